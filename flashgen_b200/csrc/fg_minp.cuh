// fg_minp.cuh — sampling with min-p beside penalties, temperature, top-k and top-p
// (fg_sample_min_p). For every row, y being the penalised logits over the temperature:
//   A    = {j : y_j >= max y + log(min_p)}, cut to the K largest (ties kept)
//   kept = A in descending order while the mass before a token is <= top_p * mass(A)
//   id   = the first kept token whose inclusive mass exceeds u * mass(kept)
// with masses e^(y_j - max y), as integers round(2^S e^(y - max y)) (S = 62 - log2 V: 2^-46
// of the largest mass at V = 128256): sums do not depend on their order, ties share one
// mass, and a decision is nearly as sharp as a 64-bit one.
//
// min-p bounds what can be drawn by the row's maximum alone. So rows_kernel reads each
// logit once, compares it with a bound that rises with the maximum seen so far and keeps
// the few that reach it; everything else is decided on those in shared memory, without a sort
// of them all: counts and masses of 1024 bins of y name the bin that holds a decision, and
// that bin's members alone are put in order. Rows whose candidates do not fit there (no
// min-p and no small top-k, or flat rows) go to wide_kernel, which does the same over whole
// rows, a cluster each.
//
// Measured (one B200, kernels alone, inputs rotated, one draw of rows and parameters each; other
// draws have other shares of flat and unbounded rows: the last two 130 to 150 and 170 to 245 as
// whole calls): 1 x 256000 fp32 18.7 us; 256 x 32000 bf16 masked, mixed parameters 61; 1024 x
// 128256 bf16 153; 512 x 128256 bf16, mixed, with histories 237. A sort of every row's candidates, 64-bit exponentials and loads to registers together
// took 1036 us for the 1024 rows, the step that replaced the three 460.
#pragma once

#include <cfloat>

#include "fg_row.cuh"

namespace fg {
namespace minp {

constexpr int NT = 256;            // threads of rows_kernel
constexpr int STAGES = 3;          // of a thread's ring of copies
constexpr int UNROLL = 3;          // 16-byte chunks of a stage
constexpr int CAP = 4096;          // candidates of a CTA's slice, and of a row
constexpr int RBINS = 1024;        // bins of their masses
constexpr int MEMBERS = 1024;      // tokens of one bin that are put in order
constexpr int MAX_K = 512;         // top-k that rows_kernel takes without min-p
constexpr int MAX_G = 16;          // CTAs that share a row
constexpr int WIDE_G = 8;          // in wide_kernel
constexpr int HIST_CAP = 4096;     // history ids of a row that rows_kernel takes
constexpr int WNT = 512;           // threads of wide_kernel
constexpr int BINS = 2048;         // of a radix step
constexpr int RING_BYTES = STAGES * UNROLL * NT * 16;
constexpr int ROW_FILTER = 2048, FILTER_WORDS = 4096;   // words of bits that say which columns may be in the history

struct Params {
    const void* logits;
    int64_t row_stride;
    int32_t batch, vocab;
    int64_t vocab_offset, vocab_total;
    const int32_t* hist_ids;
    const int64_t* hist_offsets;
    const float* temperature;
    const float* top_p;
    const int32_t* top_k;
    const float* min_p;
    const float* rep;
    const float* pres;
    const float* freq;
    const uint8_t* greedy;
    const float* uniforms;
    int64_t* out_ids;
    int32_t* out_status;
    float* out_probs;
    float* out_logprobs;
    int32_t* out_kept;
    uint8_t* marks;            // [B]: rows handed to wide_kernel
    uint2* tables;             // wide_kernel's history tables, one per cluster
    int32_t penalties;         // histories and any of the three penalties are given
    int32_t only;              // rows with min_p == 0 are left as they are
    int32_t hist_max_len;
    int32_t slots, wide_slots; // of a history table (powers of two)
    int32_t mass_shift;        // S
};

__device__ __forceinline__ void wait_prerequisites() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Cluster address of `p`'s counterpart in CTA `rank`, and loads from one.
__device__ __forceinline__ uint32_t mapa(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ uint32_t ld_cluster(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t ld_cluster64(uint32_t a) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}

// A row's parameters, the same in every thread.
struct Row {
    RowP p;
    bool greedy;
    int K;               // top-k; 0: off
    float min_p;
    int64_t h0, h1;      // its history
};
__device__ __forceinline__ Row load_row(const Params& P, int r) {
    Row row;
    row.h0 = row.h1 = 0;
    if (P.penalties) {
        row.h0 = __ldg(P.hist_offsets + r);
        row.h1 = __ldg(P.hist_offsets + r + 1);
    }
    RowP& p = row.p;
    p.T = P.temperature ? __ldg(P.temperature + r) : 1.0f;
    p.top_p = P.top_p ? __ldg(P.top_p + r) : 1.0f;
    p.u = __ldg(P.uniforms + r);
    const int k = P.top_k ? __ldg(P.top_k + r) : 0;
    row.min_p = P.min_p ? __ldg(P.min_p + r) : 0.0f;
    const bool has = row.h1 > row.h0;
    p.rep = P.rep ? __ldg(P.rep + r) : 1.0f;
    p.pres = P.pres ? __ldg(P.pres + r) : 0.0f;
    p.freq = P.freq ? __ldg(P.freq + r) : 0.0f;
    p.rep_on = has && p.rep != 1.0f;
    p.pres_on = has && p.pres != 0.0f;
    p.freq_on = has && p.freq != 0.0f;
    p.pen = p.rep_on || p.pres_on || p.freq_on;
    p.bad = 0;
    if (p.rep != p.rep || p.pres != p.pres || p.freq != p.freq) p.bad |= FG_ROW_BAD_PARAM;
    row.greedy = (P.greedy && __ldg(P.greedy + r) != 0) || p.T == 0.0f;
    if (!row.greedy) {
        if (!(p.T > 0.0f && p.T < INFINITY) || !(p.top_p > 0.0f && p.top_p <= 1.0f) ||
            !(row.min_p >= 0.0f && row.min_p <= 1.0f))
            p.bad |= FG_ROW_BAD_PARAM;
        if (!(p.u >= 0.0f && p.u < 1.0f)) p.bad |= FG_ROW_BAD_UNIFORM;
    }
    p.temp_on = !row.greedy && p.T != 1.0f;
    p.rT = p.temp_on ? __frcp_rn(p.T) : 1.0f;
    p.use_p = !row.greedy && p.top_p < 1.0f;
    p.cls = row.greedy ? RC_GREEDY : RC_FULL;
    p.K = 0;
    row.K = !row.greedy && k > 0 && k < P.vocab ? k : 0;
    return row;
}
// log(min_p): -inf without min-p, 0 for greedy rows.
__device__ __forceinline__ double log_min_p(const Row& row) {
    return row.greedy || row.min_p == 1.0f ? 0.0 : row.min_p > 0.0f ? log(double(row.min_p)) : -INFINITY;
}

__device__ __forceinline__ void write_row(const Params& P, int r, int64_t id, float logprob, int kept, uint32_t status) {
    P.out_ids[r] = id;
    if (P.out_logprobs) P.out_logprobs[r] = logprob;
    if (P.out_kept) P.out_kept[r] = kept;
    if (P.out_status) P.out_status[r] = int(status);
}
__device__ __forceinline__ void write_error(const Params& P, int r, uint32_t status) {
    write_row(P, r, -1, __int_as_float(0x7fc00000), 0, status);
}

// Masses: round(2^S e^(y - top)), right to 2^-42 of the mass. 64-bit
// exponentials at the rate of this machine's 64-bit units were the longest part of a row's
// decisions (3900 candidates: 11 us of 60), so e^d is taken in pairs of 32-bit numbers, by
// table and polynomial (P. T. P. Tang, "Table-driven implementation of the exponential
// function in IEEE floating-point arithmetic", ACM TOMS 15(2), 1989): with n the nearest
// integer to d 64 / log 2, e^d = 2^(n / 64) e^r and |r| <= log 2 / 128; the table has
// 2^(j / 64) as pairs.
struct ExpPairs {
    float v[64][2];
    constexpr ExpPairs() : v() {
        for (int j = 0; j < 64; ++j) {
            double t = 1.0, term = 1.0;   // e^x by its series, x = j log 2 / 64 < 0.69
            for (int i = 1; i < 24; ++i) {
                term *= j * (0.69314718055994530942 / 64.0) / i;
                t += term;
            }
            v[j][0] = float(t);
            v[j][1] = float(t - double(v[j][0]));
        }
    }
};
__device__ constexpr ExpPairs kExpPairs{};
struct ExpTable {   // in shared memory
    float2 v[64];
    __device__ __forceinline__ void fill() {   // by the first 64 threads
        if (threadIdx.x < 64) v[threadIdx.x] = make_float2(kExpPairs.v[threadIdx.x][0], kExpPairs.v[threadIdx.x][1]);
    }
};
__device__ __forceinline__ uint64_t mass_of(float y, float top, const ExpTable& T, int shift) {
    // d = y - top exactly, as a pair
    const float d = __fsub_rn(y, top), back = __fadd_rn(d, top);
    const float dl = __fadd_rn(__fsub_rn(y, back), __fsub_rn(__fsub_rn(back, d), top));
    if (!(d > -44.0f)) return 0;   // 2^-63
    // log 2 / 64 in three parts, of which the first two have 12 bits: n takes no more
    constexpr float kPerLog2 = 92.332482616893656877f;              // 64 / log 2
    constexpr float kC1 = 0x1.62ep-7f, kC2 = 0x1.0cp-21f, kC3 = -2.9760223436840126e-11f;
    const float n = rintf(d * kPerLog2);
    float rh = fmaf(-n, kC2, fmaf(-n, kC1, d));                     // both steps exact
    float rl = fmaf(-n, kC3, dl);
    const float sum = __fadd_rn(rh, rl);
    rl = __fadd_rn(__fsub_rn(rh, sum), rl);
    rh = sum;
    // e^r - 1 as a pair
    const float q = __fmul_rn(rh, rh), ql = fmaf(rh, rh, -q);       // r^2
    const float cubic = __fmul_rn(__fmul_rn(q, rh), fmaf(rh, fmaf(rh, 1.0f / 120.0f, 1.0f / 24.0f), 1.0f / 6.0f));
    const float half = __fmul_rn(0.5f, q);
    const float sh = __fadd_rn(rh, half);
    const float sl = __fadd_rn(__fadd_rn(__fsub_rn(half, __fsub_rn(sh, rh)), fmaf(rl, rh, rl)), fmaf(0.5f, ql, cubic));
    // 2^(n / 64) e^r in units of 2^-S: the table's part, its product's high part and the rest
    const int k = int(n), j = k & 63;
    const float2 t = T.v[j];
    const float wh = __fmul_rn(t.x, sh);
    const float wl = __fadd_rn(fmaf(t.x, sh, -wh), fmaf(t.x, sl, fmaf(t.y, sh, t.y)));
    const int e = shift + ((k - j) >> 6);                            // 62 at most
    if (e < -1) return 0;
    // a unit of the sum is 2^-(62 - e) of the result's: its bits below that are rounded once
    const float up = 0x1p62f;
    const int64_t m = __float2ll_rn(t.x * (up * 0.25f)) + __float2ll_rn(wh * (up * 0.25f)) + __float2ll_rn(wl * (up * 0.25f));
    const int down = 60 - e;                                         // m is in units of 2^-60
    return down <= 0 ? uint64_t(m) << -down : (uint64_t(m) + (uint64_t(1) << (down - 1))) >> down;
}
// The smallest key that min-p keeps below a maximum of `top`: y >= top + log(min_p) in 64 bits.
__device__ __forceinline__ uint32_t least_key(double log_min_p, float top) {
    if (!(log_min_p > -INFINITY)) return KEY_NEG_INF + 1u;
    const uint32_t k = fkey(__double2float_ru(double(top) + log_min_p));
    return k > KEY_NEG_INF ? k : KEY_NEG_INF + 1u;
}
// What of a sum stays below a share of it: floor(share * sum).
__device__ __forceinline__ uint64_t part_of(float share, uint64_t sum) {
    const uint64_t t = uint64_t(double(share) * double(sum));
    return t < sum ? t : sum - 1;
}

// ---------------------------------------------------------------------------
// History: the distinct columns of [c_lo, c_hi) with their counts, then with their
// penalised values, in an open-addressed table of (column, count or value).
// ---------------------------------------------------------------------------
__device__ __forceinline__ int find_slot(const uint2* table, uint32_t mask, uint32_t col) {
    uint32_t h = col_hash(col, mask);
    for (uint32_t i = 0; i <= mask; ++i, h = (h + 1u) & mask) {
        const uint32_t k = *reinterpret_cast<const volatile uint32_t*>(&table[h].x);
        if (k == col) return int(h);
        if (k == kEmptySlot) return -1;
    }
    return -1;
}
// Inserts the row's ids; all threads. The table is empty. Returns status bits.
template <int THREADS, int WORDS>
__device__ __forceinline__ uint32_t count_history(const Params& P, const Row& row, uint2* table, uint32_t mask,
                                                  int64_t c_lo, int64_t c_hi, uint32_t* filter) {
    uint32_t bad = 0;
    constexpr int AHEAD = 4;   // loads of ids in flight
    for (int64_t at = row.h0 + threadIdx.x; at < row.h1; at += AHEAD * THREADS) {
        int32_t ids[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) ids[j] = at + j * THREADS < row.h1 ? __ldg(P.hist_ids + at + j * THREADS) : 0;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (at + j * THREADS >= row.h1) break;
            const int64_t id = ids[j];
            if (id < 0 || id >= P.vocab_total) {
                bad |= FG_ROW_BAD_HISTORY;
                continue;
            }
            const int64_t c = id - P.vocab_offset;
            if (c < c_lo || c >= c_hi) continue;
            uint32_t h = col_hash(uint32_t(c), mask);
            bool done = false;
            for (uint32_t n = 0; n <= mask && !done; ++n) {
                const uint32_t k = atomicCAS(&table[h].x, kEmptySlot, uint32_t(c));
                done = k == kEmptySlot || k == uint32_t(c);
                if (done) atomicAdd(&table[h].y, 1u);
                h = (h + 1u) & mask;
            }
            if (!done) bad |= FG_ROW_BAD_PARAM;   // more distinct ids than hist_max_len allows
            if constexpr (WORDS > 0) {
                const uint32_t b = uint32_t(c - c_lo) & (WORDS * 32 - 1);
                atomicOr(&filter[b >> 5], 1u << (b & 31));
            }
        }
    }
    return bad;
}

// ---------------------------------------------------------------------------
// rows_kernel: one cluster of G CTAs a row, each a slice of it.
//
// Bound: HBM reads and, as 1024 x 128256 bf16 run at 2.6 TB/s in all (101 us, issue slots 38 %),
// the starts and ends of rows that no copy covers and the last flat rows. A
// 16-byte chunk costs a packed maximum and one comparison; the chunks that reach the bound, a
// few hundred of a row, are looked at element by element. The copies go through a ring in shared
// memory: the candidates leave loads to registers little L1. Three CTAs an SM. With histories
// two, and one where the caller's longest is above 2048 ids: the table is sized by that bound,
// whatever the rows have. 1024 x 128256 bf16, histories of 64 ids: 127 us a call with a bound of
// 64, 142 with 2048, 244 with 4096 (no histories: 89).
// ---------------------------------------------------------------------------
struct Shared {
    uint32_t top;        // key of the largest (penalised) logit seen
    uint32_t least;      // key of a lower bound of the K-th largest logit
    uint32_t count;      // candidates
    uint32_t count_out;  // of this slice, as the others read it
    uint32_t flags;      // row status bits
    uint32_t n;          // members of a bin
    uint32_t bin, bin_count, before_count, kth;
    uint64_t before_mass;
    double log_min_p;
    uint32_t warp[NT / 32], other[NT / 32];
    uint64_t sums[NT / 32];
};
struct Candidate {
    float x;
    uint32_t col;
};

template <int DT>
__device__ __forceinline__ float chunk_max(const uint4& q) {
    if constexpr (DT == FG_DTYPE_F32) {
        return fmax_nan(fmax_nan(__uint_as_float(q.x), __uint_as_float(q.y)),
                        fmax_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
    } else if constexpr (DT == FG_DTYPE_F16) {
        const __half2* h = reinterpret_cast<const __half2*>(&q);
        const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return fmax_nan(__low2float(m), __high2float(m));
    } else {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return fmax_nan(__low2float(m), __high2float(m));
    }
}

// Where in a chunk its largest element is (`m`, not NaN).
template <int DT>
__device__ __forceinline__ int place_of(const uint4& q, float m) {
    float x[Elem<DT>::VEC];
    Elem<DT>::unpack(q, x);
    int at = 0;
#pragma unroll
    for (int j = 1; j < Elem<DT>::VEC; ++j) at = x[j] == m ? j : at;
    return at;
}

// Counts and masses of bins, the masses as two words: 64-bit atomics on shared memory
// serialise far more.
struct Bins32 {
    uint32_t *count, *lo, *hi;
    __device__ __forceinline__ void add(uint32_t b, uint64_t m) const {
        reds_add(&count[b], 1u);
        const uint32_t l = uint32_t(m);
        uint32_t h = uint32_t(m >> 32);
        if (l) h += atoms_add(&lo[b], l) + l < l;
        if (h) reds_add(&hi[b], h);
    }
    __device__ __forceinline__ uint64_t mass(uint32_t b) const { return uint64_t(hi[b]) << 32 | lo[b]; }
};
// The bin of y below the row's maximum: of equal width down to `span` (32 at most, where a
// mass is a unit or nothing), the last one for all that lies further below. Every step is
// monotone, so bins are in the order of their keys.
__device__ __forceinline__ float bin_scale(double log_min_p, int bins) {
    return float(bins - 1) / fmaxf(1e-3f, fminf(32.0f, float(-log_min_p)));
}
__device__ __forceinline__ uint32_t bin_of(float top, float y, float scale, int bins) {
    return min(uint32_t(bins - 1), uint32_t((top - y) * scale));
}

// `n` (a power of two, at least 32) numbers in descending order, by all threads.
template <int THREADS>
__device__ __forceinline__ void sort_descending(uint64_t* v, int n) {
    for (int size = 2; size <= n; size <<= 1)
        for (int d = size >> 1; d > 0; d >>= 1) {
            for (int i = threadIdx.x; i < n / 2; i += THREADS) {
                const int a = 2 * i - (i & (d - 1)), b = a + d;
                const uint64_t x = v[a], y = v[b];
                if (((a & size) == 0) == (x < y)) {
                    v[a] = y;
                    v[b] = x;
                }
            }
            __syncthreads();
        }
}

// A bound below which no logit can be kept when the largest is `top`. The slack covers the
// roundings of x / T, of the maximum's quotient and of this product. Finite, so that -inf is below it.
__device__ __forceinline__ float bound_of(const Row& row, float top, float span) {
    return fmaxf(row.greedy ? top : top - span - 0x1p-20f * (fabsf(top) + span), -FLT_MAX);
}

__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_committed() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_done() {
    asm volatile("cp.async.wait_group %0;" :: "n"(LEFT) : "memory");
}

// Dynamic shared memory: the ring of copies (after the stream: bins and members of a bin),
// the candidates, the history's table.
template <int DT>
__global__ void __launch_bounds__(NT, 3) rows_kernel(const Params P, const int G) {
    using E = Elem<DT>;
    constexpr int VEC = E::VEC;
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ Shared S;
    __shared__ ExpTable T;
    Candidate* cand = reinterpret_cast<Candidate*>(dyn + RING_BYTES);
    uint2* table = reinterpret_cast<uint2*>(cand + CAP);
    uint32_t* filter = reinterpret_cast<uint32_t*>(table + P.slots);
    uint64_t* members = reinterpret_cast<uint64_t*>(dyn);
    Bins32 bins;
    bins.count = reinterpret_cast<uint32_t*>(members + MEMBERS);
    bins.lo = bins.count + RBINS;
    bins.hi = bins.lo + RBINS;
    static_assert(MEMBERS * 8 + RBINS * 12 <= RING_BYTES, "bins and members take the ring's place");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / G;
    const uint32_t rank = G > 1 ? cluster_rank() : 0;
    wait_prerequisites();
    launch_dependents();

    const Geom g = row_geom<E::SIZE>(P.logits, P.row_stride, P.vocab, r);
    const int nch = int(g.ibytes / 16);
    const int ch0 = int(int64_t(nch) * rank / G), ch1 = int(int64_t(nch) * (rank + 1) / G);
    const uint4* chunks = reinterpret_cast<const uint4*>(g.interior);
    const uint32_t ring = smem_u32(dyn) + 16 * tid;       // this thread's places, NT chunks apart
    // stage k of the slice: its chunks ch0 + (k UNROLL + i) NT + tid
    auto fetch = [&](int k) {
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int c = ch0 + (k * UNROLL + i) * NT + tid;
            if (c < ch1) copy_async(ring + (k % STAGES * UNROLL + i) * NT * 16, chunks + c);
        }
        copies_committed();
    };
    const int stages = (ch1 - ch0 + UNROLL * NT - 1) / (UNROLL * NT);

    // the first copies go out before anything else is known of the row
#pragma unroll
    for (int k = 0; k < STAGES; ++k) fetch(k);
    const Row row = load_row(P, r);
    if (rank == 0 && tid == 0) P.marks[r] = 0;
    // a lower bound of the K-th largest comes from K chunks of the first stages
    const bool by_k = row.K > 0 && row.K <= MAX_K;
    auto hand_on = [&]() {
        if (rank == 0 && tid == 0) P.marks[r] = 1;
    };
    if (P.only && row.min_p == 0.0f) {
        copies_done<0>();
        return;
    }
    if (row.p.bad && !P.out_probs) {
        if (rank == 0 && tid == 0) write_error(P, r, row.p.bad);
        copies_done<0>();
        return;
    }
    if (P.out_probs || (!row.greedy && row.min_p == 0.0f && !by_k) || row.h1 - row.h0 > HIST_CAP) {
        hand_on();
        copies_done<0>();
        return;
    }
    const bool first = rank == 0, last = int(rank) == G - 1;
    const int c_lo = first ? 0 : g.head + ch0 * VEC, c_hi = last ? P.vocab : g.head + ch1 * VEC;
    const uint32_t mask = uint32_t(P.slots) - 1u;
    const bool pen = row.p.pen;
    T.fill();
    if (tid == 0) {
        S.top = KEY_NEG_INF;
        S.least = KEY_NEG_INF;
        S.count = 0;
        S.flags = 0;
        S.log_min_p = log_min_p(row);   // (64 bits, by one thread: a microsecond of every thread's otherwise)
    }
    if (pen) {
        for (int i = tid; i <= int(mask); i += NT) table[i] = make_uint2(kEmptySlot, 0u);
        for (int i = tid; i < ROW_FILTER; i += NT) filter[i] = 0u;
    }
    __syncthreads();
    if (pen) {
        const uint32_t bad = count_history<NT, ROW_FILTER>(P, row, table, mask, c_lo, c_hi, filter);
        if (bad) atomicOr(&S.flags, bad);
        __syncthreads();
        uint32_t top = KEY_NEG_INF;
        constexpr int AHEAD = 8;   // loads of logits in flight
        for (int base = tid; base <= int(mask); base += AHEAD * NT) {
            uint2 e[AHEAD];
            float x[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                e[j] = base + j * NT <= int(mask) ? table[base + j * NT] : make_uint2(kEmptySlot, 0u);
                x[j] = e[j].x != kEmptySlot ? E::load(g.row, e[j].x) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (e[j].x == kEmptySlot) continue;
                const float v = penalize(row.p, x[j], e[j].y);
                table[base + j * NT].y = __float_as_uint(v);
                if (v != v) atomicOr(&S.flags, uint32_t(FG_ROW_NAN));
                else top = max(top, fkey(v));
            }
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) atomicMax(&S.top, top);
    }
    auto in_history = [&](uint32_t col) {
        if (!pen) return false;
        const uint32_t b = (col - uint32_t(c_lo)) & (ROW_FILTER * 32 - 1);
        return (filter[b >> 5] >> (b & 31) & 1u) != 0u && find_slot(table, mask, col) >= 0;
    };
    const float span = row.greedy ? 0.0f : -logf(row.min_p) * row.p.T;

    // the maximum of the ring's first filling, over what is not in the history
    constexpr int HELD = STAGES * UNROLL;
    {
        copies_done<0>();
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int c = ch0 + i * NT + tid;
            if (c >= ch1) break;
            const uint4 q = lds_v4(ring + i * NT * 16);
            const float m = chunk_max<DT>(q);
            if (!(m > top)) continue;
            // (a chunk whose largest is in the history counts for none: the stream sees to the rest of it)
            if (!pen || !in_history(uint32_t(g.head + c * VEC + place_of<DT>(q, m)))) top = m;
        }
        const uint32_t key = __reduce_max_sync(0xffffffffu, fkey(top));
        if (lane == 0) atomicMax(&S.top, key);
        __syncthreads();
        if (by_k) {
            // the largest key, to 2^-17 of its range, that K chunks of the ring reach: the K-th
            // largest logit is no smaller. A chunk whose largest is in the history counts for none
            uint32_t key_of[HELD];
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                const int c = ch0 + i * NT + tid;
                key_of[i] = 0u;
                if (c >= ch1) continue;
                const uint4 q = lds_v4(ring + i * NT * 16);
                const float m = chunk_max<DT>(q);
                if (m == m && (!pen || !in_history(uint32_t(g.head + c * VEC + place_of<DT>(q, m))))) key_of[i] = fkey(m);
            }
            uint32_t lo = KEY_NEG_INF, hi = S.top;
            for (int step = 0; step < 17 && hi > lo; ++step) {
                const uint32_t mid = lo + (hi - lo + 1) / 2;
                uint32_t n = 0;
#pragma unroll
                for (int i = 0; i < HELD; ++i) n += key_of[i] >= mid;
                n = __reduce_add_sync(0xffffffffu, n);
                uint32_t* sums = step & 1 ? S.warp : S.other;   // by turns: one barrier a step
                if (lane == 0) sums[warp] = n;
                __syncthreads();
                n = 0;
#pragma unroll
                for (int w = 0; w < NT / 32; ++w) n += sums[w];
                if (n >= uint32_t(row.K)) lo = mid;
                else hi = mid - 1;
            }
            if (tid == 0) S.least = lo;
            __syncthreads();
        }
    }

    float seen = -INFINITY, bound = -INFINITY;   // the largest logit known here; what it bounds
    // (the K-th largest's ties after the division may lie a rounding below it)
    auto with_k = [&](uint32_t key) {
        const float x = funkey(key);
        if (by_k && x > -INFINITY) bound = fmaxf(bound, x - 0x1p-20f * fabsf(x));
    };
    // the logits of a warp, one a lane, that are not below the bound (or NaN) become candidates
    auto take = [&](float x, uint32_t col, bool in) {
        if (in && !(x > -INFINITY)) {
            if (x != x && !in_history(col)) atomicOr(&S.flags, uint32_t(FG_ROW_NAN));
            in = false;
        }
        in = in && !in_history(col);
        const uint32_t who = __ballot_sync(0xffffffffu, in);
        if (who == 0) return;
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&S.count, __popc(who));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
        if (in && at < uint32_t(CAP)) cand[at] = {x, col};
        if (__any_sync(0xffffffffu, in && x > seen)) {
            const uint32_t key = __reduce_max_sync(0xffffffffu, in ? fkey(x) : 0u);
            if (lane == 0) atomicMax(&S.top, key);
        }
    };
    // A thread's chunks of a stage, in the ring from `place` on (the first is chunk c0, the others
    // NT chunks apart): their elements that reach the bound take places together, and come out of
    // the ring one by one, so that a warp's steps are those of its busiest lane. Columns of the
    // history and NaN leave -inf in their places.
    auto scan = [&](uint32_t place, int c0) {
        uint32_t mine = 0;               // VEC bits a chunk
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const uint4 q = lds_v4(place + i * NT * 16);
            if (c0 + i * NT >= ch1 || chunk_max<DT>(q) < bound) continue;
            float x[VEC];
            E::unpack(q, x);
#pragma unroll
            for (int j = 0; j < VEC; ++j) mine |= uint32_t(!(x[j] < bound)) << (i * VEC + j);
        }
        if (mine == 0u) return;
        uint32_t at = atomicAdd(&S.count, uint32_t(__popc(mine)));
        float most = -INFINITY;
        do {
            const int b = __ffs(mine) - 1, i = b / VEC, j = b % VEC;
            mine &= mine - 1u;
            const uint32_t from = place + i * NT * 16 + j * E::SIZE, col = uint32_t(g.head + (c0 + i * NT) * VEC + j);
            float x;
            if constexpr (DT == FG_DTYPE_F32) x = __uint_as_float(lds_u32(from));
            else if constexpr (DT == FG_DTYPE_F16) x = __half2float(__ushort_as_half(uint16_t(lds_u16(from))));
            else x = __uint_as_float(lds_u16(from) << 16);
            if (in_history(col)) x = -INFINITY;
            if (x != x) {
                atomicOr(&S.flags, uint32_t(FG_ROW_NAN));
                x = -INFINITY;
            }
            most = fmaxf(most, x);
            if (at < uint32_t(CAP)) cand[at] = {x, col};
            ++at;
        } while (mine);
        if (most > seen) atomicMax(&S.top, fkey(most));
    };
    static_assert(UNROLL * VEC <= 32, "a bit for each element of a stage");
    // columns [lo, hi) one by one (fewer than a chunk), by the first warp
    auto scan_columns = [&](int lo, int hi) {
        if (warp != 0) return;
        for (int c = lo; c < hi; c += 32) {
            const bool in = c + lane < hi;
            const float x = in ? E::load(g.row, c + lane) : 0.0f;
            take(x, uint32_t(c + lane), in && !(x < bound));
        }
    };
    auto scan_ragged = [&]() {
        if (first) scan_columns(0, g.head);
        if (last) scan_columns(g.tail0, P.vocab);
    };
    uint32_t top_key = 0, flags = 0;
    bool sick = false, flat = false;
    // A second pass where too many logits reached the bounds of their moments: with the final
    // bound (from L2)
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        if (pass == 0) {
            seen = funkey(S.top);
            bound = bound_of(row, seen, span);
            with_k(S.least);
        }
#pragma unroll 1
        for (int k = 0; k < stages; ++k) {
            copies_done<STAGES - 1>();
            if (pass == 0) {
                seen = funkey(*reinterpret_cast<volatile uint32_t*>(&S.top));
                bound = bound_of(row, seen, span);
                with_k(S.least);
                // a flat row: too many before half of it, when the bound has hardly risen any more
                flat = 2 * k < stages && *reinterpret_cast<volatile uint32_t*>(&S.count) > 3u * CAP / 2u;
                if (flat) break;
            }
            scan(ring + k % STAGES * (UNROLL * NT * 16), ch0 + k * UNROLL * NT + tid);
            fetch(k + STAGES);   // (past the slice: an empty group, which keeps the count)
        }
        scan_ragged();
        copies_done<0>();
        __syncthreads();
        if (pass == 1) break;
        // the whole row's maximum and flags
        top_key = S.top;
        flags = S.flags;
        uint32_t least = S.least;
        if (G > 1) {
            cluster_sync();
            const uint32_t peer = uint32_t(min(lane, G - 1));
            top_key = __reduce_max_sync(0xffffffffu, ld_cluster(mapa(&S.top, peer)));
            least = __reduce_max_sync(0xffffffffu, ld_cluster(mapa(&S.least, peer)));
            flags = __reduce_or_sync(0xffffffffu, ld_cluster(mapa(&S.flags, peer)));
            // (S.top and S.flags stay as they are until the last cluster_sync)
        }
        sick = (flags & FG_ROW_NAN) || top_key <= KEY_NEG_INF || !(funkey(top_key) < INFINITY);
        seen = INFINITY;                          // from here on nothing raises the maximum
        bound = bound_of(row, funkey(top_key), span);
        with_k(least);
        // (what a slice without the end of its stream knows of the row does not matter: it is handed on)
        flat = __syncthreads_or(flat);
        const bool over = S.count > uint32_t(CAP);
        if (!over || sick || flat) break;
        __syncthreads();
        if (tid == 0) S.count = 0;
#pragma unroll
        for (int k = 0; k < STAGES; ++k) fetch(k);
        __syncthreads();
    }
    const float top_x = funkey(top_key);
    __syncthreads();
    if (pen && !sick) {
        for (int i = tid; i <= int(mask); i += NT) {
            const float x = __uint_as_float(table[i].y);
            if (table[i].x == kEmptySlot || !(x >= bound) || !(x > -INFINITY)) continue;
            const uint32_t at = atomicAdd(&S.count, 1u);
            if (at < uint32_t(CAP)) cand[at] = {x, table[i].x};
        }
        __syncthreads();
    }
    constexpr uint32_t FLAT = 0xffffffffu;        // this slice's stream was not gone through
    if (tid == 0) S.count_out = flat ? FLAT : S.count;
    __syncthreads();
    if (G > 1) cluster_sync();                    // every slice's candidates stand
    const uint32_t slice_count = lane < G ? (G > 1 ? ld_cluster(mapa(&S.count_out, uint32_t(lane))) : S.count_out) : 0u;
    const bool over = __any_sync(0xffffffffu, slice_count > uint32_t(CAP));
    if (__any_sync(0xffffffffu, slice_count == FLAT)) sick = false;   // what is known of the row is not all of it

    // greedy rows with NaN or without a finite maximum: wide_kernel knows their first place
    const bool wide = (sick && row.greedy) || (!sick && over);
    // (finite logits may divide to an infinity: the divided maximum says what the row has)
    const float top = ydiv(row.p, top_x);
    const uint32_t errors = (flags & (FG_ROW_NAN | FG_ROW_BAD_PARAM)) |
                            (flags & FG_ROW_NAN ? 0u : top == -INFINITY    ? uint32_t(FG_ROW_ALL_MASKED)
                                                     : !(top < INFINITY) ? uint32_t(FG_ROW_POS_INF) : 0u);
    const bool decide = !wide && !(flags & FG_ROW_BAD_PARAM) && (row.greedy || !errors);
    const uint32_t least_k = row.greedy ? top_key : least_key(S.log_min_p, top);
    if (G > 1) {
        // the other slices' candidates come to the first CTA, by a warp each
        for (int peer = warp; peer < G; peer += NT / 32) {
            const uint32_t n = __shfl_sync(0xffffffffu, slice_count, peer);
            if (rank != 0 || !decide || peer == 0) continue;
            const uint32_t src = mapa(cand, uint32_t(peer));
            for (uint32_t j = lane; j < n; j += 32) {
                const uint64_t c = ld_cluster64(src + 8 * j);   // {x, col}
                if (fkey(ydiv(row.p, __uint_as_float(uint32_t(c)))) < least_k) continue;
                const uint32_t at = atomicAdd(&S.count, 1u);
                if (at < uint32_t(CAP)) cand[at] = {__uint_as_float(uint32_t(c)), uint32_t(c >> 32)};
            }
        }
        cluster_sync();                           // nobody leaves while its candidates may be read
    }
    if (rank == 0) {
        if (wide) {
            hand_on();
        } else if (!decide) {
            if (tid == 0) write_error(P, r, flags | errors);
        } else {
            // ---- the keys of all candidates
            for (int i = tid; i < RBINS; i += NT) bins.count[i] = bins.lo[i] = bins.hi[i] = 0u;
            __syncthreads();
            const int n = int(S.count);
            uint64_t* keys = reinterpret_cast<uint64_t*>(cand);      // in place: key, ~column; 0: not kept
            const float per_bin = bin_scale(S.log_min_p, RBINS);
            const uint32_t status = flags | (row.greedy ? uint32_t(FG_ROW_GREEDY) : 0u);
            if (n > CAP) {
                hand_on();
            } else if (row.greedy) {
                uint32_t col = 0xffffffffu;
                for (int i = tid; i < n; i += NT)
                    if (fkey(cand[i].x) == top_key) col = min(col, cand[i].col);
                col = __reduce_min_sync(0xffffffffu, col);
                if (lane == 0) S.warp[warp] = col;
                __syncthreads();
                if (tid == 0) {
                    for (int w = 1; w < NT / 32; ++w) col = min(col, S.warp[w]);
                    write_row(P, r, int64_t(col), 0.0f, 1, status);
                }
            } else {
                for (int i = tid; i < n; i += NT) {
                    const Candidate c = cand[i];
                    const float y = ydiv(row.p, c.x);
                    const uint32_t key = fkey(y);
                    keys[i] = key < least_k ? 0 : uint64_t(key) << 32 | uint32_t(~c.col);
                    if (key >= least_k)
                        bins.add(bin_of(top, y, per_bin, RBINS), mass_of(y, top, T, P.mass_shift));
                }
                __syncthreads();
                // each thread PB neighbouring bins and what lies above them
                constexpr int PB = RBINS / NT;
                uint64_t bm[PB], above_m = 0, all = 0;
                uint32_t bn[PB], above_n = 0, count = 0;
#pragma unroll
                for (int j = 0; j < PB; ++j) {
                    bm[j] = bins.mass(tid * PB + j);
                    bn[j] = bins.count[tid * PB + j];
                    above_m += bm[j];
                    above_n += bn[j];
                }
                {
                    const uint64_t im = warp_incl_scan_u64(above_m, lane);
                    const uint32_t in = warp_incl_scan_u32(above_n, lane);
                    if (lane == 31) {
                        S.sums[warp] = im;
                        S.warp[warp] = in;
                    }
                    __syncthreads();
                    above_m = im - above_m;
                    above_n = in - above_n;
#pragma unroll
                    for (int w = 0; w < NT / 32; ++w) {
                        if (w < warp) {
                            above_m += S.sums[w];
                            above_n += S.warp[w];
                        }
                        all += S.sums[w];
                        count += S.warp[w];
                    }
                    __syncthreads();
                }
                // The members of the bin in which the count or mass from the top passes `target`, with
                // their places in descending order: a few by counting what lies above each of them,
                // more by sorting. False where there are too many.
                constexpr int PM = MEMBERS / NT;
                uint64_t mk[PM], mm[PM], mb[PM];  // this thread's members, their masses, the mass before each
                int mi[PM];                       // their places in the bin; -1: none
                auto open_bin = [&](bool by_mass, uint64_t target, uint32_t floor_key) {
                    uint64_t m = above_m;
                    uint32_t c = above_n;
#pragma unroll
                    for (int j = 0; j < PB; ++j) {
                        const uint64_t from = by_mass ? m : c, to = from + (by_mass ? bm[j] : bn[j]);
                        if (from <= target && target < to) {
                            S.bin = tid * PB + j;
                            S.bin_count = bn[j];
                            S.before_mass = m;
                            S.before_count = c;
                        }
                        m += bm[j];
                        c += bn[j];
                    }
                    if (tid == 0) S.n = 0;
                    __syncthreads();
                    if (S.bin_count > uint32_t(MEMBERS)) return false;
                    const uint32_t b = S.bin;
                    for (int i = tid; i < n; i += NT) {
                        const uint64_t k = keys[i];
                        if (uint32_t(k >> 32) < floor_key || k == 0) continue;
                        if (bin_of(top, funkey(uint32_t(k >> 32)), per_bin, RBINS) == b)
                            members[atomicAdd(&S.n, 1u)] = k;
                    }
                    __syncthreads();
                    const int have = int(S.n);
#pragma unroll
                    for (int j = 0; j < PM; ++j) mi[j] = -1;
                    if (have <= 64) {
                        uint64_t* masses = members + 64;
                        if (tid < have) {
                            mk[0] = members[tid];
                            masses[tid] = mm[0] = mass_of(funkey(uint32_t(mk[0] >> 32)), top, T, P.mass_shift);
                        }
                        __syncthreads();
                        if (tid < have) {
                            mb[0] = S.before_mass;
                            mi[0] = 0;
                            for (int i = 0; i < have; ++i)
                                if (members[i] > mk[0]) {
                                    ++mi[0];
                                    mb[0] += masses[i];
                                }
                        }
                        return true;
                    }
                    int room = 128;
                    while (room < have) room <<= 1;
                    for (int i = have + tid; i < room; i += NT) members[i] = 0;
                    __syncthreads();
                    sort_descending<NT>(members, room);
                    uint64_t sum = 0;
#pragma unroll
                    for (int j = 0; j < PM; ++j) {
                        const int i = tid * PM + j;
                        if (i < have) {
                            mi[j] = i;
                            mk[j] = members[i];
                            mm[j] = mass_of(funkey(uint32_t(mk[j] >> 32)), top, T, P.mass_shift);
                            sum += mm[j];
                        }
                    }
                    const uint64_t im = warp_incl_scan_u64(sum, lane);
                    if (lane == 31) S.sums[warp] = im;
                    __syncthreads();
                    uint64_t before = S.before_mass + im - sum;
                    for (int w = 0; w < warp; ++w) before += S.sums[w];
#pragma unroll
                    for (int j = 0; j < PM; ++j)
                        if (mi[j] >= 0) {
                            mb[j] = before;
                            before += mm[j];
                        }
                    __syncthreads();
                    return true;
                };
                // what lies above the bin and the members that `in` says: their number and mass
                auto count_members = [&](auto in, uint32_t& number, uint64_t& mass) {
                    uint32_t c = 0;
                    uint64_t m = 0;
#pragma unroll
                    for (int j = 0; j < PM; ++j)
                        if (mi[j] >= 0 && in(mk[j], mb[j])) {
                            ++c;
                            m += mm[j];
                        }
                    c = __reduce_add_sync(0xffffffffu, c);
                    m = warp_incl_scan_u64(m, lane);
                    if (lane == 31) {
                        S.sums[warp] = m;
                        S.warp[warp] = c;
                    }
                    __syncthreads();
                    number = S.before_count;
                    mass = S.before_mass;
                    for (int w = 0; w < NT / 32; ++w) {
                        number += S.warp[w];
                        mass += S.sums[w];
                    }
                    __syncthreads();
                };
                bool fits = true;
                uint32_t floor_key = least_k;
                if (row.K > 0 && uint32_t(row.K) < count) {
                    fits = open_bin(false, uint64_t(row.K - 1), floor_key);
                    if (fits) {
#pragma unroll
                        for (int j = 0; j < PM; ++j)
                            if (mi[j] >= 0 && int(S.before_count) + mi[j] == row.K - 1) S.kth = uint32_t(mk[j] >> 32);
                        __syncthreads();
                        floor_key = S.kth;
                        count_members([&](uint64_t k, uint64_t) { return uint32_t(k >> 32) >= floor_key; }, count, all);
                    }
                }
                uint64_t kept = all;
                if (fits && row.p.use_p) {
                    const uint64_t limit = part_of(row.p.top_p, all);
                    fits = open_bin(true, limit, floor_key);
                    if (fits) count_members([&](uint64_t, uint64_t before) { return before <= limit; }, count, kept);
                }
                const uint64_t target = fits ? part_of(row.p.u, kept) : 0;
                fits = fits && open_bin(true, target, floor_key);
                if (fits) {
#pragma unroll
                    for (int j = 0; j < PM; ++j)
                        if (mi[j] >= 0 && mb[j] <= target && target < mb[j] + mm[j]) {
                            const double y = double(funkey(uint32_t(mk[j] >> 32))) - double(top);
                            const double sum = double(kept) / double(uint64_t(1) << P.mass_shift);
                            write_row(P, r, int64_t(~uint32_t(mk[j])), float(y - log(sum)), int(count), status);
                        }
                } else {
                    hand_on();
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// wide_kernel: the rows that rows_kernel has marked, one after the other on clusters of G
// CTAs, each a slice of the row. The first pass leaves the order-preserving key of every y in
// shared memory (CACHED; where a slice does not fit, every pass works them out anew). Counts
// and masses of all that min-p keeps go into 2048 bins of y, summed over the cluster through
// distributed shared memory; each decision then looks for its bin and puts that bin's
// members in order, or, where many share it (ties), searches by their keys' bits.
// ---------------------------------------------------------------------------
struct WideShared {
    uint32_t red32[WNT / 32];
    uint64_t red64[WNT / 32];
    uint32_t top, arg, nan_col, flags;   // this CTA's, read by the others
    uint16_t rows[WNT];
    uint32_t ties;
    uint32_t n;                          // members that this CTA has found, read by the first
    uint32_t bin, before_count, at_count;
    uint64_t before_mass, at_mass;
    uint32_t key, found_count, found_at; // a search's result, read from the first CTA
    uint64_t found_mass;
    uint32_t first;                      // place of the key's first member
};
// The bins of one step: this CTA's, its share of the cluster's, and all of the cluster's
// (of the steps by keys, and of the first one, which every search of the row begins with).
struct Bins {
    Bins32 mine;
    uint64_t* own_mass;
    uint64_t* all_mass;
    uint64_t* top_mass;
    uint32_t* own_count;
    uint32_t* all_count;
    uint32_t* top_count;
};
constexpr int bins_bytes(int G) { return 12 * (3 * BINS + BINS / G); }
constexpr int KEY_PAD = 16;              // keys that a cache has beside a slice's

// What a search has found: a key, the columns that share it and what lies above it.
struct Found {
    uint32_t key;
    uint64_t before_mass, at_mass;
    uint32_t before_count, at_count;
};

// This CTA's slice of a row, and its keys.
template <int DT, bool CACHED>
struct Slice {
    using E = Elem<DT>;
    static constexpr int VEC = E::VEC;
    const Row& row;
    Geom g;
    int ch0, ch1, c_lo, c_hi;
    bool first, last;
    const uint2* table;      // the history, and which columns may be in it
    uint32_t mask;
    const uint32_t* filter;
    uint32_t* cache;         // key of column c at c - c_lo + skew: the chunks' keys on 16-byte boundaries
    int skew;

    // (greedy rows: of the penalised logit itself)
    __device__ __forceinline__ uint32_t key_of(int c, float x, bool& nan) const {
        if (!CACHED && row.p.pen) {
            const uint32_t b = uint32_t(c - c_lo) & (FILTER_WORDS * 32 - 1);
            if (filter[b >> 5] >> (b & 31) & 1u) {
                const int at = find_slot(table, mask, uint32_t(c));
                if (at >= 0) x = penalize(row.p, x, *reinterpret_cast<const volatile uint32_t*>(&table[at].y));
            }
        }
        nan = x != x;
        return nan ? 0u : fkey(ydiv(row.p, x));
    }
    // The logits' keys, eight (four) at a time and the ragged ones one by one: f(column, n, keys, which are NaN).
    template <class F>
    __device__ __forceinline__ void read(F f) const {
        const int ragged = (first ? g.head : 0) + (last ? c_hi - g.tail0 : 0), heads = first ? g.head : 0;
        if (int(threadIdx.x) < ragged) {    // fewer than a warp's lanes
            const int c = int(threadIdx.x) < heads ? int(threadIdx.x) : g.tail0 + int(threadIdx.x) - heads;
            bool nan;
            uint32_t k[VEC];
            k[0] = key_of(c, E::load(g.row, c), nan);
            f(c, 1, k, nan ? 1u : 0u);
        }
        const uint4* chunks = reinterpret_cast<const uint4*>(g.interior);
        for (int b = ch0; b < ch1; b += 4 * WNT) {
            uint4 q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int ch = b + i * WNT + int(threadIdx.x);
                if (ch < ch1) q[i] = __ldg(chunks + ch);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int ch = b + i * WNT + int(threadIdx.x);
                if (ch >= ch1) continue;
                float x[VEC];
                E::unpack(q[i], x);
                uint32_t k[VEC], nans = 0;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    bool nan;
                    k[j] = key_of(g.head + ch * VEC + j, x[j], nan);
                    nans |= uint32_t(nan) << j;
                }
                f(g.head + ch * VEC, VEC, k, nans);
            }
        }
    }
    // f(column, key) for every column of the slice (CACHED: after `read` has filled the cache)
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        if constexpr (CACHED) {
#pragma unroll 4
            for (int c = c_lo + int(threadIdx.x); c < c_hi; c += WNT) f(c, cache[c - c_lo + skew]);
        } else {
            read([&](int c, int n, const uint32_t* k, uint32_t) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (j < n) f(c + j, k[j]);
            });
        }
    }
    __device__ __forceinline__ uint32_t key_at(int c) const {
        if constexpr (CACHED) return cache[c - c_lo + skew];
        bool nan;
        return key_of(c, E::load(g.row, c), nan);
    }
};

// The cluster's counts and masses by `bin` (below 0: not counted), in every CTA.
template <class S_, class F>
__device__ __forceinline__ void fill_bins(const S_& slice, const Bins& B, int G, int rank, F bin, float top,
                                          const ExpTable& T, int shift, uint64_t* all_mass, uint32_t* all_count) {
    const int tid = threadIdx.x, per = BINS / G;
    for (int i = tid; i < BINS; i += WNT) B.mine.count[i] = B.mine.lo[i] = B.mine.hi[i] = 0u;
    __syncthreads();
    slice.each([&](int, uint32_t k) {
        const int b = bin(k);
        if (b >= 0) B.mine.add(uint32_t(b), mass_of(funkey(k), top, T, shift));
    });
    cluster_sync();
    for (int i = tid; i < per; i += WNT) {
        const int at = rank * per + i;
        uint32_t lo[WIDE_G], hi[WIDE_G], n[WIDE_G];
#pragma unroll
        for (int c = 0; c < WIDE_G; ++c) {
            lo[c] = c < G ? ld_cluster(mapa(&B.mine.lo[at], c)) : 0u;
            hi[c] = c < G ? ld_cluster(mapa(&B.mine.hi[at], c)) : 0u;
            n[c] = c < G ? ld_cluster(mapa(&B.mine.count[at], c)) : 0u;
        }
        uint64_t m = 0;
        uint32_t count = 0;
#pragma unroll
        for (int c = 0; c < WIDE_G; ++c) {
            m += uint64_t(hi[c]) << 32 | lo[c];
            count += n[c];
        }
        B.own_mass[i] = m;
        B.own_count[i] = count;
    }
    cluster_sync();
#pragma unroll
    for (int j = 0; j < BINS / WNT; ++j) {
        const int i = j * WNT + tid;
        all_mass[i] = ld_cluster64(mapa(&B.own_mass[i % per], i / per));
        all_count[i] = ld_cluster(mapa(&B.own_count[i % per], i / per));
    }
    __syncthreads();
}
// The first bin up to whose end the count or mass passes `target`, f being what lies before the
// bins; f is then what lies before that bin, and the bin's own.
__device__ __forceinline__ uint32_t locate(WideShared& S, Found& f, bool by_mass, uint64_t target,
                                           const uint64_t* all_mass, const uint32_t* all_count) {
    constexpr int PB = BINS / WNT;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint64_t m[PB], sm = 0;
    uint32_t n[PB], sn = 0;
#pragma unroll
    for (int j = 0; j < PB; ++j) {
        m[j] = all_mass[tid * PB + j];
        n[j] = all_count[tid * PB + j];
        sm += m[j];
        sn += n[j];
    }
    const uint64_t im = warp_incl_scan_u64(sm, lane);
    const uint32_t in = warp_incl_scan_u32(sn, lane);
    if (lane == 31) {
        S.red64[warp] = im;
        S.red32[warp] = in;
    }
    __syncthreads();
    uint64_t bm = f.before_mass + im - sm;
    uint32_t bn = f.before_count + in - sn;
#pragma unroll
    for (int w = 0; w < WNT / 32; ++w)
        if (w < warp) {
            bm += S.red64[w];
            bn += S.red32[w];
        }
#pragma unroll
    for (int j = 0; j < PB; ++j) {
        const uint64_t from = by_mass ? bm : bn, to = from + (by_mass ? m[j] : n[j]);
        if (from <= target && target < to) {
            S.bin = uint32_t(tid * PB + j);
            S.before_mass = bm;
            S.before_count = bn;
            S.at_mass = m[j];
            S.at_count = n[j];
        }
        bm += m[j];
        bn += n[j];
    }
    __syncthreads();
    f.before_mass = S.before_mass;
    f.before_count = S.before_count;
    f.at_mass = S.at_mass;
    f.at_count = S.at_count;
    const uint32_t b = S.bin;
    __syncthreads();
    return b;
}
// The n-th column, in ascending order, that has key k, in every CTA.
template <class S_>
__device__ __forceinline__ uint32_t column_of(const S_& slice, WideShared& S, int G, int rank, uint32_t k, uint32_t n) {
    // each thread a run of the slice's neighbours
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = slice.c_hi - slice.c_lo, step = (len + WNT - 1) / WNT;
    const int a = slice.c_lo + min(len, tid * step), z = min(slice.c_hi, a + step);
    uint32_t ties = 0;
    for (int c = a; c < z; ++c) ties += slice.key_at(c) == k;
    const uint32_t upto = warp_incl_scan_u32(ties, lane);
    if (lane == 31) S.red32[warp] = upto;
    __syncthreads();
    uint32_t before = upto - ties, mine = 0;
    for (int w = 0; w < WNT / 32; ++w) {
        if (w < warp) before += S.red32[w];
        mine += S.red32[w];
    }
    if (tid == 0) {
        S.ties = mine;
        S.bin = 0xffffffffu;
    }
    cluster_sync();
    for (int c = 0; c < rank; ++c) before += ld_cluster(mapa(&S.ties, c));
    if (before <= n && n < before + ties) {
        uint32_t left = n - before;
        for (int c = a; c < z; ++c)
            if (slice.key_at(c) == k && left-- == 0) {
                S.bin = uint32_t(c);
                break;
            }
    }
    cluster_sync();
    uint32_t col = lane < G ? ld_cluster(mapa(&S.bin, lane)) : 0xffffffffu;
    col = __reduce_min_sync(0xffffffffu, col);
    cluster_sync();
    return col;
}

template <int DT, bool CACHED>
__global__ void __launch_bounds__(WNT, 1) wide_kernel(const Params P, const int G) {
    using E = Elem<DT>;
    constexpr int VEC = E::VEC;
    constexpr int NW = WNT / 32;
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ WideShared S;
    __shared__ ExpTable T;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = int(cluster_rank());
    const int per = BINS / G;
    uint64_t* members = reinterpret_cast<uint64_t*>(dyn);   // of a bin: this CTA's, and in the first CTA all
    uint64_t* all_members = members + MEMBERS;
    Bins B;
    B.all_mass = all_members + MEMBERS;
    B.top_mass = B.all_mass + BINS;
    B.own_mass = B.top_mass + BINS;
    B.mine.count = reinterpret_cast<uint32_t*>(B.own_mass + per);
    B.mine.lo = B.mine.count + BINS;
    B.mine.hi = B.mine.lo + BINS;
    B.all_count = B.mine.hi + BINS;
    B.top_count = B.all_count + BINS;
    B.own_count = B.top_count + BINS;
    uint32_t* filter = B.own_count + per;
    uint32_t* cache = filter;   // (one or the other)
    T.fill();
    wait_prerequisites();
    uint2* table = P.tables + int64_t(blockIdx.x / G) * P.wide_slots;
    const uint32_t mask = uint32_t(P.wide_slots) - 1u;

    // the marked rows, in ascending order, by turns to the clusters
    const int clusters = gridDim.x / G, mine_of = blockIdx.x / G;
    int marked = 0;   // so far
    for (int base = 0; base < P.batch; base += WNT) {
        const bool mark = base + tid < P.batch && P.marks[base + tid] != 0;
        const uint32_t vote = __ballot_sync(0xffffffffu, mark);
        __syncthreads();
        if (lane == 0) S.red32[warp] = __popc(vote);
        __syncthreads();
        int at = __popc(vote & ((1u << lane) - 1u)), found = 0;
        for (int w = 0; w < NW; ++w) {
            if (w < warp) at += int(S.red32[w]);
            found += int(S.red32[w]);
        }
        if (mark) S.rows[at] = uint16_t(tid);
        __syncthreads();
        // the first of them whose turn is this cluster's
        int item = (mine_of - marked % clusters + clusters) % clusters;
        marked += found;
        for (; item < found; item += clusters) {
            const int r = base + S.rows[item];
            const Row row = load_row(P, r);
            const Geom g = row_geom<E::SIZE>(P.logits, P.row_stride, P.vocab, r);
            const int nch = int(g.ibytes / 16);
            Slice<DT, CACHED> slice{row, g};
            slice.ch0 = int(int64_t(nch) * rank / G);
            slice.ch1 = int(int64_t(nch) * (rank + 1) / G);
            slice.first = rank == 0;
            slice.last = rank == G - 1;
            slice.c_lo = slice.first ? 0 : g.head + slice.ch0 * VEC;
            slice.c_hi = slice.last ? P.vocab : g.head + slice.ch1 * VEC;
            slice.table = table;
            slice.mask = mask;
            slice.filter = filter;
            slice.cache = cache;
            slice.skew = slice.first ? (VEC - g.head % VEC) % VEC : 0;
            const bool pen = row.p.pen;

            if (tid == 0) {
                S.flags = 0;
                S.top = KEY_NEG_INF;
                S.arg = 0xffffffffu;
                S.nan_col = 0xffffffffu;
            }
            if (pen) {
                // the cluster shares one table; its CTAs insert and look up columns of their own
                for (int i = rank * WNT + tid; i <= int(mask); i += G * WNT) table[i] = make_uint2(kEmptySlot, 0u);
                if constexpr (!CACHED)
                    for (int i = tid; i < FILTER_WORDS; i += WNT) filter[i] = 0u;
            }
            cluster_sync();
            if (pen) {
                const uint32_t bad = count_history<WNT, CACHED ? 0 : FILTER_WORDS>(P, row, table, mask, slice.c_lo,
                                                                                  slice.c_hi, filter);
                if (bad) atomicOr(&S.flags, bad);
                __syncthreads();
            }
            // ---- keys, the maximum and its first column, the first NaN
            {
                uint32_t top = KEY_NEG_INF, arg = 0xffffffffu, nan_col = 0xffffffffu;
                auto meet = [&](int c, uint32_t k, bool nan) {
                    if (nan) nan_col = min(nan_col, uint32_t(c));
                    else if (k > top || (k == top && uint32_t(c) < arg)) {
                        top = k;
                        arg = uint32_t(c);
                    }
                };
                if constexpr (CACHED) {
                    // all columns' keys (0: NaN), then the history's over them
                    slice.read([&](int c, int n, const uint32_t* k, uint32_t) {
                        uint32_t* to = cache + (c - slice.c_lo + slice.skew);
                        if (n == VEC) {
#pragma unroll
                            for (int j = 0; j < VEC; j += 4)
                                *reinterpret_cast<uint4*>(to + j) = make_uint4(k[j], k[j + 1], k[j + 2], k[j + 3]);
                        } else {
                            to[0] = k[0];
                        }
                    });
                    __syncthreads();
                    if (pen) {
                        for (int i = tid; i <= int(mask); i += WNT) {
                            const uint2 e = __ldcg(table + i);
                            if (e.x == kEmptySlot || int(e.x) < slice.c_lo || int(e.x) >= slice.c_hi) continue;
                            const float x = penalize(row.p, E::load(g.row, e.x), e.y);
                            cache[int(e.x) - slice.c_lo + slice.skew] = x != x ? 0u : fkey(ydiv(row.p, x));
                        }
                        __syncthreads();
                    }
                    slice.each([&](int c, uint32_t k) { meet(c, k, k == 0u); });
                } else {
                    slice.read([&](int c, int n, const uint32_t* k, uint32_t nans) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j)
                            if (j < n) meet(c + j, k[j], nans >> j & 1u);
                    });
                }
                const uint32_t wtop = __reduce_max_sync(0xffffffffu, top);
                const uint32_t warg = __reduce_min_sync(0xffffffffu, top == wtop ? arg : 0xffffffffu);
                nan_col = __reduce_min_sync(0xffffffffu, nan_col);
                if (lane == 0) {
                    S.red32[warp] = wtop;
                    S.red64[warp] = warg;
                    if (nan_col != 0xffffffffu) atomicMin(&S.nan_col, nan_col);
                }
                __syncthreads();
                if (tid == 0)
                    for (int w = 0; w < NW; ++w)
                        if (S.red32[w] > S.top || (S.red32[w] == S.top && uint32_t(S.red64[w]) < S.arg)) {
                            S.top = S.red32[w];
                            S.arg = uint32_t(S.red64[w]);
                        }
            }
            cluster_sync();
            const uint32_t peer = uint32_t(min(lane, G - 1));
            uint32_t top_key = ld_cluster(mapa(&S.top, peer)), arg = ld_cluster(mapa(&S.arg, peer));
            uint32_t nan_col = ld_cluster(mapa(&S.nan_col, peer)), flags = ld_cluster(mapa(&S.flags, peer));
            {
                const uint32_t k = __reduce_max_sync(0xffffffffu, top_key);
                arg = __reduce_min_sync(0xffffffffu, top_key == k ? arg : 0xffffffffu);
                top_key = k;
                nan_col = __reduce_min_sync(0xffffffffu, nan_col);
                flags = __reduce_or_sync(0xffffffffu, flags);
            }
            const float top = funkey(top_key);
            uint32_t errors = row.p.bad | (flags & FG_ROW_BAD_PARAM);
            if (!row.greedy) {
                if (nan_col != 0xffffffffu) errors |= FG_ROW_NAN;
                else if (top_key <= KEY_NEG_INF) errors |= FG_ROW_ALL_MASKED;
                else if (!(top < INFINITY)) errors |= FG_ROW_POS_INF;
            }
            const uint32_t status = flags | errors | FG_ROW_GENERAL_PATH | (row.greedy ? uint32_t(FG_ROW_GREEDY) : 0u);
            // what is drawn, and the kept set: keys above cut_key, and at cut_key the columns up to cut_col
            int drawn = -1;
            uint32_t cut_key = 0, cut_col = 0;
            uint64_t kept = 0;
            const double unit = double(uint64_t(1) << P.mass_shift);
            if (!errors && row.greedy) {
                // the first NaN counts as the maximum; a row of -inf has its first column
                drawn = int(nan_col != 0xffffffffu ? nan_col : arg);
                if (rank == 0 && tid == 0) write_row(P, r, drawn, 0.0f, 1, status);
            } else if (errors) {
                if (rank == 0 && tid == 0) write_error(P, r, status);
            } else {
                const double log_p = log_min_p(row);
                uint32_t floor_key = least_key(log_p, top);
                const float per_bin = bin_scale(log_p, BINS);
                auto top_bin = [&](uint32_t k) { return bin_of(top, funkey(k), per_bin, BINS); };
                fill_bins(slice, B, G, rank, [&](uint32_t k) { return k >= floor_key ? int(top_bin(k)) : -1; }, top, T,
                          P.mass_shift, B.top_mass, B.top_count);
                // everything that min-p keeps
                uint64_t all = 0;
                uint32_t count = 0;
#pragma unroll
                for (int j = 0; j < BINS / WNT; ++j) {
                    all += B.top_mass[j * WNT + tid];
                    count += B.top_count[j * WNT + tid];
                }
                all = warp_incl_scan_u64(all, lane);
                count = __reduce_add_sync(0xffffffffu, count);
                if (lane == 31) {
                    S.red64[warp] = all;
                    S.red32[warp] = count;
                }
                __syncthreads();
                all = 0;
                count = 0;
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    all += S.red64[w];
                    count += S.red32[w];
                }
                __syncthreads();
                kept = all;
                cut_key = floor_key;
                uint32_t kept_count = count, cut_ties = 0xffffffffu;   // of the columns at cut_key
                // top-k (0), the top-p cut (1), the draw (2)
#pragma unroll 1
                for (int step = 0; step < 3; ++step) {
                    if (step == 0 && !(row.K > 0 && uint32_t(row.K) < count)) continue;
                    if (step == 1 && !row.p.use_p) continue;
                    const bool by_mass = step > 0;
                    const uint64_t target = step == 0   ? uint64_t(row.K - 1)
                                            : step == 1 ? part_of(row.p.top_p, all)
                                                        : part_of(row.p.u, kept);
                    // the key at which the count or mass from the top passes the target
                    Found f{0u, 0, 0, 0, 0};
                    const uint32_t b = locate(S, f, by_mass, target, B.top_mass, B.top_count);
                    const bool in_order = f.at_count <= uint32_t(MEMBERS);
                    if (in_order) {
                        if (tid == 0) S.n = 0;
                        __syncthreads();
                        slice.each([&](int c, uint32_t k) {
                            if (k >= floor_key && top_bin(k) == b)
                                members[atomicAdd(&S.n, 1u)] = uint64_t(k) << 32 | uint32_t(~uint32_t(c));
                        });
                        cluster_sync();
                        if (rank == 0) {
                            // a warp or two for each CTA's members, behind those of the CTAs before it
                            const uint32_t n = lane < G ? ld_cluster(mapa(&S.n, uint32_t(lane))) : 0u;
                            const uint32_t upto = warp_incl_scan_u32(n, lane);
                            const int have = int(__shfl_sync(0xffffffffu, upto, 31));
                            const int c = warp % G;
                            const int cn = int(__shfl_sync(0xffffffffu, n, c)), to = int(__shfl_sync(0xffffffffu, upto, c)) - cn;
                            for (int i = warp / G * 32 + lane; i < cn; i += NW / G * 32)
                                all_members[to + i] = ld_cluster64(mapa(&members[i], uint32_t(c)));
                            int room = 32;
                            while (room < have) room <<= 1;
                            for (int i = have + tid; i < room; i += WNT) all_members[i] = 0;
                            __syncthreads();
                            sort_descending<WNT>(all_members, room);
                            // the element that passes the target, then all that share its key
                            constexpr int PM = MEMBERS / WNT;
                            uint64_t m[PM], sum = 0;
#pragma unroll
                            for (int j = 0; j < PM; ++j) {
                                const int i = tid * PM + j;
                                m[j] = i < have ? mass_of(funkey(uint32_t(all_members[i] >> 32)), top, T, P.mass_shift) : 0;
                                sum += m[j];
                            }
                            const uint64_t im = warp_incl_scan_u64(sum, lane);
                            if (lane == 31) S.red64[warp] = im;
                            __syncthreads();
                            uint64_t at_mass = f.before_mass + im - sum;
                            for (int w = 0; w < warp; ++w) at_mass += S.red64[w];
                            if (!by_mass) {
                                if (tid == 0) S.key = uint32_t(all_members[target - f.before_count] >> 32);
                            } else {
                                uint64_t before = at_mass;
#pragma unroll
                                for (int j = 0; j < PM; ++j) {
                                    if (before <= target && target < before + m[j])
                                        S.key = uint32_t(all_members[tid * PM + j] >> 32);
                                    before += m[j];
                                }
                            }
                            __syncthreads();
                            const uint32_t key = S.key;
                            uint32_t same = 0;
#pragma unroll
                            for (int j = 0; j < PM; ++j) {
                                const int i = tid * PM + j;
                                if (i < have && uint32_t(all_members[i] >> 32) == key) {
                                    ++same;
                                    if (i == 0 || uint32_t(all_members[i - 1] >> 32) != key) {
                                        S.first = uint32_t(i);
                                        S.found_count = f.before_count + uint32_t(i);
                                        S.found_mass = at_mass;
                                    }
                                }
                                at_mass += m[j];
                            }
                            same = __reduce_add_sync(0xffffffffu, same);
                            if (lane == 0) S.red32[warp] = same;
                            __syncthreads();
                            if (tid == 0) {
                                for (int w = 1; w < NW; ++w) same += S.red32[w];
                                S.found_at = same;
                            }
                            __syncthreads();
                        }
                        cluster_sync();
                        f.key = ld_cluster(mapa(&S.key, 0));
                        f.before_count = ld_cluster(mapa(&S.found_count, 0));
                        f.before_mass = ld_cluster64(mapa(&S.found_mass, 0));
                        f.at_count = ld_cluster(mapa(&S.found_at, 0));
                        f.at_mass = f.at_count * mass_of(funkey(f.key), top, T, P.mass_shift);
                    } else {
                        // many share the bin: by the keys' bits, highest first (the bins' order is descending)
                        uint32_t key = 0;
                        int shift = 32;
#pragma unroll 1
                        for (int level = 0; level < 3; ++level) {
                            const int bits = level < 2 ? 11 : 10;
                            const uint32_t above = shift == 32 ? 0u : 0xffffffffu << shift, low = (1u << bits) - 1u;
                            shift -= bits;
                            fill_bins(slice, B, G, rank, [&](uint32_t k) {
                                return k >= floor_key && ((k ^ key) & above) == 0u && top_bin(k) == b
                                           ? int(low - (k >> shift & low)) : -1;
                            }, top, T, P.mass_shift, B.all_mass, B.all_count);
                            key |= (low - locate(S, f, by_mass, target, B.all_mass, B.all_count)) << shift;
                        }
                        f.key = key;
                    }
                    if (step == 0) {
                        floor_key = cut_key = f.key;
                        kept = all = f.before_mass + f.at_mass;
                        kept_count = f.before_count + f.at_count;
                    } else {
                        const uint64_t m = f.at_mass / f.at_count;
                        const uint32_t nth = uint32_t((target - f.before_mass) / m);   // of those that share the key
                        if (step == 1) {
                            cut_key = f.key;
                            cut_ties = min(f.at_count, nth + 1);
                            kept = f.before_mass + cut_ties * m;
                            kept_count = f.before_count + cut_ties;
                        } else {
                            // (without probabilities the first CTA alone writes, and may know the place)
                            if (in_order && !P.out_probs)
                                drawn = rank == 0 ? int(~uint32_t(all_members[S.first + nth])) : 0;
                            else
                                drawn = int(column_of(slice, S, G, rank, f.key, nth));
                            if (rank == 0 && tid == 0) {
                                const double y = double(funkey(f.key)) - double(top);
                                write_row(P, r, drawn, float(y - log(double(kept) / unit)), int(kept_count), status);
                            }
                        }
                    }
                }
                if (P.out_probs) cut_col = cut_ties == 0xffffffffu ? 0xffffffffu : column_of(slice, S, G, rank, cut_key, cut_ties - 1);
            }
            if (P.out_probs) {
                float* out = P.out_probs + int64_t(r) * P.vocab;
                const double all = double(kept);
                slice.each([&](int c, uint32_t k) {
                    float p = 0.0f;
                    if (drawn >= 0) {
                        if (row.greedy) p = c == drawn ? 1.0f : 0.0f;
                        else if (k > cut_key || (k == cut_key && uint32_t(c) <= cut_col))
                            p = float(exp(double(funkey(k)) - double(top)) * unit / all);
                    }
                    out[c] = p;
                });
            }
            cluster_sync();   // the next row's state replaces what the others may still read
        }
    }
}

}  // namespace minp
}  // namespace fg
