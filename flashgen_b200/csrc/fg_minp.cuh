// fg_minp.cuh — sampling with min-p beside penalties, temperature, top-k and top-p
// (fg_sample_min_p). For every row, y being the penalised logits over the temperature:
//   A    = {j : y_j >= max y + log(min_p)}, cut to the K largest (ties kept)
//   kept = A in descending order while the mass before a token is <= top_p * mass(A)
//   id   = the first kept token whose inclusive mass exceeds u * mass(kept)
// with masses e^(y_j - max y), as integers round(2^S e^(y - max y)) from 64-bit
// exponentials: sums do not depend on their order, and a decision is as sharp as a
// 64-bit one (S = 62 - log2 V: 2^-46 of the largest mass at V = 128256).
//
// min-p bounds what can be drawn by the row's maximum alone. So rows_kernel reads each
// logit once, compares it with a bound that rises with the maximum seen so far and keeps
// the few that reach it; everything else is decided on those, sorted in shared memory.
// Rows whose candidates do not fit there (no min-p and no small top-k, or flat rows) go to
// wide_kernel, which selects by radix over the whole row.
#pragma once

#include "fg_row.cuh"

namespace fg {
namespace minp {

constexpr int NT = 256;            // threads of rows_kernel
constexpr int UNROLL = 8;          // 16-byte chunks a thread has in flight
constexpr int CAP = 2048;          // candidates of a CTA's slice, and of a row
constexpr int MAX_G = 8;           // CTAs that share a row
constexpr int HIST_CAP = 4096;     // history ids of a row that rows_kernel takes
constexpr int WNT = 512;           // threads of wide_kernel
constexpr int BINS = 2048;         // of a radix step
constexpr int FILTER_WORDS = 4096; // bits that say which columns may be in the history

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
    int32_t hist_max_len;
    int32_t slots, wide_slots; // of a history table (powers of two)
    int32_t mass_shift;        // S
    int32_t cache;             // keys that wide_kernel keeps in shared memory (0: none)
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
    double log_min_p;    // -inf without min-p
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
    row.log_min_p = row.greedy || row.min_p == 1.0f ? 0.0 : row.min_p > 0.0f ? log(double(row.min_p)) : -INFINITY;
    return row;
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

// round(2^S e^(y - top))
__device__ __forceinline__ uint64_t mass_of(float y, float top, double scale) {
    return __double2ull_rn(exp(double(y) - double(top)) * scale);
}
// The smallest key that min-p keeps below a maximum of `top`: y >= top + log(min_p) in 64 bits.
__device__ __forceinline__ uint32_t least_key(const Row& row, float top) {
    if (!(row.log_min_p > -INFINITY)) return KEY_NEG_INF + 1u;
    const uint32_t k = fkey(__double2float_ru(double(top) + row.log_min_p));
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
template <int THREADS>
__device__ __forceinline__ uint32_t count_history(const Params& P, const Row& row, uint2* table, uint32_t mask,
                                                  int64_t c_lo, int64_t c_hi, uint32_t* filter) {
    uint32_t bad = 0;
    for (int64_t i = row.h0 + threadIdx.x; i < row.h1; i += THREADS) {
        const int64_t id = __ldg(P.hist_ids + i);
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
        if (filter) {
            const uint32_t b = uint32_t(c - c_lo) & (FILTER_WORDS * 32 - 1);
            atomicOr(&filter[b >> 5], 1u << (b & 31));
        }
    }
    return bad;
}

// ---------------------------------------------------------------------------
// rows_kernel: one cluster of G CTAs a row, each a slice of it.
//
// Bound: HBM reads. A 16-byte chunk costs a packed maximum and one comparison; the chunks
// that reach the bound, a few hundred of a row, are looked at element by element.
// ---------------------------------------------------------------------------
struct Shared {
    uint32_t top;        // key of the largest (penalised) logit seen
    uint32_t least;      // key of a lower bound of the K-th largest logit
    uint32_t count;      // candidates
    uint32_t flags;      // row status bits
    uint32_t n;          // sorted candidates
    uint32_t nk, np, at;
    uint32_t warp[NT / 32];
    uint64_t sums[NT / 32];
    uint64_t total;
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

// A bound below which no logit can be kept when the largest is `top`. The slack covers the
// roundings of x / T, of the maximum's quotient and of this product.
__device__ __forceinline__ float bound_of(const Row& row, float top, float span) {
    if (row.greedy) return top;
    return top - span - 0x1p-20f * (fabsf(top) + span);
}

template <int DT>
__global__ void __launch_bounds__(NT) rows_kernel(const Params P, const int G) {
    using E = Elem<DT>;
    constexpr int VEC = E::VEC;
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ Shared S;
    Candidate* cand = reinterpret_cast<Candidate*>(dyn);
    uint64_t* sorted = reinterpret_cast<uint64_t*>(dyn + CAP * sizeof(Candidate));
    uint2* table = reinterpret_cast<uint2*>(dyn + CAP * (sizeof(Candidate) + 8));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / G;
    const uint32_t rank = G > 1 ? cluster_rank() : 0;
    wait_prerequisites();
    launch_dependents();

    if (rank == 0 && tid == 0) P.marks[r] = 0;
    const Row row = load_row(P, r);
    // a lower bound of the K-th largest comes from K chunks of the first tile
    const bool by_k = row.K > 0 && row.K <= CAP / 4;
    auto hand_on = [&]() {
        if (rank == 0 && tid == 0) P.marks[r] = 1;
    };
    if (row.p.bad && !P.out_probs) {
        if (rank == 0 && tid == 0) write_error(P, r, row.p.bad);
        return;
    }
    if (P.out_probs || (!row.greedy && row.min_p == 0.0f && !by_k) || row.h1 - row.h0 > HIST_CAP) {
        hand_on();
        return;
    }
    const Geom g = row_geom<E::SIZE>(P.logits, P.row_stride, P.vocab, r);
    const int nch = int(g.ibytes / 16);
    const int ch0 = int(int64_t(nch) * rank / G), ch1 = int(int64_t(nch) * (rank + 1) / G);
    const bool first = rank == 0, last = int(rank) == G - 1;
    const int c_lo = first ? 0 : g.head + ch0 * VEC, c_hi = last ? P.vocab : g.head + ch1 * VEC;
    const uint4* chunks = reinterpret_cast<const uint4*>(g.interior);
    const uint32_t mask = uint32_t(P.slots) - 1u;
    const bool pen = row.p.pen;

    // the first tile's loads go out before anything waits
    uint4 q[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
        const int c = ch0 + i * NT + tid;
        if (c < ch1) q[i] = __ldg(chunks + c);
    }
    if (tid == 0) {
        S.top = KEY_NEG_INF;
        S.least = KEY_NEG_INF;
        S.count = 0;
        S.flags = 0;
        S.n = 0;
    }
    if (pen)
        for (int i = tid; i <= int(mask); i += NT) table[i] = make_uint2(kEmptySlot, 0u);
    __syncthreads();
    if (pen) {
        const uint32_t bad = count_history<NT>(P, row, table, mask, c_lo, c_hi, nullptr);
        if (bad) atomicOr(&S.flags, bad);
        __syncthreads();
        uint32_t top = KEY_NEG_INF;
        for (int i = tid; i <= int(mask); i += NT) {
            if (table[i].x == kEmptySlot) continue;
            const float x = penalize(row.p, E::load(g.row, table[i].x), table[i].y);
            table[i].y = __float_as_uint(x);
            if (x != x) atomicOr(&S.flags, uint32_t(FG_ROW_NAN));
            else top = max(top, fkey(x));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) atomicMax(&S.top, top);
    }
    auto in_history = [&](uint32_t col) { return pen && find_slot(table, mask, col) >= 0; };
    const float span = row.greedy ? 0.0f : float(-row.log_min_p) * row.p.T;

    // the first tile's maximum, over what is not in the history
    {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int c = ch0 + i * NT + tid;
            if (c >= ch1) break;
            if (!(chunk_max<DT>(q[i]) > top)) continue;
            float x[VEC];
            E::unpack(q[i], x);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (x[j] > top && !in_history(uint32_t(g.head + c * VEC + j))) top = x[j];
        }
        const uint32_t key = __reduce_max_sync(0xffffffffu, fkey(top));
        if (lane == 0) atomicMax(&S.top, key);
        __syncthreads();
        if (by_k) {
            // the largest key, to 2^-11 of its range, that K chunks of the tile reach (the K-th
            // largest logit is no smaller); a chunk with history columns counts for none
            uint32_t key_of[UNROLL];
#pragma unroll
            for (int i = 0; i < UNROLL; ++i) {
                const int c = ch0 + i * NT + tid;
                key_of[i] = 0u;
                if (c >= ch1) continue;
                bool clean = true;
                if (pen)
                    for (int j = 0; j < VEC; ++j) clean = clean && !in_history(uint32_t(g.head + c * VEC + j));
                const float m = chunk_max<DT>(q[i]);
                if (clean && m == m) key_of[i] = fkey(m);
            }
            uint32_t lo = KEY_NEG_INF, hi = S.top;
            for (int step = 0; step < 20 && hi - lo > 1u; ++step) {
                const uint32_t mid = lo + (hi - lo + 1) / 2;
                uint32_t n = 0;
#pragma unroll
                for (int i = 0; i < UNROLL; ++i) n += key_of[i] >= mid;
                n = __reduce_add_sync(0xffffffffu, n);
                if (lane == 0) S.warp[warp] = n;
                __syncthreads();
                n = 0;
#pragma unroll
                for (int w = 0; w < NT / 32; ++w) n += S.warp[w];
                __syncthreads();
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
    auto refresh = [&](uint32_t key) {
        seen = funkey(key);
        bound = bound_of(row, seen, span);
        with_k(S.least);
    };
    auto take = [&](float x, uint32_t col) {     // a logit that is not below the bound, or NaN
        if (!(x > -INFINITY)) {
            if (x != x && !in_history(col)) atomicOr(&S.flags, uint32_t(FG_ROW_NAN));
            return;
        }
        if (in_history(col)) return;
        if (x > seen) atomicMax(&S.top, fkey(x));
        const uint32_t at = atomicAdd(&S.count, 1u);
        if (at < uint32_t(CAP)) cand[at] = {x, col};
    };
    auto scan_chunk = [&](const uint4& v, int c) {
        if (chunk_max<DT>(v) < bound) return;
        float x[VEC];
        E::unpack(v, x);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (!(x[j] < bound)) take(x[j], uint32_t(g.head + c * VEC + j));
    };
    auto scan_ragged = [&]() {
        if (first)
            for (int c = tid; c < g.head; c += NT) {
                const float x = E::load(g.row, c);
                if (!(x < bound)) take(x, uint32_t(c));
            }
        if (last)
            for (int c = g.tail0 + tid; c < P.vocab; c += NT) {
                const float x = E::load(g.row, c);
                if (!(x < bound)) take(x, uint32_t(c));
            }
    };
    refresh(S.top);
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
        const int c = ch0 + i * NT + tid;
        if (c < ch1) scan_chunk(q[i], c);
    }
    for (int base = ch0 + UNROLL * NT; base < ch1; base += UNROLL * NT) {
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int c = base + i * NT + tid;
            if (c < ch1) q[i] = __ldg(chunks + c);
        }
        refresh(*reinterpret_cast<volatile uint32_t*>(&S.top));
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int c = base + i * NT + tid;
            if (c < ch1) scan_chunk(q[i], c);
        }
    }
    scan_ragged();
    __syncthreads();

    // the whole row's maximum and flags
    uint32_t top_key = S.top, flags = S.flags, least = S.least;
    if (G > 1) {
        cluster_sync();
        for (int i = 0; i < G; ++i) {
            top_key = max(top_key, ld_cluster(mapa(&S.top, i)));
            least = max(least, ld_cluster(mapa(&S.least, i)));
            flags |= ld_cluster(mapa(&S.flags, i));
        }
        // (S.top and S.flags stay as they are until the last cluster_sync)
    }
    const float top_x = funkey(top_key);
    seen = INFINITY;                              // from here on nothing raises the maximum
    bound = bound_of(row, top_x, span);
    with_k(least);
    bool over = S.count > uint32_t(CAP);
    const bool sick = (flags & FG_ROW_NAN) || top_key <= KEY_NEG_INF || !(top_x < INFINITY);
    __syncthreads();
    if (over && !sick) {
        // too many while the maximum was still rising: once more with the final bound (from L2)
        if (tid == 0) S.count = 0;
        __syncthreads();
        for (int c = ch0 + tid; c < ch1; c += NT) scan_chunk(__ldg(chunks + c), c);
        scan_ragged();
        __syncthreads();
    }
    if (pen && !sick) {
        for (int i = tid; i <= int(mask); i += NT) {
            const float x = __uint_as_float(table[i].y);
            if (table[i].x == kEmptySlot || !(x >= bound) || !(x > -INFINITY)) continue;
            const uint32_t at = atomicAdd(&S.count, 1u);
            if (at < uint32_t(CAP)) cand[at] = {x, table[i].x};
        }
        __syncthreads();
    }
    if (G > 1) cluster_sync();                    // every slice's candidates stand
    over = false;
    for (int i = 0; i < G; ++i) over = over || (G > 1 ? ld_cluster(mapa(&S.count, i)) : S.count) > uint32_t(CAP);

    if (rank == 0) {
        // greedy rows with NaN or without a finite maximum: wide_kernel knows their first place
        const bool wide = (sick && row.greedy) || (!sick && over);
        const uint32_t errors = (flags & (FG_ROW_NAN | FG_ROW_BAD_PARAM)) |
                                (flags & FG_ROW_NAN ? 0u : top_key <= KEY_NEG_INF ? uint32_t(FG_ROW_ALL_MASKED)
                                                         : !(top_x < INFINITY)    ? uint32_t(FG_ROW_POS_INF) : 0u);
        if (wide) {
            hand_on();
        } else if ((flags & FG_ROW_BAD_PARAM) || (!row.greedy && (errors || !(ydiv(row.p, top_x) < INFINITY)))) {
            if (tid == 0) write_error(P, r, errors ? flags | errors : flags | FG_ROW_POS_INF);
        } else {
            // ---- the candidates, exactly: (key of y, ~column), so that larger comes first
            const float top = ydiv(row.p, top_x);
            const uint32_t least_k = row.greedy ? top_key : least_key(row, top);
            for (int i = 0; i < G; ++i) {
                const uint32_t n = G > 1 ? ld_cluster(mapa(&S.count, i)) : S.count;
                const uint32_t src = G > 1 ? mapa(cand, i) : smem_u32(cand);
                for (uint32_t j = tid; j < n; j += NT) {
                    const uint64_t c = ld_cluster64(src + 8 * j);   // {x, col}
                    const uint32_t key = fkey(ydiv(row.p, __uint_as_float(uint32_t(c))));
                    if (key < least_k) continue;
                    const uint32_t at = atomicAdd(&S.n, 1u);
                    if (at < uint32_t(CAP)) sorted[at] = uint64_t(key) << 32 | uint32_t(~uint32_t(c >> 32));
                }
            }
            __syncthreads();
            const int n = int(S.n);
            if (n > CAP) {
                hand_on();
            } else {
                int room = 32;
                while (room < n) room <<= 1;
                for (int i = n + tid; i < room; i += NT) sorted[i] = 0;
                __syncthreads();
                // bitonic, descending
                for (int size = 2; size <= room; size <<= 1)
                    for (int d = size >> 1; d > 0; d >>= 1) {
                        for (int i = tid; i < room / 2; i += NT) {
                            const int a = 2 * i - (i & (d - 1)), b = a + d;
                            const uint64_t u = sorted[a], v = sorted[b];
                            if (((a & size) == 0) == (u < v)) {
                                sorted[a] = v;
                                sorted[b] = u;
                            }
                        }
                        __syncthreads();
                    }
                const uint32_t status = flags | (row.greedy ? uint32_t(FG_ROW_GREEDY) : 0u);
                if (row.greedy) {
                    if (tid == 0) write_row(P, r, int64_t(~uint32_t(sorted[0])) + P.vocab_offset, 0.0f, 1, status);
                } else {
                    // each thread the masses of CAP / NT neighbours
                    constexpr int PER = CAP / NT;
                    const double scale = double(uint64_t(1) << P.mass_shift);
                    const uint32_t kth = row.K > 0 && row.K < n ? uint32_t(sorted[row.K - 1] >> 32) : 0u;
                    uint64_t m[PER], sum = 0;
                    uint32_t mine = 0;
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        const int i = tid * PER + j;
                        const uint32_t key = i < n ? uint32_t(sorted[i] >> 32) : 0u;
                        const bool in = i < n && key >= kth;
                        m[j] = in ? mass_of(funkey(key), top, scale) : 0;
                        mine += in;
                        sum += m[j];
                    }
                    uint64_t upto = warp_incl_scan_u64(sum, lane);
                    mine = __reduce_add_sync(0xffffffffu, mine);
                    if (lane == 31) S.sums[warp] = upto;
                    if (lane == 0) S.warp[warp] = mine;
                    if (tid == 0) S.at = 0xffffffffu;
                    __syncthreads();
                    uint64_t total = 0, before = upto - sum;
                    int nk = 0;
#pragma unroll
                    for (int w = 0; w < NT / 32; ++w) {
                        if (w < warp) before += S.sums[w];
                        total += S.sums[w];
                        nk += int(S.warp[w]);
                    }
                    __syncthreads();
                    // top-p: the tokens whose mass before them is within its share
                    int np = nk;
                    uint64_t kept = total;
                    if (row.p.use_p) {
                        const uint64_t limit = part_of(row.p.top_p, total);
                        uint64_t at = before, part = 0;
                        uint32_t count = 0;
#pragma unroll
                        for (int j = 0; j < PER; ++j) {
                            if (tid * PER + j < nk && at <= limit) {
                                ++count;
                                part += m[j];
                            }
                            at += m[j];
                        }
                        count = __reduce_add_sync(0xffffffffu, count);
                        part = warp_incl_scan_u64(part, lane);
                        if (lane == 31) {
                            S.sums[warp] = part;
                            S.warp[warp] = count;
                        }
                        __syncthreads();
                        np = 0;
                        kept = 0;
#pragma unroll
                        for (int w = 0; w < NT / 32; ++w) {
                            np += int(S.warp[w]);
                            kept += S.sums[w];
                        }
                    }
                    const uint64_t target = part_of(row.p.u, kept);
                    uint64_t at = before;
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        at += m[j];
                        if (tid * PER + j < np && at > target && at - m[j] <= target) S.at = tid * PER + j;
                    }
                    __syncthreads();
                    if (tid == 0) {
                        const uint64_t c = sorted[S.at];
                        const double y = double(funkey(uint32_t(c >> 32))) - double(top);
                        write_row(P, r, int64_t(~uint32_t(c)) + P.vocab_offset,
                                  float(y - log(double(kept) / scale)), np, status);
                    }
                }
            }
        }
    }
    if (G > 1) cluster_sync();                    // nobody leaves while its candidates may be read
}

// ---------------------------------------------------------------------------
// wide_kernel: the rows of the list, one after the other on clusters of G CTAs, each a
// slice of the row. The first pass leaves the order-preserving key of every y in shared
// memory (where it fits); then each decision is a radix search over the keys by count or
// by mass: 2048 bins of the highest bits, then of the next ones among the keys that
// share those, summed over the cluster through distributed shared memory.
// ---------------------------------------------------------------------------
struct WideShared {
    uint32_t red32[WNT / 32];
    uint64_t red64[WNT / 32];
    uint32_t top, arg, nan_col, flags;   // this CTA's, read by the others
    uint16_t rows[WNT];
    uint32_t ties;
    uint32_t bin;
    uint64_t before_mass, at_mass;
    uint32_t before_count, at_count;
};
// The bins of one radix step: this CTA's, its share of the cluster's, and all of the cluster's.
struct Bins {
    uint64_t* mass;
    uint32_t* count;
    uint64_t* own_mass;
    uint32_t* own_count;
    uint64_t* all_mass;
    uint32_t* all_count;
    uint64_t* top_mass;          // of the highest bits, kept for every search of the row
    uint32_t* top_count;
};
constexpr int bins_bytes(int G) { return 12 * (3 * BINS + BINS / G); }

// Where a search has come to: keys with `prefix` above `shift` bits, what lies above them.
struct Found {
    uint32_t key;                // low bits cleared below `shift`
    int shift;
    uint64_t before_mass, at_mass;
    uint32_t before_count, at_count;
};

template <int DT>
__global__ void __launch_bounds__(WNT, 1) wide_kernel(const Params P, const int G) {
    using E = Elem<DT>;
    constexpr int VEC = E::VEC;
    constexpr int NW = WNT / 32;
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ WideShared S;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = cluster_rank();
    const int per = BINS / G;
    Bins B;
    B.mass = reinterpret_cast<uint64_t*>(dyn);
    B.all_mass = B.mass + BINS;
    B.top_mass = B.all_mass + BINS;
    B.own_mass = B.top_mass + BINS;
    B.count = reinterpret_cast<uint32_t*>(B.own_mass + per);
    B.all_count = B.count + BINS;
    B.top_count = B.all_count + BINS;
    B.own_count = B.top_count + BINS;
    uint32_t* filter = B.own_count + per;
    uint32_t* cache = filter + (P.penalties ? FILTER_WORDS : 0);
    wait_prerequisites();
    uint2* table = P.tables + int64_t(blockIdx.x / G) * P.wide_slots;
    const uint32_t mask = uint32_t(P.wide_slots) - 1u;

    // the rows that carry rows_kernel's mark, in ascending order, by turns to the clusters
    const int clusters = gridDim.x / G, mine_of = blockIdx.x / G;
    int marked = 0;   // so far
    for (int base = 0; base < P.batch; base += WNT) {
      const bool mark = base + tid < P.batch &&
                        *reinterpret_cast<const volatile uint8_t*>(&P.marks[base + tid]) != 0;
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
        const int ch0 = int(int64_t(nch) * rank / G), ch1 = int(int64_t(nch) * (rank + 1) / G);
        const bool first = rank == 0, last = int(rank) == G - 1;
        const int c_lo = first ? 0 : g.head + ch0 * VEC, c_hi = last ? P.vocab : g.head + ch1 * VEC;
        const bool pen = row.p.pen;
        const bool cached = P.cache > 0;

        if (tid == 0) {
            S.flags = 0;
            S.top = KEY_NEG_INF;
            S.arg = 0xffffffffu;
            S.nan_col = 0xffffffffu;
        }
        if (pen) {
            // the cluster shares one table; its CTAs insert and look up columns of their own
            for (int i = int(rank) * WNT + tid; i <= int(mask); i += G * WNT) table[i] = make_uint2(kEmptySlot, 0u);
            for (int i = tid; i < FILTER_WORDS; i += WNT) filter[i] = 0u;
        }
        cluster_sync();
        if (pen) {
            const uint32_t bad = count_history<WNT>(P, row, table, mask, c_lo, c_hi, filter);
            if (bad) atomicOr(&S.flags, bad);
            __syncthreads();
        }
        // the key of column c (greedy rows: of the penalised logit itself)
        auto key_at = [&](int c, float x, bool* nan) {
            if (pen) {
                const uint32_t b = uint32_t(c - c_lo) & (FILTER_WORDS * 32 - 1);
                if (filter[b >> 5] >> (b & 31) & 1u) {
                    const int s = find_slot(table, mask, uint32_t(c));
                    if (s >= 0) x = penalize(row.p, x, *reinterpret_cast<const volatile uint32_t*>(&table[s].y));
                }
            }
            *nan = x != x;
            return *nan ? 0u : fkey(ydiv(row.p, x));
        };
        // every column of the slice: f(column, key, nan), in no order
        auto each = [&](auto f) {
            if (first)
                for (int c = tid; c < g.head; c += WNT) {
                    bool nan;
                    const uint32_t k = key_at(c, E::load(g.row, c), &nan);
                    f(c, k, nan);
                }
            const uint4* chunks = reinterpret_cast<const uint4*>(g.interior);
            for (int b = ch0; b < ch1; b += 4 * WNT) {
                uint4 q[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int ch = b + i * WNT + tid;
                    if (ch < ch1) q[i] = __ldg(chunks + ch);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int ch = b + i * WNT + tid;
                    if (ch >= ch1) break;
                    float x[VEC];
                    E::unpack(q[i], x);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        bool nan;
                        const int c = g.head + ch * VEC + j;
                        const uint32_t k = key_at(c, x[j], &nan);
                        f(c, k, nan);
                    }
                }
            }
            if (last)
                for (int c = g.tail0 + tid; c < P.vocab; c += WNT) {
                    bool nan;
                    const uint32_t k = key_at(c, E::load(g.row, c), &nan);
                    f(c, k, nan);
                }
        };
        auto each_key = [&](auto f) {   // the same without the NaN
            if (cached) {
                for (int i = tid; i < c_hi - c_lo; i += WNT) f(c_lo + i, cache[i]);
            } else {
                each([&](int c, uint32_t k, bool) { f(c, k); });
            }
        };
        // ---- keys, the maximum and its first column, the first NaN
        {
            uint32_t top = KEY_NEG_INF, arg = 0xffffffffu, nan_col = 0xffffffffu;
            each([&](int c, uint32_t k, bool nan) {
                if (cached) cache[c - c_lo] = k;
                if (nan) nan_col = min(nan_col, uint32_t(c));
                else if (k > top || (k == top && uint32_t(c) < arg)) {
                    top = k;
                    arg = uint32_t(c);
                }
            });
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
        uint32_t top_key = KEY_NEG_INF, arg = 0xffffffffu, nan_col = 0xffffffffu, flags = 0;
        for (int i = 0; i < G; ++i) {
            const uint32_t k = ld_cluster(mapa(&S.top, i)), a = ld_cluster(mapa(&S.arg, i));
            if (k > top_key || (k == top_key && a < arg)) {
                top_key = k;
                arg = a;
            }
            nan_col = min(nan_col, ld_cluster(mapa(&S.nan_col, i)));
            flags |= ld_cluster(mapa(&S.flags, i));
        }
        const float top = funkey(top_key);
        uint32_t errors = row.p.bad | (flags & FG_ROW_BAD_PARAM);
        if (!row.greedy) {
            if (nan_col != 0xffffffffu) errors |= FG_ROW_NAN;
            else if (top_key <= KEY_NEG_INF) errors |= FG_ROW_ALL_MASKED;
            else if (!(top < INFINITY)) errors |= FG_ROW_POS_INF;
        }
        const uint32_t status = flags | errors | FG_ROW_GENERAL_PATH | (row.greedy ? uint32_t(FG_ROW_GREEDY) : 0u);
        // what is drawn: the column's key, and the kept set: keys above cut_key, and at cut_key the
        // columns up to cut_col
        int drawn = -1;
        uint32_t cut_key = 0, cut_col = 0, kept_count = 0;
        uint64_t kept = 0;
        const double scale = double(uint64_t(1) << P.mass_shift);
        if (!errors && row.greedy) {
            // the first NaN counts as the maximum; a row of -inf has its first column
            drawn = int(nan_col != 0xffffffffu ? nan_col : arg);
            if (rank == 0 && tid == 0) write_row(P, r, drawn + P.vocab_offset, 0.0f, 1, status);
            cut_key = nan_col != 0xffffffffu ? 0xffffffffu : top_key;
            cut_col = uint32_t(drawn);
            kept = uint64_t(1) << P.mass_shift;
        } else if (errors) {
            if (rank == 0 && tid == 0) write_error(P, r, status);
        } else {
            uint32_t floor_key = least_key(row, top);
            // bins of the keys that are >= floor_key and share `at`'s bits above `shift + bits`
            auto fill = [&](uint32_t at, int shift, int bits, uint64_t* all_mass, uint32_t* all_count) {
                for (int i = tid; i < BINS; i += WNT) {
                    B.mass[i] = 0;
                    B.count[i] = 0;
                }
                __syncthreads();
                const uint32_t above = shift + bits >= 32 ? 0u : 0xffffffffu << (shift + bits);
                const uint32_t low = (1u << bits) - 1u;
                each_key([&](int, uint32_t k) {
                    if (k < floor_key || ((k ^ at) & above)) return;
                    const uint32_t b = k >> shift & low;
                    atomicAdd(&B.count[b], 1u);
                    const uint64_t m = mass_of(funkey(k), top, scale);
                    if (m) atomicAdd(reinterpret_cast<unsigned long long*>(&B.mass[b]), (unsigned long long)m);
                });
                cluster_sync();
                for (int i = tid; i < per; i += WNT) {
                    uint64_t m = 0;
                    uint32_t n = 0;
                    for (int c = 0; c < G; ++c) {
                        m += ld_cluster64(mapa(&B.mass[rank * per + i], c));
                        n += ld_cluster(mapa(&B.count[rank * per + i], c));
                    }
                    B.own_mass[i] = m;
                    B.own_count[i] = n;
                }
                cluster_sync();
                for (int i = tid; i < BINS; i += WNT) {
                    all_mass[i] = ld_cluster64(mapa(&B.own_mass[i % per], i / per));
                    all_count[i] = ld_cluster(mapa(&B.own_count[i % per], i / per));
                }
                __syncthreads();
            };
            // the first bin, from the top, up to whose end there are more than `target` (count or mass)
            auto descend = [&](Found& f, int bits, bool by_mass, uint64_t target, const uint64_t* all_mass,
                               const uint32_t* all_count) {
                constexpr int PB = BINS / WNT;
                uint64_t m[PB], sm = 0;
                uint32_t n[PB], sn = 0;
#pragma unroll
                for (int j = 0; j < PB; ++j) {
                    const int b = BINS - 1 - (tid * PB + j);
                    m[j] = all_mass[b];
                    n[j] = all_count[b];
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
                for (int w = 0; w < warp; ++w) {
                    bm += S.red64[w];
                    bn += S.red32[w];
                }
#pragma unroll
                for (int j = 0; j < PB; ++j) {
                    const uint64_t from = by_mass ? bm : bn, to = from + (by_mass ? m[j] : n[j]);
                    if (from <= target && target < to) {
                        S.bin = uint32_t(BINS - 1 - (tid * PB + j));
                        S.before_mass = bm;
                        S.before_count = bn;
                        S.at_mass = m[j];
                        S.at_count = n[j];
                    }
                    bm += m[j];
                    bn += n[j];
                }
                __syncthreads();
                f.shift -= bits;
                f.key |= S.bin << f.shift;
                f.before_mass = S.before_mass;
                f.before_count = S.before_count;
                f.at_mass = S.at_mass;
                f.at_count = S.at_count;
                __syncthreads();
            };
            // the key at which the count or mass from the top passes `target`
            fill(0u, 21, 11, B.top_mass, B.top_count);
            auto search = [&](bool by_mass, uint64_t target) {
                Found f{0u, 32, 0, 0, 0, 0};
                descend(f, 11, by_mass, target, B.top_mass, B.top_count);
                fill(f.key, 10, 11, B.all_mass, B.all_count);
                descend(f, 11, by_mass, target, B.all_mass, B.all_count);
                fill(f.key, 0, 10, B.all_mass, B.all_count);
                descend(f, 10, by_mass, target, B.all_mass, B.all_count);
                return f;
            };
            // everything that min-p keeps
            uint64_t all = 0;
            uint32_t count = 0;
            for (int i = tid; i < BINS; i += WNT) {
                all += B.top_mass[i];
                count += B.top_count[i];
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
            for (int w = 0; w < NW; ++w) {
                all += S.red64[w];
                count += S.red32[w];
            }
            __syncthreads();
            if (row.K > 0 && uint32_t(row.K) < count) {
                const Found f = search(false, uint64_t(row.K - 1));
                floor_key = f.key;
                all = f.before_mass + f.at_mass;
                count = f.before_count + f.at_count;
            }
            kept = all;
            kept_count = count;
            cut_key = floor_key;
            uint32_t cut_ties = 0xffffffffu;      // of the columns at cut_key
            if (row.p.use_p) {
                const uint64_t limit = part_of(row.p.top_p, all);
                const Found f = search(true, limit);
                const uint64_t m = f.at_mass / f.at_count;
                const uint64_t n = min(uint64_t(f.at_count), (limit - f.before_mass) / m + 1);
                cut_key = f.key;
                cut_ties = uint32_t(n);
                kept = f.before_mass + n * m;
                kept_count = f.before_count + uint32_t(n);
            }
            const uint64_t target = part_of(row.p.u, kept);
            const Found f = search(true, target);
            const uint32_t nth = uint32_t((target - f.before_mass) / (f.at_mass / f.at_count));
            // the n-th column, in ascending order, that has key k (0xffffffff: there is none)
            auto column_of = [&](uint32_t k, uint32_t n) {
                // columns in order: each thread a run of the slice's neighbours
                const int len = c_hi - c_lo, step = (len + WNT - 1) / WNT;
                const int a = min(len, tid * step), z = min(len, a + step);
                auto key_in_order = [&](int i) {
                    if (cached) return cache[i];
                    bool nan;
                    return key_at(c_lo + i, E::load(g.row, c_lo + i), &nan);
                };
                uint32_t ties = 0;
                for (int i = a; i < z; ++i) ties += key_in_order(i) == k;
                const uint32_t upto = warp_incl_scan_u32(ties, lane);
                if (lane == 31) S.red32[warp] = upto;
                __syncthreads();
                uint32_t before = upto - ties, mine = 0;
                for (int w = 0; w < NW; ++w) {
                    if (w < warp) before += S.red32[w];
                    mine += S.red32[w];
                }
                if (tid == 0) {
                    S.ties = mine;
                    S.bin = 0xffffffffu;
                }
                cluster_sync();
                for (uint32_t c = 0; c < rank; ++c) before += ld_cluster(mapa(&S.ties, c));
                if (before <= n && n < before + ties) {
                    uint32_t left = n - before;
                    for (int i = a; i < z; ++i)
                        if (key_in_order(i) == k && left-- == 0) {
                            S.bin = uint32_t(c_lo + i);
                            break;
                        }
                }
                cluster_sync();
                uint32_t col = 0xffffffffu;
                for (int c = 0; c < G; ++c) col = min(col, ld_cluster(mapa(&S.bin, c)));
                cluster_sync();
                return col;
            };
            drawn = int(column_of(f.key, nth));
            if (P.out_probs) cut_col = cut_ties == 0xffffffffu ? 0xffffffffu : column_of(cut_key, cut_ties - 1);
            if (rank == 0 && tid == 0) {
                const double y = double(funkey(f.key)) - double(top);
                write_row(P, r, drawn + P.vocab_offset, float(y - log(double(kept) / scale)), int(kept_count), status);
            }
        }
        if (P.out_probs) {
            float* out = P.out_probs + int64_t(r) * P.vocab;
            const double all = double(kept);
            each_key([&](int c, uint32_t k) {
                float p = 0.0f;
                if (drawn >= 0) {
                    if (row.greedy) p = c == drawn ? 1.0f : 0.0f;
                    else if (k > cut_key || (k == cut_key && uint32_t(c) <= cut_col))
                        p = float(exp(double(funkey(k)) - double(top)) * scale / all);
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
