// fg_logprobs.cuh — log probabilities of given tokens with entropy, rank and
// top alternatives (fg_token_logprobs), and their gradient with respect to the
// logits (fg_token_logprobs_grad).
//
// With m the row's largest logit, c = log2(e) / T and y_j = (x_j - m) c:
//   S = sum_j 2^y_j, Q = sum_j 2^y_j y_j, L2 = log2 S
//   log p_t = ln2 (y_t - L2),  H = ln2 (L2 - Q / S)
// Terms with 2^y_j = 0 (masked columns) add nothing to Q.
#pragma once

#include "fg_common.cuh"

namespace fg {
namespace lp {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float Y_MIN = -1000.0f;   // 2^Y_MIN is 0 in fp32: below it a term is exactly 0

struct Params {
    const void* logits;
    int64_t row_stride;
    int32_t vocab;
    int32_t top;
    const int64_t* tokens;
    const float* temperature;
    float* out_logprobs;
    float* out_entropy;
    float* out_max;
    float* out_logsum;
    int32_t* out_rank;
    int64_t* out_top_ids;
    float* out_top_logprobs;
    int32_t* out_status;
};

struct GradParams {
    const void* logits;
    int64_t row_stride;
    int32_t vocab;
    const int64_t* tokens;
    const float* temperature;
    const float* max;
    const float* logsum;
    const float* entropy;
    const float* grad_logprobs;
    const float* grad_entropy;
    void* out_grad;
    int64_t grad_stride;
};

// The stream's previous kernel is done and its results visible (launches may begin earlier).
__device__ __forceinline__ void wait_prerequisites() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Temperatures: positive, finite and not subnormal (1 / T stays finite).
__device__ __forceinline__ bool temperature_ok(float T) { return T >= 1.17549435e-38f && T < INFINITY; }

// ---------------------------------------------------------------------------
// Forward: one pass over the logits.
//
// A thread takes 16-byte chunks four at a time and keeps, in 32 bits: its largest
// logit; S and Q (above) against a reference that follows its largest logit (lazily: a
// sum may grow to 2^64 above it, so it is rescaled about once); the count of the
// logits ahead of the token's. S and Q are sums of 2^y and 2^y y with y = x c - r:
// one FMA a logit, the same r in every term, so r's rounding cancels in log2 S + r.
// That holds while the rounding is small: |r| stays below FAR, where it is at most half
// a unit of y. A thread whose largest logit is below -3/4 FAR / c keeps no reference, and
// a row whose maximum is not within FAR / (2 c) of 0 is summed a second time, from the
// differences x - m: in the other rows all that was left out is FAR / 4 below the
// maximum, where 2^y is 0.
//
// Alternatives without a second pass over the row: each thread leaves the maxima of up
// to SLOTS stretches of its chunks. The top-th largest of 32 or 64 group maxima bounds
// the top-th largest logit from below, so every alternative lies in a stretch whose maximum
// reaches the bound; there are few, and only their chunks are read again (from L2).
// What reaches the bound is gathered, and a candidate's place is the number of
// candidates ahead of it.
//
// Two kernels share this. rows_kernel: persistent CTAs, CTAS_PER_SM an SM, a row each
// at a time; a thread copies its own chunks to shared memory DEPTH steps ahead
// (asynchronously, no other thread reads them), across the end of a row, so the next
// row's logits arrive while a row is finished. row_kernel: a cluster of G CTAs a row,
// for batches that leave SMs idle otherwise.
//
// Bound: HBM, one read of the logits, for fp32; instruction issue and the rows' ends for
// 16-bit logits (8 instructions and one ex2 a logit). Measured: rows_kernel, 4096 x 152064
// fp32 369 us (6.8 TB/s); 1024 x 128256 bf16 53 us (5.0 TB/s; issue 65 %, ex2 pipe 63 %),
// with 20 alternatives 66 us; 777 x 50257 bf16, one alternative, 28 us. row_kernel: 1 x 256000
// fp32, 20 alternatives, 9.5 us (one launch and a chain of latencies). CTAs an SM, those
// 1024 rows without and with alternatives: two take 4 and 6 us more than three, four 6 and 6
// (fewer steps in flight each).
// ---------------------------------------------------------------------------
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CTAS_PER_SM = 3;       // of rows_kernel
constexpr int UNROLL_LOG = 2;
constexpr int UNROLL = 1 << UNROLL_LOG;   // chunks a thread takes at a time
constexpr int STEP = UNROLL * THREADS;
constexpr int DEPTH = 3;             // steps in flight in rows_kernel
constexpr int RING_BYTES = DEPTH * STEP * 16;
constexpr int SLOTS = 8;             // stretches of a thread's chunks
constexpr int GROUPS = 64;           // of THREADS / 64 neighbouring lanes, for the bound
constexpr int LANES = THREADS / GROUPS;
constexpr int MAX_G = 8;
constexpr int STRETCHES = 64;        // a warp reads again
constexpr int CAND = 256;            // candidates held at once
constexpr float R_STEP = 64.0f;      // how far above its reference a term may be (in log2)
constexpr float FAR = 0x1p24f;       // how far from 0 a reference may be (in log2)

// Order of the alternatives: larger logit first, then smaller id. A larger code
// comes first; 0 is below every element's code.
__device__ __forceinline__ uint64_t order_code(float x, int32_t j) {
    return (uint64_t(fkey(x)) << 32) | uint32_t(~j);
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
          "l"(*reinterpret_cast<uint64_t*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}

// Chunk arithmetic per type. FLOOR replaces -inf (and anything below) in the sums so
// that no term is 0 * inf; the one-pass sums are valid while the row's maximum stays
// well above it and near enough to 0, and x c finite (one_pass_ok); other rows are
// summed again.
template <int DT> struct Chunk;
template <> struct Chunk<FG_DTYPE_F32> {
    static constexpr int WORDS = 4;
    __device__ __forceinline__ static bool one_pass_ok(float m, float c) {
        return c > 1e-20f && c < 1e8f && fabsf(m * c) < 0.5f * FAR;   // (so |m| < 1e27)
    }
    // the largest logit of the words, NaN if any is
    __device__ __forceinline__ static float max_of(const uint32_t* w, int n) {
        float m = __uint_as_float(w[0]);
        for (int i = 1; i < n; ++i) m = fmax_nan(m, __uint_as_float(w[i]));
        return m;
    }
    __device__ __forceinline__ static float2 floored(const uint32_t* w, int pair) {
        return make_float2(fmaxf(__uint_as_float(w[2 * pair]), -1e30f), fmaxf(__uint_as_float(w[2 * pair + 1]), -1e30f));
    }
    static constexpr int PAIRS = 2;   // per chunk
    // the next value below x (finite)
    __device__ __forceinline__ static float below(float x) {
        const uint32_t u = __float_as_uint(x);
        return __uint_as_float(x == 0.0f ? 0x80000001u : (u >> 31) ? u + 1 : u - 1);
    }
    using Threshold = float;
    __device__ __forceinline__ static Threshold threshold(float x) { return x; }
    struct Count {   // logits above a threshold
        int n = 0;
        __device__ __forceinline__ void add(const uint32_t* w, Threshold t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) n += __uint_as_float(w[i]) > t ? 1 : 0;
        }
        __device__ __forceinline__ int take() {
            const int k = n;
            n = 0;
            return k;
        }
    };
};
template <class T2, int DT> struct Chunk16 {
    static constexpr int WORDS = 4;
    static constexpr int PAIRS = 4;
    __device__ __forceinline__ static T2 pack(uint32_t w) { return *reinterpret_cast<T2*>(&w); }
    __device__ __forceinline__ static float max_of(const uint32_t* w, int n) {
        T2 m = pack(w[0]);
        for (int i = 1; i < n; ++i) m = __hmax2_nan(m, pack(w[i]));
        const float2 f = unpack(*reinterpret_cast<uint32_t*>(&m));
        return fmax_nan(f.x, f.y);
    }
    __device__ __forceinline__ static float2 unpack(uint32_t w) {
        if constexpr (DT == FG_DTYPE_F16) return __half22float2(*reinterpret_cast<__half2*>(&w));
        else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    __device__ __forceinline__ static float2 floored(const uint32_t* w, int pair) {
        const uint32_t low = DT == FG_DTYPE_F16 ? 0xfbfffbffu : 0xf149f149u;   // -65504; -9.95e29
        T2 x = __hmax2(pack(w[pair]), pack(low));
        return unpack(*reinterpret_cast<uint32_t*>(&x));
    }
    __device__ __forceinline__ static float below(float x) {
        uint32_t u = DT == FG_DTYPE_F16 ? uint32_t(__half_as_ushort(__float2half_rn(x))) : __float_as_uint(x) >> 16;
        u = x == 0.0f ? 0x8001u : (u >> 15) ? u + 1 : u - 1;
        return DT == FG_DTYPE_F16 ? __half2float(__ushort_as_half(uint16_t(u))) : __uint_as_float(u << 16);
    }
    using Threshold = uint32_t;   // twice
    __device__ __forceinline__ static Threshold threshold(float x) {
        const uint32_t u = DT == FG_DTYPE_F16 ? uint32_t(__half_as_ushort(__float2half_rn(x))) : __float_as_uint(x) >> 16;
        return u | (u << 16);
    }
    // A comparison leaves 0xffff in each half that is above. The plain sum of these
    // words is 2^16 (L - H) - L for L low and H high halves above: no unpacking while
    // L and H stay below 2^15.
    struct Count {
        uint32_t n = 0;
        __device__ __forceinline__ void add(const uint32_t* w, Threshold t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) n += __hgt2_mask(pack(w[i]), pack(t));
        }
        __device__ __forceinline__ int take() {
            const uint32_t low = (0u - n) & 0xffffu;
            const uint32_t high = (low - ((n + low) >> 16)) & 0xffffu;
            n = 0;
            return int(low + high);
        }
    };
};
template <> struct Chunk<FG_DTYPE_F16> : Chunk16<__half2, FG_DTYPE_F16> {
    __device__ __forceinline__ static bool one_pass_ok(float m, float c) {
        return m > -60000.0f && c > 0.03f && c < 1e8f && fabsf(m * c) < 0.5f * FAR;
    }
};
template <> struct Chunk<FG_DTYPE_BF16> : Chunk16<__nv_bfloat162, FG_DTYPE_BF16> {
    __device__ __forceinline__ static bool one_pass_ok(float m, float c) {
        return Chunk<FG_DTYPE_F32>::one_pass_ok(m, c);
    }
};

// Running sums of one thread, even and odd logits apart.
struct Sums {
    float2 s = {0.0f, 0.0f}, q = {0.0f, 0.0f};
    float r = 0.0f;                  // the reference, in log2
    float limit;                     // logits above it move the reference
    bool set = false;
    __device__ __forceinline__ explicit Sums(float T) : limit(fmaxf(-9.9e29f, -0.75f * FAR * LN2 * T)) {}
    __device__ __forceinline__ void follow(float m, float c) {   // m: the largest of the next logits
        if (m > limit) {
            const float to = m * c;
            const float f = set ? exp2_fast(r - to) : 0.0f;
            const float d = set ? r - to : 0.0f;
            q = make_float2(f * fmaf(d, s.x, q.x), f * fmaf(d, s.y, q.y));
            s = make_float2(f * s.x, f * s.y);
            r = to;
            limit = m + R_STEP / c;
            set = true;
        }
    }
    // a step's sums on their own first: the long sums' rounding errors stay few
    struct Part {
        float2 s = {0.0f, 0.0f}, q = {0.0f, 0.0f};
    };
    __device__ __forceinline__ void term(Part& p, float2 x, float c) const {   // floored logits
        const float2 y = fma2(x, make_float2(c, c), make_float2(-r, -r));
        const float2 e = make_float2(exp2_fast(y.x), exp2_fast(y.y));
        p.s = add2(p.s, e);
        p.q = fma2(e, y, p.q);
    }
    __device__ __forceinline__ void add(const Part& p) {
        s = add2(s, p.s);
        q = add2(q, p.q);
    }
};

// The warp's maximum, NaN if any lane has one (redux on fp32, sm_100a).
__device__ __forceinline__ float warp_max_nan(float x) {
    float m;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
    return m;
}

// What a warp, a CTA and a row add up to: S and Q against the largest logit.
struct alignas(16) Stats {   // (other CTAs write one as 16 bytes)
    float m, s, q;
    int n;   // logits ahead of the token's
};
__device__ __forceinline__ Stats merge(const Stats& a, float m, float c) {   // a against a larger maximum m
    Stats r = a;
    if (a.m != m) {
        const float d = fmaxf((a.m - m) * c, Y_MIN);
        const float f = exp2_fast(d);
        r.q = f * fmaf(d, a.s, a.q);
        r.s = f * a.s;
    }
    r.m = m;
    return r;
}

// The k-th largest of 32 or 64 group maxima, one or two a lane: a warp-wide bitonic
// sort (of both halves, then of the larger ones of both). Counting for each how many
// exceed it has no chain of shuffles, but more to issue: 1024 x 128256 bf16, 20
// alternatives, 68.5 us against 66.2.
template <bool TWO>
__device__ __forceinline__ float kth_largest(float a, float b, int k, int lane) {
    constexpr uint32_t ALL = 0xffffffffu;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const bool keep_max = ((lane & size) == 0) == ((lane & d) == 0);
            const float o = __shfl_xor_sync(ALL, a, d);
            a = keep_max ? fmaxf(a, o) : fminf(a, o);
            if (TWO) {
                const float p = __shfl_xor_sync(ALL, b, d);
                b = keep_max ? fmaxf(b, p) : fminf(b, p);
            }
        }
    if (TWO) {
        a = fmaxf(a, __shfl_xor_sync(ALL, b, 31));   // descending a against ascending b
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const float o = __shfl_xor_sync(ALL, a, d);
            a = (lane & d) == 0 ? fmaxf(a, o) : fminf(a, o);
        }
    }
    return __shfl_sync(ALL, a, k - 1);
}

// A row's place in shared memory; what a row leaves before its first barrier alternates
// between two places, since a thread may be a row ahead of another by then.
struct alignas(128) Shared {
    Stats warp[2][WARPS];
    float groups[2][GROUPS];
    int count[2];                                // candidates
    uint16_t stretch[WARPS][STRETCHES];          // thread | slot << 8
    float slots[SLOTS][THREADS];                 // a thread's stretches' maxima (its own column)
    uint64_t cand[CAND];
};
struct alignas(16) ClusterShared {
    Stats cta[MAX_G];                            // every CTA of the cluster writes its entry
    uint64_t lists[MAX_G][FG_LOGPROB_MAX_TOP];   // the CTAs' best (in the first CTA)
};

__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// One row's geometry and parameters: scalars before the first and after the last
// whole chunk, and this CTA's chunks.
template <int DT>
struct Row {
    static constexpr int VEC = Elem<DT>::VEC, SIZE = Elem<DT>::SIZE;
    const char* p;
    int64_t r, tok;
    int V, head, nvec, tail, c0, c1;
    int tchunk;        // chunks before the token's count equal logits as ahead of it, the others do not
    float T, xt, c;
    typename Chunk<DT>::Threshold above, from;   // thresholds after and before the token
    bool given;
    __device__ __forceinline__ Row(const Params& P, int64_t row, int part, int parts)
        : Row(P, row, part, parts, P.tokens ? P.tokens[row] : -1, P.temperature ? P.temperature[row] : 1.0f,
              token_logit(P, row, P.tokens ? P.tokens[row] : -1)) {}
    __device__ __forceinline__ static float token_logit(const Params& P, int64_t row, int64_t token) {
        return token >= 0 && token < P.vocab ? Elem<DT>::load(P.logits, row * P.row_stride + token) : INFINITY;
    }
    __device__ __forceinline__ Row(const Params& P, int64_t row, int part, int parts, int64_t token, float temperature,
                                   float logit)
        : r(row), tok(token), T(temperature), xt(logit) {
        p = reinterpret_cast<const char*>(P.logits) + r * P.row_stride * SIZE;
        V = P.vocab;
        head = min(V, int((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / SIZE);
        nvec = (V - head) / VEC;
        tail = V - head - nvec * VEC;
        c0 = nvec / parts * part + min(part, nvec % parts);
        c1 = c0 + nvec / parts + (part < nvec % parts ? 1 : 0);
        given = tok >= 0 && tok < V;
        c = LOG2E / T;
        tchunk = !given || tok < head ? -1 : int((tok - head) / VEC);
        above = Chunk<DT>::threshold(xt);
        from = Chunk<DT>::threshold(Chunk<DT>::below(xt));
    }
    __device__ __forceinline__ const uint4* chunks() const {
        return reinterpret_cast<const uint4*>(p + int64_t(head) * SIZE);
    }
    __device__ __forceinline__ int id(int chunk) const { return head + chunk * VEC; }
    __device__ __forceinline__ int scalar_id(int i) const { return i < head ? i : V - tail + (i - head); }
};

// What one thread gathers in the pass.
template <int DT>
struct Pass {
    using C = Chunk<DT>;
    Sums acc;
    typename C::Count above;
    float vmax = -INFINITY;   // NaN if any logit is
    float smax = -INFINITY;   // of the stretch at hand
    int n = 0;
    __device__ __forceinline__ explicit Pass(const Row<DT>& row) : acc(row.T) {}
    // a step is done: at the end of a stretch of 2^log steps its maximum is left behind
    __device__ __forceinline__ void stretch(Shared& sh, int step, int log, bool last) {
        if (((step + 1) & ((1 << log) - 1)) == 0 || last) {
            sh.slots[step >> log][threadIdx.x] = smax;
            smax = -INFINITY;
        }
    }
    // U chunks (those past the row's end hold -inf); t[u]: the threshold of chunk u
    template <int U>
    __device__ __forceinline__ void take(const uint32_t (&w)[4 * U], const Row<DT>& row,
                                         const typename C::Threshold (&t)[U]) {
        const float m = C::max_of(w, U * 4);
        vmax = fmax_nan(vmax, m);
        smax = fmaxf(smax, m);
        acc.follow(m, row.c);
        Sums::Part part;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < C::PAIRS; ++i) acc.term(part, C::floored(w + 4 * u, i), row.c);
        acc.add(part);
        if (m >= row.xt) {   // (chunks past the end hold -inf: never above a threshold)
#pragma unroll
            for (int u = 0; u < U; ++u) above.add(w + 4 * u, t[u]);
        }
    }
    // UNROLL chunks from the ci-th on
    __device__ __forceinline__ void take(const uint32_t (&w)[4 * UNROLL], const Row<DT>& row, int ci) {
        typename C::Threshold t[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) t[u] = ci + u * THREADS < row.tchunk ? row.from : row.above;
        take<UNROLL>(w, row, t);
    }
    // at least every 512 steps: 2^15 above in a half would be too many
    __device__ __forceinline__ void settle() { n += above.take(); }
    // The ragged ends, a logit a thread, and the equal logits in the token's own chunk.
    // Their loads are begun before the pass, so that its end does not wait for them.
    float end, own;
    __device__ __forceinline__ void begin(const Row<DT>& row, int scalars, int tid) {
        end = -INFINITY;
        own = __int_as_float(0x7fc00000);
        if (tid < scalars) end = Elem<DT>::load(row.p, row.scalar_id(tid));
        if (row.tchunk >= row.c0 && row.tchunk < row.c1 && tid < Row<DT>::VEC && row.id(row.tchunk) + tid < row.tok)
            own = Elem<DT>::load(row.p, row.id(row.tchunk) + tid);
    }
    __device__ __forceinline__ void ends(const Row<DT>& row, int scalars, int tid) {
        settle();
        if (tid < scalars) {
            const float low = DT == FG_DTYPE_F16 ? -65504.0f : -1e30f;
            vmax = fmax_nan(vmax, end);
            acc.follow(end, row.c);
            Sums::Part part;
            acc.term(part, make_float2(fmaxf(end, low), low), row.c);   // (low adds 0)
            acc.add(part);
            if (row.given) n += (end > row.xt || (end == row.xt && row.scalar_id(tid) < row.tok)) ? 1 : 0;
        }
        n += own == row.xt ? 1 : 0;
        // nothing is below -inf: a masked token has every logit before it ahead of it
        if (tid == 0 && row.xt == -INFINITY) n += max(0, min(row.c1, row.tchunk) - row.c0) * Row<DT>::VEC;
    }
};

// Steps of a stretch (its log2), so that SLOTS stretches hold all steps.
__device__ __forceinline__ int stretch_log(int steps) {
    int log = 0;
    while ((SLOTS << log) < steps) ++log;
    return log;
}

template <int DT>
__device__ __forceinline__ uint4 no_logits() {   // a chunk of -inf
    const uint32_t w = DT == FG_DTYPE_F32 ? 0xff800000u : DT == FG_DTYPE_F16 ? 0xfc00fc00u : 0xff80ff80u;
    return make_uint4(w, w, w, w);
}

// From the threads' sums to the row's results; chunk i of the CTA's belongs to thread
// (i - c0) % THREADS.
template <int DT, bool TOP, bool CLUSTER>
__device__ __forceinline__ void finish_row(const Params& P, Shared& sh, ClusterShared* cl, const Row<DT>& row,
                                           const Pass<DT>& pass, int scalars, int part, int G, int flip) {
    constexpr int VEC = Elem<DT>::VEC;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float c = row.c, T = row.T, vmax = pass.vmax;
    const int64_t r = row.r;
    const uint4* chunks = row.chunks();

    // ---- the warp, then the CTA ----
    if (TOP) {
        float gm = vmax;
#pragma unroll
        for (int d = 1; d < LANES; d <<= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, d));
        if ((lane & (LANES - 1)) == 0) sh.groups[flip][tid / LANES] = gm;
    }
    {
        Stats st;
        st.m = warp_max_nan(vmax);
        st.n = __reduce_add_sync(0xffffffffu, pass.n);
        st.s = st.q = 0.0f;
        if (pass.acc.set) {
            const float d = fmaxf(fmaf(-st.m, c, pass.acc.r), Y_MIN);   // the reference against the warp's maximum
            const float f = exp2_fast(d);
            st.s = f * (pass.acc.s.x + pass.acc.s.y);
            st.q = f * fmaf(d, pass.acc.s.x + pass.acc.s.y, pass.acc.q.x + pass.acc.q.y);
        }
        float2 sq = make_float2(st.s, st.q);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
            sq = add2(sq, make_float2(__shfl_xor_sync(0xffffffffu, sq.x, d), __shfl_xor_sync(0xffffffffu, sq.y, d)));
        st.s = sq.x;
        st.q = sq.y;
        if (lane == 0) sh.warp[flip][warp] = st;
    }
    __syncthreads();
    if (tid == 0) sh.count[flip ^ 1] = 0;   // everyone is done with the row before
    // the sums of up to 16 entries, a lane an entry (same_max: all against one maximum)
    auto fold = [&](const Stats* from, int count, bool same_max) {
        Stats st{-INFINITY, 0.0f, 0.0f, 0};
        if (lane < count) st = from[lane];
        const float m = warp_max_nan(st.m);
        if (!same_max) st = merge(st, m, c);
        st.n = __reduce_add_sync(0xffffffffu, st.n);
        float2 sq = make_float2(st.s, st.q);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1)
            sq = add2(sq, make_float2(__shfl_xor_sync(0xffffffffu, sq.x, d), __shfl_xor_sync(0xffffffffu, sq.y, d)));
        return Stats{m, __shfl_sync(0xffffffffu, sq.x, 0), __shfl_sync(0xffffffffu, sq.y, 0), st.n};
    };
    // Every warp needs the row's maximum; its sums only where results are written.
    Stats all{0.0f, 0.0f, 0.0f, 0};
    if (CLUSTER || TOP || warp == 0) all = fold(sh.warp[flip], WARPS, false);
    else all.m = warp_max_nan(sh.warp[flip][lane & (WARPS - 1)].m);

    // ---- alternatives: the candidates of this CTA ----
    int ncand = 0;
    if (TOP) {
        // 32 groups are enough for a tight bound up to 16 alternatives (of n groups the
        // k-th largest maximum lets about n (H_n - H_(n - k)) logits through: 31 for k = 20,
        // but 130 for k = 32; of 64 groups 24 and 44)
        const float g0 = sh.groups[flip][2 * lane], g1 = sh.groups[flip][2 * lane + 1];
        const float bound = P.top <= 16 ? kth_largest<false>(fmaxf(g0, g1), 0.0f, P.top, lane)
                                        : kth_largest<true>(g0, g1, P.top, lane);
        const bool wins = vmax >= bound;
        const uint32_t winners = __ballot_sync(0xffffffffu, wins);
        auto put = [&](uint64_t code) {
            const int at = atomicAdd(&sh.count[flip], 1);
            if (at < CAND) sh.cand[at] = code;
        };
        if (bound > -INFINITY) {
            // the warp's stretches that reach the bound, their chunks a lane each
            const int steps = (row.c1 - row.c0 + STEP - 1) / STEP, log = stretch_log(steps);
            const int used = (steps + (1 << log) - 1) >> log;
            int total = 0;
            if (winners) {
#pragma unroll
                for (int i = 0; i < SLOTS; ++i) {
                    const bool in = wins && i < used && sh.slots[i][tid] >= bound;
                    const uint32_t b = __ballot_sync(0xffffffffu, in);
                    const int at = total + __popc(b & ((1u << lane) - 1));
                    if (in && at < STRETCHES) sh.stretch[warp][at] = uint16_t(tid | (i << 8));
                    total += __popc(b);
                }
            }
            __syncwarp();
            if (total > STRETCHES) {
                if (lane == 0) atomicAdd(&sh.count[flip], CAND + 1);   // too many
                total = 0;
            }
#pragma unroll 2
            for (int i = lane; i < total << (log + UNROLL_LOG); i += 32) {
                const int e = sh.stretch[warp][i >> (log + UNROLL_LOG)], k = i & ((UNROLL << log) - 1);
                const int ci = row.c0 + (((e >> 8) << log) + (k >> UNROLL_LOG)) * STEP + (k & (UNROLL - 1)) * THREADS + (e & 255);
                if (ci < row.c1) {
                    const uint4 v = __ldg(chunks + ci);
                    if (Chunk<DT>::max_of(&v.x, 4) >= bound) {
                        float x[VEC];
                        Elem<DT>::unpack(v, x);
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            if (x[e] >= bound) put(order_code(x[e], row.id(ci) + e));
                    }
                }
            }
            if (tid < scalars && pass.end >= bound) put(order_code(pass.end, row.scalar_id(tid)));
        }
        __syncthreads();
        ncand = sh.count[flip];
        if (ncand > CAND || !(bound > -INFINITY)) {
            // too many at or above the bound (ties, long runs in order), or a bound of -inf:
            // each warp keeps its best 32 in its lanes and inserts what beats the last
            __syncthreads();
            if (tid == 0) sh.count[flip] = 0;
            __syncthreads();
            uint64_t best = 0;
            auto insert = [&](uint64_t code) {
                uint32_t better;
                while ((better = __ballot_sync(0xffffffffu, code > shfl_u64(best, 31)))) {
                    const uint64_t v = shfl_u64(code, __ffs(better) - 1);
                    const uint64_t up = shfl_up_u64(best, 1);
                    const int place = __popc(__ballot_sync(0xffffffffu, best > v));
                    best = lane < place ? best : lane == place ? v : up;
                    if (lane == __ffs(better) - 1) code = 0;
                }
            };
            // the warp's chunks in the order of their ids, four loads in flight: once the list
            // is full, a chunk counts only with a logit above its last (a later equal one loses)
            for (int first = row.c0 + (tid & ~31); first < row.c1; first += 4 * THREADS) {
                uint4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    v[u] = no_logits<DT>();
                    const int ci = first + u * THREADS + lane;
                    if (ci < row.c1) v[u] = __ldg(chunks + ci);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int ci = first + u * THREADS + lane;
                    const uint64_t last = shfl_u64(best, 31);
                    const bool above = last == 0 || Chunk<DT>::max_of(&v[u].x, 4) > funkey(uint32_t(last >> 32));
                    if (!__any_sync(0xffffffffu, ci < row.c1 && above)) continue;
                    float x[VEC];
                    Elem<DT>::unpack(v[u], x);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) insert(ci < row.c1 ? order_code(x[e], row.id(ci) + e) : 0);
                }
            }
            if (scalars > 0 && warp == 0)
                insert(lane < scalars ? order_code(pass.end, row.scalar_id(lane)) : 0);
            if (lane >= P.top) best = 0;
            if (best != 0) put(best);
            __syncthreads();
            ncand = min(CAND, sh.count[flip]);
        }
    }
    // a candidate's place is the number of candidates ahead of it
    auto place_of = [&](uint64_t code) {
        int ahead = 0;
#pragma unroll 4
        for (int i = 0; i < ncand; ++i) ahead += sh.cand[i] > code;
        return ahead;
    };

    // ---- the row ----
    if constexpr (CLUSTER) {
        cluster_wait();
        if (warp == 0 && lane < G) {
            const uint32_t to = cluster_addr(&cl->cta[part], lane);
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};"
                         :: "r"(to), "f"(all.m), "f"(all.s), "f"(all.q), "f"(__int_as_float(all.n)) : "memory");
        }
        if (TOP) {
            const uint32_t lists = cluster_addr(&cl->lists[part][0], 0);
            if (tid < ncand) {
                const int place = place_of(sh.cand[tid]);
                if (place < P.top)
                    asm volatile("st.shared::cluster.u64 [%0], %1;"
                                 :: "r"(lists + 8 * place), "l"(sh.cand[tid]) : "memory");
            }
            if (tid < P.top && tid >= ncand)
                asm volatile("st.shared::cluster.u64 [%0], %1;" :: "r"(lists + 8 * tid), "l"(uint64_t(0)) : "memory");
        }
        cluster_arrive();
        cluster_wait();
        all = fold(cl->cta, G, false);
    }
    const float m = all.m;
    int status = 0;
    if (isnan(m)) status |= FG_ROW_NAN;
    if (m == INFINITY) status |= FG_ROW_POS_INF;
    if (m == -INFINITY) status |= FG_ROW_ALL_MASKED;
    if (!temperature_ok(T) || row.tok >= row.V) status |= FG_ROW_BAD_PARAM;
    const bool bad = (status & ~FG_ROW_ALL_MASKED) != 0;
    const bool empty = m == -INFINITY;

    if (!bad && !empty && !Chunk<DT>::one_pass_ok(m, c)) {
        // the sums again, as differences from the row's maximum
        float s = 0.0f, q = 0.0f;
        auto add = [&](float x) {
            const float y = fmaxf((x - m) * c, Y_MIN);
            const float e = exp2_fast(y);
            s += e;
            q = fmaf(e, y, q);
        };
        for (int ci = row.c0 + tid; ci < row.c1; ci += THREADS) {
            float x[VEC];
            Elem<DT>::unpack(__ldg(chunks + ci), x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) add(x[e]);
        }
        if (tid < scalars) add(Elem<DT>::load(row.p, row.scalar_id(tid)));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, d);
            q += __shfl_xor_sync(0xffffffffu, q, d);
        }
        __syncthreads();
        if (lane == 0) sh.warp[flip][warp] = Stats{m, s, q, 0};
        __syncthreads();
        Stats again = fold(sh.warp[flip], WARPS, true);
        if constexpr (CLUSTER) {
            cluster_arrive();   // everyone has read the first round's entries
            cluster_wait();
            if (warp == 0 && lane < G) {
                const uint32_t to = cluster_addr(&cl->cta[part], lane);
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};"
                             :: "r"(to), "f"(m), "f"(again.s), "f"(again.q), "f"(0.0f) : "memory");
            }
            cluster_arrive();
            cluster_wait();
            again = fold(cl->cta, G, true);
        }
        all.s = again.s;
        all.q = again.q;
    }
    if (part != 0) return;
    const float l2 = log2f(all.s);
    const float nan = __int_as_float(0x7fc00000);
    // one expression for the token and the alternatives: the same id has the same bits
    auto logprob = [&](float x) { return __fmaf_rn(-LN2, l2, __fdiv_rn(x - m, T)); };
    if (tid == 0) {
        const float lpt = row.tok < 0 ? 0.0f : empty ? -INFINITY : logprob(row.xt);
        if (P.out_logprobs) P.out_logprobs[r] = bad ? nan : lpt;
        if (P.out_entropy) P.out_entropy[r] = bad ? nan : empty ? 0.0f : LN2 * (l2 - all.q / all.s);
        if (P.out_max) P.out_max[r] = m;
        if (P.out_logsum) P.out_logsum[r] = bad ? nan : empty ? -INFINITY : LN2 * l2;
        if (P.out_rank) P.out_rank[r] = (bad || row.tok < 0) ? -1 : all.n;
        if (P.out_status) P.out_status[r] = status;
    }
    if (TOP) {
        auto write = [&](int i, bool none, uint64_t code) {
            const float x = funkey(uint32_t(code >> 32));
            if (P.out_top_ids) P.out_top_ids[r * P.top + i] = (none || bad) ? -1 : int64_t(uint32_t(~uint32_t(code)));
            if (P.out_top_logprobs)
                P.out_top_logprobs[r * P.top + i] =
                    bad ? nan : (none || x == -INFINITY) ? -INFINITY : logprob(x);
        };
        if constexpr (CLUSTER) {
            // G lists in order, an entry a thread
            const int g = tid / FG_LOGPROB_MAX_TOP, j = tid % FG_LOGPROB_MAX_TOP;
            if (g < G && j < P.top) {
                const uint64_t code = cl->lists[g][j];
                int place = 0;
                // each list is in order: halving, not counting (1 x 256000 f32: 9.5 us against 10.6)
                for (int o = 0; o < G; ++o) {
                    int ahead = 0;
#pragma unroll
                    for (int d = FG_LOGPROB_MAX_TOP; d > 0; d >>= 1)
                        if (ahead + d <= P.top && cl->lists[o][ahead + d - 1] > code) ahead += d;
                    place += ahead;
                }
                if (code != 0 && place < P.top) write(place, false, code);
            }
        } else if (tid < ncand) {
            const int place = place_of(sh.cand[tid]);
            if (place < P.top) write(place, false, sh.cand[tid]);
        }
        // past the vocabulary's end, and rows that have no alternatives to name
        if (tid < P.top && (tid >= row.V || bad)) write(tid, true, 0);
    }
}

template <int DT, bool TOP>
__global__ void __launch_bounds__(THREADS) row_kernel(const Params P, const int G) {
    __shared__ Shared sh;
    __shared__ ClusterShared cl;
    static_assert(MAX_G * FG_LOGPROB_MAX_TOP <= THREADS && CAND <= THREADS && THREADS <= 256, "a thread an entry");
    const int tid = threadIdx.x, part = blockIdx.x % G;
    cluster_arrive();   // the others' shared memory stands once all have arrived
    if (tid == 0) sh.count[0] = 0;
    wait_prerequisites();
    const Row<DT> row(P, blockIdx.x / G, part, G);
    const uint4* chunks = row.chunks();
    Pass<DT> pass(row);
    const int scalars = part == 0 ? row.head + row.tail : 0;
    pass.begin(row, scalars, tid);
    const int steps = (row.c1 - row.c0 + STEP - 1) / STEP, log = stretch_log(steps);
    uint4 ahead[UNROLL];
    auto fetch = [&](int step) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int ci = row.c0 + step * STEP + u * THREADS + tid;
            ahead[u] = no_logits<DT>();
            if (ci < row.c1) ahead[u] = __ldg(chunks + ci);
        }
    };
    fetch(0);
    for (int step = 0; step < steps; ++step) {
        uint32_t w[UNROLL * 4];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            w[4 * u] = ahead[u].x; w[4 * u + 1] = ahead[u].y; w[4 * u + 2] = ahead[u].z; w[4 * u + 3] = ahead[u].w;
        }
        fetch(step + 1);
        pass.take(w, row, row.c0 + step * STEP + tid);
        if (TOP) pass.stretch(sh, step, log, step + 1 == steps);
        if ((step & 511) == 511) pass.settle();
    }
    pass.ends(row, scalars, tid);
    finish_row<DT, TOP, true>(P, sh, &cl, row, pass, scalars, part, G, 0);
}

static_assert(sizeof(Shared) % 128 == 0 && offsetof(ClusterShared, cta) % 16 == 0 && sizeof(Stats) == 16, "alignment");

template <int DT, bool TOP>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) rows_kernel(const Params P, const int64_t batch) {
    extern __shared__ __align__(128) uint4 ring[];   // [DEPTH][UNROLL][THREADS]
    __shared__ Shared sh;
    constexpr int SIZE = Elem<DT>::SIZE;
    const int tid = threadIdx.x;
    const uint32_t ring0 = smem_u32(ring) + 16 * tid, ring1 = ring0 + RING_BYTES;
    if (tid == 0) sh.count[0] = 0;
    wait_prerequisites();

    // ---- the copies: `left` chunks of row `next` from `src` on ----
    int64_t next = blockIdx.x;
    const char* src = nullptr;
    int left = 0;
    auto open = [&]() {
        const char* p = reinterpret_cast<const char*>(P.logits) + next * P.row_stride * SIZE;
        const int head = min(P.vocab, int((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / SIZE);
        left = (P.vocab - head) / Elem<DT>::VEC;
        src = p + int64_t(head) * SIZE + 16 * tid;
    };
    // one step of this thread into a place of the ring (an empty step past the last row)
    auto fetch = [&](uint32_t place) {
        if (left >= STEP) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                             :: "r"(place + 16 * THREADS * u), "l"(src + 16 * THREADS * u) : "memory");
        } else if (left > 0) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
                if (tid + u * THREADS < left)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                 :: "r"(place + 16 * THREADS * u), "l"(src + 16 * THREADS * u) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        src += 16 * STEP;
        left -= STEP;
        while (left <= 0 && next + gridDim.x < batch) {
            next += gridDim.x;
            open();
        }
    };
    open();
    while (left <= 0 && next + gridDim.x < batch) {
        next += gridDim.x;
        open();
    }
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) fetch(ring0 + i * 16 * STEP);

    uint32_t place = ring0;
    int flip = 0;
    int64_t tok = P.tokens ? P.tokens[blockIdx.x] : -1;
    float T = P.temperature ? P.temperature[blockIdx.x] : 1.0f;
    float xt = Row<DT>::token_logit(P, blockIdx.x, tok);
    for (int64_t r = blockIdx.x; r < batch; r += gridDim.x, flip ^= 1) {
        const Row<DT> row(P, r, 0, 1, tok, T, xt);
        const bool more = r + gridDim.x < batch;
        if (more) {   // the next row's, for when its turn comes
            if (P.tokens) tok = P.tokens[r + gridDim.x];
            if (P.temperature) T = P.temperature[r + gridDim.x];
        }
        Pass<DT> pass(row);
        const int scalars = row.head + row.tail;
        pass.begin(row, scalars, tid);
        auto turn = [&]() {   // the values are used: the place is free
            fetch(place);
            place += 16 * STEP;
            if (place == ring1) place = ring0;
        };
        const int steps = (row.nvec + STEP - 1) / STEP, log = stretch_log(steps);
        int c0 = 0, step = 0;
        for (; c0 + STEP <= row.nvec; c0 += STEP, ++step) {
            asm volatile("cp.async.wait_group %0;" :: "n"(DEPTH - 1) : "memory");
            uint32_t w[UNROLL * 4];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const uint4 v = lds_v4(place + 16 * THREADS * u);
                w[4 * u] = v.x; w[4 * u + 1] = v.y; w[4 * u + 2] = v.z; w[4 * u + 3] = v.w;
            }
            if (unsigned(row.tchunk - c0) < unsigned(STEP)) {   // the token's own step
                pass.take(w, row, c0 + tid);
            } else {
                typename Chunk<DT>::Threshold t[UNROLL];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) t[u] = c0 < row.tchunk ? row.from : row.above;
                pass.template take<UNROLL>(w, row, t);
            }
            turn();
            if (TOP) pass.stretch(sh, step, log, step + 1 == steps);
            if ((step & 511) == 511) pass.settle();
        }
        if (c0 < row.nvec) {
            asm volatile("cp.async.wait_group %0;" :: "n"(DEPTH - 1) : "memory");
            if (row.nvec - c0 <= THREADS) {
                // one chunk a thread: the work of one (444 x 50257 bf16: 18.7 us, as a whole step 20.4)
                const int ci = c0 + tid;
                const uint4 v = ci < row.nvec ? lds_v4(place) : no_logits<DT>();
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                const typename Chunk<DT>::Threshold t[1] = {ci < row.tchunk ? row.from : row.above};
                pass.template take<1>(w, row, t);
            } else {
                uint32_t w[UNROLL * 4];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    uint4 v = no_logits<DT>();
                    if (c0 + tid + u * THREADS < row.nvec) v = lds_v4(place + 16 * THREADS * u);
                    w[4 * u] = v.x; w[4 * u + 1] = v.y; w[4 * u + 2] = v.z; w[4 * u + 3] = v.w;
                }
                pass.take(w, row, c0 + tid);
            }
            turn();
            if (TOP) pass.stretch(sh, step, log, true);
        }
        if (more) xt = Row<DT>::token_logit(P, r + gridDim.x, tok);
        pass.ends(row, scalars, tid);
        finish_row<DT, TOP, false>(P, sh, nullptr, row, pass, scalars, 0, 1, flip);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------------------
// Gradient: dx_j = p_j (a + b y_j) + 1[j == t] g / T with y_j = (x_j - m) c - L2,
// p_j = 2^y_j, a = -(g + h H) / T and b = -h ln2 / T.
//
// Bound: HBM, the logits read and the gradient written once. Work is cut along the
// gradient's 16-byte chunks; where the logits' rows are offset against the
// gradient's, a thread takes the two chunks around its own and shifts them together.
// Measured: 1024 x 128256 bf16 85 us (6.2 TB/s; two chunks in flight a thread 4 us more,
// one step a CTA 16 more), 2048 x 50257 fp32 128 us (6.4 TB/s; 17 more, 16 more); 333 x
// 32001 f16 13.6 us; 8 x 50257 fp32 2.9 us.
// ---------------------------------------------------------------------------
constexpr int GRAD_THREADS = 256;
constexpr int GRAD_UNROLL = 4;   // chunks in flight a thread

// Coherent loads: the gradient may overwrite the logits.
template <int DT>
__device__ __forceinline__ float load_rw(const char* row, int64_t j) {
    if constexpr (DT == FG_DTYPE_F32) return reinterpret_cast<const float*>(row)[j];
    else if constexpr (DT == FG_DTYPE_F16) return __half2float(reinterpret_cast<const __half*>(row)[j]);
    else return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[j]);
}

// The 16 bytes that start `shift` bytes into a:b.
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int shift) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (shift & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (shift & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (shift & 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

struct GradRow {
    float m, c, l2, a, b;
    __device__ __forceinline__ float at(float x) const {
        const float y = fmaxf(fmaf(x - m, c, -l2), Y_MIN);
        return exp2_fast(y) * fmaf(b, y, a);
    }
    __device__ __forceinline__ float2 at(float2 x) const {
        float2 y = fma2(add2(x, make_float2(-m, -m)), make_float2(c, c), make_float2(-l2, -l2));
        y = make_float2(fmaxf(y.x, Y_MIN), fmaxf(y.y, Y_MIN));
        const float2 d = fma2(make_float2(b, b), y, make_float2(a, a));
        return make_float2(exp2_fast(y.x) * d.x, exp2_fast(y.y) * d.y);
    }
};

template <int DT>
__device__ __forceinline__ uint4 pack_chunk(const float (&x)[Elem<DT>::VEC]) {
    uint32_t w[4];
    if constexpr (DT == FG_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == FG_DTYPE_F16) {
                const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// CTA blockIdx.x: part blockIdx.x % per_row of row blockIdx.x / per_row.
template <int DT>
__global__ void __launch_bounds__(GRAD_THREADS) logprob_grad_kernel(const GradParams P, const int per_row) {
    wait_prerequisites();
    constexpr int VEC = Elem<DT>::VEC, SIZE = Elem<DT>::SIZE;
    const int64_t r = blockIdx.x / per_row;
    const int part = blockIdx.x % per_row, tid = threadIdx.x;
    const int V = P.vocab;
    const char* in = reinterpret_cast<const char*>(P.logits) + r * P.row_stride * SIZE;
    char* out = reinterpret_cast<char*>(P.out_grad) + r * P.grad_stride * SIZE;
    const int64_t tok = P.tokens ? P.tokens[r] : -1;
    const float T = P.temperature ? P.temperature[r] : 1.0f;
    const float g = (P.grad_logprobs && tok >= 0) ? P.grad_logprobs[r] : 0.0f;
    const float h = P.grad_entropy ? P.grad_entropy[r] : 0.0f;
    GradRow G;
    G.m = P.max[r];
    G.l2 = P.logsum[r] * LOG2E;
    G.c = LOG2E / T;
    G.a = -(g + (h != 0.0f ? h * P.entropy[r] : 0.0f)) / T;
    G.b = -h * LN2 / T;
    const bool bad = !temperature_ok(T) || tok >= V || isnan(G.l2) || isnan(G.m);
    const bool zero = (g == 0.0f && h == 0.0f) || (G.m == -INFINITY && !bad);
    if (bad) G.a = __int_as_float(0x7fc00000);
    const float hit = g / T;

    const int head = min(V, int((16 - (reinterpret_cast<uintptr_t>(out) & 15)) & 15) / SIZE);
    const int nvec = (V - head) / VEC;
    uint4* dst = reinterpret_cast<uint4*>(out + int64_t(head) * SIZE);
    const char* src = in + int64_t(head) * SIZE;
    const int shift = int(reinterpret_cast<uintptr_t>(src) & 15);
    const uint4* aligned = reinterpret_cast<const uint4*>(src - shift);
    // chunks whose two aligned neighbours lie within the row
    const int safe0 = shift > head * SIZE ? 1 : 0;
    const int safe1 = shift == 0 ? nvec : (V - head) * SIZE + shift >= 32 ? ((V - head) * SIZE + shift) / 16 - 1 : 0;
    const int c0 = int(int64_t(nvec) * part / per_row), c1 = int(int64_t(nvec) * (part + 1) / per_row);
    for (int first = c0 + tid; first < c1; first += GRAD_UNROLL * GRAD_THREADS) {
        uint4 v[GRAD_UNROLL];
        if (!zero) {
#pragma unroll
            for (int u = 0; u < GRAD_UNROLL; ++u) {
                const int i = first + u * GRAD_THREADS;
                if (i >= c1) break;
                if (shift == 0) {
                    v[u] = aligned[i];
                } else if (i >= safe0 && i < safe1) {
                    v[u] = shifted(aligned[i], aligned[i + 1], shift);
                } else {
                    float x[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) x[e] = load_rw<DT>(src, int64_t(i) * VEC + e);
                    v[u] = pack_chunk<DT>(x);   // back to the bits they came from
                }
            }
        }
#pragma unroll
        for (int u = 0; u < GRAD_UNROLL; ++u) {
            const int i = first + u * GRAD_THREADS;
            if (i >= c1) break;
            float x[VEC];
            if (zero) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[e] = 0.0f;
            } else {
                Elem<DT>::unpack(v[u], x);
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const float2 d = G.at(make_float2(x[e], x[e + 1]));
                    x[e] = d.x;
                    x[e + 1] = d.y;
                }
                const int64_t at = tok - (head + int64_t(i) * VEC);
                if (at >= 0 && at < VEC) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (e == at) x[e] += hit;
                }
            }
            dst[i] = pack_chunk<DT>(x);
        }
    }
    // the ragged ends, an element a thread
    const int tail = V - head - nvec * VEC;
    if (part == 0 && tid < head + tail) {
        const int j = tid < head ? tid : V - tail + (tid - head);
        float d = 0.0f;
        if (!zero) {
            d = G.at(load_rw<DT>(in, j));
            if (j == tok) d += hit;
        }
        Elem<DT>::store(out, j, d);
    }
}

}  // namespace lp
}  // namespace fg
