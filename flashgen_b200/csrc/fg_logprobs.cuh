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


// Temperatures: positive, finite and not subnormal (1 / T stays finite).
__device__ __forceinline__ bool temperature_ok(float T) { return T >= 1.17549435e-38f && T < INFINITY; }

// ---------------------------------------------------------------------------
// Forward: one pass over the logits.
//
// A cluster of G CTAs takes a row, each a slice of its 16-byte chunks. A thread
// streams its chunks four at a time and keeps, in 32 bits: its largest logit; S and
// Q (below) against a reference that follows its largest logit (lazily: a sum may
// grow to 2^64 above it, so it is rescaled about once); the count of the logits ahead
// of the token's. S and Q are sums of 2^y and 2^y y with y = x c - r: one FMA a
// logit, the same r in every term, so r's rounding cancels in log2 S + r.
//
// Alternatives without a second pass over the row: the top-th largest of 64 group
// maxima bounds the top-th largest logit from below, so every alternative lies with a
// thread whose own maximum reaches the bound; there are few such threads, and only
// their chunks are read again (from L2). What reaches the bound is gathered, and a
// candidate's place is the number of candidates ahead of it.
//
// Bound: HBM, one read of the logits. The work per 16-bit logit is 5.5 instructions
// and one ex2, about two thirds of what the SMs can issue in that time.
// ---------------------------------------------------------------------------
constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int UNROLL = 4;            // chunks in flight a thread
constexpr int GROUPS = 64;           // of THREADS / 64 = 8 lanes
constexpr int MAX_G = 16;
constexpr int CAND = 1024;           // candidates held at once
constexpr float R_STEP = 64.0f;      // how far above its reference a term may be (in log2)

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
// well above it and x c stays finite (one_pass_ok), other rows are summed again.
template <int DT> struct Chunk;
template <> struct Chunk<FG_DTYPE_F32> {
    static constexpr int WORDS = 4;
    __device__ __forceinline__ static bool one_pass_ok(float m, float c) {
        return m > -1e29f && m < 1e29f && c < 1e8f && c > 1e-20f;
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
    struct Count {
        int n = 0;
        __device__ __forceinline__ void add(const uint32_t* w, float xt, bool or_equal) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = __uint_as_float(w[i]);
                n += (or_equal ? x >= xt : x > xt) ? 1 : 0;
            }
        }
        __device__ __forceinline__ int take() { return n; }
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
    struct Count {
        T2 n = pack(0u);   // up to 16 in each half
        __device__ __forceinline__ void add(const uint32_t* w, float xt, bool or_equal) {
            T2 t;
            if constexpr (DT == FG_DTYPE_F16) t = __float2half2_rn(xt);
            else t = __float2bfloat162_rn(xt);
            if (or_equal) {
#pragma unroll
                for (int i = 0; i < 4; ++i) n = __hadd2(n, __hge2(pack(w[i]), t));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) n = __hadd2(n, __hgt2(pack(w[i]), t));
            }
        }
        __device__ __forceinline__ int take() {
            const float2 f = unpack(*reinterpret_cast<uint32_t*>(&n));
            return int(f.x + f.y);
        }
    };
};
template <> struct Chunk<FG_DTYPE_F16> : Chunk16<__half2, FG_DTYPE_F16> {
    __device__ __forceinline__ static bool one_pass_ok(float m, float c) { return m > -60000.0f && c > 0.03f && c < 1e8f; }
};
template <> struct Chunk<FG_DTYPE_BF16> : Chunk16<__nv_bfloat162, FG_DTYPE_BF16> {
    __device__ __forceinline__ static bool one_pass_ok(float m, float c) {
        return Chunk<FG_DTYPE_F32>::one_pass_ok(m, c);
    }
};

// Running sums of one thread.
struct Sums {
    float s = 0.0f, q = 0.0f;
    float r = 0.0f;                  // the reference, in log2
    float limit = -9.9e29f;          // logits above it move the reference
    bool set = false;
    __device__ __forceinline__ void follow(float m, float c) {   // m: the largest of the next logits
        if (m > limit) {
            const float to = m * c;
            const float f = set ? exp2_fast(r - to) : 0.0f;
            q = set ? f * fmaf(r - to, s, q) : 0.0f;
            s *= f;
            r = to;
            limit = m + R_STEP / c;
            set = true;
        }
    }
    __device__ __forceinline__ void add(float x, float c) {   // x floored
        const float y = fmaf(x, c, -r);
        const float e = exp2_fast(y);
        s += e;
        q = fmaf(e, y, q);
    }
};

// What a warp, a CTA and a row add up to: S and Q against the largest logit.
struct Stats {
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

// The top-th largest of 64 values, two a lane (a warp-wide bitonic sort of both
// halves, then the larger ones of both).
__device__ __forceinline__ float kth_of_64(float a, float b, int k, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const bool keep_max = ((lane & size) == 0) == ((lane & d) == 0);
            const float oa = __shfl_xor_sync(0xffffffffu, a, d), ob = __shfl_xor_sync(0xffffffffu, b, d);
            a = keep_max ? fmaxf(a, oa) : fminf(a, oa);
            b = keep_max ? fmaxf(b, ob) : fminf(b, ob);
        }
    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, b, 31));   // descending a against ascending b
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, a, d);
        a = (lane & d) == 0 ? fmaxf(a, o) : fminf(a, o);
    }
    return __shfl_sync(0xffffffffu, a, k - 1);
}

struct Shared {
    Stats warp[WARPS];
    Stats cta[MAX_G];                       // every CTA of the cluster writes its entry
    float groups[GROUPS];
    int count;                              // candidates
    uint64_t cand[CAND];
    uint64_t lists[MAX_G][FG_LOGPROB_MAX_TOP];   // the CTAs' best (in the first CTA)
};

__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// One row's geometry: scalars before the first and after the last whole chunk, and
// this CTA's chunks.
template <int DT>
struct Row {
    static constexpr int VEC = Elem<DT>::VEC, SIZE = Elem<DT>::SIZE;
    const char* p;
    int V, head, nvec, tail, c0, c1;
    __device__ __forceinline__ Row(const Params& P, int64_t r, int part, int parts) {
        p = reinterpret_cast<const char*>(P.logits) + r * P.row_stride * SIZE;
        V = P.vocab;
        head = min(V, int((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / SIZE);
        nvec = (V - head) / VEC;
        tail = V - head - nvec * VEC;
        c0 = int(int64_t(nvec) * part / parts);
        c1 = int(int64_t(nvec) * (part + 1) / parts);
    }
    __device__ __forceinline__ const uint4* chunks() const {
        return reinterpret_cast<const uint4*>(p + int64_t(head) * SIZE);
    }
    __device__ __forceinline__ int id(int chunk) const { return head + chunk * VEC; }
    __device__ __forceinline__ int scalar_id(int i) const { return i < head ? i : V - tail + (i - head); }
};

template <int DT, bool TOP>
__global__ void __launch_bounds__(THREADS, 2) logprob_kernel(const Params P, const int G) {
    __shared__ Shared sh;
    constexpr int VEC = Elem<DT>::VEC;
    using C = Chunk<DT>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r = blockIdx.x / G;
    const int part = blockIdx.x % G;
    if (G > 1) cluster_arrive();   // the others' shared memory stands once all have arrived
    const Row<DT> row(P, r, part, G);
    const int V = row.V;
    const int64_t tok = P.tokens ? P.tokens[r] : -1;
    const float T = P.temperature ? P.temperature[r] : 1.0f;
    const bool given = tok >= 0 && tok < V;
    const float c = LOG2E / T;
    const float xt = given ? Elem<DT>::load(row.p, tok) : INFINITY;
    // chunks before the token's count equal logits as ahead of it, the others do not
    const int tchunk = !given || tok < row.head ? -1 : int((tok - row.head) / VEC);
    if (tid == 0) sh.count = 0;

    // ---- the pass ----
    const uint4* chunks = row.chunks();
    Sums acc;
    float vmax = -INFINITY;
    int n = 0;
    for (int c0 = row.c0 + tid; c0 < row.c1; c0 += UNROLL * THREADS) {
        uint32_t w[UNROLL * 4];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int ci = c0 + u * THREADS;
            const uint32_t none = DT == FG_DTYPE_F32 ? 0xff800000u : DT == FG_DTYPE_F16 ? 0xfc00fc00u : 0xff80ff80u;
            uint4 v = make_uint4(none, none, none, none);   // -inf
            if (ci < row.c1) v = __ldg(chunks + ci);
            w[4 * u] = v.x; w[4 * u + 1] = v.y; w[4 * u + 2] = v.z; w[4 * u + 3] = v.w;
        }
        const float m = C::max_of(w, UNROLL * 4);
        vmax = fmax_nan(vmax, m);
        acc.follow(m, c);
        float2 s2 = make_float2(0.0f, 0.0f), q2 = make_float2(0.0f, 0.0f);
        const float2 cc = make_float2(c, c), rr = make_float2(-acc.r, -acc.r);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < C::PAIRS; ++i) {
                const float2 y = fma2(C::floored(w + 4 * u, i), cc, rr);
                const float2 e = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                s2 = add2(s2, e);
                q2 = fma2(e, y, q2);
            }
        acc.s += s2.x + s2.y;
        acc.q += q2.x + q2.y;
        typename C::Count cnt;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int ci = c0 + u * THREADS;
            if (ci < row.c1) cnt.add(w + 4 * u, xt, ci < tchunk);
        }
        n += cnt.take();
    }
    // the ragged ends, a logit a thread, and the equal logits in the token's own chunk
    const int scalars = part == 0 ? row.head + row.tail : 0;
    if (tid < scalars) {
        const int j = row.scalar_id(tid);
        const float x = Elem<DT>::load(row.p, j);
        vmax = fmax_nan(vmax, x);
        acc.follow(x, c);
        acc.add(fmaxf(x, DT == FG_DTYPE_F16 ? -65504.0f : -1e30f), c);
        if (given) n += (x > xt || (x == xt && j < tok)) ? 1 : 0;
    }
    if (tchunk >= row.c0 && tchunk < row.c1 && tid < VEC) {
        const int j = row.id(tchunk) + tid;
        if (j < tok && Elem<DT>::load(row.p, j) == xt) n += 1;
    }

    // ---- the warp, then the CTA ----
    float wm = vmax;
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) wm = fmax_nan(wm, __shfl_xor_sync(0xffffffffu, wm, d));
    if (TOP && (lane & 7) == 0) sh.groups[tid >> 3] = wm;
#pragma unroll
    for (int d = 8; d < 32; d <<= 1) wm = fmax_nan(wm, __shfl_xor_sync(0xffffffffu, wm, d));
    {
        Stats st{wm, 0.0f, 0.0f, n};
        if (acc.set) {
            const float d = fmaxf(fmaf(-wm, c, acc.r), Y_MIN);   // the reference against the warp's maximum
            const float f = exp2_fast(d);
            st.s = f * acc.s;
            st.q = f * fmaf(d, acc.s, acc.q);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            st.s += __shfl_xor_sync(0xffffffffu, st.s, d);
            st.q += __shfl_xor_sync(0xffffffffu, st.q, d);
            st.n += __shfl_xor_sync(0xffffffffu, st.n, d);
        }
        if (lane == 0) sh.warp[warp] = st;
    }
    __syncthreads();
    auto fold = [&](const Stats* from, int count, bool recount) {   // every warp the same, a lane an entry
        Stats st{-INFINITY, 0.0f, 0.0f, 0};
        if (lane < count) st = from[lane];
        float m = st.m;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
        if (!recount) st = merge(st, m, c);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            st.s += __shfl_xor_sync(0xffffffffu, st.s, d);
            st.q += __shfl_xor_sync(0xffffffffu, st.q, d);
            st.n += __shfl_xor_sync(0xffffffffu, st.n, d);
        }
        st.m = m;
        return st;
    };
    Stats all = fold(sh.warp, WARPS, false);

    // ---- alternatives: the candidates of this CTA ----
    int ncand = 0;
    if (TOP) {
        const float bound = kth_of_64(sh.groups[lane], sh.groups[lane + 32], P.top, lane);
        const uint32_t winners = __ballot_sync(0xffffffffu, vmax >= bound);
        auto load_chunk = [&](int ci, float (&x)[VEC]) { Elem<DT>::unpack(__ldg(chunks + ci), x); };
        // gather: winner by winner, a chunk a lane
        auto put = [&](uint64_t code) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < CAND) sh.cand[at] = code;
        };
        auto each_winner = [&](auto visit) {
            for (uint32_t m = winners; m; m &= m - 1) {
                const int first = row.c0 + (tid & ~31) + __ffs(m) - 1;
                for (int c0 = first; c0 < row.c1; c0 += 32 * THREADS) visit(c0 + lane * THREADS);
            }
        };
        if (bound > -INFINITY) {
            each_winner([&](int ci) {
                if (ci < row.c1) {
                    float x[VEC];
                    load_chunk(ci, x);
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (x[e] >= bound) put(order_code(x[e], row.id(ci) + e));
                }
            });
            if (tid < scalars) {
                const float x = Elem<DT>::load(row.p, row.scalar_id(tid));
                if (x >= bound) put(order_code(x, row.scalar_id(tid)));
            }
        }
        __syncthreads();
        ncand = sh.count;
        if (ncand > CAND || !(bound > -INFINITY)) {
            // too many at or above the bound (ties, long runs in order), or a bound of -inf:
            // each warp keeps its best 32 in its lanes and inserts what beats the last
            __syncthreads();
            if (tid == 0) sh.count = 0;
            __syncthreads();
            uint64_t best = 0;
            auto insert = [&](uint64_t code) {
                uint32_t better;
                while ((better = __ballot_sync(0xffffffffu, code > __shfl_sync(0xffffffffu, best, 31)))) {
                    const uint64_t v = shfl_u64(code, __ffs(better) - 1);
                    const uint64_t up = shfl_up_u64(best, 1);
                    const int place = __popc(__ballot_sync(0xffffffffu, best > v));
                    best = lane < place ? best : lane == place ? v : up;
                    if (lane == __ffs(better) - 1) code = 0;
                }
            };
            each_winner([&](int ci) {
                float x[VEC];
                const bool in = ci < row.c1;
                if (in) load_chunk(ci, x);
#pragma unroll
                for (int e = 0; e < VEC; ++e) insert(in ? order_code(x[e], row.id(ci) + e) : 0);
            });
            if (scalars > 0 && warp == 0)
                insert(lane < scalars ? order_code(Elem<DT>::load(row.p, row.scalar_id(lane)), row.scalar_id(lane)) : 0);
            if (best != 0) put(best);
            __syncthreads();
            ncand = sh.count;
        }
    }
    // a candidate's place is the number of candidates ahead of it
    auto place_of = [&](uint64_t code, const uint64_t* from, int count) {
        int ahead = 0;
        for (int i = 0; i < count; ++i) ahead += from[i] > code;
        return ahead;
    };

    // ---- the row ----
    if (G > 1) {
        cluster_wait();
        if (warp == 0 && lane < G) {
            const uint32_t to = cluster_addr(&sh.cta[part], lane);
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};"
                         :: "r"(to), "f"(all.m), "f"(all.s), "f"(all.q), "f"(__int_as_float(all.n)) : "memory");
        }
        if (TOP) {
            const uint32_t lists = cluster_addr(&sh.lists[part][0], 0);
            for (int i = tid; i < ncand; i += THREADS) {
                const int place = place_of(sh.cand[i], sh.cand, ncand);
                if (place < P.top)
                    asm volatile("st.shared::cluster.u64 [%0], %1;" :: "r"(lists + 8 * place), "l"(sh.cand[i]) : "memory");
            }
            if (tid < P.top && tid >= ncand)
                asm volatile("st.shared::cluster.u64 [%0], %1;" :: "r"(lists + 8 * tid), "l"(uint64_t(0)) : "memory");
        }
        cluster_arrive();
        cluster_wait();
        all = fold(sh.cta, G, false);
    }
    const float m = all.m;
    int status = 0;
    if (isnan(m)) status |= FG_ROW_NAN;
    if (m == INFINITY) status |= FG_ROW_POS_INF;
    if (m == -INFINITY) status |= FG_ROW_ALL_MASKED;
    if (!temperature_ok(T) || tok >= V) status |= FG_ROW_BAD_PARAM;
    const bool bad = (status & ~FG_ROW_ALL_MASKED) != 0;
    const bool empty = m == -INFINITY;

    if (!bad && !empty && !C::one_pass_ok(m, c)) {
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
        if (lane == 0) sh.warp[warp] = Stats{m, s, q, 0};
        __syncthreads();
        Stats again = fold(sh.warp, WARPS, true);
        if (G > 1) {
            cluster_arrive();   // everyone has read the first round's entries
            cluster_wait();
            if (warp == 0 && lane < G) {
                const uint32_t to = cluster_addr(&sh.cta[part], lane);
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};"
                             :: "r"(to), "f"(m), "f"(again.s), "f"(again.q), "f"(0.0f) : "memory");
            }
            cluster_arrive();
            cluster_wait();
            again = fold(sh.cta, G, true);
        }
        all.s = again.s;
        all.q = again.q;
    }
    if (part != 0) return;
    const float l2 = log2f(all.s);
    const float nan = __int_as_float(0x7fc00000);
    if (tid == 0) {
        const float lpt = tok < 0 ? 0.0f : empty ? -INFINITY : (xt - m) / T - LN2 * l2;
        if (P.out_logprobs) P.out_logprobs[r] = bad ? nan : lpt;
        if (P.out_entropy) P.out_entropy[r] = bad ? nan : empty ? 0.0f : LN2 * (l2 - all.q / all.s);
        if (P.out_max) P.out_max[r] = m;
        if (P.out_logsum) P.out_logsum[r] = bad ? nan : empty ? -INFINITY : LN2 * l2;
        if (P.out_rank) P.out_rank[r] = (bad || tok < 0) ? -1 : all.n;
        if (P.out_status) P.out_status[r] = status;
    }
    if (TOP) {
        auto write = [&](int i, bool none, uint64_t code) {
            const float x = funkey(uint32_t(code >> 32));
            if (P.out_top_ids) P.out_top_ids[r * P.top + i] = (none || bad) ? -1 : int64_t(uint32_t(~uint32_t(code)));
            if (P.out_top_logprobs)
                P.out_top_logprobs[r * P.top + i] =
                    bad ? nan : (none || x == -INFINITY) ? -INFINITY : (x - m) / T - LN2 * l2;
        };
        const uint64_t* from = G > 1 ? &sh.lists[0][0] : sh.cand;
        const int count = G > 1 ? G * FG_LOGPROB_MAX_TOP : ncand;
        int valid = ncand;   // what there is to place
        if (G > 1) valid = V;
        for (int i = tid; i < count; i += THREADS) {
            if (G > 1 && (i & (FG_LOGPROB_MAX_TOP - 1)) >= P.top) continue;
            const uint64_t code = from[i];
            if (code == 0) continue;
            int place = 0;
            if (G > 1) {
                for (int g = 0; g < G; ++g)
                    for (int j = 0; j < P.top; ++j) place += sh.lists[g][j] > code;
            } else {
                place = place_of(code, from, count);
            }
            if (place < P.top) write(place, false, code);
        }
        // past the vocabulary's end, and rows that have no alternatives to name
        for (int i = tid; i < P.top; i += THREADS)
            if (i >= min(valid, V) || bad) write(i, true, 0);
    }
}

// ---------------------------------------------------------------------------
// Gradient: dx_j = p_j (a + b y_j) + 1[j == t] g / T with y_j = (x_j - m) c - L2,
// p_j = 2^y_j, a = -(g + h H) / T and b = -h ln2 / T.
//
// Bound: HBM, the logits read and the gradient written once. Work is cut along the
// gradient's 16-byte chunks; where the logits' rows are offset against the
// gradient's, a thread takes the two chunks around its own and shifts them together.
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
