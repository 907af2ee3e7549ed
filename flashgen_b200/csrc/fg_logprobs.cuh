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

constexpr int THREADS = 256;

// Temperatures: positive, finite and not subnormal (1 / T stays finite).
__device__ __forceinline__ bool temperature_ok(float T) { return T >= 1.17549435e-38f && T < INFINITY; }

// Order of the alternatives: larger logit first, then smaller id. A larger code
// comes first; 0 is below every element's code.
__device__ __forceinline__ uint64_t order_code(float x, int32_t j) {
    return (uint64_t(fkey(x)) << 32) | uint32_t(~j);
}
__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <class T, class F>
__device__ __forceinline__ T block_reduce(T v, F f, T* buf) {
    const int tid = threadIdx.x;
    buf[tid] = v;
    __syncthreads();
    for (int d = THREADS / 2; d > 0; d >>= 1) {
        if (tid < d) buf[tid] = f(buf[tid], buf[tid + d]);
        __syncthreads();
    }
    v = buf[0];
    __syncthreads();
    return v;
}

// One CTA per row, three passes over it and one more per alternative.
template <int DT>
__global__ void __launch_bounds__(THREADS) logprob_kernel(const Params P) {
    __shared__ uint64_t buf64[THREADS];
    float* bufF = reinterpret_cast<float*>(buf64);
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const int V = P.vocab;
    const char* row = reinterpret_cast<const char*>(P.logits) + r * P.row_stride * Elem<DT>::SIZE;
    const int64_t tok = P.tokens ? P.tokens[r] : -1;
    const float T = P.temperature ? P.temperature[r] : 1.0f;

    float m = -INFINITY;
    for (int j = tid; j < V; j += THREADS) m = fmax_nan(m, Elem<DT>::load(row, j));
    m = block_reduce(m, [](float a, float b) { return fmax_nan(a, b); }, bufF);
    int status = 0;
    if (isnan(m)) status |= FG_ROW_NAN;
    if (m == INFINITY) status |= FG_ROW_POS_INF;
    if (m == -INFINITY) status |= FG_ROW_ALL_MASKED;
    if (!temperature_ok(T) || tok >= V) status |= FG_ROW_BAD_PARAM;
    const bool bad = (status & ~FG_ROW_ALL_MASKED) != 0;
    const bool empty = m == -INFINITY;
    const float c = LOG2E / T;

    float s = 0.0f, q = 0.0f, cnt = 0.0f;
    const float xt = (tok >= 0 && tok < V) ? Elem<DT>::load(row, tok) : 0.0f;
    if (!bad) {
        for (int j = tid; j < V; j += THREADS) {
            const float x = Elem<DT>::load(row, j);
            if (!empty) {
                const float y = fmaxf((x - m) * c, Y_MIN);
                const float e = exp2f(y);
                s += e;
                q += e * y;
            }
            cnt += (x > xt || (x == xt && j < tok)) ? 1.0f : 0.0f;
        }
    }
    auto add = [](float a, float b) { return a + b; };
    s = block_reduce(s, add, bufF);
    q = block_reduce(q, add, bufF);
    cnt = block_reduce(cnt, add, bufF);
    const float l2 = log2f(s);
    const float nan = __int_as_float(0x7fc00000);
    if (tid == 0) {
        float lpt = tok < 0 ? 0.0f : empty ? -INFINITY : (xt - m) / T - LN2 * l2;
        if (P.out_logprobs) P.out_logprobs[r] = bad ? nan : lpt;
        if (P.out_entropy) P.out_entropy[r] = bad ? nan : empty ? 0.0f : LN2 * (l2 - q / s);
        if (P.out_max) P.out_max[r] = m;
        if (P.out_logsum) P.out_logsum[r] = bad ? nan : LN2 * l2;
        if (P.out_rank) P.out_rank[r] = (bad || tok < 0) ? -1 : int32_t(cnt);
        if (P.out_status) P.out_status[r] = status;
    }
    uint64_t last = ~0ull;
    for (int i = 0; i < P.top; ++i) {
        uint64_t best = 0;
        if (!bad)
            for (int j = tid; j < V; j += THREADS) {
                const uint64_t o = order_code(Elem<DT>::load(row, j), j);
                if (o < last) best = max_u64(best, o);
            }
        best = block_reduce(best, [](uint64_t a, uint64_t b) { return max_u64(a, b); }, buf64);
        last = best;
        if (tid == 0) {
            const bool none = bad || best == 0;
            const float x = funkey(uint32_t(best >> 32));
            if (P.out_top_ids) P.out_top_ids[r * P.top + i] = none ? -1 : int64_t(uint32_t(~uint32_t(best)));
            if (P.out_top_logprobs)
                P.out_top_logprobs[r * P.top + i] =
                    bad ? nan : (none || x == -INFINITY) ? -INFINITY : (x - m) / T - LN2 * l2;
        }
    }
}

// A coherent load: the gradient may overwrite the logits.
template <int DT>
__device__ __forceinline__ float load_rw(const char* row, int64_t j) {
    if constexpr (DT == FG_DTYPE_F32) return reinterpret_cast<const float*>(row)[j];
    else if constexpr (DT == FG_DTYPE_F16) return __half2float(reinterpret_cast<const __half*>(row)[j]);
    else return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[j]);
}

// dx_j = p_j (a + b y_j) + 1[j == t] g / T with y_j = (x_j - m) c - L2,
// p_j = 2^y_j, a = -(g + h H) / T and b = -h ln2 / T.
template <int DT>
__global__ void __launch_bounds__(THREADS) logprob_grad_kernel(const GradParams P) {
    const int64_t r = blockIdx.y;
    const int V = P.vocab;
    const char* row = reinterpret_cast<const char*>(P.logits) + r * P.row_stride * Elem<DT>::SIZE;
    char* out = reinterpret_cast<char*>(P.out_grad) + r * P.grad_stride * Elem<DT>::SIZE;
    const int64_t tok = P.tokens ? P.tokens[r] : -1;
    const float T = P.temperature ? P.temperature[r] : 1.0f;
    const float g = (P.grad_logprobs && tok >= 0) ? P.grad_logprobs[r] : 0.0f;
    const float h = P.grad_entropy ? P.grad_entropy[r] : 0.0f;
    const float m = P.max[r];
    const float l2 = P.logsum[r] * LOG2E;
    const float c = LOG2E / T;
    float a = -(g + (h != 0.0f ? h * P.entropy[r] : 0.0f)) / T;
    const float b = -h * LN2 / T;
    const bool bad = !temperature_ok(T) || tok >= V || isnan(l2) || isnan(m);
    const bool zero = (g == 0.0f && h == 0.0f) || (m == -INFINITY && !bad);
    if (bad) a = __int_as_float(0x7fc00000);
    for (int j = blockIdx.x * THREADS + threadIdx.x; j < V; j += gridDim.x * THREADS) {
        float d = 0.0f;
        if (!zero) {
            const float y = fmaxf((load_rw<DT>(row, j) - m) * c - l2, Y_MIN);
            d = exp2f(y) * (a + b * y);
            if (j == tok) d += g / T;
        }
        Elem<DT>::store(out, j, d);
    }
}

}  // namespace lp
}  // namespace fg
