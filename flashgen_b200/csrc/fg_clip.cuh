// fg_clip.cuh — the global norm of a list of gradients and the gradients scaled to
// at most a given norm (fg_clip_grad_norm):
//   norm = scale * sqrt(sum_i sum_j g_ij^2),   out_ij = g_ij * c,
//   c    = scale * min(1, max_norm / (norm + 1e-6))
//
// Two launches over all tensors of one pair of types (more for lists of mixed types, or
// of over MAX_TENSORS): norm_kernel leaves one partial sum a CTA, scale_kernel
// adds them up in every CTA (a few hundred numbers, in the same order everywhere) and
// scales. Tensors are cut into chunks of 16 KB, numbered through the list; a CTA takes
// every gridDim-th chunk, so neither many small tensors nor one large one leave SMs
// idle, and the sums do not depend on timing. scale_kernel goes through the chunks
// backwards: what norm_kernel read last is still in L2.
#pragma once

#include "fg_common.cuh"

namespace fg {
namespace clip {

constexpr int THREADS = 256, UNROLL = 4;
constexpr int CHUNK_BYTES = THREADS * UNROLL * 16;   // of a tensor's gradients
constexpr int MAX_TENSORS = 96;                      // of a launch: their list is a kernel parameter (4 KB at most)
constexpr int MAX_GRID = 1184;                       // CTAs, and partial sums, of a launch

struct Item {
    const void* in;
    void* out;            // null: norm only
    int64_t count;
    uint32_t first;       // number of its first chunk
    uint16_t wide_in, wide_out;   // 16-byte loads; stores of a whole vector
};
struct List {
    Item items[MAX_TENSORS];
    int32_t count;
    uint32_t chunks;
};

__device__ __forceinline__ void wait_prerequisites() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The sum of v over the block, in every thread, added in one fixed order.
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[THREADS / 32];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) sum += part[i];
    __syncthreads();
    return sum;
}

// The squares of one 16-byte vector. In fp32 while their sum is far from both ends of
// its range (then squares that underflow are below 2^-46 of it, and eight roundings are
// far below the one of the result); otherwise, but for vectors of zeros, in 64 bits.
template <int DT>
__device__ __forceinline__ double squares(const uint4& q) {
    float x[Elem<DT>::VEC];
    Elem<DT>::unpack(q, x);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < Elem<DT>::VEC; ++i) s = fmaf(x[i], x[i], s);
    if (s >= 0x1p-80f && s <= 0x1p100f) return double(s);
    double d = 0.0;
    if (((q.x | q.y | q.z | q.w) & (DT == FG_DTYPE_F32 ? 0x7fffffffu : 0x7fff7fffu)) != 0u) {
#pragma unroll
        for (int i = 0; i < Elem<DT>::VEC; ++i) d = fma(double(x[i]), double(x[i]), d);
    }
    return d;
}

// The squares of elements [lo, hi) of a tensor (one chunk), this thread's share.
template <int DT>
__device__ __forceinline__ double chunk_squares(const Item& it, int64_t lo, int64_t hi) {
    constexpr int VEC = Elem<DT>::VEC;
    double sum = 0.0;
    int64_t done = lo;
    if (it.wide_in) {
        const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(it.in) + lo * Elem<DT>::SIZE);
        const int vecs = int((hi - lo) / VEC);
        uint4 q[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (u * THREADS + int(threadIdx.x) < vecs) q[u] = __ldg(p + u * THREADS + threadIdx.x);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (u * THREADS + int(threadIdx.x) < vecs) sum += squares<DT>(q[u]);
        done = lo + int64_t(vecs) * VEC;
    }
#pragma unroll 4
    for (int64_t i = done + threadIdx.x; i < hi; i += THREADS) {
        const double x = double(Elem<DT>::load(it.in, i));
        sum = fma(x, x, sum);
    }
    return sum;
}

// The tensor that holds chunk c, searched from tensor t on.
__device__ __forceinline__ int item_of(const List& L, uint32_t c, int t) {
    while (t + 1 < L.count && L.items[t + 1].first <= c) ++t;
    return t;
}
// Bound: HBM reads: 805 million bf16 gradients 223 us, 7.2 TB/s.
template <int DT>
__global__ void __launch_bounds__(THREADS, 6) norm_kernel(const __grid_constant__ List L, double* partial) {
    wait_prerequisites();
    launch_dependents();
    double sum = 0.0;
    int t = 0;
    for (uint32_t c = blockIdx.x; c < L.chunks; c += gridDim.x) {
        t = item_of(L, c, t);
        const Item& it = L.items[t];
        constexpr int64_t STEP = CHUNK_BYTES / Elem<DT>::SIZE;
        const int64_t lo = int64_t(c - it.first) * STEP, hi = lo + STEP < it.count ? lo + STEP : it.count;
        sum += chunk_squares<DT>(it, lo, hi);
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The partial sums of several norm launches as one.
__global__ void __launch_bounds__(THREADS) total_kernel(const double* partial, int64_t count, double* total) {
    wait_prerequisites();
    launch_dependents();
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += THREADS) sum += partial[i];
    sum = block_sum(sum);
    if (threadIdx.x == 0) *total = sum;
}

// What a thread loads and stores at once: 16 bytes of the wider type, so that both are
// neighbouring bytes across a warp (16-byte loads of 16-bit gradients with two stores of 32-bit
// results each wrote half sectors: 805 million bf16 gradients 990 us, 4.9 TB/s).
template <int DT, int ODT>
struct Vector {
    static constexpr int N = 16 / (Elem<DT>::SIZE > Elem<ODT>::SIZE ? Elem<DT>::SIZE : Elem<ODT>::SIZE);
};
template <int BYTES> struct Words;
template <> struct Words<16> { using T = uint4; };
template <> struct Words<8> { using T = uint2; };

template <int DT, int N, class W>
__device__ __forceinline__ void unpack(const W& q, float (&x)[N]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&q);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (DT == FG_DTYPE_F32) x[i] = __uint_as_float(w[i]);
        else if constexpr (DT == FG_DTYPE_BF16) x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else x[i] = __half2float(__ushort_as_half(uint16_t(i & 1 ? w[i / 2] >> 16 : w[i / 2])));
    }
}
template <int ODT, int N, class W>
__device__ __forceinline__ W pack(const float (&x)[N]) {
    W q;
    uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (ODT == FG_DTYPE_F32) {
            w[i] = __float_as_uint(x[i]);
        } else if (i % 2 == 0) {
            if constexpr (ODT == FG_DTYPE_F16) {
                const __half2 h = __floats2half2_rn(x[i], x[i + 1]);
                w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[i], x[i + 1]);
                w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
    }
    return q;
}

template <int DT, int ODT>
__device__ __forceinline__ void scale_chunk(const Item& it, int64_t lo, int64_t hi, float c) {
    constexpr int N = Vector<DT, ODT>::N;
    using In = typename Words<N * Elem<DT>::SIZE>::T;
    using Out = typename Words<N * Elem<ODT>::SIZE>::T;
    constexpr int LOADS = CHUNK_BYTES / int(sizeof(In)) / THREADS;
    int64_t done = lo;
    if (it.wide_in && it.wide_out) {
        const In* p = reinterpret_cast<const In*>(reinterpret_cast<const char*>(it.in) + lo * Elem<DT>::SIZE);
        Out* o = reinterpret_cast<Out*>(reinterpret_cast<char*>(it.out) + lo * Elem<ODT>::SIZE);
        const int vecs = int((hi - lo) / N);
        In q[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u)
            if (u * THREADS + int(threadIdx.x) < vecs) q[u] = __ldcs(p + u * THREADS + threadIdx.x);
#pragma unroll
        for (int u = 0; u < LOADS; ++u)
            if (u * THREADS + int(threadIdx.x) < vecs) {
                float x[N];
                unpack<DT>(q[u], x);
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] *= c;
                __stcs(o + u * THREADS + threadIdx.x, pack<ODT, N, Out>(x));
            }
        done = lo + int64_t(vecs) * N;
    }
    // (not through the read-only cache: the result may replace what is read)
#pragma unroll 4
    for (int64_t i = done + threadIdx.x; i < hi; i += THREADS) {
        float x;
        if constexpr (DT == FG_DTYPE_F32) x = reinterpret_cast<const float*>(it.in)[i];
        else if constexpr (DT == FG_DTYPE_F16) x = __half2float(reinterpret_cast<const __half*>(it.in)[i]);
        else x = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(it.in)[i]);
        Elem<ODT>::store(it.out, i, x * c);
    }
}

// Bound: HBM, the second read as far as L2 does not hold it and the write: 805 million bf16
// gradients into fp32 830 us, 5.8 TB/s.
template <int DT, int ODT>
__global__ void __launch_bounds__(THREADS, 6) scale_kernel(const __grid_constant__ List L, const double* partial,
                                                        int64_t count, float max_norm, float scale, float* out_norm) {
    wait_prerequisites();
    launch_dependents();
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += THREADS) sum += partial[i];
    sum = block_sum(sum);
    const float norm = float(sqrt(sum) * double(scale));
    if (blockIdx.x == 0 && threadIdx.x == 0 && out_norm) *out_norm = norm;
    // (without a limit nothing is clipped, whatever the norm: infinity over infinity is no ratio)
    const float ratio = max_norm < INFINITY || norm != norm ? __fdiv_rn(max_norm, norm + 1e-6f) : 1.0f;
    const float c = scale * (ratio < 1.0f || ratio != ratio ? ratio : 1.0f);
    int t = 0;
    uint32_t top = L.chunks;   // chunks from here on are done
    while (t + 1 < L.count) ++t;
    for (uint32_t k = blockIdx.x; k < top; k += gridDim.x) {
        const uint32_t ch = top - 1 - k;
        while (t > 0 && L.items[t].first > ch) --t;
        const Item& it = L.items[t];
        // gradients that stay as they are
        if (c == 1.0f && it.out == it.in) continue;
        constexpr int64_t STEP = CHUNK_BYTES / Elem<DT>::SIZE;
        const int64_t lo = int64_t(ch - it.first) * STEP, hi = lo + STEP < it.count ? lo + STEP : it.count;
        scale_chunk<DT, ODT>(it, lo, hi, c);
    }
}

}  // namespace clip
}  // namespace fg
