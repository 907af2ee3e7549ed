// fg_linear.cuh — the fused linear block out = act(x W^T + bias) + residual and its
// gradients (fg_linear, fg_linear_grad).
//
// One product kernel serves all three products. The contiguous dimension of the result
// lies on the accumulator's 128 lanes and the other one on its columns, so that a few
// tokens take a narrow tile and waste no tensor-core rows:
//   out [m, n]:  lanes n, columns m, sum over k;  A = W [n, k],  B = x [m, k]
//   dx  [m, k]:  lanes k, columns m, sum over n;  A = W [n, k],  B = dz [m, n]
//   dW  [n, k]:  lanes k, columns n, sum over m;  A = x [m, k],  B = dz [m, n]
// A and B are read as they lie in memory: the operand descriptors say which dimension of
// a tile is the contiguous one (K-major, or MN-major where the sum runs across rows).
#pragma once

#include "fg_linear.h"
#include "fg_tcgen05.cuh"

namespace fg {
namespace lin {

// ---- activations -----------------------------------------------------------
// In fp32, for results of 16 bits: e^x by ex2 (2 ulp) of a product. Written so that
// small values keep their relative precision: the complementary error function in place
// of 1 + erf, the logistic function in place of 1 + tanh.
__device__ __forceinline__ float exp_fast(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}
// s = 1 / (1 + e^-z) and 1 - s, neither by cancellation
__device__ __forceinline__ void logistic(float z, float& s, float& rest) {
    const float t = exp_fast(-fabsf(z)), q = __fdividef(1.0f, 1.0f + t);
    s = z >= 0.0f ? q : t * q;
    rest = z >= 0.0f ? t * q : q;
    if (z != z) s = rest = z;
}
// The first alone (of powers that do not leave the range).
__device__ __forceinline__ float logistic(float z) {
    const float t = exp_fast(-fabsf(z));
    return __fdividef(z < 0.0f ? t : 1.0f, 1.0f + t);
}
constexpr float kGeluC = 0.7978845608028654f, kGeluD = 0.044715f;   // sqrt(2 / pi); the cubic term

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == FG_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if constexpr (ACT == FG_ACT_SILU) return z * logistic(z);
    if constexpr (ACT == FG_ACT_GELU) return 0.5f * z * erfcf(-0.7071067811865476f * z);
    if constexpr (ACT == FG_ACT_GELU_TANH)
        return z * logistic(2.0f * kGeluC * fmaf(kGeluD * z * z, z, z));
    return z;
}
template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == FG_ACT_RELU) return z > 0.0f ? 1.0f : z != z ? z : 0.0f;
    if constexpr (ACT == FG_ACT_SILU) {
        float s, r;
        logistic(z, s, r);
        return fmaf(r == 0.0f ? 0.0f : z * s, r, s);
    }
    if constexpr (ACT == FG_ACT_GELU) {
        const float density = 0.3989422804014327f * exp_fast(-0.5f * z * z);
        return 0.5f * erfcf(-0.7071067811865476f * z) + (density == 0.0f ? 0.0f : z * density);
    }
    if constexpr (ACT == FG_ACT_GELU_TANH) {
        float s, r;
        logistic(2.0f * kGeluC * fmaf(kGeluD * z * z, z, z), s, r);
        const float both = s * r;
        return s + (both == 0.0f ? 0.0f : z * both * 2.0f * kGeluC * fmaf(3.0f * kGeluD * z, z, 1.0f));
    }
    return 1.0f;
}
// All of x, one choice for them together.
template <int N>
__device__ __forceinline__ void activate_all(int act, float (&x)[N]) {
    switch (act) {
        case FG_ACT_RELU:
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = activate<FG_ACT_RELU>(x[i]);
            break;
        case FG_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = activate<FG_ACT_GELU>(x[i]);
            break;
        case FG_ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = activate<FG_ACT_GELU_TANH>(x[i]);
            break;
        case FG_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = activate<FG_ACT_SILU>(x[i]);
            break;
        default: break;
    }
}

template <int DT>
__device__ __forceinline__ float from_bits(uint16_t b) {
    if constexpr (DT == FG_DTYPE_F16) return __half2float(__ushort_as_half(b));
    else return __uint_as_float(uint32_t(b) << 16);
}
template <int DT>
__device__ __forceinline__ uint16_t to_bits(float x) {
    if constexpr (DT == FG_DTYPE_F16) return __half_as_ushort(__float2half_rn(x));
    else return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

// ---- the product -----------------------------------------------------------
constexpr int A_BYTES = TILE_L * TILE_K * 2;
constexpr int BLOCK_BYTES = 64 * TILE_K * 2;       // an MN-major box: 64 elements by 64 steps of K
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
template <int DT> struct Pieces { static constexpr int STEPS = DT == FG_DTYPE_BF16 ? 256 : 64; };   // of K, one accumulation

struct Control {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES];
    uint64_t acc_full[MAX_ACC], acc_empty[MAX_ACC], drain;
    uint32_t tmem;
    int abort;      // someone's wait ran out: everyone stops waiting
};

// An MN-major tile of 16-bit elements: blocks of 64 (128 bytes a step of K, 128-byte
// swizzle), eight steps of K 1024 bytes apart, the next 64 elements BLOCK_BYTES further.
// 16 steps of K are 2048 bytes.
__device__ __forceinline__ uint64_t mn_desc(uint32_t smem) {
    return uint64_t((smem & 0x3ffffu) >> 4) | (uint64_t(BLOCK_BYTES >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ void tmem_ld16(float (&v)[16], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ float load_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// This thread's lane of the results, N neighbouring columns at a time.
template <int DT>
struct Lane {
    const Params& P;
    bool in;               // the lane is one of the result's
    float bias;
    const uint16_t* residual;
    uint16_t* out;
    float* preact;
    __device__ __forceinline__ Lane(const Params& p, int l) : P(p), in(l < p.L) {
        bias = P.bias && in ? from_bits<DT>(reinterpret_cast<const uint16_t*>(P.bias)[l]) : 0.0f;
        residual = P.residual ? reinterpret_cast<const uint16_t*>(P.residual) + l : nullptr;
        out = reinterpret_cast<uint16_t*>(P.out) + l;
        preact = P.preact ? P.preact + l : nullptr;
    }
    template <int N>
    __device__ __forceinline__ void load(int c, uint16_t (&r)[N]) const {
        if (!residual || !in) return;
        const uint16_t* p = residual + int64_t(c) * P.residual_stride;
        if (c + N <= P.C) {
#pragma unroll
            for (int i = 0; i < N; ++i, p += P.residual_stride) r[i] = *p;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i, p += P.residual_stride)
                if (c + i < P.C) r[i] = *p;
        }
    }
    template <int N>
    __device__ __forceinline__ void store(int c, float (&x)[N], const uint16_t (&r)[N]) const {
        if (!in) return;
        const int n = min(N, P.C - c);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] += bias;
        if (preact) {
            float* p = preact + int64_t(c) * P.preact_stride;
#pragma unroll
            for (int i = 0; i < N; ++i, p += P.preact_stride)
                if (i < n) *p = x[i];
        }
        activate_all(P.act, x);
        if (residual) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] += from_bits<DT>(r[i]);
        }
        uint16_t* p = out + int64_t(c) * P.out_stride;
        if (n == N) {
#pragma unroll
            for (int i = 0; i < N; ++i, p += P.out_stride) *p = to_bits<DT>(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i, p += P.out_stride)
                if (i < n) *p = to_bits<DT>(x[i]);
        }
    }
};

// Tile t's place: along the lanes within a band of BAND tiles first, then along the columns, so
// that what runs at the same time is a square of the result and shares its operands in L2.
constexpr int BAND = 8;
__device__ __forceinline__ void place_of(const Params& P, int t, int& lt, int& ct) {
    const int band = t / (BAND * P.nc), l0 = band * BAND, high = min(BAND, P.nl - l0), in = t - l0 * P.nc;
    lt = l0 + in % high;
    ct = in / high;
}

// N pairs of columns, GROUPS apart from pair p on: the splits' parts of them, which lie in the
// CTAs' shared memory `at` bytes behind `ring`, added in the order of the splits. All parts of
// a few pairs, or one split's parts of several, are on their way together.
constexpr int GROUPS = EPI_WARPS * 32 / TILE_L;
template <int DT, int N>
__device__ __forceinline__ void add_parts(const Params& P, const Lane<DT>& out, const uint8_t* ring, uint32_t at, int c0,
                                          int p, int pairs) {
    constexpr int TOGETHER = N == 1 ? MAX_SPLITS : 2;
    float x[N][2] = {};
    uint16_t r[N][2] = {};
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (p + j * GROUPS < pairs) out.load(c0 + 2 * (p + j * GROUPS), r[j]);
#pragma unroll 1
    for (int q = 0; q < P.splits; q += TOGETHER) {
        float part[TOGETHER][N][2];
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int c = 2 * min(p + j * GROUPS, pairs - 1) + i;
                    part[k][j][i] = q + k < P.splits ? load_cluster(tc::mapa(ring, q + k) + at + c * TILE_L * 4) : 0.0f;
                }
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) x[j][i] += part[k][j][i];
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (p + j * GROUPS < pairs && c0 + 2 * (p + j * GROUPS) < P.C) out.store(c0 + 2 * (p + j * GROUPS), x[j], r[j]);
}

// Persistent over its tiles, one CTA an SM (CG = 1) or a pair of CTAs for two (CG = 2:
// 256 lanes). Warp 0 loads (TMA), warp 1 issues the products, eight warps are the
// epilogue, two for each quarter of the accumulator's lanes. Accumulators take turns, so
// that one tile's epilogue runs beside the next one's products.
//
// Where a call has too few tiles for the machine, a cluster of `splits` CTAs takes one
// tile, each a part of the sum over K; the parts meet in shared memory, where every CTA
// adds up its share of the columns, in the order of the parts.
//
// The tensor core truncates when it accumulates (about 0.05 n units of 2^-23 over n
// elements of one sign), so the sum is taken in pieces, which the epilogue adds with
// rounding: of 4096 for float16 (an eighth of half a unit of the result at most), of 16384
// for bfloat16 (a twentieth). bfloat16 with pieces of 4096 instead: 4096 tokens, 16384 x 4096
// 397 us against 384, a training step of 16384 tokens, 4096 x 4096, 1276 against 1257; sums of
// 8192 no difference.
//
// Bound: the weight's bytes for a few tokens (1 token, 4096 x 4096, bf16: 10 us with its 33.6 MB,
// floor 5.1; the launch, the ring's fill and the parts' exchange are the rest), the tensor pipe
// for many (8192 tokens, 4096 x 4096, launches alone: forward with SiLU, residual and fp32 sums
// 200 us, dx 179 us = 1.53 PFLOP/s, tensor pipe active 83 %; dW 206 us, 256 tiles over 74 pairs),
// in a long loop at the clock that the power limit leaves. 1024 tokens: 34 us, one wave of 64 pairs whose start and epilogue no other tile covers.
//
// Every wait is bounded (P.wait_ns). Where one runs out, the CTA (and its pair) stops
// waiting, the epilogue writes NaN for what it has not stored, and the CTA lets its
// products and copies in flight come to an end before it frees the tensor memory.
template <int CG, int DT, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(THREADS, 1)
product_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap, const Params P) {
    extern __shared__ uint8_t dyn[];
    __shared__ Control C;
    uint8_t* ring = dyn + ((1024 - (smem_u32(dyn) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 || P.splits > 1 ? tc::cta_rank() : 0;
    const uint32_t half = CG == 2 ? rank : 0;                 // of the pair
    const int split = CG == 1 && P.splits > 1 ? int(rank) : 0;
    const int S = P.stages;
    const int cols = P.nt / CG;                               // of B in this CTA
    const int stage_bytes = A_BYTES + cols * TILE_K * 2;
    const int nk_all = (P.K + TILE_K - 1) / TILE_K;
    const int k_lo = nk_all * split / P.splits, nk = nk_all * (split + 1) / P.splits - k_lo;   // this CTA's steps
    constexpr int PIECE = Pieces<DT>::STEPS;
    const int tiles = P.nl * P.nc;
    const int share = CG * P.splits;                          // CTAs of a tile
    const int first = blockIdx.x / share, step = gridDim.x / share;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&C.full[s], 1);
            mbar_init(&C.empty[s], 1);
        }
        for (int i = 0; i < P.accs; ++i) {
            mbar_init(&C.acc_full[i], i == P.withhold ? 2 : 1);
            mbar_init(&C.acc_empty[i], CG * EPI_WARPS);
        }
        mbar_init(&C.drain, 1);
        C.abort = 0;
        fence_mbar_init();
        tc::prefetch_map(&amap);
        tc::prefetch_map(&bmap);
    }
    if (warp == 1) {
        tc::tmem_alloc<CG>(&C.tmem, P.tmem_cols);
        tc::fence_before();
    }
    __syncthreads();
    if (CG == 2) tc::cluster_sync();   // both CTAs' barriers stand
    tc::fence_after();
    const uint32_t tmem = C.tmem;
    tc::wait_prerequisites();
    tc::launch_dependents();

    auto give_up = [&]() {   // (the pair's other CTA cannot go on alone)
        *reinterpret_cast<volatile int*>(&C.abort) = 1;
        if (CG == 2) tc::store_cluster(tc::mapa(&C.abort, rank ^ 1), 1);
    };
    if (warp == 0) {
        if (lane == 0) {
            // operands written by the kernel before: ordinary stores, read here by TMA
            asm volatile("fence.proxy.async.global;" ::: "memory");
            const uint32_t ring_a = smem_u32(ring);
            const uint32_t full0 = CG == 2 ? tc::mapa(&C.full[0], 0) : smem_u32(&C.full[0]);
            int stage = 0;
            uint32_t parity = 1;   // of the ring's previous round: a fresh barrier counts as passed with parity 1
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                int lt, ct;
                place_of(P, t, lt, ct);
                const int l0 = (lt * CG + half) * TILE_L, c0 = ct * P.nt + half * cols;
                for (int k = k_lo; k < k_lo + nk; ++k) {
                    if (!mbar_wait(&C.empty[stage], parity, &C.abort, P.wait_ns)) { ok = false; break; }
                    if (half == 0) mbar_arrive_expect_tx(&C.full[stage], CG * stage_bytes);
                    const uint32_t a = ring_a + stage * stage_bytes, b = a + A_BYTES, bar = full0 + 8 * stage;
                    if constexpr (A_MN) {
                        tc::tma_load_2d<CG>(a, &amap, l0, k * TILE_K, bar);
                        tc::tma_load_2d<CG>(a + BLOCK_BYTES, &amap, l0 + 64, k * TILE_K, bar);
                    } else {
                        tc::tma_load_2d<CG>(a, &amap, k * TILE_K, l0, bar);
                    }
                    if constexpr (B_MN) {
                        for (int c = 0; c < cols; c += 64)
                            tc::tma_load_2d<CG>(b + c / 64 * BLOCK_BYTES, &bmap, c0 + c, k * TILE_K, bar);
                    } else {
                        tc::tma_load_2d<CG>(b, &bmap, k * TILE_K, c0, bar);
                    }
                    if (++stage == S) {
                        stage = 0;
                        parity ^= 1;
                    }
                }
            }
            if (!ok) give_up();
        }
    } else if (warp == 1) {
        if (lane == 0 && half == 0) {
            const uint32_t idesc = tc::instr_desc(DT, TILE_L * CG, P.nt) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);
            const uint32_t ring_a = smem_u32(ring);
            const uint64_t a0 = A_MN ? mn_desc(ring_a) : tc::operand_desc(ring_a);
            const uint64_t b0 = B_MN ? mn_desc(ring_a + A_BYTES) : tc::operand_desc(ring_a + A_BYTES);
            constexpr int A_STEP = A_MN ? 128 : 2, B_STEP = B_MN ? 128 : 2;   // 16 elements of K, in 16 bytes
            int stage = 0, acc = 0;
            uint32_t parity = 0, acc_parity = 1;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                for (int k0 = 0; k0 < nk && ok; k0 += PIECE) {
                    const int k1 = min(nk, k0 + PIECE);
                    if (!mbar_wait(&C.acc_empty[acc], acc_parity, &C.abort, P.wait_ns)) { ok = false; break; }
                    tc::fence_after();
                    const uint32_t d = tmem + acc * P.nt;
                    for (int k = k0; k < k1; ++k) {
                        if (!mbar_wait(&C.full[stage], parity, &C.abort, P.wait_ns)) { ok = false; break; }
                        tc::fence_after();
                        const uint64_t ad = a0 + uint32_t(stage * stage_bytes) / 16;
                        const uint64_t bd = b0 + uint32_t(stage * stage_bytes) / 16;
#pragma unroll
                        for (int i = 0; i < TILE_K / 16; ++i)
                            tc::mma<CG>(d, ad + A_STEP * i, bd + B_STEP * i, idesc, k > k0 || i > 0);
                        tc::commit<CG>(&C.empty[stage]);
                        if (++stage == S) {
                            stage = 0;
                            parity ^= 1;
                        }
                    }
                    if (ok) tc::commit<CG>(&C.acc_full[acc]);
                    if (++acc == P.accs) {
                        acc = 0;
                        acc_parity ^= 1;
                    }
                }
            }
            if (!ok) give_up();
            // no product is in flight when this thread is done, whatever the others made of them
            tc::commit_here<CG>(&C.drain);
            mbar_wait_for(&C.drain, 0, WAIT_LIMIT_NS);
        }
    } else {
        const int quarter = warp & 3, part = (warp - 2) >> 2;
        constexpr int PARTS = EPI_WARPS / 4;
        const uint32_t empty_bar = CG == 2 ? tc::mapa(&C.acc_empty[0], 0) : smem_u32(&C.acc_empty[0]);
        const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
        int acc = 0;
        uint32_t acc_parity = 0;
        auto free_acc = [&](int which) {   // an accumulator is read
            tc::fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) tc::arrive_cluster(empty_bar + 8 * which);
                else mbar_arrive_a(empty_bar + 8 * which);
            }
        };
        auto next_acc = [&]() {
            if (++acc == P.accs) {
                acc = 0;
                acc_parity ^= 1;
            }
        };
        bool gone = false;   // gave up
        for (int t = first; t < tiles; t += step) {
            int lt, ct;
            place_of(P, t, lt, ct);
            const int c0 = ct * P.nt;
            const Lane<DT> out(P, (lt * CG + half) * TILE_L + quarter * 32 + lane);
            // the residual's columns come ahead: the first before the products are done
            uint16_t next[16] = {};
            if (P.splits == 1 && !gone) out.load(c0 + part * 16, next);
            int before = -1;
            for (int k0 = 0; k0 < nk && !gone; k0 += PIECE) {
                // a wait of the whole warp: all lanes go on or none
                gone = !__all_sync(0xffffffffu, mbar_wait(&C.acc_full[acc], acc_parity, &C.abort, P.wait_ns));
                if (gone) break;
                tc::fence_after();
                if (before >= 0) {
                    // this warp's columns of a piece take what the one before it holds
#pragma unroll 1
                    for (int i = part * 16; i < P.nt; i += 16 * PARTS) {
                        float x[16], y[16];
                        tmem_ld16(x, lanes + acc * P.nt + i);
                        tmem_ld16(y, lanes + before * P.nt + i);
                        tc::tmem_wait_ld(x);
                        tc::tmem_wait_ld(y);
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] += y[j];
                        tc::tmem_st8(x, lanes + acc * P.nt + i);
                        tc::tmem_st8(x + 8, lanes + acc * P.nt + i + 8);
                    }
                    tc::tmem_wait_st();
                    free_acc(before);
                }
                before = acc;
                if (k0 + PIECE < nk) next_acc();
            }
            if (gone) {
                if (lane == 0) give_up();
                __syncwarp();
                if (P.splits == 1)
                    for (int i = part * 16; i < P.nt && c0 + i < P.C; i += 16 * PARTS) {
                        float x[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] = __int_as_float(0x7fc00000);
                        out.store(c0 + i, x, next);
                    }
                continue;
            }
            const uint32_t at = lanes + acc * P.nt;
            if (P.splits == 1) {
#pragma unroll 1
                for (int i = part * 16; i < P.nt; i += 16 * PARTS) {
                    if (c0 + i >= P.C) break;
                    float x[16];
                    uint16_t r[16];
                    tmem_ld16(x, at + i);
#pragma unroll
                    for (int j = 0; j < 16; ++j) r[j] = next[j];
                    if (i + 16 * PARTS < P.nt) out.load(c0 + i + 16 * PARTS, next);
                    tc::tmem_wait_ld(x);
                    out.store(c0 + i, x, r);
                }
            } else {
                // this part of the sum, where the ring was: [column][lane]
                float* sums = reinterpret_cast<float*>(ring) + quarter * 32 + lane;
#pragma unroll 1
                for (int i = part * 16; i < P.nt; i += 16 * PARTS) {
                    float x[16];
                    tmem_ld16(x, at + i);
                    tc::tmem_wait_ld(x);
#pragma unroll
                    for (int j = 0; j < 16; ++j) sums[(i + j) * TILE_L] = x[j];
                }
            }
            free_acc(acc);
            next_acc();
        }
    }
    tc::fence_before();
    __syncthreads();
    const bool aborted = *reinterpret_cast<volatile int*>(&C.abort) != 0;
    if (aborted) {   // copies in flight land before the CTA goes on: a wait by time
        for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 10000000;) {}
        if (P.splits > 1)
            for (int i = threadIdx.x; i < P.nt * TILE_L; i += THREADS)
                reinterpret_cast<float*>(ring)[i] = __int_as_float(0x7fc00000);
    }
    __syncwarp();
    if (CG == 1 && P.splits > 1) {
        tc::cluster_sync();   // every part stands
        if (warp >= 2) {
            int lt, ct;
            place_of(P, first, lt, ct);
            const int c0 = ct * P.nt;
            const int tid = threadIdx.x - 64, l = tid % TILE_L;
            const Lane<DT> out(P, lt * TILE_L + l);
            // this CTA's columns (an even number), two at a time by each part of the threads
            const int lo = P.nt * split / P.splits, pairs = (P.nt * (split + 1) / P.splits - lo) / 2;
            const int group = tid / TILE_L;
            const uint32_t at = smem_u32(reinterpret_cast<float*>(ring) + l) - smem_u32(ring) + lo * TILE_L * 4;
            if (pairs <= GROUPS) {
                if (group < pairs) add_parts<DT, 1>(P, out, ring, at, c0 + lo, group, pairs);
            } else {
#pragma unroll 1
                for (int p = group; p < pairs; p += 4 * GROUPS) add_parts<DT, 4>(P, out, ring, at, c0 + lo, p, pairs);
            }
        }
    }
    if (CG == 2 || P.splits > 1) tc::cluster_sync();   // no CTA leaves while another may still reach it
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_free<CG>(tmem, P.tmem_cols);
    }
}

// ---- before the products ---------------------------------------------------
// Rows on 16-byte boundaries, as TMA wants them: a copy of [rows, dim] with a stride of
// a multiple of eight elements. Bound: HBM; taken for odd sizes and strides only.
__global__ void __launch_bounds__(256) align_kernel(const uint16_t* src, int64_t src_stride, uint16_t* dst,
                                                    int64_t dst_stride, int64_t rows, int dim) {
    tc::wait_prerequisites();
    tc::launch_dependents();
    const int vecs = int(dst_stride / 8);
    const int64_t all = rows * vecs;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / vecs;
        const int k = int(i % vecs) * 8;
        const uint16_t* p = src + row * src_stride + k;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = k + 2 * j < dim ? p[2 * j] : 0u, hi = k + 2 * j + 1 < dim ? p[2 * j + 1] : 0u;
            w[j] = lo | hi << 16;
        }
        *reinterpret_cast<uint4*>(dst + row * dst_stride + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// dz = g * act'(z), rounded to the operands' type for the products, and its column sums
// (of the products before rounding) over blocks of SLOPE_ROWS rows for the bias. A warp takes
// 256 columns of a row, eight a thread; the block's warps the rows by turns. Bound: HBM (z in
// fp32: a rounded z would cost the slope its last bits): 8192 x 4096 52 us, 5.2 TB/s.
constexpr int SLOPE_ROWS = 32, SLOPE_THREADS = 256, SLOPE_COLS = 256;
struct SlopeParams {
    const uint16_t* grad;
    const float* preact;      // null: act is none
    uint16_t* dz;             // null: the gradient serves as it is
    float* sums;              // [row blocks][outer], or null
    int64_t grad_stride, preact_stride, dz_stride;
    int32_t tokens, outer;
    int32_t wide;             // rows of grad and preact on 16-byte boundaries
};
template <int DT, int ACT>
__global__ void __launch_bounds__(SLOPE_THREADS) slope_kernel(const SlopeParams P) {
    __shared__ float part[SLOPE_THREADS / 32][SLOPE_COLS];
    tc::wait_prerequisites();
    tc::launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n0 = blockIdx.x * SLOPE_COLS, n = n0 + lane * 8;
    const int m0 = blockIdx.y * SLOPE_ROWS, m1 = min(P.tokens, m0 + SLOPE_ROWS);
    const bool whole = P.wide && n + 8 <= P.outer;
    float sum[8] = {};
    if (n < P.outer) {
#pragma unroll 2
        for (int m = m0 + warp; m < m1; m += SLOPE_THREADS / 32) {
            const uint16_t* g = P.grad + int64_t(m) * P.grad_stride + n;
            float x[8], y[8];
            if (whole) {
                Elem<DT>::unpack(__ldg(reinterpret_cast<const uint4*>(g)), x);
                if constexpr (ACT != FG_ACT_NONE) {
                    const float4* z = reinterpret_cast<const float4*>(P.preact + int64_t(m) * P.preact_stride + n);
                    const float4 a = __ldg(z), b = __ldg(z + 1);
                    y[0] = a.x; y[1] = a.y; y[2] = a.z; y[3] = a.w;
                    y[4] = b.x; y[5] = b.y; y[6] = b.z; y[7] = b.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[j] = n + j < P.outer ? from_bits<DT>(g[j]) : 0.0f;
                    y[j] = 0.0f;
                    if constexpr (ACT != FG_ACT_NONE)
                        if (n + j < P.outer) y[j] = P.preact[int64_t(m) * P.preact_stride + n + j];
                }
            }
            if constexpr (ACT != FG_ACT_NONE) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= slope<ACT>(y[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += x[j];
            if (P.dz) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = to_bits<DT>(x[2 * j]) | uint32_t(to_bits<DT>(x[2 * j + 1])) << 16;
                *reinterpret_cast<uint4*>(P.dz + int64_t(m) * P.dz_stride + n) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    if (P.sums) {
#pragma unroll
        for (int j = 0; j < 8; ++j) part[warp][lane * 8 + j] = sum[j];
        __syncthreads();
        const int c = threadIdx.x;
        float s = part[0][c];
#pragma unroll
        for (int w = 1; w < SLOPE_THREADS / 32; ++w) s += part[w][c];
        if (n0 + c < P.outer) P.sums[int64_t(blockIdx.y) * P.outer + n0 + c] = s;
    }
}

// The bias's gradient: the row blocks' sums, added in order by 32 threads a column group.
template <int DT>
__global__ void __launch_bounds__(256) bias_kernel(const float* sums, int blocks, int outer, uint16_t* out) {
    tc::wait_prerequisites();
    tc::launch_dependents();
    // eight parts of the blocks for each of 32 neighbouring columns
    __shared__ float part[8][32];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), p = threadIdx.x >> 5;
    float s = 0.0f;
    if (col < outer) {
#pragma unroll 8
        for (int b = blocks * p / 8; b < blocks * (p + 1) / 8; ++b) s += sums[int64_t(b) * outer + col];
    }
    part[p][threadIdx.x & 31] = s;
    __syncthreads();
    if (p == 0 && col < outer) {
        s = part[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
        out[col] = to_bits<DT>(s);
    }
}

}  // namespace lin
}  // namespace fg
