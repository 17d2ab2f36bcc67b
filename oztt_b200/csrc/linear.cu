// SPDX-License-Identifier: Apache-2.0
//
// The matrix product of a network layer with its epilogue, and its gradients, in BF16 and FP16 on the
// 5th-generation tensor cores (sm_100a). No counterpart in the reference, whose products are FP64 only.
//
//     forward    z = x w^T + b,  y = act(z) + r           x [m x k], w [n x k], b [n], r, y, z [m x n]
//     backward   dz = dy * act'(z),  dx = dz w,  dw = dz^T x,  db = the sum of dz over its m rows
//
// Every product is out[i][j] = sum_t Q(i, t) P(j, t): P, the operand of the output's columns j (contiguous in
// memory), is the 128-row side of the tensor-core tile, so that a warp of the epilogue owns neighbouring
// columns; Q, the operand of the output's rows i, is the other side, as narrow as 16 rows for a single token.
// Either operand may have its reduction index t contiguous (K-major) or its row index (MN-major): the weight
// serves the forward product and dx, and dz and x serve dw, as they lie in memory.
//
// Sums are held in 32 bits (the tensor core's accumulator) and joined in 32 bits; the bias, the activation and
// the residual are applied to the 32-bit sum, and each output is rounded once. dz is rounded once to the
// operands' type, since the tensor core takes it so; db is summed from dz before that rounding.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "launch.cuh"
#include "runtime.cuh"
#include "tensor_core.cuh"

namespace oztt {

// Both of launch.cuh.
constexpr int MOST_WORDS = 64;  // devices beyond share the last
static std::atomic<int*> known_words{nullptr};
int* error_word(int device) {
    static std::mutex mu;
    if (!known_words) {
        std::lock_guard<std::mutex> lock(mu);
        if (!known_words) {
            int* words = nullptr;
            cudaError_t failed;
            {
                OutsideCapture outside;
                failed = cudaHostAlloc(&words, MOST_WORDS * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
            }
            if (failed != cudaSuccess) {  // the next call tries again
                cudaGetLastError();
                throw Error(OZTT_ERUNTIME,
                            std::string("linear: no pinned host memory for the error words: ") + cudaGetErrorString(failed));
            }
            std::fill(words, words + MOST_WORDS, 0);
            known_words = words;
        }
    }
    return known_words + std::min(device, MOST_WORDS - 1);
}
void check_earlier_calls(int device) {
    if (device < 0) throw Error(OZTT_EINVAL, "device_id must be nonnegative");
    if (!known_words) return;  // no product has run
    if (const int code = __atomic_exchange_n(error_word(device), 0, __ATOMIC_RELAXED))
        throw Error(OZTT_ERUNTIME, "linear: a kernel of an earlier call gave up waiting (code " + std::to_string(code) +
                                       "); that call's outputs are not valid");
}

namespace layer {

using namespace gemm;

constexpr uint32_t BP = 128;            // rows of P in a tile
constexpr uint32_t BK = 64;             // reduction elements per stage: 128 bytes, one swizzle row
constexpr uint32_t UK = 16;             // reduction elements of one tcgen05.mma
constexpr uint32_t P_BYTES = BP * BK * 2;
constexpr uint32_t THREADS = 192;       // warp 0 loads, warp 1 issues the products, warps 2-5 read the sums
constexpr uint32_t MN_BOX = 64;         // rows of one MN-major box: 128 bytes
constexpr uint32_t MN_BOX_BYTES = MN_BOX * BK * 2;
constexpr uint32_t MAX_SPLIT = 16;      // CTAs of a cluster that share one tile's reduction

// A 16-bit matrix by its pointer and strides in elements.
struct View {
    void* p;
    int64_t rs, cs;
};

struct Epilogue {
    uint64_t rows, cols;                 // of the output
    View out, pre, res;                  // pre and res may be null
    const void* bias;                    // may be null
    int64_t bias_stride;
    int32_t act;                         // OZTT_ACT_*
    int32_t vec;                         // columns that one access may take: 1, 4, 8 or 16
};

// ---- activations in 32 bits ----------------------------------------------------------------------
// On pairs of values (one instruction of the packed FP32 pipe each), with the two special functions 2^x and 1/x by
// the hardware's approximations (2^-22): a pass over dz issues 11 (SILU) to 18 (GELU) instructions an element so, with
// scalar ones more than twice as many. Only those two flush: a factor 2^x below 2^-126 is zero, so results below |z| 2^-126 in size may be too. Sums, biases,
// residuals and products keep subnormal values, as the tensor cores do.
__device__ __forceinline__ f32x2 exp2_2(f32x2 x) {
    float a, b;
    unpk2(x, a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    return pk2(a, b);
}
__device__ __forceinline__ f32x2 reciprocal2(f32x2 x) {
    float a, b;
    unpk2(x, a, b);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
    return pk2(a, b);
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTanhScale = 0.7978845608028654f;  // sqrt(2/pi)
constexpr float kTanhCube = 0.044715f;

// 1 / (1 + 2^x): the logistic function of -x ln 2
__device__ __forceinline__ f32x2 logistic2(f32x2 x) { return reciprocal2(plus2(splat2(1.0f), exp2_2(x))); }

// The normal distribution's cumulative function, and e = exp(-z^2 / 2) on the way. In the lower tail it is
// e erfcx(|z| / sqrt 2) / 2, and that factor, smooth and between 1/2 and 0, is t (a1 + t (a2 + ... + t a6)) with
// t = 1 / (1 + 0.29 |z|): coefficients fitted for the least of the largest errors, by linear programming over a grid of
// [0, 13.6], within 2^-13.8 of itself everywhere and 8.1e-8 absolutely. So the tail is right relative to its own size as
// far as BF16 reaches, and the upper half to 2.5e-7 in 32-bit arithmetic. No branch, and no cancellation.
__device__ __forceinline__ f32x2 normal_cdf2(f32x2 z, f32x2& e) {
    const f32x2 size = z & 0x7FFFFFFF7FFFFFFFull;
    const f32x2 t = reciprocal2(fused2(splat2(0.29f), size, splat2(1.0f)));
    f32x2 q = fused2(splat2(-0.0882913856f), t, splat2(0.283034694f));
    q = fused2(q, t, splat2(-0.0906950769f));
    q = fused2(q, t, splat2(0.177939345f));
    q = fused2(q, t, splat2(0.101187212f));
    q = fused2(q, t, splat2(0.116825293f));
    e = exp2_2(times2(times2(z, splat2(-0.5f * kLog2e)), z));
    float tail0, tail1, z0, z1;
    unpk2(times2(times2(q, t), e), tail0, tail1);
    unpk2(z, z0, z1);
    return pk2(z0 < 0.0f ? tail0 : 1.0f - tail0, z1 < 0.0f ? tail1 : 1.0f - tail1);
}

// gelu_tanh is z (1 + tanh u) / 2 = z / (1 + exp(-2u)): no cancellation in the lower tail.
template <int ACT>
__device__ __forceinline__ f32x2 activate2(f32x2 z) {
    if constexpr (ACT == OZTT_ACT_RELU) {
        float a, b;
        unpk2(z, a, b);
        asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(a));
        asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(b));
        return pk2(a, b);
    } else if constexpr (ACT == OZTT_ACT_GELU) {
        f32x2 e;
        return times2(z, normal_cdf2(z, e));
    } else if constexpr (ACT == OZTT_ACT_GELU_TANH) {
        constexpr float c = -2.0f * kTanhScale * kLog2e;
        return times2(z, logistic2(times2(z, fused2(splat2(c * kTanhCube), times2(z, z), splat2(c)))));
    } else if constexpr (ACT == OZTT_ACT_SILU) {
        return times2(z, logistic2(times2(z, splat2(-kLog2e))));
    }
    return z;
}
// dz of a pair: dy times the activation's derivative at z.
template <int ACT>
__device__ __forceinline__ f32x2 through_slope2(f32x2 dy, f32x2 z) {
    if constexpr (ACT == OZTT_ACT_RELU) {
        float d0, d1, z0, z1;
        unpk2(dy, d0, d1);
        unpk2(z, z0, z1);
        return pk2(z0 > 0.0f ? d0 : 0.0f * d0, z1 > 0.0f ? d1 : 0.0f * d1);
    } else if constexpr (ACT == OZTT_ACT_GELU) {
        f32x2 e;
        const f32x2 c = normal_cdf2(z, e);
        return times2(dy, fused2(times2(z, splat2(0.3989422804014327f)), e, c));
    } else if constexpr (ACT == OZTT_ACT_SILU) {
        // z s(z) with s the logistic function: s + z s (1 - s) = s (1 + z (1 - s))
        const f32x2 s = logistic2(times2(z, splat2(-kLog2e)));
        return times2(times2(dy, s), fused2(z, sub2(splat2(1.0f), s), splat2(1.0f)));
    } else if constexpr (ACT == OZTT_ACT_GELU_TANH) {
        // z s(u): s + z u' s (1 - s), u' = a + b z^2, summed as s + a t + b z (z t) with t = z s (1 - s), which is zero long
        // before a power of z alone would leave the range. (db of 8192 x 16384: 104 us, 99 with the powers first, whose
        // products are NaN from 1.2e13 on; 105 and 107 with z or z^2 cut off by scalar instructions.)
        constexpr float c = -2.0f * kTanhScale * kLog2e;
        const f32x2 s = logistic2(times2(z, fused2(splat2(c * kTanhCube), times2(z, z), splat2(c))));
        const f32x2 t = times2(z, times2(s, sub2(splat2(1.0f), s)));
        const f32x2 slope = fused2(splat2(2.0f * kTanhScale), t, s);
        return times2(dy, fused2(splat2(6.0f * kTanhScale * kTanhCube), times2(z, times2(z, t)), slope));
    }
    return dy;
}

// FP16 (HALF) or BF16 values by their bits; a pair has its first value in the low half.
template <bool HALF>
__device__ __forceinline__ float to_f32(uint32_t v) {
    return HALF ? __half2float(__ushort_as_half((unsigned short)v)) : __uint_as_float(v << 16);
}
template <bool HALF>
__device__ __forceinline__ uint16_t from_f32(float v) {
    return HALF ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
template <bool HALF>
__device__ __forceinline__ f32x2 unpack(uint32_t w) {
    if (HALF) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        return pk2(f.x, f.y);
    }
    return pk2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <bool HALF>
__device__ __forceinline__ uint32_t pack(f32x2 v) {
    uint32_t w;
    float lo, hi;
    unpk2(v, lo, hi);
    if (HALF)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// 16-bit values w.. by one access of 8, 16 or (stores) 32 bytes.
__device__ __forceinline__ void load_words(const uint16_t* p, uint32_t (&w)[2]) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
}
__device__ __forceinline__ void load_words(const uint16_t* p, uint32_t (&w)[4]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
}
__device__ __forceinline__ void store_words(uint16_t* p, const uint32_t (&w)[2]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_words(uint16_t* p, const uint32_t (&w)[4]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_words(uint16_t* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// ---- the tile product ----------------------------------------------------------------------------
struct Product {
    CUtensorMap p, q;
    Epilogue e;
    uint32_t tiles_p, tiles_q, num_kb;   // tiles along the output's columns and rows; 64-element blocks to sum
    uint32_t idesc;
    uint32_t p_mn, q_mn;                 // 1: the operand is MN-major
};
// One or two products of one launch (dx and dw of a backward pass): the tiles of the first, then the second's.
template <int COUNT>
struct Products {
    Product of[COUNT];
    uint32_t tiles0, tiles;              // the first's, and all
    // the product of a tile, whose number becomes one among the product's own
    __device__ __forceinline__ const Product& at(uint32_t& tile) const {
        if (COUNT == 1 || tile < tiles0) return of[0];
        tile -= tiles0;
        return of[COUNT - 1];
    }
};

__device__ __forceinline__ void tma_load_2d(const CUtensorMap* map, uint32_t dst, uint64_t* bar, int32_t c0,
                                            int32_t c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
        : "memory");
}

// Shared-memory descriptor of a 128-byte-swizzled operand: 8-row (K-major) or 8-k (MN-major) groups 1024 bytes
// apart; MN-major operands wider than 64 rows continue one box (8 KB) further.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, uint32_t mn) {
    const uint64_t lead = mn ? (MN_BOX_BYTES >> 4) : 1u;
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (lead << 16) | ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1u << 46) |
           ((uint64_t)2u << 61);
}

__device__ __forceinline__ void umma_16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

__device__ __forceinline__ float ld_cluster_f1(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// One operand's 64-element block of the reduction into shared memory: one box of `rows` rows when K-major, one
// for every 64 rows when MN-major. Coordinates outside the matrix read as zero.
__device__ __forceinline__ void load_operand(const CUtensorMap* map, uint32_t dst, uint64_t* bar, int32_t row,
                                             int32_t k, uint32_t rows, uint32_t mn) {
    if (mn) {
        for (uint32_t b = 0; b < rows / MN_BOX; ++b)
            tma_load_2d(map, dst + b * MN_BOX_BYTES, bar, row + (int32_t)(b * MN_BOX), k);
    } else {
        tma_load_2d(map, dst, bar, k, row);
    }
}

// 2 N sums through the activation: the choice is made once for all.
template <int N>
__device__ __forceinline__ void activate_all(f32x2 (&z)[N], int act) {
    switch (act) {
#define OZTT_CASE(A) \
    case A:          \
        _Pragma("unroll") for (int q = 0; q < N; ++q) z[q] = activate2<A>(z[q]); \
        break;
        OZTT_CASE(OZTT_ACT_RELU)
        OZTT_CASE(OZTT_ACT_GELU)
        OZTT_CASE(OZTT_ACT_GELU_TANH)
        OZTT_CASE(OZTT_ACT_SILU)
#undef OZTT_CASE
        default: break;
    }
}

__device__ __forceinline__ uint16_t* element(const View& v, uint64_t i, uint64_t j) {
    return reinterpret_cast<uint16_t*>(v.p) + (int64_t)i * v.rs + (int64_t)j * v.cs;
}

// Activation, residual and the stores of 2 N neighbouring columns, their bias added: every one of them exists, and the
// views take accesses of so many values. out, pre (or null): where they go; r: the residual's words, if has_res.
template <bool HALF, int N>
__device__ __forceinline__ void finish_vector(uint16_t* out, uint16_t* pre, bool has_res, int act, f32x2 (&z)[N],
                                              const uint32_t (&r)[N]) {
    uint32_t w[N];
    if (pre) {
#pragma unroll
        for (int q = 0; q < N; ++q) w[q] = pack<HALF>(z[q]);
        store_words(pre, w);
    }
    activate_all<N>(z, act);
    if (has_res) {
#pragma unroll
        for (int q = 0; q < N; ++q) z[q] = plus2(z[q], unpack<HALF>(r[q]));
    }
#pragma unroll
    for (int q = 0; q < N; ++q) w[q] = pack<HALF>(z[q]);
    store_words(out, w);
}
// A lane's values by accesses of one value: where the first of them lies in each view, and how far apart they are.
struct Scattered {
    uint16_t *out, *pre;
    const uint16_t* res;
    int64_t out_step, pre_step, res_step;
    // from (i, j) on, in steps of di rows and dj columns
    __device__ __forceinline__ Scattered(const Epilogue& e, uint64_t i, uint64_t j, int64_t di, int64_t dj)
        : out(element(e.out, i, j)), pre(e.pre.p ? element(e.pre, i, j) : nullptr), res(e.res.p ? element(e.res, i, j) : nullptr),
          out_step(di * e.out.rs + dj * e.out.cs), pre_step(di * e.pre.rs + dj * e.pre.cs),
          res_step(di * e.res.rs + dj * e.res.cs) {}
    template <int N>
    __device__ __forceinline__ void advance() {
        out += N * out_step;
        if (pre) pre += N * pre_step;
        if (res) res += N * res_step;
    }
};
// The same as finish_vector for N values, of which the first `count` are inside the output.
template <bool HALF, int N>
__device__ __forceinline__ void finish_scattered(const Scattered& at, uint32_t count, int act, const float (&sums)[N]) {
    uint16_t r[N];
    f32x2 z[(N + 1) / 2];
    const auto each = [&](auto* p, int64_t step, auto&& f) {
#pragma unroll
        for (uint32_t q = 0; q < N; ++q, p += step)
            if (q < count) f(p, q);
    };
    if (at.res) each(at.res, at.res_step, [&](const uint16_t* p, uint32_t q) { r[q] = *p; });
#pragma unroll
    for (int q = 0; q < (N + 1) / 2; ++q) z[q] = pk2(sums[2 * q], 2 * q + 1 < N ? sums[2 * q + 1 < N ? 2 * q + 1 : 0] : 0.0f);
    const auto store = [&](uint16_t* p, int64_t step) {
        each(p, step, [&](uint16_t* to, uint32_t q) { *to = (uint16_t)(pack<HALF>(z[q / 2]) >> (16 * (q & 1))); });
    };
    if (at.pre) store(at.pre, at.pre_step);
    activate_all(z, act);
    if (at.res) {
#pragma unroll
        for (int q = 0; q < (N + 1) / 2; ++q)
            z[q] = plus2(z[q], pk2(to_f32<HALF>(r[2 * q]), 2 * q + 1 < N ? to_f32<HALF>(r[2 * q + 1 < N ? 2 * q + 1 : 0]) : 0.0f));
    }
    store(at.out, at.out_step);
}
template <bool HALF>
__device__ __forceinline__ float bias_at(const Epilogue& e, uint64_t j) {
    return e.bias && j < e.cols ? to_f32<HALF>(reinterpret_cast<const uint16_t*>(e.bias)[(int64_t)j * e.bias_stride]) : 0.0f;
}

// One tile of 128 output columns by BQ output rows per cluster; the CTAs of a cluster share the reduction: each
// sums its stretch of it in tensor memory and lays the 32-bit sums down in its own shared memory (where the
// operand stages were), then each finishes its share of the rows, adding the stretches in the cluster's order
// through distributed shared memory, so the result does not depend on timing.
template <bool HALF, int COUNT, int BQ, int STAGES, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS)
    product_kernel(const __grid_constant__ Products<COUNT> ps, int* err) {
    constexpr uint32_t Q_BYTES = BQ * BK * 2;
    constexpr uint32_t STAGE_BYTES = P_BYTES + Q_BYTES;
    constexpr uint32_t TMEM_COLS = BQ < 32 ? 32 : BQ;
    static_assert(STAGES * STAGE_BYTES >= BQ * BP * 4, "the sums take the place of the operand stages");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* done_bar = empty_bar + STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t split;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
    const uint32_t rank = cluster_rank();
    uint32_t tile = blockIdx.x / split;
    const Product& pr = ps.at(tile);
    const Epilogue& e = pr.e;
    const uint32_t tp = tile % pr.tiles_p, tq = tile / pr.tiles_p;
    const uint32_t p_mn = pr.p_mn, q_mn = pr.q_mn;
    const uint32_t kb0 = (uint32_t)((uint64_t)pr.num_kb * rank / split);
    const uint32_t kb1 = (uint32_t)((uint64_t)pr.num_kb * (rank + 1) / split);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < STAGES; ++s) {
            mbar_init(full_bar + s, 1);
            mbar_init(empty_bar + s, 1);
        }
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    overlap_launches();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t stage = 0, phase = 0, filled = 0, last_phase = 0;
            bool ok = true;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(empty_bar + stage, phase ^ 1u, abort_flag, err, ERR_WAIT_PRODUCER)) {
                    ok = false;
                    break;
                }
                mbar_expect_tx(full_bar + stage, STAGE_BYTES);
                const uint32_t sp = smem_u32(smem + stage * STAGE_BYTES);
                load_operand(&pr.p, sp, full_bar + stage, (int32_t)(tp * BP), (int32_t)(kb * BK), BP, p_mn);
                load_operand(&pr.q, sp + P_BYTES, full_bar + stage, (int32_t)(tq * BQ), (int32_t)(kb * BK), BQ, q_mn);
                filled |= 1u << stage;
                last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (!ok)  // every load this thread issued lands before the CTA may exit
                for (uint32_t st = 0; st < STAGES; ++st)
                    if (filled & (1u << st)) mbar_wait_drain(full_bar + st, (last_phase >> st) & 1u, 200000000ull);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            const uint32_t step_p = p_mn ? UK * 128u : UK * 2u, step_q = q_mn ? UK * 128u : UK * 2u, idesc = pr.idesc;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(full_bar + stage, phase, abort_flag, err, ERR_WAIT_MMA_FULL)) break;
                tc_fence_after();
                const uint32_t sp = smem_u32(smem + stage * STAGE_BYTES), sq = sp + P_BYTES;
#pragma unroll
                for (uint32_t k = 0; k < BK / UK; ++k)
                    umma_16(tmem_base, operand_desc(sp + k * step_p, p_mn), operand_desc(sq + k * step_q, q_mn), idesc,
                            kb != kb0 || k != 0);
                umma_commit(empty_bar + stage);
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            umma_commit(done_bar);  // every product issued so far; also when a wait gave up
            mbar_wait_drain(done_bar, 0, 1000000000ull);
        }
    } else {
        // lane l of quarter w holds output column 32 w + l; the sums go to sums[row][column]
        const uint32_t quarter = warp & 3u;
        float* sums = reinterpret_cast<float*>(smem) + quarter * 32u + lane;
        const bool any = mbar_wait(done_bar, 0, abort_flag, err, ERR_WAIT_EPILOGUE) && kb1 > kb0;
        tc_fence_after();
        if (any) {
            const uint32_t tbase = tmem_base + ((quarter * 32u) << 16);
            constexpr int STEP = BQ < 32 ? 16 : 32;
#pragma unroll 1
            for (uint32_t c = 0; c < BQ; c += STEP) {
                uint32_t v[STEP];
                if constexpr (STEP == 32)
                    tmem_ld32(tbase + c, v);
                else
                    tmem_ld16(tbase + c, v);
#pragma unroll
                for (int q = 0; q < STEP; ++q) sums[(c + q) * BP] = __uint_as_float(v[q]);
            }
        } else {  // an empty stretch of the reduction
            for (uint32_t c = 0; c < BQ; ++c) sums[c * BP] = 0.0f;
        }
        tc_fence_before();
    }
    __syncthreads();
    if (split > 1) cluster_sync();

    // a lane finishes 4 neighbouring columns where the views allow it, else 4 columns 32 apart
    const uint64_t j0 = (uint64_t)tp * BP;
    const bool vec = e.vec >= 4 && j0 + BP <= e.cols;
    uint64_t col[4];
    float bias[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        col[q] = j0 + (vec ? lane * 4 + q : lane + 32 * q);
        bias[q] = bias_at<HALF>(e, col[q]);
    }
    const uint32_t r0 = BQ * rank / split, r1 = BQ * (rank + 1) / split;
    for (uint32_t r = r0 + warp; r < r1; r += THREADS / 32) {
        const uint64_t i = (uint64_t)tq * BQ + r;
        if (i >= e.rows) break;
        float z[4] = {bias[0], bias[1], bias[2], bias[3]};
        const uint32_t row = smem_u32(smem) + r * (BP * 4);
        if (vec) {
            uint32_t res[2] = {0, 0};
            if (e.res.p) load_words(element(e.res, i, col[0]), res);
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (uint32_t c = 0; c < split; ++c) {
                const float4 v = ld_cluster_f4(map_to(row + lane * 16, c));
                acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
            }
            f32x2 sum[2] = {pk2(z[0] + acc.x, z[1] + acc.y), pk2(z[2] + acc.z, z[3] + acc.w)};
            finish_vector<HALF, 2>(element(e.out, i, col[0]), e.pre.p ? element(e.pre, i, col[0]) : nullptr, e.res.p, e.act,
                                   sum, res);
        } else {
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t c = 0; c < split; ++c) {
                const uint32_t at = map_to(row + lane * 4, c);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[q] += ld_cluster_f1(at + 128 * q);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) z[q] += acc[q];
            if (col[0] < e.cols)
                finish_scattered<HALF, 4>(Scattered(e, i, col[0], 0, 32), (uint32_t)min((e.cols - col[0] + 31) / 32, (uint64_t)4),
                                          e.act, z);
        }
    }
    __syncthreads();
    if (split > 1) cluster_sync();  // no CTA leaves while another may read its sums
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS)
                     : "memory");
    }
}

// ---- the pair product: large outputs -----------------------------------------------------------
// The same product on CTA pairs (cta_group::2): a tile of 256 output columns by BQ output rows, each CTA of the
// pair holding 128 of the columns and half of Q's rows, so that shared memory feeds the tensor cores with the
// fewest bytes. Persistent: the pairs walk over the tiles, the sums of one tile are finished from one half of
// tensor memory while the next tile accumulates in the other. Sixteen warps finish them (the latencies of the path
// from tensor memory to the stores need so many), each 32 columns of a quarter of the rows: 8 rows at a time go
// through a patch of shared memory of the warp's own, from which a lane takes 8 neighbouring columns of a row, so
// that bias, activation, residual and stores run on 16-byte accesses. Bound by the tensor pipe where the sum is long, by
// the stores where it is short.
// TURNED, for outputs that take 32-byte accesses and have no residual: the operands change sides, a lane of tensor
// memory is a row of the output and holds its neighbouring columns, which go to memory as they are, a whole sector a
// lane and store. 8192 x 8192 x 64: 34.8 us, through patches 54.0 (stores alone 18); 4096 x 4096 x 512 18.7 and 22.3;
// 8192 x 4096 x 4096 188 and 192; with a residual, which a lane would read a sector at a time too, the patches are
// faster: 8192 x 8192 x 256 82.9 us, turned 97.7.
constexpr uint32_t PAIR_STAGES_BYTES = 196608;
constexpr uint32_t FINISHERS = 16;
constexpr uint32_t PAIR_THREADS = (2 + FINISHERS) * 32;  // warp 0 loads, warp 1 issues, the others finish
constexpr uint32_t PATCH_ROWS = 8, PATCH_LD = 36;  // padded: neither its rows nor its columns share banks
constexpr uint32_t PATCH_BYTES = PATCH_ROWS * PATCH_LD * 4;
constexpr uint32_t GROUP_Q = 8;         // rows of tiles that the running pairs share in L2
constexpr uint64_t PEER_DRAIN_NS = 5000000ull;

__device__ __forceinline__ void tma_load_2d_pair(const CUtensorMap* map, uint32_t dst, uint32_t bar_cluster, int32_t c0,
                                                 int32_t c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void load_operand_pair(const CUtensorMap* map, uint32_t dst, uint32_t bar_cluster,
                                                  int32_t row, int32_t k, uint32_t rows, uint32_t mn) {
    if (mn) {
        for (uint32_t b = 0; b < rows / MN_BOX; ++b)
            tma_load_2d_pair(map, dst + b * MN_BOX_BYTES, bar_cluster, row + (int32_t)(b * MN_BOX), k);
    } else {
        tma_load_2d_pair(map, dst, bar_cluster, k, row);
    }
}
__device__ __forceinline__ void umma_16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Tile number -> its product, tile column tp and tile row tq: groups of GROUP_Q tile rows, each walked column by
// column.
template <int COUNT>
__device__ __forceinline__ const Product& tile_at(const Products<COUNT>& ps, uint32_t tile, uint32_t& tp, uint32_t& tq) {
    const Product& pr = ps.at(tile);
    const uint32_t span = GROUP_Q * pr.tiles_p, g = tile / span, first = g * GROUP_Q;
    const uint32_t size = min(pr.tiles_q - first, GROUP_Q), r = tile - g * span;
    tq = first + r % size;
    tp = r / size;
    return pr;
}

template <bool HALF, int COUNT, int BQ, bool TURNED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    pair_product_kernel(const __grid_constant__ Products<COUNT> ps, int* err) {
    constexpr uint32_t HALF_Q = BQ / 2;
    constexpr uint32_t STAGE_BYTES = P_BYTES + HALF_Q * BK * 2;
    constexpr uint32_t STAGES = PAIR_STAGES_BYTES / STAGE_BYTES;
    constexpr uint32_t TMEM_COLS = 2 * BQ;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* patches = reinterpret_cast<float*>(smem + STAGES * STAGE_BYTES);
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES + FINISHERS * PATCH_BYTES);
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* tfull_bar = empty_bar + STAGES;
    uint64_t* tempty_bar = tfull_bar + 2;
    uint64_t* drain_bar = tempty_bar + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t first_tile = blockIdx.x >> 1, tile_step = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < STAGES; ++s) {
            mbar_init(full_bar + s, 1);
            mbar_init(empty_bar + s, 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            mbar_init(tfull_bar + a, 1);
            mbar_init(tempty_bar + a, 2 * FINISHERS);  // the finishing warps of both CTAs
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer's barriers are initialised before anything is signalled across the pair
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    // With idle pairs' SMs on the device, the next kernel starts when this one ends: its blocks would all find room on those
    // SMs and share them, where they could have the whole device a moment later (backward pass of 777 x 1535 x 1001 and the
    // next call's: 25.6 us, 29.6 when they may start early; with every SM taken 1 to 2 us the other way).
    overlap_launches(2 * ps.tiles > gridDim.x);

    if (warp == 0) {
        if (lane == 0) {
            uint32_t stage = 0, phase = 0, filled = 0, last_phase = 0;
            bool ok = true, issued = false;
            for (uint32_t tile = first_tile; ok && tile < ps.tiles; tile += tile_step) {
                uint32_t tp, tq;
                const Product& pr = tile_at(ps, tile, tp, tq);
                const uint32_t num_kb = pr.num_kb, p_mn = pr.p_mn, q_mn = pr.q_mn;
                const CUtensorMap *map_p = &pr.p, *map_q = &pr.q;
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait(empty_bar + stage, phase ^ 1u, abort_flag, err, ERR_WAIT_PRODUCER)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) mbar_expect_tx(full_bar + stage, 2 * STAGE_BYTES);
                    const uint32_t full_leader = map_to(smem_u32(full_bar + stage), 0);
                    const uint32_t sp = smem_u32(smem + stage * STAGE_BYTES);
                    load_operand_pair(map_p, sp, full_leader, (int32_t)(tp * 2 * BP + rank * BP), (int32_t)(kb * BK), BP,
                                      p_mn);
                    load_operand_pair(map_q, sp + P_BYTES, full_leader, (int32_t)(tq * BQ + rank * HALF_Q),
                                      (int32_t)(kb * BK), HALF_Q, q_mn);
                    issued = true;
                    filled |= 1u << stage;
                    last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok) {  // let the loads this thread issued land before the CTA may exit
                if (rank == 0) {
                    for (uint32_t st = 0; st < STAGES; ++st)
                        if (filled & (1u << st)) mbar_wait_drain(full_bar + st, (last_phase >> st) & 1u, 200000000ull);
                } else if (issued) {  // the peer's loads complete on the leader's barriers: wait a fixed time
                    const uint64_t t0 = global_timer_ns();
                    while (global_timer_ns() - t0 < PEER_DRAIN_NS) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            for (uint32_t tile = first_tile; ok && tile < ps.tiles; tile += tile_step) {
                uint32_t own = tile;
                const Product& pr = ps.at(own);
                const uint32_t num_kb = pr.num_kb, p_mn = pr.p_mn, q_mn = pr.q_mn, idesc = pr.idesc;
                const uint32_t step_p = p_mn ? UK * 128u : UK * 2u, step_q = q_mn ? UK * 128u : UK * 2u;
                if (!mbar_wait(tempty_bar + acc, acc_phase ^ 1u, abort_flag, err, ERR_WAIT_MMA_EMPTY)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * BQ;
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait(full_bar + stage, phase, abort_flag, err, ERR_WAIT_MMA_FULL)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sp = smem_u32(smem + stage * STAGE_BYTES), sq = sp + P_BYTES;
#pragma unroll
                    for (uint32_t k = 0; k < BK / UK; ++k)
                        umma_16_pair(d_tmem, operand_desc(sp + k * step_p, p_mn),
                                     operand_desc(sq + k * step_q, q_mn), idesc, (kb | k) != 0u);
                    const uint32_t eb = smem_u32(empty_bar + stage);
                    umma_commit_pair(eb);
                    umma_commit_pair(map_to(eb, 1));
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                const uint32_t tb = smem_u32(tfull_bar + acc);
                umma_commit_pair(tb);
                umma_commit_pair(map_to(tb, 1));
                acc ^= 1u;
                if (acc == 0) acc_phase ^= 1u;
            }
            // Every product this thread issued completes before the columns of either CTA are freed.
            umma_commit_pair(smem_u32(drain_bar));
            mbar_wait_drain(drain_bar, 0, 1000000000ull);
        }
    } else {
        // 32 columns (a quarter of the CTA's) by a quarter of the tile's rows
        constexpr uint32_t ROWS = BQ / (FINISHERS / 4);
        const uint32_t quarter = warp & 3u, c0 = ((warp - 2) >> 2) * ROWS;
        float* patch = patches + (warp - 2) * (PATCH_BYTES / 4);
        const uint32_t prow = lane >> 2, pcol = (lane & 3u) * 8u;
        uint32_t acc = 0, acc_phase = 0;
        for (uint32_t tile = first_tile; tile < ps.tiles; tile += tile_step) {
            uint32_t tp, tq;
            const Product& pr = tile_at(ps, tile, tp, tq);
            const Epilogue& e = pr.e;
            if constexpr (TURNED) {  // 32 rows by a quarter of the tile's columns
                const uint64_t i0 = (uint64_t)tp * 2 * BP + rank * BP + quarter * 32u, j0 = (uint64_t)tq * BQ + c0;
                const uint32_t cols = i0 < e.rows && j0 < e.cols ? (uint32_t)min((uint64_t)ROWS, e.cols - j0) : 0;
                const bool mine = i0 + lane < e.rows, has_bias = e.bias;
                uint16_t* out = element(e.out, i0 + lane, j0);
                uint16_t* pre = e.pre.p ? element(e.pre, i0 + lane, j0) : nullptr;
                if (has_bias) {
                    __syncwarp();  // the tile before has read its own
#pragma unroll
                    for (uint32_t c = 0; c < ROWS; c += 32) patch[c + lane] = bias_at<HALF>(e, j0 + c + lane);
                    __syncwarp();
                }
                if (!mbar_wait(tfull_bar + acc, acc_phase, abort_flag, err, ERR_WAIT_EPILOGUE)) break;
                tc_fence_after();
                const uint32_t tbase = tmem_base + ((quarter * 32u) << 16) + acc * BQ + c0;
#pragma unroll 1
                for (uint32_t c = 0; c < cols; c += 16) {
                    uint32_t v[16];
                    __syncwarp();
                    tmem_ld16(tbase + c, v);
                    f32x2 z[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q) z[q] = pk2(__uint_as_float(v[2 * q]), __uint_as_float(v[2 * q + 1]));
                    if (has_bias) {
                        const ulonglong2* b = reinterpret_cast<const ulonglong2*>(patch + c);
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const ulonglong2 x = b[q];
                            z[2 * q] = plus2(z[2 * q], x.x), z[2 * q + 1] = plus2(z[2 * q + 1], x.y);
                        }
                    }
                    if (!mine) continue;
                    if (c + 16 <= cols) {
                        finish_vector<HALF, 8>(out + c, pre ? pre + c : nullptr, false, e.act, z, {});
                    } else {
                        float f[16];
#pragma unroll
                        for (int q = 0; q < 8; ++q) unpk2(z[q], f[2 * q], f[2 * q + 1]);
                        finish_scattered<HALF, 16>(Scattered(e, i0 + lane, j0 + c, 0, 1), cols - c, e.act, f);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_remote_relaxed(map_to(smem_u32(tempty_bar + acc), 0));
                acc ^= 1u;
                if (acc == 0) acc_phase ^= 1u;
                continue;
            }
            const uint64_t j0 = (uint64_t)tp * 2 * BP + rank * BP + quarter * 32u;
            const uint64_t i0 = (uint64_t)tq * BQ + c0;
            const bool vec = e.vec >= 8 && j0 + 32 <= e.cols;
            f32x2 bias[4];
            float lane_bias = 0.0f;
            if (vec) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    bias[q] = pk2(bias_at<HALF>(e, j0 + pcol + 2 * q), bias_at<HALF>(e, j0 + pcol + 2 * q + 1));
            } else {
                lane_bias = bias_at<HALF>(e, j0 + lane);
            }
            const uint32_t rows = j0 < e.cols && i0 < e.rows ? (uint32_t)min((uint64_t)ROWS, e.rows - i0) : 0;
            // this lane's place in the first patch; the next is 8 rows further
            uint16_t* out = element(e.out, i0 + prow, j0 + pcol);
            uint16_t* pre = element(e.pre, i0 + prow, j0 + pcol);
            const uint16_t* res = element(e.res, i0 + prow, j0 + pcol);
            if (vec && e.res.p)
                for (uint32_t c = prow; c < rows; c += PATCH_ROWS) prefetch_l2(res + (c - prow) * e.res.rs);
            if (!mbar_wait(tfull_bar + acc, acc_phase, abort_flag, err, ERR_WAIT_EPILOGUE)) break;
            tc_fence_after();
            const uint32_t tbase = tmem_base + ((quarter * 32u) << 16) + acc * BQ + c0;
            if (vec) {
                const bool has_pre = e.pre.p, has_res = e.res.p;
#pragma unroll 1
                for (uint32_t c = 0; c < rows; c += PATCH_ROWS) {
                    const bool mine = c + prow < rows;
                    uint32_t r[4] = {}, v[8];
                    if (has_res && mine) load_words(res, r);
                    tmem_ld8(tbase + c, v);
                    __syncwarp();  // the patch has been read
#pragma unroll
                    for (int q = 0; q < 8; ++q) patch[q * PATCH_LD + lane] = __uint_as_float(v[q]);
                    __syncwarp();
                    const ulonglong2* p = reinterpret_cast<const ulonglong2*>(patch + prow * PATCH_LD + pcol);
                    const ulonglong2 x = p[0], y = p[1];
                    f32x2 z[4] = {plus2(x.x, bias[0]), plus2(x.y, bias[1]), plus2(y.x, bias[2]), plus2(y.y, bias[3])};
                    if (mine) finish_vector<HALF, 4>(out, has_pre ? pre : nullptr, has_res, e.act, z, r);
                    out += PATCH_ROWS * e.out.rs;
                    pre += PATCH_ROWS * e.pre.rs;
                    res += PATCH_ROWS * e.res.rs;
                }
            } else {
                Scattered at(e, i0, j0 + lane, 1, 0);
#pragma unroll 1
                for (uint32_t c = 0; c < rows; c += PATCH_ROWS) {
                    uint32_t v[8];
                    tmem_ld8(tbase + c, v);
                    float z[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q) z[q] = __uint_as_float(v[q]) + lane_bias;
                    finish_scattered<HALF, 8>(at, j0 + lane < e.cols ? rows - c : 0, e.act, z);
                    at.advance<8>();
                }
            }
            // the sums have been read: all that the arrival has to tell; a releasing one would also
            // wait for the stores
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_remote_relaxed(map_to(smem_u32(tempty_bar + acc), 0));
            acc ^= 1u;
            if (acc == 0) acc_phase ^= 1u;
        }
    }
    __syncthreads();
    cluster_sync();  // no CTA frees its tensor memory or exits while the pair may still use it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS)
                     : "memory");
    }
}

// ---- few rows ------------------------------------------------------------------------------------
// The product for up to 4 output rows (single tokens), on the 32-bit pipe: bound by the bytes of P, of which each
// is read once, and by the time to the first of them, so nothing is set up: a warp streams 4 rows of P (VEC: 16
// bytes a lane) along their reduction index and multiplies them by the rows of Q, which the first-level cache
// keeps. With few rows of P the warps of a block share their reduction and join through shared memory, in order.
// One row, BF16: 4096 x 4096 in 7.2 us (4.7 TB/s), 14080 x 3520 in 19.7 (5.0), 16384 x 16384 in 89 (6.0); with 2
// columns a warp 8.7, 24.0 and 97.6, with four accesses ahead in place of two 9.7, 20.2 and 110.7.
constexpr int FEW_COLS = 4;  // output columns (rows of P) of a warp
template <bool HALF, int M, bool VEC>
__global__ void __launch_bounds__(256)
    few_rows_kernel(const uint16_t* p, int64_t ldp, const uint16_t* q, int64_t ldq,
                    const uint32_t red, const __grid_constant__ Epilogue e) {
    __shared__ float sums[8][FEW_COLS * M];
    constexpr uint32_t STEP = VEC ? 256 : 32;  // reduction elements of a warp's access
    constexpr int AHEAD = VEC ? 2 : M > 2 ? 4 : 8;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const uint64_t j0 = blockIdx.x * (uint64_t)FEW_COLS;
    overlap_launches();
    const uint16_t* row[FEW_COLS];  // columns past the last one read it again
#pragma unroll
    for (int c = 0; c < FEW_COLS; ++c) row[c] = p + (int64_t)min(j0 + c, e.cols - 1) * ldp;
    f32x2 acc[M][FEW_COLS] = {};  // two sums, of every other element (access)
    for (uint32_t t0 = warp * STEP; t0 < red; t0 += warps * STEP * AHEAD) {
        if constexpr (VEC) {
            uint32_t w[AHEAD][FEW_COLS][4], x[AHEAD][M][4];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const uint32_t t = t0 + a * warps * STEP + lane * 8;
#pragma unroll
                for (int c = 0; c < FEW_COLS; ++c) {
                    w[a][c][0] = w[a][c][1] = w[a][c][2] = w[a][c][3] = 0;
                    if (t < red) load_words(row[c] + t, w[a][c]);  // red is a multiple of 8
                }
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    x[a][m][0] = x[a][m][1] = x[a][m][2] = x[a][m][3] = 0;
                    if (t < red) load_words(q + m * ldq + t, x[a][m]);
                }
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
#pragma unroll
                for (int h = 0; h < 4; ++h)
#pragma unroll
                    for (int c = 0; c < FEW_COLS; ++c) {
                        const f32x2 v = unpack<HALF>(w[a][c][h]);
#pragma unroll
                        for (int m = 0; m < M; ++m) acc[m][c] = fused2(v, unpack<HALF>(x[a][m][h]), acc[m][c]);
                    }
        } else {
            uint16_t w[AHEAD][FEW_COLS], x[AHEAD][M];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const uint32_t t = t0 + a * warps * STEP + lane;
#pragma unroll
                for (int c = 0; c < FEW_COLS; ++c) w[a][c] = t < red ? row[c][t] : 0;
#pragma unroll
                for (int m = 0; m < M; ++m) x[a][m] = t < red ? q[m * ldq + t] : 0;
            }
#pragma unroll
            for (int a = 0; a < AHEAD; a += 2)
#pragma unroll
                for (int c = 0; c < FEW_COLS; ++c)
#pragma unroll
                    for (int m = 0; m < M; ++m)
                        acc[m][c] = fused2(pk2(to_f32<HALF>(w[a][c]), to_f32<HALF>(w[a + 1][c])),
                                         pk2(to_f32<HALF>(x[a][m]), to_f32<HALF>(x[a + 1][m])), acc[m][c]);
        }
    }
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int c = 0; c < FEW_COLS; ++c) {
            float even, odd;
            unpk2(acc[m][c], even, odd);
            even += odd;
#pragma unroll
            for (int d = 16; d; d >>= 1) even += __shfl_xor_sync(0xFFFFFFFFu, even, d);
            if (lane == 0) sums[warp][m * FEW_COLS + c] = even;
        }
    __syncthreads();
    if (threadIdx.x < FEW_COLS * M) {
        const uint64_t i = threadIdx.x / FEW_COLS, j = j0 + threadIdx.x % FEW_COLS;
        float z[1] = {bias_at<HALF>(e, j)};
        for (uint32_t w = 0; w < warps; ++w) z[0] += sums[w][threadIdx.x];
        if (j < e.cols) finish_scattered<HALF, 1>(Scattered(e, i, j, 0, 0), 1, e.act, z);
    }
}

// ---- few terms -----------------------------------------------------------------------------------
// out[i][j] = the sum of up to T products, for dw of a few tokens, whose output the tiles of the tensor cores finish at
// 3.9 TB/s at most. Up to 4 terms are bound by the stores, more by the products on the 32-bit pipe. A warp keeps 256
// columns of P (8 a lane, contiguous) in registers and walks down 8 or 16 rows, one 16-byte store a lane and row, the
// terms' factors of a row read from shared memory. 4480 x 8576 from 2, 4 and 8 terms: 12.3, 12.6 and 22.8 us (stores
// alone 10.6, at 7.3 TB/s), by tiles 24; 1024 x 1024 2.3, 2.1 and 3.9, by tiles 6.7. 8 terms with 8 rows a warp take 15 %
// longer, with 4 columns a lane 10 %.
template <int T>
constexpr uint32_t TERM_ROWS = T > 4 ? 16 : 8;
template <bool HALF, int T>
__global__ void __launch_bounds__(256)
    few_terms_kernel(const uint16_t* p, int64_t p_term, const uint16_t* q, int64_t q_row,
                     int64_t q_term, const uint32_t red, View out, uint64_t rows, uint64_t cols) {
    constexpr uint32_t ROWS = TERM_ROWS<T>;
    __shared__ __align__(16) float factors[8 * ROWS][T];  // of the block's rows
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t j = blockIdx.x * 256ull + lane * 8, i0 = blockIdx.y * (8ull * ROWS);
    overlap_launches();
    for (uint32_t k = threadIdx.x; k < 8 * ROWS * T; k += 256) {
        const uint32_t r = k % (8 * ROWS), t = k / (8 * ROWS);
        const float a = t < red && i0 + r < rows ? to_f32<HALF>(q[(int64_t)(i0 + r) * q_row + t * q_term]) : 0.0f;
        factors[r][t] = a;
    }
    f32x2 x[T][4];
#pragma unroll
    for (uint32_t t = 0; t < T; ++t) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (t < red && j < cols) load_words(p + t * p_term + j, w);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[t][c] = unpack<HALF>(w[c]);
    }
    __syncthreads();
    const uint32_t r0 = warp * ROWS;
    if (j >= cols || i0 + r0 >= rows) return;  // (cols is a multiple of 8)
    const uint32_t count = (uint32_t)min((uint64_t)ROWS, rows - i0 - r0);
    uint16_t* to = element(out, i0 + r0, j);
#pragma unroll 2
    for (uint32_t r = 0; r < count; ++r) {
        f32x2 sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t t = 0; t < T; ++t) {
            const f32x2 a = splat2(factors[r0 + r][t]);
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] = fused2(a, x[t][c], sum[c]);
        }
        uint32_t w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = pack<HALF>(sum[c]);
        store_words(to, w);
        to += out.rs;
    }
}

// ---- passes over memory --------------------------------------------------------------------------

// Copies of operands whose base or rows do not start on 16 bytes, which the tensor copies cannot read:
// dst[o][i] = src[o * so + i * si], rows ld apart (a multiple of 8, zero beyond `inner`). Up to 4 in one launch.
// Bound by memory: a warp takes 1024 elements of a row by aligned 16-byte loads and shifts them to their places, all
// loads ahead of the first store. 4095 x 4097 and 16 x 4097 together: 12.6 us of a call (67 MB moved, 5.3 TB/s).
struct Pack {
    const uint16_t* src;
    int64_t so, si;
    uint64_t outer, inner, ld;
    uint16_t* dst;
    uint64_t end;  // units of this copy and those before it: PACK_GROUPS groups of 8 elements of a row
};
struct Packs {
    Pack of[4];
    uint32_t count;
};
constexpr uint32_t PACK_AHEAD = 4, PACK_GROUPS = 32 * PACK_AHEAD;
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Packs packs) {
    const uint32_t lane = threadIdx.x & 31;
    overlap_launches();
    const uint64_t all = packs.of[packs.count - 1].end, step = (uint64_t)gridDim.x * (blockDim.x >> 5);
    for (uint64_t t = blockIdx.x * (uint64_t)(blockDim.x >> 5) + (threadIdx.x >> 5); t < all; t += step) {
        uint32_t c = 0;
        while (t >= packs.of[c].end) ++c;
        const Pack& k = packs.of[c];
        const uint64_t unit = t - (c ? packs.of[c - 1].end : 0), per_row = (k.ld / 8 + PACK_GROUPS - 1) / PACK_GROUPS;
        const uint64_t o = (unit | per_row) >> 32 ? unit / per_row : (uint32_t)unit / (uint32_t)per_row;
        const uint64_t i0 = ((unit - o * per_row) * PACK_GROUPS + lane) * 8;
        const uint16_t* row = k.src + (int64_t)o * k.so;
        uint16_t* to = k.dst + o * k.ld;
        uint32_t v[PACK_AHEAD][8], valid[PACK_AHEAD];
        // contiguous elements come from the one or two aligned 16 bytes that hold a group's
        const uint32_t shift = k.si == 1 ? (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u : 0;
#pragma unroll
        for (uint32_t a = 0; a < PACK_AHEAD; ++a) {
            const uint64_t i = i0 + a * 256;
            valid[a] = (uint32_t)min((uint64_t)8, i < k.inner ? k.inner - i : 0);
            uint4 x = make_uint4(0, 0, 0, 0), y = x;
            if (k.si == 1) {
                const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row + i) - shift);
                if (valid[a]) x = from[0];
                if (shift + 2 * valid[a] > 16) y = from[1];
            } else {
                uint32_t w[4];
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) {
                    const uint16_t* at = row + (int64_t)(i + 2 * q) * k.si;
                    w[q] = (2 * q < valid[a] ? (uint32_t)at[0] : 0u) | (2 * q + 1 < valid[a] ? (uint32_t)at[k.si] << 16 : 0u);
                }
                x = make_uint4(w[0], w[1], w[2], w[3]);
            }
            v[a][0] = x.x, v[a][1] = x.y, v[a][2] = x.z, v[a][3] = x.w;
            v[a][4] = y.x, v[a][5] = y.y, v[a][6] = y.z, v[a][7] = y.w;
        }
#pragma unroll
        for (uint32_t a = 0; a < PACK_AHEAD; ++a) {
#pragma unroll
            for (int s = 2; s; s >>= 1)
                if (shift >> 2 & s) {
#pragma unroll
                    for (int q = 0; q + s < 8; ++q) v[a][q] = v[a][q + s];
                }
            uint32_t w[4];
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) {
                w[q] = shift & 2 ? __funnelshift_r(v[a][q], v[a][q + 1], 16) : v[a][q];
                if (valid[a] < 2 * q + 2) w[q] = valid[a] > 2 * q ? w[q] & 0xFFFFu : 0;
            }
            if (i0 + a * 256 < k.ld) store_words(to + i0 + a * 256, w);
        }
    }
}

// dz = dy * act'(z) into dz (rows ld apart; may be null), and the sums of its columns in 32 bits. A block takes 128
// columns (a lane 8 neighbouring ones by 16-byte accesses with VEC, else 8 that are 16 apart) by `span` rows, 16 at a
// time; the blocks of a cluster lie below one another and join their sums, always in the same order, through
// distributed shared memory: into db where one cluster covers all rows, else into partial[cluster][n] for db_kernel.
// (db and partial may be null.) Bound by memory, which many warps with few accesses each keep busier than few with
// many: 8192 x 16384 BF16, one read for db alone: 42 us with 8 blocks on an SM and one row ahead, 61 us with 2 and
// four (41 at the rate of a copy); two reads with gelu_tanh: 104 us with 4 blocks and two rows ahead, half as
// long again with 2 and four (82); strips of 64 columns take 6 % longer with RELU.
constexpr uint32_t DZ_COLS = 128, DZ_ROWS = 16, DZ_CLUSTER = 8;
constexpr uint32_t DZ_LANES = DZ_COLS / 8;
template <bool HALF, bool VEC, int ACT>
__global__ void __launch_bounds__(256, !VEC ? 3 : ACT == OZTT_ACT_NONE ? 8 : 4)
    dz_kernel(View dy, View z, uint64_t m, uint64_t n, uint64_t span, uint16_t* __restrict__ dz, uint64_t ld,
              float* __restrict__ partial, uint16_t* __restrict__ db, int64_t db_stride) {
    constexpr uint32_t DZ_AHEAD = ACT == OZTT_ACT_NONE ? 1 : 2;
    __shared__ float sums[DZ_ROWS][DZ_COLS];
    __shared__ float block_sums[DZ_COLS];
    const uint32_t r = threadIdx.x / DZ_LANES, l = threadIdx.x % DZ_LANES;
    const uint32_t l0 = VEC ? l * 8 : l;
    constexpr uint32_t DJ = VEC ? 1 : DZ_LANES;
    const uint64_t j0 = blockIdx.x * (uint64_t)DZ_COLS + l0;
    const uint64_t i0 = min(blockIdx.y * span, m) + r, i1 = min((blockIdx.y + 1) * span, m);
    // the columns that exist: with VEC (n a multiple of 8) all or none
    const uint32_t cols = j0 >= n ? 0 : VEC ? 8 : (uint32_t)min((n - j0 + DJ - 1) / DJ, (uint64_t)8);
    overlap_launches();
    f32x2 sum[4] = {};
    if (cols && i0 < i1) {
        const uint16_t *py = element(dy, i0, j0), *pz = element(z, i0, j0);
        uint16_t* pd = dz + i0 * ld + j0;
        const int64_t step_y = DZ_ROWS * dy.rs, step_z = DZ_ROWS * z.rs, step_d = DZ_ROWS * (int64_t)ld;
        uint32_t left = (uint32_t)((i1 - i0 + DZ_ROWS - 1) / DZ_ROWS);  // of this thread's rows
        while (left) {
            uint32_t g[DZ_AHEAD][4], s[DZ_AHEAD][4];
#pragma unroll
            for (uint32_t a = 0; a < DZ_AHEAD; ++a) {
                if (a >= left) break;
                if constexpr (VEC) {
                    load_words(py + a * step_y, g[a]);
                    if (ACT != OZTT_ACT_NONE) load_words(pz + a * step_z, s[a]);
                } else {
#pragma unroll
                    for (uint32_t q = 0; q < 4; ++q) {
                        const auto pair = [&](const uint16_t* p, int64_t cs) {
                            return (2 * q < cols ? (uint32_t)p[(int64_t)(2 * q * DJ) * cs] : 0u) |
                                   (2 * q + 1 < cols ? (uint32_t)p[(int64_t)((2 * q + 1) * DJ) * cs] << 16 : 0u);
                        };
                        g[a][q] = pair(py + a * step_y, dy.cs);
                        if (ACT != OZTT_ACT_NONE) s[a][q] = pair(pz + a * step_z, z.cs);
                    }
                }
            }
#pragma unroll
            for (uint32_t a = 0; a < DZ_AHEAD; ++a) {
                if (a >= left) break;
                uint32_t w[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f32x2 v = unpack<HALF>(g[a][q]);
                    if (ACT != OZTT_ACT_NONE) v = through_slope2<ACT>(v, unpack<HALF>(s[a][q]));
                    sum[q] = plus2(sum[q], v);
                    w[q] = pack<HALF>(v);
                }
                if (!dz) continue;
                if constexpr (VEC) {
                    store_words(pd + a * step_d, w);
                } else {
#pragma unroll
                    for (uint32_t q = 0; q < 8; ++q)
                        if (q < cols) pd[a * step_d + q * DJ] = (uint16_t)(w[q >> 1] >> (16 * (q & 1)));
                }
            }
            py += DZ_AHEAD * step_y;
            pz += DZ_AHEAD * step_z;
            pd += DZ_AHEAD * step_d;
            left -= min(left, DZ_AHEAD);
        }
    }
    if (!partial && !db) return;  // the same for every block
#pragma unroll
    for (int q = 0; q < 4; ++q) unpk2(sum[q], sums[r][l0 + 2 * q * DJ], sums[r][l0 + (2 * q + 1) * DJ]);
    __syncthreads();
    if (threadIdx.x < DZ_COLS) {
        float total = 0.0f;
#pragma unroll 8
        for (uint32_t w = 0; w < DZ_ROWS; ++w) total += sums[w][threadIdx.x];
        block_sums[threadIdx.x] = total;
    }
    __syncthreads();
    cluster_sync();
    if (cluster_rank() == 0 && threadIdx.x < DZ_COLS) {
        uint32_t blocks;
        asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
        const uint64_t j = blockIdx.x * (uint64_t)DZ_COLS + threadIdx.x;
        float total = 0.0f;
        for (uint32_t c = 0; c < blocks; ++c) total += ld_cluster_f1(map_to(smem_u32(block_sums + threadIdx.x), c));
        if (j < n) {
            if (db)
                db[(int64_t)j * db_stride] = from_f32<HALF>(total);
            else
                partial[blockIdx.y / blocks * n + j] = total;
        }
    }
    cluster_sync();  // no block leaves while its sums may be read
}

// db from the clusters' sums: a block takes 32 columns, each warp every eighth cluster.
template <bool HALF>
__global__ void __launch_bounds__(256) db_kernel(const float* partial, uint64_t clusters, uint64_t n,
                                                 uint16_t* __restrict__ db, int64_t stride) {
    __shared__ float sums[8][32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t j = blockIdx.x * 32ull + lane;
    overlap_launches();
    float sum = 0.0f;
    if (j < n)
        for (uint64_t b = warp; b < clusters; b += 8) sum += partial[b * n + j];
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp || j >= n) return;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) total += sums[w][lane];
    db[(int64_t)j * stride] = from_f32<HALF>(total);
}

// ---- host side -----------------------------------------------------------------------------------

// Operand of a product: rows x red elements, element (r, t) at p[r * rs + t * ks].
struct Operand {
    const void* p;
    uint64_t rows, red;
    int64_t rs, ks;
    bool mn = false;
    int64_t at = -1;  // where it will lie in the call's scratch memory, if it does
};

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows of scratch matrices: whole lines of 128 bytes, which is what a row of a tensor copy's box reads (with rows a
// multiple of 16 bytes apart that read takes two).
static uint64_t padded(uint64_t elements) { return round_up(elements, 64); }

// One call's scratch memory: laid out first, then allocated at once, and the operands' copies made in one launch.
struct Source {  // of scratch memory: the caller's, or (alloc null) the stream-ordered allocator
    oztt_allocator alloc;
    void* context;
};
struct Scratch {
    int device;
    cudaStream_t st;
    Source source;
    uint64_t bytes = 0;
    uint8_t* base = nullptr;
    DevBuf buf;
    Packs packs;
    uint64_t pack_at[4];
    Scratch(int d, cudaStream_t s, Source from) : device(d), st(s), source(from), buf(s) { packs.count = 0; }
    int64_t reserve(uint64_t size) {
        const uint64_t at = bytes;
        bytes += round_up(std::max<uint64_t>(size, 1), 256);
        return (int64_t)at;
    }
    template <class T>
    T* at(int64_t offset) const {
        return reinterpret_cast<T*>(base + offset);
    }
    void place(Operand& o) const {
        if (o.at >= 0) o.p = at<uint8_t>(o.at);
    }
    void allocate() {
        if (bytes && source.alloc) {
            base = static_cast<uint8_t*>(source.alloc(source.context, bytes));
            if (!base) throw Error(OZTT_ENOMEM, "no scratch memory of " + std::to_string(bytes) + " bytes");
            if (reinterpret_cast<uintptr_t>(base) & 255) throw Error(OZTT_EINVAL, "scratch memory must start on 256 bytes");
        } else if (bytes) {
            buf.alloc(bytes);
            base = buf.as<uint8_t>();
        }
        if (!packs.count) return;
        for (uint32_t c = 0; c < packs.count; ++c) packs.of[c].dst = at<uint16_t>((int64_t)pack_at[c]);
        const unsigned grid = (unsigned)std::min<uint64_t>((packs.of[packs.count - 1].end + 7) / 8, multiprocessors(device) * 32);
        launch_overlapped(pack_kernel, dim3(grid), 256, 0, dim3(0), st, packs);
    }
    // The operand as the tensor copies can read it: as it lies (K-major, or MN-major where allowed), or a copy.
    void settle(Operand& o, bool allow_mn) {
        if (o.red == 1) o.ks = 1;  // a stride that no element uses
        if (o.rows == 1) o.rs = (int64_t)round_up(o.red, 8);
        const bool base = o.at >= 0 || aligned16(o.p);
        if (o.ks == 1 && o.rs % 8 == 0 && o.rs >= (int64_t)o.red && base) return;
        if (o.red == 1) o.ks = (int64_t)round_up(o.rows, 8);
        if (allow_mn && (o.rs == 1 || o.rows == 1) && o.ks % 8 == 0 && o.ks >= (int64_t)o.rows && base) {
            o.mn = true;
            return;
        }
        if (o.at >= 0) throw Error(OZTT_ERUNTIME, "linear: a scratch matrix that the tensor copies cannot read");
        // packed along the contiguous index, so that the copy reads and writes neighbouring elements
        const bool mn = allow_mn && o.rs == 1 && o.ks != 1;
        const uint64_t outer = mn ? o.red : o.rows, inner = mn ? o.rows : o.red, ld = padded(inner);
        const uint32_t c = packs.count++;
        packs.of[c] = {static_cast<const uint16_t*>(o.p), mn ? o.ks : o.rs, mn ? o.rs : o.ks, outer, inner, ld, nullptr,
                       (c ? packs.of[c - 1].end : 0) + outer * ((ld / 8 + PACK_GROUPS - 1) / PACK_GROUPS)};
        o.at = reserve(outer * ld * 2);
        pack_at[c] = (uint64_t)o.at;
        o.mn = mn;
        (mn ? o.ks : o.rs) = (int64_t)ld;
        (mn ? o.rs : o.ks) = 1;
    }
};

static CUtensorMap operand_map(const Operand& o, int half, uint32_t box_rows) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {std::max<uint64_t>(1, o.mn ? o.rows : o.red), std::max<uint64_t>(1, o.mn ? o.red : o.rows)};
    const cuuint64_t strides[1] = {(cuuint64_t)(o.mn ? o.ks : o.rs) * 2};
    const cuuint32_t box[2] = {64, o.mn ? BK : box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = encode_fn()(&map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                   const_cast<void*>(o.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw Error(OZTT_ERUNTIME, "cuTensorMapEncodeTiled failed for an operand of a layer product");
    return map;
}

// A product to be done: operands as the tensor copies read them, and its epilogue.
struct Task {
    Operand p, q;
    Epilogue e;
};

template <bool HALF>
static Product describe(const Task& t, uint32_t tile_p, uint32_t tile_q, uint32_t box_q, bool turned) {
    Product pr;
    const Operand &p = turned ? t.q : t.p, &q = turned ? t.p : t.q;
    pr.p = operand_map(p, HALF, BP);
    pr.q = operand_map(q, HALF, box_q);
    pr.e = t.e;
    pr.tiles_p = (uint32_t)(((turned ? t.e.rows : t.e.cols) + tile_p - 1) / tile_p);
    pr.tiles_q = (uint32_t)(((turned ? t.e.cols : t.e.rows) + tile_q - 1) / tile_q);
    pr.num_kb = (uint32_t)((t.p.red + BK - 1) / BK);
    pr.p_mn = p.mn;
    pr.q_mn = q.mn;
    // kind::f16: 32-bit sums, A and B of one type, their majors, N = tile_q, M = tile_p
    const uint32_t type = HALF ? 0u : 1u;
    pr.idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)p.mn << 15) | ((uint32_t)q.mn << 16) |
               ((tile_q >> 3) << 17) | ((tile_p >> 4) << 24);
    return pr;
}
template <bool HALF, int COUNT>
static Products<COUNT> describe_all(const Task* tasks, uint32_t tile_p, uint32_t tile_q, uint32_t box_q, bool turned) {
    Products<COUNT> ps;
    uint64_t tiles = 0;
    for (int i = 0; i < COUNT; ++i) {
        ps.of[i] = describe<HALF>(tasks[i], tile_p, tile_q, box_q, turned);
        tiles += (uint64_t)ps.of[i].tiles_p * ps.of[i].tiles_q;
    }
    if (tiles >= (1ull << 28)) throw Error(OZTT_EINVAL, "linear: problem too large");
    ps.tiles0 = ps.of[0].tiles_p * ps.of[0].tiles_q;
    ps.tiles = (uint32_t)tiles;
    return ps;
}

// How many clusters of `size` blocks of a kernel the device runs at once, a block to an SM. known: what was asked before,
// for each device and size.
using Room = std::atomic<int>[KNOWN_DEVICES][MAX_SPLIT + 1];
template <class Kernel>
static uint32_t room_for(Kernel* kernel, uint32_t smem, uint32_t size, int device, Room& known) {
    int n = device < KNOWN_DEVICES ? known[device][size].load() : 0;
    if (!n) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(size);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        OZTT_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
        if (device < KNOWN_DEVICES) known[device][size].store(n > 0 ? n : -1);
    }
    return n > 0 ? (uint32_t)n : 0;
}

template <bool HALF, int COUNT, int BQ, int STAGES, int CTAS>
static void launch_tiles(const Task* tasks, int device, cudaStream_t st) {
    constexpr uint32_t SMEM = STAGES * (P_BYTES + BQ * BK * 2) + 256 + 1024;
    static std::atomic<uint64_t> allowed{0};
    auto* kernel = product_kernel<HALF, COUNT, BQ, STAGES, CTAS>;
    allow_smem(kernel, SMEM, allowed, true);
    const Products<COUNT> ps = describe_all<HALF, COUNT>(tasks, BP, BQ, BQ, false);
    // With few tiles the reduction is shared by a cluster of CTAs, each with at least two blocks of it: by as many, up to
    // 8, as let all clusters find room in the device's parts at once, two CTAs to an SM (5 x 4480 x 8576, 35 tiles: 17.0 us
    // with 6, 23.6 with 8 in two turns); by 16 where they do with a CTA to an SM (16 x 512 x 16384: 8.7 us, 12.4 with 8;
    // 128 x 1024 x 4096, where they do not: 13.9 and 8.7).
    static_assert(CTAS == 2, "the room below is that of two CTAs to an SM");
    const uint32_t shortest = std::min(ps.of[0].num_kb, ps.of[COUNT - 1].num_kb);
    static Room known;
    const uint32_t sms = multiprocessors(device);
    const auto alone = [&](uint32_t size) { return room_for(kernel, SMEM, size, device, known); };
    uint32_t split = 1;
    if (shortest / MAX_SPLIT >= 2 && ps.tiles * MAX_SPLIT <= sms && ps.tiles <= alone(MAX_SPLIT))
        split = MAX_SPLIT;
    else
        for (uint32_t s = std::min<uint32_t>(8, shortest / 2); s > 1 && split == 1; --s)
            if (ps.tiles * s <= 2 * sms && ps.tiles <= std::max(2 * alone(s), alone((s + 1) / 2))) split = s;
    launch_overlapped(kernel, dim3(ps.tiles * split), THREADS, SMEM, dim3(split), st, ps, error_word(device));
}

template <bool HALF, int COUNT, int BQ, bool TURNED>
static void launch_pairs(const Task* tasks, int device, cudaStream_t st) {
    constexpr uint32_t SMEM = PAIR_STAGES_BYTES + FINISHERS * PATCH_BYTES + 256 + 1024;
    static std::atomic<uint64_t> allowed{0};
    auto* kernel = pair_product_kernel<HALF, COUNT, BQ, TURNED>;
    allow_smem(kernel, SMEM, allowed);
    const Products<COUNT> ps = describe_all<HALF, COUNT>(tasks, 2 * BP, BQ, BQ / 2, TURNED);
    launch_overlapped(kernel, dim3(2 * std::min(ps.tiles, multiprocessors(device) / 2)), PAIR_THREADS, SMEM, dim3(0), st, ps, error_word(device));
}

template <bool HALF, int M, bool VEC>
static void launch_few(const Task& t, int device, cudaStream_t st) {
    auto* kernel = few_rows_kernel<HALF, M, VEC>;
    const uint64_t blocks = (t.e.cols + FEW_COLS - 1) / FEW_COLS;
    // enough warps to keep the memory busy (16 on every SM), as long as each has a few accesses
    uint32_t warps = 1;
    while (warps < 8 && blocks * warps < 16 * multiprocessors(device) && t.p.red / (warps * 2) >= 512) warps *= 2;
    launch_overlapped(kernel, dim3((unsigned)blocks), warps * 32, 0, dim3(0), st, static_cast<const uint16_t*>(t.p.p), t.p.rs,
           static_cast<const uint16_t*>(t.q.p), t.q.rs, (uint32_t)t.p.red, t.e);
}

// Whether the streaming kernel takes a product, its operands as they lie: one row; or up to 4 where P would have to be
// copied for the tiles (measured, us: 1 x 4096 x 4096 7.2, by tiles 10.3; 4 x 4096 x 16384 38.3, by tiles 26.8;
// 4 x 4095 x 4097 24.7, by tiles with the copy 31.0).
static bool takes_vectors(const Task& t) {
    return aligned16(t.p.p) && t.p.rs % 8 == 0 && t.p.red % 8 == 0 && (t.q.at >= 0 || aligned16(t.q.p));
}
static bool few_rows(const Task& t) {
    return t.p.red && t.p.ks == 1 && t.q.ks == 1 && (t.e.rows == 1 || (t.e.rows <= 4 && !takes_vectors(t)));
}
// A sum of up to 8 terms without an epilogue, over columns that P has side by side, goes to the kernel for those; one of 7
// or 8 as long as the output is below 40 million elements (us, here and by tiles: 8 terms 4096 x 4096 12.1 and 12.6,
// 4480 x 8576 22.8 and 23.9, 6144 x 6144 22.5 and 21.7, 8192 x 8192 38.4 and 34.4, 12288 x 12288 77.0 and 74.5; 6 terms
// 35.2 and 35.1 at 8192 x 8192, 71.2 and 74.5 at 12288 x 12288).
static bool few_terms(const Task& t) {
    const Epilogue& e = t.e;
    return t.p.red && (t.p.red <= 6 || (t.p.red <= 8 && e.rows * e.cols < 40000000)) && t.p.mn && e.vec >= 8 &&
           e.cols % 8 == 0 && e.rows <= 65535 * 64 && e.act == OZTT_ACT_NONE && !e.bias && !e.pre.p && !e.res.p;
}
static uint64_t blocks_of(const Task& t) { return (t.p.red + BK - 1) / BK; }
static uint64_t pair_tiles_of(const Task& t) { return ((t.e.rows + 255) / 256) * ((t.e.cols + 255) / 256); }
// Two products share a launch, and its tiles' size, where one launch less counts or their tiles fill up one another's
// waves: with short sums, or few tiles that still keep every pair busy as long as the longest sum lasts. (dx + dw, us,
// one launch and two: 512 x 1024 x 1024 11 and 16, 1024^3 12.7 and 19.0, 2048^3 30.6 and 33.9, but 8192 x 1024 x 1024 58
// and 41, 8192 x 16384 x 4096 1922 and 1706: pairs that work on products of unlike length drift apart, and what one has
// read has left L2 when the next wants it.) One with few rows takes narrower tiles.
static bool together(const Task* tasks, int count, uint64_t sms) {
    if (count < 2 || std::min(tasks[0].e.rows, tasks[1].e.rows) <= 64) return false;
    const uint64_t b0 = blocks_of(tasks[0]), b1 = blocks_of(tasks[1]), t0 = pair_tiles_of(tasks[0]), t1 = pair_tiles_of(tasks[1]);
    // (up to two waves of pairs, and seven tenths of one busy all the time)
    return std::max(b0, b1) <= 24 || (t0 + t1 <= sms && t0 * b0 + t1 * b1 >= sms * 13 / 37 * std::max(b0, b1));
}

template <bool HALF>
static void launch_few_terms(const Task& t, cudaStream_t st) {
    const auto go = [&](auto* kernel, uint32_t block_rows) {
        const dim3 grid((unsigned)((t.e.cols + 255) / 256), (unsigned)((t.e.rows + block_rows - 1) / block_rows));
        launch_overlapped(kernel, grid, 256, 0, dim3(0), st, static_cast<const uint16_t*>(t.p.p), t.p.ks,
                          static_cast<const uint16_t*>(t.q.p), t.q.rs, t.q.ks, (uint32_t)t.p.red, t.e.out, t.e.rows, t.e.cols);
    };
    if (t.p.red == 1)
        go(few_terms_kernel<HALF, 1>, 8 * TERM_ROWS<1>);
    else if (t.p.red == 2)
        go(few_terms_kernel<HALF, 2>, 8 * TERM_ROWS<2>);
    else if (t.p.red <= 4)
        go(few_terms_kernel<HALF, 4>, 8 * TERM_ROWS<4>);
    else
        go(few_terms_kernel<HALF, 8>, 8 * TERM_ROWS<8>);
}

// The products of one call, out = epilogue(Q P^T), p the operand of the output's columns and q of its rows: what
// there is to do (the number returned, moved to the front), and the scratch memory for it.
static int plan(Task* tasks, int count, Scratch& scratch) {
    int live = 0;
    for (int i = 0; i < count; ++i) {
        Task t = tasks[i];
        Epilogue& e = t.e;
        if (e.rows == 0 || e.cols == 0) continue;
        if (e.rows >= (1ull << 31) || e.cols >= (1ull << 31) || t.p.red >= (1ull << 31))
            throw Error(OZTT_EINVAL, "linear: dimensions must be below 2^31");
        const auto takes = [&](int n) {
            const auto fits = [n](const View& v) {
                return !v.p || (v.cs == 1 && v.rs % n == 0 && reinterpret_cast<uintptr_t>(v.p) % (2 * n) == 0);
            };
            return fits(e.out) && fits(e.pre) && fits(e.res);
        };
        e.vec = takes(16) ? 16 : takes(8) ? 8 : takes(4) ? 4 : 1;
        tasks[live++] = t;
    }
    for (int i = 0; i < live; ++i) {
        Task& t = tasks[i];
        if (few_rows(t)) continue;
        if (t.p.red) {
            scratch.settle(t.p, true);
            scratch.settle(t.q, t.e.rows > 32 || t.q.at >= 0);  // (dz is made after the copies, so never copied itself)
        } else {  // nothing is read: any valid address and stride for the tensor maps
            t.p.at = t.q.at = scratch.reserve(256);
            t.p.rs = t.q.rs = 8;
            t.p.ks = t.q.ks = 1;
            t.p.rows = t.q.rows = 1;
        }
    }
    return live;
}

template <bool HALF>
static void run(Task* tasks, int count, const Scratch& scratch, cudaStream_t st) {
    if (!count) return;
    const uint32_t sms = multiprocessors(scratch.device);
    if (count == 2 && !together(tasks, count, sms)) {
        run<HALF>(tasks, 1, scratch, st);
        run<HALF>(tasks + 1, 1, scratch, st);
        return;
    }
    if (count == 2 && tasks[1].p.red > tasks[0].p.red) std::swap(tasks[0], tasks[1]);  // the longest tiles first
    uint64_t rows = 0, pair_tiles = 0, tiles = 0, blocks = 0;
    bool empty = false, wide = true, narrow = true;  // boxes of less than 64 rows have no MN-major form
    for (int i = 0; i < count; ++i) {
        scratch.place(tasks[i].p);
        scratch.place(tasks[i].q);
        const Epilogue& e = tasks[i].e;
        rows = std::max(rows, e.rows);
        pair_tiles += pair_tiles_of(tasks[i]);
        tiles += ((e.rows + 127) / 128) * ((e.cols + 127) / 128);
        blocks = std::max(blocks, blocks_of(tasks[i]));
        empty = empty || tasks[i].p.red == 0;
        wide = wide && e.vec >= 16 && !e.res.p;
        narrow = narrow && !tasks[i].q.mn;
    }
    if (count == 1 && few_rows(tasks[0])) {
        const Task& t = tasks[0];
        const auto go = rows == 1   ? (takes_vectors(t) ? launch_few<HALF, 1, true> : launch_few<HALF, 1, false>)
                        : rows == 2 ? launch_few<HALF, 2, false>
                        : rows == 3 ? launch_few<HALF, 3, false>
                                    : launch_few<HALF, 4, false>;
        return go(t, scratch.device, st);
    }
    if (count == 1 && few_terms(tasks[0])) return launch_few_terms<HALF>(tasks[0], st);
    // Which tiles, by what was measured (us, BF16, single products):
    //   output      sum    64 rows  128 rows  pairs
    //   512x4096    1024     12.1     13.3     11.5      pairs from half the device's SMs on, and from a third where
    //   512x4096    4096     26.8     23.7     27.3      the sum is short (up to 24 blocks): their tiles need a third
    //   1024x4096   4096     52.3     37.7     28.9      of the bytes from L2, but leave more SMs idle when few
    //   512x2048    1024      9.8     10.5     11.2      64 rows where 128 would leave most SMs idle or the sum is
    //   256x2048    4096     12.0     13.7     25.6      short, since the CTAs of a split sum join sooner
    //   512x2048    4096     17.2     15.9     26.1
    if (!empty && rows > 128 && (pair_tiles >= sms / 4 || (pair_tiles >= sms * 6 / 37 && blocks <= 24))) {
        if (wide)
            count == 2 ? launch_pairs<HALF, 2, 256, true>(tasks, scratch.device, st) : launch_pairs<HALF, 1, 256, true>(tasks, scratch.device, st);
        else
            count == 2 ? launch_pairs<HALF, 2, 256, false>(tasks, scratch.device, st) : launch_pairs<HALF, 1, 256, false>(tasks, scratch.device, st);
    } else if (rows <= 16 && narrow)
        launch_tiles<HALF, 1, 16, 6, 2>(tasks, scratch.device, st);
    else if (rows <= 32 && narrow)
        launch_tiles<HALF, 1, 32, 5, 2>(tasks, scratch.device, st);
    else if (rows <= 64 || tiles <= 32 || blocks <= 24)
        count == 2 ? launch_tiles<HALF, 2, 64, 4, 2>(tasks, scratch.device, st) : launch_tiles<HALF, 1, 64, 4, 2>(tasks, scratch.device, st);
    else
        count == 2 ? launch_tiles<HALF, 2, 128, 3, 2>(tasks, scratch.device, st) : launch_tiles<HALF, 1, 128, 3, 2>(tasks, scratch.device, st);
}

template <bool HALF>
static auto dz_variant(bool vec, int act) {
    switch (act) {
#define OZTT_CASE(A) \
    case A: return vec ? dz_kernel<HALF, true, A> : dz_kernel<HALF, false, A>
        OZTT_CASE(OZTT_ACT_RELU);
        OZTT_CASE(OZTT_ACT_GELU);
        OZTT_CASE(OZTT_ACT_GELU_TANH);
        OZTT_CASE(OZTT_ACT_SILU);
#undef OZTT_CASE
        default: return vec ? dz_kernel<HALF, true, OZTT_ACT_NONE> : dz_kernel<HALF, false, OZTT_ACT_NONE>;
    }
}

static View view(const oztt_view& v) { return {v.data, v.row_stride, v.col_stride}; }

static bool half_of(int32_t format, const char* who) {
    if (format == OZTT_FMT_BF16) return false;
    if (format == OZTT_FMT_FP16) return true;
    throw Error(OZTT_EINVAL, std::string(who) + ": the format must be BF16 or FP16");
}
static void check_act(int32_t act, const char* who) {
    if (act < OZTT_ACT_NONE || act > OZTT_ACT_SILU) throw Error(OZTT_EINVAL, std::string(who) + ": unknown activation");
}
// An output of rows x cols that two of its elements would not share.
static void check_output(const oztt_view& v, uint64_t rows, uint64_t cols, const char* what) {
    if (v.data && ((rows > 1 && v.row_stride == 0) || (cols > 1 && v.col_stride == 0)))
        throw Error(OZTT_EINVAL, std::string(what) + ": an output's strides must not be zero");
}
static void check_view(const oztt_view& v, bool needed, const char* what) {
    if (!v.data) {
        if (needed) throw Error(OZTT_EINVAL, std::string(what) + " is missing");
        return;
    }
    if (reinterpret_cast<uintptr_t>(v.data) & 1) throw Error(OZTT_EINVAL, std::string(what) + " must be 2-byte aligned");
    if (v.row_stride < 0 || v.col_stride < 0) throw Error(OZTT_EINVAL, std::string(what) + ": strides must not be negative");
}

template <bool HALF>
static void forward(int device, const oztt_linear& a, Source source, cudaStream_t st) {
    check_act(a.activation, "linear");
    const bool some = a.m && a.n, sum = some && a.k;
    check_view(a.x, sum, "linear: x");
    check_view(a.w, sum, "linear: w");
    check_view(a.y, some, "linear: y");
    check_view(a.bias, false, "linear: bias");
    check_view(a.residual, false, "linear: residual");
    check_view(a.pre, false, "linear: pre");
    check_output(a.y, a.m, a.n, "linear: y");
    check_output(a.pre, a.m, a.n, "linear: pre");
    if (!some) return;
    DeviceScope scope(device);
    check_earlier_calls(device);
    Epilogue e{};
    e.rows = a.m;
    e.cols = a.n;
    e.out = view(a.y);
    e.pre = view(a.pre);
    e.res = view(a.residual);
    e.bias = a.bias.data;
    e.bias_stride = a.bias.col_stride;
    e.act = a.activation;
    Task t{{a.w.data, a.n, a.k, a.w.row_stride, a.w.col_stride}, {a.x.data, a.m, a.k, a.x.row_stride, a.x.col_stride}, e};
    Scratch scratch(device, st, source);
    const int count = plan(&t, 1, scratch);
    scratch.allocate();
    run<HALF>(&t, count, scratch, st);
}

template <bool HALF>
static void backward(int device, const oztt_linear_grad& a, Source source, cudaStream_t st) {
    check_act(a.activation, "linear_backward");
    const bool act = a.activation != OZTT_ACT_NONE, mn = a.m && a.n;
    check_view(a.dy, mn, "linear_backward: dy");
    check_view(a.pre, mn && act, "linear_backward: pre (the sums before the activation)");
    check_view(a.x, a.dw.data && a.m && a.k, "linear_backward: x");
    check_view(a.w, a.dx.data && a.n && a.k, "linear_backward: w");
    check_view(a.dx, false, "linear_backward: dx");
    check_view(a.dw, false, "linear_backward: dw");
    check_view(a.db, false, "linear_backward: db");
    check_output(a.dx, a.m, a.k, "linear_backward: dx");
    check_output(a.dw, a.n, a.k, "linear_backward: dw");
    check_output(a.db, 1, a.n, "linear_backward: db");
    DeviceScope scope(device);
    check_earlier_calls(device);
    const View dy = view(a.dy), z = act ? view(a.pre) : View{};
    const auto fits = [](const View& v) { return !v.p || (v.cs == 1 && v.rs % 8 == 0 && aligned16(v.p)); };
    const bool products = mn && ((a.dx.data && a.k) || (a.dw.data && a.k));
    // dz is written where an activation makes it, or where the products cannot read dy as it lies: one pass for both
    // of them and for db
    const bool write = products && (act || !fits(dy)), sum = mn && a.db.data;
    // clusters of up to 8 blocks, one below the other, as many as spread over the device; at least 16 rows a block,
    // and up to 128 rows a block no second cluster, nor the launch that joins the clusters' sums
    const uint64_t ld = padded(a.n), strips = (a.n + DZ_COLS - 1) / DZ_COLS, most = (a.m + DZ_ROWS - 1) / DZ_ROWS;
    uint32_t cluster = 1;
    while (cluster < DZ_CLUSTER && cluster * 2 <= most) cluster *= 2;
    uint64_t clusters = 1;
    if (mn && most > 8 * cluster) clusters = std::max<uint64_t>(1, std::min(most / cluster, multiprocessors(device) * 4 / (strips * cluster)));
    if (strips >= (1ull << 31)) throw Error(OZTT_EINVAL, "linear_backward: problem too large");

    Scratch scratch(device, st, source);
    const int64_t dz_at = write ? scratch.reserve(a.m * ld * 2) : -1;
    const int64_t sums_at = sum && clusters > 1 ? scratch.reserve(clusters * a.n * 4) : -1;
    const View dz = write ? View{nullptr, (int64_t)ld, 1} : dy;
    Task tasks[2];
    int count = 0;
    Epilogue e{};
    e.act = OZTT_ACT_NONE;
    if (a.dx.data) {  // dx[i][t] = sum_n dz[i][n] w[n][t]
        e.rows = a.m;
        e.cols = a.k;
        e.out = view(a.dx);
        tasks[count++] = {{a.w.data, a.k, a.n, a.w.col_stride, a.w.row_stride}, {dz.p, a.m, a.n, dz.rs, dz.cs, false, dz_at}, e};
    }
    if (a.dw.data) {  // dw[n][t] = sum_i dz[i][n] x[i][t]
        e.rows = a.n;
        e.cols = a.k;
        e.out = view(a.dw);
        tasks[count++] = {{a.x.data, a.k, a.m, a.x.col_stride, a.x.row_stride}, {dz.p, a.n, a.m, dz.cs, dz.rs, false, dz_at}, e};
    }
    count = plan(tasks, count, scratch);
    scratch.allocate();
    auto* db = static_cast<uint16_t*>(a.db.data);
    if (write || sum)
        launch_overlapped(dz_variant<HALF>(fits(dy) && fits(z) && a.n % 8 == 0, a.activation),
                          dim3((unsigned)strips, (unsigned)(clusters * cluster)), 256, 0, dim3(1, cluster, 1), st, dy, z, a.m,
                          a.n, round_up((a.m + clusters * cluster - 1) / (clusters * cluster), DZ_ROWS),
                          write ? scratch.at<uint16_t>(dz_at) : nullptr, ld, sums_at >= 0 ? scratch.at<float>(sums_at) : nullptr,
                          sum && sums_at < 0 ? db : nullptr, a.db.col_stride);
    if (db && a.n && (sums_at >= 0 || !a.m))  // without rows: zeros
        launch_overlapped(db_kernel<HALF>, dim3((unsigned)((a.n + 31) / 32)), 256, 0, dim3(0), st,
                          a.m ? scratch.at<float>(sums_at) : nullptr, a.m ? clusters : 0, a.n, db, a.db.col_stride);
    run<HALF>(tasks, count, scratch, st);
}

}  // namespace layer
}  // namespace oztt

extern "C" int oztt_linear_forward_in(int device_id, const oztt_linear* args, oztt_allocator alloc, void* context,
                                      void* stream, char* err, size_t errlen) {
    return oztt::guarded(err, errlen, [&] {
        if (!args) throw oztt::Error(OZTT_EINVAL, "linear: no arguments");
        const auto run = oztt::layer::half_of(args->format, "linear") ? oztt::layer::forward<true> : oztt::layer::forward<false>;
        run(device_id, *args, {alloc, context}, reinterpret_cast<cudaStream_t>(stream));
    });
}
extern "C" int oztt_linear_forward(int device_id, const oztt_linear* args, void* stream, char* err, size_t errlen) {
    return oztt_linear_forward_in(device_id, args, nullptr, nullptr, stream, err, errlen);
}

extern "C" int oztt_linear_backward_in(int device_id, const oztt_linear_grad* args, oztt_allocator alloc, void* context,
                                       void* stream, char* err, size_t errlen) {
    return oztt::guarded(err, errlen, [&] {
        if (!args) throw oztt::Error(OZTT_EINVAL, "linear_backward: no arguments");
        const auto run = oztt::layer::half_of(args->format, "linear_backward") ? oztt::layer::backward<true> : oztt::layer::backward<false>;
        run(device_id, *args, {alloc, context}, reinterpret_cast<cudaStream_t>(stream));
    });
}
extern "C" int oztt_linear_backward(int device_id, const oztt_linear_grad* args, void* stream, char* err,
                                    size_t errlen) {
    return oztt_linear_backward_in(device_id, args, nullptr, nullptr, stream, err, errlen);
}

extern "C" int oztt_layer_status(int device_id, char* err, size_t errlen) {
    return oztt::guarded(err, errlen, [&] { oztt::check_earlier_calls(device_id); });
}

// Puts a wait's error code where a kernel would have put it, for the test of how the next call reports it.
extern "C" int oztt_test_device_error(int device_id, int32_t code, char* err, size_t errlen);
extern "C" int oztt_test_linear_error(int32_t code, char* err, size_t errlen) { return oztt_test_device_error(0, code, err, errlen); }
extern "C" int oztt_test_device_error(int device_id, int32_t code, char* err, size_t errlen) {
    return oztt::guarded(err, errlen, [&] { *oztt::error_word(device_id) = code; });
}
