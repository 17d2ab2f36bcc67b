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

#include "device_scope.cuh"
#include "runtime.cuh"
#include "tensor_core.cuh"

namespace oztt {
namespace layer {

using namespace gemm;

constexpr uint32_t BP = 128;            // rows of P in a tile
constexpr uint32_t BK = 64;             // reduction elements per stage: 128 bytes, one swizzle row
constexpr uint32_t UK = 16;             // reduction elements of one tcgen05.mma
constexpr uint32_t P_BYTES = BP * BK * 2;
constexpr uint32_t THREADS = 192;       // warp 0 loads, warp 1 issues the products, warps 2-5 read the sums
constexpr uint32_t MN_BOX = 64;         // rows of one MN-major box: 128 bytes
constexpr uint32_t MN_BOX_BYTES = MN_BOX * BK * 2;
constexpr uint32_t MAX_SPLIT = 8;       // CTAs of a cluster that share one tile's reduction

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
    int32_t act, half;                   // OZTT_ACT_*; 1: FP16, 0: BF16
    int32_t vec;                         // 4 columns at a time: unit column strides and 8-byte aligned rows
};

// ---- activations in 32 bits ----------------------------------------------------------------------
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }
constexpr float kTanhScale = 0.7978845608028654f;  // sqrt(2/pi)
constexpr float kTanhCube = 0.044715f;

// gelu_tanh is z (1 + tanh u) / 2 = z sigmoid(2u): no cancellation in the lower tail.
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case OZTT_ACT_RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case OZTT_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case OZTT_ACT_GELU_TANH: {
            const float u = kTanhScale * (z + kTanhCube * z * z * z);
            return z * sigmoid(2.0f * u);
        }
        case OZTT_ACT_SILU: return z * sigmoid(z);
        default: return z;
    }
}
__device__ __forceinline__ float slope(float z, int act) {
    switch (act) {
        case OZTT_ACT_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
        case OZTT_ACT_GELU:
            return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * __expf(-0.5f * z * z) * 0.3989422804014327f;
        case OZTT_ACT_GELU_TANH: {
            const float s = sigmoid(2.0f * kTanhScale * (z + kTanhCube * z * z * z));
            return s + 2.0f * z * s * (1.0f - s) * kTanhScale * (1.0f + 3.0f * kTanhCube * z * z);
        }
        case OZTT_ACT_SILU: {
            const float s = sigmoid(z);
            return s * (1.0f + z * (1.0f - s));
        }
        default: return 1.0f;
    }
}

__device__ __forceinline__ float to_f32(uint16_t v, int half) {
    return half ? __half2float(__ushort_as_half(v)) : __uint_as_float((uint32_t)v << 16);
}
__device__ __forceinline__ uint16_t from_f32(float v, int half) {
    return half ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// ---- the tile product ----------------------------------------------------------------------------
struct Product {
    uint32_t tiles_p, num_kb;            // tiles along the output's columns; 64-element blocks of the reduction
    uint32_t idesc;
    uint32_t p_mn, q_mn;                 // 1: the operand is MN-major
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

// Bias, activation, residual and the stores of four neighbouring columns j .. j+3 of row i.
__device__ __forceinline__ void finish4(const Epilogue& e, uint64_t i, uint64_t j, float4 acc, const float (&bias)[4]) {
    float z[4] = {acc.x + bias[0], acc.y + bias[1], acc.z + bias[2], acc.w + bias[3]};
    const bool whole = e.vec && j + 3 < e.cols;
    uint16_t* out = reinterpret_cast<uint16_t*>(e.out.p) + (int64_t)i * e.out.rs + (int64_t)j * e.out.cs;
    uint16_t* pre = reinterpret_cast<uint16_t*>(e.pre.p) + (int64_t)i * e.pre.rs + (int64_t)j * e.pre.cs;
    const uint16_t* res = reinterpret_cast<const uint16_t*>(e.res.p) + (int64_t)i * e.res.rs + (int64_t)j * e.res.cs;
    if (whole) {
        float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (e.res.p) {
            const ushort4 v = *reinterpret_cast<const ushort4*>(res);
            r[0] = to_f32(v.x, e.half), r[1] = to_f32(v.y, e.half), r[2] = to_f32(v.z, e.half), r[3] = to_f32(v.w, e.half);
        }
        if (e.pre.p)
            *reinterpret_cast<ushort4*>(pre) = make_ushort4(from_f32(z[0], e.half), from_f32(z[1], e.half),
                                                            from_f32(z[2], e.half), from_f32(z[3], e.half));
#pragma unroll
        for (int q = 0; q < 4; ++q) z[q] = activate(z[q], e.act) + r[q];
        *reinterpret_cast<ushort4*>(out) = make_ushort4(from_f32(z[0], e.half), from_f32(z[1], e.half),
                                                        from_f32(z[2], e.half), from_f32(z[3], e.half));
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (j + q >= e.cols) continue;
            if (e.pre.p) pre[q * e.pre.cs] = from_f32(z[q], e.half);
            float y = activate(z[q], e.act);
            if (e.res.p) y += to_f32(res[q * e.res.cs], e.half);
            out[q * e.out.cs] = from_f32(y, e.half);
        }
    }
}

// One tile of 128 output columns by BQ output rows per cluster; the CTAs of a cluster share the reduction: each
// sums its stretch of it in tensor memory and lays the 32-bit sums down in its own shared memory (where the
// operand stages were), then each finishes its share of the rows, adding the stretches in the cluster's order
// through distributed shared memory, so the result does not depend on timing.
template <int BQ, int STAGES, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS)
    product_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ, const Product pr,
                   const Epilogue e, int* err) {
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
    const uint32_t tile = blockIdx.x / split;
    const uint32_t tp = tile % pr.tiles_p, tq = tile / pr.tiles_p;
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
                load_operand(&tmP, sp, full_bar + stage, (int32_t)(tp * BP), (int32_t)(kb * BK), BP, pr.p_mn);
                load_operand(&tmQ, sp + P_BYTES, full_bar + stage, (int32_t)(tq * BQ), (int32_t)(kb * BK), BQ, pr.q_mn);
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
            const uint32_t step_p = pr.p_mn ? UK * 128u : UK * 2u, step_q = pr.q_mn ? UK * 128u : UK * 2u;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(full_bar + stage, phase, abort_flag, err, ERR_WAIT_MMA_FULL)) break;
                tc_fence_after();
                const uint32_t sp = smem_u32(smem + stage * STAGE_BYTES), sq = sp + P_BYTES;
#pragma unroll
                for (uint32_t k = 0; k < BK / UK; ++k)
                    umma_16(tmem_base, operand_desc(sp + k * step_p, pr.p_mn), operand_desc(sq + k * step_q, pr.q_mn),
                            pr.idesc, kb != kb0 || k != 0);
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

    const uint64_t j = (uint64_t)tp * BP + lane * 4;
    if (j < e.cols) {
        float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (e.bias) {
            const uint16_t* b = reinterpret_cast<const uint16_t*>(e.bias);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (j + q < e.cols) bias[q] = to_f32(b[(int64_t)(j + q) * e.bias_stride], e.half);
        }
        const uint32_t r0 = BQ * rank / split, r1 = BQ * (rank + 1) / split;
        const uint32_t mine = smem_u32(smem) + lane * 16;
        for (uint32_t r = r0 + warp; r < r1; r += THREADS / 32) {
            const uint64_t i = (uint64_t)tq * BQ + r;
            if (i >= e.rows) break;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (split == 1) {
                acc = *reinterpret_cast<const float4*>(smem + r * (BP * 4) + lane * 16);
            } else {
                for (uint32_t c = 0; c < split; ++c) {
                    const float4 v = ld_cluster_f4(map_to(mine + r * (BP * 4), c));
                    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
                }
            }
            finish4(e, i, j, acc, bias);
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

// ---- passes over memory --------------------------------------------------------------------------

// dst[o][i] = src[o * so + i * si], rows ld apart (ld a multiple of 8, zero beyond `inner`): operands whose base
// or rows do not start on 16 bytes, which the tensor copies cannot read.
__global__ void __launch_bounds__(256) pack_kernel(const uint16_t* __restrict__ src, int64_t so, int64_t si,
                                                   uint64_t outer, uint64_t inner, uint16_t* __restrict__ dst,
                                                   uint64_t ld) {
    const uint64_t per_row = ld / 8, count = outer * per_row;
    for (uint64_t t = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; t < count; t += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t o = t / per_row, i = (t - o * per_row) * 8;
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint64_t i0 = i + 2 * q;
            const uint32_t lo = i0 < inner ? src[(int64_t)o * so + (int64_t)i0 * si] : 0;
            const uint32_t hi = i0 + 1 < inner ? src[(int64_t)o * so + (int64_t)(i0 + 1) * si] : 0;
            w[q] = lo | (hi << 16);
        }
        *reinterpret_cast<uint4*>(dst + o * ld + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// dz = dy * act'(z) into dz (rows ld apart; may be null), and the sums of its columns over this block's rows in
// 32 bits into partial[block row][n] (may be null). Block (x, y): 32 columns each of 8 warps by ROWS rows.
constexpr uint32_t DZ_ROWS = 64;
__global__ void __launch_bounds__(256) dz_kernel(View dy, View z, uint64_t m, uint64_t n, int act, int half,
                                                 uint16_t* __restrict__ dz, uint64_t ld, float* __restrict__ partial) {
    const uint64_t j = blockIdx.x * 256ull + threadIdx.x;
    const uint64_t i0 = blockIdx.y * (uint64_t)DZ_ROWS, i1 = min(i0 + DZ_ROWS, m);
    if (j >= n) return;
    const uint16_t* gy = reinterpret_cast<const uint16_t*>(dy.p) + (int64_t)j * dy.cs;
    const uint16_t* gz = reinterpret_cast<const uint16_t*>(z.p) + (int64_t)j * z.cs;
    float sum = 0.0f;
    for (uint64_t i = i0; i < i1; ++i) {
        float v = to_f32(gy[(int64_t)i * dy.rs], half);
        if (act != OZTT_ACT_NONE) v *= slope(to_f32(gz[(int64_t)i * z.rs], half), act);
        sum += v;
        if (dz) dz[i * ld + j] = from_f32(v, half);
    }
    if (partial) partial[blockIdx.y * n + j] = sum;
}

__global__ void __launch_bounds__(256) db_kernel(const float* __restrict__ partial, uint64_t blocks, uint64_t n,
                                                 int half, uint16_t* __restrict__ db, int64_t stride) {
    const uint64_t j = blockIdx.x * 256ull + threadIdx.x;
    if (j >= n) return;
    float sum = 0.0f;
    for (uint64_t b = 0; b < blocks; ++b) sum += partial[b * n + j];
    db[(int64_t)j * stride] = from_f32(sum, half);
}

// ---- host side -----------------------------------------------------------------------------------

// The word that a kernel's bounded wait writes when it gives up: host memory that every device reaches, looked
// at by the next call, since these calls do not wait for their kernels.
static int* error_word() {
    static int* word = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        if (cudaHostAlloc(&word, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped) == cudaSuccess)
            *word = 0;
        else
            word = nullptr, cudaGetLastError();
    });
    if (!word) throw Error(OZTT_ERUNTIME, "linear: no pinned host memory for the error word");
    return word;
}
static void check_earlier_calls() {
    volatile int* w = error_word();
    if (const int code = *w) {
        *w = 0;
        throw Error(OZTT_ERUNTIME, "linear: a kernel of an earlier call gave up waiting (code " + std::to_string(code) +
                                       "); that call's outputs are not valid");
    }
}

// Operand of a product: rows x red elements, element (r, t) at p[r * rs + t * ks].
struct Operand {
    const void* p;
    uint64_t rows, red;
    int64_t rs, ks;
    bool mn = false;
};

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The operand as the tensor copies can read it: as it lies (K-major, or MN-major where allowed), or packed.
static void settle(Operand& o, bool allow_mn, DevBuf& buf, cudaStream_t st) {
    if (o.red == 1) o.ks = 1;  // a stride that no element uses
    if (o.rows == 1) o.rs = (int64_t)round_up(o.red, 8);
    const bool base = aligned16(o.p);
    if (o.ks == 1 && o.rs % 8 == 0 && o.rs >= (int64_t)o.red && base) return;
    if (o.red == 1) o.ks = (int64_t)round_up(o.rows, 8);
    if (allow_mn && o.rs == 1 && o.ks % 8 == 0 && o.ks >= (int64_t)o.rows && base) {
        o.mn = true;
        return;
    }
    // packed along the contiguous index, so that the copy reads and writes neighbouring elements
    const bool mn = allow_mn && o.rs == 1 && o.ks != 1;
    const uint64_t outer = mn ? o.red : o.rows, inner = mn ? o.rows : o.red, ld = round_up(inner, 8);
    buf.alloc(outer * ld * 2);
    const unsigned grid = (unsigned)std::min<uint64_t>((outer * (ld / 8) + 255) / 256, 148 * 16);
    pack_kernel<<<grid, 256, 0, st>>>(static_cast<const uint16_t*>(o.p), mn ? o.ks : o.rs, mn ? o.rs : o.ks, outer,
                                      inner, buf.as<uint16_t>(), ld);
    OZTT_CUDA(cudaGetLastError());
    o.p = buf.p;
    o.mn = mn;
    (mn ? o.ks : o.rs) = (int64_t)ld;
    (mn ? o.rs : o.ks) = 1;
}

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

template <int BQ, int STAGES, int CTAS>
static void launch_tile(const Operand& p, const Operand& q, const Epilogue& e, cudaStream_t st) {
    constexpr uint32_t SMEM = STAGES * (P_BYTES + BQ * BK * 2) + 256 + 1024;
    auto* kernel = product_kernel<BQ, STAGES, CTAS>;
    Product pr;
    pr.tiles_p = (uint32_t)((e.cols + BP - 1) / BP);
    pr.num_kb = (uint32_t)((p.red + BK - 1) / BK);
    pr.p_mn = p.mn;
    pr.q_mn = q.mn;
    // kind::f16: 32-bit sums, A and B of one type, their majors, N = BQ, M = 128
    const uint32_t type = e.half ? 0u : 1u;
    pr.idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)p.mn << 15) | ((uint32_t)q.mn << 16) |
               ((BQ >> 3) << 17) | ((BP >> 4) << 24);
    const uint64_t tiles = (uint64_t)pr.tiles_p * ((e.rows + BQ - 1) / BQ);
    // With few tiles the reduction is shared by up to 8 CTAs, as long as the CTAs are resident at once and each
    // keeps at least four blocks of it.
    uint32_t split = 1;
    while (split < MAX_SPLIT && tiles * split * 2 <= 148 * CTAS && pr.num_kb / (split * 2) >= 4) split *= 2;
    if (tiles * split >= (1ull << 31)) throw Error(OZTT_EINVAL, "linear: problem too large");
    const CUtensorMap tp = operand_map(p, e.half, BP), tq = operand_map(q, e.half, BQ);
    OZTT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * split), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    OZTT_CUDA(cudaLaunchKernelEx(&cfg, kernel, tp, tq, pr, e, error_word()));
}

// out = epilogue(Q P^T): p the operand of the output's columns, q of its rows.
static void product(Operand p, Operand q, Epilogue e, cudaStream_t st) {
    if (e.rows == 0 || e.cols == 0) return;
    if (e.rows >= (1ull << 31) || e.cols >= (1ull << 31) || p.red >= (1ull << 31))
        throw Error(OZTT_EINVAL, "linear: dimensions must be below 2^31");
    DevBuf bp(st), bq(st);
    if (p.red) {
        settle(p, true, bp, st);
        settle(q, e.rows > 32, bq, st);
    } else {  // nothing is read: any valid address and stride for the tensor maps
        bp.alloc(256);
        p.p = q.p = bp.p;
        p.rs = q.rs = 8;
        p.ks = q.ks = 1;
        p.rows = q.rows = 1;
    }
    const auto fits = [](const View& v) { return !v.p || (v.cs == 1 && v.rs % 4 == 0 && (reinterpret_cast<uintptr_t>(v.p) & 7) == 0); };
    e.vec = fits(e.out) && fits(e.pre) && fits(e.res);
    if (e.rows <= 16)
        launch_tile<16, 6, 2>(p, q, e, st);
    else if (e.rows <= 32)
        launch_tile<32, 5, 2>(p, q, e, st);
    else if (e.rows <= 64)
        launch_tile<64, 4, 2>(p, q, e, st);
    else
        launch_tile<128, 3, 2>(p, q, e, st);
}

static View view(const oztt_view& v) { return {v.data, v.row_stride, v.col_stride}; }

static int half_of(int32_t format, const char* who) {
    if (format == OZTT_FMT_BF16) return 0;
    if (format == OZTT_FMT_FP16) return 1;
    throw Error(OZTT_EINVAL, std::string(who) + ": the format must be BF16 or FP16");
}
static void check_act(int32_t act, const char* who) {
    if (act < OZTT_ACT_NONE || act > OZTT_ACT_SILU) throw Error(OZTT_EINVAL, std::string(who) + ": unknown activation");
}
static void check_view(const oztt_view& v, bool needed, const char* what) {
    if (!v.data) {
        if (needed) throw Error(OZTT_EINVAL, std::string(what) + " is missing");
        return;
    }
    if (reinterpret_cast<uintptr_t>(v.data) & 1) throw Error(OZTT_EINVAL, std::string(what) + " must be 2-byte aligned");
    if (v.row_stride < 0 || v.col_stride < 0) throw Error(OZTT_EINVAL, std::string(what) + ": strides must not be negative");
}

static void forward(int device, const oztt_linear& a, cudaStream_t st) {
    const int half = half_of(a.format, "linear");
    check_act(a.activation, "linear");
    const bool some = a.m && a.n, sum = some && a.k;
    check_view(a.x, sum, "linear: x");
    check_view(a.w, sum, "linear: w");
    check_view(a.y, some, "linear: y");
    check_view(a.bias, false, "linear: bias");
    check_view(a.residual, false, "linear: residual");
    check_view(a.pre, false, "linear: pre");
    if (!some) return;
    DeviceScope scope(device);
    check_earlier_calls();
    Epilogue e{};
    e.rows = a.m;
    e.cols = a.n;
    e.out = view(a.y);
    e.pre = view(a.pre);
    e.res = view(a.residual);
    e.bias = a.bias.data;
    e.bias_stride = a.bias.col_stride;
    e.act = a.activation;
    e.half = half;
    product({a.w.data, a.n, a.k, a.w.row_stride, a.w.col_stride}, {a.x.data, a.m, a.k, a.x.row_stride, a.x.col_stride},
            e, st);
}

static void backward(int device, const oztt_linear_grad& a, cudaStream_t st) {
    const int half = half_of(a.format, "linear_backward");
    check_act(a.activation, "linear_backward");
    const bool act = a.activation != OZTT_ACT_NONE, mn = a.m && a.n;
    check_view(a.dy, mn, "linear_backward: dy");
    check_view(a.pre, mn && act, "linear_backward: pre (the sums before the activation)");
    check_view(a.x, a.dw.data && a.m && a.k, "linear_backward: x");
    check_view(a.w, a.dx.data && a.n && a.k, "linear_backward: w");
    check_view(a.dx, false, "linear_backward: dx");
    check_view(a.dw, false, "linear_backward: dw");
    check_view(a.db, false, "linear_backward: db");
    DeviceScope scope(device);
    check_earlier_calls();
    View dz = view(a.dy);
    DevBuf dz_buf(st), sums(st);
    const bool products = (a.dx.data && a.m && a.k) || (a.dw.data && a.n && a.k);
    if (mn && ((act && products) || a.db.data)) {
        const uint64_t ld = round_up(a.n, 8), blocks = (a.m + DZ_ROWS - 1) / DZ_ROWS;
        if (blocks > 65535 * 32768ull) throw Error(OZTT_EINVAL, "linear_backward: problem too large");
        const bool store = act && products;
        if (store) dz_buf.alloc(a.m * ld * 2);
        if (a.db.data) sums.alloc(blocks * a.n * 4);
        for (uint64_t b0 = 0; b0 < blocks; b0 += 65535) {  // the grid's limit of block rows
            const uint64_t nb = std::min<uint64_t>(65535, blocks - b0), i0 = b0 * DZ_ROWS;
            const auto below = [&](View v) { return View{v.p ? static_cast<uint16_t*>(v.p) + (int64_t)i0 * v.rs : nullptr, v.rs, v.cs}; };
            dz_kernel<<<dim3((unsigned)((a.n + 255) / 256), (unsigned)nb), 256, 0, st>>>(
                below(dz), below(view(a.pre)), a.m - i0, a.n, a.activation, half,
                store ? dz_buf.as<uint16_t>() + i0 * ld : nullptr, ld, a.db.data ? sums.as<float>() + b0 * a.n : nullptr);
            OZTT_CUDA(cudaGetLastError());
        }
        if (store) dz = {dz_buf.p, (int64_t)ld, 1};
    }
    if (a.db.data && a.n) {
        const uint64_t blocks = (a.m + DZ_ROWS - 1) / DZ_ROWS;
        db_kernel<<<(unsigned)((a.n + 255) / 256), 256, 0, st>>>(sums.as<float>(), blocks, a.n, half,
                                                                static_cast<uint16_t*>(a.db.data), a.db.col_stride);
        OZTT_CUDA(cudaGetLastError());
    }
    Epilogue e{};
    e.half = half;
    e.act = OZTT_ACT_NONE;
    if (a.dx.data) {  // dx[i][t] = sum_n dz[i][n] w[n][t]
        e.rows = a.m;
        e.cols = a.k;
        e.out = view(a.dx);
        product({a.w.data, a.k, a.n, a.w.col_stride, a.w.row_stride}, {dz.p, a.m, a.n, dz.rs, dz.cs}, e, st);
    }
    if (a.dw.data) {  // dw[n][t] = sum_i dz[i][n] x[i][t]
        e.rows = a.n;
        e.cols = a.k;
        e.out = view(a.dw);
        product({a.x.data, a.k, a.m, a.x.col_stride, a.x.row_stride}, {dz.p, a.n, a.m, dz.cs, dz.rs}, e, st);
    }
}

}  // namespace layer
}  // namespace oztt

extern "C" int oztt_linear_forward(int device_id, const oztt_linear* args, void* stream, char* err, size_t errlen) {
    return oztt::guarded(err, errlen, [&] {
        if (!args) throw oztt::Error(OZTT_EINVAL, "linear: no arguments");
        oztt::layer::forward(device_id, *args, reinterpret_cast<cudaStream_t>(stream));
    });
}

extern "C" int oztt_linear_backward(int device_id, const oztt_linear_grad* args, void* stream, char* err,
                                    size_t errlen) {
    return oztt::guarded(err, errlen, [&] {
        if (!args) throw oztt::Error(OZTT_EINVAL, "linear_backward: no arguments");
        oztt::layer::backward(device_id, *args, reinterpret_cast<cudaStream_t>(stream));
    });
}
