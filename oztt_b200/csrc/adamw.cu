// SPDX-License-Identifier: Apache-2.0
//
// One AdamW step over many tensors in one launch. No counterpart in the reference, which trains nothing.
//
//     g = grad * scale
//     m' = b1 m + (1 - b1) g,   v' = b2 v + (1 - b2) g^2
//     p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// in 32 bits, from BF16, FP16 or FP32 parameters and gradients; with a 32-bit master copy of a parameter the step
// is taken on the copy and the parameter receives its rounding. The moments lie in flat buffers, each tensor's part
// starting on a block of 256 elements.
//
// 8-bit moments. Each block of 256 elements stores one exponent E (a byte) for m and one for v, and a byte for each
// element: for m a sign, 4 exponent and 3 mantissa bits, for v 5 exponent and 3 mantissa bits. A code c > 0 stands
// for the binary32 number whose bits are (8 E + c) << 20, so that codes are the leading bits of the number itself
// and neither a table nor a division is needed; c = 0 is zero. E is the largest that leaves room for the block's
// largest magnitude rounded up: 15 (m) or 31 (v) binades below it are representable. Rounding is stochastic, with
// 16 random bits for each number hashed from the element's position and the step's seed: a moment that decays by a
// few thousandths a step would never leave its code under rounding to nearest. A v > 0 is not stored as 0 (its
// root divides the step). The step itself uses the unrounded m' and v'.
//
// Bound by memory: with 8-bit moments 10 bytes an element (BF16 parameter and gradient), with 32-bit moments,
// FP32 parameter and gradient 28. A warp takes a block of 256 elements, 8 neighbouring ones a lane, so that every
// access is a wide one and a block's largest magnitude is one warp reduction.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <vector>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device_scope.cuh"
#include "runtime.cuh"

namespace oztt {
namespace adamw {

constexpr uint32_t BLOCK = OZTT_ADAMW_BLOCK;  // elements that share an exponent
constexpr uint32_t CHUNK = 32;                // blocks of one CTA
constexpr uint32_t WARPS = 8;

struct Tensor {
    void* param;
    const void* grad;
    float* master;
    uint64_t count;
    uint32_t block0;    // its first block in the moments
    uint32_t chunk0;    // its first chunk in this launch
    uint32_t param_type, grad_type;
};
template <int CAP>
struct Table {
    uint32_t count;
    Tensor t[CAP];
};
struct Moments {
    void *m, *v;
    uint8_t *m_exp, *v_exp;
};
struct Hyper {
    float beta1, one_minus_beta1, beta2, one_minus_beta2;
    float decay;       // 1 - lr wd
    float step_size;   // lr / (1 - b1^t)
    float root_scale;  // 1 / sqrt(1 - b2^t)
    float eps;
    uint32_t seed;
    const float* grad_scale;
};

__device__ __forceinline__ float half_bits(uint32_t v, uint32_t type) {
    return type == OZTT_TYPE_FP16 ? __half2float(__ushort_as_half((unsigned short)v)) : __uint_as_float(v << 16);
}
__device__ __forceinline__ uint32_t to_half_bits(float v, uint32_t type) {
    return type == OZTT_TYPE_FP16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// Eight neighbouring elements from index i on; `whole`: all eight exist and the address takes 16-byte accesses.
__device__ __forceinline__ void load8(const void* p, uint32_t type, uint64_t i, uint64_t n, bool whole, float (&x)[8]) {
    if (type == OZTT_TYPE_FP32) {
        const float* f = static_cast<const float*>(p) + i;
        if (whole) {
            const float4 a = reinterpret_cast<const float4*>(f)[0], b = reinterpret_cast<const float4*>(f)[1];
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = i + e < n ? f[e] : 0.0f;
        }
    } else {
        const uint16_t* h = static_cast<const uint16_t*>(p) + i;
        if (whole) {
            const uint4 a = *reinterpret_cast<const uint4*>(h);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = half_bits((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu, type);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = i + e < n ? half_bits(h[e], type) : 0.0f;
        }
    }
}
__device__ __forceinline__ void store8(void* p, uint32_t type, uint64_t i, uint64_t n, bool whole, const float (&x)[8]) {
    if (type == OZTT_TYPE_FP32) {
        float* f = static_cast<float*>(p) + i;
        if (whole) {
            reinterpret_cast<float4*>(f)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4*>(f)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e < n) f[e] = x[e];
        }
    } else {
        uint16_t* h = static_cast<uint16_t*>(p) + i;
        if (whole) {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = to_half_bits(x[2 * q], type) | (to_half_bits(x[2 * q + 1], type) << 16);
            *reinterpret_cast<uint4*>(h) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e < n) h[e] = (uint16_t)to_half_bits(x[e], type);
        }
    }
}

__device__ __forceinline__ bool takes16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// 32 random bits for position i: multiplications by odd numbers (the fractions of the golden ratio and of the
// square roots of 3 and 2) and shifts, modulo 2^32. The low half rounds m, the high half v.
__device__ __forceinline__ uint32_t random_bits(uint32_t i, uint32_t seed) {
    uint32_t h = i * 0x9E3779B9u + seed;
    h = (h ^ (h >> 16)) * 0xBB67AE85u;
    h = (h ^ (h >> 15)) * 0x6A09E667u;
    return h ^ (h >> 16);
}

// The exponent byte of a block whose largest magnitude has these bits, for codes of `top` binades.
__device__ __forceinline__ uint32_t block_exponent(uint32_t largest, uint32_t top) {
    const int e = (int)((largest + 0xFFFFFu) >> 23) - (int)top;
    return (uint32_t)min(max(e, 0), 254 - (int)top);
}

template <int CAP, int BITS>
__global__ void __launch_bounds__(WARPS * 32)
    adamw_kernel(const __grid_constant__ Table<CAP> table, const Moments mo, const Hyper h) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t lo = 0, hi = table.count;  // the tensor of this chunk
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (table.t[mid].chunk0 <= blockIdx.x)
            lo = mid;
        else
            hi = mid;
    }
    const Tensor& t = table.t[lo];
    const uint64_t n = t.count;
    const bool aligned = takes16(t.param) && takes16(t.grad) && takes16(t.master);
    const float scale = h.grad_scale ? *h.grad_scale : 1.0f;
    const uint64_t first = (uint64_t)(blockIdx.x - t.chunk0) * CHUNK;
    for (uint32_t b = warp; b < CHUNK; b += WARPS) {
        const uint64_t i = (first + b) * BLOCK + lane * 8;  // in the tensor
        if ((first + b) * BLOCK >= n) break;
        const uint64_t block = t.block0 + first + b;
        const uint64_t at = block * BLOCK + lane * 8;  // in the moments
        const bool whole = aligned && i + 8 <= n;
        float p[8], g[8], m[8], v[8];
        load8(t.grad, t.grad_type, i, n, whole, g);
        if (t.master)
            load8(t.master, OZTT_TYPE_FP32, i, n, whole, p);
        else
            load8(t.param, t.param_type, i, n, whole, p);
        if constexpr (BITS == 32) {
            load8(mo.m, OZTT_TYPE_FP32, at, at + 8, true, m);
            load8(mo.v, OZTT_TYPE_FP32, at, at + 8, true, v);
        } else {
            const uint2 cm = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(mo.m) + at);
            const uint2 cv = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(mo.v) + at);
            const uint32_t bm = (uint32_t)mo.m_exp[block] << 23, bv = (uint32_t)mo.v_exp[block] << 23;
            const uint32_t wm[2] = {cm.x, cm.y}, wv[2] = {cv.x, cv.y};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t c = (wm[e >> 2] >> (8 * (e & 3))) & 0xFFu, d = (wv[e >> 2] >> (8 * (e & 3))) & 0xFFu;
                const uint32_t mag = c & 0x7Fu;
                m[e] = __uint_as_float((mag ? (mag << 20) + bm : 0u) | ((c & 0x80u) << 24));
                v[e] = __uint_as_float(d ? (d << 20) + bv : 0u);
            }
        }
        // each product and sum rounded by itself, so that what is rounded to 8 bits is the same on every path
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float ge = h.grad_scale ? __fmul_rn(g[e], scale) : g[e];
            m[e] = __fadd_rn(__fmul_rn(h.beta1, m[e]), __fmul_rn(h.one_minus_beta1, ge));
            v[e] = __fadd_rn(__fmul_rn(h.beta2, v[e]), __fmul_rn(__fmul_rn(h.one_minus_beta2, ge), ge));
            float root;
            asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v[e]));
            p[e] = p[e] * h.decay - h.step_size * __fdividef(m[e], root * h.root_scale + h.eps);
        }
        if (t.master) store8(t.master, OZTT_TYPE_FP32, i, n, whole, p);
        store8(t.param, t.param_type, i, n, whole, p);
        if constexpr (BITS == 32) {
            store8(mo.m, OZTT_TYPE_FP32, at, at + 8, true, m);
            store8(mo.v, OZTT_TYPE_FP32, at, at + 8, true, v);
        } else {
            uint32_t largest_m = 0, largest_v = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                largest_m = max(largest_m, __float_as_uint(m[e]) & 0x7FFFFFFFu);
                largest_v = max(largest_v, __float_as_uint(v[e]) & 0x7FFFFFFFu);
            }
            const uint32_t em = block_exponent(__reduce_max_sync(0xFFFFFFFFu, largest_m), 15);
            const uint32_t ev = block_exponent(__reduce_max_sync(0xFFFFFFFFu, largest_v), 31);
            uint32_t wm[2] = {0, 0}, wv[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t r = random_bits((uint32_t)at + e, h.seed);
                const uint32_t xm = __float_as_uint(m[e]), am = xm & 0x7FFFFFFFu, xv = __float_as_uint(v[e]);
                const int cm = min(max((int)((am + ((r & 0xFFFFu) << 4)) >> 20) - (int)(em << 3), 0), 127);
                const int cv = min(max((int)((xv + ((r >> 16) << 4)) >> 20) - (int)(ev << 3), xv ? 1 : 0), 255);
                wm[e >> 2] |= ((uint32_t)cm | ((xm >> 24) & 0x80u)) << (8 * (e & 3));
                wv[e >> 2] |= (uint32_t)cv << (8 * (e & 3));
            }
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(mo.m) + at) = make_uint2(wm[0], wm[1]);
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(mo.v) + at) = make_uint2(wv[0], wv[1]);
            if (lane == 0) {
                mo.m_exp[block] = (uint8_t)em;
                mo.v_exp[block] = (uint8_t)ev;
            }
        }
    }
}

// The values of 8-bit moments in BF16, which holds each exactly: 8 codes a thread.
__global__ void __launch_bounds__(256) moments_kernel(const Moments mo, uint64_t groups, uint4* __restrict__ m_out,
                                                      uint4* __restrict__ v_out) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < groups; i += gridDim.x * 256ull) {
        const uint2 cm = reinterpret_cast<const uint2*>(mo.m)[i], cv = reinterpret_cast<const uint2*>(mo.v)[i];
        const uint32_t bm = (uint32_t)mo.m_exp[i / (BLOCK / 8)] << 7, bv = (uint32_t)mo.v_exp[i / (BLOCK / 8)] << 7;
        const uint32_t wm[2] = {cm.x, cm.y}, wv[2] = {cv.x, cv.y};
        uint32_t om[4] = {0, 0, 0, 0}, ov[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t c = (wm[e >> 2] >> (8 * (e & 3))) & 0xFFu, d = (wv[e >> 2] >> (8 * (e & 3))) & 0xFFu;
            const uint32_t mag = c & 0x7Fu;
            om[e >> 1] |= ((mag ? (mag << 4) + bm : 0u) | ((c & 0x80u) << 8)) << (16 * (e & 1));
            ov[e >> 1] |= (d ? (d << 4) + bv : 0u) << (16 * (e & 1));
        }
        m_out[i] = make_uint4(om[0], om[1], om[2], om[3]);
        v_out[i] = make_uint4(ov[0], ov[1], ov[2], ov[3]);
    }
}

// ---- host side -----------------------------------------------------------------------------------

constexpr int MOST = 600;  // tensors of one launch: the kernel's parameters hold 32764 bytes

template <int CAP>
static void launch(const std::vector<Tensor>& list, uint32_t chunks, int bits, const Moments& mo, const Hyper& h,
                   cudaStream_t st) {
    static_assert(sizeof(Table<CAP>) + sizeof(Moments) + sizeof(Hyper) <= 32764, "kernel parameters");
    Table<CAP> table;
    table.count = (uint32_t)list.size();
    std::copy(list.begin(), list.end(), table.t);
    if (bits == 32)
        adamw_kernel<CAP, 32><<<chunks, WARPS * 32, 0, st>>>(table, mo, h);
    else
        adamw_kernel<CAP, 8><<<chunks, WARPS * 32, 0, st>>>(table, mo, h);
    OZTT_CUDA(cudaGetLastError());
}

static Moments check_moments(const oztt_adamw_moments* s, bool some, const char* who) {
    if (!s) throw Error(OZTT_EINVAL, std::string(who) + ": no moments");
    if (s->bits != 8 && s->bits != 32) throw Error(OZTT_EINVAL, std::string(who) + ": the moments must have 8 or 32 bits");
    if (some) {
        if (!s->m || !s->v || (s->bits == 8 && (!s->m_exp || !s->v_exp)))
            throw Error(OZTT_EINVAL, std::string(who) + ": a buffer of the moments is missing");
        if ((reinterpret_cast<uintptr_t>(s->m) | reinterpret_cast<uintptr_t>(s->v)) & 15)
            throw Error(OZTT_EINVAL, std::string(who) + ": the moments must be 16-byte aligned");
    }
    return {s->m, s->v, s->m_exp, s->v_exp};
}

static void step(int device, const oztt_adamw_tensor* tensors, uint64_t count, const oztt_adamw_moments* state,
                 const oztt_adamw_hyper* hp, cudaStream_t st) {
    if (!hp || (count && !tensors)) throw Error(OZTT_EINVAL, "adamw: no arguments");
    const auto in = [](double x, double lo, double hi) { return x >= lo && x < hi; };  // false for NaN
    if (!in(hp->beta1, 0, 1) || !in(hp->beta2, 0, 1)) throw Error(OZTT_EINVAL, "adamw: the betas must be in [0, 1)");
    if (!in(hp->lr, 0, HUGE_VAL) || !in(hp->eps, 0, HUGE_VAL) || !in(hp->weight_decay, 0, HUGE_VAL))
        throw Error(OZTT_EINVAL, "adamw: lr, eps and weight_decay must be finite and not negative");
    if (hp->step < 1) throw Error(OZTT_EINVAL, "adamw: steps are counted from 1");
    if (reinterpret_cast<uintptr_t>(hp->grad_scale) & 3) throw Error(OZTT_EINVAL, "adamw: grad_scale must be 4-byte aligned");
    bool some = false;
    uint64_t blocks = 0;
    for (uint64_t i = 0; i < count; ++i) {
        const oztt_adamw_tensor& t = tensors[i];
        const auto ok = [](int32_t type) { return type >= OZTT_TYPE_BF16 && type <= OZTT_TYPE_FP32; };
        const auto size = [](int32_t type) { return type == OZTT_TYPE_FP32 ? 4u : 2u; };
        if (!ok(t.param_type) || !ok(t.grad_type))
            throw Error(OZTT_EINVAL, "adamw: tensor " + std::to_string(i) + ": the types must be BF16, FP16 or FP32");
        blocks += t.count / BLOCK + (t.count % BLOCK != 0);
        if (!t.count || !t.grad) continue;
        if (!t.param) throw Error(OZTT_EINVAL, "adamw: tensor " + std::to_string(i) + ": the parameter is missing");
        if (reinterpret_cast<uintptr_t>(t.param) % size(t.param_type) || reinterpret_cast<uintptr_t>(t.grad) % size(t.grad_type) ||
            reinterpret_cast<uintptr_t>(t.master) % 4)
            throw Error(OZTT_EINVAL, "adamw: tensor " + std::to_string(i) + ": a pointer is not aligned to its type");
        some = true;
    }
    if (blocks >= (1ull << 32)) throw Error(OZTT_EINVAL, "adamw: too many elements");
    const Moments mo = check_moments(state, some, "adamw");
    if (!some) return;
    DeviceScope scope(device);
    Hyper h;
    h.beta1 = (float)hp->beta1;
    h.one_minus_beta1 = (float)(1.0 - hp->beta1);
    h.beta2 = (float)hp->beta2;
    h.one_minus_beta2 = (float)(1.0 - hp->beta2);
    h.decay = (float)(1.0 - hp->lr * hp->weight_decay);
    h.step_size = (float)(hp->lr / (1.0 - std::pow(hp->beta1, (double)hp->step)));
    h.root_scale = (float)(1.0 / std::sqrt(1.0 - std::pow(hp->beta2, (double)hp->step)));
    h.eps = (float)hp->eps;
    h.seed = hp->seed;
    h.grad_scale = hp->grad_scale;

    std::vector<Tensor> list;
    list.reserve(std::min<uint64_t>(count, MOST));
    uint64_t chunks = 0;
    uint32_t block0 = 0;
    const auto flush = [&] {
        if (list.empty()) return;
        if (list.size() <= 32)
            launch<32>(list, (uint32_t)chunks, state->bits, mo, h, st);
        else if (list.size() <= 160)
            launch<160>(list, (uint32_t)chunks, state->bits, mo, h, st);
        else
            launch<MOST>(list, (uint32_t)chunks, state->bits, mo, h, st);
        list.clear();
        chunks = 0;
    };
    for (uint64_t i = 0; i < count; ++i) {
        const oztt_adamw_tensor& t = tensors[i];
        const uint64_t nb = t.count / BLOCK + (t.count % BLOCK != 0), nc = (nb + CHUNK - 1) / CHUNK;
        if (t.count && t.grad) {
            if (list.size() == MOST || chunks + nc >= (1ull << 31)) flush();
            list.push_back({t.param, t.grad, t.master, t.count, block0, (uint32_t)chunks, (uint32_t)t.param_type,
                            (uint32_t)t.grad_type});
            chunks += nc;
        }
        block0 += (uint32_t)nb;
    }
    flush();
}

static void values(int device, const oztt_adamw_moments* state, uint64_t blocks, uint16_t* m_out, uint16_t* v_out,
                   cudaStream_t st) {
    const Moments mo = check_moments(state, blocks != 0, "adamw_values");
    if (state->bits != 8) throw Error(OZTT_EINVAL, "adamw_values: only 8-bit moments are encoded");
    if (!blocks) return;
    if (!m_out || !v_out || ((reinterpret_cast<uintptr_t>(m_out) | reinterpret_cast<uintptr_t>(v_out)) & 15))
        throw Error(OZTT_EINVAL, "adamw_values: the outputs must be given and 16-byte aligned");
    DeviceScope scope(device);
    const uint64_t groups = blocks * (BLOCK / 8);
    const unsigned grid = (unsigned)std::min<uint64_t>((groups + 255) / 256, 148 * 8);
    moments_kernel<<<grid, 256, 0, st>>>(mo, groups, reinterpret_cast<uint4*>(m_out), reinterpret_cast<uint4*>(v_out));
    OZTT_CUDA(cudaGetLastError());
}

}  // namespace adamw
}  // namespace oztt

extern "C" int oztt_adamw_step(int device_id, const oztt_adamw_tensor* tensors, uint64_t count,
                               const oztt_adamw_moments* moments, const oztt_adamw_hyper* hyper, void* stream,
                               char* err, size_t errlen) {
    return oztt::guarded(err, errlen, [&] {
        oztt::adamw::step(device_id, tensors, count, moments, hyper, reinterpret_cast<cudaStream_t>(stream));
    });
}

extern "C" int oztt_adamw_values(int device_id, const oztt_adamw_moments* moments, uint64_t blocks, uint16_t* m_out,
                                 uint16_t* v_out, void* stream, char* err, size_t errlen) {
    return oztt::guarded(err, errlen, [&] {
        oztt::adamw::values(device_id, moments, blocks, m_out, v_out, reinterpret_cast<cudaStream_t>(stream));
    });
}
