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
// Bound by memory: with 8-bit moments 10 bytes an element (BF16 parameter and gradient), 16 with a master, with
// 32-bit moments, FP32 parameter and gradient 28. A warp takes a block of 256 elements, 8 neighbouring ones a lane, by
// accesses of 8 to 32 bytes that together cover whole lines; a block's largest magnitude is one warp reduction. The
// codes are taken apart and put together two at a time in 16-bit halves, and the arithmetic is on the packed FP32
// pipe: about 60 instructions an element, which the memory still covers.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <vector>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "launch.cuh"
#include "runtime.cuh"

namespace oztt {
namespace adamw {

constexpr uint32_t BLOCK = OZTT_ADAMW_BLOCK;  // elements that share an exponent
constexpr uint32_t LEAST_CHUNK = 8, MOST_CHUNK = 64;  // blocks of one CTA
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
    uint32_t count, chunk;  // tensors; blocks of a chunk
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
    float minus_zero;  // -0, by a route the compiler does not see through
    const float* grad_scale;
};

// Eight neighbouring elements as they lie in memory: 16-bit ones in the first four words.
template <bool WIDE>
struct Words {
    uint32_t w[WIDE ? 8 : 4];
};
// `whole`: all eight exist and the address takes one access for them (32 bytes wide for 32-bit ones, so that a warp's
// accesses cover whole lines); else those of index below n, zeros beyond.
template <bool WIDE>
__device__ __forceinline__ void load(Words<WIDE>& x, const void* p, uint64_t i, uint64_t n, bool whole) {
    if (whole) {
        if constexpr (WIDE) {
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(x.w[0]), "=r"(x.w[1]), "=r"(x.w[2]), "=r"(x.w[3]), "=r"(x.w[4]), "=r"(x.w[5]),
                           "=r"(x.w[6]), "=r"(x.w[7])
                         : "l"(static_cast<const float*>(p) + i)
                         : "memory");
        } else {
            const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
            x.w[0] = v.x, x.w[1] = v.y, x.w[2] = v.z, x.w[3] = v.w;
        }
    } else if (WIDE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x.w[e % (WIDE ? 8 : 4)] = i + e < n ? static_cast<const uint32_t*>(p)[i + e] : 0;
    } else {
        const uint16_t* q = static_cast<const uint16_t*>(p) + i;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            x.w[e] = (i + 2 * e < n ? (uint32_t)q[2 * e] : 0u) | (i + 2 * e + 1 < n ? (uint32_t)q[2 * e + 1] << 16 : 0u);
    }
}
template <bool WIDE>
__device__ __forceinline__ void store(const Words<WIDE>& x, void* p, uint64_t i, uint64_t n, bool whole) {
    if (whole) {
        if constexpr (WIDE)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<float*>(p) + i),
                         "r"(x.w[0]), "r"(x.w[1]), "r"(x.w[2]), "r"(x.w[3]), "r"(x.w[4]), "r"(x.w[5]), "r"(x.w[6]),
                         "r"(x.w[7])
                         : "memory");
        else
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
    } else if (WIDE) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i + e < n) static_cast<uint32_t*>(p)[i + e] = x.w[e % (WIDE ? 8 : 4)];
    } else {
        uint16_t* q = static_cast<uint16_t*>(p) + i;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i + e < n) q[e] = (uint16_t)(x.w[e / 2] >> (16 * (e & 1)));
    }
}
template <bool WIDE>
__device__ __forceinline__ void values(const Words<WIDE>& x, uint32_t type, f32x2 (&v)[4]) {
    if (WIDE) {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = pk2(__uint_as_float(x.w[(2 * q) % (WIDE ? 8 : 4)]), __uint_as_float(x.w[(2 * q + 1) % (WIDE ? 8 : 4)]));
    } else if (type == OZTT_TYPE_FP16) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x.w[q]));
            v[q] = pk2(f.x, f.y);
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = pk2(__uint_as_float(x.w[q] << 16), __uint_as_float(x.w[q] & 0xFFFF0000u));
    }
}
__device__ __forceinline__ Words<true> wide_words(const f32x2 (&v)[4]) {
    Words<true> x;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        x.w[2 * q] = (uint32_t)v[q];
        x.w[2 * q + 1] = (uint32_t)(v[q] >> 32);
    }
    return x;
}
__device__ __forceinline__ Words<false> half_words(const f32x2 (&v)[4], uint32_t type) {
    Words<false> x;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float lo, hi;
        unpk2(v[q], lo, hi);
        if (type == OZTT_TYPE_FP16)
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x.w[q]) : "f"(hi), "f"(lo));
        else
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(x.w[q]) : "f"(hi), "f"(lo));
    }
    return x;
}

__device__ __forceinline__ bool takes_vectors(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

// 32 random bits for position i: multiplications by odd numbers (the fractions of the golden ratio and of the
// square roots of 3 and 2) and shifts, modulo 2^32. The low half rounds m, the high half v.
__device__ __forceinline__ void random_halves(uint32_t h, uint32_t& low, uint32_t& high) {  // of h = i * kGolden + seed
    h = (h ^ (h >> 16)) * 0xBB67AE85u;
    h = (h ^ (h >> 15)) * 0x6A09E667u;
    high = h >> 16;
    low = (h ^ high) & 0xFFFFu;
}
constexpr uint32_t kGolden = 0x9E3779B9u;

// The exponent byte of a block whose largest magnitude has these bits, for codes of `top` binades.
__device__ __forceinline__ uint32_t block_exponent(uint32_t largest, uint32_t top) {
    const int e = (int)((largest + 0xFFFFFu) >> 23) - (int)top;
    return (uint32_t)min(max(e, 0), 254 - (int)top);
}

// The exponents of a CTA's blocks, of one byte each: read and written together, since a byte read from a sector that
// other SMs write bytes of waits microseconds (242 million elements with a master: 1108 us when each warp read its
// own, 671 so).
struct Exponents {
    uint8_t m[MOST_CHUNK], v[MOST_CHUNK];
};

// The leading 16 bits of two values from the two low (high) codes of a word, base = 8 E: (c << 4) + (E << 7), the
// base added where min(c << 4, 16) is not zero.
__device__ __forceinline__ uint32_t m_values(uint32_t word, bool high, uint32_t base) {
    const uint32_t c = __byte_perm(word, 0, high ? 0x4342u : 0x4140u), mag = (c & 0x007F007Fu) * 16u;
    return (__viaddmin_u16x2(mag, 0, 0x00100010u) * base + mag) | ((c << 8) & 0x80008000u);
}
__device__ __forceinline__ uint32_t v_values(uint32_t word, bool high, uint32_t base) {
    const uint32_t d = __byte_perm(word, 0, high ? 0x4342u : 0x4140u) * 16u;
    return __viaddmin_u16x2(d, 0, 0x00100010u) * base + d;
}

// The eight moments of a lane as they lie in memory.
template <int BITS>
struct Kept {
    Words<true> m, v;
    __device__ __forceinline__ void read(const Moments& mo, uint64_t block, uint32_t lane, const Exponents&, uint32_t) {
        load(m, mo.m, block * BLOCK + lane * 8, ~0ull, true);
        load(v, mo.v, block * BLOCK + lane * 8, ~0ull, true);
    }
    __device__ __forceinline__ void decode(f32x2 (&dm)[4], f32x2 (&dv)[4]) const {
        values(m, OZTT_TYPE_FP32, dm);
        values(v, OZTT_TYPE_FP32, dv);
    }
    static __device__ __forceinline__ void write(const Moments& mo, uint64_t block, uint32_t lane, Exponents&, uint32_t,
                                                 uint32_t, const f32x2 (&dm)[4], const f32x2 (&dv)[4]) {
        store(wide_words(dm), mo.m, block * BLOCK + lane * 8, ~0ull, true);
        store(wide_words(dv), mo.v, block * BLOCK + lane * 8, ~0ull, true);
    }
};
template <>
struct Kept<8> {
    uint2 m, v;
    uint32_t em, ev;
    __device__ __forceinline__ void read(const Moments& mo, uint64_t block, uint32_t lane, const Exponents& ex, uint32_t b) {
        m = reinterpret_cast<const uint2*>(mo.m)[block * (BLOCK / 8) + lane];
        v = reinterpret_cast<const uint2*>(mo.v)[block * (BLOCK / 8) + lane];
        em = ex.m[b];
        ev = ex.v[b];
    }
    __device__ __forceinline__ void decode(f32x2 (&dm)[4], f32x2 (&dv)[4]) const {
        const uint32_t wm[2] = {m.x, m.y}, wv[2] = {v.x, v.y}, bm = em << 3, bv = ev << 3;
        const auto two = [](uint32_t x) { return pk2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u)); };
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            dm[q] = two(m_values(wm[q >> 1], q & 1, bm));
            dv[q] = two(v_values(wv[q >> 1], q & 1, bv));
        }
    }
    // The leading 16 bits of a magnitude with its random number added, less the base: the code and 4 bits below it,
    // clamped to the code's range, two at a time.
    static __device__ __forceinline__ void write(const Moments& mo, uint64_t block, uint32_t lane, Exponents& ex, uint32_t b,
                                                 uint32_t seed, const f32x2 (&dm)[4], const f32x2 (&dv)[4]) {
        float fm[8], fv[8], large_m = 0.0f, large_v = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) unpk2(dm[q], fm[2 * q], fm[2 * q + 1]), unpk2(dv[q], fv[2 * q], fv[2 * q + 1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) large_m = fmaxf(large_m, fabsf(fm[e])), large_v = fmaxf(large_v, fv[e]);
        const uint32_t xm = block_exponent(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(large_m)), 15);
        const uint32_t xv = block_exponent(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(large_v)), 31);
        const uint32_t less_m = (0x10000u - (xm << 7)) * 0x10001u & (xm ? ~0u : 0u);  // both halves: -(E << 7)
        const uint32_t less_v = (0x10000u - (xv << 7)) * 0x10001u & (xv ? ~0u : 0u);
        const uint32_t h = ((uint32_t)block * BLOCK + lane * 8) * kGolden + seed;
        uint32_t cm[4], cv[4], sign[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t ym[2], yv[2], least[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t low, high;
                random_halves(h + (2 * q + e) * kGolden, low, high);
                ym[e] = low * 16u + __float_as_uint(fabsf(fm[2 * q + e]));
                const uint32_t size = __float_as_uint(fv[2 * q + e]);
                yv[e] = high * 16u + size;
                least[e] = __viaddmin_u32(size, 0xFFFFFu, 0x1FFFFFu);  // its leading half is 0x10 or more where v > 0: code 1
            }
            cm[q] = __viaddmin_s16x2_relu(__byte_perm(ym[0], ym[1], 0x7632), less_m, 0x07FF07FFu) >> 4;
            cv[q] = __viaddmax_u16x2(__viaddmin_s16x2_relu(__byte_perm(yv[0], yv[1], 0x7632), less_v, 0x0FFF0FFFu), 0,
                                     __byte_perm(least[0], least[1], 0x7632)) >> 4;
            sign[q] = __byte_perm(__float_as_uint(fm[2 * q]), __float_as_uint(fm[2 * q + 1]), 0x0073);
        }
        const auto bytes = [](const uint32_t (&c)[4], int i) { return __byte_perm(c[i], c[i + 1], 0x6420); };
        const auto signs = [&](int i) { return __byte_perm(sign[i], sign[i + 1], 0x5410) & 0x80808080u; };
        reinterpret_cast<uint2*>(mo.m)[block * (BLOCK / 8) + lane] = make_uint2(bytes(cm, 0) | signs(0), bytes(cm, 2) | signs(2));
        reinterpret_cast<uint2*>(mo.v)[block * (BLOCK / 8) + lane] = make_uint2(bytes(cv, 0), bytes(cv, 2));
        if (lane == 0) {
            ex.m[b] = (uint8_t)xm;
            ex.v[b] = (uint8_t)xv;
        }
    }
};

// A warp's blocks of one chunk. P32: the step is taken on 32-bit values (an FP32 parameter or a master); G32: the
// gradient is FP32.
template <int BITS, bool P32, bool G32>
__device__ __forceinline__ void chunk(const Tensor& t, uint64_t first, uint32_t blocks, uint32_t warp, uint32_t lane,
                                      const Moments& mo, const Hyper& h, Exponents& ex) {
    const uint64_t n = t.count;
    const bool aligned = takes_vectors(t.param) && takes_vectors(t.grad) && takes_vectors(t.master);
    void* const source = t.master ? t.master : t.param;
    const uint32_t ptype = t.param_type, gtype = t.grad_type;
    const f32x2 none = splat2(h.minus_zero);  // a sum with it keeps a product's own rounding, and cannot be fused away
    const f32x2 scale = splat2(h.grad_scale ? *h.grad_scale : 1.0f);
    for (uint32_t b = warp; b < blocks; b += WARPS) {
        const uint64_t i = (first + b) * BLOCK + lane * 8, block = t.block0 + first + b;
        const bool whole = aligned && i + 8 <= n;
        f32x2 g[4], p[4], m[4], v[4];
        {
            Words<G32> wg;
            Words<P32> wp;
            Kept<BITS> kept;
            kept.read(mo, block, lane, ex, b);
            load(wg, t.grad, i, n, whole);
            load(wp, source, i, n, whole);
            values(wg, gtype, g);
            values(wp, ptype, p);
            kept.decode(m, v);
        }
        // m and v: each product and sum rounded by itself, so that what is rounded to 8 bits is the same on every path
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (h.grad_scale) g[q] = fused2(g[q], scale, none);
            m[q] = plus2(fused2(splat2(h.beta1), m[q], none), fused2(splat2(h.one_minus_beta1), g[q], none));
            v[q] = plus2(fused2(splat2(h.beta2), v[q], none),
                         fused2(fused2(splat2(h.one_minus_beta2), g[q], none), g[q], none));
            float r0, r1;
            unpk2(v[q], r0, r1);
            asm("sqrt.approx.f32 %0, %0;" : "+f"(r0));
            asm("sqrt.approx.f32 %0, %0;" : "+f"(r1));
            unpk2(fused2(pk2(r0, r1), splat2(h.root_scale), splat2(h.eps)), r0, r1);
            asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r0));  // never of a subnormal number, unless eps is one
            asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r1));
            p[q] = fused2(fused2(m[q], pk2(r0, r1), none), splat2(-h.step_size), fused2(p[q], splat2(h.decay), none));
        }
        if (P32) {
            store(wide_words(p), source, i, n, whole);
            if (ptype != OZTT_TYPE_FP32)
                store(half_words(p, ptype), t.param, i, n, whole);
            else if (t.master)  // an FP32 parameter beside its master: the same value
                store(wide_words(p), t.param, i, n, whole);
        } else {
            store(half_words(p, ptype), t.param, i, n, whole);
        }
        Kept<BITS>::write(mo, block, lane, ex, b, h.seed, m, v);
    }
}

template <int CAP, int BITS>
__global__ void __launch_bounds__(WARPS * 32)
    adamw_kernel(const __grid_constant__ Table<CAP> table, const __grid_constant__ Moments mo,
                 const __grid_constant__ Hyper h) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t lo = 0, hi = table.count;  // the tensor of this chunk
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (table.t[mid].chunk0 <= blockIdx.x)
            lo = mid;
        else
            hi = mid;
    }
    overlap_launches();
    const Tensor& t = table.t[lo];
    const uint64_t first = (uint64_t)(blockIdx.x - t.chunk0) * table.chunk;
    const uint64_t left = (t.count - first * BLOCK + BLOCK - 1) / BLOCK;
    const uint32_t blocks = (uint32_t)min(left, (uint64_t)table.chunk);
    __shared__ Exponents ex;
    const auto exponents = [&](auto&& each) {
        for (uint32_t b = threadIdx.x; b < blocks; b += WARPS * 32) each(b, t.block0 + first + b);
    };
    if constexpr (BITS == 8) {
        exponents([&](uint32_t b, uint64_t block) { ex.m[b] = mo.m_exp[block], ex.v[b] = mo.v_exp[block]; });
        __syncthreads();
    }
    const bool p32 = t.master || t.param_type == OZTT_TYPE_FP32, g32 = t.grad_type == OZTT_TYPE_FP32;
    if (p32 && g32)
        chunk<BITS, true, true>(t, first, blocks, warp, lane, mo, h, ex);
    else if (p32)
        chunk<BITS, true, false>(t, first, blocks, warp, lane, mo, h, ex);
    else if (g32)
        chunk<BITS, false, true>(t, first, blocks, warp, lane, mo, h, ex);
    else
        chunk<BITS, false, false>(t, first, blocks, warp, lane, mo, h, ex);
    if constexpr (BITS == 8) {
        __syncthreads();
        exponents([&](uint32_t b, uint64_t block) { mo.m_exp[block] = ex.m[b], mo.v_exp[block] = ex.v[b]; });
    }
}

// The values of 8-bit moments in BF16, which holds each exactly: 16 codes of each a thread.
__global__ void __launch_bounds__(256) moments_kernel(const Moments mo, uint64_t groups, uint16_t* __restrict__ m_out,
                                                      uint16_t* __restrict__ v_out) {
    overlap_launches();
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < groups; i += gridDim.x * 256ull) {
        const uint4 cm = reinterpret_cast<const uint4*>(mo.m)[i], cv = reinterpret_cast<const uint4*>(mo.v)[i];
        const uint32_t bm = (uint32_t)mo.m_exp[i / (BLOCK / 16)] << 3, bv = (uint32_t)mo.v_exp[i / (BLOCK / 16)] << 3;
        const uint32_t wm[4] = {cm.x, cm.y, cm.z, cm.w}, wv[4] = {cv.x, cv.y, cv.z, cv.w};
        Words<true> om, ov;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            om.w[q] = m_values(wm[q >> 1], q & 1, bm);
            ov.w[q] = v_values(wv[q >> 1], q & 1, bv);
        }
        store(om, m_out, i * 8, ~0ull, true);  // (8 words, of two values each)
        store(ov, v_out, i * 8, ~0ull, true);
    }
}

// ---- host side -----------------------------------------------------------------------------------

constexpr int MOST = 600;  // tensors of one launch: the kernel's parameters hold 32764 bytes

template <int CAP>
static void launch(std::vector<Tensor>& list, uint64_t blocks, int bits, const Moments& mo, const Hyper& h,
                   cudaStream_t st) {
    static_assert(sizeof(Table<CAP>) + sizeof(Moments) + sizeof(Hyper) <= 32764, "kernel parameters");
    Table<CAP> table;
    table.count = (uint32_t)list.size();
    // Few blocks a CTA while the device is not full, then more, up to 64 (32 with 32-bit moments): the CTAs that run at
    // one time stay within a stretch of each buffer. Measured at 242 million elements, 8 bits with a master, 64: 621 us,
    // 32: 636, 512: 676; 32 bits, 32: 1039 us, 128: 1081, 512: 1107.
    const uint32_t most = bits == 8 ? MOST_CHUNK : MOST_CHUNK / 2;
    table.chunk = LEAST_CHUNK;
    while (table.chunk < most && blocks / table.chunk > 8 * multiprocessors(current_device())) table.chunk *= 2;
    uint32_t chunks = 0;
    for (Tensor& t : list) {
        t.chunk0 = chunks;
        chunks += (uint32_t)(((t.count + BLOCK - 1) / BLOCK + table.chunk - 1) / table.chunk);
    }
    std::copy(list.begin(), list.end(), table.t);
    auto* kernel = bits == 32 ? adamw_kernel<CAP, 32> : adamw_kernel<CAP, 8>;
    launch_overlapped(kernel, dim3(chunks), WARPS * 32, 0, dim3(0), st, table, mo, h);
}

static Moments check_moments(const oztt_adamw_moments* s, bool some, const char* who) {
    if (!s) throw Error(OZTT_EINVAL, std::string(who) + ": no moments");
    if (s->bits != 8 && s->bits != 32) throw Error(OZTT_EINVAL, std::string(who) + ": the moments must have 8 or 32 bits");
    if (some) {
        if (!s->m || !s->v || (s->bits == 8 && (!s->m_exp || !s->v_exp)))
            throw Error(OZTT_EINVAL, std::string(who) + ": a buffer of the moments is missing");
        if ((reinterpret_cast<uintptr_t>(s->m) | reinterpret_cast<uintptr_t>(s->v)) & 31)
            throw Error(OZTT_EINVAL, std::string(who) + ": the moments must be 32-byte aligned");
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
    check_earlier_calls(device);  // gradients of a product that gave up are not applied
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
    h.minus_zero = -0.0f;
    h.grad_scale = hp->grad_scale;

    std::vector<Tensor> list;
    list.reserve(std::min<uint64_t>(count, MOST));
    uint64_t live_blocks = 0;
    uint32_t block0 = 0;
    const auto flush = [&] {
        if (list.empty()) return;
        if (list.size() <= 32)
            launch<32>(list, live_blocks, state->bits, mo, h, st);
        else if (list.size() <= 160)
            launch<160>(list, live_blocks, state->bits, mo, h, st);
        else
            launch<MOST>(list, live_blocks, state->bits, mo, h, st);
        list.clear();
        live_blocks = 0;
    };
    for (uint64_t i = 0; i < count; ++i) {
        const oztt_adamw_tensor& t = tensors[i];
        const uint64_t nb = t.count / BLOCK + (t.count % BLOCK != 0);
        if (t.count && t.grad) {
            if (list.size() == MOST) flush();
            list.push_back({t.param, t.grad, t.master, t.count, block0, 0, (uint32_t)t.param_type, (uint32_t)t.grad_type});
            live_blocks += nb;
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
    if (!m_out || !v_out || ((reinterpret_cast<uintptr_t>(m_out) | reinterpret_cast<uintptr_t>(v_out)) & 31))
        throw Error(OZTT_EINVAL, "adamw_values: the outputs must be given and 32-byte aligned");
    DeviceScope scope(device);
    check_earlier_calls(device);
    const uint64_t groups = blocks * (BLOCK / 16);
    const unsigned grid = (unsigned)std::min<uint64_t>((groups + 255) / 256, multiprocessors(device) * 32);
    launch_overlapped(moments_kernel, dim3(grid), 256, 0, dim3(0), st, mo, groups, m_out, v_out);
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
