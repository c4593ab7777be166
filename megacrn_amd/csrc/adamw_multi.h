// adamw_multi.h - AdamW over many tensors in one pass, moments in 32 or in 8 bits (gfx950, wave64).
//
//   g' = factor g      m = b1 m + (1 - b1) g'      v = b2 v + ((1 - b2) g') g'
//   p = (1 - lr wd) p - lr / (1 - b1^s) * m / (sqrt(v) / sqrt(1 - b2^s) + eps)
//
// 8-bit moments: blocks of 64 elements share a power-of-two scale (one byte, biased by 127), so that scaling is exact.  m is a
// signed float of 4 exponent and 3 mantissa bits (bias 7), v an unsigned one of 5 and 3 (bias 15): v needs the octaves, since its
// square root has to be told from 0 wherever m is.  Both are rounded up or down at random, with the chances that make the
// expected value exact: a step moves v by 0.1 % (b2 = 0.999) while neighbouring codes lie 6 - 12 % apart, so v rounded to the
// nearest code could never decay.  The random bits are a function of (seed, tensor, step, element): a run can be repeated bit for
// bit.  A v above 0 never gets code 0, which would divide m by eps.  What is not finite is held as NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "adamw_multi_api.h"

// The moments are defined as single rounded operations: no contraction of a product and a sum, here or in what is inlined.
#pragma clang fp contract(off)

namespace mcrn {

__host__ __device__ __forceinline__ unsigned adamw_mix(unsigned x) {      // xor-shifts and odd multipliers (fractions of sqrt 2, sqrt 3)
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ unsigned adamw_key_of(unsigned seed, int id, unsigned step) {
    return adamw_mix(seed + 0x9E3779B9u * (unsigned)(id + 1) + adamw_mix(step));
}

struct AdamwF32 {
    static constexpr bool WIDE = true;
    static __device__ __forceinline__ void load4(const void* p, long long i, float* v) {
        const float4 r = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
    }
    static __device__ __forceinline__ float load1(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store4(void* p, long long i, const float* v) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
    }
    static __device__ __forceinline__ void store1(void* p, long long i, float v) { static_cast<float*>(p)[i] = v; }
};
struct AdamwBf16 {
    static constexpr bool WIDE = false;
    static __device__ __forceinline__ uint32_t down(float f) {            // to the nearest, ties to even; NaN stays NaN
        const uint32_t u = __float_as_uint(f);
        if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
        return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
    }
    static __device__ __forceinline__ void load4(const void* p, long long i, float* v) {
        const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xffff0000u);
        v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xffff0000u);
    }
    static __device__ __forceinline__ float load1(const void* p, long long i) {
        return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
    }
    static __device__ __forceinline__ void store4(void* p, long long i, const float* v) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = make_uint2(down(v[0]) | (down(v[1]) << 16), down(v[2]) | (down(v[3]) << 16));
    }
    static __device__ __forceinline__ void store1(void* p, long long i, float v) { static_cast<uint16_t*>(p)[i] = (uint16_t)down(v); }
};

// the tensor that this block works on: the last one whose first block is not behind it (one compare a lane)
template <class P> __device__ __forceinline__ int adamw_tensor(const P& p) {
    const int lane = threadIdx.x & 63;
    const unsigned first = lane < p.nt ? p.t[lane < p.nt ? lane : 0].blk0 : 0xffffffffu;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(blockIdx.x >= first)) - 1);
}

// largest of the 16 lanes that hold a block of 64 elements
template <int CTRL> __device__ __forceinline__ unsigned adamw_max_dpp(unsigned v) {
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
    return v > o ? v : o;
}
__device__ __forceinline__ unsigned adamw_row_max(unsigned v) {
    v = adamw_max_dpp<0xB1>(v);           // neighbours
    v = adamw_max_dpp<0x4E>(v);           // pairs
    v = adamw_max_dpp<0x141>(v);          // halves of 8, mirrored
    return adamw_max_dpp<0x140>(v);       // halves of 16, mirrored
}
__device__ __forceinline__ unsigned adamw_finite_bits(float x) {
    const unsigned u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
template <bool SECOND> __device__ __forceinline__ float adamw_decode(unsigned code, int scale) {
    // the code's exponent and mantissa in a float's places, then the difference of the biases and the scale as one power of two
    if (SECOND) {
        const float v = __builtin_amdgcn_ldexpf(__uint_as_float(code << 20), scale - 15);
        return code == 0xffu ? __uint_as_float(0x7fc00000u) : v;
    }
    const float v = __builtin_amdgcn_ldexpf(__uint_as_float(((code & 0x7fu) << 20) | ((code & 0x80u) << 24)), scale - 7);
    return (code & 0x7fu) == 0x7fu ? __uint_as_float(0x7fc00000u) : v;
}
template <bool SECOND> __device__ __forceinline__ unsigned adamw_encode(float x, int scale, unsigned bits16) {
    const float t = __builtin_amdgcn_ldexpf(fabsf(x), (SECOND ? 15 : 7) - scale);
    unsigned code = (__float_as_uint(t) + (bits16 << 4)) >> 20;
    if (SECOND) code = x > 0.f && code == 0u ? 1u : code;
    const bool finite = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
    code = finite ? code : (SECOND ? 0xffu : 0x7fu);
    return SECOND ? code : code | ((__float_as_uint(x) >> 24) & 0x80u);
}

__device__ __forceinline__ double adamw_block_sum(double s, double* sh) {      // in every thread; sh: one double a wave
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// What the gradients are multiplied by: grad_scale, and max_norm / norm where the norm over all tensors is larger.  Every block adds the
// partial sums (a few hundred, from L2) in the same order: no further launch, no counter, the same number everywhere.
__device__ __forceinline__ float adamw_factor(const AdamwP& p, double* sh) {
    double s = 0.0;
    for (int j = threadIdx.x; j < p.parts; j += 256) s += p.part[j];
    s = adamw_block_sum(s, sh);
    const float norm = (float)(sqrt(s) * (double)p.grad_scale);
    if (p.norm && blockIdx.x == 0 && threadIdx.x == 0) p.norm[0] = norm;
    const float c = p.max_norm / (norm + 1e-6f);
    return p.grad_scale * (c > 1.f ? 1.f : c);                // a NaN norm makes every gradient NaN
}

// One block: `per` runs of 1024 elements of one tensor, four neighbours a thread.
template <class X, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwP p) {
    const int ti = adamw_tensor(p);
    if (ti < 0) return;
    const AdamwT t = p.t[ti];
    float step_size = t.step_size, inv_bc2 = t.inv_bc2, decay = t.decay;
    unsigned key = t.key;
    if (p.dyn) { const AdamwDyn d = p.dyn[t.id]; step_size = d.step_size; inv_bc2 = d.inv_bc2; decay = d.decay; key = d.key; }
    __shared__ double sh[4];
    const float factor = p.parts ? adamw_factor(p, sh) : p.grad_scale;
    const long long first = (long long)(blockIdx.x - t.blk0) * p.per * 1024;
    for (int r = 0; r < p.per; ++r) {
        const long long i = first + r * 1024 + threadIdx.x * 4;
        if (first + r * 1024 >= t.n) return;
        const bool whole = i + 4 <= t.n, some = i < t.n;
        const bool vec = whole && (t.flags & ADAMW_VEC);
        const long long a = t.off + i;
        float g[4] = {0.f, 0.f, 0.f, 0.f}, w[4] = {0.f, 0.f, 0.f, 0.f}, m[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
        if (some) {                       // the arenas reach to the end of the block of 64: four of their elements at a time
            if (vec) X::load4(t.g, i, g);
            else for (int k = 0; k < 4; ++k) if (i + k < t.n) g[k] = X::load1(t.g, i + k);
            if (!X::WIDE) AdamwF32::load4(p.master, a, w);
            else if (vec) X::load4(t.p, i, w);
            else for (int k = 0; k < 4; ++k) if (i + k < t.n) w[k] = X::load1(t.p, i + k);
            if (BITS == 32) {
                AdamwF32::load4(p.m, a, m);
                AdamwF32::load4(p.v, a, v);
            } else {
                const uint32_t cm = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.m) + a);
                const uint32_t cv = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.v) + a);
                const int sm = p.ms[a / ADAMW_BLOCK], sv = p.vs[a / ADAMW_BLOCK];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    m[k] = adamw_decode<false>((cm >> (8 * k)) & 0xffu, sm);
                    v[k] = adamw_decode<true>((cv >> (8 * k)) & 0xffu, sv);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float gk = g[k] * factor;
            m[k] = p.b1 * m[k] + p.c1 * gk;
            v[k] = p.b2 * v[k] + (p.c2 * gk) * gk;
            w[k] = w[k] * decay - step_size * (m[k] / (sqrtf(v[k]) * inv_bc2 + p.eps));
        }
        if (i + 4 > t.n) {                // what lies behind the tensor's end stays 0 (a factor that is not finite would make it NaN)
#pragma unroll
            for (int k = 0; k < 4; ++k) if (i + k >= t.n) m[k] = v[k] = w[k] = 0.f;
        }
        if (some) {
            if (vec) X::store4(t.p, i, w);
            else for (int k = 0; k < 4; ++k) if (i + k < t.n) X::store1(t.p, i + k, w[k]);
            if (!X::WIDE) AdamwF32::store4(p.master, a, w);
        }
        if (BITS == 32) {
            if (some) { AdamwF32::store4(p.m, a, m); AdamwF32::store4(p.v, a, v); }
        } else {
            unsigned tm = 0, tv = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned um = adamw_finite_bits(m[k]), uv = adamw_finite_bits(v[k]);
                tm = tm > um ? tm : um;
                tv = tv > uv ? tv : uv;
            }
            const int em = (int)(adamw_row_max(tm) >> 23), ev = (int)(adamw_row_max(tv) >> 23);
            const int sm = em > 8 ? em - 7 : 1, sv = ev > 16 ? ev - 15 : 1;
            unsigned cm = 0, cv = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned long long e = (unsigned long long)(i + k);
                const unsigned bits = adamw_mix((unsigned)e * 0x9E3779B9u + (unsigned)(e >> 32) * 0x85157AF5u + key);
                cm |= adamw_encode<false>(m[k], sm, bits & 0xffffu) << (8 * k);
                cv |= adamw_encode<true>(v[k], sv, bits >> 16) << (8 * k);
            }
            if (some) {
                *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.m) + a) = cm;
                *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.v) + a) = cv;
                if ((threadIdx.x & 15) == 0) {
                    p.ms[a / ADAMW_BLOCK] = (uint8_t)sm;
                    p.vs[a / ADAMW_BLOCK] = (uint8_t)sv;
                }
            }
        }
    }
}

// Sums of squares in 64 bits (the squares of floats are exact there), one a block; adamw_kernel adds them in their order.
template <class X>
__global__ __launch_bounds__(256) void adamw_norm_kernel(AdamwNormP p) {
    const int ti = adamw_tensor(p);
    double s = 0.0;
    if (ti >= 0) {
        const AdamwT t = p.t[ti];
        const long long first = (long long)(blockIdx.x - t.blk0) * p.per * 1024, end = min(t.n, first + p.per * 1024ll);
        long long i = first + threadIdx.x * 4;
        constexpr int U = 8;                                  // loads in flight
        if (t.flags & ADAMW_VEC) {
            for (; first + (i - first) / 1024 * 1024 + U * 1024 <= end; i += U * 1024) {
                float g[U][4];
#pragma unroll
                for (int u = 0; u < U; ++u) X::load4(t.g, i + u * 1024, g[u]);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s = fma((double)g[u][k], (double)g[u][k], s);
            }
        }
        for (; i < end; i += 1024) {
            float g[4] = {0.f, 0.f, 0.f, 0.f};
            if (i + 4 <= end && (t.flags & ADAMW_VEC)) X::load4(t.g, i, g);
            else for (int k = 0; k < 4; ++k) if (i + k < end) g[k] = X::load1(t.g, i + k);
#pragma unroll
            for (int k = 0; k < 4; ++k) s = fma((double)g[k], (double)g[k], s);
        }
    }
    __shared__ double sh[4];
    s = adamw_block_sum(s, sh);
    if (threadIdx.x == 0) p.part[p.blk0 + blockIdx.x] = s;
}

// Steps counted on the device (a captured step is replayed with its own numbers): one thread a tensor.
__global__ void adamw_prep_kernel(AdamwPrepP p) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= p.nt || !((p.has[i >> 6] >> (i & 63)) & 1ull)) return;
    const int k = p.base + i, s = p.step[k] + 1;
    p.step[k] = s;
    AdamwDyn d;
    d.step_size = (float)(p.lr[k] / (1.0 - pow(p.b1, (double)s)));
    d.inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(p.b2, (double)s)));
    d.decay = (float)(1.0 - p.lr[k] * p.wd[k]);
    d.key = adamw_key_of(p.seed, k, (unsigned)s);
    p.dyn[k] = d;
}

// The values that codes stand for, four a thread: m (blockIdx.y 0) and v.
__global__ __launch_bounds__(256) void adamw_unpack_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ ms, const uint8_t* __restrict__ v,
                                                           const uint8_t* __restrict__ vs, float* __restrict__ om, float* __restrict__ ov, long long n4) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) return;
    const bool second = blockIdx.y != 0;
    const uint32_t c = reinterpret_cast<const uint32_t*>(second ? v : m)[i];
    const int s = (second ? vs : ms)[i * 4 / ADAMW_BLOCK];
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = second ? adamw_decode<true>((c >> (8 * k)) & 0xffu, s) : adamw_decode<false>((c >> (8 * k)) & 0xffu, s);
    AdamwF32::store4(second ? ov : om, i * 4, x);
}

}  // namespace mcrn
