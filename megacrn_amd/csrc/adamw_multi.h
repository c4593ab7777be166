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

typedef float AdamwV4 __attribute__((ext_vector_type(4)));
typedef __bf16 AdamwH4 __attribute__((ext_vector_type(4)));
// NT: what is streamed once through a step that is larger than the caches (launch_adamw) leaves them alone
template <bool NT, class V> __device__ __forceinline__ V adamw_ld(const void* p) {
    return NT ? __builtin_nontemporal_load(static_cast<const V*>(p)) : *static_cast<const V*>(p);
}
template <bool NT, class V> __device__ __forceinline__ void adamw_st(void* p, V v) {
    if (NT) __builtin_nontemporal_store(v, static_cast<V*>(p));
    else *static_cast<V*>(p) = v;
}
struct AdamwF32 {
    typedef float S;
    static constexpr bool WIDE = true;
    template <bool NT> static __device__ __forceinline__ void load4(const void* p, long long i, float* v) {
        const AdamwV4 r = adamw_ld<NT, AdamwV4>(static_cast<const float*>(p) + i);
        v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
    }
    template <bool NT> static __device__ __forceinline__ void store4(void* p, long long i, const float* v) {
        const AdamwV4 r = {v[0], v[1], v[2], v[3]};
        adamw_st<NT>(static_cast<float*>(p) + i, r);
    }
};
struct AdamwBf16 {
    typedef __bf16 S;
    static constexpr bool WIDE = false;
    template <bool NT> static __device__ __forceinline__ void load4(const void* p, long long i, float* v) {
        typedef uint32_t U2 __attribute__((ext_vector_type(2)));
        const U2 r = adamw_ld<NT, U2>(static_cast<const uint16_t*>(p) + i);
        v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xffff0000u);
        v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xffff0000u);
    }
    template <bool NT> static __device__ __forceinline__ void store4(void* p, long long i, const float* v) {
        const AdamwH4 r = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};       // to the nearest, ties to even, by the hardware
        adamw_st<NT>(static_cast<__bf16*>(p) + i, r);
    }
};
template <class X> __device__ __forceinline__ float adamw_load1(const void* p, long long i) { return (float)static_cast<const typename X::S*>(p)[i]; }
template <class X> __device__ __forceinline__ void adamw_store1(void* p, long long i, float v) { static_cast<typename X::S*>(p)[i] = (typename X::S)v; }

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
// four codes -> values.  m: the hardware's own format (e4m3), times the scale.  v: the code's exponent and mantissa in a float's places, then
// the difference of the biases and the scale as one power of two (what is below the format's normal numbers is so below the float's).
__device__ __forceinline__ void adamw_decode_m(unsigned codes, int scale, float* m) {
    const float s = __uint_as_float((unsigned)scale << 23);
    m[0] = __builtin_amdgcn_cvt_f32_fp8(codes, 0) * s;
    m[1] = __builtin_amdgcn_cvt_f32_fp8(codes, 1) * s;
    m[2] = __builtin_amdgcn_cvt_f32_fp8(codes, 2) * s;
    m[3] = __builtin_amdgcn_cvt_f32_fp8(codes, 3) * s;
}
__device__ __forceinline__ void adamw_decode_v(unsigned codes, int scale, float* v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const unsigned c = (codes >> (8 * k)) & 0xffu;
        v[k] = c == 0xffu ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(__uint_as_float(c << 20), scale - 15);
    }
}
// value -> code.  FINITE: the caller has seen that every value of the wave is
template <bool FINITE> __device__ __forceinline__ unsigned adamw_encode_m(float x, int scale, unsigned bits) {
    const float t = __builtin_amdgcn_ldexpf(fabsf(x), 7 - scale);
    unsigned code = (__float_as_uint(t) + ((bits & 0xffffu) << 4)) >> 20;
    if (!FINITE) code = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u ? code : 0x7fu;
    return code | ((__float_as_uint(x) >> 24) & 0x80u);
}
template <bool FINITE> __device__ __forceinline__ unsigned adamw_encode_v(float x, int scale, unsigned bits) {
    const float t = __builtin_amdgcn_ldexpf(x, 15 - scale);
    const unsigned least = __float_as_uint(x) < 1u ? __float_as_uint(x) : 1u;      // what is above 0 stays above 0
    unsigned code = (__float_as_uint(t) + ((bits >> 12) & 0xffff0u)) >> 20;
    code = code > least ? code : least;
    if (!FINITE) code = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u ? code : 0xffu;
    return code;
}
__device__ __forceinline__ unsigned adamw_max4(unsigned a, unsigned b, unsigned c, unsigned d) {
    const unsigned x = a > b ? a : b, y = c > d ? c : d;
    return x > y ? x : y;
}

__device__ __forceinline__ double adamw_block_sum(double s, double* sh) {      // in every thread; sh: one double a wave
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// What the gradients are multiplied by: grad_scale, and max_norm / norm where the norm over all tensors is larger, from the partial sums in
// their order (the same number whoever adds them).
__device__ __forceinline__ float adamw_factor(const double* part, int parts, float grad_scale, float max_norm, float* norm_out, double* sh) {
    double s = 0.0;
    for (int j = threadIdx.x; j < parts; j += 256) s += part[j];
    s = adamw_block_sum(s, sh);
    const float norm = (float)(sqrt(s) * (double)grad_scale);
    if (norm_out && threadIdx.x == 0) norm_out[0] = norm;
    const float c = max_norm / (norm + 1e-6f);
    return grad_scale * (c > 1.f ? 1.f : c);                  // a NaN norm makes every gradient NaN
}
// One block, for steps of many blocks: 473 us with 129 K blocks that each add 523 sums (132 M parameters in bf16, 8-bit moments), 406 so.
// Small steps let every block add them, which saves the launch (9 us of work in all).
__global__ __launch_bounds__(256) void adamw_factor_kernel(const double* part, int parts, float grad_scale, float max_norm, float* norm, float* factor) {
    __shared__ double sh[4];
    const float f = adamw_factor(part, parts, grad_scale, max_norm, norm, sh);
    if (threadIdx.x == 0) factor[0] = f;
}

// What a thread reads for its four neighbours of a run.
template <int BITS> struct AdamwRaw {
    float g[4], w[4], m[4], v[4];
    unsigned cm, cv;
    int sm, sv;
};
// i: first of the four, a: its place in the arenas (which reach to the end of the block of 64: always four elements there).  WHOLE: the
// run lies inside the tensor and can be read four elements at a time.
template <class X, int BITS, bool NT, bool WHOLE>
__device__ __forceinline__ void adamw_read(const AdamwP& p, const AdamwT& t, long long i, AdamwRaw<BITS>& r) {
    const long long a = t.off + i;
    const bool some = WHOLE || i < t.n;
    if (WHOLE) {
        X::template load4<NT>(t.g, i, r.g);
        if (X::WIDE) X::template load4<NT>(t.p, i, r.w);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            r.g[k] = i + k < t.n ? adamw_load1<X>(t.g, i + k) : 0.f;
            r.w[k] = X::WIDE && i + k < t.n ? adamw_load1<X>(t.p, i + k) : 0.f;
            r.m[k] = r.v[k] = 0.f;
        }
    }
    if (some) {
        if (!X::WIDE) AdamwF32::load4<NT>(p.master, a, r.w);
        if (BITS == 32) {
            AdamwF32::load4<NT>(p.m, a, r.m);
            AdamwF32::load4<NT>(p.v, a, r.v);
        }
    }
    if (BITS == 8) {
        r.cm = some ? adamw_ld<NT, unsigned>(static_cast<const uint8_t*>(p.m) + a) : 0u;
        r.cv = some ? adamw_ld<NT, unsigned>(static_cast<const uint8_t*>(p.v) + a) : 0u;
        r.sm = some ? p.ms[a / ADAMW_BLOCK] : 1;
        r.sv = some ? p.vs[a / ADAMW_BLOCK] : 1;
    }
}
template <class X, int BITS, bool NT, bool WHOLE>
__device__ __forceinline__ void adamw_update(const AdamwP& p, const AdamwT& t, const AdamwDyn& h, float factor, long long i, AdamwRaw<BITS>& r) {
    const long long a = t.off + i;
    if (BITS == 8) {
        adamw_decode_m(r.cm, r.sm, r.m);
        adamw_decode_v(r.cv, r.sv, r.v);
    }
    float root[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float g = r.g[k] * factor;
        r.m[k] = p.b1 * r.m[k] + p.c1 * g;
        r.v[k] = p.b2 * r.v[k] + (p.c2 * g) * g;
        // root and reciprocal by the hardware, each off by one unit of the last place: below the rounding of the update itself
        root[k] = __builtin_amdgcn_sqrtf(r.v[k]);
    }
    // The hardware's root of a subnormal v (below 2^-126) is 0.  That moves the denominator by less than 2^-63 inv_bc2: below its rounding with any eps
    // above 2^-38 inv_bc2 (1.2e-10 at b2 = 0.999).  A smaller eps has small v scaled.
    if (__builtin_amdgcn_readfirstlane(h.inv_bc2 * 0x1p-38f > p.eps)) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (r.v[k] < 0x1p-96f) root[k] = __builtin_amdgcn_sqrtf(r.v[k] * 0x1p64f) * 0x1p-32f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float q = r.m[k] * __builtin_amdgcn_rcpf(root[k] * h.inv_bc2 + p.eps);
        r.w[k] = __builtin_fmaf(-h.step_size, q, r.w[k] * h.decay);
    }
    const bool some = WHOLE || i < t.n;
    if (!WHOLE) {                         // what lies behind the tensor's end stays 0 (a factor that is not finite would make it NaN)
#pragma unroll
        for (int k = 0; k < 4; ++k) if (i + k >= t.n) r.m[k] = r.v[k] = r.w[k] = 0.f;
    }
    if (WHOLE) X::template store4<NT>(t.p, i, r.w);
    else for (int k = 0; k < 4; ++k) if (i + k < t.n) adamw_store1<X>(t.p, i + k, r.w[k]);
    if (some && !X::WIDE) AdamwF32::store4<NT>(p.master, a, r.w);
    if (BITS == 32) {
        if (some) { AdamwF32::store4<NT>(p.m, a, r.m); AdamwF32::store4<NT>(p.v, a, r.v); }
        return;
    }
    unsigned um[4], uv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) { um[k] = __float_as_uint(r.m[k]) & 0x7fffffffu; uv[k] = __float_as_uint(r.v[k]); }
    unsigned tm = adamw_max4(um[0], um[1], um[2], um[3]), tv = adamw_max4(uv[0], uv[1], uv[2], uv[3]);
    const bool finite = !__any(tm >= 0x7f800000u || tv >= 0x7f800000u);
    if (!finite) {                        // the scale comes from the values that are
#pragma unroll
        for (int k = 0; k < 4; ++k) { um[k] = adamw_finite_bits(r.m[k]); uv[k] = adamw_finite_bits(r.v[k]); }
        tm = adamw_max4(um[0], um[1], um[2], um[3]);
        tv = adamw_max4(uv[0], uv[1], uv[2], uv[3]);
    }
    const int em = (int)(adamw_row_max(tm) >> 23), ev = (int)(adamw_row_max(tv) >> 23);
    const int sm = em > 8 ? em - 7 : 1, sv = ev > 16 ? ev - 15 : 1;
    const unsigned e0 = (unsigned)i * 0x9E3779B9u + (unsigned)((unsigned long long)i >> 32) * 0x85157AF5u + h.key;
    unsigned cm = 0, cv = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {         // i is a multiple of 4: i + k has the same upper 32 bits
        const unsigned bits = adamw_mix(e0 + (unsigned)k * 0x9E3779B9u);
        cm |= (finite ? adamw_encode_m<true>(r.m[k], sm, bits) : adamw_encode_m<false>(r.m[k], sm, bits)) << (8 * k);
        cv |= (finite ? adamw_encode_v<true>(r.v[k], sv, bits) : adamw_encode_v<false>(r.v[k], sv, bits)) << (8 * k);
    }
    if (some) {
        adamw_st<NT>(static_cast<uint8_t*>(p.m) + a, cm);
        adamw_st<NT>(static_cast<uint8_t*>(p.v) + a, cv);
        if ((threadIdx.x & 15) == 0) {
            p.ms[a / ADAMW_BLOCK] = (uint8_t)sm;
            p.vs[a / ADAMW_BLOCK] = (uint8_t)sv;
        }
    }
}

// One block: a run of 1024 elements of one tensor, four neighbours a thread; what hides the loads is the other blocks of the compute unit.  (2 - 8 runs a
// block, the next one read while one is computed: 654 - 671 us where one takes 634, 132 M fp32 parameters; 362 - 408 against 353 in bf16 with 8-bit moments.)
// Bound: bytes - 28 an element (f32, 32-bit moments), 16 (f32 with 8-bit moments; bf16 with masters and 8-bit moments).  The 8-bit form takes about
// 63 vector instructions an element, just below what its bytes leave room for; wave-wide tests and whole runs without lane conditions made it
// so (125 before: 429 us where it takes 351).  Measured (6.2 TB/s for a large copy): 132 M parameters f32 3.70 GB in 640 us = 5.8 TB/s, bf16 with 8-bit
// moments 2.12 GB in 351 us = 6.0 TB/s; 46 M f32 with 8-bit moments 0.74 GB in 119 us = 6.2 TB/s; 389 K parameters of 14 tensors 5 us.
template <class X, int BITS, bool NT>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwP p) {
    const int ti = adamw_tensor(p);
    if (ti < 0) return;
    const AdamwT t = p.t[ti];
    AdamwDyn d = {t.step_size, t.inv_bc2, t.decay, t.key};
    if (p.dyn) d = p.dyn[t.id];
    const long long first = (long long)(blockIdx.x - t.blk0) * 1024, i = first + threadIdx.x * 4;
    const bool whole = (t.flags & ADAMW_VEC) && first + 1024 <= t.n;
    __shared__ double sh[4];
    AdamwRaw<BITS> r;
    if (whole) adamw_read<X, BITS, NT, true>(p, t, i, r);      // in flight while the sums are added
    const float factor = p.factor ? p.factor[0] : p.parts ? adamw_factor(p.part, p.parts, p.grad_scale, p.max_norm, blockIdx.x ? nullptr : p.norm, sh) : p.grad_scale;
    if (whole) {
        adamw_update<X, BITS, NT, true>(p, t, d, factor, i, r);
    } else {
        adamw_read<X, BITS, NT, false>(p, t, i, r);
        adamw_update<X, BITS, NT, false>(p, t, d, factor, i, r);
    }
}

// Sums of squares in 64 bits (the squares of floats are exact there), one a block; adamw_kernel adds them in their order.  Bound: bytes; about 512
// blocks with 8 loads in flight a thread read 528 MB in 89 us = 5.9 TB/s (one load in flight: 186 us), and leave few sums to add.
template <class X, bool NT>
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
                for (int u = 0; u < U; ++u) X::template load4<NT>(t.g, i + u * 1024, g[u]);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s = fma((double)g[u][k], (double)g[u][k], s);
            }
        }
        for (; i < end; i += 1024) {
            float g[4] = {0.f, 0.f, 0.f, 0.f};
            if (i + 4 <= end && (t.flags & ADAMW_VEC)) X::template load4<NT>(t.g, i, g);
            else for (int k = 0; k < 4; ++k) if (i + k < end) g[k] = adamw_load1<X>(t.g, i + k);
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

// The values that codes stand for, four of each arena a thread: 132 M elements, 1.32 GB in 222 us = 6.0 TB/s.
template <bool NT>
__global__ __launch_bounds__(256) void adamw_unpack_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ ms, const uint8_t* __restrict__ v,
                                                           const uint8_t* __restrict__ vs, float* __restrict__ om, float* __restrict__ ov, long long n4) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) return;
    const unsigned cm = adamw_ld<NT, unsigned>(m + i * 4), cv = adamw_ld<NT, unsigned>(v + i * 4);
    float x[4], y[4];
    adamw_decode_m(cm, ms[i * 4 / ADAMW_BLOCK], x);
    adamw_decode_v(cv, vs[i * 4 / ADAMW_BLOCK], y);
    AdamwF32::store4<NT>(om, i * 4, x);
    AdamwF32::store4<NT>(ov, i * 4, y);
}

}  // namespace mcrn
