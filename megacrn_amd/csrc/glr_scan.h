// glr_scan.h - gated linear recurrence over long sequences, forward and backward (gfx950, wave64).
//
//   a = sigmoid(gate), c = phi(cand):      h_t = h_{t-1} + (1 - a_t)(c_t - h_{t-1})
//   backward, with lam_t the gradient of h_t:   lam_t = dout_t + a_{t+1} lam_{t+1},   lam_{T-1} += dlast
//     dcand = lam (1 - a) phi'(c)      dgate = sum over the gate's channels of lam a (1 - a)(h_{t-1} - c)      dstate = a_0 lam_0
//
// Both directions are first-order recurrences y' = A y + X whose maps compose: (A1, X1) then (A2, X2) = (A1 A2, A2 X1 + X2).
// A block of 256 threads covers CL channel lanes (V channels each) x SEG = 256 / CL time segments of GLR_K steps.  A thread loads
// its GLR_K steps into registers, reduces them to one map, the block composes the SEG maps through LDS, and the thread runs its steps
// again from the state that enters its segment: every input is read from HBM once, whatever SEG is.  The block walks the time axis
// tile by tile (SEG * GLR_K steps), the loads of the next tile in flight while the current one is computed.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "glr_scan_api.h"

namespace mcrn {

constexpr int GLR_THREADS = 256;

// ---- storage types --------------------------------------------------------------------------------------------------
struct GlrF32 {
    typedef float S;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
struct GlrBf16 {
    typedef uint16_t S;
    static __device__ __forceinline__ float up(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ uint16_t down(float f) {          // round to nearest even; NaN stays NaN
        uint32_t u = __float_as_uint(f);
        if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
        return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
    }
};
struct GlrF16 {
    typedef _Float16 S;
    static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 down(float f) { return (_Float16)f; }
};

template <class X, int V> struct alignas(sizeof(typename X::S) * V) GlrVec { typename X::S e[V]; };

template <class X, int V> __device__ __forceinline__ GlrVec<X, V> glr_load(const void* p, long long at) {
    return *reinterpret_cast<const GlrVec<X, V>*>(static_cast<const typename X::S*>(p) + at);
}
template <class X, int V> __device__ __forceinline__ void glr_store(void* p, long long at, const float* v) {
    GlrVec<X, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.e[i] = X::down(v[i]);
    *reinterpret_cast<GlrVec<X, V>*>(static_cast<typename X::S*>(p) + at) = r;
}

// ---- the functions of a step -----------------------------------------------------------------------------------------
__device__ __forceinline__ float glr_exp(float x) {       // e^x, x <= 0, ~1 ulp: the product x log2(e) carries its rounding error along
    const float L2E = 1.44269502162933349609f, L2E_LO = 1.92596299112661746887e-8f;    // log2(e) = L2E + L2E_LO
    const float t = x * L2E;
    const float lo = fmaf(x, L2E_LO, fmaf(x, L2E, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return t < -126.f ? 0.f : fmaf(e, lo * 0.693147182464599609375f, e);
}
// sigmoid(-|g|) with the sign of g: z.  1 - a = z > 0 ? z : 1 + z, a (1 - a) = |z| - z^2; neither form cancels.
__device__ __forceinline__ float glr_z(float g) {
    const float e = glr_exp(-fabsf(g));
    return copysignf(e * __builtin_amdgcn_rcpf(1.f + e), g);
}
__device__ __forceinline__ float glr_w(float z) { return (int)__float_as_uint(z) >= 0 ? z : 1.f + z; }
__device__ __forceinline__ float glr_tanh(float u) {
    const float e = glr_exp(-2.f * fabsf(u));
    const float far = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), u);
    const float q = u * u;                                // near 0 the quotient cancels: Taylor's series to u^11, off by < 2^-25 below 0.35
    float s = fmaf(q, -1382.f / 155925.f, 62.f / 2835.f);
    s = fmaf(q, s, -17.f / 315.f);
    s = fmaf(q, s, 2.f / 15.f);
    s = fmaf(q, s, -1.f / 3.f);
    return fabsf(u) < 0.35f ? fmaf(u * q, s, u) : far;
}

// ---- where a thread works ----------------------------------------------------------------------------------------------
struct GlrAt {
    int b, chunk, cl, seg, t0, t1;
    int n, ch;                 // node and first channel of the thread's V channels
    int gi, gl, part;          // its gate's index in (.., G), its lane among the gate's lanes, its part
    bool active;
};
template <int V, int CL, bool SHARED> __device__ __forceinline__ GlrAt glr_where(const GlrP& p) {
    GlrAt w;
    unsigned blk = blockIdx.x;
    const unsigned tile = blk % (unsigned)p.tiles;
    blk /= (unsigned)p.tiles;
    w.b = (int)(blk % (unsigned)p.B);
    w.chunk = (int)(blk / (unsigned)p.B) + p.first;
    w.cl = (int)threadIdx.x % CL;
    w.seg = (int)threadIdx.x / CL;
    w.t0 = w.chunk * p.chunk;
    w.t1 = min(p.T, w.t0 + p.chunk);
    if (SHARED) {              // L lanes a (gate, part): channels behind the gate's last stay idle
        const long long unit = (long long)tile * (CL / p.L) + w.cl / p.L;
        const int D = p.H / p.G;
        w.gl = w.cl % p.L;
        w.part = (int)(unit % p.parts);
        const long long ng = unit / p.parts;
        const int d = (w.part * p.L + w.gl) * V;
        w.active = ng < (long long)p.N * p.G && d < D;
        w.n = w.active ? (int)(ng / p.G) : 0;
        w.gi = w.active ? (int)(ng % p.G) : 0;
        w.ch = w.active ? w.gi * D + d : 0;
    } else {
        const long long q = (long long)tile * CL + w.cl;
        const int hv = p.H / V;
        w.active = q < p.nq;
        w.n = w.active ? (int)(q / hv) : 0;
        w.ch = w.active ? (int)(q % hv) * V : 0;
        w.gi = w.ch;
        w.gl = 0;
        w.part = 0;
    }
    return w;
}

// The maps of the block's SEG segments, composed: `enter` = what reaches the thread's segment when `carry` reaches the tile's first one
// (its last, REV), and carry = what leaves the tile.  A[], X[] = the thread's own map.  lds: SEG x CL x V pairs, its own in every other call.
template <int V, int CL, bool REV>
__device__ __forceinline__ void glr_block_scan(float2* lds, int cl, int seg, const float* A, const float* X, float* carry, float* enter) {
    constexpr int SEG = GLR_THREADS / CL;
#pragma unroll
    for (int i = 0; i < V; ++i) lds[(seg * V + i) * CL + cl] = make_float2(A[i], X[i]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float h = carry[i], e = h;
#pragma unroll
        for (int j = 0; j < SEG; ++j) {
            const int s = REV ? SEG - 1 - j : j;
            const float2 m = lds[(s * V + i) * CL + cl];
            e = s == seg ? h : e;
            h = fmaf(m.x, h, m.y);
        }
        enter[i] = e;
        carry[i] = h;
    }
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// AGG: only the chunk's map is wanted (agg[chunk][b][A | X][N*H]); otherwise the chunk starts from the state that the maps of the chunks before it give.
template <class X, int V, int CL, bool SHARED, bool AGG>
__global__ __launch_bounds__(GLR_THREADS) void glr_fwd_kernel(GlrP p) {
    constexpr int K = GLR_K, SEG = GLR_THREADS / CL, VG = SHARED ? 1 : V;
    __shared__ float2 lds[SEG > 1 ? 2 : 1][SEG > 1 ? SEG * CL * V : 1];
    const GlrAt w = glr_where<V, CL, SHARED>(p);
    const long long NH = (long long)p.N * p.H, hoff = (long long)w.n * p.H + w.ch;
    const long long g_at = w.b * p.g_sb + w.n * p.g_sn + w.gi, c_at = w.b * p.c_sb + w.n * p.c_sn + w.ch, m_at = w.b * p.m_sb + w.n * p.m_sn;
    int par = 0;

    float carry[V], prod[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { carry[i] = 0.f; prod[i] = 1.f; }
    if (!AGG) {
        if (p.h0 && w.active) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = p.h0[w.b * NH + hoff + i];
        }
        for (int j = 0; j < w.chunk; ++j) {               // the chunks before this one
            const float* g = p.agg + ((long long)j * p.B + w.b) * 2 * NH + hoff;
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = fmaf(g[i], carry[i], g[NH + i]);
        }
    }

    GlrVec<X, VG> rg[K];
    GlrVec<X, V> rc[K];
    uint8_t rm[K];
    auto fetch = [&](int tb) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int t = min(tb + w.seg * K + k, w.t1 - 1);
            rg[k] = glr_load<X, VG>(p.gate, g_at + t * p.g_st);
            rc[k] = glr_load<X, V>(p.cand, c_at + t * p.c_st);
            rm[k] = p.mask ? p.mask[m_at + t * p.m_st] : (uint8_t)1;
        }
    };
    if (w.t0 < w.t1) fetch(w.t0);
    for (int tb = w.t0; tb < w.t1; tb += SEG * K) {
        const int ts = tb + w.seg * K;
        float ww[K][V], cc[K][V];                         // 1 - a and phi(cand); a masked step is w = 0, c = 0
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool on = rm[k] != 0 && ts + k < w.t1;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float wi = (SHARED && i) ? ww[k][0] : glr_w(glr_z(X::up(rg[k].e[SHARED ? 0 : i])));
                ww[k][i] = on ? wi : 0.f;
                cc[k][i] = on ? X::up(rc[k].e[i]) : 0.f;
            }
        }
        if (tb + SEG * K < w.t1) fetch(tb + SEG * K);
        if (p.act) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) cc[k][i] = glr_tanh(cc[k][i]);
        }
        float h[V];
        if (SEG > 1 || AGG) {
            float A[V], Xl[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A[i] = 1.f; Xl[i] = 0.f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    A[i] = fmaf(-ww[k][i], A[i], A[i]);
                    Xl[i] = fmaf(ww[k][i], cc[k][i] - Xl[i], Xl[i]);
                }
            }
            if (AGG) {
                if (SEG == 1) {
#pragma unroll
                    for (int i = 0; i < V; ++i) { carry[i] = fmaf(A[i], carry[i], Xl[i]); prod[i] *= A[i]; }
                } else {
                    // the product of the tile's A: the same composition from carry 1 with X = 0
                    float none[V], dummy[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) none[i] = 0.f;
                    glr_block_scan<V, CL, false>(lds[par], w.cl, w.seg, A, Xl, carry, dummy);
                    par ^= 1;
                    glr_block_scan<V, CL, false>(lds[par], w.cl, w.seg, A, none, prod, dummy);
                    par ^= 1;
                }
                continue;
            }
            glr_block_scan<V, CL, false>(lds[par], w.cl, w.seg, A, Xl, carry, h);
            par ^= 1;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) h[i] = carry[i];
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < V; ++i) h[i] = fmaf(ww[k][i], cc[k][i] - h[i], h[i]);
            const int t = ts + k;
            if (w.active && t < w.t1 && p.out) glr_store<X, V>(p.out, ((long long)w.b * p.T + t) * NH + hoff, h);
        }
        if (p.ckpt && w.active && ts + K < p.T) {         // the state before step ts + K
            const long long nck = (p.T - 1) / K;
            glr_store<GlrF32, V>(p.ckpt, ((long long)w.b * nck + ts / K) * NH + hoff, h);
        }
        if (SEG == 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = h[i];
        }
    }
    if (!w.active || w.seg != 0) return;
    if (AGG) {
        float* g = p.agg + ((long long)w.chunk * p.B + w.b) * 2 * NH + hoff;
#pragma unroll
        for (int i = 0; i < V; ++i) { g[i] = prod[i]; g[NH + i] = carry[i]; }
    } else if (p.last && w.chunk == p.S - 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) p.last[w.b * NH + hoff + i] = carry[i];
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------
// Walks the time axis from its end; `carry` is mu_{t+1} = a_{t+1} lam_{t+1}, what reaches step t from the steps behind it.
template <class X, int V, int CL, bool SHARED, bool AGG>
__global__ __launch_bounds__(GLR_THREADS) void glr_bwd_kernel(GlrP p) {
    constexpr int K = GLR_K, SEG = GLR_THREADS / CL, VG = SHARED ? 1 : V;
    __shared__ float2 lds[SEG > 1 ? 2 : 1][SEG > 1 ? SEG * CL * V : 1];
    const GlrAt w = glr_where<V, CL, SHARED>(p);
    const long long NH = (long long)p.N * p.H, hoff = (long long)w.n * p.H + w.ch;
    const long long g_at = w.b * p.g_sb + w.n * p.g_sn + w.gi, c_at = w.b * p.c_sb + w.n * p.c_sn + w.ch, m_at = w.b * p.m_sb + w.n * p.m_sn;
    const long long d_at = w.b * p.d_sb + w.n * p.d_sn + w.ch, nck = (p.T - 1) / K;
    int par = 0;

    float carry[V], prod[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { carry[i] = 0.f; prod[i] = 1.f; }
    if (!AGG) {
        if (p.dlast && w.active) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = p.dlast[w.b * NH + hoff + i];
        }
        for (int j = p.S - 1; j > w.chunk; --j) {         // the chunks behind this one
            const float* g = p.agg + ((long long)j * p.B + w.b) * 2 * NH + hoff;
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = fmaf(g[i], carry[i], g[NH + i]);
        }
    }

    GlrVec<X, VG> rg[K];
    GlrVec<X, V> rc[K], rd[K];
    GlrVec<GlrF32, V> rs;                                 // the state before the segment's first step
    uint8_t rm[K];
    auto fetch = [&](int tb) {
        const int ts = tb + w.seg * K;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int t = min(ts + k, w.t1 - 1);
            rg[k] = glr_load<X, VG>(p.gate, g_at + t * p.g_st);
            if (!AGG) rc[k] = glr_load<X, V>(p.cand, c_at + t * p.c_st);
            if (p.dout) rd[k] = glr_load<X, V>(p.dout, d_at + t * p.d_st);
            rm[k] = p.mask ? p.mask[m_at + t * p.m_st] : (uint8_t)1;
        }
        if (!AGG) {
#pragma unroll
            for (int i = 0; i < V; ++i) rs.e[i] = 0.f;
            if (ts == 0) {
                if (p.h0) rs = glr_load<GlrF32, V>(p.h0, w.b * NH + hoff);
            } else if (ts < w.t1) {                       // f32: out_{ts-1} is that state
                rs = p.dtype == GLR_F32 ? glr_load<GlrF32, V>(p.out, ((long long)w.b * p.T + ts - 1) * NH + hoff)
                                        : glr_load<GlrF32, V>(p.ckpt, ((long long)w.b * nck + ts / K - 1) * NH + hoff);
            }
        }
    };
    const int span = SEG * K, ntile = (w.t1 - w.t0 + span - 1) / span;
    if (ntile > 0) fetch(w.t0 + (ntile - 1) * span);
    for (int it = ntile - 1; it >= 0; --it) {
        const int tb = w.t0 + it * span, ts = tb + w.seg * K;
        float ww[K][V], wc[K][V], q[K][V], dd[K][V];      // 1 - a, its product with phi', a (1 - a)(h_{t-1} - c), dout
        float h[V];
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = AGG ? 0.f : rs.e[i];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool in = ts + k < w.t1, on = rm[k] != 0 && in;
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!SHARED || i == 0) z = on ? glr_z(X::up(rg[k].e[SHARED ? 0 : i])) : 0.f;
                ww[k][i] = glr_w(z);
                q[k][i] = fmaf(-z, z, fabsf(z));
                dd[k][i] = in && p.dout ? X::up(rd[k].e[i]) : 0.f;
                wc[k][i] = !AGG && on ? X::up(rc[k].e[i]) : 0.f;
            }
        }
        if (it > 0) fetch(tb - span);
        if (!AGG && p.act) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) wc[k][i] = glr_tanh(wc[k][i]);
        }
        if (!AGG) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float c = wc[k][i], diff = c - h[i];
                    q[k][i] *= -diff;
                    h[i] = fmaf(ww[k][i], diff, h[i]);
                    wc[k][i] = p.act ? ww[k][i] * fmaf(-c, c, 1.f) : ww[k][i];
                }
        }
        float mu[V];
        if (SEG > 1 || AGG) {
            float A[V], Xl[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A[i] = 1.f; Xl[i] = 0.f;
#pragma unroll
                for (int k = K - 1; k >= 0; --k) {
                    A[i] = fmaf(-ww[k][i], A[i], A[i]);
                    const float lam = Xl[i] + dd[k][i];
                    Xl[i] = fmaf(-ww[k][i], lam, lam);
                }
            }
            if (AGG) {
                if (SEG == 1) {
#pragma unroll
                    for (int i = 0; i < V; ++i) { carry[i] = fmaf(A[i], carry[i], Xl[i]); prod[i] *= A[i]; }
                } else {
                    float none[V], dummy[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) none[i] = 0.f;
                    glr_block_scan<V, CL, true>(lds[par], w.cl, w.seg, A, Xl, carry, dummy);
                    par ^= 1;
                    glr_block_scan<V, CL, true>(lds[par], w.cl, w.seg, A, none, prod, dummy);
                    par ^= 1;
                }
                continue;
            }
            glr_block_scan<V, CL, true>(lds[par], w.cl, w.seg, A, Xl, carry, mu);
            par ^= 1;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) mu[i] = carry[i];
        }
#pragma unroll
        for (int k = K - 1; k >= 0; --k) {
            const int t = ts + k;
            float dc[V], dg[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float lam = mu[i] + dd[k][i];
                dc[i] = lam * wc[k][i];
                dg[i] = lam * q[k][i];
                mu[i] = fmaf(-ww[k][i], lam, lam);
            }
            const long long row = ((long long)w.b * p.T + t) * p.N + w.n;
            if (w.active && t < w.t1) glr_store<X, V>(p.dcand, row * p.H + w.ch, dc);
            if (!SHARED) {
                if (w.active && t < w.t1) glr_store<X, VG>(p.dgate, row * p.G + w.gi, dg);
            } else {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) s += w.active ? dg[i] : 0.f;
                for (int o = p.L >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
                if (w.active && w.gl == 0 && t < w.t1) {
                    if (p.parts == 1) glr_store<X, 1>(p.dgate, row * p.G + w.gi, &s);
                    else p.part[(row * p.G + w.gi) * p.parts + w.part] = s;
                }
            }
        }
        if (SEG == 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = mu[i];
        }
    }
    if (!w.active || w.seg != 0) return;
    if (AGG) {
        float* g = p.agg + ((long long)w.chunk * p.B + w.b) * 2 * NH + hoff;
#pragma unroll
        for (int i = 0; i < V; ++i) { g[i] = prod[i]; g[NH + i] = carry[i]; }
    } else if (p.dstate && w.chunk == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) p.dstate[w.b * NH + hoff + i] = carry[i];
    }
}

// the parts of a gate whose channels fill more than one wave, added in their order
template <class X>
__global__ void glr_parts_kernel(const float* __restrict__ part, int parts, long long n, void* __restrict__ dgate) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
    for (int j = 0; j < parts; ++j) s += part[i * parts + j];
    glr_store<X, 1>(dgate, i, &s);
}

}  // namespace mcrn
