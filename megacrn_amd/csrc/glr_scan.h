// glr_scan.h - gated linear recurrence over long sequences, forward and backward (gfx950, wave64).
//
//   a = sigmoid(gate), c = phi(cand):      h_t = a_t h_{t-1} + (1 - a_t) c_t
//   backward, with lam_t the gradient of h_t:   lam_t = dout_t + a_{t+1} lam_{t+1},   lam_{T-1} += dlast
//     dcand = lam (1 - a) phi'(c)      dgate = sum over the gate's channels of lam a (1 - a)(h_{t-1} - c)      dstate = a_0 lam_0
//
// Both directions are first-order recurrences y' = A y + X whose maps compose: (A1, X1) then (A2, X2) = (A1 A2, A2 X1 + X2).
// A block of 256 threads covers CL channel lanes (V channels each) x SEG = 256 / CL time segments of K steps.  A thread loads its K
// steps into registers, reduces them to one map, the block composes the SEG maps (lanes of a wave by row swaps, waves through LDS),
// and the thread runs its steps from the state that enters its segment: every input is read from HBM once, whatever SEG is.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "glr_scan_api.h"

namespace mcrn {

constexpr int GLR_THREADS = 256;
// the scheduler does not move work across: a phase's temporaries die before the next one's live (else occupancy falls by a wave)
#define GLR_PHASE() __builtin_amdgcn_sched_barrier(0)
// a value is computed here and not where it is used: moved behind the wait, it would keep all its operands in registers
#define GLR_HERE(x) asm volatile("" : "+v"(x))
enum { GLR_WALK = 0, GLR_AGG = 1, GLR_CHAIN = 2 };

// ---- storage types --------------------------------------------------------------------------------------------------
struct GlrF32 {
    typedef float S;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
struct GlrBf16 {
    typedef __bf16 S;
    static __device__ __forceinline__ float up(__bf16 v) { return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, v) << 16); }
    static __device__ __forceinline__ __bf16 down(float f) { return (__bf16)f; }     // to the nearest, ties to even, by the hardware
};
struct GlrF16 {
    typedef _Float16 S;
    static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 down(float f) { return (_Float16)f; }
};

// aligned to its elements only (global memory takes any alignment): what rows of any length need
template <class X, int V> struct GlrVec { typename X::S e[V]; };

// element i; a pair of bf16 is taken apart in its 32-bit word
template <class X, int V> __device__ __forceinline__ float glr_up(const GlrVec<X, V>& r, int i) { return X::up(r.e[i]); }
template <> __device__ __forceinline__ float glr_up<GlrBf16, 4>(const GlrVec<GlrBf16, 4>& r, int i) {
    const uint2 w = __builtin_bit_cast(uint2, r);
    const uint32_t u = i < 2 ? w.x : w.y;
    return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
}
// Addresses: a base that is the same for the whole block (scalar registers, advanced by scalar adds) + 32 bits of a lane's own bytes
template <class X, int V> __device__ __forceinline__ GlrVec<X, V> glr_load(const char* base, uint32_t off) {
    return *reinterpret_cast<const GlrVec<X, V>*>(base + off);
}
template <int BYTES> struct GlrWord { typedef uint32_t T __attribute__((ext_vector_type(BYTES / 4))); };
template <> struct GlrWord<4> { typedef uint32_t T; };
template <> struct GlrWord<2> { typedef uint16_t T; };
// r where `on`, else zeros: pairs of 16-bit elements are not taken apart for it
template <class X, int V> __device__ __forceinline__ void glr_only(bool on, GlrVec<X, V>& r) {
    typedef typename GlrWord<sizeof(r)>::T T;
    T w = __builtin_bit_cast(T, r);
    if constexpr (sizeof(r) > 4) {
#pragma unroll
        for (unsigned j = 0; j < sizeof(r) / 4; ++j) w[j] = on ? w[j] : 0u;
    } else {
        w = on ? w : (T)0;
    }
    r = __builtin_bit_cast(GlrVec<X, V>, w);
}
// NT: past the caches, for sequences larger than these; `on`: else zeros
template <class X, int V, bool NT = false> __device__ __forceinline__ void glr_store(char* base, uint32_t off, const float* v, bool on = true) {
    GlrVec<X, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.e[i] = X::down(v[i]);
    glr_only<X, V>(on, r);
    typedef typename GlrWord<sizeof(r)>::T T;
    typedef T Loose __attribute__((aligned(sizeof(typename X::S))));
    if (NT) __builtin_nontemporal_store(__builtin_bit_cast(T, r), reinterpret_cast<Loose*>(base + off));
    else *reinterpret_cast<GlrVec<X, V>*>(base + off) = r;
}
struct GlrYes { static constexpr bool value = true; };
struct GlrNo { static constexpr bool value = false; };
// K rows of a thread, from row seg * K of the tile on.  What lies behind the tile's last row `end` reads that one instead: one minimum a
// row.  ONCE (no loop around it): whole tiles go without, by scalar bases (in a loop the second path costs registers, and spills).
template <class X, int V, int K, bool ONCE>
__device__ __forceinline__ void glr_rows(GlrVec<X, V>* r, const char* base, uint32_t lane, uint32_t st, int seg, bool full, int end) {
    if (ONCE && full) {
        const uint32_t off = lane + (uint32_t)(seg * K) * st;
#pragma unroll
        for (int k = 0; k < K; ++k) r[k] = glr_load<X, V>(base + (uint64_t)k * st, off);
    } else {
        uint32_t off = lane + (uint32_t)(seg * K) * st, most = 0xffffffffu;
        if (!full) {
            const int at = min(seg * K, end);
            off = lane + (uint32_t)at * st;
            most = (uint32_t)(end - at) * st;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const uint32_t o = (uint32_t)k * st;
            r[k] = glr_load<X, V>(base, off + (o < most ? o : most));
        }
    }
}
struct GlrByte {
    typedef uint8_t S;
};

// Steps that keep the state - masked, or behind the last one (`left` steps are there): bit k of a word is 1 where step k moves it, and the candidate of
// one that does not becomes 0.  FLAT: a word for each channel, since these may belong to two nodes (`over` of them to the second, rn); their candidates
// become 0 behind the conversion (elements of a pair are not taken apart for it).
template <int V, bool FLAT> struct GlrMoves {
    unsigned w[FLAT ? V : 1];
    __device__ __forceinline__ bool at(int k, int i) const { return (w[FLAT ? i : 0] >> k) & 1u; }
};
template <class X, int V, int K, bool FLAT>
__device__ __forceinline__ void glr_masked(GlrMoves<V, FLAT>& m, int left, bool mask, int over, const GlrVec<GlrByte, 1>* rm, const GlrVec<GlrByte, 1>* rn,
                                           GlrVec<X, V>* rc) {
    unsigned one = 0, two = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        one |= (k < left && (!mask || rm[k].e[0] != 0) ? 1u : 0u) << k;
        if (FLAT) two |= (k < left && (!mask || rn[k].e[0] != 0) ? 1u : 0u) << k;
        if (!FLAT) glr_only<X, V>((one >> k) & 1u, rc[k]);
    }
    m.w[0] = one;
    if (FLAT) {
#pragma unroll
        for (int i = 0; i < V; ++i) m.w[i] = V - i > over ? one : two;
    }
}

// ---- the functions of a step -----------------------------------------------------------------------------------------
// The arithmetic is fp32 whatever the inputs' type: the states behind it are.
// e^x, x <= 0.  The rounding of t = x log2 e would be an error of |x| u; x - t ln 2 is what it left out.  The factor is above log2 e by a little more than
// that rounding, so the rest is never negative and a clamp to [0, 1] (part of the instruction) only drops the NaN of an infinite x.  Off by 4 u, 7 u below -17.
__device__ __forceinline__ float glr_exp(float x) {
    const float t = x * 1.44269514083862304688f, e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, __builtin_amdgcn_fmed3f(fmaf(t, -0.693147182464599609375f, x), 0.f, 1.f), e);
}
// A gate is held as n: |n| is the smaller one of a = sigmoid(g) and w = 1 - a, with the relative error of the exponential (which cannot overflow)
// however little is kept or forgotten; the sign is g's.  The larger one is 1 - |n| and never formed: a x = x - |n| x for an open gate (n >= 0),
// |n| x for a closed one.  GLR_HOLD is the closed gate with a = 1, a step that is masked: it keeps x whatever x is, infinities among it.  (a formed as 1 - w has lost all its bits at g = -17, w formed as 1 - a at g = 17.)
__device__ __forceinline__ float glr_gate(float g) {
    const float e = glr_exp(-fabsf(g));
    return copysignf(e * __builtin_amdgcn_rcpf(1.f + e), g);
}
constexpr float GLR_HOLD = -1.f;
// Open: x, closed: y - by the sign's mask and one bit-select (the empty statement keeps the compiler from comparing, twice, and selecting through VCC)
__device__ __forceinline__ float glr_pick(float n, float x, float y) {
    int closed = (int)__float_as_uint(n) >> 31;
    asm("" : "+v"(closed));
    return __uint_as_float(((unsigned)closed & __float_as_uint(y)) | (~(unsigned)closed & __float_as_uint(x)));
}
// w = 1 - a, and a w: the larger one of a and w has all its bits as 1 - |n|
__device__ __forceinline__ float glr_w(float n) { return glr_pick(n, 0.f, 1.f) + n; }
__device__ __forceinline__ float glr_aw(float n) { return fmaf(-fabsf(n), fabsf(n), fabsf(n)); }
// a x
__device__ __forceinline__ float glr_keep(float n, float x) { return fmaf(-n, x, glr_pick(n, x, 0.f)); }
constexpr float GLR_2L2E = 2.88539004325866699219f;        // 2 log2(e)
// 1 - 2 / (1 + e^2u): off by 3 units of 2^-24 whatever u is, which shows relatively near 0: below 3/8 the odd polynomial of degree 7 whose largest
// relative error there is smallest (1.2 u, 2.2 u with its roundings; the coefficients by linear programming over 3000 Chebyshev points).
__device__ __forceinline__ float glr_tanh(float u) {
    const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * GLR_2L2E)), 1.f);
    const float q = u * u;
    const float s = fmaf(q, fmaf(q, -0.04848729074001312256f, 0.13289725780487060547f), -0.33332332968711853027f);
    return fabsf(u) < 0.375f ? fmaf(u * q, s, u) : far;
}

// c - h, what a step goes towards; where it goes nowhere (n = +0: a gate that is wholly open) an infinite state stays what it is
__device__ __forceinline__ float glr_diff(float n, float c, float h) { return c - (__float_as_uint(n) == 0u ? 0.f : h); }
// a h + w c, as h + w (c - h) or as c - a (c - h)
__device__ __forceinline__ float glr_next(float n, float c, float h, float diff) { return fmaf(n, diff, glr_pick(n, h, c)); }

// ---- where a thread works ----------------------------------------------------------------------------------------------
struct GlrAt {
    int b, chunk, cl, seg, t0, t1;
    int n, ch;                 // node and first channel of the thread's V channels
    int n2;                    // node of the last one (FLAT)
    int gi, gl, part;          // its gate's index in (.., G), its lane among the gate's lanes, its part
    bool active;
};
// CHAIN: the chunk is the next one of the block's channels that no block has taken yet, so that the block which has to hand over the
// state has started before; REV: from the last chunk on
template <int V, int CL, int GATES, bool CHAIN, bool REV> __device__ __forceinline__ GlrAt glr_where(const GlrP& p) {
    GlrAt w;
    unsigned blk = blockIdx.x;
    const unsigned tile = blk % (unsigned)p.tiles;
    blk /= (unsigned)p.tiles;
    w.b = (int)(blk % (unsigned)p.B);
    __shared__ int taken;
    int mine = 0;
    if (CHAIN && threadIdx.x == 0) mine = (int)atomicAdd(p.ticket + (tile + (unsigned)w.b * (unsigned)p.tiles), 1u);
    w.cl = (int)threadIdx.x % CL;
    w.seg = (int)threadIdx.x / CL;
    if (GATES == GLR_SHARED) { // L lanes a (gate, part): channels behind the gate's last stay idle
        const unsigned unit = tile * (unsigned)(CL / p.L) + w.cl / p.L;
        const int D = p.H / p.G;
        w.gl = w.cl % p.L;
        w.part = (int)(unit % (unsigned)p.parts);
        const unsigned ng = unit / (unsigned)p.parts;
        const int d = (w.part * p.L + w.gl) * V;
        w.active = ng < (unsigned)p.N * (unsigned)p.G && d < D;
        w.n = w.active ? (int)(ng / (unsigned)p.G) : 0;
        w.gi = w.active ? (int)(ng % (unsigned)p.G) : 0;
        w.ch = w.active ? w.gi * D + d : 0;
    } else if (GATES == GLR_FLAT) {      // channels of all nodes behind one another; the last vector reaches back over the one before
        const unsigned q = tile * CL + w.cl, NH = (unsigned)p.N * (unsigned)p.H;
        w.active = q < (unsigned)p.nq;
        const unsigned c = w.active ? min(q * V, NH - V) : 0u;
        w.n = (int)(c / (unsigned)p.H);
        w.ch = (int)(c % (unsigned)p.H);
        w.n2 = w.ch + V > p.H ? w.n + 1 : w.n;
        w.gi = w.ch;
        w.gl = 0;
        w.part = 0;
    } else {
        const unsigned q = tile * CL + w.cl, hv = p.H / V;
        w.active = q < (unsigned)p.nq;
        w.n = w.active ? (int)(q / hv) : 0;
        w.ch = w.active ? (int)(q % hv) * V : 0;
        w.gi = w.ch;
        w.gl = 0;
        w.part = 0;
    }
    if (CHAIN) {
        if (threadIdx.x == 0) taken = mine;
        __syncthreads();
        w.chunk = __builtin_amdgcn_readfirstlane(taken);
        if (REV) w.chunk = p.S - 1 - w.chunk;
    } else {
        w.chunk = (int)(blk / (unsigned)p.B) + p.first;
    }
    w.t0 = w.chunk * p.chunk;
    w.t1 = min(p.T, w.t0 + p.chunk);
    return w;
}

// ---- composing the maps of a block's segments ---------------------------------------------------------------------------
__device__ __forceinline__ float glr_f(unsigned u) { return __uint_as_float(u); }
__device__ __forceinline__ unsigned glr_u(float f) { return __float_as_uint(f); }

// First part: the thread's own map A[], X[] -> EA[], EX[], the wave's segments before the thread's (behind it, REV), and the waves' maps in
// lds (GLR_THREADS / 64 x CL x V pairs, its own in every other call).
template <int V, int CL, bool REV>
__device__ __forceinline__ void glr_scan_maps(float2* lds, int cl, const float* A, const float* X, float* EA, float* EX) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const bool odd = threadIdx.x & 16, upper = threadIdx.x & 32;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float TA = A[i], TX = X[i];
        EA[i] = 1.f; EX[i] = 0.f;
        if (CL == 16) {                                    // four segments a wave, one in each row of 16 lanes
            const auto sa = __builtin_amdgcn_permlane16_swap(glr_u(TA), glr_u(TA), false, false);      // even rows' values, odd rows' values
            const auto sx = __builtin_amdgcn_permlane16_swap(glr_u(TX), glr_u(TX), false, false);
            const float a0 = glr_f(sa[0]), a1 = glr_f(sa[1]), x0 = glr_f(sx[0]), x1 = glr_f(sx[1]);
            const bool second = REV ? !odd : odd;
            const float ea = second ? (REV ? a1 : a0) : 1.f, ex = second ? (REV ? x1 : x0) : 0.f;
            const float pa = a0 * a1, px = REV ? fmaf(a0, x1, x0) : fmaf(a1, x0, x1);
            const auto qa = __builtin_amdgcn_permlane32_swap(glr_u(pa), glr_u(pa), false, false);
            const auto qx = __builtin_amdgcn_permlane32_swap(glr_u(px), glr_u(px), false, false);
            const float b0 = glr_f(qa[0]), b1 = glr_f(qa[1]), y0 = glr_f(qx[0]), y1 = glr_f(qx[1]);
            const bool later = REV ? !upper : upper;
            EX[i] = later ? fmaf(ea, REV ? y1 : y0, ex) : ex;
            EA[i] = later ? ea * (REV ? b1 : b0) : ea;
            TA = b0 * b1;
            TX = REV ? fmaf(b0, y1, y0) : fmaf(b1, y0, y1);
        }
        if (CL == 64 || (threadIdx.x & 63) < CL) lds[(wave * V + i) * CL + cl] = make_float2(TA, TX);
        GLR_PHASE();
    }
    __syncthreads();
}
// Second part: `enter` = what reaches the thread's segment when `carry` reaches the tile's first one (its last, REV); carry = what leaves the
// tile; prod *= the product of all A (AGG).
template <int V, int CL, bool REV, bool AGG>
__device__ __forceinline__ void glr_scan_carry(const float2* lds, int cl, const float* EA, const float* EX, float* carry, float* prod, float* enter) {
    constexpr int W = GLR_THREADS / 64;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float h = carry[i], e = h;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int s = REV ? W - 1 - j : j;
            const float2 m = lds[(s * V + i) * CL + cl];
            if (s == wave) e = h;
            h = fmaf(m.x, h, m.y);
            if (AGG) prod[i] *= m.x;
        }
        enter[i] = CL == 16 ? fmaf(EA[i], e, EX[i]) : e;
        carry[i] = h;
        GLR_PHASE();
    }
}

// Splits (WALK with more than one chunk): carry = what the maps of `n` chunks, one behind the other in the order of the walk, make of it.
// The segments' threads take a run of chunks each, then the runs are composed as segments are.  at: the first one's A, X at at[NH];
// step: from one to the next.
template <int V, int CL>
__device__ __forceinline__ void glr_chunks_before(float2* lds, const GlrAt& w, const float* at, long long step, long long NH, int n, float* carry) {
    constexpr int SEG = GLR_THREADS / CL;
    const int per = (n + SEG - 1) / SEG, j0 = w.seg * per, j1 = min(n, j0 + per);
    float A[V], X[V], EA[V], EX[V], none[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { A[i] = 1.f; X[i] = 0.f; }
#pragma unroll 4
    for (int j = j0; j < j1; ++j) {
        const float* g = at + j * step;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float a = g[i], x = g[NH + i];
            X[i] = fmaf(a, X[i], x);
            A[i] *= a;
        }
    }
    glr_scan_maps<V, CL, false>(lds, w.cl, A, X, EA, EX);
    glr_scan_carry<V, CL, false, false>(lds, w.cl, EA, EX, carry, none, none);
}

// ---- handing the state from block to block (CHAIN) ------------------------------------------------------------------------
// A word of all ones says that the state is not there yet (a state of that NaN pattern is sent as the usual NaN).  Each word is valid by
// itself: no fence, no flag.  The wait ends: see glr_where; the bound only turns a broken workspace into NaN instead of a hang.
template <int V> __device__ __forceinline__ void glr_send(unsigned* at, const float* v) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const unsigned u = glr_u(v[i]);
        __hip_atomic_store(at + i, u == 0xffffffffu ? 0x7fc00000u : u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
template <int V> __device__ __forceinline__ void glr_receive(const unsigned* at, float* v) {
    for (int tries = 0; tries < (1 << 22); ++tries) {
        bool there = true;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const unsigned u = __hip_atomic_load(at + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            v[i] = glr_f(u);
            there = there && u != 0xffffffffu;
        }
        if (there) return;
        __builtin_amdgcn_s_sleep(2);
    }
}
__global__ void glr_clear_kernel(unsigned* __restrict__ words, long long tickets, long long n) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) words[i] = i < tickets ? 0u : 0xffffffffu;
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// Bound: bytes (gate, cand in, out out) for f32, vector instructions for the 16-bit types, whose bytes are half: a step takes about 36 an element and
// 4 transcendental ones (gate 8, tanh 11, map 8, the rest loads, scan and stores).  fp32 states ask for them: of a month's 254 us a tanh without its
// polynomial saved 27, maps from 1 - a alone 11, an exponential without its rest 5.  Four waves a SIMD (128 registers) hide loads and hand-overs
// without a second set of buffers, which would halve them.  Measured (MI355X, a large copy runs at 6.2 TB/s): a week of
// 4 x 207 sensors, f32, 1.28 GB in 219 us = 5.8 TB/s; a month of 325 sensors, bf16, 1.12 GB in 242 us = 4.6 TB/s; a window of 64 x 12 x 207, f32, 122 MB
// in 24 us.
// WALK: the block walks its chunk tile by tile, from the state that the maps of the chunks before it give (one chunk: from h0).
// AGG: only the chunk's map is wanted (agg[chunk][b][A | X][N*H]).  CHAIN: the chunk is one tile, its state comes from the block before.
template <class X, int V, int K, int CL, int GATES, int MODE>
__global__ __launch_bounds__(GLR_THREADS, (MODE == GLR_WALK && CL < 256) || (GATES == GLR_FLAT && sizeof(typename X::S) == 4) ? 3 : 4) void glr_fwd_kernel(GlrP p) {
    constexpr bool SHARED = GATES == GLR_SHARED, FLAT = GATES == GLR_FLAT, AGG = MODE == GLR_AGG, CHAIN = MODE == GLR_CHAIN, REV = false;
    constexpr int SEG = GLR_THREADS / CL, VG = SHARED ? 1 : V, W = GLR_THREADS / 64, span = SEG * K;
    typedef typename X::S S;
    __shared__ float2 lds[SEG > 1 ? 2 : 1][SEG > 1 ? W * CL * V : 1];
    const GlrAt w = glr_where<V, CL, GATES, CHAIN, REV>(p);
    const long long NH = (long long)p.N * p.H, hoff = (long long)w.n * p.H + w.ch;
    const long long es = sizeof(S), rb = NH * es;          // bytes of an element, of a row of out
    const char* pg = static_cast<const char*>(p.gate) + (w.b * p.g_sb + w.t0 * p.g_st) * es;
    const char* pc = static_cast<const char*>(p.cand) + (w.b * p.c_sb + w.t0 * p.c_st) * es;
    const char* pm = reinterpret_cast<const char*>(p.mask) + (w.b * p.m_sb + w.t0 * p.m_st);
    char* po = static_cast<char*>(p.out) + ((long long)w.b * p.T + w.t0) * rb;
    const uint32_t lg = (uint32_t)((w.n * p.g_sn + w.gi) * es), lc = (uint32_t)((w.n * p.c_sn + w.ch) * es), lm = (uint32_t)(w.n * p.m_sn);
    const uint32_t lo = (uint32_t)(hoff * es) + (uint32_t)(w.seg * K) * (uint32_t)rb;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    int par = 0;

    float carry[V], prod[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { carry[i] = 0.f; prod[i] = 1.f; }
    if (!AGG) {
        if (p.h0 && w.active && (!CHAIN || w.chunk == 0)) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = p.h0[w.b * NH + hoff + i];
        }
        if (SEG > 1 && p.last == p.h0) {                   // in place: every wave has its state before the first barrier, behind which another may overwrite it
#pragma unroll
            for (int i = 0; i < V; ++i) GLR_HERE(carry[i]);
        }
        if (!CHAIN && CL == 16 && w.chunk > 0) {           // the chunks before this one
            const long long step = (long long)p.B * 2 * NH;
            glr_chunks_before<V, CL>(lds[1], w, p.agg + (long long)w.b * 2 * NH + hoff, step, NH, w.chunk, carry);
        }
    }

    for (int tb = w.t0; tb < w.t1; tb += span) {
        const int ts = tb + w.seg * K;
        const bool full = tb + span <= w.t1;
        // a wave behind the last step only takes part in the scan (CHAIN: as its steps are masked; the other path's zeros would be written to 64
        // registers by every wave)
        const bool live = SEG == 1 || CHAIN || tb + wave * (64 / CL) * K < w.t1;
        float nn[K][V], cc[K][V];                          // the gate (glr_gate) and phi(cand); a masked step is GLR_HOLD, c = 0
        if (live) {
            GlrVec<X, VG> rg[K];
            GlrVec<X, V> rc[K];
            GlrVec<GlrByte, 1> rm[K], rn[FLAT ? K : 1];    // (FLAT: of the last channel's node)
            const int end = w.t1 - 1 - tb;
            glr_rows<X, VG, K, CHAIN>(rg, pg, lg, (uint32_t)(p.g_st * es), w.seg, full, end);
            glr_rows<X, V, K, CHAIN>(rc, pc, lc, (uint32_t)(p.c_st * es), w.seg, full, end);
            if (p.mask) glr_rows<GlrByte, 1, K, CHAIN>(rm, pm, lm, (uint32_t)p.m_st, w.seg, full, end);
            if (FLAT && p.mask) glr_rows<GlrByte, 1, K, CHAIN>(rn, pm, (uint32_t)(w.n2 * p.m_sn), (uint32_t)p.m_st, w.seg, full, end);
            GlrMoves<V, FLAT> moves = {};
            if (p.mask || !full) glr_masked<X, V, K, FLAT>(moves, w.t1 - ts, p.mask, w.ch + V - p.H, rm, rn, rc);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    nn[k][i] = (SHARED && i) ? nn[k][0] : glr_gate(glr_up<X, VG>(rg[k], SHARED ? 0 : i));
                    cc[k][i] = glr_up<X, V>(rc[k], i);
                }
            if (p.mask || !full) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        nn[k][i] = moves.at(k, i) ? nn[k][i] : GLR_HOLD;
                        if (FLAT) cc[k][i] = moves.at(k, i) ? cc[k][i] : 0.f;
                    }
            }
            if (p.act) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) cc[k][i] = glr_tanh(cc[k][i]);
            }
        } else if (SEG > 1) {                              // its map is the identity (a branch around the maps would cost a copy of each)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) nn[k][i] = cc[k][i] = 0.f;
        }
        GLR_PHASE();
        pg += span * p.g_st * es;
        pc += span * p.c_st * es;
        pm += span * p.m_st;
        float h[V];
        if (SEG > 1 || AGG) {
            float A[V], Xl[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A[i] = 1.f; Xl[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int k = 0; k < K; ++k) {              // from here on nn, cc hold the maps up to each step
                    A[i] = glr_keep(nn[k][i], A[i]);
                    Xl[i] = glr_next(nn[k][i], cc[k][i], Xl[i], cc[k][i] - Xl[i]);
                    nn[k][i] = A[i];
                    cc[k][i] = Xl[i];
                }
            float EA[V], EX[V];
            glr_scan_maps<V, CL, REV>(lds[par], w.cl, A, Xl, EA, EX);
            if (CHAIN && w.chunk > 0 && w.active) glr_receive<V>(p.carry + ((long long)(w.chunk - 1) * p.B + w.b) * NH + hoff, carry);
            glr_scan_carry<V, CL, REV, AGG>(lds[par], w.cl, EA, EX, carry, prod, h);
            if (CHAIN && w.chunk < p.S - 1 && w.active && w.seg == 0) glr_send<V>(p.carry + ((long long)w.chunk * p.B + w.b) * NH + hoff, carry);
            par ^= 1;
            if (AGG) continue;
            GLR_PHASE();
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) h[i] = carry[i];
        }
        float o[V];
        auto steps = [&](auto nt) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (SEG > 1) o[i] = fmaf(nn[k][i], h[i], cc[k][i]);
                    else o[i] = h[i] = glr_next(nn[k][i], cc[k][i], h[i], glr_diff(nn[k][i], cc[k][i], h[i]));
                }
                if (w.active && p.out && (full || ts + k < w.t1)) glr_store<X, V, decltype(nt)::value>(po + k * rb, lo, o);
            }
        };
        if (live) {
            if (p.nt) steps(GlrYes());
            else steps(GlrNo());
        }
        po += span * rb;
        if (p.ckpt && w.active && ts + K < p.T) {          // the state before step ts + K
            const long long nck = (p.T - 1) / K;
            glr_store<GlrF32, V>(reinterpret_cast<char*>(p.ckpt + ((long long)w.b * nck + tb / K) * NH), (uint32_t)((w.seg * NH + hoff) * 4), o);
        }
        if (SEG == 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = h[i];
        }
        if (CHAIN) break;
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
// sum over the L lanes of a gate, in every one of them
template <int CTRL> __device__ __forceinline__ float glr_add_dpp(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float glr_lane_sum(float s, int L) {
    if (L > 1) s = glr_add_dpp<0xB1>(s);                   // neighbours
    if (L > 2) s = glr_add_dpp<0x4E>(s);                   // pairs
    if (L > 4) s = glr_add_dpp<0x141>(s);                  // halves of 8 lanes, mirrored
    if (L > 8) s = glr_add_dpp<0x140>(s);                  // halves of 16 lanes, mirrored
    if (L > 16) s += __shfl_xor(s, 16, 64);
    if (L > 32) s += __shfl_xor(s, 32, 64);
    return s;
}

// Bound: bytes.  The states are not read but run again from the one before each K-th step (out for f32, kept apart for 16-bit types): 3 1/8 rows in
// and 2 out instead of 4 and 2, and the 16-bit types' states come in fp32.  Two waves a SIMD: four values of 8 steps x 4 channels stay in
// registers between the scan and the second run (a third wave would spill).  Measured: the week above 2.19 GB in 396 us = 5.5 TB/s, the
// window 208 MB in 35 us = 5.9 TB/s.
// Walks the time axis from its end; `carry` is mu_{t+1} = a_{t+1} lam_{t+1}, what reaches step t from the steps behind it.
template <class X, int V, int K, int CL, int GATES, int MODE>
__global__ __launch_bounds__(GLR_THREADS, 2) void glr_bwd_kernel(GlrP p) {
    constexpr bool SHARED = GATES == GLR_SHARED, FLAT = GATES == GLR_FLAT, AGG = MODE == GLR_AGG, CHAIN = MODE == GLR_CHAIN, REV = true;
    constexpr int SEG = GLR_THREADS / CL, VG = SHARED ? 1 : V, W = GLR_THREADS / 64, span = SEG * K;
    typedef typename X::S S;
    __shared__ float2 lds[SEG > 1 ? 2 : 1][SEG > 1 ? W * CL * V : 1];
    const GlrAt w = glr_where<V, CL, GATES, CHAIN, REV>(p);
    const long long NH = (long long)p.N * p.H, NG = (long long)p.N * p.G, hoff = (long long)w.n * p.H + w.ch, nck = (p.T - 1) / K;
    const long long es = sizeof(S), rb = NH * es, gb = NG * es;
    const int ntile = (w.t1 - w.t0 + span - 1) / span, tl = w.t0 + (ntile - 1) * span;      // tiles, first step of the last one
    const char* pg = static_cast<const char*>(p.gate) + (w.b * p.g_sb + tl * p.g_st) * es;
    const char* pc = static_cast<const char*>(p.cand) + (w.b * p.c_sb + tl * p.c_st) * es;
    const char* pd = static_cast<const char*>(p.dout) + (w.b * p.d_sb + tl * p.d_st) * es;
    const char* pm = reinterpret_cast<const char*>(p.mask) + (w.b * p.m_sb + tl * p.m_st);
    char* pdc = static_cast<char*>(p.dcand) + ((long long)w.b * p.T + tl) * rb;
    char* pdg = static_cast<char*>(p.dgate) + ((long long)w.b * p.T + tl) * gb;
    const uint32_t lg = (uint32_t)((w.n * p.g_sn + w.gi) * es), lc = (uint32_t)((w.n * p.c_sn + w.ch) * es), lm = (uint32_t)(w.n * p.m_sn);
    const uint32_t ld = (uint32_t)((w.n * p.d_sn + w.ch) * es), ldc = (uint32_t)(hoff * es) + (uint32_t)(w.seg * K) * (uint32_t)rb;
    const uint32_t ldg = (uint32_t)(((long long)w.n * p.G + w.gi) * es) + (uint32_t)(w.seg * K) * (uint32_t)gb;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    int par = 0;

    float carry[V], prod[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { carry[i] = 0.f; prod[i] = 1.f; }
    if (!AGG) {
        if (p.dlast && w.active && (!CHAIN || w.chunk == p.S - 1)) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = p.dlast[w.b * NH + hoff + i];
        }
        if (!CHAIN && CL == 16 && w.chunk < p.S - 1) {     // the chunks behind this one
            const long long step = (long long)p.B * 2 * NH;
            glr_chunks_before<V, CL>(lds[1], w, p.agg + ((long long)(p.S - 1) * p.B + w.b) * 2 * NH + hoff, -step, NH, p.S - 1 - w.chunk, carry);
        }
    }

    for (int it = ntile - 1; it >= 0; --it) {
        const int tb = w.t0 + it * span, ts = tb + w.seg * K;
        const bool full = tb + span <= w.t1;
        const bool live = SEG == 1 || tb + wave * (64 / CL) * K < w.t1;       // a wave behind the last step only takes part in the scan
        GlrMoves<V, FLAT> moves = {};
        float nn[K][V], wc[K][V], q[K][V], dd[K][V];       // the gate, (1 - a) phi', a (1 - a)(h_{t-1} - c), dout
        if (live) {
            GlrVec<X, VG> rg[K];
            GlrVec<X, V> rc[K], rd[K];
            GlrVec<GlrF32, V> rs;                          // the state before the segment's first step
            GlrVec<GlrByte, 1> rm[K], rn[FLAT ? K : 1];    // (FLAT: of the last channel's node)
            const int end = w.t1 - 1 - tb;
            glr_rows<X, VG, K, CHAIN>(rg, pg, lg, (uint32_t)(p.g_st * es), w.seg, full, end);
            if (!AGG) glr_rows<X, V, K, CHAIN>(rc, pc, lc, (uint32_t)(p.c_st * es), w.seg, full, end);
            if (p.dout) {
                glr_rows<X, V, K, CHAIN>(rd, pd, ld, (uint32_t)(p.d_st * es), w.seg, full, end);
            } else {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) rd[k].e[i] = (S)0.f;
            }
            if (p.mask) glr_rows<GlrByte, 1, K, CHAIN>(rm, pm, lm, (uint32_t)p.m_st, w.seg, full, end);
            if (FLAT && p.mask) glr_rows<GlrByte, 1, K, CHAIN>(rn, pm, (uint32_t)(w.n2 * p.m_sn), (uint32_t)p.m_st, w.seg, full, end);
            if (p.mask || !full) {
                glr_masked<X, V, K, FLAT>(moves, w.t1 - ts, p.mask, w.ch + V - p.H, rm, rn, rc);
#pragma unroll
                for (int k = 0; k < K; ++k) glr_only<X, V>(ts + k < w.t1, rd[k]);      // behind the last step dout is 0
            }
            if (!AGG) {
#pragma unroll
                for (int i = 0; i < V; ++i) rs.e[i] = 0.f;
                if (ts == 0) {
                    if (p.h0) rs = glr_load<GlrF32, V>(reinterpret_cast<const char*>(p.h0 + w.b * NH), (uint32_t)(hoff * 4));
                } else if (ts < w.t1) {                    // f32: out_{ts-1} is that state
                    const float* at = p.dtype == GLR_F32 ? static_cast<const float*>(p.out) + ((long long)w.b * p.T + tb - 1) * NH : p.ckpt + ((long long)w.b * nck + tb / K - 1) * NH;
                    rs = glr_load<GlrF32, V>(reinterpret_cast<const char*>(at), (uint32_t)(hoff * 4) + (uint32_t)(p.dtype == GLR_F32 ? w.seg * K : w.seg) * (uint32_t)(NH * 4));
                }
            }
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    nn[k][i] = (SHARED && i) ? nn[k][0] : glr_gate(glr_up<X, VG>(rg[k], SHARED ? 0 : i));
                    if (!AGG) wc[k][i] = glr_up<X, V>(rc[k], i);
                }
            if (p.mask || !full) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        nn[k][i] = moves.at(k, i) ? nn[k][i] : GLR_HOLD;
                        if (FLAT && !AGG) wc[k][i] = moves.at(k, i) ? wc[k][i] : 0.f;
                    }
            }
            if (!AGG && p.act) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) wc[k][i] = glr_tanh(wc[k][i]);
            }
            GLR_PHASE();
            if (!AGG) {
                float h[V];
#pragma unroll
                for (int i = 0; i < V; ++i) h[i] = rs.e[i];
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float n = nn[k][i], c = wc[k][i], diff = glr_diff(n, c, h[i]);
                        q[k][i] = glr_aw(n) * -diff;
                        h[i] = glr_next(n, c, h[i], diff);
                        wc[k][i] = p.act ? glr_w(n) * fmaf(-c, c, 1.f) : glr_w(n);
                        GLR_HERE(q[k][i]);
                        GLR_HERE(wc[k][i]);
                    }
                GLR_PHASE();
            }
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) dd[k][i] = glr_up<X, V>(rd[k], i);
        }
        GLR_PHASE();
        pg -= span * p.g_st * es;
        pc -= span * p.c_st * es;
        pd -= span * p.d_st * es;
        pm -= span * p.m_st;
        float mu[V];
        if (SEG > 1 || AGG) {
            float A[V], Xl[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A[i] = 1.f; Xl[i] = 0.f;
            }
            if (live) {
#pragma unroll
                for (int i = 0; i < V; ++i)
#pragma unroll
                for (int k = K - 1; k >= 0; --k) {
                    A[i] = glr_keep(nn[k][i], A[i]);
                    Xl[i] = glr_keep(nn[k][i], Xl[i] + dd[k][i]);
                }
            }
            float EA[V], EX[V];
            glr_scan_maps<V, CL, REV>(lds[par], w.cl, A, Xl, EA, EX);
            if (CHAIN && w.chunk < p.S - 1 && w.active) glr_receive<V>(p.carry + ((long long)(w.chunk + 1) * p.B + w.b) * NH + hoff, carry);
            glr_scan_carry<V, CL, REV, AGG>(lds[par], w.cl, EA, EX, carry, prod, mu);
            if (CHAIN && w.chunk > 0 && w.active && w.seg == 0) glr_send<V>(p.carry + ((long long)w.chunk * p.B + w.b) * NH + hoff, carry);
            par ^= 1;
            if (AGG) continue;
            GLR_PHASE();
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) mu[i] = carry[i];
        }
        auto steps = [&](auto nt, auto masked) {
#pragma unroll
            for (int k = K - 1; k >= 0; --k) {
                const bool in = w.active && (full || ts + k < w.t1);
                float dc[V], dg[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float lam = mu[i] + dd[k][i];
                    dc[i] = lam * wc[k][i];
                    dg[i] = lam * q[k][i];
                    mu[i] = glr_keep(nn[k][i], lam);
                    if (FLAT && decltype(masked)::value) {
                        const bool o = moves.at(k, i);
                        dc[i] = o ? dc[i] : 0.f;
                        dg[i] = o ? dg[i] : 0.f;
                    }
                }
                const bool on = FLAT || !decltype(masked)::value || moves.at(k, 0);        // masked: 0, whatever lam is and the step holds
                if (in) glr_store<X, V, decltype(nt)::value>(pdc + k * rb, ldc, dc, on);
                if (!SHARED) {
                    if (in) glr_store<X, VG, decltype(nt)::value>(pdg + k * gb, ldg, dg, on);
                } else {
                    float s = 0.f;
#pragma unroll
                    for (int i = 0; i < V; ++i) s += dg[i];
                    s = glr_lane_sum(w.active && on ? s : 0.f, p.L);
                    if (in && w.gl == 0) {
                        if (p.parts == 1) glr_store<X, 1>(pdg + k * gb, ldg, &s);
                        else p.part[((((long long)w.b * p.T + ts + k) * p.N + w.n) * p.G + w.gi) * p.parts + w.part] = s;
                    }
                }
            }
        };
        if (live) {
            if (p.mask) {
                if (p.nt) steps(GlrYes(), GlrYes());
                else steps(GlrNo(), GlrYes());
            } else {
                if (p.nt) steps(GlrYes(), GlrNo());
                else steps(GlrNo(), GlrNo());
            }
        }
        pdc -= span * rb;
        pdg -= span * gb;
        if (SEG == 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = mu[i];
        }
        if (CHAIN) break;
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
    glr_store<X, 1>(static_cast<char*>(dgate) + i * sizeof(typename X::S), 0, &s);
}

}  // namespace mcrn
