// glr_scan_unit.hip - gated linear recurrence (glr_scan.h): plan and launches
#include "glr_scan.h"

namespace mcrn {

static long long up_div(long long a, long long b) { return (a + b - 1) / b; }

// Steps a thread holds.  T alone decides, so that a backward finds the checkpoints of its forward.
int glr_steps(int T) { return T <= 1 ? 1 : T <= 4 || (T > 8 && T <= 12) ? 4 : GLR_K; }

int glr_tile(const GlrP& p) { return GLR_THREADS / p.CL * p.K; }

bool glr_plan(GlrP& p, bool backward) {
    const size_t size = p.dtype == GLR_F32 ? 4 : 2;
    const int D = p.H / p.G;
    const bool shared = D > 1;
    // Four channels a thread (16 bytes of f32, 8 of the 16-bit types), at any alignment.  A number of channels that 4 does not divide: vectors run
    // over the ends of the nodes where these lie behind one another (FLAT), else one channel a thread (3 x 3110 x 206 x 37, f32, both
    // directions: 947 us so, 611 flat; 11 x 666 x 229 x 42, bf16, forward: 269 : 149).  FLAT's last vector reaches back over channels of the one
    // before: not while `last` overwrites the state that both read.
    const long long NH = (long long)p.N * p.H;
    auto dense = [&](long long sn) { return p.N == 1 || sn == p.H; };
    const bool flat = !shared && p.H % 4 && p.H >= 3 && NH >= 4 && NH < (1ll << 31) && !p.one && dense(p.g_sn) && dense(p.c_sn) &&
                      !(p.last && p.last == p.h0) && !(backward && p.dout && !dense(p.d_sn));
    p.gates = shared ? GLR_SHARED : flat ? GLR_FLAT : GLR_OWN;
    p.V = flat || (shared ? D : p.H) % 4 == 0 ? 4 : 1;
    p.nq = flat ? up_div(NH, 4) : (long long)p.N * (p.H / p.V);
    auto cover = [&](int CL) {
        p.CL = CL;
        if (shared) {
            const int lanes = (D + p.V - 1) / p.V, most = CL < 64 ? CL : 64;
            p.L = 1;
            while (p.L < lanes && p.L < most) p.L *= 2;
            p.parts = (lanes + p.L - 1) / p.L;
            p.tiles = up_div((long long)p.N * p.G * p.parts, CL / p.L);
        } else {
            p.L = p.parts = 1;
            p.tiles = up_div(p.nq, CL);
        }
        return p.tiles * p.B;
    };
    // What is written leaves nothing of itself in the last-level cache (256 MB) when it is larger: past the caches then.  A week of 4 x 207 sensors,
    // both directions: 622 us so, 652 without; a window of 12 steps, whose outputs the caches hold: 85 so with the loads too, 80 without.
    p.nt = (double)p.B * p.T * p.N * (p.H + (backward ? p.G : 0)) * size > 256e6;
    p.S = 1;
    p.first = 0;
    p.chain = false;
    p.chunk = p.T > 0 ? p.T : 1;
    p.K = glr_steps(p.T);
    long long blocks = cover(256);
    if (p.T > GLR_K && p.K == GLR_K && blocks < 512) {
        const int span = GLR_THREADS / 16 * GLR_K;
        // From here on fewer than 512 blocks of 256 channel lanes: time is cut over the lanes of a block as well.
        //  - 64 lanes x 4 segments, the block walking its tiles: up to 32 steps, and up to 288 where that still makes 400 blocks.  Fewer blocks leave the
        //    card idle (260, 100 steps: 28.5 us forward so, 25.8 in 16 lanes; with gradients 208 blocks 53 : 50, 312 blocks 65 : 63, 432 blocks, 96
        //    steps, 68 : 78).  How long such a walk pays depends on how many rounds the blocks take: both directions, 64 lanes : 16 lanes at 160, 224, 288, 320
        //    and 512 steps, 432 blocks f32 109 : 138, 162 : 178, 204 : 235, 224 : 242, 349 : 365; 462 blocks bf16, a gate a node, 75 : 96, 100 : 107,
        //    125 : 143, 139 : 153, 218 : 213; 828 blocks f32 228 : 250, 324 : 287, 415 : 404, 457 : 412, 728 : 619.  288 stands between where the last two cross.
        //  - 16 lanes x 16 segments, a block for every 128 steps, each handing its state to the next (chain), while a chunk of all blocks holds
        //    about as much as the card reads during a hand-over (1.6 us): 64 blocks of 16 bytes a lane and step (f32, 20161 steps, both directions, chain : split:
        //    128 tiles 1184 us : 1531, 64 tiles 702 : 781 (forward alone 336 : 324), 32 tiles 515 : 407), more of fewer bytes (f16, 14362 steps, 128 tiles
        //    564 : 600, 96 tiles 470 : 455).
        //  - fewer: the chunks' maps first (they need no state), then every chunk from the maps before it.  Inputs are read twice.
        const int quarter = GLR_THREADS / 64 * GLR_K;
        if (p.T <= quarter || (p.T <= 9 * quarter && cover(64) >= 400)) {
            cover(64);
        } else if ((blocks = cover(16)) * p.V * (long long)size >= 64 * 16 && p.T > span && blocks * up_div(p.T, span) <= GLR_BLOCKS) {
            p.chain = true;
            p.chunk = span;
            p.S = (int)up_div(p.T, span);
        } else if (p.T > span && !(p.last && p.last == p.h0)) {      // (a split reads h0 in every chunk: not while it is overwritten)
            long long S = up_div(1024, blocks);
            S = S > 256 ? 256 : S;
            const long long most = up_div(p.T, span);
            S = S > most ? most : S;
            p.chunk = (int)(up_div(up_div(p.T, S), span) * span);
            p.S = (int)up_div(p.T, p.chunk);
        }
    }
    // indexes in 32 bits; the grids of the walk, of the chain's clearing and of the gates' parts
    const long long words = p.chain ? p.tiles * p.B + (long long)p.S * p.B * NH : 0, sums = backward && p.parts > 1 ? (long long)p.B * p.T * p.N * p.G : 0;
    return p.tiles * p.CL < (1ll << 31) && (long long)p.N * p.G * p.parts < (1ll << 31) && p.tiles * p.B * p.S <= GLR_BLOCKS &&
           up_div(words, GLR_THREADS) <= GLR_BLOCKS && up_div(sums, GLR_THREADS) <= GLR_BLOCKS;
}

// [tickets | states] or [chunk aggregates], then the partial gate gradients; each part 256-byte aligned
static size_t chain_words(const GlrP& p) { return (size_t)(p.tiles * p.B) + (size_t)p.S * p.B * p.N * p.H; }
static size_t head_bytes(const GlrP& p) {
    const size_t n = p.chain ? chain_words(p) * 4 : p.S > 1 ? (size_t)p.S * p.B * 2 * p.N * p.H * 4 : 0;
    return (n + 255) / 256 * 256;
}
size_t glr_ws_bytes(const GlrP& p, bool backward) {
    return head_bytes(p) + (backward && p.parts > 1 ? (size_t)p.B * p.T * p.N * p.G * p.parts * 4 : 0);
}
void glr_place(GlrP& p, void* ws) {
    p.agg = (float*)ws;
    p.ticket = (unsigned*)ws;
    p.carry = p.ticket + p.tiles * p.B;
    p.part = (float*)((char*)ws + head_bytes(p));
}

template <class X, int V, int K, int CL, int GATES> static hipError_t run(const GlrP& p0, bool backward, hipStream_t st, int* launches) {
    GlrP p = p0;
    const unsigned one = (unsigned)(p.tiles * p.B);
    const dim3 block(GLR_THREADS);
    (void)hipGetLastError();
    if (CL == 16 && p.chain) {
        const long long words = (long long)chain_words(p);
        hipLaunchKernelGGL(glr_clear_kernel, dim3((unsigned)up_div(words, 256)), dim3(256), 0, st, p.ticket, p.tiles * p.B, words);
        if (backward) hipLaunchKernelGGL((glr_bwd_kernel<X, V, GLR_K, 16, GATES, GLR_CHAIN>), dim3(one * p.S), block, 0, st, p);
        else hipLaunchKernelGGL((glr_fwd_kernel<X, V, GLR_K, 16, GATES, GLR_CHAIN>), dim3(one * p.S), block, 0, st, p);
        ++*launches;
    } else {
        if (CL == 16 && p.S > 1) {                        // maps of the chunks that others start from
            p.first = backward ? 1 : 0;
            if (backward) hipLaunchKernelGGL((glr_bwd_kernel<X, V, GLR_K, 16, GATES, GLR_AGG>), dim3(one * (p.S - 1)), block, 0, st, p);
            else hipLaunchKernelGGL((glr_fwd_kernel<X, V, GLR_K, 16, GATES, GLR_AGG>), dim3(one * (p.S - 1)), block, 0, st, p);
            p.first = 0;
            ++*launches;
        }
        if (backward) hipLaunchKernelGGL((glr_bwd_kernel<X, V, K, CL, GATES, GLR_WALK>), dim3(one * p.S), block, 0, st, p);
        else hipLaunchKernelGGL((glr_fwd_kernel<X, V, K, CL, GATES, GLR_WALK>), dim3(one * p.S), block, 0, st, p);
    }
    ++*launches;
    if (backward && p.parts > 1) {
        const long long n = (long long)p.B * p.T * p.N * p.G;
        hipLaunchKernelGGL((glr_parts_kernel<X>), dim3((unsigned)up_div(n, 256)), dim3(256), 0, st, p.part, p.parts, n, p.dgate);
        ++*launches;
    }
    return hipGetLastError();
}

template <class X, int V, int GATES> static hipError_t run_v(const GlrP& p, bool backward, hipStream_t st, int* launches) {
    if (p.K == 1) return run<X, V, 1, 256, GATES>(p, backward, st, launches);
    if (p.K == 4) return run<X, V, 4, 256, GATES>(p, backward, st, launches);
    if (p.CL == 256) return run<X, V, GLR_K, 256, GATES>(p, backward, st, launches);
    if (p.CL == 64) return run<X, V, GLR_K, 64, GATES>(p, backward, st, launches);
    return run<X, V, GLR_K, 16, GATES>(p, backward, st, launches);
}
template <class X> static hipError_t run_x(const GlrP& p, bool backward, hipStream_t st, int* launches) {
    if (p.gates == GLR_SHARED) return p.V == 4 ? run_v<X, 4, GLR_SHARED>(p, backward, st, launches) : run_v<X, 1, GLR_SHARED>(p, backward, st, launches);
    if (p.gates == GLR_FLAT) return run_v<X, 4, GLR_FLAT>(p, backward, st, launches);
    return p.V == 4 ? run_v<X, 4, GLR_OWN>(p, backward, st, launches) : run_v<X, 1, GLR_OWN>(p, backward, st, launches);
}
static hipError_t launch(const GlrP& p, bool backward, hipStream_t st, int* launches) {
    if (p.dtype == GLR_F32) return run_x<GlrF32>(p, backward, st, launches);
    if (p.dtype == GLR_BF16) return run_x<GlrBf16>(p, backward, st, launches);
    return run_x<GlrF16>(p, backward, st, launches);
}
hipError_t launch_glr_forward(const GlrP& p, hipStream_t st, int* launches) { return launch(p, false, st, launches); }
hipError_t launch_glr_backward(const GlrP& p, hipStream_t st, int* launches) { return launch(p, true, st, launches); }

}  // namespace mcrn
