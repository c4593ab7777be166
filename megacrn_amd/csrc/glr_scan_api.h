// glr_scan_api.h - parameter block and host entry points of the gated linear recurrence (glr_scan.h, compiled in
// glr_scan_unit.hip).  engine.hip includes only this file.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stddef.h>

namespace mcrn {

enum { GLR_F32 = 0, GLR_BF16 = 1, GLR_F16 = 2 };
enum { GLR_OWN = 0, GLR_SHARED = 1, GLR_FLAT = 2 };

// h_t = a_t h_{t-1} + (1 - a_t) phi(cand_t), a_t = sigmoid(gate_t); a step whose mask byte is 0 keeps the state.
// gate (B,T,N,G), cand (B,T,N,H), D = H / G channels share a gate; strides in elements, the last dimension is contiguous.
struct GlrP {
    int B, T, N, H, G, dtype, act;          // act: 0 phi(c) = c, 1 phi = tanh
    const void *gate, *cand;
    long long g_sb, g_st, g_sn, c_sb, c_st, c_sn;
    const uint8_t* mask;                    // nullable
    long long m_sb, m_st, m_sn;
    const float* h0;                        // (B,N,H) or NULL = zeros
    void* out;                              // (B,T,N,H) contiguous, NULL = not wanted (forward only)
    float* last;                            // (B,N,H), may be h0 itself (forward only)
    float* ckpt;                            // (B, ceil(T/K) - 1, N, H) states before steps K, 2 K, .. (K = glr_steps(T)); NULL = not wanted.
                                            // f32: never written, the backward reads the same states from `out`
    // backward
    const void* dout;                       // (B,T,N,H) or NULL = zeros
    long long d_sb, d_st, d_sn;
    const float* dlast;                     // (B,N,H) or NULL = zeros
    void *dgate, *dcand;                    // (B,T,N,G), (B,T,N,H) contiguous
    float* dstate;                          // (B,N,H) or NULL = not wanted
    // plan (glr_plan)
    int one;                                // not 0: plan without GLR_FLAT
    int gates;                              // GLR_OWN: channels of a node; GLR_SHARED: G < H; GLR_FLAT: channels of all nodes behind one another
    int V, K, CL, S, L, parts;              // channels and steps a thread, channel lanes a block, chunks of the time axis,
    int chunk, first;                       // lanes and parts of a shared gate's channels; steps a chunk, first chunk of the launch
    long long nq, tiles;                    // channel vectors of a batch entry, blocks that cover them
    bool nt;                                // outputs go past the caches
    bool chain;                             // a chunk is one tile and takes its state from the block before it
    float *agg, *part;                      // workspace: chunk aggregates, partial gate gradients,
    unsigned *ticket, *carry;               // chunks taken of each tile, states behind the chunks (chain)
};

constexpr long long GLR_BLOCKS = (1ll << 24) - 1;     // a launch counts its work items in 32 bits: blocks of 256
constexpr int GLR_K = 8;                    // steps a thread holds in registers, at most = distance of the checkpoints
int glr_steps(int T);

bool glr_plan(GlrP& p, bool backward);      // fills the plan; false: too large
size_t glr_ws_bytes(const GlrP& p, bool backward);
int glr_tile(const GlrP& p);                 // steps of a block's tile
void glr_place(GlrP& p, void* ws);          // the plan's parts of the workspace
hipError_t launch_glr_forward(const GlrP& p, hipStream_t st, int* launches);
hipError_t launch_glr_backward(const GlrP& p, hipStream_t st, int* launches);

}  // namespace mcrn
