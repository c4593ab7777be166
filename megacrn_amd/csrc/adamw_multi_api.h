// adamw_multi_api.h - parameter blocks and host entry points of the AdamW step over many tensors (adamw_multi.h, compiled in
// adamw_multi_unit.hip).  engine.hip includes only this file.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stddef.h>

namespace mcrn {

constexpr int ADAMW_BLOCK = 64;           // elements that share a scale of the 8-bit moments; the arenas' tensors start on it
constexpr int ADAMW_TENSORS = 60;         // tensors a launch carries in its arguments (64 B each, below the 4 KB an argument block holds)

constexpr long long ADAMW_BLOCKS = (1ll << 24) - 1;   // a launch counts its work items in 32 bits: blocks of 256, 1024 elements each

enum { ADAMW_VEC = 1 };                   // AdamwT::flags: parameter and gradient can be read four elements at a time

struct AdamwT {                           // one tensor of a launch
    void* p;
    const void* g;
    long long n, off;                     // elements; where its moments start in the arenas
    unsigned blk0;                        // first block of the launch that works on it
    unsigned key;                         // of its random bits
    float step_size, inv_bc2, decay;      // lr / (1 - b1^s), 1 / sqrt(1 - b2^s), 1 - lr wd
    int flags;
    int id;                               // its number among all tensors
    int pad;
};
static_assert(sizeof(AdamwT) == 64, "AdamwT is sized for the argument block");

struct AdamwDyn { float step_size, inv_bc2, decay; unsigned key; };   // the same from device counters

struct AdamwP {
    AdamwT t[ADAMW_TENSORS];
    int nt;                               // tensors; a block works on 1024 elements
    void *m, *v;                          // arenas: float, or codes
    uint8_t *ms, *vs;                     // scale bytes, one for each 64 elements
    float* master;                        // arena of fp32 parameters (16-bit ones only)
    const float* factor;                  // what the gradients are multiplied by, or NULL: each block takes it from
    const double* part;                   // the sums of squares of the gradients; parts = 0: grad_scale, no clipping
    int parts;
    float max_norm;
    float* norm;                          // receives the norm, or NULL
    const AdamwDyn* dyn;                  // NULL: the tensors' own values
    float grad_scale, b1, c1, b2, c2, eps;   // c = 1 - b
};
struct AdamwNormP {
    AdamwT t[ADAMW_TENSORS];
    int nt, per;                          // tensors; runs of 1024 elements a block
    unsigned blk0;                        // first partial sum of this launch
    double* part;
};
struct AdamwPrepP {
    const double *lr, *wd;                // device, one for each tensor
    int* step;                            // device, counted up for every tensor that has a gradient
    AdamwDyn* dyn;
    unsigned long long has[64];           // bit i of word w: tensor 64 w + i has a gradient
    int nt, base;
    unsigned seed;
    double b1, b2;
};

unsigned adamw_key(unsigned seed, int id, unsigned step);
// elements: of the whole step, for the choice of what streams past the caches
hipError_t launch_adamw(const AdamwP& p, unsigned blocks, long long elements, int dtype, int bits, hipStream_t st);
hipError_t launch_adamw_norm(const AdamwNormP& p, unsigned blocks, long long elements, int dtype, hipStream_t st);
hipError_t launch_adamw_factor(const AdamwP& p, float* factor, hipStream_t st);
hipError_t launch_adamw_prep(const AdamwPrepP& p, hipStream_t st);
hipError_t launch_adamw_unpack(const uint8_t* m, const uint8_t* ms, const uint8_t* v, const uint8_t* vs, long long n, float* om, float* ov, hipStream_t st);

}  // namespace mcrn
