// adamw_multi_unit.hip - AdamW over many tensors (adamw_multi.h): launches
#include "adamw_multi.h"

namespace mcrn {

unsigned adamw_key(unsigned seed, int id, unsigned step) { return adamw_key_of(seed, id, step); }

// A step that moves more than this leaves nothing of itself in the last-level cache (256 MB): it streams past the caches
static const double STREAM = 256e6;

template <bool NT> static void main_kernel(const AdamwP& p, dim3 grid, int dtype, int bits, hipStream_t st) {
    const dim3 block(256);
    if (dtype == 0 && bits == 32) hipLaunchKernelGGL((adamw_kernel<AdamwF32, 32, NT>), grid, block, 0, st, p);
    else if (dtype == 0) hipLaunchKernelGGL((adamw_kernel<AdamwF32, 8, NT>), grid, block, 0, st, p);
    else if (bits == 32) hipLaunchKernelGGL((adamw_kernel<AdamwBf16, 32, NT>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((adamw_kernel<AdamwBf16, 8, NT>), grid, block, 0, st, p);
}
hipError_t launch_adamw(const AdamwP& p, unsigned blocks, long long elements, int dtype, int bits, hipStream_t st) {
    (void)hipGetLastError();
    const double each = (dtype == 0 ? 12 : 14) + (bits == 32 ? 16 : 4);
    if (elements * each > STREAM) main_kernel<true>(p, dim3(blocks), dtype, bits, st);
    else main_kernel<false>(p, dim3(blocks), dtype, bits, st);
    return hipGetLastError();
}
hipError_t launch_adamw_norm(const AdamwNormP& p, unsigned blocks, long long elements, int dtype, hipStream_t st) {
    (void)hipGetLastError();
    const bool nt = elements * (dtype == 0 ? 4.0 : 2.0) > STREAM;
    if (dtype == 0 && nt) hipLaunchKernelGGL((adamw_norm_kernel<AdamwF32, true>), dim3(blocks), dim3(256), 0, st, p);
    else if (dtype == 0) hipLaunchKernelGGL((adamw_norm_kernel<AdamwF32, false>), dim3(blocks), dim3(256), 0, st, p);
    else if (nt) hipLaunchKernelGGL((adamw_norm_kernel<AdamwBf16, true>), dim3(blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((adamw_norm_kernel<AdamwBf16, false>), dim3(blocks), dim3(256), 0, st, p);
    return hipGetLastError();
}
hipError_t launch_adamw_factor(const AdamwP& p, float* factor, hipStream_t st) {
    (void)hipGetLastError();
    hipLaunchKernelGGL(adamw_factor_kernel, dim3(1), dim3(256), 0, st, p.part, p.parts, p.grad_scale, p.max_norm, p.norm, factor);
    return hipGetLastError();
}
hipError_t launch_adamw_prep(const AdamwPrepP& p, hipStream_t st) {
    (void)hipGetLastError();
    hipLaunchKernelGGL(adamw_prep_kernel, dim3((unsigned)((p.nt + 63) / 64)), dim3(64), 0, st, p);
    return hipGetLastError();
}
hipError_t launch_adamw_unpack(const uint8_t* m, const uint8_t* ms, const uint8_t* v, const uint8_t* vs, long long n, float* om, float* ov, hipStream_t st) {
    (void)hipGetLastError();
    const bool nt = n * 10.0 > STREAM;
    for (long long at = 0, most = 1ll << 33; at < n; at += most) {            // half of what a launch can hold, whole blocks of 64
        const long long n4 = (n - at < most ? n - at : most) / 4;
        const dim3 grid((unsigned)((n4 + 255) / 256));
        if (nt) hipLaunchKernelGGL((adamw_unpack_kernel<true>), grid, dim3(256), 0, st, m + at, ms + at / ADAMW_BLOCK, v + at, vs + at / ADAMW_BLOCK, om + at, ov + at, n4);
        else hipLaunchKernelGGL((adamw_unpack_kernel<false>), grid, dim3(256), 0, st, m + at, ms + at / ADAMW_BLOCK, v + at, vs + at / ADAMW_BLOCK, om + at, ov + at, n4);
    }
    return hipGetLastError();
}

}  // namespace mcrn
