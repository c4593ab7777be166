// adamw_multi_unit.hip - AdamW over many tensors (adamw_multi.h): launches
#include "adamw_multi.h"

namespace mcrn {

unsigned adamw_key(unsigned seed, int id, unsigned step) { return adamw_key_of(seed, id, step); }

hipError_t launch_adamw(const AdamwP& p, unsigned blocks, int dtype, int bits, hipStream_t st) {
    (void)hipGetLastError();
    const dim3 grid(blocks), block(256);
    if (dtype == 0 && bits == 32) hipLaunchKernelGGL((adamw_kernel<AdamwF32, 32>), grid, block, 0, st, p);
    else if (dtype == 0) hipLaunchKernelGGL((adamw_kernel<AdamwF32, 8>), grid, block, 0, st, p);
    else if (bits == 32) hipLaunchKernelGGL((adamw_kernel<AdamwBf16, 32>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((adamw_kernel<AdamwBf16, 8>), grid, block, 0, st, p);
    return hipGetLastError();
}
hipError_t launch_adamw_norm(const AdamwNormP& p, unsigned blocks, int dtype, hipStream_t st) {
    (void)hipGetLastError();
    if (dtype == 0) hipLaunchKernelGGL((adamw_norm_kernel<AdamwF32>), dim3(blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((adamw_norm_kernel<AdamwBf16>), dim3(blocks), dim3(256), 0, st, p);
    return hipGetLastError();
}
hipError_t launch_adamw_prep(const AdamwPrepP& p, hipStream_t st) {
    (void)hipGetLastError();
    hipLaunchKernelGGL(adamw_prep_kernel, dim3((unsigned)((p.nt + 63) / 64)), dim3(64), 0, st, p);
    return hipGetLastError();
}
hipError_t launch_adamw_unpack(const uint8_t* m, const uint8_t* ms, const uint8_t* v, const uint8_t* vs, long long n, float* om, float* ov, hipStream_t st) {
    (void)hipGetLastError();
    const long long n4 = n / 4;
    hipLaunchKernelGGL(adamw_unpack_kernel, dim3((unsigned)((n4 + 255) / 256), 2), dim3(256), 0, st, m, ms, v, vs, om, ov, n4);
    return hipGetLastError();
}

}  // namespace mcrn
