// mk_w4_fp16.cu -- the products with 4-bit weights for FP16 activations.
#include "mk_w4_kernel.cuh"

int w4::launch_fp16(const Args& a, int group, bool two, bool xr, int grid, cudaStream_t s) {
  return launch_type<Fp16>(a, group, two, xr, grid, s);
}
