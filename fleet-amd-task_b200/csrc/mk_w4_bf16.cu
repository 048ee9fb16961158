// mk_w4_bf16.cu -- the products with 4-bit weights for BF16 activations.
#include "mk_w4_kernel.cuh"

int w4::launch_bf16(const Args& a, int group, bool two, bool xr, int grid, cudaStream_t s) {
  return launch_type<Bf16>(a, group, two, xr, grid, s);
}
