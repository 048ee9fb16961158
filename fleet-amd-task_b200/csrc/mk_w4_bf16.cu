// mk_w4_bf16.cu -- the products with 4-bit weights for BF16 activations.
#include "mk_w4_kernel.cuh"

int w4::launch_bf16(const Args& a, int group, bool two, bool xr, int grid, cudaStream_t s) {
  return two ? launch_group<Bf16, 2>(a, group, xr, grid, s) : launch_group<Bf16, 1>(a, group, xr, grid, s);
}
