// The 4-bit products' kernels for bf16 rows, without zero points, in a unit of their own: the units compile
// side by side.
#include "nibble_launch.cuh"

namespace s1c {

void launch_nibble_bf16(const NibbleArgs& a, int group, int dev, cudaStream_t st) {
  launch_nibble<__nv_bfloat16, false>(a, group, dev, st);
}

}  // namespace s1c
