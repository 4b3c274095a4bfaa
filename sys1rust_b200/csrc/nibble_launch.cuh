// Choice of the product kernel's variant and its launch.
#pragma once
#include "launch.h"
#include "nibble.cuh"

namespace s1c {

template <typename T, int GROUP, int NT, int RT, int SPAN, int WARPS, bool ZERO>
void launch_nibble(NibbleArgs a, int dev, cudaStream_t st) {
  using W = NibbleWarp<T, GROUP, NT, RT, SPAN, WARPS, ZERO>;
  constexpr auto KERNEL = nibble_kernel<T, GROUP, NT, RT, SPAN, WARPS, ZERO>;
  constexpr int LIMIT = 227 * 1024;
  a.steps = (a.K + 127) / 128;
  a.tiles = (a.N + W::ROWS - 1) / W::ROWS;
  a.width = (a.K + 31) / 32 * 16;
  a.block = a.steps;
  const auto smem = [&] { return NibbleSmem(a.M, a.block, GROUP, W::RING, WARPS * W::PART, a.split).total; };
  a.split = NT <= 2;
  if (a.split && smem() > LIMIT) a.split = 0;
  if (!a.split) {
    a.block = (a.steps + SPAN - 1) / SPAN * SPAN;
    while (a.block > SPAN && smem() > LIMIT) a.block -= SPAN;
  }
  const int units = a.split ? a.tiles : (a.tiles + WARPS - 1) / WARPS;
  allow_smem<KERNEL>(dev);
  KERNEL<<<std::min(units, sm_count(dev)), WARPS * 32, smem(), st>>>(a);
}
template <typename T, int GROUP, bool ZERO>
void launch_nibble(const NibbleArgs& a, int dev, cudaStream_t st) {
  if (a.M <= 8) return launch_nibble<T, GROUP, 1, 1, 4, 16, ZERO>(a, dev, st);
  if (a.M <= 16) return launch_nibble<T, GROUP, 2, 1, 2, 16, ZERO>(a, dev, st);
  if (a.M <= 32) return launch_nibble<T, GROUP, 4, 2, 2, 8, ZERO>(a, dev, st);
  launch_nibble<T, GROUP, 8, 1, 2, 8, ZERO>(a, dev, st);
}
template <typename T, int GROUP>
void launch_nibble(const NibbleArgs& a, int dev, cudaStream_t st) {
  a.zeros ? launch_nibble<T, GROUP, true>(a, dev, st) : launch_nibble<T, GROUP, false>(a, dev, st);
}
template <typename T>
void launch_nibble(const NibbleArgs& a, int group, int dev, cudaStream_t st) {
  if (group == 32) return launch_nibble<T, 32>(a, dev, st);
  if (group == 64) return launch_nibble<T, 64>(a, dev, st);
  launch_nibble<T, 128>(a, dev, st);
}

}  // namespace s1c
