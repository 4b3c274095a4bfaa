// Choice of the product kernel's variant and its launch.
#pragma once
#include "launch.h"
#include "nibble.cuh"

namespace s1c {

// Launches the variant; false, and nothing, if x does not fit beside its rings. WHOLE: x passes in blocks
// of columns instead.
template <typename T, int GROUP, bool ZERO, int NT, int RT, int SPAN, int WARPS, bool WHOLE = false>
bool launch_nibble_as(NibbleArgs a, int dev, cudaStream_t st) {
  using W = NibbleWarp<T, GROUP, NT, RT, SPAN, WARPS, ZERO>;
  constexpr auto KERNEL = nibble_kernel<T, GROUP, NT, RT, SPAN, WARPS, ZERO>;
  constexpr int LIMIT = 227 * 1024;
  a.steps = (a.K + 127) / 128;
  a.tiles = (a.N + W::ROWS - 1) / W::ROWS;
  a.width = (a.K + 31) / 32 * 16;
  a.block = a.steps;
  a.split = !WHOLE;
  const auto smem = [&] { return NibbleSmem(a.M, a.block, GROUP, W::RING, WARPS * W::PART, a.split).total; };
  if (a.split && ((int64_t)a.M * a.K > LIMIT || smem() > LIMIT)) return false;
  if (!a.split) {
    a.block = std::min(a.steps, LIMIT / 2 / 128 / a.M + SPAN);
    a.block = (a.block + SPAN - 1) / SPAN * SPAN;
    while (a.block > SPAN && smem() > LIMIT) a.block -= SPAN;
  }
  const int units = a.split ? a.tiles : (a.tiles + WARPS - 1) / WARPS;
  allow_smem<KERNEL>(dev);
  // Two blocks stage x together from nine rows on: 64 x 4096 x 1024 takes 16.9 us with it and 20.9 without,
  // 16 x 50368 x 2624 35.7 and 36.4; 2 x 8192 x 4096 11.0 and 10.2.
  const int cluster = a.split && NT > 1 && units > 1 ? 2 : 1;
  launch_after(KERNEL, (unsigned)(std::min(units, sm_count(dev)) / cluster * cluster), WARPS * 32, smem(), cluster, st, a);
  return true;
}

// x in shared memory, if need be beside shorter rings; false if it does not fit. The variants are those for
// `like` rows: what fits for these fits for fewer.
template <typename T, int GROUP, bool ZERO>
bool launch_nibble_fit(const NibbleArgs& a, int like, int dev, cudaStream_t st) {
  if (like <= 8) return launch_nibble_as<T, GROUP, ZERO, 1, 1, 4, 16>(a, dev, st) || launch_nibble_as<T, GROUP, ZERO, 1, 1, 2, 16>(a, dev, st);
  if (like <= 16) return launch_nibble_as<T, GROUP, ZERO, 2, 1, 2, 16>(a, dev, st) || launch_nibble_as<T, GROUP, ZERO, 2, 1, 1, 16>(a, dev, st);
  if (like <= 32) return launch_nibble_as<T, GROUP, ZERO, 4, 2, 2, 8>(a, dev, st);
  return launch_nibble_as<T, GROUP, ZERO, 8, 1, 2, 8>(a, dev, st);
}

// Rows whose x does not fit go in as many launches as make it fit: the codes then come from the cache
// again, which costs less than passing x through each block in blocks of columns (32 x 8192 x 4096: two
// launches 35 us, columns 65 us). That is left for columns so many that not even one row fits.
template <typename T, int GROUP, bool ZERO>
void launch_nibble(const NibbleArgs& a, int dev, cudaStream_t st) {
  const int64_t out_bytes = a.out_f32 ? 4 : sizeof(T);
  for (int parts = 1; parts <= a.M; ++parts) {
    const int rows = (a.M + parts - 1) / parts;
    NibbleArgs p = a;
    p.M = rows;
    if (!launch_nibble_fit<T, GROUP, ZERO>(p, rows, dev, st)) continue;
    for (int m = rows; m < a.M; m += rows) {
      p.M = std::min(rows, a.M - m);
      p.x = static_cast<const T*>(a.x) + m * a.x_stride;
      p.out = static_cast<char*>(a.out) + m * a.out_stride * out_bytes;
      launch_nibble_fit<T, GROUP, ZERO>(p, rows, dev, st);
    }
    return;
  }
  for (int m = 0; m < a.M; m += 8) {
    NibbleArgs p = a;
    p.M = std::min(8, a.M - m);
    p.x = static_cast<const T*>(a.x) + m * a.x_stride;
    p.out = static_cast<char*>(a.out) + m * a.out_stride * out_bytes;
    launch_nibble_as<T, GROUP, ZERO, 1, 1, 4, 16, true>(p, dev, st);
  }
}
template <typename T, bool ZERO>
void launch_nibble(const NibbleArgs& a, int group, int dev, cudaStream_t st) {
  if (group == 32) return launch_nibble<T, 32, ZERO>(a, dev, st);
  if (group == 64) return launch_nibble<T, 64, ZERO>(a, dev, st);
  launch_nibble<T, 128, ZERO>(a, dev, st);
}

}  // namespace s1c
