// Products of a few rows with 4-bit weights:
//   out[m, n] = act( sum_g s[n, g] * sum_{k in g} (q[n, k] - z[n, g]) * x[m, k] + bias[n] )
// with codes q in 0..15 packed two to a byte (the even column in the low half), a scale s and,
// where given, a zero point z for each group of 32, 64 or 128 columns of a row (z = 8 otherwise).
//
// Bound by the codes' bytes up to about 16 rows. A warp takes row tiles of 16 (or 2 x 16) rows in blocks of
// 128 columns; it copies its codes to its own place in shared memory (cp.async), a span of blocks ahead, so
// it waits for no other warp, and little is spent on a code:
//
//  - Codes go to mma.m16n8k16 as f16 without arithmetic. The bits of a code at the bottom of a half are
//    the subnormal q * 2^-24, four places up q * 2^-20, and the tensor cores take subnormals exactly. One
//    32-bit word gives four operand registers with one shift and four ANDs:
//    (q0, q4), 16 (q1, q5), (q2, q6), 16 (q3, q7). x is laid out in that order, its factor 1/16 with it.
//  - Which eight columns of a block a lane's word j holds is free as long as x is laid out alike and the
//    four lanes of a row stay in one group: words of 16 neighbouring bytes for groups of 128, of 8 for 64, of 4 for
//    32. A row's 64 bytes lie in shared memory so that these reads meet no bank twice.
//  - x is brought to f16 by a power of two for each row (its largest value near 2^14), so bf16 and f16
//    inputs keep all their bits: values below 2^-28 of the row's largest lose low bits, by at most
//    2^-35 of the largest, far below an fp32 sum's own rounding.
//  - The zero point enters as the sum's first value, -z * sum_{k in g} x[m, k], from sums that are
//    formed once for each group when x is staged. Group sums and totals are fp32.
//
// Two ways to share the work of a block:
//  - x in shared memory as a whole (the rule; more rows than fit go in several launches): a block has a contiguous
//    run of row tiles and its warps equal shares of all their steps, so that a tile may be split between warps; split
//    tiles are summed in the warps' order, hence the same bits in each call;
//  - where not even one row of x fits, each warp has whole tiles, and x passes through in blocks of columns.
//
// Measured: 1 x 28672 x 8192, groups of 128: 27.2 us, 4.5 TB/s; 28672 rows more take 19.6 us more (6.2
// TB/s), so what is left is fixed: the launch, staging x (3 us), the last tiles. 16 x 50368 x 2624 with
// zero points, groups of 64: 35.7 us (2.2 TB/s), of which about 5 us stage x (two blocks together, from nine rows
// on); the warps, four on a scheduler, wait for one another's products and shared memory there. 16 warps
// were better than 12, 20 or 24 (registers). Not kept: TMA rings with a barrier for each step (38 us for
// the first case), codes loaded ahead into registers (42 us: loads share a few scoreboards, so the oldest
// waits for the newest).
#pragma once
#include "mma.cuh"

namespace s1c {

struct NibbleArgs {
  const void* x;
  const uint8_t* codes;
  const void* scales;
  const void* zeros;  // nullable: 8
  void* out;
  const float* bias;  // nullable
  int64_t x_stride, pitch, scale_stride, out_stride;
  int M, N, K, groups, act, out_f32;
  int steps;  // 128-column steps of a row
  int block;  // steps of x that are staged at a time
  int tiles;  // row tiles of the matrix
  int width;  // bytes of a row of codes
  int vec;    // x rows are 16-byte aligned
  int split;  // x fits: tiles may be split between warps
};

// Asynchronous copy of 16 bytes to shared memory; each thread waits for its own.
S1C_DEV void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
S1C_DEV void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All groups but the newest N have landed.
template <int N>
S1C_DEV void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The block's place in its cluster, the cluster's blocks, its barrier, and an address in another block.
S1C_DEV int cluster_rank() {
  int r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
S1C_DEV int cluster_blocks() {
  int r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
S1C_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
S1C_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
S1C_DEV uint32_t cluster_address(const void* p, int block) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(block));
  return r;
}
S1C_DEV void cluster_put(uint32_t at, uint4 v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
S1C_DEV void cluster_put(uint32_t at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }

// Shared memory of one block, in bytes.
struct NibbleSmem {
  int pitch;      // halves between rows of x: 64 bytes more than a multiple of 128, so that eight lanes' 16-byte
                  // pieces, of two rows, fall into different banks
  int sum_pitch;  // floats between the rows' group sums
  int ring, x, sums, parts, misc, total;
  __host__ __device__ NibbleSmem(int M, int block, int group, int ring_bytes, int part_floats, bool split) {
    pitch = (block + 1) / 2 * 256 + 32;
    sum_pitch = (block * 128 / group) | 1;
    ring = 0;
    x = ring_bytes;
    sums = x + M * pitch * 2;
    parts = sums + (M * sum_pitch * 4 + 15) / 16 * 16;
    misc = parts + (split ? part_floats * 4 : 0);
    total = misc + 2 * 64 * 4;  // row scales, maxima
  }
};

// GROUP columns share a scale; NT tiles of eight rows of x; RT tiles of 16 rows of codes; SPAN steps of
// 128 columns are copied while the span before is used; ZERO: zero points are given.
template <typename T, int GROUP, int NT, int RT, int SPAN, int WARPS, bool ZERO>
struct NibbleWarp {
  static constexpr int ROWS = 16 * RT, GP = 128 / GROUP;  // groups of a step
  static constexpr int PART = RT * NT * 4 * 32;                              // floats of a tile's totals
  static constexpr int STEP = RT * 1024, RING = WARPS * 2 * SPAN * STEP;     // bytes of a step's codes; of two spans
  static constexpr int NS = (SPAN * GP + 3) / 4;  // scales of a row and span that one of its four lanes holds
  const NibbleArgs& a;
  const float* row_scale;  // 2^-e that undoes x's scaling, for each row
  int lane;
  uint32_t x_at[NT], sum_at[NT][2];      // shared addresses; rows of x past M read the last one
  const uint8_t* code[RT][2];            // next codes of the tile being loaded; rows past N read the last one
  const uint16_t* scale[RT][2];
  const uint16_t* zero[ZERO ? RT : 1][2];
  // In the first of the two spans' copies: where this lane's 16 bytes of a row go (chunk c of its row), and
  // where its words of group 0 and (XORed) of the others are. Chunks of 16 bytes are moved by the row: all
  // of 32 bytes for groups of 64, of 16 for 32.
  uint32_t copy_at, word_at;
  uint32_t sz[2][RT][2][NS];             // (scale, zero point) of the span in use and of the next
  float total[RT][NT][4];

  S1C_DEV void setup(const uint8_t* ring_, const __half* xs, const float* sums, int pitch, int sum_pitch) {
    const int g = lane >> 2, c = lane & 3;
    const uint32_t row = smem_u32(ring_) + g * 64;
    const int move = GROUP == 128 ? 0 : GROUP == 64 ? (g >> 1 & 1) * 2 : g >> 1 & 3;  // of a chunk, by XOR
    copy_at = row + ((c ^ move) << 4);
    word_at = row + (GROUP == 128 ? c * 16 : GROUP == 64 ? (move << 4) + c * 8 : (move << 4) + c * 4);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      x_at[j] = smem_u32(xs + min(8 * j + g, a.M - 1) * pitch + c * 8);
#pragma unroll
      for (int e = 0; e < 2; ++e) sum_at[j][e] = smem_u32(sums + min(8 * j + 2 * c + e, a.M - 1) * sum_pitch);
    }
  }
  S1C_DEV void point(int tile, int step) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t n = min((int64_t)tile * ROWS + r * 16 + h * 8 + (lane >> 2), (int64_t)a.N - 1);
        code[r][h] = a.codes + n * a.pitch + step * 64 + (lane & 3) * 16;
        scale[r][h] = static_cast<const uint16_t*>(a.scales) + n * a.scale_stride + step * GP;
        if (ZERO) zero[r][h] = static_cast<const uint16_t*>(a.zeros) + n * a.scale_stride + step * GP;
      }
  }
  // Copies step S of a span to its half `side` (0 or 1). TAIL: columns past the row's codes (x is 0 there)
  // read its first ones.
  template <int S, bool TAIL>
  S1C_DEV void load(int step, uint32_t side) {
    int off = S * 64;
    if (TAIL && step * 64 + (lane & 3) * 16 >= a.width) off = (S - step) * 64 - (lane & 3) * 16;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) copy_async(copy_at + side * (SPAN * STEP) + S * STEP + (r * 2 + h) * 512, code[r][h] + off);
  }
  // A span's scales and zero points, spread over the four lanes of a row. Groups past the last read the
  // last one.
  S1C_DEV void fetch(uint32_t (&v)[RT][2][NS], int step) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int g = min(4 * i + (lane & 3), a.groups - 1 - step * GP);
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          v[r][h][i] = __ldg(scale[r][h] + g);
          if (ZERO) v[r][h][i] |= (uint32_t)__ldg(zero[r][h] + g) << 16;
        }
    }
  }
  S1C_DEV void advance() {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        code[r][h] += SPAN * 64;
        scale[r][h] += SPAN * GP;
        if (ZERO) zero[r][h] += SPAN * GP;
      }
  }
  S1C_DEV void clear() {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) total[r][j][v] = 0.f;
  }
  // Step S of the span in half `side`, whose staged x begins `ahead` columns in.
  template <int S>
  S1C_DEV void consume(int ahead, uint32_t side) {
    uint32_t words[RT][2][4];
    const uint32_t from = word_at + side * (SPAN * STEP);
    static_for<RT * 2>([&](auto X) {
      constexpr int r = decltype(X)::value / 2, h = decltype(X)::value % 2, OFF = S * STEP + decltype(X)::value * 512;
      uint32_t(&w)[4] = words[r][h];
      if constexpr (GROUP == 128) {
        const uint4 p = lds_v4<OFF>(from);
        w[0] = p.x, w[1] = p.y, w[2] = p.z, w[3] = p.w;
      } else if constexpr (GROUP == 64) {
        const uint2 p0 = lds_v2<OFF>(from), p1 = lds_v2<OFF>(from ^ 32);
        w[0] = p0.x, w[1] = p0.y, w[2] = p1.x, w[3] = p1.y;
      } else {
        static_for<4>([&](auto I) { w[decltype(I)::value] = lds_u32<OFF>(from ^ (decltype(I)::value * 16)); });
      }
    });
    static_for<GP>([&](auto Q) {
      constexpr int q = decltype(Q)::value, at = S * GP + q;
      float acc[RT][NT][4];
      uint32_t v[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) v[r][h] = __shfl_sync(0xffffffffu, sz[0][r][h][at / 4], (lane & 28) + at % 4);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float x0 = lds_f32<(S * GP + q) * 4>(sum_at[j][0] + ahead / GROUP * 4);
        const float x1 = lds_f32<(S * GP + q) * 4>(sum_at[j][1] + ahead / GROUP * 4);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float z = ZERO ? bits_f32<T>((uint16_t)(v[r][h] >> 16)) : 1.f;  // without zero points the 8 is in the sums
            acc[r][j][2 * h] = z * x0, acc[r][j][2 * h + 1] = z * x1;
          }
      }
      static_for<4 / GP>([&](auto I) {
        constexpr int i = q * (4 / GP) + decltype(I)::value;
        uint32_t lo[RT][4], hi[RT][4];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t word = words[r][h][i], up = word >> 8;
            lo[r][h] = word & 0x000f000fu, lo[r][h + 2] = word & 0x00f000f0u;
            hi[r][h] = up & 0x000f000fu, hi[r][h + 2] = up & 0x00f000f0u;
          }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 b = lds_v4<S * 256 + i * 64>(x_at[j] + ahead * 2);
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            mma_f16(acc[r][j], lo[r], b.x, b.y);
            mma_f16(acc[r][j], hi[r], b.z, b.w);
          }
        }
      });
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float s = bits_f32<T>((uint16_t)v[r][h]);
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 2 * h; e < 2 * h + 2; ++e) total[r][j][e] = fmaf(s, acc[r][j][e], total[r][j][e]);
        }
    });
  }
  S1C_DEV void put(float* part) const {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[((r * NT + j) * 4 + e) * 32 + lane] = total[r][j][e];
  }
  S1C_DEV void add(const float* part) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) total[r][j][e] += part[((r * NT + j) * 4 + e) * 32 + lane];
  }
  // Bias, activation (0 none, 1 ReLU, 2 GELU with erf) and one rounding.
  S1C_DEV void store(int tile) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t n = (int64_t)tile * ROWS + r * 16 + e / 2 * 8 + g;
        if (n >= a.N) continue;
        const float b = a.bias ? a.bias[n] : 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int m = 8 * j + 2 * c + e % 2;
          if (m >= a.M) continue;
          float y = total[r][j][e] * (fminf(row_scale[m], 1.f) * 0x1p24f) * fmaxf(row_scale[m], 1.f);  // nothing in between underflows
          if (a.bias) y += b;
          if (a.act == 1) y = y < 0.f ? 0.f : y;  // keeps NaN
          if (a.act == 2) y = 0.5f * y * (1.f + erff(y * 0.70710678118654752f));
          const int64_t at = m * a.out_stride + n;
          if (a.out_f32)
            static_cast<float*>(a.out)[at] = y;
          else
            static_cast<T*>(a.out)[at] = from_f32<T>(y);
        }
      }
  }
};

// Stages columns [first, first + passes * 256) of x: f16 by a power of two for each row, in the order of
// the codes, and the groups' sums times -2^-24 (-8 * 2^-24 without zero points). A pair (row, part of its
// passes) belongs to one warp. PAIR: a block that is one of two in its cluster takes every second row, from
// `rank` on, and writes what it has staged to the other block too.
template <typename T, int GROUP, int WARPS, bool ZERO, bool PAIR>
S1C_DEV void nibble_stage(const NibbleArgs& a, __half* xs, float* sums, float* row_scale, uint32_t* tops, int pitch, int sum_pitch,
                          int first, int passes, int groups, int rank = 0, int blocks = 1) {
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  int rows = a.M;
  if constexpr (PAIR) rows = (a.M - rank + blocks - 1) / blocks;  // none for the second block of a single row
  const int parts = rows >= WARPS ? 1 : WARPS / (PAIR ? max(rows, 1) : rows);
  // where the lane's eight columns go among the 16 pieces of their 128: word j of lane c
  const int i = lane % 16;
  const int j = GROUP == 128 ? i % 4 : GROUP == 64 ? i / 8 * 2 + i % 2 : i / 4, c = GROUP == 128 ? i / 4 : GROUP == 64 ? i % 8 / 2 : i % 4;
  const int place = lane / 16 * 128 + (j * 4 + c) * 8;
  for (int p = w; p < rows * parts; p += WARPS) {
    const int m = PAIR ? rank + p / parts * blocks : p / parts;
    const int s0 = p % parts * passes / parts, s1 = (p % parts + 1) * passes / parts;
    uint32_t top = 0;
#pragma unroll 4
    for (int s = s0; s < s1; ++s) {
      const int k = first + s * 256 + lane * 8;
      uint32_t v[4] = {};
      const uint16_t* src = static_cast<const uint16_t*>(a.x) + m * a.x_stride + k;
      if (a.vec && k + 8 <= a.K) {
        const uint4 u = *reinterpret_cast<const uint4*>(src);
        v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < a.K) v[e / 2] |= (uint32_t)src[e] << (16 * (e % 2));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(fabsf(bits_f32<T>((uint16_t)(v[e / 2] >> (16 * (e % 2)))))));
      *reinterpret_cast<uint4*>(xs + m * pitch + s * 256 + place) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) atomicMax(&tops[m], top);
  }
  __syncthreads();
  if (PAIR && blocks > 1) cluster_wait();
  for (int p = w; p < rows * parts; p += WARPS) {
    const int m = PAIR ? rank + p / parts * blocks : p / parts;
    const int s0 = p % parts * passes / parts, s1 = (p % parts + 1) * passes / parts;
    // 2^up brings the largest value to [2^14, 2^15); rows with an infinity or NaN keep theirs
    const int e = (int)(tops[m] >> 23) - 127, up = e == 128 ? 0 : min(14 - e, 126);
    const float by = __uint_as_float((uint32_t)(127 + up) << 23);
    if (lane == 0) row_scale[m] = __uint_as_float((uint32_t)(127 - up) << 23);
    if (PAIR && blocks > 1 && lane == 0)
      cluster_put(cluster_address(row_scale + m, rank ^ 1), __uint_as_float((uint32_t)(127 - up) << 23));
#pragma unroll 2
    for (int s = s0; s < s1; ++s) {
      uint4* slot = reinterpret_cast<uint4*>(xs + m * pitch + s * 256 + place);
      const uint4 u = *slot;
      const uint32_t v[4] = {u.x, u.y, u.z, u.w};
      float f[8], sum = 0.f;
#pragma unroll
      for (int e2 = 0; e2 < 8; ++e2) f[e2] = bits_f32<T>((uint16_t)(v[e2 / 2] >> (16 * (e2 % 2)))) * by, sum += f[e2];
      const uint4 staged = make_uint4(pack_f16x2(f[0], f[4]), pack_f16x2(f[1] * 0.0625f, f[5] * 0.0625f), pack_f16x2(f[2], f[6]),
                                      pack_f16x2(f[3] * 0.0625f, f[7] * 0.0625f));
      *slot = staged;
      if (PAIR && blocks > 1) cluster_put(cluster_address(slot, rank ^ 1), staged);
#pragma unroll
      for (int o = 1; o < GROUP / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const int g = (s * 256 + lane * 8) / GROUP;
      if (lane % (GROUP / 8) == 0 && g < groups) {
        const float start = sum * (ZERO ? -0x1p-24f : -0x1p-21f);
        sums[m * sum_pitch + g] = start;
        if (PAIR && blocks > 1) cluster_put(cluster_address(sums + m * sum_pitch + g, rank ^ 1), start);
      }
    }
  }
}

template <typename T, int GROUP, int NT, int RT, int SPAN, int WARPS, bool ZERO>
__global__ void __launch_bounds__(WARPS * 32) nibble_kernel(const NibbleArgs a) {
  using W = NibbleWarp<T, GROUP, NT, RT, SPAN, WARPS, ZERO>;
  extern __shared__ __align__(128) uint8_t base[];
  pdl_trigger();
  const int rank = NT > 1 ? cluster_rank() : 0, blocks = NT > 1 ? cluster_blocks() : 1;
  if (blocks > 1) cluster_arrive();  // nibble_stage waits: the other block has begun
  pdl_wait();
  const bool split = a.split;
  const NibbleSmem sm(a.M, a.block, GROUP, W::RING, WARPS * W::PART, split);
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  __half* xs = reinterpret_cast<__half*>(base + sm.x);
  float* sums = reinterpret_cast<float*>(base + sm.sums);
  float* parts = reinterpret_cast<float*>(base + sm.parts);
  float* row_scale = reinterpret_cast<float*>(base + sm.misc);
  uint32_t* tops = reinterpret_cast<uint32_t*>(row_scale + 64);

  W p{a, row_scale, lane};
  p.setup(base + sm.ring + w * 2 * SPAN * W::STEP, xs, sums, sm.pitch, sm.sum_pitch);
  if (threadIdx.x < 64) tops[threadIdx.x] = 0;

  // This warp's spans f0 .. f0 + count - 1; span f is span f % spans of its tile f / spans.
  const int spans = (a.steps + SPAN - 1) / SPAN;
  int first, count, f0 = 0;
  if (split) {
    first = (int)((int64_t)a.tiles * blockIdx.x / gridDim.x);
    const int64_t all = ((int64_t)a.tiles * (blockIdx.x + 1) / gridDim.x - first) * spans;
    f0 = (int)(all * w / WARPS);
    count = (int)(all * (w + 1) / WARPS) - f0;
  } else {
    const int64_t supers = (a.tiles + WARPS - 1) / WARPS;
    count = (int)((supers - blockIdx.x + gridDim.x - 1) / gridDim.x) * spans;
    first = blockIdx.x * WARPS + w;
  }
  const int stride = split ? 1 : (int)gridDim.x * WARPS;
  int tile = first + f0 / spans * stride, step = f0 % spans * SPAN;  // the span to be used
  int next_tile = tile, next_step = step, left = count;              // the span to be loaded, and how many are left
  const auto load = [&](auto S, uint32_t side) {
    constexpr int s = decltype(S)::value;
    if (left > 0) {
      if (next_step + SPAN < a.steps)
        p.template load<s, false>(next_step + s, side);
      else if (next_step + s < a.steps)
        p.template load<s, true>(next_step + s, side);
    }
    copy_commit();  // a group for each step, so that waiting can count them
  };
  const auto loaded = [&] {
    --left;
    if (next_step + SPAN < a.steps) {
      next_step += SPAN;
      p.advance();
    } else {
      next_step = 0, next_tile += stride;
      p.point(next_tile, 0);
    }
  };
  p.point(tile, step);
  static_for<SPAN>([&](auto S) { load(S, 0); });
  if (left > 0) p.fetch(p.sz[0], next_step);
  loaded();
  __syncthreads();
  if (split) {
    nibble_stage<T, GROUP, WARPS, ZERO, (NT > 1)>(a, xs, sums, row_scale, tops, sm.pitch, sm.sum_pitch, 0, (a.steps + 1) / 2, a.steps * W::GP, rank, blocks);
    if (blocks > 1) cluster_arrive(), cluster_wait();  // the other block's rows have landed
    __syncthreads();
  }
  p.clear();
  bool whole = step == 0;      // the tile's first span is in `total`
  int at = split ? step : 0;   // step within the staged part of x
  for (int i = 0; i < count; ++i) {
    if (!split && at == 0) {
      // the next columns of x; a tile's totals so far go over to its new row scales, which only grow
      float old[NT][2];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) old[j][e] = row_scale[min(a.M - 1, 8 * j + 2 * (lane & 3) + e)];
      if (step == 0 && threadIdx.x < 64) tops[threadIdx.x] = 0;
      __syncthreads();
      const int steps = min(a.block, a.steps - step);
      nibble_stage<T, GROUP, WARPS, ZERO, (NT > 1)>(a, xs, sums, row_scale, tops, sm.pitch, sm.sum_pitch, step * 128, (steps + 1) / 2, steps * W::GP);
      __syncthreads();
      if (step) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float by = old[j][e % 2] / row_scale[min(a.M - 1, 8 * j + 2 * (lane & 3) + e % 2)];
#pragma unroll
            for (int r = 0; r < RT; ++r) p.total[r][j][e] *= by;
          }
      }
    }
    const int have = a.steps - step;
    const uint32_t side = i & 1;
    if (left > 0) p.fetch(p.sz[1], next_step);
    if (left > 0 && have >= SPAN && next_step + SPAN < a.steps) {
      // whole spans: no step to ask about
      static_for<SPAN>([&](auto S) {
        constexpr int s = decltype(S)::value;
        p.template load<s, false>(0, side ^ 1);
        copy_commit();
        copy_wait<SPAN>();
        __syncwarp();
        p.template consume<s>(at * 128, side);
      });
    } else {
      static_for<SPAN>([&](auto S) {
        constexpr int s = decltype(S)::value;
        load(S, side ^ 1);
        copy_wait<SPAN>();
        __syncwarp();
        if (s < have) p.template consume<s>(at * 128, side);
      });
    }
    loaded();
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < W::NS; ++j) p.sz[0][r][h][j] = p.sz[1][r][h][j];
    const bool done = have <= SPAN;
    if (done || (split && i == count - 1 && !whole)) {
      if (whole)
        p.store(tile);
      else
        p.put(parts + w * W::PART);  // a piece that begins inside its tile
      p.clear();
      whole = true;
    }
    step += SPAN, at += SPAN;
    if (done) step = 0, tile += stride, at = 0;
    if (!split && at == a.block) at = 0;
  }
  if (!split) return;
  // Tiles split between warps: the warp with the first piece, which it still holds, adds the later ones in
  // order.
  __syncthreads();
  const int end = f0 + count, t0 = (end - 1) / spans * spans;
  if (count == 0 || end % spans == 0 || t0 < f0) return;
  const int64_t all = ((int64_t)a.tiles * (blockIdx.x + 1) / gridDim.x - first) * spans;
  for (int o = w + 1; o < WARPS; ++o) {
    const int o0 = (int)(all * o / WARPS), o1 = (int)(all * (o + 1) / WARPS);
    if (o0 == o1) continue;
    p.add(parts + o * W::PART);
    if (o1 >= t0 + spans) break;
  }
  p.store(first + t0 / spans);
}

}  // namespace s1c
