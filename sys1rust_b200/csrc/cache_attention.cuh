// Causal attention of new rows over the 8-bit paged cache of kvcache.cuh. A sequence of L cached
// rows has c query rows, the last c positions: query i stands at p = L - c + i and sees the keys
// j <= p, with j >= p - window where a window is given, on pages inside the cache.
//   o = sum_j softmax_j(scale * q . k_j) v_j,   lse = ln sum_j exp(scale * q . k_j)
// A query that sees no key gets o = 0 and lse = -inf.
//
// The rows of a key head are (query row, query head of its group); a tile of 16 is the m of
// mma.m16n8k16. Keys pass in tiles of 32, by TMA from their pages (swizzled, so that the reads below are free
// of bank conflicts), with a running maximum and sum. Codes become f16 operands in registers:
//
//  - keys: the byte code + 128 at the bottom of a half is the subnormal (code + 128) * 2^-24, which the tensor
//    cores take exactly; the products' sum starts at -128 * 2^-24 * sum(q), so nothing is subtracted. q is
//    scaled by a power of two for each row to about 2^14, which keeps all bits of bf16 and f16. The order of dimensions inside the
//    sum is free: a lane's 32-bit word holds four neighbours.
//  - values: the sum runs over keys, so a register pairs two keys' codes of one dimension; words of two
//    keys are interleaved by byte permutes, put under the exponent of 1024 and 1152 subtracted.
//  - a page's value scale differs from its neighbours' inside one sum, so it goes into the weight: with t = log2(scale /
//    largest scale of the block), the weight is exp2(s + t - m + 14.5), m a running maximum of s + t, and the sum of
//    the softmax adds weight * 2^-t. m follows the true maximum only when that is 1.25 ahead, so outputs are
//    seldom rescaled. Weights are held as f16: at most 2^15.75, with all 11 bits down to 2^-28 of the
//    largest; scores, maxima, sums and outputs are fp32.
//
// Few query rows (bound by the cache's bytes): each warp has its own tiles of the block's keys and its own ring
// of loads, so nothing waits inside the loop; the four warps' results are joined at the end. Many rows (bound by
// the tensor cores and the codes' conversion): each warp has its own 16 rows, and the tiles are shared. Long
// caches are split over blocks, whose results a second kernel joins.
#pragma once
#include <cuda.h>
#include <limits.h>

#include "kvcache.cuh"
#include "mma.cuh"

namespace s1c {

struct CacheAttnArgs {
  const void* q;
  void* out;
  float* lse;  // nullable
  int64_t q_stride, out_stride;
  const int* cu;     // [n + 1] query rows
  const int* len;    // [n] cached rows, the query rows' own among them
  const int* table;  // [n, max_pages]
  int n, heads, max_pages, max_q, window;
  int tiles;         // row tiles (of a block) that a sequence has at most
  int chunk;         // keys of a block, a multiple of 128
  int chunks;        // blocks that share a sequence's keys
  float scale_log2;  // scale * log2(e)
  float* part;       // [n * max_q * heads, chunks, dim]: normalised outputs of the chunks
  float* part_lse;   // [n * max_q * heads, chunks]: their log2 sums
};

constexpr int CATT_WARPS = 4, CATT_TK = 32, CATT_PAGES = 128;  // keys of a tile; pages of a chunk at most

template <int D, bool SHARE>
struct CacheAttnSmem {
  static constexpr int TILE = 2 * CATT_TK * D;  // keys and values of a tile
  static constexpr int STAGES = SHARE ? 4 : D == 128 ? 2 : 4;
  static constexpr int RINGS = SHARE ? 1 : CATT_WARPS;
  alignas(1024) uint8_t ring[RINGS][STAGES][TILE];
  uint4 q[SHARE ? CATT_WARPS : 1][D / 16][32];  // operands of the query rows
  uint64_t full[RINGS][STAGES], empty[STAGES];
  float4 page[CATT_PAGES + 2];  // key scale * 2^24, t, 2^-t, page (-1 outside the cache: 0, -inf, 0)
  float top[CATT_WARPS];
  float row_m[CATT_WARPS][16], row_l[CATT_WARPS][16];
};

template <typename T, int D, bool SHARE>
__global__ void __launch_bounds__(CATT_WARPS * 32, 3)
cache_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const CacheView c,
                       const CacheAttnArgs a) {
  using S = CacheAttnSmem<D, SHARE>;
  extern __shared__ uint8_t raw[];
  S& sm = *reinterpret_cast<S*>(raw + (1024 - smem_u32(raw) % 1024) % 1024);
  constexpr int ROWS = SHARE ? 16 * CATT_WARPS : 16, QK = D / 16, SEG = D / 32;
  const int tid = threadIdx.x, w = tid / 32, lane = tid % 32, g = lane >> 2, cq = lane & 3;
  const int G = a.heads / c.heads;

  // later row tiles have more keys: they come first
  const int h = blockIdx.x % c.heads, seq = blockIdx.x / c.heads % a.n, qt = a.tiles - 1 - blockIdx.x / c.heads / a.n;
  const int first = a.cu[seq], count = a.cu[seq + 1] - first, L = a.len[seq];
  const int rows = min(count, a.max_q) * G, row0 = qt * ROWS;
  pdl_trigger();
  if (row0 >= rows) return;
  const int chunk = blockIdx.y;
  // keys that some row of the block sees, in this chunk
  const int pos0 = L - count + row0 / G, pos1 = L - count + (min(row0 + ROWS, rows) - 1) / G;
  const int window = a.window < 0 ? INT_MAX / 2 : min(a.window, INT_MAX / 2);  // positions stay below that
  const int reach = (int)min((int64_t)a.max_pages * c.page, (int64_t)INT_MAX / 2);
  const int lo = max(max(0, pos0 - window) / CATT_TK * CATT_TK, chunk * a.chunk);
  const int hi = (int)min((int64_t)min(pos1 + 1, reach), ((int64_t)chunk + 1) * a.chunk);
  const int tiles = hi > lo ? (hi - lo + CATT_TK - 1) / CATT_TK : 0;
  const int shift = 31 - __clz(c.page);  // page is a power of two

  // this warp's rows
  const int wrow0 = SHARE ? row0 + w * 16 : row0;
  int64_t at_row[2];
  int head[2];
  int qpos[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = min(wrow0 + g + 8 * e, rows - 1);
    at_row[e] = first + r / G;
    head[e] = h * G + r % G;
    qpos[e] = L - count + r / G;
  }

  if (tiles > 0) {
    if (tid == 0) {
#pragma unroll
      for (int i = 0; i < S::STAGES; ++i) {
        for (int r = 0; r < S::RINGS; ++r) mbar_init(&sm.full[r][i], 1);
        mbar_init(&sm.empty[i], CATT_WARPS);
      }
      fence_barrier_init();
    }
    // the chunk's pages and scales
    const int p0 = lo >> shift, pages = ((hi - 1) >> shift) - p0 + 1;
    float top = 0.f;
    for (int i = tid; i < pages + 2; i += CATT_WARPS * 32) {
      const int page = i < pages ? cache_page(a.table, a.max_pages, seq, p0 + i, c.num_pages) : -1;
      float ks = 0.f, vs = 0.f;
      if (page >= 0) {
        const int64_t slot = (int64_t)page * c.heads + h;
        ks = c.scales[0][slot], vs = c.scales[1][slot];
      }
      sm.page[i] = make_float4(ks * 0x1p24f, vs, 0.f, __int_as_float(page));
      top = fmaxf(top, vs);
    }
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) sm.top[w] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sm.top[0], sm.top[1]), fmaxf(sm.top[2], sm.top[3]));
    for (int i = tid; i < pages + 2; i += CATT_WARPS * 32) {
      float4 e = sm.page[i];
      // scales below 2^-60 of the largest (and zero ones, whose codes are zero) count as that
      const float l2 = top > 0.f ? fmaxf(log2f(e.y / top), -60.f) : 0.f;
      const bool in = __float_as_int(e.w) >= 0;
      e.y = in ? l2 : -INFINITY, e.z = in ? exp2f(-l2) : 0.f;
      sm.page[i] = e;
    }
    __syncthreads();
  }
  const float v_top = tiles > 0 ? fmaxf(fmaxf(sm.top[0], sm.top[1]), fmaxf(sm.top[2], sm.top[3])) : 0.f;

  // Loads of tile i into its slot, by a whole warp: a lane for each page (one, or two of 16 rows). Pages outside the
  // cache are not read.
  const int per = min(c.page, CATT_TK), boxes = CATT_TK / per;
  const auto issue = [&](int i) {
    const int ring = SHARE ? 0 : w, slot = (SHARE ? i : i / CATT_WARPS) % S::STAGES;
    const int at = lo + i * CATT_TK + lane * per;
    uint64_t* bar = &sm.full[ring][slot];
    const int page = lane < boxes && at < hi ? __float_as_int(sm.page[(at >> shift) - (lo >> shift)].w) : -1;
    const int count = __popc(__ballot_sync(0xffffffffu, page >= 0));
    if (lane == 0) mbar_arrive_expect_tx(bar, count * 2 * per * D);
    __syncwarp();
    if (page >= 0) {
      const int y = (page * c.heads + h) * c.page + (at & (c.page - 1));
      tma_load_2d(sm.ring[ring][slot] + lane * per * D, &k_map, bar, 0, y);
      tma_load_2d(sm.ring[ring][slot] + CATT_TK * D + lane * per * D, &v_map, bar, 0, y);
    }
    __syncwarp();
  };
  const int step = SHARE ? 1 : CATT_WARPS, begin = SHARE ? 0 : w;
  if (!SHARE || w == 0)
    for (int s = 0; s < (SHARE ? S::STAGES - 1 : S::STAGES); ++s)
      if (begin + s * step < tiles) issue(begin + s * step);

  // q as operands: lane (g, cq) holds dimensions 16 i + 4 cq .. + 3 of rows g and g + 8
  float factor[2], start[2];
  {
  uint32_t qa[QK][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const T* q = static_cast<const T*>(a.q) + at_row[e] * a.q_stride + head[e] * D + cq * 4;
    float f[QK][4], top = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < QK; ++i) {
      const uint2 v = *reinterpret_cast<const uint2*>(q + i * 16);
      f[i][0] = bits_f32<T>((uint16_t)v.x), f[i][1] = bits_f32<T>((uint16_t)(v.x >> 16));
      f[i][2] = bits_f32<T>((uint16_t)v.y), f[i][3] = bits_f32<T>((uint16_t)(v.y >> 16));
#pragma unroll
      for (int j = 0; j < 4; ++j) top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(fabsf(f[i][j]))));
    }
    for (int o = 1; o < 4; o <<= 1)
      top = __uint_as_float(max(__float_as_uint(top), __shfl_xor_sync(0xffffffffu, __float_as_uint(top), o)));
    const int ex = (int)(__float_as_uint(top) >> 23) - 127, up = ex == 128 ? 0 : min(14 - ex, 100);
    const float by = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
    for (int i = 0; i < QK; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[i][j] *= by, sum += f[i][j];
      qa[i][e] = pack_f16x2(f[i][0], f[i][1]), qa[i][e + 2] = pack_f16x2(f[i][2], f[i][3]);
    }
    for (int o = 1; o < 4; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    factor[e] = a.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
    start[e] = sum * -0x1p-17f;  // -128 * 2^-24
  }
  if (SHARE || w == 0)
#pragma unroll
    for (int i = 0; i < QK; ++i) sm.q[SHARE ? w : 0][i][lane] = make_uint4(qa[i][0], qa[i][1], qa[i][2], qa[i][3]);
  if (SHARE)
    __syncwarp();
  else
    __syncthreads();
  }
  const uint32_t q_at = smem_u32(&sm.q[SHARE ? w : 0][0][lane]);

  // shared offsets in a slot: the swizzle moves a row's 16-byte pieces by the row (128-byte rows) or by half of it
  const int kr = D == 128 ? g : (g & 4) | (g & 1) << 1 | (g >> 1 & 1);
  uint32_t k_at[QK], v_at[2][SEG];
#pragma unroll
  for (int i = 0; i < QK; ++i) k_at[i] = kr * D + ((i ^ (D == 128 ? kr & 7 : kr >> 1 & 3)) << 4) + cq * 4;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int n = 2 * cq + e, t = D == 128 ? n : (n & 4) | (n & 1) << 1 | (n >> 1 & 1);
#pragma unroll
    for (int s = 0; s < SEG; ++s)
      v_at[e][s] = CATT_TK * D + t * D + (((2 * s + (g >> 2)) ^ (D == 128 ? t & 7 : t >> 1 & 3)) << 4) + (g & 3) * 4;
  }
  // where the columns 2 cq, 2 cq + 1 of a tile of scores stand among its eight keys
  const int kc0 = D == 128 ? 2 * cq : (cq & 2) << 1 | (cq & 1), kc1 = D == 128 ? 2 * cq + 1 : kc0 + 2;

  float o[SEG * 4][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < SEG * 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

  bool broken = false;
  int turn = 0;  // tiles this ring has been through
  for (int i = begin; i < tiles; i += step, ++turn) {
    const int slot = turn % S::STAGES;
    const uint32_t phase = turn / S::STAGES & 1;
    if (SHARE && w == 0 && i + S::STAGES - 1 < tiles) {
      // the slot of tile i - 1, when all warps are through with it
      const int prev = (i + S::STAGES - 1) % S::STAGES;
      if (i > 0 && !broken && !mbar_wait_warp(&sm.empty[prev], ((i - 1) / S::STAGES) & 1, nullptr, 0, nullptr)) broken = true;
      if (!broken) issue(i + S::STAGES - 1);
    }
    if (!broken && !mbar_wait_warp(&sm.full[SHARE ? 0 : w][slot], phase, nullptr, 0, nullptr)) broken = true;
    if (broken) break;
    const uint32_t base = smem_u32(sm.ring[SHARE ? 0 : w][slot]);
    const int key = lo + i * CATT_TK, pg = (key >> shift) - (lo >> shift);

    // scores, in units of the key scale * factor
    float s[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j][0] = s[j][1] = start[0], s[j][2] = s[j][3] = start[1];
    static_for<QK>([&](auto DD) {
      constexpr int d = decltype(DD)::value;
      const uint32_t at = base + k_at[d];
      const uint4 qv = lds_v4<d * 512>(q_at);
      const uint32_t qa[4] = {qv.x, qv.y, qv.z, qv.w};
      static_for<4>([&](auto J) {
        constexpr int j = decltype(J)::value;
        const uint32_t v = lds_u32<j * 8 * D>(at) ^ 0x80808080u;
        mma_f16(s[j], qa, __byte_perm(v, 0, 0x4140), __byte_perm(v, 0, 0x4342));
      });
    });
    // log2 of the weights; masked where the tile is not seen in whole
    const bool open = key + CATT_TK - 1 <= qpos[0] && key >= qpos[1] - window && key + CATT_TK <= hi;
    float top[2] = {-INFINITY, -INFINITY}, inv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 p = sm.page[pg + (((key & (c.page - 1)) + j * 8) >> shift)];
      inv[j] = p.z;
      const float f0 = factor[0] * p.x, f1 = factor[1] * p.x;
      s[j][0] = fmaf(s[j][0], f0, p.y), s[j][1] = fmaf(s[j][1], f0, p.y);
      s[j][2] = fmaf(s[j][2], f1, p.y), s[j][3] = fmaf(s[j][3], f1, p.y);
    }
    if (!__all_sync(0xffffffffu, open)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // key + 8 j + kc within [qpos - window, min(qpos, hi - 1)]
        const int last = min(qpos[e], hi - 1) - key, from = qpos[e] - window - key;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j * 8 + kc0 > last || j * 8 + kc0 < from) s[j][2 * e] = -INFINITY;
          if (j * 8 + kc1 > last || j * 8 + kc1 < from) s[j][2 * e + 1] = -INFINITY;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e / 2] = fmaxf(top[e / 2], s[j][e]);
    bool grows = false;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
      grows |= top[e] > m[e] + 1.25f;
    }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float n = fmaxf(m[e], top[e]), keep = m[e] == -INFINITY ? 0.f : exp2f(m[e] - n);
        m[e] = n, l[e] *= keep;
#pragma unroll
        for (int i2 = 0; i2 < SEG * 4; ++i2) o[i2][2 * e] *= keep, o[i2][2 * e + 1] *= keep;
      }
    }
    // weights times 2^14.5, and their sum without the value scales
    const float off[2] = {m[0] == -INFINITY ? 0.f : 14.5f - m[0], m[1] == -INFINITY ? 0.f : 14.5f - m[1]};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = exp2_approx(s[j][e] + off[e / 2]);
        l[e / 2] = fmaf(s[j][e], inv[j], l[e / 2]);
      }
    // outputs
    uint32_t pa[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      pa[k][0] = pack_f16x2(s[2 * k][0], s[2 * k][1]), pa[k][1] = pack_f16x2(s[2 * k][2], s[2 * k][3]);
      pa[k][2] = pack_f16x2(s[2 * k + 1][0], s[2 * k + 1][1]), pa[k][3] = pack_f16x2(s[2 * k + 1][2], s[2 * k + 1][3]);
    }
#pragma unroll
    for (int q = 0; q < SEG; ++q) {
      const uint32_t at0 = base + v_at[0][q], at1 = base + v_at[1][q];
      static_for<2>([&](auto KK) {
        constexpr int k = decltype(KK)::value;
        uint32_t b[4][2];
        static_for<2>([&](auto E) {
          constexpr int e = decltype(E)::value;
          const uint32_t x = lds_u32<(k * 16 + e * 8) * D>(at0) ^ 0x80808080u, y = lds_u32<(k * 16 + e * 8) * D>(at1) ^ 0x80808080u;
          const uint32_t even = __byte_perm(x, y, 0x6420), odd = __byte_perm(x, y, 0x7531);
          b[0][e] = code_pair(__byte_perm(even, 0x64646464u, 0x4240)), b[1][e] = code_pair(__byte_perm(odd, 0x64646464u, 0x4240));
          b[2][e] = code_pair(__byte_perm(even, 0x64646464u, 0x4341)), b[3][e] = code_pair(__byte_perm(odd, 0x64646464u, 0x4341));
        });
#pragma unroll
        for (int d = 0; d < 4; ++d) mma_f16(o[q * 4 + d], pa[k], b[d][0], b[d][1]);
      });
    }
    if (SHARE) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[slot]);
    } else {
      __syncwarp();
      if (i + S::STAGES * step < tiles) issue(i + S::STAGES * step);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
  }

  // One row's result: o / l and log2 of the sum. Without a key l is 0: o = 0 and -inf.
  const auto put = [&](int64_t grow, int hd, int d, const float* v, int n, float sum, float max_) {
    const float by = sum == 0.f ? 0.f : v_top / sum, log_sum = sum == 0.f ? -INFINITY : max_ - 14.5f + log2f(sum);
    if (a.chunks > 1) {
      const int64_t at = ((int64_t)(seq * a.max_q + (grow - first)) * a.heads + hd) * a.chunks + chunk;
      for (int i = 0; i < n; ++i) a.part[at * D + d + i] = v[i] * by;
      if (d == 0) a.part_lse[at] = log_sum;
    } else {
      T* dst = static_cast<T*>(a.out) + grow * a.out_stride + hd * D + d;
      for (int i = 0; i < n; ++i) dst[i] = from_f32<T>(v[i] * by);
      if (a.lse && d == 0) a.lse[grow * a.heads + hd] = log_sum * 0.69314718055994531f;
    }
  };
  if (SHARE) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (wrow0 + g + 8 * e >= rows) continue;
#pragma unroll
      for (int q = 0; q < SEG; ++q) {
        // n = 2 cq and 2 cq + 1 of the four tiles: eight neighbouring dimensions
        float v[8];
#pragma unroll
        for (int d = 0; d < 4; ++d) v[d] = o[q * 4 + d][2 * e], v[4 + d] = o[q * 4 + d][2 * e + 1];
        put(at_row[e], head[e], q * 32 + cq * 8, v, 8, l[e], m[e]);
      }
    }
    return;
  }
  // join the four warps
  __syncthreads();  // the rings are free
  float* all = reinterpret_cast<float*>(sm.ring[0][0]);  // [warp][16][D]
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = g + 8 * e;
    if (cq == 0) sm.row_m[w][r] = m[e], sm.row_l[w][r] = l[e];
#pragma unroll
    for (int q = 0; q < SEG; ++q)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        all[(w * 16 + r) * D + q * 32 + cq * 8 + d] = o[q * 4 + d][2 * e];
        all[(w * 16 + r) * D + q * 32 + cq * 8 + 4 + d] = o[q * 4 + d][2 * e + 1];
      }
  }
  __syncthreads();
  for (int i = tid; i < 16 * D / 4; i += CATT_WARPS * 32) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    if (row0 + r >= rows) break;
    float big = -INFINITY, sum = 0.f, v[4] = {};
    for (int x = 0; x < CATT_WARPS; ++x) big = fmaxf(big, sm.row_m[x][r]);
    for (int x = 0; x < CATT_WARPS; ++x) {
      const float by = sm.row_m[x][r] == -INFINITY ? 0.f : exp2f(sm.row_m[x][r] - big);
      sum += sm.row_l[x][r] * by;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += all[(x * 16 + r) * D + d + e] * by;
    }
    put(first + (row0 + r) / G, h * G + (row0 + r) % G, d, v, 4, sum, big);
  }
}

// Joins the chunks of a row: weights 2^(lse - max). One block for each row and head; its warps share the
// chunks, several loads of each in flight, and are summed in order.
template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) cache_attention_join_kernel(const CacheAttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float tops[WARPS], sums[WARPS], outs[WARPS][D];
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t item = blockIdx.x;  // (sequence, row, head)
  const int head = (int)(item % a.heads), i = (int)(item / a.heads % a.max_q);
  const int64_t seq = item / a.heads / a.max_q;
  pdl_wait();
  const int first = a.cu[seq];
  if (i >= a.cu[seq + 1] - first) return;
  const float* lse = a.part_lse + item * a.chunks;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < a.chunks; s += WARPS * 32) top = fmaxf(top, lse[s]);
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[w] = top;
  __syncthreads();
  for (int j = 0; j < WARPS; ++j) top = fmaxf(top, tops[j]);
  float sum = 0.f, o[E] = {};
  if (top != -INFINITY) {
#pragma unroll 8
    for (int s = w; s < a.chunks; s += WARPS) {
      const float by = exp2f(lse[s] - top);
      const float* p = a.part + (item * a.chunks + s) * D + lane * E;
      float v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = p[e];
      sum += by;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += by == 0.f ? 0.f : by * v[e];  // a chunk without a key has written no output
    }
  }
  if (lane == 0) sums[w] = sum;
#pragma unroll
  for (int e = 0; e < E; ++e) outs[w][lane * E + e] = o[e];
  __syncthreads();
  sum = 0.f;
  for (int j = 0; j < WARPS; ++j) sum += sums[j];
  const int64_t row = first + i;
  for (int d = threadIdx.x; d < D; d += WARPS * 32) {
    float v = 0.f;
    for (int j = 0; j < WARPS; ++j) v += outs[j][d];
    static_cast<T*>(a.out)[row * a.out_stride + head * D + d] = from_f32<T>(sum == 0.f ? 0.f : v / sum);
  }
  if (a.lse && threadIdx.x == 0) a.lse[row * a.heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace s1c
