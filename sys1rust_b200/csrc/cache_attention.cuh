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
//    scaled by a power of two for each row to about 2^14, which keeps all bits of bf16 and f16. The order of
//    dimensions inside the sum is free: a lane's 32-bit word holds four neighbours.
//  - values: the sum runs over keys, so a register pairs two keys' codes of one dimension; words of two
//    keys are interleaved by byte permutes, put under the exponent of 1024 and 1152 subtracted.
//  - a page's value scale differs from its neighbours' inside one sum, so it goes into the weight: with t =
//    log2(scale / largest scale of the block), the weight is exp2(s + t - m + 14), m a running maximum of s + t,
//    and the sum of the softmax adds weight * 2^-t (scales more than 2^90 apart: weights of its own). m follows
//    the true maximum only when that is 1.75 ahead, so outputs are seldom rescaled. Weights are held as f16 (two
//    of them for f16 results): at most 2^15.75, with all 11 bits down to 2^-28 of the largest; scores, maxima,
//    sums and outputs are fp32.
//
// Few query rows (bound by the cache's bytes): each warp has its own tiles of the block's keys and its own
// ring of loads, so nothing waits inside the loop; the four warps' results are joined at the end. Long
// caches are split over blocks, whose results a second kernel joins.
//
// A wait that runs out makes the rows of its block NaN.
//
// Many rows: a block of 128 rows on the 5th-generation tensor cores. Four warps convert a tile of 64 keys
// once for all rows, to f16 in shared memory (whole codes, so no scale enters before the scores); one
// thread issues S = Q K^T into one of two buffers of TMEM, a tile ahead, and O += P V; four warps have a
// row in each thread, and write the weights P over the scores they come from, where the second product
// reads them as its first operand.
//
// Measured: 64 sequences of 4096 to 8192 keys, 32 heads on 8 of 128, pages of 16: 163 us, 4.8 TB/s. Its 850
// instructions for a tile of 32 keys, most of them conversions, fill half of the issue slots; at three blocks an SM
// (168 registers) a scheduler has three warps, and waits for their dependent instructions the other half. 1 x
// 131072 keys in f16: 40 us, 3.4 TB/s (36 us with weights of 11 bits), with one round of blocks and 3 us to join them;
// 1 x 700: 8.1 us, two launches. Prompts, 4 x 512 rows over 2048 to 4096 keys, 16 heads on 4: 115 us, 465 TFLOP/s;
// on mma.m16n8k16 the same took 326 us, of shared memory reads. There 256 blocks lie unevenly on 148 SMs, and
// the softmax threads wait for the scores a third of the time.
#pragma once
#include <cuda.h>
#include <limits.h>

#include "kvcache.cuh"
#include "mma.cuh"
#include "tmem.cuh"

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
  uint64_t wait_ns = S1C_WAIT_BUDGET_NS;  // of a wait; rows of a block in which one runs out become NaN
  int beyond = 0;                         // bytes that a tile waits for beyond its own (a self-test: they never come)
};

constexpr int CATT_TK = 32;   // keys of a tile: few rows
constexpr int CATP_TK = 64;   // many rows
constexpr int CATT_BOX = 32;  // rows of a TMA box at most

constexpr int ATTN_BEYOND = 4;  // entries of the list of pages behind the last page

// What a block works on: `rows` rows from row0 on of one sequence and key head, keys [lo, hi) in `tiles` tiles.
struct AttnUnit {
  int h, seq, first, count, L, rows, row0, chunk, lo, hi, tiles, window, shift, G;
  bool wide = false;  // value scales more than 2^90 apart
};
template <int ROWS, int TK>
S1C_DEV bool attn_unit(const CacheView& c, const CacheAttnArgs& a, AttnUnit& u) {
  // later row tiles have more keys: they come first
  u.h = blockIdx.x % c.heads, u.seq = blockIdx.x / c.heads % a.n, u.G = a.heads / c.heads;
  u.first = a.cu[u.seq], u.count = a.cu[u.seq + 1] - u.first, u.L = a.len[u.seq];
  u.rows = min(u.count, a.max_q) * u.G, u.row0 = (a.tiles - 1 - blockIdx.x / c.heads / a.n) * ROWS;
  if (u.row0 >= u.rows) return false;
  u.chunk = blockIdx.y;
  u.shift = 31 - __clz(c.page);                                          // page is a power of two
  u.window = a.window < 0 ? INT_MAX / 2 : min(a.window, INT_MAX / 2);  // positions stay below that
  // keys that some row sees, in this chunk
  const int pos0 = u.L - u.count + u.row0 / u.G, pos1 = u.L - u.count + (min(u.row0 + ROWS, u.rows) - 1) / u.G;
  const int reach = (int)min((int64_t)a.max_pages * c.page, (int64_t)INT_MAX / 2);
  u.lo = max(max(0, pos0 - u.window) / CATT_BOX * CATT_BOX, u.chunk * a.chunk);
  u.hi = (int)min((int64_t)min(pos1 + 1, reach), ((int64_t)u.chunk + 1) * a.chunk);
  u.tiles = u.hi > u.lo ? (u.hi - u.lo + TK - 1) / TK : 0;
  return true;
}

// The chunk's pages: (key scale * 2^24, t, 2^-t, page), a few more than there are, without a page (-1) 0,
// -inf, 0. Returns the largest value scale, which the outputs are multiplied by. All threads call.
//
// 2^-t times a weight stays in range down to t = -90: the sum is then below 2^(15.75 + 90 + 14) for the 2^14 keys
// of a chunk. Where scales lie further apart (padding of any bits may have got into a page), u.wide is set, and
// the sum is formed from weights of its own, without t (attn_wide). Zero scales, whose codes are zero, count as the
// smallest t.
template <int WARPS>
S1C_DEV float attn_pages(const CacheView& c, const CacheAttnArgs& a, AttnUnit& u, float4* list, float2* ends) {
  const int tid = threadIdx.x, p0 = u.lo >> u.shift, pages = ((u.hi - 1) >> u.shift) - p0 + 1;  // and more behind them than a tile has
  float top = 0.f, low = INFINITY;  // the largest scale, the smallest but 0
  for (int i = tid; i < pages + ATTN_BEYOND; i += WARPS * 32) {
    const int page = i < pages ? cache_page(a.table, a.max_pages, u.seq, p0 + i, c.num_pages) : -1;
    float ks = 0.f, vs = 0.f;
    if (page >= 0) {
      const int64_t slot = (int64_t)page * c.heads + u.h;
      ks = c.scales[0][slot], vs = c.scales[1][slot] + 0.f;  // no -0
    }
    list[i] = make_float4(ks * 0x1p24f, vs, 0.f, __int_as_float(page));
    top = fmaxf(top, vs), low = vs > 0.f ? fminf(low, vs) : low;
  }
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));  // not negative: ordered as integers are
  low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(low)));
  if (tid % 32 == 0) ends[tid / 32] = make_float2(top, low);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WARPS; ++i) top = fmaxf(top, ends[i].x), low = fminf(low, ends[i].y);
  u.wide = low < top * 0x1p-90f;
  for (int i = tid; i < pages + ATTN_BEYOND; i += WARPS * 32) {
    float4 e = list[i];
    const float l2 = !(top > 0.f) ? 0.f : u.wide ? fmaxf(log2f(e.y) - log2f(top), -300.f) : fmaxf(log2f(e.y / top), -90.f);
    const bool in = __float_as_int(e.w) >= 0;
    e.y = in ? l2 : -INFINITY, e.z = in && !u.wide ? exp2f(-l2) : 0.f;
    list[i] = e;
  }
  __syncthreads();
  return top;
}

// A running maximum and sum of exp2(score) in shared memory, one for each row of a thread: (maximum, sum).
template <int N>
S1C_DEV void attn_wide_add(float2& w, float top, const float (&scores)[N]) {
  const float n = fmaxf(w.x, top), from = n == -INFINITY ? 0.f : n;
  w.y *= exp2f(w.x - from);
  w.x = n;
#pragma unroll
  for (int i = 0; i < N; ++i) w.y += exp2_approx(scores[i] - from);
}
// What outputs o are multiplied by, by and with log2 of the sum, where scales lie far apart: o is in units of
// v_top * 2^(m - 14).
S1C_DEV float attn_wide_out(float o, float v_top, float m, float2 w) {
  return w.y == 0.f ? 0.f : (float)((double)o * v_top * exp2((double)m - 14.0 - w.x) / w.y);
}

// TMA of one tile's keys and values to `dst`, by a whole warp: a lane for each page or 32 rows of one.
// Pages outside the cache are not read.
template <int D, int TK>
S1C_DEV void attn_issue(const CacheView& c, const CacheAttnArgs& a, const AttnUnit& u, const float4* list, const CUtensorMap& k_map, const CUtensorMap& v_map, int i,
                        uint8_t* dst, uint64_t* bar) {
  const int lane = threadIdx.x % 32, per = min(c.page, CATT_BOX), boxes = TK / per;
  const int at = u.lo + i * TK + lane * per;
  const int page = lane < boxes && at < u.hi ? __float_as_int(list[(at >> u.shift) - (u.lo >> u.shift)].w) : -1;
  const int count = __popc(__ballot_sync(0xffffffffu, page >= 0));
  if (lane == 0) mbar_arrive_expect_tx(bar, count * 2 * per * D + a.beyond);
  __syncwarp();
  if (page >= 0) {
    const int y = (page * c.heads + u.h) * c.page + (at & (c.page - 1));
    tma_load_2d(dst + lane * per * D, &k_map, bar, 0, y);
    tma_load_2d(dst + TK * D + lane * per * D, &v_map, bar, 0, y);
  }
  __syncwarp();
}

// A row's power of two, which brings its largest value to [2^14, 2^15), and the factor that undoes it. A row with
// an infinity or NaN counts as zeros, marked by a factor of -0, up to its end, where its sum becomes NaN if it
// has seen a key: nothing of it can then reach a place without one.
S1C_DEV float attn_up(float top, float scale, float& factor) {
  const int up = min(14 - ((int)(__float_as_uint(top) >> 23) - 127), 100);
  factor = top < INFINITY ? scale * __uint_as_float((uint32_t)(127 - up) << 23) + 0.f : -0.f;
  return __uint_as_float((uint32_t)(127 + up) << 23);
}
S1C_DEV float attn_sum(float l, float m, float factor) { return __float_as_uint(factor) == 0x80000000u && m != -INFINITY ? NAN : l; }

// One thread's part of two query rows, g and g + 8 of a tile from row `r0` on (rows past the last repeat it).
struct AttnRows {
  int64_t at[2];
  int head[2], pos[2];
  float factor[2];       // scale * log2(e) and what undoes the rows' scaling; -0: not finite
  float start[2];        // -128 * 2^-24 * sum(q)
  float m[2], l[2];      // running maximum and sum
  S1C_DEV void setup(const AttnUnit& u, int r0) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = min(r0 + (int)(threadIdx.x % 32) / 4 + 8 * e, u.rows - 1);
      at[e] = u.first + r / u.G, head[e] = u.h * u.G + r % u.G, pos[e] = u.L - u.count + r / u.G;
      m[e] = -INFINITY, l[e] = 0.f;
    }
  }
  // The rows as f16 operands. The columns 2 cq, 2 cq + 1 (and those 8 on) of operand i are dimensions 16 i
  // + 4 cq .. + 3, the order of a lane's word of codes.
  template <typename T, int D>
  S1C_DEV void operands(const CacheAttnArgs& a, uint32_t (&qa)[D / 16][4]) {
    const int cq = threadIdx.x % 4;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const T* q = static_cast<const T*>(a.q) + at[e] * a.q_stride + head[e] * D;
      float f[D / 16][4], top = 0.f, sum = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint2 v = *reinterpret_cast<const uint2*>(q + i * 16 + cq * 4);
        f[i][0] = bits_f32<T>((uint16_t)v.x), f[i][1] = bits_f32<T>((uint16_t)(v.x >> 16));
        f[i][2] = bits_f32<T>((uint16_t)v.y), f[i][3] = bits_f32<T>((uint16_t)(v.y >> 16));
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max_nan(top, fabsf(f[i][j]));
      }
      for (int o = 1; o < 4; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float by = attn_up(top, a.scale_log2, factor[e]);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[i][j] = top < INFINITY ? f[i][j] * by : 0.f, sum += f[i][j];
        qa[i][e] = pack_f16x2(f[i][0], f[i][1]), qa[i][e + 2] = pack_f16x2(f[i][2], f[i][3]);
      }
      for (int o = 1; o < 4; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      start[e] = sum * -0x1p-17f;
    }
  }
  // Scores (in units of the key scale * factor) of a tile that begins at `key` to weights times 2^14; the
  // sums take them, and the outputs o are rescaled when the maximum has grown. kc0, kc1: where a lane's two
  // columns stand among eight keys.
  template <int N>
  S1C_DEV void weights(const CacheView& c, const AttnUnit& u, const float4* list, int key, int kc0, int kc1, float2* wide, float (&s)[4][4],
                       float (&o)[N][4]) {
    const bool open = key + CATT_TK - 1 <= pos[0] && key >= pos[1] - u.window && key + CATT_TK <= u.hi;
    float top[2] = {-INFINITY, -INFINITY}, inv[4];
    const int pg = (key >> u.shift) - (u.lo >> u.shift);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 p = list[pg + (((key & (c.page - 1)) + j * 8) >> u.shift)];
      inv[j] = p.z;
      const float f0 = factor[0] * p.x, f1 = factor[1] * p.x;
      s[j][0] = fmaf(s[j][0], f0, p.y), s[j][1] = fmaf(s[j][1], f0, p.y);
      s[j][2] = fmaf(s[j][2], f1, p.y), s[j][3] = fmaf(s[j][3], f1, p.y);
    }
    if (!__all_sync(0xffffffffu, open)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // key + 8 j + kc within [pos - window, min(pos, hi - 1)]
        const int last = min(pos[e], u.hi - 1) - key, from = pos[e] - u.window - key;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j * 8 + kc0 > last || j * 8 + kc0 < from) s[j][2 * e] = -INFINITY;
          if (j * 8 + kc1 > last || j * 8 + kc1 < from) s[j][2 * e + 1] = -INFINITY;
        }
      }
    }
    if (u.wide) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float r[8], big = -INFINITY;  // scores without t
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float t = list[pg + (((key & (c.page - 1)) + j / 2 * 8) >> u.shift)].y;
          r[j] = t == -INFINITY ? t : s[j / 2][2 * e + j % 2] - t;
          big = fmaxf(big, r[j]);
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        attn_wide_add(wide[e], big, r);
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
      grows |= top[e] > m[e] + 1.75f;
    }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // each row by its own scores alone, so that its bits do not depend on the rows beside it
        const float n = top[e] > m[e] + 1.75f ? top[e] : m[e], keep = m[e] == -INFINITY ? 0.f : exp2f(m[e] - n);
        m[e] = n, l[e] *= keep;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i][2 * e] *= keep, o[i][2 * e + 1] *= keep;
      }
    }
    const float off[2] = {m[0] == -INFINITY ? 0.f : 14.f - m[0], m[1] == -INFINITY ? 0.f : 14.f - m[1]};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = exp2_approx(s[j][e] + off[e / 2]);
        l[e / 2] = fmaf(s[j][e], inv[j], l[e / 2]);
      }
  }
  S1C_DEV void finish(const AttnUnit& u, float2* wide) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (u.wide) {
        wide[e].y += __shfl_xor_sync(0xffffffffu, wide[e].y, 1);
        wide[e].y += __shfl_xor_sync(0xffffffffu, wide[e].y, 2);
        wide[e].y = attn_sum(wide[e].y, m[e], factor[e]);
      }
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      l[e] = attn_sum(l[e], m[e], factor[e]);
    }
  }
};

// Weights are rounded to 11 bits for a bf16 result, whose own rounding to 8 bits is eight times as large. A result in
// f16 would be a quarter further from its exact value (2.6e-4 instead of 2.1e-4 for one row over 131072 keys), so
// there a second product takes what the rounding has left of each weight: 22 bits together. That costs 12 to 17 %
// (36 -> 40 us for that row; bf16 would take 191 instead of 170 us for 64 rows over 4096 to 8192 keys, 134
// instead of 115 us for 4 x 512 rows, for the same distance of 1.7e-3 from the exact values).
template <typename T>
constexpr bool ATTN_SPLIT = false;
template <>
constexpr bool ATTN_SPLIT<__half> = true;
// Two weights as f16, and what that leaves of them.
S1C_DEV uint32_t attn_split(float x, float y, uint32_t& rest) {
  const uint32_t v = pack_f16x2(x, y);
  const float2 f = unpack_f16x2(v);
  rest = pack_f16x2(x - f.x, y - f.y);
  return v;
}
// The weights of a tile as operands of two products over 16 keys each.
template <bool SPLIT>
S1C_DEV void attn_pack(const float (&s)[4][4], uint32_t (&pa)[2][4], uint32_t (&pr)[2][4]) {
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = s[2 * k + i / 2][i % 2 * 2], y = s[2 * k + i / 2][i % 2 * 2 + 1];
      pa[k][i] = SPLIT ? attn_split(x, y, pr[k][i]) : pack_f16x2(x, y);
    }
}

// N neighbouring dimensions, from d on, of one row's result: v * by, by = v_top / sum, with log2 of the sum,
// top - 14 + log2(sum), beside dimension 0. Without a key the sum is 0: outputs 0 and -inf.
S1C_DEV float attn_by(float v_top, float sum) { return sum == 0.f ? 0.f : v_top / sum; }
S1C_DEV float attn_log(float top, float sum) { return sum == 0.f ? -INFINITY : top - 14.f + log2f(sum); }
template <typename T, int D, int N>
S1C_DEV void attn_put(const CacheAttnArgs& a, const AttnUnit& u, int64_t row, int head, int d, const float (&v)[N], float by, float log_sum) {
  if (a.chunks > 1) {
    const int64_t at = ((u.seq * (int64_t)a.max_q + (row - u.first)) * a.heads + head) * a.chunks + u.chunk;
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(a.part + at * D + d + i) = make_float4(v[i] * by, v[i + 1] * by, v[i + 2] * by, v[i + 3] * by);
    if (d == 0) a.part_lse[at] = log_sum;
  } else {
    uint2* dst = reinterpret_cast<uint2*>(static_cast<T*>(a.out) + row * a.out_stride + head * D + d);
#pragma unroll
    for (int i = 0; i < N; i += 4) dst[i / 4] = make_uint2(pack2<T>(v[i] * by, v[i + 1] * by), pack2<T>(v[i + 2] * by, v[i + 3] * by));
    if (a.lse && d == 0) a.lse[row * a.heads + head] = log_sum * 0.69314718055994531f;
  }
}

// Few query rows.
constexpr int CATT_WARPS = 4, CATT_PAGES = 128;  // pages of a chunk at most

template <int D>
struct CacheAttnSmem {
  static constexpr int TILE = 2 * CATT_TK * D;  // keys and values of a tile
  static constexpr int STAGES = D == 128 ? 2 : 4;
  alignas(1024) uint8_t ring[CATT_WARPS][STAGES][TILE];
  uint4 q[D / 16][32];  // operands of the query rows
  uint64_t full[CATT_WARPS][STAGES];
  float4 page[CATT_PAGES + ATTN_BEYOND];
  float2 top[CATT_WARPS];
  float row_m[CATT_WARPS][16], row_l[CATT_WARPS][16];
  float2 wide[CATT_WARPS * 32][2], row_wide[CATT_WARPS][16];
};

template <typename T, int D>
__global__ void __launch_bounds__(CATT_WARPS * 32, 3)
cache_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const CacheView c,
                       const CacheAttnArgs a) {
  using S = CacheAttnSmem<D>;
  extern __shared__ uint8_t raw[];
  S& sm = *reinterpret_cast<S*>(raw + (1024 - smem_u32(raw) % 1024) % 1024);
  constexpr int QK = D / 16, SEG = D / 32;
  const int tid = threadIdx.x, w = tid / 32, lane = tid % 32, g = lane >> 2, cq = lane & 3;
  pdl_trigger();
  pdl_wait();
  AttnUnit u;
  if (!attn_unit<16, CATT_TK>(c, a, u)) return;
  float v_top = 0.f;
  if (u.tiles > 0) {
    if (tid < CATT_WARPS * S::STAGES) {
      mbar_init(&sm.full[0][tid], 1);
      fence_barrier_init();
    }
    v_top = attn_pages<CATT_WARPS>(c, a, u, sm.page, sm.top);
  }
  const auto issue = [&](int i) {
    const int slot = i / CATT_WARPS % S::STAGES;
    attn_issue<D, CATT_TK>(c, a, u, sm.page, k_map, v_map, i, sm.ring[w][slot], &sm.full[w][slot]);
  };
  for (int s = 0; s < S::STAGES; ++s)
    if (w + s * CATT_WARPS < u.tiles) issue(w + s * CATT_WARPS);

  AttnRows row;
  row.setup(u, u.row0);
  float2* wide = sm.wide[tid];
  if (u.wide) wide[0] = wide[1] = make_float2(-INFINITY, 0.f);
  {
    uint32_t qa[QK][4];
    row.operands<T, D>(a, qa);
    if (w == 0)
#pragma unroll
      for (int i = 0; i < QK; ++i) sm.q[i][lane] = make_uint4(qa[i][0], qa[i][1], qa[i][2], qa[i][3]);
    __syncthreads();
  }
  const uint32_t q_at = smem_u32(&sm.q[0][lane]);

  // shared offsets in a slot: the swizzle moves a row's 16-byte pieces by the row (128-byte rows) or by
  // half of it
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

  float o[SEG * 4][4];
#pragma unroll
  for (int i = 0; i < SEG * 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

  int turn = 0;  // tiles this ring has been through
  bool late = false;
  for (int i = w; i < u.tiles; i += CATT_WARPS, ++turn) {
    const int slot = turn % S::STAGES;
    if (!mbar_wait_warp(&sm.full[w][slot], turn / S::STAGES & 1, nullptr, 0, nullptr, a.wait_ns)) {
      late = true;
      // what is in flight lands before the block ends
      for (int j = 0; j < S::STAGES && i + j * CATT_WARPS < u.tiles; ++j)
        mbar_wait_warp(&sm.full[w][(turn + j) % S::STAGES], (turn + j) / S::STAGES & 1, nullptr, 0, nullptr, a.wait_ns);
      break;
    }
    const uint32_t base = smem_u32(sm.ring[w][slot]);

    float s[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j][0] = s[j][1] = row.start[0], s[j][2] = s[j][3] = row.start[1];
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
    row.weights(c, u, sm.page, u.lo + i * CATT_TK, kc0, kc1, wide, s, o);
    uint32_t pa[2][4], pr[2][4];
    attn_pack<ATTN_SPLIT<T>>(s, pa, pr);
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
        for (int d = 0; d < 4; ++d) {
          mma_f16(o[q * 4 + d], pa[k], b[d][0], b[d][1]);
          if (ATTN_SPLIT<T>) mma_f16(o[q * 4 + d], pr[k], b[d][0], b[d][1]);
        }
      });
    }
    __syncwarp();
    if (i + S::STAGES * CATT_WARPS < u.tiles) issue(i + S::STAGES * CATT_WARPS);
  }
  row.finish(u, wide);

  if (__syncthreads_or(late)) {  // also: the rings are free
    const float none[4] = {};
    for (int i = tid; i < 16 * D / 4 && u.row0 + i / (D / 4) < u.rows; i += CATT_WARPS * 32) {
      const int r = u.row0 + i / (D / 4);
      attn_put<T, D>(a, u, u.first + r / u.G, u.h * u.G + r % u.G, i % (D / 4) * 4, none, NAN, NAN);
    }
    return;
  }
  // join the four warps; a lane has eight neighbouring dimensions of each 32
  float* all = reinterpret_cast<float*>(sm.ring[0][0]);  // [warp][16][D]
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = g + 8 * e;
    if (cq == 0) sm.row_m[w][r] = row.m[e], sm.row_l[w][r] = row.l[e];
    if (cq == 0 && u.wide) sm.row_wide[w][r] = wide[e];
#pragma unroll
    for (int q = 0; q < SEG; ++q) {
      float4* at = reinterpret_cast<float4*>(all + (w * 16 + r) * D + q * 32 + cq * 8);
      at[0] = make_float4(o[q * 4][2 * e], o[q * 4 + 1][2 * e], o[q * 4 + 2][2 * e], o[q * 4 + 3][2 * e]);
      at[1] = make_float4(o[q * 4][2 * e + 1], o[q * 4 + 1][2 * e + 1], o[q * 4 + 2][2 * e + 1], o[q * 4 + 3][2 * e + 1]);
    }
  }
  __syncthreads();
  for (int i = tid; i < 16 * D / 4; i += CATT_WARPS * 32) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    if (u.row0 + r >= u.rows) break;
    float big = -INFINITY, sum = 0.f, v[4] = {};
#pragma unroll
    for (int x = 0; x < CATT_WARPS; ++x) big = fmaxf(big, sm.row_m[x][r]);
#pragma unroll
    for (int x = 0; x < CATT_WARPS; ++x) {
      const float by = sm.row_m[x][r] == -INFINITY ? 0.f : exp2f(sm.row_m[x][r] - big);
      const float4 p = *reinterpret_cast<const float4*>(all + (x * 16 + r) * D + d);
      sum += sm.row_l[x][r] * by;
      v[0] += p.x * by, v[1] += p.y * by, v[2] += p.z * by, v[3] += p.w * by;
    }
    float by = attn_by(v_top, sum), log_sum = attn_log(big, sum);
    if (u.wide) {
      float2 all2 = make_float2(-INFINITY, 0.f);
      for (int x = 0; x < CATT_WARPS; ++x) {
        const float2 p = sm.row_wide[x][r];
        const float none[1] = {-INFINITY};
        attn_wide_add(all2, p.x, none);
        if (p.x != -INFINITY) all2.y += p.y * exp2f(p.x - all2.x);
      }
      for (int x = 0; x < 4; ++x) v[x] = attn_wide_out(v[x], v_top, big, all2);
      by = 1.f, log_sum = attn_log(all2.x + 14.f, all2.y);
    }
    attn_put<T, D>(a, u, u.first + (u.row0 + r) / u.G, u.h * u.G + (u.row0 + r) % u.G, d, v, by, log_sum);
  }
}

// Many query rows: warps 0 to 3 softmax (thread = row = TMEM lane), 4 to 7 conversion, 8 products.
constexpr int CATP_ROWS = 128, CATP_WARPS = 9, CATP_PAGES = 256;
// TMEM columns: scores (then weights, f16 pairs, over the first 32 columns, and what is left of them, over the
// others) of even tiles [0, 64), of odd tiles [64, 128); outputs from 128 on
constexpr uint32_t CATP_TMEM = 256, CATP_TMEM_O = 128;

template <int D>
struct CachePromptSmem {
  // blocks of 64 dimensions, rows of 128 bytes, 16-byte pieces XORed with the row: the 128-byte swizzle of
  // the products' operands
  alignas(1024) uint8_t q[D / 64][CATP_ROWS * 128];
  alignas(1024) uint8_t k[D / 64][CATP_TK * 128];
  alignas(1024) uint8_t v[2][D / 64][CATP_TK * 128];
  alignas(1024) uint8_t codes[2 * CATP_TK * D];  // one tile's keys and values as they are in the cache
  float4 page[CATP_PAGES + ATTN_BEYOND];
  float2 top[CATP_WARPS];
  uint64_t raw_full, raw_free, q_full, k_full, k_free, v_full[2], s_full[2], p_full[2], pv_done[2], o_full, drain;
  uint32_t tmem;
  int abort;
  float2 wide[CATP_ROWS];
};

template <typename T, int D>
__global__ void __launch_bounds__(CATP_WARPS * 32, 2)
cache_prompt_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const CacheView c,
                    const CacheAttnArgs a) {
  using S = CachePromptSmem<D>;
  extern __shared__ uint8_t raw[];
  S& sm = *reinterpret_cast<S*>(raw + (1024 - smem_u32(raw) % 1024) % 1024);
  const int tid = threadIdx.x, w = tid / 32, lane = tid % 32;
  pdl_wait();
  AttnUnit u;
  if (!attn_unit<CATP_ROWS, CATP_TK>(c, a, u)) return;
  // the softmax threads' rows; those past the last repeat it
  const int r = min(u.row0 + tid % CATP_ROWS, u.rows - 1);
  const int64_t at_row = u.first + r / u.G;
  const int head = u.h * u.G + r % u.G, pos = u.L - u.count + r / u.G;
  const bool real = w < 4 && u.row0 + tid < u.rows;
  if (u.tiles == 0) {
    const float zero[8] = {};
    if (real)
      for (int d = 0; d < D; d += 8) attn_put<T, D>(a, u, at_row, head, d, zero, 0.f, -INFINITY);
    return;
  }
  if (tid == 0) {
    mbar_init(&sm.raw_full, 1), mbar_init(&sm.raw_free, 4), mbar_init(&sm.q_full, 4), mbar_init(&sm.k_full, 4), mbar_init(&sm.k_free, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&sm.v_full[i], 4), mbar_init(&sm.s_full[i], 1), mbar_init(&sm.p_full[i], 4), mbar_init(&sm.pv_done[i], 1);
    mbar_init(&sm.o_full, 1), mbar_init(&sm.drain, 1);
    sm.abort = 0;
    fence_barrier_init();
  }
  if (w == 8) {
    tmem_alloc(&sm.tmem, CATP_TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  const float v_top = attn_pages<CATP_WARPS>(c, a, u, sm.page, sm.top);  // with barriers of the block
  // Only now: a kernel that is scheduled early may hold TMEM while it waits for this one, so each block has
  // its own first.
  pdl_trigger();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  volatile int* abort = &sm.abort;

  if (w == 8) {
    if (lane == 0) {
      constexpr uint32_t idS = idesc_f16_f32(CATP_ROWS, CATP_TK, false), idO = idesc_f16_f32(CATP_ROWS, 64, true);
      const auto scores = [&](int i) {
        if (!mbar_wait(&sm.k_full, i & 1, nullptr, 0, abort, a.wait_ns)) return false;
        tc_fence_after();
#pragma unroll
        for (int b = 0; b < D / 64; ++b)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16(tmem + 64 * (i & 1), sdesc_kmajor_sw128(smem_u32(sm.q[b]) + k * 32), sdesc_kmajor_sw128(smem_u32(sm.k[b]) + k * 32), idS,
                      (b | k) ? 1u : 0u);
        umma_commit(&sm.s_full[i & 1]);
        umma_commit(&sm.k_free);
        return true;
      };
      bool ok = mbar_wait(&sm.q_full, 0, nullptr, 0, abort, a.wait_ns) && scores(0) && (u.tiles < 2 || scores(1));
      for (int i = 0; ok && i < u.tiles; ++i) {
        const int b = i & 1;
        ok = mbar_wait(&sm.p_full[b], i >> 1 & 1, nullptr, 0, abort, a.wait_ns) && mbar_wait(&sm.v_full[b], i >> 1 & 1, nullptr, 0, abort, a.wait_ns);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int n = 0; n < D / 64; ++n)
#pragma unroll
          for (int k = 0; k < CATP_TK / (ATTN_SPLIT<T> ? 8 : 16); ++k)  // the weights, then what is left of them
            umma_bf16_ts(tmem + CATP_TMEM_O + 64 * n, tmem + 64 * b + 8 * k, sdesc_mnmajor_sw128(smem_u32(sm.v[b][n]) + k % 4 * 2048), idO,
                         (i | k) ? 1u : 0u);
        umma_commit(&sm.pv_done[b]);
        if (i == u.tiles - 1) umma_commit(&sm.o_full);
        // scores two tiles on, over the weights that this product, issued before them, reads
        if (i + 2 < u.tiles) ok = scores(i + 2);
      }
      umma_commit(&sm.drain);
      mbar_wait(&sm.drain, 0, nullptr, 0, nullptr, a.wait_ns);
    }
  } else if (w >= 4) {
    // 16 codes at a time: 64 x D / 16 pieces of keys and as many of values over 128 threads
    constexpr int ITEMS = CATP_TK * (D / 16) / 128;
    const int t = tid - 128;
    int i = 0, issued = 1;  // tiles taken, tiles asked for
    if (w == 4) attn_issue<D, CATP_TK>(c, a, u, sm.page, k_map, v_map, 0, sm.codes, &sm.raw_full);
    for (; i < u.tiles; ++i) {
      if (!mbar_wait_warp(&sm.raw_full, i & 1, nullptr, 0, abort, a.wait_ns)) break;
      uint4 codes[2][ITEMS];
#pragma unroll
      for (int x = 0; x < 2 * ITEMS; ++x) {
        const int j = t + x % ITEMS * 128, row = j / (D / 16), piece = j % (D / 16);
        codes[x / ITEMS][x % ITEMS] =
            *reinterpret_cast<const uint4*>(sm.codes + (x / ITEMS * CATP_TK + row) * D + ((piece ^ (D == 128 ? row & 7 : row >> 1 & 3)) << 4));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.raw_free);
      if (w == 4 && i + 1 < u.tiles) {  // the next tile may come when all codes are in registers
        if (!mbar_wait_warp(&sm.raw_free, i & 1, nullptr, 0, abort, a.wait_ns)) break;
        attn_issue<D, CATP_TK>(c, a, u, sm.page, k_map, v_map, i + 1, sm.codes, &sm.raw_full);
        ++issued;
      }
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        // the product that read this buffer last
        if (which == 0 && i > 0 && !mbar_wait_warp(&sm.k_free, (i - 1) & 1, nullptr, 0, abort, a.wait_ns)) goto done;
        if (which == 1 && i > 1 && !mbar_wait_warp(&sm.pv_done[i & 1], ((i >> 1) - 1) & 1, nullptr, 0, abort, a.wait_ns)) goto done;
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
          const int j = t + x * 128, row = j / (D / 16), piece = j % (D / 16);
          const uint4 in4 = codes[which][x];
          const uint32_t in[4] = {in4.x, in4.y, in4.z, in4.w};
          uint32_t out[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t v = in[e] ^ 0x80808080u;
            out[2 * e] = code_pair(__byte_perm(v, 0x64646464u, 0x4140)), out[2 * e + 1] = code_pair(__byte_perm(v, 0x64646464u, 0x4342));
          }
          uint8_t* dst = (which ? sm.v[i & 1][piece / 4] : sm.k[piece / 4]) + row * 128;
          const int p0 = piece % 4 * 2;
          *reinterpret_cast<uint4*>(dst + ((p0 ^ (row & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
          *reinterpret_cast<uint4*>(dst + (((p0 + 1) ^ (row & 7)) << 4)) = make_uint4(out[4], out[5], out[6], out[7]);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(which ? &sm.v_full[i & 1] : &sm.k_full);
      }
    }
  done:
    // what is in flight lands before the block ends
    if (w == 4 && i < u.tiles) mbar_wait_warp(&sm.raw_full, (issued - 1) & 1, nullptr, 0, nullptr, a.wait_ns);
  } else {
    // the row as f16, in the order of the products' operand
    float factor;
    {
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + at_row * a.q_stride + head * D);
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        float x[8];
        unpack8<T>(q[i], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(x[j]));
      }
      const float by = attn_up(top, a.scale_log2 * 0x1p-24f, factor);  // the list's key scales have 2^24
#pragma unroll 4
      for (int i = 0; i < D / 8; ++i) {
        float x[8];
        unpack8<T>(top < INFINITY ? q[i] : make_uint4(0, 0, 0, 0), x);
        *reinterpret_cast<uint4*>(sm.q[i / 8] + tid * 128 + ((i % 8 ^ (tid & 7)) << 4)) =
            make_uint4(pack_f16x2(x[0] * by, x[1] * by), pack_f16x2(x[2] * by, x[3] * by), pack_f16x2(x[4] * by, x[5] * by),
                       pack_f16x2(x[6] * by, x[7] * by));
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full);
    }
    const uint32_t lanes = (uint32_t)(w * 32) << 16;
    float m = -INFINITY, l = 0.f;
    if (u.wide) sm.wide[tid] = make_float2(-INFINITY, 0.f);
    bool ok = true;
    for (int i = 0; i < u.tiles; ++i) {
      const int b = i & 1, key = u.lo + i * CATP_TK, pg = (key >> u.shift) - (u.lo >> u.shift), in = key & (c.page - 1);
      // columns that this row sees: [from, upto)
      const int upto = min(pos + 1, u.hi) - key, from = pos - u.window - key;
      if (!mbar_wait_warp(&sm.s_full[b], i >> 1 & 1, nullptr, 0, abort, a.wait_ns)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (u.wide) {  // a first look at the scores
        float2 all = sm.wide[tid];
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          const float4 p = sm.page[pg + ((in + 16 * j) >> u.shift)];
          float r[16], big = -INFINITY;
          tmem_ld16(tmem + lanes + 64 * b + 16 * j, r);
          if (p.y == -INFINITY) continue;
#pragma unroll
          for (int x = 0; x < 16; ++x) r[x] = 16 * j + x >= from && 16 * j + x < upto ? r[x] * (factor * p.x) : -INFINITY, big = fmaxf(big, r[x]);
          attn_wide_add(all, big, r);
        }
        sm.wide[tid] = all;
      }
      float s[64];
      tmem_ld32x2(tmem + lanes + 64 * b, true, true, s);
      const bool open = __all_sync(0xffffffffu, from <= 0 && upto >= CATP_TK);
      float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, inv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 p = sm.page[pg + ((in + 16 * j) >> u.shift)];
        const float f = factor * p.x;
        inv[j] = p.z;
#pragma unroll
        for (int x = 16 * j; x < 16 * j + 16; ++x) s[x] = fmaf(s[x], f, p.y);
      }
      if (!open) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int x0 = min(max(from - 32 * half, 0), 32), x1 = min(max(upto - 32 * half, 0), 32);
          const uint32_t see = (x1 >= 32 ? 0xffffffffu : (1u << x1) - 1u) & ~(x0 >= 32 ? 0xffffffffu : (1u << x0) - 1u);
#pragma unroll
          for (int x = 0; x < 32; ++x) s[32 * half + x] = (see & (1u << x)) ? s[32 * half + x] : -INFINITY;
        }
      }
#pragma unroll
      for (int x = 0; x < 64; ++x) part[x & 3] = fmaxf(part[x & 3], s[x]);
      const float top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
      float keep = 1.f;
      if (top > m + 1.75f) {
        keep = m == -INFINITY ? 0.f : exp2f(m - top);
        l *= keep;
        m = top;
      }
      if (i > 0 && __any_sync(0xffffffffu, keep != 1.f)) {
        // the outputs so far, when the product before has completed
        if (!mbar_wait_warp(&sm.pv_done[b ^ 1], (i - 1) >> 1 & 1, nullptr, 0, abort, a.wait_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int x = 0; x < D; x += 16) {
          float t[16];
          tmem_ld16(tmem + lanes + CATP_TMEM_O + x, t);
#pragma unroll
          for (int y = 0; y < 16; ++y) t[y] *= keep;
          tmem_st16(tmem + lanes + CATP_TMEM_O + x, t);
        }
      }
      const float off = m == -INFINITY ? 0.f : 14.f - m;
      float pk[32], pr[ATTN_SPLIT<T> ? 32 : 1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float sum = 0.f;
#pragma unroll
        for (int x = 8 * j; x < 8 * j + 8; ++x) {
          const float p0 = exp2_approx(s[2 * x] + off), p1 = exp2_approx(s[2 * x + 1] + off);
          sum += p0 + p1;
          if constexpr (ATTN_SPLIT<T>) {
            uint32_t rest;
            pk[x] = __uint_as_float(attn_split(p0, p1, rest));
            pr[x] = __uint_as_float(rest);
          } else {
            pk[x] = __uint_as_float(pack_f16x2(p0, p1));
          }
        }
        l = fmaf(sum, inv[j], l);
      }
      tmem_st32(tmem + lanes + 64 * b, pk);
      if constexpr (ATTN_SPLIT<T>) tmem_st32(tmem + lanes + 64 * b + 32, pr);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[b]);
    }
    if (ok && mbar_wait_warp(&sm.o_full, 0, nullptr, 0, abort, a.wait_ns)) {
      tc_fence_after();
#pragma unroll 1
      for (int d = 0; d < D; d += 32) {
        float t[32];
        tmem_ld32(tmem + lanes + CATP_TMEM_O + d, t);
        const float sum = attn_sum(l, m, factor);
        float by = attn_by(v_top, sum), log_sum = attn_log(m, sum);
        if (u.wide) {
          const float2 all = make_float2(sm.wide[tid].x, attn_sum(sm.wide[tid].y, m, factor));
#pragma unroll
          for (int x = 0; x < 32; ++x) t[x] = attn_wide_out(t[x], v_top, m, all);
          by = 1.f, log_sum = attn_log(all.x + 14.f, all.y);
        }
        if (real) attn_put<T, D>(a, u, at_row, head, d, t, by, log_sum);
      }
    } else if (real) {  // a wait has run out
      const float none[8] = {};
#pragma unroll 1
      for (int d = 0; d < D; d += 8) attn_put<T, D>(a, u, at_row, head, d, none, NAN, NAN);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (w == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, CATP_TMEM);
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
  pdl_trigger();
  const int head = (int)(item % a.heads), i = (int)(item / a.heads % a.max_q);
  const int64_t seq = item / a.heads / a.max_q;
  pdl_wait();
  const int first = a.cu[seq];
  if (i >= a.cu[seq + 1] - first) return;
  const float* lse = a.part_lse + item * a.chunks;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < a.chunks; s += WARPS * 32) top = max_nan(top, lse[s]);  // NaN: so is the row
  for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[w] = top;
  __syncthreads();
  for (int j = 0; j < WARPS; ++j) top = max_nan(top, tops[j]);
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
      for (int e = 0; e < E; ++e) o[e] += by == 0.f ? 0.f : by * v[e];  // 0 also times an output past fp32
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
