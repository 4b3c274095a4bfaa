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
// of loads, so nothing waits inside the loop; the four warps' results are joined at the end. Long caches are split
// over blocks, whose results a second kernel joins. Many rows (bound by the tensor cores and the conversion of the
// codes): each warp has its own 16 rows, and a block converts a tile of keys once for all of them, to f16 in
// shared memory, while it works on the tile before.
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

constexpr int CATT_TK = 32;  // keys of a tile

// What a block works on: `rows` rows from row0 on of one sequence and key head, keys [lo, hi) in `tiles` tiles.
struct AttnUnit {
  int h, seq, first, count, L, rows, row0, chunk, lo, hi, tiles, window, shift, G;
};
template <int ROWS>
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
  u.lo = max(max(0, pos0 - u.window) / CATT_TK * CATT_TK, u.chunk * a.chunk);
  u.hi = (int)min((int64_t)min(pos1 + 1, reach), ((int64_t)u.chunk + 1) * a.chunk);
  u.tiles = u.hi > u.lo ? (u.hi - u.lo + CATT_TK - 1) / CATT_TK : 0;
  return true;
}

// The chunk's pages: (key scale * 2^24, t, 2^-t, page), two more than there are, without a page (-1) 0, -inf, 0. Returns the
// largest value scale, which the outputs are multiplied by. All threads call.
template <int WARPS>
S1C_DEV float attn_pages(const CacheView& c, const CacheAttnArgs& a, const AttnUnit& u, float4* list, float* tops) {
  const int tid = threadIdx.x, p0 = u.lo >> u.shift, pages = ((u.hi - 1) >> u.shift) - p0 + 1;
  float top = 0.f;
  for (int i = tid; i < pages + 2; i += WARPS * 32) {
    const int page = i < pages ? cache_page(a.table, a.max_pages, u.seq, p0 + i, c.num_pages) : -1;
    float ks = 0.f, vs = 0.f;
    if (page >= 0) {
      const int64_t slot = (int64_t)page * c.heads + u.h;
      ks = c.scales[0][slot], vs = c.scales[1][slot];
    }
    list[i] = make_float4(ks * 0x1p24f, vs, 0.f, __int_as_float(page));
    top = fmaxf(top, vs);
  }
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (tid % 32 == 0) tops[tid / 32] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WARPS; ++i) top = fmaxf(top, tops[i]);
  for (int i = tid; i < pages + 2; i += WARPS * 32) {
    float4 e = list[i];
    // scales below 2^-60 of the largest (and zero ones, whose codes are zero) count as that
    const float l2 = top > 0.f ? fmaxf(log2f(e.y / top), -60.f) : 0.f;
    const bool in = __float_as_int(e.w) >= 0;
    e.y = in ? l2 : -INFINITY, e.z = in ? exp2f(-l2) : 0.f;
    list[i] = e;
  }
  __syncthreads();
  return top;
}

// TMA of one tile's keys and values to `dst`, by a whole warp: a lane for each page (one, or two of 16 rows). Pages outside
// the cache are not read.
template <int D>
S1C_DEV void attn_issue(const CacheView& c, const AttnUnit& u, const float4* list, const CUtensorMap& k_map, const CUtensorMap& v_map, int i,
                        uint8_t* dst, uint64_t* bar) {
  const int lane = threadIdx.x % 32, per = min(c.page, CATT_TK), boxes = CATT_TK / per;
  const int at = u.lo + i * CATT_TK + lane * per;
  const int page = lane < boxes && at < u.hi ? __float_as_int(list[(at >> u.shift) - (u.lo >> u.shift)].w) : -1;
  const int count = __popc(__ballot_sync(0xffffffffu, page >= 0));
  if (lane == 0) mbar_arrive_expect_tx(bar, count * 2 * per * D);
  __syncwarp();
  if (page >= 0) {
    const int y = (page * c.heads + u.h) * c.page + (at & (c.page - 1));
    tma_load_2d(dst + lane * per * D, &k_map, bar, 0, y);
    tma_load_2d(dst + CATT_TK * D + lane * per * D, &v_map, bar, 0, y);
  }
  __syncwarp();
}

// One thread's part of two query rows, g and g + 8 of a tile from row `r0` on (rows past the last repeat it).
struct AttnRows {
  int64_t at[2];
  int head[2], pos[2];
  float factor[2];       // scale * log2(e) and what undoes the rows' scaling
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
  // The rows as f16 operands. The columns 2 cq, 2 cq + 1 (and those 8 on) of operand i are dimensions 16 i + 4 cq .. + 3 (QUADS, the order
  // of a lane's word of codes), or 16 i + 2 cq, + 1 (and 8 on).
  template <typename T, int D, bool QUADS>
  S1C_DEV void operands(const CacheAttnArgs& a, uint32_t (&qa)[D / 16][4]) {
    const int cq = threadIdx.x % 4;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const T* q = static_cast<const T*>(a.q) + at[e] * a.q_stride + head[e] * D;
      float f[D / 16][4], top = 0.f, sum = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        uint32_t lo, hi;
        if (QUADS) {
          const uint2 v = *reinterpret_cast<const uint2*>(q + i * 16 + cq * 4);
          lo = v.x, hi = v.y;
        } else {
          lo = *reinterpret_cast<const uint32_t*>(q + i * 16 + cq * 2), hi = *reinterpret_cast<const uint32_t*>(q + i * 16 + 8 + cq * 2);
        }
        f[i][0] = bits_f32<T>((uint16_t)lo), f[i][1] = bits_f32<T>((uint16_t)(lo >> 16));
        f[i][2] = bits_f32<T>((uint16_t)hi), f[i][3] = bits_f32<T>((uint16_t)(hi >> 16));
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max_nan(top, fabsf(f[i][j]));
      }
      for (int o = 1; o < 4; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      // 2^up brings the largest value to [2^14, 2^15); rows with an infinity or NaN keep theirs
      const int ex = (int)(__float_as_uint(top) >> 23) - 127, up = ex == 128 ? 0 : min(14 - ex, 100);
      const float by = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[i][j] *= by, sum += f[i][j];
        qa[i][e] = pack_f16x2(f[i][0], f[i][1]), qa[i][e + 2] = pack_f16x2(f[i][2], f[i][3]);
      }
      for (int o = 1; o < 4; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      factor[e] = a.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
      start[e] = sum * -0x1p-17f;
    }
  }
  // Scores (in units of the key scale * factor) of a tile that begins at `key` to weights times 2^14.5; the sums take them, and the
  // outputs o are rescaled when the maximum has grown. kc0, kc1: where a lane's two columns stand among eight keys.
  template <int N>
  S1C_DEV void weights(const CacheView& c, const AttnUnit& u, const float4* list, int key, int kc0, int kc1, float (&s)[4][4], float (&o)[N][4]) {
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
        for (int i = 0; i < N; ++i) o[i][2 * e] *= keep, o[i][2 * e + 1] *= keep;
      }
    }
    const float off[2] = {m[0] == -INFINITY ? 0.f : 14.5f - m[0], m[1] == -INFINITY ? 0.f : 14.5f - m[1]};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = exp2_approx(s[j][e] + off[e / 2]);
        l[e / 2] = fmaf(s[j][e], inv[j], l[e / 2]);
      }
  }
  S1C_DEV void finish() {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
  }
};

// The weights of a tile as operands of two products over 16 keys each.
S1C_DEV void attn_pack(const float (&s)[4][4], uint32_t (&pa)[2][4]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    pa[k][0] = pack_f16x2(s[2 * k][0], s[2 * k][1]), pa[k][1] = pack_f16x2(s[2 * k][2], s[2 * k][3]);
    pa[k][2] = pack_f16x2(s[2 * k + 1][0], s[2 * k + 1][1]), pa[k][3] = pack_f16x2(s[2 * k + 1][2], s[2 * k + 1][3]);
  }
}

// N neighbouring dimensions, from d on, of one row's result: v * v_top / sum, with log2 of the sum beside dimension 0. Without a
// key the sum is 0: outputs 0 and -inf.
template <typename T, int D, int N>
S1C_DEV void attn_put(const CacheAttnArgs& a, const AttnUnit& u, int64_t row, int head, int d, const float (&v)[N], float v_top, float sum, float top) {
  const float by = sum == 0.f ? 0.f : v_top / sum, log_sum = sum == 0.f ? -INFINITY : top - 14.5f + log2f(sum);
  if (a.chunks > 1) {
    const int64_t at = ((u.seq * (int64_t)a.max_q + (row - u.first)) * a.heads + head) * a.chunks + u.chunk;
#pragma unroll
    for (int i = 0; i < N; i += 2) *reinterpret_cast<float2*>(a.part + at * D + d + i) = make_float2(v[i] * by, v[i + 1] * by);
    if (d == 0) a.part_lse[at] = log_sum;
  } else {
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + row * a.out_stride + head * D + d);
#pragma unroll
    for (int i = 0; i < N; i += 2) dst[i / 2] = pack2<T>(v[i] * by, v[i + 1] * by);
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
  float4 page[CATT_PAGES + 2];
  float top[CATT_WARPS];
  float row_m[CATT_WARPS][16], row_l[CATT_WARPS][16];
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
  AttnUnit u;
  if (!attn_unit<16>(c, a, u)) return;
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
    attn_issue<D>(c, u, sm.page, k_map, v_map, i, sm.ring[w][slot], &sm.full[w][slot]);
  };
  for (int s = 0; s < S::STAGES; ++s)
    if (w + s * CATT_WARPS < u.tiles) issue(w + s * CATT_WARPS);

  AttnRows row;
  row.setup(u, u.row0);
  {
    uint32_t qa[QK][4];
    row.operands<T, D, true>(a, qa);
    if (w == 0)
#pragma unroll
      for (int i = 0; i < QK; ++i) sm.q[i][lane] = make_uint4(qa[i][0], qa[i][1], qa[i][2], qa[i][3]);
    __syncthreads();
  }
  const uint32_t q_at = smem_u32(&sm.q[0][lane]);

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

  float o[SEG * 4][4];
#pragma unroll
  for (int i = 0; i < SEG * 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

  int turn = 0;  // tiles this ring has been through
  for (int i = w; i < u.tiles; i += CATT_WARPS, ++turn) {
    const int slot = turn % S::STAGES;
    if (!mbar_wait_warp(&sm.full[w][slot], turn / S::STAGES & 1, nullptr, 0, nullptr)) break;
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
    row.weights(c, u, sm.page, u.lo + i * CATT_TK, kc0, kc1, s, o);
    uint32_t pa[2][4];
    attn_pack(s, pa);
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
    __syncwarp();
    if (i + S::STAGES * CATT_WARPS < u.tiles) issue(i + S::STAGES * CATT_WARPS);
  }
  row.finish();

  // join the four warps; a lane has eight neighbouring dimensions of each 32
  __syncthreads();  // the rings are free
  float* all = reinterpret_cast<float*>(sm.ring[0][0]);  // [warp][16][D]
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = g + 8 * e;
    if (cq == 0) sm.row_m[w][r] = row.m[e], sm.row_l[w][r] = row.l[e];
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
    attn_put<T, D>(a, u, u.first + (u.row0 + r) / u.G, u.h * u.G + (u.row0 + r) % u.G, d, v, v_top, sum, big);
  }
}

// Many query rows.
constexpr int CATP_WARPS = 8, CATP_STAGES = 2, CATP_PAGES = 256;

template <int D>
struct CachePromptSmem {
  alignas(1024) uint8_t ring[CATP_STAGES][2 * CATT_TK * D];  // codes of keys and values
  // two tiles as f16, keys (codes + 128) * 2^-24, values as codes; 16-byte pieces of a row XORed with the row
  alignas(1024) uint8_t half[2][2][CATT_TK * D * 2];
  uint4 q[CATP_WARPS][D / 16][32];
  uint64_t full[CATP_STAGES];
  float4 page[CATP_PAGES + 2];
  float top[CATP_WARPS];
};

template <typename T, int D>
__global__ void __launch_bounds__(CATP_WARPS * 32, 2)
cache_prompt_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const CacheView c,
                    const CacheAttnArgs a) {
  using S = CachePromptSmem<D>;
  extern __shared__ uint8_t raw[];
  S& sm = *reinterpret_cast<S*>(raw + (1024 - smem_u32(raw) % 1024) % 1024);
  constexpr int QK = D / 16, ROWS = 16 * CATP_WARPS;
  const int tid = threadIdx.x, w = tid / 32, lane = tid % 32, g = lane >> 2, cq = lane & 3;
  pdl_trigger();
  AttnUnit u;
  if (!attn_unit<ROWS>(c, a, u)) return;
  float v_top = 0.f;
  if (u.tiles > 0) {
    if (tid < CATP_STAGES) {
      mbar_init(&sm.full[tid], 1);
      fence_barrier_init();
    }
    v_top = attn_pages<CATP_WARPS>(c, a, u, sm.page, sm.top);
  }
  const auto issue = [&](int i) {
    attn_issue<D>(c, u, sm.page, k_map, v_map, i, sm.ring[i % CATP_STAGES], &sm.full[i % CATP_STAGES]);
  };
  if (w == 0)
    for (int s = 0; s < CATP_STAGES; ++s)
      if (s < u.tiles) issue(s);

  AttnRows row;
  row.setup(u, u.row0 + w * 16);
  {
    uint32_t qa[QK][4];
    row.operands<T, D, false>(a, qa);
#pragma unroll
    for (int i = 0; i < QK; ++i) sm.q[w][i][lane] = make_uint4(qa[i][0], qa[i][1], qa[i][2], qa[i][3]);
    __syncwarp();
  }
  const uint32_t q_at = smem_u32(&sm.q[w][0][lane]);

  // conversion: 16 codes of a row at a time
  constexpr int ITEMS = 2 * CATT_TK * (D / 16) / (CATP_WARPS * 32);
  static_assert(ITEMS >= 1, "a thread converts at least 16 codes");
  const auto item = [&](int x, int& which, int& r, int& piece) {
    const int i = tid + x * CATP_WARPS * 32;
    which = i / (CATT_TK * (D / 16)), r = i / (D / 16) % CATT_TK, piece = i % (D / 16);
  };
  uint4 codes[ITEMS];
  const auto fetch = [&](int slot) {
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
      int which, r, piece;
      item(x, which, r, piece);
      codes[x] = *reinterpret_cast<const uint4*>(sm.ring[slot] + (which * CATT_TK + r) * D + ((piece ^ (D == 128 ? r & 7 : r >> 1 & 3)) << 4));
    }
  };
  const auto convert = [&](int buffer) {
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
      int which, r, piece;
      item(x, which, r, piece);
      const uint32_t in[4] = {codes[x].x, codes[x].y, codes[x].z, codes[x].w};
      uint32_t out[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t v = in[j] ^ 0x80808080u;
        if (which) {
          out[2 * j] = code_pair(__byte_perm(v, 0x64646464u, 0x4140)), out[2 * j + 1] = code_pair(__byte_perm(v, 0x64646464u, 0x4342));
        } else {
          out[2 * j] = __byte_perm(v, 0, 0x4140), out[2 * j + 1] = __byte_perm(v, 0, 0x4342);
        }
      }
      uint8_t* dst = sm.half[buffer][which] + r * D * 2;
      *reinterpret_cast<uint4*>(dst + (((2 * piece) ^ (r & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
      *reinterpret_cast<uint4*>(dst + (((2 * piece + 1) ^ (r & 7)) << 4)) = make_uint4(out[4], out[5], out[6], out[7]);
    }
  };
  bool broken = false;
  const auto arrived = [&](int i) {
    if (!broken && !mbar_wait_warp(&sm.full[i % CATP_STAGES], i / CATP_STAGES & 1, nullptr, 0, nullptr)) broken = true;
  };

  // addresses for ldmatrix: matrices (keys 0-7, 8 columns), (keys 0-7, next 8), (keys 8-15, ..), (keys 8-15, ..) of the keys, and
  // of the values (keys 0-7, dims), (keys 8-15, dims), and the next dims
  const int mr = lane & 7, mi = lane >> 3;
  const uint32_t k_at = smem_u32(sm.half[0][0]) + ((mi >> 1) * 8 + mr) * D * 2 + (((mi & 1) ^ mr) << 4);
  const uint32_t v_at = smem_u32(sm.half[0][1]) + ((mi & 1) * 8 + mr) * D * 2 + (((mi >> 1) ^ mr) << 4);
  constexpr int BUFFER = 2 * CATT_TK * D * 2;

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  const int last = __reduce_max_sync(0xffffffffu, row.pos[1]), from = __reduce_min_sync(0xffffffffu, row.pos[0]) - u.window;

  if (u.tiles > 0) {
    arrived(0);
    fetch(0);
    convert(0);
    __syncthreads();
  }
  for (int i = 0; i < u.tiles; ++i) {
    const int key = u.lo + i * CATT_TK, b = i & 1;
    // the codes of tile i have been converted: their slot is free
    if (w == 0 && i + CATP_STAGES < u.tiles) issue(i + CATP_STAGES);
    const bool more = i + 1 < u.tiles;
    if (more) {
      arrived(i + 1);
      fetch((i + 1) % CATP_STAGES);
    }
    const bool mine = !broken && key <= last && key + CATT_TK > from;  // some row of this warp sees a key
    float s[4][4];
    if (mine) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j][0] = s[j][1] = row.start[0], s[j][2] = s[j][3] = row.start[1];
      static_for<QK>([&](auto DD) {
        constexpr int d = decltype(DD)::value;
        const uint4 qv = lds_v4<d * 512>(q_at);
        const uint32_t qa[4] = {qv.x, qv.y, qv.z, qv.w};
        const uint32_t at = (k_at ^ (d << 5)) + b * BUFFER;
        uint32_t k0[4], k1[4];
        ldmatrix<0>(at, k0);
        ldmatrix<16 * D * 2>(at, k1);
        mma_f16(s[0], qa, k0[0], k0[1]);
        mma_f16(s[1], qa, k0[2], k0[3]);
        mma_f16(s[2], qa, k1[0], k1[1]);
        mma_f16(s[3], qa, k1[2], k1[3]);
      });
    }
    if (more) convert(b ^ 1);
    if (mine) {
      row.weights(c, u, sm.page, key, 2 * cq, 2 * cq + 1, s, o);
      uint32_t pa[2][4];
      attn_pack(s, pa);
      static_for<D / 16>([&](auto DD) {
        constexpr int d = decltype(DD)::value;
        const uint32_t at = (v_at ^ (d << 5)) + b * BUFFER;
        uint32_t v0[4], v1[4];
        ldmatrix_t<0>(at, v0);
        ldmatrix_t<16 * D * 2>(at, v1);
        mma_f16(o[2 * d], pa[0], v0[0], v0[1]);
        mma_f16(o[2 * d + 1], pa[0], v0[2], v0[3]);
        mma_f16(o[2 * d], pa[1], v1[0], v1[1]);
        mma_f16(o[2 * d + 1], pa[1], v1[2], v1[3]);
      });
    }
    __syncthreads();
  }
  row.finish();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (u.row0 + w * 16 + g + 8 * e >= u.rows) continue;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const float v[2] = {o[i][2 * e], o[i][2 * e + 1]};
      attn_put<T, D>(a, u, row.at[e], row.head[e], i * 8 + cq * 2, v, v_top, row.l[e], row.m[e]);
    }
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
