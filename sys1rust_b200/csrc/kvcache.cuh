// A paged cache of keys and values held in 8 bits: pages [num_pages, kv_heads, page, head_dim] of
// int8 codes and one fp32 scale for each page and head, a value being code * scale.
//
// Writing. A sequence's rows stand at consecutive positions; position p lies in row p % page of the
// page its table names at p / page. For a page and head that new rows fall into
//   s = max(s_old, fl32(max |new| / 127)), s_old = the page's scale if earlier rows of the sequence
// stand in it, else 0; a new value becomes round-half-even(x / s), and where s grew the earlier codes
// become round-half-even(code * s_old / s), both of the exact quotient.
//
// Measured on eight ragged prompts of up to 8192 rows (8 heads of 128, pages of 64): write 70 us and read
// 74 us for 300 MB each, 4.1 TB/s. Issue slots are two thirds (write) and half (read) used; beside its rows each kernel
// stores 250 MB of its own arguments to local memory, which every thread copies because it indexes their arrays by
// blockIdx.z. A quotient costs one product, with an exact second look only near a half
// (an IEEE division for each value took 224 us, the second look inside the unrolled code 144 us, of
// instruction fetches).
#pragma once
#include "mma.cuh"

namespace s1c {

struct CacheView {
  int8_t* codes[2];  // keys, values
  float* scales[2];
  int num_pages, page, heads, dim;
};

struct CacheRows {
  void* rows[2];  // [rows, heads, dim] of the keys and of the values, row strides in elements
  int64_t stride[2];
  const int* cu;     // [n + 1]
  const int* start;  // [n] position of a sequence's first row
  const int* table;  // [n, max_pages]
  int max_pages, units;  // write: pages a sequence can touch; read: blocks for a sequence
  int most;              // rows a sequence has at most
};

// The page of position `pos`, or -1 where the table has none or names one outside the cache.
S1C_DEV int cache_page(const int* table, int64_t max_pages, int seq, int64_t at, int num_pages) {
  if (at < 0 || at >= max_pages) return -1;
  const int p = table[seq * max_pages + at];
  return p >= 0 && p < num_pages ? p : -1;
}

// round-half-even(x / s) of the exact quotient, for |x| <= about 127 s and s >= 2^-100. The product with
// the rounded reciprocal is within 1 of it. Where x / s is near a half, x is a multiple of s's last place
// (a 16-bit type's x has at most 11 bits and is at least s / 2), so the remainder x - n s is exact in fp32
// and its comparison with s / 2 decides; elsewhere its sign relative to s / 2 survives the rounding.
S1C_DEV int quantise(float x, float s, float inv) {
  float n = rintf(x * inv);
  const float d = fmaf(-n, s, x), h = 0.5f * s;
  const bool odd = (int)n & 1;
  if (d > h || (d == h && odd)) n += 1.f;
  if (d < -h || (d == -h && odd)) n -= 1.f;
  return (int)n;
}

// Low bytes of four words.
S1C_DEV uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Eight quotients x * by rounded to bytes by the place that adding 1.5 * 2^23 gives them; false where one
// is so near a half that the product's error (below 3e-5) could decide, or is not finite.
S1C_DEV bool quantise_fast(const float (&x)[8], float by, uint32_t (&q)[2]) {
  float worst = 0.f;
  uint32_t n[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = x[j] * by, r = v + 12582912.f;
    n[j] = __float_as_uint(r);
    worst = max_nan(worst, fabsf(v - (r - 12582912.f)));
  }
  q[0] = low_bytes(n[0], n[1], n[2], n[3]), q[1] = low_bytes(n[4], n[5], n[6], n[7]);
  return worst < 0.4999f;
}

template <typename T>
S1C_DEV void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = bits_f32<T>((uint16_t)(w[j / 2] >> (16 * (j % 2))));
}

// One block for each page that new rows can touch, head, and keys or values. Bound by the rows' bytes;
// the new rows stay in registers between the maximum and the codes, so each is read once (8 x 16 B a
// thread at the largest page), and a value costs about nine instructions.
template <typename T>
__global__ void __launch_bounds__(128) cache_write_kernel(const CacheView c, const CacheRows r) {
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.x / r.units, h = blockIdx.y, kv = blockIdx.z;
  const int first = r.cu[seq], start = r.start[seq];
  const int count = min(r.cu[seq + 1] - first, r.most);
  if (count <= 0 || start < 0) return;
  const int shift = 31 - __clz(c.page), vshift = c.dim == 128 ? 4 : 3;  // 16 or 8 vectors of eight values in a row
  const int64_t at = (start >> shift) + blockIdx.x % r.units;
  const int64_t lo = max((int64_t)start, at << shift), hi = min((int64_t)start + count, (at + 1) << shift);
  if (lo >= hi) return;
  const int page = cache_page(r.table, r.max_pages, seq, at, c.num_pages);
  if (page < 0) return;
  const int old = (int)(lo - (at << shift)), vecs = (int)(hi - lo) << vshift;
  const T* src = static_cast<const T*>(r.rows[kv]) + (first + (lo - start)) * r.stride[kv] + h * c.dim;
  const int64_t slot = (int64_t)page * c.heads + h;
  int8_t* dst = c.codes[kv] + slot * c.page * c.dim;
  float* scale = c.scales[kv] + slot;

  const auto vec = [&](int i) {
    const int e = threadIdx.x + i * 128;
    return ld_once(src + (e >> vshift) * r.stride[kv] + (e & ((1 << vshift) - 1)) * 8);
  };
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (threadIdx.x + i * 128 < vecs) v[i] = vec(i);
  const float had = old ? *scale : 0.f;
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (threadIdx.x + i * 128 < vecs) {
      float x[8];
      unpack8<T>(v[i], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(x[j]));
    }
  if (!(top < INFINITY)) {  // rare: the largest of the finite ones
    top = 0.f;
#pragma unroll 1
    for (int i = 0; threadIdx.x + i * 128 < vecs; ++i) {
      float x[8];
      unpack8<T>(vec(i), x);
      for (int j = 0; j < 8; ++j)
        if (fabsf(x[j]) < INFINITY) top = fmaxf(top, fabsf(x[j]));
    }
  }
  __shared__ float tops[4];
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();  // also: every thread holds the old scale before it is replaced
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float s = fmaxf(had, top / 127.f);
  if (threadIdx.x == 0) *scale = s;
  const float inv = 1.f / s;
  const bool fast = s >= 0x1p-100f;
  uint32_t again = 0;  // vectors that need the exact way, which is kept out of the unrolled code
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = threadIdx.x + i * 128;
    if (e < vecs) {
      float x[8];
      unpack8<T>(v[i], x);
      uint32_t q[2];
      if (!(quantise_fast(x, inv, q) && fast)) again |= 1u << i;
      *reinterpret_cast<uint2*>(dst + (old * c.dim + e * 8)) = make_uint2(q[0], q[1]);
    }
  }
#pragma unroll 1
  for (; again; again &= again - 1) {
    const int i = __ffs(again) - 1;
    float x[8];
    unpack8<T>(vec(i), x);
    uint32_t q[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      int n = 0;
      if (fabsf(x[j]) < INFINITY)
        n = fast ? quantise(x[j], s, inv) : s > 0.f ? (int)fmin(fmax(rint((double)x[j] / s), -127.0), 127.0) : 0;
      else if (x[j] == x[j])
        n = x[j] > 0.f ? 127 : -127;
      q[j / 4] |= (uint32_t)(n & 255) << (8 * (j % 4));
    }
    *reinterpret_cast<uint2*>(dst + (old * c.dim + (threadIdx.x + i * 128) * 8)) = make_uint2(q[0], q[1]);
  }
  if (old && s > had) {
    const float by = had * inv;
#pragma unroll 1
    for (int e = threadIdx.x; e < old << vshift; e += 128) {
      uint2* at8 = reinterpret_cast<uint2*>(dst + e * 8);
      const uint2 was = *at8;
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = (float)(int8_t)((j < 4 ? was.x : was.y) >> (8 * (j % 4)));
      uint32_t q[2];
      if (!(quantise_fast(x, by, q) && fast)) {
        q[0] = q[1] = 0;
        for (int j = 0; j < 8; ++j) q[j / 4] |= (uint32_t)((int)rint((double)x[j] * had / s) & 255) << (8 * (j % 4));
      }
      *at8 = make_uint2(q[0], q[1]);
    }
  }
}

// Rows read back: value = code * scale, rounded once. A block has 128 rows (of 64 values: 256) of one head,
// a thread 16 values (16 B of codes, 32 B of output) of four of them; rows on pages outside the cache are
// written as 0. A byte code becomes fp32 under the exponent of 2^23.
template <typename T>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheView c, const CacheRows r) {
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.x / r.units, h = blockIdx.y, kv = blockIdx.z;
  const int first = r.cu[seq], count = min(r.cu[seq + 1] - first, r.most), start = r.start[seq];
  const int shift = 31 - __clz(c.page), vshift = c.dim == 128 ? 3 : 2;
  const int d = (threadIdx.x & ((1 << vshift) - 1)) * 16, per = 256 >> vshift;
  const int row0 = blockIdx.x % r.units * 4 * per + (threadIdx.x >> vshift);
  const bool whole = reinterpret_cast<uintptr_t>(r.rows[kv]) % 32 == 0 && r.stride[kv] % 16 == 0;
  uint4 q[4];
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = row0 + i * per, pos = start + row;
    q[i] = make_uint4(0, 0, 0, 0), s[i] = 0.f;
    if (row >= count || pos < 0) continue;
    const int page = cache_page(r.table, r.max_pages, seq, pos >> shift, c.num_pages);
    if (page < 0) continue;
    const int64_t slot = (int64_t)page * c.heads + h;
    q[i] = ld_once(c.codes[kv] + ((slot << shift) + (pos & (c.page - 1))) * c.dim + d);
    s[i] = c.scales[kv][slot];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = row0 + i * per;
    if (row >= count) continue;
    const uint32_t in[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
    uint32_t out[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w = in[j / 2] ^ 0x80808080u;
      const float lo = __uint_as_float(__byte_perm(w, 0x4b000000u, j % 2 ? 0x7442 : 0x7440)) - 8388736.f;
      const float hi = __uint_as_float(__byte_perm(w, 0x4b000000u, j % 2 ? 0x7443 : 0x7441)) - 8388736.f;
      out[j] = pack2<T>(lo * s[i], hi * s[i]);
    }
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(r.rows[kv]) + (first + row) * r.stride[kv] + h * c.dim + d);
    if (whole) {
      st_32(dst, out);
    } else {
      dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
      dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
  }
}

}  // namespace s1c
