// A paged cache of keys and values held in 8 bits: pages [num_pages, kv_heads, page, head_dim] of
// int8 codes and one fp32 scale for each page and head, a value being code * scale.
//
// Writing. A sequence's rows stand at consecutive positions; position p lies in row p % page of the
// page its table names at p / page. For a page and head that new rows fall into
//   s = max(s_old, fl32(max |new| / 127)), s_old = the page's scale if earlier rows of the sequence
// stand in it, else 0; a new value becomes round-half-even(x / s), and where s grew the earlier codes
// become round-half-even(code * s_old / s), both of the exact quotient.
#pragma once
#include "common.cuh"

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
S1C_DEV int cache_page(const int* table, int64_t max_pages, int seq, int at, int num_pages) {
  if (at < 0 || at >= max_pages) return -1;
  const int p = table[seq * max_pages + at];
  return p >= 0 && p < num_pages ? p : -1;
}

// round-half-even(x / s) of the exact quotient, for |x| <= about 127 s and s >= 2^-100. The product
// with the rounded reciprocal is within 1 of it. Where x / s is near a half, x is a multiple of s's last place
// (a 16-bit type's x has at most 11 bits and is at least s / 2), so the remainder x - n s is exact in fp32 and its comparison with s / 2
// decides; elsewhere its sign relative to s / 2 survives the rounding.
S1C_DEV int quantise(float x, float s, float inv) {
  float n = rintf(x * inv);
  const float d = fmaf(-n, s, x), h = 0.5f * s;
  const bool odd = (int)n & 1;
  if (d > h || (d == h && odd)) n += 1.f;
  if (d < -h || (d == -h && odd)) n -= 1.f;
  return (int)n;
}

// One block for each page that new rows can touch, head, and keys or values. Bound by the rows' bytes;
// the new rows stay in registers between the maximum and the codes, so each is read once (8 x 16 B a
// thread at the largest page).
template <typename T>
__global__ void __launch_bounds__(128) cache_write_kernel(const CacheView c, const CacheRows r) {
  const int seq = blockIdx.x / r.units, h = blockIdx.y, kv = blockIdx.z;
  const int first = r.cu[seq], start = r.start[seq];
  const int count = min(r.cu[seq + 1] - first, r.most);
  if (count <= 0 || start < 0) return;
  const int64_t at = (int64_t)start / c.page + blockIdx.x % r.units;
  const int64_t lo = max((int64_t)start, at * c.page), hi = min((int64_t)start + count, (at + 1) * c.page);
  if (lo >= hi) return;
  const int page = cache_page(r.table, r.max_pages, seq, (int)at, c.num_pages);
  if (page < 0) return;
  const int old = (int)(lo - at * c.page), rows = (int)(hi - lo), vecs = c.dim / 8;
  const T* src = static_cast<const T*>(r.rows[kv]) + (first + (lo - start)) * r.stride[kv] + h * c.dim;
  const int64_t slot = (int64_t)page * c.heads + h;
  int8_t* dst = c.codes[kv] + slot * c.page * c.dim;
  float* scale = c.scales[kv] + slot;

  uint4 v[8];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = threadIdx.x + i * 128;
    if (e < rows * vecs) {
      v[i] = *reinterpret_cast<const uint4*>(src + (e / vecs) * r.stride[kv] + (e % vecs) * 8);
      const T* x = reinterpret_cast<const T*>(&v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = fabsf(to_f32(x[j]));
        if (f < INFINITY) top = fmaxf(top, f);
      }
    }
  }
  __shared__ float tops[4];
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  const float had = old ? *scale : 0.f;
  __syncthreads();  // also: every thread holds the old scale before it is replaced
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float s = fmaxf(had, top / 127.f);
  if (threadIdx.x == 0) *scale = s;
  const float inv = 1.f / s;
  const bool fast = s >= 0x1p-100f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = threadIdx.x + i * 128;
    if (e < rows * vecs) {
      const T* x = reinterpret_cast<const T*>(&v[i]);
      uint32_t q[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = to_f32(x[j]);
        int n = 0;
        if (fabsf(f) < INFINITY)
          n = fast ? quantise(f, s, inv) : s > 0.f ? (int)fmin(fmax(rint((double)f / s), -127.0), 127.0) : 0;
        else if (f == f)
          n = f > 0.f ? 127 : -127;
        q[j / 4] |= (uint32_t)(n & 255) << (8 * (j % 4));
      }
      *reinterpret_cast<uint2*>(dst + (old + e / vecs) * c.dim + (e % vecs) * 8) = make_uint2(q[0], q[1]);
    }
  }
  if (old && s > had) {
    for (int e = threadIdx.x; e < old * c.dim; e += 128)
      dst[e] = (int8_t)rint((double)dst[e] * had / s);
  }
}

// Rows read back: value = code * scale, rounded once. A thread takes 16 values (16 B of codes, 32 B
// of output); rows on pages outside the cache are written as 0.
template <typename T>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheView c, const CacheRows r) {
  const int seq = blockIdx.x / r.units, kv = blockIdx.y;
  const int first = r.cu[seq], count = min(r.cu[seq + 1] - first, r.most), start = r.start[seq];
  const int vecs = c.dim / 16, per = c.heads * vecs;
  const int64_t e = (int64_t)(blockIdx.x % r.units) * 256 + threadIdx.x;
  const int64_t row = e / per;
  if (row >= count) return;
  const int h = (int)(e % per) / vecs, d = (int)(e % per) % vecs * 16;
  const int64_t pos = start + row;
  const int page = pos < 0 ? -1 : cache_page(r.table, r.max_pages, seq, (int)(pos / c.page), c.num_pages);
  uint4 q = make_uint4(0, 0, 0, 0);
  float s = 0.f;
  if (page >= 0) {
    const int64_t slot = (int64_t)page * c.heads + h;
    q = *reinterpret_cast<const uint4*>(c.codes[kv] + (slot * c.page + pos % c.page) * c.dim + d);
    s = c.scales[kv][slot];
  }
  T out[16];
  const int8_t* b = reinterpret_cast<const int8_t*>(&q);
#pragma unroll
  for (int j = 0; j < 16; ++j) out[j] = from_f32<T>((float)b[j] * s);
  uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(r.rows[kv]) + (first + row) * r.stride[kv] + h * c.dim + d);
  dst[0] = reinterpret_cast<const uint4*>(out)[0];
  dst[1] = reinterpret_cast<const uint4*>(out)[1];
}

}  // namespace s1c
