// Causal attention of new rows over the 8-bit paged cache of kvcache.cuh. A sequence of L cached
// rows has c query rows, the last c positions: query i stands at p = L - c + i and sees the keys
// j <= p, with j >= p - window where a window is given, on pages inside the cache.
//   o = sum_j softmax_j(scale * q . k_j) v_j,   lse = ln sum_j exp(scale * q . k_j)
// A query that sees no key gets o = 0 and lse = -inf.
#pragma once
#include "kvcache.cuh"

namespace s1c {

struct CacheAttnArgs {
  const void* q;
  void* out;
  float* lse;  // nullable
  int64_t q_stride, out_stride;
  const int* cu;     // [n + 1] query rows
  const int* len;    // [n] cached rows, the query rows' own among them
  const int* table;  // [n, max_pages]
  int heads, max_pages, max_q, window;
  float scale_log2;  // scale * log2(e)
};

// One warp for each query row and head: a running maximum and sum over the keys, a lane holding
// dim / 32 of the dimensions.
template <typename T, int D>
__global__ void __launch_bounds__(128) cache_attention_rows_kernel(const CacheView c, const CacheAttnArgs a) {
  constexpr int E = D / 32;
  const int seq = blockIdx.x / a.max_q, i = blockIdx.x % a.max_q, lane = threadIdx.x % 32;
  const int head = blockIdx.y * 4 + threadIdx.x / 32;
  const int first = a.cu[seq], count = a.cu[seq + 1] - first;
  if (i >= count || head >= a.heads) return;
  const int h = head / (a.heads / c.heads);
  const int64_t row = first + i;
  const T* q = static_cast<const T*>(a.q) + row * a.q_stride + head * D + lane * E;
  float qf[E], o[E] = {};
  for (int e = 0; e < E; ++e) qf[e] = to_f32(q[e]) * a.scale_log2;
  const int64_t pos = (int64_t)a.len[seq] - count + i;
  float top = -INFINITY, sum = 0.f;
  for (int64_t j = a.window < 0 ? 0 : max((int64_t)0, pos - a.window); j <= pos; ++j) {
    const int page = cache_page(a.table, a.max_pages, seq, (int)(j / c.page), c.num_pages);
    if (page < 0) continue;
    const int64_t slot = (int64_t)page * c.heads + h;
    const int64_t at = (slot * c.page + j % c.page) * D + lane * E;
    float s = 0.f;
    for (int e = 0; e < E; ++e) s += qf[e] * (float)c.codes[0][at + e];
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= c.scales[0][slot];
    const float m = fmaxf(top, s), keep = exp2f(top - m), p = exp2f(s - m);
    const float vs = p * c.scales[1][slot];
    sum = sum * keep + p;
    for (int e = 0; e < E; ++e) o[e] = o[e] * keep + vs * (float)c.codes[1][at + e];
    top = m;
  }
  T* out = static_cast<T*>(a.out) + row * a.out_stride + head * D + lane * E;
  for (int e = 0; e < E; ++e) out[e] = from_f32<T>(sum > 0.f ? o[e] / sum : 0.f);
  if (a.lse && lane == 0) a.lse[row * a.heads + head] = (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace s1c
