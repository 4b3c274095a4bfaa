// Host side of the token-step operators of include/s1c.h: products with 4-bit weights, the 8-bit paged
// cache, attention over it, and sampling. Each call checks its arguments, runs on the device that
// holds its output, enqueues its kernels on the caller's stream and allocates nothing.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <string>
#include <vector>

#include "errors.h"
#include "launch.h"
#include "cache_attention.cuh"
#include "kvcache.cuh"
#include "nibble.cuh"
#include "sample.cuh"

using namespace s1c;

namespace s1c {
// nibble_f16.cu and its kind
void launch_nibble_f16(const NibbleArgs& a, int group, int dev, cudaStream_t st);
void launch_nibble_bf16(const NibbleArgs& a, int group, int dev, cudaStream_t st);
void launch_nibble_f16_zeros(const NibbleArgs& a, int group, int dev, cudaStream_t st);
void launch_nibble_bf16_zeros(const NibbleArgs& a, int group, int dev, cudaStream_t st);
}  // namespace s1c

namespace {

void need(bool ok, const char* what) {
  if (!ok) throw S1cError(S1C_ERR_ARG, what);
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Pointers (null ones are) to elements of `bytes` that lie where such elements may.
template <typename... P>
void need_elements(size_t bytes, const P*... p) {
  need(((reinterpret_cast<uintptr_t>(p) % bytes == 0) && ...), "a pointer is not aligned to its element type");
}

// Makes the device that holds `p` current for the call, so that a caller with several devices needs no
// cudaSetDevice; put back at the end. Host memory that the device cannot be shown to reach is refused.
struct OnDeviceOf {
  int was = -1, device = 0;
  explicit OnDeviceOf(const void* p) {
    cudaPointerAttributes at;
    CK(cudaPointerGetAttributes(&at, p));
    need(at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged, "outputs must be device memory");
    int now = 0;
    device = at.device;
    CK(cudaGetDevice(&now));
    if (at.device != now) {
      CK(cudaSetDevice(at.device));
      was = now;
    }
  }
  ~OnDeviceOf() {
    if (was >= 0) cudaSetDevice(was);
  }
};

template <typename F>
s1c_status enter(F&& f) {
  try {
    f();
    return S1C_OK;
  } catch (const S1cError& e) {
    set_create_error(e.what());
    return e.code;
  } catch (const std::exception& e) {
    set_create_error(e.what());
    return S1C_ERR_ARG;
  } catch (...) {
    set_create_error("unknown error");
    return S1C_ERR_ARG;
  }
}

void check_half(int dtype) { need(dtype == S1C_DT_F16 || dtype == S1C_DT_BF16, "dtype must be S1C_DT_F16 or S1C_DT_BF16"); }

CacheView check_cache(const s1c_cache* c) {
  need(c && c->k_codes && c->v_codes && c->k_scales && c->v_scales, "null cache or cache buffer");
  need(c->num_pages > 0 && c->kv_heads > 0 && c->kv_heads <= 65535, "num_pages and kv_heads must be positive (kv_heads at most 65535)");
  need(c->page == 16 || c->page == 32 || c->page == 64, "page must be 16, 32 or 64");
  need(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128");
  need(aligned(c->k_codes, 16) && aligned(c->v_codes, 16), "cache codes must be 16-byte aligned");
  need_elements(4, c->k_scales, c->v_scales);
  need((int64_t)c->num_pages * c->kv_heads * c->page <= INT_MAX, "num_pages * kv_heads * page must stay below 2^31");
  return CacheView{{static_cast<int8_t*>(c->k_codes), static_cast<int8_t*>(c->v_codes)}, {c->k_scales, c->v_scales},
                   c->num_pages, c->page, c->kv_heads, c->head_dim};
}

CacheRows check_rows(const CacheView& c, const void* k, int64_t k_stride, const void* v, int64_t v_stride, const int32_t* cu,
                     const int32_t* start, const int32_t* table, int32_t max_pages, int32_t n, int32_t most) {
  need(k && v && cu && start && table, "null argument");
  need(n >= 0 && most >= 0 && max_pages > 0, "n and the row bound must not be negative, max_pages positive");
  need(k_stride >= (int64_t)c.heads * c.dim && v_stride >= (int64_t)c.heads * c.dim && k_stride % 8 == 0 && v_stride % 8 == 0,
       "row strides must hold kv_heads * head_dim values and be multiples of 8");
  need(aligned(k, 16) && aligned(v, 16), "rows must be 16-byte aligned");
  need_elements(4, cu, start, table);
  CacheRows r{};
  r.rows[0] = const_cast<void*>(k), r.rows[1] = const_cast<void*>(v);
  r.stride[0] = k_stride, r.stride[1] = v_stride;
  r.cu = cu, r.start = start, r.table = table, r.max_pages = max_pages, r.most = most;
  return r;
}

// How an attention call is laid out: blocks of 16 rows, or of 128 that share the keys' conversion; keys of a block.
// Up to 32 rows of a key head take blocks of 16 (4 key heads of 128, pages of 16, both ways in us): 16 sequences of
// 16384 keys with 32 rows 113 and 132, with 40 rows 161 and 133; 64 of 4096 with 32 rows 121 and 132, with 40 rows
// 169 and 136. A single sequence leans to either side: 16384 keys with 64 rows 23 and 26, 131072 with 24 rows 77
// and 67.
struct AttnPlan {
  bool prompt;
  int tiles, chunk, chunks;
};
constexpr int ATTN_FEW_ROWS = 32;                              // of a key head: up to here blocks of 16 rows
constexpr int ATTN_FEW_ROUND = 444, ATTN_PROMPT_ROUND = 296;  // blocks that 148 SMs hold: three each, or two of a prompt's
constexpr int ATTN_PROMPT_WHOLE = 148;                         // prompts' blocks from which keys stay together where they may
int64_t chunk_most(const CacheView& c, bool prompt) {
  return prompt ? (int64_t)CATP_PAGES * c.page - 128 : std::min<int64_t>(2048, (int64_t)CATT_PAGES * c.page);
}
AttnPlan plan_attention(const CacheView& c, int heads, int n, int max_q, int max_kv) {
  const int64_t rows = (int64_t)max_q * (heads / c.heads);
  AttnPlan p;
  p.prompt = rows > ATTN_FEW_ROWS;
  const int per = p.prompt ? CATP_ROWS : 16;
  p.tiles = (int)((rows + per - 1) / per);
  const int64_t units = (int64_t)n * c.heads * p.tiles;
  // one round of blocks
  const int64_t round = p.prompt ? ATTN_PROMPT_ROUND : ATTN_FEW_ROUND, want = (units * max_kv + round - 1) / round;
  const int64_t most = chunk_most(c, p.prompt);
  p.chunk = (int)std::max<int64_t>(128, std::min(most, (want + 127) / 128 * 128));
  if (p.prompt && units >= ATTN_PROMPT_WHOLE && max_kv <= most) p.chunk = (int)most;
  p.chunks = (int)std::max<int64_t>(1, ((int64_t)max_kv + p.chunk - 1) / p.chunk);
  return p;
}
// What a call writes there: dim + 1 numbers for each row, head and chunk.
size_t attention_partials(const AttnPlan& p, const CacheView& c, int heads, int n, int max_q) {
  return p.chunks == 1 ? 0 : (size_t)n * max_q * heads * p.chunks * (c.dim + 1) * sizeof(float);
}
// What a call needs if it splits keys at all: enough for every call with bounds up to these, so that one buffer
// serves all of them, although a smaller call may split its keys more. A chunk has its largest size, and there
// are ceil(kv / most); or at least units * kv / round keys, so ceil(round / units) of them at most, for no more
// than `per` rows and heads in each of fewer than `round` units; and 128 keys at least.
size_t attention_workspace(const CacheView& c, int heads, int n, int max_q, int max_kv) {
  const int64_t G = heads / c.heads, least = ((int64_t)max_kv + 127) / 128;
  int64_t parts = 0;
  const auto form = [&](bool prompt, int64_t q, int64_t per, int64_t round, int64_t units) {
    const int64_t items = (int64_t)n * q * heads, largest = (max_kv + chunk_most(c, prompt) - 1) / chunk_most(c, prompt);
    if (max_kv > chunk_most(c, prompt))
      parts = std::max(parts, items * largest);
    else if (prompt)
      units = std::min<int64_t>(units, ATTN_PROMPT_WHOLE);
    if (least > 1) parts = std::max(parts, std::min(items * least, per * (round + units - 1)));
  };
  form(false, std::min<int64_t>(max_q, ATTN_FEW_ROWS / G), 16, ATTN_FEW_ROUND, ATTN_FEW_ROUND);
  if (max_q * G > ATTN_FEW_ROWS) form(true, max_q, CATP_ROWS, ATTN_PROMPT_ROUND, ATTN_PROMPT_ROUND);
  return (size_t)parts * (c.dim + 1) * sizeof(float);
}

template <typename T, int D>
void launch_attention(const CacheView& c, const CacheAttnArgs& a, bool prompt, int dev, cudaStream_t st) {
  const uint64_t rows = (uint64_t)c.num_pages * c.heads * c.page;
  const uint32_t box = std::min(c.page, CATT_BOX);
  const CUtensorMap k = byte_map(c.codes[0], D, rows, D, D, box), v = byte_map(c.codes[1], D, rows, D, D, box);
  const dim3 grid((unsigned)(a.n * c.heads * a.tiles), a.chunks);
  if (prompt) {
    allow_smem<cache_prompt_kernel<T, D>>(dev);
    launch_after(cache_prompt_kernel<T, D>, grid, CATP_WARPS * 32, sizeof(CachePromptSmem<D>) + 1024, 1, st, k, v, c, a);
  } else {
    allow_smem<cache_attention_kernel<T, D>>(dev);
    launch_after(cache_attention_kernel<T, D>, grid, CATT_WARPS * 32, sizeof(CacheAttnSmem<D>) + 1024, 1, st, k, v, c, a);
  }
  if (a.chunks > 1) {
    const unsigned items = (unsigned)((int64_t)a.n * a.max_q * a.heads);
    if (a.chunks > 16)
      launch_after(cache_attention_join_kernel<T, D, 16>, items, 512, 0, 1, st, a);
    else
      launch_after(cache_attention_join_kernel<T, D, 4>, items, 128, 0, 1, st, a);
  }
}
template <typename T>
void launch_attention(const CacheView& c, const CacheAttnArgs& a, bool prompt, int dev, cudaStream_t st) {
  c.dim == 64 ? launch_attention<T, 64>(c, a, prompt, dev, st) : launch_attention<T, 128>(c, a, prompt, dev, st);
}

// Attention of `rows` queries over `keys` positions whose loads are waited for in vain; true if every row came
// out as NaN, and a call without the fault has none.
bool attention_gives_up(int device, int dim, int rows, int keys, uint64_t wait_ns) {
  struct Buffer {
    void* p = nullptr;
    explicit Buffer(size_t bytes) {
      CK(cudaMalloc(&p, bytes));
      const cudaError_t e = cudaMemset(p, 0, bytes);
      if (e != cudaSuccess) cudaFree(p);
      CK(e);
    }
    ~Buffer() { cudaFree(p); }
  };
  const int page = 16, pages = (keys + page - 1) / page;
  Buffer k((size_t)pages * page * dim), v((size_t)pages * page * dim), ks(pages * 4), vs(pages * 4), q((size_t)rows * dim * 2),
      out((size_t)rows * dim * 2), lse(rows * 4), cu(8), len(4), table(pages * 4);
  const CacheView c{{static_cast<int8_t*>(k.p), static_cast<int8_t*>(v.p)}, {static_cast<float*>(ks.p), static_cast<float*>(vs.p)}, pages, page, 1, dim};
  const AttnPlan p = plan_attention(c, 1, 1, rows, keys);
  Buffer ws(std::max<size_t>(16, attention_partials(p, c, 1, 1, rows)));
  std::vector<int> order(pages);
  for (int i = 0; i < pages; ++i) order[i] = i;
  const int ends[2] = {0, rows};
  CK(cudaMemcpy(table.p, order.data(), pages * 4, cudaMemcpyHostToDevice));
  CK(cudaMemcpy(cu.p, ends, 8, cudaMemcpyHostToDevice));
  CK(cudaMemcpy(len.p, &keys, 4, cudaMemcpyHostToDevice));
  CacheAttnArgs a{q.p, out.p, static_cast<float*>(lse.p), dim, dim, static_cast<int*>(cu.p), static_cast<int*>(len.p),
                  static_cast<int*>(table.p), 1, 1, pages, rows, -1, p.tiles, p.chunk, p.chunks, 1.f};
  a.part = static_cast<float*>(ws.p);
  a.part_lse = a.part + (size_t)rows * p.chunks * dim;
  a.wait_ns = wait_ns;
  for (int beyond : {16, 0}) {
    a.beyond = beyond;
    launch_attention<__half>(c, a, p.prompt, device, nullptr);
    CK(cudaDeviceSynchronize());
    std::vector<uint16_t> o((size_t)rows * dim);
    std::vector<float> l(rows);
    CK(cudaMemcpy(o.data(), out.p, o.size() * 2, cudaMemcpyDeviceToHost));
    CK(cudaMemcpy(l.data(), lse.p, l.size() * 4, cudaMemcpyDeviceToHost));
    const auto nan = [](uint16_t h) { return (h & 0x7fff) > 0x7c00; };
    const int64_t nans = std::count_if(o.begin(), o.end(), nan) + std::count_if(l.begin(), l.end(), [](float x) { return std::isnan(x); });
    if (nans != (beyond ? (int64_t)(o.size() + l.size()) : 0)) return false;
  }
  return true;
}

// A row is shared by a cluster of up to eight blocks, as long as there are SMs for them and each keeps a
// thousand logits.
template <typename T>
void launch_sample(SampleArgs a, int rows, int dev, cudaStream_t st) {
  int blocks = 1;
  while (blocks < SMP_CLUSTER && 2 * blocks * rows <= sm_count(dev) && a.vocab >= 2048 * blocks) blocks *= 2;
  a.slice = ((a.vocab + blocks - 1) / blocks + 7) / 8 * 8;
  a.vec = aligned(a.logits, 16) && a.stride * (int64_t)sizeof(T) % 16 == 0;
  allow_smem<sample_kernel<T>>(dev);
  launch_after(sample_kernel<T>, (unsigned)(rows * blocks), SMP_THREADS, sizeof(SampleShared), blocks, st, a);
}

}  // namespace

extern "C" {

s1c_status s1c_nibble_gemm(int32_t dtype, const void* d_x, int64_t x_stride, const void* d_codes, int64_t code_pitch,
                           const void* d_scales, const void* d_zeros, int64_t scale_stride, int32_t group, void* d_out,
                           int64_t out_stride, int32_t M, int32_t N, int32_t K, const float* d_bias, int32_t act,
                           int32_t out_f32, void* stream) {
  return enter([&] {
    check_half(dtype);
    need(d_x && d_codes && d_scales && d_out, "null argument");
    need(M >= 0 && M <= 64 && N > 0 && K > 0 && N <= (1 << 30) && K <= (1 << 30), "M must be 0 to 64, N and K 1 to 2^30");
    need(group == 32 || group == 64 || group == 128, "group must be 32, 64 or 128");
    const int64_t groups = ((int64_t)K + group - 1) / group;
    need(code_pitch % 16 == 0 && code_pitch >= ((int64_t)K + 31) / 32 * 16 && aligned(d_codes, 16),
         "codes must be 16-byte aligned, their row pitch a multiple of 16 bytes that holds K rounded up to 32 codes");
    need(x_stride >= K && out_stride >= N && scale_stride >= groups, "a row stride is shorter than its row");
    need_elements(2, d_x, d_scales, d_zeros);
    need_elements(4, d_bias);
    need_elements(out_f32 ? 4 : 2, d_out);
    need(act >= 0 && act <= 2, "act must be 0 (none), 1 (ReLU) or 2 (GELU)");
    if (M == 0) return;
    OnDeviceOf dev(d_out);
    NibbleArgs a{d_x, static_cast<const uint8_t*>(d_codes), d_scales, d_zeros, d_out, d_bias, x_stride, code_pitch,
                 scale_stride, out_stride, M, N, K, (int)groups, act, out_f32};
    a.vec = x_stride % 8 == 0 && aligned(d_x, 16);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == S1C_DT_F16)
      (d_zeros ? launch_nibble_f16_zeros : launch_nibble_f16)(a, group, dev.device, st);
    else
      (d_zeros ? launch_nibble_bf16_zeros : launch_nibble_bf16)(a, group, dev.device, st);
  });
}

s1c_status s1c_cache_write(const s1c_cache* cache, int32_t dtype, const void* d_k, int64_t k_stride, const void* d_v,
                           int64_t v_stride, const int32_t* d_cu, const int32_t* d_start, const int32_t* d_pages,
                           int32_t max_pages, int32_t n, int32_t max_new, void* stream) {
  return enter([&] {
    const CacheView c = check_cache(cache);
    check_half(dtype);
    CacheRows r = check_rows(c, d_k, k_stride, d_v, v_stride, d_cu, d_start, d_pages, max_pages, n, max_new);
    if (n == 0 || max_new == 0) return;
    r.units = (int)(((int64_t)max_new + c.page - 2) / c.page + 1);
    need((int64_t)n * r.units <= INT_MAX, "n * pages must stay below 2^31");
    OnDeviceOf dev(cache->k_codes);
    const dim3 grid((unsigned)(n * r.units), (unsigned)c.heads, 2);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == S1C_DT_F16)
      launch_after(cache_write_kernel<__half>, grid, 128, 0, 1, st, c, r);
    else
      launch_after(cache_write_kernel<__nv_bfloat16>, grid, 128, 0, 1, st, c, r);
  });
}

s1c_status s1c_cache_read(const s1c_cache* cache, int32_t dtype, void* d_k, int64_t k_stride, void* d_v, int64_t v_stride,
                          const int32_t* d_cu, const int32_t* d_start, const int32_t* d_pages, int32_t max_pages, int32_t n,
                          int32_t max_rows, void* stream) {
  return enter([&] {
    const CacheView c = check_cache(cache);
    check_half(dtype);
    CacheRows r = check_rows(c, d_k, k_stride, d_v, v_stride, d_cu, d_start, d_pages, max_pages, n, max_rows);
    if (n == 0 || max_rows == 0) return;
    const int rows = 4 * 256 / (c.dim / 16);  // of a block
    const int64_t units = ((int64_t)max_rows + rows - 1) / rows;
    need(n * units <= INT_MAX, "n * max_rows is too large for one call");
    r.units = (int)units;
    OnDeviceOf dev(d_k);
    const dim3 grid((unsigned)(n * units), (unsigned)c.heads, 2);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == S1C_DT_F16)
      launch_after(cache_read_kernel<__half>, grid, 256, 0, 1, st, c, r);
    else
      launch_after(cache_read_kernel<__nv_bfloat16>, grid, 256, 0, 1, st, c, r);
  });
}

size_t s1c_cache_attention_workspace(const s1c_cache* cache, int32_t heads, int32_t n, int32_t max_q, int32_t max_kv) {
  try {
    const CacheView c = check_cache(cache);
    if (heads <= 0 || heads % c.heads || n <= 0 || max_q <= 0 || max_kv <= 0 || max_kv > (1 << 30) || (int64_t)n * max_q > INT_MAX / heads)
      return 0;
    return attention_workspace(c, heads, n, max_q, max_kv);
  } catch (...) {
    return 0;
  }
}

s1c_status s1c_cache_attention(const s1c_cache* cache, int32_t dtype, const void* d_q, int64_t q_stride, void* d_out,
                               int64_t out_stride, float* d_lse, int32_t heads, const int32_t* d_cu, const int32_t* d_len,
                               const int32_t* d_pages, int32_t max_pages, int32_t n, int32_t max_q, int32_t max_kv,
                               int32_t window, float scale, void* d_workspace, size_t workspace_bytes, void* stream) {
  return enter([&] {
    const CacheView c = check_cache(cache);
    check_half(dtype);
    need(d_q && d_out && d_cu && d_len && d_pages, "null argument");
    need(heads > 0 && heads % c.heads == 0, "heads must be a multiple of kv_heads");
    need(n >= 0 && max_q >= 0 && max_kv >= 0 && max_kv <= (1 << 30) && max_pages > 0,
         "n, max_q and max_kv must not be negative, max_kv at most 2^30, max_pages positive");
    const int64_t width = (int64_t)heads * c.dim;
    need(q_stride >= width && out_stride >= width && q_stride % 8 == 0 && out_stride % 8 == 0 && aligned(d_q, 16) && aligned(d_out, 16),
         "q and out must be 16-byte aligned, their row strides multiples of 8 that hold heads * head_dim values");
    need(std::isfinite(scale), "scale must be finite");
    need_elements(4, d_lse, d_cu, d_len, d_pages);
    if (n == 0 || max_q == 0) return;
    need((int64_t)n * max_q <= INT_MAX / heads, "n * max_q * heads must stay below 2^31");
    const AttnPlan p = plan_attention(c, heads, n, max_q, max_kv);
    const size_t used = attention_partials(p, c, heads, n, max_q);
    const size_t bytes = used ? std::max(used, attention_workspace(c, heads, n, max_q, max_kv)) : 0;
    need(p.chunks <= 65535, "max_kv is too large");
    need(workspace_bytes >= bytes && (!bytes || (d_workspace && aligned(d_workspace, 16))),
         "workspace too small, null or not 16-byte aligned");
    OnDeviceOf dev(d_out);
    CacheAttnArgs a{d_q, d_out, d_lse, q_stride, out_stride, d_cu, d_len, d_pages, n, heads, max_pages, max_q, window,
                    p.tiles, p.chunk, p.chunks, scale * 1.4426950408889634f};
    a.part = static_cast<float*>(d_workspace);
    a.part_lse = a.part + (size_t)n * max_q * heads * p.chunks * c.dim;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == S1C_DT_F16)
      launch_attention<__half>(c, a, p.prompt, dev.device, st);
    else
      launch_attention<__nv_bfloat16>(c, a, p.prompt, dev.device, st);
  });
}

s1c_status s1c_selftest_cache_attention_timeout(int32_t device, int64_t budget_ns, int32_t* codes) {
  return enter([&] {
    need(codes && budget_ns >= 1000000 && budget_ns <= 2000000000, "budget_ns must lie in [1e6, 2e9] and codes must not be null");
    CK(cudaSetDevice(device));
    for (int i = 0; i < 4; ++i) {
      const int rows = i < 2 ? 3 : 40, keys = i % 2 ? 1000 : 100;
      codes[i] = attention_gives_up(device, 64, rows, keys, (uint64_t)budget_ns) && attention_gives_up(device, 128, rows, keys, (uint64_t)budget_ns);
    }
  });
}

s1c_status s1c_sample(int32_t dtype, const void* d_logits, int64_t row_stride, int32_t rows, int32_t vocab,
                      const float* d_temperature, const int32_t* d_top_k, const float* d_top_p, const float* d_min_p,
                      const float* d_uniform, int32_t* d_token, float* d_prob, void* stream) {
  return enter([&] {
    need(dtype == S1C_DT_F32 || dtype == S1C_DT_F16 || dtype == S1C_DT_BF16, "dtype must be S1C_DT_F32, F16 or BF16");
    need(d_logits && d_uniform && d_token, "null argument");
    need(rows >= 0 && vocab > 0 && vocab <= (1 << 18), "rows must not be negative, vocab 1 to 2^18");
    need(rows <= INT_MAX / SMP_CLUSTER, "too many rows");
    need(row_stride >= vocab, "a row stride is shorter than its row");
    need_elements(dtype == S1C_DT_F32 ? 4 : 2, d_logits);
    need_elements(4, d_temperature, d_top_k, d_top_p, d_min_p, d_uniform, d_token, d_prob);
    if (rows == 0) return;
    OnDeviceOf dev(d_token);
    SampleArgs a{d_logits, row_stride, vocab, d_temperature, d_top_k, d_top_p, d_min_p, d_uniform, d_token, d_prob};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == S1C_DT_F32)
      launch_sample<float>(a, rows, dev.device, st);
    else if (dtype == S1C_DT_F16)
      launch_sample<__half>(a, rows, dev.device, st);
    else
      launch_sample<__nv_bfloat16>(a, rows, dev.device, st);
  });
}

}  // extern "C"
