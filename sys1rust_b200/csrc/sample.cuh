// One token for each row of logits under temperature, top-k, top-p and min-p.
//
// With z_i = (max l - l_i) / T and e_i = exp(-z_i), tokens ordered by descending logit (the lowest index first
// among equals): top-k keeps the first k; top-p keeps, of these, the first and every one whose
// predecessors' mass is below p times the mass of the k; min-p keeps those with e_i >= min_p. The
// token is the first index, in ascending order, at which the kept mass summed so far exceeds u times the kept mass.
//
// No sort is needed: both filters cut the order at one value, so each is a threshold (a logit, and how
// many of its equals are kept, by index). A cluster of blocks shares a row:
//
//  1. each block copies its part to shared memory and finds the largest logit;
//  2. the counts of the logits in bins of z, 1/32 of a power of two wide, and where top-p needs it the exact
//     mass of all, give a bin below which nothing can be kept;
//  3. what stands above, a few hundred of fifty thousand as a rule, is gathered in the order of the indexes in the first
//     block, which finds the thresholds exactly, by histograms over bins of z and, inside the bin
//     that holds the cut, over the order-preserving integer of the logit, 2048 ways at a time, until one
//     value is left; and then sums and walks what is kept. More than fit are worked on in place.
//
// Masses are integers: e = m * 2^(n - 24), m an integer of 25 bits, and all e in one bin share n. So their sums are
// exact and depend neither on the order of atomics nor on how a row is shared. Logits more than 45 powers of two
// below the largest have no mass.
#pragma once
#include <cooperative_groups.h>

#include "common.cuh"

namespace s1c {

struct SampleArgs {
  const void* logits;
  int64_t stride;
  int vocab;
  const float* temperature;  // each nullable: 1, off, off, off
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int* token;
  float* prob;  // nullable
  int slice;    // logits of a block, a multiple of 8
  int vec;      // rows are 16-byte aligned
};

constexpr int SMP_THREADS = 1024, SMP_WARPS = SMP_THREADS / 32, SMP_BINS = 2048, SMP_ZBINS = 45 * 32, SMP_LIST = 8192;
constexpr int SMP_CLUSTER = 8;

// The order-preserving integer of a logit: a > b as floats exactly if it is so for the keys.
S1C_DEV uint32_t logit_key(float l) {
  const uint32_t u = __float_as_uint(l);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
S1C_DEV float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

S1C_DEV double pow2(int e) { return __hiloint2double((1023 + e) << 20, 0); }

// exp as an integer: the bin of z and m with e = m * 2^(n - 24), n from the bin. The bin comes from the rounded product (it
// only has to be monotonic); the mass adds what the difference and the product lost. 2^f by the Taylor series of
// exp(f ln 2), |f| <= 1/2: its tenth term is below 1e-10, and rounding to fp32 leaves about 5e-8.
struct SampleMass {
  float top, rate, rate_lo;  // max l, log2(e) / T in two parts
  S1C_DEV SampleMass(float top_, float T) : top(top_) {
    const double r = fmin(1.4426950408889634 / (double)T, 1e38);
    rate = (float)r, rate_lo = (float)(r - (double)rate);
  }
  S1C_DEV int bin(float l) const {
    const float t = (top - l) * rate * 32.f;
    return t < (float)SMP_ZBINS ? (int)t : SMP_ZBINS;
  }
  static S1C_DEV int power(int bin) { return -((bin + 16) >> 5); }
  S1C_DEV uint32_t mass(float l, int bin) const {
    const float d = top - l, lost = (top - d) - l, z = d * rate;
    const float more = fmaf(d, rate, -z) + fmaf(d, rate_lo, lost * rate);
    const float f = (((float)-power(bin) - z) - more) * 0.69314718055994531f;
    float g = 2.7557319e-6f;
    g = fmaf(g, f, 2.4801587e-5f);
    g = fmaf(g, f, 1.9841270e-4f);
    g = fmaf(g, f, 1.3888889e-3f);
    g = fmaf(g, f, 8.3333333e-3f);
    g = fmaf(g, f, 4.1666667e-2f);
    g = fmaf(g, f, 0.16666667f);
    g = fmaf(g, f, 0.5f);
    g = fmaf(g, f, 1.0f);
    const uint32_t e = __float_as_uint(fmaf(g, f, 1.0f));  // in (0.5, 2): the significand, doubled from 1 on
    return ((e & 0x7fffffu) | 0x800000u) << ((e >> 23) - 126);
  }
  // the same as a fixed-point number of 44 places, for sums over bins
  S1C_DEV unsigned long long fixed(float l, int bin) const { return ((unsigned long long)mass(l, bin) << 20) >> -power(bin); }
};

struct SampleShared {
  // elements of a bin; sums of the low 12 and the high 13 bits of their masses (below 2^32 for 2^18 elements)
  uint32_t count[SMP_BINS], lo[SMP_BINS], hi[SMP_BINS];
  float value[SMP_LIST];  // what step 3 works on
  int index[SMP_LIST];
  double warp_d[SMP_WARPS];
  unsigned long long warp_u[SMP_WARPS];
  uint32_t warp_a[SMP_WARPS], warp_b[SMP_WARPS];
  uint32_t key_lo, key_hi;
  int found_bin;
  uint32_t found_count;
  double found_mass;
  // read by the other blocks of the cluster
  float top;
  int at, bad;
  uint32_t listed;
  unsigned long long sum;
  S1C_DEV unsigned long long mass(int b) const { return ((unsigned long long)hi[b] << 12) + lo[b]; }
};

// What is kept: keys above `key`, and the first `need` of those equal to it.
struct SampleCut {
  uint32_t key, need;
};

// The elements of step 3: the list, or the row itself.
template <typename T>
struct SampleItems {
  const float* value;  // null: the row
  const T* row;
  int n;
  S1C_DEV float operator()(int i) const { return value ? value[i] : to_f32(row[i]) + 0.f; }
};

// First bin whose elements reach `want` (by count), or last non-empty bin whose predecessors' mass is
// below `want` (by mass), and the count and mass before it; -1 where there is none. A mass counts 2^power
// of its bin of z, or `scale`. All threads call.
template <bool MASS>
S1C_DEV void sample_find(SampleShared& s, int bins, double want, bool zbins, double scale) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int b0 = 2 * t;
  double m[2] = {0, 0};
  uint32_t c[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (b0 + j < bins) {
      c[j] = s.count[b0 + j];
      if (MASS) m[j] = (double)s.mass(b0 + j) * (zbins ? pow2(SampleMass::power(b0 + j) - 24) : scale);
    }
  double dm = m[0] + m[1];
  uint32_t dc = c[0] + c[1];
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t pc = __shfl_up_sync(0xffffffffu, dc, o);
    if (lane >= o) dc += pc;
    if (MASS) {
      const double pm = __shfl_up_sync(0xffffffffu, dm, o);
      if (lane >= o) dm += pm;
    }
  }
  if (lane == 31) s.warp_d[w] = dm, s.warp_a[w] = dc;
  if (t == 0) s.found_bin = -1;
  __syncthreads();
  double base_m = 0;
  uint32_t base_c = 0;
  for (int i = 0; i < w; ++i) base_m += s.warp_d[i], base_c += s.warp_a[i];
  const double from_m = base_m + dm - (m[0] + m[1]);
  const uint32_t from_c = base_c + dc - (c[0] + c[1]);
  double before_m = from_m;
  uint32_t before_c = from_c;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (c[j]) {
      const bool here = MASS ? before_m < want : before_c < want && before_c + c[j] >= want;
      if (here) atomicMax(&s.found_bin, b0 + j);
    }
    before_m += m[j], before_c += c[j];
  }
  __syncthreads();
  if (s.found_bin >= 0 && s.found_bin >> 1 == t) {
    const int j = s.found_bin & 1;
    s.found_mass = from_m + (j ? m[0] : 0.0);
    s.found_count = from_c + (j ? c[0] : 0u);
  }
  __syncthreads();
}

S1C_DEV void sample_clear(SampleShared& s, int bins) {
  for (int b = threadIdx.x; b < bins; b += SMP_THREADS) s.count[b] = 0, s.lo[b] = 0, s.hi[b] = 0;
}

S1C_DEV void sample_count(SampleShared& s, int b, uint32_t m) {
  atomicAdd(&s.count[b], 1u);
  atomicAdd(&s.lo[b], m & 4095u);
  atomicAdd(&s.hi[b], m >> 12);
}

// Narrows the cut inside bin `zbin` to one key. Of elements with key == limit.key only limit.need
// count, and none below it. want: the count or mass still to come inside the bin.
template <bool MASS, typename T>
S1C_DEV SampleCut sample_narrow(SampleShared& s, const SampleMass& f, const SampleItems<T>& items, int zbin, double want, SampleCut limit) {
  const int t = threadIdx.x;
  if (t == 0) s.key_lo = 0xffffffffu, s.key_hi = 0;
  __syncthreads();
  uint32_t lo = 0xffffffffu, hi = 0;
  for (int i = t; i < items.n; i += SMP_THREADS) {
    const float l = items(i);
    const uint32_t k = logit_key(l);
    if (f.bin(l) == zbin && k >= limit.key) lo = min(lo, k), hi = max(hi, k);
  }
  lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
  if (t % 32 == 0) atomicMin(&s.key_lo, lo), atomicMax(&s.key_hi, hi);
  __syncthreads();
  lo = s.key_lo, hi = s.key_hi;
  const double scale = pow2(SampleMass::power(zbin) - 24);
  for (;;) {
    const int shift = max(0, 32 - __clz(hi - lo) - 11);
    const int bins = (int)((hi - lo) >> shift) + 1;
    __syncthreads();
    sample_clear(s, bins);
    __syncthreads();
    for (int i = t; i < items.n; i += SMP_THREADS) {
      const float l = items(i);
      const uint32_t k = logit_key(l);
      if (k < lo || k > hi || k == limit.key) continue;
      if (f.bin(l) == zbin) {
        if (MASS)
          sample_count(s, (int)((hi - k) >> shift), f.mass(l, zbin));
        else
          atomicAdd(&s.count[(hi - k) >> shift], 1u);
      }
    }
    __syncthreads();
    if (t == 0 && limit.need && limit.key >= lo && limit.key <= hi) {
      const int b = (int)((hi - limit.key) >> shift);
      const unsigned long long all = (unsigned long long)f.mass(key_logit(limit.key), zbin) * limit.need;
      s.count[b] += limit.need, s.lo[b] += (uint32_t)(all & 4095u), s.hi[b] += (uint32_t)(all >> 12);
    }
    __syncthreads();
    sample_find<MASS>(s, bins, want, false, scale);
    const int b = s.found_bin;
    if (b < 0) return limit;  // every element is kept
    want -= MASS ? s.found_mass : (double)s.found_count;
    if (shift == 0) {
      const uint32_t key = hi - (uint32_t)b, equal = s.count[b];
      const double one = MASS ? f.mass(key_logit(key), zbin) * scale : 1.0;
      const double need = fmin((double)equal, fmax(1.0, ceil(want / one)));
      __syncthreads();
      return SampleCut{key, (uint32_t)need};
    }
    const uint32_t top = hi - ((uint32_t)b << shift);
    lo = max(lo, top - ((1u << shift) - 1));
    hi = top;
  }
}

// Sum over the block of an integer for each thread; all threads call.
S1C_DEV unsigned long long sample_sum(SampleShared& s, unsigned long long v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s.warp_u[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < SMP_WARPS; ++i) v += s.warp_u[i];
  return v;
}

// Step 3, by one block. total: the mass of all logits, where top-p applies without top-k.
template <typename T>
S1C_DEV void sample_choose(SampleShared& s, const SampleArgs& a, int r, const SampleMass& f, const SampleItems<T>& items, const int* index,
                           int k, float p, double least, unsigned long long total44) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
  SampleCut cut{0, 0};  // keys of finite logits are above 0: nothing is cut
  if (by_k || by_p) {
    sample_clear(s, SMP_ZBINS);
    __syncthreads();
    for (int i = t; i < items.n; i += SMP_THREADS) {
      const float l = items(i);
      const int b = f.bin(l);
      if (b < SMP_ZBINS) sample_count(s, b, f.mass(l, b));
    }
    __syncthreads();
    double total = (double)total44 * pow2(-44);  // mass of what top-k keeps
    int last = SMP_ZBINS;                        // bin of top-k's cut
    if (by_k) {
      sample_find<false>(s, SMP_ZBINS, (double)k, true, 0);
      if (s.found_bin >= 0) {
        last = s.found_bin;
        const double before = (double)s.found_count;
        cut = sample_narrow<false, T>(s, f, items, last, (double)k - before, cut);
        if (by_p) {
          // the histogram again, with the kept part of that bin alone
          unsigned long long part = 0;
          sample_clear(s, SMP_ZBINS);
          __syncthreads();
          for (int i = t; i < items.n; i += SMP_THREADS) {
            const float l = items(i);
            const int b = f.bin(l);
            if (b < last)
              sample_count(s, b, f.mass(l, b));
            else if (b == last && logit_key(l) > cut.key)
              part += f.mass(l, last);
          }
          part = sample_sum(s, part) + (unsigned long long)f.mass(key_logit(cut.key), last) * cut.need;
          if (t == 0) s.count[last] = 1, s.lo[last] = (uint32_t)(part & 4095u), s.hi[last] = (uint32_t)(part >> 12);
          __syncthreads();
        }
      }
      if (by_p) {
        const int bins = min(last + 1, SMP_ZBINS);
        double mine = 0;
        for (int j = 0; j < 2; ++j)
          if (2 * t + j < bins) mine += (double)s.mass(2 * t + j) * pow2(SampleMass::power(2 * t + j) - 24);
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0) s.warp_d[w] = mine;
        __syncthreads();
        total = 0;
        for (int i = 0; i < SMP_WARPS; ++i) total += s.warp_d[i];
        __syncthreads();
      }
    }
    if (by_p) {
      const double goal = (double)p * total;
      if (!(goal > 0.0)) {
        cut = SampleCut{logit_key(f.top), 1};
      } else {
        sample_find<true>(s, min(last + 1, SMP_ZBINS), goal, true, 0);
        const int b = s.found_bin;
        const double before = s.found_mass;
        cut = sample_narrow<true, T>(s, f, items, b, goal - before, b == last ? cut : SampleCut{0, 0});
      }
    }
  }

  // The kept mass of each warp's share of the elements, in order; equals of the cut are counted first.
  __syncthreads();
  const int share = (items.n + SMP_WARPS - 1) / SMP_WARPS, i0 = min(items.n, w * share), i1 = min(items.n, i0 + share);
  uint32_t ahead = 0;
  if (cut.need) {
    uint32_t equal = 0;
    for (int i = i0 + lane; i < i1; i += 32) equal += logit_key(items(i)) == cut.key;
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) s.warp_a[w] = equal;
    __syncthreads();
    for (int i = 0; i < w; ++i) ahead += s.warp_a[i];
  }
  const auto kept = [&](int i, uint32_t& rank, float& l, int& b) {
    l = i < i1 ? items(i) : -INFINITY;
    b = f.bin(l);
    const uint32_t key = logit_key(l);
    bool keep = i < i1 && b < SMP_ZBINS && (double)l >= least && key >= cut.key;
    if (cut.need) {
      const bool eq = i < i1 && key == cut.key;
      const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
      if (eq && rank + __popc(eqs & ((1u << lane) - 1)) >= cut.need) keep = false;
      rank += __popc(eqs);
    }
    return keep;
  };
  unsigned long long sum = 0, total = 0, base = 0;
  uint32_t rank = ahead;
  for (int j = i0; j < i1; j += 32) {
    float l;
    int b;
    if (kept(j + lane, rank, l, b)) sum += f.fixed(l, b);
  }
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s.warp_u[w] = sum;
  __syncthreads();
  for (int i = 0; i < SMP_WARPS; ++i) {
    if (i == w) base = total;
    total += s.warp_u[i];
  }
  const double goal = (double)a.uniform[r] * (double)total;
  // the warp that the goal falls into walks; past the end (u >= 1, or NaN) it is the last with mass
  int walker = -1;
  unsigned long long run = 0;
  for (int i = 0; i < SMP_WARPS; ++i) {
    if (!s.warp_u[i]) continue;
    walker = i;
    run += s.warp_u[i];
    if ((double)run > goal) break;
  }
  if (w != walker) return;
  rank = ahead;
  int token = -1;
  float prob = 0.f;
  for (int j = i0; j < i1; j += 32) {
    float l;
    int b;
    const bool keep = kept(j + lane, rank, l, b);
    const unsigned long long m = keep ? f.fixed(l, b) : 0ull;
    if (!__any_sync(0xffffffffu, m != 0)) continue;
    unsigned long long upto = m;
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t over = __ballot_sync(0xffffffffu, m && (double)(base + upto) > goal);
    const int pick = over ? __ffs(over) - 1 : 31 - __clz(__ballot_sync(0xffffffffu, m != 0));
    token = j + pick;
    prob = (float)((double)__shfl_sync(0xffffffffu, m, pick) / (double)total);
    if (over) break;
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) {
    a.token[r] = index ? index[token] : token;
    if (a.prob) a.prob[r] = prob;
  }
}

template <typename T>
__global__ void __launch_bounds__(SMP_THREADS) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(raw);
  T* part = reinterpret_cast<T*>(raw + (sizeof(SampleShared) + 15) / 16 * 16);
  auto cluster = cooperative_groups::this_cluster();
  const int blocks = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
  const int r = blockIdx.x / blocks, t = threadIdx.x, lane = t & 31, w = t >> 5;
  const T* row = static_cast<const T*>(a.logits) + r * a.stride;
  const int first = min(a.vocab, me * a.slice), n = min(a.vocab, first + a.slice) - first;
  const float T_ = a.temperature ? a.temperature[r] : 1.f;

  // 1. Largest logit and its first index; a NaN or +inf leaves no distribution.
  float top = -INFINITY;
  int at = a.vocab;
  bool bad = false;
  const auto look = [&](float l, int i) {
    bad |= !(l < INFINITY);
    if (l > top) top = l, at = i;
  };
  if (a.vec) {
    constexpr int E = 16 / sizeof(T);
    for (int i = t * E; i < n; i += SMP_THREADS * E) {
      if (i + E <= n) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + first + i));
        *reinterpret_cast<uint4*>(part + i) = v;
        const T* x = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int e = 0; e < E; ++e) look(to_f32(x[e]) + 0.f, first + i + e);
      } else {
        for (int e = i; e < n; ++e) part[e] = row[first + e], look(to_f32(part[e]) + 0.f, first + e);
      }
    }
  } else {
    for (int i = t; i < n; i += SMP_THREADS) part[i] = row[first + i], look(to_f32(part[i]) + 0.f, first + i);
  }
  for (int o = 16; o; o >>= 1) {
    const float l = __shfl_xor_sync(0xffffffffu, top, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    if (l > top || (l == top && i < at)) top = l, at = i;
  }
  if (lane == 0) s.warp_a[w] = __float_as_uint(top), s.warp_b[w] = (uint32_t)at;
  for (int b = t; b < SMP_ZBINS; b += SMP_THREADS) s.count[b] = 0;
  bad = __syncthreads_or(bad);
  const auto better = [&](float l, int j) {
    if (l > top || (l == top && j < at)) top = l, at = j;
  };
  for (int i = 0; i < SMP_WARPS; ++i) better(__uint_as_float(s.warp_a[i]), (int)s.warp_b[i]);
  if (blocks > 1) {
    if (t == 0) s.top = top, s.at = at, s.bad = bad;
    cluster.sync();
    for (int i = 0; i < blocks; ++i) {
      const SampleShared* o = cluster.map_shared_rank(&s, i);
      better(o->top, o->at), bad |= o->bad != 0;
    }
  }
  if (bad || top == -INFINITY || !(T_ > 0.f)) {
    if (t == 0 && me == 0) {
      const bool none = bad || top == -INFINITY;
      a.token[r] = none ? -1 : at;
      if (a.prob) a.prob[r] = none ? 0.f : 1.f;
    }
    if (blocks > 1) cluster.sync();  // nobody leaves while others read it
    return;
  }
  const SampleMass f(top, T_);
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f, mp = a.min_p ? a.min_p[r] : 0.f;
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f, by_m = mp > 0.f;
  // e >= min_p as a bound on the logit
  const double least = by_m ? (double)top + (double)T_ * log(fmin((double)mp, 1.0)) : -INFINITY;

  // 2. Counts of the bins, and a bin that ends before anything that is kept.
  unsigned long long total = 0;
  bool list = false;
  uint32_t listed = 0, before = 0, mine = 0;
  int bound = SMP_ZBINS - 1;
  if (by_k || by_p || by_m) {
    const bool sums = by_p && !by_k;
    for (int i = t; i < n; i += SMP_THREADS) {
      const float l = to_f32(part[i]) + 0.f;
      const int b = f.bin(l);
      if (b < SMP_ZBINS) {
        atomicAdd(&s.count[b], 1u);
        if (sums) total += f.fixed(l, b);
      }
    }
    if (sums) total = sample_sum(s, total);
    __syncthreads();
    uint32_t own[2] = {0, 0}, all[2] = {0, 0};  // counts of this thread's two bins
    for (int j = 0; j < 2; ++j)
      if (2 * t + j < SMP_ZBINS) all[j] = own[j] = s.count[2 * t + j];
    if (blocks > 1) {
      if (t == 0) s.sum = total;
      cluster.sync();
      total = 0;
      all[0] = all[1] = 0;
      for (int i = 0; i < blocks; ++i) {
        const SampleShared* o = cluster.map_shared_rank(&s, i);
        total += o->sum;
        for (int j = 0; j < 2; ++j)
          if (2 * t + j < SMP_ZBINS) all[j] += o->count[2 * t + j];
      }
    }
    // running counts, and the least mass they can have: a bin's every e is above 2^(-(bin + 1) / 32)
    float low[2];
    for (int j = 0; j < 2; ++j) low[j] = (float)all[j] * exp2f(-(2 * t + j + 1) * 0.03125f);
    uint32_t c = all[0] + all[1];
    float m = low[0] + low[1];
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t pc = __shfl_up_sync(0xffffffffu, c, o);
      const float pm = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o) c += pc, m += pm;
    }
    __syncthreads();
    if (lane == 31) s.warp_a[w] = c, s.warp_d[w] = m;
    if (t == 0) s.found_bin = SMP_ZBINS - 1;
    __syncthreads();
    for (int i = 0; i < w; ++i) c += s.warp_a[i], m += (float)s.warp_d[i];
    if (by_k || by_p) {
      const double goal = (double)p * (double)total * pow2(-44) * 1.00001;  // beyond the rounding of `low`
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t upto_c = j ? c : c - all[1];
        const float upto_m = j ? m : m - low[1];
        if (2 * t + j < SMP_ZBINS && (by_k ? upto_c >= (uint32_t)k : upto_m >= goal)) {
          atomicMin(&s.found_bin, 2 * t + j);
          break;
        }
      }
      __syncthreads();
      bound = s.found_bin;
    }
    // what min-p drops is not listed, unless top-p needs the mass of all that top-k keeps
    if (by_m && !(by_k && by_p)) bound = min(bound, (int)fmin(-log2(fmin((double)mp, 1.0)) * 32.0, (double)SMP_ZBINS) + 1);
    unsigned long long both = 0;  // listed elements: of all blocks, of this one
    for (int j = 0; j < 2; ++j)
      if (2 * t + j <= bound) both += ((unsigned long long)all[j] << 32) + own[j];
    both = sample_sum(s, both);
    listed = (uint32_t)(both >> 32), mine = (uint32_t)both;
    list = listed <= SMP_LIST;
    if (blocks > 1 && list) {
      if (t == 0) s.listed = mine;
      cluster.sync();
      for (int i = 0; i < me; ++i) before += cluster.map_shared_rank(&s, i)->listed;
    }
  }

  // 3. The list, in order, in the first block; each warp has a run of the indexes.
  if (list) {
    SampleShared* to = blocks > 1 ? cluster.map_shared_rank(&s, 0) : &s;
    const int share = ((n + SMP_WARPS - 1) / SMP_WARPS + 31) / 32 * 32, i0 = min(n, w * share), i1 = min(n, i0 + share);
    uint32_t c = 0;
    for (int i = i0 + lane; i < i1; i += 32) c += f.bin(to_f32(part[i]) + 0.f) <= bound;
    c = __reduce_add_sync(0xffffffffu, c);
    __syncthreads();
    if (lane == 0) s.warp_a[w] = c;
    __syncthreads();
    uint32_t at_ = before;
    for (int i = 0; i < w; ++i) at_ += s.warp_a[i];
    if (c)
      for (int j = i0; j < i1; j += 32) {
        const int i = j + lane;
        const float l = i < i1 ? to_f32(part[i]) + 0.f : -INFINITY;
        const bool in = i < i1 && f.bin(l) <= bound;
        const uint32_t ins = __ballot_sync(0xffffffffu, in);
        if (in) {
          const uint32_t slot = at_ + __popc(ins & ((1u << lane) - 1));
          to->value[slot] = l, to->index[slot] = first + i;
        }
        at_ += __popc(ins);
      }
  }
  if (blocks > 1) cluster.sync();
  if (me) return;
  __syncthreads();
  if (list)
    sample_choose<T>(s, a, r, f, SampleItems<T>{s.value, nullptr, (int)listed}, s.index, k, p, least, total);
  else
    sample_choose<T>(s, a, r, f, SampleItems<T>{nullptr, blocks > 1 ? row : part, a.vocab}, nullptr, k, p, least, total);
}

}  // namespace s1c
