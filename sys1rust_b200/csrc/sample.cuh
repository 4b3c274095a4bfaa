// One token for each row of logits under temperature, top-k, top-p and min-p.
//
// With z_i = (max l - l_i) / T and e_i = exp(-z_i), tokens ordered by descending logit (the lowest index
// first among equals): top-k keeps the first k; top-p keeps, of these, the first and every one whose
// predecessors' mass is below p times the mass of the k; min-p keeps those with e_i >= min_p. The token is
// the first index, in ascending order, at which the kept mass summed so far exceeds u times the kept mass.
//
// No sort is needed: both filters cut the order at one value, so each is a threshold (a logit, and how
// many of its equals are kept, by index). A cluster of blocks shares a row:
//
//  1. each block finds the largest logit of its part (which it reads again, from the cache, in each step: two
//     blocks on an SM, whose waits overlap, are worth more than a copy in shared memory);
//  2. the counts of the logits in bins of z, 1/32 of a power of two wide, and where top-p needs it the exact
//     mass of all, give a bin below which nothing can be kept;
//  3. what stands above is gathered in the order of the indexes in the first block. Up to 512 of them are
//     sorted, one by each thread. More have their thresholds found by histograms over bins of z and, inside
//     the bin that holds the cut, over the order-preserving integer of the logit, 2048 ways at a time, until
//     one value is left. What is kept is summed and walked. More than fit in the list are worked on in place.
//
// Masses are integers: e = m * 2^(n - 24), m an integer of 25 bits, and all e in one bin share n. So their
// sums are exact and depend neither on the order of atomics nor on how a row is shared. One sum is rounded:
// where top-p counts the mass of a whole row, what lies below 1/16 of the largest, or below min-p, enters as
// fp32 sums of the four or eight neighbours that a load brings, and these as integers. They do not depend on
// how a row is shared either, so a row gets the same token in every batch. Logits more than 45 powers of two
// below the largest have no mass.
//
// Measured: 1 x 50368 fp32, top-k 50 and top-p: 17.1 us, of which the exchanges of the eight blocks are
// about half; 256 x 50368 bf16, top-p and min-p: 48.5 us for three to four passes over each row (25 M warp
// instructions, issue slots 56 % used, the rest waits for loads and at barriers, with 27 of 64 warps an SM). Without a
// list (64 x 131072, no filter) 124 us. Not kept: a row in shared memory and
// one block of 1024 threads an SM (65 us for the 256 rows).
#pragma once
#include <cooperative_groups.h>

#include "mma.cuh"

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

constexpr int SMP_THREADS = 512, SMP_WARPS = SMP_THREADS / 32, SMP_BINS = 2048, SMP_ZBINS = 45 * 32, SMP_LIST = 4096;
constexpr int SMP_PER = SMP_BINS / SMP_THREADS, SMP_CLUSTER = 8;

// The order-preserving integer of a logit: a > b as floats exactly if it is so for the keys.
S1C_DEV uint32_t logit_key(float l) {
  const uint32_t u = __float_as_uint(l);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
S1C_DEV float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

S1C_DEV double pow2(int e) { return __hiloint2double((1023 + e) << 20, 0); }

// exp as an integer: the bin of z and m with e = m * 2^(n - 24), n from the bin. The bin comes from the
// rounded product (it only has to be monotonic); the mass adds what the difference and the product lost.
// 2^f by the Taylor series of exp(f ln 2), |f| <= 0.52: its tenth term is below 1e-10, and rounding to fp32
// leaves about 5e-8.
struct SampleMass {
  float top, rate, rate_lo;  // max l, log2(e) / T in two parts
  S1C_DEV SampleMass(float top_, float T) : top(top_) {
    const double r = fmin(1.4426950408889634 / (double)T, 1e38);
    rate = (float)r, rate_lo = (float)(r - (double)rate);
  }
  S1C_DEV float z(float l) const { return (top - l) * rate; }
  // 32 z to the nearest integer, by the place that adding 2^23 gives it
  static S1C_DEV int bin_of(float z) { return z < 44.5f ? __float_as_int(fmaf(z, 32.f, 8388608.f)) & 0xfff : SMP_ZBINS; }
  S1C_DEV int bin(float l) const { return bin_of(z(l)); }
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

struct alignas(16) SampleShared {
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
  int at;
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

// f(element) for all elements, each thread with every 512th, four loads in flight.
template <typename T, typename F>
S1C_DEV void sample_each(const SampleItems<T>& items, F&& f) {
  for (int i0 = threadIdx.x; i0 < items.n; i0 += 4 * SMP_THREADS) {
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = i0 + j * SMP_THREADS < items.n ? items(i0 + j * SMP_THREADS) : -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (x[j] > -INFINITY) f(x[j]);
  }
}

// First bin whose elements reach `want` (by count), or last non-empty bin whose predecessors' mass is
// below `want` (by mass), and the count and mass before it; -1 where there is none. A mass counts 2^power
// of its bin of z, or `scale`. All threads call.
template <bool MASS>
S1C_DEV void sample_find(SampleShared& s, int bins, double want, bool zbins, double scale) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int b0 = SMP_PER * t;
  double m[SMP_PER], dm = 0;
  uint32_t c[SMP_PER], dc = 0;
#pragma unroll
  for (int j = 0; j < SMP_PER; ++j) {
    const bool in = b0 + j < bins;
    c[j] = in ? s.count[b0 + j] : 0u;
    m[j] = MASS && in ? (double)s.mass(b0 + j) * (zbins ? pow2(SampleMass::power(b0 + j) - 24) : scale) : 0.0;
    dm += m[j], dc += c[j];
  }
  const double sum_m = dm;
  const uint32_t sum_c = dc;
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
  if (w == 0) {
    uint32_t c0 = lane < SMP_WARPS ? s.warp_a[lane] : 0u;
    double m0 = lane < SMP_WARPS ? s.warp_d[lane] : 0.0;
    const uint32_t c1 = c0;
    const double m1 = m0;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t pc = __shfl_up_sync(0xffffffffu, c0, o);
      if (lane >= o) c0 += pc;
      if (MASS) {
        const double pm = __shfl_up_sync(0xffffffffu, m0, o);
        if (lane >= o) m0 += pm;
      }
    }
    if (lane < SMP_WARPS) s.warp_a[lane] = c0 - c1, s.warp_d[lane] = m0 - m1;
  }
  __syncthreads();
  const double base_m = s.warp_d[w];
  const uint32_t base_c = s.warp_a[w];
  double before_m = base_m + dm - sum_m;
  uint32_t before_c = base_c + dc - sum_c;
  int here = -1;  // the last of this thread's bins that qualifies, and what is before it
  double here_m = 0;
  uint32_t here_c = 0;
#pragma unroll
  for (int j = 0; j < SMP_PER; ++j) {
    if (c[j] && (MASS ? before_m < want : before_c < want && before_c + c[j] >= want)) here = b0 + j, here_m = before_m, here_c = before_c;
    before_m += m[j], before_c += c[j];
  }
  if (here >= 0) atomicMax(&s.found_bin, here);
  __syncthreads();
  if (here >= 0 && s.found_bin == here) s.found_mass = here_m, s.found_count = here_c;
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
  sample_each(items, [&](float l) {
    const uint32_t k = logit_key(l);
    if (f.bin(l) == zbin && k >= limit.key) lo = min(lo, k), hi = max(hi, k);
  });
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
    sample_each(items, [&](float l) {
      const uint32_t k = logit_key(l);
      if (k < lo || k > hi || k == limit.key || f.bin(l) != zbin) return;
      if (MASS)
        sample_count(s, (int)((hi - k) >> shift), f.mass(l, zbin));
      else
        atomicAdd(&s.count[(hi - k) >> shift], 1u);
    });
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
  v = threadIdx.x % 32 < SMP_WARPS ? s.warp_u[threadIdx.x % 32] : 0ull;
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum of v over the threads up to this one; all threads call.
S1C_DEV unsigned long long sample_scan(SampleShared& s, unsigned long long v, unsigned long long& all) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) s.warp_u[w] = v;
  __syncthreads();
  const unsigned long long own = lane < SMP_WARPS ? s.warp_u[lane] : 0ull;
  unsigned long long sum = own;
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += u;
  }
  all = __shfl_sync(0xffffffffu, sum, 31);
  return v + __shfl_sync(0xffffffffu, sum - own, w);
}

// Step 3 for a list of up to 512, by one block: a bitonic sort of (key, place) with an element for each
// thread, then ranks and masses are at hand.
S1C_DEV void sample_choose_sorted(SampleShared& s, const SampleArgs& a, int r, const SampleMass& f, int n, int k, float p, double least,
                                  unsigned long long total) {
  const int t = threadIdx.x;
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
  unsigned long long* masses = reinterpret_cast<unsigned long long*>(s.count);  // [512]
  unsigned long long* other = reinterpret_cast<unsigned long long*>(s.lo);      // [512]
  unsigned long long v = 0;  // past the list: last in the order
  if (t < n) v = ((unsigned long long)logit_key(s.value[t]) << 32) | (uint32_t)~t;
  int width = 32;  // threads that sort: a power of two
  while (width < n) width *= 2;
  const int names = width / 32;  // warps; they meet at a barrier of their own
  if (t < width)
    for (int size = 2; size <= width; size <<= 1)
      for (int step = size / 2; step; step >>= 1) {
        unsigned long long u;
        if (step >= 32) {
          asm volatile("bar.sync 1, %0;" ::"r"(names * 32) : "memory");
          other[t] = v;
          asm volatile("bar.sync 1, %0;" ::"r"(names * 32) : "memory");
          u = other[t ^ step];
        } else {
          u = __shfl_xor_sync(0xffffffffu, v, step);
        }
        const bool larger = !(t & step) == !(t & size);  // descending runs first
        if (larger ? u > v : u < v) v = u;
      }
  // thread t now has the element of rank t
  const int place = (int)~(uint32_t)v;
  const float l = key_logit((uint32_t)(v >> 32));
  const int b = t < n ? f.bin(l) : SMP_ZBINS;
  const unsigned long long mass = b < SMP_ZBINS ? f.fixed(l, b) : 0ull;
  bool keep = mass && (double)l >= least && !(by_k && t >= k);
  if (by_p) {
    unsigned long long all;
    const unsigned long long ahead = sample_scan(s, by_k && t >= k ? 0ull : mass, all) - mass;
    if (by_k) total = all;  // mass of what top-k keeps
    if (t && !((double)ahead < (double)p * (double)total)) keep = false;
  }
  if (t < n) masses[place] = keep ? mass : 0ull;
  if (t == 0) s.found_bin = n, s.key_hi = 0;
  __syncthreads();
  const unsigned long long mine = t < n ? masses[t] : 0ull;
  unsigned long long whole;
  const unsigned long long upto = sample_scan(s, mine, whole);
  const double goal = (double)a.uniform[r] * (double)whole;
  const uint32_t over = __ballot_sync(0xffffffffu, mine && (double)upto > goal), any = __ballot_sync(0xffffffffu, mine != 0);
  if (!(t & 31)) {
    if (over) atomicMin(&s.found_bin, t + __ffs(over) - 1);
    if (any) atomicMax(&s.key_hi, (uint32_t)(t + 31 - __clz(any)));  // the last one: for u >= 1 or NaN
  }
  __syncthreads();
  const int pick = s.found_bin < n ? s.found_bin : (int)s.key_hi;
  if (t == pick) {
    a.token[r] = s.index[pick];
    if (a.prob) a.prob[r] = (float)((double)mine / (double)whole);
  }
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
    sample_each(items, [&](float l) {
      const int b = f.bin(l);
      if (b < SMP_ZBINS) sample_count(s, b, f.mass(l, b));
    });
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
          sample_each(items, [&](float l) {
            const int b = f.bin(l);
            if (b < last)
              sample_count(s, b, f.mass(l, b));
            else if (b == last && logit_key(l) > cut.key)
              part += f.mass(l, last);
          });
          part = sample_sum(s, part) + (unsigned long long)f.mass(key_logit(cut.key), last) * cut.need;
          if (t == 0) s.count[last] = 1, s.lo[last] = (uint32_t)(part & 4095u), s.hi[last] = (uint32_t)(part >> 12);
          __syncthreads();
        }
      }
      if (by_p) {
        const int bins = min(last + 1, SMP_ZBINS);
        double mine = 0;
        for (int j = SMP_PER * t; j < min(bins, SMP_PER * (t + 1)); ++j) mine += (double)s.mass(j) * pow2(SampleMass::power(j) - 24);
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
  // Masses of the kept ones of 128 elements from j on, four steps of 32 (their loads in flight together);
  // rank: equals of the cut so far.
  const auto masses = [&](int j, uint32_t& rank, unsigned long long (&m)[4]) {
    float x[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = j + q * 32 + lane < i1 ? items(j + q * 32 + lane) : -INFINITY;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      m[q] = 0;
      if (j + q * 32 >= i1) continue;
      const int b = f.bin(x[q]);
      const uint32_t key = logit_key(x[q]);
      bool keep = b < SMP_ZBINS && key >= cut.key && (least == -INFINITY || (double)x[q] >= least);
      if (cut.need) {
        const bool eq = key == cut.key;
        const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
        if (eq && rank + __popc(eqs & ((1u << lane) - 1)) >= cut.need) keep = false;
        rank += __popc(eqs);
      }
      m[q] = keep ? f.fixed(x[q], b) : 0ull;
    }
  };
  unsigned long long sum = 0, total = 0, base = 0, m[4];
  uint32_t rank = ahead;
  for (int j = i0; j < i1; j += 128) {
    masses(j, rank, m);
#pragma unroll
    for (int q = 0; q < 4; ++q) sum += m[q];
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
  // the 128 elements that it falls into, or the last ones with mass
  int at = i0;
  uint32_t at_rank = ahead;
  unsigned long long at_base = base;
  rank = ahead;
  for (int j = i0; j < i1; j += 128) {
    const uint32_t before = rank;
    masses(j, rank, m);
    sum = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) sum += m[q];
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!sum) continue;
    at = j, at_rank = before, at_base = base;
    base += sum;
    if ((double)base > goal) break;
  }
  masses(at, at_rank, m);
  int token = -1;
  float prob = 0.f;
  bool found = false;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (at + q * 32 >= i1) continue;
    unsigned long long upto = m[q];
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t any = __ballot_sync(0xffffffffu, m[q] != 0), over = __ballot_sync(0xffffffffu, m[q] && (double)(at_base + upto) > goal);
    if (any && !found) {
      const int pick = over ? __ffs(over) - 1 : 31 - __clz(any);
      token = at + q * 32 + pick;
      prob = (float)((double)__shfl_sync(0xffffffffu, m[q], pick) / (double)total);
      found = over != 0;
    }
    at_base += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) {
    a.token[r] = index ? index[token] : token;
    if (a.prob) a.prob[r] = prob;
  }
}

template <typename T>
__global__ void __launch_bounds__(SMP_THREADS, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(raw);
  pdl_trigger();
  pdl_wait();
  auto cluster = cooperative_groups::this_cluster();
  const int blocks = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
  const int r = blockIdx.x / blocks, t = threadIdx.x, lane = t & 31, w = t >> 5;
  const T* row = static_cast<const T*>(a.logits) + r * a.stride;
  const int first = min(a.vocab, me * a.slice), n = min(a.vocab, first + a.slice) - first;
  const float T_ = a.temperature ? a.temperature[r] : 1.f;

  // E logits of the part from the i-th on, -inf past its end
  constexpr int E = 16 / sizeof(T);
  const T* part = row + first;
  const auto load = [&](float (&x)[E], int i) {
    if (a.vec && i + E <= n) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(part + i));
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = to_f32(reinterpret_cast<const T*>(&v)[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = i + e < n ? to_f32(part[i + e]) : -INFINITY;
    }
  };

  // another block's shared memory, for eight lanes at a time (repeating the last block's where there are fewer)
  const auto of_block = [&](int i) { return cluster.map_shared_rank(&s, min(i % SMP_CLUSTER, blocks - 1)); };

  // 1. The largest logit; a NaN (which the maximum keeps) or +inf leaves no distribution.
  float top = -INFINITY;
#pragma unroll 4
  for (int i = t * E; i < n; i += SMP_THREADS * E) {
    float x[E];
    load(x, i);
#pragma unroll
    for (int e = 0; e < E; ++e) top = max_nan(top, x[e]);
  }
  for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s.warp_a[w] = __float_as_uint(top);
  for (int b = t; b < SMP_ZBINS; b += SMP_THREADS) s.count[b] = 0;
  __syncthreads();
  top = __uint_as_float(s.warp_a[lane % SMP_WARPS]);
  for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (blocks > 1) {
    if (t == 0) s.top = top;
    cluster.sync();
    top = of_block(lane)->top;  // each lane asks one block
    for (int o = 4; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  top += 0.f;  // -0 and 0 are equal
  const bool none = !(top < INFINITY) || top == -INFINITY;
  if (none || !(T_ > 0.f)) {
    // the first index of the largest
    int at = a.vocab;
    if (!none)
      for (int i = t; i < n; i += SMP_THREADS)
        if (to_f32(part[i]) == top) at = min(at, first + i);
    at = __reduce_min_sync(0xffffffffu, at);
    __syncthreads();
    if (lane == 0) s.warp_b[w] = (uint32_t)at;
    __syncthreads();
    at = (int)__reduce_min_sync(0xffffffffu, s.warp_b[lane % SMP_WARPS]);
    if (blocks > 1) {
      if (t == 0) s.at = at;
      cluster.sync();
      if (me == 0)
        at = (int)__reduce_min_sync(0xffffffffu, (uint32_t)of_block(lane)->at);
      cluster.sync();  // nobody leaves while others read it
    }
    if (t == 0 && me == 0) {
      a.token[r] = none ? -1 : at;
      if (a.prob) a.prob[r] = none ? 0.f : 1.f;
    }
    return;
  }
  const SampleMass f(top, T_);
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f, mp = a.min_p ? a.min_p[r] : 0.f;
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f, by_m = mp > 0.f;
  // e >= min_p as a bound on the logit; an infinite T makes all e 1
  const double least = by_m && T_ < INFINITY ? (double)top + (double)T_ * log(fmin((double)mp, 1.0)) : -INFINITY;

  // 2. Counts of the bins, and a bin that ends before anything that is kept.
  unsigned long long total = 0;
  bool list = false;
  uint32_t listed = 0, before = 0, mine = 0;
  int bound = SMP_ZBINS - 1;
  if (by_k || by_p || by_m) {
    const bool sums = by_p && !by_k;
    // what min-p drops is not counted, unless top-p needs the mass of all that top-k keeps
    if (by_m && !(by_k && by_p)) bound = min(bound, (int)fmin(-log2(fmin((double)mp, 1.0)) * 32.0, (double)SMP_ZBINS) + 1);
    const float reach = (bound + 1) * 0.03125f;
#pragma unroll 2
    for (int i = t * E; i < n; i += SMP_THREADS * E) {
      float x[E], small = 0.f;  // by the hardware's exp2: errors of 2^-22 of masses that are small or that min-p drops
      load(x, i);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float z = f.z(x[e]);
        if (z < reach) {
          const int b = SampleMass::bin_of(z);
          if (b <= bound) atomicAdd(&s.count[b], 1u);
          if (sums && z < 4.f) total += f.fixed(x[e], b);
        }
        if (sums && !(z < fminf(4.f, reach))) small += exp2_approx(-fminf(z, 200.f));
      }
      if (sums) total += (unsigned long long)(small * 0x1p44f);
    }
    if (sums) total = sample_sum(s, total);
    __syncthreads();
    // the counts of this thread's bins, in this block and in all
    constexpr int PER = (SMP_ZBINS + SMP_THREADS * 4 - 1) / (SMP_THREADS * 4) * 4;
    static_assert(PER == 4, "one vector of counts for each thread");
    const bool have = PER * t < SMP_ZBINS;
    uint4 own4 = have ? *reinterpret_cast<const uint4*>(&s.count[PER * t]) : make_uint4(0, 0, 0, 0), all4 = own4;
    if (blocks > 1) {
      if (t == 0) s.sum = total;
      cluster.sync();
      total = sums && lane < blocks ? of_block(lane)->sum : 0ull;
      all4 = make_uint4(0, 0, 0, 0);
      if (__any_sync(0xffffffffu, have)) {
        uint4 counts[SMP_CLUSTER];
#pragma unroll
        for (int i = 0; i < SMP_CLUSTER; ++i)  // all in flight together
          counts[i] = have && i < blocks ? *reinterpret_cast<const uint4*>(&of_block(i)->count[PER * t]) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < SMP_CLUSTER; ++i) all4.x += counts[i].x, all4.y += counts[i].y, all4.z += counts[i].z, all4.w += counts[i].w;
      }
      for (int o = 4; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      total = __shfl_sync(0xffffffffu, total, 0);
    }
    const uint32_t own[PER] = {own4.x, own4.y, own4.z, own4.w}, all[PER] = {all4.x, all4.y, all4.z, all4.w};
    if (by_k || by_p) {
      // running counts, and the least mass they can have: a bin's every e is above 2^(-(bin + 1) / 32)
      float low[PER], m = 0.f;
      uint32_t c = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) low[j] = (float)all[j] * exp2_approx(-(PER * t + j + 1) * 0.03125f), c += all[j], m += low[j];
      const uint32_t c1 = c;
      const float m1 = m;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t pc = __shfl_up_sync(0xffffffffu, c, o);
        const float pm = __shfl_up_sync(0xffffffffu, m, o);
        if (lane >= o) c += pc, m += pm;
      }
      __syncthreads();
      if (lane == 31) s.warp_a[w] = c, s.warp_b[w] = __float_as_uint(m);
      if (t == 0) s.found_bin = SMP_ZBINS - 1;
      __syncthreads();
      uint32_t c0 = lane < w ? s.warp_a[lane] : 0u;
      float m0 = lane < w ? __uint_as_float(s.warp_b[lane]) : 0.f;
      for (int o = 16; o; o >>= 1) c0 += __shfl_xor_sync(0xffffffffu, c0, o), m0 += __shfl_xor_sync(0xffffffffu, m0, o);
      c += c0 - c1, m += m0 - m1;  // before this thread's bins
      const double goal = (double)p * (double)total * pow2(-44) * 1.00001;  // beyond the rounding of `low`
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        c += all[j], m += low[j];
        if (have && (by_k ? c >= (uint32_t)k : m >= goal)) {
          atomicMin(&s.found_bin, PER * t + j);
          break;
        }
      }
      __syncthreads();
      bound = min(bound, s.found_bin);
    }
    unsigned long long both = 0;  // listed elements: of all blocks, of this one
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (PER * t + j <= bound) both += ((unsigned long long)all[j] << 32) + own[j];
    both = sample_sum(s, both);
    listed = (uint32_t)(both >> 32), mine = (uint32_t)both;
    list = listed <= SMP_LIST;
    if (blocks > 1 && list) {
      if (t == 0) s.listed = mine;
      cluster.sync();
      before = __reduce_add_sync(0xffffffffu, lane < me ? of_block(lane)->listed : 0u);
    }
  }

  // 3. The list, in order, in the first block; each warp has a run of the indexes.
  if (list) {
    SampleShared* to = blocks > 1 ? cluster.map_shared_rank(&s, 0) : &s;
    // the smallest key that is listed, 32 ways at a time: bins only grow as keys fall
    if (w == 0) {
      uint32_t low = 0, size = logit_key(top);  // low + size is listed
      while (size) {
        const uint32_t step = size / 32 + 1, probe = (uint32_t)min((unsigned long long)size, (unsigned long long)step * lane);
        const uint32_t in = __ballot_sync(0xffffffffu, f.bin(key_logit(low + probe)) <= bound);
        const uint32_t j = in ? __ffs(in) - 1 : 32;  // the first probe that is listed
        const unsigned long long from = j ? (unsigned long long)step * (j - 1) + 1 : 0, upto = j < 32 ? (unsigned long long)step * j : size;
        low += (uint32_t)from, size = j ? (uint32_t)(min(upto, (unsigned long long)size) - from) : 0;
      }
      if (lane == 0) s.key_lo = low;
    }
    __syncthreads();
    const float least_in = key_logit(s.key_lo);
    const int share = ((n + SMP_WARPS - 1) / SMP_WARPS + E - 1) / E * E, i0 = min(n, w * share), i1 = min(n, i0 + share);
    uint32_t c = 0;
#pragma unroll 2
    for (int i = i0 + lane * E; i < i1; i += 32 * E) {
      float x[E];
      load(x, i);
#pragma unroll
      for (int e = 0; e < E; ++e) c += x[e] >= least_in;
    }
    c = __reduce_add_sync(0xffffffffu, c);
    __syncthreads();
    if (lane == 0) s.warp_a[w] = c;
    __syncthreads();
    uint32_t slot = before + __reduce_add_sync(0xffffffffu, lane < w ? s.warp_a[lane] : 0u);
    if (c)
#pragma unroll 2
      for (int j = i0; j < i1; j += 32 * E) {
        const int i = j + lane * E;
        float x[E];
        uint32_t in = 0;
        if (i < i1) {
          load(x, i);
#pragma unroll
          for (int e = 0; e < E; ++e) in |= (uint32_t)(x[e] >= least_in) << e;
        }
        if (!__any_sync(0xffffffffu, in)) continue;
        uint32_t upto = __popc(in);
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += u;
        }
        uint32_t at = slot + upto - __popc(in);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (in >> e & 1) to->value[at] = x[e] + 0.f, to->index[at] = first + i + e, ++at;
        slot += __shfl_sync(0xffffffffu, upto, 31);
      }
  }
  if (blocks > 1) cluster.sync();
  if (me) return;
  __syncthreads();
  if (list && listed <= SMP_THREADS)
    sample_choose_sorted(s, a, r, f, (int)listed, k, p, least, total);
  else if (list)
    sample_choose<T>(s, a, r, f, SampleItems<T>{s.value, nullptr, (int)listed}, s.index, k, p, least, total);
  else
    sample_choose<T>(s, a, r, f, SampleItems<T>{nullptr, row, a.vocab}, nullptr, k, p, least, total);
}

}  // namespace s1c
