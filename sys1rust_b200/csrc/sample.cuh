// One token for each row of logits under temperature, top-k, top-p and min-p.
//
// With z_i = (l_i - max l) / T and e_i = exp(z_i), tokens ordered by descending logit (the lowest index first
// among equals): top-k keeps the first k; top-p keeps, of these, the first and every one whose
// predecessors' mass is below p times the mass of the k; min-p keeps those with e_i >= min_p. The
// token is the first index, in ascending order, at which the kept mass summed so far exceeds u times the kept mass.
//
// No sort is needed: both filters cut the order at one value, so each is a threshold (a logit, and how
// many of its equals are kept, by index). It is found by histograms: first over bins of z,
// 1/32 of a power of two wide, then, inside the bin that holds the cut, over the order-preserving integer of the logit, 2048 ways at a
// time, until one value is left.
//
// Masses are integers: e = m * 2^(n - 30), m an integer of 31 bits, and all e in one bin share n. So their sums are exact and do not depend
// on the order of atomics. Logits more than 45 powers of two below the largest have no mass.
#pragma once
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
};

constexpr int SMP_THREADS = 1024, SMP_BINS = 2048, SMP_ZBINS = 45 * 32;

// The order-preserving integer of a logit: a > b as floats exactly if it is so for the keys.
S1C_DEV uint32_t logit_key(float l) {
  const uint32_t u = __float_as_uint(l);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
S1C_DEV float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

S1C_DEV double pow2(int e) { return __hiloint2double((1023 + e) << 20, 0); }

// exp as an integer: the bin of z and m with e = m * 2^(n - 30), n from the bin. z in double (the
// difference of two logits over T has to keep its low bits), 2^f - 1 by the Taylor series of exp(f ln 2),
// |f| <= 1/2: its tenth term is below 1e-10, and rounding to fp32 leaves about 3e-8.
struct SampleMass {
  double top, rate;  // max l, log2(e) / T
  S1C_DEV int bin(float l) const {
    const double t = (top - (double)l) * rate;
    return t < 45.0 ? (int)(t * 32.0) : SMP_ZBINS;  // also of NaN (0 * inf): no mass
  }
  static S1C_DEV int power(int bin) { return -((bin + 16) >> 5); }
  S1C_DEV uint32_t mass(float l, int bin) const {
    const float f = (float)(((double)l - top) * rate - power(bin)) * 0.69314718055994531f;
    float g = 2.7557319e-6f;
    g = fmaf(g, f, 2.4801587e-5f);
    g = fmaf(g, f, 1.9841270e-4f);
    g = fmaf(g, f, 1.3888889e-3f);
    g = fmaf(g, f, 8.3333333e-3f);
    g = fmaf(g, f, 4.1666667e-2f);
    g = fmaf(g, f, 0.16666667f);
    g = fmaf(g, f, 0.5f);
    g = fmaf(g, f, 1.0f);
    return (1u << 30) + __float2int_rn(g * f * 0x1p30f);
  }
  // the same as a fixed-point number of 44 places, for sums over bins
  S1C_DEV unsigned long long fixed(float l) const {
    const int b = bin(l);
    return b == SMP_ZBINS ? 0ull : ((unsigned long long)mass(l, b) << 14) >> -power(b);
  }
};

struct SampleShared {
  uint32_t count[SMP_BINS];
  unsigned long long mass[SMP_BINS];
  double warp_d[32];
  unsigned long long warp_u[32];
  uint32_t warp_a[32], warp_b[32];
  uint32_t key_lo, key_hi;
  int found_bin;
  uint32_t found_count;
  double found_mass;
  int token;
  float prob;
};

// What is kept: keys above `key`, and the first `need` of those equal to it.
struct SampleCut {
  uint32_t key, need;
};

template <typename T>
S1C_DEV float sample_logit(const T* row, int i) {
  return to_f32(row[i]) + 0.f;  // -0 becomes 0: they are equal
}

// First bin whose elements reach `want` (by count), or last non-empty bin whose predecessors' mass is
// below `want` (by mass): found_bin, and the count and mass before it. `power` >= 0: one power for all bins is given
// by the caller as `scale`, else the bins are bins of z. -1 where there is none. All threads call.
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
      if (MASS) m[j] = (double)s.mass[b0 + j] * (zbins ? pow2(SampleMass::power(b0 + j) - 30) : scale);
    }
  double dm = m[0] + m[1];
  uint32_t dc = c[0] + c[1];
  for (int o = 1; o < 32; o <<= 1) {
    const double pm = __shfl_up_sync(0xffffffffu, dm, o);
    const uint32_t pc = __shfl_up_sync(0xffffffffu, dc, o);
    if (lane >= o) dm += pm, dc += pc;
  }
  if (lane == 31) s.warp_d[w] = dm, s.warp_a[w] = dc;
  if (t == 0) s.found_bin = -1;
  __syncthreads();
  double base_m = 0;
  uint32_t base_c = 0;
  for (int i = 0; i < w; ++i) base_m += s.warp_d[i], base_c += s.warp_a[i];
  double before_m = base_m + dm - (m[0] + m[1]);
  uint32_t before_c = base_c + dc - (c[0] + c[1]);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (c[j]) {
      const bool here = MASS ? before_m < want : before_c < want && before_c + c[j] >= want;
      if (here) atomicMax(&s.found_bin, b0 + j);
    }
    before_m += m[j], before_c += c[j];
  }
  __syncthreads();
  before_m = base_m + dm - (m[0] + m[1]), before_c = base_c + dc - (c[0] + c[1]);
  if (s.found_bin >> 1 == t && s.found_bin >= 0) {
    const int j = s.found_bin & 1;
    s.found_mass = before_m + (j ? m[0] : 0.0);
    s.found_count = before_c + (j ? c[0] : 0u);
  }
  __syncthreads();
}

S1C_DEV void sample_clear(SampleShared& s, int bins) {
  for (int b = threadIdx.x; b < bins; b += SMP_THREADS) s.count[b] = 0, s.mass[b] = 0;
}

S1C_DEV void sample_count(SampleShared& s, int b, unsigned long long m, uint32_t times) {
  atomicAdd(&s.count[b], times);
  atomicAdd(&s.mass[b], m * times);
}

// Narrows the cut inside bin `zbin` to one key. Of elements with key == limit.key only limit.need
// count, and none below it. want: the count or mass still to come inside the bin.
template <bool MASS, typename T>
S1C_DEV SampleCut sample_narrow(SampleShared& s, const SampleMass& f, const T* row, int vocab, int zbin, double want, SampleCut limit) {
  const int t = threadIdx.x;
  if (t == 0) s.key_lo = 0xffffffffu, s.key_hi = 0;
  __syncthreads();
  uint32_t lo = 0xffffffffu, hi = 0;
  for (int i = t; i < vocab; i += SMP_THREADS) {
    const float l = sample_logit(row, i);
    const uint32_t k = logit_key(l);
    if (f.bin(l) == zbin && k >= limit.key) lo = min(lo, k), hi = max(hi, k);
  }
  atomicMin(&s.key_lo, lo);
  atomicMax(&s.key_hi, hi);
  __syncthreads();
  lo = s.key_lo, hi = s.key_hi;
  const double scale = pow2(SampleMass::power(zbin) - 30);
  for (;;) {
    const int shift = max(0, 32 - __clz(hi - lo) - 11);
    const int bins = (int)((hi - lo) >> shift) + 1;
    __syncthreads();
    sample_clear(s, bins);
    __syncthreads();
    for (int i = t; i < vocab; i += SMP_THREADS) {
      const float l = sample_logit(row, i);
      const uint32_t k = logit_key(l);
      if (k < lo || k > hi || k == limit.key) continue;
      if (f.bin(l) == zbin) sample_count(s, (int)((hi - k) >> shift), f.mass(l, zbin), 1);
    }
    if (t == 0 && limit.need && limit.key >= lo && limit.key <= hi) {
      sample_count(s, (int)((hi - limit.key) >> shift), f.mass(key_logit(limit.key), zbin), limit.need);
    }
    __syncthreads();
    sample_find<MASS>(s, bins, want, false, scale);
    const int b = s.found_bin;
    if (b < 0) return limit;  // every element is kept
    const double before = MASS ? s.found_mass : (double)s.found_count;
    want -= before;
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

template <typename T>
__global__ void __launch_bounds__(SMP_THREADS) sample_kernel(const SampleArgs a) {
  __shared__ SampleShared s;
  const int r = blockIdx.x, t = threadIdx.x, lane = t & 31, w = t >> 5;
  const T* row = static_cast<const T*>(a.logits) + r * a.stride;
  const float T_ = a.temperature ? a.temperature[r] : 1.f;

  // largest logit and its first index; a NaN or +inf leaves no distribution
  float top = -INFINITY;
  int at = a.vocab;
  bool bad = false;
  for (int i = t; i < a.vocab; i += SMP_THREADS) {
    const float l = sample_logit(row, i);
    bad |= !(l < INFINITY);
    if (l > top) top = l, at = i;
  }
  for (int o = 16; o; o >>= 1) {
    const float l = __shfl_xor_sync(0xffffffffu, top, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    if (l > top || (l == top && i < at)) top = l, at = i;
  }
  bad = __syncthreads_or(bad);
  if (lane == 0) s.warp_a[w] = __float_as_uint(top), s.warp_b[w] = (uint32_t)at;
  __syncthreads();
  for (int i = 0; i < 32; ++i) {
    const float l = __uint_as_float(s.warp_a[i]);
    const int j = (int)s.warp_b[i];
    if (l > top || (l == top && j < at)) top = l, at = j;
  }
  if (bad || top == -INFINITY || !(T_ > 0.f)) {
    if (t == 0) {
      const bool none = bad || top == -INFINITY;
      a.token[r] = none ? -1 : at;
      if (a.prob) a.prob[r] = none ? 0.f : 1.f;
    }
    return;
  }
  const SampleMass f{(double)top, 1.4426950408889634 / (double)T_};
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f;
  const float mp = a.min_p ? a.min_p[r] : 0.f;
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
  // e >= min_p as a bound on the logit
  const double least = mp > 0.f ? (double)top + (double)T_ * log(fmin((double)mp, 1.0)) : -INFINITY;

  SampleCut cut{0, 0};  // keys of finite logits are above 0: nothing is cut
  if (by_k || by_p) {
    sample_clear(s, SMP_ZBINS);
    __syncthreads();
    for (int i = t; i < a.vocab; i += SMP_THREADS) {
      const float l = sample_logit(row, i);
      const int b = f.bin(l);
      if (b < SMP_ZBINS) sample_count(s, b, f.mass(l, b), 1);
    }
    __syncthreads();
    double total = 0;  // mass of what top-k keeps
    int last = SMP_ZBINS;  // bin of top-k's cut
    if (by_k) {
      sample_find<false>(s, SMP_ZBINS, (double)k, true, 0);
      last = s.found_bin;
      if (last < 0) last = SMP_ZBINS;
      if (last < SMP_ZBINS) {
        const double before = (double)s.found_count;
        cut = sample_narrow<false, T>(s, f, row, a.vocab, last, (double)k - before, cut);
        // the kept part of that bin
        unsigned long long part = 0;
        for (int i = t; i < a.vocab; i += SMP_THREADS) {
          const float l = sample_logit(row, i);
          if (logit_key(l) > cut.key && f.bin(l) == last) part += f.mass(l, last);
        }
        for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        if (lane == 0) s.warp_u[w] = part;
        __syncthreads();
        part = 0;
        for (int i = 0; i < 32; ++i) part += s.warp_u[i];
        part += (unsigned long long)f.mass(key_logit(cut.key), last) * cut.need;
        __syncthreads();
        if (by_p) {  // the histogram again: narrowing took its place
          sample_clear(s, SMP_ZBINS);
          __syncthreads();
          for (int i = t; i < a.vocab; i += SMP_THREADS) {
            const float l = sample_logit(row, i);
            const int b = f.bin(l);
            if (b < last) sample_count(s, b, f.mass(l, b), 1);
          }
          if (t == 0) {
            s.count[last] = 1;  // stands for the part of the bin that is kept
            s.mass[last] = part;
          }
          __syncthreads();
        }
      }
    }
    if (by_p) {
      const int bins = min(last + 1, SMP_ZBINS);
      double mine = 0;
      for (int j = 0; j < 2; ++j)
        if (2 * t + j < bins)
          mine += (double)s.mass[2 * t + j] * pow2(SampleMass::power(2 * t + j) - 30);
      for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
      if (lane == 0) s.warp_d[w] = mine;
      __syncthreads();
      for (int i = 0; i < 32; ++i) total += s.warp_d[i];
      __syncthreads();
      const double goal = (double)p * total;
      if (!(goal > 0.0)) {
        cut = SampleCut{logit_key(top), 1};
      } else {
        sample_find<true>(s, bins, goal, true, 0);
        const int b = s.found_bin;
        const double before = s.found_mass;
        cut = sample_narrow<true, T>(s, f, row, a.vocab, b, goal - before, b == last ? cut : SampleCut{0, 0});
      }
    }
  }

  // The kept mass of each warp's share of the indexes, in order; equals of the cut are counted first.
  __syncthreads();
  const int share = (a.vocab + 31) / 32, i0 = min(a.vocab, w * share), i1 = min(a.vocab, i0 + share);
  uint32_t equal = 0;
  for (int i = i0 + lane; i < i1; i += 32) equal += logit_key(sample_logit(row, i)) == cut.key;
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) s.warp_a[w] = equal;
  __syncthreads();
  uint32_t ahead = 0;
  for (int i = 0; i < w; ++i) ahead += s.warp_a[i];
  const double u = (double)a.uniform[r];
  unsigned long long sum = 0, total = 0, base = 0;
  for (int pass = 0; pass < 2; ++pass) {
    if (pass) {
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) s.warp_u[w] = sum;
      if (t == 0) s.token = -1;
      __syncthreads();
      for (int i = 0; i < 32; ++i) {
        if (i == w) base = total;
        total += s.warp_u[i];
      }
    }
    const double goal = u * (double)total;
    // the warp that the goal falls into walks; past the end (u >= 1, or NaN) it is the last with mass
    if (pass) {
      int walker = -1;
      unsigned long long run = 0;
      for (int i = 0; i < 32; ++i) {
        if (!s.warp_u[i]) continue;
        walker = i;
        run += s.warp_u[i];
        if ((double)run > goal) break;
      }
      if (w != walker) break;
    }
    uint32_t rank = ahead;
    int token = -1;
    float prob = 0.f;
    for (int j = i0; j < i1; j += 32) {
      const int i = j + lane;
      const float l = i < i1 ? sample_logit(row, i) : -INFINITY;
      const uint32_t key = logit_key(l);
      const bool eq = i < i1 && key == cut.key;
      const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
      const bool keep = i < i1 && l > -INFINITY && (double)l >= least && (key > cut.key || (eq && rank + __popc(eqs & ((1u << lane) - 1)) < cut.need));
      rank += __popc(eqs);
      const unsigned long long m = keep ? f.fixed(l) : 0ull;
      if (!pass) {
        sum += m;
        continue;
      }
      unsigned long long run = m;
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += v;
      }
      const uint32_t over = __ballot_sync(0xffffffffu, m && (double)(base + run) > goal);
      const uint32_t any = __ballot_sync(0xffffffffu, m != 0);
      const int pick = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : -1;
      if (pick >= 0) {
        token = j + pick;
        prob = (float)((double)__shfl_sync(0xffffffffu, m, pick) / (double)total);
      }
      if (over) break;
      base += __shfl_sync(0xffffffffu, run, 31);
    }
    if (pass && lane == 0) {
      a.token[r] = token;
      if (a.prob) a.prob[r] = prob;
    }
  }
}

}  // namespace s1c
