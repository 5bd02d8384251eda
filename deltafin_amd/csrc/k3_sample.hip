// Token sampling (include/k3_hip_sample_abi.h) by selection instead of sorting.
//
// Every limit of a row (top-k, top-p, min-p) and the draw itself is a position in one
// order of its tokens.  A position is found in two steps: in a histogram of token counts
// and weight sums over 2048 equal ranges of the logit, from the row's largest down to
// where weights vanish (or its smallest), the range in which the count or the sum crosses
// the wanted one; then, among that range's tokens, by their keys eight bits at a time, and
// by index among equal ones.  Nothing is sorted or written back.
//
// Weights are 64-bit integers (see fixed_weight): sums of them are exact, so LDS and
// global atomics may add in any order, and workgroups' histograms join without one.
//
// Launches: the rows' largest and smallest logits, the histogram (both over many
// workgroups per row), and one workgroup per row for the positions.  That one reads its
// row once more: it gathers the tokens from the top through the first range it needs, up
// to kList of them, in LDS, and most often every position lies among them.  A range that
// does not fit (thousands of near-equal logits) is walked in memory instead.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/k3_hip_sample_abi.h"
#include "k3_device.h"
#include "k3_internal.h"
#include "k3_launch.h"

namespace k3 {
namespace {

constexpr int kBins = 2048;          // of the first histogram
constexpr int kList = 12288;         // tokens that the last workgroup holds: 96 KB of its LDS
constexpr int kScanThreads = 256;    // of the passes over a row's parts
constexpr int kPickThreads = 1024;   // of the workgroup that ends a row
constexpr double kVanish = 64.0;     // weights under 2^-kVanish round to none

struct SampleArgs {
  const void* logits;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
  uint32_t* ends;      // [rows][parts][2] keys of the parts' largest and smallest logits
  uint32_t* count;     // [rows][kBins]
  uint64_t* mass;      // [rows][kBins]
  int rows, vocab, parts, part;  // parts of a row and tokens of one
  int shift;           // weight 1 is 2^shift
};

// Descending order of the logits as ascending keys; the two zeros share a key and NaN
// takes that of -inf.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (l != l) l = -INFINITY;
  if (l == 0.f) l = 0.f;
  const uint32_t u = __float_as_uint(l);
  return (u & 0x80000000u) ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key : ~key & 0x7fffffffu);
}
constexpr uint32_t kKeyMasked = 0xff800000u;  // of -inf

struct RowParams {
  float top;       // largest logit
  double rate;     // log2(e) / T; 0 where only the largest logits weigh
  double per_bin;  // bins per halving of the weight
  bool sampled;    // T > 0
};

__device__ __forceinline__ double log2_weight(const RowParams& r, float l);

// bottom_key: of the smallest logit over -inf.
__device__ __forceinline__ RowParams row_params(const SampleArgs& a, int row, uint32_t top_key,
                                                uint32_t bottom_key) {
  RowParams r;
  r.top = value_of(top_key);
  const float t = a.temperature ? a.temperature[row] : 1.f;
  r.sampled = t > 0.f;
  r.rate = r.sampled ? 1.4426950408889634 / (double)t : 0.0;
  const double range = -log2_weight(r, value_of(bottom_key));
  r.per_bin = range > 0.0 ? (double)(kBins - 2) / fmin(range, kVanish) : 0.0;
  return r;
}

// log2 of the weight of logit l, l <= top: 0 for the largest, -inf for what has none.
__device__ __forceinline__ double log2_weight(const RowParams& r, float l) {
  if (l == r.top) return 0.0;
  if (l == -INFINITY || r.top == INFINITY || !r.sampled) return -INFINITY;
  return ((double)l - (double)r.top) * r.rate;
}

// The bin of a token of log2 weight y: it never falls as y does; the last one holds what
// weighs nothing.
__device__ __forceinline__ int bin_of(const RowParams& r, double y) {
  return y > -kVanish ? min((int)(-y * r.per_bin), kBins - 2) : kBins - 1;
}

// 2^y times 2^shift, to the nearest integer: y = n + h / 64 + f with |f| <= 1 / 128,
// 2^(h / 64) from LDS and 2^f by its Taylor series (the first term left out is under 2^-52).
__device__ __forceinline__ uint64_t fixed_weight(const double* table, int shift, double y) {
  if (!(y > -kVanish)) return 0;
  const double q = rint(y * 64.0);
  const double f = (y - q * 0.015625) * 0.6931471805599453;  // times ln 2
  const int qi = (int)q;
  double e = 1.0 + f * (1.0 + f * (0.5 + f * (1.0 / 6 + f * (1.0 / 24 + f * (1.0 / 120)))));
  e *= table[qi & 63];
  return (uint64_t)rint(ldexp(e, (qi >> 6) + shift));
}

__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x * 0.015625);
}

// Calls f(logit, index) for the tokens [t0, t1) of a row, each thread of the workgroup its
// share: 16 bytes per load where they lie inside, single tokens at ragged ends.
template <typename T, typename F>
__device__ __forceinline__ void scan(const T* row, int t0, int t1, int threads, F f) {
  constexpr int kPer = 16 / (int)sizeof(T);
  constexpr int kUnroll = 4;
  const T* p = row + t0;
  const int n = t1 - t0;
  const int lead = (int)(((uintptr_t)p & 15u) / sizeof(T));  // tokens of the first chunk before p
  const int chunks = (lead + n + kPer - 1) / kPer;
  const u32x4* base = reinterpret_cast<const u32x4*>(p - lead);
  auto value = [](u32x4 v, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(v[i]);
    return __uint_as_float(i % 2 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16);
  };
  for (int c0 = threadIdx.x; c0 < chunks; c0 += kUnroll * threads) {
    u32x4 v[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int c = c0 + k * threads;
      const bool whole = c * kPer >= lead && (c + 1) * kPer <= lead + n;
      if (whole) v[k] = base[c];
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int c = c0 + k * threads;
      const bool whole = c * kPer >= lead && (c + 1) * kPer <= lead + n;
      if (whole) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) f(value(v[k], i), t0 + c * kPer + i - lead);
      } else if (c < chunks) {
        for (int i = 0; i < kPer; ++i) {
          const int t = c * kPer + i - lead;
          if (t < 0 || t >= n) continue;
          float l;
          if constexpr (sizeof(T) == 4)
            l = p[t];
          else
            l = bf16_bits_to_f32(p[t]);
          f(l, t0 + t);
        }
      }
    }
  }
}

__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = min(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}

// The keys of a row's largest logit and of its smallest over -inf (0 where there is none),
// from every thread's own; red is shared, 2 words per wave.
__device__ __forceinline__ void block_ends(uint32_t* red, int waves, uint32_t* top,
                                           uint32_t* bottom) {
  const uint32_t t = wave_min(*top), b = ~wave_min(~*bottom);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[2 * (threadIdx.x >> 6)] = t;
    red[2 * (threadIdx.x >> 6) + 1] = b;
  }
  __syncthreads();
  *top = red[0];
  *bottom = red[1];
  for (int w = 1; w < waves; ++w) {
    *top = min(*top, red[2 * w]);
    *bottom = max(*bottom, red[2 * w + 1]);
  }
}

__device__ __forceinline__ void row_ends(const SampleArgs& a, int row, uint32_t* red, int threads,
                                         uint32_t* top, uint32_t* bottom) {
  *top = 0xffffffffu;
  *bottom = 0u;
  for (int i = threadIdx.x; i < a.parts; i += threads) {
    const uint32_t* e = a.ends + 2 * ((uint64_t)row * a.parts + i);
    *top = min(*top, e[0]);
    *bottom = max(*bottom, e[1]);
  }
  block_ends(red, threads / 64, top, bottom);
}

template <typename T>
__global__ __launch_bounds__(kScanThreads) void k_sample_ends(const SampleArgs a) {
  const int row = blockIdx.y, part = blockIdx.x;
  float most = -INFINITY, least = INFINITY;  // fmaxf and fminf pass NaN by
  const int t0 = part * a.part, t1 = min(t0 + a.part, a.vocab);
  scan(static_cast<const T*>(a.logits) + (uint64_t)row * a.vocab, t0, t1, kScanThreads,
       [&](float l, int) {
         most = fmaxf(most, l);
         least = fminf(least, l == -INFINITY ? INFINITY : l);
       });
  uint32_t top = key_of(most), bottom = most > -INFINITY ? key_of(least) : 0u;
  __shared__ uint32_t red[2 * kScanThreads / 64];
  block_ends(red, kScanThreads / 64, &top, &bottom);
  if (threadIdx.x == 0) {
    uint32_t* e = a.ends + 2 * ((uint64_t)row * a.parts + part);
    e[0] = top;
    e[1] = bottom;
  }
  // this part's share of the row's histogram, for the next launch to add to
  for (int b = part * kScanThreads + threadIdx.x; b < kBins; b += a.parts * kScanThreads) {
    a.count[(uint64_t)row * kBins + b] = 0;
    a.mass[(uint64_t)row * kBins + b] = 0;
  }
}

template <typename T>
__global__ __launch_bounds__(kScanThreads) void k_sample_histogram(const SampleArgs a) {
  const int row = blockIdx.y, part = blockIdx.x;
  __shared__ uint32_t count[kBins];
  __shared__ uint64_t mass[kBins];
  __shared__ double table[64];
  __shared__ uint32_t red[2 * kScanThreads / 64];
  fill_table(table);
  for (int b = threadIdx.x; b < kBins; b += kScanThreads) {
    count[b] = 0;
    mass[b] = 0;
  }
  uint32_t top, bottom;
  row_ends(a, row, red, kScanThreads, &top, &bottom);
  const RowParams r = row_params(a, row, top, bottom);
  if (top == kKeyMasked || !r.sampled) return;  // the last launch needs no histogram
  __syncthreads();
  const int t0 = part * a.part, t1 = min(t0 + a.part, a.vocab);
  scan(static_cast<const T*>(a.logits) + (uint64_t)row * a.vocab, t0, t1, kScanThreads,
       [&](float l, int) {
         if (l != l) l = -INFINITY;
         const double y = log2_weight(r, l);
         const int b = bin_of(r, y);
         atomicAdd(&count[b], 1u);
         const uint64_t w = fixed_weight(table, a.shift, y);
         if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&mass[b]), (unsigned long long)w);
       });
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kScanThreads) {
    if (count[b] == 0) continue;
    atomicAdd(&a.count[(uint64_t)row * kBins + b], count[b]);
    if (mass[b])
      atomicAdd(reinterpret_cast<unsigned long long*>(&a.mass[(uint64_t)row * kBins + b]),
                (unsigned long long)mass[b]);
  }
}

struct PickShared {
  uint32_t count[kBins];  // running counts and masses, each bin's own included
  uint64_t mass[kBins];
  double table[64];
  uint32_t digit_count[256];
  uint64_t digit_mass[256];
  uint32_t key[kList];
  int32_t index[kList];
  uint32_t listed;
  uint32_t wave_count[kPickThreads / 64];
  uint64_t wave_mass[kPickThreads / 64];
  uint32_t red[2 * kPickThreads / 64];
  int bin;
  uint32_t digit, before;
  uint64_t mass_before;
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  return (uint64_t)__shfl_up((unsigned long long)v, d);
}
__device__ __forceinline__ void add64(uint64_t* to, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(to), (unsigned long long)v);
}

// A position in a row's order: the key of its token and what lies before that key.
struct Found {
  uint32_t key;
  uint32_t before;       // tokens of smaller keys
  uint64_t mass_before;  // and their weight
};

// One row's workgroup.  Every member is called by all of its threads.
template <typename T>
struct Picker {
  PickShared& sh;
  const SampleArgs& a;
  const T* row;
  RowParams r;
  int first = 0, last = -1;  // bins whose tokens are listed

  // The last key of the bins up to `bin`: bins never fall along the keys.  64 keys at a
  // time; with the two ends of a bin known, tokens are told by their keys alone, without
  // the fp64 of bin_of (which took half of a pass over the row).
  __device__ __forceinline__ uint32_t last_key(int bin) const {
    if (bin < 0) return key_of(r.top) - 1;
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = key_of(r.top), hi = kKeyMasked;  // lo is in, hi is not
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo - 1) / 64 + 1;
      const uint32_t at = lo + (lane + 1) * step;
      const bool in = at < hi && at > lo && bin_of(r, log2_weight(r, value_of(at))) <= bin;
      const uint32_t n = (uint32_t)__popcll(__ballot(in));
      const uint32_t next = lo + (n + 1) * step;
      lo += n * step;
      if (n < 64 && next > lo && next < hi) hi = next;
    }
    return lo;
  }

  // The histogram, as running sums.
  __device__ __forceinline__ void load_histogram(int row_index) {
    const int b = 2 * threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t* gc = a.count + (uint64_t)row_index * kBins;
    const uint64_t* gm = a.mass + (uint64_t)row_index * kBins;
    const uint32_t c0 = gc[b], c1 = gc[b + 1];
    const uint64_t m0 = gm[b], m1 = gm[b + 1];
    uint32_t c = c0 + c1;
    uint64_t m = m0 + m1;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t cu = __shfl_up(c, d);
      const uint64_t mu = shfl_up64(m, d);
      if (lane >= d) {
        c += cu;
        m += mu;
      }
    }
    if (lane == 63) {
      sh.wave_count[wave] = c;
      sh.wave_mass[wave] = m;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      c += sh.wave_count[w];
      m += sh.wave_mass[w];
    }
    sh.count[b] = c - c1;
    sh.count[b + 1] = c;
    sh.mass[b] = m - m1;
    sh.mass[b + 1] = m;
    __syncthreads();
  }

  // The first bin whose running count or mass exceeds target; there is one.
  __device__ __forceinline__ int crossing(bool by_count, uint64_t target) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int b = 2 * threadIdx.x + i;
      const uint64_t here = by_count ? sh.count[b] : sh.mass[b];
      const uint64_t ahead = b == 0 ? 0 : by_count ? sh.count[b - 1] : sh.mass[b - 1];
      if (ahead <= target && here > target) sh.bin = b;
    }
    __syncthreads();
    return sh.bin;
  }

  __device__ __forceinline__ uint32_t count_before(int bin) const {
    return bin ? sh.count[bin - 1] : 0u;
  }
  __device__ __forceinline__ uint64_t mass_before(int bin) const {
    return bin ? sh.mass[bin - 1] : 0u;
  }

  // Lists the tokens of the bin (keys up to `to`), with those of every larger logit where
  // they fit.
  __device__ __forceinline__ void list(int bin, uint32_t from, uint32_t to) {
    if (first <= bin && bin <= last) return;
    const int b0 = sh.count[bin] <= (uint32_t)kList ? 0 : bin;
    if (sh.count[bin] - count_before(b0) > (uint32_t)kList) return;  // stays in memory
    if (b0 == 0) from = 0;
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    const float most = value_of(max(from, key_of(r.top))), least = value_of(to);
    scan(row, 0, a.vocab, kPickThreads, [&](float l, int t) {
      if (!(l <= most && l >= least)) return;
      const uint32_t at = atomicAdd(&sh.listed, 1u);
      if (at >= (uint32_t)kList) return;  // the row changed under the call
      sh.key[at] = key_of(l);
      sh.index[at] = t;
    });
    __syncthreads();
    first = b0;
    last = bin;
  }

  // Calls f(key, index) for the bin's tokens, of keys from..to, each thread its share.
  template <typename F>
  __device__ __forceinline__ void each(int bin, uint32_t from, uint32_t to, F f) {
    if (first <= bin && bin <= last) {
      const int n = min((int)sh.listed, kList);
      for (int i = threadIdx.x; i < n; i += kPickThreads) {
        const uint32_t k = sh.key[i];
        if (k >= from && k <= to) f(k, sh.index[i]);
      }
    } else {
      // (the order of the values is that of their keys; NaN is in no range)
      const float most = value_of(from), least = value_of(to);
      scan(row, 0, a.vocab, kPickThreads, [&](float l, int t) {
        if (l <= most && l >= least) f(key_of(l), t);
      });
    }
  }

  // Of the 256 digits, the first at which the running count or mass (what lies before the
  // digits included) exceeds target: into sh.digit, sh.before and sh.mass_before.
  __device__ __forceinline__ void cross_digit(bool by_count, uint64_t target, uint32_t before,
                                              uint64_t mass) {
    __syncthreads();
    if (threadIdx.x < 64) {
      uint32_t c[4];
      uint64_t m[4];
      uint32_t cs = 0;
      uint64_t ms = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = sh.digit_count[4 * threadIdx.x + i];
        m[i] = sh.digit_mass[4 * threadIdx.x + i];
        cs += c[i];
        ms += m[i];
      }
      uint32_t ci = cs;
      uint64_t mi = ms;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t cu = __shfl_up(ci, d);
        const uint64_t mu = shfl_up64(mi, d);
        if ((int)threadIdx.x >= d) {
          ci += cu;
          mi += mu;
        }
      }
      uint32_t cr = before + ci - cs;
      uint64_t mr = mass + mi - ms;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t ahead = by_count ? cr : mr;
        const uint64_t here = by_count ? (uint64_t)(cr + c[i]) : mr + m[i];
        if (ahead <= target && here > target) {
          sh.digit = 4 * threadIdx.x + i;
          sh.before = cr;
          sh.mass_before = mr;
        }
        cr += c[i];
        mr += m[i];
      }
    }
    __syncthreads();
  }

  __device__ __forceinline__ void clear_digits() {
    __syncthreads();
    if (threadIdx.x < 256) {
      sh.digit_count[threadIdx.x] = 0;
      sh.digit_mass[threadIdx.x] = 0;
    }
    __syncthreads();
  }

  // The bits in which the values that `walk` shows differ, from the highest differing one
  // down; their common part goes to *common.
  template <typename W>
  __device__ __forceinline__ int differing_bits(W walk, uint32_t* common) {
    uint32_t lo = 0xffffffffu, hi = 0u;
    walk([&](uint32_t v) {
      lo = min(lo, v);
      hi = max(hi, v);
    });
    block_ends(sh.red, kPickThreads / 64, &lo, &hi);
    const uint32_t x = lo ^ hi;
    const int bits = x ? 32 - __clz((int)x) : 0;
    *common = bits == 32 ? 0u : lo >> bits << bits;
    return bits;
  }

  // The value, among those that `walk` shows (keys, if weighed), at which the running
  // count or mass exceeds target; before and mass lie ahead of all of them.
  template <typename W>
  __device__ __forceinline__ Found descend(W walk, bool by_count, bool weigh, uint64_t target,
                                           uint32_t before, uint64_t mass) {
    Found f;
    int low = differing_bits(walk, &f.key);
    f.before = before;
    f.mass_before = mass;
    while (low > 0) {
      const int width = min(low, 8);
      const int high = low;
      low -= width;
      clear_digits();
      const uint32_t prefix = high == 32 ? 0u : f.key >> high;
      walk([&](uint32_t v) {
        if (high < 32 && v >> high != prefix) return;
        const uint32_t d = (v >> low) & ((1u << width) - 1u);
        atomicAdd(&sh.digit_count[d], 1u);
        const uint64_t w = weigh ? weight(v) : 0;
        if (w) add64(&sh.digit_mass[d], w);
      });
      cross_digit(by_count, target, f.before, f.mass_before);
      f.key |= sh.digit << low;
      f.before = sh.before;
      f.mass_before = sh.mass_before;
    }
    return f;
  }

  // The first token at which the row's running count or mass exceeds target.
  __device__ __forceinline__ Found find(bool by_count, uint64_t target, int* bin_out) {
    const int bin = crossing(by_count, target);
    *bin_out = bin;
    const uint32_t from = last_key(bin - 1) + 1, to = last_key(bin);
    list(bin, from, to);
    return descend(
        [&](auto f) { each(bin, from, to, [&](uint32_t k, int) { f(k); }); }, by_count, true,
        target, count_before(bin), mass_before(bin));
  }

  // The index of rank nth (from 0) among the bin's tokens of a key.
  __device__ __forceinline__ int nth_equal(int bin, uint32_t key, uint32_t nth) {
    return (int)descend(
               [&](auto f) { each(bin, key, key, [&](uint32_t, int t) { f((uint32_t)t); }); },
               true, false, nth, 0u, 0u)
        .key;
  }

  __device__ __forceinline__ uint64_t weight(uint32_t key) const {
    return fixed_weight(sh.table, a.shift, log2_weight(r, value_of(key)));
  }

  __device__ __forceinline__ uint64_t block_sum(uint64_t m) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m += (uint64_t)__shfl_xor((unsigned long long)m, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave_mass[threadIdx.x >> 6] = m;
    __syncthreads();
    m = 0;
    for (int w = 0; w < kPickThreads / 64; ++w) m += sh.wave_mass[w];
    return m;
  }
};

template <typename T>
__global__ __launch_bounds__(kPickThreads) void k_sample_pick(const SampleArgs a) {
  __shared__ PickShared sh;
  const int ri = blockIdx.x;
  const T* row = static_cast<const T*>(a.logits) + (uint64_t)ri * a.vocab;
  uint32_t top, bottom;
  row_ends(a, ri, sh.red, kPickThreads, &top, &bottom);
  if (top == kKeyMasked) {  // nothing but -inf and NaN
    if (threadIdx.x == 0) a.tokens[ri] = -1;
    return;
  }
  const RowParams r = row_params(a, ri, top, bottom);
  if (!r.sampled) {  // the lowest index of the largest logit
    int at = a.vocab;
    scan(row, 0, a.vocab, kPickThreads, [&](float l, int t) {
      if (l == r.top) at = min(at, t);
    });
    uint32_t lo = (uint32_t)at, hi = 0u;
    block_ends(sh.red, kPickThreads / 64, &lo, &hi);
    if (threadIdx.x == 0) a.tokens[ri] = (int)lo;
    return;
  }
  fill_table(sh.table);
  Picker<T> p{sh, a, row, r};
  p.load_histogram(ri);
  int bin;
  uint64_t kept = sh.mass[kBins - 1];  // weight of the shortest prefix so far
  const int k = a.top_k ? a.top_k[ri] : 0;
  // (a first k that ends among the tokens of no weight leaves the sum as it is)
  if (k > 0 && k < a.vocab && (uint32_t)k <= sh.count[kBins - 2]) {
    const Found f = p.find(true, (uint64_t)(k - 1), &bin);
    kept = f.mass_before + (uint64_t)((uint32_t)k - f.before) * p.weight(f.key);
  }
  const float top_p = a.top_p ? a.top_p[ri] : 1.f;
  if (top_p < 1.f) {
    // the first prefix with a sum of at least top_p times the top-k one's
    const uint64_t want =
        max((uint64_t)1, (uint64_t)ceil(fmax((double)top_p, 0.0) * (double)kept));
    const Found f = p.find(false, want - 1, &bin);
    const uint64_t w = p.weight(f.key);
    kept = min(kept, f.mass_before + (want - f.mass_before + w - 1) / w * w);
  }
  const float min_p = a.min_p ? a.min_p[ri] : 0.f;
  if (min_p > 0.f) {
    const double least = log2(fmin((double)min_p, 1.0));
    bin = bin_of(r, least);
    uint64_t m = 0;
    if (p.mass_before(bin) < kept) {  // else a shorter prefix is there already
      const uint32_t from = p.last_key(bin - 1) + 1, to = p.last_key(bin);
      p.list(bin, from, to);
      p.each(bin, from, to, [&](uint32_t key, int) {
        const double y = log2_weight(r, value_of(key));
        if (y >= least) m += fixed_weight(sh.table, a.shift, y);
      });
      kept = min(kept, p.mass_before(bin) + p.block_sum(m));
    }
  }
  float u = a.u[ri];
  if (!(u < 1.f)) u = 1.f - 0x1p-24f;
  u = fmaxf(u, 0.f);
  const uint64_t target = min((uint64_t)((double)u * (double)kept), kept - 1);
  const Found f = p.find(false, target, &bin);
  const uint32_t nth = (uint32_t)((target - f.mass_before) / p.weight(f.key));
  const int t = p.nth_equal(bin, f.key, nth);
  if (threadIdx.x == 0) a.tokens[ri] = t;
}

uint64_t align256(uint64_t v) { return (v + 255) & ~255ull; }

struct SampleLayout {
  int parts, part;
  uint64_t count, mass, bytes;  // offsets of the histograms behind the parts' ends
  SampleLayout(int rows, int vocab) {
    // parts of at least 4096 tokens, about two workgroups per CU over all rows
    const int want = std::max(1, 512 / rows);
    parts = std::min(want, (vocab + 4095) / 4096);
    part = (vocab + parts - 1) / parts;
    parts = (vocab + part - 1) / part;
    count = align256(8ull * rows * parts);
    mass = count + align256(4ull * rows * kBins);
    bytes = mass + align256(8ull * rows * kBins);
  }
};

int sample_check(const K3HipSampleV1* op, bool sizes) {
  if (!op) return spine_fail(K3_SPINE_E_INVALID, "sample: null descriptor");
  if (op->abi_version != K3_SAMPLE_ABI_V1 || op->struct_bytes != sizeof(*op) || op->reserved != 0)
    return spine_fail(K3_SPINE_E_INVALID,
                      "sample: descriptor version %u, size %u or reserved field is not this ABI's",
                      op->abi_version, op->struct_bytes);
  if (op->logits_dtype != K3_DTYPE_F32 && op->logits_dtype != K3_DTYPE_BF16)
    return spine_fail(K3_SPINE_E_INVALID, "sample: logits are neither fp32 nor BF16");
  if (op->rows == 0 || op->rows > K3_SAMPLE_MAX_ROWS || op->vocabulary == 0 ||
      op->vocabulary > K3_SAMPLE_MAX_VOCABULARY)
    return spine_fail(K3_SPINE_E_INVALID,
                      "sample: rows (%u) must be 1..%u and the vocabulary (%u) 1..%u", op->rows,
                      K3_SAMPLE_MAX_ROWS, op->vocabulary, K3_SAMPLE_MAX_VOCABULARY);
  if (sizes) return K3_SPINE_OK;
  if (!op->logits || !op->u || !op->tokens)
    return spine_fail(K3_SPINE_E_INVALID, "sample: null logits, u or tokens");
  const unsigned e = op->logits_dtype == K3_DTYPE_F32 ? 4 : 2;
  if (((uintptr_t)op->logits & (e - 1)) ||
      (((uintptr_t)op->u | (uintptr_t)op->temperature | (uintptr_t)op->top_k |
        (uintptr_t)op->top_p | (uintptr_t)op->min_p | (uintptr_t)op->tokens) & 3u))
    return spine_fail(K3_SPINE_E_INVALID, "sample: a pointer is not aligned to its elements");
  const uintptr_t t0 = (uintptr_t)op->tokens, t1 = t0 + 4ull * op->rows;
  auto meets = [&](const void* p, uint64_t bytes) {
    return p && (uintptr_t)p < t1 && t0 < (uintptr_t)p + bytes;
  };
  if (meets(op->logits, (uint64_t)op->rows * op->vocabulary * e) || meets(op->u, 4ull * op->rows) ||
      meets(op->temperature, 4ull * op->rows) || meets(op->top_k, 4ull * op->rows) ||
      meets(op->top_p, 4ull * op->rows) || meets(op->min_p, 4ull * op->rows))
    return spine_fail(K3_SPINE_E_INVALID, "sample: tokens overlap an input");
  return K3_SPINE_OK;
}

template <typename T>
int sample_launch(const SampleArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.parts, (unsigned)a.rows);
  for (int step = 0; step < 3; ++step) {
    TimedLaunch tl(KC_ROUTE, st);
    if (step == 0)
      launch_timed(tl, k_sample_ends<T>, grid, dim3(kScanThreads), 0, st, a);
    else if (step == 1)
      launch_timed(tl, k_sample_histogram<T>, grid, dim3(kScanThreads), 0, st, a);
    else
      launch_timed(tl, k_sample_pick<T>, dim3((unsigned)a.rows), dim3(kPickThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
      tl.failed();
      return spine_fail(K3_SPINE_E_RUNTIME, "sample launch: %s", hipGetErrorString(e));
    }
  }
  return K3_SPINE_OK;
}

}  // namespace
}  // namespace k3

using namespace k3;

static_assert(sizeof(K3HipSampleV1) == 80, "descriptor ABI drift");

extern "C" {

uint64_t k3_hip_sample_workspace_bytes(const K3HipSampleV1* op) {
  if (sample_check(op, true) != K3_SPINE_OK) return 0;
  return SampleLayout((int)op->rows, (int)op->vocabulary).bytes;
}

int k3_hip_sample(const K3HipSampleV1* op, void* workspace, uint64_t workspace_bytes,
                  void* stream) {
  int rc = sample_check(op, false);
  if (rc != K3_SPINE_OK) return rc;
  const SampleLayout l((int)op->rows, (int)op->vocabulary);
  if (!workspace || ((uintptr_t)workspace & 255u) != 0 || workspace_bytes < l.bytes)
    return spine_fail(K3_SPINE_E_INVALID,
                      "sample: the workspace must be %llu bytes at a 256-byte boundary",
                      (unsigned long long)l.bytes);
  const hipError_t e = hipGetLastError();  // an earlier call's, not this one's
  if (e != hipSuccess)
    return spine_fail(K3_SPINE_E_RUNTIME, "sample preflight: %s", hipGetErrorString(e));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  SampleArgs a{};
  a.logits = op->logits;
  a.u = op->u;
  a.temperature = op->temperature;
  a.top_k = op->top_k;
  a.top_p = op->top_p;
  a.min_p = op->min_p;
  a.tokens = op->tokens;
  a.ends = reinterpret_cast<uint32_t*>(ws);
  a.count = reinterpret_cast<uint32_t*>(ws + l.count);
  a.mass = reinterpret_cast<uint64_t*>(ws + l.mass);
  a.rows = (int)op->rows;
  a.vocab = (int)op->vocabulary;
  a.parts = l.parts;
  a.part = l.part;
  // sums of a whole row stay under 2^62
  int bits = 0;
  while ((1u << bits) < op->vocabulary) ++bits;
  a.shift = 62 - bits;
  hipStream_t st = static_cast<hipStream_t>(stream);
  try {
    return op->logits_dtype == K3_DTYPE_F32 ? sample_launch<float>(a, st)
                                            : sample_launch<uint16_t>(a, st);
  } catch (...) {
    return spine_fail(K3_SPINE_E_RUNTIME, "sample: out of host memory");
  }
}

}  // extern "C"
