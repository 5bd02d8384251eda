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
// Launches: the rows' largest and smallest logits, the histogram, the tokens of every
// range in which one of the positions can lie (all three over many workgroups per row), and
// one workgroup per row for the positions.  The limits depend on one another (top-p on the
// weight that top-k leaves, the draw on all of them), but each lies between values that the
// histogram gives, so the candidates are one to three ranges each, a few hundred tokens;
// the last workgroup has them in LDS.  Ranges of more than kList tokens (thousands of
// near-equal logits) stay in memory and are walked there.
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
constexpr int kList = 4096;          // candidates of a row that are gathered
constexpr int kScanThreads = 512;    // of the passes over a row's parts
constexpr int kPickThreads = 1024;   // of the workgroup that ends a row
constexpr double kVanish = 64.0;     // weights under 2^-kVanish round to none

constexpr int kRanges = 4;           // top-k's, top-p's, min-p's and the draw's
// Tokens that are ranked one against all: 96 rows of 150001 take 21 us in the last launch;
// with 64 by one wave 29, 512 27, 1024 26.
constexpr int kSmall = 256;
constexpr int kRankers = kPickThreads / kSmall;  // threads per token
static_assert(kSmall * kRankers == kPickThreads && 64 % kRankers == 0,
              "a token's threads are in one wave");

// The ranges of bins in which a row's positions lie; a bin's tokens are gathered for the
// first of them that holds it.
struct RowPlan {
  int32_t first;                     // lowest index of the largest logit (T not above 0)
  int32_t listed;                    // places of the list in use
  int32_t b0[kRanges], b1[kRanges];  // first and last bin
  int32_t base[kRanges];             // place of the first in the list, or -1
  int32_t pad[2];
};
static_assert(sizeof(RowPlan) == 64, "one line per row");

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
  uint32_t* taken;     // [rows][kBins] tokens gathered
  RowPlan* plan;       // [rows]
  uint2* list;         // [rows][kList] gathered keys and indices, a range's bins in order
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
// share: 16 bytes per load, four in flight (those past the end repeat the last, so that none
// is conditional: behind a branch each waited for the one before), single tokens ahead of
// the first 16-byte boundary and behind the last.
template <typename T, typename F>
__device__ __forceinline__ void scan(const T* row, int t0, int t1, int threads, F f) {
  constexpr int kPer = 16 / (int)sizeof(T);
  constexpr int kUnroll = 4;
  const T* p = row + t0;
  const int n = max(t1 - t0, 0);
  const int off = (int)(((uintptr_t)p & 15u) / sizeof(T));
  const int head = min(n, off ? kPer - off : 0);
  const int chunks = (n - head) / kPer;
  auto one = [&](int t) {
    float l;
    if constexpr (sizeof(T) == 4)
      l = p[t];
    else
      l = bf16_bits_to_f32(p[t]);
    f(l, t0 + t);
  };
  const int tail = head + chunks * kPer;
  if ((int)threadIdx.x < head) one(threadIdx.x);
  if ((int)threadIdx.x < n - tail) one(tail + threadIdx.x);
  const u32x4* base = reinterpret_cast<const u32x4*>(p + head);
  for (int c0 = threadIdx.x; c0 < chunks; c0 += kUnroll * threads) {
    u32x4 v[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) v[k] = base[min(c0 + k * threads, chunks - 1)];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int c = c0 + k * threads;
      if (c >= chunks) break;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float l;
        if constexpr (sizeof(T) == 4)
          l = __uint_as_float(v[k][i]);
        else
          l = __uint_as_float(i % 2 ? v[k][i / 2] & 0xffff0000u : v[k][i / 2] << 16);
        f(l, t0 + head + c * kPer + i);
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
    a.taken[(uint64_t)row * kBins + b] = 0;
  }
  if (part == 0 && threadIdx.x == 0) a.plan[row].first = a.vocab;
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

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  return (uint64_t)__shfl_up((unsigned long long)v, d);
}
__device__ __forceinline__ void add64(uint64_t* to, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(to), (unsigned long long)v);
}

// A row's histogram as running counts and weights, each bin's own included, in the LDS of a
// workgroup of THREADS.  Every member is called by all of its threads.
template <int THREADS>
struct Running {
  uint32_t count[kBins];
  uint64_t mass[kBins];
  uint32_t wave_count[THREADS / 64];
  uint64_t wave_mass[THREADS / 64];
  int bin;

  __device__ __forceinline__ void load(const SampleArgs& a, int row) {
    constexpr int kPer = kBins / THREADS;
    const int b = kPer * threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t* gc = a.count + (uint64_t)row * kBins + b;
    const uint64_t* gm = a.mass + (uint64_t)row * kBins + b;
    uint32_t cv[kPer], c = 0;
    uint64_t mv[kPer], m = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      cv[i] = c += gc[i];
      mv[i] = m += gm[i];
    }
    const uint32_t own_c = c;
    const uint64_t own_m = m;
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
      wave_count[wave] = c;
      wave_mass[wave] = m;
    }
    __syncthreads();
    c -= own_c;
    m -= own_m;
    for (int w = 0; w < wave; ++w) {
      c += wave_count[w];
      m += wave_mass[w];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      count[b + i] = c + cv[i];
      mass[b + i] = m + mv[i];
    }
    __syncthreads();
  }

  __device__ __forceinline__ uint32_t count_before(int b) const { return b ? count[b - 1] : 0u; }
  __device__ __forceinline__ uint64_t mass_before(int b) const { return b ? mass[b - 1] : 0u; }

  // The first bin whose running count or weight exceeds target; there is one.
  __device__ __forceinline__ int crossing(bool by_count, uint64_t target) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBins / THREADS; ++i) {
      const int b = threadIdx.x + i * THREADS;
      const uint64_t here = by_count ? count[b] : mass[b];
      const uint64_t ahead = by_count ? count_before(b) : mass_before(b);
      if (ahead <= target && here > target) bin = b;
    }
    __syncthreads();
    return bin;
  }
};

// The last key of the bins up to `bin`, by a wave: bins never fall along the keys.  64 keys
// at a time; with the two ends of a range known, its tokens are told by their values,
// without the fp64 of bin_of (which took half of a pass over the row).
__device__ __forceinline__ uint32_t last_key(const RowParams& r, int bin) {
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

// A row's limits.
struct Limits {
  bool has_k, has_p, has_m;
  uint64_t k;       // target count of the last of the first top_k
  double p, least;  // top-p's share, min-p's log2 weight
  double u;
};

template <int THREADS>
__device__ __forceinline__ Limits row_limits(const SampleArgs& a, int row,
                                             const Running<THREADS>& h) {
  Limits l;
  const int k = a.top_k ? a.top_k[row] : 0;
  // (a first k that ends among the tokens of no weight leaves the sum as it is)
  l.has_k = k > 0 && k < a.vocab && (uint32_t)k <= h.count[kBins - 2];
  l.k = (uint64_t)(k - 1);
  const float p = a.top_p ? a.top_p[row] : 1.f;
  l.has_p = p < 1.f;
  l.p = fmax((double)p, 0.0);
  const float m = a.min_p ? a.min_p[row] : 0.f;
  l.has_m = m > 0.f;
  l.least = l.has_m ? log2(fmin((double)m, 1.0)) : 0.0;
  float u = a.u[row];
  if (!(u < 1.f)) u = 1.f - 0x1p-24f;
  l.u = (double)fmaxf(u, 0.f);
  return l;
}

// The weight that a top-p prefix has to reach, and the one that the draw has to exceed:
// both rise with the weight they are shares of.
__device__ __forceinline__ uint64_t top_p_want(const Limits& l, uint64_t kept) {
  return max((uint64_t)1, (uint64_t)ceil(l.p * (double)kept));
}
__device__ __forceinline__ uint64_t draw_target(const Limits& l, uint64_t kept) {
  return min((uint64_t)(l.u * (double)kept), kept - 1);
}

template <typename T>
__global__ __launch_bounds__(kScanThreads) void k_sample_gather(const SampleArgs a) {
  const int row = blockIdx.y, part = blockIdx.x;
  __shared__ Running<kScanThreads> h;
  __shared__ RowPlan plan;
  __shared__ uint32_t red[2 * kScanThreads / 64];
  __shared__ float most[kRanges], least[kRanges];
  __shared__ uint32_t found, key[kList], index[kList];
  uint32_t top, bottom;
  row_ends(a, row, red, kScanThreads, &top, &bottom);
  if (top == kKeyMasked) return;
  const RowParams r = row_params(a, row, top, bottom);
  const T* tokens = static_cast<const T*>(a.logits) + (uint64_t)row * a.vocab;
  const int t0 = part * a.part, t1 = min(t0 + a.part, a.vocab);
  if (!r.sampled) {
    int at = a.vocab;
    scan(tokens, t0, t1, kScanThreads, [&](float l, int t) {
      if (l == r.top) at = min(at, t);
    });
    if (at < a.vocab) atomicMin(&a.plan[row].first, at);
    return;
  }
  h.load(a, row);
  const Limits l = row_limits(a, row, h);
  // each limit's bins, from what the ones before it leave at least and at most
  uint64_t lo = h.mass[kBins - 1], hi = lo;
  int b0[kRanges], b1[kRanges];
#pragma unroll
  for (int i = 0; i < kRanges; ++i) {
    b0[i] = kBins;
    b1[i] = -1;
  }
  if (l.has_k) {
    b0[0] = b1[0] = h.crossing(true, l.k);
    lo = h.mass_before(b0[0]);
    hi = h.mass[b0[0]];
  }
  if (l.has_p) {
    b0[1] = h.crossing(false, top_p_want(l, lo) - 1);
    b1[1] = h.crossing(false, top_p_want(l, hi) - 1);
    lo = min(lo, h.mass_before(b0[1]));
    hi = min(hi, h.mass[b1[1]]);
  }
  if (l.has_m) {
    const int b = bin_of(r, l.least);
    if (h.mass_before(b) < hi) b0[2] = b1[2] = b;
    lo = min(lo, h.mass_before(b));
    hi = min(hi, h.mass[b]);
  }
  b0[3] = h.crossing(false, lo ? draw_target(l, lo) : 0);
  b1[3] = h.crossing(false, draw_target(l, hi));
  // places, while they fit, for ranges that no earlier one holds
  int base[kRanges], total = 0;
#pragma unroll
  for (int i = 0; i < kRanges; ++i) {
    base[i] = -1;
    bool held = b1[i] < 0;
#pragma unroll
    for (int k = 0; k < i; ++k) held = held || (base[k] >= 0 && b0[k] <= b0[i] && b1[i] <= b1[k]);
    if (held) continue;
    const int n = (int)(h.count[b1[i]] - h.count_before(b0[i]));
    if (n > kList - total) continue;
    base[i] = total;
    total += n;
  }
  const int wave = threadIdx.x >> 6;
  static_assert(2 * kRanges <= kScanThreads / 64, "a wave per end of a range");
#pragma unroll
  for (int i = 0; i < kRanges; ++i) {
    if (wave != i && wave != kRanges + i) continue;
    // (an empty range of values where there is none)
    float* end = wave == i ? &most[i] : &least[i];
    const float none = wave == i ? -INFINITY : INFINITY;
    const float v = base[i] < 0 ? none
                    : wave == i ? value_of(last_key(r, b0[i] - 1) + 1)
                                : value_of(last_key(r, b1[i]));
    if ((threadIdx.x & 63) == 0) *end = v;
  }
  if (threadIdx.x == 0) {
    plan.first = a.vocab;
    plan.listed = total;
#pragma unroll
    for (int i = 0; i < kRanges; ++i) {
      plan.b0[i] = b0[i];
      plan.b1[i] = b1[i];
      plan.base[i] = base[i];
    }
    found = 0;
  }
  __syncthreads();
  if (part == 0 && threadIdx.x < sizeof(RowPlan) / 4)
    reinterpret_cast<int32_t*>(&a.plan[row])[threadIdx.x] =
        reinterpret_cast<const int32_t*>(&plan)[threadIdx.x];
  float m[kRanges], s[kRanges];
#pragma unroll
  for (int i = 0; i < kRanges; ++i) {
    m[i] = most[i];
    s[i] = least[i];
  }
  scan(tokens, t0, t1, kScanThreads, [&](float v, int t) {
    bool in = false;
#pragma unroll
    for (int i = 0; i < kRanges; ++i) in = in || (v <= m[i] && v >= s[i]);
    if (!in) return;
    const uint32_t at = atomicAdd(&found, 1u);
    if (at >= (uint32_t)kList) return;  // (the row changed under the call)
    key[at] = key_of(v);
    index[at] = (uint32_t)t;
  });
  __syncthreads();
  // places by the bins' counters in memory, all at once: one at a time, as tokens were
  // found, their round trips took most of the launch
  for (uint32_t i = threadIdx.x; i < min(found, (uint32_t)kList); i += kScanThreads) {
    const int b = bin_of(r, log2_weight(r, value_of(key[i])));
    int from = 0, place = 0;
#pragma unroll
    for (int k = kRanges - 1; k >= 0; --k)
      if (base[k] >= 0 && b0[k] <= b && b <= b1[k]) {
        from = b0[k];
        place = base[k];
      }
    const uint32_t at = place + (h.count_before(b) - h.count_before(from)) +
                        atomicAdd(&a.taken[(uint64_t)row * kBins + b], 1u);
    if (at < (uint32_t)kList) a.list[(uint64_t)row * kList + at] = make_uint2(key[i], index[i]);
  }
}

struct PickShared {
  Running<kPickThreads> h;
  RowPlan plan;
  double table[64];
  uint2 list[kList];
  uint32_t digit_count[256];
  uint64_t digit_mass[256];
  ulonglong2 ranked[kSmall];  // key and index, weight
  uint32_t small;
  uint32_t red[2 * kPickThreads / 64];
  uint64_t wave_mass[kPickThreads / 64];
  uint32_t digit, before;
  uint64_t mass;
  int token;
};

// A position in a row's order.
struct Found {
  uint64_t mass;  // weight through its token
  int token;      // if asked for
};

// One row's workgroup.  Every member is called by all of its threads.
template <typename T>
struct Picker {
  PickShared& sh;
  const SampleArgs& a;
  const T* row;
  RowParams r;

  __device__ __forceinline__ uint64_t weight(uint32_t key) const {
    return fixed_weight(sh.table, a.shift, log2_weight(r, value_of(key)));
  }

  // Where a bin's tokens are: a part of the list, or a range of values in memory.
  struct Place {
    int at, n;         // n < 0: in memory
    float most, least;
  };
  __device__ __forceinline__ Place place(int bin) const {
    Place p{0, -1, 0.f, 0.f};
#pragma unroll
    for (int i = kRanges - 1; i >= 0; --i)
      if (sh.plan.b0[i] <= bin && bin <= sh.plan.b1[i] && sh.plan.base[i] >= 0) {
        const uint32_t before = sh.h.count_before(bin);
        p.at = sh.plan.base[i] + (int)(before - sh.h.count_before(sh.plan.b0[i]));
        p.n = (int)(sh.h.count[bin] - before);
        p.n = min(p.n, kList - p.at);
      }
    if (p.n < 0) {
      p.most = value_of(last_key(r, bin - 1) + 1);
      p.least = value_of(last_key(r, bin));
    }
    return p;
  }

  // Calls f(key, index) for the tokens of a bin, each thread its share.
  template <typename F>
  __device__ __forceinline__ void each(const Place& p, F f) {
    if (p.n >= 0) {
      for (int i = threadIdx.x; i < p.n; i += kPickThreads) f(sh.list[p.at + i].x, sh.list[p.at + i].y);
    } else {
      scan(row, 0, a.vocab, kPickThreads, [&](float l, int t) {
        if (l <= p.most && l >= p.least) f(key_of(l), (uint32_t)t);
      });
    }
  }

  // What lies before a set of values, what the set holds, and the bits all of them share.
  struct Part {
    uint32_t before, n;
    uint64_t mass;    // weight before it
    uint32_t prefix;  // the values' bits from `low` up, in place
    int low;
  };

  // Narrows the part to the bits in which its values differ.  walk(f) calls f(value).
  template <typename W>
  __device__ __forceinline__ void narrow(W walk, Part* part) {
    uint32_t lo = 0xffffffffu, hi = 0u;
    walk([&](uint32_t v) {
      lo = min(lo, v);
      hi = max(hi, v);
    });
    block_ends(sh.red, kPickThreads / 64, &lo, &hi);
    const uint32_t x = lo ^ hi;
    part->low = x ? 32 - __clz((int)x) : 0;
    part->prefix = part->low == 32 ? 0u : lo >> part->low << part->low;
  }

  __device__ __forceinline__ bool in(const Part& part, uint32_t v) const {
    return part.low == 32 || v >> part.low == part.prefix >> part.low;
  }

  // Narrows the part by its next (up to) eight bits, to the values at which the running
  // count or weight exceeds target.
  template <typename W>
  __device__ __forceinline__ void digit(W walk, bool by_count, bool weigh, uint64_t target,
                                        Part* part) {
    const int width = min(part->low, 8), low = part->low - width;
    __syncthreads();
    if (threadIdx.x < 256) {
      sh.digit_count[threadIdx.x] = 0;
      sh.digit_mass[threadIdx.x] = 0;
    }
    __syncthreads();
    walk([&](uint32_t v) {
      if (!in(*part, v)) return;
      const uint32_t d = (v >> low) & ((1u << width) - 1u);
      atomicAdd(&sh.digit_count[d], 1u);
      const uint64_t w = weigh ? weight(v) : 0;
      if (w) add64(&sh.digit_mass[d], w);
    });
    __syncthreads();
    if (threadIdx.x < 64) {
      uint32_t c[4], cs = 0;
      uint64_t m[4], ms = 0;
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
      uint32_t cr = part->before + ci - cs;
      uint64_t mr = part->mass + mi - ms;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t ahead = by_count ? cr : mr;
        const uint64_t here = by_count ? (uint64_t)(cr + c[i]) : mr + m[i];
        if (ahead <= target && here > target) {
          sh.digit = 4 * threadIdx.x + i;
          sh.before = cr;
          sh.mass = mr;
        }
        cr += c[i];
        mr += m[i];
      }
    }
    __syncthreads();
    part->low = low;
    part->prefix |= sh.digit << low;
    part->before = sh.before;
    part->mass = sh.mass;
    part->n = sh.digit_count[sh.digit & 255u];
  }

  // The first token at which the row's running count or weight exceeds target.
  __device__ __forceinline__ Found find(bool by_count, uint64_t target, bool ask_token) {
    const int bin = sh.h.crossing(by_count, target);
    const Place at = place(bin);
    auto keys = [&](auto f) { each(at, [&](uint32_t k, uint32_t) { f(k); }); };
    Part part;
    part.before = sh.h.count_before(bin);
    part.mass = sh.h.mass_before(bin);
    part.n = sh.h.count[bin] - part.before;
    part.prefix = 0;
    part.low = 32;
    if (part.n > kSmall) narrow(keys, &part);
    while (part.n > kSmall && part.low > 0) digit(keys, by_count, true, target, &part);
    if (part.n <= kSmall) {
      // few tokens: four threads rank each against all of them, by key and index
      __syncthreads();
      if (threadIdx.x == 0) sh.small = 0;
      __syncthreads();
      each(at, [&](uint32_t k, uint32_t t) {
        if (!in(part, k)) return;
        const uint32_t i = atomicAdd(&sh.small, 1u);
        if (i >= (uint32_t)kSmall) return;  // (the row changed under the call)
        sh.ranked[i] = make_ulonglong2((unsigned long long)k << 32 | t, weight(k));
      });
      __syncthreads();
      const int n = min((int)sh.small, kSmall), i = threadIdx.x / kRankers;
      if (i < n) {
        const ulonglong2 own = sh.ranked[i];
        uint32_t c = 0;
        uint64_t m = 0;
        for (int j = threadIdx.x % kRankers; j < n; j += kRankers) {
          const ulonglong2 other = sh.ranked[j];
          const bool ahead = other.x < own.x;
          c += ahead;
          m += ahead ? other.y : 0;
        }
#pragma unroll
        for (int d = 1; d < kRankers; d <<= 1) {
          c += __shfl_xor(c, d);
          m += (uint64_t)__shfl_xor((unsigned long long)m, d);
        }
        c += part.before;
        m += part.mass;
        const uint64_t ahead = by_count ? c : m, here = by_count ? (uint64_t)c + 1 : m + own.y;
        if (threadIdx.x % kRankers == 0 && ahead <= target && here > target) {
          sh.mass = m + own.y;
          sh.token = (int)(uint32_t)own.x;
        }
      }
      __syncthreads();
      return Found{sh.mass, sh.token};
    }
    // many tokens of one key: whole weights of it, in the order of their indices
    const uint32_t key = part.prefix;
    const uint64_t w = weight(key);
    const uint64_t nth = by_count ? target - part.before : (target - part.mass) / w;
    Found f{part.mass + (nth + 1) * w, -1};
    if (ask_token) {
      auto indices = [&](auto g) {
        each(at, [&](uint32_t k, uint32_t t) {
          if (k == key) g(t);
        });
      };
      Part p{0u, part.n, 0u, 0u, 32};
      narrow(indices, &p);
      while (p.low > 0) digit(indices, true, false, nth, &p);
      f.token = (int)p.prefix;
    }
    return f;
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
  if (!r.sampled) {
    if (threadIdx.x == 0) a.tokens[ri] = a.plan[ri].first;
    return;
  }
  fill_table(sh.table);
  if (threadIdx.x < sizeof(RowPlan) / 4)
    reinterpret_cast<int32_t*>(&sh.plan)[threadIdx.x] =
        reinterpret_cast<const int32_t*>(&a.plan[ri])[threadIdx.x];
  sh.h.load(a, ri);
  for (int i = threadIdx.x; i < min(sh.plan.listed, kList); i += kPickThreads)
    sh.list[i] = a.list[(uint64_t)ri * kList + i];
  Picker<T> p{sh, a, row, r};
  const Limits l = row_limits(a, ri, sh.h);
  uint64_t kept = sh.h.mass[kBins - 1];  // weight of the shortest prefix so far
  if (l.has_k) kept = p.find(true, l.k, false).mass;
  if (l.has_p) kept = min(kept, p.find(false, top_p_want(l, kept) - 1, false).mass);
  if (l.has_m) {
    const int bin = bin_of(r, l.least);
    if (sh.h.mass_before(bin) < kept) {  // else a shorter prefix is there already
      uint64_t m = 0;
      __syncthreads();
      p.each(p.place(bin), [&](uint32_t key, uint32_t) {
        const double y = log2_weight(r, value_of(key));
        if (y >= l.least) m += fixed_weight(sh.table, a.shift, y);
      });
      kept = min(kept, sh.h.mass_before(bin) + p.block_sum(m));
    }
  }
  const int t = p.find(false, draw_target(l, kept), true).token;
  if (threadIdx.x == 0) a.tokens[ri] = t;
}

uint64_t align256(uint64_t v) { return (v + 255) & ~255ull; }

struct SampleLayout {
  int parts, part;
  uint64_t count, mass, taken, plan, list, bytes;  // offsets behind the parts' ends
  SampleLayout(int rows, int vocab) {
    // parts of at least 4096 tokens, about two workgroups per CU over all rows
    const int want = std::max(1, 512 / rows);
    parts = std::min(want, (vocab + 4095) / 4096);
    part = (vocab + parts - 1) / parts;
    parts = (vocab + part - 1) / part;
    count = align256(8ull * rows * parts);
    mass = count + align256(4ull * rows * kBins);
    taken = mass + align256(8ull * rows * kBins);
    plan = taken + align256(4ull * rows * kBins);
    list = plan + align256(sizeof(RowPlan) * (uint64_t)rows);
    bytes = list + align256(sizeof(uint2) * (uint64_t)rows * kList);
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
  for (int step = 0; step < 4; ++step) {
    TimedLaunch tl(KC_ROUTE, st);
    if (step == 0)
      launch_timed(tl, k_sample_ends<T>, grid, dim3(kScanThreads), 0, st, a);
    else if (step == 1)
      launch_timed(tl, k_sample_histogram<T>, grid, dim3(kScanThreads), 0, st, a);
    else if (step == 2)
      launch_timed(tl, k_sample_gather<T>, grid, dim3(kScanThreads), 0, st, a);
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
  a.taken = reinterpret_cast<uint32_t*>(ws + l.taken);
  a.plan = reinterpret_cast<RowPlan*>(ws + l.plan);
  a.list = reinterpret_cast<uint2*>(ws + l.list);
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
