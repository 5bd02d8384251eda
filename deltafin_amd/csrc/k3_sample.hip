// Token sampling (include/k3_hip_sample_abi.h) by selection instead of sorting.
//
// Every limit of a row (top-k, top-p, min-p) and the draw itself is a position in one
// order of its tokens, and a position is found by a radix descent over the 32-bit keys of
// the logits: a histogram of token counts and weight sums over the top 11 key bits, the
// bin in which the count or the sum crosses the wanted one, then the next 11 bits of that
// bin's tokens and the last 10.  Nothing is sorted or written back, so the work is a few
// reads of the row.
//
// Weights are 64-bit integers (see fixed_weight): sums of them are exact, so LDS and
// global atomics may add in any order, and two workgroups' histograms join without one.
//
// Launches: the row maxima (which the weights need), the first histogram (both over many
// workgroups per row), and one workgroup per row for the descents.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/k3_hip_sample_abi.h"
#include "k3_device.h"
#include "k3_internal.h"
#include "k3_launch.h"

namespace k3 {
namespace {

constexpr int kBins = 2048;          // of the first and second digit
constexpr int kScanThreads = 256;    // of the passes over a row's parts
constexpr int kPickThreads = 1024;   // of the workgroup that ends a row

struct SampleArgs {
  const void* logits;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
  uint32_t* part_max;  // [rows][parts] keys of the parts' largest logits
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
  bool sampled;    // T > 0
};

__device__ __forceinline__ RowParams row_params(const SampleArgs& a, int row, uint32_t top_key) {
  RowParams r;
  r.top = value_of(top_key);
  const float t = a.temperature ? a.temperature[row] : 1.f;
  r.sampled = t > 0.f;
  r.rate = r.sampled ? 1.4426950408889634 / (double)t : 0.0;
  return r;
}

// log2 of the weight of logit l, l <= top: 0 for the largest, -inf for what has none.
__device__ __forceinline__ double log2_weight(const RowParams& r, float l) {
  if (l == r.top) return 0.0;
  if (l == -INFINITY || r.top == INFINITY || !r.sampled) return -INFINITY;
  return ((double)l - (double)r.top) * r.rate;
}

// Weight times 2^shift, to the nearest integer: 2^y by y = n + h / 64 + f with |f| <= 1 / 128,
// 2^(h / 64) from LDS and 2^f by its Taylor series (the first term left out is under 2^-52).
__device__ __forceinline__ uint64_t fixed_weight(const RowParams& r, const double* table, int shift,
                                                 float l) {
  const double y = log2_weight(r, l);
  if (!(y > -64.0)) return 0;
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

template <typename T>
__global__ __launch_bounds__(kScanThreads) void k_sample_max(const SampleArgs a) {
  const int row = blockIdx.y, part = blockIdx.x;
  uint32_t best = 0xffffffffu;
  const int t0 = part * a.part, t1 = min(t0 + a.part, a.vocab);
  scan(static_cast<const T*>(a.logits) + (uint64_t)row * a.vocab, t0, t1, kScanThreads,
       [&](float l, int) { best = min(best, key_of(l)); });
  best = wave_min(best);
  __shared__ uint32_t red[kScanThreads / 64];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kScanThreads / 64; ++w) best = min(best, red[w]);
    a.part_max[(uint64_t)row * a.parts + part] = best;
  }
  // this part's share of the row's histogram, for the next launch to add to
  for (int b = part * kScanThreads + threadIdx.x; b < kBins; b += a.parts * kScanThreads) {
    a.count[(uint64_t)row * kBins + b] = 0;
    a.mass[(uint64_t)row * kBins + b] = 0;
  }
}

__device__ __forceinline__ uint32_t row_top(const SampleArgs& a, int row) {
  uint32_t best = 0xffffffffu;
  for (int i = 0; i < a.parts; ++i) best = min(best, a.part_max[(uint64_t)row * a.parts + i]);
  return best;
}

template <typename T>
__global__ __launch_bounds__(kScanThreads) void k_sample_histogram(const SampleArgs a) {
  const int row = blockIdx.y, part = blockIdx.x;
  __shared__ uint32_t count[kBins];
  __shared__ uint64_t mass[kBins];
  __shared__ double table[64];
  fill_table(table);
  for (int b = threadIdx.x; b < kBins; b += kScanThreads) {
    count[b] = 0;
    mass[b] = 0;
  }
  const RowParams r = row_params(a, row, row_top(a, row));
  __syncthreads();
  const int t0 = part * a.part, t1 = min(t0 + a.part, a.vocab);
  scan(static_cast<const T*>(a.logits) + (uint64_t)row * a.vocab, t0, t1, kScanThreads,
       [&](float l, int) {
         const uint32_t b = key_of(l) >> 21;
         atomicAdd(&count[b], 1u);
         const uint64_t w = fixed_weight(r, table, a.shift, l);
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

// A position in a row's order: the key of its token and what lies before that key.
struct Found {
  uint32_t key;
  uint32_t before;       // tokens of smaller keys
  uint64_t mass_before;  // and their weight
  uint32_t equal;        // tokens of this key
};

struct PickShared {
  uint32_t count[kBins];
  uint64_t mass[kBins];
  double table[64];
  uint32_t wave_count[kPickThreads / 64];
  uint64_t wave_mass[kPickThreads / 64];
  uint32_t bin, before;
  uint64_t mass_before;
  int token;
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  return (uint64_t)__shfl_up((unsigned long long)v, d);
}

// The first bin of sh.count / sh.mass at which the running count (by_count) or mass,
// `before` included, exceeds `target`: into sh.bin, sh.before and sh.mass_before.  There
// is one.
__device__ __forceinline__ void cross(PickShared& sh, int bins, bool by_count, uint64_t target,
                                      uint32_t before, uint64_t mass_before) {
  const int b = 2 * threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t c0 = b < bins ? sh.count[b] : 0u, c1 = b < bins ? sh.count[b + 1] : 0u;
  const uint64_t m0 = b < bins ? sh.mass[b] : 0u, m1 = b < bins ? sh.mass[b + 1] : 0u;
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
  c += before;
  m += mass_before;
  for (int w = 0; w < wave; ++w) {
    c += sh.wave_count[w];
    m += sh.wave_mass[w];
  }
  // running values ahead of this thread's two bins, between them and behind them
  const uint32_t r0 = c - c0 - c1, r1 = c - c1;
  const uint64_t s0 = m - m0 - m1, s1 = m - m1;
  const uint64_t v0 = by_count ? r0 : s0, v1 = by_count ? r1 : s1, v2 = by_count ? c : m;
  if (v0 <= target && v1 > target) {
    sh.bin = b;
    sh.before = r0;
    sh.mass_before = s0;
  } else if (v1 <= target && v2 > target) {
    sh.bin = b + 1;
    sh.before = r1;
    sh.mass_before = s1;
  }
  __syncthreads();
}

// The histogram of the digit of `bits` key bits above `low`, over the row's tokens whose
// higher bits are `prefix`.
template <typename T>
__device__ __forceinline__ void digit_histogram(PickShared& sh, const SampleArgs& a, const T* row,
                                                const RowParams& r, uint32_t prefix, int low,
                                                int bits) {
  __syncthreads();
  for (int b = threadIdx.x; b < (1 << bits); b += kPickThreads) {
    sh.count[b] = 0;
    sh.mass[b] = 0;
  }
  __syncthreads();
  scan(row, 0, a.vocab, kPickThreads, [&](float l, int) {
    const uint32_t k = key_of(l);
    if (k >> (low + bits) != prefix) return;
    const uint32_t b = (k >> low) & ((1u << bits) - 1u);
    atomicAdd(&sh.count[b], 1u);
    const uint64_t w = fixed_weight(r, sh.table, a.shift, l);
    if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[b]), (unsigned long long)w);
  });
  __syncthreads();
}

__device__ __forceinline__ void first_histogram(PickShared& sh, const SampleArgs& a, int row) {
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kPickThreads) {
    sh.count[b] = a.count[(uint64_t)row * kBins + b];
    sh.mass[b] = a.mass[(uint64_t)row * kBins + b];
  }
  __syncthreads();
}

// The first token of the order at which the running count or mass exceeds target.
template <typename T>
__device__ __forceinline__ Found descend(PickShared& sh, const SampleArgs& a, int row_index,
                                         const T* row, const RowParams& r, bool by_count,
                                         uint64_t target) {
  first_histogram(sh, a, row_index);
  cross(sh, kBins, by_count, target, 0u, 0u);
  uint32_t prefix = sh.bin, before = sh.before;
  uint64_t mass_before = sh.mass_before;
  digit_histogram(sh, a, row, r, prefix, 10, 11);
  cross(sh, 2048, by_count, target, before, mass_before);
  prefix = prefix << 11 | sh.bin;
  before = sh.before;
  mass_before = sh.mass_before;
  digit_histogram(sh, a, row, r, prefix, 0, 10);
  cross(sh, 1024, by_count, target, before, mass_before);
  Found f;
  f.key = prefix << 10 | sh.bin;
  f.before = sh.before;
  f.mass_before = sh.mass_before;
  f.equal = sh.count[sh.bin];
  __syncthreads();
  return f;
}

// The token of rank `nth` (from 0) among those with the key, by index.
template <typename T>
__device__ __forceinline__ int nth_equal(PickShared& sh, const SampleArgs& a, const T* row,
                                         uint32_t key, uint32_t nth) {
  constexpr int kWaves = kPickThreads / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int share = (a.vocab + kWaves - 1) / kWaves;
  const int t0 = min(wave * share, a.vocab), t1 = min(t0 + share, a.vocab);
  auto is = [&](int t) {
    if (t >= t1) return false;
    float l;
    if constexpr (sizeof(T) == 4)
      l = row[t];
    else
      l = bf16_bits_to_f32(row[t]);
    return key_of(l) == key;
  };
  uint32_t n = 0;
  for (int t = t0; t < t1; t += 64) n += __popcll(__ballot(is(t + lane)));
  if (lane == 0) sh.wave_count[wave] = n;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += sh.wave_count[w];
  if (before <= nth && nth < before + n) {
    uint32_t left = nth - before;
    for (int t = t0; t < t1; t += 64) {
      const bool here = is(t + lane);
      const uint64_t mask = __ballot(here);
      const uint32_t m = (uint32_t)__popcll(mask);
      if (left < m) {
        if (here && (uint32_t)__popcll(mask & ((1ull << lane) - 1)) == left) sh.token = t + lane;
        break;
      }
      left -= m;
    }
  }
  __syncthreads();
  return sh.token;
}

template <typename T>
__global__ __launch_bounds__(kPickThreads) void k_sample_pick(const SampleArgs a) {
  __shared__ PickShared sh;
  const int ri = blockIdx.x;
  const T* row = static_cast<const T*>(a.logits) + (uint64_t)ri * a.vocab;
  const uint32_t top = row_top(a, ri);
  if (top == kKeyMasked) {  // nothing but -inf and NaN
    if (threadIdx.x == 0) a.tokens[ri] = -1;
    return;
  }
  fill_table(sh.table);
  const RowParams r = row_params(a, ri, top);
  if (!r.sampled) {
    const int t = nth_equal(sh, a, row, top, 0u);
    if (threadIdx.x == 0) a.tokens[ri] = t;
    return;
  }
  // the sum over the whole row, then the mass of the top-k prefix
  first_histogram(sh, a, ri);
  uint64_t total = 0;
  {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t m = sh.mass[2 * threadIdx.x] + sh.mass[2 * threadIdx.x + 1];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m += (uint64_t)__shfl_xor((unsigned long long)m, d);
    if (lane == 0) sh.wave_mass[wave] = m;
    __syncthreads();
    for (int w = 0; w < kPickThreads / 64; ++w) total += sh.wave_mass[w];
    __syncthreads();
  }
  auto weight = [&](uint32_t key) { return fixed_weight(r, sh.table, a.shift, value_of(key)); };
  uint64_t kept = total;  // weight of the shortest prefix so far
  const int k = a.top_k ? a.top_k[ri] : 0;
  if (k > 0 && k < a.vocab) {
    const Found f = descend(sh, a, ri, row, r, true, (uint64_t)(k - 1));
    kept = f.mass_before + (uint64_t)((uint32_t)k - f.before) * weight(f.key);
  }
  const float p = a.top_p ? a.top_p[ri] : 1.f;
  if (p < 1.f) {
    // the first prefix with a sum of at least p times the top-k one's
    const uint64_t want = max((uint64_t)1, (uint64_t)ceil(fmax((double)p, 0.0) * (double)kept));
    const Found f = descend(sh, a, ri, row, r, false, want - 1);
    const uint64_t w = weight(f.key);
    kept = min(kept, f.mass_before + (want - f.mass_before + w - 1) / w * w);
  }
  const float mp = a.min_p ? a.min_p[ri] : 0.f;
  if (mp > 0.f) {
    // the last key whose weight is at least min_p, by halving over the keys from the top
    const double least = log2(fmin((double)mp, 1.0));
    uint32_t lo = top, hi = kKeyMasked;  // lo is kept, hi is not
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (log2_weight(r, value_of(mid)) >= least)
        lo = mid;
      else
        hi = mid;
    }
    // weight of the tokens up to it: a sum over its bin behind the bins before
    const uint32_t bin = lo >> 21;
    first_histogram(sh, a, ri);
    uint64_t m = 0;
    for (uint32_t b = threadIdx.x; b < bin; b += kPickThreads) m += sh.mass[b];
    scan(row, 0, a.vocab, kPickThreads, [&](float l, int) {
      const uint32_t key = key_of(l);
      if (key >> 21 == bin && key <= lo) m += fixed_weight(r, sh.table, a.shift, l);
    });
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m += (uint64_t)__shfl_xor((unsigned long long)m, d);
    if ((threadIdx.x & 63) == 0) sh.wave_mass[threadIdx.x >> 6] = m;
    __syncthreads();
    m = 0;
    for (int w = 0; w < kPickThreads / 64; ++w) m += sh.wave_mass[w];
    __syncthreads();
    kept = min(kept, m);
  }
  float u = a.u[ri];
  if (!(u < 1.f)) u = 1.f - 0x1p-24f;
  u = fmaxf(u, 0.f);
  const uint64_t target = min((uint64_t)((double)u * (double)kept), kept - 1);
  const Found f = descend(sh, a, ri, row, r, false, target);
  const uint32_t nth = (uint32_t)((target - f.mass_before) / weight(f.key));
  const int t = nth_equal(sh, a, row, f.key, nth);
  if (threadIdx.x == 0) a.tokens[ri] = t;
}

uint64_t align256(uint64_t v) { return (v + 255) & ~255ull; }

struct SampleLayout {
  int parts, part;
  uint64_t count, mass, bytes;  // offsets of the histograms behind the part maxima
  SampleLayout(int rows, int vocab) {
    // parts of at least 4096 tokens, about two workgroups per CU over all rows
    const int want = std::max(1, 512 / rows);
    parts = std::min(want, (vocab + 4095) / 4096);
    part = (vocab + parts - 1) / parts;
    parts = (vocab + part - 1) / part;
    count = align256(4ull * rows * parts);
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
      launch_timed(tl, k_sample_max<T>, grid, dim3(kScanThreads), 0, st, a);
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
  a.part_max = reinterpret_cast<uint32_t*>(ws);
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
