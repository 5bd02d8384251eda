// Dense layers over many positions on the BF16 matrix cores: a projection with bias,
// activation and residual, the gated feed-forward block and its gradient
// (include/k3_hip_dense_abi.h).  The product core is k3_gemm.h; this file lays operands
// out, ends the sums and chooses tiles.
//
// fp32 activations.  x = t0 + t1 + t2, each term the BF16 nearest to what the earlier
// ones leave (24 bits in all), written once as three planes; a product is then three
// segments of the same sum.  Forward rows are first scaled by a power of two that brings
// their largest value into [1, 2), so that no term of a value within 2^-100 of it falls
// below BF16's smallest subnormal; the sum's end takes the scale back.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "k3_dense.h"
#include "k3_device.h"
#include "k3_gemm.h"
#include "k3_internal.h"
#include "k3_launch.h"
#include "k3_skinny.h"

namespace k3 {
namespace {

using namespace gemm;

enum { EPI_LINEAR = 0, EPI_GLU = 1, EPI_GRAD = 2 };

// What happens to a sum.
struct Epilogue {
  const float* rs;    // int8 row scales [n]
  const float* rs2;   // GLU: up's
  const float* bias;  // LINEAR
  const float* xs;    // [m] scale of an fp32 activation row
  const void* res;    // LINEAR
  void* out;          // [m][n]; GRAD with half: rows [0, half) of m
  void* out1;         // GLU: kept g; GRAD: rows [half, 2 half)
  void* out2;         // GLU: kept u
  int n, m;           // outputs of a row and rows (GRAD with half: 2 half)
  int half, valid;    // GRAD: rows per matrix and those that exist; half 0: one matrix
  int act, bf16;      // output type
  int vec;            // four neighbours of a row are one aligned access
};

// The nearest BF16 values, as a pair with a's low (finite values that round past the largest
// become infinite).
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  typedef float v2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2{a, b}, v2bf));
}

// Value i of a pair.
__device__ __forceinline__ float head_of(uint32_t pair, int i) {
  return __uint_as_float(i ? pair & 0xffff0000u : pair << 16);
}

// Columns n .. n + 3 (those below e.n) of a row that starts at element `row`.
__device__ __forceinline__ void store4(const Epilogue& e, void* out, uint64_t row, int n,
                                       f32x4 v) {
  if (e.vec && n + 4 <= e.n) {
    if (e.bf16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + row + n) =
          make_uint2(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]));
    else
      *reinterpret_cast<f32x4*>(static_cast<float*>(out) + row + n) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= e.n) break;
    if (e.bf16)
      static_cast<uint16_t*>(out)[row + n + i] = (uint16_t)bf16_pair(v[i], 0.f);
    else
      static_cast<float*>(out)[row + n + i] = v[i];
  }
}

__device__ __forceinline__ f32x4 load4(const Epilogue& e, const void* p, int bf16, uint64_t row,
                                       int n) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (e.vec && n + 4 <= e.n) {
    if (!bf16) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + row + n);
    const uint2 b = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + row + n);
    return f32x4{__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u),
                 __uint_as_float(b.y << 16), __uint_as_float(b.y & 0xffff0000u)};
  }
  // n < e.n; loads past the row's end repeat its last value (unconditional, as in
  // k_pack_rows) and are not used
  if (bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = bf16_bits_to_f32(static_cast<const uint16_t*>(p)[row + min(n + i, e.n - 1)]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<const float*>(p)[row + min(n + i, e.n - 1)];
  }
  return v;
}

// What columns n .. n + 3 have in common over the rows.
struct Columns {
  f32x4 rs, rs2, bias;
};
template <int EPI>
__device__ __forceinline__ Columns load_columns(const Epilogue& e, int n) {
  Columns c{};
  if constexpr (EPI != EPI_GRAD) {
    if (e.rs) c.rs = load4(e, e.rs, 0, 0, n);
    if (EPI == EPI_GLU && e.rs) c.rs2 = load4(e, e.rs2, 0, 0, n);
    if (EPI == EPI_LINEAR && e.bias) c.bias = load4(e, e.bias, 0, 0, n);
  }
  return c;
}
// What a row adds to them, requested ahead of its use.
struct RowInputs {
  f32x4 res;
  float xs;
};
template <int EPI>
__device__ __forceinline__ RowInputs load_row(const Epilogue& e, int m, int n) {
  RowInputs r{};
  if constexpr (EPI != EPI_GRAD) {
    if (e.xs) r.xs = e.xs[m];
    if (EPI == EPI_LINEAR && e.res) r.res = load4(e, e.res, e.bf16, (uint64_t)m * e.n, n);
  }
  return r;
}

// Sums v (GLU: of gate, u of up) of row m < e.m, columns n .. n + 3 of which n < e.n.
template <int EPI>
__device__ __forceinline__ void finish(const Epilogue& e, const Columns& c, const RowInputs& in,
                                       int m, int n, f32x4 v, f32x4 u) {
  if constexpr (EPI == EPI_GRAD) {
    void* out = e.out;
    int r = m;
    if (e.half) {
      if (m >= e.half) {
        out = e.out1;
        r = m - e.half;
      }
      if (r >= e.valid) return;
    }
    store4(e, out, (uint64_t)r * e.n, n, v);
    return;
  }
  const uint64_t row = (uint64_t)m * e.n;
  if (e.xs) {
    v *= in.xs;
    if constexpr (EPI == EPI_GLU) u *= in.xs;
  }
  if (e.rs) {
    v *= c.rs;
    if constexpr (EPI == EPI_GLU) u *= c.rs2;
  }
  if constexpr (EPI == EPI_GLU) {
    f32x4 h;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = activate(e.act, v[i], u[i]);
    if (e.out1) {
      store4(e, e.out1, row, n, v);
      store4(e, e.out2, row, n, u);
    }
    store4(e, e.out, row, n, h);
  } else {
    if (e.bias) v += c.bias;
    if (e.act != K3_DENSE_ACT_NONE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = unary_activation(e.act, v[i]);
    }
    if (e.res) v += in.res;
    store4(e, e.out, row, n, v);
  }
}

// A whole wave's part of a tile where all of it exists and four neighbours are one access:
// a column or two of sums (16 rows each) at a time, with the next ones' residual on its way
// (sum after sum, it took 40 of 304 us at 4096 x 7168 x 6144; all of it ahead spilled).
// n0, m0: this lane's first column and row; a sum's are n0 + 16 i and m0 + 16 j.
template <int EPI, bool kBf16, bool kInt8, int FN, int FM>
__device__ __forceinline__ void finish_inside(const Epilogue& e, void* out, int n0, int m0,
                                              const f32x4 (&acc)[FN][FM]) {
  constexpr bool kGlu = EPI == EPI_GLU;
  constexpr int kOut = kGlu ? FN / 2 : FN;  // blocks of 16 outputs
  typedef typename std::conditional<kBf16, uint2, f32x4>::type Quad;  // four outputs
  auto store = [&](void* to, uint64_t at, f32x4 v) {
    if constexpr (kBf16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(to) + at) =
          make_uint2(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]));
    else
      *reinterpret_cast<f32x4*>(static_cast<float*>(to) + at) = v;
  };
  f32x4 rs[FN], bias[FN];
  if constexpr (EPI != EPI_GRAD) {
    const f32x4 ones = {1.f, 1.f, 1.f, 1.f}, none = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const int n = n0 + 16 * (kGlu ? i / 2 : i);
      rs[i] = kInt8 ? *reinterpret_cast<const f32x4*>((kGlu && i % 2 ? e.rs2 : e.rs) + n) : ones;
      bias[i] = !kGlu && e.bias ? *reinterpret_cast<const f32x4*>(e.bias + n) : none;
    }
  }
  constexpr bool kRes = EPI == EPI_LINEAR;
  constexpr int kCols = FN > 4 ? 1 : 2;  // columns at a time
  Quad res[2][kCols][kRes ? FN : 1];
  float xs[2][kCols];
  auto request = [&](int c) {  // of columns kCols c and behind
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      const int m = m0 + 16 * (kCols * c + k);
      if constexpr (EPI != EPI_GRAD) xs[c & 1][k] = e.xs ? e.xs[m] : 1.f;
      if constexpr (kRes) {
        if (e.res) {
#pragma unroll
          for (int i = 0; i < FN; ++i)
            res[c & 1][k][i] = *reinterpret_cast<const Quad*>(
                static_cast<const uint8_t*>(e.res) +
                ((uint64_t)m * e.n + n0 + 16 * i) * (kBf16 ? 2 : 4));
        }
      }
    }
  };
  request(0);
#pragma unroll
  for (int c = 0; c < FM / kCols; ++c) {
    if (c + 1 < FM / kCols) request(c + 1);
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      const int j = kCols * c + k;
      const uint64_t at = (uint64_t)(m0 + 16 * j) * e.n + n0;
#pragma unroll
      for (int i = 0; i < kOut; ++i) {
        if constexpr (EPI == EPI_GRAD) {
          store(out, at + 16 * i, acc[i][j]);
        } else if constexpr (kGlu) {
          f32x4 g = acc[2 * i][j] * xs[c & 1][k], u = acc[2 * i + 1][j] * xs[c & 1][k];
          if constexpr (kInt8) {
            g *= rs[2 * i];
            u *= rs[2 * i + 1];
          }
          f32x4 h;
#pragma unroll
          for (int q = 0; q < 4; ++q) h[q] = activate(e.act, g[q], u[q]);
          if (e.out1) {
            store(e.out1, at + 16 * i, g);
            store(e.out2, at + 16 * i, u);
          }
          store(out, at + 16 * i, h);
        } else {
          f32x4 v = acc[i][j] * xs[c & 1][k];
          if constexpr (kInt8) v *= rs[i];
          if (e.bias) v += bias[i];
          if (e.act != K3_DENSE_ACT_NONE) {
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = unary_activation(e.act, v[q]);
          }
          if (e.res) {
            const Quad r = res[c & 1][k][i];
            if constexpr (kBf16)
              v += f32x4{head_of(r.x, 0), head_of(r.x, 1), head_of(r.y, 0), head_of(r.y, 1)};
            else
              v += r;
          }
          store(out, at + 16 * i, v);
        }
      }
    }
  }
}

// part: [splits][m][pitch] sums of a split K, in place of the epilogue.  With GLU the
// pitch runs over blocks of 16 gate and 16 up columns.
template <int BN, int BM, int NWN, int NWM, int WL, int XL, int EPI>
__global__ __launch_bounds__(64 * NWN * NWM) void k_gemm(const GemmArgs a, const Epilogue e,
                                                         float* part, int pitch) {
  constexpr bool kGlu = EPI == EPI_GLU;
  typedef Core<BN, BM, NWN, NWM, WL, XL, kGlu> C;
  __shared__ __attribute__((aligned(16))) uint8_t lds[C::kLds];
  int tn, tm;
  tile_of(blockIdx.x, a.tiles_n, a.tiles_m, &tn, &tm);
  f32x4 acc[C::FN][C::FM];
  C::run(a, lds, tn, tm, blockIdx.y, acc);

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nw = tn * BN + (wave % NWN) * C::FN * 16;  // the wave's first (GLU: pair) column
  const int mw = tm * BM + (wave / NWN) * C::FM * 16;
  const int n0 = (kGlu && !part ? nw / 2 : nw) + 4 * (lane >> 4), m0 = mw + (lane & 15);
  if (part) {
#pragma unroll
    for (int j = 0; j < C::FM; ++j) {
      const int m = m0 + 16 * j;
      if (m >= a.m) continue;
      float* row = part + ((uint64_t)blockIdx.y * a.m + m) * pitch;
#pragma unroll
      for (int i = 0; i < C::FN; ++i)
        if (n0 + 16 * i < pitch) *reinterpret_cast<f32x4*>(row + n0 + 16 * i) = acc[i][j];
    }
    return;
  }
  constexpr int kBlocks = kGlu ? C::FN / 2 : C::FN;
  // the wave's rows in its matrix (the second of a gradient's two starts at row `half`)
  const bool second = EPI == EPI_GRAD && e.half && mw >= e.half;
  const int first = second ? mw - e.half : mw;
  const int rows = EPI == EPI_GRAD && e.half ? e.valid : e.m;
  if (e.vec && first + 16 * C::FM <= rows && (kGlu ? nw / 2 : nw) + 16 * kBlocks <= e.n) {
    void* out = second ? e.out1 : e.out;
    const int r0 = first + (lane & 15);
    if (e.bf16)
      finish_inside<EPI, true, WL == L_INT8>(e, out, n0, r0, acc);
    else
      finish_inside<EPI, false, WL == L_INT8>(e, out, n0, r0, acc);
    return;
  }
#pragma unroll
  for (int j = 0; j < C::FM; ++j) {
    const int m = m0 + 16 * j;
    if (m >= e.m) continue;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const int n = n0 + 16 * i;
      if (n >= e.n) continue;
      const Columns c = load_columns<EPI>(e, n);
      const RowInputs in = load_row<EPI>(e, m, n);
      if constexpr (kGlu)
        finish<EPI>(e, c, in, m, n, acc[2 * i][j], acc[2 * i + 1][j]);
      else
        finish<EPI>(e, c, in, m, n, acc[i][j], f32x4{});
    }
  }
}

// The splits' sums in order, then the epilogue: four columns of one row per thread.
template <int EPI>
__global__ __launch_bounds__(256) void k_gemm_join(const Epilogue e, const float* part, int splits,
                                                   int pitch) {
  const int quads = (e.n + 3) / 4;
  const uint64_t total = (uint64_t)e.m * quads;
  for (uint64_t t = blockIdx.x * 256ull + threadIdx.x; t < total; t += gridDim.x * 256ull) {
    const int m = (int)(t / quads), n = 4 * (int)(t % quads);
    const uint64_t at =
        (uint64_t)m * pitch + (EPI == EPI_GLU ? (uint32_t)(n >> 4) * 32 + (n & 15) : n);
    const Columns c = load_columns<EPI>(e, n);
    const RowInputs in = load_row<EPI>(e, m, n);
    f32x4 v = {0.f, 0.f, 0.f, 0.f}, u = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
      const float* p = part + (uint64_t)s * e.m * pitch + at;
      v += *reinterpret_cast<const f32x4*>(p);
      if constexpr (EPI == EPI_GLU) u += *reinterpret_cast<const f32x4*>(p + 16);
    }
    finish<EPI>(e, c, in, m, n, v, u);
  }
}

// ------------------------------------------------------------------ operand layout
// Nearest BF16 of a finite value (the largest finite one where that overflows), an
// infinity or a quiet NaN of the others.
__device__ __forceinline__ uint32_t nearest_bf16(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7f800000u) == 0x7f800000u)
    return (u >> 16) | ((u & 0x7fffffu) ? 0x40u : 0u);
  const uint32_t r = (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
  return (r & 0x7f80u) == 0x7f80u ? u >> 16 : r;
}

// Three BF16 terms of a and of b as pairs; only the first of an infinity or NaN.  The
// hardware's convert rounds values of the last half step under infinity to it: those take
// the slow way.
__device__ __forceinline__ void terms3(float a, float b, uint32_t (&t)[3]) {
  t[0] = bf16_pair(a, b);
  const float most = fmaxf(fabsf(a), fabsf(b));
  if (!(most < 0x1.fep+127f)) t[0] = nearest_bf16(a) | nearest_bf16(b) << 16;
  const float ra = fabsf(a) < INFINITY ? a - head_of(t[0], 0) : 0.f;
  const float rb = fabsf(b) < INFINITY ? b - head_of(t[0], 1) : 0.f;
  t[1] = bf16_pair(ra, rb);
  t[2] = bf16_pair(ra - head_of(t[1], 0), rb - head_of(t[1], 1));
}

// Eight neighbouring fp32 values of a row of `cols` from column 8 g, zeros past its end.
__device__ __forceinline__ void load_eight(const float* p, int g, int cols, bool aligned,
                                           float (&v)[8]) {
  const int c = 8 * g;
  if (aligned && c + 8 <= cols) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 q = *reinterpret_cast<const f32x4*>(p + c + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * h + i] = q[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float value = p[min(c + i, cols - 1)];  // unconditional, as in pack_rows
      v[i] = c + i < cols ? value : 0.f;
    }
  }
}

// The three terms of eight values to their planes, `plane` bytes apart.
__device__ __forceinline__ void store_terms(uint8_t* d, uint64_t plane, const float (&v)[8],
                                            float scale) {
  u32x4 t[3];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t p[3];
    terms3(v[2 * q] * scale, v[2 * q + 1] * scale, p);
#pragma unroll
    for (int i = 0; i < 3; ++i) t[i][q] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) *reinterpret_cast<u32x4*>(d + i * plane) = t[i];
}

// fp32 rows to three planes [3][rows][pitch / 2] (pitch in bytes, zeros past cols), scaled by
// the power of two that brings the row's largest finite value into [1, 2), whose inverse
// goes to xs[row].  A thread takes eight neighbouring values at a time, kHeld such groups of
// a row in registers between the search for the largest and the split (rows of up to 8192
// values are read once).
constexpr int kHeld = 4;
__global__ __launch_bounds__(256) void k_split_rows(const float* __restrict__ x,
                                                    uint8_t* __restrict__ planes,
                                                    float* __restrict__ xs, int rows, int cols,
                                                    uint32_t pitch, int aligned) {
  const uint64_t plane = (uint64_t)rows * pitch;
  __shared__ float red[4];
  const int groups = (int)(pitch / 16);
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const float* p = x + (uint64_t)row * cols;
    float held[kHeld][8];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int g = threadIdx.x + 256 * k;
      if (g < groups) load_eight(p, g, cols, aligned, held[k]);
    }
    float most = 0.f;
    auto see = [&](const float (&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = fabsf(v[i]);
        most = a < INFINITY ? fmaxf(most, a) : most;
      }
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if ((int)threadIdx.x + 256 * k < groups) see(held[k]);
    for (int g = threadIdx.x + 256 * kHeld; g < groups; g += 256) {
      float v[8];
      load_eight(p, g, cols, aligned, v);
      see(v);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    __syncthreads();  // red of the row before
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    // exponents -126 .. 126, so that the scale and its inverse are normal numbers
    const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -126), 126);
    const float scale = most > 0.f ? __uint_as_float((uint32_t)(127 - e) << 23) : 1.f;
    if (threadIdx.x == 0)
      xs[row] = most > 0.f ? __uint_as_float((uint32_t)(127 + e) << 23) : 1.f;
    uint8_t* d = planes + (uint64_t)row * pitch;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int g = threadIdx.x + 256 * k;
      if (g < groups) store_terms(d + 16ull * g, plane, held[k], scale);
    }
    for (int g = threadIdx.x + 256 * kHeld; g < groups; g += 256) {
      float v[8];
      load_eight(p, g, cols, aligned, v);
      store_terms(d + 16ull * g, plane, v, scale);
    }
  }
}

// fp32 rows to three planes [3][rows_out][pitch / 2] as they are, zeros behind each and in
// the rows from `rows` on.
__device__ __forceinline__ void term_rows(const float* __restrict__ x, uint8_t* __restrict__ planes,
                                          int rows, int cols, int rows_out, uint32_t pitch,
                                          bool aligned, uint32_t block, uint32_t blocks) {
  const uint32_t groups = pitch / 16;
  const uint64_t total = (uint64_t)rows_out * groups, plane = (uint64_t)rows_out * pitch;
  for (uint64_t t = block * 256ull + threadIdx.x; t < total; t += blocks * 256ull) {
    const uint64_t row = t / groups;
    float v[8];
    load_eight(x + min(row, (uint64_t)rows - 1) * cols, (int)(t - row * groups), cols, aligned, v);
    if (row >= (uint64_t)rows) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
    store_terms(planes + 16 * t, plane, v, 1.f);
  }
}

// Rows to rows of `pitch` bytes (a multiple of 16), zeros behind each and in the rows from
// `rows` to rows_out.
template <typename T>
__device__ __forceinline__ void pack_rows(const T* __restrict__ src, u32x4* __restrict__ dst,
                                          int rows, int cols, int rows_out, uint32_t pitch,
                                          uint32_t block, uint32_t blocks) {
  constexpr int kPer = 16 / (int)sizeof(T);
  const uint32_t chunks = pitch / 16;
  const uint64_t total = (uint64_t)rows_out * chunks;
  for (uint64_t t = block * 256ull + threadIdx.x; t < total; t += blocks * 256ull) {
    const uint64_t row = t / chunks;
    const int c0 = row < (uint64_t)rows ? (int)(t - row * chunks) * kPer : cols;
    const T* p = src + min(row, (uint64_t)rows - 1) * cols;
    u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      // (loads past the end repeat the last value: behind a condition each would wait for
      // the one before)
      const uint32_t value = p[min(c0 + i, cols - 1)];
      const uint32_t b = c0 + i < cols ? value : 0u;
      v[i * (int)sizeof(T) / 4] |= b << (8 * ((i * (int)sizeof(T)) & 3));
    }
    dst[t] = v;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_pack_rows(const T* __restrict__ src, u32x4* __restrict__ dst,
                                                   int rows, int cols, int rows_out,
                                                   uint32_t pitch) {
  pack_rows<T>(src, dst, rows, cols, rows_out, pitch, blockIdx.x, gridDim.x);
}

// dg = grad f_g(g, u) and du = grad f_u(g, u) of [rows][cols] values as BF16 planes
// [terms][rows_out][2 half]: dg at columns [0, cols), du at [half, half + cols), zeros in the
// rest; half is a multiple of 8.  One term rounds to BF16, three keep all 24 bits.
__device__ __forceinline__ float widen(uint16_t b) { return bf16_bits_to_f32(b); }
__device__ __forceinline__ float widen(float f) { return f; }

// The first W values from p, n of which exist (n < 1: p is any value, none counts).
template <typename T, int W>
__device__ __forceinline__ void load_row_part(const T* p, bool vec, int n, float (&v)[W]) {
  if (W == 8 && vec && n >= 8) {
    constexpr int kPer = 16 / (int)sizeof(T);
#pragma unroll
    for (int h = 0; h < W / kPer; ++h) {
      const u32x4 q = *reinterpret_cast<const u32x4*>(p + kPer * h);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        v[kPer * h + i] = sizeof(T) == 4 ? __uint_as_float(q[i % 4])
                                         : head_of(q[i / 2 % 4], i % 2);
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float value = widen(p[max(min(i, n - 1), 0)]);  // unconditional, as in pack_rows
      v[i] = i < n ? value : 0.f;
    }
  }
}

// W neighbouring columns per thread: eight, or two where eight would leave the card to a few
// waves that each go through eight sets of exponentials (517 x 1003 fp32 12 us of 105).
template <typename T, int TERMS, int W>
__device__ __forceinline__ void gated_grad(const T* __restrict__ g, const T* __restrict__ u,
                                           const T* __restrict__ grad,
                                           uint16_t* __restrict__ planes, int rows, int cols,
                                           int rows_out, int half, int act, int vec,
                                           uint32_t block, uint32_t blocks) {
  const uint64_t plane = (uint64_t)rows_out * 2 * half;
  const uint32_t groups = (uint32_t)half / W;
  const uint64_t total = (uint64_t)rows_out * groups;
  for (uint64_t t = block * 256ull + threadIdx.x; t < total; t += blocks * 256ull) {
    const uint64_t row = t / groups;
    const int c = W * (int)(t - row * groups);
    const int n = row < (uint64_t)rows ? cols - c : 0;
    const uint64_t at = n > 0 ? row * cols + c : 0;
    float gv[W], uv[W], dv[W];
    load_row_part<T, W>(g + at, vec, n, gv);
    load_row_part<T, W>(u + at, vec, n, uv);
    load_row_part<T, W>(grad + at, vec, n, dv);
    uint32_t og[TERMS][W / 2], ou[TERMS][W / 2];
    float dg[W], du[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      dg[i] = du[i] = 0.f;
      if (i < n) {
        const float sig = 1.0f / (1.0f + expf(-gv[i]));
        if (act == K3_ACT_SILU) {
          dg[i] = dv[i] * uv[i] * (sig * (1.0f + gv[i] * (1.0f - sig)));
          du[i] = dv[i] * (gv[i] * sig);
        } else {
          const float a = tanhf(gv[i] / 4.0f), b = tanhf(uv[i] / 25.0f);
          dg[i] = dv[i] * (25.0f * b) * ((1.0f - a * a) * sig + 4.0f * a * (sig * (1.0f - sig)));
          du[i] = dv[i] * (4.0f * a * sig) * (1.0f - b * b);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < W / 2; ++q) {
      uint32_t tg[3], tu[3];
      if constexpr (TERMS == 1) {
        tg[0] = bf16_pair(dg[2 * q], dg[2 * q + 1]);
        tu[0] = bf16_pair(du[2 * q], du[2 * q + 1]);
      } else {
        terms3(dg[2 * q], dg[2 * q + 1], tg);
        terms3(du[2 * q], du[2 * q + 1], tu);
      }
#pragma unroll
      for (int k = 0; k < TERMS; ++k) {
        og[k][q] = tg[k];
        ou[k][q] = tu[k];
      }
    }
    uint16_t* o = planes + row * 2 * half + c;
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
      if constexpr (W == 8) {
        *reinterpret_cast<u32x4*>(o + k * plane) = u32x4{og[k][0], og[k][1], og[k][2], og[k][3]};
        *reinterpret_cast<u32x4*>(o + k * plane + half) =
            u32x4{ou[k][0], ou[k][1], ou[k][2], ou[k][3]};
      } else {
        *reinterpret_cast<uint32_t*>(o + k * plane) = og[k][0];
        *reinterpret_cast<uint32_t*>(o + k * plane + half) = ou[k][0];
      }
    }
  }
}

// Everything that the gradient's products read and is not in place yet, in one launch of
// workgroups with a job each: dg and du, copies of the gate, the up matrix and the
// activations.  One by one the four filled and drained the card for 4 to 8 us each (517
// rows of 1003 x 2050 in fp32: 23 us together, in one launch 12).
struct CopyJob {
  const void* src;
  uint8_t* dst;
  int rows, cols, rows_out;
  uint32_t pitch;
  uint32_t blocks;  // 0: in place already
};
struct GradJob {
  const void *g, *u, *grad;
  uint16_t* planes;
  int rows, cols, rows_out, half, act, vec;
  uint32_t blocks;
};
template <typename T, int TERMS, int W>
__global__ __launch_bounds__(256) void k_gated_grad(const GradJob d, const CopyJob gate,
                                                    const CopyJob up, const CopyJob x,
                                                    int x_aligned) {
  uint32_t block = blockIdx.x;
  if (block < d.blocks) {
    gated_grad<T, TERMS, W>(static_cast<const T*>(d.g), static_cast<const T*>(d.u),
                            static_cast<const T*>(d.grad), d.planes, d.rows, d.cols, d.rows_out,
                            d.half, d.act, d.vec, block, d.blocks);
    return;
  }
  block -= d.blocks;
  if (block < x.blocks) {
    if constexpr (TERMS == 3)
      term_rows(static_cast<const float*>(x.src), x.dst, x.rows, x.cols, x.rows_out, x.pitch,
                x_aligned, block, x.blocks);
    else
      pack_rows<uint16_t>(static_cast<const uint16_t*>(x.src), reinterpret_cast<u32x4*>(x.dst),
                          x.rows, x.cols, x.rows_out, x.pitch, block, x.blocks);
    return;
  }
  block -= x.blocks;
  const bool second = block >= gate.blocks;
  const CopyJob& w = second ? up : gate;
  if (second) block -= gate.blocks;
  pack_rows<uint16_t>(static_cast<const uint16_t*>(w.src), reinterpret_cast<u32x4*>(w.dst), w.rows,
                      w.cols, w.rows_out, w.pitch, block, w.blocks);
}

// ------------------------------------------------------------------ host
bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
uint64_t align256(uint64_t v) { return (v + 255) & ~255ull; }
uint32_t round_up(uint32_t v, uint32_t to) { return (v + to - 1) / to * to; }

// Scratch memory in the order of its taking.
struct Scratch {
  uint8_t* base;
  uint64_t used = 0;
  explicit Scratch(void* p) : base(static_cast<uint8_t*>(p)) {}
  uint8_t* take(uint64_t bytes) {
    uint8_t* p = base ? base + used : nullptr;
    used += align256(bytes);
    return p;
  }
};

unsigned grid_for(uint64_t threads) {
  return (unsigned)std::min<uint64_t>((threads + 255) / 256, 1u << 16);
}

int launched_or(TimedLaunch& tl, const char* what) {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return K3_SPINE_OK;
  tl.failed();
  return spine_fail(K3_SPINE_E_RUNTIME, "%s: %s", what, hipGetErrorString(err));
}

int launch_pack_rows(const void* src, void* dst, int elem, int rows, int cols, int rows_out,
              uint32_t pitch, hipStream_t st) {
  TimedLaunch tl(KC_SPLIT, st);
  const unsigned grid = grid_for((uint64_t)rows_out * (pitch / 16));
  if (elem == 2)
    launch_timed(tl, k_pack_rows<uint16_t>, dim3(grid), dim3(256), 0, st,
                 static_cast<const uint16_t*>(src), static_cast<u32x4*>(dst), rows, cols, rows_out,
                 pitch);
  else
    launch_timed(tl, k_pack_rows<uint8_t>, dim3(grid), dim3(256), 0, st,
                 static_cast<const uint8_t*>(src), static_cast<u32x4*>(dst), rows, cols, rows_out,
                 pitch);
  return launched_or(tl, "dense operand layout");
}

int launch_split_rows(const void* x, void* planes, float* xs, int rows, int cols, uint32_t pitch,
                      hipStream_t st) {
  TimedLaunch tl(KC_SPLIT, st);
  launch_timed(tl, k_split_rows, dim3((unsigned)std::min(rows, 1 << 16)), dim3(256), 0, st,
               static_cast<const float*>(x), static_cast<uint8_t*>(planes), xs, rows, cols, pitch,
               (int)(cols % 4 == 0 && aligned16(x)));
  return launched_or(tl, "dense activation terms");
}

// Operands that are laid out anew get a K of whole steps where K runs over their rows
// (`along`), zeros in the added ones: the rest of K that is no whole step is the slow part
// of a product.

// A matrix as an operand: in place where its rows are whole 16-byte pieces, else a
// copy of it with rows that are.
struct Matrix {
  const void* src;
  int elem, rows, cols, rows_out;
  uint32_t pitch;
  uint8_t* copy = nullptr;  // scratch of the copy
  bool copied;
  Matrix(const void* p, int elem_, int rows_, int cols_, bool along, Scratch& s)
      : src(p), elem(elem_), rows(rows_), cols(cols_), rows_out(rows_) {
    pitch = round_up((uint32_t)cols * elem, 16);
    copied = pitch != (uint32_t)cols * elem || !aligned16(p);
    if (!copied) return;
    if (along) rows_out = (int)round_up((uint32_t)rows, kStep);
    copy = s.take((uint64_t)rows_out * pitch);
  }
  const uint8_t* data() const { return copied ? copy : static_cast<const uint8_t*>(src); }
  int fill(hipStream_t st) const {
    return copied ? launch_pack_rows(src, copy, elem, rows, cols, rows_out, pitch, st) : K3_SPINE_OK;
  }
  CopyJob job() const {
    const uint32_t blocks = copied ? grid_for((uint64_t)rows_out * (pitch / 16)) : 0;
    return CopyJob{src, copy, rows, cols, rows_out, pitch, blocks};
  }
};

// Activation rows as operand planes: bf16 rows as a Matrix, fp32 rows split.
struct Activation {
  const void* src;
  bool f32;
  int rows, cols, rows_out;
  uint32_t pitch;
  uint8_t* planes = nullptr;
  float* xs = nullptr;
  bool copied = false;
  Activation(const void* p, int dtype, int rows_, int cols_, bool scaled, bool along, Scratch& s)
      : src(p), f32(dtype == K3_DTYPE_F32), rows(rows_), cols(cols_), rows_out(rows_) {
    pitch = round_up((uint32_t)cols * 2, 16);
    copied = f32 || pitch != (uint32_t)cols * 2 || !aligned16(p);
    if (!copied) return;
    if (along) rows_out = (int)round_up((uint32_t)rows, kStep);
    planes = s.take((uint64_t)terms() * rows_out * pitch);
    if (f32 && scaled) xs = reinterpret_cast<float*>(s.take(4ull * rows));
  }
  int terms() const { return f32 ? 3 : 1; }
  const uint8_t* plane(int t) const {
    if (!copied) return static_cast<const uint8_t*>(src);
    return planes + (uint64_t)t * rows_out * pitch;
  }
  int fill(hipStream_t st) const {
    if (f32) return launch_split_rows(src, planes, xs, rows, cols, pitch, st);
    return copied ? launch_pack_rows(src, planes, 2, rows, cols, rows_out, pitch, st) : K3_SPINE_OK;
  }
  CopyJob job() const {
    const uint32_t blocks = copied ? grid_for((uint64_t)rows_out * (pitch / 16)) : 0;
    return CopyJob{src, planes, rows, cols, rows_out, pitch, blocks};
  }
};

// Tiles and the split of K.
struct Plan {
  int bn, bm;  // rows of the matrix and positions of a tile
  int tiles_n, tiles_m, splits, per, pitch;
  double us;  // its estimated time
  float* part;
};

// The tile and the split of K with the smallest estimated time.  One workgroup fills a CU,
// so tiles run in rounds of as many as there are CUs; a round costs its steps, more for a
// larger tile though less per output, and about six microseconds around them; a split K
// costs writing and reading its partial sums and a launch.  Microseconds a step, measured
// on products that fill the card.  224 rows serve products that leave the last round of
// 256 half empty (4096 x 7168 outputs: 448 tiles of 256, 512 of 224, on 256 CUs; the
// gated block's pairs of 16 rows need an even number of blocks per wave and do without).
// 128 x 128 tiles, two on a CU, took 1.1 us for twice that output and lost to 256 x 128 at
// every size tried (7168 x 6144 int8 at 1024 positions 106 against 92 us; 256 x 256 in two
// splits 97).
Plan plan_product(int n, int m, int steps, bool glu, Scratch& s) {
  struct Shape {
    int bn, bm;
    double us;
  };
  static const Shape kShapes[] = {{256, 256, 1.6}, {256, 128, 0.93}, {224, 256, 1.44}};
  const int cols = glu ? (int)round_up((uint32_t)n, 16) * 2 : n;
  const int cus = std::max(1, device_cu_count());
  steps = std::max(steps, 1);
  Plan p{};
  double best = 0;
  for (const Shape& t : kShapes) {
    if (glu && t.bn == 224) continue;
    const int64_t tiles = (int64_t)((cols + t.bn - 1) / t.bn) * ((m + t.bm - 1) / t.bm);
    for (int want = 1; want <= 32 && (want == 1 || want * 4 <= steps); ++want) {
      const int per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
      const double rounds = (double)((tiles * splits + cus - 1) / cus);
      double us = rounds * (per * t.us + 6.0);
      if (splits > 1) us += 4.0 + 8.0 * splits * (double)m * cols / 5e6;
      if (best != 0 && us >= best) continue;
      p.us = best = us;
      p.bn = t.bn;
      p.bm = t.bm;
      p.per = per;
      p.splits = splits;
    }
  }
  p.tiles_n = (cols + p.bn - 1) / p.bn;
  p.tiles_m = (m + p.bm - 1) / p.bm;
  p.pitch = (int)round_up((uint32_t)cols, 4);
  if (p.splits > 1) p.part = reinterpret_cast<float*>(s.take(4ull * p.splits * m * p.pitch));
  return p;
}

template <int WL, int XL, int EPI>
int product(GemmArgs a, const Epilogue& e, const Plan& p, const char* what, hipStream_t st) {
  a.tiles_n = p.tiles_n;
  a.tiles_m = p.tiles_m;
  a.splits = p.splits;
  a.per = p.per;
  const uint64_t tiles = (uint64_t)p.tiles_n * p.tiles_m;
  if (tiles > UINT32_MAX / 512 || p.splits > 65535)
    return spine_fail(K3_SPINE_E_INVALID, "%s: too many output tiles", what);
  {
    TimedLaunch tl(KC_SPINE_MFMA, st);
    const dim3 grid((unsigned)tiles, (unsigned)p.splits);
    float* part = p.splits > 1 ? p.part : nullptr;
    if (p.bn == 224) {
      if constexpr (EPI != EPI_GLU)
        launch_timed(tl, (k_gemm<224, 256, 2, 4, WL, XL, EPI>), grid, dim3(512), 0, st, a, e, part,
                     p.pitch);
    } else if (p.bm == 256) {
      launch_timed(tl, (k_gemm<256, 256, 4, 2, WL, XL, EPI>), grid, dim3(512), 0, st, a, e, part,
                   p.pitch);
    } else {
      launch_timed(tl, (k_gemm<256, 128, 4, 2, WL, XL, EPI>), grid, dim3(512), 0, st, a, e, part,
                   p.pitch);
    }
    const int rc = launched_or(tl, what);
    if (rc != K3_SPINE_OK) return rc;
  }
  if (p.splits == 1) return K3_SPINE_OK;
  TimedLaunch tl(KC_COMBINE, st);
  launch_timed(tl, k_gemm_join<EPI>, dim3(grid_for((uint64_t)e.m * ((e.n + 3) / 4))), dim3(256), 0,
               st, e, p.part, p.splits, p.pitch);
  return launched_or(tl, what);
}

int steps_of(int k) { return k / kStep; }  // whole ones

bool vec_ok(int n, int out_elem, std::initializer_list<const void*> ptrs) {
  if (n % 4 != 0) return false;
  for (const void* p : ptrs)
    if (((uintptr_t)p & 15u) != 0) return false;
  (void)out_elem;
  return true;
}

// Few positions: the skinny kernels stream a matrix once per 16 positions with no scratch
// memory and no second launch.  Up to 16 positions they always win; beyond, where their
// time, about 0.22 us (fp32 rows: 0.3) per million weights and 16 positions behind a
// launch, is under the tiles': us on skinny / tiled kernels 7168 x 2048 bf16 at 32 positions
// 9.9 / 14.4 and at 128 27 / 19, fp32 rows 12 / 23 and 40 / 33; 7168 x 6144 fp32 rows at 32
// positions 27 / 41 and at 64 51 / 43; 1024 x 1024 at 128 positions 9.8 / 12.8.
constexpr int kSkinnyAlways = 16, kSkinnyMost = 512;
bool skinny_pays(int n, int m, int k, int x_dtype, bool glu) {
  if (m <= kSkinnyAlways) return true;
  if (m > kSkinnyMost) return false;
  const bool f32 = x_dtype == K3_DTYPE_F32;
  const double weights = (double)n * k * (glu ? 2 : 1) * 1e-6;
  const double skinny = 8.0 + (f32 ? 0.30 : 0.22) * weights * ((m + 15) / 16);
  Scratch none(nullptr);
  return skinny <= plan_product(n, m, (f32 ? 3 : 1) * steps_of(k), glu, none).us + (f32 ? 4.0 : 0.0);
}
bool skinny_linear(const K3HipLinearV1& op, SkinnyOp* sk) {
  if (op.positions > kSkinnyMost) return false;
  sk->kind = op.matrix_kind == K3_SPINE_MATRIX_INT8 ? SKINNY_INT8 : SKINNY_BF16;
  sk->w = op.weights;
  sk->row_scales = op.row_scales;
  sk->x = op.x;
  sk->x_dtype = (int)op.x_dtype;
  sk->y = op.out;
  sk->bias = op.bias;
  sk->unary = (int)op.activation;
  sk->add = op.residual;
  sk->add_bf16 = sk->out_bf16 = op.out_dtype == K3_DTYPE_BF16;
  sk->rows = (int)op.rows;
  sk->cols = (int)op.columns;
  sk->positions = (int)op.positions;
  return skinny_fits(*sk) && skinny_pays(sk->rows, sk->positions, sk->cols, sk->x_dtype, false);
}
bool skinny_gated(const K3HipGatedV1& op, SkinnyOp* sk) {
  if (op.positions > kSkinnyMost) return false;
  sk->kind = op.matrix_kind == K3_SPINE_MATRIX_INT8 ? SKINNY_INT8 : SKINNY_BF16;
  sk->w = op.gate;
  sk->w2 = op.up;
  sk->row_scales = op.gate_scales;
  sk->row_scales2 = op.up_scales;
  sk->act = (int)op.activation;
  sk->x = op.x;
  sk->x_dtype = (int)op.x_dtype;
  sk->y = op.out;
  sk->keep_gate = op.out_gate;
  sk->keep_up = op.out_up;
  sk->out_bf16 = op.out_dtype == K3_DTYPE_BF16;
  sk->rows = (int)op.rows;
  sk->cols = (int)op.columns;
  sk->positions = (int)op.positions;
  return skinny_fits(*sk) && skinny_pays(sk->rows, sk->positions, sk->cols, sk->x_dtype, true);
}
int run_skinny(const SkinnyOp& sk, const char* what, hipStream_t st) {
  if (launch_skinny(sk, KC_SPINE_MFMA, st) == K3_HIP_OK) return K3_SPINE_OK;
  return spine_fail(K3_SPINE_E_RUNTIME, "%s: %s", what, k3_hip_last_error());
}

struct LinearCall {
  Scratch s;
  Matrix w;
  Activation x;
  Plan p;
  LinearCall(const K3HipLinearV1& op, void* ws)
      : s(ws),
        w(op.weights, op.matrix_kind == K3_SPINE_MATRIX_INT8 ? 1 : 2, (int)op.rows,
          (int)op.columns, false, s),
        x(op.x, (int)op.x_dtype, (int)op.positions, (int)op.columns, true, false, s),
        p(plan_product((int)op.rows, (int)op.positions, x.terms() * steps_of((int)op.columns),
                       false, s)) {}
};

struct GatedCall {
  Scratch s;
  Matrix g, u;
  Activation x;
  Plan p;
  GatedCall(const K3HipGatedV1& op, void* ws)
      : s(ws),
        g(op.gate, op.matrix_kind == K3_SPINE_MATRIX_INT8 ? 1 : 2, (int)op.rows, (int)op.columns,
          false, s),
        u(op.up, g.elem, g.rows, g.cols, false, s),
        x(op.x, (int)op.x_dtype, (int)op.positions, (int)op.columns, true, false, s),
        p(plan_product((int)op.rows, (int)op.positions, x.terms() * steps_of((int)op.columns),
                       true, s)) {}
};

// The products of the gradient: d_x over the 2 terms() segments of (dg, gate) and
// (du, up), and both weight gradients as one product of 2 half rows.  dg and du are written
// here, so their rows and columns can be whole steps of either product's K; whether a K
// is follows from the other operand (k_x, k_w).
struct GradCall {
  Scratch s;
  Matrix g, u;
  Activation x;
  int half, terms, rows_out, k_x, k_w;
  uint16_t* planes;
  Plan px, pw;
  GradCall(const K3HipGatedGradV1& op, void* ws)
      : s(ws),
        g(op.gate, 2, (int)op.rows, (int)op.columns, true, s),
        u(op.up, 2, (int)op.rows, (int)op.columns, true, s),
        x(op.x, (int)op.dtype, (int)op.positions, (int)op.columns, false, true, s),
        half((int)round_up(op.rows, g.rows_out == u.rows_out && g.rows_out % kStep == 0 ? kStep : 8)),
        terms(x.terms()),
        rows_out(x.rows_out),
        k_x(std::min(g.rows_out, u.rows_out)),
        k_w(x.rows_out),
        planes(reinterpret_cast<uint16_t*>(s.take(4ull * terms * rows_out * half))),
        px(plan_product((int)op.columns, (int)op.positions, 2 * terms * steps_of(k_x), false, s)),
        pw(plan_product((int)op.columns, 2 * half, (terms == 3 ? 6 : 1) * steps_of(k_w), false,
                        s)) {}
};

}  // namespace

uint64_t dense_linear_workspace(const K3HipLinearV1& op) {
  SkinnyOp sk{};
  if (skinny_linear(op, &sk)) return K3_DENSE_NO_WORKSPACE;
  return K3_DENSE_NO_WORKSPACE + LinearCall(op, nullptr).s.used;
}
uint64_t dense_gated_workspace(const K3HipGatedV1& op) {
  SkinnyOp sk{};
  if (skinny_gated(op, &sk)) return K3_DENSE_NO_WORKSPACE;
  return K3_DENSE_NO_WORKSPACE + GatedCall(op, nullptr).s.used;
}
uint64_t dense_gated_grad_workspace(const K3HipGatedGradV1& op) {
  return K3_DENSE_NO_WORKSPACE + GradCall(op, nullptr).s.used;
}

int dense_linear(const K3HipLinearV1& op, void* ws, hipStream_t st) {
  SkinnyOp sk{};
  if (skinny_linear(op, &sk)) return run_skinny(sk, "linear", st);
  const LinearCall c(op, ws);
  int rc = c.w.fill(st);
  if (rc == K3_SPINE_OK) rc = c.x.fill(st);
  if (rc != K3_SPINE_OK) return rc;
  const bool int8 = op.matrix_kind == K3_SPINE_MATRIX_INT8;
  GemmArgs a{};
  a.segments = c.x.terms();
  for (int t = 0; t < a.segments; ++t) {
    a.w[t] = c.w.data();
    a.x[t] = c.x.plane(a.segments - 1 - t);  // the small terms first
  }
  a.n = (int)op.rows;
  a.m = (int)op.positions;
  a.k = (int)op.columns;
  a.ldw = c.w.pitch;
  a.kw = (int)(c.w.pitch / c.w.elem);
  a.ldx = c.x.pitch;
  a.kx = (int)(c.x.pitch / 2);
  Epilogue e{};
  e.rs = int8 ? op.row_scales : nullptr;
  e.bias = op.bias;
  e.xs = c.x.xs;
  e.res = op.residual;
  e.out = op.out;
  e.n = a.n;
  e.m = a.m;
  e.act = (int)op.activation;
  e.bf16 = op.out_dtype == K3_DTYPE_BF16;
  e.vec = vec_ok(a.n, 0, {e.rs, op.bias, op.residual, op.out});
  return int8 ? product<L_INT8, L_KMAJOR, EPI_LINEAR>(a, e, c.p, "linear", st)
              : product<L_KMAJOR, L_KMAJOR, EPI_LINEAR>(a, e, c.p, "linear", st);
}

int dense_gated(const K3HipGatedV1& op, void* ws, hipStream_t st) {
  SkinnyOp sk{};
  if (skinny_gated(op, &sk)) return run_skinny(sk, "gated feed-forward", st);
  const GatedCall c(op, ws);
  int rc = c.g.fill(st);
  if (rc == K3_SPINE_OK) rc = c.u.fill(st);
  if (rc == K3_SPINE_OK) rc = c.x.fill(st);
  if (rc != K3_SPINE_OK) return rc;
  const bool int8 = op.matrix_kind == K3_SPINE_MATRIX_INT8;
  GemmArgs a{};
  a.segments = c.x.terms();
  for (int t = 0; t < a.segments; ++t) {
    a.w[t] = c.g.data();
    a.w2[t] = c.u.data();
    a.x[t] = c.x.plane(a.segments - 1 - t);
  }
  a.n = (int)op.rows;
  a.m = (int)op.positions;
  a.k = (int)op.columns;
  a.ldw = c.g.pitch;
  a.kw = (int)(c.g.pitch / c.g.elem);
  a.ldx = c.x.pitch;
  a.kx = (int)(c.x.pitch / 2);
  Epilogue e{};
  e.rs = int8 ? op.gate_scales : nullptr;
  e.rs2 = int8 ? op.up_scales : nullptr;
  e.xs = c.x.xs;
  e.out = op.out;
  e.out1 = op.out_gate;
  e.out2 = op.out_up;
  e.n = a.n;
  e.m = a.m;
  e.act = (int)op.activation;
  e.bf16 = op.out_dtype == K3_DTYPE_BF16;
  e.vec = vec_ok(a.n, 0, {e.rs, e.rs2, op.out, op.out_gate, op.out_up});
  return int8 ? product<L_INT8, L_KMAJOR, EPI_GLU>(a, e, c.p, "gated feed-forward", st)
              : product<L_KMAJOR, L_KMAJOR, EPI_GLU>(a, e, c.p, "gated feed-forward", st);
}

int dense_gated_grad(const K3HipGatedGradV1& op, void* ws, hipStream_t st) {
  const GradCall c(op, ws);
  const char* what = "gated feed-forward gradient";
  const bool f32 = op.dtype == K3_DTYPE_F32;
  const int P = (int)op.positions, S = (int)op.rows, H = (int)op.columns;
  int rc;
  {
    TimedLaunch tl(KC_ACTIVATE, st);
    const uint64_t eights = (uint64_t)c.rows_out * (c.half / 8);
    const bool wide = eights >= 1024ull * std::max(1, device_cu_count());
    const int vec = ((uint64_t)S * (f32 ? 4 : 2)) % 16 == 0 && aligned16(op.g) &&
                    aligned16(op.u) && aligned16(op.grad);
    const GradJob d{op.g, op.u, op.grad, c.planes, P, S, c.rows_out, c.half, (int)op.activation,
                    vec, grid_for(wide ? eights : 4 * eights)};
    const CopyJob gate = c.g.job(), up = c.u.job(), x = c.x.job();
    const int x_aligned = H % 4 == 0 && aligned16(op.x);
    const dim3 grid(d.blocks + x.blocks + gate.blocks + up.blocks);
    auto go = [&](auto kernel) {
      launch_timed(tl, kernel, grid, dim3(256), 0, st, d, gate, up, x, x_aligned);
    };
    if (f32)
      wide ? go(k_gated_grad<float, 3, 8>) : go(k_gated_grad<float, 3, 2>);
    else
      wide ? go(k_gated_grad<uint16_t, 1, 8>) : go(k_gated_grad<uint16_t, 1, 2>);
    if ((rc = launched_or(tl, what)) != K3_SPINE_OK) return rc;
  }
  const uint32_t ldd = 4u * (uint32_t)c.half;  // bytes of a row of dg and du
  auto plane = [&](int t, int which) {
    return reinterpret_cast<const uint8_t*>(c.planes) + (uint64_t)t * c.rows_out * ldd +
           2ull * which * c.half;
  };
  GemmArgs a{};
  for (int t = c.terms - 1; t >= 0; --t)
    for (int which = 0; which < 2; ++which) {
      a.w[a.segments] = which ? c.u.data() : c.g.data();
      a.x[a.segments] = plane(t, which);
      ++a.segments;
    }
  a.n = H;
  a.m = P;
  a.k = a.kw = c.k_x;
  a.kx = c.half;
  a.ldw = c.g.pitch;
  a.ldx = ldd;
  Epilogue e{};
  e.out = op.d_x;
  e.n = H;
  e.m = P;
  e.bf16 = !f32;
  e.vec = vec_ok(H, 0, {op.d_x});
  rc = product<L_NMAJOR, L_KMAJOR, EPI_GRAD>(a, e, c.px, what, st);
  if (rc != K3_SPINE_OK) return rc;

  // term pairs (of dg / du, of x), the small products first
  static const int kPairs[6][2] = {{0, 2}, {2, 0}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};
  GemmArgs b{};
  b.segments = f32 ? 6 : 1;
  for (int i = 0; i < b.segments; ++i) {
    const int* t = kPairs[f32 ? i : 5];
    b.x[i] = plane(t[0], 0);
    b.w[i] = c.x.plane(t[1]);
  }
  b.n = H;
  b.m = 2 * c.half;
  b.k = b.kw = b.kx = c.k_w;
  b.ldw = c.x.pitch;
  b.ldx = ldd;
  Epilogue f{};
  f.out = op.d_gate;
  f.out1 = op.d_up;
  f.n = H;
  f.m = 2 * c.half;
  f.half = c.half;
  f.valid = S;
  f.bf16 = !f32;
  f.vec = vec_ok(H, 0, {op.d_gate, op.d_up});
  return product<L_NMAJOR, L_NMAJOR, EPI_GRAD>(b, f, c.pw, what, st);
}

}  // namespace k3
