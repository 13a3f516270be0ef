// Item tables in 4 bits and their products with a few users' rows, gfx950.
//
// A table of n rows of k values is held as E2M1 codes (sign, two exponent bits, one mantissa
// bit: 0, .5, 1, 1.5, 2, 3, 4, 6), two a byte with the even column in the low half, rows padded
// to whole groups of 32 columns (16 bytes), and one bfloat16 scale for each group of a row:
//   value[r, c] = e2m1(code[r, c]) * scale[r, c / 32]
//   out[i, r]   = sum over groups g of scale[r, g] * (sum over c in g of x[i, c] e2m1(code[r, c]))
// E2M1 is the 4-bit type that this hardware converts by itself (two codes an instruction).
#include <type_traits>

#include "rowwise.h"

namespace gnnrec {

constexpr int kGroup = 32;
constexpr int kQ4Block = 256;

__device__ __forceinline__ float e2m1(uint32_t code) {
  const uint32_t m = code & 7;
  const float v = m < 4 ? 0.5f * (float)m : (m < 6 ? (float)(m - 2) : (m == 6 ? 4.f : 6.f));
  return code & 8 ? -v : v;
}

// ---- laying a table out -------------------------------------------------------------------
// A group's scale is its largest magnitude / 6, rounded to bfloat16, and a value takes the code
// nearest to value / scale, ties to the even code. The borders between codes times the scale are
// exact in fp32 (3 bits times 8), so the comparisons decide the true quotient and nothing is
// divided. A group that holds an infinity or a NaN has a NaN scale: its row's scores are NaN.
// Four threads a group, eight values each: 32-B loads, one 4-B store.
template <class T>
__global__ __launch_bounds__(kQ4Block) void quantize_q4_kernel(int64_t n, int64_t k, int64_t ng,
                                                               const T* __restrict__ w,
                                                               int64_t ldw,
                                                               uint32_t* __restrict__ codes,
                                                               bf16_t* __restrict__ scale) {
  const int64_t base = (int64_t)blockIdx.x * kQ4Block;
  const int64_t per_row = ng * 4;
  const int64_t row_base = base / per_row;
  const uint32_t in_row = (uint32_t)(base - row_base * per_row) + threadIdx.x;
  const uint32_t q = in_row / (uint32_t)per_row, part = in_row - q * (uint32_t)per_row;
  const int64_t row = row_base + q;
  if (row >= n) return;  // four threads of a group leave together
  const int64_t c = (int64_t)part * 8;
  float v[8];
  load8(w + row * ldw + c, k - c, v);
  uint32_t top = 0;  // the magnitudes' bit patterns sort as the magnitudes, NaN above infinity
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2));
  const bool finite = top < 0x7f800000u;
  const bf16_t sb = finite ? (bf16_t)(__uint_as_float(top) / 6.f) : (bf16_t)__builtin_nanf("");
  const float s = (float)sb;
  uint32_t word = 0;
  if (s > 0.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = fabsf(v[e]);
      const uint32_t m = (uint32_t)(a > 0.25f * s) + (a >= 0.75f * s) + (a > 1.25f * s) +
                         (a >= 1.75f * s) + (a > 2.5f * s) + (a >= 3.5f * s) + (a > 5.f * s);
      word |= (m | (v[e] < 0.f ? 8u : 0u)) << (4 * e);
    }
  }
  codes[row * per_row + part] = word;
  if ((part & 3) == 0) scale[row * ng + (part >> 2)] = sb;
}

__global__ __launch_bounds__(kQ4Block) void dequantize_q4_kernel(int64_t n, int64_t k, int64_t ng,
                                                                 const uint32_t* __restrict__ codes,
                                                                 const bf16_t* __restrict__ scale,
                                                                 float* __restrict__ out,
                                                                 int64_t ldo) {
  const int64_t base = (int64_t)blockIdx.x * kQ4Block;
  const int64_t per_row = ng * 4;
  const int64_t row_base = base / per_row;
  const uint32_t in_row = (uint32_t)(base - row_base * per_row) + threadIdx.x;
  const uint32_t q = in_row / (uint32_t)per_row, part = in_row - q * (uint32_t)per_row;
  const int64_t row = row_base + q;
  if (row >= n) return;
  const int64_t c = (int64_t)part * 8;
  if (c >= k) return;
  const uint32_t word = codes[row * per_row + part];
  const float s = (float)scale[row * ng + (part >> 2)];
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e2m1(word >> (4 * e)) * s;
  store8(out + row * ldo + c, k - c, v);
}

// ---- products -----------------------------------------------------------------------------
// On the matrix cores, one 16 x 16 x 32 bf16 instruction a group: A holds the users (16 rows),
// B the codes of 16 items as bf16 (exact), and the group's 32 products are summed in fp32 before
// the group's scale multiplies them:
//   acc[user][item] += scale[item, g] * mfma(x[users, g], e2m1(codes[items, g]))
// A user's fp32 value is cut into three bf16 parts by truncation (8 + 8 + 8 bits, exact), half
// into two; the parts are further steps of the same accumulator, or, for up to four users, the
// idle rows of the same instruction (row 4 part + user), summed at the end.
//
// The codes stay row-major in memory. A lane reads 16 bytes, the 32 codes of one group of its
// row; the instruction wants a lane to hold eight codes of each group, so the four lanes of a row
// exchange their words (a 4 x 4 transposition, four permlane swaps).
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <class T>
struct Parts;
template <>
struct Parts<float> { static constexpr int n = 3; };
template <>
struct Parts<f16_t> { static constexpr int n = 2; };
template <>
struct Parts<bf16_t> { static constexpr int n = 1; };

// a's upper half and b's lower half change places; odd rows of a and even rows of b (16 lanes).
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
  const u32x2 r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
  const u32x2 r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}
// w[j] of lane row q  ->  w[q] of lane row j.
__device__ __forceinline__ void transpose4(u32x4& w) {
  uint32_t a = w[0], b = w[1], c = w[2], d = w[3];
  swap32(a, c);
  swap32(b, d);
  swap16(a, b);
  swap16(c, d);
  w = u32x4{a, b, c, d};
}

// Eight codes as bf16.
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t w) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The top 16 bits of v, and what is left of it (exact; 0 for an infinity or a NaN, whose top bits
// keep it one).
__device__ __forceinline__ uint32_t cut(float& v) {
  uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) u |= 0x400000u;  // a NaN stays one in 16 bits
  const uint32_t top = u & 0xffff0000u;
  v = (u & 0x7f800000u) == 0x7f800000u ? 0.f : v - __uint_as_float(top);
  return top;
}

// A's fragments of one group: eight values x[user, c ..] of this lane, cut into parts.
template <class T, bool FEW>
__device__ __forceinline__ void load_users(const T* __restrict__ row, bool valid, int part,
                                           int64_t c, int64_t k,
                                           bf16x8 (&a)[FEW ? 1 : Parts<T>::n]) {
  constexpr int kP = Parts<T>::n;
  float v[8];
  load8(row + c, valid ? k - c : 0, v);
  uint32_t bits[kP][8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
#pragma unroll
    for (int i = 0; i < kP; ++i) bits[i][e] = cut(v[e]);
#pragma unroll
  for (int i = 0; i < (FEW ? 1 : kP); ++i) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t lo = bits[i][2 * e], hi = bits[i][2 * e + 1];
      if (FEW) {
#pragma unroll
        for (int j = 1; j < kP; ++j) {
          lo = part == j ? bits[j][2 * e] : lo;
          hi = part == j ? bits[j][2 * e + 1] : hi;
        }
      }
      w[e] = (lo >> 16) | hi;
    }
    a[i] = __builtin_bit_cast(bf16x8, w);
  }
}

__device__ __forceinline__ void store_out(void* out, int32_t dtype, int64_t i, float v) {
  if (dtype == GNNREC_F32) ((float*)out)[i] = v;
  else if (dtype == GNNREC_BF16) ((bf16_t*)out)[i] = (bf16_t)v;
  else ((f16_t*)out)[i] = (f16_t)v;
}

struct Q4Args {
  int64_t m, ldx, n, k, ng, ldo;
  const uint32_t* codes;
  const bf16_t* scale;
  void* out;
  int32_t out_dtype;
};

// FEW: at most four users a tile. WK waves share 64 items and split the groups; WK == 1: every
// wave takes items of its own. HELD > 0: rows of at most 4 HELD groups, whose users' fragments
// stay in registers over all the wave's items.
template <class T, bool FEW, int WK, int HELD>
__global__ __launch_bounds__(WK > 4 ? WK * 64 : 256) void q4_matmul_kernel(
    const T* __restrict__ x, Q4Args p) {
  constexpr int kA = FEW ? 1 : Parts<T>::n;
  constexpr int kWaves = WK > 4 ? WK : 4;
  __shared__ f32x4 join[WK > 1 ? (WK - 1) * 4 * 64 : 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const int64_t user0 = (int64_t)blockIdx.y * (FEW ? 4 : 16);
  const int64_t user = user0 + (FEW ? (r & 3) : r);
  const int part = FEW ? r >> 2 : 0;
  const bool valid = user < p.m && part < Parts<T>::n;
  const T* xrow = x + (user < p.m ? user : 0) * p.ldx;
  const int64_t blocks4 = (p.ng + 3) >> 2;

  bf16x8 held[HELD ? HELD * 4 : 1][kA];
  if (HELD) {
#pragma unroll
    for (int g = 0; g < HELD * 4; ++g)
      load_users<T, FEW>(xrow, valid, part, (int64_t)g * kGroup + q * 8, p.k, held[g]);
  }
  const int64_t tasks = (p.n + 63) >> 6;
  const int64_t first = WK == 1 ? (int64_t)blockIdx.x * kWaves + wave : blockIdx.x;
  const int64_t step = WK == 1 ? (int64_t)gridDim.x * kWaves : gridDim.x;
  for (int64_t task = first; task < tasks; task += step) {
    const int64_t base = task * 64;
    int64_t row[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t i = base + t * 16 + r;
      row[t] = i < p.n ? i : p.n - 1;
    }
    f32x4 acc[4] = {};
    auto step4 = [&](int64_t b, const bf16x8(*a)[kA]) {
      const int64_t g0 = b * 4;
      u32x4 w[4];
      uint32_t sc[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        w[t] = u32x4{0, 0, 0, 0};
        if (g0 + q < p.ng)
          w[t] = *reinterpret_cast<const u32x4*>(p.codes + (row[t] * p.ng + g0 + q) * 4);
#pragma unroll
        for (int g = 0; g < 4; ++g)
          sc[t][g] = g0 + g < p.ng
                         ? (uint32_t)reinterpret_cast<const uint16_t*>(p.scale)[row[t] * p.ng + g0 + g]
                         : 0;
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) transpose4(w[t]);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g0 + g >= p.ng) break;
        bf16x8 now[kA];
        if (HELD) {
#pragma unroll
          for (int i = 0; i < kA; ++i) now[i] = a[g][i];
        } else {
          load_users<T, FEW>(xrow, valid, part, (g0 + g) * kGroup + q * 8, p.k, now);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const bf16x8 bf = codes_to_bf16(w[t][g]);
          f32x4 d = {};
#pragma unroll
          for (int i = kA - 1; i >= 0; --i)
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(now[i], bf, d, 0, 0, 0);
          const float s = __uint_as_float(sc[t][g] << 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(s, d[i], acc[t][i]);
        }
      }
    };
    if (HELD) {
#pragma unroll
      for (int b = 0; b < HELD; ++b) step4(b, held + b * 4);
    } else {
      const int64_t b0 = WK > 1 ? blocks4 * wave / WK : 0;
      const int64_t b1 = WK > 1 ? blocks4 * (wave + 1) / WK : blocks4;
      for (int64_t b = b0; b < b1; ++b) step4(b, held);
    }
    if (WK > 1) {
      if (wave > 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) join[((wave - 1) * 4 + t) * 64 + lane] = acc[t];
      }
      __syncthreads();
      if (wave == 0) {
        for (int v = 0; v < WK - 1; ++v)
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[t] += join[(v * 4 + t) * 64 + lane];
      }
      __syncthreads();
      if (wave > 0) continue;
    }
    // lane (q, r) holds users 4 q + i (or part q of user i) of items 16 t + r; with t and q
    // exchanged, a register is one user's 64 neighbouring items
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 v;
#pragma unroll
      for (int t = 0; t < 4; ++t) v[t] = __float_as_uint(acc[t][i]);
      transpose4(v);
      const int64_t item = base + lane;
      if (FEW) {
        float s = __uint_as_float(v[0]);
#pragma unroll
        for (int j = 1; j < Parts<T>::n; ++j) s += __uint_as_float(v[j]);
        if (user0 + i < p.m && item < p.n)
          store_out(p.out, p.out_dtype, (user0 + i) * p.ldo + item, s);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t u = user0 + 4 * j + i;
          if (u < p.m && item < p.n)
            store_out(p.out, p.out_dtype, u * p.ldo + item, __uint_as_float(v[j]));
        }
      }
    }
  }
}

template <class T, bool FEW>
static int run_matmul(const T* x, const Q4Args& p, hipStream_t stream) {
  const int64_t tasks = ceil_div(p.n, 64);
  const unsigned tiles = (unsigned)ceil_div(p.m, FEW ? 4 : 16);
  auto go = [&](auto wk, auto held) {
    constexpr int kWaves = wk.value > 4 ? wk.value : 4;
    const int64_t want = wk.value == 1 ? ceil_div(tasks, 4) : tasks;
    const unsigned grid = (unsigned)(want < 2048 ? want : 2048);
    hipLaunchKernelGGL((q4_matmul_kernel<T, FEW, wk.value, held.value>), dim3(grid, tiles),
                       dim3(kWaves * 64), 0, stream, x, p);
    return check_launch("q4_matmul");
  };
  using std::integral_constant;
  if (p.ng <= 4) return go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  if (p.ng <= 8) return go(integral_constant<int, 1>{}, integral_constant<int, 2>{});
  if (p.ng < 64) return go(integral_constant<int, 4>{}, integral_constant<int, 0>{});
  return go(integral_constant<int, 16>{}, integral_constant<int, 0>{});
}

static int check_table(const char* what, int64_t n, int64_t k, const void* codes,
                       const void* scale) {
  GNNREC_REQUIRE(n >= 0 && k >= 1 && k <= 0x3fffffff, "%s: bad table size", what);
  if (n == 0) return GNNREC_OK;
  GNNREC_REQUIRE(codes && scale, "%s: null pointer", what);
  GNNREC_REQUIRE(aligned16(codes), "%s: the codes must be 16-B aligned", what);
  GNNREC_REQUIRE(n <= (int64_t)0x7fffffff * kQ4Block / (ceil_div(k, kGroup) * 4),
                 "%s: table too large", what);
  return GNNREC_OK;
}

}  // namespace gnnrec

using namespace gnnrec;

extern "C" int gnnrec_quantize_q4(int32_t dtype, int64_t n, int64_t k, const void* w, int64_t ldw,
                                  void* codes, void* scale, gnnrec_stream_t stream) {
  GNNREC_REQUIRE(dtype_ok(dtype), "quantize_q4: unknown dtype %d", dtype);
  const int rc = check_table("quantize_q4", n, k, codes, scale);
  if (rc != GNNREC_OK || n == 0) return rc;
  GNNREC_REQUIRE(w, "quantize_q4: null pointer");
  const int64_t ng = ceil_div(k, kGroup);
  return with_dtype(dtype, [&](auto e) {
    using T = decltype(e);
    hipLaunchKernelGGL((quantize_q4_kernel<T>), dim3((unsigned)ceil_div(n * ng * 4, kQ4Block)),
                       dim3(kQ4Block), 0, as_hip(stream), n, k, ng, (const T*)w, ldw,
                       (uint32_t*)codes, (bf16_t*)scale);
    return check_launch("quantize_q4");
  });
}

extern "C" int gnnrec_dequantize_q4(int64_t n, int64_t k, const void* codes, const void* scale,
                                    float* out, int64_t ldo, gnnrec_stream_t stream) {
  const int rc = check_table("dequantize_q4", n, k, codes, scale);
  if (rc != GNNREC_OK || n == 0) return rc;
  GNNREC_REQUIRE(out, "dequantize_q4: null pointer");
  const int64_t ng = ceil_div(k, kGroup);
  hipLaunchKernelGGL(dequantize_q4_kernel, dim3((unsigned)ceil_div(n * ng * 4, kQ4Block)),
                     dim3(kQ4Block), 0, as_hip(stream), n, k, ng, (const uint32_t*)codes,
                     (const bf16_t*)scale, out, ldo);
  return check_launch("dequantize_q4");
}

extern "C" int gnnrec_q4_matmul(int32_t dtype, int32_t out_dtype, int64_t m, const void* x,
                                int64_t ldx, int64_t n, int64_t k, const void* codes,
                                const void* scale, void* out, int64_t ldo,
                                gnnrec_stream_t stream) {
  GNNREC_REQUIRE(dtype_ok(dtype) && dtype_ok(out_dtype), "q4_matmul: unknown dtype");
  const int rc = check_table("q4_matmul", n, k, codes, scale);
  if (rc != GNNREC_OK) return rc;
  GNNREC_REQUIRE(m >= 0 && m <= 65535, "q4_matmul: %lld rows of x, at most 65535",
                 (long long)m);
  if (n == 0 || m == 0) return GNNREC_OK;
  GNNREC_REQUIRE(x && out, "q4_matmul: null pointer");
  const Q4Args p{m, ldx, n, k, ceil_div(k, kGroup), ldo, (const uint32_t*)codes,
                 (const bf16_t*)scale, out, out_dtype};
  return with_dtype(dtype, [&](auto e) {
    using T = decltype(e);
    return m <= 4 ? run_matmul<T, true>((const T*)x, p, as_hip(stream))
                  : run_matmul<T, false>((const T*)x, p, as_hip(stream));
  });
}
