// Item tables in 4 bits and their products with a few users' rows, gfx950.
//
// A table of n rows of k values is held as E2M1 codes (sign, two exponent bits, one mantissa
// bit: 0, .5, 1, 1.5, 2, 3, 4, 6), two a byte with the even column in the low half, rows padded
// to whole groups of 32 columns (16 bytes), and one bfloat16 scale for each group of a row:
//   value[r, c] = e2m1(code[r, c]) * scale[r, c / 32]
//   out[i, r]   = sum over groups g of scale[r, g] * (sum over c in g of x[i, c] e2m1(code[r, c]))
// E2M1 is the 4-bit type that this hardware converts by itself (two codes an instruction).
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
// One thread an output.
template <class T, class O>
__global__ __launch_bounds__(kQ4Block) void q4_matmul_kernel(const T* __restrict__ x, int64_t ldx,
                                                             int64_t n, int64_t k, int64_t ng,
                                                             const uint32_t* __restrict__ codes,
                                                             const bf16_t* __restrict__ scale,
                                                             O* __restrict__ out, int64_t ldo) {
  const int64_t r = (int64_t)blockIdx.x * kQ4Block + threadIdx.x;
  const int64_t i = blockIdx.y;
  if (r >= n) return;
  float total = 0.f;
  for (int64_t g = 0; g < ng; ++g) {
    float s = 0.f;
    for (int p = 0; p < 4; ++p) {
      const int64_t c = g * kGroup + p * 8;
      if (c >= k) break;
      const uint32_t word = codes[(r * ng + g) * 4 + p];
      float v[8];
      load8(x + i * ldx + c, k - c, v);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < k) s = fmaf(v[e], e2m1(word >> (4 * e)), s);
    }
    total = fmaf(s, (float)scale[r * ng + g], total);
  }
  out[i * ldo + r] = (O)total;
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
  const int64_t ng = ceil_div(k, kGroup);
  return with_dtype(dtype, [&](auto e) {
    using T = decltype(e);
    return with_dtype(out_dtype, [&](auto o) {
      using O = decltype(o);
      hipLaunchKernelGGL((q4_matmul_kernel<T, O>),
                         dim3((unsigned)ceil_div(n, kQ4Block), (unsigned)m), dim3(kQ4Block), 0,
                         as_hip(stream), (const T*)x, ldx, n, k, ng, (const uint32_t*)codes,
                         (const bf16_t*)scale, (O*)out, ldo);
      return check_launch("q4_matmul");
    });
  });
}
