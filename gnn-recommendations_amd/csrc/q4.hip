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
  int64_t m, n, k, ng, ldo;
  const uint32_t* codes;
  const bf16_t* scale;
  void* out;
  int32_t out_dtype;
};

// acc[t] += the products of R groups from g0 on (R == 4: as many of four as the row has) of NT
// tiles of 16 items. Rows are given as an offset from `base`, clamped to the table's last row (a
// clamped row's results are not stored).
//
// Loads: with four groups, lane (q, r) takes 16 bytes, group g0 + q of row r of a tile; of rows
// with only two (one) groups left, a load covers two (four) tiles, so that no lane idles and the
// wave reads one contiguous piece. Either way word j of load i after the transposition holds
// eight codes of one (tile, group) in every lane row. Scales: lane l takes those of row l of the
// 64, and two swaps spread a tile's to all lane rows.
template <int NT, int R, int KA, class A>
__device__ __forceinline__ void groups(const Q4Args& p, int64_t base, int64_t g0, A&& users,
                                       f32x4 (&acc)[NT]) {
  static_assert(NT == 4 || (NT == 1 && R == 4), "a single tile always takes four groups");
  constexpr int kLoads = NT == 4 ? R : 1;  // four tiles x R groups, four pieces of 16 B a load
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int last = (int)(p.n - 1 - base < 63 ? p.n - 1 - base : 63);
  const uint32_t* codes = p.codes + (base * p.ng + g0) * 4;
  const uint16_t* scale = reinterpret_cast<const uint16_t*>(p.scale) + base * p.ng + g0;
  const int here = p.ng - g0 < 4 ? (int)(p.ng - g0) : 4;  // groups left
  u32x4 w[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = (R == 4 ? i * 16 : R == 2 ? i * 32 + (q >> 1) * 16 : q * 16) + r;
    const int g = R == 4 ? q : R == 2 ? (q & 1) : 0;
    w[i] = u32x4{0, 0, 0, 0};
    if (R < 4 || g < here)
      w[i] = *reinterpret_cast<const u32x4*>(
          codes + ((int64_t)(row < last ? row : last) * p.ng + g) * 4);
  }
  // s[h]: scales of groups g0 + 2 h and g0 + 2 h + 1
  uint32_t s[2] = {0, 0};
  {
    const int row = NT == 4 ? lane : r;
    const uint16_t* at = scale + (int64_t)(row < last ? row : last) * p.ng;
    struct __attribute__((packed)) Two { uint32_t v[2]; };
    struct __attribute__((packed)) One { uint32_t v; };
    if (R == 1) {
      s[0] = at[0];
    } else if (R == 2) {
      s[0] = reinterpret_cast<const One*>(at)->v;
    } else if (here == 4) {
      const Two v = *reinterpret_cast<const Two*>(at);
      s[0] = v.v[0], s[1] = v.v[1];
    } else {
      s[0] = at[0];
      if (here > 1) s[0] |= (uint32_t)at[1] << 16;
      if (here > 2) s[1] = at[2];
    }
  }
  uint32_t st[2][4];
#pragma unroll
  for (int h = 0; h < (R == 4 ? 2 : 1); ++h) {
    if (NT == 1) {
      st[h][0] = s[h];
    } else {
      uint32_t a = s[h], b = s[h];
      swap16(a, b);  // rows (0 0 2 2) and (1 1 3 3)
      uint32_t c = a, d = b;
      swap32(a, c);
      swap32(b, d);
      st[h][0] = a, st[h][1] = b, st[h][2] = c, st[h][3] = d;
    }
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i) transpose4(w[i]);
#pragma unroll
  for (int g = 0; g < R; ++g) {
    if (R == 4 && g >= here) break;
    const auto& a = users(g);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t word = R == 4 ? w[t][g] : R == 2 ? w[t >> 1][(t & 1) * 2 + g] : w[0][t];
      const bf16x8 bf = codes_to_bf16(word);
      f32x4 d = {};
#pragma unroll
      for (int i = KA - 1; i >= 0; --i)
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], bf, d, 0, 0, 0);
      const uint32_t sw = st[g >> 1][t];
      const float sc = __uint_as_float(g & 1 ? sw & 0xffff0000u : sw << 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(sc, d[i], acc[t][i]);
    }
  }
}

// The results of NT tiles. Lane (q, r) holds users 4 q + i of item r of a tile, or part q of user
// i; a transposition gives a register 64 neighbouring items of one user (NT == 4), or the parts
// of user q (FEW, NT == 1).
template <bool FEW, int NT, int PARTS>
__device__ __forceinline__ void store_tiles(const Q4Args& p, int64_t base, int64_t user0,
                                            const f32x4 (&acc)[NT]) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  if (NT == 4) {
    const int64_t item = base + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (user0 + i >= p.m) break;
      u32x4 v;
#pragma unroll
      for (int t = 0; t < 4; ++t) v[t] = __float_as_uint(acc[t % NT][i]);
      transpose4(v);
      if (FEW) {
        float s = __uint_as_float(v[0]);
#pragma unroll
        for (int j = 1; j < PARTS; ++j) s += __uint_as_float(v[j]);
        if (item < p.n) store_out(p.out, p.out_dtype, (user0 + i) * p.ldo + item, s);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t u = user0 + 4 * j + i;
          if (u < p.m && item < p.n)
            store_out(p.out, p.out_dtype, u * p.ldo + item, __uint_as_float(v[j]));
        }
      }
    }
  } else {
    const int64_t item = base + r;
    if (FEW) {
      u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(acc[0][i]);
      transpose4(v);
      float s = __uint_as_float(v[0]);
#pragma unroll
      for (int j = 1; j < PARTS; ++j) s += __uint_as_float(v[j]);
      if (user0 + q < p.m && item < p.n)
        store_out(p.out, p.out_dtype, (user0 + q) * p.ldo + item, s);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t u = user0 + 4 * q + i;
        if (u < p.m && item < p.n) store_out(p.out, p.out_dtype, u * p.ldo + item, acc[0][i]);
      }
    }
  }
}

// Short rows (at most 8 groups, 256 columns): the users' fragments stay in registers over all the
// items of a wave. FEW: at most four users a tile, the parts in the instruction's idle rows. HELD
// steps of four groups, the last of R.
template <class T, bool FEW, int NT, int HELD, int R>
__global__ __launch_bounds__(kQ4Block) void q4_short_kernel(const T* __restrict__ x, int64_t ldx,
                                                            Q4Args p) {
  constexpr int kA = FEW ? 1 : Parts<T>::n;
  constexpr int kHeld = (HELD - 1) * 4 + R;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const int64_t user0 = (int64_t)blockIdx.y * (FEW ? 4 : 16);
  const int64_t user = user0 + (FEW ? (r & 3) : r);
  const int part = FEW ? r >> 2 : 0;
  const bool valid = user < p.m && part < Parts<T>::n;
  bf16x8 held[kHeld][kA];
#pragma unroll
  for (int g = 0; g < kHeld; ++g)
    load_users<T, FEW>(x + (valid ? user : 0) * ldx, valid, part, (int64_t)g * kGroup + q * 8, p.k,
                       held[g]);
  const int64_t tasks = (p.n + NT * 16 - 1) / (NT * 16);
  for (int64_t task = (int64_t)blockIdx.x * 4 + wave; task < tasks; task += (int64_t)gridDim.x * 4) {
    const int64_t base = task * NT * 16;
    f32x4 acc[NT] = {};
    if (HELD == 2)
      groups<NT, 4, kA>(p, base, 0, [&](int g) -> auto& { return held[g % kHeld]; }, acc);
    groups<NT, R, kA>(p, base, (HELD - 1) * 4,
                      [&](int g) -> auto& { return held[(HELD - 1) * 4 + g]; }, acc);
    store_tiles<FEW, NT, Parts<T>::n>(p, base, user0, acc);
  }
}

// Long rows: the users come as bf16 parts (plane i at x + i * plane, rows ldx apart), from the
// table itself or from split_users_kernel. WK waves share a tile set and split its groups; their
// sums are joined through LDS in the waves' order.
template <int PARTS, bool FEW, int NT, int WK>
__global__ __launch_bounds__(WK > 4 ? WK * 64 : 256) void q4_long_kernel(
    const bf16_t* __restrict__ x, int64_t ldx, int64_t plane, Q4Args p) {
  constexpr int kA = FEW ? 1 : PARTS;
  __shared__ f32x4 join[WK > 1 ? (WK - 1) * NT * 64 : 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const int64_t user0 = (int64_t)blockIdx.y * (FEW ? 4 : 16);
  const int64_t user = user0 + (FEW ? (r & 3) : r);
  const int part = FEW ? r >> 2 : 0;
  const bool valid = user < p.m && part < PARTS;
  const bf16_t* xrow = x + (valid ? part * plane + user * ldx : 0);
  const int64_t blocks4 = (p.ng + 3) >> 2;
  const int64_t b0 = WK > 1 ? blocks4 * wave / WK : 0;
  const int64_t b1 = WK > 1 ? blocks4 * (wave + 1) / WK : blocks4;
  const int64_t tasks = (p.n + NT * 16 - 1) / (NT * 16);
  const int64_t first = WK > 1 ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  const int64_t step = WK > 1 ? gridDim.x : (int64_t)gridDim.x * 4;
  for (int64_t task = first; task < tasks; task += step) {
    const int64_t base = task * NT * 16;
    f32x4 acc[NT] = {};
#pragma unroll 2
    for (int64_t b = b0; b < b1; ++b) {
      bf16x8 a[4][kA];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int64_t c = (b * 4 + g) * kGroup + q * 8;
#pragma unroll
        for (int i = 0; i < kA; ++i) {
          a[g][i] = bf16x8{};
          if (valid && c + 8 <= p.k) {
            a[g][i] = __builtin_bit_cast(
                bf16x8, *reinterpret_cast<const Eight<bf16_t>*>(xrow + i * plane + c));
          } else if (valid && c < p.k) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c + e < p.k) a[g][i][e] = xrow[i * plane + c + e];
          }
        }
      }
      groups<NT, 4, kA>(p, base, b * 4, [&](int g) -> auto& { return a[g]; }, acc);
    }
    if (WK > 1) {
      if (wave > 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t) join[((wave - 1) * NT + t) * 64 + lane] = acc[t];
      }
      __syncthreads();
      if (wave == 0) {
        for (int v = 0; v < WK - 1; ++v)
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t] += join[(v * NT + t) * 64 + lane];
      }
      __syncthreads();  // the sums have been read before the next task's are written
      if (wave > 0) continue;
    }
    store_tiles<FEW, NT, PARTS>(p, base, user0, acc);
  }
}

// x [m, k] as bf16 parts: plane i, rows of kp = 32 ng values, zeros behind k.
template <class T>
__global__ __launch_bounds__(kQ4Block) void split_users_kernel(const T* __restrict__ x,
                                                               int64_t ldx, int64_t m, int64_t k,
                                                               int64_t kp,
                                                               bf16_t* __restrict__ parts) {
  constexpr int kP = Parts<T>::n;
  const int64_t i = (int64_t)blockIdx.x * kQ4Block + threadIdx.x;
  const int64_t per = kp / 8, row = i / per, c = (i - row * per) * 8;
  if (row >= m) return;
  float v[8];
  load8(x + row * ldx + c, k - c, v);
#pragma unroll
  for (int j = 0; j < kP; ++j) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = cut(v[2 * e]), hi = cut(v[2 * e + 1]);
      w[e] = (lo >> 16) | hi;
    }
    *reinterpret_cast<u32x4*>(parts + (j * m + row) * kp + c) = w;
  }
}

constexpr int64_t kShortGroups = 8;

template <class T, bool FEW>
static int run_short(const T* x, int64_t ldx, const Q4Args& p, hipStream_t stream) {
  auto go = [&](auto nt, auto held, auto rem) {
    const int64_t want = ceil_div(ceil_div(p.n, nt.value * 16), 4);
    hipLaunchKernelGGL((q4_short_kernel<T, FEW, nt.value, held.value, rem.value>),
                       dim3((unsigned)(want < 2048 ? want : 2048),
                            (unsigned)ceil_div(p.m, FEW ? 4 : 16)),
                       dim3(kQ4Block), 0, stream, x, ldx, p);
    return check_launch("q4_matmul");
  };
  using std::integral_constant;
  const integral_constant<int, 1> i1{};
  const integral_constant<int, 2> i2{};
  const integral_constant<int, 4> i4{};
  if (p.n < 64 * 1024) {  // one tile a wave: four times the waves
    if (p.ng <= 4) return go(i1, i1, i4);
    return go(i1, i2, i4);
  }
  switch (p.ng) {
    case 1: return go(i4, i1, i1);
    case 2: return go(i4, i1, i2);
    case 3: case 4: return go(i4, i1, i4);
    case 5: return go(i4, i2, i1);
    case 6: return go(i4, i2, i2);
    default: return go(i4, i2, i4);
  }
}

template <int PARTS, bool FEW>
static int run_long(const bf16_t* x, int64_t ldx, int64_t plane, const Q4Args& p,
                    hipStream_t stream) {
  auto go = [&](auto nt, auto wk) {
    const int64_t tasks = ceil_div(p.n, nt.value * 16);
    const int64_t want = wk.value == 1 ? ceil_div(tasks, 4) : tasks;
    hipLaunchKernelGGL((q4_long_kernel<PARTS, FEW, nt.value, wk.value>),
                       dim3((unsigned)(want < 4096 ? want : 4096),
                            (unsigned)ceil_div(p.m, FEW ? 4 : 16)),
                       dim3(wk.value > 4 ? wk.value * 64 : 256), 0, stream, x, ldx, plane, p);
    return check_launch("q4_matmul");
  };
  using std::integral_constant;
  const integral_constant<int, 1> i1{};
  const integral_constant<int, 4> i4{};
  const integral_constant<int, 8> i8{};
  if (p.n >= 64 * 4096) return go(i4, i1);
  if (p.n >= 64 * 512) return go(i4, i4);
  return p.ng >= 32 ? go(i1, i8) : go(i1, i4);
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

extern "C" int64_t gnnrec_q4_matmul_work_bytes(int32_t dtype, int64_t m, int64_t k) {
  const int64_t ng = ceil_div(k, kGroup);
  if (m <= 0 || k <= 0 || ng <= kShortGroups || dtype == GNNREC_BF16) return 0;
  return (dtype == GNNREC_F32 ? 3 : 2) * m * ng * kGroup * (int64_t)sizeof(bf16_t);
}

extern "C" int gnnrec_q4_matmul(int32_t dtype, int32_t out_dtype, int64_t m, const void* x,
                                int64_t ldx, int64_t n, int64_t k, const void* codes,
                                const void* scale, void* out, int64_t ldo, void* work,
                                gnnrec_stream_t stream) {
  GNNREC_REQUIRE(dtype_ok(dtype) && dtype_ok(out_dtype), "q4_matmul: unknown dtype");
  const int rc = check_table("q4_matmul", n, k, codes, scale);
  if (rc != GNNREC_OK) return rc;
  GNNREC_REQUIRE(m >= 0 && m <= 65535, "q4_matmul: %lld rows of x, at most 65535",
                 (long long)m);
  if (n == 0 || m == 0) return GNNREC_OK;
  GNNREC_REQUIRE(x && out, "q4_matmul: null pointer");
  GNNREC_REQUIRE(gnnrec_q4_matmul_work_bytes(dtype, m, k) == 0 || (work && aligned16(work)),
                 "q4_matmul: the workspace is missing or not 16-B aligned");
  const int64_t ng = ceil_div(k, kGroup);
  const Q4Args p{m, n, k, ng, ldo, (const uint32_t*)codes, (const bf16_t*)scale, out, out_dtype};
  const hipStream_t st = as_hip(stream);
  return with_dtype(dtype, [&](auto e) {
    using T = decltype(e);
    constexpr int kP = Parts<T>::n;
    if (ng <= kShortGroups)
      return m <= 4 ? run_short<T, true>((const T*)x, ldx, p, st)
                    : run_short<T, false>((const T*)x, ldx, p, st);
    const bf16_t* xs = (const bf16_t*)x;
    int64_t lds = ldx, plane = 0;
    if (kP > 1) {
      const int64_t kp = ng * kGroup;
      hipLaunchKernelGGL((split_users_kernel<T>),
                         dim3((unsigned)ceil_div(m * (kp / 8), kQ4Block)), dim3(kQ4Block), 0, st,
                         (const T*)x, ldx, m, k, kp, (bf16_t*)work);
      const int rc2 = check_launch("q4_matmul (users)");
      if (rc2 != GNNREC_OK) return rc2;
      xs = (const bf16_t*)work, lds = kp, plane = m * kp;
    }
    return m <= 4 ? run_long<kP, true>(xs, lds, plane, p, st)
                  : run_long<kP, false>(xs, lds, plane, p, st);
  });
}
