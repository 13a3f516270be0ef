// Item tables in 4 bits and their products with a few users' rows, gfx950.
//
// A table of n rows of k values is held as E2M1 codes (sign, two exponent bits, one mantissa
// bit: 0, .5, 1, 1.5, 2, 3, 4, 6), two a byte with the even column in the low half, rows padded
// to whole groups of 32 columns (16 bytes), and one bfloat16 scale for each group of a row:
//   value[r, c] = e2m1(code[r, c]) * scale[r, c / 32]
//   out[i, r]   = sum over groups g of scale[r, g] * (sum over c in g of x[i, c] e2m1(code[r, c]))
// E2M1 is the 4-bit type that this hardware converts by itself (two codes an instruction).
//
// Short rows are bound by the table's bytes: one user against 1M x 64 9.7 us (36 MB, which may lie
// in the 256 MB cache: 4.1 TB/s), 16 users against 1M x 256 bf16 48 us (3.7). Long rows are not:
// 8192 x 8192 and one user 13.4 us (2.8: each round of loads waits for the one before to be
// multiplied), 16 fp32 users 35 us (1.1: the users' fragments from the caches, see q4_many_kernel).
// The quantiser: 1M x 64 fp32 68 us (4.3, the VALU busy in 76 % of the cycles), bf16 59 (2.8, 86 %:
// instructions, seven comparisons a value among them).
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
  const int64_t base = block_index() * kQ4Block;
  const int64_t per_row = ng * 4;
  const int64_t row_base = base / per_row;
  const uint32_t in_row = (uint32_t)(base - row_base * per_row) + threadIdx.x;
  const uint32_t q = in_row / (uint32_t)per_row, part = in_row - q * (uint32_t)per_row;
  const int64_t row = row_base + q;
  if (row >= n) return;  // four threads of a group leave together
  const int64_t c = (int64_t)part * 8;
  float v[8];
  load8(w + row * ldw, c, k, v);
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
  const int64_t base = block_index() * kQ4Block;
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
  store8(out + row * ldo, c, k, v);
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

// Eight values cut into their bf16 parts.
template <int P>
__device__ __forceinline__ void split8(float (&v)[8], u32x4 (&parts)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = cut(v[2 * e]), hi = cut(v[2 * e + 1]);
      parts[i][e] = (lo >> 16) | hi;
    }
}

// STREAM: past the caches, which hold the codes for the next tile of users (64 users x 1M x 64:
// 73.8 -> 64.8 us; one user's scores are a small part of what is moved, and gain nothing).
template <bool STREAM>
__device__ __forceinline__ void store_out(void* out, int32_t dtype, int64_t i, float v) {
  auto put = [](auto* at, auto x) {
    if (STREAM) __builtin_nontemporal_store(x, at);
    else *at = x;
  };
  if (dtype == GNNREC_F32) put((float*)out + i, v);
  else if (dtype == GNNREC_BF16) put((bf16_t*)out + i, (bf16_t)v);
  else put((f16_t*)out + i, (f16_t)v);
}

struct Q4Args {
  int64_t m, n, k, ng, ldo;
  const uint32_t* codes;
  const bf16_t* scale;
  void* out;
  int32_t out_dtype;
};

// Codes and scales of R groups from g0 on (R == 4: as many of four as the row has) of NT tiles of
// 16 items, in flight. Rows are offsets from `base`, clamped to the table's last row, and groups
// to the row's last one, so every load is unconditional and within the table; what a clamped
// load brings is not used (a tile's results depend on their own row alone).
//
// With four groups, lane (q, r) takes 16 bytes, group g0 + q of row r of a tile; of rows with only
// two (one) groups, a load covers two (four) tiles, so that no lane idles and the wave reads one
// contiguous piece. Either way word j of load i after the transposition holds eight codes of one
// (tile, group) in every lane row. Scales: lane l takes those of row l of the 64.
template <int NT, int R>
struct Codes {
  // NT tiles x R groups, four 16-B pieces a load (of one or two tiles always four groups)
  static constexpr int kLoads = NT == 4 ? R : NT;
  u32x4 w[kLoads];
  uint32_t s[2];  // s[h]: scales of groups g0 + 2 h and g0 + 2 h + 1

  __device__ __forceinline__ void load(const Q4Args& p, int64_t base, int64_t g0) {
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int last = (int)(p.n - 1 - base < 63 ? p.n - 1 - base : 63);
    const int end = p.ng - g0 < 4 ? (int)(p.ng - g0) - 1 : 3;  // the last group of these
    const uint32_t* codes = p.codes + (base * p.ng + g0) * 4;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = (R == 4 ? i * 16 : R == 2 ? i * 32 + (q >> 1) * 16 : q * 16) + r;
      const int g = R == 4 ? min(q, end) : R == 2 ? (q & 1) : 0;
      w[i] = *reinterpret_cast<const u32x4*>(codes + ((int64_t)min(row, last) * p.ng + g) * 4);
    }
    struct __attribute__((packed)) Pair { uint32_t v; };
    const int row = min(lane & (NT * 16 - 1), last);
    const uint16_t* at = reinterpret_cast<const uint16_t*>(p.scale) + (base + row) * p.ng + g0;
    if (R == 1) {
      s[0] = at[0];
    } else {  // two at a time; a pair that would leave the row is read one earlier
      const int back0 = R == 4 && end < 1, back1 = R == 4 ? max(0, 3 - end) : 0;
      s[0] = reinterpret_cast<const Pair*>(at - back0)->v >> (16 * back0);
      if (R == 4) {
        const int o = max(2 - back1, end > 0 ? 0 : -1);
        s[1] = reinterpret_cast<const Pair*>(at + o)->v >> (16 * min(back1, 1));
      }
    }
  }

  // acc[t] += the products with users(g), the fragments of group g0 + g.
  template <int KA, class A>
  __device__ __forceinline__ void multiply(int64_t left, A&& users, f32x4 (&acc)[NT]) {
    uint32_t st[2][4];
#pragma unroll
    for (int h = 0; h < (R == 4 ? 2 : 1); ++h) {
      if (NT == 1) {
        st[h][0] = s[h];
      } else if (NT == 2) {
        uint32_t a = s[h], b = s[h];  // rows (0 1 0 1)
        swap16(a, b);
        st[h][0] = a, st[h][1] = b;
      } else {  // a tile's scales to all lane rows
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
      if (R == 4 && g >= left) break;
      bf16x8 a[KA];
      users(g, a);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t word = R == 4 ? w[t][g] : R == 2 ? w[t >> 1][(t & 1) * 2 + g] : w[0][t];
        const bf16x8 bf = codes_to_bf16(word);
        f32x4 d[KA + 1];  // d[i]: the sum of parts i and up
        d[KA] = f32x4{};
#pragma unroll
        for (int i = KA - 1; i >= 0; --i)
          d[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], bf, d[i + 1], 0, 0, 0);
        const uint32_t sw = st[g >> 1][t];
        const float sc = __uint_as_float(g & 1 ? sw & 0xffff0000u : sw << 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(sc, d[0][i], acc[t][i]);
        // The parts' sums stay alive past the last instruction of their chain (no code: nothing is
        // read here), so that none is accumulated into registers that partly hold another: the
        // compiler did that, and it has given wrong results on this hardware. 16 fp16 users x
        // 8192 x 8192: 28.1 us, and 28.0 without.
#pragma unroll
        for (int i = 1; i < KA; ++i) asm volatile("" ::"v"(d[i]), "v"(acc[t][0]));
      }
      // one group at a time: all four together would take twice the registers and half the waves
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// The results of NT tiles. Lane (q, r) holds users 4 q + i of item r of a tile, or part q of user
// i; a transposition gives a register 64 neighbouring items of one user (NT == 4), or the parts
// of user q (FEW, fewer tiles).
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
        if (item < p.n) store_out<!FEW>(p.out, p.out_dtype, (user0 + i) * p.ldo + item, s);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t u = user0 + 4 * j + i;
          if (u < p.m && item < p.n)
            store_out<!FEW>(p.out, p.out_dtype, u * p.ldo + item, __uint_as_float(v[j]));
        }
      }
    }
  } else {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t item = base + t * 16 + r;
      u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(acc[t][i]);
      if (FEW) {
        transpose4(v);
        float s = __uint_as_float(v[0]);
#pragma unroll
        for (int j = 1; j < PARTS; ++j) s += __uint_as_float(v[j]);
        if (user0 + q < p.m && item < p.n)
          store_out<!FEW>(p.out, p.out_dtype, (user0 + q) * p.ldo + item, s);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t u = user0 + 4 * q + i;
          if (u < p.m && item < p.n)
            store_out<!FEW>(p.out, p.out_dtype, u * p.ldo + item, __uint_as_float(v[i]));
        }
      }
    }
  }
}

// Many items or short rows: the workgroup cuts its users into fragments once, all groups of them,
// in LDS, and its waves walk tile sets of their own, the codes one step (four groups, or R) ahead
// through the end of a tile set into the next. FEW: at most four users a tile, their parts in the
// instruction's idle rows.
template <class T, bool FEW, int NT, int R>
__global__ __launch_bounds__(kQ4Block, FEW ? 4 : 3) void q4_walk_kernel(const T* __restrict__ x,
                                                                        int64_t ldx, Q4Args p) {
  constexpr int kP = Parts<T>::n, kA = FEW ? 1 : kP, kUsers = FEW ? 4 : 16;
  extern __shared__ u32x4 frag[];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t user0 = (int64_t)blockIdx.y * kUsers;
  const int64_t tasks = (p.n + NT * 16 - 1) / (NT * 16), stride = (int64_t)gridDim.x * 4;
  const int64_t steps = R == 4 ? (p.ng + 3) >> 2 : 1;
  int64_t task = (int64_t)blockIdx.x * 4 + wave;
  Codes<NT, R> now, next;
  if (task < tasks) now.load(p, task * NT * 16, 0);
  // rows of A that no user fills are left as they are: they reach no result that is stored
  const int users = (int)(p.m - user0 < kUsers ? p.m - user0 : kUsers), per = (int)p.ng * 4;
  for (int i = threadIdx.x; i < users * per; i += kQ4Block) {
    const int u = i / per, c = i - u * per;
    float v[8];
    load8(x + (user0 + u) * ldx, c * 8, p.k, v);
    u32x4 parts[kP];
    split8(v, parts);
#pragma unroll
    for (int j = 0; j < kP; ++j)
      frag[((c >> 2) * kA + (FEW ? 0 : j)) * 64 + (c & 3) * 16 + (FEW ? j * 4 + u : u)] = parts[j];
  }
  __syncthreads();
  while (task < tasks) {
    f32x4 acc[NT] = {};
    const int64_t base = task * NT * 16;
    task += stride;
    for (int64_t b = 0; b < steps; ++b) {
      if (b + 1 < steps) next.load(p, base, (b + 1) * 4);
      else if (task < tasks) next.load(p, task * NT * 16, 0);
      now.template multiply<kA>(
          p.ng - b * 4,
          [&](int g, bf16x8(&a)[kA]) {
#pragma unroll
            for (int i = 0; i < kA; ++i)
              a[i] = __builtin_bit_cast(bf16x8, frag[((b * 4 + g) * kA + i) * 64 + lane]);
          },
          acc);
      now = next;
    }
    store_tiles<FEW, NT, kP>(p, base, user0, acc);
  }
}

// The sums of a tile set over the WK waves that split its groups, in wave 0, in the waves' order.
template <int NT, int WK>
__device__ __forceinline__ void join_waves(f32x4 (&acc)[NT], f32x4* join) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
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
  __syncthreads();  // the sums have been read before the next tile set's are written
}

// Long rows, at most four users a tile: WK waves share a tile set and split its groups, STEPS
// steps of four groups in flight. The workgroup keeps the users' parts in LDS, row j * users + u
// padded by 64 B, cut while the first codes are on their way.
template <class T, int NT, int WK, int STEPS>
__global__ __launch_bounds__(WK * 64, 4) void q4_few_kernel(const T* __restrict__ x, int64_t ldx,
                                                         Q4Args p) {
  constexpr int kP = Parts<T>::n;
  extern __shared__ u32x4 rows[];
  __shared__ f32x4 join[(WK - 1) * NT * 64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const int64_t user0 = (int64_t)blockIdx.y * 4;
  const int users = (int)(p.m - user0 < 4 ? p.m - user0 : 4);
  const int per = (int)p.ng * 4, pitch = per + 4;  // 16-B pieces
  const int64_t steps = (p.ng + 3) >> 2;
  // a wave's steps are wave, wave + WK, ...: the waves read neighbouring pieces of the rows
  const int64_t count = (steps - wave + WK - 1) / WK;
  const int64_t tasks = (p.n + NT * 16 - 1) / (NT * 16);
  // rows of A that no user fills repeat another's: they reach no result that is stored
  const int mine = (min(r >> 2, kP - 1) * users + min(r & 3, users - 1)) * pitch + q;
  Codes<NT, 4> now[STEPS];
  auto load = [&](int64_t task, int64_t b) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int64_t step = wave + (b + i) * WK;
      now[i].load(p, task * NT * 16, (step < steps ? step : steps - 1) * 4);
    }
  };
  load(blockIdx.x, 0);
  for (int u = 0; u < users; ++u)
    for (int c = threadIdx.x; c < per; c += WK * 64) {
      float v[8];
      load8(x + (user0 + u) * ldx, c * 8, p.k, v);
      u32x4 parts[kP];
      split8(v, parts);
#pragma unroll
      for (int j = 0; j < kP; ++j) rows[(j * users + u) * pitch + c] = parts[j];
    }
  __syncthreads();
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    f32x4 acc[NT] = {};
    if (task != blockIdx.x) load(task, 0);
    for (int64_t b = 0;;) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        if (b + i >= count) break;
        const int64_t g0 = (wave + (b + i) * WK) * 4;
        now[i].template multiply<1>(
            p.ng - g0,
            [&](int g, bf16x8(&f)[1]) {
              f[0] = __builtin_bit_cast(bf16x8, rows[mine + (g0 + g) * 4]);
            },
            acc);
      }
      b += STEPS;
      if (b >= count) break;
      load(task, b);
    }
    join_waves<NT, WK>(acc, join);
    if (wave == 0) store_tiles<true, NT, kP>(p, task * NT * 16, user0, acc);
  }
}

// Long rows, more users: they come as bf16 parts in rows of whole groups (plane i at x + i *
// plane, rows ldx apart), from the table itself or from split_users_kernel, and a step's
// fragments (1 KB a group and part) are loaded from the caches with its codes, one step ahead.
// The waves split the groups, so each fragment is loaded once for every 32 (64) items: 16 fp32
// users x 8192 x 8192 move 200 MB of them beside 38 MB of codes, with one wave a SIMD resident (256
// workgroups of four), in 35 us; bf16 users, a third of the fragments, in 19.
template <int PARTS, int NT, int WK>
__global__ __launch_bounds__(WK * 64, 2) void q4_many_kernel(const bf16_t* __restrict__ x,
                                                          int64_t ldx, int64_t plane, Q4Args p) {
  __shared__ f32x4 join[(WK - 1) * NT * 64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const int64_t user0 = (int64_t)blockIdx.y * 16;
  const bf16_t* xrow = x + (user0 + r < p.m ? user0 + r : p.m - 1) * ldx + q * 8;
  const int64_t steps = (p.ng + 3) >> 2;
  const int64_t b0 = steps * wave / WK, b1 = steps * (wave + 1) / WK;
  const int64_t tasks = (p.n + NT * 16 - 1) / (NT * 16);
  struct Step {
    Codes<NT, 4> codes;
    bf16x8 a[4][PARTS];
  };
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int64_t base = task * NT * 16;
    auto load = [&](Step& s, int64_t b) {
      b = b < steps ? b : steps - 1;
      s.codes.load(p, base, b * 4);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int64_t at = b * 4 + g < p.ng ? b * 4 + g : p.ng - 1;
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
          s.a[g][i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const Eight<bf16_t>*>(
                                                     xrow + i * plane + at * kGroup));
      }
    };
    auto multiply = [&](Step& s, int64_t b, f32x4(&acc)[NT]) {
      s.codes.template multiply<PARTS>(
          p.ng - b * 4,
          [&](int g, bf16x8(&f)[PARTS]) {
#pragma unroll
            for (int i = 0; i < PARTS; ++i) f[i] = s.a[g][i];
          },
          acc);
    };
    f32x4 acc[NT] = {};
    Step one, two;
    load(one, b0);
    for (int64_t b = b0; b < b1; b += 2) {
      if (b + 1 < b1) load(two, b + 1);
      multiply(one, b, acc);
      if (b + 1 >= b1) break;
      if (b + 2 < b1) load(one, b + 2);
      multiply(two, b + 1, acc);
    }
    join_waves<NT, WK>(acc, join);
    if (wave == 0) store_tiles<false, NT, PARTS>(p, base, user0, acc);
  }
}

// x [m, k] as bf16 parts: plane i, rows of kp = 32 ng values, zeros behind k.
template <class T>
__global__ __launch_bounds__(kQ4Block) void split_users_kernel(const T* __restrict__ x,
                                                               int64_t ldx, int64_t m, int64_t k,
                                                               int64_t kp,
                                                               bf16_t* __restrict__ parts) {
  constexpr int kP = Parts<T>::n;
  const int64_t i = block_index() * kQ4Block + threadIdx.x;
  const int64_t per = kp / 8, row = i / per, c = (i - row * per) * 8;
  if (row >= m) return;
  float v[8];
  load8(x + row * ldx, c, k, v);
  u32x4 w[kP];
  split8(v, w);
#pragma unroll
  for (int j = 0; j < kP; ++j) *reinterpret_cast<u32x4*>(parts + (j * m + row) * kp + c) = w[j];
}

// Workgroups of a walk (three a CU are resident; with several user tiles each takes fewer, as the
// tiles share the codes in the caches) and of the split products. 16 users x 1M x 64 fp32: 768
// 20.7 us, 1024 23.8, 2048 25.2; 64 users: 384 a tile 72.0, 256 82.8, 512 75.8.
constexpr int64_t kWalkGrid = 768, kWalkGridTiled = 384, kSplitGrid = 1024;
// LDS that the users' fragments or rows may take: two workgroups still fit a CU (160 KB), and
// with the joined sums the rows stay below 64 KB.
constexpr int64_t kWalkBytes = 64 * 1024, kFewBytes = 50 * 1024;
// Items from which waves walk long rows alone (125 000 x 512, one user: 13.1 us, split 49.3), and
// from which they walk four tiles at a time (4 users x 30 000 x 1000: one tile 10.7 us, four
// 14.9).
constexpr int64_t kManyItems = 16384, kWideItems = 65536;
// Items from which the waves that split long rows share two tiles (8192 x 8192, one user: 13.7 us,
// one tile 15.6; 4096 x 4096: 8.4 and 6.5); eight waves from 2048 columns, four below (8000 x
// 1000: 4.3 us, eight 4.9).
constexpr int64_t kPairItems = 6144;

static int64_t parts_of(int32_t dtype) {
  return dtype == GNNREC_F32 ? 3 : dtype == GNNREC_F16 ? 2 : 1;
}

// How a product is shared out.
//  walk: a wave walks whole rows; needs all groups' fragments of a user tile in LDS (1 KB a group,
//        and for more than four users a part), and either rows of at most 256 columns (then also
//        few items are quick) or items for all waves.
//  few:  the waves of a workgroup split long rows; at most four users, whose parts fit LDS.
//  many: the same with the fragments from the caches; the rest.
enum class Q4Plan { walk, few, many };
static int64_t few_bytes(int32_t dtype, int64_t m, int64_t ng) {
  return (m < 4 ? m : 4) * parts_of(dtype) * (ng * 4 + 4) * 16;
}
static int64_t walk_bytes(int32_t dtype, int64_t m, int64_t ng) {
  return ng * (m <= 4 ? 1 : parts_of(dtype)) * 1024;
}
static Q4Plan plan_of(int32_t dtype, int64_t m, int64_t n, int64_t ng) {
  if (walk_bytes(dtype, m, ng) <= kWalkBytes && (ng <= 8 || n >= kManyItems)) return Q4Plan::walk;
  return m <= 4 && few_bytes(dtype, m, ng) <= kFewBytes ? Q4Plan::few : Q4Plan::many;
}

template <class T, bool FEW>
static int run_walk(int32_t dtype, const T* x, int64_t ldx, const Q4Args& p, hipStream_t stream) {
  auto go = [&](auto nt, auto rem) {
    const int64_t tiles = ceil_div(p.m, FEW ? 4 : 16);
    const int64_t most = tiles == 1 ? kWalkGrid : kWalkGridTiled;
    const int64_t want = ceil_div(ceil_div(p.n, nt.value * 16), 4);
    hipLaunchKernelGGL((q4_walk_kernel<T, FEW, nt.value, rem.value>),
                       dim3((unsigned)(want < most ? want : most), (unsigned)tiles),
                       dim3(kQ4Block), walk_bytes(dtype, p.m, p.ng), stream, x, ldx, p);
    return check_launch("q4_matmul");
  };
  using std::integral_constant;
  const integral_constant<int, 1> i1{};
  const integral_constant<int, 2> i2{};
  const integral_constant<int, 4> i4{};
  if (p.n < kWideItems) return p.ng == 1 ? go(i1, i1) : go(i1, i4);  // four times the waves
  return p.ng == 1 ? go(i4, i1) : p.ng == 2 ? go(i4, i2) : go(i4, i4);
}

template <class T>
static int run_few(int32_t dtype, const T* x, int64_t ldx, const Q4Args& p, hipStream_t stream) {
  auto go = [&](auto nt, auto wk, auto steps) {
    const int64_t tasks = ceil_div(p.n, nt.value * 16);
    hipLaunchKernelGGL((q4_few_kernel<T, nt.value, wk.value, steps.value>),
                       dim3((unsigned)(tasks < kSplitGrid ? tasks : kSplitGrid),
                            (unsigned)ceil_div(p.m, 4)),
                       dim3(wk.value * 64), few_bytes(dtype, p.m, p.ng), stream, x, ldx, p);
    return check_launch("q4_matmul");
  };
  using std::integral_constant;
  const integral_constant<int, 1> i1{};
  const integral_constant<int, 2> i2{};
  const integral_constant<int, 4> i4{};
  const integral_constant<int, 8> i8{};
  if (p.n >= kPairItems) return p.ng >= 64 ? go(i2, i8, i2) : go(i2, i4, i2);
  return p.ng >= 64 ? go(i1, i8, i2) : go(i1, i4, i2);
}

// Two tiles a wave set: 16 users x 8192 x 8192 fp32 35.2 us (eight waves 36.3), x 2000 x 1000 fp32
// 9.5 (four tiles 12.2), x 20 000 x 3100 bf16 20.1 (four tiles 22.4). Four where there are several
// user tiles and many items, so that a fragment serves more of them: 64 users x 7812 x 8192 fp32
// 82.6 us (two 120; bf16 48.5), x 10 000 x 1000 fp32 23.5 (25.6); but x 300 x 3000 fp32 22.2
// (17.4).
template <int PARTS>
static int run_many(const bf16_t* x, int64_t ldx, int64_t plane, const Q4Args& p,
                    hipStream_t stream) {
  auto go = [&](auto nt) {
    constexpr int kWaves = 4;
    const int64_t tasks = ceil_div(p.n, nt.value * 16);
    hipLaunchKernelGGL((q4_many_kernel<PARTS, nt.value, kWaves>),
                       dim3((unsigned)(tasks < kSplitGrid ? tasks : kSplitGrid),
                            (unsigned)ceil_div(p.m, 16)),
                       dim3(kWaves * 64), 0, stream, x, ldx, plane, p);
    return check_launch("q4_matmul");
  };
  if (p.m > 16 && p.n >= kPairItems) return go(std::integral_constant<int, 4>{});
  return go(std::integral_constant<int, 2>{});
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
    hipLaunchKernelGGL((quantize_q4_kernel<T>), wide_grid(ceil_div(n * ng * 4, kQ4Block), kQ4Block),
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
  hipLaunchKernelGGL(dequantize_q4_kernel, wide_grid(ceil_div(n * ng * 4, kQ4Block), kQ4Block),
                     dim3(kQ4Block), 0, as_hip(stream), n, k, ng, (const uint32_t*)codes,
                     (const bf16_t*)scale, out, ldo);
  return check_launch("dequantize_q4");
}

extern "C" int64_t gnnrec_q4_matmul_work_bytes(int32_t dtype, int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || !dtype_ok(dtype)) return 0;
  const int64_t ng = ceil_div(k, kGroup);
  if (plan_of(dtype, m, n, ng) != Q4Plan::many) return 0;
  if (dtype == GNNREC_BF16 && k % kGroup == 0) return 0;  // x itself is read
  return parts_of(dtype) * m * ng * kGroup * (int64_t)sizeof(bf16_t);
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
  GNNREC_REQUIRE(gnnrec_q4_matmul_work_bytes(dtype, m, n, k) == 0 || (work && aligned16(work)),
                 "q4_matmul: the workspace is missing or not 16-B aligned");
  const int64_t ng = ceil_div(k, kGroup);
  GNNREC_REQUIRE(ceil_div(m * ng * 4, kQ4Block) <= 0x7fffffff, "q4_matmul: x is too large");
  const Q4Args p{m, n, k, ng, ldo, (const uint32_t*)codes, (const bf16_t*)scale, out, out_dtype};
  const hipStream_t st = as_hip(stream);
  return with_dtype(dtype, [&](auto e) {
    using T = decltype(e);
    constexpr int kP = Parts<T>::n;
    const Q4Plan plan = plan_of(dtype, m, n, ng);
    if (plan == Q4Plan::walk)
      return m <= 4 ? run_walk<T, true>(dtype, (const T*)x, ldx, p, st)
                    : run_walk<T, false>(dtype, (const T*)x, ldx, p, st);
    if (plan == Q4Plan::few) return run_few<T>(dtype, (const T*)x, ldx, p, st);
    const bf16_t* xs = (const bf16_t*)x;
    int64_t lds = ldx, plane = 0;
    if (kP > 1 || k % kGroup) {
      const int64_t kp = ng * kGroup;
      hipLaunchKernelGGL((split_users_kernel<T>),
                         wide_grid(ceil_div(m * (kp / 8), kQ4Block), kQ4Block), dim3(kQ4Block), 0,
                         st, (const T*)x, ldx, m, k, kp, (bf16_t*)work);
      const int rc2 = check_launch("q4_matmul (users)");
      if (rc2 != GNNREC_OK) return rc2;
      xs = (const bf16_t*)work, lds = kp, plane = m * kp;
    }
    return run_many<kP>(xs, lds, plane, p, st);
  });
}
