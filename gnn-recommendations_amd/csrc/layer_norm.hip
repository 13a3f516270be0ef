// Layer norm of a table's rows, forward and backward, alone or as the block between two hops
// (LeakyReLU, dropout and the residual sum in front), gfx950.
//
//   h    = residual + keep(act(x)) s        (alone: h = x)
//   y    = (h - mean h) r w + b             r = 1 / sqrt(var h + eps), var over the row's d values
//   g    = dy w,  u = (h - mean h) r
//   dh   = r (g - mean g - u mean(g u)) + dh_out
//   dres = dh,  dx = keep ? dh s act'(x) : 0
//   dw   = sum over rows of dy u,  db = sum over rows of dy
//
// A row lives in the registers of the TPR lanes that share it, in blocks of eight columns (one
// block is one draw of the dropout's generator), so the table is read once: the mean first, then
// the deviations' own sum and square sum, whose first part corrects the rounding of the mean
// (a constant row comes out as exactly b). The backward pass forms h and the statistics again
// from its inputs: nothing is saved, and half precision loses nothing to a rounded h.
//
// dw and db: every workgroup sums its rows in registers, joins its lane groups through LDS and
// writes one partial row; a second launch adds the partial rows, each column in a fixed order
// (no atomics: equal inputs give equal bits).
//
// fp32 tables are bound by memory (the block on 2M x 64: forward 373 us, 5.5 TB/s, backward 601 us,
// 5.1, sums 5 us), wide half-precision rows too (8192 x 4096 bf16 alone: 30, 44 and 5 us). A
// half-precision block is short of both limits (100 003 x 201 fp16: 39, 62 and 4 us, 4.1 and 3.9
// TB/s with the VALU busy in 64 and 62 % of the cycles, most of it the generator's and the
// conversions' instructions). A width just above one that fills its lanes takes twice as many:
// 8192 x 4097 fp16, both passes, 172 us, 4096 columns 80.
//
// Deviations are squared in fp32: a row whose squares add up to more than it holds (64 deviations of
// 2.4e18) comes out as the bias.
#include <type_traits>

#include "rowwise.h"

namespace gnnrec {

constexpr int kNormBlock = 256;
constexpr int kNormMaxD = 16384;

struct NormIn {
  int64_t rows, d;
  const void *x, *res, *w, *b;
  int64_t ldx, ldr;
  int32_t w_f32;  // w and b (and their gradients) hold float beside a half-precision table
  int32_t dropping;  // a mask is drawn (p > 0)
  float eps;
  Drop drop;
};

// Eight values of w or b (`fill` where there is none; anything behind the row's end).
template <class T, Edge EDGE>
__device__ __forceinline__ void load_param(const void* p, int32_t f32, int64_t c, int64_t d,
                                           float fill, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fill;
  } else if (f32) {
    take8<float, EDGE, false>(fetch8<float, EDGE>((const float*)p, c, d), c, d, v);
  } else {
    take8<T, EDGE, false>(fetch8<T, EDGE>((const T*)p, c, d), c, d, v);
  }
}

// v of the lane whose number differs as CTRL (a data-parallel move within 16 lanes) says.
template <int CTRL>
__device__ __forceinline__ float moved(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}

// The sums of a and b over aligned groups of L lanes, in every lane of them: pairs and quads, then
// mirrors (a group's halves hold equal values), then the lane rows through permlane swaps.
template <int L>
__device__ __forceinline__ void lane_sum2(float& a, float& b) {
  auto step = [&](float x, float y) { a += x, b += y; };
  if (L >= 2) step(moved<0xB1>(a), moved<0xB1>(b));    // quad_perm 1 0 3 2
  if (L >= 4) step(moved<0x4E>(a), moved<0x4E>(b));    // quad_perm 2 3 0 1
  if (L >= 8) step(moved<0x141>(a), moved<0x141>(b));  // mirror within 8
  if (L >= 16) step(moved<0x140>(a), moved<0x140>(b));  // mirror within 16
  if (L >= 32) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    const u32x2 ra = __builtin_amdgcn_permlane16_swap(ua, ua, false, false);
    const u32x2 rb = __builtin_amdgcn_permlane16_swap(ub, ub, false, false);
    a = __uint_as_float(ra[0]) + __uint_as_float(ra[1]);
    b = __uint_as_float(rb[0]) + __uint_as_float(rb[1]);
  }
  if (L >= 64) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    const u32x2 ra = __builtin_amdgcn_permlane32_swap(ua, ua, false, false);
    const u32x2 rb = __builtin_amdgcn_permlane32_swap(ub, ub, false, false);
    a = __uint_as_float(ra[0]) + __uint_as_float(ra[1]);
    b = __uint_as_float(rb[0]) + __uint_as_float(rb[1]);
  }
}

// Sums a and b over the TPR lanes (or waves) that share a row.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
  lane_sum2<TPR < 64 ? TPR : 64>(a, b);
  if (TPR > 64) {  // the workgroup is one row: every thread adds the waves' sums in one order
    constexpr int kWaves = TPR / 64;
    const int w = threadIdx.x >> 6;
    __syncthreads();  // the previous sums have been read
    if ((threadIdx.x & 63) == 0) {
      red[2 * w] = a;
      red[2 * w + 1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      a += red[2 * i];
      b += red[2 * i + 1];
    }
  }
}

// A row's inputs on their way: this lane's NV blocks of each table.
template <class T, int TPR, int NV, Edge EDGE, int TABLES>
struct RowIn {
  Raw<T> raw[TABLES][NV];

  __device__ __forceinline__ void fetch(int k, const void* p, int64_t ld, int64_t row, int64_t d,
                                        int t, int from = 0, int to = NV) {
    if (!p) return;
#pragma unroll
    for (int j = from; j < to; ++j)
      raw[k][j] = fetch8<T, EDGE>((const T*)p + row * ld, (int64_t)(j * TPR + t) * 8, d);
  }
  template <bool ZERO>
  __device__ __forceinline__ void take(int k, int j, int64_t d, int t, float (&v)[8]) const {
    take8<T, EDGE, ZERO>(raw[k][j], (int64_t)(j * TPR + t) * 8, d, v);
  }
};

// One block of act(x) with its mask, and with FACTORS its derivative.
template <bool FACTORS>
__device__ __forceinline__ void activate(const NormIn& in, uint64_t key, int64_t row, uint32_t cb,
                                         float (&h)[8], float (&fx)[8]) {
  if (FACTORS) {
#pragma unroll
    for (int e = 0; e < 8; ++e) fx[e] = 1.f;
  }
  if (in.drop.slope != 1.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool pos = h[e] > 0.f;
      if (FACTORS) fx[e] = pos ? 1.f : in.drop.slope;
      h[e] = pos ? h[e] : h[e] * in.drop.slope;
    }
  }
  if (in.dropping && (int64_t)cb * 8 < in.d) {
    float f[8];
    drop_factors(in.drop, key, row, cb, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[e] = masked(h[e], f[e]);
      if (FACTORS) fx[e] *= f[e];
    }
  }
}

// h of one row from x (table 0) and the residual (table 1), and with FACTORS dx / dh. PLAIN: h is
// x. What a lane holds behind the row's end is anything.
template <bool PLAIN, bool FACTORS, int TPR, int NV, class In>
__device__ __forceinline__ void form_h(const NormIn& in, uint64_t key, const In& raw, int64_t row,
                                       int t, float (&h)[NV][8], float (&fx)[NV][8]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    raw.template take<false>(0, j, in.d, t, h[j]);
    if (PLAIN) continue;
    activate<FACTORS>(in, key, row, (uint32_t)(j * TPR + t), h[j], fx[j]);
    if (in.res) {
      float r[8];
      raw.template take<false>(1, j, in.d, t, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] += r[e];
    }
  }
}

// 1 / sqrt(v): the hardware's estimate (1 ulp) and one Newton step, over the range where neither
// leaves the normal numbers; the exact root and quotient, some thirty instructions, elsewhere.
__device__ __forceinline__ float inv_sqrt(float v) {
  if (v > 1e-30f && v < 1e30f) {
    const float r = __builtin_amdgcn_rsqf(v);
    return fmaf(r, 0.5f * fmaf(-v * r, r, 1.f), r);
  }
  return 1.f / __builtin_sqrtf(v);
}

// h -> u in place; returns r. Behind the row's end u is finite where the row is (the gradients
// there are 0, and nothing of it is stored).
template <int TPR, int NV, Edge EDGE>
__device__ __forceinline__ float normalize(const NormIn& in, int t, float (&h)[NV][8],
                                           float* red) {
  const float inv = 1.f / (float)in.d;
  const int n = (int)in.d - t * 8;  // block j of this lane has n - j TPR 8 values in the row
  float s = 0.f, unused = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += EDGE == kFull || e < n - j * TPR * 8 ? h[j][e] : 0.f;
  row_sum2<TPR>(s, unused, red);
  const float mean = s * inv;
  float s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[j][e] = EDGE == kFull || e < n - j * TPR * 8 ? h[j][e] - mean : 0.f;
      s1 += h[j][e];
      s2 = fmaf(h[j][e], h[j][e], s2);
    }
  row_sum2<TPR>(s1, s2, red);
  const float off = s1 * inv;
  const float var = fmaxf(fmaf(-off, off, s2 * inv), 0.f);
  const float r = inv_sqrt(var + in.eps);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) h[j][e] = (h[j][e] - off) * r;
  return r;
}

template <class T, int TPR, int NV, Edge EDGE, bool PLAIN>
__global__ __launch_bounds__(TPR > kNormBlock ? TPR : kNormBlock) void norm_forward_kernel(
    NormIn in, T* __restrict__ y, int64_t ldy, T* __restrict__ hout, int64_t ldh) {
  constexpr int kBlock = TPR > kNormBlock ? TPR : kNormBlock;
  constexpr bool HELD = NV == 1;  // w and b stay in registers over a lane group's rows
  __shared__ float red[2 * kBlock / 64];
  const int t = threadIdx.x % TPR;
  const uint64_t key = in.dropping ? drop_key(in.drop) : 0;
  float w[8], b[8];
  auto params = [&](int j) {
    const int64_t c = (int64_t)(j * TPR + t) * 8;
    load_param<T, EDGE>(in.w, in.w_f32, c, in.d, 1.f, w);
    load_param<T, EDGE>(in.b, in.w_f32, c, in.d, 0.f, b);
  };
  const int64_t stride = (int64_t)gridDim.x * (kBlock / TPR);
  int64_t row = (int64_t)blockIdx.x * (kBlock / TPR) + threadIdx.x / TPR;
  if (HELD && row < in.rows) params(0);
  for (; row < in.rows; row += stride) {  // the lanes of a row leave together
    RowIn<T, TPR, NV, EDGE, PLAIN ? 1 : 2> raw;
    raw.fetch(0, in.x, in.ldx, row, in.d, t);
    if (!PLAIN) raw.fetch(PLAIN ? 0 : 1, in.res, in.ldr, row, in.d, t);
    float h[NV][8], none[NV][8];
    form_h<PLAIN, false, TPR, NV>(in, key, raw, row, t, h, none);
    if (hout) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int64_t c = (int64_t)(j * TPR + t) * 8;
        store8<T, EDGE>(hout + row * ldh, c, in.d, h[j]);
      }
    }
    normalize<TPR, NV, EDGE>(in, t, h, red);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t c = (int64_t)(j * TPR + t) * 8;
      if (!HELD) params(j);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] = fmaf(h[j][e], w[e], b[e]);
      store8<T, EDGE>(y + row * ldy, c, in.d, h[j]);
    }
  }
}

// Rows of a workgroup's own fetch the next row while one is worked on (AHEAD: there are too few
// waves to hide the fetch otherwise: 8192 x 4096 bf16 143 -> 111 us). With up to 512 columns many
// waves are resident, and dy and dh are fetched when they are needed (2M x 64 fp32 block 963 -> 939
// us for fewer registers). With 1024 lanes, of 128 registers each, so is x again with its mask, and
// dw and db are summed in LDS (LATE: in registers they spilled: 5003 x 16384 bf16 743 us, in LDS
// 311).
template <class T, int TPR, int NV, Edge EDGE, bool PLAIN>
__global__ __launch_bounds__(TPR > kNormBlock ? TPR : kNormBlock,
                             NV == 1 && TPR <= 64 ? 4 : 1) void norm_backward_kernel(
    NormIn in, const T* __restrict__ dy, int64_t lddy, const T* __restrict__ dh, int64_t lddh,
    T* __restrict__ dx, int64_t lddx, T* __restrict__ dres, int64_t lddr,
    float* __restrict__ part) {
  constexpr int kBlock = TPR > kNormBlock ? TPR : kNormBlock;
  constexpr int kGroups = kBlock / TPR;
  constexpr bool AHEAD = TPR == 256 || TPR == 512, LATE = TPR > 512;
  __shared__ float red[2 * kBlock / 64];
  constexpr bool kWhenNeeded = LATE || (TPR <= 64 && NV == 1);
  constexpr int kWide = TPR * NV * 8;  // columns that a row's lanes hold
  __shared__ float join[LATE ? 2 * kWide : kBlock * 8];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.f / (float)in.d;
  const uint64_t key = in.dropping ? drop_key(in.drop) : 0;
  const int64_t stride = (int64_t)gridDim.x * kGroups;
  float aw[LATE ? 1 : NV][8] = {}, ab[LATE ? 1 : NV][8] = {};
  float* own = join + t * 8;  // LATE: this lane's columns' sums of block j at j * TPR * 8
  if (LATE) {
#pragma unroll
    for (int k = 0; k < 2 * NV; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) own[k * TPR * 8 + e] = 0.f;
  }
  constexpr int kDy = PLAIN ? 1 : 2, kDh = PLAIN ? 1 : 3;  // their places among the tables
  using In = RowIn<T, TPR, NV, EDGE, PLAIN ? 2 : 4>;
  auto fetch = [&](In& raw, int64_t row) {
    raw.fetch(0, in.x, in.ldx, row, in.d, t);
    if (!PLAIN) raw.fetch(1, in.res, in.ldr, row, in.d, t);
    if (!kWhenNeeded) {
      raw.fetch(kDy, dy, lddy, row, in.d, t);
      if (!PLAIN) raw.fetch(kDh, dh, lddh, row, in.d, t);
    }
  };
  In next;
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
  float w[8];
  if (NV == 1) load_param<T, EDGE>(in.w, in.w_f32, t * 8, in.d, 1.f, w);
  if (AHEAD && row < in.rows) fetch(next, row);
  for (; row < in.rows; row += stride) {
    In raw;
    if (AHEAD) {
      raw = next;
      if (row + stride < in.rows) fetch(next, row + stride);
    } else {
      fetch(raw, row);
    }
    float u[NV][8], fx[NV][8], g[NV][8];
    form_h<PLAIN, !LATE, TPR, NV>(in, key, raw, row, t, u, fx);
    const float r = normalize<TPR, NV, EDGE>(in, t, u, red);
    float s1 = 0.f, s2 = 0.f;
    if (kWhenNeeded) raw.fetch(kDy, dy, lddy, row, in.d, t);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      raw.template take<true>(kDy, j, in.d, t, g[j]);
      if (NV > 1) load_param<T, EDGE>(in.w, in.w_f32, (int64_t)(j * TPR + t) * 8, in.d, 1.f, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (LATE) {
          float* sum = own + j * TPR * 8 + e;
          sum[0] = fmaf(g[j][e], u[j][e], sum[0]);
          sum[kWide] += g[j][e];
        } else {
          aw[LATE ? 0 : j][e] = fmaf(g[j][e], u[j][e], aw[LATE ? 0 : j][e]);
          ab[LATE ? 0 : j][e] += g[j][e];
        }
        g[j][e] *= w[e];
        s1 += g[j][e];
        s2 = fmaf(g[j][e], u[j][e], s2);
      }
    }
    row_sum2<TPR>(s1, s2, red);
    s1 *= inv;
    s2 *= inv;
    if (kWhenNeeded && !PLAIN) raw.fetch(kDh, dh, lddh, row, in.d, t);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t c = (int64_t)(j * TPR + t) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) g[j][e] = r * (g[j][e] - fmaf(u[j][e], s2, s1));
      if (!PLAIN && dh) {
        float v[8];
        raw.template take<false>(kDh, j, in.d, t, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[j][e] += v[e];
      }
      if (!PLAIN && dres) store8<T, EDGE>(dres + row * lddr, c, in.d, g[j]);
      if (dx) {
        if (LATE && !PLAIN) {
          raw.fetch(0, in.x, in.ldx, row, in.d, t, j, j + 1);
          float a[8];
          raw.template take<false>(0, j, in.d, t, a);
          activate<true>(in, key, row, (uint32_t)(j * TPR + t), a, fx[j]);
        }
        if (!PLAIN) {
#pragma unroll
          for (int e = 0; e < 8; ++e) g[j][e] = masked(g[j][e], fx[j][e]);
        }
        store8<T, EDGE>(dx + row * lddx, c, in.d, g[j]);
      }
    }
  }
  if (!part) return;
  if (LATE) {
    float* out = part + (int64_t)blockIdx.x * 2 * in.d;
    __syncthreads();
    for (int64_t c = threadIdx.x; c < in.d; c += kBlock) {
      out[c] = join[c];
      out[in.d + c] = join[kWide + c];
    }
    return;
  }
  // this workgroup's sums: [2][d] at part + blockIdx.x * 2 d, joined over its lane groups
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e)
        join[threadIdx.x * 8 + e] = k ? ab[LATE ? 0 : j][e] : aw[LATE ? 0 : j][e];
      __syncthreads();
      constexpr int kCols = TPR * 8, kSlices = kBlock / kCols;
      if (kSlices > 1) {  // few columns: eight groups a thread, then the threads of a column
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q)
          s += join[(threadIdx.x / kCols * 8 + q) * kCols + threadIdx.x % kCols];
        __syncthreads();
        join[threadIdx.x] = s;
        __syncthreads();
      }
      constexpr int kLeft = kSlices > 1 ? kSlices : kGroups;
      for (int i = threadIdx.x; i < kCols; i += kBlock) {
        const int64_t c = (int64_t)j * kCols + i;
        if (c >= in.d) continue;
        float s = 0.f;
        for (int q = 0; q < kLeft; ++q) s += join[q * kCols + i];
        part[(int64_t)blockIdx.x * 2 * in.d + k * in.d + c] = s;
      }
    }
  }
}

// out[c] = sum over the n partial rows: 32 columns a workgroup (a line of 128 B), its threads in 32
// slices of the rows, eight loads of each in flight. 768 x 8192 values 5.2 us (16 columns, one
// load at a time: 8.5), 1024 x 128 3.8 (6.1).
constexpr int kSumCols = 32, kSumBlock = 1024;
template <class T>
__global__ __launch_bounds__(kSumBlock) void norm_sum_kernel(const float* __restrict__ part,
                                                             int64_t n, int64_t d,
                                                             T* __restrict__ dw,
                                                             T* __restrict__ db) {
  constexpr int kSlices = kSumBlock / kSumCols;
  __shared__ float red[kSlices][kSumCols + 1];
  const int lc = threadIdx.x % kSumCols, slice = threadIdx.x / kSumCols;
  const int64_t c = (int64_t)blockIdx.x * kSumCols + lc;
  float s = 0.f;
  if (c < 2 * d) {
#pragma unroll 8
    for (int64_t i = slice; i < n; i += kSlices) s += part[i * 2 * d + c];
  }
  red[slice][lc] = s;
  __syncthreads();
#pragma unroll
  for (int m = kSlices / 2; m > 0; m >>= 1) {
    if (slice < m) red[slice][lc] += red[slice + m][lc];
    __syncthreads();
  }
  if (slice == 0 && c < 2 * d) {
    T* out = c < d ? dw : db;
    if (out) out[c < d ? c : c - d] = (T)red[0][lc];
  }
}

// Lanes a row and blocks a lane by the row's width (blocks of eight columns), from one lane on (1M
// x 16 fp16 block: two lanes a row 66 us, eight 166; 1M x 32 bf16: four 125, eight 182): one wave
// holds up to 1024 columns, wider rows take a workgroup. Rows that fill every lane (a power of two
// from 16 columns on) have an instance without masks, and rows of a workgroup one for the norm
// alone, without registers for a residual and a mask.
template <int TPR, int NV, Edge EDGE, bool PLAIN>
struct Shape {
  static constexpr int tpr = TPR, nv = NV;
  static constexpr Edge edge = EDGE;
  static constexpr bool plain = PLAIN;
};
template <int TPR, int NV, class F>
static int one_wave(int64_t d, F&& f) {
  return d == TPR * NV * 8 ? f(Shape<TPR, NV, kFull, false>{})
                           : f(Shape<TPR, NV, kRagged, false>{});
}
template <int TPR, int NV, class F>
static int workgroup(int64_t d, bool plain, F&& f) {
  if (!plain) return f(Shape<TPR, NV, kRagged, false>{});
  return d == TPR * NV * 8 ? f(Shape<TPR, NV, kFull, true>{}) : f(Shape<TPR, NV, kRagged, true>{});
}
template <class F>
static int with_shape(int64_t d, bool plain, F&& f) {
  const int64_t nb = ceil_div(d, 8);
  if (d < 8) return f(Shape<1, 1, kNarrow, false>{});
  if (nb <= 2) return one_wave<2, 1>(d, f);
  if (nb <= 4) return one_wave<4, 1>(d, f);
  if (nb <= 8) return one_wave<8, 1>(d, f);
  if (nb <= 16) return one_wave<16, 1>(d, f);
  if (nb <= 32) return one_wave<32, 1>(d, f);
  if (nb <= 64) return one_wave<64, 1>(d, f);
  if (nb <= 128) return one_wave<64, 2>(d, f);
  if (nb <= 256) return workgroup<256, 1>(d, plain, f);
  if (nb <= 512) return workgroup<256, 2>(d, plain, f);
  if (nb <= 1024) return workgroup<512, 2>(d, plain, f);
  return workgroup<1024, 2>(d, plain, f);
}

// Rows a workgroup holds at a time, and workgroups of the backward pass: as many as are resident
// together (by the registers four, three or two a CU), each with one partial row. 8192 x 4096
// bf16, both passes: 768 workgroups 85.9 us, 512 88.5, 1024 96.3; 10 003 x 8192 fp32: 512 343, 768
// 364; 2M x 64 fp32 block: 1024 966, 1280 1361.
static int64_t rows_per_block(int64_t d) {
  int64_t r = 1;
  with_shape(d, false, [&](auto s) {
    r = s.tpr < kNormBlock ? kNormBlock / s.tpr : 1;
    return 0;
  });
  return r;
}
static int64_t backward_blocks(int64_t rows, int64_t d) {
  const int64_t b = ceil_div(rows, rows_per_block(d));
  const int64_t most = d <= 1024 ? 1024 : d <= 4096 ? 768 : 512;
  return b < most ? b : most;
}

static bool is_plain(const NormIn& in) {
  return !in.res && !in.dropping && in.drop.slope == 1.f;
}

static int check_norm(NormIn* in, const char* what, int32_t dtype, int32_t wdtype, int64_t rows,
                      int64_t d, const void* x, int64_t ldx, const void* res, int64_t ldr,
                      const void* w, const void* b, float eps, double p, uint64_t seed,
                      const int64_t* seed_ptr, uint32_t site, int64_t row0, float slope) {
  GNNREC_REQUIRE(dtype_ok(dtype), "%s: unknown dtype %d", what, dtype);
  GNNREC_REQUIRE(wdtype == dtype || wdtype == GNNREC_F32,
                 "%s: weight and bias must have the table's dtype or be float", what);
  GNNREC_REQUIRE(rows >= 0 && d >= 1, "%s: bad table size", what);
  if (d > kNormMaxD) {
    set_error("%s: rows of %lld values, at most %d are supported", what, (long long)d, kNormMaxD);
    return GNNREC_EUNSUPPORTED;
  }
  GNNREC_REQUIRE(eps >= 0.f, "%s: eps must not be negative", what);
  GNNREC_REQUIRE(rows <= (int64_t)0x7fffffff * rows_per_block(d), "%s: table too large", what);
  GNNREC_REQUIRE(rows == 0 || x, "%s: null pointer", what);
  Drop drop;
  if (!make_drop(&drop, what, p, seed, seed_ptr, site, row0, slope)) return GNNREC_EINVAL;
  *in = NormIn{rows, d, x, res, w, b, ldx, ldr, wdtype == GNNREC_F32, drop.border > 0, eps, drop};
  return GNNREC_OK;
}

}  // namespace gnnrec

using namespace gnnrec;

extern "C" int gnnrec_layer_norm_forward(int32_t dtype, int32_t wdtype, int64_t rows, int64_t d,
                                         const void* x, int64_t ldx, const void* res, int64_t ldr,
                                         const void* w, const void* b, float eps, double p,
                                         uint64_t seed, const int64_t* seed_ptr, uint32_t site,
                                         int64_t row0, float slope, void* y, int64_t ldy, void* h,
                                         int64_t ldh, gnnrec_stream_t stream) {
  NormIn in;
  const int rc = check_norm(&in, "layer_norm_forward", dtype, wdtype, rows, d, x, ldx, res, ldr, w,
                            b, eps, p, seed, seed_ptr, site, row0, slope);
  if (rc != GNNREC_OK || rows == 0) return rc;
  GNNREC_REQUIRE(y, "layer_norm_forward: null pointer");
  return with_dtype(dtype, [&](auto e) {
    using T = decltype(e);
    return with_shape(d, is_plain(in), [&](auto s) {
      using S = decltype(s);
      constexpr int kBlock = S::tpr > kNormBlock ? S::tpr : kNormBlock;
      // half-precision blocks are bound by instructions, and resident workgroups load w and b
      // once (100 003 x 201 fp16 block, both passes: 118 -> 110 us); the others by memory, and
      // one row a lane group keeps more of it in flight (2M x 64 fp32: 960 us, resident 1000)
      const int64_t want = ceil_div(rows, kBlock / S::tpr);
      // (a grid has fewer than 2^32 threads; its workgroups take the rows beyond in turn)
      const int64_t most = sizeof(T) == 2 && !S::plain ? 2048 : 0xffffffffll / kBlock;
      hipLaunchKernelGGL((norm_forward_kernel<T, S::tpr, S::nv, S::edge, S::plain>),
                         dim3((unsigned)(want < most ? want : most)),
                         dim3(kBlock), 0, as_hip(stream), in, (T*)y, ldy, (T*)h, ldh);
      return check_launch("layer_norm_forward");
    });
  });
}

extern "C" int64_t gnnrec_layer_norm_work_floats(int64_t rows, int64_t d) {
  if (rows <= 0 || d < 1 || d > kNormMaxD) return 0;
  return backward_blocks(rows, d) * 2 * d;
}

extern "C" int gnnrec_layer_norm_backward(int32_t dtype, int32_t wdtype, int64_t rows, int64_t d,
                                          const void* x, int64_t ldx, const void* res, int64_t ldr,
                                          const void* w, float eps, double p, uint64_t seed,
                                          const int64_t* seed_ptr, uint32_t site, int64_t row0,
                                          float slope, const void* dy, int64_t lddy,
                                          const void* dh, int64_t lddh, void* dx, int64_t lddx,
                                          void* dres, int64_t lddr, void* dw, void* db,
                                          float* work, gnnrec_stream_t stream) {
  NormIn in;
  const int rc = check_norm(&in, "layer_norm_backward", dtype, wdtype, rows, d, x, ldx, res, ldr,
                            w, nullptr, eps, p, seed, seed_ptr, site, row0, slope);
  if (rc != GNNREC_OK) return rc;
  GNNREC_REQUIRE(rows == 0 || dy, "layer_norm_backward: null pointer");
  GNNREC_REQUIRE(rows == 0 || !(dw || db) || work, "layer_norm_backward: null workspace");
  const int64_t blocks = rows > 0 ? backward_blocks(rows, d) : 0;
  if (rows > 0) {
    const int rc2 = with_dtype(dtype, [&](auto e) {
      using T = decltype(e);
      return with_shape(d, is_plain(in) && !dh && !dres, [&](auto s) {
        using S = decltype(s);
        constexpr int kBlock = S::tpr > kNormBlock ? S::tpr : kNormBlock;
        hipLaunchKernelGGL((norm_backward_kernel<T, S::tpr, S::nv, S::edge, S::plain>),
                           dim3((unsigned)blocks), dim3(kBlock), 0, as_hip(stream), in,
                           (const T*)dy, lddy, (const T*)dh, lddh, (T*)dx, lddx,
                           (T*)dres, lddr, dw || db ? work : nullptr);
        return check_launch("layer_norm_backward");
      });
    });
    if (rc2 != GNNREC_OK) return rc2;
  }
  if (!dw && !db) return GNNREC_OK;
  return with_dtype(wdtype, [&](auto e) {
    using T = decltype(e);
    hipLaunchKernelGGL((norm_sum_kernel<T>), dim3((unsigned)ceil_div(2 * d, kSumCols)),
                       dim3(kSumBlock), 0, as_hip(stream), work, blocks, d, (T*)dw, (T*)db);
    return check_launch("layer_norm_backward (sums)");
  });
}
