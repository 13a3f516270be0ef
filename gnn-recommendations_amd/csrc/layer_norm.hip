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

template <class T>
__device__ __forceinline__ void load_param(const void* p, int32_t f32, int64_t c, int64_t n,
                                           float fill, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fill;
  } else if (f32) {
    load8((const float*)p + c, n, v);
  } else {
    load8((const T*)p + c, n, v);
  }
}

// Sums a and b over the TPR lanes (or waves) that share a row.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
#pragma unroll
  for (int m = 1; m < (TPR < 64 ? TPR : 64); m <<= 1) {
    a += __shfl_xor(a, m);
    b += __shfl_xor(b, m);
  }
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

// h of one row (this lane's NV blocks) and, when there is one, its dx/dh factors.
template <class T, int TPR, int NV, bool FACTORS>
__device__ __forceinline__ void load_h(const NormIn& in, uint64_t key, int64_t row, int t,
                                       float (&h)[NV][8], float (&fx)[NV][8]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t c = (int64_t)(j * TPR + t) * 8, n = in.d - c;
    load8((const T*)in.x + row * in.ldx + c, n, h[j]);
    if (FACTORS) {
#pragma unroll
      for (int e = 0; e < 8; ++e) fx[j][e] = 1.f;
    }
    if (in.drop.slope != 1.f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool pos = h[j][e] > 0.f;
        if (FACTORS) fx[j][e] = pos ? 1.f : in.drop.slope;
        h[j][e] = pos ? h[j][e] : h[j][e] * in.drop.slope;
      }
    }
    if (in.dropping && n > 0) {
      float f[8];
      drop_factors(in.drop, key, row, (uint32_t)(j * TPR + t), f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[j][e] = f[e] != 0.f ? h[j][e] * f[e] : 0.f;
        if (FACTORS) fx[j][e] *= f[e];
      }
    }
    if (in.res) {
      float r[8];
      load8((const T*)in.res + row * in.ldr + c, n, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] += r[e];
    }
  }
}

// h -> u in place (columns behind the row's end: 0); returns r.
template <int TPR, int NV>
__device__ __forceinline__ float normalize(const NormIn& in, int t, float (&h)[NV][8],
                                           float* red) {
  const float inv = 1.f / (float)in.d;
  float s = 0.f, unused = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += h[j][e];
  row_sum2<TPR>(s, unused, red);
  const float mean = s * inv;
  float s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t n = in.d - (int64_t)(j * TPR + t) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[j][e] = e < n ? h[j][e] - mean : 0.f;
      s1 += h[j][e];
      s2 = fmaf(h[j][e], h[j][e], s2);
    }
  }
  row_sum2<TPR>(s1, s2, red);
  const float off = s1 * inv;
  const float var = fmaxf(fmaf(-off, off, s2 * inv), 0.f);
  const float r = 1.f / __builtin_sqrtf(var + in.eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t n = in.d - (int64_t)(j * TPR + t) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[j][e] = e < n ? (h[j][e] - off) * r : 0.f;
  }
  return r;
}

template <class T, int TPR, int NV>
__global__ __launch_bounds__(TPR > kNormBlock ? TPR : kNormBlock) void norm_forward_kernel(
    NormIn in, T* __restrict__ y, int64_t ldy, T* __restrict__ hout, int64_t ldh) {
  constexpr int kBlock = TPR > kNormBlock ? TPR : kNormBlock;
  __shared__ float red[2 * kBlock / 64];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (kBlock / TPR) + threadIdx.x / TPR;
  if (row >= in.rows) return;  // whole rows only: the lanes of a row leave together
  float h[NV][8], none[NV][8];
  load_h<T, TPR, NV, false>(in, in.dropping ? drop_key(in.drop) : 0, row, t, h, none);
  if (hout) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t c = (int64_t)(j * TPR + t) * 8;
      store8(hout + row * ldh + c, in.d - c, h[j]);
    }
  }
  normalize<TPR, NV>(in, t, h, red);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t c = (int64_t)(j * TPR + t) * 8, n = in.d - c;
    float w[8], b[8];
    load_param<T>(in.w, in.w_f32, c, n, 1.f, w);
    load_param<T>(in.b, in.w_f32, c, n, 0.f, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[j][e] = fmaf(h[j][e], w[e], b[e]);
    store8(y + row * ldy + c, n, h[j]);
  }
}

template <class T, int TPR, int NV>
__global__ __launch_bounds__(TPR > kNormBlock ? TPR : kNormBlock) void norm_backward_kernel(
    NormIn in, const T* __restrict__ dy, int64_t lddy, const T* __restrict__ dh, int64_t lddh,
    T* __restrict__ dx, int64_t lddx, T* __restrict__ dres, int64_t lddr,
    float* __restrict__ part) {
  constexpr int kBlock = TPR > kNormBlock ? TPR : kNormBlock;
  constexpr int kGroups = kBlock / TPR;
  __shared__ float red[2 * kBlock / 64];
  __shared__ float join[kBlock * 8];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.f / (float)in.d;
  const uint64_t key = in.dropping ? drop_key(in.drop) : 0;
  float aw[NV][8] = {}, ab[NV][8] = {};
  for (int64_t row = (int64_t)blockIdx.x * kGroups + group; row < in.rows;
       row += (int64_t)gridDim.x * kGroups) {
    float u[NV][8], fx[NV][8], g[NV][8];
    load_h<T, TPR, NV, true>(in, key, row, t, u, fx);
    const float r = normalize<TPR, NV>(in, t, u, red);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t c = (int64_t)(j * TPR + t) * 8, n = in.d - c;
      float w[8];
      load8(dy + row * lddy + c, n, g[j]);
      load_param<T>(in.w, in.w_f32, c, n, 1.f, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        aw[j][e] = fmaf(g[j][e], u[j][e], aw[j][e]);
        ab[j][e] += g[j][e];
        g[j][e] *= w[e];
        s1 += g[j][e];
        s2 = fmaf(g[j][e], u[j][e], s2);
      }
    }
    row_sum2<TPR>(s1, s2, red);
    s1 *= inv;
    s2 *= inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t c = (int64_t)(j * TPR + t) * 8, n = in.d - c;
#pragma unroll
      for (int e = 0; e < 8; ++e) g[j][e] = r * (g[j][e] - fmaf(u[j][e], s2, s1));
      if (dh) {
        float v[8];
        load8(dh + row * lddh + c, n, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[j][e] += v[e];
      }
      if (dres) store8(dres + row * lddr + c, n, g[j]);
      if (dx) {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[j][e] = fx[j][e] != 0.f ? g[j][e] * fx[j][e] : 0.f;
        store8(dx + row * lddx + c, n, g[j]);
      }
    }
  }
  if (!part) return;
  // this workgroup's sums: [2][d] at part + blockIdx.x * 2 d, joined over its lane groups
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) join[threadIdx.x * 8 + e] = k ? ab[j][e] : aw[j][e];
      __syncthreads();
      for (int i = threadIdx.x; i < TPR * 8; i += kBlock) {
        const int64_t c = (int64_t)j * TPR * 8 + i;
        if (c >= in.d) continue;
        float s = 0.f;
        for (int q = 0; q < kGroups; ++q) s += join[q * TPR * 8 + i];
        part[(int64_t)blockIdx.x * 2 * in.d + k * in.d + c] = s;
      }
    }
  }
}

// out[c] = sum over the n partial rows, 16 columns a workgroup, 64 threads a column.
constexpr int kSumCols = 16, kSumSlices = 64;
template <class T>
__global__ __launch_bounds__(kSumCols* kSumSlices) void norm_sum_kernel(
    const float* __restrict__ part, int64_t n, int64_t d, T* __restrict__ dw,
    T* __restrict__ db) {
  __shared__ float red[kSumSlices][kSumCols + 1];
  const int lc = threadIdx.x % kSumCols, slice = threadIdx.x / kSumCols;
  const int64_t c = (int64_t)blockIdx.x * kSumCols + lc;
  float s = 0.f;
  if (c < 2 * d)
    for (int64_t i = slice; i < n; i += kSumSlices) s += part[i * 2 * d + c];
  red[slice][lc] = s;
  __syncthreads();
#pragma unroll
  for (int m = kSumSlices / 2; m > 0; m >>= 1) {
    if (slice < m) red[slice][lc] += red[slice + m][lc];
    __syncthreads();
  }
  if (slice == 0 && c < 2 * d) {
    T* out = c < d ? dw : db;
    if (out) out[c < d ? c : c - d] = (T)red[0][lc];
  }
}

// Lanes a row and blocks a lane by the row's width (blocks of eight columns): one wave holds up
// to 2048 columns, wider rows take a workgroup.
template <class F>
static int with_shape(int64_t d, F&& f) {
  const int64_t nb = ceil_div(d, 8);
  if (nb <= 8) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
  if (nb <= 16) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
  if (nb <= 32) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
  if (nb <= 64) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  if (nb <= 128) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  if (nb <= 256) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
  if (nb <= 512) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
  if (nb <= 1024) return f(std::integral_constant<int, 512>{}, std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
}

// Rows a workgroup holds at a time, and workgroups of the backward pass: at most 1024 (four a
// CU), each with one partial row.
static int64_t rows_per_block(int64_t d) {
  int64_t r = 1;
  with_shape(d, [&](auto tpr, auto) {
    r = tpr.value < kNormBlock ? kNormBlock / tpr.value : 1;
    return 0;
  });
  return r;
}
static int64_t backward_blocks(int64_t rows, int64_t d) {
  const int64_t b = ceil_div(rows, rows_per_block(d));
  return b < 1024 ? b : 1024;
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
    return with_shape(d, [&](auto tpr, auto nv) {
      constexpr int kBlock = tpr.value > kNormBlock ? tpr.value : kNormBlock;
      hipLaunchKernelGGL((norm_forward_kernel<T, tpr.value, nv.value>),
                         dim3((unsigned)ceil_div(rows, kBlock / tpr.value)), dim3(kBlock), 0,
                         as_hip(stream), in, (T*)y, ldy, (T*)h, ldh);
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
      return with_shape(d, [&](auto tpr, auto nv) {
        constexpr int kBlock = tpr.value > kNormBlock ? tpr.value : kNormBlock;
        hipLaunchKernelGGL((norm_backward_kernel<T, tpr.value, nv.value>), dim3((unsigned)blocks),
                           dim3(kBlock), 0, as_hip(stream), in, (const T*)dy, lddy, (const T*)dh,
                           lddh, (T*)dx, lddx, (T*)dres, lddr, dw || db ? work : nullptr);
        return check_launch("layer_norm_backward");
      });
    });
    if (rc2 != GNNREC_OK) return rc2;
  }
  if (!dw && !db) return GNNREC_OK;
  return with_dtype(wdtype, [&](auto e) {
    using T = decltype(e);
    hipLaunchKernelGGL((norm_sum_kernel<T>), dim3((unsigned)ceil_div(2 * d, kSumCols)),
                       dim3(kSumCols * kSumSlices), 0, as_hip(stream), work, blocks, d, (T*)dw,
                       (T*)db);
    return check_launch("layer_norm_backward (sums)");
  });
}
