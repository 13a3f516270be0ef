// Dropout of a table with an optional LeakyReLU in front, forward and backward, gfx950.
//
//   y  = keep ? act(x) * s : 0              act(x) = x > 0 ? x : slope x
//   dx = keep ? dy * s * (x > 0 ? 1 : slope) : 0
//
// keep is drawn from the element's place (rowwise.h), so no mask is stored or read: the passes
// move 2 and 3 (2 without the LeakyReLU) elements a value. A dropped value is 0 whatever x
// holds there, infinities and NaN included.
//
// One thread takes one block of eight columns: one Philox block, 16-B accesses. Bound by memory:
// 2M x 64 fp32 forward 176 us (5.8 TB/s; torch's copy of 2 GiB reaches 4.9), backward 264 us (5.8);
// 65 537 x 321 bf16, rows of odd width and no alignment, 21 us each (4.0).
#include "rowwise.h"

namespace gnnrec {

constexpr int kDropBlock = 256;

template <class T, bool BWD, Edge EDGE>
__global__ __launch_bounds__(kDropBlock) void dropout_kernel(
    int64_t rows, int64_t d, int64_t nb, const T* __restrict__ x, int64_t ldx,
    const T* __restrict__ dy, int64_t lddy, T* __restrict__ out, int64_t ldo, Drop drop) {
  // items (row, block of eight columns) in row order; the 64-bit division is the block's own
  const int64_t base = block_index() * kDropBlock;
  const int64_t row_base = base / nb;
  const uint32_t in_row = (uint32_t)(base - row_base * nb) + threadIdx.x;
  const uint32_t q = in_row / (uint32_t)nb, cb = in_row - q * (uint32_t)nb;
  const int64_t row = row_base + q;
  if (row >= rows) return;
  const int64_t c = (int64_t)cb * 8;
  float f[8], v[8];
  if (!BWD) {
    const Raw<T> rx = fetch8<T, EDGE>(x + row * ldx, c, d);
    drop_factors(drop, drop_key(drop), row, cb, f);  // while the values are on their way
    take8<T, EDGE>(rx, c, d, v);
    if (drop.slope != 1.f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] > 0.f ? v[e] : v[e] * drop.slope;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = masked(v[e], f[e]);
  } else {
    const Raw<T> rdy = fetch8<T, EDGE>(dy + row * lddy, c, d);
    Raw<T> rx;
    if (drop.slope != 1.f) rx = fetch8<T, EDGE>(x + row * ldx, c, d);
    drop_factors(drop, drop_key(drop), row, cb, f);
    take8<T, EDGE>(rdy, c, d, v);
    if (drop.slope != 1.f) {
      float xv[8];
      take8<T, EDGE>(rx, c, d, xv);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = xv[e] > 0.f ? v[e] : v[e] * drop.slope;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = masked(v[e], f[e]);
  }
  store8<T, EDGE>(out + row * ldo, c, d, v);
}

template <bool BWD>
static int run_dropout(const char* what, int32_t dtype, int64_t rows, int64_t d, const void* x,
                       int64_t ldx, const void* dy, int64_t lddy, void* out, int64_t ldo, double p,
                       uint64_t seed, const int64_t* seed_ptr, uint32_t site, int64_t row0,
                       float slope, gnnrec_stream_t stream) {
  GNNREC_REQUIRE(dtype_ok(dtype), "%s: unknown dtype %d", what, dtype);
  GNNREC_REQUIRE(rows >= 0 && d >= 1 && d <= 0x7fffffff, "%s: bad table size", what);
  Drop drop;
  if (!make_drop(&drop, what, p, seed, seed_ptr, site, row0, slope)) return GNNREC_EINVAL;
  if (rows == 0) return GNNREC_OK;
  GNNREC_REQUIRE(out && (BWD ? dy : x) && (!BWD || slope == 1.f || x), "%s: null pointer", what);
  const int64_t nb = ceil_div(d, 8);
  GNNREC_REQUIRE(rows <= INT64_MAX / 8 / nb, "%s: table too large", what);
  const int64_t blocks = ceil_div(rows * nb, kDropBlock);
  GNNREC_REQUIRE(blocks <= 0x7fffffff, "%s: table too large", what);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto* kernel = d < 8        ? dropout_kernel<T, BWD, kNarrow>
                   : d % 8 == 0 ? dropout_kernel<T, BWD, kFull>
                                : dropout_kernel<T, BWD, kRagged>;
    hipLaunchKernelGGL(kernel, wide_grid(blocks, kDropBlock), dim3(kDropBlock), 0,
                       as_hip(stream), rows, d, nb, (const T*)x, ldx, (const T*)dy, lddy, (T*)out,
                       ldo, drop);
    return check_launch(what);
  });
}

}  // namespace gnnrec

using namespace gnnrec;

extern "C" int gnnrec_dropout_forward(int32_t dtype, int64_t rows, int64_t d, const void* x,
                                      int64_t ldx, void* y, int64_t ldy, double p, uint64_t seed,
                                      const int64_t* seed_ptr, uint32_t site, int64_t row0,
                                      float slope, gnnrec_stream_t stream) {
  return run_dropout<false>("dropout_forward", dtype, rows, d, x, ldx, nullptr, 0, y, ldy, p, seed,
                            seed_ptr, site, row0, slope, stream);
}

extern "C" int gnnrec_dropout_backward(int32_t dtype, int64_t rows, int64_t d, const void* x,
                                       int64_t ldx, const void* dy, int64_t lddy, void* dx,
                                       int64_t lddx, double p, uint64_t seed,
                                       const int64_t* seed_ptr, uint32_t site, int64_t row0,
                                       float slope, gnnrec_stream_t stream) {
  return run_dropout<true>("dropout_backward", dtype, rows, d, x, ldx, dy, lddy, dx, lddx, p, seed,
                           seed_ptr, site, row0, slope, stream);
}
