// What the row-wise kernels share (dropout, layer norm, the 4-bit tables): element types, loads
// and stores of eight neighbouring elements, and the dropout's counter-based generator.
#pragma once

#include "common.h"

namespace gnnrec {

// Tables of these kernels hold float, bfloat16 or half; all arithmetic is in 32 bits, and a
// result is rounded once (to nearest, ties to even) when it is stored.
using bf16_t = __bf16;
using f16_t = _Float16;

// Runs f(T{}) for the element type of a gnnrec_dtype value (already checked).
template <class F>
inline int with_dtype(int32_t t, F&& f) {
  if (t == GNNREC_F32) return f(float{});
  if (t == GNNREC_BF16) return f(bf16_t{});
  return f(f16_t{});
}
inline bool dtype_ok(int32_t t) { return t == GNNREC_F32 || t == GNNREC_BF16 || t == GNNREC_F16; }

// The grid of a kernel whose workgroups (of `block` threads) are numbered by block_index(), with
// at least `blocks` of them: HIP takes fewer than 2^32 threads in a dimension, and a table of 2^35
// values has more eights than that, so the workgroups beyond go to further rows of the grid.
inline dim3 wide_grid(int64_t blocks, int block) {
  const int64_t rows = ceil_div(blocks, 0xffffffffll / block);
  return dim3((unsigned)ceil_div(blocks, rows), (unsigned)rows);
}
__device__ __forceinline__ int64_t block_index() {
  return (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Eight neighbouring elements as they lie in memory. Aligned as one element only, so that rows of
// any width and stride load with 16-B instructions (the hardware takes unaligned vectors).
template <class T>
struct __attribute__((packed)) Eight {
  T v[8];
};
template <class T>
struct Raw {
  uint32_t w[2 * sizeof(T)];
};

// How the lanes' eights meet a row's end. kFull: every lane's eight columns lie in the row.
// kRagged: the row's last eight may be partial and lanes may start behind its end. kNarrow: the
// row has fewer than eight values.
enum Edge { kFull, kRagged, kNarrow };

// Columns c .. c + 7 of a row of d values, 0 behind its end (ZERO: also for a lane that starts
// there): fetch8 is the memory access alone, so that several are in flight, and take8 what
// follows it. No lane branches: a row's last, partial eight is read from the row's last eight
// values and shifted down, since a lane that loaded its few values one by one would hold up the
// wave for as many round trips.
template <class T, Edge EDGE>
__device__ __forceinline__ Raw<T> fetch8(const T* __restrict__ row, int64_t c, int64_t d) {
  if (EDGE != kNarrow) {
    const int64_t at = EDGE == kFull || c < d - 8 ? c : d - 8;
    return __builtin_bit_cast(Raw<T>, *reinterpret_cast<const Eight<T>*>(row + at));
  }
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < 8; ++i) e.v[i] = row[i < d ? i : d - 1];
  return __builtin_bit_cast(Raw<T>, e);
}

template <class T, Edge EDGE, bool ZERO = true>
__device__ __forceinline__ void take8(Raw<T> t, int64_t c, int64_t d, float (&v)[8]) {
  constexpr int kWords = 2 * sizeof(T), kPer = 4 / sizeof(T);  // elements a word
  if (EDGE == kRagged) {
    if (d & 7) {
      const int s = c > d - 8 ? (int)(c - d) & 7 : 0;
#pragma unroll
      for (int bit = 4; bit >= 1; bit >>= 1) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          uint32_t from;
          if (bit >= kPer) {
            from = i + bit / kPer < kWords ? t.w[i + bit / kPer] : 0u;
          } else {  // half a word
            from = (t.w[i] >> 16) | (i + 1 < kWords ? t.w[i + 1] << 16 : 0u);
          }
          t.w[i] = s & bit ? from : t.w[i];
        }
      }
    }
    if (ZERO) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) t.w[i] = c < d ? t.w[i] : 0u;
    }
  }
  const Eight<T> e = __builtin_bit_cast(Eight<T>, t);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = EDGE != kNarrow || (c == 0 && i < d) ? (float)e.v[i] : 0.f;
}

// Both at once, for any width.
template <class T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int64_t c, int64_t d,
                                      float (&v)[8]) {
  if (d >= 8) take8<T, kRagged>(fetch8<T, kRagged>(row, c, d), c, d, v);
  else take8<T, kNarrow>(fetch8<T, kNarrow>(row, c, d), c, d, v);
}

template <class T, Edge EDGE = kRagged>
__device__ __forceinline__ void store8(T* __restrict__ row, int64_t c, int64_t d,
                                       const float (&v)[8]) {
  T* p = row + c;
  if (EDGE == kFull || d - c >= 8) {
    Eight<T> t;
#pragma unroll
    for (int e = 0; e < 8; ++e) t.v[e] = (T)v[e];
    *reinterpret_cast<Eight<T>*>(p) = t;
  } else {
    const int n = (int)(d - c);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = (T)v[e];
  }
}

// ---- dropout ------------------------------------------------------------------------------
// Philox4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011): a keyed bijection of a 128-bit counter. Here the key is the seed and the
// counter (column / 8, row, site), so a block's 128 bits are the eight 16-bit draws of eight
// neighbouring columns of a row. A value depends on its place alone: not on the launch, the
// table's stride or the shard that holds the row, and the backward pass draws the same mask
// again instead of reading it.
struct Drop {
  const int64_t* seed_ptr;  // the seed in device memory (a captured graph's), or NULL
  uint64_t seed;
  uint32_t site;
  uint32_t border;  // a draw below it drops the value; 65536 drops all, 0 none
  float scale;      // 65536 / (65536 - border): the expectation is kept for the border used
  float slope;      // of the LeakyReLU in front (1: none)
  int64_t row0;     // global row of the table's first one
};

__device__ __forceinline__ uint64_t drop_key(const Drop& d) {
  return d.seed_ptr ? (uint64_t)*d.seed_ptr : d.seed;
}

__device__ __forceinline__ void philox(uint64_t key, uint32_t c0, uint64_t row, uint32_t site,
                                       uint32_t (&w)[4]) {
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
  uint32_t x0 = c0, x1 = (uint32_t)row, x2 = (uint32_t)(row >> 32), x3 = site;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)x0 * 0xD2511F53u, b = (uint64_t)x2 * 0xCD9E8D57u;
    x0 = (uint32_t)(b >> 32) ^ x1 ^ k0;
    x1 = (uint32_t)b;
    x2 = (uint32_t)(a >> 32) ^ x3 ^ k1;
    x3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = x0, w[1] = x1, w[2] = x2, w[3] = x3;
}

// v * f, and 0 where f is 0 whatever v is (an infinity, a NaN).
__device__ __forceinline__ float masked(float v, float f) {
  float r;  // the multiplication in which 0 times anything is 0: one instruction for three
  asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(v), "v"(f));
  return r;
}

// f[e] = scale where value e of block (row, cb) is kept, 0 where it is dropped.
__device__ __forceinline__ void drop_factors(const Drop& d, uint64_t key, int64_t row, uint32_t cb,
                                             float (&f)[8]) {
  uint32_t w[4];
  philox(key, cb, (uint64_t)(d.row0 + row), d.site, w);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    f[e] = ((w[e >> 1] >> (16 * (e & 1))) & 0xffffu) >= d.border ? d.scale : 0.f;
}

// Fills a Drop from the C ABI's arguments; false (and the message set) if they are unusable.
inline bool make_drop(Drop* d, const char* what, double p, uint64_t seed, const int64_t* seed_ptr,
                      uint32_t site, int64_t row0, float slope) {
  if (!(p >= 0.0 && p <= 1.0)) {
    set_error("%s: p must be between 0 and 1, got %g", what, p);
    return false;
  }
  if (row0 < 0 || row0 > (int64_t)1 << 62) {  // row0 + row stays within 63 bits
    set_error("%s: row0 must be between 0 and 2^62, got %lld", what, (long long)row0);
    return false;
  }
  const uint32_t border = (uint32_t)(p * 65536.0 + 0.5);
  *d = Drop{seed_ptr, seed, site, border,
            border < 65536 ? (float)(65536.0 / (65536 - border)) : 0.f, slope, row0};
  return true;
}

}  // namespace gnnrec
