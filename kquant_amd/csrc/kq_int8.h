// Products of 8-bit integers with a scale for each row and each column:
//
//   y[m][n] = act(sx[m] sw[n] sum over k of q[m][k] w[n][k] + bias[n]) + residual[m][n]
//
// The sums are int32 and exact (k < 2^17, so that 2^7 2^7 k stays below 2^31);
// the scaling, activation and residual are fp32, rounded once to the result's
// type.  Here: the code of a value, and the way of a tile's sums from the
// accumulators of kq_mm16.h to memory.
#pragma once

#include "kq_epilogue.h"
#include "kq_mm16.h"

namespace kq {
namespace int8 {

constexpr int64_t MAX_K = (1 << 17) - 16;  // the sums' bound, in whole 16-byte pieces

// A row's scale from the largest magnitude's bits: its product with the fp32 number
// nearest to 1 / 127, which is (1 - 2^-28) / 127, rounded once (within 9/16 of a step of
// a 127th of the magnitude, one step below the nearest in some 4.5 % of rows), and at
// least 2^-126, so that quotients by it
// need no subnormal scale.  A row with an infinity or a NaN has scale NaN (and
// codes 0): what it multiplies is NaN, and no other row is.
__device__ __forceinline__ float row_scale(uint32_t magnitude) {
  if (magnitude >= 0x7f800000u) return __builtin_nanf("");
  return fmaxf(__uint_as_float(magnitude) * 0x1.0204080000000p-7f, 0x1p-126f);
}

// The integer nearest to x / s, the even one of two, for |x| <= 127 s (1 + 2^-22)
// and inv near 1 / s.  n is off by one at most, and r = x - n s shows it: with
// s = S 2^e (S of 24 bits) r is a multiple of 2^(e-1), so every r with
// |r| <= s / 2 + 2^(e-1) is exact in fp32, a tie included, and a larger one is
// not rounded below that.
__device__ __forceinline__ int code(float x, float s, float inv) {
  float n = rintf(x * inv);
  const float r = fmaf(-n, s, x), half = 0.5f * s, away = fabsf(r);
  if (away >= half) {
    const bool odd = (int)n & 1;
    if (away > half || odd) n += r > 0.0f ? 1.0f : -1.0f;
  }
  return (int)n;
}

__device__ __forceinline__ uint32_t pack_codes(int a, int b, int c, int d) {
  return (uint32_t)(a & 0xff) | (uint32_t)(b & 0xff) << 8 | (uint32_t)(c & 0xff) << 16 | (uint32_t)d << 24;
}

// Eight values of a row as fp32, from memory's words (4 of 16-bit types, 8 of fp32).
template <int DT>
struct Eight {
  static constexpr int WORDS = DT == KQ_DT_F32 ? 8 : 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ uint32_t bits(int i) const {  // of the fp32 value
    if (DT == KQ_DT_F32) return w[i];
    const uint32_t h = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
    return DT == KQ_DT_BF16 ? h << 16 : __float_as_uint(f16_bits_to_f32(h));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  // elements [at, at + 8) of a row of `k`; vec: 16-byte pieces may be read (those past k are not)
  __device__ __forceinline__ void load(const void* row, int64_t at, int64_t k, bool vec) {
    constexpr int ES = DT == KQ_DT_F32 ? 4 : 2;
    const char* p = static_cast<const char*>(row) + at * ES;
    if (vec && at + 8 <= k) {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const mm16::u32x4_t v = *reinterpret_cast<const mm16::u32x4_t*>(p + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i + j] = v[j];
      }
      return;
    }
    clear();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (at + i >= k) break;
      if (ES == 4) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
      else w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << 16 * (i & 1);
    }
  }
  __device__ __forceinline__ uint32_t magnitude() const {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, bits(i) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ mm16::u32x2_t codes(float s, float inv) const {
    int c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = code(__uint_as_float(bits(i)), s, inv);
    mm16::u32x2_t v;
    v[0] = pack_codes(c[0], c[1], c[2], c[3]);
    v[1] = pack_codes(c[4], c[5], c[6], c[7]);
    return v;
  }
};

// ------------------------------------------------------- a tile's results --

// Of one tile: everything is at its row 0 and column 0.
struct Finish {
  const float* sx;
  const float* sw;
  char* out;
  int64_t ld;     // bytes
  Epilogue epi;   // kind EPI_OFF: no bias, activation or residual
  bool pieces;    // 16-bit results: every 8 columns of the results and the residual are a 16-byte piece
};

// Inverse of mm16::eight_columns (each of its steps is its own inverse): eight
// columns of one row, for a lane's four rows of one column, in 16-bit pairs
// w[j][0] (rows 0 and 1) and w[j][1] (2 and 3) of block j.
template <int WN>
__device__ __forceinline__ void four_rows(const mm16::u32x4_t (&q)[WN / 2], mm16::u32x2_t (&w)[WN]) {
  const bool odd = threadIdx.x & 4;
#pragma unroll
  for (int j = 0; j < WN; j += 2) {
    const mm16::u32x4_t v = q[j / 2];
    const uint32_t x0 = mm16::other_quad(odd ? v[0] : v[2]), x1 = mm16::other_quad(odd ? v[1] : v[3]);
    w[j][0] = odd ? x0 : v[0];
    w[j][1] = odd ? x1 : v[1];
    w[j + 1][0] = odd ? v[2] : x0;
    w[j + 1][1] = odd ? v[3] : x1;
  }
#pragma unroll
  for (int j = 0; j < WN; ++j) {
    uint32_t a = w[j][0], b = w[j][1];
    quad_transpose16(a, b);
    w[j][0] = a;
    w[j][1] = b;
  }
}

template <int OUT>
__device__ __forceinline__ float of16(uint32_t h) {
  return OUT == KQ_DT_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
}

// A value as it is in fp32.  Without this a product, sum or rounding to fp16 that
// follows may become one instruction with the one before it, here and not there, and
// a result would depend on the path that it took.
__device__ __forceinline__ float settled(float v) {
  asm("" : "+v"(v));
  return v;
}

// A sum scaled and finished up to the residual, in the same steps on every path.
template <int OUT, int EPI>
__device__ __forceinline__ float finished(const Epilogue& e, int sum, float sx, float sw, float bias) {
  const float t = settled((float)sum * sx);
  if (EPI == EPI_OFF) return settled(t * sw);
  const float v = settled(fmaf(t, sw, bias));
  return settled(OUT == KQ_DT_F32 ? epi_activate<EPI>(e, v) : epi_activate16<EPI>(e, v));
}
// the class decided at run time
template <int OUT>
__device__ __forceinline__ float finished_any(const Epilogue& e, int sum, float sx, float sw, float bias) {
  return e.kind == EPI_OFF       ? finished<OUT, EPI_OFF>(e, sum, sx, sw, bias)
         : e.kind == EPI_SIGMOID ? finished<OUT, EPI_SIGMOID>(e, sum, sx, sw, bias)
         : e.kind == EPI_ERF     ? finished<OUT, EPI_ERF>(e, sum, sx, sw, bias)
                                 : finished<OUT, EPI_CLAMP>(e, sum, sx, sw, bias);
}

// With the residual's bits, where there is one.
template <int OUT>
__device__ __forceinline__ float added(const Epilogue& e, float v, uint32_t bits) {
  return e.residual ? settled(v + epi_residual_value<OUT>(bits)) : v;
}

// Scales, finishes and stores a wave's blocks: rows below `rows` and columns
// below `cols` of the tile (element (i, j, r) as in mm16::each).  The scales of
// the wave's rows are in two registers, a row a lane, and reach their elements
// by lane exchanges; residuals are loaded a block row ahead.
template <int NB, int WN, int OUT, int EPI>
__device__ __forceinline__ void finish(const Finish& f, int rows, int cols, int wm, int wn, float16_t (&acc)[NB][WN],
                                       int lane) {
  static_assert(WN % 2 == 0, "column blocks in pairs");
  using mm16::u32x2_t;
  using mm16::u32x4_t;
  const int half = 4 * (lane >> 5);
  float sx[(NB + 1) / 2], sw[WN], bias[WN];
#pragma unroll
  for (int i = 0; i < (NB + 1) / 2; ++i) sx[i] = f.sx[min(wm + 64 * i + lane, rows - 1)];
#pragma unroll
  for (int j = 0; j < WN; ++j) {
    const int c = min(wn + 32 * j + (lane & 31), cols - 1);
    sw[j] = f.sw[c];
    bias[j] = EPI != EPI_OFF ? epi_bias(f.epi, c) : 0.0f;
  }
  // of element (i, j, r) with row scale s
  auto value = [&](float a, float s, int j) { return finished<OUT, EPI>(f.epi, __float_as_int(a), s, sw[j], bias[j]); };
  auto scale_of = [&](int i, int r) { return __shfl(sx[i / 2], 32 * (i & 1) + 8 * (r >> 2) + (r & 3) + half); };
  const bool residual = EPI != EPI_OFF && f.epi.residual;
  if (OUT != KQ_DT_F32 && f.pieces) {
    int row = wm + half + (lane & 3), col = wn + (lane & 28) + (lane & 4 ? 28 : 0);
    asm volatile("" : "+v"(row), "+v"(col));  // the elements' offsets are not kept from tile to tile
    u32x4_t next[4][WN / 2];  // of the four row quads to come
    auto fetch = [&](int t) {
      const int64_t at = (int64_t)min(row + 8 * t, rows - 1) * f.epi.ldr;
#pragma unroll
      for (int j = 0; j < WN / 2; ++j)
        next[t & 3][j] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(f.epi.residual) + at +
                                                           min(col + 64 * j, cols - 8));
    };
    if (residual) {
#pragma unroll
      for (int t = 0; t < 4; ++t) fetch(t);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      mm16::in_place(acc, i);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x2_t res[WN];
        if (residual) {
          four_rows<WN>(next[g], res);
          if (i + 1 < NB) fetch(4 * i + g + 4);
        }
        float s[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = scale_of(i, 4 * g + r);
        u32x4_t q[WN / 2];
        mm16::eight_columns<NB, WN, OUT == KQ_DT_F16>(acc, i, g, q, [&](int, int j, int r, float a) {
          float v = value(a, s[r & 3], j);
          if (residual) {
            const uint32_t h = res[j][(r & 3) >> 1];
            v += of16<OUT>(r & 1 ? h >> 16 : h & 0xffffu);
          }
          return residual ? settled(v) : v;
        });
        const int at = row + 32 * i + 8 * g;
        char* p = f.out + (int64_t)min(at, rows - 1) * f.ld + 2 * (int64_t)col;
#pragma unroll
        for (int j = 0; j < WN / 2; ++j)
          if (at < rows && col + 64 * j < cols) __builtin_nontemporal_store(q[j], reinterpret_cast<u32x4_t*>(p + 128 * j));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    return;
  }
  // one element a lane: 32 lanes store 32 columns of a row
  constexpr int ES = OUT == KQ_DT_F32 ? 4 : 2;
  int row = wm + half, col = wn + (lane & 31);
  asm volatile("" : "+v"(row), "+v"(col));
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    mm16::in_place(acc, i);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t res[4][WN];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < WN; ++j)
          res[r][j] = residual ? epi_residual_bits<OUT == KQ_DT_F32 ? KQ_DT_F32 : KQ_DT_BF16>(
                                     f.epi, min(row + 32 * i + 8 * g + r, rows - 1), min(col + 32 * j, cols - 1))
                               : 0u;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = row + 32 * i + 8 * g + r;
        const float s = scale_of(i, 4 * g + r);
        if (at >= rows) continue;
        char* p = f.out + (int64_t)at * f.ld + (int64_t)col * ES;
#pragma unroll
        for (int j = 0; j < WN; ++j) {
          const float v = added<OUT>(f.epi, value(acc[i][j][4 * g + r], s, j), res[r][j]);
          if (col + 32 * j >= cols) continue;
          if (OUT == KQ_DT_F32) *reinterpret_cast<float*>(p + 32 * ES * j) = v;
          else *reinterpret_cast<uint16_t*>(p + 32 * ES * j) = (uint16_t)mm16::pack16<OUT == KQ_DT_F16>(v, 0.0f);
        }
      }
    }
  }
}

}  // namespace int8
}  // namespace kq
