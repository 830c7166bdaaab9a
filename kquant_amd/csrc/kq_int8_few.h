// The int8 product for few activation rows: one pass over the weights, for the
// linear and for the products grouped by expert.
#pragma once

#include "kq_int8.h"

namespace kq {
namespace int8 {

using mm16::u32x2_t;
using mm16::u32x4_t;
using mm16::i32x4_t;

// The largest value of a wave.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}

// What bounds it: the weight bytes.  A workgroup owns 16 R weight rows and each
// of its waves a run of 128-k windows of them, so N / (16 R) workgroups of
// independent waves keep the whole chip's loads in flight.
//  * a window of 16 weight rows is 16 lines of 128 bytes: 8 lanes load a line,
//    nontemporally, and the 16-byte pieces that lane (r, g) multiplies (row r,
//    pieces g and 4 + g; the MFMA sums over any assignment of k) come out of
//    2 KiB of the wave's own LDS.
//  * rows of activations: codes are read from memory as they are multiplied;
//    up to FUSED rows in 16 or 32 bits are quantized by every workgroup itself
//    while its first weights are on their way, into LDS, which saves the launch.
//  * P windows are in flight a wave; the last ones reload the wave's final
//    window instead of branching, so the compiler counts its waits exactly.
//  * the waves' int32 sums meet in LDS: exact, in any order.
// Rows past M or N are read at the last valid row and not stored; pieces past K
// (TAIL: K is no multiple of 128) multiply zeros.
constexpr int WIN = 128;
constexpr int FEW = 64;          // rows
constexpr int FUSED = 4;         // rows
constexpr int FUSED_K = 8192;    // and elements of a row: two pieces of 8 for each of 512 threads
constexpr int DT_CODES = 4;      // a_dtype of quantized rows

struct FewArgs {
  const char* a;
  int64_t lda;  // bytes
  const float* sx;
  const int8_t* w;
  const float* sw;
  void* c;
  int64_t ldc;
  int m, n, k;
  Epilogue epi;
};

constexpr int wave_lds(int mb, int r) { return (mb < 2 ? 2 : mb) * r * 1024; }

// Weight rows from n0 and rows from m0 on, by one workgroup; every thread of it calls.
template <int DT, int OUT, int MB, int R, int P, bool TAIL>
__device__ __forceinline__ void few_rows(const FewArgs& f, int n0, int m0) {
  constexpr bool FUSE = DT != DT_CODES;
  static_assert(!FUSE || MB == 1, "rows quantized here fill one block at most");
  struct Window {
    u32x4_t w[R][2], a[MB][2];
  };
  extern __shared__ __attribute__((aligned(16))) unsigned char few_lds[];
  __shared__ uint32_t tops[FUSED][8];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int waves = (int)blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int nwin = (f.k + WIN - 1) / WIN;
  const int w_begin = wave * nwin / waves, w_end = (wave + 1) * nwin / waves;
  const int8_t* wrow[R][2];
#pragma unroll
  for (int j = 0; j < R; ++j)
#pragma unroll
    for (int q = 0; q < 2; ++q) wrow[j][q] = f.w + (int64_t)min(n0 + 16 * j + 8 * q + (lane >> 3), f.n - 1) * f.k;
  const char* arow[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) arow[i] = f.a + (int64_t)min(m0 + 16 * i + r, f.m - 1) * f.lda;
  unsigned char* const lines = few_lds + wave * wave_lds(MB, R);
  unsigned char* const codes = few_lds + waves * wave_lds(MB, R);
  const int ldcodes = nwin * WIN + 16;
  const unsigned char* const crow = codes + (r < f.m ? r : 0) * ldcodes;

  auto load_w = [&](int w, Window& v) {
    const int at = w * WIN + 16 * (lane & 7);
    const bool gone = TAIL && at >= f.k;
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        v.w[j][q] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(wrow[j][q] + (gone ? 0 : at)));
        if (gone) v.w[j][q] = u32x4_t{0u, 0u, 0u, 0u};
      }
  };
  auto load_a = [&](int w, Window& v) {
    if constexpr (!FUSE) {
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = w * WIN + 64 * h + 16 * g;
          v.a[i][h] = *reinterpret_cast<const u32x4_t*>(arow[i] + (TAIL && at >= f.k ? 0 : at));
        }
    }
  };
  i32x4_t acc[MB][R];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
  auto compute = [&](int w, Window v) {
    // the lines' pieces: row x's at c ^ x % 8, so that 8 rows' pieces fall on distinct banks; one wave's accesses to
    // LDS stay in order
    const int to = (lane >> 3) * 128 + 16 * ((lane & 7) ^ (lane >> 3));
    const int from = r * 128 + 16 * (g ^ (r & 7));  // and the piece 64 bytes on, at from ^ 64
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q) *reinterpret_cast<u32x4_t*>(lines + j * 2048 + q * 1024 + to) = v.w[j][q];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q) v.w[j][q] = *reinterpret_cast<const u32x4_t*>(lines + j * 2048 + (from ^ 64 * q));
    __builtin_amdgcn_wave_barrier();
    if constexpr (FUSE) {
#pragma unroll
      for (int h = 0; h < 2; ++h) v.a[0][h] = *reinterpret_cast<const u32x4_t*>(crow + w * WIN + 64 * h + 16 * g);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, v.a[i][h]),
                                                            __builtin_bit_cast(i32x4_t, v.w[j][h]), acc[i][j], 0, 0, 0);
  };

  // what the epilogue reads for this thread's first sum is on its way during the K loop
  constexpr int TILE = MB * R * 256;
  uint32_t bias_bits = 0, residual_bits = 0;
  float sw0 = 0.0f;
  constexpr int RES = OUT == KQ_DT_F32 ? KQ_DT_F32 : KQ_DT_BF16;
  auto load_tail = [&](int e) {
    const int n = n0 + e % (16 * R), m = m0 + e / (16 * R);
    if (e < TILE && m < f.m && n < f.n) {
      sw0 = f.sw[n];
      bias_bits = epi_bias_bits(f.epi, n);
      residual_bits = epi_residual_bits<RES>(f.epi, m, n);
    }
  };

  // (a wave without windows has w_end == w_begin: it loads a valid window and multiplies none)
  const int last = min(max(w_end - 1, w_begin), nwin - 1);
  Window v[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    load_w(min(w_begin + p, last), v[p]);
    load_a(min(w_begin + p, last), v[p]);
  }
  float sx[FUSED];
  if constexpr (FUSE) {
    const bool vec = f.lda % 16 == 0 && ((uintptr_t)f.a & 15) == 0;
    const int t = threadIdx.x, step = (int)blockDim.x * 8;
    Eight<DT> x[FUSED][2];
#pragma unroll
    for (int mm = 0; mm < FUSED; ++mm) {
      if (mm >= f.m) break;
      uint32_t top = 0u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (8 * t + i * step < f.k) x[mm][i].load(f.a + mm * f.lda, 8 * t + i * step, f.k, vec);
        else x[mm][i].clear();
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) top = max(top, x[mm][i].magnitude());
      top = wave_max(top);
      if (lane == 0) tops[mm][wave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int mm = 0; mm < FUSED; ++mm) {
      if (mm >= f.m) break;
      uint32_t top = 0u;
      for (int w = 0; w < waves; ++w) top = max(top, tops[mm][w]);
      sx[mm] = row_scale(top);
      const float inv = 1.0f / sx[mm];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = 8 * t + i * step;
        if (at < nwin * WIN) {
          u32x2_t c = {0u, 0u};
          if (top < 0x7f800000u) c = x[mm][i].codes(sx[mm], inv);
          *reinterpret_cast<u32x2_t*>(codes + mm * ldcodes + at) = c;
        }
      }
    }
    __syncthreads();
  }
  load_tail((int)threadIdx.x);
  {
    int w = w_begin;
    for (; w + P <= w_end; w += P) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        compute(w + p, v[p]);
        load_w(min(w + P + p, last), v[p]);
        load_a(min(w + P + p, last), v[p]);
      }
    }
#pragma unroll
    for (int p = 0; p < P - 1; ++p)
      if (w + p < w_end) compute(w + p, v[p]);
  }

  // D (16x16): lane holds column lane % 16, rows 4 (lane / 16) + j
  constexpr int STRIDE = wave_lds(MB, R) / 4;
  int* const red = reinterpret_cast<int*>(few_lds);
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j)
      *reinterpret_cast<i32x4_t*>(red + wave * STRIDE + (i * R + j) * 256 + lane * 4) = acc[i][j];
  __syncthreads();
  for (int e = (int)threadIdx.x; e < TILE; e += (int)blockDim.x) {
    const int n = e % (16 * R), m = e / (16 * R);
    if (m0 + m >= f.m || n0 + n >= f.n) continue;
    if (e != (int)threadIdx.x) load_tail(e);
    const int at = ((m >> 4) * R + (n >> 4)) * 256 + (16 * ((m & 15) >> 2) + (n & 15)) * 4 + (m & 3);
    int sum = red[at];
    for (int w = 1; w < waves; ++w) sum += red[w * STRIDE + at];
    float s;
    if constexpr (FUSE) {
      s = sx[0];
#pragma unroll
      for (int mm = 1; mm < FUSED; ++mm) s = m == mm ? sx[mm] : s;
    } else {
      s = f.sx[m0 + m];
    }
    const float y =
        added<OUT>(f.epi, finished_any<OUT>(f.epi, sum, s, sw0, epi_bias_value(f.epi, bias_bits)), residual_bits);
    const int64_t to = (int64_t)(m0 + m) * f.ldc + n0 + n;
    if (OUT == KQ_DT_F32) static_cast<float*>(f.c)[to] = y;
    else static_cast<uint16_t*>(f.c)[to] = (uint16_t)mm16::pack16<OUT == KQ_DT_F16>(y, 0.0f);
  }
}

template <int DT, int OUT, int MB, int R, int P, bool TAIL>
__global__ __launch_bounds__(512) void few_rows_kernel(const FewArgs f) {
  few_rows<DT, OUT, MB, R, P, TAIL>(f, (int)blockIdx.x * 16 * R, 0);  // (at most 16 MB rows)
}

}  // namespace int8
}  // namespace kq
