// 8-bit integers: rows quantized with one scale a row, and the dense linear over
// them (kq_int8.h states the product).  Rows past 64 run on the 256-column tiles
// of kq_mm16.h; up to 64 rows take one pass over the weights (few_rows_kernel).
#include "kq_int8_dense.h"
#include "kq_internal.h"

namespace kq {
namespace int8 {

using mm16::u32x2_t;
using mm16::u32x4_t;
using mm16::i32x4_t;

// ------------------------------------------------------------ quantization --

// The largest value of a wave.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}

// T threads take a row, 256 / T rows a workgroup.  The row's first 8 NV T
// elements stay in registers between its largest magnitude and its codes; what a
// longer row has besides is read again (from L2).
template <int DT, int T, int NV>
__global__ __launch_bounds__(256) void quantize_kernel(const char* __restrict__ x, int64_t ldx, int64_t rows, int64_t k,
                                                       int8_t* __restrict__ q, int64_t ldq, int64_t kp,
                                                       float* __restrict__ scale, int vec_in, int vec_out) {
  __shared__ uint32_t part[4];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (256 / T) + threadIdx.x / T;
  if (T < 256 && row >= rows) return;  // (T 256: the grid has a workgroup a row)
  const char* xr = x + row * ldx;
  Eight<DT> v[NV];
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t at = (int64_t)(t + i * T) * 8;
    if (at < k) v[i].load(xr, at, k, vec_in);
    else v[i].clear();
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) top = max(top, v[i].magnitude());
  for (int64_t at = (int64_t)(t + NV * T) * 8; at < k; at += T * 8) {
    Eight<DT> more;
    more.load(xr, at, k, vec_in);
    top = max(top, more.magnitude());
  }
  top = wave_max(top);
  if (T > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(part[0], part[1]), max(part[2], part[3]));
  }
  const float s = row_scale(top);
  const bool finite = top < 0x7f800000u;
  const float inv = 1.0f / s;
  if (t == 0) scale[row] = s;
  int8_t* qr = q + row * ldq;
  auto store = [&](const Eight<DT>& e, int64_t at) {
    u32x2_t c = {0u, 0u};
    if (finite) c = e.codes(s, inv);
    if (vec_out && at + 8 <= kp) {
      *reinterpret_cast<u32x2_t*>(qr + at) = c;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < kp) qr[at + i] = (int8_t)(c[i >> 2] >> 8 * (i & 3));
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t at = (int64_t)(t + i * T) * 8;
    if (at < kp) store(v[i], at);
  }
  for (int64_t at = (int64_t)(t + NV * T) * 8; at < kp; at += T * 8) {
    Eight<DT> more;
    if (at < k) more.load(xr, at, k, vec_in);
    else more.clear();
    store(more, at);
  }
}

// Columns [k, kp) of q are written as zeros.
static hipError_t quantize(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t k, int8_t* q, int64_t ldq,
                           int64_t kp, float* scale, hipStream_t st) {
  const int es = dtype == KQ_DT_F32 ? 4 : 2;
  const int vec_in = !kq_misaligned(x, 16) && ldx * es % 16 == 0;
  const int vec_out = !kq_misaligned(q, 8) && ldq % 8 == 0;
  auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (k <= 2048)
      quantize_kernel<DT, 64, 4><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(
          (const char*)x, ldx * es, rows, k, q, ldq, kp, scale, vec_in, vec_out);
    else
      quantize_kernel<DT, 256, 4><<<(unsigned)rows, 256, 0, st>>>((const char*)x, ldx * es, rows, k, q, ldq, kp, scale,
                                                                  vec_in, vec_out);
  };
  if (dtype == KQ_DT_BF16) run(std::integral_constant<int, KQ_DT_BF16>{});
  else if (dtype == KQ_DT_F16) run(std::integral_constant<int, KQ_DT_F16>{});
  else run(std::integral_constant<int, KQ_DT_F32>{});
  return hipGetLastError();
}

// ---------------------------------------------------------------- few rows --

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
  int m, n, k, mtiles;
  Epilogue epi;
};

constexpr int wave_lds(int mb, int r) { return (mb < 2 ? 2 : mb) * r * 1024; }

template <int DT, int OUT, int MB, int R, int P, bool TAIL>
__global__ __launch_bounds__(512) void few_rows_kernel(const FewArgs f) {
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
  // row tiles of one column tile run on one XCD, one after the other, and share its weights in that L2
  const int idx = (int)blockIdx.x / 8, xcd = (int)blockIdx.x % 8;
  const int n0 = ((idx / f.mtiles) * 8 + xcd) * 16 * R, m0 = (idx % f.mtiles) * 16 * MB;
  if (n0 >= f.n) return;
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
    constexpr int ES = DT == KQ_DT_F32 ? 4 : 2;
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
    static_assert(ES > 0, "");
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
    float y = (float)sum * s * sw0;
    if (f.epi.kind != EPI_OFF)
      y = epi_activate_any(f.epi, y + epi_bias_value(f.epi, bias_bits)) + epi_residual_value<OUT>(residual_bits);
    const int64_t to = (int64_t)(m0 + m) * f.ldc + n0 + n;
    if (OUT == KQ_DT_F32) static_cast<float*>(f.c)[to] = y;
    else static_cast<uint16_t*>(f.c)[to] = (uint16_t)mm16::pack16<OUT == KQ_DT_F16>(y, 0.0f);
  }
}

template <int DT, int OUT, int MB, int R, int P, bool TAIL>
static hipError_t launch_few(FewArgs f, hipStream_t st) {
  const int nwin = (f.k + WIN - 1) / WIN, waves = nwin < 8 ? nwin : 8;
  const size_t lds = (size_t)waves * wave_lds(MB, R) + (DT != DT_CODES ? (size_t)f.m * (nwin * WIN + 16) : 0);
  auto kern = few_rows_kernel<DT, OUT, MB, R, P, TAIL>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  f.mtiles = (f.m + 16 * MB - 1) / (16 * MB);
  const int64_t ntiles = ((int64_t)f.n + 16 * R - 1) / (16 * R);
  kern<<<(unsigned)(f.mtiles * ((ntiles + 7) / 8 * 8)), waves * 64, lds, st>>>(f);
  return hipGetLastError();
}

// Row blocks of weights a workgroup (R) and windows in flight a wave.  Cold weights, K = 7168, us by N:
//   rows       N = 12288             24576             129280
//   1     R 1  20.4          R 1, 2  28.8, 28.8        135, 132     (R 4: 20, 33, 142)
//   16    R 1  21.8          R 1, 2  39.0, 33.0        202, 160     (R 4, one window: 20.7, 37, 153)
//   32    R 1, 4  32.6, 24.8         61.0, 46.8        304, 191
//   64    R 1, 4  61.3, 34.5         119, 65.6         617, 275
// A block's reads of the activations (from L2) are shared by its R blocks; four need
// enough workgroups to cover the CUs (N = 4096: 19.7 and 23.0 at 32 rows).
template <int DT, int OUT, bool TAIL>
static hipError_t few_rows(const FewArgs& f, hipStream_t st) {
  if constexpr (DT != DT_CODES) {
    if (f.n >= 24576) return launch_few<DT, OUT, 1, 2, 2, TAIL>(f, st);
    return launch_few<DT, OUT, 1, 1, 2, TAIL>(f, st);
  } else {
    if (f.m <= 16) {
      if (f.n >= 24576) return launch_few<DT, OUT, 1, 2, 2, TAIL>(f, st);
      return launch_few<DT, OUT, 1, 1, 2, TAIL>(f, st);
    }
    if (f.m <= 32) {
      if (f.n >= 8192) return launch_few<DT, OUT, 2, 4, 2, TAIL>(f, st);
      return launch_few<DT, OUT, 2, 1, 2, TAIL>(f, st);
    }
    if (f.n >= 8192) return launch_few<DT, OUT, 4, 4, 1, TAIL>(f, st);
    return launch_few<DT, OUT, 4, 1, 2, TAIL>(f, st);
  }
}

// Whether up to FEW rows take the one-pass kernel or the tiles, where the weights
// are wide: the first reads them at 4.8 (32 rows) or 3.4 TB/s (64), the activations'
// reads beside them; the tiles at 5.9, in rounds of 0.9 us a step while they come
// from memory (N = 129280, 32 / 64 rows: 191 / 275 and 158 / 161 us; 24576 47 / 66 and 55 / 51).
static bool takes_few(int64_t m, int64_t n, int64_t k, int64_t cus) {
  if (m > FEW) return false;
  if (m <= 16) return true;
  const double bytes = (double)n * (double)k, few = bytes / (m <= 32 ? 4.8e6 : 3.4e6);
  const double rounds = (double)(((n + mm16::BN - 1) / mm16::BN + cus - 1) / cus) * 0.9 * (double)((k + 127) / 128);
  return few <= (rounds > bytes / 5.9e6 ? rounds : bytes / 5.9e6);
}

static inline int64_t up16(int64_t v) { return (v + 15) & ~(int64_t)15; }

// Rows that the few-row kernel quantizes itself.
static bool fuses(int a_dtype, int64_t m, int64_t k) {
  return a_dtype != KQ_DT_I8 && m <= FUSED && k <= FUSED_K;
}

template <int OUT>
static hipError_t few(int a_dtype, const FewArgs& f, hipStream_t st) {
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return f.k % WIN ? few_rows<DT, OUT, true>(f, st) : few_rows<DT, OUT, false>(f, st);
  };
  if (a_dtype == KQ_DT_BF16) return go(std::integral_constant<int, KQ_DT_BF16>{});
  if (a_dtype == KQ_DT_F16) return go(std::integral_constant<int, KQ_DT_F16>{});
  if (a_dtype == KQ_DT_F32) return go(std::integral_constant<int, KQ_DT_F32>{});
  return go(std::integral_constant<int, DT_CODES>{});
}

}  // namespace int8
}  // namespace kq

using namespace kq;
using namespace kq::int8;

extern "C" int kq_int8_quantize(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t k, int8_t* q, int64_t ldq,
                                float* scale, void* stream) {
  const char* fn = "kq_int8_quantize";
  if (dtype != KQ_DT_BF16 && dtype != KQ_DT_F16 && dtype != KQ_DT_F32)
    return kq_fail(KQ_ERR_INVALID, "%s: dtype must be bf16, f16 or f32", fn);
  if (rows < 0 || k < 1 || ldx < k || ldq < k)
    return kq_fail(KQ_ERR_INVALID, "%s: need rows >= 0, k >= 1, row strides of at least k (rows=%lld k=%lld strides %lld, %lld)",
                   fn, (long long)rows, (long long)k, (long long)ldx, (long long)ldq);
  if (rows > INT32_MAX / 2 || k > INT32_MAX / 2) return kq_fail(KQ_ERR_LIMIT, "%s: at most 2^30 rows and columns", fn);
  if (rows == 0) return KQ_OK;
  if (!x || !q || !scale) return kq_fail(KQ_ERR_INVALID, "%s: null buffer", fn);
  if (kq_misaligned(x, dtype == KQ_DT_F32 ? 4 : 2) || kq_misaligned(scale, 4))
    return kq_fail(KQ_ERR_INVALID, "%s: x and scale must be aligned to their type", fn);
  return kq_check_launch(quantize(dtype, x, ldx, rows, k, q, ldq, k, scale, (hipStream_t)stream), fn);
}

extern "C" int64_t kq_int8_linear_workspace_size(int a_dtype, int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 1) return -1;
  if (a_dtype == KQ_DT_I8 || fuses(a_dtype, m, k)) return 0;
  return up16(m * up16(k)) + 4 * m;  // the rows' codes and scales
}

extern "C" int kq_int8_linear(int a_dtype, const void* a, int64_t lda, const float* a_scale, const int8_t* w,
                              const float* w_scale, int64_t m, int64_t n, int64_t k, int activation, const void* bias,
                              int bias_dtype, const void* residual, int64_t ldr, int out_dtype, void* c, int64_t ldc,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "kq_int8_linear";
  const bool codes = a_dtype == KQ_DT_I8;
  if (!codes && a_dtype != KQ_DT_BF16 && a_dtype != KQ_DT_F16 && a_dtype != KQ_DT_F32)
    return kq_fail(KQ_ERR_INVALID, "%s: input dtype must be i8, bf16, f16 or f32", fn);
  if (out_dtype != KQ_DT_BF16 && out_dtype != KQ_DT_F16 && out_dtype != KQ_DT_F32)
    return kq_fail(KQ_ERR_INVALID, "%s: output dtype must be bf16, f16 or f32", fn);
  if (m < 0 || n < 0 || k < 16 || k % 16 || lda < k || (codes && lda % 16) || ldc < n || (residual && ldr < n))
    return kq_fail(KQ_ERR_INVALID,
                   "%s: need k %% 16 == 0, lda >= k (of codes a multiple of 16), ldc >= n, ldr >= n "
                   "(m=%lld n=%lld k=%lld lda=%lld ldc=%lld ldr=%lld)",
                   fn, (long long)m, (long long)n, (long long)k, (long long)lda, (long long)ldc, (long long)ldr);
  if (activation < KQ_LIN_NONE || activation > KQ_LIN_GELU_TANH)
    return kq_fail(KQ_ERR_INVALID, "%s: unknown activation %d", fn, activation);
  if (bias && bias_dtype != KQ_DT_BF16 && bias_dtype != KQ_DT_F32)
    return kq_fail(KQ_ERR_INVALID, "%s: bias dtype must be bf16 or f32", fn);
  if (k > MAX_K || m > INT32_MAX / 2 || n > INT32_MAX / 2 || (codes && lda > mm16::MAX_LD) ||
      ((m + 255) / 256) * ((n + 255) / 256) > INT32_MAX / 2)
    return kq_fail(KQ_ERR_LIMIT, "%s: at most k = %lld (the int32 sums), 2^30 rows, columns and tiles, code rows 2^22 apart",
                   fn, (long long)MAX_K);
  if (m == 0 || n == 0) return KQ_OK;
  if (!a || !w || !w_scale || !c || (codes && !a_scale)) return kq_fail(KQ_ERR_INVALID, "%s: null buffer", fn);
  const int os = out_dtype == KQ_DT_F32 ? 4 : 2;
  if (kq_misaligned(a, codes ? 16 : a_dtype == KQ_DT_F32 ? 4 : 2) || kq_misaligned(w, 16) || kq_misaligned(w_scale, 4) ||
      kq_misaligned(a_scale, 4) || kq_misaligned(c, os) || kq_misaligned(residual, os) ||
      kq_misaligned(bias, bias_dtype == KQ_DT_F32 ? 4 : 2) || kq_misaligned(workspace, 16))
    return kq_fail(KQ_ERR_INVALID, "%s: weights, codes and workspace must be 16-byte aligned, the others to their type", fn);
  const int64_t need = kq_int8_linear_workspace_size(a_dtype, m, n, k);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return kq_fail(KQ_ERR_INVALID, "%s: workspace needs %lld bytes", fn, (long long)need);
  hipStream_t st = (hipStream_t)stream;
  Epilogue e = make_epilogue(activation);
  if (activation == KQ_LIN_NONE && !bias && !residual) e.kind = EPI_OFF;
  e.bias = bias;
  e.bias_f32 = bias_dtype == KQ_DT_F32;
  e.residual = residual;
  e.ldr = ldr;
  const char* rows = (const char*)a;
  int64_t ld = lda;
  const float* sx = a_scale;
  const bool fused = fuses(a_dtype, m, k);
  if (!codes && !fused) {
    int8_t* q = (int8_t*)workspace;
    float* s = (float*)((char*)workspace + up16(m * k));
    const hipError_t err = quantize(a_dtype, a, lda, m, k, q, k, k, s, st);
    if (err != hipSuccess) return kq_check_launch(err, "kq_int8_linear/quantize");
    rows = (const char*)q;
    ld = k;
    sx = s;
  } else if (!codes) {
    ld = lda * (a_dtype == KQ_DT_F32 ? 4 : 2);
  }
  int cus = 0;
  if (m > 16 && m <= FEW) {
    int dev = 0;
    hipError_t err = st ? hipStreamGetDevice(st, &dev) : hipGetDevice(&dev);
    if (err == hipSuccess) err = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
    if (err != hipSuccess) return kq_check_launch(err, fn);
  }
  if (takes_few(m, n, k, cus > 0 ? cus : 1)) {
    const FewArgs f{rows, ld, sx, w, w_scale, c, ldc, (int)m, (int)n, (int)k, 1, e};
    const int dt = fused ? a_dtype : KQ_DT_I8;
    const hipError_t err = out_dtype == KQ_DT_BF16  ? few<KQ_DT_BF16>(dt, f, st)
                           : out_dtype == KQ_DT_F16 ? few<KQ_DT_F16>(dt, f, st)
                                                    : few<KQ_DT_F32>(dt, f, st);
    return kq_check_launch(err, fn);
  }
  DenseArgs g{};
  g.a = rows;
  g.w = (const char*)w;
  g.sx = sx;
  g.sw = w_scale;
  g.out = (char*)c;
  g.lda = (uint32_t)ld;
  g.ldw = (uint32_t)k;
  g.ld = ldc * os;
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  g.epi = e;
  g.pieces = os == 2 && n % 8 == 0 && ldc % 8 == 0 && !kq_misaligned(c, 16) &&
             (!residual || (ldr % 8 == 0 && !kq_misaligned(residual, 16)));
  return kq_check_launch(out_dtype == KQ_DT_BF16  ? dense_bf16(g, st)
                         : out_dtype == KQ_DT_F16 ? dense_f16(g, st)
                                                  : dense_f32(g, st), fn);
}
