// 8-bit integers: rows quantized with one scale a row, and the dense linear over
// them (kq_int8.h states the product).  Rows past 64 run on the 256-column tiles
// of kq_mm16.h; up to 64 rows take one pass over the weights (few_rows_kernel).
#include "kq_int8_dense.h"
#include "kq_int8_few.h"
#include "kq_internal.h"

namespace kq {
namespace int8 {

// ------------------------------------------------------------ quantization --

// T threads take a row, 256 / T rows a workgroup.  The row's first 8 NV T
// elements stay in registers between its largest magnitude and its codes; what a
// longer row has besides is read again (from L2).
template <int DT, int T, int NV>
__global__ __launch_bounds__(256) void quantize_kernel(const char* __restrict__ x, int64_t ldx, int64_t rows, int64_t k,
                                                       int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                                                       int vec_in, int vec_out) {
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
    if (vec_out && at + 8 <= k) {
      *reinterpret_cast<u32x2_t*>(qr + at) = c;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < k) qr[at + i] = (int8_t)(c[i >> 2] >> 8 * (i & 3));
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t at = (int64_t)(t + i * T) * 8;
    if (at < k) store(v[i], at);
  }
  for (int64_t at = (int64_t)(t + NV * T) * 8; at < k; at += T * 8) {
    Eight<DT> more;
    more.load(xr, at, k, vec_in);
    store(more, at);
  }
}

static hipError_t quantize(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t k, int8_t* q, int64_t ldq,
                           float* scale, hipStream_t st) {
  const int es = dtype == KQ_DT_F32 ? 4 : 2;
  const int vec_in = !kq_misaligned(x, 16) && ldx * es % 16 == 0;
  const int vec_out = !kq_misaligned(q, 8) && ldq % 8 == 0;
  auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    constexpr int64_t MOST = 1 << 23;  // rows of a launch, which has less than 2^32 threads
    for (int64_t r = 0; r < rows; r += MOST) {
      const int64_t some = rows - r < MOST ? rows - r : MOST;
      const char* xr = (const char*)x + r * ldx * es;
      if (k <= 2048)
        quantize_kernel<DT, 64, 4><<<(unsigned)((some + 3) / 4), 256, 0, st>>>(xr, ldx * es, some, k, q + r * ldq, ldq,
                                                                               scale + r, vec_in, vec_out);
      else
        quantize_kernel<DT, 256, 4><<<(unsigned)some, 256, 0, st>>>(xr, ldx * es, some, k, q + r * ldq, ldq, scale + r,
                                                                    vec_in, vec_out);
    }
  };
  if (dtype == KQ_DT_BF16) run(std::integral_constant<int, KQ_DT_BF16>{});
  else if (dtype == KQ_DT_F16) run(std::integral_constant<int, KQ_DT_F16>{});
  else run(std::integral_constant<int, KQ_DT_F32>{});
  return hipGetLastError();
}

// A code times its scale, rounded once.  The fp32 product's rest is an fp32 number
// (both are multiples of the scale's last bit); a product that is not one is taken
// as the neighbour with an odd last bit, which no border between two 16-bit
// results has, so that the second rounding goes to the exact product's side.
template <int OUT>
__device__ __forceinline__ float value_of(int code, float s) {
  const float p = (float)code * s;
  if (OUT == KQ_DT_F32) return p;
  const float rest = fmaf((float)code, s, -p);
  const uint32_t bits = __float_as_uint(p);
  if ((rest < 0.0f || rest > 0.0f) && !(bits & 1)) return __uint_as_float((rest > 0.0f) == (p > 0.0f) ? bits + 1 : bits - 1);
  return p;
}

// T threads take a row, 256 / T rows a workgroup, as in quantize_kernel; eight codes
// a thread and step.  Bound by memory (12288 x 7168: 43 us to bf16, 6.2 TB/s; 112 to fp32, 3.9, its stores 32 bytes a lane).
template <int OUT, int T>
__global__ __launch_bounds__(256) void dequantize_kernel(const int8_t* __restrict__ q, int64_t ldq,
                                                         const float* __restrict__ scale, int64_t rows, int64_t k,
                                                         char* __restrict__ out, int64_t ldo, int vec) {
  constexpr int ES = OUT == KQ_DT_F32 ? 4 : 2;
  const int64_t row = (int64_t)blockIdx.x * (256 / T) + threadIdx.x / T;
  if (row >= rows) return;
  const float s = scale[row];
  const int8_t* qr = q + row * ldq;
  char* to = out + row * ldo;
  for (int64_t at = (int64_t)(threadIdx.x % T) * 8; at < k; at += T * 8) {
    if (vec && at + 8 <= k) {
      const u32x2_t c = *reinterpret_cast<const u32x2_t*>(qr + at);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = value_of<OUT>((int)(int8_t)(c[i >> 2] >> 8 * (i & 3)), s);
#pragma unroll
      for (int i = 0; i < 8; i += 16 / ES) {
        u32x4_t w;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = ES == 4 ? __float_as_uint(v[i + j]) : mm16::pack16<OUT == KQ_DT_F16>(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<u32x4_t*>(to + ES * (at + i)) = w;
      }
    } else {
      for (int i = 0; i < 8 && at + i < k; ++i) {
        const float v = value_of<OUT>(qr[at + i], s);
        if (ES == 4) *reinterpret_cast<float*>(to + 4 * (at + i)) = v;
        else *reinterpret_cast<uint16_t*>(to + 2 * (at + i)) = (uint16_t)mm16::pack16<OUT == KQ_DT_F16>(v, 0.0f);
      }
    }
  }
}

template <int OUT>
static hipError_t dequantize(const int8_t* q, int64_t ldq, const float* scale, int64_t rows, int64_t k, void* out, int64_t ldo,
                             hipStream_t st) {
  constexpr int ES = OUT == KQ_DT_F32 ? 4 : 2;
  constexpr int64_t MOST = 1 << 23;  // rows of a launch, which has less than 2^32 threads
  const int vec = !kq_misaligned(q, 8) && ldq % 8 == 0 && !kq_misaligned(out, 16) && ldo * ES % 16 == 0;
  for (int64_t r = 0; r < rows; r += MOST) {
    const int64_t some = rows - r < MOST ? rows - r : MOST;
    char* to = (char*)out + r * ldo * ES;
    if (k <= 2048)
      dequantize_kernel<OUT, 64><<<(unsigned)((some + 3) / 4), 256, 0, st>>>(q + r * ldq, ldq, scale + r, some, k, to, ldo * ES, vec);
    else
      dequantize_kernel<OUT, 256><<<(unsigned)some, 256, 0, st>>>(q + r * ldq, ldq, scale + r, some, k, to, ldo * ES, vec);
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------- few rows --

constexpr int64_t MAX_N = 1 << 26;  // a launch of 512 threads for 16 columns has less than 2^32

template <int DT, int OUT, int MB, int R, int P, bool TAIL>
static hipError_t launch_few(const FewArgs& f, hipStream_t st) {
  const int nwin = (f.k + WIN - 1) / WIN, waves = nwin < 8 ? nwin : 8;
  const size_t lds = (size_t)waves * wave_lds(MB, R) + (DT != DT_CODES ? (size_t)f.m * (nwin * WIN + 16) : 0);
  auto kern = few_rows_kernel<DT, OUT, MB, R, P, TAIL>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  kern<<<(unsigned)((f.n + 16 * R - 1) / (16 * R)), waves * 64, lds, st>>>(f);
  return hipGetLastError();
}

// Row blocks of weights a workgroup (R) and windows in flight a wave.  Cold weights, us:
//   rows  R, windows     12288 x 7168       24576 x 7168       129280 x 7168      65536 x 4096
//   1     1, 2 / 2, 2    16.3 / 18.4        28.4 / 28.6        137 / 132          54.6 / 52.8
//   8     1, 2 / 3, 2    18.0 / 16.8        31.9 / 29.9        154 / 145          62.3 / 60.5
//         2, 2 / 4, 1    19.8 / 18.6        29.8 / 34.6        139 / 148          58.2 / 51.9
//   16    1, 2 / 3, 2    21.3 / 18.3        38.6 / 31.7        201 / 159          78.0 / 66.5
//         2, 2 / 4, 1    21.9 / 20.6        32.6 / 37.2        159 / 153          64.5 / 53.6
//   32    1, 2 / 4, 2    32.6 / 24.8        61.0 / 46.8        304 / 191
//   64    1, 2 / 4, 1    61.3 / 34.5        119  / 65.6        617 / 275
// The activations' reads (from L2) are shared by a workgroup's R blocks; its
// workgroups have to cover the CUs (N = 4096: 19.7 with R 1 and 23.0 with R 4 at 32 rows).
// (Results in bf16; 16 rows of 129280 in fp32 take 162.)  The borders in N are measured ones at K = 7168, not
// sought between these columns: a shorter K gives each wave fewer windows, which no row of the table has.
template <int DT, int OUT, bool TAIL>
static hipError_t launch_few_rows(const FewArgs& f, hipStream_t st) {
  if constexpr (DT != DT_CODES) {
    // (blocks share a workgroup's quantization too: N = 24576, 1 / 2 rows 33.6 / 38.7 us with one, 29.9 / 32.4 with three)
    if (f.n >= 24576) return launch_few<DT, OUT, 1, 3, 2, TAIL>(f, st);
    return launch_few<DT, OUT, 1, 1, 2, TAIL>(f, st);
  } else {
    if (f.m <= 16) {
      if (f.m > 4 && f.n >= 12288 && f.n < 40960) return launch_few<DT, OUT, 1, 3, 2, TAIL>(f, st);
      if (f.m > 8 && f.n >= 40960) return launch_few<DT, OUT, 1, 4, 1, TAIL>(f, st);
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

// CUs of the stream's device (of the current one without a stream); 0 where there is none.
static int64_t device_cus(hipStream_t st) {
  int dev = 0, cus = 0;
  hipError_t e = st ? hipStreamGetDevice(st, &dev) : hipGetDevice(&dev);
  if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  if (e != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return cus;
}
static int workers(int64_t cus) { return cus >= 8 ? (int)(cus / 8 * 8) : 8; }

// Whether the few-row kernel quantizes the rows itself.  Every workgroup does so
// then, beside its first weights; a launch of its own takes 4.5 us.  K = 7168, us
// over the product of codes: N = 12288, 1 / 2 / 4 rows 1.0 / 2.4 / 5.6, 24576 1.3 / 3.3 / 6.5, 129280 6 / 17 / 35.
static bool fuses(int a_dtype, int64_t m, int64_t n, int64_t k) {
  return a_dtype != KQ_DT_I8 && m <= FUSED && k <= FUSED_K && (double)m * (double)n * (double)k <= 3.5e8;
}

template <int OUT>
static hipError_t few(int a_dtype, const FewArgs& f, hipStream_t st) {
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return f.k % WIN ? launch_few_rows<DT, OUT, true>(f, st) : launch_few_rows<DT, OUT, false>(f, st);
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
  return kq_check_launch(quantize(dtype, x, ldx, rows, k, q, ldq, scale, (hipStream_t)stream), fn);
}

extern "C" int kq_int8_dequantize(const int8_t* q, int64_t ldq, const float* scale, int64_t rows, int64_t k, int out_dtype,
                                  void* out, int64_t ldo, void* stream) {
  const char* fn = "kq_int8_dequantize";
  if (out_dtype != KQ_DT_BF16 && out_dtype != KQ_DT_F16 && out_dtype != KQ_DT_F32)
    return kq_fail(KQ_ERR_INVALID, "%s: output dtype must be bf16, f16 or f32", fn);
  if (rows < 0 || k < 1 || ldq < k || ldo < k)
    return kq_fail(KQ_ERR_INVALID, "%s: need rows >= 0, k >= 1, row strides of at least k (rows=%lld k=%lld strides %lld, %lld)",
                   fn, (long long)rows, (long long)k, (long long)ldq, (long long)ldo);
  if (rows == 0) return KQ_OK;
  if (!q || !scale || !out) return kq_fail(KQ_ERR_INVALID, "%s: null buffer", fn);
  if (kq_misaligned(out, out_dtype == KQ_DT_F32 ? 4 : 2) || kq_misaligned(scale, 4))
    return kq_fail(KQ_ERR_INVALID, "%s: scale and results must be aligned to their type", fn);
  hipStream_t st = (hipStream_t)stream;
  return kq_check_launch(out_dtype == KQ_DT_BF16  ? dequantize<KQ_DT_BF16>(q, ldq, scale, rows, k, out, ldo, st)
                         : out_dtype == KQ_DT_F16 ? dequantize<KQ_DT_F16>(q, ldq, scale, rows, k, out, ldo, st)
                                                  : dequantize<KQ_DT_F32>(q, ldq, scale, rows, k, out, ldo, st),
                         fn);
}

// The rows' codes and scales.
static int64_t codes_bytes(int a_dtype, int64_t m, int64_t n, int64_t k) {
  return a_dtype == KQ_DT_I8 || fuses(a_dtype, m, n, k) ? 0 : up16(m * up16(k)) + up16(4 * m);
}

extern "C" int64_t kq_int8_linear_workspace_size(int a_dtype, int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 1) return -1;
  int64_t bytes = codes_bytes(a_dtype, m, n, k);
  if (m == 0 || n == 0 || m <= 16) return bytes;
  const int64_t cus = device_cus(nullptr);
  if (cus > 0 && !takes_few(m, n, k, cus)) bytes += dense_plan(m, n, k, workers(cus), true).bytes;
  return bytes;
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
  if (k > MAX_K || m > INT32_MAX / 2 || n > MAX_N || (codes && lda > mm16::MAX_LD) ||
      ((m + 255) / 256) * ((n + 255) / 256) > INT32_MAX / 2)
    return kq_fail(KQ_ERR_LIMIT, "%s: at most k = %lld (the int32 sums), 2^30 rows and tiles, 2^26 columns, code rows 2^22 apart",
                   fn, (long long)MAX_K);
  if (m == 0 || n == 0) return KQ_OK;
  if (!a || !w || !w_scale || !c || (codes && !a_scale)) return kq_fail(KQ_ERR_INVALID, "%s: null buffer", fn);
  const int os = out_dtype == KQ_DT_F32 ? 4 : 2;
  if (kq_misaligned(a, codes ? 16 : a_dtype == KQ_DT_F32 ? 4 : 2) || kq_misaligned(w, 16) || kq_misaligned(w_scale, 4) ||
      kq_misaligned(a_scale, 4) || kq_misaligned(c, os) || kq_misaligned(residual, os) ||
      kq_misaligned(bias, bias_dtype == KQ_DT_F32 ? 4 : 2) || kq_misaligned(workspace, 16))
    return kq_fail(KQ_ERR_INVALID, "%s: weights, codes and workspace must be 16-byte aligned, the others to their type", fn);
  const int64_t need = codes_bytes(a_dtype, m, n, k);
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
  const bool fused = fuses(a_dtype, m, n, k);
  if (!codes && !fused) {
    int8_t* q = (int8_t*)workspace;
    float* s = (float*)((char*)workspace + up16(m * k));
    const hipError_t err = quantize(a_dtype, a, lda, m, k, q, k, s, st);
    if (err != hipSuccess) return kq_check_launch(err, "kq_int8_linear/quantize");
    rows = (const char*)q;
    ld = k;
    sx = s;
  } else if (!codes) {
    ld = lda * (a_dtype == KQ_DT_F32 ? 4 : 2);
  }
  const int64_t cus = m > 16 ? device_cus(st) : 1;
  if (cus <= 0) return kq_fail(KQ_ERR_HIP, "%s: no device", fn);
  if (takes_few(m, n, k, cus)) {
    const FewArgs f{rows, ld, sx, w, w_scale, c, ldc, (int)m, (int)n, (int)k, e};
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
  const int grid = workers(cus);
  DensePlan plan = dense_plan(m, n, k, grid, true);
  const bool split = plan.slices > 1 && workspace && workspace_bytes >= need + plan.bytes;
  if (plan.slices > 1 && !split) plan = dense_plan(m, n, k, grid, false);  // without room for the planes
  g.tm = plan.tm;
  g.mtiles = (g.m + g.tm - 1) / g.tm;
  g.ntiles = (g.n + mm16::BN - 1) / mm16::BN;
  g.slices = plan.slices;
  g.ks = plan.ks;
  g.planes = split ? (int*)((char*)workspace + need) : nullptr;
  return kq_check_launch(split                     ? dense_split(g, out_dtype, grid, st)
                         : out_dtype == KQ_DT_BF16 ? dense_bf16(g, grid, st)
                         : out_dtype == KQ_DT_F16  ? dense_f16(g, grid, st)
                                                   : dense_f32(g, grid, st),
                         fn);
}
