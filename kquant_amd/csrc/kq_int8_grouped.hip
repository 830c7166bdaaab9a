// 8-bit integers grouped by expert: y[r] = sx[r] sw_g (W_g q[r]) for the rows r of
// group g, on the tiles of the 16-bit grouped product with the int8 matrix
// instructions (kq_grouped.h, kq_int8.h).
#include "kq_grouped.h"

using namespace kq;

extern "C" int kq_int8_grouped_linear(const int8_t* x, int64_t ldx, const float* x_scale, int64_t rows,
                                      const int64_t* offsets, int groups, const int8_t* w, const float* w_scale,
                                      int64_t n, int64_t k, int out_dtype, void* y, int64_t ldy, void* stream) {
  const char* fn = "kq_int8_grouped_linear";
  if (out_dtype != KQ_DT_BF16 && out_dtype != KQ_DT_F16 && out_dtype != KQ_DT_F32)
    return kq_fail(KQ_ERR_INVALID, "%s: output dtype must be bf16, f16 or f32", fn);
  if (rows < 0 || groups < 1 || n <= 0 || k <= 0 || n % 8 || k % 16 || ldx < k || ldx % 16 || ldy < n || ldy % 8)
    return kq_fail(KQ_ERR_INVALID,
                   "%s: need groups >= 1, n %% 8 == 0, k %% 16 == 0, row strides of at least k and n, multiples of 16 and 8 "
                   "(rows=%lld groups=%d n=%lld k=%lld strides %lld, %lld)",
                   fn, (long long)rows, groups, (long long)n, (long long)k, (long long)ldx, (long long)ldy);
  const int64_t tiles_n = (n + 255) / 256;
  if (groups > grouped::MAX_GROUPS || rows > INT32_MAX / 2 || k > int8::MAX_K || ldx > mm16::MAX_LD ||
      ldy > mm16::MAX_LD || n > mm16::MAX_LD || (rows / 256 + groups) * tiles_n > INT32_MAX / 2)
    return kq_fail(KQ_ERR_LIMIT, "%s: at most %d groups, 2^30 rows and tiles, k = %lld, rows of 2^22 elements", fn,
                   grouped::MAX_GROUPS, (long long)int8::MAX_K);
  if (!offsets || kq_misaligned(offsets, 8)) return kq_fail(KQ_ERR_INVALID, "%s: offsets must be int64 on the device", fn);
  if (kq_misaligned(x, 16) || kq_misaligned(w, 16) || kq_misaligned(y, 16) || kq_misaligned(x_scale, 4) ||
      kq_misaligned(w_scale, 4))
    return kq_fail(KQ_ERR_INVALID, "%s: operands must be 16-byte aligned, scales 4", fn);
  if (rows == 0) return KQ_OK;
  if (!x || !x_scale || !w || !w_scale || !y) return kq_fail(KQ_ERR_INVALID, "%s: null buffer", fn);
  const int es = out_dtype == KQ_DT_F32 ? 4 : 2;
  const grouped::Args g{(const char*)x,     (const char*)w, (char*)y,  (uint32_t)ldx, (uint32_t)k,
                        (uint32_t)(es * ldy), offsets,        rows,     groups,        (int)n,
                        (int)(k / 2),         x_scale,        w_scale};
  hipStream_t st = (hipStream_t)stream;
  int64_t grid;
  bool stream_weights;
  hipError_t e = grouped::plan<grouped::FORWARD>(g, st, grid, stream_weights);
  if (e != hipSuccess) return kq_check_launch(e, fn);
  auto run = [&](auto out) {
    constexpr int OUT = decltype(out)::value;
    auto kern = stream_weights ? grouped::grouped_kernel<grouped::FORWARD, mm16::I8, true, OUT>
                               : grouped::grouped_kernel<grouped::FORWARD, mm16::I8, false, OUT>;
    kern<<<(unsigned)grid, mm16::THREADS, 0, st>>>(g);
  };
  if (out_dtype == KQ_DT_BF16) run(std::integral_constant<int, KQ_DT_BF16>{});
  else if (out_dtype == KQ_DT_F16) run(std::integral_constant<int, KQ_DT_F16>{});
  else run(std::integral_constant<int, KQ_DT_F32>{});
  return kq_check_launch(hipGetLastError(), fn);
}
