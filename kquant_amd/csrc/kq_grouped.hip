// Matrix products grouped by expert with ragged sizes: rows sorted by group
// times that group's dense 16-bit weight, and both gradients.
//
//   forward  y[r]  = W_g x[r]                 for the rows r of group g
//   dx       dx[r] = W_g^T dy[r]
//   dw       dW_g  = sum over r of dy[r] x[r]^T
//
// All three run on the tiles of kq_mm16.h: the weight is read along its rows in
// the forward pass and across them for dx, and dw contracts over the rows of a
// group, both operands read across.  Group sizes stay on the device (offsets),
// so each workgroup numbers the tiles itself.
#include "kq_grouped.h"

namespace kq {
namespace grouped {

template <int MODE>
static hipError_t launch(int dtype, const Args& g, hipStream_t st) {
  int64_t grid;
  bool stream;
  if (const hipError_t e = plan<MODE>(g, st, grid, stream); e != hipSuccess) return e;
  auto run = [&](auto streamed) {
    constexpr bool S = MODE != DW && streamed.value;
    if (dtype == KQ_DT_F16) grouped_kernel<MODE, mm16::F16, S><<<(unsigned)grid, mm16::THREADS, 0, st>>>(g);
    else grouped_kernel<MODE, mm16::BF16, S><<<(unsigned)grid, mm16::THREADS, 0, st>>>(g);
  };
  if (stream) run(std::true_type{});
  else run(std::false_type{});
  return hipGetLastError();
}

static int check(const char* fn, int dtype, int64_t rows, int groups, int64_t n, int64_t k, int64_t ld_n, int64_t ld_k,
                 const int64_t* offsets, const void* a, const void* b, const void* c) {
  if (dtype != KQ_DT_BF16 && dtype != KQ_DT_F16) return kq_fail(KQ_ERR_INVALID, "%s: dtype must be bf16 or f16", fn);
  if (rows < 0 || groups < 1 || n <= 0 || k <= 0 || n % 8 || k % 8 || ld_n < n || ld_k < k || ld_n % 8 || ld_k % 8)
    return kq_fail(KQ_ERR_INVALID,
                   "%s: need groups >= 1, n %% 8 == 0, k %% 8 == 0, row strides of at least n and k, multiples of 8 "
                   "(rows=%lld groups=%d n=%lld k=%lld strides %lld, %lld)",
                   fn, (long long)rows, groups, (long long)n, (long long)k, (long long)ld_n, (long long)ld_k);
  const int64_t tiles_n = (n + 255) / 256, tiles_k = (k + 255) / 256;
  if (groups > MAX_GROUPS || rows > INT32_MAX / 2 || ld_n > mm16::MAX_LD || ld_k > mm16::MAX_LD ||
      (int64_t)groups * tiles_n * tiles_k > INT32_MAX / 2 ||
      (rows / 256 + groups) * (tiles_n > tiles_k ? tiles_n : tiles_k) > INT32_MAX / 2)
    return kq_fail(KQ_ERR_LIMIT, "%s: at most %d groups, 2^30 rows and tiles, rows of 2^22 elements", fn, MAX_GROUPS);
  if (!offsets || kq_misaligned(offsets, 8)) return kq_fail(KQ_ERR_INVALID, "%s: offsets must be int64 on the device", fn);
  if (kq_misaligned(a, 16) || kq_misaligned(b, 16) || kq_misaligned(c, 16))
    return kq_fail(KQ_ERR_INVALID, "%s: operands must be 16-byte aligned", fn);
  return KQ_OK;
}

}  // namespace grouped
}  // namespace kq

using namespace kq;

extern "C" int kq_grouped_linear(int dtype, const void* x, int64_t ldx, int64_t rows, const int64_t* offsets, int groups,
                                 const void* w, int64_t n, int64_t k, void* y, int64_t ldy, void* stream) {
  if (int rc = grouped::check("kq_grouped_linear", dtype, rows, groups, n, k, ldy, ldx, offsets, x, w, y)) return rc;
  if (rows == 0) return KQ_OK;
  const grouped::Args g{(const char*)x, (const char*)w, (char*)y, (uint32_t)(2 * ldx), (uint32_t)(2 * k),
                        (uint32_t)(2 * ldy), offsets, rows, groups, (int)n, (int)k};
  return kq_check_launch(grouped::launch<grouped::FORWARD>(dtype, g, (hipStream_t)stream), "kq_grouped_linear");
}

extern "C" int kq_grouped_linear_dx(int dtype, const void* dy, int64_t lddy, int64_t rows, const int64_t* offsets,
                                    int groups, const void* w, int64_t n, int64_t k, void* dx, int64_t lddx,
                                    void* stream) {
  if (int rc = grouped::check("kq_grouped_linear_dx", dtype, rows, groups, n, k, lddy, lddx, offsets, dy, w, dx)) return rc;
  if (rows == 0) return KQ_OK;
  const grouped::Args g{(const char*)dy, (const char*)w, (char*)dx, (uint32_t)(2 * lddy), (uint32_t)(2 * k),
                        (uint32_t)(2 * lddx), offsets, rows, groups, (int)n, (int)k};
  return kq_check_launch(grouped::launch<grouped::DX>(dtype, g, (hipStream_t)stream), "kq_grouped_linear_dx");
}

extern "C" int kq_grouped_linear_dw(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t rows,
                                    const int64_t* offsets, int groups, int64_t n, int64_t k, void* dw, void* stream) {
  if (int rc = grouped::check("kq_grouped_linear_dw", dtype, rows, groups, n, k, lddy, ldx, offsets, dy, x, dw)) return rc;
  const grouped::Args g{(const char*)dy, (const char*)x, (char*)dw, (uint32_t)(2 * lddy), (uint32_t)(2 * ldx),
                        (uint32_t)(2 * k), offsets, rows, groups, (int)n, (int)k};
  return kq_check_launch(grouped::launch<grouped::DW>(dtype, g, (hipStream_t)stream), "kq_grouped_linear_dw");
}
