// 8-bit integers grouped by expert: y[r] = sx[r] sw_g (W_g q[r]) for the rows r of
// group g, on the tiles of the 16-bit grouped product with the int8 matrix
// instructions (kq_grouped.h, kq_int8.h).
//
// Few rows in all (FEW_EACH a group on average) take one pass over the weights of
// each group that has rows (kq_int8_few.h), 16 rows at a time.
#include "kq_grouped.h"
#include "kq_int8_few.h"

namespace kq {
namespace int8 {

// Workgroups: 16 R weight rows of a group each, then those that clear the rows of
// no group.  Group sizes are device data: a group without rows is left at once, one of more
// than 16 reads its weights again (from the caches) for the next 16.
template <int OUT, int R, int P, bool TAIL>
__global__ __launch_bounds__(512) void grouped_few_kernel(const grouped::Args g, int k, int tiles) {
  constexpr int ES = OUT == KQ_DT_F32 ? 4 : 2;
  const int e = (int)blockIdx.x / tiles;
  if (e >= g.groups) {
    grouped::zero_rows<ES>(g, g.n, (int)blockIdx.x - g.groups * tiles, (int)gridDim.x - g.groups * tiles);
    return;
  }
  const int64_t beg = grouped::clamped(g.offsets[e], 0, g.rows), end = grouped::clamped(g.offsets[e + 1], beg, g.rows);
  FewArgs f{};
  f.a = g.rows_in + beg * g.ld_in;
  f.lda = g.ld_in;
  f.sx = g.sx + beg;
  f.w = (const int8_t*)g.other + (int64_t)e * g.n * g.ld_other;
  f.sw = g.sw + (int64_t)e * g.n;
  f.c = g.out + beg * g.ld_out;
  f.ldc = g.ld_out / ES;
  f.m = (int)(end - beg);
  f.n = g.n;
  f.k = k;
  f.epi.kind = EPI_OFF;
  const int n0 = ((int)blockIdx.x - e * tiles) * 16 * R;
  for (int m0 = 0; m0 < f.m; m0 += 16) {
    few_rows<DT_CODES, OUT, 1, R, P, TAIL>(f, n0, m0);
    __syncthreads();  // the sums have been read
  }
}

template <int OUT>
static hipError_t grouped_few(const grouped::Args& g, int k, hipStream_t st) {
  constexpr int R = 2, P = 2;
  const int tiles = (g.n + 16 * R - 1) / (16 * R), nwin = (k + WIN - 1) / WIN, waves = nwin < 8 ? nwin : 8;
  const unsigned grid = (unsigned)(g.groups * tiles + 64);
  const size_t lds = (size_t)waves * wave_lds(1, R);
  if (k % WIN) grouped_few_kernel<OUT, R, P, true><<<grid, waves * 64, lds, st>>>(g, k, tiles);
  else grouped_few_kernel<OUT, R, P, false><<<grid, waves * 64, lds, st>>>(g, k, tiles);
  return hipGetLastError();
}

// (48 groups of 4096 x 7168, whole calls of bf16 rows, us, and the tiles; of the 165 the kernel is 154: 1 row 14, 45; 16 rows 75, 73; 64 rows 165, 193; 128 rows 183, 201; 192 rows 199, 204.)
constexpr int FEW_EACH = 4;

}  // namespace int8
}  // namespace kq

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
  hipError_t e;
  if (rows <= (int64_t)int8::FEW_EACH * groups && (int64_t)groups * ((n + 31) / 32) < 1 << 22) {  // (less than 2^32 threads)
    e = out_dtype == KQ_DT_BF16  ? int8::grouped_few<KQ_DT_BF16>(g, (int)k, st)
        : out_dtype == KQ_DT_F16 ? int8::grouped_few<KQ_DT_F16>(g, (int)k, st)
                                 : int8::grouped_few<KQ_DT_F32>(g, (int)k, st);
    return kq_check_launch(e, fn);
  }
  int64_t grid;
  bool stream_weights;
  e = grouped::plan<grouped::FORWARD>(g, st, grid, stream_weights);
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
