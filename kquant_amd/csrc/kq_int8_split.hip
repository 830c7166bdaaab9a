// The int8 linear cut along k: outputs of few tiles (a router's or a small model's
// matrices) leave most CUs idle over a long k, so slices of it go to planes of
// int32 sums, which a second kernel adds (exactly) and finishes.
#include "kq_int8_dense.h"

namespace kq {
namespace int8 {

// A step of a narrow tile is bounded by its loads, in which the 256 columns' share is
// the same for every tile (256 x 12288 in tiles of 64 rows: 42 us, 33 without fragment
// reads and MFMAs; 1024 rows in tiles of 256: 94 and 49): at K = 7168 (56 steps) a round
// of tiles of 32 / 64 / 128 / 256 rows takes 28 / 35 / 52 / 77 us, so 88 + rows.
// The cut with the least rounds in all (256 x 12288: 80 us in 48 tiles of 256 rows, 39
// in 192 of 64; 512 rows 93 and 57 of 128; 1024 rows 94, 107 and 109).  Planes cost a
// launch and their bytes.
DensePlan dense_plan(int64_t m, int64_t n, int64_t k, int64_t cus, bool split) {
  DensePlan best{};
  double least = 0.0;
  const int64_t ntiles = (n + mm16::BN - 1) / mm16::BN, steps = (k + 127) / 128;
  for (int tm : {32, 64, 96, 128, 256}) {
    const int64_t tiles = (m + tm - 1) / tm * ntiles;
    for (int slices : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (slices > 1 && (!split || tiles * slices > cus || steps < 2 * slices)) break;
      const int64_t each = (steps + slices - 1) / slices, used = (steps + each - 1) / each;
      double cost = (double)((tiles * used + cus - 1) / cus) * (88 + tm) * 0.0042 * (double)each;
      if (used > 1) cost += 4.0 + (double)m * (double)n * (4.0 * (double)used + 4.0) / 4e6;
      if (least == 0.0 || cost <= least) {
        least = cost;
        best.tm = tm;
        best.slices = (int)used;
        best.ks = (int)(each * 128);
      }
    }
  }
  best.bytes = best.slices > 1 ? 4 * (int64_t)best.slices * m * n : 0;
  return best;
}

namespace {

struct Split {
  const DenseArgs& g;
  __device__ __forceinline__ int tiles() const { return mm16::worker_tiles(g.mtiles * g.ntiles * g.slices); }
  __device__ __forceinline__ void find(int i, int& m0, int& n0, int& slice) const {
    const int at = mm16::worker_number() + i * (int)gridDim.x, all = g.mtiles * g.ntiles;
    slice = at / all;
    int mt, nt;
    mm16::tile_mn(at - slice * all, g.mtiles, g.ntiles, mt, nt);
    m0 = mt * g.tm;
    n0 = nt * mm16::BN;
  }
  __device__ __forceinline__ mm16::Tile tile(int i) const {
    int m0, n0, slice;
    find(i, m0, n0, slice);
    const int k0 = slice * g.ks;
    mm16::Tile r;
    r.kc = min(g.ks, g.k - k0) / 2;
    r.rows = r.a.rows = min(g.tm, g.m - m0);
    r.cols = r.b.rows = min(mm16::BN, g.n - n0);
    r.a.base = g.a + (int64_t)m0 * g.lda + k0;
    r.a.ld = g.lda;
    r.b.base = g.w + (int64_t)n0 * g.ldw + k0;
    r.b.ld = g.ldw;
    r.a.width = r.b.width = 0;
    return r;
  }
  template <int NB, int WN>
  __device__ __forceinline__ bool epilogue(const mm16::Tile& tl, int i, int wm, int wn, float16_t (&acc)[NB][WN],
                                           int lane) const {
    int m0, n0, slice;
    find(i, m0, n0, slice);
    int* out = g.planes + ((int64_t)slice * g.m + m0) * g.n + n0;
    mm16::each<NB, WN>(tl.rows, tl.cols, wm, wn, acc, lane,
                       [&](int row, int col, float v) { out[(int64_t)row * g.n + col] = __float_as_int(v); });
    return false;
  }
};

__global__ __launch_bounds__(mm16::THREADS, 1) void split_kernel(const DenseArgs g) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[mm16::LDS_BYTES];
  const Split p{g};
  mm16::Core<false, false, mm16::I8, mm16::SMALL_ROWS, true, false, Split> core(p, lds);
  core.run();
}

template <int OUT>
__global__ __launch_bounds__(256) void join_kernel(const DenseArgs g) {
  const int64_t all = (int64_t)g.m * g.n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / g.n, n = i - m * g.n;
    int sum = 0;
    for (int s = 0; s < g.slices; ++s) sum += g.planes[s * all + i];
    constexpr int RES = OUT == KQ_DT_F32 ? KQ_DT_F32 : KQ_DT_BF16;
    const float y = added<OUT>(g.epi, finished_any<OUT>(g.epi, sum, g.sx[m], g.sw[n], epi_bias(g.epi, n)),
                               epi_residual_bits<RES>(g.epi, m, n));
    char* p = g.out + m * g.ld + n * (OUT == KQ_DT_F32 ? 4 : 2);
    if (OUT == KQ_DT_F32) *reinterpret_cast<float*>(p) = y;
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)mm16::pack16<OUT == KQ_DT_F16>(y, 0.0f);
  }
}

}  // namespace

hipError_t dense_split(const DenseArgs& g, int out, int grid, hipStream_t st) {
  split_kernel<<<(unsigned)grid, mm16::THREADS, 0, st>>>(g);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t blocks = ((int64_t)g.m * g.n + 255) / 256;
  const unsigned join = (unsigned)(blocks < 2048 ? blocks : 2048);
  if (out == KQ_DT_BF16) join_kernel<KQ_DT_BF16><<<join, 256, 0, st>>>(g);
  else if (out == KQ_DT_F16) join_kernel<KQ_DT_F16><<<join, 256, 0, st>>>(g);
  else join_kernel<KQ_DT_F32><<<join, 256, 0, st>>>(g);
  return hipGetLastError();
}

}  // namespace int8
}  // namespace kq
