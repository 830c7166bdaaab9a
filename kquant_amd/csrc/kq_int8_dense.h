// The int8 linear on the 256-column tiles of kq_mm16.h, one kernel for each
// result type and activation class (a source file a type).
#pragma once

#include "kq_int8.h"
#include "kq_internal.h"

namespace kq {
namespace int8 {

struct DenseArgs {
  const char* a;
  const char* w;
  const float* sx;
  const float* sw;
  char* out;
  uint32_t lda, ldw;  // bytes
  int64_t ld;         // bytes
  int m, n, k;
  int tm;             // rows of a tile
  int mtiles, ntiles;
  int slices, ks;     // of k, and the bytes of one (a multiple of 128)
  int* planes;        // the slices' sums [slices][m][n]
  Epilogue epi;
  int pieces;
};

hipError_t dense_bf16(const DenseArgs& g, int grid, hipStream_t st);
hipError_t dense_f16(const DenseArgs& g, int grid, hipStream_t st);
hipError_t dense_f32(const DenseArgs& g, int grid, hipStream_t st);

// How an m x n product over k is cut: the tiles' height, and slices of k where the
// tiles alone leave most CUs without one; cus workgroups run.
struct DensePlan {
  int tm, slices, ks;
  int64_t bytes;  // of the planes
};
DensePlan dense_plan(int64_t m, int64_t n, int64_t k, int64_t cus, bool split);
hipError_t dense_split(const DenseArgs& g, int out, int grid, hipStream_t st);

template <int OUT, int EPI>
struct Dense {
  const DenseArgs& g;
  __device__ __forceinline__ int tiles() const { return mm16::worker_tiles(g.mtiles * g.ntiles); }
  __device__ __forceinline__ void find(int i, int& m0, int& n0) const {
    int mt, nt;
    mm16::tile_mn(mm16::worker_number() + i * (int)gridDim.x, g.mtiles, g.ntiles, mt, nt);
    m0 = mt * g.tm;
    n0 = nt * mm16::BN;
  }
  __device__ __forceinline__ mm16::Tile tile(int i) const {
    int m0, n0;
    find(i, m0, n0);
    mm16::Tile r;
    r.kc = g.k / 2;
    r.rows = r.a.rows = min(g.tm, g.m - m0);
    r.cols = r.b.rows = min(mm16::BN, g.n - n0);
    r.a.base = g.a + (int64_t)m0 * g.lda;
    r.a.ld = g.lda;
    r.b.base = g.w + (int64_t)n0 * g.ldw;
    r.b.ld = g.ldw;
    r.a.width = r.b.width = 0;
    return r;
  }
  template <int NB, int WN>
  __device__ __forceinline__ bool epilogue(const mm16::Tile& tl, int i, int wm, int wn, float16_t (&acc)[NB][WN],
                                           int lane) const {
    constexpr int ES = OUT == KQ_DT_F32 ? 4 : 2;
    int m0, n0;
    find(i, m0, n0);
    Finish f;
    f.sx = g.sx + m0;
    f.sw = g.sw + n0;
    f.out = g.out + (int64_t)m0 * g.ld + (int64_t)n0 * ES;
    f.ld = g.ld;
    f.epi = g.epi;
    if (f.epi.bias) f.epi.bias = static_cast<const char*>(f.epi.bias) + (int64_t)n0 * (f.epi.bias_f32 ? 4 : 2);
    if (f.epi.residual)
      f.epi.residual = static_cast<const char*>(f.epi.residual) + ((int64_t)m0 * f.epi.ldr + n0) * ES;
    f.pieces = g.pieces;
    finish<NB, WN, OUT, EPI>(f, tl.rows, tl.cols, wm, wn, acc, lane);
    return tl.rows >= mm16::BM && tl.cols >= mm16::BN;
  }
};

template <int OUT, int EPI>
__global__ __launch_bounds__(mm16::THREADS, 1) void dense_kernel(const DenseArgs g) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[mm16::LDS_BYTES];
  const Dense<OUT, EPI> p{g};
  mm16::Core<false, false, mm16::I8, mm16::SMALL_ROWS, true, false, Dense<OUT, EPI>> core(p, lds);
  core.run();
}

template <int OUT>
static hipError_t dense(const DenseArgs& g, int grid, hipStream_t st) {
  auto kern = g.epi.kind == EPI_OFF       ? dense_kernel<OUT, EPI_OFF>
              : g.epi.kind == EPI_CLAMP   ? dense_kernel<OUT, EPI_CLAMP>
              : g.epi.kind == EPI_SIGMOID ? dense_kernel<OUT, EPI_SIGMOID>
                                          : dense_kernel<OUT, EPI_ERF>;
  kern<<<(unsigned)grid, mm16::THREADS, 0, st>>>(g);
  return hipGetLastError();
}

}  // namespace int8
}  // namespace kq
