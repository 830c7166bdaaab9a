// Softmax cross entropy of a vocabulary head without keeping the logits.
//
//   z[t][v] = h_t . w_v          loss_t = lse_t - z[t][y_t],  lse_t = log sum_v exp z[t][v]
//   d[t][v] = g_t (exp(z[t][v] - lse_t) - [v = y_t])
//   dh_t = sum_v d[t][v] w_v     dw_v = sum_t d[t][v] h_t
//
// with g_t = alpha u_t: alpha (one upstream gradient, over the token count for a
// mean; else the largest magnitude of the tokens' gradients) multiplies the fp32
// sums, so that the -1 of a target enters the products exactly and not as a
// rounded 1 / count, whose error all tokens would share.
//
// What bounds it: the matrix products (2 T V K flop forward, 6 T V K backward,
// a third of which recomputes z); at few tokens, the head's bytes.  The
// logits never reach memory in the forward pass: a tile's epilogue reduces its
// 64 or 128 vocabulary rows per wave to a running maximum and a sum of exponentials
// per token, and picks the target's logit.  The product is taken as W H^T, so
// a lane holds one token's logits and reduces them in registers.  The
// backward pass walks the vocabulary in pieces whose gradient d^T (bf16) fits
// a bounded workspace; a piece recomputes its logits, and its d^T then is an
// operand of both gradients' products, for dh across its rows and for dw along
// them.
//
// Tokens whose target is ignore_index are left out of every product: the
// counted rows are first gathered (their number stays on the device), so their
// values, NaN and Inf among them, reach nothing, and cost nothing.
//
// Precision: products of bf16 values are exact and sum in fp32, as do the
// exponentials, their sums and dh's planes; d is rounded to bf16 to be an
// operand (half a step, 2^-8 relative, of each term of sums that are themselves
// rounded to bf16).  Heads in MXFP8 / MXFP4 are expanded piece by piece to bf16,
// which holds their values exactly (but for those below bf16's subnormals, 2^-133).
#include "kq_internal.h"
#include "kq_mm16.h"

namespace kq {
namespace loss {

using mm16::Tile;
using mm16::u32x4_t;

enum { NONE = 0, MEAN = 1, SUM = 2 };
constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;

__shared__ __attribute__((aligned(16))) unsigned char lds[mm16::LDS_BYTES];

// dh's contraction over the vocabulary runs in slices until its tiles fill the workers; a slice's plane is written
// and read once (5 TB/s), a 64-row step of a tile takes 1.3 us.
constexpr int MAX_SLICES = 16;
__host__ __device__ inline bool slices_allowed(int64_t s, int64_t steps) { return s == 1 || s * 4 <= steps; }
__host__ __device__ inline float slices_us(int64_t s, int64_t counted, int64_t k, int64_t steps, int workers, bool planes) {
  const int64_t tiles = ((counted + 255) / 256) * ((k + 255) / 256);
  return (float)((tiles * s + workers - 1) / workers) * (float)((steps + s - 1) / s) * 1.3f +
         (s > 1 || planes ? 5.0f + (float)(s * counted * k * 8) / 5e6f : 0.0f);
}

// What the device chooses the slices from: the planes there is room for (0: dh is stored at once), a piece's
// steps of 64 vocabulary rows, K, and the workers.
struct Slicing {
  int64_t room;  // rows of planes
  int steps, k, workers;
};

// The gradient of a mean or a sum (alpha null: there is none yet, or it has a kernel of its own).
struct Upstream {
  const float* grad;
  int mean;
  float* alpha;
};

// Counted tokens in order: rows[i] the i-th one's row, place[t] its i or -1.  count[0]: their number, count[1]:
// dh's slices for it (2048 tokens of which 1434 count, V = 50257, K = 2048: dh 292 us with the slices of all
// tokens, 245 so).
__global__ __launch_bounds__(1024) void compact_kernel(const int64_t* __restrict__ target, int64_t ignore_index,
                                                       int tokens, int* __restrict__ rows, int* __restrict__ place,
                                                       int* __restrict__ count, Slicing dh, Upstream up) {
  __shared__ int wave_sum[16];
  constexpr int PER = 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int base = 0;
  for (int t0 = 0; t0 < tokens; t0 += 1024 * PER) {
    const int first = t0 + tid * PER;
    int mine = 0, keep = 0;
    for (int q = 0; q < PER; ++q)
      if (first + q < tokens && target[first + q] != ignore_index) {
        keep |= 1 << q;
        ++mine;
      }
    int upto = mine;
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    int before = base, all = 0;
    for (int w = 0; w < 16; ++w) {
      before += w < wave ? wave_sum[w] : 0;
      all += wave_sum[w];
    }
    int at = before + upto - mine;
    for (int q = 0; q < PER; ++q)
      if (first + q < tokens) {
        const bool k = keep >> q & 1;
        place[first + q] = k ? at : -1;
        if (k) rows[at++] = first + q;
      }
    base += all;
    __syncthreads();
  }
  if (tid < 64) {  // lane s - 1: s slices
    const int s = tid + 1;
    float us = __builtin_inff();
    if (dh.workers > 0 && s <= MAX_SLICES && (int64_t)s * base <= dh.room && slices_allowed(s, dh.steps))
      us = slices_us(s, base, dh.k, dh.steps, dh.workers, true);
    float least = us;
    for (int d = 1; d < 64; d <<= 1) least = fminf(least, __shfl_xor(least, d));
    const uint64_t best = __ballot(us == least && us < __builtin_inff());
    if (tid == 0) {
      count[0] = base;
      count[1] = best ? __builtin_ctzll(best) + 1 : 1;
      // none counted: gradients of zero whatever the upstream one is
      if (up.alpha) *up.alpha = base == 0 ? 0.0f : up.mean ? *up.grad / (float)base : *up.grad;
    }
  }
}

// alpha of one upstream gradient per token (see above); 1 where they are all zero.
__global__ __launch_bounds__(1024) void alpha_kernel(const float* __restrict__ grad, int tokens,
                                                     const int* __restrict__ place, float* __restrict__ alpha) {
  __shared__ float wave_max[16];
  float m = 0.0f;  // the largest finite one: another leaves u infinite or NaN, as it should
  for (int t = threadIdx.x; t < tokens; t += 1024) {
    const float v = fabsf(grad[t]);
    if (place[t] >= 0 && v < __builtin_inff()) m = fmaxf(m, v);
  }
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) m = fmaxf(m, wave_max[w]);
    *alpha = m > 0.0f ? m : 1.0f;
  }
}

__device__ __forceinline__ int tile_number(int i) { return mm16::worker_number() + i * (int)gridDim.x; }

struct Gather {
  const char* h;
  int64_t ldh;  // bytes
  const int64_t* target;
  const int* place;
  const int* count;
  int tokens, k;
  int64_t vocab;
  char* hc;      // counted rows, then zero rows up to a multiple of 8
  int* target_c;  // -1 where the target is outside the vocabulary
  // backward
  const float* lse;
  const float* grad;
  int reduction;
  const float* alpha;
  float* lse_c;
  float* u_c;  // upstream gradients over alpha
  char* dh;
  int64_t lddh;  // bytes
};

// One workgroup per token row: a counted one goes to its place, an ignored
// one's gradient is zero.
__global__ __launch_bounds__(256) void gather_kernel(Gather g) {
  const int t = blockIdx.x, count = *g.count;
  if (t >= g.tokens) {  // the zero rows behind the counted ones
    const int row = count + t - g.tokens;
    if (row < (count + 7) / 8 * 8)
      for (int c = (int)threadIdx.x * 8; c < g.k; c += 2048)
        *reinterpret_cast<u32x4_t*>(g.hc + ((int64_t)row * g.k + c) * 2) = u32x4_t{0u, 0u, 0u, 0u};
    return;
  }
  const int at = g.place[t];
  if (at >= 0) {
    for (int c = (int)threadIdx.x * 8; c < g.k; c += 2048)
      *reinterpret_cast<u32x4_t*>(g.hc + ((int64_t)at * g.k + c) * 2) =
          *reinterpret_cast<const u32x4_t*>(g.h + t * g.ldh + 2 * (int64_t)c);
    if (threadIdx.x == 0) {
      const int64_t y = g.target[t];
      const bool ok = y >= 0 && y < g.vocab;
      g.target_c[at] = ok ? (int)y : -1;
      if (g.lse_c) {
        g.lse_c[at] = g.lse[t];
        g.u_c[at] = ok ? (g.reduction == NONE ? g.grad[t] / *g.alpha : 1.0f) : __builtin_nanf("");
      }
    }
  } else if (g.dh) {
    for (int c = (int)threadIdx.x * 8; c < g.k; c += 2048)
      *reinterpret_cast<u32x4_t*>(g.dh + t * g.lddh + 2 * (int64_t)c) = u32x4_t{0u, 0u, 0u, 0u};
  }
}

// A running (maximum, sum of exp(z - maximum)) joined with another.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), ref = top == -__builtin_inff() ? 0.0f : top;
  s = s * __builtin_amdgcn_exp2f((m - ref) * LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - ref) * LOG2E);
  m = top;
}

// The logits of a vocabulary piece: W rows [first, first + rows) x counted
// tokens.  Forward: partial maxima and sums of 64 vocabulary rows each,
// part[4 tile + row / 64][token], and the targets' logits.  GRAD: d^T, row stride ldg elements, zero in the
// token columns from count up to a multiple of 8.
struct LogitArgs {
  const char* w;  // bf16 rows of the piece
  const char* hc;
  const int* count;
  const int* target_c;
  int first, rows, k, tokens;
  float2_t* part;
  int part0;  // tiles of the pieces before
  float* z_target;
  const float* lse_c;
  const float* u_c;
  char* dt;
  int ldg;
};

template <bool GRAD>
struct LogitProblem {
  LogitArgs g;
  int count, mtiles, ntiles;

  __device__ __forceinline__ int tiles() const { return mm16::worker_tiles(mtiles * ntiles); }
  __device__ __forceinline__ Tile tile(int x) const {
    const int t = tile_number(x);
    int mt, nt;
    mm16::tile_mn(t, mtiles, ntiles, mt, nt);
    const int m0 = mt * mm16::BM, n0 = nt * mm16::BN;
    Tile r;
    r.cols = min(mm16::BN, count - n0);
    r.kc = g.k;
    r.rows = min(mm16::BM, g.rows - m0);
    r.a = {g.w + (int64_t)m0 * g.k * 2, (uint32_t)g.k * 2u, r.rows, 0u};
    r.b = {g.hc + (int64_t)n0 * g.k * 2, (uint32_t)g.k * 2u, min(mm16::BN, count - n0), 0u};
    return r;
  }
  template <int NB, int WN>
  __device__ __forceinline__ bool epilogue(const Tile& tl, int x, int wm, int wn, float16_t (&acc)[NB][WN],
                                           int lane) const {
    const int t = tile_number(x);
    int mt, nt;
    mm16::tile_mn(t, mtiles, ntiles, mt, nt);
    const int v0 = g.first + mt * mm16::BM, n0 = nt * mm16::BN;
    if (GRAD) {
      int tgt[WN];
      float lse[WN], up[WN];
#pragma unroll
      for (int j = 0; j < WN; ++j) {
        const int c = n0 + wn + 32 * j + (lane & 31);
        const bool live = c < count;
        tgt[j] = live ? g.target_c[c] - v0 : -1;
        lse[j] = live ? g.lse_c[c] : 0.0f;
        up[j] = live ? g.u_c[c] : 0.0f;
      }
      char* out = g.dt + ((int64_t)mt * mm16::BM * g.ldg + n0) * 2;
      const int row = wm + 4 * (lane >> 5);
      mm16::store16<NB, WN, false>([&](int r) { return out + (uint32_t)r * ((uint32_t)g.ldg * 2u); }, tl.rows,
                                   (count + 7) / 8 * 8 - n0, wm, wn, acc, lane, [&](int i, int j, int r, float z) {
        const int at = row + 32 * i + 8 * (r >> 2) + (r & 3);
        const float p = __builtin_amdgcn_exp2f((z - lse[j]) * LOG2E) - (at == tgt[j] ? 1.0f : 0.0f);
        return n0 + wn + 32 * j + (lane & 31) < count ? up[j] * p : 0.0f;
      });
      return tl.rows >= mm16::BM && (count + 7) / 8 * 8 - n0 >= mm16::BN;
    }
    const int row = wm + 4 * (lane >> 5);  // this lane's rows: row + 32 i + 8 (r / 4) + r % 4
    float m[WN], s[WN], hit[WN];
    int at[WN];  // the target's position from this lane's first row
    bool some = false;
#pragma unroll
    for (int j = 0; j < WN; ++j) {
      m[j] = -__builtin_inff();
      s[j] = hit[j] = 0.0f;
      const int c = n0 + wn + 32 * j + (lane & 31);
      at[j] = c < count ? g.target_c[c] - v0 - row : -1;
      some |= at[j] >= 0 && at[j] < 32 * NB;
    }
    // one pass, 16 logits at a time: the sums so far are rescaled to a new maximum
    const bool any = __any(some);
    const int left = tl.rows - row;  // of this lane's rows, where the vocabulary ends in them
    const bool cut = tl.rows < wm + 32 * NB;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      mm16::in_place(acc, i);
#pragma unroll
      for (int j = 0; j < WN; ++j) {
        float z[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = acc[i][j][r];
        if (any) {
#pragma unroll
          for (int r = 0; r < 16; ++r) hit[j] = at[j] == 32 * i + 8 * (r >> 2) + (r & 3) ? z[r] : hit[j];
        }
        if (cut) {
#pragma unroll
          for (int r = 0; r < 16; ++r) z[r] = 32 * i + 8 * (r >> 2) + (r & 3) < left ? z[r] : -__builtin_inff();
        }
        float top = m[j];
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, z[r]);
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        float sum = s[j] * __builtin_amdgcn_exp2f((m[j] - ref) * LOG2E);
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f((z[r] - ref) * LOG2E);
        m[j] = top;
        s[j] = sum;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int j = 0; j < WN; ++j) {
      join(m[j], s[j], __shfl_xor(m[j], 32), __shfl_xor(s[j], 32));
      const int c = n0 + wn + 32 * j + (lane & 31);
      if (c < count) {
        if (lane < 32) {
          float2_t* part = g.part + (int64_t)(4 * (g.part0 + mt) + (wm >> 6)) * g.tokens + c;
          float2_t v;
          v[0] = m[j];
          v[1] = s[j];
          part[0] = v;
          if (NB == 4) {  // 128 rows at once: nothing is left for the second 64
            v[0] = -__builtin_inff();
            v[1] = 0.0f;
            part[g.tokens] = v;
          }
        }
        if (at[j] >= 0 && at[j] < 32 * NB && !(at[j] & 4)) g.z_target[c] = hit[j];
      }
    }
    return false;
  }
};

template <bool GRAD>
__global__ __launch_bounds__(mm16::THREADS, 1) void logit_kernel(LogitArgs g) {
  LogitProblem<GRAD> p{g, __builtin_amdgcn_readfirstlane(*g.count), 0, 0};
  p.mtiles = (g.rows + mm16::BM - 1) / mm16::BM;
  p.ntiles = (p.count + mm16::BN - 1) / mm16::BN;
  mm16::Core<false, false, false, mm16::SMALL_COLS, false, false, LogitProblem<GRAD>> core(p, lds);
  core.run();
}

// dh: d (its transpose, read across) x the piece's rows (read across), the
// vocabulary cut into slices.  One slice of one piece stores dh itself, at the
// tokens' own rows; else slices add up in fp32 planes [slice][counted token][k].
struct DhArgs {
  const char* dt;
  int ldg;
  const char* w;
  const int* count;
  const int* rows_of;
  int rows, k;
  const float* alpha;
  char* dh;  // or null
  int64_t lddh;  // bytes
  float* planes;
  int add;  // to the planes of the pieces before
};

struct DhProblem {
  DhArgs g;
  int count, slices, mtiles, ntiles;

  __device__ __forceinline__ int tiles() const { return mm16::worker_tiles(mtiles * ntiles * slices); }
  __device__ __forceinline__ Tile tile(int x) const {
    const int t = tile_number(x);
    int mt, nt;
    const int per = mtiles * ntiles, sl = t / per;
    mm16::tile_mn(t - sl * per, mtiles, ntiles, mt, nt);
    const int m0 = mt * mm16::BM, n0 = nt * mm16::BN, steps = (g.rows + mm16::BK - 1) / mm16::BK;
    const int v0 = sl * steps / slices * mm16::BK;  // slices <= 16, steps <= 2^18
    const int v1 = min((sl + 1) * steps / slices * mm16::BK, g.rows);
    Tile r;
    r.cols = mm16::BN;
    r.kc = v1 - v0;
    r.rows = min(mm16::BM, count - m0);
    r.a = {g.dt + ((int64_t)v0 * g.ldg + m0) * 2, (uint32_t)g.ldg * 2u, 0, (uint32_t)((count + 7) / 8 * 8 - m0) * 2u};
    r.b = {g.w + ((int64_t)v0 * g.k + n0) * 2, (uint32_t)g.k * 2u, 0, (uint32_t)(g.k - n0) * 2u};
    return r;
  }
  template <int NB, int WN>
  __device__ __forceinline__ bool epilogue(const Tile& tl, int x, int wm, int wn, float16_t (&acc)[NB][WN],
                                           int lane) const {
    const int t = tile_number(x);
    int mt, nt;
    const int per = mtiles * ntiles, sl = t / per;
    mm16::tile_mn(t - sl * per, mtiles, ntiles, mt, nt);
    const int m0 = mt * mm16::BM, n0 = nt * mm16::BN;
    if (g.dh) {
      const int* map = g.rows_of + m0;
      char* out = g.dh + 2 * (int64_t)n0;
      const float alpha = *g.alpha;
      mm16::store16<NB, WN, false>([&](int r) { return out + map[r] * g.lddh; }, tl.rows, g.k - n0, wm, wn, acc, lane,
                                   [&](int, int, int, float v) { return alpha * v; });
    } else {
      float* out = g.planes + ((int64_t)sl * count + m0) * g.k + n0;
      const uint32_t ld = (uint32_t)g.k;
      if (g.add)
        mm16::each(tl.rows, g.k - n0, wm, wn, acc, lane,
                   [&](int r, int c, float v) { out[(uint32_t)r * ld + (uint32_t)c] += v; });
      else
        mm16::each(tl.rows, g.k - n0, wm, wn, acc, lane,
                   [&](int r, int c, float v) { out[(uint32_t)r * ld + (uint32_t)c] = v; });
    }
    return tl.rows >= mm16::BM && g.k - n0 >= mm16::BN;
  }
};

__global__ __launch_bounds__(mm16::THREADS, 1) void dh_kernel(DhArgs g) {
  DhProblem p{g, __builtin_amdgcn_readfirstlane(g.count[0]), __builtin_amdgcn_readfirstlane(g.count[1]), 0, 0};
  p.mtiles = (p.count + mm16::BM - 1) / mm16::BM;
  p.ntiles = (g.k + mm16::BN - 1) / mm16::BN;
  mm16::Core<true, true, false, mm16::SMALL_ROWS, true, false, DhProblem> core(p, lds);
  core.run();
}

// dh at the tokens' own rows = the sum of the planes, in slice order.
__global__ __launch_bounds__(256) void dh_sum_kernel(const float* __restrict__ planes, const int* __restrict__ count, int k,
                                                     const int* __restrict__ place,
                                                     const float* __restrict__ alpha_at, char* __restrict__ dh,
                                                     int64_t lddh) {
  const int t = blockIdx.x, at = place[t];
  if (at < 0) return;
  const float alpha = *alpha_at;
  const int counted = count[0], slices = count[1];
  for (int c = (int)threadIdx.x * 4; c < k; c += 1024) {
    const float* p = planes + (int64_t)at * k + c;
    float4_t v = *reinterpret_cast<const float4_t*>(p);
    for (int s = 1; s < slices; ++s) v += *reinterpret_cast<const float4_t*>(p + (int64_t)s * counted * k);
    uint32_t* o = reinterpret_cast<uint32_t*>(dh + t * lddh + 2 * (int64_t)c);
    o[0] = f32x2_to_bf16x2_bits(alpha * v[0], alpha * v[1]);
    o[1] = f32x2_to_bf16x2_bits(alpha * v[2], alpha * v[3]);
  }
}

// dw rows of the piece: d^T (along its rows) x the counted tokens (across).
struct DwArgs {
  const char* dt;
  int ldg;
  const char* hc;
  const int* count;
  const float* alpha;
  int rows, k;
  char* dw;
};

struct DwProblem {
  DwArgs g;
  int count, mtiles, ntiles;  // count: rounded up to 8, the rows behind it are zero

  __device__ __forceinline__ int tiles() const { return mm16::worker_tiles(mtiles * ntiles); }
  __device__ __forceinline__ Tile tile(int x) const {
    const int t = tile_number(x);
    int mt, nt;
    mm16::tile_mn(t, mtiles, ntiles, mt, nt);
    const int m0 = mt * mm16::BM, n0 = nt * mm16::BN;
    Tile r;
    r.cols = mm16::BN;
    r.kc = count;
    r.rows = min(mm16::BM, g.rows - m0);
    r.a = {g.dt + (int64_t)m0 * g.ldg * 2, (uint32_t)g.ldg * 2u, r.rows, 0u};
    r.b = {g.hc + (int64_t)n0 * 2, (uint32_t)g.k * 2u, 0, (uint32_t)(g.k - n0) * 2u};
    return r;
  }
  template <int NB, int WN>
  __device__ __forceinline__ bool epilogue(const Tile& tl, int x, int wm, int wn, float16_t (&acc)[NB][WN],
                                           int lane) const {
    const int t = tile_number(x);
    int mt, nt;
    mm16::tile_mn(t, mtiles, ntiles, mt, nt);
    const int n0 = nt * mm16::BN;
    char* out = g.dw + ((int64_t)mt * mm16::BM * g.k + n0) * 2;
    const float alpha = *g.alpha;
    mm16::store16<NB, WN, false>([&](int r) { return out + (uint32_t)r * ((uint32_t)g.k * 2u); }, tl.rows, g.k - n0, wm, wn,
                                 acc, lane,
                                 [&](int, int, int, float v) { return alpha * v; });
    return tl.rows >= mm16::BM && g.k - n0 >= mm16::BN;
  }
};

__global__ __launch_bounds__(mm16::THREADS, 1) void dw_kernel(DwArgs g) {
  DwProblem p{g, (__builtin_amdgcn_readfirstlane(*g.count) + 7) / 8 * 8, 0, 0};
  p.mtiles = (g.rows + mm16::BM - 1) / mm16::BM;
  p.ntiles = (g.k + mm16::BN - 1) / mm16::BN;
  mm16::Core<false, true, false, mm16::WHOLE, false, false, DwProblem> core(p, lds);
  core.run();
}

// lse and loss of every token from its partial maxima and sums (nparts rows of
// `tokens`), 16 tokens a workgroup; 0 for the ignored ones, NaN where the
// target is outside the vocabulary.  Few workgroups of long columns: what bounds
// it is latency, so eight loads are out at a time and the columns meet in a tree
// (777 tokens, 2020 parts: 24 us one after the other, 14 so).
__global__ __launch_bounds__(1024) void combine_kernel(const float2_t* __restrict__ part, int nparts, int tokens,
                                                       const int* __restrict__ place, const int* __restrict__ target_c,
                                                       const float* __restrict__ z_target, float* __restrict__ losses,
                                                       float* __restrict__ lse) {
  __shared__ float ms[64][17], ss[64][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, t = blockIdx.x * 16 + x;
  const int at = t < tokens ? place[t] : -1;
  float m = -__builtin_inff(), s = 0.0f;
  if (at >= 0)
    for (int p = y; p < nparts; p += 64 * 8) {
      float2_t v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {  // past the end: the last one again, not joined
        const int row = p + 64 * q < nparts ? p + 64 * q : nparts - 1;
        v[q] = part[(int64_t)row * tokens + at];
      }
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (p + 64 * q < nparts) join(m, s, v[q][0], v[q][1]);
    }
  ms[y][x] = m;
  ss[y][x] = s;
  for (int w = 32; w > 0; w >>= 1) {
    __syncthreads();
    if (y < w) {
      join(m, s, ms[y + w][x], ss[y + w][x]);
      ms[y][x] = m;
      ss[y][x] = s;
    }
  }
  if (y != 0 || t >= tokens) return;
  const float l = m + LN2 * __builtin_amdgcn_logf(s);
  lse[t] = at < 0 ? 0.0f : l;
  losses[t] = at < 0 ? 0.0f : target_c[at] < 0 ? __builtin_nanf("") : l - z_target[at];
}

// The few-token form: the maxima and sums of 16 columns each, part[token][nparts],
// one workgroup a token.
__global__ __launch_bounds__(1024) void combine_few_kernel(const float2_t* __restrict__ part, int64_t nparts,
                                                           const int64_t* __restrict__ target, int64_t ignore_index,
                                                           int64_t vocab, const float* __restrict__ z_target,
                                                           float* __restrict__ losses, float* __restrict__ lse) {
  __shared__ float ms[16], ss[16];
  const int t = blockIdx.x;
  const int64_t y = target[t];
  if (y == ignore_index) {
    if (threadIdx.x == 0) losses[t] = lse[t] = 0.0f;
    return;
  }
  float m = -__builtin_inff(), s = 0.0f;
  for (int64_t p = threadIdx.x; p < nparts; p += 1024) {
    const float2_t v = part[t * nparts + p];
    join(m, s, v[0], v[1]);
  }
  for (int d = 1; d < 64; d <<= 1) join(m, s, __shfl_xor(m, d), __shfl_xor(s, d));
  if ((threadIdx.x & 63) == 0) {
    ms[threadIdx.x >> 6] = m;
    ss[threadIdx.x >> 6] = s;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) join(m, s, ms[w], ss[w]);
  const float l = m + LN2 * __builtin_amdgcn_logf(s);
  lse[t] = l;
  losses[t] = y >= 0 && y < vocab ? l - z_target[t] : __builtin_nanf("");
}

// sums[0] = the losses' sum, sums[1] = their mean over the counted tokens (NaN
// if there are none), added in 64 bits.
__global__ __launch_bounds__(1024) void sum_kernel(const float* __restrict__ losses, int tokens,
                                                   const int64_t* __restrict__ target, int64_t ignore_index,
                                                   float* __restrict__ sums) {
  __shared__ double red[1024];
  __shared__ int counts[1024];
  double s = 0.0;
  int n = 0;
  for (int t = threadIdx.x; t < tokens; t += 1024) {
    s += (double)losses[t];
    n += target[t] != ignore_index ? 1 : 0;
  }
  red[threadIdx.x] = s;
  counts[threadIdx.x] = n;
  for (int w = 512; w > 0; w >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < w) {
      red[threadIdx.x] += red[threadIdx.x + w];
      counts[threadIdx.x] += counts[threadIdx.x + w];
    }
  }
  if (threadIdx.x == 0) {
    sums[0] = (float)red[0];
    sums[1] = (float)(red[0] / (double)counts[0]);
  }
}

// ------------------------------------------------------------------- host --

constexpr int64_t PIECE_BYTES = 1ll << 30;  // of a piece's d^T, and of its expanded rows

struct Plan {
  bool few;                    // the one-pass kernel of kq_skinny.hip
  int64_t piece, pieces;       // vocabulary rows
  int slices;                  // of dh's contraction
  int64_t ldg;
  int64_t o_rows, o_place, o_count, o_target, o_lse, o_u, o_alpha, o_z, o_part, o_hc, o_w, o_dt, o_planes, bytes;
};

static int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

static Plan plan(int w_fmt, int64_t tokens, int64_t vocab, int64_t k, bool backward, int cus) {
  Plan p{};
  const bool mx = w_fmt != KQ_FMT_BF16;
  // A block-scaled head at few tokens is read as it is, once (5 tokens, V = 129280, K = 7168 E4M3: 172 us; expanded
  // to bf16 and multiplied in tiles 760 us).  A bf16 head's tiles stream it whatever the count (1.85 GB,
  // 1 / 16 / 64 tokens: 323 / 332 / 334 us, 5.5 to 5.7 TB/s).
  p.few = mx && !backward && tokens >= 1 && tokens <= 64;
  if (p.few) {
    p.o_z = 0;
    p.o_part = up(tokens * 4, 256);
    p.bytes = p.o_part + up(tokens * ((vocab + 15) / 16) * 8, 256);
    return p;
  }
  p.ldg = up(tokens > 0 ? tokens : 1, 8);
  int64_t most = vocab;
  if (mx) most = PIECE_BYTES / (2 * k);
  if (backward && PIECE_BYTES / (2 * p.ldg) < most) most = PIECE_BYTES / (2 * p.ldg);
  if (most < 256) most = 256;  // (2^20 tokens leave 512, K = 2^16 8192)
  most = most / 256 * 256;
  p.pieces = most >= vocab ? 1 : (vocab + most - 1) / most;
  p.piece = p.pieces == 1 ? vocab : up((vocab + p.pieces - 1) / p.pieces, 256);
  p.pieces = (vocab + p.piece - 1) / p.piece;
  // dh: the planes that all tokens would take; fewer counted ones may be cut finer in the same room
  p.slices = 1;
  if (backward) {
    const int64_t steps = (p.piece + 63) / 64;
    float best = 1e30f;
    for (int64_t s = 1; s <= MAX_SLICES && slices_allowed(s, steps); ++s) {
      const float t = slices_us(s, tokens, k, steps, cus, p.pieces > 1);
      if (t < best) {
        best = t;
        p.slices = (int)s;
      }
    }
  }
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  p.o_rows = take(tokens * 4);
  p.o_place = take(tokens * 4);
  p.o_count = take(8);
  p.o_target = take(tokens * 4);
  p.o_hc = take(up(tokens, 8) * k * 2);
  if (mx) p.o_w = take(p.piece * k * 2);
  if (backward) {
    p.o_lse = take(tokens * 4);
    p.o_u = take(tokens * 4);
    p.o_alpha = take(4);
    p.o_dt = take(p.piece * p.ldg * 2);
    if (p.slices > 1 || p.pieces > 1) p.o_planes = take(p.slices * tokens * k * 4);
  } else {
    p.o_z = take(tokens * 4);
    p.o_part = take(4 * p.pieces * ((p.piece + 255) / 256) * tokens * 8);
  }
  p.bytes = at;
  return p;
}

static hipError_t stream_cus(hipStream_t st, int* cus) {
  int dev = 0;
  hipError_t e = st ? hipStreamGetDevice(st, &dev) : hipGetDevice(&dev);
  if (e == hipSuccess) e = hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev);
  return e;
}

static int check(const char* fn, int w_fmt, const void* h, int64_t ldh, int64_t tokens, const void* w,
                 const uint8_t* w_scale, int64_t vocab, int64_t k, const int64_t* target, int reduction) {
  const bool mx = w_fmt == KQ_FMT_MXFP8_E4M3 || w_fmt == KQ_FMT_MXFP4_E2M1;
  if (!mx && w_fmt != KQ_FMT_BF16) return kq_fail(KQ_ERR_INVALID, "%s: unknown head format %d", fn, w_fmt);
  if (reduction < NONE || reduction > SUM) return kq_fail(KQ_ERR_INVALID, "%s: unknown reduction %d", fn, reduction);
  if (tokens < 0 || vocab <= 0 || k <= 0 || k % (mx ? 64 : 8) || ldh < k || ldh % 8)
    return kq_fail(KQ_ERR_INVALID,
                   "%s: need k %% %d == 0, ldh >= k, ldh %% 8 == 0, vocab >= 1 (tokens=%lld vocab=%lld k=%lld ldh=%lld)", fn,
                   mx ? 64 : 8, (long long)tokens, (long long)vocab, (long long)k, (long long)ldh);
  if (tokens > 1 << 20 || vocab > 1 << 24 || k > 1 << 16)
    return kq_fail(KQ_ERR_LIMIT, "%s: at most 2^20 tokens, 2^24 vocabulary rows and k = 2^16", fn);
  if (mx && !w_scale) return kq_fail(KQ_ERR_INVALID, "%s: a block-scaled head needs its scales", fn);
  if (kq_misaligned(h, 16) || kq_misaligned(w, 16) || kq_misaligned(target, 8) || kq_misaligned(w_scale, 4))
    return kq_fail(KQ_ERR_INVALID, "%s: h and w must be 16-byte aligned, target 8, scales 4", fn);
  return KQ_OK;
}

// The piece's rows in bf16: the head's own, or expanded into the workspace.
static int piece_rows(int w_fmt, const void* w, const uint8_t* w_scale, int64_t first, int64_t rows, int64_t k,
                      char* expanded, const char** out, void* stream) {
  if (w_fmt == KQ_FMT_BF16) {
    *out = (const char*)w + first * k * 2;
    return KQ_OK;
  }
  *out = expanded;
  const int64_t row = w_fmt == KQ_FMT_MXFP8_E4M3 ? k : k / 2;
  return kq_mx_dequant(w_fmt, (const char*)w + first * row, w_scale + first * (k / 32), rows, k, KQ_DT_BF16, expanded, 0,
                       stream);
}

static unsigned persistent_grid(int cus) { return cus >= 8 ? (unsigned)(cus / 8 * 8) : 8u; }

}  // namespace loss
}  // namespace kq

using namespace kq;

extern "C" int64_t kq_linear_cross_entropy_workspace_size(int w_fmt, int64_t tokens, int64_t vocab, int64_t k,
                                                          int backward) {
  if (tokens < 0 || vocab <= 0 || k <= 0 || tokens > 1 << 20 || vocab > 1 << 24 || k > 1 << 16) return -1;
  int cus = 0;
  if (loss::stream_cus(nullptr, &cus) != hipSuccess || cus <= 0) cus = 256;
  return loss::plan(w_fmt, tokens, vocab, k, backward != 0, cus).bytes;
}

extern "C" int kq_linear_cross_entropy(int w_fmt, const void* h, int64_t ldh, int64_t tokens, const void* w,
                                       const uint8_t* w_scale, int64_t vocab, int64_t k, const int64_t* target,
                                       int64_t ignore_index, float* losses, float* lse, float* sums, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  const char* fn = "kq_linear_cross_entropy";
  if (int rc = loss::check(fn, w_fmt, h, ldh, tokens, w, w_scale, vocab, k, target, loss::NONE)) return rc;
  hipStream_t st = (hipStream_t)stream;
  int cus = 0;
  if (int rc = kq_check_launch(loss::stream_cus(st, &cus), fn)) return rc;
  const loss::Plan p = loss::plan(w_fmt, tokens, vocab, k, false, cus);
  if (workspace_bytes < p.bytes || kq_misaligned(workspace, 256))
    return kq_fail(KQ_ERR_INVALID, "%s: workspace needs %lld bytes, 256-byte aligned", fn, (long long)p.bytes);
  char* ws = (char*)workspace;
  if (p.few) {
    const LossTail tail{target, (float2_t*)(ws + p.o_part), (vocab + 15) / 16, (float*)(ws + p.o_z)};
    hipError_t e = mx_skinny_loss(w_fmt, {h, nullptr, ldh, (const uint8_t*)w, w_scale, nullptr, 0, (int)tokens,
                                          (int)vocab, (int)k}, tail, st);
    if (e == hipSuccess) {
      loss::combine_few_kernel<<<(unsigned)tokens, 1024, 0, st>>>(tail.part, tail.parts, target, ignore_index, vocab,
                                                                  tail.z_target, losses, lse);
      e = hipGetLastError();
    }
    if (e == hipSuccess && sums) {
      loss::sum_kernel<<<1, 1024, 0, st>>>(losses, (int)tokens, target, ignore_index, sums);
      e = hipGetLastError();
    }
    return kq_check_launch(e, fn);
  }
  int* count = (int*)(ws + p.o_count);
  loss::compact_kernel<<<1, 1024, 0, st>>>(target, ignore_index, (int)tokens, (int*)(ws + p.o_rows),
                                           (int*)(ws + p.o_place), count, loss::Slicing{},
                                           loss::Upstream{});
  if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
  if (tokens > 0) {
    loss::Gather g{};
    g.h = (const char*)h;
    g.ldh = 2 * ldh;
    g.target = target;
    g.place = (int*)(ws + p.o_place);
    g.count = count;
    g.tokens = (int)tokens;
    g.k = (int)k;
    g.vocab = vocab;
    g.hc = ws + p.o_hc;
    g.target_c = (int*)(ws + p.o_target);
    loss::gather_kernel<<<(unsigned)tokens, 256, 0, st>>>(g);
    if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
    loss::LogitArgs a{};
    a.hc = ws + p.o_hc;
    a.count = count;
    a.target_c = g.target_c;
    a.k = (int)k;
    a.tokens = (int)tokens;
    a.part = (float2_t*)(ws + p.o_part);
    a.z_target = (float*)(ws + p.o_z);
    for (int64_t first = 0; first < vocab; first += p.piece) {
      a.first = (int)first;
      a.rows = (int)(vocab - first < p.piece ? vocab - first : p.piece);
      if (int rc = loss::piece_rows(w_fmt, w, w_scale, first, a.rows, k, ws + p.o_w, &a.w, stream)) return rc;
      loss::logit_kernel<false><<<loss::persistent_grid(cus), mm16::THREADS, 0, st>>>(a);
      if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
      a.part0 += (a.rows + mm16::BM - 1) / mm16::BM;
    }
    loss::combine_kernel<<<(unsigned)((tokens + 15) / 16), 1024, 0, st>>>(a.part, 4 * a.part0, (int)tokens, g.place,
                                                                         g.target_c, a.z_target, losses, lse);
    if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
  }
  if (!sums) return KQ_OK;
  loss::sum_kernel<<<1, 1024, 0, st>>>(losses, (int)tokens, target, ignore_index, sums);
  return kq_check_launch(hipGetLastError(), fn);
}

extern "C" int kq_linear_cross_entropy_backward(int w_fmt, const void* h, int64_t ldh, int64_t tokens, const void* w,
                                                const uint8_t* w_scale, int64_t vocab, int64_t k, const int64_t* target,
                                                int64_t ignore_index, const float* lse, const float* grad, int reduction,
                                                void* dh, int64_t lddh, void* dw, void* workspace,
                                                int64_t workspace_bytes, void* stream) {
  const char* fn = "kq_linear_cross_entropy_backward";
  if (int rc = loss::check(fn, w_fmt, h, ldh, tokens, w, w_scale, vocab, k, target, reduction)) return rc;
  if (dw && w_fmt != KQ_FMT_BF16) return kq_fail(KQ_ERR_INVALID, "%s: only a bf16 head has a gradient", fn);
  if ((dh && (lddh < k || lddh % 8)) || kq_misaligned(dh, 16) || kq_misaligned(dw, 16))
    return kq_fail(KQ_ERR_INVALID, "%s: need lddh >= k, lddh %% 8 == 0, dh and dw 16-byte aligned", fn);
  hipStream_t st = (hipStream_t)stream;
  int cus = 0;
  if (int rc = kq_check_launch(loss::stream_cus(st, &cus), fn)) return rc;
  const loss::Plan p = loss::plan(w_fmt, tokens, vocab, k, true, cus);
  if (workspace_bytes < p.bytes || kq_misaligned(workspace, 256))
    return kq_fail(KQ_ERR_INVALID, "%s: workspace needs %lld bytes, 256-byte aligned", fn, (long long)p.bytes);
  char* ws = (char*)workspace;
  int* count = (int*)(ws + p.o_count);
  float* alpha = (float*)(ws + p.o_alpha);
  const bool planes = p.slices > 1 || p.pieces > 1;
  loss::compact_kernel<<<1, 1024, 0, st>>>(
      target, ignore_index, (int)tokens, (int*)(ws + p.o_rows), (int*)(ws + p.o_place), count,
      loss::Slicing{planes ? p.slices * tokens : 0, (int)((p.piece + 63) / 64), (int)k, (int)loss::persistent_grid(cus)},
      loss::Upstream{grad, reduction == loss::MEAN, reduction == loss::NONE ? nullptr : alpha});
  if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
  if (tokens == 0 && !dw) return KQ_OK;
  loss::Gather g{};
  g.h = (const char*)h;
  g.ldh = 2 * ldh;
  g.target = target;
  g.place = (int*)(ws + p.o_place);
  g.count = count;
  g.tokens = (int)tokens;
  g.k = (int)k;
  g.vocab = vocab;
  g.hc = ws + p.o_hc;
  g.target_c = (int*)(ws + p.o_target);
  g.lse = lse;
  g.grad = grad;
  g.reduction = reduction;
  g.alpha = alpha;
  g.lse_c = (float*)(ws + p.o_lse);
  g.u_c = (float*)(ws + p.o_u);
  g.dh = (char*)dh;
  g.lddh = 2 * lddh;
  if (reduction == loss::NONE) {
    loss::alpha_kernel<<<1, 1024, 0, st>>>(grad, (int)tokens, g.place, alpha);
    if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
  }
  loss::gather_kernel<<<(unsigned)tokens + 8, 256, 0, st>>>(g);
  if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
  const unsigned grid = loss::persistent_grid(cus);
  loss::LogitArgs a{};
  a.hc = g.hc;
  a.count = count;
  a.target_c = g.target_c;
  a.k = (int)k;
  a.tokens = (int)tokens;
  a.lse_c = g.lse_c;
  a.u_c = g.u_c;
  a.dt = ws + p.o_dt;
  a.ldg = (int)p.ldg;
  for (int64_t first = 0; first < vocab; first += p.piece) {
    a.first = (int)first;
    a.rows = (int)(vocab - first < p.piece ? vocab - first : p.piece);
    if (int rc = loss::piece_rows(w_fmt, w, w_scale, first, a.rows, k, ws + p.o_w, &a.w, stream)) return rc;
    loss::logit_kernel<true><<<grid, mm16::THREADS, 0, st>>>(a);
    if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
    if (dh) {
      const loss::DhArgs d{a.dt, (int)p.ldg, a.w, count, (int*)(ws + p.o_rows), a.rows, (int)k,
                           alpha, planes ? nullptr : (char*)dh, 2 * lddh, (float*)(ws + p.o_planes), first > 0};
      loss::dh_kernel<<<grid, mm16::THREADS, 0, st>>>(d);
      if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
    }
    if (dw) {
      const loss::DwArgs d{a.dt, (int)p.ldg, g.hc, count, alpha, a.rows, (int)k, (char*)dw + first * k * 2};
      loss::dw_kernel<<<grid, mm16::THREADS, 0, st>>>(d);
      if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
    }
  }
  if (dh && planes && tokens > 0) {
    loss::dh_sum_kernel<<<(unsigned)tokens, 256, 0, st>>>((const float*)(ws + p.o_planes), count, (int)k,
                                                         g.place, alpha, (char*)dh, 2 * lddh);
    if (int rc = kq_check_launch(hipGetLastError(), fn)) return rc;
  }
  return KQ_OK;
}
