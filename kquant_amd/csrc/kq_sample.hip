// One token for each row of logits from a given uniform number, with temperature,
// top-k, top-p and min-p.
//
// Of a row l with maximum M and temperature t, w_i = exp((l_i - M) / t).  In the
// order of descending logits (ties: the lower index first) the first k tokens are
// kept, of those the shortest prefix whose weight reaches p of theirs (a token
// stays while the weight before it is below p total), of those the tokens with
// w_i >= min_p; the first token always.  So the kept tokens are a prefix of the
// order.  The draw is the first kept token, by index, whose cumulative weight
// exceeds u times the total.
//
// Which token that is must not depend on how sums are split, so weights are
// integers: w_i in units of 2^-45 (below 2^-46: zero), from an exponential in 64
// bits, and every sum of them is exact, in any order.  A border between two
// tokens is off by 2^-46 a token, the fp32 number u is 2^-24 apart from the next.
// The order of the logits is that of 32-bit keys, and with the index behind
// them of 64-bit ones without ties.
#include "kq_internal.h"
#include "kq_common.h"

namespace kq {
namespace sample {

constexpr int MAX_VOCAB = 1 << 18;  // sums of weights stay below 2^63
constexpr int UNIT = 45;            // a weight of 1 is 2^UNIT
constexpr double FAR = -33.0;       // exp(FAR) rounds to 0 units
constexpr int CHUNK = 512;          // tokens whose kept weight is summed on its own
constexpr int CHUNKS = MAX_VOCAB / CHUNK;

// One number for all rows, or one for each.
struct Setting {
  const float* rows;
  double all;
  __device__ __forceinline__ double of(int64_t r) const { return rows ? (double)rows[r] : all; }
};

struct Args {
  const char* logits;
  int64_t ld;  // bytes
  int vocab;
  int vec;     // rows are whole 16-byte pieces from aligned addresses
  const float* uniform;
  Setting temperature, top_p, min_p;
  const int* k_rows;
  int k_all;
  int64_t* token;
  float* logprob;  // may be null
};

// Larger for larger logits; -0 is 0.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// Earlier in the order: larger.
__device__ __forceinline__ uint64_t place_of(float v, int index) {
  return (uint64_t)key_of(v) << 32 | (uint32_t)~index;
}

template <int DT>
__device__ __forceinline__ float logit(const char* row, int i) {
  if (DT == KQ_DT_F32) return reinterpret_cast<const float*>(row)[i];
  const uint32_t h = reinterpret_cast<const uint16_t*>(row)[i];
  return DT == KQ_DT_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}

// exp(d) for FAR <= d <= 0 (0 below): 2^k times the Taylor sum of the rest,
// |rest| <= ln 2 / 2, to the 12th power (the next term is below 2e-16).
__device__ __forceinline__ double exp64(double d) {
  if (!(d >= FAR)) return 0.0;
  const double k = rint(d * 1.4426950408889634);
  double r = fma(-k, 0.6931471805598903, d);  // ln 2 in two parts, the first of 43 bits: k times it is exact
  r = fma(-k, 5.497923018708371e-14, r);
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)k);
}

__device__ __forceinline__ uint64_t units(double w) {
  // the sum's mantissa is w in units, rounded to nearest
  return (uint64_t)__double_as_longlong(fma(w, (double)(1ull << UNIT), 4503599627370496.0)) & 0xfffffffffffffull;
}

// A row's logits as weights.
struct Scale {
  float top;        // M
  double inv_t, M;
  __device__ __forceinline__ double distance(float v) const {
    return v == top ? 0.0 : ((double)v - M) * inv_t;  // (an infinite M: 0 or -inf)
  }
  __device__ __forceinline__ double weight(float v) const { return exp64(distance(v)); }
};

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int src) { return __shfl((unsigned long long)v, src); }
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor((unsigned long long)v, d);
  return v;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max64(v, __shfl_xor((unsigned long long)v, d));
  return v;
}
// Inclusive sums over the lanes.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t x = __shfl_up((unsigned long long)v, d);
    if (lane >= d) v += x;
  }
  return v;
}

// The whole units in f total, for 0 < f < 1, exactly; `rest`: whether it has a fraction besides.
__device__ __forceinline__ uint64_t share(double f, uint64_t total, bool& rest) {
  const uint64_t bits = (uint64_t)__double_as_longlong(f);
  const int exponent = (int)(bits >> 52);
  const uint64_t m = (bits & 0xfffffffffffffull) | (exponent ? 1ull << 52 : 0);
  const int shift = 1075 - (exponent ? exponent : 1);  // f = m 2^-shift, shift >= 53
  const uint64_t hi = __umul64hi(m, total), lo = m * total;  // below 2^116
  if (shift >= 116) {
    rest = true;
    return 0;
  }
  if (shift >= 64) {
    rest = lo != 0 || (hi & ((1ull << (shift - 64)) - 1)) != 0;
    return hi >> (shift - 64);
  }
  rest = (lo & ((1ull << shift) - 1)) != 0;
  return hi << (64 - shift) | lo >> shift;
}

// The least whole weight that reaches p total.
__device__ __forceinline__ uint64_t nucleus(double p, uint64_t total) {
  if (!(p > 0.0)) return 1;
  bool rest;
  const uint64_t v = share(p, total, rest) + (rest ? 1 : 0);
  return v ? v : 1;
}
// The draw's token is the first whose cumulative weight is larger than this.
__device__ __forceinline__ uint64_t drawn_weight(double u, uint64_t total) {
  if (!(u < 1.0)) return total - 1;
  bool rest;
  return u > 0.0 ? share(u, total, rest) : 0;
}

// --------------------------------------------------------- one row, whole --

constexpr int T = 1024;
constexpr int DIGIT = 11, BINS = 1 << DIGIT;

struct Shared {
  unsigned long long mass[BINS];
  unsigned int count[BINS];
  unsigned long long chunk[CHUNKS];
  uint64_t part[T / 64];
  uint64_t found[4];
};

// Sum of v over the workgroup, and (before) of the threads below this one.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, Shared& s, uint64_t& before) {
  const uint64_t upto = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.part[threadIdx.x >> 6] = upto;
  __syncthreads();
  uint64_t total = 0, below = 0;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    if (w < (int)(threadIdx.x >> 6)) below += s.part[w];
    total += s.part[w];
  }
  before = below + upto - v;
  return total;
}

struct Cut {
  uint64_t place;  // of the last token kept
  uint64_t mass;   // weight up to and with it
};

// The token, in the order, with which a count of k (BY_COUNT) or a weight of
// `target` units is reached; one digit of its place a pass over the row.  All
// tokens together reach it.
template <int DT, bool BY_COUNT>
__device__ __forceinline__ Cut select(const char* row, int vocab, const Scale& sc, uint64_t target, Shared& s) {
  uint64_t prefix = 0, count = 0, mass = 0;
  constexpr int SHIFTS[6] = {53, 42, 31, 20, 9, 0};
  int top = 64;
  for (int step = 0; step < 6; ++step) {
    const int shift = SHIFTS[step], bits = top - shift;
    for (int b = threadIdx.x; b < BINS; b += T) {
      s.mass[b] = 0;
      s.count[b] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < vocab; i += T) {
      const float v = logit<DT>(row, i);
      const uint64_t place = place_of(v, i);
      if (top < 64 && (place ^ prefix) >> top) continue;
      const int bin = (int)(~(place >> shift) & ((1u << bits) - 1));  // the first of the order first
      atomicAdd(&s.count[bin], 1u);
      const uint64_t w = units(sc.weight(v));
      if (w) atomicAdd(&s.mass[bin], (unsigned long long)w);
    }
    __syncthreads();
    // two bins a thread
    const int b0 = 2 * threadIdx.x;
    const uint64_t c0 = s.count[b0], c1 = s.count[b0 + 1], m0 = s.mass[b0], m1 = s.mass[b0 + 1];
    uint64_t cb, mb;
    block_scan(c0 + c1, s, cb);
    block_scan(m0 + m1, s, mb);
    cb += count;
    mb += mass;
    const uint64_t want = target;
    const uint64_t at0 = BY_COUNT ? cb : mb, v0 = BY_COUNT ? c0 : m0, v1 = BY_COUNT ? c1 : m1;
    // the one bin in which the target is reached
    const bool in0 = at0 < want && at0 + v0 >= want, in1 = at0 + v0 < want && at0 + v0 + v1 >= want;
    __syncthreads();
    if (in0 || in1) {
      s.found[0] = in0 ? b0 : b0 + 1;
      s.found[1] = in0 ? cb : cb + c0;
      s.found[2] = in0 ? mb : mb + m0;
      s.found[3] = in0 ? m0 : m1;
    }
    __syncthreads();
    prefix |= (~s.found[0] & ((1u << bits) - 1)) << shift;
    count = s.found[1];
    mass = s.found[2];
    top = shift;
  }
  return Cut{prefix, mass + s.found[3]};
}

template <int DT>
__global__ __launch_bounds__(T) void row_kernel(const Args a) {
  __shared__ Shared s;
  const int64_t r = blockIdx.x;
  const char* row = a.logits + r * a.ld;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the first of the order, and whether a NaN is among the logits
  uint64_t best = 0;
  bool nan = false;
  for (int i = threadIdx.x; i < a.vocab; i += T) {
    const float v = logit<DT>(row, i);
    nan |= v != v;
    best = max64(best, place_of(v, i));
  }
  if (nan) best = ~0ull;  // (no logit's place: its index would be -1)
  best = wave_max(best);
  if (lane == 0) s.part[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < T / 64; ++w) best = max64(best, s.part[w]);
  const float top = value_of((uint32_t)(best >> 32));
  const int first = ~(int)(uint32_t)best;
  const double t = a.temperature.of(r);
  if (best == ~0ull || top == -__builtin_inff() || !(t > 0.0)) {
    const bool none = best == ~0ull || top == -__builtin_inff();
    if (threadIdx.x == 0) {
      a.token[r] = none ? -1 : first;
      if (a.logprob) a.logprob[r] = none ? __builtin_nanf("") : 0.0f;
    }
    return;
  }
  const Scale sc{top, 1.0 / t, (double)top};
  const int k = a.k_rows ? a.k_rows[r] : a.k_all;
  const double p = a.top_p.of(r), min_p = a.min_p.of(r);
  uint64_t last = 0;  // the place of the last token kept
  uint64_t total = 0;
  if (k > 0 && k < a.vocab) {
    const Cut c = select<DT, true>(row, a.vocab, sc, (uint64_t)k, s);
    last = c.place;
    total = c.mass;
  } else if (p < 1.0) {
    uint64_t sum = 0, before;
    for (int i = threadIdx.x; i < a.vocab; i += T) sum += units(sc.weight(logit<DT>(row, i)));
    total = block_scan(sum, s, before);
  }
  if (p < 1.0) {
    last = max64(last, select<DT, false>(row, a.vocab, sc, nucleus(p, total), s).place);
  }
  auto kept = [&](float v, int i, double w) { return place_of(v, i) >= last && (w >= min_p || i == first); };
  // the kept weight of each chunk, and where the draw falls among them
  const int chunks = (a.vocab + CHUNK - 1) / CHUNK;
  for (int c = wave; c < chunks; c += T / 64) {
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < CHUNK / 64; ++j) {
      const int i = c * CHUNK + j * 64 + lane;
      if (i < a.vocab) {
        const float v = logit<DT>(row, i);
        const double w = sc.weight(v);
        if (kept(v, i, w)) sum += units(w);
      }
    }
    sum = wave_sum(sum);
    if (lane == 0) s.chunk[c] = sum;
  }
  __syncthreads();
  uint64_t before;
  const uint64_t mine = (int)threadIdx.x < chunks ? s.chunk[threadIdx.x] : 0;
  total = block_scan(mine, s, before);
  const uint64_t at = drawn_weight((double)a.uniform[r], total);
  __syncthreads();
  if (mine && before <= at && at < before + mine) {
    s.found[0] = threadIdx.x;
    s.found[1] = before;
  }
  __syncthreads();
  const int base = (int)s.found[0] * CHUNK;
  const uint64_t under = s.found[1];
  const int i = base + (int)threadIdx.x;
  uint64_t w = 0;
  float v = 0.0f;
  if ((int)threadIdx.x < CHUNK && i < a.vocab) {
    v = logit<DT>(row, i);
    const double e = sc.weight(v);
    if (kept(v, i, e)) w = units(e);
  }
  block_scan(w, s, before);
  before += under;
  if (w && before <= at && at < before + w) {
    a.token[r] = i;
    if (a.logprob) a.logprob[r] = (float)(sc.distance(v) - log((double)total * (1.0 / (double)(1ull << UNIT))));
  }
}

}  // namespace sample
}  // namespace kq

using namespace kq;

extern "C" int kq_sample_tokens(int dtype, const void* logits, int64_t ld, int64_t rows, int64_t vocab, const float* uniform,
                                const float* temperature_rows, double temperature, const int* top_k_rows, int64_t top_k,
                                const float* top_p_rows, double top_p, const float* min_p_rows, double min_p,
                                int64_t* tokens, float* logprobs, void* stream) {
  const char* fn = "kq_sample_tokens";
  if (dtype != KQ_DT_BF16 && dtype != KQ_DT_F16 && dtype != KQ_DT_F32)
    return kq_fail(KQ_ERR_INVALID, "%s: dtype must be bf16, f16 or f32", fn);
  if (rows < 0 || vocab < 1 || ld < vocab)
    return kq_fail(KQ_ERR_INVALID, "%s: need rows >= 0, vocab >= 1, a row stride of at least vocab (rows=%lld vocab=%lld ld=%lld)",
                   fn, (long long)rows, (long long)vocab, (long long)ld);
  if (vocab > sample::MAX_VOCAB || rows > INT32_MAX)
    return kq_fail(KQ_ERR_LIMIT, "%s: at most %d tokens in the vocabulary and 2^31 - 1 rows", fn, sample::MAX_VOCAB);
  if (rows == 0) return KQ_OK;
  if (!logits || !uniform || !tokens) return kq_fail(KQ_ERR_INVALID, "%s: null buffer", fn);
  const int es = dtype == KQ_DT_F32 ? 4 : 2;
  if (kq_misaligned(logits, es) || kq_misaligned(uniform, 4) || kq_misaligned(tokens, 8) || kq_misaligned(logprobs, 4) ||
      kq_misaligned(temperature_rows, 4) || kq_misaligned(top_k_rows, 4) || kq_misaligned(top_p_rows, 4) ||
      kq_misaligned(min_p_rows, 4))
    return kq_fail(KQ_ERR_INVALID, "%s: buffers must be aligned to their type", fn);
  sample::Args a{};
  a.logits = (const char*)logits;
  a.ld = ld * es;
  a.vocab = (int)vocab;
  a.vec = !kq_misaligned(logits, 16) && a.ld % 16 == 0;
  a.uniform = uniform;
  a.temperature = {temperature_rows, temperature};
  a.top_p = {top_p_rows, top_p};
  a.min_p = {min_p_rows, min_p};
  a.k_rows = top_k_rows;
  a.k_all = top_k > vocab || top_k < 0 ? 0 : (int)top_k;
  a.token = tokens;
  a.logprob = logprobs;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == KQ_DT_BF16) sample::row_kernel<KQ_DT_BF16><<<(unsigned)rows, sample::T, 0, st>>>(a);
  else if (dtype == KQ_DT_F16) sample::row_kernel<KQ_DT_F16><<<(unsigned)rows, sample::T, 0, st>>>(a);
  else sample::row_kernel<KQ_DT_F32><<<(unsigned)rows, sample::T, 0, st>>>(a);
  return kq_check_launch(hipGetLastError(), fn);
}
