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
constexpr int CHUNK = 512;          // tokens whose kept weight is summed on its own
constexpr int CHUNKS = MAX_VOCAB / CHUNK;  // no more than a workgroup's threads

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

// A constant in scalar registers: as an FMA's addend it needs no copy into the result's.
__device__ __forceinline__ double scalar(double c) {
  asm("" : "+s"(c));
  return c;
}

// A row's logits as weights.
struct Scale {
  float top;
  double M, a;  // the top (1e300 for an infinite one) and log2(e) / t
  __device__ __forceinline__ Scale() {}
  __device__ __forceinline__ Scale(float m, double t)
      : top(m),
        M(m == __builtin_inff() ? 1e300 : (double)m),
        a(fmax(fmin(1.4426950408889634 / t, 1e300), m == __builtin_inff() ? 1.0 : 0.0)) {}  // (t may be infinite)
  // log2 of a weight: 0 for the top (an infinite one too), no less than -60, which is no weight
  __device__ __forceinline__ double log2_weight(float v) const { return fmin(fmax(((double)v - M) * a, -60.0), 0.0); }
  // The weight in units, not rounded: 2^(k + UNIT) 2^f with |f| <= 1/2, 2^f by the polynomial of degree 10 that meets
  // it at the Chebyshev points (within 3e-16).  Only additions, products and FMAs: they run at the full fp64 rate.
  __device__ __forceinline__ double weight(float v) const {
    constexpr double SHIFT = 6755399441055744.0 + UNIT;  // 1.5 2^52: k + UNIT in the low word of the sum
    const double y = log2_weight(v), t = y + SHIFT;
    const double f = y - (t - SHIFT);
    double p = fma(scalar(7.072585949269223e-09), f, scalar(1.0208690299958306e-07));
    p = fma(p, f, scalar(1.321544258792169e-06));
    p = fma(p, f, scalar(1.5252657260200837e-05));
    p = fma(p, f, scalar(0.0001540353044173605));
    p = fma(p, f, scalar(0.0013333558230164974));
    p = fma(p, f, scalar(0.009618129107606888));
    p = fma(p, f, scalar(0.05550410866444772));
    p = fma(p, f, scalar(0.24022650695910097));
    p = fma(p, f, scalar(0.69314718055995));
    p = fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
  }
};

// A weight rounded to whole units: the mantissa of its sum with 2^52.
constexpr uint64_t RAW = 0x4330000000000000ull;  // the bits of 2^52
__device__ __forceinline__ uint64_t raw_units(double w) { return (uint64_t)__double_as_longlong(w + 4503599627370496.0); }
__device__ __forceinline__ uint64_t units(double w) { return raw_units(w) - RAW; }
constexpr double ONE = (double)(1ull << UNIT);

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

__device__ __forceinline__ float logprob_of(double log2_weight, uint64_t total) {
  return (float)(log2_weight * 0.6931471805599453 - log((double)total * (1.0 / ONE)));
}

// --------------------------------------------------------- one row, whole --

constexpr int T = 512;
constexpr int DIGIT = 11, BINS = 1 << DIGIT;

struct Shared {
  unsigned long long mass[BINS];
  unsigned int count[BINS];
  unsigned long long chunk[CHUNKS];
  uint64_t part[T / 64];
  uint64_t found[5];
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
  uint64_t prefix = 0, count = 0, mass = 0, own = 0;
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
    constexpr int PER = BINS / T;
    uint64_t c[PER], m[PER], cs = 0, ms = 0, cb, mb;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      cs += c[j] = s.count[PER * threadIdx.x + j];
      ms += m[j] = s.mass[PER * threadIdx.x + j];
    }
    block_scan(cs, s, cb);
    block_scan(ms, s, mb);
    cb += count;
    mb += mass;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint64_t at = BY_COUNT ? cb : mb, v = BY_COUNT ? c[j] : m[j];
      if (at < target && at + v >= target) {  // the one bin in which the target is reached
        s.found[0] = PER * threadIdx.x + j;
        s.found[1] = cb;
        s.found[2] = mb;
        s.found[3] = m[j];
        s.found[4] = c[j];
      }
      cb += c[j];
      mb += m[j];
    }
    __syncthreads();
    prefix |= (~s.found[0] & ((1u << bits) - 1)) << shift;
    count = s.found[1];
    mass = s.found[2];
    own = s.found[3];
    top = shift;
    if (shift > 0 && s.found[4] == 1) {  // one token is left: its other digits are read from it
      __syncthreads();                   // (all have read what was found)
      for (int i = threadIdx.x; i < vocab; i += T) {
        const uint64_t place = place_of(logit<DT>(row, i), i);
        if (!((place ^ prefix) >> shift)) s.found[0] = place;
      }
      __syncthreads();
      prefix = s.found[0];
      break;
    }
  }
  __syncthreads();  // (the next search writes there)
  return Cut{prefix, mass + own};
}

template <int DT>
__device__ __forceinline__ void whole_row(const Args& a, int64_t r, Shared& s) {
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
  const Scale sc(top, t);
  const int k = a.k_rows ? a.k_rows[r] : a.k_all;
  const double p = a.top_p.of(r), min_p = fmin(a.min_p.of(r), 1.0) * ONE;
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
  auto kept = [&](float v, int i, double w) { return place_of(v, i) >= last && w >= min_p; };
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
    if (a.logprob) a.logprob[r] = logprob_of(sc.log2_weight(v), total);
  }
}

template <int DT>
__global__ __launch_bounds__(T) void row_kernel(const Args a) {
  __shared__ Shared s;
  whole_row<DT>(a, blockIdx.x, s);
}

// ------------------------------------------------------- many workgroups a row --

// A row's tokens fall into bins of equal width by their distance from the top, so
// a cut falls into one bin (with top-k the weight's cut into a few, since the bins'
// weights are sums of fp32 exponentials then), and only what lies there has to be
// ordered.
// Three launches, a workgroup a slice of a row:
//   stats      the slice's first place and least logit; clears the row's bins
//   histogram  (with top-k or top-p) every bin's weight; with top-k its tokens and a
//              rough weight, since only the bins up to the count's matter then.  The
//              row's last workgroup finds the cuts' bins
//   weigh      exact weight of each chunk's tokens in the bins before the cuts, and
//              the list of the tokens in the cuts' bins; with top-k also the weight
//              of the bins that count for top-p's total only.  The row's last
//              workgroup orders the list, cuts, and finds the draw's chunk and token
// No workgroup waits for another: the last one is who finds that all others of its
// row have counted themselves.  What it reads of theirs goes to memory and comes
// from there in agent-scope accesses, all of which end before the count (a fence
// would write each workgroup's L2 back).
// A list longer than LIST (many equal logits at a cut) leaves the row to
// whole_row, in one workgroup after the three launches: a bf16 row of 129280 equal
// logits 1.25 ms with top-k or top-p, 2.4 with both (64 rows 2.5, 4.7); logits of 20
// with a spread of 0.3, which are 1/8 apart, 0.65 ms with top-p (64 rows 1.2).
// What bounds it, kernels in us.  One row of 129280: without cuts 3.5 + 8.9, with
// 3.5 + 8 + 12 - 17, nearly all of the last ones the chain of dependent reads,
// barriers and LDS steps of the row's last workgroup.  64 such rows (33 MB, 8 to
// read): stats 8.6; histogram 16 - 18; weigh 20 without cuts, 23 - 24 with top-k 50,
// where few chunks hold a token that counts, 28 - 32 with top-k 1000 or top-p, where
// most do: by difference some 5 are the exponentials (26 instructions each), 6 the last
// workgroup's sums and draw, and 4 - 9 more its list.  256 rows of 65536 in bf16
// without cuts 10 + 28, of which 16.8 M exponentials are about 11.
constexpr int SLICE_T = T;
static_assert(CHUNKS <= SLICE_T && CHUNK <= SLICE_T, "a thread for each chunk and each token of one");
constexpr int NEAR = 1024;   // listed tokens that a workgroup gathers before they go to the list
constexpr int NBINS = 2048, FAR_BIN = NBINS - 1;  // FAR_BIN: tokens of no weight
constexpr int BINS_EACH = NBINS / SLICE_T;        // a thread's bins where a workgroup looks through them
constexpr int LIST = 4096;
constexpr int COUNT_SHIFT = 44;  // a bin: tokens << 44 | weight in 2^-25
constexpr float BIN_WEIGHT = 33554432.0f;

struct Part {
  uint64_t best;
  float least;  // of the logits above -inf
  uint32_t pad;
};
struct Cuts {
  int lo, hi;         // bins of the weight's cut (lo: those before are kept); of the count's alone both its bin
  int kb;             // the count's bin (NBINS: none)
  int slow;           // the list would be too long
  int before_lo;      // tokens in the bins before lo
  int before_kb;      // and before kb
  int in_range;       // tokens in [lo, hi]
  int pad;
};
struct RowState {
  Cuts cuts;
  unsigned long long sure, middle;  // with top-k: weight of the bins before lo, and of those that only count for the total
  unsigned long long before, total; // without: of the bins before lo, and of all
  unsigned int listed;
  unsigned int arrived[2];          // workgroups that are through with the histogram, and with weighing
  unsigned int pad;
};

struct Split {
  Part* parts;                  // [rows][slices]
  unsigned long long* bins;     // [rows][NBINS]
  RowState* state;              // [rows]
  unsigned long long* chunk;    // [rows][chunks]
  unsigned long long* list;     // [rows][LIST]
  int slices, per, chunks;      // per: chunks a slice
  int filters;                  // top-k or top-p may cut
};

__device__ __forceinline__ uint64_t shared_load(const unsigned long long* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void shared_store(unsigned long long* p, uint64_t v) {
  __hip_atomic_store(p, (unsigned long long)v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this workgroup is the last of `all` to come here; its shared accesses have ended.
__device__ __forceinline__ bool last_of(unsigned int* counter, int all) {
  __shared__ bool last;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned int)(all - 1);
  __syncthreads();
  return last;
}

// What a row asks for.
struct Row {
  bool none, greedy;
  int first;          // of the order, of a greedy row
  int k;              // 0: all
  double p, min_p;    // min_p in units, no more than the top's weight
  Scale sc;
  float range, to_bin, to_exp;
  __device__ __forceinline__ bool cuts() const { return k > 0 || p < 1.0; }
};

// Half the distance from the top (the whole one may not be finite).
__device__ __forceinline__ float down(const Row& q, float v) {
  return v == q.sc.top ? 0.0f : fmaf(-0.5f, v, 0.5f * q.sc.top);
}
// The bins reach as far as weights do, or the logits: below `range` they are
// numbered from 0 to NBINS - 2.
__device__ __forceinline__ float bin_place(const Row& q, float down) {
  return down < q.range ? down * q.to_bin : (float)FAR_BIN;
}
__device__ __forceinline__ int bin_of(const Row& q, float down) { return (int)bin_place(q, down); }

__device__ __forceinline__ Row row_of(const Args& a, const Split& sp, int64_t r) {
  Row q;
  const int lane = threadIdx.x & 63;
  uint64_t best = 0;
  float least = __builtin_inff();
  for (int g = lane; g < sp.slices; g += 64) {
    const Part p = sp.parts[r * sp.slices + g];
    best = max64(best, p.best);
    least = fminf(least, p.least);
  }
  best = wave_max(best);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) least = fminf(least, __shfl_xor(least, d));
  const float top = value_of((uint32_t)(best >> 32));
  q.first = ~(int)(uint32_t)best;
  const double t = a.temperature.of(r);
  q.sc = Scale(top, t);
  q.none = best == ~0ull || top == -__builtin_inff();
  q.greedy = !(t > 0.0);
  const int k = a.k_rows ? a.k_rows[r] : a.k_all;
  q.k = k > 0 && k < a.vocab ? k : 0;
  q.p = a.top_p.of(r);
  q.min_p = fmin(a.min_p.of(r), 1.0) * ONE;
  // logits further than 32.25 t weigh less than 2^-46; the least one itself is within the range
  q.range = fmaxf(fminf(16.125f * (float)t, down(q, least) * 1.0001f), 1e-30f);
  q.to_bin = ((float)FAR_BIN - 0.5f) / q.range;
  q.to_exp = fmaxf((float)(-2.8853900817779268 / t), -3e38f);  // (the top's distance of 0 times an infinity were NaN)
  return q;
}

// Eight logits a lane of chunk c (-inf where there is none); at(j) is the index of
// the j-th, in pieces of 16 bytes where the rows are.
template <int DT>
struct Chunk {
  float v[8];
  int base, lane, vocab;
  bool vec;
  __device__ __forceinline__ int at(int j) const {
    if (!vec) return base + 64 * j + lane;
    return DT == KQ_DT_F32 ? base + 256 * (j >> 2) + 4 * lane + (j & 3) : base + 8 * lane + j;
  }
  __device__ __forceinline__ bool there(int j) const { return at(j) < vocab; }
  __device__ __forceinline__ void load(const Args& a, const char* row, int c) {
    base = c * CHUNK;
    lane = threadIdx.x & 63;
    vocab = a.vocab;
    vec = a.vec && base + CHUNK <= vocab;
    if (vec) {
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      if (DT == KQ_DT_F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(row + 4ll * (base + 256 * h + 4 * lane));
#pragma unroll
          for (int j = 0; j < 4; ++j) v[4 * h + j] = __uint_as_float(x[j]);
        }
      } else {
        const u32x4 x = *reinterpret_cast<const u32x4*>(row + 2ll * (base + 8 * lane));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t h = j & 1 ? x[j >> 1] >> 16 : x[j >> 1] & 0xffffu;
          v[j] = DT == KQ_DT_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = there(j) ? logit<DT>(row, at(j)) : -__builtin_inff();
    }
  }
};

// f(chunk, its number) of a wave's chunks first, first + the workgroup's waves, ... below end, with the next D chunks'
// logits on their way; `ready`, which may end it, runs when the first ones' are.
template <int DT, int D, class F, class R>
__device__ __forceinline__ void for_chunks(const Args& a, const char* row, int first, int end, F&& f, R&& ready) {
  constexpr int STEP = SLICE_T / 64;
  Chunk<DT> x[D];
#pragma unroll
  for (int i = 0; i < D; ++i)
    if (first + i * STEP < end) x[i].load(a, row, first + i * STEP);
  if (!ready()) return;
  // one copy of f: a kernel's code comes from memory once a CU, and costs as its data does
#pragma nounroll
  for (int c = first; c < end; c += STEP) {
    const Chunk<DT> now = x[0];
#pragma unroll
    for (int i = 0; i + 1 < D; ++i) x[i] = x[i + 1];
    if (c + D * STEP < end) x[D - 1].load(a, row, c + D * STEP);
    f(now, c);
  }
}

template <int DT>
__global__ __launch_bounds__(SLICE_T) void stats_kernel(const Args a, const Split sp) {
  __shared__ Part part[SLICE_T / 64];
  const int64_t r = blockIdx.x / sp.slices;
  const int g = (int)(blockIdx.x - r * sp.slices), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char* row = a.logits + r * a.ld;
  const float inf = __builtin_inff();
  float high = -inf, least = inf;
  int from = -1;  // this lane's chunk with `high` first
  bool nan = false;
  const int end = min((g + 1) * sp.per, sp.chunks);
  // (the median with an infinity: a maximum or minimum in one instruction, without quieting its operands first)
  auto larger = [&](float x, float y) { return __builtin_amdgcn_fmed3f(x, y, inf); };
  auto smaller = [&](float x, float y) { return __builtin_amdgcn_fmed3f(x, y, -inf); };
  for_chunks<DT, 4>(a, row, g * sp.per + wave, end, [&](const Chunk<DT>& x, int c) {
    float top = x.v[0], low = x.v[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
      top = larger(top, x.v[j]);
      low = smaller(low, x.v[j]);
      if (j & 1) nan |= __builtin_isunordered(x.v[j - 1], x.v[j]);
    }
    if (top > high) {
      high = top;
      from = c;
    }
    if (__any(low == -inf)) {  // masked logits, or the row's end
#pragma unroll
      for (int j = 0; j < 8; ++j) least = x.v[j] == -inf ? least : smaller(least, x.v[j]);
    } else {
      least = smaller(least, low);
    }
  }, [] { return true; });
  // the place itself is asked for where it is the token: a lane's tokens come in ascending order
  int where = -1;
  if (!(a.temperature.of(r) > 0.0) && from >= 0) {
    Chunk<DT> x;
    x.load(a, row, from);
#pragma unroll
    for (int j = 7; j >= 0; --j) where = x.v[j] == high ? x.at(j) : where;
  }
  const uint64_t best = wave_max(nan ? ~0ull : place_of(high, where));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) least = fminf(least, __shfl_xor(least, d));
  if (lane == 0) part[wave] = Part{best, least, 0u};
  if (sp.filters) {
    for (int b = g * SLICE_T + threadIdx.x; b < NBINS; b += sp.slices * SLICE_T) sp.bins[r * NBINS + b] = 0;
    if (g == 0 && threadIdx.x == 0) {
      sp.state[r].sure = sp.state[r].middle = 0;
      sp.state[r].listed = 0;
    }
  }
  if (g == 0 && threadIdx.x == 0) sp.state[r].arrived[0] = sp.state[r].arrived[1] = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    Part p = part[0];
#pragma unroll
    for (int w = 1; w < SLICE_T / 64; ++w) {
      p.best = max64(p.best, part[w].best);
      p.least = fminf(p.least, part[w].least);
    }
    sp.parts[r * sp.slices + g] = p;
  }
}

// The bin of the weight's cut where there is no top-k: the bins' weights are exact.
__device__ __forceinline__ Cuts find_nucleus(const Row& q, const uint64_t (&v)[BINS_EACH], RowState& state) {
  __shared__ uint64_t wave_total[SLICE_T / 64];
  __shared__ int found;
  constexpr int PER = BINS_EACH;
  uint64_t sum = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) sum += v[j];
  const uint64_t upto = wave_scan(sum);
  if ((threadIdx.x & 63) == 63) wave_total[threadIdx.x >> 6] = upto;
  __syncthreads();
  uint64_t at = upto - sum, total = 0;
#pragma unroll
  for (int w = 0; w < SLICE_T / 64; ++w) {
    if (w < (int)(threadIdx.x >> 6)) at += wave_total[w];
    total += wave_total[w];
  }
  const uint64_t target = nucleus(q.p, total);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (at < target && at + v[j] >= target) {  // one thread's
      found = threadIdx.x * PER + j;
      state.before = at;
      state.total = total;
    }
    at += v[j];
  }
  __syncthreads();
  Cuts c;
  c.lo = c.hi = found;
  c.kb = NBINS;
  c.slow = 0;
  c.before_lo = found ? 1 : 0;  // (whether the first of the order is before it)
  c.before_kb = 0;
  c.in_range = LIST;
  c.pad = 0;
  return c;
}

// The cuts' bins from the row's histogram with top-k, by all threads of a workgroup.
__device__ __forceinline__ Cuts find_cuts(const Row& q, int vocab, const uint64_t (&v)[BINS_EACH]) {
  __shared__ uint64_t wave_total[SLICE_T / 64];
  __shared__ int found[6];  // kb, lo, hi, tokens before kb, before lo, up to and with hi
  __shared__ uint64_t weights[2];  // before kb, up to and with it
  constexpr int PER = BINS_EACH;
  constexpr uint64_t WEIGHT = (1ull << COUNT_SHIFT) - 1;
  uint64_t sum = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) sum += v[j];
  const uint64_t upto = wave_scan(sum);
  if ((threadIdx.x & 63) == 63) wave_total[threadIdx.x >> 6] = upto;
  if (threadIdx.x == 0) found[1] = found[2] = FAR_BIN - 1;
  __syncthreads();
  uint64_t before = upto - sum, total = 0;
#pragma unroll
  for (int w = 0; w < SLICE_T / 64; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += wave_total[w];
    total += wave_total[w];
  }
  uint64_t up = before;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint64_t next = up + v[j];
    if ((int)(up >> COUNT_SHIFT) < q.k && (int)(next >> COUNT_SHIFT) >= q.k) {  // one thread's: 0 < k < the bins' tokens
      found[0] = threadIdx.x * PER + j;
      found[3] = (int)(up >> COUNT_SHIFT);
      weights[0] = up & WEIGHT;
      weights[1] = next & WEIGHT;
    }
    up = next;
  }
  __syncthreads();
  Cuts c;
  c.kb = found[0];
  c.before_kb = found[3];
  if (q.p < 1.0) {
    // a sum of bins is off by half a unit a token, and by 2^-16 of it (the exponential and its argument in fp32)
    const double off = 0.5 * vocab + 1.0 + ldexp((double)(total & WEIGHT), -16);
    const double least = q.p * ((double)weights[0] - off) - off, most = q.p * ((double)weights[1] + off) + off;
    uint64_t at = before;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint64_t next = at + v[j];
      const int b = threadIdx.x * PER + j;
      const double w0 = (double)(at & WEIGHT), w1 = (double)(next & WEIGHT);
      if (w1 >= least && (w0 < least || b == 0) && b < FAR_BIN) found[1] = b;
      if (w1 >= most && w0 < most && b < FAR_BIN) found[2] = b;
      at = next;
    }
    __syncthreads();
    c.lo = found[1] < c.kb ? found[1] : c.kb;
    c.hi = found[2] < c.kb ? found[2] : c.kb;
    if (c.hi < c.lo) c.hi = c.lo;  // (equal bounds met in bins of no tokens)
  } else {
    c.lo = c.hi = c.kb;
  }
  if (c.kb == FAR_BIN) {  // tokens of no weight are not told apart
    c.kb = NBINS;
    if (c.lo == FAR_BIN) c.hi = FAR_BIN - 1;
  }
  __syncthreads();
  uint64_t at = before;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int b = threadIdx.x * PER + j;
    if (b == c.lo) found[4] = (int)(at >> COUNT_SHIFT);
    at += v[j];
    if (b == c.hi) found[5] = (int)(at >> COUNT_SHIFT);
    if (b == c.kb) found[0] = (int)(v[j] >> COUNT_SHIFT);
  }
  __syncthreads();
  c.before_lo = found[4];
  c.in_range = c.hi >= c.lo ? found[5] - found[4] : 0;
  c.slow = c.in_range + (c.kb < NBINS && c.kb > c.hi ? found[0] : 0) > LIST;
  c.pad = 0;
  return c;
}

template <int DT>
__global__ __launch_bounds__(SLICE_T) void histogram_kernel(const Args a, const Split sp) {
  __shared__ unsigned long long bins[NBINS];
  const int64_t r = blockIdx.x / sp.slices;
  const int g = (int)(blockIdx.x - r * sp.slices), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char* row = a.logits + r * a.ld;
  const int end = min((g + 1) * sp.per, sp.chunks);
  Row q;
  uint64_t far = 0;
  bool run = false;
  for_chunks<DT, 2>(
      a, row, g * sp.per + wave, end,
      [&](const Chunk<DT>& x, int) {
        int b[8];
        float d[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          d[j] = down(q, x.v[j]);
          b[j] = bin_of(q, d[j]);
        }
        if (q.k > 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t w = (uint32_t)rintf(__builtin_amdgcn_exp2f(d[j] * q.to_exp) * BIN_WEIGHT);
            if (b[j] != FAR_BIN) atomicAdd(&bins[b[j]], 1ull << COUNT_SHIFT | w);
            else far += x.there(j) ? 1 : 0;
          }
        } else {
          double w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = q.sc.weight(x.v[j]);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (b[j] != FAR_BIN) atomicAdd(&bins[b[j]], (unsigned long long)units(w[j]));
        }
      },
      [&] {
        for (int b = threadIdx.x; b < NBINS; b += SLICE_T) bins[b] = 0;
        q = row_of(a, sp, r);
        run = !q.none && !q.greedy && q.cuts();
        __syncthreads();
        return run;
      });
  if (!run) return;
  if (q.k > 0) {
    far = wave_sum(far);
    if (lane == 0 && far) atomicAdd(&bins[FAR_BIN], (unsigned long long)far << COUNT_SHIFT);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < NBINS; b += SLICE_T)
    if (bins[b]) atomicAdd(&sp.bins[r * NBINS + b], bins[b]);
  RowState& state = sp.state[r];
  if (!last_of(&state.arrived[0], sp.slices)) return;
  uint64_t v[BINS_EACH];
#pragma unroll
  for (int j = 0; j < BINS_EACH; ++j) v[j] = shared_load(&sp.bins[r * NBINS + threadIdx.x * BINS_EACH + j]);
  const Cuts c = q.k > 0 ? find_cuts(q, a.vocab, v) : find_nucleus(q, v, state);
  if (threadIdx.x == 0) state.cuts = c;
}

// n <= T / 2 places, largest first: each one's rank is counted by a group of lanes.
// (A step of the sort below waits for LDS twice, 0.15 us: 256 places 6 us, so 1.5.)
__device__ __forceinline__ void rank_down(unsigned long long* v, int n, int up) {
  const int lanes = T / up < 64 ? T / up : 64;  // of a group, a power of two as `up` >= n
  const int e = (int)threadIdx.x / lanes;
  __syncthreads();
  const unsigned long long mine = e < n ? v[e] : 0ull;
  int rank = 0;
#pragma unroll 8
  for (int j = (int)threadIdx.x % lanes; j < n; j += lanes) rank += v[j] > mine ? 1 : 0;
  for (int d = 1; d < lanes; d <<= 1) rank += __shfl_xor(rank, d);
  __syncthreads();
  if (e < n && (int)threadIdx.x % lanes == 0) v[rank] = mine;
  __syncthreads();
}

// n (a power of two) places, largest first.
__device__ __forceinline__ void sort_down(unsigned long long* v, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      // pairs up to 64 apart lie in a wave's own 128 places: its accesses to LDS stay in order
      if (step > 64 || (step == 64 && size > 128) || size == 2) __syncthreads();
      __builtin_amdgcn_wave_barrier();
      for (int i = threadIdx.x; i < n / 2; i += T) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const bool down = !(lo & size);
        const unsigned long long x = v[lo], y = v[hi];
        if ((x < y) == down) {
          v[lo] = y;
          v[hi] = x;
        }
      }
    }
  __syncthreads();
}

union DrawShared {
  Shared s;
  struct {
    unsigned long long list[LIST];
    unsigned long long chunk[CHUNKS];
    uint64_t part[T / 64];
    uint64_t found[4];
    unsigned long long last;
  } d;
};

// A row's token, from what its workgroups left.
template <int DT>
__device__ __forceinline__ void draw(const Args& a, const Split& sp, int64_t r, const Row& q, const Cuts& c, DrawShared& u) {
  auto& d = u.d;
  RowState* const state = sp.state + r;
  const bool cuts = q.cuts();
  // all on its way at once
  const uint64_t my_chunk = (int)threadIdx.x < sp.chunks ? shared_load(&sp.chunk[r * sp.chunks + threadIdx.x]) : 0;
  const uint64_t my_place = cuts ? shared_load(&sp.list[r * LIST + threadIdx.x]) : 0;  // (of LIST there are, if not all written)
  int listed = 0;
  uint64_t sure = 0, middle = 0, before_lo = 0, total_of = 0;
  if (cuts) {
    listed = (int)min(__hip_atomic_load(&state->listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), (unsigned int)(LIST + 1));
    sure = shared_load(&state->sure);
    middle = shared_load(&state->middle);
    before_lo = state->before;
    total_of = state->total;
  }
  const double number = (double)a.uniform[r];
  uint64_t last = 0;    // the place of the last token kept, or none of the list is
  bool any = false;
  if (c.slow || listed > LIST) {
    whole_row<DT>(a, r, u.s);
    return;
  }
  d.chunk[threadIdx.x] = my_chunk;
  if (threadIdx.x == 0) d.last = ~0ull;
  auto scan = [&](uint64_t v, uint64_t& before) {
    const uint64_t upto = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) d.part[threadIdx.x >> 6] = upto;
    __syncthreads();
    uint64_t total = 0, below = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
      if (w < (int)(threadIdx.x >> 6)) below += d.part[w];
      total += d.part[w];
    }
    before = below + upto - v;
    return total;
  };
  if (listed) {
    int n = 2;
    while (n < listed) n <<= 1;
    if ((int)threadIdx.x < n) d.list[threadIdx.x] = (int)threadIdx.x < listed ? my_place : 0ull;
    for (int i = threadIdx.x + T; i < n; i += T) d.list[i] = i < listed ? shared_load(&sp.list[r * LIST + i]) : 0ull;
    if (n <= T / 2) rank_down(d.list, listed, n);
    else sort_down(d.list, n);
    // thread t holds places PER t .. in the order
    const int per = n > T ? n / T : 1;
    const int j0 = (int)threadIdx.x * per, j1 = min(j0 + per, listed);
    auto position = [&](int j) { return j < c.in_range ? c.before_lo + j : c.before_kb + j - c.in_range; };
    auto weight = [&](int j) { return q.sc.weight(value_of((uint32_t)(d.list[j] >> 32))); };
    uint64_t sum = 0, before;
#pragma nounroll
    for (int j = j0; j < j1; ++j)
      if (q.k == 0 || position(j) < q.k) sum += units(weight(j));
    const uint64_t allowed = scan(sum, before);
    uint64_t target = ~0ull, at = before;
    if (q.p < 1.0) {
      target = nucleus(q.p, q.k > 0 ? sure + middle + allowed : total_of);
      at += q.k > 0 ? sure : before_lo;
    }
#pragma nounroll
    for (int j = j0; j < j1; ++j) {
      const int pos = position(j);
      const double w = weight(j);
      const uint64_t m = units(w), place = d.list[j];
      const int index = ~(int)(uint32_t)place;
      if (pos == 0 || ((q.k == 0 || pos < q.k) && at < target && (q.p >= 1.0 || j < c.in_range))) {
        atomicMin(&d.last, (unsigned long long)place);
        if (m && w >= q.min_p) atomicAdd(&d.chunk[index / CHUNK], (unsigned long long)m);
      }
      at += m;
    }
    __syncthreads();
    last = d.last;
    any = last != ~0ull;
  }
  auto kept = [&](float v, int i, double w) {
    const bool in = any ? place_of(v, i) >= last : c.lo >= NBINS || bin_of(q, down(q, v)) < c.lo;
    return in && w >= q.min_p;
  };
  uint64_t before;
  if (!listed) __syncthreads();
  const uint64_t mine = d.chunk[threadIdx.x];
  const uint64_t total = scan(mine, before);
  const uint64_t at = drawn_weight(number, total);
  __syncthreads();
  if (mine && before <= at && at < before + mine) {
    d.found[0] = threadIdx.x;
    d.found[1] = before;
  }
  __syncthreads();
  const int i = (int)d.found[0] * CHUNK + (int)threadIdx.x;
  const uint64_t under = d.found[1];
  uint64_t w = 0;
  float v = 0.0f;
  if ((int)threadIdx.x < CHUNK && i < a.vocab) {
    v = logit<DT>(a.logits + r * a.ld, i);
    const double e = q.sc.weight(v);
    if (kept(v, i, e)) w = units(e);
  }
  scan(w, before);
  before += under;
  if (w && before <= at && at < before + w) {
    a.token[r] = i;
    if (a.logprob) a.logprob[r] = logprob_of(q.sc.log2_weight(v), total);
  }
}

template <int DT>
__global__ __launch_bounds__(SLICE_T, 4) void weigh_kernel(const Args a, const Split sp) {
  const int64_t r = blockIdx.x / sp.slices;
  const int g = (int)(blockIdx.x - r * sp.slices), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char* row = a.logits + r * a.ld;
  const int end = min((g + 1) * sp.per, sp.chunks);
  RowState& state = sp.state[r];
  Row q;
  Cuts c{};
  bool cuts = false, run = true, sums = false;
  float lo = 0.0f, hi = 0.0f, kb = 0.0f, min_far_kb = 0.0f;
  uint64_t sure = 0, middle = 0;
  __shared__ DrawShared u;
  __shared__ unsigned long long near[NEAR];
  __shared__ int gathered;
  __shared__ unsigned int base;
  auto list_one = [&](uint64_t place) {
    const unsigned int at = atomicAdd(&state.listed, 1u);
    if (at < LIST) shared_store(&sp.list[r * LIST + at], place);
  };
  if (threadIdx.x == 0) gathered = 0;
  for_chunks<DT, 2>(
      a, row, g * sp.per + wave, end,
      [&](const Chunk<DT>& x, int n) {
        // whether each of this lane's eight is kept for sure, or counts for the total only (what is after the count's bin
        // is dropped; without one, what is after the weight's)
        bool before[8], between[8], some = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          before[j] = true;
          between[j] = false;
        }
        if (cuts) {
          bool listed[8], any = false;
          some = false;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float b = bin_place(q, down(q, x.v[j]));  // compared as it is: the bounds are whole numbers
            before[j] = b < lo;
            listed[j] = ((b >= lo && b < hi) || (b >= kb && b < kb + 1.0f)) && x.there(j);
            between[j] = sums && b >= hi && b < min_far_kb;
            some |= before[j] || between[j];
            any |= listed[j];
          }
          if (__any(any)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (listed[j]) {
                const int at = atomicAdd(&gathered, 1);
                const uint64_t place = place_of(x.v[j], x.at(j));
                if (at < NEAR) near[at] = place;
                else list_one(place);
              }
            }
          }
        }
        uint64_t kept = 0;
        if (__any(some)) {
          // four at a time, without branches: their FMAs fill each other's latency
#pragma unroll
          for (int h = 0; h < 8; h += 4) {
            double w[4];
            if (sums) {
#pragma unroll
              for (int j = 0; j < 4; ++j) w[j] = q.sc.weight(x.v[h + j]);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint64_t m = units(w[j]);
                const bool in = before[h + j];
                sure += in ? m : 0;
                middle += between[h + j] ? m : 0;
                kept += in && w[j] >= q.min_p ? m : 0;
              }
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                w[j] = q.sc.weight(before[h + j] ? x.v[h + j] : -__builtin_inff());
              if (q.min_p > 0.0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = w[j] >= q.min_p ? w[j] : 0.0;
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) kept += raw_units(w[j]);
              kept -= 4 * RAW;
            }
          }
        }
        if (__any(kept != 0)) kept = wave_sum(kept);
        if (lane == 0) shared_store(&sp.chunk[r * sp.chunks + n], kept);
      },
      [&] {
        if (sp.filters) c = state.cuts;  // (on its way beside the slices' maxima)
        q = row_of(a, sp, r);
        __syncthreads();  // (`gathered` is 0)
        run = !q.none && !q.greedy;
        if (!run) return false;
        cuts = q.cuts();
        sums = q.k > 0 && q.p < 1.0;
        if (!cuts) {
          c.slow = 0;
          c.lo = NBINS;
        } else {
          run = !c.slow;
          lo = (float)c.lo;
          hi = (float)(c.hi + 1);
          kb = (float)c.kb;
          min_far_kb = fminf(kb, (float)FAR_BIN);
        }
        return run;
      });
  if (q.none || q.greedy) {
    if (g == 0 && threadIdx.x == 0) {
      a.token[r] = q.none ? -1 : q.first;
      if (a.logprob) a.logprob[r] = q.none ? __builtin_nanf("") : 0.0f;
    }
    return;
  }
  if (run && cuts) {
    __syncthreads();
    const int here = min(gathered, NEAR);
    if (here) {
      if (threadIdx.x == 0) base = atomicAdd(&state.listed, (unsigned int)here);
      __syncthreads();
      for (int i = threadIdx.x; i < here; i += SLICE_T)
        if (base + i < LIST) shared_store(&sp.list[r * LIST + base + i], near[i]);
    }
    if (sums) {
      sure = wave_sum(sure);
      middle = wave_sum(middle);
      if (lane == 0) {
        if (sure) atomicAdd(&state.sure, (unsigned long long)sure);
        if (middle) atomicAdd(&state.middle, (unsigned long long)middle);
      }
    }
  }
  if (last_of(&state.arrived[1], sp.slices)) draw<DT>(a, sp, r, q, c, u);
}

// Rows of at most this many tokens take one workgroup and launch.  One row, us so and in slices: 1024 tokens without
// filters 11, 15, with top-k 12, 21, with both 17, 23; 4096 11, 15, with top-k 16, 22, with both 25, 23; 2048 rows of
// 4096 34, 40, 81, 103, 131, 111.
constexpr int WHOLE_VOCAB = 4096;

// Rows of one set of launches, each set after the last one in the same workspace: 49 KiB a row of it.
constexpr int64_t MOST_ROWS = 8192;

struct Plan {
  int chunks, per, slices;
  int64_t parts, bins, state, chunk, list, bytes;  // offsets of the workspace's pieces
};

// Slices of a row: two workgroups a CU in all (64 rows of 129280 54 us, 256 of 65536 35; with half as many 60 and 41,
// with twice as many 61 and 40), and a chunk a wave at least.
static Plan plan(int64_t rows, int64_t vocab, bool filters) {
  Plan p{};
  p.chunks = (int)((vocab + CHUNK - 1) / CHUNK);
  const int waves = SLICE_T / 64;
  const int64_t all = 4096 / waves, most = all / rows < 1 ? 1 : all / rows;
  int64_t slices = (p.chunks + waves - 1) / waves;
  if (slices > most) slices = most;
  p.per = (int)((p.chunks + slices - 1) / slices);
  p.per = (p.per + waves - 1) / waves * waves;
  p.slices = (p.chunks + p.per - 1) / p.per;
  int64_t at = 0;
  auto take = [&](int64_t n) {
    const int64_t was = at;
    at += (n + 255) & ~(int64_t)255;
    return was;
  };
  p.parts = take(rows * p.slices * (int64_t)sizeof(Part));
  p.chunk = take(rows * p.chunks * 8);
  p.state = take(rows * (int64_t)sizeof(RowState));
  p.bins = take(filters ? rows * NBINS * 8 : 0);
  p.list = take(filters ? rows * LIST * 8 : 0);
  p.bytes = at;
  return p;
}

template <int DT>
static hipError_t launch(const Args& a, int64_t rows, bool filters, char* ws, hipStream_t st) {
  if (!ws) {
    row_kernel<DT><<<(unsigned)rows, T, 0, st>>>(a);
    return hipGetLastError();
  }
  if (rows > MOST_ROWS) {
    for (int64_t r = 0; r < rows; r += MOST_ROWS) {
      Args b = a;
      b.logits += r * a.ld;
      b.uniform += r;
      if (a.temperature.rows) b.temperature.rows += r;
      if (a.top_p.rows) b.top_p.rows += r;
      if (a.min_p.rows) b.min_p.rows += r;
      if (a.k_rows) b.k_rows += r;
      b.token += r;
      if (a.logprob) b.logprob += r;
      const hipError_t e = launch<DT>(b, rows - r < MOST_ROWS ? rows - r : MOST_ROWS, filters, ws, st);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  const Plan p = plan(rows, a.vocab, filters);
  const Split sp{(Part*)(ws + p.parts),
                 (unsigned long long*)(ws + p.bins),
                 (RowState*)(ws + p.state),
                 (unsigned long long*)(ws + p.chunk),
                 (unsigned long long*)(ws + p.list),
                 p.slices,
                 p.per,
                 p.chunks,
                 filters};
  const unsigned grid = (unsigned)(rows * p.slices);
  stats_kernel<DT><<<grid, SLICE_T, 0, st>>>(a, sp);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && filters) {
    histogram_kernel<DT><<<grid, SLICE_T, 0, st>>>(a, sp);
    e = hipGetLastError();
  }
  if (e == hipSuccess) {
    weigh_kernel<DT><<<grid, SLICE_T, 0, st>>>(a, sp);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace sample
}  // namespace kq

using namespace kq;

extern "C" int64_t kq_sample_tokens_workspace_size(int64_t rows, int64_t vocab, int filters) {
  if (rows < 0 || vocab < 1 || vocab > sample::MAX_VOCAB) return -1;
  if (rows == 0 || vocab <= sample::WHOLE_VOCAB) return 0;
  return sample::plan(rows < sample::MOST_ROWS ? rows : sample::MOST_ROWS, vocab, filters != 0).bytes;
}

extern "C" int kq_sample_tokens(int dtype, const void* logits, int64_t ld, int64_t rows, int64_t vocab, const float* uniform,
                                const float* temperature_rows, double temperature, const int* top_k_rows, int64_t top_k,
                                const float* top_p_rows, double top_p, const float* min_p_rows, double min_p,
                                int64_t* tokens, float* logprobs, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "kq_sample_tokens";
  if (dtype != KQ_DT_BF16 && dtype != KQ_DT_F16 && dtype != KQ_DT_F32)
    return kq_fail(KQ_ERR_INVALID, "%s: dtype must be bf16, f16 or f32", fn);
  if (rows < 0 || vocab < 1 || ld < vocab)
    return kq_fail(KQ_ERR_INVALID, "%s: need rows >= 0, vocab >= 1, a row stride of at least vocab (rows=%lld vocab=%lld ld=%lld)",
                   fn, (long long)rows, (long long)vocab, (long long)ld);
  if (vocab > sample::MAX_VOCAB || rows > (1 << 20))
    return kq_fail(KQ_ERR_LIMIT, "%s: at most %d tokens in the vocabulary and 2^20 rows", fn, sample::MAX_VOCAB);
  if (rows == 0) return KQ_OK;
  if (!logits || !uniform || !tokens) return kq_fail(KQ_ERR_INVALID, "%s: null buffer", fn);
  const int es = dtype == KQ_DT_F32 ? 4 : 2;
  if (kq_misaligned(logits, es) || kq_misaligned(uniform, 4) || kq_misaligned(tokens, 8) || kq_misaligned(logprobs, 4) ||
      kq_misaligned(temperature_rows, 4) || kq_misaligned(top_k_rows, 4) || kq_misaligned(top_p_rows, 4) ||
      kq_misaligned(min_p_rows, 4) || kq_misaligned(workspace, 16))
    return kq_fail(KQ_ERR_INVALID, "%s: buffers must be aligned to their type, the workspace 16", fn);
  const bool filters = top_k_rows || top_k > 0 || top_p_rows || top_p < 1.0;
  const int64_t need = kq_sample_tokens_workspace_size(rows, vocab, filters);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return kq_fail(KQ_ERR_INVALID, "%s: workspace needs %lld bytes", fn, (long long)need);
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
  char* ws = need > 0 ? (char*)workspace : nullptr;
  const hipError_t e = dtype == KQ_DT_BF16  ? sample::launch<KQ_DT_BF16>(a, rows, filters, ws, st)
                       : dtype == KQ_DT_F16 ? sample::launch<KQ_DT_F16>(a, rows, filters, ws, st)
                                            : sample::launch<KQ_DT_F32>(a, rows, filters, ws, st);
  return kq_check_launch(e, fn);
}
