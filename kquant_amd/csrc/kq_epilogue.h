// The linear's epilogue: c = act(x W^T + bias) + residual, in fp32 on the
// accumulated product and rounded once.
//
// The activations fall in three classes, so that a kernel whose epilogue is
// unrolled over its accumulators needs three forms and no branch per element:
//   none, relu       x below `low` becomes `low` (-inf or 0; NaN stays)
//   silu, gelu_tanh  x sigmoid(x (c1 + c3 x^2)): c = (1, 0), or (2 sqrt(2/pi),
//                    0.044715 times that), since (1 + tanh u) / 2 = sigmoid(2u)
//   gelu             x Phi(x), Phi by the rational-exponential approximation of
//                    Abramowitz and Stegun 7.1.26 for erf (|error| <= 1.5e-7)
#pragma once

#include "kq_act.h"
#include "kq_common.h"

namespace kq {

enum { EPI_OFF = 0, EPI_CLAMP = 1, EPI_SIGMOID = 2, EPI_ERF = 3 };

struct Epilogue {
  int kind;              // EPI_*
  float low, c1, c3;
  const void* bias;      // [n] or null
  int bias_f32;
  const void* residual;  // [m, n] of the output's type, or null
  int64_t ldr;
  int quads;             // bf16 results of 8-byte aligned groups of 4 columns (n, ldc, ldr, c, residual)
};

// Instead of storing the results, the softmax of the rows: part[row][column /
// 16] = (maximum, sum of exp(z - maximum)) of 16 columns, parts = ceil(n / 16),
// and z_target[row] = z[row][target[row]] where the target is a column.
struct LossTail {
  const int64_t* target;
  float2_t* part;
  int64_t parts;
  float* z_target;
};

template <int KIND>
__device__ __forceinline__ float epi_activate(const Epilogue& e, float x) {
  if (KIND == EPI_CLAMP) return x < e.low ? e.low : x;
  // arguments end where the sigmoid is 0 or 1 and the exponential 0: exp_act of an infinity is NaN
  if (KIND == EPI_SIGMOID) {
    const float s = x * fmaf(e.c3, fminf(x * x, 1e30f), e.c1);
    return x * sigmoid_act(fminf(fmaxf(s, -200.0f), 200.0f));
  }
  if (KIND == EPI_ERF) {
    const float a = fabsf(x) * 0.70710678f;
    const float t = rcp_act(fmaf(0.3275911f, a, 1.0f));
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    const float tail = 0.5f * p * t * exp_act(-fminf(a * a, 200.0f));  // (1 - erf(|x| / sqrt 2)) / 2
    return x * (x < 0.0f ? tail : 1.0f - tail);
  }
  return x;
}

// The same for results in 16 bits: the hardware's exponential and reciprocal as
// they are (a few 2^-24 of |x|; epi_activate corrects the exponential's argument).
template <int KIND>
__device__ __forceinline__ float epi_activate16(const Epilogue& e, float x) {
  if (KIND == EPI_SIGMOID) {
    constexpr float L2E = -1.44269502f;
    const float t = x * fmaf(e.c3 * L2E, fminf(x * x, 1e30f), e.c1 * L2E);
    return x * rcp_act(1.0f + __builtin_amdgcn_exp2f(t));
  }
  if (KIND == EPI_ERF) {  // as epi_activate
    const float a = fabsf(x) * 0.70710678f;
    const float t = rcp_act(fmaf(0.3275911f, a, 1.0f));
    float p = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
    p = fmaf(p, t, 0.5f * 1.421413741f);
    p = fmaf(p, t, 0.5f * -0.284496736f);
    p = fmaf(p, t, 0.5f * 0.254829592f);
    const float tail = p * t * __builtin_amdgcn_exp2f(-1.44269502f * fminf(a * a, 200.0f));
    return x * (x < 0.0f ? tail : 1.0f - tail);
  }
  return epi_activate<KIND>(e, x);
}

// the class decided at run time
__device__ __forceinline__ float epi_activate_any(const Epilogue& e, float x) {
  return e.kind == EPI_SIGMOID ? epi_activate<EPI_SIGMOID>(e, x)
         : e.kind == EPI_ERF   ? epi_activate<EPI_ERF>(e, x)
                               : epi_activate<EPI_CLAMP>(e, x);
}

// Bits as loaded (0 where there is none) and their value, apart, so that a load can be on its way for long.
__device__ __forceinline__ uint32_t epi_bias_bits(const Epilogue& e, int64_t n) {
  if (!e.bias) return 0u;
  return e.bias_f32 ? static_cast<const uint32_t*>(e.bias)[n] : static_cast<const uint16_t*>(e.bias)[n];
}
__device__ __forceinline__ float epi_bias_value(const Epilogue& e, uint32_t bits) {
  return __uint_as_float(e.bias_f32 ? bits : bits << 16);
}
__device__ __forceinline__ float epi_bias(const Epilogue& e, int64_t n) { return epi_bias_value(e, epi_bias_bits(e, n)); }

// OUT: the output's and so the residual's type (KQ_DT_BF16 or KQ_DT_F32; of int8 products KQ_DT_F16 too).
template <int OUT>
__device__ __forceinline__ uint32_t epi_residual_bits(const Epilogue& e, int64_t m, int64_t n) {
  if (!e.residual) return 0u;
  const int64_t at = m * e.ldr + n;
  return OUT == KQ_DT_F32 ? static_cast<const uint32_t*>(e.residual)[at] : static_cast<const uint16_t*>(e.residual)[at];
}
template <int OUT>
__device__ __forceinline__ float epi_residual_value(uint32_t bits) {
  if (OUT == KQ_DT_F16) return f16_bits_to_f32(bits);
  return __uint_as_float(OUT == KQ_DT_F32 ? bits : bits << 16);
}
template <int OUT>
__device__ __forceinline__ float epi_residual(const Epilogue& e, int64_t m, int64_t n) {
  return epi_residual_value<OUT>(epi_residual_bits<OUT>(e, m, n));
}

// The value at (m, n) of the matrix from its accumulated product.
template <int OUT>
__device__ __forceinline__ float epi_apply(const Epilogue& e, float x, int64_t m, int64_t n) {
  return epi_activate_any(e, x + epi_bias(e, n)) + epi_residual<OUT>(e, m, n);
}

// The activation's class and constants (KQ_LIN_*).
static inline Epilogue make_epilogue(int activation) {
  Epilogue e{};
  e.kind = activation == KQ_LIN_GELU                                     ? EPI_ERF
           : activation == KQ_LIN_SILU || activation == KQ_LIN_GELU_TANH ? EPI_SIGMOID
                                                                         : EPI_CLAMP;
  e.low = activation == KQ_LIN_RELU ? 0.0f : -__builtin_inff();
  constexpr double C = 1.5957691216057308;  // 2 sqrt(2 / pi)
  e.c1 = activation == KQ_LIN_GELU_TANH ? (float)C : 1.0f;
  e.c3 = activation == KQ_LIN_GELU_TANH ? (float)(0.044715 * C) : 0.0f;
  return e;
}

// The epilogue of the rows from m0 and the columns from n0 on.
template <int OUT>
static inline Epilogue epi_at(Epilogue e, int64_t m0, int64_t n0) {
  if (e.bias) e.bias = static_cast<const char*>(e.bias) + n0 * (e.bias_f32 ? 4 : 2);
  if (e.residual) e.residual = static_cast<const char*>(e.residual) + (m0 * e.ldr + n0) * (OUT == KQ_DT_F32 ? 4 : 2);
  return e;
}

}  // namespace kq
