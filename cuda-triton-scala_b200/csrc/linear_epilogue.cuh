// linear_epilogue.cuh -- what follows the products of a linear layer, for the SIMT and the
// tensor-core kernels: dequantisation, bias, activation, gate, residual and the one rounding
// to the output type.
//     z = float(acc) * sw[n] * sx[m]   (int8: two roundings, in that order)   or the fp32 sum
//     v = act(z + bias[n]);  gated: v = act(z_gate + b_gate) * (z_up + b_up)
//     y = round(v + residual[m, n])
// Everything up to the last line is fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "internal.h"

namespace qg {
namespace lin {

struct Epi {
  const float* sx;
  const float* sw;
  const float* bias;
  const void* residual;
  void* out;
  long long ldr, ldc;
  int N, nw;       // features, weight rows of one expert (N or 2 N)
  int out_f32;
  int act;
  int vec;         // out and residual rows take 4-feature vectors (8 bytes bf16, 16 fp32)
  int vec2;        // out and residual rows take bf16 pairs (4 bytes)
};

// SiLU and the tanh form of GELU through the fast exponential (2 + 1.17 |v| ulp) and the fast quotient (2 ulp), far below
// a bf16 step: the full-precision ones made the gated layer at 8192 x 28672 x 4096 int8 28 %
// slower than the same layer without an activation.  __fdividef gives 0 where 1 + exp(-v)
// passes 2^126, which is the limit there.
// GELU is max(v, 0) - 0.5 |v| erfc(|v| / sqrt 2), erfc(x) = exp(-x^2) P(1 / (1 + p x)) with the
// degree-5 P of Abramowitz and Stegun 7.1.26 (absolute error 1.5e-7, and no cancellation for
// negative v, where 1 + erf loses the small result); about half of erff's instructions, which
// the last tile's epilogue exposes.
__device__ __forceinline__ float gelu(float v) {
  const float a = fminf(fabsf(v), 30.f);  // exp(-a^2 / 2) is 0 from 15 on
  const float t = __fdividef(1.f, fmaf(0.3275911f * 0.70710678118654752f, a, 1.f));
  const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f),
                                   -0.284496736f), 0.254829592f);
  const float y = fmaxf(v, 0.f) - 0.5f * a * p * __expf(-0.5f * a * a);
  return v != v ? v : y;
}

__device__ __forceinline__ float activate(int act, float v) {
  switch (act) {
    case QGEMM_ACT_RELU: return v > 0.f ? v : (v != v ? v : 0.f);
    case QGEMM_ACT_GELU: return gelu(v);
    case QGEMM_ACT_GELU_TANH: {  // 0.5 v (1 + tanh u) = v / (1 + exp(-2 u))
      const float u = 0.79788456080286536f * (v + 0.044715f * v * v * v);
      return __fdividef(v, 1.f + __expf(-2.f * u));
    }
    case QGEMM_ACT_SILU: return __fdividef(v, 1.f + __expf(-v));
    default: return v;
  }
}

template <int KIND>
__device__ __forceinline__ float dequant(uint32_t word, float sw, float sx) {
  if constexpr (KIND == KIND_I8) return __fmul_rn(__fmul_rn(__int2float_rn((int)word), sw), sx);
  else return __uint_as_float(word);
}

__device__ __forceinline__ float load_out(const void* p, int f32, size_t i) {
  return f32 ? static_cast<const float*>(p)[i]
             : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_out(void* p, int f32, size_t i, float v) {
  if (f32) static_cast<float*>(p)[i] = v;
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

}  // namespace lin
}  // namespace qg
