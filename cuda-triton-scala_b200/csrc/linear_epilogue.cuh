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
  int out_f32;     // (CUDA cores; the tensor-core kernels have it as a template parameter)
  int act;
  int vec;         // out and residual rows take 4-feature vectors (8 bytes bf16, 16 fp32)
  int vec2;        // out and residual rows take bf16 pairs (4 bytes)
};

// The activations.  GELU is the same for both output types, a few units of 2^-24 of the result on
// both sides; a shorter polynomial with an absolute error (Abramowitz and Stegun 7.1.26) left
// bf16 outputs 1 % of themselves off at v = -8 and gained 1 % of the time of 4096 x 4096 x 11008.
//
// SiLU and the tanh form of GELU come in two forms.  FULL, for fp32 outputs, keeps to a few units
// of 2^-24 too.  Branch-free from the functions below: 6001 rows over 64 experts of 1544 x 2048
// with the tanh form take 120 us (118 with the short form; 147 with expf and IEEE quotients,
// whose special cases keep the 16 values of a chunk from overlapping).  Short, for bf16 outputs:
// the fast exponential (2 + 1.17 |v| ulp) and the fast quotient (2 ulp), far below a bf16
// step: expf and IEEE quotients made the gated layer at 8192 x 28672 x 4096 int8 28 % slower than
// the same layer without an activation.  __fdividef gives 0 where 1 + exp(-v) passes 2^126,
// which is the limit there.

// 2^x and 1 / x within 2^-22 and 2^-23 of themselves, where the argument and the result are
// normal numbers: one instruction each, without the handling of the rest.
__device__ __forceinline__ float exp2_normal(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float recip_normal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp(x + y) for x < 87, y a correction of x below its last place; below -87 it is exp(-87).
// x log2(e) is taken in two pieces, the product and what its rounding lost (log2(e) in two
// floats): 2^(h + l) = 2^h (1 + l ln 2) but for l^2 / 4 < 2^-36.
__device__ __forceinline__ float exp_full(float x, float y = 0.f) {
  constexpr float L = 1.4426950408889634f, L2 = (float)(1.4426950408889634 - (double)L);
  x = fmaxf(x, -87.f);
  const float h = __fmul_rn(x, L);
  float l = fmaf(x, L2, fmaf(x, L, -h));
  l = fmaf(y, L, l);
  const float p = exp2_normal(h);
  return fmaf(p, l * 0.69314718055994531f, p);
}

// v / (1 + exp(x)): the quotient by an approximate reciprocal and one step of iterative
// refinement.  x >= 87 (the reciprocal leaves the normal numbers soon after): 0 with v's sign, the
// limit, at most 1.5e-36 away (NaN where v is infinite); a divisor of one leaves v, infinite or
// not.
__device__ __forceinline__ float over_one_plus_exp(float v, float x) {
  const float d = 1.f + exp_full(x);
  const float r = recip_normal(d), q0 = __fmul_rn(v, r);
  const float q = fmaf(fmaf(-q0, d, v), r, q0);
  return d == 1.f ? v : (x >= 87.f ? 0.f * v : q);
}

// max(v, 0) - 0.5 |v| erfc(|v| / sqrt 2), erfc = exp(-v^2 / 2) t P(t), t = 1 / (1 + 0.35 |v|): P of
// degree 8 fitted to the minimax of the relative error over |v| <= 13.2 (3.2e-8); beyond, the
// second term is below the normal numbers.  v^2 / 2 enters with what its rounding lost.
__device__ __forceinline__ float gelu(float v) {
  const float a = fminf(fabsf(v), 13.2f), m = 0.5f * a, s = __fmul_rn(m, a);
  const float d = fmaf(0.35f, a, 1.f), t0 = recip_normal(d);
  const float t = fmaf(t0, fmaf(-d, t0, 1.f), t0);  // one step of Newton's
  float p = -0.058218326f;
  p = fmaf(p, t, 0.28757864f);
  p = fmaf(p, t, -0.5106589f);
  p = fmaf(p, t, 0.31744885f);
  p = fmaf(p, t, -0.045584686f);
  p = fmaf(p, t, 0.21073967f);
  p = fmaf(p, t, 0.23973787f);
  p = fmaf(p, t, 0.27971345f);
  p = fmaf(p, t, 0.2792434f);
  const float y = fmaf(-m, p * t * exp_full(-s, -fmaf(m, a, -s)), fmaxf(v, 0.f));
  return v != v ? v : y;
}

template <bool FULL>
__device__ __forceinline__ float activate(int act, float v) {
  switch (act) {
    case QGEMM_ACT_RELU: return v > 0.f ? v : (v != v ? v : 0.f);
    case QGEMM_ACT_GELU: return gelu(v);
    case QGEMM_ACT_GELU_TANH: {  // 0.5 v (1 + tanh u) = v / (1 + exp(-2 u))
      const float u = 0.79788456080286536f * (v + 0.044715f * v * v * v);
      return FULL ? over_one_plus_exp(v, -2.f * u) : __fdividef(v, 1.f + __expf(-2.f * u));
    }
    case QGEMM_ACT_SILU:
      return FULL ? over_one_plus_exp(v, -v) : __fdividef(v, 1.f + __expf(-v));
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
