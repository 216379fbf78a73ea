// linear_simt.cu -- the linear layers of linear_tcgen05.cu on CUDA cores: any K, any
// alignment, and the independent check of the tensor-core kernels (QGEMM_ALGO_SIMT).
//
// One block of 256 threads per 32 rows x 32 features of one expert, 32-deep tiles of x and w
// in shared memory, four outputs a thread; sums in int32 (int8 operands) or in fp32 with k
// ascending.  Bound by shared memory and instruction issue, not meant to be fast: shapes that
// the tensor cores take (K a multiple of 16 bytes, 16-byte aligned operands) do not come here
// unless asked for.
#include "linear_epilogue.cuh"

namespace qg {
namespace lin {

constexpr int TM = 32, TN = 32, TK = 32;

template <int KIND> struct Elem;
template <> struct Elem<KIND_I8> {
  using T = int8_t;
  using Acc = int;
  static __device__ __forceinline__ int load(const int8_t* p, size_t i) { return p[i]; }
  static __device__ __forceinline__ int mad(int a, int b, int c) { return a * b + c; }
  static __device__ __forceinline__ uint32_t word(int a) { return (uint32_t)a; }
};
template <> struct Elem<KIND_BF16> {
  using T = __nv_bfloat16;
  using Acc = float;
  static __device__ __forceinline__ float load(const __nv_bfloat16* p, size_t i) {
    return __bfloat162float(p[i]);
  }
  static __device__ __forceinline__ float mad(float a, float b, float c) {
    return __fmaf_rn(a, b, c);
  }
  static __device__ __forceinline__ uint32_t word(float a) { return __float_as_uint(a); }
};

template <int KIND, bool GATED>
__global__ void __launch_bounds__(256)
    linear_simt_kernel(const LinArgs a, Epi ep, long long tiles, int* bad) {
  using El = Elem<KIND>;
  using Acc = typename El::Acc;
  const auto* x = static_cast<const typename El::T*>(a.x);
  const auto* w = static_cast<const typename El::T*>(a.w);
  __shared__ int s_e, s_r0, s_r1;
  __shared__ Acc sx[TK][TM + 1], sg[TK][TN + 1], su[GATED ? TK : 1][TN + 1];
  const int tn = threadIdx.x % 32, tm = threadIdx.x / 32;  // feature tn, rows tm + 8 i
  const int n0 = blockIdx.x * TN, n = n0 + tn;
  for (long long tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
    // the expert and the rows of this tile: row tiles are counted expert by expert
    if (threadIdx.x == 0) {
      s_e = -1;
      if (!a.offsets) {
        if (tile * TM < a.M) { s_e = 0; s_r0 = (int)tile * TM; s_r1 = a.M; }
      } else {
        long long left = tile;
        for (int e = 0; e < a.E; ++e) {
          const int o0 = a.offsets[e], o1 = a.offsets[e + 1];
          if (o0 < 0 || o1 < o0 || o1 > a.M) {
            note_bad_index(bad);
            continue;
          }
          const int tiles = (o1 - o0 + TM - 1) / TM;
          if (left < tiles) {
            s_e = e; s_r0 = o0 + (int)left * TM; s_r1 = o1;
            break;
          }
          left -= tiles;
        }
      }
    }
    __syncthreads();
    const int e = s_e;
    if (e < 0) return;  // `tiles` is a bound where the rows are grouped
    const int r0 = s_r0, r1 = s_r1;
    Acc g[4] = {}, u[4] = {};
    const size_t wbase = (size_t)e * ep.nw;
    for (int k0 = 0; k0 < a.K; k0 += TK) {
      for (int i = threadIdx.x; i < TM * TK; i += 256) {
        const int k = i % TK, r = i / TK;
        sx[k][r] = (k0 + k < a.K && r0 + r < r1)
                       ? El::load(x, (size_t)(r0 + r) * a.ldx + k0 + k) : Acc(0);
        const bool in = k0 + k < a.K && n0 + r < a.N;
        sg[k][r] = in ? El::load(w, (wbase + n0 + r) * a.K + k0 + k) : Acc(0);
        if (GATED) su[k][r] = in ? El::load(w, (wbase + a.N + n0 + r) * a.K + k0 + k) : Acc(0);
      }
      __syncthreads();
#pragma unroll 8
      for (int k = 0; k < TK; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[i] = El::mad(sx[k][tm + 8 * i], sg[k][tn], g[i]);
          if (GATED) u[i] = El::mad(sx[k][tm + 8 * i], su[k][tn], u[i]);
        }
      }
      __syncthreads();
    }
    __syncthreads();  // s_e and the rows are read
    if (n < a.N) {
      const float swg = ep.sw ? ep.sw[wbase + n] : 1.f, bg = ep.bias ? ep.bias[wbase + n] : 0.f;
      const float swu = GATED && ep.sw ? ep.sw[wbase + a.N + n] : 1.f;
      const float bu = GATED && ep.bias ? ep.bias[wbase + a.N + n] : 0.f;
      for (int i = 0; i < 4; ++i) {
        const int row = r0 + tm + 8 * i;
        if (row >= r1) continue;
        const float s = ep.sx ? ep.sx[row] : 1.f;
        float z = dequant<KIND>(El::word(g[i]), swg, s);
        if (ep.bias) z = __fadd_rn(z, bg);
        float v = ep.out_f32 ? activate<true>(ep.act, z) : activate<false>(ep.act, z);
        if (GATED) {
          float zu = dequant<KIND>(El::word(u[i]), swu, s);
          if (ep.bias) zu = __fadd_rn(zu, bu);
          v = __fmul_rn(v, zu);
        }
        if (ep.residual) v = __fadd_rn(v, load_out(ep.residual, ep.out_f32, (size_t)row * ep.ldr + n));
        store_out(ep.out, ep.out_f32, (size_t)row * ep.ldc + n, v);
      }
    }
  }
}

}  // namespace lin

qgemm_status launch_linear_simt(qgemm_stream_s* s, const LinArgs& a) {
  using namespace lin;
  Epi ep = {};
  ep.sx = a.sx; ep.sw = a.sw; ep.bias = a.bias; ep.residual = a.residual; ep.out = a.out;
  ep.ldr = a.ldr; ep.ldc = a.ldc;
  ep.N = a.N; ep.nw = a.gated ? 2 * a.N : a.N;
  ep.out_f32 = a.out_dtype == QGEMM_F32;
  ep.act = a.act;
  // row tiles of ragged groups: at most one partial tile an expert; a grid has 65535 blocks in y
  const long long row_tiles = ((long long)a.M + TM - 1) / TM + (a.offsets ? a.E : 0);
  const dim3 grid((unsigned)(((long long)a.N + TN - 1) / TN),
                  (unsigned)(row_tiles < 65535 ? row_tiles : 65535));
  int* bad = s->index_word;
  if (a.kind == KIND_I8) {
    if (a.gated) linear_simt_kernel<KIND_I8, true><<<grid, 256, 0, s->stream>>>(a, ep, row_tiles, bad);
    else linear_simt_kernel<KIND_I8, false><<<grid, 256, 0, s->stream>>>(a, ep, row_tiles, bad);
  } else {
    if (a.gated) linear_simt_kernel<KIND_BF16, true><<<grid, 256, 0, s->stream>>>(a, ep, row_tiles, bad);
    else linear_simt_kernel<KIND_BF16, false><<<grid, 256, 0, s->stream>>>(a, ep, row_tiles, bad);
  }
  return cuda_fail(cudaGetLastError(), "linear_simt launch");
}

}  // namespace qg
