// route.cu -- tokens to experts and back: top-k routing with the counting sort that groups
// the (token, slot) pairs by expert, dispatch of the token rows into that order (copied or
// quantised to int8), and the weighted combine of the experts' rows.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <mutex>

#include "internal.h"
#include "ptx.cuh"

namespace qg {
namespace route {

constexpr int CLUSTER = 8;          // grouping CTAs of a large call (portable cluster size)

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

// A key that orders like the logit, 0 for what is never chosen (-inf, NaN).  -0 and +0 get one
// key (they are equal, the lower index wins); +inf counts as the largest finite fp32.  A bf16
// logit leaves 16 bits for the (complemented) index, so one warp reduction finds the largest
// and, among equals, the lowest index; fp32 logits need a second one for the index (at 16384
// tokens, 64 experts and k = 8 the reductions are what bounds the kernel).
template <typename T> struct Key;
template <> struct Key<float> {
  static constexpr bool kIndexed = false;
  static __device__ __forceinline__ uint32_t of(float v, int) {
    if (!(v > -INFINITY)) return 0u;
    v = fminf(v, FLT_MAX) + 0.0f;
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
  }
  static __device__ __forceinline__ int index(uint32_t) { return 0; }
};
template <> struct Key<__nv_bfloat16> {
  static constexpr bool kIndexed = true;
  static __device__ __forceinline__ uint32_t of(__nv_bfloat16 x, int e) {
    float v = __bfloat162float(x);
    if (!(v > -INFINITY)) return 0u;
    v += 0.0f;
    const uint32_t b = __float_as_uint(v) >> 16;
    const uint32_t o = (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
    return (o << 16) | (0xffffu - (uint32_t)e);
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    const uint32_t o = key >> 16;
    return fminf(__uint_as_float(((o & 0x8000u) ? (o & 0x7fffu) : (~o & 0xffffu)) << 16), FLT_MAX);
  }
  static __device__ __forceinline__ int index(uint32_t key) { return (int)(0xffffu - (key & 0xffffu)); }
};

// One token by one warp: lane l holds the logits of experts l, l + 32, ...  Each round takes
// the largest key of the warp and retires it; the softmax sum runs over the same registers.
template <typename T, int EPL>
__device__ __forceinline__ void topk_token(const T* __restrict__ logits, int E, int k,
                                           int renormalize, float* __restrict__ weights,
                                           int* __restrict__ experts, int lane) {
  using K = Key<T>;
  uint32_t key[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    key[i] = e < E ? K::of(logits[e], e) : 0u;
  }
  uint32_t best = 0;
  int at = 0;
  auto rescan = [&]() {
    best = 0;
    at = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (key[i] > best) { best = key[i]; at = i; }
  };
  rescan();
  const uint32_t top = __reduce_max_sync(0xffffffffu, best);
  const float most = K::value(top);
  float sum = 0.f;  // over every expert that can be chosen
  if (!renormalize) {
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (key[i]) sum += expf(K::value(key[i]) - most);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  }
  uint32_t won[2] = {0u, 0u};  // keys of slots lane and lane + 32
  int id[2] = {-1, -1};
  for (int j = 0; j < k; ++j) {
    const uint32_t m = j == 0 ? top : __reduce_max_sync(0xffffffffu, best);
    if (m == 0) break;
    const int mine = best == m ? lane + 32 * at : 0x7fffffff;
    const int e = K::kIndexed ? K::index(m) : __reduce_min_sync(0xffffffffu, mine);
    if (mine == e) {
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (i == at) key[i] = 0;
      rescan();
    }
    if ((j & 31) == lane) {
      won[j >> 5] = m;
      id[j >> 5] = e;
    }
  }
  float p[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) p[h] = won[h] ? expf(K::value(won[h]) - most) : 0.f;
  if (renormalize) {
    sum = p[0] + p[1];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (lane + 32 * h < k) {
      weights[lane + 32 * h] = id[h] >= 0 ? p[h] / sum : 0.f;
      experts[lane + 32 * h] = id[h];
    }
}

// Top-k of every token, a warp each, over the whole GPU (large T; route_group_kernel then
// only sorts).
template <typename T, int EPL>
__global__ void __launch_bounds__(256) route_topk_kernel(const T* __restrict__ logits,
                                                         float* __restrict__ weights,
                                                         int* __restrict__ experts, int n, int E,
                                                         int k, int renormalize) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int t = blockIdx.x * 8 + threadIdx.x / 32;
  if (t >= n) return;
  topk_token<T, EPL>(logits + (size_t)t * E, E, k, renormalize, weights + (size_t)t * k,
                     experts + (size_t)t * k, threadIdx.x % 32);
}

// Stable counting sort of the pairs by expert, in one cluster (one CTA for small T), and the
// top-k of the tokens before it when `topk` is set.  Every warp owns a run of consecutive
// tokens, a lane a token at a time.  Counts: every lane adds its pairs to the warp's own row of
// shared memory; the rows are scanned over the warps of the CTA, over the CTAs through
// distributed shared memory, and over the experts.  Positions: a token has an expert once at
// most, so the pairs of an expert among 32 tokens are a bit mask (OR-ed in shared memory), and
// a pair's rank is the number of lower bits.  Integer additions and ORs only, so the result does
// not depend on timing.  (Finding equal experts with match_any instead took 36 us at 131072
// pairs.)
template <typename T, int EPL>
__global__ void __launch_bounds__(1024, 1)
    route_group_kernel(const T* __restrict__ logits, float* __restrict__ weights,
                       int* __restrict__ experts, int* __restrict__ offsets,
                       int* __restrict__ rows, int n, int E, int k, int renormalize, int topk,
                       int csize) {
  extern __shared__ int sh[];
  const int nwarps = blockDim.x / 32;
  int* hist = sh;                                                 // [nwarps][E]
  uint32_t* mask = reinterpret_cast<uint32_t*>(sh + nwarps * E);  // [nwarps][E]
  int* total = sh + 2 * nwarps * E;                               // [E] this CTA's pairs
  int* start = total + E;                                         // [E] first position of the expert
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int cta = blockIdx.x;   // the grid is one cluster
  ptx::grid_launch_dependents();
  for (int i = threadIdx.x; i < 2 * nwarps * E; i += blockDim.x) sh[i] = 0;
  ptx::grid_dependency_wait();
  const int per = (n + csize * nwarps - 1) / (csize * nwarps);
  const long long first = (long long)(cta * nwarps + warp) * per;
  const int t0 = (int)(first < n ? first : n), t1 = (int)(first + per < n ? first + per : n);
  if (topk)
    for (int t = t0; t < t1; ++t)
      topk_token<T, EPL>(logits + (size_t)t * E, E, k, renormalize, weights + (size_t)t * k,
                         experts + (size_t)t * k, lane);
  __syncthreads();
  int* mine = hist + warp * E;
  uint32_t* bits = mask + warp * E;
  // calls fn(slot, expert) for a token's chosen experts, eight slots' loads in flight
  auto each_pair = [&](int t, auto&& fn) {
    for (int j0 = 0; j0 < k; j0 += 8) {
      int ex[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) ex[j] = j0 + j < k ? experts[(size_t)t * k + j0 + j] : -2;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ex[j] > -2) fn(j0 + j, ex[j]);
    }
  };
  for (int t = t0 + lane; t < t1; t += 32)
    each_pair(t, [&](int, int e) { if (e >= 0) atomicAdd(mine + e, 1); });
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < nwarps; ++w) {
      const int c = hist[w * E + e];
      hist[w * E + e] = run;
      run += c;
    }
    total[e] = run;
  }
  if (csize > 1) ptx::cluster_sync_all(); else __syncthreads();
  // all pairs of each expert, and how many of them lie in earlier CTAs
  int before[1024 / 256] = {};  // of experts threadIdx.x, + blockDim.x, ... (at least 256 threads)
#pragma unroll
  for (int i = 0; i < 1024 / 256; ++i) {
    const int e = threadIdx.x + i * blockDim.x;
    if (e >= E) break;
    int all = 0;
    if (csize > 1) {
      const uint32_t here = ptx::smem_u32(total + e);
      for (int c = 0; c < csize; ++c) {
        int v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];"
                     : "=r"(v) : "r"(ptx::map_to_rank(here, c)) : "memory");
        all += v;
        if (c < cta) before[i] += v;
      }
    } else {
      all = total[e];
    }
    start[e] = all;
  }
  __syncthreads();
  if (warp == 0) {  // exclusive scan over the experts
    const int chunk = (E + 31) / 32, e0 = min(E, lane * chunk), e1 = min(E, e0 + chunk);
    int sum = 0;
    for (int e = e0; e < e1; ++e) sum += start[e];
    int run = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += o;
    }
    if (cta == 0 && lane == 31) offsets[E] = run;
    run -= sum;
    for (int e = e0; e < e1; ++e) {
      const int c = start[e];
      start[e] = run;
      if (cta == 0) offsets[e] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 1024 / 256; ++i) {
    const int e = threadIdx.x + i * blockDim.x;
    if (e < E) start[e] += before[i];
  }
  __syncthreads();
  for (int b = t0; b < t1; b += 32) {  // warp-uniform
    const int t = b + lane;
    const bool in = t < t1;
    if (in) each_pair(t, [&](int, int e) { if (e >= 0) atomicOr(bits + e, 1u << lane); });
    __syncwarp();
    if (in)
      each_pair(t, [&](int j, int e) {
        rows[(size_t)t * k + j] =
            e < 0 ? -1 : start[e] + mine[e] + __popc(bits[e] & ((1u << lane) - 1u));
      });
    __syncwarp();
    if (b + 32 < t1)
      for (int e = lane; e < E; e += 32) {
        mine[e] += __popc(bits[e]);
        bits[e] = 0u;
      }
    __syncwarp();
  }
  if (csize > 1) ptx::cluster_sync_all();  // no CTA leaves while another reads its totals
}

// ---- dispatch -----------------------------------------------------------------------

// out[rows[t, j]] = x[t]: each thread holds one piece (16 bytes, or one element) of a token
// row and stores it to the token's k places; x is read once.  Bound by HBM where rows are whole
// pieces (8192 tokens x 2 bf16: K = 4096 32 us, floor 31; K = 4095, an element a thread, 137).
template <typename V>
__global__ void __launch_bounds__(256) dispatch_copy_kernel(const V* __restrict__ x,
                                                            const int* __restrict__ rows,
                                                            V* __restrict__ out, int T, int k,
                                                            int pieces, int R, int* bad) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= pieces) return;
  for (int t = blockIdx.y; t < T; t += gridDim.y) {
    const V v = x[(size_t)t * pieces + c];
    for (int j = 0; j < k; ++j) {
      const int r = __ldg(rows + (size_t)t * k + j);
      if (r >= R) {
        if (c == 0) note_bad_index(bad);
      } else if (r >= 0) {
        out[(size_t)r * pieces + c] = v;
      }
    }
  }
}

__device__ __forceinline__ int8_t quant(float v, float mul) {
  const int q = __float2int_rz(__fmul_rn(v, mul));  // NaN -> 0
  return (int8_t)(q > 127 ? 127 : (q < -128 ? -128 : q));
}

// A token per CTA, quantised once and stored to its k places.  NV > 0: the row is held in
// registers (NV pieces of 4 elements a thread: K % 4 == 0, aligned rows, K <= 8192); NV = 0: any
// row, read once for the maximum and again, and quantised, for each place (8192 tokens x 2 bf16: K =
// 4096 28 us, 4095 46; 8192 58, 8196 77).  maxAbs in the "if (v > m) m = v" form: a NaN never replaces a number.
template <typename T, int NV>
__global__ void __launch_bounds__(256) dispatch_quant_kernel(const T* __restrict__ x,
                                                             const int* __restrict__ rows,
                                                             int8_t* __restrict__ q,
                                                             float* __restrict__ sA, int k, int K,
                                                             int R, int* bad) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int t = blockIdx.x;
  const T* row = x + (size_t)t * K;
  const int tid = threadIdx.x;
  float v[NV > 0 ? NV : 1][4];
  float mx = 0.f;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = tid + 256 * i;
      if (c < K / 4) {
        if constexpr (sizeof(T) == 2) {
          const uint2 u = __ldcs(reinterpret_cast<const uint2*>(row) + c);
          v[i][0] = __uint_as_float(u.x << 16);
          v[i][1] = __uint_as_float(u.x & 0xffff0000u);
          v[i][2] = __uint_as_float(u.y << 16);
          v[i][3] = __uint_as_float(u.y & 0xffff0000u);
        } else {
          const float4 f = __ldcs(reinterpret_cast<const float4*>(row) + c);
          v[i][0] = f.x; v[i][1] = f.y; v[i][2] = f.z; v[i][3] = f.w;
        }
#pragma unroll
        for (int h = 0; h < 4; ++h)
          if (fabsf(v[i][h]) > mx) mx = fabsf(v[i][h]);
      }
    }
  } else {
    for (int i = tid; i < K; i += 256) {
      const float a = fabsf(to_f<T>(row[i]));
      if (a > mx) mx = a;
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, mx, off);
    if (o > mx) mx = o;
  }
  __shared__ float wmax[8];
  if (tid % 32 == 0) wmax[tid / 32] = mx;
  __syncthreads();
  mx = wmax[0];
#pragma unroll
  for (int w = 1; w < 8; ++w)
    if (wmax[w] > mx) mx = wmax[w];
  const float mul = mx > 1e-6f ? __fdiv_rn(127.0f, mx) : 1.0f;
  const float scale = __fdiv_rn(mx, 127.0f);
  uint32_t packed[NV > 0 ? NV : 1];
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (tid + 256 * i >= K / 4) continue;
      uint32_t b = 0;
#pragma unroll
      for (int h = 0; h < 4; ++h) b |= (uint32_t)(uint8_t)quant(v[i][h], mul) << (8 * h);
      packed[i] = b;
    }
  }
  for (int j = 0; j < k; ++j) {
    const int r = __ldg(rows + (size_t)t * k + j);
    if (r < 0) continue;
    if (r >= R) {
      if (tid == 0) note_bad_index(bad);
      continue;
    }
    if (tid == 0) sA[r] = scale;
    int8_t* dst = q + (size_t)r * K;
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = tid + 256 * i;
        if (c < K / 4) reinterpret_cast<uint32_t*>(dst)[c] = packed[i];
      }
    } else {
      for (int i = tid; i < K; i += 256) dst[i] = quant(to_f<T>(row[i]), mul);
    }
  }
}

// ---- combine ------------------------------------------------------------------------

// 8 consecutive elements as fp32 (VEC: one or two 16-byte loads, else element by element
// up to `left`).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, int left, float (&v)[8]) {
  if constexpr (VEC && sizeof(T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else if constexpr (VEC) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f<T>(p[i]) : 0.f;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ p, int left, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (VEC) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int i = 0; i < 8 && i < left; ++i) p[i] = __float2bfloat16_rn(v[i]);
    }
  } else if constexpr (VEC) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    for (int i = 0; i < 8 && i < left; ++i) p[i] = v[i];
  }
}

// out[t] = sum_j w[t, j] y[rows[t, j]] (+ residual[t]): a thread per 8 columns of a token,
// fp32 sums with j ascending.  Bound by HBM: U rows' loads are in flight a thread, as loaded
// (8 rows of bf16: 172 us at 8192 tokens of 8 rows x 4096 with 4 in flight and widened at once, 114
// to 119 this way).  Widths that are not a multiple of 8 go element by element (4095: 201 us).
template <typename TI, typename TO, bool VEC, int U>
__global__ void __launch_bounds__(128) combine_kernel(const TI* __restrict__ y,
                                                      const int* __restrict__ rows,
                                                      const float* __restrict__ weights,
                                                      const TO* residual, TO* out, int T, int k,
                                                      int N, int R, int* bad) {
  constexpr int RAW = VEC ? (int)sizeof(TI) / 2 : 1;  // 16-byte words of 8 elements
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int c = (blockIdx.x * 128 + threadIdx.x) * 8;
  if (c >= N) return;
  const int left = N - c;
  for (int t = blockIdx.y; t < T; t += gridDim.y) {
    float acc[8] = {};
    for (int j0 = 0; j0 < k; j0 += U) {
      uint4 raw[U][RAW];
      float w[U];
      int row[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        row[u] = j0 + u < k ? __ldg(rows + (size_t)t * k + j0 + u) : -1;
        w[u] = weights && j0 + u < k ? __ldg(weights + (size_t)t * k + j0 + u) : 1.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row[u] >= R) {
          if (c == 0) note_bad_index(bad);
          row[u] = -1;
        }
        if constexpr (VEC) {
#pragma unroll
          for (int h = 0; h < RAW; ++h)
            raw[u][h] = row[u] >= 0
                ? __ldcs(reinterpret_cast<const uint4*>(y + (size_t)row[u] * N + c) + h)
                : make_uint4(0u, 0u, 0u, 0u);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row[u] < 0) continue;  // a slot without a row adds nothing, whatever its weight
        float v[8];
        if constexpr (!VEC) {
          load8<TI, false>(y + (size_t)row[u] * N + c, left, v);
        } else if constexpr (sizeof(TI) == 2) {
          const uint32_t q[4] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(q[i] << 16);
            v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
          }
        } else {
#pragma unroll
          for (int h = 0; h < RAW; ++h) {
            v[4 * h] = __uint_as_float(raw[u][h].x);
            v[4 * h + 1] = __uint_as_float(raw[u][h].y);
            v[4 * h + 2] = __uint_as_float(raw[u][h].z);
            v[4 * h + 3] = __uint_as_float(raw[u][h].w);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = __fmaf_rn(w[u], v[i], acc[i]);
      }
    }
    if (residual) {
      float res[8];
      load8<TO, VEC>(residual + (size_t)t * N + c, left, res);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += res[i];
    }
    store8<TO, VEC>(out + (size_t)t * N + c, left, acc);
  }
}

// ---- launches -----------------------------------------------------------------------

// A launch that may start while the previous kernel on the stream ends (every kernel here
// waits for it before it touches memory), in clusters of `cluster` CTAs.
template <typename... P, typename... A>
cudaError_t launch(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                   int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}

// The grouping kernel's shared memory at most: 16 warps' rows of 1024 experts.
constexpr int GROUP_SMEM_MAX = (int)sizeof(int) * (2 * 16 + 2) * kMaxExperts;
static_assert(GROUP_SMEM_MAX >= (int)sizeof(int) * (2 * 32 + 2) * 512, "32 warps up to 512 experts");

// Opts a grouping kernel in to that size, once a device.  The permission belongs to the kernel,
// not to a launch: set to each call's own need, one thread's call could lower it between another
// thread's setting and its launch, which was then refused.
template <typename T, int EPL>
qgemm_status group_smem_opt_in(qgemm_stream_s* s) {
  static std::mutex mu;
  static bool done[64] = {};
  const int ord = s->dev->ordinal;
  if (ord < 0 || ord >= 64) return fail(QGEMM_ERR_UNSUPPORTED, "device ordinal %d >= 64", ord);
  std::lock_guard<std::mutex> lock(mu);
  if (!done[ord]) {
    const cudaError_t e = cudaFuncSetAttribute(
        route_group_kernel<T, EPL>, cudaFuncAttributeMaxDynamicSharedMemorySize, GROUP_SMEM_MAX);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(route_group)");
    done[ord] = true;
  }
  return QGEMM_OK;
}

template <typename T, int EPL>
qgemm_status route_t(qgemm_stream_s* s, const T* logits, float* weights, int* experts,
                     int* offsets, int* rows, int n, int E, int k, int renormalize) {
  // Top-k in the grouping kernel while its CTAs hold the tokens one to a warp; beyond that over
  // the whole GPU first (512 tokens, 64 experts, k = 8: 8.3 us against 11.2 with two to a warp;
  // 256 tokens: 8.5 in one kernel).  One CTA up to 32 tokens (7.6 us; a cluster takes 8.3).  Two
  // rows of E words a warp: 32 warps up to 512 experts.
  const int warps = E <= 512 ? 32 : 16;
  const int csize = n <= 32 ? 1 : CLUSTER;
  const bool fused = n <= warps * CLUSTER;
  if (!fused) {
    const cudaError_t e = launch(route_topk_kernel<T, EPL>, dim3((n + 7) / 8), 256, 0, s->stream,
                                 1, logits, weights, experts, n, E, k, renormalize);
    if (e != cudaSuccess) return cuda_fail(e, "route_topk launch");
  }
  const size_t smem = sizeof(int) * (size_t)(2 * warps + 2) * E;
  const auto kern = route_group_kernel<T, EPL>;
  if (smem > 48 * 1024) {
    const qgemm_status st = group_smem_opt_in<T, EPL>(s);
    if (st != QGEMM_OK) return st;
  }
  return cuda_fail(launch(kern, dim3(csize), 32 * warps, smem, s->stream, csize, logits, weights,
                          experts, offsets, rows, n, E, k, renormalize, fused ? 1 : 0, csize),
                   "route_group launch");
}

template <typename T>
qgemm_status route_e(qgemm_stream_s* s, const T* l, float* w, int* x, int* o, int* r, int n, int E,
                     int k, int rn) {
  if (E <= 32) return route_t<T, 1>(s, l, w, x, o, r, n, E, k, rn);
  if (E <= 64) return route_t<T, 2>(s, l, w, x, o, r, n, E, k, rn);
  if (E <= 128) return route_t<T, 4>(s, l, w, x, o, r, n, E, k, rn);
  if (E <= 256) return route_t<T, 8>(s, l, w, x, o, r, n, E, k, rn);
  return route_t<T, 32>(s, l, w, x, o, r, n, E, k, rn);
}

template <typename T>
cudaError_t quant_t(qgemm_stream_s* s, const T* x, const int* rows, int8_t* q, float* sA, int n,
                    int k, int K, int R) {
  const bool vec = K % 4 == 0 && aligned((uint64_t)x, 4 * sizeof(T)) && aligned((uint64_t)q, 4);
  const int nv = vec ? (K / 4 + 255) / 256 : 0;
  int* bad = s->index_word;
  const dim3 g(n);
  if (nv == 1) return launch(dispatch_quant_kernel<T, 1>, g, 256, 0, s->stream, 1, x, rows, q, sA, k, K, R, bad);
  if (nv == 2) return launch(dispatch_quant_kernel<T, 2>, g, 256, 0, s->stream, 1, x, rows, q, sA, k, K, R, bad);
  if (nv == 3 || nv == 4)
    return launch(dispatch_quant_kernel<T, 4>, g, 256, 0, s->stream, 1, x, rows, q, sA, k, K, R, bad);
  if (nv > 4 && nv <= 8)
    return launch(dispatch_quant_kernel<T, 8>, g, 256, 0, s->stream, 1, x, rows, q, sA, k, K, R, bad);
  return launch(dispatch_quant_kernel<T, 0>, g, 256, 0, s->stream, 1, x, rows, q, sA, k, K, R, bad);
}

template <typename V>
cudaError_t copy_t(qgemm_stream_s* s, const void* x, const int* rows, void* out, int n, int k,
                   int pieces, int R) {
  const dim3 g((pieces + 255) / 256, n < 65535 ? n : 65535);
  return launch(dispatch_copy_kernel<V>, g, 256, 0, s->stream, 1, static_cast<const V*>(x), rows,
                static_cast<V*>(out), n, k, pieces, R, s->index_word);
}

template <typename TI, typename TO>
cudaError_t combine_t(qgemm_stream_s* s, const void* y, const int* rows, const float* weights,
                      const void* residual, void* out, int n, int k, int N, int R) {
  const bool vec = N % 8 == 0 && aligned((uint64_t)y, 16) && aligned((uint64_t)out, 16) &&
                   aligned((uint64_t)residual, 16);
  const dim3 g((N + 1023) / 1024, n < 65535 ? n : 65535);
  const TI* yi = static_cast<const TI*>(y);
  const TO* ri = static_cast<const TO*>(residual);
  TO* o = static_cast<TO*>(out);
  int* bad = s->index_word;
  auto go = [&](auto kern) {
    return launch(kern, g, 128, 0, s->stream, 1, yi, rows, weights, ri, o, n, k, N, R, bad);
  };
  if (!vec) return go(combine_kernel<TI, TO, false, 2>);
  if (k <= 2) return go(combine_kernel<TI, TO, true, 2>);
  if (k <= 4) return go(combine_kernel<TI, TO, true, 4>);
  return go(combine_kernel<TI, TO, true, 8>);
}

}  // namespace route

qgemm_status launch_route_topk(qgemm_stream_s* s, const void* logits, int in_dtype,
                               float* weights, int* experts, int* offsets, int* rows, int T,
                               int E, int k, int renormalize) {
  using namespace route;
  return in_dtype == QGEMM_F32
             ? route_e(s, static_cast<const float*>(logits), weights, experts, offsets, rows, T, E,
                       k, renormalize)
             : route_e(s, static_cast<const __nv_bfloat16*>(logits), weights, experts, offsets,
                       rows, T, E, k, renormalize);
}

qgemm_status launch_dispatch_rows(qgemm_stream_s* s, const void* x, int in_dtype,
                                  const int* rows, void* out, float* sq, int T, int k, int K,
                                  int R) {
  using namespace route;
  if (sq)
    return cuda_fail(in_dtype == QGEMM_F32
                         ? quant_t(s, static_cast<const float*>(x), rows, static_cast<int8_t*>(out),
                                   sq, T, k, K, R)
                         : quant_t(s, static_cast<const __nv_bfloat16*>(x), rows,
                                   static_cast<int8_t*>(out), sq, T, k, K, R),
                     "dispatch_quant launch");
  const size_t row = (size_t)K * (in_dtype == QGEMM_F32 ? 4 : 2);
  cudaError_t e;
  if (row % 16 == 0 && aligned((uint64_t)x, 16) && aligned((uint64_t)out, 16))
    e = copy_t<uint4>(s, x, rows, out, T, k, (int)(row / 16), R);
  else if (in_dtype == QGEMM_F32)
    e = copy_t<uint32_t>(s, x, rows, out, T, k, K, R);
  else
    e = copy_t<uint16_t>(s, x, rows, out, T, k, K, R);
  return cuda_fail(e, "dispatch_copy launch");
}

qgemm_status launch_combine_rows(qgemm_stream_s* s, const void* y, int in_dtype,
                                 const int* rows, const float* weights, const void* residual,
                                 void* out, int out_dtype, int T, int k, int N, int R) {
  using namespace route;
  const bool fi = in_dtype == QGEMM_F32, fo = out_dtype == QGEMM_F32;
  const cudaError_t e =
      fi ? (fo ? combine_t<float, float>(s, y, rows, weights, residual, out, T, k, N, R)
               : combine_t<float, __nv_bfloat16>(s, y, rows, weights, residual, out, T, k, N, R))
         : (fo ? combine_t<__nv_bfloat16, float>(s, y, rows, weights, residual, out, T, k, N, R)
               : combine_t<__nv_bfloat16, __nv_bfloat16>(s, y, rows, weights, residual, out, T, k, N, R));
  return cuda_fail(e, "combine launch");
}

}  // namespace qg
