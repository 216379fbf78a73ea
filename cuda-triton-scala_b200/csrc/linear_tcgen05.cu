// linear_tcgen05.cu -- linear layers with their epilogue on the sm_100a tensor cores, dense
// or grouped by expert over ragged row counts.
//
//     z[m, n] = sum_k x[m, k] w[n, k]      (bf16: fp32 sums; int8: int32 sums, then scales)
//     y[m, n] = act(z + bias[n]) + residual[m, n];  gated: act(z_gate) * z_up + residual
//
// Both kernels compute the transposed tile: the weights are the MMA's A operand (M = 128
// weight rows a CTA) and the tokens its B operand.  The tokens then lie along the MMA's N,
// which is a run-time field of the instruction descriptor: a group of 44 rows costs MMAs of 48
// (or 64) columns instead of a whole 128- or 256-row tile, and one token costs a 16-column
// one.  An accumulator column is a token, a TMEM lane a feature: bias and weight scale are
// per-lane constants.  Gated layers lay 8 gate rows and the 8 up rows of the same features by
// turns, so both halves of a product meet in one warp.
//
//   linear_pair_kernel    many rows: CTA pairs (tcgen05 cta_group::2), tiles of 256 weight
//       rows x up to 256 tokens, persistent, two accumulators so that the epilogue of a tile
//       overlaps the next tile's MMAs.  Bound by the tensor pipe and, after seconds of load, by
//       the power cap: int8 gated 8192 x 28672 x 4096 0.57 ms (3.38 POPS; 0.68 under the cap),
//       bf16 4096 x 4096 x 11008 with bias, gelu and residual 261 to 264 us (1.41 PFLOP/s; 322).
//       Ungated, the epilogue spills (about 450 bytes a thread at the 168 registers that ten
//       warps leave), which shows where few k-blocks hide it: 4976 x 1728 x 328 19 us, with GELU
//       36.
//   linear_stream_kernel  few rows: one CTA per tile of up to 128 weight rows x up to 96
//       tokens, two k-blocks a stage, persistent; a cluster of 1, 2, 4 or 8 CTAs cuts K and
//       joins its partial sums through distributed shared memory in rank order (so no scratch,
//       no atomics, the same bits every time).  Bound by reading the weights once: 940 MB of
//       experts' weights in 143 us (6.6 TB/s); small layers by 3.4 us of launch, first copy and
//       exchange (1 x 4096 x 4096 bf16 with bias and residual: 8.7 us).
//
// Experts: offsets[E + 1] are read on the device; every CTA lists the experts' tiles in
// shared memory (prefix sums) and walks the same persistent schedule, so the host never
// waits for the counts.
//
// Every barrier wait is bounded; one that runs out records a code in the device error word, and
// the abort flags that it raises make every other wait of the cluster give up.  Then, once all
// warps have stopped issuing, the CTA waits for its copies and MMAs (and, where K is cut, for the
// exchange's copies) whoever gave up, frees TMEM and returns.  Those waits have a limit of their
// own: the device's may be too short for a copy to land.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstring>
#include <mutex>

#include "linear_epilogue.cuh"
#include "linear_tiles.cuh"
#include "pair_copies.cuh"
#include "ptx.cuh"

namespace qg {
namespace lin {

constexpr int BK = 128;         // bytes of K a stage: one 128-byte swizzle row
constexpr int UMMA_K = 32;      // bytes of K an MMA
constexpr int WROWS = 128;      // weight rows of a CTA's tile
constexpr int W_BYTES = WROWS * BK;          // 16 KB
constexpr int CHUNK = 16;                    // accumulator columns (tokens) read at a time
constexpr int SMEM_MAX = 232448;             // 227 KB
constexpr int BAR_BYTES = 640;
constexpr int MAX_STAGES = 32;

struct Params : Schedule {
  Epi ep;
  const int* offsets;
  int num_k_blocks;
  int rows;         // weight rows of a CTA's tile: 128, in the stream kernel a multiple of 16
  int feats;        // features of them: rows, gated rows / 2
  int stages;
  int seg_kb;       // k-blocks of one accumulator (SEG)
  int csize;        // CTAs of a cluster (stream kernel)
  int box;          // token rows of a TMA box (stream kernel)
  int tmem_cols;    // TMEM columns (stream kernel)
  int hold;         // the epilogue waits for what never comes (qgemm_debug_hold_split)
  int* err;         // a wait ran out
  int* bad;         // an offset out of range
  unsigned long long wait_ns;
};

// One thread: the table of a dense layer, one group of M rows.
__device__ __forceinline__ void dense_table(const Params& p, const Table& tb) {
  tb.row0[0] = 0;
  tb.cnt[0] = p.M;
  tb.pref[0] = 0;
  tb.pref[1] = blocks_of(p, p.M) * p.num_w_blocks;
}

// All threads: fills the experts' table.  No rows where expert_rows or kMostTiles says so.
__device__ __forceinline__ void fill_table(const Params& p, const Table& tb) {
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int o0, o1;
    if (!expert_rows(p, p.offsets, e, o0, o1) && blockIdx.x == 0) note_bad_index(p.bad);
    tb.row0[e] = o0;
    tb.cnt[e] = o1 - o0;
    tb.pref[e] = blocks_of(p, o1 - o0) * p.num_w_blocks;
  }
  __syncthreads();
  if (threadIdx.x < 32) {  // exclusive scan, a run of experts a lane
    const int lane = threadIdx.x;
    const int chunk = (p.E + 31) / 32, e0 = min(p.E, lane * chunk), e1 = min(p.E, e0 + chunk);
    long long sum = 0;
    for (int e = e0; e < e1; ++e) sum += tb.pref[e];
    long long run = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += o;
    }
    const long long all = __shfl_sync(0xffffffffu, run, 31);
    if (all > kMostTiles && lane == 0 && blockIdx.x == 0) note_bad_index(p.bad);
    if (lane == 31) tb.pref[p.E] = tiles_before(all, all);
    run -= sum;
    for (int e = e0; e < e1; ++e) {
      const int c = tb.pref[e];
      tb.pref[e] = tiles_before(run, all);
      run += c;
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void report(int* err, int code, volatile int* abort_flag) {
  *abort_flag = 1;
  if (err) atomicCAS(err, 0, code);
}

// As report(), and raises the abort flags of the other CTAs of the cluster, so that their
// waits give up at once.
__device__ __forceinline__ void report_cluster(int* err, int code, volatile int* abort_flag,
                                               int csize) {
  report(err, code, abort_flag);
  const uint32_t here = ptx::smem_u32(const_cast<int*>(abort_flag));
  for (int c = 0; c < csize; ++c) ptx::st_cluster_u32(ptx::map_to_rank(here, c), 1u);
}

// A whole warp waits; false (in every lane) when a lane's wait ran out, after reporting `code`.
__device__ __forceinline__ bool warp_wait(const Params& p, uint32_t bar, uint32_t parity,
                                          volatile int* abort_flag, int code, int csize) {
  const bool ok = ptx::mbar_wait(bar, parity, abort_flag, p.wait_ns);
  if (__all_sync(0xffffffffu, ok)) return true;
  if (threadIdx.x % 32 == 0 && !*abort_flag) report_cluster(p.err, code, abort_flag, csize);
  __syncwarp();
  return false;
}

// ---- finishing four features of a token ---------------------------------------------------

// Per-lane constants of a tile: this lane's four features (and, gated, their up rows).
template <bool GATED>
struct Feat {
  int n;            // first feature, N or more: none
  float sg[4], bg[4], su[GATED ? 4 : 1], bu[GATED ? 4 : 1];
};

template <int KIND, bool GATED>
__device__ __forceinline__ void load_feat(const Epi& ep, int e, int n, Feat<GATED>& f) {
  f.n = n;
  const size_t base = (size_t)e * ep.nw + n;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = n + i < ep.N;
    f.sg[i] = KIND == KIND_I8 && in ? __ldg(ep.sw + base + i) : 0.f;
    f.bg[i] = ep.bias && in ? __ldg(ep.bias + base + i) : 0.f;
    if constexpr (GATED) {
      f.su[i] = KIND == KIND_I8 && in ? __ldg(ep.sw + base + ep.N + i) : 0.f;
      f.bu[i] = ep.bias && in ? __ldg(ep.bias + base + ep.N + i) : 0.f;
    }
  }
}

// The residual of four features of a row, fetched before the products are needed.
template <bool F32>
__device__ __forceinline__ void load_residual(const Epi& ep, int row, int n, float (&r)[4]) {
  if (!ep.residual) return;
  const size_t at = (size_t)row * ep.ldr + n;
  if (ep.vec && n + 4 <= ep.N) {
    if constexpr (F32) {
      const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(ep.residual) + at);
      r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(
          static_cast<const __nv_bfloat16*>(ep.residual) + at);
      r[0] = __uint_as_float(u.x << 16);
      r[1] = __uint_as_float(u.x & 0xffff0000u);
      r[2] = __uint_as_float(u.y << 16);
      r[3] = __uint_as_float(u.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = n + i < ep.N ? load_out(ep.residual, F32, at + i) : 0.f;
  }
}

// ACT is a compile-time choice: the switch sits outside the loops.
template <int KIND, bool GATED, bool F32, int ACT>
__device__ __forceinline__ void finish4(const Epi& ep, const Feat<GATED>& f, int row, float sx,
                                        const uint32_t (&g)[4], const uint32_t (&u)[4],
                                        const float (&res)[4]) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = activate<F32>(ACT, __fadd_rn(dequant<KIND>(g[i], f.sg[i], sx), f.bg[i]));
    if constexpr (GATED)
      v[i] = __fmul_rn(v[i], __fadd_rn(dequant<KIND>(u[i], f.su[i], sx), f.bu[i]));
  }
  if (ep.residual) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __fadd_rn(v[i], res[i]);
  }
  const size_t at = (size_t)row * ep.ldc + f.n;
  if (ep.vec && f.n + 4 <= ep.N) {
    if constexpr (F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(ep.out) + at) =
          make_float4(v[0], v[1], v[2], v[3]);
    } else {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]);
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(ep.out) + at) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f.n + i < ep.N) store_out(ep.out, F32, at + i, v[i]);
  }
}

// ---- finishing a chunk of 16 tokens where the accumulator lies ------------------------------

// A lane's weight row: its feature (N or more: none), scale and bias.  Gated: a warp's lanes
// hold 8 gate rows, the up rows of those 8 features, 8 gate rows and their up rows.
template <bool GATED>
struct Lane {
  int f;
  float sw, b;
};

template <int KIND, bool GATED>
__device__ __forceinline__ Lane<GATED> lane_of(const Epi& ep, int e, int f0, int rows, int q,
                                               int lane) {
  Lane<GATED> l;
  l.f = f0 + (GATED ? q * 16 + lane / 16 * 8 + lane % 8 : q * 32 + lane);
  if (q * 32 + lane >= rows) l.f = ep.N + 2;  // its pair is past N too
  const size_t at = (size_t)e * ep.nw + l.f + (GATED && (lane & 8) ? ep.N : 0);
  const bool in = l.f < ep.N;
  l.sw = KIND == KIND_I8 && in ? __ldg(ep.sw + at) : 0.f;
  l.b = ep.bias && in ? __ldg(ep.bias + at) : 0.f;
  return l;
}

// r: 16 accumulator columns (tokens row0 .. row0 + 15, of which `n` exist) of this lane's
// weight row, valid after `ready`.  Gated, lanes l and l + 8 hold the gate and the up sums
// of one feature: one shuffle a token pair gives lane l the even token and lane l + 8 the odd
// one.  bf16 outputs are stored as feature pairs: one shuffle a token pair gives even lanes
// both features of the first token and odd lanes those of the second, so that a warp's store
// covers whole 32-byte sectors of two (gated: four) token rows.  Stores go straight to memory:
// through a staging buffer in shared memory (256-byte runs of a token) the int8 layer at
// 8192 x 28672 x 4096 took 827 us instead of 790.
// FULL: all 16 tokens and all of the warp's features exist.
template <int KIND, bool GATED, bool F32, int ACT, bool FULL, typename Ready>
__device__ __forceinline__ void finish_chunk_t(const Epi& ep, const Lane<GATED>& l, int row0, int n,
                                               int lane, const uint32_t (&r)[16], Ready&& ready) {
  constexpr int NV = GATED ? 8 : 16;       // values a lane finishes
  const int hi = GATED ? lane / 8 % 2 : 0; // value i is token (GATED ? 2 i + hi : i)
  const int fe = l.f & ~1;                 // packed: features fe, fe + 1
  const int odd = l.f & 1;
  const bool packed = !F32 && ep.vec2;
  // packed: pair i of this lane is token `first` + `step` i, feature fe
  const int first = GATED ? 2 * odd + hi : odd;
  constexpr int step = GATED ? 4 : 2;
  // fetched while the accumulator load is under way
  float sx = 0.f;
  if (KIND == KIND_I8 && (FULL || lane % 16 < n)) sx = __ldg(ep.sx + row0 + lane % 16);
  float res[NV];
  if (ep.residual) {
    if (packed) {
      const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(ep.residual) +
                               (size_t)(row0 + first) * ep.ldr + fe;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i, p += step * ep.ldr) {
        uint32_t w = 0;
        if (FULL || (first + step * i < n && fe + 1 < ep.N)) w = *reinterpret_cast<const uint32_t*>(p);
        else if (first + step * i < n && fe < ep.N) w = *reinterpret_cast<const uint16_t*>(p);
        res[2 * i] = __uint_as_float(w << 16);
        res[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int t = GATED ? 2 * i + hi : i;
        res[i] = FULL || (t < n && l.f < ep.N)
                     ? load_out(ep.residual, F32, (size_t)(row0 + t) * ep.ldr + l.f) : 0.f;
      }
    }
  }
  ready();
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float s = KIND == KIND_I8 ? __shfl_sync(0xffffffffu, sx, j) : 0.f;
    v[j] = __fadd_rn(dequant<KIND>(r[j], l.sw, s), l.b);
    if (!GATED) v[j] = activate<F32>(ACT, v[j]);
  }
  if constexpr (GATED) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, hi ? v[2 * i] : v[2 * i + 1], 8);
      const float gate = hi ? other : v[2 * i], up = hi ? v[2 * i + 1] : other;
      v[i] = __fmul_rn(activate<F32>(ACT, gate), up);
    }
  }
  if (packed) {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(ep.out) + (size_t)(row0 + first) * ep.ldc + fe;
#pragma unroll
    for (int i = 0; i < NV / 2; ++i, p += step * ep.ldc) {
      uint32_t w;
      if (ep.residual) {
        const float other = __shfl_xor_sync(0xffffffffu, odd ? v[2 * i] : v[2 * i + 1], 1);
        const float a = odd ? other : v[2 * i], b = odd ? v[2 * i + 1] : other;
        const __nv_bfloat162 h = __floats2bfloat162_rn(__fadd_rn(a, res[2 * i]),
                                                       __fadd_rn(b, res[2 * i + 1]));
        w = *reinterpret_cast<const uint32_t*>(&h);
      } else {  // rounded first, so that one word crosses and one byte permute sorts
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        const uint32_t mine = *reinterpret_cast<const uint32_t*>(&h);
        const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
        w = odd ? __byte_perm(other, mine, 0x7632) : __byte_perm(mine, other, 0x5410);
      }
      if (FULL || (first + step * i < n && fe + 1 < ep.N)) *reinterpret_cast<uint32_t*>(p) = w;
      else if (first + step * i < n && fe < ep.N) *reinterpret_cast<uint16_t*>(p) = (uint16_t)w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int t = GATED ? 2 * i + hi : i;
      if (FULL || (t < n && l.f < ep.N)) {
        const float y = ep.residual ? __fadd_rn(v[i], res[i]) : v[i];
        store_out(ep.out, F32, (size_t)(row0 + t) * ep.ldc + l.f, y);
      }
    }
  }
}

template <int KIND, bool GATED, bool F32, int ACT, typename Ready>
__device__ __forceinline__ void finish_chunk(const Epi& ep, const Lane<GATED>& l, int row0, int n,
                                             int lane, const uint32_t (&r)[16], Ready&& ready) {
  if (n >= 16 && __all_sync(0xffffffffu, l.f < ep.N))
    finish_chunk_t<KIND, GATED, F32, ACT, true>(ep, l, row0, n, lane, r, ready);
  else
    finish_chunk_t<KIND, GATED, F32, ACT, false>(ep, l, row0, n, lane, r, ready);
}

// SEG: r (16 fp32 accumulator columns being loaded) plus the running sums at TMEM address
// `run` where `more` is set; valid after the call.
__device__ __forceinline__ void add_running(uint32_t run, bool more, uint32_t (&r)[16]) {
  if (more) {
    uint32_t q[16];
    ptx::tmem_ld_32x32b_x16(run, q);
    ptx::tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j)
      r[j] = __float_as_uint(__fadd_rn(__uint_as_float(q[j]), __uint_as_float(r[j])));
  } else {
    ptx::tmem_wait_ld();
  }
}

// Calls fn with the activation as a compile-time constant.
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& fn) {
  switch (act) {
    case QGEMM_ACT_RELU: fn(std::integral_constant<int, QGEMM_ACT_RELU>()); break;
    case QGEMM_ACT_GELU: fn(std::integral_constant<int, QGEMM_ACT_GELU>()); break;
    case QGEMM_ACT_GELU_TANH: fn(std::integral_constant<int, QGEMM_ACT_GELU_TANH>()); break;
    case QGEMM_ACT_SILU: fn(std::integral_constant<int, QGEMM_ACT_SILU>()); break;
    default: fn(std::integral_constant<int, QGEMM_ACT_NONE>()); break;
  }
}

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ void st_shared_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Adds four accumulator words: int32, or fp32 rounding to nearest.
template <int KIND>
__device__ __forceinline__ void add_words(uint32_t (&a)[4], const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    a[i] = KIND == KIND_I8 ? a[i] + w[i]
                           : __float_as_uint(__fadd_rn(__uint_as_float(a[i]), __uint_as_float(w[i])));
}

// ---- the CTA-pair kernel -------------------------------------------------------------------
namespace pair {
constexpr int TOK = 256;                  // tokens of a tile at most (MMA N)
constexpr int TOK_BYTES = (TOK / 2) * BK; // each CTA holds half the tokens: 16 KB a stage
constexpr int STAGE_BYTES = W_BYTES + TOK_BYTES;
constexpr int BOX = 32;                   // token rows of a TMA box where half a tile has
                                          // fewer than 97 (else one box of 128)
constexpr int EPI_WARPS = 8;              // two groups of four (one warp a TMEM lane quadrant)
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int SEG_TOK = 128;              // tokens of a tile at most with SEG
}  // namespace pair

// What a pair that gave up has under way, once neither CTA issues any more and both see their
// abort flag; all threads of both.  (Out of line, as the stream kernel's: inline it lay between
// the hot code and the exit, and cost small calls 0.3 us of instruction fetch.)
namespace pair {
__device__ __noinline__ void drain(const Params& p, uint32_t bar_base, uint32_t copies,
                                   uint32_t drain_bar, volatile int* abort_flag) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = ptx::cluster_ctarank();
  if (warp == 0 && rank == 0 && lane == 0 && !settle_pair_copies(bar_base, p.stages, copies))
    report(p.err, DEVERR_TIMEOUT_DRAIN, abort_flag);
  __syncwarp();
  if (warp == 1) {  // everything that the even CTA's issuer has committed, in both CTAs
    if (rank == 0 && ptx::elect_one()) ptx::umma_commit_pair(drain_bar, 0x3);
    __syncwarp();
    if (lane == 0 && !ptx::mbar_wait(drain_bar, 0, nullptr, DRAIN_NS))
      report(p.err, DEVERR_TIMEOUT_DRAIN, abort_flag);
    __syncwarp();
  }
  __syncthreads();
  ptx::cluster_sync_all();  // neither CTA leaves before the other's copies and MMAs have ended
}
}  // namespace pair

// F32: the output's type (and the residual's), and with it the form of the activation.
template <int KIND, bool GATED, bool SEG, bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::THREADS, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tmW,
                       const __grid_constant__ CUtensorMap tmG,
                       const __grid_constant__ CUtensorMap tmX,
                       const __grid_constant__ CUtensorMap tmXs, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw_base);
  const int S = p.stages;
  const uint32_t bar_base = base + S * pair::STAGE_BYTES;
  uint8_t* gbar = gbase + S * pair::STAGE_BYTES;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (MAX_STAGES + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * MAX_STAGES + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * MAX_STAGES + 2 + a); };
  const uint32_t drain_bar = bar_base + 8u * (2 * MAX_STAGES + 4);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbar + 8 * (2 * MAX_STAGES + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbar + 8 * (2 * MAX_STAGES + 5) + 4);
  constexpr int COPIES_AT = 8 * (2 * MAX_STAGES + 6);
  static_assert(COPIES_AT + (int)sizeof(PairCopies) <= BAR_BYTES, "barriers and counts");
  static_assert((SMEM_MAX - BAR_BYTES) / pair::STAGE_BYTES <= 8, "stages that PairCopies holds");
  PairCopies* copies = reinterpret_cast<PairCopies*>(gbar + COPIES_AT);
  Table tb;
  tb.row0 = reinterpret_cast<int*>(gbar + BAR_BYTES);
  tb.cnt = tb.row0 + p.E;
  tb.pref = tb.cnt + p.E;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = ptx::cluster_ctarank();
  const int pid = blockIdx.x / 2, npairs = gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(tfull_bar(a), 1);
      ptx::mbar_init(tempty_bar(a), 2 * pair::EPI_WARPS);
    }
    ptx::mbar_init(drain_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::grid_launch_dependents();
    ptx::prefetch_tmap(GATED ? &tmG : &tmW);
    ptx::prefetch_tmap(&tmX);
    if (!p.offsets) dense_table(p, tb);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    ptx::tmem_relinquish_pair();
  }
  // everything up to here overlaps the previous kernel
  ptx::tc_fence_before();
  ptx::cluster_sync_all();
  ptx::tc_fence_after();
  ptx::grid_dependency_wait();
  if (p.offsets) fill_table(p, tb);
  const uint32_t tmem_base = *tmem_slot;
  Tile it_;

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    int stage = 0;
    uint32_t phase = 0;
    long long issued = 0;
    bool ok = true;
    for (int item = 0; ok && pair_item(p, tb, pid, npairs, item, it_); ++item) {
      if (it_.n == 0) continue;
      const int half = (it_.n + p.tok_round - 1) / p.tok_round * p.tok_round / 2;
      const int boxes = (half + pair::BOX - 1) / pair::BOX;  // 1 to 4
      const uint32_t tx = 2u * (W_BYTES + (uint32_t)boxes * pair::BOX * BK);
      const int x0 = it_.t0 + (int)rank * half;
      // this CTA's weight rows: 128 of the block's 256, or 64 gate and 64 up rows
      const int f0 = (it_.wb * 2 + (int)rank) * p.feats;
      const int w0 = it_.e * p.ep.nw + f0;
      for (int kb = 0; kb < p.num_k_blocks; ++kb) {
        if (!warp_wait(p, empty_bar(stage), phase ^ 1u, abort_flag, DEVERR_TIMEOUT_PRODUCER, 2)) {
          ok = false;
          break;
        }
        if (ptx::elect_one()) {
          copies->half[stage] = tx / 2;
          const uint32_t sw = base + stage * pair::STAGE_BYTES, sx = sw + W_BYTES;
          const uint32_t fb = ptx::map_to_rank(full_bar(stage), 0);
          if (rank == 0) ptx::mbar_arrive_expect_tx(full_bar(stage), tx);
          if constexpr (GATED) {
            // 8 gate rows, the 8 up rows of the same features, and so on: both halves of a
            // feature's product land in one warp's TMEM lanes.  One copy through the 5-D map
            // (k, row of 8, gate / up, block of 8 features, expert) where all 64 features lie
            // in whole blocks, else one copy for every 8 rows (the last features of an N that
            // is not a multiple of 8; eight copies for every tile made the layer 25 % slower)
            if (f0 + 64 <= p.ep.N / 8 * 8) {
              ptx::tma_load_5d_pair(sw, &tmG, fb, kb * BK, 0, 0, f0 / 8, it_.e);
            } else {
              for (int b = 0; b < 8; ++b) {
                ptx::tma_load_2d_pair(sw + (2 * b) * 8 * BK, &tmW, fb, kb * BK, w0 + 8 * b);
                ptx::tma_load_2d_pair(sw + (2 * b + 1) * 8 * BK, &tmW, fb, kb * BK, w0 + p.ep.N + 8 * b);
              }
            }
          } else {
            ptx::tma_load_2d_pair(sw, &tmW, fb, kb * BK, w0);
          }
          if (boxes == 4)
            ptx::tma_load_2d_pair(sx, &tmX, fb, kb * BK, x0);
          else
            for (int b = 0; b < boxes; ++b)
              ptx::tma_load_2d_pair(sx + b * pair::BOX * BK, &tmXs, fb, kb * BK, x0 + b * pair::BOX);
        }
        __syncwarp();
        ++issued;
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
    }
    if (lane == 0) copies->stages = issued;
  } else if (warp == 1) {
    // ---------------- MMA issuer (even CTA) ----------------
    if (rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      for (int item = 0; ok && pair_item(p, tb, pid, npairs, item, it_); ++item) {
        if (it_.n == 0) continue;
        const int ncol = (it_.n + p.tok_round - 1) / p.tok_round * p.tok_round;
        const uint32_t idesc = KIND == KIND_BF16 ? ptx::idesc_bf16(256, ncol)
                                                 : ptx::idesc_i8(256, ncol, false, false);
        const int seg = SEG ? p.seg_kb : p.num_k_blocks;
        for (int kb0 = 0; ok && kb0 < p.num_k_blocks; kb0 += seg) {
          const int a = it & 1;
          if (!warp_wait(p, tempty_bar(a), (uint32_t)((it >> 1) & 1) ^ 1u, abort_flag,
                         DEVERR_TIMEOUT_MMA, 2)) {
            ok = false;
            break;
          }
          ++it;
          ptx::tc_fence_after();
          const uint32_t d_tmem = tmem_base + (uint32_t)(a * 256);
          const int kb1 = min(kb0 + seg, p.num_k_blocks);
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!warp_wait(p, full_bar(stage), phase, abort_flag, DEVERR_TIMEOUT_MMA, 2)) {
              ok = false;
              break;
            }
            ptx::tc_fence_after();
            if (ptx::elect_one()) {
              const uint32_t sw = base + stage * pair::STAGE_BYTES;
              const uint64_t adesc = ptx::smem_desc_sw128(sw, 16, 1024);
              const uint64_t bdesc = ptx::smem_desc_sw128(sw + W_BYTES, 16, 1024);
#pragma unroll
              for (int kk = 0; kk < BK / UMMA_K; ++kk) {  // 32 bytes further along the swizzled rows
                const uint32_t accum = (kb != kb0 || kk != 0) ? 1u : 0u;
                if constexpr (KIND == KIND_BF16)
                  ptx::umma_bf16_pair(d_tmem, adesc + kk * (UMMA_K / 16), bdesc + kk * (UMMA_K / 16), idesc, accum);
                else
                  ptx::umma_i8_pair(d_tmem, adesc + kk * (UMMA_K / 16), bdesc + kk * (UMMA_K / 16), idesc, accum);
              }
              ptx::umma_commit_pair(empty_bar(stage), 0x3);
              if (kb + 1 == kb1) ptx::umma_commit_pair(tfull_bar(a), 0x3);
            }
            __syncwarp();
            if (++stage == S) { stage = 0; phase ^= 1u; }
          }
        }
      }
    }
  } else {
    // ---------------- epilogue (both CTAs, two groups of four warps) ----------------
    const int q = warp & 3;             // TMEM lane quadrant
    const int grp = (warp - 2) / 4;     // chunks c with c % 2 == grp
    const uint32_t te0 = ptx::map_to_rank(tempty_bar(0), 0);
    const uint32_t te1 = ptx::map_to_rank(tempty_bar(1), 0);
    const uint32_t tmem_q = tmem_base + ((uint32_t)(q * 32) << 16);
    int it = 0;
    for (int item = 0; pair_item(p, tb, pid, npairs, item, it_); ++item) {
      if (it_.n == 0) continue;
      const Lane<GATED> f =
          lane_of<KIND, GATED>(p.ep, it_.e, (it_.wb * 2 + (int)rank) * p.feats, WROWS, q, lane);
      const int chunks = (it_.n + CHUNK - 1) / CHUNK;
      // this warp's part of the residual into L2 while the MMAs run: its loads come chunk by
      // chunk, and the last tile's epilogue waits for every one
      if (p.ep.residual) {
        const int os = F32 ? 4 : 2;
        const int f0 = (it_.wb * 2 + (int)rank) * p.feats + q * (GATED ? 16 : 32);
        const char* at = static_cast<const char*>(p.ep.residual) + ((size_t)it_.t0 * p.ep.ldr + f0) * os;
        for (int t = grp * 32 + lane; t < it_.n && f0 < p.ep.N; t += 64)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(at + (size_t)t * p.ep.ldr * os));
      }
      // Waits for accumulator it & 1; a warp whose wait ran out stores nothing.
      auto acc_ready = [&]() {
        bool ok = ptx::mbar_wait(p.hold ? drain_bar : tfull_bar(it & 1),
                                 p.hold ? 0u : (uint32_t)((it >> 1) & 1), abort_flag, p.wait_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok && lane == 0 && !*abort_flag)
          report_cluster(p.err, DEVERR_TIMEOUT_EPILOGUE, abort_flag, 2);
        ptx::tc_fence_after();
        return ok;
      };
      auto acc_done = [&]() {  // this warp has read its columns
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_remote((it & 1) ? te1 : te0);
        ++it;
      };
      // SEG: the running sums of the segments before live in TMEM columns 128 ..
      const int seg = SEG ? p.seg_kb : p.num_k_blocks;
      for (int kb = 0; kb < p.num_k_blocks; kb += seg) {
        const bool ok = acc_ready();
        const uint32_t acc = tmem_q + (uint32_t)((it & 1) * 256);
        if (!ok) {
        } else if (SEG && kb + seg < p.num_k_blocks) {
          for (int c = grp; c < chunks; c += 2) {
            uint32_t r[16];
            ptx::tmem_ld_32x32b_x16(acc + (uint32_t)(c * CHUNK), r);
            add_running(tmem_q + (uint32_t)(128 + c * CHUNK), kb > 0, r);
            ptx::tmem_st_32x32b_x16(tmem_q + (uint32_t)(128 + c * CHUNK), r);
          }
          ptx::tmem_wait_st();
        } else {
          with_act(p.ep.act, [&](auto act) {
            for (int c = grp; c < chunks; c += 2) {
              uint32_t r[16];
              ptx::tmem_ld_32x32b_x16(acc + (uint32_t)(c * CHUNK), r);
              if (SEG) add_running(tmem_q + (uint32_t)(128 + c * CHUNK), kb > 0, r);
              finish_chunk<KIND, GATED, F32, decltype(act)::value>(
                  p.ep, f, it_.t0 + c * CHUNK, it_.n - c * CHUNK, lane, r,
                  [] { if (!SEG) ptx::tmem_wait_ld(); });
            }
          });
        }
        acc_done();
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();
  ptx::tc_fence_after();
  // From here nobody issues any more, and a flag that was raised is raised in both CTAs.
  if (*abort_flag) pair::drain(p, bar_base, bar_base + COPIES_AT, drain_bar, abort_flag);
  if (warp == 1) {
    __syncwarp();
    ptx::tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---- the streaming kernel ------------------------------------------------------------------
namespace strm {  // tiles of 16 to 96 tokens at most (Params::tok_max, a multiple of 16)
constexpr int THREADS = 192;   // producer, MMA issuer, four epilogue warps
constexpr int TOK = 96;        // tokens of a tile at most: more leave too few stages
constexpr int XTOK = 64;       // tokens of an exchange at most (SPLIT)
constexpr int STEP = 2;        // k-blocks of a stage: one barrier round for both
}  // namespace strm

// What a CTA that gave up has under way, once its warps issue no more; all its threads.  `issued`
// stages were filled.
namespace strm {
__device__ __noinline__ void drain(const Params& p, uint32_t bar_base, long long issued,
                                   uint32_t drain_bar, volatile int* abort_flag) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, S = p.stages;
  if (warp == 0 && lane == 0) {
    for (long long f = max(0ll, issued - S); f < issued; ++f)
      if (!ptx::mbar_wait(bar_base + 8u * (int)(f % S), (uint32_t)((f / S) & 1), nullptr, DRAIN_NS)) {
        report(p.err, DEVERR_TIMEOUT_DRAIN, abort_flag);
        break;
      }
  }
  __syncwarp();
  if (warp == 1) {
    if (ptx::elect_one()) ptx::umma_commit(drain_bar);
    __syncwarp();
    if (lane == 0 && !ptx::mbar_wait(drain_bar, 0, nullptr, DRAIN_NS))
      report(p.err, DEVERR_TIMEOUT_DRAIN, abort_flag);
    __syncwarp();
  }
  __syncthreads();
}
}  // namespace strm

// SPLIT: a cluster of csize CTAs cuts K.  The sums of a token go to the rank that finishes it,
// which adds them in rank order: each warp lays its 32 weight rows' sums out in shared memory
// ([token][32]) and sends every rank its run of tokens as one bulk copy, counted in bytes on the
// receiver's barrier (word by word with st.async, 33 tokens took 2700 cycles a tile and 128
// took 8500; DSMEM moves wide runs far better).  Otherwise a CTA finishes its own accumulator.
template <int KIND, bool GATED, bool SEG, bool F32, bool SPLIT>
__global__ void __launch_bounds__(strm::THREADS, 1)
    linear_stream_kernel(const __grid_constant__ CUtensorMap tmW,
                         const __grid_constant__ CUtensorMap tmG,
                         const __grid_constant__ CUtensorMap tmX,
                         const __grid_constant__ CUtensorMap, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw_base);
  const int S = p.stages, TOK = p.tok_max, C = SPLIT ? p.csize : 1;
  const int box = p.box;
  const uint32_t w_bytes = (uint32_t)(p.rows * BK);
  const uint32_t x_bytes = (uint32_t)(TOK * BK);
  const uint32_t stage_bytes = strm::STEP * (w_bytes + x_bytes);  // weights, then tokens
  // SPLIT: the sums that this rank sends, [warp][token][32 weight rows] words, and those of its
  // own tokens, [source rank][warp][XT / C tokens][32]
  const int XT = min(TOK, strm::XTOK);
  const uint32_t send = base + S * stage_bytes;
  const uint32_t recv = send + (SPLIT ? (uint32_t)XT * WROWS * 4u : 0u);
  const uint32_t bar_base = recv + (SPLIT ? (uint32_t)XT * WROWS * 4u : 0u);
  uint8_t* gbar = gbase + (bar_base - base);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (MAX_STAGES + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * MAX_STAGES + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * MAX_STAGES + 2 + a); };
  const uint32_t drain_bar = bar_base + 8u * (2 * MAX_STAGES + 4);
  const uint32_t rfull_bar = bar_base + 8u * (2 * MAX_STAGES + 5);   // all ranks' sums are in
  const uint32_t rempty_bar = bar_base + 8u * (2 * MAX_STAGES + 6);  // every rank has read its
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbar + 8 * (2 * MAX_STAGES + 7));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbar + 8 * (2 * MAX_STAGES + 7) + 4);
  constexpr int COUNT_AT = 8 * (2 * MAX_STAGES + 8);  // stages the producer filled
  static_assert(COUNT_AT + 8 <= BAR_BYTES, "barriers and count");
  Table tb;
  tb.row0 = reinterpret_cast<int*>(gbar + BAR_BYTES);
  tb.cnt = tb.row0 + p.E;
  tb.pref = tb.cnt + p.E;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = SPLIT ? (int)ptx::cluster_ctarank() : 0;
  const int cid = blockIdx.x / C, nclusters = gridDim.x / C;
  const uint32_t tmem_cols = (uint32_t)p.tmem_cols;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(tfull_bar(a), 1);
      ptx::mbar_init(tempty_bar(a), 4);
    }
    ptx::mbar_init(drain_bar, 1);
    ptx::mbar_init(rfull_bar, 1);
    ptx::mbar_init(rempty_bar, 4 * C);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::grid_launch_dependents();
    ptx::prefetch_tmap(GATED ? &tmG : &tmW);
    ptx::prefetch_tmap(&tmX);
    if (!p.offsets) dense_table(p, tb);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), tmem_cols);
    ptx::tmem_relinquish();
  }
  // everything up to here overlaps the previous kernel
  ptx::tc_fence_before();
  if (SPLIT) ptx::cluster_sync_all(); else __syncthreads();
  ptx::tc_fence_after();
  ptx::grid_dependency_wait();
  if (p.offsets) fill_table(p, tb);
  const uint32_t tmem_base = *tmem_slot;
  const int T = tb.pref[p.E];
  // this rank's k-blocks: whole stages, at least one (the host cuts K no finer)
  const int ksteps = (p.num_k_blocks + strm::STEP - 1) / strm::STEP;
  const int kb0 = ksteps * rank / C * strm::STEP;
  const int kb1 = min(p.num_k_blocks, ksteps * (rank + 1) / C * strm::STEP);

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    int stage = 0;
    uint32_t phase = 0;
    long long issued = 0;
    bool ok = true;
    for (int tile = cid; ok && tile < T; tile += nclusters) {
      const Tile t = tile_of(p, tb, tile, p.band);
      const int boxes = (t.n + box - 1) / box;
      const uint32_t tx = w_bytes + (uint32_t)(boxes * box * BK);
      const int f0 = t.wb * p.feats, w0 = t.e * p.ep.nw + f0;
      for (int kb = kb0; kb < kb1; kb += strm::STEP) {
        if (!warp_wait(p, empty_bar(stage), phase ^ 1u, abort_flag, DEVERR_TIMEOUT_PRODUCER, C)) {
          ok = false;
          break;
        }
        if (ptx::elect_one()) {
          const uint32_t fb = full_bar(stage);
          const int nk = min(strm::STEP, kb1 - kb);
          ptx::mbar_arrive_expect_tx(fb, (uint32_t)nk * tx);
#pragma unroll
          for (int h = 0; h < strm::STEP; ++h) {
            if (h >= nk) break;
            const uint32_t sw = base + stage * stage_bytes + h * w_bytes;
            const int ck = (kb + h) * BK;
            if constexpr (GATED) {  // gate and up rows by turns of 8, as in the pair kernel
              if (f0 + p.feats <= p.ep.N / 8 * 8) {
                ptx::tma_load_5d(sw, &tmG, fb, ck, 0, 0, f0 / 8, t.e);
              } else {
                for (int b = 0; b < p.feats / 8; ++b) {
                  ptx::tma_load_2d(sw + (2 * b) * 8 * BK, &tmW, fb, ck, w0 + 8 * b);
                  ptx::tma_load_2d(sw + (2 * b + 1) * 8 * BK, &tmW, fb, ck, w0 + p.ep.N + 8 * b);
                }
              }
            } else {
              ptx::tma_load_2d(sw, &tmW, fb, ck, w0);
            }
          }
#pragma unroll
          for (int h = 0; h < strm::STEP; ++h) {
            if (h >= nk) break;
            const uint32_t sx = base + stage * stage_bytes + strm::STEP * w_bytes + h * x_bytes;
            for (int b = 0; b < boxes; ++b)
              ptx::tma_load_2d(sx + b * box * BK, &tmX, fb, (kb + h) * BK, t.t0 + b * box);
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
    }
    if (lane == 0) *reinterpret_cast<volatile long long*>(gbar + COUNT_AT) = issued;
    __syncwarp();
    if (SPLIT) ptx::cluster_arrive();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    int stage = 0;
    uint32_t phase = 0;
    int it = 0;
    bool ok = true;
    for (int tile = cid; ok && tile < T; tile += nclusters) {
      const Tile t = tile_of(p, tb, tile, p.band);
      const int ncol = (t.n + 15) / 16 * 16;
      const uint32_t idesc = KIND == KIND_BF16 ? ptx::idesc_bf16(128, ncol)
                                               : ptx::idesc_i8(128, ncol, false, false);
      const int seg = SEG ? p.seg_kb : p.num_k_blocks;
      for (int s0 = kb0; ok && s0 < kb1; s0 += seg) {
        const int a = it & 1;
        if (!warp_wait(p, tempty_bar(a), (uint32_t)((it >> 1) & 1) ^ 1u, abort_flag,
                       DEVERR_TIMEOUT_MMA, C)) {
          ok = false;
          break;
        }
        ++it;
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(a * TOK);
        const int s1 = min(s0 + seg, kb1);
        for (int kb = s0; kb < s1; kb += strm::STEP) {
          if (!warp_wait(p, full_bar(stage), phase, abort_flag, DEVERR_TIMEOUT_MMA, C)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            // the MMA reads 128 weight rows: past p.rows they are whatever the ring holds, and
            // only lanes that nothing reads see them
            const uint32_t sw = base + stage * stage_bytes;
            const int nk = min(strm::STEP, s1 - kb);
#pragma unroll
            for (int h = 0; h < strm::STEP; ++h) {
              if (h >= nk) break;
              const uint64_t adesc = ptx::smem_desc_sw128(sw + h * w_bytes, 16, 1024);
              const uint64_t bdesc = ptx::smem_desc_sw128(sw + strm::STEP * w_bytes + h * x_bytes, 16, 1024);
#pragma unroll
              for (int kk = 0; kk < BK / UMMA_K; ++kk) {
                const uint32_t accum = (kb != s0 || h != 0 || kk != 0) ? 1u : 0u;
                if constexpr (KIND == KIND_BF16)
                  ptx::umma_bf16(d_tmem, adesc + kk * (UMMA_K / 16), bdesc + kk * (UMMA_K / 16), idesc, accum);
                else
                  ptx::umma_i8(d_tmem, adesc + kk * (UMMA_K / 16), bdesc + kk * (UMMA_K / 16), idesc, accum);
              }
            }
            ptx::umma_commit(empty_bar(stage));
            if (kb + nk >= s1) ptx::umma_commit(tfull_bar(a));
          }
          __syncwarp();
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
      }
    }
    __syncwarp();
    if (SPLIT) ptx::cluster_arrive();
  } else {
    // ---------------- epilogue ----------------
    const int q = warp & 3;     // TMEM lane quadrant
    const Epi& ep = p.ep;
    const int w4 = warp - 2;
    const int slot = XT / C;    // tokens of a rank's slice at most
    const uint32_t tmem_q = tmem_base + ((uint32_t)(q * 32) << 16);
    const uint32_t send_q = send + (uint32_t)(q * XT) * 128u;  // this warp's part
    int it = 0, xc = 0;         // accumulators read, exchanges that came in
    bool ok = true, arrived = false;
    for (int tile = cid; ok && tile < T; tile += nclusters) {
      const Tile t = tile_of(p, tb, tile, p.band);
      const bool last_tile = tile + nclusters >= T;
      const int f0 = t.wb * p.feats;
      Feat<GATED> ff;
      Lane<GATED> fl;
      if (SPLIT) {
        const int f4 = 4 * (GATED ? lane % 16 : lane);
        load_feat<KIND, GATED>(ep, t.e, f4 < p.feats ? f0 + f4 : ep.N, ff);
      }
      else fl = lane_of<KIND, GATED>(ep, t.e, f0, p.rows, q, lane);
      // One exchange: tokens x0 .. x0 + xn of the tile, whose sums this warp has laid out.
      auto exchange = [&](int x0, int xn) {
        const uint32_t phase = (uint32_t)(xc & 1);
        const int per = (xn + C - 1) / C;          // rank r finishes tokens r * per ..
        const int mine = max(0, min(per, xn - rank * per));
        const int row0 = t.t0 + x0 + rank * per;
        // the scales of this rank's tokens (32 at most), while the copies are under way
        float sxl = 1.f;
        if (KIND == KIND_I8 && lane < mine) sxl = __ldg(ep.sx + row0 + lane);
        if (threadIdx.x == 64)
          ptx::mbar_arrive_expect_tx(rfull_bar, (uint32_t)(mine * C * WROWS) * 4u);
        ptx::fence_proxy_async_smem();             // the layout -> visible to the bulk copies
        __syncwarp();
        if (lane < C) {
          const int theirs = max(0, min(per, xn - lane * per));
          if (theirs > 0)
            ptx::bulk_copy_cluster(ptx::map_to_rank(recv + (uint32_t)((rank * 4 + q) * slot) * 128u, lane),
                                   send_q + (uint32_t)(lane * per) * 128u, (uint32_t)theirs * 128u,
                                   ptx::map_to_rank(rfull_bar, lane));
        }
        ok = ptx::mbar_wait_acquire_cluster(rfull_bar, phase, abort_flag, p.wait_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        ++xc;
        const bool last = last_tile && x0 + xn >= t.n;
        if (last) {  // this warp has made its last access to another CTA
          ptx::cluster_arrive();
          arrived = true;
        }
        // this lane's four features in a source's [warp][slot][32] words: gated, gate rows and
        // up rows by turns of 8
        const int fq = GATED ? (lane % 16) / 4 : lane / 8;
        const int fw = GATED ? lane / 2 % 2 * 16 + lane % 2 * 4 : (lane % 8) * 4;
        with_act(ep.act, [&](auto act) {
          const int step = GATED ? 8 : 4;
          for (int l0 = GATED ? w4 * 2 : w4; l0 < mine; l0 += step) {  // warp-uniform
            const int l = l0 + (GATED ? lane / 16 : 0);
            const float sx = __shfl_sync(0xffffffffu, sxl, l & 31);
            if (l >= mine || ff.n >= ep.N) continue;
            float res[4];
            load_residual<F32>(ep, row0 + l, ff.n, res);
            uint32_t g[4] = {0u, 0u, 0u, 0u}, u[4] = {0u, 0u, 0u, 0u};
            for (int c = 0; c < C; ++c) {
              const uint32_t at = recv + (uint32_t)(((c * 4 + fq) * slot + l) * 32 + fw) * 4u;
              add_words<KIND>(g, ld_shared_v4(at));
              if (GATED) add_words<KIND>(u, ld_shared_v4(at + 8 * 4));
            }
            finish4<KIND, GATED, F32, decltype(act)::value>(ep, ff, row0 + l, sx, g, u, res);
          }
        });
        __syncwarp();
        // The loads above have returned (their values went into the outputs), so the arrival
        // needs no release: a cluster-scope one waited for the output stores, 2000 cycles a
        // tile.
        if (!last && lane < C) ptx::mbar_arrive_remote(ptx::map_to_rank(rempty_bar, lane));
      };
      // Before this warp lays out anything: every rank has read the exchange before (and with
      // that, the copies out of this warp's layout are done).
      auto layout_free = [&]() {
        ok = ptx::mbar_wait_acquire_cluster(rempty_bar, (uint32_t)(xc & 1) ^ 1u, abort_flag, p.wait_ns);
        ok = __all_sync(0xffffffffu, ok);
      };
      // 16 tokens' sums of this lane's weight row: finished here, or laid out (and exchanged
      // when the layout is full or the tile ends)
      auto emit = [&](int c, const uint32_t (&r)[16]) {
        if constexpr (!SPLIT) {
          with_act(ep.act, [&](auto act) {
            finish_chunk<KIND, GATED, F32, decltype(act)::value>(ep, fl, t.t0 + c, t.n - c, lane, r, [] {});
          });
        } else {
          const int x0 = c / XT * XT;
          if (c == x0) layout_free();
          if (!ok) return;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            st_shared_u32(send_q + (uint32_t)((c - x0 + j) * 32 + lane) * 4u, r[j]);
          if (c + 16 >= t.n || c + 16 == x0 + XT) exchange(x0, min(t.n - x0, XT));
        }
      };
      // SEG: the running sums of the segments before live in TMEM columns 2 TOK ..
      const int seg = SEG ? p.seg_kb : p.num_k_blocks;
      for (int s0 = kb0; ok && s0 < kb1; s0 += seg, ++it) {
        const int a = it & 1;
        ok = ptx::mbar_wait(p.hold ? drain_bar : tfull_bar(a),
                            p.hold ? 0u : (uint32_t)((it >> 1) & 1), abort_flag, p.wait_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ptx::tc_fence_after();
        const bool last_seg = !SEG || s0 + seg >= kb1;
        for (int c = 0; ok && c < t.n; c += 16) {
          uint32_t r[16];
          ptx::tmem_ld_32x32b_x16(tmem_q + (uint32_t)(a * TOK + c), r);
          if (SEG) add_running(tmem_q + (uint32_t)(2 * TOK + c), s0 > kb0, r);
          else ptx::tmem_wait_ld();
          if (!last_seg) ptx::tmem_st_32x32b_x16(tmem_q + (uint32_t)(2 * TOK + c), r);
          if (c + 16 >= t.n) {  // the accumulator is read: free before the last exchange
            if (SEG) ptx::tmem_wait_st();
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(tempty_bar(a));
          }
          if (last_seg) emit(c, r);
        }
      }
      if (!ok && lane == 0 && !*abort_flag)
        report_cluster(p.err, DEVERR_TIMEOUT_EPILOGUE, abort_flag, C);
    }
    if (SPLIT && !arrived) {
      // Given up: until the exchange that was next has come in whole, or for as long as a copy
      // could conceivably take.  A warp that has sent its sums waits here or in the exchange for
      // the other ranks', so no rank leaves while a copy from it or to it is under way.
      if (!ok) ptx::mbar_wait_acquire_cluster(rfull_bar, (uint32_t)(xc & 1), nullptr, DRAIN_NS);
      __syncwarp();
      ptx::cluster_arrive();
    }
  }

  ptx::tc_fence_before();
  const bool gave_up = __syncthreads_or(*abort_flag);
  ptx::tc_fence_after();
  // Nobody here issues any more.  A flag that another rank raises later finds this CTA's work
  // done: its epilogue has seen every accumulator.
  if (gave_up)
    strm::drain(p, bar_base, *reinterpret_cast<volatile long long*>(gbar + COUNT_AT), drain_bar, abort_flag);
  if (warp == 1) {
    __syncwarp();
    ptx::tmem_dealloc(tmem_base, tmem_cols);
  }
  if (SPLIT) ptx::cluster_wait();  // no CTA leaves while another may write or arrive in it
}

// ---- host side -----------------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// Byte map of `rows` rows of `width` bytes, `pitch` apart; boxes of 128 bytes x box_rows.
static bool make_map(CUtensorMap* m, const void* ptr, uint64_t width, uint64_t rows,
                     uint64_t pitch, uint32_t box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {width, rows};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {BK, box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The gated weights [E][2][N][K] as (k, row of 8, gate / up, block of 8 features, expert);
// features past the last whole block are outside the map.  Boxes of 128 bytes x 8 rows x both
// halves x `blocks` blocks: 16 * blocks weight rows, gate and up by turns of 8.
static bool make_gated_map(CUtensorMap* m, const void* ptr, uint64_t width, int N, int E,
                           int blocks) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[5] = {width, 8, 2, (cuuint64_t)(N / 8), (cuuint64_t)E};
  cuuint64_t strides[4] = {width, (cuuint64_t)N * width, 8 * width, 2 * (cuuint64_t)N * width};
  cuuint32_t box[5] = {BK, 8, 2, (cuuint32_t)blocks, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(ptr), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

using Kern = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap,
                      const Params);
// The kernels of an operand kind, summed in segments or not, for one output type.
struct Kerns {
  Kern pair[2], stream[2][2];  // [gated], [gated][K split]
};
template <int KIND, bool SEG, bool F32>
static constexpr Kerns kerns_of() {
  return {{linear_pair_kernel<KIND, false, SEG, F32>, linear_pair_kernel<KIND, true, SEG, F32>},
          {{linear_stream_kernel<KIND, false, SEG, F32, false>, linear_stream_kernel<KIND, false, SEG, F32, true>},
           {linear_stream_kernel<KIND, true, SEG, F32, false>, linear_stream_kernel<KIND, true, SEG, F32, true>}}};
}
static const Kerns kInt8[2] = {kerns_of<KIND_I8, false, false>(), kerns_of<KIND_I8, false, true>()};
static const Kerns kBf16[2] = {kerns_of<KIND_BF16, false, false>(), kerns_of<KIND_BF16, false, true>()};
static const Kerns kBf16Seg[2] = {kerns_of<KIND_BF16, true, false>(), kerns_of<KIND_BF16, true, true>()};
static const Kerns* const kAll[] = {&kInt8[0], &kInt8[1], &kBf16[0], &kBf16[1], &kBf16Seg[0], &kBf16Seg[1]};

static_assert(pair::SEG_TOK <= 128 && 3 * strm::TOK <= 512, "TMEM columns of SEG");

// The tensor cores add each MMA's products to the fp32 accumulator by truncation, so a sum
// over K shrinks by about 9e-10 of itself a value of K (measured: 2.1e-6 at K = 2048, 1.2e-5 at
// 11008).  A bf16 output's half step is 33 times that or more up to K = SEG_K; beyond, and for
// fp32 outputs from the first, the SEG kernels run, which start a new accumulator every SEG_KB k-blocks (512 values, 4.7e-7) and add the pieces rounding to
// nearest, into running sums in TMEM (in registers, the unrolled code ran from outside the
// instruction cache: 170 us instead of 112 for 6001 x 1544 x 2048 over 64 experts).
constexpr int SEG_KB = 8;
constexpr int SEG_K = 65536;
static_assert(SEG_KB % strm::STEP == 0, "a segment is whole stages");

// Opts the kernels in to the whole shared memory once a device, and asks how many clusters of
// 1, 2, 4 and 8 streaming CTAs the device holds at once.
struct DeviceSetup {
  bool ready = false;
  int clusters[4] = {0, 0, 0, 0};
};

static qgemm_status device_setup(qgemm_stream_s* s, const DeviceSetup** out) {
  static std::mutex mu;
  static DeviceSetup setup[64];
  const int ord = s->dev->ordinal;
  if (ord < 0 || ord >= 64) return fail(QGEMM_ERR_UNSUPPORTED, "device ordinal %d >= 64", ord);
  std::lock_guard<std::mutex> lock(mu);
  DeviceSetup& d = setup[ord];
  if (!d.ready) {
    for (const Kerns* k : kAll)
      for (int g = 0; g < 2; ++g) {
        cudaError_t e = cudaFuncSetAttribute(k->pair[g], cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
        for (int sp = 0; sp < 2 && e == cudaSuccess; ++sp)
          e = cudaFuncSetAttribute(k->stream[g][sp], cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(linear)");
      }
    for (int i = 0; i < 4; ++i) {
      const int c = 1 << i;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(s->dev->sm_count / c * c);
      cfg.blockDim = dim3(strm::THREADS);
      cfg.dynamicSmemBytes = SMEM_MAX;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = c;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kInt8[0].stream[0][1], &cfg);
      if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveClusters(linear)");
      d.clusters[i] = n;
    }
    d.ready = true;
  }
  *out = &d;
  return QGEMM_OK;
}

}  // namespace lin

bool linear_tcgen05_supported(const qgemm_device_s* d, const LinArgs& a, const char** why) {
  auto no = [&](const char* w) { if (why) *why = w; return false; };
  const int es = a.kind == KIND_I8 ? 1 : 2;
  if (!d->tcgen05) return no("device is not sm_100 (tcgen05 unavailable)");
  if (d->smem_optin < (size_t)lin::SMEM_MAX) return no("not enough shared memory per block");
  if (a.K <= 0) return no("K == 0");
  // tiles, rows and the bytes of a row are counted in 32 bits
  if (a.K > (1 << 29)) return no("K > 2^29");
  if (a.M > (1 << 30) || ((long long)a.M / 16 + a.E) * (a.N / 64 + 1) > (1ll << 30))
    return no("more than 2^30 tiles");
  if (((long long)a.K * es) % 16 != 0) return no("K is not a multiple of 16 bytes");
  if ((a.ldx * es) % 16 != 0) return no("the rows of x are not a multiple of 16 bytes apart");
  if (!aligned((uint64_t)a.x, 16) || !aligned((uint64_t)a.w, 16))
    return no("x and w must be 16-byte aligned");
  return true;
}

qgemm_status launch_linear_tcgen05(qgemm_stream_s* s, const LinArgs& a) {
  using namespace lin;
  const DeviceSetup* ds = nullptr;
  qgemm_status st = device_setup(s, &ds);
  if (st != QGEMM_OK) return st;
  const int es = a.kind == KIND_I8 ? 1 : 2, os = a.out_dtype == QGEMM_F32 ? 4 : 2;
  const int sms = s->dev->sm_count;
  Params p = {};
  p.ep.sx = a.sx; p.ep.sw = a.sw; p.ep.bias = a.bias; p.ep.residual = a.residual;
  p.ep.out = a.out; p.ep.ldr = a.ldr; p.ep.ldc = a.ldc;
  p.ep.N = a.N; p.ep.nw = a.gated ? 2 * a.N : a.N;
  p.ep.act = a.act;
  p.ep.vec = aligned((uint64_t)a.out, 4 * os) && a.ldc % 4 == 0 &&
             (!a.residual || (aligned((uint64_t)a.residual, 4 * os) && a.ldr % 4 == 0));
  p.ep.vec2 = a.out_dtype == QGEMM_BF16 && aligned((uint64_t)a.out, 4) && a.ldc % 2 == 0 &&
              (!a.residual || (aligned((uint64_t)a.residual, 4) && a.ldr % 2 == 0));
  p.offsets = a.offsets;
  p.E = a.E; p.M = a.M;
  p.num_k_blocks = (int)(((long long)a.K * es + BK - 1) / BK);
  p.err = s->dev->d_err;
  p.bad = s->index_word;
  p.hold = s->dev->hold_split;
  p.wait_ns = s->dev->wait_ns;
  p.rows = WROWS;
  const int table = ((3 * a.E + 1) * 4 + 15) / 16 * 16;
  // rows of a group if they are spread evenly; the kernels take any spread
  const int groups = a.E < a.M ? a.E : a.M;
  const int avg = (a.M + groups - 1) / groups;
  p.seg_kb = SEG_KB;
  const int f32 = a.out_dtype == QGEMM_F32;
  const bool seg = a.kind == KIND_BF16 && p.num_k_blocks > SEG_KB && (f32 || a.K > SEG_K);
  const Kerns& kerns = a.kind == KIND_I8 ? kInt8[f32] : seg ? kBf16Seg[f32] : kBf16[f32];
  // ---- the streaming kernel's cut of the work ----
  const int cap = strm::TOK;
  int tok_max, box;
  if (a.offsets) {
    // tokens of a tile: twice the even share, so that a moderate skew stays in one tile
    const int want = 2 * avg < a.M ? 2 * avg : a.M;
    tok_max = want <= 16 ? 16 : want <= 32 ? 32 : want <= 64 ? 64 : cap;
    box = tok_max < 32 ? tok_max : 32;
  } else {  // equal blocks, each one box
    const int blocks = (a.M + cap - 1) / cap;
    tok_max = ((a.M + blocks - 1) / blocks + 15) / 16 * 16;
    box = tok_max;
  }
  // K over c CTAs, and weight rows a tile, so that the rounds come out full.  A round takes the
  // longer of its k-blocks' copies and MMAs in a CTA (0.17 us each and more with more tokens,
  // 0.22 gated) and of its weights from HBM (6.2 TB/s from all SMs), and a quarter of the
  // other; a cut of K adds an exchange.  Measured against every choice at 9 shapes of 1024 to
  // 11008 features and 1 to 100 tokens (1 x 4096 x 4096 bf16: 8.9 us with c = 4, 10.1 with 2,
  // 14.7 with 1; 33 x 11008 x 4096 int8 gated: 21.2 us with c = 2 and 112 rows, 22.5 with c = 1
  // and 128).
  const int ksteps = (p.num_k_blocks + strm::STEP - 1) / strm::STEP;
  const int nblk = (avg + tok_max - 1) / tok_max;
  const long long groups_tok = (long long)groups * nblk;
  const double tok = avg < tok_max ? avg : tok_max;
  const double kb_us = (a.gated ? 0.22 : 0.17) + 0.0009 * tok;
  auto both = [](double x, double y) { return x > y ? x + 0.25 * y : y + 0.25 * x; };
  // a stage holds tok_max token rows and is filled in whole boxes
  if (tok_max % box != 0 || tok_max > strm::TOK || box > 128)
    return fail(QGEMM_ERR_UNSUPPORTED, "token tile %d in boxes of %d", tok_max, box);
  double stream_us = 0;
  int pick = 0, rows = WROWS;
  for (int i = 0; i < 4; ++i) {
    const int c = 1 << i;
    if (ds->clusters[i] < 1 || c > ksteps) continue;
    for (int r = WROWS; r >= 64; r -= 16) {
      // fewer rows a tile pay only where the counts are known and the epilogue is short (6001
      // rows over 64 experts, fp32 out: 100 us with 128 rows, 118 with 112)
      if (r < WROWS && (a.offsets || tok > 64)) continue;
      const int feats = a.gated ? r / 2 : r;
      const long long tiles = groups_tok * ((a.N + feats - 1) / feats);
      // a cut of K only where tiles are scarce: with many, its exchange is paid for every one
      // (those 6001 rows: 208 us with c = 2, 108 with c = 1)
      if (c > 1 && tiles >= 2 * sms) continue;
      const long long full = tiles / ds->clusters[i], rest = tiles - full * ds->clusters[i];
      double cta = (ksteps + c - 1) / c * strm::STEP * kb_us + 0.1;
      if (c > 1 && cta < 1.2 + 0.03 * tok) cta = 1.2 + 0.03 * tok;  // an exchange a tile
      const int ctas = c * ds->clusters[i];
      // (the token blocks of a group run side by side and share their weights in L2)
      const double tile_hbm = (double)r * a.K * es / nblk / (6.2e6 * (ctas < sms ? ctas : sms) / sms);
      const double us = (r < WROWS ? 1.03 : 1.0) * (full * both(cta, ds->clusters[i] * tile_hbm) +
                        (rest ? both(cta, rest * tile_hbm) : 0.0)) + (c > 1 ? 0.6 + 0.05 * tok : 0.0);
      if (stream_us == 0 || us < stream_us) { stream_us = us; pick = i; rows = r; }
    }
  }
  // ---- the pair kernel's time, in the same terms ----
  const int pair_feats = a.gated ? 128 : 256, pair_tok = seg ? pair::SEG_TOK : pair::TOK;
  const int pairs = sms / 2;
  const long long pair_blocks = (avg + pair_tok - 1) / pair_tok;
  const long long pair_tiles = groups * pair_blocks * ((a.N + pair_feats - 1) / pair_feats);
  const double pair_n = (double)avg / pair_blocks;
  auto pair_round = [&](long long n, double toks) {
    return p.num_k_blocks * both(0.24 + 0.0005 * toks, n * 2 * W_BYTES / 6.2e6);
  };
  const long long pfull = pair_tiles / pairs, prest = pair_tiles - pfull * pairs;
  // (SEG costs the pair kernel half its time more: 142 us against 100 streaming for those rows)
  const double pair_us = 0.5 + (seg ? 1.5 : 1.0) * pfull * pair_round(pairs, pair_n) +
      (prest ? (seg ? 1.5 : 1.0) * pair_round(prest, pair_n / (pairs / prest < 4 ? pairs / prest : 4)) : 0.0);
  // Which kernel (measured, bf16 4096 x 4096: 64 rows 12.2 us streaming, 19.5 in pairs; 256 rows
  // 19.6 and 20.6; 512 rows 32 and 25; 11008 x 4096: 96 rows 22.7 and 24.7; 128 rows 31.5 and
  // 25.6).
  const bool use_pair = pair_us < stream_us;

  cudaLaunchConfig_t cfg = {};
  cfg.stream = s->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  Kern kern;
  if (use_pair) {
    p.tok_max = pair_tok;
    // A band's tokens stay in L2 while all weights pass by once: the fewer bands, the fewer
    // times the weights come from HBM, whose power the tensor cores then lack (int8 8192 x
    // 28672 x 4096: 805 us with 32 MB of tokens a band, 815 with 16, 825 with 8; bf16 4096 x
    // 4096 x 11008: 318 us with 45 MB, 327 with 90 or 22).
    const long long block_bytes = (long long)p.tok_max * a.K * es;
    p.band = (int)(block_bytes > (48 << 20) ? 1 : (48 << 20) / block_bytes);
    p.tok_round = 32;
    p.feats = a.gated ? 64 : 128;
    p.num_w_blocks = (a.N + 2 * p.feats - 1) / (2 * p.feats);
    box = 128;
    const int fixed = BAR_BYTES + table + 1024;
    p.stages = (SMEM_MAX - fixed) / pair::STAGE_BYTES;
    cfg.dynamicSmemBytes = (size_t)fixed + (size_t)p.stages * pair::STAGE_BYTES;
    cfg.gridDim = dim3(sms / 2 * 2);
    cfg.blockDim = dim3(pair::THREADS);
    kern = kerns.pair[a.gated];
  } else {
    p.tok_max = tok_max;
    p.box = box;
    const int cols = (seg ? 3 : 2) * tok_max;  // accumulators, running sums
    p.tmem_cols = cols <= 32 ? 32 : cols <= 64 ? 64 : cols <= 128 ? 128 : cols <= 256 ? 256 : 512;
    p.tok_round = 16;
    p.band = 1 << 20;  // token blocks run fastest: neighbours share the weights
    p.csize = 1 << pick;
    p.rows = rows;
    p.feats = a.gated ? rows / 2 : rows;
    p.num_w_blocks = (a.N + p.feats - 1) / p.feats;
    const int stage = strm::STEP * (rows + tok_max) * BK;
    const int xt = tok_max < strm::XTOK ? tok_max : strm::XTOK;
    // the last stage's MMAs read a whole weight tile, past the ring if rows is small
    const int fixed = (p.csize > 1 ? 2 * xt * WROWS * 4 : 0) + BAR_BYTES + table + 1024 +
                      (stage < 2 * W_BYTES ? 2 * W_BYTES - stage : 0);
    p.stages = (SMEM_MAX - fixed) / stage;
    if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
    cfg.dynamicSmemBytes = (size_t)fixed + (size_t)p.stages * stage;
    // as many clusters as fit (the counts of the experts are not known here: at least one
    // tile each is not promised)
    const long long most = (long long)p.num_w_blocks * (a.M / tok_max + groups);
    const long long clusters = most < ds->clusters[pick] ? most : ds->clusters[pick];
    cfg.gridDim = dim3((unsigned)(clusters * p.csize));
    cfg.blockDim = dim3(strm::THREADS);
    kern = kerns.stream[a.gated][p.csize > 1];
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.csize;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  // weight boxes: all of a CTA's rows, or (gated) runs of 8 and the 5-D map over them
  CUtensorMap tmW, tmG, tmX;
  if (!make_map(&tmW, a.w, (uint64_t)a.K * es, (uint64_t)a.E * p.ep.nw, (uint64_t)a.K * es,
                a.gated ? 8 : p.rows))
    return fail(QGEMM_ERR_CUDA, "cuTensorMapEncodeTiled failed for the weights");
  tmG = tmW;  // not used where no tile of the layer lies in whole blocks of 8 features
  if (a.gated && a.N / 8 >= p.rows / 16 &&
      !make_gated_map(&tmG, a.w, (uint64_t)a.K * es, a.N, a.E, p.rows / 16))
    return fail(QGEMM_ERR_CUDA, "cuTensorMapEncodeTiled failed for the gated weights");
  if (!make_map(&tmX, a.x, (uint64_t)a.K * es, (uint64_t)a.M, (uint64_t)a.ldx * es, box))
    return fail(QGEMM_ERR_CUDA, "cuTensorMapEncodeTiled failed for x");
  CUtensorMap tmXs = tmX;  // the pair kernel's boxes for part tiles
  if (use_pair && !make_map(&tmXs, a.x, (uint64_t)a.K * es, (uint64_t)a.M, (uint64_t)a.ldx * es, pair::BOX))
    return fail(QGEMM_ERR_CUDA, "cuTensorMapEncodeTiled failed for x");
  return cuda_fail(cudaLaunchKernelEx(&cfg, kern, tmW, tmG, tmX, tmXs, p), "linear launch");
}

}  // namespace qg
