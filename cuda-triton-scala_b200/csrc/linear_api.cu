// linear_api.cu -- the extern "C" boundary of the linear layers with their epilogue and of
// the routing around the experts (include/qgemm.h): argument checks and dispatch.
#include <cuda_runtime.h>

#include "internal.h"

using namespace qg;

#define QG_TRY(expr)                     \
  do {                                   \
    qgemm_status _st = (expr);           \
    if (_st != QGEMM_OK) return _st;     \
  } while (0)

namespace {

// Addresses [p, p + rows * pitch) touched by a row-major buffer whose rows hold `width`
// bytes `pitch` bytes apart (rows > 0).
struct Range {
  uint64_t lo, hi;
};

Range range_of(uint64_t p, long long rows, unsigned long long pitch, unsigned long long width) {
  return {p, p + (unsigned long long)(rows - 1) * pitch + width};
}

bool overlap(const Range& a, const Range& b) { return a.lo < b.hi && b.lo < a.hi; }

// `rows` rows of `width` bytes, `pitch` bytes apart.
struct Rows {
  uint64_t p;
  long long rows;
  unsigned long long pitch, width;
};

// Whether two buffers share a byte.  Exact for rows of one pitch (columns of one wider buffer) and
// where one is a single run; else the ranges from first to last byte are compared.
bool overlap(const Rows& a, const Rows& b) {
  if (!overlap(range_of(a.p, a.rows, a.pitch, a.width), range_of(b.p, b.rows, b.pitch, b.width)))
    return false;
  if (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) return true;
  const unsigned long long pitch = a.rows > 1 ? a.pitch : b.pitch;
  if (a.rows == 1 && b.rows == 1) return true;
  const Rows& first = a.p <= b.p ? a : b;
  const Rows& second = a.p <= b.p ? b : a;
  const unsigned long long d = (second.p - first.p) % pitch;
  // a single run that begins first and reaches the other holds its first byte
  if (first.rows == 1) return true;
  return d < first.width || d + second.width > pitch;
}

qgemm_status need(uint64_t p, uint64_t align, const char* name) {
  if (p == 0) return fail(QGEMM_ERR_INVALID_ARG, "%s is null", name);
  if (!aligned(p, align))
    return fail(QGEMM_ERR_BAD_ALIGN, "%s is not %llu-byte aligned", name, (unsigned long long)align);
  return QGEMM_OK;
}

qgemm_status dtype_ok(int t, const char* name) {
  if (t != QGEMM_F32 && t != QGEMM_BF16)
    return fail(QGEMM_ERR_INVALID_ARG, "%s %d is neither QGEMM_F32 nor QGEMM_BF16", name, t);
  return QGEMM_OK;
}

// Rows, features and values a row at most: loops and tile counts of the kernels step past the end
// by up to a block's width in 32 bits.
constexpr int kMostSize = 1 << 30;

qgemm_status linear_entry(qgemm_stream_t s, int kind, uint64_t x, int ldx, uint64_t w,
                          uint64_t sx, uint64_t sw, uint64_t bias, uint64_t residual, int ldr,
                          uint64_t offsets, bool experts, uint64_t out, int out_dtype, int ldc,
                          int E, int M, int N, int K, int act, int gated, int algo) {
  if (M < 0 || N < 0 || K < 0)
    return fail(QGEMM_ERR_INVALID_ARG, "negative size M=%d N=%d K=%d", M, N, K);
  if (M > kMostSize || N > kMostSize || K > kMostSize)
    return fail(QGEMM_ERR_UNSUPPORTED, "size past 2^30: M=%d N=%d K=%d", M, N, K);
  if (E < 1 || E > kMaxExperts)
    return fail(QGEMM_ERR_INVALID_ARG, "E %d outside [1, %d]", E, kMaxExperts);
  QG_TRY(dtype_ok(out_dtype, "out_dtype"));
  if (act < QGEMM_ACT_NONE || act > QGEMM_ACT_SILU)
    return fail(QGEMM_ERR_INVALID_ARG, "bad activation %d", act);
  if (gated != 0 && gated != 1) return fail(QGEMM_ERR_INVALID_ARG, "gated %d is not 0 or 1", gated);
  if (algo < QGEMM_ALGO_AUTO || algo > QGEMM_ALGO_SIMT)
    return fail(QGEMM_ERR_INVALID_ARG, "bad algo %d", algo);
  if (M == 0 || N == 0) return enter(s);
  if (ldx < K) return fail(QGEMM_ERR_INVALID_ARG, "row pitch %d of x < K %d", ldx, K);
  if (ldc < N) return fail(QGEMM_ERR_INVALID_ARG, "ldc %d < N %d", ldc, N);
  if (residual && ldr < N) return fail(QGEMM_ERR_INVALID_ARG, "ldr %d < N %d", ldr, N);
  const int es = kind == KIND_I8 ? 1 : 2, os = out_dtype == QGEMM_F32 ? 4 : 2;
  const long long nw = gated ? 2ll * N : N;
  if (nw * E > 0x7fffffffll)
    return fail(QGEMM_ERR_UNSUPPORTED, "%lld weight rows exceed 2^31 - 1", nw * E);
  if (kind == KIND_I8 && K > 131071)
    return fail(QGEMM_ERR_UNSUPPORTED, "K %d > 131071: int32 sums could overflow", K);
  if (K > 0) {
    QG_TRY(need(x, es, kind == KIND_I8 ? "A" : "x"));
    QG_TRY(need(w, es, kind == KIND_I8 ? "B" : "w"));
  }
  if (kind == KIND_I8) {
    QG_TRY(need(sx, 4, "sA"));
    QG_TRY(need(sw, 4, "sB"));
  }
  QG_TRY(need(out, os, "out"));
  if (bias) QG_TRY(need(bias, 4, "bias"));
  if (residual) QG_TRY(need(residual, os, "residual"));
  if (experts) QG_TRY(need(offsets, 4, "offsets"));
  const auto rows = [](uint64_t p, long long n, unsigned long long pitch, unsigned long long width) {
    return Rows{p, n, pitch, width};
  };
  const auto run = [](uint64_t p, unsigned long long bytes) { return Rows{p, 1, bytes, bytes}; };
  const Rows o = rows(out, M, (unsigned long long)ldc * os, (unsigned long long)N * os);
  if (K > 0 && (overlap(o, rows(x, M, (unsigned long long)ldx * es, (unsigned long long)K * es)) ||
                overlap(o, run(w, (unsigned long long)(nw * E) * K * es))))
    return fail(QGEMM_ERR_INVALID_ARG, "out overlaps an operand");
  if ((kind == KIND_I8 && (overlap(o, run(sx, 4ull * M)) || overlap(o, run(sw, 4ull * nw * E)))) ||
      (bias && overlap(o, run(bias, 4ull * nw * E))) ||
      (experts && overlap(o, run(offsets, 4ull * (E + 1)))))
    return fail(QGEMM_ERR_INVALID_ARG, "out overlaps the scales, the bias or the offsets");
  if (residual && !(residual == out && ldr == ldc) &&
      overlap(o, rows(residual, M, (unsigned long long)ldr * os, (unsigned long long)N * os)))
    return fail(QGEMM_ERR_INVALID_ARG, "out overlaps the residual without being it");
  QG_TRY(enter(s));
  LinArgs a;
  a.kind = kind;
  a.x = reinterpret_cast<const void*>(x);
  a.w = reinterpret_cast<const void*>(w);
  a.sx = reinterpret_cast<const float*>(sx);
  a.sw = reinterpret_cast<const float*>(sw);
  a.bias = reinterpret_cast<const float*>(bias);
  a.residual = reinterpret_cast<const void*>(residual);
  a.out = reinterpret_cast<void*>(out);
  a.offsets = experts ? reinterpret_cast<const int*>(offsets) : nullptr;
  a.E = experts ? E : 1;
  a.M = M; a.N = N; a.K = K;
  a.ldx = ldx; a.ldr = ldr; a.ldc = ldc;
  a.out_dtype = out_dtype;
  a.act = act;
  a.gated = gated;
  const char* why = nullptr;
  const bool tc = linear_tcgen05_supported(s->dev, a, &why);
  if (algo == QGEMM_ALGO_TCGEN05 && !tc)
    return fail(QGEMM_ERR_UNSUPPORTED, "tensor-core linear layer unavailable: %s", why);
  if (tc && algo != QGEMM_ALGO_SIMT) return launch_linear_tcgen05(s, a);
  return launch_linear_simt(s, a);
}

// Sizes, types and pointers that dispatch and combine share.
qgemm_status rows_entry(qgemm_stream_t s, int in_dtype, int T, int k, int W, int R,
                        const char* width) {
  if (T < 0 || W < 0 || R < 0)
    return fail(QGEMM_ERR_INVALID_ARG, "negative size T=%d %s=%d R=%d", T, width, W, R);
  if (k < 1 || k > 64) return fail(QGEMM_ERR_INVALID_ARG, "k %d outside [1, 64]", k);
  if ((long long)T * k > 0x7fffffffll)
    return fail(QGEMM_ERR_UNSUPPORTED, "T * k exceeds 2^31 - 1");
  if (T > kMostSize || W > kMostSize)
    return fail(QGEMM_ERR_UNSUPPORTED, "size past 2^30: T=%d %s=%d", T, width, W);
  return dtype_ok(in_dtype, "in_dtype");
}

}  // namespace

extern "C" {

qgemm_status qgemm_linear_bf16_nk(qgemm_stream_t s, uint64_t x, int ldx, uint64_t w,
                                  uint64_t bias, uint64_t residual, int ldr, uint64_t out,
                                  int out_dtype, int ldc, int M, int N, int K, int act, int gated,
                                  int algo) {
  return linear_entry(s, KIND_BF16, x, ldx, w, 0, 0, bias, residual, ldr, 0, false, out,
                      out_dtype, ldc, 1, M, N, K, act, gated, algo);
}

qgemm_status qgemm_w8a8_linear(qgemm_stream_t s, uint64_t A, int lda, uint64_t B, uint64_t sA,
                               uint64_t sB, uint64_t bias, uint64_t residual, int ldr,
                               uint64_t out, int out_dtype, int ldc, int M, int N, int K, int act,
                               int gated, int algo) {
  return linear_entry(s, KIND_I8, A, lda, B, sA, sB, bias, residual, ldr, 0, false, out,
                      out_dtype, ldc, 1, M, N, K, act, gated, algo);
}

qgemm_status qgemm_expert_linear_bf16_nk(qgemm_stream_t s, uint64_t x, int ldx, uint64_t w,
                                         uint64_t bias, uint64_t offsets, uint64_t out,
                                         int out_dtype, int ldc, int E, int M, int N, int K,
                                         int act, int gated, int algo) {
  return linear_entry(s, KIND_BF16, x, ldx, w, 0, 0, bias, 0, 0, offsets, true, out, out_dtype,
                      ldc, E, M, N, K, act, gated, algo);
}

qgemm_status qgemm_w8a8_expert_linear(qgemm_stream_t s, uint64_t A, int lda, uint64_t B,
                                      uint64_t sA, uint64_t sB, uint64_t bias, uint64_t offsets,
                                      uint64_t out, int out_dtype, int ldc, int E, int M, int N,
                                      int K, int act, int gated, int algo) {
  return linear_entry(s, KIND_I8, A, lda, B, sA, sB, bias, 0, 0, offsets, true, out, out_dtype,
                      ldc, E, M, N, K, act, gated, algo);
}

qgemm_status qgemm_route_topk(qgemm_stream_t s, uint64_t logits, int in_dtype, uint64_t weights,
                              uint64_t experts, uint64_t offsets, uint64_t rows, int T, int E,
                              int k, int renormalize) {
  if (T < 0) return fail(QGEMM_ERR_INVALID_ARG, "negative size T=%d", T);
  if (E < 1 || E > kMaxExperts)
    return fail(QGEMM_ERR_INVALID_ARG, "E %d outside [1, %d]", E, kMaxExperts);
  if (k < 1 || k > E || k > 64)
    return fail(QGEMM_ERR_INVALID_ARG, "k %d outside [1, min(E, 64)]", k);
  if (renormalize != 0 && renormalize != 1)
    return fail(QGEMM_ERR_INVALID_ARG, "renormalize %d is not 0 or 1", renormalize);
  if ((long long)T * k > 0x7fffffffll)
    return fail(QGEMM_ERR_UNSUPPORTED, "T * k exceeds 2^31 - 1");
  if (T > kMostSize) return fail(QGEMM_ERR_UNSUPPORTED, "size past 2^30: T=%d", T);
  QG_TRY(dtype_ok(in_dtype, "in_dtype"));
  QG_TRY(need(offsets, 4, "offsets"));
  if (T > 0) {
    QG_TRY(need(logits, in_dtype == QGEMM_F32 ? 4 : 2, "logits"));
    QG_TRY(need(weights, 4, "weights"));
    QG_TRY(need(experts, 4, "experts"));
    QG_TRY(need(rows, 4, "rows"));
    const unsigned long long pb = (unsigned long long)T * k * 4;
    const Range in = range_of(logits, 1, 0, (unsigned long long)T * E * (in_dtype == QGEMM_F32 ? 4 : 2));
    const Range outs[4] = {{weights, weights + pb}, {experts, experts + pb}, {rows, rows + pb},
                           {offsets, offsets + 4ull * (E + 1)}};
    for (int i = 0; i < 4; ++i) {
      if (overlap(in, outs[i])) return fail(QGEMM_ERR_INVALID_ARG, "an output overlaps the logits");
      for (int j = 0; j < i; ++j)
        if (overlap(outs[i], outs[j])) return fail(QGEMM_ERR_INVALID_ARG, "two outputs overlap");
    }
  }
  QG_TRY(enter(s));
  return launch_route_topk(s, reinterpret_cast<const void*>(logits), in_dtype,
                           reinterpret_cast<float*>(weights), reinterpret_cast<int*>(experts),
                           reinterpret_cast<int*>(offsets), reinterpret_cast<int*>(rows), T, E, k,
                           renormalize);
}

qgemm_status qgemm_dispatch_rows(qgemm_stream_t s, uint64_t x, int dtype, uint64_t rows,
                                 uint64_t out, int T, int k, int K, int R) {
  QG_TRY(rows_entry(s, dtype, T, k, K, R, "K"));
  if (T == 0 || K == 0) return enter(s);
  const int es = dtype == QGEMM_F32 ? 4 : 2;
  QG_TRY(need(x, es, "x"));
  QG_TRY(need(rows, 4, "rows"));
  if (R > 0) QG_TRY(need(out, es, "out"));
  const unsigned long long row = (unsigned long long)K * es;
  const Range o = {out, out + R * row};
  if (overlap(o, {x, x + T * row}) || overlap(o, {rows, rows + 4ull * T * k}))
    return fail(QGEMM_ERR_INVALID_ARG, "out overlaps an input");
  QG_TRY(enter(s));
  return launch_dispatch_rows(s, reinterpret_cast<const void*>(x), dtype,
                              reinterpret_cast<const int*>(rows), reinterpret_cast<void*>(out),
                              nullptr, T, k, K, R);
}

qgemm_status qgemm_dispatch_rows_quantized(qgemm_stream_t s, uint64_t x, int in_dtype,
                                           uint64_t rows, uint64_t q, uint64_t sA, int T, int k,
                                           int K, int R) {
  QG_TRY(rows_entry(s, in_dtype, T, k, K, R, "K"));
  if (T == 0) return enter(s);
  const int es = in_dtype == QGEMM_F32 ? 4 : 2;
  QG_TRY(need(rows, 4, "rows"));
  if (K > 0) QG_TRY(need(x, es, "x"));
  if (R > 0) {
    QG_TRY(need(sA, 4, "sA"));
    if (K > 0) QG_TRY(need(q, 1, "q"));
  }
  const Range in = {x, x + (unsigned long long)T * K * es}, ix = {rows, rows + 4ull * T * k};
  const Range o = {q, q + (unsigned long long)R * K}, so = {sA, sA + 4ull * R};
  if (overlap(o, in) || overlap(so, in) || overlap(o, ix) || overlap(so, ix) || overlap(o, so))
    return fail(QGEMM_ERR_INVALID_ARG, "an output overlaps an input or the other output");
  QG_TRY(enter(s));
  return launch_dispatch_rows(s, reinterpret_cast<const void*>(x), in_dtype,
                              reinterpret_cast<const int*>(rows), reinterpret_cast<void*>(q),
                              reinterpret_cast<float*>(sA), T, k, K, R);
}

qgemm_status qgemm_combine_rows(qgemm_stream_t s, uint64_t y, int in_dtype, uint64_t rows,
                                uint64_t weights, uint64_t residual, uint64_t out, int out_dtype,
                                int T, int k, int N, int R) {
  QG_TRY(rows_entry(s, in_dtype, T, k, N, R, "N"));
  QG_TRY(dtype_ok(out_dtype, "out_dtype"));
  if (T == 0 || N == 0) return enter(s);
  const int es = in_dtype == QGEMM_F32 ? 4 : 2, os = out_dtype == QGEMM_F32 ? 4 : 2;
  QG_TRY(need(rows, 4, "rows"));
  if (R > 0) QG_TRY(need(y, es, "y"));
  if (weights) QG_TRY(need(weights, 4, "weights"));
  QG_TRY(need(out, os, "out"));
  if (residual) QG_TRY(need(residual, os, "residual"));
  const unsigned long long pb = 4ull * T * k, ob = (unsigned long long)T * N * os;
  const Range o = {out, out + ob};
  if (overlap(o, {y, y + (unsigned long long)R * N * es}) || overlap(o, {rows, rows + pb}) ||
      (weights && overlap(o, {weights, weights + pb})) ||
      (residual && residual != out && overlap(o, {residual, residual + ob})))
    return fail(QGEMM_ERR_INVALID_ARG, "out overlaps an input");
  QG_TRY(enter(s));
  return launch_combine_rows(s, reinterpret_cast<const void*>(y), in_dtype,
                             reinterpret_cast<const int*>(rows),
                             reinterpret_cast<const float*>(weights),
                             reinterpret_cast<const void*>(residual), reinterpret_cast<void*>(out),
                             out_dtype, T, k, N, R);
}

}  // extern "C"
