// Attention with capped scores, a distance bias and causal / prefix / document masks: argument checks, document ranges and the choice of the
// instantiation.  The kernels are in attention_{fwd,token,bwd}.inc.hpp, compiled per (type, padded head width) in kernels_attention_<type>_d<width>.hip.
#include "attention_tile.hpp"
#include "../../include/craft_hip.h"

namespace craft {

// per 32 tokens: {least, greatest document that is not negative, 1 if any is negative, 0}; two runs of groups (queries, keys) in one launch
__global__ __launch_bounds__(64) void k_document_ranges(const int* dq, int4* rq, int nq, int gq, const int* dk, int4* rk, int nk, int gk, int B) {
  const long e = (long)blockIdx.x * 64 + threadIdx.x, eq = (long)B * gq, ek = (long)B * gk;
  if (e >= eq + ek) return;
  const bool isq = e < eq;
  const long x = isq ? e : e - eq;
  const int groups = isq ? gq : gk, n = isq ? nq : nk;
  const long b = x / groups;
  const int g = (int)(x - b * groups), n0 = g * 32, n1 = min(n0 + 32, n);
  const int* d = (isq ? dq : dk) + b * n;
  int lo = 0x7fffffff, hi = -1, neg = 0;
  for (int i = n0; i < n1; ++i) {
    const int v = d[i];
    if (v < 0) neg = 1;
    else { lo = min(lo, v); hi = max(hi, v); }
  }
  (isq ? rq : rk)[x] = make_int4(lo, hi, neg, 0);
}

template <typename T>
static int by_width(const AttentionParams& p, int what, hipStream_t s) {
  if (what == 0) return p.D <= 32 ? attention_fwd_launch<T, 32>(p, s) : p.D <= 64 ? attention_fwd_launch<T, 64>(p, s) : attention_fwd_launch<T, 128>(p, s);
  if (what == 1) return p.D <= 32 ? attention_token_launch<T, 32>(p, s) : p.D <= 64 ? attention_token_launch<T, 64>(p, s) : attention_token_launch<T, 128>(p, s);
  return p.D <= 32 ? attention_bwd_launch<T, 32>(p, s) : p.D <= 64 ? attention_bwd_launch<T, 64>(p, s) : attention_bwd_launch<T, 128>(p, s);
}
static int dispatch(const AttentionParams& p, int dtype, int what, hipStream_t s) {
  return dtype == CRAFT_PREC_F16 ? by_width<_Float16>(p, what, s) : dtype == CRAFT_PREC_BF16 ? by_width<__bf16>(p, what, s) : by_width<float>(p, what, s);
}

// shape: B, Nq, Nk, H, Hk, D, then (batch, token, head) strides of the nt tensors
static int fill(AttentionParams& p, const long* shape, int nt, const float* slopes, const int* prefix, const int* doc_q, const int* doc_k, float scale, float cap,
                int causal, int dtype) {
  if (!shape || dtype < 0 || dtype > 2 || (doc_q == nullptr) != (doc_k == nullptr) || (prefix && !causal)) return CRAFT_ERR_ARG;
  if (!(cap >= 0.f) || !(cap <= 1e30f) || !(fabsf(scale) <= 1e30f)) return CRAFT_ERR_ARG;
  // 16-bit types take tanh from 1 / (1 + e^2u), off by 2^-23 of 1 however small u is: a capped score is off by cap 2^-22, 2^-10 here.  And a score
  // of zero times 2 scale / cap has to be zero, which it is not where that overflows.
  if (cap > 4096.f && dtype != CRAFT_PREC_F32) return CRAFT_ERR_UNSUPPORTED;
  if (cap > 0.f && !(fabsf(scale) / cap <= 1e30f)) return CRAFT_ERR_ARG;
  for (int i = 0; i < 6; ++i)
    if (shape[i] <= 0 || shape[i] >= (1l << 29)) return CRAFT_ERR_UNSUPPORTED;
  const long size = dtype == CRAFT_PREC_F32 ? 4 : 2, step = 16 / size;
  if (shape[3] % shape[4] || shape[5] > 128) return CRAFT_ERR_UNSUPPORTED;
  if (shape[5] % 8) return CRAFT_ERR_ALIGN;
  for (int i = 6; i < 6 + 3 * nt; ++i) {
    if (shape[i] < 0 || shape[i] % step) return CRAFT_ERR_ALIGN;
    if (i % 3 == 1 && shape[i] * size >= (1l << 24)) return CRAFT_ERR_UNSUPPORTED;        // 64 rows stay within the copies' 32-bit offsets
  }
  p = AttentionParams{};
  p.B = (int)shape[0]; p.Nq = (int)shape[1]; p.Nk = (int)shape[2]; p.H = (int)shape[3]; p.Hk = (int)shape[4]; p.D = (int)shape[5];
  long* st[5][3] = {{&p.q_b, &p.q_n, &p.q_h}, {&p.k_b, &p.k_n, &p.k_h}, {&p.v_b, &p.v_n, &p.v_h}, {&p.o_b, &p.o_n, &p.o_h}, {&p.go_b, &p.go_n, &p.go_h}};
  for (int t = 0; t < nt; ++t)
    for (int i = 0; i < 3; ++i) *st[t][i] = shape[6 + 3 * t + i];
  const float log2e = 1.44269504088896341f;
  p.scale = scale; p.cap = cap; p.c2 = scale * log2e;
  if (cap > 0.f) { p.ca = 2.f * scale / cap * log2e; p.cap2 = cap * log2e; }
  p.slopes = slopes; p.prefix = prefix; p.docq = doc_q; p.dock = doc_k; p.causal = causal ? 1 : 0;
  return 0;
}

static long range_bytes(const AttentionParams& p) { return p.docq ? 16l * p.B * ((p.Nq + 31) / 32 + (p.Nk + 31) / 32) : 0; }

static int make_ranges(AttentionParams& p, void* ws, hipStream_t s) {
  if (!p.docq) return 0;
  const int gq = (p.Nq + 31) / 32, gk = (p.Nk + 31) / 32;
  int4* rq = reinterpret_cast<int4*>(ws);
  int4* rk = rq + (long)p.B * gq;
  const long n = (long)p.B * (gq + gk);
  hipLaunchKernelGGL(k_document_ranges, dim3((unsigned)((n + 63) / 64)), dim3(64), 0, s, p.docq, rq, p.Nq, gq, p.dock, rk, p.Nk, gk, p.B);
  p.rq = rq; p.rk = rk;
  return (int)hipGetLastError();
}
static bool aligned(const void* a) { return a && (reinterpret_cast<uintptr_t>(a) & 15) == 0; }

}  // namespace craft

using namespace craft;

extern "C" {

int craft_attention_fwd(const void* q, const void* k, const void* v, const long* shape, const float* slopes, const int* prefix, const int* doc_q,
                        const int* doc_k, float scale, float cap, int causal, int dtype, int splits, void* out, float* lse, void* out_rest, void* ws,
                        long ws_bytes, void* stream) {
  AttentionParams p;
  const int rc = fill(p, shape, 4, slopes, prefix, doc_q, doc_k, scale, cap, causal, dtype);
  if (rc) return rc;
  if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(out)) return CRAFT_ERR_ALIGN;
  if (splits < 0 || splits > 65535 || (splits && (lse || out_rest)) || (reinterpret_cast<uintptr_t>(out_rest) & 15)) return CRAFT_ERR_ARG;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  p.q = q; p.k = k; p.v = v; p.out = out; p.lse = lse; p.rest = out_rest;
  if (splits) {
    if ((long)p.Nq * (p.H / p.Hk) > 1l << 20) return CRAFT_ERR_UNSUPPORTED;
    p.splits = splits;
    if (splits > 1) {
      const long rows = (long)p.B * p.Hk * p.Nq * (p.H / p.Hk) * splits;
      if (!aligned(ws) || ws_bytes < rows * (p.D + 2) * 4) return CRAFT_ERR_ARG;
      p.part_o = reinterpret_cast<float*>(ws);
      p.part_ml = p.part_o + rows * p.D;
    }
    return dispatch(p, dtype, 1, s);
  }
  if (p.docq && (!aligned(ws) || ws_bytes < range_bytes(p))) return CRAFT_ERR_ARG;
  const int rr = make_ranges(p, ws, s);
  return rr ? rr : dispatch(p, dtype, 0, s);
}

int craft_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* out_rest, const float* lse, const void* grad_out,
                        const long* shape,
                        const float* slopes, const int* prefix, const int* doc_q, const int* doc_k, float scale, float cap, int causal, int dtype,
                        int split_group, void* dq, void* dk, void* dv, void* ws, long ws_bytes, void* stream) {
  AttentionParams p;
  const int rc = fill(p, shape, 5, slopes, prefix, doc_q, doc_k, scale, cap, causal, dtype);
  if (rc) return rc;
  if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(out) || !aligned(grad_out)) return CRAFT_ERR_ALIGN;
  if ((dq && !aligned(dq)) || (dk && !aligned(dk)) || (dv && !aligned(dv))) return CRAFT_ERR_ALIGN;
  if ((dk == nullptr) != (dv == nullptr) || (split_group && !dk)) return CRAFT_ERR_ARG;
  if (!lse || (reinterpret_cast<uintptr_t>(out_rest) & 15)) return CRAFT_ERR_ARG;
  const long ranges = range_bytes(p), delta = ((long)p.B * p.H * p.Nq * 4 + 15) / 16 * 16, part = split_group ? (long)p.B * p.Nk * p.H * p.D * 4 : 0;
  // fp16: a key head's rows are cut into slices for the largest norms: as many rows as a block has groups of lanes, 1024 slices at most (a wave reads them all)
  const bool f16 = dtype == CRAFT_PREC_F16;
  const long rows = (long)p.Nq * (p.H / p.Hk) > p.Nk ? (long)p.Nq * (p.H / p.Hk) : p.Nk, each = p.D > 64 ? 16 : 32;
  const long slices = (rows + each - 1) / each < 1024 ? (rows + each - 1) / each : 1024, more = f16 ? (8 * slices * p.B * p.Hk + 15) / 16 * 16 : 0;
  if (!aligned(ws) || ws_bytes < ranges + delta + more + 2 * part) return CRAFT_ERR_ARG;
  if (!dq && !dk) return 0;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  p.q = q; p.k = k; p.v = v; p.o = out; p.o_rest = out_rest; p.go = grad_out; p.lse = const_cast<float*>(lse); p.dq = dq; p.dk = dk; p.dv = dv;
  char* w = reinterpret_cast<char*>(ws) + ranges;
  p.delta = reinterpret_cast<float*>(w);
  if (f16) { p.top = reinterpret_cast<float2*>(w + delta); p.slices = (int)slices; }
  w += delta + more;
  if (split_group) { p.part_k = reinterpret_cast<float*>(w); p.part_v = reinterpret_cast<float*>(w + part); }
  const int rr = make_ranges(p, ws, s);
  return rr ? rr : dispatch(p, dtype, 2, s);
}

}  // extern "C"
