// Forward attention: a block owns 128 queries of one head (4 waves x 32), walks over the keys in LDS tiles, and keeps the running maximum and sum
// of the softmax, the query operand and the 32 x D output in registers.
//
// Bound by the vector instructions of the softmax, which take the SIMD in turns with the matrix instructions, and at large sizes by the package's power.
// 8192 fp16 queries x 32 heads of 128, causal with a prefix of 1900: 607 .. 626 us, 0.95 PF/s, 68 % of what a large library product reaches; counters: matrix
// instructions 50 % of the SIMDs' cycles, vector instructions 44 %, at 1.5 .. 1.7 GHz.  With scores of the next tile computed under the softmax of this one the
// same 628 us stood against 628 (and capped scores were slower).  Capped, causal, 4096 bf16 tokens x 32 heads of 128: 222 us (29 % and 54 %).  fp32, 2852 tokens
// x 8 heads of 64: 242 us, 69 TF/s (the rate of an fp32 library product is 154): 45 % and 10 %, one wave to a SIMD waits for its own products.
#pragma once
#include "attention_tile.hpp"

namespace craft {

template <typename T, int DP> struct FwdShape {
  static constexpr int TK = sizeof(T) == 2 ? 64 : 32;                     // keys of a tile
  static constexpr int TILE = TK * DP * (int)sizeof(T);
  static constexpr int STAGE = 2 * TILE + 512;                            // K, V, document ids
  static constexpr int LDS = 2 * STAGE + 64;
};

template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void k_attention_fwd(AttentionParams p) {
  typedef FwdShape<T, DP> S;
  typedef typename AtFrag<T>::type frag_t;
  constexpr int TK = S::TK, NB = TK / 32;
  extern __shared__ __align__(512) unsigned char lds[];
  const unsigned lds0 = (unsigned)(size_t)(CRAFT_LDS unsigned char*)lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int nqt = (p.Nq + 127) >> 7;
  int bh, qt;
  block_of(p.B * p.H, nqt, bh, qt);
  qt = nqt - 1 - qt;                            // (the last queries of a causal row are the heaviest)
  const int b = bh / p.H, head = bh - b * p.H, kvh = head / (p.H / p.Hk);
  const int off = p.Nk - p.Nq, i0 = qt * 128, i_last = min(i0 + 127, p.Nq - 1);
  const int prefix = p.prefix ? p.prefix[b] : 0;
  // this lane's query; queries behind the last one repeat it and are not stored
  const int i = min(i0 + wave * 32 + (lane & 31), p.Nq - 1), pos = i + off;
  int lim = p.causal ? min(max(pos + 1, prefix), p.Nk) : p.Nk;            // it sees the keys below lim (of its document)
  int mydoc = 0;
  if (p.docq) { mydoc = p.docq[(long)b * p.Nq + i]; if (mydoc < 0) lim = 0; }
  int lim_lo = lim, lim_hi = lim;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { lim_lo = min(lim_lo, __shfl_xor(lim_lo, o)); lim_hi = max(lim_hi, __shfl_xor(lim_hi, o)); }
  lim_lo = __builtin_amdgcn_readfirstlane(lim_lo); lim_hi = __builtin_amdgcn_readfirstlane(lim_hi);

  frag_t qf[DP / 16];
  load_own<T, DP>(reinterpret_cast<const T*>(p.q) + b * p.q_b + (long)i * p.q_n + head * p.q_h, p.D, h, qf);
  constexpr bool RAW = !BIAS;                   // the maximum is taken of at_raw, at_mul goes into the exponential's one fma
  const float mul = at_mul<T, CAP>(p), c2 = RAW ? fmaxf(fabsf(mul), 1e-30f) : 1.f;
  if (RAW && !CAP && mul < 0.f) {
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) qf[ks] = -qf[ks];
  }
  arrived(qf);

  int t0 = 0, t1 = p.causal ? (max(min(max(i_last + off + 1, prefix), p.Nk), 0) + TK - 1) / TK : (p.Nk + TK - 1) / TK;
  int4 qr = make_int4(0, 0, 0, 0), qrw = qr;
  const int4* rk = nullptr;
  const int kgroups = (p.Nk + 31) >> 5;
  if (p.rq) {
    const int qgroups = (p.Nq + 31) >> 5;
    const int4* rq = p.rq + (long)b * qgroups;
    rk = p.rk + (long)b * kgroups;
    qr = join_ranges(rq, i0 >> 5, min((i0 >> 5) + 4, qgroups) - 1);
    qrw = rq[min((i0 >> 5) + wave, qgroups - 1)];
    tiles_of_documents<256>(rk, kgroups, NB, qr, t0, t1, tid, reinterpret_cast<int*>(lds + 2 * S::STAGE));
  }
  const int nchunk = p.D * (int)sizeof(T) / 16;
  const unsigned kst = (unsigned)(p.k_n * (long)sizeof(T)), vst = (unsigned)(p.v_n * (long)sizeof(T));
  TileCopy<T, DP, TK, 4> kc, vc;
  kc.init(wave, lane, kst, nchunk);
  vc.init(wave, lane, vst, nchunk);
  const unsigned char* kb = reinterpret_cast<const unsigned char*>(p.k) + (b * p.k_b + kvh * p.k_h) * (long)sizeof(T);
  const unsigned char* vb = reinterpret_cast<const unsigned char*>(p.v) + (b * p.v_b + kvh * p.v_h) * (long)sizeof(T);
  // the next tile from t on that has one of the block's documents, and its range
  auto next = [&](int t, int4& kr) {
    if (rk)
      for (; t < t1; ++t) {
        kr = uniform_range(join_ranges(rk, t * NB, min(t * NB + NB, kgroups) - 1));
        if (ranges_meet(kr, qr)) break;
      }
    return t;
  };
  auto stage = [&](int buf, int t) {
    const int valid = p.Nk - t * TK;
    const unsigned at = lds0 + (unsigned)buf * S::STAGE;
    kc.issue(kb + (long)t * TK * kst, kst, nchunk, valid, at, wave, lane);
    vc.issue(vb + (long)t * TK * vst, vst, nchunk, valid, at + S::TILE, wave, lane);
    if (rk && wave == 0) copy_words(p.dock + (long)b * p.Nk, (long)t * TK, p.Nk - 1, at + 2 * S::TILE, lane);
  };

  f32x16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = -INFINITY, l = 0.f;                 // the running maximum (kept up to 2^8 below the true one) and this lane's share of the sum
  const float slope2 = BIAS ? p.slopes[head] * 1.44269504088896f : 0.f;

  const float thr = RAW ? 8.f / c2 : 8.f;
  int4 kr = make_int4(0, 0, 0, 0), krn = kr;
  int t = next(t0, kr), buf = 0;
  if (t < t1) stage(0, t);
  while (t < t1) {
    wait_copies();
    __syncthreads();                            // the tile is whole; everybody has left the other buffer
    const int tn = next(t + 1, krn);
    if (tn < t1) stage(buf ^ 1, tn);
    unsigned char* V = lds + buf * S::STAGE + S::TILE;
    const int* ids = reinterpret_cast<const int*>(V + S::TILE);
    const unsigned at = lds0 + (unsigned)(buf * S::STAGE), Kr = row_addr<T, DP>(at, lane), Vc = col_addr<T, DP>(at + S::TILE, lane);
    const int k0 = t * TK;
    bool docmask = false, skip = k0 >= lim_hi;
    if (rk) {
      if (kr.z) { zero_rows<T, DP, TK>(V, ids, p.Nk - k0, tid, 256); __syncthreads(); }
      docmask = !one_document(kr, qrw);
      skip |= !ranges_meet(kr, qrw);
    }
    if (!skip) {
      f32x16 x[NB];
#pragma unroll
      for (int kbk = 0; kbk < NB; ++kbk) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[kbk][r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) at_mma(row_read<T, DP>(Kr, kbk, ks), qf[ks], x[kbk]);
      }
      if constexpr (CAP || BIAS) {
        const float away = BIAS ? (float)(pos - k0 - 4 * h) : 0.f;
#pragma unroll
        for (int kbk = 0; kbk < NB; ++kbk)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float z = at_raw<T, CAP>(p, x[kbk][r]);
            if constexpr (BIAS) z = fmaf(-slope2, fabsf(away - (float)(32 * kbk + acc_row(r))), z * mul);
            x[kbk][r] = z;
          }
      }
      if (k0 + TK > lim_lo) {
        const int room = lim - k0 - 4 * h;
#pragma unroll
        for (int kbk = 0; kbk < NB; ++kbk)
#pragma unroll
          for (int r = 0; r < 16; ++r) x[kbk][r] = 32 * kbk + acc_row(r) < room ? x[kbk][r] : -INFINITY;
      }
      if (docmask) {
#pragma unroll
        for (int kbk = 0; kbk < NB; ++kbk)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int4 d = *reinterpret_cast<const int4*>(ids + 32 * kbk + 8 * g + 4 * h);
            x[kbk][4 * g + 0] = d.x == mydoc ? x[kbk][4 * g + 0] : -INFINITY;
            x[kbk][4 * g + 1] = d.y == mydoc ? x[kbk][4 * g + 1] : -INFINITY;
            x[kbk][4 * g + 2] = d.z == mydoc ? x[kbk][4 * g + 2] : -INFINITY;
            x[kbk][4 * g + 3] = d.w == mydoc ? x[kbk][4 * g + 3] : -INFINITY;
          }
      }
      float mt = x[0][0];
#pragma unroll
      for (int kbk = 0; kbk < NB; ++kbk)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, x[kbk][r]);
      mt = fmaxf(mt, at_other_half(mt));
      // the output is rescaled only when some query's maximum has grown by more than 2^8: until then its probabilities are merely larger than one
      if (__ballot(mt > m + thr)) {
        const float mn = fmaxf(m, mt), alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c2);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      }
      const float ref = m == -INFINITY ? 0.f : m * c2;
#pragma unroll
      for (int kbk = 0; kbk < NB; ++kbk)
#pragma unroll
        for (int r = 0; r < 16; ++r) { x[kbk][r] = __builtin_amdgcn_exp2f(RAW ? fmaf(x[kbk][r], c2, -ref) : x[kbk][r] - ref); l += x[kbk][r]; }
#pragma unroll
      for (int kbk = 0; kbk < NB; ++kbk)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          const frag_t pf = at_pack<T>(x[kbk], s2);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) at_mma(col_read<T, DP>(Vc, 32 * kbk + 16 * s2, d), pf, o[d]);
        }
    }
    t = tn;
    kr = krn;
    buf ^= 1;
  }

  l += at_other_half(l);
  if (i0 + wave * 32 + (lane & 31) < p.Nq) {
    const float inv = l > 0.f ? 1.f / l : 0.f;                            // nothing seen: zero
    T* orow = reinterpret_cast<T*>(p.out) + b * p.o_b + (long)i * p.o_n + head * p.o_h;
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * d + 8 * g + 4 * h;
        if (c < p.D) {
          t4 w, rest;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float v = o[d][4 * g + j] * inv;
            w[j] = (T)v;
            rest[j] = (T)(v - (float)w[j]);
          }
          *reinterpret_cast<t4*>(orow + c) = w;
          if (sizeof(T) == 2 && p.rest) *reinterpret_cast<t4*>(reinterpret_cast<T*>(p.rest) + (((long)b * p.Nq + i) * p.H + head) * p.D + c) = rest;
        }
      }
    if (p.lse && h == 0) {
      float* lse = p.lse + ((long)bh * p.Nq + i) * at_lw<T>();
      const float big = m * c2, small = __log2f(l), sum = big + small;
      lse[0] = l > 0.f ? sum : INFINITY;
      if (at_lw<T>() == 2) lse[1] = l > 0.f ? small - (sum - big) : 0.f;
    }
  }
}

template <typename T, int DP>
int attention_fwd_launch(const AttentionParams& p, hipStream_t s) {
  typedef FwdShape<T, DP> S;
  const long blocks = (long)p.B * p.H * ((p.Nq + 127) / 128);
  if (blocks > 0x7fffffffL) return CRAFT_ERR_UNSUPPORTED;
  auto go = [&](auto tag) {
    constexpr auto kernel = decltype(tag)::value;
    if (const int rc = allow_lds<kernel>(S::LDS)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), S::LDS, s, p);
    return (int)hipGetLastError();
  };
  if (p.cap > 0.f) return p.slopes ? go(KernelTag<k_attention_fwd<T, DP, true, true>>()) : go(KernelTag<k_attention_fwd<T, DP, true, false>>());
  return p.slopes ? go(KernelTag<k_attention_fwd<T, DP, false, true>>()) : go(KernelTag<k_attention_fwd<T, DP, false, false>>());
}

}  // namespace craft
