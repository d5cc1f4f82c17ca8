// Backward attention.  With p = 2^(z - lse), delta_i = sum_d go_i o_i:
//   dv_j = sum_i p_ij go_i;  dp_ij = go_i . v_j;  ds_ij = p_ij (dp_ij - delta_i) (1 - tanh^2);  dq_i = scale sum_j ds_ij k_j;  dk_j = scale sum_i ds_ij q_i
// Two kernels, each the sole writer of its gradients (no atomics: the result does not depend on the order of the blocks): k_attention_dq owns 128
// queries and walks over the keys, k_attention_dkv owns 128 keys and walks over the queries of every head that shares them.  Both recompute the scores.
//
// Bound by the same turns of vector and matrix instructions as the forward pass, with 18 instead of 14 D operations a pair (the scores and dp twice:
// the price of one writer for each gradient).  Capped, causal, 4096 bf16 tokens x 32 heads of 128 on 8 key heads: dk, dv 368 us
// (0.75 PF/s; matrix instructions 36 %, vector instructions 41 % of the SIMDs' cycles, the rest waits for LDS), dq 288 us (0.72 PF/s; 35 % and 48 %), the sum over
// the group 24 us, delta 18 us.  fp32, 2852 tokens x 8 heads of 64: 396 and 300 us, 83 TF/s of 154 (55 % and 8 %).  fp16, 4 x 3001 tokens in documents of about
// 400, 8 heads of 64: 89 and 51 us, delta and the largest norms 12 us: two of three SIMDs' cycles wait, tiles cut by documents' borders and their ranges read in the walk.
#pragma once
#include "attention_tile.hpp"

namespace craft {

// -delta (the sums of dp start there), 16 lanes to a row
template <typename T>
__global__ __launch_bounds__(256) void k_attention_delta(AttentionParams p, float* delta) {
  const long row = (long)blockIdx.x * 16 + (threadIdx.x >> 4), rows = (long)p.B * p.Nq * p.H;
  if (row >= rows) return;                                                 // (whole 16-lane groups)
  const int head = (int)(row % p.H);
  const long bi = row / p.H, b = bi / p.Nq, i = bi - b * p.Nq;
  const int c = 8 * (threadIdx.x & 15);
  float s = 0.f;
  if (c < p.D) {
    typedef typename AtFrag<T>::type frag_t;
    const frag_t o = *reinterpret_cast<const frag_t*>(reinterpret_cast<const T*>(p.o) + b * p.o_b + i * p.o_n + head * p.o_h + c);
    const frag_t g = *reinterpret_cast<const frag_t*>(reinterpret_cast<const T*>(p.go) + b * p.go_b + i * p.go_n + head * p.go_h + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (float)o[j] * (float)g[j];
    if (sizeof(T) == 2 && p.o_rest) {
      const frag_t r = *reinterpret_cast<const frag_t*>(reinterpret_cast<const T*>(p.o_rest) + row * p.D + c);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += (float)r[j] * (float)g[j];
    }
  }
#pragma unroll
  for (int k = 8; k > 0; k >>= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 15) == 0) delta[(b * p.H + head) * p.Nq + i] = -s;
}

// The same for fp16, which also needs the largest norms for its powers of two (score_exponent): a block per (batch, key head, slice), whose
// share of the queries of the head's group and of its keys it reads, 8 or 16 lanes to a row.  Padding's rows do not count.  All loads of a row stand in front of
// its sums (one behind the other: 20 us instead of 16; as many slices as there are rows for: 12).
template <typename T>
__global__ __launch_bounds__(256) void k_attention_delta_scaled(AttentionParams p, float* delta) {
  typedef typename AtFrag<T>::type frag_t;
  __shared__ float2 red[32];
  const int bk = blockIdx.x / p.slices, slice = blockIdx.x - bk * p.slices, b = bk / p.Hk, kvh = bk - b * p.Hk, G = p.H / p.Hk;
  const int shift = p.D > 64 ? 4 : 3, groups = 256 >> shift, sub = threadIdx.x >> shift, c = 8 * (threadIdx.x & ((1 << shift) - 1));
  const bool in = c < p.D;
  const int i0 = (int)((long)p.Nq * slice / p.slices), j0 = (int)((long)p.Nk * slice / p.slices);
  const long nq = ((long)p.Nq * (slice + 1) / p.slices - i0) * G, nk = (long)p.Nk * (slice + 1) / p.slices - j0;
  float go2 = 0.f, v2 = 0.f;
  for (long r = sub; r < max(nq, nk); r += groups) {                       // (whole groups of lanes)
    const bool isq = r < nq, isk = r < nk;
    const int i = i0 + (int)(r / G), head = kvh * G + (int)(r % G);
    const long row = ((long)b * p.Nq + i) * p.H + head;
    frag_t o, g, t, v;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = g[j] = t[j] = v[j] = (T)0.f;
    int dq = 0, dk = 0;
    if (isq) {
      if (in) {
        o = *reinterpret_cast<const frag_t*>(reinterpret_cast<const T*>(p.o) + b * p.o_b + i * p.o_n + head * p.o_h + c);
        g = *reinterpret_cast<const frag_t*>(reinterpret_cast<const T*>(p.go) + b * p.go_b + i * p.go_n + head * p.go_h + c);
        if (p.o_rest) t = *reinterpret_cast<const frag_t*>(reinterpret_cast<const T*>(p.o_rest) + row * p.D + c);
      }
      if (p.docq) dq = p.docq[(long)b * p.Nq + i];
    }
    if (isk) {
      if (in) v = *reinterpret_cast<const frag_t*>(reinterpret_cast<const T*>(p.v) + b * p.v_b + (j0 + r) * p.v_n + kvh * p.v_h + c);
      if (p.dock) dk = p.dock[(long)b * p.Nk + j0 + r];
    }
    float s = 0.f, n = 0.f, m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s += (float)o[j] * (float)g[j];
      s += (float)t[j] * (float)g[j];
      n += (float)g[j] * (float)g[j];
      m += (float)v[j] * (float)v[j];
    }
    for (int k = 1 << (shift - 1); k > 0; k >>= 1) { s += __shfl_xor(s, k); n += __shfl_xor(n, k); m += __shfl_xor(m, k); }
    if (isq && c == 0) delta[((long)b * p.H + head) * p.Nq + i] = -s;
    if (n < INFINITY && dq >= 0) go2 = fmaxf(go2, n);
    if (m < INFINITY && dk >= 0) v2 = fmaxf(v2, m);
  }
  if (c == 0) red[sub] = make_float2(go2, v2);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < groups; ++k) { go2 = fmaxf(go2, red[k].x); v2 = fmaxf(v2, red[k].y); }
    p.top[(long)bk * p.slices + slice] = make_float2(go2, v2);
  }
}

template <typename T, int DP> struct BwdShape {
  static constexpr int TR = sizeof(T) == 2 && DP < 128 ? 64 : 32;         // rows of a tile (128 columns in 64-row tiles: registers spill)
  static constexpr int TILE = TR * DP * (int)sizeof(T);
  static constexpr int STAGE = 2 * TILE + 1024;                        // two operands; lse, delta, documents of 64 rows
  static constexpr int LDS = 2 * STAGE + 64;
};

// the key / value kernel's tiles.  Two 16-bit operands and two fp32 results of 128 columns leave no room for two waves to a SIMD in registers: there V is
// read from LDS (the block's 128 keys stay there), and tiles are 32 rows so that two blocks share a compute unit (558 -> 404 us for the capped 4096-token step)
template <typename T, int DP> struct DkvShape {
  static_assert(sizeof(T) == 2 || BwdShape<T, DP>::TR * at_lw<T>() <= 64, "a tile's log-sums are one copy");
  static constexpr bool VL = sizeof(T) == 2 && DP == 128;
  static constexpr int TR = VL ? 32 : BwdShape<T, DP>::TR;
  static constexpr int TILE = TR * DP * (int)sizeof(T);
  static constexpr int STAGE = 2 * TILE + 1024;
  static constexpr int V = 2 * STAGE + 512, LDS = V + (VL ? 128 * DP * (int)sizeof(T) : 0);
};

// dq: lane = query
template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 || DP < 128 ? 2 : 1)) void k_attention_dq(AttentionParams p) {
  typedef BwdShape<T, DP> S;
  typedef typename AtFrag<T>::type frag_t;
  constexpr int TK = S::TR, NB = TK / 32;
  extern __shared__ __align__(512) unsigned char lds[];
  const unsigned lds0 = (unsigned)(size_t)(CRAFT_LDS unsigned char*)lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int nqt = (p.Nq + 127) >> 7;
  int bh, qt;
  block_of(p.B * p.H, nqt, bh, qt);
  qt = nqt - 1 - qt;
  const int b = bh / p.H, head = bh - b * p.H, kvh = head / (p.H / p.Hk);
  const int off = p.Nk - p.Nq, i0 = qt * 128, i_last = min(i0 + 127, p.Nq - 1);
  const int prefix = p.prefix ? p.prefix[b] : 0;
  const int i = min(i0 + wave * 32 + (lane & 31), p.Nq - 1), pos = i + off;
  int lim = p.causal ? min(max(pos + 1, prefix), p.Nk) : p.Nk;
  int mydoc = 0;
  if (p.docq) { mydoc = p.docq[(long)b * p.Nq + i]; if (mydoc < 0) lim = 0; }
  int lim_lo = lim, lim_hi = lim;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { lim_lo = min(lim_lo, __shfl_xor(lim_lo, o)); lim_hi = max(lim_hi, __shfl_xor(lim_hi, o)); }
  lim_lo = __builtin_amdgcn_readfirstlane(lim_lo); lim_hi = __builtin_amdgcn_readfirstlane(lim_hi);

  frag_t qf[DP / 16], gf[DP / 16];
  load_own<T, DP>(reinterpret_cast<const T*>(p.q) + b * p.q_b + (long)i * p.q_n + head * p.q_h, p.D, h, qf);
  load_own<T, DP>(reinterpret_cast<const T*>(p.go) + b * p.go_b + (long)i * p.go_n + head * p.go_h, p.D, h, gf);
  const float* lp = p.lse + ((long)bh * p.Nq + i) * at_lw<T>();
  float row[3] = {lp[0], p.delta[(long)bh * p.Nq + i], at_lw<T>() == 2 ? lp[1] : 0.f};
  int ex = 0;
  if constexpr (std::is_same<T, _Float16>::value) {
    const float v2 = largest_rows(p, b * p.Hk + kvh, lane).y;
    float n = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) n += (float)gf[ks][j] * (float)gf[ks][j];
    n += at_other_half(n);
    ex = score_exponent(n < INFINITY ? n : 0.f, v2);
    row[0] -= (float)ex;
  }
  arrived(qf);
  arrived(gf);
  arrived(row);
  const float lse = row[0], delta = row[1], mul = at_mul<T, CAP>(p);

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
  auto next = [&](int t, int4& r) {
    if (rk)
      for (; t < t1; ++t) {
        r = uniform_range(join_ranges(rk, t * NB, min(t * NB + NB, kgroups) - 1));
        if (ranges_meet(r, qr)) break;
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

  f32x16 dq[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
  const float slope2 = BIAS ? p.slopes[head] * 1.44269504088896f : 0.f;

  int4 kr = make_int4(0, 0, 0, 0), krn = kr;
  int t = next(t0, kr), buf = 0;
  if (t < t1) stage(0, t);
  while (t < t1) {
    wait_copies();
    __syncthreads();
    const int tn = next(t + 1, krn);
    if (tn < t1) stage(buf ^ 1, tn);
    unsigned char* K = lds + buf * S::STAGE;
    unsigned char* V = K + S::TILE;
    const int* ids = reinterpret_cast<const int*>(V + S::TILE);
    const unsigned at = lds0 + (unsigned)(buf * S::STAGE), Kr = row_addr<T, DP>(at, lane), Kc = col_addr<T, DP>(at, lane);
    const int k0 = t * TK;
    bool docmask = false, skip = k0 >= lim_hi;
    if (rk) {
      if (kr.z) { zero_rows<T, DP, TK>(K, ids, p.Nk - k0, tid, 256); __syncthreads(); }
      docmask = !one_document(kr, qrw);
      skip |= !ranges_meet(kr, qrw);
    }
    if (!skip) {
      const bool masked = docmask || k0 + TK > lim_lo;
#pragma unroll
      for (int kbk = 0; kbk < NB; ++kbk) {
        f32x16 x, y;
#pragma unroll
        for (int r = 0; r < 16; ++r) { x[r] = 0.f; y[r] = delta; }                // dp - delta: the sum starts at -delta, which is what is stored
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          at_mma(row_read<T, DP>(Kr, kbk, ks), qf[ks], x);
          at_mma(row_read<T, DP>(Kr, kbk, ks, S::TILE), gf[ks], y);
        }
        const float away = BIAS ? (float)(pos - k0 - 32 * kbk - 4 * h) : 0.f;
        {                                                                 // in steps over all 16 scores: a score's own steps wait for one another
          if constexpr (CAP) {
            at_raws<T>(p, x);
#pragma unroll
            for (int q = 0; q < 16; ++q) y[q] *= at_slope<T>(x[q]);
          }
#pragma unroll
          for (int q = 0; q < 16; ++q)
          {
            float z = fmaf(x[q], mul, -lse);
            if constexpr (BIAS) z = fmaf(-slope2, fabsf(away - (float)acc_row(q)), z);
            x[q] = at_lw<T>() == 2 ? z - row[2] : z;
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int q = 0; q < 16; ++q) x[q] = __builtin_amdgcn_exp2f(x[q]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int q = 0; q < 16; ++q) x[q] *= y[q];
        }
        if (masked) {                                                     // a choice, not a product: what the mask hides may be inf or NaN
          const int room = lim - k0 - 32 * kbk - 4 * h;
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = acc_row(r) < room ? x[r] : 0.f;
          if (docmask) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int4 d = *reinterpret_cast<const int4*>(ids + 32 * kbk + 8 * g + 4 * h);
              x[4 * g + 0] = d.x == mydoc ? x[4 * g + 0] : 0.f;
              x[4 * g + 1] = d.y == mydoc ? x[4 * g + 1] : 0.f;
              x[4 * g + 2] = d.z == mydoc ? x[4 * g + 2] : 0.f;
              x[4 * g + 3] = d.w == mydoc ? x[4 * g + 3] : 0.f;
            }
          }
        }
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          const frag_t sf = at_pack<T>(x, s2);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) at_mma(col_read<T, DP>(Kc, 32 * kbk + 16 * s2, d), sf, dq[d]);
        }
      }
    }
    t = tn;
    kr = krn;
    buf ^= 1;
  }
  if (i0 + wave * 32 + (lane & 31) < p.Nq) {
    T* row = reinterpret_cast<T*>(p.dq) + (((long)b * p.Nq + i) * p.H + head) * p.D;
    const float scale = __builtin_ldexpf(p.scale, -ex);
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * d + 8 * g + 4 * h;
        if (c < p.D) {
          t4 w;
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = (T)(dq[d][4 * g + j] * scale);
          *reinterpret_cast<t4*>(row + c) = w;
        }
      }
  }
}

// dk, dv: lane = key
template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 || DP == 32 ? 2 : 1)) void k_attention_dkv(AttentionParams p) {
  typedef DkvShape<T, DP> S;
  typedef typename AtFrag<T>::type frag_t;
  constexpr int TQ = S::TR, NB = TQ / 32;
  constexpr bool F16 = std::is_same<T, _Float16>::value;
  extern __shared__ __align__(512) unsigned char lds[];
  const unsigned lds0 = (unsigned)(size_t)(CRAFT_LDS unsigned char*)lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int nkt = (p.Nk + 127) >> 7, G = p.H / p.Hk;
  // part_k: one block per query head, whose results a second kernel sums over the group; else one block walks over the heads of its group
  const int heads = p.part_k ? p.H : p.Hk;
  int bx, kt;
  block_of(p.B * heads, nkt, bx, kt);           // (the first keys of a causal row are the heaviest)
  const int b = bx / heads, hx = bx - b * heads, kvh = p.part_k ? hx / G : hx;
  const int head0 = p.part_k ? hx : hx * G, head1 = p.part_k ? hx + 1 : hx * G + G;
  const int off = p.Nk - p.Nq, j0 = kt * 128, jw = j0 + wave * 32;
  const int prefix = p.prefix ? p.prefix[b] : 0;
  const int key = min(jw + (lane & 31), p.Nk - 1);
  const int first = !p.causal || key < prefix ? -0x40000000 : key - off;  // the first query that sees this key
  const int mydoc = p.dock ? p.dock[(long)b * p.Nk + key] : 0;

  frag_t kf[DP / 16], vf[S::VL ? 1 : DP / 16];
  load_own<T, DP>(reinterpret_cast<const T*>(p.k) + b * p.k_b + (long)key * p.k_n + kvh * p.k_h, p.D, h, kf);
  int ex = 0;                                   // fp16 (behind the keys' loads): probabilities times 2^15, gradients of scores times 2^ex
  if constexpr (F16) {
    const float2 top = largest_rows(p, b * p.Hk + kvh, lane);
    ex = __builtin_amdgcn_readfirstlane(score_exponent(top.x, top.y));
  }
  const float xp = F16 ? 0x1p15f : 1.f, xs = F16 ? __builtin_ldexpf(1.f, ex) : 1.f;
  const int nchunk = p.D * (int)sizeof(T) / 16;
  const unsigned VTr = row_addr<T, DP>(lds0 + (unsigned)(S::V + wave * 32 * at_rowb<T, DP>()), lane);
  if constexpr (S::VL) {
    typedef TileCopy<T, DP, 128, 4> Copy;
    Copy vc;
    const unsigned vst = (unsigned)(p.v_n * (long)sizeof(T));
    vc.init(wave, lane, vst, nchunk);
    vc.issue(reinterpret_cast<const unsigned char*>(p.v) + (b * p.v_b + kvh * p.v_h + (long)j0 * p.v_n) * (long)sizeof(T), vst, nchunk, p.Nk - j0,
             lds0 + (unsigned)S::V, wave, lane);
    if (nchunk < Copy::CPR) {                           // both operands of go v come out of LDS: behind D one of them has to be zero
      wait_copies();
      __syncthreads();
      for (int c = tid; c < 128 * Copy::CPR; c += 256) {
        const int row = c / Copy::CPR;
        if (((c % Copy::CPR) ^ tile_swz<Copy::CPR>(row)) >= nchunk) *reinterpret_cast<f32x4*>(lds + S::V + c * 16) = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  } else {
    load_own<T, DP>(reinterpret_cast<const T*>(p.v) + b * p.v_b + (long)key * p.v_n + kvh * p.v_h, p.D, h, vf);
    arrived(vf);
  }
  arrived(kf);

  int t0 = !p.causal || prefix > j0 ? 0 : min(max(j0 - off, 0), p.Nq) / TQ, t1 = (p.Nq + TQ - 1) / TQ;
  int4 kr = make_int4(0, 0, 0, 0), krw = kr;
  const int4* rq = nullptr;
  const int qgroups = (p.Nq + 31) >> 5;
  if (p.rq) {
    const int kgroups = (p.Nk + 31) >> 5;
    const int4* rk = p.rk + (long)b * kgroups;
    rq = p.rq + (long)b * qgroups;
    kr = join_ranges(rk, j0 >> 5, min((j0 >> 5) + 4, kgroups) - 1);
    krw = rk[min((j0 >> 5) + wave, kgroups - 1)];
    tiles_of_documents<256>(rq, qgroups, NB, kr, t0, t1, tid, reinterpret_cast<int*>(lds + 2 * S::STAGE));
  }
  const unsigned qst = (unsigned)(p.q_n * (long)sizeof(T)), gst = (unsigned)(p.go_n * (long)sizeof(T));
  TileCopy<T, DP, TQ, 4> qc, gc;
  qc.init(wave, lane, qst, nchunk);
  gc.init(wave, lane, gst, nchunk);
  auto next = [&](int t, int4& r) {
    if (rq)
      for (; t < t1; ++t) {
        r = uniform_range(join_ranges(rq, t * NB, min(t * NB + NB, qgroups) - 1));
        if (ranges_meet(r, kr)) break;
      }
    return t;
  };
  // where the head being copied lies
  const unsigned char *qb, *gb;
  const float *lb, *db;
  auto enter = [&](int head) {
    qb = reinterpret_cast<const unsigned char*>(p.q) + (b * p.q_b + head * p.q_h) * (long)sizeof(T);
    gb = reinterpret_cast<const unsigned char*>(p.go) + (b * p.go_b + head * p.go_h) * (long)sizeof(T);
    lb = p.lse + ((long)b * p.H + head) * p.Nq * at_lw<T>();
    db = p.delta + ((long)b * p.H + head) * p.Nq;
  };
  auto stage = [&](int buf, int head, int t) {
    const int valid = p.Nq - t * TQ;
    const unsigned at = lds0 + (unsigned)buf * S::STAGE;
    qc.issue(qb + (long)t * TQ * qst, qst, nchunk, valid, at, wave, lane);
    gc.issue(gb + (long)t * TQ * gst, gst, nchunk, valid, at + S::TILE, wave, lane);
    if (wave == 0) copy_words(lb, (long)t * TQ * at_lw<T>(), (long)p.Nq * at_lw<T>() - 1, at + 2 * S::TILE, lane);
    if (wave == 1) copy_words(db, (long)t * TQ, p.Nq - 1, at + 2 * S::TILE + 256, lane);
    if (rq && wave == 2) copy_words(p.docq + (long)b * p.Nq, (long)t * TQ, p.Nq - 1, at + 2 * S::TILE + 512, lane);
    if (BIAS && wave == 3) copy_words(p.slopes, head, head, at + 2 * S::TILE + 768, lane);
  };

  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.f;

  int4 qr = make_int4(0, 0, 0, 0), qrn = qr;
  int head = head0, t = next(t0, qr), buf = 0;
  const int tfirst = t;
  const int4 qrfirst = qr;
  enter(head);
  if (t < t1) stage(0, head, t);
  while (t < t1) {
    wait_copies();
    __syncthreads();
    int tn = next(t + 1, qrn), headn = head;
    if (tn >= t1 && head + 1 < head1) { tn = tfirst; qrn = qrfirst; headn = head + 1; enter(headn); }
    if (tn < t1) stage(buf ^ 1, headn, tn);
    unsigned char* Q = lds + buf * S::STAGE;
    unsigned char* GO = Q + S::TILE;
    const float* lse = reinterpret_cast<const float*>(GO + S::TILE);
    const float* delta = lse + 64;
    const int* ids = reinterpret_cast<const int*>(delta + 64);
    const unsigned at = lds0 + (unsigned)(buf * S::STAGE), Qr = row_addr<T, DP>(at, lane), Qc = col_addr<T, DP>(at, lane);
    const int i0 = t * TQ;
    bool docmask = false, skip = p.causal && prefix <= jw && i0 + TQ - 1 + off < jw;
    if (rq) {
      if (qr.z) { zero_rows<T, DP, TQ>(Q, ids, p.Nq - i0, tid, 256); zero_rows<T, DP, TQ>(GO, ids, p.Nq - i0, tid, 256); __syncthreads(); }
      docmask = !one_document(qr, krw);
      skip |= !ranges_meet(qr, krw);
    }
    if (!skip) {
      const float mul = at_mul<T, CAP>(p), slope2 = BIAS ? delta[128] * 1.44269504088896f : 0.f;      // (behind the documents)
      const bool masked = docmask || i0 + TQ > p.Nq || (p.causal && i0 + off < jw + 31 && prefix < jw + 32);
#pragma unroll
      for (int ib = 0; ib < NB; ++ib) {
        f32x16 x, y;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = 0.f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {                                     // dp - delta: the sum starts at -delta
          const f32x4 de = *reinterpret_cast<const f32x4*>(delta + 32 * ib + 8 * g + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[4 * g + e] = de[e];
        }
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          at_mma(row_read<T, DP>(Qr, ib, ks), kf[ks], x);
          at_mma(row_read<T, DP>(Qr, ib, ks, S::TILE), S::VL ? row_read<T, DP>(VTr, 0, ks) : vf[S::VL ? 0 : ks], y);
        }
        const float away = BIAS ? (float)(key - off - i0 - 32 * ib - 4 * h) : 0.f;
        // in steps over all 16 scores: a score's own steps wait for one another
        if constexpr (CAP) {
          at_raws<T>(p, x);
#pragma unroll
          for (int r = 0; r < 16; ++r) y[r] *= at_slope<T>(x[r]);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float le[4], rest[4];
          if constexpr (at_lw<T>() == 2) {
            const f32x4 u = *reinterpret_cast<const f32x4*>(lse + 2 * (32 * ib + 8 * g + 4 * h)), v = *reinterpret_cast<const f32x4*>(lse + 2 * (32 * ib + 8 * g + 4 * h) + 4);
            le[0] = u[0]; rest[0] = u[1]; le[1] = u[2]; rest[1] = u[3]; le[2] = v[0]; rest[2] = v[1]; le[3] = v[2]; rest[3] = v[3];
          } else {
            const f32x4 u = *reinterpret_cast<const f32x4*>(lse + 32 * ib + 8 * g + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) { le[e] = u[e]; rest[e] = 0.f; }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            float z = fmaf(x[r], mul, -le[e]);
            if constexpr (BIAS) z = fmaf(-slope2, fabsf(away - (float)acc_row(r)), z);
            x[r] = at_lw<T>() == 2 ? z - rest[e] : z;
          }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(x[r]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) y[r] *= x[r];
        if (masked) {                                                     // a choice, not a product: what the mask hides may be inf or NaN
          asm volatile("" ::: "memory");                                  // (a branch of its own, not a branch or a selection per score)
          const int need = max(first, -0x20000000) - i0 - 32 * ib - 4 * h, room = p.Nq - i0 - 32 * ib - 4 * h;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            int4 di = make_int4(0, 0, 0, 0);
            if (docmask) di = *reinterpret_cast<const int4*>(ids + 32 * ib + 8 * g + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 4 * g + e, dr = e == 0 ? di.x : e == 1 ? di.y : e == 2 ? di.z : di.w;
              const bool see = (acc_row(r) >= need) & (acc_row(r) < room) & (!docmask | ((dr == mydoc) & (dr >= 0)));
              x[r] = see ? x[r] : 0.f;
              y[r] = see ? y[r] : 0.f;
            }
          }
        }
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          const frag_t pf = at_pack<T>(x, s2, xp), sf = at_pack<T>(y, s2, xs);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) {
            at_mma(col_read<T, DP>(Qc, 32 * ib + 16 * s2, d, S::TILE), pf, dv[d]);
            at_mma(col_read<T, DP>(Qc, 32 * ib + 16 * s2, d), sf, dk[d]);
          }
        }
      }
    }
    t = tn;
    qr = qrn;
    head = headn;
    buf ^= 1;
  }
  if constexpr (S::VL) wait_copies();                     // (where no tile was walked nothing else has waited for V's copy)
  if (jw + (lane & 31) < p.Nk) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const long row = (((long)b * p.Nk + key) * heads + hx) * p.D;
    const float sk = __builtin_ldexpf(p.scale, -ex), sv = 1.f / xp;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * d + 8 * g + 4 * h;
        if (c >= p.D) continue;
        if (p.part_k) {
          f32x4 wk, wv;
#pragma unroll
          for (int j = 0; j < 4; ++j) { wk[j] = dk[d][4 * g + j] * sk; wv[j] = dv[d][4 * g + j] * sv; }
          *reinterpret_cast<f32x4*>(p.part_k + row + c) = wk;
          *reinterpret_cast<f32x4*>(p.part_v + row + c) = wv;
        } else {
          t4 wk, wv;
#pragma unroll
          for (int j = 0; j < 4; ++j) { wk[j] = (T)(dk[d][4 * g + j] * sk); wv[j] = (T)(dv[d][4 * g + j] * sv); }
          *reinterpret_cast<t4*>(reinterpret_cast<T*>(p.dk) + row + c) = wk;
          *reinterpret_cast<t4*>(reinterpret_cast<T*>(p.dv) + row + c) = wv;
        }
      }
  }
}

// the heads of a group summed in their order: [rows][G][D] fp32 -> [rows][D]
template <typename T>
__global__ __launch_bounds__(256) void k_attention_group_sum(const float* pk, const float* pv, T* dk, T* dv, long n4, int G, int d4) {
  const long e = (long)blockIdx.x * 256 + threadIdx.x;
  if (e >= n4) return;
  const long row = e / d4;
  const int c = (int)(e - row * d4);
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, w = a;
  for (int g = 0; g < G; ++g) {
    const long at = ((row * G + g) * d4 + c) * 4;
    a += *reinterpret_cast<const f32x4*>(pk + at);
    w += *reinterpret_cast<const f32x4*>(pv + at);
  }
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 x, y;
#pragma unroll
  for (int j = 0; j < 4; ++j) { x[j] = (T)a[j]; y[j] = (T)w[j]; }
  *reinterpret_cast<t4*>(dk + e * 4) = x;
  *reinterpret_cast<t4*>(dv + e * 4) = y;
}

template <typename T, int DP>
int attention_bwd_launch(const AttentionParams& p, hipStream_t s) {
  typedef BwdShape<T, DP> S;
  const long rows = (long)p.B * p.Nq * p.H;
  const long bq = (long)p.B * p.H * ((p.Nq + 127) / 128), bk = (long)p.B * (p.part_k ? p.H : p.Hk) * ((p.Nk + 127) / 128);
  if ((long)p.B * p.Hk * p.slices > 0x7fffffffL) return CRAFT_ERR_UNSUPPORTED;
  if (bq > 0x7fffffffL || bk > 0x7fffffffL || (rows + 15) / 16 > 0x7fffffffL) return CRAFT_ERR_UNSUPPORTED;
  if constexpr (std::is_same<T, _Float16>::value)
    hipLaunchKernelGGL(k_attention_delta_scaled<T>, dim3((unsigned)(p.B * p.Hk * p.slices)), dim3(256), 0, s, p, const_cast<float*>(p.delta));
  else
    hipLaunchKernelGGL(k_attention_delta<T>, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, s, p, const_cast<float*>(p.delta));
  HIP_CHECK_RET(hipGetLastError());
  auto go = [&](auto tag, long blocks, int bytes) {
    constexpr auto kernel = decltype(tag)::value;
    if (const int rc = allow_lds<kernel>(bytes)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), bytes, s, p);
    return (int)hipGetLastError();
  };
  if (p.dk) {
    int rc;
    if (p.cap > 0.f) rc = p.slopes ? go(KernelTag<k_attention_dkv<T, DP, true, true>>(), bk, DkvShape<T, DP>::LDS) : go(KernelTag<k_attention_dkv<T, DP, true, false>>(), bk, DkvShape<T, DP>::LDS);
    else rc = p.slopes ? go(KernelTag<k_attention_dkv<T, DP, false, true>>(), bk, DkvShape<T, DP>::LDS) : go(KernelTag<k_attention_dkv<T, DP, false, false>>(), bk, DkvShape<T, DP>::LDS);
    if (rc) return rc;
  }
  if (p.part_k) {
    const long n4 = (long)p.B * p.Nk * p.Hk * (p.D / 4);
    if ((n4 + 255) / 256 > 0x7fffffffL) return CRAFT_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(k_attention_group_sum<T>, dim3((unsigned)((n4 + 255) / 256)), dim3(256), 0, s, p.part_k, p.part_v, reinterpret_cast<T*>(p.dk),
                       reinterpret_cast<T*>(p.dv), n4, p.H / p.Hk, p.D / 4);
    HIP_CHECK_RET(hipGetLastError());
  }
  if (!p.dq) return 0;
  if (p.cap > 0.f) return p.slopes ? go(KernelTag<k_attention_dq<T, DP, true, true>>(), bq, S::LDS) : go(KernelTag<k_attention_dq<T, DP, true, false>>(), bq, S::LDS);
  return p.slopes ? go(KernelTag<k_attention_dq<T, DP, false, true>>(), bq, S::LDS) : go(KernelTag<k_attention_dq<T, DP, false, false>>(), bq, S::LDS);
}

}  // namespace craft
