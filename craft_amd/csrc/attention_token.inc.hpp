// Attention of a few query rows over many keys (one new token of each sequence, a short chunk of tokens): the time is the keys' and values' way out
// of HBM.  The query heads that share a key head are the columns of ONE score block (row r = token r / G, head r % G of the group), so the keys are
// read once for all of them.  The keys are split over blocks and, within a block, over its waves: every wave streams its own 32-key tiles through its
// own ring of LDS stages and never meets the others before the end, where running maxima, sums and outputs are joined -- in LDS over the waves of a
// block, and by k_attention_join over the splits, each in a fixed order.
//
// 16 sequences of 32768 keys, 32 heads on 8 key heads of 128, bf16 (2.1 GB): 367 us, 5.85 TB/s (a copy of that size moves 4.9).  777 keys of 8 heads of
// 64: 6.6 us and 4.3 us for the join, behind which the host's 26 us a call stand.
#pragma once
#include "attention_tile.hpp"

namespace craft {

template <typename T, int DP> struct TokenShape {
  static constexpr int TILE = 32 * DP * (int)sizeof(T);
  static constexpr int STAGE = 2 * TILE + 512;
  static constexpr int WAVES = STAGE > 20 * 1024 ? 2 : 4;
  static constexpr int NST = STAGE * WAVES * 4 <= 144 * 1024 ? 4 : 2;     // about 64 KB of copies in flight per CU either way
  static constexpr int JOIN = WAVES * 32 * ((DP + 4) * 4 + 8);
  static constexpr int RING = WAVES * NST * STAGE;
  static constexpr int LDS = RING > JOIN ? RING : JOIN;
};

template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__((TokenShape<T, DP>::WAVES * 64)) void k_attention_token(AttentionParams p) {
  typedef TokenShape<T, DP> S;
  typedef typename AtFrag<T>::type frag_t;
  constexpr int W = S::WAVES, NST = S::NST;
  extern __shared__ __align__(512) unsigned char lds[];
  const unsigned lds0 = (unsigned)(size_t)(CRAFT_LDS unsigned char*)lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int G = p.H / p.Hk, R = p.Nq * G, nrt = (R + 31) >> 5;
  const int split = blockIdx.x % p.splits, rest = blockIdx.x / p.splits, rt = rest % nrt, bk = rest / nrt;
  const int b = bk / p.Hk, kvh = bk - b * p.Hk;
  const int off = p.Nk - p.Nq, prefix = p.prefix ? p.prefix[b] : 0;
  const int r = min(rt * 32 + (lane & 31), R - 1), i = r / G, head = kvh * G + (r - i * G), pos = i + off;
  int lim = p.causal ? min(max(pos + 1, prefix), p.Nk) : p.Nk;
  int mydoc = 0;
  if (p.docq) { mydoc = p.docq[(long)b * p.Nq + i]; if (mydoc < 0) lim = 0; }
  int lim_lo = lim, lim_hi = lim;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { lim_lo = min(lim_lo, __shfl_xor(lim_lo, o)); lim_hi = max(lim_hi, __shfl_xor(lim_hi, o)); }
  lim_lo = __builtin_amdgcn_readfirstlane(lim_lo); lim_hi = __builtin_amdgcn_readfirstlane(lim_hi);
  frag_t qf[DP / 16];
  load_own<T, DP>(reinterpret_cast<const T*>(p.q) + b * p.q_b + (long)i * p.q_n + head * p.q_h, p.D, h, qf);
  float sl[1] = {BIAS ? p.slopes[head] * 1.44269504088896f : 0.f};
  arrived(qf);
  arrived(sl);
  const float slope2 = sl[0], mul = at_mul<T, CAP>(p);

  // tiles of this split: [a0, a1); of this wave: a0 + wave, + W, ...
  const int tiles = (p.Nk + 31) >> 5, per = (tiles + p.splits - 1) / p.splits;
  const int a0 = split * per, a1 = min(min(a0 + per, tiles), (lim_hi + 31) >> 5);
  const int nchunk = p.D * (int)sizeof(T) / 16;
  const unsigned kst = (unsigned)(p.k_n * (long)sizeof(T)), vst = (unsigned)(p.v_n * (long)sizeof(T));
  typedef TileCopy<T, DP, 32, 1> Copy;
  Copy kc, vc;
  kc.init(0, lane, kst, nchunk);
  vc.init(0, lane, vst, nchunk);
  const unsigned char* kb = reinterpret_cast<const unsigned char*>(p.k) + (b * p.k_b + kvh * p.k_h) * (long)sizeof(T);
  const unsigned char* vb = reinterpret_cast<const unsigned char*>(p.v) + (b * p.v_b + kvh * p.v_h) * (long)sizeof(T);
  const unsigned ring = lds0 + (unsigned)(wave * NST * S::STAGE);
  const int last = a0 + wave + ((max(a1 - a0 - wave, 1) - 1) / W) * W;     // the wave's last tile: read again behind it, so that the count of copies in flight is fixed
  auto stage = [&](int st, int t) {
    t = min(t, last);
    const unsigned at = ring + (unsigned)st * S::STAGE;
    kc.issue(kb + (long)t * 32 * kst, kst, nchunk, p.Nk - t * 32, at, 0, lane);
    vc.issue(vb + (long)t * 32 * vst, vst, nchunk, p.Nk - t * 32, at + S::TILE, 0, lane);
    if (p.dock) copy_words(p.dock + (long)b * p.Nk, (long)t * 32, p.Nk - 1, at + 2 * S::TILE, lane);
  };

  f32x16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int q = 0; q < 16; ++q) o[d][q] = 0.f;
  float m = -INFINITY, l = 0.f;
  if (a0 + wave < a1) {
#pragma unroll
    for (int n = 0; n < NST - 1; ++n) stage(n, a0 + wave + n * W);
    int st = 0;
    for (int t = a0 + wave; t < a1; t += W) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                   // the reads of the stage that is filled next are done
      stage(st == 0 ? NST - 1 : st - 1, t + (NST - 1) * W);
      if (p.dock) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * (2 * Copy::PER + 1)) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * 2 * Copy::PER) : "memory");
      unsigned char* V = lds + (wave * NST + st) * S::STAGE + S::TILE;
      const unsigned at = ring + (unsigned)st * S::STAGE, Kr = row_addr<T, DP>(at, lane), Vc = col_addr<T, DP>(at + S::TILE, lane);
      const int* ids = reinterpret_cast<const int*>(V + S::TILE);
      const int k0 = t * 32;
      f32x16 x;
#pragma unroll
      for (int q = 0; q < 16; ++q) x[q] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) at_mma(row_read<T, DP>(Kr, 0, ks), qf[ks], x);
      const float away = BIAS ? (float)(pos - k0 - 4 * h) : 0.f;
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        float z = at_raw<T, CAP>(p, x[q]) * mul;
        if constexpr (BIAS) z = fmaf(-slope2, fabsf(away - (float)acc_row(q)), z);
        x[q] = z;
      }
      if (k0 + 32 > lim_lo) {
        const int room = lim - k0 - 4 * h;
#pragma unroll
        for (int q = 0; q < 16; ++q) x[q] = acc_row(q) < room ? x[q] : -INFINITY;
      }
      if (p.dock) {
        // (rows of a padded cache may hold anything: only this wave reads its stage, so it clears them itself)
        const int mine = ids[lane & 31];
        if (__ballot(mine < 0)) {
          for (int c = lane; c < 32 * at_cpr<T, DP>(); c += 64)
            if (ids[c / at_cpr<T, DP>()] < 0) *reinterpret_cast<f32x4*>(V + c * 16) = f32x4{0.f, 0.f, 0.f, 0.f};
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int4 d = *reinterpret_cast<const int4*>(ids + 8 * g + 4 * h);
          x[4 * g + 0] = d.x == mydoc ? x[4 * g + 0] : -INFINITY;
          x[4 * g + 1] = d.y == mydoc ? x[4 * g + 1] : -INFINITY;
          x[4 * g + 2] = d.z == mydoc ? x[4 * g + 2] : -INFINITY;
          x[4 * g + 3] = d.w == mydoc ? x[4 * g + 3] : -INFINITY;
        }
      }
      float mt = x[0];
#pragma unroll
      for (int q = 1; q < 16; ++q) mt = fmaxf(mt, x[q]);
      mt = fmaxf(mt, at_other_half(mt));
      if (__ballot(mt > m + 8.f)) {
        const float mn = fmaxf(m, mt), alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int q = 0; q < 16; ++q) o[d][q] *= alpha;
      }
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int q = 0; q < 16; ++q) { x[q] = __builtin_amdgcn_exp2f(x[q] - ref); l += x[q]; }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const frag_t pf = at_pack<T>(x, s2);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) at_mma(col_read<T, DP>(Vc, 16 * s2, d), pf, o[d]);
      }
      st = st == NST - 1 ? 0 : st + 1;
    }
  }
  l += at_other_half(l);

  // ---- join the waves
  wait_copies();
  __syncthreads();
  float* jo = reinterpret_cast<float*>(lds);                               // [W][32][DP + 4]
  float* jm = jo + W * 32 * (DP + 4);                                      // [W][32] maxima, then sums
  float* jl = jm + W * 32;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = o[d][4 * g + j];
      *reinterpret_cast<f32x4*>(jo + (wave * 32 + (lane & 31)) * (DP + 4) + 32 * d + 8 * g + 4 * h) = w;
    }
  if (h == 0) { jm[wave * 32 + (lane & 31)] = m; jl[wave * 32 + (lane & 31)] = l; }
  __syncthreads();
  typedef T t4 __attribute__((ext_vector_type(4)));
  const int cols = p.D / 4;
  for (int e = tid; e < 32 * cols; e += W * 64) {
    const int row = e / cols, c = (e - row * cols) * 4, rr = rt * 32 + row;
    if (rr >= R) continue;
    float M = jm[row], L = 0.f;
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, jm[w * 32 + row]);
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = jm[w * 32 + row], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
      L += f * jl[w * 32 + row];
      a += f * *reinterpret_cast<const f32x4*>(jo + (w * 32 + row) * (DP + 4) + c);
    }
    if (p.splits == 1) {
      const float inv = L > 0.f ? 1.f / L : 0.f;
      const int ii = rr / G, hh = kvh * G + (rr - ii * G);
      t4 w4;
#pragma unroll
      for (int j = 0; j < 4; ++j) w4[j] = (T)(a[j] * inv);
      *reinterpret_cast<t4*>(reinterpret_cast<T*>(p.out) + b * p.o_b + (long)ii * p.o_n + hh * p.o_h + c) = w4;
    } else {
      const long row_id = ((long)bk * R + rr) * p.splits + split;
      *reinterpret_cast<f32x4*>(p.part_o + row_id * p.D + c) = a;
      if (c == 0) { p.part_ml[2 * row_id] = M; p.part_ml[2 * row_id + 1] = L; }
    }
  }
}

// one block of 64 lanes per (batch, key head, row): the splits joined in their order
template <typename T>
__global__ __launch_bounds__(64) void k_attention_join(AttentionParams p) {
  const int G = p.H / p.Hk, R = p.Nq * G, lane = threadIdx.x;
  const int bk = blockIdx.x / R, rr = blockIdx.x - bk * R, b = bk / p.Hk, kvh = bk - b * p.Hk, i = rr / G, head = kvh * G + (rr - i * G);
  const long row = (long)blockIdx.x * p.splits;
  const float* ml = p.part_ml + 2 * row;
  float M = -INFINITY;
  for (int s = lane; s < p.splits; s += 64) M = fmaxf(M, ml[2 * s]);
  M = wave_max(M);
  float a0 = 0.f, a1 = 0.f, L = 0.f;
  const int c = 2 * lane;
  for (int s = 0; s < p.splits; ++s) {
    const float ms = ml[2 * s], f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - M);
    L += f * ml[2 * s + 1];
    if (c < p.D) {
      const float2 v = *reinterpret_cast<const float2*>(p.part_o + (row + s) * p.D + c);
      a0 += f * v.x; a1 += f * v.y;
    }
  }
  if (c < p.D) {
    const float inv = L > 0.f ? 1.f / L : 0.f;
    T* o = reinterpret_cast<T*>(p.out) + b * p.o_b + (long)i * p.o_n + head * p.o_h + c;
    o[0] = (T)(a0 * inv);
    o[1] = (T)(a1 * inv);
  }
}

template <typename T, int DP>
int attention_token_launch(const AttentionParams& p, hipStream_t s) {
  typedef TokenShape<T, DP> S;
  const int R = p.Nq * (p.H / p.Hk), nrt = (R + 31) / 32;
  const long blocks = (long)p.B * p.Hk * nrt * p.splits, rows = (long)p.B * p.Hk * R;
  if (blocks > 0x7fffffffL || rows > 0x7fffffffL) return CRAFT_ERR_UNSUPPORTED;
  auto go = [&](auto tag) {
    constexpr auto kernel = decltype(tag)::value;
    if (const int rc = allow_lds<kernel>(S::LDS)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(S::WAVES * 64), S::LDS, s, p);
    return (int)hipGetLastError();
  };
  int rc;
  if (p.cap > 0.f) rc = p.slopes ? go(KernelTag<k_attention_token<T, DP, true, true>>()) : go(KernelTag<k_attention_token<T, DP, true, false>>());
  else rc = p.slopes ? go(KernelTag<k_attention_token<T, DP, false, true>>()) : go(KernelTag<k_attention_token<T, DP, false, false>>());
  if (rc || p.splits == 1) return rc;
  hipLaunchKernelGGL(k_attention_join<T>, dim3((unsigned)rows), dim3(64), 0, s, p);
  return (int)hipGetLastError();
}

}  // namespace craft
