// Orthogonalising updates by Newton-Schulz products, for a list of matrices at once.
//
//   X <- G / (|G|_F + eps)   (G transposed where it has more rows than columns: m <= n)
//   steps times:  A = X X^T,   B = b A + c A^2,   X <- a X + B X
//
// Each step is three products whose sizes differ from matrix to matrix, and each needs the one before it: three launches a step for the WHOLE list, a
// block per output tile of any matrix (a table of the matrices travels in the kernel's arguments).  A and A^2 are symmetric: only their lower tiles are
// computed and written twice.
//
// Arithmetic: fp32-class.  Every operand is two fp16 planes hi + lo of its value times a power of two (22 bits and more: the scales bring the largest
// possible entry, which the spectrum bounds, just below fp16's largest number, so that lo keeps its bits), every product three MFMAs with fp32 sums.  The
// planes take the four bytes of an fp32 value.  The norm is summed in fp64: its error would scale the whole result.
//
// All operands are read along their rows: X (rows of n) for X X^T, A for A^2, and B with X^T (rows of m) for B X; the last product's epilogue writes both X
// and X^T.  X^T is kept twice (blocks of one strip read it whole while others write).  Rows and columns are padded to 64 with zeros, which the products keep.
#include "attention_tile.hpp"
#include "../../include/craft_hip.h"

namespace craft {

constexpr int NS_MAX_JOBS = 60;                      // (the table fits a kernel's 4 KB of arguments)
constexpr int NS_NORM_BLOCKS = 32;                   // partial norms of a matrix, at most

struct NsJob {
  const void* src; void* dst;
  long ld_src, ld_dst;
  long ws;                                           // byte offset of the matrix' operands in the workspace
  int rows, cols;                                    // of src and dst
  int mp, np;                                        // of X, padded
  int first;                                         // its first block in this launch
  int nb;                                            // blocks of its norm
};
struct NsParams {
  NsJob job[NS_MAX_JOBS];
  int n, dtype;
  unsigned char* ws;
  double* norm;                                      // [jobs][NS_NORM_BLOCKS]
  float eps, c0, c1;                                 // epilogue: c0 * (old value) + c1 * (product), scales folded in
  float s_x;                                         // scale of X
  int last, flip;                                    // last step; which of the two X^T is read
};

static_assert(sizeof(NsParams) <= 4096, "kernel arguments");
// a matrix' operands: X, X^T, X^T again, A, B; each [2][rows][cols] fp16
__host__ __device__ __forceinline__ long ns_x_bytes(int mp, int np) { return 4l * mp * np; }
__host__ __device__ __forceinline__ long ns_bytes(int mp, int np) { return 3 * ns_x_bytes(mp, np) + 2 * 4l * mp * mp; }
__device__ __forceinline__ _Float16* ns_x(const NsParams& p, const NsJob& j) { return reinterpret_cast<_Float16*>(p.ws + j.ws); }
__device__ __forceinline__ _Float16* ns_xt(const NsParams& p, const NsJob& j, int which) { return reinterpret_cast<_Float16*>(p.ws + j.ws + (1 + which) * ns_x_bytes(j.mp, j.np)); }
__device__ __forceinline__ _Float16* ns_a(const NsParams& p, const NsJob& j, int which) { return reinterpret_cast<_Float16*>(p.ws + j.ws + 3 * ns_x_bytes(j.mp, j.np) + which * 4l * j.mp * j.mp); }

__device__ __forceinline__ int ns_job(const NsParams& p, int block) {
  int lo = 0, hi = p.n;
  while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (p.job[m].first <= block) lo = m; else hi = m; }
  return lo;
}
__device__ __forceinline__ float ns_get(const void* p, long i, int dtype) {
  return dtype == CRAFT_PREC_F32 ? reinterpret_cast<const float*>(p)[i] : dtype == CRAFT_PREC_F16 ? (float)reinterpret_cast<const _Float16*>(p)[i] : (float)reinterpret_cast<const __bf16*>(p)[i];
}
__device__ __forceinline__ void ns_put(void* p, long i, int dtype, float v) {
  if (dtype == CRAFT_PREC_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == CRAFT_PREC_F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
  else reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
}
// 8 values as two planes
__device__ __forceinline__ void ns_split(const float (&v)[8], _Float16* hi, _Float16* lo) {
  f16x8 h, l;
#pragma unroll
  for (int i = 0; i < 8; ++i) { h[i] = (_Float16)v[i]; l[i] = (_Float16)(v[i] - (float)h[i]); }
  *reinterpret_cast<f16x8*>(hi) = h;
  *reinterpret_cast<f16x8*>(lo) = l;
}

// partial sums of squares: job.nb blocks share a matrix' rows
__global__ __launch_bounds__(256) void k_ns_norm(NsParams p) {
  __shared__ double red[4];
  const int id = ns_job(p, blockIdx.x);
  const NsJob& j = p.job[id];
  const int q = blockIdx.x - j.first;
  double s = 0.0;
  const long total = (long)j.rows * j.cols;
  for (long e = (long)q * 256 + threadIdx.x; e < total; e += (long)j.nb * 256) {
    const long r = e / j.cols;
    const double v = ns_get(j.src, r * j.ld_src + (e - r * j.cols), p.dtype);
    s += v * v;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) p.norm[id * NS_NORM_BLOCKS + q] = (red[0] + red[1]) + (red[2] + red[3]);
}

// G -> X and X^T, a block per 64 x 64 tile of X
__global__ __launch_bounds__(256) void k_ns_init(NsParams p) {
  __shared__ float t[64][65];
  const int id = ns_job(p, blockIdx.x);
  const NsJob& j = p.job[id];
  const int q = blockIdx.x - j.first, tn = j.np >> 6, ti = (q / tn) * 64, tj = (q % tn) * 64;
  double sum = 0.0;
  for (int b = 0; b < j.nb; ++b) sum += p.norm[id * NS_NORM_BLOCKS + b];
  const float f = (float)((double)p.s_x / (sqrt(sum) + (double)p.eps));
  const bool flip = j.rows > j.cols;
  const int r0 = flip ? tj : ti, c0 = flip ? ti : tj;                    // the tile of G
  for (int e = threadIdx.x; e < 64 * 64; e += 256) {
    const int r = e >> 6, c = e & 63;
    const float v = r0 + r < j.rows && c0 + c < j.cols ? ns_get(j.src, (long)(r0 + r) * j.ld_src + c0 + c, p.dtype) * f : 0.f;
    if (flip) t[c][r] = v; else t[r][c] = v;
  }
  __syncthreads();
  _Float16* x = ns_x(p, j);
  _Float16* xt = ns_xt(p, j, 0);
  const long plane = (long)j.mp * j.np;
  for (int e = threadIdx.x; e < 512; e += 256) {
    const int r = e >> 3, c = (e & 7) * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = t[r][c + i];
    _Float16* o = x + (long)(ti + r) * j.np + tj + c;
    ns_split(v, o, o + plane);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = t[c + i][r];
    o = xt + (long)(tj + r) * j.mp + ti + c;
    ns_split(v, o, o + plane);
  }
}

// One 64 x 64 tile of P Q^T, both read along their rows of K straight into MFMA operands (no operand is used twice within a wave, so LDS would not save
// a load): the 8 waves of a block share K, their partial tiles are summed in LDS in the order of the waves.
//   PHASE 0: A = X X^T;  1: B = b A + c A A^T;  2: X = a X + B (X^T)^T
template <int PHASE>
__global__ __launch_bounds__(512) void k_ns_product(NsParams p) {
  extern __shared__ __align__(16) float part[];                          // [8][64][64]
  const int id = ns_job(p, blockIdx.x);
  const NsJob& j = p.job[id];
  const int q = blockIdx.x - j.first, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  int ti, tj;
  if constexpr (PHASE < 2) {                                             // lower tiles, row by row
    ti = (int)((sqrtf(8.f * (float)q + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= q) ++ti;
    while (ti * (ti + 1) / 2 > q) --ti;
    tj = q - ti * (ti + 1) / 2;
  } else {
    const int tm = j.mp >> 6;
    tj = q / tm;
    ti = q - tj * tm;
  }
  const int K = PHASE == 0 ? j.np : j.mp;
  const _Float16* P = PHASE == 0 ? ns_x(p, j) : ns_a(p, j, PHASE - 1);
  const _Float16* Q = PHASE == 2 ? ns_xt(p, j, p.flip) : P;
  const long pp = PHASE == 0 ? (long)j.mp * j.np : (long)j.mp * j.mp, qp = PHASE == 1 ? pp : (long)j.mp * j.np;
  const int nk = K >> 4, k0 = nk * wave / 8, k1 = nk * (wave + 1) / 8;
  f32x16 acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
  const _Float16* pr = P + (long)(ti * 64 + (lane & 31)) * K + 8 * h;
  const _Float16* qr = Q + (long)(tj * 64 + (lane & 31)) * K + 8 * h;
#pragma unroll 2
  for (int k = k0; k < k1; ++k) {
    f16x8 ph[2], pl[2], qh[2], ql[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      ph[a] = *reinterpret_cast<const f16x8*>(pr + (long)a * 32 * K + 16 * k);
      pl[a] = *reinterpret_cast<const f16x8*>(pr + (long)a * 32 * K + 16 * k + pp);
      qh[a] = *reinterpret_cast<const f16x8*>(qr + (long)a * 32 * K + 16 * k);
      ql[a] = *reinterpret_cast<const f16x8*>(qr + (long)a * 32 * K + 16 * k + qp);
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        at_mma(pl[a], qh[b], acc[a][b]);
        at_mma(ph[a], ql[b], acc[a][b]);
        at_mma(ph[a], qh[b], acc[a][b]);
      }
  }
  float* mine = part + wave * 4096;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(32 * a + acc_row(r) + 4 * h) * 64 + 32 * b + (lane & 31)] = acc[a][b][r];
  __syncthreads();
  // thread: row tid / 8, 8 columns
  const int row = tid >> 3, c = (tid & 7) * 8;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += part[w * 4096 + row * 64 + c + i];
  const int gi = ti * 64 + row, gj = tj * 64 + c;
  if constexpr (PHASE == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= p.c1;
  } else if constexpr (PHASE == 1) {
    const f16x8 oh = *reinterpret_cast<const f16x8*>(P + (long)gi * K + gj), ol = *reinterpret_cast<const f16x8*>(P + (long)gi * K + gj + pp);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p.c0 * ((float)oh[i] + (float)ol[i]) + p.c1 * v[i];
  } else {
    // the old X: every thread reads its column group of X^T's rows
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const _Float16* o = Q + (long)(gj + i) * K + gi;
      v[i] = p.c0 * ((float)o[0] + (float)o[qp]) + p.c1 * v[i];
    }
  }
  __syncthreads();                                                       // (all partial tiles are read: the first becomes the finished tile)
#pragma unroll
  for (int i = 0; i < 8; ++i) part[row * 65 + c + i] = v[i];
  __syncthreads();
  if (PHASE == 2 && p.last) {
    const bool flip = j.rows > j.cols;
    const int r0 = flip ? tj * 64 : ti * 64, c0 = flip ? ti * 64 : tj * 64;
    for (int e = tid; e < 4096; e += 512) {
      const int r = e >> 6, cc = e & 63;
      if (r0 + r < j.rows && c0 + cc < j.cols) ns_put(j.dst, (long)(r0 + r) * j.ld_dst + c0 + cc, p.dtype, flip ? part[cc * 65 + r] : part[r * 65 + cc]);
    }
    return;
  }
  float u[8];                                                            // the tile's transpose: row `row`, 8 columns
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = part[(c + i) * 65 + row];
  if constexpr (PHASE < 2) {
    _Float16* out = ns_a(p, j, PHASE);
    const long plane = (long)j.mp * j.mp;
    _Float16* o = out + (long)gi * j.mp + gj;
    ns_split(v, o, o + plane);
    if (ti != tj) {
      o = out + (long)(tj * 64 + row) * j.mp + ti * 64 + c;
      ns_split(u, o, o + plane);
    }
  } else {
    const long plane = (long)j.mp * j.np;
    _Float16* o = ns_x(p, j) + (long)gi * j.np + gj;
    ns_split(v, o, o + plane);
    o = ns_xt(p, j, p.flip ^ 1) + (long)(tj * 64 + row) * j.mp + ti * 64 + c;
    ns_split(u, o, o + plane);
  }
}

// ---- the momentum in front of the products and the update behind them, over ranges of flat buffers
constexpr int MUON_MAX_SEGS = 128, MUON_CHUNK = 4096;
struct MuonSeg { long off, n; float scale; int first; };
struct MuonParams {
  MuonSeg seg[MUON_MAX_SEGS];
  int n;
  float *param, *buf, *update;
  const float* grad;
  const int* state;                                  // craft_loss_scale_update's record: word 4 found_inf, word 5 gm (float)
  float momentum, lr, decay;
  int nesterov;
};

// APPLY 0: buf = momentum buf + g, update = nesterov ? g + momentum buf : buf (g = gm x gradient);  1: param = decay param - lr scale update.
// A skipped step (found_inf) writes nothing.
template <int APPLY>
__global__ __launch_bounds__(256) void k_muon(MuonParams p) {
  if (p.state[4]) return;
  int lo = 0, hi = p.n;
  while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (p.seg[m].first <= (int)blockIdx.x) lo = m; else hi = m; }
  const MuonSeg& g = p.seg[lo];
  const float gm = __int_as_float(p.state[5]), f = p.lr * g.scale;
  const long c0 = (long)(blockIdx.x - g.first) * MUON_CHUNK, c1 = min(c0 + MUON_CHUNK, g.n);
  for (long c = c0 + threadIdx.x; c < c1; c += 256) {
    const long e = g.off + c;
    if constexpr (APPLY == 0) {
      const float d = p.grad[e] * gm, b = p.momentum * p.buf[e] + d;
      p.buf[e] = b;
      p.update[e] = p.nesterov ? d + p.momentum * b : b;
    } else {
      p.param[e] = p.param[e] * p.decay - f * p.update[e];
    }
  }
}

static int muon_launch(MuonParams& p, const long* segs, const float* scales, int n, bool apply, hipStream_t s) {
  for (int i0 = 0; i0 < n; i0 += MUON_MAX_SEGS) {
    p.n = n - i0 < MUON_MAX_SEGS ? n - i0 : MUON_MAX_SEGS;
    long blocks = 0;
    for (int i = 0; i < p.n; ++i) {
      const long* d = segs + 2 * (i0 + i);
      if (d[0] < 0 || d[1] <= 0) return CRAFT_ERR_ARG;
      p.seg[i] = MuonSeg{d[0], d[1], scales ? scales[i0 + i] : 1.f, (int)blocks};
      blocks += (d[1] + MUON_CHUNK - 1) / MUON_CHUNK;
      if (blocks > 0x7fffffffL) return CRAFT_ERR_UNSUPPORTED;
    }
    if (apply) hipLaunchKernelGGL(k_muon<1>, dim3((unsigned)blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL(k_muon<0>, dim3((unsigned)blocks), dim3(256), 0, s, p);
    HIP_CHECK_RET(hipGetLastError());
  }
  return 0;
}

}  // namespace craft

using namespace craft;

extern "C" int craft_orthogonalize(const long* jobs, int n, const float* coeffs, int steps, float eps, float s_x, float s_a, float s_b, int dtype, void* ws,
                                   long ws_bytes, void* stream) {
  if (!jobs || !coeffs || n <= 0 || n > NS_MAX_JOBS || steps < 1 || steps > 64 || dtype < 0 || dtype > 2) return CRAFT_ERR_ARG;
  if (!(eps >= 0.f) || !(s_x > 0.f) || !(s_a > 0.f) || !(s_b > 0.f) || (reinterpret_cast<uintptr_t>(ws) & 255) || !ws) return CRAFT_ERR_ARG;
  NsParams p = {};
  p.n = n; p.dtype = dtype; p.eps = eps; p.s_x = s_x;
  p.norm = reinterpret_cast<double*>(ws);
  long at = (long)n * NS_NORM_BLOCKS * 8;
  p.ws = reinterpret_cast<unsigned char*>(ws);
  long lower = 0, tiles = 0, norms = 0;
  for (int i = 0; i < n; ++i) {
    const long* d = jobs + 6 * i;                                        // src, ld_src, dst, ld_dst, rows, cols
    NsJob& j = p.job[i];
    if (!d[0] || !d[2] || d[4] <= 0 || d[5] <= 0 || d[1] < 0 || d[3] < d[5]) return CRAFT_ERR_ARG;
    if (d[4] > 65536 || d[5] > 1l << 24 || (d[5] > 65536 && d[4] > 65536)) return CRAFT_ERR_UNSUPPORTED;
    j.src = reinterpret_cast<const void*>(d[0]); j.ld_src = d[1]; j.dst = reinterpret_cast<void*>(d[2]); j.ld_dst = d[3];
    j.rows = (int)d[4]; j.cols = (int)d[5];
    const int m = j.rows < j.cols ? j.rows : j.cols, nn = j.rows < j.cols ? j.cols : j.rows;
    if (m > 32768) return CRAFT_ERR_UNSUPPORTED;
    j.mp = (m + 63) / 64 * 64; j.np = (nn + 63) / 64 * 64;
    j.ws = at;
    at += ns_bytes(j.mp, j.np);
    const long el = (long)j.rows * j.cols;
    j.nb = (int)(el / 8192 < 1 ? 1 : el / 8192 > NS_NORM_BLOCKS ? NS_NORM_BLOCKS : el / 8192);
    norms += j.nb;
    lower += (long)(j.mp / 64) * (j.mp / 64 + 1) / 2;
    tiles += (long)(j.mp / 64) * (j.np / 64);
  }
  if (at > ws_bytes) return CRAFT_ERR_ARG;
  if (lower > 0x7fffffffL || tiles > 0x7fffffffL) return CRAFT_ERR_UNSUPPORTED;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto number = [&](int what) {                                          // first blocks: 0 norms, 1 lower tiles, 2 all tiles
    int first = 0;
    for (int i = 0; i < n; ++i) {
      NsJob& j = p.job[i];
      const int tm = j.mp / 64, tn = j.np / 64;
      j.first = first;
      first += what == 0 ? j.nb : what == 1 ? tm * (tm + 1) / 2 : tm * tn;
    }
  };
  constexpr int LDS = 8 * 4096 * 4;
  const void* kernels[3] = {reinterpret_cast<const void*>(k_ns_product<0>), reinterpret_cast<const void*>(k_ns_product<1>), reinterpret_cast<const void*>(k_ns_product<2>)};
  for (const void* k : kernels) HIP_CHECK_RET(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
  number(0);
  hipLaunchKernelGGL(k_ns_norm, dim3((unsigned)norms), dim3(256), 0, s, p);
  HIP_CHECK_RET(hipGetLastError());
  number(2);
  hipLaunchKernelGGL(k_ns_init, dim3((unsigned)tiles), dim3(256), 0, s, p);
  HIP_CHECK_RET(hipGetLastError());
  for (int t = 0; t < steps; ++t) {
    const float a = coeffs[3 * t], b = coeffs[3 * t + 1], c = coeffs[3 * t + 2];
    p.flip = t & 1;
    p.last = t == steps - 1;
    number(1);
    p.c0 = 0.f; p.c1 = s_a / (s_x * s_x);
    hipLaunchKernelGGL(k_ns_product<0>, dim3((unsigned)lower), dim3(512), LDS, s, p);
    HIP_CHECK_RET(hipGetLastError());
    p.c0 = b * s_b / s_a; p.c1 = c * s_b / (s_a * s_a);
    hipLaunchKernelGGL(k_ns_product<1>, dim3((unsigned)lower), dim3(512), LDS, s, p);
    HIP_CHECK_RET(hipGetLastError());
    number(2);
    p.c0 = p.last ? a / s_x : a; p.c1 = (p.last ? 1.f / s_x : 1.f) / s_b;   // B X carries s_b s_x; the last one leaves without a scale
    hipLaunchKernelGGL(k_ns_product<2>, dim3((unsigned)tiles), dim3(512), LDS, s, p);
    HIP_CHECK_RET(hipGetLastError());
  }
  return 0;
}

extern "C" int craft_muon_momentum(const float* grad, float* buf, float* update, const long* segs, int n, float momentum, int nesterov, const void* state,
                                   void* stream) {
  if (!grad || !buf || !update || !segs || n <= 0 || !state || !(momentum >= 0.f && momentum < 1.f)) return CRAFT_ERR_ARG;
  MuonParams p = {};
  p.grad = grad; p.buf = buf; p.update = update; p.momentum = momentum; p.nesterov = nesterov; p.state = reinterpret_cast<const int*>(state);
  return muon_launch(p, segs, nullptr, n, false, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int craft_muon_apply(float* param, const float* update, const long* segs, const float* scales, int n, float lr, float weight_decay, const void* state,
                                void* stream) {
  if (!param || !update || !segs || !scales || n <= 0 || !state) return CRAFT_ERR_ARG;
  MuonParams p = {};
  p.param = param; p.update = const_cast<float*>(update); p.lr = lr; p.decay = 1.f - lr * weight_decay; p.state = reinterpret_cast<const int*>(state);
  return muon_launch(p, segs, scales, n, true, reinterpret_cast<hipStream_t>(stream));
}
