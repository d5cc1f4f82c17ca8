// LayerNorm with weights, forward and backward, any width up to 16384, fp32 / fp16 / bf16 rows.
//
//   y = xn w + b,  xn = (x - mean) rstd;      dx = rstd (g - mean(g) - xn mean(g xn)) with g = dy w,   dw = sum_rows dy xn,   db = sum_rows dy
//
// HBM-bound: x is read once forward (and the row held in registers for its two statistics, mean first, then the squares about it, in fp32), x and dy once
// backward.  A row belongs to TPR threads (16 of a wave, a wave, up to 16 waves), with one vector each up to 1024 vectors.
// The weight's and the bias' gradients are summed on the way: a thread owns the same columns of every row it meets, so its sums stay in registers over the
// block's whole share of the rows; the row groups of a block are joined in LDS, the blocks by k_layer_norm_sum -- each in a fixed order, no atomics.
// Vectors are 16 bytes at any alignment (unaligned loads and stores are native): an odd width moves its last vector back (LnCols).
//
// 16384 rows of 4096 bf16: forward 52 us (5.2 TB/s), backward 81 us (5.0 TB/s), the sum over the blocks 4 us; a copy of 256 MiB moves 5.5 TB/s, one of
// 2 GiB 4.9.  28672 rows of 256 fp32: 12 us (4.8 TB/s).  1441 rows of 1027 fp16: 6 + 11 + 4 us, latency.  Above 8192 columns the backward kernel's 1024 threads
// keep 128 .. 448 bytes each in scratch (16-bit rows of an odd width from 4096 on 36): 4096 rows of 16384, forward and backward, bf16 322 us (2.1 TB/s), fp32 494 (2.7);
// 8192 rows of 8192 take 163 (4.1 TB/s) and 272 us (4.9).
#include <type_traits>
#include "launch.hpp"
#include "../../include/craft_hip.h"

namespace craft {

constexpr int LN_MAX_WIDTH = 16384;

struct LayerNormParams {
  const void *x, *w, *b, *dy;
  void *y, *dx;
  long ldx, ldy, lddy, lddx;
  float *mean, *rstd;                 // [rows]
  float* part;                        // backward: [blocks][2][C] partial weight / bias gradients (null: not wanted)
  long rows;
  int C;
  float eps;
};

template <typename T> struct LnVec { static constexpr int N = 16 / sizeof(T); };

// A thread's vector j holds columns base .. base + N - 1 of the row, of which those below `lo` belong to its neighbour: the last vector of a row whose
// width is no multiple of N is moved back to end with the row, so that every load is one whole vector with no branch around it (a branch per vector made
// the loads of a row wait for one another: 28 us instead of 11 for the gradients of 1441 rows of 1027).  A row narrower than a vector goes element by element.
template <int N>
struct LnCols {
  int base, lo;
  __device__ __forceinline__ LnCols(int col, int C) {
    base = col + N <= C ? col : C >= N ? C - N : 0;
    lo = col;                                          // a vector behind the row owns nothing
  }
  __device__ __forceinline__ bool mine(int i, int C) const { return base + i >= lo && base + i < C; }
};

// the neighbour's columns get the values that the neighbour writes
template <typename T, int N>
__device__ __forceinline__ void ln_store(T* p, const LnCols<N>& k, int C, const float (&f)[N]) {
  typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  if (k.lo >= C) return;
  if (C >= N) {
    vec v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)f[i];
    *reinterpret_cast<vec*>(p + k.base) = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) if (k.base + i < C) p[k.base + i] = (T)f[i];
  }
}

// sums over the TPR threads of a row, on all of them.  TPR > 64: `red` [2][waves of the row][2] of the row's group, used alternately, so one barrier a
// call is enough (all threads of the block have to come)
template <int TPR, int NS>
__device__ __forceinline__ void ln_sum(float (&s)[NS], float* red, int wave_in_row, int phase) {
#pragma unroll
  for (int k = 0; k < NS; ++k)
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) s[k] += __shfl_xor(s[k], o);
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    float* r = red + phase * NW * 2;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < NS; ++k) r[wave_in_row * 2 + k] = s[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      s[k] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) s[k] += r[w * 2 + k];
    }
  }
}

// TH threads: TH / TPR rows at a time; a block walks over the rows blockIdx.x * RPB + group, + gridDim.x * RPB, ... and has the next row's vectors on
// their way while this one is worked on.
template <typename T, typename W, int TPR, int NV, int TH>
__global__ __launch_bounds__(TH) void k_layer_norm_fwd(LayerNormParams p) {
  constexpr int N = LnVec<T>::N, RPB = TH / TPR, NW = TPR > 64 ? TPR / 64 : 1;
  typedef T tvec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  __shared__ float red[RPB][2 * NW * 2];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const bool whole = p.C >= N;                        // (uniform)
  auto cols = [&](int j) { return LnCols<N>((j * TPR + t) * N, p.C); };
  const float inv = 1.f / (float)p.C;
  // the weights stay in registers, in their own type: loads arrive in order, so one inside the loop would wait for the next row
  typedef W wvec __attribute__((ext_vector_type(N), aligned(sizeof(W))));
  wvec w[NV], b[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int base = cols(j).base;
#pragma unroll
    for (int i = 0; i < N; ++i) { w[j][i] = (W)1.f; b[j][i] = (W)0.f; }
    auto get = [&](const void* q, wvec& v) {
      const W* c = reinterpret_cast<const W*>(q);
      if (whole) v = *reinterpret_cast<const wvec*>(c + base);
      else {
#pragma unroll
        for (int i = 0; i < N; ++i) if (base + i < p.C) v[i] = c[base + i];
      }
    };
    if (p.w) get(p.w, w[j]);
    if (p.b) get(p.b, b[j]);
  }
  tvec xv[NV];
  auto fetch = [&](long r) {                           // (a group without a row goes through the last one and keeps nothing of it)
    const T* q = reinterpret_cast<const T*>(p.x) + (r < p.rows ? r : p.rows - 1) * p.ldx;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int base = cols(j).base;
      if (whole) xv[j] = *reinterpret_cast<const tvec*>(q + base);
      else {
#pragma unroll
        for (int i = 0; i < N; ++i) xv[j][i] = base + i < p.C ? q[base + i] : q[0];
      }
    }
  };
  const long step = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + group;
  fetch(row);
  for (long row0 = (long)blockIdx.x * RPB; row0 < p.rows; row0 += step, row += step) {
    const bool on = row < p.rows;
    float v[NV][N];
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const LnCols<N> k = cols(j);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[j][i] = (float)xv[j][i];
        s[0] += k.mine(i, p.C) ? v[j][i] : 0.f;
      }
    }
    if (row0 + step < p.rows) fetch(row + step);
    ln_sum<TPR, 1>(s, red[group], t >> 6, 0);
    const float mean = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const LnCols<N> k = cols(j);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[j][i] -= mean;
        s[0] += k.mine(i, p.C) ? v[j][i] * v[j][i] : 0.f;
      }
    }
    ln_sum<TPR, 1>(s, red[group], t >> 6, 1);
    const float rstd = 1.f / sqrtf(s[0] * inv + p.eps);
    if (!on) continue;                                 // (behind the row's barriers)
    T* y = reinterpret_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[j][i] = v[j][i] * rstd * (float)w[j][i] + (float)b[j][i];
      ln_store<T, N>(y, cols(j), p.C, v[j]);
    }
    if (p.mean && t == 0) { p.mean[row] = mean; p.rstd[row] = rstd; }
  }
}

// 1024 threads: 1024 / TPR rows at a time; a block walks over the rows blockIdx.x * RPB + group, + gridDim.x * RPB, ...  The next row's vectors are on
// their way while this one is worked on; vectors stay in their own type until used (twice: once for the sums, once for dx), which leaves the registers to
// the sums of the weight's gradients.  TAIL: the width is no multiple of the vector (the masks it needs cost registers).
template <typename T, typename W, int TPR, int NV, bool TAIL>
__global__ __launch_bounds__(1024) void k_layer_norm_bwd(LayerNormParams p) {
  constexpr int N = LnVec<T>::N, RPB = 1024 / TPR, NW = TPR > 64 ? TPR / 64 : 1;
  typedef T tvec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  typedef W wvec __attribute__((ext_vector_type(N), aligned(sizeof(W))));
  extern __shared__ float sums[];                     // [2][C]: the row groups of a block are joined here
  __shared__ float red[RPB][2 * NW * 2];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const bool whole = !TAIL || p.C >= N;               // (uniform)
  auto cols = [&](int j) { return LnCols<N>((j * TPR + t) * N, p.C); };
  auto mine = [&](int j, int i) { return TAIL ? cols(j).mine(i, p.C) : (j * TPR + t) * N < p.C; };
  auto get = [&](auto* q, int base, auto& v) {
    if (whole) v = *reinterpret_cast<const typename std::remove_reference<decltype(v)>::type*>(q + base);
    else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = base + i < p.C ? q[base + i] : q[0];
    }
  };
  float dw[NV][N], db[NV][N];
  wvec w[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < N; ++i) { dw[j][i] = db[j][i] = 0.f; w[j][i] = (W)1.f; }
    if (p.w) get(reinterpret_cast<const W*>(p.w), cols(j).base, w[j]);
  }
  const float inv = 1.f / (float)p.C;
  int phase = 0;
  const long step = (long)gridDim.x * RPB;
  tvec xv[NV], gv[NV];
  float mean, rstd;
  auto fetch = [&](long r) {                           // (a group without a row goes through the last one and keeps nothing of it)
    const long row = r < p.rows ? r : p.rows - 1;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      get(reinterpret_cast<const T*>(p.x) + row * p.ldx, cols(j).base, xv[j]);
      get(reinterpret_cast<const T*>(p.dy) + row * p.lddy, cols(j).base, gv[j]);
    }
    mean = p.mean[row];
    rstd = p.rstd[row];
  };
  long row = (long)blockIdx.x * RPB + group;
  fetch(row);
  for (long row0 = (long)blockIdx.x * RPB; row0 < p.rows; row0 += step, row += step) {
    const bool on = row < p.rows;
    tvec x[NV], g[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) { x[j] = xv[j]; g[j] = gv[j]; }
    const float mu = mean, rs = rstd;
    if (row0 + step < p.rows) fetch(row + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = on && mine(j, i) ? (float)g[j][i] : 0.f, xn = ((float)x[j][i] - mu) * rs, gw = d * (float)w[j][i];
        dw[j][i] += d * xn;
        db[j][i] += d;
        s[0] += gw;
        s[1] += gw * xn;
      }
    if (p.dx) {
      ln_sum<TPR, 2>(s, red[group], t >> 6, phase);
      phase ^= 1;
      if (on) {
        const float m0 = s[0] * inv, m1 = s[1] * inv;
        T* dx = reinterpret_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float o[N];
#pragma unroll
          for (int i = 0; i < N; ++i) o[i] = ((float)g[j][i] * (float)w[j][i] - m0 - ((float)x[j][i] - mu) * rs * m1) * rs;
          ln_store<T, N>(dx, cols(j), p.C, o);
        }
      }
    }
  }
  if (!p.part) return;
  float* out = p.part + (long)blockIdx.x * 2 * p.C;
  for (int q = 0; q < RPB; ++q) {                     // the groups one behind the other
    if (group == q) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (mine(j, i)) {
            float* c = (RPB > 1 ? sums : out) + cols(j).base + i;
            c[0] = (q ? c[0] : 0.f) + dw[j][i];
            c[p.C] = (q ? c[p.C] : 0.f) + db[j][i];
          }
    }
    if (RPB > 1) __syncthreads();
  }
  if constexpr (RPB > 1)
    for (int c = threadIdx.x; c < 2 * p.C; c += 1024) out[c] = sums[c];
}

// [blocks][2][C] -> dw, db; a block of 512: 32 columns x 16 shares of the blocks
template <typename W>
__global__ __launch_bounds__(512) void k_layer_norm_sum(const float* part, int blocks, int C, W* dw, W* db) {
  __shared__ float red[16][33];
  const int c = threadIdx.x & 31, q = threadIdx.x >> 5, col = min((int)blockIdx.x * 32 + c, 2 * C - 1);
  float s = 0.f;
#pragma unroll 8
  for (int b = q; b < blocks; b += 16) s += part[(long)b * 2 * C + col];
  red[q][c] = s;
  __syncthreads();
  if (q == 0 && (int)blockIdx.x * 32 + c < 2 * C) {
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][c];
    if (col < C) { if (dw) dw[col] = (W)s; }
    else if (db) db[col - C] = (W)s;
  }
}

template <typename T, typename W>
static int layer_norm_run(const LayerNormParams& p, int blocks, void* dw, void* db, hipStream_t s) {
  constexpr int N = LnVec<T>::N;
  auto go = [&](auto fwd, auto bwd, int tpr) {
    if (!p.dy) {
      const int th = tpr > 512 ? tpr : 512, rpb = th / tpr;
      // what the card holds at once: three blocks of 512 threads to a compute unit (up to 74 registers), two of 1024 of one fp32 vector each (48 registers; us,
      // 16384 rows of 4096: 107, one block 143), one of those of 16 bits or more vectors (68 .. 128; 8192 rows of 8192 bf16: 68 with one, 66 with two).
      // 16384 rows of 1024 bf16 with 256 / 512 / 768 / 1024 / 2048 blocks: 25 / 17 / 15 / 17 / 18; of 4096: 87 / 58 / 50 / 58 / 54.
      const long most = (p.rows + rpb - 1) / rpb, full = th == 512 ? 768 : sizeof(T) == 4 && p.C <= 4096 ? 512 : 256;
      hipLaunchKernelGGL(fwd, dim3((unsigned)(most < full ? most : full)), dim3(th), 0, s, p);
      return (int)hipGetLastError();
    }
    const int rpb = 1024 / tpr;
    const long most = (p.rows + rpb - 1) / rpb;
    const int grid = most < blocks ? (int)most : blocks;
    const size_t lds = p.part && rpb > 1 ? (size_t)2 * p.C * 4 : 0;          // (32 KB at most: wider rows have a block of their own)
    hipLaunchKernelGGL(bwd, dim3((unsigned)grid), dim3(1024), lds, s, p);
    HIP_CHECK_RET(hipGetLastError());
    if (p.part) hipLaunchKernelGGL(k_layer_norm_sum<W>, dim3((unsigned)((2 * p.C + 31) / 32)), dim3(512), 0, s, p.part, grid, p.C, (W*)dw, (W*)db);
    return (int)hipGetLastError();
  };
  const int nv = (p.C + N - 1) / N;                    // vectors of a row
  const bool tail = p.C % N != 0;
#define LN_GO(TPR, NV) go(k_layer_norm_fwd<T, W, TPR, NV, (TPR > 512 ? TPR : 512)>, tail ? k_layer_norm_bwd<T, W, TPR, NV, true> : k_layer_norm_bwd<T, W, TPR, NV, false>, TPR)
  if (nv <= 16) return LN_GO(16, 1);
  if (nv <= 64) return LN_GO(64, 1);
  if (nv <= 128) return LN_GO(128, 1);
  if (nv <= 256) return LN_GO(256, 1);
  if (nv <= 512) return LN_GO(512, 1);
  if (nv <= 1024) return LN_GO(1024, 1);
  if constexpr (sizeof(T) == 4) if (nv > 2048) return LN_GO(1024, 4);
  return LN_GO(1024, 2);
#undef LN_GO
}

static int layer_norm_dispatch(const LayerNormParams& p, int dtype, int wdtype, int blocks, void* dw, void* db, hipStream_t s) {
  if (dtype == CRAFT_PREC_F32) return wdtype == CRAFT_PREC_F32 ? layer_norm_run<float, float>(p, blocks, dw, db, s) : CRAFT_ERR_UNSUPPORTED;
  if (dtype == CRAFT_PREC_F16)
    return wdtype == CRAFT_PREC_F32 ? layer_norm_run<_Float16, float>(p, blocks, dw, db, s)
         : wdtype == CRAFT_PREC_F16 ? layer_norm_run<_Float16, _Float16>(p, blocks, dw, db, s) : CRAFT_ERR_UNSUPPORTED;
  if (dtype == CRAFT_PREC_BF16)
    return wdtype == CRAFT_PREC_F32 ? layer_norm_run<__bf16, float>(p, blocks, dw, db, s)
         : wdtype == CRAFT_PREC_BF16 ? layer_norm_run<__bf16, __bf16>(p, blocks, dw, db, s) : CRAFT_ERR_UNSUPPORTED;
  return CRAFT_ERR_ARG;
}

static int layer_norm_check(const void* x, const void* y, long ldx, long ldy, long rows, int C, float eps, int dtype) {
  if (rows <= 0 || C <= 0 || !x || !y || !(eps >= 0.f)) return CRAFT_ERR_ARG;
  if (C > LN_MAX_WIDTH) return CRAFT_ERR_UNSUPPORTED;
  if (ldx < 0 || ldy < C) return CRAFT_ERR_ARG;
  const uintptr_t m = dtype == CRAFT_PREC_F32 ? 3 : 1;
  return ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & m) ? CRAFT_ERR_ALIGN : 0;
}

}  // namespace craft

using namespace craft;

extern "C" {

int craft_layer_norm_fwd(const void* x, long ldx, const void* w, const void* b, long rows, int C, float eps, int dtype, int wdtype, void* y, long ldy,
                         float* mean, float* rstd, void* stream) {
  const int rc = layer_norm_check(x, y, ldx, ldy, rows, C, eps, dtype);
  if (rc) return rc;
  if ((mean == nullptr) != (rstd == nullptr)) return CRAFT_ERR_ARG;
  LayerNormParams p = {};
  p.x = x; p.ldx = ldx; p.w = w; p.b = b; p.rows = rows; p.C = C; p.eps = eps; p.y = y; p.ldy = ldy; p.mean = mean; p.rstd = rstd;
  return layer_norm_dispatch(p, dtype, wdtype, 0, nullptr, nullptr, reinterpret_cast<hipStream_t>(stream));
}

int craft_layer_norm_bwd(const void* x, long ldx, const void* dy, long lddy, const void* w, const float* mean, const float* rstd, long rows, int C,
                         int dtype, int wdtype, void* dx, long lddx, void* dw, void* db, float* ws, int blocks, void* stream) {
  const int rc = layer_norm_check(x, dy, ldx, lddy < C ? C : lddy, rows, C, 0.f, dtype);
  if (rc) return rc;
  if (!mean || !rstd || lddy < 0 || (dx && lddx < C) || blocks <= 0 || blocks > (1 << 20)) return CRAFT_ERR_ARG;
  if ((dw || db) && !ws) return CRAFT_ERR_ARG;
  if (!dx && !dw && !db) return 0;
  LayerNormParams p = {};
  p.x = x; p.ldx = ldx; p.dy = dy; p.lddy = lddy; p.w = w; p.rows = rows; p.C = C; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.dx = dx; p.lddx = lddx; p.part = dw || db ? ws : nullptr;
  return layer_norm_dispatch(p, dtype, wdtype, blocks, dw, db, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
