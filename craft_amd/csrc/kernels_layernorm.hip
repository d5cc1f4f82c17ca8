// LayerNorm with weights, forward and backward, any width up to 16384, fp32 / fp16 / bf16 rows.
//
//   y = xn w + b,  xn = (x - mean) rstd;      dx = rstd (g - mean(g) - xn mean(g xn)) with g = dy w,   dw = sum_rows dy xn,   db = sum_rows dy
//
// HBM-bound: x is read once forward (and the row held in registers for its two statistics, mean first, then the squares about it, in fp32), x and dy once
// backward.  A row belongs to TPR threads (16 of a wave, a wave, 4 waves, 16 waves: the smallest that holds it with at most 4 vectors a thread).
// The weight's and the bias' gradients are summed on the way: a thread owns the same columns of every row it meets, so its sums stay in registers over the
// block's whole share of the rows; the row groups of a block are joined in LDS, the blocks by k_layer_norm_sum -- each in a fixed order, no atomics.
// Vectors are 16 bytes at any alignment (unaligned loads and stores are native): an odd width costs its last vector element by element, nothing else.
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

template <typename T> struct LnVec { static constexpr int N = 16 / sizeof(T); typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))); };

template <typename T, typename W, int N>
__device__ __forceinline__ void ln_load(const W* p, int col, int C, float (&f)[N]) {
  typedef W vec __attribute__((ext_vector_type(N), aligned(sizeof(W))));
  if (col + N <= C) {
    const vec v = *reinterpret_cast<const vec*>(p + col);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = col + i < C ? (float)p[col + i] : 0.f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void ln_store(T* p, int col, int C, const float (&f)[N]) {
  typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  if (col + N <= C) {
    vec v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)f[i];
    *reinterpret_cast<vec*>(p + col) = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) if (col + i < C) p[col + i] = (T)f[i];
  }
}

// sums over the TPR threads of a row, on all of them.  TPR > 64: `red` [2][waves of the row][2], used alternately, so one barrier a call is enough
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

template <int TPR> constexpr int ln_threads() { return TPR > 256 ? TPR : 256; }

template <typename T, typename W, int TPR, int NV>
__global__ __launch_bounds__((ln_threads<TPR>())) void k_layer_norm_fwd(LayerNormParams p) {
  constexpr int N = LnVec<T>::N, RPB = ln_threads<TPR>() / TPR;
  __shared__ float red[2 * 2 * 16];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const long row = (long)blockIdx.x * RPB + group;
  if (TPR <= 64 && row >= p.rows) return;             // (TPR > 64: one row per block, always there)
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
  float v[NV][N];
  float s[1] = {0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j) ln_load<T>(x, (j * TPR + t) * N, p.C, v[j]);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) s[0] += v[j][i];
  ln_sum<TPR, 1>(s, red, t >> 6, 0);
  const float inv = 1.f / (float)p.C, mean = s[0] * inv;
  s[0] = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = (j * TPR + t) * N + i < p.C ? v[j][i] - mean : 0.f;
      v[j][i] = d;
      s[0] += d * d;
    }
  ln_sum<TPR, 1>(s, red, t >> 6, 1);
  const float rstd = 1.f / sqrtf(s[0] * inv + p.eps);
  T* y = reinterpret_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int col = (j * TPR + t) * N;
    if (col >= p.C) continue;
    float w[N], b[N];
    if (p.w) ln_load<T>(reinterpret_cast<const W*>(p.w), col, p.C, w);
    if (p.b) ln_load<T>(reinterpret_cast<const W*>(p.b), col, p.C, b);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float o = v[j][i] * rstd;
      if (p.w) o *= w[i];
      if (p.b) o += b[i];
      v[j][i] = o;
    }
    ln_store<T>(y, col, p.C, v[j]);
  }
  if (p.mean && t == 0) { p.mean[row] = mean; p.rstd[row] = rstd; }
}

// a block walks over the rows row0 + blockIdx.x * RPB, + gridDim.x * RPB, ...
template <typename T, typename W, int TPR, int NV>
__global__ __launch_bounds__((ln_threads<TPR>())) void k_layer_norm_bwd(LayerNormParams p) {
  constexpr int N = LnVec<T>::N, TH = ln_threads<TPR>(), RPB = TH / TPR;
  extern __shared__ float sums[];                     // [2][C] when the row groups of a block are joined
  __shared__ float red[2 * 2 * 16];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  float dw[NV][N], db[NV][N], w[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < N; ++i) { dw[j][i] = db[j][i] = 0.f; w[j][i] = 1.f; }
    if (p.w) ln_load<T>(reinterpret_cast<const W*>(p.w), (j * TPR + t) * N, p.C, w[j]);
  }
  const float inv = 1.f / (float)p.C;
  int phase = 0;
  for (long row0 = (long)blockIdx.x * RPB; row0 < p.rows; row0 += (long)gridDim.x * RPB) {
    const long row = row0 + group;
    if (TPR > 64 || row < p.rows) {                   // (whole groups of at most a wave)
      const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
      const T* dy = reinterpret_cast<const T*>(p.dy) + row * p.lddy;
      float v[NV][N], g[NV][N];
#pragma unroll
      for (int j = 0; j < NV; ++j) { ln_load<T>(x, (j * TPR + t) * N, p.C, v[j]); ln_load<T>(dy, (j * TPR + t) * N, p.C, g[j]); }
      const float mean = p.mean[row], rstd = p.rstd[row];
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float xn = (v[j][i] - mean) * rstd, d = g[j][i];          // (behind the width d = 0: nothing is added)
          dw[j][i] += d * xn;
          db[j][i] += d;
          const float gw = d * w[j][i];
          s[0] += gw;
          s[1] += gw * xn;
          v[j][i] = xn;
          g[j][i] = gw;
        }
      if (p.dx) {
        ln_sum<TPR, 2>(s, red, t >> 6, phase);
        phase ^= 1;
        const float m0 = s[0] * inv, m1 = s[1] * inv;
        T* dx = reinterpret_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int col = (j * TPR + t) * N;
          if (col >= p.C) continue;
#pragma unroll
          for (int i = 0; i < N; ++i) g[j][i] = (g[j][i] - m0 - v[j][i] * m1) * rstd;
          ln_store<T>(dx, col, p.C, g[j]);
        }
      }
    }
  }
  if (!p.part) return;
  float* out = p.part + (long)blockIdx.x * 2 * p.C;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) { ln_store<float>(out, (j * TPR + t) * N, p.C, dw[j]); ln_store<float>(out + p.C, (j * TPR + t) * N, p.C, db[j]); }
  } else {
    for (int q = 0; q < RPB; ++q) {                   // the groups one behind the other
      if (group == q) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int col = (j * TPR + t) * N + i;
            if (col < p.C) {
              sums[col] = (q ? sums[col] : 0.f) + dw[j][i];
              sums[p.C + col] = (q ? sums[p.C + col] : 0.f) + db[j][i];
            }
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * p.C; c += TH) out[c] = sums[c];
  }
}

// [blocks][2][C] -> dw, db; a block of 256: 32 columns x 8 shares of the blocks
template <typename W>
__global__ __launch_bounds__(256) void k_layer_norm_sum(const float* part, int blocks, int C, W* dw, W* db) {
  __shared__ float red[8][33];
  const int c = threadIdx.x & 31, q = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < 2 * C)
    for (int b = q; b < blocks; b += 8) s += part[(long)b * 2 * C + col];
  red[q][c] = s;
  __syncthreads();
  if (q == 0 && col < 2 * C) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][c];
    if (col < C) { if (dw) dw[col] = (W)s; }
    else if (db) db[col - C] = (W)s;
  }
}

template <typename T, typename W>
static int layer_norm_run(const LayerNormParams& p, int blocks, void* dw, void* db, hipStream_t s) {
  constexpr int N = LnVec<T>::N;
  auto go = [&](auto fwd, auto bwd, int tpr, int th) {
    const int rpb = th / tpr;
    if (!p.dy) {
      const long grid = (p.rows + rpb - 1) / rpb;
      if (grid > 0x7fffffffL) return CRAFT_ERR_UNSUPPORTED;
      hipLaunchKernelGGL(fwd, dim3((unsigned)grid), dim3(th), 0, s, p);
      return (int)hipGetLastError();
    }
    const size_t lds = p.part && rpb > 1 ? (size_t)2 * p.C * 4 : 0;
    hipLaunchKernelGGL(bwd, dim3((unsigned)blocks), dim3(th), lds, s, p);
    HIP_CHECK_RET(hipGetLastError());
    if (p.part) hipLaunchKernelGGL(k_layer_norm_sum<W>, dim3((unsigned)((2 * p.C + 31) / 32)), dim3(256), 0, s, p.part, blocks, p.C, (W*)dw, (W*)db);
    return (int)hipGetLastError();
  };
#define LN_GO(TPR, NV) go(k_layer_norm_fwd<T, W, TPR, NV>, k_layer_norm_bwd<T, W, TPR, NV>, TPR, ln_threads<TPR>())
  const int nv = (p.C + N - 1) / N;                    // vectors of a row
  if (nv <= 16) return LN_GO(16, 1);
  if (nv <= 64) return LN_GO(64, 1);
  if (nv <= 128) return LN_GO(64, 2);
  if (nv <= 256) return LN_GO(64, 4);
  if (nv <= 512) return LN_GO(256, 2);
  if (nv <= 1024) return LN_GO(256, 4);
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
