// Orthogonalising updates by Newton-Schulz products, for a list of matrices at once.
//
//   X <- G / (|G|_F + eps)   (G transposed where it has more rows than columns: m <= n)
//   steps times:  A = X X^T,   B = b A + c A^2,   X <- a X + B X
//
// Each step is three products whose sizes differ from matrix to matrix, and each needs the one before it: three launches a step for the WHOLE list, a
// block per output tile of any matrix.  A and A^2 are symmetric: only their lower tiles are computed, and written twice.
//
// Arithmetic: fp32-class.  Every operand is two fp16 planes hi + lo of its value times a power of two (22 bits and more: the scales bring the largest
// possible entry, which the spectrum bounds, just below fp16's largest number, so that lo keeps its bits), every product three MFMAs with fp32 sums.  The
// planes take the four bytes of an fp32 value.  The norm is summed in fp64: its error would scale the whole result.
//
// All operands are read along their rows: X (rows of n) for X X^T, A for A^2, and B with X^T (rows of m) for B X; the last product's epilogue writes both X
// and X^T.  X^T is kept twice (blocks of one strip read it whole while others write).
//
// One 2048 x 8192 matrix: 1.86 ms, of which B X five times 202 us (three fp16 products: 1.02 PF/s, 73 % of a large library product's 1.39), X X^T 114 us
// and 14 us for the sum of its shares, B 34 + 18 us.  The 53 matrices of the CRAFT model (64 x 147 .. 1024 x 256): 306 .. 324 us in 18 launches (its operations
// are 33 us).  B X 26 us a step: it moves 142 MB (a strip of X^T once for each 64 rows of tiles, the old X, X and X^T written), 5.4 TB/s.  X X^T 22 us: 192 blocks,
// a tile's whole K in each, up to 20 steps of a wave one behind the other's loads.  B 7 us.  One 256 x 256: 106 us, 18 dependent launches of 4 .. 8 us.
//
// Rows and columns are padded to 64 (128) with zeros, which the products keep.
#include "attention_tile.hpp"
#include "../../include/craft_hip.h"

namespace craft {

constexpr int NS_MAX_JOBS = 60;                      // (the table fits the 4 KB of k_ns_table's arguments)
constexpr int NS_NORM_BLOCKS = 256;                  // partial norms of a matrix, at most
constexpr int NS_MAX_BIG = 16;                       // larger ones in one set of launches
constexpr long NS_PART_BYTES = 512l * 65536;         // partial tiles of the larger ones
constexpr int NS_SMALL = 256;                        // smaller sides up to here: k_ns_gram / k_ns_update

struct NsJob {
  const void* src; void* dst;
  long ld_src, ld_dst;
  long ws;                                           // byte offset of the matrix' operands in the workspace
  int rows, cols;                                    // of src and dst
  int mp, np;                                        // of X, padded
  short nb;                                          // blocks of its norm
  short share[3];                                    // k_ns_big: shares of K in each of the three products
};
// The kinds of launches: a matrix' first block in each.
enum { NS_NORM, NS_INIT, NS_LOWER, NS_ALL, NS_SHARED, NS_KINDS = NS_SHARED + 3 };
// The matrices' table, in the workspace: kernel arguments lie in host memory, and a search through them costs a kernel ten microseconds.  Which matrix a
// block belongs to: every lane holds one first block, a ballot finds the last that is not behind.
struct NsTable {
  NsJob job[64];
  int first[NS_KINDS][64];                           // (INT_MAX behind the last)
  int part[3][64];                                   // k_ns_big: a matrix' first partial tile
};
struct NsLoad { NsJob job[NS_MAX_JOBS]; int n, side, big; NsTable* table; };
struct NsParams {
  const NsTable* table;
  int dtype;
  unsigned char* ws;
  double* norm;                                      // [jobs][NS_NORM_BLOCKS]
  float eps, c0, c1;                                 // epilogue: c0 * (old value) + c1 * (product), scales folded in
  float s_x;                                         // scale of X
  float* part;                                       // k_ns_big: partial tiles
  int last, flip;                                    // last step; which of the two X^T is read
};
constexpr long NS_TABLE_BYTES = 8192;
static_assert(sizeof(NsLoad) <= 4096 && sizeof(NsTable) <= NS_TABLE_BYTES, "kernel arguments and the table in the workspace");

// a matrix' operands: X, X^T, X^T again, A, B; each [2][rows][cols] fp16
__host__ __device__ __forceinline__ long ns_x_bytes(int mp, int np) { return 4l * mp * np; }
__host__ __device__ __forceinline__ long ns_bytes(int mp, int np) { return 3 * ns_x_bytes(mp, np) + 2 * 4l * mp * mp; }
__device__ __forceinline__ _Float16* ns_x(const NsParams& p, const NsJob& j) { return reinterpret_cast<_Float16*>(p.ws + j.ws); }
__device__ __forceinline__ _Float16* ns_xt(const NsParams& p, const NsJob& j, int which) { return reinterpret_cast<_Float16*>(p.ws + j.ws + (1 + which) * ns_x_bytes(j.mp, j.np)); }
__device__ __forceinline__ _Float16* ns_a(const NsParams& p, const NsJob& j, int which) { return reinterpret_cast<_Float16*>(p.ws + j.ws + 3 * ns_x_bytes(j.mp, j.np) + which * 4l * j.mp * j.mp); }

// blocks of a matrix in a launch of each kind
__host__ __device__ __forceinline__ long ns_blocks(const NsJob& j, int kind, int side) {
  const long tm = j.mp / side, tn = j.np / side, lower = tm * (tm + 1) / 2, all = tm * tn;
  switch (kind) {
    case NS_NORM: return j.nb;
    case NS_INIT: return (long)(j.mp / 64) * (j.np / 64);
    case NS_LOWER: return lower;
    case NS_ALL: return all;
    default: return (kind < NS_SHARED + 2 ? lower : all) * j.share[kind - NS_SHARED];
  }
}
__global__ __launch_bounds__(64) void k_ns_table(NsLoad l) {
  const int i = threadIdx.x;
  NsTable* t = l.table;
  if (i < l.n) t->job[i] = l.job[i];
  for (int kind = 0; kind < NS_KINDS; ++kind) {
    long at = i < l.n ? ns_blocks(l.job[i], kind, l.side) : 0;
    const long mine = at;
    for (int o = 1; o < 64; o <<= 1) {                                   // sum over the lanes in front
      const long v = __shfl_up(at, o);
      if (i >= o) at += v;
    }
    t->first[kind][i] = i < l.n ? (int)(at - mine) : 0x7fffffff;
    if (kind >= NS_SHARED) t->part[kind - NS_SHARED][i] = (int)(at - mine);
  }
}
__device__ __forceinline__ int ns_job(const NsTable* t, int kind, int block, int& local) {
  const int f = t->first[kind][threadIdx.x & 63];
  const int id = 63 - __builtin_clzll(__ballot(f <= block));
  local = block - __builtin_amdgcn_readlane(f, id);
  return id;
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

// partial sums of squares: job.nb blocks share a matrix' pieces of 8192 columns of a row (of the whole matrix, where its rows are contiguous)
__global__ __launch_bounds__(1024) void k_ns_norm(NsParams p) {
  __shared__ double red[16];
  int q;
  const int id = ns_job(p.table, NS_NORM, blockIdx.x, q);
  const NsJob j = p.table->job[id];
  const bool flat = j.ld_src == j.cols;
  const long rows = flat ? 1 : j.rows, cols = flat ? (long)j.rows * j.cols : j.cols, segs = (cols + 8191) >> 13, items = rows * segs;
  double s = 0.0;
  for (long e = q; e < items; e += j.nb) {
    const long r = e / segs, c0 = (e - r * segs) * 8192 + threadIdx.x;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + 1024 * i < cols ? ns_get(j.src, r * j.ld_src + c0 + 1024 * i, p.dtype) : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += (double)v[i] * (double)v[i];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 16; ++w) s += red[w];
    p.norm[id * NS_NORM_BLOCKS + q] = s;
  }
}

// Operands lie in the order in which a wave reads them: 32 rows x 16 columns of one plane are 1 KiB, 16 bytes for each lane -- row lane & 31, columns
// 8 (lane >> 5) .. + 7 -- so that a load of an MFMA operand is one contiguous KiB.  (Rows behind one another, a load touched 32 lines and used a quarter
// of each, and 8 waves' lines overran the L1: X X^T of 128 x 2560 took 57 us.)  Element offset of the 8 columns at k (a multiple of 8) of a row:
__device__ __forceinline__ long ns_at(int row, int k, int K) {
  return (((long)(row >> 5) * (K >> 4) + (k >> 4)) * 64 + ((k >> 3) & 1) * 32 + (row & 31)) * 8;
}

// G -> X and X^T, a block per 64 x 64 tile of X
__global__ __launch_bounds__(256) void k_ns_init(NsParams p) {
  __shared__ float t[64][65];
  __shared__ double red[4];
  int q;
  const int id = ns_job(p.table, NS_INIT, blockIdx.x, q);
  const NsJob j = p.table->job[id];
  const int tn = j.np >> 6, ti = (q / tn) * 64, tj = (q % tn) * 64;
  double sum = (int)threadIdx.x < j.nb ? p.norm[id * NS_NORM_BLOCKS + threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = (red[0] + red[1]) + (red[2] + red[3]);
  // the factor as a fraction and a power of two: it is past fp32's range for a norm below 1e-34 and no eps, and subnormal for one above 1e38
  int e2;
  const float f = (float)frexp((double)p.s_x / (sqrt(sum) + (double)p.eps), &e2);
  const bool flip = j.rows > j.cols;
  const int r0 = flip ? tj : ti, c0 = flip ? ti : tj;                    // the tile of G
  for (int e = threadIdx.x; e < 64 * 64; e += 256) {
    const int r = e >> 6, c = e & 63;
    const float v = r0 + r < j.rows && c0 + c < j.cols ? ldexpf(ns_get(j.src, (long)(r0 + r) * j.ld_src + c0 + c, p.dtype), e2) * f : 0.f;
    if (flip) t[c][r] = v; else t[r][c] = v;
  }
  __syncthreads();
  _Float16* x = ns_x(p, j);
  _Float16* xt = ns_xt(p, j, 0);
  const long plane = (long)j.mp * j.np;
  for (int e = threadIdx.x; e < 512; e += 256) {
    const int r = e & 63, c = (e >> 6) * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = t[r][c + i];
    _Float16* o = x + ns_at(ti + r, tj + c, j.np);
    ns_split(v, o, o + plane);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = t[c + i][r];
    o = xt + ns_at(tj + r, ti + c, j.mp);
    ns_split(v, o, o + plane);
  }
}

__device__ __forceinline__ void ns_lower(int q, int& ti, int& tj) {      // tile q of the lower triangle, row by row
  ti = (int)((sqrtf(8.f * (float)q + 1.f) - 1.f) * 0.5f);
  while ((ti + 1) * (ti + 2) / 2 <= q) ++ti;
  while (ti * (ti + 1) / 2 > q) --ti;
  tj = q - ti * (ti + 1) / 2;
}
// acc += one 16-step of a 32 x 32 product of two-plane operands (lo lo is below the sums' own rounding)
__device__ __forceinline__ void ns_mma(const f16x8& ph, const f16x8& pl, const f16x8& qh, const f16x8& ql, f32x16& acc) {
  at_mma(pl, qh, acc);
  at_mma(ph, ql, acc);
  at_mma(ph, qh, acc);
}
__device__ __forceinline__ f16x8 ns_ld(const _Float16* q) { return *reinterpret_cast<const f16x8*>(q); }

// What leaves a finished tile t ([N][N + 1] in LDS): the last step's result to dst ...
template <int N>
__device__ __forceinline__ void ns_result(const NsParams& p, const NsJob& j, const float* t, int ti, int tj, int tid, int threads) {
  const bool flip = j.rows > j.cols;
  const int r0 = (flip ? tj : ti) * N, c0 = (flip ? ti : tj) * N;
  for (int e = tid; e < N * N; e += threads) {
    const int r = e / N, c = e % N;
    if (r0 + r < j.rows && c0 + c < j.cols) ns_put(j.dst, (long)(r0 + r) * j.ld_dst + c0 + c, p.dtype, flip ? t[c * (N + 1) + r] : t[r * (N + 1) + c]);
  }
}
// ... or the tile as planes at (ti, tj) of `out` (rows of K) and its transpose at (tj, ti) of `outt` (rows of Kt)
template <int N>
__device__ __forceinline__ void ns_planes(const float* t, _Float16* out, int K, long plane, _Float16* outt, int Kt, int ti, int tj, int tid, int threads) {
#pragma unroll 1
  for (int e = tid; e < N * N / 8; e += threads) {
    const int row = e % N, c = (e / N) * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = t[row * (N + 1) + c + i];
    _Float16* o = out + ns_at(ti * N + row, tj * N + c, K);
    ns_split(v, o, o + plane);
    if (outt) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = t[(c + i) * (N + 1) + row];
      o = outt + ns_at(tj * N + row, ti * N + c, Kt);
      ns_split(v, o, o + plane);
    }
  }
}

// ---- matrices whose smaller side is at most 256: bound by the launches' and loads' latency
// PHASE 0: A = X X^T, 1: B = b A + c A A, a block per 64 x 64 tile: the 8 waves share K and read both operands straight into MFMA operands (a wave would use none twice, so LDS would
// not save a load); their partial tiles are summed in LDS in the order of the waves.
template <int PHASE>
__global__ __launch_bounds__(512) void k_ns_gram(NsParams p) {
  extern __shared__ __align__(16) float part[];                          // [8][64][64]
  int q;
  const NsJob j = p.table->job[ns_job(p.table, NS_LOWER, blockIdx.x, q)];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  int ti, tj;
  ns_lower(q, ti, tj);
  const int K = PHASE == 0 ? j.np : j.mp;
  const _Float16* X = PHASE == 0 ? ns_x(p, j) : ns_a(p, j, 0);
  const long plane = (long)j.mp * K;
  const int nk = K >> 4, k0 = nk * wave / 8, k1 = nk * (wave + 1) / 8;
  f32x16 acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
  // a diagonal tile has one operand
  const bool diag = ti == tj;
  const _Float16* pr = X + ns_at(ti * 64, 0, K) + lane * 8;
  const _Float16* qr = X + ns_at(tj * 64, 0, K) + lane * 8;
  const long half = (long)(K >> 4) * 512;                                // 32 rows on
  f16x8 f[2][2][2], g[2][2][2];                                          // [P, Q][32 rows][plane]; the next step's on their way
  auto fetch = [&](int k) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        g[0][a][e] = ns_ld(pr + a * half + (long)k * 512 + e * plane);
        if (!diag) g[1][a][e] = ns_ld(qr + a * half + (long)k * 512 + e * plane);
      }
  };
  if (k0 < k1) fetch(k0);
#pragma unroll 1
  for (int k = k0; k < k1; ++k) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int e = 0; e < 2; ++e) { f[0][a][e] = g[0][a][e]; f[1][a][e] = diag ? g[0][a][e] : g[1][a][e]; }
    if (k + 1 < k1) fetch(k + 1);
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b) ns_mma(f[0][a][0], f[0][a][1], f[1][b][0], f[1][b][1], acc[a][b]);
  }
  float* mine = part + wave * 4096;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(32 * a + acc_row(r) + 4 * h) * 64 + 32 * b + (lane & 31)] = acc[a][b][r];
  __syncthreads();
  const int row = tid >> 3, c = (tid & 7) * 8;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += part[w * 4096 + row * 64 + c + i];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= p.c1;
  if constexpr (PHASE == 1) {
    const _Float16* old = X + ns_at(64 * ti + row, 64 * tj + c, K);
    const f16x8 oh = ns_ld(old), ol = ns_ld(old + plane);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += p.c0 * ((float)oh[i] + (float)ol[i]);
  }
  __syncthreads();                                                       // (all partial tiles are read: the first becomes the finished tile)
#pragma unroll
  for (int i = 0; i < 8; ++i) part[row * 65 + c + i] = v[i];
  __syncthreads();
  _Float16* A = ns_a(p, j, PHASE);
  ns_planes<64>(part, A, j.mp, (long)j.mp * j.mp, ti == tj ? nullptr : A, j.mp, ti, tj, tid, 512);
}

// X <- a X + B X, a block per 64 x 64 tile: 4 waves of 32 x 32, operands from memory straight into registers, the next step's on their way.  Small blocks:
// four and more to a compute unit hide one another's latency.  (With B made again in every block, instead of in a launch of its own, the
// model's step took 40 us here instead of 7 + 28.)
__global__ __launch_bounds__(256) void k_ns_update(NsParams p) {
  __shared__ float part[64 * 65];
  int q;
  const NsJob j = p.table->job[ns_job(p.table, NS_ALL, blockIdx.x, q)];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, l31 = lane & 31, sa = wave & 1, sb = wave >> 1;
  const int tm = j.mp >> 6, tj = q / tm, ti = q - tj * tm, K = j.mp, nk = K >> 4;
  const long pb = (long)K * K, px = (long)K * j.np;
  const _Float16* br = ns_a(p, j, 1) + ns_at(64 * ti + 32 * sa, 0, K) + lane * 8;
  const _Float16* xr = ns_xt(p, j, p.flip) + ns_at(64 * tj + 32 * sb, 0, K) + lane * 8;
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  f16x8 f[2][4];                                                         // [step][B hi, B lo, X^T hi, X^T lo]
  auto fetch = [&](int k) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const long at = (long)(k + u) * 512;
      f[u][0] = ns_ld(br + at); f[u][1] = ns_ld(br + at + pb); f[u][2] = ns_ld(xr + at); f[u][3] = ns_ld(xr + at + px);
    }
  };
  fetch(0);
#pragma unroll 1
  for (int k = 0; k < nk; k += 2) {                                      // (nk is a multiple of 4)
    f16x8 g[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) g[u][e] = f[u][e];
    if (k + 2 < nk) fetch(k + 2);
#pragma unroll
    for (int u = 0; u < 2; ++u) ns_mma(g[u][0], g[u][1], g[u][2], g[u][3], acc);
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) part[(32 * sa + acc_row(r) + 4 * h) * 65 + 32 * sb + l31] = acc[r] * p.c1;
  __syncthreads();
#pragma unroll
  for (int e = tid; e < 512; e += 256) {
    const int row = e & 63, c = (e >> 6) * 8;
    const _Float16* old = ns_x(p, j) + ns_at(64 * ti + row, 64 * tj + c, j.np);       // (only this block touches its tile of X)
    const f16x8 oh = ns_ld(old), ol = ns_ld(old + px);
#pragma unroll
    for (int i = 0; i < 8; ++i) part[row * 65 + c + i] += p.c0 * ((float)oh[i] + (float)ol[i]);
  }
  __syncthreads();
  if (p.last) ns_result<64>(p, j, part, ti, tj, tid, 256);
  else ns_planes<64>(part, ns_x(p, j), j.np, px, ns_xt(p, j, p.flip ^ 1), j.mp, ti, tj, tid, 256);
}

// ---- larger matrices: three launches a step, bound by the matrix units.  128 x 128 tiles, 4 waves of 64 x 64 each (12 MFMAs for 8 operand reads),
// 32 columns of K at a time by LDS-DMA into two stages, two blocks to a compute unit.
//   PHASE 0: A = X X^T;  1: B = b A + c A A;  2: X <- a X + B X.   MODE 0: whole tiles;  1: job.share[PHASE] shares of K, each leaving an fp32 tile;  2: their sum
constexpr int NS_BIG_TILE = 128 * 64, NS_BIG_STAGE = 4 * NS_BIG_TILE, NS_BIG_LDS = 128 * 129 * 4 > 2 * NS_BIG_STAGE ? 128 * 129 * 4 : 2 * NS_BIG_STAGE;
template <int PHASE, int MODE>
__global__ __launch_bounds__(256, 2) void k_ns_big(NsParams p) {
  extern __shared__ __align__(16) unsigned char lds[];
  const unsigned lds0 = (unsigned)(size_t)(CRAFT_LDS unsigned char*)lds;
  const int block = MODE == 2 ? blockIdx.x : xcd_chunk(blockIdx.x, gridDim.x);
  int q, split = 0;
  const int id = ns_job(p.table, MODE == 1 ? NS_SHARED + PHASE : PHASE < 2 ? NS_LOWER : NS_ALL, block, q);
  const NsJob j = p.table->job[id];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l31 = lane & 31;
  const int splits = MODE == 0 ? 1 : j.share[PHASE];
  if (MODE == 1) { split = q % splits; q /= splits; }
  int ti, tj;
  if constexpr (PHASE < 2) ns_lower(q, ti, tj);
  else { const int tm = j.mp >> 7; tj = q / tm; ti = q - tj * tm; }
  const int K = PHASE == 0 ? j.np : j.mp;
  const _Float16* P = PHASE == 0 ? ns_x(p, j) : ns_a(p, j, PHASE - 1);
  const _Float16* Q = PHASE == 2 ? ns_xt(p, j, p.flip) : P;
  const long pp = PHASE == 0 ? (long)j.mp * j.np : (long)j.mp * j.mp, qp = PHASE == 1 ? pp : (long)j.mp * j.np;
  const int wa = wave >> 1, wb = wave & 1;
  f32x16 acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
  // a partial tile: [wave][a][b][r / 4][lane][4]
  float* part = p.part + ((long)p.table->part[PHASE][id] + (long)q * splits) * 16384 + wave * 4096 + lane * 4;
  if constexpr (MODE < 2) {
    // a stage: [P hi, P lo, Q hi, Q lo][32-row block][16 columns] x 1 KiB; wave w copies the blocks w
    const _Float16* src[4] = {P + ns_at(ti * 128, 0, K), P + pp + ns_at(ti * 128, 0, K), Q + ns_at(tj * 128, 0, K), Q + qp + ns_at(tj * 128, 0, K)};
    const int nk = K >> 5, k0 = nk * split / splits, k1 = nk * (split + 1) / splits;
    const unsigned voff = (unsigned)wave * (unsigned)(K >> 4) * 1024u + (unsigned)lane * 16u;
    auto stage = [&](int buf, int k) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const unsigned long base = (unsigned long)(src[s] + (long)k * 1024);
        u32x4_at d;
        d[0] = __builtin_amdgcn_readfirstlane((unsigned)base);
        d[1] = __builtin_amdgcn_readfirstlane((unsigned)(base >> 32));
        d[2] = 0xffffffffu;
        d[3] = 0x00020000u;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          TileCopy<_Float16, 32, 128, 4>::one(d, voff + u * 1024u, lds0 + (unsigned)(buf * NS_BIG_STAGE + s * NS_BIG_TILE + wave * 2048 + u * 1024));
      }
    };
    if (k0 < k1) stage(0, k0);
    for (int k = k0; k < k1; ++k) {
      const int buf = (k - k0) & 1;
      wait_copies();
      __syncthreads();
      if (k + 1 < k1) stage(buf ^ 1, k + 1);
      const unsigned char* t = lds + buf * NS_BIG_STAGE + lane * 16;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        f16x8 ph[2], pl[2], qh[2], ql[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const unsigned char* r = t + ((2 * wa + a) * 2 + ks) * 1024;
          const unsigned char* c = t + ((2 * wb + a) * 2 + ks) * 1024;
          ph[a] = *reinterpret_cast<const f16x8*>(r);
          pl[a] = *reinterpret_cast<const f16x8*>(r + NS_BIG_TILE);
          qh[a] = *reinterpret_cast<const f16x8*>(c + 2 * NS_BIG_TILE);
          ql[a] = *reinterpret_cast<const f16x8*>(c + 3 * NS_BIG_TILE);
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int b = 0; b < 2; ++b) ns_mma(ph[a], pl[a], qh[b], ql[b], acc[a][b]);
      }
    }
    if constexpr (MODE == 1) {
      part += (long)split * 16384;
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(part + ((a * 2 + b) * 4 + g) * 256) = f32x4{acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
      return;
    }
    __syncthreads();
  } else {
    for (int s = 0; s < splits; ++s)                                     // in their order
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(part + (long)s * 16384 + ((a * 2 + b) * 4 + g) * 256);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[a][b][4 * g + e] += v[e];
          }
  }
  float* t = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) t[(64 * wa + 32 * a + acc_row(r) + 4 * h) * 129 + 64 * wb + 32 * b + l31] = acc[a][b][r] * p.c1;
  __syncthreads();
  if constexpr (PHASE > 0) {                                             // the old value: A's tile, or X's (only this block touches it)
    const _Float16* O = PHASE == 1 ? P : ns_x(p, j);
    const int ld = PHASE == 1 ? K : j.np;
    const long plane = PHASE == 1 ? pp : qp;
    for (int e = tid; e < 2048; e += 256) {
      const int row = e & 127, c = (e >> 7) * 8;
      const _Float16* o = O + ns_at(ti * 128 + row, tj * 128 + c, ld);
      const f16x8 oh = ns_ld(o), ol = ns_ld(o + plane);
#pragma unroll
      for (int i = 0; i < 8; ++i) t[row * 129 + c + i] += p.c0 * ((float)oh[i] + (float)ol[i]);
    }
    __syncthreads();
  }
  if (PHASE == 2 && p.last) ns_result<128>(p, j, t, ti, tj, tid, 256);
  else if constexpr (PHASE == 2) ns_planes<128>(t, ns_x(p, j), j.np, qp, ns_xt(p, j, p.flip ^ 1), j.mp, ti, tj, tid, 256);
  else {
    _Float16* out = ns_a(p, j, PHASE);
    ns_planes<128>(t, out, j.mp, (long)j.mp * j.mp, ti == tj ? nullptr : out, j.mp, ti, tj, tid, 256);
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

namespace craft {
// one set of launches: matrices that are all small or all large
static int ns_run(NsLoad& l, NsParams& p, const float* coeffs, int steps, float s_a, float s_b, hipStream_t s) {
  auto count = [&](int kind) {
    long c = 0;
    for (int i = 0; i < l.n; ++i) c += ns_blocks(l.job[i], kind, l.side);
    return c;
  };
  if (l.big) {
    // shares of K for tiles too few to fill the card: as many blocks as it holds at once (two to a compute unit), at least 256 columns of K each
    const long tiles[3] = {count(NS_LOWER), count(NS_LOWER), count(NS_ALL)};
    for (int i = 0; i < l.n; ++i)
      for (int ph = 0; ph < 3; ++ph) {
        const long most = (ph == 0 ? l.job[i].np : l.job[i].mp) / 256, want = 512 / tiles[ph];
        const long v = want < most ? want : most;
        l.job[i].share[ph] = (short)(v < 1 ? 1 : v);
      }
  }
  for (int kind = 0; kind < NS_KINDS; ++kind)
    if (count(kind) > 0x7ffffffeL) return CRAFT_ERR_UNSUPPORTED;
  auto go = [&](auto tag, int kind, int threads, int lds) {
    constexpr auto kernel = decltype(tag)::value;
    if (lds > 0) if (const int rc = allow_lds<kernel>(lds)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)count(kind)), dim3(threads), lds, s, p);
    return (int)hipGetLastError();
  };
#define NS_TRY(x) do { const int rc_ = (x); if (rc_) return rc_; } while (0)
  hipLaunchKernelGGL(k_ns_table, dim3(1), dim3(64), 0, s, l);
  HIP_CHECK_RET(hipGetLastError());
  NS_TRY(go(KernelTag<k_ns_norm>(), NS_NORM, 1024, 0));
  NS_TRY(go(KernelTag<k_ns_init>(), NS_INIT, 256, 0));
  // a product of the larger ones: whole tiles, or shares of K and their sum
  auto product = [&](auto whole, auto shared, auto sum, int ph) {
    const int kind = ph < 2 ? NS_LOWER : NS_ALL;
    if (count(NS_SHARED + ph) == count(kind)) return go(whole, kind, 256, NS_BIG_LDS);
    const int rc = go(shared, NS_SHARED + ph, 256, NS_BIG_LDS);
    return rc ? rc : go(sum, kind, 256, NS_BIG_LDS);
  };
  for (int t = 0; t < steps; ++t) {
    const float a = coeffs[3 * t], b = coeffs[3 * t + 1], c = coeffs[3 * t + 2];
    p.flip = t & 1;
    p.last = t == steps - 1;
    const float gram = s_a / (p.s_x * p.s_x), b0 = b * s_b / s_a, b1 = c * s_b / (s_a * s_a);
    const float x0 = p.last ? a / p.s_x : a, x1 = (p.last ? 1.f / p.s_x : 1.f) / s_b;      // B X carries s_b s_x; the last one leaves without a scale
    if (!l.big) {
      p.c1 = gram;
      NS_TRY(go(KernelTag<k_ns_gram<0>>(), NS_LOWER, 512, 8 * 4096 * 4));
      p.c0 = b0; p.c1 = b1;
      NS_TRY(go(KernelTag<k_ns_gram<1>>(), NS_LOWER, 512, 8 * 4096 * 4));
      p.c0 = x0; p.c1 = x1;
      NS_TRY(go(KernelTag<k_ns_update>(), NS_ALL, 256, 0));
      continue;
    }
    p.c0 = 0.f; p.c1 = gram;
    NS_TRY(product(KernelTag<k_ns_big<0, 0>>(), KernelTag<k_ns_big<0, 1>>(), KernelTag<k_ns_big<0, 2>>(), 0));
    p.c0 = b0; p.c1 = b1;
    NS_TRY(product(KernelTag<k_ns_big<1, 0>>(), KernelTag<k_ns_big<1, 1>>(), KernelTag<k_ns_big<1, 2>>(), 1));
    p.c0 = x0; p.c1 = x1;
    NS_TRY(product(KernelTag<k_ns_big<2, 0>>(), KernelTag<k_ns_big<2, 1>>(), KernelTag<k_ns_big<2, 2>>(), 2));
  }
#undef NS_TRY
  return 0;
}
}  // namespace craft

extern "C" int craft_orthogonalize(const long* jobs, int n, const float* coeffs, int steps, float eps, float s_x, float s_a, float s_b, int dtype, void* ws,
                                   long ws_bytes, void* stream) {
  if (!jobs || !coeffs || n <= 0 || steps < 1 || steps > 64 || dtype < 0 || dtype > 2) return CRAFT_ERR_ARG;
  if (!(eps >= 0.f) || !(s_x > 0.f) || !(s_a > 0.f) || !(s_b > 0.f) || (reinterpret_cast<uintptr_t>(ws) & 255) || !ws) return CRAFT_ERR_ARG;
  const bool big = (jobs[4] < jobs[5] ? jobs[4] : jobs[5]) > NS_SMALL;
  if (n > (big ? NS_MAX_BIG : NS_MAX_JOBS)) return CRAFT_ERR_ARG;
  NsLoad l = {};
  NsParams p = {};
  l.n = n; l.big = big; l.side = big ? 128 : 64;
  l.table = reinterpret_cast<NsTable*>(ws);
  p.table = l.table; p.dtype = dtype; p.eps = eps; p.s_x = s_x;
  p.ws = reinterpret_cast<unsigned char*>(ws);
  p.norm = reinterpret_cast<double*>(p.ws + NS_TABLE_BYTES);
  long at = NS_TABLE_BYTES + (long)n * NS_NORM_BLOCKS * 8;
  const int pad = l.side;
  for (int i = 0; i < n; ++i) {
    const long* d = jobs + 6 * i;                                        // src, ld_src, dst, ld_dst, rows, cols
    NsJob& j = l.job[i];
    if (!d[0] || !d[2] || d[4] <= 0 || d[5] <= 0 || d[1] < 0 || d[3] < d[5]) return CRAFT_ERR_ARG;
    const long m = d[4] < d[5] ? d[4] : d[5], nn = d[4] < d[5] ? d[5] : d[4];
    if (m > 32768 || nn > 1l << 22) return CRAFT_ERR_UNSUPPORTED;
    if ((m > NS_SMALL) != big) return CRAFT_ERR_ARG;
    j.src = reinterpret_cast<const void*>(d[0]); j.ld_src = d[1]; j.dst = reinterpret_cast<void*>(d[2]); j.ld_dst = d[3];
    j.rows = (int)d[4]; j.cols = (int)d[5];
    j.mp = (int)((m + pad - 1) / pad * pad); j.np = (int)((nn + pad - 1) / pad * pad);
    j.ws = at;
    at += ns_bytes(j.mp, j.np);
    const long el = m * nn;
    j.nb = (short)(el / 8192 < 1 ? 1 : el / 8192 > NS_NORM_BLOCKS ? NS_NORM_BLOCKS : el / 8192);
    j.share[0] = j.share[1] = j.share[2] = 1;
  }
  if (at + (big ? NS_PART_BYTES : 0) > ws_bytes) return CRAFT_ERR_ARG;
  p.part = reinterpret_cast<float*>(p.ws + at);
  return ns_run(l, p, coeffs, steps, s_a, s_b, reinterpret_cast<hipStream_t>(stream));
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
