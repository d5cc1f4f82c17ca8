// Shared pieces of the masked / capped / biased attention kernels (kernels_attention_*.hip):
//
//   z[i][j] = cap(scale * q_i . k_j) - slope_h * |pos_i - j|,   cap(x) = c tanh(x / c) or x,   pos_i = i + Nk - Nq
//   p = softmax of z over the keys a query sees,   o_i = sum_j p_ij v_j
//
// Every kernel computes its scores as 32 x 32 MFMA blocks whose A operand comes out of LDS (rows = the tokens that a block walks over) and whose
// B operand lies in registers (columns = the 32 tokens that a wave owns: lane & 31).  A lane then holds 16 scores of ONE of its own tokens, in
// accumulator order -- row 8 (r >> 2) + 4 (lane >> 5) + (r & 3) of the block in register r -- which is, with no exchange between lanes, the B operand
// of the next product over those rows: the order of a contraction is free as long as both operands use the same one, so the transposing reads of
// the A operand simply fetch their rows in accumulator order.  Probabilities and score gradients never leave their lane's registers.
//
// LDS tiles are [row][DP] in the tensors' own type, 16-byte chunks swizzled within a row (tile_swz) so that both the row reads (ds_read_b128) and
// the transposing reads (ds_read_b64_tr_b16) of a tile are free of bank conflicts.  They are filled by LDS-DMA: the copy writes LDS linearly, so the
// swizzle is applied to the global addresses of the lanes.
#pragma once
#include <atomic>
#include <type_traits>
#include "launch.hpp"

namespace craft {

// Dynamic LDS above 64 KB has to be allowed once per kernel and device (hipFuncSetAttribute takes as long as a launch).  The flags only remember that it
// was done: any thread may set them again.
template <auto Kernel>
inline int allow_lds(int bytes) {
  static std::atomic<unsigned> done{0};
  int dev = 0;
  if (const hipError_t e = hipGetDevice(&dev)) return (int)e;
  if (dev < 32 && (done.load(std::memory_order_relaxed) >> dev & 1)) return 0;
  if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) return (int)e;
  if (dev < 32) done.fetch_or(1u << dev, std::memory_order_relaxed);
  return 0;
}

template <auto Kernel> struct KernelTag { static constexpr auto value = Kernel; };

#define CRAFT_LDS __attribute__((address_space(3)))
typedef __fp16 at_fp16x4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __bf16 at_bf16x4 __attribute__((__vector_size__(4 * sizeof(__bf16))));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4_at __attribute__((ext_vector_type(4)));

struct AttentionParams {
  const void *q, *k, *v, *o, *go;              // o, go (gradient of o): backward only
  void *out, *dq, *dk, *dv;
  long q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h, o_b, o_n, o_h, go_b, go_n, go_h;   // strides in elements; the last axis is contiguous
  int B, Nq, Nk, H, Hk, D;
  float c2;                                    // scale * log2(e): scores are kept as powers of two
  float ca, cap2;                              // capped: 2 scale / cap * log2(e) and cap * log2(e)
  float scale, cap;
  const float* slopes;                         // [H], natural units
  const int *prefix, *docq, *dock;             // [B], [B][Nq], [B][Nk]; each may be null
  const int4 *rq, *rk;                         // per 32 tokens: {least document, greatest document, any negative one, 0}
  int causal;
  float* lse;                                  // [B][H][Nq] log2 of the sum of 2^z; +inf for a query that sees nothing (so that 2^(z - lse) = 0).  fp32 tensors:
                                               // [B][H][Nq][2], with what its rounding left (a log-sum of 20 is rounded by 1e-6, the whole row's gradients with it)
  void* rest; const void* o_rest;              // 16-bit: what o's rounding left, like o contiguous [B][Nq][H][D]: delta is a difference of sums that the
                                               // rounding of o would disturb as much as the gradients' own (written with lse, read for delta; may be null)
  const float* delta;                          // [B][H][Nq] -sum_d go * o
  float *part_o, *part_ml;                     // token kernel: partial results of the splits
  int splits;
  float *part_k, *part_v;                      // backward: per query head partial key / value gradients (null: written directly)
  float2* top;                                 // backward, fp16: [B * Hk][slices] the largest |go_i|^2 and |v_j|^2 (see score_exponent)
  int slices;
};

// fp16's second products.  An operand in fp16 keeps its bits between 2^-14 and 2^16 only: the probabilities of a long row, and the gradients of scores
// where the loss' own are small, would lose them or vanish; large gradients of scores would overflow though dq and dk fit.  Both are carried times a
// power of two, which the fp32 results lose again: 2^15 for probabilities (at most 1), 2^E for gradients of scores, which are at most
// |go_i| (|v_j| + |o_i|) <= 2 max|go| max|v| < 2^(15 - E).  The gradient of q has its own query's |go_i| and so its own E; those of k and v have one for a
// key head (its query heads share the sums).  Norms that are not finite do not count: their rows give inf or NaN at any scale.
// (|go| = 1e-4, 2048 tokens: dk was off by 2.7e-3 without, where rounding the result costs 3e-4.)
__device__ __forceinline__ int score_exponent(float go2, float v2) {
  const float b = 2.f * sqrtf(go2) * sqrtf(v2);
  return 15 - __builtin_amdgcn_frexp_expf(b < INFINITY ? b : 1.f);
}
// largest of the slices, by a wave; four loads on their way at a time
__device__ __forceinline__ float2 largest_rows(const AttentionParams& p, int bk, int lane) {
  const float2* top = p.top + (long)bk * p.slices;
  float2 m = make_float2(0.f, 0.f);
  for (int i = lane; i - lane < p.slices; i += 256) {
    float2 t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) t[u] = top[min(i + 64 * u, p.slices - 1)];
#pragma unroll
    for (int u = 0; u < 4; ++u) { m.x = fmaxf(m.x, t[u].x); m.y = fmaxf(m.y, t[u].y); }
  }
  return make_float2(wave_max(m.x), wave_max(m.y));
}

template <typename T> struct AtFrag { typedef f32x8 type; };
template <> struct AtFrag<_Float16> { typedef f16x8 type; };
template <> struct AtFrag<__bf16> { typedef bf16x8 type; };

// D (16 rows of contraction) += A B.  fp32: eight exact 32x32x2 products; instruction j contracts element j of both lane halves.
__device__ __forceinline__ void at_mma(const f16x8& a, const f16x8& b, f32x16& c) { c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ void at_mma(const bf16x8& a, const bf16x8& b, f32x16& c) { c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ void at_mma(const f32x8& a, const f32x8& b, f32x16& c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
}

// Chunk c (16 bytes) of row r lies at slot c ^ tile_swz(r).  CPR = chunks per row.  16 consecutive rows must reach 16 different slots of the 256-byte
// bank row (ds_read_b128), and the 64-byte segments that a transposing read takes from 4 consecutive rows must be 4 different quarters of it.
template <int CPR>
__device__ __forceinline__ int tile_swz(int r) {
  if constexpr (CPR >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (CPR == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  else return (r >> 2) & 3;
}
template <typename T, int DP> constexpr int at_cpr() { return DP * (int)sizeof(T) / 16; }

// LDS addresses.  The swizzle is an exclusive or of a chunk's number, so a lane's addresses within a tile (whose base is a multiple of its row, 512 bytes at
// most) differ from one of them by an exclusive or with a constant and an offset that the instruction adds: one register for the row reads of a tile and
// one for its transposing reads, in place of one for each column step (the gradients' kernels spilled for them).
template <typename T, int DP> constexpr int at_rowb() { return DP * (int)sizeof(T); }
// of lane's row lane & 31, columns 8 h ..
template <typename T, int DP>
__device__ __forceinline__ unsigned row_addr(unsigned tile, int lane) {
  const int row = lane & 31, h = lane >> 5, f = tile_swz<at_cpr<T, DP>()>(row);
  return tile + (unsigned)(row * at_rowb<T, DP>() + (((sizeof(T) == 2 ? h : 2 * h) ^ f) << 4));
}
// row read: columns 16 ks + 8 h .. + 7 of row 32 blk + (lane & 31); `more`: in the tile that many bytes on (one exclusive or for both)
template <typename T, int DP>
__device__ __forceinline__ typename AtFrag<T>::type row_read(unsigned addr, int blk, int ks, int more = 0) {
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<CRAFT_LDS typename AtFrag<T>::type*>((addr ^ (unsigned)(ks << 5)) + (unsigned)(blk * 32 * at_rowb<T, DP>() + more));
  } else {
    const f32x4 a = *reinterpret_cast<CRAFT_LDS f32x4*>((addr ^ (unsigned)(ks << 6)) + (unsigned)(blk * 32 * at_rowb<T, DP>() + more));
    const f32x4 b = *reinterpret_cast<CRAFT_LDS f32x4*>((addr ^ (unsigned)(ks << 6) ^ 16u) + (unsigned)(blk * 32 * at_rowb<T, DP>() + more));
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    return v;
  }
}
// of lane's part of the transposing reads
template <typename T, int DP>
__device__ __forceinline__ unsigned col_addr(unsigned tile, int lane) {
  const int h = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    const int j = lane & 15, mh = (lane >> 4) & 1, row = 4 * h + (j >> 2), c = 2 * mh + ((j & 3) >> 1);
    return tile + (unsigned)(row * at_rowb<T, DP>() + ((c ^ tile_swz<at_cpr<T, DP>()>(row)) << 4) + ((j & 1) << 3));
  } else {
    const int col = lane & 31, row = 4 * h;
    return tile + (unsigned)(row * at_rowb<T, DP>() + (((col >> 2) ^ tile_swz<at_cpr<T, DP>()>(row)) << 4) + ((col & 3) << 2));
  }
}
// transposing read: column 32 db + (lane & 31) of rows row0 + 4 h + {0..3} and row0 + 8 + 4 h + {0..3} (accumulator order), row0 a multiple of 16
template <typename T, int DP>
__device__ __forceinline__ typename AtFrag<T>::type col_read(unsigned addr, int row0, int db, int more = 0) {
  constexpr int ROWB = at_rowb<T, DP>();
  typename AtFrag<T>::type v;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {                       // 8 rows on: the swizzle's bit 1
      const unsigned at = (addr ^ (unsigned)((db << 6) | (u << 5))) + (unsigned)((row0 + 8 * u) * ROWB + more);
      if constexpr (std::is_same<T, __bf16>::value) {
        const at_bf16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((CRAFT_LDS at_bf16x4*)at);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * u + i] = x[i];
      } else {
        const at_fp16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4f16((CRAFT_LDS at_fp16x4*)at);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * u + i] = (_Float16)x[i];
      }
    }
  } else {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = at_cpr<T, DP>() >= 16 ? (i << 2) : ((i >> 1) & 1) << 2;          // tile_swz of row 8 u + 4 h + i, less that of 4 h
        const unsigned at = (addr ^ (unsigned)((db << 7) ^ (f << 4) ^ (u << 5))) + (unsigned)((row0 + 8 * u + i) * ROWB + more);
        v[4 * u + i] = *reinterpret_cast<CRAFT_LDS float*>(at);
      }
  }
  return v;
}

// 8 accumulator values (registers 8 s .. 8 s + 7) as a B operand.  16-bit types: the probabilities (at most 2^8 before normalisation) and score
// gradients are rounded to the tensors' type here, once, to nearest; their sums are taken in fp32 before the rounding.  That is one product in place of two
// or three (a value in two 16-bit planes), and it is what makes the results err more than fp32 products rounded once at the end: outputs 2.8e-4 against 2.1e-4
// (fp16) and 2.0e-3 against 1.7e-3 (bf16), dq and dk 3.5e-4 against 2.1e-4 and 2.6e-3 against 1.7e-3.
template <typename T>
__device__ __forceinline__ typename AtFrag<T>::type at_pack(const f32x16& x, int s) {
  typename AtFrag<T>::type v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (T)x[8 * s + j];
  return v;
}
// times a power of two (fp16: the product and its conversion are one instruction)
template <typename T>
__device__ __forceinline__ typename AtFrag<T>::type at_pack(const f32x16& x, int s, float f) {
  if constexpr (!std::is_same<T, _Float16>::value) return at_pack<T>(x, s);
  typename AtFrag<T>::type v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (T)(x[8 * s + j] * f);
  return v;
}

template <typename T> constexpr int at_lw() { return sizeof(T) == 4 ? 2 : 1; }       // words of a log-sum

// the row of a 32-row block that register r of a lane holds, less 4 h
__device__ __forceinline__ constexpr int acc_row(int r) { return 8 * (r >> 2) + (r & 3); }

// a value and its partner's in the other half of the wave
__device__ __forceinline__ float at_other_half(float x) { return __shfl_xor(x, 32); }

// B operand in registers: row `row` of a [.., D] matrix, columns 16 ks + 8 h .. (zero behind D; D is a multiple of 8)
template <typename T, int DP>
__device__ __forceinline__ void load_own(const T* row, int D, int h, typename AtFrag<T>::type (&f)[DP / 16]) {
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int c = 16 * ks + 8 * h;
    typename AtFrag<T>::type v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (T)0.f;
    if (c < D) v = *reinterpret_cast<const typename AtFrag<T>::type*>(row + c);
    f[ks] = v;
  }
}

// Loads into registers have arrived behind this.  The compiler waits for a load where its value is first used; inside a loop that copies by LDS-DMA
// (which it does not know of, and which its counter counts) such a wait would be for the copies just started as well.
template <typename F, int N>
__device__ __forceinline__ void arrived(F (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// LDS-DMA of ROWS rows (those from `valid` on repeat the last valid one; the chunks behind D repeat the last real one: both are only ever
// multiplied by zeros or masked) by WAVES waves; this wave's share.  Issues only: wait for vmcnt and pass a barrier before reading.
template <typename T, int DP, int ROWS, int WAVES>
struct TileCopy {
  static constexpr int CPR = at_cpr<T, DP>(), CHUNKS = ROWS * CPR, PER = CHUNKS / 64 / WAVES;
  static_assert(CHUNKS % (64 * WAVES) == 0, "whole wave instructions");
  unsigned voff[PER];
  __device__ __forceinline__ static unsigned offset(int wave, int lane, int i, unsigned stride, int nchunk, int valid) {
    const int L = (wave * PER + i) * 64 + lane, row = L / CPR, pos = L % CPR;
    const int c = min(pos ^ tile_swz<CPR>(row), nchunk - 1);
    return (unsigned)min(row, valid - 1) * stride + ((unsigned)c << 4);
  }
  __device__ __forceinline__ void init(int wave, int lane, unsigned stride, int nchunk) {
#pragma unroll
    for (int i = 0; i < PER; ++i) voff[i] = offset(wave, lane, i, stride, nchunk, ROWS);
  }
  // base: row 0 of the tile (wave-uniform); stride: bytes between rows; lds: byte address of the tile in LDS
  __device__ __forceinline__ void issue(const unsigned char* base, unsigned stride, int nchunk, int valid, unsigned lds, int wave, int lane) const {
    const unsigned long a = (unsigned long)base;
    u32x4_at d;
    d[0] = __builtin_amdgcn_readfirstlane((unsigned)a);
    d[1] = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
    d[2] = 0xffffffffu;
    d[3] = 0x00020000u;
    if (valid >= ROWS) {
#pragma unroll
      for (int i = 0; i < PER; ++i) one(d, voff[i], lds + (unsigned)(wave * PER + i) * 1024u);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) one(d, offset(wave, lane, i, stride, nchunk, valid), lds + (unsigned)(wave * PER + i) * 1024u);
    }
  }
  __device__ __forceinline__ static void one(const u32x4_at& d, unsigned v, unsigned lds) {
    const unsigned dst = __builtin_amdgcn_readfirstlane(lds);
    // (m0 holds the LDS address; a copy may follow its setting after one wait state)
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds" ::"v"(v), "s"(dst), "s"(d) : "memory", "m0");
  }
};
// 64 words base[min(first + lane, last)] -> LDS, by one wave
__device__ __forceinline__ void copy_words(const void* base, long first, long last, unsigned lds, int lane) {
  const unsigned long a = (unsigned long)base + 4ul * (unsigned long)first;
  u32x4_at d;
  d[0] = __builtin_amdgcn_readfirstlane((unsigned)a);
  d[1] = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
  d[2] = 0xffffffffu;
  d[3] = 0x00020000u;
  const unsigned v = 4u * (unsigned)min(lane, (int)min(last - first, 63l));
  const unsigned dst = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dword %0, %2, 0 offen lds" ::"v"(v), "s"(dst), "s"(d) : "memory", "m0");
}
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// zero the rows of a tile whose document is negative: what lies there may be anything, and 0 * inf is not 0.  All threads; barrier behind it.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void zero_rows(unsigned char* t, const int* docs, int valid, int tid, int nthread) {
  constexpr int CPR = at_cpr<T, DP>();
  for (int c = tid; c < ROWS * CPR; c += nthread) {
    const int row = c / CPR;
    if (docs[min(row, valid - 1)] < 0) *reinterpret_cast<f32x4*>(t + c * 16) = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// a document range over 32-token groups [g0, g1] joined (wave-uniform)
__device__ __forceinline__ int4 join_ranges(const int4* r, int g0, int g1) {
  int4 a = r[g0];
  for (int g = g0 + 1; g <= g1; ++g) {
    const int4 b = r[g];
    a.x = min(a.x, b.x); a.y = max(a.y, b.y); a.z |= b.z;
  }
  return a;
}
// the same as scalars: a range read inside the walk is read before the next tile's copies are started
__device__ __forceinline__ int4 uniform_range(const int4& a) {
  return make_int4(__builtin_amdgcn_readfirstlane(a.x), __builtin_amdgcn_readfirstlane(a.y), __builtin_amdgcn_readfirstlane(a.z), 0);
}
__device__ __forceinline__ bool ranges_meet(const int4& a, const int4& b) { return a.x <= b.y && b.x <= a.y; }
__device__ __forceinline__ bool one_document(const int4& a, const int4& b) { return !a.z && !b.z && a.x == a.y && b.x == b.y && a.x == b.x; }

// A score is at_mul * at_raw(q . k) (+ the bias), as a power of two and up to a constant of the whole row, which the softmax drops (the kept log-sums drop
// it too): the product itself; capped, with tanh(u) = 1 - 2 r, r = 1 / (1 + e^2u): -r.  fp32 tensors take the library's tanh (r is off by 2^-23 of 1).
template <typename T, bool CAP>
__device__ __forceinline__ float at_raw(const AttentionParams& p, float s) {
  if constexpr (!CAP) return s;
  else if constexpr (std::is_same<T, float>::value) return tanhf(s * p.scale / p.cap);
  else return -__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * p.ca) + 1.f);                // (exp2 = inf: 0;  exp2 = 0: -1)
}
// at_raw with a cap of 16 scores, step by step
template <typename T>
__device__ __forceinline__ void at_raws(const AttentionParams& p, f32x16& x) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = at_raw<T, true>(p, x[r]);
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= p.ca;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(x[r]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] += 1.f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = -__builtin_amdgcn_rcpf(x[r]);
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <typename T, bool CAP>
__device__ __forceinline__ float at_mul(const AttentionParams& p) { return !CAP ? p.c2 : std::is_same<T, float>::value ? p.cap2 : 2.f * p.cap2; }
// 1 - tanh^2 from at_raw
template <typename T>
__device__ __forceinline__ float at_slope(float x) {
  const float th = std::is_same<T, float>::value ? x : fmaf(2.f, x, 1.f);
  return fmaf(-th, th, 1.f);
}

// Which (head of the batch, tile) a block takes.  The blocks of a head share an XCD, whose L2 then holds that head's keys; and the tiles of all the heads
// of an XCD come with the heaviest first (tile 0 is the heaviest): under a causal mask the last blocks to start are the shortest, and no compute unit is
// left with a long one at the end.  Heads that do not divide by the 8 XCDs: head by head, in contiguous eighths of the list.
__device__ __forceinline__ void block_of(int heads, int tiles, int& head, int& tile) {
  const int total = heads * tiles, id = blockIdx.x;
  if ((heads & 7) == 0) {
    const int per = heads >> 3, slot = id >> 3;
    tile = slot / per;
    head = (id & 7) * per + slot - tile * per;
  } else {
    const int at = xcd_chunk(id, total);
    head = at / tiles;
    tile = at - head * tiles;
  }
}

// token range of a walk: the first and the last tile of [t0, t1) whose documents meet `own`, over the whole block
template <int THREADS>
__device__ __forceinline__ void tiles_of_documents(const int4* r, int groups, int gpt, const int4& own, int& t0, int& t1, int tid, int* red) {
  int lo = 0x7fffffff, hi = -1;
  for (int t = t0 + tid; t < t1; t += THREADS) {
    const int4 a = join_ranges(r, t * gpt, min(t * gpt + gpt, groups) - 1);
    if (ranges_meet(a, own)) { lo = min(lo, t); hi = max(hi, t); }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { lo = min(lo, __shfl_xor(lo, o)); hi = max(hi, __shfl_xor(hi, o)); }
  if ((tid & 63) == 0) { red[2 * (tid >> 6)] = lo; red[2 * (tid >> 6) + 1] = hi; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) { lo = min(lo, red[2 * w]); hi = max(hi, red[2 * w + 1]); }
  t0 = __builtin_amdgcn_readfirstlane(lo);
  t1 = __builtin_amdgcn_readfirstlane(hi) + 1;
  if (t1 <= 0) t0 = t1 = 0;
}

// the launchers of each (type, padded width); `what` 0 forward, 1 single tokens, 2 gradient of q, 3 gradients of k and v
template <typename T, int DP> int attention_fwd_launch(const AttentionParams& p, hipStream_t s);
template <typename T, int DP> int attention_token_launch(const AttentionParams& p, hipStream_t s);
template <typename T, int DP> int attention_bwd_launch(const AttentionParams& p, hipStream_t s);

}  // namespace craft
