// What the attention kernels share: arguments, element types, LDS tiles of rows, fragments and the second product's reads.
// The layouts are described at the top of sdpa.hip.
#pragma once
#include <cfloat>
#include <climits>
#include "lds_dma.h"

namespace attn {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;
typedef unsigned long long u64;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int WAVES = 4, ROWS = 32 * WAVES;  // rows (queries or keys) that a workgroup owns: 32 per wave

struct Strides { long long b, s, h; };       // elements

struct AttnArgs {
  const void *q, *k, *v, *o, *dout;
  Strides sq, sk, sv, sdo;
  void *out, *dq, *dk, *dv;                  // dense (B, S, heads, D)
  const void* low;                           // bf16, backward: what rounding left of o (NULL: not kept)
  void* out_low;                             // forward: where to keep it
  float *lse2, *nlse, *ndelta;               // (B, H, Sq); nlse: what the backward pass adds to log2(e) s; ndelta: -sum_d do o
  const u64* words;                          // (B, nw) mask bits, 64 keys a word; NULL: every key is visible
  float* part;                               // partial results of splits
  float* part_lse;
  int B, H, Hkv, Sq, Sk, D, nw;
  int G;                                     // few rows: query heads of a group packed into them
  int nsplit, tiles_per_split;
  int nrow;                                  // row blocks
  float scale;
  int causal;
};

// ---- element types -----------------------------------------------------------------------------------------------
template <typename T> struct El;
template <> struct El<u16> {
  static constexpr int BK = 64;              // rows of an LDS tile
  typedef u32x4 Vec4;                        // 16 bytes of a row
  static constexpr int CK = 16;              // elements of a row that one pair of 16-byte fragments covers
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct El<float> {
  static constexpr int BK = 32;
  typedef f32x4 Vec4;
  static constexpr int CK = 8;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack2(float a, float b) {      // one instruction: v_cvt_pk_bf16_f32
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// Four results as they are stored, to `at`, and (bf16, low not NULL) what their rounding left, to `low`: with it the backward
// pass forms delta from 16 bits of each result, not 8.  Where a result is infinite nothing is left.
template <typename T>
__device__ __forceinline__ void put4(T* at, u16* low, const float* x) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4*>(at) = f32x4{x[0], x[1], x[2], x[3]};
  } else {
    const u32x2 w = {pack2(x[0], x[1]), pack2(x[2], x[3])};
    *reinterpret_cast<u32x2*>(at) = w;
    if (low) {
      float rest[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        rest[j] = x[j] - __builtin_bit_cast(float, j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
        rest[j] = fabsf(rest[j]) <= FLT_MAX ? rest[j] : 0.f;
      }
      *reinterpret_cast<u32x2*>(low) = u32x2{pack2(rest[0], rest[1]), pack2(rest[2], rest[3])};
    }
  }
}

// ---- LDS tile of `El<T>::BK` rows ----------------------------------------------------------------------------------
template <typename T, int DP>
struct Tile {
  static constexpr int BK = El<T>::BK;
  static constexpr int RB = DP * (int)sizeof(T);       // bytes of a row
  static constexpr int PPR = RB / 16;                  // pieces of a row
  static constexpr int BYTES = BK * RB;
  static constexpr int NDMA = BYTES / (1024 * WAVES);  // loads per wave
  static_assert(NDMA * 1024 * WAVES == BYTES, "a tile is whole loads of every wave");

  static __device__ __forceinline__ int swizzle(int r) {
    return PPR == 4 ? (r >> 2) & 3 : PPR == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
  }
  // What a lane of one of `waves` waves loads of any tile of a tensor whose rows of D elements lie `stride` bytes apart.
  template <int N>
  struct Source {
    unsigned off[N];
    __device__ __forceinline__ Source(int waves, int wave, int lane, unsigned stride, int D) {
      const int pieces = D * (int)sizeof(T) / 16;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int slot = (j * waves + wave) * 64 + lane, r = slot / PPR, p = (slot % PPR) ^ swizzle(r);
        off[j] = p < pieces ? (unsigned)r * stride + 16u * p : DMA_OUTSIDE;
      }
    }
    // The rows of the tile at `base` whose bit of `rows` is set (all: every bit); the others arrive as zeros.
    __device__ __forceinline__ void load(char* dst, int waves, int wave, int lane, const void* base, u64 rows, u64 all) const {
      const u32x4 rs = dma_rsrc(base);
      if (rows == all) {
#pragma unroll
        for (int j = 0; j < N; ++j) dma16(rs, dst + (j * waves + wave) * 1024, off[j]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int r = ((j * waves + wave) * 64 + lane) / PPR;
          dma16(rs, dst + (j * waves + wave) * 1024, (rows >> r) & 1 ? off[j] : DMA_OUTSIDE);
        }
      }
    }
  };
  typedef Source<NDMA> Shared;             // a tile that the four waves of a workgroup load together
  static constexpr u64 ALL = BK == 64 ? ~0ull : (1ull << (BK & 63)) - 1;
  // Fragment c of row r0 + lane % 32: the lane's 16 bytes of the row's c-th 32 bytes.
  static __device__ __forceinline__ u32x4 frag(const char* t, int r0, int c, int lane) {
    const int r = lane & 31;
    return *reinterpret_cast<const u32x4*>(t + (r0 + r) * RB + (((2 * c + (lane >> 5)) ^ swizzle(r)) << 4));
  }
};

// acc (columns of the tile x lanes) += tile^T [d][row] * x[row][lane], rows r0 .. r0 + 31 of the tile, x as a result
// tile of mma() (sixteen rows a lane).
template <typename T, int DP>
struct Second;
template <int DP>
struct Second<u16, DP> {
  typedef Tile<u16, DP> TL;
  static __device__ __forceinline__ void run(f32x16 (&acc)[DP / 32], const char* t, int r0, const f32x16& x, int lane) {
    const int h = lane >> 5, sub = (lane >> 4) & 1, i = lane & 15;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      u32x4 b;
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = pack2(x[8 * c + 2 * j], x[8 * c + 2 * j + 1]);
      const int r = 4 * h + (i >> 2);                       // and r + 8; of the chunk's 16 rows
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const int p = 4 * dt + 2 * sub + ((i & 3) >> 1);
        const char* a0 = t + (r0 + 16 * c + r) * TL::RB + ((p ^ TL::swizzle(r)) << 4) + (i & 1) * 8;
        const char* a1 = t + (r0 + 16 * c + r + 8) * TL::RB + ((p ^ TL::swizzle(r + 8)) << 4) + (i & 1) * 8;
        union { struct { s16x4 lo, hi; } h; u32x4 f; } u;
        u.h.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(a0));
        u.h.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(a1));
        acc[dt] = El<u16>::mma(u.f, b, acc[dt]);
      }
    }
  }
};
template <int DP>
struct Second<float, DP> {
  typedef Tile<float, DP> TL;
  static __device__ __forceinline__ void run(f32x16 (&acc)[DP / 32], const char* t, int r0, const f32x16& x, int lane) {
    const int h = lane >> 5;
#pragma unroll
    for (int g = 0; g < 16; ++g) {
      const int r = 8 * (g >> 2) + 4 * h + (g & 3);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const int d = 32 * dt + (lane & 31);
        const float a = *reinterpret_cast<const float*>(t + (r0 + r) * TL::RB + (((d >> 2) ^ TL::swizzle(r)) << 4) + (d & 3) * 4);
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x[g], acc[dt], 0, 0, 0);
      }
    }
  }
};

// The 32 rows of a wave as fragments in registers: row p of this lane, zeros where it is not `in`.
template <typename T, int DP>
__device__ __forceinline__ void load_rows(u32x4 (&f)[DP / El<T>::CK], const T* p, int D, bool in, int lane) {
  constexpr int HALF = El<T>::CK / 2;
#pragma unroll
  for (int c = 0; c < DP / El<T>::CK; ++c) {
    const int e = c * El<T>::CK + (lane >> 5) * HALF;
    f[c] = (in && e < D) ? *reinterpret_cast<const u32x4*>(p + e) : u32x4{0, 0, 0, 0};
  }
#pragma unroll
  for (int c = 0; c < DP / El<T>::CK; ++c) settle(f[c]);
}

// Store a lane's row of an accumulator set: columns 32 dt + 8 g + 4 h + 0..3.
template <typename T, int DP>
__device__ __forceinline__ void store_rows(T* row, const f32x16 (&acc)[DP / 32], float mul, int D, int lane, u16* low = nullptr) {
  const int h = lane >> 5;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * h;
      if (d >= D) continue;
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = acc[dt][4 * g + j] * mul;
      put4<T>(row + d, low ? low + d : nullptr, w);
    }
}

// The same for 32 rows `pitch` elements apart, of which the first n exist, through 32 rows of LDS that only this wave uses:
// a row leaves in whole lines, where store_rows writes 8 or 16 bytes of each of 32 rows at a time.
template <typename T, int DP>
__device__ __forceinline__ void store_tile(char* lds, T* rows, long long pitch, int n, const f32x16 (&acc)[DP / 32], float mul, int D,
                                           int lane) {
  typedef Tile<T, DP> TL;
  constexpr int E = 16 / (int)sizeof(T);
  const int h = lane >> 5, row = lane & 31;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = acc[dt][4 * g + j] * mul;
      const int d = 32 * dt + 8 * g + 4 * h;
      char* to = lds + row * TL::RB + (((d / E) ^ TL::swizzle(row)) << 4) + d % E * (int)sizeof(T);
      if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(to) = w;
      else *reinterpret_cast<u32x2*>(to) = u32x2{pack2(w[0], w[1]), pack2(w[2], w[3])};
    }
  __builtin_amdgcn_wave_barrier();      // a wave's own stores are visible to it in order
#pragma unroll
  for (int j = 0; j < 32 * TL::PPR / 64; ++j) {
    const int slot = j * 64 + lane, r = slot / TL::PPR, d = ((slot % TL::PPR) ^ TL::swizzle(r)) * E;
    const u32x4 w = *reinterpret_cast<const u32x4*>(lds + slot * 16);
    if (r < n && d < D) *reinterpret_cast<u32x4*>(rows + r * pitch + d) = w;
  }
}

template <int DP>
__device__ __forceinline__ void clear(f32x16 (&acc)[DP / 32]) {
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
}

// lse2 of a row whose weights add up to 0.  It sees no key: -inf.  All the scores that it sees are -inf: NaN, but where it is
// one of several splits, beside which the others' scores may be finite, a number below every finite lse2.
__device__ __forceinline__ float no_weight(bool sees, int nsplit) { return sees ? (nsplit > 1 ? -FLT_MAX : NAN) : -INFINITY; }

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// Consecutive workgroups go to the eight dies in turn: workgroups with neighbouring numbers after this share a die,
// and with it the L2 that holds their keys and values.
__device__ __forceinline__ int die_order(int id, int total) {
  const int per = total >> 3, rest = total & 7, die = id & 7, at = id >> 3;
  return die < rest ? die * (per + 1) + at : die * per + rest + at;
}

// Cell, query head (or pack of G of them) and key head of unit `id`.  All cells of a key head come before the next key head: a
// die's share then holds cells of every length where their masks differ, and the heads that share keys stay together.
struct Unit { int b, hu, kvh; };
__device__ __forceinline__ Unit unit_of(const AttnArgs& a, int id, int G) {
  const int per = a.H / a.Hkv / G, rest = id / per, kvh = rest / a.B;
  return Unit{rest % a.B, kvh * per + id % per, kvh};
}

// A mask word through the scalar cache: the mask is not written while a kernel runs, and a vector load's wait would be a wait
// for the tiles in flight too.
__device__ __forceinline__ u64 word_at(const u64* words, int i) {
  return ((const __attribute__((address_space(4))) u64*)words)[__builtin_amdgcn_readfirstlane(i)];
}
// Bits of the keys of tile t that exist and are not masked.
template <int BK>
__device__ __forceinline__ u64 tile_bits(const u64* words, int Sk, int t) {
  const int left = Sk - t * BK;
  u64 w = left >= BK ? (BK == 64 ? ~0ull : (1ull << (BK & 63)) - 1) : (left > 0 ? (1ull << left) - 1 : 0);
  if (words && left > 0) w &= BK == 64 ? word_at(words, t) : word_at(words, t >> 1) >> ((t & 1) * 32);
  return w;
}

// ---- few rows (sdpa_few.hip) -----------------------------------------------------------------------------------------
constexpr int FEW = 32;                      // rows that one wave holds
// Waves of a workgroup: as many as LDS holds tiles of keys and values for.
template <typename T, int DP> constexpr int few_waves() { return 32 * DP * (int)sizeof(T) * 2 <= 16384 ? 8 : 4; }
constexpr int ONE_WAVES = 16;                // of a workgroup for one row, which needs no tiles
template <typename T, int DP> constexpr int few_bwd_waves() { return 32 * DP * (int)sizeof(T) * 2 <= 8192 ? 8 : 4; }

int few_fwd(const AttnArgs& a, int dtype, hipStream_t st);
int few_bwd(const AttnArgs& a, int dtype, hipStream_t st);

}  // namespace attn
