// Scaled dot-product attention over any number of tokens, forward and backward.
//
//   s = scale q k^T, key j hidden from row i where its mask bit is 0 or (causal) j > i + Sk - Sq
//   o = softmax(s) v;  lse2 = log2(sum exp(s)) kept for the backward pass
//   a row that sees no key: o = 0, lse2 = -inf;  one with a score of +inf, or that sees scores of -inf alone: both NaN
//   p = exp2(log2(e) s - lse2);  delta = sum_d do o;  dp = do v^T;  ds = p (dp - delta)
//   dv = p^T do;  dq = scale ds k;  dk = scale ds^T q
//
// Every product runs on the matrix cores in 32 x 32 tiles (bf16: v_mfma_f32_32x32x16_bf16, float32:
// v_mfma_f32_32x32x2_f32 in groups of four), with scores, statistics, sums and accumulators in float32.  A score tile
// is computed transposed to the way it is used next: in the result layout a lane owns one column and sixteen rows (rows
// 8 (r / 4) + 4 (lane / 32) + r % 4), which is exactly the operand layout of the next product when its summed
// dimension is taken in that order.  So probabilities never leave the registers, a row's maximum and sum are
// reductions inside a lane plus one exchange between its halves, and the other operand is read from LDS in the same order
// (bf16: ds_read_b64_tr_b16, float32: ds_read_b32).
// bf16: p and ds are rounded to bf16 for the second product (2^-8 of each term), since the matrix cores take nothing wider at
// their rate; everything else is float32.  delta is formed from o as it was stored and what that rounding left (another bf16
// value of each, kept for the backward pass alone; 2 bytes written and read per element, 0.3-1 % of a training call): from the
// stored o alone the root mean square error of dq was 3.6-6.0 thousandths of dq where one key has most of a row's weight, with
// what rounding left 2.1-3.4 (2.1: dq's own rounding).
//
// LDS tiles hold rows of DP elements (the head dimension padded to 32, 64 or 128) in 16-byte pieces, written by the
// LDS-DMA loads lane by lane; piece p of row r sits at slot p ^ swizzle(r), so that both a column of 16 rows
// (ds_read_b128) and four rows side by side (the transposing read) touch all 64 banks.  What a row or piece lies outside
// the tensor, or belongs to a masked key, is requested beyond the buffer's range and arrives as zeros: a NaN stored
// behind a masked key reaches nothing.
#include "attn_tile.h"

using namespace attn;

namespace {

// ---- forward -------------------------------------------------------------------------------------------------------
// A workgroup owns 128 rows of one (cell, head), a wave 32 of them.  Keys and values pass through two LDS buffers; the loads
// of the next tile run under the products of this one.  Bound in bf16 by the vector units at 64 columns (64 keys take 32
// exponentials, sixteen cycles each, and some hundred other instructions beside 16 products) and by both units at 128, in
// float32 by the matrix cores.  The first product's waves go first (s_setprio), so that a SIMD's other wave is left the
// vector unit.
//   16 cells of 1000 to 2000 tokens, 8 heads of 64, bf16       145 us   (168 with each die holding two cells)
//   8192 causal, 32 heads of 128, 8 of keys and values, bf16   610 us   900 TFLOP/s (633 at one priority); 628 where what
//                                                              rounding left is kept for the backward pass
//   8 x 1000 tokens, 8 heads of 64, float32                    167 us    98 TFLOP/s
// The scores of the next tile formed ahead, between this one's exponentials, gave nothing (149, 617, 173 us).
template <typename T, int DP>
__global__ void __launch_bounds__(256, DP == 128 && sizeof(T) == 4 ? 1 : 2) attn_fwd_kernel(AttnArgs a) {
  typedef Tile<T, DP> TL;
  constexpr int BK = TL::BK, NT = BK / 32;
  __shared__ __align__(16) char smem[4 * TL::BYTES];       // k, v; k, v
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = die_order(blockIdx.x, gridDim.x);
  const int split = id % a.nsplit;
  id /= a.nsplit;
  const int rb = a.nrow - 1 - id % a.nrow, unit = id / a.nrow;      // the longest causal rows first
  const Unit un = unit_of(a, unit, 1);
  const int head = un.hu, b = un.b, kvh = un.kvh;
  const int row0 = rb * ROWS + wave * 32;
  const bool live = row0 + (lane & 31) < a.Sq;
  const int qi = live ? row0 + (lane & 31) : 0;
  const int off = a.Sk - a.Sq;
  u32x4 qf[DP / El<T>::CK];
  load_rows<T, DP>(qf, (const T*)a.q + b * a.sq.b + qi * a.sq.s + head * a.sq.h, a.D, live, lane);

  const T* kb = (const T*)a.k + b * a.sk.b + kvh * a.sk.h;
  const T* vb = (const T*)a.v + b * a.sv.b + kvh * a.sv.h;
  const u64* words = a.words ? a.words + (long long)b * a.nw : nullptr;
  // keys that the workgroup's / this wave's rows can see
  const int wg_end = a.causal ? min(a.Sk, min((rb + 1) * ROWS, a.Sq) + off) : a.Sk;
  const int wave_end = a.causal ? min(a.Sk, min(row0 + 32, a.Sq) + off) : a.Sk;
  const int free_end = a.causal ? row0 + off + 1 : a.Sk;       // all of the wave's rows see the keys below
  int tile = split * a.tiles_per_split;
  const int tend = min((wg_end + BK - 1) / BK, tile + a.tiles_per_split);
  const float sl2 = a.scale * LOG2E;

  f32x16 acc[DP / 32];
  clear<DP>(acc);
  float m = -INFINITY, l = 0.f;      // the row's maximum (of q k^T) and this lane's share of its sum

  u64 bits = 0, nbits;
  auto next = [&](int t) {
    for (nbits = 0; t < tend && (nbits = tile_bits<BK>(words, a.Sk, t)) == 0;) ++t;
    return t;
  };
  const typename TL::Shared from_k(WAVES, wave, lane, (unsigned)(a.sk.s * sizeof(T)), a.D);
  const typename TL::Shared from_v(WAVES, wave, lane, (unsigned)(a.sv.s * sizeof(T)), a.D);
  auto issue = [&](int t, int buf) {
    char* to = smem + buf * 2 * TL::BYTES;
    from_k.load(to, WAVES, wave, lane, kb + (long long)t * BK * a.sk.s, nbits, TL::ALL);
    from_v.load(to + TL::BYTES, WAVES, wave, lane, vb + (long long)t * BK * a.sv.s, nbits, TL::ALL);
  };
  tile = next(tile);
  const int first = tile < tend ? tile * BK + __builtin_ctzll(nbits) : INT_MAX;      // the first visible key
  if (tile < tend) issue(tile, 0);
  int buf = 0;
  while (tile < tend) {
    bits = nbits;
    const int after = next(tile + 1);
    tile_barrier();                  // this tile has arrived, and nobody reads the other buffer any more
    if (after < tend) issue(after, buf ^ 1);
    const int key0 = tile * BK;
    if (key0 < wave_end) {
      const char* ks = smem + buf * 2 * TL::BYTES;
      const char* vs = ks + TL::BYTES;
      f32x16 s[NT];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[nt][r] = 0.f;
#pragma unroll
        for (int c = 0; c < DP / El<T>::CK; ++c) s[nt] = El<T>::mma(TL::frag(ks, 32 * nt, c, lane), qf[c], s[nt]);
      }
      __builtin_amdgcn_s_setprio(0);
      if (bits != TL::ALL || key0 + BK > free_end) {
        const int reach = a.causal ? qi + off - key0 - 4 * half : BK;      // this row sees keys up to here
        const u64 w = bits >> (4 * half);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint32_t w32 = (uint32_t)(w >> (32 * nt));
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = 8 * (r >> 2) + (r & 3);
            s[nt][r] = ((w32 >> key) & 1) && 32 * nt + key <= reach ? s[nt][r] : -INFINITY;
          }
        }
      }
      float top = s[0][0];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[nt][r]);
      top = fmaxf(top, other_half(top));
      // The running maximum is raised only when a row's scores outgrow it by 2^8 (then every accumulator is scaled);
      // below that exp2 stays far from overflow and the result is the same quotient.
      if (__any(top * sl2 > (m == -INFINITY ? -INFINITY : m * sl2 + 8.f))) {
        const float mn = fmaxf(m, top);
        const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f((m - mn) * sl2);
        l *= f;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] *= f;
        m = mn;
      }
      const float base = m == -INFINITY ? 0.f : -m * sl2;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[nt][r] = __builtin_amdgcn_exp2f(fmaf(s[nt][r], sl2, base));
          l += s[nt][r];
        }
        Second<T, DP>::run(acc, vs, 32 * nt, s[nt], lane);
      }
    }
    tile = after;
    buf ^= 1;
  }
  l += other_half(l);
  // No weight at all: the row sees no key, or only scores of -inf, whose quotient is not a number
  const float none = no_weight(first <= (a.causal ? qi + off : INT_MAX - 1), a.nsplit);
  const float inv = l == 0.f ? (none != none ? none : 0.f) : 1.f / l;
  const float lse2 = l == 0.f ? none : m * sl2 + __builtin_amdgcn_logf(l);
  if (!live) return;
  if (l == 0.f) clear<DP>(acc);      // not multiplied by 0: a value that only other rows see may be infinite
  const long long at = ((long long)b * a.Sq + qi) * a.H + head;
  if (a.nsplit > 1) {
    const long long n = (long long)a.B * a.Sq * a.H;
    store_rows<float, DP>(a.part + (split * n + at) * a.D, acc, inv, a.D, lane);
    if (half == 0) a.part_lse[split * n + at] = lse2;
  } else {
    store_rows<T, DP>((T*)a.out + at * a.D, acc, inv, a.D, lane, a.out_low ? (u16*)a.out_low + at * a.D : nullptr);
    if (half == 0 && a.lse2) a.lse2[((long long)b * a.H + head) * a.Sq + qi] = lse2;
  }
}

// The splits of one row joined: o = sum_i 2^(lse_i - lse) o_i, lse = log2(sum_i 2^lse_i).  One wave per row: a lane per
// split for the weights, then DP / 4 lanes across a result and 256 / DP splits side by side.  Bound by the latency of its
// two readings (128 rows of 16 splits: 9 us, 17 with every lane reading every split in turn).
template <typename T, int DP>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a) {
  constexpr int ACROSS = DP / 4, SIDE = 64 / ACROSS;
  const int lane = threadIdx.x & 63;
  const long long n = (long long)a.B * a.Sq * a.H, at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= n) return;
  float top = -INFINITY;
  for (int i = lane; i < a.nsplit; i += 64) top = fmaxf(top, a.part_lse[i * n + at]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float base = top == -INFINITY ? 0.f : top;
  const int side = lane / ACROSS, d = lane % ACROSS * 4;
  float total = 0.f;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < a.nsplit; i0 += 64) {
    const float w = i0 + lane < a.nsplit ? __builtin_amdgcn_exp2f(a.part_lse[(i0 + lane) * n + at] - base) : 0.f;
    total += w;
    const int m = min(64, a.nsplit - i0);
    for (int i = side; i < m + side; i += 8 * SIDE)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int of = i + k * SIDE;
        const float wi = __shfl(w, of & 63, 64);
        if (of < m && d < a.D) s += wi * *reinterpret_cast<const f32x4*>(a.part + ((i0 + of) * n + at) * a.D + d);
      }
  }
#pragma unroll
  for (int o = ACROSS; o < 64; o <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += __shfl_xor(s[j], o, 64);
  total = wave_sum(total);
  const bool lost = top == -FLT_MAX;      // keys are seen, every score is -inf
  const float inv = lost ? NAN : total == 0.f ? 0.f : 1.f / total;
  if (side == 0 && d < a.D) {
    s *= inv;
    const float w[4] = {s[0], s[1], s[2], s[3]};
    put4<T>((T*)a.out + at * a.D + d, a.out_low ? (u16*)a.out_low + at * a.D + d : nullptr, w);
  }
  if (lane == 0 && a.lse2) {
    const long long h = at % a.H, bq = at / a.H;
    a.lse2[(bq / a.Sq * a.H + h) * a.Sq + bq % a.Sq] = lost ? NAN : total == 0.f ? -INFINITY : base + __builtin_amdgcn_logf(total);
  }
}

// words[b][w]: bit i = key 64 w + i of cell b is visible.
__global__ void __launch_bounds__(256) attn_words_kernel(u64* words, const uint8_t* mask, long long ldm, int B, int Sk, int nw) {
  const int lane = threadIdx.x & 63, w = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= nw) return;
  const int key = w * 64 + lane;
  for (int b = blockIdx.y; b < B; b += gridDim.y) {
    const u64 bits = __ballot(key < Sk && mask[(long long)b * ldm + key] != 0);
    if (lane == 0) words[(long long)b * nw + w] = bits;
  }
}

// ---- backward ------------------------------------------------------------------------------------------------------
// ndelta (B, H, Sq) = -sum_d do o (o with what its rounding to bf16 left, where that was kept), from which the products dp = do v^T start, and nlse = -lse2, or -inf for a row that sees nothing: its probabilities are all 0.
// Eight lanes per row.
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(AttnArgs a) {
  const long long n = (long long)a.B * a.Sq * a.H, at = (long long)blockIdx.x * 32 + (threadIdx.x >> 3);
  if (at >= n) return;
  const long long h = at % a.H, bq = at / a.H, b = bq / a.Sq, q = bq % a.Sq;
  const T* o = (const T*)a.o + at * a.D;
  const T* low = a.low ? (const T*)a.low + at * a.D : nullptr;
  const T* g = (const T*)a.dout + b * a.sdo.b + q * a.sdo.s + h * a.sdo.h;
  constexpr int E = 16 / sizeof(T);
  float s = 0.f;
  for (int d = (threadIdx.x & 7) * E; d < a.D; d += 8 * E) {
    typedef typename El<T>::Vec4 V4;
    const V4 x = *reinterpret_cast<const V4*>(o + d), y = *reinterpret_cast<const V4*>(g + d);
    V4 z{};
    if (sizeof(T) == 2 && low) z = *reinterpret_cast<const V4*>(low + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        s = fmaf(x[j], y[j], s);
      } else {
        const float y0 = __builtin_bit_cast(float, y[j] << 16), y1 = __builtin_bit_cast(float, y[j] & 0xffff0000u);
        s = fmaf(__builtin_bit_cast(float, x[j] << 16) + __builtin_bit_cast(float, z[j] << 16), y0, s);
        s = fmaf(__builtin_bit_cast(float, x[j] & 0xffff0000u) + __builtin_bit_cast(float, z[j] & 0xffff0000u), y1, s);
      }
    }
  }
#pragma unroll
  for (int o2 = 4; o2 > 0; o2 >>= 1) s += __shfl_xor(s, o2, 64);
  if ((threadIdx.x & 7) == 0) {
    const long long stat = (b * a.H + h) * a.Sq + q;
    const float l = a.lse2[stat];
    a.nlse[stat] = l == -INFINITY ? l : -l;
    a.ndelta[stat] = -s;
  }
}

// dq of 128 rows: the forward kernel's loop with the probabilities recomputed from lse2 and ndelta as what the products
// do v^T start from.  Three products a tile, so nearer the matrix cores' bound: 8192 causal, 32 heads of 128, 8 of keys
// and values, bf16: 750 us, 1100 TFLOP/s; 8 x 1000 tokens, 8 heads of 64, float32: 246 us, 100 TFLOP/s.  A launch of its own
// beside dk, dv forms s and dp twice, seven products where five would do: one launch for both would add dq up in memory, in no
// fixed order, or keep a partial dq for every block of keys and add those (in float32 the cheaper way by its bytes: 131 MB at
// 8 x 1000 x 8 x 64, some 55 us, against 160 for two products; not built).
template <typename T, int DP>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) attn_dq_kernel(AttnArgs a) {
  typedef Tile<T, DP> TL;
  constexpr int BK = TL::BK, NT = BK / 32;
  __shared__ __align__(16) char smem[4 * TL::BYTES];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = die_order(blockIdx.x, gridDim.x);
  const int split = id % a.nsplit;
  id /= a.nsplit;
  const int rb = a.nrow - 1 - id % a.nrow, unit = id / a.nrow;
  const Unit un = unit_of(a, unit, 1);
  const int head = un.hu, b = un.b, kvh = un.kvh;
  const int row0 = rb * ROWS + wave * 32;
  const bool live = row0 + (lane & 31) < a.Sq;
  const int qi = live ? row0 + (lane & 31) : 0;
  const int off = a.Sk - a.Sq;
  const long long stat = ((long long)b * a.H + head) * a.Sq + qi;
  float base = live ? a.nlse[stat] : -INFINITY;
  const bool some = base != -INFINITY;       // a row that sees nothing has no gradient, whatever arrives in do
  float nd = some ? a.ndelta[stat] : 0.f;
  settle(base), settle(nd);
  u32x4 qf[DP / El<T>::CK], gf[DP / El<T>::CK];
  load_rows<T, DP>(qf, (const T*)a.q + b * a.sq.b + qi * a.sq.s + head * a.sq.h, a.D, some, lane);
  load_rows<T, DP>(gf, (const T*)a.dout + b * a.sdo.b + qi * a.sdo.s + head * a.sdo.h, a.D, some, lane);

  const T* kb = (const T*)a.k + b * a.sk.b + kvh * a.sk.h;
  const T* vb = (const T*)a.v + b * a.sv.b + kvh * a.sv.h;
  const u64* words = a.words ? a.words + (long long)b * a.nw : nullptr;
  const int wg_end = a.causal ? min(a.Sk, min((rb + 1) * ROWS, a.Sq) + off) : a.Sk;
  const int wave_end = a.causal ? min(a.Sk, min(row0 + 32, a.Sq) + off) : a.Sk;
  const int free_end = a.causal ? row0 + off + 1 : a.Sk;
  int tile = split * a.tiles_per_split;
  const int tend = min((wg_end + BK - 1) / BK, tile + a.tiles_per_split);
  const float sl2 = a.scale * LOG2E;

  f32x16 acc[DP / 32];
  clear<DP>(acc);

  u64 bits = 0, nbits;
  auto next = [&](int t) {
    for (nbits = 0; t < tend && (nbits = tile_bits<BK>(words, a.Sk, t)) == 0;) ++t;
    return t;
  };
  const typename TL::Shared from_k(WAVES, wave, lane, (unsigned)(a.sk.s * sizeof(T)), a.D);
  const typename TL::Shared from_v(WAVES, wave, lane, (unsigned)(a.sv.s * sizeof(T)), a.D);
  auto issue = [&](int t, int buf) {
    char* to = smem + buf * 2 * TL::BYTES;
    from_k.load(to, WAVES, wave, lane, kb + (long long)t * BK * a.sk.s, nbits, TL::ALL);
    from_v.load(to + TL::BYTES, WAVES, wave, lane, vb + (long long)t * BK * a.sv.s, nbits, TL::ALL);
  };
  tile = next(tile);
  if (tile < tend) issue(tile, 0);
  int buf = 0;
  while (tile < tend) {
    bits = nbits;
    const int after = next(tile + 1);
    tile_barrier();
    if (after < tend) issue(after, buf ^ 1);
    const int key0 = tile * BK;
    if (key0 < wave_end) {
      const char* ks = smem + buf * 2 * TL::BYTES;
      const char* vs = ks + TL::BYTES;
      const bool masked = bits != TL::ALL || key0 + BK > free_end;
      const int reach = a.causal ? qi + off - key0 - 4 * half : BK;
      const u64 w = bits >> (4 * half);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f, dp[r] = nd;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int c = 0; c < DP / El<T>::CK; ++c) {
          s = El<T>::mma(TL::frag(ks, 32 * nt, c, lane), qf[c], s);
          dp = El<T>::mma(TL::frag(vs, 32 * nt, c, lane), gf[c], dp);
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl2, base)) * dp[r];
        if (masked) {
          const uint32_t w32 = (uint32_t)(w >> (32 * nt));
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = 8 * (r >> 2) + (r & 3);
            s[r] = ((w32 >> key) & 1) && 32 * nt + key <= reach ? s[r] : 0.f;
          }
        }
        Second<T, DP>::run(acc, ks, 32 * nt, s, lane);
      }
    }
    tile = after;
    buf ^= 1;
  }
  if (!live) return;
  if (!some) clear<DP>(acc);
  const long long at = ((long long)b * a.Sq + qi) * a.H + head;
  if (a.nsplit > 1)
    store_rows<float, DP>(a.part + (split * (long long)a.B * a.Sq * a.H + at) * a.D, acc, a.scale, a.D, lane);
  else
    store_rows<T, DP>((T*)a.dq + at * a.D, acc, a.scale, a.D, lane);
}

// dk, dv of 32 W keys of one key head: a wave keeps its 32 values, (KEYS_LDS: not) its keys and both accumulators in
// registers, and the query heads of the group with their rows pass through LDS (q, do, nlse, ndelta).  Four products a tile.
// 128 bf16 columns with the keys in registers make 412 of them, one wave a SIMD, whose products and exponentials then take
// turns (8192 causal, 32 heads of 128, 8 of keys and values: 1577 us); with the keys in LDS two waves fit (1160 us, 950
// TFLOP/s, each block's rows in two halves), and in float32 nothing spills any more.  64 keys a
// wave, which halves the reads of LDS, is slower again (one wave a SIMD: 2636 us).  8 x 1000 tokens, 8 heads of 64,
// float32: 310 us, 106 TFLOP/s.
template <typename T, int DP, int W, bool KEYS_LDS>
__global__ void __launch_bounds__(64 * W, sizeof(T) == 4 && DP == 128 ? 1 : DP == 32 ? 4 : 2) attn_dkv_kernel(AttnArgs a) {
  typedef Tile<T, DP> TL;
  constexpr int BK = TL::BK, NT = BK / 32, CH = DP / El<T>::CK;
  typedef typename TL::template Source<TL::BYTES / (1024 * W)> From;
  __shared__ __align__(16) char smem[4 * TL::BYTES];       // q, do; q, do
  __shared__ __align__(16) char keys[KEYS_LDS ? 32 * W * TL::RB : 16];
  __shared__ __align__(16) float stats[2][2][64];          // nlse, ndelta
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = die_order(blockIdx.x, gridDim.x);
  const int split = id % a.nsplit;
  id /= a.nsplit;
  const int rb = id % a.nrow, unit = id / a.nrow;          // causal: the first keys are seen by the most rows
  const int kvh = unit / a.B, b = unit % a.B, group = a.H / a.Hkv;
  const int block0 = rb * 32 * W, key0 = block0 + wave * 32, key = key0 + (lane & 31), off = a.Sk - a.Sq;
  bool seen = key < a.Sk;
  if (seen && a.words) seen = (a.words[(long long)b * a.nw + (key >> 6)] >> (key & 63)) & 1;
  u32x4 kf[KEYS_LDS ? 1 : CH], vf[CH];
  {
    const long long kk = seen ? key : 0;
    if constexpr (!KEYS_LDS) load_rows<T, DP>(kf, (const T*)a.k + b * a.sk.b + kk * a.sk.s + kvh * a.sk.h, a.D, seen, lane);
    load_rows<T, DP>(vf, (const T*)a.v + b * a.sv.b + kk * a.sv.s + kvh * a.sv.h, a.D, seen, lane);
  }
  f32x16 dk[DP / 32], dv[DP / 32];
  clear<DP>(dk), clear<DP>(dv);
  const float sl2 = a.scale * LOG2E;

  // the first key of the workgroup that any row sees
  int seen0 = block0;
  if (a.words) {
    seen0 = a.Sk;
    for (int i = 32 * W / 64 - 1; i >= 0; --i) {
      const int at = block0 / 64 + i;
      const u64 w = at < a.nw ? word_at(a.words + (long long)b * a.nw, at) : 0;
      if (w) seen0 = at * 64 + __builtin_ctzll(w);
    }
  }
  // causal: rows from here on see any of the workgroup's / all of the wave's keys.  Rows before the first see none of
  // them, perhaps no key at all: they arrive as zeros, whatever their do holds
  const int first = a.causal ? max(0, seen0 - off) : 0;
  const int wave_first = a.causal ? key0 - off : 0, free_first = a.causal ? max(key0 + 31 - off, first) : 0;
  const int t0 = first / BK, tq = max(0, (a.Sq + BK - 1) / BK - t0);       // tiles per query head
  const int steps = tq * group;
  // every block's steps are divided evenly: the blocks come in the order of their work, the longest first
  int step = (int)((long long)steps * split / a.nsplit);
  const int end = (int)((long long)steps * (split + 1) / a.nsplit);
  const bool work = seen0 < a.Sk;

  if constexpr (KEYS_LDS) {
    if (work) {
      const u64* words = a.words ? a.words + (long long)b * a.nw : nullptr;
      const From from_k(W, wave, lane, (unsigned)(a.sk.s * sizeof(T)), a.D);
      for (int i = 0; i < 32 * W / BK; ++i)
        from_k.load(keys + i * TL::BYTES, W, wave, lane, (const T*)a.k + b * a.sk.b + (long long)(block0 + i * BK) * a.sk.s + kvh * a.sk.h,
                    tile_bits<BK>(words, a.Sk, block0 / BK + i), TL::ALL);
    }
  }
  const From from_q(W, wave, lane, (unsigned)(a.sq.s * sizeof(T)), a.D);
  const From from_g(W, wave, lane, (unsigned)(a.sdo.s * sizeof(T)), a.D);
  // rows outside the tensor arrive as zeros, statistics too
  auto issue = [&](int st, int buf) {
    const int head = kvh * group + st / tq, r0 = (t0 + st % tq) * BK, left = a.Sq - r0;
    u64 rows = left >= 64 ? ~0ull : (1ull << left) - 1;
    if (r0 < first) rows &= ~0ull << (first - r0);
    if (wave < 2) {
      const float* stat = (wave ? a.ndelta : a.nlse) + ((long long)b * a.H + head) * a.Sq + r0;
      dma4(dma_rsrc(stat), &stats[buf][wave][0], lane < BK && ((rows >> lane) & 1) ? 4u * lane : DMA_OUTSIDE);
    }
    rows &= TL::ALL;
    char* to = smem + buf * 2 * TL::BYTES;
    from_q.load(to, W, wave, lane, (const T*)a.q + b * a.sq.b + (long long)r0 * a.sq.s + head * a.sq.h, rows, TL::ALL);
    from_g.load(to + TL::BYTES, W, wave, lane, (const T*)a.dout + b * a.sdo.b + (long long)r0 * a.sdo.s + head * a.sdo.h, rows, TL::ALL);
  };
  if (work && step < end) issue(step, 0);
  int buf = 0;
  for (; work && step < end; ++step) {
    tile_barrier();
    if (step + 1 < end) issue(step + 1, buf ^ 1);
    const int r0 = (t0 + step % tq) * BK;
    const char* qs = smem + buf * 2 * TL::BYTES;
    const char* gs = qs + TL::BYTES;
#pragma unroll 1
    for (int nt = 0; nt < NT; ++nt) {
      const int q0 = r0 + 32 * nt;
      if (q0 + 31 < wave_first || q0 >= a.Sq) continue;
      f32x16 s, dp;
      int at = lane;
      asm volatile("" : "+v"(at));      // addresses are worked out again for every 32 rows: kept, they do not fit
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 nd = *reinterpret_cast<const f32x4*>(&stats[buf][1][32 * nt + 8 * g + 4 * half]);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * g + j] = 0.f, dp[4 * g + j] = nd[j];
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if constexpr (KEYS_LDS) s = El<T>::mma(TL::frag(qs, 32 * nt, c, at), TL::frag(keys, 32 * wave, c, at), s);
        else s = El<T>::mma(TL::frag(qs, 32 * nt, c, at), kf[c], s);
        dp = El<T>::mma(TL::frag(gs, 32 * nt, c, at), vf[c], dp);
      }
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(&stats[buf][0][32 * nt + 8 * g + 4 * half]);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * g + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + j], sl2, ls[j]));
      }
      if (q0 < free_first || q0 + 32 > a.Sq) {
        // rows that see this lane's key; the others count for nothing, also where an infinite key met their zeros
        const int from = (a.causal ? max(key - off, first) : 0) - q0 - 4 * half, to = a.Sq - q0 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = 8 * (r >> 2) + (r & 3);
          if (row < from || row >= to) s[r] = dp[r] = 0.f;
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] *= s[r];
      asm volatile("" : "+v"(at));
      Second<T, DP>::run(dv, gs, 32 * nt, s, at);
      Second<T, DP>::run(dk, qs, 32 * nt, dp, at);
    }
    buf ^= 1;
  }
  if (key >= a.Sk) return;
  // a masked key has no gradient; what its lane computed from a zero row is dropped, not multiplied
  if (!seen) clear<DP>(dk), clear<DP>(dv);
  const long long at = ((long long)b * a.Sk + key) * a.Hkv + kvh;
  if (a.nsplit > 1) {
    const long long n = (long long)a.B * a.Sk * a.Hkv;
    store_rows<float, DP>(a.part + (split * n + at) * a.D, dk, a.scale, a.D, lane);
    store_rows<float, DP>(a.part + ((a.nsplit + split) * n + at) * a.D, dv, 1.f, a.D, lane);
  } else {
    store_rows<T, DP>((T*)a.dk + at * a.D, dk, a.scale, a.D, lane);
    store_rows<T, DP>((T*)a.dv + at * a.D, dv, 1.f, a.D, lane);
  }
}

// out[i] = sum over splits of part[split][i], in split order; four elements a thread.  blockIdx.y: the second of two.
template <typename T>
__global__ void __launch_bounds__(256) attn_sum_kernel(T* out0, T* out1, const float* part, long long n, int nsplit) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const float* p = part + (blockIdx.y ? nsplit * n : 0) + i;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < nsplit; ++k) s += *reinterpret_cast<const f32x4*>(p + k * n);
  T* out = (blockIdx.y ? out1 : out0) + i;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4*>(out) = s;
  } else {
    *reinterpret_cast<u32x2*>(out) = u32x2{pack2(s[0], s[1]), pack2(s[2], s[3])};
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------
// Splits of a loop of `tiles` tiles so that `wgs` workgroups, if fewer than `least`, become about `fill`, each with at
// least four tiles.
int splits_for(long long wgs, int tiles, int least, int fill) {
  if (wgs >= least || tiles < 8) return 1;
  long long n = (fill + wgs - 1) / (wgs < 1 ? 1 : wgs);
  if (n > tiles / 4) n = tiles / 4;
  return n < 1 ? 1 : (int)n;
}

struct Plan {
  bool few;          // sdpa_few.hip: at most 32 rows
  int G, nrow, nsplit, tps;
};
int bk_of(int dtype) { return dtype == CG_BF16 ? El<u16>::BK : El<float>::BK; }

void set_splits(Plan& p, int tiles, int nsplit) {
  p.tps = tiles ? (tiles + nsplit - 1) / nsplit : 1;
  p.nsplit = tiles ? (tiles + p.tps - 1) / p.tps : 1;
}

// Rows of the forward and dq kernels.  Few rows: as many of a group's query heads as the 32 rows of a wave hold (the keys
// are read once for them), the keys divided over the waves of a workgroup, and over more workgroups where the cells and
// heads alone are few: two a CU where all keys count (one query of 32 heads, 8 of them of keys and values, 65537 x 128 bf16,
// four cells: 207 us, and 254 with eight a CU).  Forward, four a CU where a mask may leave most of a cell's keys out, since
// the longest cell ends last (16 latents and 5000 genes of 32 ragged cells, 8 heads of 64: 74 us, 86 with two a CU, 74 with
// eight; backward, which writes for every key, 114, 115 and 130).  A wave keeps two tiles (4 cells, 2 query heads over each
// of 8, 2000 x 64: bf16 12 us, float32 24; 13 and 42 with four tiles, 11 and 17 with one, but 3 cells, 4 over 1, 25000 x 64:
// 15 and 26, with one tile 20 and 35); one row's waves, with loads enough under way, one (3 cells, 25316 x 128, float32: 25 us, 34
// with four).
Plan row_plan(int B, int H, int Hkv, int Sq, int Sk, int D, int dtype, bool bwd, bool uneven) {
  Plan p{};
  const int group = H / Hkv;
  p.G = 1;
  for (int g = 2; g <= group && Sq * g <= FEW; ++g)
    if (group % g == 0) p.G = g;
  const int bytes = 64 * (D <= 32 ? 32 : D <= 64 ? 64 : 128) * (dtype == CG_BF16 ? 2 : 4);      // a wave's keys and values
  p.few = Sq <= FEW && (!bwd || (p.G == group && bytes <= 16384));
  if (p.few) {
    const bool one = !bwd && Sq * p.G == 1;
    const int waves = bwd ? (bytes <= 8192 ? 8 : 4) : one ? ONE_WAVES : bytes <= 16384 ? 8 : 4;
    const int tiles = (Sk + 31) / 32, target = uneven && !bwd ? 1024 : 512, least = one ? 1 : 2;
    const long long units = (long long)B * (H / p.G);
    p.nrow = 1;
    long long n = target / units;
    if (n > tiles / (least * waves)) n = tiles / (least * waves);
    set_splits(p, tiles, n < 1 ? 1 : (int)n);
    if (one && p.tps % 2) {      // whole mask words: a wave's batch of up to 64 keys lies in one of them
      ++p.tps;
      p.nsplit = tiles ? (tiles + p.tps - 1) / p.tps : 1;
    }
    return p;
  }
  p.G = 1;
  p.nrow = (Sq + ROWS - 1) / ROWS;
  const int tiles = (Sk + bk_of(dtype) - 1) / bk_of(dtype);
  set_splits(p, tiles, splits_for((long long)B * H * p.nrow, tiles, 512, 1024));
  return p;
}
// Blocks of keys of the dk, dv kernel: of 256 where its workgroups have eight waves, one a CU, else of 128.  Causal blocks
// differ in length; in halves, the longest first, they even out (8192 causal, 8 heads of 128: 256 blocks 1900 us, 512 halves
// 1160 and 25 for their sums, quarters 1160 and 51).
Plan key_plan(int B, int H, int Hkv, int Sq, int Sk, int D, int dtype, bool causal) {
  Plan p{};
  p.G = 1;
  const bool wide = dtype == CG_BF16 && D > 64;
  const int keys = wide ? 256 : 128;
  p.nrow = (Sk + keys - 1) / keys;
  const long long steps = (long long)((Sq + bk_of(dtype) - 1) / bk_of(dtype)) * (H / Hkv), wgs = (long long)B * Hkv * p.nrow;
  set_splits(p, (int)steps, wide ? splits_for(wgs, (int)steps, causal ? 512 : 256, 512) : splits_for(wgs, (int)steps, 512, 1024));
  return p;
}

int attn_shape_ok(int B, int H, int Hkv, int Sq, int Sk, int D, int dtype) {
  if (B < 0 || H < 1 || Hkv < 1 || Sq < 0 || Sk < 0 || D < 1 || H % Hkv != 0) return CG_ERR_BAD_ARG;
  if (dtype != CG_F32 && dtype != CG_BF16) return CG_ERR_BAD_ARG;
  if (D > 128 || D % (dtype == CG_BF16 ? 8 : 4) != 0) return CG_ERR_UNSUPPORTED;
  // a launch has fewer than 2^32 threads, up to 1024 of them for 128 rows; row numbers are 32-bit
  if ((long long)Sq * H >= (1ll << 31) || (long long)B * H * ((Sq + (ROWS - 1ll)) / ROWS) >= (1 << 22) ||
      (long long)B * Hkv * ((Sk + (ROWS - 1ll)) / ROWS) >= (1 << 22) || Sk > (1 << 30))
    return CG_ERR_UNSUPPORTED;
  return CG_OK;
}

// 16-byte pieces: the tensor's address and every stride that is used are multiples of 16 bytes; a tile's rows lie
// within 2^31 bytes.
bool operand_ok(const void* p, const Strides& s, int B, int S, int heads, int dtype) {
  const int e = dtype == CG_BF16 ? 8 : 4, size = 16 / e;
  if (((uintptr_t)p & 15) || (B > 1 && s.b % e) || (S > 1 && s.s % e) || (heads > 1 && s.h % e)) return false;
  return s.s >= 0 && (S <= 1 || s.s * size * 64 < (1ll << 31)) && s.b >= 0 && s.h >= 0;
}

#define BY_DP(KERNEL, T, ...)                              \
  do {                                                     \
    if (a.D <= 32) KERNEL<T, 32> __VA_ARGS__;              \
    else if (a.D <= 64) KERNEL<T, 64> __VA_ARGS__;         \
    else KERNEL<T, 128> __VA_ARGS__;                       \
  } while (0)

template <typename T>
int fwd_run(AttnArgs a, const Plan& p, hipStream_t st) {
  a.G = p.G, a.nrow = p.nrow, a.nsplit = p.nsplit, a.tiles_per_split = p.tps;
  if (p.few) {
    few_fwd(a, sizeof(T) == 4 ? CG_F32 : CG_BF16, st);
  } else {
    const unsigned grid = (unsigned)((long long)a.B * a.H * a.nrow * a.nsplit);
    BY_DP(attn_fwd_kernel, T, <<<grid, 256, 0, st>>>(a));
  }
  if (a.nsplit > 1)
    BY_DP(attn_join_kernel, T, <<<(unsigned)(((long long)a.B * a.Sq * a.H + 3) / 4), 256, 0, st>>>(a));
  return cg_launch_status();
}

template <typename T>
int bwd_run(AttnArgs a, const Plan& pr, const Plan& pk, hipStream_t st) {
  const long long nq = (long long)a.B * a.Sq * a.H, nk = (long long)a.B * a.Sk * a.Hkv;
  if (nq > 0) {
    attn_delta_kernel<T><<<(unsigned)((nq + 31) / 32), 256, 0, st>>>(a);
    AttnArgs r = a;
    r.G = pr.G, r.nrow = pr.nrow, r.nsplit = pr.nsplit, r.tiles_per_split = pr.tps;
    if (pr.few) {
      few_bwd(r, sizeof(T) == 4 ? CG_F32 : CG_BF16, st);
    } else {
      const unsigned grid = (unsigned)((long long)a.B * a.H * r.nrow * r.nsplit);
      BY_DP(attn_dq_kernel, T, <<<grid, 256, 0, st>>>(r));
    }
    if (r.nsplit > 1)
      attn_sum_kernel<T><<<(unsigned)((nq * a.D / 4 + 255) / 256), 256, 0, st>>>((T*)a.dq, nullptr, a.part, nq * a.D, r.nsplit);
  }
  if (nk > 0 && !(pr.few && nq > 0)) {      // the few-rows kernel has written dk and dv
    AttnArgs r = a;
    r.G = 1, r.nrow = pk.nrow, r.nsplit = pk.nsplit, r.tiles_per_split = pk.tps;
    const unsigned grid = (unsigned)((long long)a.B * a.Hkv * r.nrow * r.nsplit);
    if (a.D <= 32) attn_dkv_kernel<T, 32, 4, false><<<grid, 256, 0, st>>>(r);
    else if (a.D <= 64) attn_dkv_kernel<T, 64, 4, false><<<grid, 256, 0, st>>>(r);
    else if constexpr (sizeof(T) == 4) attn_dkv_kernel<T, 128, 4, true><<<grid, 256, 0, st>>>(r);
    else attn_dkv_kernel<T, 128, 8, true><<<grid, 512, 0, st>>>(r);
    if (r.nsplit > 1)
      attn_sum_kernel<T><<<dim3((unsigned)((nk * a.D / 4 + 255) / 256), 2), 256, 0, st>>>((T*)a.dk, (T*)a.dv, a.part, nk * a.D, r.nsplit);
  }
  return cg_launch_status();
}

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

extern "C" int cg_attention_mask_words(void* words, const uint8_t* mask, long long ldm, int B, int Sk, void* stream) {
  if (B < 0 || Sk < 0 || Sk > (1 << 30) || ldm < 0) return CG_ERR_BAD_ARG;
  if (B == 0 || Sk == 0) return CG_OK;
  if (!words || !mask) return CG_ERR_BAD_ARG;
  const int nw = (Sk + 63) / 64;
  attn_words_kernel<<<dim3((nw + 3) / 4, B < 4096 ? B : 4096), 256, 0, (hipStream_t)stream>>>((u64*)words, mask, ldm, B, Sk, nw);
  return cg_launch_status();
}

extern "C" size_t cg_attention_fwd_workspace_bytes(int B, int H, int Hkv, int Sq, int Sk, int D, int dtype) {
  if (attn_shape_ok(B, H, Hkv, Sq, Sk, D, dtype) != CG_OK || B == 0 || Sq == 0) return 0;
  const Plan p = row_plan(B, H, Hkv, Sq, Sk, D, dtype, false, true);      // the more splits
  if (p.nsplit == 1) return 0;
  const size_t n = (size_t)B * Sq * H * p.nsplit;
  return up16(n * D * 4) + n * 4;
}

extern "C" int cg_attention_fwd(void* O, float* lse2, const void* Q, long long qb, long long qs, long long qh, const void* K,
                                long long kb, long long ks, long long kh, const void* V, long long vb, long long vs,
                                long long vh, const void* words, int B, int H, int Hkv, int Sq, int Sk, int D, float scale,
                                int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return cg_attention_fwd_low(O, nullptr, lse2, Q, qb, qs, qh, K, kb, ks, kh, V, vb, vs, vh, words, B, H, Hkv, Sq, Sk, D, scale,
                              causal, dtype, workspace, workspace_bytes, stream);
}

extern "C" int cg_attention_fwd_low(void* O, void* Olow, float* lse2, const void* Q, long long qb, long long qs, long long qh, const void* K,
                                long long kb, long long ks, long long kh, const void* V, long long vb, long long vs,
                                long long vh, const void* words, int B, int H, int Hkv, int Sq, int Sk, int D, float scale,
                                int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const int ok = attn_shape_ok(B, H, Hkv, Sq, Sk, D, dtype);
  if (ok != CG_OK) return ok;
  if (!(scale > 0.f) || scale > 3e38f) return CG_ERR_BAD_ARG;
  if (B == 0 || Sq == 0) return CG_OK;
  if (!O || !Q || (Sk > 0 && (!K || !V)) || (Olow && dtype != CG_BF16)) return CG_ERR_BAD_ARG;
  const Strides sq{qb, qs, qh}, sk{kb, ks, kh}, sv{vb, vs, vh};
  if (!operand_ok(Q, sq, B, Sq, H, dtype) || !operand_ok(K, sk, B, Sk, Hkv, dtype) || !operand_ok(V, sv, B, Sk, Hkv, dtype) ||
      (((uintptr_t)O | (uintptr_t)Olow) & 15))
    return CG_ERR_UNSUPPORTED;
  const Plan p = row_plan(B, H, Hkv, Sq, Sk, D, dtype, false, words != nullptr);
  if (p.nsplit > 1 && (!workspace || ((uintptr_t)workspace & 15) ||
                       workspace_bytes < cg_attention_fwd_workspace_bytes(B, H, Hkv, Sq, Sk, D, dtype)))
    return CG_ERR_WORKSPACE;
  AttnArgs a{};
  a.q = Q, a.k = K, a.v = V, a.sq = sq, a.sk = sk, a.sv = sv, a.out = O, a.out_low = Olow, a.lse2 = lse2;
  a.words = (const u64*)words;
  a.B = B, a.H = H, a.Hkv = Hkv, a.Sq = Sq, a.Sk = Sk, a.D = D, a.nw = (Sk + 63) / 64, a.scale = scale, a.causal = causal;
  a.part = (float*)workspace;
  if (p.nsplit > 1) a.part_lse = (float*)((char*)workspace + up16((size_t)B * Sq * H * p.nsplit * D * 4));
  hipStream_t st = (hipStream_t)stream;
  return dtype == CG_F32 ? fwd_run<float>(a, p, st) : fwd_run<u16>(a, p, st);
}

extern "C" size_t cg_attention_bwd_workspace_bytes(int B, int H, int Hkv, int Sq, int Sk, int D, int dtype) {
  if (attn_shape_ok(B, H, Hkv, Sq, Sk, D, dtype) != CG_OK || B == 0) return 0;
  size_t part = 0;
  if (Sq > 0) {
    const Plan r = row_plan(B, H, Hkv, Sq, Sk, D, dtype, true, true);
    if (r.nsplit > 1) part = (size_t)B * Sq * H * r.nsplit * D * 4;
  }
  if (Sk > 0 && !(Sq > 0 && row_plan(B, H, Hkv, Sq, Sk, D, dtype, true, true).few)) {
    const Plan k = key_plan(B, H, Hkv, Sq, Sk, D, dtype, true);
    const size_t n = (size_t)B * Sk * Hkv * k.nsplit * D * 8;
    if (k.nsplit > 1 && n > part) part = n;
  }
  return up16((size_t)B * H * Sq * 8) + part;
}

extern "C" int cg_attention_bwd(void* dQ, void* dK, void* dV, const void* dO, long long gb, long long gs, long long gh,
                                const void* O, const float* lse2, const void* Q, long long qb, long long qs, long long qh,
                                const void* K, long long kb, long long ks, long long kh, const void* V, long long vb,
                                long long vs, long long vh, const void* words, int B, int H, int Hkv, int Sq, int Sk, int D,
                                float scale, int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return cg_attention_bwd_low(dQ, dK, dV, dO, gb, gs, gh, O, nullptr, lse2, Q, qb, qs, qh, K, kb, ks, kh, V, vb, vs, vh, words, B, H,
                              Hkv, Sq, Sk, D, scale, causal, dtype, workspace, workspace_bytes, stream);
}

extern "C" int cg_attention_bwd_low(void* dQ, void* dK, void* dV, const void* dO, long long gb, long long gs, long long gh,
                                const void* O, const void* Olow, const float* lse2, const void* Q, long long qb, long long qs, long long qh,
                                const void* K, long long kb, long long ks, long long kh, const void* V, long long vb,
                                long long vs, long long vh, const void* words, int B, int H, int Hkv, int Sq, int Sk, int D,
                                float scale, int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const int ok = attn_shape_ok(B, H, Hkv, Sq, Sk, D, dtype);
  if (ok != CG_OK) return ok;
  if (!(scale > 0.f) || scale > 3e38f) return CG_ERR_BAD_ARG;
  if (B == 0 || (Sq == 0 && Sk == 0)) return CG_OK;
  if ((Sq > 0 && (!dQ || !dO || !O || !lse2 || !Q)) || (Sk > 0 && (!dK || !dV || !K || !V)) || (Olow && dtype != CG_BF16))
    return CG_ERR_BAD_ARG;
  const Strides sq{qb, qs, qh}, sk{kb, ks, kh}, sv{vb, vs, vh}, sg{gb, gs, gh};
  if (!operand_ok(Q, sq, B, Sq, H, dtype) || !operand_ok(K, sk, B, Sk, Hkv, dtype) || !operand_ok(V, sv, B, Sk, Hkv, dtype) ||
      !operand_ok(dO, sg, B, Sq, H, dtype) || (((uintptr_t)O | (uintptr_t)Olow | (uintptr_t)dQ | (uintptr_t)dK | (uintptr_t)dV) & 15))
    return CG_ERR_UNSUPPORTED;
  if (workspace_bytes < cg_attention_bwd_workspace_bytes(B, H, Hkv, Sq, Sk, D, dtype) || ((uintptr_t)workspace & 15) ||
      (Sq > 0 && !workspace))
    return CG_ERR_WORKSPACE;
  AttnArgs a{};
  a.q = Q, a.k = K, a.v = V, a.o = O, a.low = Olow, a.dout = dO, a.sq = sq, a.sk = sk, a.sv = sv, a.sdo = sg;
  a.dq = dQ, a.dk = dK, a.dv = dV, a.lse2 = const_cast<float*>(lse2), a.words = (const u64*)words;
  a.B = B, a.H = H, a.Hkv = Hkv, a.Sq = Sq, a.Sk = Sk, a.D = D, a.nw = (Sk + 63) / 64, a.scale = scale, a.causal = causal;
  a.nlse = (float*)workspace, a.ndelta = a.nlse + (size_t)B * H * Sq;
  a.part = (float*)((char*)workspace + up16((size_t)B * H * Sq * 8));
  const Plan pr = row_plan(B, H, Hkv, Sq, Sk, D, dtype, true, words != nullptr), pk = key_plan(B, H, Hkv, Sq, Sk, D, dtype, causal != 0);
  hipStream_t st = (hipStream_t)stream;
  return dtype == CG_F32 ? bwd_run<float>(a, pr, pk, st) : bwd_run<u16>(a, pr, pk, st);
}
