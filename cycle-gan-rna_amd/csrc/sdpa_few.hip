// Attention of at most 32 rows over many keys: one query against a stored context, a few latent tokens that read all genes
// of a cell, the query heads of a group packed into the rows of one tile.  Bound by reading the keys and values once.
//
// Here the waves of a workgroup share the rows and divide the keys: each wave streams its own 32-key tiles through its own
// part of LDS, waits for its own loads only, and nothing meets at a barrier until the waves' partial results are joined
// through LDS at the end.  (sdpa.hip's kernels, in which the waves share the key tiles and divide the rows, leave three of
// four waves without rows here.)  The backward pass forms both orientations of the score tile from the same fragments, so
// one reading of keys and values gives dq, dk and dv; dk and dv of a tile are complete at once, because all rows are there.
//   one query, 32 heads over 8 of keys and values, 65537 x 128, 4 cells, bf16   forward 193 us, 5.6 TB/s
//   16 rows, 8 heads of 64, 32 cells of 2500 to 5000 keys, bf16                  forward 74 us, backward 114 us (dk and dv
//   written 8 bytes of a row at a time cost another 80)
// Neighbouring workgroups take neighbouring keys of one head (die_order): with the heads of a cell side by side instead
// the latter take 10 us more each.
#include "attn_tile.h"

using namespace attn;

namespace {

// A wave's own tile of 32 rows.
template <typename T, int DP>
struct WaveTile {
  typedef Tile<T, DP> TL;
  static constexpr int BYTES = 32 * TL::RB, NDMA = BYTES / 1024;
  typedef typename TL::template Source<NDMA> Own;
};

// Bits of the existing, visible keys of 32-key tile t.
__device__ __forceinline__ uint32_t bits32(const u64* words, int Sk, int t) {
  const int left = Sk - t * 32;
  uint32_t w = left >= 32 ? ~0u : (left > 0 ? (1u << left) - 1 : 0);
  if (words) w &= (uint32_t)(word_at(words, t >> 1) >> ((t & 1) * 32));
  return w;
}

// A wave's accumulator as [32 rows][DP] float32 in LDS, 16-byte pieces swizzled by the row.
template <int DP>
__device__ __forceinline__ int part_at(int row, int d) { return row * DP + ((((d >> 2) ^ row) & (DP / 4 - 1)) << 2) + (d & 3); }
template <int DP>
__device__ __forceinline__ void part_store(float* p, const f32x16 (&acc)[DP / 32], float mul, int lane) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = acc[dt][4 * g + j] * mul;
      *reinterpret_cast<f32x4*>(p + part_at<DP>(lane & 31, 32 * dt + 8 * g + 4 * (lane >> 5))) = w;
    }
}

template <typename T, int DP, int W>
__global__ void __launch_bounds__(64 * W, 1) attn_few_fwd_kernel(AttnArgs a) {
  typedef Tile<T, DP> TL;
  typedef WaveTile<T, DP> WT;
  constexpr int NL = WT::NDMA;
  __shared__ __align__(16) char smem[W * 2 * WT::BYTES];      // every wave's k, v; at the end its partial result
  __shared__ float stat[W][32][2];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = die_order(blockIdx.x, gridDim.x);
  const int split = id % a.nsplit, unit = id / a.nsplit;
  const int hu = unit % (a.H / a.G), b = unit / (a.H / a.G), kvh = hu * a.G / (a.H / a.Hkv);
  const int nrows = a.Sq * a.G, row = lane & 31, off = a.Sk - a.Sq;
  const bool live = row < nrows;
  const int qi = live ? row / a.G : 0, head = hu * a.G + (live ? row % a.G : 0);
  u32x4 qf[DP / El<T>::CK];
  load_rows<T, DP>(qf, (const T*)a.q + b * a.sq.b + qi * a.sq.s + head * a.sq.h, a.D, live, lane);
  const T* kb = (const T*)a.k + b * a.sk.b + kvh * a.sk.h;
  const T* vb = (const T*)a.v + b * a.sv.b + kvh * a.sv.h;
  const u64* words = a.words ? a.words + (long long)b * a.nw : nullptr;
  char* ks = smem + wave * 2 * WT::BYTES;
  char* vs = ks + WT::BYTES;
  const int end = min((a.Sk + 31) / 32, (split + 1) * a.tiles_per_split);
  const float sl2 = a.scale * LOG2E;
  f32x16 acc[DP / 32];
  clear<DP>(acc);
  float m = -INFINITY, l = 0.f;
  auto next = [&](int t, uint32_t& bits) {      // this wave's next tile with a visible key
    for (bits = 0; t < end && (bits = bits32(words, a.Sk, t)) == 0;) t += W;
    return t;
  };
  const typename WT::Own from_k(1, 0, lane, (unsigned)(a.sk.s * sizeof(T)), a.D);
  const typename WT::Own from_v(1, 0, lane, (unsigned)(a.sv.s * sizeof(T)), a.D);
  auto load_k = [&](int t, uint32_t bits) { from_k.load(ks, 1, 0, lane, kb + (long long)t * 32 * a.sk.s, bits, ~0u); };
  auto load_v = [&](int t, uint32_t bits) { from_v.load(vs, 1, 0, lane, vb + (long long)t * 32 * a.sv.s, bits, ~0u); };
  uint32_t bits, nbits;
  int t = next(split * a.tiles_per_split + wave, bits);
  const int first = t < end ? t * 32 + __builtin_ctz(bits) : INT_MAX;      // this wave's first visible key
  if (t < end) load_k(t, bits), load_v(t, bits);
  while (t < end) {
    lds_wait<NL>();                            // the keys are there, the values under way
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / El<T>::CK; ++c) s = El<T>::mma(TL::frag(ks, 0, c, lane), qf[c], s);
    const int tn = next(t + W, nbits);
    lds_read_wait();
    load_k(min(tn, end), nbits);                 // without a next tile: no bits, zeros arrive, the count of loads holds
    if (bits != ~0u || a.causal) {
      const int reach = a.causal ? qi + off - t * 32 - 4 * half : 32;
      const uint32_t w = bits >> (4 * half);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = 8 * (r >> 2) + (r & 3);
        s[r] = ((w >> key) & 1) && key <= reach ? s[r] : -INFINITY;
      }
    }
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = fmaxf(top, other_half(top));
    if (__any(top * sl2 > (m == -INFINITY ? -INFINITY : m * sl2 + 8.f))) {      // as in sdpa.hip: raised lazily
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
    for (int r = 0; r < 16; ++r) {
      s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl2, base));
      l += s[r];
    }
    lds_wait<NL>();                            // the values are there, the next keys under way
    Second<T, DP>::run(acc, vs, 0, s, lane);
    lds_read_wait();
    load_v(min(tn, end), nbits);
    t = tn, bits = nbits;
  }
  lds_wait<0>();
  l += other_half(l);
  // a row that sees scores of -inf alone has the lowest finite maximum, one that sees no key -inf
  if (l == 0.f && first <= (a.causal ? qi + off : INT_MAX - 1)) m = -FLT_MAX;
  if (half == 0) stat[wave][row][0] = m, stat[wave][row][1] = l;
  __syncthreads();
  // The waves' maxima and sums joined; a wave's result scaled to the common maximum and laid down, then all of them added.
  // A NaN sum (its wave's maximum may be -inf) is carried along.
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) top = fmaxf(top, stat[w][row][0]);
  const float base = top == -INFINITY ? 0.f : top;
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float lw = stat[w][row][1];
    if (lw != 0.f) total = fmaf(lw, stat[w][row][0] == base ? 1.f : __builtin_amdgcn_exp2f((stat[w][row][0] - base) * sl2), total);
  }
  const float inv = total == 0.f ? 0.f : 1.f / total, none = no_weight(top != -INFINITY, a.nsplit);
  const float mine = l == 0.f ? (total == 0.f && none != none ? none : 0.f) : (m == base ? 1.f : __builtin_amdgcn_exp2f((m - base) * sl2)) * inv;
  if (l == 0.f) clear<DP>(acc);
  float* part = reinterpret_cast<float*>(smem);
  part_store<DP>(part + wave * 32 * DP, acc, mine, lane);
  __syncthreads();
  const long long n = (long long)a.B * a.Sq * a.H;
  for (int i = threadIdx.x; i < nrows * (a.D / 4); i += 64 * W) {
    const int r = i / (a.D / 4), d = i % (a.D / 4) * 4;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) o += *reinterpret_cast<const f32x4*>(part + w * 32 * DP + part_at<DP>(r, d));
    const long long at = ((long long)b * a.Sq + r / a.G) * a.H + hu * a.G + r % a.G;
    if (a.nsplit > 1) {
      *reinterpret_cast<f32x4*>(a.part + (split * n + at) * a.D + d) = o;
    } else {
      const float x[4] = {o[0], o[1], o[2], o[3]};
      put4<T>((T*)a.out + at * a.D + d, a.out_low ? (u16*)a.out_low + at * a.D + d : nullptr, x);
    }
  }
  if (wave == 0 && half == 0 && live) {
    const float lse2 = total == 0.f ? none : top * sl2 + __builtin_amdgcn_logf(total);
    if (a.nsplit > 1) a.part_lse[split * n + ((long long)b * a.Sq + qi) * a.H + head] = lse2;
    else if (a.lse2) a.lse2[((long long)b * a.H + head) * a.Sq + qi] = lse2;
  }
}

// One row: 31 of the 32 rows of a tile's products would be nothing, and a wave's tiles follow one another at the latency of
// memory, so here the vector units do the work.  A key's 16-byte pieces lie across DP / 4 (bf16: DP / 8) lanes, a wave
// takes eight (bf16, which unpacks into twice the registers: four) loads of keys and of values at once; every group of lanes
// keeps its own keys' maximum, sum and result, and they meet at the end.  Bound by latency where the context is short (8
// heads, 513 x 64: float32 6.2 us, 17 on the matrix cores, bf16 5.8 and 7.6; 4 cells, 8 heads, 2000 x 64, bf16: 10 and 13),
// else by reading it (4 cells, 8 heads, 65537 x 128: float32 5.1, bf16 5.3 TB/s, 5.4 on the matrix cores).
template <typename T>
__device__ __forceinline__ void widen(float* f, u32x4 v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      f[j] = __builtin_bit_cast(f32x4, v)[j];
    } else {
      const u32x4 lo = v << 16, hi = v & 0xffff0000u;
      f[2 * j] = __builtin_bit_cast(f32x4, lo)[j], f[2 * j + 1] = __builtin_bit_cast(f32x4, hi)[j];
    }
  }
}
template <typename T, int DP>
__global__ void __launch_bounds__(64 * ONE_WAVES, 4) attn_one_kernel(AttnArgs a) {
  constexpr int VE = 16 / sizeof(T), LPK = DP / VE, KPW = 64 / LPK, U = sizeof(T) == 4 ? 8 : 4, BATCH = U * KPW, W = ONE_WAVES;
  static_assert(64 % BATCH == 0, "a batch lies in one mask word: splits begin at whole ones");
  __shared__ __align__(16) float part[W][DP];
  __shared__ float stat[W][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = lane / LPK, d = lane % LPK * VE;
  const int id = die_order(blockIdx.x, gridDim.x), split = id % a.nsplit, unit = id / a.nsplit;
  const int head = unit % a.H, b = unit / a.H, kvh = head / (a.H / a.Hkv);
  float q[VE];
  {
    u32x4 w = {0, 0, 0, 0};
    if (d < a.D) w = *reinterpret_cast<const u32x4*>((const T*)a.q + b * a.sq.b + head * a.sq.h + d);
    widen<T>(q, w);
  }
  const T* kb = (const T*)a.k + b * a.sk.b + kvh * a.sk.h + d;
  const T* vb = (const T*)a.v + b * a.sv.b + kvh * a.sv.h + d;
  const u64* words = a.words ? a.words + (long long)b * a.nw : nullptr;
  const int end = min(a.Sk, (split + 1) * a.tiles_per_split * 32);
  const float sl2 = a.scale * LOG2E;
  float m = -INFINITY, l = 0.f, acc[VE];
#pragma unroll
  for (int j = 0; j < VE; ++j) acc[j] = 0.f;
  for (int k0 = split * a.tiles_per_split * 32 + wave * BATCH; k0 < end; k0 += W * BATCH) {
    u64 bits = end - k0 >= 64 ? ~0ull : (1ull << (end - k0)) - 1;
    if (words) bits &= word_at(words, k0 >> 6) >> (k0 & 63);
    u32x4 k[U], v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long key = k0 + u * KPW + slot;
      k[u] = v[u] = u32x4{0, 0, 0, 0};                                  // what is not read counts as zeros
      if (d < a.D && ((bits >> (u * KPW + slot)) & 1)) {
        k[u] = *reinterpret_cast<const u32x4*>(kb + key * a.sk.s);
        v[u] = *reinterpret_cast<const u32x4*>(vb + key * a.sv.s);
      }
    }
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[VE];
      widen<T>(x, k[u]);
      s[u] = q[0] * x[0];
#pragma unroll
      for (int j = 1; j < VE; ++j) s[u] = fmaf(q[j], x[j], s[u]);
    }
#pragma unroll
    for (int o = 1; o < LPK; o <<= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) s[u] += __shfl_xor(s[u], o, 64);
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool sees = (bits >> (u * KPW + slot)) & 1;
      if (!sees) s[u] = -INFINITY;
      mn = fmaxf(mn, sees ? fmaxf(s[u], -FLT_MAX) : s[u]);      // keys that are seen: a finite maximum at the least
    }
    const float base = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f((m - base) * sl2);
    l *= f;
#pragma unroll
    for (int j = 0; j < VE; ++j) acc[j] *= f;
    m = mn;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float p = __builtin_amdgcn_exp2f((s[u] - base) * sl2);
      float x[VE];
      widen<T>(x, v[u]);
      l += p;
#pragma unroll
      for (int j = 0; j < VE; ++j) acc[j] = fmaf(p, x[j], acc[j]);
    }
  }
  // the groups of lanes, then the waves; a NaN sum, whose maximum may be -inf, is carried along
  float top = m;
#pragma unroll
  for (int o = LPK; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  float base = top == -INFINITY ? 0.f : top, f = __builtin_amdgcn_exp2f((m - base) * sl2);
  l *= f;
#pragma unroll
  for (int j = 0; j < VE; ++j) acc[j] *= f;
#pragma unroll
  for (int o = LPK; o < 64; o <<= 1) {
    l += __shfl_xor(l, o, 64);
#pragma unroll
    for (int j = 0; j < VE; ++j) acc[j] += __shfl_xor(acc[j], o, 64);
  }
  if (slot == 0)
#pragma unroll
    for (int j = 0; j < VE; ++j) part[wave][d + j] = acc[j];
  if (lane == 0) stat[wave][0] = top, stat[wave][1] = l;
  __syncthreads();
  if (threadIdx.x >= DP) return;
  top = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) top = fmaxf(top, stat[w][0]);
  base = top == -INFINITY ? 0.f : top;
  float total = 0.f, o = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    f = __builtin_amdgcn_exp2f((stat[w][0] - base) * sl2);
    total = fmaf(f, stat[w][1], total);
    o = fmaf(f, part[w][threadIdx.x], o);
  }
  const float none = no_weight(top != -INFINITY, a.nsplit);
  o = total == 0.f ? (none != none ? none : 0.f) : o * (1.f / total);
  const float lse2 = total == 0.f ? none : top * sl2 + __builtin_amdgcn_logf(total);
  const long long n = (long long)a.B * a.H, at = (long long)b * a.H + head, dd = threadIdx.x;
  if (dd < a.D) {
    if (a.nsplit > 1) a.part[(split * n + at) * a.D + dd] = o;
    else if constexpr (sizeof(T) == 4) ((float*)a.out)[at * a.D + dd] = o;
    else {
      const u16 w = f2bf(o);
      ((u16*)a.out)[at * a.D + dd] = w;
      const float rest = o - bf2f(w);
      if (a.out_low) ((u16*)a.out_low)[at * a.D + dd] = f2bf(fabsf(rest) <= FLT_MAX ? rest : 0.f);
    }
  }
  if (dd == 0) {
    if (a.nsplit > 1) a.part_lse[split * n + at] = lse2;
    else if (a.lse2) a.lse2[at] = lse2;
  }
}

// All of a group's heads are in the rows (G = H / Hkv): dk and dv are whole.
template <typename T, int DP, int W>
__global__ void __launch_bounds__(64 * W, 1) attn_few_bwd_kernel(AttnArgs a) {
  typedef Tile<T, DP> TL;
  typedef WaveTile<T, DP> WT;
  constexpr int CH = DP / El<T>::CK;
  __shared__ __align__(16) char smem[W * 4 * WT::BYTES];      // every wave's k, v; k, v; at the end its dq
  __shared__ __align__(16) char rows_[2 * WT::BYTES];         // q, do
  __shared__ __align__(16) float stats[2][32];                // nlse, ndelta
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = die_order(blockIdx.x, gridDim.x);
  const int split = id % a.nsplit, unit = id / a.nsplit;
  const int kvh = unit % a.Hkv, b = unit / a.Hkv;
  const int nrows = a.Sq * a.G, row = lane & 31, off = a.Sk - a.Sq;
  const bool live = row < nrows;
  const int qi = live ? row / a.G : 0, head = kvh * a.G + (live ? row % a.G : 0);
  const long long stat = ((long long)b * a.H + head) * a.Sq + qi;
  float base = live ? a.nlse[stat] : -INFINITY;
  const bool some = base != -INFINITY;       // a row that sees nothing takes no part, whatever arrives in do
  float nd = some ? a.ndelta[stat] : 0.f;
  settle(base), settle(nd);
  u32x4 qf[CH], gf[CH];
  load_rows<T, DP>(qf, (const T*)a.q + b * a.sq.b + qi * a.sq.s + head * a.sq.h, a.D, some, lane);
  load_rows<T, DP>(gf, (const T*)a.dout + b * a.sdo.b + qi * a.sdo.s + head * a.sdo.h, a.D, some, lane);
  char* qs = rows_;
  char* gs = rows_ + WT::BYTES;
  if (wave == 0) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = row * TL::RB + (((2 * c + half) ^ TL::swizzle(row)) << 4);
      *reinterpret_cast<u32x4*>(qs + at) = qf[c];
      *reinterpret_cast<u32x4*>(gs + at) = gf[c];
    }
    if (half == 0) stats[0][row] = some ? base : 0.f, stats[1][row] = nd;
  }
  __syncthreads();
  const uint32_t taking = (uint32_t)__ballot(some);      // the rows that take part, in every wave
  const T* kb = (const T*)a.k + b * a.sk.b + kvh * a.sk.h;
  const T* vb = (const T*)a.v + b * a.sv.b + kvh * a.sv.h;
  const u64* words = a.words ? a.words + (long long)b * a.nw : nullptr;
  const int end = min((a.Sk + 31) / 32, (split + 1) * a.tiles_per_split);
  const float sl2 = a.scale * LOG2E;
  f32x16 dq[DP / 32];
  clear<DP>(dq);
  const typename WT::Own from_k(1, 0, lane, (unsigned)(a.sk.s * sizeof(T)), a.D);
  const typename WT::Own from_v(1, 0, lane, (unsigned)(a.sv.s * sizeof(T)), a.D);
  auto load = [&](int t, uint32_t bits, int buf) {
    char* ks = smem + (wave * 2 + buf) * 2 * WT::BYTES;
    from_k.load(ks, 1, 0, lane, kb + (long long)t * 32 * a.sk.s, bits, ~0u);
    from_v.load(ks + WT::BYTES, 1, 0, lane, vb + (long long)t * 32 * a.sv.s, bits, ~0u);
  };
  int t = split * a.tiles_per_split + wave, buf = 0;
  uint32_t bits = t < end ? bits32(words, a.Sk, t) : 0;
  if (t < end) load(t, bits, 0);
  lds_wait<0>();
  for (; t < end; t += W, buf ^= 1) {
    const char* ks = smem + (wave * 2 + buf) * 2 * WT::BYTES;
    const char* vs = ks + WT::BYTES;
    lds_read_wait();                                // the other buffer's last reads
    const uint32_t nbits = t + W < end ? bits32(words, a.Sk, t + W) : 0;
    if (t + W < end) load(t + W, nbits, buf ^ 1);
    const int key0 = t * 32;
    const bool masked = bits != ~0u || a.causal;
    u32x4 kf[CH], vf[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) kf[c] = TL::frag(ks, 0, c, lane), vf[c] = TL::frag(vs, 0, c, lane);
    f32x16 s, dp;
    // keys down the registers, the lane's row: dq
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f, dp[r] = nd;
#pragma unroll
    for (int c = 0; c < CH; ++c) s = El<T>::mma(kf[c], qf[c], s), dp = El<T>::mma(vf[c], gf[c], dp);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl2, base)) * dp[r];
    if (masked) {
      const int reach = a.causal ? qi + off - key0 - 4 * half : 32;
      const uint32_t w = bits >> (4 * half);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = 8 * (r >> 2) + (r & 3);
        s[r] = ((w >> key) & 1) && key <= reach ? s[r] : 0.f;
      }
    }
    Second<T, DP>::run(dq, ks, 0, s, lane);
    // rows down the registers, the lane's key: dv, dk
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 de = *reinterpret_cast<const f32x4*>(&stats[1][8 * g + 4 * half]);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[4 * g + j] = 0.f, dp[4 * g + j] = de[j];
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) s = El<T>::mma(qf[c], kf[c], s), dp = El<T>::mma(gf[c], vf[c], dp);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 ls = *reinterpret_cast<const f32x4*>(&stats[0][8 * g + 4 * half]);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[4 * g + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + j], sl2, ls[j]));
    }
    if (taking != ~0u) {      // rows of zeros: 0 times an infinity at a visible key is none
      const uint32_t w = taking >> (4 * half);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!((w >> (8 * (r >> 2) + (r & 3))) & 1)) s[r] = dp[r] = 0.f;
    }
    if (a.causal) {
      // rows from here on see this lane's key; all of them where it is negative, which times G may pass 32 bits
      const int from = max(key0 + row - off, 0) * a.G - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + (r & 3) < from) s[r] = 0.f;
    }
    f32x16 dv[DP / 32], dk[DP / 32];
    clear<DP>(dv), clear<DP>(dk);
    Second<T, DP>::run(dv, gs, 0, s, lane);
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] *= s[r];
    Second<T, DP>::run(dk, qs, 0, dp, lane);
    if (!((bits >> row) & 1)) clear<DP>(dv), clear<DP>(dk);      // masked: dropped, not multiplied
    const long long at = (((long long)b * a.Sk + key0) * a.Hkv + kvh) * a.D, pitch = (long long)a.Hkv * a.D;
    lds_wait<0>();                             // the next keys and values; the stores then have the next tile's time
    store_tile<T, DP>(smem + (wave * 2 + buf) * 2 * WT::BYTES, (T*)a.dk + at, pitch, a.Sk - key0, dk, a.scale, a.D, lane);
    store_tile<T, DP>(smem + ((wave * 2 + buf) * 2 + 1) * WT::BYTES, (T*)a.dv + at, pitch, a.Sk - key0, dv, 1.f, a.D, lane);
    bits = nbits;
  }
  if (!some) clear<DP>(dq);
  float* part = reinterpret_cast<float*>(smem);
  __syncthreads();
  part_store<DP>(part + wave * 32 * DP, dq, a.scale, lane);
  __syncthreads();
  const long long n = (long long)a.B * a.Sq * a.H;
  for (int i = threadIdx.x; i < nrows * (a.D / 4); i += 64 * W) {
    const int r = i / (a.D / 4), d = i % (a.D / 4) * 4;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) o += *reinterpret_cast<const f32x4*>(part + w * 32 * DP + part_at<DP>(r, d));
    const long long at = ((long long)b * a.Sq + r / a.G) * a.H + kvh * a.G + r % a.G;
    if (a.nsplit > 1) {
      *reinterpret_cast<f32x4*>(a.part + (split * n + at) * a.D + d) = o;
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4*>((float*)a.dq + at * a.D + d) = o;
    } else {
      *reinterpret_cast<u32x2*>((u16*)a.dq + at * a.D + d) = u32x2{pack2(o[0], o[1]), pack2(o[2], o[3])};
    }
  }
}

template <typename T, int DP>
void fwd_launch(const AttnArgs& a, hipStream_t st) {
  if (a.Sq * a.G == 1) {
    attn_one_kernel<T, DP><<<(unsigned)((long long)a.B * a.H * a.nsplit), 64 * ONE_WAVES, 0, st>>>(a);
    return;
  }
  constexpr int W = few_waves<T, DP>();
  attn_few_fwd_kernel<T, DP, W><<<(unsigned)((long long)a.B * (a.H / a.G) * a.nsplit), 64 * W, 0, st>>>(a);
}
template <typename T, int DP>
void bwd_launch(const AttnArgs& a, hipStream_t st) {
  constexpr int W = few_bwd_waves<T, DP>();
  attn_few_bwd_kernel<T, DP, W><<<(unsigned)((long long)a.B * a.Hkv * a.nsplit), 64 * W, 0, st>>>(a);
}

}  // namespace

int attn::few_fwd(const AttnArgs& a, int dtype, hipStream_t st) {
  if (dtype == CG_F32) a.D <= 32 ? fwd_launch<float, 32>(a, st) : a.D <= 64 ? fwd_launch<float, 64>(a, st) : fwd_launch<float, 128>(a, st);
  else a.D <= 32 ? fwd_launch<u16, 32>(a, st) : a.D <= 64 ? fwd_launch<u16, 64>(a, st) : fwd_launch<u16, 128>(a, st);
  return cg_launch_status();
}
int attn::few_bwd(const AttnArgs& a, int dtype, hipStream_t st) {
  if (dtype == CG_F32) a.D <= 32 ? bwd_launch<float, 32>(a, st) : bwd_launch<float, 64>(a, st);      // wider: see row_plan
  else a.D <= 32 ? bwd_launch<u16, 32>(a, st) : a.D <= 64 ? bwd_launch<u16, 64>(a, st) : bwd_launch<u16, 128>(a, st);
  return cg_launch_status();
}
