// Dense layer y = act(x W^T + b) + r with its epilogue in the product, and its gradients, in float32 or bf16 storage.
//
//   forward   a = x W^T + b;  y = act(a) + r;  a is kept (z) for the backward pass where act is not the identity
//   backward  da = dy act'(a);  dx = da W;  dW = da^T x;  db = column sums of da     (dr = dy)
//
// The three products are one kernel: C[m][n] = sum_k A(m, k) B(n, k), where an operand lies in memory either along k (x
// and W forward, da for dx) or along its rows (W for dx; da and x for dW).  Both kinds pass through LDS as they lie, by
// LDS-DMA loads, and meet in the fragment reads: 16 bytes of a row, or for an operand along its rows the transposing
// read (bf16: ds_read_b64_tr_b16) and single words (float32).
// bf16: v_mfma_f32_32x32x16_bf16, float32: v_mfma_f32_32x32x2_f32; accumulation, bias, activation and residual in
// float32, one rounding where y (and z) is stored.  bf16 rounds da for its products, which the matrix cores ask for, and z,
// which they do not: the slope at a rounded z is off by up to |z act''(z)| 2^-8, a third of 2^-8 at most, and float32 would be 67 MB more
// written and read at 8192 x 4096, some 27 us of 290.  Large products are bound by the matrix cores, single rows by reading
// the weights.
#include "lds_dma.h"
#include "vec.h"

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;


struct Epi {
  void* Y; long long ldy;
  void* Z; long long ldz;                    // pre-activation (may be NULL)
  const void* bias;
  const void* R; long long ldr;
  int act;
  float slope;
};

struct GemmArgs {
  const void *A, *B;
  long long lda, ldb;
  int M, N, K;
  int tiles_m, tiles_n, nsplit, ksteps;      // ksteps: pipeline steps of one split
  float* part;                               // [nsplit][M][N] where nsplit > 1
  Epi e;
};

constexpr int STEP = 128;                    // bytes of k per pipeline step

template <typename T> struct Op;
template <> struct Op<u16> {
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Op<float> {
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};

// ---- activations ---------------------------------------------------------------------------------------------------
// Branch-free: the epilogue of a large product evaluates them for every element.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(1.44269504088896340736f * x); }

// Distribution function of the normal distribution at a, and bell = exp(-a^2 / 2), which the density needs too.  The tail
// behind |a| is bell t Q(t), t = 1 / (1 + 0.305 |a|); Q was fitted to it by weighted least squares over 0 <= |a| <= 14 until
// its largest relative error was least, 2^-23.3: the result is right to a share of itself however small the tail is, as the
// values and slopes of gelu are that hang on it (2^-21 in float32 arithmetic; an approximation of erf to 1.5e-7 would be off by
// 5e-5 of gelu at -3 and by 1e-2 at -8, and save 2 us of 90 at 8192 x 1024 -> 4096 bf16, forward).  FINE takes what rounding
// a^2 / 2 to the exponent of 2 leaves along (up to 2^-17 of the bell at 13): float32; bf16's own rounding is far above it.
template <bool FINE>
__device__ __forceinline__ float normal_cdf(float a, float& bell) {
  const float x = fminf(fabsf(a), 16.f), t = __builtin_amdgcn_rcpf(fmaf(0.305f, x, 1.f));      // at 16 the tail is 0
  constexpr float C = 0.72134752044448170368f;                                                 // log2(e) / 2
  const float h = x * x, u = C * h;
  bell = __builtin_amdgcn_exp2f(-u);
  if constexpr (FINE) {
    constexpr float C_REST = (float)(0.72134752044448170368 - (double)C);
    const float rest = fmaf(fmaf(x, x, -h), C, fmaf(h, C_REST, fmaf(h, C, -u)));
    bell = fmaf(-0.69314718055994530942f * rest, bell, bell);
  }
  float q = fmaf(0.0366989552f, t, -0.152987361f);
  q = fmaf(q, t, 0.185715318f);
  q = fmaf(q, t, -0.0379754268f);
  q = fmaf(q, t, 0.121020965f);
  q = fmaf(q, t, 0.103421077f);
  q = fmaf(q, t, 0.122466788f);
  q = fmaf(q, t, 0.121639736f);
  const float tail = q * (t * bell);           // of the side away from a
  return a < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float logistic(float a) { return __builtin_amdgcn_rcpf(1.f + exp_fast(-a)); }

template <int VE, bool FINE>
__device__ __forceinline__ void act_value(float* v, int act, float slope) {
  if (act == CG_ACT_LEAKY) {
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = v[i] > 0.f ? v[i] : v[i] * slope;
  } else if (act == CG_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      float bell;
      v[i] *= normal_cdf<FINE>(v[i], bell);
    }
  } else if (act == CG_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] *= logistic(v[i]);
  }
}
// d <- d act'(a)
template <int VE, bool FINE>
__device__ __forceinline__ void act_slope(float* d, const float* a, int act, float slope) {
  if (act == CG_ACT_LEAKY) {
#pragma unroll
    for (int i = 0; i < VE; ++i) d[i] = a[i] > 0.f ? d[i] : d[i] * slope;
  } else if (act == CG_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      float bell;
      const float c = normal_cdf<FINE>(a[i], bell);
      d[i] *= fmaf(a[i] * 0.39894228040143268f, bell, c);
    }
  } else if (act == CG_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float g = logistic(a[i]);
      d[i] *= g * fmaf(a[i], 1.f - g, 1.f);
    }
  }
}

// Elements c .. c + VE - 1 of row m from their float32 sums: bias, activation, residual; c < N.
template <typename T>
__device__ __forceinline__ void finish(const Epi& e, float* v, long long m, int c, int N) {
  constexpr int VE = Vec<T>::N;
  if (e.bias) {
    float b[VE];
    row_load<T>(b, (const T*)e.bias, c, N);
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] += b[i];
  }
  if (e.Z) row_store<T>((T*)e.Z + m * e.ldz, v, c, N);
  act_value<VE, sizeof(T) == 4>(v, e.act, e.slope);
  if (e.R) {
    float r[VE];
    row_load<T>(r, (const T*)e.R + m * e.ldr, c, N);
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] += r[i];
  }
  row_store<T>((T*)e.Y + m * e.ldy, v, c, N);
}

// ---- operand tiles -------------------------------------------------------------------------------------------------
// ROWS x STEP bytes of k.  COL = false: [row][STEP bytes along k]; COL = true: [k][ROWS elements].  16-byte piece p of row r
// sits at slot p ^ swizzle(r): the 16 rows of a fragment read touch all 64 banks, and the four k rows of a
// transposing read lie 64 bytes apart in them.
template <typename T, int ROWS, bool COL, int NWAVES>
struct Operand {
  static constexpr int VE = Vec<T>::N;
  static constexpr int BYTES = ROWS * STEP;
  static constexpr int NDMA = BYTES / (1024 * NWAVES);
  static_assert(NDMA * 1024 * NWAVES == BYTES, "a tile is whole loads of every wave");
  static constexpr int PPR = COL ? ROWS * (int)sizeof(T) / 16 : STEP / 16;
  unsigned off[NDMA];       // byte offset of the piece from the step's base; DMA_OUTSIDE where its row is
  int kk[NDMA];             // its k inside a step

  static __device__ __forceinline__ int swizzle(int r) {
    if (!COL && PPR == 8) return (r >> 1) & 7;
    return PPR == 4 ? (r >> 2) & 3 : PPR == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
  }
  __device__ __forceinline__ void init(long long ld, int row0, int nrows, int wave, int lane) {
#pragma unroll
    for (int j = 0; j < NDMA; ++j) {
      const int slot = (j * NWAVES + wave) * 64 + lane, r = slot / PPR, p = (slot % PPR) ^ swizzle(r);
      kk[j] = COL ? r : p * VE;
      off[j] = (COL ? row0 + p * VE : row0 + r) < nrows ? (unsigned)(r * ld * sizeof(T)) + 16u * p : DMA_OUTSIDE;
    }
  }
  // the next step has kleft k values: what lies behind them is outside from now on
  __device__ __forceinline__ void end(int kleft) {
#pragma unroll
    for (int j = 0; j < NDMA; ++j) off[j] = kk[j] < kleft ? off[j] : DMA_OUTSIDE;
  }
  // base: the tile's first row at the step's first k
  __device__ __forceinline__ void load(char* dst, const T* base, int wave) const {
    const u32x4 rs = dma_rsrc(base);
#pragma unroll
    for (int j = 0; j < NDMA; ++j)
      dma16(rs, dst + (j * NWAVES + wave) * 1024, off[j]);
  }
  // Fragment of rows r0 .. r0 + 31 (lane % 32) and the c-th 32 bytes of k.
  static __device__ __forceinline__ u32x4 frag(const char* t, int r0, int c, int lane) {
    if constexpr (!COL) {
      const int r = lane & 31;
      return *reinterpret_cast<const u32x4*>(t + (r0 + r) * STEP + (((2 * c + (lane >> 5)) ^ swizzle(r)) << 4));
    } else if constexpr (sizeof(T) == 2) {
      const int h = lane >> 5, sub = (lane >> 4) & 1, i = lane & 15;
      const int k = 16 * c + 8 * h + (i >> 2), p = (r0 >> 3) + 2 * sub + ((i & 3) >> 1);
      const char* a0 = t + k * (PPR * 16) + ((p ^ swizzle(k)) << 4) + (i & 1) * 8;
      const char* a1 = t + (k + 4) * (PPR * 16) + ((p ^ swizzle(k + 4)) << 4) + (i & 1) * 8;
      union { struct { s16x4 lo, hi; } h; u32x4 f; } u;
      u.h.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(a0));
      u.h.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(a1));
      return u.f;
    } else {
      const int r = r0 + (lane & 31), k0 = 8 * c + 4 * (lane >> 5);
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = *reinterpret_cast<const float*>(t + (k0 + j) * (PPR * 16) + (((r >> 2) ^ swizzle(k0 + j)) << 4) + (r & 3) * 4);
      return __builtin_bit_cast(u32x4, v);
    }
  }
};

// Consecutive workgroups go to the eight dies in turn: neighbours after this share a die and its L2.
__device__ __forceinline__ int die_order(int id, int total) {
  const int per = total >> 3, rest = total & 7, die = id & 7, at = id >> 3;
  return die < rest ? die * (per + 1) + at : die * per + rest + at;
}

// One BM x BN tile of C (or of one split of k) per workgroup of WM x WN waves: two LDS stages of STEP bytes of k, the loads
// of the next step under the products of this one, fragments read 32 bytes ahead of their products, one barrier a step.
// 4096 x 4096 x 4096 in bf16: 117 us forward, 119 dx, 117 dW, 79 % of the library's product (93 us); on zeros 98 us, so a
// tenth of it is the clock that falls under load.  Other forms of this loop at that size: four stages of 64 bytes with a
// counted wait, 8 waves 122, 4 waves of 128 x 128 119 us (one wave a SIMD, memory instructions spread between the products
// by hand); stages indexed at run time instead of unrolled 120.
template <typename T, int BM, int BN, int WM, int WN, bool ACOL, bool BCOL>
__global__ void __launch_bounds__(64 * WM * WN, 2) linear_gemm_kernel(GemmArgs g) {
#ifdef __HIP_DEVICE_COMPILE__      // the host pass needs the launch stub alone; it drops the stub of some instances over the body
  constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, KE = STEP / (int)sizeof(T), VE = Vec<T>::N;
  typedef Operand<T, BM, ACOL, NW> OA;
  typedef Operand<T, BN, BCOL, NW> OB;
  constexpr int STAGE = OA::BYTES + OB::BYTES;
  constexpr int LDT = 32 * TN + 4;                      // row of a wave's output exchange, float32
  static_assert(NW * 32 * LDT * 4 <= 2 * STAGE, "the output exchange fits the stages");
  __shared__ __align__(16) char smem[2 * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int id = die_order(blockIdx.x, gridDim.x);
  // the splits of a tile on different dies' turns, tiles in groups of eight rows: a die's tiles share their operands
  const int tiles = g.tiles_m * g.tiles_n, split = id / tiles;
  id -= split * tiles;
  const int group = 8 * g.tiles_n, first = id / group * 8, rows = min(8, g.tiles_m - first);
  const int tm = first + id % group % rows, tn = id % group / rows;
  const int row0 = tm * BM, col0 = tn * BN;

  OA oa;
  OB ob;
  oa.init(g.lda, row0, g.M, wave, lane);
  ob.init(g.ldb, col0, g.N, wave, lane);
  const int k0 = split * g.ksteps * KE, n = min(g.ksteps, (g.K - k0 + KE - 1) / KE);
  const T* pa = (const T*)g.A + (ACOL ? (long long)k0 * g.lda + row0 : (long long)row0 * g.lda + k0);
  const T* pb = (const T*)g.B + (BCOL ? (long long)k0 * g.ldb + col0 : (long long)col0 * g.ldb + k0);
  const long long sa = ACOL ? KE * g.lda : KE, sb = BCOL ? KE * g.ldb : KE;
  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  int kleft = min(n * KE, g.K - k0);      // of the step to be issued next
  auto issue = [&](int stage) {
    if (kleft < KE) oa.end(kleft), ob.end(kleft);
    oa.load(smem + stage * STAGE, pa, wave);
    ob.load(smem + stage * STAGE + OA::BYTES, pb, wave);
    pa += sa, pb += sb, kleft -= KE;
  };
  u32x4 fa[2][TM], fb[2][TN];
  auto read = [&](int stage, int c) {
    const char* ta = smem + stage * STAGE;
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[c & 1][i] = OA::frag(ta, wm * TM * 32 + 32 * i, c, lane);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[c & 1][j] = OB::frag(ta + OA::BYTES, wn * TN * 32 + 32 * j, c, lane);
  };
  auto step = [&](int stage) {
    tile_barrier();                    // this step has arrived, and nobody reads the other stage any more
    issue(stage ^ 1);
    read(stage, 0);
#pragma unroll
    for (int c = 0; c < STEP / 32; ++c) {
      __builtin_amdgcn_sched_barrier(0);
      if (c + 1 < STEP / 32) read(stage, c + 1);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = Op<T>::mma(fa[c & 1][i], fb[c & 1][j], acc[i][j]);
    }
  };
  if (n > 0) issue(0);
  for (int s = 0; s < n; s += 2) {     // behind the last step everything is outside: an odd count multiplies zeros once
    step(0);
    step(1);
  }
  tile_barrier();                      // every load has landed and every fragment has been read: the stages are free
  // A wave passes 32 rows x 32 TN columns at a time through its part of LDS, so that they leave as whole 16-byte vectors
  // along the rows.
  float* x = reinterpret_cast<float*>(smem) + wave * 32 * LDT;
  constexpr int VPR = 32 * TN / VE;                     // vectors of a row
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        x[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * LDT + 32 * j + (lane & 31)] = acc[i][j][r];
    // the wave's own stores are visible to it in order; no other wave touches this part
    __builtin_amdgcn_wave_barrier();
#pragma unroll 2
    for (int t = 0; t < 32 * VPR / 64; ++t) {
      const int v = t * 64 + lane, r = v / VPR, c = v % VPR * VE;
      const int m = row0 + wm * TM * 32 + 32 * i + r, cc = col0 + wn * TN * 32 + c;
      float f[VE];
#pragma unroll
      for (int q = 0; q < VE; q += 4) *reinterpret_cast<f32x4*>(f + q) = *reinterpret_cast<const f32x4*>(x + r * LDT + c + q);
      if (m < g.M && cc < g.N) {
        if (g.nsplit > 1) {
          float* p = g.part + ((long long)split * g.M + m) * g.N;
#pragma unroll
          for (int q = 0; q < VE; q += 4) row_store<float>(p, f + q, cc + q, g.N);
        } else {
          finish<T>(g.e, f, m, cc, g.N);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
#endif
}

// The splits of k added in order, then the epilogue.
template <typename T>
__global__ void __launch_bounds__(256) linear_join_kernel(GemmArgs g) {
  constexpr int VE = Vec<T>::N;
  const int vpr = (g.N + VE - 1) / VE;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)g.M * vpr) return;
  const long long m = i / vpr;
  const int c = (int)(i % vpr) * VE;
  float v[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) v[e] = 0.f;
  for (int s = 0; s < g.nsplit; ++s) {
    const float* p = g.part + ((long long)s * g.M + m) * g.N;
    float q[VE];
    side_load<VE, float>(q, p, c, g.N);
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] += q[e];
  }
  finish<T>(g.e, v, m, c, g.N);
}

// Up to four rows of x: a wave per row of W, read once, 64 vectors at a time.
template <typename T, int MR>
__global__ void __launch_bounds__(256) linear_rows_kernel(const T* X, long long ldx, const T* W, long long ldw, int M, int N,
                                                          int K, Epi e) {
  constexpr int VE = Vec<T>::N;
  const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  const T* w = W + (long long)n * ldw;
  float acc[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[m] = 0.f;
#pragma unroll 4
  for (int k = lane * VE; k < K; k += 64 * VE) {
    float a[VE];
    row_load<T>(a, w, k, K);
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      float b[VE];
      if (m < M) {
        row_load<T>(b, X + m * ldx, k, K);
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[m] = fmaf(a[i], b[i], acc[m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[m] = wave_sum(acc[m]);
  if (lane < M) {
    float v = acc[0];
#pragma unroll
    for (int m = 1; m < MR; ++m) v = lane == m ? acc[m] : v;
    if (e.bias) v += Vec<T>::get((const T*)e.bias + n);
    if (e.Z) Vec<T>::put((T*)e.Z + lane * e.ldz + n, v);
    act_value<1, sizeof(T) == 4>(&v, e.act, e.slope);
    if (e.R) v += Vec<T>::get((const T*)e.R + lane * e.ldr + n);
    Vec<T>::put((T*)e.Y + lane * e.ldy + n, v);
  }
}

// dst [rows][ldd] <- src [rows][n], zeros behind column n: an operand whose rows are not whole aligned pieces.
template <typename T>
__global__ void __launch_bounds__(256) linear_pad_kernel(T* dst, int ldd, const T* src, long long lds, long long rows, int n) {
  constexpr int VE = Vec<T>::N;
  const int vpr = ldd / VE;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * vpr) return;
  const int c = (int)(i % vpr) * VE;
  float v[VE];
  row_load<T>(v, src + i / vpr * lds, c, n);
  Vec<T>::store(dst + i / vpr * ldd + c, v);
}

// da = dy act'(z) (dense rows of ldd elements, zeros behind column N; NULL: not wanted) and the column sums of this
// workgroup's rows.  64 vectors of columns x 4 rows at a time.
template <typename T>
__global__ void __launch_bounds__(256) linear_dact_kernel(T* dA, int ldd, float* part, const T* dY, long long lddy,
                                                          const T* Z, long long ldz, int M, int N, int act, float slope) {
  constexpr int VE = Vec<T>::N;
  __shared__ float lds[3][64 * VE];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = (blockIdx.x * 64 + lane) * VE;
  float sum[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) sum[i] = 0.f;
  if (c < N)
    for (long long m = (long long)blockIdx.y * 4 + w; m < M; m += 4ll * gridDim.y) {
      float v[VE];
      row_load<T>(v, dY + m * lddy, c, N);
      if (act != CG_ACT_NONE) {
        float z[VE];
        row_load<T>(z, Z + m * ldz, c, N);
        act_slope<VE, sizeof(T) == 4>(v, z, act, slope);
      }
#pragma unroll
      for (int i = 0; i < VE; ++i) sum[i] += v[i];
      if (dA) Vec<T>::store(dA + m * ldd + c, v);       // behind column N: dy read as 0
    }
  if (!part) return;
  if (w > 0)
#pragma unroll
    for (int i = 0; i < VE; ++i) lds[w - 1][i * 64 + lane] = sum[i];
  __syncthreads();
  if (w == 0 && c < N)
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (c + i < N) part[(long long)blockIdx.y * N + c + i] = sum[i] + lds[0][i * 64 + lane] + lds[1][i * 64 + lane] + lds[2][i * 64 + lane];
}

template <typename T>
__global__ void __launch_bounds__(1024) linear_colsum_kernel(T* db, const float* part, int nb, int N) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, r = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < N)
    for (int i = r; i < nb; i += 16) s += part[(long long)i * N + c];
  lds[r][lane] = s;
  __syncthreads();
  if (r == 0 && c < N) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][lane];
    Vec<T>::put(db + c, s);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
int ve_of(int dtype) { return dtype == CG_BF16 ? 8 : 4; }
int size_of(int dtype) { return dtype == CG_BF16 ? 2 : 4; }
int padded(int n, int ve) { return (n + ve - 1) / ve * ve; }

// Can a matrix with rows of n contiguous elements be read in whole aligned 16-byte pieces?
bool pieces_ok(const void* p, long long ld, long long rows, int n, int dtype) {
  const int ve = ve_of(dtype);
  return ((uintptr_t)p & 15) == 0 && n % ve == 0 && (rows <= 1 || ld % ve == 0);
}

// Tile and splits of a product.  bf16 takes the largest tile that still gives three quarters of the CUs one (the LDS reads
// per product halve with the edge; 4096 x 4096 x 4096: 117 us with 256, 134 with 128, 191 with 64), float32, whose products are
// sixteen times as long, the 128-row tile only where there are enough for even rounds (512 x 2048 x 5000: 93 us with
// 64-row tiles, 98-122 with 128).  What leaves workgroups short of the slots that LDS allows (1, 2, 5 a CU) splits k, as
// long as a split keeps enough steps to pay for the second launch and the partial results.  bf16: 12 steps where CUs
// would stand idle (300 x 1000 x 1000: 7.9 us, in two splits 9.3; 64 x 4096 x 4096: 32 us, in four 14.6), 32 where every CU has a tile
// already (2048 x 2048 x 2048: 29 us, in two splits 35; 4096 x 1024 x 8192: 91 us, in two 81).  float32: 5
// (1000 x 600 x 200: 8.7 us, in two splits 13; 1000 x 200 x 600: 15.9 us, in three 11.8).
enum { TILE_256, TILE_128, TILE_64 };
struct GemmPlan { int kind, tiles_m, tiles_n, nsplit, ksteps; };
GemmPlan gemm_plan(int M, int N, int K, int dtype) {
  GemmPlan p{};
  static const int edge[3] = {256, 128, 64}, slots[3] = {256, 512, 1280};
  auto tiles = [&](int i) { return (long long)((M + edge[i] - 1) / edge[i]) * ((N + edge[i] - 1) / edge[i]); };
  p.kind = dtype == CG_F32 ? (tiles(TILE_128) >= 1024 ? TILE_128 : TILE_64)
           : tiles(TILE_256) >= 192 ? TILE_256 : tiles(TILE_128) >= 192 ? TILE_128 : TILE_64;
  const int ke = STEP / size_of(dtype), steps = (K + ke - 1) / ke, few = dtype == CG_F32 ? 5 : 12;
  p.tiles_m = (M + edge[p.kind] - 1) / edge[p.kind];
  p.tiles_n = (N + edge[p.kind] - 1) / edge[p.kind];
  const long long t = (long long)p.tiles_m * p.tiles_n;
  const int least = dtype == CG_BF16 && t >= 192 ? 32 : few;
  long long n = t == 0 ? 1 : slots[p.kind] / t;
  if (n > 8) n = 8;
  if (n > steps / least) n = steps / least;
  if (n < 1) n = 1;
  p.ksteps = steps ? (int)((steps + n - 1) / n) : 0;
  p.nsplit = steps ? (steps + p.ksteps - 1) / p.ksteps : 1;
  return p;
}
size_t gemm_part_bytes(int M, int N, int K, int dtype) {
  const GemmPlan p = gemm_plan(M, N, K, dtype);
  return p.nsplit > 1 ? up256((size_t)p.nsplit * M * N * 4) : 0;
}

template <typename T, bool ACOL, bool BCOL>
void gemm_run(GemmArgs g, int dtype, float* part, hipStream_t st) {
  const GemmPlan p = gemm_plan(g.M, g.N, g.K, dtype);
  g.tiles_m = p.tiles_m, g.tiles_n = p.tiles_n, g.nsplit = p.nsplit, g.ksteps = p.ksteps, g.part = part;
  const unsigned grid = (unsigned)(p.tiles_m * p.tiles_n * p.nsplit);
  if constexpr (sizeof(T) == 2) {
    if (p.kind == TILE_256) linear_gemm_kernel<T, 256, 256, 2, 4, ACOL, BCOL><<<grid, 512, 0, st>>>(g);
  }
  if (p.kind == TILE_128) linear_gemm_kernel<T, 128, 128, 2, 2, ACOL, BCOL><<<grid, 256, 0, st>>>(g);
  if (p.kind == TILE_64) linear_gemm_kernel<T, 64, 64, 2, 2, ACOL, BCOL><<<grid, 256, 0, st>>>(g);
  if (p.nsplit > 1) {
    const long long v = (long long)g.M * ((g.N + Vec<T>::N - 1) / Vec<T>::N);
    linear_join_kernel<T><<<(unsigned)((v + 255) / 256), 256, 0, st>>>(g);
  }
}

template <typename T>
const T* pad_run(void* dst, const void* src, long long ld, int rows, int n, int ldd, hipStream_t st) {
  // a launch has fewer than 2^32 threads, one for each piece: more rows take several
  const long long vpr = ldd / Vec<T>::N, most = (1ll << 31) / vpr;
  for (long long r = 0; r < rows; r += most) {
    const long long m = rows - r < most ? rows - r : most;
    linear_pad_kernel<T><<<(unsigned)((m * vpr + 255) / 256), 256, 0, st>>>((T*)dst + r * ldd, ldd, (const T*)src + r * ld, ld, m, n);
  }
  return (const T*)dst;
}

constexpr int ROWS_MAX = 4;      // rows of x up to which the weights are read by linear_rows_kernel

int linear_shape_ok(int M, int N, int K, int act, float slope, int dtype) {
  if (M < 0 || N < 1 || K < 1 || (dtype != CG_F32 && dtype != CG_BF16)) return CG_ERR_BAD_ARG;
  if (act < CG_ACT_NONE || act > CG_ACT_SILU || !(slope == slope)) return CG_ERR_BAD_ARG;
  // tiles and vectors are counted in 32 bits, offsets inside a tile too
  if ((long long)M * N >= (1ll << 38) || (long long)M * K >= (1ll << 38) || (long long)N * K >= (1ll << 38) || M > (1 << 30) ||
      N > (1 << 21) || K > (1 << 21))
    return CG_ERR_UNSUPPORTED;
  return CG_OK;
}
// byte offsets of the rows of one tile: 256 rows, or the k rows of a step
bool ld_ok(long long ld, int n, long long rows) { return rows <= 1 || (ld >= n && ld <= (1ll << 21)); }

int dact_rows(int M, int N, int ve) {      // row chunks of linear_dact_kernel
  const int cols = (N + 64 * ve - 1) / (64 * ve);
  int n = (2048 + cols - 1) / cols;
  const int most = (M + 15) / 16;
  if (n > most) n = most;
  return n < 1 ? 1 : (n > 1024 ? 1024 : n);
}

template <typename T>
int fwd_run(const void* X, long long ldx, const void* W, long long ldw, int M, int N, int K, const Epi& e, int dtype,
            char* ws, hipStream_t st) {
  if (M <= ROWS_MAX) {
    const unsigned grid = (N + 3) / 4;
    if (M == 1) linear_rows_kernel<T, 1><<<grid, 256, 0, st>>>((const T*)X, ldx, (const T*)W, ldw, M, N, K, e);
    else linear_rows_kernel<T, ROWS_MAX><<<grid, 256, 0, st>>>((const T*)X, ldx, (const T*)W, ldw, M, N, K, e);
    return cg_launch_status();
  }
  const int kp = padded(K, Vec<T>::N);
  float* part = (float*)ws;
  ws += gemm_part_bytes(M, N, K, dtype);
  GemmArgs g{};
  g.A = X, g.lda = ldx, g.B = W, g.ldb = ldw, g.M = M, g.N = N, g.K = K, g.e = e;
  if (!pieces_ok(X, ldx, M, K, dtype)) {
    g.A = pad_run<T>(ws, X, ldx, M, K, kp, st), g.lda = kp;
    ws += up256((size_t)M * kp * sizeof(T));
  }
  if (!pieces_ok(W, ldw, N, K, dtype)) g.B = pad_run<T>(ws, W, ldw, N, K, kp, st), g.ldb = kp;
  gemm_run<T, false, false>(g, dtype, part, st);
  return cg_launch_status();
}

template <typename T>
int bwd_run(void* dX, long long lddx, void* dW, void* db, const void* dY, long long lddy, const void* Z, long long ldz,
            const void* X, long long ldx, const void* W, long long ldw, int M, int N, int K, int act, float slope, int dtype,
            char* ws, hipStream_t st) {
  constexpr int VE = Vec<T>::N;
  const int kp = padded(K, VE), np = padded(N, VE);
  size_t part_bytes = gemm_part_bytes(M, K, N, dtype);
  if (gemm_part_bytes(N, K, M, dtype) > part_bytes) part_bytes = gemm_part_bytes(N, K, M, dtype);
  float* part = (float*)ws;
  ws += part_bytes;
  float* colpart = (float*)ws;
  const int chunks = dact_rows(M, N, VE);
  ws += up256((size_t)chunks * N * 4);
  const T* da = (const T*)dY;
  long long ldda = lddy;
  const bool product = (dX || dW) && M > 0, own = product && (act != CG_ACT_NONE || !pieces_ok(dY, lddy, M, N, dtype));
  T* buf = own ? (T*)ws : nullptr;
  if (own) {
    ws += up256((size_t)M * np * sizeof(T));
    da = buf, ldda = np;
  }
  if (own || db) {
    linear_dact_kernel<T><<<dim3((N + 64 * VE - 1) / (64 * VE), chunks), 256, 0, st>>>(
        buf, np, db ? colpart : nullptr, (const T*)dY, lddy, (const T*)Z, ldz, M, N, act, slope);
    if (db) linear_colsum_kernel<T><<<(N + 63) / 64, 1024, 0, st>>>((T*)db, colpart, chunks, N);
  }
  if (dX && M > 0) {      // dx (M, K) = da (along N) W (N rows along K)
    GemmArgs g{};
    g.A = da, g.lda = ldda, g.B = W, g.ldb = ldw, g.M = M, g.N = K, g.K = N;
    g.e.Y = dX, g.e.ldy = lddx;
    if (!pieces_ok(W, ldw, N, K, dtype)) {
      g.B = pad_run<T>(ws, W, ldw, N, K, kp, st), g.ldb = kp;
      ws += up256((size_t)N * kp * sizeof(T));
    }
    gemm_run<T, false, true>(g, dtype, part, st);
  }
  if (dW) {               // dW (N, K) = da^T (M rows along N) x (M rows along K)
    GemmArgs g{};
    g.A = da, g.lda = ldda, g.B = X, g.ldb = ldx, g.M = N, g.N = K, g.K = M;
    g.e.Y = dW, g.e.ldy = K;
    if (M > 0 && !pieces_ok(X, ldx, M, K, dtype)) g.B = pad_run<T>(ws, X, ldx, M, K, kp, st), g.ldb = kp;
    gemm_run<T, true, true>(g, dtype, part, st);
  }
  return cg_launch_status();
}

}  // namespace

extern "C" size_t cg_linear_fwd_workspace_bytes(int M, int N, int K, int dtype) {
  if (linear_shape_ok(M, N, K, CG_ACT_NONE, 0.f, dtype) != CG_OK || M <= ROWS_MAX) return 0;
  const size_t kp = padded(K, ve_of(dtype));
  return gemm_part_bytes(M, N, K, dtype) + up256(M * kp * size_of(dtype)) + up256(N * kp * size_of(dtype));
}

extern "C" int cg_linear_fwd(void* Y, long long ldy, void* Z, long long ldz, const void* X, long long ldx, const void* W,
                             long long ldw, const void* bias, const void* R, long long ldr, int M, int N, int K, int act,
                             float slope, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const int ok = linear_shape_ok(M, N, K, act, slope, dtype);
  if (ok != CG_OK) return ok;
  if (M == 0) return CG_OK;
  if (!Y || !X || !W || !ld_ok(ldx, K, M) || !ld_ok(ldw, K, N) || !ld_ok(ldy, N, M) || (Z && !ld_ok(ldz, N, M)) ||
      (R && !ld_ok(ldr, N, M)))
    return CG_ERR_BAD_ARG;
  const size_t need = cg_linear_fwd_workspace_bytes(M, N, K, dtype);
  if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return CG_ERR_WORKSPACE;
  const Epi e{Y, ldy, Z, ldz, bias, R, ldr, act, slope};
  hipStream_t st = (hipStream_t)stream;
  return dtype == CG_F32 ? fwd_run<float>(X, ldx, W, ldw, M, N, K, e, dtype, (char*)workspace, st)
                         : fwd_run<u16>(X, ldx, W, ldw, M, N, K, e, dtype, (char*)workspace, st);
}

extern "C" size_t cg_linear_bwd_workspace_bytes(int M, int N, int K, int dtype) {
  if (linear_shape_ok(M, N, K, CG_ACT_NONE, 0.f, dtype) != CG_OK) return 0;
  const int ve = ve_of(dtype);
  const size_t kp = padded(K, ve), np = padded(N, ve), size = size_of(dtype);
  size_t part = gemm_part_bytes(M, K, N, dtype);
  if (gemm_part_bytes(N, K, M, dtype) > part) part = gemm_part_bytes(N, K, M, dtype);
  return part + up256((size_t)dact_rows(M, N, ve) * N * 4) + up256(M * np * size) + up256(N * kp * size) + up256(M * kp * size);
}

extern "C" int cg_linear_bwd(void* dX, long long lddx, void* dW, void* db, const void* dY, long long lddy, const void* Z,
                             long long ldz, const void* X, long long ldx, const void* W, long long ldw, int M, int N, int K,
                             int act, float slope, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const int ok = linear_shape_ok(M, N, K, act, slope, dtype);
  if (ok != CG_OK) return ok;
  if (!dX && !dW && !db) return CG_ERR_BAD_ARG;
  if (M > 0 && (!dY || (act != CG_ACT_NONE && !Z) || (dX && !W) || (dW && !X))) return CG_ERR_BAD_ARG;
  if (!ld_ok(lddy, N, M) || (act != CG_ACT_NONE && !ld_ok(ldz, N, M)) || (dX && (!ld_ok(lddx, K, M) || !ld_ok(ldw, K, N))) ||
      (dW && !ld_ok(ldx, K, M)))
    return CG_ERR_BAD_ARG;
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < cg_linear_bwd_workspace_bytes(M, N, K, dtype))
    return CG_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  return dtype == CG_F32
             ? bwd_run<float>(dX, lddx, dW, db, dY, lddy, Z, ldz, X, ldx, W, ldw, M, N, K, act, slope, dtype, (char*)workspace, st)
             : bwd_run<u16>(dX, lddx, dW, db, dY, lddy, Z, ldz, X, ldx, W, ldw, M, N, K, act, slope, dtype, (char*)workspace, st);
}
