// LayerNorm over the last axis of token rows, with the residual sum in front of it: forward and backward.
//
//   s = x + r                      (r may be absent)
//   y = (s - mean) rstd w + b      mean, var over the N columns of a row, rstd = 1 / sqrt(var + eps)
//   g = dy w;  xhat = (s - mean) rstd
//   dx = rstd (g - mean(g) - xhat mean(g xhat)) + ds        (also the gradient of r)
//   dw = sum over rows of dy xhat;  db = sum over rows of dy
//
// Bound by memory from 256 float32 columns on (2^20 rows: 5.3 TB/s), every tensor passes once; below, by the latency of a row,
// which has a wave to itself (64 columns 1.8 TB/s, 16 0.5; bf16 256 2.7, 16 0.2).  A row lives in the registers of its group of threads (64, 256 or 1024,
// by its length), so the mean and then the sum of squared deviations from it are two reductions over registers (no
// cancellation of large squares).  The backward pass keeps the groups resident and walks the rows with a stride: a
// thread owns the same columns in every row, so the column sums dw and db stay in its registers, leave as one
// partial row per workgroup and are added in workgroup order by a second launch (no atomics: the same bits every time).
// Statistics and sums are float32; y, s, dx, dw, db are rounded once, when they are stored.  y is that of the unrounded
// sum; the backward pass takes s as it was stored or forms it from x and r again (bf16: the stored sum is up to 2^-8
// off, which dw would show).
#include "vec.h"

namespace {

constexpr int LN_MAX_COLS = 1 << 30;     // columns are counted in 32 bits, up to 8192 past the last
constexpr int LN_MAX_BLOCKS = 1024;      // workgroups of the backward pass: rows of partial column sums

struct LnFwd {
  void* Y; long long ldy;
  void* S; long long lds;
  const void* X; long long ldx;
  const void* R; long long ldr;
  const void *w, *b;
  float eps;
  float *mean, *rstd;
  int M, N;
};

struct LnBwd {
  void* dX; long long lddx;
  const void* dY; long long lddy;
  const void* dS; long long ldds;
  const void* S; long long lds;
  const void* R; long long ldr;
  const void* w;
  const float *mean, *rstd;
  float* part;             // [gridDim.x][2][N]: dw, db (NULL: not wanted)
  int M, N;
};

// Sums of NS values over a group of GROUP threads (a wave, or the whole workgroup); every thread gets them.  Two calls
// in a row use different `lds`: a thread that reaches the barrier of the second has read the sums of the first.
template <int GROUP, int NS>
__device__ __forceinline__ void group_sum(float* v, float* lds) {
#pragma unroll
  for (int s = 0; s < NS; ++s) v[s] = wave_sum(v[s]);
  if constexpr (GROUP > 64) {
    constexpr int W = GROUP / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0)
#pragma unroll
      for (int s = 0; s < NS; ++s) lds[s * W + wave] = v[s];
    __syncthreads();
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) t += lds[s * W + i];
      v[s] = t;
    }
  }
}

template <typename T, typename TW, int GROUP, int NV>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP) ln_fwd_kernel(LnFwd a) {
  constexpr int VE = Vec<T>::N, PER = GROUP < 256 ? 256 / GROUP : 1;
  __shared__ float lds[GROUP / 64 * 2];
  const int t = GROUP < 256 ? threadIdx.x % GROUP : threadIdx.x;
  const long long row = (long long)blockIdx.x * PER + (PER > 1 ? threadIdx.x / GROUP : 0);
  if (PER > 1 && row >= a.M) return;       // whole waves, and groups of one wave meet at no barrier
  const int N = a.N;
  float s[NV][VE];
  const T* x = (const T*)a.X + row * a.ldx;
#pragma unroll
  for (int j = 0; j < NV; ++j) row_load<T>(s[j], x, (j * GROUP + t) * VE, N);
  if (a.R) {
    const T* r = (const T*)a.R + row * a.ldr;
#pragma unroll
    for (int j = 0; j < NV; ++j) row_add<T>(s[j], r, (j * GROUP + t) * VE, N);
  }
  if (a.S) {
    T* so = (T*)a.S + row * a.lds;
#pragma unroll
    for (int j = 0; j < NV; ++j) row_store<T>(so, s[j], (j * GROUP + t) * VE, N);
  }
  float sum[1] = {0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VE; ++e) sum[0] += s[j][e];
  group_sum<GROUP, 1>(sum, lds);
  const float mean = sum[0] / (float)N;
  float sq[1] = {0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      s[j][e] -= mean;
      if ((j * GROUP + t) * VE + e < N) sq[0] = fmaf(s[j][e], s[j][e], sq[0]);
    }
  group_sum<GROUP, 1>(sq, lds + (GROUP > 64 ? GROUP / 64 : 0));
  const float rstd = 1.f / sqrtf(sq[0] / (float)N + a.eps);
  if (t == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  T* y = (T*)a.Y + row * a.ldy;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * GROUP + t) * VE;
    if (c >= N) break;
    float w[VE], b[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = 1.f, b[e] = 0.f;
    if (a.w) side_load<VE, TW>(w, (const TW*)a.w, c, N);
    if (a.b) side_load<VE, TW>(b, (const TW*)a.b, c, N);
#pragma unroll
    for (int e = 0; e < VE; ++e) s[j][e] = fmaf(s[j][e] * rstd, w[e], b[e]);
    row_store<T>(y, s[j], c, N);
  }
}

// COLS: with the column sums (four float32 values per element in registers); without, dX alone (two).
template <typename T, typename TW, int GROUP, int NV, bool COLS>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP) ln_bwd_kernel(LnBwd a) {
  constexpr int VE = Vec<T>::N, PER = GROUP < 256 ? 256 / GROUP : 1;
  __shared__ float lds[GROUP > 64 ? GROUP / 64 * 4 : 1];
  const int t = GROUP < 256 ? threadIdx.x % GROUP : threadIdx.x;
  const int grp = PER > 1 ? threadIdx.x / GROUP : 0;
  const int N = a.N;
  float dw[NV][VE], db[NV][VE];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VE; ++e) dw[j][e] = db[j][e] = 0.f;
  int parity = 0;
  for (long long row = (long long)blockIdx.x * PER + grp; row < a.M; row += (long long)gridDim.x * PER) {
    const T* so = (const T*)a.S + row * a.lds;
    const T* dy = (const T*)a.dY + row * a.lddy;
    float x[NV][VE], g[NV][VE];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      row_load<T>(x[j], so, (j * GROUP + t) * VE, N);
      row_load<T>(g[j], dy, (j * GROUP + t) * VE, N);
    }
    if (a.R) {
      const T* r = (const T*)a.R + row * a.ldr;
#pragma unroll
      for (int j = 0; j < NV; ++j) row_add<T>(x[j], r, (j * GROUP + t) * VE, N);
    }
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * GROUP + t) * VE;
      float w[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) w[e] = 1.f;
      if (a.w) side_load<VE, TW>(w, (const TW*)a.w, c, N);
#pragma unroll
      for (int e = 0; e < VE; ++e) {      // past the end of the row g is 0: x counts for nothing there
        x[j][e] = (x[j][e] - mean) * rstd;
        if constexpr (COLS) {
          db[j][e] += g[j][e];
          dw[j][e] = fmaf(g[j][e], x[j][e], dw[j][e]);
        }
        g[j][e] *= w[e];
        sum[0] += g[j][e];
        sum[1] = fmaf(g[j][e], x[j][e], sum[1]);
      }
    }
    group_sum<GROUP, 2>(sum, lds + (GROUP > 64 ? parity * (GROUP / 64 * 2) : 0));
    parity ^= 1;
    const float m1 = sum[0] / (float)N, m2 = sum[1] / (float)N;
    if (a.dX) {
      T* dx = (T*)a.dX + row * a.lddx;
      const T* ds = a.dS ? (const T*)a.dS + row * a.ldds : nullptr;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * GROUP + t) * VE;
        if (c >= N) break;
        float d[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) d[e] = 0.f;
        if (ds) row_load<T>(d, ds, c, N);
#pragma unroll
        for (int e = 0; e < VE; ++e) d[e] = fmaf(rstd, g[j][e] - m1 - x[j][e] * m2, d[e]);
        row_store<T>(dx, d, c, N);
      }
    }
  }
  if (!COLS || !a.part) return;
  float* p = a.part + (long long)blockIdx.x * 2 * N;
  if constexpr (PER == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const int c = (j * GROUP + t) * VE + e;
        if (c < N) {
          p[c] = dw[j][e];
          p[N + c] = db[j][e];
        }
      }
  } else {      // the workgroup's groups, in order
    __shared__ float acc[PER > 1 ? 2 * GROUP * NV * VE : 1];
    for (int k = 0; k < PER; ++k) {
      if (grp == k)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const int c = (j * VE + e) * GROUP + t;       // bank-conflict-free order; put right when it leaves
            acc[c] = k ? acc[c] + dw[j][e] : dw[j][e];
            acc[GROUP * NV * VE + c] = k ? acc[GROUP * NV * VE + c] + db[j][e] : db[j][e];
          }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < N; i += 256) {
      const int v = i / VE, e = i % VE, j = v / GROUP, tt = v % GROUP, c = (j * VE + e) * GROUP + tt;
      p[i] = acc[c];
      p[N + i] = acc[GROUP * NV * VE + c];
    }
  }
}

// Rows longer than a workgroup's registers: the row is read once per pass (the second and third reads come from the
// caches).
template <typename T, typename TW>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(LnFwd a) {
  constexpr int VE = Vec<T>::N;
  __shared__ float lds[32];
  const long long row = blockIdx.x;
  const int N = a.N;
  const T* x = (const T*)a.X + row * a.ldx;
  const T* r = a.R ? (const T*)a.R + row * a.ldr : nullptr;
  auto load = [&](float* s, int c) {
    row_load<T>(s, x, c, N);
    if (r) row_add<T>(s, r, c, N);
  };
  float sum[1] = {0.f};
  for (int c = threadIdx.x * VE; c < N; c += 1024 * VE) {
    float s[VE];
    load(s, c);
    if (a.S) row_store<T>((T*)a.S + row * a.lds, s, c, N);
#pragma unroll
    for (int e = 0; e < VE; ++e) sum[0] += s[e];
  }
  group_sum<1024, 1>(sum, lds);
  const float mean = sum[0] / (float)N;
  float sq[1] = {0.f};
  for (int c = threadIdx.x * VE; c < N; c += 1024 * VE) {
    float s[VE];
    load(s, c);
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (c + e < N) sq[0] = fmaf(s[e] - mean, s[e] - mean, sq[0]);
  }
  group_sum<1024, 1>(sq, lds + 16);
  const float rstd = 1.f / sqrtf(sq[0] / (float)N + a.eps);
  if (threadIdx.x == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  for (int c = threadIdx.x * VE; c < N; c += 1024 * VE) {
    float s[VE], w[VE], b[VE];
    load(s, c);
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = 1.f, b[e] = 0.f;
    if (a.w) side_load<VE, TW>(w, (const TW*)a.w, c, N);
    if (a.b) side_load<VE, TW>(b, (const TW*)a.b, c, N);
#pragma unroll
    for (int e = 0; e < VE; ++e) s[e] = fmaf((s[e] - mean) * rstd, w[e], b[e]);
    row_store<T>((T*)a.Y + row * a.ldy, s, c, N);
  }
}

template <typename T, typename TW>
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(LnBwd a) {
  constexpr int VE = Vec<T>::N;
  __shared__ float lds[32];
  const long long row = blockIdx.x;
  const int N = a.N;
  const T* so = (const T*)a.S + row * a.lds;
  const T* dy = (const T*)a.dY + row * a.lddy;
  const float mean = a.mean[row], rstd = a.rstd[row];
  auto load = [&](float* x, float* g, int c) {
    float w[VE];
    row_load<T>(x, so, c, N);
    if (a.R) row_add<T>(x, (const T*)a.R + row * a.ldr, c, N);
    row_load<T>(g, dy, c, N);
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = 1.f;
    if (a.w) side_load<VE, TW>(w, (const TW*)a.w, c, N);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      x[e] = (x[e] - mean) * rstd;
      g[e] *= w[e];
    }
  };
  float sum[2] = {0.f, 0.f};
  for (int c = threadIdx.x * VE; c < N; c += 1024 * VE) {
    float x[VE], g[VE];
    load(x, g, c);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      sum[0] += g[e];
      sum[1] = fmaf(g[e], x[e], sum[1]);
    }
  }
  group_sum<1024, 2>(sum, lds);
  const float m1 = sum[0] / (float)N, m2 = sum[1] / (float)N;
  for (int c = threadIdx.x * VE; c < N; c += 1024 * VE) {
    float x[VE], g[VE], d[VE];
    load(x, g, c);
#pragma unroll
    for (int e = 0; e < VE; ++e) d[e] = 0.f;
    if (a.dS) row_load<T>(d, (const T*)a.dS + row * a.ldds, c, N);
#pragma unroll
    for (int e = 0; e < VE; ++e) d[e] = fmaf(rstd, g[e] - m1 - x[e] * m2, d[e]);
    row_store<T>((T*)a.dX + row * a.lddx, d, c, N);
  }
}

// Partial column sums of rows too long for COLS: blockIdx.x takes 256 vectors of columns, blockIdx.y every
// gridDim.y-th row.
template <typename T>
__global__ void __launch_bounds__(256) ln_cols_kernel(LnBwd a) {
  constexpr int VE = Vec<T>::N;
  const int N = a.N;
  const long long c = ((long long)blockIdx.x * 256 + threadIdx.x) * VE;
  if (c >= N) return;
  float dw[VE], db[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) dw[e] = db[e] = 0.f;
  for (long long row = blockIdx.y; row < a.M; row += gridDim.y) {
    float x[VE], g[VE];
    row_load<T>(x, (const T*)a.S + row * a.lds, (int)c, N);
    if (a.R) row_add<T>(x, (const T*)a.R + row * a.ldr, (int)c, N);
    row_load<T>(g, (const T*)a.dY + row * a.lddy, (int)c, N);
    const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      db[e] += g[e];
      dw[e] = fmaf(g[e], (x[e] - mean) * rstd, dw[e]);
    }
  }
  float* p = a.part + (long long)blockIdx.y * 2 * N;
#pragma unroll
  for (int e = 0; e < VE; ++e)
    if (c + e < N) {
      p[c + e] = dw[e];
      p[N + c + e] = db[e];
    }
}

// dw, db <- the sums of nb partial rows.  A workgroup takes 16 columns (a row's 64 bytes): its 16 (up to 256 rows) or
// 64 threads of a column add every 16th or 64th row each, then their sums in order.  Bound by latency, so the columns
// are spread over many workgroups and eight rows are asked for at once (1024 rows of 2 x 1024: 5 us, 20 with 64 columns
// a workgroup and one row at a time).
template <typename TW>
__global__ void __launch_bounds__(1024) ln_cols_reduce_kernel(TW* dw, TW* db, const float* part, int nb, int N) {
  __shared__ float lds[16][64 + 1];
  const int col = threadIdx.x & 15, r = threadIdx.x >> 4, side = blockDim.x >> 4;
  const long long c = (long long)blockIdx.x * 16 + col;
  const float* p = part + (blockIdx.y ? N : 0) + c;
  float s = 0.f;
  if (c < N)
    for (int i = r; i < nb; i += 8 * side) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i + side * k < nb ? p[((long long)i + side * k) * 2 * N] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
  lds[col][r] = s;
  __syncthreads();
  if (threadIdx.x < 16 && c < N) {
    s = 0.f;
    for (int i = 0; i < side; ++i) s += lds[col][i];
    TW* out = blockIdx.y ? db : dw;
    if (out) Vec<TW>::put(out + c, s);
  }
}

// The group of threads that holds a row of N columns in registers, and its vectors per thread; group 0: too long.
// A wave per row while the row fits 32 elements a lane (backward with column sums: 16), then a workgroup of 256 at up to
// four vectors a thread, then 1024 threads at up to 32 elements (24 for dX).  Backward with column sums stops at
// 12 (float32) and 8 (bf16) elements of 1024 threads, where the compiler starts to spill: longer rows take two launches, the column
// sums and dX apart, and read their operands twice.
struct LnPlan { int group, nv; };
enum { LN_FWD, LN_DX, LN_DX_COLS };
LnPlan ln_plan(int N, int ve, int kind) {
  const int v = (N + ve - 1) / ve;
  const int wave_nv = (kind == LN_DX_COLS ? 16 : 32) / ve;
  if (v <= 64 * wave_nv) return {64, (v + 63) / 64};
  const int mid_nv = kind == LN_DX_COLS ? 16 / ve : 4;
  if (v <= 256 * mid_nv) return {256, (v + 255) / 256};
  const int top_nv = kind == LN_DX_COLS ? (ve == 4 ? 3 : 1) : (kind == LN_DX ? 24 : 32) / ve;
  if (v <= 1024 * top_nv) return {1024, (v + 1023) / 1024};
  return {0, 0};
}

int ln_bwd_blocks(int M, int N, int ve) {
  const LnPlan p = ln_plan(N, ve, LN_DX_COLS);
  // enough workgroups to fill the chip, few enough that the partial sums stay small beside the rows
  const int per = p.group == 64 ? 4 : 1;
  const int cap = p.group == 0 ? 64 : p.group == 1024 ? 256 : LN_MAX_BLOCKS;
  const int want = (M + per - 1) / per;
  return want < 1 ? 1 : (want < cap ? want : cap);
}

// A launch has fewer than 2^32 threads, up to 1024 of them for a row: more rows take several.
constexpr int LN_MAX_ROWS = 1 << 21;
template <typename P>
P* at_row(P* p, int m, long long ld, int size) { return p ? (P*)((char*)p + m * ld * size) : nullptr; }

template <typename T, typename TW, int GROUP, int NV>
void ln_fwd_launch(const LnFwd& a, hipStream_t st) {
  constexpr int PER = GROUP < 256 ? 256 / GROUP : 1;
  ln_fwd_kernel<T, TW, GROUP, NV><<<(unsigned)(((long long)a.M + PER - 1) / PER), GROUP < 256 ? 256 : GROUP, 0, st>>>(a);
}
template <typename T, typename TW>
int ln_fwd_run(const LnFwd& a, hipStream_t st) {
  constexpr int VE = Vec<T>::N;
  const LnPlan p = ln_plan(a.N, VE, LN_FWD);
#define CASE(G, V) if (p.group == G && p.nv == V) { ln_fwd_launch<T, TW, G, V>(a, st); return cg_launch_status(); }
  CASE(64, 1) CASE(64, 2) CASE(64, 3) CASE(64, 4)
  CASE(256, 3) CASE(256, 4)
  CASE(1024, 2) CASE(1024, 3) CASE(1024, 4)
  if constexpr (VE == 8) { CASE(256, 2) }
  if constexpr (VE == 4) { CASE(64, 5) CASE(64, 6) CASE(64, 7) CASE(64, 8) CASE(1024, 5) CASE(1024, 6) CASE(1024, 7) CASE(1024, 8) }
#undef CASE
  if (p.group != 0) return CG_ERR_UNSUPPORTED;
  ln_fwd_long_kernel<T, TW><<<a.M, 1024, 0, st>>>(a);
  return cg_launch_status();
}

template <typename T, typename TW>
int ln_bwd_run(const LnBwd& a, TW* dw, TW* db, hipStream_t st) {
  constexpr int VE = Vec<T>::N;
  const int nb = ln_bwd_blocks(a.M, a.N, VE);
  if (a.M > 0) {
    LnPlan p = ln_plan(a.N, VE, LN_DX_COLS);
    const bool together = a.part && p.group != 0;
    if (together) {
#define CASE(G, V) \
  if (p.group == G && p.nv == V) { ln_bwd_kernel<T, TW, G, V, true><<<nb, G < 256 ? 256 : G, 0, st>>>(a); p.group = -1; }
      CASE(64, 1) CASE(64, 2) CASE(256, 2)
      if constexpr (VE == 8) { CASE(256, 1) CASE(1024, 1) }
      if constexpr (VE == 4) { CASE(64, 3) CASE(64, 4) CASE(256, 3) CASE(256, 4) CASE(1024, 2) CASE(1024, 3) }
#undef CASE
      if (p.group != -1) return CG_ERR_UNSUPPORTED;
    } else {
      if (a.part) ln_cols_kernel<T><<<dim3(((a.N + VE - 1) / VE + 255) / 256, nb), 256, 0, st>>>(a);
      if (a.dX) {
        p = ln_plan(a.N, VE, LN_DX);
        const unsigned rows = (unsigned)(p.group == 64 ? ((long long)a.M + 3) / 4 : a.M);      // each walks on by as many
        const unsigned grid = rows < LN_MAX_ROWS ? rows : LN_MAX_ROWS;
#define CASE(G, V) \
  if (p.group == G && p.nv == V) { ln_bwd_kernel<T, TW, G, V, false><<<grid, G < 256 ? 256 : G, 0, st>>>(a); p.group = -1; }
        CASE(64, 1) CASE(64, 2) CASE(64, 3) CASE(64, 4)
        CASE(256, 3) CASE(256, 4)
        CASE(1024, 2) CASE(1024, 3)
        if constexpr (VE == 8) { CASE(256, 2) }
        if constexpr (VE == 4) { CASE(64, 5) CASE(64, 6) CASE(64, 7) CASE(64, 8) CASE(1024, 4) CASE(1024, 5) CASE(1024, 6) }
#undef CASE
        if (p.group > 0) return CG_ERR_UNSUPPORTED;
        if (p.group == 0) ln_bwd_long_kernel<T, TW><<<a.M, 1024, 0, st>>>(a);
      }
    }
  }
  if (a.part)
    ln_cols_reduce_kernel<TW><<<dim3((a.N + 15) / 16, db ? 2 : 1), nb <= 256 ? 256 : 1024, 0, st>>>(dw, db, a.part, a.M == 0 ? 0 : nb, a.N);
  return cg_launch_status();
}

bool ln_types_ok(int dtype, int wdtype) {
  return (dtype == CG_F32 && wdtype == CG_F32) || (dtype == CG_BF16 && (wdtype == CG_F32 || wdtype == CG_BF16));
}

}  // namespace

extern "C" size_t cg_ln_bwd_workspace_bytes(int M, int N, int dtype) {
  if (M < 0 || N < 1 || N > LN_MAX_COLS) return 0;
  return (size_t)ln_bwd_blocks(M, N, dtype == CG_BF16 ? 8 : 4) * 2 * N * sizeof(float);
}

extern "C" int cg_ln_fwd(void* Y, long long ldy, void* S, long long lds, const void* X, long long ldx, const void* R,
                         long long ldr, const void* weight, const void* bias, float eps, float* mean, float* rstd, int M,
                         int N, int dtype, int wdtype, void* stream) {
  if (M < 0 || N < 1 || (M > 0 && (!Y || !X)) || !ln_types_ok(dtype, wdtype) || (mean == nullptr) != (rstd == nullptr))
    return CG_ERR_BAD_ARG;
  if (N > LN_MAX_COLS) return CG_ERR_UNSUPPORTED;
  if (M > 1 && (ldy < N || ldx < N || (S && lds < N) || (R && ldr < N))) return CG_ERR_BAD_ARG;
  if (M == 0) return CG_OK;
  hipStream_t st = (hipStream_t)stream;
  const int size = dtype == CG_F32 ? 4 : 2;
  for (int m = 0; m < M; m += LN_MAX_ROWS) {
    const LnFwd a{at_row(Y, m, ldy, size), ldy, at_row(S, m, lds, size), lds, at_row(X, m, ldx, size), ldx, at_row(R, m, ldr, size),
                  ldr, weight, bias, eps, at_row(mean, m, 1, 4), at_row(rstd, m, 1, 4), M - m < LN_MAX_ROWS ? M - m : LN_MAX_ROWS, N};
    const int status = dtype == CG_F32 ? ln_fwd_run<float, float>(a, st)
                       : wdtype == CG_F32 ? ln_fwd_run<u16, float>(a, st) : ln_fwd_run<u16, u16>(a, st);
    if (status != CG_OK) return status;
  }
  return CG_OK;
}

extern "C" int cg_ln_bwd(void* dX, long long lddx, const void* dY, long long lddy, const void* dS, long long ldds,
                         const void* S, long long lds, const void* R, long long ldr, const void* weight,
                         const float* mean, const float* rstd, void* dweight, void* dbias, int M, int N, int dtype, int wdtype, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (M < 0 || N < 1 || (M > 0 && (!dY || !S || !mean || !rstd)) || !ln_types_ok(dtype, wdtype)) return CG_ERR_BAD_ARG;
  if (!dX && !dweight && !dbias) return CG_ERR_BAD_ARG;
  if (N > LN_MAX_COLS) return CG_ERR_UNSUPPORTED;
  if (M > 1 && ((dX && lddx < N) || lddy < N || lds < N || (dS && ldds < N) || (R && ldr < N))) return CG_ERR_BAD_ARG;
  const bool cols = dweight || dbias;
  if (cols && (!workspace || workspace_bytes < cg_ln_bwd_workspace_bytes(M, N, dtype))) return CG_ERR_WORKSPACE;
  if (M == 0 && !cols) return CG_OK;
  const LnBwd a{dX, lddx, dY, lddy, dS, ldds, S, lds, R, ldr, weight, mean, rstd, cols ? (float*)workspace : nullptr, M, N};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CG_F32) return ln_bwd_run<float, float>(a, (float*)dweight, (float*)dbias, st);
  return wdtype == CG_F32 ? ln_bwd_run<u16, float>(a, (float*)dweight, (float*)dbias, st)
                          : ln_bwd_run<u16, u16>(a, (u16*)dweight, (u16*)dbias, st);
}
