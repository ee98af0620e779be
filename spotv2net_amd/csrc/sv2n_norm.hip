// Layer norm over the last dimension, forward and backward (f32, bf16, f16).
//
//   z = (x - mean) · rstd,  rstd = 1/sqrt(var + eps),  y = z·w + b
//   g = dy·w;  dx = rstd·(g - mean(g) - z·mean(g·z));  dw = Σ_rows dy·z;  db = Σ_rows dy
//
// Both passes are bound by memory: the forward reads x once and writes y, the
// backward reads x and dy once and writes dx.  A row is held in the registers
// of TPR threads (16 B per thread and load), so taking the mean, then the mean of the
// deviations from it (added to the mean), then the squares of those left costs no second
// read and loses nothing to cancellation: a row of equal values has exactly that mean,
// z = 0 and variance 0, where a mean off by its rounding would come out scaled by rstd,
// up to 1/sqrt(eps).  (The factors 1/cols are rounded too: the first is corrected, the
// second moves a correction of a few units by far less than one.)  TPR is the smallest group that leaves a thread at most 16 elements
// (32 past rows of 8,192), since the backward holds five such arrays (x, dy, w and the
// sums of dw and db): 16 threads for a row of 128, so a wave carries four of them.
// Groups walk the rows with a stride; each thread owns the same columns in every
// row, so dw and db are summed in its registers (f32) and leave the block once,
// as a partial per block that a second launch adds in block order: no atomics,
// the same bits every run.
//
// Rows need no alignment: the 16-B loads and stores are emitted for the element's own
// alignment (the hardware takes them at any).  Only a thread's last vector can reach
// past the row; it is loaded from where it still fits (cols - V) with the elements of
// the vector before it masked, so no load branches and none leaves the row.  Rows
// shorter than a vector go element by element.
//
// The next row's loads are in flight while a row is summed, clamped to the last row
// instead of branching; a group past the last row adds zeros.
//
// MI355X, us (forward / backward with its second launch; a large copy reaches 5.0 TB/s):
//   15,360 x 400 f32      10.5 / 18.5        16,384 x 4,096 f32    97 / 158  (5.5 / 5.1 TB/s)
//   262,144 x 128 f32       45 / 81          16,384 x 8,192 bf16  100 / 153  (5.4 / 5.3 TB/s)
//   3,840 x 3,000 bf16    12.0 / 27.8        10,007 x 1,261 f16  18.2 / 25.9
// The last two are 1.3 and 1.8 (forward), 2.0 and 1.7 (backward) times a copy of their
// bytes: rows of 375 and 158 vectors leave a quarter and three eighths of the places for
// vectors empty, the backward's partials are a quarter and a fifth of its bytes again
// (written and read, 17 and 15 MB), and 360 blocks for 3,840 rows give 104 of the 256 CUs
// 22 rows and the others 11.
#include "sv2n_common.h"
#include <algorithm>
#include <type_traits>

namespace sv2n {

enum { LN_FULL = 0, LN_ODD = 1, LN_TINY = 2 };  // cols % V == 0, other, cols < V

template <typename T>
struct LnVec {
  static constexpr int V = 16 / (int)sizeof(T);
};

// Where a thread's vector k starts and which of its elements are its own
template <int MODE, int V>
struct LnAt {
  int c, skip, own;  // first column read; elements before the own ones; own ones
  __device__ __forceinline__ void set(int c0, int cols, bool last) {
    c = c0;
    skip = 0;
    own = V;
    if (!last) return;
    if (MODE == LN_TINY) {
      own = min(max(cols - c0, 0), V);
      if (own == 0) c = 0;
    } else if (c0 + V > cols) {
      c = cols - V;
      own = max(cols - c0, 0);
      skip = V - own;
    }
  }
  __device__ __forceinline__ bool has(int j) const {
    return MODE == LN_FULL ? own != 0 : MODE == LN_ODD ? j >= skip : j < own;
  }
};

// 16 B of a row as they are in memory
template <typename T>
struct LnRaw {
  T t[LnVec<T>::V];
};
template <int MODE, typename T>
__device__ __forceinline__ LnRaw<T> ln_raw(const T* __restrict__ row,
                                           const LnAt<MODE, LnVec<T>::V>& at) {
  constexpr int V = LnVec<T>::V;
  LnRaw<T> r;
  if (MODE == LN_TINY) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      r.t[j] = (T)0.f;
      if (j < at.own) r.t[j] = row[at.c + j];
    }
  } else {
    __builtin_memcpy(r.t, row + at.c, sizeof(r.t));
  }
  return r;
}
template <int MODE, typename T>
__device__ __forceinline__ void ln_st(T* __restrict__ row, const LnAt<MODE, LnVec<T>::V>& at,
                                      bool last, const float (&o)[LnVec<T>::V]) {
  constexpr int V = LnVec<T>::V;
  if (!last || at.own == V) {
    T t[V];
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = (T)o[j];
    __builtin_memcpy(row + at.c, t, sizeof(t));
  } else if (MODE != LN_FULL && at.own > 0) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (at.has(j)) row[at.c + j] = (T)o[j];
  }
}

// V elements of an optional vector p of type wdt (the value `none` where there is none)
template <int MODE, typename W, int V>
__device__ __forceinline__ void ln_ld_as(const void* __restrict__ p, const LnAt<MODE, V>& at,
                                         float (&o)[V]) {
  const W* q = (const W*)p + at.c;
  if (MODE == LN_TINY) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < at.own) o[j] = (float)q[j];
  } else {
    W t[V];
    __builtin_memcpy(t, q, sizeof(t));
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = (float)t[j];
  }
}
template <typename T, int MODE, int V>
__device__ __forceinline__ void ln_ld_w(const void* __restrict__ p, int wdt,
                                        const LnAt<MODE, V>& at, float none, float (&o)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = none;
  if (!p) return;
  if (wdt == SV2N_DT_F32) ln_ld_as<MODE, float>(p, at, o);
  else ln_ld_as<MODE, T>(p, at, o);
}

// Sum over an aligned group of G <= 64 lanes, the result in every lane: quads
// by quad_perm, 8 and 16 lanes by the row mirrors (each half is uniform by
// then), 32 and 64 by the gfx950 row swaps (v_permlane{16,32}_swap of a value
// with itself gives both partners' values).
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#define SV2N_DPP(c) __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), c, 0xF, 0xF, false))
  if (G >= 2) v += SV2N_DPP(0xB1);
  if (G >= 4) v += SV2N_DPP(0x4E);
  if (G >= 8) v += SV2N_DPP(0x141);   // row_half_mirror
  if (G >= 16) v += SV2N_DPP(0x140);  // row_mirror
#undef SV2N_DPP
  if (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (G >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Sums of s1 and s2 over a row's threads, the result in all of them.  Rows of several
// waves exchange through `red`, two buffers in turn so that one barrier does; every
// group of the block takes part in it, with or without a row.
template <int TPR>
__device__ __forceinline__ void row_sums(float& s1, float& s2, float (*red)[2], int grp, int t) {
  constexpr int G = TPR < 64 ? TPR : 64, WPR = TPR / 64;
  s1 = group_sum<G>(s1);
  s2 = group_sum<G>(s2);
  if constexpr (WPR > 1) {
    float(*mine)[2] = red + grp * WPR;
    if ((t & 63) == 0) {
      mine[t / 64][0] = s1;
      mine[t / 64][1] = s2;
    }
    __syncthreads();
    s1 = s2 = 0.f;
#pragma unroll
    for (int u = 0; u < WPR; ++u) {
      s1 += mine[u][0];
      s2 += mine[u][1];
    }
  }
}

// threads of a block
template <int TPR>
constexpr int ln_threads() { return TPR < 256 ? 256 : TPR; }
// waves per SIMD the backward's registers are fitted to
template <int TPR>
constexpr int ln_bwd_waves() { return TPR <= 256 ? 3 : 2; }

template <typename T, int TPR, int NPT, int MODE>
__global__ __launch_bounds__(ln_threads<TPR>()) void k_ln_fwd(
    const T* __restrict__ x, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b,
    int wdt, int64_t rows, int cols, float eps, T* __restrict__ y, float* __restrict__ mean,
    float* __restrict__ rstd) {
  constexpr int V = LnVec<T>::V;
  constexpr int THREADS = ln_threads<TPR>();
  constexpr int GROUPS = THREADS / TPR;
  constexpr int WPR = TPR / 64;  // waves per row (0: several rows per wave)
  constexpr int G = TPR < 64 ? TPR : 64;
  __shared__ float red[2][WPR > 1 ? THREADS / 64 : 1][2];
  const int t = threadIdx.x % TPR;
  const int grp = threadIdx.x / TPR;
  float wv[NPT][V], bv[NPT][V];
  LnAt<MODE, V> at[NPT];
#pragma unroll
  for (int k = 0; k < NPT; ++k) {
    at[k].set((k * TPR + t) * V, cols, k == NPT - 1);
    ln_ld_w<T>(w, wdt, at[k], 1.f, wv[k]);
    ln_ld_w<T>(b, wdt, at[k], 0.f, bv[k]);
  }
  const float inv_c = 1.f / (float)cols;
  // (rows of several waves: of the elements of this wave, if any)
  float inv_n = inv_c;
  if constexpr (WPR > 1) {
    int n = 0;
#pragma unroll
    for (int k = 0; k < NPT; ++k)
      n += max(0, min(64 * V, cols - k * TPR * V - (t / 64) * 64 * V));
    inv_n = 1.f / (float)max(n, 1);
  }
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  LnRaw<T> next[NPT];
  auto fetch = [&](int64_t row) {
    const T* xr = x + min(row, rows - 1) * ldx;
#pragma unroll
    for (int k = 0; k < NPT; ++k) next[k] = ln_raw<MODE>(xr, at[k]);
  };
  int64_t row = (int64_t)blockIdx.x * GROUPS + grp;
  fetch(row);
  // the block's first row decides how often it goes round: its groups stay together
  int buf = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * GROUPS; r0 < rows; r0 += step, row += step) {
    // (a deviation is from the rounded mean that the correction is added to, not from an
    // unrounded product inside a fused operation)
#pragma clang fp contract(off)
    float v[NPT][V];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[k][j] = (float)next[k].t[j];
        s += k < NPT - 1 || at[k].has(j) ? v[k][j] : 0.f;
      }
    fetch(row + step);
    s = group_sum<G>(s);
    float m = s * inv_n, m1 = 0.f, m2 = 0.f;
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) m1 += k < NPT - 1 || at[k].has(j) ? v[k][j] - m : 0.f;
    m += group_sum<G>(m1) * inv_n;
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = k < NPT - 1 || at[k].has(j) ? v[k][j] - m : 0.f;
        m2 = fmaf(d, d, m2);
      }
    m2 = group_sum<G>(m2);
    if constexpr (WPR > 1) {
      // one exchange per row (two buffers, so one barrier): the mean of the waves'
      // means by their counts, from the first one's, and Σ m2 + n·(mean_wave - mean)²
      float(*mine)[2] = red[buf] + grp * WPR;
      if ((t & 63) == 0) {
        mine[t / 64][0] = m;
        mine[t / 64][1] = m2;
      }
      __syncthreads();
      const float m0 = mine[0][0];
      float tot = 0.f, q = 0.f;
#pragma unroll
      for (int u = 0; u < WPR; ++u) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < NPT; ++k) n += max(0, min(64 * V, cols - k * TPR * V - u * 64 * V));
        tot = fmaf((float)n, mine[u][0] - m0, tot);
      }
      m = fmaf(tot, inv_c, m0);
#pragma unroll
      for (int u = 0; u < WPR; ++u) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < NPT; ++k) n += max(0, min(64 * V, cols - k * TPR * V - u * 64 * V));
        const float d = mine[u][0] - m;
        q += fmaf((float)n * d, d, mine[u][1]);
      }
      m2 = q;
      buf ^= 1;
    }
    if (row >= rows) continue;
    const float r = 1.f / sqrtf(fmaf(m2, inv_c, eps));
    if (t == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
    T* yr = y + row * (int64_t)cols;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = fmaf((v[k][j] - m) * r, wv[k][j], bv[k][j]);
      ln_st<MODE>(yr, at[k], k == NPT - 1, o);
    }
  }
}

// part [gridDim.x][2][cols]: the block's Σ dy·z and Σ dy
template <typename T, int TPR, int NPT, int MODE>
__global__ __launch_bounds__(ln_threads<TPR>(), ln_bwd_waves<TPR>()) void k_ln_bwd(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
    const void* __restrict__ w, int wdt, const float* __restrict__ mean,
    const float* __restrict__ rstd, int64_t rows, int cols, T* __restrict__ dx,
    float* __restrict__ part) {
  constexpr int V = LnVec<T>::V;
  constexpr int THREADS = ln_threads<TPR>();
  constexpr int GROUPS = THREADS / TPR;
  constexpr int WPR = TPR / 64;
  constexpr bool AHEAD = NPT * V <= 16;  // the next row's loads are in flight
  constexpr int CAP = TPR * NPT * V;  // columns a group can hold
  __shared__ float red[2][WPR > 1 ? THREADS / 64 : 1][2];
  __shared__ float acc[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? CAP : 1];
  const int t = threadIdx.x % TPR;
  const int grp = threadIdx.x / TPR;
  float wv[NPT][V], gw[NPT][V], gb[NPT][V];
  LnAt<MODE, V> at[NPT];
#pragma unroll
  for (int k = 0; k < NPT; ++k) {
    at[k].set((k * TPR + t) * V, cols, k == NPT - 1);
    ln_ld_w<T>(w, wdt, at[k], 1.f, wv[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) gw[k][j] = gb[k][j] = 0.f;
  }
  const float inv_c = 1.f / (float)cols;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  LnRaw<T> nx[NPT], nd[NPT];
  float nm, nr;
  auto fetch = [&](int64_t row) {
    row = min(row, rows - 1);
    const T* xr = x + row * ldx;
    const T* dr = dy + row * lddy;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      nx[k] = ln_raw<MODE>(xr, at[k]);
      nd[k] = ln_raw<MODE>(dr, at[k]);
    }
    nm = mean[row];
    nr = rstd[row];
  };
  int64_t row = (int64_t)blockIdx.x * GROUPS + grp;
  if (AHEAD) fetch(row);
  int buf = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * GROUPS; r0 < rows; r0 += step, row += step) {
    const bool here = row < rows;
    if (!AHEAD) fetch(row);
    float xv[NPT][V], dv[NPT][V];
    const float m = nm, r = nr;
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool mine = here && (k < NPT - 1 || at[k].has(j));
        // zeros where there is nothing of this group's (a NaN of another row, or of a
        // column that another thread adds, must not reach its sums)
        xv[k][j] = mine ? ((float)nx[k].t[j] - m) * r : 0.f;
        dv[k][j] = mine ? (float)nd[k].t[j] : 0.f;
      }
    if (AHEAD) fetch(row + step);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float z = xv[k][j], d = dv[k][j];
        gb[k][j] += d;
        gw[k][j] = fmaf(d, z, gw[k][j]);
        const float g = d * wv[k][j];
        dv[k][j] = g;
        s1 += g;
        s2 = fmaf(g, z, s2);
      }
    }
    if (dx) {
      row_sums<TPR>(s1, s2, red[buf], grp, t);
      buf ^= 1;
      if (!here) continue;
      s1 *= inv_c;
      s2 *= inv_c;
      T* o = dx + row * (int64_t)cols;
#pragma unroll
      for (int k = 0; k < NPT; ++k) {
        float ov[V];
#pragma unroll
        for (int j = 0; j < V; ++j) ov[j] = r * (dv[k][j] - fmaf(xv[k][j], s2, s1));
        ln_st<MODE>(o, at[k], k == NPT - 1, ov);
      }
    }
  }
  if (!part) return;
  float* p = part + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (GROUPS > 1) {
    // the groups' sums in group order, dw's and then db's through the same LDS
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which) __syncthreads();
#pragma unroll
      for (int k = 0; k < NPT; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (k < NPT - 1 || at[k].has(j)) acc[grp][at[k].c + j] = which ? gb[k][j] : gw[k][j];
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += THREADS) {
        float s = 0.f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) s += acc[g][c];
        p[which * cols + c] = s;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (k < NPT - 1 || at[k].has(j)) {
          p[at[k].c + j] = gw[k][j];
          p[cols + at[k].c + j] = gb[k][j];
        }
  }
}

// dw / db [cols] = Σ over the nblk partials, in block order within each of 1024 / CW
// slices and slice order after that (fixed, so the same bits every run).  CW columns a
// block: 16 keep 128 columns on 16 blocks; rows past 2,048 give blocks enough with 64,
// whose reads are whole lines (256 partials of 16,384 columns: 12.2 -> 8.9 us).
template <typename W, int CW>
__global__ __launch_bounds__(1024) void k_ln_wgrad(const float* __restrict__ part, int nblk,
                                                   int cols, W* __restrict__ dw,
                                                   W* __restrict__ db, int accumulate) {
  constexpr int S = 1024 / CW;
  __shared__ float sl[S][CW + 1];
  const int cc = threadIdx.x % CW, s = threadIdx.x / CW;
  const int c = blockIdx.x * CW + cc;  // over [0, 2·cols)
  float v = 0.f;
  if (c < 2 * cols) {
    const float* p = part + c;
#pragma unroll 8
    for (int i = s; i < nblk; i += S) v += p[(int64_t)i * 2 * cols];
  }
  sl[s][cc] = v;
  __syncthreads();
  if (s == 0 && c < 2 * cols) {
    float tot = 0.f;
#pragma unroll
    for (int u = 0; u < S; ++u) tot += sl[u][cc];
    W* o = c < cols ? dw : db;
    const int k = c < cols ? c : c - cols;
    if (o) o[k] = (W)(accumulate ? (float)o[k] + tot : tot);
  }
}

// Blocks of the backward (and so partials): at most three a CU (one of 512 threads),
// and past one a CU only while the partials stay under an eighth of the rows' bytes.
static inline int ln_bwd_blocks(int64_t rows, int tpr, int bytes) {
  const int groups = tpr < 256 ? 256 / tpr : 1;
  const int64_t need = (rows + groups - 1) / groups;
  const int64_t cap = tpr > 256 ? 256 : 768;
  const int64_t cheap = std::max<int64_t>(256, rows * 3 * bytes / 64);
  return (int)std::max<int64_t>(1, std::min({need, cap, cheap}));
}

// threads per row for a row of nv 16-B vectors with at most `most` per thread (rows past
// 8,192 elements: up to twice that in 512 threads)
static inline int ln_tpr(int64_t nv, int most) {
  for (int t : {16, 32, 64, 128, 256})
    if (nv <= (int64_t)t * most) return t;
  return 512;
}

template <typename T>
struct LnLaunch {
  static constexpr int V = LnVec<T>::V;
  static constexpr int MOST = 16 / V;
  const T* x;
  int64_t ldx;
  const void *w, *b;
  int wdt;
  int64_t rows;
  int cols;
  float eps;
  T* y;
  float *mean, *rstd;
  // backward
  const T* dy;
  int64_t lddy;
  const float *cmean, *crstd;
  T* dx;
  float* part;
  hipStream_t stream;

  template <int TPR, int NPT, int MODE>
  void launch(bool fwd) const {
    constexpr int TH = ln_threads<TPR>();
    constexpr int GR = TH / TPR;
    if (fwd) {
      const int64_t need = (rows + GR - 1) / GR;
      const int grid = (int)std::min<int64_t>(need, TPR > 256 ? 1024 : 2048);
      hipLaunchKernelGGL((k_ln_fwd<T, TPR, NPT, MODE>), dim3(grid), dim3(TH), 0, stream, x, ldx, w,
                         b, wdt, rows, cols, eps, y, mean, rstd);
    } else {
      hipLaunchKernelGGL((k_ln_bwd<T, TPR, NPT, MODE>),
                         dim3(ln_bwd_blocks(rows, TPR, (int)sizeof(T))), dim3(TH), 0, stream, dy,
                         lddy, x, ldx, w, wdt, cmean, crstd, rows, cols, dx, part);
    }
  }
  template <int TPR, int NPT>
  void go(bool fwd) const {
    if (cols % V == 0) return launch<TPR, NPT, LN_FULL>(fwd);
    if constexpr (TPR == 16 && NPT == 1)
      if (cols < V) return launch<TPR, NPT, LN_TINY>(fwd);
    launch<TPR, NPT, LN_ODD>(fwd);
  }
  // NPT is exact (every vector but a thread's last is whole): the smaller counts of a
  // group belong to the group below it, so only the reachable ones are instances
  void run(bool fwd) const {
    const int nv = (cols + V - 1) / V;
    const int tpr = ln_tpr(nv, MOST);
    const int npt = (nv + tpr - 1) / tpr;
    if constexpr (V == 4) {
      switch (tpr * 16 + npt) {
        case 16 * 16 + 1: return go<16, 1>(fwd);
        case 16 * 16 + 2: return go<16, 2>(fwd);
        case 16 * 16 + 3: return go<16, 3>(fwd);
        case 16 * 16 + 4: return go<16, 4>(fwd);
        case 32 * 16 + 3: return go<32, 3>(fwd);
        case 32 * 16 + 4: return go<32, 4>(fwd);
        case 64 * 16 + 3: return go<64, 3>(fwd);
        case 64 * 16 + 4: return go<64, 4>(fwd);
        case 128 * 16 + 3: return go<128, 3>(fwd);
        case 128 * 16 + 4: return go<128, 4>(fwd);
        case 256 * 16 + 3: return go<256, 3>(fwd);
        case 256 * 16 + 4: return go<256, 4>(fwd);
        case 512 * 16 + 3: return go<512, 3>(fwd);
        case 512 * 16 + 4: return go<512, 4>(fwd);
        case 512 * 16 + 5: return go<512, 5>(fwd);
        case 512 * 16 + 6: return go<512, 6>(fwd);
        case 512 * 16 + 7: return go<512, 7>(fwd);
        default: return go<512, 8>(fwd);
      }
    } else {
      switch (tpr * 16 + npt) {
        case 16 * 16 + 1: return go<16, 1>(fwd);
        case 16 * 16 + 2: return go<16, 2>(fwd);
        case 32 * 16 + 2: return go<32, 2>(fwd);
        case 64 * 16 + 2: return go<64, 2>(fwd);
        case 128 * 16 + 2: return go<128, 2>(fwd);
        case 256 * 16 + 2: return go<256, 2>(fwd);
        case 512 * 16 + 2: return go<512, 2>(fwd);
        case 512 * 16 + 3: return go<512, 3>(fwd);
        default: return go<512, 4>(fwd);
      }
    }
  }
};

template <typename W>
static int ln_wgrad(const float* part, int nblk, int cols, void* dw, void* db, int accumulate,
                    hipStream_t stream) {
  if (cols > 2048)
    hipLaunchKernelGGL((k_ln_wgrad<W, 64>), dim3((2 * cols + 63) / 64), dim3(1024), 0, stream, part,
                       nblk, cols, (W*)dw, (W*)db, accumulate);
  else
    hipLaunchKernelGGL((k_ln_wgrad<W, 16>), dim3((2 * cols + 15) / 16), dim3(1024), 0, stream, part,
                       nblk, cols, (W*)dw, (W*)db, accumulate);
  return (int)hipGetLastError();
}

static inline bool ln_types_ok(int dtype, int wdtype) {
  return dtype >= SV2N_DT_F32 && dtype <= SV2N_DT_F16 &&
         (wdtype == SV2N_DT_F32 || wdtype == dtype);
}
static inline int ln_bytes(int dtype) { return dtype == SV2N_DT_F32 ? 4 : 2; }

template <typename F>
static int ln_dispatch(int dtype, F&& f) {
  if (dtype == SV2N_DT_F32) return f((float*)nullptr);
  if (dtype == SV2N_DT_BF16) return f((__bf16*)nullptr);
  return f((_Float16*)nullptr);
}

}  // namespace sv2n

using namespace sv2n;

extern "C" int sv2n_layer_norm_fwd(const void* x, int64_t ldx, int dtype, const void* weight,
                                   const void* bias, int wdtype, int64_t rows, int cols, float eps,
                                   void* y, float* mean, float* rstd, hipStream_t stream) {
  if (rows < 0 || cols <= 0 || !(eps >= 0.f) || !ln_types_ok(dtype, wdtype)) return SV2N_ERR_ARG;
  if (cols > SV2N_LN_MAX_COLS || ldx < cols) return SV2N_ERR_SHAPE;
  if (rows == 0) return 0;
  if (!x || !y) return SV2N_ERR_ARG;
  if (((uintptr_t)x | (uintptr_t)y) & (ln_bytes(dtype) - 1)) return SV2N_ERR_ALIGN;
  return ln_dispatch(dtype, [&](auto* tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    LnLaunch<T> l{};
    l.x = (const T*)x; l.ldx = ldx; l.w = weight; l.b = bias; l.wdt = wdtype;
    l.rows = rows; l.cols = cols; l.eps = eps; l.y = (T*)y; l.mean = mean; l.rstd = rstd;
    l.stream = stream;
    l.run(true);
    return (int)hipGetLastError();
  });
}

extern "C" int64_t sv2n_layer_norm_bwd_workspace(int64_t rows, int cols, int dtype) {
  if (rows <= 0 || cols <= 0 || cols > SV2N_LN_MAX_COLS || !ln_types_ok(dtype, dtype)) return 0;
  const int v = 16 / ln_bytes(dtype);
  return (int64_t)ln_bwd_blocks(rows, ln_tpr((cols + v - 1) / v, 16 / v), ln_bytes(dtype)) *
         2 * cols;
}

extern "C" int sv2n_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                   int dtype, const void* weight, int wdtype, const float* mean,
                                   const float* rstd, int64_t rows, int cols, void* dx, void* dw,
                                   void* db, int accumulate, float* workspace,
                                   int64_t workspace_floats, hipStream_t stream) {
  if (rows < 0 || cols <= 0 || !ln_types_ok(dtype, wdtype)) return SV2N_ERR_ARG;
  if (cols > SV2N_LN_MAX_COLS || ldx < cols || lddy < cols) return SV2N_ERR_SHAPE;
  const bool wg = dw || db;
  if (rows > 0) {
    if (!dy || !x || !mean || !rstd) return SV2N_ERR_ARG;
    if (((uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx) & (ln_bytes(dtype) - 1))
      return SV2N_ERR_ALIGN;
    if (wg && (!workspace ||
               workspace_floats < sv2n_layer_norm_bwd_workspace(rows, cols, dtype)))
      return SV2N_ERR_WORKSPACE;
  }
  if (rows == 0 && (accumulate || !wg)) return 0;
  if (rows > 0 && !dx && !wg) return 0;
  return ln_dispatch(dtype, [&](auto* tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    int nblk = 0;
    if (rows > 0) {
      LnLaunch<T> l{};
      l.x = (const T*)x; l.ldx = ldx; l.w = weight; l.wdt = wdtype; l.rows = rows; l.cols = cols;
      l.dy = (const T*)dy; l.lddy = lddy; l.cmean = mean; l.crstd = rstd; l.dx = (T*)dx;
      l.part = wg ? workspace : nullptr;
      l.stream = stream;
      l.run(false);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
      nblk = (int)(sv2n_layer_norm_bwd_workspace(rows, cols, dtype) / (2 * cols));
    }
    if (!wg) return 0;
    if (wdtype == SV2N_DT_F32)
      return ln_wgrad<float>(workspace, nblk, cols, dw, db, accumulate, stream);
    return ln_wgrad<T>(workspace, nblk, cols, dw, db, accumulate, stream);
  });
}
