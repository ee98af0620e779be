// Layer norm over the last dimension, forward and backward (f32, bf16, f16).
//
//   z = (x - mean) · rstd,  rstd = 1/sqrt(var + eps),  y = z·w + b
//   g = dy·w;  dx = rstd·(g - mean(g) - z·mean(g·z));  dw = Σ_rows dy·z;  db = Σ_rows dy
//
// Both passes are bound by memory: the forward reads x once and writes y, the
// backward reads x and dy once and writes dx.  A row is held in the registers
// of TPR threads (16 B per thread and load), so the two-step variance (mean
// first, then the squared deviations) costs no second read and loses nothing to
// cancellation.  TPR is the smallest group that leaves a thread at most 16
// elements, since the backward holds five such arrays (x, dy, w and the sums of
// dw and db): 16 threads for a row of 128, so a wave carries four of them.
// (1,024 threads have 128 registers each: there the weight is read again per row.)
// Groups walk the rows with a stride; each thread owns the same columns in every
// row, so dw and db are summed in its registers (f32) and leave the block once,
// as a partial per block that a second launch adds in block order: no atomics,
// the same bits every run.
//
// Rows need no alignment: the 16-B loads and stores are emitted for the
// element's own alignment (the hardware takes them at any), and only the one
// vector that crosses the end of a row goes element by element.
#include "sv2n_common.h"
#include <algorithm>
#include <type_traits>

namespace sv2n {

template <typename T>
struct LnVec {
  static constexpr int V = 16 / (int)sizeof(T);
};

// V elements at p (only the first `valid` exist); absent ones read as 0
template <int V, typename T>
__device__ __forceinline__ void ln_ld(const T* __restrict__ p, int valid, float (&o)[V]) {
  if (valid >= V) {
    T t[V];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = (float)t[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      o[j] = 0.f;
      if (j < valid) o[j] = (float)p[j];
    }
  }
}
// the same of an optional vector p (the value `none` where there is none)
template <int V, typename T>
__device__ __forceinline__ void ln_ld_or(const T* __restrict__ p, int c0, int valid, float none,
                                         float (&o)[V]) {
  if (p) {
    ln_ld<V>(p + c0, valid, o);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = none;
  }
}
template <int V, typename T>
__device__ __forceinline__ void ln_st(T* __restrict__ p, int valid, const float (&o)[V]) {
  if (valid >= V) {
    T t[V];
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = (T)o[j];
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < valid) p[j] = (T)o[j];
  }
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

// threads of a block: at least 256, so that short rows still fill a block
template <int TPR>
constexpr int ln_threads() { return TPR < 256 ? 256 : TPR; }

template <typename T, typename W, int TPR, int NPT>
__global__ __launch_bounds__(ln_threads<TPR>()) void k_ln_fwd(
    const T* __restrict__ x, int64_t ldx, const W* __restrict__ w, const W* __restrict__ b,
    int64_t rows, int cols, float eps, T* __restrict__ y, float* __restrict__ mean,
    float* __restrict__ rstd) {
  constexpr int V = LnVec<T>::V;
  constexpr int THREADS = ln_threads<TPR>();
  constexpr int GROUPS = THREADS / TPR;
  constexpr int WPR = TPR / 64;  // waves per row (0: several rows per wave)
  constexpr int G = TPR < 64 ? TPR : 64;
  constexpr bool KEEP = TPR < 1024;  // the weight stays in registers
  __shared__ float red[2][WPR > 1 ? WPR : 1][2];
  const int t = threadIdx.x % TPR;
  const int grp = threadIdx.x / TPR;
  float wv[KEEP ? NPT : 1][V], bv[KEEP ? NPT : 1][V];
  int valid[NPT];
#pragma unroll
  for (int k = 0; k < NPT; ++k) {
    valid[k] = cols - (k * TPR + t) * V;
    if (KEEP) {
      ln_ld_or<V>(w, (k * TPR + t) * V, valid[k], 1.f, wv[k]);
      ln_ld_or<V>(b, (k * TPR + t) * V, valid[k], 0.f, bv[k]);
    }
  }
  const float inv_c = 1.f / (float)cols;
  int buf = 0;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + grp; row < rows;
       row += (int64_t)gridDim.x * GROUPS) {
    const T* xr = x + row * ldx;
    float v[NPT][V];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NPT; ++k) ln_ld<V>(xr + (k * TPR + t) * V, valid[k], v[k]);
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[k][j];
    s = group_sum<G>(s);
    float m, m2 = 0.f;
    if constexpr (WPR <= 1) {
      m = s * inv_c;
    } else {
      // the wave's own mean first; the waves are merged below
      const int wv0 = (t / 64) * 64 * V;
      int n = 0;
#pragma unroll
      for (int k = 0; k < NPT; ++k) n += max(0, min(64 * V, cols - k * TPR * V - wv0));
      m = n > 0 ? s / (float)n : 0.f;
    }
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[k][j] - m;
        if (j < valid[k]) m2 = fmaf(d, d, m2);
      }
    m2 = group_sum<G>(m2);
    if constexpr (WPR > 1) {
      // one exchange per row (two buffers, so one barrier): the mean of the
      // means by their counts, and Σ m2 + n·(mean_wave - mean)²
      const int wave = t / 64;
      if ((t & 63) == 0) {
        red[buf][wave][0] = m;
        red[buf][wave][1] = m2;
      }
      __syncthreads();
      float tot = 0.f, q = 0.f;
#pragma unroll
      for (int u = 0; u < WPR; ++u) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < NPT; ++k) n += max(0, min(64 * V, cols - k * TPR * V - u * 64 * V));
        tot = fmaf((float)n, red[buf][u][0], tot);
      }
      m = tot * inv_c;
#pragma unroll
      for (int u = 0; u < WPR; ++u) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < NPT; ++k) n += max(0, min(64 * V, cols - k * TPR * V - u * 64 * V));
        const float d = red[buf][u][0] - m;
        q += fmaf((float)n * d, d, red[buf][u][1]);
      }
      m2 = q;
      buf ^= 1;
    }
    const float r = 1.f / sqrtf(fmaf(m2, inv_c, eps));
    if (t == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
    T* yr = y + row * (int64_t)cols;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      constexpr int KS = KEEP ? 1 : 0;
      if (!KEEP) {
        ln_ld_or<V>(w, (k * TPR + t) * V, valid[k], 1.f, wv[0]);
        ln_ld_or<V>(b, (k * TPR + t) * V, valid[k], 0.f, bv[0]);
      }
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j)
        o[j] = fmaf((v[k][j] - m) * r, wv[KS * k][j], bv[KS * k][j]);
      ln_st<V>(yr + (k * TPR + t) * V, valid[k], o);
    }
  }
}

// part [gridDim.x][2][cols]: the block's Σ dy·z and Σ dy
template <typename T, typename W, int TPR, int NPT>
__global__ __launch_bounds__(ln_threads<TPR>()) void k_ln_bwd(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
    const W* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
    int64_t rows, int cols, T* __restrict__ dx, float* __restrict__ part) {
  constexpr int V = LnVec<T>::V;
  constexpr int THREADS = ln_threads<TPR>();
  constexpr int GROUPS = THREADS / TPR;
  constexpr int WPR = TPR / 64;
  constexpr int G = TPR < 64 ? TPR : 64;
  constexpr bool KEEP = TPR < 1024;  // the weight stays in registers
  constexpr int CAP = TPR * NPT * V;  // columns a group can hold
  __shared__ float red[2][WPR > 1 ? WPR : 1][2];
  __shared__ float acc[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? 2 * CAP : 1];
  const int t = threadIdx.x % TPR;
  const int grp = threadIdx.x / TPR;
  float wv[KEEP ? NPT : 1][V], gw[NPT][V], gb[NPT][V];
  int valid[NPT];
#pragma unroll
  for (int k = 0; k < NPT; ++k) {
    valid[k] = cols - (k * TPR + t) * V;
    if (KEEP) ln_ld_or<V>(w, (k * TPR + t) * V, valid[k], 1.f, wv[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) gw[k][j] = gb[k][j] = 0.f;
  }
  const float inv_c = 1.f / (float)cols;
  int buf = 0;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + grp; row < rows;
       row += (int64_t)gridDim.x * GROUPS) {
    float xv[NPT][V], dv[NPT][V];
    const T* xr = x + row * ldx;
    const T* dr = dy + row * lddy;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      ln_ld<V>(xr + (k * TPR + t) * V, valid[k], xv[k]);
      ln_ld<V>(dr + (k * TPR + t) * V, valid[k], dv[k]);
    }
    const float m = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      if (!KEEP) ln_ld_or<V>(w, (k * TPR + t) * V, valid[k], 1.f, wv[0]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // absent columns: dy is 0, so they add nothing whatever z is; z is kept
        // finite there (x reads 0, m and r are the row's)
        const float z = (xv[k][j] - m) * r;
        const float d = dv[k][j];
        xv[k][j] = z;
        gb[k][j] += d;
        gw[k][j] = fmaf(d, z, gw[k][j]);
        const float g = d * wv[KEEP ? k : 0][j];
        dv[k][j] = g;
        s1 += g;
        s2 = fmaf(g, z, s2);
      }
    }
    if (dx) {
      s1 = group_sum<G>(s1);
      s2 = group_sum<G>(s2);
      if constexpr (WPR > 1) {
        const int wave = t / 64;
        if ((t & 63) == 0) {
          red[buf][wave][0] = s1;
          red[buf][wave][1] = s2;
        }
        __syncthreads();
        s1 = s2 = 0.f;
#pragma unroll
        for (int u = 0; u < WPR; ++u) {
          s1 += red[buf][u][0];
          s2 += red[buf][u][1];
        }
        buf ^= 1;
      }
      s1 *= inv_c;
      s2 *= inv_c;
      T* o = dx + row * (int64_t)cols;
#pragma unroll
      for (int k = 0; k < NPT; ++k) {
        float ov[V];
#pragma unroll
        for (int j = 0; j < V; ++j) ov[j] = r * (dv[k][j] - fmaf(xv[k][j], s2, s1));
        ln_st<V>(o + (k * TPR + t) * V, valid[k], ov);
      }
    }
  }
  if (!part) return;
  float* p = part + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (GROUPS > 1) {
#pragma unroll
    for (int k = 0; k < NPT; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (k * TPR + t) * V + j;
        acc[grp][c] = gw[k][j];
        acc[grp][CAP + c] = gb[k][j];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * cols; c += THREADS) {
      const int a = c < cols ? c : CAP + c - cols;
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) s += acc[g][a];
      p[c] = s;
    }
  } else {
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      const int c0 = (k * TPR + t) * V;
      ln_st<V>(p + c0, valid[k], gw[k]);
      ln_st<V>(p + cols + c0, valid[k], gb[k]);
    }
  }
}

// dw / db [cols] = Σ over the nblk partials, in block order within each of 64
// slices and slice order after that (fixed, so the same bits every run).
// 16 columns x 64 slices per block: with 16 KiB-strided partials a thread adds
// nblk/64 values, and 128 columns still give 16 blocks.
template <typename W>
__global__ __launch_bounds__(1024) void k_ln_wgrad(const float* __restrict__ part, int nblk,
                                                   int cols, W* __restrict__ dw,
                                                   W* __restrict__ db, int accumulate) {
  __shared__ float sl[64][17];
  const int cc = threadIdx.x & 15, s = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + cc;  // over [0, 2·cols)
  float v = 0.f;
  if (c < 2 * cols) {
    const float* p = part + c;
#pragma unroll 4
    for (int i = s; i < nblk; i += 64) v += p[(int64_t)i * 2 * cols];
  }
  sl[s][cc] = v;
  __syncthreads();
  if (s == 0 && c < 2 * cols) {
    float tot = 0.f;
#pragma unroll
    for (int u = 0; u < 64; ++u) tot += sl[u][cc];
    W* o = c < cols ? dw : db;
    const int k = c < cols ? c : c - cols;
    if (o) o[k] = (W)(accumulate ? (float)o[k] + tot : tot);
  }
}

// Blocks of the backward (and so partials): enough rows per group that the
// partials stay a few per cent of the rows' bytes, at most two blocks of 256
// threads (one of 1,024) per CU.
static inline int ln_bwd_blocks(int64_t rows, int tpr) {
  const int groups = tpr < 256 ? 256 / tpr : 1;
  const int64_t need = (rows + groups - 1) / groups;
  const int64_t cap = tpr > 256 ? 256 : 512;
  return (int)std::min<int64_t>(std::max<int64_t>(need, 1), cap);
}

// threads per row for a row of nv 16-B vectors with at most `most` per thread
static inline int ln_tpr(int64_t nv, int most) {
  for (int t : {16, 32, 64, 256, 512})
    if (nv <= (int64_t)t * most) return t;
  return 1024;
}

template <typename T, typename W>
struct LnLaunch {
  static constexpr int V = LnVec<T>::V;
  static constexpr int MOST = 16 / V;
  const T* x;
  int64_t ldx;
  const W *w, *b;
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

  template <int TPR, int NPT>
  void go(bool fwd) const {
    constexpr int TH = ln_threads<TPR>();
    constexpr int GR = TH / TPR;
    if (fwd) {
      const int64_t need = (rows + GR - 1) / GR;
      const int grid = (int)std::min<int64_t>(need, TPR > 256 ? 1024 : 2048);
      hipLaunchKernelGGL((k_ln_fwd<T, W, TPR, NPT>), dim3(grid), dim3(TH), 0, stream, x, ldx, w, b,
                         rows, cols, eps, y, mean, rstd);
    } else {
      hipLaunchKernelGGL((k_ln_bwd<T, W, TPR, NPT>), dim3(ln_bwd_blocks(rows, TPR)), dim3(TH), 0,
                         stream, dy, lddy, x, ldx, w, cmean, crstd, rows, cols, dx, part);
    }
  }
  // NPT of the TPR chosen by ln_tpr; the smaller counts of a group belong to
  // the group below it, so only the reachable ones are instances
  void run(bool fwd) const {
    const int nv = (cols + V - 1) / V;
    const int tpr = ln_tpr(nv, MOST);
    const int npt = (nv + tpr - 1) / tpr;
    if constexpr (V == 4) {
      if (tpr == 16) {
        if (npt <= 1) go<16, 1>(fwd);
        else if (npt == 2) go<16, 2>(fwd);
        else if (npt == 3) go<16, 3>(fwd);
        else go<16, 4>(fwd);
      } else if (tpr == 32) {
        if (npt == 3) go<32, 3>(fwd); else go<32, 4>(fwd);
      } else if (tpr == 64) {
        if (npt == 3) go<64, 3>(fwd); else go<64, 4>(fwd);
      } else if (tpr == 256) {
        if (npt == 2) go<256, 2>(fwd);
        else if (npt == 3) go<256, 3>(fwd);
        else go<256, 4>(fwd);
      } else if (tpr == 512) {
        if (npt == 3) go<512, 3>(fwd); else go<512, 4>(fwd);
      } else {
        if (npt == 3) go<1024, 3>(fwd); else go<1024, 4>(fwd);
      }
    } else {
      if (tpr == 16) {
        if (npt <= 1) go<16, 1>(fwd); else go<16, 2>(fwd);
      } else if (tpr == 32) {
        go<32, 2>(fwd);
      } else if (tpr == 64) {
        go<64, 2>(fwd);
      } else if (tpr == 256) {
        if (npt == 1) go<256, 1>(fwd); else go<256, 2>(fwd);
      } else if (tpr == 512) {
        go<512, 2>(fwd);
      } else {
        go<1024, 2>(fwd);
      }
    }
  }
};

template <typename W>
static int ln_wgrad(const float* part, int nblk, int cols, void* dw, void* db, int accumulate,
                    hipStream_t stream) {
  hipLaunchKernelGGL((k_ln_wgrad<W>), dim3((2 * cols + 15) / 16), dim3(1024), 0, stream, part,
                     nblk, cols, (W*)dw, (W*)db, accumulate);
  return (int)hipGetLastError();
}

static inline bool ln_types_ok(int dtype, int wdtype) {
  return dtype >= SV2N_DT_F32 && dtype <= SV2N_DT_F16 &&
         (wdtype == SV2N_DT_F32 || wdtype == dtype);
}
static inline int ln_bytes(int dtype) { return dtype == SV2N_DT_F32 ? 4 : 2; }

template <typename F>
static int ln_dispatch(int dtype, int wdtype, F&& f) {
  if (dtype == SV2N_DT_F32) return f((float*)nullptr, (float*)nullptr);
  if (dtype == SV2N_DT_BF16)
    return wdtype == SV2N_DT_F32 ? f((__bf16*)nullptr, (float*)nullptr)
                                 : f((__bf16*)nullptr, (__bf16*)nullptr);
  return wdtype == SV2N_DT_F32 ? f((_Float16*)nullptr, (float*)nullptr)
                               : f((_Float16*)nullptr, (_Float16*)nullptr);
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
  return ln_dispatch(dtype, wdtype, [&](auto* tp, auto* wp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    using W = std::remove_pointer_t<decltype(wp)>;
    LnLaunch<T, W> l{};
    l.x = (const T*)x; l.ldx = ldx; l.w = (const W*)weight; l.b = (const W*)bias;
    l.rows = rows; l.cols = cols; l.eps = eps; l.y = (T*)y; l.mean = mean; l.rstd = rstd;
    l.stream = stream;
    l.run(true);
    return (int)hipGetLastError();
  });
}

extern "C" int64_t sv2n_layer_norm_bwd_workspace(int64_t rows, int cols, int dtype) {
  if (rows <= 0 || cols <= 0 || cols > SV2N_LN_MAX_COLS || !ln_types_ok(dtype, dtype)) return 0;
  const int v = 16 / ln_bytes(dtype);
  return (int64_t)ln_bwd_blocks(rows, ln_tpr((cols + v - 1) / v, 16 / v)) * 2 * cols;
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
  return ln_dispatch(dtype, wdtype, [&](auto* tp, auto* wp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    using W = std::remove_pointer_t<decltype(wp)>;
    int nblk = 0;
    if (rows > 0) {
      LnLaunch<T, W> l{};
      l.x = (const T*)x; l.ldx = ldx; l.w = (const W*)weight; l.rows = rows; l.cols = cols;
      l.dy = (const T*)dy; l.lddy = lddy; l.cmean = mean; l.crstd = rstd; l.dx = (T*)dx;
      l.part = wg ? workspace : nullptr;
      l.stream = stream;
      l.run(false);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
      nblk = (int)(sv2n_layer_norm_bwd_workspace(rows, cols, dtype) / (2 * cols));
    }
    if (!wg) return 0;
    return ln_wgrad<W>(workspace, nblk, cols, dw, db, accumulate, stream);
  });
}
