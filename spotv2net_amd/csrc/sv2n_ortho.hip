// Orthogonalising a matrix by Newton-Schulz products, and the optimiser step
// (momentum, orthogonalised update, decoupled weight decay) built on it.
//
//   X_0 = G / max(|G|_F, eps)           (transposed if G has more rows than columns: m <= n)
//   S = X Xt [m][m];  Q = b S + c S S [m][m];  X <- a X + Q X [m][n]        (`steps` times)
//
// The products are nearly all of the work and run on the f16 matrix cores at f32
// accuracy: |X|_F = 1 bounds every singular value, the polynomial bounds them
// after each step, so X, S and Q have entries below known constants and are held
// as v·2^k = hi + lo, two f16 numbers with a power-of-two scale k per operand
// (22 bits; what the scale leaves below f16's range is under 2^-38 of the bound).
// A product keeps hi·hi + hi·lo + lo·hi in f32 accumulators: three f16 products
// at 1/3 of that peak each, where an exact f32 product has 1/16 of it.  Against
// 64 bits the result is as close as one of f32 products (the steps amplify any
// rounding of the input by up to a^steps, so fewer bits are not enough for f32).
//
// S and S S are symmetric: only tiles on and below the diagonal are computed and
// each is stored twice.  Every operand is stored with its K dimension contiguous
// (X for S, Xt for Q X), so one kernel with one staging scheme serves all three
// products; the epilogue writes X and Xt of the next step.
//
// Layout of an operand: [row][K/32][plane hi, lo][32 halves], rows and K padded
// with zeros to the tile: the 32 K values a stage needs of a row are one 128-B line.
//
// Several matrices (a model's weights) share each launch: `first` maps blocks to
// matrices, so a step over four weights costs the same 3·steps + 2 launches as one.
#include "sv2n_common.h"
#include <algorithm>
#include <cmath>

namespace sv2n {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int NS_MAX = 16;      // matrices of one launch
constexpr int NS_PARTS = 512;   // most partial sums of squares of one matrix
constexpr int NS_PART_ELEMS = 8192;

struct NsMat {
  const void* g;        // [batch][rows][ld] of dtype
  int64_t ld, g_batch;
  float* buf;           // momentum [rows][cols], or NULL (plain orthogonalisation)
  void* out;            // U [batch][rows][cols] of dtype; with buf: the weight, f32
  int rows, cols;       // as given
  int m, n, mp, np;     // m <= n, padded to the tile
  int batch, flip;      // flip: X = Gt
  int dtype;
  int parts, part_rows; // partial sums of squares per matrix, rows of each
  float lr;             // the update's factor (with buf)
  _Float16 *x, *xt[2], *s, *q;
  double* part;         // [batch][parts]
};
struct NsArgs {
  NsMat mat[NS_MAX];
  int first[NS_MAX + 1];
  int count;
};
struct NsScale {
  float a, b, c;
  int kx, ks, kq;       // X, S and Q are held times 2^k
  float eps;
  float momentum, fresh; // beta and 1 - beta
  int nesterov;
  float keep;           // 1 - lr·weight_decay
};

__device__ __forceinline__ int ns_find(const NsArgs& A, int b) {
  int i = 0;
  while (i + 1 < A.count && b >= A.first[i + 1]) ++i;
  return i;
}

__device__ __forceinline__ float ns_ld(const void* p, int64_t i, int dtype) {
  if (dtype == SV2N_DT_F32) return ((const float*)p)[i];
  if (dtype == SV2N_DT_BF16) return (float)((const __bf16*)p)[i];
  return (float)((const _Float16*)p)[i];
}

// halves offset of (row, k) of the hi plane in an operand of padded depth kp; lo: + 32
__device__ __forceinline__ int64_t ns_off(int64_t row, int k, int kp) {
  return row * (2 * (int64_t)kp) + ((k >> 5) << 6) + (k & 31);
}

// the matrix the products orthogonalise: G, or its momentum update
__device__ __forceinline__ float ns_update(const NsScale& sc, float g, float buf) {
  return sc.nesterov ? fmaf(sc.momentum, buf, sc.fresh * g) : buf;
}

// ---- 1: the momentum and the partial sums of squares (in 64 bits: an f32 square
// overflows above 2^64 and is lost below 2^-75) ----
__global__ __launch_bounds__(256) void k_ns_norm(NsArgs A, NsScale sc) {
  __shared__ double red[4];
  const int mi = ns_find(A, blockIdx.x);
  const NsMat& M = A.mat[mi];
  const int local = blockIdx.x - A.first[mi];
  const int b = local / M.parts, p = local - b * M.parts;
  // tx threads along a row, the rest down the rows
  int tx = 256;
  while (tx > 1 && tx / 2 >= M.cols) tx >>= 1;
  const int ty = 256 / tx;
  const int c0 = threadIdx.x % tx, r0 = threadIdx.x / tx;
  const int64_t rbeg = (int64_t)p * M.part_rows;
  const int64_t rend = min((int64_t)M.rows, rbeg + M.part_rows);
  const int64_t base = b * M.g_batch;
  double acc = 0.0;
  for (int64_t r = rbeg + r0; r < rend; r += ty) {
    for (int c = c0; c < M.cols; c += tx) {
      float v = ns_ld(M.g, base + r * M.ld + c, M.dtype);
      if (M.buf) {
        float* bp = M.buf + r * M.cols + c;
        const float nb = fmaf(sc.momentum, *bp, sc.fresh * v);
        *bp = nb;
        v = ns_update(sc, v, nb);
      }
      acc = fma((double)v, (double)v, acc);
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) acc += __shfl_xor(acc, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) M.part[(int64_t)b * M.parts + p] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ void ns_split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// ---- 2: X_0 and its transpose as planes, one 64 x 64 tile per block ----
__global__ __launch_bounds__(256) void k_ns_split(NsArgs A, NsScale sc) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int mi = ns_find(A, blockIdx.x);
  const NsMat& M = A.mat[mi];
  int local = blockIdx.x - A.first[mi];
  const int ti = M.mp / 64, tj = M.np / 64;
  const int b = local / (ti * tj);
  local -= b * ti * tj;
  const int i0 = (local / tj) * 64, j0 = (local % tj) * 64;
  // every block adds the matrix's partials in the same order
  double acc = 0.0;
  for (int k = threadIdx.x; k < M.parts; k += 256) acc += M.part[(int64_t)b * M.parts + k];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) acc += __shfl_xor(acc, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  // NaN stays NaN (fmax would drop it)
  const double den = norm < (double)sc.eps ? (double)sc.eps : norm;
  const double inv = ldexp(1.0, sc.kx) / den;
  const int64_t base = b * M.g_batch;
  const int r0 = M.flip ? j0 : i0, c0 = M.flip ? i0 : j0;
  const int c = threadIdx.x & 63;
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int r = (threadIdx.x >> 6) + 4 * k;
    float v = 0.f;
    if (r0 + r < M.rows && c0 + c < M.cols) {
      v = ns_ld(M.g, base + (int64_t)(r0 + r) * M.ld + c0 + c, M.dtype);
      if (M.buf) v = ns_update(sc, v, M.buf[(int64_t)(r0 + r) * M.cols + c0 + c]);
      v = (float)((double)v * inv);
    }
    if (M.flip) tile[c][r] = v; else tile[r][c] = v;
  }
  __syncthreads();
  _Float16* X = M.x + (int64_t)b * 2 * M.mp * M.np;
  _Float16* XT = M.xt[0] + (int64_t)b * 2 * M.mp * M.np;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const int u = h * 256 + threadIdx.x;       // 512 groups of 8 values, then the transpose's
    const int row = (u >> 3) & 63, k0 = (u & 7) * 8;
    f16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = u < 512 ? tile[row][k0 + e] : tile[k0 + e][row];
      _Float16 a, d;
      ns_split(v, a, d);
      hi[e] = a;
      lo[e] = d;
    }
    _Float16* o = u < 512 ? X + ns_off(i0 + row, j0 + k0, M.np)
                          : XT + ns_off(j0 + row, i0 + k0, M.mp);
    *(f16x8*)o = hi;
    *(f16x8*)(o + 32) = lo;
  }
}

// LDS written by the wave's lanes is read by its other lanes after this
__device__ __forceinline__ void ns_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

enum { NS_S = 0, NS_Q = 1, NS_X = 2, NS_LAST = 3 };

// Stores a wave's 32 x 32 tile of values (LDS, stride 33) as planes with row r0
// and column (K) c0: two lanes per row, 128 B of hi and lo each.  TR: the tile's
// transpose.
template <bool TR>
__device__ __forceinline__ void ns_store(const float* t, _Float16* dst, int64_t r0, int c0, int kp) {
  const int lane = threadIdx.x & 63;
  const int row = lane >> 1, k0 = (lane & 1) * 16;
  _Float16* o = dst + ns_off(r0 + row, c0 + k0, kp);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = k0 + h * 8 + e;
      _Float16 a, d;
      ns_split(TR ? t[k * 33 + row] : t[row * 33 + k], a, d);
      hi[e] = a;
      lo[e] = d;
    }
    *(f16x8*)(o + h * 8) = hi;
    *(f16x8*)(o + h * 8 + 32) = lo;
  }
}

// ---- 3: one product ----
// D[i][j] = sum_k P[i][k] R[j][k] over TB x TB tiles, 4 waves in a 2 x 2 grid of
// TB/2 x TB/2.  A stage is 32 K values of both planes (128 B a row), staged
// through registers into one of two LDS buffers: the next stage's loads are in
// flight while this one is multiplied, one barrier a stage.  16-B slots of a row
// are swapped by (row >> 1) & 7 so that the 16 rows a quarter wave reads fall on
// different banks.
//   NS_S:  P = R = X,        S = D             (i >= j tiles, stored twice)
//   NS_Q:  P = R = S,        Q = b S + c D     (the same)
//   NS_X:  P = Q, R = Xt,    X' = a X + D      (X' and its transpose)
//   NS_LAST: as NS_X, the result goes to the caller
template <int TB, int EPI>
__global__ __launch_bounds__(256, 2) void k_ns_gemm(NsArgs A, NsScale sc, int cur) {
  constexpr int WT = TB / 2, FT = WT / 32;
  constexpr int OPB = TB * 128;              // bytes of an operand's stage
  constexpr int LD = TB * 8 / 256;           // 16-B loads per thread and operand
  __shared__ __attribute__((aligned(16))) char lds[2 * 2 * OPB];
  const int mi = ns_find(A, blockIdx.x);
  const NsMat& M = A.mat[mi];
  int local = blockIdx.x - A.first[mi];
  const int tm = M.mp / TB, tn = M.np / TB;
  int ti, tj;
  int bt;
  if (EPI == NS_S || EPI == NS_Q) {
    const int per = tm * (tm + 1) / 2;
    bt = local / per;
    local -= bt * per;
    ti = (int)((sqrtf(8.f * (float)local + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > local) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= local) ++ti;
    tj = local - ti * (ti + 1) / 2;
  } else {
    const int per = tm * tn;
    bt = local / per;
    local -= bt * per;
    ti = local % tm;
    tj = local / tm;
  }
  const int i0 = ti * TB, j0 = tj * TB;
  const int64_t xs = (int64_t)bt * 2 * M.mp * M.np, ss = (int64_t)bt * 2 * M.mp * M.mp;
  const int kp = EPI == NS_S ? M.np : M.mp;
  const _Float16* P = (EPI == NS_S ? M.x + xs : EPI == NS_Q ? M.s + ss : M.q + ss);
  const _Float16* R = (EPI == NS_S ? M.x + xs : EPI == NS_Q ? M.s + ss : M.xt[cur] + xs);

  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int wi = (wave >> 1) * WT, wj = (wave & 1) * WT;
  const char* gp[LD];
  const char* gr[LD];
#pragma unroll
  for (int l = 0; l < LD; ++l) {
    const int q = l * 256 + t, row = q >> 3, g = (q & 7) ^ ((row >> 1) & 7);
    gp[l] = (const char*)P + (int64_t)(i0 + row) * kp * 4 + g * 16;
    gr[l] = (const char*)R + (int64_t)(j0 + row) * kp * 4 + g * 16;
  }
  u32x4 sp[LD], sr[LD];
  auto fetch = [&](int st) {
#pragma unroll
    for (int l = 0; l < LD; ++l) {
      sp[l] = *(const u32x4*)(gp[l] + (int64_t)st * 128);
      sr[l] = *(const u32x4*)(gr[l] + (int64_t)st * 128);
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int l = 0; l < LD; ++l) {
      *(u32x4*)(lds + buf * 2 * OPB + (l * 256 + t) * 16) = sp[l];
      *(u32x4*)(lds + buf * 2 * OPB + OPB + (l * 256 + t) * 16) = sr[l];
    }
  };
  f32x16 acc[FT][FT];
#pragma unroll
  for (int x = 0; x < FT; ++x)
#pragma unroll
    for (int y = 0; y < FT; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;

  auto frag = [&](int buf, int op, int row, int plane, int ks) {
    const int slot = (plane * 4 + ks * 2 + (lane >> 5)) ^ ((row >> 1) & 7);
    return *(const f16x8*)(lds + buf * 2 * OPB + op * OPB + row * 128 + slot * 16);
  };
  const int nst = kp / 32;
  fetch(0);
  put(0);
  __syncthreads();
  for (int st = 0; st < nst; ++st) {
    const int buf = st & 1;
    if (st + 1 < nst) fetch(st + 1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      f16x8 ah[FT], al[FT], bh[FT], bl[FT];
#pragma unroll
      for (int x = 0; x < FT; ++x) {
        const int ra = wi + x * 32 + (lane & 31), rb = wj + x * 32 + (lane & 31);
        ah[x] = frag(buf, 0, ra, 0, ks);
        bh[x] = frag(buf, 1, rb, 0, ks);
        al[x] = frag(buf, 0, ra, 1, ks);
        bl[x] = frag(buf, 1, rb, 1, ks);
      }
#pragma unroll
      for (int x = 0; x < FT; ++x)
#pragma unroll
        for (int y = 0; y < FT; ++y) {
          acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[x], bh[y], acc[x][y], 0, 0, 0);
          acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[x], bl[y], acc[x][y], 0, 0, 0);
          acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[x], bh[y], acc[x][y], 0, 0, 0);
        }
    }
    if (st + 1 < nst) put(buf ^ 1);
    __syncthreads();
  }

  // epilogue: lane holds column j = lane & 31 and, in fours, rows i of each tile
  float* tile = (float*)lds + wave * 32 * 33;
  const float up_s = ldexpf(1.f, sc.ks - 2 * sc.kx);           // D of X Xt -> S's scale
  const float up_q = sc.c * ldexpf(1.f, sc.kq - 2 * sc.ks);    // c·D of S S -> Q's scale
  const float up_b = sc.b * ldexpf(1.f, sc.kq - sc.ks);
  const float up_x = ldexpf(1.f, -sc.kq);                      // D of Q X -> X's scale
#pragma unroll
  for (int x = 0; x < FT; ++x)
#pragma unroll
    for (int y = 0; y < FT; ++y) {
      const int ib = i0 + wi + x * 32, jb = j0 + wj + y * 32;
      const int il = 4 * (lane >> 5), jl = lane & 31;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        f16x4 ph, pl;
        if (EPI != NS_S) {
          // the old S or X at [i..i+3][j]: four values in a row of the (symmetric)
          // S, or of Xt
          const _Float16* o = R + ns_off(jb + jl, ib + 8 * r4 + il, kp);
          ph = *(const f16x4*)o;
          pl = *(const f16x4*)(o + 32);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = acc[x][y][r4 * 4 + e];
          if (EPI == NS_S) {
            v *= up_s;
          } else {
            const float old = (float)ph[e] + (float)pl[e];
            if (EPI == NS_Q) v = fmaf(up_q, v, up_b * old);
            else v = fmaf(up_x, v, sc.a * old);
          }
          tile[(8 * r4 + il + e) * 33 + jl] = v;
        }
      }
      ns_wave_sync();  // the tile is the wave's own
      if (EPI == NS_S || EPI == NS_Q) {
        _Float16* D = (EPI == NS_S ? M.s : M.q) + ss;
        ns_store<false>(tile, D, ib, jb, M.mp);
        if (ti != tj) ns_store<true>(tile, D, jb, ib, M.mp);
      } else if (EPI == NS_X) {
        ns_store<false>(tile, M.x + xs, ib, jb, M.np);
        ns_store<true>(tile, M.xt[cur ^ 1] + xs, jb, ib, M.mp);
      } else {
        const float down = ldexpf(1.f, -sc.kx);
        const float f = M.buf ? -M.lr * down : down;
        // along the caller's rows: 32 lanes a row, two rows at a time
#pragma unroll 4
        for (int p = 0; p < 16; ++p) {
          const int u = 2 * p + (lane >> 5), v = lane & 31;
          const int i = M.flip ? ib + v : ib + u, j = M.flip ? jb + u : jb + v;
          if (i >= M.m || j >= M.n) continue;
          const float val = f * (M.flip ? tile[v * 33 + u] : tile[u * 33 + v]);
          const int64_t o = (int64_t)bt * M.rows * M.cols +
                            (M.flip ? (int64_t)j * M.cols + i : (int64_t)i * M.cols + j);
          if (M.buf) {
            float* w = (float*)M.out + o;
            *w = fmaf(sc.keep, *w, val);
          } else if (M.dtype == SV2N_DT_F32) {
            ((float*)M.out)[o] = val;
          } else if (M.dtype == SV2N_DT_BF16) {
            ((__bf16*)M.out)[o] = (__bf16)val;
          } else {
            ((_Float16*)M.out)[o] = (_Float16)val;
          }
        }
      }
      ns_wave_sync();
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static inline int64_t ns_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// Largest |f| of f(x) = x·p(x²) and of q(λ) = b λ + c λ² over [0, hi]: both are
// smooth, so a grid and the polynomials' own stationary points settle it.
static void ns_bounds(double a, double b, double c, double hi, double* f_max, double* q_max) {
  auto f = [&](double x) { return std::fabs(x * (a + b * x * x + c * x * x * x * x)); };
  auto q = [&](double l) { return std::fabs(b * l + c * l * l); };
  double fm = f(hi), qm = q(hi * hi);
  // f' = a + 3 b y + 5 c y² at y = x²
  const double dis = 9 * b * b - 20 * a * c;
  if (c != 0.0) {
    if (dis >= 0.0)
      for (double s : {-1.0, 1.0}) {
        const double y = (-3 * b + s * std::sqrt(dis)) / (10 * c);
        if (y > 0.0 && y < hi * hi) fm = std::max(fm, f(std::sqrt(y)));
      }
    const double l = -b / (2 * c);
    if (l > 0.0 && l < hi * hi) qm = std::max(qm, q(l));
  } else if (b != 0.0) {
    const double y = -a / (3 * b);
    if (y > 0.0 && y < hi * hi) fm = std::max(fm, f(std::sqrt(y)));
  }
  *f_max = fm;
  *q_max = qm;
}

// The power-of-two scales of X, S and Q from the largest singular value any step
// can reach; false if the coefficients let them grow past 2^8.
static bool ns_scales(int steps, NsScale* sc) {
  double top = 1.0, hi = 1.0, qm = 0.0;
  for (int k = 0; k < steps; ++k) {
    double f, q;
    ns_bounds(sc->a, sc->b, sc->c, hi, &f, &q);
    qm = std::max(qm, q);
    top = std::max(top, f);
    hi = f;
    if (!(top <= 256.0) || !(qm <= 65536.0)) return false;
    if (hi == 0.0) break;
  }
  auto fit = [](double v) {  // largest k <= 14 with v·2^k <= 2^15
    int e;
    std::frexp(std::max(v, 1e-30), &e);  // v < 2^e
    return std::min(14, 15 - e);
  };
  sc->kx = fit(top);
  sc->ks = fit(top * top);
  sc->kq = fit(qm);
  return true;
}

// Tile of a group of matrices: 128 where that leaves at least 128 blocks for X's
// product, else 64 (more blocks, each with half the K-loop's work per stage)
static int ns_tile(const NsMat* mats, int count) {
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i)
    blocks += (int64_t)mats[i].batch * (ns_up(mats[i].m, 128) / 128) * (ns_up(mats[i].n, 128) / 128);
  return blocks >= 128 ? 128 : 64;
}

static void ns_shape(NsMat* M) {
  M->flip = M->rows > M->cols;
  M->m = std::min(M->rows, M->cols);
  M->n = std::max(M->rows, M->cols);
  int64_t pr = (NS_PART_ELEMS + M->cols - 1) / M->cols;
  pr = std::max<int64_t>(pr, (M->rows + NS_PARTS - 1) / NS_PARTS);
  M->part_rows = (int)std::min<int64_t>(pr, M->rows);
  M->parts = (M->rows + M->part_rows - 1) / M->part_rows;
}

// pads the shapes for the group's tile and lays its workspace out from `ws`
// (NULL: only counts); returns the bytes
static int64_t ns_plan(NsMat* mats, int count, int tile, char* ws) {
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    char* p = ws ? ws + off : nullptr;
    off += ns_up(bytes, 256);
    return p;
  };
  for (int i = 0; i < count; ++i) {
    NsMat& M = mats[i];
    M.mp = (int)ns_up(M.m, tile);
    M.np = (int)ns_up(M.n, tile);
    const int64_t xb = (int64_t)M.batch * M.mp * M.np * 4, sb = (int64_t)M.batch * M.mp * M.mp * 4;
    M.part = (double*)take((int64_t)M.batch * M.parts * 8);
    M.x = (_Float16*)take(xb);
    M.xt[0] = (_Float16*)take(xb);
    M.xt[1] = (_Float16*)take(xb);
    M.s = (_Float16*)take(sb);
    M.q = (_Float16*)take(sb);
  }
  return off;
}

template <typename F>
static int64_t ns_blocks(NsArgs& A, F&& per) {
  int64_t n = 0;
  for (int i = 0; i < A.count; ++i) {
    A.first[i] = (int)n;
    n += per(A.mat[i]) * A.mat[i].batch;
  }
  A.first[A.count] = (int)n;
  return n;
}

template <int TB, int EPI>
static void ns_gemm(NsArgs& A, const NsScale& sc, int cur, hipStream_t stream) {
  const int64_t n = ns_blocks(A, [](const NsMat& M) -> int64_t {
    const int64_t tm = M.mp / TB, tn = M.np / TB;
    return EPI == NS_S || EPI == NS_Q ? tm * (tm + 1) / 2 : tm * tn;
  });
  hipLaunchKernelGGL((k_ns_gemm<TB, EPI>), dim3((unsigned)n), dim3(256), 0, stream, A, sc, cur);
}

template <int TB>
static void ns_steps(NsArgs& A, const NsScale& sc, int steps, hipStream_t stream) {
  for (int s = 0; s < steps; ++s) {
    const int cur = s & 1;
    ns_gemm<TB, NS_S>(A, sc, cur, stream);
    ns_gemm<TB, NS_Q>(A, sc, cur, stream);
    if (s + 1 < steps) ns_gemm<TB, NS_X>(A, sc, cur, stream);
    else ns_gemm<TB, NS_LAST>(A, sc, cur, stream);
  }
}

static int ns_run(NsArgs& A, const NsScale& sc, int steps, int tile, hipStream_t stream) {
  int64_t n = ns_blocks(A, [](const NsMat& M) -> int64_t { return M.parts; });
  hipLaunchKernelGGL(k_ns_norm, dim3((unsigned)n), dim3(256), 0, stream, A, sc);
  n = ns_blocks(A, [](const NsMat& M) -> int64_t { return (int64_t)(M.mp / 64) * (M.np / 64); });
  hipLaunchKernelGGL(k_ns_split, dim3((unsigned)n), dim3(256), 0, stream, A, sc);
  if (tile == 128) ns_steps<128>(A, sc, steps, stream);
  else ns_steps<64>(A, sc, steps, stream);
  return (int)hipGetLastError();
}

static inline bool ns_size_ok(int64_t batch, int64_t rows, int64_t cols) {
  return batch >= 1 && rows >= 1 && cols >= 1 && rows <= SV2N_NS_MAX_SIDE &&
         cols <= SV2N_NS_MAX_SIDE && batch <= SV2N_NS_MAX_BATCH;
}
static inline bool ns_coef_ok(int steps, float a, float b, float c, float eps) {
  return steps >= 1 && steps <= SV2N_NS_MAX_STEPS && std::isfinite(a) && std::isfinite(b) &&
         std::isfinite(c) && eps > 0.f && std::isfinite(eps);
}

}  // namespace sv2n

using namespace sv2n;

extern "C" int64_t sv2n_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols) {
  if (!ns_size_ok(batch, rows, cols)) return 0;
  NsMat M{};
  M.rows = (int)rows;
  M.cols = (int)cols;
  M.batch = (int)batch;
  ns_shape(&M);
  return ns_plan(&M, 1, ns_tile(&M, 1), nullptr);
}

extern "C" int sv2n_orthogonalize(const void* g, int64_t ld, int64_t batch_stride, int dtype,
                                  int64_t batch, int64_t rows, int64_t cols, int steps, float a,
                                  float b, float c, float eps, void* out, void* workspace,
                                  int64_t workspace_bytes, hipStream_t stream) {
  if (!g || !out || dtype < SV2N_DT_F32 || dtype > SV2N_DT_F16 || !ns_coef_ok(steps, a, b, c, eps))
    return SV2N_ERR_ARG;
  if (!ns_size_ok(batch, rows, cols) || ld < cols || batch_stride < 0) return SV2N_ERR_SHAPE;
  const int es = dtype == SV2N_DT_F32 ? 4 : 2;
  if (((uintptr_t)g | (uintptr_t)out) & (es - 1)) return SV2N_ERR_ALIGN;
  NsArgs A{};
  NsScale sc{};
  sc.a = a; sc.b = b; sc.c = c; sc.eps = eps;
  if (!ns_scales(steps, &sc)) return SV2N_ERR_ARG;
  NsMat& M = A.mat[0];
  A.count = 1;
  M.g = g; M.ld = ld; M.g_batch = batch_stride; M.out = out; M.dtype = dtype;
  M.rows = (int)rows; M.cols = (int)cols; M.batch = (int)batch;
  ns_shape(&M);
  const int tile = ns_tile(&M, 1);
  if (!workspace || workspace_bytes < ns_plan(&M, 1, tile, nullptr)) return SV2N_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 255) return SV2N_ERR_ALIGN;
  ns_plan(&M, 1, tile, (char*)workspace);
  return ns_run(A, sc, steps, tile, stream);
}

// fills one group of at most NS_MAX matrices
static void ns_group(const sv2n_muon_matrix* mats, int count, double lr, NsArgs* A) {
  A->count = count;
  for (int i = 0; i < count; ++i) {
    NsMat& M = A->mat[i];
    M = NsMat{};
    M.g = mats[i].grad;
    M.buf = mats[i].momentum;
    M.out = mats[i].weight;
    M.rows = mats[i].rows;
    M.cols = mats[i].cols;
    M.ld = M.cols;
    M.batch = 1;
    M.dtype = SV2N_DT_F32;
    M.lr = (float)(lr * (double)mats[i].lr_scale);
    ns_shape(&M);
  }
}

extern "C" int64_t sv2n_muon_step_workspace(const sv2n_muon_matrix* mats, int count) {
  if (!mats || count <= 0) return 0;
  int64_t most = 0;
  for (int k = 0; k < count; k += NS_MAX) {
    const int n = std::min(NS_MAX, count - k);
    for (int i = 0; i < n; ++i)
      if (!ns_size_ok(1, mats[k + i].rows, mats[k + i].cols)) return 0;
    NsArgs A{};
    ns_group(mats + k, n, 0.0, &A);
    most = std::max(most, ns_plan(A.mat, n, ns_tile(A.mat, n), nullptr));
  }
  return most;
}

extern "C" int sv2n_muon_step(const sv2n_muon_matrix* mats, int count, double lr, double momentum,
                              int nesterov, double weight_decay, int steps, float a, float b,
                              float c, float eps, void* workspace, int64_t workspace_bytes,
                              hipStream_t stream) {
  if (count == 0) return 0;
  if (!mats || count < 0 || !ns_coef_ok(steps, a, b, c, eps) || !std::isfinite(lr) ||
      !(momentum >= 0.0 && momentum < 1.0) || !std::isfinite(weight_decay))
    return SV2N_ERR_ARG;
  for (int i = 0; i < count; ++i) {
    const sv2n_muon_matrix& M = mats[i];
    if (!M.weight || !M.grad || !M.momentum || !std::isfinite(M.lr_scale)) return SV2N_ERR_ARG;
    if (!ns_size_ok(1, M.rows, M.cols)) return SV2N_ERR_SHAPE;
    if (((uintptr_t)M.weight | (uintptr_t)M.grad | (uintptr_t)M.momentum) & 3)
      return SV2N_ERR_ALIGN;
  }
  NsScale sc{};
  sc.a = a; sc.b = b; sc.c = c; sc.eps = eps;
  sc.momentum = (float)momentum;
  sc.fresh = (float)(1.0 - momentum);
  sc.nesterov = nesterov != 0;
  sc.keep = (float)(1.0 - lr * weight_decay);
  if (!ns_scales(steps, &sc)) return SV2N_ERR_ARG;
  if (!workspace || workspace_bytes < sv2n_muon_step_workspace(mats, count))
    return SV2N_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 255) return SV2N_ERR_ALIGN;
  for (int k = 0; k < count; k += NS_MAX) {
    const int n = std::min(NS_MAX, count - k);
    NsArgs A{};
    ns_group(mats + k, n, lr, &A);
    const int tile = ns_tile(A.mat, n);
    ns_plan(A.mat, n, tile, (char*)workspace);
    const int rc = ns_run(A, sc, steps, tile, stream);
    if (rc) return rc;
  }
  return 0;
}
