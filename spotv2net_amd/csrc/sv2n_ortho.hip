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
// 64 bits the result as a whole is as close as one of f32 products (the steps amplify
// any rounding of the input by up to a^steps, so fewer bits are not enough for f32).
//
// Two cases take f32 operands and v_mfma_f32_32x32x2_f32 instead:
// - The smaller side is at most 32: the sums are so short that those 22 bits would be
//   the largest error, up to 3.6 times that of f32 products, and the work is next to
//   nothing.
// - What the pairs leave out could become a visible part of the result (ns_pairs_ok):
//   rows or columns far below the others under many steps (64 x 128, half of the rows
//   times 1e-8, 16 steps: 3.6e-3 off in pairs, 2.7e-6 in f32), or coefficients that
//   shrink X.  A step takes 1.1 (128 x 1,024), 1.8 (777 x 1,537) to 4.0 (4,096²) times
//   as long as on pairs.
//
// S and S S are symmetric: only tiles on and below the diagonal are computed and
// each is stored twice.  Every operand is stored with its K dimension contiguous
// (X for S, Xt for Q X), so one kernel with one staging scheme serves all three
// products; the epilogue writes X and Xt of the next step.
//
// Layout of an operand: MFMA fragments in order.  A block of 32 rows x 16 K values
// is 64 lanes x 8 halves (1 KiB) as v_mfma_f32_32x32x16_f16 reads it, hi plane then
// lo, blocks along K next to each other, rows and K padded with zeros: a wave's
// fragment is one contiguous KiB, from memory or LDS alike (no bank conflicts, no
// swizzle).  Inside the 16 K values lane half h holds k = 4h..4h+3 and 8+4h..8+4h+3
// (every operand agrees, so the sums do not care): that is how the accumulators
// hold a tile's rows, so the tile's transpose goes back to memory as the next
// product's fragments straight from registers.
//
// Several matrices (a model's weights) share each launch: `first` maps blocks to
// matrices, so four weights cost as many launches as one: two, and three to six a step
// (a product whose last tiles of 128 fill no round takes a second one, ns_product).
// Small and thin matrices take fewer (k_ns_qx, k_ns_thin), thin ones beside large ones
// add one and one a step.
#include "sv2n_common.h"
#include <algorithm>
#include <cmath>

namespace sv2n {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int NS_MAX = 16;      // matrices of one launch
constexpr int NS_PARTS = 1024;  // most partial sums of squares of one matrix
constexpr int NS_PART_ELEMS = 4096;
constexpr int NS_THIN_COLS = 128;  // columns of a thin matrix a block keeps
constexpr int NS_EXACT = 32;    // smaller sides up to which the products are always f32
// The bounds between variants; us of the whole five steps, in a captured graph.
// Length from which thin matrices beside small ones get launches of their own.  16 x n
// beside 128 x 128, riding along / own: n 1,024 94 / 104, 1,408 103 / 107, 1,536 110 / 105,
// 4,096 196 / 117 (beside six of 64 x 64, or 400 x 300 and 200 x 400, they cross there too).
constexpr int NS_THIN_LONG = 1408;
// Tiles of 128 that are worth a round of their own (else they are cut into tiles of 64).
// n² at 48 / 128 / 256: 1,300 (121 tiles) 471 / 265 / 263, 2,300 (324, 68 left over)
// 996 / 975 / 1,069, 2,700 (484, 228 left over) 1,308 / 1,305 / 1,752.
constexpr int NS_HALF = 128;
// Tiles of 32 of X up to which blocks make their own rows of Q.  128 x n, own / a launch
// for Q: 16 tiles 69 / 73, 256 97 / 101, 512 134 / 133, 752 172 / 166, 2,048 373 / 321.
constexpr int NS_FUSED = 512;
// Tiles of 64 of a product below which tiles of 32 are faster, 32 / 64: 400 x 400 (28 of
// S, 49 of X) 91 / 116, 704² (66, 121) 137 / 155, 768² (78, 144) 174 / 158, 1,024² (136,
// 256) 265 / 184.
constexpr int NS_TINY = 72;
// Depth of X's product from which tiles of 128 are worth it, 128 / 64: 1,024 x 2,048
// 291 / 252, 1,152 x 2,048 309 / 304, 1,260 x 3,000 394 / 406, 1,792² 545 / 604, 2,048 x
// 8,192 1,974 / 2,409.
constexpr int NS_DEEP = 1200;

struct NsMat {
  const void* g;        // [batch][rows][ld] of dtype
  int64_t ld, g_batch;
  float* buf;           // momentum [rows][cols], or NULL (plain orthogonalisation)
  void* out;            // U [batch][rows][cols] of dtype; with buf: the weight, f32
  int rows, cols;       // as given
  int m, n, mp, np;     // m <= n, padded to the tile
  int batch, flip;      // flip: X = Gt
  int dtype;
  int exact;            // f32 operands and products
  int parts, part_elems; // partial sums of squares per matrix, elements of each
  float lr;             // the update's factor (with buf)
  _Float16 *x, *xt[2], *s, *q;
  double* part;         // [batch][parts]
  float* thin;          // k_ns_thin's partial S [2][batch][np / NS_THIN_COLS][1024], or NULL
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

// halves from an operand's start to the hi fragment block of rows 32·r32.., K values
// 16·k16.. of depth kp; the lo block follows it
__device__ __forceinline__ int64_t ns_blk(int64_t r32, int k16, int kp) {
  return (r32 * (kp >> 4) + k16) << 10;
}
// the 16 K values of a block that lane half h holds, in register order
__device__ __forceinline__ int ns_k(int h, int e) { return ((e & 4) << 1) + 4 * h + (e & 3); }

// the matrix the products orthogonalise: G, or its momentum update
__device__ __forceinline__ float ns_update(const NsScale& sc, float g, float buf) {
  return sc.nesterov ? fmaf(sc.momentum, buf, sc.fresh * g) : buf;
}

// ---- 1: the momentum and the partial sums of squares (in 64 bits: an f32 square
// overflows above 2^64 and is lost below 2^-75) ----
// A block takes part_elems elements of a matrix, 16 B a thread and load where the rows
// are dense and aligned, else one by one.
template <typename T>
__global__ __launch_bounds__(256) void k_ns_norm(NsArgs A, NsScale sc) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ double red[4];
  const int mi = ns_find(A, blockIdx.x);
  const NsMat& M = A.mat[mi];
  const int local = blockIdx.x - A.first[mi];
  const int b = local / M.parts, p = local - b * M.parts;
  const int total = M.rows * M.cols;
  const int beg = p * M.part_elems, end = min(total, beg + M.part_elems);
  const T* g = (const T*)M.g + b * M.g_batch;
  float* buf = M.buf;
  double acc = 0.0;
  auto take = [&](float v, float* bp) {
    if (bp) {
      const float nb = fmaf(sc.momentum, *bp, sc.fresh * v);
      *bp = nb;
      v = ns_update(sc, v, nb);
    }
    acc = fma((double)v, (double)v, acc);
  };
  const bool vec = M.ld == M.cols && (((uintptr_t)g | (uintptr_t)buf) & 15) == 0;
  int e = beg;
  if (vec) {
    // (beg is a multiple of 8)
#pragma unroll 4
    for (int i = beg + (int)threadIdx.x * V; i + V <= end; i += 256 * V) {
      T t[V];
      __builtin_memcpy(t, __builtin_assume_aligned(g + i, 16), 16);
      float bv[V];
      if (buf) {
        __builtin_memcpy(bv, __builtin_assume_aligned(buf + i, 16), sizeof(bv));
#pragma unroll
        for (int j = 0; j < V; ++j) take((float)t[j], &bv[j]);
        __builtin_memcpy(__builtin_assume_aligned(buf + i, 16), bv, sizeof(bv));
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) take((float)t[j], nullptr);
      }
    }
    e = beg + (end - beg) / V * V;
  }
#pragma unroll 4
  for (int i = e + (int)threadIdx.x; i < end; i += 256) {
    const int r = i / M.cols, c = i - r * M.cols;
    take((float)g[r * M.ld + c], buf ? buf + i : nullptr);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) acc += __shfl_xor(acc, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) M.part[(int64_t)b * M.parts + p] = (red[0] + red[1]) + (red[2] + red[3]);
}

// A lane's 8 values of a fragment block as they are stored, and back: the hi and lo f16
// planes, or (exact) the first and the last four as f32
__device__ __forceinline__ void ns_pack(const float (&v)[8], bool exact, f16x8& hi, f16x8& lo) {
  if (exact) {
    hi = __builtin_bit_cast(f16x8, f32x4{v[0], v[1], v[2], v[3]});
    lo = __builtin_bit_cast(f16x8, f32x4{v[4], v[5], v[6], v[7]});
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[e] = (_Float16)v[e];
      lo[e] = (_Float16)(v[e] - (float)hi[e]);
    }
  }
}
__device__ __forceinline__ void ns_unpack(f16x8 hi, f16x8 lo, bool exact, float (&v)[8]) {
  if (exact) {
    const f32x4 a = __builtin_bit_cast(f32x4, hi), b = __builtin_bit_cast(f32x4, lo);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)hi[e] + (float)lo[e];
  }
}

// ---- 2: X_0 and its transpose as planes, one 64 x 64 tile per block ----
template <typename T>
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
  // the tile's elements first: their loads are in flight while the norm is added up
  const T* g = (const T*)M.g + b * M.g_batch;
  const int r0 = M.flip ? j0 : i0, c0 = M.flip ? i0 : j0;
  const int c = threadIdx.x & 63, rq = threadIdx.x >> 6;
  float v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = r0 + rq + 4 * k;
    v[k] = r < M.rows && c0 + c < M.cols ? (float)g[(int64_t)r * M.ld + c0 + c] : 0.f;
  }
  if (M.buf) {
    float m[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int r = r0 + rq + 4 * k;
      m[k] = r < M.rows && c0 + c < M.cols ? M.buf[(int64_t)r * M.cols + c0 + c] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = ns_update(sc, v[k], m[k]);
  }
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
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = rq + 4 * k;
    const float x = (float)((double)v[k] * inv);
    if (M.flip) tile[c][r] = x; else tile[r][c] = x;
  }
  __syncthreads();
  _Float16* X = M.x + (int64_t)b * 2 * M.mp * M.np;
  _Float16* XT = M.xt[0] + (int64_t)b * 2 * M.mp * M.np;
  // 8 fragment blocks of X (2 row groups x 4), then 8 of its transpose
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = threadIdx.x >> 6; u < 16; u += 4) {
    const bool tr = u >= 8;
    const int rg = (u >> 2) & 1, kg = u & 3;
    const int row = rg * 32 + (lane & 31);
    f16x8 hi, lo;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = kg * 16 + ns_k(lane >> 5, e);
      f[e] = tr ? tile[k][row] : tile[row][k];
    }
    ns_pack(f, M.exact, hi, lo);
    _Float16* o = tr ? XT + ns_blk(j0 / 32 + rg, i0 / 16 + kg, M.mp)
                     : X + ns_blk(i0 / 32 + rg, j0 / 16 + kg, M.np);
    *(f16x8*)(o + lane * 8) = hi;
    *(f16x8*)(o + 512 + lane * 8) = lo;
  }
}

// LDS written by the wave's lanes is read by its other lanes after this
__device__ __forceinline__ void ns_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

enum { NS_S = 0, NS_Q = 1, NS_X = 2, NS_LAST = 3 };

// What a product computes; D = P Rt, 32 x 32 tiles [i][j]
//   NS_S:  P = R = X,        S = D             (i >= j tiles, stored twice)
//   NS_Q:  P = R = S,        Q = b S + c D     (the same)
//   NS_X:  P = Q, R = Xt,    X' = a X + D      (X' and its transpose)
//   NS_LAST: as NS_X, the result goes to the caller
struct NsOut {
  float up, old;        // new value = up·D + old·(the old S or X there)
  float down;           // NS_LAST: to the caller's scale
};
template <int EPI>
__device__ __forceinline__ NsOut ns_out(const NsScale& sc, const NsMat& M) {
  NsOut o;
  o.old = 0.f;
  o.down = 0.f;
  if (EPI == NS_S) {
    o.up = ldexpf(1.f, sc.ks - 2 * sc.kx);
  } else if (EPI == NS_Q) {
    o.up = sc.c * ldexpf(1.f, sc.kq - 2 * sc.ks);
    o.old = sc.b * ldexpf(1.f, sc.kq - sc.ks);
  } else {
    o.up = ldexpf(1.f, -sc.kq);
    o.old = sc.a;
    o.down = ldexpf(1.f, -sc.kx) * (M.buf ? -M.lr : 1.f);
  }
  return o;
}

// One 32 x 32 tile of D (accumulator layout: lane & 31 the column j, and rows
// i = 8·(e/4) + 4·(lane/32) + e%4) at rows ib, columns jb: the new values, stored
// where the next product reads them.  `tile`: 32 x 33 floats of the wave's own LDS,
// for the orientation that registers do not give.
template <int EPI>
__device__ __forceinline__ void ns_epilogue(const f32x16& d, const NsOut& o, const NsMat& M,
                                            const NsScale& sc, const _Float16* R, int64_t bt,
                                            int ib, int jb, int cur, bool mirror, float* tile) {
  const int lane = threadIdx.x & 63, h = lane >> 5, jl = lane & 31;
  const int64_t xs = bt * 2 * M.mp * M.np, ss = bt * 2 * M.mp * M.mp;
  float v[16];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    float old[8];
    if (EPI != NS_S) {
      // the old S or X at [i][j]: R's fragment of row j (S is symmetric, R = Xt)
      const _Float16* p = R + ns_blk(jb >> 5, (ib >> 4) + g, M.mp) + lane * 8;
      ns_unpack(*(const f16x8*)p, *(const f16x8*)(p + 512), M.exact, old);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = d[g * 8 + e] * o.up;
      if (EPI != NS_S) x = fmaf(o.old, old[e], x);
      v[g * 8 + e] = x;
    }
  }
  if (EPI == NS_LAST) {
    const int64_t base = bt * M.rows * M.cols;
    if (M.flip) {
      // the caller's rows are j: through LDS, so that lanes run along i
#pragma unroll
      for (int e = 0; e < 16; ++e) tile[(8 * (e >> 2) + 4 * h + (e & 3)) * 33 + jl] = v[e];
      ns_wave_sync();
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = tile[jl * 33 + 2 * e + h];
      ns_wave_sync();
    }
    // v[e] is the element (row, col) of the caller's matrix
    const int col = (M.flip ? ib : jb) + jl;
    if (col >= M.cols) return;
    float w[16];
    if (M.buf) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int row = M.flip ? jb + 2 * e + h : ib + 8 * (e >> 2) + 4 * h + (e & 3);
        w[e] = row < M.rows ? ((const float*)M.out)[base + (int64_t)row * M.cols + col] : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int row = M.flip ? jb + 2 * e + h : ib + 8 * (e >> 2) + 4 * h + (e & 3);
      if (row >= M.rows) continue;
      const int64_t at = base + (int64_t)row * M.cols + col;
      const float x = o.down * v[e];
      if (M.buf) ((float*)M.out)[at] = fmaf(sc.keep, w[e], x);
      else if (M.dtype == SV2N_DT_F32) ((float*)M.out)[at] = x;
      else if (M.dtype == SV2N_DT_BF16) ((__bf16*)M.out)[at] = (__bf16)x;
      else ((_Float16*)M.out)[at] = (_Float16)x;
    }
    return;
  }
  // the transpose, rows j: straight from registers
  _Float16* T = EPI == NS_S ? M.s + ss : EPI == NS_Q ? M.q + ss : M.xt[cur ^ 1] + xs;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    f16x8 hi, lo;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = v[g * 8 + e];
    ns_pack(f, M.exact, hi, lo);
    _Float16* p = T + ns_blk(jb >> 5, (ib >> 4) + g, M.mp) + lane * 8;
    *(f16x8*)p = hi;
    *(f16x8*)(p + 512) = lo;
  }
  if (!mirror) return;
  // the tile itself, rows i
#pragma unroll
  for (int e = 0; e < 16; ++e) tile[(8 * (e >> 2) + 4 * h + (e & 3)) * 33 + jl] = v[e];
  ns_wave_sync();
  _Float16* D = EPI == NS_S ? M.s + ss : EPI == NS_Q ? M.q + ss : M.x + xs;
  const int kd = EPI == NS_X ? M.np : M.mp;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    f16x8 hi, lo;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = tile[jl * 33 + 16 * g + ns_k(h, e)];
    ns_pack(f, M.exact, hi, lo);
    _Float16* p = D + ns_blk(ib >> 5, (jb >> 4) + g, kd) + lane * 8;
    *(f16x8*)p = hi;
    *(f16x8*)(p + 512) = lo;
  }
  ns_wave_sync();
}

// Blocks of a launch that share operand rows run on one XCD (its own L2): the
// hardware deals blocks to the 8 XCDs in turn, so block b takes the (b / 8)-th tile of
// the (b % 8)-th eighth.
__device__ __forceinline__ int ns_xcd(int b, int n) {
  const int x = b & 7, k = b >> 3, q = n >> 3, r = n & 7;
  return x * q + min(x, r) + k;
}

struct NsTile {
  const NsMat* M;
  int bt, ti, tj;
};
// tile `b` (of TB x TB) of a launch
template <int TB, int EPI>
__device__ __forceinline__ NsTile ns_tile_of(const NsArgs& A, int b) {
  NsTile r;
  const int mi = ns_find(A, b);
  const NsMat& M = A.mat[mi];
  int local = b - A.first[mi];
  const int tm = M.mp / TB, tn = M.np / TB;
  if (EPI == NS_S || EPI == NS_Q) {
    const int per = tm * (tm + 1) / 2;
    r.bt = local / per;
    local -= r.bt * per;
    int ti = (int)((sqrtf(8.f * (float)local + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > local) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= local) ++ti;
    r.ti = ti;
    r.tj = local - ti * (ti + 1) / 2;
  } else {
    const int per = tm * tn;
    r.bt = local / per;
    local -= r.bt * per;
    // strips of 8 rows of tiles, column by column
    const int s0 = local / (8 * tn) * 8, sh = min(8, tm - s0);
    local -= s0 * tn;
    r.ti = s0 + local % sh;
    r.tj = local / sh;
  }
  r.M = &M;
  return r;
}

// The eight f32 products of a pair of exact fragments: instruction q takes every lane's
// value q, so lane half h's K values 4h + .. of both operands meet
__device__ __forceinline__ f32x16 ns_mfma_exact(const f16x8* a, const f16x8* b, f32x16 c) {
#pragma unroll
  for (int q = 0; q < 8; ++q)
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(f32x4, a[q >> 2])[q & 3],
                                             __builtin_bit_cast(f32x4, b[q >> 2])[q & 3], c, 0, 0,
                                             0);
  return c;
}

// The three f16 products of a pair of fragments
__device__ __forceinline__ f32x16 ns_mfma(const f16x8* a, const f16x8* b, f32x16 c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[0], c, 0, 0, 0);
  return c;
}

// ---- 3: one product ----
// Tiles of 32·FT a side.  Each of the block's W waves takes every W-th 16 K values of
// the whole tile: fragments go straight from memory into registers, DEPTH steps
// ahead, and nothing waits for another wave until the W sums are added at the end in
// wave order.  The wider the wave's tile, the fewer bytes a product needs (FT = 1, 2,
// 4: 4, 8, 16 KiB for 3, 12, 48 matrix instructions), so what bounds it goes from the
// caches to the matrix cores, but the fewer blocks there are and the more the sums at
// the end cost.  MI355X, one product of an f32 orthogonalisation, us:
//                                        FT = 1    FT = 2    FT = 4
//   X' of 512 x 512     (K 512)             6.1       7.5      17.9
//   S of 1,024 x 4,096  (K 4,096)          44.2      27.7      61.9
//   X' of 1,024 x 4,096 (K 1,024)          54.9      38.1      34.9
//   X' of 2,048 x 2,048                       -      70.7      55.8
//   X' of 4,096 x 4,096                       -       511       365   (1.13 Pflop/s of f16)
// FT = 4 keeps 256 accumulators and two steps of fragments in the 512 registers of the
// one wave per SIMD.  big0 >= 0 (FT = 2): the blocks are quarters of the 128 x 128 tiles
// from big0 on, what whole rounds of FT = 4 left.
template <int EPI, int FT, int W>
__global__ __launch_bounds__(64 * W, FT == 4 ? 1 : 2) void k_ns_mm(NsArgs A, NsScale sc, int cur, int big0) {
  // (deeper does not help: 2 to 5 steps measure the same.  FT = 1 and 2 are bound by the
  // 64 B a cycle that a CU's L1 hands its registers: with every load a hit they take 80 %
  // of the time, and without the products 90 to 100 %)
  constexpr int DEPTH = FT == 1 ? 4 : 2;
  constexpr int TB = 32 * FT;
  extern __shared__ float s_sum[];
  const int bx = ns_xcd(blockIdx.x, gridDim.x);
  NsTile tl;
  if (FT == 2 && big0 >= 0) {
    tl = ns_tile_of<128, EPI>(A, big0 + (bx >> 2));
    const int si = (bx >> 1) & 1, sj = bx & 1;
    // above the diagonal: its mirror's block writes it
    if ((EPI == NS_S || EPI == NS_Q) && tl.ti == tl.tj && sj > si) return;
    tl.ti = tl.ti * 2 + si;
    tl.tj = tl.tj * 2 + sj;
  } else {
    tl = ns_tile_of<TB, EPI>(A, bx);
  }
  const NsMat& M = *tl.M;
  const int64_t xs = (int64_t)tl.bt * 2 * M.mp * M.np, ss = (int64_t)tl.bt * 2 * M.mp * M.mp;
  const int kp = EPI == NS_S ? M.np : M.mp;
  const _Float16* P = EPI == NS_S ? M.x + xs : EPI == NS_Q ? M.s + ss : M.q + ss;
  const _Float16* R = EPI == NS_S ? M.x + xs : EPI == NS_Q ? M.s + ss : M.xt[cur] + xs;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t rg = (int64_t)(kp >> 4) << 10;
  const _Float16* gp = P + ns_blk(tl.ti * FT, 0, kp) + lane * 8;
  const _Float16* gr = R + ns_blk(tl.tj * FT, 0, kp) + lane * 8;
  f16x8 a[DEPTH][FT][2], b[DEPTH][FT][2];
  f32x16 acc[FT][FT];
#pragma unroll
  for (int x = 0; x < FT; ++x)
#pragma unroll
    for (int y = 0; y < FT; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
  const int nk = ((EPI == NS_S ? M.n : M.m) + 15) / 16;  // (the padding's zeros add nothing)
  auto fetch = [&](int d, int k) {
#pragma unroll
    for (int x = 0; x < FT; ++x)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        a[d][x][p] = *(const f16x8*)(gp + x * rg + (int64_t)k * 1024 + p * 512);
        b[d][x][p] = *(const f16x8*)(gr + x * rg + (int64_t)k * 1024 + p * 512);
      }
  };
  // loads past the operand's end read its last block again (not used): without a
  // branch the waits count the loads in flight
  auto run = [&](auto product) {
    auto mul = [&](int d) {
#pragma unroll
      for (int x = 0; x < FT; ++x)
#pragma unroll
        for (int y = 0; y < FT; ++y) acc[x][y] = product(a[d][x], b[d][y], acc[x][y]);
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) fetch(d, min(wave + d * W, nk - 1));
    int k = wave;
    for (; k + (DEPTH - 1) * W < nk; k += DEPTH * W) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        // (the scheduler would sink the loads to their use, and the distance with them)
        __builtin_amdgcn_sched_barrier(0);
        mul(d);
        __builtin_amdgcn_sched_barrier(0);
        fetch(d, min(k + (d + DEPTH) * W, nk - 1));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d)
      if (k + d * W < nk) mul(d);
  };
  auto f16 = [](const f16x8* p, const f16x8* q, f32x16 c) { return ns_mfma(p, q, c); };
  if constexpr (FT == 1) {
    if (M.exact) run([](const f16x8* p, const f16x8* q, f32x16 c) { return ns_mfma_exact(p, q, c); });
    else run(f16);
  } else {
    run(f16);  // (f32 operands come on FT = 1 alone)
  }
  if constexpr (FT == 4) {
    // wave w finishes the 64 x 64 quadrant (w / 2, w % 2); two quadrants' sums at a
    // time fit the LDS
    const NsOut o = ns_out<EPI>(sc, M);
    f32x16 own[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s_sum[(((q * 4 + wave) * 4 + v) * 16 + e) * 64 + lane] =
                acc[h * 2 + (v >> 1)][q * 2 + (v & 1)][e];
      __syncthreads();
      if ((wave >> 1) == h) {
        const int q = wave & 1;
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float* c = s_sum + (((q * 4) * 4 + v) * 16 + e) * 64 + lane;
            own[v >> 1][v & 1][e] = (c[0] + c[4096]) + (c[2 * 4096] + c[3 * 4096]);
          }
      }
      __syncthreads();
    }
    float* tile = s_sum + wave * 32 * 33;
#pragma unroll
    for (int v = 0; v < 4; ++v)
      ns_epilogue<EPI>(own[v >> 1][v & 1], o, M, sc, R, tl.bt,
                       tl.ti * TB + (wave >> 1) * 64 + (v >> 1) * 32,
                       tl.tj * TB + (wave & 1) * 64 + (v & 1) * 32, cur,
                       EPI == NS_X || tl.ti != tl.tj, tile);
    return;
  } else {
  f32x16 d;
  float* tile;
  int x = 0, y = 0;
  if constexpr (FT == 2) {
    // wave w finishes the tile at (w / 2, w % 2); two places' sums at a time in the LDS,
    // so that three blocks share a CU
    static_assert(W == 4, "one wave per place");
    auto sum = (float (*)[W][16][64])s_sum;  // [place of 2][wave][element][lane]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h) __syncthreads();
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[q][wave][e][lane] = acc[h][q][e];
      __syncthreads();
      if ((wave >> 1) == h) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          d[e] = (sum[wave & 1][0][e][lane] + sum[wave & 1][1][e][lane]) +
                 (sum[wave & 1][2][e][lane] + sum[wave & 1][3][e][lane]);
      }
    }
    x = wave >> 1;
    y = wave & 1;
    __syncthreads();
    tile = s_sum + wave * 32 * 33;
  } else {
    auto sum = (float (*)[W][16][64])s_sum;  // [0][wave][element][lane]
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[0][wave][e][lane] = acc[0][0][e];
    __syncthreads();
    // the waves add 16 / W elements each, the first one finishes the tile
    constexpr int EW = 16 / W;
    float part[EW];
#pragma unroll
    for (int q = 0; q < EW; ++q) {
      part[q] = 0.f;
#pragma unroll
      for (int u = 0; u < W; ++u) part[q] += sum[0][u][wave * EW + q][lane];
    }
    // slot 0 of an element is read by its own adder alone
#pragma unroll
    for (int q = 0; q < EW; ++q) sum[0][0][wave * EW + q][lane] = part[q];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int e = 0; e < 16; ++e) d[e] = sum[0][0][e][lane];
    ns_wave_sync();
    tile = &sum[0][1][0][0];
  }
  const NsOut o = ns_out<EPI>(sc, M);
  ns_epilogue<EPI>(d, o, M, sc, R, tl.bt, tl.ti * TB + x * 32, tl.tj * TB + y * 32, cur,
                   EPI == NS_X || tl.ti != tl.tj, tile);
  }
}

// ---- 3b: Q and X's product in one launch, for small matrices (mp <= 128) ----
// A 32 x 32 tile of X needs 32 rows of Q, 32 x m values from the m x m S: each block
// makes them itself (in LDS, as fragments) rather than wait for a launch that stores
// Q.  128 x 1,024: 4.3 + 4.5 us in two launches, 7.9 in one (87 -> 81 us with all steps).
// Eight waves: first Q's m / 32 tiles times
// slices of their depth, then 16 K values of X's product each.
template <int EPI>
__global__ __launch_bounds__(512, 2) void k_ns_qx(NsArgs A, NsScale sc, int cur) {
  __shared__ __attribute__((aligned(16))) float sum[8][16][64];
  __shared__ __attribute__((aligned(16))) _Float16 qf[8][2][512];
  const NsTile tl = ns_tile_of<32, EPI>(A, ns_xcd(blockIdx.x, gridDim.x));
  const NsMat& M = *tl.M;
  const int64_t xs = (int64_t)tl.bt * 2 * M.mp * M.np, ss = (int64_t)tl.bt * 2 * M.mp * M.mp;
  const _Float16 *S = M.s + ss, *R = M.xt[cur] + xs;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int kp = M.mp, nk = kp / 16;       // 4 or 8
  const int tiles = kp / 32, slices = 8 / tiles;
  const int tq = wave % tiles, sl = wave / tiles;
  auto product = [&](const f16x8* p, const f16x8* q, f32x16 c) {
    if (M.exact) return ns_mfma_exact(p, q, c);
    return ns_mfma(p, q, c);
  };
  // X's fragment of this wave's K values, in flight meanwhile
  f16x8 xb[2];
#pragma unroll
  for (int p = 0; p < 2; ++p)
    xb[p] = *(const f16x8*)(R + ns_blk(tl.tj, min(wave, nk - 1), kp) + p * 512 + lane * 8);
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  for (int k = sl; k < nk; k += slices) {
    f16x8 a[2], b[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      a[p] = *(const f16x8*)(S + ns_blk(tq, k, kp) + p * 512 + lane * 8);
      b[p] = *(const f16x8*)(S + ns_blk(tl.ti, k, kp) + p * 512 + lane * 8);
    }
    acc = product(a, b, acc);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[wave][e][lane] = acc[e];
  __syncthreads();
  if (sl < 2) {
    // (S S) is symmetric: the tile's transpose, whose lane & 31 is Q's row, is what the
    // accumulators hold as fragments; slice sl finishes 16 of the tile's 32 K values
    const NsOut o = ns_out<NS_Q>(sc, M);
    const _Float16* p = S + ns_blk(tl.ti, tq * 2 + sl, kp) + lane * 8;
    float old[8], v[8];
    ns_unpack(*(const f16x8*)p, *(const f16x8*)(p + 512), M.exact, old);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float d = 0.f;
      for (int u = 0; u < slices; ++u) d += sum[tq + tiles * u][sl * 8 + e][lane];
      v[e] = fmaf(o.old, old[e], o.up * d);
    }
    f16x8 hi, lo;
    ns_pack(v, M.exact, hi, lo);
    *(f16x8*)&qf[tq * 2 + sl][0][lane * 8] = hi;
    *(f16x8*)&qf[tq * 2 + sl][1][lane * 8] = lo;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  if (wave < nk) {
    f16x8 a[2];
    a[0] = *(const f16x8*)&qf[wave][0][lane * 8];
    a[1] = *(const f16x8*)&qf[wave][1][lane * 8];
    acc = product(a, xb, acc);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[wave][e][lane] = acc[e];
  __syncthreads();
  // two elements a wave; slot 0 of an element is read by its own adder alone
  float part[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    part[q] = 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) part[q] += sum[u][wave * 2 + q][lane];
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) sum[0][wave * 2 + q][lane] = part[q];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = sum[0][e][lane];
  ns_wave_sync();
  ns_epilogue<EPI>(acc, ns_out<EPI>(sc, M), M, sc, R, tl.bt, tl.ti * 32, tl.tj * 32, cur, true,
                   &sum[1][0][0]);
}

// ---- 4: thin matrices (m <= 32), one launch a step ----
// X is at most 32 rows tall, so a block keeps 128 of its n columns in registers, f32, and
// needs of the others only S: a launch adds the blocks' partial S in block order, makes
// Q, its columns of X' and its partial of the next S, all with f32 matrix instructions.
// A wave has 32 columns as accumulators hold them (lane & 31 the column, register e and
// lane half h the row 8·(e/4) + 4h + e%4), and S and Q the same way: S is symmetric, so
// instruction e of S S and of Q X takes register e of both operands as it is.  Only X Xt
// sums over columns and turns them in LDS.  A matrix of at most 128 columns takes all its
// steps in one launch.  Against three products a step on tiles, us: 16 x 128 66 -> 21,
// 32 x 1,024 87 -> 43, 16 x 4,096 187 -> 53 (what is left is launches).
// steps: how many this launch takes; first: from the caller's matrix (else from M.x);
// last: the result goes to the caller.  single: one block per matrix.
template <typename T>
__global__ __launch_bounds__(256) void k_ns_thin(NsArgs A, NsScale sc, int cur, int steps,
                                                 int first, int last, int single) {
  constexpr int CC = NS_THIN_COLS;
  __shared__ float xs[4][32][33];        // a wave's columns, turned
  __shared__ float red[2][4][16][64];    // the waves' sums of X Xt, two steps in turn
  __shared__ double nred[4];
  const int mi = ns_find(A, blockIdx.x);
  const NsMat& M = A.mat[mi];
  const int local = blockIdx.x - A.first[mi];
  const int chunks = M.np / CC;
  const int bt = local / chunks, ch = local - bt * chunks;
  const int t = threadIdx.x, lane = t & 63, h = lane >> 5, wave = wave_id();
  const int j = ch * CC + wave * 32 + (lane & 31);
  auto row_of = [&](int e) { return 8 * (e >> 2) + 4 * h + (e & 3); };
  float* X = (float*)M.x + (int64_t)bt * 32 * M.np;
  const float* part_in = M.thin + ((int64_t)cur * M.batch + bt) * chunks * 1024;
  float* part_out = M.thin + ((int64_t)(cur ^ 1) * M.batch + bt) * chunks * 1024;
  f32x16 x;
  if (first) {
    const T* g = (const T*)M.g + bt * M.g_batch;
    float m[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int i = row_of(e);
      const int64_t row = M.flip ? j : i, col = M.flip ? i : j;
      const bool in = i < M.m && j < M.n;
      x[e] = in ? (float)g[row * M.ld + col] : 0.f;
      m[e] = in && M.buf ? M.buf[row * M.cols + col] : 0.f;
    }
    double acc = 0.0;
    for (int k = t; k < M.parts; k += 256) acc += M.part[(int64_t)bt * M.parts + k];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) acc += __shfl_xor(acc, o, 64);
    if (lane == 0) nred[wave] = acc;
    __syncthreads();
    const double norm = sqrt((nred[0] + nred[1]) + (nred[2] + nred[3]));
    const double inv = 1.0 / (norm < (double)sc.eps ? (double)sc.eps : norm);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float u = M.buf ? ns_update(sc, x[e], m[e]) : x[e];
      x[e] = (float)((double)u * inv);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = X[(int64_t)row_of(e) * M.np + j];
  }
  // the wave's columns of X Xt
  auto gram = [&]() {
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      acc[e] = 0.f;
      xs[wave][row_of(e)][lane & 31] = x[e];
    }
    ns_wave_sync();
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const float a = xs[wave][lane & 31][2 * q + h];
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a, a, acc, 0, 0, 0);
    }
    ns_wave_sync();
    return acc;
  };
  // the block's: in every wave's registers (single), or to its partial
  auto reduce = [&](const f32x16& acc, int buf, f32x16* S) {
#pragma unroll
    for (int e = 0; e < 16; ++e) red[buf][wave][e][lane] = acc[e];
    __syncthreads();
    if (single) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        (*S)[e] = (red[buf][0][e][lane] + red[buf][1][e][lane]) +
                  (red[buf][2][e][lane] + red[buf][3][e][lane]);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int e = wave * 4 + q;
        part_out[(int64_t)ch * 1024 + e * 64 + lane] =
            (red[buf][0][e][lane] + red[buf][1][e][lane]) +
            (red[buf][2][e][lane] + red[buf][3][e][lane]);
      }
    }
  };
  f32x16 S;
#pragma unroll
  for (int e = 0; e < 16; ++e) S[e] = 0.f;
  int buf = 0;
  if (first) {
    reduce(gram(), buf, &S);
    buf ^= 1;
  } else {
    // the blocks' partials: a wave adds four registers' worth and hands them round
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const float* p = part_in + wave * 256 + lane;
#pragma unroll 4
    for (int k = 0; k < chunks; ++k)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += p[(int64_t)k * 1024 + q * 64];
#pragma unroll
    for (int q = 0; q < 4; ++q) red[buf][0][wave * 4 + q][lane] = v[q];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) S[e] = red[buf][0][e][lane];
    buf ^= 1;
  }
  for (int s = 0; s < steps; ++s) {
    f32x16 Q, y;
#pragma unroll
    for (int e = 0; e < 16; ++e) Q[e] = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) Q = __builtin_amdgcn_mfma_f32_32x32x2f32(S[e], S[e], Q, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      Q[e] = fmaf(sc.c, Q[e], sc.b * S[e]);
      y[e] = 0.f;
    }
    // (a x joins the finished sum: under it, every addition would round at its size)
#pragma unroll
    for (int e = 0; e < 16; ++e) y = __builtin_amdgcn_mfma_f32_32x32x2f32(Q[e], x[e], y, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = fmaf(sc.a, x[e], y[e]);
    if (last && s + 1 == steps) break;
    reduce(gram(), buf, &S);
    buf ^= 1;
  }
  if (!last) {
#pragma unroll
    for (int e = 0; e < 16; ++e) X[(int64_t)row_of(e) * M.np + j] = x[e];
    return;
  }
  const int64_t base = (int64_t)bt * M.rows * M.cols;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int i = row_of(e);
    if (i >= M.m || j >= M.n) continue;
    const int64_t at = base + (M.flip ? (int64_t)j * M.cols + i : (int64_t)i * M.cols + j);
    if (M.buf) {
      float* w = (float*)M.out + at;
      *w = fmaf(sc.keep, *w, -M.lr * x[e]);
    } else {
      ((T*)M.out)[at] = (T)x[e];
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static inline int64_t ns_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// What one step does to singular values in [0, hi], f(x) = x·p(x²), p(y) = a + b y + c y²:
// the largest |f|; of q(y) = b y + c y² the largest |q|; the largest |p| or |f'|, which is
// how far the step can multiply an error of X; and the least |f| over [lo, hi].  All are
// smooth, so the ends and the polynomials' own stationary points settle it.
struct NsStep {
  double f_max, q_max, gain, f_min;
};
static NsStep ns_step(double a, double b, double c, double lo, double hi) {
  auto f = [&](double x) { return x * (a + b * x * x + c * x * x * x * x); };
  auto q = [&](double y) { return std::fabs(b * y + c * y * y); };
  auto p = [&](double y) { return std::fabs(a + b * y + c * y * y); };
  auto fd = [&](double y) { return std::fabs(a + 3 * b * y + 5 * c * y * y); };
  const double top = hi * hi;
  // inside (0, top): where q and p (one shape), f' and f turn
  double turn_p = -1.0, turn_fd = -1.0, turn_f[2] = {-1.0, -1.0};
  if (c != 0.0) {
    turn_p = -b / (2 * c);
    turn_fd = -3 * b / (10 * c);
    const double dis = 9 * b * b - 20 * a * c;  // of f' = a + 3 b y + 5 c y²
    if (dis >= 0.0) {
      turn_f[0] = (-3 * b - std::sqrt(dis)) / (10 * c);
      turn_f[1] = (-3 * b + std::sqrt(dis)) / (10 * c);
    }
  } else if (b != 0.0) {
    turn_f[0] = -a / (3 * b);
  }
  auto in = [&](double y) { return y > 0.0 && y < top; };
  NsStep r;
  r.f_max = std::fabs(f(hi));
  r.q_max = q(top);
  r.gain = std::max(std::max(p(0.0), p(top)), fd(top));
  if (in(turn_p)) {
    r.q_max = std::max(r.q_max, q(turn_p));
    r.gain = std::max(r.gain, p(turn_p));
  }
  if (in(turn_fd)) r.gain = std::max(r.gain, fd(turn_fd));
  double least = std::min(f(lo), f(hi)), most = std::max(f(lo), f(hi));
  for (double y : turn_f)
    if (in(y)) {
      const double x = std::sqrt(y), v = f(x);
      r.f_max = std::max(r.f_max, std::fabs(v));
      if (x > lo) {
        least = std::min(least, v);
        most = std::max(most, v);
      }
    }
  r.f_min = least > 0.0 ? least : most < 0.0 ? -most : 0.0;
  return r;
}

// What the steps can do to X: `gain` to an error of it, `least` its smallest norm
struct NsRange {
  double gain, least;
};

// The power-of-two scales of X, S and Q from the largest singular value any step
// can reach; false if the coefficients let them grow past 2^8.
static bool ns_scales(int steps, NsScale* sc, NsRange* range) {
  // (the largest singular value of an m-row X_0 is at least 1/sqrt(m))
  double top = 1.0, hi = 1.0, lo = 1.0 / 128, qm = 0.0;
  static_assert(SV2N_NS_MAX_SIDE == 128 * 128, "lo");
  *range = {1.0, lo};
  for (int k = 0; k < steps; ++k) {
    const NsStep r = ns_step(sc->a, sc->b, sc->c, lo, hi);
    qm = std::max(qm, r.q_max);
    top = std::max(top, r.f_max);
    hi = r.f_max;
    lo = r.f_min;
    range->gain *= std::max(1.0, r.gain);
    range->least = std::min(range->least, lo);
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

// Whether pairs of f16 are as good as f32 for a matrix under these steps.  An entry held
// as a pair is off by up to 2^-39 (0.3 of it on average) however small it is, which f32
// is not.  Over the matrix that is 2^-41 sqrt(rows·cols) in the 2-norm, and the steps
// multiply it by at most `gain`: allowed up to 2^-17 of a result whose norm is near 1 or
// more.  (The default coefficients: five steps at every size, 6 to 4,096², 8 to 64 x 128.)
// And X must not shrink by more than 16, or 2^-39 comes nearer to its own entries.
static bool ns_pairs_ok(const NsMat& M, const NsRange& range) {
  return range.gain * std::sqrt((double)M.rows * M.cols) <= 16777216.0 &&
         range.least >= 1.0 / 2048;
}

static void ns_shape(NsMat* M) {
  M->flip = M->rows > M->cols;
  M->m = std::min(M->rows, M->cols);
  M->n = std::max(M->rows, M->cols);
  const int64_t total = (int64_t)M->rows * M->cols;
  const int64_t each = std::max<int64_t>(NS_PART_ELEMS, (total + NS_PARTS - 1) / NS_PARTS);
  M->part_elems = (int)ns_up(each, 8);
  M->parts = (int)((total + M->part_elems - 1) / M->part_elems);
}

// What a group's matrices are padded to: 128 where X's product (the largest) is worth
// tiles of 128: NS_HALF of them that are NS_DEEP deep, else 64
static int ns_pad(const NsMat* mats, int count) {
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i)
    if (mats[i].m >= NS_DEEP)
      tiles += (int64_t)mats[i].batch * (ns_up(mats[i].m, 128) / 128) *
               (ns_up(mats[i].n, 128) / 128);
  return tiles >= NS_HALF ? 128 : 64;
}

// Whether a group's matrices of m <= NS_EXACT go to k_ns_thin: always where the others
// (if any) have NS_TINY tiles of 64 or one is longer than NS_THIN_LONG; beside small
// matrices they ride in those launches as exact tiles instead of adding their own.
static bool ns_thin(const NsMat* mats, int count) {
  int64_t tiles = 0;
  bool others = false, any = false, longer = false;
  for (int i = 0; i < count; ++i) {
    if (mats[i].m <= NS_EXACT) {
      any = true;
      longer |= mats[i].n > NS_THIN_LONG;
    } else {
      others = true;
      tiles += (int64_t)mats[i].batch * (ns_up(mats[i].m, 64) / 64) * (ns_up(mats[i].n, 64) / 64);
    }
  }
  return any && (!others || longer || tiles >= NS_TINY);
}

// pads the shapes and lays its workspace out from `ws`
// (NULL: only counts); returns the bytes
static int64_t ns_plan(NsMat* mats, int count, int pad, char* ws) {
  int64_t off = 0;
  const bool thin = ns_thin(mats, count);
  auto take = [&](int64_t bytes) {
    char* p = ws ? ws + off : nullptr;
    off += ns_up(bytes, 256);
    return p;
  };
  for (int i = 0; i < count; ++i) {
    NsMat& M = mats[i];
    M.thin = nullptr;
    if (thin && M.m <= NS_EXACT) {
      M.mp = NS_EXACT;
      M.np = (int)ns_up(M.n, NS_THIN_COLS);
      M.part = (double*)take((int64_t)M.batch * M.parts * 8);
      M.x = (_Float16*)take((int64_t)M.batch * NS_EXACT * M.np * 4);
      M.thin = (float*)take((int64_t)2 * M.batch * (M.np / NS_THIN_COLS) * 4096);
      continue;
    }
    M.mp = (int)ns_up(M.m, pad);
    M.np = (int)ns_up(M.n, pad);
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

// Tiles of a product over the group's matrices; `pairs`: over those in pairs of f16
template <int EPI>
static int64_t ns_count(NsArgs& A, int tile, bool pairs) {
  return ns_blocks(A, [&](const NsMat& M) -> int64_t {
    const int64_t tm = M.mp / tile, tn = M.np / tile;
    return pairs && M.exact ? 0 : EPI == NS_S || EPI == NS_Q ? tm * (tm + 1) / 2 : tm * tn;
  });
}

template <int EPI, int FT, int W>
static void ns_launch(NsArgs& A, const NsScale& sc, int cur, int64_t blocks, int big0,
                      hipStream_t stream) {
  constexpr int lds = FT == 4 ? 131072 : FT == 2 ? 32768 : W * 4096;
  auto* k = k_ns_mm<EPI, FT, W>;
  if (lds > 65536)
    (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(64 * W), lds, stream, A, sc, cur, big0);
}

// A product over the group's tiles.  Tiles of 128 where they fill at least half of the
// chip's 256 CUs (one block each) in every round; fewer than that left over go on
// tiles of 64, as do products that never have so many; tiles of 32 where even those
// are under NS_TINY (the measured sides: k_ns_mm), and for f32 operands, whose products
// are the bound there already (tiles of 64, us a step: 4,096² 3,450 -> 3,780, 777 x 1,537
// 77 -> 87, 1,024² 86 -> 62).  A group is all f32 operands, or those of m <= NS_EXACT
// beside pairs with fewer than NS_TINY tiles (ns_thin).
template <int EPI>
static void ns_product(NsArgs& A, const NsScale& sc, int cur, int pad, hipStream_t stream) {
  if (ns_count<EPI>(A, 64, true) < NS_TINY) {
    ns_launch<EPI, 1, 8>(A, sc, cur, ns_count<EPI>(A, 32, false), -1, stream);
    return;
  }
  if (pad == 128) {
    const int64_t n = ns_count<EPI>(A, 128, true);
    int64_t big = n / 256 * 256;
    if (n - big >= NS_HALF) big = n;
    if (big > 0) {
      ns_launch<EPI, 4, 4>(A, sc, cur, big, -1, stream);
      if (n > big) ns_launch<EPI, 2, 4>(A, sc, cur, 4 * (n - big), (int)big, stream);
      return;
    }
  }
  ns_launch<EPI, 2, 4>(A, sc, cur, ns_count<EPI>(A, 64, true), -1, stream);
}

// Whether Q and X's product go in one launch: every matrix small enough for k_ns_qx, and
// few enough tiles that each making its rows of Q costs less than a launch
static bool ns_fused(NsArgs& A) {
  for (int i = 0; i < A.count; ++i)
    if (A.mat[i].mp > 128) return false;
  return ns_count<NS_X>(A, 32, false) <= NS_FUSED;
}

static void ns_one_step(NsArgs& A, const NsScale& sc, int s, bool last, int pad,
                        hipStream_t stream) {
  const int cur = s & 1;
  ns_product<NS_S>(A, sc, cur, pad, stream);
  if (ns_fused(A)) {
    const int64_t n = ns_count<NS_X>(A, 32, false);
    if (!last)
      hipLaunchKernelGGL(k_ns_qx<NS_X>, dim3((unsigned)n), dim3(512), 0, stream, A, sc, cur);
    else
      hipLaunchKernelGGL(k_ns_qx<NS_LAST>, dim3((unsigned)n), dim3(512), 0, stream, A, sc, cur);
    return;
  }
  ns_product<NS_Q>(A, sc, cur, pad, stream);
  if (!last) ns_product<NS_X>(A, sc, cur, pad, stream);
  else ns_product<NS_LAST>(A, sc, cur, pad, stream);
}

template <typename T>
static void ns_run_as(NsArgs& A, const NsScale& sc, int steps, int pad, hipStream_t stream) {
  int64_t n = ns_blocks(A, [](const NsMat& M) -> int64_t { return M.parts; });
  hipLaunchKernelGGL(k_ns_norm<T>, dim3((unsigned)n), dim3(256), 0, stream, A, sc);
  NsArgs B{}, H{};  // tiles, thin
  for (int i = 0; i < A.count; ++i) {
    NsArgs& to = A.mat[i].thin ? H : B;
    to.mat[to.count++] = A.mat[i];
  }
  if (H.count) {
    n = ns_blocks(H, [](const NsMat& M) -> int64_t { return M.np / NS_THIN_COLS; });
    bool single = true;
    for (int i = 0; i < H.count; ++i) single &= H.mat[i].np == NS_THIN_COLS;
    auto go = [&](int cur, int k, int first, int last) {
      hipLaunchKernelGGL(k_ns_thin<T>, dim3((unsigned)n), dim3(256), 0, stream, H, sc, cur, k, first,
                         last, (int)single);
    };
    if (single) {
      go(0, steps, 1, 1);
    } else {
      go(1, 0, 1, 0);
      for (int k = 0; k < steps; ++k) go(k & 1, 1, 0, k + 1 == steps);
    }
  }
  if (!B.count) return;
  n = ns_blocks(B, [](const NsMat& M) -> int64_t { return (int64_t)(M.mp / 64) * (M.np / 64); });
  hipLaunchKernelGGL(k_ns_split<T>, dim3((unsigned)n), dim3(256), 0, stream, B, sc);
  for (int k = 0; k < steps; ++k) ns_one_step(B, sc, k, k + 1 == steps, pad, stream);
}

// Which products a group takes: one matrix that needs f32 operands takes the group along
// (a step's launches are shared), else those of m <= NS_EXACT have them alone
static void ns_exact(NsArgs* A, const NsRange& range) {
  bool all = false;
  for (int i = 0; i < A->count; ++i)
    all |= A->mat[i].m > NS_EXACT && !ns_pairs_ok(A->mat[i], range);
  for (int i = 0; i < A->count; ++i) A->mat[i].exact = all || A->mat[i].m <= NS_EXACT;
}

static int ns_run(NsArgs& A, const NsScale& sc, int steps, int pad, hipStream_t stream) {
  const int dtype = A.mat[0].dtype;  // one for the whole group
  if (dtype == SV2N_DT_F32) ns_run_as<float>(A, sc, steps, pad, stream);
  else if (dtype == SV2N_DT_BF16) ns_run_as<__bf16>(A, sc, steps, pad, stream);
  else ns_run_as<_Float16>(A, sc, steps, pad, stream);
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
  return ns_plan(&M, 1, ns_pad(&M, 1), nullptr);
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
  NsRange range;
  if (!ns_scales(steps, &sc, &range)) return SV2N_ERR_ARG;
  NsMat& M = A.mat[0];
  A.count = 1;
  M.g = g; M.ld = ld; M.g_batch = batch_stride; M.out = out; M.dtype = dtype;
  M.rows = (int)rows; M.cols = (int)cols; M.batch = (int)batch;
  ns_shape(&M);
  ns_exact(&A, range);
  const int pad = ns_pad(&M, 1);
  if (!workspace || workspace_bytes < ns_plan(&M, 1, pad, nullptr)) return SV2N_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 255) return SV2N_ERR_ALIGN;
  ns_plan(&M, 1, pad, (char*)workspace);
  return ns_run(A, sc, steps, pad, stream);
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
    most = std::max(most, ns_plan(A.mat, n, ns_pad(A.mat, n), nullptr));
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
  NsRange range;
  if (!ns_scales(steps, &sc, &range)) return SV2N_ERR_ARG;
  if (!workspace || workspace_bytes < sv2n_muon_step_workspace(mats, count))
    return SV2N_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 255) return SV2N_ERR_ALIGN;
  for (int k = 0; k < count; k += NS_MAX) {
    const int n = std::min(NS_MAX, count - k);
    NsArgs A{};
    ns_group(mats + k, n, lr, &A);
    ns_exact(&A, range);
    const int pad = ns_pad(A.mat, n);
    ns_plan(A.mat, n, pad, (char*)workspace);
    const int rc = ns_run(A, sc, steps, pad, stream);
    if (rc) return rc;
  }
  return 0;
}
