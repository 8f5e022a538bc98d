// Newton-Schulz orthogonalisation of many matrices at once and the Muon step built on it, for gfx950.
//
//   m <- mu m + (1 - mu) g     u = mu m + (1 - mu) g (Nesterov) or m     X = u / max(|u|, eps), |u| the root of the sum of squares
//   steps times:  A = X X^T    P = b A + c A A    X <- a X + P X         (a matrix taller than wide: its transpose)
//   p <- p (1 - lr decay) - lr adjust X
//
// A matrix m x n (m <= n) lives in a workspace as [m', n'], both rounded up to 64 and zero beyond m and n, which every
// product leaves zero: no product has an edge to watch.  It stands there in panels of 32 columns, [n' / 32][m'][32], so
// that what a stage of a product copies to LDS is one piece (rows of n' elements instead: 8 to 30% slower).  Matrices of one
// shape stand one behind the other, and a launch takes the tiles of all shapes: three launches a step, whatever the
// number of matrices.  A and P are symmetric: only tiles on and above the diagonal are computed and also written
// transposed, so that a step costs m m n + m m m + 2 m m n operations instead of 4 m m n + 2 m m m.  P X reads X along its
// rows, transposed out of LDS (ds_read_b64_tr_b16).
//
// What is rounded: the products' operands are sums of two fp16 (22 bits), scaled by powers of two (X 2^12, A and P 2^10: there is
// room up to 16 and 64, the usual coefficients keep them under 2 and 8; most values lie at 1 / sqrt(n), well above the 2^-14 where
// fp16 loses bits), sums are fp32.  A product is three, high high, high low and low high (a small matrix's low low too): the result
// is off by 0.8e-6 to 2e-6, as with products of fp32, which a bf16 result's rounding of 1.7e-3 hides.
//
// Where fewer bits are asked for, the operands are one fp16.  Singular values near 0 grow 3.4-fold a step with all the noise among
// them, so it is the early roundings of X that show, and those of its term a X alone (P is small then): X is held as the sum of two
// fp16, of which the products take the first, in the first three steps.  Simulated, 512 x 600 is off by 1.3e-3 for noise and 0.9e-3,
// 1.1e-3 and 1.3e-3 for singular values that decay over two, three and four decades (1.2, 1.4, 2.4 and 3.1e-3 with a second
// fp16 in two steps; 10 to 30e-3 with iterates in bf16), 128 x 128 by up to 1.5e-3.
#include <algorithm>
#include <cmath>
#include <exception>
#include <map>
#include <tuple>
#include <vector>

#include "optim.h"

namespace strata {

typedef _Float16 f16;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int MU_PAD = 64;       // rows and columns of a matrix in the workspace are multiples of it
constexpr int MU_K = 32;         // columns that stand together there, row by row: X[np / 32][mp][32]
constexpr int MU_CHUNK = 8192;   // elements a workgroup of the momentum's pass
constexpr int MU_SUMS = 1024;    // sums of squares a matrix from which on they are added up by a launch of their own
constexpr int MU_LO_STEPS = 3;   // steps whose X has its second fp16, where not all have
constexpr int MU_PER = 40;       // tensors a launch, and shapes: kernel arguments are 4 KiB
constexpr float MU_X = 0x1p12f, MU_A = 0x1p10f;  // scales of X, and of A and P
enum { MU_P32 = 1, MU_G32 = 2, MU_TALL = 4, MU_ALIGNED = 8, MU_NESTEROV = 16, MU_STEP = 32, MU_LO = 64 };

struct MuTensor {
  void* p;           // weights, or the result of an orthogonalisation alone
  const void* g;
  float* m;          // null: u is g
  float* master;
  f16* x;            // in the workspace, [batch, m', n']
  f16* xlo;          // its second fp16
  double* part;  // sums of squares [batch, chunks]
  int64_t rows, cols;
  uint32_t first;    // the tensor's first workgroup in the launch
  uint32_t per;      // workgroups a matrix
  uint32_t flags;
  float rate, decay;  // lr adjust and 1 - lr decay
};
struct MuBatch {
  MuTensor t[MU_PER];
  int count;
  float mu, omu;     // momentum and 1 - it
  double eps;
};
static_assert(sizeof(MuBatch) <= 4096, "kernel arguments");

template <typename F>
__device__ __forceinline__ int mu_entry(int count, uint32_t wg, F first) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first(mid) <= wg) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// v, rounded to fp32.  A product or multiply-add that is converted to fp16 may otherwise be rounded straight to it
// (v_fma_mixlo_f16) where it is stored and by way of fp32 where it is subtracted, of which a second fp16 would not be the rest; and
// a matrix's result would depend on the variant of the kernel.
__device__ __forceinline__ float mu_rounded(float v) {
  asm("" : "+v"(v));
  return v;
}

// MU_X / max(norm, eps) as f 2^k: of tiny and huge updates it leaves fp32, and a product of 64 bits costs eight times two of 32.
struct MuScale {
  float f;
  int k;
  __device__ __forceinline__ float operator()(float u) const { return mu_rounded(ldexpf(u, k) * f); }  // exact, then one rounding
};
__device__ __forceinline__ MuScale mu_scale(double norm, double eps) {
  int k = 0;
  const double f = frexp(norm == 0. ? 0. : MU_X / (norm < eps ? eps : norm), &k);  // NaN stays NaN
  return {(float)f, k};
}

__device__ __forceinline__ float mu_load(const void* p, int64_t i, bool wide) {
  return wide ? ((const float*)p)[i] : (float)((const bf16*)p)[i];
}
__device__ __forceinline__ f32x4 mu_load4(const void* p, int64_t i, bool wide) {
  if (wide) return *(const f32x4*)((const float*)p + i);
  const u32x2 w = *(const u32x2*)((const bf16*)p + i);
  return (f32x4){bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
}

// ---- m <- mu m + (1 - mu) g and the sums of squares of u, 64-bit, one a workgroup ----
__global__ __launch_bounds__(256) void muon_momentum_kernel(MuBatch b) {
  const uint32_t wg = blockIdx.x;
  const MuTensor& t = b.t[mu_entry(b.count, wg, [&](int i) { return b.t[i].first; })];
  const uint32_t local = wg - t.first, mat = local / t.per, chunk = local % t.per;
  const int64_t n = t.rows * t.cols, base = mat * n, i0 = (int64_t)chunk * MU_CHUNK, i1 = min(i0 + MU_CHUNK, n);
  const int tid = threadIdx.x;
  const bool g32 = t.flags & MU_G32, nesterov = t.flags & MU_NESTEROV;
  double s = 0.;
  auto one = [&](float g, float m) {
    m = fmaf(b.mu, m, b.omu * g);
    const double u = nesterov ? fmaf(b.mu, m, b.omu * g) : m;
    s = fma(u, u, s);
    return m;
  };
  if ((t.flags & MU_ALIGNED) && i1 - i0 == MU_CHUNK) {
#pragma unroll
    for (int k = 0; k < MU_CHUNK / 1024; ++k) {
      const int64_t i = base + i0 + 1024 * k + 4 * tid;
      const f32x4 g = mu_load4(t.g, i, g32);
      if (t.m) {
        f32x4 m = *(const f32x4*)(t.m + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = one(g[e], m[e]);
        *(f32x4*)(t.m + i) = m;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fma((double)g[e], (double)g[e], s);
      }
    }
  } else {
    for (int64_t i = base + i0 + tid; i < base + i1; i += 256) {
      const float g = mu_load(t.g, i, g32);
      if (t.m) t.m[i] = one(g, t.m[i]);
      else s = fma((double)g, (double)g, s);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  __shared__ double red[4];
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) t.part[local] = ((red[0] + red[1]) + red[2]) + red[3];
}

// ---- a matrix's sums of squares, added up into the first ----
// Every tile of the next pass adds up its matrix's sums, 1024 of them 8 KiB from L2, for which a launch would cost more.  Of more
// than that a workgroup makes one, or the pass would read as the square of the matrix (4096 x 131072 without steps 1.7 instead of
// 5.4 ms, 32768 x 65536 6.2 instead of 70; 4096 x 8192 0.090 and 0.094).
__global__ __launch_bounds__(1024) void muon_norm_kernel(MuBatch b) {
  const uint32_t wg = blockIdx.x;
  const MuTensor& t = b.t[mu_entry(b.count, wg, [&](int i) { return b.t[i].first; })];
  const int tid = threadIdx.x;
  const int64_t chunks = (t.rows * t.cols + MU_CHUNK - 1) / MU_CHUNK;
  double* const part = t.part + (wg - t.first) * chunks;
  double s = 0.;
#pragma unroll 8
  for (int64_t k = tid; k < chunks; k += 1024) s += part[k];
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  __shared__ double red[16];
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();  // every sum is read
  if (tid) return;
  for (int w = 1; w < 16; ++w) s += red[w];
  part[0] = s;
}

// A tile of 64 x 64 of one matrix: `x` tile (ti, tj) of the workspace, whose source tile is the same or, of a tall
// matrix, the transposed one.
struct MuTile {
  int64_t base;   // first element of the matrix in its tensor
  int64_t at;     // first element of the tile in the workspace
  int64_t row0, col0;
  int panel;      // elements of MU_K columns there
  __device__ __forceinline__ int64_t element(int row, int col) const { return at + (int64_t)(col / MU_K) * panel + row * MU_K + col % MU_K; }
};
__device__ __forceinline__ MuTile mu_tile(const MuTensor& t, uint32_t local) {
  const bool tall = t.flags & MU_TALL;
  const int64_t m = tall ? t.cols : t.rows, n = tall ? t.rows : t.cols;
  const int64_t mt = (m + 63) / 64, nt = (n + 63) / 64;
  const uint32_t mat = local / t.per, k = local % t.per;
  const int64_t ti = k / nt, tj = k % nt;
  MuTile r;
  r.base = (int64_t)mat * t.rows * t.cols;
  r.panel = (int)mt * 64 * MU_K;
  r.at = (int64_t)mat * mt * 64 * nt * 64 + tj * (64 / MU_K) * r.panel + ti * 64 * MU_K;
  r.row0 = (tall ? tj : ti) * 64;
  r.col0 = (tall ? ti : tj) * 64;
  return r;
}

// ---- X = u / |u| as fp16 (and what that leaves, as another), zero beyond the matrix ----
__global__ __launch_bounds__(256) void muon_pack_kernel(MuBatch b) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const uint32_t wg = blockIdx.x;
  const MuTensor& t = b.t[mu_entry(b.count, wg, [&](int i) { return b.t[i].first; })];
  const uint32_t local = wg - t.first, mat = local / t.per;
  const MuTile x = mu_tile(t, local);
  const int tid = threadIdx.x;
  const bool g32 = t.flags & MU_G32, nesterov = t.flags & MU_NESTEROV, tall = t.flags & MU_TALL;
  const int64_t n = t.rows * t.cols;
  const uint32_t chunks = (uint32_t)((n + MU_CHUNK - 1) / MU_CHUNK);
  double s = 0.;
  for (uint32_t k = tid; k < (chunks > MU_SUMS ? 1 : chunks); k += 256) s += t.part[(int64_t)mat * chunks + k];
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  const double norm = sqrt(((red[0] + red[1]) + red[2]) + red[3]);
  const MuScale scale = mu_scale(norm, b.eps);
  const int r = tid >> 4, c = (tid & 15) * 4;
  auto write = [&](int row, const float (&v)[4]) {
    f16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      h[e] = (f16)v[e];
      l[e] = (f16)(v[e] - (float)h[e]);
    }
    const int64_t at = x.element(row, c);
    *(f16x4*)(t.x + at) = h;
    *(f16x4*)(t.xlo + at) = l;
  };
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t row = x.row0 + 16 * k + r, col = x.col0 + c, i = x.base + row * t.cols + col;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    auto one = [&](float g, float m) { return scale(t.m ? nesterov ? fmaf(b.mu, m, b.omu * g) : m : g); };
    if (row < t.rows) {
      if ((t.flags & MU_ALIGNED) && col + 4 <= t.cols) {
        const f32x4 g = t.m && !nesterov ? (f32x4){0.f, 0.f, 0.f, 0.f} : mu_load4(t.g, i, g32);
        const f32x4 m = t.m ? *(const f32x4*)(t.m + i) : g;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = one(g[e], m[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < t.cols) v[e] = one(mu_load(t.g, i + e, g32), t.m ? t.m[i + e] : 0.f);
      }
    }
    if (!tall) write(16 * k + r, v);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (tall) tile[16 * k + r][c + e] = v[e];
  }
  if (!tall) return;  // uniform
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) write(16 * k + r, {tile[c][16 * k + r], tile[c + 1][16 * k + r], tile[c + 2][16 * k + r], tile[c + 3][16 * k + r]});
}

// ---- the weights' update from X, or X itself ----
__global__ __launch_bounds__(256) void muon_apply_kernel(MuBatch b) {
  __shared__ float tile[64][65];
  const uint32_t wg = blockIdx.x;
  const MuTensor& t = b.t[mu_entry(b.count, wg, [&](int i) { return b.t[i].first; })];
  const MuTile x = mu_tile(t, wg - t.first);
  const int tid = threadIdx.x, r = tid >> 4, c = (tid & 15) * 4;
  const bool p32 = t.flags & MU_P32, tall = t.flags & MU_TALL, step = t.flags & MU_STEP, two = t.flags & MU_LO;
  const bool wide = (t.flags & MU_ALIGNED) && x.col0 + c + 4 <= t.cols;
  const int64_t first = x.base + (x.row0 + r) * t.cols + x.col0 + c;
  f32x4 p[4] = {}, v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t i = first + 16 * k * t.cols;
    if (!step || x.row0 + 16 * k + r >= t.rows) continue;
    if (wide) p[k] = t.master ? *(const f32x4*)(t.master + i) : mu_load4(t.p, i, p32);
    else
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (x.col0 + c + e < t.cols) p[k][e] = t.master ? t.master[i + e] : mu_load(t.p, i + e, p32);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t at = x.element(16 * k + r, c);
    const f16x4 h = *(const f16x4*)(t.x + at), l = two ? *(const f16x4*)(t.xlo + at) : (f16x4){};
#pragma unroll
    for (int e = 0; e < 4; ++e) v[k][e] = ((float)h[e] + (float)l[e]) * (1.f / MU_X);
  }
  if (tall) {  // uniform
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[c + e][16 * k + r] = v[k][e];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = tile[16 * k + r][c + e];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t i = first + 16 * k * t.cols;
    if (x.row0 + 16 * k + r >= t.rows) continue;
    if (step)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = fmaf(-t.rate, v[k][e], p[k][e] * t.decay);
    if (wide) {
      if (t.master) *(f32x4*)(t.master + i) = v[k];
      if (p32) *(f32x4*)((float*)t.p + i) = v[k];
      else *(u32x2*)((bf16*)t.p + i) = (u32x2){pack_bf16x2(v[k][0], v[k][1]), pack_bf16x2(v[k][2], v[k][3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (x.col0 + c + e >= t.cols) continue;
        if (t.master) t.master[i + e] = v[k][e];
        if (p32) ((float*)t.p)[i + e] = v[k][e];
        else ((bf16*)t.p)[i + e] = (bf16)v[k][e];
      }
    }
  }
}

// ---- the products ----
struct MuShape {
  const f16* x;   // rows of the product, K along them
  const f16* w;   // its columns: [columns, K], in UPDATE [K, columns]
  const f16* d;   // what the product is added to
  f16* out;
  int mp, np, count;
  int tiles;      // of all its matrices
  int flags;
};
struct MuGemm {
  MuShape s[MU_PER];
  uint32_t first[MU_PER];  // a shape's first workgroup
  int count;
  float alpha, beta;  // of the product and of d
};
static_assert(sizeof(MuGemm) <= 4096, "kernel arguments");
enum { MU_GRAM = 0, MU_POLY = 1, MU_UPDATE = 2 };
enum { MU_LO_IN = 1, MU_LO_OUT = 2 };  // d has, out gets its second fp16

// Chunks of 16 bytes of an LDS row of MU_K columns are stored at their index xor this: the 16 rows that an instruction's
// lanes read at one chunk lie in all banks.  (Rows that are read transposed, 4 of 64 bytes at once, are so by themselves.)
__device__ __forceinline__ int mu_swz(int row) { return (row >> 2) & 3; }

// 32 x 32 fp16 as the matrix instructions leave them, a lane with columns 8 q + 4 hi .. + 3 of row l32 in halves q & 1 of
// w[q / 2], to rows as memory has them: w[t] is columns mu_chunk(lane) .. + 7 of row 16 t + lane % 16, so that 64 lanes
// write 1 KiB in one piece.  mu_unrows is the way back.
__device__ __forceinline__ void mu_swap32(u32x4& w) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const auto r = __builtin_amdgcn_permlane32_swap(w[x], w[x + 2], false, false);
    w[x] = r[0];
    w[x + 2] = r[1];
  }
}
__device__ __forceinline__ void mu_swap16(u32x4 (&w)[2]) {
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const auto r = __builtin_amdgcn_permlane16_swap(w[0][x], w[1][x], false, false);
    w[0][x] = r[0];
    w[1][x] = r[1];
  }
}
__device__ __forceinline__ void mu_rows(u32x4 (&w)[2]) {
  mu_swap32(w[0]);
  mu_swap32(w[1]);
  mu_swap16(w);
}
__device__ __forceinline__ void mu_unrows(u32x4 (&w)[2]) {
  mu_swap16(w);
  mu_swap32(w[0]);
  mu_swap32(w[1]);
}
__device__ __forceinline__ int mu_chunk(int lane) { return 16 * ((lane >> 4) & 1) + 8 * (lane >> 5); }
// Four lanes with four columns each of one row after the other: the transpose, lane k with column k of the four rows.
__device__ __forceinline__ u32x2 mu_quads(u32x2 w, int lane) {
  const bool odd = lane & 1, up = lane & 2;
  uint32_t e[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {  // columns 2 x + odd of rows lane & ~1, + 1
    const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)w[x], 0xb1, 0xf, 0xf, true);
    e[x] = odd ? __builtin_amdgcn_perm(w[x], o, 0x07060302) : __builtin_amdgcn_perm(o, w[x], 0x05040100);
  }
  const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)(up ? e[0] : e[1]), 0x4e, 0xf, 0xf, true);
  return up ? (u32x2){o, e[1]} : (u32x2){e[0], o};
}

template <int N>
__device__ __forceinline__ void mu_wait() {  // all but the last N copies have landed
  static_assert(N < 64, "vmcnt");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

// T x T tiles of one product, by WGM x WGN waves with v_mfma_f32_32x32x16_f16, whose A operand the product's columns are: a
// lane owns four consecutive columns of one row.  Both operands (PARTS 2: and their second fp16) stream into an LDS ring of
// NST stages of MU_K columns (buffer_load ... lds); the fragments of 16 columns are read while those before them
// multiply, over the stages' borders too, so stage kt + 1 has landed when kt begins.
// Bound by the matrix instructions and the power that they draw (the clock falls from 2.4 to 1.8 GHz): 48 matrices 960 x 960 to 960 x
// 3840 of two fp16, P X 853 us (896 TFLOP/s of what it multiplies), X X^T 539; of one fp16 P X 312 us (814 TFLOP/s; a library
// product of 960 x 960 x 3840 by 12 910, of 8192^3 1216), X X^T 178 us (716 of the half that is needed; 256 x 256 tiles on the diagonal
// and the edge are 42% more, of which 32 x 32 blocks that nobody writes are left out: 209 -> 194 us in a whole step, P X 385 -> 371);
// 79% of a 256 x 256 tile's cycles in the loop issue them, its start and epilogue are 26% of P X.  128 x 128 tiles wait for L2 (16 KiB a stage of 256 cycles); of two fp16
// they multiply three times and do not; there P X takes two stages only, so that another tile of the CU multiplies during
// one's start and epilogue (24 matrices of 640 columns 140 us, with five stages and one tile a CU 163; X X^T with its longer
// contraction 98 and 87).
template <int T, int WGM, int WGN, int NST, int PARTS, int MODE>
__global__ __launch_bounds__(64 * WGM * WGN, 1) void muon_gemm_kernel(MuGemm p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr bool WT = MODE == MU_UPDATE, SYM = !WT;
  constexpr int NW = WGM * WGN, KS = MU_K / 16;
  constexpr int WTM = T / WGM, WTN = T / WGN, FM = WTM / 32, FN = WTN / 32;
  constexpr int ROWB = MU_K * 2, PB = T * ROWB, XB = PARTS * PB, STAGE = 2 * XB;  // one fp16 of an operand, an operand, a stage
  constexpr int LP = PB / 1024 / NW, COPIES = 2 * PARTS * LP;                      // 1-KiB copies a wave
  static_assert(WTM % 32 == 0 && WTN % 32 == 0 && PB % (1024 * NW) == 0 && NST >= 2, "layout");
  __shared__ __attribute__((aligned(1024))) char lds[NST * STAGE];

  const int tid = (int)__builtin_amdgcn_workitem_id_x();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  // Two waves of a SIMD are four apart: in a tile of 256 on the diagonal they have 6 to 14 blocks on and above it, of 16.
  const int wm = wave / WGN, wn = NW == 8 && SYM && wm ? WGN - 1 - wave % WGN : wave % WGN, l32 = lane & 31, hi = lane >> 5;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  // Each shape's tiles are dealt to the XCDs in blocks: one matrix's on one XCD, every XCD with its share of every shape.
  const uint32_t wg = (uint32_t)__builtin_amdgcn_workgroup_id_x();
  MuShape s = p.s[0];  // loaded while the entries are looked over
  uint32_t first = 0;
  const int entry = __builtin_popcountll(__ballot(lane < p.count && p.first[lane < MU_PER ? lane : 0] <= wg)) - 1;
  if (entry) s = p.s[entry], first = p.first[entry];
  const int id = xcd_tile_order(s.tiles, (int)(wg - first));
  const int mp = s.mp, np = s.np, flags = s.flags, count = s.count;
  const int mt = (mp + T - 1) / T, nt = (np + T - 1) / T, per = SYM ? mt * (mt + 1) / 2 : mt * nt;
  const int mat = id / per, k = id % per;
  int tm, tn;
  if (SYM) {  // the k-th pair tm <= tn
    tn = (int)((sqrtf(8.f * (float)k + 1.f) - 1.f) * 0.5f);
    tn += (tn + 1) * (tn + 2) / 2 <= k;
    tn -= tn * (tn + 1) / 2 > k;
    tm = k - tn * (tn + 1) / 2;
  } else {
    tm = k % mt;
    tn = k / mt;
  }
  const int row0 = tm * T, n0 = tn * T;
  const int64_t square = (int64_t)mp * mp, wide = (int64_t)mp * np;
  const int64_t xs = MODE == MU_GRAM ? wide : square, ws = MODE == MU_POLY ? square : wide, os = MODE == MU_UPDATE ? wide : square;
  const int cols = SYM ? mp : np, nk = (MODE == MU_GRAM ? np : mp) / MU_K;
  const int panel = mp * MU_K;  // elements of MU_K columns
  const f16* xp = s.x + mat * xs + row0 * MU_K;
  const f16* wp = s.w + mat * ws + (WT ? (int64_t)(n0 / MU_K) * panel : n0 * MU_K);
  const int64_t xlo = count * xs, wlo = count * ws;

  // A stage is MU_K columns of T rows, 16 rows a copy, or (WT) MU_K rows of T columns, half a panel's a copy.
  uint32_t xo[LP], wo[LP];
#pragma unroll
  for (int j = 0; j < LP; ++j) {
    const int u = j * NW + wave, row = 16 * u + lane / 4;
    const uint32_t chunk = ((lane % 4) ^ mu_swz(row)) * 16;
    xo[j] = row0 + row < mp ? row * ROWB + chunk : OOB;
    if (WT) wo[j] = n0 + (u / 2) * MU_K < np ? (uint32_t)(u / 2) * (panel * 2) + (u % 2) * 1024 + lane * 16 : OOB;
    else wo[j] = n0 + row < mp ? row * ROWB + chunk : OOB;
  }
  uint32_t to = lds_base + wave * 1024;  // where the next stage goes
  int staged = 0;
  // Copies c0 .. c1 of the next stage; past the last one they read nothing and write zeros that nobody reads.
  auto issue = [&](int c0, int c1) {
#pragma unroll
    for (int c = c0; c < c1; ++c) {
      const int part = c / (2 * LP), j = c % LP, w = c / LP % 2;
      const f16* const base = (w ? wp : xp) + (part ? w ? wlo : xlo : 0);
      dma_row16(make_rsrc(base, staged < nk ? OOB : 0), to + w * XB + part * PB + j * NW * 1024, w ? wo[j] : xo[j]);
    }
    if (c1 == COPIES) {
      xp += panel;
      wp += WT ? MU_K * MU_K : panel;
      ++staged;
      to = to == lds_base + wave * 1024 + (NST - 1) * STAGE ? lds_base + wave * 1024 : to + STAGE;
    }
  };
#pragma unroll
  for (int q = 0; q < NST - 1; ++q) issue(0, COPIES);

  const int gn0 = n0 + wn * WTN, gr0 = row0 + wm * WTM;
  // Over the long contraction of X X^T the products with a second fp16 have a sum of their own, 2^-11 of the other: a third of the
  // roundings (8 x 1000 off by 1.1e-6 instead of 2.2e-6, 384 x 776 by 1.55e-6 instead of 1.65e-6; the times within 1%).
  constexpr int SUMS = PARTS == 2 && MODE == MU_GRAM ? 2 : 1;
  f32x16 acc[FN][FM], low[SUMS == 2 ? FN : 1][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        acc[i][j][r] = 0.f;
        if (SUMS == 2) low[i][j][r] = 0.f;
      }

  // LDS offsets of the fragments
  uint32_t aoff[FN][WT ? 1 : KS], boff[FM][KS];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    if (WT) {
      const int r4 = (lane & 15) >> 2, c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      aoff[i][0] = XB + ((wn * WTN + 32 * i) / MU_K) * (MU_K * ROWB) + (8 * hi + r4) * ROWB + c * 16 + 8 * (lane & 1);
    } else {
      const int row = wn * WTN + 32 * i + l32;
      for (int kk = 0; kk < KS; ++kk) aoff[i][WT ? 0 : kk] = XB + row * ROWB + ((2 * kk + hi) ^ mu_swz(row)) * 16;
    }
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int row = wm * WTM + 32 * j + l32;
    for (int kk = 0; kk < KS; ++kk) boff[j][kk] = row * ROWB + ((2 * kk + hi) ^ mu_swz(row)) * 16;
  }
  auto load_frags = [&](const char* st, int kk, f16x8 (&a)[PARTS][FN], f16x8 (&b)[PARTS][FM]) {
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        if constexpr (WT) {
          const char* q = st + aoff[i][0] + part * PB + kk * 16 * ROWB;
          typedef __fp16 h16x4 __attribute__((ext_vector_type(4)));
          const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(LDS_PTR(h16x4, q)));
          const f16x4 up = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(LDS_PTR(h16x4, q + 4 * ROWB)));
          a[part][i] = __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
          a[part][i] = *(const f16x8*)(st + part * PB + aoff[i][kk]);
        }
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) b[part][j] = *(const f16x8*)(st + part * PB + boff[j][kk]);
    }
  };

  constexpr int PRODUCTS = PARTS == 2 ? 3 : 1, GROUPS = KS * PRODUCTS * FN;
  f16x8 af[2][PARTS][FN], bf[2][PARTS][FM];
  constexpr bool AHEAD = NST > 2;  // two stages: the first fragments of one are read once it has landed, while other workgroups multiply
  if constexpr (AHEAD) {
    mu_wait<(NST - 2) * COPIES>();
    lds_barrier();
    load_frags(lds, 0, af[0], bf[0]);
  }
  // The 32 x 32 blocks of 32 columns that are written: none beyond the matrix, and none below the diagonal.  The others are not
  // multiplied, which saves their power more than time: a tile's slowest wave mostly has all of its blocks.
  int blocks[FN];
  bool every = true;
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    const int c0 = gn0 + 32 * i, last = SYM ? c0 : mp - 32;
    blocks[i] = c0 < cols && gr0 <= last ? min((last - gr0) / 32 + 1, FM) : 0;
    every = every && blocks[i] == FM;
  }
  auto loop = [&](auto all) {
    const char* st = lds;
    for (int kt = 0; kt < nk; ++kt) {
      mu_wait<AHEAD ? (NST - 3) * COPIES : 0>();
      wait_lgkm0();   // the slot of kt - 1 is read, and this stage's first fragments are there: no later wait counts them
      lds_barrier();  // stage kt + 1 (or kt) landed for every wave, and the slot of kt - 1 is free
      const char* const next = st == lds + (NST - 1) * STAGE ? lds : st + STAGE;
      if constexpr (!AHEAD) load_frags(st, 0, af[0], bf[0]);
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        const int cb = kk & 1;
        if (kk + 1 < KS) load_frags(st, kk + 1, af[cb ^ 1], bf[cb ^ 1]);
        else if (AHEAD) load_frags(next, 0, af[cb ^ 1], bf[cb ^ 1]);  // after the last stage: read for nothing
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int pr = 0; pr < PRODUCTS; ++pr)
#pragma unroll
          for (int i = 0; i < FN; ++i) {
#pragma unroll
            for (int j = 0; j < FM; ++j)
              if (decltype(all)::value || j < blocks[i]) {
                f32x16& sum = SUMS == 2 && pr ? low[SUMS == 2 ? i : 0][j] : acc[i][j];
                sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[cb][PARTS == 2 && pr == 1][i], bf[cb][PARTS == 2 && pr == 2][j], sum, 0, 0, 0);
              }
            // the copies between the products: issued at once they would hold up the products behind them
            const int g = (kk * PRODUCTS + pr) * FN + i;
            __builtin_amdgcn_sched_barrier(0);
            issue(COPIES * g / GROUPS, COPIES * (g + 1) / GROUPS);
            __builtin_amdgcn_sched_barrier(0);
          }
      }
      st = next;
    }
  };
  if (every) loop(std::true_type{});
  else loop(std::false_type{});
  wait_vmcnt(0);
  if constexpr (SUMS == 2)
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] += low[i][j][r];
  // ---- epilogue, 32 x 32 at a time in registers
  f16* const __restrict__ out = s.out + mat * os;
  const int64_t olo = count * os;  // from a value's first fp16 to its second
  const f16* const __restrict__ d = s.d + mat * os;
  auto element = [&](int row, int col) { return (int64_t)(col / MU_K) * panel + row * MU_K + col % MU_K; };
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    const int c0 = gn0 + 32 * i;
    if (c0 >= cols) continue;  // cols is a multiple of 64
    u32x4 dh[FM][2], dl[FM][2];  // what the columns are added to: all their loads before their stores
    if (MODE != MU_GRAM) {
#pragma unroll
      for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int64_t at = gr0 + 32 * j < mp ? element(gr0 + 32 * j + 16 * t + (lane & 15), c0 + mu_chunk(lane)) : 0;
          dh[j][t] = *(const u32x4*)(d + at);
          dl[j][t] = flags & MU_LO_IN ? *(const u32x4*)(d + olo + at) : (u32x4){};
        }
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      // Blocks below the diagonal are mirror images in the diagonal's tiles too: of two fp16 their sums have another order.
      if (gr0 + 32 * j >= mp || (SYM && gr0 + 32 * j > c0)) continue;
      const bool mirror = SYM && gr0 + 32 * j < c0;
      float v[16];
      if (MODE != MU_GRAM) {
        mu_unrows(dh[j]);
        if (flags & MU_LO_IN) mu_unrows(dl[j]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f16x8 h = __builtin_bit_cast(f16x8, dh[j][t]), l = __builtin_bit_cast(f16x8, dl[j][t]);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float a = acc[i][j][8 * t + x];
          v[8 * t + x] = mu_rounded(MODE == MU_GRAM ? a * p.alpha : fmaf(a, p.alpha, p.beta * ((float)h[x] + (float)l[x])));
        }
      }
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        if (part && !(flags & MU_LO_OUT)) break;
        f16* const o = out + part * olo;
        u32x4 w[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f16x8 h;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            h[x] = (f16)v[8 * t + x];
            v[8 * t + x] = v[8 * t + x] - (float)h[x];
          }
          w[t] = __builtin_bit_cast(u32x4, h);
          if (mirror) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
              *(u32x2*)(o + element(c0 + 16 * t + 8 * q + 4 * hi + (lane & 3), gr0 + 32 * j + (l32 & 28))) =
                  mu_quads((u32x2){w[t][2 * q], w[t][2 * q + 1]}, lane);
          }
        }
        mu_rows(w);
#pragma unroll
        for (int t = 0; t < 2; ++t) *(u32x4*)(o + element(gr0 + 32 * j + 16 * t + (lane & 15), c0 + mu_chunk(lane))) = w[t];
      }
    }
  }
#endif
}

// ---- P and X <- a X + P X of slim matrices in one launch ----
// A whole (at most 128 x 128) and 128 columns of X lie in LDS; a workgroup makes 64 rows of P from A for itself, which costs it 0.7 us
// where a launch costs 4 to 5, and multiplies them by its columns: eight waves with a 32 x 32 block each.  The same sums in
// the same order as muon_gemm_kernel's.  Bound by latencies: eight matrices of 128 columns
// in fp32 7.8 us (P and X by themselves 5.6 and 5.7), of which the start and 160 KiB of copies are 2.
struct MuSlim {
  MuShape s[MU_PER];  // x: A, w: X
  uint32_t first[MU_PER];
  int count;
  float a, b, c;
};
static_assert(sizeof(MuSlim) <= 4096, "kernel arguments");

template <int MP, int PARTS>
__global__ __launch_bounds__(512, 1) void muon_slim_kernel(MuSlim p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int AB = MP * MP * 2, XB = MP * 128 * 2, PB = 64 * MP * 2;  // bytes of one fp16 of A, of the columns, of 64 rows of P
  __shared__ __attribute__((aligned(1024))) char lds[PARTS * (AB + XB + PB)];
  char* const xl = lds + PARTS * AB;
  char* const pl = xl + PARTS * XB;
  const int tid = (int)__builtin_amdgcn_workitem_id_x();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint32_t wg = (uint32_t)__builtin_amdgcn_workgroup_id_x();
  MuShape s = p.s[0];
  uint32_t first = 0;
  const int entry = __builtin_popcountll(__ballot(lane < p.count && p.first[lane < MU_PER ? lane : 0] <= wg)) - 1;
  if (entry) s = p.s[entry], first = p.first[entry];
  const int np = s.np, flags = s.flags, across = (np + 127) / 128, per = MP / 64 * across;
  const int id = (int)(wg - first), mat = id / per, rest = id % per, r0 = rest / across * 64, n0 = rest % across * 128;
  const int64_t wide = (int64_t)MP * np;

  // Both are whole panels, 16 rows a copy.
  auto copy = [&](const f16* from, uint32_t to, int panels) {
    for (int u = wave; u < panels * (MP / 16); u += 8) {
      const int row = 16 * (u % (MP / 16)) + lane / 4;
      const uint32_t at = (uint32_t)(u / (MP / 16)) * (MP * MU_K * 2) + row * (MU_K * 2) + ((lane % 4) ^ mu_swz(row)) * 16;
      dma_row16(make_rsrc(from, OOB), to + u * 1024, at);
    }
  };
  const int panels = min(4, (np - n0) / MU_K);  // the rest of LDS is multiplied for nobody
#pragma unroll
  for (int q = 0; q < PARTS; ++q) {
    copy(s.x + mat * (int64_t)(MP * MP) + q * s.count * (int64_t)(MP * MP), lds_base + q * AB, MP / MU_K);
    copy(s.w + mat * wide + q * s.count * wide + (int64_t)n0 * MP, lds_base + PARTS * AB + q * XB, panels);
  }
  auto place = [](int rows, int row, int col) { return (col / MU_K) * (rows * MU_K * 2) + row * (MU_K * 2) + (((col % MU_K) / 8) ^ mu_swz(row)) * 16 + (col % 8) * 2; };
  const int br = wave / 4 * 32, bc = wave % 4 * 32;  // this wave's block: of X, and of the rows of P
  wait_vmcnt(0);
  lds_barrier();

  auto multiply = [&](f32x16& acc, const f16x8 (&w)[PARTS], const f16x8 (&x)[PARTS], bool lower) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(w[0], x[0], acc, 0, 0, 0);
    if constexpr (PARTS == 2) {  // below P's diagonal in the order of the block whose image it is
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(w[lower ? 0 : 1], x[lower ? 1 : 0], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(w[lower ? 1 : 0], x[lower ? 0 : 1], acc, 0, 0, 0);
    }
  };
  const int pr = MP == 64 ? wave / 2 * 32 : br, pc = MP == 64 ? wave % 2 * 32 : bc;
  auto square = [&](bool lower) {
    f32x16 acc = {};
#pragma unroll
    for (int k = 0; k < MP; k += 16) {
      f16x8 x[PARTS], w[PARTS];
#pragma unroll
      for (int q = 0; q < PARTS; ++q) {
        x[q] = *(const f16x8*)(lds + q * AB + place(MP, r0 + pr + l32, k + 8 * hi));
        w[q] = *(const f16x8*)(lds + q * AB + place(MP, pc + l32, k + 8 * hi));
      }
      multiply(acc, w, x, lower);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = place(MP, r0 + pr + l32, pc + 8 * q + 4 * hi), to = place(64, pr + l32, pc + 8 * q + 4 * hi);
      const f16x4 dh = *(const f16x4*)(lds + at), dl = PARTS == 2 ? *(const f16x4*)(lds + AB + at) : (f16x4){};
      f16x4 h, l;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float v = mu_rounded(fmaf(acc[4 * q + x], p.c / MU_A, p.b * ((float)dh[x] + (float)dl[x])));
        h[x] = (f16)v;
        l[x] = (f16)(v - (float)h[x]);
      }
      *(f16x4*)(pl + to) = h;
      if (PARTS == 2) *(f16x4*)(pl + PB + to) = l;
    }
  };
  if (MP == 128 || wave < 4) {
    if (r0 + pr > pc) square(true);
    else square(false);
  }
  __syncthreads();

  const int c0 = n0 + bc;
  if (c0 >= np) return;
  f32x16 acc = {};
#pragma unroll
  for (int k = 0; k < MP; k += 16) {
    f16x8 x[PARTS], w[PARTS];
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      typedef __fp16 h16x4 __attribute__((ext_vector_type(4)));
      const int row = k + 8 * hi + ((lane & 15) >> 2), col = bc + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      const char* const m = xl + q * XB;
      const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(LDS_PTR(h16x4, m + place(MP, row, col))));
      const f16x4 up = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(LDS_PTR(h16x4, m + place(MP, row + 4, col))));
      w[q] = __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
      x[q] = *(const f16x8*)(pl + q * PB + place(64, br + l32, k + 8 * hi));
    }
    multiply(acc, w, x, false);
  }
  // a X: X's second fp16 from LDS, or (of the first steps where only a X has it) from memory
  const int64_t panel = MP * MU_K, block = (int64_t)(c0 / MU_K) * panel + (r0 + br) * MU_K;
  float v[16];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int at = place(MP, r0 + br + l32, bc + 8 * q + 4 * hi);
    const f16x4 h = *(const f16x4*)(xl + at);
    f16x4 l = {};
    if (PARTS == 2) l = *(const f16x4*)(xl + XB + at);
    else if (flags & MU_LO_IN) l = *(const f16x4*)(s.w + (s.count + mat) * wide + block + l32 * MU_K + 8 * q + 4 * hi);
#pragma unroll
    for (int x = 0; x < 4; ++x) v[4 * q + x] = mu_rounded(fmaf(acc[4 * q + x], 1.f / MU_A, p.a * ((float)h[x] + (float)l[x])));
  }
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    if (part && !(flags & MU_LO_OUT)) break;
    f16* const o = s.out + (part * s.count + mat) * wide + block;
    u32x4 w[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f16x8 h;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        h[x] = (f16)v[8 * t + x];
        v[8 * t + x] = v[8 * t + x] - (float)h[x];
      }
      w[t] = __builtin_bit_cast(u32x4, h);
    }
    mu_rows(w);
#pragma unroll
    for (int t = 0; t < 2; ++t) *(u32x4*)(o + (16 * t + (lane & 15)) * MU_K + mu_chunk(lane)) = w[t];
  }
#endif
}

// ---- small matrices: the whole step in one workgroup and launch ----
// X (as two fp16) and A, which P takes the place of, stay in LDS, in the workspace's layout.  Sixteen waves take a 32 x 32
// block of a product of 128 x 128 each (eight take two: 30 us, of one fp16), eight one of 64 x 64 with half of the contraction.  Bound by
// latencies and the conversions of the results: 128 x 128 alone 49 us, of one fp16 24 (eighteen launches: 77), of which a step is
// 8300 cycles with 3 x 1024 of matrix instructions, and 16000 go into u, its norm and the result.
constexpr int MU_SMALL_PER = 32;  // tensors a launch
struct MuSmall {
  MuTensor t[MU_SMALL_PER];
  float co[64][3];
  int count, steps;
  float mu, omu;
  double eps;
};
static_assert(sizeof(MuSmall) <= 4096, "kernel arguments");

// MP x n matrices, n <= NP: the shorter side rounded up to MP, the longer one to 64.
template <int MP, int NP, int PARTS>
__global__ __launch_bounds__(MP == 64 ? 512 : 1024, 1) void muon_small_kernel(MuSmall b) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int XB = MP * NP * 2, AB = MP * MP * 2;  // bytes of one fp16 of X, of A
  constexpr int HALVES = MP == 64 ? 2 : 1;           // of a contraction, to a wave each
  constexpr int NT = MP == 64 ? 512 : 1024, NW = NT / 64, UB = MP * NP / 1024 / NW;  // threads, waves, blocks of X a wave (of A one)
  __shared__ __attribute__((aligned(1024))) char lds[2 * XB + PARTS * AB + (HALVES == 2 ? MP * MP * 4 : 0)];
  __shared__ double red[NW];
  char* const xl = lds;
  char* const al = lds + 2 * XB;
  float* const shares = (float*)(al + PARTS * AB);

  const uint32_t wg = blockIdx.x;
  const MuTensor& t = b.t[mu_entry(b.count, wg, [&](int i) { return b.t[i].first; })];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, hi = lane >> 5;
  const int rows = (int)t.rows, cols = (int)t.cols, n = rows * cols;
  const bool tall = t.flags & MU_TALL, g32 = t.flags & MU_G32, p32 = t.flags & MU_P32, nesterov = t.flags & MU_NESTEROV;
  const bool aligned = t.flags & MU_ALIGNED, step = t.flags & MU_STEP;
  const int np = ((tall ? rows : cols) + 63) / 64 * 64;
  const int64_t base = (int64_t)(wg - t.first) * n;

  // Element (row, col) of a matrix of MP rows in panels of 32 columns, 16-byte chunks swizzled.
  auto place = [](int row, int col) { return (col / MU_K) * (MP * MU_K * 2) + row * (MU_K * 2) + (((col % MU_K) / 8) ^ mu_swz(row)) * 16 + (col % 8) * 2; };

  for (int i = tid; i < 2 * XB / 16; i += NT) *(u32x4*)(xl + 16 * i) = (u32x4){};
  __syncthreads();
  // Runs of four elements where they lie in one row and memory allows, or single ones.  The loops are short: a workgroup alone
  // fetches every instruction of them anew, and unrolled to the end they took three times as long.
  const float inverse = 1.f / (float)cols;
  auto row_of = [&](int e) { return (int)(((float)e + 0.5f) * inverse); };  // e / cols: off from the next one by 1 / 2 cols, e < 2^21
  auto at_of = [&](int e) {
    const int row = row_of(e), col = e - row * cols;
    return tall ? place(col, row) : place(row, col);
  };
  // u, and m <- mu m + (1 - mu) g.  u's upper and lower 16 bits take the places of X's two fp16 until the norm is known.
  double s = 0.;
  auto momentum = [&](float g, float& m) {
    m = fmaf(b.mu, m, b.omu * g);
    const float u = !t.m ? g : nesterov ? fmaf(b.mu, m, b.omu * g) : m;
    s = fma((double)u, (double)u, s);
    return __float_as_uint(u);
  };
  if (aligned) {
#pragma unroll 4
    for (int e0 = 4 * tid; e0 < n; e0 += 4 * NT) {
      const f32x4 g = mu_load4(t.g, base + e0, g32);
      f32x4 m = t.m ? *(const f32x4*)(t.m + base + e0) : (f32x4){};
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = m[e];
        u[e] = momentum(g[e], v);
        m[e] = v;
      }
      if (t.m) *(f32x4*)(t.m + base + e0) = m;
      const int at = at_of(e0);
      if (!tall) {
        *(u32x2*)(xl + at) = (u32x2){__builtin_amdgcn_perm(u[1], u[0], 0x07060302), __builtin_amdgcn_perm(u[3], u[2], 0x07060302)};
        *(u32x2*)(xl + XB + at) = (u32x2){__builtin_amdgcn_perm(u[1], u[0], 0x05040100), __builtin_amdgcn_perm(u[3], u[2], 0x05040100)};
      } else {  // four rows of one swizzle
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          *(uint16_t*)(xl + at + e * MU_K * 2) = (uint16_t)(u[e] >> 16);
          *(uint16_t*)(xl + XB + at + e * MU_K * 2) = (uint16_t)u[e];
        }
      }
    }
  } else {
#pragma unroll 4
    for (int e = tid; e < n; e += NT) {
      float m = t.m ? t.m[base + e] : 0.f;
      const uint32_t u = momentum(mu_load(t.g, base + e, g32), m);
      if (t.m) t.m[base + e] = m;
      const int at = at_of(e);
      *(uint16_t*)(xl + at) = (uint16_t)(u >> 16);
      *(uint16_t*)(xl + XB + at) = (uint16_t)u;
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  s = 0.;
#pragma unroll
  for (int w = 0; w < NW; ++w) s += red[w];
  const MuScale scale = mu_scale(sqrt(s), b.eps);
#pragma unroll 2
  for (int i = tid; i < MP * np / 4; i += NT) {
    u32x2* const hp = (u32x2*)(xl + 8 * i);
    u32x2* const lp = (u32x2*)(xl + XB + 8 * i);
    const u32x2 up = *hp, low = *lp;
    f16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = __builtin_amdgcn_perm(up[e / 2], low[e / 2], e % 2 ? 0x07060302 : 0x05040100);
      const float v = scale(__uint_as_float(u));
      h[e] = (f16)v;
      l[e] = (f16)(v - (float)h[e]);
    }
    *(f16x4*)hp = h;
    *(f16x4*)lp = l;
  }
  __syncthreads();

  typedef __fp16 h16x4 __attribute__((ext_vector_type(4)));
  auto frag = [&](const char* m, int row, int k0) { return *(const f16x8*)(m + place(row, k0 + 8 * hi)); };  // 16 columns from k0 on
  auto frag_t = [&](const char* m, int k0, int c0) {  // rows k0 .. + 15 of columns c0 .. + 31, transposed
    const int row = k0 + 8 * hi + ((lane & 15) >> 2), col = c0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(LDS_PTR(h16x4, m + place(row, col))));
    const f16x4 up = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(LDS_PTR(h16x4, m + place(row + 4, col))));
    return __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // The products with a second fp16 have a sum of their own, 2^-11 of the other, whose roundings are nothing beside it.  That of
  // two second ones is 2^-24 of a value, but of one sign on A's diagonal, which few rows show: 8 x 200 off by 0.83e-6 (0.96e-6
  // without it, 1.08e-6 in one sum; 0.77e-6 with products of fp32) in 32 us instead of 29, 128 x 128 0.77e-6 (0.84, 1.11; 1.34).
  auto multiply = [&](f32x16& acc, f32x16& low, const f16x8 (&a)[PARTS], const f16x8 (&c)[PARTS]) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], c[0], acc, 0, 0, 0);
    if constexpr (PARTS == 2) {
      low = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], c[0], low, 0, 0, 0);
      low = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], c[1], low, 0, 0, 0);
      low = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], c[1], low, 0, 0, 0);
    }
  };
  auto join = [&](f32x16& acc, const f32x16& low) {
    if constexpr (PARTS == 2)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] += low[r];
  };
  // Blocks of m m^T, m [MP, K] at stride `part` between its two fp16: of a wave, with its share of the contraction.
  auto square = [&](f32x16& acc, const char* m, int part, int K) {
    const int half = HALVES == 2 ? wave / 4 : 0, block = HALVES == 2 ? wave % 4 : wave;
    const int r0 = block / (MP / 32) * 32, k0 = half * (K / HALVES), k1 = k0 + K / HALVES;
    f32x16 low = {};
    acc = (f32x16){};
#pragma unroll 2
    for (int k = k0; k < k1; k += 32) {  // K is a multiple of 64
      f16x8 x[2][PARTS], w[2][PARTS];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
          x[kk][q] = frag(m + q * part, r0 + l32, k + 16 * kk);
          w[kk][q] = frag(m + q * part, block % (MP / 32) * 32 + l32, k + 16 * kk);
        }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) multiply(acc, low, w[kk], x[kk]);
    }
    join(acc, low);
    if constexpr (HALVES == 2) {  // the upper waves' shares are added to the lower ones'
      if (half)
#pragma unroll
        for (int r = 0; r < 4; ++r) *(f32x4*)(shares + ((block * 4 + r) * 64 + lane) * 4) = (f32x4){acc[4 * r], acc[4 * r + 1], acc[4 * r + 2], acc[4 * r + 3]};
      __syncthreads();
      if (!half)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] += shares[((block * 4 + r / 4) * 64 + lane) * 4 + r % 4];
    }
  };
  // alpha acc + beta d at block (r0, c0) of a matrix, four columns at once, written over d once every wave has read.
  auto combine = [&](f32x16& acc, const char* d, int part, bool two, int r0, int c0, float alpha, float beta) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = place(r0 + l32, c0 + 8 * q + 4 * hi);
      f16x4 h = {}, l = {};
      if (d) h = *(const f16x4*)(d + at);
      if (d && two) l = *(const f16x4*)(d + part + at);
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[4 * q + x] = fmaf(acc[4 * q + x], alpha, beta * ((float)h[x] + (float)l[x]));
    }
  };
  auto write = [&](const f32x16& acc, char* o, int part, bool two, int r0, int c0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = place(r0 + l32, c0 + 8 * q + 4 * hi);
      f16x4 h, l;
      if (two) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float v = mu_rounded(acc[4 * q + x]);
          h[x] = (f16)v;
          l[x] = (f16)(v - (float)h[x]);
        }
        *(f16x4*)(o + part + at) = l;
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) h[x] = (f16)acc[4 * q + x];
      }
      *(f16x4*)(o + at) = h;
    }
  };
  const int block = HALVES == 2 ? wave % 4 : wave, r0 = block / (MP / 32) * 32, c0 = block % (MP / 32) * 32;
  const bool mine = HALVES == 1 || wave < 4;  // holds blocks of A and P
  for (int k = 0; k < b.steps; ++k) {
    f32x16 acc;
    square(acc, xl, XB, np);
    if (mine) {
      combine(acc, nullptr, 0, false, 0, 0, MU_A / (MU_X * MU_X), 0.f);
      write(acc, al, AB, PARTS == 2, r0, c0);
    }
    __syncthreads();
    square(acc, al, AB, MP);
    if (mine) combine(acc, al, AB, PARTS == 2, r0, c0, b.co[k][2] / MU_A, b.co[k][1]);
    __syncthreads();
    if (mine) write(acc, al, AB, PARTS == 2, r0, c0);
    __syncthreads();
    f32x16 x[UB];
#pragma unroll
    for (int i = 0; i < UB; ++i) {
      const int blk = wave + NW * i, rr = blk % (MP / 32) * 32, cc = blk / (MP / 32) * 32;
      if (cc >= np) continue;
      f32x16 low = {};
      x[i] = (f32x16){};
#pragma unroll
      for (int kk = 0; kk < MP; kk += 16) {
        f16x8 w[PARTS], p[PARTS];
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
          w[q] = frag_t(xl + q * XB, kk, cc);
          p[q] = frag(al + q * AB, rr + l32, kk);
        }
        multiply(x[i], low, w, p);
      }
      join(x[i], low);
      combine(x[i], xl, XB, PARTS == 2 || k < MU_LO_STEPS, rr, cc, 1.f / MU_A, b.co[k][0]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < UB; ++i) {
      const int blk = wave + NW * i, rr = blk % (MP / 32) * 32, cc = blk / (MP / 32) * 32;
      if (cc < np) write(x[i], xl, XB, PARTS == 2 || k + 1 < MU_LO_STEPS, rr, cc);
    }
    __syncthreads();
  }

  auto value = [&](int at) { return ((float)*(const f16*)(xl + at) + (PARTS == 2 ? (float)*(const f16*)(xl + XB + at) : 0.f)) * (1.f / MU_X); };
  if (aligned) {
#pragma unroll 4
    for (int e0 = 4 * tid; e0 < n; e0 += 4 * NT) {
      f32x4 p = {}, v;
      if (step) p = t.master ? *(const f32x4*)(t.master + base + e0) : mu_load4(t.p, base + e0, p32);
      const int at = at_of(e0);
      if (!tall) {
        const f16x4 h = *(const f16x4*)(xl + at), l = PARTS == 2 ? *(const f16x4*)(xl + XB + at) : (f16x4){};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ((float)h[e] + (float)l[e]) * (1.f / MU_X);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = value(at + e * MU_K * 2);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (step) v[e] = fmaf(-t.rate, v[e], p[e] * t.decay);
      }
      if (t.master) *(f32x4*)(t.master + base + e0) = v;
      if (p32) *(f32x4*)((float*)t.p + base + e0) = v;
      else *(u32x2*)((bf16*)t.p + base + e0) = (u32x2){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    }
  } else {
#pragma unroll 4
    for (int e = tid; e < n; e += NT) {
      float v = value(at_of(e));
      if (step) v = fmaf(-t.rate, v, (t.master ? t.master[base + e] : mu_load(t.p, base + e, p32)) * t.decay);
      if (t.master) t.master[base + e] = v;
      if (p32) ((float*)t.p)[base + e] = v;
      else ((bf16*)t.p)[base + e] = (bf16)v;
    }
  }
#endif
}

// ---- the host's side ----
struct MuGroup {  // matrices of one shape and precision
  int64_t m, n, mp, np, count;
  bool precise;
  int64_t x[2], a, p;  // elements into the workspace's fp16: X and the one that takes the next, A, P
};
struct MuPlan {
  std::vector<MuGroup> groups;
  std::vector<int> of;             // a tensor's group, or -1: empty, or all are small
  std::vector<int64_t> at, parts;  // its first matrix there, and its first sum of squares
  int64_t sums = 0, halves = 0, bytes = 0;
};

// Matrices that a workgroup can take whole: the variant of muon_small_kernel, or -1.
static int mu_small(const strata_hip_muon_matrix& t) {
  const int64_t m = std::min(t.rows, t.cols), n = std::max(t.rows, t.cols);
  return m <= 64 && n <= 128 ? 0 : m <= 64 && n <= 384 ? 1 : n <= 128 ? 2 : -1;
}
// Whether a matrix's operands are two fp16.  With few singular values (at most 64) one fp16's roundings do not even out: 3 to 4e-3 of
// a row's result, 2.5e-3 of 24 x 960.  Such matrices are small beside the others of a call, and so is what three products of theirs cost.
static bool mu_precise(const strata_hip_muon_matrix& t) {
  return std::min(t.rows, t.cols) <= 64 || (t.bits ? t.bits == 22 : t.precise != 0);
}
// What a call's matrices all are.
struct MuCall {
  // Small.  Beside others such matrices go with them, whose launches they do not lengthen (two of 128 x 128 among eight
  // matrices in fp32: 109 us; first by themselves 150).
  bool small = true;
  // At most 128 on the shorter side: a step is two launches (muon_slim_kernel).
  bool slim = true;
};
static MuCall mu_call(const strata_hip_muon_matrix* ts, int64_t count) {
  MuCall c;
  for (int64_t i = 0; i < count; ++i) {
    if (!ts[i].rows || !ts[i].cols || !ts[i].batch) continue;
    c.small &= mu_small(ts[i]) >= 0;
    c.slim &= std::min(ts[i].rows, ts[i].cols) <= 128;
  }
  return c;
}
static int64_t mu_chunks(const strata_hip_muon_matrix& t) { return (t.rows * t.cols + MU_CHUNK - 1) / MU_CHUNK; }
static int64_t mu_up(int64_t n) { return (n + MU_PAD - 1) / MU_PAD * MU_PAD; }

// The sizes that the kernels' indexes and grids hold: at most 2^22 tiles of 64 x 64 in all.
static int mu_sizes(const std::string& n, const strata_hip_muon_matrix* ts, int64_t count) {
  int64_t tiles = 0;
  for (int64_t i = 0; i < count; ++i) {
    const strata_hip_muon_matrix& t = ts[i];
    if (t.rows < 0 || t.cols < 0 || t.batch < 0) return fail(STRATA_HIP_EINVAL, n + ": negative size");
    if (!t.rows || !t.cols || !t.batch) continue;
    if (t.rows > (1 << 20) || t.cols > (1 << 20) || t.batch > (1 << 20) || std::min(t.rows, t.cols) > (1 << 15) ||
        t.rows * t.cols > (1ll << 31) / t.batch || mu_up(t.rows) * mu_up(t.cols) / 4096 > (1 << 22) / t.batch ||
        (tiles += mu_up(t.rows) * mu_up(t.cols) / 4096 * t.batch) > (1 << 22))
      return fail(STRATA_HIP_EUNSUPPORTED, n + ": matrices of at most 2^20 rows and columns (the shorter side 2^15), 2^31 elements a tensor and "
                                               "2^34 together, each side counted as the next multiple of 64");
  }
  return STRATA_HIP_OK;
}

// A matrix has room for two fp16 a value of X; A and P have it where `precise`.
static MuPlan mu_plan(const strata_hip_muon_matrix* ts, int64_t count) {
  MuPlan q;
  const MuCall call = mu_call(ts, count);
  std::map<std::tuple<int64_t, int64_t, bool>, int> seen;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t m = std::min(ts[i].rows, ts[i].cols), n = std::max(ts[i].rows, ts[i].cols);
    const bool precise = mu_precise(ts[i]);
    q.at.push_back(0);
    q.parts.push_back(q.sums);
    if (m <= 0 || ts[i].batch <= 0 || call.small) {
      q.of.push_back(-1);
      continue;
    }
    const auto in = seen.emplace(std::make_tuple(m, n, precise), (int)q.groups.size());
    if (in.second) q.groups.push_back({m, n, mu_up(m), mu_up(n), 0, precise, {0, 0}, 0, 0});
    MuGroup& g = q.groups[(size_t)in.first->second];
    q.of.push_back(in.first->second);
    q.at.back() = g.count;
    g.count += ts[i].batch;
    q.sums += ts[i].batch * mu_chunks(ts[i]);
  }
  for (MuGroup& g : q.groups) {
    auto take = [&](int64_t n) {
      const int64_t at = q.halves;
      q.halves += n;
      return at;
    };
    for (int64_t& x : g.x) x = take(2 * g.count * g.mp * g.np);
    g.a = take((g.precise ? 2 : 1) * g.count * g.mp * g.mp);
    // narrow ones' P does not leave LDS in a slim call
    g.p = call.slim && g.mp == MU_PAD ? 0 : take((g.precise ? 2 : 1) * g.count * g.mp * g.mp);
  }
  q.bytes = (q.sums * 8 + 255) / 256 * 256 + q.halves * 2;
  return q;
}

static int mu_check(const std::string& n, const strata_hip_muon_args* a, bool step) {
  if (!a) return fail(STRATA_HIP_EINVAL, n + ": null args");
  if (a->count < 0 || (a->count > 0 && !a->matrices)) return fail(STRATA_HIP_EINVAL, n + ": bad list of matrices");
  if (a->steps < 0 || a->steps > 64 || (a->steps > 0 && !a->coefficients))
    return fail(STRATA_HIP_EINVAL, n + ": between 0 and 64 steps, with their coefficients");
  for (int i = 0; i < 3 * a->steps; ++i)
    if (!std::isfinite(a->coefficients[i])) return fail(STRATA_HIP_EINVAL, n + ": coefficients must be finite");
  if (!(a->eps > 0.) || !std::isfinite(a->eps)) return fail(STRATA_HIP_EINVAL, n + ": eps must be positive and finite");
  if (step && !(a->momentum >= 0. && a->momentum < 1.)) return fail(STRATA_HIP_EINVAL, n + ": momentum must lie in [0, 1)");
  if (a->adjust != STRATA_HIP_ADJUST_ORIGINAL && a->adjust != STRATA_HIP_ADJUST_MATCH_RMS_ADAMW)
    return fail(STRATA_HIP_EINVAL, n + ": bad adjust");
  if (const int rc = mu_sizes(n, a->matrices, a->count)) return rc;
  std::vector<std::pair<uintptr_t, uintptr_t>> written, read;
  for (int64_t i = 0; i < a->count; ++i) {
    const strata_hip_muon_matrix& t = a->matrices[i];
    if (!t.rows || !t.cols || !t.batch) continue;
    if (step && (!std::isfinite(t.lr) || !std::isfinite(t.weight_decay)))
      return fail(STRATA_HIP_EINVAL, n + ": lr and weight_decay must be finite");
    const bool p32 = t.param_dtype == STRATA_HIP_F32, g32 = t.grad_dtype == STRATA_HIP_F32;
    if ((!p32 && t.param_dtype != STRATA_HIP_BF16) || (!g32 && t.grad_dtype != STRATA_HIP_BF16))
      return fail(STRATA_HIP_EINVAL, n + ": matrices must be bf16 or f32");
    if (t.bits != 0 && t.bits != 11 && t.bits != 22) return fail(STRATA_HIP_EINVAL, n + ": operands have 11 or 22 bits");
    if (!t.param || !t.grad || (step && !t.momentum)) return fail(STRATA_HIP_EINVAL, n + ": null tensor");
    if (!step && t.momentum) return fail(STRATA_HIP_EINVAL, n + ": a momentum is the step's");
    if (t.master && (p32 || !step)) return fail(STRATA_HIP_EINVAL, n + ": master weights are for bf16 parameters");
    const uintptr_t ps = p32 ? 4 : 2, gs = g32 ? 4 : 2, all = (uintptr_t)(t.rows * t.cols * t.batch);
    if (((uintptr_t)t.param % ps) || ((uintptr_t)t.grad % gs) || ((uintptr_t)t.momentum % 4) || ((uintptr_t)t.master % 4))
      return fail(STRATA_HIP_EINVAL, n + ": a tensor is not aligned to its elements");
    read.emplace_back((uintptr_t)t.grad, (uintptr_t)t.grad + gs * all);
    written.emplace_back((uintptr_t)t.param, (uintptr_t)t.param + ps * all);
    if (step) written.emplace_back((uintptr_t)t.momentum, (uintptr_t)t.momentum + 4 * all);
    if (t.master) written.emplace_back((uintptr_t)t.master, (uintptr_t)t.master + 4 * all);
  }
  if (!mu_call(a->matrices, a->count).small && (!a->workspace || ((uintptr_t)a->workspace & 255)))
    return fail(STRATA_HIP_EINVAL, n + ": workspace must be given, 256-byte aligned");
  return check_ranges(n, written, read);
}

// Tiles of T x T a product of a group takes.
static int64_t mu_tiles(const MuGroup& g, int T, int mode) {
  const int64_t mt = (g.mp + T - 1) / T, nt = (g.np + T - 1) / T;
  return g.count * (mode == MU_UPDATE ? mt * nt : mt * (mt + 1) / 2);  // at most 2^22 (mu_sizes)
}
static int64_t mu_length(const MuGroup& g, int mode) { return (mode == MU_GRAM ? g.np : g.mp) / MU_K; }

// The tile of a launch, by an estimate of its cycles: rounds of the 256 CUs, each of the tiles' stages at what one costs with so
// many tiles on a CU, and what a tile costs besides; at least the longest tile alone.  Measured in cycles a stage, one
// tile alone on a CU and as many as fit: 64 x 64 240 and 480 (3), 128 x 128 530 and 850 (2), 256 x 256 1400; of two fp16
// 64 x 64 400 and 670 (2), 128 x 128 1150, in P X 1300 and 2800 (2); besides them 5000, 11000, 20000 (7000, 12000).  What it decides: 960 x 3840 alone, X X^T
// 17 us on 64 x 64, 33 on 128 x 128, 75 on 256 x 256; 72 matrices of 512 columns 53, 41, 47; 48 of 960 P X 570, 423, 362.
static int mu_tile_size(const std::vector<const MuGroup*>& groups, int mode, bool precise) {
  struct Cost {
    int tile, fit;
    double alone, more, fixed;  // a stage: alone + more for each other tile on the CU
  };
  static constexpr Cost plain[3] = {{64, 3, 240., 120., 5e3}, {128, 2, 530., 320., 11e3}, {256, 1, 1400., 0., 20e3}};
  static constexpr Cost square[2] = {{64, 2, 400., 270., 7e3}, {128, 1, 1150., 0., 12e3}}, update[2] = {{64, 2, 400., 270., 7e3}, {128, 2, 1300., 1500., 12e3}};
  const Cost* const two = mode == MU_UPDATE ? update : square;
  int best = 0;
  double least = 0.;
  for (int i = 0; i < (precise ? 2 : 3); ++i) {
    const Cost& c = precise ? two[i] : plain[i];
    double tiles = 0., stages = 0., longest = 0.;
    for (const MuGroup* g : groups) {
      const double n = (double)mu_tiles(*g, c.tile, mode), k = (double)mu_length(*g, mode);
      tiles += n;
      stages += n * k;
      longest = std::max(longest, k);
    }
    const double mean = stages / tiles, round = 256. * c.fit, full = std::floor(tiles / round), rest = std::ceil((tiles - full * round) / 256.);
    auto of = [&](double on, double k) { return k * (c.alone + c.more * (on - 1.)) + c.fixed; };
    const double t = std::max(full * of(c.fit, mean) + (rest > 0. ? of(rest, mean) : 0.), of(1., longest));
    if (!best || t < least) best = c.tile, least = t;
  }
  return best;
}

// One product of every group of one precision, the longest first: `fill` sets the operands of a shape.
template <int MODE, int PARTS, typename F>
static int mu_products_of(const MuPlan& q, MuGemm& b, hipStream_t st, F fill) {
  std::vector<const MuGroup*> order;
  for (const MuGroup& g : q.groups)
    if (g.precise == (PARTS == 2)) order.push_back(&g);
  if (order.empty()) return STRATA_HIP_OK;
  std::stable_sort(order.begin(), order.end(), [](const MuGroup* x, const MuGroup* y) { return mu_length(*x, MODE) > mu_length(*y, MODE); });
  const int T = mu_tile_size(order, MODE, PARTS == 2);
  b.count = 0;
  uint32_t tiles = 0;
  auto flush = [&]() -> int {
    if (!b.count) return STRATA_HIP_OK;
    if (T == 64) hipLaunchKernelGGL((muon_gemm_kernel<64, 2, 2, PARTS == 2 ? 4 : 6, PARTS, MODE>), dim3(tiles), dim3(256), 0, st, b);
    else if constexpr (PARTS == 2 && MODE == MU_UPDATE) hipLaunchKernelGGL((muon_gemm_kernel<128, 4, 2, 2, 2, MU_UPDATE>), dim3(tiles), dim3(512), 0, st, b);
    else if (T == 128) hipLaunchKernelGGL((muon_gemm_kernel<128, 2, 2, PARTS == 2 ? 5 : 4, PARTS, MODE>), dim3(tiles), dim3(256), 0, st, b);
    else if constexpr (PARTS == 1) hipLaunchKernelGGL((muon_gemm_kernel<256, 2, 4, 4, 1, MODE>), dim3(tiles), dim3(512), 0, st, b);
    b.count = 0;
    tiles = 0;
    return check_launch("muon products");
  };
  for (const MuGroup* g : order) {
    const int64_t n = mu_tiles(*g, T, MODE);
    if (b.count == MU_PER || tiles + n > (1 << 22))
      if (const int rc = flush()) return rc;
    b.first[b.count] = tiles;
    MuShape& s = b.s[b.count++];
    s.mp = (int)g->mp;
    s.np = (int)g->np;
    s.count = (int)g->count;
    s.tiles = (int)n;
    s.flags = PARTS == 2 ? MU_LO_IN | MU_LO_OUT : 0;
    fill(*g, s);
    tiles += (uint32_t)n;
  }
  return flush();
}

// P and P X of the groups of one height and precision.
template <int MP, int PARTS, typename F>
static int mu_slim_launch(const MuPlan& q, MuSlim& b, hipStream_t st, F fill) {
  b.count = 0;
  uint32_t tiles = 0;
  auto flush = [&]() -> int {
    if (!b.count) return STRATA_HIP_OK;
    hipLaunchKernelGGL((muon_slim_kernel<MP, PARTS>), dim3(tiles), dim3(512), 0, st, b);
    b.count = 0;
    tiles = 0;
    return check_launch("muon slim products");
  };
  for (const MuGroup& g : q.groups) {
    if (g.mp != MP || g.precise != (PARTS == 2)) continue;
    const int64_t n = g.count * (MP / 64) * ((g.np + 127) / 128);  // at most 2^22 (mu_sizes)
    if (b.count == MU_PER || tiles + n > (1 << 22))
      if (const int rc = flush()) return rc;
    b.first[b.count] = tiles;
    MuShape& s = b.s[b.count++];
    s.mp = (int)g.mp;
    s.np = (int)g.np;
    s.count = (int)g.count;
    s.tiles = (int)n;
    s.flags = PARTS == 2 ? MU_LO_IN | MU_LO_OUT : 0;
    fill(g, s);
    tiles += (uint32_t)n;
  }
  return flush();
}

template <int MODE, typename F>
static int mu_products(const MuPlan& q, MuGemm& b, hipStream_t st, F fill) {
  const int rc = mu_products_of<MODE, 1>(q, b, st, fill);
  return rc ? rc : mu_products_of<MODE, 2>(q, b, st, fill);
}

// What the kernels are told of a tensor, but for its place in the workspace.
static MuTensor mu_tensor(const strata_hip_muon_args* a, const strata_hip_muon_matrix& t, bool step) {
  MuTensor o = {};
  o.p = t.param;
  o.g = t.grad;
  o.m = t.momentum;
  o.master = t.master;
  o.rows = t.rows;
  o.cols = t.cols;
  const uintptr_t at = (uintptr_t)t.grad | (uintptr_t)t.momentum | (uintptr_t)t.param | (uintptr_t)t.master;
  o.flags = (t.param_dtype == STRATA_HIP_F32 ? MU_P32 : 0) | (t.grad_dtype == STRATA_HIP_F32 ? MU_G32 : 0) |
            (t.rows > t.cols ? MU_TALL : 0) | ((at & 15) || t.cols % 4 ? 0 : MU_ALIGNED) | (a->nesterov ? MU_NESTEROV : 0) |
            (step ? MU_STEP : 0) | (mu_precise(t) ? MU_LO : 0);
  const double adjust = a->adjust == STRATA_HIP_ADJUST_MATCH_RMS_ADAMW ? 0.2 * std::sqrt((double)std::max(t.rows, t.cols))
                                                                       : std::sqrt(std::max(1., (double)t.rows / (double)t.cols));
  o.rate = (float)(t.lr * adjust);
  o.decay = (float)(1. - t.lr * t.weight_decay);
  return o;
}

template <int MP, int NP, int PARTS>
static int mu_small_launch(const strata_hip_muon_args* a, int kind, bool step, hipStream_t st) {
  MuSmall b;
  b.count = 0;
  b.steps = a->steps;
  b.mu = (float)a->momentum;
  b.omu = (float)(1. - a->momentum);
  b.eps = a->eps;
  for (int i = 0; i < 3 * a->steps; ++i) b.co[i / 3][i % 3] = (float)a->coefficients[i];
  uint32_t wgs = 0;
  auto flush = [&]() -> int {
    if (!b.count) return STRATA_HIP_OK;
    hipLaunchKernelGGL((muon_small_kernel<MP, NP, PARTS>), dim3(wgs), dim3(MP == 64 ? 512 : 1024), 0, st, b);
    b.count = 0;
    wgs = 0;
    return check_launch("muon small");
  };
  for (int64_t i = 0; i < a->count; ++i) {
    const strata_hip_muon_matrix& t = a->matrices[i];
    if (!t.rows || !t.cols || !t.batch || mu_small(t) != kind || mu_precise(t) != (PARTS == 2)) continue;
    if (b.count == MU_SMALL_PER || wgs + t.batch > (1 << 21))  // 1024 threads each: a grid holds less than 2^32
      if (const int rc = flush()) return rc;
    b.t[b.count] = mu_tensor(a, t, step);
    b.t[b.count++].first = wgs;
    wgs += (uint32_t)t.batch;
  }
  return flush();
}

static int mu_launch(const std::string& name, const strata_hip_muon_args* a, bool step, hipStream_t st) {
  if (const int rc = mu_check(name, a, step)) return rc;
  const MuCall call = mu_call(a->matrices, a->count);
  if (call.small) {
    int kinds = 0;
    for (int64_t i = 0; i < a->count; ++i) {
      const strata_hip_muon_matrix& t = a->matrices[i];
      if (t.rows && t.cols && t.batch) kinds |= 1 << (2 * mu_small(t) + mu_precise(t));
    }
    int rc = STRATA_HIP_OK;
    if (kinds & 2) rc = mu_small_launch<64, 128, 2>(a, 0, step, st);
    if (!rc && kinds & 8) rc = mu_small_launch<64, 384, 2>(a, 1, step, st);
    if (!rc && kinds & 16) rc = mu_small_launch<128, 128, 1>(a, 2, step, st);
    if (!rc && kinds & 32) rc = mu_small_launch<128, 128, 2>(a, 2, step, st);
    return rc;
  }
  const MuPlan q = mu_plan(a->matrices, a->count);
  double* const sums = (double*)a->workspace;
  f16* const halves = (f16*)((char*)a->workspace + (q.sums * 8 + 255) / 256 * 256);
  int last = 0;  // which X a pass reads or writes

  // kind 0: momentum and sums, 1: X, 2: the update, 3: the sums of matrices that have many
  auto tensors = [&](int kind) -> int {
    MuBatch b;
    b.count = 0;
    b.mu = (float)a->momentum;
    b.omu = (float)(1. - a->momentum);
    b.eps = a->eps;
    uint32_t wgs = 0;
    auto flush = [&]() -> int {
      if (!b.count) return STRATA_HIP_OK;
      if (kind == 0) hipLaunchKernelGGL(muon_momentum_kernel, dim3(wgs), dim3(256), 0, st, b);
      else if (kind == 3) hipLaunchKernelGGL(muon_norm_kernel, dim3(wgs), dim3(1024), 0, st, b);
      else if (kind == 1) hipLaunchKernelGGL(muon_pack_kernel, dim3(wgs), dim3(256), 0, st, b);
      else hipLaunchKernelGGL(muon_apply_kernel, dim3(wgs), dim3(256), 0, st, b);
      b.count = 0;
      wgs = 0;
      return check_launch("muon elements");
    };
    for (int64_t i = 0; i < a->count; ++i) {
      if (q.of[(size_t)i] < 0) continue;
      const strata_hip_muon_matrix& t = a->matrices[i];
      const MuGroup& g = q.groups[(size_t)q.of[(size_t)i]];
      if (kind == 3 && mu_chunks(t) <= MU_SUMS) continue;
      const int64_t per = kind == 0 ? mu_chunks(t) : kind == 3 ? 1 : (g.mp / 64) * (g.np / 64), n = per * t.batch;
      if (b.count == MU_PER || wgs + n > (1 << 23))
        if (const int rc = flush()) return rc;
      MuTensor& o = b.t[b.count++];
      o = mu_tensor(a, t, step);
      o.x = halves + g.x[last] + q.at[(size_t)i] * g.mp * g.np;
      o.xlo = o.x + g.count * g.mp * g.np;
      o.part = sums + q.parts[(size_t)i];
      o.first = wgs;
      o.per = (uint32_t)per;
      wgs += (uint32_t)n;
    }
    return flush();
  };

  if (const int rc = tensors(0)) return rc;
  if (const int rc = tensors(3)) return rc;
  if (const int rc = tensors(1)) return rc;
  MuGemm b;
  for (int k = 0; k < a->steps; ++k) {
    const double* c = a->coefficients + 3 * k;
    b.alpha = MU_A / (MU_X * MU_X);
    b.beta = 0.f;
    if (const int rc = mu_products<MU_GRAM>(q, b, st, [&](const MuGroup& g, MuShape& s) {
          s.x = s.w = s.d = halves + g.x[last];
          s.out = halves + g.a;
        }))
      return rc;
    // X's second fp16 goes into the first steps
    const int lo = (k < MU_LO_STEPS ? MU_LO_IN : 0) | (k + 1 < MU_LO_STEPS ? MU_LO_OUT : 0);
    auto update = [&](const MuGroup& g, MuShape& s) {
      s.flags |= lo;
      s.w = s.d = halves + g.x[last];
      s.out = halves + g.x[last ^ 1];
    };
    if (call.slim) {
      MuSlim m;
      m.a = (float)c[0];
      m.b = (float)c[1];
      m.c = (float)c[2];
      auto both = [&](const MuGroup& g, MuShape& s) {
        update(g, s);
        s.x = halves + g.a;
      };
      int rc = mu_slim_launch<64, 2>(q, m, st, both);
      if (!rc) rc = mu_slim_launch<128, 1>(q, m, st, both);
      if (!rc) rc = mu_slim_launch<128, 2>(q, m, st, both);
      if (rc) return rc;
      last ^= 1;
      continue;
    }
    b.alpha = (float)(c[2] / MU_A);
    b.beta = (float)c[1];
    if (const int rc = mu_products<MU_POLY>(q, b, st, [&](const MuGroup& g, MuShape& s) {
          s.x = s.w = s.d = halves + g.a;
          s.out = halves + g.p;
        }))
      return rc;
    b.alpha = 1.f / MU_A;
    b.beta = (float)c[0];
    if (const int rc = mu_products<MU_UPDATE>(q, b, st, [&](const MuGroup& g, MuShape& s) {
          update(g, s);
          s.x = halves + g.p;
        }))
      return rc;
    last ^= 1;
  }
  return tensors(2);
}

static int mu_entry_point(const char* name, const strata_hip_muon_args* a, bool step, void* stream) {
  try {
    return mu_launch(name, a, step, (hipStream_t)stream);
  } catch (const std::exception&) {  // no memory for the lists, or more than a list can hold
    return fail(STRATA_HIP_EUNSUPPORTED, std::string(name) + ": out of host memory");
  }
}

}  // namespace strata

extern "C" int64_t strata_hip_muon_workspace(const strata_hip_muon_matrix* matrices, int64_t count) {
  if (!matrices || count <= 0) return 0;
  try {
    if (strata::mu_sizes("muon_workspace", matrices, count)) return -1;
    return strata::mu_plan(matrices, count).bytes;
  } catch (const std::exception&) {
    return -1;
  }
}

extern "C" int strata_hip_muon_step(const strata_hip_muon_args* a, void* stream) {
  return strata::mu_entry_point("muon_step", a, true, stream);
}

extern "C" int strata_hip_orthogonalize(const strata_hip_muon_args* a, void* stream) {
  return strata::mu_entry_point("orthogonalize", a, false, stream);
}
