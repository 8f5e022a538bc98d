// Newton-Schulz orthogonalisation of many matrices at once and the Muon step built on it, for gfx950.
//
//   m <- mu m + (1 - mu) g     u = mu m + (1 - mu) g (Nesterov) or m     X = u / max(|u|, eps), |u| the root of the sum of squares
//   steps times:  A = X X^T    P = b A + c A A    X <- a X + P X         (a matrix taller than wide: its transpose)
//   p <- p (1 - lr decay) - lr adjust X
//
// A matrix m x n (m <= n) lives in a workspace as [m', n'], both rounded up to 64 and zero beyond m and n, which every
// product leaves zero: no product has an edge to watch.  Matrices of one shape stand one behind the other, and a launch takes
// the tiles of all shapes: three launches a step, whatever the number of matrices.  A and P are symmetric: only tiles on
// and above the diagonal are computed and also written transposed, so that a step costs m m n + m m m + 2 m m n
// operations instead of 4 m m n + 2 m m m.  P X reads X along its rows, transposed out of LDS (ds_read_b64_tr_b16).
//
// What is rounded: the products' operands are fp16, scaled by powers of two (X 2^12, A and P 2^10: there is room up to
// 16 and 64, the usual coefficients keep them under 2 and 8; most values lie at 1 / sqrt(n), well above the 2^-14 where
// fp16 loses bits), sums are fp32.
// Singular values near 0 grow 3.4-fold a step with all the noise among them, so it is the early roundings
// of X that show, and those of its term a X alone (P is small then): X is held as the sum of two fp16, of which the
// products take the first, in all steps but the last two.  Simulated, the result is off by 0.3e-3 to 1.5e-3 for
// noise, decaying and low-rank spectra (3.8e-3 without the second fp16, 10 to 30e-3 with iterates in bf16), below the 1.7e-3
// of a bf16 result's own rounding.  `precise`: X, A and P are sums of two fp16 throughout and a product is three, high
// high, high low and low high: 0.2e-6 to 0.7e-6.
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
constexpr int MU_CHUNK = 8192;   // elements a workgroup of the momentum's pass
constexpr int MU_PER = 40;       // tensors a launch, and shapes: kernel arguments are 4 KiB
constexpr float MU_X = 0x1p12f, MU_A = 0x1p10f;  // scales of X, and of A and P
enum { MU_P32 = 1, MU_G32 = 2, MU_TALL = 4, MU_ALIGNED = 8, MU_NESTEROV = 16, MU_STEP = 32 };

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

// A tile of 64 x 64 of one matrix: `x` tile (ti, tj) of the workspace, whose source tile is the same or, of a tall
// matrix, the transposed one.
struct MuTile {
  int64_t base;   // first element of the matrix in its tensor
  int64_t at;     // first element of the tile in the workspace
  int64_t row0, col0;
  int64_t np;
};
__device__ __forceinline__ MuTile mu_tile(const MuTensor& t, uint32_t local) {
  const bool tall = t.flags & MU_TALL;
  const int64_t m = tall ? t.cols : t.rows, n = tall ? t.rows : t.cols;
  const int64_t mt = (m + 63) / 64, nt = (n + 63) / 64;
  const uint32_t mat = local / t.per, k = local % t.per;
  const int64_t ti = k / nt, tj = k % nt;
  MuTile r;
  r.base = (int64_t)mat * t.rows * t.cols;
  r.np = nt * 64;
  r.at = ((int64_t)mat * mt * 64 + ti * 64) * r.np + tj * 64;
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
  for (uint32_t k = tid; k < chunks; k += 256) s += t.part[(int64_t)mat * chunks + k];
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  const double norm = sqrt(((red[0] + red[1]) + red[2]) + red[3]);
  const double scale = norm == 0. ? 0. : MU_X / (norm < b.eps ? b.eps : norm);  // 64-bit: of tiny updates it leaves fp32
  const int r = tid >> 4, c = (tid & 15) * 4;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t row = x.row0 + 16 * k + r, col = x.col0 + c, i = x.base + row * t.cols + col;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    auto one = [&](float g, float m) { return (float)((double)(t.m ? nesterov ? fmaf(b.mu, m, b.omu * g) : m : g) * scale); };
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
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[16 * k + r][c + e] = v[e];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = tall ? tile[c + e][16 * k + r] : tile[16 * k + r][c + e];
      h[e] = (f16)v;
      l[e] = (f16)(v - (float)h[e]);
    }
    const int64_t at = x.at + (16 * k + r) * x.np + c;
    *(f16x4*)(t.x + at) = h;
    *(f16x4*)(t.xlo + at) = l;
  }
}

// ---- the weights' update from X, or X itself ----
__global__ __launch_bounds__(256) void muon_apply_kernel(MuBatch b) {
  __shared__ float tile[64][65];
  const uint32_t wg = blockIdx.x;
  const MuTensor& t = b.t[mu_entry(b.count, wg, [&](int i) { return b.t[i].first; })];
  const MuTile x = mu_tile(t, wg - t.first);
  const int tid = threadIdx.x, r = tid >> 4, c = (tid & 15) * 4;
  const bool p32 = t.flags & MU_P32, tall = t.flags & MU_TALL;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t at = x.at + (16 * k + r) * x.np + c;
    const f16x4 h = *(const f16x4*)(t.x + at), l = *(const f16x4*)(t.xlo + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = ((float)h[e] + (float)l[e]) * (1.f / MU_X);
      if (tall) tile[c + e][16 * k + r] = v;
      else tile[16 * k + r][c + e] = v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t row = x.row0 + 16 * k + r, col = x.col0 + c, i = x.base + row * t.cols + col;
    if (row >= t.rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (col + e >= t.cols) continue;
      float v = tile[16 * k + r][c + e];
      if (t.flags & MU_STEP) {  // uniform
        const float p = t.master ? t.master[i + e] : mu_load(t.p, i + e, p32);
        v = fmaf(-t.rate, v, p * t.decay);
      }
      if (t.master) t.master[i + e] = v;
      if (p32) ((float*)t.p)[i + e] = v;
      else ((bf16*)t.p)[i + e] = (bf16)v;
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
  uint32_t first;
  int flags;
};
struct MuGemm {
  MuShape s[MU_PER];
  int count;
  float alpha, beta;  // of the product and of d
};
static_assert(sizeof(MuGemm) <= 4096, "kernel arguments");
enum { MU_GRAM = 0, MU_POLY = 1, MU_UPDATE = 2 };
enum { MU_THREE = 1, MU_LO_IN = 2, MU_LO_OUT = 4 };  // high high, high low, low high; d has, out gets its second fp16

// 16-byte chunks of an LDS row are stored at their index xor these: rows of 64 columns read 16 bytes a lane by 32
// rows at one chunk, rows of BN columns read transposed by 8 rows at 4 chunks.
__device__ __forceinline__ int mu_swz(int row) { return (row & 7) ^ ((row >> 3) & 1); }
template <int BN>
__device__ __forceinline__ int mu_wswz(int row) {
  return BN == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
}

template <int BM, int BN, int WGM, int WGN, int NST, int MODE>
__global__ __launch_bounds__(64 * WGM * WGN, 1) void muon_gemm_kernel(MuGemm p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr bool WT = MODE == MU_UPDATE, SYM = !WT;
  static_assert(!SYM || BM == BN, "square tiles");
  constexpr int BK = 64, NW = WGM * WGN;
  constexpr int WTM = BM / WGM, WTN = BN / WGN, FM = WTM / 32, FN = WTN / 32;
  constexpr int ROWB = BK * 2, CH = ROWB / 16, RPC = 1024 / ROWB;
  constexpr int XB = BM * ROWB, STAGE = XB + BN * ROWB;
  constexpr int LPX = XB / 1024 / NW, LPW = BN * ROWB / 1024 / NW;  // 1-KiB copies a wave and stage
  constexpr int WLPR = BN / 8, WRPC = 64 / WLPR;
  constexpr int SLAB = 32 * WTN * 4;
  static_assert(WTM % 32 == 0 && WTN % 32 == 0 && LPX > 0 && LPW > 0 && NW * SLAB <= NST * STAGE, "wave tile, stage and slab layout");
  __shared__ __attribute__((aligned(1024))) char lds[NST * STAGE];

  const int tid = (int)__builtin_amdgcn_workitem_id_x();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wm = wave / WGN, wn = wave % WGN, l32 = lane & 31, hi = lane >> 5;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  // Each shape's tiles are dealt to the XCDs in blocks: one matrix's on one XCD, every XCD with its share of every shape.
  const uint32_t wg = (uint32_t)__builtin_amdgcn_workgroup_id_x();
  const MuShape& s = p.s[mu_entry(p.count, wg, [&](int i) { return p.s[i].first; })];
  const int id = xcd_tile_order(s.tiles, (int)(wg - s.first));
  const int mp = s.mp, np = s.np;
  const int mt = (mp + BM - 1) / BM, nt = (np + BN - 1) / BN, per = SYM ? mt * (mt + 1) / 2 : mt * nt;
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
  const int row0 = tm * BM, n0 = tn * BN;
  // the x operand is [mp, ldx], the w operand [mp, ldw] (its rows are columns of the product, in UPDATE the contraction)
  const int ldx = MODE == MU_GRAM ? np : mp, ldw = MODE == MU_POLY ? mp : np, ldo = MODE == MU_UPDATE ? np : mp;
  const int64_t xs = (int64_t)mp * ldx, ws = (int64_t)mp * ldw, os = (int64_t)mp * ldo;
  const int K = MODE == MU_GRAM ? np : mp, cols = SYM ? mp : np;
  const f16* const xb = s.x + mat * xs + (int64_t)row0 * ldx;
  const f16* const wb = s.w + mat * ws + (WT ? (int64_t)n0 : (int64_t)n0 * ldw);
  const int nk1 = K / BK, nk = s.flags & MU_THREE ? 3 * nk1 : nk1;

  uint32_t xo[LPX], wo[LPW];
#pragma unroll
  for (int j = 0; j < LPX; ++j) {
    const int row = RPC * (j * NW + wave) + lane / CH;
    xo[j] = row0 + row < mp ? (uint32_t)row * (uint32_t)ldx * 2u + (((lane % CH) ^ mu_swz(row)) * 16) : OOB;
  }
#pragma unroll
  for (int j = 0; j < LPW; ++j) {
    if (WT) {
      const int row = WRPC * (j * NW + wave) + lane / WLPR, chunk = (lane % WLPR) ^ mu_wswz<BN>(row);
      wo[j] = n0 + 8 * chunk < np ? (uint32_t)row * (uint32_t)ldw * 2u + chunk * 16 : OOB;
    } else {
      const int row = RPC * (j * NW + wave) + lane / CH;
      wo[j] = n0 + row < mp ? (uint32_t)row * (uint32_t)ldw * 2u + (((lane % CH) ^ mu_swz(row)) * 16) : OOB;
    }
  }
  auto issue = [&](int kt, int slot) {
    const int seg = kt / nk1, kk = kt - seg * nk1;
    const u32x4 rx = make_rsrc(xb + (seg == 2 ? s.count * xs : 0) + (int64_t)kk * BK, OOB);
    const u32x4 rw = make_rsrc(wb + (seg == 1 ? s.count * ws : 0) + (WT ? (int64_t)kk * BK * ldw : (int64_t)kk * BK), OOB);
    const uint32_t dst = lds_base + slot * STAGE + wave * 1024;
#pragma unroll
    for (int j = 0; j < LPX; ++j) dma_row16(rx, dst + j * NW * 1024, xo[j]);
#pragma unroll
    for (int j = 0; j < LPW; ++j) dma_row16(rw, dst + XB + j * NW * 1024, wo[j]);
  };

  // LDS offsets of the fragments; K sub-steps 2, 3 of K-contiguous rows are at offset ^ 64
  uint32_t aoff[FN][WT ? 1 : 2], boff[FM][2];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    if (WT) {
      const int r4 = (lane & 15) >> 2, c = (wn * WTN + 32 * i) / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      aoff[i][0] = XB + (8 * hi + r4) * (BN * 2) + ((c ^ mu_wswz<BN>(r4)) << 4) + 8 * (lane & 1);
    } else {
      const int row = wn * WTN + 32 * i + l32;
      for (int kk = 0; kk < 2; ++kk) aoff[i][WT ? 0 : kk] = XB + row * ROWB + ((2 * kk + hi) ^ mu_swz(row)) * 16;
    }
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int row = wm * WTM + 32 * j + l32;
    for (int kk = 0; kk < 2; ++kk) boff[j][kk] = row * ROWB + ((2 * kk + hi) ^ mu_swz(row)) * 16;
  }
  auto load_frags = [&](const char* st, int kk, f16x8 (&a)[FN], f16x8 (&b)[FM]) {
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if constexpr (WT) {
        const char* q = st + aoff[i][0] + kk * 16 * (BN * 2);
        typedef __fp16 h16x4 __attribute__((ext_vector_type(4)));
        const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(LDS_PTR(h16x4, q)));
        const f16x4 up = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(LDS_PTR(h16x4, q + 4 * (BN * 2))));
        a[i] = __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        a[i] = *(const f16x8*)(st + (aoff[i][kk & 1] ^ ((kk >> 1) * 64)));
      }
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) b[j] = *(const f16x8*)(st + (boff[j][kk & 1] ^ ((kk >> 1) * 64)));
  };

  f32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
#pragma unroll
  for (int q = 0; q < NST - 1; ++q)
    if (q < nk) issue(q, q);
  int rd = 0;
  for (int kt = 0; kt < nk; ++kt) {
    if (NST > 2 && kt + NST - 2 < nk) wait_vmcnt((NST - 2) * (LPX + LPW));
    else wait_vmcnt(0);
    lds_barrier();  // landed for every wave, and the slot read last step is free
    if (kt + NST - 1 < nk) issue(kt + NST - 1, rd == 0 ? NST - 1 : rd - 1);
    const char* st = lds + rd * STAGE;
    rd = rd + 1 == NST ? 0 : rd + 1;
    f16x8 af[2][FN], bfr[2][FM];
    load_frags(st, 0, af[0], bfr[0]);
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      const int cb = kk & 1;
      if (kk + 1 < BK / 16) load_frags(st, kk + 1, af[cb ^ 1], bfr[cb ^ 1]);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[cb][i], bfr[cb][j], acc[i][j], 0, 0, 0);
    }
  }

  // ---- epilogue: 32 rows of the wave's tile at a time through its slab of the ring in fp32, back as eight columns a lane
  lds_barrier();  // every wave is done reading the last stage
  constexpr int NCH = WTN / 4, LPR = WTN / 8, RPI = 64 / LPR, NIT = 32 / RPI;
  char* slab = lds + wave * SLAB;
  const int lrow = lane / LPR, lc = lane % LPR, gn = n0 + wn * WTN + 8 * lc;
  const bool mirror = SYM && tm != tn;
  f16* const out = s.out + mat * os;
  const int64_t olo = s.count * os;  // from a value's first fp16 to its second
  const f16* const d = s.d + mat * os;
  auto place = [&](int row, int chunk) { return slab + row * (WTN * 4) + ((chunk ^ (row & (NCH - 1))) << 4); };
  auto split = [&](const float (&v)[8], f16x8& h, f16x8& l) {
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      h[x] = (f16)v[x];
      l[x] = (f16)(v[x] - (float)h[x]);
    }
  };
#pragma unroll
  for (int j = 0; j < FM; ++j) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(f32x4*)place(l32, 8 * i + 2 * q + hi) = (f32x4){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int sl = RPI * it + lrow, r = row0 + wm * WTM + 32 * j + sl;
      const bool in = r < mp && gn < cols;
      const f32x4 z0 = *(const f32x4*)place(sl, 2 * lc), z1 = *(const f32x4*)place(sl, 2 * lc + 1);
      float v[8] = {z0[0], z0[1], z0[2], z0[3], z1[0], z1[1], z1[2], z1[3]};
      const int64_t at = (int64_t)r * ldo + gn;
      f16x8 h = {}, l = {};
      if (MODE != MU_GRAM && in) {
        h = *(const f16x8*)(d + at);
        if (s.flags & MU_LO_IN) l = *(const f16x8*)(d + olo + at);
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x] = MODE == MU_GRAM ? v[x] * p.alpha : fmaf(v[x], p.alpha, p.beta * ((float)h[x] + (float)l[x]));
      split(v, h, l);
      if (in) {
        *(f16x8*)(out + at) = h;
        if (s.flags & MU_LO_OUT) *(f16x8*)(out + olo + at) = l;
      }
      if (mirror) {
        *(f32x4*)place(sl, 2 * lc) = (f32x4){v[0], v[1], v[2], v[3]};
        *(f32x4*)place(sl, 2 * lc + 1) = (f32x4){v[4], v[5], v[6], v[7]};
      }
    }
    if (mirror) {  // four lanes a column, eight rows each
#pragma unroll
      for (int it = 0; it < WTN / 16; ++it) {
        const int c = 16 * it + (lane >> 2), r8 = (lane & 3) * 8;
        float v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = *(const float*)(place(r8 + x, c >> 2) + 4 * (c & 3));
        f16x8 h, l;
        split(v, h, l);
        const int r = row0 + wm * WTM + 32 * j + r8, g = n0 + wn * WTN + c;
        if (r < mp && g < mp) {
          *(f16x8*)(out + (int64_t)g * ldo + r) = h;
          if (s.flags & MU_LO_OUT) *(f16x8*)(out + olo + (int64_t)g * ldo + r) = l;
        }
      }
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
  std::vector<int> of;             // a tensor's group
  std::vector<int64_t> at, parts;  // its first matrix there, and its first sum of squares
  int64_t sums = 0, halves = 0, bytes = 0;
};

static int64_t mu_chunks(const strata_hip_muon_matrix& t) { return (t.rows * t.cols + MU_CHUNK - 1) / MU_CHUNK; }
static int64_t mu_up(int64_t n) { return (n + MU_PAD - 1) / MU_PAD * MU_PAD; }

// The sizes that the kernels' indexes and grids hold: at most 2^23 tiles of 64 x 64 a tensor.
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
  std::map<std::tuple<int64_t, int64_t, bool>, int> seen;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t m = std::min(ts[i].rows, ts[i].cols), n = std::max(ts[i].rows, ts[i].cols);
    const bool precise = ts[i].precise != 0;
    q.at.push_back(0);
    q.parts.push_back(q.sums);
    if (m <= 0 || ts[i].batch <= 0) {
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
    g.p = take((g.precise ? 2 : 1) * g.count * g.mp * g.mp);
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
  if (!written.empty() && (!a->workspace || ((uintptr_t)a->workspace & 255)))
    return fail(STRATA_HIP_EINVAL, n + ": workspace must be given, 256-byte aligned");
  return check_ranges(n, written, read);
}

// One product of every group, the longest first: `fill` sets the operands of a shape.
template <int MODE, typename F>
static int mu_products(const MuPlan& q, MuGemm& b, hipStream_t st, F fill) {
  constexpr int T = 128;
  std::vector<const MuGroup*> order;
  for (const MuGroup& g : q.groups) order.push_back(&g);
  auto length = [](const MuGroup* g) { return (MODE == MU_GRAM ? g->np : g->mp) * (g->precise ? 3 : 1); };
  std::stable_sort(order.begin(), order.end(), [&](const MuGroup* x, const MuGroup* y) { return length(x) > length(y); });
  b.count = 0;
  uint32_t tiles = 0;
  auto flush = [&]() -> int {
    if (!b.count) return STRATA_HIP_OK;
    hipLaunchKernelGGL((muon_gemm_kernel<T, T, 4, 2, 2, MODE>), dim3(tiles), dim3(512), 0, st, b);
    b.count = 0;
    tiles = 0;
    return check_launch("muon products");
  };
  for (const MuGroup* g : order) {
    const int64_t mt = (g->mp + T - 1) / T, nt = (g->np + T - 1) / T;
    const int64_t n = g->count * (MODE == MU_UPDATE ? mt * nt : mt * (mt + 1) / 2);  // at most 2^22 (mu_sizes)
    if (b.count == MU_PER || tiles + n > (1 << 22))
      if (const int rc = flush()) return rc;
    MuShape& s = b.s[b.count++];
    s.mp = (int)g->mp;
    s.np = (int)g->np;
    s.count = (int)g->count;
    s.tiles = (int)n;
    s.first = tiles;
    s.flags = g->precise ? MU_THREE | MU_LO_IN | MU_LO_OUT : 0;
    fill(*g, s);
    tiles += (uint32_t)n;
  }
  return flush();
}

static int mu_launch(const std::string& name, const strata_hip_muon_args* a, bool step, hipStream_t st) {
  if (const int rc = mu_check(name, a, step)) return rc;
  const MuPlan q = mu_plan(a->matrices, a->count);
  if (q.groups.empty()) return STRATA_HIP_OK;
  double* const sums = (double*)a->workspace;
  f16* const halves = (f16*)((char*)a->workspace + (q.sums * 8 + 255) / 256 * 256);
  int last = 0;  // which X a pass reads or writes

  // kind 0: momentum and sums, 1: X, 2: the update
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
      const int64_t per = kind == 0 ? mu_chunks(t) : (g.mp / 64) * (g.np / 64), n = per * t.batch;
      if (b.count == MU_PER || wgs + n > (1 << 23))
        if (const int rc = flush()) return rc;
      MuTensor& o = b.t[b.count++];
      o.p = t.param;
      o.g = t.grad;
      o.m = t.momentum;
      o.master = t.master;
      o.x = halves + g.x[last] + q.at[(size_t)i] * g.mp * g.np;
      o.xlo = o.x + g.count * g.mp * g.np;
      o.part = sums + q.parts[(size_t)i];
      o.rows = t.rows;
      o.cols = t.cols;
      o.first = wgs;
      o.per = (uint32_t)per;
      const uintptr_t at = (uintptr_t)t.grad | (uintptr_t)t.momentum | (uintptr_t)t.param | (uintptr_t)t.master;
      o.flags = (t.param_dtype == STRATA_HIP_F32 ? MU_P32 : 0) | (t.grad_dtype == STRATA_HIP_F32 ? MU_G32 : 0) |
                (t.rows > t.cols ? MU_TALL : 0) | ((at & 15) || t.cols % 4 ? 0 : MU_ALIGNED) | (a->nesterov ? MU_NESTEROV : 0) |
                (step ? MU_STEP : 0);
      const double adjust = a->adjust == STRATA_HIP_ADJUST_MATCH_RMS_ADAMW ? 0.2 * std::sqrt((double)std::max(t.rows, t.cols))
                                                                           : std::sqrt(std::max(1., (double)t.rows / (double)t.cols));
      o.rate = (float)(t.lr * adjust);
      o.decay = (float)(1. - t.lr * t.weight_decay);
      wgs += (uint32_t)n;
    }
    return flush();
  };

  if (const int rc = tensors(0)) return rc;
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
    b.alpha = (float)(c[2] / MU_A);
    b.beta = (float)c[1];
    if (const int rc = mu_products<MU_POLY>(q, b, st, [&](const MuGroup& g, MuShape& s) {
          s.x = s.w = s.d = halves + g.a;
          s.out = halves + g.p;
        }))
      return rc;
    b.alpha = 1.f / MU_A;
    b.beta = (float)c[0];
    // X's second fp16: into all steps but the last two, and the last one's result, which the weights take
    const int lo = (k < a->steps - 2 ? MU_LO_IN : 0) | (k + 1 < a->steps - 2 || k + 1 == a->steps ? MU_LO_OUT : 0);
    if (const int rc = mu_products<MU_UPDATE>(q, b, st, [&](const MuGroup& g, MuShape& s) {
          s.flags |= lo;
          s.x = halves + g.p;
          s.w = s.d = halves + g.x[last];
          s.out = halves + g.x[last ^ 1];
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
