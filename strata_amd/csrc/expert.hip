// The chosen experts' MLPs for gfx950: grouped matrix products over rows sorted by expert.
//
//   out[t] = residual[t] + sum over slots s of w[t, s] (gelu(x[t] W1_e^T + b1_e) W2_e^T + b2_e),  e = index[t, s]
//
// Row r of the products is the pair (t, s) = row_slot[r] of the plan; the first product
// gathers its rows of x as it copies them into LDS, so no sorted copy of x exists.  Forward:
//   h = gelu(x[t] W1_e^T + b1_e)       bf16 (the second product's operand), with gelu' for a backward
//   y = h W2_e^T + b2_e                fp32: out is rounded once
//   out[t] = residual[t] + sum_s w y   in slot order
// Backward, g = dout:
//   dw[t, s] = <g[t], y_r>             gs_r = w g[t], bf16 (an operand of dW2)
//   gz_r = w (g[t] W2_e) gelu'         bf16 (an operand of the next three)
//   dW2_e = sum_r gs_r^T h_r  db2_e = sum_r gs_r  dW1_e = sum_r gz_r^T x[t]  db1_e = sum_r gz_r
//   dx[t] = sum_s (gz W1_e)_r          rows in bf16, summed in fp32 in slot order
// Each intermediate is rounded once, where a matrix instruction needs bf16.  Every sum has
// an order fixed by the sizes and the plan: results repeat bit for bit.
#include <algorithm>

#include "common.h"

namespace strata {

__device__ __forceinline__ void gelu_both(float x, float& y, float& d) {
  // x s and its derivative s + x s (1 - s) 2u' with s = sigmoid(2u), u = sqrt(2/pi) (x + 0.044715 x^3)
  constexpr float c = 0.7978845608028654f, k1 = 2.f * 1.4426950408889634f * c;
  const float t = x * fmaf(k1 * 0.044715f, x * x, k1);
  const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-t));
  y = x * s;
  d = fmaf(y * (1.f - s), 2.f * c * fmaf(3.f * 0.044715f, x * x, 1.f), s);
}

struct ExpertGemm {
  const bf16* x;
  const int32_t* rows;   // gather: row r of the product is row rows[r] / top_k of x; or null
  const bf16* w;         // [E, N, K]
  const bf16* bias;      // [E, N] or null
  const bf16* mul;       // HIDDEN_GRAD: gelu', [P, N]
  const bf16* scale;     // HIDDEN_GRAD: the weight of each pair, by rows[r]
  const int32_t* slots;  // HIDDEN_GRAD: row_slot
  void* out;             // [P, N] bf16, OUT: fp32
  bf16* out2;            // HIDDEN: gelu' or null
  const int32_t* offsets;
  const int32_t* tiles;
  int64_t ldx;
  int top_k, N, K, nt;
};

enum { EX_HIDDEN = 0, EX_OUT = 1, EX_HIDDEN_GRAD = 2, EX_INPUT_GRAD = 3 };

template <int CH>
__device__ __forceinline__ int ex_swz(int chunk, int row) {
  return chunk ^ ((row & 7) ^ ((row >> 3) & 1));
}

// One BM x BN tile of one expert's product a workgroup: x and w tiles stream into an
// LDS ring of NST stages of 64 columns, NST - 1 stages ahead of the v_mfma_f32_32x32x16_bf16.
// The weights are the MFMA's A operand: a lane owns four consecutive columns of one row.
template <int BM, int BN, int WGM, int WGN, int NST, int MODE>
__global__ __launch_bounds__(64 * WGM * WGN) void expert_gemm_kernel(ExpertGemm p) {
  constexpr int BK = 64, NW = WGM * WGN;
  constexpr int WTM = BM / WGM, WTN = BN / WGN, FM = WTM / 32, FN = WTN / 32;
  constexpr int ROWB = BK * 2, CH = ROWB / 16, RPC = 1024 / ROWB;
  constexpr int XB = BM * ROWB, XCH = XB / 1024, STAGE = XB + BN * ROWB;
  constexpr int LPW = STAGE / 1024 / NW;
  constexpr int SLAB = WTM * WTN * 2;
  static_assert(WTM % 32 == 0 && WTN % 32 == 0 && XCH % NW == 0 && (STAGE / 1024) % NW == 0, "wave tile / stage layout");
  static_assert(NW * SLAB <= NST * STAGE, "the epilogue slabs fit the ring");
  __shared__ __attribute__((aligned(1024))) char lds[NST * STAGE];

  const int tid = (int)__builtin_amdgcn_workitem_id_x();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wm = wave / WGN, wn = wave % WGN, l32 = lane & 31, hi = lane >> 5;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  // The grid is sized for the most tiles that the pairs can make; the plan says how many there are.
  const int mt = p.tiles[0], total = mt * p.nt, id = (int)__builtin_amdgcn_workgroup_id_x();
  if (id >= total) return;
  int tm, n0;
  {
    const int wg = xcd_tile_order(total, id);
    constexpr int GRP = 8;
    const int gi = wg / (GRP * p.nt), li = wg % (GRP * p.nt), gmn = min(GRP, mt - gi * GRP);
    tm = gi * GRP + li % gmn;
    n0 = (li / gmn) * BN;
  }
  const int e = p.tiles[1 + 2 * tm], row0 = p.tiles[2 + 2 * tm];
  const int rows = min(p.offsets[e + 1] - row0, BM);  // rows of this tile
  const bf16* we = p.w + (int64_t)e * p.N * p.K;

  uint32_t voff[LPW];
#pragma unroll
  for (int j = 0; j < LPW; ++j) {
    const bool isw = j * NW >= XCH;
    const int c = j * NW + wave - (isw ? XCH : 0), row = RPC * c + lane / CH;
    const uint32_t chunk = ex_swz<CH>(lane % CH, row) * 16;
    if (isw) {
      voff[j] = n0 + row < p.N ? (uint32_t)((uint32_t)row * p.K * 2) + chunk : OOB;
    } else {
      int64_t at = row;
      if (p.rows && row < rows) at = p.rows[row0 + row] / p.top_k;
      voff[j] = row < rows ? (uint32_t)(at * p.ldx * 2) + chunk : OOB;
    }
  }
  const int nk = (p.K + BK - 1) / BK, ktail = p.K % BK;
  const char* xk = (const char*)(p.rows ? p.x : p.x + (int64_t)row0 * p.ldx);
  const char* wk = (const char*)(we + (int64_t)n0 * p.K);
  auto issue = [&](int kt, int slot) {
    const u32x4 rx = make_rsrc(xk + (int64_t)kt * BK * 2, OOB), rw = make_rsrc(wk + (int64_t)kt * BK * 2, OOB);
    const uint32_t dst = lds_base + slot * STAGE + wave * 1024;
    const bool last = ktail && kt == nk - 1;  // uniform: chunks at or past K read as zero
#pragma unroll
    for (int j = 0; j < LPW; ++j) {
      const bool isw = j * NW >= XCH;
      uint32_t vo = voff[j];
      if (last) {
        const int row = RPC * (j * NW + wave - (isw ? XCH : 0)) + lane / CH;
        if (ex_swz<CH>(lane % CH, row) * 8 >= ktail) vo = OOB;
      }
      dma_row16(isw ? rw : rx, dst + j * NW * 1024, vo);
    }
  };

  // The bias as the accumulators' first C operand (columns 8q + 4hi + e of each 32).
  const int gn0 = n0 + wn * WTN;
  f32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      u32x2 bb = {0u, 0u};
      if (MODE <= EX_OUT && p.bias) bb = *(const u32x2*)(p.bias + (int64_t)e * p.N + min(gn0 + 32 * i + 8 * q + 4 * hi, p.N - 4));
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        acc[i][j][4 * q + 0] = bf16_lo(bb[0]);
        acc[i][j][4 * q + 1] = bf16_hi(bb[0]);
        acc[i][j][4 * q + 2] = bf16_lo(bb[1]);
        acc[i][j][4 * q + 3] = bf16_hi(bb[1]);
      }
    }

  uint32_t aoff[FN][2], boff[FM][2];  // sub-steps 2, 3 flip bit 2 of the chunk: offset ^ 64
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    const int row = wn * WTN + 32 * i + l32;
    for (int kk = 0; kk < 2; ++kk) aoff[i][kk] = XB + row * ROWB + ex_swz<CH>(2 * kk + hi, row) * 16;
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int row = wm * WTM + 32 * j + l32;
    for (int kk = 0; kk < 2; ++kk) boff[j][kk] = row * ROWB + ex_swz<CH>(2 * kk + hi, row) * 16;
  }

#pragma unroll
  for (int s = 0; s < NST - 1; ++s)
    if (s < nk) issue(s, s);
  int rd = 0;
  for (int kt = 0; kt < nk; ++kt) {
    if (NST > 2 && kt + NST - 2 < nk) wait_vmcnt((NST - 2) * LPW);
    else wait_vmcnt(0);
    lds_barrier();  // landed for every wave, and the slot read last step is free
    const int wr = rd == 0 ? NST - 1 : rd - 1;
    if (kt + NST - 1 < nk) issue(kt + NST - 1, wr);
    const char* st = lds + rd * STAGE;
    rd = rd + 1 == NST ? 0 : rd + 1;
    bf16x8 af[2][FN], bfr[2][FM];
    auto load_frags = [&](int kk, int buf) {
#pragma unroll
      for (int i = 0; i < FN; ++i) af[buf][i] = *(const bf16x8*)(st + (aoff[i][kk & 1] ^ ((kk >> 1) * 64)));
#pragma unroll
      for (int j = 0; j < FM; ++j) bfr[buf][j] = *(const bf16x8*)(st + (boff[j][kk & 1] ^ ((kk >> 1) * 64)));
    };
    load_frags(0, 0);
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      const int cb = kk & 1;
      if (kk + 1 < BK / 16) load_frags(kk + 1, cb ^ 1);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[cb][i], bfr[cb][j], acc[i][j], 0, 0, 0);
    }
  }

  // ---- epilogue ----
  const int wr0 = wm * WTM;  // first row of the wave's tile
  if constexpr (MODE == EX_OUT) {  // fp32, straight from the accumulators
    float* out = (float*)p.out;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int r = wr0 + 32 * j + l32;
      if (r >= rows) continue;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int gn = gn0 + 32 * i + 8 * q + 4 * hi;
          if (gn < p.N)
            *(f32x4*)(out + (int64_t)(row0 + r) * p.N + gn) =
                (f32x4){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        }
    }
    return;
  }
  if constexpr (MODE == EX_HIDDEN_GRAD) {
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int r = wr0 + 32 * j + l32;
      const bool in = r < rows;
      const float w = in ? (float)p.scale[p.slots[row0 + r]] : 0.f;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int gn = gn0 + 32 * i + 8 * q + 4 * hi;
          u32x2 d = {0u, 0u};
          if (in && gn < p.N) d = *(const u32x2*)(p.mul + (int64_t)(row0 + r) * p.N + gn);
          acc[i][j][4 * q + 0] *= w * bf16_lo(d[0]);
          acc[i][j][4 * q + 1] *= w * bf16_hi(d[0]);
          acc[i][j][4 * q + 2] *= w * bf16_lo(d[1]);
          acc[i][j][4 * q + 3] *= w * bf16_hi(d[1]);
        }
    }
  }
  // bf16 through this wave's LDS slab, 16-byte rows out
  lds_barrier();  // every wave is done reading the ring
  constexpr int SRB = WTN * 2, CPR = WTN / 8, RPI = 64 / CPR, NIT = WTM / RPI;
  char* slab = lds + wave * SLAB;
  const int c = lane % CPR, gn = gn0 + 8 * c;
  const bool col = gn < p.N;  // N is a multiple of 8: the whole 16-byte run
  auto to_slab = [&](auto f) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int nl = 32 * i + 8 * q + 4 * hi;
#pragma unroll
        for (int j = 0; j < FM; ++j) {
          float v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) v[x] = f(acc[i][j][4 * q + x]);
          const int ml = 32 * j + l32;
          const u32x2 w2 = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
          *(u32x2*)(slab + ml * SRB + (((nl >> 3) ^ (ml & (CPR - 1))) << 4) + 8 * hi) = w2;
        }
      }
  };
  auto from_slab = [&](bf16* dst) {
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int sl = RPI * it + lane / CPR;
      if (col && wr0 + sl < rows)
        *(u32x4*)(dst + (int64_t)(row0 + wr0 + sl) * p.N + gn) = *(const u32x4*)(slab + sl * SRB + ((c ^ (sl & (CPR - 1))) << 4));
    }
  };
  if constexpr (MODE == EX_HIDDEN) {
    to_slab([](float x) {
      float y, d;
      gelu_both(x, y, d);
      return y;
    });
    from_slab((bf16*)p.out);
    if (p.out2) {
      to_slab([](float x) {
        float y, d;
        gelu_both(x, y, d);
        return d;
      });
      from_slab(p.out2);
    }
  } else {
    to_slab([](float x) { return x; });
    from_slab((bf16*)p.out);
  }
}

// ---- out[t] = residual[t] + sum over s of w y (y fp32 rows), eight channels a thread ----
struct ExpertCombine {
  const float* y;
  const bf16* yb;         // the backward's rows instead of y (no weights)
  const bf16* weights;
  const int32_t* slot_row;
  const bf16* residual;
  bf16* out;
  int64_t n, ldr;         // tokens * chunks of eight channels
  int chunks, top_k;
};

template <bool BWD>
__global__ __launch_bounds__(256) void expert_combine_kernel(ExpertCombine p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.n) return;
  const int64_t t = i / p.chunks;
  const int c = (int)(i - t * p.chunks) * 8;
  const int64_t ld = (int64_t)p.chunks * 8;
  float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (!BWD && p.residual) {
    const u32x4 r = *(const u32x4*)(p.residual + t * p.ldr + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[2 * e] = bf16_lo(r[e]);
      a[2 * e + 1] = bf16_hi(r[e]);
    }
  }
  for (int s = 0; s < p.top_k; ++s) {
    const int r = p.slot_row[t * p.top_k + s];
    if (r < 0) continue;
    if (BWD) {
      const u32x4 v = *(const u32x4*)(p.yb + (int64_t)r * ld + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[2 * e] += bf16_lo(v[e]);
        a[2 * e + 1] += bf16_hi(v[e]);
      }
    } else {
      const float w = (float)p.weights[t * p.top_k + s];
      const f32x4 u = *(const f32x4*)(p.y + (int64_t)r * ld + c), v = *(const f32x4*)(p.y + (int64_t)r * ld + c + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = fmaf(w, u[e], a[e]);
        a[4 + e] = fmaf(w, v[e], a[4 + e]);
      }
    }
  }
  *(u32x4*)(p.out + i * 8) = (u32x4){pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7])};
}

// ---- the pairs' half of the backward: gs_r = w g[t] and dw = <g[t], y_r>; a wave a pair ----
struct ExpertScatter {
  const bf16* g;  // [T, N]
  const float* y;
  const bf16* weights;
  const int32_t* slot_row;
  bf16* gs;       // or null
  bf16* dw;       // or null
  int64_t pairs;
  int top_k, N;
};

__global__ __launch_bounds__(256) void expert_scatter_kernel(ExpertScatter p) {
  const int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (s >= p.pairs) return;
  const int r = p.slot_row[s];
  if (r < 0) {
    if (p.dw && lane == 0) p.dw[s] = (bf16)0.f;
    return;
  }
  const bf16* g = p.g + s / p.top_k * p.N;
  const float* y = p.y + (int64_t)r * p.N;
  const float w = (float)p.weights[s];
  float d = 0.f;
  for (int c = lane * 8; c < p.N; c += 512) {
    const u32x4 v = *(const u32x4*)(g + c);
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = bf16_lo(v[e]), b = bf16_hi(v[e]);
      o[e] = pack_bf16x2(w * a, w * b);
      if (p.dw) d = fmaf(b, y[c + 2 * e + 1], fmaf(a, y[c + 2 * e], d));
    }
    if (p.gs) *(u32x4*)(p.gs + (int64_t)r * p.N + c) = o;
  }
  if (p.dw) {
#pragma unroll
    for (int k = 32; k; k >>= 1) d += __shfl_xor(d, k);
    if (lane == 0) p.dw[s] = (bf16)d;
  }
}

// ---- w[e] [R, C] -> wt[e] [C, R], 64 x 64 tiles through LDS ----
__global__ __launch_bounds__(256) void expert_transpose_kernel(const bf16* __restrict__ w, bf16* __restrict__ wt, int R, int C) {
  __shared__ bf16 s[64][72];
  const int64_t base = (int64_t)blockIdx.z * R * C;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, tid = threadIdx.x;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = (tid >> 3) + 32 * k, c = (tid & 7) * 8;
    if (r0 + r < R && c0 + c < C) *(u32x4*)&s[r][c] = *(const u32x4*)(w + base + (int64_t)(r0 + r) * C + c0 + c);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c = (tid >> 3) + 32 * k, r = (tid & 7) * 8;
    if (c0 + c < C && r0 + r < R) {
      bf16x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = s[r + e][c];
      *(bf16x8*)(wt + base + (int64_t)(c0 + c) * R + r0 + r) = v;
    }
  }
}

// ---- the weights' gradients: out[e] [N, K] = sum over the expert's rows of g[r, n] x[r, k] ----
// One 256 x 256 tile of one expert a workgroup, stages of 64 rows; both operands are read
// transposed out of LDS (ds_read_b64_tr_b16), the column sums of g by a ones operand.
struct ExpertWgrad {
  const bf16* g;
  const bf16* x;
  const int32_t* rows;  // gather of x, or null
  const int32_t* offsets;
  bf16* out;
  bf16* bias_out;       // [E, N] or null
  int64_t ldg, ldx;
  int N, K, nt, kt, top_k;
};

constexpr int EW_BK = 64, EW_HALF = EW_BK * 512, EW_STAGE = 2 * EW_HALF;

template <bool GATHER>
__global__ __launch_bounds__(512, 1) void expert_wgrad_kernel(ExpertWgrad p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NW = 8, LPW = EW_HALF / 1024 / NW;
  __shared__ __attribute__((aligned(1024))) char lds[2 * EW_STAGE];
  const int tid = (int)__builtin_amdgcn_workitem_id_x();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n16 = lane & 15, g4 = lane >> 4;
  const int wk = wave >> 2, wn = wave & 3;  // wave tile: 128 k x 64 n
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  int w = xcd_tile_order((int)gridDim.x, (int)__builtin_amdgcn_workgroup_id_x());
  const int tk = w % p.kt;
  w /= p.kt;
  const int tn = w % p.nt, e = w / p.nt;
  const int k0 = tk * 256, n0 = tn * 256;
  const int row0 = p.offsets[e], rows = p.offsets[e + 1] - row0;
  const int nk = (rows + EW_BK - 1) / EW_BK;

  uint32_t vx[LPW], vg[LPW];  // GATHER: vx without the row
  int rr[LPW];
#pragma unroll
  for (int j = 0; j < LPW; ++j) {
    const int row = 2 * (j * NW + wave) + (lane >> 5), c = (lane & 31) ^ ((row & 7) << 1);
    rr[j] = row;
    vx[j] = k0 + 8 * c < p.K ? (uint32_t)((GATHER ? 0 : row * p.ldx * 2) + c * 16) : OOB;
    vg[j] = n0 + 8 * c < p.N ? (uint32_t)(row * p.ldg * 2 + c * 16) : OOB;
  }
  const char* xb = (const char*)(p.x + (GATHER ? 0 : (int64_t)row0 * p.ldx) + k0);
  const char* gb = (const char*)(p.g + (int64_t)row0 * p.ldg + n0);
  uint32_t tok[LPW];  // GATHER: byte offsets of the next stage's rows of x
  auto fetch = [&](int kt) {
    if constexpr (GATHER) {
#pragma unroll
      for (int j = 0; j < LPW; ++j) {
        const int r = kt * EW_BK + rr[j];
        tok[j] = r < rows ? (uint32_t)(p.rows[row0 + r] / p.top_k) * (uint32_t)(p.ldx * 2) : 0u;
      }
    }
  };
  auto issue = [&](int kt, int slot, bool is_g) {
    const int left = rows - kt * EW_BK;
    const u32x4 r = is_g ? make_rsrc(gb + (int64_t)kt * EW_BK * p.ldg * 2, OOB)
                         : make_rsrc(GATHER ? xb : xb + (int64_t)kt * EW_BK * p.ldx * 2, OOB);
    const uint32_t dst = lds_base + slot * EW_STAGE + (is_g ? EW_HALF : 0) + wave * 1024;
#pragma unroll
    for (int j = 0; j < LPW; ++j) {
      uint32_t vo = is_g ? vg[j] : vx[j];
      if (GATHER && !is_g && vo != OOB) vo += tok[j];
      if (left < EW_BK && rr[j] >= left) vo = OOB;
      dma_row16(r, dst + j * NW * 1024, vo);
    }
  };

  const int tr = 4 * g4 + (n16 >> 2);
  auto frag_off = [&](int col) {
    const int c = col / 8 + ((n16 & 3) >> 1);
    return (uint32_t)(tr * 512 + ((c ^ ((tr & 7) << 1)) << 4) + 8 * (n16 & 1));
  };
  uint32_t ao[8], bo[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) ao[i] = frag_off(128 * wk + 16 * i);
#pragma unroll
  for (int j = 0; j < 4; ++j) bo[j] = EW_HALF + frag_off(64 * wn + 16 * j);
  auto frag = [&](const char* st, uint32_t off, int kk) {
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, st + off + kk * 32 * 512));
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, st + off + kk * 32 * 512 + 16 * 512));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  f32x4 acc[8][4], bacc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bacc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i][j] = bacc[j];
  }
  bf16x8 ones;
#pragma unroll
  for (int k = 0; k < 8; ++k) ones[k] = (bf16)1.f;
  const bool sums = p.bias_out && tk == 0 && wk == 0;  // uniform per wave
  if (nk > 0) {
    fetch(0);
    issue(0, 0, false);
    issue(0, 0, true);
    fetch(1);
  }
  for (int kt = 0; kt < nk; ++kt) {
    wait_vmcnt(0);
    lds_barrier();  // the stage has landed for every wave; the other slot is free
    const int wr = (kt + 1) & 1;
    if (kt + 1 < nk) {
      issue(kt + 1, wr, false);
      fetch(kt + 2);
    }
    const char* st = lds + (kt & 1) * EW_STAGE;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 a[8], b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = frag(st, bo[j], kk);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = frag(st, ao[i], kk);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
      if (sums) {
#pragma unroll
        for (int j = 0; j < 4; ++j) bacc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, b[j], bacc[j], 0, 0, 0);
      }
      if (kk == 0 && kt + 1 < nk) {
        __builtin_amdgcn_sched_barrier(0);
        issue(kt + 1, wr, true);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if (sums && g4 == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 64 * wn + 16 * j + n16;
      if (n < p.N) p.bias_out[(int64_t)e * p.N + n] = (bf16)bacc[j][0];
    }
  }
  bf16* out = p.out + (int64_t)e * p.N * p.K;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + 64 * wn + 16 * j + n16;
    if (n >= p.N) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k0 + 128 * wk + 16 * i + 4 * g4;
      if (k < p.K)
        *(u32x2*)(out + (int64_t)n * p.K + k) =
            (u32x2){pack_bf16x2(acc[i][j][0], acc[i][j][1]), pack_bf16x2(acc[i][j][2], acc[i][j][3])};
    }
  }
#endif
}

// Rows of a tile: 64 where an expert has fewer than 96 rows on average, else 128.
static int expert_tile(int64_t pairs, int experts) { return pairs < 96 * (int64_t)experts ? 64 : 128; }

template <int MODE>
static int launch_expert_gemm(ExpertGemm p, int64_t pairs, int experts, int tile, hipStream_t st) {
  p.nt = (p.N + tile - 1) / tile;
  const int64_t mt = pairs / tile + std::min<int64_t>(experts, pairs), total = mt * p.nt;
  if (total > 0x7fffffff) return fail(STRATA_HIP_EUNSUPPORTED, "expert_mlp: problem too large for one launch");
  if (tile == 128)
    hipLaunchKernelGGL((expert_gemm_kernel<128, 128, 4, 2, 2, MODE>), dim3((unsigned)total), dim3(512), 0, st, p);
  else
    hipLaunchKernelGGL((expert_gemm_kernel<64, 64, 2, 2, 4, MODE>), dim3((unsigned)total), dim3(256), 0, st, p);
  return check_launch("expert_gemm_kernel");
}

static int launch_wgrad(const ExpertWgrad& q, int experts, hipStream_t st) {
  ExpertWgrad p = q;
  p.nt = (p.N + 255) / 256;
  p.kt = (p.K + 255) / 256;
  const int64_t total = (int64_t)p.nt * p.kt * experts;
  if (total > 0x7fffffff) return fail(STRATA_HIP_EUNSUPPORTED, "expert_mlp_bwd: problem too large for one launch");
  if (p.rows) hipLaunchKernelGGL(expert_wgrad_kernel<true>, dim3((unsigned)total), dim3(512), 0, st, p);
  else hipLaunchKernelGGL(expert_wgrad_kernel<false>, dim3((unsigned)total), dim3(512), 0, st, p);
  return check_launch("expert_wgrad_kernel");
}

static int expert_check(const std::string& name, const strata_hip_expert_mlp_args* a) {
  if (!a) return fail(STRATA_HIP_EINVAL, name + ": null args");
  if (a->tokens < 0 || a->top_k <= 0 || a->experts <= 0 || a->dim <= 0 || a->hidden <= 0 || a->out_dim <= 0)
    return fail(STRATA_HIP_EINVAL, name + ": bad sizes");
  if (a->dim % 8 || a->hidden % 8 || a->out_dim % 8)
    return fail(STRATA_HIP_EINVAL, name + ": dim, hidden and out_dim must be multiples of 8");
  const int64_t pairs = a->tokens * (int64_t)a->top_k;
  if (a->experts > 512 || pairs > 0x7ffffff0 || a->dim > 32768 || a->hidden > 32768 || a->out_dim > 32768)
    return fail(STRATA_HIP_EUNSUPPORTED, name + ": at most 512 experts, widths 32768 and 2^31 pairs");
  if (a->tile != expert_tile(pairs, a->experts)) return fail(STRATA_HIP_EINVAL, name + ": tile is not strata_hip_expert_tile()'s");
  if (!a->w1 || !a->w2 || !a->offsets || !a->tiles) return fail(STRATA_HIP_EINVAL, name + ": null pointer");
  if (((uintptr_t)a->w1 & 15) || ((uintptr_t)a->w2 & 15) || ((uintptr_t)a->b1 & 7) || ((uintptr_t)a->b2 & 7))
    return fail(STRATA_HIP_EINVAL, name + ": weights must be 16-byte, biases 8-byte aligned");
  if (pairs == 0) return STRATA_HIP_OK;
  if (!a->x || !a->weights || !a->row_slot || !a->slot_row || !a->h || !a->y)
    return fail(STRATA_HIP_EINVAL, name + ": null pointer");
  if (((uintptr_t)a->x & 15) || ((uintptr_t)a->h & 15) || ((uintptr_t)a->y & 15) || ((uintptr_t)a->dact & 15) || a->ldx % 8 ||
      (a->tokens > 1 && a->ldx < a->dim))
    return fail(STRATA_HIP_EINVAL, name + ": x, h, y and dact must be 16-byte aligned, the row stride of x a multiple of 8");
  // the products address their rows of x (and of dout) by 32-bit offsets
  if (((a->tokens - 1) * a->ldx + a->dim) * 2 >= (int64_t)OOB - 4096 || a->tokens * a->out_dim * 2 >= (int64_t)OOB - 4096)
    return fail(STRATA_HIP_EUNSUPPORTED, name + ": tokens of 2 GiB or more in one call");
  return STRATA_HIP_OK;
}

}  // namespace strata

using namespace strata;

extern "C" int32_t strata_hip_expert_tile(int64_t pairs, int32_t experts) { return expert_tile(pairs, experts); }

extern "C" int strata_hip_expert_mlp(const strata_hip_expert_mlp_args* a, void* stream) {
  if (const int rc = expert_check("expert_mlp", a)) return rc;
  if (a->tokens == 0) return STRATA_HIP_OK;
  if (!a->out || ((uintptr_t)a->out & 15) || ((uintptr_t)a->residual & 15) ||
      (a->residual && (a->ldr % 8 || (a->tokens > 1 && a->ldr < a->out_dim))))
    return fail(STRATA_HIP_EINVAL, "expert_mlp: out and residual must be 16-byte aligned, row strides multiples of 8");
  hipStream_t st = (hipStream_t)stream;
  const int64_t pairs = a->tokens * (int64_t)a->top_k;
  ExpertGemm g = {};
  g.offsets = a->offsets;
  g.tiles = a->tiles;
  g.top_k = a->top_k;
  g.x = (const bf16*)a->x;
  g.ldx = a->ldx;
  g.rows = a->row_slot;
  g.w = (const bf16*)a->w1;
  g.bias = (const bf16*)a->b1;
  g.out = a->h;
  g.out2 = (bf16*)a->dact;
  g.N = a->hidden;
  g.K = a->dim;
  if (const int rc = launch_expert_gemm<EX_HIDDEN>(g, pairs, a->experts, a->tile, st)) return rc;
  g.x = (const bf16*)a->h;
  g.ldx = a->hidden;
  g.rows = nullptr;
  g.w = (const bf16*)a->w2;
  g.bias = (const bf16*)a->b2;
  g.out = a->y;
  g.out2 = nullptr;
  g.N = a->out_dim;
  g.K = a->hidden;
  if (const int rc = launch_expert_gemm<EX_OUT>(g, pairs, a->experts, a->tile, st)) return rc;
  ExpertCombine c = {};
  c.y = a->y;
  c.weights = (const bf16*)a->weights;
  c.slot_row = a->slot_row;
  c.residual = (const bf16*)a->residual;
  c.ldr = a->ldr;
  c.out = (bf16*)a->out;
  c.chunks = a->out_dim / 8;
  c.top_k = a->top_k;
  c.n = a->tokens * c.chunks;
  if (c.n > 0x7fffffffll * 256) return fail(STRATA_HIP_EUNSUPPORTED, "expert_mlp: problem too large for one launch");
  hipLaunchKernelGGL(expert_combine_kernel<false>, dim3((unsigned)((c.n + 255) / 256)), dim3(256), 0, st, c);
  return check_launch("expert_combine_kernel");
}

extern "C" int strata_hip_expert_mlp_bwd(const strata_hip_expert_mlp_bwd_args* b, void* stream) {
  const std::string name = "expert_mlp_bwd";
  if (!b) return fail(STRATA_HIP_EINVAL, name + ": null args");
  const strata_hip_expert_mlp_args* a = &b->fwd;
  if (const int rc = expert_check(name, a)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const int64_t pairs = a->tokens * (int64_t)a->top_k;
  const bool hid = b->dx || b->dw1 || b->db1;  // gradients below the hidden layer
  if (pairs > 0) {
    if (!b->dout || ((uintptr_t)b->dout & 15)) return fail(STRATA_HIP_EINVAL, name + ": dout must be given, 16-byte aligned");
    if ((b->dw2 || b->db2) && !b->gs) return fail(STRATA_HIP_EINVAL, name + ": gs is needed for dw2 and db2");
    if (hid && (!a->dact || !b->gz || !b->w2t)) return fail(STRATA_HIP_EINVAL, name + ": dact, gz and w2t are needed for dx, dw1 and db1");
    if (b->dx && (!b->dxs || !b->w1t)) return fail(STRATA_HIP_EINVAL, name + ": dxs and w1t are needed for dx");
  }
  if ((b->db2 && !b->dw2) || (b->db1 && !b->dw1)) return fail(STRATA_HIP_EINVAL, name + ": a bias gradient comes with its weight's");
  const void* all[] = {b->gs, b->gz, b->dxs, b->w1t, b->w2t, b->dx, b->dw1, b->dw2};
  for (const void* q : all)
    if ((uintptr_t)q & 15) return fail(STRATA_HIP_EINVAL, name + ": workspaces and gradients must be 16-byte aligned");
  if (pairs > 0 && (b->dweights || b->dw2)) {
    ExpertScatter s = {};
    s.g = (const bf16*)b->dout;
    s.y = a->y;
    s.weights = (const bf16*)a->weights;
    s.slot_row = a->slot_row;
    s.gs = b->dw2 ? (bf16*)b->gs : nullptr;
    s.dw = (bf16*)b->dweights;
    s.pairs = pairs;
    s.top_k = a->top_k;
    s.N = a->out_dim;
    hipLaunchKernelGGL(expert_scatter_kernel, dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, st, s);
    if (const int rc = check_launch("expert_scatter_kernel")) return rc;
  }
  auto transpose = [&](const void* w, void* wt, int R, int C) {
    hipLaunchKernelGGL(expert_transpose_kernel, dim3((C + 63) / 64, (R + 63) / 64, a->experts), dim3(256), 0, st,
                       (const bf16*)w, (bf16*)wt, R, C);
    return check_launch("expert_transpose_kernel");
  };
  if (b->dw2) {  // without rows: zeros
    ExpertWgrad w = {};
    w.g = (const bf16*)b->gs;
    w.x = (const bf16*)a->h;
    w.offsets = a->offsets;
    w.out = (bf16*)b->dw2;
    w.bias_out = (bf16*)b->db2;
    w.ldg = a->out_dim;
    w.ldx = a->hidden;
    w.N = a->out_dim;
    w.K = a->hidden;
    w.top_k = 1;
    if (const int rc = launch_wgrad(w, a->experts, st)) return rc;
  }
  if (!hid) return STRATA_HIP_OK;
  ExpertGemm g = {};
  g.offsets = a->offsets;
  g.tiles = a->tiles;
  g.top_k = a->top_k;
  if (pairs > 0) {
    if (const int rc = transpose(a->w2, b->w2t, a->out_dim, a->hidden)) return rc;
    g.x = (const bf16*)b->dout;
    g.ldx = a->out_dim;
    g.rows = a->row_slot;
    g.slots = a->row_slot;
    g.scale = (const bf16*)a->weights;
    g.w = (const bf16*)b->w2t;
    g.mul = (const bf16*)a->dact;
    g.out = b->gz;
    g.N = a->hidden;
    g.K = a->out_dim;
    if (const int rc = launch_expert_gemm<EX_HIDDEN_GRAD>(g, pairs, a->experts, a->tile, st)) return rc;
  }
  if (b->dw1) {
    ExpertWgrad w = {};
    w.g = (const bf16*)b->gz;
    w.x = (const bf16*)a->x;
    w.rows = a->row_slot;
    w.offsets = a->offsets;
    w.out = (bf16*)b->dw1;
    w.bias_out = (bf16*)b->db1;
    w.ldg = a->hidden;
    w.ldx = a->ldx;
    w.N = a->hidden;
    w.K = a->dim;
    w.top_k = a->top_k;
    if (const int rc = launch_wgrad(w, a->experts, st)) return rc;
  }
  if (b->dx && pairs > 0) {
    if (const int rc = transpose(a->w1, b->w1t, a->hidden, a->dim)) return rc;
    g.x = (const bf16*)b->gz;
    g.ldx = a->hidden;
    g.rows = nullptr;
    g.w = (const bf16*)b->w1t;
    g.out = b->dxs;
    g.N = a->dim;
    g.K = a->hidden;
    if (const int rc = launch_expert_gemm<EX_INPUT_GRAD>(g, pairs, a->experts, a->tile, st)) return rc;
    ExpertCombine c = {};
    c.yb = (const bf16*)b->dxs;
    c.slot_row = a->slot_row;
    c.out = (bf16*)b->dx;
    c.chunks = a->dim / 8;
    c.top_k = a->top_k;
    c.n = a->tokens * c.chunks;
    if (c.n > 0x7fffffffll * 256) return fail(STRATA_HIP_EUNSUPPORTED, name + ": problem too large for one launch");
    hipLaunchKernelGGL(expert_combine_kernel<true>, dim3((unsigned)((c.n + 255) / 256)), dim3(256), 0, st, c);
    return check_launch("expert_combine_kernel");
  }
  return STRATA_HIP_OK;
}
