// The chosen experts' MLPs for gfx950: grouped matrix products over rows sorted by expert.
//
//   out[t] = residual[t] + sum over slots s of w[t, s] (gelu(x[t] W1_e^T + b1_e) W2_e^T + b2_e),  e = index[t, s]
//
// Row r of the products is a pair (t, s) in the plan's order; products over tokens gather
// their rows as they copy them into LDS, so no sorted copy of x or dout exists.  The pair's
// weight scales its hidden row before that is rounded to bf16, so the sum over slots needs
// no weights and dW2 no scaled copy of dout:
//   h_r = w' gelu(x[t] W1_e^T + b1_e)  bf16, with gelu' in fp16 (its values lie in (-0.13, 1.13)) for a backward
//   y_r = h_r W2_e^T + w' b2_e         fp32: out is rounded once
//   out[t] = residual[t] + sum_s y     in slot order
// w' = w, or 1 where |w| < 2^-100: such a pair adds nothing, but its weight has a gradient.
// Backward, g = dout:
//   dw[t, s] = <g[t], y_r> / w'
//   gz_r = w (g[t] W2_e) gelu'         bf16 (an operand of the next three)
//   dW2_e = sum_r g[t]^T h_r  db2_e = sum_r w g[t]  dW1_e = sum_r gz_r^T x[t]  db1_e = sum_r gz_r
//   dx[t] = sum_s (gz W1_e)_r          fp32 rows, in slot order
// Each gradient then has one rounding of an operand to bf16 and its own: 2.35e-3 relative, 1.66e-3
// from rounding the result alone (h or gz in more bits would be a second half of each as operands,
// four of the six products twice; the dense MLP rounds its hidden layer alike).  The backward's
// products take the weights along their rows: they are read transposed out of LDS
// (ds_read_b64_tr_b16), no transposed copy is made.  Every sum has an order fixed by the
// sizes and the plan: results repeat bit for bit.
#include <algorithm>

#include "common.h"

namespace strata {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void gelu_both(float x, float& y, float& d) {
  // x s and its derivative s + x s (1 - s) 2u' with s = sigmoid(2u), u = sqrt(2/pi) (x + 0.044715 x^3).
  // Beyond 1e15 s is 0 or 1, and x^2, held there, stays finite: 0 times it is 0.
  constexpr float c = 0.7978845608028654f, k1 = 2.f * 1.4426950408889634f * c;
  const float xx = fminf(x * x, 1e30f);
  const float t = x * fmaf(k1 * 0.044715f, xx, k1);
  const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-t));
  y = x * s;
  d = fmaf(y * (1.f - s), 2.f * c * fmaf(3.f * 0.044715f, xx, 1.f), s);
}

// Whether a pair's weight counts as nothing, and what its row is scaled by (a weight that
// is no number scales).
__device__ __forceinline__ bool no_weight(float w) { return fabsf(w) < 0x1p-100f; }
__device__ __forceinline__ float row_scale(float w) { return no_weight(w) ? 1.f : w; }

struct ExpertGemm {
  const bf16* x;
  const bf16* w;         // [E, N, K], WT: [E, K, N]
  const bf16* bias;      // [E, N] or null
  const _Float16* mul;   // HIDDEN_GRAD: gelu', [P, N]
  void* out;             // [P, N] bf16, OUT: fp32
  _Float16* out2;        // HIDDEN: gelu' or null
  const int32_t* token;  // row_token and row_weight of the plan
  const float* weight;
  const int32_t* offsets;
  const int32_t* tiles;
  int64_t ldx;
  int N, K, nt;
  int round;             // 256 x 256 tiles that run at once
  const int32_t* index;  // without a plan: the pairs' experts and weights
  const bf16* weights;
  int pairs, top_k, experts;
};

enum { EX_HIDDEN = 0, EX_OUT = 1, EX_HIDDEN_GRAD = 2 };

// Chunks of 16 bytes of an LDS row are stored at their index xor these:
// K-contiguous rows of 128 bytes, read 16 bytes a lane by 32 rows at one chunk, and
// (WT) rows of BN columns, read transposed by 8 rows at 4 chunks: each instruction's
// lanes then spread over all banks.
__device__ __forceinline__ int ex_swz(int row) { return (row & 7) ^ ((row >> 3) & 1); }
template <int BN>
__device__ __forceinline__ int ex_wswz(int row) {
  return BN == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
}

struct ExpertTile {
  int e, row0, rows, n0;
};

// The plan by scalar loads: they are counted apart from the copies in flight.
__device__ __forceinline__ int plan_load(const int32_t* p, int i) {
  return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)p)[__builtin_amdgcn_readfirstlane(i)];
}

// BM x BN tiles of the experts' products: x and w stream into an LDS ring of NST stages of
// 64 columns (buffer_load ... lds) ahead of v_mfma_f32_32x32x16_bf16, whose A operand the
// weights are: a lane owns four consecutive columns of one row.
// BIG: 256 x 256, one workgroup a CU walks over the tiles; the last step of a tile starts
// the next one's first stage.  Otherwise one tile a workgroup and several workgroups a CU.
// TAIL: the 256 x 256 tiles of a last round that would leave half of the CUs or more idle,
// each as four 128 x 128 or sixteen 64 x 64 ones (the same sums in the same order).
// Bound by the matrix instructions and their feeding: 32768 pairs of 8 experts, 1024 -> 4096 ->
// 1024, the two products forward with what a backward needs 351 and 291 us (783 and 945 TFLOP/s; a
// dense library product of these sizes 217 and 188 without GELU, bias, gather or fp32 output), the
// backward's 330 to 350 (gelu' and the weight in the epilogue) and 291; 54% of the cycles issue MFMAs in
// the second, 43% in the first, whose epilogue writes 520 MB; no LDS conflicts, 68 - 75% of the reads
// hit L2.  Every 128 x 128 tiles instead: 20% slower; the K loop's barrier elsewhere: spills.
template <int BM, int BN, int WGM, int WGN, int NST, int MODE, bool WT, bool TAIL>
__global__ __launch_bounds__(64 * WGM * WGN, 1) void expert_gemm_kernel(ExpertGemm p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr bool BIG = BM == 256, GATHER = MODE != EX_OUT;
  constexpr int BK = 64, NW = WGM * WGN;
  constexpr int WTM = BM / WGM, WTN = BN / WGN, FM = WTM / 32, FN = WTN / 32;
  constexpr int ROWB = BK * 2, CH = ROWB / 16, RPC = 1024 / ROWB;
  constexpr int XB = BM * ROWB, XCH = XB / 1024, STAGE = XB + BN * ROWB;
  constexpr int LPX = XCH / NW, LPW = BN * ROWB / 1024 / NW;  // 1-KiB copies a wave and stage
  constexpr int WLPR = BN / 8, WRPC = 64 / WLPR;             // WT: lanes a row, rows a copy
  constexpr int SLAB = 32 * WTN * 4;
  static_assert(WTM % 32 == 0 && WTN % 32 == 0 && XCH % NW == 0 && (STAGE / 1024) % NW == 0, "wave tile / stage layout");
  static_assert(NW * SLAB <= (BIG ? STAGE : NST * STAGE) && (!BIG || NST == 2), "the epilogue slabs fit the ring");
  // BIG: what a tile needs besides its stages, copied to LDS a tile ahead and read where it is
  // used (loads into registers would wait, in order, for the copies and stores before them):
  // the rows' tokens, their weights, the columns' bias.
  constexpr int TOKENS = 0, WEIGHTS = BM * 4, BIAS = BM * 8, META = BM * 8 + BN * 2;
  __shared__ __attribute__((aligned(1024))) char lds[NST * STAGE + (BIG ? 2 * META : 0)];

  const int tid = (int)__builtin_amdgcn_workitem_id_x();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wm = wave / WGN, wn = wave % WGN, l32 = lane & 31, hi = lane >> 5;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const bool weigh = MODE != EX_OUT || p.bias, biased = MODE != EX_HIDDEN_GRAD && p.bias;  // uniform

  // The grid is sized for the most tiles that the pairs can make; the plan says how many there are.
  const int mt = plan_load(p.tiles, 0), all = mt * p.nt, wg_id = (int)__builtin_amdgcn_workgroup_id_x();
  int tail = BIG || TAIL ? all > p.round ? all % p.round : 0 : 0;
  if (2 * tail > p.round) tail = 0;
  constexpr int SUB = TAIL ? 256 / BM : 1;
  const int total = BIG ? all - tail : TAIL ? SUB * SUB * tail : all;
  if (wg_id >= total) return;
  auto tile_at = [&](int t) {
    const int wg = xcd_tile_order(all, TAIL ? all - tail + t / (SUB * SUB) : t);
    constexpr int GRP = BIG || TAIL ? 4 : 8;  // row panels x every column panel, row panel fastest
    const int gi = wg / (GRP * p.nt), li = wg % (GRP * p.nt), gmn = min(GRP, mt - gi * GRP);
    const int tm = gi * GRP + li % gmn;
    ExpertTile r;
    r.e = plan_load(p.tiles, 1 + 2 * tm);
    r.row0 = plan_load(p.tiles, 2 + 2 * tm);
    r.rows = plan_load(p.offsets, r.e + 1) - r.row0;
    r.n0 = (li / gmn) * (SUB * BN);
    if (TAIL) {
      const int sr = t / SUB % SUB, sc = t % SUB;
      r.rows = min(r.rows, SUB * BM) - BM * sr;
      r.row0 += BM * sr;
      r.n0 += BN * sc;
    }
    r.rows = min(r.rows, BM);
    return r;
  };
  const int nk = (p.K + BK - 1) / BK, ktail = p.K % BK;
  // wave w copies dwords 64 (w % 4) .. of the rows' tokens (w < 4) or weights, and of the bias
  auto issue_meta = [&](const ExpertTile& t, int buf) {
    const uint32_t dst = lds_base + NST * STAGE + buf * META;
    const int i = 64 * (wave & 3) + lane;
    const uint32_t vo = i < t.rows ? 4u * i : OOB;
    if (wave < 4) {
      if (GATHER) dma_dword(make_rsrc(p.token + t.row0, OOB), dst + TOKENS + 256 * wave, vo);
    } else if (weigh) {
      dma_dword(make_rsrc(p.weight + t.row0, OOB), dst + WEIGHTS + 256 * (wave - 4), vo);
    }
    if (biased && wave < BN / 128) {
      const int c = 128 * wave + 2 * lane;
      dma_dword(make_rsrc(p.bias + (int64_t)t.e * p.N + t.n0, OOB), dst + BIAS + 256 * wave, t.n0 + c < p.N ? 2u * c : OOB);
    }
  };
  // lane offsets of a tile's x rows (BIG: their tokens in LDS buffer buf)
  auto x_offsets = [&](const ExpertTile& t, uint32_t (&vo)[LPX], int buf) {
#pragma unroll
    for (int j = 0; j < LPX; ++j) {
      const int row = RPC * (j * NW + wave) + lane / CH;
      const uint32_t chunk = ((lane % CH) ^ ex_swz(row)) * 16;
      int64_t at = row;
      if (GATHER && BIG) at = *(const int*)(lds + NST * STAGE + buf * META + TOKENS + 4 * row);
      else if (GATHER && row < t.rows) at = p.token[t.row0 + row];
      vo[j] = row < t.rows ? (uint32_t)(at * p.ldx * 2) + chunk : OOB;
    }
  };
  auto w_offsets = [&](const ExpertTile& t, uint32_t (&vo)[LPW]) {
#pragma unroll
    for (int j = 0; j < LPW; ++j) {
      if (WT) {
        const int row = WRPC * (j * NW + wave) + lane / WLPR, chunk = (lane % WLPR) ^ ex_wswz<BN>(row);
        vo[j] = t.n0 + 8 * chunk < p.N ? (uint32_t)((uint32_t)row * p.N * 2) + chunk * 16 : OOB;
      } else {
        const int row = RPC * (j * NW + wave) + lane / CH, chunk = (lane % CH) ^ ex_swz(row);
        vo[j] = t.n0 + row < p.N ? (uint32_t)((uint32_t)row * p.K * 2) + chunk * 16 : OOB;
      }
    }
  };
  auto issue_x = [&](const ExpertTile& t, const uint32_t (&vo)[LPX], int kt, int slot) {
    const bf16* base = GATHER ? p.x : p.x + (int64_t)t.row0 * p.ldx;
    const u32x4 r = make_rsrc((const char*)base + (int64_t)kt * BK * 2, OOB);
    const uint32_t dst = lds_base + slot * STAGE + wave * 1024;
    if (ktail && kt == nk - 1) {  // uniform: chunks at or past K read as zero
#pragma unroll
      for (int j = 0; j < LPX; ++j)
        dma_row16(r, dst + j * NW * 1024, ((lane % CH) ^ ex_swz(RPC * (j * NW + wave) + lane / CH)) * 8 >= ktail ? OOB : vo[j]);
    } else {
#pragma unroll
      for (int j = 0; j < LPX; ++j) dma_row16(r, dst + j * NW * 1024, vo[j]);
    }
  };
  auto issue_w = [&](const ExpertTile& t, const uint32_t (&vo)[LPW], int kt, int slot) {
    const bf16* base = p.w + (int64_t)t.e * p.N * p.K + (WT ? (int64_t)kt * BK * p.N + t.n0 : (int64_t)t.n0 * p.K + kt * BK);
    const u32x4 r = make_rsrc(base, OOB);
    const uint32_t dst = lds_base + slot * STAGE + XB + wave * 1024;
    if (ktail && kt == nk - 1) {
#pragma unroll
      for (int j = 0; j < LPW; ++j) {
        const bool past = WT ? WRPC * (j * NW + wave) + lane / WLPR >= ktail
                             : ((lane % CH) ^ ex_swz(RPC * (j * NW + wave) + lane / CH)) * 8 >= ktail;
        dma_row16(r, dst + j * NW * 1024, past ? OOB : vo[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < LPW; ++j) dma_row16(r, dst + j * NW * 1024, vo[j]);
    }
  };

  // LDS offsets of the fragments: x (and w) for K sub-steps 0, 1 (2, 3 flip bit 2 of the chunk:
  // offset ^ 64); WT: rows 8 hi + 4 half + (lane & 15) / 4 of columns 32 i + 16 ((lane >> 4) & 1).
  uint32_t aoff[FN][WT ? 1 : 2], boff[FM][2];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    if (WT) {
      const int r4 = (lane & 15) >> 2, c = (wn * WTN + 32 * i) / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      aoff[i][0] = XB + (8 * hi + r4) * (BN * 2) + ((c ^ ex_wswz<BN>(r4)) << 4) + 8 * (lane & 1);
    } else {
      const int row = wn * WTN + 32 * i + l32;
      for (int kk = 0; kk < 2; ++kk) aoff[i][WT ? 0 : kk] = XB + row * ROWB + ((2 * kk + hi) ^ ex_swz(row)) * 16;
    }
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int row = wm * WTM + 32 * j + l32;
    for (int kk = 0; kk < 2; ++kk) boff[j][kk] = row * ROWB + ((2 * kk + hi) ^ ex_swz(row)) * 16;
  }
  auto load_frags = [&](const char* st, int kk, bf16x8 (&a)[FN], bf16x8 (&b)[FM]) {
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if constexpr (WT) {
        const char* q = st + aoff[i][0] + kk * 16 * (BN * 2);
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, q));
        const bf16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, q + 4 * (BN * 2)));
        a[i] = __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        a[i] = *(const bf16x8*)(st + (aoff[i][kk & 1] ^ ((kk >> 1) * 64)));
      }
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) b[j] = *(const bf16x8*)(st + (boff[j][kk & 1] ^ ((kk >> 1) * 64)));
  };

  f32x16 acc[FN][FM];
  ExpertTile t = tile_at(wg_id), tn = t;
  if (TAIL && (t.rows <= 0 || t.n0 >= p.N)) return;
  uint32_t xo[LPX], wo[LPW];
  int mb = 0;  // the tile's buffer
  if (BIG) {
    issue_meta(t, 0);
    wait_vmcnt(0);
    lds_barrier();
  }
  // BIG: slot rd holds the next stage to read, wr takes the next issue
  int rd = 0, wr = 1;
  bool in_flight = false;  // the tile's first stage was issued by the previous tile
  for (int ti = wg_id; ti < total; ti += (int)gridDim.x) {
    const bool more = BIG && ti + (int)gridDim.x < total;
    const int gn0 = t.n0 + wn * WTN, wr0 = wm * WTM;
    bf16x8 af[2][FN], bfr[2][FM];
    auto multiply = [&](int cb) {
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[cb][i], bfr[cb][j], acc[i][j], 0, 0, 0);
    };
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    if constexpr (BIG) {
      if (!in_flight) {
        if (ti != wg_id) {  // a product of one step: the tile's tokens are waited for here
          wait_vmcnt(0);
          lds_barrier();
        }
        x_offsets(t, xo, mb);
      }
      w_offsets(t, wo);
      if (!in_flight) {
        issue_x(t, xo, 0, rd);
        issue_w(t, wo, 0, rd);
      }
      if (more) tn = tile_at(ti + (int)gridDim.x);
      in_flight = false;
      auto kstep = [&](int kt, auto last) {
        constexpr bool LAST = decltype(last)::value;
        wait_vmcnt(0);
        lds_barrier();  // the stage has landed for every wave; slot wr is free
        if (more && kt == 0) issue_meta(tn, mb ^ 1);
        if (!LAST) {
          issue_x(t, xo, kt + 1, wr);
        } else if (more && kt > 0) {  // the next tile's first stage
          w_offsets(tn, wo);
          x_offsets(tn, xo, mb ^ 1);
          issue_x(tn, xo, 0, wr);
          issue_w(tn, wo, 0, wr);
          in_flight = true;
        }
        const char* st = lds + rd * STAGE;
        load_frags(st, 0, af[0], bfr[0]);
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
          if (kk + 1 < BK / 16) load_frags(st, kk + 1, af[(kk + 1) & 1], bfr[(kk + 1) & 1]);
          multiply(kk & 1);
          if (kk == 0 && !LAST) {  // the weights' copies behind the first MFMAs
            __builtin_amdgcn_sched_barrier(0);
            issue_w(t, wo, kt + 1, wr);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        __builtin_amdgcn_iglp_opt(1);
        rd ^= 1;
        wr ^= 1;
      };
      for (int kt = 0; kt + 1 < nk; ++kt) kstep(kt, std::false_type{});
      kstep(nk - 1, std::true_type{});
    } else {
      x_offsets(t, xo, 0);
      w_offsets(t, wo);
#pragma unroll
      for (int s = 0; s < NST - 1; ++s)
        if (s < nk) {
          issue_x(t, xo, s, s);
          issue_w(t, wo, s, s);
        }
      for (int kt = 0; kt < nk; ++kt) {
        if (NST > 2 && kt + NST - 2 < nk) wait_vmcnt((NST - 2) * (LPX + LPW));
        else wait_vmcnt(0);
        lds_barrier();  // landed for every wave, and the slot read last step is free
        const int ws = rd == 0 ? NST - 1 : rd - 1;
        if (kt + NST - 1 < nk) {
          issue_x(t, xo, kt + NST - 1, ws);
          issue_w(t, wo, kt + NST - 1, ws);
        }
        const char* st = lds + rd * STAGE;
        rd = rd + 1 == NST ? 0 : rd + 1;
        load_frags(st, 0, af[0], bfr[0]);
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
          const int cb = kk & 1;
          if (kk + 1 < BK / 16) load_frags(st, kk + 1, af[cb ^ 1], bfr[cb ^ 1]);
          multiply(cb);
        }
      }
    }

    // ---- epilogue: 32 rows of the wave's tile at a time through its LDS slab in fp32, back as
    // eight consecutive columns a lane, so that every load and store moves whole 16-byte runs of
    // a row (BIG: the slabs are in the slot read last, the other takes the next tile's stage)
    lds_barrier();  // every wave is done reading the last stage
    constexpr int NCH = WTN / 4, LPR = WTN / 8, RPI = 64 / LPR, NIT = 32 / RPI;
    char* slab = lds + (BIG ? wr * STAGE : 0) + wave * SLAB;
    const char* meta = lds + NST * STAGE + mb * META;
    const int lrow = lane / LPR, lc = lane % LPR, gn = gn0 + 8 * lc;
    const bool col = gn < p.N;  // N is a multiple of 8: the whole run
    float b8[8];
    {
      u32x4 b = {0u, 0u, 0u, 0u};
      if (biased)
        b = BIG ? *(const u32x4*)(meta + BIAS + 2 * (wn * WTN + 8 * lc)) : *(const u32x4*)(p.bias + (int64_t)t.e * p.N + min(gn, p.N - 8));
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        b8[2 * x] = bf16_lo(b[x]);
        b8[2 * x + 1] = bf16_hi(b[x]);
      }
    }
    f16x8 dv[2][NIT];  // HIDDEN_GRAD: gelu' of this pass and the next, loaded before this pass's stores
    auto load_mul = [&](int j) {
#pragma unroll
      for (int it = 0; it < NIT; ++it) {
        const int r = wr0 + 32 * j + RPI * it + lrow;
        dv[j & 1][it] = (f16x8){};
        if (col && r < t.rows) dv[j & 1][it] = *(const f16x8*)(p.mul + (int64_t)(t.row0 + r) * p.N + gn);
      }
    };
    if (MODE == EX_HIDDEN_GRAD) load_mul(0);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(f32x4*)(slab + l32 * (WTN * 4) + (((8 * i + 2 * q + hi) ^ (l32 & (NCH - 1))) << 4)) =
              (f32x4){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      if (MODE == EX_HIDDEN_GRAD && j + 1 < FM) load_mul(j + 1);
#pragma unroll
      for (int it = 0; it < NIT; ++it) {
        const int sl = RPI * it + lrow, r = wr0 + 32 * j + sl;
        const f32x4 z0 = *(const f32x4*)(slab + sl * (WTN * 4) + (((2 * lc) ^ (sl & (NCH - 1))) << 4));
        const f32x4 z1 = *(const f32x4*)(slab + sl * (WTN * 4) + (((2 * lc + 1) ^ (sl & (NCH - 1))) << 4));
        float v[8] = {z0[0], z0[1], z0[2], z0[3], z1[0], z1[1], z1[2], z1[3]};
        // the row's weight: scale of h, factor of the bias, factor of gz
        float w = 0.f;
        if (weigh) w = BIG ? *(const float*)(meta + WEIGHTS + 4 * r) : r < t.rows ? p.weight[t.row0 + r] : 0.f;
        if (MODE != EX_HIDDEN_GRAD) w = row_scale(w);
        const bool in = col && r < t.rows;
        const int64_t at = (int64_t)(t.row0 + r) * p.N + gn;
        if constexpr (MODE == EX_OUT) {
          f32x4 o0, o1;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            o0[x] = fmaf(w, b8[x], v[x]);
            o1[x] = fmaf(w, b8[4 + x], v[4 + x]);
          }
          if (in) {
            *(f32x4*)((float*)p.out + at) = o0;
            *(f32x4*)((float*)p.out + at + 4) = o1;
          }
        } else {
          f16x8 d8;
          u32x4 o;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            if constexpr (MODE == EX_HIDDEN) {
              float y, d;
              gelu_both(v[x] + b8[x], y, d);
              v[x] = y * w;
              d8[x] = (_Float16)d;
            } else {
              v[x] *= w * (float)dv[j & 1][it][x];
            }
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) o[x] = pack_bf16x2(v[2 * x], v[2 * x + 1]);
          if (in) {
            __builtin_nontemporal_store(o, (u32x4*)((bf16*)p.out + at));
            if (MODE == EX_HIDDEN && p.out2) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, d8), (u32x4*)(p.out2 + at));
          }
        }
      }
    }
    if (!BIG) return;
    t = tn;
    mb ^= 1;
  }
#endif
}

// ---- few rows an expert (a token or a handful while serving): 16 rows x 16 columns a
// workgroup, W waves with a share of K each, their sums added in LDS in wave order.  Bound by
// reading the weights, which go straight into registers: a lane reads 32 bytes of a weight row,
// four lanes its 128-byte line, and the contraction takes the columns in that order.  One token, two of
// 8 experts, 1024 -> 4096: 6.6 and 7.6 us for 16.8 MB each (2.5 and 2.2 TB/s; a launch that does
// nothing takes 2 to 3).
// DIRECT: up to 16 pairs, without a plan (the call's first launch of four): row r is pair r, and every
// wave finds its tile's expert, the tm-th that is named, and that expert's pairs from the index
// (the token's call 24.5 -> 21.9 us).
constexpr int EX_DIRECT = 16;
__device__ __forceinline__ int nth_bit(uint32_t m, int n) {
  for (int i = 0; i < n; ++i) m &= m - 1;
  return __ffs(m) - 1;  // -1: fewer than n + 1 bits
}
template <int MODE, int W, bool DIRECT>
__global__ __launch_bounds__(64 * W) void expert_few_kernel(ExpertGemm p) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ float red[W][16][20];
  const int tid = (int)__builtin_amdgcn_workitem_id_x(), wave = tid >> 6, lane = tid & 63, n16 = lane & 15, g4 = lane >> 4;
  const int id = (int)__builtin_amdgcn_workgroup_id_x();
  const int tm = id / p.nt, n0 = id % p.nt * 16;
  int e, row0 = 0, rows;
  uint32_t mine = 0u;  // DIRECT: the expert's pairs
  if constexpr (DIRECT) {
    int el = lane < p.pairs ? p.index[lane] : -1;
    if (el >= p.experts) el = -1;
    bool first = el >= 0;
    for (int s = 0; s < p.pairs; ++s) first = first && !(s < lane && __builtin_amdgcn_readlane(el, s) == el);
    const int lead = nth_bit((uint32_t)__ballot(first), tm);
    if (lead < 0) return;  // uniform: fewer experts are named
    e = __builtin_amdgcn_readlane(el, lead);
    mine = (uint32_t)__ballot(el == e);
    rows = __popc(mine);
  } else {
    if (tm >= plan_load(p.tiles, 0)) return;
    e = plan_load(p.tiles, 1 + 2 * tm);
    row0 = plan_load(p.tiles, 2 + 2 * tm);
    rows = min(plan_load(p.offsets, e + 1) - row0, 16);
  }
  auto row_at = [&](int r) { return DIRECT ? max(nth_bit(mine, r), 0) : row0 + r; };
  const bf16* w = p.w + ((int64_t)e * p.N + min(n0 + n16, p.N - 1)) * p.K;
  const bool live = n16 < rows;
  const int xr = row_at(live ? n16 : 0);
  const bf16* x = p.x + (int64_t)(MODE != EX_HIDDEN ? xr : DIRECT ? xr / p.top_k : live ? p.token[xr] : 0) * p.ldx;
  constexpr int U = 4;
  const int kc = (p.K + 64 * W - 1) / (64 * W) * 64, k0 = wave * kc, k1 = min(p.K, k0 + kc);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int k = k0; k < k1; k += 64 * U) {
    u32x4 a[U][2], b[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = k + 64 * u + 16 * g4 + 8 * h;
        a[u][h] = c < k1 ? *(const u32x4*)(w + c) : zero;
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = k + 64 * u + 16 * g4 + 8 * h;
        b[u][h] = live && c < k1 ? *(const u32x4*)(x + c) : zero;
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[u][h]), __builtin_bit_cast(bf16x8, b[u][h]),
                                                      acc, 0, 0, 0);
  }
  *(f32x4*)&red[wave][n16][4 * g4] = acc;  // row n16, columns 4 g4 .. + 3
  __syncthreads();
  const int r = tid >> 4, c = tid & 15;
  if (tid >= 256 || r >= rows || n0 + c >= p.N) return;
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) z += red[i][r][c];
  const int row = row_at(r);
  const float b = p.bias ? (float)p.bias[(int64_t)e * p.N + n0 + c] : 0.f;
  const float s = row_scale(DIRECT ? (float)p.weights[row] : p.weight[row]);
  const int64_t at = (int64_t)row * p.N + n0 + c;
  if (MODE == EX_HIDDEN) {
    float y, d;
    gelu_both(z + b, y, d);
    ((bf16*)p.out)[at] = (bf16)(y * s);
  } else {
    ((float*)p.out)[at] = fmaf(s, b, z);
  }
#endif
}

// One pair, or up to EX_FUSED (a token while serving) of at most EX_FUSED_K columns together: the second product and
// the sum over slots in one launch, 8 columns of every token a workgroup, whose 16 waves share the named
// experts and their contractions.  Two launches / this one, of 512 and 1024 columns, replayed, us (the whole call; called
// from Python the launch saved is 2.5 more): 1 pair, 4096 hidden columns 13.6 / 10.8 and 14.4 / 11.5; 2 pairs, 2048 12.2 / 11.4
// and 13.1 / 12.1, 4096 14.8 / 15.0 and 17.2 / 16.6, 5632 17.4 / 18.2 and 21.2 / 22.1; 3 pairs, 1024 11.6 / 11.3 and
// 12.3 / 11.9, 2816 14.9 / 17.0 and 17.7 / 19.5; 4 pairs, 512 11.1 / 10.7 and 12.5 / 11.7, 2048 14.3 / 16.6 and 17.2 / 18.3.
// One pair gains at every width (16384: 29.3 / 22.7 and 35.1 / 28.1); for 2 to 4 pairs limits of 6144, 8192, 9216 and 12288
// pairs x columns lose 1.4, 1.1, 1.0 and 1.4% on average over both ways of calling.
constexpr int EX_FUSED = 4, EX_FUSED_K = 9216, EX_FUSED_N = 8;
__global__ __launch_bounds__(1024) void expert_few_out_kernel(ExpertGemm p, const bf16* residual, int64_t ldr, bf16* out) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ float red[16][EX_FUSED][20];
  // a pair's expert (the index is read once), its place among the named ones (-1), the pair's among its expert's
  __shared__ int expert_of[EX_FUSED], expert_at[EX_FUSED], rank_at[EX_FUSED];
  const int tid = (int)__builtin_amdgcn_workitem_id_x(), lane = tid & 63, n16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), n0 = (int)__builtin_amdgcn_workgroup_id_x() * EX_FUSED_N;
  int el = lane < p.pairs ? p.index[lane] : -1;
  if (el < 0 || el >= p.experts) el = -1;
  int lead = lane, rank = 0;  // the first pair of this one's expert
  for (int s = 0; s < p.pairs; ++s) {
    const bool same = s < lane && __builtin_amdgcn_readlane(el, s) == el;
    lead = same ? min(lead, s) : lead;
    rank += same;
  }
  const uint32_t named = (uint32_t)__ballot(el >= 0 && lead == lane);
  const int count = __popc(named), per = count ? 16 / count : 16;
  if (wave == 0 && lane < p.pairs) {
    expert_of[lane] = el;
    expert_at[lane] = el >= 0 ? __popc(named & ((1u << lead) - 1)) : -1;
    rank_at[lane] = rank;
  }
  const int place = wave / per, part = wave % per;
  if (place < count) {  // uniform per wave
    const int e = __builtin_amdgcn_readlane(el, nth_bit(named, place));
    const uint32_t mine = (uint32_t)__ballot(el == e);
    const bool live = n16 < __popc(mine);
    const bf16* w = p.w + ((int64_t)e * p.N + n0 + n16 % EX_FUSED_N) * p.K;
    const bf16* x = p.x + (int64_t)(live ? nth_bit(mine, n16) : 0) * p.ldx;
    constexpr int U = 4;
    const int kc = (p.K + 64 * per - 1) / (64 * per) * 64, k0 = part * kc, k1 = min(p.K, k0 + kc);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int k = k0; k < k1; k += 64 * U) {
      u32x4 a[U][2], b[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = k + 64 * u + 16 * g4 + 8 * h;
          a[u][h] = n16 < EX_FUSED_N && c < k1 ? *(const u32x4*)(w + c) : zero;
          b[u][h] = live && c < k1 ? *(const u32x4*)(x + c) : zero;
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[u][h]), __builtin_bit_cast(bf16x8, b[u][h]),
                                                        acc, 0, 0, 0);
    }
    if (n16 < EX_FUSED) *(f32x4*)&red[wave][n16][4 * g4] = acc;
  }
  __syncthreads();
  const int t = tid / EX_FUSED_N, c = tid % EX_FUSED_N, n = n0 + c;  // N is a multiple of 8
  if (t * p.top_k >= p.pairs) return;
  float a = residual ? (float)residual[t * ldr + n] : 0.f;
  for (int s = 0; s < p.top_k; ++s) {
    const int pair = t * p.top_k + s, at = expert_at[pair];
    const float w = (float)p.weights[pair];
    if (at < 0 || no_weight(w)) continue;
    float z = 0.f;
    for (int i = 0; i < per; ++i) z += red[at * per + i][rank_at[pair]][c];
    a += p.bias ? fmaf(w, (float)p.bias[(int64_t)expert_of[pair] * p.N + n], z) : z;
  }
  out[(int64_t)t * p.N + n] = (bf16)a;
#endif
}

// ---- out[t] = residual[t] + sum over s of y_r, eight channels a thread; without weights: dx ----
// Bound by memory: 32768 tokens, 2 slots, 1024 channels with residual 78 us for 402 MB (5.1 TB/s); rows
// loaded past the caches, where part of what the products just wrote still is: 15 us more.
struct ExpertCombine {
  const float* y;
  const bf16* weights;    // [T, k] or null; a pair whose weight is nothing adds nothing
  const int32_t* slot_row;
  const bf16* residual;
  bf16* out;
  int64_t n, ldr;         // tokens * chunks of eight channels
  int chunks, top_k;
  int experts;            // without a plan: slot_row is the index, a pair's row the pair; else 0
};

__global__ __launch_bounds__(256) void expert_combine_kernel(ExpertCombine p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.n) return;
  const int64_t t = i / p.chunks;
  const int c = (int)(i - t * p.chunks) * 8;
  const int64_t ld = (int64_t)p.chunks * 8;
  float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (p.residual) {
    const u32x4 r = *(const u32x4*)(p.residual + t * p.ldr + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[2 * e] = bf16_lo(r[e]);
      a[2 * e + 1] = bf16_hi(r[e]);
    }
  }
  for (int s = 0; s < p.top_k; ++s) {
    int r = p.slot_row[t * p.top_k + s];
    if (p.experts) r = (uint32_t)r < (uint32_t)p.experts ? (int)t * p.top_k + s : -1;
    if (r < 0 || (p.weights && no_weight((float)p.weights[t * p.top_k + s]))) continue;
    const f32x4 u = *(const f32x4*)(p.y + (int64_t)r * ld + c), v = *(const f32x4*)(p.y + (int64_t)r * ld + c + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] += u[e];
      a[4 + e] += v[e];
    }
  }
  *(u32x4*)(p.out + i * 8) = (u32x4){pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7])};
}

// ---- dw = <g[t], y_r> / w'; a wave a pair (`pair0`: the launch's first one) ----
// Bound by memory: 32768 pairs of 1024 columns 26 us for 168 MB (6.5 TB/s, partly from the caches).
__global__ __launch_bounds__(256) void expert_dweight_kernel(const bf16* g, const float* yy, const bf16* weights,
                                                             const int32_t* slot_row, bf16* dw, int64_t pair0, int64_t pairs,
                                                             int top_k, int N) {
  const int64_t s = pair0 + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (s >= pairs) return;
  const int r = slot_row[s];
  if (r < 0) {
    if (lane == 0) dw[s] = (bf16)0.f;
    return;
  }
  g += s / top_k * N;
  const float* y = yy + (int64_t)r * N;
  float d = 0.f;
  for (int c = lane * 8; c < N; c += 512) {
    const u32x4 v = *(const u32x4*)(g + c);
    const f32x4 a = *(const f32x4*)(y + c), b = *(const f32x4*)(y + c + 4);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      d = fmaf(bf16_hi(v[e]), a[2 * e + 1], fmaf(bf16_lo(v[e]), a[2 * e], d));
      d = fmaf(bf16_hi(v[2 + e]), b[2 * e + 1], fmaf(bf16_lo(v[2 + e]), b[2 * e], d));
    }
  }
#pragma unroll
  for (int k = 32; k; k >>= 1) d += __shfl_xor(d, k);
  if (lane == 0) dw[s] = (bf16)(d / row_scale((float)weights[s]));
}

// ---- the weights' gradients: out[e] [N, K] = sum over the expert's rows of g[r, n] x[r, k] ----
// One 256 x 256 tile of one expert a workgroup, stages of 64 rows; both operands are read
// transposed out of LDS (ds_read_b64_tr_b16).  The bias's gradient is one more product, of
// ones (dW1) or the rows' weights (dW2) with the fragments of g at hand.  One of the operands
// is gathered by token.  Experts are taken by falling number of rows, so that the largest
// does not start last.
// Bound by the matrix instructions and their feeding: 32768 rows of 8 experts, 4096 x 1024, dW2 329
// and dW1 313 us (835 and 878 TFLOP/s, 41 and 44% of the cycles issue MFMAs), 298 and 276 where every
// expert has the same number of rows.
struct ExpertWgrad {
  const bf16* g;
  const bf16* x;
  const int32_t* token;
  const float* weight;  // OF_G: a row whose weight is nothing counts as zero
  const int32_t* offsets;
  bf16* out;
  bf16* bias_out;       // [E, N] or null
  float* part;          // SPLIT: [split, E, N, K], then the bias's [split, E, N]
  int64_t ldg, ldx;
  int N, K, nt, kt, experts, split;
};

constexpr int EW_BK = 64, EW_HALF = EW_BK * 512, EW_STAGE = 2 * EW_HALF;

// OF_G: g is gathered (dout), x are rows (h); else x is gathered and g are rows (gz).
// SPLIT: where the tiles are at most half as many as the CUs, an expert's rows are shared out over `split`
// workgroups, whose fp32 sums are added in order by a second launch.
template <bool OF_G, bool SPLIT>
__global__ __launch_bounds__(512, 1) void expert_wgrad_kernel(ExpertWgrad p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NW = 8, LPW = EW_HALF / 1024 / NW;
  __shared__ __attribute__((aligned(1024))) char lds[2 * EW_STAGE];
  // a stage's tokens and weights, copied three stages ahead: loads into registers would wait,
  // in order, for the copies before them
  __shared__ __attribute__((aligned(1024))) char meta[4][2][EW_BK * 4];
  const int tid = (int)__builtin_amdgcn_workitem_id_x();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n16 = lane & 15, g4 = lane >> 4;
  const int wk = wave >> 2, wn = wave & 3;  // wave tile: 128 k x 64 n
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  const int id = (int)__builtin_amdgcn_workgroup_id_x(), per = p.nt * p.kt * (SPLIT ? p.split : 1);
  int e = id / per;
  const int tile = SPLIT ? id % per / p.split : id % per, share = SPLIT ? id % per % p.split : 0;
  const int tk = tile % p.kt, tn = tile / p.kt;
  if (p.experts <= 64) {  // the e-th largest: every wave ranks the experts, one a lane
    const int n = lane < p.experts ? p.offsets[lane + 1] - p.offsets[lane] : -1;
    int before = 0;
    for (int i = 0; i < p.experts; ++i) {
      const int o = __builtin_amdgcn_readlane(n, i);
      before += o > n || (o == n && i < lane);
    }
    e = __ffsll(__ballot(lane < p.experts && before == e)) - 1;
  }
  e = __builtin_amdgcn_readfirstlane(e);
  const int k0 = tk * 256, n0 = tn * 256;
  int row0 = plan_load(p.offsets, e), rows = plan_load(p.offsets, e + 1) - row0;
  if (SPLIT) {  // whole stages
    const int chunk = ((rows + EW_BK - 1) / EW_BK + p.split - 1) / p.split * EW_BK, first = min(share * chunk, rows);
    row0 += first;
    rows = min(chunk, rows - first);
  }
  const int nk = (rows + EW_BK - 1) / EW_BK;

  uint32_t vx[LPW], vg[LPW];  // the gathered one's without the row
  int rr[LPW];
#pragma unroll
  for (int j = 0; j < LPW; ++j) {
    const int row = 2 * (j * NW + wave) + (lane >> 5), c = (lane & 31) ^ ((row & 7) << 1);
    rr[j] = row;
    vx[j] = k0 + 8 * c < p.K ? (uint32_t)((OF_G ? row * p.ldx * 2 : 0) + c * 16) : OOB;
    vg[j] = n0 + 8 * c < p.N ? (uint32_t)((OF_G ? 0 : row * p.ldg * 2) + c * 16) : OOB;
  }
  const char* xb = (const char*)(p.x + (OF_G ? (int64_t)row0 * p.ldx : 0) + k0);
  const char* gb = (const char*)(p.g + (OF_G ? 0 : (int64_t)row0 * p.ldg) + n0);
  const uint32_t ldt = (uint32_t)((OF_G ? p.ldg : p.ldx) * 2);
  const bool sums = p.bias_out && tk == 0 && wk == 0;  // uniform per wave
  const uint32_t meta_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)meta;
  auto issue_meta = [&](int kt) {  // wave 0: tokens, wave 1: weights
    const int r = kt * EW_BK + lane;
    const uint32_t vo = r < rows ? 4u * r : OOB;
    if (wave == 0) dma_dword(make_rsrc(p.token + row0, OOB), meta_base + (kt & 3) * 2 * EW_BK * 4, vo);
    if (wave == 1) dma_dword(make_rsrc(p.weight + row0, OOB), meta_base + ((kt & 3) * 2 + 1) * EW_BK * 4, vo);
  };
  uint32_t vt[LPW];  // the gathered operand's offsets of the stage issued next
  auto offsets = [&](int kt) {
#pragma unroll
    for (int j = 0; j < LPW; ++j) {
      const uint32_t vo = OF_G ? vg[j] : vx[j];
      bool in = rr[j] < rows - kt * EW_BK && vo != OOB;
      if (OF_G) in = in && !no_weight(*(const float*)(meta[kt & 3][1] + 4 * rr[j]));
      vt[j] = in ? vo + *(const uint32_t*)(meta[kt & 3][0] + 4 * rr[j]) * ldt : OOB;
    }
  };
  auto issue = [&](int kt, int slot, bool is_g) {
    const int left = rows - kt * EW_BK;
    const bool gathered = is_g == OF_G;
    const char* base = is_g ? gb : xb;
    const u32x4 r = make_rsrc(gathered ? base : base + (int64_t)kt * EW_BK * (is_g ? p.ldg : p.ldx) * 2, OOB);
    const uint32_t dst = lds_base + slot * EW_STAGE + (is_g ? EW_HALF : 0) + wave * 1024;
    if (gathered || left >= EW_BK) {
#pragma unroll
      for (int j = 0; j < LPW; ++j) dma_row16(r, dst + j * NW * 1024, gathered ? vt[j] : is_g ? vg[j] : vx[j]);
    } else {
#pragma unroll
      for (int j = 0; j < LPW; ++j) dma_row16(r, dst + j * NW * 1024, rr[j] < left ? (is_g ? vg[j] : vx[j]) : OOB);
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
  if (nk > 0) {
    issue_meta(0);
    if (nk > 1) issue_meta(1);
    if (nk > 2) issue_meta(2);
    wait_vmcnt(0);
    lds_barrier();
    offsets(0);
    issue(0, 0, OF_G);
    issue(0, 0, !OF_G);
    offsets(1);
  }
  auto stage = [&](int kt, auto with_sums) {
    wait_vmcnt(0);
    lds_barrier();  // the stage has landed for every wave; the other slot is free
    const int wr = (kt + 1) & 1;
    const bool step = kt + 1 < nk;
    if (step) issue(kt + 1, wr, OF_G);
    if (kt + 3 < nk) issue_meta(kt + 3);
    const char* st = lds + (kt & 1) * EW_STAGE;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 a[8], b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = frag(st, bo[j], kk);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = frag(st, ao[i], kk);
      if (kk == 1) offsets(kt + 2);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
      if constexpr (decltype(with_sums)::value) {
        // the bias's other operand: ones, or the weights of rows 4 g4 .. + 3 and 16 + 4 g4 .. + 3, as the fragments
        bf16x8 w8;
        const char* m = meta[kt & 3][1] + 4 * (32 * kk + 4 * g4);
        const f32x4 lo = OF_G ? *(const f32x4*)m : (f32x4){1.f, 1.f, 1.f, 1.f}, up = OF_G ? *(const f32x4*)(m + 64) : lo;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          w8[x] = (bf16)lo[x];
          w8[4 + x] = (bf16)up[x];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) bacc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w8, b[j], bacc[j], 0, 0, 0);
      }
      if (kk == 0 && step) {
        __builtin_amdgcn_sched_barrier(0);
        issue(kt + 1, wr, !OF_G);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  if (sums)
    for (int kt = 0; kt < nk; ++kt) stage(kt, std::true_type{});
  else
    for (int kt = 0; kt < nk; ++kt) stage(kt, std::false_type{});
  const int64_t of_e = SPLIT ? (int64_t)share * p.experts + e : e;
  if (sums && g4 == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 64 * wn + 16 * j + n16;
      if (n >= p.N) continue;
      if (SPLIT) p.part[(int64_t)p.split * p.experts * p.N * p.K + of_e * p.N + n] = bacc[j][0];
      else p.bias_out[of_e * p.N + n] = (bf16)bacc[j][0];
    }
  }
  if constexpr (SPLIT) {
    float* out = p.part + of_e * p.N * p.K;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 64 * wn + 16 * j + n16;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = k0 + 128 * wk + 16 * i + 4 * g4;
        if (n < p.N && k < p.K) *(f32x4*)(out + (int64_t)n * p.K + k) = acc[i][j];
      }
    }
    return;
  }
  // 16 rows n x 128 columns k at a time through this wave's 4 KiB of the ring: rows of 256 bytes out
  lds_barrier();  // every wave is done reading the last stage
  bf16* out = p.out + of_e * p.N * p.K;
  char* slab = lds + wave * 4096;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *(u32x2*)(slab + n16 * 256 + (((2 * i + (g4 >> 1)) ^ n16) << 4) + 8 * (g4 & 1)) =
          (u32x2){pack_bf16x2(acc[i][j][0], acc[i][j][1]), pack_bf16x2(acc[i][j][2], acc[i][j][3])};
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int r = 4 * it + g4, n = n0 + 64 * wn + 16 * j + r, k = k0 + 128 * wk + 8 * n16;
      const u32x4 v = *(const u32x4*)(slab + r * 256 + ((n16 ^ r) << 4));
      if (n < p.N && k < p.K) *(u32x4*)(out + (int64_t)n * p.K + k) = v;
    }
  }
#endif
}

// The shares' sums, added in order and rounded once: n elements of the weights, then nb of the bias.
__global__ __launch_bounds__(256) void expert_wgrad_sum_kernel(const float* part, bf16* out, int64_t n, bf16* bias_out, int64_t nb,
                                                               int split) {
  int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const bool bias = i >= n;
  if (bias) {
    i -= n;
    if (i >= nb) return;
    part += n * split;
    out = bias_out;
    n = nb;
  }
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < split; ++s) a += *(const f32x4*)(part + n * s + i);
  *(u32x2*)(out + i) = (u32x2){pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3])};
}

// 1: up to 16 pairs without a backward take no plan (`EX_DIRECT`); else rows of a tile.  Times of a
// whole forward replayed, us; E experts, C -> H -> C, a: pairs an expert:
//   16 (the few-rows kernel) under 4 pairs an expert without a backward (a 1, E 8, 1024 -> 4096: 36 against
//     42 with 64; a 4: 41 / 45, but E 32, 512 -> 1024 32 / 30; a 12: 50 / 47);
//   64 where the narrowest product would have fewer than 140 tiles of 128 x 128.  Over 12 families of E, k, C and H
//     (E 2 to 64, C 256 to 1024, H 384 to 4096) at 64 to 225 such tiles, forward and training, the better of the two
//     changes between 104 (E 8, 512 -> 2048) and 192 (E 64, 384 -> 384), mostly around 130 to 150, and a rule
//     loses against the better one on average 2.5% with 104, 1.1 with 128, 0.6 with 136 to 144, 0.8 with 160,
//     1.4 with 164 (E 8, 512 -> 2048: at 104 57.3 with 64 against 56.4 with 128, at 144 72.9 / 66.2; E 16, 768 ->
//     1536: at 126 50.5 / 61.1, at 162 62.4 / 56.4; E 2, 1024 -> 4096: at 112 78.8 / 80.3, at 136 105.4 / 93.5);
//   256 where an expert has two such tiles and they fill the chip (a 2048, E 8, 1024 -> 2048: 217 against
//     240 with 128; a 1024: 141 / 148; a 1024, E 32, 512 -> 1024: 150 / 154);
//   else 128, also for a few rows of many experts (a 6, E 64, 1024 -> 1024: 60 against 62 with 64).
static int expert_tile(int64_t pairs, int experts, int64_t width, bool train) {
  if (!train && pairs <= EX_DIRECT) return 1;
  if (!train && pairs < 4 * (int64_t)experts) return 16;
  if ((pairs / 128 + experts / 2) * ((width + 127) / 128) < 140) return 64;
  return pairs >= 512 * (int64_t)experts && (pairs / 256) * ((width + 255) / 256) >= 200 ? 256 : 128;
}
static int expert_tile(const strata_hip_expert_mlp_args* a) {
  return expert_tile(a->tokens * (int64_t)a->top_k, a->experts, std::min(std::min(a->dim, a->hidden), a->out_dim), a->dact != nullptr);
}

static int expert_cus() {
  static int cached[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cached[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cached[dev] = n;
  }
  return cached[dev];
}

template <int MODE, bool WT>
static int launch_expert_gemm(ExpertGemm p, int64_t pairs, int experts, int tile, hipStream_t st) {
  const int cols = tile == 1 ? 16 : tile;
  p.nt = (p.N + cols - 1) / cols;
  const int64_t mt = tile == 1 ? std::min<int64_t>(experts, pairs) : pairs / tile + std::min<int64_t>(experts, pairs), total = mt * p.nt;
  // 2^32 threads a launch (a grid of 256 x 256 tiles is not larger than the chip)
  if (total > 0x7fffffff || (tile != 256 && total * (tile <= 16 ? 1024 : tile == 64 ? 256 : 512) >= 0x100000000ll))
    return fail(STRATA_HIP_EUNSUPPORTED, "expert_mlp: problem too large for one launch");
  if constexpr (!WT && MODE != EX_HIDDEN_GRAD) {
    if (tile == 1) {
      if (p.K > 1024)
        hipLaunchKernelGGL((expert_few_kernel<MODE, 16, true>), dim3((unsigned)total), dim3(1024), 0, st, p);
      else
        hipLaunchKernelGGL((expert_few_kernel<MODE, 4, true>), dim3((unsigned)total), dim3(256), 0, st, p);
      return check_launch("expert_few_kernel");
    }
    if (tile == 16) {
      // 16 waves a workgroup for a long contraction: one token, 1024 -> 4096 24.8 us against 26.0 with 4
      // throughout (and 25.8 with 16 throughout); four tokens, 1024 -> 2048 28.5 against 27.5.
      if (p.K > 1024)
        hipLaunchKernelGGL((expert_few_kernel<MODE, 16, false>), dim3((unsigned)total), dim3(1024), 0, st, p);
      else
        hipLaunchKernelGGL((expert_few_kernel<MODE, 4, false>), dim3((unsigned)total), dim3(256), 0, st, p);
      return check_launch("expert_few_kernel");
    }
  }
  if (tile == 256) {
    p.round = expert_cus();
    hipLaunchKernelGGL((expert_gemm_kernel<256, 256, 2, 4, 2, MODE, WT, false>), dim3((unsigned)std::min<int64_t>(total, p.round)),
                       dim3(512), 0, st, p);
    if (total > p.round) {
      // The tail in 64 x 64 tiles where they are expected to fit the chip at one a CU, an expert's last tile being
      // half full on average: 16 tiles, 4096 -> 1024, 45 -> 28 us (a whole training pass 1843 -> 1810); 64 tiles
      // of 1024 -> 4096 in 64 x 64 ones: the pass 10 us slower.
      const int64_t tail = (pairs / tile + experts / 2) * p.nt % p.round;
      if (16 * tail <= p.round)
        hipLaunchKernelGGL((expert_gemm_kernel<64, 64, 2, 2, 4, MODE, WT, true>), dim3((unsigned)(p.round / 2 * 16)), dim3(256), 0, st, p);
      else
        hipLaunchKernelGGL((expert_gemm_kernel<128, 128, 4, 2, 4, MODE, WT, true>), dim3((unsigned)(p.round / 2 * 4)), dim3(512), 0, st, p);
    }
  } else if (tile == 128) {
    // A ring of four stages (one workgroup a CU) where one round of workgroups is expected, else of two
    // (two a CU): 4000 pairs, 16 experts, 768 columns of 1536 30 -> 23 us, 1536 of 768 26 against 28.
    if ((pairs / tile + experts / 2) * p.nt <= expert_cus())
      hipLaunchKernelGGL((expert_gemm_kernel<128, 128, 4, 2, 4, MODE, WT, false>), dim3((unsigned)total), dim3(512), 0, st, p);
    else
      hipLaunchKernelGGL((expert_gemm_kernel<128, 128, 4, 2, 2, MODE, WT, false>), dim3((unsigned)total), dim3(512), 0, st, p);
  }
  else
    hipLaunchKernelGGL((expert_gemm_kernel<64, 64, 2, 2, 4, MODE, WT, false>), dim3((unsigned)total), dim3(256), 0, st, p);
  return check_launch("expert_gemm_kernel");
}

// Shares of an expert's rows in its weights' gradients: as many as fill the chip, of four stages or
// more on average.  A whole forward and backward with one share / with these: 32768 tokens, 2 experts,
// 128 -> 512 887 / 172 us; 8000, 2 of 2, 512 -> 1024 534 / 250; 16000, 2 of 8, 512 -> 512 420 / 306;
// 1000, 2 of 2, 512 -> 512 110 / 100 (shares of two stages 97, of eight 110).
// CUS is the whole chip's number, not the current device's: a caller sizes the workspace by this rule, maybe
// while another device is current than the launch's.
static int wgrad_split(int64_t pairs, int experts, int N, int K) {
  constexpr int64_t CUS = 256;
  const int64_t tiles = (int64_t)experts * ((N + 255) / 256) * ((K + 255) / 256);
  return (int)std::max<int64_t>(1, std::min<int64_t>({CUS / tiles, pairs / experts / (4 * EW_BK), 32}));
}
static int64_t wgrad_space(int64_t pairs, int experts, int N, int K) {
  const int split = wgrad_split(pairs, experts, N, K);
  return split > 1 ? (int64_t)split * experts * N * (K + 1) : 0;
}

template <bool OF_G>
static int launch_wgrad(ExpertWgrad p, int64_t pairs, float* space, hipStream_t st) {
  p.nt = (p.N + 255) / 256;
  p.kt = (p.K + 255) / 256;
  p.split = wgrad_split(pairs, p.experts, p.N, p.K);
  p.part = space;
  const int64_t total = (int64_t)p.nt * p.kt * p.experts * p.split;
  if (total * 512 >= 0x100000000ll) return fail(STRATA_HIP_EUNSUPPORTED, "expert_mlp_bwd: problem too large for one launch");
  if (p.split == 1) {
    hipLaunchKernelGGL((expert_wgrad_kernel<OF_G, false>), dim3((unsigned)total), dim3(512), 0, st, p);
    return check_launch("expert_wgrad_kernel");
  }
  if (!space || ((uintptr_t)space & 15)) return fail(STRATA_HIP_EINVAL, "expert_mlp_bwd: wspace is needed, 16-byte aligned");
  hipLaunchKernelGGL((expert_wgrad_kernel<OF_G, true>), dim3((unsigned)total), dim3(512), 0, st, p);
  if (const int rc = check_launch("expert_wgrad_kernel")) return rc;
  const int64_t n = (int64_t)p.experts * p.N * p.K, nb = p.bias_out ? (int64_t)p.experts * p.N : 0;
  hipLaunchKernelGGL(expert_wgrad_sum_kernel, dim3((unsigned)((n + nb + 1023) / 1024)), dim3(256), 0, st, space, p.out, n, p.bias_out,
                     nb, p.split);
  return check_launch("expert_wgrad_sum_kernel");
}

static int launch_combine(ExpertCombine c, int64_t tokens, int width, hipStream_t st) {
  c.chunks = width / 8;
  c.n = tokens * c.chunks;
  if (c.n >= 0xffffff00ll) return fail(STRATA_HIP_EUNSUPPORTED, "expert_mlp: problem too large for one launch");
  hipLaunchKernelGGL(expert_combine_kernel, dim3((unsigned)((c.n + 255) / 256)), dim3(256), 0, st, c);
  return check_launch("expert_combine_kernel");
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
  if (pairs > 0 && a->tile != expert_tile(a)) return fail(STRATA_HIP_EINVAL, name + ": tile is not strata_hip_expert_tile()'s");
  const bool plan = a->tile != 1;
  if (!a->w1 || !a->w2 || (plan && (!a->offsets || !a->tiles))) return fail(STRATA_HIP_EINVAL, name + ": null pointer");
  if (((uintptr_t)a->w1 & 15) || ((uintptr_t)a->w2 & 15) || ((uintptr_t)a->b1 & 15) || ((uintptr_t)a->b2 & 15))
    return fail(STRATA_HIP_EINVAL, name + ": weights and biases must be 16-byte aligned");
  if (pairs == 0) return STRATA_HIP_OK;
  if (!a->dact && name != "expert_mlp") return fail(STRATA_HIP_EINVAL, name + ": dact is needed");
  if (!a->x || !a->weights || (plan && (!a->row_token || !a->row_weight)) || !a->slot_row || !a->h || !a->y)
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

extern "C" int32_t strata_hip_expert_tile(int64_t pairs, int32_t experts, int32_t dim, int32_t hidden, int32_t out_dim,
                                          int32_t train) {
  return expert_tile(pairs, experts, std::min(std::min(dim, hidden), out_dim), train != 0);
}

extern "C" int64_t strata_hip_expert_mlp_bwd_workspace(int64_t pairs, int32_t experts, int32_t dim, int32_t hidden, int32_t out_dim) {
  if (pairs <= 0 || experts <= 0 || dim <= 0 || hidden <= 0 || out_dim <= 0) return 0;
  return std::max(wgrad_space(pairs, experts, out_dim, hidden), wgrad_space(pairs, experts, hidden, dim));
}

extern "C" int strata_hip_expert_mlp(const strata_hip_expert_mlp_args* a, void* stream) {
  if (const int rc = expert_check("expert_mlp", a)) return rc;
  if (a->tokens == 0) return STRATA_HIP_OK;
  if (!a->out || ((uintptr_t)a->out & 15) || ((uintptr_t)a->residual & 15) ||
      (a->residual && (a->ldr % 8 || (a->tokens > 1 && a->ldr < a->out_dim))))
    return fail(STRATA_HIP_EINVAL, "expert_mlp: out and residual must be 16-byte aligned, row strides multiples of 8");
  hipStream_t st = (hipStream_t)stream;
  const int64_t pairs = a->tokens * (int64_t)a->top_k;
  ExpertGemm g = {};
  g.token = a->row_token;
  g.weight = a->row_weight;
  g.offsets = a->offsets;
  g.tiles = a->tiles;
  g.index = a->slot_row;
  g.weights = (const bf16*)a->weights;
  g.pairs = (int)std::min<int64_t>(pairs, EX_DIRECT);
  g.top_k = a->top_k;
  g.experts = a->experts;
  g.x = (const bf16*)a->x;
  g.ldx = a->ldx;
  g.w = (const bf16*)a->w1;
  g.bias = (const bf16*)a->b1;
  g.out = a->h;
  g.out2 = (_Float16*)a->dact;
  g.N = a->hidden;
  g.K = a->dim;
  if (const int rc = launch_expert_gemm<EX_HIDDEN, false>(g, pairs, a->experts, a->tile, st)) return rc;
  g.x = (const bf16*)a->h;
  g.ldx = a->hidden;
  g.w = (const bf16*)a->w2;
  g.bias = (const bf16*)a->b2;
  g.out = a->y;
  g.N = a->out_dim;
  g.K = a->hidden;
  if (a->tile == 1 && (pairs == 1 || (pairs <= EX_FUSED && pairs * a->hidden <= EX_FUSED_K))) {
    hipLaunchKernelGGL(expert_few_out_kernel, dim3((unsigned)(a->out_dim / EX_FUSED_N)), dim3(1024), 0, st, g, (const bf16*)a->residual,
                       a->ldr, (bf16*)a->out);
    return check_launch("expert_few_out_kernel");
  }
  if (const int rc = launch_expert_gemm<EX_OUT, false>(g, pairs, a->experts, a->tile, st)) return rc;
  ExpertCombine c = {};
  c.y = a->y;
  c.weights = (const bf16*)a->weights;
  c.slot_row = a->slot_row;
  c.residual = (const bf16*)a->residual;
  c.ldr = a->ldr;
  c.out = (bf16*)a->out;
  c.top_k = a->top_k;
  c.experts = a->tile == 1 ? a->experts : 0;
  return launch_combine(c, a->tokens, a->out_dim, st);
}

extern "C" int strata_hip_expert_mlp_bwd(const strata_hip_expert_mlp_bwd_args* b, void* stream) {
  const std::string name = "expert_mlp_bwd";
  if (!b) return fail(STRATA_HIP_EINVAL, name + ": null args");
  const strata_hip_expert_mlp_args* a = &b->fwd;
  if (const int rc = expert_check(name, a)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const int64_t pairs = a->tokens * (int64_t)a->top_k;
  const bool hid = b->dx || b->dw1;  // gradients below the hidden layer
  if (pairs > 0) {
    if (!b->dout || ((uintptr_t)b->dout & 15)) return fail(STRATA_HIP_EINVAL, name + ": dout must be given, 16-byte aligned");
    if (hid && !b->gz) return fail(STRATA_HIP_EINVAL, name + ": gz is needed for dx and dw1");
    if (b->dx && !b->dxs) return fail(STRATA_HIP_EINVAL, name + ": dxs is needed for dx");
  }
  if ((b->db2 && !b->dw2) || (b->db1 && !b->dw1)) return fail(STRATA_HIP_EINVAL, name + ": a bias gradient comes with its weight's");
  const void* all[] = {b->gz, b->dxs, b->dx, b->dw1, b->dw2, b->db1, b->db2};
  for (const void* q : all)
    if ((uintptr_t)q & 15) return fail(STRATA_HIP_EINVAL, name + ": workspaces and gradients must be 16-byte aligned");
  if (pairs > 0 && b->dweights) {
    constexpr int64_t MOST = 1ll << 25;  // pairs a launch: 2^31 threads
    for (int64_t p0 = 0; p0 < pairs; p0 += MOST) {
      hipLaunchKernelGGL(expert_dweight_kernel, dim3((unsigned)((std::min(pairs - p0, MOST) + 3) / 4)), dim3(256), 0, st,
                         (const bf16*)b->dout, a->y, (const bf16*)a->weights, a->slot_row, (bf16*)b->dweights, p0, pairs, a->top_k,
                         a->out_dim);
      if (const int rc = check_launch("expert_dweight_kernel")) return rc;
    }
  }
  ExpertWgrad w = {};
  w.token = a->row_token;
  w.weight = a->row_weight;
  w.offsets = a->offsets;
  w.experts = a->experts;
  if (b->dw2) {  // without rows: zeros
    w.g = (const bf16*)b->dout;
    w.x = (const bf16*)a->h;
    w.out = (bf16*)b->dw2;
    w.bias_out = (bf16*)b->db2;
    w.ldg = a->out_dim;
    w.ldx = a->hidden;
    w.N = a->out_dim;
    w.K = a->hidden;
    if (const int rc = launch_wgrad<true>(w, pairs, b->wspace, st)) return rc;
  }
  ExpertGemm g = {};
  g.token = a->row_token;
  g.weight = a->row_weight;
  g.offsets = a->offsets;
  g.tiles = a->tiles;
  if (hid && pairs > 0) {
    g.x = (const bf16*)b->dout;
    g.ldx = a->out_dim;
    g.w = (const bf16*)a->w2;
    g.mul = (const _Float16*)a->dact;
    g.out = b->gz;
    g.N = a->hidden;
    g.K = a->out_dim;
    if (const int rc = launch_expert_gemm<EX_HIDDEN_GRAD, true>(g, pairs, a->experts, a->tile, st)) return rc;
  }
  if (b->dw1) {
    w.g = (const bf16*)b->gz;
    w.x = (const bf16*)a->x;
    w.out = (bf16*)b->dw1;
    w.bias_out = (bf16*)b->db1;
    w.ldg = a->hidden;
    w.ldx = a->ldx;
    w.N = a->hidden;
    w.K = a->dim;
    if (const int rc = launch_wgrad<false>(w, pairs, b->wspace, st)) return rc;
  }
  if (b->dx && pairs > 0) {
    g.x = (const bf16*)b->gz;
    g.ldx = a->hidden;
    g.w = (const bf16*)a->w1;
    g.out = b->dxs;
    g.N = a->dim;
    g.K = a->hidden;
    if (const int rc = launch_expert_gemm<EX_OUT, true>(g, pairs, a->experts, a->tile, st)) return rc;
    ExpertCombine c = {};
    c.y = b->dxs;
    c.slot_row = a->slot_row;
    c.out = (bf16*)b->dx;
    c.top_k = a->top_k;
    return launch_combine(c, a->tokens, a->dim, st);
  }
  return STRATA_HIP_OK;
}
