// Routing of tokens to experts for gfx950: scores, choice and weights; their gradient;
// and the order in which the experts' products take the chosen rows.
//
//   s = softmax(l) over the experts that are not masked, or 1 / (1 + exp(-l))
//   key = s + bias (the logit itself where there is neither a bias nor a group)
//   the top_groups groups with the largest sums of their two best keys stay
//   index = the top_k largest keys left, the lower expert of two equal ones, -1 where none is left
//   w = scale * s[index] (/ sum of the chosen s)
//
// A logit or bias that is not finite masks its expert (in the softmax's sum too).
//
// Renormalised weights of chosen scores that are all small are ratios of exponentials, relative
// to the largest chosen logit m: s_i / s_j = exp(l_i - l_j) for a softmax, and for a sigmoid up to 1 + e^m.
// Below a sum of 2^-30 weights and gradient are formed so: scores themselves are denormal in 32 bits
// below a logit of -87 and 0 below -103, and 1 / sum is infinite.  Scores that are 0 in
// 64 bits too (ROUTE_ZERO_*) give weights of 0.
//
// L lanes take a token, EPL (up to 8) consecutive experts each: the best key of a lane is found in
// its registers, the token's by log2(L) exchanges, so a round of the choice costs a wave
// 3 EPL + 6 log2(L) operations for 64 / L tokens.  Bound by those operations and their latency:
// [65536, 64] fp32, 8 of 64 in 4 of 8 groups with a bias 27.2 us replayed (17 MB read in 4), its gradient 11.0
// (38 MB, 3.5 TB/s); a training router's call is then bound by the host (two launches and autograd).
//
// Keys s + bias are first compared in 32 bits.  Where two that are compared lie closer together
// than those are off by (a token in some hundred), the wave chooses again in 64 bits.
#include "route.h"

namespace strata {

struct RouteParams {
  const void* logits;
  const float* bias;
  void* weights;
  int32_t* index;
  const void* dweights;  // backward
  void* dlogits;
  int64_t tokens, ld;
  int experts, top_k, score, groups, top_groups, renormalize;
  float scale;
};

constexpr int ROUTE_MAX_K = 64;
constexpr float ROUTE_SMALL = 0x1p-30f;         // a sum of chosen scores under it is formed from the logits
constexpr float ROUTE_ZERO_SOFTMAX = -745.f;    // exp of less is 0 in 64 bits
constexpr float ROUTE_ZERO_SIGMOID = -709.75f;  // exp of minus less is infinite there

// LDS written by lanes of a wave is read by others of the same wave.
__device__ __forceinline__ void wave_sync() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// The choice of one token by its L lanes, into sel (scores) and chosen (experts) in LDS.  l: this
// lane's logits, -inf where masked.  WIDE: keys are scores + bias, else the logits.  Returns
// whether two keys (or groups) that were compared lie too close together for KEY's scores.
template <typename KEY, bool WIDE, int EPL, int L>
__device__ __forceinline__ bool route_choose(const RouteParams& p, const float (&l)[EPL], const float (&bias)[EPL], int lane,
                                             char* scratch, float* sel, int* chosen) {
  constexpr KEY NONE = -__builtin_inf();
  constexpr bool CHECK = WIDE && sizeof(KEY) == 4;
  const int e0 = lane * EPL;
  KEY key[EPL], sc[EPL];
  if (p.score == STRATA_HIP_SCORE_SOFTMAX) {
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < EPL; ++i) top = fmaxf(top, l[i]);
    top = group_max<L>(top);
    KEY sum = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      sc[i] = l[i] > -__builtin_inff() ? exp_of((KEY)l[i] - (KEY)top) : (KEY)0;
      sum += sc[i];
    }
    sum = group_sum<L>(sum);
    if (sizeof(KEY) == 8) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) sc[i] = sum > 0 ? sc[i] / sum : (KEY)0;
    } else {
      const KEY r = sum > 0 ? (KEY)1 / sum : (KEY)0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) sc[i] *= r;
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) sc[i] = l[i] > -__builtin_inff() ? (KEY)1 / ((KEY)1 + exp_of(-(KEY)l[i])) : (KEY)0;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) key[i] = l[i] > -__builtin_inff() ? (WIDE ? sc[i] + (KEY)bias[i] : (KEY)l[i]) : NONE;
  bool close = false;
  // What two 32-bit keys have to be apart, in units of 1 + |key|.  With u = 6e-8 an exponential is within 2 u,
  // a sigmoid within 3.5 u, a softmax score within 16 u (its sum has 13 roundings: 8 scores a lane at most,
  // exchanged by 64 lanes at most) and a sum with the bias u further: 2 x 4.5 u and 2 x 17 u, with a margin of 2.
  // Groups' sums of two keys: twice that.
  const float apart = p.score == STRATA_HIP_SCORE_SOFTMAX ? 4e-6f : 1e-6f;
  auto near = [&](KEY a, KEY b) { return CHECK && fabsf((float)(a - b)) <= apart * (1.f + fabsf((float)a)); };
  if (WIDE && p.groups > 1) {
    KEY* keys = (KEY*)scratch;
    KEY* rank = keys + EPL * L;
    int* stays = (int*)(rank + p.groups);
    const int per = p.experts / p.groups;
#pragma unroll
    for (int i = 0; i < EPL; ++i) keys[e0 + i] = key[i];
    wave_sync();
    for (int g = lane; g < p.groups; g += L) {
      KEY a = NONE, b = NONE;
      for (int i = 0; i < per; ++i) {
        const KEY k = keys[g * per + i];
        b = k > b ? (k > a ? a : k) : b;
        a = k > a ? k : a;
      }
      rank[g] = b > NONE ? a + b : a;
    }
    wave_sync();
    for (int g = lane; g < p.groups; g += L) {  // a group stays if fewer than top_groups come before it
      const KEY mine = rank[g];
      int before = 0, sure = 0, may = 0;
      const float room = 2.f * apart * (1.f + fabsf((float)mine));
      for (int j = 0; j < p.groups; ++j) {
        const KEY o = rank[j];
        before += o > mine || (o == mine && j < g);
        if (CHECK && j != g) {
          sure += o > mine + room;
          may += o >= mine - room;
        }
      }
      stays[g] = before < p.top_groups;
      if (CHECK && mine > NONE) close |= (sure < p.top_groups) != (may < p.top_groups);
    }
    wave_sync();
    int g = e0 / per, in = e0 - g * per;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      if (e0 + i < p.experts && !stays[g]) key[i] = NONE;
      if (++in == per) {
        in = 0;
        ++g;
      }
    }
  }
  KEY last = NONE;
  const int rounds = p.top_k + (CHECK && p.top_k < p.experts ? 1 : 0);  // the first one left out is compared too
  for (int s = 0; s < rounds; ++s) {
    KEY best = NONE;
    KEY bs = 0;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (key[i] > best) {
        best = key[i];
        bs = sc[i];
        at = e0 + i;
      }
    const int own = at;
    butterfly<L>([&](auto d) {
      const KEY o = swap_lane<decltype(d)::value>(best);
      const int oa = swap_lane<decltype(d)::value>(at);
      if (o > best || (o == best && oa < at)) {
        best = o;
        at = oa;
      }
    });
    const bool some = best > NONE;
    if (CHECK && s > 0 && some) close |= near(last, best);
    last = best;
    if (s == p.top_k) break;
    if (some ? own == at : lane == 0) {  // the chosen expert's lane
      sel[s] = some ? (float)bs : 0.f;
      chosen[s] = some ? at : -1;
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (e0 + i == at) key[i] = NONE;
  }
  return close;
}

template <typename T, bool WIDE, bool VEC, int EPL, int L>
__global__ __launch_bounds__(256) void route_kernel(RouteParams p) {
  constexpr int TOK = 256 / L;
  extern __shared__ char smem[];  // a token: [top_k] scores, [top_k] experts; with groups the choice's scratch
  const int tid = threadIdx.x, lane = tid % L, tok = tid / L;
  const int64_t t = (int64_t)blockIdx.x * TOK + tok;
  const bool live = t < p.tokens;  // the other lanes of a wave follow with masked logits
  const int E = p.experts, e0 = lane * EPL, left = live ? max(E - e0, 0) : 0;
  float l[EPL], bias[EPL];
  route_row<T, EPL, VEC>(p.logits, t * p.ld + e0, left, __builtin_inff(), l);
#pragma unroll
  for (int i = 0; i < EPL; ++i) bias[i] = 0.f;
  if (WIDE && p.bias) route_row<float, EPL, VEC>(p.bias, e0, left, 0.f, bias);
#pragma unroll
  for (int i = 0; i < EPL; ++i) l[i] = is_finite(l[i]) && is_finite(bias[i]) ? l[i] : -__builtin_inff();
  float* sel = (float*)smem + tok * 2 * p.top_k;
  int* chosen = (int*)sel + p.top_k;
  const size_t fixed = ((size_t)TOK * p.top_k * 8 + 15) & ~(size_t)15;
  char* scratch = smem + fixed + (size_t)tok * (EPL * L + 2 * p.groups) * 8;
  const bool close = route_choose<float, WIDE, EPL, L>(p, l, bias, lane, scratch, sel, chosen);
  if constexpr (WIDE) {
    if (__any(close)) {
      wave_sync();
      route_choose<double, WIDE, EPL, L>(p, l, bias, lane, scratch, sel, chosen);
    }
  }
  wave_sync();
  if (!live) return;
  float total = 0.f;
  for (int s = 0; s < p.top_k; ++s) total += sel[s];
  if (p.renormalize && total < ROUTE_SMALL) {  // the same for a token's lanes
    auto logit = [&](int s) { return chosen[s] >= 0 ? route_load<T>(p.logits, t * p.ld + chosen[s]) : -__builtin_inff(); };
    float m = -__builtin_inff(), top = 0.f, sum = 0.f;
#pragma unroll 1
    for (int s = 0; s < p.top_k; ++s) m = fmaxf(m, logit(s));
    if (p.score == STRATA_HIP_SCORE_SOFTMAX) {
      top = -__builtin_inff();
#pragma unroll 1
      for (int e = lane; e < E; e += L) {
        const float x = route_load<T>(p.logits, t * p.ld + e);
        if (is_finite(x) && !(WIDE && p.bias && !is_finite(p.bias[e]))) top = fmaxf(top, x);
      }
      top = group_max<L>(top);
    }
    if (m - top >= (p.score == STRATA_HIP_SCORE_SOFTMAX ? ROUTE_ZERO_SOFTMAX : ROUTE_ZERO_SIGMOID)) {  // not with nothing chosen
#pragma unroll 1
      for (int s = 0; s < p.top_k; ++s) sum += expf(logit(s) - m);
      const float f = p.scale / sum;
#pragma unroll 1
      for (int s = lane; s < p.top_k; s += L) {
        route_store<T>(p.weights, t * p.top_k + s, expf(logit(s) - m) * f);
        p.index[t * p.top_k + s] = chosen[s];
      }
      return;
    }
  }
  const float f = p.renormalize ? p.scale / (total > 0.f ? total : 1.f) : p.scale;
  for (int s = lane; s < p.top_k; s += L) {
    route_store<T>(p.weights, t * p.top_k + s, sel[s] * f);
    p.index[t * p.top_k + s] = chosen[s];
  }
}

// The gradient at the logits.  With c the scale, S the sum of the chosen scores and a the
// sum of dw s over them:  ds = c dw, or c / S (dw - a / S) renormalised;
// softmax: dl = s (ds - sum of s ds), the sum zero when renormalised; sigmoid: dl = ds s (1 - s).
// The chosen slots' dw reach their experts' lanes through a row of LDS; renormalised, less the first
// slot's (a common part of them changes nothing): one chosen expert, or equal dw, would leave the
// roundings of dw in the place of a gradient of zero.
template <typename T, bool VEC, int EPL, int L>
__global__ __launch_bounds__(256) void route_bwd_kernel(RouteParams p) {
  constexpr int TOK = 256 / L;
  constexpr uint32_t FREE = 0x7fc0beefu;  // not chosen: no product makes these bits
  extern __shared__ char smem[];           // [TOK][EPL * L] dw by expert
  const int tid = threadIdx.x, lane = tid % L, tok = tid / L;
  const int64_t t = (int64_t)blockIdx.x * TOK + tok;
  const bool live = t < p.tokens;
  const int E = p.experts, e0 = lane * EPL, left = live ? max(E - e0, 0) : 0;
  float* row = (float*)smem + tok * (EPL * L);
  float l[EPL], bias[EPL], sc[EPL], om[EPL], dw[EPL];  // om: 1 - s of the sigmoid
  route_row<T, EPL, VEC>(p.logits, t * p.ld + e0, left, __builtin_inff(), l);
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    bias[i] = 0.f;
    row[e0 + i] = __uint_as_float(FREE);
  }
  if (p.bias) route_row<float, EPL, VEC>(p.bias, e0, left, 0.f, bias);
  wave_sync();
  if (live) {
    const int first = p.index[t * p.top_k];
    const float common = p.renormalize && first >= 0 && first < E ? route_load<T>(p.dweights, t * p.top_k) : 0.f;
    for (int s = lane; s < p.top_k; s += L) {
      const int at = p.index[t * p.top_k + s];
      if (at >= 0 && at < E) row[at] = route_load<T>(p.dweights, t * p.top_k + s) - common;
    }
  }
  const float NONE = -__builtin_inff();
  float top = NONE;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    l[i] = is_finite(l[i]) && is_finite(bias[i]) ? l[i] : NONE;
    top = fmaxf(top, l[i]);
  }
  if (p.score == STRATA_HIP_SCORE_SOFTMAX) {
    top = group_max<L>(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      sc[i] = l[i] > NONE ? expf(l[i] - top) : 0.f;
      om[i] = 0.f;
      sum += sc[i];
    }
    sum = group_sum<L>(sum);
    const float r = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sc[i] *= r;
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float x = expf(-fabsf(l[i]));  // in (0, 1]
      const float a = 1.f / (1.f + x), b = x * a;
      sc[i] = l[i] > NONE ? (l[i] >= 0.f ? a : b) : 0.f;
      om[i] = l[i] >= 0.f ? b : a;
    }
  }
  wave_sync();
  float S = 0.f, a = 0.f;
  bool chosen[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    dw[i] = row[e0 + i];
    chosen[i] = __float_as_uint(dw[i]) != FREE;
    S += chosen[i] ? sc[i] : 0.f;
    a = chosen[i] ? fmaf(dw[i], sc[i], a) : a;
  }
  S = group_sum<L>(S);
  a = group_sum<L>(a);
  if (p.renormalize && S < ROUTE_SMALL) {  // the same for a token's lanes: ratios in the place of scores
    const bool softmax = p.score == STRATA_HIP_SCORE_SOFTMAX;
    float m = NONE;
#pragma unroll
    for (int i = 0; i < EPL; ++i) m = chosen[i] ? fmaxf(m, l[i]) : m;
    m = group_max<L>(m);
    if (m - (softmax ? top : 0.f) >= (softmax ? ROUTE_ZERO_SOFTMAX : ROUTE_ZERO_SIGMOID)) {
      S = 0.f;
      a = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (chosen[i]) {
          sc[i] = expf(l[i] - m);
          S += sc[i];
          a = fmaf(dw[i], sc[i], a);
        }
      S = group_sum<L>(S);
      a = group_sum<L>(a);
    }
  }
  const bool norm = p.renormalize && S > 0.f;
  const float c = norm ? p.scale / S : p.scale, mean = norm ? a / S : 0.f;
  const float back = p.renormalize ? 0.f : p.scale * a;
  if (!live) return;
  float dl[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const float ds = chosen[i] ? c * (dw[i] - mean) : 0.f;
    dl[i] = l[i] > NONE ? (p.score == STRATA_HIP_SCORE_SOFTMAX ? sc[i] * (ds - back) : ds * sc[i] * om[i]) : 0.f;
  }
  if constexpr (VEC && EPL >= 4) {
    if (left >= EPL) {
#pragma unroll
      for (int k = 0; k < EPL / 4; ++k) {
        if constexpr (sizeof(T) == 4)
          *(f32x4*)((float*)p.dlogits + t * E + e0 + 4 * k) = (f32x4){dl[4 * k], dl[4 * k + 1], dl[4 * k + 2], dl[4 * k + 3]};
        else
          *(u32x2*)((bf16*)p.dlogits + t * E + e0 + 4 * k) =
              (u32x2){pack_bf16x2(dl[4 * k], dl[4 * k + 1]), pack_bf16x2(dl[4 * k + 2], dl[4 * k + 3])};
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (i < left) route_store<T>(p.dlogits, t * E + e0 + i, dl[i]);
}

// ---------------------------------------------------------------------------
// The plan: the chosen (token, slot) pairs in the order of their experts, pairs of one
// expert in their own order, by a counting sort whose result depends on nothing else.
//   row_token[r], row_weight[r]  the token and the weight of row r's pair
//   slot_row[s]  the row of pair s, -1 where its index names no expert
//   offsets[e]   the first row of expert e; offsets[E] the number of rows
//   tiles        [n, then n pairs (expert, first row)]: `tile` rows of one expert each
// Pairs are taken PLAN_N at a time: counted per block, the blocks' counts summed, and placed by
// block, wave and lane (the lanes of a wave that name the same expert find each other by one
// ballot per bit of the expert's number).  Bound by latency: 2 pairs 4.3 us in one launch, 4050
// of 24 experts 2 + 6, 65536 of 8 5 + 10 in two (three launches, the sums in one of their own: 23).
// ---------------------------------------------------------------------------
constexpr int PLAN_N = 1024, PLAN_WAVES = PLAN_N / 64, PLAN_MAX_E = ROUTE_MAX_E;

struct PlanParams {
  const int32_t* index;
  const bf16* weights;
  int32_t* row_token;
  float* row_weight;
  int32_t* slot_row;
  int32_t* offsets;
  int32_t* tiles;
  int32_t* counts;  // [blocks][E]
  int64_t n;        // pairs
  int experts, top_k, tile, bits, blocks;
};

__device__ __forceinline__ int plan_expert(const PlanParams& p, int64_t s) {
  const int e = s < p.n ? p.index[s] : -1;
  return e >= 0 && e < p.experts ? e : -1;
}

__global__ __launch_bounds__(PLAN_N) void plan_count_kernel(PlanParams p) {
  __shared__ int cnt[PLAN_MAX_E];
  const int tid = threadIdx.x;
  for (int e = tid; e < p.experts; e += PLAN_N) cnt[e] = 0;
  __syncthreads();
  const int e = plan_expert(p, (int64_t)blockIdx.x * PLAN_N + tid);
  if (e >= 0) atomicAdd(&cnt[e], 1);
  __syncthreads();
  for (int i = tid; i < p.experts; i += PLAN_N) p.counts[(int64_t)blockIdx.x * p.experts + i] = cnt[i];
}

// Every expert's first row, into total[e], from its number of rows there (both in LDS); `write`:
// also the plan's offsets and tiles.
__device__ __forceinline__ void plan_offsets(const PlanParams& p, int* total, int tid, bool write) {
  __shared__ int row0[PLAN_MAX_E + 1], tile0[PLAN_MAX_E + 1];
  if (tid < 64) {  // one wave scans, 8 experts a lane
    constexpr int PER = PLAN_MAX_E / 64;
    int r[PER], t[PER], rs = 0, ts = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = tid * PER + i, n = e < p.experts ? total[e] : 0;
      r[i] = rs;
      t[i] = ts;
      rs += n;
      ts += (n + p.tile - 1) / p.tile;
    }
    int ra = rs, ta = ts;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int a = __shfl_up(ra, d), b = __shfl_up(ta, d);
      if (tid >= d) {
        ra += a;
        ta += b;
      }
    }
    ra -= rs;
    ta -= ts;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      row0[tid * PER + i] = ra + r[i];
      tile0[tid * PER + i] = ta + t[i];
    }
    if (tid == 63) {
      row0[PLAN_MAX_E] = ra + rs;
      tile0[PLAN_MAX_E] = ta + ts;
    }
  }
  __syncthreads();
  for (int e = tid; e < p.experts; e += PLAN_N) total[e] = row0[e];
  if (write) {
    for (int e = tid; e < p.experts; e += PLAN_N) p.offsets[e] = row0[e];
    const int tiles = tile0[PLAN_MAX_E];
    for (int i = tid; i < tiles; i += PLAN_N) {  // the last expert whose tiles start at or before i
      int lo = 0, hi = p.experts - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tile0[mid] <= i) lo = mid;
        else hi = mid - 1;
      }
      p.tiles[1 + 2 * i] = lo;
      p.tiles[2 + 2 * i] = row0[lo] + (i - tile0[lo]) * p.tile;
    }
    if (tid == 0) {
      p.offsets[p.experts] = row0[PLAN_MAX_E];
      p.tiles[0] = tiles;
    }
  }
  __syncthreads();
}

// Sums over the blocks' counts of expert tid % w (w: experts rounded up to a power of two), by
// PLAN_N / w threads an expert: all of them into total[e] (LDS), those before this thread's run
// of blocks, or before block `mine`, returned.
__device__ __forceinline__ int plan_sum(const PlanParams& p, int* total, int* part, int w, int b0, int b1, int mine) {
  const int tid = threadIdx.x, seg = PLAN_N / w, e = tid % w, g = tid / w;
  int s = 0, m = 0;
  if (e < p.experts) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) {
      const int v = p.counts[(int64_t)b * p.experts + e];
      s += v;
      m += b < mine ? v : 0;
    }
  }
  part[tid] = s;
  part[PLAN_N + tid] = m;
  __syncthreads();
  int before = 0, all = 0, mm = 0;
  const int per = (p.blocks + seg - 1) / seg, used = (p.blocks + per - 1) / per;  // runs that hold blocks
  for (int k = 0; k < used; ++k) {
    const int v = part[k * w + e];
    before += k < g ? v : 0;
    all += v;
    mm += part[PLAN_N + k * w + e];
  }
  if (e < p.experts && g == 0) total[e] = all;
  __syncthreads();
  return mine >= 0 ? mm : before;
}

// The blocks' counts become each block's first row of each expert.
__global__ __launch_bounds__(PLAN_N) void plan_scan_kernel(PlanParams p) {
  __shared__ int total[PLAN_MAX_E], part[2 * PLAN_N];
  const int tid = threadIdx.x, E = p.experts, w = 1 << p.bits, e = tid % w, g = tid / w;
  const int per = (p.blocks + PLAN_N / w - 1) / (PLAN_N / w), b0 = min(g * per, p.blocks), b1 = min(b0 + per, p.blocks);
  const int before = plan_sum(p, total, part, w, b0, b1, -1);
  plan_offsets(p, total, tid, true);
  if (e < E) {
    int at = total[e] + before;
    for (int b = b0; b < b1; ++b) {
      int32_t* c = p.counts + (int64_t)b * E + e;
      const int v = *c;
      *c = at;
      at += v;
    }
  }
}

// ONE: the whole plan in one block.  SUMS: every block sums the counts of the blocks before it
// itself (the first also writes offsets and tiles), in the place of a launch of plan_scan_kernel.
template <bool ONE, bool SUMS>
__global__ __launch_bounds__(PLAN_N) void plan_place_kernel(PlanParams p) {
  extern __shared__ int cnt[];  // [PLAN_WAVES][E] counts, then first rows; + [E] totals
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, E = p.experts;
  int* total = cnt + PLAN_WAVES * E;
  for (int i = tid; i < PLAN_WAVES * E; i += PLAN_N) cnt[i] = 0;
  __syncthreads();
  const int64_t s = (int64_t)blockIdx.x * PLAN_N + tid;
  const int e = plan_expert(p, s);
  uint64_t same = __ballot(e >= 0);
  for (int b = 0; b < p.bits; ++b) {
    const uint64_t m = __ballot((e >> b) & 1);
    same &= ((e >> b) & 1) ? m : ~m;
  }
  const int rank = __popcll(same & ((1ull << lane) - 1));
  if (e >= 0 && rank == 0) cnt[wave * E + e] = __popcll(same);
  __syncthreads();
  if (ONE) {
    for (int i = tid; i < E; i += PLAN_N) {
      int n = 0;
      for (int w = 0; w < PLAN_WAVES; ++w) n += cnt[w * E + i];
      total[i] = n;
    }
    __syncthreads();
    plan_offsets(p, total, tid, true);
  }
  if (SUMS) {
    __shared__ int part[2 * PLAN_N];
    const int w = 1 << p.bits, g = tid / w, per = (p.blocks + PLAN_N / w - 1) / (PLAN_N / w);
    const int b0 = min(g * per, p.blocks), before = plan_sum(p, total, part, w, b0, min(b0 + per, p.blocks), blockIdx.x);
    plan_offsets(p, total, tid, blockIdx.x == 0);
    if (g == 0 && tid < E) total[tid] += before;
    __syncthreads();
  }
  for (int i = tid; i < E; i += PLAN_N) {
    int at = ONE || SUMS ? total[i] : p.counts[(int64_t)blockIdx.x * E + i];
    for (int w = 0; w < PLAN_WAVES; ++w) {
      const int n = cnt[w * E + i];
      cnt[w * E + i] = at;
      at += n;
    }
  }
  __syncthreads();
  if (s < p.n) {
    const int r = e >= 0 ? cnt[wave * E + e] + rank : -1;
    p.slot_row[s] = r;
    if (r >= 0) {
      p.row_token[r] = (int32_t)s / p.top_k;
      p.row_weight[r] = (float)p.weights[s];
    }
  }
}

// f(experts a lane, lanes a token).
template <typename F>
static int route_width(int experts, F f) {
  using std::integral_constant;
  if (experts <= 8) return f(integral_constant<int, 1>{}, integral_constant<int, 8>{});
  if (experts <= 16) return f(integral_constant<int, 2>{}, integral_constant<int, 8>{});
  if (experts <= 32) return f(integral_constant<int, 4>{}, integral_constant<int, 8>{});
  if (experts <= 64) return f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
  if (experts <= 128) return f(integral_constant<int, 8>{}, integral_constant<int, 16>{});
  if (experts <= 256) return f(integral_constant<int, 8>{}, integral_constant<int, 32>{});
  return f(integral_constant<int, 8>{}, integral_constant<int, 64>{});
}

// Rows of whole 16-byte runs: logits and bias aligned, experts a multiple of 4 (a lane's run of experts
// is then whole or, the last one of 8, read one by one).
static bool route_aligned(const strata_hip_expert_route_args* a, const float* bias) {
  return a->experts % 4 == 0 && ((uintptr_t)a->logits & 15) == 0 && ((uintptr_t)bias & 15) == 0;
}

static int route_params(const char* name, const strata_hip_expert_route_args* a, RouteParams& p) {
  const std::string n(name);
  if (!a) return fail(STRATA_HIP_EINVAL, n + ": null args");
  if (a->tokens < 0 || a->experts <= 0 || a->top_k <= 0) return fail(STRATA_HIP_EINVAL, n + ": bad tokens, experts or top_k");
  if (a->dtype != STRATA_HIP_F32 && a->dtype != STRATA_HIP_BF16) return fail(STRATA_HIP_EINVAL, n + ": bad dtype");
  if (a->score != STRATA_HIP_SCORE_SOFTMAX && a->score != STRATA_HIP_SCORE_SIGMOID) return fail(STRATA_HIP_EINVAL, n + ": bad score");
  if (a->experts > PLAN_MAX_E || a->top_k > ROUTE_MAX_K)
    return fail(STRATA_HIP_EUNSUPPORTED, n + ": at most 512 experts and top_k 64");
  if (a->groups < 1 || a->experts % a->groups || a->top_groups < 1 || a->top_groups > a->groups)
    return fail(STRATA_HIP_EINVAL, n + ": groups must divide the experts and top_groups lie in 1 .. groups");
  if (a->top_k > a->experts / a->groups * a->top_groups)
    return fail(STRATA_HIP_EINVAL, n + ": top_k exceeds the experts that may be chosen");
  if (a->tokens > 1 && a->ld < a->experts) return fail(STRATA_HIP_EINVAL, n + ": row stride smaller than the row");
  if (!(fabsf(a->scale) < __builtin_inff())) return fail(STRATA_HIP_EINVAL, n + ": scale must be finite");
  if (a->tokens * (int64_t)a->top_k > 0x7fffffff) return fail(STRATA_HIP_EUNSUPPORTED, n + ": more than 2^31 - 1 chosen pairs");
  p = {};
  p.logits = a->logits;
  p.bias = a->bias;
  p.weights = a->weights;
  p.index = a->index;
  p.dweights = a->dweights;
  p.dlogits = a->dlogits;
  p.tokens = a->tokens;
  p.ld = a->tokens > 1 ? a->ld : a->experts;
  p.experts = a->experts;
  p.top_k = a->top_k;
  p.score = a->score;
  p.groups = a->groups;
  p.top_groups = a->top_groups;
  p.renormalize = a->renormalize;
  p.scale = a->scale;
  return STRATA_HIP_OK;
}

}  // namespace strata

extern "C" int strata_hip_expert_route(const strata_hip_expert_route_args* a, void* stream) {
  using namespace strata;
  RouteParams p;
  if (const int rc = route_params("expert_route", a, p)) return rc;
  if (p.tokens == 0) return STRATA_HIP_OK;
  if (!p.logits || !p.weights || !p.index) return fail(STRATA_HIP_EINVAL, "expert_route: null pointer");
  const bool wide = p.bias || p.groups > 1, vec = route_aligned(a, p.bias) && (p.ld % 4) == 0;
  return route_width(p.experts, [&](auto epl, auto l) {
    constexpr int EPL = decltype(epl)::value, L = decltype(l)::value;
    constexpr int TOK = 256 / L;
    // At most 64 KiB: with E experts rounded up to EPL * L and no more groups or slots than experts, 2048 EPL (3 E + min(E, 64)) / E.
    const size_t smem = (((size_t)TOK * p.top_k * 8 + 15) & ~(size_t)15) + (p.groups > 1 ? (size_t)TOK * (EPL * L + 2 * p.groups) * 8 : 0);
    const int64_t wgs = (p.tokens + TOK - 1) / TOK;
    if (smem > 65536 || wgs * 256 >= 0x100000000ll)
      return fail(STRATA_HIP_EUNSUPPORTED, "expert_route: problem too large for one launch");
    const dim3 grid((unsigned)wgs);
    auto go = [&](auto t, auto w, auto v) {
      hipLaunchKernelGGL((route_kernel<decltype(t), decltype(w)::value, decltype(v)::value, EPL, L>), grid, dim3(256), smem,
                         (hipStream_t)stream, p);
    };
    auto with = [&](auto t, auto w) {
      if (vec) go(t, w, std::true_type{});
      else go(t, w, std::false_type{});
    };
    if (a->dtype == STRATA_HIP_F32) {
      if (wide) with(0.f, std::true_type{});
      else with(0.f, std::false_type{});
    } else {
      if (wide) with((bf16)0.f, std::true_type{});
      else with((bf16)0.f, std::false_type{});
    }
    return check_launch("expert_route");
  });
}

extern "C" int strata_hip_expert_route_bwd(const strata_hip_expert_route_args* a, void* stream) {
  using namespace strata;
  RouteParams p;
  if (const int rc = route_params("expert_route_bwd", a, p)) return rc;
  if (p.tokens == 0) return STRATA_HIP_OK;
  if (!p.logits || !p.dweights || !p.index || !p.dlogits) return fail(STRATA_HIP_EINVAL, "expert_route_bwd: null pointer");
  const bool vec = route_aligned(a, p.bias) && (p.ld % 4) == 0 && ((uintptr_t)p.dlogits & 15) == 0;
  return route_width(p.experts, [&](auto epl, auto l) {
    constexpr int EPL = decltype(epl)::value, L = decltype(l)::value, TOK = 256 / L;
    const int64_t wgs = (p.tokens + TOK - 1) / TOK;
    if (wgs * 256 >= 0x100000000ll) return fail(STRATA_HIP_EUNSUPPORTED, "expert_route_bwd: problem too large for one launch");
    const dim3 grid((unsigned)wgs);
    auto go = [&](auto t, auto v) {
      hipLaunchKernelGGL((route_bwd_kernel<decltype(t), decltype(v)::value, EPL, L>), grid, dim3(256), (size_t)TOK * EPL * L * 4,
                         (hipStream_t)stream, p);
    };
    auto with = [&](auto t) {
      if (vec) go(t, std::true_type{});
      else go(t, std::false_type{});
    };
    if (a->dtype == STRATA_HIP_F32) with(0.f);
    else with((bf16)0.f);
    return check_launch("expert_route_bwd");
  });
}

extern "C" int64_t strata_hip_expert_plan_workspace(int64_t pairs, int32_t experts) {
  if (pairs <= strata::PLAN_N || experts <= 0) return 0;
  return (pairs + strata::PLAN_N - 1) / strata::PLAN_N * experts;
}

extern "C" int strata_hip_expert_plan(const strata_hip_expert_plan_args* a, void* stream) {
  using namespace strata;
  if (!a) return fail(STRATA_HIP_EINVAL, "expert_plan: null args");
  if (a->pairs < 0 || a->experts <= 0 || a->tile <= 0 || a->top_k <= 0 || a->pairs % a->top_k)
    return fail(STRATA_HIP_EINVAL, "expert_plan: bad sizes");
  if (a->experts > PLAN_MAX_E) return fail(STRATA_HIP_EUNSUPPORTED, "expert_plan: at most 512 experts");
  if (a->pairs > 0x7ffffff0) return fail(STRATA_HIP_EUNSUPPORTED, "expert_plan: too many pairs");
  if (!a->offsets || !a->tiles || (a->pairs > 0 && (!a->index || !a->weights || !a->row_token || !a->row_weight || !a->slot_row)))
    return fail(STRATA_HIP_EINVAL, "expert_plan: null pointer");
  PlanParams p;
  p.index = a->index;
  p.weights = (const bf16*)a->weights;
  p.row_token = a->row_token;
  p.row_weight = a->row_weight;
  p.top_k = a->top_k;
  p.slot_row = a->slot_row;
  p.offsets = a->offsets;
  p.tiles = a->tiles;
  p.counts = a->workspace;
  p.n = a->pairs;
  p.experts = a->experts;
  p.tile = a->tile;
  p.bits = 0;
  while ((1 << p.bits) < a->experts) ++p.bits;
  p.blocks = (int)((a->pairs + PLAN_N - 1) / PLAN_N);
  hipStream_t st = (hipStream_t)stream;
  const size_t smem = (size_t)(PLAN_WAVES + 1) * a->experts * 4;
  if (p.blocks <= 1) {
    hipLaunchKernelGGL((plan_place_kernel<true, false>), dim3(1), dim3(PLAN_N), smem, st, p);
    return check_launch("expert_plan");
  }
  if (!a->workspace) return fail(STRATA_HIP_EINVAL, "expert_plan: null workspace");
  hipLaunchKernelGGL(plan_count_kernel, dim3((unsigned)p.blocks), dim3(PLAN_N), 0, st, p);
  // Up to 32768 counts every block sums them itself; beyond, that reading (the counts times the
  // blocks) costs more than the launch of one workgroup that sums them once.
  if ((int64_t)p.blocks * p.experts <= 32768) {
    hipLaunchKernelGGL((plan_place_kernel<false, true>), dim3((unsigned)p.blocks), dim3(PLAN_N), smem, st, p);
  } else {
    hipLaunchKernelGGL(plan_scan_kernel, dim3(1), dim3(PLAN_N), 0, st, p);
    hipLaunchKernelGGL((plan_place_kernel<false, false>), dim3((unsigned)p.blocks), dim3(PLAN_N), smem, st, p);
  }
  return check_launch("expert_plan");
}
