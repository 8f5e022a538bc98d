// Routing of tokens to experts for gfx950: scores, choice and weights; their gradient;
// and the order in which the experts' products take the chosen rows.
//
//   s = softmax(l) over the experts that are not masked, or 1 / (1 + exp(-l))
//   key = s + bias (the logit itself where there is neither a bias nor a group)
//   the top_groups groups with the largest sums of their two best keys stay
//   index = the top_k largest keys left, the lower expert of two equal ones, -1 where none is left
//   w = scale * s[index] (/ sum of the chosen s)
//
// A logit or bias that is not finite masks its expert.  Two keys s + bias of one token lie
// closer together than 32-bit scores resolve in about one token of 1e5, so scores that
// decide are held in 64 bits (v_fma_f64 issues at the rate of v_fma_f32 here).
//
// L lanes take a token, EPL consecutive experts each: the best key of a lane is found in
// its registers, the token's by log2(L) exchanges, so a round of the choice costs a wave
// EPL + 3 log2(L) operations for 64 / L tokens.
#include "common.h"

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

template <typename T>
__device__ __forceinline__ float route_load(const void* p, int64_t i) {
  return (float)((const T*)p)[i];
}
template <typename T>
__device__ __forceinline__ void route_store(void* p, int64_t i, float v) {
  ((T*)p)[i] = (T)v;
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < __builtin_inff(); }

template <int L, typename V>
__device__ __forceinline__ V group_max(V v) {
#pragma unroll
  for (int d = 1; d < L; d <<= 1) {
    const V o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}
template <int L, typename V>
__device__ __forceinline__ V group_sum(V v) {
#pragma unroll
  for (int d = 1; d < L; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// KEY: the type that scores and keys are held in, double where they decide.
template <typename T, typename KEY, int EPL, int L>
__global__ __launch_bounds__(256) void route_kernel(RouteParams p) {
  constexpr int TOK = 256 / L;
  constexpr KEY NONE = -__builtin_inf();
  extern __shared__ char smem[];  // [TOK][top_k] scores; with groups [TOK][EPL * L] keys and [TOK][groups] sums before them
  const int tid = threadIdx.x, lane = tid % L, tok = tid / L;
  const int64_t t = (int64_t)blockIdx.x * TOK + tok;
  const bool live = t < p.tokens;  // the other lanes of a wave wait for nobody: they follow with masked keys
  const int E = p.experts, e0 = lane * EPL;
  KEY key[EPL];
  KEY sc[EPL];
  KEY top = NONE;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const bool in = live && e0 + i < E;
    float l = in ? route_load<T>(p.logits, t * p.ld + e0 + i) : __builtin_inff();
    if (in && p.bias && !is_finite(p.bias[e0 + i])) l = __builtin_inff();
    key[i] = is_finite(l) ? (KEY)l : NONE;
    top = key[i] > top ? key[i] : top;
  }
  if (p.score == STRATA_HIP_SCORE_SOFTMAX) {
    top = group_max<L>(top);
    KEY sum = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      sc[i] = key[i] > NONE ? exp_of(key[i] - top) : (KEY)0;
      sum += sc[i];
    }
    sum = group_sum<L>(sum);
    const KEY r = sum > 0 ? (KEY)1 / sum : (KEY)0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sc[i] = sizeof(KEY) == 8 ? (sum > 0 ? sc[i] / sum : (KEY)0) : sc[i] * r;
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) sc[i] = key[i] > NONE ? (KEY)1 / ((KEY)1 + exp_of(-key[i])) : (KEY)0;
  }
  if (p.bias || p.groups > 1) {
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (key[i] > NONE) key[i] = sc[i] + (p.bias ? (KEY)p.bias[e0 + i] : (KEY)0);
  }
  float* sel = (float*)smem + tok * p.top_k;
  if (p.groups > 1) {
    KEY* keys = (KEY*)(smem + ((TOK * p.top_k * 4 + 15) & ~15)) + tok * (EPL * L);
    KEY* rank = (KEY*)(smem + ((TOK * p.top_k * 4 + 15) & ~15)) + TOK * (EPL * L) + tok * p.groups;
    const int per = E / p.groups;
#pragma unroll
    for (int i = 0; i < EPL; ++i) keys[e0 + i] = key[i];
    __syncthreads();
    for (int g = lane; g < p.groups; g += L) {
      KEY a = NONE, b = NONE;
      for (int i = 0; i < per; ++i) {
        const KEY k = keys[g * per + i];
        if (k > a) {
          b = a;
          a = k;
        } else if (k > b) {
          b = k;
        }
      }
      rank[g] = b > NONE ? a + b : a;
    }
    __syncthreads();
    // a group stays if fewer than top_groups come before it
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      if (!(key[i] > NONE)) continue;
      const int g = (e0 + i) / per;
      const KEY mine = rank[g];
      int before = 0;
      for (int j = 0; j < p.groups; ++j) before += rank[j] > mine || (rank[j] == mine && j < g);
      if (before >= p.top_groups) key[i] = NONE;
    }
  }
  // the choice, one slot a round
  float total = 0.f;
  for (int s = 0; s < p.top_k; ++s) {
    KEY best = NONE;
    float bs = 0.f;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (key[i] > best) {
        best = key[i];
        bs = (float)sc[i];
        at = e0 + i;
      }
#pragma unroll
    for (int d = 1; d < L; d <<= 1) {
      const KEY o = __shfl_xor(best, d);
      const float os = __shfl_xor(bs, d);
      const int oa = __shfl_xor(at, d);
      if (o > best || (o == best && oa < at)) {
        best = o;
        bs = os;
        at = oa;
      }
    }
    const bool some = best > NONE;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (e0 + i == at) key[i] = NONE;
    total += bs;
    if (lane == 0) {
      sel[s] = some ? bs : 0.f;
      if (live) p.index[t * p.top_k + s] = some ? at : -1;
    }
  }
  __syncthreads();
  if (!live) return;
  const float f = p.renormalize ? p.scale / (total > 0.f ? total : 1.f) : p.scale;
  for (int s = lane; s < p.top_k; s += L) route_store<T>(p.weights, t * p.top_k + s, sel[s] * f);
}

// The gradient at the logits.  With c the scale, S the sum of the chosen scores and a the
// sum of dw s over them:  ds = c dw, or c / S (dw - a / S) renormalised;
// softmax: dl = s (ds - sum of s ds), the sum zero when renormalised; sigmoid: dl = ds s (1 - s).
template <typename T, int EPL, int L>
__global__ __launch_bounds__(256) void route_bwd_kernel(RouteParams p) {
  constexpr int TOK = 256 / L;
  const int tid = threadIdx.x, lane = tid % L, tok = tid / L;
  const int64_t t = (int64_t)blockIdx.x * TOK + tok;
  const bool live = t < p.tokens;
  const int E = p.experts, e0 = lane * EPL;
  float l[EPL], sc[EPL], om[EPL], dw[EPL];  // om: 1 - s of the sigmoid
  bool chosen[EPL];
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const bool in = live && e0 + i < E;
    l[i] = in ? route_load<T>(p.logits, t * p.ld + e0 + i) : __builtin_inff();
    if (in && p.bias && !is_finite(p.bias[e0 + i])) l[i] = __builtin_inff();
    l[i] = is_finite(l[i]) ? l[i] : -__builtin_inff();
    top = fmaxf(top, l[i]);
    dw[i] = 0.f;
    chosen[i] = false;
  }
  const float NONE = -__builtin_inff();
  if (p.score == STRATA_HIP_SCORE_SOFTMAX) {
    top = group_max<L>(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      sc[i] = l[i] > NONE ? expf(l[i] - top) : 0.f;
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
  float S = 0.f, a = 0.f;
  for (int s = 0; s < p.top_k; ++s) {
    const int at = live ? p.index[t * p.top_k + s] : -1;
    const float d = live ? route_load<T>(p.dweights, t * p.top_k + s) : 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (e0 + i == at) {
        chosen[i] = true;
        dw[i] = d;
        S += sc[i];
        a = fmaf(d, sc[i], a);
      }
  }
  S = group_sum<L>(S);
  a = group_sum<L>(a);
  const bool norm = p.renormalize && S > 0.f;
  const float c = norm ? p.scale / S : p.scale, mean = norm ? a / S : 0.f;
  const float back = p.renormalize ? 0.f : p.scale * a;
  if (!live) return;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    if (e0 + i >= E) continue;
    const float ds = chosen[i] ? c * (dw[i] - mean) : 0.f;
    const float dl = p.score == STRATA_HIP_SCORE_SOFTMAX ? sc[i] * (ds - back) : ds * sc[i] * om[i];
    route_store<T>(p.dlogits, t * E + e0 + i, l[i] > NONE ? dl : 0.f);
  }
}

// ---------------------------------------------------------------------------
// The plan: the chosen (token, slot) pairs in the order of their experts, pairs of one
// expert in their own order, by a counting sort whose result depends on nothing else.
//   row_token[r], row_weight[r]  the token and the weight of row r's pair
//   slot_row[s]  the row of pair s, -1 where its index names no expert
//   offsets[e]   the first row of expert e; offsets[E] the number of rows
//   tiles        [n, then n pairs (expert, first row)]: `tile` rows of one expert each
// Pairs are taken PLAN_N at a time: counted per block, the blocks' counts summed, and placed by block, wave and lane (the lanes of a wave that name the same
// expert find each other by one ballot per bit of the expert's number).
// ---------------------------------------------------------------------------
constexpr int PLAN_N = 1024, PLAN_WAVES = PLAN_N / 64, PLAN_MAX_E = 512;

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
  for (int k = 0; k < seg; ++k) {
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

// Lanes a token and experts a lane.
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
  const bool wide = p.bias || p.groups > 1;
  return route_width(p.experts, [&](auto epl, auto l) {
    constexpr int EPL = decltype(epl)::value, L = decltype(l)::value, TOK = 256 / L;
    const dim3 grid((unsigned)((p.tokens + TOK - 1) / TOK));
    size_t smem = ((size_t)TOK * p.top_k * 4 + 15) & ~(size_t)15;
    if (p.groups > 1) smem += (size_t)TOK * (EPL * L + p.groups) * 8;
    auto go = [&](auto t) {
      using T = decltype(t);
      if (wide) hipLaunchKernelGGL((route_kernel<T, double, EPL, L>), grid, dim3(256), smem, (hipStream_t)stream, p);
      else hipLaunchKernelGGL((route_kernel<T, float, EPL, L>), grid, dim3(256), smem, (hipStream_t)stream, p);
    };
    if (a->dtype == STRATA_HIP_F32) go(0.f);
    else go((bf16)0.f);
    return check_launch("expert_route");
  });
}

extern "C" int strata_hip_expert_route_bwd(const strata_hip_expert_route_args* a, void* stream) {
  using namespace strata;
  RouteParams p;
  if (const int rc = route_params("expert_route_bwd", a, p)) return rc;
  if (p.tokens == 0) return STRATA_HIP_OK;
  if (!p.logits || !p.dweights || !p.index || !p.dlogits) return fail(STRATA_HIP_EINVAL, "expert_route_bwd: null pointer");
  return route_width(p.experts, [&](auto epl, auto l) {
    constexpr int EPL = decltype(epl)::value, L = decltype(l)::value, TOK = 256 / L;
    const dim3 grid((unsigned)((p.tokens + TOK - 1) / TOK));
    if (a->dtype == STRATA_HIP_F32) hipLaunchKernelGGL((route_bwd_kernel<float, EPL, L>), grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL((route_bwd_kernel<bf16, EPL, L>), grid, dim3(256), 0, (hipStream_t)stream, p);
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
  if (a->pairs < 0 || a->experts <= 0 || a->tile <= 0 || a->top_k <= 0 || a->pairs % a->top_k) return fail(STRATA_HIP_EINVAL, "expert_plan: bad sizes");
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
