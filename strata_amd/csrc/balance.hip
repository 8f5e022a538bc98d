// What keeps the routing to experts balanced, for gfx950: the balance loss, the z-loss of the logits and the
// experts' load; their gradient at the logits.
//
//   s = softmax(l) over a token's experts that are not masked, or sigmoid(l) divided by the sum of the token's
//   a sequence of n tokens that have an expert left:  f = E load / (k n),  P = sum over its tokens of s / n
//   balance = mean over the sequences (of n > 0) of sum over experts of f P     z = mean over all tokens of lse^2
// with lse the log-sum-exp of a token's logits, load an expert's number of entries in the index.  A sequence whose
// load is even has a balance of 1.  No gradient flows through load:
//   dl = g (s (f - sum f s) [1 - sigmoid(l)]) / (n sequences) + gz 2 lse softmax(l) / tokens
// A sigmoid's scores are the softmax of the sigmoid's logarithms min(l, 0) - log(1 + exp(-|l|)), so scores that are
// all small keep their ratios.
//
// A lane holds 8 consecutive experts of a token and L lanes a token, so that a token's row is read in 16-byte runs
// and needs log2(L) exchanges.  A workgroup takes a run of one sequence's tokens and leaves an fp32 sum of scores and
// a load for every expert; one workgroup (of many sequences one for each 64, and another one) adds these up in 64 bits, in an order
// fixed by the sizes.  Loads are integers, so that LDS atomics may add them in any order.
//
// Bound by the operations, exponentials of 32 bits (five an element with sigmoid scores), and for few tokens by the three
// launches: 65536 tokens of 64 experts in fp32 27 us for the sums (0.6 TB/s), 17 to add 512 workgroups' up, 29 for the gradient
// (1.2 TB/s); 1350 of 24 in bf16 6.4, 5.8 and 4.2.  A call's host path is 17 us, with its backward through autograd 96, so a
// training step meets the kernels' time only where it is captured or the GPU lags behind.
#include <algorithm>

#include "route.h"

namespace strata {

struct BalanceParams {
  const void* logits;
  const int32_t* index;
  float* balance;
  float* z;
  int32_t* load;
  float* state;  // [0] 1 / sequences that count, [1] 2 / tokens that count, then f / n, [sequences, experts]
  const float* dbalance;
  const float* dz;
  void* dlogits;
  float* sums;      // a workgroup's sums of scores [wgs, experts], then
  int32_t* counts;  // its loads [wgs, experts]
  double* zs;       // its sum of lse^2
  int32_t* tokens_of;  // its tokens that count
  double* balances;    // of more than BAL_GROUP sequences: a finishing workgroup's sum over them,
  int32_t* counted;    // its sequences that count,
  int32_t* loads;      // and its load [finishing workgroups, experts]
  int64_t per, ld;     // tokens of a sequence
  int64_t run;         // tokens of a workgroup
  int64_t first;       // the launch's first token (backward)
  int experts, top_k, score, sequences, wgs_of;  // workgroups of a sequence
};

constexpr int BAL_EPL = 8;
constexpr int BAL_GROUP = 64;  // sequences that one workgroup adds up
constexpr float BAL_NONE = -__builtin_inff();

// The token's scores and log-sum-exp from its logits (-inf where masked); soft: the softmax, where it is not the score.
template <int L, bool SIGMOID>
__device__ __forceinline__ void balance_scores(const float (&l)[BAL_EPL], float (&s)[BAL_EPL], float (&soft)[BAL_EPL], float& lse) {
  float top = BAL_NONE, sum = 0.f;
#pragma unroll
  for (int i = 0; i < BAL_EPL; ++i) top = fmaxf(top, l[i]);
  top = group_max<L>(top);
  const bool some = top > BAL_NONE;
#pragma unroll
  for (int i = 0; i < BAL_EPL; ++i) {
    soft[i] = some ? expf(l[i] - top) : 0.f;
    sum += soft[i];
  }
  sum = group_sum<L>(sum);
  lse = some ? top + logf(sum) : 0.f;
  const float r = some ? 1.f / sum : 0.f;
#pragma unroll
  for (int i = 0; i < BAL_EPL; ++i) soft[i] *= r;
  if constexpr (SIGMOID) {
    // relative to the largest logit's logarithm
    const float best = some ? fminf(top, 0.f) - log1pf(expf(-fabsf(top))) : 0.f;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < BAL_EPL; ++i) {
      s[i] = l[i] > BAL_NONE ? expf(fminf(l[i], 0.f) - log1pf(expf(-fabsf(l[i]))) - best) : 0.f;
      sum += s[i];
    }
    sum = group_sum<L>(sum);
    const float q = some ? 1.f / sum : 0.f;
#pragma unroll
    for (int i = 0; i < BAL_EPL; ++i) s[i] *= q;
  } else {
#pragma unroll
    for (int i = 0; i < BAL_EPL; ++i) s[i] = soft[i];
  }
}

template <typename T, bool VEC, int L>
__device__ __forceinline__ void balance_row(const BalanceParams& p, int64_t t, int e0, int left, float (&l)[BAL_EPL]) {
  route_row<T, BAL_EPL, VEC>(p.logits, t * p.ld + e0, left, __builtin_inff(), l);
#pragma unroll
  for (int i = 0; i < BAL_EPL; ++i) l[i] = is_finite(l[i]) ? l[i] : BAL_NONE;
}

template <typename T, bool VEC, bool SIGMOID, int L>
__global__ __launch_bounds__(256) void balance_stats_kernel(BalanceParams p) {
  constexpr int TOK = 256 / L, W = BAL_EPL * L;
  __shared__ float rows[4][W];
  __shared__ int hist[W];
  __shared__ double zred[4];
  __shared__ int nred[4];
  const int tid = threadIdx.x, lane = tid % L, tok = tid / L, E = p.experts, e0 = lane * BAL_EPL;
  const int seq = blockIdx.x / p.wgs_of, part = blockIdx.x % p.wgs_of;
  const int64_t first = seq * p.per, t0 = first + min(part * p.run, p.per), t1 = first + min((part + 1) * p.run, p.per);
  for (int e = tid; e < W; e += 256) hist[e] = 0;
  __syncthreads();
  float acc[BAL_EPL];
#pragma unroll
  for (int i = 0; i < BAL_EPL; ++i) acc[i] = 0.f;
  double z = 0.;
  int n = 0;
  for (int64_t t = t0; t < t1; t += TOK) {
    float l[BAL_EPL], s[BAL_EPL], soft[BAL_EPL], lse;
    const bool live = t + tok < t1;
    balance_row<T, VEC, L>(p, t + tok, e0, live ? E - e0 : 0, l);
    balance_scores<L, SIGMOID>(l, s, soft, lse);
    float top = BAL_NONE;
#pragma unroll
    for (int i = 0; i < BAL_EPL; ++i) {
      acc[i] += s[i];
      top = fmaxf(top, l[i]);
    }
    if (group_max<L>(top) > BAL_NONE && lane == 0) {
      ++n;
      z = fma((double)lse, (double)lse, z);
    }
  }
  for (int64_t i = t0 * p.top_k + tid; i < t1 * p.top_k; i += 256) {
    const int e = p.index[i];
    if ((uint32_t)e < (uint32_t)E) atomicAdd(&hist[e], 1);
  }
#pragma unroll
  for (int d = L; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < BAL_EPL; ++i) acc[i] += __shfl_xor(acc[i], d);
  if ((tid & 63) < L)
#pragma unroll
    for (int i = 0; i < BAL_EPL; ++i) rows[tid >> 6][e0 + i] = acc[i];
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    z += __shfl_xor(z, d);
    n += __shfl_xor(n, d);
  }
  if ((tid & 63) == 0) {
    zred[tid >> 6] = z;
    nred[tid >> 6] = n;
  }
  __syncthreads();
  for (int e = tid; e < E; e += 256) {
    p.sums[(int64_t)blockIdx.x * E + e] = ((rows[0][e] + rows[1][e]) + rows[2][e]) + rows[3][e];
    p.counts[(int64_t)blockIdx.x * E + e] = hist[e];
  }
  if (tid == 0) {
    p.zs[blockIdx.x] = ((zred[0] + zred[1]) + zred[2]) + zred[3];
    p.tokens_of[blockIdx.x] = nred[0] + nred[1] + nred[2] + nred[3];
  }
}

// The sum of lse^2 and the tokens that count, over all workgroups: valid in thread 0.
struct BalanceTotals {
  double z;
  int64_t n;
};
__device__ __forceinline__ BalanceTotals balance_totals(const BalanceParams& p) {
  constexpr int NW = 16;
  __shared__ double zred[NW];
  __shared__ int64_t nred[NW];
  const int tid = threadIdx.x;
  double z = 0.;
  int64_t n = 0;
  for (int b = tid; b < p.sequences * p.wgs_of; b += 1024) {
    z += p.zs[b];
    n += p.tokens_of[b];
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    z += __shfl_xor(z, d);
    n += __shfl_xor(n, d);
  }
  if ((tid & 63) == 0) {
    zred[tid >> 6] = z;
    nred[tid >> 6] = n;
  }
  __syncthreads();
  if (tid == 0)
    for (int w = 1; w < NW; ++w) {
      z += zred[w];
      n += nred[w];
    }
  return {z, n};
}
__device__ __forceinline__ void balance_results(const BalanceParams& p, double balance, int counted, BalanceTotals t) {
  const double ig = counted ? 1. / counted : 0., in = t.n ? 1. / (double)t.n : 0.;
  *p.balance = (float)(balance * ig);
  *p.z = (float)(t.z * in);
  p.state[0] = (float)ig;
  p.state[1] = (float)(2. * in);
}

// The workgroups' sums added up, of BAL_GROUP sequences a workgroup: a sequence is taken by 16 / (sequences, rounded up to a power
// of two) waves, one at least, that share its workgroups; a lane takes every 64th expert.  16 sequences take 2.6 us: 65536
// tokens of 64 experts in 1024 sequences 185 us by one workgroup, 41 by several, in 65536 10600 and 214; 8192 tokens in 128 46 and 37.
__global__ __launch_bounds__(1024) void balance_finish_kernel(BalanceParams p) {
  constexpr int NW = 16, EL = ROUTE_MAX_E / 64;
  __shared__ double sum[NW][ROUTE_MAX_E];
  __shared__ int cnt[NW][ROUTE_MAX_E];
  __shared__ int load[ROUTE_MAX_E];
  __shared__ double each[NW];
  __shared__ int some[NW];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, E = p.experts;
  const int first = blockIdx.x * BAL_GROUP, G = gridDim.x == 1 ? p.sequences : min(p.sequences, first + BAL_GROUP);
  int slots = 1;  // sequences at a time
  while (slots < G - first && slots < NW) slots *= 2;
  const int per = NW / slots, share = wave % per, slot = wave / per;
  for (int e = tid; e < E; e += 1024) load[e] = 0;
  double balance = 0.;  // thread 0
  int counted = 0;
  for (int g0 = first; g0 < G; g0 += slots) {
    const int g = g0 + slot;
    double a[EL];
    int c[EL];
#pragma unroll
    for (int i = 0; i < EL; ++i) {
      a[i] = 0.;
      c[i] = 0;
    }
    int ng = 0;
    if (g < G) {
      for (int b = lane; b < p.wgs_of; b += 64) ng += p.tokens_of[g * p.wgs_of + b];
#pragma unroll
      for (int d = 32; d; d >>= 1) ng += __shfl_xor(ng, d);
#pragma unroll 4
      for (int b = share; b < p.wgs_of; b += per) {
        const int64_t row = (int64_t)(g * p.wgs_of + b) * E;
#pragma unroll
        for (int i = 0; i < EL; ++i) {
          const int e = 64 * i + lane;
          if (e < E) {
            a[i] += p.sums[row + e];
            c[i] += p.counts[row + e];
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < EL; ++i) {
      sum[wave][64 * i + lane] = a[i];
      cnt[wave][64 * i + lane] = c[i];
    }
    __syncthreads();
    if (share == 0) {
      double term = 0.;
      if (g < G) {
        const double inv = ng > 0 ? 1. / (double)ng : 0.;
        for (int e = lane; e < E; e += 64) {
          double s = 0.;
          int k = 0;
          for (int w = 0; w < per; ++w) {
            s += sum[wave + w][e];
            k += cnt[wave + w][e];
          }
          const double f = (double)k * E * inv / p.top_k;
          term += f * s * inv;
          p.state[2 + (int64_t)g * E + e] = (float)(f * inv);
          atomicAdd(&load[e], k);
        }
      }
#pragma unroll
      for (int d = 32; d; d >>= 1) term += __shfl_xor(term, d);
      if (lane == 0) {
        each[slot] = term;
        some[slot] = g < G && ng > 0;
      }
    }
    __syncthreads();
    if (tid == 0)
      for (int k = 0; k < slots; ++k) {
        balance += each[k];
        counted += some[k];
      }
  }
  __syncthreads();
  int32_t* const loads = gridDim.x == 1 ? p.load : p.loads + (int64_t)blockIdx.x * E;
  for (int e = tid; e < E; e += 1024) loads[e] = load[e];
  if (gridDim.x == 1) {  // uniform
    const BalanceTotals t = balance_totals(p);
    if (tid == 0) balance_results(p, balance, counted, t);
  } else if (tid == 0) {
    p.balances[blockIdx.x] = balance;
    p.counted[blockIdx.x] = counted;
  }
}

// What the finishing workgroups (at most 1024) have, added up.
__global__ __launch_bounds__(1024) void balance_join_kernel(BalanceParams p) {
  constexpr int NW = 16;
  __shared__ int load[ROUTE_MAX_E];
  __shared__ double bred[NW];
  __shared__ int cred[NW];
  const int tid = threadIdx.x, E = p.experts, groups = (p.sequences + BAL_GROUP - 1) / BAL_GROUP;
  if (tid < ROUTE_MAX_E) load[tid] = 0;
  double balance = tid < groups ? p.balances[tid] : 0.;
  int counted = tid < groups ? p.counted[tid] : 0;
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    balance += __shfl_xor(balance, d);
    counted += __shfl_xor(counted, d);
  }
  if ((tid & 63) == 0) {
    bred[tid >> 6] = balance;
    cred[tid >> 6] = counted;
  }
  __syncthreads();
  int k = 0;  // an expert's share of the workgroups, of those that 1024 threads hold at once
  const int at = tid % E, shares = 1024 / E, share = tid / E;
  if (share < shares)
#pragma unroll 8
    for (int g = share; g < groups; g += shares) k += p.loads[(int64_t)g * E + at];
  if (share < shares) atomicAdd(&load[at], k);
  const BalanceTotals t = balance_totals(p);
  if (tid < E) p.load[tid] = load[tid];  // a barrier behind the last of them
  if (tid == 0) {
    for (int w = 1; w < NW; ++w) {
      balance += bred[w];
      counted += cred[w];
    }
    balance_results(p, balance, counted, t);
  }
}

template <typename T, bool VEC, bool SIGMOID, int L>
__global__ __launch_bounds__(256) void balance_bwd_kernel(BalanceParams p) {
  constexpr int TOK = 256 / L;
  const int tid = threadIdx.x, lane = tid % L, tok = tid / L, E = p.experts, e0 = lane * BAL_EPL;
  const int64_t t = p.first + (int64_t)blockIdx.x * TOK + tok, total = p.per * p.sequences;
  const bool live = t < total;
  const int left = live ? E - e0 : 0;
  float l[BAL_EPL], s[BAL_EPL], soft[BAL_EPL], f[BAL_EPL], lse;
  const float gb = p.dbalance ? *p.dbalance * p.state[0] : 0.f, gz = p.dz ? *p.dz * p.state[1] : 0.f;
  balance_row<T, VEC, L>(p, t, e0, left, l);
  route_row<float, BAL_EPL, false>(p.state, 2 + (live ? t / p.per : 0) * E + e0, left, 0.f, f);
  balance_scores<L, SIGMOID>(l, s, soft, lse);
  float mean = 0.f;
#pragma unroll
  for (int i = 0; i < BAL_EPL; ++i) mean = fmaf(f[i], s[i], mean);
  mean = group_sum<L>(mean);
  if (!live) return;
  float dl[BAL_EPL];
  const float zf = gz * lse;
#pragma unroll
  for (int i = 0; i < BAL_EPL; ++i) {
    float d = gb * (s[i] * (f[i] - mean));
    if (SIGMOID) {
      const float x = expf(-fabsf(l[i]));
      d *= (l[i] >= 0.f ? x : 1.f) / (1.f + x);  // 1 - sigmoid(l)
    }
    dl[i] = l[i] > BAL_NONE ? fmaf(zf, soft[i], d) : 0.f;
  }
  const int64_t at = t * E + e0;
  if constexpr (VEC) {
    if (left >= BAL_EPL) {
      if constexpr (sizeof(T) == 4) {
        *(f32x4*)((float*)p.dlogits + at) = (f32x4){dl[0], dl[1], dl[2], dl[3]};
        *(f32x4*)((float*)p.dlogits + at + 4) = (f32x4){dl[4], dl[5], dl[6], dl[7]};
      } else {
        *(u32x4*)((bf16*)p.dlogits + at) =
            (u32x4){pack_bf16x2(dl[0], dl[1]), pack_bf16x2(dl[2], dl[3]), pack_bf16x2(dl[4], dl[5]), pack_bf16x2(dl[6], dl[7])};
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < BAL_EPL; ++i)
    if (i < left) route_store<T>(p.dlogits, at + i, dl[i]);
}

// f(lanes a token), of 8 experts each.
template <typename F>
static int balance_width(int experts, F f) {
  using std::integral_constant;
  if (experts <= 8) return f(integral_constant<int, 1>{});
  if (experts <= 16) return f(integral_constant<int, 2>{});
  if (experts <= 32) return f(integral_constant<int, 4>{});
  if (experts <= 64) return f(integral_constant<int, 8>{});
  if (experts <= 128) return f(integral_constant<int, 16>{});
  if (experts <= 256) return f(integral_constant<int, 32>{});
  return f(integral_constant<int, 64>{});
}

// Workgroups of a sequence: whole rounds of a workgroup's tokens, up to 512 workgroups in all and 65536 sums
// for the one that adds them up.
static int64_t balance_wgs(int64_t per, int64_t sequences, int experts) {
  int lanes = 1;
  while (8 * lanes < experts) lanes *= 2;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(512, 65536 / experts) / sequences);
  const int64_t tok = 256 / lanes, rounds = (per + tok - 1) / tok;
  return std::min(most, rounds);
}

// Workgroups that add up sequences for one more: none where one does it all.
static int64_t balance_groups(int64_t sequences) {
  return sequences > BAL_GROUP ? (sequences + BAL_GROUP - 1) / BAL_GROUP : 0;
}

static int balance_sizes(const std::string& n, int64_t tokens, int64_t sequences, int experts, int top_k) {
  if (tokens < 0 || sequences <= 0 || experts <= 0 || top_k <= 0)
    return fail(STRATA_HIP_EINVAL, n + ": bad tokens, sequences, experts or top_k");
  if (experts > ROUTE_MAX_E) return fail(STRATA_HIP_EUNSUPPORTED, n + ": at most 512 experts");
  if (tokens > 0x7fffffff / top_k || sequences > (1 << 16))
    return fail(STRATA_HIP_EUNSUPPORTED, n + ": more than 2^31 - 1 chosen pairs or 65536 sequences");
  return STRATA_HIP_OK;
}

static int balance_params(const std::string& n, const strata_hip_expert_balance_args* a, BalanceParams& p) {
  if (!a) return fail(STRATA_HIP_EINVAL, n + ": null args");
  if (const int rc = balance_sizes(n, a->tokens, a->sequences, a->experts, a->top_k)) return rc;
  if (a->tokens % a->sequences) return fail(STRATA_HIP_EINVAL, n + ": the tokens are no whole number for each sequence");
  if (a->dtype != STRATA_HIP_F32 && a->dtype != STRATA_HIP_BF16) return fail(STRATA_HIP_EINVAL, n + ": bad dtype");
  if (a->score != STRATA_HIP_SCORE_SOFTMAX && a->score != STRATA_HIP_SCORE_SIGMOID) return fail(STRATA_HIP_EINVAL, n + ": bad score");
  if (a->tokens > 1 && a->ld < a->experts) return fail(STRATA_HIP_EINVAL, n + ": row stride smaller than the row");
  if (!a->state || ((uintptr_t)a->state & 3)) return fail(STRATA_HIP_EINVAL, n + ": null state");
  if (a->tokens > 0 && !a->logits) return fail(STRATA_HIP_EINVAL, n + ": null pointer");
  p = {};
  p.logits = a->logits;
  p.index = a->index;
  p.balance = a->balance;
  p.z = a->z;
  p.load = a->load;
  p.state = a->state;
  p.dbalance = a->dbalance;
  p.dz = a->dz;
  p.dlogits = a->dlogits;
  p.per = a->tokens / a->sequences;
  p.ld = a->tokens > 1 ? a->ld : a->experts;
  p.experts = a->experts;
  p.top_k = a->top_k;
  p.score = a->score;
  p.sequences = (int)a->sequences;
  return STRATA_HIP_OK;
}

// go(T, VEC, SIGMOID) with the call's type, whether its rows are whole 16-byte runs, and its score.
template <typename F>
static void balance_pick(const strata_hip_expert_balance_args* a, bool vec, F go) {
  auto score = [&](auto t, auto v) {
    if (a->score == STRATA_HIP_SCORE_SIGMOID) go(t, v, std::true_type{});
    else go(t, v, std::false_type{});
  };
  auto rows = [&](auto t) {
    if (vec) score(t, std::true_type{});
    else score(t, std::false_type{});
  };
  if (a->dtype == STRATA_HIP_F32) rows(0.f);
  else rows((bf16)0.f);
}

static bool balance_aligned(const strata_hip_expert_balance_args* a) {
  return a->experts % 4 == 0 && (a->tokens <= 1 || a->ld % 4 == 0) && ((uintptr_t)a->logits & 15) == 0;
}

}  // namespace strata

extern "C" int64_t strata_hip_expert_balance_workspace(int64_t tokens, int64_t sequences, int32_t experts) {
  if (const int rc = strata::balance_sizes("expert_balance_workspace", tokens, sequences, experts, 1)) return rc == STRATA_HIP_EUNSUPPORTED ? -1 : 0;
  if (tokens == 0) return 0;
  return strata::balance_wgs(tokens / sequences, sequences, experts) * sequences * (12 + 8 * (int64_t)experts) +
         strata::balance_groups(sequences) * (12 + 4 * (int64_t)experts);
}

extern "C" int strata_hip_expert_balance(const strata_hip_expert_balance_args* a, void* stream) {
  using namespace strata;
  BalanceParams p;
  if (const int rc = balance_params("expert_balance", a, p)) return rc;
  if (!p.balance || !p.z || !p.load) return fail(STRATA_HIP_EINVAL, "expert_balance: null pointer");
  const hipStream_t st = (hipStream_t)stream;
  const int64_t groups = a->tokens > 0 ? balance_groups(p.sequences) : 0;  // (without tokens all are 0)
  if (a->tokens > 0) {
    if (!p.index || !a->workspace || ((uintptr_t)a->workspace & 7))
      return fail(STRATA_HIP_EINVAL, "expert_balance: index and workspace must be given, the workspace 8-byte aligned");
    p.wgs_of = (int)balance_wgs(p.per, p.sequences, p.experts);
    const int64_t wgs = (int64_t)p.wgs_of * p.sequences;
    p.zs = (double*)a->workspace;
    p.balances = p.zs + wgs;
    p.tokens_of = (int32_t*)(p.balances + groups);
    p.counted = p.tokens_of + wgs;
    p.loads = p.counted + groups;
    p.sums = (float*)(p.loads + groups * p.experts);
    p.counts = (int32_t*)(p.sums + wgs * p.experts);
    const int rc = balance_width(p.experts, [&](auto lanes) {
      constexpr int L = decltype(lanes)::value, TOK = 256 / L;
      const int64_t rounds = (p.per + TOK - 1) / TOK;
      p.run = (rounds + p.wgs_of - 1) / p.wgs_of * TOK;
      balance_pick(a, balance_aligned(a), [&](auto t, auto v, auto s) {
        hipLaunchKernelGGL((balance_stats_kernel<decltype(t), decltype(v)::value, decltype(s)::value, L>), dim3((unsigned)wgs), dim3(256), 0,
                           st, p);
      });
      return check_launch("expert_balance");
    });
    if (rc) return rc;
  }
  hipLaunchKernelGGL(balance_finish_kernel, dim3((unsigned)std::max<int64_t>(groups, 1)), dim3(1024), 0, st, p);
  if (const int rc = check_launch("expert_balance sums")) return rc;
  if (!groups) return STRATA_HIP_OK;
  hipLaunchKernelGGL(balance_join_kernel, dim3(1), dim3(1024), 0, st, p);
  return check_launch("expert_balance joined sums");
}

extern "C" int strata_hip_expert_balance_bwd(const strata_hip_expert_balance_args* a, void* stream) {
  using namespace strata;
  BalanceParams p;
  if (const int rc = balance_params("expert_balance_bwd", a, p)) return rc;
  if (a->tokens == 0) return STRATA_HIP_OK;
  if (!p.dlogits) return fail(STRATA_HIP_EINVAL, "expert_balance_bwd: null pointer");
  const bool vec = balance_aligned(a) && ((uintptr_t)p.dlogits & 15) == 0 && p.experts % 8 == 0;
  return balance_width(p.experts, [&](auto lanes) {
    constexpr int L = decltype(lanes)::value, TOK = 256 / L;
    constexpr int64_t MOST = 0xffffffff / 256;  // workgroups: a grid holds less than 2^32 threads
    for (; p.first < a->tokens; p.first += MOST * TOK) {
      const int64_t wgs = std::min(MOST, (a->tokens - p.first + TOK - 1) / TOK);
      balance_pick(a, vec, [&](auto t, auto v, auto s) {
        hipLaunchKernelGGL((balance_bwd_kernel<decltype(t), decltype(v)::value, decltype(s)::value, L>), dim3((unsigned)wgs), dim3(256), 0,
                           (hipStream_t)stream, p);
      });
      if (const int rc = check_launch("expert_balance_bwd")) return rc;
    }
    return (int)STRATA_HIP_OK;
  });
}
