// AdamW over many tensors for gfx950, with the clipping of the gradients by their
// global norm and moments held in 32 or in 8 bits.
//
//   c = min(1, max_norm / (|all gradients| + 1e-6)),  g <- c g
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2        t <- t + 1
//   p <- p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// 8-bit moments: 256 consecutive elements share one fp32 scale each for m and v, the
// largest magnitude among them.  A code stands for
//   m = scale * sign(c) (c / 127)^2, c in -127 .. 127      v = scale * ((c + 1) / 256)^2, c in 0 .. 255
// and is the nearest one in the root's domain: the quadratic spacing keeps 2 to 3
// digits of values down to 1e-4 of their block's largest, and v, which divides, is never
// below 1.5e-5 of it.  Decays and sums run in 64 bits there (v_fma_f64 issues at the
// rate of v_fma_f32 here), so a code does not depend on how 32-bit sums round: beside a
// border between two codes one such rounding moves the state by a whole code.  The
// norm's sum of squares runs in 64 bits too, in an order fixed by the sizes.
//
// Bound by memory with 32-bit moments: 133M bf16 elements with masters, twelve blocks 960 wide, 561 us
// for 3.72 GB (6.6 TB/s, some of the gradients out of the caches) and 102 for the 266 MB of the norm
// (2.6 TB/s: reading alone reaches 3.8 to 4.0 here); with 8-bit moments by operations and latency: 59M
// bf16 elements 173 us for 0.60 GB (3.4 TB/s).  Few or small tensors: by the host, 1.5 us a tensor
// (its checks and pointers), which a captured step does not pay.
// The tensors' addresses travel in the launch's arguments, so nothing
// is kept between calls; the step count lives on the device, so a captured step counts on.
#include <algorithm>
#include <cmath>
#include <exception>
#include <unordered_map>
#include <vector>

#include "optim.h"

namespace strata {

constexpr int AW_BLOCK = 256;    // elements per 8-bit scale
constexpr int AW_CHUNK = 4096;   // elements per workgroup of the step
constexpr int AW_SUM = 16384;    // elements per workgroup of the sum of squares
constexpr int AW_HEAD = 8;       // doubles before the partial sums
constexpr int AW_PER = 48;       // tensors per launch: 80 bytes each in 4 KiB of arguments
constexpr int AW_COUNTS = 448;   // step counts per launch of their own
constexpr float AW_TINY = 0x1p-100f;  // the places of 8-bit codes under such a scale are found 2^100 larger: 65536 / scale leaves 32 bits
enum { AW_P32 = 1, AW_G32 = 2, AW_ALIGNED = 4, AW_COUNT_SHIFT = 8 };  // above: which step count is the tensor's

struct AwTensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* ms;
  float* vs;
  float* master;
  int64_t n;
  float lr;
  float decay;     // 1 - lr * weight_decay
  uint32_t first;  // the tensor's first workgroup in the launch
  uint32_t flags;
};
struct AwBatch {
  AwTensor t[AW_PER];
  int count;
  float eps;
  double b1, b2;
  const double* head;    // what aw_head_kernel left for each step count, see there
};
struct SumBatch {
  const void* g[3 * AW_PER];
  int64_t n[3 * AW_PER];
  uint32_t first[3 * AW_PER];
  uint32_t wide[3 * AW_PER];  // 1: fp32, 0: bf16; 2: 16-byte aligned
  int count;
  double* part;
};
static_assert(sizeof(AwBatch) <= 4096 && sizeof(SumBatch) <= 4096, "kernel arguments");

// What nothing reads again before the next step passes the caches by (non-temporal), so that the
// gradients, which the sum of squares has just read, are still there for the step: 133M bf16
// elements with masters and clipping 787 -> 673 us, 30M 187 -> 155, 2M 29 -> 22 (everything
// non-temporal, the sum's reading too: 729, 163, 22).  Parameters are stored as usual, for the next forward.
template <typename V>
__device__ __forceinline__ V load_once(const void* p) { return __builtin_nontemporal_load((const V*)p); }
template <typename V>
__device__ __forceinline__ void store_once(void* p, V v) { __builtin_nontemporal_store(v, (V*)p); }

// Last entry whose first workgroup is at or before `wg`.
template <typename F>
__device__ __forceinline__ int find_entry(int count, uint32_t wg, F first) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first(mid) <= wg) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ---- sum of squares: one 64-bit partial per AW_SUM elements ----
__global__ __launch_bounds__(256) void aw_sum_kernel(SumBatch b) {
  const uint32_t wg = blockIdx.x;
  const int e = find_entry(b.count, wg, [&](int i) { return b.first[i]; });
  const int64_t i0 = (int64_t)(wg - b.first[e]) * AW_SUM, i1 = min(i0 + AW_SUM, b.n[e]);
  const uint32_t wide = b.wide[e];
  const int tid = threadIdx.x;
  double s = 0.;
  if ((wide & 2) && i1 - i0 == AW_SUM) {  // whole and aligned: eight 16-byte loads in flight a thread
    constexpr int U = 8;
    const int rounds = (wide & 1) ? AW_SUM / (1024 * U) : AW_SUM / (2048 * U);
    const char* q = (const char*)b.g[e] + i0 * ((wide & 1) ? 4 : 2) + 16 * tid;
    for (int k = 0; k < rounds; ++k, q += 4096 * U) {
      u32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = *(const u32x4*)(q + 4096 * u);
      if (wide & 1) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const double x = __uint_as_float(v[u][j]);
            s = fma(x, x, s);
          }
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const double lo = bf16_lo(v[u][j]), hi = bf16_hi(v[u][j]);
            s = fma(lo, lo, s);
            s = fma(hi, hi, s);
          }
      }
    }
  } else {
    for (int64_t i = i0 + tid; i < i1; i += 256) {
      const double x = (wide & 1) ? ((const float*)b.g[e])[i] : (float)((const bf16*)b.g[e])[i];
      s = fma(x, x, s);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  __shared__ double red[4];
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) b.part[wg] = ((red[0] + red[1]) + red[2]) + red[3];
}

// ---- what every element of the tensors of one step count shares: head[0] the factor c,
// [1] 1 / (1 - b1^t), [2] 1 / sqrt(1 - b2^t), [3] 1 where the step is left out (a norm that is not finite).
struct AwNorm {
  const double* part;
  int64_t parts;
  double* norm;  // or null: no clipping
  double max_norm, b1, b2;
};

// c and whether the step is left out, in thread 0 of 1024; the partial sums in a fixed order.
__device__ __forceinline__ void aw_clip(const AwNorm& a, double& c, bool& skip) {
  __shared__ double red[16];
  const int tid = threadIdx.x;
  c = 1.;
  skip = false;
  if (a.norm) {
    double s = 0.;
    for (int64_t i = tid; i < a.parts; i += 1024) s += a.part[i];
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) {
      for (int k = 1; k < 16; ++k) s += red[k];
      const double nrm = sqrt(s);
      *a.norm = nrm;
      skip = !(nrm < __builtin_inf());
      c = fmin(1., a.max_norm / (nrm + 1e-6));
    }
  }
}
__device__ __forceinline__ void aw_count(const AwNorm& a, double* head, int64_t* step, double c, bool skip) {
  const int64_t t = *step + (skip ? 0 : 1);
  *step = t;
  head[0] = c;
  head[1] = 1. / (1. - pow(a.b1, (double)t));
  head[2] = 1. / sqrt(1. - pow(a.b2, (double)t));
  head[3] = skip ? 1. : 0.;
}

__global__ __launch_bounds__(1024) void aw_head_kernel(AwNorm a, double* head, int64_t* step) {
  double c;
  bool skip;
  aw_clip(a, c, skip);
  if (threadIdx.x == 0) aw_count(a, head, step, c, skip);
}

// Several counts, each with its head: the factor is the same for all.
struct AwCounts {
  int64_t* step[AW_COUNTS];
  int count;
};
static_assert(sizeof(AwCounts) + sizeof(AwNorm) + 8 <= 4096, "kernel arguments");
__global__ __launch_bounds__(1024) void aw_heads_kernel(AwNorm a, double* heads, AwCounts s) {
  __shared__ double shared_c;
  __shared__ int shared_skip;
  double c;
  bool skip;
  aw_clip(a, c, skip);
  if (threadIdx.x == 0) {
    shared_c = c;
    shared_skip = skip;
  }
  __syncthreads();
  const int k = threadIdx.x;
  if (k < s.count) aw_count(a, heads + 4 * k, s.step[k], shared_c, shared_skip != 0);
}

// ---- the step ----
struct AwShared {
  float c, rate, rbc2, eps, decay, b1, b2, omb1, omb2;
  double db1, db2, dg1, dg2;  // decays, and (1 - b1) c, (1 - b2) c^2
};

// FAST: within 2 u instead of 1/2 u in the root and in the quotient (v_sqrt_f32 and v_rcp_f32,
// a root of less than 2^-96 taken of 2^32 times it), where the step is bound by its operations.
template <bool FAST>
__device__ __forceinline__ float aw_update(const AwShared& s, float p, float m, float v) {
  if (FAST) {
    float root;
    if (s.eps >= 1e-10f) {  // uniform; a root under 2^-48 is then nothing beside eps
      root = __builtin_amdgcn_sqrtf(v);
    } else {
      const bool small = v < 0x1p-96f;
      root = __builtin_amdgcn_sqrtf(small ? v * 0x1p32f : v) * (small ? 0x1p-16f : 1.f);
    }
    return fmaf(p, s.decay, -(s.rate * m) * __builtin_amdgcn_rcpf(fmaf(root, s.rbc2, s.eps)));
  }
  const float denom = fmaf(__builtin_sqrtf(v), s.rbc2, s.eps);
  return fmaf(p, s.decay, -(s.rate * m) / denom);
}

__device__ __forceinline__ float load1(const void* p, int64_t i, bool wide) {
  return wide ? ((const float*)p)[i] : (float)((const bf16*)p)[i];
}

// Four consecutive elements from a 16-byte (fp32) or 8-byte (bf16) run.  ONCE: non-temporal; not with
// 8-bit moments, where all of a step's data is small enough to meet the caches (30M fp32 elements
// 129 -> 116 us without).
template <bool ONCE>
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i, bool wide) {
  if (wide) return ONCE ? load_once<f32x4>((const float*)p + i) : *(const f32x4*)((const float*)p + i);
  const u32x2 w = ONCE ? load_once<u32x2>((const bf16*)p + i) : *(const u32x2*)((const bf16*)p + i);
  return (f32x4){bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
}
__device__ __forceinline__ void store4(void* p, int64_t i, bool wide, f32x4 v) {
  if (wide) *(f32x4*)((float*)p + i) = v;
  else *(u32x2*)((bf16*)p + i) = (u32x2){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// 32-bit moments: 256 threads x 4 elements x 4 rounds.
template <bool P32, bool G32, bool MASTER>
__device__ __forceinline__ void aw_chunk32(const AwTensor& t, const AwShared& s, int64_t i0, int tid) {
  float* m = (float*)t.m;
  float* v = (float*)t.v;
  auto one = [&](float g, float& mm, float& vv, float pp) {
    g *= s.c;
    mm = fmaf(s.omb1, g, s.b1 * mm);
    vv = fmaf(s.omb2 * g, g, s.b2 * vv);
    return aw_update<false>(s, pp, mm, vv);
  };
  if ((t.flags & AW_ALIGNED) && i0 + AW_CHUNK <= t.n) {
    f32x4 g[4], mm[4], vv[4], pp[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t i = i0 + 1024 * k + 4 * tid;
      g[k] = load4<true>(t.g, i, G32);
      mm[k] = load_once<f32x4>(m + i);
      vv[k] = load_once<f32x4>(v + i);
      pp[k] = MASTER ? load_once<f32x4>(t.master + i) : load4<true>(t.p, i, P32);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t i = i0 + 1024 * k + 4 * tid;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float a = mm[k][e], b = vv[k][e];
        pp[k][e] = one(g[k][e], a, b, pp[k][e]);
        mm[k][e] = a;
        vv[k][e] = b;
      }
      store_once<f32x4>(m + i, mm[k]);
      store_once<f32x4>(v + i, vv[k]);
      if (MASTER) store_once<f32x4>(t.master + i, pp[k]);
      store4(t.p, i, P32, pp[k]);
    }
    return;
  }
  const int64_t i1 = min(i0 + AW_CHUNK, t.n);
  for (int64_t i = i0 + tid; i < i1; i += 256) {
    float a = m[i], b = v[i];
    const float p = one(load1(t.g, i, G32), a, b, MASTER ? t.master[i] : load1(t.p, i, P32));
    m[i] = a;
    v[i] = b;
    if (MASTER) t.master[i] = p;
    if (P32) ((float*)t.p)[i] = p;
    else ((bf16*)t.p)[i] = (bf16)p;
  }
}

__device__ __forceinline__ double aw_value_m(int c, double scale) {
  const double r = (double)c * (1. / 127.);
  return (c < 0 ? -(r * r) : r * r) * scale;
}
__device__ __forceinline__ double aw_value_v(int c, double scale) {
  const double r = (double)(c + 1) * (1. / 256.);
  return r * r * scale;
}
// A code found in 32 bits, held to its borders (k +- 1/2)^2 scale in 64.
__device__ __forceinline__ int aw_settle(int k, double x, double scale, double steps, int lo, int hi) {
  const double q = x * (steps * steps), up = (double)k + .5, dn = (double)k - .5;
  if (k < hi && q > up * up * scale) ++k;
  else if (k > lo && q < dn * dn * scale) --k;
  return k;
}

// 8-bit moments: 32 lanes take a block of 256, eight consecutive elements each; a workgroup's
// chunk is two rounds of eight blocks.  VALU and memory are close here (some 50 operations, four of
// them roots or reciprocals, for 10 bytes of a bf16 element): squares of codes are exact in
// 32 bits, so that a moment costs two conversions, four products and a sum in 64 bits; these round
// one by one, as the formula writes them, because a decayed scale and a share of a bf16 gradient
// often add up to exactly half way between two 32-bit scales (0.9 s + 0.1 g); the largest magnitude
// is taken of the bits (one that is no number stays: the block's scale then says so); and whether
// any of a lane's sixteen codes is within 8e-5 of a border (a 32-bit place is off by at most 7e-5)
// is asked once, in a seventh of all waves with yes.  VEC: a whole aligned run of eight, else `left` elements one by one.
template <bool P32, bool G32, bool MASTER, bool VEC>
__device__ __forceinline__ void aw_block8(const AwTensor& t, const AwShared& s, int64_t i, int left) {
#pragma clang fp contract(off)
  const int64_t blk = i / AW_BLOCK;
  int8_t* mc = (int8_t*)t.m;
  uint8_t* vc = (uint8_t*)t.v;
  float g[8], p[8];
  uint32_t wm[2] = {0u, 0u}, wv[2] = {0u, 0u};  // four codes a word
  const float scm = t.ms[blk], scv = t.vs[blk];
  if constexpr (VEC) {
    const u32x2 a = load_once<u32x2>(mc + i), b = load_once<u32x2>(vc + i);
    const f32x4 x0 = load4<false>(t.g, i, G32), x1 = load4<false>(t.g, i + 4, G32);
    const f32x4 y0 = MASTER ? load_once<f32x4>(t.master + i) : load4<false>(t.p, i, P32);
    const f32x4 y1 = MASTER ? load_once<f32x4>(t.master + i + 4) : load4<false>(t.p, i + 4, P32);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g[e] = x0[e];
      g[4 + e] = x1[e];
      p[e] = y0[e];
      p[4 + e] = y1[e];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      wm[h] = a[h];
      wv[h] = b[h];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool in = k < left;
      g[k] = in ? load1(t.g, i + k, G32) : 0.f;
      p[k] = in ? (MASTER ? t.master[i + k] : load1(t.p, i + k, P32)) : 0.f;
      wm[k >> 2] |= (in ? (uint32_t)(uint8_t)mc[i + k] : 0u) << (8 * (k & 3));
      wv[k >> 2] |= (in ? (uint32_t)vc[i + k] : 0u) << (8 * (k & 3));
    }
  }
  const double sm = (double)scm * s.db1, sv = (double)scv * (1. / 65536.);
  double m[8], v[8];
  float mf[8], vf[8];
  uint32_t am = 0u, av = 0u;  // bits of the largest magnitudes
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float cm = (float)(int)(int8_t)(wm[k >> 2] >> (8 * (k & 3)));
    const float cv = (float)((wv[k >> 2] >> (8 * (k & 3))) & 255u) + 1.f;
    const double gd = (double)g[k];
    m[k] = (double)(cm * fabsf(cm)) * (1. / 16129.) * sm + s.dg1 * gd;  // 127^2 / 16129 is 1
    v[k] = (double)(cv * cv) * sv * s.db2 + s.dg2 * gd * gd;            // the first product is exact
    mf[k] = (float)m[k];
    vf[k] = (float)v[k];
    if (VEC || k < left) {  // rounding keeps the order: the largest rounded is the largest, rounded
      am = max(am, __float_as_uint(mf[k]) & 0x7fffffffu);
      av = max(av, __float_as_uint(vf[k]) & 0x7fffffffu);
    }
    p[k] = aw_update<true>(s, p[k], mf[k], vf[k]);
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    am = max(am, (uint32_t)__shfl_xor((int)am, d));
    av = max(av, (uint32_t)__shfl_xor((int)av, d));
  }
  const float fm = __uint_as_float(am), fv = __uint_as_float(av);
  float fms = fm, fvs = fv;
  if (fm < AW_TINY) {  // the same for a block's lanes
    fms *= 0x1p100f;
#pragma unroll
    for (int k = 0; k < 8; ++k) mf[k] = (float)(m[k] * 0x1p100);
  }
  if (fv < AW_TINY) {
    fvs *= 0x1p100f;
#pragma unroll
    for (int k = 0; k < 8; ++k) vf[k] = (float)(v[k] * 0x1p100);
  }
  const float im = fms > 0.f ? 16129.f / fms : 0.f, iv = fvs > 0.f ? 65536.f / fvs : 0.f;
  int km[8], kv[8];
  float dev = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = __builtin_amdgcn_sqrtf(fabsf(mf[k]) * im), b = fmaxf(__builtin_amdgcn_sqrtf(vf[k] * iv), 1.f);
    const float ra = rintf(a), rb = rintf(b);
    dev = fmaxf(dev, fmaxf(fabsf(a - ra), fabsf(b - rb)));
    km[k] = (int)fminf(ra, 127.f);  // a block whose scale is no number or infinite: any code
    kv[k] = (int)fminf(rb, 256.f);
  }
  if (dev > 0.49992f) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      km[k] = aw_settle(km[k], fabs(m[k]), (double)fm, 127., 0, 127);
      kv[k] = aw_settle(kv[k], v[k], (double)fv, 256., 1, 256);
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) km[k] = mf[k] < 0.f ? -km[k] : km[k];
  if ((threadIdx.x & 31) == 0) {
    t.ms[blk] = fm;
    t.vs[blk] = fv;
  }
  if constexpr (VEC) {
    u32x2 a = {0u, 0u}, b = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e >> 2] |= (uint32_t)(km[e] & 255) << (8 * (e & 3));
      b[e >> 2] |= (uint32_t)(kv[e] - 1) << (8 * (e & 3));
    }
    const f32x4 y0 = {p[0], p[1], p[2], p[3]}, y1 = {p[4], p[5], p[6], p[7]};
    if (MASTER) {
      store_once<f32x4>(t.master + i, y0);
      store_once<f32x4>(t.master + i + 4, y1);
    }
    if (P32) {
      store4(t.p, i, true, y0);
      store4(t.p, i + 4, true, y1);
    } else {
      *(u32x4*)((bf16*)t.p + i) =
          (u32x4){pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])};
    }
    store_once<u32x2>(mc + i, a);
    store_once<u32x2>(vc + i, b);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k >= left) continue;
      mc[i + k] = (int8_t)km[k];
      vc[i + k] = (uint8_t)(kv[k] - 1);
      if (MASTER) t.master[i + k] = p[k];
      if (P32) ((float*)t.p)[i + k] = p[k];
      else ((bf16*)t.p)[i + k] = (bf16)p[k];
    }
  }
}

template <bool P32, bool G32, bool MASTER>
__device__ __forceinline__ void aw_chunk8(const AwTensor& t, const AwShared& s, int64_t i0, int tid) {
#pragma unroll 1
  for (int k = 0; k < AW_CHUNK / 2048; ++k) {
    const int64_t i = i0 + 2048 * k + 8 * tid;
    if (i0 + 2048 * k + (tid / 32) * AW_BLOCK >= t.n) return;  // whole groups of 32 lanes leave
    // every lane of a block takes the same path: they exchange their largest magnitudes
    const int64_t end = i0 + 2048 * k + (tid / 32 + 1) * AW_BLOCK;
    if ((t.flags & AW_ALIGNED) && end <= t.n) aw_block8<P32, G32, MASTER, true>(t, s, i, 8);
    else aw_block8<P32, G32, MASTER, false>(t, s, i, (int)min((int64_t)8, t.n - i));  // past the end: none
  }
}

template <bool Q8>
__global__ __launch_bounds__(256) void aw_step_kernel(AwBatch b) {
  const uint32_t wg = blockIdx.x;
  if (b.head[3] != 0.) return;
  const int e = find_entry(b.count, wg, [&](int i) { return b.t[i].first; });
  const AwTensor t = b.t[e];
  const double* head = b.head + 4 * (t.flags >> AW_COUNT_SHIFT);
  AwShared s;
  const double c = head[0];
  s.c = (float)c;
  s.rate = t.lr * (float)head[1];
  s.rbc2 = (float)head[2];
  s.eps = b.eps;
  s.decay = t.decay;
  s.db1 = b.b1;
  s.db2 = b.b2;
  s.dg1 = (1. - b.b1) * c;
  s.dg2 = (1. - b.b2) * (c * c);
  s.b1 = (float)b.b1;
  s.b2 = (float)b.b2;
  s.omb1 = (float)(1. - b.b1);
  s.omb2 = (float)(1. - b.b2);
  const int64_t i0 = (int64_t)(wg - t.first) * AW_CHUNK;
  const int tid = threadIdx.x;
  const bool p32 = t.flags & AW_P32, g32 = t.flags & AW_G32;
  auto go = [&](auto P, auto G, auto M) {
    constexpr bool p_ = decltype(P)::value, g_ = decltype(G)::value, m_ = decltype(M)::value;
    if (Q8) aw_chunk8<p_, g_, m_>(t, s, i0, tid);
    else aw_chunk32<p_, g_, m_>(t, s, i0, tid);
  };
  if (p32) {
    if (g32) go(std::true_type{}, std::true_type{}, std::false_type{});
    else go(std::true_type{}, std::false_type{}, std::false_type{});
  } else if (t.master) {
    if (g32) go(std::false_type{}, std::true_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{}, std::true_type{});
  } else {
    if (g32) go(std::false_type{}, std::true_type{}, std::false_type{});
    else go(std::false_type{}, std::false_type{}, std::false_type{});
  }
}

// ---- the values that 8-bit states stand for ----
__global__ __launch_bounds__(256) void aw_values_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales,
                                                        float* __restrict__ out, int64_t n, int is_signed) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const double sc = (double)scales[i / AW_BLOCK];
  uint32_t w = 0;
  const int left = (int)min((int64_t)4, n - i);
  if (left == 4) w = *(const uint32_t*)(codes + i);
  else
    for (int e = 0; e < left; ++e) w |= (uint32_t)codes[i + e] << (8 * e);
  f32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = (w >> (8 * e)) & 255;
    o[e] = (float)(is_signed ? aw_value_m((int)(int8_t)c, sc) : aw_value_v(c, sc));
  }
  if (left == 4) *(f32x4*)(out + i) = o;
  else
    for (int e = 0; e < left; ++e) out[i + e] = o[e];
}

static int64_t aw_parts(const strata_hip_adamw_tensor* t, int64_t count) {
  int64_t parts = 0;
  for (int64_t i = 0; i < count; ++i) parts += t[i].n > 0 ? (t[i].n + AW_SUM - 1) / AW_SUM : 0;
  return parts;
}

// The distinct step counts of a call (`of`: which one each tensor has), in the order of their first tensors.
struct AwSteps {
  std::vector<int64_t*> each;
  std::vector<uint32_t> of;
};

static void aw_steps(const strata_hip_adamw_args* a, int64_t* const* steps, AwSteps& s) {
  if (!steps) {
    s.each.push_back(a->step);
    return;
  }
  std::unordered_map<int64_t*, uint32_t> seen;
  s.of.resize((size_t)a->count);
  for (int64_t i = 0; i < a->count; ++i) {
    const auto at = seen.emplace(steps[i], (uint32_t)s.each.size());
    if (at.second) s.each.push_back(steps[i]);
    s.of[(size_t)i] = at.first->second;
  }
}

static int aw_check(const strata_hip_adamw_args* a, const AwSteps& steps) {
  for (const int64_t* step : steps.each)
    if (!step || ((uintptr_t)step & 7)) return fail(STRATA_HIP_EINVAL, "adamw_step: step must be given, 8-byte aligned");
  if (!a->workspace || ((uintptr_t)a->workspace & 7))
    return fail(STRATA_HIP_EINVAL, "adamw_step: workspace must be given, 8-byte aligned");
  if (steps.each.size() > 0xffffff) return fail(STRATA_HIP_EUNSUPPORTED, "adamw_step: too many step counts for one call");
  if (!(a->beta1 >= 0. && a->beta1 < 1. && a->beta2 >= 0. && a->beta2 < 1.))
    return fail(STRATA_HIP_EINVAL, "adamw_step: betas must lie in [0, 1)");
  if (!(a->eps >= 0.) || !std::isfinite(a->eps))
    return fail(STRATA_HIP_EINVAL, "adamw_step: eps must be finite and not negative");
  if (!std::isfinite(a->max_norm) || (a->max_norm > 0. && (!a->norm || ((uintptr_t)a->norm & 7))))
    return fail(STRATA_HIP_EINVAL, "adamw_step: max_norm must be finite and norm given with it, 8-byte aligned");
  std::vector<std::pair<uintptr_t, uintptr_t>> written, read;
  written.reserve((size_t)a->count * 6 + steps.each.size());
  read.reserve((size_t)a->count);
  for (const int64_t* step : steps.each) written.emplace_back((uintptr_t)step, (uintptr_t)step + 8);
  int64_t chunks = 0;
  for (int64_t i = 0; i < a->count; ++i) {
    const strata_hip_adamw_tensor& t = a->tensors[i];
    if (t.n < 0) return fail(STRATA_HIP_EINVAL, "adamw_step: negative size");
    if (t.n == 0) continue;
    if (!std::isfinite(t.lr) || !std::isfinite(t.weight_decay))
      return fail(STRATA_HIP_EINVAL, "adamw_step: lr and weight_decay must be finite");
    const bool p32 = t.param_dtype == STRATA_HIP_F32, g32 = t.grad_dtype == STRATA_HIP_F32;
    if ((!p32 && t.param_dtype != STRATA_HIP_BF16) || (!g32 && t.grad_dtype != STRATA_HIP_BF16))
      return fail(STRATA_HIP_EINVAL, "adamw_step: parameters and gradients must be bf16 or f32");
    if (t.state_bits != 32 && t.state_bits != 8) return fail(STRATA_HIP_EINVAL, "adamw_step: state_bits must be 32 or 8");
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return fail(STRATA_HIP_EINVAL, "adamw_step: null tensor");
    if (t.state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale))
      return fail(STRATA_HIP_EINVAL, "adamw_step: 8-bit states need their scales");
    if (p32 && t.master) return fail(STRATA_HIP_EINVAL, "adamw_step: master weights are for bf16 parameters");
    const uintptr_t ps = p32 ? 4 : 2, gs = g32 ? 4 : 2, ss = t.state_bits / 8;
    if (((uintptr_t)t.param % ps) || ((uintptr_t)t.grad % gs) || ((uintptr_t)t.exp_avg % ss) || ((uintptr_t)t.exp_avg_sq % ss) ||
        ((uintptr_t)t.master % 4) || ((uintptr_t)t.exp_avg_scale % 4) || ((uintptr_t)t.exp_avg_sq_scale % 4))
      return fail(STRATA_HIP_EINVAL, "adamw_step: a tensor is not aligned to its elements");
    auto add = [&](const void* p, uintptr_t bytes) { written.emplace_back((uintptr_t)p, (uintptr_t)p + bytes); };
    read.emplace_back((uintptr_t)t.grad, (uintptr_t)t.grad + gs * t.n);
    add(t.param, ps * t.n);
    add(t.exp_avg, ss * t.n);
    add(t.exp_avg_sq, ss * t.n);
    if (t.master) add(t.master, 4 * t.n);
    if (t.state_bits == 8) {
      add(t.exp_avg_scale, 4 * ((t.n + AW_BLOCK - 1) / AW_BLOCK));
      add(t.exp_avg_sq_scale, 4 * ((t.n + AW_BLOCK - 1) / AW_BLOCK));
    }
    chunks += (t.n + AW_CHUNK - 1) / AW_CHUNK;
  }
  if (chunks > 0xffffff) return fail(STRATA_HIP_EUNSUPPORTED, "adamw_step: too many elements for one call");
  return check_ranges("adamw_step", written, read);
}

static int aw_launch(const strata_hip_adamw_args* a, int64_t* const* steps, hipStream_t st) {
  if (!a) return fail(STRATA_HIP_EINVAL, "adamw_step: null args");
  if (a->count < 0 || (a->count > 0 && !a->tensors)) return fail(STRATA_HIP_EINVAL, "adamw_step: bad tensor list");
  AwSteps counts;
  aw_steps(a, steps, counts);
  if (const int rc = aw_check(a, counts)) return rc;
  double* part = a->workspace + AW_HEAD;
  int64_t parts = 0;
  if (a->max_norm > 0.) {
    SumBatch b;
    b.count = 0;
    uint32_t wgs = 0;
    auto flush = [&]() -> int {
      if (!b.count) return STRATA_HIP_OK;
      b.part = part + parts;
      hipLaunchKernelGGL(aw_sum_kernel, dim3(wgs), dim3(256), 0, st, b);
      parts += wgs;
      b.count = 0;
      wgs = 0;
      return check_launch("adamw sum of squares");
    };
    for (int64_t i = 0; i < a->count; ++i) {
      const strata_hip_adamw_tensor& t = a->tensors[i];
      if (t.n == 0) continue;
      const int k = b.count++;
      b.g[k] = t.grad;
      b.n[k] = t.n;
      b.first[k] = wgs;
      b.wide[k] = (t.grad_dtype == STRATA_HIP_F32 ? 1u : 0u) | (((uintptr_t)t.grad & 15) ? 0u : 2u);
      wgs += (uint32_t)((t.n + AW_SUM - 1) / AW_SUM);
      if (b.count == 3 * AW_PER)
        if (const int rc = flush()) return rc;
    }
    if (const int rc = flush()) return rc;
  }
  const bool clip = a->max_norm > 0.;
  const AwNorm norm = {part, parts, clip ? a->norm : nullptr, a->max_norm, a->beta1, a->beta2};
  double* heads = a->workspace;
  if (counts.each.size() == 1) {
    hipLaunchKernelGGL(aw_head_kernel, dim3(1), dim3(1024), 0, st, norm, heads, counts.each[0]);
    if (const int rc = check_launch("adamw head")) return rc;
  } else {
    heads = part + aw_parts(a->tensors, a->count);
    AwCounts c;
    size_t k = 0;
    do {  // without a tensor: the norm alone
      c.count = (int)std::min(counts.each.size() - k, (size_t)AW_COUNTS);
      std::copy_n(counts.each.begin() + k, c.count, c.step);
      hipLaunchKernelGGL(aw_heads_kernel, dim3(1), dim3(1024), 0, st, norm, heads + 4 * k, c);
      if (const int rc = check_launch("adamw heads")) return rc;
      k += AW_COUNTS;
    } while (k < counts.each.size());
  }
  AwBatch b;
  b.count = 0;
  b.eps = (float)a->eps;
  b.b1 = a->beta1;
  b.b2 = a->beta2;
  b.head = heads;
  for (const bool q8 : {false, true}) {  // a launch takes tensors of one kind of moments
    uint32_t wgs = 0;
    auto flush = [&]() -> int {
      if (!b.count) return STRATA_HIP_OK;
      if (q8) hipLaunchKernelGGL(aw_step_kernel<true>, dim3(wgs), dim3(256), 0, st, b);
      else hipLaunchKernelGGL(aw_step_kernel<false>, dim3(wgs), dim3(256), 0, st, b);
      b.count = 0;
      wgs = 0;
      return check_launch("adamw step");
    };
    for (int64_t i = 0; i < a->count; ++i) {
      const strata_hip_adamw_tensor& t = a->tensors[i];
      if (t.n == 0 || (t.state_bits == 8) != q8) continue;
      AwTensor& o = b.t[b.count++];
      o.p = t.param;
      o.g = t.grad;
      o.m = t.exp_avg;
      o.v = t.exp_avg_sq;
      o.ms = t.exp_avg_scale;
      o.vs = t.exp_avg_sq_scale;
      o.master = t.master;
      o.n = t.n;
      o.lr = (float)t.lr;
      o.decay = (float)(1. - t.lr * t.weight_decay);
      o.first = wgs;
      const uintptr_t all = (uintptr_t)t.param | (uintptr_t)t.grad | (uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq | (uintptr_t)t.master;
      o.flags = (t.param_dtype == STRATA_HIP_F32 ? AW_P32 : 0) | (t.grad_dtype == STRATA_HIP_F32 ? AW_G32 : 0) |
                ((all & 15) ? 0 : AW_ALIGNED) | (steps ? counts.of[(size_t)i] << AW_COUNT_SHIFT : 0);
      wgs += (uint32_t)((t.n + AW_CHUNK - 1) / AW_CHUNK);
      if (b.count == AW_PER)
        if (const int rc = flush()) return rc;
    }
    if (const int rc = flush()) return rc;
  }
  return STRATA_HIP_OK;
}

}  // namespace strata

extern "C" int64_t strata_hip_adamw_workspace(const strata_hip_adamw_tensor* tensors, int64_t count) {
  if (!tensors || count <= 0) return strata::AW_HEAD;
  return strata::AW_HEAD + strata::aw_parts(tensors, count);
}

extern "C" int strata_hip_adamw_step(const strata_hip_adamw_args* a, void* stream) {
  try {
    return strata::aw_launch(a, nullptr, (hipStream_t)stream);
  } catch (const std::exception&) {  // no memory for the lists, or more than a list can hold
    return strata::fail(STRATA_HIP_EUNSUPPORTED, "adamw_step: out of host memory");
  }
}

extern "C" int strata_hip_adamw_step_counts(const strata_hip_adamw_args* a, int64_t* const* steps, void* stream) {
  if (!steps) return strata::fail(STRATA_HIP_EINVAL, "adamw_step: null steps");
  try {
    return strata::aw_launch(a, steps, (hipStream_t)stream);
  } catch (const std::exception&) {  // no memory for the lists, or more than a list can hold
    return strata::fail(STRATA_HIP_EUNSUPPORTED, "adamw_step: out of host memory");
  }
}

extern "C" int strata_hip_adamw_state_values(const strata_hip_adamw_values_args* a, void* stream) {
  using namespace strata;
  if (!a) return fail(STRATA_HIP_EINVAL, "adamw_state_values: null args");
  if (a->n < 0) return fail(STRATA_HIP_EINVAL, "adamw_state_values: negative size");
  if (a->n == 0) return STRATA_HIP_OK;
  if (!a->codes || !a->scales || !a->out) return fail(STRATA_HIP_EINVAL, "adamw_state_values: null pointer");
  if (((uintptr_t)a->codes & 3) || ((uintptr_t)a->scales & 3) || ((uintptr_t)a->out & 15))
    return fail(STRATA_HIP_EINVAL, "adamw_state_values: codes must be 4-byte, out 16-byte aligned");
  const int64_t wgs = (a->n + 1023) / 1024;
  if (wgs > 0xffffff) return fail(STRATA_HIP_EUNSUPPORTED, "adamw_state_values: too many elements for one call");
  hipLaunchKernelGGL(aw_values_kernel, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)a->codes,
                     a->scales, a->out, a->n, a->is_signed);
  return check_launch("adamw state values");
}
