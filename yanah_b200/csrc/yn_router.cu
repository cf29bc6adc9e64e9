// Routing of rows of router logits by a rule (softmax or sigmoid scores, a
// balance bias, groups of experts, top k, renormalised weights), and its C ABI.
// No counterpart in the reference, whose routers are softmax top-k without a
// bias (mlx_backend.py:308-316; that form is yn_route).
//
// Mathematics, per row of logits z: s_e = exp(z_e - m) / sum or 1 / (1 +
// exp(-z_e)); c_e = s_e + b_e orders the experts; a group's score is the sum of
// its `group_top` largest c; the k largest c inside the `top_groups` best groups
// are chosen (ties: lower id first) and weighted by s, not c.
//
// The order is that of exact arithmetic, as far as 64 bits have it. Without a bias and groups c is a
// monotone function of z, so the logits themselves are compared. Otherwise the
// row is ordered in fp32, whose error on c is bounded (below); only where two
// neighbours of the chosen order, or the last group in and the first one out,
// are nearer than that bound are the candidates, or the groups, ordered in fp64.
//
// One warp per row, keys in registers: L = 32 / (groups rounded up to a power of
// two) lanes hold one group, element i of a lane being expert
// (lane / L) * per_group + lane % L + i * L; where the groups fill their lanes and the
// row is aligned, a lane has consecutive experts instead, read in wide pieces (16384 x
// 256 in 8 groups, bias: 19.5 us, 24.0 one by one with the groups ranked by shuffles).
// A row is at most 4 KB, so the kernel is bound by issuing instructions (three quarters
// of all cycles, 1.4 us of memory traffic), not by memory, and more warps per SM change
// nothing (10 or 12 blocks: 24.0 and 24.8 us then). The choice takes few of them: the
// k-th largest of the 32 lane maxima (k redux) bounds the k-th largest key from
// below; the keys that reach it, little more than k, are gathered one per lane and
// placed by counting the larger ones.
#include <cuda_runtime.h>

#include <string>
#include <type_traits>

#include "yanah_b200.h"
#include "yn_common.cuh"
#include "yn_internal.h"

namespace ynb {

constexpr int RT_WARPS = 4;          // rows per block
constexpr int RT_MAX_E = 1024;
constexpr int RT_MAX_K = 31;         // lane k holds the first expert not chosen
constexpr uint32_t RT_NONE = 0x007FFFFFu;   // f32_ukey(-inf): experts that take no part

struct RouterArgs {
  const void* z;
  long long ld;
  long long rows;
  const float* bias;
  const uint8_t* avail;
  int32_t* ids;
  float* w;
  int E, K, G, per, L, log_l, kept, group_top;
  bool softmax, norm;
  float scale;
};

template <typename T>
YN_DEV float rt_load(const void* z, long long i);
template <>
YN_DEV float rt_load<float>(const void* z, long long i) { return __ldg(reinterpret_cast<const float*>(z) + i); }
template <>
YN_DEV float rt_load<__nv_bfloat16>(const void* z, long long i) {
  return bf16_to_f32(__ldg(reinterpret_cast<const uint16_t*>(z) + i));
}
template <>
YN_DEV float rt_load<__half>(const void* z, long long i) {
  return f16_to_f32(__ldg(reinterpret_cast<const uint16_t*>(z) + i));
}

// N consecutive values in pieces of up to 16 bytes.
template <int N, typename T>
YN_DEV void rt_load_wide(const T* p, float (&v)[N]) {
  constexpr int W = N * sizeof(T) < 16 ? N * sizeof(T) / 4 : 4, PER = 4 / sizeof(T);   // words of a piece, values of a word
#pragma unroll
  for (int i = 0; i < N; i += W * PER) {
    uint32_t w[W];
    if constexpr (W == 1) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p + i));
    } else if constexpr (W == 2) {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(p + i));
      w[0] = q.x, w[1] = q.y;
    } else {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p + i));
      w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    }
#pragma unroll
    for (int j = 0; j < W * PER; ++j) {
      if constexpr (sizeof(T) == 4) v[i + j] = __uint_as_float(w[j]);
      else if constexpr (std::is_same_v<T, __half>) v[i + j] = f16_to_f32((uint16_t)(w[j / 2] >> (16 * (j & 1))));
      else v[i + j] = __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
    }
  }
}

YN_DEV double warp_max_f64(double v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, m));
  return v;
}
YN_DEV double warp_sum_f64(double v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
// 2^x and 1 / (1 + e^-z) by the hardware's approximations (2 and 1 ulp; 0 below 2^-126).
YN_DEV float rt_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float RT_LOG2E = 1.44269504088896341f;
YN_DEV float rt_sigmoid(float z) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + rt_ex2(-RT_LOG2E * z)));
  return r;
}

// A lane's part of a row: its elements are experts first + (i << log_l), i < count.
struct RtLane {
  int first, count;
  YN_DEV RtLane(const RouterArgs& a, int lane) {
    const int g = lane >> a.log_l, at = lane & (a.L - 1);
    first = g * a.per + at;
    count = g < a.G && at < a.per ? (a.per - at + a.L - 1) >> a.log_l : 0;
  }
};

// The two largest values of the lane, merged over the L lanes of its group, as the group's score.
template <typename F>
YN_DEV F rt_group_score(const RouterArgs& a, F hi, F lo, F none) {
  for (int m = 1; m < a.L; m <<= 1) {
    const F h2 = __shfl_xor_sync(0xffffffffu, hi, m), l2 = __shfl_xor_sync(0xffffffffu, lo, m);
    const F mn = hi < h2 ? hi : h2, mx = hi < h2 ? h2 : hi, l = lo < l2 ? l2 : lo;
    hi = mx;
    lo = mn < l ? l : mn;
  }
  return a.group_top > 1 && lo != none ? hi + lo : hi;
}
// Whether the lane's group is among the `kept` best by score, ties to the lower group.
YN_DEV bool rt_group_kept_f64(const RouterArgs& a, int lane, double score) {
  const int g = lane >> a.log_l;
  int rank = 0;
  for (int o = 0; o < a.G; ++o) {
    const double s = __shfl_sync(0xffffffffu, score, o << a.log_l);
    rank += s > score || (s == score && o < g);
  }
  return g < a.G && rank < a.kept;
}
// The same in fp32, a redux per kept group. far: the distance between the last group in and the
// first one out.
YN_DEV bool rt_group_kept(const RouterArgs& a, int lane, float score, float* far) {
  const int g = lane >> a.log_l;
  uint32_t k = g < a.G && (lane & (a.L - 1)) == 0 ? f32_ukey(score) : 0u, top = 0, groups = 0;
  for (int j = 0; j < a.kept; ++j) {
    top = __reduce_max_sync(0xffffffffu, k);
    const int w = __ffs(__ballot_sync(0xffffffffu, k == top)) - 1;
    groups |= 1u << (w >> a.log_l);
    if (lane == w) k = 0;
  }
  const uint32_t out = __reduce_max_sync(0xffffffffu, k);
  *far = out <= RT_NONE ? __int_as_float(0x7f800000) : f32_from_ukey(top) - f32_from_ukey(out);
  return (groups >> g) & 1u;
}

// A row's scores in fp64: 1 / sum exp(z - m) of a softmax (1 for sigmoids).
template <typename T>
YN_DEV double rt_inv_sum_f64(const RouterArgs& a, const RtLane& own, long long row, double m) {
  double sum = 0.0;
  for (int i = 0; i < own.count; ++i) {
    const int e = own.first + (i << a.log_l);
    const double z = rt_load<T>(a.z, row * a.ld + e);
    if (z > -__longlong_as_double(0x7ff0000000000000LL) && (!a.avail || a.avail[e])) sum += z == m ? 1.0 : exp(z - m);
  }
  return 1.0 / warp_sum_f64(sum);
}
// Choice value of expert e, which takes part; -inf where its bias takes it out.
template <typename T>
YN_DEV double rt_choice_f64(const RouterArgs& a, long long row, int e, double m, double inv) {
  const double z = rt_load<T>(a.z, row * a.ld + e);
  const double s = !a.softmax ? 1.0 / (1.0 + exp(-z)) : z == m ? inv : exp(z - m) * inv;
  if (!a.bias) return s;
  const double none = -__longlong_as_double(0x7ff0000000000000LL), c = s + (double)a.bias[e];
  return c > none ? c : none;
}

// The groups kept, decided in fp64.
template <typename T>
__device__ __noinline__ bool rt_groups_f64(const RouterArgs& a, long long row, int lane, double m) {
  const double none = -__longlong_as_double(0x7ff0000000000000LL);
  const RtLane own(a, lane);
  const double inv = a.softmax ? rt_inv_sum_f64<T>(a, own, row, m) : 1.0;
  double hi = none, lo = none;
  for (int i = 0; i < own.count; ++i) {
    const int e = own.first + (i << a.log_l);
    const float z = rt_load<T>(a.z, row * a.ld + e);
    if (!(z > -__int_as_float(0x7f800000)) || (a.avail && !a.avail[e])) continue;
    const double c = rt_choice_f64<T>(a, row, e, m, inv);
    if (c > hi) { lo = hi; hi = c; }
    else if (c > lo) lo = c;
  }
  return rt_group_kept_f64(a, lane, rt_group_score(a, hi, lo, none));
}

// The place of this lane's candidate (id, or -1) among the n <= 32 candidates, by fp64.
template <typename T>
__device__ __noinline__ int rt_place_f64(const RouterArgs& a, long long row, int lane, int id, int n, double m) {
  const double none = -__longlong_as_double(0x7ff0000000000000LL);
  const double inv = a.softmax ? rt_inv_sum_f64<T>(a, RtLane(a, lane), row, m) : 1.0;
  const double c = id >= 0 ? rt_choice_f64<T>(a, row, id, m, inv) : none;
  int place = 0;
  for (int q = 0; q < n; ++q) {
    const double o = __shfl_sync(0xffffffffu, c, q);
    const int oid = __shfl_sync(0xffffffffu, id, q);
    place += o > c || (o == c && oid < id);
  }
  return place;
}

// The row's choice from the values of the kept groups in fp64, one after another; lane
// j < K returns the id at place j. For rows with more near candidates than lanes.
template <typename T>
__device__ __noinline__ int rt_choose_f64(const RouterArgs& a, long long row, int lane, bool in, double m, double* val) {
  const double none = -__longlong_as_double(0x7ff0000000000000LL);
  const RtLane own(a, lane);
  const double inv = a.softmax ? rt_inv_sum_f64<T>(a, own, row, m) : 1.0;
  for (int i = 0; i < own.count; ++i) {
    const int e = own.first + (i << a.log_l);
    const float z = rt_load<T>(a.z, row * a.ld + e);
    const bool on = in && z > -__int_as_float(0x7f800000) && (!a.avail || a.avail[e]);
    val[e] = on ? rt_choice_f64<T>(a, row, e, m, inv) : none;
  }
  int mine = -1;
  for (int j = 0; j < a.K; ++j) {
    double best = none;
    int at = RT_MAX_E;
    for (int i = 0; i < own.count; ++i) {
      const int e = own.first + (i << a.log_l);
      if (val[e] > best) { best = val[e]; at = e; }
    }
    const double top = warp_max_f64(best);
    const int id = (int)__reduce_min_sync(0xffffffffu, best == top ? (unsigned)at : (unsigned)RT_MAX_E);
    if (top == none) break;
    if (at == id) val[id] = none;
    if (lane == j) mine = id;
  }
  return mine;
}

// NV: elements per lane. BY_SCORE: the order needs the scores (a bias or groups);
// otherwise the logits order the experts.
// WHOLE: the row has 32 * NV experts, whose groups fill their lanes, and is aligned: a lane
// takes NV consecutive ones in wide loads and asks for no bounds.
template <typename T, int NV, bool BY_SCORE, bool WHOLE>
__global__ void __launch_bounds__(32 * RT_WARPS) k_router(const RouterArgs a) {
  extern __shared__ double rt_smem[];   // BY_SCORE: E doubles per warp
  __shared__ unsigned long long cand[RT_WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * RT_WARPS + warp;
  if (row >= a.rows) return;
  const float inf = __int_as_float(0x7f800000);
  const RtLane own(a, lane);
  const int first = WHOLE ? NV * lane : own.first;
  auto expert = [&](int i) { return WHOLE ? first + i : first + (i << a.log_l); };
  auto there = [&](int i) { return WHOLE || i < own.count; };
  float v[NV];
  if (WHOLE) {
    rt_load_wide<NV>(reinterpret_cast<const T*>(a.z) + row * a.ld + first, v);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = there(i) ? rt_load<T>(a.z, row * a.ld + expert(i)) : -inf;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = fmaxf(v[i], -inf);   // NaN too
  if (a.avail) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (there(i) && !a.avail[expert(i)]) v[i] = -inf;
  }
  float m = -inf, sum = 0.0f, tol = 0.0f;
  if (BY_SCORE || (a.softmax && !a.norm)) {
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, v[i]);
    m = f32_from_ukey(__reduce_max_sync(0xffffffffu, f32_ukey(m)));
    if (a.softmax) {
#pragma unroll
      for (int i = 0; i < NV; ++i)   // all +inf logits share the mass
        sum += v[i] == -inf ? 0.0f : v[i] == m ? 1.0f : rt_ex2((v[i] - m) * RT_LOG2E);
      sum = warp_sum_f32(sum);
    }
  }
  uint32_t key[NV];
  bool in = true;   // the lane's group is kept
  if (BY_SCORE) {
    // |c - exact| <= tol + 2^-24 |c|, tol relative to the row's largest score: e^x as
    // 2^(x log2 e) is off by 2 ulp and the rounding of its exponent, 1.2 |x| ulp, and |x| e^x
    // <= 0.4 for x <= 0, so the exponentials stay within 2^-21 of the largest; the softmax sum
    // of at most 64 terms a lane and 5 shuffled adds within 69 * 2^-24 < 5e-6 of itself. Sigmoids of
    // a row whose largest logit m is far below 0 are e^z too, relative to a largest score of e^m: the
    // exponent's rounding and that of log2 e are 7.3e-8 |z| of e^z, which is largest at m (|z| e^z
    // falls from z = -1 on; 0.4 is its maximum). Scores below 1e-30 are not told apart.
    const float inv = a.softmax ? 1.0f / sum : 1.0f;
    tol = (a.softmax ? 1.6e-5f * inv : (2.0e-6f + 1.0e-7f * fminf(fmaxf(-m, 0.0f), 100.0f)) * rt_sigmoid(m)) + 1e-30f;
    float hi = -inf, lo = -inf, b[NV];
    if (WHOLE && a.bias) {
      rt_load_wide<NV>(a.bias + first, b);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) b[i] = a.bias && there(i) ? __ldg(a.bias + expert(i)) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float s = a.softmax ? (v[i] == m ? inv : rt_ex2((v[i] - m) * RT_LOG2E) * inv) : rt_sigmoid(v[i]);
      const float c = v[i] > -inf ? fmaxf(s + b[i], -inf) : -inf;   // a bias of -inf or NaN takes the expert out
      lo = fmaxf(lo, fminf(hi, c));
      hi = fmaxf(hi, c);
      // without a bias the logits have the scores' order, exactly
      key[i] = f32_ukey(a.bias ? c : v[i]);
    }
    if (a.G > 1) {
      float far;
      in = rt_group_kept(a, lane, rt_group_score(a, hi, lo, -inf), &far);
      // the largest of the lanes' two values: a score's terms are rounded by 2^-24 of theirs
      const float mag = __uint_as_float(__reduce_max_sync(
          0xffffffffu, __float_as_uint(hi == -inf ? 0.0f : lo == -inf ? fabsf(hi) : fmaxf(fabsf(hi), fabsf(lo)))));
      if (far <= 4.0f * tol + 5.0e-7f * mag) in = rt_groups_f64<T>(a, row, lane, (double)m);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = f32_ukey(v[i]);
  }
  // The first K (one more where neighbours are compared), descending, ties to the lower id.
  const bool compared = BY_SCORE && a.bias;
  const int places = compared ? a.K + 1 : a.K;
  uint32_t cur = 0, bound = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) cur = max(cur, key[i]);
  cur = in ? cur : 0u;
  for (int j = 0; j < places; ++j) {
    bound = __reduce_max_sync(0xffffffffu, cur);
    if (cur == bound) cur = 0;   // equal lane maxima go together: the bound is lower then, and still one
  }
  if (compared && bound > RT_NONE) {   // whatever might be as large as the bound in exact arithmetic is a candidate too
    const float c = f32_from_ukey(bound);
    bound = f32_ukey(fmaxf(c - 2.0f * tol - 2.5e-7f * fabsf(c), -3.402823466e38f));
  }
  bound = in ? max(bound, RT_NONE + 1u) : ~0u;
  // one lane's candidates side by side, the lanes one after another (their order does not matter)
  int own_n = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) own_n += key[i] >= bound;
  const unsigned below = (1u << lane) - 1u;
  const unsigned b1 = __ballot_sync(0xffffffffu, own_n > 0), b2 = __ballot_sync(0xffffffffu, own_n > 1);
  int at = __popc(b1 & below) + __popc(b2 & below), n = __popc(b1) + __popc(b2);
  for (int q = 2; __any_sync(0xffffffffu, own_n > q); ++q) {   // three or more in one lane: seldom
    const unsigned bq = __ballot_sync(0xffffffffu, own_n > q);
    at += __popc(bq & below);
    n += __popc(bq);
  }
  if (n <= 32) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (key[i] >= bound)
        cand[warp][at++] = ((unsigned long long)key[i] << 32) | (0xFFFFFFFFu - (uint32_t)expert(i));
  }
  int mine = -1;
  uint32_t my_key = 0;
  __syncwarp();
  if (n <= 32) {
    const unsigned long long c = lane < n ? cand[warp][lane] : 0;
    int place = 0;
#pragma unroll 4
    for (int q = 0; q < n; ++q) place += cand[warp][q] > c;
    __syncwarp();
    if (lane < n) cand[warp][place] = c;
    __syncwarp();
    if (lane < n) {
      mine = (int)(0xFFFFFFFFu - (uint32_t)cand[warp][lane]);
      my_key = (uint32_t)(cand[warp][lane] >> 32);
    }
  } else {
    // many near keys, or k near 32: one after another, two redux each
    for (int j = 0; j < places; ++j) {
      uint32_t best = RT_NONE;
      int bi = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in && key[i] > best) { best = key[i]; bi = i; }
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      if (top == RT_NONE) break;
      const int e = best == top ? expert(bi) : RT_MAX_E;
      const int id = (int)__reduce_min_sync(0xffffffffu, (unsigned)e);
      if (e == id) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (i == bi) key[i] = 0;
      }
      if (lane == j) { mine = id; my_key = top; }
    }
  }
  float z = mine >= 0 ? rt_load<T>(a.z, row * a.ld + mine) : -inf;
  if (compared) {
    const int nid = __shfl_down_sync(0xffffffffu, mine, 1);
    const uint32_t nk = __shfl_down_sync(0xffffffffu, my_key, 1);
    bool near = false;
    if (lane < a.K && mine >= 0 && nid >= 0) {   // K < 32: lane K has the first one left out
      const float c = f32_from_ukey(my_key), nc = f32_from_ukey(nk);
      near = c - nc <= 2.0f * tol + 2.5e-7f * fmaxf(fabsf(c), fabsf(nc));
      // equal logits with equal biases are equal in exact arithmetic too, except at the last place: what is
      // near the first one left out is not looked at
      if (near && lane < a.K - 1)
        near = z != rt_load<T>(a.z, row * a.ld + nid) || __ldg(a.bias + mine) != __ldg(a.bias + nid);
    }
    if (__any_sync(0xffffffffu, near)) {
      if (n <= 32) {
        const int place = rt_place_f64<T>(a, row, lane, mine, n, (double)m);
        __syncwarp();
        if (lane < n) cand[warp][place] = (unsigned long long)mine;
        __syncwarp();
        if (lane < n) mine = (int)cand[warp][lane];
      } else {
        mine = rt_choose_f64<T>(a, row, lane, in, (double)m, rt_smem + (size_t)warp * a.E);
      }
      z = mine >= 0 ? rt_load<T>(a.z, row * a.ld + mine) : -inf;
    }
  }
  if (lane >= a.K) { mine = -1; z = -inf; }
  // Weights from the chosen logits alone, relative to the largest of them (M) where
  // they are renormalised, so that scores far below the row's largest keep their ratio.
  float w;
  if (a.norm) {
    const float M = f32_from_ukey(__reduce_max_sync(0xffffffffu, f32_ukey(z)));
    const bool rel = a.softmax || M < 0.0f;
    const float e = expf(rel ? (z == M ? 0.0f : z - M) : -z);   // z = -inf: 0, or infinity
    w = a.softmax ? e : __fdividef(rel ? e : 1.0f, 1.0f + (rel ? expf(z) : e));
    w = z == -inf ? 0.0f : w;
    const float t = warp_sum_f32(w);
    w = t > 0.0f ? __fdividef(w, t) * a.scale : 0.0f;
  } else {
    if (a.softmax) w = z == -inf ? 0.0f : (z == m ? 1.0f : expf(z - m)) / sum * a.scale;
    else w = z == -inf ? 0.0f : 1.0f / (1.0f + expf(-z)) * a.scale;
  }
  if (lane < a.K) {
    a.ids[row * a.K + lane] = mine;
    a.w[row * a.K + lane] = w;
  }
}

template <typename T, int NV, bool BY_SCORE>
void launch_router_nv(const RouterArgs& a, dim3 grid, size_t smem, cudaStream_t st) {
  const dim3 b(32 * RT_WARPS);
  constexpr size_t ZA = NV * sizeof(T) < 16 ? NV * sizeof(T) : 16, BA = NV * 4 < 16 ? NV * 4 : 16;
  // groups that are a power of two fill their lanes
  const bool whole = a.E == 32 * NV && a.G * a.L == 32 && reinterpret_cast<uintptr_t>(a.z) % ZA == 0 &&
                     (a.ld * sizeof(T)) % ZA == 0 && reinterpret_cast<uintptr_t>(a.bias) % BA == 0;
  if constexpr (NV <= 32) {
    if (whole) {
      k_router<T, NV, BY_SCORE, true><<<grid, b, smem, st>>>(a);
      return;
    }
  }
  k_router<T, NV, BY_SCORE, false><<<grid, b, smem, st>>>(a);
}

template <typename T, bool BY_SCORE>
void launch_router(const RouterArgs& a, int nv, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.rows + RT_WARPS - 1) / RT_WARPS);
  const size_t smem = BY_SCORE ? (size_t)RT_WARPS * a.E * sizeof(double) : 0;
  if (nv <= 2) launch_router_nv<T, 2, BY_SCORE>(a, grid, smem, st);
  else if (nv <= 4) launch_router_nv<T, 4, BY_SCORE>(a, grid, smem, st);
  else if (nv <= 8) launch_router_nv<T, 8, BY_SCORE>(a, grid, smem, st);
  else if (nv <= 16) launch_router_nv<T, 16, BY_SCORE>(a, grid, smem, st);
  else if (nv <= 32) launch_router_nv<T, 32, BY_SCORE>(a, grid, smem, st);
  else launch_router_nv<T, 64, BY_SCORE>(a, grid, smem, st);
}

}  // namespace ynb

using namespace ynb;

extern "C" int yn_route_scored(const yn_route_rule* rule, const void* logits, int32_t dtype, int64_t row_stride,
                               int64_t rows, const float* bias, const uint8_t* available, int32_t* ids,
                               float* weights, void* stream) {
  if (!rule) return host_fail(YN_E_INVALID, "null argument");
  const yn_route_rule& r = *rule;
  if (r.n_experts < 1 || r.top_k < 1 || r.top_k > r.n_experts)
    return host_fail(YN_E_INVALID, "top_k must be in [1, n_experts]");
  if (r.n_experts > RT_MAX_E || r.top_k > RT_MAX_K)
    return host_fail(YN_E_UNSUPPORTED, "at most 1024 experts and top_k 31");
  if (r.score != YN_SCORE_SOFTMAX && r.score != YN_SCORE_SIGMOID)
    return host_fail(YN_E_INVALID, "score must be YN_SCORE_SOFTMAX or YN_SCORE_SIGMOID");
  if (r.n_groups < 1 || r.n_experts % r.n_groups || r.top_groups < 1 || r.top_groups > r.n_groups)
    return host_fail(YN_E_INVALID, "n_groups must divide n_experts, top_groups must be in [1, n_groups]");
  if (r.n_groups > 32) return host_fail(YN_E_UNSUPPORTED, "at most 32 groups");
  if (r.group_top != 1 && r.group_top != 2) return host_fail(YN_E_INVALID, "group_top must be 1 or 2");
  if (r.top_k > r.top_groups * (r.n_experts / r.n_groups))
    return host_fail(YN_E_INVALID, "top_k is larger than the kept groups");
  if (dtype != YN_F32 && dtype != YN_BF16 && dtype != YN_F16) return host_fail(YN_E_INVALID, "unknown dtype");
  if (rows < 0 || rows > 0x7fffffffLL || row_stride < r.n_experts)
    return host_fail(YN_E_INVALID, "rows must be in [0, 2^31), row_stride at least n_experts");
  if (rows == 0) return YN_OK;
  if (!logits || !ids || !weights) return host_fail(YN_E_INVALID, "null argument");
  if (!host_aligned(dtype == YN_F32 ? 4 : 2, logits) || !host_aligned(4, bias, ids, weights))
    return host_fail(YN_E_INVALID, "logits, bias, ids and weights must be aligned to their elements");
  RouterArgs a{};
  a.z = logits;
  a.ld = row_stride;
  a.rows = rows;
  a.bias = bias;
  a.avail = available;
  a.ids = ids;
  a.w = weights;
  a.E = r.n_experts;
  a.K = r.top_k;
  // keeping every group is the same as having none
  a.G = r.top_groups == r.n_groups ? 1 : r.n_groups;
  a.per = a.E / a.G;
  int p2 = 1;
  while (p2 < a.G) p2 *= 2;
  a.L = 32 / p2;
  while ((1 << a.log_l) < a.L) ++a.log_l;
  a.kept = r.top_groups;
  a.group_top = r.group_top;
  a.softmax = r.score == YN_SCORE_SOFTMAX;
  a.norm = r.norm_topk != 0;
  a.scale = r.scale;
  const bool by_score = bias || a.G > 1;
  const int nv = (a.per + a.L - 1) / a.L;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == YN_F32) by_score ? launch_router<float, true>(a, nv, st) : launch_router<float, false>(a, nv, st);
  else if (dtype == YN_BF16)
    by_score ? launch_router<__nv_bfloat16, true>(a, nv, st) : launch_router<__nv_bfloat16, false>(a, nv, st);
  else by_score ? launch_router<__half, true>(a, nv, st) : launch_router<__half, false>(a, nv, st);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return host_fail(YN_E_CUDA, std::string("yn_route_scored: ") + cudaGetErrorString(e));
  return YN_OK;
}
