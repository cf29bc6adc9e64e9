// Log probabilities of given tokens, their ranks, the rows' entropies and the
// likeliest alternatives, and their C ABI. No counterpart in the reference, which
// compares greedy choices of the verify pass (speculative.py:121-193).
//
// Per row of logits z with maximum m at token *:  R = sum over the others of
// exp(z - m), log S = log1p(R), logprob = (z[t] - m) - log S, entropy = log S -
// sum exp(z - m)(z - m) / S. The sum leaves the largest term out so that log S
// keeps its relative accuracy when that term has nearly all the mass.
//
// Bound by reading the logits once. A thread holds VPT 16-byte pieces of the row in
// registers (all loads in flight at once), takes their maximum and sums their
// exponentials relative to it, one ex2 per element and two fp32 values per
// instruction elsewhere (fma.rn.f32x2); pieces and threads are joined by rescaling two
// sums. A thread's R is its sum less one, off by 2^-23: where the row's R comes out small
// one warp sums the pieces of the thread that holds the maximum again without it.
// The alternatives cost little beside that: the n-th largest of the block's 32
// quarter-warp maxima (or of its 256 thread maxima) bounds the n-th largest element from
// below, and only the threads that reach it, little more than n, have their elements
// looked at again, a warp for each (from L2).
// Few rows are split over the blocks of a cluster, whose parts the first of them joins
// through distributed shared memory: one launch, no workspace. The parts take the bound of
// the alternatives from all of them, so that they have few candidates together (1 x 151936
// fp32, 20 alternatives: 9.2 us, 14.5 with bounds of their own). 4096 x 65536 bf16 with 8
// alternatives: 115 us, 4.7 TB/s, bound by instruction issue (62% of the cycles; 91 us without
// tokens and alternatives).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "yanah_b200.h"
#include "yn_common.cuh"
#include "yn_internal.h"

namespace ynb {

constexpr int LP_THREADS = 256;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_MAX_TOP = 64;
constexpr int LP_CAND = 1024;        // candidates of one chunk that are ranked by counting
constexpr int LP_MAX_SPLITS = 8;     // blocks of one row: a portable cluster
constexpr float LP_LOG2E = 1.44269504088896341f;
constexpr float LP_LN2 = 0.69314718055994531f;

// Sums of a part of a row: maximum m (-inf: nothing in it), R = sum exp(z - m)
// without one largest term, D = sum exp(z - m) (z - m).
struct LpSums {
  float m, R, D;
  int rank;   // elements of the part that come before the given token
};
struct LpArgs {
  const uint8_t* z;
  long long ld, rows;
  int V, n_top, splits, split_vecs;
  const int32_t* tokens;
  float* logprob;
  float* entropy;
  int32_t* rank;
  int32_t* top_ids;
  float* top_lp;
};

template <typename T>
struct LpType;
template <>
struct LpType<float> {
  static constexpr int PER = 4;
  static constexpr uint32_t NEG = 0xFF800000u;
  YN_DEV static void unpack(uint32_t w, float* f) { f[0] = __uint_as_float(w); }
  YN_DEV static uint32_t max_nan(uint32_t a, uint32_t b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
    return __float_as_uint(d);
  }
  // -inf as a finite value whose exponential is 0 against any maximum above -4096
  YN_DEV static uint32_t floor(uint32_t a) { return __float_as_uint(fmaxf(__uint_as_float(a), -1e30f)); }
  YN_DEV static float load(const void* p) { return __ldg(reinterpret_cast<const float*>(p)); }
  // how many values of `a` are above `t` (a value in both halves, for 16-bit types), added to `c`
  YN_DEV static uint32_t splat(float t) { return __float_as_uint(t); }
  YN_DEV static void count(uint32_t a, uint32_t t, uint32_t& c) { c += __uint_as_float(a) > __uint_as_float(t); }
  YN_DEV static int counted(uint32_t c) { return (int)c; }
};
template <>
struct LpType<__nv_bfloat16> {
  static constexpr int PER = 8;
  static constexpr uint32_t NEG = 0xFF80FF80u;
  YN_DEV static void unpack(uint32_t w, float* f) {
    f[0] = __uint_as_float(w << 16);
    f[1] = __uint_as_float(w & 0xFFFF0000u);
  }
  YN_DEV static uint32_t max_nan(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  YN_DEV static uint32_t floor(uint32_t a) {
    uint32_t d;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(0xF149F149u));   // -1e30
    return d;
  }
  YN_DEV static float load(const void* p) { return bf16_to_f32(__ldg(reinterpret_cast<const uint16_t*>(p))); }
  YN_DEV static uint32_t splat(float t) { return (__float_as_uint(t) >> 16) * 0x10001u; }
  YN_DEV static void count(uint32_t a, uint32_t t, uint32_t& c) {   // counts of at most 256 are exact in bf16
    __nv_bfloat162 x = *reinterpret_cast<__nv_bfloat162*>(&a), y = *reinterpret_cast<__nv_bfloat162*>(&t);
    __nv_bfloat162 s = __hadd2(*reinterpret_cast<__nv_bfloat162*>(&c), __hgt2(x, y));
    c = *reinterpret_cast<uint32_t*>(&s);
  }
  YN_DEV static int counted(uint32_t c) {
    return (int)(__uint_as_float(c << 16) + __uint_as_float(c & 0xFFFF0000u));
  }
};
template <>
struct LpType<__half> {
  static constexpr int PER = 8;
  static constexpr uint32_t NEG = 0xFC00FC00u;
  YN_DEV static void unpack(uint32_t w, float* f) {
    f[0] = f16_to_f32((uint16_t)(w & 0xFFFFu));
    f[1] = f16_to_f32((uint16_t)(w >> 16));
  }
  YN_DEV static uint32_t max_nan(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  YN_DEV static uint32_t floor(uint32_t a) {
    uint32_t d;
    asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(0xFBFFFBFFu));   // -65504
    return d;
  }
  YN_DEV static float load(const void* p) { return f16_to_f32(__ldg(reinterpret_cast<const uint16_t*>(p))); }
  YN_DEV static uint32_t splat(float t) { return __half_as_ushort(__float2half_rn(t)) * 0x10001u; }
  YN_DEV static void count(uint32_t a, uint32_t t, uint32_t& c) {
    __half2 s = __hadd2(*reinterpret_cast<__half2*>(&c), __hgt2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&t)));
    c = *reinterpret_cast<uint32_t*>(&s);
  }
  YN_DEV static int counted(uint32_t c) {
    return (int)(f16_to_f32((uint16_t)(c & 0xFFFFu)) + f16_to_f32((uint16_t)(c >> 16)));
  }
};

// The largest value of the type below a finite t, as fp32.
template <typename T>
YN_DEV float lp_below(float t) {
  constexpr uint32_t step = sizeof(T) == 4 ? 1u : std::is_same_v<T, __half> ? 0u : 0x10000u;
  if constexpr (step == 0) {
    const uint16_t h = __half_as_ushort(__float2half_rn(__fadd_rn(t, 0.0f)));
    return f16_to_f32(h == 0 ? (uint16_t)0x8001u : (uint16_t)(h & 0x8000u ? h + 1 : h - 1));
  } else {
    const uint32_t b = __float_as_uint(__fadd_rn(t, 0.0f));
    return __uint_as_float(b == 0 ? 0x80000000u + step : b & 0x80000000u ? b + step : b - step);
  }
}

// The elements of a 16-byte vector, in order.
template <typename T>
YN_DEV void lp_unpack(const uint4& v, float (&f)[LpType<T>::PER]) {
  constexpr int W = LpType<T>::PER / 4;
  LpType<T>::unpack(v.x, f);
  LpType<T>::unpack(v.y, f + W);
  LpType<T>::unpack(v.z, f + 2 * W);
  LpType<T>::unpack(v.w, f + 3 * W);
}

// Two fp32 values per instruction.
YN_DEV uint64_t lp_pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
YN_DEV void lp_unpair(uint64_t d, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(d)); }
YN_DEV uint64_t lp_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
YN_DEV uint64_t lp_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

YN_DEV float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Joins part b to part a (the ranks apart).
YN_DEV void lp_join(LpSums& a, const LpSums& b) {
  const float inf = __int_as_float(0x7f800000);
  const bool up = b.m > a.m;
  const float hm = up ? b.m : a.m, hR = up ? b.R : a.R, hD = up ? b.D : a.D;
  const float lm = up ? a.m : b.m, lR = up ? a.R : b.R, lD = up ? a.D : b.D;
  const float d = hm == lm ? 0.0f : lm - hm, f = lm == -inf ? 0.0f : lp_ex2(d * LP_LOG2E);   // both +inf: d = 0
  a.m = hm;
  a.R = fmaf(f, 1.0f + lR, hR);
  a.D = f > 0.0f ? fmaf(f, fmaf(d, 1.0f + lR, lD), hD) : hD;
}

// The join of the 32 lanes' parts, on every lane. own: R and D of the one lane (`first`) whose
// maximum is taken, which are not in those returned.
YN_DEV LpSums lp_warp_join(const LpSums& s, float2* own, int* first) {
  const float inf = __int_as_float(0x7f800000);
  LpSums o;
  o.m = f32_from_ukey(__reduce_max_sync(0xffffffffu, f32_ukey(s.m)));
  const bool top = s.m == o.m;
  *first = __ffs(__ballot_sync(0xffffffffu, top)) - 1;
  const float d = top ? 0.0f : s.m - o.m, f = s.m == -inf ? 0.0f : top ? 1.0f : lp_ex2(d * LP_LOG2E);
  const bool other = (int)(threadIdx.x & 31) != *first && f > 0.0f;
  *own = make_float2(__shfl_sync(0xffffffffu, s.R, *first), __shfl_sync(0xffffffffu, s.D, *first));
  o.R = warp_sum_f32(other ? f * (1.0f + s.R) : 0.0f);
  o.D = warp_sum_f32(other ? f * fmaf(d, 1.0f + s.R, s.D) : 0.0f);
  o.rank = __reduce_add_sync(0xffffffffu, s.rank);
  return o;
}

// A row's answer from its sums and log S, by one thread. z_tok: the token's logit.
YN_DEV void lp_write(const LpArgs& a, long long row, const LpSums& s, float ls, bool nan, int tok, float z_tok) {
  const float inf = __int_as_float(0x7f800000), none = __int_as_float(0x7fc00000);
  if (a.entropy) a.entropy[row] = nan ? none : s.m == -inf ? 0.0f : ls - s.D / (1.0f + s.R);
  if (!a.tokens) return;
  const bool ok = !nan && tok >= 0 && tok < a.V;
  a.rank[row] = ok ? s.rank : -1;
  a.logprob[row] = !ok ? none : z_tok == -inf ? -inf : z_tok == s.m ? -ls : (z_tok - s.m) - ls;
}
YN_DEV void lp_write_top(const LpArgs& a, long long row, int j, unsigned long long key, float m, float log_s, bool nan) {
  const float z = f32_from_ukey((uint32_t)(key >> 32));
  a.top_ids[row * a.n_top + j] = key && !nan ? (int32_t)(0xFFFFFFFFu - (uint32_t)key) : -1;
  a.top_lp[row * a.n_top + j] = nan ? log_s : !key ? -__int_as_float(0x7f800000) : z == m ? -log_s : (z - m) - log_s;
}

// Largest 64-bit key over the block, on every thread. buf: LP_WARPS words that no
// other call since the last barrier but one uses.
YN_DEV unsigned long long lp_block_max(unsigned long long k, unsigned long long* buf) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = ((unsigned long long)hi << 32) | lo;
  __syncthreads();
  unsigned long long best = buf[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) best = best < buf[w] ? buf[w] : best;
  return best;
}

template <typename T, int VPT, bool SPLIT>
__global__ void __launch_bounds__(LP_THREADS, 1024 / LP_THREADS) k_logprobs(const LpArgs a) {
  using L = LpType<T>;
  constexpr int PER = L::PER;
  constexpr uint32_t KEY_NEG = 0x007FFFFFu;   // f32_ukey(-inf)
  __shared__ uint32_t tkey[LP_THREADS], gkey[32];
  __shared__ LpSums wsum[LP_WARPS];
  __shared__ float2 wown[LP_WARPS];
  __shared__ int wfirst[LP_WARPS];
  __shared__ int n_cand;
  __shared__ unsigned long long cand[LP_CAND], list[LP_MAX_TOP], buf[2][LP_WARPS];
  __shared__ LpSums part;
  __shared__ int part_nan, part_have, list_end[LP_MAX_SPLITS];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row = blockIdx.x / a.splits;
  const int split = (int)(blockIdx.x % a.splits);
  const float inf = __int_as_float(0x7f800000);
  const float z_big = sizeof(T) == 4 ? 3.402823466e38f : std::is_same_v<T, __half> ? 65504.0f : 3.38953139e38f;
  const uint8_t* p = a.z + (size_t)row * a.ld * sizeof(T);
  // Vectors are aligned: the row's first element is element `lead` of vector 0, and
  // what a vector holds beside the row lies inside the same 16 bytes as an element of it.
  const int lead = (int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
  const uint8_t* base = p - lead * sizeof(T);
  const int n_vecs = (int)(((long long)lead + a.V + PER - 1) / PER);
  const int v0 = split * a.split_vecs, v1 = min(n_vecs, v0 + a.split_vecs);
  const int tok = a.tokens ? a.tokens[row] : -1;
  const bool ranked = tok >= 0 && tok < a.V;
  const float z_tok = ranked ? L::load(p + (size_t)tok * sizeof(T)) : inf;
  const int tv = ranked ? (int)(((long long)lead + tok) / PER) : 0;

  LpSums sums = {-inf, 0.0f, 0.0f, 0};
  bool bad = false;            // a NaN
  uint32_t tk = KEY_NEG;       // key of the thread's maximum
  if (tid == 0) n_cand = 0;
  for (int c0 = v0; c0 < v1; c0 += LP_THREADS * VPT) {
    uint4 v[VPT];
    const uint8_t* at0 = base + ((size_t)c0 + tid) * 16;
    if (c0 + LP_THREADS * VPT <= v1) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) v[i] = ldg_nc_v4(at0 + i * (LP_THREADS * 16));
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        v[i] = c0 + i * LP_THREADS + tid < v1 ? ldg_nc_v4(at0 + i * (LP_THREADS * 16))
                                              : make_uint4(L::NEG, L::NEG, L::NEG, L::NEG);
    }
    if ((c0 == 0 && lead) || c0 + LP_THREADS * VPT >= n_vecs) {  // what lies outside the row reads as -inf
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int at = c0 + i * LP_THREADS + tid;
        if (at != 0 && at != n_vecs - 1) continue;
        const long long e0 = (long long)at * PER - lead;
        uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (e0 + j < 0 || e0 + j >= a.V) {
            if (PER == 4) w[j] = L::NEG;
            else w[j / 2] = (j & 1) ? (w[j / 2] & 0xFFFFu) | (L::NEG & 0xFFFF0000u)
                                    : (w[j / 2] & 0xFFFF0000u) | (L::NEG & 0xFFFFu);
          }
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    uint32_t mx = L::NEG;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      mx = L::max_nan(mx, L::max_nan(L::max_nan(v[i].x, v[i].y), L::max_nan(v[i].z, v[i].w)));
    float tm;
    {
      float f[2];
      L::unpack(mx, f);
      tm = PER == 4 ? f[0] : (f[0] > f[1] || f[0] != f[0] ? f[0] : f[1]);
    }
    bad |= tm != tm;
    if (tm > -inf) {
      // y is (z - tm) log2(e) + del, del the rounding of tm log2(e), which is taken out of the sums
      LpSums c = {tm, 0.0f, 0.0f, 0};
      if (fabsf(tm) < 4096.0f) {
        const float ml = tm * LP_LOG2E, del = fmaf(tm, LP_LOG2E, -ml);
        const uint64_t l2 = lp_pair(LP_LOG2E, LP_LOG2E), ml2 = lp_pair(-ml, -ml);
        uint64_t r2 = 0, d2 = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const uint4 q = make_uint4(L::floor(v[i].x), L::floor(v[i].y), L::floor(v[i].z), L::floor(v[i].w));
          float f[PER];
          lp_unpack<T>(q, f);
#pragma unroll
          for (int j = 0; j < PER; j += 2) {
            const uint64_t y = lp_fma2(lp_pair(f[j], f[j + 1]), l2, ml2);
            float y0, y1;
            lp_unpair(y, y0, y1);
            const uint64_t e = lp_pair(lp_ex2(y0), lp_ex2(y1));
            r2 = lp_add2(r2, e);
            d2 = lp_fma2(e, y, d2);
          }
        }
        float r0, r1, d0, d1;
        lp_unpair(r2, r0, r1);
        lp_unpair(d2, d0, d1);
        const float s = r0 + r1, f = lp_ex2(-del);
        c.R = fmaf(f, s, -1.0f);
        c.D = f * fmaf(-del, s, d0 + d1) * LP_LN2;
      } else {
        // maxima so large that del is not small, or infinite: the pieces again, one at a time, the
        // subtraction first
        int cnt = 0;
        float d = 0.0f;
#pragma unroll 1
        for (int i = 0; i < VPT; ++i) {
          const int at = c0 + i * LP_THREADS + tid;
          if (at >= v1) break;
          float f[PER];
          lp_unpack<T>(ldg_nc_v4(base + (size_t)at * 16), f);
          const long long e0 = (long long)at * PER - lead;
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            if (e0 + j < 0 || e0 + j >= a.V) continue;
            const bool top = f[j] == tm;
            const float y = fmaxf((f[j] - tm) * LP_LOG2E, -200.0f), e = top ? 0.0f : lp_ex2(y);
            cnt += top;
            c.R += e;
            d = top ? d : fmaf(e, y, d);
          }
        }
        c.R += (float)(cnt - 1);
        c.D = d * LP_LN2;
      }
      lp_join(sums, c);
      tk = max(tk, f32_ukey(tm));
    }
    if (ranked && tm >= z_tok) {
      if (z_tok > -inf) {
        // before the token's own vector equal logits count too: above the value just below
        const uint32_t above = L::splat(z_tok), from = L::splat(z_tok < inf ? lp_below<T>(z_tok) : z_big);
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int at = c0 + i * LP_THREADS + tid;
          const uint32_t t = at < tv ? from : above;
          L::count(v[i].x, t, c);
          L::count(v[i].y, t, c);
          L::count(v[i].z, t, c);
          L::count(v[i].w, t, c);
        }
        sums.rank += L::counted(c);
      } else {
        // a barred token: every logit above -inf, and before its own vector the barred ones too
        const uint32_t above = L::splat(-inf);
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int at = c0 + i * LP_THREADS + tid;
          if (at >= tv) {
            L::count(v[i].x, above, c);
            L::count(v[i].y, above, c);
            L::count(v[i].z, above, c);
            L::count(v[i].w, above, c);
          } else if (at < v1) {
            sums.rank += at ? PER : PER - lead;
          }
        }
        sums.rank += L::counted(c);
      }
      if (tv >= c0 && tv < min(v1, c0 + LP_THREADS * VPT) && (tv - c0) % LP_THREADS == tid) {
        // inside it, those of a lower id
        for (int j = 0; j < PER; ++j) {
          const long long e = (long long)tv * PER + j - lead;
          if (e >= 0 && e < tok) sums.rank += L::load(p + e * sizeof(T)) == z_tok;
        }
      }
    }
  }
  {
    float2 own;
    int first;
    sums = lp_warp_join(sums, &own, &first);
    if (lane == 0) {
      wsum[warp] = sums;
      wown[warp] = own;
      wfirst[warp] = first;
    }
    uint32_t g = tk;
#pragma unroll
    for (int o = LP_THREADS / 64; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % (LP_THREADS / 32) == 0) gkey[tid / (LP_THREADS / 32)] = g;
    if (a.n_top > 32) tkey[tid] = tk;
  }
  const bool nan = __syncthreads_or(bad) != 0;
  if (a.n_top) {
    uint32_t t = 0;
    if (a.n_top <= 32) {
      // every warp takes the n-th largest of the 32 (equal ones go together: lower, and still a bound);
      // of a split row the 32 are maxima over all parts, so that the parts have few candidates together
      uint32_t g = gkey[lane];
      if constexpr (SPLIT) {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        for (int q = 0; q < a.splits; ++q) g = max(g, cluster.map_shared_rank(gkey, q)[lane]);
      }
      for (int j = 0; j < a.n_top; ++j) {
        t = __reduce_max_sync(0xffffffffu, g);
        if (g == t) g = 0;
      }
    } else {
      uint32_t k[LP_WARPS];   // the n-th largest thread maximum, its low 16 bits left out
#pragma unroll
      for (int w = 0; w < LP_WARPS; ++w) k[w] = tkey[lane + 32 * w];
      for (int b = 31; b >= 16; --b) {
        const uint32_t x = t | (1u << b);
        int c = 0;
#pragma unroll
        for (int w = 0; w < LP_WARPS; ++w) c += k[w] >= x;
        if (__reduce_add_sync(0xffffffffu, c) >= a.n_top) t = x;
      }
    }
    t = max(t, KEY_NEG + 1);
    const float least = f32_from_ukey(t);
    // the elements of each of the warp's threads that reach the bound, a lane per vector
    for (unsigned who = __ballot_sync(0xffffffffu, tk >= t); who; who &= who - 1) {
      for (int at = v0 + 32 * warp + __ffs(who) - 1 + lane * LP_THREADS; at < v1; at += 32 * LP_THREADS) {
        const uint4 q = ldg_nc_v4(base + (size_t)at * 16);
        const uint32_t w = L::max_nan(L::max_nan(q.x, q.y), L::max_nan(q.z, q.w));
        float f[PER];
        L::unpack(w, f);
        if (at > 0 && at < n_vecs - 1 && !(f[0] >= least || (PER == 8 && f[1] >= least))) continue;
        lp_unpack<T>(q, f);
        const long long e0 = (long long)at * PER - lead;
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (f[j] >= least && e0 + j >= 0 && e0 + j < a.V) {
            const int n = atomicAdd(&n_cand, 1);
            if (n < LP_CAND) cand[n] = ((unsigned long long)f32_ukey(f[j]) << 32) | (0xFFFFFFFFu - (uint32_t)(e0 + j));
          }
      }
      __syncwarp();
    }
  }
  if (warp == 0) {
    const LpSums none = {-inf, 0.0f, 0.0f, 0};
    // a warp's sums are whole where another warp has the maximum
    LpSums s = lane < LP_WARPS ? wsum[lane] : none;
    const float2 own = lane < LP_WARPS ? wown[lane] : make_float2(0.0f, 0.0f), apart = make_float2(s.R, s.D);
    s.R += own.x;
    s.D += own.y;
    float2 whole;
    int w0;
    sums = lp_warp_join(s, &whole, &w0);
    float2 rest = wown[w0];   // of the thread that holds the maximum
    sums.R += __shfl_sync(0xffffffffu, apart.x, w0);
    sums.D += __shfl_sync(0xffffffffu, apart.y, w0);
    if (sums.R + rest.x < 0.25f && fabsf(sums.m) < inf) {
      float r = 0.0f, d = 0.0f;
      int cnt = 0;
      for (int at = v0 + 32 * w0 + wfirst[w0] + lane * LP_THREADS; at < v1; at += 32 * LP_THREADS) {
        float f[PER];
        lp_unpack<T>(ldg_nc_v4(base + (size_t)at * 16), f);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const long long e = (long long)at * PER + j - lead;
          if (e < 0 || e >= a.V) continue;
          const float y = fmaxf((f[j] - sums.m) * LP_LOG2E, -200.0f), x = f[j] == sums.m ? 0.0f : lp_ex2(y);
          cnt += f[j] == sums.m;
          r += x;
          d = fmaf(x, y, d);
        }
      }
      rest.x = warp_sum_f32(r) + (float)(__reduce_add_sync(0xffffffffu, cnt) - 1);
      rest.y = warp_sum_f32(d) * LP_LN2;
    }
    sums.R += rest.x;
    sums.D += rest.y;
  }
  if (a.n_top) __syncthreads();
  int have = 0;
  if (a.n_top) {
    int n = n_cand;
    if (n > LP_CAND) {
      // many equal or ascending logits: the n largest one after another, over the whole part
      unsigned long long prev = ~0ull;
      __syncthreads();   // n_cand and cand have been read by all
      n = 0;
      for (int q = 0; q < a.n_top; ++q) {
        unsigned long long best = 0;
        for (int at = v0 + tid; at < v1; at += LP_THREADS) {
          float f[PER];
          lp_unpack<T>(ldg_nc_v4(base + (size_t)at * 16), f);
          const long long e0 = (long long)at * PER - lead;
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const unsigned long long k = ((unsigned long long)f32_ukey(f[j]) << 32) | (0xFFFFFFFFu - (uint32_t)(e0 + j));
            if (e0 + j >= 0 && e0 + j < a.V && f[j] > -inf && k < prev && k > best) best = k;
          }
        }
        prev = lp_block_max(best, buf[q & 1]);
        if (!prev) break;
        if (tid == 0) list[q] = prev;
        ++n;
      }
    } else {
      // each candidate placed by how many are larger (keys are distinct)
      for (int i = tid; i < n; i += LP_THREADS) {
        const unsigned long long k = cand[i];
        int place = 0;
        for (int q = 0; q < n; ++q) place += cand[q] > k;
        if (place < a.n_top) list[place] = k;
      }
    }
    have = min(n, a.n_top);
    __syncthreads();
  }
  bool row_nan = nan;
  if constexpr (SPLIT) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) {
      part = sums;
      part_nan = nan;
      part_have = have;
    }
    cluster.sync();
    if (split == 0) {
      if (warp == 0) {
        LpSums s = {-inf, 0.0f, 0.0f, 0};
        if (lane < a.splits) {
          s = *cluster.map_shared_rank(&part, lane);
          row_nan = *cluster.map_shared_rank(&part_nan, lane) != 0;
        }
        float2 own;
        int first;
        sums = lp_warp_join(s, &own, &first);
        sums.R += own.x;
        sums.D += own.y;
        int end = lane < a.splits ? *cluster.map_shared_rank(&part_have, lane) : 0;
#pragma unroll
        for (int o = 1; o < LP_MAX_SPLITS; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, end, o);
          if (lane >= o) end += v;
        }
        if (lane < a.splits) list_end[lane] = end;
      }
      row_nan = __syncthreads_or(row_nan) != 0;
      if (a.n_top) {
        // the parts' lists one after another, then placed as the candidates above
        for (int i = tid; i < a.splits * a.n_top; i += LP_THREADS) {
          const int q = i / a.n_top, j = i - q * a.n_top, at = q ? list_end[q - 1] : 0;
          if (at + j < list_end[q]) cand[at + j] = cluster.map_shared_rank(list, q)[j];
        }
        __syncthreads();
        const int n = list_end[a.splits - 1];
        for (int i = tid; i < n; i += LP_THREADS) {
          const unsigned long long k = cand[i];
          int place = 0;
          for (int q = 0; q < n; ++q) place += cand[q] > k;
          if (place < a.n_top) list[place] = k;
        }
        __syncthreads();
        have = min(n, a.n_top);
      }
    }
    cluster.sync();   // no block leaves while its parts are read
    if (split != 0) return;
  }
  if (warp == 0) {
    const float ls = row_nan ? __int_as_float(0x7fc00000) : log1pf(sums.R);
    if (lane == 0) lp_write(a, row, sums, ls, row_nan, tok, z_tok);
    for (int j = lane; j < a.n_top; j += 32) lp_write_top(a, row, j, j < have ? list[j] : 0ull, sums.m, ls, row_nan);
  }
}

// How a row is split: enough blocks for two on every SM when the rows alone are fewer,
// each with at least one 16-byte load per thread.
int lp_splits(long long rows, long long vecs) {
  int s = 1;
  while (s < LP_MAX_SPLITS && rows * 2 * s <= 2 * 148 && vecs >= 2 * s * LP_THREADS) s *= 2;
  return s;
}

template <typename T, int VPT>
cudaError_t launch_logprobs_vpt(const LpArgs& a, cudaStream_t st) {
  if (a.splits == 1) {
    k_logprobs<T, VPT, false><<<(unsigned)a.rows, LP_THREADS, 0, st>>>(a);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)(a.rows * a.splits));
  c.blockDim = dim3(LP_THREADS);
  c.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = a.splits;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  c.attrs = &at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, k_logprobs<T, VPT, true>, a);
}
// Pieces per thread: all of a short part at once, else 8.
template <typename T>
cudaError_t launch_logprobs(const LpArgs& a, cudaStream_t st) {
  if (a.split_vecs <= LP_THREADS) return launch_logprobs_vpt<T, 1>(a, st);
  if (a.split_vecs <= 2 * LP_THREADS) return launch_logprobs_vpt<T, 2>(a, st);
  if (a.split_vecs <= 4 * LP_THREADS) return launch_logprobs_vpt<T, 4>(a, st);
  return launch_logprobs_vpt<T, 8>(a, st);
}

}  // namespace ynb

using namespace ynb;

namespace {
int lp_size(int dtype) { return dtype == YN_F32 ? 4 : dtype == YN_BF16 || dtype == YN_F16 ? 2 : 0; }
}  // namespace

extern "C" int yn_token_logprobs(const void* logits, int32_t dtype, int64_t row_stride, int64_t rows, int64_t vocab,
                                 const int32_t* tokens, int32_t n_top, float* logprob, float* entropy, int32_t* rank,
                                 int32_t* top_ids, float* top_logprobs, void* stream) {
  const int size = lp_size(dtype);
  if (!size) return host_fail(YN_E_INVALID, "unknown dtype");
  if (vocab < 1 || rows < 0 || row_stride < vocab) return host_fail(YN_E_INVALID, "row_stride must be at least vocab, vocab at least 1");
  if (vocab > 0x7fffff00LL || rows > 0x7fffffffLL / LP_MAX_SPLITS)
    return host_fail(YN_E_UNSUPPORTED, "vocab below 2^31 - 255, at most 8388607 rows");
  if (n_top < 0 || n_top > LP_MAX_TOP || n_top > vocab) return host_fail(YN_E_INVALID, "n_top must be in [0, min(64, vocab)]");
  if (rows == 0) return YN_OK;
  if (!logits || (tokens && (!logprob || !rank)) || (n_top && (!top_ids || !top_logprobs)))
    return host_fail(YN_E_INVALID, "null argument");
  if (!host_aligned(size, logits) || !host_aligned(4, tokens, logprob, entropy, rank, top_ids, top_logprobs))
    return host_fail(YN_E_INVALID, "logits, tokens and outputs must be aligned to their elements");
  LpArgs a{};
  a.z = reinterpret_cast<const uint8_t*>(logits);
  a.ld = row_stride;
  a.rows = rows;
  a.V = (int)vocab;
  a.n_top = n_top;
  const long long vecs = (vocab * size + 15) / 16 + 1;   // one more: a row may start inside a vector
  a.splits = lp_splits(rows, vecs);
  a.split_vecs = (int)((vecs + a.splits - 1) / a.splits);
  a.tokens = tokens;
  a.logprob = logprob;
  a.entropy = entropy;
  a.rank = rank;
  a.top_ids = top_ids;
  a.top_lp = top_logprobs;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == YN_F32    ? launch_logprobs<float>(a, st)
                        : dtype == YN_BF16 ? launch_logprobs<__nv_bfloat16>(a, st)
                                           : launch_logprobs<__half>(a, st);
  if (e != cudaSuccess) return host_fail(YN_E_CUDA, std::string("yn_token_logprobs: ") + cudaGetErrorString(e));
  return YN_OK;
}
