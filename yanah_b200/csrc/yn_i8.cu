// Rows in 8-bit integers, the products of few rows (dp4a), the grouping and the
// joining of the experts' products, and the C ABI of all of it. The tensor-core
// product of many rows is in yn_i8.cuh.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "yanah_b200.h"
#include "yn_common.cuh"
#include "yn_i8.cuh"
#include "yn_internal.h"

namespace ynb {

// Element type at run time, where a load is not what a kernel waits for.
YN_DEV float i8_load(int dt, const void* p, size_t i) {
  return dt == YN_F32 ? I8In<float>::load(p, i) : dt == YN_BF16 ? I8In<__nv_bfloat16>::load(p, i) : I8In<__half>::load(p, i);
}
YN_DEV void i8_store(int dt, void* p, size_t i, float v) {
  if (dt == YN_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == YN_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// ------------------------------------------------------------- row codes
constexpr int I8_QT = 128;     // threads of a row
constexpr long long I8_QWARP = 1184;   // rows from which a warp each fills the device (8 per SM)

// The largest magnitude, then the codes, by N threads per row: a block where there are few
// rows, a warp where there are many (no barrier, 8 loads in flight per lane). Rows of up to
// N * 8 * HOLD elements are read once, longer ones a second time from L2. The codes go to row
// `to[j]` for each of the `copies` entries of the row's list (or to the row itself): a row's
// codes are made once for all of its experts. late: the kernel before makes the lists, not the
// rows, and is waited for when the codes are made.
template <typename T, bool VEC, int N, int HOLD>
__global__ void __launch_bounds__(I8_QT) k_i8_quant(const void* x, long long ldx, long long rows, int K, const int* n_rows,
                                                    const int32_t* to, int copies, int8_t* codes, long long ldc,
                                                    float* scales, bool late) {
  __shared__ uint32_t buf[I8_QT / 32];
  i8_launch_next();
  if (!late) i8_wait_previous();
  const size_t row = blockIdx.x * (size_t)(I8_QT / N) + threadIdx.x / N, base = row * (size_t)ldx;
  if (row >= (size_t)(n_rows ? *n_rows : rows)) return;
  const int tid = threadIdx.x % N, n8 = VEC ? K / 8 : 0;
  I8Raw<T> raw[HOLD], one;
  uint32_t m = 0;
  auto max8 = [&](const I8Raw<T>& r) {
    float g[8];
    r.get(g);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, i8_abs_bits(g[j]));
  };
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (tid + i * N < n8) raw[i].load(x, base + 8 * (size_t)(tid + i * N));
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (tid + i * N < n8) max8(raw[i]);
  for (int at = tid + HOLD * N; at < n8; at += N) {
    one.load(x, base + 8 * (size_t)at);
    max8(one);
  }
  for (int k = 8 * n8 + tid; k < K; k += N) m = max(m, i8_abs_bits(I8In<T>::load(x, base + k)));
  const I8Row q(N == 32 ? __reduce_max_sync(0xffffffffu, m) : block_max_u32(m, buf));
  auto code8 = [&](const I8Raw<T>& r) {
    float g[8];
    uint32_t w[2];
    r.get(g);
    q.codes<sizeof(T) == 2>(g, w);
    return make_uint2(w[0], w[1]);
  };
  uint2 c[HOLD];
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (tid + i * N < n8) c[i] = code8(raw[i]);
  if (late) i8_wait_previous();
  // lane j of every warp has destination j
  const int lane = threadIdx.x & 31, n_to = to ? copies : 1;
  const int dest = lane < n_to ? (to ? to[row * copies + lane] : (int)row) : -1;
  if (tid < n_to && dest >= 0) scales[dest] = q.scale();
  for (int j = 0; j < n_to; ++j) {
    const int r = __shfl_sync(0xffffffffu, dest, j);
    if (r < 0) continue;
    uint2* at = reinterpret_cast<uint2*>(codes + (long long)r * ldc) + tid;
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (tid + i * N < n8) at[i * N] = c[i];
  }
  for (int i = HOLD * N; i < n8; i += N) {
    if (i + tid < n8) {
      one.load(x, base + 8 * (size_t)(i + tid));
      c[0] = code8(one);
    }
    for (int j = 0; j < n_to; ++j) {
      const int r = __shfl_sync(0xffffffffu, dest, j);
      if (r >= 0 && i + tid < n8) reinterpret_cast<uint2*>(codes + (long long)r * ldc)[i + tid] = c[0];
    }
  }
  for (int k = 8 * n8 + tid; k < K; k += N) {
    const float g[4] = {I8In<T>::load(x, base + k), 0.0f, 0.0f, 0.0f};
    uint32_t w[1];
    q.codes<sizeof(T) == 2>(g, w);
    const int8_t b = (int8_t)w[0];
    for (int j = 0; j < n_to; ++j) {
      const long long r = to ? to[row * copies + j] : (long long)row;
      if (r >= 0) codes[r * ldc + k] = b;
    }
  }
}

// Kernels of one call follow one another without a gap (programmatic launch): all but the first
// are launched with this. Each waits for the one before it itself.
template <typename... P, typename... A>
void launch_after(void (*kern)(P...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t lc{};
  lc.gridDim = grid;
  lc.blockDim = dim3(block);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  lc.attrs = &at;
  lc.numAttrs = 1;
  (void)cudaLaunchKernelEx(&lc, kern, static_cast<P>(args)...);   // its error is the caller's cudaGetLastError
}

int launch_quant(int dt, const void* x, long long ldx, long long rows, int K, const int* n_rows, const int32_t* to, int copies,
                 int8_t* codes, long long ldc, float* scales, bool first, cudaStream_t st) {
  const size_t size = dt == YN_F32 ? 4 : 2;
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * size) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(codes) % 8 == 0 && ldc % 8 == 0;
  const bool warps = vec && rows >= I8_QWARP && K <= 4096;
  const dim3 g((unsigned)(warps ? (rows + I8_QT / 32 - 1) / (I8_QT / 32) : rows));
  auto go = [&](auto kern) {
    if (first) kern<<<g, I8_QT, 0, st>>>(x, ldx, rows, K, n_rows, to, copies, codes, ldc, scales, false);
    else launch_after(kern, g, I8_QT, 0, st, x, ldx, rows, K, n_rows, to, copies, codes, ldc, scales, to != nullptr);
  };
#define YN_Q(T)                                                       \
  if (warps) go(k_i8_quant<T, true, 32, sizeof(T) == 4 ? 6 : 8>);     \
  else if (vec) go(k_i8_quant<T, true, I8_QT, 4>);                    \
  else go(k_i8_quant<T, false, I8_QT, 4>)
  if (dt == YN_F32) { YN_Q(float); }
  else if (dt == YN_BF16) { YN_Q(__nv_bfloat16); }
  else { YN_Q(__half); }
#undef YN_Q
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? YN_OK : host_fail(YN_E_CUDA, std::string("row codes: ") + cudaGetErrorString(e));
}

// ------------------------------------------------- few rows: dp4a products
constexpr int I8_GT = 256;           // threads
constexpr int I8_GW = I8_GT / 32;
constexpr int I8_GK = 512;           // codes of K that a warp takes in one step, 16 per lane

YN_DEV int dot16(const uint4& a, const uint4& b, int acc) {
  acc = __dp4a((int)a.x, (int)b.x, acc);
  acc = __dp4a((int)a.y, (int)b.y, acc);
  acc = __dp4a((int)a.z, (int)b.z, acc);
  return __dp4a((int)a.w, (int)b.w, acc);
}

// 16 codes from column `off` of a row of K (off < K), zero past its end.
YN_DEV uint4 i8_codes16(const int8_t* row, int off, int K) {
  if (off + 16 <= K) return ldg_nc_v4(row + off);
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; off + i < K; ++i) w[i >> 2] |= (uint32_t)(uint8_t)row[off + i] << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Codes and scale of one row of K elements into shared memory by `n` threads (the whole
// block, or one warp), zero up to KP. The elements are read twice (from L1 or L2 the second
// time): rows are a few KB.
template <bool BLOCK, typename T>
YN_DEV void i8_row_smem_t(const void* x, size_t base, int K, int KP, int8_t* codes, float* scale, uint32_t* buf) {
  const int at = BLOCK ? threadIdx.x : threadIdx.x & 31, n = BLOCK ? (int)blockDim.x : 32;
  const bool vec = (reinterpret_cast<uintptr_t>(reinterpret_cast<const T*>(x) + base) & 15u) == 0;
  const int n8 = vec ? K / 8 : 0;
  uint32_t m = 0;
#pragma unroll 2
  for (int i = at; i < n8; i += n) {
    I8Raw<T> r;
    float f[8];
    r.load(x, base + 8 * (size_t)i);
    r.get(f);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, i8_abs_bits(f[j]));
  }
  for (int k = 8 * n8 + at; k < K; k += n) m = max(m, i8_abs_bits(I8In<T>::load(x, base + k)));
  if (BLOCK) m = block_max_u32(m, buf);
  else m = __reduce_max_sync(0xffffffffu, m);
  const I8Row q(m);
  if (at == 0) *scale = q.scale();
#pragma unroll 2
  for (int i = at; i < KP / 8; i += n) {
    I8Raw<T> r;
    float f[8];
    if (i < n8) {
      r.load(x, base + 8 * (size_t)i);
      r.get(f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 8 * i + j < K ? I8In<T>::load(x, base + 8 * i + j) : 0.0f;
    }
    uint32_t w[2];
    q.codes<sizeof(T) == 2>(f, w);
    *reinterpret_cast<uint2*>(codes + 8 * i) = make_uint2(w[0], w[1]);
  }
}
template <bool BLOCK>
YN_DEV void i8_row_smem(int dt, const void* x, size_t base, int K, int KP, int8_t* codes, float* scale, uint32_t* buf) {
  if (dt == YN_F32) i8_row_smem_t<BLOCK, float>(x, base, K, KP, codes, scale, buf);
  else if (dt == YN_BF16) i8_row_smem_t<BLOCK, __nv_bfloat16>(x, base, K, KP, codes, scale, buf);
  else i8_row_smem_t<BLOCK, __half>(x, base, K, KP, codes, scale, buf);
}

struct I8Mat {
  const int8_t* codes;
  const float* scales;
  long long row_stride, mat_stride, scale_stride;
};

// R rows of codes (row pointers) times T rows in shared memory: per-lane sums, then the
// whole dot product on every lane.
template <int R, int T, int U>
YN_DEV void i8_dots(const int8_t* const (&w)[R], const int8_t* xs, int KP, int K, int lane, int (&acc)[R][T]) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < T; ++t) acc[r][t] = 0;
  for (int k0 = 0; k0 < K; k0 += U * I8_GK) {
    uint4 a[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int off = k0 + u * I8_GK + 16 * lane;
#pragma unroll
      for (int r = 0; r < R; ++r) a[u][r] = off < K ? i8_codes16(w[r], off, K) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int off = k0 + u * I8_GK + 16 * lane;
      if (off < K) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const uint4 x = *reinterpret_cast<const uint4*>(xs + t * KP + off);
#pragma unroll
          for (int r = 0; r < R; ++r) acc[r][t] = dot16(a[u][r], x, acc[r][t]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < T; ++t) acc[r][t] = __reduce_add_sync(0xffffffffu, acc[r][t]);
}

// y (T, N) of T <= 5 rows (linear_few): every block makes the rows' codes itself (they are a few KB),
// then its warps take 4 output channels at a time through the matrix, which is read once:
// bound by that read with one row (2048 x 151936: 47.6 us, 6.54 TB/s), with more by the
// products too (three rows 51.8 us). A lane copies its own 16 codes of 4 channels per step into a ring of
// its warp (cp.async, I8_FS steps deep, 144 KB in flight per SM) and reads them back itself,
// so that neither the products nor the sums over lanes stop the copies and no thread waits
// for another. With five rows the ring took 59 us, loads into registers instead (8 per lane in
// flight) 71 us, twice as many of them 91 us.
constexpr int I8_FR = 4;    // channels per step
constexpr int I8_FS = 4;    // steps in the ring
constexpr int I8_FRING = I8_FS * I8_FR * I8_GK;   // bytes per warp

YN_DEV void i8_copy16(uint32_t dst, const void* src, int bytes) {   // bytes past `bytes` become 0
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <int T>
__global__ void __launch_bounds__(I8_GT, 3) k_i8_few(int dt, const void* x, long long ldx, int K, int KP, const I8Mat w,
                                                     int N, int odt, void* y, long long ldy) {
  extern __shared__ __align__(16) int8_t few_smem[];   // rings, then the rows' codes
  __shared__ float sx[T];
  __shared__ uint32_t buf[I8_GW];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int8_t* xs = few_smem + I8_GW * I8_FRING;
  const uint32_t ring = smem_u32(few_smem + warp * I8_FRING) + 16 * lane;
  const int NC = KP / I8_GK;
  const long long stride = (long long)gridDim.x * I8_GW * I8_FR, n_first = ((long long)blockIdx.x * I8_GW + warp) * I8_FR;
  // the step that is copied next
  long long cn = n_first;
  int cc = 0, cslot = 0;
  auto copy = [&]() {
    if (cn < N) {
      const int off = cc * I8_GK + 16 * lane, bytes = min(16, max(0, K - off));
#pragma unroll
      for (int r = 0; r < I8_FR; ++r) {
        const long long n = cn + r < N ? cn + r : (long long)N - 1;
        i8_copy16(ring + cslot * (I8_FR * I8_GK) + r * I8_GK, w.codes + n * w.row_stride + (bytes ? off : 0), bytes);
      }
      cslot = cslot + 1 < I8_FS ? cslot + 1 : 0;
      if (++cc == NC) {
        cc = 0;
        cn += stride;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < I8_FS - 1; ++i) copy();
  if (T == 1) i8_row_smem<true>(dt, x, 0, K, KP, xs, sx, buf);
  else if (warp < T) i8_row_smem<false>(dt, x, (size_t)warp * ldx, K, KP, xs + warp * KP, sx + warp, buf);
  __syncthreads();
  int slot = 0;
  for (long long n0 = n_first; n0 < N; n0 += stride) {
    int acc[I8_FR][T];
#pragma unroll
    for (int r = 0; r < I8_FR; ++r)
#pragma unroll
      for (int t = 0; t < T; ++t) acc[r][t] = 0;
    for (int c = 0; c < NC; ++c) {
      asm volatile("cp.async.wait_group %0;" ::"n"(I8_FS - 2) : "memory");
      uint4 a[I8_FR];
#pragma unroll
      for (int r = 0; r < I8_FR; ++r)
        a[r] = *reinterpret_cast<const uint4*>(few_smem + warp * I8_FRING + slot * (I8_FR * I8_GK) + r * I8_GK + 16 * lane);
      slot = slot + 1 < I8_FS ? slot + 1 : 0;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const uint4 q = *reinterpret_cast<const uint4*>(xs + t * KP + c * I8_GK + 16 * lane);
#pragma unroll
        for (int r = 0; r < I8_FR; ++r) acc[r][t] = dot16(a[r], q, acc[r][t]);
      }
      copy();   // into the slot read one step ago
    }
    // every lane gets all sums; lane r * T + t writes one
    float out = 0.0f;
#pragma unroll
    for (int r = 0; r < I8_FR; ++r)
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const int v = __reduce_add_sync(0xffffffffu, acc[r][t]);
        if (lane == r * T + t) out = (float)v;
      }
    const int r = lane / T, t = lane - r * T;
    if (r < I8_FR && n0 + r < N) i8_store(odt, y, (size_t)t * ldy + n0 + r, out * sx[t] * __ldg(w.scales + n0 + r));
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Few (row, expert) pairs: gate and up of 2 units per warp, the pair's row codes made by
// every block, SwiGLU in fp32 to act (pairs, I).
__global__ void __launch_bounds__(I8_GT) k_i8_up_few(int dt, const void* x, long long ldx, int H, int HP, const int32_t* ids,
                                                     int k, int E, const I8Mat gate, const I8Mat up, int I, float* act,
                                                    int* err) {
  extern __shared__ __align__(16) int8_t xs[];
  __shared__ float sx;
  __shared__ uint32_t buf[I8_GW];
  const int p = blockIdx.y, e = ids[p], warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  i8_launch_next();
  if (e < 0 || e >= E) {
    if (e != -1 && threadIdx.x == 0 && blockIdx.x == 0) raise_error(i8_err(err), YN_ERR_BAD_EXPERT);
    return;
  }
  i8_row_smem<true>(dt, x, (size_t)(p / k) * ldx, H, HP, xs, &sx, buf);
  __syncthreads();
  const int u0 = 2 * (blockIdx.x * I8_GW + warp);
  if (u0 >= I) return;
  const int u1 = u0 + 1 < I ? u0 + 1 : u0;
  const int8_t* g = gate.codes + e * gate.mat_stride;
  const int8_t* v = up.codes + e * up.mat_stride;
  const int8_t* rows[4] = {g + u0 * gate.row_stride, v + u0 * up.row_stride, g + u1 * gate.row_stride,
                           v + u1 * up.row_stride};
  int acc[4][1];
  i8_dots<4, 1, 2>(rows, xs, HP, H, lane, acc);
  if (lane < 2 && u0 + lane < I) {
    const int u = u0 + lane;
    const float gv = (float)(lane ? acc[2][0] : acc[0][0]) * sx * gate.scales[e * gate.scale_stride + u];
    const float uv = (float)(lane ? acc[3][0] : acc[1][0]) * sx * up.scales[e * up.scale_stride + u];
    act[(size_t)p * I + u] = i8_swiglu(gv, uv);
  }
}

// The down products of a row's experts and their weighted sum: a block makes the codes of
// the row's k activations, its warps take 2 outputs each through all k experts, 4 experts'
// rows in flight at a time, the first of them before the activations are there.
constexpr int I8_DJ = 4;
__global__ void __launch_bounds__(I8_GT) k_i8_down_few(const float* act, int I, int IP, const int32_t* ids, const float* wts,
                                                       int k, int E, const I8Mat down, int H, int odt, const void* res,
                                                       long long ldr, void* out, long long ldo) {
  extern __shared__ __align__(16) int8_t as[];
  __shared__ float sa[32];
  const int t = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h0 = 2 * (blockIdx.x * I8_GW + warp), h1 = h0 + 1 < H ? h0 + 1 : h0;
  const bool work = h0 < H;
  const int mine = lane < k ? ids[(size_t)t * k + lane] : -1;   // lane j: the row's expert j
  const float w_mine = lane < k ? wts[(size_t)t * k + lane] : 0.0f;
  uint4 a[I8_DJ][2];
  // rows of experts j0.. from column off on
  auto load = [&](int j0, int off) {
#pragma unroll
    for (int q = 0; q < I8_DJ; ++q) {
      const int e = __shfl_sync(0xffffffffu, mine, (j0 + q) & 31);
      const bool on = work && j0 + q < k && e >= 0 && e < E && off < I;
      const int8_t* d = down.codes + (on ? e * down.mat_stride : 0);
      a[q][0] = on ? i8_codes16(d + h0 * down.row_stride, off, I) : make_uint4(0, 0, 0, 0);
      a[q][1] = on ? i8_codes16(d + h1 * down.row_stride, off, I) : make_uint4(0, 0, 0, 0);
    }
  };
  load(0, 16 * lane);
  i8_wait_previous();
  for (int j = warp; j < k; j += I8_GW) {
    const int e = __shfl_sync(0xffffffffu, mine, j);
    if (e >= 0 && e < E) i8_row_smem_t<false, float>(act, ((size_t)t * k + j) * I, I, IP, as + j * IP, sa + j, nullptr);
  }
  __syncthreads();
  if (!work) return;
  float sum = 0.0f;   // of output h0 + (lane & 1)
  for (int j0 = 0; j0 < k; j0 += I8_DJ) {
    int acc[I8_DJ][2];
#pragma unroll
    for (int q = 0; q < I8_DJ; ++q) acc[q][0] = acc[q][1] = 0;
    for (int k0 = 0; k0 < I; k0 += I8_GK) {
      const int off = k0 + 16 * lane;
      if (j0 + k0 > 0) load(j0, off);
      if (off < I) {
#pragma unroll
        for (int q = 0; q < I8_DJ; ++q) {
          if (j0 + q >= k) break;
          const uint4 x = *reinterpret_cast<const uint4*>(as + (j0 + q) * IP + off);
          acc[q][0] = dot16(a[q][0], x, acc[q][0]);
          acc[q][1] = dot16(a[q][1], x, acc[q][1]);
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int q = 0; q < I8_DJ; ++q) {
      const int e = __shfl_sync(0xffffffffu, mine, (j0 + q) & 31);
      const float w = __shfl_sync(0xffffffffu, w_mine, (j0 + q) & 31);
      const int d0 = __reduce_add_sync(0xffffffffu, acc[q][0]), d1 = __reduce_add_sync(0xffffffffu, acc[q][1]);
      if (j0 + q >= k || e < 0 || e >= E) continue;
      sum = fmaf(w, (float)(lane & 1 ? d1 : d0) * sa[j0 + q] * __ldg(down.scales + e * down.scale_stride + (lane & 1 ? h1 : h0)), sum);
    }
  }
  if (lane < 2 && h0 + lane < H) {
    const size_t h = h0 + lane;
    i8_store(odt, out, (size_t)t * ldo + h, (res ? i8_load(odt, res, (size_t)t * ldr + h) : 0.0f) + sum);
  }
}

// --------------------------------------------- many rows: grouping, joining
constexpr int I8_PLAN_T = 1024;
constexpr int I8_PLAN_B = 8;     // blocks, one cluster
constexpr int I8_PLAN_Q = 4;     // pairs that a thread has in registers at a time
constexpr int I8_MAX_E = 1024;

// Pairs of one expert made contiguous and cut into chunks of at most NB rows. Which place
// a pair takes inside its expert does not change its product. pair_of: (row, column) ->
// pair, -1 where there is no expert. n_out[0] = chunks, [1] = pairs. The blocks of a
// cluster count a part of the pairs each, read one another's counts through distributed
// shared memory, and all make the same scan over the experts (16384 pairs: one block alone
// took 11 us, most of it atomics on popular experts).
__global__ void __cluster_dims__(I8_PLAN_B, 1, 1) __launch_bounds__(I8_PLAN_T)
    k_i8_plan(const int32_t* ids, int P, int E, int NB, int32_t* pair_of, I8Chunk* chunks, int* n_out, int* err) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ int cnt[I8_MAX_E], base_of[I8_MAX_E];
  __shared__ int2 ws[I8_PLAN_T / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, me = (int)cluster.block_rank();
  i8_launch_next();
  cnt[tid] = 0;
  __syncthreads();
  // part of the pairs: rounds of I8_PLAN_B * I8_PLAN_T * Q
  const int round = I8_PLAN_B * I8_PLAN_T * I8_PLAN_Q, rounds = (P + round - 1) / round;
  for (int k = 0; k < rounds; ++k) {
    const int i0 = k * round + me * (I8_PLAN_T * I8_PLAN_Q) + tid;
    int e[I8_PLAN_Q];
#pragma unroll
    for (int q = 0; q < I8_PLAN_Q; ++q) e[q] = i0 + q * I8_PLAN_T < P ? ids[i0 + q * I8_PLAN_T] : -1;
#pragma unroll
    for (int q = 0; q < I8_PLAN_Q; ++q) {
      const int i = i0 + q * I8_PLAN_T;
      if (i >= P) break;
      if (e[q] >= 0 && e[q] < E) pair_of[i] = atomicAdd(&cnt[e[q]], 1);   // place inside this block's share
      else {
        pair_of[i] = -1;
        if (e[q] != -1) raise_error(i8_err(err), YN_ERR_BAD_EXPERT);
      }
    }
  }
  cluster.sync();
  int c = 0, before = 0;   // expert tid: pairs of all blocks, and of those before this one
#pragma unroll
  for (int b = 0; b < I8_PLAN_B; ++b) {
    const int v = *cluster.map_shared_rank(&cnt[tid], b);
    c += v;
    before += b < me ? v : 0;
  }
  const int nc = (c + NB - 1) / NB;
  int2 inc = make_int2(c, nc);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, inc.x, o), b = __shfl_up_sync(0xffffffffu, inc.y, o);
    if (lane >= o) { inc.x += a; inc.y += b; }
  }
  if (lane == 31) ws[warp] = inc;
  __syncthreads();
  // the warps before: every warp sums its own
  int2 v = ws[lane];
  int2 base = lane < warp ? v : make_int2(0, 0);
  base.x = __reduce_add_sync(0xffffffffu, base.x);
  base.y = __reduce_add_sync(0xffffffffu, base.y);
  const int start = base.x + inc.x - c, at = base.y + inc.y - nc;
  base_of[tid] = start + before;
  if (me == tid % I8_PLAN_B)   // the blocks share the writing of the list
    for (int i = 0; i < nc; ++i) chunks[at + i] = I8Chunk{tid, start + i * NB, min(NB, c - i * NB)};
  if (me == 0 && tid == I8_PLAN_T - 1) {
    n_out[0] = at + nc;
    n_out[1] = start + c;
  }
  __syncthreads();
  for (int k = 0; k < rounds; ++k) {
    const int i0 = k * round + me * (I8_PLAN_T * I8_PLAN_Q) + tid;
    int e[I8_PLAN_Q], place[I8_PLAN_Q];
#pragma unroll
    for (int q = 0; q < I8_PLAN_Q; ++q) {
      const int i = i0 + q * I8_PLAN_T;
      place[q] = i < P ? pair_of[i] : -1;
      e[q] = i < P ? ids[i] : 0;
    }
#pragma unroll
    for (int q = 0; q < I8_PLAN_Q; ++q)
      if (place[q] >= 0) pair_of[i0 + q * I8_PLAN_T] = place[q] + base_of[e[q]];
  }
  cluster.sync();   // no block leaves while its counts are read
}

// out[t] = residual[t] + sum_j w_j y[pair_of[t][j]] in fp32, columns in order, rounded once: the
// products y stay fp32 until then, as they do in k_i8_down_few, so that a row comes out the same
// in a batch of any size.
// One row of the batch per blockIdx.x, 8 outputs per thread; VEC: residual and out in 16-byte pieces.
template <typename O, bool VEC>
__global__ void __launch_bounds__(128) k_i8_combine(const float* y, long long ldy, const int32_t* pair_of, const float* w, int k,
                                                    int H, const void* res, long long ldr, void* out, long long ldo) {
  i8_wait_previous();
  const size_t t = blockIdx.x;
  const int lane = threadIdx.x & 31, h = 8 * (blockIdx.y * 128 + threadIdx.x);
  const int p_mine = lane < k ? pair_of[t * k + lane] : -1;   // lane j: the row's pair j
  const float w_mine = lane < k ? w[t * k + lane] : 0.0f;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  const bool on = h < H;
  for (int j0 = 0; j0 < k; j0 += 4) {
    I8Raw<float> r[4];
    float wj[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {   // 4 rows of y in flight
      const int p = __shfl_sync(0xffffffffu, p_mine, (j0 + q) & 31);
      wj[q] = __shfl_sync(0xffffffffu, w_mine, (j0 + q) & 31);
      if (j0 + q >= k || p < 0) wj[q] = 0.0f;
      if (on && j0 + q < k && p >= 0) r[q].load(y, (size_t)p * ldy + h);   // rows of y are padded to whole pieces
      else r[q] = I8Raw<float>{};
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[8];
      r[q].get(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(wj[q], v[i], acc[i]);
    }
  }
  if (!on) return;
  if (VEC && h + 8 <= H) {
    if (res) {
      I8Raw<O> r;
      float v[8];
      r.load(res, t * ldr + h);
      r.get(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += v[i];
    }
    uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<O*>(out) + t * ldo + h);
    if constexpr (sizeof(O) == 4) {
      o[0] = make_uint4(__float_as_uint(acc[0]), __float_as_uint(acc[1]), __float_as_uint(acc[2]), __float_as_uint(acc[3]));
      o[1] = make_uint4(__float_as_uint(acc[4]), __float_as_uint(acc[5]), __float_as_uint(acc[6]), __float_as_uint(acc[7]));
    } else {
      o[0] = make_uint4(i8_pack2<O>(acc[0], acc[1]), i8_pack2<O>(acc[2], acc[3]), i8_pack2<O>(acc[4], acc[5]),
                        i8_pack2<O>(acc[6], acc[7]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (h + i < H) {
      const float r = res ? I8In<O>::load(res, t * ldr + h + i) : 0.0f;
      reinterpret_cast<O*>(out)[t * ldo + h + i] = i8_out<O>(r + acc[i]);
    }
}
template <typename O>
void launch_combine(const float* y, long long ldy, const int32_t* pair_of, const float* w, int k, int H, long long rows,
                    const void* res, long long ldr, void* out, long long ldo, cudaStream_t st) {
  const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (ldo * sizeof(O)) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(res) % 16 == 0 && (ldr * sizeof(O)) % 16 == 0;
  const dim3 g((unsigned)rows, (H + 1023) / 1024);
  if (vec) launch_after(k_i8_combine<O, true>, g, 128, 0, st, y, ldy, pair_of, w, k, H, res, ldr, out, ldo);
  else launch_after(k_i8_combine<O, false>, g, 128, 0, st, y, ldy, pair_of, w, k, H, res, ldr, out, ldo);
}

// ---------------------------------------------------------------- host side
size_t up_to(size_t v, size_t m) { return (v + m - 1) / m * m; }

int tmap(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  TmapEncode fn;
  int rc = host_tmap_encode(&fn);
  if (rc) return rc;
  const cuuint32_t one[5] = {1u, 1u, 1u, 1u, 1u};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? YN_OK : host_fail(YN_E_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
}
// The rows' codes in boxes of 16, 32, 64 and 128 rows.
int tmap_rows(I8Maps* maps, const void* base, long long cols, long long rows, long long stride) {
  for (int i = 0; i < I8_BMAPS; ++i) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {128u, 16u << i};
    const int rc = tmap(&maps->b[i], base, 2, dims, strides, box);
    if (rc) return rc;
  }
  return YN_OK;
}
// The matrices' rows: (K, rows, matrices), or (K, matrices, rows) where the matrices are interleaved row by
// row. cuTensorMapEncodeTiled asks that each stride be a multiple of the one before; a map whose strides
// are not so is accepted, but its boxes may touch memory past the last row.
bool mats_first(const yn_i8_mat& w) { return w.n_mats > 1 && w.rows > 1 && w.mat_stride < w.row_stride; }
bool strides_in_order(const yn_i8_mat& w) {
  if (w.n_mats == 1 || w.rows == 1) return true;
  if (mats_first(w)) return w.row_stride % w.mat_stride == 0 && w.row_stride / w.mat_stride >= w.n_mats;
  return w.mat_stride % w.row_stride == 0 && w.mat_stride / w.row_stride >= w.rows;
}
int tmap_mats(CUtensorMap* m, const yn_i8_mat& w, int box_rows) {
  const int r = mats_first(w) ? 2 : 1, e = 3 - r;   // places of the rows and of the matrices
  cuuint64_t dims[3], strides[2];
  cuuint32_t box[3];
  dims[0] = (cuuint64_t)w.cols;
  dims[r] = (cuuint64_t)w.rows;
  dims[e] = (cuuint64_t)w.n_mats;
  strides[r - 1] = (cuuint64_t)(w.n_mats > 1 && w.rows == 1 ? w.mat_stride : w.row_stride);
  strides[e - 1] = (cuuint64_t)(w.n_mats > 1 ? w.mat_stride : w.row_stride * (int64_t)w.rows);
  box[0] = 128u;
  box[r] = (cuuint32_t)box_rows;
  box[e] = 1u;
  return tmap(m, w.codes, 3, dims, strides, box);
}

int sm_count(int* out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev);
  return e == cudaSuccess ? YN_OK : host_fail(YN_E_CUDA, std::string("device attributes: ") + cudaGetErrorString(e));
}

template <typename O, bool UP, int NB>
int launch_gemm(const I8Gemm& a, const I8Maps& maps, long long max_tiles, cudaStream_t st) {
  const void* kern = reinterpret_cast<const void*>(k_i8_gemm<O, UP, NB>);
  int rc = host_set_smem(kern, I8Cfg<NB>::SMEM), sms = 0;
  if (rc || (rc = sm_count(&sms))) return rc;
  const unsigned grid = 2 * (unsigned)std::max<long long>(1, std::min<long long>(max_tiles, sms / 2));
  launch_after(k_i8_gemm<O, UP, NB>, grid, I8_THREADS, I8Cfg<NB>::SMEM, st, a, maps);   // after the rows' codes
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? YN_OK : host_fail(YN_E_CUDA, std::string("8-bit product: ") + cudaGetErrorString(e));
}
// Rows per tile: 64 where most tiles have few rows (their time is the weights' way from HBM,
// and the smaller stages keep more of them in flight), else 256.
template <typename O, bool UP>
int launch_gemm_nb(int nb, const I8Gemm& a, const I8Maps& maps, long long max_tiles, cudaStream_t st) {
  if (max_tiles > 0x3fffffff) return host_fail(YN_E_UNSUPPORTED, "more than 2^30 tiles");
  return nb <= 64 ? launch_gemm<O, UP, 64>(a, maps, max_tiles, st) : launch_gemm<O, UP, 256>(a, maps, max_tiles, st);
}
int launch_gemm_out(int odt, int nb, const I8Gemm& a, const I8Maps& maps, long long max_tiles, cudaStream_t st) {
  if (odt == YN_F32) return launch_gemm_nb<float, false>(nb, a, maps, max_tiles, st);
  if (odt == YN_BF16) return launch_gemm_nb<__nv_bfloat16, false>(nb, a, maps, max_tiles, st);
  return launch_gemm_nb<__half, false>(nb, a, maps, max_tiles, st);
}

bool dtype_ok(int dt) { return dt == YN_F32 || dt == YN_BF16 || dt == YN_F16; }
int dtype_size(int dt) { return dt == YN_F32 ? 4 : 2; }
I8Mat mat_of(const yn_i8_mat& w) {
  return I8Mat{reinterpret_cast<const int8_t*>(w.codes), w.scales, w.row_stride, w.mat_stride, w.scale_stride};
}

constexpr int I8_MAX_K = 131072;   // 127^2 * 131072 < 2^31
// Rows of a product on dp4a: one row of any matrix that fits, and a few where a launch counts (small
// matrices) or where every block's work on their codes does not (short rows). K x N, us with 1 to 5 rows
// on dp4a and, with any of them, on the tensor cores, which have the codes made first:
//   2048 x 4096     5.0   6.2   6.4   7.0   7.4   |  8.4      4096 x 4096    6.9   9.7  10.2  10.3  11.2  | 11.1
//   2048 x 8192     6.6   7.8   8.4   8.7   9.7   |  9.2      8192 x 1024    8.3  14.4  14.7  19.0  21.2  | 17.2
//   2048 x 16384    8.5  10.5  11.0  11.9  13.1   | 10.9      8192 x 2048    8.9  15.0  15.3  19.3  21.5  | 17.5
//   2048 x 65536   22.7  24.8  26.0  28.0  30.5   | 26.2     16384 x 1024   13.0  33.4  35.0  35     38   | 29.9
//   2048 x 151936  47.6  50.8  51.8  55    62     | 51 to 52  2560 x 40000  17.8  20.6  21.8  23.5  29    | 21.2
//   1536 x 40000   12.2  13.4  14.2  16.0  17.5   | 14.8      4096 x 16384  13.4  17.2  21.3  23    25    | 15.6
constexpr int I8_FEW = 3, I8_FEW_MEDIUM = 4, I8_FEW_SMALL = 5;
constexpr long long I8_SMALL = 8ll << 20, I8_MEDIUM = 16ll << 20;   // codes of the matrix
constexpr long long I8_FEW_CODES = 6 * 1024, I8_FEW_CODES_MEDIUM = 24 * 1024;   // codes of the rows

int check_mat(const yn_i8_mat& w, const char* what) {
  const std::string n(what);
  if (!w.codes || !w.scales) return host_fail(YN_E_INVALID, n + ": null pointer");
  if (w.n_mats < 1 || w.rows < 1 || w.cols < 1) return host_fail(YN_E_INVALID, n + ": empty matrix");
  if (w.cols > I8_MAX_K) return host_fail(YN_E_UNSUPPORTED, n + ": at most 131072 columns (32-bit sums)");
  if (reinterpret_cast<uintptr_t>(w.codes) % 16 || w.row_stride % 16 || (w.n_mats > 1 && w.mat_stride % 16))
    return host_fail(YN_E_INVALID, n + ": rows of codes must start at multiples of 16 bytes");
  if (!host_aligned(4, w.scales)) return host_fail(YN_E_INVALID, n + ": scales must be aligned to their element");
  if (w.row_stride < w.cols || (w.n_mats > 1 && (w.mat_stride < w.cols || w.scale_stride < w.rows)))
    return host_fail(YN_E_INVALID, n + ": rows or matrices overlap");
  if (!strides_in_order(w))
    return host_fail(YN_E_UNSUPPORTED, n + ": matrices must lie one after another, whole rows apart, or be interleaved row by row");
  if (w.row_stride >= (1ll << 40) || w.mat_stride >= (1ll << 40)) return host_fail(YN_E_UNSUPPORTED, n + ": stride above 2^40");
  return YN_OK;
}

bool linear_few(long long rows, long long k, long long n) {
  if (rows == 1) return up_to(k, I8_GK) <= 96 * 1024;
  if (n * k > I8_MEDIUM) return rows <= I8_FEW && rows * k <= I8_FEW_CODES;
  return rows <= (n * k <= I8_SMALL ? I8_FEW_SMALL : I8_FEW_MEDIUM) && rows * k <= I8_FEW_CODES_MEDIUM;
}

template <int T>
int launch_few(int dt, const void* x, long long ldx, int K, const I8Mat& w, int N, int odt, void* y, long long ldy, int sms,
               cudaStream_t st) {
  const int KP = (int)up_to(K, I8_GK);
  const size_t smem = (size_t)T * KP + I8_GW * I8_FRING;
  const int rc = host_set_smem(reinterpret_cast<const void*>(k_i8_few<T>), 96 * 1024 + I8_GW * I8_FRING);
  if (rc) return rc;
  const int grid = std::min((N + I8_FR * I8_GW - 1) / (I8_FR * I8_GW), 3 * sms);
  k_i8_few<T><<<grid, I8_GT, smem, st>>>(dt, x, ldx, K, KP, w, N, odt, y, ldy);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? YN_OK : host_fail(YN_E_CUDA, std::string("8-bit product: ") + cudaGetErrorString(e));
}

// Workspace of the experts' products.
struct ExpertsWs {
  size_t n_out, pair_of, chunks, codes, sx, act, acodes, sa, y, total;
  long long ldc, lda, ldac, ldy;
  int nb;
};
// Rows per chunk of an expert, by the pairs per expert (see launch_gemm_nb). On 512 experts of 3 MB 64
// and 256 rows take 118 and 139 us at 5 pairs per expert, 154 and 181 at 10, 210 and 242 at 20, 325 and
// 336 at 40; on 64 experts of 9 MB 98 and 98 us at 7.5, 116 and 119 at 19, 137 and 137 at 38, 174 and 165
// at 75, 255 and 211 at 150.
int chunk_rows(long long pairs, int E) { return pairs <= 40ll * E ? 64 : 256; }
// Pairs that go to the dp4a kernels: two launches instead of six, but they read an expert's matrices
// for every pair. The two ways meet at about 120 MB of such reads: 30 pairs on 3 MB experts take 26 us so
// and 32 us grouped (40: 30 and 31, 50: 39 and 34), 8 pairs on 9 MB experts 21.5 and 27 us (16: 36 and 28).
bool experts_few(long long pairs, int k, int H, int I) {
  return (pairs <= 8 || (pairs <= 64 && pairs * 3 * H * I <= 120000000ll)) && up_to(H, I8_GK) <= 96 * 1024 &&
         k * up_to(I, I8_GK) <= 96 * 1024;
}

ExpertsWs experts_ws(long long rows, int k, int E, int H, int I) {
  ExpertsWs L{};
  size_t o = 0;
  auto take = [&](size_t b) { const size_t at = o; o = up_to(o + b, 256); return at; };
  const size_t P = (size_t)rows * k;
  if (experts_few((long long)P, k, H, I)) {
    L.act = take(P * I * 4);
    L.total = o;
    return L;
  }
  L.nb = chunk_rows((long long)P, E);
  L.ldc = (long long)up_to(H, 16);
  L.lda = (long long)up_to(I, 4);
  L.ldac = (long long)up_to(I, 16);
  L.ldy = (long long)up_to(H, 16);
  L.n_out = take(8);
  L.pair_of = take(P * 4);
  L.chunks = take((E + P / L.nb + 1) * sizeof(I8Chunk));
  L.codes = take(P * L.ldc);
  L.sx = take(P * 4);
  L.act = take(P * L.lda * 4);
  L.acodes = take(P * L.ldac);
  L.sa = take(P * 4);
  L.y = take(P * L.ldy * 4);
  L.total = o;
  return L;
}

}  // namespace ynb

using namespace ynb;

extern "C" int yn_i8_quant_rows(const void* x, int32_t dtype, int64_t row_stride, int64_t rows, int32_t cols, void* codes,
                                int64_t code_stride, float* scales, void* stream) {
  if (!dtype_ok(dtype)) return host_fail(YN_E_INVALID, "unknown dtype");
  if (rows < 0 || rows > 0x7fffffffLL || cols < 1 || row_stride < cols || code_stride < cols)
    return host_fail(YN_E_INVALID, "rows must be in [0, 2^31), strides at least cols, cols at least 1");
  if (rows == 0) return YN_OK;
  if (!x || !codes || !scales) return host_fail(YN_E_INVALID, "null argument");
  if (!host_aligned(dtype_size(dtype), x) || !host_aligned(4, scales))
    return host_fail(YN_E_INVALID, "x and scales must be aligned to their elements");
  return launch_quant(dtype, x, row_stride, rows, cols, nullptr, nullptr, 1, reinterpret_cast<int8_t*>(codes), code_stride, scales, true,
                      reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t yn_i8_linear_ws_bytes(int64_t rows, int32_t cols) {
  if (rows < 1 || cols < 1 || linear_few(rows, cols, I8_MEDIUM + 1)) return 0;   // few rows of a large matrix are few of any
  return up_to((size_t)rows * up_to(cols, 16), 256) + (size_t)rows * 4;
}

extern "C" int yn_i8_linear(const yn_i8_mat* w, const void* x, int32_t dtype, int64_t x_stride, int64_t rows, void* y,
                            int32_t y_dtype, int64_t y_stride, void* ws, size_t ws_bytes, void* stream) {
  if (!w) return host_fail(YN_E_INVALID, "null argument");
  int rc = check_mat(*w, "matrix");
  if (rc) return rc;
  if (w->n_mats != 1) return host_fail(YN_E_INVALID, "one matrix");
  if (!dtype_ok(dtype) || !dtype_ok(y_dtype)) return host_fail(YN_E_INVALID, "unknown dtype");
  if (rows < 0 || rows > 0x7fffff00LL || x_stride < w->cols || y_stride < w->rows)
    return host_fail(YN_E_INVALID, "rows must be in [0, 2^31 - 256), strides at least the row lengths");
  if (rows == 0) return YN_OK;
  if (!x || !y) return host_fail(YN_E_INVALID, "null argument");
  if (!host_aligned(dtype_size(dtype), x) || !host_aligned(dtype_size(y_dtype), y))
    return host_fail(YN_E_INVALID, "x and y must be aligned to their elements");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (linear_few(rows, w->cols, w->rows)) {
    const I8Mat m = mat_of(*w);
    int sms = 0;
    if ((rc = sm_count(&sms))) return rc;
#define YN_FEW(T) \
  case T: return launch_few<T>(dtype, x, x_stride, w->cols, m, w->rows, y_dtype, y, y_stride, sms, st)
    switch ((int)rows) {
      YN_FEW(1);
      YN_FEW(2);
      YN_FEW(3);
      YN_FEW(4);
      YN_FEW(5);
    }
#undef YN_FEW
  }
  if (!ws || reinterpret_cast<uintptr_t>(ws) % 256 || ws_bytes < yn_i8_linear_ws_bytes(rows, w->cols))
    return host_fail(YN_E_INVALID, "workspace too small or not 256-byte aligned");
  int8_t* codes = reinterpret_cast<int8_t*>(ws);
  const long long ldc = (long long)up_to(w->cols, 16);
  float* sx = reinterpret_cast<float*>(codes + up_to((size_t)rows * ldc, 256));
  if ((rc = launch_quant(dtype, x, x_stride, rows, w->cols, nullptr, nullptr, 1, codes, ldc, sx, true, st))) return rc;
  I8Gemm a{};
  a.rows = (int)rows;
  a.channels = w->rows;
  a.K = w->cols;
  a.half = 128;
  a.sx = sx;
  a.sw = w->scales;
  a.y = y;
  a.y_stride = y_stride;
  a.pairs = reinterpret_cast<uintptr_t>(y) % 4 == 0 && y_stride % 2 == 0;
  // 33 to 64 rows are the same on either tile where the weights' way counts (2048 x 151936: 57.2 and 57.7
  // us), and faster on the larger one elsewhere (2048 x 16384, 64 rows: 11.5 and 9.7)
  const int nb = rows <= 32 ? 64 : 256;
  int sms = 0;
  if ((rc = sm_count(&sms))) return rc;
  const long long pairs = std::max(1, sms / 2), rounds = (w->rows + 256 * pairs - 1) / (256 * pairs);
  if (nb == 64 && rounds > 1) {
    // bound by the weights' way from HBM: tiles that come out even over the pairs of SMs (6 rows of
    // 2048 x 151936: 53.6 -> 52.8 us, of 2048 x 65536 27.7 -> 26.2)
    a.half = (int)(up_to((size_t)((w->rows + rounds * pairs - 1) / (rounds * pairs)), 4) / 2);
  }
  I8Maps maps{};
  if ((rc = tmap_mats(&maps.a, *w, a.half)) || (rc = tmap_rows(&maps, codes, w->cols, rows, ldc))) return rc;
  const long long tiles = (long long)((rows + nb - 1) / nb) * ((w->rows + 2 * a.half - 1) / (2 * a.half));
  return launch_gemm_out(y_dtype, nb, a, maps, tiles, st);
}

extern "C" size_t yn_i8_experts_ws_bytes(int64_t rows, int32_t top_k, int32_t n_experts, int32_t hidden, int32_t inter,
                                         int32_t dtype) {
  if (rows < 1 || top_k < 1 || n_experts < 1 || hidden < 1 || inter < 1 || !dtype_ok(dtype)) return 0;
  return experts_ws(rows, top_k, n_experts, hidden, inter).total;
}

extern "C" int yn_i8_experts(const yn_i8_mat* gate, const yn_i8_mat* up, const yn_i8_mat* down, const void* x, int32_t dtype,
                             int64_t x_stride, int64_t rows, const int32_t* ids, const float* weights, int32_t top_k,
                             const void* residual, int64_t res_stride, void* out, int64_t out_stride, void* ws,
                             size_t ws_bytes, void* stream) {
  return yn_i8_experts_err(gate, up, down, x, dtype, x_stride, rows, ids, weights, top_k, residual, res_stride, out,
                           out_stride, ws, ws_bytes, nullptr, stream);
}

extern "C" int yn_i8_experts_err(const yn_i8_mat* gate, const yn_i8_mat* up, const yn_i8_mat* down, const void* x,
                                 int32_t dtype, int64_t x_stride, int64_t rows, const int32_t* ids, const float* weights,
                                 int32_t top_k, const void* residual, int64_t res_stride, void* out, int64_t out_stride,
                                 void* ws, size_t ws_bytes, int32_t* err, void* stream) {
  if (!gate || !up || !down) return host_fail(YN_E_INVALID, "null argument");
  int rc = check_mat(*gate, "gate");
  if (rc || (rc = check_mat(*up, "up")) || (rc = check_mat(*down, "down"))) return rc;
  const int E = gate->n_mats, H = gate->cols, I = gate->rows;
  if (up->n_mats != E || up->rows != I || up->cols != H || down->n_mats != E || down->rows != H || down->cols != I)
    return host_fail(YN_E_INVALID, "gate and up are (E, I, H), down is (E, H, I)");
  if (E > I8_MAX_E || top_k < 1 || top_k > 32) return host_fail(YN_E_UNSUPPORTED, "at most 1024 experts, top_k in [1, 32]");
  if (!dtype_ok(dtype)) return host_fail(YN_E_INVALID, "unknown dtype");
  if (rows < 0 || rows > (1 << 22) / top_k || x_stride < H || out_stride < H || (residual && res_stride < H))
    return host_fail(YN_E_INVALID, "rows * top_k must be in [0, 2^22], strides at least hidden");
  if (rows == 0) return YN_OK;
  if (!x || !ids || !weights || !out || !ws) return host_fail(YN_E_INVALID, "null argument");
  if (!host_aligned(dtype_size(dtype), x, out, residual) || !host_aligned(4, ids, weights, err))
    return host_fail(YN_E_INVALID, "rows, ids, weights and the error word must be aligned to their elements");
  const ExpertsWs L = experts_ws(rows, top_k, E, H, I);
  if (ws_bytes < L.total || reinterpret_cast<uintptr_t>(ws) % 256)
    return host_fail(YN_E_INVALID, "workspace too small or not 256-byte aligned");
  uint8_t* b = reinterpret_cast<uint8_t*>(ws);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int P = (int)(rows * top_k);
  const I8Mat mg = mat_of(*gate), mu = mat_of(*up), md = mat_of(*down);
  if (experts_few(P, top_k, H, I)) {
    float* act = reinterpret_cast<float*>(b + L.act);
    const int HP = (int)up_to(H, I8_GK), IP = (int)up_to(I, I8_GK);
    const size_t ds = (size_t)top_k * IP;
    if ((HP > 40 * 1024 && (rc = host_set_smem(reinterpret_cast<const void*>(k_i8_up_few), 96 * 1024))) ||
        (ds > 40 * 1024 && (rc = host_set_smem(reinterpret_cast<const void*>(k_i8_down_few), 96 * 1024))))
      return rc;
    k_i8_up_few<<<dim3((I + 2 * I8_GW - 1) / (2 * I8_GW), P), I8_GT, HP, st>>>(dtype, x, x_stride, H, HP, ids, top_k, E, mg, mu,
                                                                             I, act, err);
    launch_after(k_i8_down_few, dim3((H + 2 * I8_GW - 1) / (2 * I8_GW), (unsigned)rows), I8_GT, ds, st, act, I, IP, ids, weights,
                 top_k, E, md, H, dtype, residual, res_stride, out, out_stride);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? YN_OK : host_fail(YN_E_CUDA, std::string("experts: ") + cudaGetErrorString(e));
  }
  int* n_out = reinterpret_cast<int*>(b + L.n_out);
  int32_t* pair_of = reinterpret_cast<int32_t*>(b + L.pair_of);
  I8Chunk* chunks = reinterpret_cast<I8Chunk*>(b + L.chunks);
  int8_t* codes = reinterpret_cast<int8_t*>(b + L.codes);
  float* sx = reinterpret_cast<float*>(b + L.sx);
  float* act = reinterpret_cast<float*>(b + L.act);
  int8_t* acodes = reinterpret_cast<int8_t*>(b + L.acodes);
  float* sa = reinterpret_cast<float*>(b + L.sa);
  float* y = reinterpret_cast<float*>(b + L.y);
  k_i8_plan<<<I8_PLAN_B, I8_PLAN_T, 0, st>>>(ids, P, E, L.nb, pair_of, chunks, n_out, err);
  if ((rc = launch_quant(dtype, x, x_stride, rows, H, nullptr, pair_of, top_k, codes, L.ldc, sx, false, st))) return rc;
  const long long max_chunks = E + P / L.nb + 1;
  I8Maps maps{};
  I8Gemm g{};
  if ((rc = tmap_mats(&maps.a, *gate, 16)) || (rc = tmap_mats(&maps.a_up, *up, 16)) ||
      (rc = tmap_rows(&maps, codes, H, P, L.ldc)))
    return rc;
  g.mats_first = mats_first(*gate);
  g.up_mats_first = mats_first(*up);
  g.chunks = chunks;
  g.err = err;
  g.n_chunks = n_out;
  g.rows = P;
  g.channels = I;
  g.K = H;
  g.sx = sx;
  g.sw = gate->scales;
  g.sw_up = up->scales;
  g.sw_stride = gate->scale_stride;
  g.sw_up_stride = up->scale_stride;
  g.y = act;
  g.y_stride = L.lda;
  const long long tu = max_chunks * ((I + 127) / 128), td = max_chunks * ((H + 255) / 256);
  rc = launch_gemm_nb<float, true>(L.nb, g, maps, tu, st);
  if (rc) return rc;
  if ((rc = launch_quant(YN_F32, act, L.lda, P, I, n_out + 1, nullptr, 1, acodes, L.ldac, sa, false, st))) return rc;
  I8Maps md2{};
  if ((rc = tmap_mats(&md2.a, *down, 128)) || (rc = tmap_rows(&md2, acodes, I, P, L.ldac))) return rc;
  I8Gemm d{};
  d.chunks = chunks;
  d.err = err;
  d.n_chunks = n_out;
  d.rows = P;
  d.channels = H;
  d.K = I;
  d.half = 128;
  d.mats_first = mats_first(*down);
  d.sx = sa;
  d.sw = down->scales;
  d.sw_stride = down->scale_stride;
  d.y = y;
  d.y_stride = L.ldy;
  if ((rc = launch_gemm_nb<float, false>(L.nb, d, md2, td, st))) return rc;
  if (dtype == YN_BF16)
    launch_combine<__nv_bfloat16>(y, L.ldy, pair_of, weights, top_k, H, rows, residual, res_stride, out, out_stride, st);
  else if (dtype == YN_F16)
    launch_combine<__half>(y, L.ldy, pair_of, weights, top_k, H, rows, residual, res_stride, out, out_stride, st);
  else launch_combine<float>(y, L.ldy, pair_of, weights, top_k, H, rows, residual, res_stride, out, out_stride, st);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? YN_OK : host_fail(YN_E_CUDA, std::string("experts: ") + cudaGetErrorString(e));
}

extern "C" int yn_i8_error(void* stream, int32_t* code_out) {
  if (!code_out) return host_fail(YN_E_INVALID, "null argument");
  // A word that reads 0 is not cleared: a kernel of another stream may set it meanwhile. One that does not
  // read 0 takes no further error until it is cleared, and one caller at a time does that.
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, g_i8_err);
  if (e == cudaSuccess) e = cudaMemcpyAsync(code_out, p, 4, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *code_out) e = cudaMemsetAsync(p, 0, 4, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  return e == cudaSuccess ? YN_OK : host_fail(YN_E_CUDA, std::string("yn_i8_error: ") + cudaGetErrorString(e));
}
