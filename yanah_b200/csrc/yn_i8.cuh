// Matrix products in 8-bit integers: rows (tokens) and output channels each with one
// fp32 scale, y[t][r] = (sum_k qx[t][k] qw[r][k]) * sx[t] * sw[r], the sum exact in 32
// bits (127^2 * 131072 < 2^31). No counterpart in the reference, whose 8-bit matrices
// are group-affine (mlx_backend.py:305-306).
//
// Row codes: a = max |x|, scale = a / 127, q = the whole number nearest to 127 x / a,
// ties to even. The nearest one exactly: x with an 8- or 11-bit mantissa meets ties
// often (x = a / 2), so quotients within 2^-14 of a tie are taken again in fp64, where
// neither product nor quotient can reach or leave a tie by rounding.
#pragma once
#include <type_traits>

#include "yn_common.cuh"
#include "yn_tcgen05.cuh"

namespace ynb {

// Error word of these kernels, one per device: first error wins (yn_i8_error).
__device__ int g_i8_err;

template <typename T>
struct I8In;
template <>
struct I8In<float> {
  YN_DEV static float load(const void* p, size_t i) { return reinterpret_cast<const float*>(p)[i]; }
};
template <>
struct I8In<__nv_bfloat16> {
  YN_DEV static float load(const void* p, size_t i) { return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]); }
};
template <>
struct I8In<__half> {
  YN_DEV static float load(const void* p, size_t i) { return f16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]); }
};
template <typename T>
YN_DEV T i8_out(float v);
template <>
YN_DEV float i8_out<float>(float v) { return v; }
template <>
YN_DEV __nv_bfloat16 i8_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
YN_DEV __half i8_out<__half>(float v) { return __float2half_rn(v); }

template <typename O>
YN_DEV uint32_t i8_pack2(float lo, float hi) {
  if constexpr (std::is_same_v<O, __half>) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

// Element by element; 8 at a time where rows are 16-byte aligned.
template <typename T>
YN_DEV void i8_load8(const void* p, size_t i, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i)[0];
    const float4 b = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint16_t h = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
      if constexpr (std::is_same_v<T, __half>) f[j] = f16_to_f32(h);
      else f[j] = bf16_to_f32(h);
    }
  }
}

// A row's quantiser. A row with an infinity or a NaN has a NaN scale and codes of 0, so
// that its products are NaN and no other row's; a row of zeros has scale 0.
struct I8Row {
  float amax, inv;
  bool exact;   // 127 / amax outside fp32: every code in fp64
  YN_DEV I8Row(uint32_t amax_bits) {
    amax = __uint_as_float(amax_bits);
    exact = amax < 1e-30f;
    inv = amax > 0.0f && amax_bits < 0x7F800000u && !exact ? __fdiv_rn(127.0f, amax) : 0.0f;
    if (amax_bits >= 0x7F800000u) exact = false;
  }
  YN_DEV float scale() const {
    return __float_as_uint(amax) >= 0x7F800000u ? __int_as_float(0x7fc00000) : __fdiv_rn(amax, 127.0f);
  }
  // The codes of N values (N a multiple of 4), four to a word. Adding 1.5 * 2^23 rounds y to
  // the nearest whole number, ties to even, and leaves it in the low bits.
  template <int N>
  YN_DEV void codes(const float (&x)[N], uint32_t (&out)[N / 4]) const {
    float t[N];
    bool near = exact;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = __fmul_rn(x[i], inv);
      t[i] = __fadd_rn(y, 12582912.0f);
      near |= fabsf(__fsub_rn(y, __fsub_rn(t[i], 12582912.0f))) > 0.5f - 6.2e-5f;
    }
    if (near) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float y = __fmul_rn(x[i], inv);
        if (exact || fabsf(__fsub_rn(y, __fsub_rn(t[i], 12582912.0f))) > 0.5f - 6.2e-5f)
          t[i] = amax > 0.0f ? __fadd_rn((float)rint(127.0 * (double)x[i] / (double)amax), 12582912.0f) : 12582912.0f;
      }
    }
    const bool none = __float_as_uint(amax) >= 0x7F800000u;   // infinities and NaN stay out of the codes
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint32_t lo = __byte_perm(__float_as_uint(t[4 * i]), __float_as_uint(t[4 * i + 1]), 0x0040);
      const uint32_t hi = __byte_perm(__float_as_uint(t[4 * i + 2]), __float_as_uint(t[4 * i + 3]), 0x0040);
      out[i] = none ? 0u : __byte_perm(lo, hi, 0x5410);
    }
  }
};
YN_DEV uint32_t i8_abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

YN_DEV uint32_t block_max_u32(uint32_t v, uint32_t* buf) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t m = buf[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) m = max(m, buf[w]);
  return m;
}

// The tensor-core product. One tile: 128 output channels of one matrix x up to NB rows.
// A = the channels' codes, B = the rows' codes, both K-major in the 128-byte swizzled
// layout by TMA, 128 codes of K per stage (four tcgen05.mma kind::i8 of K 32); the
// accumulator is channels (TMEM lanes) x rows (columns), int32. UP doubles A: the same
// 128 units of the gate and of the up matrix into two accumulators, so that a thread of
// the epilogue holds both and SwiGLU needs no exchange.
struct I8Chunk {
  int e, p0, n;   // matrix, first row, rows (1..NB)
};

struct I8Gemm {
  const I8Chunk* chunks;   // null: one matrix, chunk c = rows [c * NB, ...) of `rows`
  const int* n_chunks;     // device count of `chunks`
  int rows, channels, K;
  const float* sx;         // (rows) row scales
  const float* sw;         // channel scales, sw_stride per matrix
  const float* sw_up;
  long long sw_stride, sw_up_stride;
  void* y;                 // (rows, y_stride): output, or UP: int16 activations
  long long y_stride;
  int store_cols;          // columns of a row that may be written: channels, or more where rows are padded
  bool pairs;              // 16-bit outputs may be written two channels at a time (4-byte aligned rows)
  float* bscale;           // UP: (rows, ceil(channels / 32)) scales of the activations' blocks
};
struct I8Maps {
  CUtensorMap a, a_up, b;
};

YN_DEV void i8_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// int32 accumulate (D format 2 at bits 4-5), signed 8-bit A and B (format 1), both
// K-major, N >> 3 at bits 17-22, M = 128 at bits 24-28
YN_DEV uint32_t i8_idesc(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
YN_DEV void i8_tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// 16 consecutive 32-bit columns of this thread's TMEM lane; wait with i8_ld_wait.
YN_DEV void i8_ld16(uint32_t taddr, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
// The wait takes the registers through it, so that nothing reads them before it.
YN_DEV void i8_ld_wait(int (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}

constexpr int I8_EPW = 16;                   // epilogue warps (warp % 4: TMEM lanes 32 (warp % 4)..+31)
constexpr int I8_MW = I8_EPW, I8_LW = I8_EPW + 1;
constexpr int I8_THREADS = 32 * (I8_EPW + 2);
constexpr int I8_A_BYTES = 128 * 128;

template <bool UP, int NB>
struct I8Cfg {
  static constexpr int STAGE = (UP ? 2 : 1) * I8_A_BYTES + NB * 128;
  static constexpr int FIT = (224 * 1024) / STAGE;
  static constexpr int S = FIT < 8 ? FIT : 8;          // stages in flight
  static constexpr int COLS = (UP ? 2 : 1) * NB;       // TMEM columns of one accumulator, two of them
  static constexpr int SMEM = 1024 + S * STAGE + (2 * S + 4) * 8 + 16;
  static_assert(2 * COLS <= 512, "two accumulators have to fit TMEM");
};

// SiLU(g) * u in fp32.
YN_DEV float i8_swiglu(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

// Warp-specialised and persistent: the loader warp fills a ring of stages by TMA, the
// MMA warp multiplies them into one of two accumulators, the epilogue warps drain the
// other. Waits are bounded as in the other tensor-core kernels: on a timeout the error
// word is set and every role leaves its loop.
template <typename O, bool UP, int NB>
__global__ void __launch_bounds__(I8_THREADS, 1) k_i8_gemm(const I8Gemm a, const __grid_constant__ I8Maps maps) {
  using F = I8Cfg<UP, NB>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + F::S * F::STAGE);
  uint64_t* empty = full + F::S;
  uint64_t* acc_full = empty + F::S;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* err = &g_i8_err;

  const int UT = (a.channels + 127) / 128;
  const int n_chunks = a.chunks ? *a.n_chunks : (a.rows + NB - 1) / NB;
  const long long n_tiles = (long long)n_chunks * UT;
  const int NK = (a.K + 127) / 128;
  if (tid == 0) {
    for (int s = 0; s < F::S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 32 * I8_EPW);
    }
    fence_mbar_init();
  }
  if (warp == I8_MW) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  // A list's tiles go unit by unit through a chunk, so that neighbours share the rows; a
  // single matrix's go chunk by chunk through 128 channels, so that they share the weights.
  auto tile = [&](long long ti, int& u0) -> I8Chunk {
    if (a.chunks) {
      const int c = (int)(ti / UT);
      u0 = 128 * (int)(ti - (long long)c * UT);
      return a.chunks[c];
    }
    const int u = (int)(ti / n_chunks), c = (int)(ti - (long long)u * n_chunks);
    u0 = 128 * u;
    return I8Chunk{0, c * NB, min(NB, a.rows - c * NB)};
  };

  if (warp < I8_EPW) {
    const int m = 32 * (warp & 3) + lane, part = warp >> 2;
    long long j = 0;
    for (long long ti = blockIdx.x; ti < n_tiles; ti += gridDim.x, ++j) {
      int u0;
      const I8Chunk c = tile(ti, u0);
      const int b = (int)(j & 1), r = u0 + m;
      const bool in = r < a.channels;
      const float sw = in ? a.sw[c.e * a.sw_stride + r] : 0.0f;
      const float su = UP && in ? a.sw_up[c.e * a.sw_up_stride + r] : 0.0f;
      ok = mbar_wait_bounded(&acc_full[b], (uint32_t)(j >> 1) & 1, err);
      ok = __all_sync(0xffffffffu, ok) != 0;
      if (!ok) break;
      tc_fence_after();
      const uint32_t base = tmem + (uint32_t)(b * F::COLS) + ((uint32_t)(32 * (warp & 3)) << 16);
      // A lane holds one channel of 16 rows: two lanes exchange so that each writes two adjacent
      // channels of every second row (even lanes the even rows).
      const bool odd = lane & 1, two = (r | 1) < a.store_cols;
      const uint32_t sel = odd ? 0x3276u : 0x5410u;
      for (int c0 = 16 * part; c0 < c.n; c0 += 4 * I8_EPW) {
        int v[16], w[16];
        i8_ld16(base + (uint32_t)c0, v);
        if (UP) i8_ld16(base + (uint32_t)(NB + c0), w);
        const int left = c.n - c0;
        const float sx = lane < min(16, left) ? a.sx[c.p0 + c0 + lane] : 0.0f;
        i8_ld_wait(v);
        if (UP) i8_ld_wait(w);
        const long long row = c.p0 + c0;
        if (UP) {
          // 16 bits relative to the largest of these 32 units: off by at most 2^-16 of it, 1/516 of
          // a step of the 8-bit code that follows
          uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<int16_t*>(a.y) + (row + odd) * a.y_stride + (r & ~1));
          float bm = 0.0f;
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            float t[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float s = __shfl_sync(0xffffffffu, sx, k + i);
              const float act = i8_swiglu((float)v[k + i] * s * sw, (float)w[k + i] * s * su);
              const uint32_t mb = __reduce_max_sync(0xffffffffu, i8_abs_bits(act));
              const float m = __uint_as_float(mb);
              if (lane == k + i) bm = m;
              t[i] = fmaf(act, m > 0.0f ? __fdividef(32767.0f, m) : 0.0f, 12582912.0f);   // the code in the low bits
            }
            const uint32_t own = __byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x5410);
            const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
            if (k + odd < left && (r & ~1) < a.channels) out[(size_t)k * a.y_stride / 2] = __byte_perm(own, other, sel);
          }
          if (lane < min(16, left) && u0 + 32 * (warp & 3) < a.channels)
            a.bscale[(row + lane) * ((a.channels + 31) / 32) + (u0 >> 5) + (warp & 3)] = bm;
        } else if (sizeof(O) == 2 && a.pairs) {
          uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<O*>(a.y) + (row + odd) * a.y_stride + (r & ~1));
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const float f0 = (float)v[k] * __shfl_sync(0xffffffffu, sx, k) * sw;
            const float f1 = (float)v[k + 1] * __shfl_sync(0xffffffffu, sx, k + 1) * sw;
            const uint32_t own = i8_pack2<O>(f0, f1);
            const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
            const uint32_t pk = __byte_perm(own, other, sel);
            if (k + odd < left) {
              if (two) out[(size_t)k * a.y_stride / 2] = pk;
              else if ((r & ~1) < a.channels)
                reinterpret_cast<uint16_t*>(out)[(size_t)k * a.y_stride] = (uint16_t)pk;
            }
          }
        } else {
          O* out = reinterpret_cast<O*>(a.y) + row * a.y_stride + r;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float f = (float)v[k] * __shfl_sync(0xffffffffu, sx, k) * sw;
            if (k < left && in) out[(size_t)k * a.y_stride] = i8_out<O>(f);
          }
        }
      }
      tc_fence_before();
      mbar_arrive1(&acc_empty[b]);
    }
  } else if (warp == I8_MW) {
    long long g = 0, j = 0;
    for (long long ti = blockIdx.x; ti < n_tiles && ok; ti += gridDim.x, ++j) {
      int u0;
      const I8Chunk c = tile(ti, u0);
      const int b = (int)(j & 1);
      if (j >= 2) ok = mbar_wait_bounded(&acc_empty[b], (uint32_t)((j >> 1) - 1) & 1, err);
      ok = __all_sync(0xffffffffu, ok) != 0;
      if (!ok) break;
      tc_fence_after();
      const uint32_t idesc = i8_idesc((c.n + 15) & ~15), dcol = tmem + (uint32_t)(b * F::COLS);
      for (int kc = 0; kc < NK; ++kc, ++g) {
        const int s = (int)(g % F::S);
        ok = mbar_wait_bounded(&full[s], (uint32_t)(g / F::S) & 1, err);
        ok = __all_sync(0xffffffffu, ok) != 0;
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t abase = smem_u32(smem + s * F::STAGE), bbase = abase + (UP ? 2 : 1) * I8_A_BYTES;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t acc = kc > 0 || k > 0 ? 1u : 0u;
            i8_mma(dcol, tc_desc(abase + 32 * k), tc_desc(bbase + 32 * k), idesc, acc);
            if (UP) i8_mma(dcol + NB, tc_desc(abase + I8_A_BYTES + 32 * k), tc_desc(bbase + 32 * k), idesc, acc);
          }
          tc_commit(&empty[s]);
          if (kc == NK - 1) tc_commit(&acc_full[b]);
        }
        __syncwarp();
      }
    }
    // the last commits must land before TMEM is released (bounded)
    if (ok && lane == 0 && j > 0) (void)mbar_wait_bounded(&acc_full[(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1, err);
    __syncwarp();
  } else {
    long long g = 0;
    for (long long ti = blockIdx.x; ti < n_tiles && ok; ti += gridDim.x) {
      int u0;
      const I8Chunk c = tile(ti, u0);
      for (int kc = 0; kc < NK; ++kc, ++g) {
        const int s = (int)(g % F::S);
        if (g >= F::S) ok = mbar_wait_bounded(&empty[s], (uint32_t)(g / F::S - 1) & 1, err);
        ok = __all_sync(0xffffffffu, ok) != 0;
        if (!ok) break;
        if (lane == 0) {
          uint8_t* st = smem + s * F::STAGE;
          mbar_arrive_expect_tx(&full[s], F::STAGE);
          i8_tma_3d(st, &maps.a, 128 * kc, u0, c.e, &full[s]);
          if (UP) i8_tma_3d(st + I8_A_BYTES, &maps.a_up, 128 * kc, u0, c.e, &full[s]);
          tc_tma_rows(st + (UP ? 2 : 1) * I8_A_BYTES, &maps.b, 128 * kc, c.p0, &full[s]);
        }
        __syncwarp();
      }
    }
    // every stage filled must have been read (its copies and MMAs done) before the block ends
    for (int s = 0; s < F::S && ok; ++s) {
      const long long last = g - 1 - ((g - 1 - s) % F::S + F::S) % F::S;   // last stage number in slot s
      if (last >= 0 && last < g) ok = mbar_wait_bounded(&empty[s], (uint32_t)(last / F::S) & 1, err);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == I8_MW) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace ynb
