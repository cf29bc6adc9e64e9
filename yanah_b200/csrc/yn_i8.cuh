// Matrix products in 8-bit integers: rows (tokens) and output channels each with one
// fp32 scale, y[t][r] = (sum_k qx[t][k] qw[r][k]) * sx[t] * sw[r], the sum exact in 32
// bits (127^2 * 131072 < 2^31). No counterpart in the reference, whose 8-bit matrices
// are group-affine (mlx_backend.py:305-306).
//
// Row codes: a = max |x|, scale = a / 127, q = the whole number nearest to 127 x / a,
// ties to even. The nearest one exactly: x with an 8- or 11-bit mantissa meets ties
// often (x = a / 2), so quotients within 2^-14 of a tie are settled by the remainder 127 x -
// q a, which fp32 holds exactly for 16-bit inputs, or for fp32 inputs taken again in fp64,
// where neither product nor quotient can reach or leave a tie by rounding.
#pragma once
#include <type_traits>

#include "yn_common.cuh"
#include "yn_tcgen05.cuh"

namespace ynb {

// Error word of the calls that were given none of their own, one per device: first error wins (yn_i8_error).
__device__ int g_i8_err;
YN_DEV int* i8_err(int* own) { return own ? own : &g_i8_err; }

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

// 8 elements as they lie in memory (16-byte aligned), and as fp32.
template <typename T>
struct I8Raw {
  uint4 v[sizeof(T) / 2];
  YN_DEV void load(const void* p, size_t i) {
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p) + i);
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) v[j] = q[j];
  }
  YN_DEV void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
      const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          f[4 * j + i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same_v<T, __half>) {
          f[2 * i] = f16_to_f32((uint16_t)(w[i] & 0xFFFFu));
          f[2 * i + 1] = f16_to_f32((uint16_t)(w[i] >> 16));
        } else {
          f[2 * i] = __uint_as_float(w[i] << 16);
          f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
      }
    }
  }
};

// A row's quantiser. A row with an infinity or a NaN has a NaN scale and codes of 0, so
// that its products are NaN and no other row's; a row of zeros has scale 0.
struct I8Row {
  float amax, inv;
  bool wide;   // 127 x or 127 / amax outside fp32: every code in fp64
  YN_DEV I8Row(uint32_t amax_bits) {
    amax = __uint_as_float(amax_bits);
    wide = amax < 1e-30f || (amax > 1e36f && amax_bits < 0x7F800000u);
    inv = amax_bits < 0x7F800000u && !wide ? __fdiv_rn(127.0f, amax) : 0.0f;
  }
  YN_DEV float scale() const {
    return __float_as_uint(amax) >= 0x7F800000u ? __int_as_float(0x7fc00000) : __fdiv_rn(amax, 127.0f);
  }
  // The codes of N values (N a multiple of 4), four to a word. Adding 1.5 * 2^23 rounds y to
  // the nearest whole number, ties to even, and leaves it in the low bits. Near a tie it is
  // settled from the remainder 127 x - q amax: for 16-bit inputs (NARROW) both terms have at
  // most 18 bits and fp32 has it exactly, else fp64.
  template <bool NARROW, int N>
  YN_DEV void codes(const float (&x)[N], uint32_t (&out)[N / 4]) const {
    float t[N];
    bool near = wide;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = __fmul_rn(x[i], inv);
      t[i] = __fadd_rn(y, 12582912.0f);
      near |= fabsf(__fsub_rn(y, __fsub_rn(t[i], 12582912.0f))) > 0.5f - 6.2e-5f;
    }
    if (near) {
      if (NARROW && !wide) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float q = __fsub_rn(t[i], 12582912.0f), d = fmaf(-q, amax, 127.0f * x[i]), a = 2.0f * fabsf(d);
          if (a > amax || (a == amax && (__float_as_int(t[i]) & 1))) t[i] += copysignf(1.0f, d);
        }
      } else {
#pragma unroll 1
        for (int k = 0; k < N; ++k) {   // one division in the code, N in a row that needs them
          float xv = 0.0f;
#pragma unroll
          for (int i = 0; i < N; ++i) xv = i == k ? x[i] : xv;
          const float q = amax > 0.0f ? (float)rint(127.0 * (double)xv / (double)amax) : 0.0f;
#pragma unroll
          for (int i = 0; i < N; ++i) t[i] = i == k ? __fadd_rn(q, 12582912.0f) : t[i];
        }
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

// The tensor-core product, by pairs of blocks (a cluster of two SMs, tcgen05 cta_group::2).
// One tile: 256 channels of one matrix x up to NB rows, each block with 128 of the channels
// (its own TMEM lanes) and half of the rows' codes in its shared memory; the pair's MMA (M
// 256, kind::i8) reads both halves, so a row's codes cross from L2 once per pair and a stage
// moves 32 KB per SM for 512 cycles of MMA where one block alone would move 48 KB (4096 rows
// of 64 experts: 334 us, 346 with single blocks). 4096 x 2048 x 16384 takes 92 us in single
// launches, 66 without its loads and its epilogue. Run after run the card's power limit holds it.
// A = the channels' codes, B = the rows' codes, both K-major in the 128-byte swizzled layout
// by TMA, 128 codes of K per stage (four MMAs of K 32); the accumulator is channels (lanes) x
// rows (columns), int32. UP interleaves 16 rows of the gate matrix with 16 of the up matrix,
// so that lanes l and l + 16 of an epilogue warp hold gate and up of the same unit.
struct I8Chunk {
  int e, p0, n;   // matrix, first row, rows (1..NB)
};

struct I8Gemm {
  const I8Chunk* chunks;   // null: one matrix, chunk c = rows [c * NB, ...) of `rows`
  const int* n_chunks;     // device count of `chunks`
  int rows, channels, K;
  int half;                // channels of a block's tile, even, 128 at most (UP: 64 units)
  const float* sx;         // (rows) row scales
  const float* sw;         // channel scales, sw_stride per matrix
  const float* sw_up;
  long long sw_stride, sw_up_stride;
  void* y;                 // (rows, y_stride): output, or UP: fp32 activations
  long long y_stride;
  int* err;                // error word, null: the device's
  bool mats_first, up_mats_first;   // map a (a_up) is (K, matrices, rows) instead of (K, rows, matrices)
  bool pairs;              // 16-bit outputs may be written two channels at a time (4-byte aligned rows)
};
// Tensor maps. a: the matrices' rows, boxes of 128 (UP: gate and up by a map each, boxes of 16; one map
// over both, whose strides are not in order, read past the end of the matrices). b[i]: the rows' codes,
// boxes of 16 << i.
constexpr int I8_BMAPS = 4;
struct I8Maps {
  CUtensorMap a, a_up, b[I8_BMAPS];
};

// A kernel of a call may be launched while the one before it runs (launch_after): it sets itself
// up, then waits until that one is done and its writes can be seen. Every thread of it waits, so
// that a kernel that is done has all before it done.
YN_DEV void i8_launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
YN_DEV void i8_wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

YN_DEV void i8_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Arrival on the barrier at this offset in both blocks once the MMAs issued so far are done.
YN_DEV void i8_commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// int32 accumulate (D format 2 at bits 4-5), signed 8-bit A and B (format 1), both
// K-major, N >> 3 at bits 17-22, M = 256 at bits 24-28
YN_DEV uint32_t i8_idesc(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (16u << 24);
}
// One thread of a converged warp. Under its predicate the compiler keeps the operands of copies and
// products in uniform registers; under `lane == 0` it moves each of them there for every instruction.
YN_DEV bool i8_elect() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
YN_DEV uint32_t i8_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address of block 0's copy of a barrier.
YN_DEV uint32_t i8_leader(uint64_t* bar) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(bar)));
  return a;
}
YN_DEV void i8_arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
YN_DEV void i8_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Copies and commits complete a barrier of this block by themselves; only where threads of the other
// block arrive does a wait have to acquire from the cluster, which costs far more.
template <bool CLUSTER>
YN_DEV bool i8_try_wait(uint64_t* bar, uint32_t phase) {
  uint32_t ok;
  if (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(phase)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(phase)
        : "memory");
  return ok != 0;
}
// A wait of one thread, at most 1 s: on a timeout the error word is set and every role leaves
// its loop.
template <bool CLUSTER = false>
YN_DEV bool i8_wait1(uint64_t* bar, uint32_t phase, int* err) {
  if (i8_try_wait<CLUSTER>(bar, phase)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!i8_try_wait<CLUSTER>(bar, phase))
    if (globaltimer_ns() - t0 > 1000000000ull) {
      raise_error(err, YN_ERR_BULK_TIMEOUT);
      return false;
    }
  return true;
}
// The same of a whole warp.
YN_DEV bool i8_wait(uint64_t* bar, uint32_t phase, int* err) { return __all_sync(0xffffffffu, i8_wait1(bar, phase, err)) != 0; }
// Tile copies of this block whose bytes are counted on a barrier of the pair's first block.
YN_DEV void i8_tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(cluster_bar)
      : "memory");
}
YN_DEV void i8_tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint32_t cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(cluster_bar)
      : "memory");
}
// 16 consecutive 32-bit columns of this thread's TMEM lane. The wait takes the registers
// through it, so that nothing reads them before it.
YN_DEV void i8_ld16(uint32_t taddr, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}

constexpr int I8_EPW = 16;                   // epilogue warps (warp % 4: TMEM lanes 32 (warp % 4)..+31)
constexpr int I8_MW = I8_EPW, I8_LW = I8_EPW + 1;
constexpr int I8_THREADS = 32 * (I8_EPW + 2);
constexpr int I8_A_BYTES = 128 * 128;        // a block's channels, one stage

template <int NB>
struct I8Cfg {
  static constexpr int STAGE = I8_A_BYTES + NB / 2 * 128;
  static constexpr int FIT = (224 * 1024) / STAGE;
  static constexpr int S = FIT < 8 ? FIT : 8;          // stages in flight: with 8 of 18 KB HBM is as fast as it gets
  static constexpr int ACC = 512 / NB < 4 ? 512 / NB : 4;   // accumulators of NB columns in TMEM
  static constexpr int GROUPS = NB <= 64 ? ACC : 1;         // groups of epilogue warps, a tile each
  static constexpr int SPLIT = I8_EPW / 4 / GROUPS;         // warps of a group on the same 32 lanes
  static constexpr int PIECES = NB / (16 * SPLIT);          // 16-column pieces of such a warp
  static constexpr int SMEM = 1024 + S * STAGE + (2 * S + 2 * ACC) * 8 + 16;
  static_assert(NB % 32 == 0 && NB <= 256, "two accumulators have to fit TMEM");
  static_assert(2 * SMEM > 228 * 1024, "each block takes an SM's whole TMEM: no two may share one");
};

// SiLU(g) * u in fp32.
YN_DEV float i8_swiglu(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

// Warp-specialised and persistent: in both blocks a loader warp fills a ring of stages by
// TMA and epilogue warps drain the accumulators; the first block's MMA warp multiplies for
// both, into one of the accumulators while the others are drained.
// full[s] (first block): the bytes of both blocks' stage s; empty[s] (each block): its MMAs
// are done; acc_full[b] (each block); acc_empty[b] (first block): the accumulator's epilogue warps of both.
template <typename O, bool UP, int NB>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8_THREADS, 1)
    k_i8_gemm(const I8Gemm a, const __grid_constant__ I8Maps maps) {
  using F = I8Cfg<NB>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + F::S * F::STAGE);
  uint64_t* empty = full + F::S;
  uint64_t* acc_full = empty + F::S;
  uint64_t* acc_empty = acc_full + F::ACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + F::ACC);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)i8_rank();
  int* err = i8_err(a.err);

  const int tile_half = UP ? 64 : a.half, TILE = 2 * tile_half;   // units or channels of a block's and of a pair's tile
  const int UT = (a.channels + TILE - 1) / TILE;
  const int step = (int)(gridDim.x >> 1), t0 = (int)(blockIdx.x >> 1), NK = (a.K + 127) / 128;
  i8_launch_next();
  if (tid == 0) {
    for (int s = 0; s < F::S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < F::ACC; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * I8_EPW / F::GROUPS);
    }
    fence_mbar_init();
  }
  if (warp == I8_MW) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  i8_cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  i8_wait_previous();
  const int n_chunks = a.chunks ? *a.n_chunks : (a.rows + NB - 1) / NB, n_tiles = n_chunks * UT;
  // A list's tiles go unit by unit through a chunk, so that neighbours share the rows; a
  // single matrix's go chunk by chunk through its channels, so that they share the weights.
  // Every role looks its tiles up two ahead.
  struct Tile {
    I8Chunk c;
    int u0;
  };
  auto tile = [&](int ti) -> Tile {
    if (ti >= n_tiles) return Tile{I8Chunk{0, 0, 0}, 0};
    if (a.chunks) {
      const int c = ti / UT;
      return Tile{a.chunks[c], TILE * (ti - c * UT) + tile_half * rank};
    }
    const int u = ti / n_chunks, c = ti - u * n_chunks;
    return Tile{I8Chunk{0, c * NB, min(NB, a.rows - c * NB)}, TILE * u + tile_half * rank};
  };
  Tile next = tile(t0), after = tile(t0 + step);

  if (warp < I8_EPW) {
    // Tiles of few rows are short (4 stages of K 512 come in 1.6 us) and draining one is a chain of
    // TMEM loads, exchanges and stores that takes longer: every accumulator has warps of its own then,
    // which take every 4th tile (2048 x 512 experts, 166 MB: 49 -> 41 us). All warps on each tile
    // is better for long ones (4096 x 2048 x 16384: 115 us, 121 us in groups, when measured). A tile's scales are
    // loaded while the group's tile before it is drained.
    const int q = warp & 3, group = (warp >> 2) % F::GROUPS, part = (warp >> 2) / F::GROUPS;
    const int r_in = UP ? 16 * q + (lane & 15) : 32 * q + lane, ahead = F::GROUPS * step;
    struct Scales {
      float sw, su, sx[F::PIECES];
    };
    auto scales = [&](const Tile& t) -> Scales {
      Scales o;
      const int r = t.u0 + r_in;
      const bool in = r < a.channels && t.c.n > 0;
      o.sw = in ? a.sw[t.c.e * a.sw_stride + r] : 0.0f;
      o.su = UP && in ? a.sw_up[t.c.e * a.sw_up_stride + r] : 0.0f;
#pragma unroll
      for (int i = 0; i < F::PIECES; ++i) {
        const int col = 16 * (part + F::SPLIT * i) + lane;
        o.sx[i] = lane < 16 && col < t.c.n ? a.sx[t.c.p0 + col] : 0.0f;
      }
      return o;
    };
    next = tile(t0 + group * step);
    after = tile(t0 + group * step + ahead);
    Scales sc = scales(next);
    int j = group;
    for (int ti = t0 + group * step; ti < n_tiles; ti += ahead, j += F::GROUPS) {
      const I8Chunk c = next.c;
      const int u0 = next.u0, r = u0 + r_in, b = j % F::ACC;
      const float sw = sc.sw, su = sc.su;
      float sxs[F::PIECES];
#pragma unroll
      for (int i = 0; i < F::PIECES; ++i) sxs[i] = sc.sx[i];
      next = after;
      after = tile(ti + 2 * ahead);
      sc = scales(next);
      const bool mine = UP || r_in < tile_half, in = mine && r < a.channels;
      ok = i8_wait(&acc_full[b], (uint32_t)(j / F::ACC) & 1, err);
      if (!ok) break;
      tc_fence_after();
      const uint32_t base = tmem + (uint32_t)(b * NB) + ((uint32_t)(32 * q) << 16);
#pragma unroll
      for (int i = 0; i < F::PIECES; ++i) {
        const int c0 = 16 * (part + F::SPLIT * i);
        if (c0 >= c.n) break;
        const int left = c.n - c0;
        const long long row = c.p0 + c0;
        const float sx = sxs[i];
        int v[16];
        i8_ld16(base + (uint32_t)c0, v);
        if (UP) {
          // lanes below 16 take the even rows, the others the odd ones
          const bool up = lane & 16;
          float* out = reinterpret_cast<float*>(a.y) + (row + up) * a.y_stride + r;
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const int got = __shfl_xor_sync(0xffffffffu, up ? v[k] : v[k + 1], 16);
            const float s = __shfl_sync(0xffffffffu, sx, k + up);
            const float g = (float)(up ? got : v[k]) * s * sw, u = (float)(up ? v[k + 1] : got) * s * su;
            if (k + up < left && in) out[(size_t)k * a.y_stride] = i8_swiglu(g, u);
          }
        } else if (sizeof(O) == 2 && a.pairs) {
          // two lanes exchange so that each writes two adjacent channels of every second row
          // (even lanes the even rows)
          const bool odd = lane & 1, two = (r | 1) < a.channels;
          const uint32_t sel = odd ? 0x3276u : 0x5410u;
          uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<O*>(a.y) + (row + odd) * a.y_stride + (r & ~1));
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const float f0 = (float)v[k] * __shfl_sync(0xffffffffu, sx, k) * sw;
            const float f1 = (float)v[k + 1] * __shfl_sync(0xffffffffu, sx, k + 1) * sw;
            const uint32_t own = i8_pack2<O>(f0, f1);
            const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
            const uint32_t pk = __byte_perm(own, other, sel);
            if (k + odd < left && mine) {
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
      __syncwarp();
      if (lane == 0) i8_arrive_at(i8_leader(&acc_empty[b]));
    }
  } else if (warp == I8_MW) {
    // One elected thread: few MMAs wait in the tensor core's queue, so what it does between them
    // counts (4096 x 2048 x 16384: 92 us; 104 by lane 0, 116 by whole warps that elected one per step).
    if (i8_elect() && rank == 0) {
      int j = 0, s = 0;
      uint32_t full_phase = 0;
      const uint64_t a0 = tc_desc(smem_u32(smem)), b0 = tc_desc(smem_u32(smem) + I8_A_BYTES);
      for (int ti = t0; ti < n_tiles && ok; ti += step, ++j) {
        const int n = next.c.n, b = j % F::ACC;
        next = after;
        after = tile(ti + 2 * step);
        if (j >= F::ACC) ok = i8_wait1<true>(&acc_empty[b], (uint32_t)(j / F::ACC - 1) & 1, err);
        tc_fence_after();
        const uint32_t idesc = i8_idesc((n + 31) & ~31), dcol = tmem + (uint32_t)(b * NB);
        for (int kc = 0; kc < NK && ok; ++kc) {
          ok = i8_wait1(&full[s], full_phase, err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t ad = a0 + (uint32_t)(s * (F::STAGE >> 4)), bd = b0 + (uint32_t)(s * (F::STAGE >> 4));
#pragma unroll
          for (int k = 0; k < 4; ++k) i8_mma(dcol, ad + 2 * k, bd + 2 * k, idesc, kc > 0 || k > 0 ? 1u : 0u);
          i8_commit_both(&empty[s]);
          if (kc == NK - 1) i8_commit_both(&acc_full[b]);
          if (++s == F::S) {
            s = 0;
            full_phase ^= 1;
          }
        }
      }
      // the last commits must land before TMEM is released (bounded)
      if (ok && j > 0) (void)i8_wait1(&acc_full[(j - 1) % F::ACC], (uint32_t)((j - 1) / F::ACC) & 1, err);
    }
    __syncwarp();
  } else {
    if (i8_elect()) {
      int s = 0, used = 0;
      uint32_t empty_phase = 1;   // the first round finds the ring empty
      for (int ti = t0; ti < n_tiles && ok; ti += step) {
        const I8Chunk c = next.c;
        const int u0 = next.u0;
        next = after;
        after = tile(ti + 2 * step);
        const int half = ((c.n + 31) & ~31) >> 1, row = c.p0 + rank * half;   // this block's half of the MMA's rows
        const int bi = half <= 16 ? 0 : half <= 32 ? 1 : half <= 64 ? 2 : 3;
        const uint32_t bytes = 2u * ((UP ? 128u : (uint32_t)tile_half) + (16u << bi)) * 128u;
        for (int kc = 0; kc < NK; ++kc) {
          if (used == F::S) ok = i8_wait1(&empty[s], empty_phase, err);
          else ++used;
          if (!ok) break;
          uint8_t* st = smem + s * F::STAGE;
          const uint32_t bar = i8_leader(&full[s]);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
          auto weights = [&](void* dst, const CUtensorMap* map, bool first, int r) {
            i8_tma_3d(dst, map, 128 * kc, first ? c.e : r, first ? r : c.e, bar);
          };
          if (UP) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              weights(st + 4096 * i, &maps.a, a.mats_first, u0 + 16 * i);
              weights(st + 4096 * i + 2048, &maps.a_up, a.up_mats_first, u0 + 16 * i);
            }
          } else {
            weights(st, &maps.a, a.mats_first, u0);
          }
          i8_tma_2d(st + I8_A_BYTES, &maps.b[bi], 128 * kc, row, bar);
          if (++s == F::S) {
            s = 0;
            empty_phase ^= 1;
          }
        }
      }
      // every stage filled must have been read (its copies and MMAs done) before the block ends: the
      // ring's `used` slots, the oldest first
      if (used < F::S) {
        s = 0;
        empty_phase = 0;
      }
      for (int i = 0; i < used && ok; ++i) {
        ok = i8_wait1(&empty[s], empty_phase, err);
        if (++s == F::S) {
          s = 0;
          empty_phase ^= 1;
        }
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  i8_cluster_sync();   // neither block leaves, or gives its TMEM back, while the other may still signal it
  tc_fence_after();
  if (warp == I8_MW) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace ynb
