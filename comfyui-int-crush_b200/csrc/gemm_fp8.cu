// Product of two e4m3 matrices with a scale for each block of 128:
//   out[m, n] = sum_b s_a[m, b] s_w[n / 128, b] sum_{k in block b} x[m, k] w[n, k] + bias[n]
// on tcgen05 (kind::f8f6f4).
//
// Persistent, one CTA per SM, 12 warps: warp 0 TMA producer, warp 1 MMA issuer,
// warps 4-11 the sums.  Tokens are the MMA's rows (TMEM lanes), features its
// columns, so that a thread owns one token row and a block's factor
// s_a * s_w is one number a thread: a weight block is 128 features wide and a
// warp's columns lie in one.  The 128 products of a block are summed on the
// tensor core (fp32 in tensor memory, accumulation off at the block's first
// MMA); the warps read the block's sums, hand the buffer back, and add them, times the
// factor, onto fp32 registers, 32 columns while the next 32 come out of tensor
// memory.  That is full of buffers (two of 256 columns, or four of 128): a block's
// MMAs run while the block before is read.
//
// Large problems: pairs of CTAs (cta_group::2), 256 x 256 a pair, every CTA
// staging half of each operand; 256 x 128 or one CTA's 128 x 128 where that leaves
// fewer SMs without a tile (launch_gemm_fp8).  Where the tiles are fewer than the
// SMs, clusters of CTAs share a tile's blocks: each pushes its partial sums to the
// CTAs that own their rows, which add them in rank order.
//
// What bounds it: the way of a block's sums.  512 clocks of MMAs, but 850 to 950 a
// block (256 x 256): 300 of FMAs a scheduler, the first columns' 130 from tensor
// memory, 100 to 150 for each question to a barrier beside the MMAs' operand
// reads, which take all of shared memory's width at full rate.  Two values an FMA
// instruction were slower (as many moves to pair them).  4608 x 12288 -> 4096: 238 us,
// 1950 TFLOP/s; 65520 x 5120 -> 13824: 4.87 ms, 1905 TFLOP/s under the power cap (1480
// to 1530 MHz); one row of 5120 x 5120: 9.4 us, 2.8 TB/s.
#include <string.h>

#include <atomic>
#include <type_traits>

namespace ic {

template <int BN_, bool PAIR_>
struct F8Cfg {
  static constexpr int BN = BN_;
  static constexpr bool PAIR = PAIR_;
  static constexpr int BM = 128;                       // rows of a CTA
  static constexpr int A_BYTES = BM * 128;
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;    // features that a CTA stages
  static constexpr int STAGE = A_BYTES + B_ROWS * 128;
  static constexpr int NST = BN == 256 ? 6 : PAIR ? 8 : 4;
  static constexpr int NB = 512 / BN;                  // buffers of tensor memory
  static constexpr int CPT = BN / 2;                   // columns of a thread (8 warps: 4 x 32 rows, 2 halves)
  static constexpr int OFF_STG = NST * STAGE;          // output staging, 4 KB a warp
  // a cluster's partial sums: of every CTA, the rows that this one adds up (they
  // lie over the staging, which a cluster does not use)
  static constexpr int PARTS = PAIR ? 0 : (128 + 8) * 128 * 4;
  static constexpr int OFF_BAR = OFF_STG + (PARTS > 8 * 4096 ? PARTS : 8 * 4096);
  static constexpr int SMEM = OFF_BAR + 256;
  static constexpr int THREADS = 384;
  // with 128 columns a thread: 384 x 168 registers
  static constexpr RegisterSplit REGS = {128, 40, 256, 232};
  static_assert(SMEM <= 232448, "shared memory");
};

struct F8Args {
  int M, N, kb;                 // kb: blocks along K
  int m_tiles, n_tiles;
  int splits;                   // CTAs of a cluster that share a tile's blocks
  const float* s_a;
  long long sa_row, sa_block;
  const float* s_w;
  long long sw_row, sw_block;
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  long long ldo;
  int tma_store;
  int a_rows;                   // rows of x that a CTA stages: 128, or fewer where there are
};

__device__ __forceinline__ void mma_f8_on(uint32_t on, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mma_f8_2_on(uint32_t on, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ uint32_t f8_elect() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on;
}
__device__ __forceinline__ void f8_commit_on(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(bar)), "r"(on)
      : "memory");
}
// on this barrier of both CTAs of the pair
__device__ __forceinline__ void f8_commit2_on(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}"
      ::"r"(smem_u32(bar)), "r"(on)
      : "memory");
}
// D = F32, A and B = e4m3 (format 0), both K-major
__host__ __device__ constexpr uint32_t idesc_f8(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void f8_tie(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void st_cluster4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

// Whether a phase is complete, without waiting for it.
__device__ __forceinline__ bool f8_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// A wait that was asked about beforehand: `early` is f8_test's answer, taken
// while there was other work.  Asking takes 100 to 150 clocks beside the MMAs'
// operand reads, also where the phase is long complete.
__device__ __forceinline__ bool f8_wait(bool early, uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (__all_sync(0xffffffffu, early)) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort));
}

// Tiles in groups of 8 row tiles, features slowest inside a group, so that the
// CTAs of a wave share rows and features in L2.
template <typename A>
__device__ __forceinline__ void f8_tile(const A& a, int tile, int& mt, int& nt) {
  constexpr int G = 8;
  const int per = G * a.n_tiles;
  const int g = tile / per, r = tile - g * per;
  const int rows = min(G, a.m_tiles - g * G);
  nt = r / rows;
  mt = g * G + r - nt * rows;
}

template <typename C>
__global__ void __launch_bounds__(C::THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                const __grid_constant__ CUtensorMap tm_o, const F8Args a) {
  constexpr int NST = C::NST, BN = C::BN, CPT = C::CPT, NB = C::NB;
  constexpr bool PAIR = C::PAIR;
  extern __shared__ __align__(1024) uint8_t smem[];   // no static shared memory: the declared alignment holds
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);   // [NST] TMA -> MMA
  uint64_t* empty = full + NST;                                       // [NST] MMA -> TMA
  uint64_t* acc_full = empty + NST;                                   // [NB] MMA -> sums
  uint64_t* acc_empty = acc_full + NB;                                // [NB] sums -> MMA (8 warps of each CTA)
  uint64_t* drain = acc_empty + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(drain + 2);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();       // of the pair, or of the split
  const bool leader = !PAIR || rank == 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NST; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, PAIR ? 16 : 8);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc2(tmem_slot, NB * BN);
      tmem_relinquish2();
    } else {
      tmem_alloc(tmem_slot, NB * BN);
      tmem_relinquish();
    }
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_o);
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR || a.splits > 1) cluster_sync_all();   // the others are there, their barriers initialised
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  const int tiles = a.m_tiles * a.n_tiles;
  const int first = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x / a.splits;
  const int step = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x / a.splits;
  // this CTA's blocks of a tile
  int kb0 = 0, kb1 = a.kb;
  if (!PAIR && a.splits > 1) {
    kb0 = (int)((long long)a.kb * rank / a.splits);
    kb1 = (int)((long long)a.kb * (rank + 1) / a.splits);
  }
  // what a cluster's CTA adds up: rows [rank * share, ...) of the tile, a lane four
  // columns from nc on, whose biases are here early
  int mt0 = 0, share = 1, nc = 0;
  float bias4[4] = {0.f, 0.f, 0.f, 0.f};
  const uint32_t parts = smem_u32(smem) + C::OFF_STG;
  if (!PAIR && a.splits > 1) {
    int nt0;
    f8_tile(a, first, mt0, nt0);
    share = (min(128, a.M - mt0 * 128) + a.splits - 1) / a.splits;
    nc = nt0 * BN + 4 * lane;
    if (a.bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (nc + j < a.N) bias4[j] = load_any(a.bias, a.bias_dtype, nc + j);
    }
  }
  constexpr int TILE_M = PAIR ? 256 : 128;
  const int m_off = PAIR ? (int)rank * 128 : 0;
  const uint32_t ring = smem_u32(smem);

  if (warp < 4) {
    if constexpr (CPT == 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS.few));
    if (warp == 0) {
      // ------------------------------------------------------------ producer
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true, early = false;
        for (int t = first; ok && t < tiles; t += step) {
          int mt, nt;
          f8_tile(a, t, mt, nt);
          const int row = mt * TILE_M + m_off, col = nt * BN + (PAIR ? (int)rank * C::B_ROWS : 0);
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const uint32_t s = it % NST, ph = (it / NST) & 1u;
            if (!early && !mbar_wait(empty + s, ph ^ 1u, abort_flag)) { ok = false; break; }
            uint8_t* st = smem + s * C::STAGE;
            if constexpr (PAIR) {
              // both halves count on the leader's barrier
              if (leader) mbar_arrive_expect_tx(full + s, 2 * (a.a_rows * 128 + C::B_ROWS * 128));
              const uint32_t bar = mapa_u32(smem_u32(full + s), 0u);
              tma_load_2d_pair(st, &tm_x, bar, kb * 128, row);
              tma_load_2d_pair(st + C::A_BYTES, &tm_w, bar, kb * 128, col);
            } else {
              mbar_arrive_expect_tx(full + s, a.a_rows * 128 + C::B_ROWS * 128);
              tma_load_2d(st, &tm_x, full + s, kb * 128, row);
              tma_load_2d(st + C::A_BYTES, &tm_w, full + s, kb * 128, col);
            }
            early = f8_test(empty + (it + 1) % NST, (((it + 1) / NST) & 1u) ^ 1u);
          }
        }
        // every copy issued lands before the CTA may leave, whoever gave up.  A
        // pair's count on the leader's barriers, and where one of the two gave up
        // before the other not all of them can be waited for there: those land in a
        // millisecond, as they do in microseconds.
        if (leader) {
          volatile int never = 0;
          for (uint32_t u = it > NST ? it - NST : 0; u < it; ++u) mbar_wait(full + u % NST, (u / NST) & 1u, &never);
        }
        if (PAIR && (!ok || *abort_flag)) {
          const uint64_t t0 = globaltimer();
          while (globaltimer() - t0 < 1000000) {}
        }
      }
    } else if (warp == 1 && leader) {
      // ---------------------------------------------------------- MMA issuer
      const uint32_t on = f8_elect();
      constexpr uint32_t idesc = idesc_f8(PAIR ? 256 : 128, BN);
      uint32_t it = 0;
      bool ok = true, staged = false, freed = false;
      for (int t = first; ok && t < tiles; t += step) {
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t s = it % NST, b = it % NB;
          // operands first: the buffer is what comes last
          ok = f8_wait(staged, full + s, (it / NST) & 1u, abort_flag) &&
               f8_wait(freed, acc_empty + b, ((it / NB) & 1u) ^ 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint64_t ad = smem_desc_sw128(ring + s * C::STAGE);
          const uint64_t bd = smem_desc_sw128(ring + s * C::STAGE + C::A_BYTES);
          const uint32_t d = tmem + b * BN;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (PAIR) mma_f8_2_on(on, d, ad + 2 * k, bd + 2 * k, idesc, k > 0);
            else mma_f8_on(on, d, ad + 2 * k, bd + 2 * k, idesc, k > 0);
          }
          if constexpr (PAIR) {
            f8_commit2_on(on, acc_full + b);
            f8_commit2_on(on, empty + s);
          } else {
            f8_commit_on(on, acc_full + b);
            f8_commit_on(on, empty + s);
          }
          staged = f8_test(full + (it + 1) % NST, ((it + 1) / NST) & 1u);
          freed = f8_test(acc_empty + (it + 1) % NB, (((it + 1) / NB) & 1u) ^ 1u);
        }
      }
      // all MMAs are done before tensor memory is freed
      // (committed by the lane that issued them)
      volatile int never = 0;
      if (on) {
        if constexpr (PAIR) mma_commit2_local(drain);
        else mma_commit(drain);
      }
      __syncwarp();
      mbar_wait(drain, 0, &never);
    }
  } else {
    // ------------------------------------------------------------------ sums
    if constexpr (CPT == 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS.many));
    const int e = warp - 4, q = e & 3, half = e >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(half * CPT);
    uint8_t* stg = smem + C::OFF_STG + e * 4096;
    uint32_t it = 0;
    bool ok = true, early = false;
    for (int t = first; ok && t < tiles; t += step) {
      int mt, nt;
      f8_tile(a, t, mt, nt);
      const int m0 = mt * TILE_M + m_off + 32 * q, n0 = nt * BN + half * CPT;
      const bool rows = m0 < a.M;   // or 32 rows that are not there
      const float* sa = a.s_a + (long long)min(m0 + lane, a.M - 1) * a.sa_row + kb0 * a.sa_block;
      const float* sw = a.s_w + (long long)(min(n0, a.N - 1) / 128) * a.sw_row + kb0 * a.sw_block;
      float acc[CPT];
#pragma unroll
      for (int j = 0; j < CPT; ++j) acc[j] = 0.f;
      // biases of columns n0 + lane + 32 i, here early
      float bias[CPT / 32];
      if (!(!PAIR && a.splits > 1)) {
#pragma unroll
        for (int i = 0; i < CPT / 32; ++i) {
          const int n = n0 + 32 * i + lane;
          bias[i] = a.bias && n < a.N ? load_any(a.bias, a.bias_dtype, n) : 0.f;
        }
      }
      // factors of two blocks ahead
      float fa[2], fw[2];
      fa[0] = __ldg(sa);
      fw[0] = __ldg(sw);
      sa += kb1 - kb0 > 1 ? a.sa_block : 0;
      sw += kb1 - kb0 > 1 ? a.sw_block : 0;
      fa[1] = __ldg(sa);
      fw[1] = __ldg(sw);
      // 32 columns at a time, the next ones on their way from tensor memory while
      // these are added; a block's last 32 after its buffer is handed back
      uint32_t r[2][32];
      constexpr int NC = CPT / 32;
      for (int kb2 = kb0; ok && kb2 < kb1; kb2 += 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (kb2 + i < kb1) {
            const uint32_t b = it % NB;
            ok = f8_wait(early, acc_full + b, (it / NB) & 1u, abort_flag);
            if (!ok) break;
            ++it;
            tc_fence_after();
            if (!rows) {
              __syncwarp();
              if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(mapa_u32(smem_u32(acc_empty + b), 0u));
                else mbar_arrive(acc_empty + b);
              }
              early = f8_test(acc_full + it % NB, (it / NB) & 1u);
              continue;
            }
            const float f = fa[i] * fw[i];
            const uint32_t src = lanes + b * BN;
            tmem_ld32(src, r[0]);
            if (kb2 + i + 2 < kb1) {
              sa += a.sa_block;
              sw += a.sw_block;
              fa[i] = __ldg(sa);
              fw[i] = __ldg(sw);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              tmem_wait_ld();
              f8_tie(r[c & 1]);
              if (c + 1 < NC) {
                tmem_ld32(src + 32 * (c + 1), r[(c + 1) & 1]);
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[32 * c + j] = fmaf(__uint_as_float(r[c & 1][j]), f, acc[32 * c + j]);
              }
            }
            // all is read: the buffer is the next MMAs'
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (PAIR) mbar_arrive_cluster(mapa_u32(smem_u32(acc_empty + b), 0u));
              else mbar_arrive(acc_empty + b);
            }
            early = f8_test(acc_full + it % NB, (it / NB) & 1u);
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[CPT - 32 + j] = fmaf(__uint_as_float(r[1][j]), f, acc[CPT - 32 + j]);
          }
        }
      }
      if (!ok) break;
      if (!PAIR && a.splits > 1) {
        // this CTA's partial sums to the CTAs that add them up.  16-byte chunks of a
        // row are XORed with the row's number, or all lanes would use the same banks.
        if (m0 + lane < a.M) {
          const int r = 32 * q + lane, owner = r / share;
          const uint32_t to = mapa_u32(parts + (rank * share + r - owner * share) * 512, owner);
#pragma unroll
          for (int c = 0; c < CPT / 4; ++c)
            st_cluster4(to + (((half * (CPT / 4) + c) ^ lane) << 4), acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
        }
        break;   // one tile a cluster
      }
      if (a.bias) {
        // to all lanes through the staging, once the box before has left it
        if (lane == 0) bulk_wait_read0();
        __syncwarp();
#pragma unroll
        for (int i = 0; i < CPT / 32; ++i) reinterpret_cast<float*>(stg)[32 * i + lane] = bias[i];
        __syncwarp();
#pragma unroll
        for (int j = 0; j < CPT / 4; ++j) {
          const float4 v = reinterpret_cast<const float4*>(stg)[j];
          acc[4 * j] += v.x; acc[4 * j + 1] += v.y; acc[4 * j + 2] += v.z; acc[4 * j + 3] += v.w;
        }
        __syncwarp();
      }
      // 4 KB of output at a time: 32 rows of 128 bytes, 128-byte-swizzled
      const int per = a.out_dtype == IC_DTYPE_F32 ? 32 : 64;   // columns
#pragma unroll
      for (int c = 0; c < CPT / 32; ++c) {
        const int n = n0 + 32 * c;   // 32 columns: a whole row of the box in fp32, half of one else
        const bool begin = per == 32 || (c & 1) == 0, end = per == 32 || (c & 1) == 1;
        if (begin) {
          if (lane == 0) bulk_wait_read0();   // the box before has left
          __syncwarp();
        }
        if (per == 32) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float* v = acc + 32 * c + 4 * j;
            *reinterpret_cast<float4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 u = make_float2(acc[32 * c + 8 * j + 2 * i], acc[32 * c + 8 * j + 2 * i + 1]);
              if (a.out_dtype == IC_DTYPE_F16) {
                const __half2 h = __floats2half2_rn(u.x, u.y);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
              } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(u.x, u.y);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
              }
            }
            const int chunk = 4 * (c & 1) + j;
            *reinterpret_cast<uint4*>(stg + lane * 128 + ((chunk ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        if (end) {
          const int nb = per == 32 ? n : n - 32;
          if (a.tma_store) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && nb < a.N && m0 < a.M) {
              tma_store_2d(&tm_o, stg, nb, m0);
              bulk_commit();
            }
          } else {
            __syncwarp();
            const int rows = min(32, a.M - m0);
            for (int r = 0; r < rows; ++r) {
              if (per == 32) {
                if (nb + lane < a.N)
                  reinterpret_cast<float*>(a.out)[(long long)(m0 + r) * a.ldo + nb + lane] =
                      *reinterpret_cast<const float*>(stg + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
              } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const int x = lane + 32 * i;
                  if (nb + x < a.N)
                    reinterpret_cast<uint16_t*>(a.out)[(long long)(m0 + r) * a.ldo + nb + x] =
                        *reinterpret_cast<const uint16_t*>(stg + r * 128 + (((x >> 3) ^ (r & 7)) << 4) + (x & 7) * 2);
                }
              }
            }
            __syncwarp();
          }
        }
      }
    }
    if (lane == 0) bulk_wait0();   // the output has left before the CTA does
  }
  tc_fence_before();
  __syncthreads();
  if (!PAIR && a.splits > 1) {
    // the sums of all CTAs of the cluster, in rank order
    cluster_sync_all();
#pragma unroll 1
    for (int lr = warp; lr < share; lr += C::THREADS / 32) {
      const int r = (int)rank * share + lr;
      const long long m = mt0 * 128 + r;
      if (r >= 128 || m >= a.M) break;
      const float4* from = reinterpret_cast<const float4*>(smem + C::OFF_STG + lr * 512 + ((lane ^ (r & 31)) << 4));
      float4 sum = make_float4(bias4[0], bias4[1], bias4[2], bias4[3]);
#pragma unroll 1
      for (int p = 0; p < a.splits; ++p) {
        const float4 v = from[p * share * 32];
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
      }
      const long long at = m * a.ldo + nc;
      if (a.tma_store && nc + 4 <= a.N) {   // 8 or 16 aligned bytes
        if (a.out_dtype == IC_DTYPE_F32) {
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at) = sum;
        } else {
          const bool f16 = a.out_dtype == IC_DTYPE_F16;
          const __half2 h0 = __floats2half2_rn(sum.x, sum.y), h1 = __floats2half2_rn(sum.z, sum.w);
          const __nv_bfloat162 g0 = __floats2bfloat162_rn(sum.x, sum.y), g1 = __floats2bfloat162_rn(sum.z, sum.w);
          *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + at) =
              make_uint2(f16 ? *reinterpret_cast<const uint32_t*>(&h0) : *reinterpret_cast<const uint32_t*>(&g0),
                         f16 ? *reinterpret_cast<const uint32_t*>(&h1) : *reinterpret_cast<const uint32_t*>(&g1));
        }
      } else {
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (nc + j < a.N) store_out(a.out, a.out_dtype, at + j, v[j]);
      }
    }
  }
  // neither CTA of a pair leaves while the other may reach its shared memory
  if constexpr (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc2(tmem, NB * BN);
    else tmem_dealloc(tmem, NB * BN);
  }
}

// ============================================================== host side

static bool f8_tmap(CUtensorMap* m, CUtensorMapDataType dt, const void* p, uint64_t inner, uint64_t outer, uint64_t ld_bytes,
                    uint32_t box_inner, uint32_t box_outer) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {inner, outer}, strides[1] = {ld_bytes};
  const cuuint32_t box[2] = {box_inner, box_outer}, es[2] = {1, 1};
  return fn(m, dt, 2, const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct F8Operands {
  const void *x, *w;
  long long M, K, N, ldx, ldw;
};

template <typename C>
static cudaError_t f8_launch(const F8Operands& o, F8Args a, int splits, cudaStream_t st) {
  constexpr int TILE_M = C::PAIR ? 256 : 128;
  a.m_tiles = (a.M + TILE_M - 1) / TILE_M;
  a.n_tiles = (a.N + C::BN - 1) / C::BN;
  a.splits = splits;
  // (rows that are not staged keep what shared memory held; they end in rows of D that nobody reads)
  a.a_rows = a.M < 128 ? (a.M + 7) / 8 * 8 : 128;
  CUtensorMap tx, tw, to;
  memset(&to, 0, sizeof(to));
  if (!f8_tmap(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, o.x, o.K, o.M, o.ldx, 128, a.a_rows) ||
      !f8_tmap(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, o.w, o.K, o.N, o.ldw, 128, C::B_ROWS))
    return cudaErrorInvalidValue;
  const int es = a.out_dtype == IC_DTYPE_F32 ? 4 : 2;
  a.tma_store = a.ldo * es % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  if (a.tma_store &&
      !f8_tmap(&to, a.out_dtype == IC_DTYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, a.out,
               a.N, a.M, a.ldo * es, 128 / es, 32))
    return cudaErrorInvalidValue;
  auto kern = gemm_fp8_kernel<C>;
  cudaError_t e = set_smem_once(kern, C::SMEM);
  if constexpr (C::CPT == 128) {
    static std::atomic<unsigned long long> devices{0};
    if (e == cudaSuccess) e = split_fits_once(kern, C::REGS, devices);
  }
  if (e != cudaSuccess) return e;
  const long long tiles = (long long)a.m_tiles * a.n_tiles;
  const int cluster = C::PAIR ? 2 : splits;
  long long grid = tiles * cluster;
  if (splits == 1) {
    const long long most = num_sms() / cluster * cluster;
    if (grid > most) grid = most;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, tx, tw, to, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Clusters of `splits` CTAs that the device holds at once (45 of 3, 33 of 4, 15 of 7
// or 8 on 148 SMs: they do not fill its processor groups).  Asked once a device.
static long long f8_clusters(int splits) {
  static std::atomic<int> known[64][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  std::atomic<int>& at = known[dev & 63][splits];
  if (at.load()) return at.load();
  using C = F8Cfg<128, false>;
  auto kern = gemm_fp8_kernel<C>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim.x = splits;
  a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(840 * 8);   // a multiple of every size
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.attrs = a;
  cfg.numAttrs = 1;
  int n = 0;
  if (set_smem_once(kern, C::SMEM) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    n = 0;
  }
  if (n > 0) at.store(n);
  return n;
}

// The cheapest way to deal the tiles out, in ns as measured (every SM at work, 1500
// to 1900 MHz): a block of 128 along K takes 560 in a pair's 256 x 256, 375 in its
// 256 x 128, 400 in one CTA's 128 x 128; a tile's output 1000 to 1500; a cluster's
// exchange 2500.  Tiles beyond whole rounds wait for a round of their own.
// (4608 x 12288 -> 4096: 240, 298 and 316 us; 256 x 8192 -> 4096: 32.7, 29.9 and 28.6, in
// clusters of two 20.9.  The first is a tenth too cheap here: of 768 x 2048 -> 8192, in
// 23.3, 21.7 and 22.0, it is taken, by 20.9 against 21.0.)
cudaError_t launch_gemm_fp8(const F8Operands& o, const F8Args& a, cudaStream_t st) {
  const long long sms = num_sms();
  const auto rounds = [](long long tiles, long long places) { return (double)((tiles + places - 1) / places); };
  const long long m128 = (o.M + 127) / 128, m256 = (o.M + 255) / 256, n128 = (o.N + 127) / 128, n256 = (o.N + 255) / 256;
  const double wide = rounds(m256 * n256, sms / 2) * (560. * a.kb + 1500), pair = rounds(m256 * n128, sms / 2) * (375. * a.kb + 1000);
  const double one = rounds(m128 * n128, sms) * (400. * a.kb + 1000);
  int splits = 1;
  for (int n = 2; n <= 8 && m128 * n128 * n <= sms && a.kb >= 2 * n; ++n)
    if (m128 * n128 <= f8_clusters(n)) splits = n;
  const double shared = splits > 1 ? 400. * ((a.kb + splits - 1) / splits) + 3500 : wide;
  if (wide <= pair && wide <= one && wide <= shared) return f8_launch<F8Cfg<256, true>>(o, a, 1, st);
  if (pair <= one && pair <= shared) return f8_launch<F8Cfg<128, true>>(o, a, 1, st);
  return f8_launch<F8Cfg<128, false>>(o, a, shared < one ? splits : 1, st);
}

}  // namespace ic
