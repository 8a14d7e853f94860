// The many-request adapters for many rows: both products as streams through
// shared memory.  One warp feeds rings with TMA, eight warps of 16 rows each
// compute.  HBM bounds both: loads and stores in flight take no registers here,
// which is what limits lora_down_kernel and lora_up_kernel at this size (8 x
// 4095 rows, 5120 to 13824 columns, rank 32, one sample without an adapter:
// 263 us for the first product register-fed, 77 us here; second 520 us and 360
// us here, 5.0 TB/s).
#include "ic_common.cuh"
#include "lora_feed.h"

namespace ic {

__device__ __forceinline__ void bulk_wait_read1() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// The ids of a tile's 128 rows and the adapters among them, in shared memory
// (warp 0 builds the list; a __syncthreads before and after).  Returns their
// number; `bad`: some id names no adapter.
__device__ __forceinline__ int lora_tile_list(const int* ids, int* list, int lane, bool& bad) {
  int n = 0;
  bad = false;
  for (int q = 0; q < 4; ++q) {
    const int id = ids[32 * q + lane];
    bad = __any_sync(0xffffffffu, id == -2) || bad;
    for (unsigned todo = __ballot_sync(0xffffffffu, id >= 0); todo;) {
      const int ad = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
      todo &= ~__ballot_sync(0xffffffffu, id == ad);
      bool old = false;
      for (int i = lane; i < n; i += 32) old = old || list[i] == ad;
      if (!__any_sync(0xffffffffu, old)) {
        if (lane == 0) list[n] = ad;
        ++n;
      }
      __syncwarp();
    }
  }
  return n;
}

// ------------------------------------------------------------------- down
// mid[split][m] = x[m] @ down_a^T over a part of K, for tiles of 128 rows with
// at most two adapters in each 16 rows (others: lora_down_kernel).  Blocks of
// 64 k, 128B-swizzled, read as MMA fragments by ldmatrix without bank
// conflicts, in two rings: 128 rows of x, and R rows of down for each of the
// tile's adapters in turn.  A warp takes part in its rows' adapters only, with
// a set of sums for each, so no row's sum sees another adapter.
template <int NT>
struct LdCfg {
  static constexpr int SX = 4, SD = 6;
  static constexpr int X = 128 * 128;
  static constexpr int DOWN = NT * 8 * 128;            // 1024 or more
  static constexpr int OFF_DOWN = SX * X;
  static constexpr int OFF_IDS = OFF_DOWN + SD * DOWN;
  static constexpr int OFF_BAR = OFF_IDS + 1024;       // ids of the rows, adapters among them
  static constexpr int SMEM = OFF_BAR + 256;
  static constexpr int THREADS = 32 * (kLoraWarps + 1);
};

template <typename T, int NT>
__global__ void __launch_bounds__(LdCfg<NT>::THREADS)
lora_down_stream_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_down,
                        const LoraArgs a) {
  using C = LdCfg<NT>;
  constexpr int SX = C::SX, SD = C::SD;
  extern __shared__ __align__(1024) uint8_t smem[];   // no static shared memory: the declared alignment holds
  int* ids = reinterpret_cast<int*>(smem + C::OFF_IDS);
  int* list = ids + 128;
  uint64_t* x_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);   // [SX] TMA -> warps
  uint64_t* x_empty = x_full + SX;                                     // [SX] warps -> TMA
  uint64_t* d_full = x_empty + SX;                                     // [SD]
  uint64_t* d_empty = d_full + SD;                                     // [SD]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(d_empty + SD);
  volatile int* count = abort_flag + 1;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int64_t m0 = (int64_t)blockIdx.x * 128;

  if (threadIdx.x == 0) {
    for (int i = 0; i < SX; ++i) {
      mbar_init(x_full + i, 1);
      mbar_init(x_empty + i, kLoraWarps);
    }
    for (int i = 0; i < SD; ++i) {
      mbar_init(d_full + i, 1);
      mbar_init(d_empty + i, kLoraWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < 128) ids[threadIdx.x] = lora_id(a, m0 + threadIdx.x, 1, 0);
  __syncthreads();
  bool more = false;
  int a0 = -1, a1 = -1;   // this warp's adapters
  if (warp < kLoraWarps) more = lora_two(lane < 16 ? ids[16 * warp + lane] : -1, 0xffffu, a0, a1);
  if (__syncthreads_or(more)) return;
  if (warp == 0) {
    bool bad;
    const int n = lora_tile_list(ids, list, lane, bad);
    if (lane == 0) *count = n;
  }
  __syncthreads();
  const int passes = *count;
  if (passes == 0) return;
  const int all = (int)((a.K + 63) / 64), per = (all + a.splits - 1) / a.splits;
  const int k0 = min((int)blockIdx.y * per, all), steps = min(k0 + per, all) - k0;

  if (warp == kLoraWarps) {
    if (lane == 0) {
      volatile int never = 0;
      lora_feed<SX, SD>(
          steps, passes, [&](int i) { return mbar_wait(x_empty + i % SX, ((i / SX) & 1) ^ 1, abort_flag); },
          [&](int i) {
            mbar_arrive_expect_tx(x_full + i % SX, C::X);
            tma_load_2d(smem + i % SX * C::X, &tm_x, x_full + i % SX, 64 * (k0 + i), (int)m0);
          },
          [&](int i) { mbar_wait(x_full + i % SX, (i / SX) & 1, &never); },
          [&](int u) { return mbar_wait(d_empty + u % SD, ((u / SD) & 1) ^ 1, abort_flag); },
          [&](int u, int i, int p) {
            mbar_arrive_expect_tx(d_full + u % SD, C::DOWN);
            tma_load_2d(smem + C::OFF_DOWN + u % SD * C::DOWN, &tm_down, d_full + u % SD, 64 * (k0 + i), list[p] * a.R);
          },
          [&](int u) { mbar_wait(d_full + u % SD, (u / SD) & 1, &never); });
    }
    return;
  }
  float acc[2][NT][4];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[q][j][0] = acc[q][j][1] = acc[q][j][2] = acc[q][j][3] = 0.f;
  // ldmatrix: lane i names row i % 8 of matrix i / 8.  x: rows 0-7 | 8-15 at k,
  // then at k + 8; down: ranks 0-7 at k, k + 8, then ranks 8-15
  const int row = warp * 16 + (lane & 15), xc = lane >> 4;
  const int rank = (lane & 7) + 8 * (lane >> 4), dc = (lane >> 3) & 1;
  const uint32_t base = smem_u32(smem);
  const auto product = [&](float (&c)[NT][4], uint32_t xs, uint32_t ds) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {   // 16 k: chunks 2k, 2k + 1
      uint32_t xf[4];
      ldmatrix4(xf, xs + row * 128 + (((2 * k + xc) ^ (row & 7)) << 4));
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        // (8 ranks: the second pair of matrices is the first again)
        const int r = NT == 1 ? lane & 7 : 8 * j + rank;
        uint32_t df[4];
        ldmatrix4(df, ds + r * 128 + (((2 * k + dc) ^ (r & 7)) << 4));
        lora_mma<T>(c[j], xf[0], xf[1], xf[2], xf[3], df[0], df[1]);
        if constexpr (NT > 1) lora_mma<T>(c[j + 1], xf[0], xf[1], xf[2], xf[3], df[2], df[3]);
      }
    }
  };
  bool ok = true;
  int u = 0;
  for (int i = 0; i < steps; ++i) {
    const int st = i % SX;
    ok = __all_sync(0xffffffffu, mbar_wait(x_full + st, (i / SX) & 1, abort_flag));
    if (!ok) return;
    for (int p = 0; p < passes; ++p, ++u) {
      const int su = u % SD, ad = list[p];
      ok = __all_sync(0xffffffffu, mbar_wait(d_full + su, (u / SD) & 1, abort_flag));
      if (!ok) return;
      const uint32_t xs = base + st * C::X, ds = base + C::OFF_DOWN + su * C::DOWN;
      if (ad == a0) product(acc[0], xs, ds);
      else if (ad == a1) product(acc[1], xs, ds);
      __syncwarp();
      if (lane == 0) mbar_arrive(d_empty + su);
    }
    if (lane == 0) mbar_arrive(x_empty + st);
  }
  const int g = lane >> 2, t = lane & 3;
  float* mid = a.mid + (int64_t)blockIdx.y * a.M * a.Rp;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t m = m0 + 16 * warp + 8 * h + g;
    const int id = ids[16 * warp + 8 * h + g];
    if (id < 0) continue;
    const bool second = id != a0;
    // ranks past R: rows of another adapter, zeros in mid
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = 8 * j + 2 * t;
      const float v0 = second ? acc[1][j][2 * h] : acc[0][j][2 * h];
      const float v1 = second ? acc[1][j][2 * h + 1] : acc[0][j][2 * h + 1];
      if (8 * j < a.Rp)
        *reinterpret_cast<float2*>(mid + m * a.Rp + r) = make_float2(r < a.R ? v0 : 0.f, r + 1 < a.R ? v1 : 0.f);
    }
  }
}

// --------------------------------------------------------------------- up
// out[m] = T(base[m] + mid[m] @ up_a^T), tiles of 128 rows, blocks of 64
// columns.  Two rings: the base block, and an up block (64 rows) for each of
// the adapters among the tile's rows in turn.  A warp adds the product in
// place to its rows of that adapter and sends its 16 rows off by TMA store
// after the last one; the base stage is refilled when its stores have read it.
// Rows without an adapter pass unchanged; fragments of mid stay in registers.
template <int KS>
struct LsCfg {
  static constexpr int SB = KS <= 2 ? 5 : 4, SU = 4;   // two CTAs fit an SM
  static constexpr int BASE = 128 * 128;              // 128 rows x 64 elements, 128B-swizzled
  static constexpr int UP = 64 * KS * 32;             // 64 rows of up to 16 * KS ranks
  static constexpr int OFF_UP = SB * BASE;
  static constexpr int OFF_IDS = OFF_UP + SU * UP;
  static constexpr int OFF_BAR = OFF_IDS + 1024;      // ids of the rows, adapters among them
  static constexpr int SMEM = OFF_BAR + 256;
  static constexpr int THREADS = 32 * (kLoraWarps + 1);
};

template <typename T, int KS>
__global__ void __launch_bounds__(LsCfg<KS>::THREADS)
lora_up_stream_kernel(const __grid_constant__ CUtensorMap tm_base, const __grid_constant__ CUtensorMap tm_up,
                      const __grid_constant__ CUtensorMap tm_out, const LoraArgs a, int cols_per_cta) {
  using C = LsCfg<KS>;
  constexpr int SB = C::SB, SU = C::SU;
  constexpr int FORM = KS % 2 == 0 ? 2 : 1;
  constexpr int STEP = FORM == 2 ? 2 : 1;
  extern __shared__ __align__(1024) uint8_t smem[];   // no static shared memory: the declared alignment holds
  int* ids = reinterpret_cast<int*>(smem + C::OFF_IDS);
  int* list = ids + 128;
  uint64_t* b_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);   // [SB] TMA -> warps
  uint64_t* b_empty = b_full + SB;                                     // [SB] stores have read -> TMA
  uint64_t* u_full = b_empty + SB;                                     // [SU]
  uint64_t* u_empty = u_full + SU;                                     // [SU]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(u_empty + SU);
  volatile int* count = abort_flag + 1;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int64_t m0 = (int64_t)blockIdx.x * 128;
  const bool has_base = a.base != nullptr;

  if (threadIdx.x == 0) {
    for (int i = 0; i < SB; ++i) {
      mbar_init(b_full + i, 1);
      mbar_init(b_empty + i, kLoraWarps);
    }
    for (int i = 0; i < SU; ++i) {
      mbar_init(u_full + i, 1);
      mbar_init(u_empty + i, kLoraWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < 128) {
    const int id = lora_id(a, m0 + threadIdx.x, 1, 0);
    ids[threadIdx.x] = id;
    if (id == -2) set_dev_error(IC_DEV_ERR_INDEX);
  }
  __syncthreads();
  if (warp == 0) {
    bool bad;
    const int n = lora_tile_list(ids, list, lane, bad);
    if (lane == 0) *count = n == 0 && !bad && a.base == a.out && a.ldb == a.ldo ? -1 : n;   // -1: already there
  }
  __syncthreads();
  const int passes = *count;
  if (passes < 0) return;
  const int64_t n0 = (int64_t)blockIdx.y * cols_per_cta;
  const int blocks = (int)((min(n0 + cols_per_cta, a.N) - n0 + 63) / 64);

  if (warp == kLoraWarps) {
    if (lane == 0) {
      volatile int never = 0;
      lora_feed<SB, SU>(
          blocks, passes, [&](int i) { return mbar_wait(b_empty + i % SB, ((i / SB) & 1) ^ 1, abort_flag); },
          [&](int i) {
            if (has_base) {
              mbar_arrive_expect_tx(b_full + i % SB, C::BASE);
              tma_load_2d(smem + i % SB * C::BASE, &tm_base, b_full + i % SB, (int)n0 + 64 * i, (int)m0);
            } else {
              mbar_arrive(b_full + i % SB);
            }
          },
          [&](int i) { mbar_wait(b_full + i % SB, (i / SB) & 1, &never); },
          [&](int u) { return mbar_wait(u_empty + u % SU, ((u / SU) & 1) ^ 1, abort_flag); },
          [&](int u, int i, int p) {
            mbar_arrive_expect_tx(u_full + u % SU, 128 * a.R);
            tma_load_2d(smem + C::OFF_UP + u % SU * C::UP, &tm_up, u_full + u % SU, 0,
                        list[p] * (int)a.N + (int)n0 + 64 * i);
          },
          [&](int u) { mbar_wait(u_full + u % SU, (u / SU) & 1, &never); });
    }
    return;
  }
  const int g = lane >> 2, t = lane & 3;
  const int id0 = ids[16 * warp + g], id1 = ids[16 * warp + 8 + g];
  uint32_t hi[1][KS][4], lo[1][KS][4];
  float grow[1][2];
  {
    const int id = ids[16 * warp + (lane & 15)];
    const unsigned mine = __ballot_sync(0xffffffffu, id >= 0) & 0xffffu;
    lora_mid_fragments<T, KS, 1, FORM>(a, m0 + 16 * warp, mine, id, g, t, hi, lo, grow);
  }
  const bool nan = __any_sync(0xffffffffu, id0 == -2 || id1 == -2);
  bool ok = true;
  int u = 0;
  for (int i = 0; ok && i < blocks; ++i) {
    const int st = i % SB;
    ok = __all_sync(0xffffffffu, mbar_wait(b_full + st, (i / SB) & 1, abort_flag));
    if (!ok) break;
    uint8_t* rows = smem + st * C::BASE + warp * 2048;
    if (!has_base) {
#pragma unroll
      for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(rows + (32 * q + lane) * 16) = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
    }
    for (int p = 0; p < passes; ++p, ++u) {
      const int su = u % SU, ad = list[p];
      ok = __all_sync(0xffffffffu, mbar_wait(u_full + su, (u / SU) & 1, abort_flag));
      if (!ok) break;
      if (__any_sync(0xffffffffu, id0 == ad || id1 == ad)) {
        const uint8_t* up = smem + C::OFF_UP + su * C::UP;
#pragma unroll
        for (int j = 0; j < 8; ++j) {   // 8 columns
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < KS; k += STEP) {
            const int r = lora_rank<FORM>(k, t);
            const uint8_t* v8 = up + (8 * j + g) * (2 * a.R) + 2 * r;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (r < a.R) {
              if constexpr (FORM == 2) {
                v = *reinterpret_cast<const uint4*>(v8);
              } else {
                const uint2 w = *reinterpret_cast<const uint2*>(v8);
                v.x = w.x;
                v.y = w.y;
              }
            }
            lora_mma<T>(acc, hi[0][k][0], hi[0][k][1], hi[0][k][2], hi[0][k][3], v.x, v.y);
            lora_mma<T>(acc, lo[0][k][0], lo[0][k][1], lo[0][k][2], lo[0][k][3], v.x, v.y);
            if constexpr (FORM == 2) {
              lora_mma<T>(acc, hi[0][k + 1][0], hi[0][k + 1][1], hi[0][k + 1][2], hi[0][k + 1][3], v.z, v.w);
              lora_mma<T>(acc, lo[0][k + 1][0], lo[0][k + 1][1], lo[0][k + 1][2], lo[0][k + 1][3], v.z, v.w);
            }
          }
          // columns 8j + 2t, + 1 of rows g and g + 8, where they are this adapter's
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if ((h ? id1 : id0) != ad) continue;
            uint32_t* at = reinterpret_cast<uint32_t*>(rows + (8 * h + g) * 128 + ((j ^ g) << 4) + 4 * t);
            const uint32_t w = *at;
            T e[2];
            memcpy(e, &w, 4);
            *at = pack2(DT<T>::from_f(fmaf(acc[2 * h], grow[0][h], DT<T>::to_f(e[0]))),
                        DT<T>::from_f(fmaf(acc[2 * h + 1], grow[0][h], DT<T>::to_f(e[1]))));
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(u_empty + su);
    }
    if (!ok) break;
    if (nan) {
      const T v = DT<T>::from_f(__int_as_float(0x7fc00000));
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if ((h ? id1 : id0) == -2)
          for (int q = 0; q < 8; ++q) *reinterpret_cast<uint32_t*>(rows + (8 * h + g) * 128 + 16 * q + 4 * t) = pack2(v, v);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (m0 + 16 * warp < a.M) tma_store_2d(&tm_out, rows, (int)n0 + 64 * i, (int)m0 + 16 * warp);
      bulk_commit();
      bulk_wait_read1();   // the block before has been read
      if (i > 0) mbar_arrive(b_empty + (i - 1) % SB);
    }
  }
  if (lane == 0) bulk_wait0();   // the stores are done before the CTA leaves
}

// ---------------------------------------------------------------- host side
static bool ls_map(CUtensorMap* m, bool bf, const void* p, int64_t inner, int64_t outer, int64_t ld, int box_inner,
                   int box_outer, CUtensorMapSwizzle sw) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer};
  cuuint32_t one[2] = {1, 1};
  return fn(m, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(p), dims,
            strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int NT>
static cudaError_t lora_down_stream_t(const LoraArgs& a, cudaStream_t st) {
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  using C = LdCfg<NT>;
  CUtensorMap tx, td;
  if (!ls_map(&tx, BF, a.x, a.K, a.M, a.ldx, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !ls_map(&td, BF, a.down, a.K, (int64_t)a.n * a.R, a.K, 64, NT * 8, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  auto kern = lora_down_stream_kernel<T, NT>;
  const cudaError_t e = set_smem_once(kern, C::SMEM);
  if (e != cudaSuccess) return e;
  kern<<<dim3((unsigned)((a.M + 127) / 128), (unsigned)a.splits), C::THREADS, C::SMEM, st>>>(tx, td, a);
  return cudaGetLastError();
}

template <typename T, int KS>
static cudaError_t lora_up_stream_t(const LoraArgs& a, cudaStream_t st) {
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  using C = LsCfg<KS>;
  CUtensorMap tb{}, tu, to;
  if ((a.base && !ls_map(&tb, BF, a.base, a.N, a.M, a.ldb, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B)) ||
      !ls_map(&tu, BF, a.up, a.R, (int64_t)a.n * a.N, a.R, a.R, 64, CU_TENSOR_MAP_SWIZZLE_NONE) ||
      !ls_map(&to, BF, a.out, a.N, a.M, a.ldo, 64, 16, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  auto kern = lora_up_stream_kernel<T, KS>;
  const cudaError_t e = set_smem_once(kern, C::SMEM);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (a.M + 127) / 128;
  // two CTAs run on an SM: columns for at least four waves of them, so that
  // the last one is short
  int cols = 256;
  while (cols < 4096 && tiles * ((a.N + 2 * cols - 1) / (2 * cols)) >= 8 * num_sms()) cols *= 2;
  const dim3 grid((unsigned)tiles, (unsigned)((a.N + cols - 1) / cols));
  kern<<<grid, C::THREADS, C::SMEM, st>>>(tb, tu, to, a, cols);
  return cudaGetLastError();
}

}  // namespace ic
