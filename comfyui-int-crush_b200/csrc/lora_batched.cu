// Low-rank adapters of many requests at once, beside a shared projection:
//
//   out[m] = T(base[m] + scale_a * (x[m] @ down_a^T) @ up_a^T),  a = ids[m / rows_per_id]
//
// Two kernels: "down" streams x and the adapters' down matrices into fp32
// partial sums mid[split][m][r]; "up" adds the splits in a fixed order and
// streams base -> out.  Rows find their adapter themselves: a warp holds 16
// or 32 rows, and goes over the distinct adapters among them (one pass each,
// found by ballot).  In a pass the rows of other adapters are not loaded and
// their sums are dropped, so each row is read once and gets exactly its own
// adapter's sum, whatever the order of the requests and whatever another
// request's adapter holds; no sort, no host knowledge of the ids.
//
// The products run on register-fed m16n8k16 MMAs without shared memory: the
// order of the summed index inside a block is permuted alike for both
// operands so that a lane's 16- or 8-byte load is its fragment.  At rank 16
// to 64 an adapter does 2R operations per 2-byte value of x and out, far
// below what makes the tensor pipe the limit: HBM bounds the large calls, the
// two launches the small ones.
//
// Roundings: x, down and up are exact in the products, all sums are fp32.
// The MMA takes 16-bit operands, so mid enters the second product as the sum
// of two 16-bit values (hi + lo, 16 bits of precision or more); a row of fp16
// is scaled by a power of two first, so that it neither overflows nor loses
// lo to subnormals.  One rounding at the end.
#include "ic_common.cuh"

#include <type_traits>

namespace ic {

struct LoraArgs {
  const void* x; int64_t ldx;          // [M, K]
  int64_t M, K, N;
  int R, Rp;                           // rank, and its multiple of 8 (mid's row)
  int r0, Rc;                          // the down kernel's share of the ranks
  const void* down;                    // [n, R, K]
  const void* up;                      // [n, N, R]
  const int32_t* ids;                  // [ceil(M / rows_per_id)], < 0: none
  int64_t rows_per_id;
  const float* scales;                 // [n] or NULL (ones)
  int n;
  const void* base; int64_t ldb;       // [M, N] or NULL (zeros)
  void* out; int64_t ldo;
  float* mid; int splits;              // [splits, M, Rp]
  int streamed;                        // lora_stream.cu takes part
};

constexpr int kLoraWarps = 8;
// Rows from which lora_stream.cu takes over (2777 rows of runs of four adapters,
// 5120 to 5120 columns, rank 24: 45 us with it, 69 us without).
constexpr int kLoraStreamRows = 1024;

template <typename T>
__device__ __forceinline__ void lora_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight values of a row at k, zeros past K.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 lora_ld8(const T* row, int64_t k, int64_t K) {
  if constexpr (VEC) {
    return k < K ? __ldg(reinterpret_cast<const uint4*>(row + k)) : make_uint4(0u, 0u, 0u, 0u);
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < K ? row[k + i] : DT<T>::from_f(0.f);
    uint4 v;
    memcpy(&v, e, 16);
    return v;
  }
}

// Lane i's adapter: row m0 + i of a tile of `rows` rows; -1 past M or for
// none, -2 for an id that names no adapter.
__device__ __forceinline__ int lora_id(const LoraArgs& a, int64_t m0, int rows, int lane) {
  const int64_t m = m0 + lane;
  if (lane >= rows || m >= a.M) return -1;
  // M < 2^31
  const int id = __ldg(a.ids + (a.rows_per_id == 1 ? (uint32_t)m : (uint32_t)m / (uint32_t)a.rows_per_id));
  return id < 0 ? -1 : id < a.n ? id : -2;
}

// The first two adapters among 16 rows (bits of `rows` in a ballot; -1: none),
// and whether there are more.
__device__ __forceinline__ bool lora_two(int id, unsigned rows, int& a0, int& a1) {
  const unsigned act = __ballot_sync(0xffffffffu, id >= 0) & rows;
  a0 = __shfl_sync(0xffffffffu, id, act ? __ffs(act) - 1 : 0);
  const unsigned rest = act & ~__ballot_sync(0xffffffffu, id == a0);
  a1 = __shfl_sync(0xffffffffu, id, rest ? __ffs(rest) - 1 : 0);
  const unsigned more = rest & ~__ballot_sync(0xffffffffu, id == a1);
  if (!act) a0 = -1;
  if (!rest) a1 = -1;
  return more != 0;
}

// Whether a tile of 128 rows has more than two adapters in one of its groups of
// 16 rows, which lora_down_stream_kernel leaves to lora_down_kernel.  The two add
// up K in different orders, so a row's last bits depend on its neighbours' ids.
__device__ __forceinline__ bool lora_tile_left(const LoraArgs& a, int64_t tile0, int lane) {
  bool left = false;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int id = lora_id(a, tile0 + 32 * q, 32, lane);
    int a0, a1;
    left = lora_two(id, 0xffffu, a0, a1) || left;
    left = lora_two(id, 0xffff0000u, a0, a1) || left;
  }
  return left;
}

// mid partials.  The CTA's warps share a tile of 16 * MT rows and cut its part
// of K between them.  blockIdx: row tiles and K parts (in turns, beside the
// stream kernel), passes (pass p is taken by the CTA with z = p % gridDim.z).
template <typename T, int NT, int MT, bool VEC>
__global__ void __launch_bounds__(32 * kLoraWarps) lora_down_kernel(const LoraArgs a) {
  constexpr int ROWS = 16 * MT;
  __shared__ float red[kLoraWarps / 2][ROWS][NT * 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* down = reinterpret_cast<const T*>(a.down);
  const int64_t steps = (a.K + 31) / 32;
  const int64_t per = (steps + a.splits - 1) / a.splits;

  for (int64_t m0 = (int64_t)blockIdx.x * ROWS; m0 < a.M; m0 += (int64_t)gridDim.x * ROWS) {
    if (a.streamed && !lora_tile_left(a, m0 / 128 * 128, lane)) continue;   // lora_down_stream_kernel's
    const int id = lora_id(a, m0, ROWS, lane);
    for (int part = blockIdx.y; part < a.splits; part += gridDim.y) {
      const int64_t s0 = part * per, s1 = min(s0 + per, steps);
      unsigned todo = __ballot_sync(0xffffffffu, id >= 0);
      for (unsigned pass = 0; todo; ++pass) {
        const int ad = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
        const unsigned match = __ballot_sync(0xffffffffu, id == ad);
        todo &= ~match;
        if (pass % gridDim.z != blockIdx.z) continue;
        const T* dn = down + ((int64_t)ad * a.R + a.r0) * a.K;
        bool on[MT][2];
        const T* xr[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = 16 * i + 8 * h + g;
            on[i][h] = (match >> r) & 1u;
            xr[i][h] = x + (m0 + (on[i][h] ? r : 0)) * a.ldx;
          }
        float acc[MT][NT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
#pragma unroll (NT <= 4 ? 4 : 2)
        for (int64_t s = s0 + warp; s < s1; s += kLoraWarps) {
          const int64_t k = s * 32 + 8 * t;
          uint4 xv[MT][2];
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              xv[i][h] = on[i][h] ? lora_ld8<T, VEC>(xr[i][h], k, a.K) : make_uint4(0u, 0u, 0u, 0u);
          uint4 dv[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j)
            dv[j] = j * 8 + g < a.Rc ? lora_ld8<T, VEC>(dn + (int64_t)(j * 8 + g) * a.K, k, a.K)
                                     : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              lora_mma<T>(acc[i][j], xv[i][0].x, xv[i][1].x, xv[i][0].y, xv[i][1].y, dv[j].x, dv[j].y);
              lora_mma<T>(acc[i][j], xv[i][0].z, xv[i][1].z, xv[i][0].w, xv[i][1].w, dv[j].z, dv[j].w);
            }
        }
        // the warps (all in this pass together) add up pairwise, in a fixed order
#pragma unroll
        for (int o = kLoraWarps / 2; o > 0; o >>= 1) {
          float* slot = &red[warp & (o - 1)][0][0];
          if (warp >= o && warp < 2 * o) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  *reinterpret_cast<float2*>(slot + (16 * i + 8 * h + g) * (NT * 8) + j * 8 + 2 * t) =
                      make_float2(acc[i][j][2 * h], acc[i][j][2 * h + 1]);
          }
          __syncthreads();
          if (warp < o) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const float2 v = *reinterpret_cast<const float2*>(slot + (16 * i + 8 * h + g) * (NT * 8) + j * 8 + 2 * t);
                  acc[i][j][2 * h] += v.x;
                  acc[i][j][2 * h + 1] += v.y;
                }
          }
          __syncthreads();
        }
        if (warp != 0) continue;
        float* mid = a.mid + (int64_t)part * a.M * a.Rp + a.r0;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = 16 * i + 8 * h + g;
            if (!((match >> r) & 1u)) continue;
#pragma unroll
            for (int j = 0; j < NT; ++j)
              if (a.r0 + j * 8 < a.Rp)
                *reinterpret_cast<float2*>(mid + (m0 + r) * a.Rp + j * 8 + 2 * t) =
                    make_float2(acc[i][j][2 * h], acc[i][j][2 * h + 1]);
          }
      }
    }
  }
}

// Ranks of a lane's MMA operand values: step k of 16 ranks, e = 0..3.  FORM 2
// takes 16-byte loads of 8 ranks for two steps, FORM 1 8-byte loads, FORM 0
// single values.
template <int FORM>
__device__ __forceinline__ int lora_rank(int k, int t) {
  return FORM == 2 ? 32 * (k >> 1) + 8 * t + 4 * (k & 1) : 16 * k + 4 * t;
}

// An up row's operand values of steps k0 .. k0 + 1 (FORM 2) or k0, zeros past R.
template <typename T, int FORM>
__device__ __forceinline__ uint4 lora_ld_up(const T* row, int k0, int t, int R) {
  const int r = lora_rank<FORM>(k0, t);
  if constexpr (FORM == 2) {
    return r < R ? __ldg(reinterpret_cast<const uint4*>(row + r)) : make_uint4(0u, 0u, 0u, 0u);
  } else if constexpr (FORM == 1) {
    const uint2 v = r < R ? __ldg(reinterpret_cast<const uint2*>(row + r)) : make_uint2(0u, 0u);
    return make_uint4(v.x, v.y, 0u, 0u);
  } else {
    T e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = r + i < R ? row[r + i] : DT<T>::from_f(0.f);
    uint2 v;
    memcpy(&v, e, 8);
    return make_uint4(v.x, v.y, 0u, 0u);
  }
}

// Eight values of a base row at n (plain loads: out may be base).
template <typename T, bool VEC>
__device__ __forceinline__ uint4 lora_row8(const T* row, int64_t n, int64_t N) {
  if constexpr (VEC) {
    return n < N ? *reinterpret_cast<const uint4*>(row + n) : make_uint4(0u, 0u, 0u, 0u);
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = n + i < N ? row[n + i] : DT<T>::from_f(0.f);
    uint4 v;
    memcpy(&v, e, 16);
    return v;
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(T lo, T hi) {
  T e[2] = {lo, hi};
  uint32_t v;
  memcpy(&v, e, 4);
  return v;
}

// mid fragments (scale included) of rows m0 + r with bit r of `mine`, as hi + lo
// 16-bit values, and the power of two that was taken out of an fp16 row.  id:
// row m0 + lane's adapter.
template <typename T, int KS, int MT, int FORM>
__device__ __forceinline__ void lora_mid_fragments(const LoraArgs& a, int64_t m0, unsigned mine, int id, int g, int t,
                                                   uint32_t (&hi)[MT][KS][4], uint32_t (&lo)[MT][KS][4],
                                                   float (&grow)[MT][2]) {
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 16 * i + 8 * h + g;
      float v[KS][4];
#pragma unroll
      for (int k = 0; k < KS; ++k) v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.f;
      const int rid = __shfl_sync(0xffffffffu, id, r);
      if ((mine >> r) & 1u) {
#pragma unroll 4
        for (int sp = 0; sp < a.splits; ++sp) {
          const float* row = a.mid + ((int64_t)sp * a.M + m0 + r) * a.Rp;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            const int rk = lora_rank<FORM>(k, t);
            if (rk < a.Rp) {
              const float4 q = *reinterpret_cast<const float4*>(row + rk);
              v[k][0] += q.x; v[k][1] += q.y; v[k][2] += q.z; v[k][3] += q.w;
            }
          }
        }
        const float sc = a.scales ? __ldg(a.scales + rid) : 1.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[k][e] *= sc;
      }
      grow[i][h] = 1.f;
      if constexpr (std::is_same<T, __half>::value) {
        float mx = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(v[k][e]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int ex = (int)(__float_as_uint(mx) >> 23) - 127;
        if (mx == 0.f || ex == 128) ex = 0;
        ex = max(-126, min(126, ex));
        const float shrink = __uint_as_float((uint32_t)(127 - ex) << 23);
        grow[i][h] = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[k][e] *= shrink;
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        T h4[4], l4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h4[e] = DT<T>::from_f(v[k][e]);
          const float rest = v[k][e] - DT<T>::to_f(h4[e]);
          l4[e] = DT<T>::from_f(isfinite(rest) ? rest : 0.f);
        }
        // row half h holds registers h (values 0, 1) and 2 + h (values 2, 3)
        hi[i][k][h] = pack2(h4[0], h4[1]);
        hi[i][k][2 + h] = pack2(h4[2], h4[3]);
        lo[i][k][h] = pack2(l4[0], l4[1]);
        lo[i][k][2 + h] = pack2(l4[2], l4[3]);
      }
    }
}

// out = base + mid @ up^T.  A warp holds the mid fragments of 16 * MT rows
// (KS steps of 16 ranks) and goes over blocks of 32 columns.  Column 2c + e
// of MMA tile j stands for column 8c + 2j + e of the block, so a lane ends up
// with 8 consecutive outputs of a row.  ACROSS: the CTA's warps take eight row
// tiles and the same columns (many rows: an up row is fetched into L1 once for
// all of them), otherwise one row tile and a share of the columns each.
// blockIdx: row tiles, column parts, passes as above (rows without an adapter
// belong to z = 0).
// Above rank 128 (KS = 16) the fragments do not fit the registers: 0.8 to 1.3 KB
// a thread lie in local memory.  8 x 4095 rows, 5120 to 13824 columns, both
// products: rank 12 (not streamed) 686 us, 32 (streamed) 461, 128 1795, 192 4131.
template <typename T, int KS, int MT, bool VECO, int FORM, bool ACROSS>
__global__ void __launch_bounds__(32 * kLoraWarps) lora_up_kernel(const LoraArgs a, int cols_per_cta) {
  constexpr int ROWS = 16 * MT;
  constexpr int STEP = FORM == 2 ? 2 : 1;   // steps per up load
  static_assert(KS % STEP == 0, "two steps to a load");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int64_t m0 = ((int64_t)blockIdx.x * (ACROSS ? kLoraWarps : 1) + (ACROSS ? warp : 0)) * ROWS;
  if (m0 >= a.M) return;
  const T* up = reinterpret_cast<const T*>(a.up);
  const T* base = reinterpret_cast<const T*>(a.base);
  T* out = reinterpret_cast<T*>(a.out);
  const int id = lora_id(a, m0, ROWS, lane);
  const unsigned active = __ballot_sync(0xffffffffu, id >= 0);
  const unsigned bad = __ballot_sync(0xffffffffu, id == -2);
  if (bad && lane == 0) set_dev_error(IC_DEV_ERR_INDEX);

  // rows with an adapter that this CTA writes, and without
  unsigned mine = 0, bare = 0;
  unsigned passes = 0;
  for (unsigned todo = active; todo; ++passes) {
    const int ad = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
    const unsigned match = __ballot_sync(0xffffffffu, id == ad);
    todo &= ~match;
    if (passes % gridDim.z == blockIdx.z) mine |= match;
  }
  if (blockIdx.z == 0) {
    const int64_t left = a.M - m0;
    bare = left >= ROWS ? (ROWS == 32 ? 0xffffffffu : (1u << ROWS) - 1u) : (1u << left) - 1u;
    bare &= ~active;
    if (base == out && a.ldb == a.ldo) bare &= bad;   // already there
  }
  if (!(mine | bare)) return;

  uint32_t hi[MT][KS][4], lo[MT][KS][4];
  float grow[MT][2];
  lora_mid_fragments<T, KS, MT, FORM>(a, m0, mine, id, g, t, hi, lo, grow);

  const int64_t n_begin = (int64_t)blockIdx.y * cols_per_cta + (ACROSS ? 0 : 32 * warp);
  const int64_t n_end = min((int64_t)(blockIdx.y + 1) * cols_per_cta, a.N);
  constexpr int64_t kNext = ACROSS ? 32 : 32 * kLoraWarps;
  const auto load_base = [&](uint4 (&bv)[MT][2], int64_t nb, unsigned match) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 16 * i + 8 * h + g;
        bv[i][h] = make_uint4(0u, 0u, 0u, 0u);
        if (base && ((match >> r) & 1u)) bv[i][h] = lora_row8<T, VECO>(base + (m0 + r) * a.ldb, nb + 8 * t, a.N);
      }
  };
  const auto load_up = [&](uint4 (&uv)[KS / STEP][4], int64_t nb, int ad) {
    const T* u = up + (int64_t)ad * a.N * a.R;
#pragma unroll
    for (int k = 0; k < KS; k += STEP)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t nrow = nb + 8 * (g >> 1) + 2 * j + (g & 1);
        uv[k / STEP][j] = nrow < a.N ? lora_ld_up<T, FORM>(u + nrow * a.R, k, t, a.R) : make_uint4(0u, 0u, 0u, 0u);
      }
  };
  const auto block = [&](const uint4 (&bv)[MT][2], const uint4 (&uv)[KS / STEP][4], int64_t nb, int ad, unsigned match) {
    float acc[MT][4][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
    if (ad >= 0) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4& u = uv[k / STEP][j];
            const uint32_t b0 = k % STEP ? u.z : u.x, b1 = k % STEP ? u.w : u.y;
            lora_mma<T>(acc[i][j], hi[i][k][0], hi[i][k][1], hi[i][k][2], hi[i][k][3], b0, b1);
            lora_mma<T>(acc[i][j], lo[i][k][0], lo[i][k][1], lo[i][k][2], lo[i][k][3], b0, b1);
          }
    }
    const int64_t nc = nb + 8 * t;   // this lane's 8 columns
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 16 * i + 8 * h + g;
        if (!((match >> r) & 1u)) continue;
        T e[8], o[8];
        memcpy(e, &bv[i][h], 16);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float v = DT<T>::to_f(e[2 * j + q]);
            if (ad >= 0) v = fmaf(acc[i][j][2 * h + q], grow[i][h], v);
            else if (ad == -2) v = __int_as_float(0x7fc00000);
            o[2 * j + q] = DT<T>::from_f(v);
          }
        T* row = out + (m0 + r) * a.ldo;
        if constexpr (VECO) {
          if (nc < a.N) {
            uint4 w;
            memcpy(&w, o, 16);
            *reinterpret_cast<uint4*>(row + nc) = w;
          }
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (nc + q < a.N) row[nc + q] = o[q];
        }
      }
  };

  const int first = __shfl_sync(0xffffffffu, id, mine ? __ffs(mine) - 1 : 0);
  if (!bare && __ballot_sync(0xffffffffu, id == first) == mine) {
    // one adapter for all rows: the next block's loads run under this one
    uint4 bv[MT][2], uv[KS / STEP][4];
    load_base(bv, n_begin, mine);
    load_up(uv, n_begin, first);
    for (int64_t nb = n_begin; nb < n_end; nb += kNext) {
      uint4 bn[MT][2], un[KS / STEP][4];
      if constexpr (KS <= 4) {   // more ranks leave no registers for it
        load_base(bn, nb + kNext < n_end ? nb + kNext : a.N, mine);
        load_up(un, nb + kNext < n_end ? nb + kNext : a.N, first);
      }
      block(bv, uv, nb, first, mine);
      if constexpr (KS <= 4) {
#pragma unroll
        for (int i = 0; i < MT; ++i) { bv[i][0] = bn[i][0]; bv[i][1] = bn[i][1]; }
#pragma unroll
        for (int k = 0; k < KS / STEP; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) uv[k][j] = un[k][j];
      } else if (nb + kNext < n_end) {
        load_base(bv, nb + kNext, mine);
        load_up(uv, nb + kNext, first);
      }
    }
    return;
  }
  for (int64_t nb = n_begin; nb < n_end; nb += kNext)
    for (unsigned todo = mine | bare; todo;) {
      const int ad = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
      const unsigned match = __ballot_sync(0xffffffffu, id == ad) & (mine | bare);
      todo &= ~match;
      uint4 bv[MT][2], uv[KS / STEP][4];
      load_base(bv, nb, match);
      if (ad >= 0) load_up(uv, nb, ad);
      block(bv, uv, nb, ad, match);
    }
}

}  // namespace ic

#include "lora_stream.cu"

namespace ic {

// ---------------------------------------------------------------- launches
struct LoraPlan {
  int stream;
  int mt_down, splits, z_down;
  int mt_up, across, cols, z_up;
};

// Rules on sizes.  Down: a CTA takes one tile of 16 rows (32 where that still
// gives every SM two CTAs) and its eight warps cut K; K is cut further over
// CTAs while there are fewer than two per SM, two 32-wide steps per warp at
// least.  Up: tiles of 32 rows (16 for up to 16, or above rank 64); eight row
// tiles per CTA once that fills the SMs twice, else one tile and 256 columns;
// as many columns as leave four CTAs per SM.  Passes go over CTAs only while
// that keeps the grid small (a CTA without a pass ends at once).
static LoraPlan lora_plan(int64_t M, int64_t K, int64_t N, int R, int n, bool stream) {
  LoraPlan p;
  const int sms = num_sms();
  const int64_t steps = (K + 31) / 32;
  p.stream = stream;
  p.mt_down = R <= 64 && (M + 31) / 32 >= 2 * sms ? 2 : 1;
  const int64_t tiles = (M + 16 * p.mt_down - 1) / (16 * p.mt_down);
  int64_t s = (2 * sms + tiles - 1) / tiles;
  const int64_t most = steps / (2 * kLoraWarps);
  s = s < most ? s : most;
  if (stream) {   // tiles of 128 rows, eight 64-wide steps at least in a part
    const int64_t t128 = (M + 127) / 128, k64 = (K + 511) / 512;
    s = (3 * sms + t128 - 1) / t128;
    s = s < k64 ? s : k64;
  }
  p.splits = (int)(s < 1 ? 1 : s > 16 ? 16 : s);
  const int zn = n < 16 ? n : 16;
  p.z_down = tiles * p.splits * zn <= 8 * sms ? zn : 1;
  p.mt_up = M <= 16 || R > 64 ? 1 : 2;
  const int64_t rows = 16 * p.mt_up, groups = (M + rows * kLoraWarps - 1) / (rows * kLoraWarps);
  p.across = groups * ((N + 255) / 256) >= 2 * sms;
  const int64_t units = p.across ? groups : (M + rows - 1) / rows;
  int cols = 32 * kLoraWarps;
  while (cols < 4096 && units * ((N + 2 * cols - 1) / (2 * cols)) >= 4 * sms) cols *= 2;
  p.cols = cols;
  p.z_up = !p.across && units * ((N + cols - 1) / cols) * zn <= 8 * sms ? zn : 1;
  return p;
}

// Sizes that lora_stream.cu takes, if the rows are aligned for TMA.
static bool lora_stream_sizes(int64_t M, int64_t K, int64_t N, int R, int n) {
  return M >= kLoraStreamRows && R <= 64 && R % 8 == 0 && K % 8 == 0 && N % 8 == 0 && K >= 64 && N >= 64 &&
         (int64_t)n * N < (1LL << 31) && (int64_t)n * R < (1LL << 31);
}

int64_t lora_workspace(int64_t M, int64_t K, int64_t N, int R, int n) {
  int splits = lora_plan(M, K, N, R, n, false).splits;
  if (lora_stream_sizes(M, K, N, R, n)) {   // either, by the alignment of the rows
    const int s = lora_plan(M, K, N, R, n, true).splits;
    splits = s > splits ? s : splits;
  }
  return (int64_t)splits * M * ((R + 7) / 8 * 8);
}

template <typename T, int NT, bool VEC>
static cudaError_t lora_down_t(const LoraArgs& a, const LoraPlan& p, cudaStream_t st) {
  const int64_t rows = 16 * p.mt_down;
  // beside the stream kernel most tiles are not this one's: few CTAs look them over
  int64_t tiles = (a.M + rows - 1) / rows;
  int64_t parts = p.splits;
  if (a.streamed) {
    const int64_t most = 2 * num_sms();
    tiles = tiles < most ? tiles : most;
    parts = parts < most / tiles ? parts : most / tiles;
  }
  const dim3 grid((unsigned)tiles, (unsigned)parts, (unsigned)p.z_down);
  if constexpr (NT <= 8) {
    if (p.mt_down == 2) {
      lora_down_kernel<T, NT, 2, VEC><<<grid, 32 * kLoraWarps, 0, st>>>(a);
      return cudaGetLastError();
    }
  }
  lora_down_kernel<T, NT, 1, VEC><<<grid, 32 * kLoraWarps, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T, int KS, int MT>
static cudaError_t lora_up_m(const LoraArgs& a, const LoraPlan& p, bool vec, bool wide, cudaStream_t st) {
  const int64_t rows = 16 * MT * (p.across ? kLoraWarps : 1);
  const dim3 grid((unsigned)((a.M + rows - 1) / rows), (unsigned)((a.N + p.cols - 1) / p.cols), (unsigned)p.z_up);
  const int th = 32 * kLoraWarps;
  constexpr int WIDE = KS % 2 == 0 ? 2 : 1;
  if (!vec) lora_up_kernel<T, KS, MT, false, 0, false><<<grid, th, 0, st>>>(a, p.cols);
  else if (p.across && wide) lora_up_kernel<T, KS, MT, true, WIDE, true><<<grid, th, 0, st>>>(a, p.cols);
  else if (p.across) lora_up_kernel<T, KS, MT, true, 1, true><<<grid, th, 0, st>>>(a, p.cols);
  else if (wide) lora_up_kernel<T, KS, MT, true, WIDE, false><<<grid, th, 0, st>>>(a, p.cols);
  else lora_up_kernel<T, KS, MT, true, 1, false><<<grid, th, 0, st>>>(a, p.cols);
  return cudaGetLastError();
}

template <typename T, int KS>
static cudaError_t lora_up_t(const LoraArgs& a, LoraPlan p, bool vec, bool wide, cudaStream_t st) {
  if (!vec && p.across) {   // odd rows: one tile per CTA
    p.across = 0;
    p.z_up = 1;
  }
  if constexpr (KS <= 4) {
    if (p.mt_up == 2) return lora_up_m<T, KS, 2>(a, p, vec, wide, st);
  }
  return lora_up_m<T, KS, 1>(a, p, vec, wide, st);
}

template <typename T>
static cudaError_t lora_t(LoraArgs a, cudaStream_t st) {
  const auto al = [](const void* q, int by) { return (reinterpret_cast<uintptr_t>(q) & (by - 1)) == 0; };
  const bool vec = al(a.x, 16) && al(a.down, 16) && a.ldx % 8 == 0 && a.K % 8 == 0;
  const bool veco = (!a.base || (al(a.base, 16) && a.ldb % 8 == 0)) && al(a.out, 16) && a.ldo % 8 == 0 && a.N % 8 == 0;
  const bool vecu = veco && al(a.up, 8) && a.R % 4 == 0, wide = al(a.up, 16) && a.R % 8 == 0;
  const bool stream = vec && vecu && wide && lora_stream_sizes(a.M, a.K, a.N, a.R, a.n);
  const LoraPlan p = lora_plan(a.M, a.K, a.N, a.R, a.n, stream);
  a.splits = p.splits;
  a.streamed = stream;
  cudaError_t e = cudaSuccess;
  if (stream) {
    e = a.R <= 8 ? lora_down_stream_t<T, 1>(a, st) : a.R <= 16 ? lora_down_stream_t<T, 2>(a, st)
        : a.R <= 32 ? lora_down_stream_t<T, 4>(a, st) : lora_down_stream_t<T, 8>(a, st);
    if (e != cudaSuccess) return e;
  }
#define IC_DOWN(NT) e = vec ? lora_down_t<T, NT, true>(c, p, st) : lora_down_t<T, NT, false>(c, p, st)
  // (16 or more rows of a request together: 16 rows have at most two adapters,
  // and the stream leaves nothing)
  const int todo = stream && a.rows_per_id >= 16 ? 0 : a.R;
  for (int r0 = 0; r0 < todo; r0 += 128) {   // accumulators hold 128 ranks
    LoraArgs c = a;
    c.r0 = r0;
    c.Rc = a.R - r0 < 128 ? a.R - r0 : 128;
    if (c.Rc <= 8) IC_DOWN(1);
    else if (c.Rc <= 16) IC_DOWN(2);
    else if (c.Rc <= 32) IC_DOWN(4);
    else if (c.Rc <= 64) IC_DOWN(8);
    else IC_DOWN(16);
    if (e != cudaSuccess) return e;
  }
#undef IC_DOWN
  if (stream)
    return a.R <= 16 ? lora_up_stream_t<T, 1>(a, st) : a.R <= 32 ? lora_up_stream_t<T, 2>(a, st) : lora_up_stream_t<T, 4>(a, st);
  if (a.R <= 16) return lora_up_t<T, 1>(a, p, vecu, wide, st);
  if (a.R <= 32) return lora_up_t<T, 2>(a, p, vecu, wide, st);
  if (a.R <= 64) return lora_up_t<T, 4>(a, p, vecu, wide, st);
  if (a.R <= 128) return lora_up_t<T, 8>(a, p, vecu, wide, st);
  return lora_up_t<T, 16>(a, p, vecu, wide, st);
}

cudaError_t launch_lora_batched(const LoraArgs& a, int dtype, cudaStream_t st) {
  if (a.M == 0 || a.N == 0) return cudaSuccess;
  return dtype == IC_DTYPE_BF16 ? lora_t<__nv_bfloat16>(a, st) : lora_t<__half>(a, st);
}

}  // namespace ic
