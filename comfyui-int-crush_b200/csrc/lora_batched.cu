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
};

constexpr int kLoraWarps = 8;

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

// Barrier of one row group's warps (ids 1..15; 0 is __syncthreads').
__device__ __forceinline__ void group_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
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
  const int id = __ldg(a.ids + m / a.rows_per_id);
  return id < 0 ? -1 : id < a.n ? id : -2;
}

// mid partials.  A warp takes 16 * MT rows; WK warps share them and cut the
// CTA's part of K between them, 8 / WK row groups per CTA.  blockIdx: row
// groups, K parts, passes (pass p is taken by the CTA with z = p % gridDim.z).
template <typename T, int NT, int MT, int WK, bool VEC>
__global__ void __launch_bounds__(32 * kLoraWarps) lora_down_kernel(const LoraArgs a) {
  constexpr int ROWS = 16 * MT;
  constexpr int WR = kLoraWarps / WK;
  __shared__ float red[kLoraWarps / 2][ROWS][NT * 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rg = warp / WK, kw = warp % WK;
  const int64_t m0 = ((int64_t)blockIdx.x * WR + rg) * ROWS;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* down = reinterpret_cast<const T*>(a.down);

  const int id = lora_id(a, m0, ROWS, lane);
  const int64_t steps = (a.K + 31) / 32;
  const int64_t per = (steps + a.splits - 1) / a.splits;
  const int64_t s0 = (int64_t)blockIdx.y * per, s1 = min(s0 + per, steps);

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
#pragma unroll 2
    for (int64_t s = s0 + kw; s < s1; s += WK) {
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
    // the WK warps of a row group (all in this pass together) add up
    // pairwise, in a fixed order
#pragma unroll
    for (int o = WK / 2; o > 0; o >>= 1) {
      float* slot = &red[rg * (WK / 2) + (kw & (o - 1))][0][0];
      if (kw >= o && kw < 2 * o) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              *reinterpret_cast<float2*>(slot + (16 * i + 8 * h + g) * (NT * 8) + j * 8 + 2 * t) =
                  make_float2(acc[i][j][2 * h], acc[i][j][2 * h + 1]);
      }
      group_sync(1 + rg, 32 * WK);
      if (kw < o) {
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
      group_sync(1 + rg, 32 * WK);
    }
    if (kw != 0) continue;
    float* mid = a.mid + (int64_t)blockIdx.y * a.M * a.Rp + a.r0;
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

// Four values of an up row at r, zeros past R.
template <typename T, bool VEC>
__device__ __forceinline__ uint2 lora_ld4(const T* row, int r, int R) {
  if constexpr (VEC) {
    return r < R ? __ldg(reinterpret_cast<const uint2*>(row + r)) : make_uint2(0u, 0u);
  } else {
    T e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = r + i < R ? row[r + i] : DT<T>::from_f(0.f);
    uint2 v;
    memcpy(&v, e, 8);
    return v;
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

// out = base + mid @ up^T.  A warp holds the mid fragments of 16 * MT rows
// (KS steps of 16 ranks) and goes over blocks of 32 columns.  Column 2c + e
// of MMA tile j stands for column 8c + 2j + e of the block, so a lane ends up
// with 8 consecutive outputs of a row.  blockIdx: row tiles, column parts,
// passes as above (rows without an adapter belong to z = 0).
template <typename T, int KS, int MT, bool VECO, bool VECB>
__global__ void __launch_bounds__(32 * kLoraWarps) lora_up_kernel(const LoraArgs a, int cols_per_cta) {
  constexpr int ROWS = 16 * MT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int64_t m0 = (int64_t)blockIdx.x * ROWS;
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

  // mid fragments (scale included), as hi + lo 16-bit values
  uint32_t hi[MT][KS][4], lo[MT][KS][4];
  float grow[MT][2];   // power of two taken out of an fp16 row
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
        for (int sp = 0; sp < a.splits; ++sp) {
          const float* row = a.mid + ((int64_t)sp * a.M + m0 + r) * a.Rp;
#pragma unroll
          for (int k = 0; k < KS; ++k)
            if (16 * k + 4 * t < a.Rp) {
              const float4 q = *reinterpret_cast<const float4*>(row + 16 * k + 4 * t);
              v[k][0] += q.x; v[k][1] += q.y; v[k][2] += q.z; v[k][3] += q.w;
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
        // row half h holds registers h (ranks 4t, 4t+1) and 2 + h (4t+2, 4t+3)
        hi[i][k][h] = pack2(h4[0], h4[1]);
        hi[i][k][2 + h] = pack2(h4[2], h4[3]);
        lo[i][k][h] = pack2(l4[0], l4[1]);
        lo[i][k][2 + h] = pack2(l4[2], l4[3]);
      }
    }

  const int64_t n_begin = (int64_t)blockIdx.y * cols_per_cta;
  const int64_t n_end = min(n_begin + cols_per_cta, a.N);
  for (int64_t nb = n_begin + 32 * warp; nb < n_end; nb += 32 * kLoraWarps) {
    const int64_t nc = nb + 8 * t;   // this lane's 8 columns
    for (unsigned todo = mine | bare; todo;) {
      const int ad = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
      const unsigned match = __ballot_sync(0xffffffffu, id == ad) & (mine | bare);
      todo &= ~match;
      uint4 bv[MT][2];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 16 * i + 8 * h + g;
          bv[i][h] = make_uint4(0u, 0u, 0u, 0u);
          if (base && ((match >> r) & 1u)) bv[i][h] = lora_row8<T, VECO>(base + (m0 + r) * a.ldb, nc, a.N);
        }
      float acc[MT][4][4];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
      if (ad >= 0) {
        const T* u = up + (int64_t)ad * a.N * a.R;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint2 uv[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int64_t nrow = nb + 8 * (g >> 1) + 2 * j + (g & 1);
            uv[j] = nrow < a.N ? lora_ld4<T, VECB>(u + nrow * a.R, 16 * k + 4 * t, a.R) : make_uint2(0u, 0u);
          }
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              lora_mma<T>(acc[i][j], hi[i][k][0], hi[i][k][1], hi[i][k][2], hi[i][k][3], uv[j].x, uv[j].y);
              lora_mma<T>(acc[i][j], lo[i][k][0], lo[i][k][1], lo[i][k][2], lo[i][k][3], uv[j].x, uv[j].y);
            }
        }
      }
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
    }
  }
}

// ---------------------------------------------------------------- launches
struct LoraPlan {
  int mt_down, wk, splits, z_down;
  int mt_up, cols, z_up;
};

// Rules on sizes: few rows put all eight warps of a CTA on one 16-row tile's
// K range and cut K further over CTAs until about two CTAs per SM run; many
// rows take 32-row warp tiles.  Passes go over CTAs only while that keeps the
// grid small (a CTA without a pass ends at once).
static LoraPlan lora_plan(int64_t M, int64_t K, int64_t N, int R, int n) {
  LoraPlan p;
  const int sms = num_sms();
  const int64_t steps = (K + 31) / 32;
  const bool few = M <= 16 * (int64_t)sms;
  p.mt_down = few || R > 64 ? 1 : 2;
  p.wk = few ? 8 : 2;
  const int64_t groups = (M + 16 * p.mt_down * (kLoraWarps / p.wk) - 1) / (16 * p.mt_down * (kLoraWarps / p.wk));
  int64_t s = (2 * sms + groups - 1) / groups;
  s = s < steps / p.wk ? s : steps / p.wk;
  s = s < 1 ? 1 : s > 16 ? 16 : s;
  p.splits = (int)s;
  const int zn = n < 16 ? n : 16;
  p.z_down = groups * s * zn <= 8 * sms ? zn : 1;
  p.mt_up = M <= 16 || R > 64 ? 1 : 2;
  const int64_t tiles = (M + 16 * p.mt_up - 1) / (16 * p.mt_up);
  int cols = 32 * kLoraWarps;
  while (cols < 2048 && tiles * ((N + 2 * cols - 1) / (2 * cols)) >= 8 * sms) cols *= 2;
  p.cols = cols;
  p.z_up = tiles * ((N + cols - 1) / cols) * zn <= 8 * sms ? zn : 1;
  return p;
}

int64_t lora_workspace(int64_t M, int64_t K, int64_t N, int R, int n) {
  return (int64_t)lora_plan(M, K, N, R, n).splits * M * ((R + 7) / 8 * 8);
}

template <typename T, int NT, bool VEC>
static cudaError_t lora_down_t(const LoraArgs& a, const LoraPlan& p, cudaStream_t st) {
  const int64_t rows = 16 * p.mt_down * (kLoraWarps / p.wk);
  const dim3 grid((unsigned)((a.M + rows - 1) / rows), (unsigned)p.splits, (unsigned)p.z_down);
  if (p.wk == 8) lora_down_kernel<T, NT, 1, 8, VEC><<<grid, 32 * kLoraWarps, 0, st>>>(a);
  else if (p.mt_down == 1) lora_down_kernel<T, NT, 1, 2, VEC><<<grid, 32 * kLoraWarps, 0, st>>>(a);
  else if constexpr (NT <= 8) lora_down_kernel<T, NT, 2, 2, VEC><<<grid, 32 * kLoraWarps, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T, int KS>
static cudaError_t lora_up_t(const LoraArgs& a, const LoraPlan& p, bool veco, bool vecb, cudaStream_t st) {
  const int64_t rows = 16 * p.mt_up;
  const dim3 grid((unsigned)((a.M + rows - 1) / rows), (unsigned)((a.N + p.cols - 1) / p.cols), (unsigned)p.z_up);
  const int th = 32 * kLoraWarps;
#define IC_UP(MT)                                                                         \
  if (veco && vecb) lora_up_kernel<T, KS, MT, true, true><<<grid, th, 0, st>>>(a, p.cols); \
  else lora_up_kernel<T, KS, MT, false, false><<<grid, th, 0, st>>>(a, p.cols);
  if constexpr (KS <= 4) {
    if (p.mt_up == 2) { IC_UP(2) return cudaGetLastError(); }
  }
  IC_UP(1)
#undef IC_UP
  return cudaGetLastError();
}

template <typename T>
static cudaError_t lora_t(const LoraArgs& a, cudaStream_t st) {
  const LoraPlan p = lora_plan(a.M, a.K, a.N, a.R, a.n);
  const auto al = [](const void* q, int by) { return (reinterpret_cast<uintptr_t>(q) & (by - 1)) == 0; };
  const bool vec = al(a.x, 16) && al(a.down, 16) && a.ldx % 8 == 0 && a.K % 8 == 0;
  const bool veco = (!a.base || (al(a.base, 16) && a.ldb % 8 == 0)) && al(a.out, 16) && a.ldo % 8 == 0 && a.N % 8 == 0;
  const bool vecb = al(a.up, 8) && a.R % 4 == 0;
#define IC_DOWN(NT) e = vec ? lora_down_t<T, NT, true>(c, p, st) : lora_down_t<T, NT, false>(c, p, st)
  for (int r0 = 0; r0 < a.R; r0 += 128) {   // accumulators hold 128 ranks
    LoraArgs c = a;
    c.r0 = r0;
    c.Rc = a.R - r0 < 128 ? a.R - r0 : 128;
    cudaError_t e;
    if (c.Rc <= 8) IC_DOWN(1);
    else if (c.Rc <= 16) IC_DOWN(2);
    else if (c.Rc <= 32) IC_DOWN(4);
    else if (c.Rc <= 64) IC_DOWN(8);
    else IC_DOWN(16);
    if (e != cudaSuccess) return e;
  }
#undef IC_DOWN
  if (a.R <= 16) return lora_up_t<T, 1>(a, p, veco, vecb, st);
  if (a.R <= 32) return lora_up_t<T, 2>(a, p, veco, vecb, st);
  if (a.R <= 64) return lora_up_t<T, 4>(a, p, veco, vecb, st);
  if (a.R <= 128) return lora_up_t<T, 8>(a, p, veco, vecb, st);
  return lora_up_t<T, 16>(a, p, veco, vecb, st);
}

cudaError_t launch_lora_batched(LoraArgs a, int dtype, cudaStream_t st) {
  if (a.M == 0 || a.N == 0) return cudaSuccess;
  a.splits = lora_plan(a.M, a.K, a.N, a.R, a.n).splits;
  return dtype == IC_DTYPE_BF16 ? lora_t<__nv_bfloat16>(a, st) : lora_t<__half>(a, st);
}

}  // namespace ic
