// Cross attention to an encoder's states: masks, the kernel for few query
// rows, and the join of split keys.  (Many rows: cross_attention_tc.cu.)
//
//   o[b, l, h] = sum_j p_j v[b, j, hk] / sum_j p_j,
//   p_j = exp(scale * q[b, l, h] . k[b, j, hk] + mask[b, j]),  hk = h / (H / Hk)
//
// over the keys that sample b sees: j < kv_lens[b], mask not false and not
// -inf.  A key that is not seen does not count whatever its k and v hold; a
// sample that sees none gets zeros.
#include "cross_attention.cuh"

#include <type_traits>

namespace ic {

// ------------------------------------------------------------------- masks
// bias[b, j] = log2(e) * (mask[b, j] - max_j mask[b, j]), -inf for a key that
// is not seen (rows padded to a multiple of 128 with it), and ends[b] = 1 +
// the last key that is seen.  A constant added to all of a sample's scores
// cancels in the softmax; taking the largest mask value away keeps the sums
// exact where every mask value is a type's lowest (-65504 + s would lose
// 16 bits of s).  One CTA per sample: at 512 to 16384 keys it is one launch's
// latency, whatever the layout.
template <typename M>
__device__ __forceinline__ float mask_value(const void* mask, int64_t i) {
  if constexpr (std::is_same<M, uint8_t>::value)
    return reinterpret_cast<const uint8_t*>(mask)[i] ? 0.f : -INFINITY;
  else if constexpr (std::is_same<M, float>::value)
    return reinterpret_cast<const float*>(mask)[i];
  else
    return DT<M>::to_f(reinterpret_cast<const M*>(mask)[i]);
}

template <typename M>
__global__ void __launch_bounds__(1024) xattn_mask_kernel(const void* mask, int64_t ld, const int32_t* kv_lens,
                                                          int64_t Lk, int64_t Lkp, float* bias, int32_t* ends) {
  __shared__ float wmax[32];
  __shared__ int wend[32];
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t len = Lk;
  if (kv_lens) len = max((int64_t)0, min((int64_t)kv_lens[b], Lk));
  float mx = -INFINITY;
  for (int64_t j = threadIdx.x; j < len; j += 1024) mx = fmaxf(mx, mask_value<M>(mask, b * ld + j));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) wmax[warp] = mx;
  __syncthreads();
  mx = wmax[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  int end = 0;
  for (int64_t j = threadIdx.x; j < Lkp; j += 1024) {
    const float m = j < len ? mask_value<M>(mask, b * ld + j) : -INFINITY;
    const float v = m == -INFINITY ? -INFINITY : (m - mx) * kLog2e;
    bias[b * Lkp + j] = v;
    if (!(v == -INFINITY)) end = (int)j + 1;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) end = max(end, __shfl_xor_sync(0xffffffffu, end, o));
  if (lane == 0) wend[warp] = end;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) end = max(end, wend[w]);
    ends[b] = end;
  }
}

// --------------------------------------------------------------- few rows
// The rows of one key head (Lq tokens times the query heads that share it)
// in tiles of 16; four warps go over the keys in blocks of 16, each warp its
// own blocks, and the keys are split over CTAs when there are few tiles.
// A lane's 16-byte loads of K (row = key, chunk of 8 elements) are MMA
// fragments as they are, with the order of the summed elements permuted alike
// in Q, and V's fragments pair two keys of one element by a byte permutation
// of two loads.  What bounds it is the stream of K and V from HBM and the
// warps' own instructions beside it, so the next block is in flight (8 KB a
// warp at D = 128) while one is computed, as asynchronous copies to a ring of
// the warp's own in shared memory: every lane reads back what it copied, so the
// ring needs no barrier, and its registers leave room for three CTAs per SM (168
// of them; above D = 64, with a mask, or above 96 without, 12 to 52 bytes a thread
// go to local memory).
// 8 single tokens of 32 heads over 8 key heads of 128, 1024 to 8192 keys (151
// MB): 46 us with the join, 3.3 TB/s, as the tcgen05 kernel; loads straight to
// registers 49 us.  The copies alone take 44 us of that, the arithmetic alone 22.
// Softmax: scores, references (kXattnUp) and sums in fp32.  p enters the product
// with V rounded to the activation type, which is the MMA's operand type, its
// sum unrounded: at most u sum_j p_j |v_j| beside the output's own rounding.
constexpr int kXsWarps = 4;

template <typename T>
__device__ __forceinline__ void xs_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int NC>
struct XsCfg {
  static constexpr int NH = (NC + 1) / 2;              // 64-element halves of V
  static constexpr int LOADS = 2 * NC + 4 * NH;        // of a lane for a block
  static constexpr int STAGES = 2;                     // one in use, one in flight
  static constexpr int RING = kXsWarps * STAGES * LOADS * 512;
  static constexpr int JOIN = kXsWarps * 16 * (64 * NH + 4) * 4;
  static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

// NC: 32-element chunks of the head (D <= 32 * NC).
template <typename T, int NC, bool BIAS>
__global__ void __launch_bounds__(32 * kXsWarps, 3) xattn_rows_kernel(const XattnArgs a) {
  using C = XsCfg<NC>;
  constexpr int NH = C::NH, S = C::STAGES;
  constexpr int DP = 64 * NH;
  extern __shared__ __align__(16) uint8_t ring[];
  float (*so)[16][DP + 4] = reinterpret_cast<float (*)[16][DP + 4]>(ring);   // after the loop
  __shared__ float sm[kXsWarps][16], sl[kXsWarps][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int group = a.H / a.Hk;
  const int64_t rows = a.Lq * group, tiles = (rows + 15) / 16;
  const int64_t bh = blockIdx.x / tiles;
  const int64_t b = bh / a.Hk;
  const int hk = (int)(bh % a.Hk);
  const int64_t row0 = (blockIdx.x - bh * tiles) * 16;
  const T* kp = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* vp = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];

  const int end = xattn_end(a, b);
  // parts of the same length for every sample: a short one has fewer of them,
  // and a part past its end nothing to do
  const int blocks = (end + 15) / 16;
  const int blk0 = (int)blockIdx.y * a.part_blocks, blk1 = min(blk0 + a.part_blocks, blocks);
  if (blk0 >= blocks && blockIdx.y > 0) return;

  uint4 qv[2][NC];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t r = row0 + 8 * h + g;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      qv[h][c] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows && 32 * c + 8 * t < a.D)
        qv[h][c] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + b * a.qs[0] +
                                                        r / group * a.qs[1] + (hk * group + r % group) * a.qs[2] +
                                                        32 * c + 8 * t));
    }
  }
  float o[NH][8][4];
#pragma unroll
  for (int i = 0; i < NH; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};   // references, sums
  const float sc = a.scale * kLog2e;

  const uint32_t mine = smem_u32(ring) + warp * S * C::LOADS * 512 + lane * 16;
  // K rows 8i + g, chunk t of 32 elements; V rows 2t, + 1, + 8, + 9 (this lane's
  // keys), chunk g of 64.  A key past the end is not read (zeros).
  const T* kl = kp + g * a.ks[1] + 8 * t;
  const T* vl = vp + 2 * t * a.vs[1] + 8 * g;
  const bool full_d = a.D == 32 * NC && NC % 2 == 0;
  const auto copy = [&](int blk, int stage) {
    const uint32_t to = mine + stage * C::LOADS * 512;
    const T* k0 = kl + (int64_t)(16 * blk) * a.ks[1];
    const T* v0 = vl + (int64_t)(16 * blk) * a.vs[1];
    if (full_d && blk < blk1 && 16 * blk + 16 <= end) {
#pragma unroll
      for (int i = 0; i < 2; ++i, k0 += 8 * a.ks[1])
#pragma unroll
        for (int c = 0; c < NC; ++c) cp_async16(to + (i * NC + c) * 512, k0 + 32 * c, true);
#pragma unroll
      for (int e = 0; e < 4; ++e, v0 += e == 2 ? 7 * a.vs[1] : a.vs[1])
#pragma unroll
        for (int i = 0; i < NH; ++i) cp_async16(to + (2 * NC + e * NH + i) * 512, v0 + 64 * i, true);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const bool on = blk < blk1 && 16 * blk + 8 * i + g < end && 32 * c + 8 * t < a.D;
          cp_async16(to + (i * NC + c) * 512, on ? k0 + 8 * i * a.ks[1] + 32 * c : kp, on);
        }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < NH; ++i) {
          const int r = (e & 1) + 8 * (e >> 1);
          const bool on = blk < blk1 && 16 * blk + 2 * t + r < end && 64 * i + 8 * g < a.D;
          cp_async16(to + (2 * NC + e * NH + i) * 512, on ? v0 + r * a.vs[1] + 64 * i : vp, on);
        }
    }
    cp_async_commit();
  };
  const auto load_bias = [&](float (&bs)[4], int blk) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = blk * 16 + 2 * t + (e & 1) + 8 * (e >> 1);
      bs[e] = 0.f;
      if constexpr (BIAS) {
        if (blk < blk1) bs[e] = __ldg(a.bias + b * a.Lkp + j);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) copy(blk0 + warp + kXsWarps * i, i);
  float bs[4], bn[4];
  load_bias(bs, blk0 + warp);
  int stage = 0;
  for (int blk = blk0 + warp; blk < blk1; blk += kXsWarps) {
    copy(blk + kXsWarps * (S - 1), stage == 0 ? S - 1 : stage - 1);   // the stage used last
    load_bias(bn, blk + kXsWarps);
    cp_async_wait<S - 1>();
    uint4 kv[2][NC], vv[NH][4];
    const uint8_t* from = ring + (mine - smem_u32(ring)) + stage * C::LOADS * 512;
    bool seen[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      seen[e] = blk * 16 + 2 * t + (e & 1) + 8 * (e >> 1) < end && !(BIAS && bs[e] == -INFINITY);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < NC; ++c) kv[i][c] = *reinterpret_cast<const uint4*>(from + (i * NC + c) * 512);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        vv[i][e] = *reinterpret_cast<const uint4*>(from + (2 * NC + e * NH + i) * 512);
        if (BIAS && !seen[e]) vv[i][e] = make_uint4(0u, 0u, 0u, 0u);   // 0 * NaN is not 0
      }
    float s[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        xs_mma<T>(s[i], qv[0][c].x, qv[1][c].x, qv[0][c].y, qv[1][c].y, kv[i][c].x, kv[i][c].y);
        xs_mma<T>(s[i], qv[0][c].z, qv[1][c].z, qv[0][c].w, qv[1][c].w, kv[i][c].z, kv[i][c].w);
      }
    }
    // row h (g, g + 8), key e -> s[e >> 1][2h + (e & 1)]
    float x[2][4], mx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = s[e >> 1][2 * h + (e & 1)];
        x[h][e] = seen[e] ? (BIAS ? fmaf(y, sc, bs[e]) : y * sc) : -INFINITY;
        mx[h] = fmaxf(mx[h], x[h][e]);
      }
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
    }
    if (__any_sync(0xffffffffu, xattn_moves<T>(mx[0], m[0]) || xattn_moves<T>(mx[1], m[1]))) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float nm = fmaxf(m[h], mx[h] - kXattnUp<T>);
        const float f = nm == m[h] ? 1.f : ex2(m[h] - nm);
        m[h] = nm;
        l[h] *= f;
#pragma unroll
        for (int i = 0; i < NH; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            o[i][j][2 * h] *= f;
            o[i][j][2 * h + 1] *= f;
          }
      }
    }
    uint32_t p[2][2];   // [row][key pair]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float ref = m[h] == -INFINITY ? 0.f : m[h];
      float e4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        e4[e] = ex2(x[h][e] - ref);
        l[h] += e4[e];
      }
      p[h][0] = pack16<T>(e4[0], e4[1]);
      p[h][1] = pack16<T>(e4[2], e4[3]);
    }
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      const uint32_t w[4][4] = {{vv[i][0].x, vv[i][0].y, vv[i][0].z, vv[i][0].w},
                                {vv[i][1].x, vv[i][1].y, vv[i][1].z, vv[i][1].w},
                                {vv[i][2].x, vv[i][2].y, vv[i][2].z, vv[i][2].w},
                                {vv[i][3].x, vv[i][3].y, vv[i][3].z, vv[i][3].w}};
      // tile j's column g is element 64 i + 8 g + j
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
        xs_mma<T>(o[i][j], p[0][0], p[1][0], p[0][1], p[1][1], __byte_perm(w[0][j >> 1], w[1][j >> 1], sel),
                  __byte_perm(w[2][j >> 1], w[3][j >> 1], sel));
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) bs[e] = bn[e];
    stage = stage == S - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  __syncthreads();   // the ring becomes the joined sums
  // join the warps: row sums over the quad first
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (t == 0) {
      sm[warp][8 * h + g] = m[h];
      sl[warp][8 * h + g] = l[h];
    }
#pragma unroll
    for (int i = 0; i < NH; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int j = 0; j < 8; j += 4)
          *reinterpret_cast<float4*>(&so[warp][8 * h + g][64 * i + 8 * (2 * t + q) + j]) =
              make_float4(o[i][j][2 * h + q], o[i][j + 1][2 * h + q], o[i][j + 2][2 * h + q], o[i][j + 3][2 * h + q]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * (DP / 8); i += 32 * kXsWarps) {
    const int r = i / (DP / 8), d = i % (DP / 8) * 8;
    const int64_t row = row0 + r;
    if (row >= rows || d >= a.D) continue;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kXsWarps; ++w) mm = fmaxf(mm, sm[w][r]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kXsWarps; ++w) {
      const float f = ex2(sm[w][r] - ref);
      sum = fmaf(sl[w][r], f, sum);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(so[w][r][d + e], f, v[e]);
    }
    const int64_t lq = row / group, h = hk * group + row % group;
    xattn_put<T>(a, b, lq, (int)h, (int)blockIdx.y, d, v, mm, sum);
  }
}

// ------------------------------------------------------------------- join
// One thread per 8 elements of an output row: the splits' sums weighted to
// their largest reference, in split order.
template <typename T>
__global__ void __launch_bounds__(128) xattn_join_kernel(const XattnArgs a) {
  const int dq = a.D / 8;
  const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int64_t rows = a.B * a.Lq * a.H;
  if (i >= rows * dq) return;
  const int64_t row = i / dq;
  const int d = (int)(i % dq) * 8;
  // parts that the sample has (the tcgen05 kernel writes all)
  int splits = a.splits;
  if (a.part_blocks) {
    const int blocks = (xattn_end(a, row / a.H / a.Lq) + 15) / 16;
    splits = max(1, min(splits, (blocks + a.part_blocks - 1) / a.part_blocks));
  }
  float mm = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) mm = fmaxf(mm, a.part_ml[(s * rows + row) * 2]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (s * rows + row) * 2);
    const float f = ex2(ml.x - ref);
    const float4* p = reinterpret_cast<const float4*>(a.part_o + (s * rows + row) * a.D + d);
    const float4 lo = p[0], hi = p[1];
    sum = fmaf(ml.y, f, sum);
    v[0] = fmaf(lo.x, f, v[0]); v[1] = fmaf(lo.y, f, v[1]); v[2] = fmaf(lo.z, f, v[2]); v[3] = fmaf(lo.w, f, v[3]);
    v[4] = fmaf(hi.x, f, v[4]); v[5] = fmaf(hi.y, f, v[5]); v[6] = fmaf(hi.z, f, v[6]); v[7] = fmaf(hi.w, f, v[7]);
  }
  const int64_t h = row % a.H, bl = row / a.H;
  xattn_store8<T>(a, bl / a.Lq, bl % a.Lq, (int)h, d, v, sum);
}

// ---------------------------------------------------------------- launches
// The tcgen05 kernel takes over above 8 query rows of a key head (tokens times
// heads), and for fewer from 2^15 rows of keys in the batch.  Measured, few-rows
// against tcgen05 kernel: 1 x 8 rows, 24 heads, 512 keys 9.9 / 10.6 us, 16 rows
// 11.5 / 10.6; 8 x 1 token, 32 heads over 8, 1024 keys 20.5 / 15.2; 1 token of 24
// heads over 512 keys 9.5 / 10.4, of 8 heads over 77 keys 3.9 / 5.3.
constexpr int64_t kTcRows = 8, kTcKeys = 1 << 15;
// Items per SM that its keys are split for: 8 x 1 token of 32 heads over 8, 1024
// to 8192 keys: one 59 us, two 46.6, four 47.5, eight 52.
constexpr int64_t kTcItems = 2;

// Splits of the few-rows kernel: four CTAs per SM, with at least 8 blocks of 16
// keys (two per warp) in a part (the case above: two CTAs per SM 57 us, three
// 48 to 53, four 46, six 50 to 55, ten 52).
static int rows_splits(int64_t B, int64_t Lq, int64_t Lk, int H, int Hk) {
  const int64_t ctas = (Lq * (H / Hk) + 15) / 16 * B * Hk;
  const int64_t blocks = (Lk + 15) / 16;
  int64_t s = (4 * (int64_t)num_sms() + ctas - 1) / ctas;
  const int64_t most = (blocks + 7) / 8;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

// Splits and slots of the tcgen05 kernel: two query tiles per CTA share K and
// V; with too few tiles for that to fill the SMs, one, and then the keys are
// split with two tiles of 128 at least in a part.
static int tc_splits(int64_t B, int64_t Lq, int64_t Lk, int H, int Hk, int* slots) {
  const int64_t sms = num_sms();
  const int64_t packed = xattn_packed(H, Hk);
  const int64_t tiles = H / Hk / packed * ((Lq * packed + 127) / 128);
  *slots = B * Hk * tiles <= sms ? 1 : 2;
  const int64_t items = B * Hk * ((tiles + *slots - 1) / *slots);
  int64_t s = kTcItems * sms / items;
  const int64_t most = ((Lk + 127) / 128 + 1) / 2;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

XattnPlan xattn_plan(int64_t B, int64_t Lq, int64_t Lk, int H, int Hk, int D, int mask_kind) {
  XattnPlan p;
  p.slots = 0;
  if (Lk == 0) p.splits = 1;
  else if (Lq * (H / Hk) > kTcRows || B * Hk * Lk >= kTcKeys) p.splits = tc_splits(B, Lq, Lk, H, Hk, &p.slots);
  else p.splits = rows_splits(B, Lq, Lk, H, Hk);
  p.Lkp = mask_kind ? (Lk + 127) / 128 * 128 : 0;
  const int64_t rows = B * Lq * H;
  p.part_floats = p.splits > 1 ? ((int64_t)p.splits * rows * (D + 2) + 3) / 4 * 4 : 0;
  p.floats = p.part_floats + (mask_kind ? B * p.Lkp + (B + 3) / 4 * 4 : 0);
  return p;
}

template <typename T, bool BIAS>
static cudaError_t launch_rows(const XattnArgs& a, cudaStream_t st) {
  const int64_t tiles = (a.Lq * (a.H / a.Hk) + 15) / 16 * a.B * a.Hk;
  if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)tiles, (unsigned)a.splits);
  const auto go = [&](auto* kern, int smem) {
    const cudaError_t e = set_smem_once(kern, smem);
    if (e != cudaSuccess) return e;
    kern<<<grid, 32 * kXsWarps, smem, st>>>(a);
    return cudaGetLastError();
  };
  if (a.D <= 32) return go(xattn_rows_kernel<T, 1, BIAS>, XsCfg<1>::SMEM);
  if (a.D <= 64) return go(xattn_rows_kernel<T, 2, BIAS>, XsCfg<2>::SMEM);
  if (a.D <= 96) return go(xattn_rows_kernel<T, 3, BIAS>, XsCfg<3>::SMEM);
  return go(xattn_rows_kernel<T, 4, BIAS>, XsCfg<4>::SMEM);
}

template <typename T>
static cudaError_t launch_xattn_t(const XattnArgs& a, int slots, cudaStream_t st) {
  cudaError_t e = slots ? launch_xattn_tc<T>(a, slots, st)
                        : a.bias ? launch_rows<T, true>(a, st) : launch_rows<T, false>(a, st);
  if (e != cudaSuccess || a.splits == 1) return e;
  const int64_t n = a.B * a.Lq * a.H * (a.D / 8);
  xattn_join_kernel<T><<<(unsigned)((n + 127) / 128), 128, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_cross_attention(XattnArgs a, int dtype, const void* mask, int mask_kind, int64_t ld_mask,
                                   float* workspace, cudaStream_t st) {
  if (a.B == 0 || a.Lq == 0) return cudaSuccess;
  XattnPlan p = xattn_plan(a.B, a.Lq, a.Lk, a.H, a.Hk, a.D, mask_kind);
  // the tcgen05 kernel takes row maxima before the scale: only with a positive
  // one.  Others are nobody's ordinary call: the few-rows kernel, unsplit.
  if (p.slots && !(a.scale > 0.f)) p.slots = 0, p.splits = 1;
  a.splits = p.splits;
  a.part_blocks = p.slots ? 0 : (int)(((a.Lk + 15) / 16 + p.splits - 1) / p.splits);
  a.Lkp = p.Lkp;
  a.part_o = workspace;
  a.part_ml = workspace + p.part_floats / (a.D + 2) * a.D;
  if (mask_kind) {
    float* bias = workspace + p.part_floats;
    int32_t* ends = reinterpret_cast<int32_t*>(bias + a.B * p.Lkp);
    const unsigned n = (unsigned)a.B;
    switch (mask_kind) {
      case IC_MASK_BOOL:
        xattn_mask_kernel<uint8_t><<<n, 1024, 0, st>>>(mask, ld_mask, a.kv_lens, a.Lk, p.Lkp, bias, ends);
        break;
      case IC_MASK_F16:
        xattn_mask_kernel<__half><<<n, 1024, 0, st>>>(mask, ld_mask, a.kv_lens, a.Lk, p.Lkp, bias, ends);
        break;
      case IC_MASK_BF16:
        xattn_mask_kernel<__nv_bfloat16><<<n, 1024, 0, st>>>(mask, ld_mask, a.kv_lens, a.Lk, p.Lkp, bias, ends);
        break;
      default:
        xattn_mask_kernel<float><<<n, 1024, 0, st>>>(mask, ld_mask, a.kv_lens, a.Lk, p.Lkp, bias, ends);
    }
    a.bias = bias;
    a.ends = ends;
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return dtype == IC_DTYPE_BF16 ? launch_xattn_t<__nv_bfloat16>(a, p.slots, st) : launch_xattn_t<__half>(a, p.slots, st);
}

}  // namespace ic
