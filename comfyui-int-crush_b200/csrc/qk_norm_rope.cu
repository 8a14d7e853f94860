// Per-head RMS norm of queries and keys with the position rotation, one pass.
//
//   y = x * rsqrt(mean_D(x^2) + eps) * gamma              (fp32)
//   interleaved: pairs (2i, 2i+1), half: pairs (i, i + rot/2), i < rot/2:
//     (a, b) -> (a cos - b sin, b cos + a sin), cos / sin = table[position][i]
//   elements past rot keep y; one rounding to the activation type.
//
// Bound by HBM: 4 bytes per element against ~8 instructions.  One head's
// vector sits in D/8 lanes of one warp (16 bytes each, rounded up to a power
// of two), so the mean is a shuffle reduction, and a group of lanes takes up
// to kHeads heads of one token: their loads are all in flight together and
// the token's table row and gamma are read once for all of them.  A half
// layout's partner chunk comes by shuffle of the raw 16-bit pairs when rot/2
// is a multiple of 8, otherwise element by element from the row (an L1 hit);
// every lane reads before any lane of the warp writes, so the output may be
// the input.
#include "ic_common.cuh"

namespace ic {

struct QkArgs {
  // 0: queries, 1: keys; strides in elements over batch, token, head
  const void* x[2];
  void* y[2];
  int64_t xs[2][3], ys[2][3];
  const float* gamma[2];          // [D] or NULL (ones)
  int heads[2];
  int units[2];                   // head groups of a token
  int per_unit[2];                // heads in each (the last may have fewer)
  int64_t B, Lq;                  // tokens of a sample
  int D, rot;
  float eps;
  const float* cosp;              // [table, rot / 2]
  const float* sinp;
  int64_t table;
  const int32_t* positions;       // [B, L] or NULL (the token's own index)
};

constexpr int kQkThreads = 256;
constexpr int kQkHeads = 8;

// LAYOUT 0: no rotation, 1: interleaved, 2: half with rot/2 % 8 == 0,
// 3: half, any even rot.  LANES: lanes of a head's vector.
template <typename T, int LANES, int LAYOUT>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_kernel(const QkArgs a) {
  const int lane = threadIdx.x & (LANES - 1);
  const int per_token = a.units[0] + a.units[1];
  const int64_t unit = ((int64_t)blockIdx.x * kQkThreads + threadIdx.x) / LANES;
  const int64_t tokens = a.B * a.Lq;
  // lanes past the end keep running (shuffles below name the whole warp)
  const int64_t token = unit / per_token < tokens ? unit / per_token : tokens - 1;
  const bool live = unit / per_token < tokens;
  const int u = (int)(unit % per_token);
  const int which = u < a.units[0] ? 0 : 1;
  const int h0 = (which ? u - a.units[0] : u) * a.per_unit[which];
  const int nh = min(a.per_unit[which], a.heads[which] - h0);
  const int64_t b = token / a.Lq, l = token - b * a.Lq;
  const int d0 = lane * 8;
  const bool on = live && d0 < a.D;
  const T* x = reinterpret_cast<const T*>(a.x[which]) + b * a.xs[which][0] + l * a.xs[which][1] +
               (int64_t)h0 * a.xs[which][2];
  T* y = reinterpret_cast<T*>(a.y[which]) + b * a.ys[which][0] + l * a.ys[which][1] + (int64_t)h0 * a.ys[which][2];

  uint4 raw[kQkHeads];
#pragma unroll
  for (int h = 0; h < kQkHeads; ++h) {
    raw[h] = make_uint4(0u, 0u, 0u, 0u);
    if (on && h < nh) raw[h] = *reinterpret_cast<const uint4*>(x + (int64_t)h * a.xs[which][2] + d0);
  }
  float g[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = 1.f;
  if (on && a.gamma[which]) {
    const float4 lo = __ldg(reinterpret_cast<const float4*>(a.gamma[which] + d0));
    const float4 hi = __ldg(reinterpret_cast<const float4*>(a.gamma[which] + d0) + 1);
    g[0] = lo.x; g[1] = lo.y; g[2] = lo.z; g[3] = lo.w;
    g[4] = hi.x; g[5] = hi.y; g[6] = hi.z; g[7] = hi.w;
  }

  // the token's angles: element i of this lane turns with c[i], s[i]; the
  // partner enters with +s (second of a pair) or -s (first of a pair)
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { c[i] = 1.f; s[i] = 0.f; }
  const int half = a.rot >> 1;
  bool bad = false;
  if constexpr (LAYOUT != 0) {
    int64_t pos = l;
    if (a.positions) pos = __ldg(a.positions + token);
    bad = pos < 0 || pos >= a.table;
    if (bad) {
      // no table row: the token's heads become NaN and the error word says so
      if (live && lane == 0) set_dev_error(IC_DEV_ERR_INDEX);
    } else if (d0 < a.rot) {
      const float* ct = a.cosp + pos * half;
      const float* st = a.sinp + pos * half;
      if constexpr (LAYOUT == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (d0 + 2 * i < a.rot) {
            const float cv = __ldg(ct + d0 / 2 + i), sv = __ldg(st + d0 / 2 + i);
            c[2 * i] = c[2 * i + 1] = cv;
            s[2 * i] = -sv;
            s[2 * i + 1] = sv;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = d0 + i;
          if (d < a.rot) {
            const int j = d < half ? d : d - half;
            c[i] = __ldg(ct + j);
            const float sv = __ldg(st + j);
            s[i] = d < half ? -sv : sv;
          }
        }
      }
    }
  }

  // LAYOUT 3 reads partners from memory: all of them before any store
  [[maybe_unused]] T part[LAYOUT == 3 ? kQkHeads : 1][8];
  if constexpr (LAYOUT == 3) {
#pragma unroll
    for (int h = 0; h < kQkHeads; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        part[h][i] = DT<T>::from_f(0.f);
        if (on && h < nh && d < a.rot) {
          const int pd = d < half ? d + half : d - half;
          part[h][i] = x[(int64_t)h * a.xs[which][2] + pd];
        }
      }
    __syncwarp();
  }
  // gamma of the partner element (half layouts)
  [[maybe_unused]] float pg[8];
  if constexpr (LAYOUT >= 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + i;
      pg[i] = 1.f;
      if (d < a.rot && a.gamma[which]) pg[i] = __ldg(a.gamma[which] + (d < half ? d + half : d - half));
    }
  }

  float ss[kQkHeads];
#pragma unroll
  for (int h = 0; h < kQkHeads; ++h) {
    const T* e = reinterpret_cast<const T*>(&raw[h]);
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) { const float f = DT<T>::to_f(e[i]); v = fmaf(f, f, v); }
    ss[h] = v;
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
    for (int h = 0; h < kQkHeads; ++h) ss[h] += __shfl_xor_sync(0xffffffffu, ss[h], o);

#pragma unroll
  for (int h = 0; h < kQkHeads; ++h) {
    const float r = rsqrtf(ss[h] / (float)a.D + a.eps);
    const T* e = reinterpret_cast<const T*>(&raw[h]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = DT<T>::to_f(e[i]) * r * g[i];
    float o[8];
    if constexpr (LAYOUT == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = v[i];
    } else if constexpr (LAYOUT == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = d0 + i < a.rot ? fmaf(v[i], c[i], v[i ^ 1] * s[i]) : v[i];
    } else {
      T pe[8];
      if constexpr (LAYOUT == 2) {
        // chunk lane +- half/8 holds the partners; lanes past rot keep their own
        const int src = d0 < half ? lane + half / 8 : (d0 < a.rot ? lane - half / 8 : lane);
        uint4 pr;
        pr.x = __shfl_sync(0xffffffffu, raw[h].x, src, LANES);
        pr.y = __shfl_sync(0xffffffffu, raw[h].y, src, LANES);
        pr.z = __shfl_sync(0xffffffffu, raw[h].z, src, LANES);
        pr.w = __shfl_sync(0xffffffffu, raw[h].w, src, LANES);
        const T* q = reinterpret_cast<const T*>(&pr);
#pragma unroll
        for (int i = 0; i < 8; ++i) pe[i] = q[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) pe[i] = part[h][i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        o[i] = d0 + i < a.rot ? fmaf(v[i], c[i], DT<T>::to_f(pe[i]) * r * pg[i] * s[i]) : v[i];
    }
    if (bad) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = __int_as_float(0x7fc00000);
    }
    if (on && h < nh) {
      T t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = DT<T>::from_f(o[i]);
      uint4 w;
      memcpy(&w, t, 16);
      *reinterpret_cast<uint4*>(y + (int64_t)h * a.ys[which][2] + d0) = w;
    }
  }
}

template <typename T, int LANES>
static cudaError_t launch_qk_l(const QkArgs& a, int layout, unsigned blocks, cudaStream_t st) {
  switch (layout) {
    case 0: qk_norm_rope_kernel<T, LANES, 0><<<blocks, kQkThreads, 0, st>>>(a); break;
    case 1: qk_norm_rope_kernel<T, LANES, 1><<<blocks, kQkThreads, 0, st>>>(a); break;
    case 2: qk_norm_rope_kernel<T, LANES, 2><<<blocks, kQkThreads, 0, st>>>(a); break;
    default: qk_norm_rope_kernel<T, LANES, 3><<<blocks, kQkThreads, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_qk_t(const QkArgs& a, int layout, cudaStream_t st) {
  int lanes = 4;
  while (lanes * 8 < a.D) lanes *= 2;
  const int64_t threads = a.B * a.Lq * (a.units[0] + a.units[1]) * lanes;
  const unsigned blocks = (unsigned)((threads + kQkThreads - 1) / kQkThreads);
  switch (lanes) {
    case 4: return launch_qk_l<T, 4>(a, layout, blocks, st);
    case 8: return launch_qk_l<T, 8>(a, layout, blocks, st);
    case 16: return launch_qk_l<T, 16>(a, layout, blocks, st);
    default: return launch_qk_l<T, 32>(a, layout, blocks, st);
  }
}

// heads shared evenly over the fewest groups of at most kQkHeads
static void qk_units(QkArgs& a) {
  for (int i = 0; i < 2; ++i) {
    a.units[i] = (a.heads[i] + kQkHeads - 1) / kQkHeads;
    a.per_unit[i] = a.units[i] ? (a.heads[i] + a.units[i] - 1) / a.units[i] : 1;
    a.units[i] = a.heads[i] ? (a.heads[i] + a.per_unit[i] - 1) / a.per_unit[i] : 0;
  }
}

// layout: 0 interleaved, 1 half (rot 0: none)
cudaError_t launch_qk_norm_rope(QkArgs a, int dtype, int layout, cudaStream_t st) {
  if (a.B == 0 || a.Lq == 0 || a.heads[0] + a.heads[1] == 0) return cudaSuccess;
  qk_units(a);
  const int form = a.rot == 0 ? 0 : layout == 0 ? 1 : (a.rot / 2) % 8 == 0 ? 2 : 3;
  return dtype == IC_DTYPE_BF16 ? launch_qk_t<__nv_bfloat16>(a, form, st) : launch_qk_t<__half>(a, form, st);
}

}  // namespace ic
