// Per-head RMS norm of queries and keys with the position rotation, one pass.
//
//   y = x * rsqrt(mean_D(x^2) + eps) * gamma              (fp32)
//   interleaved: pairs (2i, 2i+1), half: pairs (i, i + rot/2), i < rot/2:
//     (a, b) -> (a cos - b sin, b cos + a sin), cos / sin = table[position][i]
//   elements past rot keep y; one rounding to the activation type.
//
// Bound by HBM (4 bytes per element), with the instruction issue close behind
// (7 to 8 instructions per element).  One head's
// vector sits in D/8 lanes of one warp (16 bytes each, rounded up to a power
// of two), so the mean is a shuffle reduction.  A group of lanes takes several
// heads of one token, two at a time, the next two's loads in flight meanwhile;
// the token's table row and gamma are read once for all of them and folded
// into two factors per element, for itself and for its partner.  A half
// layout's partner chunk comes by shuffle of the raw 16-bit pairs when rot/2
// is a multiple of 8, otherwise element by element from the row (an L1 hit);
// every lane reads before any lane of the warp writes, so the output may be
// the input.  80 registers for three CTAs per SM; the half layout (LAYOUT 2)
// keeps 32 to 44 bytes a thread in local memory for it.
#include "cross_attention.cuh"   // pack16

namespace ic {

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

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
  unsigned total;                 // units of all tokens
  int D, rot;
  float eps;
  const float* cosp;              // [table, rot / 2]
  const float* sinp;
  int tvec;                       // table rows take 16-byte loads
  int64_t table;
  const int32_t* positions;       // [B, L] or NULL (the token's own index)
};

constexpr int kQkThreads = 256;
constexpr int kQkHeads = 2;       // heads at a time

// LAYOUT 0: no rotation, 1: interleaved, 2: half with rot/2 % 8 == 0,
// 3: half, any even rot.  LANES: lanes of a head's vector.
template <typename T, int LANES, int LAYOUT>
__global__ void __launch_bounds__(kQkThreads, LAYOUT == 3 ? 2 : 3) qk_norm_rope_kernel(const QkArgs a) {
  const int lane = threadIdx.x & (LANES - 1);
  const unsigned per_token = a.units[0] + a.units[1];
  const unsigned unit = blockIdx.x * (kQkThreads / LANES) + threadIdx.x / LANES;
  // lanes past the end keep running (shuffles below name the whole warp)
  const bool live = unit < a.total;
  const unsigned token = (live ? unit : a.total - 1) / per_token;
  const int u = (int)((live ? unit : a.total - 1) - token * per_token);
  const int which = u < a.units[0] ? 0 : 1;
  const int h0 = (which ? u - a.units[0] : u) * a.per_unit[which];
  const int nh = min(a.per_unit[which], a.heads[which] - h0);
  const unsigned b = token / (unsigned)a.Lq;
  const int64_t l = token - b * (unsigned)a.Lq;
  const int d0 = lane * 8;
  const bool on = live && d0 < a.D;
  const int64_t xh = a.xs[which][2], yh = a.ys[which][2];
  const T* x = reinterpret_cast<const T*>(a.x[which]) + b * a.xs[which][0] + l * a.xs[which][1] + h0 * xh + d0;
  T* y = reinterpret_cast<T*>(a.y[which]) + b * a.ys[which][0] + l * a.ys[which][1] + h0 * yh + d0;

  uint4 raw[kQkHeads], next[kQkHeads];
  const auto load = [&](uint4 (&to)[kQkHeads], int hb) {
#pragma unroll
    for (int h = 0; h < kQkHeads; ++h) {
      to[h] = make_uint4(0u, 0u, 0u, 0u);
      if (on && hb + h < nh) to[h] = *reinterpret_cast<const uint4*>(x + (hb + h) * xh);
    }
  };
  load(raw, 0);

  // f[i], p[i]: y_i = r * (x_i f_i + partner_i p_i)
  float f[8], p[8];
  const float* gam = a.gamma[which];
#pragma unroll
  for (int i = 0; i < 8; ++i) { f[i] = 1.f; p[i] = 0.f; }
  if (on && gam) {
    const float4 lo = __ldg(reinterpret_cast<const float4*>(gam + d0));
    const float4 hi = __ldg(reinterpret_cast<const float4*>(gam + d0) + 1);
    f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w;
    f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
  }
  const int half = a.rot >> 1;
  bool bad = false;
  if constexpr (LAYOUT != 0) {
    int64_t pos = l;
    if (a.positions) pos = __ldg(a.positions + token);
    bad = pos < 0 || pos >= a.table;
    if (bad) {
      // no table row: the token's heads become NaN and the error word says so
      if (live && lane == 0) set_dev_error(IC_DEV_ERR_INDEX);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = p[i] = __int_as_float(0x7fc00000);
    } else if (d0 < a.rot) {
      const float* ct = a.cosp + pos * half;
      const float* st = a.sinp + pos * half;
      if constexpr (LAYOUT == 1) {
        float c[4], s[4];
        if (a.tvec && d0 + 8 <= a.rot) {
          const float4 cv = __ldg(reinterpret_cast<const float4*>(ct + d0 / 2));
          const float4 sv = __ldg(reinterpret_cast<const float4*>(st + d0 / 2));
          c[0] = cv.x; c[1] = cv.y; c[2] = cv.z; c[3] = cv.w;
          s[0] = sv.x; s[1] = sv.y; s[2] = sv.z; s[3] = sv.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool in = d0 + 2 * i < a.rot;
            c[i] = in ? __ldg(ct + d0 / 2 + i) : 1.f;
            s[i] = in ? __ldg(st + d0 / 2 + i) : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[2 * i] = -f[2 * i + 1] * s[i];
          p[2 * i + 1] = f[2 * i] * s[i];
          f[2 * i] *= c[i];
          f[2 * i + 1] *= c[i];
        }
      } else {
        const bool first = d0 < half;
        float c[8], s[8], pg[8];
        if (LAYOUT == 2 && a.tvec) {   // the chunk lies in one half
          const int j = first ? d0 : d0 - half;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const float4 cv = __ldg(reinterpret_cast<const float4*>(ct + j) + v);
            const float4 sv = __ldg(reinterpret_cast<const float4*>(st + j) + v);
            c[4 * v] = cv.x; c[4 * v + 1] = cv.y; c[4 * v + 2] = cv.z; c[4 * v + 3] = cv.w;
            s[4 * v] = sv.x; s[4 * v + 1] = sv.y; s[4 * v + 2] = sv.z; s[4 * v + 3] = sv.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int d = d0 + i, j = d < half ? d : d - half;
            c[i] = d < a.rot ? __ldg(ct + j) : 1.f;
            s[i] = d < a.rot ? __ldg(st + j) : 0.f;
          }
        }
        if (!gam) {
#pragma unroll
          for (int i = 0; i < 8; ++i) pg[i] = 1.f;
        } else if (LAYOUT == 2) {
          const float4* pp = reinterpret_cast<const float4*>(gam + (first ? d0 + half : d0 - half));
          const float4 lo = __ldg(pp), hi = __ldg(pp + 1);
          pg[0] = lo.x; pg[1] = lo.y; pg[2] = lo.z; pg[3] = lo.w;
          pg[4] = hi.x; pg[5] = hi.y; pg[6] = hi.z; pg[7] = hi.w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int d = d0 + i;
            pg[i] = d < a.rot ? __ldg(gam + (d < half ? d + half : d - half)) : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = pg[i] * (d0 + i < half ? -s[i] : s[i]);
          f[i] *= c[i];
        }
      }
    }
  }
  // partner chunk of LAYOUT 2: lane +- half/8; lanes past rot keep their own
  [[maybe_unused]] const int src = d0 < half ? lane + half / 8 : (d0 < a.rot ? lane - half / 8 : lane);
  // all of this lane's elements turn (lanes past the head: no matter)
  const bool whole = d0 + 8 <= a.rot || d0 >= a.D;
  const float inv_d = 1.f / (float)a.D;

  // The groups of a warp may belong to queries and to keys and so leave this loop
  // at different turns; the shuffles name the whole warp all the same, which holds
  // because a lane that leaves the loop leaves the kernel: nothing may come after it.
  for (int hb = 0; hb < a.per_unit[which]; hb += kQkHeads) {
    load(next, hb + kQkHeads);   // of other heads: nothing that is written before it is read
    // partners from memory (LAYOUT 3): all of them before any store
    [[maybe_unused]] uint32_t part[LAYOUT == 3 ? kQkHeads : 1][4];
    if constexpr (LAYOUT == 3) {
#pragma unroll
      for (int h = 0; h < kQkHeads; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          T e[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int d = d0 + 2 * i + k;
            e[k] = DT<T>::from_f(0.f);
            if (on && hb + h < nh && d < a.rot) e[k] = x[(hb + h) * xh + 2 * i + k + (d < half ? half : -half)];
          }
          memcpy(&part[h][i], e, 4);
        }
      __syncwarp();
    }
    float v[kQkHeads][8], ss[kQkHeads];
#pragma unroll
    for (int h = 0; h < kQkHeads; ++h) {
      const uint32_t w[4] = {raw[h].x, raw[h].y, raw[h].z, raw[h].w};
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = unpack2<T>(w[i]);
        v[h][2 * i] = t.x;
        v[h][2 * i + 1] = t.y;
        sum.x = fmaf(t.x, t.x, sum.x);
        sum.y = fmaf(t.y, t.y, sum.y);
      }
      ss[h] = sum.x + sum.y;
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
      for (int h = 0; h < kQkHeads; ++h) ss[h] += __shfl_xor_sync(0xffffffffu, ss[h], o);

#pragma unroll
    for (int h = 0; h < kQkHeads; ++h) {
      const float r = rsqrtf(fmaf(ss[h], inv_d, a.eps));
      [[maybe_unused]] uint32_t pr[4] = {0u, 0u, 0u, 0u};
      if constexpr (LAYOUT == 2) {
        pr[0] = __shfl_sync(0xffffffffu, raw[h].x, src, LANES);
        pr[1] = __shfl_sync(0xffffffffu, raw[h].y, src, LANES);
        pr[2] = __shfl_sync(0xffffffffu, raw[h].z, src, LANES);
        pr[3] = __shfl_sync(0xffffffffu, raw[h].w, src, LANES);
      } else if constexpr (LAYOUT == 3) {
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = part[h][i];
      }
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        float2 w = make_float2(0.f, 0.f);
        if constexpr (LAYOUT == 1) w = make_float2(v[h][i + 1], v[h][i]);
        else if constexpr (LAYOUT >= 2) w = unpack2<T>(pr[i / 2]);
        o[i] = v[h][i] * f[i];
        o[i + 1] = v[h][i + 1] * f[i + 1];
        if constexpr (LAYOUT != 0) {
          // an element past rot takes nothing from its neighbours, not even NaN
          if (whole || d0 + i < a.rot) o[i] = fmaf(w.x, p[i], o[i]);
          if (whole || d0 + i + 1 < a.rot) o[i + 1] = fmaf(w.y, p[i + 1], o[i + 1]);
        }
      }
      if (on && hb + h < nh) {
        uint4 w;
        w.x = pack16<T>(o[0] * r, o[1] * r);
        w.y = pack16<T>(o[2] * r, o[3] * r);
        w.z = pack16<T>(o[4] * r, o[5] * r);
        w.w = pack16<T>(o[6] * r, o[7] * r);
        *reinterpret_cast<uint4*>(y + (hb + h) * yh) = w;
      }
    }
#pragma unroll
    for (int h = 0; h < kQkHeads; ++h) raw[h] = next[h];
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
  const unsigned per_block = kQkThreads / lanes;
  const unsigned blocks = (a.total + per_block - 1) / per_block;
  switch (lanes) {
    case 4: return launch_qk_l<T, 4>(a, layout, blocks, st);
    case 8: return launch_qk_l<T, 8>(a, layout, blocks, st);
    case 16: return launch_qk_l<T, 16>(a, layout, blocks, st);
    default: return launch_qk_l<T, 32>(a, layout, blocks, st);
  }
}

// Heads of a token in a group of lanes: 16, which reads a table row once for 16
// heads, as long as that gives every SM its three CTAs twice or more; fewer for fewer
// tokens (one token of 32 + 8 heads: a head each).  Shared evenly over the
// groups.
static void qk_units(QkArgs& a) {
  int lanes = 4;
  while (lanes * 8 < a.D) lanes *= 2;
  const int64_t want = (int64_t)num_sms() * 8 * (kQkThreads / lanes);
  int most = 16;
  while (most > 1 && a.B * a.Lq * ((a.heads[0] + most - 1) / most + (a.heads[1] + most - 1) / most) < want) most /= 2;
  for (int i = 0; i < 2; ++i) {
    const int units = (a.heads[i] + most - 1) / most;
    a.per_unit[i] = units ? (a.heads[i] + units - 1) / units : 1;
    a.units[i] = (a.heads[i] + a.per_unit[i] - 1) / a.per_unit[i];
  }
  a.total = (unsigned)(a.B * a.Lq * (a.units[0] + a.units[1]));
  a.tvec = (a.rot / 2) % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.cosp) | reinterpret_cast<uintptr_t>(a.sinp)) & 15) == 0;
}

// layout: 0 interleaved, 1 half (rot 0: none)
cudaError_t launch_qk_norm_rope(QkArgs a, int dtype, int layout, cudaStream_t st) {
  if (a.B == 0 || a.Lq == 0 || a.heads[0] + a.heads[1] == 0) return cudaSuccess;
  qk_units(a);
  const int form = a.rot == 0 ? 0 : layout == 0 ? 1 : (a.rot / 2) % 8 == 0 ? 2 : 3;
  return dtype == IC_DTYPE_BF16 ? launch_qk_t<__nv_bfloat16>(a, form, st) : launch_qk_t<__half>(a, form, st);
}

}  // namespace ic
