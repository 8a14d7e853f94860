// Group norm with an activation, channels last: x [B, L, C], a group of a sample
// is C / G neighbouring channels of all its L rows.
//   y = act((x - mean) / sqrt(var + eps) * gamma + beta), var biased
// in fp32, rounded once: to x's type, or to e4m3 with a scale for each block of
// 128 channels of a row (quant_fp8.cu).
//
// Every thread keeps 8 neighbouring channels (16 bytes) of rows that are a fixed
// step apart, and for each channel the sums of x - x0 and (x - x0)^2 with x0 the
// first value it sees (no cancellation where the mean is far from 0).  They
// become mean and sum of squared deviations, and those of several channels,
// threads, CTAs and clusters are joined as
//   mean = sum n_i mean_i / N,  M2 = sum M2_i + n_i (mean_i - mean)^2
// in a fixed order.
//
// Two forms.  A sample that fits the shared memory of a cluster of up to 8 CTAs
// is read once: each CTA keeps its rows in shared memory while the statistics
// cross the cluster.  Others take two launches: statistics of runs of rows, a
// cluster's worth each, into a workspace, then the norm; the second walks
// the rows from the end, where L2 still holds them.
#include <type_traits>

namespace ic {

constexpr int kGnThreads = 512;

struct GnArgs {
  const void* x;
  long long L, x_batch, x_row;
  int B, C, G, Cg;
  int vec;                  // rows of x and y can be taken 16 bytes at a time
  int cols;                 // threads of a row: C / 8, rounded up to 16 for e4m3 blocks
  int slots;                // rows that a CTA holds side by side
  int sub;                  // channels of a thread that share a group: 1, 2, 4 or 8
  const void *gamma, *beta;
  int gamma_dtype, beta_dtype;
  float eps;
  void* y;
  long long y_batch, y_row;
  uint8_t* q;               // e4m3 rows [B L, ldq], or null
  long long ldq;
  float* s;
  long long s_row, s_block;
  int width;                // C rounded up to 16
  long long chunk;          // rows of a CTA
  int cluster, cluster_shift;   // CTAs of a cluster, a power of two
  int runs;                 // clusters of a sample
  long long span;           // rows of a cluster
  float2* part;             // [B, runs, G] mean, M2
};

constexpr int kGnRing = 8;   // rows of a thread on their way to shared memory

// 8 channels of a row to shared memory: one asynchronous 16-byte copy, or n
// values one by one.  Committed by gn_commit; only the thread that fetched reads them.
template <typename T>
__device__ __forceinline__ void gn_fetch(uint4* dst, const T* p, int n, bool vec) {
  if (vec) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(p) : "memory");
  } else {
    const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? u[i] : 0;
    *dst = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
}
__device__ __forceinline__ void gn_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void gn_arrived() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

template <typename T> struct Gn8 {
  uint4 w;
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[8], int n, bool vec) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if (vec) {
      *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
      unsigned short* o = reinterpret_cast<unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) o[i] = (unsigned short)(u[i / 2] >> (16 * (i & 1)));
    }
  }
};

template <int ACT>
__device__ __forceinline__ float gn_act(float y) {
  if (ACT == 1) return __fdividef(y, 1.f + __expf(-y));
  if (ACT == 2) return 0.5f * y * (1.f + erff(y * 0.70710678f));
  if (ACT == 3) return 0.5f * y * (1.f + tanhf(0.79788456f * (y + 0.044715f * y * y * y)));
  return y;
}

// Two equal counts n of a channel each, joined.
__device__ __forceinline__ void gn_pair(float& mean, float& m2, float mean2, float m22, float n) {
  const float d = mean2 - mean;
  mean = fmaf(0.5f, d, mean);
  m2 = fmaf(0.5f * n * d, d, m2 + m22);
}

// Sum over the warp, the same bits in all lanes.
__device__ __forceinline__ float gn_warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// A thread's factors: mean, rstd gamma and beta of its 8 channels.
struct GnFactors {
  float mean[8], a[8], b[8];
  // channels [c0, c0 + 8) of a vector of C
  static __device__ __forceinline__ void vector(float (&v)[8], const void* p, int dtype, int c0, int C, float none) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = none;
    if (!p) return;
    if (dtype != IC_DTYPE_F32 && c0 + 8 <= C && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned short*>(p) + c0);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t h = i & 1 ? u[i / 2] >> 16 : u[i / 2] & 0xffffu;
        v[i] = dtype == IC_DTYPE_F16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < C) v[i] = load_any(p, dtype, c0 + i);
  }
  __device__ __forceinline__ void load(const GnArgs& g, const float2* fin, int c0) {
    vector(a, g.gamma, g.gamma_dtype, c0, g.C, 1.f);
    vector(b, g.beta, g.beta_dtype, c0, g.C, 0.f);
    int group = c0 / g.Cg, left = (group + 1) * g.Cg - c0;   // channels up to the next group
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = fin[min(group, g.G - 1)];
      mean[i] = f.x;
      a[i] *= f.y;
      if (--left == 0) {
        ++group;
        left = g.Cg;
      }
    }
  }
};

// Norm, activation and output of 8 channels of row l of sample b.  For e4m3 the
// 16 threads of a block of 128 channels (half a warp) come here together.
template <typename T, bool F8, int ACT>
__device__ __forceinline__ void gn_finish(const GnArgs& g, const GnFactors& f, const Gn8<T>& in, long long b, long long l,
                                          int v) {
  float y[8];
  in.get(y);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = gn_act<ACT>(fmaf(y[i] - f.mean[i], f.a[i], f.b[i]));
  if constexpr (!F8) {
    Gn8<T>::store(reinterpret_cast<T*>(g.y) + b * g.y_batch + l * g.y_row + 8 * v, y, g.C - 8 * v, g.vec != 0);
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (8 * v + i >= g.C) y[i] = 0.f;
      top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
    }
    const uint32_t half = 0xffffu << (threadIdx.x & 16);
#pragma unroll
    for (int d = 8; d; d >>= 1) top = max(top, __shfl_xor_sync(half, top, d));
    const F8Scale sc = f8_scale(__uint_as_float(top));
    const long long row = b * g.L + l;
    uint2 o;
    if (sc.s <= 3.4e38f) {
      o = make_uint2(f8_four(y[0], y[1], y[2], y[3], sc), f8_four(y[4], y[5], y[6], y[7], sc));
    } else {
      o = make_uint2(f8_four_div(y[0], y[1], y[2], y[3], sc.s), f8_four_div(y[4], y[5], y[6], y[7], sc.s));
    }
    if (8 * v < g.width) *reinterpret_cast<uint2*>(g.q + row * g.ldq + 8 * v) = o;
    if ((v & 15) == 0 && 8 * v < g.C) g.s[row * g.s_row + (v >> 4) * g.s_block] = sc.s;
  }
}

// Where a CTA works: its sample, rows and threads.
struct GnPlace {
  int b, run, rank, s0, v0, wide;
  long long lo, hi;
  bool busy;
  __device__ __forceinline__ GnPlace(const GnArgs& g) {
    const int t = threadIdx.x, unit = (int)blockIdx.x >> g.cluster_shift;
    rank = (int)blockIdx.x - (unit << g.cluster_shift);
    b = unit / g.runs;
    run = unit - b * g.runs;
    lo = min(g.L, run * g.span + rank * g.chunk);
    hi = min(g.L, lo + g.chunk);
    wide = g.slots == 1 ? kGnThreads : g.cols;   // columns a pass
    s0 = g.slots == 1 ? 0 : t / g.cols;
    v0 = t - s0 * g.cols;
    busy = s0 < g.slots;
  }
};

// Statistics of a cluster's rows (`KEEP`: the whole sample, kept in shared memory
// and normalised; else into the workspace).
template <typename T, bool KEEP, bool F8, int ACT>
__global__ void __launch_bounds__(kGnThreads, KEEP ? 1 : 2) gn_stats_kernel(const GnArgs g) {
  extern __shared__ __align__(1024) uint8_t smem[];
  // the norm's launch may begin, its CTAs wait for the statistics themselves
  if (!KEEP) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int shift = 31 - __clz(g.sub), per = 8 >> shift;          // entries of a thread
  const int width = g.cols * per;                                 // of a slot
  float2* sums = reinterpret_cast<float2*>(smem);                 // [slots, width]
  float2* own = sums + g.slots * width;                           // [G] this CTA's
  float2* fin = own + g.G;                                        // [G] mean, rstd (KEEP)
  // KEEP: [chunk, cols], else [kGnRing, threads]
  uint4* kept = reinterpret_cast<uint4*>(smem + (((g.slots * width + (KEEP ? 2 : 1) * g.G) * 8 + 15) & ~15));
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const GnPlace at(g);
  const int rows = (int)(at.hi - at.lo);
  // slot i takes rows i, i + slots, ...: more of them the first `rest` slots
  const int least = rows / g.slots, rest = rows - least * g.slots;
  const int mine = at.busy ? least + (at.s0 < rest) : 0;          // this thread's rows
  const long long step = g.slots * g.x_row;
  const T* x = reinterpret_cast<const T*>(g.x) + at.b * g.x_batch + (at.lo + at.s0) * g.x_row;
  const int keep_step = KEEP ? g.slots * g.cols : kGnThreads;
  if (at.busy) {
    for (int v = at.v0; v < g.cols; v += at.wide) {
      const int n = g.C - 8 * v;   // <= 0: a column that only fills up a block
      if (n <= 0) continue;
      const T* p = x + 8 * v;
      uint4* keep = KEEP ? kept + at.s0 * g.cols + v : kept + t;
      if (KEEP) {   // all of them at once
        for (int r = 0; r < mine; ++r, p += step) gn_fetch(keep + r * keep_step, p, n, g.vec != 0);
        gn_commit();
        gn_arrived<0>();
      } else {
#pragma unroll
        for (int r = 0; r < kGnRing; ++r) {
          if (r < mine) gn_fetch(keep + r * keep_step, p, n, g.vec != 0);
          p += step;
          gn_commit();
        }
      }
      float x0[8], s[8], q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x0[i] = s[i] = q[i] = 0.f;
      for (int r0 = 0; r0 < mine; r0 += kGnRing) {
#pragma unroll
        for (int k = 0; k < kGnRing; ++k) {
          const int r = r0 + k;
          if (r < mine) {
            if (!KEEP) gn_arrived<kGnRing - 1>();
            Gn8<T> in;
            in.w = keep[(KEEP ? r : k) * keep_step];
            float f[8];
            in.get(f);
            if (r == 0) {
#pragma unroll
              for (int j = 0; j < 8; ++j) x0[j] = f[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float d = f[j] - x0[j];
              s[j] += d;
              q[j] = fmaf(d, d, q[j]);
            }
            if (!KEEP) {
              if (r + kGnRing < mine) gn_fetch(keep + k * keep_step, p, n, g.vec != 0);
              p += step;
              gn_commit();
            }
          }
        }
      }
      if (!KEEP) gn_arrived<0>();
      const float count = (float)mine, inv = mine ? 1.f / count : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[i] = fmaxf(0.f, q[i] - s[i] * s[i] * inv);
        s[i] = fmaf(s[i], inv, x0[i]);
      }
      // channels of one group, two by two
#pragma unroll
      for (int w = 1; w < 8; w *= 2)
        if (w < g.sub) {
#pragma unroll
          for (int i = 0; i < 8; i += 2 * w) gn_pair(s[i], q[i], s[i + w], q[i + w], count * w);
        }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((i & (g.sub - 1)) == 0 && i < n) sums[at.s0 * width + v * per + (i >> shift)] = make_float2(s[i], q[i]);
    }
  }
  __syncthreads();
  // a warp joins the entries of a group: from slot sl and column e on, 32 at a
  // time.  Means are summed as differences from the first one's: of a mean far
  // from 0 only its own rounding is lost.
  const int entries = g.Cg >> shift;   // of a group and slot
  const int dq = 32 / entries, dr = 32 - dq * entries, sl0 = lane / entries, e0 = lane - sl0 * entries;
  for (int i = warp; i < g.G; i += kGnThreads / 32) {
    const float2* from = sums + i * entries;
    const float ref = from[0].x, total = (float)max(rows, 1) * (float)g.Cg;
    float sum = 0.f, dev = 0.f;
    for (int sl = sl0, e = e0; sl < g.slots;) {
      sum = fmaf((float)((least + (sl < rest)) << shift), from[sl * width + e].x - ref, sum);
      sl += dq;
      e += dr;
      if (e >= entries) { e -= entries; ++sl; }
    }
    const float mean = ref + gn_warp_sum(sum) / total;
    for (int sl = sl0, e = e0; sl < g.slots;) {
      const float2 v = from[sl * width + e];
      const float d = v.x - mean;
      dev += fmaf((float)((least + (sl < rest)) << shift) * d, d, v.y);
      sl += dq;
      e += dr;
      if (e >= entries) { e -= entries; ++sl; }
    }
    dev = gn_warp_sum(dev);
    if (lane == 0) own[i] = make_float2(mean, dev);
  }
  cluster_sync_all();
  // the cluster's CTAs, a lane each
  if (KEEP || at.rank == 0) {
    const long long run_lo = at.run * g.span;
    const int p = lane & (g.cluster - 1);
    const long long first = min(g.L, run_lo + p * g.chunk);
    const float count = (float)(min(g.L, first + g.chunk) - first) * (float)g.Cg;
    const float total = (float)(min(g.L, run_lo + g.span) - run_lo) * (float)g.Cg;
    for (int i0 = 0; i0 < g.G; i0 += kGnThreads >> g.cluster_shift) {
      const int i = i0 + (t >> g.cluster_shift);
      float2 v;
      const uint32_t where = mapa_u32(smem_u32(own + min(i, g.G - 1)), p);
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(where) : "memory");
      const float ref = __shfl_sync(0xffffffffu, v.x, lane & ~(g.cluster - 1));
      float sum = count * (v.x - ref);
      for (int d = 1; d < g.cluster; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float mean = ref + sum / total, dev = v.x - mean;
      float m2 = fmaf(count * dev, dev, v.y);
      for (int d = 1; d < g.cluster; d *= 2) m2 += __shfl_xor_sync(0xffffffffu, m2, d);
      if (p == 0 && i < g.G) {
        if (KEEP) fin[i] = make_float2(mean, 1.f / sqrtf(m2 / total + g.eps));
        else g.part[((long long)at.b * g.runs + at.run) * g.G + i] = make_float2(mean, m2);
      }
    }
  }
  if (KEEP) {
    __syncthreads();
    if (at.busy) {
      for (int v = at.v0; v < g.cols; v += at.wide) {
        GnFactors f;
        f.load(g, fin, 8 * v);
        const bool in_row = 8 * v < g.C;
        if (!F8 && !in_row) continue;
        const uint4* keep = kept + at.s0 * g.cols + v;
        for (int r = 0; r < mine; ++r) {
          Gn8<T> in;
          in.w = in_row ? keep[r * keep_step] : make_uint4(0, 0, 0, 0);
          gn_finish<T, F8, ACT>(g, f, in, at.b, at.lo + at.s0 + r * g.slots, v);
        }
      }
    }
  }
  cluster_sync_all();   // nobody leaves while another CTA may read its shared memory
}

// The norm from the workspace's statistics, with the first launch's shares of the
// rows, each from its end.
template <typename T, bool F8, int ACT>
__global__ void __launch_bounds__(kGnThreads, 2) gn_apply_kernel(const GnArgs g) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;          // [kGnRing, threads]
  float2* fin = reinterpret_cast<float2*>(smem + kGnRing * kGnThreads * 16);   // [G] mean, rstd
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const GnPlace at(g);
  const int rows = (int)(at.hi - at.lo) - at.s0;
  const int mine = at.busy && rows > 0 ? (rows + g.slots - 1) / g.slots : 0;   // this thread's rows
  const long long step = g.slots * g.x_row;
  const T* x = reinterpret_cast<const T*>(g.x) + at.b * g.x_batch + (at.hi - 1 - at.s0) * g.x_row;
  const auto begin = [&](int v) {
    const T* p = x + 8 * v;
#pragma unroll
    for (int r = 0; r < kGnRing; ++r) {
      if (r < mine && 8 * v < g.C) gn_fetch(ring + r * kGnThreads, p, g.C - 8 * v, g.vec != 0);
      p -= step;
      gn_commit();
    }
  };
  if (at.v0 < g.cols) begin(at.v0);   // x is no output of the first launch
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float total = (float)g.L * (float)g.Cg;
  const float2* part = g.part + (long long)at.b * g.runs * g.G;
  for (int i = warp; i < g.G; i += kGnThreads / 32) {
    // two runs a lane at most (kGnRuns)
    float2 v[2];
    float count[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = lane + 32 * k;
      const long long a = min(g.L, j * g.span);
      v[k] = __ldcg(part + min(j, g.runs - 1) * g.G + i);
      count[k] = j < g.runs ? (float)(min(g.L, a + g.span) - a) * (float)g.Cg : 0.f;
    }
    const float ref = __shfl_sync(0xffffffffu, v[0].x, 0);
    const float mean = ref + gn_warp_sum(fmaf(count[0], v[0].x - ref, count[1] * (v[1].x - ref))) / total;
    float dev = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float d = v[k].x - mean;
      dev += count[k] > 0.f ? fmaf(count[k] * d, d, v[k].y) : 0.f;
    }
    dev = gn_warp_sum(dev);
    if (lane == 0) fin[i] = make_float2(mean, 1.f / sqrtf(dev / total + g.eps));
  }
  __syncthreads();
  for (int v = at.v0; v < g.cols; v += at.wide) {
    if (v != at.v0) begin(v);
    GnFactors f;
    f.load(g, fin, 8 * v);
    const int n = g.C - 8 * v;
    const T* p = x + 8 * v - kGnRing * step;
    long long l = at.hi - 1 - at.s0;
    for (int r0 = 0; r0 < mine; r0 += kGnRing) {
#pragma unroll 2
      for (int k = 0; k < kGnRing; ++k) {
        const int r = r0 + k;
        if (r < mine) {
          gn_arrived<kGnRing - 1>();
          Gn8<T> in;
          in.w = n > 0 ? ring[k * kGnThreads] : make_uint4(0, 0, 0, 0);
          if (F8 || n > 0) gn_finish<T, F8, ACT>(g, f, in, at.b, l, v);
          if (r + kGnRing < mine && n > 0) gn_fetch(ring + k * kGnThreads, p, n, g.vec != 0);
          p -= step;
          l -= g.slots;
          gn_commit();
        }
      }
    }
    gn_arrived<0>();
  }
}

// ============================================================== host side

constexpr int kGnCluster = 8;
constexpr int kGnRuns = 64;        // of a sample, what the norm's warps join
constexpr int kGnShared = 200 * 1024;

struct GnPlan {
  int cols, slots, sub, cluster, runs;
  long long chunk;           // rows of a CTA of the first launch
  bool keep;                 // one launch
  int shared;
  long long floats;          // workspace
};

static GnPlan gn_plan(long long B, long long L, long long C, long long G, bool f8) {
  GnPlan p;
  p.cols = (int)((C + 7) / 8);
  if (f8) p.cols = (p.cols + 15) / 16 * 16;
  p.slots = p.cols <= kGnThreads ? kGnThreads / p.cols : 1;
  p.sub = 1;
  while (p.sub < 8 && C / G % (2 * p.sub) == 0) p.sub *= 2;
  const long long sums = (long long)p.slots * p.cols * (8 / p.sub);
  const long long head = ((sums + 2 * G) * 8 + 15) / 16 * 16;
  const long long row = (long long)p.cols * 16;
  // one launch: as few CTAs as keep a sample, but several where it has rows for them
  const long long most = (kGnShared - head) / row;   // rows of a CTA
  p.keep = most > 0 && L <= most * kGnCluster;
  if (p.keep) {
    p.cluster = 1;
    while (p.cluster < kGnCluster && (p.cluster * most < L || L >= 2 * p.cluster * (long long)p.slots)) p.cluster *= 2;
    p.chunk = (L + p.cluster - 1) / p.cluster;
    p.runs = 1;
    p.shared = (int)(head + p.chunk * row);
    p.floats = 0;
    return p;
  }
  const long long ctas = 2LL * num_sms();
  p.cluster = kGnCluster;
  long long runs = ctas / kGnCluster / B;
  const long long useful = (L + 4LL * p.slots * kGnCluster - 1) / (4LL * p.slots * kGnCluster);   // 4 rows a thread at least
  runs = runs < useful ? runs : useful;
  p.runs = (int)(runs < 1 ? 1 : runs > kGnRuns ? kGnRuns : runs);
  p.chunk = ((L + p.runs - 1) / p.runs + p.cluster - 1) / p.cluster;
  p.shared = (int)(((sums + G) * 8 + 15) / 16 * 16) + kGnRing * kGnThreads * 16;
  p.floats = 2 * B * p.runs * G;
  return p;
}

template <typename T, bool F8, int ACT>
static cudaError_t gn_launch(GnArgs a, const GnPlan& p, cudaStream_t st) {
  a.cols = p.cols;
  a.slots = p.slots;
  a.sub = p.sub;
  a.cluster = p.cluster;
  a.cluster_shift = 31 - __builtin_clz(p.cluster);
  a.runs = p.runs;
  a.chunk = p.chunk;
  a.span = p.chunk * p.cluster;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)((long long)a.B * p.runs * p.cluster));
  cfg.blockDim = dim3(kGnThreads);
  cfg.dynamicSmemBytes = p.shared;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (p.keep) {
    auto kern = gn_stats_kernel<T, true, F8, ACT>;
    cudaError_t e = set_smem_once(kern, 227 * 1024);
    return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, kern, a);
  }
  auto stats = gn_stats_kernel<T, false, false, 0>;
  auto apply = gn_apply_kernel<T, F8, ACT>;
  cudaError_t e = set_smem_once(stats, 227 * 1024);
  if (e == cudaSuccess) e = set_smem_once(apply, 227 * 1024);
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, stats, a);
  if (e != cudaSuccess) return e;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.dynamicSmemBytes = kGnRing * kGnThreads * 16 + a.G * 8;
  return cudaLaunchKernelEx(&cfg, apply, a);
}

template <typename T, bool F8>
static cudaError_t gn_launch_act(const GnArgs& a, const GnPlan& p, int act, cudaStream_t st) {
  if (act == 0) return gn_launch<T, F8, 0>(a, p, st);
  if (act == 1) return gn_launch<T, F8, 1>(a, p, st);
  if (act == 2) return gn_launch<T, F8, 2>(a, p, st);
  return gn_launch<T, F8, 3>(a, p, st);
}

cudaError_t launch_group_norm(const GnArgs& a, const GnPlan& p, int dtype, int act, cudaStream_t st) {
  if (dtype == IC_DTYPE_F16) return a.q ? gn_launch_act<__half, true>(a, p, act, st) : gn_launch_act<__half, false>(a, p, act, st);
  return a.q ? gn_launch_act<__nv_bfloat16, true>(a, p, act, st) : gn_launch_act<__nv_bfloat16, false>(a, p, act, st);
}

}  // namespace ic
