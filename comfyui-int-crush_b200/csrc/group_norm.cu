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
  const void *gamma, *beta;
  int gamma_dtype, beta_dtype;
  float eps;
  int act;
  void* y;
  long long y_batch, y_row;
  uint8_t* q;               // e4m3 rows [B L, ldq], or null
  long long ldq;
  float* s;
  long long s_row, s_block;
  int width;                // C rounded up to 16
  long long chunk;          // rows of a CTA
  int cluster;              // CTAs of a cluster
  int runs;                 // clusters of a sample
  long long span;           // rows of a cluster
  float2* part;             // [B, runs, G] mean, M2
};

template <typename T> struct Gn8 {
  uint4 w;
  // channels [0, n) of p; all 8 in one load where `vec`
  __device__ __forceinline__ void load(const T* p, int n, bool vec) {
    if (vec) {
      w = *reinterpret_cast<const uint4*>(p);
    } else {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? u[i] : 0;
      w = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    }
  }
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

__device__ __forceinline__ float gn_act(float y, int act) {
  if (act == 1) return __fdividef(y, 1.f + __expf(-y));
  if (act == 2) return 0.5f * y * (1.f + erff(y * 0.70710678f));
  if (act == 3) return 0.5f * y * (1.f + tanhf(0.79788456f * (y + 0.044715f * y * y * y)));
  return y;
}

// Rows [lo, hi) of a CTA; n rows fall to slot i of `slots`.
__device__ __forceinline__ long long gn_slot_rows(long long rows, int slot, int slots) {
  return (rows - slot + slots - 1) / slots;
}

// mean and M2 of one group from n entries, by one warp in a fixed order;
// all lanes get the result.  at(i, count, mean, m2) reads entry i.  Means are
// summed as differences from the first one's: of a mean far from 0 only its
// own rounding is lost.
template <typename F>
__device__ __forceinline__ float2 gn_join(int n, float total, F at) {
  const int lane = threadIdx.x & 31;
  float sum = 0.f, count, ref, m2;
  at(0, count, ref, m2);
  for (int i = lane; i < n; i += 32) {
    float mean;
    at(i, count, mean, m2);
    sum = fmaf(count, mean - ref, sum);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  const float all = ref + sum / total;
  float dev = 0.f;
  for (int i = lane; i < n; i += 32) {
    float mean;
    at(i, count, mean, m2);
    const float d = mean - all;
    dev += fmaf(count * d, d, m2);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) dev += __shfl_xor_sync(0xffffffffu, dev, d);
  return make_float2(all, dev);
}

// A thread's factors: mean, rstd gamma and beta of its 8 channels.
struct GnFactors {
  float mean[8], a[8], b[8];
  __device__ __forceinline__ void load(const GnArgs& g, const float2* fin, int c0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + i;
      mean[i] = a[i] = b[i] = 0.f;
      if (c < g.C) {
        const float2 f = fin[c / g.Cg];
        mean[i] = f.x;
        a[i] = f.y * (g.gamma ? load_any(g.gamma, g.gamma_dtype, c) : 1.f);
        if (g.beta) b[i] = load_any(g.beta, g.beta_dtype, c);
      }
    }
  }
};

// Norm, activation and output of 8 channels of row l of sample b.  For e4m3 the
// 16 threads of a block of 128 channels (half a warp) come here together.
template <typename T, bool F8>
__device__ __forceinline__ void gn_finish(const GnArgs& g, const GnFactors& f, const Gn8<T>& in, long long b, long long l,
                                          int v) {
  float y[8];
  in.get(y);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = gn_act(fmaf(y[i] - f.mean[i], f.a[i], f.b[i]), g.act);
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

// Statistics of a cluster's rows (`KEEP`: the whole sample, kept in shared memory
// and normalised; else into the workspace).
template <typename T, bool KEEP, bool F8>
__global__ void __launch_bounds__(kGnThreads, KEEP ? 1 : 2) gn_stats_kernel(const GnArgs g) {
  extern __shared__ __align__(1024) uint8_t smem[];
  float2* sums = reinterpret_cast<float2*>(smem);                 // [slots, 8 cols]
  float2* own = sums + (size_t)g.slots * g.cols * 8;              // [G] this CTA's
  float2* fin = own + g.G;                                        // [G] mean, rstd (KEEP)
  uint4* kept = reinterpret_cast<uint4*>(smem + ((((size_t)g.slots * g.cols * 8 + 2 * (size_t)g.G) * 8 + 15) & ~(size_t)15));
  if (!KEEP) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int rank = (int)cluster_ctarank();
  const long long unit = blockIdx.x / g.cluster;
  const long long b = unit / g.runs, run = unit - b * g.runs;
  const long long lo = min(g.L, run * g.span + rank * g.chunk), hi = min(g.L, lo + g.chunk);
  const int slot = t / g.cols, col = t - slot * g.cols;
  const T* x = reinterpret_cast<const T*>(g.x) + b * g.x_batch;
  const int wide = g.slots == 1 ? kGnThreads : g.cols;   // columns a pass
  if (slot < g.slots || g.slots == 1) {
    const int v0 = g.slots == 1 ? t : col, s0 = g.slots == 1 ? 0 : slot;
    for (int v = v0; v < g.cols; v += wide) {
      const int n = g.C - 8 * v;   // <= 0: a column that only fills up a block
      float x0[8], s[8], q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x0[i] = s[i] = q[i] = 0.f;
      if (n > 0) {
        const T* p = x + 8 * v;
        const auto one = [&](const Gn8<T>& in) {
          float f[8];
          in.get(f);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float d = f[i] - x0[i];
            s[i] += d;
            q[i] = fmaf(d, d, q[i]);
          }
        };
        long long l = lo + s0;
        uint4* keep = kept + (size_t)s0 * g.cols + v;
        const size_t keep_step = (size_t)g.slots * g.cols;
        if (l < hi) {
          Gn8<T> in;
          in.load(p + l * g.x_row, n, g.vec != 0);
          in.get(x0);
        }
        constexpr int U = 4;
        for (; l + (U - 1) * g.slots < hi; l += U * g.slots) {
          Gn8<T> in[U];
#pragma unroll
          for (int i = 0; i < U; ++i) in[i].load(p + (l + i * g.slots) * g.x_row, n, g.vec != 0);
#pragma unroll
          for (int i = 0; i < U; ++i) {
            if (KEEP) { *keep = in[i].w; keep += keep_step; }
            one(in[i]);
          }
        }
        for (; l < hi; l += g.slots) {
          Gn8<T> in;
          in.load(p + l * g.x_row, n, g.vec != 0);
          if (KEEP) { *keep = in.w; keep += keep_step; }
          one(in);
        }
        const float rows = (float)gn_slot_rows(hi - lo, s0, g.slots);
        const float inv = rows > 0.f ? 1.f / rows : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n) sums[(size_t)s0 * g.cols * 8 + 8 * v + i] = make_float2(fmaf(s[i], inv, x0[i]), fmaxf(0.f, q[i] - s[i] * s[i] * inv));
      }
    }
  }
  __syncthreads();
  const float rows = (float)(hi - lo);
  for (int i = warp; i < g.G; i += kGnThreads / 32) {
    const float2 r = gn_join(g.Cg * g.slots, fmaxf(rows, 1.f) * (float)g.Cg, [&](int j, float& count, float& mean, float& m2) {
      const int sl = j / g.Cg;
      const float2 v = sums[(size_t)sl * g.cols * 8 + i * g.Cg + (j - sl * g.Cg)];
      count = (float)gn_slot_rows(hi - lo, sl, g.slots);
      mean = v.x;
      m2 = v.y;
    });
    if (lane == 0) own[i] = r;
  }
  cluster_sync_all();
  // the cluster's CTAs in rank order
  const long long run_lo = run * g.span;
  if (KEEP || rank == 0) {
    for (int i = t; i < g.G; i += kGnThreads) {
      const auto of = [&](int p, float& count, float2& v) {
        const long long a = min(g.L, run_lo + p * g.chunk);
        count = (float)(min(g.L, a + g.chunk) - a) * (float)g.Cg;
        const uint32_t at = mapa_u32(smem_u32(own + i), p);
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
      };
      float total = 0.f, sum = 0.f, ref = 0.f;
      for (int p = 0; p < g.cluster; ++p) {
        float count;
        float2 v;
        of(p, count, v);
        if (p == 0) ref = v.x;
        total += count;
        sum = fmaf(count, v.x - ref, sum);
      }
      const float mean = ref + sum / total;
      float m2 = 0.f;
      for (int p = 0; p < g.cluster; ++p) {
        float count;
        float2 v;
        of(p, count, v);
        const float d = v.x - mean;
        m2 += fmaf(count * d, d, v.y);
      }
      if (KEEP) fin[i] = make_float2(mean, 1.f / sqrtf(m2 / total + g.eps));
      else g.part[(b * g.runs + run) * g.G + i] = make_float2(mean, m2);
    }
  }
  if (KEEP) {
    __syncthreads();
    if (slot < g.slots || g.slots == 1) {
      const int v0 = g.slots == 1 ? t : col, s0 = g.slots == 1 ? 0 : slot;
      for (int v = v0; v < g.cols; v += wide) {
        GnFactors f;
        f.load(g, fin, 8 * v);
        const bool in_row = 8 * v < g.C;
        if (!F8 && !in_row) continue;
        const uint4* keep = kept + (size_t)s0 * g.cols + v;
        for (long long l = lo + s0; l < hi; l += g.slots, keep += (size_t)g.slots * g.cols) {
          Gn8<T> in;
          in.w = in_row ? *keep : make_uint4(0, 0, 0, 0);
          gn_finish<T, F8>(g, f, in, b, l, v);
        }
      }
    }
  }
  cluster_sync_all();   // nobody leaves while another CTA may read its shared memory
}

// The norm from the workspace's statistics.
template <typename T, bool F8>
__global__ void __launch_bounds__(kGnThreads, 2) gn_apply_kernel(const GnArgs g) {
  extern __shared__ __align__(1024) uint8_t smem[];
  float2* fin = reinterpret_cast<float2*>(smem);   // [G] mean, rstd
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const long long unit = gridDim.x - 1 - blockIdx.x;   // from the end
  const long long per = (g.L + g.chunk - 1) / g.chunk;
  const long long b = unit / per, lo = (unit - b * per) * g.chunk, hi = min(g.L, lo + g.chunk);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = warp; i < g.G; i += kGnThreads / 32) {
    const float total = (float)g.L * (float)g.Cg;
    const float2 r = gn_join(g.runs, total, [&](int j, float& count, float& mean, float& m2) {
      const float2 v = __ldcg(g.part + (b * g.runs + j) * g.G + i);
      const long long a = min(g.L, j * g.span);
      count = (float)(min(g.L, a + g.span) - a) * (float)g.Cg;
      mean = v.x;
      m2 = v.y;
    });
    if (lane == 0) fin[i] = make_float2(r.x, 1.f / sqrtf(r.y / total + g.eps));
  }
  __syncthreads();
  const int slot = t / g.cols, col = t - slot * g.cols;
  if (!(slot < g.slots || g.slots == 1)) return;
  const int wide = g.slots == 1 ? kGnThreads : g.cols;
  const int v0 = g.slots == 1 ? t : col, s0 = g.slots == 1 ? 0 : slot;
  const T* x = reinterpret_cast<const T*>(g.x) + b * g.x_batch;
  for (int v = v0; v < g.cols; v += wide) {
    GnFactors f;
    f.load(g, fin, 8 * v);
    const int n = g.C - 8 * v;
    if (!F8 && n <= 0) continue;
    const T* p = x + 8 * v;
    long long l = lo + s0;
    constexpr int U = 4;
    for (; l < hi; l += U * g.slots) {
      Gn8<T> in[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        in[i].w = make_uint4(0, 0, 0, 0);
        if (n > 0 && l + i * g.slots < hi) in[i].load(p + (l + i * g.slots) * g.x_row, n, g.vec != 0);
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (l + i * g.slots < hi) gn_finish<T, F8>(g, f, in[i], b, l + i * g.slots, v);
    }
  }
}

// ============================================================== host side

constexpr int kGnCluster = 8;
constexpr int kGnShared = 200 * 1024;

struct GnPlan {
  int cols, slots, cluster, runs;
  long long chunk;           // rows of a CTA of the first launch
  long long apply_chunk;     // of the second, 0: there is none
  int shared, apply_shared;
  long long floats;          // workspace
};

static GnPlan gn_plan(long long B, long long L, long long C, long long G, bool f8) {
  GnPlan p;
  p.cols = (int)((C + 7) / 8);
  if (f8) p.cols = (p.cols + 15) / 16 * 16;
  p.slots = p.cols <= kGnThreads ? kGnThreads / p.cols : 1;
  const long long head = (((long long)p.slots * p.cols * 8 + 2 * G) * 8 + 15) / 16 * 16;
  const long long row = (long long)p.cols * 16;
  // one launch: as few CTAs as keep a sample, but several where it has rows for them
  const long long most = (kGnShared - head) / row;   // rows of a CTA
  if (most > 0 && L <= most * kGnCluster) {
    p.cluster = 1;
    while (p.cluster < kGnCluster && (p.cluster * most < L || L >= 2 * p.cluster * (long long)p.slots)) p.cluster *= 2;
    p.chunk = (L + p.cluster - 1) / p.cluster;
    p.runs = 1;
    p.shared = (int)(head + p.chunk * row);
    p.apply_chunk = 0;
    p.apply_shared = 0;
    p.floats = 0;
    return p;
  }
  const long long ctas = 2LL * num_sms();
  p.cluster = kGnCluster;
  long long runs = ctas / kGnCluster / B;
  const long long useful = (L + 4LL * p.slots * kGnCluster - 1) / (4LL * p.slots * kGnCluster);   // 4 rows a thread at least
  runs = runs < useful ? runs : useful;
  p.runs = (int)(runs < 1 ? 1 : runs);
  p.chunk = ((L + p.runs - 1) / p.runs + p.cluster - 1) / p.cluster;
  p.shared = (int)head;
  p.apply_chunk = 8LL * p.slots;   // 8 rows a thread
  p.apply_shared = (int)(G * 8);
  p.floats = 2 * B * p.runs * G;
  return p;
}

template <typename T, bool F8>
static cudaError_t gn_launch(GnArgs a, const GnPlan& p, cudaStream_t st) {
  a.cols = p.cols;
  a.slots = p.slots;
  a.cluster = p.cluster;
  a.runs = p.runs;
  a.chunk = p.chunk;
  a.span = p.chunk * p.cluster;
  const bool keep = p.apply_chunk == 0;
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
  cudaError_t e = keep ? set_smem_once(gn_stats_kernel<T, true, F8>, 227 * 1024) : set_smem_once(gn_stats_kernel<T, false, false>, 227 * 1024);
  if (e != cudaSuccess) return e;
  e = keep ? cudaLaunchKernelEx(&cfg, gn_stats_kernel<T, true, F8>, a) : cudaLaunchKernelEx(&cfg, gn_stats_kernel<T, false, false>, a);
  if (e != cudaSuccess || keep) return e;
  a.chunk = p.apply_chunk;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)(a.B * ((a.L + a.chunk - 1) / a.chunk)));
  cfg.dynamicSmemBytes = p.apply_shared;
  e = set_smem_once(gn_apply_kernel<T, F8>, 227 * 1024);
  if (e != cudaSuccess) return e;
  return cudaLaunchKernelEx(&cfg, gn_apply_kernel<T, F8>, a);
}

cudaError_t launch_group_norm(const GnArgs& a, const GnPlan& p, int dtype, cudaStream_t st) {
  if (dtype == IC_DTYPE_F16) return a.q ? gn_launch<__half, true>(a, p, st) : gn_launch<__half, false>(a, p, st);
  return a.q ? gn_launch<__nv_bfloat16, true>(a, p, st) : gn_launch<__nv_bfloat16, false>(a, p, st);
}

}  // namespace ic
