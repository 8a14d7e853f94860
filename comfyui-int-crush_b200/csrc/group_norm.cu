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
// Two forms.  What fits the shared memory of clusters of up to 16 CTAs is read
// once: each CTA keeps its rows in shared memory while the statistics cross the
// cluster; a sample's groups are dealt to several clusters (`parts`), as they have
// nothing to do with one another, until the SMs are busy.  Others take two
// launches: statistics of runs of rows, a cluster's worth each, into a
// workspace, then the norm; the second takes the rows from the end, which the first
// read last, so that L2 still holds some of them.
//
// 2 x 256 x 1280 with SiLU: 6.9 us, most of it code that runs once.  1024 x 1024 x 128
// with SiLU: 151 us, where 805 MB (x twice, y) at 6.55 TB/s are 123: the statistics
// take 48 us on average and 60 with the CTAs that read from far memory, the norm 78,
// at three quarters of the instruction slots and half of the special functions'.
#include <atomic>
#include <type_traits>

namespace ic {

constexpr int kGnThreads = 512;

struct GnArgs {
  const void* x;
  long long L, x_batch, x_row;
  int C, G, Cg;             // channels and groups of a part
  int parts;                // of a sample
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
  int cluster, cluster_shift;   // CTAs of a cluster, a power of two
  int runs;                 // clusters of a part
  // tiles of `tile` rows (all of a CTA's, or kGnRing a thread), dealt to a part's
  // CTAs in turn: `deal` each, the first `more` CTAs one more; the last tile lacks
  // `lack` rows
  int tile, deal, more, lack;
  float2* part;             // [B, parts, G, runs] mean, M2
  int* tiles;               // [B, parts] tiles that CTAs of the second launch have taken
};

// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t gn_two(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void gn_untwo(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t gn_add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t gn_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t gn_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t gn_neg2(uint64_t a) { return a ^ 0x8000000080000000ull; }

// the largest magnitude of three, a NaN (positive) if one is
__device__ __forceinline__ float gn_top3(float a, float b, float c) {
  float v;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}

constexpr int kGnRing = 8;   // rows of a thread on their way to shared memory
constexpr int kGnLaneRuns = 5;   // runs of a part that a lane of the second launch joins, at most

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

// 8 values of 16 bits as four pairs in fp32, and back
template <typename T>
__device__ __forceinline__ void gn_unpack(const uint4& w, uint64_t (&v)[4]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      v[i] = gn_two(f.x, f.y);
    } else {
      v[i] = gn_two(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    }
  }
}
template <typename T>
__device__ __forceinline__ void gn_store(T* p, const float (&v)[8], int n, bool vec) {
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

constexpr float kGnLog2e = 1.4426950408889634f;
__device__ __forceinline__ float gn_ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float gn_rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float gn_max_nan(float a, float b) {   // a NaN where one is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The activation of a thread's 8 values.  SiLU and GELU (tanh) are y / (1 + 2^z)
// (1 + tanh(u) = 2 / (1 + exp(-2 u))); where 2^z is too large for its reciprocal
// the quotient is a signed 0.
template <int ACT, bool F8>
__device__ __forceinline__ void gn_act8(float (&y)[8]) {
  if constexpr (ACT == 1 && !F8) {
    // SiLU to 16 bits: one reciprocal for two values (these functions run at a
    // quarter of the other instructions' rate; 1024 x 1024 x 128: 150.5 us, 156.8 with
    // a reciprocal each).  Denominators times 2^-63, so that the product of two
    // stays in range for y down to -86.6; values below count as that one, whose SiLU
    // is -2e-36.  The exponent's maximum drops a NaN, which would reach its
    // neighbour, the quotient's keeps it.
    constexpr float kLow = -86.6f, k = 1.0842021724855044e-19f;   // 2^-63
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float a = k + gn_ex2(fmaf(fmaxf(y[i], kLow), -kGnLog2e, -63.f));
      const float b = k + gn_ex2(fmaf(fmaxf(y[i + 1], kLow), -kGnLog2e, -63.f));
      const float r = gn_rcp(a * b);
      y[i] = gn_max_nan(y[i], kLow) * (r * b * k);
      y[i + 1] = gn_max_nan(y[i + 1], kLow) * (r * a * k);
    }
  } else if constexpr (ACT == 1 || ACT == 3) {
    // A reciprocal each: fewer instructions (300000 x 128 to e4m3 with SiLU: 66.5 us,
    // 70.3 with one for two; 1024 x 1024 x 128 with GELU (tanh): 161.7 and 172).
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float z = ACT == 1 ? y[i] * -kGnLog2e : -2.f * 0.7978845608028654f * kGnLog2e * fmaf(0.044715f * y[i], y[i] * y[i], y[i]);
      y[i] *= gn_rcp(1.f + gn_ex2(z));
    }
  } else if constexpr (ACT == 2) {
    // y Phi(y), Phi(-t) = exp(-t^2 / 2) P(u) for t >= 0 with u = 1 / (1 + 0.2325 t): the
    // form of Hastings' approximations of erfc ("Approximations for Digital
    // Computers", 1955), the polynomial fitted to exp(t^2 / 2) Phi(-t) for its largest
    // relative error, 9e-8 for t up to 13.3 (beyond, y Phi(y) is below the normal
    // numbers).  1 + erf(y / sqrt 2) loses all digits below -5.5, and erff takes
    // longer: 1024 x 1024 x 128 in 227 us, 188 like this, 322 with erfcf.
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = fabsf(y[i]), u = gn_rcp(fmaf(0.2325f, t, 1.f));
      float p = fmaf(-0.06954354047775269f, u, 0.24090537428855896f);
      p = fmaf(p, u, -0.19213353097438812f);
      p = fmaf(p, u, 0.21811789274215698f);
      p = fmaf(p, u, 0.01670587807893753f);
      p = fmaf(p, u, 0.10224095731973648f);
      p = fmaf(p, u, 0.09084631502628326f);
      p = fmaf(p, u, 0.09286066889762878f);
      p *= u * gn_ex2(t * t * (-0.5f * kGnLog2e));
      y[i] *= y[i] < 0.f ? p : 1.f - p;
    }
  }
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

// A thread's factors: -mean, rstd gamma and beta of its 8 channels, in pairs.
// (a x + b with b = beta - mean a would save an addition, but a constant group,
// whose rstd is large, would show b's rounding.)
struct GnFactors {
  uint64_t m[4], a[4], b[4];
  // channels [c0, c0 + 8) of a vector, n of them there
  static __device__ __forceinline__ void vector(float (&v)[8], const void* p, int dtype, int c0, int n, float none) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = none;
    if (!p) return;
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p) + c0;
    if (dtype != IC_DTYPE_F32 && n >= 8 && (reinterpret_cast<uintptr_t>(h) & 15) == 0) {
      const uint4 w = *reinterpret_cast<const uint4*>(h);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t e = i & 1 ? u[i / 2] >> 16 : u[i / 2] & 0xffffu;
        v[i] = dtype == IC_DTYPE_F16 ? __half2float(__ushort_as_half((unsigned short)e)) : __uint_as_float(e << 16);
      }
      return;
    }
#pragma unroll 1
    for (int i = 0; i < 8; ++i)
      if (i < n) {
        const float e = load_any(p, dtype, c0 + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = i == j ? e : v[j];
      }
  }
  // column v of the part that begins at channel c
  __device__ __forceinline__ void load(const GnArgs& g, const float2* fin, int c, int v) {
    float m_[8], a_[8], b_[8];
    vector(a_, g.gamma, g.gamma_dtype, c + 8 * v, g.C - 8 * v, 1.f);
    vector(b_, g.beta, g.beta_dtype, c + 8 * v, g.C - 8 * v, 0.f);
    int group = 8 * v / g.Cg, left = (group + 1) * g.Cg - 8 * v;   // channels up to the next group
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = fin[min(group, g.G - 1)];
      m_[i] = -f.x;
      a_[i] *= f.y;
      if (--left == 0) {
        ++group;
        left = g.Cg;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = gn_two(m_[2 * i], m_[2 * i + 1]);
      a[i] = gn_two(a_[2 * i], a_[2 * i + 1]);
      b[i] = gn_two(b_[2 * i], b_[2 * i + 1]);
    }
  }
};

// rows of CTA c of a part
__device__ __forceinline__ int gn_rows(const GnArgs& g, int c) {
  const int last = g.more ? g.more - 1 : (g.runs << g.cluster_shift) - 1;
  return (g.deal + (c < g.more)) * g.tile - (c == last ? g.lack : 0);
}
// of a cluster
__device__ __forceinline__ int gn_run_rows(const GnArgs& g, int run) {
  int n = 0;
  for (int i = 0; i < g.cluster; ++i) n += gn_rows(g, (run << g.cluster_shift) + i);
  return n;
}

// Where a CTA works: its sample, part and threads; c: its number in the part.
struct GnPlace {
  int b, part, run, rank, c, s0, v0, wide;
  bool busy;
  __device__ __forceinline__ GnPlace(const GnArgs& g) {
    const int t = threadIdx.x, unit = (int)blockIdx.x >> g.cluster_shift;
    rank = (int)blockIdx.x - (unit << g.cluster_shift);
    const int bp = unit / g.runs;
    run = unit - bp * g.runs;
    b = bp / g.parts;
    part = bp - b * g.parts;
    c = (run << g.cluster_shift) + rank;
    wide = g.slots == 1 ? kGnThreads : g.cols;   // columns a pass
    s0 = g.slots == 1 ? 0 : t / g.cols;
    v0 = t - s0 * g.cols;
    busy = s0 < g.slots;
  }
};

// Where a thread's column v of row l goes, and `rows` rows further on.
template <typename T, bool F8> struct GnOut {
  T* y;
  uint8_t* q;
  float* s;
  long long step, s_step;
  __device__ __forceinline__ GnOut(const GnArgs& g, const GnPlace& at, long long l, int v, int rows) {
    const int c = at.part * g.C + 8 * v;
    if (F8) {
      const long long row = at.b * g.L + l;
      q = g.q + row * g.ldq + c;
      s = g.s + row * g.s_row + (c >> 7) * g.s_block;
      step = rows * g.ldq;
      s_step = rows * g.s_row;
    } else {
      y = reinterpret_cast<T*>(g.y) + at.b * g.y_batch + l * g.y_row + c;
      step = rows * g.y_row;
    }
  }
  __device__ __forceinline__ void next() {
    if (F8) {
      q += step;
      s += s_step;
    } else {
      y += step;
    }
  }
};

// Norm, activation and output of 8 channels of a row.  For e4m3 the 16 threads of
// a block of 128 channels (half a warp) come here together.
template <typename T, bool F8, int ACT>
__device__ __forceinline__ void gn_finish(const GnArgs& g, const GnFactors& f, const uint4& in, const GnOut<T, F8>& o, int v) {
  uint64_t x[4];
  gn_unpack<T>(in, x);
  float y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) gn_untwo(gn_fma2(gn_add2(x[i], f.m[i]), f.a[i], f.b[i]), y[2 * i], y[2 * i + 1]);
  gn_act8<ACT, F8>(y);
  const int n = g.C - 8 * v;
  if constexpr (!F8) {
    gn_store(o.y, y, n, g.vec != 0);
  } else {
    // Scale and quotients as they are defined (quant_fp8.cu), the quotients from a
    // reciprocal to a unit (300000 x 128 with SiLU: 66.5 us, 65.7 without their
    // correction, 71.9 a value at a time).  A scale that is infinite has 0 for its
    // reciprocal, a NaN a NaN; both correct against 0, so that the block's finite
    // values become 0, or NaN.  (y = -0 becomes +0: its sign would cost 1%.)
    if (n < 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = i < n ? y[i] : 0.f;
    }
    const float top = gn_top3(gn_top3(gn_top3(y[0], y[1], y[2]), y[3], y[4]), gn_top3(y[5], y[6], y[7]), 0.f);
    const float amax = __uint_as_float(__reduce_max_sync(0xffffu << (threadIdx.x & 16), __float_as_uint(top)));
    const F8Scale of448 = {kF8Max, 1.f / kF8Max};
    const float s = amax <= 3.4028235e38f ? f8_quotient(fmaxf(amax, kF8AmaxMin), of448) : amax;
    float inv = gn_rcp(s);
    if (inv > 0.f) inv = fmaf(inv, fmaf(-s, inv, 1.f), inv);   // (a NaN stays, a 0 too)
    const float minus = inv > 0.f ? -s : 0.f;
    const uint64_t by = gn_two(inv, inv), less = gn_two(minus, minus);
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t z = gn_two(y[2 * i], y[2 * i + 1]), r = gn_mul2(z, by);
      float lo, hi;
      gn_untwo(gn_fma2(gn_fma2(r, less, z), by, r), lo, hi);
      p[i] = f8_pair(lo, hi);
    }
    const uint2 w = make_uint2(p[0] | p[1] << 16, p[2] | p[3] << 16);
    if (8 * v < g.width) *reinterpret_cast<uint2*>(o.q) = w;
    if ((v & 15) == 0 && n > 0) *o.s = s;
  }
}

// Statistics of a cluster's rows (`KEEP`: all rows of a part, kept in shared memory
// and normalised; else into the workspace).
template <typename T, bool KEEP, bool F8, int ACT>
__global__ void __launch_bounds__(kGnThreads, 2) gn_stats_kernel(const GnArgs g) {
  extern __shared__ __align__(1024) uint8_t smem[];
  // the norm's launch may begin, its CTAs wait for the statistics themselves
  if (!KEEP) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int shift = 31 - __clz(g.sub), per = 8 >> shift;          // entries of a thread
  const int width = (g.cols * per) | 1;                           // of a slot, odd: slots lie in other banks
  float2* sums = reinterpret_cast<float2*>(smem);                 // [slots, width]
  float2* own = sums + g.slots * width;                           // [G] this CTA's
  float2* fin = own + g.G;                                        // [G] mean, rstd (KEEP)
  // KEEP: [chunk, cols], else [kGnRing, threads]
  uint4* kept = reinterpret_cast<uint4*>(smem + (((g.slots * width + (KEEP ? 2 : 1) * g.G) * 8 + 15) & ~15));
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const GnPlace at(g);
  const int rows = gn_rows(g, at.c);
  // slot i takes rows i, i + slots, ...: more of them the first `rest` slots
  const int least = rows / g.slots, rest = rows - least * g.slots;
  const int mine = at.busy ? least + (at.s0 < rest) : 0;          // this thread's rows
  const long long step = g.slots * g.x_row;
  const long long jump = (long long)((g.runs << g.cluster_shift) - 1) * g.tile * g.x_row;   // to the next tile
  const T* x = reinterpret_cast<const T*>(g.x) + at.b * g.x_batch + at.part * g.C + ((long long)at.c * g.tile + at.s0) * g.x_row;
  const int keep_step = KEEP ? g.slots * g.cols : kGnThreads;
  // the second launch's CTAs begin with a tile each
  if (!KEEP && at.run == 0 && at.rank == 0 && t == 0) g.tiles[at.b * g.parts + at.part] = g.runs << g.cluster_shift;
  if (at.busy) {
    for (int v = at.v0; v < g.cols; v += at.wide) {
      const int n = g.C - 8 * v;   // <= 0: a column that only fills up a block
      if (n <= 0) continue;
      const T* p = x + 8 * v;
      uint4* keep = KEEP ? kept + at.s0 * g.cols + v : kept + t;
      if (KEEP) {   // all of them at once
        uint4* to = keep;
        for (int r = 0; r < mine; ++r, p += step, to += keep_step) gn_fetch(to, p, n, g.vec != 0);
        gn_commit();
        gn_arrived<0>();
      } else {
#pragma unroll
        for (int r = 0; r < kGnRing; ++r) {
          if (r < mine) gn_fetch(keep + r * keep_step, p, n, g.vec != 0);
          p += step;
          gn_commit();
        }
        p += jump;
      }
      uint64_t x0[4], s2[4], q2[4];   // -x0
#pragma unroll
      for (int i = 0; i < 4; ++i) x0[i] = s2[i] = q2[i] = 0;
      const auto add = [&](const uint4& in, bool first) {
        uint64_t f[4];
        gn_unpack<T>(in, f);
        if (first) {
#pragma unroll
          for (int j = 0; j < 4; ++j) x0[j] = gn_neg2(f[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t d = gn_add2(f[j], x0[j]);
          s2[j] = gn_add2(s2[j], d);
          q2[j] = gn_fma2(d, d, q2[j]);
        }
      };
      if (KEEP) {
        const uint4* from = keep;
#pragma unroll 2
        for (int r = 0; r < mine; ++r, from += keep_step) add(*from, r == 0);
      } else {
        for (int r0 = 0; r0 < mine; r0 += kGnRing) {
#pragma unroll
          for (int k = 0; k < kGnRing; ++k) {
            if (r0 + k < mine) {
              gn_arrived<kGnRing - 1>();
              add(keep[k * keep_step], r0 + k == 0);
              if (r0 + k + kGnRing < mine) gn_fetch(keep + k * keep_step, p, n, g.vec != 0);
              p += step;
              gn_commit();
            }
          }
          p += jump;
        }
        gn_arrived<0>();
      }
      const float count = (float)mine, inv = mine ? __frcp_rn(count) : 0.f;
      float s[8], q[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float z[2];
        gn_untwo(s2[i], s[2 * i], s[2 * i + 1]);
        gn_untwo(q2[i], q[2 * i], q[2 * i + 1]);
        gn_untwo(x0[i], z[0], z[1]);
#pragma unroll
        for (int j = 2 * i; j < 2 * i + 2; ++j) {
          // (squares beyond fp32's range: infinite, and not NaN, of which the maximum
          // would make 0)
          const float d = s[j] * inv;
          q[j] = q[j] <= 3.4028235e38f ? fmaxf(0.f, fmaf(-s[j], d, q[j])) : q[j];
          s[j] = d - z[j & 1];
        }
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
  const float inv_total = __frcp_rn((float)max(rows, 1) * (float)g.Cg);
  for (int i = warp; i < g.G; i += kGnThreads / 32) {
    const float2* from = sums + i * entries;
    const float ref = from[0].x;
    float mean = ref, dev = 0.f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      float sum = 0.f;
      for (int sl = sl0, e = e0; sl < g.slots;) {
        const float2 v = from[sl * width + e];
        const float count = (float)((least + (sl < rest)) << shift), d = v.x - mean;
        sum += pass ? fmaf(count * d, d, v.y) : count * d;
        sl += dq;
        e += dr;
        if (e >= entries) { e -= entries; ++sl; }
      }
      sum = gn_warp_sum(sum);
      if (pass) dev = sum;
      else mean = fmaf(sum, inv_total, ref);
    }
    if (lane == 0) own[i] = make_float2(mean, dev);
  }
  __syncwarp();
  if (g.cluster > 1) cluster_sync_all();
  else __syncthreads();
  // the cluster's CTAs, a lane each
  if (KEEP || at.rank == 0) {
    const int p = lane & (g.cluster - 1);
    const float count = (float)gn_rows(g, (at.run << g.cluster_shift) + p) * (float)g.Cg;
    const float inv = __frcp_rn((float)gn_run_rows(g, at.run) * (float)g.Cg);
    for (int i0 = 0; i0 < g.G; i0 += kGnThreads >> g.cluster_shift) {
      const int i = i0 + (t >> g.cluster_shift);
      float2 v;
      const uint32_t where = mapa_u32(smem_u32(own + min(i, g.G - 1)), p);
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(where) : "memory");
      const float ref = __shfl_sync(0xffffffffu, v.x, lane & ~(g.cluster - 1));
      float sum = count * (v.x - ref);
      for (int d = 1; d < g.cluster; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float mean = fmaf(sum, inv, ref), dev = v.x - mean;
      float m2 = fmaf(count * dev, dev, v.y);
      for (int d = 1; d < g.cluster; d *= 2) m2 += __shfl_xor_sync(0xffffffffu, m2, d);
      if (p == 0 && i < g.G) {
        if (KEEP) fin[i] = make_float2(mean, rsqrtf(fmaf(m2, inv, g.eps)));
        else g.part[((long long)(at.b * g.parts + at.part) * g.G + i) * g.runs + at.run] = make_float2(mean, m2);
      }
    }
  }
  if (KEEP) {
    __syncthreads();
    if (at.busy) {
      for (int v = at.v0; v < g.cols; v += at.wide) {
        const bool in_row = 8 * v < g.C;
        if (!F8 && !in_row) continue;
        GnFactors f;
        f.load(g, fin, at.part * g.C, v);
        const uint4* from = kept + at.s0 * g.cols + v;
        GnOut<T, F8> o(g, at, (long long)at.c * g.tile + at.s0, v, g.slots);
#pragma unroll 2
        for (int r = 0; r < mine; ++r, from += keep_step, o.next())
          gn_finish<T, F8, ACT>(g, f, in_row ? *from : make_uint4(0, 0, 0, 0), o, v);
      }
    }
  }
  // nobody leaves while another CTA may read its shared memory (threads without a
  // row come here before the others of their warp)
  __syncwarp();
  if (g.cluster > 1) cluster_sync_all();
}

// The norm from the workspace's statistics, tile by tile from the last row on.  A
// CTA takes the next tile when it has time: those far from the memory that they
// read need a third longer for the same rows.  (Every value goes by its own row
// and the statistics, whoever computes it.)
template <typename T, bool F8, int ACT>
__global__ void __launch_bounds__(kGnThreads, 2) gn_apply_kernel(const GnArgs g) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;          // [kGnRing, threads]
  float2* fin = reinterpret_cast<float2*>(smem + kGnRing * kGnThreads * 16);   // [G] mean, rstd
  int* box = reinterpret_cast<int*>(fin + g.G);                        // [2] a tile taken
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const GnPlace at(g);
  const int tiles = (int)((g.L + g.tile - 1) / g.tile);
  const long long step = g.slots * g.x_row;
  const T* x = reinterpret_cast<const T*>(g.x) + at.b * g.x_batch + at.part * g.C;
  // this thread's rows of the i-th tile from the end, and how many
  const auto first = [&](int i) { return (long long)(tiles - 1 - i) * g.tile + at.s0; };
  const auto number = [&](int i) {
    const long long left = g.L - first(i);
    return !at.busy || i >= tiles || left <= 0 ? 0 : left >= g.tile ? kGnRing : (int)min((long long)kGnRing, (left + g.slots - 1) / g.slots);
  };
  int cur = at.c, have = number(cur);
  {   // x is no output of the first launch
    const T* p = x + (have ? first(cur) * g.x_row : 0) + 8 * at.v0;
#pragma unroll
    for (int r = 0; r < kGnRing; ++r) {
      if (r < have && 8 * at.v0 < g.C) gn_fetch(ring + r * kGnThreads, p + r * step, g.C - 8 * at.v0, g.vec != 0);
      gn_commit();
    }
  }
  float count[kGnLaneRuns];
#pragma unroll
  for (int k = 0; k < kGnLaneRuns; ++k) {
    const int j = lane + 32 * k;
    count[k] = j < g.runs ? (float)gn_run_rows(g, j) * (float)g.Cg : 0.f;
  }
  const float inv = __frcp_rn((float)g.L * (float)g.Cg);
  const float2* part = g.part + (long long)(at.b * g.parts + at.part) * g.runs * g.G;
  int* taken = g.tiles + at.b * g.parts + at.part;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0) box[0] = atomicAdd(taken, 1);
#pragma unroll 2
  for (int i = warp; i < g.G; i += kGnThreads / 32) {
    float2 w[kGnLaneRuns];
#pragma unroll
    for (int k = 0; k < kGnLaneRuns; ++k) w[k] = __ldcg(part + (long long)i * g.runs + min(lane + 32 * k, g.runs - 1));
    const float ref = __shfl_sync(0xffffffffu, w[0].x, 0);
    float sum = 0.f, dev = 0.f;
#pragma unroll
    for (int k = 0; k < kGnLaneRuns; ++k) sum = fmaf(count[k], w[k].x - ref, sum);
    const float mean = fmaf(gn_warp_sum(sum), inv, ref);
#pragma unroll
    for (int k = 0; k < kGnLaneRuns; ++k) {
      const float d = w[k].x - mean;
      if (count[k] > 0.f) dev += fmaf(count[k] * d, d, w[k].y);
    }
    dev = gn_warp_sum(dev);
    if (lane == 0) fin[i] = make_float2(mean, rsqrtf(fmaf(dev, inv, g.eps)));
  }
  __syncthreads();
  GnFactors f;
  f.load(g, fin, at.part * g.C, min(at.v0, g.cols - 1));
  int next = box[0];
  for (int it = 1; cur < tiles; ++it) {
    int got = 0;
    if (threadIdx.x == 0) got = atomicAdd(taken, 1);
    const int then = number(next);
    for (int v = at.v0; v < g.cols; v += at.wide) {
      if (at.wide < g.cols) f.load(g, fin, at.part * g.C, v);
      // what the ring is filled up with: this tile's next columns, or the next tile
      const bool more = v + at.wide < g.cols;
      const int vn = more ? v + at.wide : at.v0, hn = 8 * vn < g.C ? (more ? have : then) : 0;
      const T* p = x + (hn ? first(more ? cur : next) * g.x_row : 0) + 8 * vn;
      const int n = g.C - 8 * v;
      GnOut<T, F8> o(g, at, first(cur), v, g.slots);
#pragma unroll 4
      for (int r = 0; r < kGnRing; ++r) {
        if (r < have) {
          gn_arrived<kGnRing - 1>();
          if (F8 || n > 0) gn_finish<T, F8, ACT>(g, f, n > 0 ? ring[r * kGnThreads] : make_uint4(0, 0, 0, 0), o, v);
          o.next();
        }
        if (r < hn) gn_fetch(ring + r * kGnThreads, p, g.C - 8 * vn, g.vec != 0);
        p += step;
        gn_commit();
      }
    }
    if (threadIdx.x == 0) box[it & 1] = got;
    __syncthreads();
    cur = next;
    have = then;
    next = box[it & 1];
  }
  gn_arrived<0>();
}

// ============================================================== host side

constexpr int kGnShared = 200 * 1024, kGnHalf = 110 * 1024;   // one and two CTAs an SM
constexpr int kGnRuns = 32 * kGnLaneRuns;

struct GnPlan {
  int parts, cols, slots, sub, cluster, runs;
  long long tile;            // rows: all of a CTA's (one launch), or kGnRing a thread
  bool keep;                 // one launch
  int shared;
  long long floats;          // workspace
};

// parts: C and G are one part's
static void gn_threads(GnPlan& p, long long C, long long G, bool f8) {
  p.cols = (int)((C + 7) / 8);
  if (f8) p.cols = (p.cols + 15) / 16 * 16;
  p.slots = p.cols <= kGnThreads ? kGnThreads / p.cols : 1;
  p.sub = 1;
  while (p.sub < 8 && C / G % (2 * p.sub) == 0) p.sub *= 2;
}

// CTAs in clusters of 1 << shift that the device holds at once, `two` on an SM (of 4
// and more they do not fill its processor groups: 132 of 148 in clusters of 4,
// 120 of 8, 112 of 16).  Asked once a device; without one, seven eighths.
static long long gn_places(int dev, long long sms, int shift, bool two) {
  static std::atomic<int> known[64][5][2];
  std::atomic<int>& at = known[dev & 63][shift][two];
  if (at.load()) return at.load();
  int clusters = 0;
  auto kern = gn_stats_kernel<__half, true, false, 1>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim.x = 1u << shift;
  a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(16384);
  cfg.blockDim = dim3(kGnThreads);
  cfg.dynamicSmemBytes = two ? kGnHalf : kGnShared;
  cfg.attrs = a;
  cfg.numAttrs = 1;
  const bool asked = set_smem_once(kern, 227 * 1024) == cudaSuccess &&
                     cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                     cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) == cudaSuccess;
  if (!asked) (void)cudaGetLastError();
  const long long guess = shift < 2 ? sms : sms * 7 / 8 >> shift << shift;
  const long long n = asked && clusters > 0 ? (long long)clusters << shift : asked ? 0 : two ? 2 * guess : guess;
  if (n > 0) at.store((int)n);
  return n;
}

static GnPlan gn_plan(long long B, long long L, long long C, long long G, bool f8) {
  GnPlan p;
  const long long sms = num_sms();
  // One launch where what a cluster keeps fits.  A part is whole groups and whole
  // 16-byte columns (128 channels for e4m3).  The cheapest of the ways to deal it
  // out, in clocks as they were measured: a CTA takes 6000 and 0.3 a value, two that
  // share an SM 7500 and 0.6, a cluster's exchange 3500; rows in pieces below 64
  // bytes half as much again.
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  long long ones[5], twos[5];
  for (int i = 0; i < 5; ++i) {
    ones[i] = gn_places(dev, sms, i, false);
    twos[i] = gn_places(dev, sms, i, true);
  }
  double best = 0;
  for (long long parts = 1; parts <= G && parts <= 4 * sms; ++parts) {
    if (G % parts || (parts > 1 && C / parts % (f8 ? 128 : 8))) continue;
    GnPlan t;
    t.parts = (int)parts;
    gn_threads(t, C / parts, G / parts, f8);
    const long long sums = (long long)t.slots * ((t.cols * (8 / t.sub)) | 1);
    const long long head = ((sums + 2 * (G / parts)) * 8 + 15) / 16 * 16;
    const long long most = (kGnShared - head) / ((long long)t.cols * 16);   // rows of a CTA
    if (most <= 0) continue;
    int shift = 0;
    for (t.cluster = 1; t.cluster <= 16; t.cluster *= 2, ++shift) {
      t.tile = (L + t.cluster - 1) / t.cluster;
      const long long ctas = B * parts * t.cluster;
      if (t.tile > most || ctas > (1LL << 30)) continue;
      t.shared = (int)(head + t.tile * t.cols * 16);
      const long long one = ones[shift], two = t.shared <= kGnHalf ? twos[shift] : 0;
      if (one <= 0) continue;   // clusters of this size do not fit at all
      const double values = (double)t.tile * t.cols * 8 * (C / parts < 32 ? 1.5 : 1.0);
      double cost = (double)((ctas + one - 1) / one) * (6000 + 0.3 * values);
      if (two > 0) {
        const double shared = (double)((ctas + two - 1) / two) * (7500 + 0.6 * values);
        if (ctas > one && shared < cost) cost = shared;
      }
      if (t.cluster > 1) cost += 3500;
      if (best && cost >= best) continue;
      best = cost;
      t.runs = 1;
      t.keep = true;
      t.floats = 0;
      p = t;
    }
  }
  // Two launches: 22000, and 0.27 a value at all SMs' rate.
  if (best && best <= 22000 + 0.27 * (double)B * (double)L * (double)C / sms) return p;
  p.parts = 1;
  p.keep = false;
  gn_threads(p, C, G, f8);
  p.cluster = 2;   // (of four or eight, not as many as the SMs have room for fit at once: a few were left for a second wave)
  long long runs = 2 * sms / p.cluster / B;
  p.tile = (long long)p.slots * kGnRing;
  const long long useful = (L + p.tile * p.cluster - 1) / (p.tile * p.cluster);   // each has a tile
  runs = runs < useful ? runs : useful;
  p.runs = (int)(runs < 1 ? 1 : runs > kGnRuns ? kGnRuns : runs);
  const long long sums = (long long)p.slots * ((p.cols * (8 / p.sub)) | 1);
  p.shared = (int)(((sums + G) * 8 + 15) / 16 * 16) + kGnRing * kGnThreads * 16;
  p.floats = 2 * B * p.runs * G + B;
  return p;
}

template <typename T, bool F8, int ACT>
static cudaError_t gn_launch(GnArgs a, const GnPlan& p, long long B, cudaStream_t st) {
  a.parts = p.parts;
  a.C /= p.parts;
  a.G /= p.parts;
  if (p.parts > 1) a.width = a.C;
  a.cols = p.cols;
  a.slots = p.slots;
  a.sub = p.sub;
  a.cluster = p.cluster;
  a.cluster_shift = 31 - __builtin_clz(p.cluster);
  a.runs = p.runs;
  const long long tiles = (a.L + p.tile - 1) / p.tile, ctas = (long long)p.runs * p.cluster;
  a.tile = (int)p.tile;
  a.deal = (int)(tiles / ctas);
  a.more = (int)(tiles % ctas);
  a.lack = (int)(tiles * p.tile - a.L);
  a.tiles = reinterpret_cast<int*>(a.part + B * p.runs * a.G);   // (two launches have one part)
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(B * p.parts * p.runs * p.cluster));
  cfg.blockDim = dim3(kGnThreads);
  cfg.dynamicSmemBytes = p.shared;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (p.keep) {
    auto kern = gn_stats_kernel<T, true, F8, ACT>;
    cudaError_t e = set_smem_once(kern, 227 * 1024);
    if (e == cudaSuccess && p.cluster > 8) {
      static std::atomic<unsigned long long> devices{0};   // that the attribute is set on
      int dev = 0;
      cudaGetDevice(&dev);
      if (!(devices.load() >> (dev & 63) & 1)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) devices.fetch_or(1ull << (dev & 63));
      }
    }
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
  cfg.dynamicSmemBytes = kGnRing * kGnThreads * 16 + a.G * 8 + 8;
  return cudaLaunchKernelEx(&cfg, apply, a);
}

template <typename T, bool F8>
static cudaError_t gn_launch_act(const GnArgs& a, const GnPlan& p, long long B, int act, cudaStream_t st) {
  if (act == 0) return gn_launch<T, F8, 0>(a, p, B, st);
  if (act == 1) return gn_launch<T, F8, 1>(a, p, B, st);
  if (act == 2) return gn_launch<T, F8, 2>(a, p, B, st);
  return gn_launch<T, F8, 3>(a, p, B, st);
}

cudaError_t launch_group_norm(const GnArgs& a, const GnPlan& p, int64_t B, int dtype, int act, cudaStream_t st) {
  if (dtype == IC_DTYPE_F16) return a.q ? gn_launch_act<__half, true>(a, p, B, act, st) : gn_launch_act<__half, false>(a, p, B, act, st);
  return a.q ? gn_launch_act<__nv_bfloat16, true>(a, p, B, act, st) : gn_launch_act<__nv_bfloat16, false>(a, p, B, act, st);
}

}  // namespace ic
