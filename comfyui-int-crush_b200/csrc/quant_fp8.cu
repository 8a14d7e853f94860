// Values to e4m3 with a scale for each block of 128: rows of activations
// (1 x 128) or weights (128 x 128).
//   s = RN32(max(max |x|, 1e-8) / 448),  q = RN_e4m3(RN32(x / s))
// A NaN makes its block's scale NaN, an infinity infinite (its own value NaN,
// the others 0), so that neither is lost in a product.
//
// One pass; HBM bounds it.  65520 x 5120 bf16: 170 us, 6.0 TB/s (92% of a copy);
// weights 13824 x 5120: 44.7 us, 4.7 TB/s (a CTA's loads, its maximum and its stores
// follow one another; an SM's CTAs cover for each other in part).
#include <type_traits>

namespace ic {

constexpr float kF8Max = 448.f, kF8AmaxMin = 1e-8f;

// A block's scale and the reciprocal that its quotients start from.
struct F8Scale {
  float s, inv;
};
__device__ __forceinline__ F8Scale f8_scale(float amax) {
  F8Scale r;
  r.s = __fdiv_rn(amax < kF8AmaxMin ? kF8AmaxMin : amax, kF8Max);   // (a NaN stays)
  r.inv = __frcp_rn(r.s);
  return r;
}
// x / s for |x| <= 448 s, s finite: the product with the correctly rounded
// reciprocal, corrected by its remainder (Markstein, "Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990): 3 instructions where
// the division takes about ten.  Where the remainder is below the subnormals
// the quotient is far below e4m3's least value.  (The remainder is taken
// negative: so the quotient of -0 is -0.)
__device__ __forceinline__ float f8_quotient(float x, const F8Scale& f) {
  const float q = x * f.inv;
  return fmaf(-fmaf(q, f.s, -x), f.inv, q);
}
// two values to e4m3, ties to even, the first in the low byte
__device__ __forceinline__ uint32_t f8_pair(float lo, float hi) {
  uint16_t v;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v) : "f"(hi), "f"(lo));
  return v;
}
__device__ __forceinline__ uint32_t f8_four(float a, float b, float c, float d, const F8Scale& f) {
  return f8_pair(f8_quotient(a, f), f8_quotient(b, f)) | f8_pair(f8_quotient(c, f), f8_quotient(d, f)) << 16;
}
__device__ __forceinline__ uint32_t f8_four_div(float a, float b, float c, float d, float s) {
  return f8_pair(__fdiv_rn(a, s), __fdiv_rn(b, s)) | f8_pair(__fdiv_rn(c, s), __fdiv_rn(d, s)) << 16;
}

// 16 values of a lane as they are read: |x| by its bits, which order like the
// values with infinities above them and NaN above those.
template <typename T> struct F8In {   // 16-bit types
  uint32_t w[8];
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    return max(m & 0xffffu, m >> 16);
  }
  static __device__ __forceinline__ float top_value(uint32_t bits) {
    if (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)bits));
    return __uint_as_float(bits << 16);
  }
  __device__ __forceinline__ void get4(int i, float (&v)[4]) const {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t p = w[2 * i + j];
      if (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      } else {
        v[2 * j] = __uint_as_float(p << 16);
        v[2 * j + 1] = __uint_as_float(p & 0xffff0000u);
      }
    }
  }
  // values [0, n) of p, 8 at a time where `vec` (then n is a multiple of 8)
  __device__ __forceinline__ void load(const T* p, int n, bool vec) {
    if (vec) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (8 * h < n) v = __ldg(reinterpret_cast<const uint4*>(p) + h);
        w[4 * h] = v.x; w[4 * h + 1] = v.y; w[4 * h + 2] = v.z; w[4 * h + 3] = v.w;
      }
    } else {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = (2 * i < n ? (uint32_t)__ldg(u + 2 * i) : 0u) | (2 * i + 1 < n ? (uint32_t)__ldg(u + 2 * i + 1) << 16 : 0u);
    }
  }
};
template <> struct F8In<float> {
  uint32_t w[16];
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  }
  static __device__ __forceinline__ float top_value(uint32_t bits) { return __uint_as_float(bits); }
  __device__ __forceinline__ void get4(int i, float (&v)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[4 * i + j]);
  }
  __device__ __forceinline__ void load(const float* p, int n, bool vec) {
    if (vec) {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (4 * h < n) v = __ldg(reinterpret_cast<const uint4*>(p) + h);
        w[4 * h] = v.x; w[4 * h + 1] = v.y; w[4 * h + 2] = v.z; w[4 * h + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = i < n ? __ldg(reinterpret_cast<const uint32_t*>(p) + i) : 0u;
    }
  }
};

struct F8QuantArgs {
  const void* x;
  long long M, ldx;
  int K, kb, width;        // width: K rounded up to 16, zeros behind K
  uint8_t* q;
  long long ldq;
  float* s;
  long long s_row, s_block;
  int vec;
};

// 16 values to 16 bytes.  fp32 inputs take the division itself: the quotient's
// last bit is only checked for 16-bit ones.
template <typename T>
__device__ __forceinline__ uint4 f8_bytes(const F8In<T>& in, const F8Scale& f) {
  uint32_t w[4];
  const bool plain = !std::is_same<T, float>::value && f.s <= 3.4e38f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[4];
    in.get4(i, v);
    w[i] = plain ? f8_four(v[0], v[1], v[2], v[3], f) : f8_four_div(v[0], v[1], v[2], v[3], f.s);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Activations.  8 lanes hold a block (16 values each: 32 bytes in, 16 out), a
// warp 4 rows of one block column and R such groups of rows, all loads ahead
// of the first maximum.  The rows of a warp are neighbours, so that with the
// scales stored block by block (s_row 1) their four stores share a sector.
template <typename T, int R>
__global__ void __launch_bounds__(256) quant_fp8_rows_kernel(const F8QuantArgs a) {
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long group = unit / a.kb;
  const int b = (int)(unit - group * a.kb);
  const long long m0 = group * (4 * R) + (lane >> 3);
  if (group * (4 * R) >= a.M) return;
  const int k = b * 128 + (lane & 7) * 16;
  F8In<T> in[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const long long m = m0 + 4 * i;
    const int n = m < a.M ? max(0, min(16, a.K - k)) : 0;
    in[i].load(reinterpret_cast<const T*>(a.x) + (n > 0 ? m * a.ldx + k : 0), n, a.vec != 0);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    uint32_t top = in[i].top();
#pragma unroll
    for (int d = 4; d; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const F8Scale f = f8_scale(F8In<T>::top_value(top));
    const uint4 v = f8_bytes<T>(in[i], f);
    const long long m = m0 + 4 * i;
    if (m < a.M) {
      if (k < a.width) *reinterpret_cast<uint4*>(a.q + m * a.ldq + k) = v;
      if ((lane & 7) == 0) a.s[m * a.s_row + b * a.s_block] = f.s;
    }
  }
}

// Weights: a CTA per 128 x 128 block, its values in registers: 32 a thread of 16 warps
// for 16-bit types (13824 x 5120: 44.7 us, 47.3 with 64 of 8 warps), 64 of 8 warps for
// fp32 (62.5 us, 64.4 with 32 of 16 warps).
template <typename T>
constexpr int kF8SquareWarps = sizeof(T) == 2 ? 16 : 8;

template <typename T>
__global__ void __launch_bounds__(32 * kF8SquareWarps<T>) quant_fp8_square_kernel(const F8QuantArgs a) {
  constexpr int W = kF8SquareWarps<T>, R = 32 / W;   // warps, rows a thread
  __shared__ uint32_t tops[W];
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long m0 = (long long)blockIdx.y * 128 + warp * (4 * R) + (lane >> 3);
  const int k = b * 128 + (lane & 7) * 16;
  F8In<T> in[R];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const long long m = m0 + 4 * i;
    const int n = m < a.M ? max(0, min(16, a.K - k)) : 0;
    in[i].load(reinterpret_cast<const T*>(a.x) + (n > 0 ? m * a.ldx + k : 0), n, a.vec != 0);
    top = max(top, in[i].top());
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i) top = max(top, tops[i]);
  const F8Scale f = f8_scale(F8In<T>::top_value(top));
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const long long m = m0 + 4 * i;
    if (m < a.M && k < a.width) *reinterpret_cast<uint4*>(a.q + m * a.ldq + k) = f8_bytes<T>(in[i], f);
  }
  if (threadIdx.x == 0) a.s[(long long)blockIdx.y * a.s_row + b * a.s_block] = f.s;
}

template <typename T>
static cudaError_t f8_quant_launch(const F8QuantArgs& a, int rows, cudaStream_t st) {
  if (rows == 128) {
    quant_fp8_square_kernel<T><<<dim3(a.kb, (unsigned)((a.M + 127) / 128)), 32 * kF8SquareWarps<T>, 0, st>>>(a);
  } else if ((a.M + 15) / 16 * a.kb >= 8LL * num_sms()) {
    quant_fp8_rows_kernel<T, 4><<<(unsigned)(((a.M + 15) / 16 * a.kb + 7) / 8), 256, 0, st>>>(a);
  } else {
    // few blocks: four rows a warp, so that more warps share them
    quant_fp8_rows_kernel<T, 1><<<(unsigned)(((a.M + 3) / 4 * a.kb + 7) / 8), 256, 0, st>>>(a);
  }
  return cudaGetLastError();
}

cudaError_t launch_quant_fp8(const F8QuantArgs& a, int dtype, int rows, cudaStream_t st) {
  if (dtype == IC_DTYPE_F16) return f8_quant_launch<__half>(a, rows, st);
  if (dtype == IC_DTYPE_BF16) return f8_quant_launch<__nv_bfloat16>(a, rows, st);
  return f8_quant_launch<float>(a, rows, st);
}

}  // namespace ic
