// Declarations shared by the cross-attention kernels.
#pragma once

#include <math.h>

#include <type_traits>

#include "ic_common.cuh"

namespace ic {

constexpr float kLog2e = 1.4426950408889634f;

struct XattnArgs {
  // strides in elements over batch, token, head; the head's elements are
  // contiguous
  const void* q; int64_t qs[3];
  const void* k; int64_t ks[3];
  const void* v; int64_t vs[3];
  void* o; int64_t os[3];
  int64_t B, Lq, Lk;
  int H, Hk, D;
  float scale;
  const int32_t* kv_lens;      // [B] or NULL
  const float* bias;           // [B, Lkp] from xattn_mask_kernel, or NULL
  const int32_t* ends;         // [B], with bias
  int64_t Lkp;
  int splits;                  // parts of the keys
  int part_blocks;             // few-rows kernel: blocks of 16 keys in a part
  float* part_o;               // [splits, B, Lq, H, D] with splits > 1
  float* part_ml;              // [splits, B, Lq, H, 2]: reference (log2), sum
};

struct XattnPlan {
  int slots;                   // 0: few-rows kernel, else query tiles per item of the tcgen05 one
  int splits;
  int64_t Lkp;
  int64_t part_floats;
  int64_t floats;              // workspace
};

// Query heads of a key head that share a tile of the tcgen05 kernel.
inline int xattn_packed(int H, int Hk) {
  const int group = H / Hk;
  return 128 % group == 0 ? group : 1;
}

template <typename T>
cudaError_t launch_xattn_tc(const XattnArgs& a, int slots, cudaStream_t st);   // cross_attention_tc.cu
XattnPlan xattn_plan(int64_t B, int64_t Lq, int64_t Lk, int H, int Hk, int D, int mask_kind);

// 1 + the last key that sample b may see
__device__ __forceinline__ int xattn_end(const XattnArgs& a, int64_t b) {
  if (a.ends) return __ldg(a.ends + b);
  if (a.kv_lens) return max(0, min(__ldg(a.kv_lens + b), (int)a.Lk));
  return (int)a.Lk;
}

// A row's weights are p = 2^(x - ref) of its scores x in units of log2.  The
// reference follows the running maximum: it is set kXattnUp<T> below it and stays
// until the maximum is more than kXattnRoom<T> above it, so that most tiles
// rescale nothing.  In fp16 the largest weight so lies between 2^7 and 2^15, and
// the others are held to 2^-32 of it; with the maximum itself as reference it is
// 2^-25, and 2^15 keys of little weight could lose as much as the output's own
// rounding.  bf16 has fp32's range and needs neither.
template <typename T>
constexpr float kXattnUp = std::is_same<T, __half>::value ? 7.f : 0.f;
template <typename T>
constexpr float kXattnRoom = 8.f + kXattnUp<T>;
// (as a difference: ref + room would round where scores are large)
template <typename T>
__device__ __forceinline__ bool xattn_moves(float mx, float ref) {
  return mx - ref > kXattnRoom<T>;
}

// 2^x (the hardware's approximation, 2 ulp; 2^-inf = 0)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight output elements: v / sum, zeros for a row that saw no key.
template <typename T>
__device__ __forceinline__ void xattn_store8(const XattnArgs& a, int64_t b, int64_t l, int h, int d,
                                             const float (&v)[8], float sum) {
  const float r = sum == 0.f ? 0.f : 1.f / sum;
  uint4 w;
  w.x = pack16<T>(v[0] * r, v[1] * r);
  w.y = pack16<T>(v[2] * r, v[3] * r);
  w.z = pack16<T>(v[4] * r, v[5] * r);
  w.w = pack16<T>(v[6] * r, v[7] * r);
  *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.o) + b * a.os[0] + l * a.os[1] + h * a.os[2] + d) = w;
}

// A finished row part: to the output, or to the splits' partial sums.
template <typename T>
__device__ __forceinline__ void xattn_put(const XattnArgs& a, int64_t b, int64_t l, int h, int split, int d,
                                          const float (&v)[8], float m, float sum) {
  if (a.splits == 1) {
    xattn_store8<T>(a, b, l, h, d, v, sum);
    return;
  }
  const int64_t row = ((split * a.B + b) * a.Lq + l) * a.H + h;
  float4* p = reinterpret_cast<float4*>(a.part_o + row * a.D + d);
  p[0] = make_float4(v[0], v[1], v[2], v[3]);
  p[1] = make_float4(v[4], v[5], v[6], v[7]);
  if (d == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m, sum);
}

}  // namespace ic
