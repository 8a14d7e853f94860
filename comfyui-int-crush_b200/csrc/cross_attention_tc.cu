// Cross attention for many query rows on tcgen05 (kind::f16).
//
// Persistent, one CTA per SM, 16 warps.  A work item is one key head of one
// sample with one or two tiles of 128 query rows (all query heads that share the
// key head in turn for each token, where their number divides 128) ("slots"; the slots share the
// K and V tiles), over the item's part of the keys in tiles of 128:
//   S_s = Q_s K^T            128 x 128 into tensor memory
//   P_s = 2^(S_s c - m)      registers, written back over S_s as 16-bit pairs
//   O_s += P_s V             A operand from tensor memory, V as it lies in
//                            memory (rows = keys: the MN-major B operand)
// Tensor memory: S_0 | S_1 | O_0 | O_1, 128 columns each.
//
// Warps 0-3 / 4-7: softmax of slot 0 / 1, one row per thread (no shuffles).
// Warp 8: TMA producer (Q slots, a ring of K and V tiles).  Warp 9: MMA
// issuer.  Warp 10: zeroes the V rows of keys that are not seen (P is 0 there,
// but 0 * NaN is not) when there are lengths or a mask.  Warps 12-15: O out of
// tensor memory, over the row sums, to global memory.
// The MMAs of one slot run while the other slot's softmax does; P V starts when
// three quarters of P are written; the next item's first S is issued behind the
// last P V, so that nothing drains between items.
// What bounds it: a slot's turn from S to the next S.  Of its about 3000 clocks
// at D = 128 the softmax takes 1900 (the 128 exponentials of a row alone 1024,
// at 16 a clock per SM), P V's rest and the next S 1100; the MMAs of both slots
// (64 to 73 clocks for 128 x 128 x 16) fill 2200 of them.  S cannot run ahead:
// O and S of two slots take all 512 columns, so P lies over S.  Measured and
// not kept (8190 rows, 512 keys, 40 heads, 89 us): P through shared memory with
// S ahead 105 us (P's traffic on top of what the MMAs read), a part of the
// exponentials as polynomials 90 to 94, hand-interleaved 93 and more.
// 2 x 32760 rows, 512 keys, 40 heads of 128: 620 to 630 us, 1100 TFLOP/s, at
// 1965 MHz (three launches with pauses); 731 us, 940 TFLOP/s, back to back for
// seconds, where the power cap holds the clock at 1510 MHz (graph replays and
// single calls alike).
//
// S, the reference of a row's weights (kXattnUp), the row sum and O are fp32; the
// reference moves on few tiles, where O is rescaled in tensor memory.  P is
// rounded to the activation type, the MMA's operand type (at most u sum_j p_j
// |v_j| beside the output's own rounding), the row sum is not.
#include "cross_attention.cuh"

#include <type_traits>

namespace ic {

template <int DP>
struct XtCfg {
  static constexpr int PANELS = DP / 64;            // 64-element panels of 128 rows, 128B-swizzled
  static constexpr int TILE = PANELS * 16384;
  static constexpr int NST = DP == 128 ? 5 : 8;     // ring stages (K and V tiles in turn)
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_ML = OFF_KV + NST * TILE;   // row references and sums, [2 slots][128] float2
  static constexpr int OFF_BAR = OFF_ML + 2048;
  static constexpr int SMEM = OFF_BAR + 512;
  static constexpr int THREADS = 512;
  // 512 x 128 registers; the many where a thread holds a row of S
  static constexpr RegisterSplit REGS = {256, 72, 256, 184};
};

// n / d for 0 <= n < 2^30 by a multiplication: m = ceil(2^(30 + l) / d) with
// 2^l >= d is exact there (Granlund & Montgomery, "Division by invariant
// integers using multiplication", 1994).
struct XtDiv {
  uint32_t d, m, shift;
};
static XtDiv xt_div(uint32_t d) {
  uint32_t l = 0;
  while ((1u << l) < d) ++l;
  return {d, (uint32_t)((((uint64_t)1 << (30 + l)) + d - 1) / d), 30 + l};
}
__device__ __forceinline__ int xt_quot(const XtDiv& v, int n) { return (int)(((uint64_t)(uint32_t)n * v.m) >> v.shift); }

struct XtArgs {
  XattnArgs x;
  XtDiv by_split, by_head, by_hk, by_tiles;   // splits, items of a key head, key heads, query tiles of a head
  int slots;          // query tiles of an item: 1 or 2
  int group;          // query heads of a key head
  int packed;         // of them in a tile: row r is token r / packed, head r % packed
  int pack_shift;     // log2
  int tiles_per_head; // tiles of `packed` heads
  int tiles;          // query tiles of a key head
  int wide;           // output rows take 32-byte stores
  int items;
  int qm[2], km[2], vm[2];   // 0 where the batch / head stride is 0 (coordinate 0), else 1
};

struct XtItem {
  int64_t b;
  int hk, split, tile0, nslots, end, key0, nt;
};

__device__ __forceinline__ XtItem xt_item(const XtArgs& a, int i) {
  XtItem t;
  const int tiles = a.tiles;
  const int i0 = xt_quot(a.by_split, i);
  t.split = i - i0 * (int)a.by_split.d;
  const int bh = xt_quot(a.by_head, i0);
  t.tile0 = (i0 - bh * (int)a.by_head.d) * a.slots;
  t.nslots = min(a.slots, tiles - t.tile0);
  const int b = xt_quot(a.by_hk, bh);
  t.hk = bh - b * a.x.Hk;
  t.b = b;
  t.end = xattn_end(a.x, t.b);
  const int kt = (t.end + 127) / 128;
  const int per = xt_quot(a.by_split, kt + a.x.splits - 1);
  const int t0 = min(t.split * per, kt);
  t.nt = min(t0 + per, kt) - t0;
  t.key0 = t0 * 128;
  return t;
}
// first head and first token of slot s
__device__ __forceinline__ void xt_slot(const XtArgs& a, const XtItem& t, int s, int& h, int& l0) {
  const int q = t.tile0 + s;
  const int sub = xt_quot(a.by_tiles, q);
  h = t.hk * a.group + (sub << a.pack_shift);
  l0 = (q - sub * a.tiles_per_head) * (128 >> a.pack_shift);
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// MN-major operand in the 128-byte-swizzled layout: 64 contiguous elements
// per row, 8-row groups 1024 bytes apart (stride offset), panels of 64
// elements 16384 bytes apart (leading offset).
__device__ __forceinline__ uint64_t smem_desc_mn128(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(16384u >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1u << 46 | (uint64_t)2u << 61;
}

// The registers of a tcgen05.ld are valid after the wait: tie them to it.
__device__ __forceinline__ void tie32(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31]));
}

// The MMA warp stays converged, so that descriptors live in uniform registers;
// only the issue itself is one lane's (`on`).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on;
}
__device__ __forceinline__ void mma_f16_on(uint32_t on, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts_on(uint32_t on, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                              uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mma_commit_on(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(bar)), "r"(on)
      : "memory");
}

// 32 bytes at once (32-byte aligned)
__device__ __forceinline__ void st_global32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t two(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void untwo(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ bool all_lanes(bool ok) { return __all_sync(0xffffffffu, ok); }

template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(XtCfg<DP>::THREADS, 1)
xattn_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const XtArgs a) {
  using C = XtCfg<DP>;
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  constexpr int NST = C::NST;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;   // no static shared memory: the declared alignment holds
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);   // [2] TMA -> MMA
  uint64_t* q_empty = q_full + 2;       // [2] the item's last S is done -> TMA
  uint64_t* s_full = q_empty + 2;       // [2] S is done -> softmax
  uint64_t* p_part = s_full + 2;        // [2] P's first 96 keys are written, O rescaled -> MMA (4 warps)
  uint64_t* p_full = p_part + 2;        // [2] all of P is written -> MMA (4 warps)
  uint64_t* o_full = p_full + 2;        // [2] the item's last P V is done -> epilogue
  uint64_t* o_empty = o_full + 2;       // [2] O is read -> MMA (4 warps)
  uint64_t* l_full = o_empty + 2;       // [2] row references and sums are there -> epilogue (4 warps)
  uint64_t* l_empty = l_full + 2;       // [2] and read -> softmax (4 warps)
  uint64_t* kv_full = l_empty + 2;      // [NST] TMA -> MMA, cleaner
  uint64_t* kv_empty = kv_full + NST;   // [NST] MMA -> TMA
  uint64_t* ready = kv_empty + NST;     // [NST] cleaner -> MMA
  uint64_t* drain = ready + NST;        // all MMAs are done, at the end
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(drain + 2);

  // values that are the same in all lanes, said so by the broadcast: the role
  // branches and the MMA warp's descriptors then compile as warp-uniform
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_part + i, 4);
      mbar_init(p_full + i, 4);
      mbar_init(l_full + i, 4);
      mbar_init(l_empty + i, 4);
      mbar_init(o_full + i, 1);
      mbar_init(o_empty + i, 4);
    }
    for (int i = 0; i < NST; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
      mbar_init(ready + i, 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const bool clean = BIAS || a.x.kv_lens != nullptr;
  const uint32_t kv_base = smem_u32(smem) + C::OFF_KV;
  float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
  const auto next_item = [&](int& i, XtItem& t) {
    for (; i < a.items; i += gridDim.x) {
      t = xt_item(a, i);
      if (t.nt) return true;
    }
    return false;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(XtCfg<DP>::REGS.few));
    if (warp == 8) {
      // ------------------------------------------------------------ producer
      if (lane == 0) {
        uint32_t use = 0, qn[2] = {0, 0};
        bool ok = true;
        const auto load_kv = [&](const CUtensorMap* tm, const XtItem& t, const int* mul, int key) {
          const uint32_t st = use % NST;
          if (!mbar_wait(kv_empty + st, ((use / NST) & 1u) ^ 1u, abort_flag)) return false;
          mbar_arrive_expect_tx(kv_full + st, C::TILE);
#pragma unroll
          for (int p = 0; p < C::PANELS; ++p)
            tma_load_4d(kv_base + st * C::TILE + p * 16384, tm, kv_full + st, 64 * p, t.hk * mul[1], key,
                        (int)t.b * mul[0]);
          ++use;
          return true;
        };
        const auto load_q = [&](const XtItem& t, int s) {
          if (!mbar_wait(q_empty + s, (qn[s] & 1u) ^ 1u, abort_flag)) return false;
          int h, l0;
          xt_slot(a, t, s, h, l0);
          mbar_arrive_expect_tx(q_full + s, C::TILE);
#pragma unroll
          for (int p = 0; p < C::PANELS; ++p)
            tma_load_4d(smem_u32(smem) + s * C::TILE + p * 16384, &tm_q, q_full + s, 64 * p, h * a.qm[1], l0,
                        (int)t.b * a.qm[0]);
          ++qn[s];
          return true;
        };
        XtItem t;
        for (int i = blockIdx.x; ok && next_item(i, t); i += gridDim.x) {
          // K first: its stage frees before the Q slots of the item before
          ok = load_kv(&tm_k, t, a.km, t.key0) && load_q(t, 0) && (t.nslots < 2 || load_q(t, 1)) &&
               load_kv(&tm_v, t, a.vm, t.key0);
          for (int j = 1; ok && j < t.nt; ++j)
            ok = load_kv(&tm_k, t, a.km, t.key0 + 128 * j) && load_kv(&tm_v, t, a.vm, t.key0 + 128 * j);
        }
        // every copy issued lands before the CTA may leave, whoever gave up
        volatile int never = 0;
        for (uint32_t u = use > NST ? use - NST : 0; u < use; ++u) mbar_wait(kv_full + u % NST, (u / NST) & 1u, &never);
        for (int s = 0; s < 2; ++s)
          if (qn[s]) mbar_wait(q_full + s, (qn[s] - 1) & 1u, &never);
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------- MMA issuer
      const uint32_t on = elect_one();
      const int ksteps = (a.x.D + 15) / 16;
      const uint32_t i_pv = idesc_f16(128, ksteps * 16, BF) | (1u << 16);   // B is MN-major
      uint32_t use = 0, qph = 0, hph = 0, pph = 0, oph = 3;   // a phase bit per slot
      const auto tile_wait = [&](uint32_t u) {
        return all_lanes(mbar_wait((clean ? ready : kv_full) + u % NST, (u / NST) & 1u, abort_flag));
      };
      const auto slot_wait = [&](uint64_t* bar, uint32_t& ph, int s) {
        const uint32_t parity = (ph >> s) & 1u;
        ph ^= 1u << s;
        return all_lanes(mbar_wait(bar + s, parity, abort_flag));
      };
      // keys of tile j of an item, rounded to the MMA's step
      const auto width = [&](const XtItem& t, int j) { return min(128, (t.end - t.key0 - 128 * j + 15) / 16 * 16); };
      const auto issue_s = [&](int s, uint32_t u, int n, bool last) {
        const uint64_t dq = smem_desc_sw128(smem_u32(smem) + s * C::TILE);
        const uint64_t dk = smem_desc_sw128(kv_base + (u % NST) * C::TILE);
        const uint32_t idesc = idesc_f16(128, n, BF);
        const auto step = [&](int k) {   // offsets in descriptor units (16 bytes)
          const uint32_t off = (k >> 2) * (16384 >> 4) + (k & 3) * (32 >> 4);
          mma_f16_on(on, tmem + s * 128, dq + off, dk + off, idesc, k > 0);
        };
        if (ksteps == DP / 16) {
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) step(k);
        } else {
#pragma unroll 1
          for (int k = 0; k < ksteps; ++k) step(k);
        }
        mma_commit_on(on, s_full + s);
        if (last) mma_commit_on(on, q_empty + s);
      };
      // P V over the steps [k0, k1) of 16 keys
      const auto issue_pv = [&](int s, uint32_t u, int k0, int k1, uint32_t accumulate) {
        const uint64_t dv = smem_desc_mn128(kv_base + (u % NST) * C::TILE) + k0 * (2048 >> 4);
        const uint32_t pa = tmem + s * 128 + k0 * 8;
        const auto step = [&](int k) {
          mma_f16_ts_on(on, tmem + 256 + s * 128, pa + k * 8, dv + k * (2048 >> 4), i_pv, k > 0 ? 1u : accumulate);
        };
        if (k1 - k0 == 6) {
#pragma unroll
          for (int k = 0; k < 6; ++k) step(k);
        } else {
#pragma unroll 1
          for (int k = 0; k < k1 - k0; ++k) step(k);
        }
      };
      const auto next_uniform = [&](int& i, XtItem& t) {
        const bool got = next_item(i, t);
        t.end = uniform(t.end);
        t.nt = uniform(t.nt);
        t.key0 = uniform(t.key0);
        return all_lanes(got);
      };
      int i = blockIdx.x;
      XtItem t, nx;
      bool have = next_uniform(i, t), ok = true;
      if (have) {
        ok = tile_wait(use);
        for (int s = 0; ok && s < t.nslots; ++s) {
          ok = slot_wait(q_full, qph, s);
          if (ok) issue_s(s, use, width(t, 0), t.nt == 1);
        }
        if (ok) mma_commit_on(on, kv_empty + use % NST);
        ++use;
      }
      while (have && ok) {
        i += gridDim.x;
        const bool more = next_uniform(i, nx);
        for (int j = 0; ok && j < t.nt; ++j) {
          const bool last = j == t.nt - 1;
          const uint32_t uv = use, uk = use + 1;   // V of this tile, the K tile after it
          const int n = last ? (more ? width(nx, 0) : 0) : width(t, j + 1);
          const int nslots = n ? (last ? nx.nslots : t.nslots) : 0;   // slots whose next S uses uk
          const int steps = width(t, j) / 16;
          ok = tile_wait(uv);
          for (int s = 0; ok && s < max(t.nslots, nslots); ++s) {
            // everything that the next S needs first, so that it follows P V at once
            if (s < nslots) {
              if (s == 0) ok = tile_wait(uk);
              if (ok && last) ok = slot_wait(q_full, qph, s);
              if (!ok) break;
            }
            if (s < t.nslots) {
              if (j == 0) ok = slot_wait(o_empty, oph, s);
              ok = ok && slot_wait(p_part, hph, s);
              if (!ok) break;
              tc_fence_after();
              issue_pv(s, uv, 0, min(steps, 6), j > 0);
              ok = slot_wait(p_full, pph, s);
              if (!ok) break;
              tc_fence_after();
              issue_pv(s, uv, 6, steps, 1u);
              if (last) mma_commit_on(on, o_full + s);
            }
            if (s < nslots) issue_s(s, uk, n, last ? nx.nt == 1 : j + 2 == t.nt);
          }
          if (!ok) break;
          mma_commit_on(on, kv_empty + uv % NST);
          if (n) mma_commit_on(on, kv_empty + uk % NST);
          use += 2;
        }
        t = nx;
        have = more;
      }
      // MMAs in flight and their arrivals end before tensor memory is freed and
      // the CTA leaves
      volatile int never = 0;
      mma_commit_on(on, drain);
      mbar_wait(drain, 0, &never);
    } else if (warp == 10) {
      // ------------------------------------------------------------- cleaner
      if (clean) {
        uint32_t use = 0;
        bool ok = true;
        const auto pass = [&](bool got) {   // the tile may be used
          __syncwarp();
          if (got && lane == 0) mbar_arrive(ready + use % NST);
          ++use;
          return got;
        };
        const auto landed = [&]() { return all_lanes(mbar_wait(kv_full + use % NST, (use / NST) & 1u, abort_flag)); };
        XtItem t;
        for (int i = blockIdx.x; ok && next_item(i, t); i += gridDim.x) {
          for (int j = 0; ok && j < t.nt; ++j) {
            ok = pass(landed());   // a K tile
            ok = ok && landed();
            if (!ok) break;
            const uint32_t st = use % NST;
            {
              const int k0 = t.key0 + 128 * j;
              const int rows = min(128, (t.end - k0 + 15) / 16 * 16);   // rows that the MMA reads
              unsigned hide[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int key = k0 + 32 * q + lane;
                bool no = key >= t.end;
                if constexpr (BIAS) no = no || __ldg(a.x.bias + t.b * a.x.Lkp + key) == -INFINITY;
                hide[q] = __ballot_sync(0xffffffffu, no && 32 * q + lane < rows);
              }
              if (hide[0] | hide[1] | hide[2] | hide[3]) {
                uint8_t* tile = smem + C::OFF_KV + st * C::TILE;
                // lane: 16-byte chunk of a row; 8 chunks per panel
                const int sub = lane / (8 * C::PANELS), ch = lane % (8 * C::PANELS);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  if (hide[q])
                    for (int r = sub; r < 32; r += 32 / (8 * C::PANELS))
                      if ((hide[q] >> r) & 1u)
                        *reinterpret_cast<uint4*>(tile + (ch >> 3) * 16384 + (32 * q + r) * 128 + (ch & 7) * 16) =
                            make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async_smem();
              }
            }
            pass(true);
          }
        }
      }
    } else if (warp >= 12) {
      // ------------------------------------------------------------ epilogue
      const int w = warp & 3;
      const uint32_t lane_base = (uint32_t)(w * 32) << 16;
      const bool split = a.x.splits > 1;
      uint32_t ph[2] = {0, 0};
      bool ok = true;
      for (int i = blockIdx.x; ok && i < a.items; i += gridDim.x) {
        const XtItem t = xt_item(a, i);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (s >= t.nslots || !ok) continue;
          int h, l0;
          xt_slot(a, t, s, h, l0);
          const int row_in_tile = w * 32 + lane;
          const int64_t l = l0 + (row_in_tile >> a.pack_shift);
          h += row_in_tile & (a.packed - 1);
          float m = -INFINITY, sum = 0.f;
          if (t.nt) {
            ok = all_lanes(mbar_wait(l_full + s, ph[s], abort_flag));
            if (!ok) continue;
            const float2 v = ml[s * 128 + w * 32 + lane];
            m = v.x;
            sum = v.y;
            __syncwarp();
            if (lane == 0) mbar_arrive(l_empty + s);
            ok = all_lanes(mbar_wait(o_full + s, ph[s], abort_flag));
            if (!ok) continue;
            ph[s] ^= 1u;
            tc_fence_after();
          }
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          const uint64_t ii = two(inv, inv);
#pragma unroll 1
          for (int q = 0; 32 * q < a.x.D; ++q) {
            uint32_t o[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0u;
            if (t.nt) {
              tmem_ld32(tmem + 256 + s * 128 + lane_base + 32 * q, o);
              tmem_wait_ld();
              tie32(o);
            }
            if (l >= a.x.Lq) {
              // past the sample's rows
            } else if (split) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                if (32 * q + e < a.x.D) {
                  float v[8];
#pragma unroll
                  for (int f = 0; f < 8; ++f) v[f] = __uint_as_float(o[e + f]);
                  xattn_put<T>(a.x, t.b, l, h, t.split, 32 * q + e, v, m, sum);
                }
              }
            } else {
              T* row = reinterpret_cast<T*>(a.x.o) + t.b * a.x.os[0] + l * a.x.os[1] + h * a.x.os[2] + 32 * q;
#pragma unroll
              for (int e = 0; e < 32; e += 16) {
                uint32_t v[8];
#pragma unroll
                for (int f = 0; f < 8; ++f) {
                  float lo, hi;
                  untwo(mul2(two(__uint_as_float(o[e + 2 * f]), __uint_as_float(o[e + 2 * f + 1])), ii), lo, hi);
                  v[f] = pack16<T>(lo, hi);
                }
                if (a.wide) {
                  if (32 * q + e < a.x.D) st_global32(row + e, v);
                } else {
                  if (32 * q + e < a.x.D) *reinterpret_cast<uint4*>(row + e) = make_uint4(v[0], v[1], v[2], v[3]);
                  if (32 * q + e + 8 < a.x.D) *reinterpret_cast<uint4*>(row + e + 8) = make_uint4(v[4], v[5], v[6], v[7]);
                }
              }
            }
            __syncwarp();   // the next tcgen05.ld is the whole warp's
          }
          if (t.nt) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty + s);
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(XtCfg<DP>::REGS.many));
    // ------------------------------------------------------------- softmax
    const int s = warp >> 2, w = warp & 3;
    const uint32_t lane_base = (uint32_t)(w * 32) << 16;
    const uint32_t ts = tmem + s * 128 + lane_base, to = tmem + 256 + s * 128 + lane_base;
    const float c = a.x.scale * kLog2e;   // > 0: scores in units of log2 are S c
    uint32_t sn = 0, ln = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < a.items; i += gridDim.x) {
      const XtItem t = xt_item(a, i);
      if (s >= t.nslots || t.nt == 0) continue;
      float m = -INFINITY, sum = 0.f;
      for (int j = 0; j < t.nt; ++j) {
        const int k0 = t.key0 + 128 * j;
        const int rem = t.end - k0;          // keys of this tile (>= 128: all)
        ok = all_lanes(mbar_wait(s_full + s, sn & 1u, abort_flag));
        if (!ok) break;
        ++sn;
        tc_fence_after();
        uint32_t r[4][32];
        tmem_ld32(ts, r[0]);
        tmem_ld32(ts + 32, r[1]);
        tmem_wait_ld();
        tie32(r[0]);
        tie32(r[1]);
        tmem_ld32(ts + 64, r[2]);
        tmem_ld32(ts + 96, r[3]);
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const auto maxima = [&](int q) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            m4[2 * (q & 1)] = fmaxf(fmaxf(m4[2 * (q & 1)], __uint_as_float(r[q][e])), __uint_as_float(r[q][e + 1]));
            m4[2 * (q & 1) + 1] = fmaxf(fmaxf(m4[2 * (q & 1) + 1], __uint_as_float(r[q][e + 2])), __uint_as_float(r[q][e + 3]));
          }
        };
        if (!BIAS && rem >= 128) {
          maxima(0);
          maxima(1);
        }
        tmem_wait_ld();
        tie32(r[2]);
        tie32(r[3]);
        if (rem < 128) {
          // columns past the keys: whatever the tile held
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t keep = rem >= 32 * q + 32 ? 0xffffffffu : rem <= 32 * q ? 0u : (1u << (rem - 32 * q)) - 1u;
#pragma unroll
            for (int e = 0; e < 32; ++e) r[q][e] = (keep >> e) & 1u ? r[q][e] : 0xff800000u;   // -inf
          }
          if constexpr (!BIAS) {
            maxima(0);
            maxima(1);
          }
        }
        float mx;
        if constexpr (BIAS) {
          const float4* bias = reinterpret_cast<const float4*>(a.x.bias + t.b * a.x.Lkp + k0);
          mx = -INFINITY;
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 b4 = __ldg(bias + 8 * q + e / 4);
              const float bb[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
              for (int f = 0; f < 4; ++f) {
                const float x = bb[f] == -INFINITY ? -INFINITY : fmaf(__uint_as_float(r[q][e + f]), c, bb[f]);
                r[q][e + f] = __float_as_uint(x);
                mx = fmaxf(mx, x);
              }
            }
        } else {
          maxima(2);
          maxima(3);
          mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        }
        if constexpr (!BIAS) mx *= c;
        // (P V of the tile before is done: this S was issued behind it)
        if (__any_sync(0xffffffffu, xattn_moves<T>(mx, m))) {
          const float nm = xattn_moves<T>(mx, m) ? mx - kXattnUp<T> : m;
          const float f = nm == m ? 1.f : ex2(m - nm);
          m = nm;
          sum *= f;
          if (j > 0) {
#pragma unroll 1
            for (int q = 0; 16 * q < a.x.D; ++q) {
              uint32_t o[16];
              tmem_ld16(to + 16 * q, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                asm volatile("" : "+r"(o[e]));   // valid after the wait
                o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              }
              tmem_st16(to + 16 * q, o);
            }
            tmem_wait_st();
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const uint64_t cc = two(BIAS ? 1.f : c, BIAS ? 1.f : c), rr = two(-ref, -ref);
        uint64_t add[2] = {two(sum, 0.f), two(0.f, 0.f)};
        // 32 columns at a time; a block's exponentials are issued ahead of the
        // sums and the packing of the block before, which fill their latency
        const auto finish = [&](int q) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float p0 = __uint_as_float(r[q][e]), p1 = __uint_as_float(r[q][e + 1]);
            add[(e >> 1) & 1] = add2(add[(e >> 1) & 1], two(p0, p1));
            p[e / 2] = pack16<T>(p0, p1);
          }
          tmem_st16(ts + 16 * q, p);
          if (q >= 2) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive((q == 3 ? p_full : p_part) + s);
          }
        };
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const uint64_t x = fma2(two(__uint_as_float(r[q][e]), __uint_as_float(r[q][e + 1])), cc, rr);
            float p0, p1;
            untwo(x, p0, p1);
            r[q][e] = __float_as_uint(ex2(p0));
            r[q][e + 1] = __float_as_uint(ex2(p1));
          }
          if (q > 0) finish(q - 1);
        }
        finish(3);
        float s0, s1;
        untwo(add2(add[0], add[1]), s0, s1);
        sum = s0 + s1;
      }
      if (!ok) break;
      ok = all_lanes(mbar_wait(l_empty + s, (ln & 1u) ^ 1u, abort_flag));
      if (!ok) break;
      ++ln;
      ml[s * 128 + w * 32 + lane] = make_float2(m, sum);
      __syncwarp();
      if (lane == 0) mbar_arrive(l_full + s);
    }
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- host side
// [elements, heads, tokens, batch] of a strided tensor.  A stride of 0 is one
// entry that every coordinate maps to; a dimension of one entry takes any
// stride.
static bool xt_map(CUtensorMap* m, bool bf, const void* p, const int64_t* st, int64_t D, int64_t heads, int64_t tokens,
                   int64_t batch, int box_heads, int* mul) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  mul[0] = st[0] == 0 ? 0 : 1;
  mul[1] = st[2] == 0 ? 0 : 1;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)(mul[1] ? heads : 1), (cuuint64_t)tokens,
                        (cuuint64_t)(mul[0] ? batch : 1)};
  const int64_t el[3] = {st[2], st[1], st[0]};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) strides[i] = dims[i + 1] == 1 ? 16 * ((cuuint64_t)D / 8) : (cuuint64_t)el[i] * 2;
  cuuint32_t box[4] = {64, (cuuint32_t)box_heads, (cuuint32_t)(128 / box_heads), 1};
  cuuint32_t one[4] = {1, 1, 1, 1};
  return fn(m, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(p), dims,
            strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, bool BIAS>
static cudaError_t launch_xt(const CUtensorMap (&m)[3], const XtArgs& a, cudaStream_t st) {
  auto kern = xattn_tc_kernel<T, DP, BIAS>;
  static std::atomic<unsigned long long> devices{0};
  cudaError_t e = set_smem_once(kern, XtCfg<DP>::SMEM);
  if (e == cudaSuccess) e = split_fits_once(kern, XtCfg<DP>::REGS, devices);
  if (e != cudaSuccess) return e;
  const int grid = a.items < num_sms() ? a.items : num_sms();
  kern<<<grid, XtCfg<DP>::THREADS, XtCfg<DP>::SMEM, st>>>(m[0], m[1], m[2], a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_xattn_tc(const XattnArgs& x, int slots, cudaStream_t st) {
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  XtArgs a;
  a.x = x;
  a.slots = slots;
  a.group = x.H / x.Hk;
  a.packed = x.qs[2] != 0 ? xattn_packed(x.H, x.Hk) : 1;
  for (a.pack_shift = 0; (1 << a.pack_shift) < a.packed;) ++a.pack_shift;
  a.tiles_per_head = (int)((x.Lq * a.packed + 127) / 128);
  const int64_t tiles = (int64_t)(a.group / a.packed) * a.tiles_per_head;
  const int64_t per_head = (tiles + slots - 1) / slots;
  const int64_t items = x.B * x.Hk * per_head * x.splits;
  if (items + num_sms() >= (1 << 30) || tiles >= (1 << 30)) return cudaErrorInvalidValue;
  a.tiles = (int)tiles;
  a.items = (int)items;
  a.wide = x.D % 16 == 0 && (reinterpret_cast<uintptr_t>(x.o) & 31) == 0 && x.os[0] % 16 == 0 && x.os[1] % 16 == 0 &&
           x.os[2] % 16 == 0;
  a.by_split = xt_div((uint32_t)x.splits);
  a.by_head = xt_div((uint32_t)per_head);
  a.by_hk = xt_div((uint32_t)x.Hk);
  a.by_tiles = xt_div((uint32_t)a.tiles_per_head);
  CUtensorMap m[3];
  if (!xt_map(&m[0], BF, x.q, x.qs, x.D, x.H, x.Lq, x.B, a.packed, a.qm) ||
      !xt_map(&m[1], BF, x.k, x.ks, x.D, x.Hk, x.Lk, x.B, 1, a.km) ||
      !xt_map(&m[2], BF, x.v, x.vs, x.D, x.Hk, x.Lk, x.B, 1, a.vm))
    return cudaErrorInvalidValue;
  if (x.D <= 64) return x.bias ? launch_xt<T, 64, true>(m, a, st) : launch_xt<T, 64, false>(m, a, st);
  return x.bias ? launch_xt<T, 128, true>(m, a, st) : launch_xt<T, 128, false>(m, a, st);
}

}  // namespace ic
