// extern "C" entry points of the attention-side operators (declared in
// include/intcrush_b200.h).  Each validates its arguments, launches on the
// caller's stream and returns a status code; no exception crosses the ABI.
#include <string.h>

namespace ic {

cudaError_t attention_device_error(int* word, bool store) {
  return store ? cudaMemcpyToSymbol(g_ic_dev_error, word, sizeof(int)) : cudaMemcpyFromSymbol(word, g_ic_dev_error, sizeof(int));
}

static int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return IC_OK;
  return set_error(IC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

static bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool is16(int dtype) { return dtype == IC_DTYPE_F16 || dtype == IC_DTYPE_BF16; }

// A tensor of 16-bit heads that is read or written 16 bytes at a time.
static bool head_layout_ok(const void* p, const int64_t* strides) {
  return at16(p) && strides[0] % 8 == 0 && strides[1] % 8 == 0 && strides[2] % 8 == 0;
}

}  // namespace ic

extern "C" {

int ic_qk_norm_rope(const void* q, void* q_out, int64_t H, const void* k, void* k_out, int64_t Hk, int dtype,
                    int64_t B, int64_t L, int64_t D, const int64_t* strides, const float* q_gamma,
                    const float* k_gamma, float eps, int layout, int64_t rot, const float* cos_table,
                    const float* sin_table, int64_t table_rows, const int32_t* positions, void* stream) {
  using namespace ic;
  const char* me = "ic_qk_norm_rope";
  clear_error();
  if (!is16(dtype)) return set_error(IC_ERR_ARG, "%s: dtype must be f16 or bf16", me);
  if (B < 0 || L < 0 || H < 0 || Hk < 0) return set_error(IC_ERR_ARG, "%s: negative size", me);
  if (D <= 0 || D % 8 || D > 256)
    return set_error(IC_ERR_UNSUPPORTED, "%s: head size must be a multiple of 8 up to 256, got %lld", me, (long long)D);
  if (rot < 0 || rot > D || rot % 2)
    return set_error(IC_ERR_ARG, "%s: rot must be even and in [0, %lld], got %lld", me, (long long)D, (long long)rot);
  if (layout != IC_ROPE_INTERLEAVED && layout != IC_ROPE_HALF)
    return set_error(IC_ERR_ARG, "%s: layout must be 0 (interleaved) or 1 (half)", me);
  if (!strides) return set_error(IC_ERR_ARG, "%s: strides is NULL", me);
  if (B == 0 || L == 0 || H + Hk == 0) return IC_OK;
  if ((H && (!q || !q_out)) || (Hk && (!k || !k_out))) return set_error(IC_ERR_ARG, "%s: NULL tensor", me);
  if (rot && (!cos_table || !sin_table)) return set_error(IC_ERR_ARG, "%s: a rotation needs cos and sin tables", me);
  if (rot && !positions && table_rows < L)
    return set_error(IC_ERR_ARG, "%s: %lld table rows for %lld tokens", me, (long long)table_rows, (long long)L);
  if (rot && table_rows <= 0) return set_error(IC_ERR_ARG, "%s: empty tables", me);
  const void* xs[2] = {q, k};
  void* ys[2] = {q_out, k_out};
  const float* gs[2] = {q_gamma, k_gamma};
  QkArgs a;
  memset(&a, 0, sizeof(a));
  const int64_t hs[2] = {H, Hk};
  for (int i = 0; i < 2; ++i) {
    if (!hs[i]) continue;
    if (!head_layout_ok(xs[i], strides + 6 * i) || !head_layout_ok(ys[i], strides + 6 * i + 3) || !at16(gs[i]))
      return set_error(IC_ERR_ARG, "%s: tensors and gammas must be 16-byte aligned, strides multiples of 8", me);
    if (hs[i] > 65536) return set_error(IC_ERR_UNSUPPORTED, "%s: more than 65536 heads", me);
    a.x[i] = xs[i];
    a.y[i] = ys[i];
    a.gamma[i] = gs[i];
    a.heads[i] = (int)hs[i];
    for (int j = 0; j < 3; ++j) {
      a.xs[i][j] = strides[6 * i + j];
      a.ys[i][j] = strides[6 * i + 3 + j];
    }
  }
  // units of a launch: 16 heads of a token at least, or one head when there
  // are few
  if (B > (1LL << 30) / L || B * L > (1LL << 30) / ((H + 15) / 16 + (Hk + 15) / 16))
    return set_error(IC_ERR_UNSUPPORTED, "%s: too many rows for one launch", me);
  a.B = B;
  a.Lq = L;
  a.D = (int)D;
  a.rot = (int)rot;
  a.eps = eps;
  a.cosp = cos_table;
  a.sinp = sin_table;
  a.table = table_rows;
  a.positions = rot ? positions : nullptr;
  return launched(launch_qk_norm_rope(a, dtype, layout, (cudaStream_t)stream), "ic_qk_norm_rope launch");
}

static int lora_sizes(const char* me, int64_t M, int64_t K, int64_t N, int64_t R, int64_t n) {
  using namespace ic;
  if (M < 0 || N < 0 || K <= 0 || n <= 0) return set_error(IC_ERR_ARG, "%s: bad M/K/N/adapters (%lld, %lld, %lld, %lld)", me,
                                                          (long long)M, (long long)K, (long long)N, (long long)n);
  if (R < 1 || R > 256) return set_error(IC_ERR_UNSUPPORTED, "%s: rank must be 1..256, got %lld", me, (long long)R);
  if (M > 0x7fffffffLL || K > 0x7fffffffLL || N > 65535LL * 256 || n > 0x7fffffffLL)
    return set_error(IC_ERR_UNSUPPORTED, "%s: size too large", me);
  return IC_OK;
}

int64_t ic_lora_batched_workspace(int64_t M, int64_t K, int64_t N, int64_t R, int64_t n) {
  if (lora_sizes("ic_lora_batched_workspace", M, K, N, R, n) != IC_OK) return -1;
  return M ? ic::lora_workspace(M, K, N, (int)R, (int)n) : 0;
}

int ic_lora_batched(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* down, const void* up,
                    int64_t R, int64_t n, const int32_t* ids, int64_t rows_per_id, const float* scales,
                    const void* base, int64_t ldb, void* out, int64_t N, int64_t ldo, float* workspace,
                    int64_t workspace_elems, void* stream) {
  using namespace ic;
  const char* me = "ic_lora_batched";
  clear_error();
  if (!is16(dtype)) return set_error(IC_ERR_ARG, "%s: dtype must be f16 or bf16", me);
  const int bad = lora_sizes(me, M, K, N, R, n);
  if (bad != IC_OK) return bad;
  if (rows_per_id <= 0) return set_error(IC_ERR_ARG, "%s: rows_per_id must be positive", me);
  if (rows_per_id > 0x7fffffffLL) rows_per_id = 0x7fffffffLL;   // M is below that
  if (ldx < K || ldo < N || (base && ldb < N))
    return set_error(IC_ERR_ARG, "%s: a row stride is shorter than its row", me);
  if (M == 0 || N == 0) return IC_OK;
  if (!x || !down || !up || !ids || !out) return set_error(IC_ERR_ARG, "%s: NULL tensor", me);
  if (!workspace || !at16(workspace) || workspace_elems < lora_workspace(M, K, N, (int)R, (int)n))
    return set_error(IC_ERR_ARG, "%s: needs a 16-byte aligned workspace of %lld floats, got %lld", me,
                     (long long)lora_workspace(M, K, N, (int)R, (int)n), (long long)workspace_elems);
  LoraArgs a;
  memset(&a, 0, sizeof(a));
  a.x = x; a.ldx = ldx; a.M = M; a.K = K; a.N = N;
  a.R = (int)R; a.Rp = ((int)R + 7) / 8 * 8;
  a.down = down; a.up = up; a.ids = ids; a.rows_per_id = rows_per_id; a.scales = scales; a.n = (int)n;
  a.base = base; a.ldb = ldb; a.out = out; a.ldo = ldo; a.mid = workspace;
  return launched(launch_lora_batched(a, dtype, (cudaStream_t)stream), "ic_lora_batched launch");
}

static int xattn_sizes(const char* me, int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D,
                       int mask_kind) {
  using namespace ic;
  if (B < 0 || Lq < 0 || Lk < 0 || H <= 0 || Hk <= 0 || H % Hk)
    return set_error(IC_ERR_ARG, "%s: bad sizes: batch %lld, queries %lld, keys %lld, heads %lld over %lld", me,
                     (long long)B, (long long)Lq, (long long)Lk, (long long)H, (long long)Hk);
  if (D <= 0 || D % 8 || D > 128)
    return set_error(IC_ERR_UNSUPPORTED, "%s: head size must be a multiple of 8 up to 128, got %lld", me, (long long)D);
  if (mask_kind < IC_MASK_NONE || mask_kind > IC_MASK_F32)
    return set_error(IC_ERR_ARG, "%s: mask kind %d", me, mask_kind);
  if (H > 65536 || Lq > (1LL << 30) || Lk > (1LL << 30) || B > (1LL << 30) || B * H > (1LL << 30) ||
      (Lq + 16) * H > (1LL << 40) / (B + 1))
    return set_error(IC_ERR_UNSUPPORTED, "%s: too many rows for one launch", me);
  return IC_OK;
}

int64_t ic_cross_attention_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D,
                                     int mask_kind) {
  if (xattn_sizes("ic_cross_attention_workspace", B, Lq, Lk, H, Hk, D, mask_kind) != IC_OK) return -1;
  return B && Lq ? ic::xattn_plan(B, Lq, Lk, (int)H, (int)Hk, (int)D, mask_kind).floats : 0;
}

int ic_cross_attention(const void* q, const void* k, const void* v, void* out, int dtype, int64_t B, int64_t Lq,
                       int64_t Lk, int64_t H, int64_t Hk, int64_t D, const int64_t* strides, float scale,
                       const int32_t* kv_lens, const void* mask, int mask_kind, int64_t ld_mask, float* workspace,
                       int64_t workspace_elems, void* stream) {
  using namespace ic;
  const char* me = "ic_cross_attention";
  clear_error();
  if (!is16(dtype)) return set_error(IC_ERR_ARG, "%s: dtype must be f16 or bf16", me);
  const int bad = xattn_sizes(me, B, Lq, Lk, H, Hk, D, mask_kind);
  if (bad != IC_OK) return bad;
  if (!strides) return set_error(IC_ERR_ARG, "%s: strides is NULL", me);
  if (B == 0 || Lq == 0) return IC_OK;
  if (!q || !out || (Lk && (!k || !v)) || (mask_kind && Lk && !mask)) return set_error(IC_ERR_ARG, "%s: NULL tensor", me);
  if (mask_kind && ld_mask != 0 && ld_mask < Lk) return set_error(IC_ERR_ARG, "%s: ld_mask < keys", me);
  if (!head_layout_ok(q, strides) || !head_layout_ok(out, strides + 9) ||
      (Lk && (!head_layout_ok(k, strides + 3) || !head_layout_ok(v, strides + 6))))
    return set_error(IC_ERR_ARG, "%s: tensors must be 16-byte aligned, strides multiples of 8", me);
  for (int i = 0; i < 12; ++i) {
    const int64_t tokens = i < 3 || i >= 9 ? Lq : Lk;
    if (strides[i] < 0 || strides[i] >= (1LL << 38))
      return set_error(IC_ERR_ARG, "%s: strides must be in [0, 2^38)", me);
    if (i % 3 == 1 && strides[i] == 0 && tokens > 1)
      return set_error(IC_ERR_ARG, "%s: a token stride of 0 with more than one token", me);
    if (strides[i] == 0 && ((i == 9 && B > 1) || (i == 11 && H > 1)))
      return set_error(IC_ERR_ARG, "%s: out overlaps itself", me);
  }
  const XattnPlan p = xattn_plan(B, Lq, Lk, (int)H, (int)Hk, (int)D, mask_kind);
  if (p.floats && (!workspace || !at16(workspace) || workspace_elems < p.floats))
    return set_error(IC_ERR_ARG, "%s: needs a 16-byte aligned workspace of %lld floats, got %lld", me,
                     (long long)p.floats, (long long)workspace_elems);
  XattnArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q; a.k = k; a.v = v; a.o = out;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = strides[i];
    a.ks[i] = strides[3 + i];
    a.vs[i] = strides[6 + i];
    a.os[i] = strides[9 + i];
  }
  a.B = B; a.Lq = Lq; a.Lk = Lk; a.H = (int)H; a.Hk = (int)Hk; a.D = (int)D;
  a.scale = scale;
  a.kv_lens = kv_lens;
  return launched(launch_cross_attention(a, dtype, mask, mask_kind, ld_mask, workspace, (cudaStream_t)stream),
                  "ic_cross_attention launch");
}

}  // extern "C"
