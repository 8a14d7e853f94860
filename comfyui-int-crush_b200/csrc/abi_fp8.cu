// extern "C" entry points of the 8-bit floating point linear (declared in
// include/intcrush_b200.h).  Each validates its arguments, launches on the
// caller's stream and returns a status code; no exception crosses the ABI.
#include <string.h>

#include <utility>

namespace ic {

cudaError_t fp8_device_error(int* word, bool store) {
  return store ? cudaMemcpyToSymbol(g_ic_dev_error, word, sizeof(int)) : cudaMemcpyFromSymbol(word, g_ic_dev_error, sizeof(int));
}

static int f8_launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return IC_OK;
  return set_error(IC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
static bool f8_at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool f8_float(int dtype) { return dtype == IC_DTYPE_F16 || dtype == IC_DTYPE_BF16 || dtype == IC_DTYPE_F32; }
// a code of a sizes structure; what no int holds is no code
static int f8_code(int64_t v) { return v == (int)v ? (int)v : -1; }
static int64_t f8_up(int64_t n, int64_t m) { return (n + m - 1) / m; }

constexpr int64_t kF8Rows = 0x7fffffffLL - 1024;   // row and column numbers are 32-bit in the kernels
constexpr int64_t kF8Stride = 1LL << 38;           // of a tensor map

}  // namespace ic

extern "C" {

int ic_quantize_fp8_block(const void* x, void* q, float* s, const ic_quantize_fp8_sizes* sizes, void* stream) {
  using namespace ic;
  const char* me = "ic_quantize_fp8_block";
  clear_error();
  if (!sizes) return set_error(IC_ERR_ARG, "%s: sizes is NULL", me);
  const int64_t M = sizes->M, K = sizes->K, ldx = sizes->ldx, ldq = sizes->ldq, s_row = sizes->s_row, s_block = sizes->s_block;
  const int dtype = f8_code(sizes->dtype), rows = f8_code(sizes->rows);
  if (!f8_float(dtype)) return set_error(IC_ERR_ARG, "%s: dtype must be f16, bf16 or f32", me);
  if (M < 0 || K <= 0 || ldx < K) return set_error(IC_ERR_ARG, "%s: bad M/K/ldx (%lld, %lld, %lld)", me, (long long)M, (long long)K, (long long)ldx);
  if (rows != 1 && rows != 128) return set_error(IC_ERR_ARG, "%s: rows of a block must be 1 or 128, got %d", me, rows);
  if (M == 0) return IC_OK;
  if (!x || !q || !s) return set_error(IC_ERR_ARG, "%s: NULL tensor", me);
  const int64_t width = f8_up(K, 16) * 16;
  if (ldq < width || ldq % 16 || !f8_at16(q))
    return set_error(IC_ERR_ARG, "%s: q must be 16-byte aligned, its row stride a multiple of 16 and at least %lld", me, (long long)width);
  const int es = dtype == IC_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % es) return set_error(IC_ERR_ARG, "%s: x is not aligned to its type", me);
  const int64_t kb = f8_up(K, 128);
  if (M > kF8Rows || K > kF8Rows || f8_up(M, 4) * kb > (1LL << 33) || (rows == 128 && f8_up(M, 128) > 65535))
    return set_error(IC_ERR_UNSUPPORTED, "%s: too many blocks for one launch", me);
  F8QuantArgs a;
  memset(&a, 0, sizeof(a));
  a.x = x; a.M = M; a.ldx = ldx; a.K = (int)K; a.kb = (int)kb; a.width = (int)width;
  a.q = static_cast<uint8_t*>(q); a.ldq = ldq; a.s = s; a.s_row = s_row; a.s_block = s_block;
  a.vec = f8_at16(x) && K % (16 / es) == 0 && (ldx % (16 / es) == 0 || M == 1);
  return f8_launched(launch_quant_fp8(a, dtype, rows, (cudaStream_t)stream), "ic_quantize_fp8_block launch");
}

int ic_gemm_fp8_block(const void* x, const void* w, const float* s_a, const float* s_w, const void* bias, void* out,
                      const ic_gemm_fp8_sizes* sizes, void* stream) {
  using namespace ic;
  const char* me = "ic_gemm_fp8_block";
  clear_error();
  if (!sizes) return set_error(IC_ERR_ARG, "%s: sizes is NULL", me);
  const int64_t M = sizes->M, K = sizes->K, N = sizes->N, ldx = sizes->ldx, ldw = sizes->ldw, ldo = sizes->ldo;
  const int bias_dtype = f8_code(sizes->bias_dtype), out_dtype = f8_code(sizes->out_dtype);
  if (M < 0 || N < 0 || K <= 0) return set_error(IC_ERR_ARG, "%s: bad M/N/K (%lld, %lld, %lld)", me, (long long)M, (long long)N, (long long)K);
  if (!f8_float(out_dtype) || (bias && !f8_float(bias_dtype)))
    return set_error(IC_ERR_ARG, "%s: out and bias must be f16, bf16 or f32", me);
  if (ldx < K || ldw < K || ldo < N) return set_error(IC_ERR_ARG, "%s: a row stride is shorter than its row", me);
  if (M == 0 || N == 0) return IC_OK;
  if (!x || !w || !s_a || !s_w || !out) return set_error(IC_ERR_ARG, "%s: NULL tensor", me);
  if (!f8_at16(x) || !f8_at16(w) || ldx % 16 || ldw % 16)
    return set_error(IC_ERR_ARG, "%s: x and w must be 16-byte aligned with row strides that are multiples of 16", me);
  const int es = out_dtype == IC_DTYPE_F32 ? 4 : 2, bs = bias_dtype == IC_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(out) % es || (bias && reinterpret_cast<uintptr_t>(bias) % bs))
    return set_error(IC_ERR_ARG, "%s: out or bias is not aligned to its type", me);
  if (M > kF8Rows || N > kF8Rows || K > kF8Rows || ldx >= kF8Stride || ldw >= kF8Stride || ldo >= kF8Stride ||
      f8_up(M, 128) * f8_up(N, 128) > (1LL << 30))
    return set_error(IC_ERR_UNSUPPORTED, "%s: size too large", me);
  F8Operands o = {x, w, M, K, N, ldx, ldw};
  F8Args a;
  memset(&a, 0, sizeof(a));
  a.M = (int)M; a.N = (int)N; a.kb = (int)f8_up(K, 128);
  a.s_a = s_a; a.sa_row = sizes->sa_row; a.sa_block = sizes->sa_block;
  a.s_w = s_w; a.sw_row = sizes->sw_row; a.sw_block = sizes->sw_block;
  a.bias = bias; a.bias_dtype = bias_dtype; a.out = out; a.out_dtype = out_dtype; a.ldo = ldo;
  return f8_launched(launch_gemm_fp8(o, a, (cudaStream_t)stream), "ic_gemm_fp8_block launch");
}

static int gn_sizes(const char* me, int64_t B, int64_t L, int64_t C, int64_t groups) {
  using namespace ic;
  if (B < 0 || L < 0 || C <= 0 || groups <= 0 || C % groups)
    return set_error(IC_ERR_ARG, "%s: bad sizes: batch %lld, rows %lld, %lld channels in %lld groups", me, (long long)B,
                     (long long)L, (long long)C, (long long)groups);
  if (C > 8192) return set_error(IC_ERR_UNSUPPORTED, "%s: at most 8192 channels, got %lld", me, (long long)C);
  if (B > (1LL << 24) || L > kF8Rows || B * L > (1LL << 33)) return set_error(IC_ERR_UNSUPPORTED, "%s: too many rows for one launch", me);
  return IC_OK;
}

// Whether two of n x m runs of `width` elements, `far` and `near` apart, share one.
static bool gn_overlap(int64_t n, int64_t far, int64_t m, int64_t near, int64_t width) {
  if (n == 1 || m == 1) return (n > 1 && far < width) || (m > 1 && near < width);
  if (near > far) {
    std::swap(n, m);
    std::swap(far, near);
  }
  if (near < width) return true;
  const __int128 last = (__int128)(m - 1) * near;   // (any strides are let in here)
  for (int64_t j = 1; j < n && (__int128)j * far < last + width; ++j) {
    const __int128 at = (__int128)j * far, i = at / near, r = at - i * near;
    if ((i < m && r < width) || (i + 1 < m && near - r < width)) return true;
  }
  return false;
}

int64_t ic_group_norm_workspace(int64_t B, int64_t L, int64_t C, int64_t groups, int quantize) {
  if (gn_sizes("ic_group_norm_workspace", B, L, C, groups) != IC_OK) return -1;
  return B && L ? ic::gn_plan(B, L, C, groups, quantize != 0).floats : 0;
}

int ic_group_norm(const void* x, const void* gamma, const void* beta, float eps, void* y, void* q, float* s, float* workspace,
                  const ic_group_norm_sizes* sizes, void* stream) {
  using namespace ic;
  const char* me = "ic_group_norm";
  clear_error();
  if (!sizes) return set_error(IC_ERR_ARG, "%s: sizes is NULL", me);
  const int64_t B = sizes->B, L = sizes->L, C = sizes->C, groups = sizes->groups, x_batch = sizes->x_batch, x_row = sizes->x_row;
  const int64_t y_batch = sizes->y_batch, y_row = sizes->y_row, ldq = sizes->ldq, workspace_elems = sizes->floats;
  const int dtype = f8_code(sizes->dtype), activation = f8_code(sizes->activation);
  const int gamma_dtype = f8_code(sizes->gamma_dtype), beta_dtype = f8_code(sizes->beta_dtype);
  if (dtype != IC_DTYPE_F16 && dtype != IC_DTYPE_BF16) return set_error(IC_ERR_ARG, "%s: dtype must be f16 or bf16", me);
  const int bad = gn_sizes(me, B, L, C, groups);
  if (bad != IC_OK) return bad;
  if ((gamma && !f8_float(gamma_dtype)) || (beta && !f8_float(beta_dtype)))
    return set_error(IC_ERR_ARG, "%s: gamma and beta must be f16, bf16 or f32", me);
  if (activation < 0 || activation > 3) return set_error(IC_ERR_ARG, "%s: activation must be 0..3, got %d", me, activation);
  if (!(eps >= 0.f)) return set_error(IC_ERR_ARG, "%s: eps must not be negative", me);
  if (B == 0 || L == 0) return IC_OK;
  if (!x || (!y == !q) || (q && !s)) return set_error(IC_ERR_ARG, "%s: NULL tensor: one of y and q (with s) is written", me);
  if (x_batch < 0 || x_row < C || (y && (y_batch < 0 || y_row < C)))
    return set_error(IC_ERR_ARG, "%s: a row stride is shorter than its row", me);
  if (y && B > 1 && y_batch < C) return set_error(IC_ERR_ARG, "%s: y overlaps itself", me);
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 1)
    return set_error(IC_ERR_ARG, "%s: x or y is not aligned to its type", me);
  const auto off = [](const void* p, int dt) { return reinterpret_cast<uintptr_t>(p) % (dt == IC_DTYPE_F32 ? 4 : 2) != 0; };
  if ((gamma && off(gamma, gamma_dtype)) || (beta && off(beta, beta_dtype)))
    return set_error(IC_ERR_ARG, "%s: gamma or beta is not aligned to its type", me);
  const int64_t width = f8_up(C, 16) * 16;
  if (q && (ldq < width || ldq % 16 || !f8_at16(q)))
    return set_error(IC_ERR_ARG, "%s: q must be 16-byte aligned, its row stride a multiple of 16 and at least %lld", me, (long long)width);
  const GnPlan p = gn_plan(B, L, C, groups, q != nullptr);
  if (p.floats && (!workspace || !f8_at16(workspace) || workspace_elems < p.floats))
    return set_error(IC_ERR_ARG, "%s: needs a 16-byte aligned workspace of %lld floats, got %lld", me, (long long)p.floats,
                     (long long)workspace_elems);
  if (y && gn_overlap(B, y_batch, L, y_row, C)) return set_error(IC_ERR_ARG, "%s: y overlaps itself", me);
  GnArgs a;
  memset(&a, 0, sizeof(a));
  a.x = x; a.L = L; a.C = (int)C; a.G = (int)groups; a.Cg = (int)(C / groups);
  a.x_batch = x_batch; a.x_row = x_row;
  a.vec = C % 8 == 0 && f8_at16(x) && x_row % 8 == 0 && (x_batch % 8 == 0 || B == 1) &&
          (!y || (f8_at16(y) && y_row % 8 == 0 && (y_batch % 8 == 0 || B == 1)));
  a.gamma = gamma; a.gamma_dtype = gamma_dtype; a.beta = beta; a.beta_dtype = beta_dtype;
  a.eps = eps;
  a.y = y; a.y_batch = y_batch; a.y_row = y_row;
  a.q = static_cast<uint8_t*>(q); a.ldq = ldq; a.s = s; a.s_row = sizes->s_row; a.s_block = sizes->s_block; a.width = (int)width;
  a.part = reinterpret_cast<float2*>(workspace);
  return f8_launched(launch_group_norm(a, p, B, dtype, activation, (cudaStream_t)stream), "ic_group_norm launch");
}

}  // extern "C"
