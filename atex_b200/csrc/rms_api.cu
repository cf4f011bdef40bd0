// C ABI of the RMS normalisation and of the residual norms' gradients: argument checks, the
// choice of a kernel, workspace carving and the launches (include/nvnorms.h).
//
// The reference normalises by mean and variance only and leaves the residual stream to
// separate TensorFlow ops (atex/nv_norms/python/ops/nv_norm_ops.py:85-99); these entry points
// have no counterpart there.
#include "../../include/nvnorms.h"
#include "nvn_host.h"

namespace nvn {

namespace {

struct Shape {
  int capacity, pf, forms;
};
#define X(I, TPR, VPT, RB, MINB, PF, FORMS) {TPR * VPT, PF, FORMS},
const Shape kFwdShapes[] = {NVN_RMS_FWD_SHAPES(X)};
const Shape kBwdShapes[] = {NVN_RMS_BWD_SHAPES(X)};
const Shape kNarrowShapes[] = {NVN_RMS_NARROW_SHAPES(X)};
#undef X

// Smallest shape of the form that holds `nvec` accesses, or -1; held rings only for large tensors
// unless nothing else fits.
int pick(const Shape* table, int n, int form, int64_t nvec, int64_t tensor_bytes) {
  int best = -1;
  for (int pass = 0; pass < 2 && best < 0; ++pass)
    for (int i = 0; i < n; ++i) {
      const Shape& t = table[i];
      if ((t.forms >> form & 1) == 0 || t.capacity < nvec) continue;
      if (pass == 0 && t.pf >= 10 && tensor_bytes < kRmsHeldMinBytes) continue;
      if (best < 0 || t.capacity < table[best].capacity) best = i;
    }
  return best;
}

typedef cudaError_t (*RowsRmsFn)(int, int, int, const RowsResArgs&, cudaStream_t, bool, RowsPlan*);
RowsRmsFn rows_rms_fn(int dtype, bool bwd) {
  if (dtype == NVN_F32) return bwd ? rows_rms_f32_bwd : rows_rms_f32_fwd;
  if (dtype == NVN_F16) return bwd ? rows_rms_f16_bwd : rows_rms_f16_fwd;
  return bwd ? rows_rms_bf16_bwd : rows_rms_bf16_fwd;
}

struct Plan {
  int epv, shape;        // shape < 0: the kernels for any width
  int64_t partial_rows;  // backward
  size_t off_coef, bytes;
};

int plan(int form, int dtype, bool bwd, int64_t N, int64_t D, size_t align, size_t par_align, Plan* p) {
  const bool rms = !bwd || form != 2;
  const int NR = rms ? 1 : 2;
  *p = {};
  p->epv = pick_epv(dtype, D, align, par_align);
  const bool full = p->epv == full_epv(dtype);
  const int64_t tensor_bytes = N * D * static_cast<int64_t>(dtype_size(dtype));
  const Shape* table = !full ? kNarrowShapes : (bwd ? kBwdShapes : kFwdShapes);
  const size_t count = !full ? sizeof(kNarrowShapes) : (bwd ? sizeof(kBwdShapes) : sizeof(kFwdShapes));
  p->shape = pick(table, static_cast<int>(count / sizeof(Shape)), form, D / p->epv, tensor_bytes);
  if (!bwd) return NVN_OK;
  if (p->shape >= 0) {
    RowsResArgs a = {};
    a.N = N;
    a.D = D;
    RowsPlan rp;
    const cudaError_t e = rows_rms_fn(dtype, true)(form, p->epv, p->shape, a, nullptr, true, &rp);
    if (e != cudaSuccess) return fail_cuda(e);
    p->partial_rows = rp.partial_rows;
  } else {
    if (!full) p->epv = 1;
    p->partial_rows = generic_slices(N, D, p->epv);
  }
  p->off_coef = align_up(static_cast<size_t>(p->partial_rows) * NR * D * 4, 256);
  p->bytes = p->off_coef + (p->shape < 0 ? align_up(static_cast<size_t>(N) * NR * 4, 256) : 0);
  return NVN_OK;
}

// The access width, hence the plan, depends on the alignment the call arrives with.
size_t workspace(int form, int dtype, int64_t N, int64_t D) {
  if (!valid_dtype(dtype) || N <= 0 || D <= 0) return 0;
  size_t most = 0;
  Plan p;
  for (size_t al : {size_t(16), size_t(8), size_t(4), size_t(2)})
    if (plan(form, dtype, true, N, D, al, 16, &p) == NVN_OK && p.bytes > most) most = p.bytes;
  return most;
}

int forward(int dtype, const void* x, const void* residual, const float* gamma, int64_t N, int64_t D,
            float eps, void* sum_out, void* y, float* inv_rms, cudaStream_t s) {
  RowsResArgs a = {};
  a.x = x;
  a.res = residual;
  a.sum_out = sum_out;
  a.gamma = gamma;
  a.out = y;
  a.ivar = inv_rms;
  a.N = N;
  a.D = D;
  a.C = 1;
  a.eps = eps;
  const size_t align = residual != nullptr ? common_alignment({x, residual, sum_out, y})
                                           : common_alignment({x, y});
  const int form = residual != nullptr ? 1 : 0;
  Plan p;
  const int st = plan(form, dtype, false, N, D, align, common_alignment({gamma}), &p);
  if (st != NVN_OK) return st;
  cudaError_t e;
  if (p.shape >= 0) {
    a.status = device_status_word();
    RowsPlan rp;
    e = rows_rms_fn(dtype, false)(form, p.epv, p.shape, a, s, false, &rp);
  } else {
    e = generic_launch(dtype, p.epv == full_epv(dtype), false, true, a, nullptr, 0, s);
  }
  return e == cudaSuccess ? NVN_OK : fail_cuda(e);
}

int backward(int form, int dtype, const void* dy, const void* dsum, const void* x, const float* gamma,
             const float* mean, const float* inv, int64_t N, int64_t D, void* dx, float* dgamma,
             float* dbeta, void* ws, size_t ws_bytes, cudaStream_t s) {
  if (ws == nullptr || !aligned(ws, 256)) return NVN_ERR_WORKSPACE;
  const size_t align = dsum != nullptr ? common_alignment({dy, x, dsum, dx}) : common_alignment({dy, x, dx});
  Plan p;
  const int st = plan(form, dtype, true, N, D, align, common_alignment({gamma}), &p);
  if (st != NVN_OK) return st;
  if (ws_bytes < p.bytes) return NVN_ERR_WORKSPACE;
  RowsResArgs a = {};
  a.x = x;
  a.dy = dy;
  a.res = dsum;
  a.gamma = gamma;
  a.mean_in = mean;
  a.ivar_in = inv;
  a.out = dx;
  a.ws = static_cast<float*>(ws);
  a.N = N;
  a.D = D;
  a.C = 1;
  cudaError_t e;
  if (p.shape >= 0) {
    a.status = device_status_word();
    RowsPlan rp;
    e = rows_rms_fn(dtype, true)(form, p.epv, p.shape, a, s, false, &rp);
  } else {
    e = generic_launch(dtype, p.epv == full_epv(dtype), true, form != 2, a,
                       reinterpret_cast<float*>(static_cast<char*>(ws) + p.off_coef),
                       static_cast<int>(p.partial_rows), s);
  }
  if (e != cudaSuccess) return fail_cuda(e);
  e = form == 2 ? colreduce_launch(a.ws, p.partial_rows, D, dgamma, dbeta, s)
                : colsum_launch(a.ws, p.partial_rows, D, dgamma, s);
  return e == cudaSuccess ? NVN_OK : fail_cuda(e);
}

int zero(float* v, int64_t n, cudaStream_t s) {
  const cudaError_t e = cudaMemsetAsync(v, 0, static_cast<size_t>(n) * 4, s);
  return e == cudaSuccess ? NVN_OK : fail_cuda(e);
}

}  // namespace

}  // namespace nvn

using namespace nvn;

extern "C" {

int nvn_rms_fwd(int dtype, const void* x, const float* gamma, int64_t N, int64_t D, float epsilon,
                void* y, float* inv_rms, void* stream) {
  if (!valid_dtype(dtype) || N < 0 || D < 0) return NVN_ERR_INVALID_ARGUMENT;
  if (N == 0 || D == 0) return empty_statistics(inv_rms, N, static_cast<cudaStream_t>(stream));
  if (x == nullptr || gamma == nullptr || y == nullptr) return NVN_ERR_INVALID_ARGUMENT;
  return forward(dtype, x, nullptr, gamma, N, D, epsilon, nullptr, y, inv_rms,
                 static_cast<cudaStream_t>(stream));
}

int nvn_rms_fwd_residual(int dtype, const void* x, const void* residual, const float* gamma,
                         int64_t N, int64_t D, float epsilon, void* sum_out, void* y,
                         float* inv_rms, void* stream) {
  if (!valid_dtype(dtype) || N < 0 || D < 0) return NVN_ERR_INVALID_ARGUMENT;
  if (N == 0 || D == 0) return empty_statistics(inv_rms, N, static_cast<cudaStream_t>(stream));
  if (x == nullptr || residual == nullptr || gamma == nullptr || sum_out == nullptr || y == nullptr ||
      sum_out == y)
    return NVN_ERR_INVALID_ARGUMENT;
  return forward(dtype, x, residual, gamma, N, D, epsilon, sum_out, y, inv_rms,
                 static_cast<cudaStream_t>(stream));
}

size_t nvn_rms_bwd_workspace_bytes(int dtype, int64_t N, int64_t D) {
  const size_t a = workspace(0, dtype, N, D), b = workspace(1, dtype, N, D);
  return a > b ? a : b;
}

int nvn_rms_bwd(int dtype, const void* dy, const void* dsum, const void* x, const float* gamma,
                const float* inv_rms, int64_t N, int64_t D, void* dx, float* dgamma,
                void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_dtype(dtype) || N < 0 || D < 0) return NVN_ERR_INVALID_ARGUMENT;
  if (D == 0) return NVN_OK;
  if (dgamma == nullptr) return NVN_ERR_INVALID_ARGUMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (N == 0) return zero(dgamma, D, s);
  if (dy == nullptr || x == nullptr || gamma == nullptr || inv_rms == nullptr || dx == nullptr)
    return NVN_ERR_INVALID_ARGUMENT;
  return backward(dsum != nullptr ? 1 : 0, dtype, dy, dsum, x, gamma, nullptr, inv_rms, N, D, dx,
                  dgamma, nullptr, workspace, workspace_bytes, s);
}

size_t nvn_ln_bwd_residual_workspace_bytes(int dtype, int64_t N, int64_t D) {
  return workspace(2, dtype, N, D);
}

int nvn_ln_bwd_residual(int dtype, const void* dy, const void* dsum, const void* x,
                        const float* gamma, const float* mean, const float* inv_std, int64_t N,
                        int64_t D, void* dx, float* dgamma, float* dbeta, void* workspace,
                        size_t workspace_bytes, void* stream) {
  if (!valid_dtype(dtype) || N < 0 || D < 0) return NVN_ERR_INVALID_ARGUMENT;
  if (D == 0) return NVN_OK;
  if (dgamma == nullptr || dbeta == nullptr) return NVN_ERR_INVALID_ARGUMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (N == 0) {
    const int st = zero(dgamma, D, s);
    return st != NVN_OK ? st : zero(dbeta, D, s);
  }
  if (dy == nullptr || dsum == nullptr || x == nullptr || gamma == nullptr || mean == nullptr ||
      inv_std == nullptr || dx == nullptr)
    return NVN_ERR_INVALID_ARGUMENT;
  return backward(2, dtype, dy, dsum, x, gamma, mean, inv_std, N, D, dx, dgamma, dbeta, workspace,
                  workspace_bytes, s);
}

}  // extern "C"
