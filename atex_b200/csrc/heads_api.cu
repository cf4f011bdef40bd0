// C ABI of the per-head normalisation with rotary positions: argument checks, the access width,
// workspace and launches (include/nvnorms.h).  No counterpart in the reference.
#include "../../include/nvnorms.h"
#include "nvn_host.h"

namespace nvn {

namespace {

constexpr int64_t kMaxHeadDim = 512;    // 32 lanes of 16 elements
constexpr int64_t kMaxHeads = 65535;

typedef cudaError_t (*HeadsFn)(int, bool, int, HeadArgs&, cudaStream_t, bool, HeadPlan*);
HeadsFn heads_fn(int dtype, bool bwd) {
  if (dtype == NVN_F32) return bwd ? heads_f32_bwd : heads_f32_fwd;
  if (dtype == NVN_F16) return bwd ? heads_f16_bwd : heads_f16_fwd;
  return bwd ? heads_bf16_bwd : heads_bf16_fwd;
}

int vectors_per_part(int norm) { return norm == NVN_NORM_RMS ? 1 : (norm == NVN_NORM_LAYER ? 2 : 0); }

// The strides that matter: an extent of one has none.
void strides(const nvn_head_problem& p, const nvn_heads& v, int64_t (&to)[3]) {
  to[0] = p.batch > 1 ? v.stride_batch : 0;
  to[1] = p.tokens > 1 ? v.stride_token : 0;
  to[2] = v.heads > 1 ? v.stride_head : 0;
}

bool fits(int v, size_t es, const void* ptr, const int64_t (&s)[3]) {
  return reinterpret_cast<uintptr_t>(ptr) % (v * es) == 0 && s[0] % v == 0 && s[1] % v == 0 && s[2] % v == 0;
}

int check(const nvn_head_problem* p) {
  if (p == nullptr || !valid_dtype(p->dtype) || p->norm < NVN_NORM_NONE || p->norm > NVN_NORM_LAYER ||
      p->batch < 0 || p->tokens < 0 || p->head_dim < 1 || p->pairs < 0 || 2 * p->pairs > p->head_dim ||
      p->q.heads < 1 || (p->k.data != nullptr && p->k.heads < 1))
    return NVN_ERR_INVALID_ARGUMENT;
  if (p->pairs > 0 && (p->axes < 1 || (p->position_bytes != 4 && p->position_bytes != 8)))
    return NVN_ERR_INVALID_ARGUMENT;
  if (p->head_dim > kMaxHeadDim) return NVN_ERR_LIMIT;
  if (p->q.heads > kMaxHeads || (p->k.data != nullptr && p->k.heads > kMaxHeads)) return NVN_ERR_UNSUPPORTED;
  if (p->tokens > 0 && p->batch > 0x7fffffffLL / p->tokens) return NVN_ERR_UNSUPPORTED;
  return NVN_OK;
}

int check_pointers(const nvn_head_problem* p, bool bwd) {
  if (p->q.data == nullptr) return NVN_ERR_INVALID_ARGUMENT;
  if (p->pairs > 0 && (p->positions == nullptr || p->inv_freq == nullptr || p->pair_axis == nullptr))
    return NVN_ERR_INVALID_ARGUMENT;
  const bool k = p->k.data != nullptr;
  if (p->norm != NVN_NORM_NONE && (p->scale_q == nullptr || (k && p->scale_k == nullptr)))
    return NVN_ERR_INVALID_ARGUMENT;
  if (p->norm == NVN_NORM_LAYER && !bwd && (p->offset_q == nullptr || (k && p->offset_k == nullptr)))
    return NVN_ERR_INVALID_ARGUMENT;
  return NVN_OK;
}

// Fills the arguments and returns the access width: the widest that divides head_dim, the
// rotated range and every stride, and that every address is aligned to.
int fill(const nvn_head_problem& p, const nvn_heads* const (&out)[2], const nvn_heads* const (&dy)[2],
         HeadArgs* a) {
  *a = {};
  const size_t es = dtype_size(p.dtype);
  const nvn_heads* const in[2] = {&p.q, &p.k};
  a->parts = p.k.data != nullptr ? 2 : 1;
  const bool il = p.interleaved != 0;
  int v = full_epv(p.dtype);
  auto shrink = [&](const void* ptr, const int64_t(&s)[3]) {
    while (v > 1 && !fits(v, es, ptr, s)) v /= 2;
  };
  while (v > 1 && (p.head_dim % v != 0 || (!il && p.pairs % v != 0))) v /= 2;
  for (int i = 0; i < a->parts; ++i) {
    HeadPart& h = a->part[i];
    h.heads = static_cast<int>(in[i]->heads);
    h.x = in[i]->data;
    strides(p, *in[i], h.xs);
    shrink(h.x, h.xs);
    if (out[i] != nullptr) {
      h.out = out[i]->data;
      strides(p, *out[i], h.os);
      shrink(h.out, h.os);
    }
    if (dy[i] != nullptr) {
      h.dy = dy[i]->data;
      strides(p, *dy[i], h.ds);
      shrink(h.dy, h.ds);
    }
  }
  a->param[0] = p.scale_q;
  a->param[1] = p.offset_q;
  a->param[2] = p.scale_k;
  a->param[3] = p.offset_k;
  a->positions = p.positions;
  a->inv_freq = p.inv_freq;
  a->pair_axis = p.pair_axis;
  a->ps[0] = p.axes > 1 ? p.position_stride_axis : 0;
  a->ps[1] = p.batch > 1 ? p.position_stride_batch : 0;
  a->ps[2] = p.tokens > 1 ? p.position_stride_token : 0;
  a->pos64 = p.position_bytes == 8;
  a->axes = p.axes;
  a->pairs = static_cast<int>(p.pairs);
  a->N = p.batch * p.tokens;
  a->T = p.tokens;
  a->tdiv = head_divider(p.tokens);
  a->hd = static_cast<int>(p.head_dim);
  a->inv_hd = 1.0f / static_cast<float>(p.head_dim);
  a->eps = p.epsilon;
  return v;
}

bool matches(const nvn_heads& in, const nvn_heads* out) {
  return out != nullptr && out->data != nullptr && out->heads == in.heads;
}

}  // namespace

}  // namespace nvn

using namespace nvn;

extern "C" {

int nvn_head_norm_rotary_fwd(const nvn_head_problem* p, const nvn_heads* q_out, const nvn_heads* k_out,
                             void* stream) {
  int st = check(p);
  if (st != NVN_OK) return st;
  if (p->batch == 0 || p->tokens == 0) return NVN_OK;
  st = check_pointers(p, false);
  if (st != NVN_OK) return st;
  const bool k = p->k.data != nullptr;
  if (!matches(p->q, q_out) || (k && !matches(p->k, k_out))) return NVN_ERR_INVALID_ARGUMENT;
  HeadArgs a;
  const int v = fill(*p, {q_out, k ? k_out : nullptr}, {nullptr, nullptr}, &a);
  HeadPlan plan;
  const cudaError_t e = heads_fn(p->dtype, false)(p->norm, p->interleaved != 0, v, a,
                                                  static_cast<cudaStream_t>(stream), false, &plan);
  return e == cudaSuccess ? NVN_OK : fail_cuda(e);
}

size_t nvn_head_norm_rotary_bwd_workspace_bytes(const nvn_head_problem* p) {
  if (check(p) != NVN_OK || p->batch == 0 || p->tokens == 0 || vectors_per_part(p->norm) == 0) return 0;
  HeadArgs a;
  const int widest = fill(*p, {nullptr, nullptr}, {nullptr, nullptr}, &a);
  size_t most = 0;
  // the outputs' alignment, which is not known here, may narrow the accesses
  for (int v = widest; v >= 1; v /= 2) {
    HeadPlan plan;
    if (heads_fn(p->dtype, true)(p->norm, p->interleaved != 0, v, a, nullptr, true, &plan) != cudaSuccess) {
      (void)cudaGetLastError();
      return 0;
    }
    if (plan.ws_bytes > most) most = plan.ws_bytes;
  }
  return align_up(most, 256);
}

int nvn_head_norm_rotary_bwd(const nvn_head_problem* p, const nvn_heads* q_grad, const nvn_heads* k_grad,
                             const nvn_heads* dq, const nvn_heads* dk, float* dparams, void* workspace,
                             size_t workspace_bytes, void* stream) {
  int st = check(p);
  if (st != NVN_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool k = p->k.data != nullptr;
  const int64_t cols = (k ? 2 : 1) * vectors_per_part(p->norm) * p->head_dim;
  if (cols > 0 && dparams == nullptr) return NVN_ERR_INVALID_ARGUMENT;
  if (p->batch == 0 || p->tokens == 0) {
    if (cols == 0) return NVN_OK;
    const cudaError_t e = cudaMemsetAsync(dparams, 0, static_cast<size_t>(cols) * 4, s);
    return e == cudaSuccess ? NVN_OK : fail_cuda(e);
  }
  st = check_pointers(p, true);
  if (st != NVN_OK) return st;
  if (!matches(p->q, q_grad) || !matches(p->q, dq) || (k && (!matches(p->k, k_grad) || !matches(p->k, dk))))
    return NVN_ERR_INVALID_ARGUMENT;
  if (cols > 0 && (workspace == nullptr || !aligned(workspace, 256))) return NVN_ERR_WORKSPACE;
  HeadArgs a;
  const int v = fill(*p, {dq, k ? dk : nullptr}, {q_grad, k ? k_grad : nullptr}, &a);
  a.ws = static_cast<float*>(workspace);
  a.ws_bytes = workspace_bytes;
  HeadPlan plan;
  cudaError_t e = heads_fn(p->dtype, true)(p->norm, p->interleaved != 0, v, a, s, false, &plan);
  if (e != cudaSuccess) return fail_cuda(e);
  if (plan.ws_bytes > workspace_bytes) return NVN_ERR_WORKSPACE;
  if (e == cudaSuccess && cols > 0) e = colsum_launch(a.ws, plan.grid, cols, dparams, s);
  return e == cudaSuccess ? NVN_OK : fail_cuda(e);
}

}  // extern "C"
