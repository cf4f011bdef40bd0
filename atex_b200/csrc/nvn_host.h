// Host-side declarations shared by the kernel translation units and the C ABI.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>

struct nvn_dp_comm;

namespace nvn {

// Arguments of the row-cached kernels (rows_kernels.cuh).  `out` is y (forward)
// or dx (backward); `mean` / `ivar` are forward outputs, `mean_in` / `ivar_in`
// backward inputs.  C is the channel count when gamma / beta are indexed by
// row % C (InstanceNorm "NC..."), unused otherwise.
struct RowsArgs {
  const void* x;
  const void* dy;
  const float* gamma;
  const float* beta;
  const float* mean_in;
  const float* ivar_in;
  void* out;
  float* mean;
  float* ivar;
  float* ws;
  int64_t N;
  int64_t D;
  int64_t C;
  float eps;
  int* status;  // device status word: set non-zero when a bounded wait gave up
};

// Arguments of the residual-add forward (rows_fwd_kernel<..., RES = true>): the row that is
// normalised is s = T(x + res), which is also written to sum_out.  A type of its own, so
// that the parameter block - and with it the generated code - of every other instantiation
// of the row kernels stays what their shapes were tuned with.
struct RowsResArgs : RowsArgs {
  const void* res;
  void* sum_out;
};

struct RowsPlan {
  int grid;
  int block;
  int cluster;
  int tpr;
  int vpt;
  int epv;
  int rb;
  int load_mode;  // 0 plain, 1 register prefetch, 2..9 TMA ring with that many stages,
                  // >= 10 held TMA ring with (load_mode - 10) stages
  int partial_rows;  // rows of [2][D] dgamma/dbeta partials the backward kernel writes
};

// Cluster kernels for LayerNorm rows of thousands of vectors (rows_wide.cu): a row must
// fill one of the compiled shapes exactly (wide_ok).  Backward leaves `partial_rows` rows of
// [2][D] dgamma / dbeta partials in RowsArgs::ws.
struct WidePlan {
  int grid;
  int block;
  int cluster;
  int vpt;
  int stages;
  int partial_rows;
};
bool wide_ok(int64_t nvec, bool bwd);
// `forced`: index of a shape of rows_wide.cu to use instead of the default for the row's
// width (tuning runs), or -1.
cudaError_t wide_launch(int dtype, bool bwd, int forced, const RowsArgs& a, cudaStream_t s,
                        bool dry_run, WidePlan* plan);

// On-chip channels-last InstanceNorm (nlc_onchip.cu): one CTA holds a whole batch item in
// shared memory.  nlc_onchip_ok: the item fits and C / vector divides the CTA size.  The
// backward launch leaves per-item (dgamma, dbeta) contributions in colpart[N][2][C].
bool nlc_onchip_ok(int dtype, bool bwd, int64_t C, int64_t D);
cudaError_t nlc_onchip_launch(int dtype, bool bwd, const void* dy, const void* x,
                              const float* gamma, const float* beta, const float* mean_in,
                              const float* ivar_in, int64_t N, int64_t C, int64_t D, float eps,
                              void* out, float* mean, float* ivar, float* colpart, int* status,
                              cudaStream_t s);

// Persistent channels-last InstanceNorm for items far larger than shared memory
// (nlc_stream.cu): one cooperative launch per direction, the tail of every item stays on
// chip between the statistics and the normalisation.  nlc_stream_ok: 128-bit accesses, a
// power-of-two number (<= 32) of channel vectors, C <= 256 (whether the items are large
// enough to be worth it is the dispatcher's decision).  `ws` holds
// nlc_stream_workspace_bytes; the backward launch leaves colpart[N][2][C].  `block`: 512
// threads (one CTA per SM) or 256 (two per SM).  `groups`: CTA groups that work on
// different items at the same time (clamped to N and to the grid).  `row_channels` > 0: row
// mode for channel-first tensors - the N items are contiguous rows of D * C elements (pass
// C = the vector width and D = row length / C), item n being row (n / row_channels,
// n % row_channels) with gamma[n % row_channels]; mean / ivar are [N], colpart is
// [N / row_channels][2][row_channels].
bool nlc_stream_ok(int dtype, int64_t N, int64_t C, int64_t D);
size_t nlc_stream_workspace_bytes(bool bwd, int64_t N, int64_t C);
cudaError_t nlc_stream_launch(int dtype, bool bwd, const void* dy, const void* x,
                              const float* gamma, const float* beta, const float* mean_in,
                              const float* ivar_in, int64_t N, int64_t C, int64_t D, float eps,
                              void* out, float* mean, float* ivar, void* ws, float* colpart,
                              int* status, int block, int groups, int64_t row_channels,
                              cudaStream_t s);

// Warp-per-item channels-last InstanceNorm for small items (nlc_small.cu): any dtype, C and
// alignment, C <= 32 and D * C <= 4096 elements.  Backward leaves colpart[N][2][C].
bool nlc_small_ok(int64_t C, int64_t D);
cudaError_t nlc_small_launch(int dtype, bool bwd, const void* dy, const void* x,
                             const float* gamma, const float* beta, const float* mean_in,
                             const float* ivar_in, int64_t N, int64_t C, int64_t D, float eps,
                             void* out, float* mean, float* ivar, float* colpart, cudaStream_t s);

// Launch configuration for a kernel that follows the kernel it depends on in the same
// stream and calls griddep_wait() (nvn_common.cuh) before reading that kernel's output:
// its launch overlaps the predecessor's tail.  `attr` must outlive the launch call.
inline cudaLaunchConfig_t dependent_launch_config(dim3 grid, dim3 block, size_t smem,
                                                  cudaStream_t s, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr->val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// Remembers `e` for nvn_last_cuda_error() and clears it; returns NVN_ERR_CUDA.
int fail_cuda(cudaError_t e);

// The statistics of n rows without elements are not a number: a mean over nothing (all bits set
// is a NaN).  `v` may be null.
int empty_statistics(float* v, int64_t n, cudaStream_t s);

inline bool aligned(const void* p, size_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}
inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
// codes of nvn_dtype: 0 = float, 1 = half, 2 = bfloat16
inline size_t dtype_size(int dtype) { return dtype == 0 ? 4 : 2; }
inline int full_epv(int dtype) { return dtype == 0 ? 4 : 8; }
inline bool valid_dtype(int d) { return d >= 0 && d <= 2; }

// Largest power-of-two alignment (capped at 16) shared by all the pointers given.
inline size_t common_alignment(std::initializer_list<const void*> ptrs) {
  uintptr_t bits = 0;
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p);
  size_t a = 16;
  while (a > 1 && (bits & (a - 1)) != 0) a >>= 1;
  return a;
}

// Elements per access for rows of width D: the widest of (full, full/2, full/4) that
// divides D and fits the alignment, else single elements.
// `align` is the activations' alignment, `par_align` that of the fp32 parameters, which are
// read e floats at a time in accesses of at most 16 bytes.
inline int pick_epv(int dtype, int64_t D, size_t align, size_t par_align) {
  const int V = full_epv(dtype);
  const size_t es = dtype_size(dtype);
  for (int e = V; e >= 2; e >>= 1)
    if (D % e == 0 && e * es <= align && std::min<size_t>(16, e * 4) <= par_align) return e;
  return 1;
}

int device_sm_count();
void count_launch();
// Whether the row kernels are launched with the programmatic-stream-serialization
// attribute (their launch then overlaps the predecessor's tail); see variant key `pdl`.
bool use_dependent_launch();

// Function attributes (the opt-in to more than 48 KB of dynamic shared memory, non-portable
// cluster sizes) belong to one device's context, and one process may drive several devices
// (a TensorFlow process owns every GPU of the node).  `mask` is a kernel's own set of device
// ordinals whose context already has the attributes; `set` runs with the calling thread's
// current device when that device is not in the set yet.  Two threads may both run `set`
// the first time: the calls are idempotent.
template <typename F>
inline cudaError_t once_per_device(std::atomic<uint64_t>& mask, F&& set) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  // ordinals beyond 63 are not remembered: every call sets the attributes again
  const uint64_t bit = (dev >= 0 && dev < 64) ? (1ull << dev) : 0;
  if (bit != 0 && (mask.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
  e = set();
  if (e != cudaSuccess) return e;
  if (bit != 0) mask.fetch_or(bit, std::memory_order_release);
  return cudaSuccess;
}
// What a launcher remembers of its kernel's residency: a count below 2^20 for one key (bytes of
// dynamic shared memory) per device, because SM counts may differ.  A key that changes from call
// to call is asked for again; ordinals beyond 63 always are.
struct ResidencyCache {
  std::atomic<int64_t> slot[64] = {};   // (key << 20) | count
  int get(int dev, size_t key) const {  // 0: not known
    const int64_t c = dev >= 0 && dev < 64 ? slot[dev].load(std::memory_order_relaxed) : 0;
    return c != 0 && static_cast<size_t>(c >> 20) == key ? static_cast<int>(c & 0xfffff) : 0;
  }
  void put(int dev, size_t key, int count) {
    if (dev >= 0 && dev < 64)
      slot[dev].store((static_cast<int64_t>(key) << 20) | count, std::memory_order_relaxed);
  }
};

// Device address of the library's status word on the current device (nullptr on failure).
int* device_status_word();

// Row-group shapes: X(index, TPR, VPT, CS, RB, PR, MINB, PF)
//   TPR threads per row, VPT vectors per thread, CS CTAs per cluster, RB rows in
//   flight per row group, PR gamma/beta cached in registers, MINB the CTA size for
//   row groups smaller than a CTA (0 = 256 threads), PF load mode: 0 = plain loads,
//   1 = register prefetch of the next row batch, 2..9 = TMA (cp.async.bulk) ring in
//   shared memory with that many stages, 10 + s = (backward) held ring of s stages: the
//   row batch stays in its stage until dx is written and is read from there twice.
// "Light" kernels keep only the row itself in registers (LayerNorm forward,
// InstanceNorm forward/backward); "heavy" is LayerNorm backward, which adds the
// per-column dgamma/dbeta accumulators and therefore spreads a row over more
// threads.  Capacity of a shape is TPR*VPT*CS vectors; the dispatcher takes the
// first entry (in listing order) among those of the smallest sufficient capacity.
#ifndef NVN_ROW_SHAPES_LIGHT
#define NVN_ROW_SHAPES_LIGHT(X)                                                              \
  X(0, 4, 1, 1, 4, 1, 0, 1)     X(1, 8, 1, 1, 4, 1, 0, 1)     X(2, 8, 2, 1, 4, 1, 0, 3)      \
  X(3, 32, 1, 1, 4, 1, 0, 3)    X(4, 32, 2, 1, 2, 1, 0, 3)    X(5, 32, 4, 1, 2, 1, 0, 3)     \
  X(6, 128, 2, 1, 1, 1, 128, 1)  X(7, 128, 4, 1, 1, 1, 0, 2)   X(8, 256, 4, 1, 1, 1, 0, 2)    \
  X(9, 512, 4, 1, 1, 1, 0, 2)   X(10, 512, 8, 1, 1, 0, 0, 1)  X(11, 512, 4, 4, 1, 1, 0, 1)   \
  X(12, 512, 8, 4, 1, 0, 0, 1)  X(13, 512, 8, 8, 1, 0, 0, 1)  X(14, 512, 8, 16, 1, 0, 0, 1)  \
  /* three or five vectors per thread: widths of 3 * 2^k and 5 * 2^k elements */            \
  X(15, 32, 3, 1, 2, 1, 0, 3)   X(16, 64, 3, 1, 2, 1, 0, 3)   X(17, 128, 3, 1, 1, 1, 0, 2)   \
  X(18, 128, 5, 1, 1, 1, 0, 2)  X(19, 256, 3, 1, 1, 1, 0, 2)  X(20, 256, 5, 1, 1, 1, 0, 2)   \
  X(21, 512, 3, 1, 1, 1, 0, 2)
#endif

// In the heavy table a held-ring entry (PF >= 10) is followed by the register-prefetch
// entry of the same capacity: the held ring wins once the problem is large enough to be
// bandwidth-bound, the other on small problems, where the ring's start-up shows.
#ifndef NVN_ROW_SHAPES_HEAVY
#define NVN_ROW_SHAPES_HEAVY(X)                                                              \
  X(0, 4, 1, 1, 4, 1, 128, 3)      X(1, 8, 1, 1, 4, 1, 128, 3)     X(2, 16, 1, 1, 4, 1, 128, 3) \
  X(3, 32, 1, 1, 4, 1, 128, 3)     X(4, 32, 2, 1, 2, 1, 128, 3)    X(5, 64, 2, 1, 2, 1, 128, 3) \
  X(6, 128, 2, 1, 2, 1, 128, 12)   X(7, 64, 4, 1, 1, 1, 128, 1)                                \
  X(8, 128, 4, 1, 1, 1, 128, 13)   X(9, 256, 2, 1, 2, 1, 0, 1)                                 \
  X(10, 256, 4, 1, 1, 1, 0, 12)    X(11, 512, 2, 1, 1, 1, 0, 1)                                \
  X(12, 512, 4, 1, 1, 1, 0, 12)    X(13, 512, 2, 2, 1, 1, 0, 1)                                \
  X(14, 128, 4, 8, 2, 1, 128, 12)  X(15, 512, 2, 4, 1, 1, 0, 1)                                \
  X(16, 128, 4, 16, 2, 1, 128, 12) X(17, 512, 2, 8, 1, 1, 0, 1)                                \
  X(18, 512, 2, 16, 1, 1, 0, 1)    X(19, 512, 4, 16, 1, 0, 0, 1)                               \
  /* three or five vectors per thread: widths of 3 * 2^k and 5 * 2^k elements */            \
  X(20, 32, 3, 1, 2, 1, 128, 3)    X(21, 64, 3, 1, 2, 1, 128, 12)  X(22, 128, 3, 1, 1, 1, 128, 13) \
  X(23, 128, 5, 1, 1, 1, 128, 12)  X(24, 256, 3, 1, 1, 1, 0, 12)   X(25, 512, 3, 1, 1, 1, 0, 12)
#endif

// InstanceNorm "NC..." backward for rows of more than 2048 vectors.  The light table's wide
// shapes hold 8 vectors per thread, which the backward kernel (x-hat and dy of the batch in
// registers across the reduction) cannot afford at 512 threads; these shapes keep at most 4
// vectors per thread or hold the batch in the ring.  Indices start at 256; wider rows take
// the two-phase kernels.
#ifndef NVN_ROW_SHAPES_AFFINE_WIDE
#define NVN_ROW_SHAPES_AFFINE_WIDE(X)                                                        \
  X(256, 256, 4, 4, 1, 0, 0, 1)    X(257, 512, 4, 4, 1, 0, 0, 1)
#endif
constexpr int kAffineWideBase = 256;

// Rows accessed with less than 128 bits per access (64-, 32-bit or single elements: widths
// that are not a multiple of the vector, misaligned buffers) share this coarser table.
#define NVN_ROW_SHAPES_SCALAR(X)                                                             \
  X(0, 8, 4, 1, 2, 0, 0, 1) X(1, 32, 8, 1, 1, 0, 0, 1) X(2, 256, 8, 1, 1, 0, 0, 1)           \
  X(3, 512, 8, 2, 1, 0, 0, 1) X(4, 512, 8, 8, 1, 0, 0, 1) X(5, 512, 8, 16, 1, 0, 0, 1)

// One entry point per (dtype, direction) translation unit.  `epv` (elements per access: the
// full 128-bit width, or 4 / 2 / 1) selects the family, `row_affine` the InstanceNorm
// "NC..." parameter indexing.
// With dry_run the plan is filled in and nothing is launched.
#define NVN_DECLARE_ROWS(NAME)                                                              \
  cudaError_t NAME(bool row_affine, int epv, int shape, const RowsArgs& a, cudaStream_t s, \
                   bool dry_run, RowsPlan* plan);
NVN_DECLARE_ROWS(rows_f32_fwd)
NVN_DECLARE_ROWS(rows_f32_bwd)
NVN_DECLARE_ROWS(rows_f16_fwd)
NVN_DECLARE_ROWS(rows_f16_bwd)
NVN_DECLARE_ROWS(rows_bf16_fwd)
NVN_DECLARE_ROWS(rows_bf16_bwd)

// LayerNorm forward fused with the residual add that precedes it in a pre-norm transformer
// block (rows_res_inst.cu): s = T(x + res) is written to a.sum_out and normalised in the same
// pass.  Covers rows of up to 4096 128-bit vectors with 128-bit accesses; rows_res_ok says
// whether a problem qualifies (the C ABI falls back to an add kernel plus the plain forward).
bool rows_res_ok(int dtype, int64_t D, size_t align, size_t par_align);
cudaError_t rows_res_launch(int dtype, const RowsResArgs& a, cudaStream_t s);
cudaError_t rows_res_f32(const RowsResArgs& a, cudaStream_t s);
cudaError_t rows_res_f16(const RowsResArgs& a, cudaStream_t s);
cudaError_t rows_res_bf16(const RowsResArgs& a, cudaStream_t s);
cudaError_t residual_add_f32(const void* x, const void* res, void* out, int64_t count, cudaStream_t s);
cudaError_t residual_add_f16(const void* x, const void* res, void* out, int64_t count, cudaStream_t s);
cudaError_t residual_add_bf16(const void* x, const void* res, void* out, int64_t count, cudaStream_t s);
// The fallback's element-wise s = T(x + res) for any size and alignment.
cudaError_t residual_add_launch(int dtype, const void* x, const void* res, void* sum_out,
                                int64_t count, cudaStream_t s);

// RMS normalisation and the residual norms' gradients (rows_rms_inst.cu), one entry point per
// (dtype, direction).  `form`: forward 0 = RMS, 1 = RMS of s = T(x + res); backward 0 = RMS,
// 1 = RMS with the residual branch's gradient (a.res) added to dx, 2 = LayerNorm with it.
// RMS reads no mean and no beta; its partial rows are [D] instead of [2][D].
//
// Their shapes: X(index, TPR, VPT, RB, MINB, PF, FORMS), gamma always in registers, one CTA per
// row; FORMS is the set of forms (bit `form`) that may take the entry.  The smallest sufficient
// capacity is used, held rings (PF >= 10) from kRmsHeldMinBytes on.  Measured on B200, each
// against the LayerNorm tables' shape of the same width:
//   forward: small CTAs that keep the next row in registers beat the rings, whose barriers the
//     one reduction does not hide (bf16 [32768, 4096] plain 97 -> 84 us, residual 181 -> 170 us,
//     where 192 threads, 64 of them with a vector less, beat 128 that fit); wide rows of the residual
//     form load on demand ([16384, 8192] 186 -> 166 us, [4096, 32768] 219 -> 177 us).
//   backward: two stages and a warp or two per row (f16 [65536, 1024] LayerNorm 93 -> 85 us, bf16
//     [32768, 2048] RMS residual 107 -> 84 us).  Where three tensors are read, two rows at once and
//     CTAs of 256 threads, whose half as many partial rows cost less to write and read, win again
//     (bf16 [32768, 4096] RMS residual 169 -> 159 us, LayerNorm 161 us); with two tensors one row
//     does (134 -> 125 us).
constexpr int64_t kRmsHeldMinBytes = 32ll << 20;
#define NVN_RMS_FWD_SHAPES(X)                                                                  \
  X(0, 4, 1, 4, 128, 1, 3)    X(1, 8, 1, 4, 128, 1, 3)    X(2, 8, 2, 4, 128, 1, 3)              \
  X(3, 16, 2, 4, 128, 1, 3)   X(4, 64, 1, 2, 128, 1, 3)   X(5, 32, 3, 2, 128, 1, 3)             \
  X(6, 64, 2, 2, 128, 1, 3)   X(7, 64, 3, 1, 128, 1, 3)   X(8, 128, 2, 1, 128, 1, 1)            \
  X(9, 64, 4, 1, 128, 1, 2)   X(10, 128, 3, 1, 128, 1, 3) X(11, 128, 4, 1, 128, 1, 1)           \
  X(12, 192, 3, 1, 128, 1, 2) X(13, 160, 4, 1, 128, 1, 3) X(14, 192, 4, 1, 128, 1, 3)           \
  X(15, 512, 2, 1, 0, 1, 1)   X(16, 256, 4, 1, 0, 0, 2)   X(17, 320, 4, 1, 0, 1, 1)             \
  X(18, 320, 4, 1, 0, 0, 2)   X(19, 384, 4, 1, 0, 1, 1)   X(20, 384, 4, 1, 0, 0, 2)             \
  X(21, 512, 4, 1, 0, 1, 3)   X(22, 512, 8, 1, 0, 0, 3)
#define NVN_RMS_BWD_SHAPES(X)                                                                 \
  X(0, 4, 1, 4, 128, 1, 7)      X(1, 8, 1, 4, 128, 1, 7)      X(2, 8, 2, 4, 128, 12, 7)       \
  X(3, 16, 1, 4, 128, 1, 7)     X(4, 16, 2, 4, 128, 12, 7)    X(5, 32, 1, 4, 128, 1, 7)       \
  X(6, 32, 2, 4, 128, 12, 7)    X(7, 32, 2, 2, 128, 1, 7)     X(8, 32, 3, 2, 128, 12, 7)      \
  X(9, 32, 3, 1, 128, 1, 7)     X(10, 32, 4, 2, 128, 12, 1)   X(11, 64, 2, 2, 0, 12, 6)       \
  X(12, 32, 4, 1, 128, 1, 7)    X(13, 64, 3, 2, 128, 12, 7)   X(14, 64, 3, 1, 128, 1, 7)      \
  X(15, 64, 4, 2, 128, 12, 3)   X(16, 64, 4, 2, 0, 12, 4)     X(17, 128, 2, 1, 128, 1, 7)     \
  X(18, 128, 3, 1, 128, 12, 7)  X(19, 128, 3, 1, 128, 1, 7)   X(20, 256, 2, 1, 0, 12, 1)      \
  X(21, 256, 2, 2, 0, 12, 6)    X(22, 256, 2, 1, 0, 1, 3)     X(23, 128, 4, 1, 128, 1, 4)     \
  X(24, 128, 5, 1, 128, 12, 7)  X(25, 320, 2, 1, 0, 1, 7)     X(26, 256, 3, 1, 0, 12, 7)      \
  X(27, 256, 3, 1, 0, 1, 7)     X(28, 256, 4, 1, 0, 12, 7)    X(29, 512, 2, 1, 0, 1, 7)       \
  X(30, 512, 3, 1, 0, 12, 7)    X(31, 512, 4, 1, 0, 12, 7)
// Accesses of less than 128 bits.  Against the LayerNorm table: f16 [12345, 1001] 20.3 -> 12.5 us
// forward, 58 -> 34 us LayerNorm backward; bf16 [29363, 2347] residual 258 -> 122 us.  The widest
// entry holds 16 values of four tensors per thread, too many with the dbeta sums (f16 [4000, 7031]
// LayerNorm 152 us, 106 us by the kernels for any width).  Those figures are of single elements; 16-bit
// widths that four divides and eight does not hold four times the values in the same entries, and their
// gradients spill (0.2 to 4.8 KB a thread).
#define NVN_RMS_NARROW_SHAPES(X)                                                               \
  X(0, 8, 4, 2, 128, 1, 7)    X(1, 32, 4, 4, 128, 1, 7)   X(2, 32, 8, 2, 128, 1, 7)             \
  X(3, 32, 16, 1, 128, 1, 7)  X(4, 64, 16, 1, 128, 1, 7)  X(5, 128, 16, 1, 128, 1, 7)           \
  X(6, 256, 10, 1, 0, 1, 7)   X(7, 512, 8, 1, 0, 1, 7)    X(8, 512, 16, 1, 0, 1, 3)
#define NVN_DECLARE_ROWS_RMS(NAME)                                                      \
  cudaError_t NAME(int form, int epv, int shape, const RowsResArgs& a, cudaStream_t s, \
                   bool dry_run, RowsPlan* plan);
NVN_DECLARE_ROWS_RMS(rows_rms_f32_fwd)
NVN_DECLARE_ROWS_RMS(rows_rms_f32_bwd)
NVN_DECLARE_ROWS_RMS(rows_rms_f16_fwd)
NVN_DECLARE_ROWS_RMS(rows_rms_f16_bwd)
NVN_DECLARE_ROWS_RMS(rows_rms_bf16_fwd)
NVN_DECLARE_ROWS_RMS(rows_rms_bf16_bwd)

// The same operators for any row width (rows_generic.cu): `vec` = 128-bit accesses, else
// single elements.  a.res may be null (no residual).  Backward: `coef` holds [N][rms ? 1 : 2]
// floats of scratch and a.ws `slices` partial rows (generic_slices).
int generic_slices(int64_t N, int64_t D, int epv);
cudaError_t generic_launch(int dtype, bool vec, bool bwd, bool rms, const RowsResArgs& a,
                           float* coef, int slices, cudaStream_t s);

// out[c] = sum over `rows` partial rows of `cols` floats, in a fixed order (launched as a
// dependent of the kernel before it).
cudaError_t colsum_launch(const float* partials, int64_t rows, int64_t cols, float* out,
                          cudaStream_t s);

// Per-head normalisation with rotary positions (head_rotary.cuh).  Strides are in elements,
// in the order batch, token, head; the elements of a head are contiguous.
struct HeadDiv {   // division by a fixed number: see fast_div
  unsigned mul;
  int shift;       // < 0: the divisor is 1
};
struct HeadPart {  // the queries or the keys
  const void* x;
  const void* dy;
  void* out;
  int64_t xs[3], ds[3], os[3];
  int64_t x_row, d_row, o_row;  // between the heads of a group of rows
  int heads;       // groups of rows per token
  HeadDiv div;     // by heads
};
inline HeadDiv head_divider(int64_t d) {
  if (d <= 1) return {0, -1};
  int s = 1;
  while ((int64_t(1) << s) < d) ++s;
  const uint64_t m = ((uint64_t(1) << (31 + s)) + static_cast<uint64_t>(d) - 1) / static_cast<uint64_t>(d);
  return {static_cast<unsigned>(m), s - 1};
}
struct HeadArgs {
  HeadPart part[2];
  int parts;
  const float* param[4];  // scale and offset of the queries, scale and offset of the keys
  float* ws;              // partial rows [grid][parts][1 or 2][hd]
  size_t ws_bytes;
  const void* positions;
  const double* inv_freq;
  const int32_t* pair_axis;
  int64_t ps[3];          // strides of positions: axis, batch, token
  int pos64, axes, pairs;
  int64_t N, T, tiles;    // N = batch * tokens
  HeadDiv tdiv;           // by T
  HeadDiv adiv;           // by across
  int across, down;       // the angle table is made by `down` tokens of `across` pairs at a time
  int hd, hd4, tph, pstride;
  int tile;               // tokens of a block
  int q_steps, all_steps; // steps of a block: one row for every group of lanes each, queries first
  int steps, pieces;      // steps of a tile, tiles of a block
  int rows;               // rows of a tile
  float inv_hd, eps;
};
struct HeadPlan {
  int v;                  // elements per access
  int grid;               // CTAs = partial rows
  size_t smem;
  size_t ws_bytes;        // of the partial rows; nothing is launched when HeadArgs has fewer
};
// `bwd`, `norm` (0 none, 1 root mean square, 2 mean and variance), `interleaved` select the
// kernel; the launcher sets the layout (hd4, tph, pstride, tile ... rows, tiles) itself.  With dry_run nothing is launched.
#define NVN_DECLARE_HEADS(NAME)                                                                \
  cudaError_t NAME(int norm, bool interleaved, int v, HeadArgs& a, cudaStream_t s, bool dry_run, \
                   HeadPlan* plan);
NVN_DECLARE_HEADS(heads_f32_fwd)
NVN_DECLARE_HEADS(heads_f32_bwd)
NVN_DECLARE_HEADS(heads_f16_fwd)
NVN_DECLARE_HEADS(heads_f16_bwd)
NVN_DECLARE_HEADS(heads_bf16_fwd)
NVN_DECLARE_HEADS(heads_bf16_bwd)

// Deterministic second stage of the dgamma / dbeta reduction: sums P partial
// rows of [2][F] floats (dgamma then dbeta) in a fixed order.
// `scratch` (optional, `scratch_rows` rows of [2F] floats, 16-byte aligned) lets the kernel
// split very many partial rows into slabs when there are few columns.
constexpr int64_t kColreduceScratchRows = 256;
cudaError_t colreduce_launch(const float* partials, int64_t P, int64_t F, float* dgamma,
                             float* dbeta, cudaStream_t s, float* scratch = nullptr,
                             int64_t scratch_rows = 0);

// Column reduction fused with the all-reduce over peer memory (colreduce_dp.cu).  Needs
// 2F % 4 == 0.
cudaError_t colreduce_allreduce_launch(const float* partials, int64_t P, int64_t F,
                                       const struct ::nvn_dp_comm* comm, float* dgamma,
                                       float* dbeta, cudaStream_t s);
cudaError_t dp_finish_launch(int64_t F, const struct ::nvn_dp_comm* comm, float* dgamma,
                             float* dbeta, cudaStream_t s);

}  // namespace nvn
