// Row-cached kernels of the RMS normalisation and of the residual norms' gradients:
// instantiations of rows_fwd_kernel<..., RMS> and rows_bwd_kernel<..., RMS, DRES> for one
// (dtype, direction) pair, compiled six times with -DNVN_T={0,1,2} and -DNVN_BWD={0,1}.
//
//   forward    y = x inv g, inv = 1/sqrt(mean(x^2) + eps); with RES the row is s = T(x + res)
//   backward   xh = x inv, gy = dy g:  dx = inv (gy - xh mean(gy xh)) [+ dsum],  dg = sum dy xh
//              and the LayerNorm gradient with dsum (its plain form is in rows_inst.cu)
//
// A row belongs to one CTA: up to 4096 vectors forward, 2048 backward; wider rows take
// rows_generic.cu.
#include "rows_kernels.cuh"

#if NVN_T == 0
using T = float;
#define NVN_TNAME f32
#elif NVN_T == 1
using T = __half;
#define NVN_TNAME f16
#else
using T = __nv_bfloat16;
#define NVN_TNAME bf16
#endif

#if NVN_BWD
#define NVN_DIR bwd
#else
#define NVN_DIR fwd
#endif

#define NVN_CAT4_(a, b, c, d) a##_##b##_##c##_##d
#define NVN_CAT4(a, b, c, d) NVN_CAT4_(a, b, c, d)

namespace nvn {

namespace {

constexpr bool kBwd = NVN_BWD != 0;

// FORM: forward 0 = RMS, 1 = RMS behind the residual add; backward 0 = RMS, 1 = RMS with the
// residual branch's gradient, 2 = LayerNorm with it.
template <int EPV, int TPR, int VPT, int RB, bool PR, int MINB, int PF, bool EXACT, int FORM>
cudaError_t launch_exact(const RowsResArgs& a, cudaStream_t stream, bool dry_run, RowsPlan* plan) {
  constexpr int BLOCK = RowBlock<TPR, MINB>::kBlock;
  constexpr int RPC = RowBlock<TPR, MINB>::kRowsPerCta;
  constexpr bool TMA = PF >= 2;
  constexpr bool THIRD = FORM != 0;                         // one tensor more than the plain form
  constexpr int NT = (kBwd ? 2 : 1) + (THIRD ? 1 : 0);      // tensors of a ring stage
  using Args = typename std::conditional<THIRD, RowsResArgs, RowsArgs>::type;
  size_t ring = 0;
  if constexpr (TMA) {
    constexpr size_t kStageRows = static_cast<size_t>(RPC) * RB * NT * (PF >= 10 ? PF - 10 : PF);
    static_assert(sizeof(Pack<T, EPV>) == 16, "ring copies move 16 bytes at least");
    static_assert(kStageRows * TPR * VPT * EPV * sizeof(T) <= (PF >= 10 ? kMaxHeldRingBytes : kMaxRingBytes),
                  "the ring of the widest row this shape holds must fit");
    ring = kStageRows * static_cast<size_t>(a.D) * sizeof(T);
  }
  void (*kernel)(const Args);
  if constexpr (kBwd) {
    kernel = rows_bwd_kernel<T, EPV, TPR, VPT, 1, RB, PR, MINB, PF, EXACT, false, FORM != 2, THIRD>;
  } else {
    kernel = rows_fwd_kernel<T, EPV, TPR, VPT, 1, RB, PR, MINB, PF, EXACT, false, THIRD, true>;
  }
  static ResidencyCache resident;   // CTAs on the device, by ring bytes
  static std::atomic<uint64_t> prepared{0};
  if constexpr (TMA) {
    const cudaError_t e = once_per_device(prepared, [&]() -> cudaError_t {
      cudaFuncAttributes fa;
      const cudaError_t e1 = cudaFuncGetAttributes(&fa, kernel);
      if (e1 != cudaSuccess) return e1;
      const size_t room = 227 * 1024 - fa.sharedSizeBytes - 1024;
      const size_t most = PF >= 10 ? kMaxHeldRingBytes : kMaxRingBytes;
      return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(most < room ? most : room));
    });
    if (e != cudaSuccess) return e;
  }
  int dev = -1;   // a size may be asked for without a device
  if (cudaGetDevice(&dev) != cudaSuccess) (void)cudaGetLastError();
  int units = resident.get(dev, ring);
  if (units == 0) {
    units = resident_units(kernel, BLOCK, 1, ring);
    resident.put(dev, ring, units);
  }
  const int64_t need = (a.N + RPC * RB - 1) / (RPC * RB);
  const int64_t use = need < units ? need : units;
  *plan = {};
  plan->grid = static_cast<int>(use);
  plan->block = BLOCK;
  plan->cluster = 1;
  plan->tpr = TPR;
  plan->vpt = VPT;
  plan->epv = EPV;
  plan->rb = RB;
  plan->load_mode = PF;
  plan->partial_rows = static_cast<int>(use);
  if (dry_run) return cudaSuccess;

  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(plan->grid), 1, 1);
  cfg.blockDim = dim3(BLOCK, 1, 1);
  cfg.dynamicSmemBytes = ring;
  cfg.stream = stream;
  // as for the LayerNorm kernels: dependent launches for short kernels only
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed =
      use_dependent_launch() && a.N * a.D * static_cast<int64_t>(sizeof(T)) <= (int64_t(128) << 20)
          ? 1
          : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<const Args&>(a));
}

template <int EPV, int TPR, int VPT, int RB, int MINB, int PF, int FORMS, int FORM>
cudaError_t launch_one(const RowsResArgs& a, cudaStream_t s, bool dry, RowsPlan* plan) {
  if constexpr ((FORMS >> FORM & 1) == 0) {
    return cudaErrorInvalidValue;  // another form's entry
  } else if constexpr (EPV != VecTraits<T>::kFull) {
    return launch_exact<EPV, TPR, VPT, RB, true, MINB, PF, false, FORM>(a, s, dry, plan);
  } else {
    return a.D == static_cast<int64_t>(TPR) * VPT * EPV
               ? launch_exact<EPV, TPR, VPT, RB, true, MINB, PF, true, FORM>(a, s, dry, plan)
               : launch_exact<EPV, TPR, VPT, RB, true, MINB, PF, false, FORM>(a, s, dry, plan);
  }
}

template <int EPV, int FORM>
cudaError_t launch_form(int shape, const RowsResArgs& a, cudaStream_t s, bool dry, RowsPlan* plan) {
#define X(I, TPR, VPT, RB, MINB, PF, FORMS) \
  case I:                                   \
    return launch_one<EPV, TPR, VPT, RB, MINB, PF, FORMS, FORM>(a, s, dry, plan);
  if constexpr (EPV != VecTraits<T>::kFull) {
    switch (shape) { NVN_RMS_NARROW_SHAPES(X) }
  } else if constexpr (kBwd) {
    switch (shape) { NVN_RMS_BWD_SHAPES(X) }
  } else {
    switch (shape) { NVN_RMS_FWD_SHAPES(X) }
  }
#undef X
  return cudaErrorInvalidValue;
}

template <int EPV>
cudaError_t launch_epv(int form, int shape, const RowsResArgs& a, cudaStream_t s, bool dry,
                       RowsPlan* plan) {
  if (form == 0) return launch_form<EPV, 0>(shape, a, s, dry, plan);
  if (form == 1) return launch_form<EPV, 1>(shape, a, s, dry, plan);
  if constexpr (kBwd) {
    if (form == 2) return launch_form<EPV, 2>(shape, a, s, dry, plan);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t NVN_CAT4(rows, rms, NVN_TNAME, NVN_DIR)(int form, int epv, int shape,
                                                     const RowsResArgs& a, cudaStream_t s,
                                                     bool dry_run, RowsPlan* plan) {
  constexpr int V = VecTraits<T>::kFull;
  if (epv == V) return launch_epv<V>(form, shape, a, s, dry_run, plan);
  if (epv == 1) return launch_epv<1>(form, shape, a, s, dry_run, plan);
  if (epv == 2) return launch_epv<2>(form, shape, a, s, dry_run, plan);
  if constexpr (V == 8) {
    if (epv == 4) return launch_epv<4>(form, shape, a, s, dry_run, plan);
  }
  return cudaErrorInvalidValue;
}

}  // namespace nvn
