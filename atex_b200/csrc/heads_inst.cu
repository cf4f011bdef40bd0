// Instantiates the per-head normalisation and rotary kernels (head_rotary.cuh) for one
// (dtype, direction) pair; compiled six times with -DNVN_T={0,1,2} and -DNVN_BWD={0,1}.
#include "head_rotary.cuh"

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

#define NVN_CAT3_(a, b, c) a##_##b##_##c
#define NVN_CAT3(a, b, c) NVN_CAT3_(a, b, c)

namespace nvn {

namespace {

constexpr bool kBwd = NVN_BWD != 0;
constexpr int kMaxRows = kBwd ? 256 : 512;   // of a tile (its addresses: 3 buffers of 32 bytes a row)
constexpr int kTableBytes = 48 * 1024;   // most that a tile's angles may take

inline int round4(int v) { return (v + 3) / 4 * 4; }

template <int V, int NORM, bool IL, int FULL, bool PAD, int R>
cudaError_t launch_kernel(HeadArgs a, cudaStream_t s, bool dry_run, HeadPlan* plan) {
  auto kernel = head_kernel<T, V, NORM, IL, kBwd, FULL, PAD, R>;
  constexpr int BLOCK = head_block(R);
  constexpr int SPT = HeadTraits<V>::SPT;
  constexpr int NV = NORM;
  const int slots = (a.hd + 2 * V - 1) / (2 * V);
  a.tph = 1;
  while (a.tph * SPT < slots) a.tph *= 2;
  if (a.tph > 32) return cudaErrorInvalidValue;
  a.pstride = a.tph * SPT * V * 2;
  a.across = a.pairs < BLOCK ? (a.pairs > 0 ? a.pairs : 1) : BLOCK;
  a.down = BLOCK / a.across;
  a.adiv = head_divider(a.across);
  a.hd4 = round4(a.hd);
  // A tile is up to eight steps of the CTA.  Tokens are dealt out so that the CTAs that fit on the
  // GPU at once take the same number of tiles; when there are fewer tokens than CTAs a tile is a
  // piece of one token's rows.
  const int groups = BLOCK / a.tph;
  for (int i = 0; i < a.parts; ++i) {   // R heads are one row of work
    HeadPart& h = a.part[i];
    h.heads /= R;
    h.div = head_divider(h.heads);
    h.x_row = h.xs[2];
    h.d_row = h.ds[2];
    h.o_row = h.os[2];
    h.xs[2] *= R;
    h.ds[2] *= R;
    h.os[2] *= R;
  }
  const int hq = a.part[0].heads, hk = a.parts > 1 ? a.part[1].heads : 0;
  const int most_steps = kMaxRows / R / groups < 8 ? kMaxRows / R / groups : 8;
  const int64_t ctas = static_cast<int64_t>(device_sm_count()) * head_ctas(kBwd, R, NORM, PAD);
  int64_t tile = static_cast<int64_t>(most_steps) * groups / (hq + hk);
  // what one CTA's tables may take so that the registers, and not they, set the CTAs per SM
  constexpr size_t kSlots = kBwd && R > 1 ? R * SPT * 4 * BLOCK * 16 : 0;
  const size_t fixed =
      static_cast<size_t>(2 * NV * a.hd4 + (kBwd ? 2 * NV * 16 * BLOCK : 0)) * 4 + kSlots;
  int64_t room = (227 * 1024) / head_ctas(kBwd, R, NORM, PAD) - 1024 - static_cast<int64_t>(fixed) -
                 3 * 32 * (most_steps + 2) * groups;
  if (room > kTableBytes) room = kTableBytes;
  // (unless that leaves too few rows to fill the steps: a CTA less is the smaller loss)
  const int64_t fits = room / (3 * 4 * a.pstride);
  if (tile > fits && fits * (hq + hk) >= 3 * groups) tile = fits;
  if (tile > kTableBytes / (3 * 4 * a.pstride)) tile = kTableBytes / (3 * 4 * a.pstride);
  if (tile < 1) tile = 1;
  const int64_t waves = (a.N + tile * ctas - 1) / (tile * ctas);
  tile = (a.N + waves * ctas - 1) / (waves * ctas);
  a.tile = static_cast<int>(tile);
  const int64_t blocks = (a.N + a.tile - 1) / a.tile;
  a.q_steps = static_cast<int>((static_cast<int64_t>(a.tile) * hq + groups - 1) / groups);
  a.all_steps = a.q_steps + static_cast<int>((static_cast<int64_t>(a.tile) * hk + groups - 1) / groups);
  a.steps = a.all_steps < most_steps + 2 ? a.all_steps : most_steps;
  while (a.steps > 1 && blocks * ((a.all_steps + a.steps - 2) / (a.steps - 1)) <= ctas) --a.steps;
  a.pieces = (a.all_steps + a.steps - 1) / a.steps;
  a.tiles = blocks * a.pieces;
  a.rows = a.steps * groups;
  const size_t smem = fixed + static_cast<size_t>(3) * (32 * a.rows + 4 * a.tile * a.pstride);
  static std::atomic<uint64_t> prepared{0};
  cudaError_t e = once_per_device(prepared, [&]() -> cudaError_t {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(kSlots) + kTableBytes + 3 * 32 * (kMaxRows + 2 * BLOCK) +
                                    (2 * NV * 512 + (kBwd ? 2 * NV * 16 * BLOCK : 0)) * 4);
  });
  if (e != cudaSuccess) return e;
  // persistent: tables and (backward) the parameter sums of a CTA serve all its tiles
  static ResidencyCache resident_per_sm;   // CTAs per SM, by shared bytes
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int per_sm = resident_per_sm.get(dev, smem);
  if (per_sm == 0) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, BLOCK, smem);
    if (e != cudaSuccess) return e;
    if (per_sm < 1) per_sm = 1;
    resident_per_sm.put(dev, smem, per_sm);
  }
  const int64_t resident = static_cast<int64_t>(per_sm) * device_sm_count();
  const int64_t grid = a.tiles < resident ? a.tiles : resident;
  plan->v = V;
  plan->grid = static_cast<int>(grid);
  plan->smem = smem;
  plan->ws_bytes = kBwd ? static_cast<size_t>(grid) * a.parts * NV * a.hd * 4 : 0;
  if (dry_run || plan->ws_bytes > a.ws_bytes) return cudaSuccess;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(BLOCK, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  // dependent launches for short kernels only, as for the row kernels
  attr[0].val.programmaticStreamSerializationAllowed =
      use_dependent_launch() &&
              a.N * (hq + hk) * R * a.hd * static_cast<int64_t>(sizeof(T)) <= (int64_t(128) << 20)
          ? 1
          : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int V, int NORM, bool IL, int R>
cudaError_t launch_full(HeadArgs& a, cudaStream_t s, bool dry, HeadPlan* plan) {
  const bool pad = (a.hd != 64 && a.hd != 128 && a.hd != 256) || 2 * a.pairs != a.hd;
#define NVN_HEADS(FULL)                                                      \
  return pad ? launch_kernel<V, NORM, IL, FULL, true, R>(a, s, dry, plan)    \
             : launch_kernel<V, NORM, IL, FULL, false, R>(a, s, dry, plan)
  if (a.hd <= 64) NVN_HEADS(4);
  if (a.hd <= 128) NVN_HEADS(8);
  NVN_HEADS(16);
#undef NVN_HEADS
}

template <int V, int NORM, bool IL>
cudaError_t launch(HeadArgs& a, cudaStream_t s, bool dry, HeadPlan* plan) {
  if constexpr (V == VecTraits<T>::kFull) {
    if (a.hd > 32 && a.hd <= 256 && a.hd % (2 * V) == 0 && a.pairs % V == 0) {
      // Two heads at once in 16 bits, when they pair up and there is work for every CTA (bf16
      // [16, 2048, 32+8, 128] forward 124 -> 111 us, f16 [2, 17550, 16+16, 64] with layer norm 67
      // -> 61 us); with fewer rows one head at a time spreads over more CTAs, and fp32 rows are
      // twice as long and would not fit in the registers.
      if constexpr (sizeof(T) == 2) {
        const int hq = a.part[0].heads, hk = a.parts > 1 ? a.part[1].heads : 0;
        const int groups = head_block(1) / (a.hd <= 64 ? 4 : (a.hd <= 128 ? 8 : 16));
        if (hq % 2 == 0 && hk % 2 == 0 &&
            a.N * (hq + hk) >= static_cast<int64_t>(device_sm_count()) * head_ctas(kBwd, 1, NORM, false) * groups)
          return launch_full<V, NORM, IL, 2>(a, s, dry, plan);
      }
      return launch_full<V, NORM, IL, 1>(a, s, dry, plan);
    }
  }
  return launch_kernel<V, NORM, IL, 0, false, 1>(a, s, dry, plan);
}

template <int V>
cudaError_t launch_v(int norm, bool il, HeadArgs& a, cudaStream_t s, bool dry, HeadPlan* plan) {
  if (norm == 0) return il ? launch<V, 0, true>(a, s, dry, plan) : launch<V, 0, false>(a, s, dry, plan);
  if (norm == 1) return il ? launch<V, 1, true>(a, s, dry, plan) : launch<V, 1, false>(a, s, dry, plan);
  return il ? launch<V, 2, true>(a, s, dry, plan) : launch<V, 2, false>(a, s, dry, plan);
}

}  // namespace

cudaError_t NVN_CAT3(heads, NVN_TNAME, NVN_DIR)(int norm, bool interleaved, int v, HeadArgs& a,
                                                 cudaStream_t s, bool dry_run, HeadPlan* plan) {
  if constexpr (VecTraits<T>::kFull == 8) {
    if (v == 8) return launch_v<8>(norm, interleaved, a, s, dry_run, plan);
  }
  if (v == 4) return launch_v<4>(norm, interleaved, a, s, dry_run, plan);
  if (v == 2) return launch_v<2>(norm, interleaved, a, s, dry_run, plan);
  return launch_v<1>(norm, interleaved, a, s, dry_run, plan);
}

}  // namespace nvn
