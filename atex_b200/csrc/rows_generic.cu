// RMS normalisation and residual norm gradients for rows that the row-cached kernels of
// rows_rms_inst.cu do not hold (wider than a CTA's registers, or wide and of a width that
// rules out vector accesses), and the column sum that ends their gradients.
//
//   forward    one CTA per row: pass 1 sums the squares (and writes s = T(x + res)), pass 2
//              reads the row again - from L2 - and writes y.
//   backward   rms_rowsum_kernel: one CTA per row, the row's mean(gy xh) (and mean(gy) for
//              LayerNorm);  rms_columns_kernel: a thread owns EPV columns of a slice of rows,
//              writes dx and keeps dgamma (dbeta) of its columns in registers;  the partial
//              rows of the slices are summed by colsum_kernel in a fixed order.
//
// Bound by HBM: the second pass over x (and dy) misses L2 once a tensor is far larger than
// it, so forward moves up to 3 tensor passes for 2 counted, backward 5 for 3.
#include "nvn_common.cuh"
#include "nvn_host.h"

namespace nvn {

namespace {

constexpr int kRowBlock = 512;
constexpr int kColBlock = 128;

template <typename T, int EPV, bool RES>
__global__ void __launch_bounds__(kRowBlock) rms_generic_fwd_kernel(const RowsResArgs a) {
  using M = typename MathSel<EPV>::M;
  using E = typename M::E;
  constexpr int NE = MathSel<EPV>::NE;
  using P = Pack<T, EPV>;
  __shared__ ReduceSmem<1, kRowBlock> sm;
  int phase = 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t rowvecs = a.D / EPV;
  const float inv_D = 1.0f / static_cast<float>(a.D);
  // squares are scaled down by a power of two, at least as many as a thread adds: see rows_fwd_kernel
  float squares = 1.f;
  if constexpr (kSquaresOverflow<T>) {
    for (int64_t n = (rowvecs + kRowBlock - 1) / kRowBlock * EPV; n > 1; n = (n + 1) / 2) squares *= 2.f;
  }
  const E down = M::bcast(1.f / squares);
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const P* xp = reinterpret_cast<const P*>(a.x) + row * rowvecs;
    const P* rp = reinterpret_cast<const P*>(a.res) + (RES ? row * rowvecs : 0);
    P* sp = reinterpret_cast<P*>(a.sum_out) + (RES ? row * rowvecs : 0);
    P* yp = reinterpret_cast<P*>(a.out) + row * rowvecs;
    E acc = M::bcast(0.f);
    for (int64_t i = tid; i < rowvecs; i += kRowBlock) {
      E v[NE];
      unpack<T, EPV>(load_keep<T, EPV>(reinterpret_cast<const T*>(xp + i)), v);
      if constexpr (RES) {
        E r[NE];
        unpack<T, EPV>(load_keep<T, EPV>(reinterpret_cast<const T*>(rp + i)), r);
#pragma unroll
        for (int e = 0; e < NE; ++e) v[e] = M::add(v[e], r[e]);
        const P s = repack<T, EPV>(v);
        sp[i] = s;
        unpack<T, EPV>(s, v);
      }
#pragma unroll
      for (int e = 0; e < NE; ++e) acc = M::fma(kSquaresOverflow<T> ? M::mul(v[e], down) : v[e], v[e], acc);
    }
    float q[1] = {M::hsum(acc) * (inv_D * squares)};  // the thread's share of the mean: see rows_fwd_kernel
    // the thread reads back only what it wrote itself (s), or what nobody has written (x)
    const P* back = RES ? sp : xp;
    group_allreduce<1, kRowBlock, kRowBlock, 1>(q, sm, phase, warp, lane);
    const float inv = rsqrtf(q[0] + a.eps);
    const E iv2 = M::bcast(inv);
    for (int64_t i = tid; i < rowvecs; i += kRowBlock) {
      E v[NE], g[NE];
      unpack<T, EPV>(load_keep<T, EPV>(reinterpret_cast<const T*>(back + i)), v);
      load_param_lanes<EPV>(a.gamma, i * EPV, g);
#pragma unroll
      for (int e = 0; e < NE; ++e) v[e] = M::mul(M::mul(v[e], iv2), g[e]);
      yp[i] = repack<T, EPV>(v);
    }
    if (tid == 0 && a.ivar != nullptr) a.ivar[row] = inv;
  }
}

// coef[row][NR]: mean(gy) (LayerNorm only), mean(gy xh)
template <typename T, int EPV, bool RMS>
__global__ void __launch_bounds__(kRowBlock) rms_rowsum_kernel(const RowsResArgs a, float* coef) {
  using M = typename MathSel<EPV>::M;
  using E = typename M::E;
  constexpr int NE = MathSel<EPV>::NE;
  constexpr int NR = RMS ? 1 : 2;
  using P = Pack<T, EPV>;
  __shared__ ReduceSmem<NR, kRowBlock> sm;
  int phase = 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t rowvecs = a.D / EPV;
  const float inv_D = 1.0f / static_cast<float>(a.D);
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const P* xp = reinterpret_cast<const P*>(a.x) + row * rowvecs;
    const P* dyp = reinterpret_cast<const P*>(a.dy) + row * rowvecs;
    const E nm = M::bcast(RMS ? 0.f : -a.mean_in[row]);
    const E iv2 = M::bcast(a.ivar_in[row]);
    E r0 = M::bcast(0.f), r1 = M::bcast(0.f);
    for (int64_t i = tid; i < rowvecs; i += kRowBlock) {
      E v[NE], d[NE], g[NE];
      unpack<T, EPV>(load_keep<T, EPV>(reinterpret_cast<const T*>(xp + i)), v);
      unpack<T, EPV>(load_keep<T, EPV>(reinterpret_cast<const T*>(dyp + i)), d);
      load_param_lanes<EPV>(a.gamma, i * EPV, g);
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        d[e] = M::mul(d[e], g[e]);
        if constexpr (!RMS) r0 = M::add(r0, d[e]);
        r1 = M::fma(d[e], M::mul(RMS ? v[e] : M::add(v[e], nm), iv2), r1);
      }
    }
    float red[NR];
    if constexpr (!RMS) red[0] = M::hsum(r0);
    red[NR - 1] = M::hsum(r1);
    group_allreduce<NR, kRowBlock, kRowBlock, 1>(red, sm, phase, warp, lane);
    if (tid == 0) {
#pragma unroll
      for (int k = 0; k < NR; ++k) coef[row * NR + k] = red[k] * inv_D;
    }
  }
}

// a.ws: partial rows [gridDim.y][NR][D]
template <typename T, int EPV, bool RMS>
__global__ void __launch_bounds__(kColBlock)
    rms_columns_kernel(const RowsResArgs a, const float* __restrict__ coef, int64_t rows_per_slice) {
  using M = typename MathSel<EPV>::M;
  using E = typename M::E;
  constexpr int NE = MathSel<EPV>::NE;
  constexpr int NR = RMS ? 1 : 2;
  using P = Pack<T, EPV>;
  const int64_t rowvecs = a.D / EPV;
  const int64_t vec = static_cast<int64_t>(blockIdx.x) * kColBlock + threadIdx.x;
  if (vec >= rowvecs) return;
  const int64_t r_begin = static_cast<int64_t>(blockIdx.y) * rows_per_slice;
  const int64_t r_end = r_begin + rows_per_slice < a.N ? r_begin + rows_per_slice : a.N;
  const P* xp = reinterpret_cast<const P*>(a.x) + vec;
  const P* dyp = reinterpret_cast<const P*>(a.dy) + vec;
  const P* dsp = reinterpret_cast<const P*>(a.res) + vec;
  const bool third = a.res != nullptr;
  P* op = reinterpret_cast<P*>(a.out) + vec;
  E g[NE], dg[NE], db[NE];
  load_param_lanes<EPV>(a.gamma, vec * EPV, g);
#pragma unroll
  for (int e = 0; e < NE; ++e) dg[e] = db[e] = M::bcast(0.f);
  // Wide rows leave few slices, so a slice may have any number of rows: their terms are added 256 at
  // a time and the sums of those joined, in shared memory (registers are short), which keeps an fp32
  // sum of n terms to 256 + n / 256 roundings instead of n.  A thread has slots of its own.
  constexpr int kTogether = 256;
  __shared__ E joined[NR * NE][kColBlock];
#pragma unroll
  for (int e = 0; e < NR * NE; ++e) joined[e][threadIdx.x] = M::bcast(0.f);
  auto join = [&]() {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      joined[e][threadIdx.x] = dg[e] = M::add(joined[e][threadIdx.x], dg[e]);
      if constexpr (!RMS) joined[NE + e][threadIdx.x] = db[e] = M::add(joined[NE + e][threadIdx.x], db[e]);
    }
  };
  constexpr int U = 4;   // rows in flight per thread
  int64_t next_join = r_begin + kTogether;
  for (int64_t r0 = r_begin; r0 < r_end; r0 += U) {
    if (r0 == next_join) {
      join();
#pragma unroll
      for (int e = 0; e < NE; ++e) dg[e] = db[e] = M::bcast(0.f);
      next_join += kTogether;
    }
    P px[U], pd[U], ps[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u < r_end) {
        px[u] = load_stream<T, EPV>(reinterpret_cast<const T*>(xp + (r0 + u) * rowvecs), 0);
        pd[u] = load_stream<T, EPV>(reinterpret_cast<const T*>(dyp + (r0 + u) * rowvecs), 0);
        if (third) ps[u] = load_stream<T, EPV>(reinterpret_cast<const T*>(dsp + (r0 + u) * rowvecs), 0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + u;
      if (row < r_end) {
        E v[NE], d[NE];
        unpack<T, EPV>(px[u], v);
        unpack<T, EPV>(pd[u], d);
        const float iv = __ldg(a.ivar_in + row);
        const E iv2 = M::bcast(iv);
        const E nm = M::bcast(RMS ? 0.f : -__ldg(a.mean_in + row));
        const E nm0 = M::bcast(RMS ? 0.f : -__ldg(coef + row * NR));
        const E nm1 = M::bcast(-__ldg(coef + row * NR + NR - 1));
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          v[e] = M::mul(RMS ? v[e] : M::add(v[e], nm), iv2);
          dg[e] = M::fma(d[e], v[e], dg[e]);
          if constexpr (!RMS) db[e] = M::add(db[e], d[e]);
          d[e] = M::mul(d[e], g[e]);
          v[e] = RMS ? M::fma(v[e], nm1, d[e]) : M::add(d[e], M::fma(v[e], nm1, nm0));
        }
        if (third) {
          E s[NE];
          unpack<T, EPV>(ps[u], s);
#pragma unroll
          for (int e = 0; e < NE; ++e) v[e] = M::fma(v[e], iv2, s[e]);
        } else {
#pragma unroll
          for (int e = 0; e < NE; ++e) v[e] = M::mul(v[e], iv2);
        }
        store_stream<T, EPV>(reinterpret_cast<T*>(op + row * rowvecs), 0, repack<T, EPV>(v));
      }
    }
  }
  join();
  float* w = a.ws + static_cast<int64_t>(blockIdx.y) * NR * a.D;
  store_param_lanes<EPV>(w, vec * EPV, dg);
  if constexpr (!RMS) store_param_lanes<EPV>(w + a.D, vec * EPV, db);
}

template <typename T, int EPV>
cudaError_t fwd_t(const RowsResArgs& a, cudaStream_t s) {
  const int64_t most = static_cast<int64_t>(device_sm_count()) * 4;  // 4 CTAs of 512 threads fill an SM
  const unsigned grid = static_cast<unsigned>(a.N < most ? a.N : most);
  count_launch();
  if (a.res != nullptr) {
    rms_generic_fwd_kernel<T, EPV, true><<<grid, kRowBlock, 0, s>>>(a);
  } else {
    rms_generic_fwd_kernel<T, EPV, false><<<grid, kRowBlock, 0, s>>>(a);
  }
  return cudaGetLastError();
}

template <typename T, int EPV, bool RMS>
cudaError_t bwd_t(const RowsResArgs& a, float* coef, int slices, cudaStream_t s) {
  const int64_t most = static_cast<int64_t>(device_sm_count()) * 4;
  count_launch();
  rms_rowsum_kernel<T, EPV, RMS>
      <<<static_cast<unsigned>(a.N < most ? a.N : most), kRowBlock, 0, s>>>(a, coef);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t tiles = (a.D / EPV + kColBlock - 1) / kColBlock;
  count_launch();
  rms_columns_kernel<T, EPV, RMS>
      <<<dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(slices)), kColBlock, 0, s>>>(
          a, coef, (a.N + slices - 1) / slices);
  return cudaGetLastError();
}

template <typename T>
cudaError_t generic_t(bool vec, bool bwd, bool rms, const RowsResArgs& a, float* coef, int slices,
                      cudaStream_t s) {
  constexpr int V = VecTraits<T>::kFull;
  if (!bwd) return vec ? fwd_t<T, V>(a, s) : fwd_t<T, 1>(a, s);
  if (rms) return vec ? bwd_t<T, V, true>(a, coef, slices, s) : bwd_t<T, 1, true>(a, coef, slices, s);
  return vec ? bwd_t<T, V, false>(a, coef, slices, s) : bwd_t<T, 1, false>(a, coef, slices, s);
}

// ---- column sum ---------------------------------------------------------------
// Block (X, 1024 / X): thread (tx, ty) adds rows ty, ty + TY, ... of column tx in increasing order;
// the TY sums are then added in a fixed order, so that every run gives the same bits.  The partial
// rows come out of L2 and the kernel is a chain of its latencies: up to 2048 columns take X = 8
// (a sector of each row), four times the CTAs and a quarter of the rows per thread of X = 32 (the
// rotary gradients of f16 [14, 3, 32+8, 160] 8.4 -> 7.2 us and f32 [43, 23, 2+1, 128] 7.8 -> 7.3
// us, both kernels).
constexpr int kSumThreads = 1024;

template <int X>
__global__ void __launch_bounds__(kSumThreads)
    colsum_kernel(const float* __restrict__ partials, int64_t rows, int64_t cols,
                  float* __restrict__ out) {
  constexpr int TY = kSumThreads / X;
  constexpr int U = 4;   // loads in flight; the additions keep their order
  __shared__ float tile[32][X + 1];
  const int tid = threadIdx.x, tx = tid % X, ty = tid / X;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * X + tx;
  griddep_launch_dependents();
  griddep_wait();  // the partial rows come from the kernel launched just before
  float s = 0.f;
  if (col < cols) {
    int64_t p = ty;
    for (; p + (U - 1) * TY < rows; p += U * TY) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = partials[(p + u * TY) * cols + col];
#pragma unroll
      for (int u = 0; u < U; ++u) s += v[u];
    }
    for (; p < rows; p += TY) s += partials[p * cols + col];
  }
  // the lanes of a warp that share a column, then the 32 warps
#pragma unroll
  for (int off = X; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if (tid % 32 < X) tile[tid / 32][tx] = s;
  __syncthreads();
  if (tid < X && col < cols) {
    float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 32; ++k) t[k % 4] += tile[k][tx];
    out[col] = (t[0] + t[1]) + (t[2] + t[3]);
  }
}

template <int X>
cudaError_t colsum_t(const float* partials, int64_t rows, int64_t cols, float* out, cudaStream_t s) {
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = dependent_launch_config(
      dim3(static_cast<unsigned>((cols + X - 1) / X)), dim3(kSumThreads), 0, s, &attr);
  count_launch();
  return cudaLaunchKernelEx(&cfg, colsum_kernel<X>, partials, rows, cols, out);
}

}  // namespace

int generic_slices(int64_t N, int64_t D, int epv) {
  // enough (column tile, slice) CTAs for eight per SM, at least eight rows in a slice
  const int64_t tiles = (D / epv + kColBlock - 1) / kColBlock;
  int64_t n = static_cast<int64_t>(device_sm_count()) * 8 / tiles;
  if (n > (N + 7) / 8) n = (N + 7) / 8;
  return static_cast<int>(n < 1 ? 1 : n);
}

cudaError_t generic_launch(int dtype, bool vec, bool bwd, bool rms, const RowsResArgs& a,
                           float* coef, int slices, cudaStream_t s) {
  if (dtype == 0) return generic_t<float>(vec, bwd, rms, a, coef, slices, s);
  if (dtype == 1) return generic_t<__half>(vec, bwd, rms, a, coef, slices, s);
  return generic_t<__nv_bfloat16>(vec, bwd, rms, a, coef, slices, s);
}

cudaError_t colsum_launch(const float* partials, int64_t rows, int64_t cols, float* out,
                          cudaStream_t s) {
  return cols <= 2048 ? colsum_t<8>(partials, rows, cols, out, s)
                      : colsum_t<32>(partials, rows, cols, out, s);
}

}  // namespace nvn
