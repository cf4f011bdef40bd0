// Per-head normalisation and rotary positions on several axes, fused: attention queries and
// keys [batch, token, head, head_dim] are read once, normalised over head_dim (root mean
// square, mean and variance, or not at all), scaled, rotated and written once.
//
//   c  = x (rms) or x - mean(x);  xh = c / sqrt(mean(c^2) + eps);  n = xh g (+ b)
//   pair p of a head turns by  angle = position[axis(p), token] * inv_freq(p):
//       (u, v) -> (u cos - v sin, u sin + v cos)
//   gradient: dn = the rotation turned back on dy;  dg = sum dn xh, db = sum dn over batch,
//   tokens and heads;  gy = dn g;  dx = inv (gy [- mean(gy)] - xh mean(gy xh)).  The statistics
//   are formed again from x, whose row sits in registers anyway: one more shuffle reduction in
//   place of two more tensors.
//
// Both directions are bound by HBM: 2 (forward) or 3 (gradient) passes over q and k.
//
// Layout.  A head is a row of head_dim elements; TPH lanes of a warp (a power of two) own it, 16
// elements each, as SPT slots of two vectors (A, B) of V elements:
//   split pairs (p, p + pairs):   slot s < pairs / V is A = [sV, sV + V), B = the same + pairs,
//                                 so a thread holds both halves of its V pairs
//   interleaved (2p, 2p + 1):     slot s is the 2V elements from 2sV on, V pairs as well
//   behind the rotated elements a slot is 2V plain elements.
// In every form slot s turns by the V angles from pair sV on.
//
// A CTA takes a tile of consecutive tokens with all their heads, queries and keys: the angles of
// a token are the same for all of them and are computed once per tile into shared memory - in 64
// bits up to the fraction of a turn, because a position of a million times a frequency has no
// fraction left in 32.  The rows of the tile are dealt to the groups of TPH lanes; each group
// keeps R rows in flight, and those of the first batch are fetched before the angles are computed.
#pragma once

#include "nvn_common.cuh"
#include "nvn_host.h"

namespace nvn {

constexpr int kHeadBlock = 256;

// n / d for n < 2^31 by a multiplication: with 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d),
// m d - 2^(31+s) < d <= 2^s, so floor(n m / 2^(31+s)) is exact.
__device__ __forceinline__ unsigned fast_div(unsigned n, const HeadDiv& d) {
  return d.shift < 0 ? n : __umulhi(n, d.mul) >> d.shift;
}

template <typename T, int V>
struct HeadTraits {
  static constexpr int SPT = 8 / V;                       // slots per thread
  using P = Pack<T, V>;
};

// Element column of vector `half` of slot s.
template <int V, bool IL>
__device__ __forceinline__ int head_col(int s, int half, int pairs) {
  if (!IL && s * V < pairs) return half == 0 ? s * V : s * V + pairs;
  return (2 * s + half) * V;
}

// (a, b) -> (a cos - b sin, a sin + b cos), or the other way round for SIGN < 0; `c`, `sn` are the
// V cosines and sines of the slot.
template <int V, bool IL, int SIGN>
__device__ __forceinline__ void head_turn(float (&a)[V], float (&b)[V], const float* c,
                                          const float* sn, bool rot_a, bool rot_b) {
  if constexpr (!IL || V == 1) {
    if (rot_a) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float s = SIGN > 0 ? sn[e] : -sn[e];
        const float u = fmaf(a[e], c[e], -(b[e] * s));
        b[e] = fmaf(a[e], s, b[e] * c[e]);
        a[e] = u;
      }
    }
  } else {
    if (rot_a) {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float s = SIGN > 0 ? sn[e / 2] : -sn[e / 2];
        const float u = fmaf(a[e], c[e / 2], -(a[e + 1] * s));
        a[e + 1] = fmaf(a[e], s, a[e + 1] * c[e / 2]);
        a[e] = u;
      }
    }
    if (rot_b) {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float s = SIGN > 0 ? sn[(V + e) / 2] : -sn[(V + e) / 2];
        const float u = fmaf(b[e], c[(V + e) / 2], -(b[e + 1] * s));
        b[e + 1] = fmaf(b[e], s, b[e + 1] * c[(V + e) / 2]);
        b[e] = u;
      }
    }
  }
}

template <int N>
__device__ __forceinline__ void head_reduce(float (&v)[N], int tph) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    if (off < tph) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void head_unpack(const Pack<T, V>& p, float (&f)[V]) {
  typename MathSel<V>::M::E lanes[MathSel<V>::NE];
  unpack<T, V>(p, lanes);
  if constexpr (V == 1) {
    f[0] = lanes[0];
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      f[2 * i] = lanes[i].x;
      f[2 * i + 1] = lanes[i].y;
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> head_pack(const float (&f)[V]) {
  typename MathSel<V>::M::E lanes[MathSel<V>::NE];
  if constexpr (V == 1) {
    lanes[0] = f[0];
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) lanes[i] = make_float2(f[2 * i], f[2 * i + 1]);
  }
  return repack<T, V>(lanes);
}

// NORM: 0 none, 1 root mean square, 2 mean and variance.  IL: interleaved pairs.
template <typename T, int V, int NORM, bool IL, bool BWD>
__global__ void __launch_bounds__(kHeadBlock) head_kernel(const HeadArgs a) {
  constexpr int SPT = HeadTraits<T, V>::SPT;
  using P = Pack<T, V>;
  constexpr int R = (BWD ? 2 : 4) / (sizeof(T) == 4 ? 2 : 1);   // rows in flight per group
  constexpr int NV = NORM == 0 ? 0 : (NORM == 1 ? 1 : 2);       // parameter vectors per part
  // dynamic shared memory: cos [tile][pstride], sin [tile][pstride], parameters [2][NV][hd4],
  // gradient sums [2][NV][16][kHeadBlock] (backward)
  extern __shared__ __align__(16) float head_smem[];
  float* const cos_t = head_smem;
  float* const sin_t = cos_t + a.tile * a.pstride;
  float* const par = sin_t + a.tile * a.pstride;
  float* const sums = par + 2 * NV * a.hd4;

  const int tid = threadIdx.x;
  const int tph = a.tph;
  const int lane = tid & (tph - 1);
  const int group = tid / tph;
  const int groups = kHeadBlock / tph;
  const int pairs = a.pairs;
  const int vectors = a.hd / V;

  griddep_launch_dependents();
  griddep_wait();
  if constexpr (NV > 0) {
    for (int i = tid; i < 2 * NV * a.hd4; i += kHeadBlock) {
      const int which = i / a.hd4, col = i - which * a.hd4;
      const float* src = NV == 1 ? a.param[2 * which] : a.param[which];
      par[i] = src != nullptr && col < a.hd ? __ldg(src + col) : 0.f;
    }
  }

  // this thread's vectors
  int col[SPT][2];
  bool valid[SPT][2], rot[SPT][2];
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int s = lane + i * tph;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      col[i][h] = head_col<V, IL>(s, h, pairs);
      valid[i][h] = !IL && s * V < pairs ? true : 2 * s + h < vectors;
      rot[i][h] = (!IL || V == 1) ? s * V < pairs : (2 * s + h) * V < 2 * pairs;
    }
  }

  P xr[R][SPT][2], dr[BWD ? R : 1][SPT][2];
  // Row `u` of a part's tile: its token in the tile and its element offsets.
  auto fetch = [&](int part, int64_t n0, int base, int rows) {
    const HeadPart& hp = a.part[part];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int u = base + r * groups + group;
      const bool on = u < rows;
      const unsigned lt = fast_div(static_cast<unsigned>(u), hp.div);
      const int64_t h = u - static_cast<int>(lt) * hp.heads;
      const unsigned n = static_cast<unsigned>(n0) + lt;
      const unsigned b = fast_div(n, a.tdiv);
      const int64_t t = n - b * static_cast<unsigned>(a.T);
      const T* xp = static_cast<const T*>(hp.x) + (b * hp.xs[0] + t * hp.xs[1] + h * hp.xs[2]);
      const T* dp = static_cast<const T*>(hp.dy);
      if constexpr (BWD) dp += b * hp.ds[0] + t * hp.ds[1] + h * hp.ds[2];
#pragma unroll
      for (int i = 0; i < SPT; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (on && valid[i][k]) {
            if (!BWD || NORM != 0) xr[r][i][k] = load_stream<T, V>(xp, col[i][k]);
            if constexpr (BWD) dr[r][i][k] = load_stream<T, V>(dp, col[i][k]);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              xr[r][i][k].v[e] = Cvt<T>::from_f32(0.f);
              if constexpr (BWD) dr[r][i][k].v[e] = Cvt<T>::from_f32(0.f);
            }
          }
        }
    }
  };

  bool first = true;
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t n0 = tile * a.tile;
    const int tokens = static_cast<int>(a.N - n0 < a.tile ? a.N - n0 : a.tile);
    fetch(0, n0, 0, tokens * a.part[0].heads);
    // the angles of the tile's tokens
    if (!first) __syncthreads();   // everybody is past the previous tile's table
    for (int i = tid; i < tokens * pairs; i += kHeadBlock) {
      const int lt = i / pairs, p = i - lt * pairs;
      const unsigned n = static_cast<unsigned>(n0) + lt;
      const unsigned b = fast_div(n, a.tdiv);
      const int64_t t = n - b * static_cast<unsigned>(a.T);
      const int axis = __ldg(a.pair_axis + p);
      float c = 1.f, s = 0.f;
      if (axis >= 0 && axis < a.axes) {
        const int64_t at = axis * a.ps[0] + b * a.ps[1] + t * a.ps[2];
        const double pos = a.pos64 ? static_cast<double>(__ldg(static_cast<const long long*>(a.positions) + at))
                                   : static_cast<double>(__ldg(static_cast<const int*>(a.positions) + at));
        double turns = pos * __ldg(a.inv_freq + p) * 0.15915494309189533577;   // 1 / (2 pi)
        turns -= rint(turns);
        sincospif(2.f * static_cast<float>(turns), &s, &c);
      }
      cos_t[lt * a.pstride + p] = c;
      sin_t[lt * a.pstride + p] = s;
    }
    __syncthreads();

#pragma unroll 1
    for (int part = 0; part < a.parts; ++part) {
      const HeadPart& hp = a.part[part];
      const int rows = tokens * hp.heads;
      float g[SPT][2][V], off[SPT][2][V];
      float dg[SPT][2][V], db[SPT][2][V];
#pragma unroll
      for (int i = 0; i < SPT; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float* pv = par + part * NV * a.hd4 + (valid[i][k] ? col[i][k] + e : 0);
            if constexpr (NORM != 0) g[i][k][e] = pv[0];
            if constexpr (NORM == 2 && !BWD) off[i][k][e] = pv[a.hd4];
            if constexpr (BWD && NORM != 0) {
              const float* sv = sums + (part * NV * 16 + (i * 2 + k) * V + e) * kHeadBlock + tid;
              dg[i][k][e] = first ? 0.f : sv[0];
              if constexpr (NORM == 2) db[i][k][e] = first ? 0.f : sv[16 * kHeadBlock];
            }
          }
      for (int base = 0; base < rows; base += groups * R) {
        if (part > 0 || base > 0) fetch(part, n0, base, rows);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int u = base + r * groups + group;
          const bool on = u < rows;
          const unsigned lt = on ? fast_div(static_cast<unsigned>(u), hp.div) : 0;
          const float* ct = cos_t + lt * a.pstride;
          const float* st = sin_t + lt * a.pstride;
          float x[SPT][2][V], d[SPT][2][V];
#pragma unroll
          for (int i = 0; i < SPT; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              head_unpack<T, V>(xr[r][i][k], x[i][k]);
              if constexpr (BWD) head_unpack<T, V>(dr[r][i][k], d[i][k]);
            }
          float inv = 1.f;
          if constexpr (BWD) {
#pragma unroll
            for (int i = 0; i < SPT; ++i) {
              const int p0 = (lane + i * tph) * V;
              float c[V], s[V];
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const bool in = p0 + e < pairs;
                c[e] = in ? ct[p0 + e] : 1.f;
                s[e] = in ? st[p0 + e] : 0.f;
              }
              head_turn<V, IL, -1>(d[i][0], d[i][1], c, s, rot[i][0], rot[i][1]);
            }
          }
          if constexpr (NORM == 2) {
            float m[1] = {0.f};
#pragma unroll
            for (int i = 0; i < SPT; ++i)
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) m[0] += x[i][k][e];
            head_reduce<1>(m, tph);
            m[0] *= a.inv_hd;
#pragma unroll
            for (int i = 0; i < SPT; ++i)
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) x[i][k][e] = valid[i][k] ? x[i][k][e] - m[0] : 0.f;
          }
          if constexpr (NORM != 0) {
            // sum of squares; backward: sum gy c and, for mean and variance, sum gy beside it
            constexpr int NR = BWD ? NORM + 1 : 1;
            float red[NR];
#pragma unroll
            for (int k = 0; k < NR; ++k) red[k] = 0.f;
#pragma unroll
            for (int i = 0; i < SPT; ++i)
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                  red[0] = fmaf(x[i][k][e], x[i][k][e], red[0]);
                  if constexpr (BWD) {
                    const float gy = d[i][k][e] * g[i][k][e];
                    red[1] = fmaf(gy, x[i][k][e], red[1]);
                    if constexpr (NORM == 2) red[2] += gy;
                  }
                }
#pragma unroll
            for (int k = 0; k < NR; ++k) red[k] *= a.inv_hd;   // shares of means: no overflow in the sum
            head_reduce<NR>(red, tph);
            // a group without a row must not put 0 * inf into the parameter sums
            inv = on ? rsqrtf(red[0] + a.eps) : 0.f;
            if constexpr (BWD) {
              const float m1 = red[1] * inv;
              const float m0 = NORM == 2 ? red[NORM] : 0.f;
#pragma unroll
              for (int i = 0; i < SPT; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                  for (int e = 0; e < V; ++e) {
                    const float xh = x[i][k][e] * inv;
                    dg[i][k][e] = fmaf(d[i][k][e], xh, dg[i][k][e]);
                    if constexpr (NORM == 2) db[i][k][e] += d[i][k][e];
                    const float gy = fmaf(d[i][k][e], g[i][k][e], -m0);
                    d[i][k][e] = fmaf(-m1, xh, gy) * inv;
                  }
            } else {
#pragma unroll
              for (int i = 0; i < SPT; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                  for (int e = 0; e < V; ++e)
                    x[i][k][e] = NORM == 2 ? fmaf(x[i][k][e] * inv, g[i][k][e], off[i][k][e])
                                           : x[i][k][e] * inv * g[i][k][e];
            }
          }
          if constexpr (!BWD) {
#pragma unroll
            for (int i = 0; i < SPT; ++i) {
              const int p0 = (lane + i * tph) * V;
              float c[V], s[V];
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const bool in = p0 + e < pairs;
                c[e] = in ? ct[p0 + e] : 1.f;
                s[e] = in ? st[p0 + e] : 0.f;
              }
              head_turn<V, IL, 1>(x[i][0], x[i][1], c, s, rot[i][0], rot[i][1]);
            }
          }
          if (on) {
            const int64_t h = u - static_cast<int>(lt) * hp.heads;
            const unsigned n = static_cast<unsigned>(n0) + lt;
            const unsigned b = fast_div(n, a.tdiv);
            const int64_t t = n - b * static_cast<unsigned>(a.T);
            T* op = static_cast<T*>(hp.out) + (b * hp.os[0] + t * hp.os[1] + h * hp.os[2]);
#pragma unroll
            for (int i = 0; i < SPT; ++i)
#pragma unroll
              for (int k = 0; k < 2; ++k)
                if (valid[i][k]) {
                  if constexpr (BWD) {
                    store_stream<T, V>(op, col[i][k], head_pack<T, V>(d[i][k]));
                  } else {
                    store_stream<T, V>(op, col[i][k], head_pack<T, V>(x[i][k]));
                  }
                }
          }
        }
      }
      if constexpr (BWD && NORM != 0) {
#pragma unroll
        for (int i = 0; i < SPT; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              float* sv = sums + (part * NV * 16 + (i * 2 + k) * V + e) * kHeadBlock + tid;
              sv[0] = dg[i][k][e];
              if constexpr (NORM == 2) sv[16 * kHeadBlock] = db[i][k][e];
            }
      }
    }
    first = false;
  }

  if constexpr (BWD && NORM != 0) {
    // the CTA's sums of the groups, in group order: one partial row [parts][NV][hd]
    __syncthreads();
    float* w = a.ws + static_cast<int64_t>(blockIdx.x) * a.parts * NV * a.hd;
    for (int o = tid; o < a.parts * NV * 16 * tph; o += kHeadBlock) {
      const int vec = o / (16 * tph), rest = o - vec * 16 * tph;
      const int el = rest / tph, ln = rest - el * tph;
      const int s = ln + el / (2 * V) * tph, half = el / V % 2;
      const bool in = (!IL && s * V < pairs) || 2 * s + half < vectors;
      if (!in) continue;
      float t = 0.f;
      for (int gr = 0; gr < groups; ++gr) t += sums[(vec * 16 + el) * kHeadBlock + gr * tph + ln];
      w[vec * a.hd + head_col<V, IL>(s, half, pairs) + el % V] = t;
    }
  }
}

}  // namespace nvn
