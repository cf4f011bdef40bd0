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
// Both directions move 2 (forward) or 3 (gradient) passes over q and k and are bound by HBM when
// there are rows enough: bf16, 32+8 packed heads of 128, 32768 tokens forward 116 us (5.8 TB/s, 89 % of
// the measured copy rate), 16384 tokens gradient 91 us (5.6 TB/s, 85 %).  What stands between that and
// the copy rate is a row's dependent chain (unpack, sums, shuffles, rotation) on 16 to 20 warps an SM.
//
// Layout.  A head is a row of head_dim elements; TPH lanes of a warp (a power of two) own it, 16
// elements each, as SPT slots of two vectors (A, B) of V elements:
//   split pairs (p, p + pairs):   slot s < pairs / V is A = [sV, sV + V), B = the same + pairs,
//                                 so a thread holds both halves of its V pairs
//   interleaved (2p, 2p + 1):     slot s is the 2V elements from 2sV on, V pairs as well; a head of
//                                 whole slots (FULL below) takes A = [sV, sV + V) and B half a head
//                                 behind it, so that neighbouring lanes copy neighbouring vectors
//   behind the rotated elements a slot is 2V plain elements.
//
// A CTA takes tiles: a block of consecutive tokens with all their heads, queries and keys - or, when
// a token has more rows than a tile, or tokens are few, a piece of the block's rows.  The angles of a
// token are the same for all its heads and are computed once per tile into shared memory - in 64
// bits up to the fraction of a turn, because a position of a million times a frequency has no
// fraction left in 32; cosine and sine are fp32 functions of the fraction rounded to fp32, corrected
// by what the rounding dropped (1.3 units of 2^-24 at worst, measured; a rounded 64-bit value has
// 0.5).  Where each row of a tile begins is worked out once as well, by one thread a
// row (done by every lane for every row it was a fifth of the instructions).  The rows of a tile
// are dealt to the groups of TPH lanes; while a group works on a row its next one is already on the
// way into registers, across the ends of parts and tiles too.  The tables (angles, row addresses)
// have three buffers, so that one barrier per tile is enough: tile i reads buffer i, its last rows
// fetch from the addresses of buffer i + 1, and the barrier in tile i + 1 stands between the last
// read of buffer i and its refill in tile i + 2.
#pragma once

#include "nvn_common.cuh"
#include "nvn_host.h"

namespace nvn {

// Threads per CTA, and the CTAs per SM that the registers are limited for: with two rows at once
// 5 (backward 4) small CTAs of up to 102 (128) registers, with offsets or padding one fewer of 128
// (168); with one row 3 (2) of 80 (128).  Spilling to fit a fourth cost more than it gave (88 -> 115 us).  Small
// CTAs for one row were slower (f32 [3, 1025, 10+2, 80] gradient 17.5 -> 20.0 us).
__host__ __device__ constexpr int head_block(int rows) { return rows > 1 ? 128 : 256; }
__host__ __device__ constexpr int head_ctas(bool bwd, int rows, int norm, bool pad) {
  return bwd ? (rows > 1 ? (norm == 2 || (norm == 1 && pad) ? 3 : 4) : 2)
             : (rows > 1 ? (norm == 2 || pad ? 4 : 5) : 3);
}

// n / d for n < 2^31 by a multiplication: with 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d),
// m d - 2^(31+s) < d <= 2^s, so floor(n m / 2^(31+s)) is exact.
__device__ __forceinline__ unsigned fast_div(unsigned n, const HeadDiv& d) {
  return d.shift < 0 ? n : __umulhi(n, d.mul) >> d.shift;
}

template <int V>
struct HeadTraits {
  static constexpr int SPT = 8 / V;             // slots per thread
  static constexpr int CW = V < 4 ? V : 4;      // floats of one access to the angle table
  static constexpr int CHUNKS = V / CW;         // accesses for a slot's cosines
};

// Element column of vector `half` of slot s.
template <int V, bool IL, int FULL>
__device__ __forceinline__ int head_col(int s, int half, int pairs, int hd) {
  if (IL && FULL != 0) return s * V + half * (hd / 2);
  if (!IL && s * V < pairs) return half == 0 ? s * V : s * V + pairs;
  return (2 * s + half) * V;
}

// Angle table of one token: [cos, sin][chunk][slot][CW], so that neighbouring lanes read
// neighbouring 16-byte words.
template <int V, bool IL, int FULL>
__device__ __forceinline__ int head_table_at(int p, bool sine, int nslots, int hd) {
  constexpr int CW = HeadTraits<V>::CW, CHUNKS = HeadTraits<V>::CHUNKS;
  int s = p / V, e = p % V;
  if constexpr (IL && FULL != 0) {   // vector v = 2p / V is slot v's A, or slot (v - half)'s B
    const int v = p / (V / 2), half = hd / (2 * V);
    s = v < half ? v : v - half;
    e = p % (V / 2) + (v < half ? 0 : V / 2);
  }
  return (((sine ? CHUNKS : 0) + e / CW) * nslots + s) * CW + e % CW;
}

// The V cosines (or sines) of slot s.
template <int V>
__device__ __forceinline__ void head_table_read(const float* tab, bool sine, int s, int nslots,
                                                float (&out)[V]) {
  constexpr int CW = HeadTraits<V>::CW, CHUNKS = HeadTraits<V>::CHUNKS;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const float* p = tab + (((sine ? CHUNKS : 0) + c) * nslots + s) * CW;
    if constexpr (CW == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      out[4 * c] = v.x;
      out[4 * c + 1] = v.y;
      out[4 * c + 2] = v.z;
      out[4 * c + 3] = v.w;
    } else if constexpr (CW == 2) {
      const float2 v = *reinterpret_cast<const float2*>(p);
      out[0] = v.x;
      out[1] = v.y;
    } else {
      out[0] = *p;
    }
  }
}

__device__ __forceinline__ float2 neg(float2 v) { return make_float2(-v.x, -v.y); }
__device__ __forceinline__ float neg(float v) { return -v; }

// (a, b) -> (a cos - b sin, a sin + b cos), turned back for SIGN < 0.
// `left` is the number of the slot's pairs that are rotated, for interleaved pairs whose rotated
// range ends inside a vector (an infinity beside it must not meet a sine of zero); with WHOLE a
// vector is rotated or not.
template <int V, bool IL, int SIGN, bool WHOLE, typename E, int NE>
__device__ __forceinline__ void head_turn(E (&a)[NE], E (&b)[NE], const float (&c)[V],
                                          const float (&sn)[V], bool rot_a, bool rot_b, int left) {
  using M = typename MathSel<V>::M;
  if constexpr (!IL || V == 1) {
    if (rot_a) {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        E cc, ss;
        if constexpr (V == 1) {
          cc = c[0];
          ss = sn[0];
        } else {
          cc = make_float2(c[2 * e], c[2 * e + 1]);
          ss = make_float2(sn[2 * e], sn[2 * e + 1]);
        }
        const E bs = M::mul(b[e], ss), as = M::mul(a[e], ss);
        a[e] = M::fma(a[e], cc, SIGN > 0 ? neg(bs) : bs);
        b[e] = M::fma(b[e], cc, SIGN > 0 ? as : neg(as));
      }
    }
  } else {
    auto turn = [&](E& v, int e) {
      const float cc = c[e], ss = SIGN < 0 ? -sn[e] : sn[e];
      const float u = fmaf(v.x, cc, -(v.y * ss));
      const float w = fmaf(v.x, ss, v.y * cc);
      if (WHOLE || e < left) v = make_float2(u, w);
    };
    if (rot_a) {
#pragma unroll
      for (int e = 0; e < NE; ++e) turn(a[e], e);
    }
    if (rot_b) {
#pragma unroll
      for (int e = 0; e < NE; ++e) turn(b[e], NE + e);
    }
  }
}

template <int FULL, int N>
__device__ __forceinline__ void head_reduce(float (&v)[N], int tph) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    if (off < (FULL != 0 ? FULL : tph)) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    }
  }
}

// V consecutive floats of shared memory as math lanes.
template <int V>
__device__ __forceinline__ void head_lanes(const float* p, typename MathSel<V>::M::E (&out)[MathSel<V>::NE]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 v = reinterpret_cast<const float4*>(p)[i];
      out[2 * i] = make_float2(v.x, v.y);
      out[2 * i + 1] = make_float2(v.z, v.w);
    }
  } else if constexpr (V == 2) {
    out[0] = *reinterpret_cast<const float2*>(p);
  } else {
    out[0] = *p;
  }
}

// The same, to shared memory of a thread's own: element e of vector j is word
// ((j V + e) / CW) CW BLOCK + CW thread + e % CW, so that a warp's accesses are contiguous.
template <int V, int BLOCK>
__device__ __forceinline__ void head_sums_load(const float* p, int j, typename MathSel<V>::M::E (&out)[MathSel<V>::NE]) {
  constexpr int CW = HeadTraits<V>::CW;
#pragma unroll
  for (int c = 0; c < V / CW; ++c) {
    const float* q = p + (j * (V / CW) + c) * CW * BLOCK;
    if constexpr (CW == 4) {
      const float4 v = *reinterpret_cast<const float4*>(q);
      out[2 * c] = make_float2(v.x, v.y);
      out[2 * c + 1] = make_float2(v.z, v.w);
    } else if constexpr (CW == 2) {
      out[0] = *reinterpret_cast<const float2*>(q);
    } else {
      out[0] = *q;
    }
  }
}
template <int V, int BLOCK>
__device__ __forceinline__ void head_sums_store(float* p, int j, const typename MathSel<V>::M::E (&in)[MathSel<V>::NE]) {
  constexpr int CW = HeadTraits<V>::CW;
#pragma unroll
  for (int c = 0; c < V / CW; ++c) {
    float* q = p + (j * (V / CW) + c) * CW * BLOCK;
    if constexpr (CW == 4) {
      *reinterpret_cast<float4*>(q) = make_float4(in[2 * c].x, in[2 * c].y, in[2 * c + 1].x, in[2 * c + 1].y);
    } else if constexpr (CW == 2) {
      *reinterpret_cast<float2*>(q) = in[0];
    } else {
      *q = in[0];
    }
  }
}

// Turns every slot of R rows of one token by its angles.
template <int V, bool IL, int SIGN, int FULL, int R, int SPT, typename E, int NE>
__device__ __forceinline__ void head_rotate(E (&v)[R][SPT][2][NE], const float* tab, int nslots,
                                            const int (&slot_of)[SPT], const bool (&rot)[SPT][2], int pairs) {
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    float c[V], s[V];
    head_table_read<V>(tab, false, slot_of[i], nslots, c);
    head_table_read<V>(tab, true, slot_of[i], nslots, s);
#pragma unroll
    for (int r = 0; r < R; ++r)
      head_turn<V, IL, SIGN, FULL != 0>(v[r][i][0], v[r][i][1], c, s, rot[i][0], rot[i][1],
                                        pairs - slot_of[i] * V);
  }
}

// 16 bytes from global to shared memory; cp.async.wait_all of the same thread makes them visible.
__device__ __forceinline__ void head_copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}

// Where a row (the first of R) is read, and where it goes: null for one that is none.
struct alignas(16) HeadSource {
  const void* x;
  const void* dy;
};
struct alignas(16) HeadTarget {
  void* out;
  int angles;   // of the row's token, in the tile's table
  int unused;
};

// NORM: 0 none, 1 root mean square, 2 mean and variance.  IL: interleaved pairs.
// R: rows a group works on at once, neighbouring heads of one token: they share its angles and the
// parameters, and their reductions overlap.
// FULL: lanes per head (4, 8, 16) of heads that are whole slots, rotated slot by slot (in 16 bits
// head_dim a multiple of 16 up to 256 and pairs of 8): the reduction is fixed.  Without PAD the
// head fills its lanes and is rotated whole; with PAD lanes behind its last slot repeat that slot -
// only their sums and stores are left out, where predicates around every access cost a tenth of
// the time.  0: any head.
template <typename T, int V, int NORM, bool IL, bool BWD, int FULL, bool PAD, int R>
__global__ void __launch_bounds__(head_block(R), head_ctas(BWD, R, NORM, PAD)) head_kernel(const HeadArgs a) {
  constexpr int BLOCK = head_block(R);
  constexpr int SPT = HeadTraits<V>::SPT;
  using M = typename MathSel<V>::M;
  using E = typename M::E;
  constexpr int NE = MathSel<V>::NE;
  using P = Pack<T, V>;
  constexpr int NV = NORM;                         // parameter vectors per part
  constexpr bool READ_X = !BWD || NORM != 0;       // without a norm the gradient needs no x
  // The next rows wait in registers, or - two rows of two tensors would take 32 - in 16-byte slots
  // of shared memory that the thread copies to and reads back itself.
  constexpr bool ASYNC = BWD && R > 1;
  static_assert(!ASYNC || sizeof(P) == 16, "cp.async moves 16 bytes here");
  // dynamic shared memory: gradient sums [2][NV][16][threads] (backward), the threads' slots
  // [R][SPT][2][x, dy][threads] (two rows backward), three buffers of row
  // addresses [rows] (where x and dy are read; where the result goes, and the row's angles),
  // parameters [2][NV][hd4], three buffers of angles [tile][pstride]
  extern __shared__ __align__(16) float head_smem[];
  float* const sums = head_smem;
  P* const slots = reinterpret_cast<P*>(sums + (BWD ? 2 * NV * 16 * BLOCK : 0)) + threadIdx.x;
  HeadSource* const sources = reinterpret_cast<HeadSource*>(slots - threadIdx.x + (ASYNC ? R * SPT * 4 * BLOCK : 0));
  HeadTarget* const targets = reinterpret_cast<HeadTarget*>(sources + 3 * a.rows);
  float* const par = reinterpret_cast<float*>(targets + 3 * a.rows);
  float* const tables = par + 2 * NV * a.hd4;
  const int table_floats = a.tile * a.pstride;

  const int tid = threadIdx.x;
  const int tph = FULL != 0 ? FULL : a.tph;
  const int lane = tid & (tph - 1);
  const int group = tid / tph;
  const int groups = BLOCK / tph;
  const int glog = 31 - __clz(groups);
  const int nslots = SPT * tph;
  const int pairs = a.pairs;
  const int vectors = a.hd / V;

  griddep_launch_dependents();
  griddep_wait();
  // this thread's vectors
  int col[SPT][2];
  int slot_of[SPT];
  bool valid[SPT][2], rot[SPT][2], ok[SPT];
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    int s = lane + i * tph;
    ok[i] = !PAD || 2 * s < vectors;
    if (!ok[i]) s = vectors / 2 - 1;
    slot_of[i] = s;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      col[i][h] = head_col<V, IL, FULL>(s, h, pairs, a.hd);
      valid[i][h] = FULL != 0 || (!IL && s * V < pairs) || 2 * s + h < vectors;
      rot[i][h] = (FULL != 0 && !PAD) ||
                  ((!IL || V == 1) ? s * V < pairs : col[i][h] < 2 * pairs);
    }
  }

  // A tile's block of tokens and its first step (a step is one row for every group).
  auto place = [&](int64_t tile, int64_t& block, int& first) {
    block = tile;
    first = 0;
    if (a.pieces > 1) {
      block = tile / a.pieces;
      first = static_cast<int>(tile - block * a.pieces) * a.steps;
    }
  };
  // Where row i of a tile begins; nowhere for the rows that fill up a part's last step or lie
  // behind the last token.
  auto row_at = [&](unsigned n0, int tokens, int first, int i, HeadSource& src, HeadTarget& dst) {
    const int part = first + (i >> glog) >= a.q_steps ? 1 : 0;
    const HeadPart& hp = a.part[part];
    const int u = i + ((first - (part ? a.q_steps : 0)) << glog);
    const int lt = static_cast<int>(fast_div(static_cast<unsigned>(u), hp.div));
    const int h = u - lt * hp.heads;
    src = {nullptr, nullptr};
    dst = {nullptr, 0, 0};
    if (lt < tokens) {
      const unsigned n = n0 + lt, b = fast_div(n, a.tdiv);
      const int64_t t = n - b * static_cast<unsigned>(a.T);
      src.x = static_cast<const T*>(hp.x) + (b * hp.xs[0] + t * hp.xs[1] + static_cast<int64_t>(h) * hp.xs[2]);
      if constexpr (BWD) src.dy = static_cast<const T*>(hp.dy) + (b * hp.ds[0] + t * hp.ds[1] + static_cast<int64_t>(h) * hp.ds[2]);
      dst.out = static_cast<T*>(hp.out) + (b * hp.os[0] + t * hp.os[1] + static_cast<int64_t>(h) * hp.os[2]);
      dst.angles = lt * a.pstride;
    }
  };
  const int a_row = static_cast<int>(fast_div(tid, a.adiv));   // of the angle table
  auto tokens_of = [&](int64_t block) {
    const int64_t left = a.N - block * a.tile;
    return static_cast<int>(left < a.tile ? left : a.tile);
  };
  // The tables of a tile: angles, and where each row begins.
  auto make_tables = [&](int64_t tile, int buf) {
    int64_t block;
    int first;
    place(tile, block, first);
    const int tokens = tokens_of(block);
    const unsigned n0 = static_cast<unsigned>(block * a.tile);
    float* tab = tables + buf * table_floats;
    const int steps = a.all_steps - first < a.steps ? a.all_steps - first : a.steps;
    for (int i = tid; i < steps * groups; i += BLOCK) {
      HeadSource src;
      HeadTarget dst;
      row_at(n0, tokens, first, i, src, dst);
      sources[buf * a.rows + i] = src;
      targets[buf * a.rows + i] = dst;
    }
    // a thread keeps its pair over several tokens
    for (int p = tid - a_row * a.across; a_row < a.down && p < pairs; p += a.across) {
      const int axis = __ldg(a.pair_axis + p);
      const bool turns_p = axis >= 0 && axis < a.axes;
      const double freq = __ldg(a.inv_freq + p) * 0.15915494309189533577;   // 1 / (2 pi): in turns
      float* const cos_p = tab + head_table_at<V, IL, FULL>(p, false, nslots, a.hd);
      float* const sin_p = tab + head_table_at<V, IL, FULL>(p, true, nslots, a.hd);
      for (int lt = a_row; lt < tokens; lt += a.down) {
        float c = 1.f, s = 0.f;
        if (turns_p) {
          const unsigned n = n0 + lt, b = fast_div(n, a.tdiv);
          const int64_t at = axis * a.ps[0] + b * a.ps[1] + static_cast<int64_t>(n - b * static_cast<unsigned>(a.T)) * a.ps[2];
          const double pos = a.pos64 ? static_cast<double>(__ldg(static_cast<const long long*>(a.positions) + at))
                                     : static_cast<double>(__ldg(static_cast<const int*>(a.positions) + at));
          const double turns = pos * freq, part = turns - rint(turns);
          const float rounded = static_cast<float>(part);
          sincospif(2.f * rounded, &s, &c);
          // What fp32 drops of the fraction turns by d < 1e-7 more.  Left out, it would be twice the
          // error of the functions themselves.
          const float d = 6.28318530717958647692f * static_cast<float>(part - static_cast<double>(rounded));
          const float cd = c * d;
          c = fmaf(-s, d, c);
          s += cd;
        }
        cos_p[lt * a.pstride] = c;
        sin_p[lt * a.pstride] = s;
      }
    }
  };

  P xr[R][SPT][2], dr[R][SPT][2];
  auto slot = [&](int r, int i, int k, int tensor) -> P* {
    return slots + (((r * SPT + i) * 2 + k) * 2 + tensor) * BLOCK;
  };
  auto clear = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < SPT; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          P zero;
#pragma unroll
          for (int e = 0; e < V; ++e) zero.v[e] = Cvt<T>::from_f32(0.f);
          if constexpr (ASYNC) {
            *slot(r, i, k, 0) = zero;
            *slot(r, i, k, 1) = zero;
          } else {
            xr[r][i][k] = dr[r][i][k] = zero;
          }
        }
  };
  // Starts the loads of a group's rows.
  auto fetch = [&](const HeadSource src, int part) {
    if (src.x != nullptr) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const T* xp = static_cast<const T*>(src.x) + (R > 1 ? r * a.part[part].x_row : 0);
        const T* dp = static_cast<const T*>(src.dy) + (R > 1 ? r * a.part[part].d_row : 0);
#pragma unroll
        for (int i = 0; i < SPT; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (valid[i][k]) {
              if constexpr (ASYNC) {
                if constexpr (READ_X) head_copy16(slot(r, i, k, 0), xp + col[i][k]);
                head_copy16(slot(r, i, k, 1), dp + col[i][k]);
              } else {
                if constexpr (READ_X) xr[r][i][k] = load_stream<T, V>(xp, col[i][k]);
                if constexpr (BWD) dr[r][i][k] = load_stream<T, V>(dp, col[i][k]);
              }
            }
      }
    }
    if constexpr (BWD) {
      // a group without a row adds nothing to the parameter sums (a branch of the whole warp,
      // which hardly any warp takes)
      if (__any_sync(0xffffffffu, src.x == nullptr)) {
        if (src.x == nullptr) clear();
      }
    }
  };
  // vectors that no row fills stay zero
  if constexpr (!ASYNC) {
    clear();
  } else if constexpr (FULL == 0) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < SPT; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (!valid[i][k]) *slot(r, i, k, 0) = *slot(r, i, k, 1) = P{};
  }

  auto fill_parameters = [&]() {
    if constexpr (NV > 0) {
      for (int i = tid; i < 2 * NV * a.hd4; i += BLOCK) {
        const int which = i / a.hd4, col = i - which * a.hd4;
        const float* src = NV == 1 ? a.param[2 * which] : a.param[which];
        par[i] = src != nullptr && col < a.hd ? __ldg(src + col) : 0.f;
      }
    }
    // slots behind the rotated pairs turn by nothing
    const int plain = (FULL != 0 ? a.hd / 2 : nslots * V) - pairs;
    for (int i = tid; i < 3 * a.tile * plain; i += BLOCK) {
      const int row = i / plain, p = pairs + i - row * plain;
      tables[row * a.pstride + head_table_at<V, IL, FULL>(p, false, nslots, a.hd)] = 1.f;
      tables[row * a.pstride + head_table_at<V, IL, FULL>(p, true, nslots, a.hd)] = 0.f;
    }
    if constexpr (BWD && NORM != 0) {
      for (int i = tid; i < 2 * NV * 16 * BLOCK; i += BLOCK) sums[i] = 0.f;
    }
  };
  const int64_t tile0 = blockIdx.x;
  {  // the first row is on its way while the first tables are made
    int64_t block;
    int first;
    place(tile0, block, first);
    HeadSource src;
    HeadTarget dst;
    row_at(static_cast<unsigned>(block * a.tile), tokens_of(block), first, group, src, dst);
    fetch(src, first < a.q_steps ? 0 : 1);
  }
  make_tables(tile0, 0);
  fill_parameters();
  __syncthreads();
  int buf = 0;
  for (int64_t tile = tile0; tile < a.tiles; tile += gridDim.x) {
    const bool more = tile + gridDim.x < a.tiles;
    const int next_buf = buf == 2 ? 0 : buf + 1;
    if (more) make_tables(tile + gridDim.x, next_buf);
    if (tile != tile0 || more) __syncthreads();
    int64_t block;
    int first;
    place(tile, block, first);
    const float* tab = tables + buf * table_floats;
    const int end = a.all_steps - first < a.steps ? a.all_steps - first : a.steps;
    int next_part = 0;
    if (more) {
      int64_t next_block;
      int next_first;
      place(tile + gridDim.x, next_block, next_first);
      next_part = next_first < a.q_steps ? 0 : 1;
    }
    const int q_end = a.q_steps - first < end ? (a.q_steps > first ? a.q_steps - first : 0) : end;
#pragma unroll 1
    for (int part = q_end > 0 ? 0 : 1; part < a.parts; ++part) {
      const int stop = part == 0 ? q_end : end;
      const HeadPart& hp = a.part[part];
      E g[SPT][2][NE], dg[SPT][2][NE], db[SPT][2][NE];
#pragma unroll
      for (int i = 0; i < SPT; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if constexpr (NORM != 0)
            head_lanes<V>(par + part * NV * a.hd4 + (valid[i][k] ? col[i][k] : 0), g[i][k]);
        }
      float* const mine = sums + part * NV * 16 * BLOCK + tid * HeadTraits<V>::CW;
      if constexpr (BWD && NORM != 0) {
#pragma unroll
        for (int i = 0; i < SPT; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            head_sums_load<V, BLOCK>(mine, i * 2 + k, dg[i][k]);
            if constexpr (NORM == 2) head_sums_load<V, BLOCK>(mine + 16 * BLOCK, i * 2 + k, db[i][k]);
          }
      }
#pragma unroll 1
      for (int step = part == 0 ? 0 : q_end; step < stop; ++step) {
        E x[R][SPT][2][NE], d[R][SPT][2][NE];
        if constexpr (ASYNC) asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < SPT; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if constexpr (ASYNC) {
                if constexpr (READ_X) unpack<T, V>(*slot(r, i, k, 0), x[r][i][k]);
                unpack<T, V>(*slot(r, i, k, 1), d[r][i][k]);
              } else {
                if constexpr (READ_X) unpack<T, V>(xr[r][i][k], x[r][i][k]);
                if constexpr (BWD) unpack<T, V>(dr[r][i][k], d[r][i][k]);
              }
            }
        // the group's next rows, of this tile or the next
        if (step + 1 < end) {
          fetch(sources[buf * a.rows + ((step + 1) << glog) + group], step + 1 < q_end ? 0 : 1);
        } else if (more) {
          fetch(sources[next_buf * a.rows + group], next_part);
        }
        const HeadTarget dst = targets[buf * a.rows + (step << glog) + group];
        const bool on = dst.out != nullptr;
        const float* tt = tab + dst.angles;
        if constexpr (BWD) head_rotate<V, IL, -1, FULL, R>(d, tt, nslots, slot_of, rot, pairs);
        if constexpr (NORM == 2) {
          float m[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            m[r] = 0.f;
#pragma unroll
            for (int i = 0; i < SPT; ++i) {
              E acc = M::bcast(0.f);
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < NE; ++e) acc = M::add(acc, x[r][i][k][e]);
              if (ok[i]) m[r] += M::hsum(acc);
            }
          }
          head_reduce<FULL>(m, tph);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const E nm = M::bcast(-m[r] * a.inv_hd);
#pragma unroll
            for (int i = 0; i < SPT; ++i)
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < NE; ++e)
                  x[r][i][k][e] = valid[i][k] ? M::add(x[r][i][k][e], nm) : M::bcast(0.f);
          }
        }
        if constexpr (NORM != 0) {
          // sum of squares; backward: sum gy c and, for mean and variance, sum gy beside it
          constexpr int NR = BWD ? NORM + 1 : 1;
          // squares scaled down by a power of two, as many as a lane adds at once: see rows_fwd_kernel.
          // (Up to 3 % for heads bound by instructions.  Adding again only where a sum overflowed
          // costs the gradient registers: bf16 16384 tokens 91 -> 109 us.)
          constexpr float kSquares = kSquaresOverflow<T> ? 2 * V : 1;
          const E down = M::bcast(1.f / kSquares);
          float red[NR * R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int k = 0; k < NR; ++k) red[r * NR + k] = 0.f;
#pragma unroll
            for (int i = 0; i < SPT; ++i) {
              E acc[NR];
#pragma unroll
              for (int k = 0; k < NR; ++k) acc[k] = M::bcast(0.f);
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                  acc[0] = M::fma(kSquares > 1.f ? M::mul(x[r][i][k][e], down) : x[r][i][k][e], x[r][i][k][e], acc[0]);
                  if constexpr (BWD) {
                    const E gy = M::mul(d[r][i][k][e], g[i][k][e]);
                    acc[1] = M::fma(gy, x[r][i][k][e], acc[1]);
                    if constexpr (NORM == 2) acc[NORM] = M::add(acc[NORM], gy);
                  }
                }
#pragma unroll
              for (int k = 0; k < NR; ++k)   // shares of means: no overflow in the sum over the lanes
                if (ok[i]) red[r * NR + k] += M::hsum(acc[k]) * (k == 0 ? a.inv_hd * kSquares : a.inv_hd);
            }
          }
          head_reduce<FULL>(red, tph);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            // a group without a row must not put 0 * inf into the parameter sums
            const float inv = on ? rsqrtf(red[r * NR] + a.eps) : 0.f;
            const E iv = M::bcast(inv);
            if constexpr (BWD) {
              const E nm1 = M::bcast(-red[r * NR + 1] * inv);
              const E nm0 = M::bcast(NORM == 2 ? -red[r * NR + NORM] : 0.f);
#pragma unroll
              for (int i = 0; i < SPT; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                  for (int e = 0; e < NE; ++e) {
                    E& de = d[r][i][k][e];
                    const E xh = M::mul(x[r][i][k][e], iv);
                    dg[i][k][e] = M::fma(de, xh, dg[i][k][e]);
                    if constexpr (NORM == 2) db[i][k][e] = M::add(db[i][k][e], de);
                    const E gy = NORM == 2 ? M::fma(de, g[i][k][e], nm0) : M::mul(de, g[i][k][e]);
                    de = M::mul(M::fma(nm1, xh, gy), iv);
                  }
            } else {
#pragma unroll
              for (int i = 0; i < SPT; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  E be[NE];   // the offsets stay in shared memory: registers are short here
                  if constexpr (NORM == 2)
                    head_lanes<V>(par + (part * NV + 1) * a.hd4 + (valid[i][k] ? col[i][k] : 0), be);
#pragma unroll
                  for (int e = 0; e < NE; ++e) {
                    const E xh = M::mul(x[r][i][k][e], iv);
                    x[r][i][k][e] = NORM == 2 ? M::fma(xh, g[i][k][e], be[e]) : M::mul(xh, g[i][k][e]);
                  }
                }
            }
          }
        }
        if constexpr (!BWD) head_rotate<V, IL, 1, FULL, R>(x, tt, nslots, slot_of, rot, pairs);
        if (on) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            T* op = static_cast<T*>(dst.out) + (R > 1 ? r * hp.o_row : 0);
#pragma unroll
            for (int i = 0; i < SPT; ++i)
#pragma unroll
              for (int k = 0; k < 2; ++k)
                if (valid[i][k] && ok[i]) {
                  if constexpr (BWD) {
                    store_stream<T, V>(op, col[i][k], repack<T, V>(d[r][i][k]));
                  } else {
                    store_stream<T, V>(op, col[i][k], repack<T, V>(x[r][i][k]));
                  }
                }
          }
        }
      }
      if constexpr (BWD && NORM != 0) {
#pragma unroll
        for (int i = 0; i < SPT; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            head_sums_store<V, BLOCK>(mine, i * 2 + k, dg[i][k]);
            if constexpr (NORM == 2) head_sums_store<V, BLOCK>(mine + 16 * BLOCK, i * 2 + k, db[i][k]);
          }
      }
    }
    buf = next_buf;
  }

  if constexpr (BWD && NORM != 0) {
    // the CTA's sums of the groups, in group order: one partial row [parts][NV][hd]
    __syncthreads();
    float* w = a.ws + static_cast<int64_t>(blockIdx.x) * a.parts * NV * a.hd;
    constexpr int CW = HeadTraits<V>::CW;
    for (int o = tid; o < a.parts * NV * 16 * tph; o += BLOCK) {
      const int vec = o / (16 * tph), rest = o - vec * 16 * tph;
      const int el = rest / tph, ln = rest - el * tph;
      const int s = ln + el / (2 * V) * tph, half = el / V % 2;
      const bool in = FULL != 0 ? 2 * s < vectors : (!IL && s * V < pairs) || 2 * s + half < vectors;
      if (!in) continue;
      float t = 0.f;
      for (int gr = 0; gr < groups; ++gr)
        t += sums[(vec * 16 + el / CW * CW) * BLOCK + (gr * tph + ln) * CW + el % CW];
      w[vec * a.hd + head_col<V, IL, FULL>(s, half, pairs, a.hd) + el % V] = t;
    }
  }
}

}  // namespace nvn
