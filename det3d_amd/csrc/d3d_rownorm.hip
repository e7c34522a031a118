// Row norms and the join of a block (include/d3d.h, d3d_row_join_*):
//
//   forward   u = post(f);  h = x + alpha s act(g) u;  z = pre(h)            (f absent: h = x)
//   backward  dH = dh + pre^T(dz);  dx = dH;  du = alpha s act(g) dH;  df = post^T(du);  dg = alpha s u act'(g) dH
//             column sums: ds = alpha sum dH act(g) u, dw = sum dz hhat, db = sum dz, and the post norm's from du and fhat
//   norm^T    with xhat = (x - mu) r and d = w dy:  r (d - mean(d) - xhat mean(d xhat));  rms has no mu and no mean(d)
//
// Bound by HBM: a few dozen f32 operations a value against 8 to 40 bytes.  So one pass: T lanes own a row and keep it in
// registers (NV vectors of E values a lane) from the first load to the last store; the sums of a row go over the T lanes, in
// registers up to a wave, through LDS beyond it.  The variance is a second sum over the registers, around the mean that the
// first gave: no cancellation.  The backward pass recomputes u, h and their statistics from x and f (or from their 8-bit
// codes) instead of reading saved ones.
//
// Join of [8192, 4096] bf16 with both norms, a full gate and e4m3 rows: forward 76 us (404 MB, 5.3 TB/s), backward 137 us (471 MB,
// 3.4 TB/s: 700 vector instructions a row and wave, which the SIMDs issue in two thirds of the time), fold 8 us.  Norm of
// [60013, 128] f32 with int8 rows: forward 15 to 20 us, backward 15 us (70 MB each), fold 5 us.  Join of [65021, 64] f32 with the post
// norm alone: forward 10.5 us (50 MB), backward 14 (67 MB), with f in int8 12.6 and 12.6 (54 MB each), fold 5.
#include "d3d_act8.h"
#include <string.h>
#include <type_traits>


template <int T, int NT, int N> __device__ __forceinline__ void row_sum(float *v, float (&lds)[2][N][NT / 64], int &slot) {
  const auto add = [](uint32_t l, uint32_t r) { return __float_as_uint(__uint_as_float(l) + __uint_as_float(r)); };
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = __uint_as_float(a8_lanes<T < 64 ? T : 64>(__float_as_uint(v[k]), add));
  if constexpr (T > 64) {
    constexpr int W = T / 64;  // waves of a row
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) lds[slot][k][wave] = v[k];
    }
    d3d_lds_barrier();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) t += lds[slot][k][first + w];
      v[k] = t;
    }
    slot ^= 1;
  }
}

struct RjArgs {
  D3dRowJoin a;
  D3dRowJoinGrads g;
  float inv_c;
  int pitch;
  float *part;  // backward: the blocks' column sums, [blocks][rj_slabs(sums)][c]
  int sums;
};

// T lanes own a row, NV vectors of E values each; RPB rows to a block of NT threads; ANY: rows of any alignment and width
template <bool BF16_, int T_, int NV_, bool ANY_> struct RjShape {
  static constexpr bool BF16 = BF16_, ANY = ANY_;
  static constexpr int E = BF16_ ? 8 : 4, T = T_, NV = NV_;
  static constexpr int NT = T > 256 ? T : 256, RPB = NT / T, EPL = E * NV;
};

// act(g) and, with DA, its derivative: p = 1 / (1 + 2^(-g log2 e)).  Exponential and reciprocal are the hardware's, one step off at
// most each; what is rounded in the exponent weighs |g|, so p is off by at most (1.25 |g| + 5) 2^-24 of its value (sigmoid(-10) by 9
// steps), and below the smallest normal number (g < -87.3) by as much as that.  The slope is p - p p: for large g, where it
// vanishes, off by at most 5 2^-24 in all
template <bool DA> __device__ __forceinline__ void rj_act(int act, float g, float &a, float &da) {
  const float p = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896341f));
  if (act == D3D_GATE_SIGMOID) {
    a = p;
    if constexpr (DA) da = fmaf(-p, p, p);
  } else {
    a = g * p;
    if constexpr (DA) da = fmaf(a, 1.f - p, p);
  }
}

// a [c] vector's values of this lane (`absent` where there is none, 0 behind its end), times `factor`; kept in registers over the rows
template <class S> __device__ __forceinline__ void rj_vector(const float *w, float absent, float factor, int lane, int c, float *v) {
#pragma unroll
  for (int k = 0; k < S::NV; ++k) {
    const int at = (k * S::T + lane) * S::E;
#pragma unroll
    for (int j = 0; j < S::E; ++j) v[k * S::E + j] = at + j < c ? absent * factor : 0.f;
    if (w == nullptr) continue;
    if constexpr (S::ANY) {
#pragma unroll
      for (int j = 0; j < S::E; ++j)
        if (at + j < c) v[k * S::E + j] = w[at + j] * factor;
    } else if (at < c) {
#pragma unroll
      for (int j = 0; j < S::E; j += 4) {
        const float4 q = *(const float4 *)(w + at + j);
        v[k * S::E + j] = q.x * factor;
        v[k * S::E + j + 1] = q.y * factor;
        v[k * S::E + j + 2] = q.z * factor;
        v[k * S::E + j + 3] = q.w * factor;
      }
    }
  }
}

// v - mu in place (layer) and r; values behind the row's end stay zero
template <class S>
__device__ __forceinline__ float rj_normalise(int kind, float eps, float inv_c, int lane, int c, float *v,
                                              float (&lds1)[2][1][S::NT / 64], int &slot) {
  if (kind == D3D_NORM_LAYER) {
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < S::EPL; ++j) s[0] += v[j];
    row_sum<S::T, S::NT, 1>(s, lds1, slot);
    const float mu = s[0] * inv_c;
#pragma unroll
    for (int k = 0; k < S::NV; ++k) {
      const int at = (k * S::T + lane) * S::E;
#pragma unroll
      for (int j = 0; j < S::E; ++j) v[k * S::E + j] -= (S::ANY ? at + j : at) < c ? mu : 0.f;
    }
  }
  float q[1] = {0.f};
#pragma unroll
  for (int j = 0; j < S::EPL; ++j) q[0] = fmaf(v[j], v[j], q[0]);
  row_sum<S::T, S::NT, 1>(q, lds1, slot);
  return rsqrtf(fmaf(q[0], inv_c, eps));
}

template <class S, int FMT> __global__ void __launch_bounds__(S::NT) row_join_fwd_kernel(RjArgs p) {
  constexpr int E = S::E, T = S::T, NV = S::NV, EB = S::BF16 ? 2 : 4;
  constexpr bool ANY = S::ANY;
  constexpr int GL = A8_GROUP / E < T ? A8_GROUP / E : T;
  using Row = A8Row<S::BF16, E>;
  __shared__ float lds1[2][1][S::NT / 64];
  int slot = 0;
  const D3dRowJoin &a = p.a;
  const int lane = threadIdx.x & (T - 1), sub = threadIdx.x / T;
  const int c = a.c;
  float pw[S::EPL], pb[S::EPL], sc[S::EPL], qw[S::EPL], qb[S::EPL];
  if (a.f) {
    rj_vector<S>(a.post_weight, 1.f, 1.f, lane, c, pw);
    rj_vector<S>(a.post_bias, 0.f, 1.f, lane, c, pb);
    rj_vector<S>(a.scale, 1.f, a.alpha, lane, c, sc);
  }
  if (a.pre_kind) {
    rj_vector<S>(a.pre_weight, 1.f, 1.f, lane, c, qw);
    rj_vector<S>(a.pre_bias, 0.f, 1.f, lane, c, qb);
  }
  for (int64_t base = (int64_t)blockIdx.x * S::RPB; base < a.n; base += (int64_t)gridDim.x * S::RPB) {
    const bool mine = S::RPB == 1 || base + sub < a.n;
    const int64_t row = mine ? base + sub : a.n - 1;
    typename Row::Raw rx[NV], rf[NV], rg[NV];
    float ag = 1.f, dag;
    // every load of the row first
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int at = (k * T + lane) * E;
      const bool in = at < c;
      rx[k] = in ? Row::template get<ANY>((const char *)a.x + row * a.x_stride * EB, at, c) : Row::zero();
      if (a.f) rf[k] = in ? Row::template get<ANY>((const char *)a.f + row * a.f_stride * EB, at, c) : Row::zero();
      if (a.gate_cols > 1) rg[k] = in ? Row::template get<ANY>((const char *)a.gate + row * a.gate_stride * EB, at, c) : Row::zero();
    }
    if (a.gate_cols == 1) A8Row<S::BF16, 1>::load(a.gate, row * a.gate_stride, &ag);
    float h[S::EPL];
#pragma unroll
    for (int k = 0; k < NV; ++k) Row::template open<ANY>(rx[k], (k * T + lane) * E, c, h + k * E);
    if (a.x_codes) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int at = (k * T + lane) * E;
        A8Held<FMT, E, GL>::store(a.x_codes, a.x_scales, row, p.pitch, at, mine && at < p.pitch, h + k * E);
      }
    }
    if (a.f) {
      float f[S::EPL];
#pragma unroll
      for (int k = 0; k < NV; ++k) Row::template open<ANY>(rf[k], (k * T + lane) * E, c, f + k * E);
      if (a.f_codes) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int at = (k * T + lane) * E;
          A8Held<FMT, E, GL>::store(a.f_codes, a.f_scales, row, p.pitch, at, mine && at < p.pitch, f + k * E);
        }
      }
      float r = 1.f;
      if (a.post_kind) r = rj_normalise<S>(a.post_kind, a.post_eps, p.inv_c, lane, c, f, lds1, slot);
      if (a.gate_cols == 1 && a.gate_act != D3D_GATE_NONE) rj_act<false>(a.gate_act, ag, ag, dag);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float g[E];
#pragma unroll
        for (int j = 0; j < E; ++j) g[j] = ag;
        const int at = (k * T + lane) * E;
        if (a.gate_cols > 1) {
          Row::template open<ANY>(rg[k], at, c, g);
          if (a.gate_act != D3D_GATE_NONE) {
#pragma unroll
            for (int j = 0; j < E; ++j) rj_act<false>(a.gate_act, g[j], g[j], dag);
          }
        }
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const int q = k * E + j;
          h[q] = fmaf(sc[q] * g[j], fmaf(f[q] * r, pw[q], pb[q]), h[q]);
        }
        if (mine && at < c) Row::template put<ANY>((char *)a.h + row * c * EB, at, c, h + k * E);
      }
    }
    if (a.pre_kind) {
      const float r = rj_normalise<S>(a.pre_kind, a.pre_eps, p.inv_c, lane, c, h, lds1, slot);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int at = (k * T + lane) * E;
#pragma unroll
        for (int j = 0; j < E; ++j) h[k * E + j] = fmaf(h[k * E + j] * r, qw[k * E + j], qb[k * E + j]);
        if (mine && at < c) Row::template put<ANY>((char *)a.z + row * c * EB, at, c, h + k * E);
      }
    }
  }
}

// The column sums of a launch: which pairs are asked for (bit 0: sum e fhat | sum e with e = act(g) dH, of which the gradients of
// scale, post weight and post bias are multiples; bit 1: sum dz hhat | sum dz, those of pre weight and pre bias)
__host__ __device__ static inline int rj_slabs(int sums) { return ((sums & 1) + (sums >> 1)) * 2; }

// the block's: every lane's sums over the rows that it saw, added over the block's row groups in their order, into the block's slab
template <int E, int T, int NV, int NT>
__device__ __forceinline__ void rj_columns(const float *const *accs, int sums, int c, float *lds, float *dst) {
  constexpr int RPB = NT / T, EPL = E * NV;
  const int lane = threadIdx.x & (T - 1), sub = threadIdx.x / T;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    if (!(sums >> (a / 2) & 1)) continue;
    const float *acc = accs[a];
    if constexpr (RPB == 1) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const int at = (k * T + lane) * E + j;
          if (at < c) dst[at] = acc[k * E + j];
        }
    } else {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < E; ++j) lds[sub * (T * EPL) + (k * T + lane) * E + j] = acc[k * E + j];
      __syncthreads();
      for (int at = threadIdx.x; at < c; at += NT) {
        float t = 0.f;
#pragma unroll
        for (int s = 0; s < RPB; ++s) t += lds[s * (T * EPL) + at];
        dst[at] = t;
      }
    }
    dst += c;
  }
}

// E values of a [c] vector in LDS
template <class S> __device__ __forceinline__ void rj_shared(const float *w, int at, float *v) {
#pragma unroll
  for (int j = 0; j < S::E; j += 4) *(float4 *)(v + j) = *(const float4 *)(w + at + j);
}

// The backward pass keeps x (then h), f, dH and the gate of a row in registers, four column sums over the rows beside them (32
// registers of a lane with 8 values), and the [c] vectors in LDS: with those in registers too it takes 180 of them, two waves to a
// SIMD in place of four, and [8192, 4096] bf16 took 201 us in place of 169 (137 now: no lane branches around its part of the
// vectors, and the sums over lanes leave LDS alone).
// HELD: 0 rows as they are, 1 + format: codes
template <class S, int HELD> __global__ void __launch_bounds__(S::NT, S::EPL > 4 && S::NT < 512 ? 3 : 4) row_join_bwd_kernel(RjArgs p) {
  constexpr int E = S::E, T = S::T, NV = S::NV, EB = S::BF16 ? 2 : 4;
  constexpr bool ANY = S::ANY;
  constexpr int FMT = HELD == 2 ? D3D_ACT8_E4M3 : D3D_ACT8_INT8;
  using Row = A8Row<S::BF16, E>;
  using Code = A8Held<FMT, E, 1>;
  using In = typename std::conditional<HELD != 0, Code, Row>::type;  // what x and f come as
  __shared__ float lds1[2][1][S::NT / 64], lds2[2][2][S::NT / 64], lds3[2][3][S::NT / 64];
  // post weight | post bias | alpha scale | pre weight; behind the rows the block's column sums
  extern __shared__ __attribute__((aligned(16))) float vec[];
  int slot1 = 0, slot2 = 0, slot3 = 0;
  const D3dRowJoin &a = p.a;
  const D3dRowJoinGrads &g = p.g;
  const int lane = threadIdx.x & (T - 1), sub = threadIdx.x / T;
  const int c = a.c;
  constexpr int cp = T * S::EPL;  // the vectors' length in LDS: zeros behind the row's end, so that no lane needs a branch
  const bool has_f = HELD ? a.f_codes != nullptr : a.f != nullptr;
  float *const pw = vec, *const pb = vec + cp, *const sc = vec + 2 * cp, *const qw = vec + 3 * cp;
  for (int i = threadIdx.x; i < cp; i += S::NT) {
    const bool in = i < c;
    pw[i] = !in ? 0.f : (a.post_weight ? a.post_weight[i] : 1.f);
    pb[i] = !in ? 0.f : (a.post_bias ? a.post_bias[i] : 0.f);
    sc[i] = !in ? 0.f : (a.scale ? a.alpha * a.scale[i] : a.alpha);
    qw[i] = !in ? 0.f : (a.pre_weight ? a.pre_weight[i] : 1.f);
  }
  __syncthreads();
  float s_ef[S::EPL], s_e[S::EPL], s_qw[S::EPL], s_qb[S::EPL];
#pragma unroll
  for (int j = 0; j < S::EPL; ++j) s_ef[j] = s_e[j] = s_qw[j] = s_qb[j] = 0.f;

  for (int64_t base = (int64_t)blockIdx.x * S::RPB; base < a.n; base += (int64_t)gridDim.x * S::RPB) {
    const bool mine = S::RPB == 1 || base + sub < a.n;
    const int64_t row = mine ? base + sub : a.n - 1;
    // every load of the row first.  A row behind the last takes part in the sums over lanes with zero gradients
    typename In::Raw rx[NV], rf[NV];
    typename Row::Raw rg[NV], rdh[NV], rdz[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int at = (k * T + lane) * E;
      const bool in = at < c;
      // (x is read for the pre norm's statistics alone; without it h below is computed from zeros and dropped: a branch around that
      // too costs the widest f32 rows registers, [4096, 8191] 297 us in place of 274)
      if constexpr (HELD != 0) {
        rx[k] = in && a.pre_kind ? Code::fetch(a.x_codes, a.x_scales, row, p.pitch, at) : Code::zero();
        if (has_f) rf[k] = in ? Code::fetch(a.f_codes, a.f_scales, row, p.pitch, at) : Code::zero();
      } else {
        rx[k] = in && a.pre_kind ? Row::template get<ANY>((const char *)a.x + row * a.x_stride * EB, at, c) : Row::zero();
        if (has_f) rf[k] = in ? Row::template get<ANY>((const char *)a.f + row * a.f_stride * EB, at, c) : Row::zero();
      }
      rg[k] = in && a.gate_cols > 1 ? Row::template get<ANY>((const char *)a.gate + row * a.gate_stride * EB, at, c) : Row::zero();
      rdz[k] = in && mine && g.dz ? Row::template get<ANY>((const char *)g.dz + row * g.dz_stride * EB, at, c) : Row::zero();
      rdh[k] = in && mine && g.dh ? Row::template get<ANY>((const char *)g.dh + row * g.dh_stride * EB, at, c) : Row::zero();
    }
    float ag = 1.f, dag = 0.f;
    if (a.gate_cols == 1) A8Row<S::BF16, 1>::load(a.gate, row * a.gate_stride, &ag);

    float h[S::EPL], f[S::EPL];  // x, then h, then hhat | f, then fhat
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if constexpr (HELD != 0) Code::unpack(rx[k], h + k * E);
      else Row::template open<ANY>(rx[k], (k * T + lane) * E, c, h + k * E);
    }
    float fr = 1.f;
    if (has_f) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if constexpr (HELD != 0) Code::unpack(rf[k], f + k * E);
        else Row::template open<ANY>(rf[k], (k * T + lane) * E, c, f + k * E);
      }
      if (a.post_kind) {
        fr = rj_normalise<S>(a.post_kind, a.post_eps, p.inv_c, lane, c, f, lds1, slot1);
#pragma unroll
        for (int j = 0; j < S::EPL; ++j) f[j] *= fr;
      }
      if (a.gate_cols == 1) {
        dag = 1.f;
        if (a.gate_act != D3D_GATE_NONE) rj_act<true>(a.gate_act, ag, ag, dag);
      }
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int at = (k * T + lane) * E;
        float m[E], w[E], b[E], s[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
          m[j] = ag;
        }
        if (a.gate_cols > 1) {
          float unused;
          Row::template open<ANY>(rg[k], at, c, m);
          if (a.gate_act != D3D_GATE_NONE) {
#pragma unroll
            for (int j = 0; j < E; ++j) rj_act<false>(a.gate_act, m[j], m[j], unused);
          }
        }
        rj_shared<S>(pw, at, w);
        rj_shared<S>(pb, at, b);
        rj_shared<S>(sc, at, s);
#pragma unroll
        for (int j = 0; j < E; ++j)  // (behind the row's end everything is zero)
          h[k * E + j] = fmaf(s[j] * m[j], fmaf(f[k * E + j], w[j], b[j]), h[k * E + j]);
      }
    }
    float d[S::EPL];  // dH
    if (a.pre_kind) {
      const float hr = rj_normalise<S>(a.pre_kind, a.pre_eps, p.inv_c, lane, c, h, lds1, slot1);
      float s2[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int at = (k * T + lane) * E;
        float dz[E], w[E];
        Row::template open<ANY>(rdz[k], at, c, dz);
        rj_shared<S>(qw, at, w);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const int q = k * E + j;
          h[q] *= hr;
          d[q] = dz[j] * w[j];
          s2[0] = fmaf(d[q], h[q], s2[0]);
          s2[1] += d[q];
        }
        if (mine) {  // (not 0 times a NaN of the last row)
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const int q = k * E + j;
            s_qw[q] = fmaf(dz[j], h[q], s_qw[q]);
            s_qb[q] += dz[j];
          }
        }
      }
      row_sum<T, S::NT, 2>(s2, lds2, slot2);
      const float m2 = s2[0] * p.inv_c, m1 = a.pre_kind == D3D_NORM_LAYER ? s2[1] * p.inv_c : 0.f;
#pragma unroll
      for (int j = 0; j < S::EPL; ++j) d[j] = hr * (fmaf(-h[j], m2, d[j]) - m1);
    } else {
#pragma unroll
      for (int j = 0; j < S::EPL; ++j) d[j] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int at = (k * T + lane) * E;
      float dh[E];
      Row::template open<ANY>(rdh[k], at, c, dh);
      const bool in = at < c;
#pragma unroll
      for (int j = 0; j < E; ++j) d[k * E + j] += dh[j];  // (behind the row's end the mean's share: the scale there is zero)
      if (g.dx && mine && in) Row::template put<ANY>((char *)g.dx + row * c * EB, at, c, d + k * E);
    }
    if (!has_f) continue;
    float s3[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int at = (k * T + lane) * E;
      float m[E], dm[E], dg[E], w[E], b[E], s[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        m[j] = ag;
        dm[j] = 1.f;
      }
      if (a.gate_cols > 1) {  // (act(g) and act'(g) from the gate as it came: cheaper than to keep them)
        Row::template open<ANY>(rg[k], at, c, m);
        if (a.gate_act != D3D_GATE_NONE) {
#pragma unroll
          for (int j = 0; j < E; ++j) rj_act<true>(a.gate_act, m[j], m[j], dm[j]);
        }
      }
      rj_shared<S>(pw, at, w);
      rj_shared<S>(pb, at, b);
      rj_shared<S>(sc, at, s);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int q = k * E + j;
        const float e = d[q] * m[j];
        dg[j] = d[q] * s[j] * fmaf(f[q], w[j], b[j]);
        s3[2] += dg[j];
        dg[j] *= dm[j];
        if (mine) {
          s_ef[q] = fmaf(e, f[q], s_ef[q]);
          s_e[q] += e;
        }
        d[q] = e * s[j] * w[j];
        s3[0] = fmaf(d[q], f[q], s3[0]);
        s3[1] += d[q];
      }
      if (g.dgate && a.gate_cols > 1 && mine && at < c) Row::template put<ANY>((char *)g.dgate + row * c * EB, at, c, dg);
    }
    row_sum<T, S::NT, 3>(s3, lds3, slot3);
    if (g.dgate && a.gate_cols == 1 && mine && lane == 0) {
      const float v = s3[2] * dag;
      A8Row<S::BF16, 1>::store(g.dgate, row, &v);
    }
    const float m2 = s3[0] * p.inv_c, m1 = a.post_kind == D3D_NORM_LAYER ? s3[1] * p.inv_c : 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int at = (k * T + lane) * E;
      if (a.post_kind) {
#pragma unroll
        for (int j = 0; j < E; ++j) d[k * E + j] = fr * (fmaf(-f[k * E + j], m2, d[k * E + j]) - m1);
      }
      if (g.df && mine && at < c) Row::template put<ANY>((char *)g.df + row * c * EB, at, c, d + k * E);
    }
  }
  const float *const accs[4] = {s_ef, s_e, s_qw, s_qb};
  if (p.sums) rj_columns<E, T, NV, S::NT>(accs, p.sums, c, vec, p.part + (int64_t)blockIdx.x * rj_slabs(p.sums) * c);
}

// The blocks' slabs added up, 32 columns a block of threads, 32 parts of the slabs side by side, the parts in a tree (one thread a
// column over all slabs took 117 us for 512 of them: as many dependent loads), and the gradients from the sums: with A = sum e fhat
// and B = sum e,  ds = alpha (w A + b B),  dw = alpha s A,  db = alpha s B
__global__ void __launch_bounds__(1024) row_join_fold_kernel(const float *__restrict__ part, int blocks, int sums, D3dRowJoin a, D3dRowJoinGrads g) {
  __shared__ float lds[2][32][33];
  const int c = a.c, slabs = rj_slabs(sums), x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int tiles = (c + 31) / 32, pair = blockIdx.x / tiles, i = blockIdx.x % tiles * 32 + x;
  const int64_t step = (int64_t)slabs * c;
  float t0 = 0.f, t1 = 0.f;
  if (i < c) {
    const float *src = part + (int64_t)pair * 2 * c + i;
#pragma unroll 8
    for (int b = y; b < blocks; b += 32) {
      t0 += src[b * step];
      t1 += src[b * step + c];
    }
  }
  lds[0][y][x] = t0;
  lds[1][y][x] = t1;
  __syncthreads();
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    if (y < m) {
      lds[0][y][x] += lds[0][y + m][x];
      lds[1][y][x] += lds[1][y + m][x];
    }
    __syncthreads();
  }
  if (y != 0 || i >= c) return;
  t0 = lds[0][0][x];
  t1 = lds[1][0][x];
  if ((sums & 1) && pair == 0) {
    const float s = a.scale ? a.alpha * a.scale[i] : a.alpha;
    if (g.dscale) g.dscale[i] = a.alpha * fmaf(a.post_weight ? a.post_weight[i] : 1.f, t0, a.post_bias ? a.post_bias[i] * t1 : 0.f);
    if (g.dpost_weight) g.dpost_weight[i] = s * t0;
    if (g.dpost_bias) g.dpost_bias[i] = s * t1;
  } else {
    if (g.dpre_weight) g.dpre_weight[i] = t0;
    if (g.dpre_bias) g.dpre_bias[i] = t1;
  }
}

#define RJ_MAXC 8192
// blocks of the backward pass: at most four waves to a SIMD, and behind the first 256 blocks two row groups to a block, since every
// block writes its column sums and the fold reads them ([2057, 333] f32: 15.1 + 5.2 us, with one row group 14.6 + 7.8)
static int rj_blocks_bwd(int64_t n, int rpb, int nt) {
  const int64_t nb = (n + rpb - 1) / rpb, most = 256 * (1024 / nt);
  const int64_t two = nb > 512 ? (nb + 1) / 2 : (nb > 256 ? 256 : nb);
  return (int)(two > most ? most : two);
}

static int rj_check(const D3dRowJoin *a, bool backward, const char *who) {
  D3D_REQUIRE(a, "%s: null pointer", who);
  D3D_REQUIRE(a->dtype == D3D_F32 || a->dtype == D3D_BF16, "%s: dtype %d", who, a->dtype);
  D3D_REQUIRE(a->fmt == D3D_ACT8_INT8 || a->fmt == D3D_ACT8_E4M3, "%s: format %d", who, a->fmt);
  D3D_REQUIRE(a->n >= 1 && a->n < ((int64_t)1 << 40) && a->c >= 1 && a->c <= RJ_MAXC, "%s: %lld rows of %d channels (1 to %d)", who,
              (long long)a->n, a->c, RJ_MAXC);
  const bool held = a->x_codes != nullptr;
  // (without a pre norm the backward pass does not read x: neither it nor its codes are asked for)
  D3D_REQUIRE(a->x || (backward && (held || !a->pre_kind)), "%s: no rows", who);
  D3D_REQUIRE(!a->x || a->x_stride >= a->c, "%s: x rows %lld elements apart", who, (long long)a->x_stride);
  D3D_REQUIRE(!a->f || a->f_stride >= a->c, "%s: f rows %lld elements apart", who, (long long)a->f_stride);
  D3D_REQUIRE(held == (a->x_scales != nullptr) && (a->f_codes != nullptr) == (a->f_scales != nullptr), "%s: codes without scales", who);
  const bool has_f = a->f || a->f_codes;
  D3D_REQUIRE(!backward || !held || !has_f || a->f_codes, "%s: x is held in 8 bits, f is not", who);
  D3D_REQUIRE(!has_f || (backward && !a->f_codes) || held == (a->f_codes != nullptr) || (!a->pre_kind && a->f_codes),
              "%s: x and f are held together", who);
  D3D_REQUIRE(backward || a->f || !a->f_codes, "%s: codes of f without f", who);
  D3D_REQUIRE(a->post_kind >= 0 && a->post_kind <= 2 && a->pre_kind >= 0 && a->pre_kind <= 2, "%s: norm kinds %d, %d", who, a->post_kind, a->pre_kind);
  D3D_REQUIRE(a->post_eps >= 0.f && a->pre_eps >= 0.f, "%s: negative eps", who);
  D3D_REQUIRE(has_f || (a->pre_kind && !a->post_kind && !a->gate && !a->scale), "%s: without f there is the pre norm alone", who);
  D3D_REQUIRE(a->gate ? (a->gate_cols == 1 || a->gate_cols == a->c) && a->gate_stride >= a->gate_cols : a->gate_cols == 0, "%s: gate of %d columns", who, a->gate_cols);
  D3D_REQUIRE(a->gate_act >= D3D_GATE_NONE && a->gate_act <= D3D_GATE_SILU, "%s: gate_act %d", who, a->gate_act);
  D3D_REQUIRE((((uintptr_t)a->x_codes | (uintptr_t)a->f_codes) & 15) == 0, "%s: codes are not aligned to 16 bytes", who);
  return D3D_OK;
}
// may the rows, and the float32 vectors over the channels, be moved 16 bytes at a time?
static bool rj_vectors(const D3dRowJoin *a, const D3dRowJoinGrads *g) {
  const int eb = a->dtype == D3D_BF16 ? 2 : 4;
  bool v = a8_vectors(a->x, a->x_stride, a->c, eb) && a8_vectors(a->f, a->f_stride, a->c, eb) && a8_vectors(a->h, a->c, a->c, eb) &&
           a8_vectors(a->z, a->c, a->c, eb) && a->c % (16 / eb) == 0;
  for (const void *w : {(const void *)a->scale, (const void *)a->post_weight, (const void *)a->post_bias, (const void *)a->pre_weight, (const void *)a->pre_bias})
    v = v && ((uintptr_t)w & 15) == 0;
  if (a->gate_cols > 1) v = v && a8_vectors(a->gate, a->gate_stride, a->c, eb);
  if (g) {
    v = v && a8_vectors(g->dh, g->dh_stride, a->c, eb) && a8_vectors(g->dz, g->dz_stride, a->c, eb) &&
        a8_vectors(g->dx, a->c, a->c, eb) && a8_vectors(g->df, a->c, a->c, eb);
    if (a->gate_cols > 1) v = v && a8_vectors(g->dgate, a->c, a->c, eb);
  }
  return v;
}

// The shape of the launch by the number of 16-byte vectors in a row: the fewest lanes that hold it with one vector each (4 values in
// f32, 8 in bf16); f32 rows of more than 512 vectors take two a lane.  go(RjShape) launches.
template <bool BF16, bool ANY, class Go> static int rj_pick(int c, Go &&go) {
  const int units = (c + (BF16 ? 8 : 4) - 1) / (BF16 ? 8 : 4);
  if (units <= 8) return go(RjShape<BF16, 8, 1, ANY>{});
  if (units <= 16) return go(RjShape<BF16, 16, 1, ANY>{});
  if (units <= 32) return go(RjShape<BF16, 32, 1, ANY>{});
  if (units <= 64) return go(RjShape<BF16, 64, 1, ANY>{});
  if (units <= 128) return go(RjShape<BF16, 128, 1, ANY>{});
  if (units <= 256) return go(RjShape<BF16, 256, 1, ANY>{});
  if (units <= 512) return go(RjShape<BF16, 512, 1, ANY>{});
  if constexpr (BF16) return go(RjShape<BF16, 1024, 1, ANY>{});
  else if (units <= 1024) return go(RjShape<BF16, 512, 2, ANY>{});
  else return go(RjShape<BF16, 1024, 2, ANY>{});
}
template <class Go> static int rj_for(const D3dRowJoin *a, bool vec, Go &&go) {
  if (a->dtype == D3D_BF16) return vec ? rj_pick<true, false>(a->c, go) : rj_pick<true, true>(a->c, go);
  return vec ? rj_pick<false, false>(a->c, go) : rj_pick<false, true>(a->c, go);
}

extern "C" int d3d_row_join_fwd(const D3dRowJoin *a, d3d_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  int rc = rj_check(a, false, "d3d_row_join_fwd");
  if (rc) return rc;
  D3D_REQUIRE((a->h || !a->f) && (a->z || !a->pre_kind), "d3d_row_join_fwd: null output");
  const bool vec = rj_vectors(a, nullptr);
  RjArgs p;
  memset(&p, 0, sizeof(p));
  p.a = *a;
  p.inv_c = 1.f / (float)a->c;
  p.pitch = a8_pitch(a->c);
  rj_for(a, vec, [&](auto shape) {
    using S = decltype(shape);
    const int64_t nb = (a->n + S::RPB - 1) / S::RPB;
    // (a block keeps the [c] vectors in registers from row to row: enough blocks to fill the chip, no more)
    const int64_t most = 256 * (2048 / S::NT);
    const dim3 grid((unsigned)(nb > most ? most : nb));
    if (a->fmt == D3D_ACT8_INT8) hipLaunchKernelGGL((row_join_fwd_kernel<S, D3D_ACT8_INT8>), grid, dim3(S::NT), 0, stream, p);
    else hipLaunchKernelGGL((row_join_fwd_kernel<S, D3D_ACT8_E4M3>), grid, dim3(S::NT), 0, stream, p);
    return D3D_OK;
  });
  D3D_LAUNCH_TRY("row_join_fwd_kernel");
  return D3D_OK;
}

// workspace of the column sums: the blocks' slabs, of one pair of sums where a single result is asked for (two results may belong to
// different pairs).  The rows of a block follow from the width and the type alone
extern "C" size_t d3d_row_join_ws_floats(int64_t n, int c, int dtype, int sums) {
  if (n < 1 || c < 1 || c > RJ_MAXC || sums < 1 || sums > 5 || (dtype != D3D_F32 && dtype != D3D_BF16)) return 0;
  D3dRowJoin a;
  memset(&a, 0, sizeof(a));
  a.c = c;
  a.dtype = dtype;
  const int blocks = rj_for(&a, true, [&](auto shape) {
    using S = decltype(shape);
    return rj_blocks_bwd(n, S::RPB, S::NT);
  });
  return (size_t)blocks * rj_slabs(sums == 1 ? 1 : 3) * (size_t)c;
}

extern "C" int d3d_row_join_bwd(const D3dRowJoin *a, const D3dRowJoinGrads *g, d3d_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  int rc = rj_check(a, true, "d3d_row_join_bwd");
  if (rc) return rc;
  D3D_REQUIRE(g, "d3d_row_join_bwd: null pointer");
  const bool has_f = a->f || a->f_codes;
  D3D_REQUIRE(!g->dh || g->dh_stride >= a->c, "d3d_row_join_bwd: dh rows %lld elements apart", (long long)g->dh_stride);
  D3D_REQUIRE(!g->dz || g->dz_stride >= a->c, "d3d_row_join_bwd: dz rows %lld elements apart", (long long)g->dz_stride);
  D3D_REQUIRE(!g->dz || a->pre_kind, "d3d_row_join_bwd: dz without a pre norm");
  D3D_REQUIRE(has_f || (!g->dh && !g->df), "d3d_row_join_bwd: dh / df without f");
  D3D_REQUIRE(!g->dgate || a->gate, "d3d_row_join_bwd: dgate without a gate");
  D3D_REQUIRE((!g->dscale || a->scale) && (!g->dpost_weight || a->post_weight) && (!g->dpost_bias || a->post_bias) &&
                  (!g->dpre_weight || a->pre_weight) && (!g->dpre_bias || a->pre_bias),
              "d3d_row_join_bwd: the gradient of an absent vector");
  const int sums = (g->dscale || g->dpost_weight || g->dpost_bias ? 1 : 0) | (g->dpre_weight || g->dpre_bias ? 2 : 0);
  const bool vec = rj_vectors(a, g);
  RjArgs p;
  memset(&p, 0, sizeof(p));
  p.a = *a;
  p.g = *g;
  p.inv_c = 1.f / (float)a->c;
  p.pitch = a8_pitch(a->c);
  p.sums = sums;
  const int held = (a->pre_kind ? a->x_codes : a->f_codes) ? 1 + a->fmt : 0;
  int blocks = 0;
  rc = rj_for(a, vec, [&](auto shape) {
    using S = decltype(shape);
    blocks = rj_blocks_bwd(a->n, S::RPB, S::NT);
    if (sums) {
      const size_t need = (size_t)blocks * rj_slabs(sums) * a->c;
      if (!g->ws || g->ws_floats < need)
        return d3d_set_error(D3D_ECAPACITY, "d3d_row_join_bwd: workspace of %zu floats, %zu needed", (size_t)g->ws_floats, need);
      p.part = g->ws;
    }
    const dim3 grid((unsigned)blocks), block(S::NT);
    const size_t lds = (S::RPB > 4 ? S::RPB : 4) * (size_t)S::T * S::EPL * sizeof(float);
    const void *fn = held == 0 ? (const void *)row_join_bwd_kernel<S, 0>
                               : (held == 1 ? (const void *)row_join_bwd_kernel<S, 1> : (const void *)row_join_bwd_kernel<S, 2>);
    if (lds > 48 * 1024) D3D_HIP_TRY(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    if (held == 0) hipLaunchKernelGGL((row_join_bwd_kernel<S, 0>), grid, block, lds, stream, p);
    else if (held == 1) hipLaunchKernelGGL((row_join_bwd_kernel<S, 1>), grid, block, lds, stream, p);
    else hipLaunchKernelGGL((row_join_bwd_kernel<S, 2>), grid, block, lds, stream, p);
    return D3D_OK;
  });
  if (rc) return rc;
  D3D_LAUNCH_TRY("row_join_bwd_kernel");
  if (sums) {
    const unsigned nb = (unsigned)((a->c + 31) / 32 * (rj_slabs(sums) / 2));
    hipLaunchKernelGGL(row_join_fold_kernel, dim3(nb), dim3(1024), 0, stream, p.part, blocks, sums, *a, *g);
    D3D_LAUNCH_TRY("row_join_fold_kernel");
  }
  return D3D_OK;
}
