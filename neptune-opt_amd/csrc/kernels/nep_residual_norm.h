// nep_residual_norm.h -- the norms after and before a block, fused with its gate and residual
// scale, and their gradients (gfx950).
//
// Per row of n columns, with the residual stream x, the block's output y, an optional gate g and
// scale s (RMS norms, eps inside the root):
//   u = y rate_y (rate_y = rsqrt(mean y^2 + eps)), c = u gamma_after       or c = y without that norm
//   r = x + s g c          h = r rate_r gamma_before, rate_r = rsqrt(mean r^2 + eps)
// r and h are each rounded once; h is the norm of the unrounded r.
//
// Gradient, for dr of r and dh of h, with k = r rate_r and a = gamma_before dh:
//   dx = dr + rate_r (a - k mean(a k))                 dgamma_before = sum over rows of dh k
//   dc = s g dx      dg = s c dx                       dgamma_after  = sum over rows of dc u
//   dy = rate_y (b - u mean(b u)), b = gamma_after dc  or dy = dc
// The second mean needs dx, and so the first, but is linear in it:
//   sum b u = sum w (dr + rate_r a) - rate_r mean(a k) sum w k,   w = s g gamma_after u,
// so one reduction of three sums serves a row.  x is read again instead of r: the same bytes, and r in
// 32 bits.
//
// HBM-bound: the forward pass reads x and y and writes r and h, the gradient reads x, y, dr and dh and
// writes dx and dy, once each; rows stay in registers as packed words.
#pragma once

namespace nep {

constexpr int kGateNone = 0, kGateRows = 1, kGateGroup = 2;   // a gate row per row, or per group of rows

// A row of up to TPR * NV * VEC columns: slot u of lane t holds the columns from (u TPR + t) VEC.
// ANY: rows of any alignment and width (a slot over the end is taken element by element).
template <class St, int TPR, int NV, bool ANY>
struct NormRow {
  typedef typename St::T T;
  static constexpr int VEC = St::kVec;
  static constexpr int COLS = TPR * NV * VEC;
  __device__ static __forceinline__ int at(int u, int t) { return (u * TPR + t) * VEC; }
  __device__ static __forceinline__ u32x4 edge(const T* p, int e, int n) {
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = e + j < n ? St::load(p + e + j) : 0.0f;
    return St::pack(v);
  }
  // columns past n read as zero
  template <bool STREAM>
  __device__ static __forceinline__ void load(u32x4* w, const T* p, int n, int t, bool live) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int e = at(u, t);
      w[u] = u32x4{0u, 0u, 0u, 0u};
      if (!live) continue;
      if (e + VEC <= n) w[u] = ANY ? load16_any(p + e) : STREAM ? load16(p + e) : load16_cached(p + e);
      else if (ANY && e < n) w[u] = edge(p, e, n);
    }
  }
  __device__ static __forceinline__ void store(T* p, int e, int n, const float* v) {
    if (e + VEC <= n) {
      if constexpr (ANY) store16_any(p + e, St::pack(v));
      else store16(p + e, St::pack(v));
    } else if (ANY && e < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (e + j < n) St::store(p + e + j, v[j]);
    }
  }
};

// N sums over the TPR lanes of a row; `lds` holds N floats per wave and is not read by anyone still
// when the next call writes it (callers alternate between two).
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float* v, float* lds) {
  constexpr int G = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = group_sum<G>(v[i]);
  if constexpr (TPR > 64) {
    constexpr int WPR = TPR / 64;
    const int wave = threadIdx.x >> 6, first = (wave / WPR) * WPR;
    if (lane_id() == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[wave * N + i] = v[i];
    }
    __syncthreads();
    float r[WPR][N];
#pragma unroll
    for (int w = 0; w < WPR; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) r[w][i] = lds[(first + w) * N + i];
#pragma unroll
    for (int s = 1; s < WPR; s *= 2)
#pragma unroll
      for (int w = 0; w < WPR; w += 2 * s)
#pragma unroll
        for (int i = 0; i < N; ++i) r[w][i] += r[w + s][i];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = r[0][i];
  }
}

template <class St, int TPR, int NV, bool ANY, bool AFTER, int GATE, int WG>
__device__ __forceinline__ void residual_norm_forward(
    const typename St::T* __restrict__ x, const typename St::T* __restrict__ y,
    const typename St::T* __restrict__ gate, const typename St::T* __restrict__ after,
    const typename St::T* __restrict__ before, typename St::T* __restrict__ residual,
    typename St::T* __restrict__ normed, float* __restrict__ stats, i64 rows, int n, i64 stride_x,
    i64 stride_y, i64 group, float scale, float eps) {
  typedef NormRow<St, TPR, NV, ANY> Row;
  constexpr int VEC = St::kVec;
  __shared__ float lds[2][WG / 64];
  const int t = threadIdx.x % TPR;
  const i64 row = (i64)blockIdx.x * (WG / TPR) + threadIdx.x / TPR;
  const bool live = row < rows;
  const i64 at = live ? row : 0;
  u32x4 xw[NV], yw[NV], gw[NV], aw[NV], bw[NV];
  Row::template load<true>(yw, y + at * stride_y, n, t, live);
  Row::template load<true>(xw, x + at * stride_x, n, t, live);
  if constexpr (GATE == kGateRows) Row::template load<true>(gw, gate + at * n, n, t, live);
  if constexpr (GATE == kGateGroup) Row::template load<false>(gw, gate + at / group * n, n, t, live);
  if constexpr (AFTER) Row::template load<false>(aw, after, n, t, live);
  Row::template load<false>(bw, before, n, t, live);
  const float mean = 1.0f / (float)n;
  float rate_y = 1.0f;
  if constexpr (AFTER) {
    float total = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      float v[VEC];
      St::unpack(yw[u], v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) total = __builtin_fmaf(v[j], v[j], total);
    }
    row_sums<TPR, 1>(&total, lds[0]);
    rate_y = frsq(__builtin_fmaf(total, mean, eps));
  }
  float r[NV][VEC], total = 0.0f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    float v[VEC], g[VEC], a[VEC];
    St::unpack(xw[u], r[u]);
    St::reunpack(yw[u], v);
    if constexpr (GATE != kGateNone) St::unpack(gw[u], g);
    if constexpr (AFTER) St::unpack(aw[u], a);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float c = v[j];
      if constexpr (AFTER) c = c * rate_y * a[j];
      if constexpr (GATE != kGateNone) c *= g[j];
      r[u][j] = __builtin_fmaf(scale, c, r[u][j]);
      total = __builtin_fmaf(r[u][j], r[u][j], total);
    }
  }
  row_sums<TPR, 1>(&total, lds[1]);
  const float rate_r = frsq(__builtin_fmaf(total, mean, eps));
  if (!live) return;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int e = Row::at(u, t);
    float b[VEC], h[VEC];
    St::unpack(bw[u], b);
#pragma unroll
    for (int j = 0; j < VEC; ++j) h[j] = r[u][j] * rate_r * b[j];
    Row::store(residual + row * n, e, n, r[u]);
    Row::store(normed + row * n, e, n, h);
  }
  if (stats != nullptr && t == 0) {
    stats[2 * row] = rate_y;
    stats[2 * row + 1] = rate_r;
  }
}

// The workgroup's sums of `acc` over its rows (WG / TPR at a time) into fp32 `out`, or rounded into
// `rounded` where the workgroup has seen all rows.
template <class St, int TPR, int NV, int WG>
__device__ __forceinline__ void norm_columns(float (&acc)[NV][St::kVec], float* lds, float* out,
                                             typename St::T* rounded, int n) {
  constexpr int VEC = St::kVec, COLS = TPR * NV * VEC, RPW = WG / TPR;
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  __syncthreads();                                   // the last sums have been read
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int j = 0; j < VEC; j += 4)
      *(u32x4*)(lds + slot * COLS + (u * TPR + t) * VEC + j) =
          u32x4{as_u32(acc[u][j]), as_u32(acc[u][j + 1]), as_u32(acc[u][j + 2]), as_u32(acc[u][j + 3])};
  __syncthreads();
  for (int e = threadIdx.x; e < n; e += WG) {
    float v = lds[e];
    for (int s = 1; s < RPW; ++s) v += lds[s * COLS + e];
    if (rounded != nullptr) St::store(rounded + e, v);
    else out[e] = v;
  }
}

// A workgroup of WG lanes walks a chunk of rows, WG / TPR at a time, the next rows' words in flight
// under the arithmetic of these, and keeps the column sums in registers: one partial row per workgroup
// and quantity (256 workgroups: 3% of the bytes at 16384 x 4096).
//   chunks: `per_group` chunks of `chunk` rows in each gate group, or (per_group 0) one chunk of
//   `chunk` whole groups of `group` rows.
//   sums: fp32 [2][chunks][n] for dgamma_after and dgamma_before, then [chunks][n] for the gate's
//   (only with per_group > 1; a group that one workgroup sees whole is written rounded).
template <class St, int TPR, int NV, bool ANY, bool AFTER, int GATE, int WG>
__device__ __forceinline__ void residual_norm_backward(
    const typename St::T* __restrict__ dres, const typename St::T* __restrict__ dnormed,
    const typename St::T* __restrict__ x, const typename St::T* __restrict__ y,
    const typename St::T* __restrict__ gate, const typename St::T* __restrict__ after,
    const typename St::T* __restrict__ before, const float* __restrict__ stats,
    typename St::T* __restrict__ dx, typename St::T* __restrict__ dy,
    typename St::T* __restrict__ dgate, typename St::T* __restrict__ dafter,
    typename St::T* __restrict__ dbefore, float* __restrict__ sums, i64 rows, int n, i64 stride_dr,
    i64 stride_dn, i64 stride_x, i64 stride_y, i64 group, i64 chunk, i64 per_group, float scale) {
  typedef NormRow<St, TPR, NV, ANY> Row;
  constexpr int VEC = St::kVec, RPW = WG / TPR, COLS = Row::COLS;
  __shared__ __attribute__((aligned(16))) float lds[RPW * COLS];
  __shared__ float sums3[2][3 * (WG / 64)];
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const float mean = 1.0f / (float)n;
  const i64 chunks = gridDim.x;
  // 16 columns a lane and more: their sums and words leave no registers for the next row's words or
  // for the gammas and the gate, which come from the caches at each row instead
  constexpr bool kLean = NV * VEC >= 16;
  u32x4 aw[NV], bw[NV], gw[NV];
  auto weights = [&](i64 gi) {
    if constexpr (AFTER) Row::template load<false>(aw, after, n, t, true);
    Row::template load<false>(bw, before, n, t, true);
    if constexpr (GATE == kGateGroup) Row::template load<false>(gw, gate + gi * n, n, t, true);
  };
  float da[NV][VEC], db[NV][VEC], dg[NV][VEC];
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int j = 0; j < VEC; ++j) da[u][j] = db[u][j] = dg[u][j] = 0.0f;

  const i64 g0 = per_group ? blockIdx.x / per_group : blockIdx.x * chunk;
  const i64 g1 = per_group ? g0 + 1 : (g0 + chunk < rows / group ? g0 + chunk : rows / group);
  int turn = 0;
  for (i64 gi = g0; gi < g1; ++gi) {
    const i64 first = gi * group + (per_group ? blockIdx.x % per_group * chunk : 0);
    const i64 end = per_group && first + chunk < (gi + 1) * group ? first + chunk : (gi + 1) * group;
    if constexpr (!kLean) weights(gi);
    u32x4 nx[NV], ny[NV], nr[NV], nh[NV], ng[GATE == kGateRows ? NV : 1];
    float nrate_y = 0.0f, nrate_r = 0.0f;
    auto fetch = [&](i64 base) {
      const i64 row = base + slot;
      const bool live = row < end;
      const i64 at = live ? row : 0;
      Row::template load<true>(nx, x + at * stride_x, n, t, live);
      Row::template load<true>(ny, y + at * stride_y, n, t, live);
      Row::template load<true>(nr, dres + at * stride_dr, n, t, live && dres != nullptr);
      Row::template load<true>(nh, dnormed + at * stride_dn, n, t, live);
      if constexpr (GATE == kGateRows) Row::template load<true>(ng, gate + at * n, n, t, live);
      nrate_y = live ? stats[2 * at] : 0.0f;         // (a lane group without a row adds zeros)
      nrate_r = live ? stats[2 * at + 1] : 0.0f;
    };
    if (!kLean && first < end) fetch(first);
    for (i64 base = first; base < end; base += RPW) {
      const i64 row = base + slot;
      const bool live = row < end;
      if constexpr (kLean) {
        fetch(base);
        weights(gi);
      }
      u32x4 xw[NV], yw[NV], rw[NV], hw[NV];
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        xw[u] = nx[u];
        yw[u] = ny[u];
        rw[u] = nr[u];
        hw[u] = nh[u];
        if constexpr (GATE == kGateRows) gw[u] = ng[u];
      }
      const float rate_y = AFTER ? nrate_y : 1.0f, rate_r = nrate_r;
      if (!kLean && base + RPW < end) fetch(base + RPW);
      // per element: the block's unit output, s g, its share of r, r / its norm, gamma_before dh
      auto element = [&](int u, int j, const float* xv, const float* yv, const float* hv, const float* gv,
                         const float* av, const float* bv, float& unit, float& w, float& c, float& k, float& a) {
        unit = yv[j] * rate_y;
        c = AFTER ? unit * av[j] : unit;
        w = GATE != kGateNone ? scale * gv[j] : scale;
        k = __builtin_fmaf(w, c, xv[j]) * rate_r;
        a = hv[j] * bv[j];
      };
      float s3[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float xv[VEC], yv[VEC], rv[VEC], hv[VEC], gv[VEC], av[VEC], bv[VEC];
        St::unpack(xw[u], xv);
        St::unpack(yw[u], yv);
        St::unpack(rw[u], rv);
        St::unpack(hw[u], hv);
        if constexpr (GATE != kGateNone) St::unpack(gw[u], gv);
        if constexpr (AFTER) St::unpack(aw[u], av);
        St::unpack(bw[u], bv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float unit, w, c, k, a;
          element(u, j, xv, yv, hv, gv, av, bv, unit, w, c, k, a);
          s3[0] = __builtin_fmaf(a, k, s3[0]);
          if constexpr (AFTER) {
            const float wc = w * c;
            s3[1] = __builtin_fmaf(wc, __builtin_fmaf(rate_r, a, rv[j]), s3[1]);
            s3[2] = __builtin_fmaf(wc, k, s3[2]);
          }
        }
      }
      row_sums<TPR, AFTER ? 3 : 1>(s3, sums3[turn]);
      turn ^= 1;
      const float m1 = s3[0] * mean;
      const float m2 = AFTER ? (s3[1] - rate_r * m1 * s3[2]) * mean : 0.0f;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int e = Row::at(u, t);
        float xv[VEC], yv[VEC], rv[VEC], hv[VEC], gv[VEC], av[VEC], bv[VEC], ox[VEC], oy[VEC], og[VEC];
        St::reunpack(xw[u], xv);
        St::reunpack(yw[u], yv);
        St::reunpack(rw[u], rv);
        St::reunpack(hw[u], hv);
        if constexpr (GATE != kGateNone) St::reunpack(gw[u], gv);
        if constexpr (AFTER) St::reunpack(aw[u], av);
        St::reunpack(bw[u], bv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float unit, w, c, k, a;
          element(u, j, xv, yv, hv, gv, av, bv, unit, w, c, k, a);
          ox[j] = __builtin_fmaf(rate_r, __builtin_fmaf(-k, m1, a), rv[j]);
          const float dc = w * ox[j];
          if constexpr (AFTER) {
            oy[j] = rate_y * __builtin_fmaf(-unit, m2, dc * av[j]);
            da[u][j] = __builtin_fmaf(dc, unit, da[u][j]);
          } else {
            oy[j] = dc;
          }
          db[u][j] = __builtin_fmaf(hv[j], k, db[u][j]);
          if constexpr (GATE != kGateNone) {
            og[j] = scale * ox[j] * c;
            if constexpr (GATE == kGateGroup) dg[u][j] += og[j];
          }
        }
        if (!live) continue;
        Row::store(dx + row * n, e, n, ox);
        Row::store(dy + row * n, e, n, oy);
        if constexpr (GATE == kGateRows) Row::store(dgate + row * n, e, n, og);
      }
    }
    if constexpr (GATE == kGateGroup) {
      const bool whole = per_group <= 1;
      norm_columns<St, TPR, NV, WG>(dg, lds, sums + (2 * chunks + blockIdx.x) * n,
                                    whole ? dgate + gi * n : nullptr, n);
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) dg[u][j] = 0.0f;
    }
  }
  if constexpr (AFTER)
    norm_columns<St, TPR, NV, WG>(da, lds, sums + (i64)blockIdx.x * n, chunks == 1 ? dafter : nullptr, n);
  norm_columns<St, TPR, NV, WG>(db, lds, sums + (chunks + blockIdx.x) * n, chunks == 1 ? dbefore : nullptr, n);
}

// Column sums of `count` fp32 partial rows, in their order within each of 8 interleaved runs and
// then over the runs.  A workgroup of 256 takes 32 columns of one output row: blockIdx.y 0 and 1 are
// dgamma_after and dgamma_before (over all chunks), 2 + i is gate group i (over its per_group chunks).
template <class St>
__device__ __forceinline__ void residual_norm_join(const float* __restrict__ sums,
                                                   typename St::T* __restrict__ dafter,
                                                   typename St::T* __restrict__ dbefore,
                                                   typename St::T* __restrict__ dgate, int n, i64 chunks,
                                                   i64 per_group) {
  __shared__ float part[8][32];
  const int c = threadIdx.x & 31, run = threadIdx.x >> 5, e = blockIdx.x * 32 + c;
  const i64 which = blockIdx.y;
  typename St::T* out = which == 0 ? dafter : which == 1 ? dbefore : dgate + (which - 2) * n;
  if (which == 0 && dafter == nullptr) return;
  const i64 first = which < 2 ? which * chunks : 2 * chunks + (which - 2) * per_group;
  const i64 count = which < 2 ? chunks : per_group;
  float v = 0.0f;
  if (e < n) {
    const float* p = sums + first * n + e;
    i64 i = run;
    for (; i + 24 < count; i += 32) {
      const float a = p[i * n], b = p[(i + 8) * n], d = p[(i + 16) * n], f = p[(i + 24) * n];
      v += a;
      v += b;
      v += d;
      v += f;
    }
    for (; i < count; i += 8) v += p[i * n];
  }
  part[run][c] = v;
  __syncthreads();
  if (run == 0 && e < n) {
#pragma unroll
    for (int r = 1; r < 8; ++r) v += part[r][c];
    St::store(out + e, v);
  }
}

}  // namespace nep
