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
// writes dx and dy, once each; rows stay in registers as packed words.  Forward bf16 16384 x 4096 91-95 us
// (5.7-5.9 TB/s; one slot a lane, two and four within 4%), 65536 x 256 24 us; gradient 143-146 us, fp32
// 8192 x 4096 138, bf16 16384 x 8192 280; 16384 columns 144-204 us per 0.8 GB (of any
// alignment 192-320), where registers run out.
#pragma once

namespace nep {

typedef float f32x4n __attribute__((ext_vector_type(4)));

constexpr int kGateNone = 0, kGateRows = 1, kGateGroup = 2;   // a gate row per row, or per group of rows

// How rows are read: whole 16-byte words; any alignment and width from one word up; fewer columns than a
// word holds, one by one.
constexpr int kWords = 0, kAnyRows = 1, kFewColumns = 2;
constexpr u32 kBufferWord3 = 0x00020000u;          // gfx9 raw buffer descriptor, dword 3
constexpr u32 kNowhere = 0x80000000u;              // past every buffer: reads as zero, is not written
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, 0x7fffffff, (int)kBufferWord3);
}

// A row of up to TPR * NV * VEC columns: slot u of lane t holds the columns from (u TPR + t) VEC.
//  * kWords: buffer accesses, lanes and rows past the end at an offset past the buffer, so that no
//    access is in a branch: the waits for loads in flight then count the accesses behind them exactly.
//    (In branches each wait is for everything in flight, the next row's loads among it.)
//  * kAnyRows: a slot over the end is loaded from the row's last VEC columns and shifted when it is used
//    (its columns one by one would be waited for in front of the row's arithmetic).
template <class St, int TPR, int NV, int ACCESS>
struct NormRow {
  typedef typename St::T T;
  static constexpr int VEC = St::kVec;
  static constexpr int COLS = TPR * NV * VEC;
  __device__ static __forceinline__ int at(int u, int t) { return (u * TPR + t) * VEC; }
  // Words of the row `local` rows behind row0 (the wavefront's first); to be settled.
  template <bool STREAM>
  __device__ static __forceinline__ void load(u32x4* w, const T* p, i64 row0, i64 stride, int local, bool live,
                                              int n, int t) {
    if constexpr (ACCESS == kWords) {
      const __amdgpu_buffer_rsrc_t r = buffer_at(p + row0 * stride);
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int e = at(u, t);
        const u32 off = live && e < n ? (u32)(local * (int)stride + e) * (u32)sizeof(T) : kNowhere;
        w[u] = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, STREAM ? 2 : 0);
      }
    } else if constexpr (ACCESS == kAnyRows) {
      const T* q = p + row0 * stride + (live ? (i64)local * stride : 0);
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int e = at(u, t);
        w[u] = load16_any(q + (e + VEC <= n ? e : n - VEC));
      }
    } else {
      const T* q = p + row0 * stride + (live ? (i64)local * stride : 0);
      float v[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = j < n && t == 0 ? St::load(q + j) : 0.0f;
      w[0] = St::pack(v);
    }
  }
  // columns past n, and rows that are none, become zero
  __device__ static __forceinline__ void settle(u32x4* w, int n, int t, bool live) {
    if constexpr (ACCESS == kWords) return;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int over = ACCESS == kAnyRows ? at(u, t) + VEC - n : 0;
      if (!live || over >= VEC) {
        w[u] = u32x4{0u, 0u, 0u, 0u};
      } else if (over > 0) {
        u32x4 x = w[u];
        if constexpr (VEC == 8) {
          if (over & 4) x = u32x4{x.z, x.w, 0u, 0u};
          if (over & 2) x = u32x4{x.y, x.z, x.w, 0u};
          if (over & 1)
            x = u32x4{__builtin_amdgcn_alignbit(x.y, x.x, 16), __builtin_amdgcn_alignbit(x.z, x.y, 16),
                      __builtin_amdgcn_alignbit(x.w, x.z, 16), x.w >> 16};
        } else {
          if (over & 2) x = u32x4{x.z, x.w, 0u, 0u};
          if (over & 1) x = u32x4{x.y, x.z, x.w, 0u};
        }
        w[u] = x;
      }
    }
  }
  // a vector of n columns, settled
  __device__ static __forceinline__ void vector(u32x4* w, const T* p, int n, int t) {
    load<false>(w, p, 0, 0, 0, true, n, t);
    settle(w, n, t, true);
  }
  // words v[u] of the row `local` behind row0 of a contiguous output
  __device__ static __forceinline__ void store(T* p, i64 row0, int local, bool live, int u, int n, int t,
                                               const float* v) {
    const int e = at(u, t);
    if constexpr (ACCESS == kWords) {
      const u32 off = live && e < n ? (u32)(local * n + e) * (u32)sizeof(T) : kNowhere;
      __builtin_amdgcn_raw_buffer_store_b128(St::pack(v), buffer_at(p + row0 * n), off, 0, 2);
    } else if (live) {
      T* q = p + (row0 + local) * n + e;
      if (e + VEC <= n) {
        store16_any(q, St::pack(v));
      } else if (e < n) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (e + j < n) St::store(q + j, v[j]);
      }
    }
  }
};

// A lane's row: `local` rows behind the wavefront's first, which is `first` rows into the workgroup's
// (the same in every lane, so that addresses are scalar).
template <int TPR>
struct LaneRow {
  int first, local;
  __device__ __forceinline__ LaneRow() {
    constexpr int PER = TPR < 64 ? 64 / TPR : 1;     // rows of a wavefront
    first = __builtin_amdgcn_readfirstlane(TPR < 64 ? (int)(threadIdx.x / 64) * PER : (int)(threadIdx.x / TPR));
    local = TPR < 64 ? (int)(threadIdx.x % 64) / TPR : 0;
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
    // every group of WPR lanes reads the waves' sums and adds them (held whole, they would take N WPR
    // registers)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = group_sum<WPR>(lds[(first + lane_id() % WPR) * N + i]);
  }
}

// ---------------------------------------------------------------- an 8-bit output
// h in 8 bits, h ~ scale q: blocks of GROUP columns (of the whole row, 0) have an fp32 scale each,
//   scale = max|h| / M, M the format's largest value, or the least power of two that is no less (POWER),
// and at least 2^-126, the least normal number; q = h / scale rounded to the format, half to even.  A block
// with an infinity or NaN has that for a scale, so that scale q is not finite in any of its columns.
// Seven bytes an element in 16 bits, as the forward pass's eight HBM-bound: bf16 16384 x 4096 gated 79.8 us (5.9
// TB/s), fp16 5331 x 2999 in blocks of 32 20.2 (5.6).
constexpr int kSameType = 0, kE4M3 = 1, kE5M2 = 2, kInt8 = 3;

template <int FORMAT>
struct Format;
template <>
struct Format<kE4M3> {
  static constexpr float kMost = 448.0f;             // 1.75 2^8
  static constexpr u32 kExponent = 8, kFraction = 0x600000u;
  __device__ static __forceinline__ u32 pack(const float* v) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (u32)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  }
};
template <>
struct Format<kE5M2> {
  static constexpr float kMost = 57344.0f;           // 1.75 2^15
  static constexpr u32 kExponent = 15, kFraction = 0x600000u;
  __device__ static __forceinline__ u32 pack(const float* v) {
    const int lo = __builtin_amdgcn_cvt_pk_bf8_f32(v[0], v[1], 0, false);
    return (u32)__builtin_amdgcn_cvt_pk_bf8_f32(v[2], v[3], lo, true);
  }
};
template <>
struct Format<kInt8> {
  static constexpr float kMost = 127.0f;             // (1 + 63/64) 2^6
  static constexpr u32 kExponent = 6, kFraction = 0x7e0000u;
  __device__ static __forceinline__ u32 pack(const float* v) {
    u32 w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float r = __builtin_rintf(v[j]);         // (NaN becomes -127)
      const int i = (int)__builtin_fminf(__builtin_fmaxf(r, -127.0f), 127.0f);
      w |= ((u32)i & 0xffu) << (8 * j);
    }
    return w;
  }
};

// The scale of a block whose largest magnitude has the bits `most` (a NaN's are above an infinity's).
template <int FORMAT, bool POWER>
__device__ __forceinline__ float block_scale(u32 most) {
  typedef Format<FORMAT> F;
  if (most >= 0x7f800000u) return as_f32(most);
  if constexpr (POWER) {
    // up to the next exponent where the fraction is above that of M
    const int b = (int)((most + (0x7fffffu - F::kFraction)) & 0x7f800000u) - (int)(F::kExponent << 23);
    return as_f32((u32)(b > 0x00800000 ? b : 0x00800000));
  }
  return __builtin_fmaxf(div_rn(as_f32(most), F::kMost), 0x1p-126f);
}

template <int G>
__device__ __forceinline__ u32 group_most(u32 v) {
  auto up = [](u32 a, u32 b) { return a > b ? a : b; };
  if constexpr (G >= 2) v = up(v, partner_u32<1>(v));
  if constexpr (G >= 4) v = up(v, partner_u32<2>(v));
  if constexpr (G >= 8) v = up(v, partner_u32<4>(v));
  if constexpr (G >= 16) v = up(v, partner_u32<8>(v));
  if constexpr (G >= 32) v = up(v, partner_u32<16>(v));
  if constexpr (G >= 64) v = up(v, partner_u32<32>(v));
  return v;
}
// over the TPR lanes of a row; `lds` holds a word per wave
template <int TPR>
__device__ __forceinline__ u32 row_most(u32 v, u32* lds) {
  v = group_most<(TPR < 64 ? TPR : 64)>(v);
  if constexpr (TPR > 64) {
    constexpr int WPR = TPR / 64;
    const int wave = threadIdx.x >> 6, first = (wave / WPR) * WPR;
    if (lane_id() == 0) lds[wave] = v;
    __syncthreads();
    v = group_most<WPR>(lds[first + lane_id() % WPR]);
  }
  return v;
}

// Columns (u TPR + t) VEC ... of the row `local` behind row0: VEC values in 8 bits.
template <int FORMAT, int VEC, int ACCESS>
__device__ __forceinline__ void store_8bit(unsigned char* p, i64 row0, int local, bool live, int e, int n,
                                           const float* v) {
  typedef u32 u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
  typedef u32 u32_any __attribute__((aligned(1)));
  u32 w[VEC / 4];
#pragma unroll
  for (int j = 0; j < VEC / 4; ++j) w[j] = Format<FORMAT>::pack(v + 4 * j);
  if constexpr (ACCESS == kWords) {
    const u32 off = live && e < n ? (u32)(local * n + e) : kNowhere;
    const __amdgpu_buffer_rsrc_t r = buffer_at(p + row0 * n);
    if constexpr (VEC == 8) __builtin_amdgcn_raw_buffer_store_b64(u32x2{w[0], w[1]}, r, off, 0, 2);
    else __builtin_amdgcn_raw_buffer_store_b32(w[0], r, off, 0, 2);
  } else if (live) {
    unsigned char* q = p + (row0 + local) * n + e;
    if (e + VEC <= n) {
      if constexpr (VEC == 8) *(u32x2_any*)q = u32x2{w[0], w[1]};
      else *(u32_any*)q = w[0];
    } else if (e < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (e + j < n) q[j] = (unsigned char)(w[j / 4] >> (8 * (j % 4)));
    }
  }
}

// (FORMAT other than kSameType: `normed` is in that format, `scales` has a number per block)
template <class St, int TPR, int NV, int ACCESS, bool AFTER, int GATE, int WG, int FORMAT = kSameType,
          int GROUP = 0, bool POWER = false>
__device__ __forceinline__ void residual_norm_forward(
    const typename St::T* __restrict__ x, const typename St::T* __restrict__ y,
    const typename St::T* __restrict__ gate, const typename St::T* __restrict__ after,
    const typename St::T* __restrict__ before, typename St::T* __restrict__ residual,
    void* __restrict__ normed, float* __restrict__ stats, i64 rows, int n, i64 stride_x,
    i64 stride_y, i64 group, float scale, float eps, float* __restrict__ scales = nullptr) {
  typedef NormRow<St, TPR, NV, ACCESS> Row;
  constexpr int VEC = St::kVec;
  __shared__ float lds[2][WG / 64];
  const int t = threadIdx.x % TPR;
  const LaneRow<TPR> lane;
  const i64 row0 = (i64)blockIdx.x * (WG / TPR) + lane.first, row = row0 + lane.local;
  const bool live = row < rows;
  const i64 safe = row0 < rows ? row0 : 0;           // a wavefront without a row reads the first
  u32x4 xw[NV], yw[NV], gw[NV], aw[NV], bw[NV];
  Row::template load<true>(yw, y, safe, stride_y, lane.local, live, n, t);
  Row::template load<true>(xw, x, safe, stride_x, lane.local, live, n, t);
  if constexpr (GATE == kGateRows) Row::template load<true>(gw, gate, safe, n, lane.local, live, n, t);
  // (rows of one wavefront may be in different groups)
  const i64 gate0 = safe / group;
  if constexpr (GATE == kGateGroup)
    Row::template load<false>(gw, gate, gate0, n, live ? (int)(row / group - gate0) : 0, live, n, t);
  if constexpr (AFTER) Row::template load<false>(aw, after, 0, 0, 0, true, n, t);
  Row::template load<false>(bw, before, 0, 0, 0, true, n, t);
  Row::settle(yw, n, t, live);
  Row::settle(xw, n, t, live);
  if constexpr (GATE != kGateNone) Row::settle(gw, n, t, live);
  if constexpr (AFTER) Row::settle(aw, n, t, true);
  Row::settle(bw, n, t, true);
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
  if constexpr (FORMAT == kSameType) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      float b[VEC], h[VEC];
      St::unpack(bw[u], b);
#pragma unroll
      for (int j = 0; j < VEC; ++j) h[j] = r[u][j] * rate_r * b[j];
      Row::store(residual, row0, lane.local, live, u, n, t, r[u]);
      Row::store((typename St::T*)normed, row0, lane.local, live, u, n, t, h);
    }
  } else {
    // the lanes of a block are neighbours: its columns are a power of two, and so many lanes hold a row or
    // several blocks of one slot
    constexpr int LANES = GROUP == 0 ? TPR : GROUP / VEC < TPR ? GROUP / VEC : TPR;
    static_assert(GROUP == 0 || LANES <= 64, "a block is in one wavefront");
    static_assert(GROUP == 0 || NV == 1 || TPR * VEC % GROUP == 0, "a slot holds whole blocks");
    __shared__ u32 lds_most[WG / 64];
    u32 most[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      float b[VEC];
      St::unpack(bw[u], b);
      Row::store(residual, row0, lane.local, live, u, n, t, r[u]);
      most[u] = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        r[u][j] = r[u][j] * rate_r * b[j];
        const u32 bits = as_u32(r[u][j]) & 0x7fffffffu;
        most[u] = bits > most[u] ? bits : most[u];
      }
      if constexpr (GROUP > 0) most[u] = group_most<LANES>(most[u]);
      else if (u > 0) most[0] = most[u] > most[0] ? most[u] : most[0];
    }
    if constexpr (GROUP == 0) most[0] = row_most<TPR>(most[0], lds_most);
    const int blocks = GROUP == 0 ? 1 : (n + GROUP - 1) / GROUP;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int e = Row::at(u, t);
      const float s = block_scale<FORMAT, POWER>(most[GROUP == 0 ? 0 : u]);
      const float inverse = is_finite(s) ? div_rn(1.0f, s) : 0.0f;
      float h[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        // the quotient, by one step from the product: without it twice as many values land on the other side of
        // a rounding as with a division
        h[j] = r[u][j] * inverse;
        if constexpr (!POWER) h[j] = __builtin_fmaf(__builtin_fmaf(-h[j], s, r[u][j]), inverse, h[j]);
      }
      store_8bit<FORMAT, VEC, ACCESS>((unsigned char*)normed, row0, lane.local, live, e, n, h);
      if (live && e < n && (GROUP == 0 ? u == 0 && t == 0 : t % LANES == 0))
        scales[row * blocks + (GROUP == 0 ? 0 : e / GROUP)] = s;
    }
  }
  if (stats != nullptr && t == 0 && live) {
    stats[2 * row] = rate_y;
    stats[2 * row + 1] = rate_r;
  }
}

// A workgroup's column sums, for each of the three quantities: in registers, or in LDS where a lane has
// 16 columns (its own, so without a barrier).
template <class St, int TPR, int NV, int WG, bool IN_LDS>
struct ColumnSums {
  typedef typename St::T T;
  static constexpr int VEC = St::kVec, COLS = TPR * NV * VEC, RPW = WG / TPR;
  static_assert(!IN_LDS || RPW == 1, "a lane owns its columns");
  float acc[IN_LDS ? 1 : NV][VEC];
  float* lds;      // COLS floats of its own (IN_LDS), or RPW * COLS shared by the workgroup's sums

  __device__ __forceinline__ ColumnSums(float* l, int t) : lds(l) { clear(t); }
  __device__ __forceinline__ f32x4n* at(int u, int t, int j) const {
    return (f32x4n*)(lds + (u * TPR + t) * VEC + j);
  }
  __device__ __forceinline__ void clear(int t) {
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        if constexpr (IN_LDS) *at(u, t, j) = f32x4n{0.0f, 0.0f, 0.0f, 0.0f};
        else acc[u][j] = acc[u][j + 1] = acc[u][j + 2] = acc[u][j + 3] = 0.0f;
      }
  }
  __device__ __forceinline__ void add(int u, int t, const float* v) {
    if constexpr (IN_LDS) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) *at(u, t, j) += f32x4n{v[j], v[j + 1], v[j + 2], v[j + 3]};
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[u][j] += v[j];
    }
  }
  // over the workgroup's rows, into fp32 `out`, or rounded into `rounded` where it has seen them all
  __device__ __forceinline__ void write(int slot, int t, float* out, T* rounded, int n) {
    if constexpr (RPW > 1) {
      __syncthreads();                               // the last sums have been read
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int j = 0; j < VEC; j += 4)
          *(f32x4n*)(lds + slot * COLS + (u * TPR + t) * VEC + j) =
              f32x4n{acc[u][j], acc[u][j + 1], acc[u][j + 2], acc[u][j + 3]};
      __syncthreads();
      for (int e = threadIdx.x; e < n; e += WG) {
        float v = lds[e];
        for (int s = 1; s < RPW; ++s) v += lds[s * COLS + e];
        if (rounded != nullptr) St::store(rounded + e, v);
        else out[e] = v;
      }
    } else {
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int e = (u * TPR + t) * VEC + j;
          if (e >= n) continue;
          float v;
          if constexpr (IN_LDS) v = lds[e];
          else v = acc[u][j];
          if (rounded != nullptr) St::store(rounded + e, v);
          else out[e] = v;
        }
    }
  }
};

// A workgroup of WG lanes walks a chunk of rows, WG / TPR at a time, and keeps the column sums, one
// partial row per workgroup and quantity (256 workgroups: 3% of the bytes at 16384 x 4096).  With up to 8
// columns a lane the next rows' words are in flight under the arithmetic of these, the gammas and the
// gate stay in registers as packed words, and an element's terms are kept from the sums to the results; with 16
// there are no registers for that: a row's words and the gammas are read when it is begun, and the sums of
// dgamma_after and of a group's gate are in LDS.
//   `per_group` workgroups share each group of `group` rows, or (per_group 0) each takes whole groups: between
//   129 and 255 groups, and a little above 256, that leaves CUs idle (bf16 16384 x 4096 in 128 groups 159 us,
//   129 263, 200 174, 256 158, 257 248, 512 157).
//   Rows and groups are dealt in turn, so that the workgroups walk through memory together: in
//   contiguous chunks, 512 KB apart at bf16 16384 x 4096, they meet in the same memory channels (160-166
//   us; in turn 148-150; with exact waits, above, 143-146, 5.6 TB/s).
//   sums: fp32 [2][chunks][n] for dgamma_after and dgamma_before, then [chunks][n] for the gate's
//   (only with per_group > 1; a group that one workgroup sees whole is written rounded).
template <class St, int TPR, int NV, int ACCESS, bool AFTER, int GATE, int WG>
__device__ __forceinline__ void residual_norm_backward(
    const typename St::T* __restrict__ dres, const typename St::T* __restrict__ dnormed,
    const typename St::T* __restrict__ x, const typename St::T* __restrict__ y,
    const typename St::T* __restrict__ gate, const typename St::T* __restrict__ after,
    const typename St::T* __restrict__ before, const float* __restrict__ stats,
    typename St::T* __restrict__ dx, typename St::T* __restrict__ dy,
    typename St::T* __restrict__ dgate, typename St::T* __restrict__ dafter,
    typename St::T* __restrict__ dbefore, float* __restrict__ sums, i64 rows, int n, i64 stride_dr,
    i64 stride_dn, i64 stride_x, i64 stride_y, i64 group, i64 per_group, float scale) {
  typedef NormRow<St, TPR, NV, ACCESS> Row;
  constexpr int VEC = St::kVec, RPW = WG / TPR, COLS = Row::COLS;
  constexpr bool kLean = NV * VEC >= 16;
  constexpr int SHARED = kLean ? (AFTER + (GATE == kGateGroup)) * COLS : RPW > 1 ? RPW * COLS : 0;
  static_assert(!kLean || RPW == 1, "sums of 16 columns a lane are the lane's own");
  static_assert(SHARED >= (kLean && AFTER ? COLS : 0) + (kLean && GATE == kGateGroup ? COLS : 0) &&
                    SHARED >= (RPW > 1 ? RPW * COLS : 0), "the sums' LDS");
  __shared__ __attribute__((aligned(16))) float lds[SHARED ? SHARED : 4];
  __shared__ float sums3[2][3 * (WG / 64)];
  const int t = threadIdx.x % TPR;
  const LaneRow<TPR> lane;
  const int slot = lane.first + lane.local;
  const float mean = 1.0f / (float)n;
  const i64 chunks = gridDim.x;
  // sums that a form has not (da without AFTER, dg without a group's gate) stay out of LDS: no part of it is theirs
  ColumnSums<St, TPR, NV, WG, kLean && AFTER> da(lds, t);
  constexpr int GATE_AT = kLean && AFTER ? COLS : 0;
  ColumnSums<St, TPR, NV, WG, kLean && GATE == kGateGroup> dg(lds + GATE_AT, t);
  ColumnSums<St, TPR, NV, WG, false> db(lds, t);

  // words of gamma_after, gamma_before and the group's gate
  u32x4 aw[NV], bw[NV], gw[NV];
  auto weights = [&](i64 gate_row) {
    if constexpr (AFTER) Row::vector(aw, after, n, t);
    Row::vector(bw, before, n, t);
    if constexpr (GATE == kGateGroup) Row::vector(gw, gate + gate_row * n, n, t);
  };

  const i64 g0 = per_group ? blockIdx.x / per_group : blockIdx.x;
  const i64 g1 = per_group ? g0 + 1 : rows / group, step = RPW * (per_group ? per_group : 1);
  int turn = 0;
  for (i64 gi = g0; gi < g1; gi += chunks) {
    const i64 first = gi * group + (per_group ? blockIdx.x % per_group * RPW : 0), end = (gi + 1) * group;
    if constexpr (!kLean) weights(gi);
    u32x4 nx[NV], ny[NV], nr[NV], nh[NV], ng[GATE == kGateRows ? NV : 1];
    u32x2 nrate;
    // no row: zeros, for a lane group that has none adds them (the addresses are the first row's)
    auto fetch = [&](i64 base) {
      const i64 row0 = base + lane.first, safe = row0 < end ? row0 : first;
      const bool live = row0 + lane.local < end;
      Row::template load<true>(nx, x, safe, stride_x, lane.local, live, n, t);
      Row::template load<true>(ny, y, safe, stride_y, lane.local, live, n, t);
      Row::template load<true>(nr, dres != nullptr ? dres : dnormed, safe, dres != nullptr ? stride_dr : stride_dn,
                               lane.local, live && dres != nullptr, n, t);
      Row::template load<true>(nh, dnormed, safe, stride_dn, lane.local, live, n, t);
      if constexpr (GATE == kGateRows) Row::template load<true>(ng, gate, safe, n, lane.local, live, n, t);
      nrate = __builtin_amdgcn_raw_buffer_load_b64(buffer_at(stats + 2 * safe), live ? 8u * lane.local : kNowhere,
                                                   0, 0);
    };
    if (first >= end) continue;
    if constexpr (!kLean) {
      fetch(first);
      // as many writes as a row makes, to nowhere: the first wait counts what every other does
      if constexpr (ACCESS == kWords) {
        const __amdgpu_buffer_rsrc_t none = buffer_at(dx);
#pragma unroll
        for (int i = 0; i < (GATE == kGateRows ? 3 : 2) * NV; ++i)
          __builtin_amdgcn_raw_buffer_store_b128(u32x4{0u, 0u, 0u, 0u}, none, kNowhere, 0, 2);
      }
    }
    for (i64 base = first; base < end; base += step) {
      const i64 row0 = base + lane.first;
      const bool live = row0 + lane.local < end;
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
      const u32x2 rate = nrate;
      if constexpr (!kLean) {
        fetch(base + step);
        __builtin_amdgcn_sched_barrier(0);
      }
      Row::settle(xw, n, t, live);
      Row::settle(yw, n, t, live);
      Row::settle(rw, n, t, live && dres != nullptr);
      Row::settle(hw, n, t, live);
      if constexpr (GATE == kGateRows) Row::settle(gw, n, t, live);
      const float rate_y = AFTER ? as_f32(rate.x) : 1.0f, rate_r = as_f32(rate.y);
      // an element's unit output, the residual over its norm k, gamma_before dh; its share c and s g are
      // made again from the words (kept too, they would not fit the 128 registers of 1024 lanes)
      struct Terms {
        float unit[VEC], k[VEC], a[VEC];
      };
      auto share = [&](int u, const Terms& e, float* g2, float* c, float* w) {
        if constexpr (AFTER) St::reunpack(aw[u], g2);
        if constexpr (GATE != kGateNone) St::reunpack(gw[u], w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          w[j] = GATE != kGateNone ? scale * w[j] : scale;
          c[j] = AFTER ? e.unit[j] * g2[j] : e.unit[j];
        }
      };
      auto terms = [&](int u, Terms& e, float* g2, float* c, float* w) {
        float xv[VEC], yv[VEC], hv[VEC], bv[VEC];
        St::reunpack(xw[u], xv);
        St::reunpack(yw[u], yv);
        St::reunpack(hw[u], hv);
        St::reunpack(bw[u], bv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) e.unit[j] = yv[j] * rate_y;
        share(u, e, g2, c, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          e.k[j] = __builtin_fmaf(w[j], c[j], xv[j]) * rate_r;
          e.a[j] = hv[j] * bv[j];
        }
      };
      Terms kept[kLean ? 1 : NV];
      float s3[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        Terms& e = kept[kLean ? 0 : u];
        float rv[VEC], g2[VEC], c[VEC], w[VEC];
        terms(u, e, g2, c, w);
        St::reunpack(rw[u], rv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          s3[0] = __builtin_fmaf(e.a[j], e.k[j], s3[0]);
          if constexpr (AFTER) {
            const float wc = w[j] * c[j];
            s3[1] = __builtin_fmaf(wc, __builtin_fmaf(rate_r, e.a[j], rv[j]), s3[1]);
            s3[2] = __builtin_fmaf(wc, e.k[j], s3[2]);
          }
        }
      }
      row_sums<TPR, AFTER ? 3 : 1>(s3, sums3[turn]);
      turn ^= 1;
      const float m1 = s3[0] * mean;
      const float m2 = AFTER ? (s3[1] - rate_r * m1 * s3[2]) * mean : 0.0f;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        Terms& e = kept[kLean ? 0 : u];
        float rv[VEC], hv[VEC], ox[VEC], oy[VEC], og[VEC], ca[VEC], cb[VEC], g2[VEC], c[VEC], w[VEC];
        if constexpr (kLean) terms(u, e, g2, c, w);
        else share(u, e, g2, c, w);
        St::reunpack(rw[u], rv);
        St::reunpack(hw[u], hv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ox[j] = __builtin_fmaf(rate_r, __builtin_fmaf(-e.k[j], m1, e.a[j]), rv[j]);
          const float dc = w[j] * ox[j];
          oy[j] = AFTER ? rate_y * __builtin_fmaf(-e.unit[j], m2, dc * g2[j]) : dc;
          ca[j] = dc * e.unit[j];
          cb[j] = hv[j] * e.k[j];
          og[j] = scale * ox[j] * c[j];
        }
        if constexpr (AFTER) da.add(u, t, ca);
        db.add(u, t, cb);
        if constexpr (GATE == kGateGroup) dg.add(u, t, og);
        Row::store(dx, row0, lane.local, live, u, n, t, ox);
        Row::store(dy, row0, lane.local, live, u, n, t, oy);
        if constexpr (GATE == kGateRows) Row::store(dgate, row0, lane.local, live, u, n, t, og);
      }
    }
    if constexpr (GATE == kGateGroup) {
      dg.write(slot, t, sums + (2 * chunks + blockIdx.x) * n, per_group <= 1 ? dgate + gi * n : nullptr, n);
      dg.clear(t);
    }
  }
  if constexpr (AFTER) da.write(slot, t, sums + (i64)blockIdx.x * n, chunks == 1 ? dafter : nullptr, n);
  db.write(slot, t, sums + (chunks + blockIdx.x) * n, chunks == 1 ? dbefore : nullptr, n);
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
