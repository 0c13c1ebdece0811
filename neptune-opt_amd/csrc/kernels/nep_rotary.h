// nep_rotary.h -- rotary positions of queries and keys, and their gradients (gfx950).
//
// Pair i of the first `part` elements of a head is turned by theta = 2 pi frac(position turns_i):
//   (a, b) -> m (a cos theta - b sin theta, a sin theta + b cos theta)
// with pairs (2i, 2i+1) (interleaved) or (i, i + part/2); the elements from `part` on are copied.  The
// gradient is the transpose: the same with -theta.
//
// Angles: position * turns_i in 64 bits (a position of 2^20 in 32 bits would be off by up to 2^-5 of a
// turn for the fastest pair), reduced there to the nearest quarter turn, so that the 32-bit sine and
// cosine see at most pi/4: their Taylor series to x^9 and x^10 are within 2^-28 of the value there, and
// the quarter turns are exact.
//
// HBM-bound: every element is read once and written once.  A lane owns one 16-byte slot of a token,
// computes its angles once and walks `per` heads with them, queries and keys alike; consecutive lanes are
// consecutive slots, then tokens.  In the half layout the two lanes of a pair of slots exchange their words
// (each half's lanes a power of two, some idle), so that a wavefront reads whole rows of a head; halves
// shorter than a word, or of more lanes than a wavefront has, are read by one lane as two slots.
#pragma once

namespace nep {

// sine and cosine of `turn` full turns
__device__ __forceinline__ void sincos_turns(double turn, float& s, float& c) {
  const double quarters = __builtin_rint(4.0 * turn);
  const float x = (float)(6.283185307179586476925 * __builtin_fma(-0.25, quarters, turn));
  const float z = x * x;
  // x - x^3/3! + ... and 1 - x^2/2! + ... by Horner's rule
  float ps = __builtin_fmaf(z, 2.755731922e-6f, -1.984126984e-4f);
  ps = __builtin_fmaf(z, ps, 8.333333333e-3f);
  ps = __builtin_fmaf(z, ps, -1.666666667e-1f);
  const float sx = __builtin_fmaf(x * z, ps, x);
  float pc = __builtin_fmaf(z, -2.755731922e-7f, 2.480158730e-5f);
  pc = __builtin_fmaf(z, pc, -1.388888889e-3f);
  pc = __builtin_fmaf(z, pc, 4.166666667e-2f);
  pc = __builtin_fmaf(z, pc, -0.5f);
  const float cx = __builtin_fmaf(z, pc, 1.0f);
  const int q = (int)__builtin_fma(-4.0, __builtin_floor(0.25 * quarters), quarters);   // 0..3
  s = (q & 1) ? cx : sx;
  c = (q & 1) ? sx : cx;
  if (q & 2) s = -s;
  if (q == 1 || q == 2) c = -c;
}

constexpr int kHalves = 0, kPairs = 1, kExchanged = 2;
// the word of lane ^ distance (a power of two below 64)
__device__ __forceinline__ u32x4 exchanged(const u32x4& w, int distance) {
  u32x4 r;
  if (distance == 8) {                               // row_ror:8 inside 16 lanes
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (u32)__builtin_amdgcn_mov_dpp((int)w[i], 0x128, 0xF, 0xF, false);
  } else {
    const int from = (lane_id() ^ distance) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (u32)__builtin_amdgcn_ds_bpermute(from, (int)w[i]);
  }
  return r;
}

// One 16-byte slot of a row from element e; ANY: of any alignment, up to `count` elements.
template <class St, bool ANY>
__device__ __forceinline__ u32x4 slot_load(const typename St::T* p, int count) {
  if constexpr (!ANY) return load16(p);
  if (count >= St::kVec) return load16_any(p);
  float v[St::kVec];
#pragma unroll
  for (int j = 0; j < St::kVec; ++j) v[j] = j < count ? St::load(p + j) : 0.0f;
  return St::pack(v);
}
template <class St, bool ANY>
__device__ __forceinline__ void slot_store(typename St::T* p, const u32x4& w, int count) {
  if constexpr (!ANY) {
    store16(p, w);
  } else if (count >= St::kVec) {
    store16_any(p, w);
  } else {
    float v[St::kVec];
    St::unpack(w, v);
#pragma unroll
    for (int j = 0; j < St::kVec; ++j)
      if (j < count) St::store(p + j, v[j]);
  }
}

// tokens = batch * seq; a token has `turned` slots of pairs and then the slots of its copied rest,
// `slots` in all.  Outputs are contiguous [batch, heads, seq, dim].
template <class St, typename Px, int LAYOUT, bool ANY>
__device__ __forceinline__ void rotary(const typename St::T* __restrict__ q,
                                       const typename St::T* __restrict__ k,
                                       const Px* __restrict__ positions,
                                       const double* __restrict__ turns,
                                       typename St::T* __restrict__ qo,
                                       typename St::T* __restrict__ ko, u32 tokens, u32 seq, int dim,
                                       int part, u32 slots, u32 turned, int heads_q, int heads_k,
                                       int per, i64 qsb, i64 qsh, i64 qss, i64 ksb, i64 ksh, i64 kss,
                                       i64 psb, i64 pss, float sign, float magnitude) {
  typedef typename St::T T;
  constexpr int VEC = St::kVec, PAIRS = LAYOUT == kPairs ? VEC / 2 : VEC;
  constexpr int AHEAD = 4;                          // heads in flight per lane
  const u32 id = blockIdx.x * 256u + threadIdx.x;
  const u32 token = id / slots, slot = id - token * slots;
  if (token >= tokens) return;
  const u32 b = token / seq, s = token - b * seq;
  const int half = part / 2;
  const bool turn = slot < turned, second = LAYOUT == kExchanged && turn && slot >= turned / 2;
  // first element and elements of the slot, whose run starts at `from`; of a run that is no multiple of VEC
  // the last slot overlaps its neighbour (both write the same values)
  const int from = !turn ? part : second ? half : 0;
  const int run = !turn ? dim - part : LAYOUT == kPairs ? part : half;
  const int at = (int)(!turn ? slot - turned : second ? slot - turned / 2 : slot) * VEC, back = run - VEC;
  if (at >= run) return;                             // (its partner has none either)
  const int e = from + (ANY && at > back ? (back > 0 ? back : 0) : at);
  const int count = run;
  float cs[PAIRS], sn[PAIRS];
  if (turn) {
    const double at = (double)positions[b * psb + s * pss];
    const int first = LAYOUT == kPairs ? e / 2 : e - from;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const double t = first + i < half ? at * turns[first + i] : 0.0;
      sincos_turns(t, sn[i], cs[i]);
      // (exchanged: the second half's slot is b, and b' = b cos + a sin)
      sn[i] *= LAYOUT == kExchanged && !second ? -(sign * magnitude) : sign * magnitude;
      cs[i] *= magnitude;
    }
  }
  const int h1 = heads_q + heads_k, h0 = blockIdx.y * per, end = h0 + per < h1 ? h0 + per : h1;
  const T* qrow = q + b * qsb + s * qss + e;
  const T* krow = k + b * ksb + s * kss + e;
  T* qout = qo + ((i64)b * heads_q * seq + s) * dim + e;
  T* kout = ko + ((i64)b * heads_k * seq + s) * dim + e;
  const i64 ostep = (i64)seq * dim;
  for (int h = h0; h < end; h += AHEAD) {
    u32x4 w0[AHEAD], w1[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (h + i >= end) continue;
      const T* p = h + i < heads_q ? qrow + (h + i) * qsh : krow + (h + i - heads_q) * ksh;
      w0[i] = slot_load<St, ANY>(p, count);
      if (LAYOUT == kHalves && turn) w1[i] = slot_load<St, ANY>(p + half, count);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (h + i >= end) continue;
      T* o = h + i < heads_q ? qout + (h + i) * ostep : kout + (h + i - heads_q) * ostep;
      if (turn) {
        if constexpr (LAYOUT == kExchanged) {
          float own[VEC], other[VEC];
          St::unpack(w0[i], own);
          St::unpack(exchanged(w0[i], (int)turned / 2), other);
#pragma unroll
          for (int j = 0; j < VEC; ++j) own[j] = __builtin_fmaf(other[j], sn[j], own[j] * cs[j]);
          w0[i] = St::pack(own);
        } else if constexpr (LAYOUT == kPairs) {
          float v[VEC];
          St::unpack(w0[i], v);
#pragma unroll
          for (int j = 0; j < PAIRS; ++j) {
            const float a = v[2 * j], c = v[2 * j + 1];
            v[2 * j] = __builtin_fmaf(a, cs[j], -(c * sn[j]));
            v[2 * j + 1] = __builtin_fmaf(a, sn[j], c * cs[j]);
          }
          w0[i] = St::pack(v);
        } else {
          float a[VEC], c[VEC], x[VEC], y[VEC];
          St::unpack(w0[i], a);
          St::unpack(w1[i], c);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            x[j] = __builtin_fmaf(a[j], cs[j], -(c[j] * sn[j]));
            y[j] = __builtin_fmaf(a[j], sn[j], c[j] * cs[j]);
          }
          w0[i] = St::pack(x);
          slot_store<St, ANY>(o + half, St::pack(y), count);
        }
      }
      slot_store<St, ANY>(o, w0[i], count);
    }
  }
}

}  // namespace nep
