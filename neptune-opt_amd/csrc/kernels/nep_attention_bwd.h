// nep_attention_bwd.h -- gradients of the online-softmax attention fold on gfx950 MFMA (bf16 or
// fp16 in, fp32 accumulation).
//
// With t_ij = scale q_i.k_j, P_ij = exp(t_ij - lse_i) on the visible pairs (0 elsewhere) and the
// forward pass's O and lse,
//   delta_i = dO_i.O_i - dlse_i        dP_ij = dO_i.v_j       dS_ij = P_ij (dP_ij - delta_i)
//   dV_j = sum_i P_ij dO_i             dK_j = scale sum_i dS_ij q_i
//   dQ_i = scale sum_j dS_ij k_j
// P is recomputed tile by tile from lse, so no score matrix is stored.
//
// Three stages per call, none with an atomic: results do not depend on the order of workgroups.
//  * attention_bwd_rows: delta of every query row, and the rows' start values -lse/scale.
//  * attention_bwd_kv: a workgroup keeps K and V of its keys (in registers, or K in LDS) and walks the query
//    tiles (dK and dV stay in registers, four products per pair).
//  * attention_bwd_q: a workgroup keeps Q and dO of its queries and walks the key tiles (three
//    products per pair).
// The last two share a launch, dQ's workgroups behind the others: apart and together, causal 2x8x1500x128
// 97 and 57 us, 2x16x2048x128 198 and 146, 7x4x576x256 88 and 55, 1x4x8192x128 438 and 284, full
// 8x12x777x64 95 and 90; causal 4x32x4096x128 the same within 1%.  (Long calls of head dim 64 lose 1%, dQ's
// workgroups being three to a CU alone.)  Five products instead of seven, with one stage, would add dQ
// across key blocks: fp32 atomics, whose order changes results, or an fp32 copy of dQ per key block.
//
// Bound by the matrix cores at the rate that this card's power allows a product: full bf16 2x16x4096x128
// takes 760 to 770 us for the call's 962 GFLOP (1260 TFLOP/s), a library product of 8192^3 1165 to 1350.  Causal
// 4x32x4096x128: 1924 GFLOP, and the pairs hidden in tiles on the diagonal, in 1810 to 1940 us from card to card;
// a workgroup's start and end (11 us: its rows, its gradients; one to a CU) are as long for half the tiles, and
// on the diagonal its waves wait for each other (with that, 19 to 22 us).
// Head dim 64 (fp16 full 8x12x777: 69 to 80 us the call) passes as many LDS reads and exponentials for
// half the products, and 7% of rows past the end; its last workgroups leave CUs idle.
//
// Inside a tile P is computed beside the products of dP, dS beside those of dV (in attention_bwd_q P of one
// block beside the next block's S, and dS beside the first half of dQ's products), each LDS read two steps
// before its MFMAs: causal 4x32x4096x128 7% less than in the order S, dP, P, dS, products; full
// 2x16x4096x128 874 us so and 768.  (The same order of blocks in attention_bwd_kv keeps the tile's rows and spills:
// 1009 us, 1065.)
//
// Mapping (v_mfma_f32_32x32x16): attention_bwd_kv computes S[i][j] with A = Q rows from LDS and
// B = K rows in registers, so lane l holds key l % 32 and registers hold queries
// 8*(r/4) + 4*(l/32) + r%4.  That register order is the contraction order of dV^T += dO^T P and
// dK^T += Q^T dS with P and dS straight from the registers as B; their A operand, rows of dO^T and
// Q^T, comes from the same LDS tiles through ds_read_b64_tr_b16 (4 rows of 16 columns per 16
// lanes, transposed), two reads of 4 queries per operand.  attention_bwd_q is the mirror image:
// S^T with A = K rows, B = Q rows in registers, dQ^T += K^T dS^T.
//
// -lse_i/scale and -delta_i are the start values of the S and dP accumulators in attention_bwd_kv
// (per register there), so P = exp2(c S) and dS = P dP without another operation.
//
// P and dS are rounded to the input type for their products (half a step, bf16 2^-8, fp16 2^-11
// relative; the sums are fp32), the rounding that Q, K, V and dO themselves carry.  fp16 holds
// 2^14 P (a normal number down to 2^-28; two more bits are left for a P past 1, which large scores' rounding
// may make) and dS times a power of two that keeps it below 2^15;
// both are divided out of the fp32 sums exactly.  By Cauchy-Schwarz (delta_i + dlse_i averages the dP_ij)
//   |dP_ij - delta_i| <= |dO_i| max|v| + |delta_i| <= 2 |dO_i| max|v| + |dlse_i|
// For dQ_i the power is the query's own, from the first bound.  For dK_j, a sum over queries, the words of
// all of them share one, from the second: of the queries that a wave's keys are walked with, under the mask
// from the tile of its first key on.  A dS below 2^-29 of that bound is a subnormal there, off by up to
// 2^-39 of the bound: it weighs only where every query that a key matters to has a gradient as much
// smaller than another of those queries'.
#pragma once

namespace nep {

constexpr int kBwdTile = 64;            // rows per staged tile

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct BwdIn;
template <>
struct BwdIn<__bf16> {
  static constexpr bool kScaled = false;
  static constexpr float kLift = 0.0f;              // log2 of the factor on P
  static constexpr u32 kExponent = 0x7f807f80u;     // exponent bits of a packed pair
};
template <>
struct BwdIn<_Float16> {
  static constexpr bool kScaled = true;
  static constexpr float kLift = 14.0f;
  static constexpr u32 kExponent = 0x7c007c00u;
};

// Whether one of the two 16-bit values of a word is infinite or NaN (exponent all ones: the
// xor leaves a zero half).  A finite pair never reports; with a non-finite low half the other
// half does not matter.
template <typename T>
__device__ __forceinline__ u32 pair_nonfinite(u32 w) {
  const u32 t = (w & BwdIn<T>::kExponent) ^ BwdIn<T>::kExponent;
  return (t - 0x00010001u) & ~t & 0x80008000u;
}

// Row r of a tile (D 16-bit values, CH = D/8 chunks of 16 bytes) keeps chunk c at position
// c ^ bwd_swizzle(r).  Two kinds of reads meet the 64 LDS banks (256 bytes a clock): 16 consecutive
// rows of one chunk, which must spread over the 16 chunk positions of a bank sweep, and for the
// transposed reads 4 consecutive rows of 4 chunks (one 64-byte window each), so rows differing in
// their low two bits go to different windows.
template <int D>
__device__ __forceinline__ int bwd_swizzle(int row) {
  if constexpr (D >= 128) return ((row & 3) << 2) | ((row >> 2) & 3);
  else return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);   // two rows per sweep
}

// One tile operand's way into LDS: piece i of wave w fills the 1 KB block i*W + w.  LDS chunk L is
// row L / CH, position L % CH.  Where the rows of one round of all waves are a multiple of 16 the
// swizzle is the same in every piece and one offset serves them.
template <int D, int W, int ROWS = kBwdTile>
struct BwdTile {
  static constexpr int CH = D / 8;
  static constexpr int BYTES = ROWS * D * 2;
  static constexpr int PIECES = BYTES / 1024 / W;
  static constexpr int ROUND = 64 * W / CH;            // rows per round
  static constexpr int OFFS = ROUND % 16 == 0 ? 1 : PIECES;
  static_assert(PIECES >= 1, "a wave moves at least one block");
  int offs[OFFS];
  int step;

  __device__ __forceinline__ BwdTile(int wave, int lane, i64 stride) {
#pragma unroll
    for (int i = 0; i < OFFS; ++i) {
      const int chunk = (i * W + wave) * 64 + lane, row = chunk / CH, p = chunk % CH;
      offs[i] = (int)((i64)row * stride * 2) + ((p ^ bwd_swizzle<D>(row)) << 4);
    }
    step = (int)((i64)ROUND * stride * 2);
  }
  // rows [row0, row0 + ROWS) of `base`; those at or past `count` read as zero
  template <typename T>
  __device__ __forceinline__ void load(const T* base, i64 stride, int row0, int count, int wave,
                                       unsigned char* dst) const {
    const int rows = min(ROWS, count - row0);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(base + (i64)row0 * stride), (short)0, (int)(((i64)(rows - 1) * stride + D) * 2),
        (int)kRawBufferWord3);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if constexpr (OFFS == 1) dma16(r, dst + (i * W + wave) * 1024, offs[0] + i * step, 0);
      else dma16(r, dst + (i * W + wave) * 1024, offs[i], 0);
    }
  }
};

// Operand reads of the 32 rows from `sub` of a tile.
template <typename T, int D>
struct BwdRead {
  typedef typename AttnIn<T>::vec8 vec8;
  int row_off, sw, tr_off[2], tr_sw[2];

  __device__ __forceinline__ explicit BwdRead(int lane) {
    const int l32 = lane & 31, hi = lane >> 5;
    row_off = l32 * (D * 2);
    sw = bwd_swizzle<D>(l32) ^ hi;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = 8 * u + 4 * hi + ((lane & 15) >> 2);
      tr_off[u] = row * (D * 2) + (lane & 1) * 8;
      tr_sw[u] = (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ bwd_swizzle<D>(row);
    }
  }
  // row lane % 32, columns [16 s + 8 (lane / 32), + 8)
  __device__ __forceinline__ vec8 row(const unsigned char* tile, int sub, int s) const {
    return *(const vec8*)(tile + sub * (D * 2) + row_off + (((2 * (s & 7)) ^ sw) << 4) + (s >> 3) * 256);
  }
  // column 32 a + lane % 32 of the rows 16 cs + {4 hi + 0..3, 8 + 4 hi + 0..3}
  __device__ __forceinline__ vec8 column(const unsigned char* tile, int sub, int cs, int a) const {
    typedef __attribute__((address_space(3))) s16x4* lds4;
    const unsigned char* p = tile + (sub + 16 * cs) * (D * 2);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds4)(p + tr_off[0] + (((4 * (a & 3)) ^ tr_sw[0]) << 4) + (a >> 2) * 256));
    const s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds4)(p + tr_off[1] + (((4 * (a & 3)) ^ tr_sw[1]) << 4) + (a >> 2) * 256));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 w = __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(vec8, w);
  }
  // whether the 32 rows hold an infinity or NaN (the answer is the wave's)
  __device__ __forceinline__ bool nonfinite(const unsigned char* tile, int sub) const {
    u32 bad = 0;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const u32x4 w = *(const u32x4*)(tile + sub * (D * 2) + row_off +
                                      (((2 * (s & 7)) ^ sw) << 4) + (s >> 3) * 256);
      bad |= pair_nonfinite<T>(w.x) | pair_nonfinite<T>(w.y) | pair_nonfinite<T>(w.z) |
             pair_nonfinite<T>(w.w);
    }
    return __builtin_amdgcn_ballot_w64(bad != 0) != 0;
  }
};

// B operand of contraction step cs from a 32x32 accumulator's packed pairs.
template <typename T>
__device__ __forceinline__ typename AttnIn<T>::vec8 packed_operand(const u32* pk, int cs) {
  u32x4 w;
  w.x = pk[4 * cs + 0];
  w.y = pk[4 * cs + 1];
  w.z = pk[4 * cs + 2];
  w.w = pk[4 * cs + 3];
  return __builtin_bit_cast(typename AttnIn<T>::vec8, w);
}

// fp16's power of two on dS for a bound on |dP_ij - delta_i|, behind the one on P: with bound < 2^e,
// 2^14 P (dP - delta) 2^(1 - e) stays below 2^15.  Returns 1 - e.
__device__ __forceinline__ int bwd_exponent(float bound) {
  const int e = (int)(as_u32(bound) >> 23) - 126;
  return 1 - min(max(e, -100), 100);
}
// The most of `n` bounds that are `step` apart (the wave's).
__device__ __forceinline__ float bwd_most(const float* __restrict__ bounds, int step, int n, int lane) {
  float m = 0.0f;
  for (int i = lane; i < n; i += 64) m = __builtin_fmaxf(m, bounds[step * i]);
  return group_max<64>(m);
}

// delta_i and the start values of every query row, and fp16's bounds.  start[bh][sqp] holds
// -lse/scale + lift (with rows from sq to sqp, a multiple of 64, at -inf: their P is 0), and
// ndelta[bh][sqp] -delta_i (0 there).  A workgroup of 256 threads takes 64 query rows, D/8 lanes a
// row; with fp16 the workgroups behind them take 64 keys each and bound |v|.  bounds: per 64 rows of queries
// (|dO|, |dlse|), then per 64 keys |v|.  Rows with an infinity or NaN are left out of the bounds: what they
// reach is not finite whatever the scale.
// Rows that see at most 64 keys (the first tile under the causal mask) take delta + dlse as the sum of
// P_ij dP_ij over their keys instead: with few keys O is as large as a row of V, and its rounding, times
// dO, weighs on every dS of the row (relative 2-norm errors of dQ and dK, bf16 causal 2x4x77x64, are 1.61
// times a rounded fp32 result's with dO.O and 1.44 so; 1.50 and 1.42 at 900 rows).
// HBM-bound: O and dO are read once (and V in fp16).
template <typename T, int D>
__device__ __forceinline__ void attention_bwd_rows(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ o, const T* __restrict__ go, const T* __restrict__ v,
    const float* __restrict__ lse, const float* __restrict__ glse, float* __restrict__ start,
    float* __restrict__ ndelta, float* __restrict__ bounds, int heads, int sq, int sk, int units,
    i64 qsb, i64 qsh, i64 qss, i64 ksb, i64 ksh, i64 kss, i64 osb, i64 osh, i64 oss, i64 gsb, i64 gsh,
    i64 gss, i64 vsb, i64 vsh, i64 vss, float scale, float scale_log2, int causal) {
  typedef AttnIn<T> In;
  typedef typename In::vec8 vec8;
  constexpr int LPR = D / 8, RPP = 256 / LPR;     // lanes per row, rows per pass
  constexpr bool kScaled = BwdIn<T>::kScaled;
  __shared__ float wmax[2][4];
  __shared__ float dots[2][kBwdTile];
  const int nq = (sq + kBwdTile - 1) / kBwdTile, nk = (sk + kBwdTile - 1) / kBwdTile;
  const int tid = threadIdx.x, c = tid % LPR;
  // tiles of a head whose rows see at most 64 keys: the first workgroups', whose chain of loads and products
  // is longer than the others'
  const int few = sk <= kBwdTile ? nq : causal ? 1 : 0, group = (int)blockIdx.x - units * few;
  if (group < 0) {
    const int id = blockIdx.x, bh = id / few, t = id % few, b = bh / heads, h = bh % heads;
    // a wave takes 32 queries (its lanes) by 32 keys (its registers); rows past the end are the last
    const int wave = tid >> 6, l32 = tid & 31, hi = (tid >> 5) & 1, j0 = 32 * (wave >> 1);
    const int i = t * kBwdTile + 32 * (wave & 1) + l32, qi = min(i, sq - 1), kj = min(j0 + l32, sk - 1);
    const T* qr = q + b * qsb + h * qsh + (i64)qi * qss + 8 * hi;
    const T* gr = go + b * gsb + h * gsh + (i64)qi * gss + 8 * hi;
    const T* kr = k + b * ksb + h * ksh + (i64)kj * kss + 8 * hi;
    const T* vr = v + b * vsb + h * vsh + (i64)kj * vss + 8 * hi;
    const float shift = -lse[(i64)bh * sq + qi] * kLog2e;
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
      s = In::mfma(*(const vec8*)(kr + 16 * x), *(const vec8*)(qr + 16 * x), s);
      dp = In::mfma(*(const vec8*)(vr + 16 * x), *(const vec8*)(gr + 16 * x), dp);
    }
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = j0 + 8 * (r >> 2) + 4 * hi + (r & 3);
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale_log2, shift));
      sum += j < sk && (!causal || j <= i) ? p * dp[r] : 0.0f;
    }
    u32 lower, upper;
    pair_u32<32>(as_u32(sum), lower, upper);
    if (hi == 0) dots[wave >> 1][32 * (wave & 1) + l32] = as_f32(lower) + as_f32(upper);
    __syncthreads();
    const int row = t * kBwdTile + tid;
    if (tid < kBwdTile)
      ndelta[(i64)bh * nq * kBwdTile + row] =
          row < sq ? (glse != nullptr ? glse[(i64)bh * sq + row] : 0.0f) - (dots[0][tid] + dots[1][tid]) : 0.0f;
    return;
  }
  const bool keys = kScaled && group >= units * nq;
  const int id = keys ? group - units * nq : group, n = keys ? nk : nq;
  const int bh = id / n, t = id % n;
  const int b = bh / heads, h = bh % heads;
  float gm = 0.0f, lm = 0.0f;
  if (!keys) {
    const T* op = o + b * osb + h * osh;
    const T* gp = go + b * gsb + h * gsh;
    const i64 row0 = (i64)bh * nq * kBwdTile;
    u32x4 ow[kBwdTile / RPP], gw[kBwdTile / RPP];
#pragma unroll
    for (int i = 0; i < kBwdTile / RPP; ++i) {
      const int row = t * kBwdTile + i * RPP + tid / LPR;
      ow[i] = gw[i] = u32x4{0u, 0u, 0u, 0u};
      if (row < sq) {
        ow[i] = load16_cached(op + (i64)row * oss + 8 * c);
        gw[i] = load16_cached(gp + (i64)row * gss + 8 * c);
      }
    }
#pragma unroll
    for (int i = 0; i < kBwdTile / RPP; ++i) {
      const int row = t * kBwdTile + i * RPP + tid / LPR;
      float dot = 0.0f, g2 = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        dot = __builtin_fmaf(In::lo(ow[i][w]), In::lo(gw[i][w]), dot);
        dot = __builtin_fmaf(In::hi(ow[i][w]), In::hi(gw[i][w]), dot);
        if constexpr (kScaled) {
          g2 = __builtin_fmaf(In::lo(gw[i][w]), In::lo(gw[i][w]), g2);
          g2 = __builtin_fmaf(In::hi(gw[i][w]), In::hi(gw[i][w]), g2);
        }
      }
      dot = group_sum<LPR>(dot);
      float dl = 0.0f;
      if (row < sq && glse != nullptr) dl = glse[(i64)bh * sq + row];
      if constexpr (kScaled) {
        g2 = group_sum<LPR>(g2);
        gm = is_finite(g2) ? __builtin_fmaxf(gm, g2) : gm;
        lm = is_finite(dl) ? __builtin_fmaxf(lm, __builtin_fabsf(dl)) : lm;
      }
      if (c == 0) {
        start[row0 + row] =
            row < sq ? -lse[(i64)bh * sq + row] / scale + BwdIn<T>::kLift / (scale * kLog2e) : -kInf;
        if (t >= few) ndelta[row0 + row] = row < sq ? dl - dot : 0.0f;
      }
    }
  } else {
    const T* vp = v + b * vsb + h * vsh;
#pragma unroll
    for (int i = 0; i < kBwdTile / RPP; ++i) {
      const int row = t * kBwdTile + i * RPP + tid / LPR;
      float v2 = 0.0f;
      if (row < sk) {
        const u32x4 w = load16_cached(vp + (i64)row * vss + 8 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v2 = __builtin_fmaf(In::lo(w[j]), In::lo(w[j]), v2);
          v2 = __builtin_fmaf(In::hi(w[j]), In::hi(w[j]), v2);
        }
      }
      v2 = group_sum<LPR>(v2);
      gm = is_finite(v2) ? __builtin_fmaxf(gm, v2) : gm;
    }
  }
  if constexpr (kScaled) {
    gm = group_max<64>(gm);
    lm = group_max<64>(lm);
    if ((tid & 63) == 0) {
      wmax[0][tid >> 6] = gm;
      wmax[1][tid >> 6] = lm;
    }
    __syncthreads();
    if (tid == 0) {
      float m[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        m[i] = __builtin_fmaxf(__builtin_fmaxf(wmax[i][0], wmax[i][1]),
                               __builtin_fmaxf(wmax[i][2], wmax[i][3]));
      // the fp32 sum of up to 256 squares is within 2^-15 of its value
      const float norm = __builtin_sqrtf(m[0]) * 1.001f;
      if (keys) {
        bounds[(i64)units * nq * 2 + id] = norm;
      } else {
        bounds[2 * id] = norm;
        bounds[2 * id + 1] = m[1];
      }
    }
  }
}

// Gradients of [j0, j0 + count) keys in plain fp32, for a workgroup whose key range shares a tile
// with queries hidden from some of its keys and holding inf or NaN in Q or dO (0 * inf in the
// products above would reach those keys).  16 adjacent lanes hold a key's row (D/16 dims each);
// hidden pairs are skipped.  Of the queries [i_begin, i_end).
template <typename T, int D, bool CAUSAL, int W, class Store>
__device__ void attention_bwd_exact_kv(const T* __restrict__ qp, const T* __restrict__ kp,
                                       const T* __restrict__ vp, const T* __restrict__ gp,
                                       const float* __restrict__ start,
                                       const float* __restrict__ ndelta, int j0, int count, int sk,
                                       int i_begin, int i_end, i64 qss, i64 kss, i64 vss, i64 gss,
                                       float scale, float scale_log2, Store store) {
  typedef AttnIn<T> In;
  constexpr int DQ = D / 16;
  const int tid = threadIdx.x, c = tid & 15;
  for (int r0 = j0; r0 < j0 + count; r0 += W * 4) {
    const int j = r0 + (tid >> 4);
    const bool active = j < sk;
    float kv[DQ], vv[DQ], dk[DQ], dv[DQ];
#pragma unroll
    for (int d = 0; d < DQ; d += 2) {
      const u32 a = active ? *(const u32*)(kp + (i64)j * kss + c * DQ + d) : 0u;
      const u32 b = active ? *(const u32*)(vp + (i64)j * vss + c * DQ + d) : 0u;
      kv[d] = In::lo(a);
      kv[d + 1] = In::hi(a);
      vv[d] = In::lo(b);
      vv[d + 1] = In::hi(b);
      dk[d] = dk[d + 1] = dv[d] = dv[d + 1] = 0.0f;
    }
    for (int i = CAUSAL ? max(i_begin, r0) : i_begin; i < i_end; ++i) {
      const T* qr = qp + (i64)i * qss + c * DQ;
      const T* gr = gp + (i64)i * gss + c * DQ;
      float s = 0.0f, dp = 0.0f;
#pragma unroll
      for (int d = 0; d < DQ; d += 2) {
        const u32 a = *(const u32*)(qr + d), b = *(const u32*)(gr + d);
        s = __builtin_fmaf(In::lo(a), kv[d], s);
        s = __builtin_fmaf(In::hi(a), kv[d + 1], s);
        dp = __builtin_fmaf(In::lo(b), vv[d], dp);
        dp = __builtin_fmaf(In::hi(b), vv[d + 1], dp);
      }
      s = group_sum<16>(s);
      dp = group_sum<16>(dp);
      if (active && (!CAUSAL || i >= j)) {
        const float p =
            __builtin_amdgcn_exp2f((s + start[i]) * scale_log2) * exp2_int(-(int)BwdIn<T>::kLift);
        const float ds = p * (dp + ndelta[i]) * scale;
#pragma unroll
        for (int d = 0; d < DQ; d += 2) {
          const u32 a = *(const u32*)(qr + d), b = *(const u32*)(gr + d);
          dk[d] = __builtin_fmaf(ds, In::lo(a), dk[d]);
          dk[d + 1] = __builtin_fmaf(ds, In::hi(a), dk[d + 1]);
          dv[d] = __builtin_fmaf(p, In::lo(b), dv[d]);
          dv[d + 1] = __builtin_fmaf(p, In::hi(b), dv[d + 1]);
        }
      }
    }
    if (active) {
#pragma unroll
      for (int d = 0; d < DQ; d += 4) {
        store(0, j, c * DQ + d, dk[d], dk[d + 1], dk[d + 2], dk[d + 3]);
        store(1, j, c * DQ + d, dv[d], dv[d + 1], dv[d + 2], dv[d + 3]);
      }
    }
  }
}

// The same for dQ of the queries [i0, i0 + count), over the keys [j_begin, j_end).
template <typename T, int D, bool CAUSAL, int W, class Store>
__device__ void attention_bwd_exact_q(const T* __restrict__ qp, const T* __restrict__ kp,
                                      const T* __restrict__ vp, const T* __restrict__ gp,
                                      const float* __restrict__ start,
                                      const float* __restrict__ ndelta, int i0, int count, int sq,
                                      int j_begin, int j_end, i64 qss, i64 kss, i64 vss, i64 gss,
                                      float scale, float scale_log2, Store store) {
  typedef AttnIn<T> In;
  constexpr int DQ = D / 16;
  const int tid = threadIdx.x, c = tid & 15;
  for (int r0 = i0; r0 < i0 + count; r0 += W * 4) {
    const int i = r0 + (tid >> 4);
    const bool active = i < sq;
    float qv[DQ], gv[DQ], dq[DQ];
#pragma unroll
    for (int d = 0; d < DQ; d += 2) {
      const u32 a = active ? *(const u32*)(qp + (i64)i * qss + c * DQ + d) : 0u;
      const u32 b = active ? *(const u32*)(gp + (i64)i * gss + c * DQ + d) : 0u;
      qv[d] = In::lo(a);
      qv[d + 1] = In::hi(a);
      gv[d] = In::lo(b);
      gv[d + 1] = In::hi(b);
      dq[d] = dq[d + 1] = 0.0f;
    }
    const float st = active ? start[i] : -kInf, nd = active ? ndelta[i] : 0.0f;
    const int end = CAUSAL ? min(j_end, r0 + W * 4) : j_end;
    for (int j = j_begin; j < end; ++j) {
      const T* kr = kp + (i64)j * kss + c * DQ;
      const T* vr = vp + (i64)j * vss + c * DQ;
      float s = 0.0f, dp = 0.0f;
#pragma unroll
      for (int d = 0; d < DQ; d += 2) {
        const u32 a = *(const u32*)(kr + d), b = *(const u32*)(vr + d);
        s = __builtin_fmaf(In::lo(a), qv[d], s);
        s = __builtin_fmaf(In::hi(a), qv[d + 1], s);
        dp = __builtin_fmaf(In::lo(b), gv[d], dp);
        dp = __builtin_fmaf(In::hi(b), gv[d + 1], dp);
      }
      s = group_sum<16>(s);
      dp = group_sum<16>(dp);
      if (active && (!CAUSAL || j <= i)) {
        const float p =
            __builtin_amdgcn_exp2f((s + st) * scale_log2) * exp2_int(-(int)BwdIn<T>::kLift);
        const float ds = p * (dp + nd) * scale;
#pragma unroll
        for (int d = 0; d < DQ; d += 2) {
          const u32 a = *(const u32*)(kr + d);
          dq[d] = __builtin_fmaf(ds, In::lo(a), dq[d]);
          dq[d + 1] = __builtin_fmaf(ds, In::hi(a), dq[d + 1]);
        }
      }
    }
    if (active) {
#pragma unroll
      for (int d = 0; d < DQ; d += 4)
        store(i, c * DQ + d, dq[d], dq[d + 1], dq[d + 2], dq[d + 3]);
    }
  }
}

// S and dP of kernels with more than 256 registers: d = c + a b with d in vector registers, from a zero,
// a given or its own c.  The compiler keeps the accumulators of every MFMA of such a kernel in AGPRs, of
// which there are 256: the gradients take them (all, for dK and dV from head dim 128 up), S and dP beside
// them would spill, and each of their values would cost a move before its exponential.  (`mfma_settle`
// stands between the last of a chain and the first other use of d: the wait states are the program's here,
// 12 after an MFMA of 8 passes, as the compiler leaves after its own; the MFMAs between are among them.)
// B_AGPR: b is kept in AGPRs.
template <typename T, bool B_AGPR>
__device__ __forceinline__ void mfma_vgpr(typename AttnIn<T>::vec8 a, typename AttnIn<T>::vec8 b,
                                          f32x16& c) {
  if constexpr (__is_same(T, __bf16)) {
    if constexpr (B_AGPR) asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "a"(b));
    else asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  } else {
    if constexpr (B_AGPR) asm("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "a"(b));
    else asm("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  }
}
template <typename T>
__device__ __forceinline__ f32x16 mfma_vgpr_from(typename AttnIn<T>::vec8 a, typename AttnIn<T>::vec8 b,
                                                 const f32x16& c) {
  f32x16 d;
  if constexpr (__is_same(T, __bf16))
    asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %3" : "=&v"(d) : "v"(a), "v"(b), "v"(c));
  else
    asm("v_mfma_f32_32x32x16_f16 %0, %1, %2, %3" : "=&v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}
template <typename T, bool B_AGPR>
__device__ __forceinline__ f32x16 mfma_vgpr_zero(typename AttnIn<T>::vec8 a, typename AttnIn<T>::vec8 b) {
  f32x16 d;
  if constexpr (__is_same(T, __bf16)) {
    if constexpr (B_AGPR) asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "a"(b));
    else asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "v"(b));
  } else {
    if constexpr (B_AGPR) asm("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "a"(b));
    else asm("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "v"(b));
  }
  return d;
}
template <int STATES>
__device__ __forceinline__ void mfma_settle(f32x16& c) {
  asm volatile("s_nop %1" : "+v"(c) : "n"(STATES - 1));
}
template <int STATES>
__device__ __forceinline__ void mfma_settle(f32x16 (&c)[1]) {
  mfma_settle<STATES>(c[0]);
}
template <int STATES>
__device__ __forceinline__ void mfma_settle(f32x16 (&c)[2]) {
  asm volatile("s_nop %2" : "+v"(c[0]), "+v"(c[1]) : "n"(STATES - 1));
}
// Nothing moves across: the steps of the loops below stand in the order they were written, each with the
// next step's LDS reads in flight and vector operations beside its MFMAs.
// The registers of an MFMA's c are free for other values once the next MFMA has been issued.
__device__ __forceinline__ void mfma_read(const f32x16& c) { asm volatile("" : : "v"(c)); }
__device__ __forceinline__ void step_end() { __builtin_amdgcn_sched_barrier(0); }
// Three workgroups of head dim 64 share a CU without the mask, by 168 registers (6 spilled in bf16, 9 in fp16): K
// in LDS, and LDS reads one step before their MFMAs instead of two.  fp16 8x12x777 79 us, 87 with two workgroups; 32x12x777 272, 293;
// bf16 4x16x2048 239, 249.  (The mask's branch takes registers: causal 4x32x4096 1279 us, 1003 with two.)
template <int D, bool CAUSAL>
constexpr bool kThree = D == 64 && !CAUSAL;
template <int D, bool CAUSAL>
constexpr int kSteps = kThree<D, CAUSAL> ? 1 : 2;   // that an LDS read is issued before its MFMAs

// A wave's 32 output rows (acc holds their transpose) go through its own 32 * D * 2 bytes of LDS,
// 16-byte chunks XORed by row, and out as whole rows of 16 bytes per lane.  Written from the
// accumulators they would be 8-byte pieces of 32 rows each (a workgroup's end at head dim 128 took
// 8 us longer so).
template <typename T, int D>
__device__ __forceinline__ void bwd_store_rows(unsigned char* stage, const f32x16 (&acc)[D / 32],
                                               float factor, T* __restrict__ out, int row0, int rows,
                                               int lane) {
  typedef AttnIn<T> In;
  constexpr int CPR = D / 8, SW = CPR < 16 ? CPR - 1 : 15, RPI = 64 / CPR;
  const int l32 = lane & 31, hi = lane >> 5;
#pragma unroll
  for (int a = 0; a < D / 32; ++a)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u32x2 w;
      w.x = In::pack2(acc[a][4 * g] * factor, acc[a][4 * g + 1] * factor);
      w.y = In::pack2(acc[a][4 * g + 2] * factor, acc[a][4 * g + 3] * factor);
      *(u32x2*)(stage + l32 * (D * 2) + (((4 * a + g) ^ (l32 & SW)) << 4) + 8 * hi) = w;
    }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 32 / RPI; ++i) {
    const int row = RPI * i + lane / CPR, c = lane % CPR;
    const u32x4 w = *(const u32x4*)(stage + row * (D * 2) + ((c ^ (row & SW)) << 4));
    if (row0 + row < rows) store16(out + (i64)(row0 + row) * D + 8 * c, w);
  }
  __builtin_amdgcn_wave_barrier();
}

// A tile buffer, an object of its own, the same for both stages where one kernel holds them.
template <int BYTES, int ID>
__device__ __forceinline__ unsigned char* bwd_tile() {
  __shared__ __attribute__((aligned(1024))) unsigned char tile[BYTES];
  return tile;
}

// dK and dV.  W waves of 32 KB keys each; a wave's V rows and its dK^T and dV^T stay in registers, its K
// rows too (in LDS where dK and dV take every AGPR, D KB = 256, and where three workgroups share a CU); the
// workgroup's Q and dO tiles are staged for all of its waves.  From head dim 128 on a SIMD has one wave: at
// KB = 2 every operand read from LDS feeds two MFMAs, which halves the LDS traffic of KB = 1 (at 32 keys a
// wave the four SIMDs' operand reads alone fill the LDS's 128 bytes a clock: full 2x16x4096x128 872 to 881
// us, 770 with two blocks).  Under the mask two blocks of head dim 128, and 256, spill 9 to 40 registers a lane.
// PARTS: each block's query tiles are taken in parts of `per` (64-row tiles, from the block's first);
// of a block with more than one, each part's fp32 sums go to `sums` [part][bh][key][dK, dV][D] for
// attention_bwd_join.
template <typename T, int D, bool CAUSAL, int W, int KB, bool PARTS>
__device__ __forceinline__ void attention_bwd_kv(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    const T* __restrict__ go, const float* __restrict__ start, const float* __restrict__ ndelta,
    const float* __restrict__ bounds, T* __restrict__ dk, T* __restrict__ dv,
    float* __restrict__ sums, int units, int heads, int sq, int sk, i64 qsb, i64 qsh, i64 qss,
    i64 ksb, i64 ksh, i64 kss, i64 vsb, i64 vsh, i64 vss, i64 gsb, i64 gsh, i64 gss, float scale,
    float scale_log2, int per, int group) {
  typedef AttnIn<T> In;
  typedef typename In::vec8 vec8;
  constexpr int BN = 32 * KB * W;                    // keys per workgroup
  constexpr int KSTEPS = D / 16, DBLK = D / 32;
  constexpr int ROWS = D <= 128 ? kBwdTile : 32;     // queries per staged tile
  constexpr int TILE = ROWS * D * 2;
  constexpr bool kOwn = D * KB >= 128;               // more than 256 registers
  // K takes no vector register where dK and dV take every AGPR, or three workgroups a CU
  constexpr bool kKeysInLds = D * KB >= 256 || kThree<D, CAUSAL>;
  constexpr int kAhead = kSteps<D, CAUSAL>;
  constexpr bool kScaled = BwdIn<T>::kScaled;
  unsigned char *const qbuf0 = bwd_tile<TILE, 0>(), *const qbuf1 = bwd_tile<TILE, 1>(),
                *const gbuf0 = bwd_tile<TILE, 2>(), *const gbuf1 = bwd_tile<TILE, 3>();
  __shared__ __attribute__((aligned(1024))) unsigned char kall[kKeysInLds ? BN * D * 2 : 16];
  __shared__ __attribute__((aligned(1024))) float sbuf0[2 * kBwdTile];
  __shared__ __attribute__((aligned(1024))) float sbuf1[2 * kBwdTile];

  const int nkb = (sk + BN - 1) / BN, nq = (sq + kBwdTile - 1) / kBwdTile;
  const int bh = group % units, id = group / units;
  const int kb_id = PARTS ? id % nkb : id, part = PARTS ? id / nkb : 0;   // whole parts first
  const int b = bh / heads, h = bh % heads;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hi = lane >> 5;
  const int k0 = kb_id * BN, kw = k0 + wave * 32 * KB;
  const bool idle = kw >= sk;                        // a wave without a key
  const T* qp = q + b * qsb + h * qsh;
  const T* kp = k + b * ksb + h * ksh;
  const T* vp = v + b * vsb + h * vsh;
  const T* gp = go + b * gsb + h * gsh;
  const float* st = start + (i64)bh * nq * kBwdTile;
  const float* nd = ndelta + (i64)bh * nq * kBwdTile;
  // causal: key j is seen by the queries from j on
  constexpr int PER = kBwdTile / ROWS;
  const int tiles = (sq + ROWS - 1) / ROWS, first = CAUSAL ? k0 / ROWS : 0;
  const int t0 = first + part * per * PER;
  const int t1 = PARTS ? min(tiles, t0 + per * PER) : tiles;
  if (PARTS && part > 0 && t0 >= tiles) return;      // the block has fewer parts
  const bool whole = !PARTS || tiles - first <= per * PER;

  vec8 kreg[kKeysInLds ? 1 : KB][kKeysInLds ? 1 : KSTEPS], vreg[KB][KSTEPS];
#pragma unroll
  for (int x = 0; x < KB; ++x) {
    const int j = kw + 32 * x + l32;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      vreg[x][s] = vec8{};
      if constexpr (!kKeysInLds) kreg[x][s] = vec8{};
      if (j < sk) {
        if constexpr (!kKeysInLds) kreg[x][s] = *(const vec8*)(kp + (i64)j * kss + 16 * s + 8 * hi);
        vreg[x][s] = *(const vec8*)(vp + (i64)j * vss + 16 * s + 8 * hi);
      }
    }
  }
  int lift = 0;
  if constexpr (kScaled) {
    const int nk = (sk + kBwdTile - 1) / kBwdTile;
    const int from = max(t0 / PER, CAUSAL ? kw / kBwdTile : 0), to = (t1 + PER - 1) / PER;
    const float* rows = bounds + 2 * ((i64)bh * nq + from);
    lift = bwd_exponent(2.0f * bwd_most(rows, 2, to - from, lane) *
                            bwd_most(bounds + 2 * (i64)units * nq + (i64)bh * nk, 1, nk, lane) +
                        bwd_most(rows + 1, 2, to - from, lane));
  }
  const float ds_mul = exp2_int(lift);

  const BwdTile<D, W, ROWS> qdma(wave, lane, qss), gdma(wave, lane, gss);
  const BwdRead<T, D> rd(lane);
  auto issue = [&](int tile, unsigned char* qd, unsigned char* gd, float* sd) {
    qdma.load(qp, qss, tile * ROWS, sq, wave, qd);
    gdma.load(gp, gss, tile * ROWS, sq, wave, gd);
    if (wave < 2) {
      const float* src = (wave == 0 ? st : nd) + (i64)tile * ROWS;
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          (void*)src, (short)0, ROWS * 4, (int)kRawBufferWord3);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (__attribute__((address_space(3))) void*)(sd + wave * kBwdTile), 4, lane * 4, 0, 0, 0);
    }
  };

  f32x16 dka[KB][DBLK], dva[KB][DBLK];
#pragma unroll
  for (int x = 0; x < KB; ++x)
#pragma unroll
    for (int a = 0; a < DBLK; ++a) dka[x][a] = dva[x][a] = f32x16{};
  bool bad = false;

  auto body = [&](int tile, const unsigned char* qt, const unsigned char* gt, const float* sv) {
#pragma unroll
    for (int sub = 0; sub < ROWS; sub += 32) {
      const int i0 = tile * ROWS + sub;
      if (CAUSAL && i0 + 31 < kw) continue;          // every pair hidden
      if (i0 >= sq) continue;
      auto starts = [&](const float* p) {            // per register: its query's value
        f32x16 c;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 w = *(const f32x4*)(p + sub + 8 * g + 4 * hi);
#pragma unroll
          for (int r = 0; r < 4; ++r) c[4 * g + r] = w[r];
        }
        return c;
      };
      auto kop = [&](int x, int t) {
        if constexpr (kKeysInLds) return rd.row(kall, wave * 32 * KB + 32 * x, t);
        else return kreg[x][t];
      };
      // every step's operands, read kAhead steps before
      vec8 rows[2 * KSTEPS + kAhead], keys[KB][KSTEPS + kAhead], columns[4 * DBLK + kAhead];
      auto read_step = [&](int n) {
        if (n < 2 * KSTEPS) rows[n] = n < KSTEPS ? rd.row(qt, sub, n) : rd.row(gt, sub, n - KSTEPS);
        if (n < KSTEPS) {
#pragma unroll
          for (int x = 0; x < KB; ++x) keys[x][n] = kop(x, n);
        }
        if (n >= 2 * KSTEPS) {
          const int m = n - 2 * KSTEPS, cs = m / DBLK % 2;
          if (m < 4 * DBLK) columns[m] = rd.column(m < 2 * DBLK ? gt : qt, sub, cs, m % DBLK);
        }
      };
      f32x16 s[KB], dp[KB], c = starts(sv);
#pragma unroll
      for (int n = 0; n < kAhead; ++n) read_step(n);
#pragma unroll
      for (int t = 0; t < KSTEPS; ++t) {
        read_step(t + kAhead);
#pragma unroll
        for (int x = 0; x < KB; ++x) {
          if constexpr (kOwn) {
            if (t == 0) s[x] = mfma_vgpr_from<T>(rows[t], keys[x][t], c);
            else mfma_vgpr<T, false>(rows[t], keys[x][t], s[x]);
          } else {
            s[x] = In::mfma(rows[t], keys[x][t], t == 0 ? c : s[x]);
          }
        }
        if (kOwn && t == 1) mfma_read(c);
        if (t == KSTEPS - 2) c = starts(sv + kBwdTile);
        if constexpr (kOwn) step_end();
      }
      // P of the first elements while the products of dP go on
      constexpr int LATE = KSTEPS > 4 ? 2 : 1, PER_STEP = (16 * KB + KSTEPS - LATE - 1) / (KSTEPS - LATE);
#pragma unroll
      for (int t = 0; t < KSTEPS; ++t) {
        read_step(KSTEPS + t + kAhead);
#pragma unroll
        for (int x = 0; x < KB; ++x) {
          if constexpr (kOwn) {
            if (t == 0) dp[x] = mfma_vgpr_from<T>(rows[KSTEPS + t], vreg[x][t], c);
            else mfma_vgpr<T, false>(rows[KSTEPS + t], vreg[x][t], dp[x]);
          } else {
            dp[x] = In::mfma(rows[KSTEPS + t], vreg[x][t], t == 0 ? c : dp[x]);
          }
        }
        if (kOwn && t == 1) mfma_read(c);
        if (kOwn && t == LATE) mfma_settle<12 - LATE>(s);
        if (t >= LATE) {
#pragma unroll
          for (int e = (t - LATE) * PER_STEP; e < (t - LATE + 1) * PER_STEP && e < 16 * KB; ++e)
            s[e / 16][e % 16] = __builtin_amdgcn_exp2f(s[e / 16][e % 16] * scale_log2);
        }
        if constexpr (kOwn) step_end();
      }
      if constexpr (kOwn) mfma_settle<12>(dp);
      // rows past the end are zero and P = 2^-inf, but not where K or V of the lane's key is
      // infinite or NaN: they are hidden too
      if ((CAUSAL && i0 < kw + 32 * KB - 1) || i0 + 32 > sq) {
        if (CAUSAL) bad |= rd.nonfinite(qt, sub) | rd.nonfinite(gt, sub);
        const int end = sq - i0 - 4 * hi;
#pragma unroll
        for (int x = 0; x < KB; ++x) {
          const int first_seen = CAUSAL ? kw + 32 * x + l32 - i0 - 4 * hi : 0;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int row = 8 * (r >> 2) + (r & 3);
            if (row < first_seen || row >= end) s[x][r] = dp[x][r] = 0.0f;
          }
        }
      }
      u32 pk[KB][8], dk2[KB][8];
      auto pack_p = [&](int x, int w) { pk[x][w] = In::pack2(s[x][2 * w], s[x][2 * w + 1]); };
      auto pack_ds = [&](int x, int w) {
        float u = s[x][2 * w], v = s[x][2 * w + 1];
        if constexpr (kScaled) {
          u *= ds_mul;
          v *= ds_mul;
        }
        dk2[x][w] = In::pack2(u * dp[x][2 * w], v * dp[x][2 * w + 1]);
      };
#pragma unroll
      for (int x = 0; x < KB; ++x)
#pragma unroll
        for (int w = 0; w < 4; ++w) pack_p(x, w);
      if constexpr (kOwn) step_end();
      // dV; beside it the rest of P, then dS
      constexpr int WORDS_STEP = (4 * KB + DBLK - 1) / DBLK, LATER = (8 * KB + DBLK - 1) / DBLK;
#pragma unroll
      for (int n = 0; n < 2 * DBLK; ++n) {
        read_step(2 * KSTEPS + n + kAhead);
#pragma unroll
        for (int x = 0; x < KB; ++x)
          dva[x][n % DBLK] = In::mfma(columns[n], packed_operand<T>(pk[x], n / DBLK), dva[x][n % DBLK]);
        // words in the order they are needed: P's 4..7 before the second half, then dS's 0..7
        if (n < DBLK) {
#pragma unroll
          for (int w = n * WORDS_STEP; w < (n + 1) * WORDS_STEP && w < 4 * KB; ++w) pack_p(w / 4, 4 + w % 4);
        } else {
#pragma unroll
          for (int w = (n - DBLK) * LATER; w < (n - DBLK + 1) * LATER && w < 8 * KB; ++w) pack_ds(w / 8, w % 8);
        }
        if constexpr (kOwn) step_end();
      }
#pragma unroll
      for (int n = 0; n < 2 * DBLK; ++n) {
        read_step(2 * KSTEPS + 2 * DBLK + n + kAhead);
#pragma unroll
        for (int x = 0; x < KB; ++x)
          dka[x][n % DBLK] = In::mfma(columns[2 * DBLK + n], packed_operand<T>(dk2[x], n / DBLK), dka[x][n % DBLK]);
        if constexpr (kOwn) step_end();
      }
    }
  };

  // Tile t is used from buffers t % 2 while the loads of tile t+1 fill the others (last read in
  // iteration t-1, before this iteration's barrier).
  auto landed = []() { __builtin_amdgcn_s_waitcnt(0x0F70); };   // vmcnt(0)
  if (t0 < t1) {
    if constexpr (kKeysInLds) {
      const BwdTile<D, W, ROWS> kdma(wave, lane, kss);
#pragma unroll
      for (int r = 0; r < BN; r += ROWS)
        if (k0 + r < sk) kdma.load(kp, kss, k0 + r, sk, wave, kall + r * D * 2);
    }
    issue(t0, qbuf0, gbuf0, sbuf0);
    for (int tile = t0; tile < t1; tile += 2) {
      landed();
      __syncthreads();
      if (tile + 1 < t1) issue(tile + 1, qbuf1, gbuf1, sbuf1);
      if (!idle) body(tile, qbuf0, gbuf0, sbuf0);
      landed();
      __syncthreads();
      if (tile + 2 < t1) issue(tile + 2, qbuf0, gbuf0, sbuf0);
      if (!idle && tile + 1 < t1) body(tile + 1, qbuf1, gbuf1, sbuf1);
    }
  }

  const i64 row0 = (i64)bh * sk;
  float* const part_rows = PARTS ? sums + ((i64)part * units + bh) * sk * 2 * D : nullptr;
  auto store = [&](int which, int j, int d, float a0, float a1, float a2, float a3) {
    if (!whole) {
      *(f32x4*)(part_rows + ((i64)j * 2 + which) * D + d) = f32x4{a0, a1, a2, a3};
    } else {
      u32x2 w;
      w.x = In::pack2(a0, a1);
      w.y = In::pack2(a2, a3);
      *(u32x2*)((which ? dv : dk) + (row0 + j) * D + d) = w;
    }
  };
  if constexpr (CAUSAL) {
    if (__syncthreads_or(bad)) {
      attention_bwd_exact_kv<T, D, CAUSAL, W>(qp, kp, vp, gp, st, nd, k0, BN, sk, t0 * ROWS,
                                              min(sq, t1 * ROWS), qss, kss, vss, gss, scale,
                                              scale_log2, store);
      return;
    }
  }
  const float pf = exp2_int(-(int)BwdIn<T>::kLift), sf = scale * pf * exp2_int(-lift);
  if (whole) {
    if constexpr (!CAUSAL) __syncthreads();          // every wave is done with the tiles
    static_assert(W <= 4, "one tile buffer for each wave");
    unsigned char* stage = wave == 0 ? qbuf0 : wave == 1 ? qbuf1 : wave == 2 ? gbuf0 : gbuf1;
#pragma unroll
    for (int x = 0; x < KB; ++x) {
      bwd_store_rows<T, D>(stage, dka[x], sf, dk + row0 * D, kw + 32 * x, sk, lane);
      bwd_store_rows<T, D>(stage, dva[x], pf, dv + row0 * D, kw + 32 * x, sk, lane);
    }
  } else {
#pragma unroll
    for (int x = 0; x < KB; ++x) {
      const int j = kw + 32 * x + l32;
      if (j >= sk) continue;
#pragma unroll
      for (int a = 0; a < DBLK; ++a)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = 32 * a + 8 * g + 4 * hi;
          store(0, j, d, dka[x][a][4 * g] * sf, dka[x][a][4 * g + 1] * sf,
                dka[x][a][4 * g + 2] * sf, dka[x][a][4 * g + 3] * sf);
          store(1, j, d, dva[x][a][4 * g] * pf, dva[x][a][4 * g + 1] * pf,
                dva[x][a][4 * g + 2] * pf, dva[x][a][4 * g + 3] * pf);
        }
    }
  }
}

// dQ.  W waves of 32 QB queries each; a wave's Q and dO rows and its dQ^T stay in registers, the
// workgroup's K and V tiles are staged for all of its waves.  PARTS: as above, over the key tiles, with
// `sums` [part][bh][query][D].
template <typename T, int D, bool CAUSAL, int W, int QB, bool PARTS>
__device__ __forceinline__ void attention_bwd_q(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    const T* __restrict__ go, const float* __restrict__ start, const float* __restrict__ ndelta,
    const float* __restrict__ bounds, T* __restrict__ dq, float* __restrict__ sums, int units,
    int heads, int sq, int sk, i64 qsb, i64 qsh, i64 qss, i64 ksb, i64 ksh, i64 kss, i64 vsb,
    i64 vsh, i64 vss, i64 gsb, i64 gsh, i64 gss, float scale, float scale_log2, int per, int group) {
  typedef AttnIn<T> In;
  typedef typename In::vec8 vec8;
  constexpr int BM = 32 * QB * W;
  constexpr int KSTEPS = D / 16, DBLK = D / 32;
  constexpr int ROWS = D <= 128 ? kBwdTile : 32;     // keys per staged tile, as attention_bwd_kv's
  constexpr int TILE = ROWS * D * 2;
  constexpr bool kScaled = BwdIn<T>::kScaled;
  constexpr int kAhead = kSteps<D, CAUSAL>;
  constexpr bool kOwn = D * QB >= 128;              // more than 256 registers
  unsigned char *const kbuf0 = bwd_tile<TILE, 0>(), *const kbuf1 = bwd_tile<TILE, 1>(),
                *const vbuf0 = bwd_tile<TILE, 2>(), *const vbuf1 = bwd_tile<TILE, 3>();

  const int nqb = (sq + BM - 1) / BM, nq = (sq + kBwdTile - 1) / kBwdTile;
  const int nk = (sk + kBwdTile - 1) / kBwdTile;
  const int bh = group % units, id = group / units;
  // heaviest first: under the causal mask those of the most keys, otherwise the whole ones
  const int at = PARTS ? id % nqb : id, qb = CAUSAL ? nqb - 1 - at : at, part = PARTS ? id / nqb : 0;
  const int b = bh / heads, h = bh % heads;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hi = lane >> 5;
  const int q0 = qb * BM, qw = q0 + wave * 32 * QB;
  const bool idle = qw >= sq;                        // a wave without a query
  const T* qp = q + b * qsb + h * qsh;
  const T* kp = k + b * ksb + h * ksh;
  const T* vp = v + b * vsb + h * vsh;
  const T* gp = go + b * gsb + h * gsh;
  const float* st = start + (i64)bh * nq * kBwdTile;
  const float* nd = ndelta + (i64)bh * nq * kBwdTile;
  constexpr int PER = kBwdTile / ROWS;
  const int tiles = (sk + ROWS - 1) / ROWS, last = CAUSAL ? min(tiles, (q0 + BM + ROWS - 1) / ROWS) : tiles;
  const int t0 = PARTS ? part * per * PER : 0;
  const int t1 = PARTS ? min(last, t0 + per * PER) : last;
  if (PARTS && part > 0 && t0 >= last) return;       // the block has fewer parts
  const bool whole = !PARTS || last <= per * PER;

  vec8 qreg[QB][KSTEPS], greg[QB][KSTEPS];
  float shift[QB], minus[QB];
#pragma unroll
  for (int x = 0; x < QB; ++x) {
    const int i = qw + 32 * x + l32;
    shift[x] = i < sq ? st[i] * scale_log2 : -kInf;
    minus[x] = i < sq ? nd[i] : 0.0f;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      qreg[x][s] = greg[x][s] = vec8{};
      if (i < sq) {
        qreg[x][s] = *(const vec8*)(qp + (i64)i * qss + 16 * s + 8 * hi);
        greg[x][s] = *(const vec8*)(gp + (i64)i * gss + 16 * s + 8 * hi);
      }
    }
  }
  int lift[QB];                                      // a query's power of two on dS
  float most = 0.0f;                                 // |v|
  if constexpr (kScaled) most = bwd_most(bounds + 2 * (i64)units * nq + (i64)bh * nk, 1, nk, lane);
#pragma unroll
  for (int x = 0; x < QB; ++x) {
    lift[x] = 0;
    if constexpr (kScaled) {
      float g2 = 0.0f;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = (float)greg[x][s][j];
          g2 = __builtin_fmaf(w, w, g2);
        }
      u32 lower, upper;
      pair_u32<32>(as_u32(g2), lower, upper);
      lift[x] = bwd_exponent(__builtin_sqrtf(as_f32(lower) + as_f32(upper)) * 1.001f * most +
                             __builtin_fabsf(minus[x]));
      shift[x] += (float)lift[x];                    // on P
    }
  }
  if constexpr (kOwn) {
#pragma unroll
    for (int x = 0; x < QB; ++x)
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) asm("" : "+a"(greg[x][s]));
  }
  const BwdTile<D, W, ROWS> kdma(wave, lane, kss), vdma(wave, lane, vss);
  const BwdRead<T, D> rd(lane);
  auto issue = [&](int tile, unsigned char* kd, unsigned char* vd) {
    kdma.load(kp, kss, tile * ROWS, sk, wave, kd);
    vdma.load(vp, vss, tile * ROWS, sk, wave, vd);
  };

  f32x16 dqa[QB][DBLK];
#pragma unroll
  for (int x = 0; x < QB; ++x)
#pragma unroll
    for (int a = 0; a < DBLK; ++a) dqa[x][a] = f32x16{};
  bool bad = false;

  auto body = [&](int tile, const unsigned char* kt, const unsigned char* vt) {
#pragma unroll
    for (int sub = 0; sub < ROWS; sub += 32) {
      const int j0 = tile * ROWS + sub;
      if (CAUSAL && j0 > qw + 32 * QB - 1) continue;   // every pair hidden
      if (j0 >= sk) continue;
      // the operands of every step, read kAhead steps before
      constexpr int ROWS_STEPS = 2 * QB * KSTEPS;
      vec8 rows[2 * KSTEPS], columns[2 * DBLK];
      auto read_step = [&](int n) {
        if (n < ROWS_STEPS) {
          const int x = n / KSTEPS % QB, t = n % KSTEPS;
          if (x == 0) {
            if (n < KSTEPS) rows[t] = rd.row(kt, sub, t);
            else rows[KSTEPS + t] = rd.row(vt, sub, t);
          }
        } else if (n < ROWS_STEPS + 2 * DBLK) {
          const int m = n - ROWS_STEPS;
          columns[m] = rd.column(kt, sub, m / DBLK, m % DBLK);
        }
      };
      f32x16 s[QB], dp[QB];
      auto exponentials = [&](int x, int from, int to) {
#pragma unroll
        for (int r = from; r < to && r < 16; ++r)
          s[x][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][r], scale_log2, shift[x]));
      };
      // S of one block of queries after the other, and then dP; P of a block beside the products behind its S
      constexpr int LATE = KSTEPS > 4 ? 2 : 1, PER_STEP = (16 + KSTEPS - LATE - 1) / (KSTEPS - LATE);
#pragma unroll
      for (int n = 0; n < kAhead; ++n) read_step(n);
#pragma unroll
      for (int n = 0; n < 2 * QB * KSTEPS; ++n) {
        const int x = n / KSTEPS % QB, t = n % KSTEPS, chain = n / KSTEPS;
        read_step(n + kAhead);
        if (chain < QB) {
          if constexpr (kOwn) {
            if (t == 0) s[x] = mfma_vgpr_zero<T, false>(rows[t], qreg[x][t]);
            else mfma_vgpr<T, false>(rows[t], qreg[x][t], s[x]);
          } else {
            s[x] = In::mfma(rows[t], qreg[x][t], t == 0 ? f32x16{} : s[x]);
          }
        } else {
          if constexpr (kOwn) {
            if (t == 0) dp[x] = mfma_vgpr_zero<T, true>(rows[KSTEPS + t], greg[x][t]);
            else mfma_vgpr<T, true>(rows[KSTEPS + t], greg[x][t], dp[x]);
          } else {
            dp[x] = In::mfma(rows[KSTEPS + t], greg[x][t], t == 0 ? f32x16{} : dp[x]);
          }
        }
        if (chain >= 1 && chain <= QB && t >= LATE) {
          if (kOwn && t == LATE) mfma_settle<12 - LATE>(s[chain - 1]);
          exponentials(chain - 1, (t - LATE) * PER_STEP, (t - LATE + 1) * PER_STEP);
        }
        if constexpr (kOwn) step_end();
      }
      if constexpr (kOwn) mfma_settle<12>(dp[QB - 1]);
      const bool masked = (CAUSAL && j0 + 31 > qw) || j0 + 32 > sk;
      if (masked) {
        if (CAUSAL) bad |= rd.nonfinite(kt, sub);
#pragma unroll
        for (int x = 0; x < QB; ++x) {
          const int i = qw + 32 * x + l32;
          const int end = (CAUSAL ? min(sk, i + 1) : sk) - j0 - 4 * hi;   // register rows from it on
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) >= end) {
              s[x][r] = 0.0f;
              dp[x][r] = -minus[x];
            }
        }
      }
      u32 pk[QB][8];
      auto pack_ds = [&](int x, int w) {
        pk[x][w] = In::pack2(s[x][2 * w] * (dp[x][2 * w] + minus[x]),
                             s[x][2 * w + 1] * (dp[x][2 * w + 1] + minus[x]));
      };
#pragma unroll
      for (int x = 0; x < QB; ++x)
#pragma unroll
        for (int w = 0; w < 4; ++w) pack_ds(x, w);
      if constexpr (kOwn) step_end();
      constexpr int WORDS_STEP = (4 * QB + DBLK - 1) / DBLK;
#pragma unroll
      for (int n = 0; n < 2 * DBLK; ++n) {
        read_step(ROWS_STEPS + n + kAhead);
#pragma unroll
        for (int x = 0; x < QB; ++x)
          dqa[x][n % DBLK] = In::mfma(columns[n], packed_operand<T>(pk[x], n / DBLK), dqa[x][n % DBLK]);
        if (n < DBLK) {
#pragma unroll
          for (int w = n * WORDS_STEP; w < (n + 1) * WORDS_STEP && w < 4 * QB; ++w) pack_ds(w / 4, 4 + w % 4);
        }
        if constexpr (kOwn) step_end();
      }
    }
  };

  auto landed = []() { __builtin_amdgcn_s_waitcnt(0x0F70); };   // vmcnt(0)
  if (t0 < t1) {
    issue(t0, kbuf0, vbuf0);
    for (int tile = t0; tile < t1; tile += 2) {
      landed();
      __syncthreads();
      if (tile + 1 < t1) issue(tile + 1, kbuf1, vbuf1);
      if (!idle) body(tile, kbuf0, vbuf0);
      landed();
      __syncthreads();
      if (tile + 2 < t1) issue(tile + 2, kbuf0, vbuf0);
      if (!idle && tile + 1 < t1) body(tile + 1, kbuf1, vbuf1);
    }
  }

  const i64 row0 = (i64)bh * sq;
  float* const part_rows = PARTS ? sums + ((i64)part * units + bh) * sq * D : nullptr;
  auto store = [&](int i, int d, float a0, float a1, float a2, float a3) {
    if (!whole) {
      *(f32x4*)(part_rows + (i64)i * D + d) = f32x4{a0, a1, a2, a3};
    } else {
      u32x2 w;
      w.x = In::pack2(a0, a1);
      w.y = In::pack2(a2, a3);
      *(u32x2*)(dq + (row0 + i) * D + d) = w;
    }
  };
  if constexpr (CAUSAL) {
    if (__syncthreads_or(bad)) {
      attention_bwd_exact_q<T, D, CAUSAL, W>(qp, kp, vp, gp, st, nd, q0, BM, sq, t0 * ROWS,
                                             min(sk, t1 * ROWS), qss, kss, vss, gss, scale,
                                             scale_log2, store);
      return;
    }
  }
  float sf[QB];
#pragma unroll
  for (int x = 0; x < QB; ++x) sf[x] = scale * exp2_int(-(int)BwdIn<T>::kLift) * exp2_int(-lift[x]);
  if (whole) {
    if constexpr (!CAUSAL) __syncthreads();          // every wave is done with the tiles
    static_assert(W <= 4, "one tile buffer for each wave");
    unsigned char* stage = wave == 0 ? kbuf0 : wave == 1 ? kbuf1 : wave == 2 ? vbuf0 : vbuf1;
#pragma unroll
    for (int x = 0; x < QB; ++x)
      bwd_store_rows<T, D>(stage, dqa[x], sf[x], dq + row0 * D, qw + 32 * x, sq, lane);
  } else {
#pragma unroll
    for (int x = 0; x < QB; ++x) {
      const int i = qw + 32 * x + l32;
      if (i >= sq) continue;
#pragma unroll
      for (int a = 0; a < DBLK; ++a)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          store(i, 32 * a + 8 * g + 4 * hi, dqa[x][a][4 * g] * sf[x], dqa[x][a][4 * g + 1] * sf[x],
                dqa[x][a][4 * g + 2] * sf[x], dqa[x][a][4 * g + 3] * sf[x]);
    }
  }
}

// The parts' fp32 sums of the rows whose block of `block` rows had more than one part of `per` tiles,
// added in the order of the parts and rounded once.  KV: `len` keys a head and (dK, dV) of a key side by
// side; a block's tiles are those of the `other` queries, from its own keys' on under the causal mask.
// Otherwise `len` queries; the tiles are the keys', up to its own queries'.
template <typename T, int D, bool KV>
__device__ __forceinline__ void attention_bwd_join(const float* __restrict__ sums, T* __restrict__ a,
                                                   T* __restrict__ b, i64 rows, int len, int other,
                                                   int block, int per, int causal) {
  typedef AttnIn<T> In;
  constexpr int N = KV ? 2 * D : D;
  const i64 at = ((i64)blockIdx.x * 256 + threadIdx.x) * 4;
  const i64 all = rows * N;
  if (at >= all) return;
  const i64 row = at / N;
  const int c = (int)(at % N), r0 = (int)(row % len) / block * block;
  int tiles = (other + kBwdTile - 1) / kBwdTile;
  if (causal) tiles = KV ? tiles - r0 / kBwdTile : min(tiles, (r0 + block + kBwdTile - 1) / kBwdTile);
  const int parts = (tiles + per - 1) / per;
  if (parts <= 1) return;                            // written by its workgroup
  f32x4 t = *(const f32x4*)(sums + at);
  for (int p = 1; p < parts; ++p) t += *(const f32x4*)(sums + p * all + at);
  u32x2 w;
  w.x = In::pack2(t[0], t[1]);
  w.y = In::pack2(t[2], t[3]);
  T* out = KV && c >= D ? b + row * D + (c - D) : a + row * D + c;
  *(u32x2*)out = w;
}

}  // namespace nep
