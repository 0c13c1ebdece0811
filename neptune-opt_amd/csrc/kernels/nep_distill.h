// nep_distill.h -- distillation from a teacher's top logits, and its gradient (gfx950).
//
// Per row, student logits z[0..n), temperature T, and a teacher's list of entries (t_k, i_k):
//   p = softmax(t / T) over the list's present entries (i_k >= 0)      q = softmax(z / T)
//   loss = T^2 sum_k p_k (log p_k - log q_{i_k})
//   dloss/dz_i = T (q_i - sum of p_k with i_k = i), times the row's upstream gradient
// The row's state (max m, sum s of exp((z - m) / T)) is kept for the gradient instead of its
// logsumexp: (z - m) is exact to an ulp of itself where z - lse would lose lse's ulp.
//
// A list without a present entry, or with all of them -inf, has loss 0 and gradient 0 whatever the
// row holds.  An entry with p = 0 adds nothing; one with p > 0 at a student logit of -inf makes the
// loss +inf (its gradient is finite).  An index of n or more makes the row's loss and gradient NaN,
// and is never read through.
//
// HBM-bound: the loss reads the row once (running max and sum per lane, rescaled when the max
// moves), the gradient reads it once and writes it once.  bf16 16384 x 32000 with 64 entries: loss 151 us
// (7.0 TB/s), gradient 355 (5.9); 7168 x 32003 gradient 158 (5.8); 16384 x 4096 27 and 58 (5.5, 4.8: the
// list's chain of index, column and sums is as long as the row); fp32 4096 x 32000 78 and 173.
#pragma once

namespace nep {

// TPR lanes hold a row: a wavefront (WG holds several rows, no barrier) or the whole workgroup.
template <int TPR>
struct RowLanes {
  static constexpr int kWaves = TPR > 64 ? TPR / 64 : 1;
  static_assert(TPR >= 64 && TPR <= 1024, "a row has a wavefront at least");
  __device__ static __forceinline__ void sync() {
    if constexpr (TPR > 64) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
  }
  // N reductions in one exchange; `lds` has N floats a wave, and the next call may use the same
  template <bool MAX, int N>
  __device__ static __forceinline__ void reduce(float (&v)[N], float* lds) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = MAX ? group_max<64>(v[i]) : group_sum<64>(v[i]);
    if constexpr (TPR > 64) {
      __syncthreads();
      if (lane_id() == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) lds[(threadIdx.x >> 6) * N + i] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float w = lds[(lane_id() % kWaves) * N + i];
        v[i] = MAX ? group_max<kWaves>(w) : group_sum<kWaves>(w);
      }
    }
  }
  __device__ static __forceinline__ bool any(bool b) {
    if constexpr (TPR > 64) return __syncthreads_or(b ? 1 : 0) != 0;
    else return __builtin_amdgcn_ballot_w64(b) != 0;
  }
};

// The whole words of a row (those of its Span), read through a buffer, zero past the end.  No access is in a
// branch, so a wait for one tile leaves the next one in flight (in branches the waits are for everything,
// and a tile is not started until the one before it is done).
// LINES: word 0 is the start of the cache line that the row's first word is in, and the lanes before `skip`
// take the first word too (and write the same value): a wavefront's words are whole lines.  For the gradient
// of wide rows, which writes them: 7168 rows of 32003 159 us, 167 from the first word on; the loss, and
// rows that a wavefront holds, lose by the longer row (16384 rows of 1000 13.6 us, 14.7).
constexpr u32 kPastRow = 0x80000000u;
template <class St, class Sp, bool LINES>
struct RowWords {
  __amdgpu_buffer_rsrc_t row;
  int skip, words;
  i64 line;                                          // column of word 0

  __device__ __forceinline__ RowWords(const typename St::T* rp, const Sp& sp) {
    skip = LINES ? (int)(((u64)(rp + sp.v0) >> 4) & 7) : 0;
    line = sp.v0 - skip * St::kVec;
    words = sp.v1 > sp.v0 ? skip + (int)((sp.v1 - sp.v0) / St::kVec) : 0;
    row = __builtin_amdgcn_make_buffer_rsrc((void*)(rp + line), (short)0, 0x7fffffff, 0x00020000);
  }
  // words first + u TPR + t of a tile
  template <int TPR, int UNROLL>
  __device__ __forceinline__ void load(int first, int t, u32x4* w) const {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = first + u * TPR + t;
      w[u] = __builtin_amdgcn_raw_buffer_load_b128(row, i < words ? (u32)at(i) * 16u : kPastRow, 0, 2);
    }
  }
  __device__ __forceinline__ int at(int i) const { return LINES && i < skip ? skip : i; }
};

// Element `i` of a buffer (kPastRow: zero), of 2, 4 or 8 bytes.
template <typename T>
__device__ __forceinline__ T load_element(__amdgpu_buffer_rsrc_t r, u32 i) {
  const u32 off = i == kPastRow ? kPastRow : i * (u32)sizeof(T);
  if constexpr (sizeof(T) == 8) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
  else if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
  else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t elements_at(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, 0x7fffffff, 0x00020000);
}

// A row's entries, EPL per lane: entry k of lane t is t + k TPR.  They are asked for before the row's first
// words and looked at behind them, so that the columns they name are asked for while those are in flight.
template <class St, class Lt, typename Ix, int TPR, int EPL>
struct TeacherList {
  float e[EPL];      // t_k, then exp((t_k - max) / T) / sum = p_k
  float d[EPL];      // (t_k - max)
  float z[EPL];      // the student's logit there
  int at[EPL];       // column, -1 where absent
  float top, total;  // max and sum of the exponentials
  bool empty, bad;
  typename Lt::T raw[EPL];
  Ix index[EPL];

  __device__ __forceinline__ void ask(const typename Lt::T* t, const Ix* ix, int count, int lane, bool live) {
    const __amdgpu_buffer_rsrc_t tops = elements_at(t), indices = elements_at(ix);
#pragma unroll
    for (int k = 0; k < EPL; ++k) {
      const u32 i = live && lane + k * TPR < count ? (u32)(lane + k * TPR) : kPastRow;
      index[k] = load_element<Ix>(indices, i);
      raw[k] = load_element<typename Lt::T>(tops, i);
    }
  }
  __device__ __forceinline__ void look(const typename St::T* row, int count, i64 n, int lane, bool live) {
    const __amdgpu_buffer_rsrc_t logits = elements_at(row);
    bad = false;
#pragma unroll
    for (int k = 0; k < EPL; ++k) {
      const bool here = live && lane + k * TPR < count && index[k] >= 0;
      bad |= here && (i64)index[k] >= n;
      at[k] = here && (i64)index[k] < n ? (int)index[k] : -1;
      e[k] = at[k] < 0 ? -kInf : Lt::load(&raw[k]);
      const typename St::T v = load_element<typename St::T>(logits, at[k] < 0 ? kPastRow : (u32)at[k]);
      z[k] = St::load(&v);
    }
  }
  // this lane's largest t (a NaN is no maximum, but it counts as present)
  __device__ __forceinline__ float largest() const {
    float m = -kInf;
#pragma unroll
    for (int k = 0; k < EPL; ++k) m = __builtin_fmaxf(m, is_nan(e[k]) ? -3.0e38f : e[k]);
    return m;
  }
  // with the list's largest: the exponentials, this lane's sum of them
  __device__ __forceinline__ float exponentials(float list_top, float c) {
    top = list_top;
    const float ref = top == -kInf ? 0.0f : top;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < EPL; ++k) {
      d[k] = e[k] - ref;
      e[k] = at[k] < 0 ? 0.0f : __builtin_amdgcn_exp2f(d[k] * c);
      s += e[k];
    }
    return s;
  }
  __device__ __forceinline__ void normalise(float list_total, bool any_bad) {
    total = list_total;
    bad = any_bad;
    empty = top == -kInf && !bad;
    const float inv = __builtin_amdgcn_rcpf(total);   // total is at least 1
#pragma unroll
    for (int k = 0; k < EPL; ++k) e[k] *= inv;
  }
};

// Loss and state of each row.  c = log2(e) / T, inv_t = 1 / T, t2 = T^2.
template <class St, class Lt, typename Ix, int TPR, int UNROLL, int ACCESS, int EPL, int WG>
__device__ __forceinline__ void distill_forward(const typename St::T* __restrict__ z,
                                                const typename Lt::T* __restrict__ top_logits,
                                                const Ix* __restrict__ index,
                                                float* __restrict__ loss,
                                                float* __restrict__ stats, i64 rows, i64 n,
                                                i64 stride_z, i64 stride_t, i64 stride_i,
                                                int count, float c, float inv_t, float t2) {
  typedef RowLanes<TPR> R;
  typedef Span<St, TPR, ACCESS> Sp;
  constexpr int VEC = St::kVec;
  __shared__ float lds[2 * R::kWaves];
  const int t = threadIdx.x % TPR;
  const i64 row = (i64)blockIdx.x * (WG / TPR) + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  const bool live = row < rows;
  const typename St::T* rp = z + (live ? row : 0) * stride_z;
  TeacherList<St, Lt, Ix, TPR, EPL> list;
  list.ask(top_logits + (live ? row : 0) * stride_t, index + (live ? row : 0) * stride_i, count, t, live);
  const Sp sp(rp, 0, live ? n : 0);
  const RowWords<St, Sp, false> row_words(rp, sp);
  const int words = row_words.words;
  u32x4 cur[UNROLL];
  row_words.template load<TPR, UNROLL>(0, t, cur);
  list.look(rp, count, n, t, live);
  float m = -kInf, s = 0.0f;
  auto move = [&](float tile_max) {
    if (tile_max > m) {
      s *= m == -kInf ? 0.0f : __builtin_amdgcn_exp2f((m - tile_max) * c);
      m = tile_max;
    }
    return m == -kInf ? 0.0f : m;
  };
  auto tile = [&]() {
    float tm = -kInf;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float v[VEC];
      St::unpack(cur[u], v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) tm = __builtin_fmaxf(tm, v[j]);
    }
    const float ref = move(tm);
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float v[VEC];
      St::unpack(cur[u], v);
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        a += __builtin_amdgcn_exp2f((v[j] - ref) * c);
        b += __builtin_amdgcn_exp2f((v[j + 1] - ref) * c);
      }
    }
    s += a + b;
  };
  typename Sp::Rest rest;
  if constexpr (ACCESS == kRagged) sp.load_rest(rest, rp, t);
  int at = 0;
  for (; at + UNROLL * TPR <= words; at += UNROLL * TPR) {
    u32x4 next[UNROLL];
    row_words.template load<TPR, UNROLL>(at + UNROLL * TPR, t, next);
    tile();
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) cur[u] = next[u];
  }
  if (at < words) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (at + u * TPR + t >= words)
        cur[u] = u32x4{St::kNegInfWord, St::kNegInfWord, St::kNegInfWord, St::kNegInfWord};
    tile();
  }
  if constexpr (ACCESS == kRagged) {
    float tm = -kInf;
#pragma unroll
    for (int u = 0; u < Sp::RU; ++u) tm = __builtin_fmaxf(tm, rest.s[u]);
    const float ref = move(tm);
#pragma unroll
    for (int u = 0; u < Sp::RU; ++u) s += __builtin_amdgcn_exp2f((rest.s[u] - ref) * c);
  }
  float tops[2] = {m, list.largest()};
  R::template reduce<true, 2>(tops, lds);
  const float top = tops[0];
  float totals[2] = {m == -kInf ? s : s * __builtin_amdgcn_exp2f((m - top) * c), list.exponentials(tops[1], c)};
  R::template reduce<false, 2>(totals, lds);
  const float total = totals[0];
  list.normalise(totals[1], R::any(list.bad));
  // log p_k - log q_k = ((t_k - max t) - (z_k - max z)) / T - log(total t) + log(total z), with the
  // hardware's logarithm (an ulp; both arguments are at least 1)
  const float gap = (__builtin_amdgcn_logf(total) - __builtin_amdgcn_logf(list.total)) * 0.6931471805599453f;
  float term = 0.0f;
#pragma unroll
  for (int k = 0; k < EPL; ++k)
    if (list.at[k] >= 0 && !(list.e[k] == 0.0f))
      term += list.e[k] * ((list.d[k] - (list.z[k] - top)) * inv_t + gap);
  float terms[1] = {term};
  R::template reduce<false, 1>(terms, lds);
  if (live && t == 0) {
    loss[row] = list.bad ? __builtin_nanf("") : list.empty ? 0.0f : t2 * terms[0];
    if (stats != nullptr) {
      stats[2 * row] = top;
      stats[2 * row + 1] = total;
    }
  }
}

// Gradient of each row, its columns in gridDim.y parts of `per` (a multiple of a word's; the state is given,
// so a part needs nothing of the others).  The part is written as T g q first; the list's columns are then written
// again, whole, by the lanes that hold their entries, after a barrier behind which the first writes
// are complete.  An index that comes twice is found by a hash of LDS bits (never missed; a false
// alarm costs the search): each of its entries then sums p over the list in the list's order, so
// all of them write the same value.
template <class St, class Lt, typename Ix, int TPR, int UNROLL, int ACCESS, int EPL, int WG>
__device__ __forceinline__ void distill_backward(const float* __restrict__ grad,
                                                 const typename St::T* __restrict__ z,
                                                 const typename Lt::T* __restrict__ top_logits,
                                                 const Ix* __restrict__ index,
                                                 const float* __restrict__ stats,
                                                 typename St::T* __restrict__ dz, i64 rows, i64 n,
                                                 i64 stride_g, i64 stride_z, i64 stride_t,
                                                 i64 stride_i, int count, float c, float temperature,
                                                 i64 per) {
  typedef RowLanes<TPR> R;
  typedef Span<St, TPR, ACCESS> Sp;
  constexpr int VEC = St::kVec, STEP = TPR * VEC, RPW = WG / TPR;
  constexpr int HASH = 1 << 15;                    // bits of a row's table
  __shared__ float lds[R::kWaves];
  __shared__ u32 seen[RPW][HASH / 32];
  __shared__ float list_p[RPW][TPR * EPL];
  __shared__ int list_at[RPW][TPR * EPL];
  const int t = threadIdx.x % TPR, slot = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  const i64 row = (i64)blockIdx.x * RPW + slot;
  const bool live = row < rows;
  const typename St::T* rp = z + (live ? row : 0) * stride_z;
  typename St::T* op = dz + (live ? row : 0) * n;
  const i64 c0 = blockIdx.y * per, c1 = c0 + per < n ? c0 + per : n;
  const Sp sp(rp, c0, live ? c1 : c0);
  const RowWords<St, Sp, (TPR > 64)> row_words(rp, sp);
  const int words = row_words.words;
  TeacherList<St, Lt, Ix, TPR, EPL> list;
  list.ask(top_logits + (live ? row : 0) * stride_t, index + (live ? row : 0) * stride_i, count, t, live);
  u32x4 cur[UNROLL];
  row_words.template load<TPR, UNROLL>(0, t, cur);
  list.look(rp, count, n, t, live);
  const float g = live ? grad[row * stride_g] * temperature : 0.0f;
  const float top = live ? stats[2 * row] : 0.0f, total = live ? stats[2 * row + 1] : 1.0f;
#pragma unroll
  for (int i = t; i < HASH / 32; i += TPR) seen[slot][i] = 0u;
  float reduced[1] = {list.largest()};
  R::template reduce<true, 1>(reduced, lds);
  reduced[0] = list.exponentials(reduced[0], c);
  R::template reduce<false, 1>(reduced, lds);
  list.normalise(reduced[0], R::any(list.bad));
  R::sync();                                       // the table is clear
  bool twice = false;
#pragma unroll
  for (int k = 0; k < EPL; ++k) {
    list_p[slot][t + k * TPR] = list.e[k];
    list_at[slot][t + k * TPR] = list.at[k];
    if (list.at[k] >= 0) {
      const u32 h = (u32)list.at[k] & (HASH - 1);
      twice |= (atomicOr(&seen[slot][h >> 5], 1u << (h & 31)) >> (h & 31)) & 1u;
    }
  }
  // NaN where the list's probabilities are (their sum is 1 otherwise), and for an index past the row
  const float scale = list.bad || is_nan(list.total) ? __builtin_nanf("") : g / total;
  const float ref = top == -kInf ? 0.0f : top;
  auto value = [&](float v) { return scale * __builtin_amdgcn_exp2f((v - ref) * c); };
  if (list.empty) {
    for (i64 e = sp.v0 + (i64)t * VEC; e < sp.v1; e += STEP) store_vec<ACCESS>(op + e, u32x4{0u, 0u, 0u, 0u});
    if constexpr (ACCESS == kRagged)
      for (int i = t; i < sp.rest; i += TPR) St::store(op + sp.column(i), 0.0f);
  } else {
    typename Sp::Rest rest;
    if constexpr (ACCESS == kRagged) sp.load_rest(rest, rp, t);
    typename St::T* ow = op + row_words.line;
    auto put = [&](int u, int at) {
      float v[VEC];
      St::unpack(cur[u], v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = value(v[j]);
      store_vec<ACCESS>(ow + (i64)row_words.at(at + u * TPR + t) * VEC, St::pack(v));
    };
    // as many writes as a tile makes, to nowhere: the first wait counts what every other does
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      __builtin_amdgcn_raw_buffer_store_b32(0u, row_words.row, kPastRow + 4u * u, 0, 0);
    int at = 0;
    for (; at + UNROLL * TPR <= words; at += UNROLL * TPR) {
      u32x4 next[UNROLL];
      row_words.template load<TPR, UNROLL>(at + UNROLL * TPR, t, next);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) put(u, at);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) cur[u] = next[u];
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (at + u * TPR + t < words) put(u, at);
    if constexpr (ACCESS == kRagged) sp.store_rest(rest, op, t, value);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);              // vmcnt(0): this wave's writes are done
  R::sync();
  if (list.empty || list.bad) twice = false;
  twice = R::any(twice);
  if (list.empty || list.bad) return;
#pragma unroll
  for (int k = 0; k < EPL; ++k) {
    if (list.at[k] < c0 || list.at[k] >= c1) continue;   // absent, or another part's
    float p = list.e[k];
    if (twice) {
      p = 0.0f;
      for (int i = 0; i < count; ++i) p += list_at[slot][i] == list.at[k] ? list_p[slot][i] : 0.0f;
    }
    St::store(op + list.at[k], g * (__builtin_amdgcn_exp2f((list.z[k] - ref) * c) / total - p));
  }
}

}  // namespace nep
