// nep_embedding.h -- embedding lookup with a scale, and the table's gradient by sorted tokens (gfx950).
//
//   out[i] = scale * table[token i]               dtable[v] = scale * sum over i with token i = v of grad[i]
// A negative token stands for none: a row of zeros, and no gradient.  A token of `vocab` or more has a row
// of NaN and no gradient; neither is read through.  Products and sums are fp32, rounded once.
//
// Gradient.  The tokens are sorted (by token, then by position), so that every row of the table is the sum
// of one run of sorted entries, added in one order, without atomics:
//   sort    pieces of the tokens, each by a workgroup in LDS, while the others clear the table
//   merge   (more than one piece) an entry's place is its own in its piece and those of the other pieces'
//           entries in front of it, found by bisection
//   sums    a wavefront adds a chunk of entries over its columns, several rows in flight; runs that end
//           inside the chunk are written, the others' parts are kept in fp32
//   join    the parts of each run of several chunks, in order
#pragma once

namespace nep {

typedef float f32x4e __attribute__((ext_vector_type(4)));

// How rows are read and written: aligned 16-byte words; words of any alignment, the last one from the
// row's end (so that it overlaps the one before it); fewer columns than a word holds, one by one.
constexpr int kRowWords = 0, kRowAny = 1, kRowFew = 2;

template <class St, int ACCESS, bool STREAM>
__device__ __forceinline__ u32x4 row_word(const typename St::T* p, int n) {
  if constexpr (ACCESS == kRowWords) return STREAM ? load16(p) : load16_cached(p);
  else if constexpr (ACCESS == kRowAny) return load16_any(p);
  else {
    float v[St::kVec];
#pragma unroll
    for (int j = 0; j < St::kVec; ++j) v[j] = j < n ? St::load(p + j) : 0.0f;
    return St::pack(v);
  }
}

// First column of the word that lane position `at` of a row holds.
template <class St, int ACCESS>
__device__ __forceinline__ int word_column(int at, int n) {
  const int e = at * St::kVec;
  return ACCESS == kRowAny && e + St::kVec > n ? n - St::kVec : e;
}

// COUNT values v to the elements of type Ot behind p, those in front of `from` left alone.
template <class Ot, int ACCESS, int COUNT>
__device__ __forceinline__ void store_values(typename Ot::T* p, const float* v, int n, int from) {
  constexpr int PER = Ot::kVec;
  if (ACCESS != kRowFew && from == 0) {
#pragma unroll
    for (int j = 0; j < COUNT; j += PER) {
      if constexpr (ACCESS == kRowWords) store16(p + j, Ot::pack(v + j));
      else store16_any(p + j, Ot::pack(v + j));
    }
  } else {
#pragma unroll
    for (int j = 0; j < COUNT; ++j)
      if (j >= from && (ACCESS != kRowFew || j < n)) Ot::store(p + j, v[j]);
  }
}

// ---------------------------------------------------------------- lookup
// TPR lanes a row, U words a lane in flight and tile.
template <class St, class Ix, int TPR, int U, int ACCESS>
__device__ __forceinline__ void embedding(const Ix* __restrict__ tokens, const typename St::T* __restrict__ table,
                                          typename St::T* __restrict__ out, i64 rows, int n, i64 vocab,
                                          i64 stride_i, i64 stride_t, float scale) {
  constexpr int VEC = St::kVec;
  const int t = threadIdx.x % TPR;
  const i64 row = (i64)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;
  const i64 token = (i64)tokens[row * stride_i];
  const bool known = token >= 0 && token < vocab;
  const float fill = token < 0 ? 0.0f : __builtin_nanf("");
  const typename St::T* from = table + (known ? token : 0) * stride_t;
  typename St::T* to = out + row * n;
  for (int first = blockIdx.y * TPR * U; first * VEC < n; first += gridDim.y * TPR * U) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = first + u * TPR + t;
      if (known && at * VEC < n) w[u] = row_word<St, ACCESS, false>(from + word_column<St, ACCESS>(at, n), n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = first + u * TPR + t;
      if (at * VEC >= n) continue;
      float v[VEC];
      St::unpack(w[u], v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = known ? v[j] * scale : fill;
      store_values<St, ACCESS, VEC>(to + word_column<St, ACCESS>(at, n), v, n, 0);
    }
  }
}

// ---------------------------------------------------------------- sorting the tokens
constexpr int kDigit = 9;                            // bits of a digit at most
constexpr int kPerLane = 4;                          // entries of a lane

// Sums of the lanes before each lane, over the workgroup; `lds` holds an int per wavefront.
template <int WAVES>
__device__ __forceinline__ int exclusive_sum(int v, int* lds) {
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __builtin_amdgcn_ds_bpermute((lane - d) * 4, s);
    s += lane >= d ? o : 0;
  }
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) before += w < wave ? lds[w] : 0;
  return before + s - v;
}

// Piece blockIdx.x of THREADS * kPerLane tokens: keys (the token, or `vocab` for an absent one) and
// positions in order, to its place in `keys` and `positions`.  A stable sort by `passes` digits of `width`
// bits, from the last: a wavefront's lanes with one digit are found by a ballot for each of its bits.
template <class Ix, int THREADS>
__device__ __forceinline__ void sort_tokens(const Ix* __restrict__ tokens, u32* __restrict__ keys,
                                            u32* __restrict__ positions, i64 count, i64 vocab, i64 stride_i,
                                            int width, int passes) {
  constexpr int WAVES = THREADS / 64, PIECE = THREADS * kPerLane, COUNTERS = WAVES << kDigit;
  constexpr int MINE = COUNTERS / THREADS;           // counters of a lane
  __shared__ u16 counters[WAVES][1 << kDigit];
  __shared__ u32 lds_keys[PIECE], lds_positions[PIECE];
  __shared__ int sums[WAVES];
  const int lane = lane_id(), wave = threadIdx.x >> 6, place = wave * 64 * kPerLane + lane;
  const i64 first = (i64)blockIdx.x * PIECE;
  u32 key[kPerLane], position[kPerLane];
#pragma unroll
  for (int r = 0; r < kPerLane; ++r) {
    const i64 i = first + place + r * 64;
    const i64 token = i < count ? (i64)tokens[i * stride_i] : -1;
    key[r] = (u32)(token >= 0 && token < vocab ? token : vocab);
    position[r] = (u32)i;
  }
  volatile u16* mine = counters[wave];
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * width, digits = 1 << width;
    for (int d = lane; d < digits; d += 64) mine[d] = 0;
    int rank[kPerLane];
#pragma unroll
    for (int r = 0; r < kPerLane; ++r) {
      const u32 digit = (key[r] >> shift) & (digits - 1);
      u64 same = ~0ull;
      for (int b = 0; b < width; ++b) {
        const bool bit = (digit >> b) & 1;
        const u64 set = __builtin_amdgcn_ballot_w64(bit);
        same &= bit ? set : ~set;
      }
      const int before = __builtin_amdgcn_mbcnt_hi((u32)(same >> 32), __builtin_amdgcn_mbcnt_lo((u32)same, 0));
      const int base = mine[digit];
      if (before == 0) mine[digit] = (u16)(base + __builtin_popcountll(same));
      rank[r] = base + before;
    }
    __syncthreads();
    // counters by (digit, wavefront) become the sums of those in front
    int own[MINE], total = 0;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int c = threadIdx.x * MINE + i;
      own[i] = c < digits * WAVES ? counters[c % WAVES][c / WAVES] : 0;
      total += own[i];
    }
    int before = exclusive_sum<WAVES>(total, sums);
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int c = threadIdx.x * MINE + i;
      if (c < digits * WAVES) counters[c % WAVES][c / WAVES] = (u16)before;
      before += own[i];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kPerLane; ++r) {
      const int to = rank[r] + mine[(key[r] >> shift) & (digits - 1)];
      lds_keys[to] = key[r];
      lds_positions[to] = position[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kPerLane; ++r) {
      key[r] = lds_keys[place + r * 64];
      position[r] = lds_positions[place + r * 64];
    }
  }
#pragma unroll
  for (int r = 0; r < kPerLane; ++r) {
    const i64 i = first + place + r * 64;
    keys[i] = key[r];
    positions[i] = position[r];
  }
}

// The first `pieces` workgroups sort, the others (if any) write zeros over `bytes` bytes from the 16-byte
// aligned `table`.
template <class Ix, int THREADS>
__device__ __forceinline__ void embedding_sort(const Ix* __restrict__ tokens, u32* __restrict__ keys,
                                               u32* __restrict__ positions, char* __restrict__ table, i64 count,
                                               i64 vocab, i64 stride_i, i64 bytes, int width, int passes,
                                               int pieces) {
  if ((int)blockIdx.x < pieces) {
    sort_tokens<Ix, THREADS>(tokens, keys, positions, count, vocab, stride_i, width, passes);
    return;
  }
  const i64 words = bytes / 16, at = (i64)(blockIdx.x - pieces) * THREADS + threadIdx.x;
  const i64 step = (i64)(gridDim.x - pieces) * THREADS;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (i64 w = at; w < words; w += step) store16(table + w * 16, zero);
  for (i64 b = words * 16 + at * 2; b < bytes; b += step * 2) *(u16*)(table + b) = 0;
}

// Entries of `keys[0..size)` (in order) that are less than `key`, or not more.
__device__ __forceinline__ int count_before(const u32* keys, int size, u32 key, bool or_same) {
  int lo = 0, n = size;
  while (n > 0) {
    const int half = n >> 1;
    const u32 k = keys[lo + half];
    const bool up = or_same ? k <= key : k < key;
    lo = up ? lo + half + 1 : lo;
    n = up ? n - half - 1 : half;
  }
  return lo;
}

// blockIdx.x: 256 * kPerLane entries of the pieces of PIECE entries.  Entries past `count` have the last
// places, and are not written.
template <int PIECE>
__device__ __forceinline__ void embedding_merge(const u32* __restrict__ keys, const u32* __restrict__ positions,
                                                u32* __restrict__ keys_out, u32* __restrict__ positions_out,
                                                i64 count, int pieces) {
  constexpr int SHARE = 256 * kPerLane;
  __shared__ u32x4 words[PIECE / 4];
  const u32* other = (const u32*)words;
  const int piece = (int)(((i64)blockIdx.x * SHARE) / PIECE);
  const i64 first = (i64)blockIdx.x * SHARE;
  u32 key[kPerLane], position[kPerLane];
  i64 to[kPerLane];
#pragma unroll
  for (int r = 0; r < kPerLane; ++r) {
    const i64 i = first + r * 256 + threadIdx.x;
    key[r] = keys[i];
    position[r] = positions[i];
    to[r] = i - (i64)piece * PIECE;
  }
  for (int p = 0; p < pieces; ++p) {
    if (p == piece) continue;
    __syncthreads();
    for (int w = threadIdx.x; w < PIECE / 4; w += 256) words[w] = load16_cached(keys + (i64)p * PIECE + w * 4);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kPerLane; ++r) to[r] += count_before(other, PIECE, key[r], p < piece);
  }
#pragma unroll
  for (int r = 0; r < kPerLane; ++r)
    if ((i64)position[r] < count && to[r] < count) {
      keys_out[to[r]] = key[r];
      positions_out[to[r]] = position[r];
    }
}

// ---------------------------------------------------------------- sums
// A finished row: scale * acc, plus what the row holds already (ADD).
template <class Ot, int ACCESS, bool ADD, int VEC>
__device__ __forceinline__ void write_row(typename Ot::T* row, const float* acc, float scale, int at, int column,
                                          int n) {
  float v[VEC];
  // an overlapping word's first columns are its neighbour's
  const int from = ADD ? at * VEC - column : 0;
  if constexpr (ADD) {
    if constexpr (ACCESS == kRowFew) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = j < n ? Ot::load(row + j) : 0.0f;
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j += Ot::kVec)
        Ot::unpack(row_word<Ot, ACCESS, true>(row + column + j, n), v + j);
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) v[j] = ADD ? __builtin_fmaf(scale, acc[j], v[j]) : scale * acc[j];
  store_values<Ot, ACCESS, VEC>(row + column, v, n, from);
}

// Chunk blockIdx.x of `chunk` entries (a multiple of 64 or less than it), columns of the word of lane
// blockIdx.y * 256 + threadIdx.x.  parts: [chunks][2][lanes][VEC] fp32, of the run that the chunk before
// began (0), and of the one that begins here and goes on (1).
template <class St, class Ot, int ACCESS, bool ADD>
__device__ __forceinline__ void embedding_sums(const typename St::T* __restrict__ grad,
                                               const u32* __restrict__ keys, const u32* __restrict__ positions,
                                               typename Ot::T* __restrict__ table, float* __restrict__ parts,
                                               i64 count, int n, u32 vocab, i64 stride_g, i64 stride_t, int chunk,
                                               float scale) {
  constexpr int VEC = St::kVec, FLIGHT = 8;
  const int lane = lane_id(), at = blockIdx.y * 256 + threadIdx.x;
  const int wave_at = __builtin_amdgcn_readfirstlane(at - lane);
  if (wave_at * VEC >= n) return;
  const bool active = at * VEC < n;
  const int column = active ? word_column<St, ACCESS>(at, n) : 0;
  const i64 first = (i64)blockIdx.x * chunk, end = first + chunk < count ? first + chunk : count;
  const i64 lanes = (i64)gridDim.y * 256;
  float* part = parts + ((i64)blockIdx.x * 2 * lanes + at) * VEC;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
  u32 current = keys[first];
  if (current >= vocab) return;                      // absent tokens are last
  // whether the current run began in front of this chunk
  bool before = first > 0 && keys[first - 1] == current;
  auto flush = [&](bool goes_on) {
    if (!active) return;
    if (before || goes_on) {
      float* p = part + (before ? 0 : lanes * VEC);
#pragma unroll
      for (int j = 0; j < VEC; j += 4) *(f32x4e*)(p + j) = f32x4e{acc[j], acc[j + 1], acc[j + 2], acc[j + 3]};
    } else {
      write_row<Ot, ACCESS, ADD, VEC>(table + (i64)current * stride_t, acc, scale, at, column, n);
    }
  };
  const typename St::T* base = grad + column;
  for (i64 i0 = first; i0 < end; i0 += 64) {
    const bool here = i0 + lane < end;
    const u32 key = here ? keys[i0 + lane] : vocab, position = here ? positions[i0 + lane] : 0;
    const int live = __builtin_popcountll(__builtin_amdgcn_ballot_w64(key < vocab));
    for (int s = 0; s < live; s += FLIGHT) {
      u32x4 w[FLIGHT];
#pragma unroll
      for (int j = 0; j < FLIGHT; ++j) {
        // (entries past the last one read its row again)
        const int e = s + j < live ? s + j : live - 1;
        const u32 p = (u32)__builtin_amdgcn_readlane((int)position, e);
        if (active) w[j] = row_word<St, ACCESS, true>(base + (i64)p * stride_g, n);
      }
#pragma unroll
      for (int j = 0; j < FLIGHT; ++j) {
        if (s + j < live) {
          const u32 k = (u32)__builtin_amdgcn_readlane((int)key, s + j);
          if (k != current) {
            flush(false);
            before = false;
            current = k;
#pragma unroll
            for (int c = 0; c < VEC; ++c) acc[c] = 0.0f;
          }
          float v[VEC];
          St::unpack(w[j], v);
#pragma unroll
          for (int c = 0; c < VEC; ++c) acc[c] += v[c];
        }
      }
    }
  }
  flush(end < count && keys[end] == current);
}

// The run that begins in chunk blockIdx.x and goes on behind it, if there is one: its parts, over the
// columns of the words of the 64 lanes of blockIdx.y.  The parts are dealt to the workgroup's WAVES
// wavefronts in turn and their sums added in order.
template <class St, class Ot, int ACCESS, bool ADD, int WAVES>
__device__ __forceinline__ void embedding_join(const u32* __restrict__ keys, const float* __restrict__ parts,
                                               typename Ot::T* __restrict__ table, i64 count, int n, u32 vocab,
                                               i64 stride_t, int chunk, int chunks, i64 lanes, float scale) {
  constexpr int VEC = St::kVec, FLIGHT = 4;
  __shared__ float lds[WAVES][64][VEC + 4];
  const i64 first = (i64)blockIdx.x * chunk, end = first + chunk;
  if (end >= count) return;
  const u32 key = keys[end - 1];
  if (key >= vocab || keys[end] != key) return;
  if (first > 0 && keys[first] == key && keys[first - 1] == key) return;    // it began earlier
  // chunks whose first entry is of this run
  int lo = (int)blockIdx.x + 1, hi = chunks;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (keys[(i64)mid * chunk] == key) lo = mid;
    else hi = mid;
  }
  const int items = hi - (int)blockIdx.x;            // this chunk's part, and one of each behind it
  const int lane = lane_id(), wave = threadIdx.x >> 6, at = blockIdx.y * 64 + lane;
  const float* mine = parts + ((i64)blockIdx.x * 2 * lanes + at) * VEC;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
  for (int i0 = wave; i0 < items; i0 += WAVES * FLIGHT) {
    f32x4e v[FLIGHT][VEC / 4];
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      const int i = i0 + f * WAVES;
      const i64 slot = i == 0 ? lanes * VEC : (i64)i * 2 * lanes * VEC;
#pragma unroll
      for (int j = 0; j < VEC; j += 4)
        v[f][j / 4] = i < items ? *(const f32x4e*)(mine + slot + j) : f32x4e{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += v[f][j / 4][j % 4];
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) lds[wave][lane][j] = acc[j];
  __syncthreads();
  if (wave > 0 || at * VEC >= n) return;
  const int waves = items < WAVES ? items : WAVES;
  for (int w = 1; w < waves; ++w)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += lds[w][lane][j];
  write_row<Ot, ACCESS, ADD, VEC>(table + (i64)key * stride_t, acc, scale, at,
                                  word_column<St, ACCESS>(at, n), n);
}

}  // namespace nep
