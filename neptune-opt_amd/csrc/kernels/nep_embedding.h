// nep_embedding.h -- embedding lookup with a scale, and the table's gradient by sorted tokens (gfx950).
//
//   out[i] = scale * table[token i]               dtable[v] = scale * sum over i with token i = v of grad[i]
// A negative token stands for none: a row of zeros, and no gradient.  A token of `vocab` or more has a row
// of NaN and no gradient; neither is read through.  Products and sums are fp32, rounded once.
//
// Gradient.  The tokens are put in order, equal ones by position, so that every row of the table is the sum of
// one run of entries, added in one order, without atomics:
//   order   the tokens' places, by counting
//   sums    a wavefront adds a chunk of entries over its columns, several rows in flight; runs that end
//           inside the chunk are written, the others' parts are kept in fp32; further workgroups clear the
//           rows that no token names
//   join    the parts of each run of several chunks, in order
// or, of few tokens, by one launch in which each row's first token finds the others.
//
// HBM-bound: the lookup reads and writes a row per token (bf16 16384 x 4096 28 us, 7.1 TB/s), the gradient reads a
// row per token and writes the table's (16384 tokens of 128256 x 4096 223 us: order 9, sums and clearing 202 at 5.8
// TB/s, join 7; fp16 55087 tokens of 32003 x 1001 60 us: 16, 40, 5).
#pragma once

namespace nep {

typedef float f32x4e __attribute__((ext_vector_type(4)));

// How rows are read and written: aligned 16-byte words; words of any alignment, the last one from the
// row's end (so that it overlaps the one before it); fewer columns than a word holds, one by one.
constexpr int kRowWords = 0, kRowAny = 1, kRowFew = 2;

template <class St, int ACCESS, bool STREAM>
__device__ __forceinline__ u32x4 row_word(const typename St::T* p, int n) {
  if constexpr (ACCESS == kRowWords) return STREAM ? load16(p) : load16_cached(p);
  else if constexpr (ACCESS == kRowAny) return STREAM ? load16_any_once(p) : load16_any(p);
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

// ---------------------------------------------------------------- tokens in order
constexpr int kMostKeys = 1024;                      // rows of the table that a workgroup counts
constexpr int kMostTokenStride = 16;

// Sums of the lanes before each lane, over the workgroup, and of all; `lds` holds an int per wavefront.
template <int WAVES>
__device__ __forceinline__ int exclusive_sum(int v, int* lds, int& all) {
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __builtin_amdgcn_ds_bpermute((lane - d) * 4, s);
    s += lane >= d ? o : 0;
  }
  __syncthreads();                                   // the last sums have been read
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    before += w < wave ? lds[w] : 0;
    all += lds[w];
  }
  return before + s - v;
}

// In a wavefront: what its lanes have stored in LDS is there for its other lanes' reads behind, and is read before their
// stores behind.  (LDS takes a wavefront's accesses in order; this keeps the compiler to it.)
__device__ __forceinline__ void lanes_meet() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The tokens by (token mod W, token / W), then by position, W = 2^log_shares workgroups: workgroup w has the
// tokens that are w mod W, and its places are behind those of the workgroups before it.  Each of its wavefronts
// walks a run of the positions (of less than 2^22), lists its tokens and counts them (and those of earlier
// workgroups); when the counters have become places, the list goes there.  Every workgroup reads all tokens (from L2, a
// few instructions for 64 of them), and none waits for another: 65536 tokens of 32000 rows 20 us, 262144 113, 1048576
// 458; above 2^18 rows there are more workgroups (262144 tokens of 2^20 rows 176 us, of 2^24 2326).  Frequent tokens, often neighbours, spread over
// the workgroups; a wavefront whose list is too short walks its run again, and empties it when it is full.
// `named` gets a byte for each row of the table: whether a token names it.  Places behind the last token
// have the key `vocab`.
template <class Ix, int WAVES>
__device__ __forceinline__ void embedding_order(const Ix* __restrict__ tokens, u32* __restrict__ keys,
                                                u32* __restrict__ positions, unsigned char* __restrict__ named,
                                                i64 count, u32 vocab, i64 stride_i, int log_shares) {
  constexpr int THREADS = WAVES * 64, BATCHES = 4, GROUP = 64 * BATCHES, LIST = 1024;
  __shared__ int counters[WAVES][kMostKeys];
  __shared__ u32 list[WAVES][LIST];                  // key / W, and the position in the run behind it
  __shared__ int sums[WAVES];
  static_assert(kMostKeys <= 1 << 10, "32 bits hold an entry");
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const u32 share = blockIdx.x, mask = (1u << log_shares) - 1;
  const int mine = share < vocab ? (int)((vocab - 1 - share) >> log_shares) + 1 : 0;    // keys
  for (int k = lane; k < mine; k += 64) counters[wave][k] = 0;
  lanes_meet();
  const i64 run = ((count + THREADS - 1) / THREADS) * 64;
  const i64 first = wave * run < count ? wave * run : count, end = first + run < count ? first + run : count;
  // A group of positions, through a buffer: no load is in a branch, so that the wait for one group leaves the next
  // in flight (in branches 55087 tokens 18 us, so 16).  Past the run's end nothing is read and the tokens are absent.
  // (strides are at most kMostTokenStride, so that a run's bytes stay below 2^30)
  const u32 step = (u32)stride_i * (u32)sizeof(Ix);
  const __amdgpu_buffer_rsrc_t run_words = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(tokens + first * stride_i), (short)0, end > first ? (int)((end - first - 1) * step + sizeof(Ix)) : 0,
      (int)0x00020000);
  const int size = (int)(end - first);
  auto load = [&](int i0, Ix* token) {
#pragma unroll
    for (int b = 0; b < BATCHES; ++b) {
      const u32 at = (u32)(i0 + b * 64 + lane) * step;
      if constexpr (sizeof(Ix) == 8) {
        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(run_words, at, 0, 0);
        token[b] = (Ix)((u64)w.x | (u64)w.y << 32);
      } else {
        token[b] = (Ix)__builtin_amdgcn_raw_buffer_load_b32(run_words, at, 0, 0);
      }
    }
  };
  // The remainder of a token, which is the workgroup that it belongs to; an unknown token is of none.  (`left`:
  // tokens of the run from the batch on)
  auto owner = [&](Ix token, int left) -> u32 {
    bool known = (u32)token < vocab;
    if constexpr (sizeof(Ix) == 8) known = known && (u32)((u64)token >> 32) == 0;
    u32 of = known ? (u32)token & mask : ~0u;
    if (left < 64 * BATCHES) of = lane < left ? of : ~0u;                // (the run's last group)
    return of;
  };
  // every group of the wavefront's run, the next one's tokens in flight
  auto walk = [&](auto each) {
    Ix a[BATCHES], b[BATCHES];
    load(0, a);
    for (int i0 = 0; i0 < size; i0 += 2 * GROUP) {
      load(i0 + GROUP, b);
      each(i0, a);
      load(i0 + 2 * GROUP, a);
      each(i0 + GROUP, b);
    }
  };
  int listed = 0;
  // a batch's own tokens (there is room for a batch), to the list
  auto note = [&](bool own, u64 some, u32 key, int position) {
    const int at = listed + __builtin_amdgcn_mbcnt_hi((u32)(some >> 32), __builtin_amdgcn_mbcnt_lo((u32)some, 0));
    if (own) list[wave][at] = (key >> log_shares) << 22 | (u32)position;
    listed += __builtin_popcountll(some);
  };
  auto tally = [&]() {                               // counts the list's tokens
    lanes_meet();
    for (int l = lane; l < listed; l += 64)
      __hip_atomic_fetch_add(&counters[wave][list[wave][l] >> 22], 1, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_WORKGROUP);
    lanes_meet();
  };
  int earlier = 0;                                   // of the wavefront
  bool whole = true;                                 // the list holds all of them
  walk([&](int i0, const Ix* token) {
#pragma unroll
    for (int b = 0; b < BATCHES; ++b) {
      const u32 of = owner(token[b], size - i0 - b * 64);
      earlier += __builtin_popcountll(__builtin_amdgcn_uicmp(of, share, 36));    // less than
      const u64 some = __builtin_amdgcn_uicmp(of, share, 32);                    // equal
      if (some == 0) continue;
      if (listed + 64 > LIST) {
        tally();
        listed = 0;
        whole = false;
      }
      note(of == share, some, (u32)token[b], i0 + b * 64 + lane);
    }
  });
  tally();
  int base;
  exclusive_sum<WAVES>(lane == 0 ? earlier : 0, sums, base);         // (its barriers are behind all counts)
  for (int k0 = 0; k0 < mine; k0 += THREADS) {
    const int k = k0 + threadIdx.x;
    int total = 0, all;
    if (k < mine) {
#pragma unroll
      for (int w = 0; w < WAVES; ++w) total += counters[w][k];
    }
    int place = base + exclusive_sum<WAVES>(total, sums, all);
    if (k < mine) {
      named[((u32)k << log_shares) | share] = total > 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const int c = counters[w][k];
        counters[w][k] = place;
        place += c;
      }
    }
    base += all;
  }
  __syncthreads();
  if (share == mask)
    for (i64 i = base + (int)threadIdx.x; i < count; i += THREADS) keys[i] = vocab;
  // the list's tokens, which are in order of their positions, to their places
  const int bits = mine > 1 ? 32 - __builtin_clz(mine - 1) : 0;
  auto empty = [&]() {
    lanes_meet();
    for (int l0 = 0; l0 < listed; l0 += 64) {
      const bool here = l0 + lane < listed;
      const u32 entry = here ? list[wave][l0 + lane] : 0;
      const int k = (int)(entry >> 22);
      u64 same = __builtin_amdgcn_ballot_w64(here);
      for (int b = 0; b < bits; ++b) {
        const bool bit = (k >> b) & 1;
        const u64 set = __builtin_amdgcn_ballot_w64(bit);
        same &= bit ? set : ~set;
      }
      const int before = __builtin_amdgcn_mbcnt_hi((u32)(same >> 32), __builtin_amdgcn_mbcnt_lo((u32)same, 0));
      if (here) {
        // (the wavefront's own counters: its reads and writes stay in order)
        volatile int* counter = &counters[wave][k];
        const int place = *counter + before;
        if (before == 0) *counter = place + __builtin_popcountll(same);
        keys[place] = (u32)k << log_shares | share;
        positions[place] = (u32)first + (entry & 0x3fffffu);
      }
      lanes_meet();
    }
  };
  if (whole) {
    empty();
    return;
  }
  listed = 0;
  walk([&](int i0, const Ix* token) {
#pragma unroll
    for (int b = 0; b < BATCHES; ++b) {
      const u32 of = owner(token[b], size - i0 - b * 64);
      const u64 some = __builtin_amdgcn_uicmp(of, share, 32);
      if (some == 0) continue;
      if (listed + 64 > LIST) {
        empty();
        listed = 0;
      }
      note(of == share, some, (u32)token[b], i0 + b * 64 + lane);
    }
  });
  empty();
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

// Zeros to the rows that no token names, four words a lane: of rows of up to 64 words, 2^log_lanes lanes each; or of
// one row, in 2^log_tiles wavefronts.  The wavefronts walk the table's memory in order, 4 KB each, so that few of
// the memory's pages are open and the wait for `named` is hidden (1.05 GB by workgroups of a wavefront 171 us, by
// larger ones with four words a lane 182-196, a word a lane 157, but not behind a load).
// `named` has a byte for each row from `base` on.
template <class St, int ACCESS>
__device__ __forceinline__ void clear_rows(const unsigned char* named, u32 base, typename St::T* __restrict__ table,
                                           u32 block, int n, u32 vocab, int log_lanes, int log_tiles) {
  constexpr int WORDS = 4;
  const int lane = lane_id();
  const u32x4 zero = {0u, 0u, 0u, 0u};
  auto clear = [&](u32 row, int at) {
    typename St::T* p = table + (i64)row * n + word_column<St, ACCESS>(at, n);
    if constexpr (ACCESS == kRowWords) *(u32x4*)p = zero;
    else if constexpr (ACCESS == kRowAny) *(u32x4_any*)p = zero;
    else
      for (int j = 0; j < n; ++j) St::store(p + j, 0.0f);
  };
  if (log_lanes < 7) {
    const int rows = 64 >> log_lanes, at = lane & ((1 << log_lanes) - 1);
    const u32 first = block * (WORDS * rows) + (lane >> log_lanes);
    bool empty[WORDS];
#pragma unroll
    for (int u = 0; u < WORDS; ++u) empty[u] = first + u * rows < vocab && !named[first + u * rows - base];
#pragma unroll
    for (int u = 0; u < WORDS; ++u)
      if (empty[u] && at * St::kVec < n) clear(first + u * rows, at);
  } else {
    const u32 row = block >> log_tiles;
    const int first = (int)(block & ((1u << log_tiles) - 1)) * 64 * WORDS + lane;
    if (row >= vocab || named[row - base]) return;
#pragma unroll
    for (int u = 0; u < WORDS; ++u)
      if ((first + u * 64) * St::kVec < n) clear(row, first + u * 64);
  }
}

// Workgroup (a wavefront) b < sums: chunk b / columns of `chunk` entries, columns of the word of lane
// (b % columns) * 64 + lane; the workgroups behind clear the other rows.  parts: [chunks][2][lanes][VEC] fp32,
// of the run that the chunk before began (0), and of the one that begins here and goes on (1).
template <class St, class Ot, int ACCESS, bool ADD>
__device__ __forceinline__ void embedding_sums(const typename St::T* __restrict__ grad,
                                               const u32* __restrict__ keys, const u32* __restrict__ positions,
                                               const unsigned char* __restrict__ named,
                                               typename Ot::T* __restrict__ table, float* __restrict__ parts,
                                               i64 count, int n, u32 vocab, i64 stride_g, i64 stride_t, int chunk,
                                               int columns, u32 sums, int log_lanes, int log_tiles, float scale) {
  constexpr int VEC = St::kVec, FLIGHT = 8;
  if constexpr (!ADD) {
    if (blockIdx.x >= sums) {
      clear_rows<Ot, ACCESS>(named, 0, table, blockIdx.x - sums, n, vocab, log_lanes, log_tiles);
      return;
    }
  }
  const u32 number = blockIdx.x / columns;           // of the chunk
  const int lane = lane_id(), at = (blockIdx.x - number * columns) * 64 + lane;
  const bool active = at * VEC < n;
  const int column = active ? word_column<St, ACCESS>(at, n) : 0;
  const i64 first = (i64)number * chunk, end = first + chunk < count ? first + chunk : count;
  const i64 lanes = (i64)columns * 64;
  float* part = parts + ((i64)number * 2 * lanes + at) * VEC;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
  u32 current = keys[first];
  const u32 last = keys[first > 0 ? first - 1 : 0], next = keys[end < count ? end : count - 1];
  if (current >= vocab) return;                      // absent tokens are last
  bool before = first > 0 && last == current;        // the current run began in front of this chunk
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
  flush(end < count && next == current);
}

// The run that begins in chunk blockIdx.x and goes on behind it, if there is one: its parts, over the words of
// the 64 lanes of blockIdx.y.  The WAVES wavefronts take the parts in turn, and their sums are added in order.
template <class St, class Ot, int ACCESS, bool ADD, int WAVES>
__device__ __forceinline__ void embedding_join(const u32* __restrict__ keys, const float* __restrict__ parts,
                                               typename Ot::T* __restrict__ table, i64 count, int n, u32 vocab,
                                               i64 stride_t, int chunk, int chunks, float scale) {
  constexpr int VEC = St::kVec, FLIGHT = 8;
  __shared__ float lds[WAVES][64][VEC + 4];
  const i64 first = (i64)blockIdx.x * chunk, end = first + chunk;
  if (end >= count) return;
  const u32 key = keys[end - 1], behind = keys[end], begin = keys[first], before = keys[first > 0 ? first - 1 : 0];
  if (key >= vocab || behind != key) return;
  if (first > 0 && begin == key && before == key) return;                  // it began earlier
  const int lane = lane_id();
  int items = 1;                                     // this chunk's part, and one of each that begins with the run
  for (int c0 = (int)blockIdx.x + 1; c0 < chunks; c0 += 64) {
    const bool goes_on = c0 + lane < chunks && keys[(i64)(c0 + lane) * chunk] == key;
    const u64 ends = ~__builtin_amdgcn_ballot_w64(goes_on);
    items += ends != 0 ? (int)__builtin_ctzll(ends) : 64;
    if (ends != 0) break;
  }
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), at = blockIdx.y * 64 + lane;
  const i64 lanes = (i64)gridDim.y * 64;
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
  for (int w = 1; w < WAVES && w < items; ++w)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += lds[w][lane][j];
  write_row<Ot, ACCESS, ADD, VEC>(table + (i64)key * stride_t, acc, scale, at,
                                  word_column<St, ACCESS>(at, n), n);
}

// ---------------------------------------------------------------- few tokens
constexpr int kFewTokens = 512;

// Up to kFewTokens tokens in one launch (512 of 1000 x 768 fp32 5.2 us, ordered 13.5; 256 of 32000 x 4096 bf16
// 35.7, 41.2; 512 times one token 15-18, ordered 12-14, and twice that with 1024).  Workgroup b < sums: the row of
// token b / columns where that is its first, over the words of 64 lanes; its four wavefronts take the row's tokens
// in turn, and their sums are added in order.  The workgroups behind mark the tokens of the rows that they clear in
// LDS.
template <class St, class Ot, class Ix, int ACCESS, bool ADD>
__device__ __forceinline__ void embedding_few(const Ix* __restrict__ tokens, const typename St::T* __restrict__ grad,
                                              typename Ot::T* __restrict__ table, int count, int n, u32 vocab,
                                              i64 stride_i, i64 stride_g, i64 stride_t, int columns, u32 sums,
                                              int log_lanes, int log_tiles, float scale) {
  constexpr int VEC = St::kVec, FLIGHT = 8, WAVES = 4, LANES = 64 * WAVES, EACH = kFewTokens / LANES;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), tid = threadIdx.x;
  u32 key[EACH];                                     // of tokens tid, tid + LANES, ...
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = e * LANES + tid;
    const i64 token = i < count ? (i64)tokens[i * stride_i] : -1;
    key[e] = token >= 0 && token < (i64)vocab ? (u32)token : ~0u;
  }
  if constexpr (!ADD) {
    __shared__ u32 marks[256];                       // a byte for each of 1024 rows
    unsigned char* named = (unsigned char*)marks;
    if (blockIdx.x >= sums) {
      const u32 block = blockIdx.x - sums, per = 64 >> (log_lanes < 6 ? log_lanes : 6);
      const u32 base = log_lanes < 7 ? block * (WAVES * 4 * per) : block * WAVES >> log_tiles;
      marks[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EACH; ++e)
        if (key[e] - base < 1024) named[key[e] - base] = 1;              // (of at most 16 * 64 rows)
      __syncthreads();
      clear_rows<Ot, ACCESS>(named, base, table, block * WAVES + wave, n, vocab, log_lanes, log_tiles);
      return;
    }
  }
  __shared__ u32 keys[kFewTokens];
  __shared__ u16 list[kFewTokens];
  __shared__ int found[EACH][WAVES];
  __shared__ float lds[WAVES][64][VEC + 4];
  const int number = blockIdx.x / columns, at = (blockIdx.x - number * columns) * 64 + lane;
#pragma unroll
  for (int e = 0; e < EACH; ++e) keys[e * LANES + tid] = key[e];
  __syncthreads();
  const u32 mine = keys[number];
  bool first = mine != ~0u;
  u64 same[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    same[e] = __builtin_amdgcn_ballot_w64(key[e] == mine);
    if (lane == 0) found[e][wave] = __builtin_popcountll(same[e]);
    first = first && !(key[e] == mine && e * LANES + tid < number);
  }
  if (__syncthreads_or(!first)) return;
  int items = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    int place = items + __builtin_amdgcn_mbcnt_hi((u32)(same[e] >> 32), __builtin_amdgcn_mbcnt_lo((u32)same[e], 0));
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      place += w < wave ? found[e][w] : 0;
      items += found[e][w];
    }
    if (key[e] == mine) list[place] = (u16)(e * LANES + tid);
  }
  __syncthreads();
  const bool active = at * VEC < n;
  const int column = active ? word_column<St, ACCESS>(at, n) : 0;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
  for (int i0 = wave; i0 < items; i0 += WAVES * FLIGHT) {
    u32x4 w[FLIGHT];
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      const int i = i0 + f * WAVES;
      const i64 row = (i64)list[i < items ? i : i0] * stride_g;
      if (active) w[f] = row_word<St, ACCESS, true>(grad + row + column, n);
    }
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      if (i0 + f * WAVES < items) {
        float v[VEC];
        St::unpack(w[f], v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += v[j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) lds[wave][lane][j] = acc[j];
  __syncthreads();
  if (wave > 0 || !active) return;
  for (int w = 1; w < WAVES && w < items; ++w)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += lds[w][lane][j];
  write_row<Ot, ACCESS, ADD, VEC>(table + (i64)mine * stride_t, acc, scale, at, column, n);
}

}  // namespace nep
