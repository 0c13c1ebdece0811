// nep_gradients.h -- the 2-norm of many tensors together, and their scaling to a largest norm (gfx950).
//
//   norm = sqrt(sum over all elements of g^2)          out = g * min(1, max_norm / norm)
// Squares and sums are fp64: the square of an fp32 number neither overflows nor vanishes there, and the
// conversion and the FMA are hidden behind the loads.  The norm is rounded to fp32 once and the factor comes
// from the rounded norm, so that a norm computed before gives the same bits.  A norm that is an infinity or
// NaN has no factor: the elements stay as they are.
//
// Lists of up to kTensors tensors are given by value, in a launch's arguments: nothing is copied to the device, and
// a captured launch keeps its own list.  Longer ones (up to kMostTensors a launch) are put together in device memory
// by small launches that hold a part each (0.9 GB in 290 tensors: 135 us so, 148 by three launches of the sums).
// The elements are dealt to the workgroups in turn, in pieces of `piece` elements that do not cross tensors; a
// workgroup finds a piece's tensor among the first pieces' numbers, in LDS, by two ballots (the arguments lie far
// away, so each is read once).
//
// HBM-bound: the norm reads its tensors once (0.89 GB bf16 135 us, 6.6 TB/s), a scaling reads them again and writes
// (0.54 GB bf16 into fp32 83 + 295 us, 5.5 TB/s; 0.1 GB fp16 20 + 38).
#pragma once

namespace nep {

constexpr int kTensors = 112;                        // 3584 bytes; all arguments stay below 4096
constexpr int kMostTensors = 4096;
constexpr int kSumLanes = 1024;
constexpr int kPieceLanes = 256;                     // lanes that share a piece
constexpr u32 kAtOnce = kSumLanes / kPieceLanes;     // pieces that a workgroup has at a time

struct alignas(16) TensorEntry {
  const void* in;
  void* out;
  u64 count;                                         // elements, at least one
  u32 first;                                         // number of its first piece
  u32 kind;                                          // types of in and out
};
struct TensorList {
  TensorEntry entry[kTensors];
};

// in and out
constexpr u32 kF32 = 0, kBF16 = 1, kF16 = 2, kBF16ToF32 = 3, kF16ToF32 = 4;

__device__ __forceinline__ void copy_entry_words(u32x4* to, const TensorEntry* from, int count) {
  for (int i = threadIdx.x; i < 2 * count; i += kSumLanes) to[i] = ((const u32x4*)from)[i];
}
// A part of a long list, to its place.
__device__ __forceinline__ void gradient_list(const TensorList& list, int count, TensorEntry* __restrict__ to) {
  copy_entry_words((u32x4*)to, list.entry, count);
}

// A list as a workgroup sees it: a short one is copied to LDS (FAR false), of a long one the numbers of the first
// pieces.
template <bool FAR>
struct Tensors {
  static constexpr int MOST = FAR ? kMostTensors : kTensors;
  const TensorEntry* entries;
  const u32* firsts;
  int count, step;

  // `lds`: room for a list by value; `numbers`: MOST words.  All lanes, once.
  __device__ __forceinline__ Tensors(const TensorEntry* given, int n, u32x4* lds, u32* numbers)
      : entries(FAR ? given : (const TensorEntry*)lds), firsts(numbers), count(n), step((n + 63) / 64) {
    if constexpr (!FAR) copy_entry_words(lds, given, n);
    for (int i = threadIdx.x; i < n; i += kSumLanes) numbers[i] = given[i].first;
    __syncthreads();
  }
  // The entry that piece p (of a wavefront) belongs to: the last with a first piece of p or less (the first has 0).
  __device__ __forceinline__ TensorEntry entry(u32 p) const {
    const int lane = lane_id(), at = lane * step;
    const u64 low = __builtin_amdgcn_ballot_w64(at < count && firsts[at < count ? at : 0] <= p);
    const int begin = (__builtin_popcountll(low) - 1) * step, i = begin + lane;
    const u64 in = __builtin_amdgcn_ballot_w64(lane < step && i < count && firsts[i < count ? i : 0] <= p);
    const TensorEntry e = entries[begin + __builtin_popcountll(in) - 1];
    // (the same in every lane, so that addresses are scalar)
    auto same = [](u64 v) {
      return (u64)(u32)__builtin_amdgcn_readfirstlane((int)(u32)v) |
             (u64)(u32)__builtin_amdgcn_readfirstlane((int)(u32)(v >> 32)) << 32;
    };
    return {(const void*)same((u64)e.in), (void*)same((u64)e.out), same(e.count),
            (u32)__builtin_amdgcn_readfirstlane((int)e.first), (u32)__builtin_amdgcn_readfirstlane((int)e.kind)};
  }
};

// Sum over the workgroup of kSumLanes lanes, the same in every lane.  (lds: a double per wavefront)
__device__ __forceinline__ double workgroup_sum(double v, double* lds) {
  const int lane = lane_id();
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) {
    const u64 b = __builtin_bit_cast(u64, v);
    const int from = (lane ^ d) * 4;
    const u64 lo = (u32)__builtin_amdgcn_ds_bpermute(from, (int)(u32)b);
    const u64 hi = (u32)__builtin_amdgcn_ds_bpermute(from, (int)(u32)(b >> 32));
    v += __builtin_bit_cast(double, lo | hi << 32);
  }
  if (lane == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < kSumLanes / 64; ++w) total += lds[w];
  return total;
}

// Squares of elements [first, end) of p, added to acc, by kPieceLanes lanes.
template <class St>
__device__ __forceinline__ void add_squares(const typename St::T* p, i64 first, i64 end, double& acc) {
  constexpr int VEC = St::kVec, FLIGHT = 4;
  const int lane = threadIdx.x % kPieceLanes;
  const i64 words = (end - first) / VEC;
  p += first;
  for (i64 w0 = 0; w0 < words; w0 += kPieceLanes * FLIGHT) {
    u32x4 w[FLIGHT];
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      const i64 i = w0 + f * kPieceLanes + lane;
      w[f] = i < words ? load16_any_once(p + i * VEC) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      float v[VEC];
      St::unpack(w[f], v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc = __builtin_fma((double)v[j], (double)v[j], acc);
    }
  }
  const i64 rest = words * VEC + lane;
  if (rest < end - first) {
    const double v = (double)St::load(p + rest);
    acc = __builtin_fma(v, v, acc);
  }
}

// The squares of the pieces first, first + step, ...: a lane's share.
template <class List>
__device__ __forceinline__ double piece_squares(const List& tensors, u32 first, u32 step, u32 pieces, int piece) {
  double acc = 0.0;
  for (u32 p = first; p < pieces; p += step) {
    const TensorEntry e = tensors.entry(p);
    const i64 from = (i64)(p - e.first) * piece;
    const i64 end = from + piece < (i64)e.count ? from + piece : (i64)e.count;
    if (e.kind == kF32) add_squares<F32>((const float*)e.in, from, end, acc);
    else if (e.kind == kBF16 || e.kind == kBF16ToF32) add_squares<BF16>((const u16*)e.in, from, end, acc);
    else add_squares<F16>((const _Float16*)e.in, from, end, acc);
  }
  return acc;
}

template <bool FAR>
__device__ __forceinline__ void gradient_sums(const TensorEntry* list, int count, u32 pieces, int piece,
                                              double* __restrict__ sums) {
  __shared__ double lds[kSumLanes / 64];
  __shared__ u32x4 words[FAR ? 1 : 2 * kTensors];
  __shared__ u32 numbers[Tensors<FAR>::MOST];
  const Tensors<FAR> tensors(list, count, words, numbers);
  const u32 group = __builtin_amdgcn_readfirstlane(threadIdx.x / kPieceLanes);
  const double acc = piece_squares(tensors, blockIdx.x * kAtOnce + group, gridDim.x * kAtOnce, pieces, piece);
  const double total = workgroup_sum(acc, lds);
  if (threadIdx.x == 0) sums[blockIdx.x] = total;
}

// The norm from the workgroups' sums.
__device__ __forceinline__ float norm_of(const double* __restrict__ sums, int count) {
  __shared__ double lds[kSumLanes / 64];
  double acc = 0.0;
  for (int i = threadIdx.x; i < count; i += kSumLanes) acc += sums[i];
  return (float)__builtin_sqrt(workgroup_sum(acc, lds));
}

__device__ __forceinline__ void gradient_norm(const double* __restrict__ sums, int count, float* __restrict__ norm) {
  const float v = norm_of(sums, count);
  if (threadIdx.x == 0) *norm = v;
}

// A lane's values fill the word that it writes: eight bytes of 16-bit numbers make a word of fp32 (half the words
// of a store's lines at a time, by words read whole, 417 us; so 274, for 1.6 GB read and written).
template <class St, class Ot>
__device__ __forceinline__ void scale_elements(const typename St::T* p, typename Ot::T* q, i64 first, i64 end,
                                               float factor) {
  typedef u32 u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
  constexpr int VEC = Ot::kVec, FLIGHT = St::kVec == VEC ? 4 : 8;
  const int lane = threadIdx.x % kPieceLanes;
  const i64 words = (end - first) / VEC;
  p += first;
  q += first;
  for (i64 w0 = 0; w0 < words; w0 += kPieceLanes * FLIGHT) {
    u32x4 w[FLIGHT];
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      const i64 i = w0 + f * kPieceLanes + lane;
      if (i >= words) continue;
      if constexpr (St::kVec == VEC) {
        w[f] = load16_any_once(p + i * VEC);
      } else {
        const u32x2 half = __builtin_nontemporal_load(reinterpret_cast<const u32x2_any*>(p + i * VEC));
        w[f] = u32x4{half.x, half.y, 0u, 0u};
      }
    }
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      const i64 i = w0 + f * kPieceLanes + lane;
      if (i >= words) continue;
      float v[St::kVec];
      St::unpack(w[f], v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] *= factor;
      store16_any(q + i * VEC, Ot::pack(v));
    }
  }
  const i64 rest = words * VEC + lane;
  if (rest < end - first) Ot::store(q + rest, St::load(p + rest) * factor);
}

__device__ __forceinline__ float factor_of(float norm, float max_norm) {
  return is_finite(norm) && norm > max_norm ? div_rn(max_norm, norm) : 1.0f;
}

// The pieces first, first + step, ... times `factor`.
template <class List>
__device__ __forceinline__ void scale_pieces(const List& tensors, u32 first, u32 step, u32 pieces, int piece,
                                             float factor) {
  for (u32 p = first; p < pieces; p += step) {
    const TensorEntry e = tensors.entry(p);
    if (factor == 1.0f && e.in == e.out) continue;
    const i64 from = (i64)(p - e.first) * piece;
    const i64 end = from + piece < (i64)e.count ? from + piece : (i64)e.count;
    if (e.kind == kF32) scale_elements<F32, F32>((const float*)e.in, (float*)e.out, from, end, factor);
    else if (e.kind == kBF16) scale_elements<BF16, BF16>((const u16*)e.in, (u16*)e.out, from, end, factor);
    else if (e.kind == kF16) scale_elements<F16, F16>((const _Float16*)e.in, (_Float16*)e.out, from, end, factor);
    else if (e.kind == kBF16ToF32) scale_elements<BF16, F32>((const u16*)e.in, (float*)e.out, from, end, factor);
    else scale_elements<F16, F32>((const _Float16*)e.in, (float*)e.out, from, end, factor);
  }
}

// `sums` null: the norm is given.  `copies`: whether an entry's out is not its in.
template <bool FAR>
__device__ __forceinline__ void gradient_scale(const TensorEntry* list, int count, u32 pieces, int piece,
                                               const double* __restrict__ sums, int n_sums,
                                               const float* __restrict__ given, float* __restrict__ norm_out,
                                               float max_norm, int copies) {
  const float norm = sums != nullptr ? norm_of(sums, n_sums) : *given;
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  const float factor = factor_of(norm, max_norm);
  if (factor == 1.0f && !copies) return;
  __shared__ u32x4 words[FAR ? 1 : 2 * kTensors];
  __shared__ u32 numbers[Tensors<FAR>::MOST];
  const Tensors<FAR> tensors(list, count, words, numbers);
  const u32 group = __builtin_amdgcn_readfirstlane(threadIdx.x / kPieceLanes);
  scale_pieces(tensors, blockIdx.x * kAtOnce + group, gridDim.x * kAtOnce, pieces, piece, factor);
}

// A short list of few elements by one workgroup: the norm, and where `scale` is set the scaling behind it.
__device__ __forceinline__ void gradient_one(const TensorEntry* list, int count, u32 pieces, int piece,
                                             float* __restrict__ norm_out, float max_norm, int scale, int copies) {
  __shared__ double lds[kSumLanes / 64];
  __shared__ u32x4 words[2 * kTensors];
  __shared__ u32 numbers[kTensors];
  const Tensors<false> tensors(list, count, words, numbers);
  const u32 group = __builtin_amdgcn_readfirstlane(threadIdx.x / kPieceLanes);
  // (the sum's barrier is behind all reads)
  const float norm = (float)__builtin_sqrt(workgroup_sum(piece_squares(tensors, group, kAtOnce, pieces, piece), lds));
  if (threadIdx.x == 0) *norm_out = norm;
  const float factor = factor_of(norm, max_norm);
  if (!scale || (factor == 1.0f && !copies)) return;
  scale_pieces(tensors, group, kAtOnce, pieces, piece, factor);
}

}  // namespace nep
