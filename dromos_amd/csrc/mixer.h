// What the operators of a linear-attention mixer (lx_rotate, lx_causal_conv, lx_linear_attention) share: the device's view of a call's
// rows and of the states that sequences keep, and the bounds that keep every access inside them whatever the numbers in device
// memory are.
#pragma once

#include "tile_mfma.h"

namespace dro {

struct MixBatch {
  const int32_t* rows;
  const int32_t* lengths;
  int seqs, max_rows, T;
};

// One sequence of a call: its first row, the position of that row, and the rows [first, stop) of it that count.
struct MixSpan {
  int row0, lead, first, stop;
  bool begins;  // with this call: no state to go on from
};

__host__ __device__ __forceinline__ int mix_clamp(int v, int low, int high) { return v < low ? low : v > high ? high : v; }

__host__ __device__ __forceinline__ MixSpan mix_span_of(const MixBatch& b, int from, int to, int length) {
  MixSpan p;
  p.row0 = mix_clamp(from, 0, b.T);
  const int end = mix_clamp(to, 0, b.T), n = end > p.row0 ? end - p.row0 : 0;
  p.lead = b.lengths ? mix_clamp(length, 0, 1 << 30) - n : 0;
  p.first = p.lead < 0 ? -p.lead : 0;
  p.stop = n < b.max_rows ? n : b.max_rows;
  p.begins = b.lengths && p.lead <= 0;
  return p;
}

// The numbers are asked for at once: no address depends on a branch. Without rows a sequence has one; without lengths none begins.
__device__ __forceinline__ MixSpan mix_span(const MixBatch& b, int s) {
  const int from = b.rows ? b.rows[s] : s, to = b.rows ? b.rows[s + 1] : s + 1, length = b.lengths ? b.lengths[s] : 0;
  return mix_span_of(b, from, to, length);
}

// A call's rows fall into pieces of up to `size` rows of one sequence. Piece j of sequence s is number rows[s] / size + s + j: numbers do not
// meet, since a sequence of n rows has at most (rows[s] + n) / size + 1 - rows[s] / size pieces, and there are fewer than
// T / size + seqs. Where no sequence has more than one piece, number s is sequence s.
struct MixPieces {
  int size;
  int single;
};

inline MixPieces mix_pieces(const MixBatch& b, int size) { return {size, !b.rows || b.max_rows <= size}; }
inline int64_t mix_piece_count(const MixBatch& b, const MixPieces& p) { return p.single ? b.seqs : static_cast<int64_t>(b.T) / p.size + b.seqs; }

// The last sequence whose number is not behind w, as every wavefront finds it for itself, 64 candidates at a time; -1 where there is none. Numbers
// ascend.
template <typename Number>
__device__ __forceinline__ int mix_last(int seqs, int64_t w, Number number) {
  if (seqs == 1) return number(0) <= w ? 0 : -1;
  const int lane = threadIdx.x % kWave;
  int low = 0, count = seqs;
  while (true) {
    const int step = (count + kWave - 1) / kWave, at = lane * step;
    const bool here = at < count && number(low + (at < count ? at : 0)) <= w;
    const uint64_t set = __ballot(here);
    if (!set) return -1;
    const int last = (kWave - 1 - __builtin_clzll(set)) * step;
    low += last;
    count = count - last < step ? count - last : step;
    if (count <= 1) return __builtin_amdgcn_readfirstlane(low);
  }
}

// The sequence of piece w and the piece's number in it; false where there is none.
__device__ __forceinline__ bool mix_find(const MixBatch& b, const MixPieces& p, int64_t w, int& s, int& j) {
  if (p.single) {
    s = static_cast<int>(w), j = 0;
    return w < b.seqs;
  }
  auto number = [&](int i) { return static_cast<int64_t>(mix_clamp(b.rows[i], 0, b.T) / p.size) + i; };
  s = mix_last(b.seqs, w, number);
  const int64_t of = s < 0 ? w : w - number(s);
  j = static_cast<int>(of);
  return s >= 0 && of <= b.T / p.size;
}

// The same among the sequences of more than one piece alone, which start more than `size` rows apart: piece j of sequence s is number
// 2 (rows[s] / size) + j, which a sequence of n > size rows, (rows[s] + n) / size - rows[s] / size >= 1 whole sizes apart from the next one, does not
// exceed, and all of them are fewer than 2 (T / size). The last sequence that starts in a size is the one, if any is.
__device__ __forceinline__ bool mix_find_long(const MixBatch& b, int size, int64_t w, int& s, int& j) {
  auto number = [&](int i) { return 2 * static_cast<int64_t>(mix_clamp(b.rows[i], 0, b.T) / size); };
  s = mix_last(b.seqs, w, number);
  const int64_t of = s < 0 ? w : w - number(s);
  j = static_cast<int>(of);
  return s >= 0 && of <= b.T / size;
}

// Whether those numbers find all pieces of sequence s, as they do wherever rows ascend: if they find its first and last ones, then those between them, since a
// search for a later number never ends in front of one for an earlier one. Both searches in one.
__device__ __forceinline__ bool mix_all_found(const MixBatch& b, int size, int s, const MixSpan& span) {
  if (b.seqs == 1) return true;
  const int lane = threadIdx.x % kWave, first = 2 * (span.row0 / size), last = first + (span.stop - 1) / size;  // at most 2 T / size
  int low = 0, count = b.seqs;
  while (true) {
    const int step = (count + kWave - 1) / kWave, at = lane * step;
    const int number = 2 * (mix_clamp(b.rows[low + (at < count ? at : 0)], 0, b.T) / size);
    const uint64_t before_first = __ballot(at < count && number <= first), before_last = __ballot(at < count && number <= last);
    if (!before_first) return false;
    const int pick = kWave - 1 - __builtin_clzll(before_last);
    if (pick != kWave - 1 - __builtin_clzll(before_first)) return false;
    low += pick * step;
    count = count - pick * step < step ? count - pick * step : step;
    if (count <= 1) return __builtin_amdgcn_readfirstlane(low) == s;
  }
}

struct MixStates {
  const void* in;
  void* out;
  const int32_t* slots;
  int count;
};

// The slot of sequence s, or -1.
__device__ __forceinline__ int mix_slot(const MixStates& t, int s) {
  const int slot = t.slots ? t.slots[s] : s;
  return slot >= 0 && slot < t.count ? slot : -1;
}

// v / (1 + exp(-v)), right to 2^-21, of any v: the exponent's product in two parts, one reciprocal in place of a division. Below -87, where that would be
// no normal number, nothing (the value is less than 2e-36).
__device__ __forceinline__ float quick_silu(float v) {
  const float x = fminf(fmaxf(-v, -87.0f), 87.0f), t = x * 1.44269502f;
  const float rest = __builtin_fmaf(x, 1.44269502f, -t);  // what t's rounding left, exactly
  float e = __builtin_amdgcn_exp2f(t);
  e = __builtin_fmaf(e, __builtin_fmaf(x, 1.334976e-8f, rest * 0.693147181f), e);  // log2(e) - 1.44269502 is 1.92596e-8
  return v * (v < -87.0f ? 0.0f : __builtin_amdgcn_rcpf(1.0f + e));
}

inline bool mix_type(lx_dtype t) { return t == LX_F32 || t == LX_BF16; }
inline int mix_size(int type) { return type == LX_BF16 ? 2 : 4; }
// Whether a tensor of rows can be moved `bytes` bytes at a time.
inline bool mix_aligned(const void* p, int64_t ld, int type, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * mix_size(type) % bytes == 0;
}

// Host side: 0 or the status to refuse with. Positions, and what is added to them on the way, stay below 2^31.
inline int mix_check(const lx_kv8_batch* b, int T) {
  if (T < 0 || T >= (1 << 30)) return kInvalid;
  if (!b || b->seqs < 0 || b->seqs > (1 << 30) || b->max_rows < 0) return kInvalid;
  return kOk;
}
inline int mix_check_states(const lx_states* s) {
  return s && (s->in || s->out) && s->count < 0 ? kInvalid : kOk;
}
inline MixBatch mix_batch(const lx_kv8_batch& b, int T) {
  const int seqs = b.rows || b.seqs < T ? b.seqs : T;  // without rows a sequence has row s
  const int most = b.rows ? (b.max_rows < T ? b.max_rows : T) : (b.max_rows < 1 ? 0 : 1);
  return {b.rows, b.lengths, seqs, most, T};
}
inline MixStates mix_states(const lx_states* s) { return s ? MixStates{s->in, s->out, s->slots, s->count} : MixStates{}; }

// Eight values as bf16, `wide` where they can be read 16 (bf16) or 32 (f32) bytes at a time.
__device__ __forceinline__ u32x4 load_eight_bf16(const void* p, int type, bool wide, int64_t i) {
  u32x4 r;
  if (type == LX_BF16) {
    const uint16_t* const h = static_cast<const uint16_t*>(p) + i;
    if (wide) return *reinterpret_cast<const u32x4*>(h);
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = h[2 * j] | static_cast<uint32_t>(h[2 * j + 1]) << 16;
  } else {
    const float* const f = static_cast<const float*>(p) + i;
    float v[8];
    if (wide) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(f), b = *reinterpret_cast<const f32x4*>(f + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = f[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_bit_cast(uint32_t, pack_bf16(v[2 * j], v[2 * j + 1]));
  }
  return r;
}

// Four values, `wide` where they can be moved 8 (bf16) or 16 (f32) bytes at a time.
__device__ __forceinline__ f32x4 load_four(const void* p, int type, bool wide, int64_t i) {
  f32x4 v;
  if (!wide) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = load_as_f32(p, type, i + j);
  } else if (type == LX_BF16) {
    const u32x2 r = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t a = r.x, b = r.y;
    v = f32x4{__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u), __uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)};
  } else {
    v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
  }
  return v;
}

__device__ __forceinline__ void store_four(void* p, int type, bool wide, int64_t i, const f32x4& v) {
  if (!wide) {
#pragma unroll
    for (int j = 0; j < 4; ++j) store_from_f32(p, type, i + j, v[j]);
  } else if (type == LX_BF16) {
    const u32x2 r = {__builtin_bit_cast(uint32_t, pack_bf16(v[0], v[1])), __builtin_bit_cast(uint32_t, pack_bf16(v[2], v[3]))};
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p) + i) = r;
  } else {
    *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = v;
  }
}

}  // namespace dro
