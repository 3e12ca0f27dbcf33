// lx_causal_conv: a short causal convolution along each sequence, a filter of its own for every channel, the last inputs kept between calls.
//
// Bytes decide: x is read once (and again the width - 1 rows in front of a piece, from L2), y written once. A thread takes
// eight channels of a piece of a sequence's rows and slides over them with the last rows in registers, four rows ahead on their way. The first
// piece of a sequence reads the rows it kept, and leaves the new ones (no other piece looks at either), so `in` and `out` may
// be the same. A single token is a chain of loads: the sequence's bounds and slot, its kept rows; filters are asked for before the first of them.
// 4096 rows of 10240 channels, bf16, four taps: 33.4 us (5.0 TB/s; 61.0 us a row at a time), 64 sequences of one row of them
// 5.6 us (12.9 us with filters read a value at a time). Five sequences of 611 rows of 2050 channels f32, which only two at a time are aligned: 9.5 us
// (15.0 us one at a time).
#include "mixer.h"

namespace dro {
namespace {

constexpr int kMaxWidth = 8;  // taps
constexpr int kAhead = 4;     // rows on their way

struct ConvArgs {
  const void* x;
  const void* w;
  const void* bias;
  void* y;
  int64_t ld_x, ld_y;
  int x_type, w_type, y_type, width, silu, C;
  int blocks;  // workgroups side by side in a row
  int w_wide;  // the filters of eight channels can be read 16 bytes at a time
  MixBatch b;
  MixPieces pieces;
  MixStates states;
};

// V channels as they lie in memory: eight, two or one.
template <int V>
struct Channels {
  u32x4 low, high;
};
template <>
struct Channels<2> {
  u32x2 v;
};
template <>
struct Channels<1> {
  uint32_t v;
};

template <int V>
__device__ __forceinline__ Channels<V> load_raw(const void* p, int type, int64_t i) {
  Channels<V> r{};
  if constexpr (V == 1) {
    r.v = type == LX_BF16 ? static_cast<const uint16_t*>(p)[i] : static_cast<const uint32_t*>(p)[i];
  } else if constexpr (V == 2) {
    if (type == LX_BF16) r.v.x = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i);
    else r.v = *reinterpret_cast<const u32x2*>(static_cast<const float*>(p) + i);
  } else if (type == LX_BF16) {
    r.low = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
  } else {
    const u32x4* const q = reinterpret_cast<const u32x4*>(static_cast<const float*>(p) + i);
    r.low = q[0], r.high = q[1];
  }
  return r;
}

template <int V>
__device__ __forceinline__ void store_raw(void* p, int type, int64_t i, const Channels<V>& r) {
  if constexpr (V == 1) {
    if (type == LX_BF16) static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(r.v);
    else static_cast<uint32_t*>(p)[i] = r.v;
  } else if constexpr (V == 2) {
    if (type == LX_BF16) *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p) + i) = r.v.x;
    else *reinterpret_cast<u32x2*>(static_cast<float*>(p) + i) = r.v;
  } else if (type == LX_BF16) {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) = r.low;
  } else {
    u32x4* const q = reinterpret_cast<u32x4*>(static_cast<float*>(p) + i);
    q[0] = r.low, q[1] = r.high;
  }
}

template <int V>
__device__ __forceinline__ void values_of(const Channels<V>& r, int type, float (&v)[V]) {
  const bool half = type == LX_BF16;
  if constexpr (V == 1) {
    v[0] = __uint_as_float(half ? r.v << 16 : r.v);
  } else if constexpr (V == 2) {
    const uint32_t x = r.v.x, y = r.v.y;
    v[0] = __uint_as_float(half ? x << 16 : x);
    v[1] = __uint_as_float(half ? x & 0xffff0000u : y);
  } else if (half) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t two = r.low[j / 2];
      v[j] = __uint_as_float(j % 2 ? two & 0xffff0000u : two << 16);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t low = r.low[j], high = r.high[j];
      v[j] = __uint_as_float(low), v[4 + j] = __uint_as_float(high);
    }
  }
}

// Stored past the caches that the next kernel's other XCDs do not share.
template <int V>
__device__ __forceinline__ void store_values(void* p, int type, int64_t i, const float (&v)[V]) {
  if constexpr (V == 8) {
    if (type == LX_BF16) {
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __builtin_bit_cast(uint32_t, pack_bf16(v[2 * j], v[2 * j + 1]));
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i));
    } else {
      f32x4* const q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + i);
      __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, q);
      __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, q + 1);
    }
  } else if constexpr (V == 2) {
    if (type == LX_BF16) *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p) + i) = __builtin_bit_cast(uint32_t, pack_bf16(v[0], v[1]));
    else *reinterpret_cast<f32x2*>(static_cast<float*>(p) + i) = f32x2{v[0], v[1]};
  } else {
    store_from_f32(p, type, i, v[0]);
  }
}

// W: taps, or 0 for any number of them up to kMaxWidth.
template <int V, int W>
__global__ void __launch_bounds__(256) conv_kernel(const ConvArgs p) {
  constexpr int kTaps = W ? W : kMaxWidth;
  const unsigned piece = blockIdx.x / p.blocks;
  const int channel = (static_cast<int>(blockIdx.x % p.blocks) * 256 + static_cast<int>(threadIdx.x)) * V;
  const bool mine = channel < p.C;
  const int at = mine ? channel : 0, width = W ? W : p.width, kept = width - 1;
  float weight[kTaps][V], bias[V];
  if (V == 8 && W && p.w_wide) {
    constexpr int kPieces = W ? W : 1;
    Channels<8> raw[kPieces];  // eight values each of the eight filters
#pragma unroll
    for (int t = 0; t < kPieces; ++t) raw[t] = load_raw<8>(p.w, p.w_type, static_cast<int64_t>(at) * W + 8 * t);
    float flat[kPieces][8];
#pragma unroll
    for (int t = 0; t < kPieces; ++t) values_of<8>(raw[t], p.w_type, flat[t]);
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
      for (int t = 0; t < kTaps; ++t) weight[t][c] = flat[(c * W + t) / 8 % kPieces][(c * W + t) % 8];
  } else {
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
      for (int t = 0; t < kTaps; ++t) weight[t][c] = t < width ? load_as_f32(p.w, p.w_type, static_cast<int64_t>(at + c) * width + t) : 0.0f;
  }
#pragma unroll
  for (int c = 0; c < V; ++c) bias[c] = 0.0f;
  if (p.bias) {
    if (V == 8 && p.w_wide) {
      values_of<V>(load_raw<V>(p.bias, p.w_type, at), p.w_type, bias);
    } else {
#pragma unroll
      for (int c = 0; c < V; ++c) bias[c] = load_as_f32(p.bias, p.w_type, at + c);
    }
  }

  int s, j;
  if (!mix_find(p.b, p.pieces, piece, s, j)) return;
  const MixSpan span = mix_span(p.b, s);
  const int slot = mix_slot(p.states, s);
  const int begin = max(span.first, j * p.pieces.size), end = min(span.stop, (j + 1) * p.pieces.size);
  if (begin >= end || !mine) return;
  const bool reads = p.states.in && slot >= 0 && !span.begins;
  const int64_t state_at = static_cast<int64_t>(slot) * kept * p.C + channel, x_at = static_cast<int64_t>(span.row0) * p.ld_x + channel;
  // Row i of the sequence; the kept ones in front of the first that counts.
  auto input = [&](int i) -> Channels<V> {
    if (i >= span.first) return load_raw<V>(p.x, p.x_type, x_at + i * p.ld_x);
    const int back = i - span.first + kept;
    return reads && back >= 0 ? load_raw<V>(p.states.in, p.x_type, state_at + static_cast<int64_t>(back) * p.C) : Channels<V>{};
  };
  Channels<V> next[kAhead], before[kTaps];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) next[i] = load_raw<V>(p.x, p.x_type, x_at + min(begin + i, end - 1) * p.ld_x);
#pragma unroll
  for (int t = 0; t + 1 < kTaps; ++t)
    if (t < kept) before[t] = input(begin - kept + t);
  // What the sequence keeps: read before anything is written, since `out` may be `in`.
  if (span.first >= j * p.pieces.size && span.first < (j + 1) * p.pieces.size && p.states.out && slot >= 0) {
    Channels<V> last[kTaps];
#pragma unroll
    for (int t = 0; t + 1 < kTaps; ++t)
      if (t < kept) last[t] = input(span.stop - kept + t);
#pragma unroll
    for (int t = 0; t + 1 < kTaps; ++t)
      if (t < kept) store_raw<V>(p.states.out, p.x_type, state_at + static_cast<int64_t>(t) * p.C, last[t]);
  }
  float seen[kTaps][V];  // the last rows, the newest at kept - 1
#pragma unroll
  for (int t = 0; t + 1 < kTaps; ++t)
    if (t < kept) values_of<V>(before[t], p.x_type, seen[t]);
  for (int i0 = begin; i0 < end; i0 += kAhead) {
    Channels<V> now[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) now[i] = next[i];
    if (i0 + kAhead < end) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) next[i] = load_raw<V>(p.x, p.x_type, x_at + min(i0 + kAhead + i, end - 1) * p.ld_x);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i >= end) break;
      float x[V], y[V];
      values_of<V>(now[i], p.x_type, x);
#pragma unroll
      for (int c = 0; c < V; ++c) {
        y[c] = bias[c];
#pragma unroll
        for (int t = 0; t + 1 < kTaps; ++t)
          if (t < kept) y[c] = __builtin_fmaf(weight[t][c], seen[t][c], y[c]);
        float last = weight[kTaps - 1][c];
        if (!W) {
#pragma unroll
          for (int t = 0; t < kTaps; ++t) last = t == kept ? weight[t][c] : last;
        }
        y[c] = __builtin_fmaf(last, x[c], y[c]);
#pragma unroll
        for (int t = 0; t + 1 < kTaps; ++t) {
          if (t + 1 < kept) seen[t][c] = seen[t + 1][c];
          else if (t + 1 == kept) seen[t][c] = x[c];
        }
      }
      if (p.silu) {
        // A bf16 result does not see the last bits of the exponent: 2^-17 of the value for |y| < 64, against a rounding of 2^-8.
        if (p.y_type == LX_BF16) {
#pragma unroll
          for (int c = 0; c < V; ++c) y[c] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y[c] * -1.44269504f));
        } else {
#pragma unroll
          for (int c = 0; c < V; ++c) y[c] = quick_silu(y[c]);
        }
      }
      store_values<V>(p.y, p.y_type, static_cast<int64_t>(span.row0 + i0 + i) * p.ld_y + channel, y);
    }
  }
}

template <int V, int W>
int launch(ConvArgs p, hipStream_t s) {
  p.blocks = (p.C + 256 * V - 1) / (256 * V);
  // Rows of a piece: a filter is read for each and so are the rows in front of it, so many of them as long as eight wavefronts a unit of the device remain. 4096 rows of
  // 10240 channels: 33.4 us by 32 rows, 34.4 by 16; 2400 rows of 2050 f32 channels, half as many threads: 12.3 us and 9.5.
  const int64_t threads = static_cast<int64_t>(p.b.T) * p.blocks * 256;
  const int size = threads / 32 >= 512 * static_cast<int64_t>(compute_units()) ? 32 : 16;
  p.pieces = mix_pieces(p.b, size);
  const int64_t groups = mix_piece_count(p.b, p.pieces) * p.blocks;
  if (groups * 256 > kMaxGridThreads) return kInvalid;
  hipLaunchKernelGGL((conv_kernel<V, W>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, s, p);
  return status_of(hipGetLastError());
}

template <int V>
int launch_width(const ConvArgs& p, hipStream_t s) {
  return p.width == 4 ? launch<V, 4>(p, s) : p.width == 3 ? launch<V, 3>(p, s) : p.width == 2 ? launch<V, 2>(p, s) : launch<V, 0>(p, s);
}

}  // namespace
}  // namespace dro

using namespace dro;

extern "C" {

int lx_causal_conv(const void* x, lx_dtype x_dtype, int ld_x, const void* weight, const void* bias, lx_dtype w_dtype, int width, lx_act act,
                   const lx_kv8_batch* batch, const lx_states* states, void* y, lx_dtype y_dtype, int ld_y, int T, int C, void* stream) {
  if (int st = mix_check(batch, T)) return fail(st);
  if (int st = mix_check_states(states)) return fail(st);
  if (width < 2 || width > kMaxWidth || C < 0 || C > (1 << 24) || (act != LX_ACT_NONE && act != LX_ACT_SILU)) return fail(kInvalid);
  if (!mix_type(x_dtype) || !mix_type(w_dtype) || !mix_type(y_dtype)) return fail(kInvalid);
  if (T == 0 || C == 0 || batch->seqs == 0) return kOk;
  if (!x || !weight || !y || x == y || (T > 1 && (ld_x < C || ld_y < C))) return fail(kInvalid);
  ConvArgs p{};
  p.x = x, p.w = weight, p.bias = bias, p.y = y;
  p.ld_x = ld_x, p.ld_y = ld_y, p.x_type = x_dtype, p.w_type = w_dtype, p.y_type = y_dtype;
  p.width = width, p.silu = act == LX_ACT_SILU, p.C = C;
  p.b = mix_batch(*batch, T);
  p.states = mix_states(states);
  if (p.b.max_rows == 0 || p.b.seqs == 0) return kOk;
  auto in = [&](const void* t, int64_t ld, int type, int values) { return mix_aligned(t, T > 1 ? ld : 0, type, values == 8 ? 16 : values * mix_size(type)); };
  auto all = [&](int values) {
    return C % values == 0 && in(x, ld_x, x_dtype, values) && in(y, ld_y, y_dtype, values) && (!p.states.in || mix_aligned(p.states.in, C, x_dtype, values == 8 ? 16 : values * mix_size(x_dtype))) &&
           (!p.states.out || mix_aligned(p.states.out, C, x_dtype, values == 8 ? 16 : values * mix_size(x_dtype)));
  };
  p.w_wide = reinterpret_cast<uintptr_t>(weight) % 16 == 0 && reinterpret_cast<uintptr_t>(bias) % 16 == 0;
  hipStream_t s = as_stream(stream);
  const int st = all(8) ? launch_width<8>(p, s) : all(2) ? launch_width<2>(p, s) : launch_width<1>(p, s);
  return st ? fail(st) : kOk;
}

}  // extern "C"
