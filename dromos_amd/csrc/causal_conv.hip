// lx_causal_conv: a short causal convolution along each sequence, a filter of its own for every channel, the last inputs kept between calls.
//
// Bytes decide: x is read once (and again the width - 1 rows in front of a piece, from L2), y written once. A thread takes
// eight channels of a piece of up to kRows rows and slides over them with the last rows in registers, four rows ahead on their way. The first
// piece of a sequence reads the rows it kept, and leaves the new ones (no other piece looks at either), so `in` and `out` may
// be the same. Single tokens are a piece each: a chain of rows, lengths and slots, then the kept rows.
#include "mixer.h"

namespace dro {
namespace {

constexpr int kRows = 16;     // of a piece
constexpr int kMaxWidth = 8;  // taps

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

// V channels as they lie in memory: eight, or one.
template <int V>
struct Channels {
  u32x4 low, high;
};
template <>
struct Channels<1> {
  uint32_t v;
};

template <int V>
__device__ __forceinline__ Channels<V> load_raw(const void* p, int type, int64_t i) {
  Channels<V> r;
  if constexpr (V == 1) {
    r.v = type == LX_BF16 ? static_cast<const uint16_t*>(p)[i] : static_cast<const uint32_t*>(p)[i];
  } else if (type == LX_BF16) {
    r.low = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
    r.high = r.low;
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
  } else if (type == LX_BF16) {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) = r.low;
  } else {
    u32x4* const q = reinterpret_cast<u32x4*>(static_cast<float*>(p) + i);
    q[0] = r.low, q[1] = r.high;
  }
}

template <int V>
__device__ __forceinline__ Channels<V> no_channels() {
  Channels<V> r{};
  return r;
}

template <int V>
__device__ __forceinline__ void values_of(const Channels<V>& r, int type, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = __uint_as_float(type == LX_BF16 ? r.v << 16 : r.v);
  } else {
    const bool half = type == LX_BF16;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t two = r.low[j / 2], four = r.low[2 + j / 2], low = r.low[j], high = r.high[j];
      v[j] = __uint_as_float(half ? (j % 2 ? two & 0xffff0000u : two << 16) : low);
      v[4 + j] = __uint_as_float(half ? (j % 2 ? four & 0xffff0000u : four << 16) : high);
    }
  }
}

template <int V>
__device__ __forceinline__ void store_values(void* p, int type, int64_t i, const float (&v)[V]) {
  if constexpr (V == 1) {
    store_from_f32(p, type, i, v[0]);
  } else {
    store_four(p, type, true, i, f32x4{v[0], v[1], v[2], v[3]});
    store_four(p, type, true, i + 4, f32x4{v[4], v[5], v[6], v[7]});
  }
}

template <int V, int W>
__global__ void __launch_bounds__(256) conv_kernel(const ConvArgs p) {
  const int64_t piece = blockIdx.x / p.blocks;
  const int channel = (static_cast<int>(blockIdx.x % p.blocks) * 256 + static_cast<int>(threadIdx.x)) * V;
  int s, j;
  if (!mix_find(p.b, p.pieces, piece, s, j)) return;
  const MixSpan span = mix_span(p.b, s);
  const int begin = max(span.first, j * p.pieces.size), end = min(span.stop, (j + 1) * p.pieces.size);
  if (begin >= end || channel >= p.C) return;
  const int width = W ? W : p.width, kept = width - 1;
  constexpr int kTaps = W ? W : kMaxWidth;

  float weight[kTaps][V], bias[V];
#pragma unroll
  for (int c = 0; c < V; ++c) {
    bias[c] = p.bias ? load_as_f32(p.bias, p.w_type, channel + c) : 0.0f;
#pragma unroll
    for (int t = 0; t < kTaps; ++t) weight[t][c] = t < width ? load_as_f32(p.w, p.w_type, static_cast<int64_t>(channel + c) * width + t) : 0.0f;
  }
  const int slot = mix_slot(p.states, s);
  const bool reads = p.states.in && slot >= 0 && !span.begins;
  const int64_t state_at = static_cast<int64_t>(slot) * kept * p.C + channel;
  // The row `i` rows behind the sequence's first one that counts; the kept ones in front of it.
  auto input = [&](int i) -> Channels<V> {
    if (i >= span.first) return load_raw<V>(p.x, p.x_type, (static_cast<int64_t>(span.row0) + i) * p.ld_x + channel);
    const int back = i - span.first + kept;
    return reads && back >= 0 ? load_raw<V>(p.states.in, p.x_type, state_at + static_cast<int64_t>(back) * p.C) : no_channels<V>();
  };
  float seen[kTaps][V];  // the last rows, the newest last
#pragma unroll
  for (int t = 0; t + 1 < kTaps; ++t) {
    if (t < kept) values_of<V>(input(begin - kept + t), p.x_type, seen[t]);
  }
  // What the sequence keeps: read before anything is written, since `out` may be `in`.
  const bool keeps = span.first >= j * p.pieces.size && span.first < (j + 1) * p.pieces.size && p.states.out && slot >= 0;
  if (keeps) {
    Channels<V> last[kTaps];
#pragma unroll
    for (int t = 0; t + 1 < kTaps; ++t)
      if (t < kept) last[t] = input(span.stop - kept + t);
#pragma unroll
    for (int t = 0; t + 1 < kTaps; ++t)
      if (t < kept) store_raw<V>(p.states.out, p.x_type, state_at + static_cast<int64_t>(t) * p.C, last[t]);
  }
  for (int i = begin; i < end; ++i) {
    float now[V], y[V];
    values_of<V>(load_raw<V>(p.x, p.x_type, (static_cast<int64_t>(span.row0) + i) * p.ld_x + channel), p.x_type, now);
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
      y[c] = __builtin_fmaf(last, now[c], y[c]);
      if (p.silu) y[c] = quick_silu(y[c]);
#pragma unroll
      for (int t = 0; t + 1 < kTaps; ++t) {
        if (t + 1 < kept) seen[t][c] = seen[t + 1][c];
        else if (t + 1 == kept) seen[t][c] = now[c];
      }
    }
    store_values<V>(p.y, p.y_type, (static_cast<int64_t>(span.row0) + i) * p.ld_y + channel, y);
  }
}

template <int V, int W>
int launch(ConvArgs p, hipStream_t s) {
  p.blocks = (p.C + 256 * V - 1) / (256 * V);
  const int64_t groups = mix_piece_count(p.b, p.pieces) * p.blocks;
  if (groups * 256 > kMaxGridThreads) return kInvalid;
  hipLaunchKernelGGL((conv_kernel<V, W>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, s, p);
  return status_of(hipGetLastError());
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
  p.pieces = mix_pieces(p.b, kRows);
  p.states = mix_states(states);
  if (p.b.max_rows == 0 || p.b.seqs == 0) return kOk;
  auto in16 = [&](const void* t, int64_t ld, int type) { return mix_aligned(t, T > 1 ? ld : 0, type, 16); };
  const bool wide = C % 8 == 0 && in16(x, ld_x, x_dtype) && in16(y, ld_y, y_dtype) && (!p.states.in || in16(p.states.in, C, x_dtype)) &&
                    (!p.states.out || in16(p.states.out, C, x_dtype));
  hipStream_t s = as_stream(stream);
  int st;
  if (wide) st = width == 4 ? launch<8, 4>(p, s) : width == 3 ? launch<8, 3>(p, s) : width == 2 ? launch<8, 2>(p, s) : launch<8, 0>(p, s);
  else st = width == 4 ? launch<1, 4>(p, s) : launch<1, 0>(p, s);
  return st ? fail(st) : kOk;
}

}  // extern "C"
