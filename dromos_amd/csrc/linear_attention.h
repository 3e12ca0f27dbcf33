// The arguments of lx_linear_attention's kernels, and what they share: the decay of a token.
#pragma once

#include "mixer.h"

namespace dro {

struct LinearArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* x;  // the decay's numbers of each row
  const float* rate;
  const float* bias;
  const float* skip;
  const void* gate;
  void* out;
  int64_t ld_q, ld_k, ld_v, ld_x, ld_gate, ld_out;
  int type, x_type, gate_type, out_type;
  int kind, heads, k_heads, group, dk, dv;
  int wide;  // every row can be moved 16 bytes at a time
  float scale;
  MixBatch b;
  MixStates states;
};

// Below this exp() times any f32 is zero: logarithms of decays are held above it, so that sums of them and differences of sums stay
// numbers (and exact) where a state is forgotten altogether.
constexpr float kForgotten = -200.0f;

// z / (1 + exp(-z)) as a gate of bf16 results, whose rounding is 2^-8: right to 2^-21 near zero, 2^-24 |z| beyond.
__device__ __forceinline__ float gate_of(float z) { return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }

// The functions of a decay without the library's care for every argument: a wavefront makes a chunk's while the others wait for it. log(1 + u), u in 0 .. 1, and
// e^x - 1, -0.5 < x <= 0, to a few steps of the result: what rounding 1 + u (or e^x) leaves off cancels in the quotient (Kahan).
__device__ __forceinline__ float quick_log1p(float u) {
  const float w = 1.0f + u, d = w - 1.0f;
  return d == 0.0f ? u : __builtin_amdgcn_logf(w) * 0.693147181f * (u * __builtin_amdgcn_rcpf(d));
}
__device__ __forceinline__ float quick_exp(float x) {
  const float t = x * 1.44269502f, rest = __builtin_fmaf(x, 1.44269502f, -t), e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, __builtin_fmaf(x, 1.334976e-8f, rest * 0.693147181f), e);  // log2(e) - 1.44269502 is 1.92596e-8
}
__device__ __forceinline__ float quick_expm1(float x) {
  const float e = quick_exp(x), d = e - 1.0f;
  return d == 0.0f ? x : d * x * __builtin_amdgcn_rcpf(__builtin_amdgcn_logf(e) * 0.693147181f);
}

// e^log in two parts: rounded, near 1, it is off to the same side time after time. The first is rounded down and the second above nothing, 2^-149 at least, so that the state's
// products with both have one sign and an infinite one stays what it is.
struct Fade {
  float high, low;
};
__device__ __forceinline__ Fade fade_from(float high, float low) {
  if (low < 0.0f) {
    const float below = __int_as_float(__float_as_int(high) - 1);
    low += high - below, high = below;
  }
  return {high, high > 0.0f ? fmaxf(low, 0x1p-149f) : 0.0f};
}
__device__ __forceinline__ Fade fade_of(float log) {
  const float less = quick_expm1(log), high = 1.0f + less;
  return log > -0.5f ? fade_from(high, less - (high - 1.0f)) : fade_from(quick_exp(log), 0.0f);
}

// A head's decays: what they are made of but for a row's own number.
struct HeadDecay {
  float rate, bias;
};
__device__ __forceinline__ HeadDecay head_decay(const LinearArgs& p, int head) {
  return {p.rate ? p.rate[head] : p.kind == LX_DECAY_STEP ? -1.0f : 1.0f, p.bias ? p.bias[head] : 0.0f};
}
// A row's own number (1: none), as it lies in memory: asked for well before it is used.
__device__ __forceinline__ uint32_t decay_raw(const LinearArgs& p, int64_t row, int head) {
  if (p.kind == LX_DECAY_HEAD) return 0x3f800000u;
  const int64_t at = row * p.ld_x + head;
  return p.x_type == LX_BF16 ? static_cast<const uint16_t*>(p.x)[at] : static_cast<const uint32_t*>(p.x)[at];
}
// The decay's logarithm and the weight of the update of a row and head.
__device__ __forceinline__ void decay_of(const LinearArgs& p, const HeadDecay& d, uint32_t raw, float& log, float& weight) {
  float x = __uint_as_float(p.x_type == LX_BF16 && p.kind != LX_DECAY_HEAD ? raw << 16 : raw);
  weight = 1.0f;
  if (p.kind == LX_DECAY_STEP) {
    const float t = x + d.bias;
    x = fmaxf(t, 0.0f) + quick_log1p(quick_exp(fmaxf(-fabsf(t), -100.0f)));  // log(1 + exp(t))
    weight = x = t != t ? t : x;
  }
  log = x * d.rate;
  log = log < kForgotten ? kForgotten : log > -kForgotten ? -kForgotten : log;
}

}  // namespace dro
