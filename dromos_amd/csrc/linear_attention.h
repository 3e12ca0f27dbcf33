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

// Below this exp() is zero in f32 (and in f64): logarithms of decays are held above it, so that sums of them and differences of
// sums stay numbers where a state is forgotten altogether.
constexpr float kForgotten = -1e4f;

// The decay's logarithm and the weight of the update of a row and head.
__device__ __forceinline__ void decay_of(const LinearArgs& p, int64_t row, int head, float& log, float& weight) {
  weight = 1.0f;
  if (p.kind == LX_DECAY_HEAD) {
    log = p.rate[head];
  } else {
    const float x = load_as_f32(p.x, p.x_type, row * p.ld_x + head);
    if (p.kind == LX_DECAY_LOG) {
      log = p.rate ? x * p.rate[head] : x;
    } else {
      const float t = p.bias ? x + p.bias[head] : x;
      weight = fmaxf(t, 0.0f) + log1pf(expf(-fabsf(t)));  // log(1 + exp(t))
      weight = t != t ? t : weight;
      log = p.rate ? weight * p.rate[head] : -weight;
    }
  }
  log = log < kForgotten ? kForgotten : log;
}

}  // namespace dro
