// lx_linear_attention, token by token: single tokens and a few drafted ones.
//
// S = e^g S + b k v^T, out = scale S^T q: of every value of the state two multiply-adds a token, and eight bytes of memory a call.
// Bytes decide, so a state is read once and written once, in pieces that are whole lines, everything asked for before the first use: a
// wavefront takes 4 COLS columns of one head's state (all its rows: no other wavefront is waited for), four columns a lane,
// 64 / COLS parts of the rows. The columns' sums over the rows cross the lanes once a token.
#pragma once

#include "linear_attention.h"

namespace dro {

// COLS lanes side by side in a row of the state; ROWS rows of it a lane.
template <int COLS, int ROWS>
__global__ void __launch_bounds__(256, ROWS >= 32 ? 2 : 4) linear_step_kernel(const LinearArgs p) {
  static_assert(COLS == 4 || COLS == 8, "lanes of a row");
  static_assert(ROWS % 8 == 0, "keys are read eight at a time");
  const int lane = threadIdx.x % kWave;
  const int blocks = (p.dv + 4 * COLS - 1) / (4 * COLS);
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * (blockDim.x / kWave) + threadIdx.x / kWave;
  const int64_t unit = wave / blocks;
  const int s = static_cast<int>(unit / p.heads), head = static_cast<int>(unit % p.heads);
  if (s >= p.b.seqs) return;
  const MixSpan span = mix_span(p.b, s);
  if (span.first >= span.stop) return;
  const int column = static_cast<int>(wave % blocks) * (4 * COLS) + lane % COLS * 4;
  const int row0 = lane / COLS * ROWS;  // of the state
  const bool mine = column < p.dv;
  const int slot = mix_slot(p.states, s);
  const int64_t size = static_cast<int64_t>(p.dk) * p.dv;
  const int64_t at = (static_cast<int64_t>(slot) * p.heads + head) * size + static_cast<int64_t>(row0) * p.dv + column;

  f32x4 state[ROWS];
  const bool reads = p.states.in && slot >= 0 && !span.begins && mine;
#pragma unroll
  for (int i = 0; i < ROWS; i += 8)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      state[i + j] = reads && row0 + i < p.dk ? *reinterpret_cast<const f32x4*>(static_cast<const float*>(p.states.in) + at + static_cast<int64_t>(i + j) * p.dv) : f32x4{};

  const int k_head = head / p.group;
  const float skip = p.skip ? p.skip[head] : 0.0f;
  u32x4 key[ROWS / 8], query[ROWS / 8];
  f32x4 value;
  float log, weight;
  auto ask = [&](int i) {
    const int64_t row = span.row0 + i;
    const int64_t k_at = static_cast<int64_t>(k_head) * p.dk + row0;
#pragma unroll
    for (int r = 0; r < ROWS / 8; ++r) {
      const bool in = row0 + 8 * r < p.dk;
      key[r] = in ? load_eight_bf16(p.k, p.type, p.wide, row * p.ld_k + k_at + 8 * r) : u32x4{};
      query[r] = in ? load_eight_bf16(p.q, p.type, p.wide, row * p.ld_q + k_at + 8 * r) : u32x4{};
    }
    value = mine ? load_four(p.v, p.type, p.wide, row * p.ld_v + static_cast<int64_t>(head) * p.dv + column) : f32x4{};
    if (p.type != LX_BF16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) value[j] = bf16_bits_to_f32(f32_to_bf16_bits(value[j]));
    }
    decay_of(p, row, head, log, weight);
  };
  ask(span.first);
  for (int i = span.first; i < span.stop; ++i) {
    u32x4 ks[ROWS / 8], qs[ROWS / 8];
#pragma unroll
    for (int r = 0; r < ROWS / 8; ++r) ks[r] = key[r], qs[r] = query[r];
    const f32x4 v = value * weight;
    const float now = log;
    if (i + 1 < span.stop) ask(i + 1);
    f32x4 o = {};
    // e^g in two parts: rounded, near 1, it is off to the same side token after token (after 4096 tokens of a memory as long, 3e-4 were
    // missing).
    const float less = expm1f(now), slow = 1.0f + less, fade = now > -0.5f ? slow : expf(now), left = now > -0.5f ? less - (slow - 1.0f) : 0.0f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const uint32_t two_k = ks[r / 8][r % 8 / 2], two_q = qs[r / 8][r % 8 / 2];
      const float k = __uint_as_float(r % 2 ? two_k & 0xffff0000u : two_k << 16), q = __uint_as_float(r % 2 ? two_q & 0xffff0000u : two_q << 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        state[r][j] = __builtin_fmaf(state[r][j], fade, __builtin_fmaf(state[r][j], left, k * v[j]));
        o[j] = __builtin_fmaf(q, state[r][j], o[j]);
      }
      if (r % 2) __builtin_amdgcn_sched_barrier(0);  // left alone, products of all rows are made before the first sum, in registers that are not there
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (COLS == 4) o[j] += dpp_move<0x124>(o[j]);  // row_ror:4
      o[j] += dpp_move<0x128>(o[j]);                 // row_ror:8
      float a, b;
      swap_halves<true>(o[j], a, b);
      const float half = a + b;
      swap_halves<false>(half, a, b);
      o[j] = (a + b) * p.scale;
    }
    if (mine && lane < COLS) finish_four(p, span.row0 + i, head, column, o, skip);
  }
  if (!p.states.out || slot < 0 || !mine) return;
#pragma unroll
  for (int i = 0; i < ROWS; i += 8)
    if (row0 + i < p.dk) {
#pragma unroll
      for (int j = 0; j < 8; ++j) *reinterpret_cast<f32x4*>(static_cast<float*>(p.states.out) + at + static_cast<int64_t>(i + j) * p.dv) = state[i + j];
    }
}

}  // namespace dro
