// lx_linear_attention, token by token: single tokens and a few drafted ones.
//
// S = e^g S + b k v^T, out = scale S^T q: of every value of the state two multiply-adds a token, and eight bytes of memory a call.
// Bytes decide, so a state is read once and written once, in pieces that are whole lines, everything asked for before the first use: a
// wavefront takes 4 COLS columns of one head's state (all its rows: no other wavefront is waited for), four columns a lane,
// 64 / COLS parts of the rows. The columns' sums over the rows cross the lanes once a token. 64 sequences of a token, 128 heads of 128 by 64: 90.8 us, 5.0 TB/s, the
// rate of a copy; 8 sequences of 5 drafted tokens 17.6 us, where a token's sums wait for the last one's state; one of 32 heads of 128 by 128 4.5 us, a launch and a
// chain of loads.
#pragma once

#include <type_traits>

#include "linear_attention.h"

namespace dro {

// COLS lanes side by side in a row of the state; ROWS rows of it a lane. Sums over the rows are made in the same order by four lanes of up to 16 rows and by eight of up to
// 32, whose two halves are summed apart: which of them a call takes goes by the number of its sequences, and no sequence's bits may. PLAIN: queries, keys, values and gates bf16 that can be moved 16 bytes at
// a time (everything else in its own kernel: the registers of its loads would be missing here). f32 queries, keys and values are rounded to bf16 as by chunks, so that
// a token is the same to either form, and as lx_gemm_w's BF16 math rounds its rows.
template <int COLS, int ROWS, bool PLAIN>
__global__ void __launch_bounds__(256, ROWS >= 32 ? 2 : 3) linear_step_kernel(const LinearArgs p) {
  static_assert(COLS == 4 || COLS == 8, "lanes of a row");
  static_assert(ROWS % 8 == 0, "keys are read eight at a time");
  const int lane = threadIdx.x % kWave;
  const unsigned blocks = (p.dv + 4 * COLS - 1) / (4 * COLS);
  const unsigned wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), unit = wave / blocks;
  const int s = unit / p.heads, head = unit % p.heads;
  if (s >= p.b.seqs) return;
  const MixSpan span = mix_span(p.b, s);
  if (span.first >= span.stop) return;
  const int column = wave % blocks * (4 * COLS) + lane % COLS * 4;
  const int row0 = lane / COLS * ROWS;  // of the state
  const bool mine = column < p.dv;
  const int slot = __builtin_amdgcn_readfirstlane(mix_slot(p.states, s));
  const int64_t size = static_cast<int64_t>(p.dk) * p.dv, base = (static_cast<int64_t>(slot) * p.heads + head) * size;
  const unsigned from = static_cast<unsigned>(row0 * p.dv + column);  // rows are told apart by what all lanes share

  f32x4 state[ROWS];
  const bool reads = p.states.in && slot >= 0 && !span.begins && mine;
#pragma unroll
  for (int i = 0; i < ROWS; i += 8) {
    const float* const rows = static_cast<const float*>(p.states.in) + base + static_cast<int64_t>(i) * p.dv;
#pragma unroll
    for (int j = 0; j < 8; ++j) state[i + j] = f32x4{};
    if (reads && row0 + i < p.dk) {
#pragma unroll
      for (int j = 0; j < 8; ++j) state[i + j] = *reinterpret_cast<const f32x4*>(rows + static_cast<int64_t>(j) * p.dv + from);
    }
  }

  const int k_head = head / p.group, rows = span.stop - span.first;
  const int64_t first = static_cast<int64_t>(span.row0) + span.first, k_at = static_cast<int64_t>(k_head) * p.dk + row0, v_at = static_cast<int64_t>(head) * p.dv + column;
  // What a token brings, one token ahead on its way. The gate too: asked for at an output's end, each token would wait for it.
  // Numbers are made of it where they are used: here they would be waited for.
  u32x4 key[ROWS / 8], query[ROWS / 8];
  using Four = std::conditional_t<PLAIN, u32x2, f32x4>;
  Four value, gate = {};
  auto ask = [&](int i) {
    const int64_t row = first + i;
#pragma unroll
    for (int r = 0; r < ROWS / 8; ++r) {  // places behind the state's last row are read somewhere else, and count nothing
      const int64_t at = row0 + 8 * r < p.dk ? k_at + 8 * r : static_cast<int64_t>(k_head) * p.dk;
      key[r] = load_eight_bf16(p.k, PLAIN ? LX_BF16 : p.type, PLAIN || p.wide, row * p.ld_k + at);
      query[r] = load_eight_bf16(p.q, PLAIN ? LX_BF16 : p.type, PLAIN || p.wide, row * p.ld_q + at);
    }
    const int64_t at = mine ? v_at : static_cast<int64_t>(head) * p.dv;
    if constexpr (PLAIN) {
      value = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p.v) + row * p.ld_v + at);
      if (p.gate) gate = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p.gate) + row * p.ld_gate + at);
    } else {
      value = load_four(p.v, p.type, p.wide, row * p.ld_v + at);
      if (p.gate) gate = load_four(p.gate, p.gate_type, p.wide, row * p.ld_gate + at);
#pragma unroll
      for (int j = 0; j < 4; ++j) value[j] = bf16_bits_to_f32(f32_to_bf16_bits(value[j]));
    }
  };
  auto four_of = [](const Four& x) {
    if constexpr (PLAIN) {
      const uint32_t a = x.x, b = x.y;
      return f32x4{__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u), __uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)};
    } else {
      return x;
    }
  };
  ask(0);

  // The decays, a token a lane. e^g in two parts: rounded, near 1, it is off to the same side token after token: up to 2^-25 of
  // the state for each of as many tokens as it remembers.
  const float skip = p.skip ? p.skip[head] : 0.0f;
  float fades, lefts, weights = 1.0f;
  {
    float log = 0.0f;
    if (lane < rows) decay_of(p, head_decay(p, head), decay_raw(p, first + lane, head), log, weights);
    const Fade fade = fade_of(log);
    fades = fade.high, lefts = fade.low;
  }
  auto of_token = [&](float v, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i)); };

  for (int i = 0; i < rows; ++i) {
    u32x4 ks[ROWS / 8], qs[ROWS / 8];
#pragma unroll
    for (int r = 0; r < ROWS / 8; ++r) ks[r] = row0 + 8 * r < p.dk ? key[r] : u32x4{}, qs[r] = row0 + 8 * r < p.dk ? query[r] : u32x4{};
    float fade = of_token(fades, i);
    const float left = of_token(lefts, i), weight = of_token(weights, i);
    asm("s_nop 1" : "+s"(fade));  // a lane's value read into a scalar: two cycles before the instructions below, which the compiler does not look into
    const f32x4 raw = four_of(value), z = four_of(gate), v = raw * weight;
    if (i + 1 < rows) ask(i + 1);
    constexpr int kSums = COLS == 8 && ROWS > 8 ? 2 : 1;
    f32x4 sums[kSums] = {};
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      f32x4& o = sums[r * kSums / ROWS];
      const uint32_t two_k = ks[r / 8][r % 8 / 2], two_q = qs[r / 8][r % 8 / 2];
      const float k = __uint_as_float(r % 2 ? two_k & 0xffff0000u : two_k << 16), q = __uint_as_float(r % 2 ? two_q & 0xffff0000u : two_q << 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // In place: the compiler would make the new state in registers of its own.
        const float add = __builtin_fmaf(state[r][j], left, k * v[j]);
        float in = state[r][j];
        asm("v_fma_f32 %0, %0, %1, %2" : "+v"(in) : "s"(fade), "v"(add));
        state[r][j] = in;
        o[j] = __builtin_fmaf(q, in, o[j]);
      }
      if (r % 2) __builtin_amdgcn_sched_barrier(0);  // left alone, products of all rows are made before the first sum, in registers that are not there
    }
    f32x4 o = sums[0];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (COLS == 4) o[j] += dpp_move<0x124>(o[j]);                // row_ror:4
      if (kSums > 1) o[j] += dpp_move<0x128>(sums[kSums - 1][j]);  // as that adds them: the first rows' half and the last ones', then those between
      o[j] += dpp_move<0x128>(o[j]);                               // row_ror:8
      float a, b;
      swap_halves<true>(o[j], a, b);
      const float half = a + b;
      swap_halves<false>(half, a, b);
      o[j] = (a + b) * p.scale;
    }
    if (mine && lane < COLS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = __builtin_fmaf(skip, raw[j], o[j]);
        if (p.gate) o[j] *= quick_silu(z[j]);
      }
      store_four(p.out, p.out_type, p.wide, (first + i) * p.ld_out + v_at, o);
    }
  }
  if (!p.states.out || slot < 0 || !mine) return;
#pragma unroll
  for (int i = 0; i < ROWS; i += 8) {
    float* const rows = static_cast<float*>(p.states.out) + base + static_cast<int64_t>(i) * p.dv;
    if (row0 + i < p.dk) {
#pragma unroll
      for (int j = 0; j < 8; ++j) *reinterpret_cast<f32x4*>(rows + static_cast<int64_t>(j) * p.dv + from) = state[i + j];
    }
  }
}

}  // namespace dro
