// lx_linear_attention by chunks of 64 tokens, on the matrix cores.
//
// With G_i the sum of the decays' logarithms of a chunk up to token i, b_j the weight of an update and S the state in front of the chunk
//   out_i = scale (e^{G_i} S^T q_i + sum_{j <= i} (q_i . k_j) e^{G_i - G_j} b_j v_j)
//   S    <- e^{G_63} S + sum_j k_j (e^{G_63 - G_j} b_j v_j)^T
// Every exponent is a difference of sums at most 0, formed from sums in 64 bits (as two f32): nothing overflows, and near tokens lose nothing where the sums
// are large. What is rounded to go into a product (weights, scaled values, the state) goes in as two bf16, a value and what its
// rounding left: with one, a state would be right to 2^-9 only, and results carry its error on from chunk to chunk.
//
// A wavefront owns 32 columns of a head's state, all its rows, in registers, for the whole of a sequence's part. Its layout is what
// makes that work: v_mfma_f32_32x32x16 leaves a lane with four neighbouring rows, and four others 8 further, of its column. Rows and columns are given to
// the instruction in the order (0-3, 8-11, 4-7, 12-15) of every 16 (the transposing reads of LDS take any four neighbours from anywhere), and
// so a lane's eight values are neighbours: the state is the next product's operand as it lies, an output's eight values are one
// store. Products are transposed, out^T = S^T Q^T + V^T P^T, so that a row's factors are a lane's own.
//
// Queries, keys and values of a chunk stand in LDS, read along rows (16 bytes a lane) and across (ds_read_tr16), units of 16 bytes swizzled so that both
// fall on all banks. The weights P of a head are made once by its wavefronts, 32 x 32 tiles on and below the diagonal, and shared through
// LDS. Heads that read the same keys go into one workgroup by twos where they are 64 columns or fewer. The next chunk is on its way in
// registers meanwhile.
//
// Long sequences are cut into parts where there are too few workgroups: a first kernel leaves each part's own sum (keys and values
// only), a second one runs through them and leaves the state in front of every part, and this one starts from there.
#pragma once

#include "linear_attention.h"

namespace dro {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kChunk = 64;

struct ChunkArgs {
  LinearArgs l;
  int size;         // rows of a part, whole chunks
  int single;       // no sequence has more than one part
  int64_t numbers;  // of parts that the launch counts to
  int across;       // workgroups of a part and key head
  float* sums;      // [2 (T / size)] states [heads, dk, dv]: parts' sums, then the states in front of them
  double* logs;     // [2 (T / size), heads] logarithms (base 2) of what the parts leave of what was in front of them
};

// Where 16-byte unit `unit` of row `row` lies in a tile of rows of `kPitch` bytes (128, 256 or 512): its place in the row is turned by the row's low bits, so
// that sixteen rows' units of one place fall on all banks, and so do four neighbouring rows' of four neighbouring places.
template <int kPitch>
__host__ __device__ constexpr int turn_of(int row) {
  return kPitch == 128 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3);
}
template <int kPitch>
__device__ __forceinline__ int tile_place(int row, int unit) {
  return row * kPitch + 16 * (unit ^ turn_of<kPitch>(row));
}
// The same from the place of a row and unit that share no bits with `row` and `unit`: constants leave an exclusive or and an offset of an
// instruction (with every address by itself, 64 of them live through the loop in registers that are not there).
template <int kPitch>
__device__ __forceinline__ int tile_place(int from, int row, int unit) {
  return (from ^ 16 * (unit ^ turn_of<kPitch>(row))) + row * kPitch;
}

__device__ __forceinline__ bf16x8 eight_at(const uint8_t* lds, int at) { return *reinterpret_cast<const bf16x8*>(lds + at); }

// The operand of rows across a tile: eight rows 16 s + 8 h .. + 7 of 32 columns, in the order (0-3, 8-11, 4-7, 12-15) of every 16. A lane asks for four
// neighbouring columns of a row and gets four rows of a column; here is where its four lie, of columns 0 .. 31 and s = 0, for
// either half of the eight rows.
template <int kPitch>
__device__ __forceinline__ int across_place(int column, int half) {
  const int lane = threadIdx.x % kWave, m = lane % 16, h = lane / 32;
  const int from = column + lane / 16 % 2 * 16 + (m % 2 * 8 | m % 4 / 2 * 4);
  return tile_place<kPitch>(8 * h + 4 * half + m / 4, from / 8) + from % 8 * 2;
}
__device__ __forceinline__ bf16x8 across(const uint8_t* lds, int at0, int at1) {
  union {
    s16x4 half[2];
    bf16x8 whole;
  } r;
  r.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at0));
  r.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at1));
  return r.whole;
}

// Eight f32 as bf16, and what their rounding leaves as bf16.
__device__ __forceinline__ void split_eight(const float (&v)[8], bf16x8& high, bf16x8& low) {
  u32x4 a, b;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t two = __builtin_bit_cast(uint32_t, pack_bf16(v[2 * j], v[2 * j + 1]));
    a[j] = two;
    b[j] = __builtin_bit_cast(uint32_t, pack_bf16(v[2 * j] - __uint_as_float(two << 16), v[2 * j + 1] - __uint_as_float(two & 0xffff0000u)));
  }
  high = __builtin_bit_cast(bf16x8, a);
  low = __builtin_bit_cast(bf16x8, b);
}

// A sum over the wavefront's lanes up to and with each one, in 64 bits.
template <int CTRL, int ROWS>
__device__ __forceinline__ double scan_step(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xf, true);
  const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xf, true);
  return v + __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
}
__device__ __forceinline__ double wave_scan(double v) {
  v = scan_step<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v = scan_step<0x112, 0xf>(v);
  v = scan_step<0x114, 0xf>(v);
  v = scan_step<0x118, 0xf>(v);
  v = scan_step<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  return scan_step<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
}

// What of a state is left by a decay: x e^log, or x + x (e^log - 1) where little fades, whose rounding does not go to one side.
struct Fade {
  float factor;
  bool slow;
};
__device__ __forceinline__ Fade fade_of(double log2_of) {
  const float log = static_cast<float>(log2_of * 0.69314718055994530942);
  const bool slow = log > -0.5f;
  return {slow ? expm1f(log) : expf(log), slow};
}

// The numbers of a chunk's tokens.
struct Tokens {
  float g_high[kChunk], g_low[kChunk];  // G_i, base 2
  float h_high[kChunk], h_low[kChunk];  // G_j - log2(b_j)
  float update[kChunk];                 // e^{G_63 - G_j} b_j
  float seen[kChunk];                   // e^{G_i}
  double whole, none;                   // G_63; whole 16 bytes
};

template <int DK, int TW, int TEAMS>
struct ChunkTiles {
  static constexpr int kWaves = TW * TEAMS, kThreads = kWave * kWaves;
  static constexpr int kColumns = 32 * kWaves;
  static constexpr int kKeyPitch = 2 * DK, kValuePitch = 2 * kColumns;
  static constexpr int kKeyBytes = kChunk * kKeyPitch, kValueBytes = kChunk * kValuePitch;
  static constexpr int kBlock = 32 * 64;             // a 32 x 32 tile of weights, bf16
  static constexpr int kWeightBytes = 2 * 3 * kBlock;  // of a head: tiles (0, 0), (0, 1), (1, 1) as values, then what their rounding left
  static constexpr int kKeys = 0, kValues = kKeys + kKeyBytes, kTokens = kValues + kValueBytes;
  static constexpr int kQueries = kTokens + 2 * TEAMS * static_cast<int>(sizeof(Tokens)), kWeights = kQueries + kKeyBytes;
  static constexpr int kSumBytes = kQueries, kBytes = kWeights + TEAMS * kWeightBytes;
};

// OUT: outputs and states; otherwise a part's sum of a long sequence only.
template <int DK, int TW, int TEAMS, bool OUT>
__global__ void __launch_bounds__(kWave * TW * TEAMS, DK == 256 ? 1 : 2) linear_chunk_kernel(const ChunkArgs c) {
  using L = ChunkTiles<DK, TW, TEAMS>;
  extern __shared__ __attribute__((aligned(256))) uint8_t lds[];
  const LinearArgs& p = c.l;
  // Workgroups that read the same keys follow one another on one die.
  const int64_t turn = blockIdx.x / 8, unit = turn / c.across * 8 + blockIdx.x % 8;
  const int beside = static_cast<int>(turn % c.across), k_head = static_cast<int>(unit % p.k_heads);
  const int64_t number = unit / p.k_heads;
  if (number >= c.numbers) return;
  int s, j;
  if (OUT ? !mix_find(p.b, MixPieces{c.size, c.single}, number, s, j) : !mix_find_long(p.b, c.size, number, s, j)) return;
  MixSpan span = mix_span(p.b, s);
  span.row0 = __builtin_amdgcn_readfirstlane(span.row0), span.first = __builtin_amdgcn_readfirstlane(span.first);
  span.stop = __builtin_amdgcn_readfirstlane(span.stop), span.begins = __builtin_amdgcn_readfirstlane(span.begins);
  const int begin = max(span.first, j * c.size), end = min(span.stop, (j + 1) * c.size);
  const bool split = span.stop > c.size;
  if (begin >= end || (!OUT && (!split || end == span.stop))) return;
  // A sequence's part has a place of its own: those of more than one part are more than `size` rows each.
  const int64_t place = 2 * static_cast<int64_t>(span.row0 / c.size) + j;

  const int lane = threadIdx.x % kWave, h = lane / 32, n = lane % 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), team = wave / TW, mate = wave % TW;
  const int blocks = (p.dv + 32 * TW - 1) / (32 * TW);  // TEAMS > 1: one
  const int head0 = k_head * p.group + (TEAMS > 1 ? beside * TEAMS : beside / blocks);
  const int head_end = (k_head + 1) * p.group;
  const int column0 = TEAMS > 1 ? 0 : beside % blocks * 32 * TW;
  const int head = min(head0 + team, head_end - 1);
  const bool idle = head0 + team >= head_end;
  const int column = column0 + 32 * mate + (n / 16 * 16 + (n % 4 | n / 4 % 2 * 8 | n / 8 % 2 * 4));  // the lane's of the state
  const int64_t first_row = span.row0 + begin;
  const int rows = end - begin, chunks = (rows + kChunk - 1) / kChunk;

  Tokens* const tokens = reinterpret_cast<Tokens*>(lds + L::kTokens) + 2 * team;
  // Where the lane's first reads lie: row n of the keys (and queries), the columns of the keys and of its values, row n of its values and of the weights.
  const int key_row = tile_place<L::kKeyPitch>(n, h);
  const int key_column[2] = {across_place<L::kKeyPitch>(0, 0), across_place<L::kKeyPitch>(0, 1)};
  const int value_column[2] = {L::kValues + across_place<L::kValuePitch>(32 * wave, 0), L::kValues + across_place<L::kValuePitch>(32 * wave, 1)};
  const int value_row = tile_place<L::kValuePitch>(n, 4 * wave + h);
  const int weight_row = team * L::kWeightBytes + 64 * n + 16 * (n >> 2 & 3);
  auto read_keys = [&](int row, int k) { return eight_at(lds, L::kKeys + tile_place<L::kKeyPitch>(key_row, row, 2 * k)); };
  auto read_queries = [&](int row, int k) { return eight_at(lds, L::kQueries + tile_place<L::kKeyPitch>(key_row, row, 2 * k)); };
  auto keys_across = [&](int x, int k) {  // keys' values 32 x .. of tokens 16 k ..
    return across(lds, L::kKeys + tile_place<L::kKeyPitch>(key_column[0], 16 * k, 4 * x), L::kKeys + tile_place<L::kKeyPitch>(key_column[1], 16 * k, 4 * x));
  };
  auto values_across = [&](int k) { return across(lds, value_column[0] + 16 * k * L::kValuePitch, value_column[1] + 16 * k * L::kValuePitch); };

  // ---- the next chunk on its way --------------------------------------------------------------------------------------
  constexpr int kKeyLoads = kChunk * DK / 8 / L::kThreads, kValueLoads = kChunk * L::kColumns / 8 / L::kThreads;
  u32x4 next_k[kKeyLoads], next_q[OUT ? kKeyLoads : 1], next_v[kValueLoads];
  const bool whole_tiles = p.dk == DK && head0 + TEAMS <= head_end && column0 + 32 * TW <= p.dv;  // no column is nobody's
  const bool plain = p.type == LX_BF16 && p.wide && whole_tiles;
  // Where a thread's first loads of a whole chunk lie, from the chunk's first row on; the others follow rows further.
  constexpr int kKeyStep = L::kThreads / (DK / 8), kValueStep = L::kThreads / (L::kColumns / 8);
  const int my_key = threadIdx.x % (DK / 8) * 8, my_value = threadIdx.x % (L::kColumns / 8);
  const unsigned k_from = static_cast<unsigned>(threadIdx.x / (DK / 8) * p.ld_k + k_head * p.dk + my_key);
  const unsigned q_from = static_cast<unsigned>(threadIdx.x / (DK / 8) * p.ld_q + k_head * p.dk + my_key);
  const unsigned v_from = static_cast<unsigned>(threadIdx.x / (L::kColumns / 8) * p.ld_v + (head0 + my_value / (4 * TW)) * p.dv + column0 + my_value % (4 * TW) * 8);
  auto ask = [&](int chunk) {
    const int64_t row0 = first_row + static_cast<int64_t>(chunk) * kChunk;
    const int last = min(kChunk, rows - chunk * kChunk) - 1;
    if (plain && last == kChunk - 1) {
      auto at = [](const void* x, int64_t i, unsigned from) { return *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(x) + i + from); };
#pragma unroll
      for (int e = 0; e < kKeyLoads; ++e) {
        next_k[e] = at(p.k, (row0 + e * kKeyStep) * p.ld_k, k_from);
        if constexpr (OUT) next_q[e] = at(p.q, (row0 + e * kKeyStep) * p.ld_q, q_from);
      }
#pragma unroll
      for (int e = 0; e < kValueLoads; ++e) next_v[e] = at(p.v, (row0 + e * kValueStep) * p.ld_v, v_from);
      return;
    }
#pragma unroll
    for (int e = 0; e < kKeyLoads; ++e) {
      const int row = min(static_cast<int>(threadIdx.x) / (DK / 8) + e * kKeyStep, last);
      const int64_t from = static_cast<int64_t>(k_head) * p.dk + (my_key < p.dk ? my_key : 0);
      next_k[e] = load_eight_bf16(p.k, p.type, p.wide, (row0 + row) * p.ld_k + from);
      if constexpr (OUT) next_q[e] = load_eight_bf16(p.q, p.type, p.wide, (row0 + row) * p.ld_q + from);
    }
#pragma unroll
    for (int e = 0; e < kValueLoads; ++e) {
      const int row = min(static_cast<int>(threadIdx.x) / (L::kColumns / 8) + e * kValueStep, last);
      const int of = min(head0 + my_value / (4 * TW), head_end - 1), d = column0 + my_value % (4 * TW) * 8;
      next_v[e] = load_eight_bf16(p.v, p.type, p.wide, (row0 + row) * p.ld_v + static_cast<int64_t>(of) * p.dv + (d < p.dv ? d : 0));
    }
  };
  const int key_place = tile_place<L::kKeyPitch>(threadIdx.x / (DK / 8), my_key / 8);
  const int value_place = tile_place<L::kValuePitch>(threadIdx.x / (L::kColumns / 8), my_value);
  auto put = [&](int chunk) {
    const int m = min(kChunk, rows - chunk * kChunk);
    auto all = [&](auto in) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < kKeyLoads; ++e) {
        const bool there = in(static_cast<int>(threadIdx.x) / (DK / 8) + e * kKeyStep < m && my_key < p.dk);
        const int at = tile_place<L::kKeyPitch>(key_place, e * kKeyStep, 0);
        *reinterpret_cast<u32x4*>(lds + L::kKeys + at) = there ? next_k[e] : u32x4{};
        if constexpr (OUT) *reinterpret_cast<u32x4*>(lds + L::kQueries + at) = there ? next_q[e] : u32x4{};
      }
#pragma unroll
      for (int e = 0; e < kValueLoads; ++e) {
        const bool there = in(static_cast<int>(threadIdx.x) / (L::kColumns / 8) + e * kValueStep < m && head0 + my_value / (4 * TW) < head_end &&
                              column0 + my_value % (4 * TW) * 8 < p.dv);
        *reinterpret_cast<u32x4*>(lds + L::kValues + tile_place<L::kValuePitch>(value_place, e * kValueStep, 0)) = there ? next_v[e] : u32x4{};
      }
    };
    if (m == kChunk && whole_tiles) all([](bool) { return true; });
    else all([](bool in) { return in; });
  };
  // The decay's numbers, a token a lane: asked for two chunks ahead, made ready one ahead, by the team's last wavefront.
  const bool counts = mate == TW - 1;
  float next_log = 0.0f, next_weight = 1.0f;
  auto ask_decay = [&](int chunk) {
    next_log = 0.0f, next_weight = 1.0f;
    if (chunk * kChunk + lane < rows) decay_of(p, first_row + static_cast<int64_t>(chunk) * kChunk + lane, head, next_log, next_weight);
  };
  auto put_decay = [&](int chunk) {
    Tokens& t = tokens[chunk % 2];
    const double g = wave_scan(static_cast<double>(next_log) * 1.44269504088896340736);
    const float b = next_weight == 1.0f ? 0.0f : fminf(fmaxf(__builtin_amdgcn_logf(next_weight), -1e5f), 1e5f);
    const double more = g - static_cast<double>(next_weight != next_weight ? next_weight : b);
    const uint64_t u = __builtin_bit_cast(uint64_t, g);
    const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(u), kWave - 1), high = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), kWave - 1);
    const double whole = __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
    t.g_high[lane] = static_cast<float>(g);
    t.g_low[lane] = static_cast<float>(g - static_cast<double>(static_cast<float>(g)));
    t.h_high[lane] = static_cast<float>(more);
    t.h_low[lane] = static_cast<float>(more - static_cast<double>(static_cast<float>(more)));
    t.update[lane] = __builtin_amdgcn_exp2f(static_cast<float>(whole - more));
    t.seen[lane] = __builtin_amdgcn_exp2f(static_cast<float>(g));
    if (lane == 0) t.whole = whole;
  };

  // ---- the state ------------------------------------------------------------------------------------------------------
  f32x16 state[DK / 32] = {};
  const int slot = __builtin_amdgcn_readfirstlane(mix_slot(p.states, s));
  const bool mine = column < p.dv && !idle;
  const int64_t state_size = static_cast<int64_t>(p.dk) * p.dv;
  const unsigned state_from = static_cast<unsigned>(8 * h * p.dv + column);
  auto each_state = [&](float* base, auto use) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < DK / 32; ++t)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        if (!mine || 32 * t + 16 * a + 8 * h >= p.dk) continue;
        float* const row = base + static_cast<int64_t>(32 * t + 16 * a) * p.dv;
#pragma unroll
        for (int r = 0; r < 8; ++r) use((row + static_cast<int64_t>(r) * p.dv)[state_from], t, 8 * a + r);
      }
  };
  if constexpr (OUT) {
    float* from = nullptr;
    if (split) from = c.sums + (place * p.heads + head) * state_size;
    else if (p.states.in && slot >= 0 && !span.begins) from = const_cast<float*>(static_cast<const float*>(p.states.in)) + (static_cast<int64_t>(slot) * p.heads + head) * state_size;
    if (from) each_state(from, [&](float& x, int t, int r) { state[t][r] = x; });
  }
  const float skip = p.skip ? p.skip[head] : 0.0f;
  double part_log = 0.0;

  if (counts) {
    ask_decay(0);
    put_decay(0);
    ask_decay(1);
  }
  ask(0);
  put(0);
  __syncthreads();
  for (int chunk = 0; chunk < chunks; ++chunk) {
    const Tokens& t = tokens[chunk % 2];
    const int m = min(kChunk, rows - chunk * kChunk);
    const bool more = chunk + 1 < chunks, two = m > 32;
    if (more) ask(chunk + 1);
    __builtin_amdgcn_sched_barrier(0);
    f32x16 out[2] = {};
    if constexpr (OUT) {
      // Weights: tile `block` has tokens 32 jb .. of rows 32 ib ..
      auto weigh = [&](int block) {
        const int jb = block == 2, ib = block > 0;
        f32x16 w = {};
#pragma unroll
        for (int k = 0; k < DK / 16; ++k)
          w = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_keys(32 * jb, k), read_queries(32 * ib, k), w, 0, 0, 0);
        const float g_high = t.g_high[32 * ib + n], g_low = t.g_low[32 * ib + n];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int token = 8 * g + 4 * h;  // of the tile's, and the three behind it
          const f32x4 h_high = *reinterpret_cast<const f32x4*>(t.h_high + 32 * jb + token), h_low = *reinterpret_cast<const f32x4*>(t.h_low + 32 * jb + token);
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = w[4 * g + e] * __builtin_amdgcn_exp2f((g_high - h_high[e]) + (g_low - h_low[e]));
            if (jb == ib) v[e] = token + e <= n ? v[e] : 0.0f;
          }
          const uint32_t a = __builtin_bit_cast(uint32_t, pack_bf16(v[0], v[1])), b = __builtin_bit_cast(uint32_t, pack_bf16(v[2], v[3]));
          const u32x2 left = {__builtin_bit_cast(uint32_t, pack_bf16(v[0] - __uint_as_float(a << 16), v[1] - __uint_as_float(a & 0xffff0000u))),
                              __builtin_bit_cast(uint32_t, pack_bf16(v[2] - __uint_as_float(b << 16), v[3] - __uint_as_float(b & 0xffff0000u)))};
          uint8_t* const at = lds + L::kWeights + block * L::kBlock + (weight_row ^ 16 * g) + 8 * h;
          *reinterpret_cast<u32x2*>(at) = u32x2{a, b};
          *reinterpret_cast<u32x2*>(at + 3 * L::kBlock) = left;
        }
      };
      if constexpr (TW == 2) {
        if (mate == 0) {
          weigh(0);
          if (two) weigh(1);
        } else if (two) {
          weigh(2);
        }
      } else if (mate < 3 && (two || mate == 0)) {
        weigh(mate);
      }
      __builtin_amdgcn_sched_barrier(0);
      // What the rows see of the state: queries read one step ahead.
      bf16x8 q[2][2];
      auto read = [&](int k) {
        q[k % 2][0] = read_queries(0, k);
        q[k % 2][1] = read_queries(32, k);
      };
      read(0);
#pragma unroll
      for (int k = 0; k < DK / 16; ++k) {
        if (k + 1 < DK / 16) read(k + 1);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = state[k / 2][k % 2 * 8 + e];
        bf16x8 high, low;
        split_eight(v, high, low);
        out[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(high, q[k % 2][0], out[0], 0, 0, 0);
        out[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(high, q[k % 2][1], out[1], 0, 0, 0);
        out[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(low, q[k % 2][0], out[0], 0, 0, 0);
        out[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(low, q[k % 2][1], out[1], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) out[i] *= t.seen[32 * i + n];
    }
    if (counts && more) {
      put_decay(chunk + 1);
      ask_decay(chunk + 2);
    }
    if constexpr (OUT) __syncthreads();

    // Gates of the usual type are asked for here.
    const bool gates = OUT && p.gate && p.wide && p.gate_type == LX_BF16;
    u32x4 gate[2][2];
    if (gates) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int d = column0 + 32 * mate + 16 * a + 8 * h;
          const int64_t row = first_row + static_cast<int64_t>(chunk) * kChunk + min(32 * i + n, m - 1);
          gate[i][a] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.gate) + row * p.ld_gate + static_cast<int64_t>(head) * p.dv + (d < p.dv ? d : 0));
        }
    }
    bf16x8 v[kChunk / 16];
#pragma unroll
    for (int k = 0; k < kChunk / 16; ++k) v[k] = values_across(k);
    if constexpr (OUT) {
      auto weight_unit = [&](int block, int k, int low) {  // of row n, tokens 16 k + 8 h .. of the tile
        return eight_at(lds, L::kWeights + (block + 3 * low) * L::kBlock + ((weight_row ^ 16 * h) ^ 32 * k));
      };
      // A weight of nothing times an infinity or a NaN of a later token is no number: those are taken out of the product, and what rows behind
      // them see of them is added by itself.
      float odd = 0.0f;
#pragma unroll
      for (int k = 0; k < kChunk / 16; ++k) {
        const u32x4 raw = __builtin_bit_cast(u32x4, v[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd = __builtin_amdgcn_fdot2_f32_bf16(as_bf16x2(raw[e]), as_bf16x2(0), odd, false);
      }
      const bool some_odd = __any(odd != odd);
      if (some_odd) {
#pragma unroll
        for (int k = 0; k < kChunk / 16; ++k) {
          u32x4 raw = __builtin_bit_cast(u32x4, v[k]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if ((raw[e] & 0x7f80u) == 0x7f80u) raw[e] &= 0xffff0000u;
            if ((raw[e] & 0x7f800000u) == 0x7f800000u) raw[e] &= 0xffffu;
          }
          v[k] = __builtin_bit_cast(bf16x8, raw);
        }
        for (int token = 0; token < m; ++token) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (token > 32 * i + n || 32 * i >= m) continue;
            const int in = token % 32;
            const uint8_t* const at = lds + L::kWeights + (i + token / 32) * L::kBlock + (weight_row ^ 16 * (in / 8)) + in % 8 * 2;
            const float weight = bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(at)) + bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(at + 3 * L::kBlock));
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              const u32x4 eight = __builtin_bit_cast(u32x4, eight_at(lds, L::kValues + tile_place<L::kValuePitch>(token, 4 * wave + 2 * a + h)));
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t pair = eight[e / 2], value = e % 2 ? pair & 0xffff0000u : pair << 16;
                if ((value & 0x7f800000u) == 0x7f800000u) out[i][8 * a + e] += weight * __uint_as_float(value);
              }
            }
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < kChunk / 16; ++k) {
#pragma unroll
        for (int low = 0; low < 2; ++low) {
          if (k < 2) out[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[k], weight_unit(0, k, low), out[0], 0, 0, 0);
          if (two) out[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[k], weight_unit(1 + k / 2, k % 2, low), out[1], 0, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (some_odd) {
#pragma unroll
        for (int k = 0; k < kChunk / 16; ++k) v[k] = values_across(k);
      }
    }
    // The state behind the chunk.
    const double whole = t.whole;
    const Fade fade = fade_of(whole);
    if (__builtin_amdgcn_readfirstlane(fade.slow)) {
#pragma unroll
      for (int x = 0; x < DK / 32; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) state[x][r] = __builtin_fmaf(state[x][r], fade.factor, state[x][r]);
    } else {
#pragma unroll
      for (int x = 0; x < DK / 32; ++x) state[x] *= fade.factor;
    }
    part_log += whole;
#pragma unroll
    for (int k = 0; k < kChunk / 16; ++k) {
      const u32x4 raw = __builtin_bit_cast(u32x4, v[k]);
      const f32x4 w0 = *reinterpret_cast<const f32x4*>(t.update + 16 * k + 8 * h), w1 = *reinterpret_cast<const f32x4*>(t.update + 16 * k + 8 * h + 4);
      float scaled[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t pair = raw[e / 2];
        scaled[e] = __uint_as_float(e % 2 ? pair & 0xffff0000u : pair << 16) * (e < 4 ? w0[e % 4] : w1[e % 4]);
      }
      bf16x8 high, low;
      split_eight(scaled, high, low);
#pragma unroll
      for (int x = 0; x < DK / 32; ++x) {
        const bf16x8 key = keys_across(x, k);
        state[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(key, high, state[x], 0, 0, 0);
        state[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(key, low, state[x], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (OUT) {
      if (!idle) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (32 * i + n >= m) continue;
          const int64_t row = first_row + static_cast<int64_t>(chunk) * kChunk + 32 * i + n;
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const int d = column0 + 32 * mate + 16 * a + 8 * h;
            if (d >= p.dv) continue;
            const u32x4 eight = __builtin_bit_cast(u32x4, eight_at(lds, L::kValues + tile_place<L::kValuePitch>(value_row, 32 * i, 2 * a)));
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t pair = eight[e / 2];
              o[e] = out[i][8 * a + e] * p.scale;
              if (p.skip) o[e] = __builtin_fmaf(skip, __uint_as_float(e % 2 ? pair & 0xffff0000u : pair << 16), o[e]);
            }
            const int64_t at = static_cast<int64_t>(head) * p.dv + d;
            if (gates) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t pair = gate[i][a][e / 2];
                o[e] *= quick_silu(__uint_as_float(e % 2 ? pair & 0xffff0000u : pair << 16));
              }
            } else if (p.gate) {
#pragma unroll
              for (int e = 0; e < 8; e += 4) {
                const f32x4 z = load_four(p.gate, p.gate_type, p.wide, row * p.ld_gate + at + e);
#pragma unroll
                for (int f = 0; f < 4; ++f) o[e + f] *= quick_silu(z[f]);
              }
            }
            if (p.wide && p.out_type == LX_BF16) {
              const u32x4 packed = {__builtin_bit_cast(uint32_t, pack_bf16(o[0], o[1])), __builtin_bit_cast(uint32_t, pack_bf16(o[2], o[3])),
                                    __builtin_bit_cast(uint32_t, pack_bf16(o[4], o[5])), __builtin_bit_cast(uint32_t, pack_bf16(o[6], o[7]))};
              *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.out) + row * p.ld_out + at) = packed;
            } else {
              store_four(p.out, p.out_type, p.wide, row * p.ld_out + at, f32x4{o[0], o[1], o[2], o[3]});
              store_four(p.out, p.out_type, p.wide, row * p.ld_out + at + 4, f32x4{o[4], o[5], o[6], o[7]});
            }
          }
        }
      }
    }
    __syncthreads();
    if (more) {
      put(chunk + 1);
      __syncthreads();
    }
  }

  float* to = nullptr;
  if constexpr (OUT) {
    if (p.states.out && slot >= 0 && end == span.stop) to = static_cast<float*>(p.states.out) + (static_cast<int64_t>(slot) * p.heads + head) * state_size;
  } else {
    to = c.sums + (place * p.heads + head) * state_size;
    if (!idle && mate == 0 && lane == 0 && column0 == 0) c.logs[place * p.heads + head] = part_log;
  }
  if (to) each_state(to, [&](float& x, int t, int r) { x = state[t][r]; });
}

// The states in front of a long sequence's parts, where their sums were: four values a thread, all parts in order.
__global__ void __launch_bounds__(256) linear_parts_kernel(const ChunkArgs c) {
  const LinearArgs& p = c.l;
  const int64_t state_size = static_cast<int64_t>(p.dk) * p.dv, fours = p.heads * state_size / 4;
  const int64_t groups = (fours + 255) / 256;
  int s, j;
  if (!mix_find_long(p.b, c.size, 2 * (blockIdx.x / groups), s, j) || j != 0) return;
  const MixSpan span = mix_span(p.b, s);
  if (span.stop <= c.size) return;
  const int64_t i = blockIdx.x % groups * 256 + threadIdx.x;
  if (i >= fours) return;
  const int head = static_cast<int>(4 * i / state_size), parts = (span.stop + c.size - 1) / c.size;
  const int64_t place = 2 * static_cast<int64_t>(span.row0 / c.size);
  const int slot = mix_slot(p.states, s);
  f32x4 state = {};
  if (p.states.in && slot >= 0 && !span.begins) state = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p.states.in) + static_cast<int64_t>(slot) * p.heads * state_size + 4 * i);
  const int skipped = min(span.first / c.size, parts);  // parts in front of position 0 have left no sum
  for (int k = skipped; k < parts; ++k) {
    f32x4* const at = reinterpret_cast<f32x4*>(c.sums + (place + k) * p.heads * state_size + 4 * i);
    const f32x4 before = state;
    if (k + 1 < parts) {
      const f32x4 sum = *at;
      const Fade fade = fade_of(c.logs[(place + k) * p.heads + head]);
#pragma unroll
      for (int e = 0; e < 4; ++e) state[e] = (fade.slow ? __builtin_fmaf(state[e], fade.factor, state[e]) : state[e] * fade.factor) + sum[e];
    }
    *at = before;
  }
}

}  // namespace dro
