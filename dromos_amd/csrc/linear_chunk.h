// lx_linear_attention by chunks of 64 tokens, on the matrix cores.
//
// With G_i the sum of the decays' logarithms of a chunk up to token i, b_j the weight of an update and S the state in front of the chunk
//   out_i = scale (e^{G_i} S^T q_i + sum_{j <= i} (q_i . k_j) e^{G_i - G_j} b_j v_j)
//   S    <- e^{G_63} S + sum_j k_j (e^{G_63 - G_j} b_j v_j)^T
// Every exponent is a difference of sums at most 0, formed from sums in 64 bits (as two f32 each): nothing overflows, and near tokens lose nothing where the sums
// are large. What is rounded to go into a product goes in as bf16 terms, a value, what its rounding left, and so on: three of the values that a state is made of
// (24 bits; with two, states were right to 2.6e-6, with one to 2^-9, and what a state has lost goes on from chunk to chunk), and of the state and the weights where results
// are f32; two of those, 2^-17 of them, where results are rounded to bf16, 2^-8 of them, in any case (one result in 400 to 7000 is another one, mostly its neighbour; three terms there
// too: 4096 tokens 190 us in place of 135, 16384 tokens 146 and 137, the wide prompts 139 and 127).
//
// A wavefront owns 32 columns of a head's state in registers, all rows or (of more than 128 keys) one half of them, for the whole of a sequence's part. Its layout is what
// makes that work: v_mfma_f32_32x32x16 leaves a lane with four neighbouring rows, and four others 8 further, of its column. Rows and columns are given to
// the instruction in the order (0-3, 8-11, 4-7, 12-15) of every 16 (the transposing reads of LDS take any four neighbours from anywhere), and
// so a lane's eight values are neighbours: the state is the next product's operand as it lies, an output's eight values are one
// store. Products are transposed, out^T = S^T Q^T + V^T P^T, so that a row's factors are a lane's own.
// Halves give each other what they have for the other's 32 tokens through LDS (a wavefront with all 256 rows leaves a SIMD to itself: eight prompts of up to 2048
// of 8 heads of 256 by 256, with two terms throughout and a kernel between sums and outputs, 168 us, 150 by halves).
//
// Queries, keys and values of a chunk stand in LDS, read along rows (16 bytes a lane) and across (ds_read_tr16), units of 16 bytes swizzled so that both
// fall on all banks. The weights P of a head are made once by its wavefronts, 32 x 32 tiles on and below the diagonal, and shared through
// LDS. Heads that read the same keys go into one workgroup by twos where they are 64 columns or fewer. The next chunk is on its way in
// registers meanwhile.
//
// Long sequences are cut into parts where there are too few workgroups: a first kernel leaves each part's own sum (keys and values
// only), and this one starts from the sums in front of its part; where there are many, a kernel in between runs through them and leaves the state in front of every
// part.
//
// What bounds it: a wavefront's vector arithmetic (terms, exponentials, skips, gates: 1370 instructions a chunk) and its products (104, 3300 cycles), one after
// another in each of the two wavefronts that a SIMD has registers for. 4096 tokens of 128 heads of 128 by 64, 16 to a key head: 128 - 135 us (devices differ; sums 38,
// outputs 105), 16384 of 16 heads of 128 by 128 133 - 137 us (42, 16 in between, 82), eight prompts of up to 2048 of 8 heads of 256 by 256 126 us (43, 93).
#pragma once

#include <type_traits>

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
  int sums_only;    // sequences have few parts at most: nothing runs through them in between
  float* sums;      // [2 (T / size), heads] states as wavefronts hold them: parts' sums, and what a sequence goes on from or the states in front of the parts
  double* logs;     // [2 (T / size), heads] logarithms of what the parts leave of what was in front of them
};

// A state as the wavefronts' registers hold it, for the parts of long sequences: columns by 32s, rows by 32s, then four registers by four of all
// lanes (as rows and columns, a lane's values would be 64 loads of four bytes: 4 us of a part's 45).
__host__ __device__ __forceinline__ int64_t part_values(int dk, int dv) { return static_cast<int64_t>(dk <= 64 ? 64 : dk <= 128 ? 128 : 256) * ((dv + 31) / 32 * 32); }
// Lane n's column of 32.
__device__ __forceinline__ int lane_column(int n) { return n / 16 * 16 + (n % 4 | n / 4 % 2 * 8 | n / 8 % 2 * 4); }

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
// neighbouring columns of a row and gets four rows of a column; here is where its four lie, of columns 0 .. 31 and s = 0, for the first four of
// the eight rows.
template <int kPitch>
__device__ __forceinline__ int across_place(int column) {
  const int lane = threadIdx.x % kWave, m = lane % 16, h = lane / 32;
  const int from = column + lane / 16 % 2 * 16 + (m % 2 * 8 | m % 4 / 2 * 4);
  return tile_place<kPitch>(8 * h + m / 4, from / 8) + from % 8 * 2;
}
// The operand of tile `at` (a whole 256 bytes), from that place, of rows 16 s .. and columns 8 unit .. further.
template <int kPitch>
__device__ __forceinline__ bf16x8 across(const uint8_t* lds, int at, int from, int s, int unit) {
  const int at0 = at + tile_place<kPitch>(from, 16 * s, unit), at1 = at + tile_place<kPitch>(from, 16 * s + 4, unit);
  union {
    s16x4 half[2];
    bf16x8 whole;
  } r;
  r.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at0));
  r.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at1));
  return r.whole;
}

// Two f32 as bf16, what their rounding leaves as bf16, and so on, TERMS of them. Values that are not used again: taken off by one instruction each, in
// place (a dot product with minus one and nothing; an infinity or a NaN of one is one of the other's rest too, which is summed with it). KEPT: by two at first.
template <bool KEPT, int TERMS>
__device__ __forceinline__ void split_two(float x, float y, uint32_t (&term)[TERMS]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    const bf16x2 two = pack_bf16(x, y);
    term[t] = __builtin_bit_cast(uint32_t, two);
    if (t + 1 == TERMS) break;
    if (KEPT && t == 0) {
      x -= __uint_as_float(term[t] << 16), y -= __uint_as_float(term[t] & 0xffff0000u);
    } else {
      uint32_t first = 0x0000bf80u, second = 0xbf800000u;
      asm("" : "+s"(first), "+s"(second));  // as constants of the instruction they are something else
      x = __builtin_amdgcn_fdot2_f32_bf16(two, as_bf16x2(first), x, false);
      y = __builtin_amdgcn_fdot2_f32_bf16(two, as_bf16x2(second), y, false);
    }
  }
}
template <bool KEPT, int TERMS>
__device__ __forceinline__ void split_eight(const float (&v)[8], bf16x8 (&term)[TERMS]) {
  u32x4 all[TERMS];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t two[TERMS];
    split_two<KEPT>(v[2 * j], v[2 * j + 1], two);
#pragma unroll
    for (int t = 0; t < TERMS; ++t) all[t][j] = two[t];
  }
#pragma unroll
  for (int t = 0; t < TERMS; ++t) term[t] = __builtin_bit_cast(bf16x8, all[t]);
}

// A sum over the wavefront's lanes up to and with each one, of 64-bit integers.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t scan_step(int64_t v) {
  const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, true);
  const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, true);
  return v + static_cast<int64_t>(static_cast<uint64_t>(high) << 32 | low);
}
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
  v = scan_step<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v = scan_step<0x112, 0xf>(v);
  v = scan_step<0x114, 0xf>(v);
  v = scan_step<0x118, 0xf>(v);
  v = scan_step<0x142, 0xa>(v);     // row_bcast:15 into rows 1 and 3
  return scan_step<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
}

// The numbers of a chunk's tokens. G_i (base 2) is a sum of integers of 2^-47, to which a logarithm is rounded in 64 bits, and exact beyond that (131072 tokens are off by
// less than 2^-30 of a state however slow their decay; from f32's `x - floor(x)`, 1 - 2^-24 at most, they were by 1e-5): its nearest 256th and a rest of either sign, as exact as
// f32 is near nothing. Logarithms of 200 at most keep the sum of 64 below 2^62 and its 256ths within 24 bits.
// The factor of a row's weight of a token is a product where nothing in it can overflow or is large enough to lose bits: with R the sum up to the row's
// half of the chunk, e^{G_i - R} times e^{R - G_j} b_j (`quick`: G falls by 24 at most in either half, and the scale is no extreme). Otherwise it is made from the difference.
// b and the scale are factors throughout: as parts of an exponent, their logarithms' roundings were 2^-21 of an update of 1000.
struct Tokens {
  float row[kChunk];     // quick: scale e^{G_i - R}; otherwise b_i
  float column[kChunk];  // quick: e^{R - G_j} b_j, R of the token's own half; otherwise the rest of G_j
  float other[kChunk];   // quick: the same with R of the second half, of tokens of the first one; otherwise the 256ths of G_i
  float update[kChunk];  // e^{G_63 - G_j} b_j
  float seen[kChunk];    // scale e^{G_i}
  float fade;            // e^{G_63}, and what its rounding left of the chunks before
  float left;            // what its own rounding leaves, of a call's last chunk: no further one follows the state; next to nothing otherwise
  float whole;           // the logarithm of e^{G_63}
  int quick;
};

template <int DK, int TW, int TEAMS, int HALVES, int TERMS>
struct ChunkTiles {
  static constexpr int kWaves = TW * TEAMS, kThreads = kWave * kWaves * HALVES;
  static constexpr int kColumns = 32 * kWaves;
  static constexpr int kKeyPitch = 2 * DK, kValuePitch = 2 * kColumns;
  static constexpr int kKeyBytes = kChunk * kKeyPitch, kValueBytes = kChunk * kValuePitch;
  static constexpr int kBlock = 32 * 64;             // a 32 x 32 tile of weights, bf16
  static constexpr int kWeightBytes = TERMS * 3 * kBlock;  // of a head: tiles (0, 0), (0, 1), (1, 1) as values, then what their rounding left
  static constexpr int kKeys = 0, kValues = kKeys + kKeyBytes, kTokens = kValues + kValueBytes;
  // Places in a tile are made by exclusive ors: it begins at a whole 256 bytes.
  static constexpr int kQueries = kTokens + (2 * TEAMS * static_cast<int>(sizeof(Tokens)) + 255) / 256 * 256, kWeights = kQueries + kKeyBytes;
  // What a wavefront of one half of the rows has for the other half's, one 32 x 32 tile each.
  static constexpr int kExchange = kWeights + TEAMS * kWeightBytes, kTileBytes = 4 * 32 * 32;
  static constexpr int kSumBytes = kQueries, kBytes = kExchange + (HALVES > 1 ? kWaves * HALVES * kTileBytes : 0);
};

// A part of a tensor as a buffer: what is read behind its end is zero and what is stored there is dropped, without a branch (behind which the
// compiler would not know how many loads are on their way, and wait for all).
constexpr unsigned kOutside = 0x80000000u;  // no buffer here is as long
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 buffer_load(__amdgpu_buffer_rsrc_t b, unsigned at) { return __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0); }
__device__ __forceinline__ void buffer_store(__amdgpu_buffer_rsrc_t b, unsigned at, u32x4 v) { __builtin_amdgcn_raw_buffer_store_b128(v, b, at, 0, 0); }
// Bytes of m rows of `width` values, `ld` apart.
__device__ __forceinline__ int rows_bytes(int m, int64_t ld, int width, int size) { return m > 0 ? ((m - 1) * static_cast<int>(ld) + width) * size : 0; }

// OUT: outputs and states; otherwise a part's sum of a long sequence only. PLAIN: bf16 that can be moved 16 bytes at a time, gates bf16 or
// none (everything else in its own kernel: its loads and stores, a value at a time perhaps, would cost this one registers). Two wavefronts a SIMD, but for heads of 128 keys and up to 64
// columns that share no keys: their workgroups of two wavefronts load twice as many keys a lane, 52 registers of which would be spilled. By one wavefront a SIMD and by two: 4096 tokens of 32
// heads of 128 by 64 69 us and 106, 16384 of 8 heads of 128 by 48 79 and 116, four sequences of 512 of 16 heads 33 and 44, eight of up to 2048 59 and 100.
template <int DK, int TW, int TEAMS, int HALVES, bool OUT, bool PLAIN, int TERMS>
__global__ void __launch_bounds__(kWave * TW * TEAMS * HALVES, DK == 128 && TW * TEAMS * HALVES == 2 ? 1 : 2) linear_chunk_kernel(const ChunkArgs c) {
  using L = ChunkTiles<DK, TW, TEAMS, HALVES, TERMS>;
  constexpr int kRows = DK / HALVES;  // of the state, a wavefront's
  extern __shared__ __attribute__((aligned(256))) uint8_t lds[];
  const LinearArgs& p = c.l;
  // Workgroups that read the same keys follow one another on one die.
  const unsigned turn = blockIdx.x / 8, unit = turn / c.across * 8 + blockIdx.x % 8, number = unit / p.k_heads;
  const int beside = turn % c.across, k_head = unit % p.k_heads;
  if (number >= c.numbers) return;
  int s, j;
  if (OUT ? !mix_find(p.b, MixPieces{c.size, c.single}, number, s, j) : !mix_find_long(p.b, c.size, number, s, j)) return;
  MixSpan span = mix_span(p.b, s);
  const int slot = __builtin_amdgcn_readfirstlane(mix_slot(p.states, s));
  span.row0 = __builtin_amdgcn_readfirstlane(span.row0), span.first = __builtin_amdgcn_readfirstlane(span.first);
  span.stop = __builtin_amdgcn_readfirstlane(span.stop), span.begins = __builtin_amdgcn_readfirstlane(span.begins);
  const int begin = max(span.first, j * c.size), end = min(span.stop, (j + 1) * c.size);
  // A sequence whose parts have not all been found (its rows do not ascend) has left no states between them.
  const bool split = span.stop > c.size && (!OUT || mix_all_found(p.b, c.size, s, span));
  // The last part leaves no sum; where nothing runs through the sums afterwards, its place takes the state that the sequence goes on from: read in the
  // outputs' kernel, it may have been replaced already.
  const bool last = end == span.stop, keeps = !OUT && last && c.sums_only && p.states.in && slot >= 0 && !span.begins;
  if (begin >= end || (!OUT && (!split || (last && !keeps)))) return;
  // A sequence's part has a place of its own: those of more than one part are more than `size` rows each.
  const int64_t place = 2 * static_cast<int64_t>(span.row0 / c.size) + j;

  const int lane = threadIdx.x % kWave, h = lane / 32, n = lane % 32;
  const int number_of_wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = HALVES > 1 ? number_of_wave / L::kWaves : 0;
  const int wave = number_of_wave - half * L::kWaves, team = wave / TW, mate = wave % TW;  // by columns
  const int blocks = (p.dv + 32 * TW - 1) / (32 * TW);  // TEAMS > 1: one
  const int head0 = k_head * p.group + (TEAMS > 1 ? beside * TEAMS : beside / blocks);
  const int head_end = (k_head + 1) * p.group;
  const int column0 = TEAMS > 1 ? 0 : beside % blocks * 32 * TW;
  const int head = min(head0 + team, head_end - 1);
  const bool idle = head0 + team >= head_end;
  const int column = column0 + 32 * mate + lane_column(n);  // the lane's of the state
  const int64_t first_row = static_cast<int64_t>(span.row0) + begin;
  const int rows = end - begin, chunks = keeps ? 0 : (rows + kChunk - 1) / kChunk;

  // ---- the next chunk on its way --------------------------------------------------------------------------------------
  constexpr int kKeyLoads = kChunk * DK / 8 / L::kThreads, kValueLoads = kChunk * L::kColumns / 8 / L::kThreads;
  u32x4 next_k[kKeyLoads], next_q[OUT ? kKeyLoads : 1], next_v[kValueLoads];
  const bool whole_tiles = p.dk == DK && head0 + TEAMS <= head_end && column0 + 32 * TW <= p.dv;  // no column is nobody's
  // Where a thread's first loads of a whole chunk lie, from the chunk's first row on; the others follow rows further.
  constexpr int kKeyStep = L::kThreads / (DK / 8), kValueStep = L::kThreads / (L::kColumns / 8);
  const int my_key_row = threadIdx.x / (DK / 8), my_value_row = threadIdx.x / (L::kColumns / 8);
  const int my_key = threadIdx.x % (DK / 8) * 8, my_value = threadIdx.x % (L::kColumns / 8);
  const int my_head = min(head0 + my_value / (4 * TW), head_end - 1), my_value_at = column0 + my_value % (4 * TW) * 8;
  const bool my_key_in = my_key < p.dk, my_value_in = my_value_at < p.dv && head0 + my_value / (4 * TW) < head_end;
  const unsigned k_column = k_head * p.dk + (my_key_in ? my_key : 0), v_column = my_head * p.dv + (my_value_in ? my_value_at : 0);
  const unsigned k_from = my_key_in ? 2 * (static_cast<unsigned>(my_key_row * p.ld_k) + k_column) : kOutside;
  const unsigned q_from = my_key_in ? 2 * (static_cast<unsigned>(my_key_row * p.ld_q) + k_column) : kOutside;
  const unsigned v_from = my_value_in ? 2 * (static_cast<unsigned>(my_value_row * p.ld_v) + v_column) : kOutside;
  auto ask = [&](int chunk) __attribute__((always_inline)) {
    const int64_t row0 = first_row + static_cast<int64_t>(chunk) * kChunk;
    if constexpr (PLAIN) {  // behind the last chunk too: of nothing
      const int m = min(kChunk, rows - chunk * kChunk), keys = p.k_heads * p.dk, all = p.heads * p.dv;
      const auto k = buffer_of(static_cast<const uint16_t*>(p.k) + row0 * p.ld_k, rows_bytes(m, p.ld_k, keys, 2));
      const auto q = buffer_of(static_cast<const uint16_t*>(p.q) + row0 * p.ld_q, rows_bytes(m, p.ld_q, keys, 2));
      const auto v = buffer_of(static_cast<const uint16_t*>(p.v) + row0 * p.ld_v, rows_bytes(m, p.ld_v, all, 2));
#pragma unroll
      for (int e = 0; e < kKeyLoads; ++e) {
        next_k[e] = buffer_load(k, k_from + e * static_cast<unsigned>(2 * kKeyStep * p.ld_k));
        if constexpr (OUT) next_q[e] = buffer_load(q, q_from + e * static_cast<unsigned>(2 * kKeyStep * p.ld_q));
      }
#pragma unroll
      for (int e = 0; e < kValueLoads; ++e) next_v[e] = buffer_load(v, v_from + e * static_cast<unsigned>(2 * kValueStep * p.ld_v));
      return;
    }
    const int last = min(kChunk, rows - chunk * kChunk) - 1;
    auto load = [&](const void* x, int64_t i) { return load_eight_bf16(x, p.type, p.wide, i); };
#pragma unroll
    for (int e = 0; e < kKeyLoads; ++e) {
      const int64_t row = row0 + min(my_key_row + e * kKeyStep, last);
      if constexpr (OUT) next_q[e] = load(p.q, row * p.ld_q + k_column);
      next_k[e] = load(p.k, row * p.ld_k + k_column);
      __builtin_amdgcn_sched_barrier(0);  // one after another: f32 values of all of them do not fit
    }
#pragma unroll
    for (int e = 0; e < kValueLoads; ++e) {
      next_v[e] = load(p.v, (row0 + min(my_value_row + e * kValueStep, last)) * p.ld_v + v_column);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Behind the last chunk: values that nobody reads, so that the registers are known to be free until the next ones are asked for.
  auto ask_nothing = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < kKeyLoads; ++e) {
      if constexpr (OUT) next_q[e] = u32x4{};
      next_k[e] = u32x4{};
    }
#pragma unroll
    for (int e = 0; e < kValueLoads; ++e) next_v[e] = u32x4{};
  };
  ask(0);
  constexpr bool kEach = TW * HALVES >= 4;  // a head's wavefronts make one tile of weights each

  // ---- the decays -----------------------------------------------------------------------------------------------------
  // A token a lane: asked for two chunks ahead, made ready one ahead, by the team's last wavefront.
  Tokens* const tokens = reinterpret_cast<Tokens*>(lds + L::kTokens) + 2 * team;
  // The scale is part of the rows' factors.
  const bool counts = mate == TW - 1 && half == HALVES - 1;
  const HeadDecay head_numbers = head_decay(p, head);
  uint32_t next_raw;
  float carried = 0.0f;
  auto ask_decay = [&](int chunk) {
    next_raw = decay_raw(p, first_row + min(chunk * kChunk + lane, rows - 1), head);
  };
  auto put_decay = [&](int chunk) {
    Tokens& t = tokens[chunk % 2];
    float log, weight;
    decay_of(p, head_numbers, next_raw, log, weight);
    if (chunk * kChunk + lane >= rows) log = 0.0f, weight = 1.0f;
    const double units = static_cast<double>(log) * (1.4426950408889634 * 0x1p47);
    const int64_t g = wave_scan(log == log ? static_cast<int64_t>(rint(units)) : 0), nearest = (g + (int64_t{1} << 38)) >> 39;
    const float high = static_cast<float>(static_cast<int>(nearest)) * 0x1p-8f, rest = static_cast<float>(g - (nearest << 39)) * 0x1p-47f;
    auto of = [](float x, int token) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), token)); };
    const float last_high = of(high, kWave - 1), last_rest = of(rest, kWave - 1);
    // A NaN of a logarithm is one of its token's weight.
    const float by = weight + (log - log);
    if constexpr (OUT) {
      const float half_high = of(high, 31), half_rest = of(rest, 31);
      const float from_high = lane < 32 ? 0.0f : half_high, from_rest = lane < 32 ? 0.0f : half_rest, most = weight == weight ? fmaxf(weight, 1.0f) : 1.0f;
      const bool quick = half_high > -24.0f && last_high - half_high > -24.0f && __all(most < 0x1p60f) && fabsf(p.scale) > 0x1p-100f && fabsf(p.scale) < 0x1p100f;
      if (quick) {
        t.row[lane] = __builtin_amdgcn_exp2f((high - from_high) + (rest - from_rest)) * p.scale;
        t.column[lane] = __builtin_amdgcn_exp2f((from_high - high) + (from_rest - rest)) * by;
        t.other[lane] = __builtin_amdgcn_exp2f((half_high - high) + (half_rest - rest)) * by;
      } else {
        t.row[lane] = by;
        t.column[lane] = rest;
        t.other[lane] = high;
      }
      if (lane == 0) t.quick = quick;
      t.seen[lane] = __builtin_amdgcn_exp2f(high + rest) * p.scale;
    }
    t.update[lane] = __builtin_amdgcn_exp2f((last_high - high) + (last_rest - rest)) * by;
    // What a factor's rounding leaves goes into the next one, and behind the last one into the state itself: one that lasts many chunks, or many calls of one, does not drift.
    const float whole = (last_high + last_rest) * 0.693147181f;
    const Fade fade = fade_of(whole);
    const float more = __builtin_fmaf(fade.high, carried, fade.low), factor = fade.high + more;
    const float left = more - (factor - fade.high);
    const Fade last = fade_from(factor, OUT && (chunk + 1) * kChunk >= rows ? left : 0.0f);  // a part's sum takes the nearest factor alone
    carried = left * __builtin_amdgcn_rcpf(factor);
    if (!(fabsf(carried) < 1.0f)) carried = 0.0f;
    if (lane == 0) t.whole = whole, t.fade = last.high, t.left = last.low;
  };
  if (counts) ask_decay(0);

  // ---- the state ------------------------------------------------------------------------------------------------------
  f32x16 state[kRows / 32] = {};
  const bool mine = column < p.dv && !idle;
  const int64_t state_size = static_cast<int64_t>(p.dk) * p.dv;
  const unsigned state_from = static_cast<unsigned>((half * kRows + 8 * h) * p.dv + column);
  auto each_state = [&](float* base, auto use) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kRows / 32; ++t)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        if (!mine || half * kRows + 32 * t + 16 * a + 8 * h >= p.dk) continue;
        float* const row = base + static_cast<int64_t>(32 * t + 16 * a) * p.dv;
#pragma unroll
        for (int r = 0; r < 8; ++r) use((row + static_cast<int64_t>(r) * p.dv)[state_from], t, 8 * a + r);
      }
  };
  const int64_t part_size = part_values(p.dk, p.dv);
  f32x4* const part = reinterpret_cast<f32x4*>(c.sums + (place * p.heads + head) * part_size) + (column0 / 32 + mate) * (DK / 32 * 4 * kWave) + half * (kRows / 32 * 4 * kWave);
  const bool goes_on = p.states.in && slot >= 0 && !span.begins;
  if (OUT ? !split && goes_on : keeps) {
    float* const from = const_cast<float*>(static_cast<const float*>(p.states.in)) + (static_cast<int64_t>(slot) * p.heads + head) * state_size;
    each_state(from, [&](float& x, int t, int r) { state[t][r] = x; });
  }
  if (OUT && split && column0 + 32 * mate < p.dv) {
    auto take = [&](int k, Fade fade) {
      const f32x4* const from = part + (k - j) * p.heads * (part_size / 4);
      f32x4 four[kRows / 8];
#pragma unroll
      for (int i = 0; i < kRows / 8; ++i) four[i] = from[i * kWave + lane];
#pragma unroll
      for (int i = 0; i < kRows / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          state[i / 4][i % 4 * 4 + e] = __builtin_fmaf(state[i / 4][i % 4 * 4 + e], fade.high, __builtin_fmaf(state[i / 4][i % 4 * 4 + e], fade.low, four[i][e]));
    };
    if (!c.sums_only) take(j, Fade{0.0f, 0.0f});
    else if (goes_on) take((span.stop - 1) / c.size, Fade{0.0f, 0.0f});
    for (int k = c.sums_only ? span.first / c.size : j; k < j; ++k) take(k, fade_of(static_cast<float>(c.logs[(place + k - j) * p.heads + head])));
  }
  const float skip = p.skip ? p.skip[head] : 0.0f;
  double part_log = 0.0;

  // ---- places in LDS --------------------------------------------------------------------------------------------------
  // `now` of a place: what is made of it is made anew for each chunk (the compiler would keep every address from chunk to chunk, in registers that
  // then hold none of what is on its way).
  auto now = [](int place) {
    asm("" : "+v"(place));
    return place;
  };
  const int key_place = tile_place<L::kKeyPitch>(my_key_row, my_key / 8), value_place = tile_place<L::kValuePitch>(my_value_row, my_value);
  auto put = [&](int chunk) __attribute__((always_inline)) {
    const int m = min(kChunk, rows - chunk * kChunk);
    auto all = [&](auto in) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < kKeyLoads; ++e) {
        const bool there = in(my_key_row + e * kKeyStep < m && my_key_in);
        const int at = tile_place<L::kKeyPitch>(key_place, e * kKeyStep, 0);
        if constexpr (OUT) *reinterpret_cast<u32x4*>(lds + L::kQueries + at) = there ? next_q[e] : u32x4{};
        *reinterpret_cast<u32x4*>(lds + L::kKeys + at) = there ? next_k[e] : u32x4{};
      }
#pragma unroll
      for (int e = 0; e < kValueLoads; ++e) {
        const bool there = in(my_value_row + e * kValueStep < m && my_value_in);
        *reinterpret_cast<u32x4*>(lds + L::kValues + tile_place<L::kValuePitch>(value_place, e * kValueStep, 0)) = there ? next_v[e] : u32x4{};
      }
    };
    if (PLAIN || (m == kChunk && whole_tiles)) all([](bool) { return true; });
    else all([](bool in) { return in; });
  };
  // Where the lane's first reads lie: row n of the keys (and queries), the columns of the keys and of its values, row n of the weights.
  const int key_row = tile_place<L::kKeyPitch>(n, h);
  const int key_column = across_place<L::kKeyPitch>(half * kRows), value_column = across_place<L::kValuePitch>(32 * wave);
  const int weight_row = L::kWeights + team * L::kWeightBytes + 64 * n + 16 * (n >> 2 & 3);
  auto values_across = [&](int k) { return across<L::kValuePitch>(lds, L::kValues, value_column, k, 0); };
  const int my_column = column0 + 32 * mate + 8 * h;  // the lane's outputs of a row: 16 a .. from here on
  const int out_place = static_cast<int>(n * p.ld_out) + my_column, gate_place = 2 * (static_cast<int>(n * p.ld_gate) + my_column);

  if (counts) {
    put_decay(0);
    ask_decay(1);
  }
  put(0);
  __syncthreads();
  for (int chunk = 0; chunk < chunks; ++chunk) {
    const Tokens& t = tokens[chunk % 2];
    const int m = min(kChunk, rows - chunk * kChunk);
    const bool more = chunk + 1 < chunks, two = m > 32;
    const int64_t row0 = first_row + static_cast<int64_t>(chunk) * kChunk;
    auto ask_next = [&]() __attribute__((always_inline)) {
      if (PLAIN || more) ask(chunk + 1);
      else ask_nothing();
      __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (!OUT) ask_next();
    f32x16 out[2] = {};
    if constexpr (OUT) {
      // Weights, in tiles of 32 rows by 32 tokens: (0, 0), (1, 0), (1, 1).
      const int from = now(key_row), to = now(weight_row), here = now(n);  // compared anew: kept, the results cost more scalar registers than there are
      auto put_weights = [&](int block, int g, const float (&v)[4]) __attribute__((always_inline)) {
        uint32_t x[TERMS], y[TERMS];
        split_two<false>(v[0], v[1], x);
        split_two<false>(v[2], v[3], y);
        uint8_t* const at = lds + block * L::kBlock + (to ^ 16 * g) + 8 * h;
#pragma unroll
        for (int term = 0; term < TERMS; ++term) *reinterpret_cast<u32x2*>(at + 3 * L::kBlock * term) = u32x2{x[term], y[term]};
      };
      // Tokens 8 g + 4 h .. + 3 of the tile's. `kind`: the tile is one on the diagonal (1), the one below it (0), or either (2).
      auto weigh = [&](auto kind, int block, const f32x16& w, int g) __attribute__((always_inline)) {
        constexpr int kKind = decltype(kind)::value;
        const int token = 8 * g + 4 * h, jb = block == 2;
        const float row = t.row[32 * (block > 0) + n];
        const f32x4 columns = *reinterpret_cast<const f32x4*>((kKind == 1 || (kKind == 2 && block != 1) ? t.column + 32 * jb : t.other) + token);
        const int until = kKind == 2 && block == 1 ? 32 : here;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = w[4 * g + e] * row * columns[e];
          if (kKind != 0) v[e] = token + e <= until ? v[e] : 0.0f;
        }
        put_weights(block, g, v);
      };
      // The same from differences, a tile at a time.
      auto weigh_far = [&](int block) __attribute__((always_inline)) {
        const int jb = block == 2, ib = block > 0, until = jb == ib ? here : 32;
        f32x16 w = {};
#pragma unroll
        for (int k = 0; k < DK / 16; ++k) {
          w = __builtin_amdgcn_mfma_f32_32x32x16_bf16(eight_at(lds, L::kKeys + jb * 32 * L::kKeyPitch + (from ^ 32 * k)),
                                                      eight_at(lds, L::kQueries + ib * 32 * L::kKeyPitch + (from ^ 32 * k)), w, 0, 0, 0);
          if (k % 2) __builtin_amdgcn_sched_barrier(0);  // no more reads ahead than registers
        }
        const float high = t.other[32 * ib + n], rest = t.column[32 * ib + n];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int token = 8 * g + 4 * h;
          const f32x4 highs = *reinterpret_cast<const f32x4*>(t.other + 32 * jb + token), rests = *reinterpret_cast<const f32x4*>(t.column + 32 * jb + token);
          const f32x4 by = *reinterpret_cast<const f32x4*>(t.row + 32 * jb + token);
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = w[4 * g + e] * __builtin_amdgcn_exp2f((high - highs[e]) + (rest - rests[e])) * by[e] * p.scale;
            v[e] = token + e <= until ? v[e] : 0.0f;
          }
          put_weights(block, g, v);
        }
      };
      // What the rows see of the state, and the products of `kTiles` tiles of weights, which read the same queries; a step's operands are made ready one
      // ahead. `block`: the first tile (two: (0, 0) and (1, 0), of the same keys).
      auto see = [&](auto tiles, int block) __attribute__((always_inline)) {
        constexpr int kTiles = decltype(tiles)::value, kSteps = kRows / 16;
        const int from_half = HALVES > 1 ? from ^ 32 * kSteps * half : from;
        f32x16 w[2] = {};
        bf16x8 q[2][2], k[2], held[2][TERMS];
        const int keys_at = L::kKeys + (kTiles == 1 && block == 2) * 32 * L::kKeyPitch;
        auto ready = [&](int step) __attribute__((always_inline)) {
          const int now = step % 2;
          q[now][0] = eight_at(lds, L::kQueries + (from_half ^ 32 * step));
          q[now][1] = eight_at(lds, L::kQueries + 32 * L::kKeyPitch + (from_half ^ 32 * step));
          if constexpr (kTiles > 0) k[now] = eight_at(lds, keys_at + (from_half ^ 32 * step));
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = state[step / 2][step % 2 * 8 + e];
          split_eight<true>(v, held[now]);
        };
        // A wavefront with products goes in front of one with vector arithmetic (here and below: 126.6 us without for the 4096 tokens, 124.3 then).
        __builtin_amdgcn_s_setprio(1);
        ready(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
          const int now = step % 2;
          if (step + 1 < kSteps) ready(step + 1);
          out[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(held[now][0], q[now][0], out[0], 0, 0, 0);
          out[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(held[now][0], q[now][1], out[1], 0, 0, 0);
          if constexpr (kTiles == 2) w[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[now], q[now][0], w[0], 0, 0, 0);
          if constexpr (kTiles == 2) w[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[now], q[now][1], w[1], 0, 0, 0);
          if constexpr (kTiles == 1) {
            if (block == 0) w[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[now], q[now][0], w[0], 0, 0, 0);
            else w[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[now], q[now][1], w[0], 0, 0, 0);
          }
#pragma unroll
          for (int term = 1; term < TERMS; ++term) {
            out[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(held[now][term], q[now][0], out[0], 0, 0, 0);
            out[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(held[now][term], q[now][1], out[1], 0, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (kTiles > 0 && HALVES > 1) {  // the tile's products of the other half's keys
          const int from_other = from_half ^ 32 * kSteps, queries_at = L::kQueries + (block > 0) * 32 * L::kKeyPitch;
#pragma unroll
          for (int step = 0; step < kSteps; ++step) {
            w[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(eight_at(lds, keys_at + (from_other ^ 32 * step)), eight_at(lds, queries_at + (from_other ^ 32 * step)), w[0], 0, 0, 0);
            if (step % 4 == 3) __builtin_amdgcn_sched_barrier(0);
          }
        }
        if constexpr (kTiles > 0) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (kEach) weigh(std::integral_constant<int, 2>(), block, w[0], g);
            else weigh(std::integral_constant<int, 1>(), block, w[0], g);
            if constexpr (kTiles > 1) weigh(std::integral_constant<int, 0>(), 1, w[1], g);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      };
      // Of two wavefronts a head the first one makes tiles (0, 0) and (1, 0), the other, which has the decays, (1, 1); of more the first three one each.
      const int maker = half * TW + mate, block = kEach ? maker : 2 * maker;
      const bool makes = maker == 0 || (maker < 3 && two);
      if (!__builtin_amdgcn_readfirstlane(t.quick)) {
        if (makes) weigh_far(block);
        if (!kEach && mate == 0 && two) weigh_far(1);
        see(std::integral_constant<int, 0>(), 0);
      } else if (!kEach && mate == 0 && two) {
        see(std::integral_constant<int, kEach ? 0 : 2>(), 0);
      } else if (makes) {
        see(std::integral_constant<int, 1>(), block);
      } else {
        see(std::integral_constant<int, 0>(), 0);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) out[i] *= t.seen[32 * i + n];
      if constexpr (HALVES > 1) {  // a half keeps the rows of its own number
        const f32x16 give = half ? out[0] : out[1];
        if (half) out[0] = out[1];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *reinterpret_cast<f32x4*>(lds + L::kExchange + number_of_wave * L::kTileBytes + 16 * (r * kWave + lane)) = f32x4{give[4 * r], give[4 * r + 1], give[4 * r + 2], give[4 * r + 3]};
      }
    }
    if (counts && more) {
      put_decay(chunk + 1);
      ask_decay(chunk + 2);
    }
    // Gates are asked for here: earlier, they would take registers from what went before.
    constexpr int kOutTiles = 2 / HALVES;  // of 32 rows, a wavefront's; tile i has the rows from 32 (i + half) on
    u32x4 gate[kOutTiles][2];
    if (OUT && PLAIN && p.gate) {
      const unsigned from = now(gate_place);
      const auto g = buffer_of(static_cast<const uint16_t*>(p.gate) + row0 * p.ld_gate + static_cast<int64_t>(head) * p.dv, rows_bytes(m, p.ld_gate, p.dv, 2));
#pragma unroll
      for (int i = 0; i < kOutTiles; ++i)
#pragma unroll
        for (int a = 0; a < 2; ++a) gate[i][a] = buffer_load(g, from + (i + half) * static_cast<unsigned>(64 * p.ld_gate) + 32 * a);
    }
    if constexpr (OUT) ask_next();  // not before the products of the state have left their registers
    if constexpr (OUT) __syncthreads();
    if constexpr (OUT && HALVES > 1) {
      const int other = number_of_wave + (half ? -L::kWaves : L::kWaves);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 four = *reinterpret_cast<const f32x4*>(lds + L::kExchange + other * L::kTileBytes + 16 * (r * kWave + lane));
#pragma unroll
        for (int e = 0; e < 4; ++e) out[0][4 * r + e] += four[e];
      }
    }

    bf16x8 v[kChunk / 16];
#pragma unroll
    for (int k = 0; k < kChunk / 16; ++k) v[k] = values_across(k);
    if constexpr (OUT) {
      // A weight of nothing times an infinity or a NaN of a later token is no number: those are taken out of the product, and what rows behind
      // them see of them is added by itself.
      float odd[2] = {};
#pragma unroll
      for (int k = 0; k < kChunk / 16; ++k) {
        const u32x4 raw = __builtin_bit_cast(u32x4, v[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd[e % 2] = __builtin_amdgcn_fdot2_f32_bf16(as_bf16x2(raw[e]), as_bf16x2(0), odd[e % 2], false);
      }
      const bool some_odd = __any(odd[0] + odd[1] != 0.0f);
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
          for (int i = 0; i < kOutTiles; ++i) {
            if (token > 32 * (i + half) + n || 32 * (i + half) >= m) continue;
            const int in = token % 32;
            const uint8_t* const at = lds + (i + half + token / 32) * L::kBlock + (weight_row ^ 16 * (in / 8)) + in % 8 * 2;
            float weight = 0.0f;
#pragma unroll
            for (int term = TERMS - 1; term >= 0; --term) weight += bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(at + 3 * L::kBlock * term));
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
      // The weights' products, the gates' factors meanwhile.
      const int from = now(weight_row ^ 16 * h);
      auto weight_unit = [&](int block, int k, int term) {  // of row n, tokens 16 k + 8 h .. of the tile
        return eight_at(lds, (block + 3 * term) * L::kBlock + (from ^ 32 * k));
      };
#pragma unroll
      for (int k = 0; k < kChunk / 16; ++k)
#pragma unroll
        for (int term = 0; term < TERMS; ++term) {
          if (k < 2 && half == 0) out[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[k], weight_unit(0, k, term), out[0], 0, 0, 0);
          if (two && HALVES == 1) out[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[k], weight_unit(1 + k / 2, k % 2, term), out[1], 0, 0, 0);
          if (two && half) out[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[k], weight_unit(1 + k / 2, k % 2, term), out[0], 0, 0, 0);
        }
      __builtin_amdgcn_sched_barrier(0);
      if (some_odd) {
#pragma unroll
        for (int k = 0; k < kChunk / 16; ++k) v[k] = values_across(k);
      }
      // The skip, as token by token (as part of a row's weight of its own token, it was two terms of a bf16 result: 4096 tokens 130 us in place of 131, one result in 2000 another one
      // in place of one in 7000).
      if (p.skip) {
#pragma unroll
        for (int i = 0; i < kOutTiles; ++i)
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const u32x4 eight = __builtin_bit_cast(u32x4, eight_at(lds, L::kValues + tile_place<L::kValuePitch>(now(32 * (i + half) + n), 4 * wave + 2 * a + h)));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t pair = eight[e / 2];
              out[i][8 * a + e] = __builtin_fmaf(skip, __uint_as_float(e % 2 ? pair & 0xffff0000u : pair << 16), out[i][8 * a + e]);
            }
          }
      }
      if constexpr (PLAIN) {
        const bool short_out = p.out_type == LX_BF16;
        const int size = short_out ? 2 : 4;
        const auto to = buffer_of(static_cast<char*>(p.out) + (row0 * p.ld_out + static_cast<int64_t>(head) * p.dv) * size, idle ? 0 : rows_bytes(m, p.ld_out, p.dv, size));
        const unsigned from = now(out_place);
#pragma unroll
        for (int i = 0; i < kOutTiles; ++i)
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = out[i][8 * a + e];
            if (p.gate) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t pair = gate[i][a][e / 2];
                const float z = __uint_as_float(e % 2 ? pair & 0xffff0000u : pair << 16);
                o[e] *= TERMS > 2 ? quick_silu(z) : gate_of(z);
              }
            }
            const unsigned at = my_column + 16 * a < p.dv ? (from + (i + half) * static_cast<unsigned>(32 * p.ld_out) + 16 * a) * size : kOutside;
            if (short_out) {
              buffer_store(to, at, u32x4{__builtin_bit_cast(uint32_t, pack_bf16(o[0], o[1])), __builtin_bit_cast(uint32_t, pack_bf16(o[2], o[3])),
                                         __builtin_bit_cast(uint32_t, pack_bf16(o[4], o[5])), __builtin_bit_cast(uint32_t, pack_bf16(o[6], o[7]))});
            } else {
              buffer_store(to, at, u32x4{__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])});
              buffer_store(to, at + 16, u32x4{__float_as_uint(o[4]), __float_as_uint(o[5]), __float_as_uint(o[6]), __float_as_uint(o[7])});
            }
          }
      } else if (!idle) {
#pragma unroll
        for (int i = 0; i < kOutTiles; ++i) {
          if (32 * (i + half) + n >= m) continue;
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            if (my_column + 16 * a >= p.dv) continue;
            const int64_t column_at = static_cast<int64_t>(head) * p.dv + my_column + 16 * a, row = row0 + 32 * (i + half) + n;
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = out[i][8 * a + e];
            if (p.gate) {
#pragma unroll
              for (int e = 0; e < 8; e += 4) {
                const f32x4 z = load_four(p.gate, p.gate_type, p.wide, row * p.ld_gate + column_at + e);
#pragma unroll
                for (int f = 0; f < 4; ++f) o[e + f] *= quick_silu(z[f]);
              }
            }
            store_four(p.out, p.out_type, p.wide, row * p.ld_out + column_at, f32x4{o[0], o[1], o[2], o[3]});
            store_four(p.out, p.out_type, p.wide, row * p.ld_out + column_at + 4, f32x4{o[4], o[5], o[6], o[7]});
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // The state behind the chunk: a step's keys and scaled values made ready one ahead.
    {
      const float fade = t.fade;
      const int from = now(key_column);
      if constexpr (!OUT) part_log += t.whole;
      constexpr int kTerms = 3;
      bf16x8 key[2][kRows / 32], scaled_v[2][kTerms];
      auto ready = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < kRows / 32; ++x)
          key[k % 2][x] = across<L::kKeyPitch>(lds, L::kKeys, from, k, 4 * x);  // columns 32 x .. of tokens 16 k ..
        const u32x4 raw = __builtin_bit_cast(u32x4, v[k]);
        const f32x4 w0 = *reinterpret_cast<const f32x4*>(t.update + 16 * k + 8 * h), w1 = *reinterpret_cast<const f32x4*>(t.update + 16 * k + 8 * h + 4);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t pair = raw[e / 2];
          x[e] = __uint_as_float(e % 2 ? pair & 0xffff0000u : pair << 16) * (e < 4 ? w0[e % 4] : w1[e % 4]);
        }
        split_eight<false>(x, scaled_v[k % 2]);
      };
      const float left = t.left;
      __builtin_amdgcn_s_setprio(1);
      ready(0);
      // A branch around the second factor, or the compiler's own sum, costs registers that are not there (45 spilled, 184 us for the 4096 tokens): always, in place.
#pragma unroll
      for (int x = 0; x < kRows / 32; ++x) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if constexpr (OUT) {
            float in = state[x][e];
            const float rest = in * left;  // and by this it is known to be there
            asm("v_fma_f32 %0, %0, %1, %2" : "+v"(in) : "v"(fade), "v"(rest));
            state[x][e] = in;
          } else {
            state[x][e] *= fade;
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (OUT) asm volatile("s_nop 1");  // products do not wait for what they are not told of
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < kChunk / 16; ++k) {
        if (k + 1 < kChunk / 16) ready(k + 1);
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
#pragma unroll
          for (int x = 0; x < kRows / 32; ++x) state[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(key[k % 2][x], scaled_v[k % 2][term], state[x], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();
    if (more) {
      put(chunk + 1);
      __syncthreads();
    }
  }

  if constexpr (OUT) {
    if (p.states.out && slot >= 0 && last)
      each_state(static_cast<float*>(p.states.out) + (static_cast<int64_t>(slot) * p.heads + head) * state_size, [&](float& x, int t, int r) { x = state[t][r]; });
  } else if (!idle && column0 + 32 * mate < p.dv) {
#pragma unroll
    for (int i = 0; i < kRows / 8; ++i) part[i * kWave + lane] = f32x4{state[i / 4][i % 4 * 4], state[i / 4][i % 4 * 4 + 1], state[i / 4][i % 4 * 4 + 2], state[i / 4][i % 4 * 4 + 3]};
    if (mate == 0 && half == 0 && lane == 0 && column0 == 0) c.logs[place * p.heads + head] = part_log;
  }
}

// The states in front of a long sequence's parts, where their sums were: four values a thread, all parts in order.
__global__ void __launch_bounds__(256) linear_parts_kernel(const ChunkArgs c) {
  const LinearArgs& p = c.l;
  const int64_t part_size = part_values(p.dk, p.dv), fours = p.heads * part_size / 4;
  const unsigned groups = static_cast<unsigned>((fours + 255) / 256);
  int s, j;
  if (!mix_find_long(p.b, c.size, 2 * (blockIdx.x / groups), s, j) || j != 0) return;
  const MixSpan span = mix_span(p.b, s);
  const int slot = mix_slot(p.states, s);
  if (span.stop <= c.size || !mix_all_found(p.b, c.size, s, span)) return;
  const int64_t i = static_cast<int64_t>(blockIdx.x % groups) * 256 + threadIdx.x;
  if (i >= fours) return;
  const int head = static_cast<int>(4 * i / part_size), of_head = static_cast<int>(i - head * (part_size / 4)), parts = (span.stop + c.size - 1) / c.size;
  const int64_t place = 2 * static_cast<int64_t>(span.row0 / c.size);
  f32x4 state = {};
  if (p.states.in && slot >= 0 && !span.begins) {
    // Four neighbouring rows of a column.
    const int lane = of_head % kWave, quad = of_head / kWave % 4, tiles = p.dk <= 64 ? 2 : p.dk <= 128 ? 4 : 8, t = of_head / kWave / 4 % tiles;
    const int row = 32 * t + quad / 2 * 16 + lane / 32 * 8 + quad % 2 * 4, column = of_head / kWave / 4 / tiles * 32 + lane_column(lane % 32);
    const float* const from = static_cast<const float*>(p.states.in) + ((static_cast<int64_t>(slot) * p.heads + head) * p.dk + row) * p.dv + column;
    if (row < p.dk && column < p.dv) {
#pragma unroll
      for (int e = 0; e < 4; ++e) state[e] = from[e * p.dv];
    }
  }
  // Parts in front of position 0 have left no sum. Several at a time: one by one, each would wait for a load behind the last one's store.
  constexpr int kTogether = 8;
  for (int k0 = span.first / c.size; k0 < parts; k0 += kTogether) {
    const int last = parts - 1;
    f32x4 sum[kTogether];
    double log[kTogether];
#pragma unroll
    for (int e = 0; e < kTogether; ++e) {
      if (k0 + e >= last) break;  // the last part leaves no sum
      const int64_t at = place + k0 + e;
      sum[e] = reinterpret_cast<const f32x4*>(c.sums + at * p.heads * part_size)[i];
      log[e] = c.logs[at * p.heads + head];
    }
#pragma unroll
    for (int e = 0; e < kTogether; ++e) {
      if (k0 + e > last) break;
      reinterpret_cast<f32x4*>(c.sums + (place + k0 + e) * p.heads * part_size)[i] = state;
      if (k0 + e == last) break;
      const Fade fade = fade_of(static_cast<float>(log[e]));
#pragma unroll
      for (int x = 0; x < 4; ++x) state[x] = __builtin_fmaf(state[x], fade.high, __builtin_fmaf(state[x], fade.low, sum[e][x]));
    }
  }
}

}  // namespace dro
