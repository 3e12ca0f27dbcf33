// lx_kv8_attention for many rows a sequence (prompts and pieces of prompts): the matrix cores decide.
//
// The mathematics is kv8_stream.h's. A workgroup takes 128 rows of one of the cache's heads, 32 a wavefront, and walks their
// tokens 64 at a time (128 of heads of 64 values). What the wavefronts share is made once: the tile's key codes become
// bf16 rows in LDS, its value codes f16 columns (transposed on the way, in registers), while the tile before it is worked on;
// one barrier a tile. A wavefront multiplies 32 keys by its 32 rows (S^T = K Q^T, v_mfma_f32_32x32x16): a lane then holds 16
// scores of one row, tokens 8 a + 4 h + b (h = lane / 32), and a sum over 16 tokens takes its eight of them as they
// lie, so the value columns are stored in that order and weights never change lanes.
//
// What bounds it. 4096 rows of 32 heads of 128: 137 GFLOP in 158 .. 176 us (devices differ), 780 .. 870 TFLOP/s where a large plain product
// reaches 1220. A wavefront has 1024 cycles of matrix work a tile and takes about 4600, reads, scores' arithmetic (one maximum, one
// multiply-add, one exponential, half a conversion and one sum a score) and matrix work one after another; two a SIMD fill one
// another's gaps in part: the matrix cores are busy 40 % of the time, vector arithmetic half of it. Heads of 64 have twice the
// score arithmetic for a matrix instruction: 4096 rows of 32 heads 105 us, 655 TFLOP/s.
// LDS rows are swizzled by 16-byte pieces so that the 32 rows of a read fall on all banks.
#pragma once

#include "kv8_stream.h"

namespace dro {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileRowsOfWave = 32;
constexpr int kTileWaves = 4;
constexpr int kTileRowsOfGroup = kTileRowsOfWave * kTileWaves;

// Tokens of a tile: 16 KB of keys and 16 KB of values in LDS, twice.
template <int DIM>
constexpr int tile_tokens() {
  return 8192 / DIM;
}

// What the scheduler is told to group: matrix instructions, reads of LDS, vector arithmetic.
constexpr int kMatrix = 0x8, kReads = 0x100, kVector = 0x2;

// Where 16-byte piece `piece` of a row lies in its row. Sixteen rows that a read takes a piece of each fall on sixteen places of
// the 256 bytes that the banks are wide, and eight neighbouring lanes that write (neighbouring rows, or of the keys' image every
// other piece of a row, which is why its even pieces come first) on eight places of 128.
template <int kPitch>
__device__ __forceinline__ int swizzled(int row, int piece) {
  return piece ^ (kPitch % 256 == 0 ? row & 15 : (row ^ row >> 3) & 7);
}
template <int DIM>
__device__ __forceinline__ int key_place(int row, int piece) {
  return 16 * swizzled<2 * DIM>(row, piece % 2 * (DIM / 16) + piece / 2);
}

// Dims 4 quad .. 4 quad + 3 of a row's sums, which lie in the rows of the value image that start DIM / 4 apart: quad
// 16 a + 8 b + 4 h + c.
template <int DIM>
__device__ __forceinline__ f32x4 four_dims(const f32x16 (&acc)[DIM / 32], int a, int b, int c) {
  f32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int row = k * (DIM / 4) + 16 * a + 8 * b + c;
    v[k] = acc[row / 32][row % 32 / 8 * 4 + c];
  }
  return v;
}

template <int F, int DIM>
__global__ void __launch_bounds__(256, 2) tile_kernel(const AttentionArgs p) {
  static_assert(DIM == 64 || DIM == 128, "a tile's 16 KB images");
  constexpr int kTok = tile_tokens<DIM>(), kKeyPitch = 2 * DIM, kValuePitch = 2 * kTok;
  constexpr int kKeyBytes = kTok * kKeyPitch, kBuffer = 2 * kKeyBytes;
  extern __shared__ __attribute__((aligned(256))) uint8_t lds[];  // two buffers of keys and values
  __shared__ __attribute__((aligned(32))) float key_scale[kMaxRuns], value_log[kMaxRuns];
  __shared__ int holes;
  const Kv8Cache& c = p.c;
  const int head = blockIdx.x % c.heads;
  int64_t rest = blockIdx.x / c.heads;
  const int split = static_cast<int>(rest % p.splits);
  rest /= p.splits;
  // Later rows see more tokens: they go first. Where all workgroups are resident at once, two a compute unit, the second of them
  // starts from the other end, so that a unit has a long one and a short one (2048 rows of 32 heads of 128: 67 -> 59 us).
  const int turn = static_cast<int>(rest % p.row_tiles), seq = static_cast<int>(rest / p.row_tiles);
  const int half = (p.row_tiles + 1) / 2;
  const int tile = p.fold && turn >= half ? turn - half : p.row_tiles - 1 - turn;
  const RowTile t = row_tile(p, seq, tile, kTileRowsOfGroup);
  if (t.count <= 0) return;
  const int64_t start = t.begin + static_cast<int64_t>(split) * p.chunk;
  if (start >= t.end && split > 0) return;
  const bool alone = static_cast<int64_t>(t.begin) + p.chunk >= t.end;
  const int part_begin = static_cast<int>(start), part_end = static_cast<int>(min(start + p.chunk, static_cast<int64_t>(t.end)));

  const int lane = threadIdx.x % kWave, h = lane / 32, n = lane % 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int my_first = t.first + kTileRowsOfWave * wave;  // the wavefront's rows
  const int my_count = min(t.first + t.count - my_first, kTileRowsOfWave);
  const int lead = t.span.length - t.span.rows;
  const int pos = lead + (my_first + n) / p.group;
  const int low_pos = lead + my_first / p.group, high_pos = lead + (my_first + max(my_count, 1) - 1) / p.group;
  bf16x8 q[DIM / 16];
  {
    const int flat = my_first + n, token = flat / p.group;
    const int64_t at = n < my_count ? (t.span.row0 + token) * p.ld_q + static_cast<int64_t>(head * p.group + flat % p.group) * DIM : 0;
    load_query(p, n < my_count, at, [&](int k) { return 16 * k + 8 * h; }, q);
  }
  f32x16 acc[DIM / 32] = {};
  float base = kNothing, term_base = kNothing, total = 0.0f;

  // What a wavefront brings of a tile: a run, or two of heads of 64: its key rows 16 bytes a lane and load, and eight tokens by
  // four dims of its values a lane.
  constexpr int kKeyLoads = 2;
  auto key_run = [&](int e) { return DIM == 64 ? 2 * wave + e : wave; };     // of load e, in the tile
  auto key_piece = [&](int e) { return DIM == 64 ? lane : lane + 64 * e; };  // of the run's rows
  const int value_run = DIM == 64 ? 2 * wave + lane / 32 : wave;
  const int value_half = lane / (DIM / 4) % 2, quad = lane % (DIM / 4);
  u32x4 key_codes[kKeyLoads];
  uint32_t value_codes[8];
  // Lane kRunsOfWave * i + e holds where the wavefront's run e of the window's tile i lies: -1 where it has none, or no page.
  constexpr int kTileRuns = kTok / kRun, kRunsOfWave = kTileRuns / kTileWaves;
  static_assert(kMaxRuns == kWave * kTileWaves, "a lane a run");
  int my_run = -1;
  // The codes of the window's tile i on their way.
  auto ask = [&](int i) {
    auto place = [&](int e) { return static_cast<int64_t>(max(__builtin_amdgcn_readlane(my_run, kRunsOfWave * i + e), 0)) * (kRun * DIM); };
#pragma unroll
    for (int e = 0; e < kKeyLoads; ++e) key_codes[e] = *reinterpret_cast<const u32x4*>(c.k + place(DIM == 64 ? e : 0) + 16 * key_piece(e));
    const uint8_t* at = c.v + place(0);
    if constexpr (DIM == 64) at = lane < 32 ? at : c.v + place(1);
    at += 4 * value_half * DIM + 4 * quad;
#pragma unroll
    for (int k = 0; k < 8; ++k) value_codes[k] = *reinterpret_cast<const uint32_t*>(at + (k % 4 + 8 * (k / 4)) * DIM);
  };
  // The codes asked for into LDS. `first`: the tile's first token; `clean`: every place of the tile holds a token.
  auto put = [&](uint8_t* buffer, int i, int first, bool clean) {
#pragma unroll
    for (int e = 0; e < kKeyLoads; ++e) {
      const int row = kRun * key_run(e) + key_piece(e) / (DIM / 16), column = key_piece(e) % (DIM / 16);
      uint8_t* const at = buffer + row * kKeyPitch;
      *reinterpret_cast<bf16x8*>(at + key_place<DIM>(row, 2 * column)) = weight_fragment<F>(key_codes[e], 0, 0);
      *reinterpret_cast<bf16x8*>(at + key_place<DIM>(row, 2 * column + 1)) = weight_fragment<F>(key_codes[e], 0, 1);
    }
    if (!clean) {  // codes of places without a token (NaNs perhaps) times a weight of nothing have to be nothing
      bool there = __builtin_amdgcn_readlane(my_run, kRunsOfWave * i) >= 0;
      if constexpr (DIM == 64) there = lane < 32 ? there : __builtin_amdgcn_readlane(my_run, kRunsOfWave * i + 1) >= 0;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (!there || first + kRun * value_run + 4 * value_half + k % 4 + 8 * (k / 4) >= t.span.length) value_codes[k] = 0;
    }
    uint32_t two[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t x = flipped<F>(value_codes[2 * k]), y = flipped<F>(value_codes[2 * k + 1]);
      two[k][0] = __builtin_amdgcn_perm(y, x, 0x05010400u);
      two[k][1] = __builtin_amdgcn_perm(y, x, 0x07030602u);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      f16x2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = f % 2 ? pair_of<F, true>(two[k][f / 2]) : pair_of<F, false>(two[k][f / 2]);
      // Dim 4 quad + f is row f DIM / 4 + quad of the image, so that neighbouring lanes write neighbouring rows.
      const int row = f * (DIM / 4) + quad;
      *reinterpret_cast<f16x8*>(buffer + kKeyBytes + row * kValuePitch + 16 * swizzled<kValuePitch>(row, 2 * value_run + value_half)) = __builtin_bit_cast(f16x8, v);
    }
  };

  for (int64_t from = part_begin; from < part_end; from += kMaxRuns * kRun) {
    const int window = static_cast<int>(from);  // up to kMaxRuns runs from here
    const int stop = static_cast<int>(min(from + kMaxRuns * kRun, static_cast<int64_t>(part_end)));
    const int runs = (stop - window + kRun - 1) / kRun;
    // Where the window's runs lie (-1: no page, no tokens), and their scales.
    __syncthreads();
    if (threadIdx.x == 0) holes = 0;
    __syncthreads();
    const int mine = lane / kRunsOfWave * kTileRuns + kRunsOfWave * wave + lane % kRunsOfWave;  // the lane's run of the window
    float ks = 0.0f, vs = 0.0f;
    my_run = -1;
    if (mine < runs) {
      const int token = window + kRun * mine, page = kv8_page(c, p.b, seq, token);
      if (page >= 0) {
        const int64_t at = kv8_row(c, page, head) + token % c.page;
        my_run = static_cast<int>(at / kRun);
        ks = c.k_scale[at >> c.block_shift] * fabsf(p.scale) * 1.4426950408889634f;
        vs = fabsf(c.v_scale[at >> c.block_shift]);
      } else {
        holes = 1;
      }
    }
    key_scale[mine] = my_run >= 0 ? ks : __builtin_nanf("");  // a NaN: nothing of the run is seen
    value_log[mine] = __builtin_amdgcn_logf(vs);
    __syncthreads();
    const bool whole = !holes;
    const int tiles = (runs * kRun + kTok - 1) / kTok;
    auto clean = [&](int i) { return whole && window + (i + 1) * kTok <= min(stop, t.span.length); };
    ask(0);
    put(lds, 0, window, clean(0));
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      const uint8_t* const keys = lds + (i % 2) * kBuffer;
      const uint8_t* const values = keys + kKeyBytes;
      const int at = window + i * kTok;
      const bool more = i + 1 < tiles;
      if (more) ask(i + 1);
      float ks[kTileRuns], vl[kTileRuns];
#pragma unroll
      for (int j = 0; j < kTileRuns; ++j) {
        ks[j] = key_scale[i * kTileRuns + j];
        vl[j] = value_log[i * kTileRuns + j];
      }
      const bool some = my_count > 0 && at <= high_pos && (p.window == 0 || at + kTok > static_cast<int64_t>(low_pos) - p.window + 1);
      if (some) {
        // The wavefronts of a SIMD take turns: the one that feeds the matrix cores goes first (176 -> 169 us on a 4096-row prompt).
        __builtin_amdgcn_s_setprio(1);
        f32x16 s[kTok / 32] = {};
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k)
#pragma unroll
          for (int b = 0; b < kTok / 32; ++b) {
            const int row = 32 * b + n;
            const bf16x8 a = *reinterpret_cast<const bf16x8*>(keys + row * kKeyPitch + key_place<DIM>(row, 2 * k + h));
            s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, q[k], s[b], 0, 0, 0);
          }
        // Six reads ahead of the matrix instructions, not one or two (162 -> 150 us).
        __builtin_amdgcn_sched_group_barrier(kReads, 6, 0);
#pragma unroll
        for (int e = 0; e < 10; ++e) {
          __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
          __builtin_amdgcn_sched_group_barrier(kReads, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMatrix, 6, 0);
        __builtin_amdgcn_s_setprio(0);
        const bool plain = clean(i) && at + kTok - 1 <= low_pos && (p.window == 0 || at > static_cast<int64_t>(high_pos) - p.window);
        if (!plain) {
#pragma unroll
          for (int j = 0; j < kTok / kRun; ++j) {
            const bool there = ks[j] == ks[j];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int token = at + kRun * j + 8 * (e / 4) + 4 * h + e % 4;
              const bool hidden = !there || token > pos || (p.window > 0 && token <= pos - p.window);
              s[j / 2][8 * (j % 2) + e] = hidden ? -__builtin_inff() : s[j / 2][8 * (j % 2) + e] * ks[j];
            }
            ks[j] = 1.0f;
          }
        }
        float m = -__builtin_inff(), most_term = m;
#pragma unroll
        for (int j = 0; j < kTok / kRun; ++j) {
          float r = s[j / 2][8 * (j % 2)];
#pragma unroll
          for (int e = 1; e < 8; ++e) r = fmaxf(r, s[j / 2][8 * (j % 2) + e]);
          r *= ks[j];
          m = fmaxf(m, r);
          most_term = fmaxf(most_term, r + vl[j]);
        }
        if (__any(m > base + kSlack || most_term > term_base + kSlack)) {
          float x0, x1;
          swap_halves<false>(m, x0, x1);
          m = fmaxf(fmaxf(x0, x1) - kTermBits, base);
          swap_halves<false>(most_term, x0, x1);
          most_term = fmaxf(fmaxf(x0, x1) - kTermBits, term_base);
          total *= __builtin_amdgcn_exp2f(base - m);
          const float keep = __builtin_amdgcn_exp2f(term_base - most_term);
#pragma unroll
          for (int f = 0; f < DIM / 32; ++f) acc[f] *= keep;
          base = m;
          term_base = most_term;
        }
        const float least = kLeastLift - base;
        // A run's weights are made while the matrix cores work on the one before it, from values that were read before that.
        f16x8 a[2][DIM / 32];
        auto read_values = [&](int j, f16x8 (&to)[DIM / 32]) {
#pragma unroll
          for (int f = 0; f < DIM / 32; ++f) {
            const int row = 32 * f + n;
            to[f] = *reinterpret_cast<const f16x8*>(values + row * kValuePitch + 16 * swizzled<kValuePitch>(row, 2 * j + h));
          }
        };
        if (DIM == 128) __builtin_amdgcn_s_setprio(1);
        read_values(0, a[0]);
#pragma unroll
        for (int j = 0; j < kTok / kRun; ++j) {
          if (j + 1 < kTok / kRun) read_values(j + 1, a[(j + 1) % 2]);
          const float lift = fmaxf(vl[j] - term_base, least);
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j / 2][8 * (j % 2) + e], ks[j], lift));
          const f16x2 v[4] = {pack_f16(w[0], w[1]), pack_f16(w[2], w[3]), pack_f16(w[4], w[5]), pack_f16(w[6], w[7])};
          float sum = w[0];
#pragma unroll
          for (int e = 1; e < 8; ++e) sum += w[e];
          total = __builtin_fmaf(sum, __builtin_amdgcn_exp2f(-base - lift), total);
          const f16x8 terms = __builtin_bit_cast(f16x8, v);
#pragma unroll
          for (int f = 0; f < DIM / 32; ++f) acc[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[j % 2][f], terms, acc[f], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      if (more) put(lds + ((i + 1) % 2) * kBuffer, i + 1, at + kTok, clean(i + 1));
      __syncthreads();
    }
  }

  float x0, x1;
  swap_halves<false>(total, x0, x1);
  const float sum = x0 + x1;
  if (n >= my_count) return;
  const float root = term_root(term_base, base);
  if (alone) {
    const int flat = my_first + n;
    const int64_t at = (t.span.row0 + flat / p.group) * p.ld_out + static_cast<int64_t>(head * p.group + flat % p.group) * DIM;
    const float factor = root * over_weights(sum);
#pragma unroll
    for (int a = 0; a < DIM / 64; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int k = 0; k < 4; ++k) store_four(p, at + 4 * (16 * a + 8 * b + 4 * h + k), four_dims<DIM>(acc, a, b, k) * root * factor);
  } else {
    float* const part = partial_at<DIM>(p, (static_cast<int64_t>(seq) * p.row_tiles + tile) * c.heads + head, split, kTileRowsOfGroup);
    const int row = kTileRowsOfWave * wave + n;
#pragma unroll
    for (int a = 0; a < DIM / 64; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<f32x4*>(part + row * DIM + 4 * (16 * a + 8 * b + 4 * h + k)) = four_dims<DIM>(acc, a, b, k) * root * root;
    if (h == 0) {
      part[kTileRowsOfGroup * DIM + 2 * row] = base;
      part[kTileRowsOfGroup * DIM + 2 * row + 1] = sum;
    }
  }
}

template <int DIM>
constexpr int tile_lds_bytes() {
  return 2 * 2 * 2 * DIM * tile_tokens<DIM>();
}

}  // namespace dro
