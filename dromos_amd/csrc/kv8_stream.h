// lx_kv8_attention for few rows a sequence: the cache is streamed once, so its bytes decide.
//
// Mathematics. o = sum_t w_t v_t / sum_t w_t with w_t = 2^(c_t - m), c_t = (q . k_t) * scale * log2 e, m a score near the
// largest c so far: one pass over the keys, sums and values rescaled by 2^(m_old - m_new) where a much larger score comes. Scores are taken the other
// way round, S^T = K Q^T, sixteen keys (A) by sixteen rows (B): a lane then holds the scores of one row (lane % 16) and four
// keys, which is the layout in which O^T = V^T P^T wants its B operand, so weights never change lanes, and a row's
// rescaling is its lanes' own. The matrix instruction sums over k in any order that both operands agree on: keys are read 16
// bytes a lane as they lie, and a lane's slots of a sum over tokens are the four of one run of 16 and the four of the next
// that it holds weights of. Values are read DIM / 16 bytes a lane and token (16 lanes a row) and transposed by bytes in
// registers, two permutations for four tokens' pairs. Key codes become bf16 exactly, as the queries are; value codes become
// f16 exactly. A key block's scale multiplies its scores; a value block's scale u goes into its weights as an exponent: the
// matrix cores take terms 2^(c + log2 u - n), one multiply-add and one exponential, rounded to f16: three more bits than bf16, so
// these roundings (2^-11 of each term) stay well below the result's own. n is a row's reference for c + log2 u, as m is for c, so
// f16's range is spent on what the row sees and on nothing else. Either follows only where a token is 2^8 ahead of it. Terms are held
// times 2^7: the largest is 2^15 at most, one 2^-21 of the reference's still a normal number, one under 2^-32 nothing, and most
// steps leave the sums as they are. A token counts in the sum of weights however small its values are: that adds up the terms
// before they are rounded, in f32, and takes log2 u off again once per run. A block's exponent is 2^-60 of its weights' at least,
// so its terms are numbers in f32 (and nothing in f16) where its scale is 0.
//
// Split. A workgroup takes one sequence, 16 RT rows of one of the cache's heads (rows of a head: its tokens' query heads,
// token after token) and up to kMaxRuns runs of 16 tokens of it. Its four wavefronts take 64 tokens at a time in turn (32 of
// heads wider than 128) and keep sums of their own; the workgroup adds them up at its end, in order. Where a sequence has several
// such parts they leave their sums in the workspace, and a second kernel adds those, in order.
//
// What bounds it (heads of 128, int8 or fp8). One sequence of 131072 tokens: 50.6 us for 268 MB, 5.3 TB/s, the rate of a copy.
// 32 of up to 4096 tokens, as uneven as they come: 35.9 us where their bytes want 27, the longest one's workgroups end last. 8 of 5 rows
// (20 a head, two tiles' worth of registers): 23.0 us where their bytes want 12.6; parts are cut by the longest possible sequence, so
// 256 of 512 workgroups find a token, one a unit, and its four wavefronts wait for memory in each of four steps. 517 tokens: 9.5 us,
// two steps of a wavefront whose every load follows one before it.
#pragma once

#include "kv8.h"
#include "tile_mfma.h"

namespace dro {

constexpr int kStreamWaves = 4, kStreamThreads = kStreamWaves * kWave;
constexpr int kMaxRuns = 256;  // runs of 16 tokens a workgroup takes at most

// Runs a wavefront takes at a time: four, or two where four runs' codes and the sums (DIM * RT / 4 registers) would not fit
// the 256 registers that two wavefronts a SIMD leave each.
template <int DIM>
constexpr int step_runs() {
  return DIM <= 128 ? 4 : 2;
}

struct AttentionArgs {
  Kv8Cache c;
  Kv8Batch b;
  const void* q;
  void* out;
  float* partial;
  int64_t ld_q, ld_out;
  int q_dtype, out_dtype, group, window;
  float scale;
  int wide_q;                    // q is bf16 and can be read 16 bytes at a time
  int wide_out;                  // out can be written 8 (bf16) or 16 (f32) bytes at a time
  int fold;                      // see kv8_tile.h
  int row_tiles, splits, chunk;  // chunk: tokens of a part, a multiple of 256, 16 * kMaxRuns at most (tiles of 128 rows: any number)
};

// What one tile of rows of a sequence attends to.
struct RowTile {
  Kv8Span span;
  int first, count;      // flat rows (token * group + query head) of the tile
  int low_pos, high_pos; // positions of its first and last row
  int begin, end;        // tokens that any of its rows sees: begin is a multiple of 16; begin >= end: none
};

__device__ __forceinline__ RowTile row_tile(const AttentionArgs& p, int seq, int tile, int per_tile) {
  RowTile t;
  t.span = kv8_span(p.b, p.c.page, seq);
  const int rows = min(t.span.rows, p.b.max_rows) * p.group;
  t.first = tile * per_tile;
  t.count = min(rows - t.first, per_tile);
  const int lead = t.span.length - t.span.rows;
  t.low_pos = lead + t.first / p.group;
  t.high_pos = lead + (t.first + max(t.count, 1) - 1) / p.group;
  t.end = t.count > 0 ? t.high_pos + 1 : 0;
  const int64_t first_seen = p.window > 0 ? static_cast<int64_t>(t.low_pos) - p.window + 1 : 0;
  t.begin = first_seen > 0 ? static_cast<int>(first_seen) & ~(kRun - 1) : 0;
  return t;
}

// Where a partial sum lies: 16 RT rows of DIM sums, then a row's largest score and sum of weights.
template <int DIM>
__device__ __forceinline__ float* partial_at(const AttentionArgs& p, int64_t item, int split, int per_tile) {
  return p.partial + (item * p.splits + split) * per_tile * (DIM + 2);
}

// The bytes of a run's key rows that a lane holds: 16 at 16 g of every 64, and its values': DIM / 16 of four tokens.
template <int DIM>
struct KeyRegs {
  u32x4 w[DIM / 64];
};
template <int DIM>
struct ValueRegs {
  uint32_t w[4][DIM / 64];
};

template <int DIM>
__device__ __forceinline__ void load_keys(KeyRegs<DIM>& r, const uint8_t* run, int lane_off) {
#pragma unroll
  for (int c = 0; c < DIM / 64; ++c) r.w[c] = *reinterpret_cast<const u32x4*>(run + lane_off + 64 * c);
}

template <int DIM>
__device__ __forceinline__ void load_values(ValueRegs<DIM>& r, const uint8_t* run, int lane_off) {
  typedef uint32_t vec __attribute__((ext_vector_type(DIM / 64 == 3 ? 3 : DIM / 64), aligned(4)));
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (DIM == 64) {
      r.w[t][0] = *reinterpret_cast<const uint32_t*>(run + lane_off + t * DIM);
    } else {
      const vec v = *reinterpret_cast<const vec*>(run + lane_off + t * DIM);
#pragma unroll
      for (int j = 0; j < DIM / 64; ++j) r.w[t][j] = v[j];
    }
  }
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Two neighbouring codes of a dword (the low or the high pair) as f16. An int8 code with its top bit flipped is code + 128; as
// the low byte under 0x64 it is the half 1024 + 128 + code.
template <int F, bool HIGH>
__device__ __forceinline__ f16x2 pair_of(uint32_t d) {
  if constexpr (F == LX_W_FP8) {
    return __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d, 1.0f, HIGH));
  } else {
    const uint32_t h = __builtin_amdgcn_perm(0x64646464u, d, HIGH ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(f16x2, h) - f16x2{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
  }
}

// The bytes of value codes as pair_of takes them.
template <int F>
__device__ __forceinline__ uint32_t flipped(uint32_t d) {
  return F == LX_W_INT8 ? d ^ 0x80808080u : d;
}

__device__ __forceinline__ f16x2 pack_f16(float a, float b) { return f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)}; }

// Row references less 7 (terms and weights are held times 2^7); how far a score or a term may be ahead of them before they follow;
// and what they are until a row sees a token.
constexpr float kTermBits = 7.0f, kSlack = 8.0f + kTermBits, kNothing = -1e30f;
constexpr float kLeastLift = -60.0f;  // a term over its weight, at least (log2)

// Sums of terms times this, twice, are relative to the reference `base`, as the sum of weights is, and held times 2^-32: sums over 2^17
// tokens of values of f32's whole range (which their mean may have) are in it then, and values from 2^-101 on.
__device__ __forceinline__ float term_root(float term_base, float base) { return __builtin_amdgcn_exp2f(0.5f * (term_base - base) - 16.0f); }

// What such a sum has to be multiplied by. No token: 0; no number: that.
__device__ __forceinline__ float over_weights(float sum) { return sum > 0.0f ? 0x1p32f / sum : sum == 0.0f ? 0.0f : sum; }

// N eights of a query's values, `stride` values apart from `at` on, as the matrix instruction's operands; f32 ones are rounded to
// bf16 here. A negative scale's sign goes to them, so that the scales of the scores never turn a largest one into a smallest.
// A row that is none is read as row 0's and becomes zeros.
template <int N, typename Offset>
__device__ __forceinline__ void load_query(const AttentionArgs& p, bool have, int64_t at, Offset offset, bf16x8 (&q)[N]) {
  u32x4 w[N];
  if (p.wide_q) {
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.q) + at + offset(k));
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      bf16x2 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = pack_bf16(load_as_f32(p.q, p.q_dtype, at + offset(k) + 2 * j), load_as_f32(p.q, p.q_dtype, at + offset(k) + 2 * j + 1));
      w[k] = __builtin_bit_cast(u32x4, v);
    }
  }
  const uint32_t sign = p.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
  for (int k = 0; k < N; ++k) q[k] = __builtin_bit_cast(bf16x8, have ? w[k] ^ sign : u32x4{0u, 0u, 0u, 0u});
}

// Four consecutive values of a result.
__device__ __forceinline__ void store_four(const AttentionArgs& p, int64_t at, f32x4 v) {
  if (!p.wide_out) {
#pragma unroll
    for (int k = 0; k < 4; ++k) store_from_f32(p.out, p.out_dtype, at + k, v[k]);
  } else if (p.out_dtype == LX_BF16) {
    const bf16x2 two[2] = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.out) + at) = __builtin_bit_cast(u32x2, two);
  } else {
    *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + at) = v;
  }
}

template <int F, int DIM, int RT>
__global__ void __launch_bounds__(kStreamThreads, 2) stream_kernel(const AttentionArgs p) {
  constexpr int kC = DIM / 64, kTiles = DIM / 16, kPerTile = 16 * RT, kRuns = step_runs<DIM>(), kStep = kRuns * kRun;
  __shared__ float wave_top[kStreamWaves][kPerTile], wave_sum_of[kStreamWaves][kPerTile];
  __shared__ float sums[kStreamWaves][16][DIM + 4];
  const Kv8Cache& c = p.c;
  const int head = blockIdx.x % c.heads;
  // The first parts of all sequences go first: later ones may have nothing to do, and workgroups that do lie side by side evenly
  // (16 streams of up to 8192 tokens: with a sequence's parts side by side 160 compute units had all the work).
  const int rest = blockIdx.x / c.heads, items = p.b.seqs * p.row_tiles;
  const int split = rest / items, tile = rest % items % p.row_tiles, seq = rest % items / p.row_tiles;
  const int lane = threadIdx.x % kWave, g = lane / 16, i = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);

  // A lane holds one run of its wavefront's: lane kRuns * e + j run j of its step e, so the runs and scales that a step needs
  // come out of registers. A part begins at a multiple of its length unless a window moves it, so its line of the page table is
  // asked for together with the sequence's bounds.
  static_assert(kMaxRuns == kStreamWaves * kWave, "a lane a run");
  const int mine = (lane / kRuns * kStreamWaves + wave) * kRuns + lane % kRuns;
  const int32_t* const line = p.b.table + static_cast<int64_t>(seq) * p.b.ld_table;
  const int most = p.b.ld_table - 1;
  auto page_of = [&](int64_t token) { return line[min(static_cast<int>(token / c.page), most)]; };
  int page = -1;
  if (most >= 0 && p.window == 0) page = page_of(static_cast<int64_t>(split) * p.chunk + kRun * mine);
  const RowTile t = row_tile(p, seq, tile, kPerTile);
  if (t.count <= 0) return;
  const int64_t start = t.begin + static_cast<int64_t>(split) * p.chunk;
  if (start >= t.end && split > 0) return;
  const bool alone = static_cast<int64_t>(t.begin) + p.chunk >= t.end;  // the only part: the rows are written at once
  const int token0 = static_cast<int>(start), stop = static_cast<int>(min(start + p.chunk, static_cast<int64_t>(t.end)));
  const int runs = (stop - token0 + kRun - 1) / kRun;  // none where the rows see nothing
  const int steps = (runs + kRuns - 1) / kRuns;
  if (p.window > 0 && mine < runs) page = page_of(token0 + kRun * mine);
  int run = -1;  // where the run lies; none, or none of the cache's pages: no tokens
  if (mine < runs && page >= 0 && page < c.pages) run = static_cast<int>((kv8_row(c, page, head) + (token0 + kRun * mine) % c.page) / kRun);
  const int64_t scale_at = static_cast<int64_t>(max(run, 0)) * kRun >> c.block_shift;
  const float ks = c.k_scale[scale_at], vs = c.v_scale[scale_at];
  const int key_off = i * DIM + 16 * g, value_off = 4 * g * DIM + i * (DIM / 16);
  KeyRegs<DIM> keys[kRuns];
  ValueRegs<DIM> values[kRuns];
  auto ask_keys = [&](auto where) {
#pragma unroll
    for (int j = 0; j < kRuns; ++j) load_keys<DIM>(keys[j], c.k + static_cast<int64_t>(max(where(j), 0)) * (kRun * DIM), key_off);
  };
  auto ask_values = [&](auto where) {
#pragma unroll
    for (int j = 0; j < kRuns; ++j) load_values<DIM>(values[j], c.v + static_cast<int64_t>(max(where(j), 0)) * (kRun * DIM), value_off);
  };
  // Everything the first step needs is on its way before anything is waited for; a wavefront without a step reads run 0.
  auto run_in = [&](int e) { return [&, e](int j) { return __builtin_amdgcn_readlane(run, e * kRuns + j); }; };
  ask_keys(run_in(0));
  // The rows' queries: row 16 r + i, dims 64 c + 16 g + 8 h .. + 8 (the key's bytes of the same lane group).
  bf16x8 q[RT][2 * kC];
  int pos[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int flat = t.first + 16 * r + i, token = flat / p.group;
    const bool have = 16 * r + i < t.count;
    pos[r] = t.span.length - t.span.rows + token;
    const int64_t at = have ? (t.span.row0 + token) * p.ld_q + static_cast<int64_t>(head * p.group + flat % p.group) * DIM : 0;
    load_query(p, have, at, [&](int k) { return 64 * (k / 2) + 16 * g + 8 * (k % 2); }, q[r]);
  }
  ask_values(run_in(0));
  // Scales of the runs: of the scores, and of the values (a run that is none may have any there).
  const float key_scale = ks * fabsf(p.scale) * 1.4426950408889634f;
  const float value_log = run >= 0 ? __builtin_amdgcn_logf(fabsf(vs)) : -__builtin_inff();
  const bool whole = !__any(mine < runs && run < 0);
  auto from_lane = [](float v, int from) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), from)); };

  f32x4 acc[RT][kTiles] = {};
  float base[RT], term_base[RT], total[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    base[r] = term_base[r] = kNothing;
    total[r] = 0.0f;
  }
  for (int e = 0, step = wave; step < steps; ++e, step += kStreamWaves) {
    const int at = token0 + step * kStep;
    f32x4 s[RT][kRuns];
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int cc = 0; cc < kC; ++cc)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16x8 a = weight_fragment<F>(keys[j].w[cc], 0, h);
#pragma unroll
          for (int r = 0; r < RT; ++r) s[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[r][2 * cc + h], s[r][j], 0, 0, 0);
        }
    }
    const bool more = step + kStreamWaves < steps;
    if (more) ask_keys(run_in(e + 1));
    // Every token of the step is seen by every row?
    const bool plain = whole && at + kStep - 1 <= t.low_pos && (p.window == 0 || at > static_cast<int64_t>(t.high_pos) - p.window);
    float ks[kRuns], vl[kRuns];
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
      ks[j] = from_lane(key_scale, e * kRuns + j);
      vl[j] = from_lane(value_log, e * kRuns + j);
    }
    if (!plain) {
#pragma unroll
      for (int j = 0; j < kRuns; ++j) {
        const bool there = __builtin_amdgcn_readlane(run, e * kRuns + j) >= 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int token = at + kRun * j + 4 * g + k;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const bool hidden = !there || token > pos[r] || (p.window > 0 && token <= pos[r] - p.window);
            s[r][j][k] = hidden ? -__builtin_inff() : s[r][j][k] * ks[j];
          }
          // Codes of places without a token (NaNs perhaps) times a weight of nothing have to be nothing.
          if (!there || token >= t.span.length)
#pragma unroll
            for (int d = 0; d < kC; ++d) values[j].w[k][d] = 0;
        }
        ks[j] = 1.0f;
      }
    }
    f16x8 terms[RT][kRuns / 2];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float m = -__builtin_inff(), n = m;
#pragma unroll
      for (int j = 0; j < kRuns; ++j) {
        const float most = fmaxf(fmaxf(s[r][j][0], s[r][j][1]), fmaxf(s[r][j][2], s[r][j][3])) * ks[j];
        m = fmaxf(m, most);
        n = fmaxf(n, most + vl[j]);
      }
      if (__any(m > base[r] + kSlack || n > term_base[r] + kSlack)) {
        auto of_row = [](float v) {
          float a, b;
          swap_halves<true>(v, a, b);
          v = fmaxf(a, b);
          swap_halves<false>(v, a, b);
          return fmaxf(a, b);
        };
        m = fmaxf(of_row(m) - kTermBits, base[r]);
        n = fmaxf(of_row(n) - kTermBits, term_base[r]);
        total[r] *= __builtin_amdgcn_exp2f(base[r] - m);
        const float keep = __builtin_amdgcn_exp2f(term_base[r] - n);
#pragma unroll
        for (int f = 0; f < kTiles; ++f) acc[r][f] *= keep;
        base[r] = m;
        term_base[r] = n;
      }
      const float least = kLeastLift - base[r];
#pragma unroll
      for (int j = 0; j < kRuns; j += 2) {
        f16x2 v[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float lift = fmaxf(vl[j + e] - term_base[r], least);
          float w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][j + e][k], ks[j + e], lift));
          v[2 * e] = pack_f16(w[0], w[1]);
          v[2 * e + 1] = pack_f16(w[2], w[3]);
          const float per = __builtin_amdgcn_exp2f(-base[r] - lift);
#pragma unroll
          for (int k = 0; k < 4; ++k) total[r] = __builtin_fmaf(w[k], per, total[r]);
        }
        terms[r][j / 2] = __builtin_bit_cast(f16x8, v);
      }
    }
#pragma unroll
    for (int j = 0; j < kRuns; j += 2)
#pragma unroll
      for (int d = 0; d < kC; ++d) {
        // Dword d of the eight tokens' bytes: [pair of tokens][low, high two dims]
        uint32_t two[4][2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t x = flipped<F>(values[j + e / 2].w[2 * (e % 2)][d]), y = flipped<F>(values[j + e / 2].w[2 * (e % 2) + 1][d]);
          two[e][0] = __builtin_amdgcn_perm(y, x, 0x05010400u);
          two[e][1] = __builtin_amdgcn_perm(y, x, 0x07030602u);
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          f16x2 v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = f % 2 ? pair_of<F, true>(two[e][f / 2]) : pair_of<F, false>(two[e][f / 2]);
          const f16x8 a = __builtin_bit_cast(f16x8, v);
#pragma unroll
          for (int r = 0; r < RT; ++r) acc[r][4 * d + f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, terms[r][j / 2], acc[r][4 * d + f], 0, 0, 0);
        }
      }
    if (more) ask_values(run_in(e + 1));
  }

  // The wavefronts' sums together.
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float a, b;
    swap_halves<true>(total[r], a, b);
    const float w = a + b;
    swap_halves<false>(w, a, b);
    if (g == 0) {
      wave_top[wave][16 * r + i] = base[r];
      wave_sum_of[wave][16 * r + i] = a + b;
    }
  }
  __syncthreads();
  auto row_top = [&](int row) {
    float m = wave_top[0][row];
#pragma unroll
    for (int w = 1; w < kStreamWaves; ++w) m = fmaxf(m, wave_top[w][row]);
    return m;
  };
  float* const part = alone ? nullptr : partial_at<DIM>(p, (static_cast<int64_t>(seq) * p.row_tiles + tile) * c.heads + head, split, kPerTile);
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (16 * r >= t.count) break;
    const int row = 16 * r + i;
    const float m = row_top(row);
    const float root = term_root(term_base[r], m);
    if (r > 0) __syncthreads();
    // Tile f of a lane: dims kTiles * (4 g + e) + f.
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int f = 0; f < kTiles; f += 4) {
        f32x4 v = {acc[r][f][e], acc[r][f + 1][e], acc[r][f + 2][e], acc[r][f + 3][e]};
        *reinterpret_cast<f32x4*>(&sums[wave][i][kTiles * (4 * g + e) + f]) = v * root * root;
      }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * (DIM / 4); e += kStreamThreads) {
      const int local = e / (DIM / 4), d = 4 * (e % (DIM / 4)), row = 16 * r + local;
      if (row >= t.count) continue;
      const float m = row_top(row);
      float sum = 0.0f;
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kStreamWaves; ++w) {
        const float keep = wave_top[w][row] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(wave_top[w][row] - m);
        sum += wave_sum_of[w][row] * keep;
        v += *reinterpret_cast<const f32x4*>(&sums[w][local][d]);
      }
      if (alone) {
        const int flat = t.first + row;
        const int64_t at = (t.span.row0 + flat / p.group) * p.ld_out + static_cast<int64_t>(head * p.group + flat % p.group) * DIM + d;
        store_four(p, at, v * over_weights(sum));
      } else {
        *reinterpret_cast<f32x4*>(part + row * DIM + d) = v;
        if (d == 0) {
          part[kPerTile * DIM + 2 * row] = m;
          part[kPerTile * DIM + 2 * row + 1] = sum;
        }
      }
    }
  }
}

// The parts of one row added up, in a fixed order. A row of one of the cache's heads is DIM / 4 threads; with up to kFewParts
// parts they read them one after another. More parts are dealt out to the 1024 / DIM such groups of a whole workgroup, whose
// sums are then added. (One group over 64 parts took 35 us of a call's 57; a workgroup for each of 48880 rows of two parts 110 of 243.)
constexpr int kFewParts = 8;

template <int DIM>
__global__ void __launch_bounds__(256) combine_kernel(const AttentionArgs p, int per_tile, int rows) {
  constexpr int kLanes = DIM / 4, kGroups = 256 / kLanes, kAtOnce = 4;
  __shared__ float tops[kGroups], sums_of[kGroups];
  __shared__ f32x4 sums[kGroups][kLanes];
  const Kv8Cache& c = p.c;
  const bool few = p.splits <= kFewParts;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int64_t which = few ? static_cast<int64_t>(blockIdx.x) * kGroups + group : blockIdx.x;
  const int row = static_cast<int>(which % rows);
  const int64_t item = which / rows;
  const int head = static_cast<int>(item % c.heads), tile = static_cast<int>(item / c.heads % p.row_tiles);
  const int64_t seq = item / c.heads / p.row_tiles;
  if (few && group >= kGroups) return;  // heads of 192: 16 threads too many
  if (seq >= p.b.seqs) return;
  const RowTile t = row_tile(p, static_cast<int>(seq), tile, per_tile);
  if (row >= t.count || static_cast<int64_t>(t.begin) + p.chunk >= t.end) return;
  const int parts = (t.end - t.begin + p.chunk - 1) / p.chunk;
  const float* const first = partial_at<DIM>(p, item, 0, per_tile);
  const int64_t pitch = static_cast<int64_t>(per_tile) * (DIM + 2);
  const int begin = few ? 0 : group < kGroups ? group : parts, step = few ? 1 : kGroups;
  float m = -__builtin_inff(), sum = 0.0f;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  // Sums and marks (largest score, sum of weights) of kAtOnce parts are asked for together; the last part again for those behind it.
  for (int s = begin; s < parts; s += kAtOnce * step) {
    f32x2 marks[kAtOnce];
    f32x4 data[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const float* const part = first + min(s + k * step, parts - 1) * pitch;
      marks[k] = *reinterpret_cast<const f32x2*>(part + per_tile * DIM + 2 * row);
      data[k] = *reinterpret_cast<const f32x4*>(part + row * DIM + 4 * lane);
    }
    float now = m;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) now = fmaxf(now, marks[k].x);
    const float base = now == -__builtin_inff() ? 0.0f : now, keep = __builtin_amdgcn_exp2f(m - base);
    sum *= keep;
    v *= keep;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const float w = s + k * step < parts ? __builtin_amdgcn_exp2f(marks[k].x - base) : 0.0f;
      sum += marks[k].y * w;
      v += data[k] * w;
    }
    m = now;
  }
  if (!few) {
    if (group < kGroups) {
      sums[group][lane] = v;
      if (lane == 0) {
        tops[group] = m;
        sums_of[group] = sum;
      }
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) m = fmaxf(m, tops[g]);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    sum = 0.0f;
    v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const float w = __builtin_amdgcn_exp2f(tops[g] - base);
      sum += sums_of[g] * w;
      v += sums[g][lane] * w;
    }
  }
  const int flat = t.first + row;
  const int64_t at = (t.span.row0 + flat / p.group) * p.ld_out + static_cast<int64_t>(head * p.group + flat % p.group) * DIM + 4 * lane;
  store_four(p, at, v * over_weights(sum));
}

}  // namespace dro
