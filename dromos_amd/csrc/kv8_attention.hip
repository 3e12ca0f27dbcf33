// lx_kv8_attention: softmax attention of a call's rows over the 8-bit paged cache. The kernels are in kv8_stream.h (few rows a sequence)
// and kv8_tile.h (many).
#include "kv8_tile.h"

namespace dro {
namespace {

// How a call is cut up: from the host's numbers alone, so that a captured call does not depend on what the device holds.
struct Plan {
  bool tiles;          // kv8_tile.h's kernel
  int per_tile;        // rows of a tile
  int row_tiles;       // tiles a sequence
  int tile_rows;       // rows of its fullest tile
  int splits, chunk;
  int64_t workgroups, combiners;  // of the attention, and of the sums of its parts
  bool fits;                      // the device can be asked for that many
};

// Whether `rows` rows (tokens times query heads of a head of the cache) are taken in tiles of 128 by kv8_tile.h's kernel. Below 97
// rows a sequence tiles of 32 rows that stream the cache (again from L2 for each) are ahead: 8 streams of up to 8191
// tokens at 40 / 64 / 96 / 128 rows 41.3 / 42.1 / 50.3 / 62.8 us, in tiles of 128 rows 47.6 / 48.9 / 52.1 / 54.3. Sums of 32 rows of
// heads wider than 128 leave the tile kernel's wavefronts too few registers
// (2048 rows of 16 heads of 256 behind 2048 tokens: 246 us against 352; 260 with sums of unrounded terms).
bool in_tiles(int64_t rows, int dim) { return rows > 96 && dim <= 128; }

// Heads of 256 leave no registers for the sums of 32 rows.
int rows_per_tile(int64_t rows, int dim) { return in_tiles(rows, dim) ? kTileRowsOfGroup : rows <= 16 || dim == 256 ? 16 : 32; }

// Tiles with rows, of all heads: no more than T fills, and one begun for each sequence.
int64_t busy_tiles(int64_t seqs, int64_t row_tiles, int per, int heads, int64_t T, int group) {
  const int64_t items = seqs * row_tiles * heads, filled = (T * group / per + seqs) * heads;
  return items < filled ? items : filled;
}

// One part where there is a workgroup a unit. Tiles of 128 rows need a quarter more: a unit with one of them alone is half idle
// (1024 rows behind 7168 tokens, 264 workgroups: 208 us, in two parts 152).
bool one_part(int64_t busy, bool tiles, int units) { return 4 * busy >= (tiles ? 5 : 4) * units; }

// One sequence's parts are equally long. Several are of different lengths (which only the device knows): twice as many parts
// then even out what the compute units have, 16 streams of up to 8192 tokens 41 -> 38 us, 8 of exactly 8192 33 -> 34. Rows in
// two tiles of sixteen leave room for two workgroups a unit only: 8 streams of 5 rows 28.7 us, with twice the parts 34.8.
int64_t parts_wanted(int64_t busy, bool tiles, int64_t seqs, int per, int units) {
  const int each = seqs > 1 && per == 16 ? 4 : 2;
  return busy <= 0 || one_part(busy, tiles, units) ? 1 : (each * units + busy - 1) / busy;
}

int64_t tokens_held(const lx_kv8& c, const lx_kv8_batch& b) {
  const int64_t held = static_cast<int64_t>(b.ld_table) * c.page;
  return held < b.max_length ? held : b.max_length;
}

// Enough parts that the device has about two workgroups a compute unit, none shorter than 256 tokens (a step of each
// wavefront); one part where sequences and heads alone make a workgroup a unit.
Plan plan_for(const lx_kv8& c, const lx_kv8_batch& b, int T, int q_heads, int window) {
  Plan p{};
  const int group = q_heads / c.heads;
  const int64_t most = b.max_rows < T ? b.max_rows : T;
  const int64_t rows = most * group;
  p.tiles = in_tiles(rows, c.dim);
  p.per_tile = rows_per_tile(rows, c.dim);
  const int per = p.per_tile;
  const int64_t row_tiles = (rows + per - 1) / per, limit = kMaxGridThreads / 256;
  if (row_tiles > limit || row_tiles * b.seqs > limit || row_tiles * b.seqs * c.heads > limit) return p;
  p.row_tiles = static_cast<int>(row_tiles);
  p.tile_rows = static_cast<int>(rows < per ? rows : per);
  // What a tile's rows see: all tokens, or the window, the tile's own and the run that the window begins in.
  int64_t length = tokens_held(c, b);
  const int64_t windowed = static_cast<int64_t>(window) + per / group + 2 + kRun;
  if (window > 0 && windowed < length) length = windowed;
  const int64_t items = static_cast<int64_t>(b.seqs) * p.row_tiles * c.heads;
  const int64_t want = parts_wanted(busy_tiles(b.seqs, p.row_tiles, per, c.heads, T, group), p.tiles, b.seqs, per, compute_units());
  int64_t chunk = (length + want - 1) / want;
  chunk = (chunk + 255) / 256 * 256;
  // Parts cost a second kernel (about 4 us); one part costs a step of each wavefront more for every 256 tokens (1.6 us).
  if (length <= 768) chunk = 768;
  if (chunk < 256) chunk = 256;
  if (chunk > kMaxRuns * kRun && !p.tiles) chunk = kMaxRuns * kRun;
  if (p.tiles && want <= 1) chunk = 0x7fffff00;
  p.chunk = static_cast<int>(chunk);
  p.splits = static_cast<int>((length + chunk - 1) / chunk);
  if (p.splits < 1) p.splits = 1;
  p.workgroups = items * p.splits;
  const int64_t combined = items * p.tile_rows, each_time = p.splits <= kFewParts ? 1024 / c.dim : 1;
  p.combiners = p.splits > 1 ? (combined + each_time - 1) / each_time : 0;
  p.fits = p.workgroups <= limit && p.combiners <= limit;
  return p;
}

// Bytes of partial sums of `row_tiles` tiles of `per` rows a sequence at most, whatever the window: it may have as many parts as are
// wanted of 256 tokens, or of the longest there are.
int64_t partial_bytes(int64_t seqs, int64_t row_tiles, int per, bool tiles, int heads, int dim, int64_t whole, int64_t want) {
  const int64_t runs = (whole + 255) / 256, longest = (whole + kMaxRuns * kRun - 1) / (kMaxRuns * kRun);
  int64_t parts = want < runs ? want : runs;
  if (!tiles && parts < longest) parts = longest;
  return parts > 1 ? seqs * row_tiles * heads * parts * per * (dim + 2) * static_cast<int64_t>(sizeof(float)) : 0;
}

// The workspace of a call and of every smaller one: fewer rows or sequences fill fewer compute units, are cut into more parts for
// it, and may leave more partial sums than the call itself. From one part on those only grow with rows and sequences; in front of
// that there are few numbers of tiles and sequences to look at (about as many tiles, of all heads and sequences, as compute units).
int64_t workspace_for(const lx_kv8& c, const lx_kv8_batch& b, int T, int q_heads) {
  const int group = q_heads / c.heads, units = compute_units();
  const int64_t rows = static_cast<int64_t>(b.max_rows < T ? b.max_rows : T) * group, whole = tokens_held(c, b), limit = kMaxGridThreads / 256;
  int64_t most = 0;
  // The rows that have tiles of one height, from the last on.
  for (int64_t last = rows, first; last > 0; last = first - 1) {
    const int per = rows_per_tile(last, c.dim);
    const bool tiles = in_tiles(last, c.dim);
    first = tiles ? 97 : per == 32 ? 17 : 1;
    // n tiles a sequence, in calls of as few rows as have them. Whether one part is enough.
    auto look_at = [&](int64_t seqs, int64_t n) {
      const int64_t least = n * per - per + 1 > first ? n * per - per + 1 : first;
      const int64_t busy = busy_tiles(seqs, n, per, c.heads, (least + group - 1) / group, group);
      if (n <= limit && n * seqs <= limit && n * seqs * c.heads <= limit) {
        const int64_t bytes = partial_bytes(seqs, n, per, tiles, c.heads, c.dim, whole, parts_wanted(busy, tiles, seqs, per, units));
        most = bytes > most ? bytes : most;
      }
      return one_part(busy, tiles, units);
    };
    const int64_t most_tiles = (last + per - 1) / per;
    for (int64_t n = (first + per - 1) / per; n <= most_tiles;) {
      const bool alone = look_at(1, n);
      bool enough = alone;
      for (int64_t seqs = 2; seqs <= b.seqs && !enough; ++seqs) enough = look_at(seqs, n);
      look_at(b.seqs, n);
      n = alone && n < most_tiles ? most_tiles : n + 1;
    }
  }
  return most;
}

template <int F, int DIM>
int stream(const AttentionArgs& a, const Plan& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.workgroups));
  if (p.tiles) {
    if constexpr (DIM <= 128) {
      allow_lds(reinterpret_cast<const void*>(&tile_kernel<F, DIM>), tile_lds_bytes<DIM>());
      hipLaunchKernelGGL((tile_kernel<F, DIM>), grid, dim3(256), tile_lds_bytes<DIM>(), s, a);
    }
  } else if (p.per_tile == 16) {
    hipLaunchKernelGGL((stream_kernel<F, DIM, 1>), grid, dim3(kStreamThreads), 0, s, a);
  } else {
    if constexpr (DIM < 256) hipLaunchKernelGGL((stream_kernel<F, DIM, 2>), grid, dim3(kStreamThreads), 0, s, a);
  }
  if (int st = status_of(hipGetLastError())) return st;
  if (p.splits == 1) return kOk;
  hipLaunchKernelGGL((combine_kernel<DIM>), dim3(static_cast<unsigned>(p.combiners)), dim3(256), 0, s, a, p.per_tile, p.tile_rows);
  return status_of(hipGetLastError());
}

template <int F>
int attention(const AttentionArgs& a, const Plan& p, hipStream_t s) {
  switch (a.c.dim) {
    case 64: return stream<F, 64>(a, p, s);
    case 128: return stream<F, 128>(a, p, s);
    case 192: return stream<F, 192>(a, p, s);
    default: return stream<F, 256>(a, p, s);
  }
}

}  // namespace
}  // namespace dro

using namespace dro;

extern "C" {

int lx_kv8_attention(const void* q, lx_dtype q_dtype, int ld_q, const lx_kv8* cache, const lx_kv8_batch* batch, void* out,
                     lx_dtype out_dtype, int ld_out, int T, int q_heads, float scale, int window, void* workspace, void* stream) {
  if (int st = kv8_check_cache(cache)) return fail(st);
  if (int st = kv8_check_batch(batch, T, *cache)) return fail(st);
  if ((q_dtype != LX_F32 && q_dtype != LX_BF16) || (out_dtype != LX_F32 && out_dtype != LX_BF16) || window < 0) return fail(kInvalid);
  if (q_heads < 1 || q_heads > 65536 || q_heads % cache->heads != 0) return fail(kInvalid);
  if (T == 0 || batch->seqs == 0 || batch->max_rows == 0) return kOk;
  const int64_t width = static_cast<int64_t>(q_heads) * cache->dim;
  if (!q || !out || (T > 1 && (ld_q < width || ld_out < width))) return fail(kInvalid);
  const Plan plan = plan_for(*cache, *batch, T, q_heads, window);
  if (!plan.fits || (plan.splits > 1 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))) return fail(kInvalid);
  AttentionArgs a{};
  a.c = kv8_cache(*cache);
  a.b = kv8_batch(*batch, T);
  a.q = q, a.out = out, a.partial = static_cast<float*>(workspace), a.ld_q = ld_q, a.ld_out = ld_out;
  a.q_dtype = q_dtype, a.out_dtype = out_dtype, a.group = q_heads / cache->heads, a.scale = scale;
  a.window = window >= batch->max_length ? 0 : window;  // none sees as far
  a.wide_q = q_dtype == LX_BF16 && reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld_q % 8 == 0;
  a.wide_out = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ld_out % 4 == 0;
  a.fold = batch->seqs == 1 && plan.workgroups <= 2 * compute_units();
  a.row_tiles = plan.row_tiles, a.splits = plan.splits, a.chunk = plan.chunk;
  return cache->type == LX_W_INT8 ? attention<LX_W_INT8>(a, plan, as_stream(stream)) : attention<LX_W_FP8>(a, plan, as_stream(stream));
}

int64_t lx_kv8_attention_workspace_bytes(const lx_kv8* cache, const lx_kv8_batch* batch, int T, int q_heads) {
  if (kv8_check_cache(cache) || kv8_check_batch(batch, T, *cache) || T == 0 || batch->seqs == 0 || batch->max_rows == 0) return 0;
  if (q_heads < 1 || q_heads > 65536 || q_heads % cache->heads != 0) return 0;
  return workspace_for(*cache, *batch, T, q_heads);
}

// For tests, without a device (256 compute units): {rows of a tile, tiles a sequence, parts, tokens of a part, workgroups, partial
// sums' bytes, the workspace's bytes} of a call. Returns 0, or the status that the call is refused with.
LX_API int dromos_kv8_plan(const lx_kv8* cache, const lx_kv8_batch* batch, int T, int q_heads, int window, int64_t* out) {
  if (int st = kv8_check_cache(cache)) return st;
  if (int st = kv8_check_batch(batch, T, *cache)) return st;
  const Plan p = plan_for(*cache, *batch, T, q_heads, window);
  if (!p.fits) return kInvalid;
  out[0] = p.per_tile, out[1] = p.row_tiles, out[2] = p.splits, out[3] = p.chunk, out[4] = p.workgroups;
  out[5] = p.splits > 1 ? p.workgroups * p.per_tile * (cache->dim + 2) * static_cast<int64_t>(sizeof(float)) : 0;
  out[6] = lx_kv8_attention_workspace_bytes(cache, batch, T, q_heads);
  return kOk;
}

}  // extern "C"
