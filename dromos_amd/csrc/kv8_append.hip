// lx_kv8_append: keys and values of a call's rows into the 8-bit paged cache, rotated by their positions on the way (queries
// too), and lx_kv8_dequantize, the cache back as bf16.
//
// A scale belongs to a block of tokens and a head, so the unit of work is one such block as far as this call writes it: its
// largest magnitude has to be known before its first code. A workgroup reads it once and holds it in registers (a lane has
// eight values of a token's head, up to four tokens). Tokens of the block from earlier calls keep their codes while their scale
// still covers the new ones; where it has to grow they are read, rescaled and written again (a block holds 128 tokens at most).
// Queries are turned by workgroups of their own, four heads each, so that a model with few heads in its cache has enough of them.
//
// A prompt is bound by bytes. A single token is bound by the latency of what it has to follow: the rows' bounds and lengths (every
// wavefront looks through them by itself), the page table, the block's scale; its values are asked for before the first of them.
#include "kv8.h"
#include "rotation.h"
#include "tile_mfma.h"

namespace dro {
namespace {

struct AppendArgs {
  Kv8Cache c;
  Kv8Batch b;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  const float* freq;
  int64_t ld_q, ld_k, ld_v, ld_out;
  int dtype, out_dtype, rot, interleaved, q_heads;
  int tokens;          // of a block that a call writes at most
  unsigned queries;    // the first workgroup that turns queries
  int query_rows;      // rows of one of those
  int rows_per_group;  // rows a workgroup looks at for blocks that begin there
  int wide;            // q, k, v and q_out can be moved 16 (bf16) or 32 (f32) bytes at a time
};

// A lane's eight values of a head: four pairs that a rotation turns. Where the pairs are (i, i + rot / 2) they lie in two
// runs of four, otherwise in one run of eight.
struct Unit {
  int a, b;  // first value of either run of four
  bool turned;
};

__device__ __forceinline__ Unit unit_of(const AppendArgs& p, int u) {
  Unit n;
  const int pair = 4 * u;
  n.turned = pair < p.rot / 2;
  const bool split = n.turned && !p.interleaved;
  n.a = split ? pair : 2 * pair;
  n.b = split ? pair + p.rot / 2 : 2 * pair + 4;
  return n;
}

// The eight values as they lie in memory: bf16 (HALF: where they can be moved 8 bytes at a time), or f32.
template <bool HALF>
struct RawUnit {
  u32x4 w[HALF ? 1 : 2];
};

template <bool HALF>
__device__ __forceinline__ RawUnit<HALF> load_unit(const void* x, int dtype, bool wide, int64_t at, const Unit& n) {
  RawUnit<HALF> r;
  if constexpr (HALF) {
    const uint16_t* const h = static_cast<const uint16_t*>(x) + at;
    const u32x2 lo = *reinterpret_cast<const u32x2*>(h + n.a), hi = *reinterpret_cast<const u32x2*>(h + n.b);
    r.w[0] = u32x4{lo.x, lo.y, hi.x, hi.y};
  } else if (wide) {
    const float* const f = static_cast<const float*>(x) + at;
    r.w[0] = *reinterpret_cast<const u32x4*>(f + n.a);
    r.w[1] = *reinterpret_cast<const u32x4*>(f + n.b);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.w[0][j] = __float_as_uint(load_as_f32(x, dtype, at + n.a + j));
      r.w[1][j] = __float_as_uint(load_as_f32(x, dtype, at + n.b + j));
    }
  }
  return r;
}

// v[0 .. 3] and v[4 .. 7]: the two runs of four.
template <bool HALF>
__device__ __forceinline__ void values_of(const RawUnit<HALF>& r, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (HALF) {
      const uint32_t two = r.w[0][j / 2];
      v[j] = __uint_as_float(j % 2 ? two & 0xffff0000u : two << 16);
    } else {
      const uint32_t one = r.w[j / 4][j % 4];
      v[j] = __uint_as_float(one);
    }
  }
}

// Stored past the caches that the attention's other XCDs do not share (4096 rows 29.8 -> 28.2 us, 2048 of heads of 256 19.8 -> 17.3).
template <bool HALF>
__device__ __forceinline__ void store_unit(void* x, int dtype, bool wide, int64_t at, const Unit& n, const float* v) {
  if (HALF || wide) {
    if (dtype == LX_BF16) {
      uint16_t* const h = static_cast<uint16_t*>(x) + at;
      auto two = [&](int j) { return __builtin_bit_cast(uint32_t, pack_bf16(v[j], v[j + 1])); };
      __builtin_nontemporal_store(u32x2{two(0), two(2)}, reinterpret_cast<u32x2*>(h + n.a));
      __builtin_nontemporal_store(u32x2{two(4), two(6)}, reinterpret_cast<u32x2*>(h + n.b));
    } else {
      float* const f = static_cast<float*>(x) + at;
      __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(f + n.a));
      __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, reinterpret_cast<f32x4*>(f + n.b));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      store_from_f32(x, dtype, at + n.a + j, v[j]);
      store_from_f32(x, dtype, at + n.b + j, v[4 + j]);
    }
  }
}

// Quarter turns a position of a unit's four frequencies.
__device__ __forceinline__ void quarters_of(const AppendArgs& p, const Unit& n, int pair, double (&quarters)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) quarters[j] = n.turned ? static_cast<double>(p.freq[pair + j]) * 0.63661977236758134308 : 0.0;
}

__device__ __forceinline__ void turn(bool interleaved, const float* c, const float* s, float* v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int x = interleaved ? 2 * j : j, y = interleaved ? 2 * j + 1 : 4 + j;
    const float a = v[x], b = v[y];
    v[x] = a * c[j] - b * s[j];
    v[y] = b * c[j] + a * s[j];
  }
}

// The largest magnitude that is a number (neither infinite nor a NaN).
__device__ __forceinline__ float top_of(const float* v, float top) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float m = fabsf(v[j]);
    top = fmaxf(top, m < __builtin_inff() ? m : 0.0f);
  }
  return top;
}

// Four codes as a dword. A NaN becomes 0: a code that is no number would reach rows that do not see its token, as nothing
// times a NaN on the matrix cores.
template <int F>
__device__ __forceinline__ uint32_t encode_four(const float* v, float inverse) {
  float c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    c[j] = v[j] * inverse;
    c[j] = c[j] == c[j] ? c[j] : 0.0f;
  }
  if constexpr (F == LX_W_FP8) {
    return e4m3_encode_four(c);
  } else {
    uint32_t d = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) d |= (static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(rintf(c[j]), -127.0f), 127.0f))) & 0xffu) << (8 * j);
    return d;
  }
}

// The sequence row r belongs to, or -1, and its rows and length: a lane a sequence, in every wavefront by itself.
__device__ __forceinline__ int sequence_of(const Kv8Batch& b, int page, int r, Kv8Span& span) {
  if (!b.rows) {
    if (r >= b.seqs) return -1;
    span = kv8_span_of(b, page, r, r + 1, b.lengths[r]);
    return r;
  }
  const int lane = threadIdx.x % kWave;
  for (int base = 0; base < b.seqs; base += kWave) {
    const int s = min(base + lane, b.seqs - 1);
    const int from = b.rows[s], to = b.rows[s + 1], length = b.lengths[s];
    const uint64_t here = __ballot(base + lane < b.seqs && r >= clamp_int(from, 0, b.T) && r < clamp_int(to, 0, b.T));
    if (here) {
      const int l = __builtin_ctzll(here);
      span = kv8_span_of(b, page, __builtin_amdgcn_readlane(from, l), __builtin_amdgcn_readlane(to, l), __builtin_amdgcn_readlane(length, l));
      return base + l;
    }
  }
  return -1;
}

constexpr int kQueryHeads = 4;  // of a workgroup that turns queries

// The queries of rows first .. stop - 1 (no more than the workgroup has slots), heads q_head .. q_head + heads - 1. A thread's slot is
// a row, whose angles it makes once for all heads, or (where a workgroup has one row) a head. What it turns is asked for before
// its row's place is looked up.
template <int kThreads, bool HALF>
__device__ __forceinline__ void turn_queries(const AppendArgs& p, int first, int stop, int q_head, int heads) {
  const int dim = p.c.dim, units = dim / 8, slots = kThreads / units, slot = threadIdx.x / units;
  const bool one = stop - first == 1;
  const int base = one ? slot : 0, step = one ? slots : 1, row = one ? first : first + slot;
  const Unit n = unit_of(p, threadIdx.x % units);
  double quarters[4];
  quarters_of(p, n, 4 * (threadIdx.x % units), quarters);
  RawUnit<HALF> raw[kQueryHeads];
  const int64_t at = static_cast<int64_t>(q_head) * dim;
#pragma unroll
  for (int k = 0; k < kQueryHeads; ++k) {
    if (k > 0 && k * step >= heads) break;
    raw[k] = load_unit<HALF>(p.q, p.dtype, p.wide, min(row, p.b.T - 1) * p.ld_q + at + min(base + k * step, heads - 1) * dim, n);
  }
  int position = -1;
  for (int r = first; r < stop;) {
    Kv8Span span;
    if (sequence_of(p.b, p.c.page, r, span) < 0) {
      ++r;
      continue;
    }
    const int end = min(stop, span.row0 + span.rows);
    if (row >= r && row < end && row - span.row0 < p.b.max_rows) position = span.length - span.rows + (row - span.row0);
    r = end;
  }
  if (position < 0 || slot >= slots) return;
  float c4[4], s4[4];
  angles(quarters, position, c4, s4);
#pragma unroll
  for (int k = 0; k < kQueryHeads; ++k) {
    const int head = base + k * step;
    if (head >= heads) break;
    float q8[8];
    values_of(raw[k], q8);
    if (n.turned) turn(p.interleaved, c4, s4, q8);
    store_unit<HALF>(p.q_out, p.out_dtype, p.wide, row * p.ld_out + at + head * dim, n, q8);
    __builtin_amdgcn_sched_barrier(0);  // one head after another: all at once take 210 registers
  }
}

// The first workgroups are some rows and one of the cache's heads each, those behind them (from `queries` on) some rows and four
// query heads. P: tokens of a block that a thread holds values of.
template <int F, int kThreads, int P, bool HALF>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs p) {
  constexpr float kTop = F == LX_W_INT8 ? 127.0f : 448.0f;
  __shared__ float tops[2][kThreads / kWave];
  const Kv8Cache& c = p.c;
  if (blockIdx.x >= p.queries) {
    const unsigned fours = (p.q_heads + kQueryHeads - 1) / kQueryHeads, which = blockIdx.x - p.queries;
    const int q_head = which % fours * kQueryHeads, from = which / fours * p.query_rows;
    turn_queries<kThreads, HALF>(p, from, min(p.b.T, from + p.query_rows), q_head, min(kQueryHeads, p.q_heads - q_head));
    return;
  }
  const int first = blockIdx.x / c.heads * p.rows_per_group, stop = min(p.b.T, first + p.rows_per_group);
  const int dim = c.dim, units = dim / 8, slots = kThreads / units, slot = threadIdx.x / units, head = blockIdx.x % c.heads;
  const bool busy = slot < slots;
  const Unit n = unit_of(p, threadIdx.x % units);
  const int pair = 4 * (threadIdx.x % units);
  double quarters[4];
  quarters_of(p, n, pair, quarters);
  RawUnit<HALF> keys[P], values[P];
  auto ask = [&](int row0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (i > 0 && i * slots >= p.tokens) break;
      const int64_t row = min(row0 + slot + i * slots, p.b.T - 1);
      keys[i] = load_unit<HALF>(p.k, p.dtype, p.wide, row * p.ld_k + head * dim, n);
      values[i] = load_unit<HALF>(p.v, p.dtype, p.wide, row * p.ld_v + head * dim, n);
    }
  };
  const bool early = p.rows_per_group == 1;  // the row is likely to begin a piece
  if (early) ask(first);
  for (int r = first; r < stop;) {
    Kv8Span span;
    const int s = sequence_of(p.b, c.page, r, span);
    if (s < 0) {
      ++r;
      continue;
    }
    const Kv8Piece piece = kv8_piece(span, p.b.max_rows, c.block_shift, r);
    if (!piece.own) {
      r = piece.next;
      continue;
    }
    const int position = piece.position, begin = piece.begin, tokens = piece.end - piece.position;
    if (!early) ask(r);
    const int page = kv8_page(c, p.b, s, begin);
    r = piece.next;
    if (page < 0) continue;
    const int64_t row0 = kv8_row(c, page, head) + begin % c.page;  // the block's first token row
    float* const scales[2] = {const_cast<float*>(c.k_scale) + (row0 >> c.block_shift), const_cast<float*>(c.v_scale) + (row0 >> c.block_shift)};
    const bool kept = position > begin;
    const float held[2] = {*scales[0], *scales[1]};
    const float old[2] = {kept ? held[0] : 0.0f, kept ? held[1] : 0.0f};
    float k8[P][8], top[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float v8[8];
      values_of(keys[i], k8[i]);
      values_of(values[i], v8);
      const int token = slot + i * slots;
      if (busy && token < tokens) {
        if (n.turned) {
          float c4[4], s4[4];
          angles(quarters, position + token, c4, s4);
          turn(p.interleaved, c4, s4, k8[i]);
        }
        top[0] = top_of(k8[i], top[0]);
        top[1] = top_of(v8, top[1]);
      }
    }
#pragma unroll
    for (int part = 0; part < 2; ++part) top[part] = wave_max(top[part]);
    // The barriers also part the scales as every thread has read them from those that one writes.
    __syncthreads();
    if (threadIdx.x % kWave == 0) {
      tops[0][threadIdx.x / kWave] = top[0];
      tops[1][threadIdx.x / kWave] = top[1];
    }
    __syncthreads();
    float inverse[2];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      float most = tops[part][0];
#pragma unroll
      for (int w = 1; w < kThreads / kWave; ++w) most = fmaxf(most, tops[part][w]);
      const float scale = fmaxf(most > 0.0f ? fmaxf(most / kTop, 0x1p-126f) : 0.0f, old[part]);
      inverse[part] = scale > 0.0f ? 1.0f / scale : 0.0f;
      if (threadIdx.x == 0) *scales[part] = scale;
      if (scale > old[part]) {  // the tokens that stay: none where kept is false
        uint8_t* const codes = const_cast<uint8_t*>(part ? c.v : c.k) + row0 * dim;
        const float factor = old[part] / scale;
        for (int i = threadIdx.x; i < (position - begin) * units; i += kThreads) {
          u32x2* const word = reinterpret_cast<u32x2*>(codes) + i;
          const u32x2 was = *word;
          float v[8];
          decode_dword<F>(was.x, v);
          decode_dword<F>(was.y, v + 4);
          *word = u32x2{encode_four<F>(v, factor), encode_four<F>(v + 4, factor)};
        }
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int token = slot + i * slots;
      if (!busy || token >= tokens) continue;
      float v8[8];
      values_of(values[i], v8);
      const int64_t row = (row0 + (position - begin) + token) * dim;
      uint8_t* const kc = const_cast<uint8_t*>(c.k) + row;
      uint8_t* const vc = const_cast<uint8_t*>(c.v) + row;
      *reinterpret_cast<uint32_t*>(kc + n.a) = encode_four<F>(k8[i], inverse[0]);
      *reinterpret_cast<uint32_t*>(kc + n.b) = encode_four<F>(k8[i] + 4, inverse[0]);
      *reinterpret_cast<uint32_t*>(vc + n.a) = encode_four<F>(v8, inverse[1]);
      *reinterpret_cast<uint32_t*>(vc + n.b) = encode_four<F>(v8 + 4, inverse[1]);
    }
  }
}

// Sixteen codes a thread: 16 bytes in, 32 out; keys, then values. What one grid line does not hold goes to the next. Stored past the caches
// (4288 tokens of 8 heads of 128 7.4 -> 6.5 us, 6336 of them 11.4 -> 9.5).
template <int F>
__global__ void __launch_bounds__(256) dequantize_cache_kernel(const Kv8Cache c, uint16_t* k, uint16_t* v, int64_t pieces) {
  const int64_t i = (blockIdx.z * static_cast<int64_t>(gridDim.x) + blockIdx.x) * 256 + threadIdx.x;
  const bool values = blockIdx.y == 1;
  uint16_t* const out = values ? v : k;
  if (i >= pieces || !out) return;
  const u32x4 w = reinterpret_cast<const u32x4*>(values ? c.v : c.k)[i];
  const int per_row = c.dim / 16;
  // A head's pieces of a row are few: no division of 64 bits by what is no power of two but 192 / 16.
  const int64_t row = per_row == 12 ? i / 12 : i >> (per_row == 4 ? 2 : per_row == 8 ? 3 : 4);
  const float s = (values ? c.v_scale : c.k_scale)[row >> c.block_shift];
  u32x4 out4[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x[4];
    const uint32_t d = w[j];
    decode_dword<F>(d, x);
    out4[j / 2][2 * (j & 1)] = __builtin_bit_cast(uint32_t, pack_bf16(x[0] * s, x[1] * s));
    out4[j / 2][2 * (j & 1) + 1] = __builtin_bit_cast(uint32_t, pack_bf16(x[2] * s, x[3] * s));
  }
  __builtin_nontemporal_store(out4[0], reinterpret_cast<u32x4*>(out) + 2 * i);
  __builtin_nontemporal_store(out4[1], reinterpret_cast<u32x4*>(out) + 2 * i + 1);
}

bool aligned(const void* p, int64_t ld, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (dtype == LX_BF16 ? 2 : 4) % 16 == 0;
}

// Rows a workgroup looks at. Short sequences: one, which mostly begins a piece or goes with the one before it (8 sequences of 5 rows
// by fours: 10.6 us, workgroups that look for several sequences one after another; one by one: 7). Longer ones: about as
// many as a sequence has, up to a block's, so that about one piece begins there.
int rows_per_group(int block, int seqs, int T) {
  const int each = T / (seqs > 0 ? seqs : 1);
  int n = 1;
  while (each >= 16 && n < block && 2 * n <= each) n *= 2;
  return n;
}

template <int F, int kThreads, int P, bool HALF>
int launch(AppendArgs p, hipStream_t stream) {
  const int slots = kThreads / (p.c.dim / 8);
  p.query_rows = p.rows_per_group < slots ? p.rows_per_group : slots;
  const int64_t keys = static_cast<int64_t>((p.b.T + p.rows_per_group - 1) / p.rows_per_group) * p.c.heads;
  const int64_t queries = static_cast<int64_t>((p.b.T + p.query_rows - 1) / p.query_rows) * ((p.q_heads + kQueryHeads - 1) / kQueryHeads);
  if ((keys + queries) * kThreads > kMaxGridThreads) return fail(kInvalid);
  p.queries = static_cast<unsigned>(keys);
  hipLaunchKernelGGL((append_kernel<F, kThreads, P, HALF>), dim3(static_cast<unsigned>(keys + queries)), dim3(kThreads), 0, stream, p);
  return status_of(hipGetLastError());
}

// The fewest threads that hold a block's part in P tokens each.
template <int F, bool HALF>
int append(const AppendArgs& p, hipStream_t stream) {
  const int units = p.c.dim / 8;
  if (p.tokens <= 64 / units) return launch<F, 64, 1, HALF>(p, stream);
  if (p.tokens <= 2 * (256 / units)) return launch<F, 256, 2, HALF>(p, stream);
  if (p.tokens <= 4 * (512 / units)) return launch<F, 512, 4, HALF>(p, stream);
  return launch<F, 1024, 4, HALF>(p, stream);
}

}  // namespace
}  // namespace dro

using namespace dro;

extern "C" {

int lx_kv8_append(const lx_kv8* cache, const lx_kv8_batch* batch, const void* q, const void* k, const void* v, lx_dtype dtype, int ld_q,
                  int ld_k, int ld_v, void* q_out, lx_dtype q_out_dtype, int ld_q_out, const float* freq, int rot, int interleaved, int T,
                  int q_heads, void* stream) {
  if (int st = kv8_check_cache(cache)) return fail(st);
  if (int st = kv8_check_batch(batch, T, *cache)) return fail(st);
  if ((dtype != LX_F32 && dtype != LX_BF16) || (q && q_out_dtype != LX_F32 && q_out_dtype != LX_BF16)) return fail(kInvalid);
  if (rot < 0 || rot > cache->dim || rot % 8 != 0) return fail(kInvalid);
  if (T == 0 || batch->seqs == 0 || batch->max_rows == 0) return kOk;
  if (!k || !v || (rot > 0 && !freq) || !q != !q_out) return fail(kInvalid);
  const int64_t kv = static_cast<int64_t>(cache->heads) * cache->dim, width = static_cast<int64_t>(q_heads) * cache->dim;
  if (q && (q_heads < 1 || q_heads % cache->heads != 0 || q_heads > 65536)) return fail(kInvalid);
  if (T > 1 && (ld_k < kv || ld_v < kv || (q && (ld_q < width || ld_q_out < width)))) return fail(kInvalid);
  AppendArgs p{};
  p.c = kv8_cache(*cache);
  p.b = kv8_batch(*batch, T);
  p.q = q, p.k = k, p.v = v, p.q_out = q_out, p.freq = freq;
  p.ld_q = ld_q, p.ld_k = ld_k, p.ld_v = ld_v, p.ld_out = ld_q_out;
  p.dtype = dtype, p.out_dtype = q_out_dtype, p.rot = rot, p.interleaved = interleaved != 0;
  p.q_heads = q ? q_heads : 0;
  p.wide = aligned(k, ld_k, dtype) && aligned(v, ld_v, dtype) && (!q || (aligned(q, ld_q, dtype) && aligned(q_out, ld_q_out, q_out_dtype)));
  p.tokens = p.b.max_rows < cache->block ? p.b.max_rows : cache->block;
  p.rows_per_group = rows_per_group(cache->block, batch->seqs, T);
  hipStream_t s = as_stream(stream);
  const bool half = p.wide && dtype == LX_BF16;
  if (cache->type == LX_W_INT8) return half ? append<LX_W_INT8, true>(p, s) : append<LX_W_INT8, false>(p, s);
  return half ? append<LX_W_FP8, true>(p, s) : append<LX_W_FP8, false>(p, s);
}

int lx_kv8_dequantize(const lx_kv8* cache, void* k, void* v, void* stream) {
  if (int st = kv8_check_cache(cache)) return fail(st);
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 != 0) return fail(kInvalid);
  const Kv8Cache c = kv8_cache(*cache);
  const int64_t pieces = static_cast<int64_t>(c.pages) * c.heads * c.page * (c.dim / 16);
  if (!k && !v) return kOk;
  const int64_t groups = (pieces + 255) / 256, line = groups < (1 << 23) ? groups : 1 << 23;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(line), 2, static_cast<unsigned>((groups + line - 1) / line)), dim3(256), 0, as_stream(stream), c,
                       static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), pieces);
  };
  if (cache->type == LX_W_INT8) go(dequantize_cache_kernel<LX_W_INT8>);
  else go(dequantize_cache_kernel<LX_W_FP8>);
  return status_of(hipGetLastError());
}

// For tests, on host memory and without a device: what the kernel makes of a call's rows. Every piece that it stores, as
// {sequence, first token, its page or -1, tokens, first row}, `capacity` of them at most; returns how many there are.
LX_API int dromos_kv8_pieces(const lx_kv8* cache, const lx_kv8_batch* batch, int T, int* out, int capacity) {
  if (kv8_check_cache(cache) || kv8_check_batch(batch, T, *cache)) return -1;
  const Kv8Cache c = kv8_cache(*cache);
  const Kv8Batch b = kv8_batch(*batch, T);
  const int per = rows_per_group(cache->block, batch->seqs, T);
  int n = 0;
  for (int first = 0; first < T; first += per) {
    for (int r = first; r < T && r < first + per;) {
      int s = -1;
      for (int i = 0; i < b.seqs && s < 0; ++i) {
        const Kv8Span span = kv8_span(b, c.page, i);
        if (r >= span.row0 && r < span.row0 + span.rows) s = i;
      }
      if (s < 0) {
        ++r;
        continue;
      }
      const Kv8Piece piece = kv8_piece(kv8_span(b, c.page, s), b.max_rows, c.block_shift, r);
      if (piece.own) {
        const int five[5] = {s, piece.position, kv8_page(c, b, s, piece.begin), piece.end - piece.position, r};
        for (int i = 0; i < 5 && n < capacity; ++i) out[5 * n + i] = five[i];
        ++n;
      }
      r = piece.next;
    }
  }
  return n;
}

}  // extern "C"
