// lx_kv8_append: keys and values of a call's rows into the 8-bit paged cache, rotated by their positions on the way (queries
// too), and lx_kv8_dequantize, the cache back as bf16.
//
// A scale belongs to a block of tokens and a head, so the unit of work is one such block as far as this call writes it: its
// largest magnitude has to be known before its first code. Tokens of the block from earlier calls keep their codes while
// their scale still covers the new ones; where it has to grow they are read, rescaled and written again (a block holds 128
// tokens at most).
#include "kv8.h"

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
  int dtype, out_dtype, rot, interleaved, group;
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

// v[0..3] and v[4..7]: the two runs of four, from `at` on.
__device__ __forceinline__ void load_unit(const void* x, int dtype, bool wide, int64_t at, const Unit& n, float* v) {
  if (!wide) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = load_as_f32(x, dtype, at + n.a + j);
      v[4 + j] = load_as_f32(x, dtype, at + n.b + j);
    }
  } else if (dtype == LX_BF16) {
    const uint16_t* const h = static_cast<const uint16_t*>(x) + at;
    const u32x2 lo = *reinterpret_cast<const u32x2*>(h + n.a), hi = *reinterpret_cast<const u32x2*>(h + n.b);
    decode_dword<LX_W_BF16>(lo.x, v);
    decode_dword<LX_W_BF16>(lo.y, v + 2);
    decode_dword<LX_W_BF16>(hi.x, v + 4);
    decode_dword<LX_W_BF16>(hi.y, v + 6);
  } else {
    const float* const f = static_cast<const float*>(x) + at;
    const f32x4 lo = *reinterpret_cast<const f32x4*>(f + n.a), hi = *reinterpret_cast<const f32x4*>(f + n.b);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = lo[j];
      v[4 + j] = hi[j];
    }
  }
}

__device__ __forceinline__ void store_unit(void* x, int dtype, bool wide, int64_t at, const Unit& n, const float* v) {
  if (wide && dtype == LX_BF16) {
    uint16_t* const h = static_cast<uint16_t*>(x) + at;
    auto two = [&](int j) { return f32_to_bf16_bits(v[j]) | static_cast<uint32_t>(f32_to_bf16_bits(v[j + 1])) << 16; };
    *reinterpret_cast<u32x2*>(h + n.a) = u32x2{two(0), two(2)};
    *reinterpret_cast<u32x2*>(h + n.b) = u32x2{two(4), two(6)};
  } else if (wide) {
    float* const f = static_cast<float*>(x) + at;
    *reinterpret_cast<f32x4*>(f + n.a) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(f + n.b) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      store_from_f32(x, dtype, at + n.a + j, v[j]);
      store_from_f32(x, dtype, at + n.b + j, v[4 + j]);
    }
  }
}

// The cosines and sines of a unit's four angles position * freq. The product of a 31-bit and a 24-bit number is right to
// 2^-53 in 64 bits; whole turns are taken off it there, in two steps, so what is left of a far position is as good as of a
// near one. The rest r is split into an f32 and what that lacks: cos(r + e) = cos r - e sin r.
__device__ __forceinline__ void angles(const float* freq, int pair, int position, float* c, float* s) {
  constexpr double kTurn = 6.283185307179586477, kTurnRest = 2.4492935982947064e-16, kPerTurn = 0.15915494309189533577;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double angle = static_cast<double>(position) * static_cast<double>(freq[pair + j]);
    const double turns = rint(angle * kPerTurn);
    const double r = fma(-turns, kTurnRest, fma(-turns, kTurn, angle));
    const float near = static_cast<float>(r), rest = static_cast<float>(r - static_cast<double>(near));
    float sin_near, cos_near;
    sincosf(near, &sin_near, &cos_near);
    c[j] = __builtin_fmaf(-rest, sin_near, cos_near);
    s[j] = __builtin_fmaf(rest, cos_near, sin_near);
  }
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

// Which sequence row r belongs to, or -1: the sequences' bounds are looked at by all threads at once.
template <int kThreads>
__device__ int sequence_of(const Kv8Batch& b, int r, int* found) {
  if (!b.rows) return r < b.seqs ? r : -1;
  __syncthreads();
  if (threadIdx.x == 0) *found = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < b.seqs; s += kThreads) {
    const int first = clamp_int(b.rows[s], 0, b.T), end = clamp_int(b.rows[s + 1], 0, b.T);
    if (r >= first && r < end) *found = s;
  }
  __syncthreads();
  return *found;
}

// blockIdx.x: rows; blockIdx.y: the cache's head, whose query heads it rotates too.
template <int F, int kThreads>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs p) {
  constexpr float kTop = F == LX_W_INT8 ? 127.0f : 448.0f;
  __shared__ int found;
  __shared__ float tops[2][kThreads / kWave];
  const Kv8Cache& c = p.c;
  const int dim = c.dim, units = dim / 8, slots = kThreads / units;
  const int slot = threadIdx.x / units, head = blockIdx.y;
  const bool busy = slot < slots;
  const Unit n = unit_of(p, threadIdx.x % units);
  const int pair = 4 * (threadIdx.x % units);
  const int stop = min(p.b.T, static_cast<int>(blockIdx.x + 1) * p.rows_per_group);
  for (int r = blockIdx.x * p.rows_per_group; r < stop;) {
    const int s = sequence_of<kThreads>(p.b, r, &found);
    if (s < 0) {
      ++r;
      continue;
    }
    const Kv8Span span = kv8_span(p.b, c.page, s);
    const Kv8Piece piece = kv8_piece(span, c.block_shift, r);
    if (!piece.own) {
      r = piece.next;
      continue;
    }
    const int lead = span.length - span.rows, position = piece.position, begin = piece.begin, end = piece.end, next = piece.next;
    const int page = kv8_page(c, p.b, s, begin);
    float c4[4], s4[4], k8[8], v8[8], top_k = 0.0f, top_v = 0.0f;
    auto keys = [&](int t) {
      const int64_t row = span.row0 + (t - lead);
      load_unit(p.k, p.dtype, p.wide, row * p.ld_k + head * dim, n, k8);
      load_unit(p.v, p.dtype, p.wide, row * p.ld_v + head * dim, n, v8);
      if (n.turned) {
        angles(p.freq, pair, t, c4, s4);
        turn(p.interleaved, c4, s4, k8);
      }
    };
    for (int t = position + slot; busy && t < end; t += slots) {
      keys(t);
      top_k = top_of(k8, top_k);
      top_v = top_of(v8, top_v);
      if (p.q) {
        const int64_t row = span.row0 + (t - lead);
        for (int g = 0; g < p.group; ++g) {
          const int at = (head * p.group + g) * dim;
          float q8[8];
          load_unit(p.q, p.dtype, p.wide, row * p.ld_q + at, n, q8);
          if (n.turned) turn(p.interleaved, c4, s4, q8);
          store_unit(p.q_out, p.out_dtype, p.wide, row * p.ld_out + at, n, q8);
        }
      }
    }
    if (page >= 0) {
      top_k = wave_max(top_k);
      top_v = wave_max(top_v);
      __syncthreads();
      if (threadIdx.x % kWave == 0) {
        tops[0][threadIdx.x / kWave] = top_k;
        tops[1][threadIdx.x / kWave] = top_v;
      }
      const int64_t row0 = kv8_row(c, page, head) + begin % c.page;  // the block's first token row
      const int64_t at = row0 >> c.block_shift;
      float* const scales[2] = {const_cast<float*>(c.k_scale) + at, const_cast<float*>(c.v_scale) + at};
      const bool kept = position > begin;
      const float old[2] = {kept ? *scales[0] : 0.0f, kept ? *scales[1] : 0.0f};
      __syncthreads();
      float scale[2], inverse[2];
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        float top = tops[part][0];
#pragma unroll
        for (int w = 1; w < kThreads / kWave; ++w) top = fmaxf(top, tops[part][w]);
        scale[part] = top > 0.0f ? fmaxf(top / kTop, 0x1p-126f) : 0.0f;
        // Every thread has read the old scales before the barrier; one writes the new ones.
        scale[part] = fmaxf(scale[part], old[part]);
        inverse[part] = scale[part] > 0.0f ? 1.0f / scale[part] : 0.0f;
        if (threadIdx.x == 0) *scales[part] = scale[part];
        uint8_t* const codes = const_cast<uint8_t*>(part ? c.v : c.k) + row0 * dim;
        if (scale[part] > old[part]) {  // the tokens that stay: none where kept is false
          const float factor = old[part] / scale[part];
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
      for (int t = position + slot; busy && t < end; t += slots) {
        keys(t);
        const int64_t row = (row0 + (t - begin)) * dim;
        uint8_t* const kc = const_cast<uint8_t*>(c.k) + row;
        uint8_t* const vc = const_cast<uint8_t*>(c.v) + row;
        *reinterpret_cast<uint32_t*>(kc + n.a) = encode_four<F>(k8, inverse[0]);
        *reinterpret_cast<uint32_t*>(kc + n.b) = encode_four<F>(k8 + 4, inverse[0]);
        *reinterpret_cast<uint32_t*>(vc + n.a) = encode_four<F>(v8, inverse[1]);
        *reinterpret_cast<uint32_t*>(vc + n.b) = encode_four<F>(v8 + 4, inverse[1]);
      }
    }
    r = next;
  }
}

// Sixteen codes a thread: 16 bytes in, 32 out.
template <int F>
__global__ void __launch_bounds__(256) dequantize_cache_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scale,
                                                               uint16_t* __restrict__ out, int64_t pieces, int pieces_per_block_row,
                                                               int block_shift) {
  const int64_t i = blockIdx.x * static_cast<int64_t>(256) + threadIdx.x;
  if (i >= pieces) return;
  const u32x4 w = reinterpret_cast<const u32x4*>(codes)[i];
  const float s = scale[i / pieces_per_block_row >> block_shift];
  u32x4 out4[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float v[4];
    const uint32_t d = w[j];
    decode_dword<F>(d, v);
    out4[j / 2][2 * (j & 1)] = f32_to_bf16_bits(v[0] * s) | static_cast<uint32_t>(f32_to_bf16_bits(v[1] * s)) << 16;
    out4[j / 2][2 * (j & 1) + 1] = f32_to_bf16_bits(v[2] * s) | static_cast<uint32_t>(f32_to_bf16_bits(v[3] * s)) << 16;
  }
  reinterpret_cast<u32x4*>(out)[2 * i] = out4[0];
  reinterpret_cast<u32x4*>(out)[2 * i + 1] = out4[1];
}

bool aligned(const void* p, int64_t ld, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (dtype == LX_BF16 ? 2 : 4) % 16 == 0;
}

// Rows a workgroup looks at: about as many as a sequence has, so that about one block begins there, up to a block's.
int rows_per_group(int block, int seqs, int T) {
  int n = 1;
  while (n < block && 2 * n <= T / (seqs > 0 ? seqs : 1)) n *= 2;
  return n;
}

template <int F>
int append(const AppendArgs& p, hipStream_t stream) {
  const dim3 grid((p.b.T + p.rows_per_group - 1) / p.rows_per_group, p.c.heads);
  hipLaunchKernelGGL((append_kernel<F, 256>), grid, dim3(256), 0, stream, p);
  return status_of(hipGetLastError());
}

}  // namespace
}  // namespace dro

using namespace dro;

extern "C" {

int lx_kv8_append(const lx_kv8* cache, const lx_kv8_batch* batch, const void* q, const void* k, const void* v, lx_dtype dtype, int ld_q,
                  int ld_k, int ld_v, void* q_out, lx_dtype q_out_dtype, int ld_q_out, const float* freq, int rot, int interleaved, int T,
                  int q_heads, void* stream) {
  if (int st = kv8_check_cache(cache)) return fail(st);
  if (int st = kv8_check_batch(batch, T)) return fail(st);
  if ((dtype != LX_F32 && dtype != LX_BF16) || (q && q_out_dtype != LX_F32 && q_out_dtype != LX_BF16)) return fail(kInvalid);
  if (rot < 0 || rot > cache->dim || rot % 8 != 0) return fail(kInvalid);
  if (T == 0 || batch->seqs == 0) return kOk;
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
  p.group = q ? q_heads / cache->heads : 0;
  p.wide = aligned(k, ld_k, dtype) && aligned(v, ld_v, dtype) && (!q || (aligned(q, ld_q, dtype) && aligned(q_out, ld_q_out, q_out_dtype)));
  p.rows_per_group = rows_per_group(cache->block, batch->seqs, T);
  hipStream_t s = as_stream(stream);
  return cache->type == LX_W_INT8 ? append<LX_W_INT8>(p, s) : append<LX_W_FP8>(p, s);
}

int lx_kv8_dequantize(const lx_kv8* cache, void* k, void* v, void* stream) {
  if (int st = kv8_check_cache(cache)) return fail(st);
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 != 0) return fail(kInvalid);
  const Kv8Cache c = kv8_cache(*cache);
  const int64_t pieces = static_cast<int64_t>(c.pages) * c.heads * c.page * (c.dim / 16);
  if ((pieces + 255) / 256 > 0x7fffffff) return fail(kInvalid);
  const dim3 grid(static_cast<unsigned>((pieces + 255) / 256));
  for (int part = 0; part < 2; ++part) {
    void* const out = part ? v : k;
    if (!out) continue;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, as_stream(stream), part ? c.v : c.k, part ? c.v_scale : c.k_scale,
                         static_cast<uint16_t*>(out), pieces, c.dim / 16, c.block_shift);
    };
    if (cache->type == LX_W_INT8) go(dequantize_cache_kernel<LX_W_INT8>);
    else go(dequantize_cache_kernel<LX_W_FP8>);
    if (int st = status_of(hipGetLastError())) return st;
  }
  return kOk;
}

// For tests, on host memory and without a device: what the kernel makes of a call's rows. Every piece that it stores, as
// {sequence, first token, its page or -1, tokens, first row}, `capacity` of them at most; returns how many there are.
LX_API int dromos_kv8_pieces(const lx_kv8* cache, const lx_kv8_batch* batch, int T, int* out, int capacity) {
  if (kv8_check_cache(cache) || kv8_check_batch(batch, T)) return -1;
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
      const Kv8Piece piece = kv8_piece(kv8_span(b, c.page, s), c.block_shift, r);
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
