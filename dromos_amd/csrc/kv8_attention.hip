// lx_kv8_attention: softmax attention of a call's rows over the 8-bit paged cache.
#include "kv8.h"

namespace dro {
namespace {

struct AttentionArgs {
  Kv8Cache c;
  Kv8Batch b;
  const void* q;
  void* out;
  int64_t ld_q, ld_out;
  int q_dtype, out_dtype, group, window;
  float scale;
};

// A wavefront a row and query head: 64 tokens at a time, a lane scoring one token, then a lane adding up four values of the head.
template <int F>
__global__ void __launch_bounds__(64) attention_simple_kernel(const AttentionArgs p) {
  __shared__ float weight[kWave];
  __shared__ float query[256];
  const Kv8Cache& c = p.c;
  const int lane = threadIdx.x, row = blockIdx.x, q_head = blockIdx.y, head = q_head / p.group, dim = c.dim;
  int seq = -1;
  for (int s = 0; s < p.b.seqs && seq < 0; ++s) {
    const Kv8Span span = kv8_span(p.b, c.page, s);
    if (row >= span.row0 && row < span.row0 + span.rows) seq = s;
  }
  if (seq < 0) return;
  const Kv8Span span = kv8_span(p.b, c.page, seq);
  for (int d = lane; d < dim; d += kWave) {
    const float v = load_as_f32(p.q, p.q_dtype, row * p.ld_q + static_cast<int64_t>(q_head) * dim + d);
    query[d] = bf16_bits_to_f32(f32_to_bf16_bits(v));
  }
  __syncthreads();
  const int last = span.length - span.rows + (row - span.row0);
  const int first = p.window > 0 && last >= p.window ? last - p.window + 1 : 0;
  float top = -__builtin_inff(), sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int t0 = first; t0 <= last; t0 += kWave) {
    const int t = t0 + lane;
    const int page = t <= last ? kv8_page(c, p.b, seq, t) : -1;
    const int64_t at = page >= 0 ? kv8_row(c, page, head) + t % c.page : -1;
    float s = -__builtin_inff();
    if (at >= 0) {
      float dot = 0.0f;
      for (int d = 0; d < dim; d += 4) {
        float v[4];
        decode_dword<F>(*reinterpret_cast<const uint32_t*>(c.k + at * dim + d), v);
#pragma unroll
        for (int j = 0; j < 4; ++j) dot = __builtin_fmaf(v[j], query[d + j], dot);
      }
      s = dot * c.k_scale[at >> c.block_shift] * p.scale;
    }
    const float now = fmaxf(top, wave_max(s));
    if (now == -__builtin_inff()) continue;
    const float keep = expf(top - now), e = expf(s - now);
    sum = sum * keep + wave_sum(e);
    top = now;
    __syncthreads();
    weight[lane] = at >= 0 ? e * c.v_scale[at >> c.block_shift] : 0.0f;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] *= keep;
    for (int i = 0; i < kWave; ++i) {
      const int64_t other = __shfl(at, i);
      if (other < 0) continue;
      if (4 * lane < dim) {
        float v[4];
        decode_dword<F>(*reinterpret_cast<const uint32_t*>(c.v + other * dim + 4 * lane), v);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(weight[i], v[j], acc[j]);
      }
    }
  }
  if (4 * lane >= dim) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    store_from_f32(p.out, p.out_dtype, row * p.ld_out + static_cast<int64_t>(q_head) * dim + 4 * lane + j, sum > 0.0f ? acc[j] / sum : 0.0f);
}

}  // namespace
}  // namespace dro

using namespace dro;

extern "C" {

int lx_kv8_attention(const void* q, lx_dtype q_dtype, int ld_q, const lx_kv8* cache, const lx_kv8_batch* batch, void* out,
                     lx_dtype out_dtype, int ld_out, int T, int q_heads, float scale, int window, void* workspace, void* stream) {
  if (int st = kv8_check_cache(cache)) return fail(st);
  if (int st = kv8_check_batch(batch, T)) return fail(st);
  if ((q_dtype != LX_F32 && q_dtype != LX_BF16) || (out_dtype != LX_F32 && out_dtype != LX_BF16) || window < 0) return fail(kInvalid);
  if (q_heads < 1 || q_heads > 65536 || q_heads % cache->heads != 0) return fail(kInvalid);
  if (T == 0 || batch->seqs == 0) return kOk;
  const int64_t width = static_cast<int64_t>(q_heads) * cache->dim;
  if (!q || !out || (T > 1 && (ld_q < width || ld_out < width))) return fail(kInvalid);
  AttentionArgs p{};
  p.c = kv8_cache(*cache);
  p.b = kv8_batch(*batch, T);
  p.q = q, p.out = out, p.ld_q = ld_q, p.ld_out = ld_out;
  p.q_dtype = q_dtype, p.out_dtype = out_dtype, p.group = q_heads / cache->heads, p.window = window, p.scale = scale;
  (void)workspace;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(T, q_heads), dim3(kWave), 0, as_stream(stream), p); };
  if (cache->type == LX_W_INT8) go(attention_simple_kernel<LX_W_INT8>);
  else go(attention_simple_kernel<LX_W_FP8>);
  return status_of(hipGetLastError());
}

int64_t lx_kv8_attention_workspace_bytes(const lx_kv8* cache, const lx_kv8_batch* batch, int T, int q_heads) {
  if (kv8_check_cache(cache) || kv8_check_batch(batch, T) || T == 0 || batch->seqs == 0 || q_heads < 1) return 0;
  return 0;
}

}  // extern "C"
