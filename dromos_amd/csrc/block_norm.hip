// lx_block_norm: what stands between two blocks of a layer. The block's output goes through its norm, gate and scale into the
// residual stream, and the sum through the norm in front of the next block, in one pass over the row.
//
// Bytes decide: y, h and the gate are read once, h and x written once, and a row stays in its workgroup's registers between
// (four vectors of eight values a thread at most, 32768 values a row). A workgroup takes one row. Its sums are f32: a
// thread's values in order, then a wavefront's tree, then the wavefronts in order, so a row's bits depend on its width only.
#include "common.h"

namespace dro {
namespace {

constexpr int kMaxWidth = 32768;

struct NormArgs {
  const void* y;
  const void* post_w;
  const void* post_b;
  const void* gate;
  const void* h;
  void* h_out;
  const void* w;
  const void* b;
  void* x;
  int64_t ld_y, ld_gate, ld_h, ld_x;
  int y_type, h_type, w_type, x_type;
  float alpha, beta, eps;
  int H;
  int layer;
};

// V consecutive values.
template <int V>
__device__ __forceinline__ void load_values(const void* p, int type, int64_t i, float* v) {
  if constexpr (V == 1) {
    v[0] = load_as_f32(p, type, i);
  } else if (type == LX_BF16) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t d = w[j];
      decode_dword<LX_W_BF16>(d, v + 2 * j);
    }
  } else {
    const f32x4* const q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
    const f32x4 lo = q[0], hi = q[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = lo[j];
      v[4 + j] = hi[j];
    }
  }
}

template <int V>
__device__ __forceinline__ void store_values(void* p, int type, int64_t i, const float* v) {
  if constexpr (V == 1) {
    store_from_f32(p, type, i, v[0]);
  } else if (type == LX_BF16) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = f32_to_bf16_bits(v[2 * j]) | static_cast<uint32_t>(f32_to_bf16_bits(v[2 * j + 1])) << 16;
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) = w;
  } else {
    f32x4* const q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + i);
    q[0] = f32x4{v[0], v[1], v[2], v[3]};
    q[1] = f32x4{v[4], v[5], v[6], v[7]};
  }
}

template <int kThreads>
__device__ __forceinline__ float row_sum(float v, float* shared) {
  v = wave_sum(v);
  if constexpr (kThreads == kWave) return v;
  __syncthreads();
  if (threadIdx.x % kWave == 0) shared[threadIdx.x / kWave] = v;
  __syncthreads();
  float s = shared[0];
#pragma unroll
  for (int i = 1; i < kThreads / kWave; ++i) s += shared[i];
  return s;
}

// v <- (v - mean) / sqrt(mean of squares + eps) * w (+ b); the mean only where `layer`. Values behind the row are not touched.
template <int kThreads, int V, int N>
__device__ __forceinline__ void norm_row(const NormArgs& a, const void* w, const void* b, float (&v)[N][V], float* shared) {
  const float per = 1.0f / static_cast<float>(a.H);
  if (a.layer) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (static_cast<int>(i * kThreads + threadIdx.x) * V < a.H)
#pragma unroll
        for (int j = 0; j < V; ++j) s += v[i][j];
    const float mean = row_sum<kThreads>(s, shared) * per;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] -= mean;
  }
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (static_cast<int>(i * kThreads + threadIdx.x) * V < a.H)
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[i][j] * v[i][j];
  const float f = 1.0f / sqrtf(row_sum<kThreads>(s, shared) * per + a.eps);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * kThreads + threadIdx.x) * V;
    if (at < a.H) {
      float u[V];
      load_values<V>(w, a.w_type, at, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = v[i][j] * f * u[j];
      if (b) {
        load_values<V>(b, a.w_type, at, u);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] += u[j];
      }
    }
  }
}

// V: 8 where every row and vector can be moved 16 bytes at a time, otherwise 1. N: vectors of a thread.
template <int kThreads, int V, int N>
__global__ void __launch_bounds__(kThreads) block_norm_kernel(const NormArgs a) {
  __shared__ float shared[kThreads / kWave];
  const int64_t row = blockIdx.x;
  float v[N][V];
  if (a.y) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (i * kThreads + threadIdx.x) * V;
      if (at < a.H) load_values<V>(a.y, a.y_type, row * a.ld_y + at, v[i]);
    }
    if (a.post_w) norm_row<kThreads, V, N>(a, a.post_w, a.post_b, v, shared);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (i * kThreads + threadIdx.x) * V;
      if (at >= a.H) continue;
      float u[V];
      if (a.gate) {
        load_values<V>(a.gate, a.y_type, row * a.ld_gate + at, u);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] *= u[j];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] *= a.alpha;
      if (a.beta != 0.0f) {
        load_values<V>(a.h, a.h_type, row * a.ld_h + at, u);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = a.beta * u[j] + v[i][j];
      }
      store_values<V>(a.h_out, a.h_type, row * a.ld_h + at, v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (i * kThreads + threadIdx.x) * V;
      if (at < a.H) load_values<V>(a.h, a.h_type, row * a.ld_h + at, v[i]);
    }
  }
  if (!a.w) return;
  norm_row<kThreads, V, N>(a, a.w, a.b, v, shared);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * kThreads + threadIdx.x) * V;
    if (at < a.H) store_values<V>(a.x, a.x_type, row * a.ld_x + at, v[i]);
  }
}

bool aligned(const void* p, int64_t ld, int type) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (type == LX_BF16 ? 2 : 4) % 16 == 0;
}

// The fewest threads that hold the row in N vectors each.
template <int V, int N>
int launch(const NormArgs& a, int T, hipStream_t s) {
  const dim3 grid(T);
  const int per = (a.H + V * N - 1) / (V * N);
  if (per <= 64) hipLaunchKernelGGL((block_norm_kernel<64, V, N>), grid, dim3(64), 0, s, a);
  else if (per <= 256) hipLaunchKernelGGL((block_norm_kernel<256, V, N>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((block_norm_kernel<1024, V, N>), grid, dim3(1024), 0, s, a);
  return status_of(hipGetLastError());
}

}  // namespace
}  // namespace dro

using namespace dro;

extern "C" {

int lx_block_norm(lx_norm norm, const void* y, lx_dtype y_dtype, int ld_y, const void* post_weight, const void* post_bias,
                  const void* gate, int ld_gate, float alpha, float beta, const void* h, void* h_out, lx_dtype h_dtype, int ld_h,
                  const void* weight, const void* bias, lx_dtype w_dtype, void* x, lx_dtype x_dtype, int ld_x, float eps, int T, int H,
                  void* stream) {
  if (norm != LX_NORM_RMS && norm != LX_NORM_LAYER) return fail(kInvalid);
  if (T < 0 || H < 0 || H > kMaxWidth) return fail(kInvalid);
  if (T == 0 || H == 0) return kOk;
  auto known = [](lx_dtype t) { return t == LX_F32 || t == LX_BF16; };
  if (!known(h_dtype) || (y && !known(y_dtype)) || (weight && !known(x_dtype))) return fail(kInvalid);
  if ((weight || (y && post_weight)) && !known(w_dtype)) return fail(kInvalid);
  if (y ? !h_out || (beta != 0.0f && !h) : !h || !weight) return fail(kInvalid);
  if (weight && !x) return fail(kInvalid);
  if (T > 1 && (ld_h < H || (y && ld_y < H) || (weight && ld_x < H) || (y && gate && ld_gate != 0 && ld_gate < H))) return fail(kInvalid);
  NormArgs a{};
  a.y = y;
  a.post_w = y ? post_weight : nullptr, a.post_b = a.post_w ? post_bias : nullptr;
  a.gate = y ? gate : nullptr;
  a.h = h, a.h_out = h_out;
  a.w = weight, a.b = weight ? bias : nullptr, a.x = x;
  a.ld_y = ld_y, a.ld_gate = ld_gate, a.ld_h = ld_h, a.ld_x = ld_x;
  a.y_type = y_dtype, a.h_type = h_dtype, a.w_type = w_dtype, a.x_type = x_dtype;
  a.alpha = alpha, a.beta = beta, a.eps = eps, a.H = H, a.layer = norm == LX_NORM_LAYER;
  const bool wide = H % 8 == 0 && aligned(y, ld_y, y_dtype) && aligned(a.gate, a.gate ? ld_gate : 0, y_dtype) &&
                    aligned(y && beta == 0.0f ? nullptr : h, ld_h, h_dtype) && aligned(y ? h_out : nullptr, ld_h, h_dtype) &&
                    aligned(a.post_w, 0, w_dtype) && aligned(a.post_b, 0, w_dtype) && aligned(a.w, 0, w_dtype) &&
                    aligned(a.b, 0, w_dtype) && aligned(weight ? x : nullptr, weight ? ld_x : 0, x_dtype);
  hipStream_t s = as_stream(stream);
  if (wide) return H <= 8192 ? launch<8, 1>(a, T, s) : H <= 16384 ? launch<8, 2>(a, T, s) : launch<8, 4>(a, T, s);
  return H <= 8192 ? launch<1, 8>(a, T, s) : launch<1, 32>(a, T, s);
}

}  // extern "C"
