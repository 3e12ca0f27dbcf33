// lx_block_norm: what stands between two blocks of a layer. The block's output goes through its norm, gate and scale into the
// residual stream, and the sum through the norm in front of the next block, in one pass over the row.
//
// Bytes decide: y, h and the gate are read once, h and x written once, and a row stays in its workgroup's registers between
// (four vectors of eight values a thread at most, 32768 values a row). A workgroup takes one row. Sums are f32, in
// an order that goes by the width and by whether all rows and vectors can be moved 16 bytes at a time, and with it a row's bits: they
// do not depend on how many rows there are.
#include "tile_mfma.h"

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
  int64_t row0;
  int H;
  int layer;
};

// V consecutive values as they lie in memory: eight bf16 (in `low`) or f32, or one value as f32.
template <int V>
struct Raw {
  u32x4 low, high;
};
template <>
struct Raw<1> {
  float v;
};

// `in`: whether there are such values; eight are asked for in any case (i is inside the row then too).
template <int V>
__device__ __forceinline__ Raw<V> load_raw(const void* p, int type, int64_t i, bool in) {
  Raw<V> r;
  if constexpr (V == 1) {
    r.v = in ? load_as_f32(p, type, i) : 0.0f;
  } else if (type == LX_BF16) {
    r.low = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
    r.high = r.low;
  } else {
    const u32x4* const q = reinterpret_cast<const u32x4*>(static_cast<const float*>(p) + i);
    r.low = q[0];
    r.high = q[1];
  }
  return r;
}

template <int V>
__device__ __forceinline__ void values_of(const Raw<V>& r, int type, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = r.v;
  } else {
    const bool half = type == LX_BF16;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t two = r.low[j / 2], four = r.low[2 + j / 2], low = r.low[j], high = r.high[j];
      v[j] = __uint_as_float(half ? (j % 2 ? two & 0xffff0000u : two << 16) : low);
      v[4 + j] = __uint_as_float(half ? (j % 2 ? four & 0xffff0000u : four << 16) : high);
    }
  }
}

// Stored past the caches that the next kernel's other XCDs do not share (8192 rows of 4096: 74 -> 63 us).
template <int V>
__device__ __forceinline__ void store_values(void* p, int type, int64_t i, const float* v) {
  if constexpr (V == 1) {
    store_from_f32(p, type, i, v[0]);
  } else if (type == LX_BF16) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = __builtin_bit_cast(uint32_t, pack_bf16(v[2 * j], v[2 * j + 1]));
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i));
  } else {
    f32x4* const q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + i);
    __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, q);
    __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, q + 1);
  }
}

// The row's sum, in every thread: of a thread's vectors (`parts` holds a sum of each, or one of all four), then a wavefront's
// tree, then the wavefronts in order, first those of every thread's first vector: one vector in 1024 threads and two in 512
// give the same bits. Wavefronts that are none have left zeros in `shared` (a loop over the others would wait for one read
// after another, 59 -> 68 us on 4096 rows of 8192).
template <int P>
__device__ __forceinline__ float row_sum(const float (&parts)[P], float* shared) {
  const int waves = blockDim.x / kWave;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float v = wave_sum(parts[i]);
    if (threadIdx.x % kWave == 0) shared[i * waves + threadIdx.x / kWave] = v;
  }
  __syncthreads();
  f32x4 w[4 * P];
#pragma unroll
  for (int i = 0; i < 4 * P; ++i) w[i] = reinterpret_cast<const f32x4*>(shared)[i];
  float s = w[0][0];
#pragma unroll
  for (int i = 1; i < 16 * P; ++i) s += w[i / 4][i % 4];
  return s;
}

// v <- (v - mean) / sqrt(mean of squares + eps) * w (+ b); the mean only where `layer`. Vectors behind the row count as zeros.
// weight(i, u): the weights of vector i.
template <int V, int N, typename Weight>
__device__ __forceinline__ void norm_row(const NormArgs& a, Weight weight, const void* b, const bool (&in)[N], const int (&at)[N], float (&v)[N][V],
                                         float* shared) {
  const float per = 1.0f / static_cast<float>(a.H);
  constexpr int P = V * N == 16 ? 2 : 1;
  if (a.layer) {
    float s[P] = {};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s[i % P] += in[i] ? v[i][j] : 0.0f;
    const float mean = row_sum<P>(s, shared) * per;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] -= mean;
  }
  float s[P] = {};
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) s[i % P] += in[i] ? v[i][j] * v[i][j] : 0.0f;
  const float f = 1.0f / sqrtf(row_sum<P>(s, shared) * per + a.eps);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float u[V];
    weight(i, u);
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = v[i][j] * f * u[j];
    if (b) {
      values_of<V>(load_raw<V>(b, a.w_type, at[i], in[i]), a.w_type, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] += u[j];
    }
    if (V == 1 && N == 32 && i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // no more reads ahead than registers
  }
}

// V: 8 where every row and vector can be moved 16 bytes at a time, otherwise 1. N: vectors of a thread. Eight wavefronts a SIMD
// where a thread has one: what is on its way at once comes from them (with every input of a row asked for first, in 72 registers
// and five wavefronts, 4096 rows of 8192 took 84 us instead of 58).
template <int V, int N>
__global__ void __launch_bounds__(1024, V * N == 32 ? 4 : 8) block_norm_kernel(const NormArgs a) {
  __shared__ __attribute__((aligned(16))) float shared[32];
  if (threadIdx.x < 32) shared[threadIdx.x] = 0.0f;
  const int64_t row = a.row0 + blockIdx.x;
  bool in[N];
  int at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    at[i] = static_cast<int>(i * blockDim.x + threadIdx.x) * V;
    in[i] = at[i] < a.H;
    at[i] = in[i] ? at[i] : 0;  // read again, not used
  }
  const bool reads_h = !a.y || a.beta != 0.0f;
  float v[N][V];
  if (a.y) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      values_of<V>(load_raw<V>(a.y, a.y_type, row * a.ld_y + at[i], in[i]), a.y_type, v[i]);
    }
    if (a.post_w)
      norm_row<V, N>(a, [&](int i, float (&u)[V]) __attribute__((always_inline)) {
        values_of<V>(load_raw<V>(a.post_w, a.w_type, at[i], in[i]), a.w_type, u);
      }, a.post_b, in, at, v, shared);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float u[V];
    if (!a.y) {
      values_of<V>(load_raw<V>(a.h, a.h_type, row * a.ld_h + at[i], in[i]), a.h_type, v[i]);
      continue;
    }
    if (a.gate) {
      values_of<V>(load_raw<V>(a.gate, a.y_type, row * a.ld_gate + at[i], in[i]), a.y_type, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] *= u[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] *= a.alpha;
    if (reads_h) {
      values_of<V>(load_raw<V>(a.h, a.h_type, row * a.ld_h + at[i], in[i]), a.h_type, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = a.beta * u[j] + v[i][j];
    }
    if (in[i]) store_values<V>(a.h_out, a.h_type, row * a.ld_h + at[i], v[i]);
    if (V == 1 && N == 32 && i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // no more reads ahead than registers
  }
  if (!a.w) return;
  norm_row<V, N>(a, [&](int i, float (&u)[V]) __attribute__((always_inline)) {
    values_of<V>(load_raw<V>(a.w, a.w_type, at[i], in[i]), a.w_type, u);
  }, a.b, in, at, v, shared);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (in[i]) store_values<V>(a.x, a.x_type, row * a.ld_x + at[i], v[i]);
}

bool aligned(const void* p, int64_t ld, int type) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (type == LX_BF16 ? 2 : 4) % 16 == 0;
}

// Rows that cannot be moved 16 bytes at a time are read a value a lane: 4096 rows of 8191 values 159 us, of 8192 51. Four vectors a
// thread (more than 16384 values) leave four wavefronts a SIMD: 1024 rows of 32768 63 us, 2048 of 16384 52.
// As many threads as the row has vectors for N each, up to 1024; of single values half as many each where there are threads for it.
template <int V, int N>
int launch(NormArgs a, int T, hipStream_t s) {
  constexpr int kEach = V == 1 ? N / 2 : V * N;
  const int wanted = ((a.H + kEach - 1) / kEach + kWave - 1) / kWave * kWave, threads = wanted < 1024 ? wanted : 1024;
  const int most = static_cast<int>(kMaxGridThreads / threads);  // rows of a launch
  for (int row = 0; row < T; row += most) {
    a.row0 = row;
    hipLaunchKernelGGL((block_norm_kernel<V, N>), dim3(T - row < most ? T - row : most), dim3(threads), 0, s, a);
    if (int st = status_of(hipGetLastError())) return st;
    if (T - row <= most) break;
  }
  return kOk;
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
  // Two vectors a thread where there are rows for four workgroups a compute unit (8192 rows of 4096: 62.5 -> 57 us; 512 rows 6.6 -> 9.2).
  if (wide) return H <= 8192 && (H <= 2048 || T < 4 * compute_units()) ? launch<8, 1>(a, T, s) : H <= 16384 ? launch<8, 2>(a, T, s) : launch<8, 4>(a, T, s);
  return H <= 8192 ? launch<1, 8>(a, T, s) : launch<1, 32>(a, T, s);
}

}  // extern "C"
