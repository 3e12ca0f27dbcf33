// lx_rotate: queries and keys turned by their rows' positions; lx_rotary_frequencies: the frequencies of long contexts, on the host.
//
// Bytes decide: x is read once and y written once. A row's angles are the same for all its heads, so a workgroup makes them
// once for a few rows (a thread an angle, in 64 bits), leaves cosines and sines in LDS and goes over the rows' heads, PAIRS pairs a lane. A
// call of few rows has several workgroups a row, each with some of the heads.
#include <cmath>

#include "mixer.h"
#include "rotation.h"

namespace dro {
namespace {

constexpr int kMaxDim = 1024;
constexpr int kAngles = 512;  // of a workgroup's rows together, and of one row at most
constexpr int kMostRows = 8;  // of a workgroup

struct RotateArgs {
  const void* x;
  void* y;
  const int32_t* positions;
  const float* freq;
  int64_t ld_x, ld_y;
  int x_type, y_type, rot, interleaved, T, heads, dim;
  int rows;   // of a workgroup
  int parts;  // workgroups of the same rows, `per` units each
  int per;
  float amplitude;
  MixBatch b;
};

// The position of row t, or false where it belongs to nobody.
__device__ __forceinline__ bool position_of(const RotateArgs& p, int t, int& position) {
  if (p.positions) {
    position = p.positions[t];
    return true;
  }
  int s, j;
  // Pieces of one row: piece t + s is row t of sequence s, if it is in there; the last sequence that starts at t or before has it.
  if (!p.b.rows) {
    s = t;
    if (s >= p.b.seqs) return false;
  } else {
    s = mix_last(p.b.seqs, t, [&](int i) { return p.b.rows[i]; });
    if (s < 0) return false;
  }
  const MixSpan span = mix_span(p.b, s);
  j = t - span.row0;
  position = span.lead + j;
  return j >= span.first && j < span.stop;
}

// PAIRS pairs of a head: two runs of PAIRS values (the first values of the pairs and the second ones, or where neighbours are
// pairs the run's halves).
template <int PAIRS>
struct Run {
  float a[PAIRS], b[PAIRS];
};

template <int N>
__device__ __forceinline__ void load_run(const void* p, int type, int64_t i, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
    if (N == 8 && type == LX_BF16) {
      const u32x4 r = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t two = r[j / 2];
        v[j] = __uint_as_float(j % 2 ? two & 0xffff0000u : two << 16);
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const f32x4 four = load_four(p, type, true, i + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k + j] = four[j];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = load_as_f32(p, type, i + j);
  }
}

template <int N>
__device__ __forceinline__ void store_run(void* p, int type, int64_t i, const float (&v)[N]) {
  if constexpr (N % 4 == 0) {
    if (N == 8 && type == LX_BF16) {
      u32x4 r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = __builtin_bit_cast(uint32_t, pack_bf16(v[2 * j], v[2 * j + 1]));
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) = r;
    } else {
#pragma unroll
      for (int k = 0; k < N; k += 4) store_four(p, type, true, i + k, f32x4{v[k], v[k + 1], v[k + 2], v[k + 3]});
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) store_from_f32(p, type, i + j, v[j]);
  }
}

// A head is dim / (2 PAIRS) units (rounded up where PAIRS is 1: an odd dim's last unit is one value). The first rot / (2 PAIRS) are turned.
template <int PAIRS>
__global__ void __launch_bounds__(256) rotate_kernel(const RotateArgs p) {
  __shared__ __attribute__((aligned(16))) float cosines[kAngles], sines[kAngles];
  __shared__ int found[kMostRows], place[kMostRows];
  const int64_t first = static_cast<int64_t>(blockIdx.x / p.parts) * p.rows;
  const int part = blockIdx.x % p.parts, half = p.rot / 2;
  const int rows = static_cast<int>(p.T - first < p.rows ? p.T - first : p.rows);
  for (int r = threadIdx.x / kWave; r < rows; r += 256 / kWave) {  // every lane of a wavefront alike
    int position = 0;
    const bool in = position_of(p, static_cast<int>(first) + r, position);
    if (threadIdx.x % kWave == 0) found[r] = in, place[r] = position;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * half; i += 256) {
    const int r = i / half, n = i % half;
    const double quarters[1] = {static_cast<double>(p.freq[n]) * 0.63661977236758134308};
    float c[1], s[1];
    angles(quarters, place[r], c, s);
    cosines[i] = c[0] * p.amplitude;
    sines[i] = s[0] * p.amplitude;
  }
  __syncthreads();
  const int units = (p.dim + 2 * PAIRS - 1) / (2 * PAIRS), turned = half / PAIRS, of_row = units * p.heads;
  const int stop = min(of_row, (part + 1) * p.per);
  for (int r = 0; r < rows; ++r) {
    if (!found[r]) continue;
    const int64_t x_row = (first + r) * p.ld_x, y_row = (first + r) * p.ld_y;
    for (int i = part * p.per + static_cast<int>(threadIdx.x); i < stop; i += 256) {
      const int head = i / units, u = i % units;
      const bool turns = u < turned, split = turns && !p.interleaved;
      const int a_at = head * p.dim + (split ? PAIRS * u : 2 * PAIRS * u), b_at = split ? a_at + half : a_at + PAIRS;
      const bool both = PAIRS > 1 || turns || 2 * u + 1 < p.dim;
      Run<PAIRS> v;
      load_run<PAIRS>(p.x, p.x_type, x_row + a_at, v.a);
      if (both) load_run<PAIRS>(p.x, p.x_type, x_row + b_at, v.b);
      if (turns) {
        const float* const c = cosines + r * half + PAIRS * u;
        const float* const s = sines + r * half + PAIRS * u;
        Run<PAIRS> w = v;
        if (p.interleaved) {
#pragma unroll
          for (int j = 0; j < PAIRS; ++j) {
            const int at = 2 * j;
            float& ra = at < PAIRS ? w.a[at % PAIRS] : w.b[at % PAIRS];
            float& rb = at + 1 < PAIRS ? w.a[(at + 1) % PAIRS] : w.b[(at + 1) % PAIRS];
            const float a = ra, b = rb;
            ra = a * c[j] - b * s[j];
            rb = b * c[j] + a * s[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < PAIRS; ++j) {
            w.a[j] = v.a[j] * c[j] - v.b[j] * s[j];
            w.b[j] = v.b[j] * c[j] + v.a[j] * s[j];
          }
        }
        v = w;
      }
      store_run<PAIRS>(p.y, p.y_type, y_row + a_at, v.a);
      if (both) store_run<PAIRS>(p.y, p.y_type, y_row + b_at, v.b);
    }
  }
}

template <int PAIRS>
int launch(RotateArgs p, hipStream_t s) {
  const int half = p.rot / 2, of_row = (p.dim + 2 * PAIRS - 1) / (2 * PAIRS) * p.heads;
  // As many rows a workgroup as have an angle a thread, fewer where that leaves compute units without one.
  int rows = half ? 256 / half : kMostRows;
  rows = rows < 1 ? 1 : rows > kMostRows ? kMostRows : rows;
  const int spread = (p.T + 2 * compute_units() - 1) / (2 * compute_units());
  p.rows = rows < spread ? rows : spread;
  const int64_t groups = (static_cast<int64_t>(p.T) + p.rows - 1) / p.rows;
  // Rows of their own workgroups only where those are few: a part has 256 units at least.
  int64_t parts = (2 * compute_units() + groups - 1) / groups;
  const int most = (of_row + 255) / 256;
  p.parts = static_cast<int>(parts < most ? parts : most);
  p.per = (of_row + p.parts - 1) / p.parts;
  if (groups * p.parts * 256 > kMaxGridThreads) return kInvalid;
  hipLaunchKernelGGL((rotate_kernel<PAIRS>), dim3(static_cast<unsigned>(groups * p.parts)), dim3(256), 0, s, p);
  return status_of(hipGetLastError());
}

}  // namespace
}  // namespace dro

using namespace dro;

extern "C" {

int lx_rotary_frequencies(lx_rope kind, double base, int rot, double factor, double original, double low, double high, float* freq,
                          float* amplitude) {
  if (kind < LX_ROPE_PLAIN || kind > LX_ROPE_WAVES || rot < 0 || rot > kMaxDim || rot % 2 != 0) return fail(kInvalid);
  auto fine = [](double v) { return v > 0.0 && v < 1e300; };
  if (!fine(base) || base <= 1.0) return fail(kInvalid);
  if (kind != LX_ROPE_PLAIN && (!fine(factor) || factor < 1.0)) return fail(kInvalid);
  if (kind == LX_ROPE_BASE && rot < 4 && rot != 0) return fail(kInvalid);
  if ((kind == LX_ROPE_PARTS || kind == LX_ROPE_WAVES) && (!fine(original) || !fine(low) || !fine(high) || low >= high)) return fail(kInvalid);
  constexpr double kTurn = 6.28318530717958647693;
  if (amplitude) *amplitude = kind == LX_ROPE_PARTS ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
  if (!freq) return kOk;
  if (kind == LX_ROPE_BASE && rot) base *= std::pow(factor, static_cast<double>(rot) / (rot - 2));
  auto dimension = [&](double turns) { return rot * std::log(original / (kTurn * turns)) / (2.0 * std::log(base)); };
  double from = 0.0, to = 0.0;
  if (kind == LX_ROPE_PARTS) {
    from = std::floor(dimension(high)), to = std::ceil(dimension(low));
    from = from < 0.0 ? 0.0 : from;
    to = to > rot - 1.0 ? rot - 1.0 : to;
  }
  for (int i = 0; i < rot / 2; ++i) {
    const double f = std::pow(base, -2.0 * i / rot);
    double kept = 1.0;  // of the plain frequency; the rest is slowed by the factor
    if (kind == LX_ROPE_LINEAR) kept = 0.0;
    if (kind == LX_ROPE_PARTS) kept = i <= from ? 1.0 : i >= to ? 0.0 : 1.0 - (i - from) / (to - from);
    if (kind == LX_ROPE_WAVES) kept = (original * f / kTurn - low) / (high - low);
    kept = kept < 0.0 ? 0.0 : kept > 1.0 ? 1.0 : kept;
    freq[i] = static_cast<float>(kept == 1.0 ? f : f * (kept + (1.0 - kept) / factor));
  }
  return kOk;
}

int lx_rotate(const void* x, lx_dtype x_dtype, int ld_x, void* y, lx_dtype y_dtype, int ld_y, const lx_kv8_batch* batch,
              const int32_t* positions, const float* freq, float amplitude, int rot, int interleaved, int T, int heads, int dim, void* stream) {
  if (positions ? T < 0 || T >= (1 << 30) : mix_check(batch, T) != kOk) return fail(kInvalid);
  if (heads < 0 || dim < 0 || dim > kMaxDim || rot < 0 || rot > dim || rot % 2 != 0) return fail(kInvalid);
  if (!mix_type(x_dtype) || !mix_type(y_dtype)) return fail(kInvalid);
  if (T == 0 || heads == 0 || dim == 0 || (!positions && batch->seqs == 0)) return kOk;
  const int64_t width = static_cast<int64_t>(heads) * dim;
  if (!x || !y || (rot && !freq) || width >= (int64_t{1} << 31) || static_cast<int64_t>(T) * heads >= (int64_t{1} << 31)) return fail(kInvalid);
  if (T > 1 && (ld_x < width || ld_y < width)) return fail(kInvalid);
  if (!positions && !batch->lengths) return fail(kInvalid);
  if (x == y && (x_dtype != y_dtype || (T > 1 && ld_x != ld_y))) return fail(kInvalid);
  RotateArgs p{};
  p.x = x, p.y = y, p.positions = positions, p.freq = freq;
  p.ld_x = ld_x, p.ld_y = ld_y, p.x_type = x_dtype, p.y_type = y_dtype;
  p.rot = rot, p.interleaved = interleaved != 0, p.T = T, p.heads = heads, p.dim = dim, p.amplitude = amplitude;
  if (!positions) p.b = mix_batch(*batch, T);
  if (!positions && (p.b.max_rows == 0 || p.b.seqs == 0)) return kOk;
  auto in = [&](int bytes) {
    return mix_aligned(x, T > 1 ? ld_x : 0, x_dtype, x_dtype == LX_BF16 ? bytes : 16) && mix_aligned(y, T > 1 ? ld_y : 0, y_dtype, y_dtype == LX_BF16 ? bytes : 16);
  };
  hipStream_t s = as_stream(stream);
  int st;
  if (dim % 16 == 0 && rot % 16 == 0 && in(16)) st = launch<8>(p, s);
  else if (dim % 8 == 0 && rot % 8 == 0 && in(8)) st = launch<4>(p, s);
  else st = launch<1>(p, s);
  return st ? fail(st) : kOk;
}

}  // extern "C"
