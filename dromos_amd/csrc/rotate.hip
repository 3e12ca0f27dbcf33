// lx_rotate: queries and keys turned by their rows' positions; lx_rotary_frequencies: the frequencies of long contexts, on the host.
//
// Bytes decide: x is read once and y written once. A row's angles are the same for all its heads, so a workgroup makes them
// once for a few rows (a thread an angle, in 64 bits), leaves cosines and sines in LDS and goes over the rows' heads, PAIRS pairs a lane, the
// next ones on their way meanwhile. A call of few rows has several workgroups a row, each with some of the heads. Rows of 36 heads of 128
// values bf16, half of each turned, 125 MB read and written together: 28.4 us (4.4 TB/s; 40.3 us with a unit's place divided out anew each time and
// nothing on its way; two units on their way 29.7); 1 row of 40 heads: 3.4 to 4.2 us, a launch and one chain of loads.
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
  int parts;  // workgroups of the same rows, `per` heads each
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

// A run as it lies in memory.
template <int N>
struct Raw {
  u32x4 w[N == 8 ? 2 : 1];
};

template <int N>
__device__ __forceinline__ Raw<N> load_raw(const void* p, int type, int64_t i) {
  Raw<N> r{};
  if (type == LX_BF16) {
    const uint16_t* const h = static_cast<const uint16_t*>(p) + i;
    if constexpr (N == 8) r.w[0] = *reinterpret_cast<const u32x4*>(h);
    else if constexpr (N == 4) r.w[0].xy = *reinterpret_cast<const u32x2*>(h);
    else r.w[0].x = *h;
  } else {
    const uint32_t* const f = static_cast<const uint32_t*>(p) + i;
    if constexpr (N == 1) {
      r.w[0].x = *f;
    } else {
#pragma unroll
      for (int k = 0; k < N / 4; ++k) r.w[k] = reinterpret_cast<const u32x4*>(f)[k];
    }
  }
  return r;
}

template <int N>
__device__ __forceinline__ void values_of(const Raw<N>& r, int type, float (&v)[N]) {
  const bool half = type == LX_BF16;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t two = r.w[0][j / 2], one = r.w[j / 4][j % 4];
    v[j] = __uint_as_float(half ? (j % 2 ? two & 0xffff0000u : two << 16) : one);
  }
}

template <int N>
__device__ __forceinline__ void store_run(void* p, int type, int64_t i, const float (&v)[N]) {
  if constexpr (N % 4 == 0) {
    if (N == 8 && type == LX_BF16) {
      u32x4 r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = __builtin_bit_cast(uint32_t, pack_bf16(v[2 * j], v[2 * j + 1]));
      __builtin_nontemporal_store(r, reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i));
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
  // Unit u of head `head` of row r, 256 units further at each turn; the next one's values on their way meanwhile.
  const int units = (p.dim + 2 * PAIRS - 1) / (2 * PAIRS), turned = half / PAIRS, low = part * p.per, high = min(p.heads, low + p.per);
  const int heads = high - low, all = rows * heads * units;
  const int step_u = 256 % units, step_heads = 256 / units, step_r = step_heads / heads, step_head = step_heads % heads;
  int u = threadIdx.x % units, head = threadIdx.x / units % heads, r = threadIdx.x / units / heads;
  auto places = [&](int& a_at, int& b_at) {
    const bool split = u < turned && !p.interleaved;
    a_at = (low + head) * p.dim + (split ? PAIRS * u : 2 * PAIRS * u);
    b_at = split ? a_at + half : a_at + PAIRS;
    return PAIRS > 1 || u < turned || 2 * u + 1 < p.dim;  // whether there is a second run
  };
  Raw<PAIRS> a, b;
  auto ask = [&]() {
    int a_at, b_at;
    const bool both = places(a_at, b_at);
    const int64_t row = (first + r) * p.ld_x;
    a = load_raw<PAIRS>(p.x, p.x_type, row + a_at);
    b = both ? load_raw<PAIRS>(p.x, p.x_type, row + b_at) : a;
  };
  if (static_cast<int>(threadIdx.x) < all) ask();
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
  for (int i = threadIdx.x; i < all; i += 256) {
    int a_at, b_at;
    const bool both = places(a_at, b_at), turns = u < turned;
    const int mine = r, at = r * half + PAIRS * u;
    Run<PAIRS> v;
    values_of<PAIRS>(a, p.x_type, v.a);
    values_of<PAIRS>(b, p.x_type, v.b);
    u += step_u, head += step_head, r += step_r;
    if (u >= units) u -= units, ++head;
    if (head >= heads) head -= heads, ++r;
    if (i + 256 < all) ask();
    if (!found[mine]) continue;
    if (turns) {
      float c[PAIRS], s[PAIRS];
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) c[j] = cosines[at + j], s[j] = sines[at + j];
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
          float& x = 2 * j < PAIRS ? v.a[2 * j % PAIRS] : v.b[2 * j % PAIRS];
          float& y = 2 * j + 1 < PAIRS ? v.a[(2 * j + 1) % PAIRS] : v.b[(2 * j + 1) % PAIRS];
          const float a = x, b = y;
          x = a * c[j] - b * s[j];
          y = b * c[j] + a * s[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
          const float a = v.a[j], b = v.b[j];
          v.a[j] = a * c[j] - b * s[j];
          v.b[j] = b * c[j] + a * s[j];
        }
      }
    }
    const int64_t row = (first + mine) * p.ld_y;
    store_run<PAIRS>(p.y, p.y_type, row + a_at, v.a);
    if (both) store_run<PAIRS>(p.y, p.y_type, row + b_at, v.b);
  }
}

template <int PAIRS>
int launch(RotateArgs p, hipStream_t s) {
  const int half = p.rot / 2, units = (p.dim + 2 * PAIRS - 1) / (2 * PAIRS);
  // As many rows a workgroup as have an angle a thread, fewer where that makes fewer than four workgroups a unit of the device: all of them are there at
  // once then (6820 rows: 28.4 us; eight workgroups a unit, seven of them at work on average, 31.7 us).
  int rows = half ? 256 / half : kMostRows;
  rows = rows < 1 ? 1 : rows > kMostRows ? kMostRows : rows;
  const int spread = (p.T + 4 * compute_units() - 1) / (4 * compute_units());
  p.rows = rows < spread ? rows : spread;
  const int64_t groups = (static_cast<int64_t>(p.T) + p.rows - 1) / p.rows;
  // Several workgroups a row where rows are few, a unit a thread at least: a row of 256 heads of 128 3.1 us, 8.2 by one.
  const int64_t wanted = (2 * compute_units() + groups - 1) / groups, most = (static_cast<int64_t>(units) * p.heads + 255) / 256;
  const int64_t parts = wanted < most ? wanted : most;
  p.per = static_cast<int>((p.heads + parts - 1) / parts);
  p.parts = (p.heads + p.per - 1) / p.per;
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
