// The angles of rotary positions, as lx_kv8_append and lx_rotate turn queries and keys by them.
#pragma once

#include "common.h"

namespace dro {

// The cosines and sines of N angles at a position, from quarter turns a position. The product of a 31-bit and a 53-bit number is right to 2^-53 in 64 bits, and so is the
// second of them: the angle is off by 2^-52 of itself. Whole quarter turns are taken off it there, so up to 2^26 radians what is left of a far position
// is as good as of a near one, to f32's rounding (2^-25); at 2^31 it is 2^-21 off. The rest u, an eighth of a turn at most, goes into Taylor's series in f32 (what they leave
// off is below 2^-29 and 2^-32).
template <int N>
__device__ __forceinline__ void angles(const double (&quarters)[N], int position, float* c, float* s) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const double turned = static_cast<double>(position) * quarters[j], whole = rint(turned);
    const float u = static_cast<float>((turned - whole) * 1.57079632679489661923), x = u * u;
    float a = __builtin_fmaf(x, 1.0f / 362880.0f, -1.0f / 5040.0f), b = __builtin_fmaf(x, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    a = __builtin_fmaf(x, a, 1.0f / 120.0f);
    b = __builtin_fmaf(x, b, -1.0f / 720.0f);
    a = __builtin_fmaf(x, a, -1.0f / 6.0f);
    b = __builtin_fmaf(x, b, 1.0f / 24.0f);
    a = __builtin_fmaf(x * u, a, u);  // sin u
    b = __builtin_fmaf(x, b, -0.5f);
    b = __builtin_fmaf(x, b, 1.0f);  // cos u
    const int quadrant = static_cast<int>(static_cast<long long>(whole)) & 3;
    c[j] = quadrant & 1 ? a : b;
    s[j] = quadrant & 1 ? b : a;
    if (quadrant == 1 || quadrant == 2) c[j] = -c[j];
    if (quadrant >= 2) s[j] = -s[j];
  }
}

}  // namespace dro
