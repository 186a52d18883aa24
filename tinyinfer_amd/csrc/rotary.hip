// Rotary positions of rows x [batch][heads][rows][D]: y = x with its first R dims turned,
// the pairs (a, b) of angle w = t f_i becoming (a cos w - b sin w, a sin w + b cos w) times
// the amplitude, the others as they are.
//
// A lane holds the cosines and sines of its 8 pairs (rotary.hpp) and walks over heads,
// which share them: they cost about 300 vector instructions, a head's values 70.
#include "rotary.hpp"

namespace tia {
namespace {

// Position of row i of request b.
__device__ __forceinline__ int64_t position_of(const RotateArgs& a, int b, int i) {
  return a.per_row ? int64_t(a.positions[int64_t(b) * a.rows + i]) : int64_t(a.positions[b]) + i;
}

// D and R multiples of 16: units of 16 values.
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a, int units, int chunk) {
  const unsigned at = blockIdx.x * 256 + threadIdx.x, up = unsigned(units);  // (below 2^31: rows * dim is)
  const int b = int(blockIdx.z), row = int(at / up), u = int(at % up);
  if (row >= a.rows) return;
  const RowUnit unit = row_unit(a.rotary, u);
  const int h0 = int(blockIdx.y) * chunk, h1 = min(a.heads, h0 + chunk);
  const uint16_t* x = a.x.at + b * a.x.batch + row * a.x.row;
  uint16_t* y = a.y + (int64_t(b) * a.heads * a.rows + row) * a.dim;
  const int64_t step = int64_t(a.rows) * a.dim;
  if (!unit.turned) {
#pragma unroll 4
    for (int h = h0; h < h1; ++h) {
      store_half8(y + h * step + unit.first, load_half8(x + h * a.x.head + unit.first));
      store_half8(y + h * step + unit.second, load_half8(x + h * a.x.head + unit.second));
    }
    return;
  }
  const Turns t(a.rotary, u, position_of(a, b, row));
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    half8_t p = load_half8(x + h * a.x.head + unit.first), q = load_half8(x + h * a.x.head + unit.second);
    turn_unit(t, a.rotary.interleaved, p, q);
    store_half8(y + h * step + unit.first, p);
    store_half8(y + h * step + unit.second, q);
  }
}

// Any D and even R: a lane has one pair, or one value from R on.
__global__ __launch_bounds__(256) void rotate_pairs_kernel(RotateArgs a, int chunk) {
  const int pairs = a.rotary.rotated / 2, units = a.dim - pairs;
  const unsigned at = blockIdx.x * 256 + threadIdx.x, up = unsigned(units);  // (below 2^31: rows * dim is)
  const int b = int(blockIdx.z), row = int(at / up), u = int(at % up);
  if (row >= a.rows) return;
  const int h0 = int(blockIdx.y) * chunk, h1 = min(a.heads, h0 + chunk);
  const uint16_t* x = a.x.at + b * a.x.batch + row * a.x.row;
  uint16_t* y = a.y + (int64_t(b) * a.heads * a.rows + row) * a.dim;
  const int64_t step = int64_t(a.rows) * a.dim;
  if (u >= pairs) {
    for (int h = h0; h < h1; ++h) y[h * step + pairs + u] = x[h * a.x.head + pairs + u];
    return;
  }
  const int first = a.rotary.interleaved ? 2 * u : u, second = a.rotary.interleaved ? 2 * u + 1 : pairs + u;
  float c, s;
  turn_of(a.rotary.turns[u], position_of(a, b, row), a.rotary.amplitude, c, s);
  for (int h = h0; h < h1; ++h) {
    f16 p = __builtin_bit_cast(f16, x[h * a.x.head + first]), q = __builtin_bit_cast(f16, x[h * a.x.head + second]);
    turn_pair(c, s, p, q);
    y[h * step + first] = __builtin_bit_cast(uint16_t, p);
    y[h * step + second] = __builtin_bit_cast(uint16_t, q);
  }
}

}  // namespace

hipError_t rotate(const RotateArgs& a, hipStream_t stream) {
  const bool wide = a.dim % 16 == 0 && a.rotary.rotated % 16 == 0;
  const int units = wide ? a.dim / 16 : a.dim - a.rotary.rotated / 2;
  const int64_t groups = (int64_t(a.rows) * units + 255) / 256;
  int64_t chunks = 1;
  while (chunks < a.heads && groups * a.batch * chunks < 1024) chunks *= 2;
  const int chunk = int((a.heads + chunks - 1) / chunks);
  const dim3 grid(unsigned(groups), unsigned((a.heads + chunk - 1) / chunk), unsigned(a.batch));
  if (wide) hipLaunchKernelGGL(rotate_kernel, grid, dim3(256), 0, stream, a, units, chunk);
  else hipLaunchKernelGGL(rotate_pairs_kernel, grid, dim3(256), 0, stream, a, chunk);
  return hipGetLastError();
}

}  // namespace tia
