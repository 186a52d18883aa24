// Rotary positions of rows x [batch][heads][rows][D]: y = x with its first R dims turned,
// the pairs (a, b) of angle w = t f_i becoming (a cos w - b sin w, a sin w + b cos w) times
// the amplitude, the others as they are.
//
// A lane holds the cosines and sines of its 8 pairs (rotary.hpp) and walks over heads,
// which share them: they cost about 300 vector instructions, a head's values 70.
//
// What bounds it: memory (2 requests of 32 heads of 128, 6001 rows: 41 us, 4.8 TB/s of reads and
// writes, 35.6 where the output's block stays partly in the last cache; vector units 40 % busy; 8 of 25
// heads of 64, 777 rows: 9.7, launch and ramp 3 of them), and the launch for single tokens (32 of 24
// heads of 64: 3.6 us).  Dims that are no multiple of 16: 8- or 4-byte pieces (8 of 32 heads of 80, 2000 rows, 40
// dims turned 62 us, 2.6 TB/s, 20 dims 77).
#include "rotary.hpp"

namespace tia {
namespace {

// Position of row i of request b.
__device__ __forceinline__ int64_t position_of(const RotateArgs& a, int b, int i) {
  return a.per_row ? int64_t(a.positions[int64_t(b) * a.rows + i]) : int64_t(a.positions[b]) + i;
}

// D and R multiples of 16: units of 16 values.  flat (HC 1): heads lie side by side, too.
template <int HC>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a, int units, int chunk) {
  constexpr bool flat = HC == 1;
  const unsigned at = blockIdx.x * 256 + threadIdx.x, up = unsigned(units);  // (below 2^31: rows * dim is)
  const unsigned rows = unsigned(a.rows), piece = at / up, above = flat ? piece / rows : 0;
  const int b = int(blockIdx.z), row = int(piece - above * rows), u = int(at % up);
  const int h0 = flat ? int(above) : int(blockIdx.y) * chunk, h1 = min(a.heads, h0 + chunk);
  if (row >= a.rows || h0 >= a.heads) return;
  const RowUnit unit = row_unit(a.rotary, u);
  uint16_t* y = a.y + (int64_t(b) * a.heads * a.rows + row) * a.dim + unit.first;
  turn_heads<HC>(a.rotary, unit, u, position_of(a, b, row), a.x.at + b * a.x.batch + row * a.x.row, a.x.head, y,
                 int64_t(a.rows) * a.dim, unit.second - unit.first, h0, h1);
}

// Any D and even R: a lane has W pairs, or W values from R on (W divides both counts).
template <int W>
__global__ __launch_bounds__(256) void rotate_pairs_kernel(RotateArgs a, int chunk) {
  const int pairs = a.rotary.rotated / 2, units = (a.dim - pairs) / W;
  const unsigned at = blockIdx.x * 256 + threadIdx.x;
  const int b = int(blockIdx.z), row = int(at / unsigned(units)), u = W * int(at % unsigned(units));
  if (row >= a.rows) return;
  const int h0 = int(blockIdx.y) * chunk, h1 = min(a.heads, h0 + chunk);
  const uint16_t* x = a.x.at + b * a.x.batch + row * a.x.row;
  uint16_t* y = a.y + (int64_t(b) * a.heads * a.rows + row) * a.dim;
  const int64_t step = int64_t(a.rows) * a.dim;
  if (u >= pairs) {
    for (int h = h0; h < h1; ++h) __builtin_memcpy(y + h * step + pairs + u, x + h * a.x.head + pairs + u, 2 * W);
    return;
  }
  const bool interleaved = a.rotary.interleaved;
  const int first = interleaved ? 2 * u : u, second = interleaved ? 2 * u + W : pairs + u;
  float c[W], s[W];
  const int64_t t = position_of(a, b, row);
#pragma unroll
  for (int i = 0; i < W; ++i) turn_of(a.rotary.turns[u + i], t, a.rotary.amplitude, c[i], s[i]);
#pragma unroll 2
  for (int h = h0; h < h1; ++h) {
    f16 v[2 * W];
    __builtin_memcpy(v, x + h * a.x.head + first, 2 * W);
    __builtin_memcpy(v + W, x + h * a.x.head + second, 2 * W);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (interleaved) turn_pair(c[i], s[i], v[2 * i], v[2 * i + 1]);
      else turn_pair(c[i], s[i], v[i], v[W + i]);
    }
    __builtin_memcpy(y + h * step + first, v, 2 * W);
    __builtin_memcpy(y + h * step + second, v + W, 2 * W);
  }
}

}  // namespace

hipError_t rotate(const RotateArgs& a, hipStream_t stream) {
  const bool wide = a.dim % 16 == 0 && a.rotary.rotated % 16 == 0;
  const int pairs = a.rotary.rotated / 2, plain = a.dim - a.rotary.rotated;
  const int w = (pairs | plain) % 4 == 0 ? 4 : (pairs | plain) % 2 == 0 ? 2 : 1;  // (of the narrow kernel)
  const int units = wide ? a.dim / 16 : (pairs + plain) / w;
  const int64_t lanes = int64_t(a.rows) * units;
  // Short rows: one head to a lane, so that a request of a few tokens fills its workgroups (64
  // requests of 32 heads of 128, one token: 4.1 us; 7.0 with lanes that walk over heads).
  if (wide && lanes < 256) {
    const dim3 grid(unsigned((lanes * a.heads + 255) / 256), 1, unsigned(a.batch));
    hipLaunchKernelGGL(rotate_kernel<1>, grid, dim3(256), 0, stream, a, units, 1);
    return hipGetLastError();
  }
  const int64_t groups = (lanes + 255) / 256;
  // Heads to a lane: as many as leave 1024 workgroups, four a CU (8 requests of 25 heads of 64, 777
  // rows: 10.7 us, 11.1 with 512 and 13.1 with 4096; 2 of 32 of 128, 6001 rows: 35.6, 36.2 and 35.3).
  int64_t chunks = 1;
  while (chunks < a.heads && groups * a.batch * chunks < 1024) chunks *= 2;
  const int chunk = int((a.heads + chunks - 1) / chunks);
  const dim3 grid(unsigned(groups), unsigned((a.heads + chunk - 1) / chunk), unsigned(a.batch));
  if (!wide) {
    const auto kernel = w == 4 ? rotate_pairs_kernel<4> : w == 2 ? rotate_pairs_kernel<2> : rotate_pairs_kernel<1>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a, chunk);
    return hipGetLastError();
  }
  if (chunk < 4) hipLaunchKernelGGL(rotate_kernel<2>, grid, dim3(256), 0, stream, a, units, chunk);
  else hipLaunchKernelGGL(rotate_kernel<4>, grid, dim3(256), 0, stream, a, units, chunk);
  return hipGetLastError();
}

}  // namespace tia
