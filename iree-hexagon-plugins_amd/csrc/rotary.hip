// Rotary positions of packed rows: pair i of a head's first 2 * half dims is
// turned by t = position * frequency[i], the position that of the pair's axis,
//   y1 = x1 cos t - x2 sin t, y2 = x2 cos t + x1 sin t
// with (x1, x2) = (x[i], x[half + i]), or (x[2 i], x[2 i + 1]) interleaved; the
// dims past them are copied.
//
// A workgroup takes a token or a few: its threads first compute the half
// (cos, sin) of each into LDS, which all of the token's query and KV heads then
// share. The angle's product is made and reduced to part of a turn in 64 bits
// (a far position times a frequency has lost the turn's fraction in 32), the
// sine and cosine of that part in 32. A piece is 16 bytes of either side of the
// pairs; operands that 16-byte accesses do not fit go an element at a time. Bound
// by memory: 8191 rows of 32 and 8 heads of 128 (168 MB) take 25.4 us, 6.6 TB/s
// (30 a call among others); 64 rows 3.4, start to end.
#include "device_common.h"
#include "kernels_internal.h"

namespace ihp {

namespace {

constexpr int kRotaryThreads = 256;
// (cos, sin) of a workgroup's tokens: 128 pairs each, 16 tokens at most.
constexpr int kRotaryPairs = 2048;
typedef float f32x2 __attribute__((ext_vector_type(2)));

// N pairs of halves, or interleaved neighbours, from `in` to `out`.
template <int N>
struct RotaryVector;
template <>
struct RotaryVector<8> {
  typedef f16x8 type;
};
template <>
struct RotaryVector<1> {
  typedef f16 type;
};

// One pair turned by t = (cos, sin). The roundings are written out
// so that both kinds of access give the same bits.
__device__ __forceinline__ void turn_pair(f16 a, f16 b, f32x2 t, f16 *ya,
                                          f16 *yb) {
  const float x1 = a, x2 = b;
  float y1 = __builtin_fmaf(x1, t[0], -__fmul_rn(x2, t[1]));
  float y2 = __builtin_fmaf(x2, t[0], __fmul_rn(x1, t[1]));
  asm("" : "+v"(y1), "+v"(y2));  // not one instruction with the conversion
  *ya = (f16)y1;
  *yb = (f16)y2;
}

}  // namespace

// WIDE: 16 bytes at a time.
template <bool WIDE, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(Rotary r) {
  constexpr int VEC = WIDE ? 8 : 1;  // elements of one access
  typedef typename RotaryVector<VEC>::type Vec;
  __shared__ f32x2 turns[kRotaryPairs];
  const int tid = threadIdx.x;
  const int heads = r.heads[0] + r.heads[1], items = heads * r.pieces;
  for (int64_t row0 = (int64_t)blockIdx.x * r.tokens; row0 < r.rows;
       row0 += (int64_t)gridDim.x * r.tokens) {
    const int rows =
        r.rows - row0 < r.tokens ? (int)(r.rows - row0) : r.tokens;
    for (int i = tid; i < rows * r.half; i += kRotaryThreads) {
      const int row = i / r.half, pair = i - row * r.half;
      const int axis = (pair >= r.ends[0]) + (pair >= r.ends[1]) +
                       (pair >= r.ends[2]);
      const int position = r.positions[axis * r.position_stride + row0 + row];
      const double turn =
          (double)position * (double)r.frequencies[pair] * 0.15915494309189535;
      float s, c;
      sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
      turns[i] = f32x2{c, s};
    }
    __syncthreads();
    for (int i = tid; i < rows * items; i += kRotaryThreads) {
      const int row = i / items, at = i - row * items;
      int head = at / r.pieces;
      const int piece = at - head * r.pieces;
      const int which = head >= r.heads[0];
      head -= which ? r.heads[0] : 0;
      const f16 *in = r.in[which] + (row0 + row) * r.in_strides[which][0] +
                      head * r.in_strides[which][1];
      f16 *out = r.out[which] + (row0 + row) * r.out_strides[which][0] +
                 head * r.out_strides[which][1];
      const f32x2 *turn = turns + row * r.half;
      if (piece >= r.rotated) {  // dims past the rotated ones
        const int d = 2 * r.half + (piece - r.rotated) * VEC;
        *(Vec *)(out + d) = *(const Vec *)(in + d);
      } else if (INTERLEAVED && WIDE) {
        const int d = piece * 8;
        const f16x8 x = *(const f16x8 *)(in + d);
        f16x8 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f16 ya, yb;
          turn_pair(x[2 * e], x[2 * e + 1], turn[d / 2 + e], &ya, &yb);
          y[2 * e] = ya;
          y[2 * e + 1] = yb;
        }
        *(f16x8 *)(out + d) = y;
      } else if (WIDE) {
        const int d = piece * 8;
        const f16x8 a = *(const f16x8 *)(in + d);
        const f16x8 b = *(const f16x8 *)(in + r.half + d);
        f16x8 ya, yb;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f16 y1, y2;
          turn_pair(a[e], b[e], turn[d + e], &y1, &y2);
          ya[e] = y1;
          yb[e] = y2;
        }
        *(f16x8 *)(out + d) = ya;
        *(f16x8 *)(out + r.half + d) = yb;
      } else {
        const int d1 = INTERLEAVED ? 2 * piece : piece;
        const int d2 = INTERLEAVED ? 2 * piece + 1 : r.half + piece;
        f16 y1, y2;
        turn_pair(in[d1], in[d2], turn[piece], &y1, &y2);
        out[d1] = y1;
        out[d2] = y2;
      }
    }
    __syncthreads();  // before the next tokens' turns
  }
}

hipError_t launch_rotary(const Rotary &rotary, void *stream) {
  Rotary r = rotary;
  // Tokens of few pieces share a workgroup.
  const int items = (r.heads[0] + r.heads[1]) * r.pieces;
  int tokens = kRotaryThreads / items;
  const int most = r.half > 0 ? kRotaryPairs / r.half : 16;
  tokens = tokens > 16 ? 16 : tokens < 1 ? 1 : tokens;
  r.tokens = tokens < most ? tokens : most;
  const void *kernels[2][2] = {
      {(const void *)&rotary_kernel<false, false>,
       (const void *)&rotary_kernel<false, true>},
      {(const void *)&rotary_kernel<true, false>,
       (const void *)&rotary_kernel<true, true>}};
  void *args[] = {&r};
  // A launch has fewer than 2^32 threads.
  const int64_t wgs = ((int64_t)r.rows + r.tokens - 1) / r.tokens;
  const int64_t most_wgs = (int64_t)1 << 22;
  return hipLaunchKernel(kernels[r.wide][r.interleaved],
                         dim3((unsigned)(wgs < most_wgs ? wgs : most_wgs)),
                         dim3(kRotaryThreads), args, 0, (hipStream_t)stream);
}

const KernelEntry *rotary_kernels(int *count) {
  static const KernelEntry all[] = {
      {"rotary_elements", (const void *)&rotary_kernel<false, false>, kRotaryThreads, 0},
      {"rotary_elements_interleaved", (const void *)&rotary_kernel<false, true>, kRotaryThreads, 0},
      {"rotary", (const void *)&rotary_kernel<true, false>, kRotaryThreads, 0},
      {"rotary_interleaved", (const void *)&rotary_kernel<true, true>, kRotaryThreads, 0},
  };
  *count = (int)(sizeof(all) / sizeof(all[0]));
  return all;
}

}  // namespace ihp
