// Rotary embedding from positions on several axes.
//
// Pair i of a head's channels turns by the angle a_i = pos[axis_i][token] * f_i:
//   y0 = x0 cos a_i - x1 sin a_i,   y1 = x1 cos a_i + x0 sin a_i
// with (x0, x1) = channels (2 i, 2 i + 1), or (i, i + pairs); channels from 2 * pairs on are copied.  The inverse
// (the gradient) turns by -a_i.  The angle is taken in fp64 as a share of a full turn, reduced to half a turn
// either way, and only then rounded to fp32, so a position far out costs no accuracy; the rotation is fp32 and
// rounded once.
//
// Bound by HBM: each channel is read once and written once, positions are 12 bytes a token (75,600 tokens, 2 x 40 heads
// of 128 channels in bf16: 578 us, 5.4 TB/s; a plain copy of as much reaches 4.9).  The angles' sines are
// computed where they are used, once for all heads that a wave (or, element by element, a workgroup) takes.
#include <math.h>

#include "common.h"
#include "kv_cache.h"

namespace pasa {

namespace {

constexpr int kMaxPairs = 128;
constexpr int kRows = 4;  // of q or k that a lane has under way
constexpr double kInvTwoPi = 0.15915494309189533576888;

__device__ __forceinline__ double position(const RopeAxesParams& p, int64_t at) {
  if (p.pos_type == kPosI32) return (double)((const int32_t*)p.pos)[at];
  if (p.pos_type == kPosI64) return (double)((const int64_t*)p.pos)[at];
  return (double)((const float*)p.pos)[at];
}

// Cosine and sine of pair j's angle for token (b, s).
__device__ __forceinline__ float2 turn_of(const RopeAxesParams& p, int j, int64_t b, int64_t s) {
  const int ax = min(max(p.axis[j], 0), p.axes - 1);
  double turn = position(p, ax * p.pos_axis + b * p.pos_b + s * p.pos_s) * p.inv_freq[j] * kInvTwoPi;
  turn -= rint(turn);
  float sn, cn;
  sincospif((float)(2.0 * turn), &sn, &cn);
  return make_float2(cn, p.inverse ? -sn : sn);
}

// One element at a time: any stride, alignment and number of pairs.  A workgroup for each token; its heads read the
// sines from LDS.
template <typename T>
__global__ __launch_bounds__(256) void rope_axes_scalar(RopeAxesParams p) {
  __shared__ float2 cs[kMaxPairs];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x / p.S, s = blockIdx.x - b * p.S;
  for (int j = tid; j < p.pairs; j += 256) cs[j] = turn_of(p, j, b, s);
  __syncthreads();
  const int units = p.D - p.pairs;  // a pair, or a channel to copy
  const int heads = p.t[0].heads + p.t[1].heads;
  for (int i = tid; i < heads * units; i += 256) {
    int h = i / units;
    const int u = i - h * units;
    const int w = h >= p.t[0].heads;
    if (w) h -= p.t[0].heads;
    const RopeAxesTensor& x = p.t[w];
    const T* in = (const T*)x.in + b * x.in_b + s * x.in_s + h * x.in_h;
    T* out = (T*)x.out + b * x.out_b + s * x.out_s + h * x.out_h;
    if (u < p.pairs) {
      const int c0 = p.halves ? u : 2 * u, c1 = p.halves ? u + p.pairs : 2 * u + 1;
      const float x0 = (float)in[c0], x1 = (float)in[c1];
      const float2 a = cs[u];
      out[c0] = (T)(x0 * a.x - x1 * a.y);
      out[c1] = (T)(x1 * a.x + x0 * a.y);
    } else {
      const int c = p.pairs + u;
      out[c] = in[c];
    }
  }
}

// 16 bytes at a time, where the channels, strides and pairs allow it (64 tokens of 48 heads: 4.5 us, element by element
// 8.2; 8,192 tokens: 33 and 72).  A wave takes a token, or a part of its heads: a lane has one 16-byte unit of a head's channels
// (HALVES: two, whose channels are each other's pairs), 64 / units heads lie side by side in the wave.  The lanes share
// out the pairs' angles, and through LDS each gets the sines of its own, which stay in registers for all heads.
template <typename T, bool HALVES>
__global__ __launch_bounds__(256) void rope_axes_vec(RopeAxesParams p, int units, int parts) {
  constexpr int V = 16 / sizeof(T);
  constexpr int N = HALVES ? 2 : 1;  // 16-byte pieces of a lane
  constexpr int P = HALVES ? V : V / 2;
  __shared__ float2 turn[4][kMaxPairs];
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t n = wave / parts;
  if (n >= p.B * p.S) return;
  const int64_t b = n / p.S, s = n - b * p.S;
  const int rows = 64 / units;  // heads of a wave
  const int row = lane / units, u = lane - row * units;
  const int turning = HALVES ? p.pairs / V : 2 * p.pairs / V;  // units that turn; the others are copied
  const bool turns = u < turning;
  const int c0 = HALVES && !turns ? 2 * p.pairs + (u - turning) * V : u * V;
  const int first = row < rows ? (int)(wave - n * parts) * rows + row : 1 << 30, step = rows * parts;

  struct Piece { T v[V]; };
  auto load = [&](const RopeAxesTensor& x, int h, Piece (&d)[kRows][N]) {
    const T* in = (const T*)x.in + b * x.in_b + s * x.in_s + c0;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (h + k * step >= x.heads) continue;
      const T* from = in + (h + k * step) * x.in_h;
      __builtin_memcpy(&d[k][0], __builtin_assume_aligned(from, 16), 16);
      if (HALVES && turns) __builtin_memcpy(&d[k][N - 1], __builtin_assume_aligned(from + p.pairs, 16), 16);
    }
  };
  Piece d[kRows][N];
  load(p.t[0], first, d);
  float2* mine = turn[threadIdx.x >> 6];
  for (int j = lane; j < p.pairs; j += 64) mine[j] = turn_of(p, j, b, s);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's own: no barrier
  __builtin_amdgcn_wave_barrier();
  float2 cs[P];
  if (turns) {
#pragma unroll
    for (int i = 0; i < P; ++i) cs[i] = mine[(HALVES ? c0 : c0 >> 1) + i];
  }
  for (int w = 0; w < 2; ++w) {
    const RopeAxesTensor& x = p.t[w];
    T* out = (T*)x.out + b * x.out_b + s * x.out_s + c0;
    for (int h = first; h < x.heads; h += kRows * step) {
      if (w || h != first) load(x, h, d);
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        if (h + k * step >= x.heads) continue;
        if (turns) {
#pragma unroll
          for (int i = 0; i < P; ++i) {
            T& y0 = HALVES ? d[k][0].v[i] : d[k][0].v[2 * i];
            T& y1 = HALVES ? d[k][N - 1].v[i] : d[k][0].v[2 * i + 1];
            const float x0 = (float)y0, x1 = (float)y1;
            y0 = (T)(x0 * cs[i].x - x1 * cs[i].y);
            y1 = (T)(x1 * cs[i].x + x0 * cs[i].y);
          }
        }
        T* to = out + (h + k * step) * x.out_h;
        __builtin_memcpy(__builtin_assume_aligned(to, 16), &d[k][0], 16);
        if (HALVES && turns) __builtin_memcpy(__builtin_assume_aligned(to + p.pairs, 16), &d[k][N - 1], 16);
      }
    }
  }
}

// Whether every head's channels, and the pairs in them, are whole 16-byte pieces.
bool in_pieces(const RopeAxesParams& p) {
  const int v = p.dtype == 2 ? 4 : 8;
  if (p.D % v || (p.halves ? p.pairs : 2 * p.pairs) % v) return false;
  for (const RopeAxesTensor& t : p.t) {
    if (((uintptr_t)t.in | (uintptr_t)t.out) & 15u) return false;
    for (int64_t st : {t.in_b, t.in_s, t.in_h, t.out_b, t.out_s, t.out_h})
      if (st % v) return false;
  }
  return true;
}

template <typename T>
void launch(const RopeAxesParams& p, hipStream_t stream) {
  const int64_t all = p.B * p.S;
  if (!in_pieces(p)) {
    hipLaunchKernelGGL(rope_axes_scalar<T>, dim3((unsigned)all), dim3(256), 0, stream, p);
    return;
  }
  const int v = 16 / (int)sizeof(T);
  const int units = (p.halves ? p.D - p.pairs : p.D) / v, rows = 64 / units;
  // Few tokens: their heads are shared out until the chip has its waves, each computing the sines again (64 tokens of 48
  // heads: 6.8 us with a wave to a token, 4.5 with 16; 8,192 tokens: 33 and 66).
  const int most = max(p.t[0].heads, p.t[1].heads);
  int parts = 1;
  while (parts < 16 && all * parts < 8192 && parts * rows < most) parts *= 2;
  const dim3 grid((unsigned)((all * parts + 3) / 4));
  if (p.halves)
    hipLaunchKernelGGL((rope_axes_vec<T, true>), grid, dim3(256), 0, stream, p, units, parts);
  else
    hipLaunchKernelGGL((rope_axes_vec<T, false>), grid, dim3(256), 0, stream, p, units, parts);
}

}  // namespace

hipError_t launch_rope_axes(const RopeAxesParams& p, hipStream_t stream) {
  if (p.dtype == 0)
    launch<__bf16>(p, stream);
  else if (p.dtype == 1)
    launch<_Float16>(p, stream);
  else
    launch<float>(p, stream);
  return hipGetLastError();
}

}  // namespace pasa
