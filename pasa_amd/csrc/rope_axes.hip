// Rotary embedding from positions on several axes.
//
// Pair i of a head's channels turns by the angle a_i = pos[axis_i][token] * f_i:
//   y0 = x0 cos a_i - x1 sin a_i,   y1 = x1 cos a_i + x0 sin a_i
// with (x0, x1) = channels (2 i, 2 i + 1), or (i, i + pairs); channels from 2 * pairs on are copied.  The inverse
// (the gradient) turns by -a_i.  The angle is taken in fp64 as a share of a full turn, reduced to half a turn
// either way, and only then rounded to fp32, so a position far out costs no accuracy; the rotation is fp32 and
// rounded once.
//
// Bound by HBM: each channel is read once and written once, positions are 12 bytes a token.  A workgroup computes
// the sines of its tokens once, into LDS, and all heads of q and k read them there.
#include <math.h>

#include "common.h"
#include "kv_cache.h"

namespace pasa {

namespace {

constexpr int kMaxPairs = 128;
constexpr int kMaxTokens = 8;  // tokens of a workgroup
constexpr double kInvTwoPi = 0.15915494309189533576888;

__device__ __forceinline__ double position(const RopeAxesParams& p, int64_t at) {
  if (p.pos_type == kPosI32) return (double)((const int32_t*)p.pos)[at];
  if (p.pos_type == kPosI64) return (double)((const int64_t*)p.pos)[at];
  return (double)((const float*)p.pos)[at];
}

// One element at a time: any stride, alignment and number of pairs.
template <typename T>
__global__ __launch_bounds__(256) void rope_axes_scalar(RopeAxesParams p, int toks) {
  __shared__ float2 cs[kMaxTokens][kMaxPairs];
  const int tid = threadIdx.x;
  const int64_t n0 = (int64_t)blockIdx.x * toks;
  const int64_t all = p.B * p.S;
  const int cnt = (int)min((int64_t)toks, all - n0);
  for (int i = tid; i < cnt * p.pairs; i += 256) {
    const int t = i / p.pairs, j = i - t * p.pairs;
    const int64_t n = n0 + t, b = n / p.S, s = n - b * p.S;
    const int ax = min(max(p.axis[j], 0), p.axes - 1);
    double turn = position(p, ax * p.pos_axis + b * p.pos_b + s * p.pos_s) * p.inv_freq[j] * kInvTwoPi;
    turn -= rint(turn);
    float sn, cn;
    sincospif((float)(2.0 * turn), &sn, &cn);
    cs[t][j] = make_float2(cn, p.inverse ? -sn : sn);
  }
  __syncthreads();
  const int rest = p.D - 2 * p.pairs;
  const int units = p.pairs + rest;  // a pair, or a channel to copy
  const int heads = p.t[0].heads + p.t[1].heads;
  for (int i = tid; i < cnt * heads * units; i += 256) {
    const int u = i % units, th = i / units;
    const int t = th / heads;
    int h = th - t * heads;
    const int w = h >= p.t[0].heads;
    if (w) h -= p.t[0].heads;
    const RopeAxesTensor& x = p.t[w];
    const int64_t n = n0 + t, b = n / p.S, s = n - b * p.S;
    const T* in = (const T*)x.in + b * x.in_b + s * x.in_s + h * x.in_h;
    T* out = (T*)x.out + b * x.out_b + s * x.out_s + h * x.out_h;
    if (u < p.pairs) {
      const int c0 = p.halves ? u : 2 * u, c1 = p.halves ? u + p.pairs : 2 * u + 1;
      const float x0 = (float)in[c0], x1 = (float)in[c1];
      const float2 a = cs[t][u];
      out[c0] = (T)(x0 * a.x - x1 * a.y);
      out[c1] = (T)(x1 * a.x + x0 * a.y);
    } else {
      const int c = p.pairs + u;
      out[c] = in[c];
    }
  }
}

}  // namespace

hipError_t launch_rope_axes(const RopeAxesParams& p, hipStream_t stream) {
  const int64_t all = p.B * p.S;
  const int toks = 1;
  const int64_t wgs = (all + toks - 1) / toks;
  if (wgs > 0x7fffffff) return hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs);
  if (p.dtype == 0)
    hipLaunchKernelGGL(rope_axes_scalar<__bf16>, grid, dim3(256), 0, stream, p, toks);
  else if (p.dtype == 1)
    hipLaunchKernelGGL(rope_axes_scalar<_Float16>, grid, dim3(256), 0, stream, p, toks);
  else
    hipLaunchKernelGGL(rope_axes_scalar<float>, grid, dim3(256), 0, stream, p, toks);
  return hipGetLastError();
}

}  // namespace pasa
