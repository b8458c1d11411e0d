// New keys and values into the cache in 8 bits.
//
// Token t goes to slot = page * page_size + offset; slots that are negative or past the cache are skipped.  Tokens that
// follow each other in consecutive slots of one page are a run, and a run is written by one workgroup for each head and
// for k and v.  With amax the largest finite magnitude of the run's values:
//   e = smallest integer with amax <= 448 * 2 ** e, in [-50, 50];  in a page that goes on (offset > 0) at least the
//       page's own exponent
//   code = e4m3(x * 2 ** -e), to nearest, ties to even; what is not finite is stored as NaN
// and where e rises, the page's other codes are scaled by 2 ** (old e - e).  A run at offset 0 begins the page anew.
#include "common.h"
#include "kv_cache.h"

namespace pasa {

namespace {

constexpr int kMaxPage = 128;

// e4m3 of x * inv (|x * inv| <= 448 for finite x, or clamped to it); what is not finite becomes NaN.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  const float y = fminf(fmaxf(x * inv, -448.f), 448.f);
  const uint32_t c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xffu;
  const bool finite = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
  return finite ? c : 0x7fu;
}

__device__ __forceinline__ uint8_t rescaled(uint8_t c, float f) {
  if ((c & 0x7f) == 0x7f) return c;
  const float y = __builtin_amdgcn_cvt_f32_fp8((int)c, 0) * f;
  return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xff);
}

// Smallest e with amax <= 448 * 2 ** e: 448 = 1.75 * 2 ** 8.
__device__ __forceinline__ int exponent_of(float amax) {
  const uint32_t b = __float_as_uint(amax);
  if (b < 0x00800000u) return kKvExpMin;  // zero and subnormal
  const int x = (int)(b >> 23) - 127;
  const int e = x - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kKvExpMin), kKvExpMax);
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

template <typename T>
__global__ __launch_bounds__(256) void kv_append(KvAppendParams p, int window) {
  __shared__ int64_t slots[64 + kMaxPage + 1];  // of tokens t0 - 1 ..
  __shared__ float wave_max[4];
  const int tid = threadIdx.x, nt = blockDim.x;
  const int h = blockIdx.y, is_v = blockIdx.z;
  const int page = 1 << p.c.page_log2;
  const int64_t t0 = (int64_t)blockIdx.x * window;
  const int64_t t1 = min(p.tokens, t0 + window);
  const int64_t end = min(p.tokens, t1 + page);
  const int64_t limit = (int64_t)p.c.num_pages << p.c.page_log2;
  for (int64_t t = t0 - 1 + tid; t < end; t += nt) {
    const int64_t s = t < 0 ? -2 : p.slots[t];
    slots[t - (t0 - 1)] = s < 0 || s >= limit ? -2 : s;
  }
  __syncthreads();
  const T* x = (const T*)p.x[is_v] + h * p.head_stride[is_v];
  int8_t* exps = is_v ? p.c.v_exp : p.c.k_exp;
  uint8_t* codes = is_v ? p.c.v : p.c.k;
  const int D = p.c.head_dim, dim = p.c.dim;

  for (int64_t t = t0; t < t1; ++t) {
    const int i = (int)(t - t0) + 1;
    const int64_t s = slots[i];
    const int off = (int)(s & (page - 1));
    if (s < 0 || (slots[i - 1] == s - 1 && off != 0)) continue;  // no slot, or inside an earlier token's run
    int n = 1;
    while (off + n < page && t + n < end && slots[i + n] == s + n) ++n;

    float most = 0.f;
    for (int e = tid; e < n * D; e += nt) {
      const int j = e / D, d = e - j * D;
      const float a = fabsf((float)x[(t + j) * p.tok_stride[is_v] + d]);
      if (a < INFINITY) most = fmaxf(most, a);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) most = fmaxf(most, __shfl_xor(most, m, 64));
    __syncthreads();  // the last run's maxima are read
    if ((tid & 63) == 0) wave_max[tid >> 6] = most;
    const int64_t at = (s >> p.c.page_log2) * p.c.heads + h;
    const int had = off == 0 ? kKvExpMin : min(max((int)exps[at], kKvExpMin), kKvExpMax);
    __syncthreads();
    for (int w = 0; w < nt / 64; ++w) most = fmaxf(most, wave_max[w]);
    const int e_new = max(had, exponent_of(most));
    const float inv = exp2_int(-e_new);
    uint8_t* out = codes + at * ((int64_t)page * dim);
    if (off != 0 && e_new != had) {
      const float f = exp2_int(max(had - e_new, -126));
      for (int e = tid; e < page * dim; e += nt) {
        const int j = is_v ? e & (page - 1) : e / dim;
        if (j < off || j >= off + n) out[e] = rescaled(out[e], f);
      }
    }
    for (int e = tid; e < n * dim; e += nt) {
      const int j = e / dim, d = e - j * dim;
      const uint32_t c = d < D ? code_of((float)x[(t + j) * p.tok_stride[is_v] + d], inv) : 0u;
      out[is_v ? d * page + off + j : (off + j) * dim + d] = (uint8_t)c;
    }
    if (tid == 0) exps[at] = (int8_t)e_new;
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppendParams& p, hipStream_t stream) {
  const int window = p.tokens <= 1024 ? 1 : 64;
  const int64_t wgs = (p.tokens + window - 1) / window;
  if (wgs > 0x7fffffff || p.c.heads > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs, (unsigned)p.c.heads, 2);
  const dim3 block(window == 1 ? 64 : 256);
  if (p.dtype == 0)
    hipLaunchKernelGGL(kv_append<__bf16>, grid, block, 0, stream, p, window);
  else if (p.dtype == 1)
    hipLaunchKernelGGL(kv_append<_Float16>, grid, block, 0, stream, p, window);
  else
    hipLaunchKernelGGL(kv_append<float>, grid, block, 0, stream, p, window);
  return hipGetLastError();
}

}  // namespace pasa
