// New keys and values into the cache in 8 bits.
//
// Token t goes to slot = page * page_size + offset; slots that are negative or past the cache are skipped.  Tokens that
// follow each other in consecutive slots of one page are a run, and a run is written by one workgroup for each head and
// for k and v.  With amax the largest finite magnitude of the run's values:
//   e = smallest integer with amax <= 448 * 2 ** e, in [-50, 50];  in a page that goes on (offset > 0) at least the
//       page's own exponent
//   code = e4m3(x * 2 ** -e), to nearest, ties to even; what is not finite is stored as NaN
// and where e rises, the page's other codes are scaled by 2 ** (old e - e).  A run at offset 0 begins the page anew.
//
// Bound by HBM: 2 bytes in and 1 out of each value (10,800 tokens x 40 heads x 128 channels: 84 us, 3.9 TB/s; single
// values at a time, 623).  A thread's item is four tokens x eight channels, and the workgroup
// has as many threads as a page has items, so that a run stays in registers between the maximum and the codes.  k goes out as 8 bytes a token, v as words of
// four tokens, which is the way round it lies in the cache; runs of 16 tokens and more pass through LDS so that its rows
// leave in 16-byte pieces.  16-bit values are compared and converted two at a time as they lie in memory.
#include <type_traits>

#include "common.h"
#include "kv_cache.h"

namespace pasa {

namespace {

constexpr int kMaxPage = 128;
constexpr int kMaxThreads = 512;  // 128 tokens x 128 channels / (4 * 8)

// e4m3 of y, |y| <= 448 (or clamped to it); what is not finite becomes NaN.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  const float y = fminf(fmaxf(x * inv, -448.f), 448.f);
  const uint32_t c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xffu;
  const bool finite = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
  return finite ? c : 0x7fu;
}

// A word of codes times f (a power of two below 1), but for the bytes in `keep` and NaN.
__device__ __forceinline__ uint32_t rescaled4(uint32_t w, float f, uint32_t keep) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * f, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * f, 0, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_cvt_f32_fp8((int)w, 2) * f, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * f, v, true);
  const uint32_t nan = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  keep |= nan | (nan - (nan >> 7));
  return (w & keep) | ((uint32_t)v & ~keep);
}

// Bytes of a word whose positions p0 .. p0 + 3 lie in [a, b).
__device__ __forceinline__ uint32_t bytes_in(int p0, int a, int b) {
  uint32_t m = 0u;
#pragma unroll
  for (int k = 0; k < 4; ++k) m |= p0 + k >= a && p0 + k < b ? 0xffu << (8 * k) : 0u;
  return m;
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

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// Two 16-bit values to two codes of x * 2 ** -e (scale: 2 ** e), into the half `hi` of a word.
template <typename T>
__device__ __forceinline__ s16x2_t pair_codes(s16x2_t w, uint32_t x, float scale, bool hi) {
  if constexpr (std::is_same_v<T, __bf16>)
    return hi ? __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2_t, x), scale, true)
              : __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2_t, x), scale, false);
  else
    return hi ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2_t, x), scale, true)
              : __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2_t, x), scale, false);
}

// Eight channels of a token as they lie in memory.
template <typename T>
struct Raw {
  static constexpr int W = 2 * sizeof(T);  // words
  uint32_t w[W];
  __device__ __forceinline__ void load(const T* x, int d0, int D, bool vec) {
    if (vec && d0 + 8 <= D) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(x + d0)[i];
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    } else {
      T v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = d0 + i < D ? x[d0 + i] : (T)0.f;
      __builtin_memcpy(w, v, sizeof(v));
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else if constexpr (std::is_same_v<T, __bf16>) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    else return (float)__builtin_bit_cast(f16x2_t, w[i >> 1])[i & 1];
  }
};

// An item's largest magnitude as the bits of its type (in both halves of the word for a 16-bit one): as unsigned
// numbers they are in the magnitudes' order, infinity and NaN above all others.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Raw<T> (&r)[4]) {
  uint32_t top = 0u;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < Raw<T>::W; ++i) {
      if constexpr (sizeof(T) == 4)
        top = max(top, r[k].w[i] & 0x7fffffffu);
      else
        top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, top), __builtin_bit_cast(u16x2_t, r[k].w[i] & 0x7fff7fffu)));
    }
  return top;
}
template <typename T>
__device__ __forceinline__ float from_bits(uint32_t top) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(top);
  const uint32_t t = max(top & 0xffffu, top >> 16);
  if constexpr (std::is_same_v<T, __bf16>) return __uint_as_float(t << 16);
  else return (float)__builtin_bit_cast(f16x2_t, t)[0];
}

// Codes of channels 4 i .. 4 i + 3 of a token, and of channel i of four tokens.  careful: some value of the run is not
// finite, or past the largest exponent.
template <typename T>
__device__ __forceinline__ uint32_t codes_along(const Raw<T>& r, int i, int e, bool careful) {
  const float inv = exp2_int(-e);
  if (careful) return code_of(r.at(4 * i), inv) | code_of(r.at(4 * i + 1), inv) << 8 | code_of(r.at(4 * i + 2), inv) << 16 | code_of(r.at(4 * i + 3), inv) << 24;
  if constexpr (sizeof(T) == 4) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(r.at(4 * i) * inv, r.at(4 * i + 1) * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(r.at(4 * i + 2) * inv, r.at(4 * i + 3) * inv, w, true);
  } else {
    s16x2_t w = {0, 0};
    w = pair_codes<T>(w, r.w[2 * i], exp2_int(e), false);
    return __builtin_bit_cast(uint32_t, pair_codes<T>(w, r.w[2 * i + 1], exp2_int(e), true));
  }
}
template <typename T>
__device__ __forceinline__ uint32_t codes_across(const Raw<T> (&r)[4], int i, int e, bool careful) {
  const float inv = exp2_int(-e);
  if (careful) return code_of(r[0].at(i), inv) | code_of(r[1].at(i), inv) << 8 | code_of(r[2].at(i), inv) << 16 | code_of(r[3].at(i), inv) << 24;
  if constexpr (sizeof(T) == 4) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(r[0].at(i) * inv, r[1].at(i) * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(r[2].at(i) * inv, r[3].at(i) * inv, w, true);
  } else {
    const uint32_t pick = i & 1 ? 0x07060302u : 0x05040100u;  // the same half of two words
    s16x2_t w = {0, 0};
    w = pair_codes<T>(w, __builtin_amdgcn_perm(r[1].w[i >> 1], r[0].w[i >> 1], pick), exp2_int(e), false);
    return __builtin_bit_cast(uint32_t, pair_codes<T>(w, __builtin_amdgcn_perm(r[3].w[i >> 1], r[2].w[i >> 1], pick), exp2_int(e), true));
  }
}

// The run of n tokens from token t on, at slot s and those behind it.  ALL: by the whole workgroup, else by one wave.
template <typename T, bool ALL>
__device__ __forceinline__ void append_run(const KvAppendParams& p, int h, int is_v, int64_t t, int64_t s, int n, float* wave_max, uint32_t* vt) {
  const int tid = ALL ? threadIdx.x : threadIdx.x & 63, threads = ALL ? blockDim.x : 64;
  const T* x = (const T*)p.x[is_v] + h * p.head_stride[is_v];
  const int64_t tok_stride = p.tok_stride[is_v];
  const bool vec = p.vec[is_v];
  int8_t* exps = is_v ? p.c.v_exp : p.c.k_exp;
  uint8_t* codes = is_v ? p.c.v : p.c.k;
  const int page = 1 << p.c.page_log2, off = (int)(s & (page - 1));
  const int D = p.c.head_dim, dim = p.c.dim, chunks = dim >> 3, chunks_log2 = dim == 128 ? 4 : 3;

  // Item (pg, c): positions 4 pg .. + 3 of the page, channels 8 c .. + 7.
  const int pg0 = off >> 2, items = (((off + n + 3) >> 2) - pg0) << chunks_log2;
  // One item a thread at most: the threads are a page's items, or the run is short enough for a wave.
  const int pos = 4 * (pg0 + (tid >> chunks_log2)), d0 = 8 * (tid & (chunks - 1));
  Raw<T> raw[4];
  {
    const T* from = x + (t + pos - off) * tok_stride;
#pragma unroll
    for (int k = 0; k < 4; ++k, from += tok_stride) {
      const int j = pos + k - off;
      if (tid < items && j >= 0 && j < n) raw[k].load(from, d0, D, vec);
      else raw[k].zero();
    }
  }
  const int64_t at = (s >> p.c.page_log2) * p.c.heads + h;
  const int had = off == 0 ? kKvExpMin : min(max((int)exps[at], kKvExpMin), kKvExpMax);
  float most = from_bits<T>(top_bits<T>(raw));
  const bool odd = !(most < INFINITY);  // something is not finite: it does not count
  if (__any(odd)) {
    most = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(raw[k].at(e));
        most = a < INFINITY ? fmaxf(most, a) : most;
      }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) most = fmaxf(most, __shfl_xor(most, m, 64));
  bool careless;
  if constexpr (ALL) {
    if ((tid & 63) == 0) wave_max[tid >> 6] = most;
    careless = !__syncthreads_or(odd);
    for (int w = 0; w < threads / 64; ++w) most = fmaxf(most, wave_max[w]);
  } else {
    careless = !__any(odd);
  }
  const int e_new = max(had, exponent_of(most));
  const bool careful = !careless || e_new == kKvExpMax;
  uint8_t* out = codes + at * ((int64_t)page * dim);
  if (tid == 0) exps[at] = (int8_t)e_new;  // (every thread has read it: the barrier above, or its wave's own order)
  if (off != 0 && e_new != had) {
    const float f = exp2_int(had - e_new);
    uint32_t* words = reinterpret_cast<uint32_t*>(out);
    for (int e = tid; e < page * dim / 4; e += threads) {
      const int pos = is_v ? 4 * e & (page - 1) : 4 * e / dim;
      const uint32_t mine = is_v ? bytes_in(pos, off, off + n) : pos >= off && pos < off + n ? 0xffffffffu : 0u;
      if (mine != 0xffffffffu) {
        // The run's own bytes of the word are written below, after a barrier.
        const uint32_t old = words[e], now = rescaled4(old, f, mine);
        if (now != old) words[e] = now;
      }
    }
    if constexpr (ALL) {
      __syncthreads();
    } else {
      __threadfence_block();  // the wave's stores arrive before those that follow
      __builtin_amdgcn_wave_barrier();
    }
  }
  const bool through_lds = ALL && is_v && n >= 16;
  const int row_words = page / 4 + 1;
  if (tid < items) {
    if (!is_v) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = pos + k - off;
        if (j < 0 || j >= n) continue;
        *reinterpret_cast<uint2*>(out + (pos + k) * dim + d0) =
            make_uint2(codes_along<T>(raw[k], 0, e_new, careful), codes_along<T>(raw[k], 1, e_new, careful));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = codes_across<T>(raw, i, e_new, careful);
        if (through_lds) {
          vt[(d0 + i) * row_words + (pos >> 2)] = w;
        } else {
          uint8_t* to = out + (d0 + i) * page + pos;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (pos + k >= off && pos + k < off + n) to[k] = (uint8_t)(w >> (8 * k));
        }
      }
    }
  }
  if (through_lds) {
    __syncthreads();
    // 16 positions of a channel at a time; the first and last of the run may be cut.
    const int u0 = off >> 4, units = ((off + n + 15) >> 4) - u0;
    for (int e = tid; e < units * dim; e += threads) {
      const int d = e / units, pos = 16 * (u0 + e - d * units);
      const uint32_t* from = vt + d * row_words + (pos >> 2);
      uint8_t* to = out + d * page + pos;
      if (pos >= off && pos + 16 <= off + n) {
        *reinterpret_cast<uint4*>(to) = make_uint4(from[0], from[1], from[2], from[3]);
      } else {
        for (int k = max(off - pos, 0); k < min(off + n - pos, 16); ++k) to[k] = (uint8_t)(from[k >> 2] >> (8 * (k & 3)));
      }
    }
  }
}

// blockIdx.x: the runs that begin among `window` tokens; y: the head; z: k or v.  Runs of up to 64 items (one of a lane's)
// are the waves', one each; the workgroup takes the longer ones together.
template <typename T>
__global__ __launch_bounds__(kMaxThreads, sizeof(T) == 4 ? 4 : 6) void kv_append(KvAppendParams p, int window) {
  __shared__ int64_t slots[64 + kMaxPage + 1];  // of tokens t0 - 1 ..
  __shared__ float wave_max[kMaxThreads / 64];
  __shared__ uint64_t long_runs;
  extern __shared__ uint32_t vt[];  // v's codes, dim rows of page / 4 words and one more: rows start in other banks
  const int tid = threadIdx.x, lane = tid & 63, threads = blockDim.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.y, is_v = blockIdx.z;
  const int page = 1 << p.c.page_log2;
  const int64_t t0 = (int64_t)blockIdx.x * window;
  const int64_t t1 = min(p.tokens, t0 + window);
  const int64_t end = min(p.tokens, t1 + page);
  const int64_t limit = (int64_t)p.c.num_pages << p.c.page_log2;
  if (tid == 0) long_runs = 0u;
  for (int64_t t = t0 - 1 + tid; t < end; t += threads) {
    const int64_t s = t < 0 ? -2 : p.slots[t];
    slots[t - (t0 - 1)] = s < 0 || s >= limit ? -2 : s;
  }
  __syncthreads();

  // A token begins a run unless the one before it has the slot before, in the same page.
  uint64_t starts;
  {
    const int i = lane + 1;
    const bool in = t0 + lane < t1;
    const int64_t s = in ? slots[i] : -2;
    starts = __ballot(s >= 0 && !(slots[in ? i - 1 : 0] == s - 1 && (s & (page - 1)) != 0));
  }
  // The length of the run at token t0 + i - 1: how many of the next tokens have the next slots.
  auto length = [&](int i) {
    const int64_t t = t0 + i - 1, s = slots[i];
    const int off = (int)(s & (page - 1));
    auto follows = [&](int k) { return off + k < page && t + k < end && slots[i + k] == s + k; };
    const uint64_t m0 = __ballot(follows(1 + lane)), m1 = __ballot(follows(65 + lane));
    return 1 + (~m0 ? __builtin_ctzll(~m0) : 64 + (~m1 ? __builtin_ctzll(~m1) : 64));
  };
  int turn = 0;
  for (uint64_t left = starts; left != 0u; left &= left - 1) {
    if (turn++ % (threads / 64) != wave) continue;
    const int i = __builtin_ctzll(left) + 1, n = length(i);
    const int64_t s = slots[i];
    const int off = (int)(s & (page - 1));
    if (((off + n + 3) / 4 - off / 4) * (p.c.dim / 8) <= 64)
      append_run<T, false>(p, h, is_v, t0 + i - 1, s, n, wave_max, vt);
    else if (lane == 0)
      atomicOr((unsigned long long*)&long_runs, left & -left);
  }
  __syncthreads();
  for (uint64_t left = long_runs; left != 0u; left &= left - 1) {
    const int i = __builtin_ctzll(left) + 1, n = length(i);
    append_run<T, true>(p, h, is_v, t0 + i - 1, slots[i], n, wave_max, vt);
    __syncthreads();  // wave_max and vt are read before the next run
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppendParams& p, hipStream_t stream) {
  // A workgroup for 64 tokens, or fewer where that leaves less than 2,048 workgroups: runs of single tokens have a wave
  // each, and one behind the other takes 3 us (64 tokens x 8 heads in 64 pages: 6.6 us with a workgroup for each, 54 for
  // all 64 in one; 1,024 tokens x 8 heads: in runs of 64 13.5 for 8 a workgroup, 40 for one; in single ones 23 and 44).
  const int64_t halves = 2 * p.tokens * p.c.heads / 2048;
  int window = 1;
  while (window < 64 && 2 * window <= halves) window *= 2;
  const int64_t wgs = (p.tokens + window - 1) / window;
  if (wgs > 0x7fffffff || p.c.heads > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs, (unsigned)p.c.heads, 2);
  const int items = (p.c.dim << p.c.page_log2) / 32;
  const dim3 block(items < 64 ? 64 : items);
  const size_t lds = p.c.dim * ((1 << p.c.page_log2) / 4 + 1) * sizeof(uint32_t);
  if (p.dtype == 0)
    hipLaunchKernelGGL(kv_append<__bf16>, grid, block, lds, stream, p, window);
  else if (p.dtype == 1)
    hipLaunchKernelGGL(kv_append<_Float16>, grid, block, lds, stream, p, window);
  else
    hipLaunchKernelGGL(kv_append<float>, grid, block, lds, stream, p, window);
  return hipGetLastError();
}

}  // namespace pasa
