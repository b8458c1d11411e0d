// Softmax attention to the key/value cache in 8 bits.
//
// Request r has n new tokens (rows of q) and len[r] cached ones, its own included.  Token i of it sits at position
// pos = len - n + i and sees the keys j with j < len, j <= pos if causal, j > pos - window with a window, and a page in
// the table.  With a page's exponents ke, ve:
//   s_j = scale 2^ke q.k8_j,   o = sum_j 2^(s_j - m) 2^ve v8_j / sum_j 2^(s_j - m)        (scale holds log2 e)
// m is a running maximum of s_j + ve (short of it by at most 8), so that p_j = 2^(s_j + ve - m + 7) <= 2^15 carries the
// page's scale and stays inside fp16's normal numbers down to 2^-21 of 2^m; the row sum takes p_j 2^-ve, which is exact.
// Rows that see no key get 0, and -inf as the logarithm of their sum.
//
// The codes go to the matrix unit as they lie in memory.  Both products contract over what is contiguous in the cache,
// and a contraction may run in any order, so a lane's operand is 16 consecutive bytes, widened in registers: e4m3 is
// exact in both 16-bit types.  q.k runs in q's type, p.v in fp16 whatever q's type is: p then has 11 bits, not 8.
// Per 64-key tile, lane (m, g) = (lane % 16, lane / 16):
//   S^T = K Q^T   A row m of 16-key tile t is key 16 (m / 4) + 4 t + m % 4, so that the lane's 16 results are
//                 keys 16 g .. 16 g + 15 of row m of q: one page, one pair of exponents
//   O^T += V^T P^T  A row m of 16-channel tile dt is channel 16 dt + m, k-slots keys 16 g + 8 u .. + 7 of step u:
//                 the lane's own results as they stand, and 16 bytes of V
#include <math.h>

#include <type_traits>

#include "common.h"
#include "kv_cache.h"

namespace pasa {

namespace {

constexpr float kShift = 7.f;
constexpr float kSlack = 8.f;
constexpr float kLn2 = 0.69314718055994530942f;

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// Eight e4m3 codes as eight values of a 16-bit type, exactly.
__device__ __forceinline__ f16x8_t widen_f16(uint32_t lo, uint32_t hi) {
  const f16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
  const f16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const f16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
  const f16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return (f16x8_t){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ bf16x8_t widen_bf16(uint32_t lo, uint32_t hi) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return (bf16x8_t){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <typename E>
__device__ __forceinline__ typename E::vec8 widen(uint32_t lo, uint32_t hi) {
  if constexpr (std::is_same_v<E, F16>) return widen_f16(lo, hi);
  else return widen_bf16(lo, hi);
}

// A byte mask of the first n (0 .. 4) bytes of a word.
__device__ __forceinline__ uint32_t first_bytes(int n) {
  return n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
}
// 0x80 in each byte that is e4m3's NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// A word of codes with 0 in the place of each NaN.
__device__ __forceinline__ uint32_t finite_bytes(uint32_t w) {
  const uint32_t n = nan_bytes(w);
  return w & ~(n | (n - (n >> 7)));
}

// The requests' first rows of q, clamped to the rows that there are.
// (tokens * q_heads < 2^31: row numbers fit 32 bits.)
__device__ __forceinline__ int first_token(const KvAttnParams& p, int r) {
  return min(max(p.cu_q[r], 0), (int)p.tokens);
}

// Tile `id` of the launch: request r (requests: the rows behind the last one), its first token and rows, the tile's first
// row, and the request's length.  The tiles of a request are numbered from floor(first row / TILE) + r, which leaves room
// for every request's last, part-filled one without a sum over the requests before it.
struct TileOf {
  int r, tok0, rows, row0, raw_len;
  int front;  // tile 0 only: the first request's first token
};
template <int TILE>
__device__ __forceinline__ TileOf find_tile(const KvAttnParams& p, int id) {
  // The last request whose number is at or before id: 64 candidates at a time, one for each lane, which in the last round
  // (the only one for up to 63 requests) also has its request's length.
  TileOf t;
  if (p.cu_q == nullptr) {  // the same for all: no more numbers than tiles
    t.rows = p.per_request * p.group;
    const int each = (t.rows + TILE - 1) / TILE;
    t.r = id / each;
    t.tok0 = t.r * p.per_request;
    t.row0 = (id - t.r * each) * TILE;
    t.raw_len = max(p.lens[t.r], 0);
    t.front = 0;
    return t;
  }
  const int lane = threadIdx.x & 63;
  int lo = 0, n = p.requests + 1;
  auto number = [&](int first, int r) { return first * p.group / TILE + r; };
  while (n > 64) {
    const int step = (n + 63) >> 6, at = lo + min(lane * step, n - 1);
    const int before = max(__popcll(__ballot(lane * step < n && number(first_token(p, at), at) <= id)), 1) - 1;
    lo += before * step;
    n = min(step, n - before * step);
  }
  const int at = min(lo + lane, p.requests);
  const int first = first_token(p, at), len = p.lens[min(at, p.requests - 1)];
  const int i = max(__popcll(__ballot(lane < n && number(first, at) <= id)), 1) - 1;
  t.r = lo + i;
  t.tok0 = __builtin_amdgcn_readlane(first, i);
  const int tok1 = t.r == p.requests ? (int)p.tokens : i < 63 ? __builtin_amdgcn_readlane(first, min(i + 1, 63)) : first_token(p, t.r + 1);
  t.rows = (max(tok1, t.tok0) - t.tok0) * p.group;
  t.row0 = (id - number(t.tok0, t.r)) * TILE;
  t.raw_len = max(__builtin_amdgcn_readlane(len, i), 0);
  t.front = __builtin_amdgcn_readlane(first, 0);  // (only request 0 has a number that tile 0 reaches)
  return t;
}

// What position pos of a request of len keys sees: [sees_lo, sees_hi).
__device__ __forceinline__ int sees_lo(const KvAttnParams& p, int64_t pos, int len) {
  return p.window ? (int)min(max(pos - p.window + 1, (int64_t)0), (int64_t)len) : 0;
}
__device__ __forceinline__ int sees_hi(const KvAttnParams& p, int64_t pos, int len) {
  return p.causal ? (int)min(max(pos + 1, (int64_t)0), (int64_t)len) : len;
}

__device__ __forceinline__ void store_rowpart(const KvAttnParams& p, int64_t tok, int head, int d, float x) {
  if (d >= p.c.head_dim) return;
  const int64_t at = tok * p.o_tok + head * p.o_head + d;
  if (p.f16) ((_Float16*)p.o)[at] = (_Float16)x;
  else ((__bf16*)p.o)[at] = (__bf16)x;
}

// log of a row's sum from its maximum (with the page's exponent) and l.  l's own exponent goes to the maximum first:
// what the page's scale put into both cancels there exactly.
__device__ __forceinline__ float row_lse(float top, float l) {
  if (l == 0.f) return -INFINITY;
  int x;
  const float frac = frexpf(l, &x);
  return kLn2 * ((top + ((float)x - kShift)) + __log2f(frac));
}

// n of the rows of no request, from row0 of token tok0 on.
template <int DIM>
__device__ __forceinline__ void zero_rows(const KvAttnParams& p, int hk, int z, int tok0, int row0, int n) {
  if (!p.zero_tail || z != 0 || p.splits != 1) return;  // with parts, the join writes them
  for (int64_t e = threadIdx.x; e < (int64_t)n * DIM; e += blockDim.x) {
    const int i = row0 + (int)(e / DIM);
    const int64_t tok = tok0 + i / p.group;
    const int head = hk * p.group + i % p.group;
    store_rowpart(p, tok, head, (int)(e % DIM), 0.f);
    if (e % DIM == 0 && p.lse) p.lse[tok * p.q_heads + head] = -INFINITY;
  }
}

// Four channels from d on, times inv.
__device__ __forceinline__ void store4(const KvAttnParams& p, int64_t tok, int head, int d, const f32x4_t& x, float inv) {
  if (p.o_vec && d + 4 <= p.c.head_dim) {
    uint2 w;
    if (p.f16) w = make_uint2(F16::pack2(x[0] * inv, x[1] * inv), F16::pack2(x[2] * inv, x[3] * inv));
    else w = make_uint2(Bf16::pack2(x[0] * inv, x[1] * inv), Bf16::pack2(x[2] * inv, x[3] * inv));
    *reinterpret_cast<uint2*>((uint16_t*)p.o + tok * p.o_tok + head * p.o_head + d) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) store_rowpart(p, tok, head, d + k, x[k] * inv);
  }
}

// A row of q as B operands: channels 64 (s / 2) + 16 g + 8 (s % 2) .. + 7 for k-step s.
template <typename E, int KS>
__device__ __forceinline__ void load_q(const KvAttnParams& p, int64_t tok, int head, int g, typename E::vec8 (&qf)[KS]) {
  const uint16_t* row = (const uint16_t*)p.q + tok * p.q_tok + head * p.q_head;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d0 = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (p.q_vec && d0 + 8 <= p.c.head_dim) {
      const uint4 x = *reinterpret_cast<const uint4*>(row + d0);
      w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d0 + e < p.c.head_dim) w[e >> 1] |= (uint32_t)row[d0 + e] << (16 * (e & 1));
    }
    qf[s] = as_vec8<E>((u32x4_t){w[0], w[1], w[2], w[3]});
  }
}

// The largest of a lane's scores of row tile q, with the page's scales.
template <int NQ>
__device__ __forceinline__ float lane_max(const f32x4_t (&s)[4][NQ], int q, float sc, float ve) {
  float mx = fmaxf(s[0][q][0], s[0][q][1]);
#pragma unroll
  for (int e = 2; e < 16; e += 2) mx = fmaxf(fmaxf(s[e >> 2][q][e & 3], s[e >> 2][q][(e & 3) + 1]), mx);
  return fmaf(mx, sc, ve);
}

// The running maxima, and o and l scaled where one rose.  A rise by less than kSlack is left alone: p then stays below
// 2^(kShift + kSlack), inside fp16, and scaling o's registers is rare.
template <int DT, int NQ>
__device__ __forceinline__ void raise_max(const float (&mx)[NQ], float (&m_run)[NQ], float (&l_run)[NQ], f32x4_t (&o)[DT][NQ]) {
  bool rise = false;
#pragma unroll
  for (int q = 0; q < NQ; ++q) rise = rise | (mx[q] > m_run[q] + kSlack);
  if (__builtin_expect(!__any(rise), 1)) return;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const float m_new = fmaxf(m_run[q], quad16_max(mx[q]));
    const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run[q] - m_new);
    m_run[q] = m_new;
    l_run[q] *= alpha;
    // In place (a plain product makes the compiler copy all of o on the path around it).
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = o[dt][q][i];
        asm("v_mul_f32 %0, %1, %0" : "+v"(x) : "v"(alpha));
        o[dt][q][i] = x;
      }
  }
}

// Scores of row tile q to p, as two k-steps of B operands, and their sum to l (inv: 2^-ve).
template <int NQ>
__device__ __forceinline__ void weights(const f32x4_t (&s)[4][NQ], int q, float sc, float ve, float inv, float m_run, float& l_run,
                                        f16x8_t& p0, f16x8_t& p1) {
  const float off = m_run == -INFINITY ? 0.f : ve - m_run + kShift;
  float sum[2] = {0.f, 0.f};
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const f32x4_t& x = s[e >> 1][q];
    const float a = fast_exp2(fmaf(x[2 * (e & 1)], sc, off));
    const float b = fast_exp2(fmaf(x[2 * (e & 1) + 1], sc, off));
    w[e] = F16::pack2(a, b);
    sum[0] += a;
    sum[1] += b;
  }
  p0 = as_vec8<F16>((u32x4_t){w[0], w[1], w[2], w[3]});
  p1 = as_vec8<F16>((u32x4_t){w[4], w[5], w[6], w[7]});
  l_run = fmaf(sum[0] + sum[1], inv, l_run);
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ int page_exp(int e) { return min(max(e, kKvExpMin), kKvExpMax); }

// 0x8000 in each 16-bit half that is an infinity or NaN (among widened codes: NaN).
__device__ __forceinline__ uint32_t nan_halves(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }

// A tile in LDS that not every row sees whole and that holds a NaN among its values, which must not reach rows that do not
// see its key.  The outputs that it does reach become NaN: 1 at each NaN times 1 at each key that the row sees is above 0
// there.  The products themselves then run on the values without NaN (finite_halves).
template <int DT>
__device__ __forceinline__ void poison_step(const unsigned char* vs, int lane, bool here, int jv, const int (&lo)[2], const int (&hi)[2],
                                            f32x4_t (&o)[DT][2]) {
  uint64_t hits = 0u;  // bit 8 dt + 4 q + i
#pragma unroll 1
  for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      f32x4_t hit = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f16x8_t a = *(reinterpret_cast<const f16x8_t*>(vs + (2 * dt + u) * 1024) + lane);
        f16x8_t ind, seen;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = jv + 8 * u + e;
          ind[e] = (_Float16)(a[e] != a[e] ? 1.f : 0.f);
          seen[e] = (_Float16)(here && j >= lo[q] && j < hi[q] ? 1.f : 0.f);
        }
        hit = F16::mfma16(ind, seen, hit);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (hit[i] > 0.f) hits |= 1ull << (8 * dt + 4 * q + i);
    }
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((hits >> (8 * dt + 4 * q + i)) & 1u) o[dt][q][i] = __uint_as_float(0x7fc00000u);
}

__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  const uint32_t n = nan_halves(w);
  return w & ~(n | (n - (n >> 15)));
}

// ---- few rows --------------------------------------------------------------------
// A workgroup has 16 * NQ rows of one key head; its eight waves take the 64-key tiles in turn, straight from memory into
// registers, and their sums are joined in LDS.  blockIdx.z: a part of the keys.  Bound by the bytes of the keys: eight
// waves a compute unit, each with a tile of 16 KB in flight, ask for more than HBM gives.  2 tokens x 75,600 keys of 40
// heads of 128 channels: 270 us with the join, 5.7 TB/s where a plain read of as much reaches 6.2; 64 tokens to ragged
// lengths up to 8,192, 8 heads: 131 us, 4.3 TB/s (four waves a workgroup: 145).
template <typename E, int DIM, int NQ>
__global__ __launch_bounds__(512, 2) void kv_attn_rows(KvAttnParams p) {
  constexpr int WAVES = 8;
  constexpr int TILE = 16 * NQ, KS = DIM / 32, DT = DIM / 16, HF = DIM / 64;
  using vec8 = typename E::vec8;
  __shared__ float so[WAVES][TILE][DIM + 4];
  __shared__ float sm[WAVES][TILE], sl[WAVES][TILE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int hk = blockIdx.y, z = blockIdx.z;
  const KvCache& c = p.c;
  const int page = 1 << c.page_log2;

  const TileOf tile_of = find_tile<TILE>(p, blockIdx.x);
  if (blockIdx.x == 0 && tile_of.front > 0) zero_rows<DIM>(p, hk, z, 0, 0, tile_of.front * p.group);
  const int r = tile_of.r, tok0 = tile_of.tok0, rows = tile_of.rows, row0 = tile_of.row0, raw_len = tile_of.raw_len;
  if (row0 < 0 || row0 >= rows) return;  // below 0: row starts that do not ascend
  if (r == p.requests) {
    zero_rows<DIM>(p, hk, z, tok0, row0, min(TILE, rows - row0));
    return;
  }
  const int len = (int)min(min((int64_t)raw_len, p.max_kv), p.width << c.page_log2);
  const int64_t pos_base = (int64_t)raw_len - rows / p.group;
  const int32_t* table = p.tables + r * p.table_stride;

  // What the tile's rows see together, in tiles of 64 keys; this part's share of them.
  const int last = min(row0 + TILE, rows) - 1;
  const int klo = sees_lo(p, pos_base + row0 / p.group, len), khi = sees_hi(p, pos_base + last / p.group, len);
  const int tile_lo = klo >> 6, tile_hi = max(tile_lo, (khi + 63) >> 6);
  const int per = (tile_hi - tile_lo + p.splits - 1) / p.splits;
  const int tb = min(tile_lo + z * per, tile_hi), te = min(tb + per, tile_hi);

  // Pages of the lane's K row and of its keys 16 g .. + 15 in a tile, -1 where there is none.
  auto page_of = [&](int j) -> int {
    const int id = table[min(j, len - 1) >> c.page_log2];
    return j < len && (unsigned)id < (unsigned)c.num_pages ? id : -1;
  };
  // A tile's K is asked for when the scores of the one before are done, its V when the sums are, into the same registers.
  int kid = -1, vid = -1, ke_n = 0, ve_n = 0;
  bool here_n = false;
  auto look_up = [&](int tile) {
    kid = page_of(tile * 64 + 16 * (m >> 2));
    vid = page_of(tile * 64 + 16 * g);
  };
  uint4 kr[4][HF], vr[DT];
  auto fetch_k = [&](int tile) {
    const int j = tile * 64 + 16 * (m >> 2);
    const uint8_t* kp = c.k + ((((int64_t)max(kid, 0) * c.heads + hk) << c.page_log2) + (j & (page - 1)) + (m & 3)) * DIM + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int f = 0; f < HF; ++f) kr[t][f] = *reinterpret_cast<const uint4*>(kp + 4 * t * DIM + 64 * f);
  };
  const uint8_t* vp = c.v;
  auto fetch_v = [&](int tile) {
    const int64_t at = (int64_t)max(vid, 0) * c.heads + hk;
    vp = c.v + (((at * DIM) + m) << c.page_log2) + ((tile * 64 + 16 * g) & (page - 1));
    here_n = vid >= 0;
    ke_n = c.k_exp[at];
    ve_n = c.v_exp[at];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vr[dt] = *reinterpret_cast<const uint4*>(vp + ((16 * dt) << c.page_log2));
  };
  if (tb + wave < te) {
    look_up(tb + wave);
    fetch_k(tb + wave);
    fetch_v(tb + wave);
    if (tb + wave + WAVES < te) look_up(tb + wave + WAVES);
  }

  // This lane's rows: what they see is [lo, hi).
  vec8 qf[NQ][KS];
  int lo[NQ], hi[NQ];
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    const int i = min(row0 + 16 * t + m, rows - 1), tok = i / p.group;
    lo[t] = sees_lo(p, pos_base + tok, len);
    hi[t] = sees_hi(p, pos_base + tok, len);
    load_q<E, KS>(p, tok0 + tok, hk * p.group + (i - tok * p.group), g, qf[t]);
  }

  f32x4_t o[DT][NQ];
  float l_run[NQ], m_run[NQ];
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    l_run[t] = 0.f;
    m_run[t] = -INFINITY;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt][t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }

  // Bytes of the lane's keys jv .. + 15 that are the request's.
  auto kept = [&](int jv, bool here) {
    const int n = here ? min(max(len - jv, 0), 16) : 0;
    return make_uint4(first_bytes(n), first_bytes(n - 4), first_bytes(n - 8), first_bytes(n - 12));
  };
  uint32_t poison = 0u;

  for (int tile = tb + wave; tile < te; tile += WAVES) {
    const int jv = tile * 64 + 16 * g;
    const bool here = here_n;
    const int ke = page_exp(ke_n), ve = page_exp(ve_n);
    const bool more = tile + WAVES < te;

    f32x4_t s[4][NQ];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int q = 0; q < NQ; ++q) s[t][q] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int f = 0; f < HF; ++f) {
        const vec8 a0 = widen<E>(kr[t][f].x, kr[t][f].y), a1 = widen<E>(kr[t][f].z, kr[t][f].w);
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          s[t][q] = E::mfma16(a0, qf[q][2 * f], s[t][q]);
          s[t][q] = E::mfma16(a1, qf[q][2 * f + 1], s[t][q]);
        }
      }

    if (more) fetch_k(tile + WAVES);

    // Keys that a row does not see: key jv + e for e below a and from b on.  Codes behind the last key are whatever the
    // page held: zero times them has to be zero.  So has zero times a NaN that the row does not see; the products run
    // without NaN, and the outputs that one does reach become NaN behind the loop.
    bool all_seen = here;
#pragma unroll
    for (int q = 0; q < NQ; ++q) all_seen = all_seen & (lo[q] <= jv) & (jv + 16 <= hi[q]);
    if (!__all(all_seen)) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int a = here ? lo[q] - jv : 16, b = here ? hi[q] - jv : 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = s[e >> 2][q][e & 3];
          s[e >> 2][q][e & 3] = ((e >= a) & (e < b)) ? x : -INFINITY;
        }
      }
      const uint4 keep = kept(jv, here);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        uint4& w = vr[dt];
        w = make_uint4(w.x & keep.x, w.y & keep.y, w.z & keep.z, w.w & keep.w);
        poison |= nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w);
        w = make_uint4(finite_bytes(w.x), finite_bytes(w.y), finite_bytes(w.z), finite_bytes(w.w));
      }
    }
    const float sc = p.scale * exp2_int(ke), inv = exp2_int(-ve);
    f16x8_t pf[2][NQ];
    float mx[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) mx[q] = lane_max<NQ>(s, q, sc, (float)ve);
    raise_max<DT, NQ>(mx, m_run, l_run, o);
#pragma unroll
    for (int q = 0; q < NQ; ++q) weights<NQ>(s, q, sc, (float)ve, inv, m_run[q], l_run[q], pf[0][q], pf[1][q]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const f16x8_t a0 = widen_f16(vr[dt].x, vr[dt].y), a1 = widen_f16(vr[dt].z, vr[dt].w);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        o[dt][q] = F16::mfma16(a0, pf[0][q], o[dt][q]);
        o[dt][q] = F16::mfma16(a1, pf[1][q], o[dt][q]);
      }
    }
    if (more) {
      fetch_v(tile + WAVES);
      if (tile + 2 * WAVES < te) look_up(tile + 2 * WAVES);
    }
  }

  // NaN among the values of tiles that not every row sees whole: 1 at each times 1 at each key that a row sees is above 0
  // where it reaches the row.
  if (__any(poison != 0u)) {
    for (int tile = tb + wave; tile < te; tile += WAVES) {
      look_up(tile);
      fetch_v(tile);
      const int jv = tile * 64 + 16 * g;
      const uint4 keep = kept(jv, here_n);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        f16x8_t seen[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) seen[e >> 3][e & 7] = (_Float16)(here_n && jv + e >= lo[q] && jv + e < hi[q] ? 1.f : 0.f);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint4& w = vr[dt];  // e4m3's 1.0 in the place of each NaN
          const uint32_t ind[4] = {(nan_bytes(w.x & keep.x) >> 7) * 0x38u, (nan_bytes(w.y & keep.y) >> 7) * 0x38u,
                                   (nan_bytes(w.z & keep.z) >> 7) * 0x38u, (nan_bytes(w.w & keep.w) >> 7) * 0x38u};
          f32x4_t hit = F16::mfma16(widen_f16(ind[0], ind[1]), seen[0], (f32x4_t){0.f, 0.f, 0.f, 0.f});
          hit = F16::mfma16(widen_f16(ind[2], ind[3]), seen[1], hit);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[dt][q][i] = hit[i] > 0.f ? __uint_as_float(0x7fc00000u) : o[dt][q][i];
        }
      }
    }
  }

  // Join the waves.
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const float l = quad16_sum(l_run[q]);
    if (g == 0) {
      sm[wave][16 * q + m] = m_run[q];
      sl[wave][16 * q + m] = l;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(&so[wave][16 * q + m][16 * dt + 4 * g]) = o[dt][q];
  }
  __syncthreads();
  for (int e = tid; e < TILE * DIM / 4; e += 64 * WAVES) {
    const int i = e / (DIM / 4), d = (e % (DIM / 4)) * 4;
    const int row = row0 + i;
    if (row >= rows) break;
    const int64_t tok = tok0 + row / p.group;
    const int head = hk * p.group + row % p.group;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sm[w][i]);
    float l = 0.f;
    f32x4_t acc = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int w = 0; w < WAVES; ++w) {
      const float f = sm[w][i] == -INFINITY ? 0.f : fast_exp2(sm[w][i] - top);
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(&so[w][i][d]);
      l += f * sl[w][i];
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += f * x[k];
    }
    if (p.splits == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      store4(p, tok, head, d, acc, inv);
      if (d == 0 && p.lse) p.lse[tok * p.q_heads + head] = row_lse(top, l);
    } else {
      const int64_t at = (int64_t)z * p.tokens * p.q_heads + tok * p.q_heads + head;
      *reinterpret_cast<f32x4_t*>(p.part_o + at * DIM + d) = acc;
      if (d == 0) {
        p.part_ml[2 * at] = top;
        p.part_ml[2 * at + 1] = l;
      }
    }
  }
}

// ---- many rows --------------------------------------------------------------------
// A workgroup has 128 rows of one key head, or 256 where there are as many and the head dim is 128, 32 a wave, and walks
// the keys in tiles of 64.  A tile's codes come from memory once for the workgroup: each thread widens 16-byte pieces and
// writes them to LDS as the operands that the waves' MFMAs read (1 KB pieces, lane after lane: no bank conflicts either
// way).  Widening once for 256 rows costs a thread 32 conversions a tile; widening behind the LDS read would cost 256.
// Bound by the SIMDs' issue: an MFMA of 16 cycles has 32 rows x 64 keys x 32 channels / 4, and between two of them go the
// scale, exponential, sum, maximum and rounding of two scores (about 11 cycles at head dim 128, twice that at 64) and the
// LDS reads.  3,600 tokens x 75,600 keys of 40 heads of 128 channels: 14.3 ms with 16-row tiles, 9.65 with 128 rows, 6.2
// with 256 (half the LDS reads and widening a row) and the scores a tile ahead, 5.2 with K three tiles deep: 1.08 PFLOP/s,
// where the chip's matrix products reach 1.37.  12 requests of 1,500 tokens on 6,000 keys, 32 heads of 64 channels: 1.13 ms,
// 0.78 PFLOP/s.
template <int DIM, int WAVES>
struct KvTile {
  static constexpr int ROWS = 32 * WAVES;
  static constexpr int KS = DIM / 32, DT = DIM / 16, HF = DIM / 64;
  static constexpr int NP = 4 * HF / WAVES;  // 1 KB pieces of K, and of V, that a wave brings of a tile
  static constexpr int KBYTES = 64 * DIM * 2, VBYTES = KBYTES;
  static_assert(NP >= 1, "every wave brings a piece");
  // With one piece a wave there are registers to fetch a tile two steps before it is widened, and LDS to hold K three
  // tiles deep, so that a step's first operands are read before the barrier that opens it; else one and two.
  static constexpr int SETS = NP == 1 ? 2 : 1, KBUFS = NP == 1 ? 3 : 2;
};

constexpr int kAhead = 4;  // LDS reads in flight

// Workgroup barrier behind this wave's LDS writes, with its last N LDS reads still in flight (LDS answers in order; N
// reads have to be there, behind the last write).
template <int N>
__device__ __forceinline__ void barrier_lds() {
  __builtin_amdgcn_s_waitcnt(0xC07F | (N << 8));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// UNI: pages of 64 tokens and more, so that a tile has one page and its number stays in scalar registers.
template <typename E, int DIM, int WAVES, bool UNI>
__global__ __launch_bounds__(64 * WAVES, 2) void kv_attn_tiles(KvAttnParams p, int tiles, int items, int per_xcd) {
  using C = KvTile<DIM, WAVES>;
  constexpr int KS = C::KS, DT = C::DT, NP = C::NP;
  constexpr int SETS = C::SETS, KBUFS = C::KBUFS;
  using vec8 = typename E::vec8;
  __shared__ __attribute__((aligned(1024))) unsigned char Ks[KBUFS][C::KBYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char Vs[2][C::VBYTES];
  __shared__ int nan_tile;  // the last tile, of those seen in part, that held a NaN among its values
  // Workgroup n runs on XCD n % 8, which takes a contiguous run of (head, part of the keys, tile): the tiles of a
  // head sweep the same keys at the same time and find them in the XCD's L2.
  const int slot = blockIdx.x >> 3, item = (blockIdx.x & 7) * per_xcd + slot;
  if (item >= items) return;
  const int hz = item / tiles, hk = hz / p.splits, z = hz - hk * p.splits;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  const KvCache& c = p.c;
  const int page = 1 << c.page_log2;

  const int id = tiles - 1 - (item - hz * tiles);  // with a causal mask the last have most to do
  const TileOf tile_of = find_tile<C::ROWS>(p, id);
  if (id == 0 && tile_of.front > 0) zero_rows<DIM>(p, hk, z, 0, 0, tile_of.front * p.group);
  const int r = tile_of.r, tok0 = tile_of.tok0, rows = tile_of.rows, row0 = tile_of.row0, raw_len = tile_of.raw_len;
  if (row0 < 0 || row0 >= rows) return;
  if (r == p.requests) {
    zero_rows<DIM>(p, hk, z, tok0, row0, min(C::ROWS, rows - row0));
    return;
  }
  const int len = (int)min(min((int64_t)raw_len, p.max_kv), p.width << c.page_log2);
  const int64_t pos_base = (int64_t)raw_len - rows / p.group;
  const int32_t* table = p.tables + r * p.table_stride;

  // This lane's row of row tile q: its token within the request, and its head.
  const int wrow = row0 + 32 * wave;
  auto row_of = [&](int q, int& tok, int& head) {
    const int i = min(wrow + 16 * q + m, rows - 1);
    tok = i / p.group;
    head = hk * p.group + (i - tok * p.group);
  };
  const int last = min(row0 + C::ROWS, rows) - 1;
  const int klo = sees_lo(p, pos_base + row0 / p.group, len), khi = sees_hi(p, pos_base + last / p.group, len);
  const int tile_lo = klo >> 6, tile_hi = max(tile_lo, (khi + 63) >> 6);
  const int per = (tile_hi - tile_lo + p.splits - 1) / p.splits;
  const int tb = min(tile_lo + z * per, tile_hi), te = min(tb + per, tile_hi);

  vec8 qf[2][KS];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    int tok, head;
    row_of(q, tok, head);
    load_q<E, KS>(p, tok0 + tok, head, g, qf[q]);
  }

  f32x4_t o[DT][2];
  float l_run[2] = {0.f, 0.f}, m_run[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt][q] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

  // Tiles [wb, we) are seen whole by every row, and all of their pages are there.
  int wb = max(tb, (sees_lo(p, pos_base + last / p.group, len) + 63) >> 6);
  int we = min(te, sees_hi(p, pos_base + row0 / p.group, len) >> 6);
  if (wb < we) {
    const int end = (we * 64 - 1) >> c.page_log2;
    int gone = 0;
    for (int e = ((wb * 64) >> c.page_log2) + tid; e <= end; e += 64 * WAVES) gone |= (unsigned)table[e] >= (unsigned)c.num_pages;
    if (__syncthreads_or(gone)) wb = we = te;
  } else {
    wb = we = te;
  }

  // Pieces of a tile that this thread brings: of 16-key tile kt of K row m's 16 channels 64 f + 16 g .. of NP halves f
  // from kf on; of V channels 16 (NP wave + n) + m, keys 16 g .. + 15.  Their pages are looked up a step ahead.
  const int kt = wave & 3, kf = WAVES == 8 ? wave >> 2 : 0;
  const uint32_t k_lane = ((UNI ? 16 * (m >> 2) : 0) + 4 * kt + (m & 3)) * DIM + 64 * kf + 16 * g;
  const uint32_t v_lane = ((16 * NP * wave + m) << c.page_log2) + (UNI ? 16 * g : 0);
  auto k_key = [&](int tile) { return UNI ? tile * 64 : tile * 64 + 16 * (m >> 2); };
  auto v_key = [&](int tile) { return UNI ? tile * 64 : tile * 64 + 16 * g; };
  uint4 kr[SETS][NP], vr[SETS][NP];
  int ke_n[SETS], ve_n[SETS];  // exponents of the lane's keys 16 g .. + 15
  auto load_k = [&](uint4 (&to)[NP], int tile, int id) {
    const uint8_t* at = c.k + ((((int64_t)id * c.heads + hk) << c.page_log2) + (k_key(tile) & (page - 1))) * DIM + k_lane;
#pragma unroll
    for (int n = 0; n < NP; ++n) to[n] = *reinterpret_cast<const uint4*>(at + 64 * n);
  };
  auto fetch_k = [&](int set, int tile, int id) { load_k(kr[set], tile, id); };
  auto fetch_v = [&](int set, int tile, int id) {
    const int64_t row = (int64_t)id * c.heads + hk;
    const uint8_t* at = c.v + ((row * DIM) << c.page_log2) + (v_key(tile) & (page - 1)) + v_lane;
#pragma unroll
    for (int n = 0; n < NP; ++n) vr[set][n] = *reinterpret_cast<const uint4*>(at + ((16 * n) << c.page_log2));
    ke_n[set] = c.k_exp[row];
    ve_n[set] = c.v_exp[row];
  };
  // Half u of piece n, widened, into buffer b.
  auto stage_k = [&](int b, int n, int u, const uint4& x) {
    vec8* d = reinterpret_cast<vec8*>(Ks[0] + b * C::KBYTES + (kt * KS + 2 * (kf + n) + u) * 1024) + lane;
    d[0] = u ? widen<E>(x.z, x.w) : widen<E>(x.x, x.y);
  };
  auto stage_v = [&](int b, int n, int u, const uint4& x) {
    f16x8_t* d = reinterpret_cast<f16x8_t*>(Vs[b] + (NP * wave + n) * 2048 + u * 1024) + lane;
    d[0] = u ? widen_f16(x.z, x.w) : widen_f16(x.x, x.y);
  };
  auto stage_all = [&](int b, const uint4 (&x)[NP], auto stage) {
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) stage(b, n, u, x[n]);
  };
  auto scores = [&](int b, f32x4_t (&s)[4][2]) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int q = 0; q < 2; ++q) s[t][q] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const vec8 a = *(reinterpret_cast<const vec8*>(Ks[b] + (t * KS + k) * 1024) + lane);
#pragma unroll
        for (int q = 0; q < 2; ++q) s[t][q] = E::mfma16(a, qf[q][k], s[t][q]);
      }
  };
  auto pv = [&](int b, const f16x8_t (&pf)[2][2], auto fix) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const f16x8_t a = as_vec8<F16>(fix(*(reinterpret_cast<const uint4*>(Vs[b] + (2 * dt + u) * 1024) + lane)));
#pragma unroll
        for (int q = 0; q < 2; ++q) o[dt][q] = F16::mfma16(a, pf[u][q], o[dt][q]);
      }
  };

  auto as_is = [](const uint4& w) { return w; };

  // Tiles that some row sees in part, or whose pages are not all there: one at a time.
  auto part_tiles = [&](int t0, int t1) {
    if (t0 >= t1) return;
    int lo[2], hi[2];  // what the lane's rows see
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int tok, head;
      row_of(q, tok, head);
      lo[q] = sees_lo(p, pos_base + tok, len);
      hi[q] = sees_hi(p, pos_base + tok, len);
    }
    auto page_of = [&](int j) -> int {
      const int id = j < len ? table[j >> c.page_log2] : -1;
      return (unsigned)id < (unsigned)c.num_pages ? id : -1;
    };
    // A tile is fetched while the one before is computed, its page numbers a tile before that.
    int kid = page_of(k_key(t0)), vid = page_of(v_key(t0));
    bool here_n = false;
    auto fetch = [&](int tile) {
      here_n = vid >= 0;
      fetch_k(0, tile, max(kid, 0));
      fetch_v(0, tile, max(vid, 0));
      if (tile + 1 < t1) {
        kid = page_of(k_key(tile + 1));
        vid = page_of(v_key(tile + 1));
      }
    };
    fetch(t0);
    if (tid == 0) nan_tile = -1;
    for (int tile = t0; tile < t1; ++tile) {
      const bool here = here_n;
      const int jv = tile * 64 + 16 * g;
      const int nb = here ? min(max(len - jv, 0), 16) : 0;  // codes behind the last key are whatever the page held
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        uint4& x = vr[0][n];
        x = make_uint4(x.x & first_bytes(nb), x.y & first_bytes(nb - 4), x.z & first_bytes(nb - 8), x.w & first_bytes(nb - 12));
      }
      const int ke = page_exp(ke_n[0]), ve = page_exp(ve_n[0]);
      uint32_t nan = 0u;
#pragma unroll
      for (int n = 0; n < NP; ++n) nan |= nan_bytes(vr[0][n].x) | nan_bytes(vr[0][n].y) | nan_bytes(vr[0][n].z) | nan_bytes(vr[0][n].w);
      barrier_lds_reads_done();
      stage_all(0, kr[0], stage_k);
      stage_all(0, vr[0], stage_v);
      if (nan) nan_tile = tile;
      if (tile + 1 < t1) fetch(tile + 1);
      barrier_lds_reads_done();
      // Key jv + e is hidden from row tile q for e below a[q] and from b[q] on.
      int a[2], b[2];
      bool some = false, whole = true;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        a[q] = here ? lo[q] - jv : 16;
        b[q] = here ? hi[q] - jv : 0;
        some = some | (max(a[q], 0) < min(b[q], 16));
        whole = whole & (a[q] <= 0) & (b[q] >= 16);
      }
      if (wrow >= rows || !__any(some)) continue;  // the wave has no row here, but the other waves' tiles to bring
      f32x4_t s[4][2];
      scores(0, s);
      if (!__all(whole)) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x = s[e >> 2][q][e & 3];
            s[e >> 2][q][e & 3] = ((e >= a[q]) & (e < b[q])) ? x : -INFINITY;
          }
      }
      const float sc = p.scale * exp2_int(ke), vf = (float)ve, inv = exp2_int(-ve);
      f16x8_t pf[2][2];
      float mx[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) mx[q] = lane_max<2>(s, q, sc, vf);
      raise_max<DT, 2>(mx, m_run, l_run, o);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        weights<2>(s, q, sc, vf, inv, m_run[q], l_run[q], pf[0][q], pf[1][q]);
      }
      if (__builtin_amdgcn_readfirstlane(nan_tile) != tile) {
        pv(0, pf, as_is);
      } else {
        poison_step<DT>(Vs[0], lane, here, jv, lo, hi, o);
        pv(0, pf, [](const uint4& w) { return make_uint4(finite_halves(w.x), finite_halves(w.y), finite_halves(w.z), finite_halves(w.w)); });
      }
    }
  };

  part_tiles(tb, wb);
  if (wb < we) {
    // Scores run a tile ahead of the weights and sums: in step `tile` s holds the tile's scores, V of the tile and K of the
    // next KBUFS - 1 are in LDS.  The scores of the next tile and the weights of this one need nothing of each other, nor
    // do the sums and the widening of what comes next: matrix and vector instructions run in each other's time.
    // The step widens K of tile + KBUFS and V of tile + 1 from one register set, and fetches the same SETS - 1 tiles on.
    constexpr int KN = KBUFS + SETS - 1, VN = SETS;
    auto clip = [&](int tile) { return min(tile, we - 1); };
    // Page of the lane's key j.  With UNI it is the tile's: the number comes through a vector load all the same (a
    // scalar one would make every wait for an LDS read a wait for it), is read from one lane a step later, and K's
    // serves V KN - VN steps after.
    auto look = [&](int j) { return table[j >> c.page_log2]; };
    auto uni = [](int id) { return UNI ? __builtin_amdgcn_readfirstlane(id) : id; };
    f32x4_t sa[4][2], sb[4][2];
    float sc, vf, inv, mx[2];
    auto scales = [&](int set) {
      const int ke = page_exp(uni(ke_n[set])), ve = page_exp(uni(ve_n[set]));
      sc = p.scale * exp2_int(ke);
      vf = (float)ve;
      inv = exp2_int(-ve);
    };
    // All that step wb finds in LDS and in its registers is asked for at once, the page numbers first.
    int ks[KN + 1], vs[VN + 1];
#pragma unroll
    for (int n = 0; n <= KN; ++n) ks[n] = look(k_key(clip(wb + n)));
#pragma unroll
    for (int n = 0; n <= VN; ++n) vs[n] = UNI ? ks[n] : look(v_key(clip(wb + n)));
    uint4 k0[KBUFS][NP];
#pragma unroll
    for (int n = 0; n < KBUFS; ++n) load_k(k0[n], clip(wb + n), uni(ks[n]));
    fetch_v(0, wb, uni(vs[0]));
    if constexpr (SETS == 2) {
      fetch_v(1, clip(wb + 1), uni(vs[1]));
      fetch_k(1, clip(wb + KBUFS), uni(ks[KBUFS]));
    }
    // What step wb fetches: K of wb + KN (and, with UNI, the pages of the tiles between that and V's), V of wb + VN.
    int kid = ks[KN], vid = vs[VN];
    int mid[KN - VN];
#pragma unroll
    for (int n = 0; n < KN - VN; ++n) mid[n] = UNI ? uni(ks[VN + n]) : 0;
    barrier_lds_reads_done();
#pragma unroll
    for (int n = 0; n < KBUFS; ++n) stage_all(n, k0[n], stage_k);
    stage_all(0, vr[0], stage_v);
    scales(0);
    barrier_lds_reads_done();
    scores(0, sa);
#pragma unroll
    for (int q = 0; q < 2; ++q) mx[q] = lane_max<2>(sa, q, sc, vf);
    // (KBUFS == 2: K of the tile after next goes where the scores were just read.)
    uint4 first[kAhead];
    int kb = 0;  // (tile - wb) % KBUFS
    auto k_at = [&](int b) { return Ks[0] + b * C::KBYTES; };
    auto k_read = [&](const unsigned char* at, int f) { return *(reinterpret_cast<const uint4*>(at + ((f % 4) * KS + f / 4) * 1024) + lane); };
    if constexpr (KBUFS == 3) {
#pragma unroll
      for (int f = 0; f < kAhead; ++f) first[f] = k_read(k_at(1), f);
    }
    barrier_lds_reads_done();
    // last: no step follows, so that nothing but LDS writes is in flight at the barrier, which waits for them.
    auto step = [&](int tile, int b, f32x4_t (&s)[4][2], f32x4_t (&sn)[4][2], auto last) {
      constexpr bool FIRST = KBUFS == 3 && !decltype(last)::value;
      const int fs = SETS == 2 ? b : 0, ss = SETS == 2 ? b ^ 1 : 0;  // sets to fetch into, to widen from
      const int kb1 = kb + 1 == KBUFS ? 0 : kb + 1, kb2 = kb1 + 1 == KBUFS ? 0 : kb1 + 1;
      const unsigned char* k_src = k_at(kb1);
      int kid1 = 0, vid1 = 0;
      // The next step's page numbers are asked for before the tiles, whose loads then need not be waited for with them.
      auto look_next = [&] {
        kid1 = look(k_key(clip(tile + 1 + KN)));
        if (!UNI) vid1 = look(v_key(clip(tile + 1 + VN)));
      };
      int last_id = 0;
      auto fetch_next_k = [&] {
        last_id = uni(kid);
        fetch_k(fs, clip(tile + KN), last_id);
      };
      auto fetch_next_v = [&] { fetch_v(fs, clip(tile + VN), UNI ? mid[0] : vid); };
      if constexpr (SETS == 1) {
        fetch_next_k();
        fetch_next_v();
        look_next();
      }
      raise_max<DT, 2>(mx, m_run, l_run, o);
      // One operand at a time, read kAhead operands before, and its two MFMAs; between them, first the weights of 32 / NF
      // scores, then a piece of the next tiles' codes widened and a share of the maxima.  The order is fixed
      // (sched_barrier): left alone, the compiler reads each operand where it is used and runs the two kinds apart.
      constexpr int NF = KS * 4, PAIRS = 16 / NF;  // operands of K, and of V
      static_assert(NF == 2 * DT && NF % (4 * NP) == 0, "two operands for each channel tile of V and each piece to widen");
      uint4 fr[2 * NF];
      auto read = [&](int f) {
        if (f >= 2 * NF) return;
        const int v = f - NF;
        fr[f] = f < NF ? k_read(k_src, f) : *(reinterpret_cast<const uint4*>(Vs[b] + (2 * (v % DT) + v / DT) * 1024) + lane);
      };
#pragma unroll
      for (int f = 0; f < kAhead; ++f) {
        if constexpr (KBUFS == 3) fr[f] = first[f];
        else read(f);
      }
      float off[2], sum[2] = {0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 2; ++q) off[q] = vf - m_run[q] + kShift;
      uint32_t w[2][8];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        read(f + kAhead);
#pragma unroll
        for (int q = 0; q < 2; ++q)
          sn[f % 4][q] = E::mfma16(as_vec8<E>(fr[f]), qf[q][f / 4], f < 4 ? (f32x4_t){0.f, 0.f, 0.f, 0.f} : sn[f % 4][q]);
#pragma unroll
        for (int n = f * PAIRS; n < (f + 1) * PAIRS; ++n) {
          const int q = n & 1, e = n >> 1;
          const f32x4_t& x = s[e >> 1][q];
          const float p0 = fast_exp2(fmaf(x[2 * (e & 1)], sc, off[q]));
          const float p1 = fast_exp2(fmaf(x[2 * (e & 1) + 1], sc, off[q]));
          w[q][e] = F16::pack2(p0, p1);
          sum[q] += p0 + p1;
          asm volatile("" : "+v"(sum[q]));  // added here: sunk behind the loop, the sums would keep 32 weights in registers
        }
        if constexpr (SETS == 2) {
          if (f == 0) look_next();
          if (f == NF / 4) fetch_next_k();
          if (f == NF / 2) fetch_next_v();
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      f16x8_t pf[2][2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        l_run[q] = fmaf(sum[q], inv, l_run[q]);
        pf[0][q] = as_vec8<F16>((u32x4_t){w[q][0], w[q][1], w[q][2], w[q][3]});
        pf[1][q] = as_vec8<F16>((u32x4_t){w[q][4], w[q][5], w[q][6], w[q][7]});
        mx[q] = -INFINITY;
      }
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        read(NF + f + kAhead);
#pragma unroll
        for (int q = 0; q < 2; ++q) o[f % DT][q] = F16::mfma16(as_vec8<F16>(fr[NF + f]), pf[f / DT][q], o[f % DT][q]);
        constexpr int EVERY = NF / (4 * NP);  // one half of a piece of K, then of V, every so many operands
        if (f % EVERY == EVERY - 1) {
          const int i = f / EVERY;
          if (i < 2 * NP) stage_k(kb, i / 2, i % 2, kr[ss][i / 2]);
          else stage_v(b ^ 1, i / 2 - NP, i % 2, vr[ss][i / 2 - NP]);
        }
#pragma unroll
        for (int n = f * PAIRS; n < (f + 1) * PAIRS; ++n) {
          const int q = n & 1, e = n >> 1;
          const f32x4_t& x = sn[e >> 1][q];
          mx[q] = fmaxf(fmaxf(x[2 * (e & 1)], x[2 * (e & 1) + 1]), mx[q]);
          asm volatile("" : "+v"(mx[q]));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (FIRST) {
#pragma unroll
        for (int f = 0; f < kAhead; ++f) first[f] = k_read(k_at(kb2), f);
      }
      scales(ss);
#pragma unroll
      for (int q = 0; q < 2; ++q) mx[q] = fmaf(mx[q], sc, vf);
      kid = kid1;
      if (UNI) {
#pragma unroll
        for (int n = 0; n < KN - VN - 1; ++n) mid[n] = mid[n + 1];
        mid[KN - VN - 1] = last_id;
      } else {
        vid = vid1;
      }
      kb = kb1;
      barrier_lds<FIRST ? kAhead : 0>();
    };
    auto finish = [&](int b, const f32x4_t (&s)[4][2]) {
      f16x8_t pf[2][2];
      raise_max<DT, 2>(mx, m_run, l_run, o);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        weights<2>(s, q, sc, vf, inv, m_run[q], l_run[q], pf[0][q], pf[1][q]);
      }
      pv(b, pf, as_is);
    };
    int tile = wb;
    for (; tile + 2 < we; tile += 2) {
      step(tile, 0, sa, sb, std::false_type{});
      step(tile + 1, 1, sb, sa, std::false_type{});
    }
    if (tile + 1 < we) {
      step(tile, 0, sa, sb, std::true_type{});
      finish(1, sb);
    } else {
      finish(0, sa);
    }
  }
  part_tiles(we, te);

#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const float l = quad16_sum(l_run[q]);
    if (wrow + 16 * q + m >= rows) continue;
    int tok, head;
    row_of(q, tok, head);
    const int64_t at_tok = tok0 + tok;
    if (p.splits == 1) {
      const float w = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) store4(p, at_tok, head, 16 * dt + 4 * g, o[dt][q], w);
      if (g == 0 && p.lse) p.lse[at_tok * p.q_heads + head] = row_lse(m_run[q], l);
    } else {
      const int64_t at = ((int64_t)z * p.tokens + at_tok) * p.q_heads + head;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(p.part_o + at * DIM + 16 * dt + 4 * g) = o[dt][q];
      if (g == 0) {
        p.part_ml[2 * at] = m_run[q];
        p.part_ml[2 * at + 1] = l;
      }
    }
  }
}

// Join the parts of the keys: one wave a row.  Lane z has part z's maximum and sum (there are at most 64).
template <int DIM>
__global__ __launch_bounds__(256) void kv_attn_join(KvAttnParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t all = p.tokens * p.q_heads;
  if (row >= all) return;
  const int64_t tok = row / p.q_heads;
  const int head = (int)(row - tok * p.q_heads);
  const bool none = p.cu_q != nullptr && (tok >= first_token(p, p.requests) || tok < first_token(p, 0));  // of no request
  if (none && !p.zero_tail) return;
  constexpr int N = DIM / 64;
  float top = -INFINITY, l = 0.f, f = 0.f, acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  if (!none) {
    if (lane < p.splits) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * (lane * all + row));
      top = ml.x;
      l = ml.y;
    }
    float most = top;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
    // A part without keys has l = 0; its maximum is -inf, as beside a NaN l where NaN is all that a row sees.
    f = top == -INFINITY ? 0.f : fast_exp2(top - most);
    l = wave_sum(l == 0.f ? 0.f : f * l);
    top = most;
    const float* part = p.part_o + row * DIM + N * lane;
    for (int z = 0; z < p.splits; z += 8) {
      float x[8][N];
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int k = 0; k < N; ++k) x[n][k] = part[min(z + n, p.splits - 1) * all * DIM + k];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float fz = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), min(z + n, 63)));
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += z + n < p.splits ? fz * x[n][k] : 0.f;
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int k = 0; k < N; ++k) store_rowpart(p, tok, head, N * lane + k, acc[k] * inv);
  if (lane == 0 && p.lse) p.lse[row] = row_lse(top, l);
}

// Tile numbers that a head of the launch has.  With row starts some have no rows, often every second one (a request of less than a tile):
// their number is odd, so that those that have some fall to all XCDs and compute units, which take workgroups in turn
// (1 request, 96 rows a head, 32,768 keys of 40 heads: 206 us at 2 numbers a head, 129 at 3).
int64_t tile_numbers(const KvAttnParams& p, int rows) {
  if (p.cu_q == nullptr) return (int64_t)p.requests * (((int64_t)p.per_request * p.group + rows - 1) / rows);
  return (p.tokens * p.group / rows + p.requests + 1) | 1;
}

template <typename E, int DIM, int NQ>
hipError_t launch_rows(const KvAttnParams& p, hipStream_t stream) {
  const int64_t tiles = tile_numbers(p, 16 * NQ);
  if (tiles > 0x7fffffff || p.c.heads > 65535 || p.splits > 64) return hipErrorInvalidValue;
  const dim3 grid((unsigned)tiles, (unsigned)p.c.heads, (unsigned)p.splits);
  hipLaunchKernelGGL((kv_attn_rows<E, DIM, NQ>), grid, dim3(512), 0, stream, p);
  return hipGetLastError();
}

template <typename E, int DIM, int WAVES>
hipError_t launch_tiles(const KvAttnParams& p, hipStream_t stream) {
  const int64_t tiles = tile_numbers(p, KvTile<DIM, WAVES>::ROWS);
  const int64_t items = tiles * p.c.heads * p.splits;
  const int64_t per_xcd = (items + 7) / 8;
  if (per_xcd * 8 > 0x7fffffff) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(per_xcd * 8)), block(64 * WAVES);
  if (p.c.page_log2 >= 6)
    hipLaunchKernelGGL((kv_attn_tiles<E, DIM, WAVES, true>), grid, block, 0, stream, p, (int)tiles, (int)items, (int)per_xcd);
  else
    hipLaunchKernelGGL((kv_attn_tiles<E, DIM, WAVES, false>), grid, block, 0, stream, p, (int)tiles, (int)items, (int)per_xcd);
  return hipGetLastError();
}

template <typename E, int DIM>
hipError_t launch_any(const KvAttnParams& p, int rows, hipStream_t stream) {
  hipError_t e = hipErrorInvalidValue;
  if (rows == 16) e = launch_rows<E, DIM, 1>(p, stream);
  else if (rows == 32) e = launch_rows<E, DIM, 2>(p, stream);
  else if (rows == 128) e = launch_tiles<E, DIM, 4>(p, stream);
  else if constexpr (DIM == 128) e = launch_tiles<E, DIM, 8>(p, stream);
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t wgs = (p.tokens * p.q_heads + 3) / 4;
  if (wgs > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kv_attn_join<DIM>, dim3((unsigned)wgs), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

// Tile and parts of the keys, from the sizes that the host knows.  Tiles of 16 rows are bound by the bytes of the keys, of
// 32 by those and the widening, of 128 and 256 by the matrix units (rates of long runs, in us).  The tile is the one that
// holds a request's rows, with the best parts of each measured: 16 requests, 4,096 keys of 8 heads of 128 channels, 12 rows
// a request and key head: 30 us with 16, 33 with 32 rows; 24: 45, 34; 48: 32 rows 48, 128 rows 54; 96: 80, 59; 128: 128
// rows 62, 256 rows 81; 160: 95, 84; 512: 148, 130 us.  The workgroups run in rounds of as many as the
// chip holds at once; more parts of the keys make the last round shorter, but a workgroup begins and ends for some us and
// its sums pass through memory and a second launch.  Parts are added while that gains 3%: workgroups that sweep the same
// keys at the same time share them in L2, and the more rounds there are the further they drift apart (3,600 tokens x
// 75,600 of 40 heads: 6.08 ms whole, 5.00 in 2 parts, 5.07 in 4, 5.36 in 5).
KvAttnPlan kv_attn_plan(int64_t tokens, int requests, int q_heads, int kv_heads, int dim, int64_t max_kv) {
  const int group = q_heads / kv_heads;
  const int64_t mean = (tokens * group + requests - 1) / requests;
  KvAttnPlan plan;
  plan.rows = mean <= 16 ? 16 : mean <= 64 ? 32 : mean <= 128 || dim != 128 ? 128 : 256;
  plan.splits = 1;
  const bool few = plan.rows <= 32;
  // Four tiles a wave at most: one launch (1 token to 1,560 of 12 heads: 14.0 us on the GPU, 10.5 in four parts with their
  // join, but a second launch costs the host about 4 us of a call that takes it 13).
  if (few && max_kv <= 2048) return plan;
  const double tiles = (double)((mean + plan.rows - 1) / plan.rows), wgs = tiles * requests * kv_heads;
  const double slots = plan.rows == 128 ? 512 : 256;
  const double work_us = few ? 2.0 * tiles * requests * max_kv * kv_heads * dim / (plan.rows == 16 ? 5.5e6 : 3.6e6) : 4.0 * tokens * max_kv * q_heads * dim / 1.1e9;
  const double part_us = 2.0 * tokens * q_heads * (dim + 2) * sizeof(float) / 4.5e6;  // written and read
  const int64_t most = (max_kv + 511) / 512 < 64 ? (max_kv + 511) / 512 : 64;        // eight tiles a part at least
  double best = 0.0;
  for (int n = 1; n <= most; ++n) {
    const double used = wgs * n, rounds = ceil(used / slots);
    const double t = work_us * rounds * slots / used + (few ? 3.0 : 10.0) * rounds + (n > 1 ? 4.0 + n * part_us : 0.0);
    if (n == 1 || t < 0.97 * best) {
      best = t;
      plan.splits = n;
    }
  }
  return plan;
}

hipError_t launch_kv_attn(const KvAttnParams& p, hipStream_t stream) {
  const KvAttnPlan plan = kv_attn_plan(p.tokens, p.requests, p.q_heads, p.c.heads, p.c.dim, p.max_kv);
  if (plan.splits != p.splits) return hipErrorInvalidValue;
  if (p.c.dim == 128) return p.f16 ? launch_any<F16, 128>(p, plan.rows, stream) : launch_any<Bf16, 128>(p, plan.rows, stream);
  if (p.c.dim == 64) return p.f16 ? launch_any<F16, 64>(p, plan.rows, stream) : launch_any<Bf16, 64>(p, plan.rows, stream);
  return hipErrorInvalidValue;
}

}  // namespace pasa
