// The key/value cache in 8 bits: its layout, and the launchers of the kernels on it (kv_tables.hip,
// kv_append.hip, kv_attn.hip) and of the rotary embedding from positions (rope_axes.hip).
//
// A cache holds num_pages pages of page_size tokens (a power of two, 16 .. 128) for each of kv_heads heads:
//   k      [page][head][token][dim]   e4m3 codes, a token's channels together
//   v      [page][head][dim][token]   e4m3 codes, a channel's tokens together
//   k_exp, v_exp [page][head]         int8: a value is its code times 2 ** exponent
// dim is 64 or 128; channels from head_dim on hold zeros.  V lies the other way round because both products of the
// attention contract over what is contiguous here (channels for q.k, tokens for p.v): a lane's MFMA operand is
// 16 consecutive bytes of either, so a tile goes from memory into the matrix unit without a transposition.
// The scale is a power of two, so that a page whose largest value grows is rescaled without a second rounding
// (but of what falls into e4m3's subnormals), and applying it is exact.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace pasa {

constexpr int kKvExpMin = -50;  // exponents of a page; the attention folds them into the softmax's exponent,
constexpr int kKvExpMax = 50;   // whose fp32 range (2 ** +-126) they leave room in

struct KvCache {
  uint8_t* k;
  uint8_t* v;
  int8_t* k_exp;
  int8_t* v_exp;
  int num_pages;
  int heads;
  int page_log2;
  int dim;       // 64 or 128
  int head_dim;  // <= dim
};

// ---- rotary embedding (rope_axes.hip) --------------------------------------------
struct RopeAxesTensor {
  const void* in;  // nullptr: skipped
  void* out;
  int64_t in_b, in_s, in_h;  // strides in elements; the channels are contiguous
  int64_t out_b, out_s, out_h;
  int heads;
};
constexpr int kPosI32 = 0, kPosI64 = 1, kPosF32 = 2;
struct RopeAxesParams {
  RopeAxesTensor t[2];
  const void* pos;
  int pos_type;
  int64_t pos_axis, pos_b, pos_s;  // strides of positions in elements
  const double* inv_freq;          // [pairs], radians per position
  const int32_t* axis;             // [pairs]
  int axes;
  int64_t B, S;
  int D, pairs;
  int halves;  // pairs (i, i + pairs), else (2 i, 2 i + 1)
  int inverse;
  int dtype;  // pasa_dtype_t
};
hipError_t launch_rope_axes(const RopeAxesParams& p, hipStream_t stream);

// ---- block tables (kv_tables.hip) ------------------------------------------------
constexpr int kMaxTableRequests = 4096;
struct KvTablesParams {
  int32_t* tables;  // [requests, width], rows `stride` apart
  int64_t stride;
  int64_t width;
  const int32_t* lens;
  const int32_t* new_tokens;
  int requests;
  const int32_t* free_pages;
  int64_t free_cap;
  const int32_t* num_free;
  int page_log2;
  int64_t tokens;
  int32_t* cu_q;
  int64_t* slots;
  int32_t* positions;
  int32_t* lens_out;
  int32_t* num_free_out;
};
hipError_t launch_kv_tables(const KvTablesParams& p, hipStream_t stream);

// ---- append (kv_append.hip) ------------------------------------------------------
struct KvAppendParams {
  KvCache c;
  const void* x[2];       // k, v
  int64_t tok_stride[2];  // elements
  int64_t head_stride[2];
  bool vec[2];  // eight channels can be loaded in 16-byte pieces
  const int64_t* slots;
  int64_t tokens;
  int dtype;
};
hipError_t launch_kv_append(const KvAppendParams& p, hipStream_t stream);

// ---- attention (kv_attn.hip) -----------------------------------------------------
struct KvAttnParams {
  KvCache c;
  const void* q;
  void* o;
  float* lse;  // [tokens, q_heads] or nullptr
  int64_t q_tok, q_head, o_tok, o_head;  // strides in elements
  const int32_t* tables;
  int64_t table_stride;
  int64_t width;
  const int32_t* lens;
  const int32_t* cu_q;  // nullptr: tokens / requests for each request
  int requests;
  int64_t tokens;
  int per_request;  // tokens / requests
  int q_heads;
  int group;        // q_heads / heads
  int64_t max_kv;   // keys from here on are not looked at
  int64_t window;   // 0: none
  int causal;
  int zero_tail;    // rows of no request are set to zero
  int q_vec, o_vec; // rows of q / o are 16-byte aligned
  float scale;      // softmax scale * log2 e
  int f16;          // q and o are fp16, else bf16
  int splits;
  float* part_o;    // [splits, tokens * q_heads, dim]
  float* part_ml;   // [splits, tokens * q_heads, 2]
};
struct KvAttnPlan {
  int rows;    // rows of a workgroup's tile: 16 or 32 (few), 128 or 256
  int splits;
};
KvAttnPlan kv_attn_plan(int64_t tokens, int requests, int q_heads, int kv_heads, int dim, int64_t max_kv);
hipError_t launch_kv_attn(const KvAttnParams& p, hipStream_t stream);

}  // namespace pasa
