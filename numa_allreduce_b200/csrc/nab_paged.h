// Decode over a paged KV cache: block tables and slots (nab_paged.cu), head
// norm + rotation + append (nab_paged.cu), attention (nab_paged_attn.cu).
//
// Pages are [num_pages, Hkv, P, D]: the rows of one (page, kv head) are
// contiguous. Slot s of a token is page * P + row. A request's block table
// row lists its pages in the order of its positions.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace nab {

constexpr int kMaxPagedRequests = 8192;

struct AssignPagesArgs {
  const int* cached;       // [B] positions already held
  const int* starts;       // [B + 1] first token row of each request; null: one token each
  int* tables;             // [B, M], row stride table_stride
  int64_t table_stride;
  const int* free_pages;   // [F]
  const int* taken;        // [1] entries of free_pages already used
  int* positions;          // [T]
  int64_t* slots;          // [T]
  int* lengths;            // [B]
  int* taken_out;          // [1]
  int B, M, F, T, P;
};
void assign_pages(cudaStream_t s, const AssignPagesArgs& a, int sms);

struct RopeAppendArgs {
  const void* qkv;         // [T, (Hq + 2 Hkv) * D], row stride qkv_stride
  int64_t qkv_stride;
  const float* cos_t;      // [max_pos, R / 2]
  const float* sin_t;
  const int* positions;    // [T]
  const int64_t* slots;    // [T], negative: the token is not stored
  const void* q_norm;      // [D] or null
  const void* k_norm;      // [D] or null
  void* q_out;             // [T, Hq, D]
  void* k_pages;
  void* v_pages;
  int64_t T, num_slots;
  int Hq, Hkv, D, R, P, max_pos;
  float eps;
};
// dtype: kF16 or kBF16 (qkv, norms, pages and q_out share it).
void rope_append_paged(cudaStream_t s, const RopeAppendArgs& a, int dtype, bool interleaved, int sms);

struct PagedAttnArgs {
  const void* q;           // [B, Hq, D], batch stride q_stride
  int64_t q_stride;
  const void* k_pages;
  const void* v_pages;
  const int* tables;       // [B, M], row stride table_stride
  int64_t table_stride;
  const int* lengths;      // [B]
  void* out;               // [B, Hq, D]
  float* ws;               // paged_attention_ws_floats() floats
  int64_t num_pages;
  int B, M, P, Hq, Hkv, D;
  float scale;
};
int64_t paged_attention_ws_floats(int B, int M, int P, int Hq, int Hkv, int D, int sms);
void paged_attention(cudaStream_t s, const PagedAttnArgs& a, int dtype, int sms);

}  // namespace nab
