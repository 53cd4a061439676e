// Shared definitions of the paged key-value cache's kernels.
#pragma once

#include "attn_common.h"

namespace cmpext3 {

// n / d for 0 <= n < 2^31 as a product: s = ceil(log2 d), m = floor(2^(31+s) / d)
// + 1 exceeds the quotient's scale by less than 2^s / 2^(31+s), too little to
// reach the next whole number.
struct Div {
  uint32_t m;
  int s;
};
__device__ __forceinline__ int quot(int n, uint32_t m, int s) { return (int)(__umulhi((uint32_t)n << 1, m) >> s); }

inline Div div_by(int d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  return {(uint32_t)((1ull << (31 + s)) / (uint32_t)d + 1), s};
}

// The sequences' pages and lengths (all on the device).
struct PageMap {
  const int32_t* table;  // [B][width], row stride `stride`
  int64_t stride;
  int width;
  const int32_t* lens;      // tokens of each sequence, the new ones among them
  const int32_t* new_lens;  // new tokens among the call's S columns; null: S
  int num_pages, page_size;
};

struct AppendParams {
  const void *k, *v, *q;
  void *q_out, *k_pages, *v_pages, *bounds;
  int64_t k_b, k_h, k_s, v_b, v_h, v_s, q_b, q_h, q_s, o_b, o_h, o_s;
  int64_t kp_p, kp_h, kp_s, vp_p, vp_h, vp_s, kb_p, kb_h, kb_e;
  int B, H, Hkv, S, D;
  PageMap map;
  const int32_t* positions;
  const float *cos, *sin;
  int rows, rot, interleaved;
  int64_t rot_s;
};

struct PagedAttnParams {
  const void *q, *k, *v;
  void* o;
  int64_t q_b, q_h, q_s, o_b, o_h, o_s;
  int64_t kp_p, kp_h, kp_s, vp_p, vp_h, vp_s;
  int B, H, Hkv, S, D;
  PageMap map;
  const int32_t* selected;
  int n_selected;
  float c;          // |scale| * log2(e)
  uint32_t q_sign;  // XORed into Q words when scale < 0
  void* workspace;  // null: sequences are not split
  size_t workspace_bytes;
};

struct SelectParams {
  const void *q, *bounds;
  int32_t* selected;
  int64_t q_b, q_h, kb_p, kb_h, kb_e;
  int B, H, Hkv, D;
  PageMap map;
  Div by_ps;
  int n_selected;
  void* workspace;
};

hipError_t launch_paged_append(const AppendParams& p, int dtype, hipStream_t s);
hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, hipStream_t s);
size_t paged_attn_workspace(int dtype, int B, int H, int Hkv, int S, int D, int page_size, int width, int n_selected);
hipError_t launch_paged_select(const SelectParams& p, int dtype, hipStream_t s);
size_t paged_select_workspace(int B, int Hkv, int width);

__device__ __forceinline__ int block_y() { return (int)__builtin_amdgcn_workgroup_id_y(); }
__device__ __forceinline__ int block_z() { return (int)__builtin_amdgcn_workgroup_id_z(); }

// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// Tokens of sequence b (0: none), and how many of the S columns are new.
__device__ __forceinline__ int seq_len(const PageMap& m, int b) { return max(m.lens[b], 0); }
// The same for readers: a sequence longer than its table row (an error) as one
// token longer, so that sums with it stay in 32 bits (the host bounds the row).
__device__ __forceinline__ int seq_len_held(const PageMap& m, int b) {
  return min(seq_len(m, b), m.width * m.page_size + 1);
}
__device__ __forceinline__ int seq_new(const PageMap& m, int b, int S, int len) {
  const int n = m.new_lens ? min(max(m.new_lens[b], 0), S) : S;
  return min(n, len);
}
// The page in column `col` of sequence b's table row, -1 when there is none.
__device__ __forceinline__ int page_at(const PageMap& m, int b, int64_t col) {
  if (col < 0 || col >= m.width) return -1;
  const int p = m.table[b * m.stride + col];
  return p >= 0 && p < m.num_pages ? p : -1;
}

}  // namespace cmpext3
