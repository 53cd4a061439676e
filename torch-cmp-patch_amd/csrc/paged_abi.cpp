// C ABI of the paged key-value cache: argument checks and kernel dispatch.
// Unsupported input is reported by return code and nothing is launched.
#include <float.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <mutex>

#include "../../include/cmpext3_paged.h"
#include "paged_common.h"

namespace cmpext3 {
// Held while a call's launches are submitted to a workspace (attn_abi.cpp): a
// selection hands its scores from one launch to the next there, and the
// attention calls that share a stream's workspace hand over mask bits, so no
// other call's launch may come between.
std::mutex& space_lock(const void* space);
}  // namespace cmpext3

namespace {

constexpr int kMaxColumns = 16;  // query columns of an attention call

int elem_size(int dtype) { return dtype == CMPEXT3_DTYPE_F32 ? 4 : dtype == CMPEXT3_DTYPE_F16 || dtype == CMPEXT3_DTYPE_BF16 ? 2 : 0; }

// Sizes, dtype, heads, head dim: what every call has.
int check_shape(int dtype, int B, int H, int Hkv, int S, int D, int num_pages, int page_size, int width) {
  const int es = elem_size(dtype);
  if (es == 0) return CMPEXT3_E_DTYPE;
  if (B < 0 || S < 0 || H < 1 || Hkv < 1 || H % Hkv != 0) return CMPEXT3_E_INVALID;
  if (num_pages < 1 || page_size < 1 || width < 0) return CMPEXT3_E_INVALID;
  if (D < 1 || D > 256 || D * es % 16 != 0) return CMPEXT3_E_HEAD_DIM;
  // 32-bit row and token indices
  if ((int64_t)B * H * S * (D * es / 16) > INT32_MAX / 2) return CMPEXT3_E_TOO_LARGE;
  if (((int64_t)width + 1) * page_size > INT32_MAX - 4096) return CMPEXT3_E_TOO_LARGE;
  return CMPEXT3_OK;
}

// A tensor's base and the strides of its dims with more than one index: whole
// 16-byte chunks, no negative step.
int check_tensor(const void* base, const int64_t str[3], int64_t n0, int64_t n1, int64_t n2, int es) {
  if (!base || !str) return CMPEXT3_E_INVALID;
  if ((uintptr_t)base & 15u) return CMPEXT3_E_ALIGN;
  const int64_t n[3] = {n0, n1, n2};
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 1) continue;
    if (str[i] < 0) return CMPEXT3_E_INVALID;
    if (str[i] * es % 16 != 0) return CMPEXT3_E_ALIGN;
  }
  return CMPEXT3_OK;
}

// A page's rows must not overlap (the kernels bound a page by its last row),
// and 16 of them (a tile) are addressed with 32-bit byte offsets.
int check_rows(const int64_t str[3], int page_size, int D, int es) {
  if (page_size > 1 && str[2] < D) return CMPEXT3_E_INVALID;
  if (page_size > 1 && str[2] * es > INT32_MAX / 32) return CMPEXT3_E_TOO_LARGE;
  return CMPEXT3_OK;
}

int check_map(const int32_t* table, int width, int64_t stride, int B, const int32_t* lens) {
  if (!lens || (!table && width > 0)) return CMPEXT3_E_INVALID;
  if (B > 1 && width > 0 && stride < 0) return CMPEXT3_E_INVALID;
  if (((uintptr_t)table | (uintptr_t)lens) & 3u) return CMPEXT3_E_ALIGN;
  return CMPEXT3_OK;
}

cmpext3::PageMap map_of(const int32_t* table, int width, int64_t stride, const int32_t* lens, const int32_t* new_lens,
                        int num_pages, int page_size) {
  return {table, stride, width, lens, new_lens, num_pages, page_size};
}

int done(hipError_t e) { return e == hipSuccess ? CMPEXT3_OK : CMPEXT3_E_LAUNCH; }

#define CHECKED(call)                     \
  do {                                    \
    const int rc_ = (call);               \
    if (rc_ != CMPEXT3_OK) return rc_;    \
  } while (0)

}  // namespace

extern "C" {

int cmpext3_paged_append(const void* k, const void* v, const void* q, void* q_out, void* k_pages, void* v_pages,
                         void* key_bounds, int dtype, int B, int H, int H_kv, int S, int D, int num_pages,
                         int page_size, const int64_t k_str[3], const int64_t v_str[3], const int64_t q_str[3],
                         const int64_t qo_str[3], const int64_t kp_str[3], const int64_t vp_str[3],
                         const int64_t kb_str[3], const int32_t* page_table, int table_width, int64_t table_stride,
                         const int32_t* seq_lens, const int32_t* new_lens, const int32_t* positions,
                         const float* cos, const float* sin, int table_rows, int rot, int64_t rot_stride,
                         int interleaved, hipStream_t stream) {
  CHECKED(check_shape(dtype, B, q ? H : H_kv, H_kv, S, D, num_pages, page_size, table_width));
  const int es = elem_size(dtype);
  if (B == 0 || S == 0) return CMPEXT3_OK;
  if ((q == nullptr) != (q_out == nullptr) || (cos == nullptr) != (sin == nullptr) || (q && !cos))
    return CMPEXT3_E_INVALID;
  CHECKED(check_tensor(k, k_str, B, H_kv, S, es));
  CHECKED(check_tensor(v, v_str, B, H_kv, S, es));
  if (q) {
    CHECKED(check_tensor(q, q_str, B, H, S, es));
    CHECKED(check_tensor(q_out, qo_str, B, H, S, es));
  }
  CHECKED(check_tensor(k_pages, kp_str, num_pages, H_kv, page_size, es));
  CHECKED(check_tensor(v_pages, vp_str, num_pages, H_kv, page_size, es));
  CHECKED(check_rows(kp_str, page_size, D, es));
  CHECKED(check_rows(vp_str, page_size, D, es));
  if (key_bounds) CHECKED(check_tensor(key_bounds, kb_str, num_pages, H_kv, 2, es));
  CHECKED(check_map(page_table, table_width, table_stride, B, seq_lens));
  if (q && q == q_out) return CMPEXT3_E_INVALID;
  // 32-bit item numbers, and a grid of less than 2^32 threads
  if ((int64_t)B * S * (2 * (int64_t)H_kv + (q ? H : 0)) * (D * es / 16) > INT32_MAX / 2 ||
      (key_bounds && (int64_t)B * H_kv * (S / page_size + 2) > (1 << 23)))
    return CMPEXT3_E_TOO_LARGE;
  if (((uintptr_t)new_lens | (uintptr_t)positions | (uintptr_t)cos | (uintptr_t)sin) & 3u) return CMPEXT3_E_ALIGN;
  if (cos && (rot < 2 || rot % 2 != 0 || rot > D || table_rows < 1 || (table_rows > 1 && rot_stride < 0)))
    return CMPEXT3_E_INVALID;

  cmpext3::AppendParams p;
  memset(&p, 0, sizeof p);
  p.k = k; p.v = v; p.q = q; p.q_out = q_out;
  p.k_pages = k_pages; p.v_pages = v_pages; p.bounds = key_bounds;
  p.k_b = k_str[0]; p.k_h = k_str[1]; p.k_s = k_str[2];
  p.v_b = v_str[0]; p.v_h = v_str[1]; p.v_s = v_str[2];
  if (q) {
    p.q_b = q_str[0]; p.q_h = q_str[1]; p.q_s = q_str[2];
    p.o_b = qo_str[0]; p.o_h = qo_str[1]; p.o_s = qo_str[2];
  }
  p.kp_p = kp_str[0]; p.kp_h = kp_str[1]; p.kp_s = kp_str[2];
  p.vp_p = vp_str[0]; p.vp_h = vp_str[1]; p.vp_s = vp_str[2];
  if (key_bounds) { p.kb_p = kb_str[0]; p.kb_h = kb_str[1]; p.kb_e = kb_str[2]; }
  p.B = B; p.H = q ? H : 0; p.Hkv = H_kv; p.S = S; p.D = D;
  p.map = map_of(page_table, table_width, table_stride, seq_lens, new_lens, num_pages, page_size);
  p.positions = positions;
  p.cos = cos; p.sin = sin;
  p.rows = table_rows; p.rot = cos ? rot : 0; p.interleaved = interleaved != 0;
  p.rot_s = table_rows > 1 ? rot_stride : 0;
  return done(cmpext3::launch_paged_append(p, dtype, stream));
}

size_t cmpext3_paged_attn_workspace_size(int dtype, int B, int H, int H_kv, int S, int D, int page_size,
                                         int table_width, int n_selected) {
  if (check_shape(dtype, B, H, H_kv, S, D, 1, page_size, table_width) != CMPEXT3_OK) return 0;
  if (B == 0 || S == 0 || S > kMaxColumns || n_selected < 0) return 0;
  return cmpext3::paged_attn_workspace(dtype, B, H, H_kv, S, D, page_size, table_width, n_selected);
}

int cmpext3_paged_attn(const void* q, const void* k_pages, const void* v_pages, void* o, int dtype, int B, int H,
                       int H_kv, int S, int D, int num_pages, int page_size, const int64_t q_str[3],
                       const int64_t kp_str[3], const int64_t vp_str[3], const int64_t o_str[3],
                       const int32_t* page_table, int table_width, int64_t table_stride, const int32_t* seq_lens,
                       const int32_t* new_lens, const int32_t* selected, int n_selected, float scale,
                       void* workspace, size_t workspace_bytes, hipStream_t stream) {
  CHECKED(check_shape(dtype, B, H, H_kv, S, D, num_pages, page_size, table_width));
  const int es = elem_size(dtype);
  if (S > kMaxColumns) return CMPEXT3_E_TOO_LARGE;
  if (B == 0 || S == 0) return CMPEXT3_OK;
  if (!isfinite(scale) || (selected && n_selected < 1)) return CMPEXT3_E_INVALID;
  CHECKED(check_tensor(q, q_str, B, H, S, es));
  CHECKED(check_tensor(o, o_str, B, H, S, es));
  CHECKED(check_tensor(k_pages, kp_str, num_pages, H_kv, page_size, es));
  CHECKED(check_tensor(v_pages, vp_str, num_pages, H_kv, page_size, es));
  CHECKED(check_rows(kp_str, page_size, D, es));
  CHECKED(check_rows(vp_str, page_size, D, es));
  CHECKED(check_map(page_table, table_width, table_stride, B, seq_lens));
  if (((uintptr_t)new_lens | (uintptr_t)selected) & 3u) return CMPEXT3_E_ALIGN;
  if ((uintptr_t)workspace & 15u) return CMPEXT3_E_ALIGN;
  if (selected && (int64_t)n_selected * ((page_size + 15) / 16) * 16 > INT32_MAX - 4096) return CMPEXT3_E_TOO_LARGE;

  cmpext3::PagedAttnParams p;
  memset(&p, 0, sizeof p);
  p.q = q; p.k = k_pages; p.v = v_pages; p.o = o;
  p.q_b = q_str[0]; p.q_h = q_str[1]; p.q_s = q_str[2];
  p.o_b = o_str[0]; p.o_h = o_str[1]; p.o_s = o_str[2];
  p.kp_p = kp_str[0]; p.kp_h = kp_str[1]; p.kp_s = page_size > 1 ? kp_str[2] : D;
  p.vp_p = vp_str[0]; p.vp_h = vp_str[1]; p.vp_s = page_size > 1 ? vp_str[2] : D;
  p.B = B; p.H = H; p.Hkv = H_kv; p.S = S; p.D = D;
  p.map = map_of(page_table, table_width, table_stride, seq_lens, new_lens, num_pages, page_size);
  p.selected = selected;
  p.n_selected = selected ? n_selected : 0;
  // above 0, so that a key left out stays at -inf: at the least normal number a
  // finite score is 0 to every digit
  p.c = fmaxf(fabsf(scale) * cmpext3::kLog2e, FLT_MIN);
  p.q_sign = scale < 0.f ? (es == 4 ? 0x80000000u : 0x80008000u) : 0u;
  p.workspace = workspace;
  p.workspace_bytes = workspace ? workspace_bytes : 0;
  std::unique_lock<std::mutex> submit(cmpext3::space_lock(workspace), std::defer_lock);
  if (p.workspace) submit.lock();
  return done(cmpext3::launch_paged_attn(p, dtype, stream));
}

size_t cmpext3_paged_select_workspace_size(int B, int H_kv, int table_width) {
  if (B < 1 || H_kv < 1 || table_width < 1) return 0;
  return cmpext3::paged_select_workspace(B, H_kv, table_width);
}

int cmpext3_paged_select(const void* q, const void* key_bounds, int32_t* selected, int dtype, int B, int H, int H_kv,
                         int D, int num_pages, int page_size, const int64_t q_str[3], const int64_t kb_str[3],
                         const int32_t* page_table, int table_width, int64_t table_stride, const int32_t* seq_lens,
                         int n_selected, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  CHECKED(check_shape(dtype, B, H, H_kv, 1, D, num_pages, page_size, table_width));
  const int es = elem_size(dtype);
  if (n_selected < 1) return CMPEXT3_E_INVALID;
  if ((int64_t)B * H_kv * n_selected > INT32_MAX / 2 || (int64_t)B * H_kv * (table_width + 64ll) > INT32_MAX / 2)
    return CMPEXT3_E_TOO_LARGE;
  if (B > 65535 || H_kv > 65535) return CMPEXT3_E_TOO_LARGE;  // grid
  if (B == 0) return CMPEXT3_OK;
  if (!selected) return CMPEXT3_E_INVALID;
  CHECKED(check_tensor(q, q_str, B, H, 1, es));
  CHECKED(check_tensor(key_bounds, kb_str, num_pages, H_kv, 2, es));
  CHECKED(check_map(page_table, table_width, table_stride, B, seq_lens));
  if ((uintptr_t)selected & 3u || (uintptr_t)workspace & 15u) return CMPEXT3_E_ALIGN;
  const size_t need = cmpext3_paged_select_workspace_size(B, H_kv, table_width);
  if (need > 0 && (!workspace || workspace_bytes < need)) return CMPEXT3_E_INVALID;

  cmpext3::SelectParams p;
  memset(&p, 0, sizeof p);
  p.q = q; p.bounds = key_bounds; p.selected = selected;
  p.q_b = q_str[0]; p.q_h = q_str[1];
  p.kb_p = kb_str[0]; p.kb_h = kb_str[1]; p.kb_e = kb_str[2];
  p.B = B; p.H = H; p.Hkv = H_kv; p.D = D;
  p.map = map_of(page_table, table_width, table_stride, seq_lens, nullptr, num_pages, page_size);
  p.by_ps = cmpext3::div_by(page_size);
  p.n_selected = n_selected;
  p.workspace = workspace;
  std::unique_lock<std::mutex> submit(cmpext3::space_lock(workspace), std::defer_lock);
  if (workspace) submit.lock();
  return done(cmpext3::launch_paged_select(p, dtype, stream));
}

}  // extern "C"
