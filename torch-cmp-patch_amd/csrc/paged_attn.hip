// Host side of the paged attention: head dim buckets, workgroups, workspace.
#include <string.h>

#include "paged_attn.h"

namespace cmpext3 {

hipError_t launch_paged_attn_f16(const AttnArgs& a, int wgs, hipStream_t s);
hipError_t launch_paged_attn_bf16(const AttnArgs& a, int wgs, hipStream_t s);
hipError_t launch_paged_attn_f32(const AttnArgs& a, int wgs, hipStream_t s);

namespace {

int bucket(int dtype, int D) {
  if (dtype == 2) return (D + 63) / 64 * 64;
  return D <= 64 ? 64 : D <= 160 ? (D + 31) / 32 * 32 : (D + 63) / 64 * 64;
}

// Query rows of a unit.
int unit_rows(int dtype, int D, int rows) {
  return kRows * pg_row_blocks(bucket(dtype, D) * (dtype == 2 ? 4 : 2), rows);
}
// Rows of a part in the workspace.
int slot_rows(int dtype, int D, int rows) {
  const int n = unit_rows(dtype, D, rows);
  return rows < n ? rows : n;
}
int64_t unit_count(int dtype, int B, int H, int Hkv, int S, int D) {
  const int rows = H / Hkv * S, n = unit_rows(dtype, D, rows);
  return (int64_t)B * Hkv * ((rows + n - 1) / n);
}

// Workgroups that the CUs hold at once.
int full_house(int dtype, int D) {
  const int lds = 160 * 1024 / (pg_lds(bucket(dtype, D), dtype == 2 ? 4 : 2) + 512);
  const int n = device_cus() * (lds < kPerCu ? lds : kPerCu);
  return n < kMaxWgs ? n : kMaxWgs;
}

// Workgroups of a launch: what the CUs hold at once, or fewer when the table
// rows do not hold that many shares of kMinTiles tiles.
int workgroups(int dtype, int B, int H, int Hkv, int S, int D, int page_size, int width, int n_selected) {
  const int n = full_house(dtype, D);
  const int64_t units = unit_count(dtype, B, H, Hkv, S, D);
  const int64_t cols = n_selected > 0 ? n_selected : width;
  const int64_t tiles = units * cols * ((page_size + kTile - 1) / kTile);
  const int64_t most = units + (tiles + kSetup * units) / pg_min_tiles(dtype == 2 ? 4 : 2);
  return most < n ? (int)most : n;
}

}  // namespace

size_t paged_attn_workspace(int dtype, int B, int H, int Hkv, int S, int D, int page_size, int width, int n_selected) {
  const int n = workgroups(dtype, B, H, Hkv, S, D, page_size, width, n_selected);
  // tiles are counted in 32 bits: a table for more is read in whole units
  const int64_t cols = n_selected > 0 ? n_selected : width;
  const int64_t units = unit_count(dtype, B, H, Hkv, S, D);
  if (n <= 1 || width == 0 || units * (cols * ((page_size + kTile - 1) / kTile) + kSetup) > INT32_MAX / 2) return 0;
  return kExchangeCounterBytes + (size_t)n * 2 * slot_rows(dtype, D, H / Hkv * S) * (bucket(dtype, D) / 4 + 1) * sizeof(f32x4);
}

hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, hipStream_t s) {
  const int ps = p.map.page_size;
  const size_t need = paged_attn_workspace(dtype, p.B, p.H, p.Hkv, p.S, p.D, ps, p.map.width, p.n_selected);
  int wgs = workgroups(dtype, p.B, p.H, p.Hkv, p.S, p.D, ps, p.map.width, p.n_selected);
  const int G = p.H / p.Hkv, ur = unit_rows(dtype, p.D, G * p.S), blocks = (G * p.S + ur - 1) / ur, tpp = (ps + kTile - 1) / kTile;
  const int es = dtype == 2 ? 4 : 2;
  AttnArgs a;
  memset(&a, 0, sizeof a);
  a.lens = p.map.lens; a.news = p.map.new_lens; a.table = p.map.table; a.selected = p.selected;
  a.t_str = p.map.stride;
  a.B = p.B; a.S = p.S; a.U = p.Hkv * blocks; a.cap = p.map.width * ps;
  a.nsel = p.n_selected; a.width = p.map.width; a.ps = ps; a.tpp = tpp;
  a.by_ps = div_by(ps); a.by_tpp = div_by(tpp); a.by_blocks = div_by(blocks); a.by_s = div_by(p.S);
  a.exact = ps % kTile == 0;
  a.full = full_house(dtype, p.D) > device_cus() ? full_house(dtype, p.D) : 0;
  a.G = G; a.blocks = blocks; a.rows = G * p.S; a.slot_rows = slot_rows(dtype, p.D, G * p.S); a.num_pages = p.map.num_pages;
  a.k = (const char*)p.k; a.v = (const char*)p.v;
  a.kp_p = p.kp_p * es; a.kp_h = p.kp_h * es; a.vp_p = p.vp_p * es; a.vp_h = p.vp_h * es;
  a.ks_b = (int)p.kp_s * es; a.vs_b = (int)p.vp_s * es; a.row_b = p.D * es; a.D = p.D;
  a.q = p.q; a.q_b = p.q_b; a.q_h = p.q_h; a.q_s = p.q_s;
  a.o = p.o; a.o_b = p.o_b; a.o_h = p.o_h; a.o_s = p.o_s;
  a.c = p.c; a.q_sign = p.q_sign;
  if (need > 0 && p.workspace && p.workspace_bytes >= need) {
    a.cnt = (int*)p.workspace;
    a.ws = (f32x4*)((char*)p.workspace + kExchangeCounterBytes);
    a.split = 1;
  }
  if (dtype == 0) return launch_paged_attn_f16(a, wgs, s);
  if (dtype == 1) return launch_paged_attn_bf16(a, wgs, s);
  return launch_paged_attn_f32(a, wgs, s);
}

}  // namespace cmpext3
