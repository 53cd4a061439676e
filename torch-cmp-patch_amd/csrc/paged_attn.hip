// Attention of new tokens over a paged key-value cache: a few query rows per
// K/V head, a long sweep over keys that lie in pages.
//
// Such a launch moves almost nothing but K and V and is bound by the bytes it
// keeps in flight from HBM.  Nothing on the host knows the sequences' lengths,
// so the work is dealt out on the device:
//
//  * A unit is a (sequence, K/V head, block of 16 query rows); its keys are cut
//    into tiles of 16 slots, none across a page.  All units' tiles in a row are
//    one sequence of work, of which every workgroup takes an equal, contiguous
//    share (its prefix sum over the batch is the first thing a workgroup
//    does), so ragged batches load the chip evenly and a single long sequence
//    spreads over all of it.
//  * A workgroup's share is a list of segments, each within one unit.  Its four
//    waves take a segment's tiles in turn; every wave streams its own tiles
//    through a ring of stages in LDS filled by buffer_load ... lds (no staging
//    registers, no barriers), one buffer descriptor per tile: the page's
//    address is in its base, 64 bits wide, and its last valid slot is its end,
//    so slots behind the sequence read as zeros whatever they hold.
//  * A lane holds the page numbers of one of the wave's next 64 tiles (one
//    load of the table per 64 tiles, checked there), read back by v_readlane.
//  * Scores S^T = K Q^T and O^T = V^T P^T on 16x16 MFMAs (16x16x32 and 16x16x16
//    for fp16 and bf16, 16x16x4 for fp32), exact online softmax in the exp2
//    domain with fp32 state.  For fp16 and bf16 the weights are rounded to the
//    tensors' type for the second product; their sum takes the rounded values,
//    so the weights still add up to 1.
//  * End of a segment: the waves' (O, m, l) meet in LDS.  A unit that is one
//    segment is written out; otherwise each of its workgroups leaves its part
//    in the workspace and counts itself in, and the last one joins the parts in
//    their order and puts the counter back to zero.  Nobody waits for another
//    workgroup.
#include "paged_common.h"

namespace cmpext3 {

namespace {

typedef _Float16 f16x4p __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2p __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2p __attribute__((ext_vector_type(2)));
typedef short i16x4p __attribute__((ext_vector_type(4)));
typedef float f32x2p __attribute__((ext_vector_type(2)));

template <typename T> struct Mma;
template <> struct Mma<_Float16> {
  static __device__ __forceinline__ f32x4 qk(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 pv(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4p, a), __builtin_bit_cast(f16x4p, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2p){a, b}, f16x2p));
  }
  static __device__ __forceinline__ float sum2(uint32_t w, float acc) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2p, w), (f16x2p){1.0f16, 1.0f16}, acc, false);
  }
};
template <> struct Mma<__bf16> {
  static __device__ __forceinline__ f32x4 qk(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 pv(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4p, a), __builtin_bit_cast(i16x4p, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2p){a, b}, bf16x2p));
  }
  static __device__ __forceinline__ float sum2(uint32_t w, float acc) {
    const bf16x2p one = {(__bf16)1.0f, (__bf16)1.0f};
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2p, w), one, acc, false);
  }
};

constexpr int kRows = 16;        // query rows of a unit at most
constexpr int kTile = 16;        // slots of a tile
constexpr int kMaxWgs = 1024;    // workgroups of a launch at most (counters: one each)
constexpr int kMinTiles = 16;    // tiles of a workgroup's share at least
constexpr int kMergeLoads = 8;   // loads of one merging thread in flight together

// Waves per workgroup and stages per wave: as many stages as 128 KB of LDS
// hold, four at most.
constexpr int pg_waves(int rb) { return rb > 512 ? 2 : 4; }  // rb: bytes of a row in LDS
constexpr int pg_stages(int rb) {
  const int n = 128 * 1024 / (pg_waves(rb) * 2 * kTile * rb);
  return n < 4 ? n : 4;
}

// Physical 16-byte chunk of logical chunk c in LDS row r (nc chunks a row): XOR
// inside every whole group of 8 chunks, so that the fragment reads below (8
// rows, one chunk; 4 rows, two chunks; one row, 8 chunks) touch distinct banks.
__device__ __forceinline__ int pg_swz(int r, int c, int nc) {
  const int f = ((r & 3) << 1) | ((r >> 2) & 1);
  return c < (nc & ~7) ? (c ^ f) : c;
}

struct Plan {
  f32x4* ws;  // parts: [workgroup][first or last segment][row] (DK / 4 + 1) float4: O, then (m, l, 0, 0)
  int* cnt;   // a counter for the unit that a workgroup's last segment begins
  int split;  // 0: whole units, dealt out in turn
};

// Tiles of sequence b, 0 when nothing of it is read (no tokens, no new ones, or
// longer than its table row).
template <bool SEL>
__device__ __forceinline__ int tiles_of(const PagedAttnParams& p, int b, int tpp) {
  const int len = seq_len_held(p.map, b), ps = p.map.page_size;
  if (len == 0 || seq_new(p.map, b, p.S, len) == 0 || len > p.map.width * ps) return 0;
  if (SEL) return p.n_selected * tpp;
  const int full = len / ps;
  return full * tpp + (len - full * ps + kTile - 1) / kTile;
}

__device__ __forceinline__ float xor_f(float x, int m) { return __shfl_xor(x, m); }

template <typename T, int DK, bool SEL>
__global__ __launch_bounds__(pg_waves(DK * sizeof(T)) * 64, 1) void paged_attn(PagedAttnParams p, Plan a) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int ES = sizeof(T);
  constexpr int RB = DK * ES;           // bytes of a K/V row in LDS
  constexpr int NW = pg_waves(RB), NS = pg_stages(RB), NT = NW * 64;
  constexpr int NC = RB / 16;           // 16-byte chunks per row
  constexpr int BLK = kTile * RB;
  constexpr int IB = BLK / 1024;        // DMA instructions per 16 rows
  constexpr int STAGE = 2 * BLK;
  constexpr int IPT = 2 * IB;
  constexpr int KS = NC / 4;            // 16-byte chunks of a score operand per lane
  constexpr int NDB = DK / 16;          // float4 accumulators of a lane
  constexpr int DQ = DK / 4;            // float4 vectors of an output row
  constexpr int MOS = DK + 4;           // row stride (floats) of the waves' states
  constexpr int RING = NW * NS * STAGE;
  static_assert(BLK % 1024 == 0 && NC % 4 == 0 && (!F32 || DK % 64 == 0), "head dim bucket");
  static_assert(NS >= 1 && IPT * (NS - 1) <= 63, "vmcnt range");
  static_assert(NW * kRows * MOS * 4 + 2 * NW * kRows * 4 + 16 <= RING, "the waves' states fit the ring");
  __shared__ __attribute__((aligned(16))) unsigned char lds[RING];
  __shared__ int64_t s_wsum[NW];
  __shared__ int64_t s_at[2];
  __shared__ int s_b, s_flag;

  const int tid = thread_x(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wg = block_x(), nwg = (int)gridDim.x;
  const int c = lane & 15, g = lane >> 4;
  const int G = p.H / p.Hkv, rows_all = G * p.S, RBLK = (rows_all + kRows - 1) / kRows;
  const int U = p.Hkv * RBLK;           // units of a sequence
  const int ps = p.map.page_size, tpp = (ps + kTile - 1) / kTile;
  const int D = p.D;

  // ---- this workgroup's share [lo, hi) of all tiles, and the sequence it begins in
  int64_t lo = 0, hi = 0, share = 0, extra = 0;
  int b = 0;
  int64_t base = 0;  // tiles before sequence b
  if (a.split) {
    const int per = (p.B + NT - 1) / NT;
    const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
    int64_t mine = 0;
    for (int i = b0; i < b1; ++i) mine += (int64_t)tiles_of<SEL>(p, i, tpp) * U;
    int64_t inc = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t up = __shfl_up(inc, d);
      if (lane >= d) inc += up;
    }
    if (lane == 63) s_wsum[wave] = inc;
    __syncthreads();
    int64_t total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < wave) before += s_wsum[w];
      total += s_wsum[w];
    }
    const int64_t ex = before + inc - mine;
    const int64_t want = total / kMinTiles;
    const int n = want < 1 ? 1 : want < nwg ? (int)want : nwg;
    if (total > 0 && wg < n) {
      share = total / n;
      extra = total - share * n;
      lo = wg * share + (wg < extra ? wg : extra);
      hi = lo + share + (wg < extra ? 1 : 0);
      if (lo >= ex && lo < ex + mine) {
        int64_t at = ex;
        for (int i = b0; i < b1; ++i) {
          const int64_t t = (int64_t)tiles_of<SEL>(p, i, tpp) * U;
          if (lo < at + t) {
            s_b = i;
            s_at[0] = at;
            break;
          }
          at += t;
        }
      }
    }
    __syncthreads();
    if (lo < hi) {
      b = __builtin_amdgcn_readfirstlane(s_b);
      base = s_at[0];
    }
  }
  // the workgroup that holds tile x
  auto wg_of = [&](int64_t x) {
    const int64_t edge = (share + 1) * extra;
    return (int)(x < edge ? x / (share + 1) : extra + (x - edge) / share);
  };

  // ---- constant per-lane offsets
  // DMA: instruction i writes LDS bytes [1024 i, 1024 i + 1024); lane l's 16
  // bytes land at 1024 i + 16 l: row r, physical chunk pc, holding logical
  // chunk pg_swz(r, pc) of slot r.  Chunks past the head dim read zeros.
  const int ks_b = (int)p.kp_s * ES, vs_b = (int)p.vp_s * ES;
  int kdo[IB], vdo[IB];
#pragma unroll
  for (int i = 0; i < IB; ++i) {
    const int pos = 1024 * i + 16 * lane;
    const int r = pos / RB, lc = pg_swz(r, (pos - r * RB) / 16, NC);
    const bool in = 16 * lc < D * ES;
    kdo[i] = in ? r * ks_b + 16 * lc : (int)0x80000000u;
    vdo[i] = in ? r * vs_b + 16 * lc : (int)0x80000000u;
  }
  int kro[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) kro[ks] = c * RB + 16 * pg_swz(c, 4 * ks + g, NC);

  typedef __attribute__((address_space(3))) unsigned char lds_u8;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)lds;
  const uint32_t ring = lds0 + (uint32_t)(wave * NS * STAGE);
  float* const mo = (float*)lds;
  float* const mm = mo + NW * kRows * MOS;
  float* const ml = mm + NW * kRows;
  const float cmul = p.c;
  auto weight = [](float m, float mx) { return m == -INFINITY ? 0.f : fast_exp2(m - mx); };

  int unit = a.split ? 0 : wg;  // whole units: the one to do next
  int64_t x = lo;
  bool more = a.split ? x < hi : unit < p.B * U;
  while (more) {
    // ---- the next segment: tiles [ta, tb) of unit (b, i), one of `parts`, the part-th
    int nt, i, ta = 0, tb, parts = 1, part = 0, w0 = 0;
    if (a.split) {
      nt = __builtin_amdgcn_readfirstlane(tiles_of<SEL>(p, b, tpp));
      while (x >= base + (int64_t)nt * U) {
        base += (int64_t)nt * U;
        ++b;
        nt = __builtin_amdgcn_readfirstlane(tiles_of<SEL>(p, b, tpp));
      }
      i = (int)((x - base) / nt);
      const int64_t u0 = base + (int64_t)i * nt, u1 = u0 + nt;
      ta = (int)(x - u0);
      tb = (int)((hi < u1 ? hi : u1) - u0);
      w0 = ta == 0 ? wg : wg_of(u0);
      parts = (tb == nt ? wg : wg_of(u1 - 1)) - w0 + 1;
      part = wg - w0;
      x = u0 + tb;
      more = x < hi;
    } else {
      b = unit / U;
      i = unit - b * U;
      nt = __builtin_amdgcn_readfirstlane(tiles_of<SEL>(p, b, tpp));
      tb = nt;
      unit += nwg;
      more = unit < p.B * U;
      if (nt == 0) continue;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    const int hk = __builtin_amdgcn_readfirstlane(i / RBLK);
    const int row0 = (i - hk * RBLK) * kRows;
    const int R = min(kRows, rows_all - row0);
    const int len = __builtin_amdgcn_readfirstlane(seq_len_held(p.map, b));
    const int fresh = __builtin_amdgcn_readfirstlane(seq_new(p.map, b, p.S, len));
    const int mine = tb - ta > wave ? (tb - ta - wave + NW - 1) / NW : 0;  // tiles of this wave

    // offset (elements) of this unit's row r in a [B, H, S, D] tensor
    auto row_of = [&](int r, int64_t h_str, int64_t s_str) {
      const int hr = (row0 + r) / p.S;
      return (int64_t)(hk * G + hr) * h_str + (int64_t)(row0 + r - hr * p.S) * s_str;
    };
    // row c sees the keys before `limit`; every row those before `sure`
    int limit = 0;
    if (c < R) {
      const int col = (row0 + c) % p.S;
      limit = col < fresh ? len - fresh + col + 1 : 0;
    }
    const int sure = p.S == 1 ? len : 0;

    u32x4 qf[KS];
    {
      const T* qrow = (const T*)p.q + b * p.q_b + (c < R ? row_of(c, p.q_h, p.q_s) : 0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int ch = 4 * ks + g;
        u32x4 w = c < R && ch * 16 < D * ES ? *(const u32x4*)((const char*)qrow + 16 * ch) : (u32x4){0u, 0u, 0u, 0u};
        qf[ks] = w ^ (u32x4){p.q_sign, p.q_sign, p.q_sign, p.q_sign};
      }
    }

    // ---- pages of this wave's tiles [64 k, 64 k + 64): lane l those of tile 64 k + l
    int my_page = 0, my_pos = 0;  // page number (-1: nothing to read), position of the tile's first key
    bool bad = false;
    auto fetch = [&](int k) {
      const int j = 64 * k + lane, t = ta + wave + NW * j;
      my_page = -1;
      my_pos = 0;
      if (j < mine) {
        const int e = t / tpp, sub = t - e * tpp;
        const int col = SEL ? p.selected[((int64_t)b * p.Hkv + hk) * p.n_selected + e] : e;
        if (col >= 0) {
          my_page = (int64_t)col * ps < len ? page_at(p.map, b, col) : -1;
          my_pos = col * ps + sub * kTile;
          bad |= my_page < 0;
        }
      }
    };
    // this wave's tile j into stage j % NS
    auto issue = [&](int j) {
      const int page = __builtin_amdgcn_readlane(my_page, j & 63);
      const int pos = __builtin_amdgcn_readlane(my_pos, j & 63);
      const int slot = pos % ps;
      const int n = page < 0 ? 0 : min(min(kTile, ps - slot), len - pos);  // valid slots (<= 0: none)
      const char* kb = (const char*)p.k + ((int64_t)max(page, 0) * p.kp_p + hk * p.kp_h + slot * p.kp_s) * ES;
      const char* vb = (const char*)p.v + ((int64_t)max(page, 0) * p.vp_p + hk * p.vp_h + slot * p.vp_s) * ES;
      const u32x4 krw = uniform_rsrc_words(kb, n > 0 ? (int64_t)(n - 1) * ks_b + D * ES : 0);
      const u32x4 vrw = uniform_rsrc_words(vb, n > 0 ? (int64_t)(n - 1) * vs_b + D * ES : 0);
      const uint32_t st = ring + (uint32_t)((j % NS) * STAGE);
#pragma unroll
      for (int q = 0; q < IB; ++q) lds_dma16(krw, st + 1024 * q, kdo[q], 0);
#pragma unroll
      for (int q = 0; q < IB; ++q) lds_dma16(vrw, st + BLK + 1024 * q, vdo[q], 0);
    };

    f32x4 oacc[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) oacc[db] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;

    fetch(0);
    // (pages, positions) of the tile at hand: the lanes move on to the next 64
    // tiles when the first tile past them is issued, up to NS tiles ahead
    int pos_q[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      pos_q[j] = 0;
      if (j < mine) {
        pos_q[j] = __builtin_amdgcn_readlane(my_pos, j);
        if (__builtin_amdgcn_readlane(my_page, j) < 0) pos_q[j] = -1;
        issue(j);
      }
    }

    for (int j = 0; j < mine; ++j) {
      const int behind = min(NS - 1, mine - 1 - j);
      if (behind >= 3) wait_vmcnt<3 * IPT <= 63 ? 3 * IPT : 63>();
      else if (behind == 2) wait_vmcnt<2 * IPT <= 63 ? 2 * IPT : 63>();
      else if (behind == 1) wait_vmcnt<IPT <= 63 ? IPT : 63>();
      else wait_vmcnt<0>();
      const unsigned char* st = lds + (wave * NS + j % NS) * STAGE;
      const int pos = pos_q[0];
#pragma unroll
      for (int q = 0; q + 1 < NS; ++q) pos_q[q] = pos_q[q + 1];

      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 kk = *(const u32x4*)(st + kro[ks]);
        if constexpr (F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kk[e]), __uint_as_float(qf[ks][e]), s, 0, 0, 0);
        } else {
          s = Mma<T>::qk(kk, qf[ks], s);
        }
      }
      float xs[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) xs[e] = s[e] * cmul;
      const int slots = min(kTile, ps - pos % ps);
      if (pos < 0 || pos + kTile > sure || slots < kTile) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (pos < 0 || pos + 4 * g + e >= limit || 4 * g + e >= slots) xs[e] = -INFINITY;
      }
      float mt = fmaxf(fmaxf(xs[0], xs[1]), fmaxf(xs[2], xs[3]));
      mt = fmaxf(mt, xor_f(mt, 16));
      mt = fmaxf(mt, xor_f(mt, 32));
      if (__builtin_amdgcn_ballot_w64(mt > m_run)) {  // some row's maximum rises
        const float m_new = fmaxf(m_run, mt);
        const float alpha = weight(m_run, m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db) oacc[db] *= alpha;
      }
      const float m_sub = m_run == -INFINITY ? 0.f : m_run;
      float pe[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) pe[e] = fast_exp2(xs[e] - m_sub);
      const unsigned char* vs = st + BLK;
      if constexpr (F32) {
        l_run += (pe[0] + pe[1]) + (pe[2] + pe[3]);
        // 64 columns at a time: MFMA j takes columns 4 m + j (a lane's 16-byte
        // read is one slot's chunk, an element for each of the four)
#pragma unroll
        for (int db = 0; db < NDB; db += 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            const u32x4 v = *(const u32x4*)(vs + r * RB + 16 * pg_swz(r, 4 * db + c, NC));
#pragma unroll
            for (int q = 0; q < 4; ++q)
              oacc[db + q] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[q]), pe[e], oacc[db + q], 0, 0, 0);
          }
        }
      } else {
        u32x2 pb;
        pb[0] = Mma<T>::pack(pe[0], pe[1]);
        pb[1] = Mma<T>::pack(pe[2], pe[3]);
        l_run = Mma<T>::sum2(pb[1], Mma<T>::sum2(pb[0], l_run));
        // 16 lanes of group g read slots 4g .. 4g+3 x 16 columns, transposed:
        // lane c receives column 16 db + c of the four
        const int r = 4 * g + (c >> 2), ch = (c & 3) >> 1;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          typedef __attribute__((address_space(3))) i16x4p lds_i16x4;
          const unsigned char* at = vs + r * RB + 16 * pg_swz(r, 2 * db + ch, NC) + 8 * (c & 1);
          const i16x4p v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at);
          oacc[db] = Mma<T>::pv(__builtin_bit_cast(u32x2, v), pb, oacc[db]);
        }
      }
      if (j + NS < mine) {
        if (((j + NS) & 63) == 0) fetch((j + NS) >> 6);
        pos_q[NS - 1] = __builtin_amdgcn_readlane(my_pos, (j + NS) & 63);
        if (__builtin_amdgcn_readlane(my_page, (j + NS) & 63) < 0) pos_q[NS - 1] = -1;
        // this stage's LDS reads have returned before its next tile's loads go out
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        issue(j + NS);
      }
    }

    // ---- the waves' states meet in LDS: [wave][row][DK] O, then m, l
    float lrow = l_run + xor_f(l_run, 16);
    lrow += xor_f(lrow, 32);
    if (__builtin_amdgcn_ballot_w64(bad)) lrow = __builtin_nanf("");  // a page that is none: the unit's rows are NaN
    wait_vmcnt<0>();
    lds_barrier();  // every wave is done with its ring
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      // fp32: accumulators 4 k .. 4 k + 3 hold columns 64 k + 16 g + 4 e + (0 .. 3)
      if constexpr (F32) {
        const int k4 = db & ~3, e = db & 3;
        *(f32x4*)(mo + (wave * kRows + c) * MOS + 16 * k4 + 16 * g + 4 * e) =
            (f32x4){oacc[k4][e], oacc[k4 + 1][e], oacc[k4 + 2][e], oacc[k4 + 3][e]};
      } else {
        *(f32x4*)(mo + (wave * kRows + c) * MOS + 16 * db + 4 * g) = oacc[db];
      }
    }
    if (g == 0) {
      mm[wave * kRows + c] = m_run;
      ml[wave * kRows + c] = lrow;
    }
    lds_barrier();

    const int nu = R * DQ;  // (row, 4 columns) vectors of the output
    T* const og = (T*)p.o + b * p.o_b;
    auto inverse = [](float l) { return l == 0.f ? 0.f : 1.f / l; };
    auto store_out = [&](int r, int k, f32x4 o, float inv) {
      if (4 * k >= D) return;
      T* const at = og + row_of(r, p.o_h, p.o_s) + 4 * k;
      if constexpr (F32) {
        *(f32x4*)at = o * inv;
      } else {
        u32x2 w;
        w[0] = Mma<T>::pack(o[0] * inv, o[1] * inv);
        w[1] = Mma<T>::pack(o[2] * inv, o[3] * inv);
        *(u32x2*)at = w;
      }
    };
    const __amdgpu_buffer_rsrc_t wsr =
        uniform_rsrc(parts > 1 ? (const void*)a.ws : (const void*)p.o,
                     parts > 1 ? (int64_t)nwg * 2 * kRows * (DQ + 1) * 16 : 16);
    // slot of part q's row r: a part that begins the unit is its workgroup's
    // last segment, the others are their workgroups' first
    auto slot = [&](int q, int r, int k) { return ((((w0 + q) * 2 + (q == 0 ? 1 : 0)) * kRows + r) * (DQ + 1) + k) * 16; };
    for (int u = tid; u < nu; u += NT) {
      const int r = u / DQ, k = u - r * DQ;
      float mw[NW], mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        mw[w] = mm[w * kRows + r];
        mx = fmaxf(mx, mw[w]);
      }
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = weight(mw[w], mx);
        l = __builtin_fmaf(ml[w * kRows + r], f, l);
        o += *(const f32x4*)(mo + (w * kRows + r) * MOS + 4 * k) * f;
      }
      if (parts == 1) {
        store_out(r, k, o, inverse(l));
      } else {
        // device-scope (aux 16 = sc1) stores, coherent across the XCDs' L2s
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), wsr, slot(part, r, k), 0, 16);
        if (k == 0)
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, ((f32x4){mx, l, 0.f, 0.f})), wsr,
                                                 slot(part, r, DQ), 0, 16);
      }
    }
    bool last = false;
    if (parts > 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      lds_barrier();  // every wave's stores are done
      if (tid == 0) {
        const int old = __hip_atomic_fetch_add(a.cnt + w0, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (old == parts - 1) __hip_atomic_store(a.cnt + w0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_flag = old == parts - 1;
      }
      lds_barrier();
      last = __builtin_amdgcn_readfirstlane(s_flag) != 0;
      asm volatile("" ::: "memory");  // the loads of the parts stay after the count
    }
    if (last) {
      // ---- join the unit's parts: (1) every part's (m, l) of every row, then
      // per row (one wave each) the weight of each part, over the total; (2)
      // every thread sums its share of the weighted vectors, the parts spread
      // over S groups of threads whose sums meet in LDS.  Fixed assignment and
      // order: the same result whichever workgroup joins.
      auto ld = [&](int off) { return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(wsr, off, 0, 16)); };
      const int n = parts;
      // rows at a time, so that their weights fit the ring's LDS whatever the parts
      const int rstep = min(R, max(1, (RING - NT * 16 - 64) / (8 * n)));
      for (int r0 = 0; r0 < R; r0 += rstep) {
        const int rn = min(rstep, R - r0);
        float* const wq = (float*)lds;  // [row][part]
        float* const lq = wq + rn * n;
        for (int k = tid; k < rn * n; k += NT) {
          const int r = k / n, q = k - r * n;
          const f32x4 e = ld(slot(q, r0 + r, DQ));
          wq[k] = e[0];
          lq[k] = e[1];
        }
        lds_barrier();
        for (int r = wave; r < rn; r += NW) {
          float* const wr = wq + r * n;
          const float* const lr = lq + r * n;
          float mx = -INFINITY;
          for (int q = lane; q < n; q += 64) mx = fmaxf(mx, wr[q]);
#pragma unroll
          for (int m = 32; m >= 1; m >>= 1) mx = fmaxf(mx, xor_f(mx, m));
          float L = 0.f;
          for (int q = lane; q < n; q += 64) L = __builtin_fmaf(lr[q], weight(wr[q], mx), L);
#pragma unroll
          for (int m = 32; m >= 1; m >>= 1) L += xor_f(L, m);
          const float inv = inverse(L);
          for (int q = lane; q < n; q += 64) wr[q] = weight(wr[q], mx) * inv;
        }
        lds_barrier();
        const int nv = rn * DQ;
        const int S = nv >= NT ? 1 : NT / nv;
        f32x4* const acc = (f32x4*)(lds + ((2 * rn * n * 4 + 15) & ~15));
        for (int u0 = 0; u0 < nv; u0 += NT / S) {
          const int t = tid % (NT / S), sg = tid / (NT / S), u = u0 + t;
          f32x4 o = {0.f, 0.f, 0.f, 0.f};
          if (u < nv && sg < S) {
            const int r = u / DQ, k = u - r * DQ;
            const float* const wr = wq + r * n;
            for (int q0 = sg; q0 < n; q0 += kMergeLoads * S) {
              f32x4 v[kMergeLoads];
#pragma unroll
              for (int z = 0; z < kMergeLoads; ++z) {
                const int q = q0 + z * S;
                v[z] = q < n ? ld(slot(q, r0 + r, k)) : (f32x4){0.f, 0.f, 0.f, 0.f};
              }
#pragma unroll
              for (int z = 0; z < kMergeLoads; ++z) {
                const int q = q0 + z * S;
                if (q < n) o += v[z] * wr[q];
              }
            }
            if (S == 1) store_out(r0 + r, k, o, 1.f);
          }
          if (S > 1) {  // nv < NT: one pass
            if (sg < S && u < nv) acc[sg * nv + u] = o;
            lds_barrier();
            if (tid < nv) {
              f32x4 sum = acc[tid];
              for (int s2 = 1; s2 < S; ++s2) sum += acc[s2 * nv + tid];
              store_out(r0 + tid / DQ, tid % DQ, sum, 1.f);
            }
          }
        }
        lds_barrier();  // the weights have been read
      }
    }
    lds_barrier();  // the LDS is free for the next segment
  }

  // ---- places nothing was read for: zeros, NaN where the sequence is longer than its table row
  for (int bb = wg; bb < p.B; bb += nwg) {
    if (tiles_of<SEL>(p, bb, tpp) > 0) continue;
    const int len = seq_len_held(p.map, bb);
    const bool err = len > p.map.width * ps && seq_new(p.map, bb, p.S, len) > 0;
    const uint32_t w = err ? (F32 ? 0x7fc00000u : 0x7fff7fffu) : 0u;
    const int nc = D * ES / 16;
    for (int u = tid; u < p.H * p.S * nc; u += NT) {
      const int r = u / nc, h = r / p.S;
      *(u32x4*)((char*)p.o + (bb * p.o_b + h * p.o_h + (r - h * p.S) * p.o_s) * ES + 16 * (u - r * nc)) = (u32x4){w, w, w, w};
    }
  }
}

int bucket(int dtype, int D) {
  if (dtype == 2) return (D + 63) / 64 * 64;
  return D <= 64 ? 64 : D <= 160 ? (D + 31) / 32 * 32 : (D + 63) / 64 * 64;
}

// Workgroups of a launch: what the CUs hold at once, or fewer when the table
// rows do not hold that many shares of kMinTiles tiles.
int workgroups(int dtype, int B, int H, int Hkv, int S, int D, int page_size, int width, int n_selected) {
  const int rb = bucket(dtype, D) * (dtype == 2 ? 4 : 2);
  const int lds = pg_waves(rb) * pg_stages(rb) * 2 * kTile * rb;
  int n = device_cus() * (160 * 1024 / (lds + 4096));
  if (n > kMaxWgs) n = kMaxWgs;
  const int64_t units = (int64_t)B * Hkv * ((H / Hkv * S + kRows - 1) / kRows);
  const int64_t cols = n_selected > 0 ? n_selected : width;
  const int64_t tiles = units * cols * ((page_size + kTile - 1) / kTile);
  const int64_t most = (tiles + kMinTiles - 1) / kMinTiles;
  return most < 1 ? 1 : most < n ? (int)most : n;
}

template <typename T, int DK>
hipError_t launch_dk(const PagedAttnParams& p, const Plan& a, int wgs, hipStream_t s) {
  const dim3 grid(wgs), block(pg_waves(DK * sizeof(T)) * 64);
  if (p.n_selected > 0) hipLaunchKernelGGL((paged_attn<T, DK, true>), grid, block, 0, s, p, a);
  else hipLaunchKernelGGL((paged_attn<T, DK, false>), grid, block, 0, s, p, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch16(const PagedAttnParams& p, const Plan& a, int wgs, hipStream_t s) {
  switch (bucket(0, p.D)) {
    case 64: return launch_dk<T, 64>(p, a, wgs, s);
    case 96: return launch_dk<T, 96>(p, a, wgs, s);
    case 128: return launch_dk<T, 128>(p, a, wgs, s);
    case 160: return launch_dk<T, 160>(p, a, wgs, s);
    case 192: return launch_dk<T, 192>(p, a, wgs, s);
  }
  return launch_dk<T, 256>(p, a, wgs, s);
}

}  // namespace

size_t paged_attn_workspace(int dtype, int B, int H, int Hkv, int S, int D, int page_size, int width, int n_selected) {
  const int n = workgroups(dtype, B, H, Hkv, S, D, page_size, width, n_selected);
  if (n <= 1) return 0;
  return kExchangeCounterBytes + (size_t)n * 2 * kRows * (bucket(dtype, D) / 4 + 1) * sizeof(f32x4);
}

hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, hipStream_t s) {
  const int ps = p.map.page_size;
  const size_t need = paged_attn_workspace(dtype, p.B, p.H, p.Hkv, p.S, p.D, ps, p.map.width, p.n_selected);
  int wgs = workgroups(dtype, p.B, p.H, p.Hkv, p.S, p.D, ps, p.map.width, p.n_selected);
  Plan a = {nullptr, nullptr, 0};
  if (need > 0 && p.workspace && p.workspace_bytes >= need) {
    a.cnt = (int*)p.workspace;
    a.ws = (f32x4*)((char*)p.workspace + kExchangeCounterBytes);
    a.split = 1;
  }
  if (dtype == 0) return launch16<_Float16>(p, a, wgs, s);
  if (dtype == 1) return launch16<__bf16>(p, a, wgs, s);
  switch (bucket(2, p.D)) {
    case 64: return launch_dk<float, 64>(p, a, wgs, s);
    case 128: return launch_dk<float, 128>(p, a, wgs, s);
    case 192: return launch_dk<float, 192>(p, a, wgs, s);
  }
  return launch_dk<float, 256>(p, a, wgs, s);
}

}  // namespace cmpext3
