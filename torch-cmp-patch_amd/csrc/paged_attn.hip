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
//    domain with fp32 state.  For fp16 and bf16 a weight enters the second
//    product in two parts, its value rounded to the tensors' type and the
//    rounded rest (the matrix units are idle for most of the time anyway).
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
  // what rounding a and b to w left, rounded
  static __device__ __forceinline__ uint32_t rest(uint32_t w, float a, float b) {
    const f16x2p h = __builtin_bit_cast(f16x2p, w);
    return pack(a - (float)h[0], b - (float)h[1]);
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
  static __device__ __forceinline__ uint32_t rest(uint32_t w, float a, float b) {
    return pack(a - __uint_as_float(w << 16), b - __uint_as_float(w & 0xffff0000u));
  }
};

constexpr int kRows = 16;        // query rows of a unit at most
constexpr int kTile = 16;        // slots of a tile
constexpr int kMaxWgs = 1024;    // workgroups of a launch at most (counters: one each)
constexpr int kMinTiles = 16;    // tiles of a workgroup's share at least
constexpr int kWhole = 32;       // tiles of a unit that is never split
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

// lds_dma16 of a buffer whose descriptor a v_readlane may just have written (the
// tile's own, or one that the compiler brings back from a lane): a vector
// instruction's SGPR is not there for a memory instruction before five wait
// states have passed, and the compiler does not see into the assembly.
__device__ __forceinline__ void lds_dma16_fresh(const u32x4& rs, uint32_t lds_byte, int voff) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rs), "{m0}"(lds_byte) : "memory");
}

struct Plan {
  f32x4* ws;  // parts: [workgroup][first or last segment][row] (DK / 4 + 1) float4: O, then (m, l, 0, 0)
  int* cnt;   // a counter for the unit that a workgroup's last segment begins
  int split;  // 0: whole units, dealt out in turn
  int group;  // query heads per K/V head
  int blocks; // row blocks per (sequence, K/V head)
  int units;  // of a sequence
  int tpp;    // tiles per page
};

// A sequence as the launch sees it.
struct Seq {
  int len, fresh;  // tokens, new ones among the columns
  int tiles;       // 0: nothing of it is read (no tokens, no new ones, or longer than its table row)
};
template <bool SEL>
__device__ __forceinline__ Seq seq_of(const PagedAttnParams& p, int b, int tpp) {
  Seq s;
  const int ps = p.map.page_size;
  s.len = seq_len_held(p.map, b);
  s.fresh = seq_new(p.map, b, p.S, s.len);
  if (s.fresh == 0 || s.len > p.map.width * ps) s.tiles = 0;
  else if (SEL) s.tiles = p.n_selected * tpp;
  else if (tpp * kTile == ps) s.tiles = (s.len + kTile - 1) / kTile;
  else s.tiles = s.len / ps * tpp + (s.len % ps + kTile - 1) / kTile;
  return s;
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
  __shared__ int s_flag;

  const int tid = thread_x(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wg = block_x(), nwg = (int)gridDim.x;
  const int c = lane & 15, g = lane >> 4;
  const int G = a.group, rows_all = G * p.S, U = a.units;
  const int ps = p.map.page_size, tpp = a.tpp;
  const int D = p.D;

  // ---- this workgroup's share [lo, hi) of all tiles.  Every wave sums over the
  // batch by itself (a lane takes `per` sequences in a row), so nothing waits.
  const int per = (p.B + 63) / 64;
  Seq held = {0, 0, 0};  // per == 1: lane b's is sequence b
  int b = 0, base = 0;   // the sequence at hand, the tiles before it
  int lo = 0, hi = 0, share = 0, extra = 0;
  bool idle = !a.split;  // a sequence has no tiles
  // sequence of the batch, the same for every lane
  auto seq_at = [&](int i) {
    Seq s;
    if (per == 1) {
      s.len = __builtin_amdgcn_readlane(held.len, i);
      s.fresh = __builtin_amdgcn_readlane(held.fresh, i);
      s.tiles = __builtin_amdgcn_readlane(held.tiles, i);
    } else {
      s = seq_of<SEL>(p, i, tpp);
      s.len = __builtin_amdgcn_readfirstlane(s.len);
      s.fresh = __builtin_amdgcn_readfirstlane(s.fresh);
      s.tiles = __builtin_amdgcn_readfirstlane(s.tiles);
    }
    return s;
  };
  if (per == 1 && lane < p.B) held = seq_of<SEL>(p, lane, tpp);
  if (a.split) {
    const int b0 = min(lane * per, p.B), b1 = min(b0 + per, p.B);
    int tiles = 0, busy = 0;
    if (per == 1) {
      tiles = held.tiles;
      busy = tiles > 0;
    } else {
      for (int i = b0; i < b1; ++i) {
        const int t = seq_of<SEL>(p, i, tpp).tiles;
        tiles += t;
        busy += t > 0;
      }
    }
    int inc = tiles, all = busy;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(inc, d), more = __shfl_xor(all, d);
      if (lane >= d) inc += up;
      all += more;
    }
    all = __builtin_amdgcn_readfirstlane(all);
    idle = all < p.B;
    const int total = __builtin_amdgcn_readlane(inc, 63) * U;
    // as many shares as workgroups, but of kMinTiles tiles at least, or a unit each
    const int n = min(nwg, max(total / kMinTiles, all * U));
    if (wg < n) {
      share = total / n;
      extra = total - share * n;
      lo = wg * share + min(wg, extra);
      hi = lo + share + (wg < extra ? 1 : 0);
      // units of kWhole tiles or fewer are not split: a share begins (and ends)
      // behind the unit its border falls into
      auto border = [&](int x, int& seq, int& before) {
        if (x >= total) return total;
        const uint64_t in = __builtin_amdgcn_ballot_w64((inc - tiles) * U <= x && x < inc * U);
        const int at = (int)__builtin_ctzll(in);
        before = __builtin_amdgcn_readlane(inc - tiles, at) * U;
        seq = at * per;
        Seq s = seq_at(seq);
        while (x >= before + s.tiles * U) {
          before += s.tiles * U;
          s = seq_at(++seq);
        }
        if (s.tiles > kWhole) return x;
        const int i = (x - before + s.tiles - 1) / s.tiles;
        return before + i * s.tiles;
      };
      int seq = 0, before = 0;
      hi = border(hi, seq, before);
      lo = border(lo, b, base);
    }
  }
  // the workgroup that holds tile x of a unit that may be split
  auto wg_of = [&](int x) {
    const int edge = (share + 1) * extra;
    return x < edge ? x / (share + 1) : extra + (x - edge) / share;
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

  int unit = wg;  // whole units: the one to do next
  int x = lo;
  bool more = a.split ? x < hi : unit < p.B * U;
  while (more) {
    // ---- the next segment: tiles [ta, tb) of unit (b, i), one of `parts`, the part-th
    Seq seq;
    int i, ta = 0, tb, parts = 1, part = 0, w0 = 0;
    if (a.split) {
      seq = seq_at(b);
      while (x >= base + seq.tiles * U) {
        base += seq.tiles * U;
        seq = seq_at(++b);
      }
      i = (x - base) / seq.tiles;
      const int u0 = base + i * seq.tiles, u1 = u0 + seq.tiles;
      ta = x - u0;
      tb = min(hi, u1) - u0;
      if (ta > 0 || tb < seq.tiles) {
        w0 = ta == 0 ? wg : wg_of(u0);
        parts = (tb == seq.tiles ? wg : wg_of(u1 - 1)) - w0 + 1;
        part = wg - w0;
      }
      x = u0 + tb;
      more = x < hi;
    } else {
      b = unit / U;
      i = unit - b * U;
      seq = seq_at(b);
      tb = seq.tiles;
      unit += nwg;
      more = unit < p.B * U;
      if (tb == 0) continue;
    }
    const int len = seq.len, fresh = seq.fresh;
    const int hk = a.blocks == 1 ? i : i / a.blocks;
    const int row0 = (i - hk * a.blocks) * kRows;
    const int R = min(kRows, rows_all - row0);
    const int mine = tb - ta > wave ? (tb - ta - wave + NW - 1) / NW : 0;  // tiles of this wave

    // offset (elements) of this unit's row r in a [B, H, S, D] tensor
    auto row_of = [&](int r, int64_t h_str, int64_t s_str) {
      if (p.S == 1) return (int64_t)(hk * G + row0 + r) * h_str;
      const int hr = (row0 + r) / p.S;
      return (int64_t)(hk * G + hr) * h_str + (int64_t)(row0 + r - hr * p.S) * s_str;
    };
    // row c sees the keys before `limit`; every row those before `sure`
    int limit = 0;
    if (c < R) {
      const int col = p.S == 1 ? 0 : (row0 + c) % p.S;
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

    // ---- what this wave's tiles [64 k, 64 k + 64) read, lane l's that of tile
    // 64 k + l: the page's address at the tile's first slot and the bytes from
    // there that hold keys (K and V), the position of the first key and the
    // tile's slots
    uint32_t ka[2], va[2];
    int kn = 0, vn = 0, pos0 = 0, slots0 = 0;
    bool bad = false;
    auto fetch = [&](int k) {
      const int j = 64 * k + lane, t = ta + wave + NW * j;
      int page = -1;
      kn = vn = pos0 = slots0 = 0;
      int slot = 0;
      if (j < mine) {
        const int e = tpp == 1 ? t : t / tpp;
        slot = (t - e * tpp) * kTile;
        const int col = SEL ? p.selected[((int64_t)b * p.Hkv + hk) * p.n_selected + e] : e;
        if (col >= 0) {
          page = col <= (len - 1) / ps ? page_at(p.map, b, col) : -1;
          bad |= page < 0;
          pos0 = page < 0 ? 0 : col * ps + slot;
          slots0 = page < 0 ? 0 : min(min(kTile, ps - slot), max(len - pos0, 0));
        }
      }
      if (slots0 > 0) {
        kn = (slots0 - 1) * ks_b + D * ES;
        vn = (slots0 - 1) * vs_b + D * ES;
      }
      const uint64_t kb = (uint64_t)((const char*)p.k + (max(page, 0) * p.kp_p + hk * p.kp_h + slot * p.kp_s) * ES);
      const uint64_t vb = (uint64_t)((const char*)p.v + (max(page, 0) * p.vp_p + hk * p.vp_h + slot * p.vp_s) * ES);
      ka[0] = (uint32_t)kb;
      ka[1] = (uint32_t)(kb >> 32) & 0xffffu;
      va[0] = (uint32_t)vb;
      va[1] = (uint32_t)(vb >> 32) & 0xffffu;
    };
    auto at_lane = [](uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    // this wave's tile j into stage j % NS
    auto issue = [&](int j) {
      const int l = j & 63;
      const u32x4 krw = {at_lane(ka[0], l), at_lane(ka[1], l), at_lane(kn, l), 0x00020000u};
      const u32x4 vrw = {at_lane(va[0], l), at_lane(va[1], l), at_lane(vn, l), 0x00020000u};
      const uint32_t st = ring + (uint32_t)((j % NS) * STAGE);
#pragma unroll
      for (int q = 0; q < IB; ++q) lds_dma16_fresh(krw, st + 1024 * q, kdo[q]);
#pragma unroll
      for (int q = 0; q < IB; ++q) lds_dma16_fresh(vrw, st + BLK + 1024 * q, vdo[q]);
    };

    f32x4 oacc[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) oacc[db] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;

    fetch(0);
    // (position, slots) of the tiles in flight: the lanes move on to the next 64
    // tiles when the first of those is issued, up to NS tiles ahead
    int pos_q[NS], slots_q[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      pos_q[j] = slots_q[j] = 0;
      if (j < mine) {
        pos_q[j] = __builtin_amdgcn_readlane(pos0, j);
        slots_q[j] = __builtin_amdgcn_readlane(slots0, j);
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
      const int pos = pos_q[0], slots = slots_q[0];
#pragma unroll
      for (int q = 0; q + 1 < NS; ++q) {
        pos_q[q] = pos_q[q + 1];
        slots_q[q] = slots_q[q + 1];
      }

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
      if (slots < kTile || pos + kTile > sure) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * g + e >= slots || pos + 4 * g + e >= limit) xs[e] = -INFINITY;
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
      l_run += (pe[0] + pe[1]) + (pe[2] + pe[3]);
      const unsigned char* vs = st + BLK;
      if constexpr (F32) {
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
        u32x2 pb, pl;
        pb[0] = Mma<T>::pack(pe[0], pe[1]);
        pb[1] = Mma<T>::pack(pe[2], pe[3]);
        pl[0] = Mma<T>::rest(pb[0], pe[0], pe[1]);
        pl[1] = Mma<T>::rest(pb[1], pe[2], pe[3]);
        // 16 lanes of group g read slots 4g .. 4g+3 x 16 columns, transposed:
        // lane c receives column 16 db + c of the four
        const int r = 4 * g + (c >> 2), ch = (c & 3) >> 1;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          typedef __attribute__((address_space(3))) i16x4p lds_i16x4;
          const unsigned char* at = vs + r * RB + 16 * pg_swz(r, 2 * db + ch, NC) + 8 * (c & 1);
          const i16x4p v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at);
          oacc[db] = Mma<T>::pv(__builtin_bit_cast(u32x2, v), pb, oacc[db]);
          oacc[db] = Mma<T>::pv(__builtin_bit_cast(u32x2, v), pl, oacc[db]);
        }
      }
      if (j + NS < mine) {
        if (((j + NS) & 63) == 0) fetch((j + NS) >> 6);
        pos_q[NS - 1] = __builtin_amdgcn_readlane(pos0, (j + NS) & 63);
        slots_q[NS - 1] = __builtin_amdgcn_readlane(slots0, (j + NS) & 63);
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
  for (int bb = idle ? wg : p.B; bb < p.B; bb += nwg) {
    const Seq seq = seq_of<SEL>(p, bb, tpp);
    if (seq.tiles > 0) continue;
    const bool err = seq.len > p.map.width * ps && seq.fresh > 0;
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
  const int64_t most = tiles / kMinTiles > units ? tiles / kMinTiles : units;
  return most < n ? (int)most : n;
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
  // tiles are counted in 32 bits: a table for more is read in whole units
  const int64_t cols = n_selected > 0 ? n_selected : width;
  const int64_t units = (int64_t)B * Hkv * ((H / Hkv * S + kRows - 1) / kRows);
  if (n <= 1 || units * cols * ((page_size + kTile - 1) / kTile) > INT32_MAX - kMaxWgs) return 0;
  return kExchangeCounterBytes + (size_t)n * 2 * kRows * (bucket(dtype, D) / 4 + 1) * sizeof(f32x4);
}

hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, hipStream_t s) {
  const int ps = p.map.page_size;
  const size_t need = paged_attn_workspace(dtype, p.B, p.H, p.Hkv, p.S, p.D, ps, p.map.width, p.n_selected);
  int wgs = workgroups(dtype, p.B, p.H, p.Hkv, p.S, p.D, ps, p.map.width, p.n_selected);
  const int G = p.H / p.Hkv, blocks = (G * p.S + kRows - 1) / kRows, tpp = (ps + kTile - 1) / kTile;
  Plan a = {nullptr, nullptr, 0, G, blocks, p.Hkv * blocks, tpp};
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
