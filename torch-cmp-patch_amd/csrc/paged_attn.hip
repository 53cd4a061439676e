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
#include <string.h>

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
constexpr int kPerCu = 2;        // workgroups per CU at most
constexpr int kMinTiles = 16;    // tiles of a workgroup's share at least
constexpr int kSetup = 6;        // what a unit costs beside its tiles, in tiles
constexpr int kWhole = 32;       // tiles of a unit that is never split
constexpr int kLongShare = 48;   // tiles of a share from which one workgroup a CU is enough
constexpr int kMergeLoads = 8;   // parts of one merging thread in flight together

// Waves per workgroup and stages per wave: as many stages as 64 KB of LDS hold,
// four at most, so that two workgroups fit a CU.  More in flight is no faster
// (bf16 [16,16/8,4096,128]: 54.3 us with 128 KB a CU, 52.0 with 64).
constexpr int pg_waves(int rb) { return rb > 512 ? 2 : 4; }  // rb: bytes of a row in LDS
constexpr int pg_stages(int rb) {
  const int n = 64 * 1024 / (pg_waves(rb) * 2 * kTile * rb);
  return n < 1 ? 1 : n < 4 ? n : 4;
}
// LDS of a workgroup: the rings, later the waves' states in the same place
constexpr int pg_lds(int dk, int es) {
  const int nw = pg_waves(dk * es), ring = nw * pg_stages(dk * es) * 2 * kTile * dk * es;
  const int states = nw * kRows * (dk + 6) * 4;
  return ring > states ? ring : states;
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

struct AttnArgs {
  const int32_t *lens, *news, *table, *selected;
  int64_t t_str;
  int B, S, U, cap;        // U: units of a sequence; cap: keys a table row holds
  int nsel, width, ps, tpp;  // tpp: tiles per page
  Div by_ps, by_tpp, by_blocks, by_s;
  int split, exact, full;  // split 0: whole units, dealt out in turn; exact: pages are whole tiles; full: workgroups the CUs hold
  int G, blocks, rows, num_pages;  // query heads per K/V head, row blocks and rows of a K/V head
  const char *k, *v;
  int64_t kp_p, kp_h, vp_p, vp_h;  // bytes
  int ks_b, vs_b, row_b, D;        // bytes of a slot's stride, of a row
  const void* q;
  int64_t q_b, q_h, q_s;
  void* o;
  int64_t o_b, o_h, o_s;
  float c;
  uint32_t q_sign;
  f32x4* ws;  // parts: [workgroup][first or last segment][row] (DK / 4 + 1) float4: O, then (m, l, 0, 0)
  int* cnt;   // a counter for the unit that a workgroup's last segment begins
};
typedef const __attribute__((address_space(4))) AttnArgs* ArgsPtr;
// The arguments, read anew from here on: a phase of the kernel loads those it
// uses, and none has to stay in (or spill from) scalar registers between
// phases.
__device__ __forceinline__ ArgsPtr anew(ArgsPtr p) {
  asm volatile("" : "+s"(p));
  return p;
}

// A sequence as the launch sees it.
struct Seq {
  int len, fresh;  // tokens, new ones among the columns
  int tiles;       // 0: nothing of it is read (no tokens, no new ones, or longer than its table row)
};
template <bool SEL>
__device__ __forceinline__ Seq seq_from(ArgsPtr p, int len, int fresh) {
  Seq s;
  s.len = min(max(len, 0), p->cap + 1);
  s.fresh = min(min(max(fresh, 0), p->S), s.len);
  if (s.fresh == 0 || s.len > p->cap) s.tiles = 0;
  else if (SEL) s.tiles = p->nsel * p->tpp;
  else if (p->exact) s.tiles = (s.len + kTile - 1) / kTile;
  else {
    const int full = quot(s.len, p->by_ps.m, p->by_ps.s);
    s.tiles = full * p->tpp + (s.len - full * p->ps + kTile - 1) / kTile;
  }
  return s;
}

template <bool SEL>
__device__ __forceinline__ Seq seq_of(ArgsPtr p, int b) {
  return seq_from<SEL>(p, p->lens[b], p->news ? p->news[b] : p->S);
}

__device__ __forceinline__ float xor_f(float x, int m) { return __shfl_xor(x, m); }
// max / sum over the lanes 16 and 32 apart
__device__ __forceinline__ float rows_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xhalf_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float rows_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xhalf_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

template <typename T, int DK, bool SEL>
__global__ __launch_bounds__(pg_waves(DK * sizeof(T)) * 64, 1) void paged_attn(AttnArgs) {
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
  constexpr int LDS = pg_lds(DK, ES);   // the ring, then the waves' states
  static_assert(LDS >= RING && LDS >= NW * kRows * (MOS + 2) * 4, "the waves' states fit");
  __shared__ __attribute__((aligned(16))) unsigned char lds[LDS];
  __shared__ int s_flag;

  const int tid = thread_x(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wg = block_x(), nwg = (int)gridDim.x;
  const int c = lane & 15, g = lane >> 4;
  const ArgsPtr args = (ArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();

  // the lane's own lengths are on their way while the offsets below are made
  int my_len = 0, my_new = 0;
  {
    const ArgsPtr p = anew(args);
    if (lane < p->B) {
      my_len = p->lens[lane];
      my_new = p->news ? p->news[lane] : p->S;
    }
  }

  // ---- constant per-lane offsets
  // DMA: instruction i writes LDS bytes [1024 i, 1024 i + 1024); lane l's 16
  // bytes land at 1024 i + 16 l: row r, physical chunk pc, holding logical
  // chunk pg_swz(r, pc) of slot r.  Chunks past the head dim read zeros.
  int kdo[IB], vdo[IB];
  {
    const ArgsPtr p = anew(args);
    const int ks_b = p->ks_b, vs_b = p->vs_b, row_b = p->row_b;
#pragma unroll
    for (int i = 0; i < IB; ++i) {
      const int pos = 1024 * i + 16 * lane;
      const int r = pos / RB, lc = pg_swz(r, (pos - r * RB) / 16, NC);
      const bool in = 16 * lc < row_b;
      kdo[i] = in ? r * ks_b + 16 * lc : (int)0x80000000u;
      vdo[i] = in ? r * vs_b + 16 * lc : (int)0x80000000u;
    }
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
  // ---- this workgroup's share [lo, hi) of all units, counted in tiles (plus
  // kSetup for each unit's own cost).  Every wave sums over the batch by itself
  // (a lane takes `per` sequences in a row), so nothing waits.
  int b = 0, base = 0;  // the sequence at hand, what lies before it
  int x = 0, hi = 0, share = 1;
  bool idle = true;     // a sequence has no tiles
  int depth = NS;       // stages in use
  Seq held = {0, 0, 0};  // B <= 64: lane b's is sequence b
  auto weight_of = [](int tiles) { return tiles > 0 ? tiles + kSetup : 0; };
  // sequence i of the batch, the same for every lane
  auto seq_at = [&](int i) {
    Seq s = held;
    const ArgsPtr p = anew(args);
    if (p->B > 64) {
      s = seq_of<SEL>(p, i);
      i = 0;
    }
    s.len = __builtin_amdgcn_readlane(s.len, i);
    s.fresh = __builtin_amdgcn_readlane(s.fresh, i);
    s.tiles = __builtin_amdgcn_readlane(s.tiles, i);
    return s;
  };
  {
    const ArgsPtr p = anew(args);
    const int B = p->B, U = p->U, per = (B + 63) >> 6;
    int sum = 0, busy = 0;
    if (per == 1) {
      held = seq_from<SEL>(p, my_len, my_new);
      sum = weight_of(held.tiles);
      busy = held.tiles > 0;
    } else {
      for (int k = 0, i = lane * per; k < per && i < B; ++k, ++i) {
        const int t = seq_of<SEL>(p, i).tiles;
        sum += weight_of(t);
        busy += t > 0;
      }
    }
    if (p->split) {
      const int inc = wave_scan(sum);
      const int total = __builtin_amdgcn_readlane(inc, 63) * U;
      const int all = __builtin_amdgcn_readlane(wave_scan(busy), 63);
      idle = all < B;
      // as many shares as workgroups, but of kMinTiles at least, or a unit each
      int n = min(nwg, max(total / kMinTiles, all * U));
      // Two workgroups a CU, one setting up or joining while the other streams:
      // each with half of its stages, as what waits in the memory's queues
      // delays whatever a set-up needs (ragged fp16 batch 53.4 us with all, 48.7
      // with half).  Where units are long and few, nothing but the sweep counts:
      // one workgroup with all stages (bf16 [16,16/8,4096,128] 54.3 -> 52.0 us).
      if (n == p->full) {
        if (all * U < n / 2 && total / (n / 2) >= kLongShare) n /= 2;
        else depth = (NS + 1) / 2;
      }
      if (wg < n) {
        share = (int)(((uint32_t)total + (uint32_t)n - 1u) / (uint32_t)n);
        x = wg * share;
        hi = min(x + share, total);
        const uint64_t in = __builtin_amdgcn_ballot_w64((inc - sum) * U <= x && x < inc * U);
        if (x < hi) {
          const int at = (int)__builtin_ctzll(in);
          base = __builtin_amdgcn_readlane(inc - sum, at) * U;
          b = at * per;
        }
      }
    } else {
      x = wg;
      hi = B * U;
    }
  }

  auto weight = [](float m, float mx) { return m == -INFINITY ? 0.f : fast_exp2(m - mx); };

  while (x < hi) {
    // ---- the next segment: tiles [ta, tb) of unit (b, i), one of `parts`, the part-th
    Seq seq;
    int i, ta = 0, tb, parts = 1, part = 0, w0 = 0;
    const ArgsPtr p = anew(args);
    if (p->split) {
      const int U = p->U;
      seq = seq_at(b);
      int w = weight_of(seq.tiles);
      while (x >= base + w * U) {
        base += w * U;
        seq = seq_at(++b);
        w = weight_of(seq.tiles);
      }
      i = (int)((uint32_t)(x - base) / (uint32_t)w);
      const int u0 = base + i * w, u1 = u0 + w, x0 = x;
      x = u1;
      tb = seq.tiles;
      if (tb <= kWhole) {  // never split: its first workgroup's
        if (x0 > u0) continue;
      } else if (x0 > u0 || hi < u1) {
        // the workgroup that holds tile 0 has part 0
        ta = max(x0 - u0 - kSetup, 0);
        tb = min(min(hi, u1) - u0 - kSetup, tb);
        if (tb <= ta) continue;
        w0 = ta == 0 ? wg : (int)((uint32_t)(u0 + kSetup) / (uint32_t)share);
        part = wg - w0;
        parts = (tb == seq.tiles ? wg : (int)((uint32_t)(u1 - 1) / (uint32_t)share)) - w0 + 1;
      }
    } else {
      b = x / p->U;
      i = x - b * p->U;
      x += nwg;
      seq = seq_at(b);
      tb = seq.tiles;
      if (tb == 0) continue;
    }
    const int len = seq.len, fresh = seq.fresh, S = p->S;
    const int hk = quot(i, p->by_blocks.m, p->by_blocks.s);
    const int row0 = (i - hk * p->blocks) * kRows;
    const int R = min(kRows, p->rows - row0);
    const int head0 = hk * p->G;
    const int mine = tb - ta > wave ? (tb - ta - wave + NW - 1) / NW : 0;  // tiles of this wave

    // this unit's row r: query head head0 + h, column r - h S
    auto head_of = [&](int r, int& col) {
      const ArgsPtr p = anew(args);
      const int h = quot(row0 + r, p->by_s.m, p->by_s.s);
      col = row0 + r - h * p->S;
      return head0 + h;
    };
    // ---- what this wave's tiles [64 k, 64 k + 64) read, lane l's that of tile
    // 64 k + l: the page's address at the tile's first slot and the bytes from
    // there that hold keys (K and V), the position of the first key and the
    // tile's slots
    uint32_t ka[2], va[2];
    int kn = 0, vn = 0, pos0 = 0, slots0 = 0;
    bool bad = false;
    int page = -1, first = 0;  // between the two steps
    auto look_up = [&](int k) {
      const ArgsPtr p = anew(args);
      const int j = 64 * k + lane, t = ta + wave + NW * j;
      page = -1;
      pos0 = first = 0;
      if (j < mine) {
        const int e = quot(t, p->by_tpp.m, p->by_tpp.s);
        first = (t - e * p->tpp) * kTile;
        const int col = SEL ? p->selected[((int64_t)b * (p->U / p->blocks) + hk) * p->nsel + e] : e;
        pos0 = -1;
        if (col >= 0) {
          pos0 = (int64_t)col * p->ps < len ? col * p->ps + first : 0;
          if (!SEL || (int64_t)col * p->ps < len) page = p->table[b * p->t_str + col];
        }
      }
    };
    auto take = [&](int k) {
      const ArgsPtr p = anew(args);
      kn = vn = slots0 = 0;
      const bool wanted = 64 * k + lane < mine && pos0 >= 0;
      if (page < 0 || page >= p->num_pages) {
        bad |= wanted;
        page = -1;
      } else if (wanted) {
        slots0 = min(min(kTile, p->ps - first), max(len - pos0, 0));
      }
      pos0 = max(pos0, 0);
      const int ks_b = p->ks_b, vs_b = p->vs_b;
      if (slots0 > 0) {
        kn = (slots0 - 1) * ks_b + p->row_b;
        vn = (slots0 - 1) * vs_b + p->row_b;
      }
      const uint64_t kb = (uint64_t)(p->k + max(page, 0) * p->kp_p + hk * p->kp_h + (int64_t)first * ks_b);
      const uint64_t vb = (uint64_t)(p->v + max(page, 0) * p->vp_p + hk * p->vp_h + (int64_t)first * vs_b);
      ka[0] = (uint32_t)kb;
      ka[1] = (uint32_t)(kb >> 32) & 0xffffu;
      va[0] = (uint32_t)vb;
      va[1] = (uint32_t)(vb >> 32) & 0xffffu;
    };
    look_up(0);

    // row c sees the keys before `limit`; every row those before `sure`
    int limit = 0;
    const int sure = S == 1 ? len : 0;
    u32x4 qf[KS];
    {
      const ArgsPtr p = anew(args);
      int col;
      const int h = head_of(c, col);
      if (c < R && col < fresh) limit = len - fresh + col + 1;
      const char* qrow = (const char*)p->q + (b * p->q_b + (c < R ? h * p->q_h + col * p->q_s : 0)) * ES;
      const uint32_t sg = p->q_sign;
      const int end = c < R ? p->row_b : 0;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int at = 64 * ks + 16 * g;
        const u32x4 w = at < end ? *(const u32x4*)(qrow + at) : (u32x4){0u, 0u, 0u, 0u};
        qf[ks] = w ^ (u32x4){sg, sg, sg, sg};
      }
    }

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
    const float cmul = anew(args)->c;

    take(0);
    // (position, slots) of the tiles in flight: the lanes move on to the next 64
    // tiles when the first of those is issued, up to NS tiles ahead
    int pos_q[NS], slots_q[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      pos_q[j] = slots_q[j] = 0;
      if (j < mine && j < depth) {
        pos_q[j] = __builtin_amdgcn_readlane(pos0, j);
        slots_q[j] = __builtin_amdgcn_readlane(slots0, j);
        issue(j);
      }
    }

    for (int j = 0; j < mine; ++j) {
      const int behind = min(depth - 1, mine - 1 - j);
      if (NS > 3 && behind == 3) wait_vmcnt<(NS > 3 ? 3 * IPT : 0)>();
      else if (NS > 2 && behind == 2) wait_vmcnt<(NS > 2 ? 2 * IPT : 0)>();
      else if (NS > 1 && behind == 1) wait_vmcnt<(NS > 1 ? IPT : 0)>();
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
      const float mt = rows_max(fmaxf(fmaxf(xs[0], xs[1]), fmaxf(xs[2], xs[3])));
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
      const int ahead = j + depth;
      if (ahead < mine) {
        if ((ahead & 63) == 0) {
          look_up(ahead >> 6);
          take(ahead >> 6);
        }
#pragma unroll
        for (int q = 0; q < NS; ++q) {
          if (q == depth - 1) {
            pos_q[q] = __builtin_amdgcn_readlane(pos0, ahead & 63);
            slots_q[q] = __builtin_amdgcn_readlane(slots0, ahead & 63);
          }
        }
        // this stage's LDS reads have returned before its next tile's loads go out
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        issue(ahead);
      }
    }

    // ---- the waves' states meet in LDS: [wave][row][DK] O, then m, l
    float lrow = rows_sum(l_run);
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
    auto inverse = [](float l) { return l == 0.f ? 0.f : 1.f / l; };
    auto store_out = [&](int r, int k, f32x4 o, float inv) {
      const ArgsPtr p = anew(args);
      if (4 * k >= p->D) return;
      int col;
      const int h = head_of(r, col);
      T* const at = (T*)p->o + b * p->o_b + h * p->o_h + col * p->o_s + 4 * k;
      if constexpr (F32) {
        *(f32x4*)at = o * inv;
      } else {
        u32x2 w;
        w[0] = Mma<T>::pack(o[0] * inv, o[1] * inv);
        w[1] = Mma<T>::pack(o[2] * inv, o[3] * inv);
        *(u32x2*)at = w;
      }
    };
    const ArgsPtr pe_args = anew(args);
    const __amdgpu_buffer_rsrc_t wsr =
        uniform_rsrc(parts > 1 ? (const void*)pe_args->ws : (const void*)pe_args->o,
                     parts > 1 ? (int64_t)nwg * 2 * kRows * (DQ + 1) * 16 : 16);
    int* const cnt = pe_args->cnt;
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
        const int old = __hip_atomic_fetch_add(cnt + w0, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (old == parts - 1) __hip_atomic_store(cnt + w0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
      if (n <= kMergeLoads) {
        // few parts: every thread loads all of its vectors and their (m, l) at once
        for (int u = tid; u < nu; u += NT) {
          const int r = u / DQ, k = u - r * DQ;
          f32x4 e[kMergeLoads], v[kMergeLoads];
#pragma unroll
          for (int q = 0; q < kMergeLoads; ++q) {
            const int at = min(q, n - 1);
            e[q] = ld(slot(at, r, DQ));
            v[q] = ld(slot(at, r, k));
          }
          float mx = -INFINITY, L = 0.f;
#pragma unroll
          for (int q = 0; q < kMergeLoads; ++q) mx = fmaxf(mx, e[q][0]);
          f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < kMergeLoads; ++q) {
            const float f = q < n ? weight(e[q][0], mx) : 0.f;
            if (q < n) L = __builtin_fmaf(e[q][1], f, L);
            if (q < n) o += v[q] * f;
          }
          store_out(r, k, o, inverse(L));
        }
      } else {
      // rows at a time, so that their weights fit the ring's LDS whatever the parts
      const int rstep = min(R, max(1, (LDS - NT * 16 - 64) / (8 * n)));
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
    }
    lds_barrier();  // the LDS is free for the next segment
  }

  // ---- places nothing was read for: zeros, NaN where the sequence is longer than its table row
  const ArgsPtr p = anew(args);
  for (int bb = idle ? wg : p->B; bb < p->B; bb += nwg) {
    const Seq seq = seq_of<SEL>(p, bb);
    if (seq.tiles > 0) continue;
    const bool err = seq.len > p->cap && seq.fresh > 0;
    const uint32_t w = err ? (F32 ? 0x7fc00000u : 0x7fff7fffu) : 0u;
    const int nc = p->row_b / 16, n = p->U / p->blocks * p->rows * nc;
    for (int u = tid; u < n; u += NT) {
      const int r = u / nc, h = quot(r, p->by_s.m, p->by_s.s);
      *(u32x4*)((char*)p->o + (bb * p->o_b + h * p->o_h + (r - h * p->S) * p->o_s) * ES + 16 * (u - r * nc)) = (u32x4){w, w, w, w};
    }
  }
}

int bucket(int dtype, int D) {
  if (dtype == 2) return (D + 63) / 64 * 64;
  return D <= 64 ? 64 : D <= 160 ? (D + 31) / 32 * 32 : (D + 63) / 64 * 64;
}

// Workgroups that the CUs hold at once.
int full_house(int dtype, int D) {
  const int n = device_cus() * min(kPerCu, 160 * 1024 / (pg_lds(bucket(dtype, D), dtype == 2 ? 4 : 2) + 512));
  return n < kMaxWgs ? n : kMaxWgs;
}

// Workgroups of a launch: what the CUs hold at once, or fewer when the table
// rows do not hold that many shares of kMinTiles tiles.
int workgroups(int dtype, int B, int H, int Hkv, int S, int D, int page_size, int width, int n_selected) {
  const int n = full_house(dtype, D);
  const int64_t units = (int64_t)B * Hkv * ((H / Hkv * S + kRows - 1) / kRows);
  const int64_t cols = n_selected > 0 ? n_selected : width;
  const int64_t tiles = units * cols * ((page_size + kTile - 1) / kTile);
  const int64_t most = (tiles + kSetup * units) / kMinTiles > units ? (tiles + kSetup * units) / kMinTiles : units;
  return most < n ? (int)most : n;
}

template <typename T, int DK>
hipError_t launch_dk(const AttnArgs& a, int wgs, hipStream_t s) {
  const dim3 grid(wgs), block(pg_waves(DK * sizeof(T)) * 64);
  if (a.nsel > 0) hipLaunchKernelGGL((paged_attn<T, DK, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((paged_attn<T, DK, false>), grid, block, 0, s, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch16(const AttnArgs& a, int wgs, hipStream_t s) {
  switch (bucket(0, a.D)) {
    case 64: return launch_dk<T, 64>(a, wgs, s);
    case 96: return launch_dk<T, 96>(a, wgs, s);
    case 128: return launch_dk<T, 128>(a, wgs, s);
    case 160: return launch_dk<T, 160>(a, wgs, s);
    case 192: return launch_dk<T, 192>(a, wgs, s);
  }
  return launch_dk<T, 256>(a, wgs, s);
}

}  // namespace

size_t paged_attn_workspace(int dtype, int B, int H, int Hkv, int S, int D, int page_size, int width, int n_selected) {
  const int n = workgroups(dtype, B, H, Hkv, S, D, page_size, width, n_selected);
  // tiles are counted in 32 bits: a table for more is read in whole units
  const int64_t cols = n_selected > 0 ? n_selected : width;
  const int64_t units = (int64_t)B * Hkv * ((H / Hkv * S + kRows - 1) / kRows);
  if (n <= 1 || width == 0 || units * (cols * ((page_size + kTile - 1) / kTile) + kSetup) > INT32_MAX / 2) return 0;
  return kExchangeCounterBytes + (size_t)n * 2 * kRows * (bucket(dtype, D) / 4 + 1) * sizeof(f32x4);
}

hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, hipStream_t s) {
  const int ps = p.map.page_size;
  const size_t need = paged_attn_workspace(dtype, p.B, p.H, p.Hkv, p.S, p.D, ps, p.map.width, p.n_selected);
  int wgs = workgroups(dtype, p.B, p.H, p.Hkv, p.S, p.D, ps, p.map.width, p.n_selected);
  const int G = p.H / p.Hkv, blocks = (G * p.S + kRows - 1) / kRows, tpp = (ps + kTile - 1) / kTile;
  const int es = dtype == 2 ? 4 : 2;
  AttnArgs a;
  memset(&a, 0, sizeof a);
  a.lens = p.map.lens; a.news = p.map.new_lens; a.table = p.map.table; a.selected = p.selected;
  a.t_str = p.map.stride;
  a.B = p.B; a.S = p.S; a.U = p.Hkv * blocks; a.cap = p.map.width * ps;
  a.nsel = p.n_selected; a.width = p.map.width; a.ps = ps; a.tpp = tpp;
  a.by_ps = div_by(ps); a.by_tpp = div_by(tpp); a.by_blocks = div_by(blocks); a.by_s = div_by(p.S);
  a.exact = ps % kTile == 0;
  a.full = full_house(dtype, p.D);
  a.G = G; a.blocks = blocks; a.rows = G * p.S; a.num_pages = p.map.num_pages;
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
  if (dtype == 0) return launch16<_Float16>(a, wgs, s);
  if (dtype == 1) return launch16<__bf16>(a, wgs, s);
  switch (bucket(2, p.D)) {
    case 64: return launch_dk<float, 64>(a, wgs, s);
    case 128: return launch_dk<float, 128>(a, wgs, s);
    case 192: return launch_dk<float, 192>(a, wgs, s);
  }
  return launch_dk<float, 256>(a, wgs, s);
}

}  // namespace cmpext3
