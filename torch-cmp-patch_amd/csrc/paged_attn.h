// Attention of new tokens over a paged key-value cache: a few query rows per
// K/V head, a long sweep over keys that lie in pages.
//
// Such a launch moves almost nothing but K and V and is bound by the bytes it
// keeps in flight from HBM (measured on MI355X: bf16 [16,16/8,1,4096,128] 51.8
// us, 5.2 TB/s; [1,16/8,1,131072,256] 189 us, 5.7 TB/s), small ones by the
// latency of their dependent loads (bf16 [1,16/8,1,300,128] 8.4 us).  Nothing on
// the host knows the sequences' lengths, so the work is dealt out on the device:
//
//  * A unit is a (sequence, K/V head, up to 64 query rows); its keys are cut
//    into tiles of 16 slots, none across a page.  All units' tiles in a row are
//    one sequence of work, of which every workgroup takes an equal, contiguous
//    share (every wave sums over the batch first), so ragged batches load the
//    chip evenly and a single long sequence spreads over all of it.  Short
//    units stay whole; where shares are short, units are cut one by one.
//  * A workgroup's share is a list of segments, each within one unit.  Its four
//    waves take a segment's tiles in turn; every wave streams its own tiles
//    through a ring of stages in LDS filled by buffer_load ... lds (no staging
//    registers, no barriers), one buffer descriptor per tile: the page's
//    address is in its base, 48 bits wide, and its last valid slot is its end,
//    so slots behind the sequence read as zeros whatever they hold.
//  * A lane makes the descriptors of one of the wave's next 64 tiles (one load
//    of the table per 64 tiles, checked there), read back by v_readlane.
//  * Scores S^T = K Q^T and O^T = V^T P^T on 16x16 MFMAs (16x16x32 and 16x16x16
//    for fp16 and bf16, 16x16x4 for fp32), exact online softmax in the exp2
//    domain with fp32 state (scaled and set off against the maximum in one fma,
//    so that only the rounding of the common maximum stays, and cancels).  For
//    fp16 and bf16 a weight enters the second product in two parts, its value
//    rounded to the tensors' type and the rounded rest (the matrix units are
//    idle for most of the time anyway), whose product with an infinity is no
//    number: then the wave sweeps once more.
//  * End of a segment: the waves' (O, m, l) meet in LDS.  A unit that is one
//    segment is written out; otherwise each of its workgroups leaves its part
//    in the workspace and counts itself in, and the last of every eight
//    neighbours joins them, and so on up.  Nobody waits for another workgroup.
#pragma once

#include "paged_common.h"

namespace cmpext3 {

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

constexpr int kRows = 16;        // query rows of a block
constexpr int kTile = 16;        // slots of a tile
constexpr int kMaxWgs = 1024;    // workgroups of a launch at most (counters: one each)
constexpr int kSetup = 6;        // what a unit costs beside its tiles, in tiles
constexpr int kShortCut = 40;    // tiles of a part up to which units are cut by themselves
constexpr int kLongShare = 48;   // tiles of a share from which one workgroup a CU is enough
constexpr int kJoin = 8;         // parts joined at once

// Waves per workgroup, workgroups per CU at most, and stages per wave: as many as
// 64 KB of LDS hold, from one to four, so that two workgroups fit a CU (one where
// a stage of fp32 above D = 128 takes more).  More in flight is no faster (bf16
// [16,16/8,4096,128]: 54.3 us with 128 KB a CU, 52.0 with 64); two workgroups of
// two waves are slower than one of four (fp32 [33,40/10,3,1000,192] 121.6 us, 88.5).
constexpr int kWaves = 4;
constexpr int kPerCu = 2;
constexpr int pg_stages(int rb) {
  const int n = 64 * 1024 / (kWaves * 2 * kTile * rb);
  return n < 1 ? 1 : n < 4 ? n : 4;
}
// LDS of a workgroup: the rings, later the waves' states in the same place
constexpr int pg_lds(int dk, int es) {
  const int nw = kWaves, ring = nw * pg_stages(dk * es) * 2 * kTile * dk * es;
  const int states = nw * kRows * (dk + 6) * 4;
  return ring > states ? ring : states;
}

// Tiles of a workgroup's share at least: four a wave (two in fp32, whose products
// take longer).
constexpr int pg_min_tiles(int es) { return kWaves * (es == 4 ? 2 : 4); }

// Blocks of 16 query rows that a unit takes together, each K and V fragment read
// once for all of them: as many as the rows fill and half of the registers hold
// (two workgroups a CU).  bf16 [4,32/1,1,16384,128] 36.5 us with one, 26.6 with
// two; [7,40/5,8,8k..16k,128] 143 with one, 84.9 with two, 92.7 with four and one
// workgroup a CU.
constexpr int pg_row_blocks(int rb, int rows) {
  const int most = rb <= 128 ? 4 : rb <= 256 ? 2 : 1;
  const int n = rows <= kRows ? 1 : rows <= 2 * kRows ? 2 : 4;
  return n < most ? n : most;
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

template <bool V> struct Const {
  static constexpr bool value = V;
};

struct AttnArgs {
  const int32_t *lens, *news, *table, *selected;
  int64_t t_str;
  int B, S, U, cap;        // U: units of a sequence; cap: keys a table row holds
  int nsel, width, ps, tpp;  // tpp: tiles per page
  Div by_ps, by_tpp, by_blocks, by_s;
  int split, exact, full;  // split 0: whole units, dealt out in turn; exact: pages are whole tiles; full: workgroups the CUs hold, two each (0: one each)
  int G, blocks, rows, num_pages;  // query heads per K/V head, units and rows of a K/V head
  int slot_rows;                   // rows of a part in the workspace
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

template <typename T, int DK, int NR, bool SEL>
__global__ __launch_bounds__(kWaves * 64, pg_lds(DK, sizeof(T)) > 80 * 1024 ? 1 : 2) void paged_attn(AttnArgs) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int ES = sizeof(T);
  constexpr int RB = DK * ES;           // bytes of a K/V row in LDS
  constexpr int NW = kWaves, NS = pg_stages(RB), NT = NW * 64;
  constexpr int NC = RB / 16;           // 16-byte chunks per row
  constexpr int BLK = kTile * RB;
  constexpr int IB = BLK / 1024;        // DMA instructions per 16 rows
  constexpr int STAGE = 2 * BLK;
  constexpr int IPT = 2 * IB;
  constexpr int KS = NC / 4;            // 16-byte chunks of a score operand per lane
  constexpr int NDB = DK / 16;          // float4 accumulators of a lane
  constexpr int DQ = DK / 4;            // float4 vectors of an output row
  constexpr int MOS = DK + 4;           // row stride (floats) of the waves' states
  constexpr int ROWS = NR * kRows;      // query rows of a unit at most
  // tiles of a unit that is never split: a join costs about that many (fp32
  // products take longer).  bf16 [1,16/8,1,300,128] 7.7 us whole, 10.7 in parts;
  // fp32 [2,20/5,2,500,128] 18.7 us with 32 here, 12.2 with 16.
  constexpr int kWhole = F32 ? 16 : 32;
  constexpr int kMinTiles = pg_min_tiles(ES);
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
  int cut = 0;          // > 0: units are cut by themselves
  auto weight_of = [](int tiles) { return tiles > 0 ? tiles + kSetup : 0; };
  auto parts_of = [&](int tiles, int cut) {
    if (tiles <= kWhole) return tiles == 0 ? 0 : 1;
    const int n = (int)((uint32_t)(weight_of(tiles) + cut - 1) / (uint32_t)cut);
    return n > kJoin && n <= kJoin + kJoin / 2 ? kJoin : n;  // a little longer sweeps for a level of the join
  };
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
      const int units = all * U;
      int n = min(nwg, max(total / kMinTiles, units));
      // Two workgroups a CU, one setting up or joining while the other streams:
      // each with half of its stages, as what waits in the memory's queues
      // delays whatever a set-up needs (ragged fp16 batch 53.4 us with all, 48.7
      // with half).  Where units are long and few, nothing but the sweep counts:
      // one workgroup with all stages (bf16 [16,16/8,4096,128] 54.3 -> 52.0 us).
      const bool alone = n == p->full && units < n / 2 && total / (n / 2) >= kLongShare;
      if (alone) n /= 2;
      // Short shares: a second segment costs as much as the share itself.  Every
      // unit is cut by itself, into parts of `cut` at most, a workgroup each.
      if (per == 1 && !alone && units < nwg) {
        cut = max(kMinTiles, (int)((uint32_t)total / (uint32_t)(nwg - units)) + 1);
        if (cut > kShortCut) cut = 0;
      }
      if (cut > 0) {
        const int own = parts_of(held.tiles, cut), upto = wave_scan(own);
        const int last = __builtin_amdgcn_readlane(upto, 63) * U;
        if (p->full > 0 && 2 * last > p->full) depth = (NS + 1) / 2;
        if (wg < last) {
          x = wg;
          hi = wg + 1;
          const int at = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64((upto - own) * U <= x && x < upto * U));
          base = __builtin_amdgcn_readlane(upto - own, at) * U;
          b = at;
        }
      } else if (wg < n) {
        if (n == p->full) depth = (NS + 1) / 2;
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
    if (cut > 0) {
      seq = seq_at(b);
      parts = parts_of(seq.tiles, cut);
      i = (int)((uint32_t)(x - base) / (uint32_t)parts);
      part = x - base - i * parts;
      w0 = wg - part;
      ta = (int)((uint32_t)(part * seq.tiles) / (uint32_t)parts);
      tb = (int)((uint32_t)((part + 1) * seq.tiles) / (uint32_t)parts);
      x = hi;
    } else if (p->split) {
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
    const int row0 = (i - hk * p->blocks) * ROWS;
    const int R = min(ROWS, p->rows - row0);
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

    // row 16 z + c sees the keys before `limit[z]`; every row those before `sure`
    int limit[NR];
    const int sure = S == 1 ? len : 0;
    u32x4 qf[NR][KS];
    {
      const ArgsPtr p = anew(args);
      const uint32_t sg = p->q_sign;
#pragma unroll
      for (int z = 0; z < NR; ++z) {
        const int r = 16 * z + c;
        int col;
        const int h = head_of(r, col);
        limit[z] = r < R && col < fresh ? len - fresh + col + 1 : 0;
        const char* qrow = (const char*)p->q + (b * p->q_b + (r < R ? h * p->q_h + col * p->q_s : 0)) * ES;
        const int end = r < R ? p->row_b : 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int at = 64 * ks + 16 * g;
          const u32x4 w = at < end ? *(const u32x4*)(qrow + at) : (u32x4){0u, 0u, 0u, 0u};
          qf[z][ks] = w ^ (u32x4){sg, sg, sg, sg};
        }
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

    f32x4 oacc[NR][NDB];
    float m_run[NR], l_run[NR];
    const float cmul = anew(args)->c;

    // A sum that is no number: an infinity in V met the rest of its weight's
    // rounding, or a value that some rows do not see met their weight of 0.  The
    // wave sweeps its tiles once more, carefully.
    auto sweep = [&](auto kind) {
      constexpr bool careful = decltype(kind)::value;
#pragma unroll
      for (int z = 0; z < NR; ++z) {
        m_run[z] = -INFINITY;
        l_run[z] = 0.f;
#pragma unroll
        for (int db = 0; db < NDB; ++db) oacc[z][db] = (f32x4){0.f, 0.f, 0.f, 0.f};
      }
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

        // fp32: four sums of every fourth product (shorter chains: sums closer to the
        // exact ones, and no product waits for the last)
        f32x4 s[NR], more[NR][3];
#pragma unroll
        for (int z = 0; z < NR; ++z) s[z] = more[z][0] = more[z][1] = more[z][2] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4 kk = *(const u32x4*)(st + kro[ks]);
#pragma unroll
          for (int z = 0; z < NR; ++z) {
            if constexpr (F32) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                f32x4& sum = e == 0 ? s[z] : more[z][e - 1];
                sum = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kk[e]), __uint_as_float(qf[z][ks][e]), sum, 0, 0, 0);
              }
            } else {
              s[z] = Mma<T>::qk(kk, qf[z][ks], s[z]);
            }
          }
        }
        float pe[NR][4];
        u32x2 pb[NR], pl[NR];  // fp16, bf16: rounded weights, and what the rounding left
#pragma unroll
        for (int z = 0; z < NR; ++z) {
          if constexpr (F32) s[z] = (s[z] + more[z][0]) + (more[z][1] + more[z][2]);
          float xs[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) xs[e] = s[z][e];
          if (slots < kTile || pos + kTile > sure) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (4 * g + e >= slots || pos + 4 * g + e >= limit[z]) xs[e] = -INFINITY;
          }
          const float mt = cmul * rows_max(fmaxf(fmaxf(xs[0], xs[1]), fmaxf(xs[2], xs[3])));
          if (__builtin_amdgcn_ballot_w64(mt > m_run[z])) {  // some row's maximum rises
            const float m_new = fmaxf(m_run[z], mt);
            const float alpha = weight(m_run[z], m_new);
            m_run[z] = m_new;
            l_run[z] *= alpha;
#pragma unroll
            for (int db = 0; db < NDB; ++db) oacc[z][db] *= alpha;
          }
          const float m_sub = m_run[z] == -INFINITY ? 0.f : m_run[z];
#pragma unroll
          for (int e = 0; e < 4; ++e) pe[z][e] = fast_exp2(__builtin_fmaf(xs[e], cmul, -m_sub));
          l_run[z] += (pe[z][0] + pe[z][1]) + (pe[z][2] + pe[z][3]);
          if constexpr (!F32) {
            pb[z][0] = Mma<T>::pack(pe[z][0], pe[z][1]);
            pb[z][1] = Mma<T>::pack(pe[z][2], pe[z][3]);
            pl[z][0] = Mma<T>::rest(pb[z][0], pe[z][0], pe[z][1]);
            pl[z][1] = Mma<T>::rest(pb[z][1], pe[z][2], pe[z][3]);
          }
        }
        const unsigned char* vs = st + BLK;
        if constexpr (careful) {
          // rows of one limit at a time, the values behind it blanked
          const bool cut_off = S > 1 && pos + kTile > len - fresh + 1;
          for (int i = cut_off ? 0 : fresh - 1; i < fresh; ++i) {
            const int upto = cut_off ? len - fresh + 1 + i : INT32_MAX;
#pragma unroll
            for (int z = 0; z < NR; ++z) {
              const bool these = !cut_off || limit[z] == upto;
              if constexpr (F32) {
#pragma unroll
                for (int db = 0; db < NDB; db += 4) {
                  f32x4 t[4] = {};
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int r = 4 * g + e;
                    const u32x4 v = *(const u32x4*)(vs + r * RB + 16 * pg_swz(r, 4 * db + c, NC));
                    const bool in = pos + r < upto;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                      t[q] = __builtin_amdgcn_mfma_f32_16x16x4f32(in ? __uint_as_float(v[q]) : 0.f, pe[z][e], t[q], 0, 0, 0);
                  }
#pragma unroll
                  for (int q = 0; q < 4; ++q)
                    if (these) oacc[z][db + q] += t[q];
                  __builtin_amdgcn_sched_barrier(0);
                }
              } else {
                const int r = 4 * g + (c >> 2), ch = (c & 3) >> 1, left = upto - pos - 4 * g;
                const uint32_t m0 = (left > 0 ? 0xffffu : 0u) | (left > 1 ? 0xffff0000u : 0u);
                const uint32_t m1 = (left > 2 ? 0xffffu : 0u) | (left > 3 ? 0xffff0000u : 0u);
#pragma unroll
                for (int db = 0; db < NDB; ++db) {
                  typedef __attribute__((address_space(3))) i16x4p lds_i16x4;
                  const unsigned char* at = vs + r * RB + 16 * pg_swz(r, 2 * db + ch, NC) + 8 * (c & 1);
                  const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at)) & (u32x2){m0, m1};
                  const f32x4 t = Mma<T>::pv(v, pb[z], (f32x4){0.f, 0.f, 0.f, 0.f});
                  if (these) oacc[z][db] += t;
                  __builtin_amdgcn_sched_barrier(0);  // one at a time: few registers
                }
              }
            }
          }
        } else if constexpr (F32) {
          // 64 columns at a time: MFMA j takes columns 4 m + j (a lane's 16-byte
          // read is one slot's chunk, an element for each of the four)
#pragma unroll
          for (int db = 0; db < NDB; db += 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 4 * g + e;
              const u32x4 v = *(const u32x4*)(vs + r * RB + 16 * pg_swz(r, 4 * db + c, NC));
#pragma unroll
              for (int z = 0; z < NR; ++z)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  oacc[z][db + q] =
                      __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[q]), pe[z][e], oacc[z][db + q], 0, 0, 0);
            }
          }
        } else {
          // 16 lanes of group g read slots 4g .. 4g+3 x 16 columns, transposed:
          // lane c receives column 16 db + c of the four
          const int r = 4 * g + (c >> 2), ch = (c & 3) >> 1;
#pragma unroll
          for (int db = 0; db < NDB; ++db) {
            typedef __attribute__((address_space(3))) i16x4p lds_i16x4;
            const unsigned char* at = vs + r * RB + 16 * pg_swz(r, 2 * db + ch, NC) + 8 * (c & 1);
            const i16x4p v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at);
#pragma unroll
            for (int z = 0; z < NR; ++z) {
              oacc[z][db] = Mma<T>::pv(__builtin_bit_cast(u32x2, v), pb[z], oacc[z][db]);
              oacc[z][db] = Mma<T>::pv(__builtin_bit_cast(u32x2, v), pl[z], oacc[z][db]);
            }
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
    };
    sweep(Const<false>());
    float test = 0.f;
#pragma unroll
    for (int z = 0; z < NR; ++z)
#pragma unroll
      for (int db = 0; db < NDB; ++db) test += (oacc[z][db][0] + oacc[z][db][1]) + (oacc[z][db][2] + oacc[z][db][3]);
    if (__builtin_amdgcn_ballot_w64(test != test)) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's last LDS reads
      look_up(0);
      sweep(Const<true>());
    }

    // ---- end of the segment: outputs, or the workgroup's part of them
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
                     parts > 1 ? (int64_t)nwg * 2 * pe_args->slot_rows * (DQ + 1) * 16 : 16);
    int* const cnt = pe_args->cnt;
    const int slot_rows = pe_args->slot_rows;
    // slot of part q's row r: a part that begins the unit is its workgroup's
    // last segment, the others are their workgroups' first.  Device-scope (aux
    // 16 = sc1) accesses, coherent across the XCDs' L2s.
    auto slot = [&](int q, int r, int k) { return ((((w0 + q) * 2 + (q == 0 ? 1 : 0)) * slot_rows + r) * (DQ + 1) + k) * 16; };
    auto ld = [&](int off) { return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(wsr, off, 0, 16)); };
    auto st = [&](int off, f32x4 v) { __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), wsr, off, 0, 16); };
    const bool lost = __builtin_amdgcn_ballot_w64(bad) != 0;  // a page that is none: the unit's rows are NaN
    wait_vmcnt<0>();
    lds_barrier();  // every wave is done with its ring
    // the waves' states meet in LDS, 16 rows at a time: [wave][row][DK] O, then m, l
#pragma unroll
    for (int z = 0; z < NR; ++z) {
      if (16 * z >= R) break;
      if (z > 0) lds_barrier();  // the last rows have been read
      const float lrow = lost ? __builtin_nanf("") : rows_sum(l_run[z]);
      if (limit[z] <= 0) {  // sees nothing, whatever V holds
#pragma unroll
        for (int db = 0; db < NDB; ++db) oacc[z][db] = (f32x4){0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        // fp32: accumulators 4 k .. 4 k + 3 hold columns 64 k + 16 g + 4 e + (0 .. 3)
        if constexpr (F32) {
          const int k4 = db & ~3, e = db & 3;
          *(f32x4*)(mo + (wave * kRows + c) * MOS + 16 * k4 + 16 * g + 4 * e) =
              (f32x4){oacc[z][k4][e], oacc[z][k4 + 1][e], oacc[z][k4 + 2][e], oacc[z][k4 + 3][e]};
        } else {
          *(f32x4*)(mo + (wave * kRows + c) * MOS + 16 * db + 4 * g) = oacc[z][db];
        }
      }
      if (g == 0) {
        mm[wave * kRows + c] = m_run[z];
        ml[wave * kRows + c] = lrow;
      }
      lds_barrier();
      for (int u = tid; u < min(kRows, R - 16 * z) * DQ; u += NT) {
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
          store_out(16 * z + r, k, o, inverse(l));
        } else {
          st(slot(part, 16 * z + r, k), o);
          if (k == 0) st(slot(part, 16 * z + r, DQ), (f32x4){mx, l, 0.f, 0.f});
        }
      }
    }

    // ---- join the unit's parts as a tree: the last of every eight neighbours to
    // arrive joins them, all its loads in one round, and stands for them among
    // the next eight; the last of all writes the output.  Which parts join, and
    // in which order they are summed, does not hang on who arrives last.
    int at = part, n = parts, stride = 1;
    for (int level = 0; n > 1; ++level) {
      const int first = at & -kJoin, members = min(kJoin, n - first);
      const bool all = n <= kJoin;
      if (members > 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();  // every wave's stores are done
        if (tid == 0) {
          // (a counter's workgroup is not the unit's last, which may begin the next unit)
          int* const ctr = cnt + level * kMaxWgs + w0 + first * stride;
          const int old = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          if (old == members - 1) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          s_flag = old == members - 1;
        }
        lds_barrier();
        if (!__builtin_amdgcn_readfirstlane(s_flag)) break;
        asm volatile("" ::: "memory");  // the loads of the parts stay after the count
        float* const sums = (float*)lds;  // [row] (m, l)
        for (int u = tid; u < R * DQ; u += NT) {
          const int r = u / DQ, k = u - r * DQ;
          f32x4 e[kJoin], v[kJoin];
#pragma unroll
          for (int q = 0; q < kJoin; ++q) {
            const int of = (first + min(q, members - 1)) * stride;
            e[q] = ld(slot(of, r, DQ));
            v[q] = ld(slot(of, r, k));
          }
          float mx = -INFINITY, l = 0.f;
#pragma unroll
          for (int q = 0; q < kJoin; ++q) mx = fmaxf(mx, e[q][0]);
          f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < kJoin; ++q) {
            if (q < members) {
              const float f = weight(e[q][0], mx);
              l = __builtin_fmaf(e[q][1], f, l);
              o += v[q] * f;
            }
          }
          if (all) {
            store_out(r, k, o, inverse(l));
          } else {
            st(slot(first * stride, r, k), o);
            if (k == 0) {
              sums[2 * r] = mx;
              sums[2 * r + 1] = l;
            }
          }
        }
        if (all) break;
        lds_barrier();  // every row's (m, l) of the parts have been read
        for (int r = tid; r < R; r += NT) st(slot(first * stride, r, DQ), (f32x4){sums[2 * r], sums[2 * r + 1], 0.f, 0.f});
      }
      at /= kJoin;
      n = (n + kJoin - 1) / kJoin;
      stride *= kJoin;
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

template <typename T, int DK, int NR>
hipError_t launch_nr(const AttnArgs& a, int wgs, hipStream_t s) {
  const dim3 grid(wgs), block(kWaves * 64);
  if (a.nsel > 0) hipLaunchKernelGGL((paged_attn<T, DK, NR, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((paged_attn<T, DK, NR, false>), grid, block, 0, s, a);
  return hipGetLastError();
}

template <typename T, int DK>
hipError_t launch_dk(const AttnArgs& a, int wgs, hipStream_t s) {
  const int nr = pg_row_blocks(DK * sizeof(T), a.rows);
  if constexpr (pg_row_blocks(DK * sizeof(T), 64) >= 4) {
    if (nr == 4) return launch_nr<T, DK, 4>(a, wgs, s);
  }
  if constexpr (pg_row_blocks(DK * sizeof(T), 64) >= 2) {
    if (nr == 2) return launch_nr<T, DK, 2>(a, wgs, s);
  }
  return launch_nr<T, DK, 1>(a, wgs, s);
}

// Head dim buckets: 64, 96, 128, 160, 192, 256; fp32: 64, 128, 192, 256.
template <typename T>
hipError_t launch_type(const AttnArgs& a, int wgs, hipStream_t s) {
  if (a.D <= 64) return launch_dk<T, 64>(a, wgs, s);
  if constexpr (sizeof(T) == 2) {
    if (a.D <= 96) return launch_dk<T, 96>(a, wgs, s);
    if (a.D <= 128) return launch_dk<T, 128>(a, wgs, s);
    if (a.D <= 160) return launch_dk<T, 160>(a, wgs, s);
  }
  if (a.D <= 128) return launch_dk<T, 128>(a, wgs, s);
  if (a.D <= 192) return launch_dk<T, 192>(a, wgs, s);
  return launch_dk<T, 256>(a, wgs, s);
}

}  // namespace cmpext3
