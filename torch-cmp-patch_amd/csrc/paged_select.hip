// The pages of each sequence that its new token attends to.
//
// A page's score for a K/V head bounds the products of its keys with the
// head's queries: sum over queries h and channels d of max(q lo, q hi), which
// is sum over d of Q+ hi + Q- lo with Q+ (Q-) the sum of the queries' positive
// (negative) parts.  All of it in 64 bits: products of the inputs are exact
// there, and a page near the border falls on the same side whatever the order
// of the sums.  The scores are written as integers of the same order.
//
// paged_scores reads every page's bounds once and is bound by that: 8 to 64
// lanes take a page (a 16-byte chunk of lo and of hi each, its Q+ and Q- in
// registers), four steps of pages in flight (measured on MI355X: 8 heads x 8192
// pages of 128 fp16 channels 10.2 us, 3.3 TB/s; with the choice 19.5 us, and 20.1
// before it got faster, against 22.6 with two steps in flight and 20.1 with eight).
//
// paged_best takes the best of each (sequence, head) with one workgroup, whose
// waves hold a range of columns each.  The border is found by histograms of 2048
// bins: first 256 an octave around one of the scores, then, while more than 64
// scores share the border's bin, the range of those in equal parts; 64 or fewer
// are ranked by comparing all with all.  Which columns are taken is then a
// ballot per 64 columns, so they are written in ascending order, equal scores
// from the lowest column on.  7.5 us for 8 rows of 8192 (latency: barriers and
// LDS atomics of one workgroup a row).
//
// paged_short does both for rows of up to 1024 pages, a workgroup a row: 9.5 us
// for 16 x 8 rows of 256 pages (10.0 with the call's own; 12.2 in two launches).
#include "paged_common.h"

namespace cmpext3 {

namespace {

constexpr uint64_t kBest = ~0ull;
constexpr int kSteps = 4;     // steps of pages of a wave, all in flight together
constexpr int kBins = 2048;
constexpr int kShort = 1024;  // pages of a row that one launch scores and chooses

// Order of doubles as order of unsigned integers; NaN above everything.
__device__ __forceinline__ uint64_t order_of(double x) {
  if (x != x) return kBest;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// Pages of sequence b that its table row holds.
__device__ __forceinline__ int pages_of(const SelectParams& p, int b) {
  return min(quot(seq_len_held(p.map, b) + p.map.page_size - 1, p.by_ps.m, p.by_ps.s), p.map.width);
}

// Element e of a 16-byte chunk.
template <typename T>
__device__ __forceinline__ float elem(const u32x4& w, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
  else if constexpr (__is_same(T, __bf16)) return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e >> 1] >> (16 * (e & 1))));
}

template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
// Sum over groups of LG lanes (8, 16, 32 or 64), in every lane.
template <int LG>
__device__ __forceinline__ double group_sum(double x) {
  x += dpp<0xb1>(x);   // lanes 1 apart
  x += dpp<0x4e>(x);   // 2 apart
  x += dpp<0x141>(x);  // the other four of eight (mirrored)
  if (LG >= 16) x += dpp<0x140>(x);  // the other eight of sixteen
  if (LG >= 32) x += __shfl_xor(x, 16);
  if (LG >= 64) x += __shfl_xor(x, 32);
  return x;
}

// Q+ and Q- of a K/V head in the 16-byte chunk c.
template <typename T>
struct Weights {
  static constexpr int N = 16 / sizeof(T);  // elements of a chunk
  double up[N], down[N];
  int c;
  bool on;
  __device__ __forceinline__ void load(const SelectParams& p, int b, int hk, int chunk) {
    const int G = p.H / p.Hkv;
    c = chunk;
    on = c * N < p.D;
#pragma unroll
    for (int e = 0; e < N; ++e) up[e] = down[e] = 0;
    if (!on) return;
    const T* q = (const T*)p.q + b * p.q_b + hk * G * p.q_h + c * N;
    for (int g = 0; g < G; ++g) {
      const u32x4 w = *(const u32x4*)(q + g * p.q_h);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float x = elem<T>(w, e);
        down[e] += x < 0.f ? (double)x : 0.0;
        up[e] += x < 0.f ? 0.0 : (double)x;  // and a NaN
      }
    }
  }
};

// The bounds of kSteps steps of 64 / LG pages from this lane's column col0 on: the
// page numbers are on their way before the sequence's length is known, the
// bounds while the weights are made.
template <typename T, int LG>
struct Bounds {
  int page[kSteps];
  u32x4 lo[kSteps], hi[kSteps];
  __device__ __forceinline__ void look(const SelectParams& p, int b, int col0) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) page[s] = page_at(p.map, b, col0 + s * (64 / LG));
  }
  __device__ __forceinline__ void load(const SelectParams& p, int hk, int col0, int pages, int c) {
    constexpr int N = 16 / sizeof(T), PW = 64 / LG;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if (col0 + s * PW >= pages) page[s] = -1;
      lo[s] = hi[s] = (u32x4){0u, 0u, 0u, 0u};
      if (c * N < p.D && page[s] >= 0) {
        const T* at = (const T*)p.bounds + page[s] * p.kb_p + hk * p.kb_h + c * N;
        lo[s] = *(const u32x4*)at;
        hi[s] = *(const u32x4*)(at + p.kb_e);
      }
    }
  }
};

// put(column, key) of those pages.
template <typename T, int LG, typename Put>
__device__ __forceinline__ void score_pages(const Bounds<T, LG>& read, const Weights<T>& w, int col0, int pages, Put put) {
  constexpr int N = Weights<T>::N, PW = 64 / LG;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    double sum = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      sum = __builtin_fma(w.up[e], (double)elem<T>(read.hi[s], e), sum);
      sum = __builtin_fma(w.down[e], (double)elem<T>(read.lo[s], e), sum);
    }
    sum = group_sum<LG>(sum);
    if (__builtin_amdgcn_ballot_w64(sum != sum)) {
      // a zero part may have met an infinite bound: without the zero parts
      double t = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (w.up[e] != 0) t = __builtin_fma(w.up[e], (double)elem<T>(read.hi[s], e), t);
        if (w.down[e] != 0) t = __builtin_fma(w.down[e], (double)elem<T>(read.lo[s], e), t);
      }
      t = group_sum<LG>(t);
      if (sum != sum) sum = t;
    }
    const int col = col0 + s * PW;
    if (w.c == 0 && col < pages) put(col, read.page[s] >= 0 ? order_of(sum) : kBest);
  }
}

template <typename T, int LG>
__global__ __launch_bounds__(256) void paged_scores(SelectParams p, uint64_t* keys) {
  constexpr int PW = 64 / LG;        // pages of a wave's step
  const int hk = block_y(), b = block_z();
  const int lane = thread_x() & 63, wave = thread_x() >> 6;
  const int col0 = (block_x() * 4 + wave) * kSteps * PW + lane / LG;
  Bounds<T, LG> e;
  e.look(p, b, col0);
  const int pages = pages_of(p, b);
  if (block_x() * 4 * kSteps * PW >= pages) return;
  e.load(p, hk, col0, pages, lane & (LG - 1));
  Weights<T> w;
  w.load(p, b, hk, lane & (LG - 1));
  uint64_t* row = keys + ((int64_t)b * p.Hkv + hk) * p.map.width;
  score_pages<T, LG>(e, w, col0, pages, [&](int c, uint64_t k) { row[c] = k; });
}

__device__ __forceinline__ uint64_t wave_min(uint64_t x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)x, m);
    x = o < x ? o : x;
  }
  return x;
}

// Sum of the waves' numbers before this wave's.
template <int NW>
__device__ __forceinline__ int before_wave(const int* sums, int lane, int wave) {
  const int v = lane < NW ? sums[lane] : 0;
  return __builtin_amdgcn_readlane(wave_scan(v) - v, __builtin_amdgcn_readfirstlane(wave));
}

struct BestShared {
  int hist[kBins];
  uint64_t mn[16], mx[16], cand[64], key;
  int cand_col[64], sum[16], pick[3], cands, col;
};

// The K best columns of a row of `pages` scores, load(column) each, with NW
// waves that take a contiguous range of columns each, in steps of 64.  HELD:
// the steps' keys stay in registers, else every round loads them again.
template <int NW, int HELD, typename Load>
__device__ __forceinline__ void best(BestShared& sh, int pages, int K, int32_t* out, Load load) {
  const int tid = thread_x(), lane = tid & 63, wave = tid >> 6;
  for (int j = min(pages, K) + tid; j < K; j += NW * 64) out[j] = -1;
  if (pages <= K) {
    for (int j = tid; j < pages; j += NW * 64) out[j] = j;
    return;
  }
  const int m = pages - 1;  // the last page is in; the K - 1 best of m others
  if (tid == 0) out[K - 1] = m;
  if (K == 1) return;
  const int steps = (m + NW * 64 - 1) / (NW * 64);
  const int first = wave * steps * 64 + lane;
  uint64_t held[HELD > 0 ? HELD : 1];
  if constexpr (HELD > 0) {
#pragma unroll
    for (int s = 0; s < HELD; ++s) {
      const int c = first + 64 * s;
      held[s] = s < steps && c < m ? load(c) : 0;  // 0: below every key
    }
  }
  const uint64_t ref = load(0);
  // f(key, column) for this lane's columns
  auto each = [&](auto f) {
    if constexpr (HELD > 0) {
#pragma unroll
      for (int s = 0; s < HELD; ++s)
        if (s < steps) f(held[s], first + 64 * s);
    } else {
      for (int s = 0; s < steps; ++s) f(first + 64 * s < m ? load(first + 64 * s) : 0, first + 64 * s);
    }
  };

  // Taken are the keys above `key`, and those equal to it up to column `col`.
  // The border lies among the keys in [lo, hi], of which `need` are taken.
  uint64_t lo = 1, hi = kBest, key;
  int need = K - 1, col = INT32_MAX;
  for (int round = 0;; ++round) {
    for (int j = tid; j < kBins; j += NW * 64) sh.hist[j] = 0;
    int shift = 44;
    const int64_t zero = (int64_t)(ref >> 44) - kBins / 2;  // the first round's bin 0
    if (round > 0) {
      uint64_t mn = kBest, mx = 0;
      each([&](uint64_t k, int) {
        if (k >= lo && k <= hi) {
          mn = k < mn ? k : mn;
          mx = k > mx ? k : mx;
        }
      });
      mn = wave_min(mn);
      mx = ~wave_min(~mx);
      if (lane == 0) {
        sh.mn[wave] = mn;
        sh.mx[wave] = mx;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        mn = sh.mn[w] < mn ? sh.mn[w] : mn;
        mx = sh.mx[w] > mx ? sh.mx[w] : mx;
      }
      lo = mn;
      hi = mx;
      if (lo == hi) {  // equal keys: the `need` lowest columns
        int eq = 0;
        each([&](uint64_t k, int) { eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k == lo)); });
        if (lane == 0) sh.sum[wave] = eq;
        __syncthreads();
        int before = before_wave<NW>(sh.sum, lane, wave);
        if (before < need && before + eq >= need)
          each([&](uint64_t k, int c) {
            const uint64_t in = __builtin_amdgcn_ballot_w64(k == lo);
            if (k == lo && before + __builtin_popcountll(in & (lane ? ~0ull >> (64 - lane) : 0ull)) == need - 1) sh.col = c;
            before += __builtin_popcountll(in);
          });
        __syncthreads();
        key = lo;
        col = sh.col;
        break;
      }
      const int bits = 64 - __builtin_clzll(hi - lo);
      shift = bits > 11 ? bits - 11 : 0;
    } else {
      __syncthreads();
    }
    // Scores of one sequence and head are of one magnitude: the first round takes
    // 256 bins an octave around one of them, without a look at their range.
    each([&](uint64_t k, int) {
      if (k < lo || k > hi) return;
      int64_t bin = round > 0 ? (int64_t)((k - lo) >> shift) : (int64_t)(k >> 44) - zero;
      bin = bin < 0 ? 0 : bin > kBins - 1 ? kBins - 1 : bin;
      atomicAdd(&sh.hist[(int)bin], 1);
    });
    __syncthreads();
    // from the top: the bin in which the count reaches `need`
    constexpr int BT = kBins / (NW * 64);  // bins of a thread
    int mine = 0, h[BT];
#pragma unroll
    for (int j = 0; j < BT; ++j) {
      h[j] = sh.hist[kBins - 1 - (tid * BT + j)];
      mine += h[j];
    }
    int inc = wave_scan(mine);
    if (lane == 63) sh.sum[wave] = inc;
    if (tid == 0) sh.cands = 0;
    __syncthreads();
    int above = inc - mine + before_wave<NW>(sh.sum, lane, wave);
#pragma unroll
    for (int j = 0; j < BT; ++j) {
      if (above < need && above + h[j] >= need) {
        sh.pick[0] = kBins - 1 - (tid * BT + j);
        sh.pick[1] = above;
        sh.pick[2] = h[j];
      }
      above += h[j];
    }
    __syncthreads();
    const int bin = sh.pick[0], inside = sh.pick[2];
    need -= sh.pick[1];
    if (round > 0) {
      const uint64_t top = lo + ((uint64_t)(bin + 1) << shift) - 1;
      lo += (uint64_t)bin << shift;
      hi = top < hi && top >= lo ? top : hi;
    } else {  // the outermost bins hold all that lies beyond them
      if (bin < kBins - 1) hi = ((uint64_t)(zero + bin + 1) << 44) - 1;
      if (bin > 0) lo = (uint64_t)(zero + bin) << 44;
    }
    if (inside == need) {  // all of the bin
      key = lo - 1;
      col = -1;
      break;
    }
    if (inside <= 64) {  // few: each is compared with all, by NW lanes together
      each([&](uint64_t k, int c) {
        if (k >= lo && k <= hi) {
          const int i = atomicAdd(&sh.cands, 1);
          sh.cand[i] = k;
          sh.cand_col[i] = c;
        }
      });
      __syncthreads();
      const int i = tid / NW;
      if (i < inside) {
        const uint64_t k = sh.cand[i];
        const int c = sh.cand_col[i];
        int rank = 0;
        for (int j = tid % NW; j < inside; j += NW) {
          const uint64_t o = sh.cand[j];
          rank += o > k || (o == k && sh.cand_col[j] < c);
        }
#pragma unroll
        for (int d = 1; d < NW; d <<= 1) rank += __shfl_xor(rank, d);
        if (rank == need - 1) {
          sh.key = k;
          sh.col = c;
        }
      }
      __syncthreads();
      key = sh.key;
      col = sh.col;
      break;
    }
    __syncthreads();
  }

  int before = 0;
  auto taken = [&](uint64_t k, int c) { return k > key || (k == key && c <= col); };
  each([&](uint64_t k, int c) { before += __builtin_popcountll(__builtin_amdgcn_ballot_w64(taken(k, c))); });
  __syncthreads();
  if (lane == 0) sh.sum[wave] = before;
  __syncthreads();
  before = before_wave<NW>(sh.sum, lane, wave);
  each([&](uint64_t k, int c) {
    const uint64_t in = __builtin_amdgcn_ballot_w64(taken(k, c));
    if (taken(k, c)) out[before + __builtin_popcountll(in & (lane ? ~0ull >> (64 - lane) : 0ull))] = c;
    before += __builtin_popcountll(in);
  });
}

template <int NW, int HELD>
__global__ __launch_bounds__(NW * 64) void paged_best(SelectParams p, const uint64_t* all) {
  __shared__ BestShared sh;
  const int hk = block_x(), b = block_y();
  const uint64_t* keys = all + ((int64_t)b * p.Hkv + hk) * p.map.width;
  best<NW, HELD>(sh, pages_of(p, b), p.n_selected, p.selected + ((int64_t)b * p.Hkv + hk) * p.n_selected,
                 [&](int c) { return keys[c]; });
}

// Both in one launch, a workgroup a row: rows of up to kShort pages.
template <typename T, int LG>
__global__ __launch_bounds__(1024) void paged_short(SelectParams p) {
  __shared__ BestShared sh;
  __shared__ uint64_t keys[kShort];
  constexpr int PW = 64 / LG;
  const int hk = block_x(), b = block_y();
  const int lane = thread_x() & 63, wave = thread_x() >> 6;
  Bounds<T, LG> e;
  e.look(p, b, wave * kSteps * PW + lane / LG);
  const int pages = pages_of(p, b);
  if (pages > p.n_selected && p.n_selected > 1) {
    e.load(p, hk, wave * kSteps * PW + lane / LG, pages, lane & (LG - 1));
    Weights<T> w;
    w.load(p, b, hk, lane & (LG - 1));
    for (int c0 = wave * kSteps * PW; c0 < pages;) {
      score_pages<T, LG>(e, w, c0 + lane / LG, pages, [&](int c, uint64_t k) { keys[c] = k; });
      c0 += 16 * kSteps * PW;
      if (c0 < pages) {
        e.look(p, b, c0 + lane / LG);
        e.load(p, hk, c0 + lane / LG, pages, lane & (LG - 1));
      }
    }
    __syncthreads();
  }
  best<16, kShort / 1024>(sh, pages, p.n_selected, p.selected + ((int64_t)b * p.Hkv + hk) * p.n_selected,
                          [&](int c) { return keys[c]; });
}

template <typename T, int LG>
void launch_lg(const SelectParams& p, hipStream_t s) {
  uint64_t* keys = (uint64_t*)p.workspace;
  const dim3 rows(p.Hkv, p.B);
  if (p.map.width <= kShort) {
    hipLaunchKernelGGL((paged_short<T, LG>), rows, dim3(1024), 0, s, p);
    return;
  }
  const int per = 4 * kSteps * (64 / LG);
  hipLaunchKernelGGL((paged_scores<T, LG>), dim3((p.map.width + per - 1) / per, p.Hkv, p.B), dim3(256), 0, s, p, keys);
  if (p.map.width <= 16 * 64 * 8) hipLaunchKernelGGL((paged_best<16, 8>), rows, dim3(1024), 0, s, p, keys);
  else hipLaunchKernelGGL((paged_best<16, 0>), rows, dim3(1024), 0, s, p, keys);
}

template <typename T>
hipError_t launch(const SelectParams& p, hipStream_t s) {
  const int chunks = p.D * (int)sizeof(T) / 16;
  if (chunks <= 8) launch_lg<T, 8>(p, s);
  else if (chunks <= 16) launch_lg<T, 16>(p, s);
  else if (chunks <= 32) launch_lg<T, 32>(p, s);
  else if constexpr (sizeof(T) == 4) launch_lg<T, 64>(p, s);
  return hipGetLastError();
}

}  // namespace

size_t paged_select_workspace(int B, int Hkv, int width) { return (size_t)B * Hkv * width * sizeof(uint64_t); }

hipError_t launch_paged_select(const SelectParams& p, int dtype, hipStream_t s) {
  if (dtype == 0) return launch<_Float16>(p, s);
  if (dtype == 1) return launch<__bf16>(p, s);
  return launch<float>(p, s);
}

}  // namespace cmpext3
