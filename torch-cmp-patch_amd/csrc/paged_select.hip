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
// registers), four steps of pages in flight.
//
// paged_best takes the best of each (sequence, head) with one workgroup, whose
// waves hold a range of columns each.  The border is found by histograms:
// the range of the keys still in question is cut into 2048 equal bins, the bin
// that holds the border is the next range (scores of one magnitude spread
// evenly over it: two rounds for most inputs).  Which columns are taken is
// then a ballot per 64 columns, so they are written in ascending order, equal
// scores from the lowest column on.
#include "paged_common.h"

namespace cmpext3 {

namespace {

constexpr uint64_t kBest = ~0ull;
constexpr int kSteps = 4;     // steps of pages of a wave, all in flight together
constexpr int kBins = 2048;

// Order of doubles as order of unsigned integers; NaN above everything.
__device__ __forceinline__ uint64_t order_of(double x) {
  if (x != x) return kBest;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// Pages of sequence b that its table row holds.
__device__ __forceinline__ int pages_of(const PageMap& m, int b) {
  return min((seq_len_held(m, b) + m.page_size - 1) / m.page_size, m.width);
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

template <typename T, int LG>
__global__ __launch_bounds__(256) void paged_scores(SelectParams p, uint64_t* keys) {
  constexpr int N = 16 / sizeof(T);  // elements of a chunk
  constexpr int PW = 64 / LG;        // pages of a wave's step
  const int hk = block_y(), b = block_z(), G = p.H / p.Hkv;
  const int lane = thread_x() & 63, wave = thread_x() >> 6;
  const int pages = pages_of(p.map, b);
  const int c0 = (block_x() * 4 + wave) * kSteps * PW + lane / LG;
  if (block_x() * 4 * kSteps * PW >= pages) return;
  const int c = lane & (LG - 1);
  const bool on = c * N < p.D;

  int page[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) page[s] = c0 + s * PW < pages ? page_at(p.map, b, c0 + s * PW) : -1;

  double up[N], down[N];
#pragma unroll
  for (int e = 0; e < N; ++e) up[e] = down[e] = 0;
  if (on) {
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
  u32x4 lo[kSteps], hi[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    lo[s] = hi[s] = (u32x4){0u, 0u, 0u, 0u};
    if (on && page[s] >= 0) {
      const T* at = (const T*)p.bounds + page[s] * p.kb_p + hk * p.kb_h + c * N;
      lo[s] = *(const u32x4*)at;
      hi[s] = *(const u32x4*)(at + p.kb_e);
    }
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    double sum = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      sum = __builtin_fma(up[e], (double)elem<T>(hi[s], e), sum);
      sum = __builtin_fma(down[e], (double)elem<T>(lo[s], e), sum);
    }
    sum = group_sum<LG>(sum);
    if (__builtin_amdgcn_ballot_w64(sum != sum)) {
      // a zero part may have met an infinite bound: without the zero parts
      double t = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (up[e] != 0) t = __builtin_fma(up[e], (double)elem<T>(hi[s], e), t);
        if (down[e] != 0) t = __builtin_fma(down[e], (double)elem<T>(lo[s], e), t);
      }
      t = group_sum<LG>(t);
      if (sum != sum) sum = t;
    }
    const int col = c0 + s * PW;
    if (c == 0 && col < pages)
      keys[((int64_t)b * p.Hkv + hk) * p.map.width + col] = page[s] >= 0 ? order_of(sum) : kBest;
  }
}

__device__ __forceinline__ uint64_t wave_min(uint64_t x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)x, m);
    x = o < x ? o : x;
  }
  return x;
}

// NW waves, each with a contiguous range of columns in steps of 64; HELD: the
// steps' keys stay in registers, else each round reads them again.
template <int NW, int HELD>
__global__ __launch_bounds__(NW * 64) void paged_best(SelectParams p, const uint64_t* all) {
  __shared__ uint64_t s_min[NW], s_max[NW];
  __shared__ int hist[kBins];
  __shared__ int s_sum[NW], s_pick[3], s_gt[NW], s_eq[NW];
  const int tid = thread_x(), lane = tid & 63, wave = tid >> 6;
  const int hk = block_x(), b = block_y(), K = p.n_selected;
  const int pages = pages_of(p.map, b);
  const uint64_t* keys = all + ((int64_t)b * p.Hkv + hk) * p.map.width;
  int32_t* out = p.selected + ((int64_t)b * p.Hkv + hk) * K;
  for (int j = min(pages, K) + tid; j < K; j += NW * 64) out[j] = -1;
  if (pages <= K) {
    for (int j = tid; j < pages; j += NW * 64) out[j] = j;
    return;
  }
  const int m = pages - 1;  // the last page is in; the K - 1 best of m others
  if (K == 1) {
    if (tid == 0) out[0] = m;
    return;
  }
  const int steps = (m + NW * 64 - 1) / (NW * 64);
  const int first = wave * steps * 64 + lane;
  uint64_t held[HELD > 0 ? HELD : 1];
  if constexpr (HELD > 0) {
#pragma unroll
    for (int s = 0; s < HELD; ++s) {
      const int c = first + 64 * s;
      held[s] = s < steps && c < m ? keys[c] : 0;  // 0: below every key
    }
  }
  // f(key, column) for this lane's columns
  auto each = [&](auto f) {
    if constexpr (HELD > 0) {
#pragma unroll
      for (int s = 0; s < HELD; ++s)
        if (s < steps) f(held[s], first + 64 * s);
    } else {
      for (int s = 0; s < steps; ++s) f(first + 64 * s < m ? keys[first + 64 * s] : 0, first + 64 * s);
    }
  };

  // the keys in question are those in [lo, hi]; `need` of them are taken
  uint64_t lo = 1, hi = kBest;
  int need = K - 1;
  bool ties = false;  // all of them are equal
  for (;;) {
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
      s_min[wave] = mn;
      s_max[wave] = mx;
    }
    for (int j = tid; j < kBins; j += NW * 64) hist[j] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      mn = s_min[w] < mn ? s_min[w] : mn;
      mx = s_max[w] > mx ? s_max[w] : mx;
    }
    lo = mn;
    hi = mx;
    if (lo == hi) {
      ties = true;
      break;
    }
    const int bits = 64 - __builtin_clzll(hi - lo);
    const int shift = bits > 11 ? bits - 11 : 0;
    each([&](uint64_t k, int) {
      if (k >= lo && k <= hi) atomicAdd(&hist[(int)((k - lo) >> shift)], 1);
    });
    __syncthreads();
    // from the top: the bin in which the count reaches `need`
    constexpr int BT = kBins / (NW * 64);  // bins of a thread
    int mine = 0, h[BT];
#pragma unroll
    for (int j = 0; j < BT; ++j) {
      h[j] = hist[kBins - 1 - (tid * BT + j)];
      mine += h[j];
    }
    int inc = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(inc, d);
      if (lane >= d) inc += u;
    }
    if (lane == 63) s_sum[wave] = inc;
    __syncthreads();
    int above = inc - mine;
    for (int w = 0; w < wave; ++w) above += s_sum[w];
#pragma unroll
    for (int j = 0; j < BT; ++j) {
      if (above < need && above + h[j] >= need) {
        s_pick[0] = kBins - 1 - (tid * BT + j);
        s_pick[1] = above;
        s_pick[2] = h[j];
      }
      above += h[j];
    }
    __syncthreads();
    const uint64_t bin = (uint64_t)s_pick[0];
    need -= s_pick[1];
    const int inside = s_pick[2];
    const uint64_t top = lo + ((bin + 1) << shift) - 1;
    lo += bin << shift;
    hi = top < hi && top >= lo ? top : hi;
    __syncthreads();
    if (inside == need) break;  // all of the bin
  }

  // taken: keys above hi, and of those in [lo, hi] all, or the first `need`
  int gt = 0, eq = 0;
  each([&](uint64_t k, int) {
    gt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k > hi));
    eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k >= lo && k <= hi));
  });
  if (lane == 0) {
    s_gt[wave] = gt;
    s_eq[wave] = eq;
  }
  __syncthreads();
  gt = eq = 0;
  for (int w = 0; w < wave; ++w) {
    gt += s_gt[w];
    eq += s_eq[w];
  }
  const int most = ties ? need : INT32_MAX;
  const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
  each([&](uint64_t k, int c) {
    const uint64_t g = __builtin_amdgcn_ballot_w64(k > hi), e = __builtin_amdgcn_ballot_w64(k >= lo && k <= hi);
    const int eb = eq + __builtin_popcountll(e & below);
    const bool in_e = k >= lo && k <= hi;
    if (k > hi || (in_e && eb < most)) out[gt + __builtin_popcountll(g & below) + min(eb, most)] = c;
    gt += __builtin_popcountll(g);
    eq += __builtin_popcountll(e);
  });
  if (tid == 0) out[K - 1] = m;
}

template <typename T, int LG>
void scores(const SelectParams& p, uint64_t* keys, hipStream_t s) {
  const int per = 4 * kSteps * (64 / LG);
  hipLaunchKernelGGL((paged_scores<T, LG>), dim3((p.map.width + per - 1) / per, p.Hkv, p.B), dim3(256), 0, s, p, keys);
}

template <typename T>
hipError_t launch(const SelectParams& p, hipStream_t s) {
  uint64_t* keys = (uint64_t*)p.workspace;
  const int chunks = p.D * (int)sizeof(T) / 16;
  if (p.map.width > 0) {
    if (chunks <= 8) scores<T, 8>(p, keys, s);
    else if (chunks <= 16) scores<T, 16>(p, keys, s);
    else if (chunks <= 32) scores<T, 32>(p, keys, s);
    else if constexpr (sizeof(T) == 4) scores<T, 64>(p, keys, s);
  }
  const dim3 grid(p.Hkv, p.B);
  if (p.map.width <= 4 * 64 * 4) hipLaunchKernelGGL((paged_best<4, 4>), grid, dim3(256), 0, s, p, keys);
  else if (p.map.width <= 16 * 64 * 8) hipLaunchKernelGGL((paged_best<16, 8>), grid, dim3(1024), 0, s, p, keys);
  else hipLaunchKernelGGL((paged_best<16, 0>), grid, dim3(1024), 0, s, p, keys);
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
