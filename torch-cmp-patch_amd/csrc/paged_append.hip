// Appending new tokens to a paged key-value cache, with the rotary position
// embedding applied on the way.
//
// Bound by HBM for prompts (every row is read once and written once; measured on
// MI355X: bf16 4 x 2048 tokens of 16 + 8 + 8 heads of 128 with bounds 30.3 us,
// 4.5 TB/s) and by the latency of its loads for single tokens (16 of them 3.3
// us): lengths, then the page number and the rotation's row, while the rows
// themselves, which depend on neither, are on their way.
//
// A lane takes one unit of a row: with pairs (d, d + rot / 2) the two 16-byte
// chunks that turn together, else one chunk.  Lanes run over a token's units,
// then over its heads (K, V and Q in a row), then over tokens, so that a
// workgroup reads what a projection left in one stretch and a rotation's row
// once for all of a token's heads.
//
// With key bounds, keys of more than one token a call are taken by runs instead: the new tokens
// of one sequence that fall into one page.  A wave takes a (sequence, run,
// head); the run ends with its page, so the page's bounds are the wave's own:
// kept in registers, joined over the wave's token lanes, written once.
#include "paged_common.h"

namespace cmpext3 {

namespace {

template <typename T>
__device__ __forceinline__ float get_elem(uint32_t w, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  else if constexpr (__is_same(T, __bf16)) return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> (16 * (e & 1))));
}

// The elements of a 16-byte chunk.
template <typename T>
struct Elem {
  static constexpr int N = 16 / (int)sizeof(T);
  static __device__ __forceinline__ float get(const u32x4& w, int e) { return get_elem<T>(w[e * (int)sizeof(T) / 4], e); }
  static __device__ __forceinline__ u32x4 put(const float* x) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = __float_as_uint(x[i]);
      else
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (T)x[2 * i]) |
               (uint32_t)__builtin_bit_cast(uint16_t, (T)x[2 * i + 1]) << 16;
    }
    return w;
  }
  static __device__ __forceinline__ u32x4 all(uint32_t v) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v;
    return w;
  }
  static __device__ __forceinline__ u32x4 nan() { return all(sizeof(T) == 4 ? 0x7fc00000u : 0x7fff7fffu); }
};

// N angles' cosines or sines.
template <int N>
__device__ __forceinline__ void angles(const float* at, float* x) {
  typedef f32x4 four __attribute__((aligned(4)));
  typedef u32x2 two __attribute__((aligned(4)));
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      const f32x4 v = *(const four*)(at + k);
      x[k] = v[0]; x[k + 1] = v[1]; x[k + 2] = v[2]; x[k + 3] = v[3];
    }
  } else {
    static_assert(N == 2, "a chunk's pairs");
    const u32x2 v = *(const two*)at;
    x[0] = __uint_as_float(v[0]);
    x[1] = __uint_as_float(v[1]);
  }
}

// How a row is rotated.
enum Mode {
  kCopy,   // not at all
  kHalf,   // pairs (d, d + rot / 2) in whole 16-byte chunks
  kSkew,   // the same where a half is no whole number of chunks
  kSide,   // pairs (2 d, 2 d + 1) in whole chunks
  kAny     // anything else: element by element
};

struct Shape {
  int units, pairs;  // units of a row; the first `pairs` of them are two chunks, a half apart
  int half, rest;    // channels of a half, and behind the rotated ones
  int heads;         // heads of a token in the first section: V and Q, and K where it takes no runs
  int runs;          // second section: runs per (sequence, head)
  int first;         // workgroups of the first section
  int q_at, v_at;    // where V's and Q's heads begin in a token's
  Div by_units, by_heads, by_s, by_ps, by_runs, by_groups;
};

// A chunk in memory: at a multiple of 16 bytes, or of 4.
template <bool SKEW> struct Words { typedef u32x4 type; };
template <> struct Words<true> { typedef u32x4 type __attribute__((aligned(4))); };

// One unit of a row: a chunk or two, and those rotated.
template <typename T, int MODE>
struct Unit {
  typedef Elem<T> E;
  static constexpr int N = E::N;
  static constexpr bool kTwo = MODE == kHalf || MODE == kSkew;  // the chunks of a pair turn together
  typedef typename Words<MODE == kSkew>::type W;
  int e0, e1;  // the chunks' first channels; e1 < 0: one chunk
  u32x4 x0, x1;
  __device__ __forceinline__ Unit(int u, const Shape& sh) {
    e0 = kTwo && u >= sh.pairs ? u * N - sh.pairs * N : u * N;
    if constexpr (MODE == kSkew) {
      // the last chunk of a part ends with it: what it shares with the one
      // before is written twice, the same
      e0 = u < sh.pairs ? min(e0, sh.half - N) : 2 * sh.half + min(e0, sh.rest - N);
    } else if (kTwo && u >= sh.pairs) {
      e0 += 2 * sh.half;
    }
    e1 = kTwo && u < sh.pairs ? e0 + sh.half : -1;
  }
  __device__ __forceinline__ void load(const T* row) {
    x0 = *(const W*)(row + e0);
    x1 = x0;
    if constexpr (kTwo) {
      if (e1 >= 0) x1 = *(const W*)(row + e1);
    }
  }
  // by the angles of one row of the tables
  __device__ __forceinline__ void rotate(const T* row, const AppendParams& p, const float* cs, const float* sn) {
    const int d0 = e0;
    if constexpr (kTwo) {
      if (e1 < 0) return;
      float a[N], b[N], c[N], s[N];
      angles<N>(cs + d0, c);
      angles<N>(sn + d0, s);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float x = E::get(x0, e), y = E::get(x1, e);
        a[e] = x * c[e] - y * s[e];
        b[e] = y * c[e] + x * s[e];
      }
      x0 = E::put(a);
      x1 = E::put(b);
    } else if constexpr (MODE == kSide) {
      if (d0 >= p.rot) return;
      float a[N], c[N / 2], s[N / 2];
      angles<N / 2>(cs + d0 / 2, c);
      angles<N / 2>(sn + d0 / 2, s);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float x = E::get(x0, e), y = E::get(x0, e + 1);
        a[e] = x * c[e / 2] - y * s[e / 2];
        a[e + 1] = y * c[e / 2] + x * s[e / 2];
      }
      x0 = E::put(a);
    } else if constexpr (MODE == kAny) {
      const int h = p.rot / 2;
      if (d0 >= p.rot) return;
      float a[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int d = d0 + e;
        const int j = p.interleaved ? d / 2 : d < h ? d : d - h;
        const bool low = p.interleaved ? (d & 1) == 0 : d < h;
        const float x = E::get(x0, e);
        a[e] = x;
        if (d < p.rot) {
          const float y = (float)row[p.interleaved ? (low ? d + 1 : d - 1) : (low ? d + h : d - h)];
          a[e] = low ? x * cs[j] - y * sn[j] : x * cs[j] + y * sn[j];
        }
      }
      x0 = E::put(a);
    }
  }
  __device__ __forceinline__ void store(T* row) const {
    *(W*)(row + e0) = x0;
    if constexpr (kTwo) {
      if (e1 >= 0) *(W*)(row + e1) = x1;
    }
  }
  __device__ __forceinline__ void fill(const u32x4& w) { x0 = x1 = w; }
};

// Lowest and highest values of one chunk's channels.
template <typename U>
struct Range {
  typedef typename U::E E;
  typedef typename U::W W;
  static constexpr int N = E::N;
  float lo[N], hi[N];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      lo[e] = INFINITY;
      hi[e] = -INFINITY;
    }
  }
  __device__ __forceinline__ void take(const u32x4& w) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      lo[e] = fminf(lo[e], E::get(w, e));
      hi[e] = fmaxf(hi[e], E::get(w, e));
    }
  }
  __device__ __forceinline__ void take(const Range& o) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      lo[e] = fminf(lo[e], o.lo[e]);
      hi[e] = fmaxf(hi[e], o.hi[e]);
    }
  }
  // over the lanes of the same unit, `units` apart, `n` of them, into the first
  __device__ __forceinline__ void join(int lane, int t, int n, int units) {
    for (int d = 1; d < n; d <<= 1) {
      const bool in = t + d < n;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float l = __shfl(lo[e], (lane + d * units) & 63), h = __shfl(hi[e], (lane + d * units) & 63);
        lo[e] = in ? fminf(lo[e], l) : lo[e];
        hi[e] = in ? fmaxf(hi[e], h) : hi[e];
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* lows, T* highs, bool anew) {
    if (!anew) {
      const u32x4 a = *(const W*)lows, z = *(const W*)highs;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        lo[e] = fminf(lo[e], E::get(a, e));
        hi[e] = fmaxf(hi[e], E::get(z, e));
      }
    }
    *(W*)lows = E::put(lo);
    *(W*)highs = E::put(hi);
  }
};

// Keys of a run with their page's bounds.
template <typename T, int MODE, int WAVES>
__device__ __forceinline__ void append_run(const AppendParams& p, const Shape& sh, int wg) {
  typedef Unit<T, MODE> U;
  const int lane = thread_x() & 63, wave = __builtin_amdgcn_readfirstlane(thread_x() >> 6);
  const int rest = quot(wg, sh.by_runs.m, sh.by_runs.s), run = wg - rest * sh.runs;
  constexpr int heads = 4 / WAVES;  // a workgroup's
  const int groups = (p.Hkv + heads - 1) / heads;
  const int b = quot(rest, sh.by_groups.m, sh.by_groups.s);
  const int head = (rest - b * groups) * heads + (WAVES == 1 ? wave : 0);
  if (head >= p.Hkv) return;
  const int len = seq_len(p.map, b), n = seq_new(p.map, b, p.S, len);
  const int pos0 = len - n, ps = p.map.page_size;
  const int64_t col = (int64_t)quot(pos0, sh.by_ps.m, sh.by_ps.s) + run;
  const int64_t start = col * ps - pos0;  // the page's slot 0 as a column
  if (start >= n) return;
  const int i0 = start > 0 ? (int)start : 0, i1 = start + ps < n ? (int)(start + ps) : n;
  const int page = page_at(p.map, b, col);
  if (page < 0) return;
  const int TL = 64 / sh.units, t = quot(lane, sh.by_units.m, sh.by_units.s), u = lane - t * sh.units;
  const T* src = (const T*)p.k + b * p.k_b + head * p.k_h;
  T* dst = (T*)p.k_pages + page * p.kp_p + head * p.kp_h;
  const Unit<T, MODE> at(u, sh);
  Range<U> r0, r1;
  r0.clear();
  r1.clear();
  bool some = false;
  if (t < TL) {
    // one step at a time: a second in flight takes more registers than it hides
    // (bf16 4 x 2048 tokens 31.3 us with two, 30.3 with one; 8 x 80 8.4, 8.1)
#pragma unroll 1
    for (int i = i0 + t + (WAVES == 1 ? 0 : wave * TL); i < i1; i += TL * WAVES) {
      const T* row = src + i * p.k_s;
      Unit<T, MODE> w = at;
      w.load(row);
      bool ok = true;
      if constexpr (MODE != kCopy) {
        const int a = p.positions ? p.positions[(int64_t)b * p.S + i] : pos0 + i;
        ok = a >= 0 && a < p.rows;
        if (ok) w.rotate(row, p, p.cos + a * p.rot_s, p.sin + a * p.rot_s);
      }
      if (ok) {
        w.store(dst + (i - start) * p.kp_s);
        r0.take(w.x0);
        if constexpr (Unit<T, MODE>::kTwo) r1.take(w.x1);
        some = true;
      }
    }
  }
  if (WAVES == 1 && !__builtin_amdgcn_ballot_w64(some)) return;
  r0.join(lane, t, TL, sh.units);
  if constexpr (Unit<T, MODE>::kTwo) r1.join(lane, t, TL, sh.units);
  if constexpr (WAVES > 1) {  // the four waves' bounds meet in the first
    __shared__ Range<U> far[3][2][64];
    __shared__ int any;
    if (thread_x() == 0) any = 0;
    __syncthreads();
    if (some) any = 1;
    if (wave > 0 && t == 0) {
      far[wave - 1][0][lane] = r0;
      if constexpr (Unit<T, MODE>::kTwo) far[wave - 1][1][lane] = r1;
    }
    __syncthreads();
    if (wave > 0 || !any) return;
    if (t == 0)
      for (int w = 0; w < 3; ++w) {
        r0.take(far[w][0][lane]);
        if constexpr (Unit<T, MODE>::kTwo) r1.take(far[w][1][lane]);
      }
  }
  if (t != 0) return;
  const bool anew = start >= 0;  // the page begins with a new token
  T* edge = (T*)p.bounds + page * p.kb_p + head * p.kb_h;
  r0.store(edge + at.e0, edge + p.kb_e + at.e0, anew);
  if constexpr (Unit<T, MODE>::kTwo) {
    if (at.e1 >= 0) r1.store(edge + at.e1, edge + p.kb_e + at.e1, anew);
  }
}

// RUNS: waves of a run in the second section, 0 without one (its registers, and
// the LDS of four waves, would cost the others residency: fp16 chunks 10.1 us
// with it compiled in, 9.5 without).
template <typename T, int MODE, int RUNS>
__global__ __launch_bounds__(256) void paged_append(AppendParams p, Shape sh) {
  typedef Unit<T, MODE> U;
  if constexpr (RUNS > 0) {
    if (block_x() >= sh.first) {
      append_run<T, MODE, RUNS>(p, sh, block_x() - sh.first);
      return;
    }
  }
  const int item = block_x() * 256 + thread_x();
  const int rest = quot(item, sh.by_units.m, sh.by_units.s), u = item - rest * sh.units;
  const int token = quot(rest, sh.by_heads.m, sh.by_heads.s);
  int head = rest - token * sh.heads;
  const int b = quot(token, sh.by_s.m, sh.by_s.s), i = token - b * p.S;
  if (b >= p.B) return;
  const int kind = head >= sh.q_at ? 2 : head >= sh.v_at ? 1 : 0;  // Q, V, K
  head -= kind == 2 ? sh.q_at : kind == 1 ? sh.v_at : 0;
  const T* row = kind == 0   ? (const T*)p.k + b * p.k_b + head * p.k_h + i * p.k_s
                 : kind == 1 ? (const T*)p.v + b * p.v_b + head * p.v_h + i * p.v_s
                             : (const T*)p.q + b * p.q_b + head * p.q_h + i * p.q_s;
  Unit<T, MODE> w(u, sh);
  w.load(row);
  const int len = seq_len(p.map, b), n = seq_new(p.map, b, p.S, len);
  const bool fresh = i < n;
  if (!fresh && kind != 2) return;
  const int pos = fresh ? len - n + i : 0;
  const int col = quot(pos, sh.by_ps.m, sh.by_ps.s), slot = pos - col * p.map.page_size;
  const int page = fresh ? page_at(p.map, b, col) : -1;
  bool ok = page >= 0;
  if constexpr (MODE != kCopy) {
    const int a = p.positions ? p.positions[token] : pos;
    ok = ok && a >= 0 && a < p.rows;
    if (kind != 1 && ok) w.rotate(row, p, p.cos + a * p.rot_s, p.sin + a * p.rot_s);
  }
  if (kind == 2) {
    if (!fresh) w.fill(U::E::all(0));
    else if (!ok) w.fill(U::E::nan());
    w.store((T*)p.q_out + b * p.o_b + head * p.o_h + i * p.o_s);
    return;
  }
  if (!ok) return;
  w.store(kind == 0 ? (T*)p.k_pages + page * p.kp_p + head * p.kp_h + slot * p.kp_s
                    : (T*)p.v_pages + page * p.vp_p + head * p.vp_h + slot * p.vp_s);
  if (kind == 0 && p.bounds) {  // one token a call: its page's bounds are this unit's alone
    T* edge = (T*)p.bounds + page * p.kb_p + head * p.kb_h;
    Range<U> r;
    r.clear();
    r.take(w.x0);
    r.store(edge + w.e0, edge + p.kb_e + w.e0, slot == 0);
    if constexpr (Unit<T, MODE>::kTwo) {
      if (w.e1 >= 0) {
        Range<U> z;
        z.clear();
        z.take(w.x1);
        z.store(edge + w.e1, edge + p.kb_e + w.e1, slot == 0);
      }
    }
  }
}

template <typename T, int RUNS>
void launch_mode(const AppendParams& p, const Shape& sh, Mode mode, unsigned wgs, hipStream_t s) {
  const dim3 grid(wgs), block(256);
  if (mode == kCopy) hipLaunchKernelGGL((paged_append<T, kCopy, RUNS>), grid, block, 0, s, p, sh);
  else if (mode == kHalf) hipLaunchKernelGGL((paged_append<T, kHalf, RUNS>), grid, block, 0, s, p, sh);
  else if (mode == kSkew) hipLaunchKernelGGL((paged_append<T, kSkew, RUNS>), grid, block, 0, s, p, sh);
  else if (mode == kSide) hipLaunchKernelGGL((paged_append<T, kSide, RUNS>), grid, block, 0, s, p, sh);
  else hipLaunchKernelGGL((paged_append<T, kAny, RUNS>), grid, block, 0, s, p, sh);
}

template <typename T>
hipError_t launch(const AppendParams& p, hipStream_t s) {
  constexpr int N = 16 / (int)sizeof(T);
  const int h = p.rot / 2, ps = p.map.page_size;
  const bool by_runs = p.bounds && p.S > 1;
  Shape sh;
  sh.half = h;
  sh.rest = p.D - p.rot;
  // halves that are no whole chunks take skewed ones, where each part of the
  // row holds one and words keep their 4 bytes (bf16 [36,20/5,1081,72] with 36
  // rotated: 77 us, element by element 136)
  const bool skew = h >= N && h * sizeof(T) % 4 == 0 && (sh.rest == 0 || sh.rest >= N);
  const Mode mode = p.rot == 0        ? kCopy
                    : p.interleaved   ? (p.rot % N == 0 ? kSide : kAny)
                    : h % N == 0      ? kHalf
                    : skew            ? kSkew
                                      : kAny;
  const bool two = mode == kHalf || mode == kSkew;
  sh.pairs = two ? (h + N - 1) / N : 0;
  sh.units = two ? sh.pairs + (sh.rest + N - 1) / N : p.D / N;
  sh.v_at = by_runs ? 0 : p.Hkv;
  sh.q_at = sh.v_at + p.Hkv;
  sh.heads = sh.q_at + p.H;
  const int64_t items = (int64_t)p.B * p.S * sh.heads * sh.units;
  sh.first = (int)((items + 255) / 256);
  // pages that S tokens beginning in any slot touch at most
  sh.runs = by_runs ? (p.S - 1 + ps - 1) / ps + 1 : 1;
  // a run of more tokens than a wave takes in two steps goes to four waves
  const int waves = by_runs && (ps < p.S ? ps : p.S) * sh.units > 2 * 64 ? 4 : 1;
  const int heads = 4 / waves, groups = (p.Hkv + heads - 1) / heads;
  const int64_t second = by_runs ? (int64_t)p.B * groups * sh.runs : 0;
  sh.by_units = div_by(sh.units);
  sh.by_heads = div_by(sh.heads);
  sh.by_s = div_by(p.S);
  sh.by_ps = div_by(ps);
  sh.by_runs = div_by(sh.runs);
  sh.by_groups = div_by(groups);
  const unsigned wgs = (unsigned)(sh.first + second);
  if (!by_runs) launch_mode<T, 0>(p, sh, mode, wgs, s);
  else if (waves == 1) launch_mode<T, 1>(p, sh, mode, wgs, s);
  else launch_mode<T, 4>(p, sh, mode, wgs, s);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(const AppendParams& p, int dtype, hipStream_t s) {
  if (dtype == 0) return launch<_Float16>(p, s);
  if (dtype == 1) return launch<__bf16>(p, s);
  return launch<float>(p, s);
}

}  // namespace cmpext3
