// Appending new tokens to a paged key-value cache, with the rotary position
// embedding applied on the way.
//
// Work is cut by runs: the new tokens of one sequence that fall into one page.
// One wave takes a (sequence, run, head) of K, V or Q, a lane one 16-byte chunk
// of a token's row and as many tokens at a time as chunks fit the wave.  A run
// ends with its page, so its keys' channel bounds are the wave's own: they are
// kept in registers, joined over the wave's token lanes and written once.
#include "paged_common.h"

namespace cmpext3 {

namespace {

template <typename T> struct Elem;
template <> struct Elem<_Float16> {
  static constexpr int N = 8;  // elements of a 16-byte chunk
  static __device__ float get(const u32x4& w, int e) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e >> 1] >> (16 * (e & 1))));
  }
  static __device__ u32x4 put(const float* x) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i]) |
             (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]) << 16;
    return w;
  }
  static __device__ u32x4 nan() { return (u32x4){0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu}; }
};
template <> struct Elem<__bf16> {
  static constexpr int N = 8;
  static __device__ float get(const u32x4& w, int e) {
    return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  }
  static __device__ u32x4 put(const float* x) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x[2 * i]) |
             (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x[2 * i + 1]) << 16;
    return w;
  }
  static __device__ u32x4 nan() { return (u32x4){0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu}; }
};
template <> struct Elem<float> {
  static constexpr int N = 4;
  static __device__ float get(const u32x4& w, int e) { return __uint_as_float(w[e]); }
  static __device__ u32x4 put(const float* x) {
    return (u32x4){__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
  }
  static __device__ u32x4 nan() { return (u32x4){0x7fc00000u, 0x7fc00000u, 0x7fc00000u, 0x7fc00000u}; }
};

// Chunk c of a row, rotated by the angles in (cs, sn): the partner of element
// d < rot / 2 is d + rot / 2 (or its neighbour, when pairs lie side by side).
template <typename T>
__device__ u32x4 rotated(const T* row, int c, const AppendParams& p, const float* cs, const float* sn) {
  constexpr int N = Elem<T>::N;
  const u32x4 w = *(const u32x4*)(row + c * N);
  const int d0 = c * N, h = p.rot / 2;
  if (d0 >= p.rot) return w;
  float x[N], o[N];
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = Elem<T>::get(w, e);
  if (p.interleaved) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const int j = (d0 + e) / 2;
      const bool in = d0 + e < p.rot;
      const float a = in ? cs[j] : 1.f, s = in ? sn[j] : 0.f;
      o[e] = in ? x[e] * a - x[e + 1] * s : x[e];
      o[e + 1] = in ? x[e + 1] * a + x[e] * s : x[e + 1];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int d = d0 + e;
      if (d < h) o[e] = x[e] * cs[d] - (float)row[d + h] * sn[d];
      else if (d < p.rot) o[e] = x[e] * cs[d - h] + (float)row[d - h] * sn[d - h];
      else o[e] = x[e];
    }
  }
  return Elem<T>::put(o);
}

template <typename T>
__global__ __launch_bounds__(64) void paged_append(AppendParams p) {
  constexpr int N = Elem<T>::N;
  const int lane = threadIdx.x, run = blockIdx.x, b = blockIdx.z;
  int head = blockIdx.y;
  const int kind = head < p.Hkv ? 0 : head < 2 * p.Hkv ? 1 : 2;  // K, V, Q
  head -= kind * p.Hkv;
  const int len = seq_len(p.map, b), n = seq_new(p.map, b, p.S, len);
  const int pos0 = len - n, ps = p.map.page_size;
  const int64_t col = (int64_t)(pos0 / ps) + run;
  const int64_t start = col * ps - pos0;  // the page's slot 0 as a column
  const int last = kind == 2 ? p.S : n;
  if (start >= last) return;
  const int i0 = start > 0 ? (int)start : 0, i1 = start + ps < last ? (int)(start + ps) : last;
  const int page = page_at(p.map, b, col);
  const int C = p.D / N, TL = 64 / C;  // chunks of a row, tokens at a time
  const int t = lane / C, c = lane - t * C;
  const bool on = t < TL;

  const T* src = kind == 0   ? (const T*)p.k + b * p.k_b + head * p.k_h
                 : kind == 1 ? (const T*)p.v + b * p.v_b + head * p.v_h
                             : (const T*)p.q + b * p.q_b + head * p.q_h;
  const int64_t src_s = kind == 0 ? p.k_s : kind == 1 ? p.v_s : p.q_s;
  T* dst = kind == 0   ? (T*)p.k_pages + max(page, 0) * p.kp_p + head * p.kp_h
           : kind == 1 ? (T*)p.v_pages + max(page, 0) * p.vp_p + head * p.vp_h
                       : (T*)p.q_out + b * p.o_b + head * p.o_h;
  const int64_t dst_s = kind == 0 ? p.kp_s : kind == 1 ? p.vp_s : p.o_s;
  const bool edges = kind == 0 && p.bounds != nullptr && page >= 0;
  float lo[N], hi[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    lo[e] = INFINITY;
    hi[e] = -INFINITY;
  }
  if (on) {
    for (int i = i0 + t; i < i1; i += TL) {
      const T* row = src + i * src_s;
      if (i >= n) {  // a padding column of Q
        *(u32x4*)(dst + i * dst_s + c * N) = (u32x4){0u, 0u, 0u, 0u};
        continue;
      }
      const int at = p.positions ? p.positions[(int64_t)b * p.S + i] : pos0 + i;
      const bool ok = page >= 0 && (p.rot == 0 || (at >= 0 && at < p.rows));
      u32x4 w = Elem<T>::nan();
      if (ok) w = kind == 1 || p.rot == 0 ? *(const u32x4*)(row + c * N)
                                          : rotated<T>(row, c, p, p.cos + at * p.rot_s, p.sin + at * p.rot_s);
      if (ok || kind == 2) *(u32x4*)(dst + (kind == 2 ? i : i - start) * dst_s + c * N) = w;
      if (edges && ok) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float x = Elem<T>::get(w, e);
          lo[e] = fminf(lo[e], x);
          hi[e] = fmaxf(hi[e], x);
        }
      }
    }
  }
  if (!edges) return;
  // the token lanes' bounds meet in token lane 0
  float l0[N], h0[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    l0[e] = lo[e];
    h0[e] = hi[e];
    for (int s = 1; s < TL; ++s) {
      l0[e] = fminf(l0[e], __shfl(lo[e], (s * C + lane) & 63));
      h0[e] = fmaxf(h0[e], __shfl(hi[e], (s * C + lane) & 63));
    }
  }
  if (t != 0) return;
  T* edge = (T*)p.bounds + page * p.kb_p + head * p.kb_h + c * N;
  if (start < 0) {  // the page held keys before
    const u32x4 a = *(const u32x4*)edge, z = *(const u32x4*)(edge + p.kb_e);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      l0[e] = fminf(l0[e], Elem<T>::get(a, e));
      h0[e] = fmaxf(h0[e], Elem<T>::get(z, e));
    }
  }
  *(u32x4*)edge = Elem<T>::put(l0);
  *(u32x4*)(edge + p.kb_e) = Elem<T>::put(h0);
}

}  // namespace

hipError_t launch_paged_append(const AppendParams& p, int dtype, hipStream_t s) {
  const int ps = p.map.page_size;
  // pages that S tokens beginning in any slot touch at most
  const int64_t runs = ((int64_t)p.S - 1 + ps - 1) / ps + 1;
  const dim3 grid((unsigned)runs, 2 * p.Hkv + p.H, p.B), block(64);
  if (dtype == 0) hipLaunchKernelGGL(paged_append<_Float16>, grid, block, 0, s, p);
  else if (dtype == 1) hipLaunchKernelGGL(paged_append<__bf16>, grid, block, 0, s, p);
  else hipLaunchKernelGGL(paged_append<float>, grid, block, 0, s, p);
  return hipGetLastError();
}

}  // namespace cmpext3
