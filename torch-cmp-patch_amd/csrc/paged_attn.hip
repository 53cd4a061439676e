// Attention of new tokens over a paged key-value cache: one wave per query
// row, 64 keys at a time (a lane weighs one key, then sums the values of its
// channels), with the running maximum and sum of an online softmax.
#include "paged_common.h"

namespace cmpext3 {

namespace {

template <typename T>
__global__ __launch_bounds__(64) void paged_attn(PagedAttnParams p) {
  __shared__ float qs[256], ws[64];
  const int lane = threadIdx.x, h = blockIdx.y, b = blockIdx.z, i = blockIdx.x;
  const int hk = h / (p.H / p.Hkv), D = p.D, ps = p.map.page_size;
  const int len = seq_len_held(p.map, b), n = seq_new(p.map, b, p.S, len);
  const int limit = i < n ? len - n + i + 1 : 0;
  const int pages = (len + ps - 1) / ps;
  for (int d = lane; d < D; d += 64) {
    const float x = (float)((const T*)p.q)[b * p.q_b + h * p.q_h + i * p.q_s + d];
    qs[d] = p.q_sign ? -x : x;
  }
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  bool bad = (int64_t)len > (int64_t)p.map.width * ps;
  const int entries = p.selected ? p.n_selected : pages;
  for (int s = 0; s < entries && !bad; ++s) {
    int col = s;
    if (p.selected) {
      col = p.selected[((int64_t)b * p.Hkv + hk) * p.n_selected + s];
      if (col < 0) continue;
    }
    const int page = col < pages ? page_at(p.map, b, col) : -1;
    if (page < 0) {
      bad = len > 0;
      continue;
    }
    const int first = col * ps;
    const T* k = (const T*)p.k + page * p.kp_p + hk * p.kp_h;
    const T* v = (const T*)p.v + page * p.vp_p + hk * p.vp_h;
    const int cnt = min(ps, limit - first);
    for (int s0 = 0; s0 < cnt; s0 += 64) {
      const int j = s0 + lane;
      float x = -INFINITY;
      if (j < cnt) {
        x = 0.f;
        for (int d = 0; d < D; ++d) x += qs[d] * (float)k[j * p.kp_s + d];
        x *= p.c;
      }
      float mt = x;
      for (int w = 32; w >= 1; w >>= 1) mt = fmaxf(mt, __shfl_xor(mt, w));
      const float m2 = fmaxf(m, mt);
      const float f = m2 == -INFINITY ? 0.f : m2;
      const float a = exp2f(m - f), e = j < cnt ? exp2f(x - f) : 0.f;
      m = m2;
      float sum = e;
      for (int w = 32; w >= 1; w >>= 1) sum += __shfl_xor(sum, w);
      l = l * a + sum;
      __syncthreads();
      ws[lane] = e;
      __syncthreads();
      for (int z = 0; z < 4; ++z) {
        const int d = lane + 64 * z;
        if (d >= D) break;
        o[z] *= a;
        for (int t = 0; t < min(64, cnt - s0); ++t) o[z] += ws[t] * (float)v[(s0 + t) * p.vp_s + d];
      }
    }
  }
  for (int z = 0; z < 4; ++z) {
    const int d = lane + 64 * z;
    if (d >= D) break;
    const float r = bad ? __builtin_nanf("") : l > 0.f || l != l ? o[z] / l : 0.f;
    ((T*)p.o)[b * p.o_b + h * p.o_h + i * p.o_s + d] = (T)r;
  }
}

}  // namespace

size_t paged_attn_workspace(int, int, int, int, int, int, int, int, int) { return 0; }

hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, hipStream_t s) {
  const dim3 grid(p.S, p.H, p.B), block(64);
  if (dtype == 0) hipLaunchKernelGGL(paged_attn<_Float16>, grid, block, 0, s, p);
  else if (dtype == 1) hipLaunchKernelGGL(paged_attn<__bf16>, grid, block, 0, s, p);
  else hipLaunchKernelGGL(paged_attn<float>, grid, block, 0, s, p);
  return hipGetLastError();
}

}  // namespace cmpext3
