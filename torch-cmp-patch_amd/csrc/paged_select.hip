// The pages of each sequence that its new token attends to.
//
// A page's score for a K/V head bounds the products of its keys with the
// head's queries: sum over queries h and channels d of max(q lo, q hi), which
// is sum over d of Q+ hi + Q- lo with Q+ (Q-) the sum of the queries' positive
// (negative) parts.  All of it in 64 bits: products of the inputs are exact
// there, and a page near the border falls on the same side whatever the order
// of the sums.  One kernel writes the scores as integers of the same order,
// the next takes the best of each (sequence, head).
#include "paged_common.h"

namespace cmpext3 {

namespace {

constexpr uint64_t kBest = ~0ull;

// Order of doubles as order of unsigned integers; NaN above everything.
__device__ uint64_t order_of(double x) {
  if (x != x) return kBest;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

template <typename T>
__global__ __launch_bounds__(256) void paged_scores(SelectParams p, uint64_t* keys) {
  __shared__ double up[256], down[256];
  const int hk = blockIdx.y, b = blockIdx.z, G = p.H / p.Hkv, D = p.D;
  const int len = seq_len_held(p.map, b), ps = p.map.page_size;
  const int pages = min((len + ps - 1) / ps, p.map.width);
  if ((int)blockIdx.x * 256 >= pages) return;
  for (int d = threadIdx.x; d < D; d += 256) {
    double u = 0, w = 0;
    for (int g = 0; g < G; ++g) {
      const float x = (float)((const T*)p.q)[b * p.q_b + (hk * G + g) * p.q_h + d];
      if (x < 0) w += (double)x;
      else u += (double)x;  // and a NaN
    }
    up[d] = u;
    down[d] = w;
  }
  __syncthreads();
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= pages) return;
  uint64_t key = kBest;
  const int page = page_at(p.map, b, col);
  if (page >= 0) {
    const T* e = (const T*)p.bounds + page * p.kb_p + hk * p.kb_h;
    double s = 0;
    for (int d = 0; d < D; ++d) s += up[d] * (double)(float)e[p.kb_e + d] + down[d] * (double)(float)e[d];
    if (s != s) {  // a zero part met an infinite bound, perhaps: without the zero parts
      s = 0;
      for (int d = 0; d < D; ++d) {
        if (up[d] != 0) s += up[d] * (double)(float)e[p.kb_e + d];
        if (down[d] != 0) s += down[d] * (double)(float)e[d];
      }
    }
    key = order_of(s);
  }
  keys[((int64_t)b * p.Hkv + hk) * p.map.width + col] = key;
}

__global__ __launch_bounds__(256) void paged_best(SelectParams p, const uint64_t* all) {
  __shared__ int taken[256];
  const int hk = blockIdx.x, b = blockIdx.y;
  const int len = seq_len_held(p.map, b), ps = p.map.page_size, K = p.n_selected;
  const int pages = min((len + ps - 1) / ps, p.map.width);
  const uint64_t* keys = all + ((int64_t)b * p.Hkv + hk) * p.map.width;
  int32_t* out = p.selected + ((int64_t)b * p.Hkv + hk) * K;
  int done = 0;
  for (int c0 = 0; c0 < pages; c0 += 256) {
    const int c = c0 + threadIdx.x;
    int in = 0;
    if (c < pages) {
      int above = 0;  // better pages, the last one among them
      for (int j = 0; j < pages; ++j)
        above += j != c && (j == pages - 1 || keys[j] > keys[c] || (keys[j] == keys[c] && j < c));
      in = c == pages - 1 || above < K;
    }
    __syncthreads();
    taken[threadIdx.x] = in;
    __syncthreads();
    int before = 0, total = 0;
    for (int t = 0; t < 256; ++t) {
      total += taken[t];
      if (t < (int)threadIdx.x) before += taken[t];
    }
    if (in) out[done + before] = c;
    done += total;
  }
  for (int j = done + threadIdx.x; j < K; j += 256) out[j] = -1;
}

template <typename T>
hipError_t launch(const SelectParams& p, hipStream_t s) {
  uint64_t* keys = (uint64_t*)p.workspace;
  if (p.map.width > 0)
    hipLaunchKernelGGL(paged_scores<T>, dim3((p.map.width + 255) / 256, p.Hkv, p.B), dim3(256), 0, s, p, keys);
  hipLaunchKernelGGL(paged_best, dim3(p.Hkv, p.B), dim3(256), 0, s, p, keys);
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
