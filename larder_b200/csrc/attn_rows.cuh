// Attention one query row a warp, on CUDA cores in fp32: lane l holds D / 32 of the row's dims, keys are taken one at a
// time with an online softmax. Exact masking: a key that the row does not see is never read. The fp32 path of the paged
// cache's attention and of packed prompts.
#pragma once

#include "common.cuh"
#include "kv8.cuh"

namespace lb2 {
namespace arows {

// Keys and values of one sequence and KV head, a row at a time: E values of the lane.
template <int E>
struct PagedKeys {
  const uint8_t* pages;
  const float* scales;
  const int32_t* table;  // the sequence's row
  int Hkv, hk, page, num_pages;
  int d0;
  __device__ __forceinline__ void load(int n, float* k, float* v) const {
    const int id = table[n / page], r = n % page;
    if (id < 0 || id >= num_pages) {
      report_bad_index(111);
#pragma unroll
      for (int e = 0; e < E; ++e) k[e] = v[e] = 0.f;
      return;
    }
    const int64_t s = int64_t(id) * 2 * Hkv + hk;
    const uint8_t* kp = pages + (s * page + r) * (32 * E) + d0;
    const uint8_t* vp = kp + int64_t(Hkv) * page * (32 * E);
    const float ks = scales[s], vs = scales[s + Hkv];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      uint32_t a, b, lo, hi;
      a = *reinterpret_cast<const uint16_t*>(kp + e);
      b = *reinterpret_cast<const uint16_t*>(vp + e);
      kv8::dec4(a | b << 16, lo, hi);
      const float2 f = kv8::half2_f(lo), g = kv8::half2_f(hi);
      k[e] = f.x * ks, k[e + 1] = f.y * ks;
      v[e] = g.x * vs, v[e + 1] = g.y * vs;
    }
  }
};

template <typename T, int E>
struct PlainKeys {
  const T* k0;
  const T* v0;
  int64_t k_st, v_st;
  __device__ __forceinline__ void load(int n, float* k, float* v) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      k[e] = to_f<T>(k0[n * k_st + e]);
      v[e] = to_f<T>(v0[n * v_st + e]);
    }
  }
};

// softmax(scale q K^T) V over keys 0 .. n - 1 for one row; zeros for n <= 0. x: the lane's E values of q, then of o.
template <int E, typename Keys>
__device__ __forceinline__ void attend_row(const Keys& keys, int n, float scale, float* x) {
  float q[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) q[e] = x[e] * scale, x[e] = 0.f;
  for (int i = 0; i < n; ++i) {
    float k[E], v[E], s = 0.f;
    keys.load(i, k, v);
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float m1 = fmaxf(m, s);  // (a NaN score stays out of m and reaches l and x through w)
    const float mu = m1 == -INFINITY ? 0.f : m1;
    const float f = expf(m - mu), w = expf(s - mu);
    l = l * f + w;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = fmaf(w, v[e], x[e] * f);
    m = m1;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] *= inv;
}

struct PagedParams {
  const void* q;
  void* o;
  int64_t q_st[3], o_st[3];
  const uint8_t* pages;
  const float* scales;
  const int32_t* table;
  int64_t table_st;
  const int32_t* kv_len;
  int B, Hq, Hkv, T, page, num_pages, max_pages, causal;
  float scale;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) paged_kernel(const PagedParams p) {
  constexpr int E = D / 32;
  const int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w >= int64_t(p.B) * p.Hq * p.T) return;
  const int d0 = (threadIdx.x & 31) * E;
  const int t = int(w % p.T), h = int(w / p.T % p.Hq), b = int(w / p.T / p.Hq);
  const T* q = static_cast<const T*>(p.q) + b * p.q_st[0] + h * p.q_st[1] + t * p.q_st[2] + d0;
  T* o = static_cast<T*>(p.o) + b * p.o_st[0] + h * p.o_st[1] + t * p.o_st[2] + d0;
  const int len = int(min(int64_t(max(p.kv_len[b], 0)), int64_t(p.max_pages) * p.page));
  if (len != p.kv_len[b] && d0 == 0) report_bad_index(111);
  PagedKeys<E> keys{p.pages, p.scales, p.table + b * p.table_st, p.Hkv, h / (p.Hq / p.Hkv), p.page, p.num_pages, d0};
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = to_f<T>(q[e]);
  attend_row<E>(keys, p.causal ? len - p.T + 1 + t : len, p.scale, x);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = from_f<T>(x[e]);
}

struct PackedParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  int64_t q_st[2], k_st[2], v_st[2], o_st[2];  // H, T
  const int32_t* cu;
  int S, Hq, Hkv, T;
  float scale;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) packed_kernel(const PackedParams p) {
  constexpr int E = D / 32;
  const int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w >= int64_t(p.Hq) * p.T) return;
  const int d0 = (threadIdx.x & 31) * E;
  const int row = int(w / p.Hq), h = int(w % p.Hq), hk = h / (p.Hq / p.Hkv);
  int lo = 0, hi = p.S;  // the last s with cu[s] <= row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu[mid] <= row) lo = mid; else hi = mid;
  }
  const int first = p.cu[lo];
  const bool mine = first >= 0 && row >= first && row < p.cu[lo + 1];  // else a row of no sequence: zeros
  T* o = static_cast<T*>(p.o) + h * p.o_st[0] + row * p.o_st[1] + d0;
  const T* q = static_cast<const T*>(p.q) + h * p.q_st[0] + row * p.q_st[1] + d0;
  PlainKeys<T, E> keys{static_cast<const T*>(p.k) + hk * p.k_st[0] + int64_t(max(first, 0)) * p.k_st[1] + d0,
                       static_cast<const T*>(p.v) + hk * p.v_st[0] + int64_t(max(first, 0)) * p.v_st[1] + d0, p.k_st[1],
                       p.v_st[1]};
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = to_f<T>(q[e]);
  attend_row<E>(keys, mine ? row - first + 1 : 0, p.scale, x);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = from_f<T>(x[e]);
}

}  // namespace arows
}  // namespace lb2
