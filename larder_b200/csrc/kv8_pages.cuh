// Pages of the paged 8-bit cache (kv8.cuh) moved about: whole pages copied, and sequences compacted to the tokens kept.
#pragma once

#include "common.cuh"
#include "kv8.cuh"
#include "rope.cuh"

namespace lb2 {
namespace kv8 {

constexpr int STATUS_COPY = 150, STATUS_COMPACT = 151;  // an id or position out of range (lb2_status)

struct CopyParams {
  const uint8_t* from;
  const float* from_scales;
  uint8_t* to;
  float* to_scales;
  const int32_t* src;
  const int32_t* dst;
  int n, from_num, to_num;
  int heads;      // scales a page: 2 Hkv
  int64_t bytes;  // a page's codes
};

constexpr int COPY_THREADS = 256;

__global__ void __launch_bounds__(COPY_THREADS) copy_kernel(const CopyParams p) {
  const int i = blockIdx.y;
  const int s = p.src[i], d = p.dst[i];
  if (s < 0 || s >= p.from_num || d < 0 || d >= p.to_num) {
    if (threadIdx.x == 0) report_bad_index(STATUS_COPY);
    return;
  }
  const uint4* x = reinterpret_cast<const uint4*>(p.from + s * p.bytes);
  uint4* y = reinterpret_cast<uint4*>(p.to + d * p.bytes);
  for (int64_t e = int64_t(blockIdx.x) * COPY_THREADS + threadIdx.x; e < p.bytes / 16; e += int64_t(gridDim.x) * COPY_THREADS)
    y[e] = x[e];
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e < p.heads; e += COPY_THREADS)
      p.to_scales[int64_t(d) * p.heads + e] = p.from_scales[int64_t(s) * p.heads + e];
}

struct CompactParams {
  uint8_t* pages;
  float* scales;
  const int32_t* table;
  const int32_t* keep;
  const int32_t* cu;
  const int32_t* to;
  const int32_t* start;
  const uint64_t* turns;
  int64_t table_st, to_st;
  int B, Hkv, T, D, R, num_pages, max_pages, max_to;
  int lpage;  // log2 of page
  int interleaved;
};

// The page that block piece i writes: of sequence b, its moved tokens [t0, t0 + n), into page `id` (out of range: none).
struct CompactPiece {
  int b, t0, n, id;
  int64_t first;  // position of the page's first token
  int row0;       // index of token t0 in keep
};

// Sequence b's pieces start at cu[b] / page + b, which leaves room for its pages (n tokens fill at most n / page + 1).
__device__ __forceinline__ bool compact_piece(const CompactParams& p, int i, CompactPiece& w) {
  auto base = [&](int s) { return (min(max(p.cu[s], 0), p.T) >> p.lpage) + s; };
  int lo = 0, hi = p.B;  // base(lo) <= i, and base(hi) > i or hi == B
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, s = lo + (threadIdx.x & 31) * step;
    const uint32_t le = __ballot_sync(0xffffffffu, s < hi && (s == lo || base(s) <= i));
    const int k = 31 - __clz(le);
    lo += k * step;
    hi = min(hi, lo + step);
  }
  w.b = lo;
  const int j = i - base(lo), page = 1 << p.lpage;
  const int c0 = p.cu[lo], c1 = p.cu[lo + 1], r0 = min(max(c0, 0), p.T), n = min(max(c1, r0), p.T) - r0;
  const bool lead = threadIdx.x == 0;
  if (lead && j == 0 && (c0 != r0 || c1 != r0 + n)) report_bad_index(STATUS_COMPACT);
  if (j < 0 || int64_t(j) << p.lpage >= n) return false;
  w.t0 = j << p.lpage;
  w.n = min(n - w.t0, page);
  w.row0 = r0 + w.t0;
  const int s0 = p.start[lo];
  w.first = int64_t(s0) + w.t0;
  const int64_t pj = w.first >> p.lpage;
  w.id = s0 >= 0 && (s0 & (page - 1)) == 0 && pj < p.max_to ? p.to[lo * p.to_st + pj] : -1;
  if (w.id >= 0 && w.id < p.num_pages) return true;
  if (lead) report_bad_index(STATUS_COMPACT);
  return false;
}

// Where token t of the piece lies: its page's first (page, K / V, head) slot for head 0 of K and the row in it; -1 where it
// cannot be read. pos: its old position.
__device__ __forceinline__ int64_t compact_slot(const CompactParams& p, const CompactPiece& w, int t, int& pos) {
  pos = p.keep[w.row0 + t];
  const int j = pos >> p.lpage;
  const int id = pos >= 0 && j < p.max_pages ? p.table[w.b * p.table_st + j] : -1;
  if (id < 0 || id >= p.num_pages) {
    report_bad_index(STATUS_COMPACT);
    return -1;
  }
  return int64_t(id) * 2 * p.Hkv;
}

// Any number of rotated dims: an element at a time, walked twice.
__global__ void __launch_bounds__(128) compact_any_kernel(const CompactParams p) {
  __shared__ float red[4];
  CompactPiece w;
  if (!compact_piece(p, blockIdx.x, w)) return;
  const int kind = blockIdx.y & 1, h = blockIdx.y >> 1, D = p.D, page = 1 << p.lpage;
  const int rot = kind == 0 ? p.R : 0, R2 = rot >> 1, cnt = w.n * D;
  auto value = [&](int i) {
    const int t = i / D, d = i - t * D;
    int pos;
    const int64_t s = compact_slot(p, w, t, pos);
    if (s < 0) return 0.f;
    const int64_t slot = s + kind * p.Hkv + h;
    const uint8_t* x = p.pages + (slot * page + (pos & (page - 1))) * D;
    const float scale = p.scales[slot];
    auto held = [&](int e) {
      uint32_t lo, hi;
      dec4(x[e], lo, hi);
      return half2_f(lo).x * scale;
    };
    const float v = held(d);
    if (d >= rot) return v;
    int f, o;
    float sg;
    if (p.interleaved) {
      f = d >> 1, o = d ^ 1, sg = d & 1 ? 1.f : -1.f;
    } else {
      f = d < R2 ? d : d - R2, o = d < R2 ? d + R2 : d - R2, sg = d < R2 ? -1.f : 1.f;
    }
    const float2 z = rope::turn_cs(uint64_t(w.first + t - pos) * p.turns[f]);
    return v * z.x + sg * held(o) * z.y;
  };
  float m = 0.f;
  for (int i = threadIdx.x; i < cnt; i += 128) m = fmaxf(m, finite_abs(value(i)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float now = scale_of(m), inv = scale_inv(now);
  const int64_t slot = (int64_t(w.id) * 2 + kind) * p.Hkv + h;
  if (threadIdx.x == 0) p.scales[slot] = now;
  uint8_t* dst = p.pages + slot * page * D;
  for (int i = 4 * threadIdx.x; i < cnt; i += 4 * 128)
    *reinterpret_cast<uint32_t*>(dst + i) =
        enc4(value(i) * inv, value(i + 1) * inv, value(i + 2) * inv, value(i + 3) * inv);
}

}  // namespace kv8
}  // namespace lb2
