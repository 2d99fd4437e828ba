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

// HBM-bound: a page is read once and written once, 16 KB a block, every thread's four loads in flight before its stores.
constexpr int COPY_THREADS = 256, COPY_HELD = 4;

__global__ void __launch_bounds__(COPY_THREADS) copy_kernel(const CopyParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int i = blockIdx.y;
  const int s = p.src[i], d = p.dst[i];
  if (s < 0 || s >= p.from_num || d < 0 || d >= p.to_num) {
    if (threadIdx.x == 0 && blockIdx.x == 0) report_bad_index(STATUS_COPY);
    return;
  }
  const uint4* x = reinterpret_cast<const uint4*>(p.from + s * p.bytes);
  uint4* y = reinterpret_cast<uint4*>(p.to + d * p.bytes);
  const int end = int(p.bytes / 16), at = blockIdx.x * (COPY_THREADS * COPY_HELD) + threadIdx.x;
  uint4 v[COPY_HELD];
#pragma unroll
  for (int k = 0; k < COPY_HELD; ++k)
    if (at + k * COPY_THREADS < end) v[k] = x[at + k * COPY_THREADS];
#pragma unroll
  for (int k = 0; k < COPY_HELD; ++k)
    if (at + k * COPY_THREADS < end) y[at + k * COPY_THREADS] = v[k];
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
  int hpb;    // heads a block takes in turn
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
  asm volatile("griddepcontrol.wait;" ::: "memory");
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

// Rotated dims in whole units of 16. A block takes a page of K or of V and p.hpb heads in turn; a thread holds U units, a unit
// being 16 of a token's dims whose partners under the rotation lie in it too: 8 dims and the 8 that they are paired with (half
// layout), or 16 in a row. So the codes are read once, the angles of a page are formed once for the block's heads, and
// between the two the page's largest magnitude is found in registers; the next head's codes are on their way meanwhile.
template <int THREADS, int U, int D>
__global__ void __launch_bounds__(THREADS) compact_kernel(const CompactParams p) {
  constexpr int UPR = D / 16;  // units a token
  __shared__ uint32_t red[2][THREADS / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  CompactPiece w;
  if (!compact_piece(p, blockIdx.x, w)) return;
  const int groups = (p.Hkv + p.hpb - 1) / p.hpb, kind = blockIdx.y >= groups;
  const int h0 = (int(blockIdx.y) - kind * groups) * p.hpb, h1 = min(h0 + p.hpb, p.Hkv);
  const int page = 1 << p.lpage, tid = threadIdx.x, turned = kind == 0 ? p.R / 16 : 0;
  const int64_t head = int64_t(page) * D;  // codes of a head's page
  const uint8_t* src[U];                   // the unit's codes of head h0 (null: nothing to read)
  const float* sc[U];
  int a0[U], a1[U], pos[U];                // where its two halves lie in a row; its old position
  int64_t dst[U];
  bool live[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int x = i * THREADS + tid, t = x / UPR, q = x % UPR;
    live[i] = t < w.n;
    a0[i] = 16 * q, a1[i] = 16 * q + 8;
    if (q < turned && !p.interleaved) a0[i] = 8 * q, a1[i] = p.R / 2 + 8 * q;
    src[i] = nullptr;
    sc[i] = nullptr;
    pos[i] = 0;
    if (live[i]) {
      const int64_t s = compact_slot(p, w, t, pos[i]);
      if (s >= 0) {
        const int64_t slot = s + kind * p.Hkv + h0;
        src[i] = p.pages + slot * head + (pos[i] & (page - 1)) * D;
        sc[i] = p.scales + slot;
      }
    }
    dst[i] = ((int64_t(w.id) * 2 + kind) * p.Hkv + h0) * head + t * D;
  }
  uint2 c[U][2];
  float f[U];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      c[i][0] = c[i][1] = make_uint2(0, 0);
      f[i] = 0.f;
      if (src[i]) {
        const uint8_t* x = src[i] + (h - h0) * head;
        c[i][0] = *reinterpret_cast<const uint2*>(x + a0[i]);
        c[i][1] = *reinterpret_cast<const uint2*>(x + a1[i]);
        f[i] = sc[i][h - h0];
      }
    }
  };
  load(h0);
  float2 z[U][8];  // the unit's angles
  if (turned) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int x = i * THREADS + tid, t = x / UPR, q = x % UPR;
      if (!live[i] || q >= turned) continue;
      const uint64_t by = uint64_t(w.first + t - pos[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[i][e] = rope::turn_cs(by * p.turns[8 * q + e]);
    }
  }
  for (int h = h0; h < h1; ++h) {
    float y[U][16];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t lo, hi;
          dec4(e ? c[i][k].y : c[i][k].x, lo, hi);
          const float2 a = half2_f(lo), b = half2_f(hi);
          float* o = y[i] + 8 * k + 4 * e;
          o[0] = a.x * f[i], o[1] = a.y * f[i], o[2] = b.x * f[i], o[3] = b.y * f[i];
        }
    }
    if (h + 1 < h1) load(h + 1);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (turned && (i * THREADS + tid) % UPR < turned) {
        auto turn = [](float& a, float& b, float2 z) {
          const float x = a;
          a = x * z.x - b * z.y;
          b = b * z.x + x * z.y;
        };
        if (p.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) turn(y[i][2 * e], y[i][2 * e + 1], z[i][e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) turn(y[i][e], y[i][8 + e], z[i][e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e += 2) m = max3_abs(m, y[i][e], y[i][e + 1]);  // (NaN is passed over)
    }
    if (m == INFINITY) {  // rare: held infinities of a page whose scale is near fp32's end
      m = 0.f;
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, finite_abs(y[i][e]));
    }
    const int turn = (h - h0) & 1;
    const uint32_t wm = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    if ((tid & 31) == 0) red[turn][tid >> 5] = wm;
    __syncthreads();
    uint32_t all = red[turn][0];
#pragma unroll
    for (int k = 1; k < THREADS / 32; ++k) all = max(all, red[turn][k]);
    const float now = scale_of(__uint_as_float(all)), inv = scale_inv(now);
    if (tid == 0) p.scales[(int64_t(w.id) * 2 + kind) * p.Hkv + h] = now;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (!live[i]) continue;
      uint8_t* o = p.pages + dst[i] + (h - h0) * head;
      uint2 e[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float* v = y[i] + 8 * k;
        e[k] = make_uint2(enc4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv), enc4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
      }
      *reinterpret_cast<uint2*>(o + a0[i]) = e[0];
      *reinterpret_cast<uint2*>(o + a1[i]) = e[1];
    }
  }
}

}  // namespace kv8
}  // namespace lb2
