// Pages of the paged 8-bit cache (kv8.cuh) moved about: whole pages copied, and sequences compacted to the tokens kept.
#pragma once

#include <cfloat>

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

// HBM-bound: a page is read once and written once, 16 KB a block, every thread's four loads in flight before its stores. 4000
// pages of 131 KB into another pool take 156 us, 6.71 TB/s; four pages 7 us a call, nearly all of it the host's.
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
  int planes;  // (K or V, head) pairs a block takes
};

// The page that block piece i writes: of sequence b, its moved tokens [t0, t0 + n), into page `id` (out of range: none).
struct CompactPiece {
  int b, t0, n, id;
  int64_t first;  // position of the page's first token
  int row0;       // index of token t0 in keep
};

// Sequence b's pieces start at cu[b] / page + b, which leaves room for its pages (n tokens fill at most n / page + 1).
__device__ __forceinline__ bool compact_piece(const CompactParams& p, int i, CompactPiece& w) {
  auto base = [&](int c, int s) { return (min(max(c, 0), p.T) >> p.lpage) + s; };
  const int lane = threadIdx.x & 31;
  int lo = 0, c0, c1, s0;
  if (p.B < 32) {  // a lane a sequence: one round of loads
    const int c = p.cu[min(lane, p.B)], s = p.start[min(lane, p.B - 1)];
    lo = 31 - __clz(__ballot_sync(0xffffffffu, lane < p.B && (lane == 0 || base(c, lane) <= i)));
    c0 = __shfl_sync(0xffffffffu, c, lo), c1 = __shfl_sync(0xffffffffu, c, lo + 1), s0 = __shfl_sync(0xffffffffu, s, lo);
  } else {
    int hi = p.B;  // base(lo) <= i, and base(hi) > i or hi == B
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, s = lo + lane * step;
      const uint32_t le = __ballot_sync(0xffffffffu, s < hi && (s == lo || base(p.cu[s], s) <= i));
      const int k = 31 - __clz(le);
      lo += k * step;
      hi = min(hi, lo + step);
    }
    c0 = p.cu[lo], c1 = p.cu[lo + 1], s0 = p.start[lo];
  }
  w.b = lo;
  const int j = i - base(c0, lo), page = 1 << p.lpage, r0 = min(max(c0, 0), p.T), n = min(max(c1, r0), p.T) - r0;
  const bool lead = threadIdx.x == 0;
  if (lead && j == 0 && (c0 != r0 || c1 != r0 + n)) report_bad_index(STATUS_COMPACT);
  if (j < 0 || int64_t(j) << p.lpage >= n) return false;
  w.t0 = j << p.lpage;
  w.n = min(n - w.t0, page);
  w.row0 = r0 + w.t0;
  w.first = int64_t(s0) + w.t0;
  const int64_t pj = w.first >> p.lpage;
  w.id = s0 >= 0 && (s0 & (page - 1)) == 0 && pj < p.max_to ? p.to[lo * p.to_st + pj] : -1;
  return true;
}

// (Apart from the search: the loads of the page id and of the tokens' positions then run at once.)
__device__ __forceinline__ bool compact_page(const CompactParams& p, const CompactPiece& w) {
  if (w.id >= 0 && w.id < p.num_pages) return true;
  if (threadIdx.x == 0) report_bad_index(STATUS_COMPACT);
  return false;
}

// The first (page, K / V, head) slot of the page that holds sequence b's position; -1 where it cannot be read.
__device__ __forceinline__ int64_t compact_slot(const CompactParams& p, int b, int pos) {
  const int j = pos >> p.lpage;
  const int id = pos >= 0 && j < p.max_pages ? p.table[b * p.table_st + j] : -1;
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
  if (!compact_piece(p, blockIdx.x, w) || !compact_page(p, w)) return;
  const int kind = blockIdx.y & 1, h = blockIdx.y >> 1, D = p.D, page = 1 << p.lpage;
  const int rot = kind == 0 ? p.R : 0, R2 = rot >> 1, cnt = w.n * D;
  auto value = [&](int i) {
    const int t = i / D, d = i - t * D;
    const int pos = p.keep[w.row0 + t];
    const int64_t s = compact_slot(p, w.b, pos);
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

// (cos, sin) of `frac` 2^-64 turns, from its upper 32 bits: the nearest quarter turn, and Taylor's series on the rest, |x| <=
// pi / 4: to x^9 and x^8, which leave out 2e-9 and 3e-8. Half the instructions of sincospi, which set the kernel's pace.
__device__ __forceinline__ float2 quarter_cs(uint64_t frac) {
  const uint32_t hi = uint32_t(frac >> 32), q = (hi + 0x20000000u) >> 30;
  const float x = float(int32_t(hi - (q << 30))) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float x2 = x * x;
  float s = fmaf(x2, 1.f / 362880.f, -1.f / 5040.f);
  s = fmaf(x2, s, 1.f / 120.f);
  s = fmaf(x2, s, -1.f / 6.f);
  s = fmaf(x * x2, s, x);
  float c = fmaf(x2, 1.f / 40320.f, -1.f / 720.f);
  c = fmaf(x2, c, 1.f / 24.f);
  c = fmaf(x2, c, -0.5f);
  c = fmaf(x2, c, 1.f);
  const float a = q & 1 ? s : c, b = q & 1 ? c : s;
  return make_float2(__uint_as_float(__float_as_uint(a) ^ (((q + 1) & 2) << 30)), __uint_as_float(__float_as_uint(b) ^ ((q & 2) << 30)));
}

// The largest finite magnitude of 16 codes times f.
__device__ __noinline__ float held_max(uint2 a, uint2 b, float f) {
  float m = 0.f;
  for (int k = 0; k < 4; ++k) {
    uint32_t lo, hi;
    dec4(k == 0 ? a.x : k == 1 ? a.y : k == 2 ? b.x : b.y, lo, hi);
    const float2 x = half2_f(lo), y = half2_f(hi);
    m = fmaxf(fmaxf(m, fmaxf(finite_abs(x.x * f), finite_abs(x.y * f))), fmaxf(finite_abs(y.x * f), finite_abs(y.y * f)));
  }
  return m;
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Four codes times r, to the nearest codes.
__device__ __forceinline__ uint32_t times(uint32_t c, __half2 r) {
  uint32_t lo, hi, x;
  dec4(c, lo, hi);
  const __half2 a = __hmul2(*reinterpret_cast<__half2*>(&lo), r), b = __hmul2(*reinterpret_cast<__half2*>(&hi), r);
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f16x2 lo, %1;\n\tcvt.rn.satfinite.e4m3x2.f16x2 hi, %2;\n\tmov.b32 %0, {lo, hi};\n\t}"
      : "=r"(x)
      : "r"(*reinterpret_cast<const uint32_t*>(&a)), "r"(*reinterpret_cast<const uint32_t*>(&b)));
  return x;
}

// Rotated dims in whole units of 16. A block takes a page of p.planes (K or V, head) pairs; a thread holds U units of each,
// a unit being 16 of a token's dims whose partners under the rotation lie in it too: 8 dims and the 8 that they are
// paired with (half layout), or 16 in a row. So the codes are read once, the angles of a page are formed once for the block's
// heads, and the page's largest magnitude is found in between.
// A block begins with a chain of four loads (bounds, positions, pages, codes), some 4 us, and needs few instructions after it:
// what counts is the bytes in flight, so H planes' codes are asked for at once, and one barrier serves their maxima. Half of 16 x
// up to 8192 tokens of 4 heads x 128 (pages of 32, interleaved turns) take 35 us, 3.0 TB/s, with conversions on half of the ALU's
// time (a plane at a time 44, both layouts in one kernel 39 to 45); two thirds of 3 x up to 16390 of 2 x 256 17 us (25 with 90
// registers a thread, one block an SM).
template <int THREADS, int U, int H, int D, int LAYOUT>  // LAYOUT: 0 no turns, 1 halves, 2 interleaved
__global__ void __launch_bounds__(THREADS, !LAYOUT ? 1024 / THREADS : U == 1 ? 768 / THREADS : 1) compact_kernel(const CompactParams p) {
  constexpr int UPR = D / 16, WARPS = THREADS / 32;
  constexpr bool TURN = LAYOUT != 0;
  __shared__ uint32_t red[2][H][WARPS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  CompactPiece w;
  if (!compact_piece(p, blockIdx.x, w)) return;
  const int l0 = blockIdx.y * p.planes, l1 = min(l0 + p.planes, 2 * p.Hkv);
  const int page = 1 << p.lpage, tid = threadIdx.x, turned = TURN && l0 < p.Hkv ? p.R / 16 : 0;
  const int head = page * D;  // codes of a plane of a page
  int pos[U];
#pragma unroll
  for (int i = 0; i < U; ++i) pos[i] = (i * THREADS + tid) / UPR < w.n ? p.keep[w.row0 + (i * THREADS + tid) / UPR] : 0;
  if (!compact_page(p, w)) return;
  const uint8_t* src[U];  // the unit's codes of plane 0 (null: nothing to read)
  const float* sc[U];
  int at[U], by[U];       // where the unit's first half lies in a plane of K; how far the second one is from it
  int more[U];            // and how far on the unit lies in a plane of V
  bool live[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int x = i * THREADS + tid, t = x / UPR, q = x % UPR;
    live[i] = t < w.n;
    const bool halves = LAYOUT == 1 && q < turned;
    const int d0 = halves ? 8 * q : 16 * q;
    by[i] = halves ? p.R / 2 : 8;
    at[i] = t * D + d0;
    more[i] = 16 * q - d0;
    src[i] = nullptr;
    sc[i] = nullptr;
    if (live[i]) {
      const int64_t slot = compact_slot(p, w.b, pos[i]);
      if (slot >= 0) {
        src[i] = p.pages + slot * head + (pos[i] & (page - 1)) * D + d0;
        sc[i] = p.scales + slot;
      }
    }
  }
  uint2 c[H][U][2];
  float f[H][U];
  float2 zc[TURN ? U : 1][4], zs[TURN ? U : 1][4];  // the unit's angles: cosines and sines of pairs 2 e, 2 e + 1
  // a turned unit's codes as values, turned (its scale is left out: a power of two); in pairs y[e], y[4 + e] of what is turned
  // together, each two neighbours
  auto values = [&](const uint2* x, int i, bool turn_it, float2* y) {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 2; ++k) dec4(x[k].x, w[4 * k], w[4 * k + 1]), dec4(x[k].y, w[4 * k + 2], w[4 * k + 3]);
    constexpr bool mixed = LAYOUT == 2;  // two neighbours are a pair
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = half2_f(w[mixed ? 2 * e : e]), b = half2_f(w[mixed ? 2 * e + 1 : 4 + e]);
      y[e] = mixed ? make_float2(a.x, b.x) : a;
      y[4 + e] = mixed ? make_float2(a.y, b.y) : b;
    }
    if (!TURN || !turn_it || (i * THREADS + tid) % UPR >= turned) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 c = zc[TURN ? i : 0][e], s = zs[TURN ? i : 0][e], a = y[e], b = y[4 + e];
      y[e] = fma2(a, c, mul2(b, make_float2(-s.x, -s.y)));
      y[4 + e] = fma2(b, c, mul2(a, s));
    }
  };
  int round = 0;
#pragma unroll 1
  for (int l = l0; l < l1; l += H, round ^= 1) {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < U; ++i) {
        c[h][i][0] = c[h][i][1] = make_uint2(0, 0);
        f[h][i] = 0.f;
        if (src[i] && l + h < l1) {
          // (K's planes hold units as they are turned, V's 16 dims in a row)
          const bool v = l + h >= p.Hkv;
          const uint8_t* x = src[i] + int64_t(l + h) * head + (v ? more[i] : 0);
          c[h][i][0] = *reinterpret_cast<const uint2*>(x);
          c[h][i][1] = *reinterpret_cast<const uint2*>(x + (v ? 8 : by[i]));
          f[h][i] = sc[i][l + h];
        }
      }
    if (TURN && turned && l == l0) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int x = i * THREADS + tid, q = x % UPR;
        if (!live[i] || q >= turned) continue;
        const uint64_t shift = uint64_t(w.first + x / UPR - pos[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = quarter_cs(shift * p.turns[8 * q + 2 * e]), b = quarter_cs(shift * p.turns[8 * q + 2 * e + 1]);
          zc[TURN ? i : 0][e] = make_float2(a.x, b.x), zs[TURN ? i : 0][e] = make_float2(a.y, b.y);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const bool turn_it = TURN && turned && l + h < p.Hkv;
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        float mi = 0.f;
        if (turn_it) {
          float2 y[8];
          values(c[h][i], i, true, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) mi = max3_abs(mi, y[e].x, y[e].y);  // (NaN is passed over)
        } else {  // codes rise with their magnitudes
          uint32_t m2 = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t u = k & 1 ? c[h][i][k >> 1].y : c[h][i][k >> 1].x;
            m2 = max_u16x2(m2, max_u16x2(u & 0x7f007f00u, u << 8 & 0x7f007f00u));
          }
          const uint32_t top = max(m2 >> 16, m2 & 0xffffu);
          uint32_t lo, hi;
          dec4(top >> 8, lo, hi);
          mi = top == 0x7f00u ? INFINITY : half2_f(lo).x;  // (NaN codes: looked at again)
        }
        mi *= f[h][i];
        if (!(mi < INFINITY)) mi = held_max(c[h][i][0], c[h][i][1], f[h][i]);  // rare: NaN, or infinities near fp32's end
        m = fmaxf(m, mi);
      }
      const uint32_t wm = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
      if ((tid & 31) == 0) red[round][h][tid >> 5] = wm;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (l + h >= l1) break;
      const bool turn_it = TURN && turned && l + h < p.Hkv;
      uint32_t all = red[round][h][0];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) all = max(all, red[round][h][k]);
      const float now = scale_of(__uint_as_float(all)), inv = scale_inv(now);
      const int64_t slot = int64_t(w.id) * 2 * p.Hkv + l + h;
      if (tid == 0) p.scales[slot] = now;
      uint8_t* out = p.pages + slot * head;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (!live[i]) continue;
        const float r = f[h][i] * inv;  // what the codes are multiplied by
        uint2 e[2];
        if (turn_it || !(r <= 32768.f) || (__float_as_uint(f[h][i]) & 0x7fffffu) != 0) {
          float2 y[8];
          values(c[h][i], i, turn_it, y);
          // (past fp32's range only where all codes are zeros or NaN: zeros stay zeros)
          const float rf = r > FLT_MAX ? FLT_MAX : r;
          const float2 r2 = make_float2(rf, rf);
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = mul2(y[e], r2);
          if (LAYOUT == 2) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              e[k] = make_uint2(enc4(y[2 * k].x, y[4 + 2 * k].x, y[2 * k].y, y[4 + 2 * k].y),
                                enc4(y[2 * k + 1].x, y[5 + 2 * k].x, y[2 * k + 1].y, y[5 + 2 * k].y));
          } else {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              e[k] = make_uint2(enc4(y[4 * k].x, y[4 * k].y, y[4 * k + 1].x, y[4 * k + 1].y),
                                enc4(y[4 * k + 2].x, y[4 * k + 2].y, y[4 * k + 3].x, y[4 * k + 3].y));
          }
        } else if (r == 1.f) {
          e[0] = c[h][i][0], e[1] = c[h][i][1];
        } else {
          // a power of two times a code in f16: exact down to 2^-21, and below 2^-10 every code is 0
          const __half2 r2 = __float2half2_rn(r);
#pragma unroll
          for (int k = 0; k < 2; ++k) e[k] = make_uint2(times(c[h][i][k].x, r2), times(c[h][i][k].y, r2));
        }
        const bool v = l + h >= p.Hkv;
        const int o = at[i] + (v ? more[i] : 0);
        *reinterpret_cast<uint2*>(out + o) = e[0];
        *reinterpret_cast<uint2*>(out + o + (v ? 8 : by[i])) = e[1];
      }
    }
  }
}

}  // namespace kv8
}  // namespace lb2
