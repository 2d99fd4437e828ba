// The paged 8-bit KV cache: appending keys (rotated on the way) and values, and the codes' arithmetic.
//
// pages [num_pages, 2 (K, V), Hkv, page, D] e4m3 codes; scales [num_pages, 2, Hkv] fp32, one for each page and head of K
// and of V; table [B, max_pages] int32, a sequence's pages in order. A held value is code * scale. A scale is the least
// power of two s with max |x| <= 448 s over the page's tokens of that head (0 for none but zeros): dividing by it is
// exact, so a value is rounded once, to e4m3's 4 significant bits (a scale of max / 448 would use the top of the range a
// little better, but e4m3 keeps its relative precision down to 2^-15 of the top), and when a later token raises the page's
// scale the held codes are divided by a power of two: exact but for codes that reach e4m3's subnormals (below 2^-15 of the
// page's largest value). The result does not depend on how the tokens are cut into calls, but for those.
// Infinities are held as +-448 s (of the call that brings them, or the first scale but 0), NaN as NaN; neither sets the scale.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "rope.cuh"

namespace lb2 {
namespace kv8 {

constexpr float CODE_MAX = 448.f;

// Four floats -> four e4m3 codes (x[0] in the low byte), to nearest even, saturating.
__device__ __forceinline__ uint32_t enc4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// Four codes -> two f16 pairs: (c0, c1) and (c2, c3). Every e4m3 value is an f16 value.
__device__ __forceinline__ void dec4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float2 half2_f(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// The scale of a largest magnitude (>= 0, finite): the least power of two s >= 2^-126 with m <= 448 s; 0 for m = 0.
__device__ __forceinline__ float scale_of(float m) {
  if (!(m > 0.f)) return 0.f;
  const uint32_t u = __float_as_uint(m);
  const int e = int(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return __uint_as_float(uint32_t(max(e, 1)) << 23);
}
// What values are multiplied by before they are rounded to codes: 1 / s of a scale (a power of two between 2^-126 and
// 2^121). For 0, where every finite value is 0, it is 1: infinities then saturate as anywhere else (times 0 they were NaN).
__device__ __forceinline__ float scale_inv(float s) {
  return s > 0.f ? __uint_as_float((254u << 23) - __float_as_uint(s)) : 1.f;
}

struct AppendParams {
  uint8_t* pages;
  float* scales;
  const int32_t* table;
  int64_t table_st;
  const void* x[2];   // k, v [B, Hkv, T, D] (packed: [1, Hkv, rows, D])
  int64_t st[2][3];   // B, H, T
  const int32_t* start;
  const int32_t* lens;  // new tokens of each sequence, or nullptr: T each
  const int32_t* cu;    // packed: rows [cu[b], cu[b + 1]) are b's, or nullptr
  const uint64_t* turns;
  int B, Hkv, T, D, R, page, num_pages, max_pages, touched;
  int lpage, lupr;  // log2 of page and of a row's units (D / 16)
  int hpb;          // heads a block takes in turn
  int interleaved;
  float amp;
};

constexpr int STATUS_APPEND = 110;  // a page id or position out of range (lb2_status)

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// The sequence and page (b, j-th page that its new tokens reach) of block i. With T tokens each there are `touched` blocks
// a sequence. Packed, sequence b's blocks start at cu[b] / page + 2 b, which leaves room for every page its tokens can
// reach at any alignment (n tokens touch at most n / page + 2): a 32-way search, each warp for itself.
__device__ __forceinline__ bool find_page(const AppendParams& p, int i, int& b, int& j) {
  if (!p.cu) {
    b = p.touched == 1 ? i : i / p.touched;
    j = i - b * p.touched;
    return true;
  }
  auto base = [&](int s) { return (min(max(p.cu[s], 0), p.T) >> p.lpage) + 2 * s; };
  int lo = 0, hi = p.B;  // base(lo) <= i, and base(hi) > i or hi == B
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, s = lo + (threadIdx.x & 31) * step;
    const uint32_t le = __ballot_sync(0xffffffffu, s < hi && (s == lo || base(s) <= i));
    const int k = 31 - __clz(le);
    lo += k * step;
    hi = min(hi, lo + step);
  }
  b = lo;
  j = i - base(lo);
  return j >= 0;
}

// One block's work: a page of sequence b that its new tokens reach, K or V, of heads h on.
struct Piece {
  int b, h, kind;
  int lo, hi;       // the page's new rows
  int id;           // physical page, or out of range
  int64_t base;     // position of the page's first token
  int64_t row0;     // source row of page row lo
  int64_t slot;     // (page, K / V, head) index of the scale
};

__device__ __forceinline__ bool piece_of(const AppendParams& p, Piece& w) {
  // K / V and the head groups vary fastest, so that the blocks that run together read whole token rows
  const int groups = (p.Hkv + p.hpb - 1) / p.hpb, i = blockIdx.x / (2 * groups), g = blockIdx.x - i * 2 * groups;
  w.kind = g >= groups;
  w.h = (g - w.kind * groups) * p.hpb;
  int j;
  if (!find_page(p, i, w.b, j)) return false;
  const int n0 = p.start[w.b];
  const int r0 = p.cu ? p.cu[w.b] : 0;
  const int n = p.cu ? min(p.cu[w.b + 1], p.T) - r0 : p.lens ? min(p.lens[w.b], p.T) : p.T;
  if (n <= 0 || n0 < 0 || r0 < 0) return false;
  const int64_t pj = int64_t(n0 >> p.lpage) + j;  // the sequence's page
  w.base = pj << p.lpage;
  if (w.base >= int64_t(n0) + n) return false;
  w.lo = int(max(int64_t(n0) - w.base, int64_t(0)));
  w.hi = int(min(int64_t(n0) + n - w.base, int64_t(p.page)));
  w.row0 = int64_t(r0) + (w.base + w.lo - n0);
  w.id = pj < p.max_pages ? p.table[w.b * p.table_st + pj] : -1;
  w.slot = (int64_t(w.id) * 2 + w.kind) * p.Hkv + w.h;
  return true;
}

__device__ __forceinline__ bool bad_page(const AppendParams& p, const Piece& w) {
  if (w.id >= 0 && w.id < p.num_pages) return false;
  if (threadIdx.x == 0) report_bad_index(STATUS_APPEND);
  return true;
}

// Rescales the page's held codes (rows before lo) where its scale grew from `was` to 1 / inv.
template <int THREADS>
__device__ __forceinline__ void rescale_held(uint8_t* dst, int bytes, float was, float now, float inv) {
  if (now == was || !(was > 0.f)) return;
  const float ratio = was * inv;
  for (int i = threadIdx.x; i < bytes / 16; i += THREADS) {
    uint4 w = reinterpret_cast<uint4*>(dst)[i];
    uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t a, c;
      dec4(u[e], a, c);
      const float2 f = half2_f(a), g = half2_f(c);
      u[e] = enc4(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
    }
    reinterpret_cast<uint4*>(dst)[i] = w;
  }
}

// Any strides, alignment and number of rotated dims: an element at a time, walked twice (the second time from L1 / L2).
template <typename T>
__global__ void __launch_bounds__(128) append_any_kernel(const AppendParams p) {
  __shared__ float red[4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Piece w;
  if (!piece_of(p, w) || bad_page(p, w)) return;
  const T* x = static_cast<const T*>(p.x[w.kind]) + (p.cu ? 0 : w.b * p.st[w.kind][0]) + w.h * p.st[w.kind][1];
  const int rot = w.kind == 0 ? p.R : 0, R2 = rot >> 1;
  const int D = p.D, cnt = (w.hi - w.lo) * D;
  auto value = [&](int i) {
    const int r = i / D, d = i - r * D;
    const T* xr = x + (w.row0 + r) * p.st[w.kind][2];
    const float v = to_f<T>(xr[d]);
    if (d >= rot) return v;
    int f, o;
    float sg;
    if (p.interleaved) {
      f = d >> 1, o = d ^ 1, sg = d & 1 ? 1.f : -1.f;
    } else {
      f = d < R2 ? d : d - R2, o = d < R2 ? d + R2 : d - R2, sg = d < R2 ? -1.f : 1.f;
    }
    const float2 z = rope::turn_cs(uint64_t(w.base + w.lo + r) * p.turns[f]);
    return p.amp * (v * z.x + sg * to_f<T>(xr[o]) * z.y);
  };
  float m = 0.f;
  for (int i = threadIdx.x; i < cnt; i += 128) m = fmaxf(m, finite_abs(value(i)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  const float was = w.lo > 0 ? p.scales[w.slot] : 0.f;
  __syncthreads();  // (every thread has read the old scale)
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float now = fmaxf(was, scale_of(m)), inv = scale_inv(now);
  if (threadIdx.x == 0) p.scales[w.slot] = now;
  uint8_t* dst = p.pages + w.slot * int64_t(p.page) * D;
  rescale_held<128>(dst, w.lo * D, was, now, inv);
  for (int i = 4 * threadIdx.x; i < cnt; i += 4 * 128)
    *reinterpret_cast<uint32_t*>(dst + w.lo * D + i) =
        enc4(value(i) * inv, value(i + 1) * inv, value(i + 2) * inv, value(i + 3) * inv);
}

// Two fp32 products, or products and sums, in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\t"
      "mov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// The largest magnitude of three (NaN is passed over).
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The largest finite magnitude of M loads of V values.
template <typename T, int V, int M>
__device__ __forceinline__ float max_raw(const rope::Raw<T, V>* r) {
  float mk = 0.f;
  if constexpr (sizeof(T) == 2) {  // two values an instruction (NaN is passed over)
    using V2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const V2* h = reinterpret_cast<const V2*>(r);
    V2 m2 = __habs2(h[0]);
#pragma unroll
    for (int e = 1; e < 4 * M; ++e) m2 = __hmax2(m2, __habs2(h[e]));
    mk = fmaxf(fmaxf(to_f<T>(m2.x), to_f<T>(m2.y)), 0.f);
  } else {
    const float* f = reinterpret_cast<const float*>(r);
#pragma unroll
    for (int e = 0; e < V * M; e += 2) mk = max3_abs(mk, f[e], f[e + 1]);
  }
  if (mk == INFINITY) {  // rare
    mk = 0.f;
#pragma unroll
    for (int g = 0; g < M; ++g) {
      float f[V];
      r[g].get(f);
#pragma unroll
      for (int e = 0; e < V; ++e) mk = fmaxf(mk, finite_abs(f[e]));
    }
  }
  return mk;
}

// Four codes straight from two words of 16-bit pairs. f16: x 2^k is exact in f16 (|x 2^k| <= 448; what falls under 2^-14
// rounds to code 0 either way) unless 2^k itself leaves f16's range.
template <typename T>
struct Pair {
  static __device__ __forceinline__ bool direct(float) { return false; }
  static __device__ __forceinline__ uint32_t enc4(uint32_t, uint32_t, float) { return 0; }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ bool direct(float inv) { return inv >= 0x1p-14f && inv <= 0x1p15f; }
  static __device__ __forceinline__ uint32_t enc4(uint32_t a, uint32_t b, float inv) {
    const __half2 k = __float2half2_rn(inv);
    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&a), k), y = __hmul2(*reinterpret_cast<const __half2*>(&b), k);
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f16x2 lo, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f16x2 hi, %2;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r)
        : "r"(*reinterpret_cast<const uint32_t*>(&x)), "r"(*reinterpret_cast<const uint32_t*>(&y)));
    return r;
  }
};

// Rows of 16-byte groups: the page's new rows are held in registers, read once. A unit is two groups of 8 elements: in
// the rotated half layout a group and its partners R / 2 on, elsewhere neighbours; a thread has one unit of K rows. The
// block takes `hpb` heads in turn, the next one's loads in flight while it works: the angles of its rows serve them all
// (in shared memory, each thread its own).
// Bound for long prompts by latency: 2 x 16384 tokens of 8 heads x 128 (f16) take 50 us, 4050 GB/s of the 2 bytes read and 1
// written a value, with half the issue slots used (49 %), no pipe above 35 % and 31 % of the warps resident, which wait for
// loads and at each head's barrier; the same loads and stores without rotation and conversion take 35 us. Two
// products an instruction (f32x2) and word-wise maxima keep a value of V at about 4 instructions, one of K at 7. Single
// tokens are bound by the chain start -> table -> scale (64 sequences: 3 us).
// Pages of 128 tokens at head dim 256 take 1024 threads of 64 registers, which spill (bytes stored / loaded: bf16 168 / 124,
// f16 168 / 156, fp32 480 / 348): 2 x 8192 tokens of 4 heads take 47 us in bf16 (2130 GB/s), 88 us in fp32 (1910). The 256
// threads of three blocks an SM have 80 and spill a little (32 / 36, 32 / 56, 252 / 176); the other forms spill nothing.
template <typename T, int THREADS, int K, int OCC = THREADS == 256 ? 3 : 1>
__global__ void __launch_bounds__(THREADS, OCC) append_kernel(const AppendParams p) {
  constexpr int WARPS = THREADS / 32;
  constexpr int V = 16 / int(sizeof(T)), N = 8 / V;  // values a load, loads a group
  extern __shared__ __align__(16) float4 zsm[];  // [4 K][THREADS]: each thread's angles, two cosines and their sines a word
  __shared__ __align__(16) uint32_t red[2][WARPS < 4 ? 4 : WARPS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Piece w;
  if (!piece_of(p, w)) return;
  const int D = p.D, u = threadIdx.x & ((1 << p.lupr) - 1), first = threadIdx.x >> p.lupr;
  const int rpp = THREADS >> p.lupr;
  const int mine = (w.hi - w.lo - first + rpp - 1) / rpp;  // rows of this thread (a unit each; <= 0 for none)
  const int rot = w.kind == 0 ? p.R : 0, R2 = rot >> 1;
  const bool half = !p.interleaved && u * 8 < R2;
  const int a = half ? u * 8 : u * 16, c = half ? a + R2 : a + 8;
  const bool turn = half || (p.interleaved && a < rot);  // (R is a multiple of 16: a unit is rotated whole or not at all)
  const int64_t hst = p.st[w.kind][1], tst = p.st[w.kind][2];
  const T* x = static_cast<const T*>(p.x[w.kind]) + (p.cu ? 0 : w.b * p.st[w.kind][0]) + w.h * hst +
               (w.row0 + first) * tst + a;  // this thread's first row
  const int64_t kst = rpp * tst;
  const int nh = min(p.hpb, p.Hkv - w.h);
  rope::Raw<T, V> next[K][2 * N];
  auto fetch = [&] {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k < mine)
#pragma unroll
        for (int g = 0; g < N; ++g) {
          next[k][g].load(x + k * kst + g * V);
          next[k][N + g].load(x + k * kst + (c - a) + g * V);
        }
  };
  fetch();
  if (bad_page(p, w)) return;  // (the same for every thread)
  float was = w.lo > 0 ? p.scales[w.slot] : 0.f;
  float4* zt = zsm + threadIdx.x;
  if (turn) {
    uint64_t f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = p.turns[half ? a + e : (a >> 1) + e];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k >= mine) break;
      const uint64_t pos = uint64_t(w.base + w.lo + first + k * rpp);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 a = rope::turn_cs(pos * f[2 * e]), b = rope::turn_cs(pos * f[2 * e + 1]);
        zt[(k * 4 + e) * THREADS] = make_float4(a.x * p.amp, b.x * p.amp, a.y * p.amp, b.y * p.amp);
      }
    }
  }
  uint8_t* page = p.pages + w.slot * (int64_t(D) << p.lpage);
  uint8_t* out = page + (w.lo + first) * D + a;  // this thread's first row
  const int page_bytes = D << p.lpage, held = w.lo * D;
  for (int i = 0; i < nh; ++i, page += page_bytes, out += page_bytes) {
    rope::Raw<T, V> raw[K][2 * N];  // the rows as they lie: what a unit that is not rotated is encoded from
    float2 y[K][8];                 // or rotated: the unit's two groups, two values a word
    uint32_t m = 0;                 // the largest finite magnitude, as the bits of a float
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k >= mine) break;
#pragma unroll
      for (int g = 0; g < 2 * N; ++g) raw[k][g] = next[k][g];
      float mk = 0.f;
      if (turn) {
#pragma unroll
        for (int g = 0; g < 2 * N; ++g) raw[k][g].get(reinterpret_cast<float*>(y[k]) + g * V);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 z = zt[(k * 4 + e) * THREADS];
          const float2 co = make_float2(z.x, z.y), si = make_float2(z.z, z.w), ns = make_float2(-z.z, -z.w);
          if (half) {  // partners in two words
            const float2 x0 = y[k][e], x1 = y[k][4 + e];
            y[k][e] = fma2(x1, ns, mul2(x0, co));
            y[k][4 + e] = fma2(x0, si, mul2(x1, co));
          } else {  // a pair a word: two words a step
            const float2 p0 = y[k][2 * e], p1 = y[k][2 * e + 1];
            const float2 x0 = make_float2(p0.x, p1.x), x1 = make_float2(p0.y, p1.y);
            const float2 y0 = fma2(x1, ns, mul2(x0, co)), y1 = fma2(x0, si, mul2(x1, co));
            y[k][2 * e] = make_float2(y0.x, y1.x);
            y[k][2 * e + 1] = make_float2(y0.y, y1.y);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) mk = max3_abs(mk, y[k][e].x, y[k][e].y);
        if (mk == INFINITY) {  // rare: the largest of the finite
          mk = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) mk = fmaxf(mk, fmaxf(finite_abs(y[k][e].x), finite_abs(y[k][e].y)));
        }
      } else {
        mk = max_raw<T, V, 2 * N>(raw[k]);
      }
      m = max(m, __float_as_uint(mk));
    }
    const float old = was;
    if (i + 1 < nh) {
      x += hst;
      fetch();
      if (w.lo > 0) was = p.scales[w.slot + i + 1];
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (WARPS > 1) {
      uint32_t* r = red[i & 1];  // (the other half may still be read by warps behind)
      if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = m;
      __syncthreads();  // (every thread has read the old scale)
      if constexpr (WARPS == 2) {
        m = max(r[0], r[1]);
      } else {
#pragma unroll
        for (int q = 0; q < WARPS; q += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(r + q);
          m = max(max(m, max(v.x, v.y)), max(v.z, v.w));
        }
      }
    } else {
      __syncwarp();
    }
    const float now = fmaxf(old, scale_of(__uint_as_float(m))), inv = scale_inv(now);
    if (threadIdx.x == 0) p.scales[w.slot + i] = now;
    if (held) rescale_held<THREADS>(page, held, old, now, inv);
    const float2 i2 = make_float2(inv, inv);
    const bool words = sizeof(T) == 2 && !turn && Pair<T>::direct(inv);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k >= mine) break;
      uint32_t code[4];
      if (words) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint4 v = raw[k][g * N].u;
          code[2 * g] = Pair<T>::enc4(v.x, v.y, inv);
          code[2 * g + 1] = Pair<T>::enc4(v.z, v.w, inv);
        }
      } else {
        if (!turn)
#pragma unroll
          for (int g = 0; g < 2 * N; ++g) raw[k][g].get(reinterpret_cast<float*>(y[k]) + g * V);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float2 s = mul2(y[k][2 * g], i2), t = mul2(y[k][2 * g + 1], i2);
          code[g] = enc4(s.x, s.y, t.x, t.y);
        }
      }
      uint8_t* d = out + k * rpp * D;
      if (half) {
        *reinterpret_cast<uint2*>(d) = make_uint2(code[0], code[1]);
        *reinterpret_cast<uint2*>(d + (c - a)) = make_uint2(code[2], code[3]);
      } else {
        *reinterpret_cast<uint4*>(d) = make_uint4(code[0], code[1], code[2], code[3]);
      }
    }
  }
}

}  // namespace kv8
}  // namespace lb2
