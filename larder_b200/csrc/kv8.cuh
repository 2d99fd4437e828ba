// The paged 8-bit KV cache: appending keys (rotated on the way) and values, and the codes' arithmetic.
//
// pages [num_pages, 2 (K, V), Hkv, page, D] e4m3 codes; scales [num_pages, 2, Hkv] fp32, one for each page and head of K
// and of V; table [B, max_pages] int32, a sequence's pages in order. A held value is code * scale. A scale is the least
// power of two s with max |x| <= 448 s over the page's tokens of that head (0 for none but zeros): dividing by it is
// exact, so a value is rounded once, to e4m3's 4 significant bits (a scale of max / 448 would use the top of the range a
// little better, but e4m3 keeps its relative precision down to 2^-15 of the top), and when a later token raises the page's
// scale the held codes are divided by a power of two: exact but for codes that reach e4m3's subnormals (below 2^-15 of the
// page's largest value). The result does not depend on how the tokens are cut into calls, but for those.
// Infinities are held as +-448 s, NaN as NaN; neither sets the scale.
#pragma once

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
// 1 / s of a scale (a power of two between 2^-126 and 2^121); 0 for 0.
__device__ __forceinline__ float scale_inv(float s) {
  return s > 0.f ? __uint_as_float((254u << 23) - __float_as_uint(s)) : 0.f;
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
  int interleaved;
  float amp;
};

constexpr int STATUS_APPEND = 110;  // a page id or position out of range (lb2_status)

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// One block a (page that a sequence's new tokens reach, head, K or V): the rows' largest magnitude after rotation, the
// page's new scale, held codes rescaled where it grew, the new rows' codes. Rows are walked twice (the second time from
// L1 / L2).
template <typename T>
__global__ void __launch_bounds__(128) append_kernel(const AppendParams p) {
  __shared__ float red[4];
  const int kind = blockIdx.y & 1, h = blockIdx.y >> 1;
  int b, j;
  {
    b = blockIdx.x / p.touched;
    j = blockIdx.x - b * p.touched;
  }
  const int n0 = p.start[b];
  const int r0 = p.cu ? p.cu[b] : 0;
  const int n = p.cu ? min(p.cu[b + 1], p.T) - r0 : p.lens ? min(p.lens[b], p.T) : p.T;
  if (n <= 0 || n0 < 0 || r0 < 0) return;
  const int64_t pj = int64_t(n0 / p.page) + j;  // the sequence's page
  const int64_t base = pj * p.page;
  if (base >= int64_t(n0) + n) return;
  const int lo = int(max(int64_t(n0) - base, int64_t(0)));                      // first new row of the page
  const int hi = int(min(int64_t(n0) + n - base, int64_t(p.page)));             // past the last
  const int id = pj < p.max_pages ? p.table[b * p.table_st + pj] : -1;
  if (id < 0 || id >= p.num_pages) {
    if (threadIdx.x == 0) report_bad_index(STATUS_APPEND);
    return;
  }
  const T* x = static_cast<const T*>(p.x[kind]) + (p.cu ? 0 : b * p.st[kind][0]) + h * p.st[kind][1];
  const int64_t row0 = int64_t(r0) + (base + lo - n0);  // source row of page row lo
  const int rot = kind == 0 ? p.R : 0, R2 = rot >> 1;
  const int D = p.D, cnt = (hi - lo) * D;
  auto value = [&](int i) {
    const int r = i / D, d = i - r * D;
    const T* xr = x + (row0 + r) * p.st[kind][2];
    const float v = to_f<T>(xr[d]);
    if (d >= rot) return v;
    int f, o;
    float sg;
    if (p.interleaved) {
      f = d >> 1, o = d ^ 1, sg = d & 1 ? 1.f : -1.f;
    } else {
      f = d < R2 ? d : d - R2, o = d < R2 ? d + R2 : d - R2, sg = d < R2 ? -1.f : 1.f;
    }
    const float2 z = rope::turn_cs(uint64_t(base + lo + r) * p.turns[f]);
    return p.amp * (v * z.x + sg * to_f<T>(xr[o]) * z.y);
  };
  float m = 0.f;
  for (int i = threadIdx.x; i < cnt; i += 128) m = fmaxf(m, finite_abs(value(i)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const int64_t slot = (int64_t(id) * 2 + kind) * p.Hkv + h;
  const float was = lo > 0 ? p.scales[slot] : 0.f;
  const float now = fmaxf(was, scale_of(m));
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) p.scales[slot] = now;
  uint8_t* dst = p.pages + slot * int64_t(p.page) * D;
  const float inv = scale_inv(now);
  if (now != was && was > 0.f) {
    const float ratio = was * inv;
    for (int i = threadIdx.x; i < lo * D / 4; i += 128) {
      uint32_t a, c;
      dec4(reinterpret_cast<uint32_t*>(dst)[i], a, c);
      const float2 f = half2_f(a), g = half2_f(c);
      reinterpret_cast<uint32_t*>(dst)[i] = enc4(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
    }
  }
  for (int i = 4 * threadIdx.x; i < cnt; i += 4 * 128)
    *reinterpret_cast<uint32_t*>(dst + lo * D + i) =
        enc4(value(i) * inv, value(i + 1) * inv, value(i + 2) * inv, value(i + 3) * inv);
}

}  // namespace kv8
}  // namespace lb2
