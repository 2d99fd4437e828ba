// Rotary positions: rotation of the first R of a head's D values by the row's position, pair i by the angle
// position * w_i, in the half layout (pairs i, i + R / 2) or the interleaved one (pairs 2 i, 2 i + 1):
//   y0 = amp (x0 cos - x1 sin),  y1 = amp (x1 cos + x0 sin),  dims from R on pass unchanged.
// The inverse negates the angle: with the same amp it is the gradient (the transposed map).
//
// The angles come as `turns`: F_i = round(2^64 w_i / 2 pi), 64-bit fractions of a turn. position * F_i in 64-bit
// wrap-around arithmetic is the angle's fraction of a turn, exact to position * 2^-65 turns, so that an angle keeps full
// fp32 accuracy at any position (position * w_i in fp32 is off by 0.004 radians at 100 000) and no table of positions is
// read. sincospi takes the reduced angle. Every scaling for long contexts is a choice of F_i and amp by the host.
//
// HBM-bound: a row is read once and written once. A block takes a few tokens and a group of their heads; it forms each
// token's R / 2 (cos, sin) pairs once, in shared memory, while the rows' first loads are in flight.
#pragma once

#include "common.cuh"

namespace lb2 {
namespace rope {

struct Params {
  const void* x;
  void* y;
  int64_t x_st[3], y_st[3];  // B, H, T
  const int32_t* pos;
  int64_t p_st;  // batch stride of pos (0: one row of positions for every b)
  const uint64_t* turns;
  int B, H, T, D, R;
  int interleaved, inverse;
  float amp;
  int tok, hg;  // tokens and heads a block takes
};

// (cos, sin) of `frac` 2^-64 turns.
__device__ __forceinline__ float2 turn_cs(uint64_t frac) {
  const float h = __ll2float_rn(static_cast<long long>(frac)) * 0x1p-63f;  // half turns, in [-1, 1]
  float s, c;
  sincospif(h, &s, &c);
  return make_float2(c, s);
}

constexpr int THREADS = 256;

// V elements a load (16 bytes, or one element for the strides, alignments and widths that 16 bytes do not fit).
template <typename T, int V>
struct Vec {
  T e[V];
};
template <typename T, int V>
__device__ __forceinline__ void ld_vec(const T* p, float* f) {
  if constexpr (V == 1) {
    f[0] = to_f<T>(p[0]);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f<T>(h[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void st_vec(T* p, const float* f) {
  if constexpr (V == 1) {
    p[0] = from_f<T>(f[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
}

// A unit is two groups of V elements: in the half layout's rotated part elements [V u, V u + V) and their partners
// R / 2 on; elsewhere two neighbouring groups, each with its pairs inside (V == 1 takes pairs too: (2 u, 2 u + 1)).
template <typename T, int V>
__global__ void __launch_bounds__(THREADS) rope_kernel(const Params p) {
  extern __shared__ float2 cs[];  // [tok][R / 2]
  const int R2 = p.R >> 1, upr = p.D / (2 * V);  // units a row
  const int ntok = p.B * p.T;                   // < 2^31: checked by the launcher
  const int tok0 = blockIdx.x * p.tok, h0 = blockIdx.y * p.hg;
  const int nt = min(p.tok, ntok - tok0), nh = min(p.hg, p.H - h0);
  for (int i = threadIdx.x; i < nt * R2; i += THREADS) {
    const int t = i / R2, f = i - t * R2;
    const int row = tok0 + t, b = row / p.T;
    const int64_t pos = p.pos[b * p.p_st + (row - b * p.T)];
    float2 c = turn_cs(uint64_t(pos) * p.turns[f]);
    c.x *= p.amp;
    c.y *= p.inverse ? -p.amp : p.amp;
    cs[i] = c;
  }
  __syncthreads();
  const int units = nt * nh * upr;
  for (int i = threadIdx.x; i < units; i += THREADS) {
    const int u = i % upr, th = i / upr, t = th % nt, h = h0 + th / nt;
    const int row = tok0 + t, b = row / p.T, s = row - b * p.T;
    const T* x = static_cast<const T*>(p.x) + b * p.x_st[0] + h * p.x_st[1] + s * p.x_st[2];
    T* y = static_cast<T*>(p.y) + b * p.y_st[0] + h * p.y_st[1] + s * p.y_st[2];
    const bool half = !p.interleaved && u * V < R2;
    const int a = half ? u * V : 2 * u * V, c = half ? a + R2 : a + V;
    float xa[V], xc[V];
    ld_vec<T, V>(x + a, xa);
    ld_vec<T, V>(x + c, xc);
    const float2* w = cs + t * R2;
    if (half || (V == 1 && a < p.R)) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 z = w[half ? a + e : a >> 1];
        const float x0 = xa[e], x1 = xc[e];
        xa[e] = x0 * z.x - x1 * z.y;
        xc[e] = x1 * z.x + x0 * z.y;
      }
    } else if (p.interleaved) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float* f = g ? xc : xa;
        const int at = g ? c : a;
#pragma unroll
        for (int e = 0; e + 1 < V; e += 2) {
          if (at + e < p.R) {
            const float2 z = w[(at + e) >> 1];
            const float x0 = f[e], x1 = f[e + 1];
            f[e] = x0 * z.x - x1 * z.y;
            f[e + 1] = x1 * z.x + x0 * z.y;
          }
        }
      }
    }
    st_vec<T, V>(y + a, xa);
    st_vec<T, V>(y + c, xc);
  }
}

}  // namespace rope
}  // namespace lb2
