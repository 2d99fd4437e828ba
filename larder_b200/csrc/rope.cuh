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
// token's R / 2 (cos, sin) pairs once, in shared memory, while its rows' loads are in flight. 8192 tokens of 32 heads x 128
// (f16) take 26 us, 5130 GB/s (66 us with four fp32 rows a thread held unpacked, at two blocks an SM; 39 us with the
// angles read from shared memory for every row); one token for each of 16 sequences takes 2.4 us behind another kernel.
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
  int ltok, hg;  // tokens (log2) and heads a block takes
};

// (cos, sin) of `frac` 2^-64 turns.
__device__ __forceinline__ float2 turn_cs(uint64_t frac) {
  const float h = __ll2float_rn(static_cast<long long>(frac)) * 0x1p-63f;  // half turns, in [-1, 1]
  float s, c;
  sincospif(h, &s, &c);
  return make_float2(c, s);
}

constexpr int THREADS = 256;

// V elements a load: 16 bytes, or one element for the strides, alignments and widths that 16 bytes do not fit.
template <typename T, int V>
struct Raw {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* f) const {
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f<T>(h[i]);
  }
};
template <typename T>
struct Raw<T, 1> {
  T u;
  __device__ __forceinline__ void load(const T* p) { u = *p; }
  __device__ __forceinline__ void get(float* f) const { f[0] = to_f<T>(u); }
};
template <typename T, int V>
__device__ __forceinline__ void ld_vec(const T* p, float* f) {
  Raw<T, V> r;
  r.load(p);
  r.get(f);
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

// N (cos, sin) pairs from shared memory, two a load.
template <int N>
__device__ __forceinline__ void ld_pairs(const float2* w, float2* z) {
  if constexpr (N == 1) {
    z[0] = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float4 v = *reinterpret_cast<const float4*>(w + i);
      z[i] = make_float2(v.x, v.y);
      z[i + 1] = make_float2(v.z, v.w);
    }
  }
}

// Rotates the neighbouring pairs of V values.
template <int V>
__device__ __forceinline__ void turn_pairs(float* f, const float2* z) {
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    const float x0 = f[e], x1 = f[e + 1];
    f[e] = x0 * z[e / 2].x - x1 * z[e / 2].y;
    f[e + 1] = x1 * z[e / 2].x + x0 * z[e / 2].y;
  }
}

// A unit is two groups of V elements: in the half layout's rotated part elements [V u, V u + V) and their partners
// R / 2 on; in what it leaves alone, and in the interleaved layout, whose pairs lie inside a group, groups half the part
// apart, so that neighbouring lanes access neighbouring groups (V == 1, interleaved: the pair (2 u, 2 u + 1)).
// A thread has one unit of K rows (token, head), all loaded before the block's angles are formed.
template <typename T, int V, int K>
__global__ void __launch_bounds__(THREADS, 3) rope_kernel(const Params p) {
  extern __shared__ __align__(16) float2 cs[];  // [tokens][R / 2]
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int R2 = p.R >> 1, upr = p.D / (2 * V);  // units a row
  const int ntok = p.B * p.T;                   // < 2^31: checked by the launcher
  const int tok0 = blockIdx.x << p.ltok, h0 = blockIdx.y * p.hg;
  const int nt = min(1 << p.ltok, ntok - tok0), nh = min(p.hg, p.H - h0);
  const int rpp = upr < THREADS ? THREADS / upr : 1;  // rows a pass
  const int first = threadIdx.x / upr;
  for (int u0 = 0; u0 < upr; u0 += THREADS) {  // (once, but for single elements of rows wider than the block)
    const int u = u0 + threadIdx.x - first * upr;
    const bool mine = first < rpp && u < upr;
    const bool half = !p.interleaved && u * V < R2;
    const bool pair = V == 1 && p.interleaved;
    const int from = p.interleaved || half ? 0 : p.R;  // the part the unit lies in: [from, from + 2 apart)
    const int apart = half ? R2 : (p.D - from) >> 1;
    const int a = pair ? 2 * u : from + (u - (from >> 1) / V) * V, c = pair ? a + 1 : a + apart;
    Raw<T, V> ra[K], rc[K];
    int64_t yo[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int th = first + k * rpp, t = th & ((1 << p.ltok) - 1), h = th >> p.ltok;
      yo[k] = -1;
      if (mine && t < nt && h < nh) {
        const int row = tok0 + t, b = p.B == 1 ? 0 : row / p.T, s = row - b * p.T;
        const T* x = static_cast<const T*>(p.x) + b * p.x_st[0] + (h0 + h) * p.x_st[1] + s * p.x_st[2];
        yo[k] = b * p.y_st[0] + (h0 + h) * p.y_st[1] + s * p.y_st[2];
        ra[k].load(x + a);
        rc[k].load(x + c);
      }
    }
    if (u0 == 0) {
      for (int i = threadIdx.x; i < nt * R2; i += THREADS) {
        const int t = i / R2, f = i - t * R2;
        const int row = tok0 + t, b = p.B == 1 ? 0 : row / p.T;
        const int64_t pos = p.pos[b * p.p_st + (row - b * p.T)];
        float2 z = turn_cs(uint64_t(pos) * p.turns[f]);
        z.x *= p.amp;
        z.y *= p.inverse ? -p.amp : p.amp;
        cs[i] = z;
      }
      __syncthreads();
    }
    // The unit's angles: all its rows are of one token (the tokens divide a pass's rows).
    const float2* w = cs + (first & ((1 << p.ltok) - 1)) * R2;
    const bool turn_c = p.interleaved && !pair && c < p.R, turn_a = p.interleaved && !pair && a < p.R;
    float2 z[V];  // half, or an interleaved pair: of pair e; interleaved groups: a's V / 2 pairs, then c's
    if (half || (pair && a < p.R)) {
      ld_pairs<V>(w + (half ? a : a >> 1), z);
    } else if constexpr (V > 1) {
      if (turn_a) ld_pairs<V / 2>(w + (a >> 1), z);
      if (turn_c) ld_pairs<V / 2>(w + (c >> 1), z + V / 2);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (yo[k] < 0) continue;
      float xa[V], xc[V];
      ra[k].get(xa);
      rc[k].get(xc);
      if (half || (pair && a < p.R)) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float x0 = xa[e], x1 = xc[e];
          xa[e] = x0 * z[e].x - x1 * z[e].y;
          xc[e] = x1 * z[e].x + x0 * z[e].y;
        }
      } else if constexpr (V > 1) {
        if (turn_a) turn_pairs<V>(xa, z);
        if (turn_c) turn_pairs<V>(xc, z + V / 2);
      }
      T* y = static_cast<T*>(p.y) + yo[k];
      st_vec<T, V>(y + a, xa);
      st_vec<T, V>(y + c, xc);
    }
  }
}

}  // namespace rope
}  // namespace lb2
