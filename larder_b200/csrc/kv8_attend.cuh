// Attention of a few query rows over the paged 8-bit KV cache (kv8.cuh), split over the keys: HBM-bound.
//
//   o = softmax(scale q (code_k s_k)^T) (code_v s_v)
//
// A persistent CTA an SM streams its run of 64-key tiles. The call's tiles, ordered (b, KV head, row block, tile), are cut
// into equal runs, one a CTA, cut again where a (b, head, row block) ends, so that every SM streams the same number of
// bytes whatever the lengths; the partials (max, sum, unnormalised o) of a run's pieces are merged by combine_kernel,
// launched behind as a programmatic dependent. All G T query rows of a KV head share each pass over its codes.
//
// The codes reach shared memory as they lie (TMA boxes of a page's rows, 128-byte swizzled, 64-byte at D = 64), 1 byte a
// value, and turn into f16 MMA operands in registers: every e4m3 value is an f16 value, so nothing is rounded there, and
// cvt.rn.f16x2.e4m3x2 runs at 64 lanes a clock on an SM (measured), 128 codes against the 23 codes a clock that HBM
// delivers an SM. Products run on mma.sync m16n8k16 f16 (fp32 accumulate) with the keys, then the head dim, in M = 16 and
// the query rows in N = 8 columns. (mma.sync m16n8k32 on e4m3 itself would need the query and the weights split into two
// or three e4m3 terms.)
//  - S^T = K Q^T: a lane takes 16 consecutive bytes of a key, its share of four k-steps: the dims inside a 64-byte segment
//    are permuted alike in the query's fragments. The key of row q of an 8-row block is chosen so that neighbouring quads
//    read different halves of the 128-byte lines (no bank conflicts).
//  - O^T += V^T P^T: ldmatrix.trans on 16-bit units gives a lane two dims of two keys; one byte permute and two
//    conversions make them the operand pairs of two dims (rows quad and quad + 8 of the MMA are dims 2 quad, 2 quad + 1).
// bf16 query rows go to f16 exactly: a row is shifted by a power of two (its largest value to [2^14, 2^15)), which the
// score's factor undoes; bf16's 8 bits fit f16's 11 down to 2^-28 of the row's largest value.
//
// Softmax in base 2, fp32. The weights carry the values' scale: p'_n = 2^(s_n + log2 s_v - m + 7), m the running maximum of
// s_n + log2 s_v, and l = sum p'_n / s_v, so that o = sum p'_n code_n / l, with pages' scales far apart too. Only the
// products' weights are rounded, to f16; the sums are fp32. The maximum lags by up to 2^8 (below), so a row's largest
// p' lies between 2^7 and 2^15, the upper end of f16's range: weights down to 2^-21 of it at least keep f16's 11 bits, smaller
// ones lose one a power of two and are 0 below 2^-32 of it, which is what a key that dominates the sum with a value of 0
// leaves the others.
//
// A NaN code under a weight of 0 would spread to rows that do not see it: values past the length are zeroed in shared
// memory; with several rows of different horizons, combine_kernel takes a row that came out NaN again, key by key
// (attn_rows.cuh), which reads only what the row sees.
#pragma once

#include <cfloat>

#include "attn_rows.cuh"
#include "common.cuh"
#include "kv8.cuh"

namespace lb2 {
namespace kv8attn {

constexpr int BK = 64;       // keys a tile
constexpr int MAX_B = 1024;  // sequences a launch (the prefix table in shared memory); larger batches go in several
constexpr float TOP = 7.f;   // a weight at the running maximum is 2^TOP
constexpr int STATUS = 112;  // where (lb2_status): 112 a page id or length, 113.. waits

// NT: 8-row tiles of query rows a warp; MK: 16-key blocks of a tile a warp (two give it two independent chains of
// products); RG: row groups (sets of warps taking the same tile for other rows); KG: key groups (sets of warps taking
// every KG-th tile). At head dim 256 two warps share a warp's work (DS = 2), each with half the dims: O and the query's
// fragments then fit the registers up to 24 rows, so that a key's conversion serves them all; the two add their halves of
// the scores through shared memory.
template <int D, int NT, int RG, int MK, int KG>
struct Cfg {
  static constexpr int DS = D == 256 ? 2 : 1;
  static constexpr int DW = D / DS;             // dims a warp
  static constexpr int RP = 8 * NT * RG;  // rows of a block, padded
  static constexpr int SL = 4 / MK;       // key slices of a tile
  static constexpr int WARPS = DS * SL * RG * KG;
  static constexpr int NP = 4;            // producer warps: they take the tiles in turn
  static constexpr int THREADS = (WARPS + NP) * 32;
  static constexpr int BW = D < 128 ? D : 128;  // bytes a box row
  static constexpr int TILE = BK * D;           // bytes of a K (or V) tile
  static constexpr int STAGE = 2 * TILE;
  static constexpr bool Q_REGS = NT * DW <= 256;
  static constexpr int QBYTES = Q_REGS ? 0 : RG * NT * (D / 64) * 32 * 32;
  static constexpr int PART_REGS = NT * (DW / 16 + 1);          // float4 a lane: O and (m, l) of a warp's rows
  static constexpr int PART = WARPS / 2 * PART_REGS * 32 * 16;  // half the warps' parts
  static constexpr int XCH = DS > 1 ? 2 * WARPS * MK * NT * 32 * 16 : 0;  // two tiles' half scores of every warp
  static constexpr int JOIN = PART > XCH ? PART : XCH;  // (one area: a barrier lies between the two uses)
  static constexpr int FIXED = QBYTES + JOIN + 2 * WARPS * 8 * NT * 4 + (2 * MAX_B + 1) * 4 + 1024 + 1024;
  static constexpr int FIT = (232448 - FIXED) / (STAGE + 80);
  // A multiple of both, so that a stage only ever serves one producer warp and one key group, whose waits on it then
  // follow its phases in order (a wait two phases ahead would pass at once).
  static constexpr int STEP = KG > NP ? KG : NP;
  static constexpr int STAGES = (FIT > 16 ? 16 : FIT) / STEP * STEP;
  static constexpr int Q_OFF = STAGES * STAGE;
  static constexpr int PART_OFF = Q_OFF + QBYTES;
  static constexpr int QMAX = DS > 1 ? 2 * WARPS * 8 * NT * 4 : 0;  // two items' largest query values by half
  static constexpr int QMAX_OFF = PART_OFF + JOIN;
  static constexpr int SC_OFF = QMAX_OFF + QMAX;                // [STAGES][4 slices of 16 keys] Slice
  static constexpr int PREFIX_OFF = SC_OFF + STAGES * 64;        // [MAX_B + 1]
  static constexpr int LENS_OFF = PREFIX_OFF + (MAX_B + 1) * 4;  // [MAX_B]
  static constexpr int BAR_OFF = (LENS_OFF + MAX_B * 4 + 15) / 16 * 16;
  static constexpr int SMEM = BAR_OFF + 2 * STAGES * 8 + 16 + 1024;
  static_assert(STEP % KG == 0 && STEP % NP == 0 && STAGES >= 2 * KG && SMEM <= 232448, "shared memory budget");
};

struct Params {
  arows::PagedParams a;  // the call's arguments
  float* ws_o;           // [slots][rpb][D]
  float* ws_ml;          // [slots][rpb][2]
  int G, rows;           // query rows a KV head: G T
  int nrb, rpb;          // row blocks a KV head, rows a block
  int grid;
  int box;     // tokens a TMA box: min(page, BK)
  int lpage;   // log2(page)
  int wide_q;  // q rows may be read 16 bytes at a time
  float scale_log2;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// Byte offset of (key row r, 16-byte chunk c) in a tile: boxes of BW bytes a row, [D / BW][BK][BW], swizzled.
template <int D>
__device__ __forceinline__ uint32_t at(int r, int c) {
  if constexpr (D == 64) return uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  return uint32_t((c >> 3) * (BK * 128) + r * 128 + (((c ^ r) & 7) << 4));
}

// The key (0..7) in row i of an 8-key block: consecutive rows differ in bit 2 (bit 0 at D = 64), see above.
template <int D>
__device__ __forceinline__ int key_of(int i) {
  if constexpr (D == 64) return i;
  return (i >> 1) | ((i & 1) << 2);
}

// How many runs the call's tiles are cut into: one a CTA, but none without a tile (the grid is sized by the table's
// width, the lengths are read on the device). Every slot between a pair's first and last run is thus written.
__device__ __forceinline__ int64_t runs_of(const Params& p, int64_t total) { return min(int64_t(p.grid), total); }

// One piece of work: tiles [i0, i1) of sequence b for head-and-row-block hb (KV head hb / nrb, block hb % nrb).
struct Item {
  int b, hb, i0, i1, len, slot;
};

// The CTA's items in order; prefix[b] counts, for one head and row block, the tiles of the sequences before b.
struct Sched {
  const int* prefix;
  const int* lens;
  int B, H, cur, end;
  __device__ __forceinline__ Sched(const Params& p, const int* prefix_, const int* lens_)
      : prefix(prefix_), lens(lens_), B(p.a.B), H(p.a.Hkv * p.nrb) {
    const int64_t total = int64_t(prefix[B]) * H, runs = runs_of(p, total), c = blockIdx.x;
    cur = c < runs ? int(c * total / runs) : 0;
    end = c < runs ? int((c + 1) * total / runs) : 0;
  }
  __device__ __forceinline__ bool next(Item& it) {
    if (cur >= end) return false;
    const int key = cur / H;
    int lo = 0, hi = B;  // the largest b with prefix[b] <= key
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= key) lo = mid; else hi = mid;
    }
    const int base = prefix[lo] * H, nt = prefix[lo + 1] - prefix[lo];
    it.b = lo;
    it.len = lens[lo];
    it.hb = (cur - base) / nt;
    it.i0 = cur - base - it.hb * nt;
    const int stop = min(end, base + (it.hb + 1) * nt);
    it.i1 = it.i0 + stop - cur;
    it.slot = int(blockIdx.x) + lo * H + it.hb;
    cur = stop;
    return true;
  }
};

__device__ __forceinline__ int seq_len(const Params& p, int b) {
  return int(min(int64_t(max(p.a.kv_len[b], 0)), int64_t(p.a.max_pages) << p.lpage));
}

template <typename T, int D, int NT, int RG, int MK, int KG>
__global__ void __launch_bounds__(Cfg<D, NT, RG, MK, KG>::THREADS, 1)
    attend_kernel(const __grid_constant__ CUtensorMap map, const Params p) {
  using C = Cfg<D, NT, RG, MK, KG>;
  constexpr int STAGES = C::STAGES, WARPS = C::WARPS, SL = C::SL, DS = C::DS, DW = C::DW, SEG = DW / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* prefix = reinterpret_cast<int*>(sm + C::PREFIX_OFF);
  int* lens = reinterpret_cast<int*>(sm + C::LENS_OFF);
  float4* scl = reinterpret_cast<float4*>(sm + C::SC_OFF);
  float4* part = reinterpret_cast<float4*>(sm + C::PART_OFF);  // [WARPS / 2][PART_REGS][32 lanes]
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);
  uint64_t* empty = full + STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], DS * SL * RG);
    }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&map);
  }
  // A programmatic dependent of the stream's previous kernel: global memory is read only past this point.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int b = threadIdx.x; b < p.a.B; b += C::THREADS) {
    const int len = seq_len(p, b);
    if (len != p.a.kv_len[b] && blockIdx.x == 0) report_bad_index(STATUS);
    lens[b] = len;
    prefix[b + 1] = (len + BK - 1) / BK;
  }
  __syncthreads();
  if (warp == 0) {
    int run = 0;
    for (int base = 0; base < p.a.B; base += 32) {
      int x = base + lane < p.a.B ? prefix[base + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (base + lane < p.a.B) prefix[base + lane + 1] = run + x;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) prefix[0] = 0;
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Sched sched(p, prefix, lens);
  Item it;

  if (warp >= WARPS) {
    // ------------------------------------------------------------------ producer warps
    // Page ids and scales come 32 pages at a time, a lane a page, the next 32 loaded while these are used. A tile's boxes
    // (a page's rows, K or V, 128 bytes wide) are issued by a lane each. One warp's chain of instructions for a tile
    // (about 800 clocks) is slower than the tile's bytes arrive, so several warps take the tiles in turn.
    constexpr int NB = D / C::BW;  // boxes across a row
    constexpr int NP = C::NP;
    const int sub = BK / p.box;    // boxes down a tile
    const int per = p.box < (1 << p.lpage) ? (1 << p.lpage) / p.box : 1;  // tiles a page (128-token pages: 2)
    // lane = ((page in tile) NB + box) 2 + (K, V); lanes 0 .. 3 also write a slice of 16 keys' scales
    const int kv = lane & 1, bx = (lane >> 1) % NB, pg = (lane >> 1) / NB;
    const bool mine = pg < sub;
    const int dst = kv * C::TILE + bx * (BK * C::BW) + pg * p.box * C::BW;
    const int sp = (lane & 3) * 16 / p.box;
    int gt = warp - WARPS, done = 0;  // this warp's next tile; tiles of the items before
    int st = gt, phase = 1;           // its stage; parity of the stage's use before (1 at first: passes at once)
    bool ok = true;
    while (ok && sched.next(it)) {
      const int hk = it.hb / p.nrb;
      const int32_t* row = p.a.table + it.b * p.a.table_st;
      const int npages = (it.len + (1 << p.lpage) - 1) >> p.lpage;
      // page j of the sequence: id (-1: past the sequence), K scale, V scale
      auto fetch = [&](int j, int& id, float& ks, float& vs) {
        id = -1, ks = vs = 0.f;
        if (j < npages) {
          id = row[j];
          if (id < 0 || id >= p.a.num_pages) {
            report_bad_index(STATUS);
            id = -1;
          } else {
            const float* s = p.a.scales + int64_t(id) * 2 * p.a.Hkv + hk;
            ks = s[0], vs = s[p.a.Hkv];
          }
        }
      };
      int j0 = (it.i0 * BK) >> p.lpage;  // first page of the current 32
      int id, nid = -1;
      float ks, vs, nks = 0.f, nvs = 0.f;
      fetch(j0 + lane, id, ks, vs);
      bool ahead = false;  // the next 32 are on their way (asked for once a tile has been issued: a load is waited for)
      const int tiles = it.i1 - it.i0;
      for (; gt - done < tiles; gt += NP) {
        const int i = it.i0 + gt - done;
        const int j = (i * BK) >> p.lpage;  // first page of the tile
        if (j - j0 >= 32) {                 // (a tile's pages never straddle: a tile has 1, 2 or 4; steps are below 32)
          j0 += 32;
          if (!ahead) fetch(j0 + lane, nid, nks, nvs);
          id = nid, ks = nks, vs = nvs;
          ahead = false;
        }
        bool w = true;
        if (lane == 0 && !mbar_try_wait(&empty[st], phase)) w = !*abort_flag && mbar_wait(&empty[st], phase, STATUS + 1);
        if (!__shfl_sync(0xffffffffu, w, 0)) {
          ok = false;
          break;
        }
        const int pid = __shfl_sync(0xffffffffu, id, j - j0 + (mine ? pg : 0));
        const bool go = mine && pid >= 0;
        if (go)
          tma_load_4d(sm + st * C::STAGE + dst, &map, bx * C::BW, per > 1 ? (i & (per - 1)) * BK : 0, kv * p.a.Hkv + hk,
                      pid, &full[st]);
        const float a = __shfl_sync(0xffffffffu, ks, j - j0 + sp), c = __shfl_sync(0xffffffffu, vs, j - j0 + sp);
        // the slice's K scale; its V scale's logarithm (at least -100), the reciprocal of that power, what it leaves out
        if (lane < 4) {
          const float lv = fmaxf(lg2(c), -100.f);
          scl[st * 4 + lane] = make_float4(a, lv, ex2(-lv), lv == -100.f ? c * 0x1p100f : 1.f);
        }
        const uint32_t n = __popc(__ballot_sync(0xffffffffu, go));
        __syncwarp();  // the scales are written before lane 0's arrival
        if (lane == 0) mbar_arrive_expect_tx(&full[st], n * uint32_t(p.box * C::BW));
        if ((st += NP) >= STAGES) st -= STAGES, phase ^= 1;
        if (!ahead) {
          ahead = true;
          fetch(j0 + 32 + lane, nid, nks, nvs);
        }
      }
      done += tiles;
    }
    if (!ok && lane == 0) *abort_flag = 1;
    // Drain: the last copies this warp issued have landed before the CTA ends.
    if (lane == 0)
      for (int g = gt - NP; g >= 0 && g > gt - NP - STAGES; g -= NP) mbar_wait(&full[g % STAGES], (g / STAGES) & 1, STATUS + 2);
    return;
  }

  // ------------------------------------------------------------------ consumer warps
  const int quad = lane >> 2, qid = lane & 3;
  const int sl = warp % SL, rg = (warp / SL) % RG, kg = warp / (SL * RG) % KG, dh = warp / (SL * RG * KG);
  const int Tq = p.a.T;
  uint32_t qf[C::Q_REGS ? NT : 1][C::Q_REGS ? SEG : 1][8];  // this row's 16 dims of each 64-dim segment
  uint4* qsm = reinterpret_cast<uint4*>(sm + C::Q_OFF);     // [RG][NT][SEG][2][32 lanes]
  rope::Raw<T, 8> raw[NT][SEG][2];  // the warp's dims of the query rows as they lie
  auto load_q = [&](const Item& w) {
    const int hk = w.hb / p.nrb, r0 = (w.hb - hk * p.nrb) * p.rpb, r1 = min(p.rows, r0 + p.rpb);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + (rg * NT + nt) * 8 + quad;
      const int g = Tq == 1 ? r : r / Tq, t = r - g * Tq;
      const T* src = static_cast<const T*>(p.a.q) + w.b * p.a.q_st[0] + int64_t(hk * p.G + g) * p.a.q_st[1] +
                     t * p.a.q_st[2] + dh * DW + 16 * qid;
#pragma unroll
      for (int s = 0; s < SEG; ++s) {
        const T* from = src + 64 * s;
        if (r >= r1) {
          raw[nt][s][0].u = raw[nt][s][1].u = make_uint4(0, 0, 0, 0);
        } else if (p.wide_q) {
          raw[nt][s][0].load(from);
          raw[nt][s][1].load(from + 8);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) reinterpret_cast<T*>(&raw[nt][s][e >> 3].u)[e & 7] = from[e];
        }
      }
    }
  };
  constexpr bool AHEAD = NT == 1 && DS == 1;  // where registers allow, the next item's rows are loaded while this one's parts are merged
  bool have_q = false;
  float4* xch = reinterpret_cast<float4*>(sm + C::PART_OFF);  // [2 tiles][DS][WARPS / 2][MK NT][32 lanes]
  float* qmax = reinterpret_cast<float*>(sm + C::QMAX_OFF);  // [2 items][DS][WARPS / 2][8 NT]
  const int pair = warp % (WARPS / 2);
  int seen = 0, st = kg, phase = 0;  // tiles of the items before; this key group's next stage and its parity
  int xpar = 0, qpar = 0;
  bool ok = true;
  while (sched.next(it)) {
    const int hk = it.hb / p.nrb, r0 = (it.hb - hk * p.nrb) * p.rpb, r1 = min(p.rows, r0 + p.rpb);  // the block's rows
    // Query fragments: lane (quad, qid) holds dims 64 s + 16 qid .. + 15 of row quad of each row tile.
    if (!have_q) load_q(it);
    float fac[NT][2];
    int lim[NT][2], ex[NT];
    constexpr bool SHIFT = !std::is_same<T, __half>::value;
    if constexpr (SHIFT) {  // the exponent of each row's largest value
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mx = 0.f;
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
          __nv_bfloat162 m = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw[nt][s][g].u);
#pragma unroll
            for (int e = 0; e < 4; ++e) m = __hmax2(m, __habs2(h[e]));  // (NaN is passed over)
          }
          mx = fmaxf(mx, fmaxf(__low2float(m), __high2float(m)));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if constexpr (DS > 1) {  // of both halves of the dims
          if (qid == 0) qmax[((qpar * 2 + dh) * (WARPS / 2) + pair) * 8 * NT + nt * 8 + quad] = mx;
        }
        ex[nt] = __float_as_int(mx);
      }
      if constexpr (DS > 1) {
        asm volatile("bar.sync %0, 64;" ::"r"(2 + pair) : "memory");
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          ex[nt] = __float_as_int(fmaxf(__int_as_float(ex[nt]), qmax[((qpar * 2 + 1 - dh) * (WARPS / 2) + pair) * 8 * NT + nt * 8 + quad]));
        qpar ^= 1;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) ex[nt] = ex[nt] > 0 ? min(max((ex[nt] >> 23) - 127, -112), 127) : 14;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // bf16: times 2^(14 - ex), 14 - ex in [-113, 126]; f16 goes as it is
      const float up = SHIFT ? __uint_as_float(uint32_t(127 + 14 - ex[nt]) << 23) : 1.f;
#pragma unroll
      for (int s = 0; s < SEG; ++s) {
        uint32_t w[8];
        if constexpr (SHIFT) {
          float x[16];
          raw[nt][s][0].get(x);
          raw[nt][s][1].get(x + 8);
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = pack2<__half>(x[2 * e] * up, x[2 * e + 1] * up);
        } else {
          const uint4 a = raw[nt][s][0].u, b = raw[nt][s][1].u;
          w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        }
        if constexpr (C::Q_REGS) {
#pragma unroll
          for (int e = 0; e < 8; ++e) qf[nt][s][e] = w[e];
        } else if (sl == 0 && kg == 0) {
          uint4* d = qsm + ((rg * NT + nt) * (DS * SEG) + dh * SEG + s) * 64 + lane;
          d[0] = make_uint4(w[0], w[1], w[2], w[3]);
          d[32] = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // for columns 2 qid + e: the row whose fragments quad 2 qid + e holds
        fac[nt][e] = p.scale_log2;
        if constexpr (SHIFT) {  // times 2^(ex - 14), as two powers so that neither leaves fp32's range
          const int d = __shfl_sync(0xffffffffu, ex[nt], (2 * qid + e) * 4) - 14;
          fac[nt][e] = fac[nt][e] * __uint_as_float(uint32_t(127 + d / 2) << 23) * __uint_as_float(uint32_t(127 + d - d / 2) << 23);
        }
        // the row's last key (rows past the block's are zeros that see what the others see; nothing of them is kept)
        const int rr = r0 + (rg * NT + nt) * 8 + 2 * qid + e;
        lim[nt][e] = p.a.causal && Tq > 1 ? it.len - Tq + rr % Tq : it.len - 1;
      }
    }
    const int all_see = p.a.causal ? it.len - Tq : it.len - 1;  // the last key that every row sees
    if constexpr (!C::Q_REGS) asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");

    float m_run[NT][2], l_run[NT][2], acc[NT][DW / 16][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt][0] = m_run[nt][1] = -FLT_MAX;
      l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < DW / 16; ++j) acc[nt][j][0] = acc[nt][j][1] = acc[nt][j][2] = acc[nt][j][3] = 0.f;
    }
    const int turn = (kg - seen) & (KG - 1);  // this key group takes the item's tiles turn, turn + KG, ...
    const int i0 = it.i0 + turn, parts = SL * min(KG, it.i1 - it.i0);  // parts of a row that hold something
    seen += it.i1 - it.i0;
    for (int i = i0; i < it.i1; i += KG) {
      if (!mbar_try_wait(&full[st], phase) && (*abort_flag || !mbar_wait(&full[st], phase, STATUS + 3))) {
        ok = false;
        if constexpr (DS == 1) break;  // (DS > 1: the pair leaves together, below)
      }
      uint8_t* kt = sm + st * C::STAGE;
      uint8_t* vt = kt + C::TILE;
      const int kbase = i * BK + sl * 16 * MK;  // the warp's first key
      const int nvalid = min(16 * MK, max(0, it.len - kbase));
      if (nvalid < 16 * MK) {  // values past the length: zeros, so that P = 0 meets no NaN code
        for (int e = lane; e < (16 * MK - nvalid) * (DW / 16); e += 32) {
          const int r = sl * 16 * MK + nvalid + e / (DW / 16), c = dh * (DW / 16) + e % (DW / 16);
          *reinterpret_cast<uint4*>(vt + at<D>(r, c)) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      // (with few independent products the k-steps alternate between two accumulators: shorter chains)
      constexpr int KSP = MK * NT <= 2 ? 2 : 1;
      float s[MK][NT][4], s2[KSP > 1 ? MK : 1][KSP > 1 ? NT : 1][4];
#pragma unroll
      for (int mk = 0; mk < MK; ++mk)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[mk][nt][0] = s[mk][nt][1] = s[mk][nt][2] = s[mk][nt][3] = 0.f;
          if constexpr (KSP > 1) s2[mk][nt][0] = s2[mk][nt][1] = s2[mk][nt][2] = s2[mk][nt][3] = 0.f;
        }
#pragma unroll
      for (int sg = 0; sg < SEG; ++sg) {
        uint4 ka[MK], kb[MK];
#pragma unroll
        for (int mk = 0; mk < MK; ++mk) {
          const int kr = (sl * MK + mk) * 16 + key_of<D>(quad);
          ka[mk] = *reinterpret_cast<const uint4*>(kt + at<D>(kr, dh * (DW / 16) + 4 * sg + qid));
          kb[mk] = *reinterpret_cast<const uint4*>(kt + at<D>(kr + 8, dh * (DW / 16) + 4 * sg + qid));
        }
        uint32_t qs[NT][8];
        if constexpr (!C::Q_REGS) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4* d = qsm + ((rg * NT + nt) * (DS * SEG) + dh * SEG + sg) * 64 + lane;
            const uint4 u = d[0], v = d[32];
            qs[nt][0] = u.x, qs[nt][1] = u.y, qs[nt][2] = u.z, qs[nt][3] = u.w;
            qs[nt][4] = v.x, qs[nt][5] = v.y, qs[nt][6] = v.z, qs[nt][7] = v.w;
          }
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
          for (int mk = 0; mk < MK; ++mk) {
            uint32_t a0, a1, a2, a3;
            kv8::dec4(w == 0 ? ka[mk].x : w == 1 ? ka[mk].y : w == 2 ? ka[mk].z : ka[mk].w, a0, a2);
            kv8::dec4(w == 0 ? kb[mk].x : w == 1 ? kb[mk].y : w == 2 ? kb[mk].z : kb[mk].w, a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint32_t* q = C::Q_REGS ? qf[C::Q_REGS ? nt : 0][C::Q_REGS ? sg : 0] : qs[nt];
              if (KSP > 1 && (w & 1))
                mma16816(s2[KSP > 1 ? mk : 0][KSP > 1 ? nt : 0], a0, a1, a2, a3, q[2 * w], q[2 * w + 1]);
              else
                mma16816(s[mk][nt], a0, a1, a2, a3, q[2 * w], q[2 * w + 1]);
            }
          }
        }
      }
      if constexpr (KSP > 1) {
#pragma unroll
        for (int mk = 0; mk < MK; ++mk)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[mk][nt][e] += s2[mk][nt][e];
      }
      if constexpr (DS > 1) {  // the pair's halves of the scores (buffers alternate, so one barrier a tile is enough)
        constexpr int XW = MK * NT * 32;  // float4 a warp
        float4* mine = xch + ((xpar * 2 + dh) * (C::WARPS / 2) + pair) * XW + lane;
        const float4* other = xch + ((xpar * 2 + 1 - dh) * (C::WARPS / 2) + pair) * XW + lane;
        xpar ^= 1;
#pragma unroll
        for (int mk = 0; mk < MK; ++mk)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mine[(mk * NT + nt) * 32] = make_float4(s[mk][nt][0], s[mk][nt][1], s[mk][nt][2], s[mk][nt][3]);
        uint32_t both;  // the waits of both held: else both leave
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
            : "=r"(both)
            : "r"(uint32_t(ok)), "r"(2 + pair)
            : "memory");
        if (!both) {
          ok = false;
          break;
        }
#pragma unroll
        for (int mk = 0; mk < MK; ++mk)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float4 o = other[(mk * NT + nt) * 32];
            s[mk][nt][0] += o.x, s[mk][nt][1] += o.y, s[mk][nt][2] += o.z, s[mk][nt][3] += o.w;
          }
      }
      float ks[MK], lv[MK], iv[MK], rest[MK];
      bool odd = false;  // (uniform in the warp)
#pragma unroll
      for (int mk = 0; mk < MK; ++mk) {
        const float4 sc = scl[st * 4 + sl * MK + mk];
        ks[mk] = sc.x, lv[mk] = sc.y, iv[mk] = sc.z, rest[mk] = sc.w;
        odd = odd || rest[mk] != 1.f;
      }
      // Scores in base 2 with the values' scale, against the row's running maximum less TOP (what m_run holds). It moves
      // only when a score passes the maximum by more than 8 (weights up to 2^15 lose nothing in f16), so most tiles need no
      // exchange between lanes; before a row's first key it is the least finite number, which every score but -inf passes
      // (-inf itself would make keys whose scores are all -inf NaN).
      const bool whole = kbase + 16 * MK - 1 <= all_see;
      float t[MK][NT][4];
      auto against = [&] {  // t = score - (maximum - TOP); the lane's largest
        float top = -INFINITY;
#pragma unroll
        for (int mk = 0; mk < MK; ++mk)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float f0 = fac[nt][0] * ks[mk], f1 = fac[nt][1] * ks[mk];
            const float b0 = lv[mk] - m_run[nt][0], b1 = lv[mk] - m_run[nt][1];
            float* x = t[mk][nt];
            const float* y = s[mk][nt];
            x[0] = fmaf(y[0], f0, b0), x[1] = fmaf(y[1], f1, b1), x[2] = fmaf(y[2], f0, b0), x[3] = fmaf(y[3], f1, b1);
            if (!whole) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (kbase + 16 * mk + key_of<D>(quad) + 8 * (e >> 1) > lim[nt][e & 1]) x[e] = -INFINITY;
            }
            top = fmaxf(fmaxf(top, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
          }
        return top;
      };
      if (__any_sync(0xffffffffu, against() > TOP + 8.f)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = m_run[nt][e] + TOP;
#pragma unroll
            for (int mk = 0; mk < MK; ++mk)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float x = fmaf(s[mk][nt][2 * h + e], fac[nt][e] * ks[mk], lv[mk]);
                if (kbase + 16 * mk + key_of<D>(quad) + 8 * h <= lim[nt][e]) mx = fmaxf(mx, x);
              }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx -= TOP;
            const float corr = ex2(m_run[nt][e] - mx);
            m_run[nt][e] = mx;
            l_run[nt][e] *= corr;
#pragma unroll
            for (int j = 0; j < DW / 16; ++j) {
              acc[nt][j][e] *= corr;
              acc[nt][j][2 + e] *= corr;
            }
          }
        against();
      }
      uint32_t pb[NT][MK][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mk = 0; mk < MK; ++mk) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = ex2(t[mk][nt][e]);
          l_run[nt][0] = fmaf(x[0] + x[2], iv[mk], l_run[nt][0]);
          l_run[nt][1] = fmaf(x[1] + x[3], iv[mk], l_run[nt][1]);
          if (odd) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] *= rest[mk];
          }
          pb[nt][mk][0] = movm_t(pack2<__half>(x[0], x[1]));
          pb[nt][mk][1] = movm_t(pack2<__half>(x[2], x[3]));
        }
      }
      const uint32_t vbase = smem_u32(vt);
#pragma unroll
      for (int c = 0; c < DW / 16; c += 2) {  // 32 dims: matrices (keys 0-7, 8-15) x (chunks c, c + 1)
#pragma unroll
        for (int mk = 0; mk < MK; ++mk) {
          uint32_t v[4];
          const int r = (sl * MK + mk) * 16 + ((lane >> 3) & 1) * 8 + key_of<D>(lane & 7);
          ldsm_x4_t(vbase + at<D>(r, dh * (DW / 16) + c + (lane >> 4)), v);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a0, a1, a2, a3;
            kv8::dec4(__byte_perm(v[2 * h], 0, 0x3120), a0, a1);
            kv8::dec4(__byte_perm(v[2 * h + 1], 0, 0x3120), a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(acc[nt][c + h], a0, a1, a2, a3, pb[nt][mk][0], pb[nt][mk][1]);
          }
        }
      }
      if (nvalid < 16 * MK) fence_proxy_async_shared();  // the zeros precede the next copy into this stage
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if ((st += KG) >= STAGES) st -= STAGES, phase ^= 1;
    }

    // ------------------------------------------------------------------ the item's partial
    // The parts of a row (one a key slice and key group) meet in a tree through shared memory, each warp's registers as
    // they lie (a lane's counterpart is the same lane); the warps of part 0 write the merged partial.
    Sched ahead = sched;
    Item nx;
    have_q = AHEAD && ahead.next(nx);
    if (have_q) load_q(nx);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 4);
        l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 8);
        l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 16);
      }
    uint32_t all_ok;  // every warp's waits held: else all leave. (Also: the previous item's parts have been read.)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all_ok)
        : "r"(uint32_t(ok)), "n"(WARPS * 32)
        : "memory");
    if (!all_ok) {
      if (lane == 0) *abort_flag = 1;
      break;
    }
    const int pi = turn * SL + sl;
#pragma unroll 1  // (one copy of the code: at an item's end it is fetched cold)
    for (int half = SL * KG / 2; half > 0; half >>= 1) {
      if (half >= parts) continue;  // (the same for every warp)
      if (pi >= half && pi < 2 * half) {
        float4* d = part + (((pi - half) * RG + rg) * DS + dh) * C::PART_REGS * 32 + lane;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          *d = make_float4(m_run[nt][0], m_run[nt][1], l_run[nt][0], l_run[nt][1]);
          d += 32;
#pragma unroll
          for (int j = 0; j < DW / 16; ++j, d += 32) *d = make_float4(acc[nt][j][0], acc[nt][j][1], acc[nt][j][2], acc[nt][j][3]);
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
      if (pi < half) {
        const float4* d = part + ((pi * RG + rg) * DS + dh) * C::PART_REGS * 32 + lane;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float4 x = *d;
          d += 32;
          const float xm[2] = {x.x, x.y}, xl[2] = {x.z, x.w};
          float f[2], g[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mn = fmaxf(m_run[nt][e], xm[e]);
            f[e] = ex2(m_run[nt][e] - mn);
            g[e] = ex2(xm[e] - mn);
            m_run[nt][e] = mn;
            l_run[nt][e] = l_run[nt][e] * f[e] + xl[e] * g[e];
          }
#pragma unroll
          for (int j = 0; j < DW / 16; ++j, d += 32) {
            const float4 o = *d;
            acc[nt][j][0] = acc[nt][j][0] * f[0] + o.x * g[0];
            acc[nt][j][1] = acc[nt][j][1] * f[1] + o.y * g[1];
            acc[nt][j][2] = acc[nt][j][2] * f[0] + o.z * g[0];
            acc[nt][j][3] = acc[nt][j][3] * f[1] + o.w * g[1];
          }
        }
      }
      if (half > 1 || DS > 1) asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
    }
    if (pi == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = (rg * NT + nt) * 8 + 2 * qid + e;
          if (r >= r1 - r0) continue;
          const size_t out = size_t(it.slot) * p.rpb + r;
          if (quad == 0 && dh == 0) *reinterpret_cast<float2*>(p.ws_ml + 2 * out) = make_float2(m_run[nt][e], l_run[nt][e]);
#pragma unroll
          for (int j = 0; j < DW / 16; ++j)
            *reinterpret_cast<float2*>(p.ws_o + out * D + dh * DW + 16 * j + 2 * quad) =
                make_float2(acc[nt][j][e], acc[nt][j][2 + e]);
        }
    }
  }
}

// Merges the partials of each (b, KV head, row block): a block for eight rows of each, a warp a row. The pair's partials sit in consecutive
// slots, found from its first and last tile.
template <typename T, int D>
__global__ void __launch_bounds__(256) combine_kernel(const Params p) {
  constexpr int E = D / 32, HELD = 8;
  __shared__ int s_tiles[2][8];
  const int H = p.a.Hkv * p.nrb, b = blockIdx.x / H, hb = blockIdx.x - b * H;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  int before = 0, total = 0;
  for (int i = tid; i < p.a.B; i += 256) {
    const int t = (seq_len(p, i) + BK - 1) / BK;
    total += t;
    if (i < b) before += t;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane == 0) s_tiles[0][w] = before, s_tiles[1][w] = total;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) before += s_tiles[0][i], total += s_tiles[1][i];
  const int len = seq_len(p, b), nt = (len + BK - 1) / BK;
  int first = 0, nparts = 0;
  if (nt > 0) {  // CTA of tile t: the largest c with floor(c total / runs) <= t, i.e. ((t + 1) runs - 1) / total
    const int64_t tt = int64_t(total) * H, t0 = int64_t(before) * H + int64_t(hb) * nt, runs = runs_of(p, tt);
    const int c0 = int(((t0 + 1) * runs - 1) / tt), c1 = int(((t0 + nt) * runs - 1) / tt);
    first = c0 + blockIdx.x;
    nparts = c1 - c0 + 1;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int hk = hb / p.nrb, r0 = (hb - hk * p.nrb) * p.rpb, nrows = min(p.rows - r0, p.rpb);
  for (int r = blockIdx.y * 8 + w; r < nrows; r += 8 * gridDim.y) {
    float x[E], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
    for (int k0 = 0; k0 < nparts; k0 += HELD) {  // HELD partials' loads in flight at once
      float2 ml[HELD];
      float y[HELD][E];
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        const size_t at = size_t(first + min(k0 + k, nparts - 1)) * p.rpb + r;
        ml[k] = *reinterpret_cast<const float2*>(p.ws_ml + 2 * at);
        const float* src = p.ws_o + at * D + lane * E;
        if constexpr (E == 2) {
          const float2 v = *reinterpret_cast<const float2*>(src);
          y[k][0] = v.x, y[k][1] = v.y;
        } else {
#pragma unroll
          for (int e = 0; e < E; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(src + e);
            y[k][e] = v.x, y[k][e + 1] = v.y, y[k][e + 2] = v.z, y[k][e + 3] = v.w;
          }
        }
      }
      float m1 = M;
#pragma unroll
      for (int k = 0; k < HELD; ++k) m1 = fmaxf(m1, k0 + k < nparts ? ml[k].x : -INFINITY);
      const float mu = m1 == -INFINITY ? 0.f : m1, f = ex2(M - mu);
      L *= f;
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] *= f;
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        if (k0 + k >= nparts) continue;
        const float g = ex2(ml[k].x - mu);
        L = fmaf(ml[k].y, g, L);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = fmaf(y[k][e], g, x[e]);
      }
      M = m1;
    }
    const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] *= inv;
      nan = nan || x[e] != x[e];
    }
    const int rr = r0 + r, h = hk * p.G + rr / p.a.T, t = rr % p.a.T;
    if (p.a.causal && p.a.T > 1 && __any_sync(0xffffffffu, nan)) {
      // A NaN: the row's own, or a later token's under a weight of 0. The row again, reading only what it sees.
      const T* q = static_cast<const T*>(p.a.q) + b * p.a.q_st[0] + h * p.a.q_st[1] + t * p.a.q_st[2] + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = to_f<T>(q[e]);
      arows::PagedKeys<E> keys{p.a.pages, p.a.scales, p.a.table + b * p.a.table_st, p.a.Hkv, hk, p.a.page,
                               p.a.num_pages, lane * E};
      arows::attend_row<E>(keys, len - p.a.T + 1 + t, p.a.scale, x);
    }
    T* o = static_cast<T*>(p.a.o) + b * p.a.o_st[0] + h * p.a.o_st[1] + t * p.a.o_st[2] + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = from_f<T>(x[e]);
  }
}

}  // namespace kv8attn
}  // namespace lb2
