// Attention of packed chunks of new tokens over the paged 8-bit KV cache (kv8.cuh) on tcgen05.
//
//   o = softmax(scale q (code_k s_k)^T) (code_v s_v)
//
// A row is a (token, query head) of one KV head, the G heads of a token side by side, so that all rows that share K and V
// share the passes over them: an item is a block of 256 rows (128 at head dim 256) of one sequence and KV head, over 128-key
// tiles up to its last row's horizon. The codes are read from the pages into registers, turned into f16 (every e4m3 value is
// one) and stored as the swizzled operand tiles of both products: once for a block's 256 rows, and no raw tile passes
// through shared memory, whose bandwidth is the products' too.
//
// The tensor pipe works on units, (row tile of 128, half a key tile) pairs, over four S buffers in turn: S_i = Q K^T into buffer
// i % 4, warpgroup i % 2 turns it into P_i (in its place), O += P_i V, S_{i+4}. A warpgroup's next scores are thus ready when it
// is done with the last ones.
//  - more than 128 rows, head dim 64 and 128: unit i is row tile i % 2 of half tile i / 2; each warpgroup has its own rows.
//  - up to 128 rows there: unit i is half tile i of the one row tile; each warpgroup has its own maximum, sum and O over its
//    half of the keys, joined at the end.
//  - head dim 256 (O takes half the tensor memory): unit i is half tile i; the warpgroups share the rows' maximum, handed on
//    from unit to unit, and O; each sums its own units' weights.
//
// Work is cut evenly whatever the lengths: the call's (row tile, key tile) steps in order, cut into equal runs, one a CTA (one
// CTA an SM). An item that a cut parts is merged from fp32 partials by combine_kernel, launched behind as a programmatic
// dependent; its parts are known from the steps alone, so every sum is formed in the same order in every run of a call.
//
// Measured (bf16, 32 / 8 heads x 128): 2048 new of 32768 tokens 1.24 ms, 860 TFLOP/s, half of what the products alone could run
// at; what bounds it is the number of instructions, 10 000 warp instructions for 256 rows x 128 keys, at two a clock and SM (softmax 4 300,
// conversion 2 200, the rest barriers, schedules and issue). f16, 24 / 2 heads x 256, 1001 of up to 16390: 0.42 ms, 800 TFLOP/s.
// 33 of 777 tokens: 29 us, the life of one CTA and the merge.
//
// Softmax in base 2, fp32, one thread a row. As in kv8_attend.cuh the weights carry the values' scale, p' = 2^(s + log2 s_v -
// m), m the running maximum of s + log2 s_v less 7, l = sum p' / s_v, o = sum p' code_v / l; the maximum moves when it is
// passed by more than 8, so p' reaches 2^15, the upper end of f16, and keeps f16's 11 bits down to 2^-21 of the largest; scores
// too large for that arithmetic take a path of their own (loud_weights). bf16 queries go to f16, a row shifted by a power of two
// that the score's factor undoes, its largest value to [2^14, 2^15): exactly down to 2^-31 of that value, and off by 2^-39 of it at
// most below (half a step of f16's subnormals).
//
// A NaN code under a weight of 0 would spread to rows that do not see it. Keys past an item's horizon are stored as zeros; a
// row that comes out NaN is looked at again at the end (row_again), and where a value that it does not see is to blame, taken
// again reading only what it sees.
//
// Roles (640 threads): warps 0-3, 4-7 softmax and epilogue (warp w: TMEM lanes of quarter w % 4), 8-15 codes and queries into
// shared memory, 16 and 19 issue the products P V and S, 17 reads the page table and scales ahead, 18 lists the CTA's pieces.
#pragma once

#include <cfloat>

#include "attn_prefill.cuh"
#include "attn_prefill2.cuh"
#include "attn_rows.cuh"
#include "common.cuh"
#include "kv8.cuh"
#include "wait_clock.cuh"

namespace lb2 {
namespace kv8chunk {

constexpr int BM = 128, BN = 128;  // rows of a row tile, keys of a key tile
constexpr int BH = 64;             // keys of a unit: half a key tile
constexpr int MAX_B = 1024;        // sequences a launch
constexpr int THREADS = 640;
constexpr int CONV_WARP = 8, CONV_WARPS = 8, MMA_WARP = 16, TABLE_WARP = 17, PLAN_WARP = 18, SCORE_WARP = 19;
constexpr int CT = CONV_WARPS * 32;  // threads that turn codes into operands
constexpr int PIECES = 4;          // pieces of work listed ahead
constexpr int TABLES = 8;          // key tiles whose page ids and scales are held
constexpr uint32_t WHOLE = 256;    // a tile whose 128 keys are all there
constexpr float TOP = 7.f;         // a weight at the running maximum is 2^TOP
constexpr float LOUD = 1 << 20;    // from a maximum of this size on, fp32 numbers are 2^-3 and more apart
constexpr int STATUS_PLAN = 158;
constexpr int STATUS = arows::STATUS_CHUNK;  // lb2_status: 140 lengths and page ids, 141.. waits

// What a CTA does of one item: key tiles kt0 .. kt0 + nt - 1. No units: the end of the list.
struct Piece {
  int b, lo, n, len, hk, f0, rows, horizon, kt0, nt, units;
  int pair, whole;
  int slot;    // of its partial, where it is not the whole item
  int nparts;  // of an item that it begins and does not end, else 0
  int pad;
};

template <int D>
struct Cfg {
  static constexpr bool WIDE = D == 256;
  static constexpr int QT = WIDE ? 1 : 2;         // row tiles of an item
  static constexpr int RB = BM * QT;
  // A stage of the operand ring: a tile's K or V, or a half tile's (the keys of a unit) at head dim 256, where two tiles' K and V
  // do not fit: a half is free again after its unit. Boxes of 64 dims, 128 bytes a key.
  static constexpr int SPT = WIDE ? 2 : 1;        // stages of a K (or V) tile
  static constexpr int SK = BN / SPT;             // keys of a stage
  static constexpr int BOX = SK * 128;            // bytes of a stage's box
  static constexpr int STAGE = SK * D * 2;
  static constexpr int NS = D == 64 ? 6 : 4;
  static constexpr int QTILE = BM * D * 2;
  static constexpr int K_OFF = QT * QTILE;
  static constexpr int TAB_OFF = K_OFF + NS * STAGE;           // [TABLES][8] float4 of a 16-key slice's scales
  static constexpr int ID_OFF = TAB_OFF + TABLES * 8 * 16;     // [TABLES][8] int64: where the pages' K of the head begin; -1: none
  static constexpr int FAR_OFF = ID_OFF + TABLES * 8 * 8;      // [TABLES] the slices whose weights' sums are formed apart
  static constexpr int FAC_OFF = FAR_OFF + TABLES * 4;         // [2 items][RB] the rows' score factors
  static constexpr int ML_OFF = FAC_OFF + 2 * RB * 4;          // [2][128] float2
  static constexpr int MSH_OFF = ML_OFF + 2 * BM * 8;          // [128] the shared maximum
  static constexpr int PREFIX_OFF = MSH_OFF + BM * 4;          // [MAX_B + 3] int64
  static constexpr int RANGE_OFF = PREFIX_OFF + (MAX_B + 3) * 8;  // [MAX_B + 2] Range
  static constexpr int PIECE_OFF = (RANGE_OFF + (MAX_B + 2) * 12 + 15) / 16 * 16;  // [PIECES] Piece
  static constexpr int BAR_BYTES = 640;
  static constexpr int BAR_OFF = PIECE_OFF + PIECES * int(sizeof(Piece));
  static constexpr int SMEM = BAR_OFF + BAR_BYTES + 1024;
  static constexpr int O_COL = 2 * BN;            // O, or the two warpgroups' O at O_COL and O_COL + D
  static_assert(PREFIX_OFF % 8 == 0 && SMEM <= 232448, "shared memory budget");
  static_assert(O_COL + QT * D <= 512, "TMEM budget");
};

struct Params {
  arows::ChunkParams c;
  float* ws_o;   // [2 grid][D / 4][RB][4]
  float* ws_ml;  // [2 grid][2][RB]
  int4* rec;     // [grid][2]: the item that the CTA begins and does not end
  int G;
  int lpage;
  int first, last;       // the launch has the call's first, last sequences
  int wide_q, wide_o;    // 16-byte query loads; bytes an output store may take: 32, 16 or 0 (an element)
  int flip;              // a negative scale: the queries' signs
  int min_units;         // units a CTA at least
  float scale_log2;
};

// The sequences as ranges of rows: range 0 the rows before the first, range b + 1 sequence b, the last the rows behind (both
// without keys).
struct Range {
  int lo, n, len;
};

__device__ __forceinline__ Range range_of(const Params& p, int r) {
  const int B = p.c.a.B, T = p.c.a.T;
  Range x{0, 0, 0};
  if (r == 0) {
    if (p.first) x.n = min(max(p.c.cu[0], 0), T);
  } else if (r == B + 1) {
    x.lo = min(max(p.c.cu[B], 0), T);
    if (p.last) x.n = T - x.lo;
  } else {
    const arows::ChunkRange c = arows::chunk_range(p.c, r - 1, STATUS, false);
    x.lo = c.lo, x.n = c.hi - c.lo, x.len = c.len;
  }
  return x;
}

struct Block {
  int rows, horizon, tiles, units;
  bool pair;
};

template <int RB>
__device__ __forceinline__ Block block_of(const Params& p, const Range& x, int k) {
  Block b;
  b.rows = min(RB, x.n * p.G - k * RB);
  const int last = (k * RB + b.rows - 1) / p.G;  // token
  b.horizon = p.c.a.causal ? max(x.len - (x.n - 1 - last), 0) : x.len;
  if (x.len == 0) b.horizon = 0;
  b.tiles = max(1, (b.horizon + BN - 1) / BN);
  b.pair = RB > BM && b.rows > BM;
  b.units = b.pair ? 2 * b.tiles : b.tiles;
  return b;
}

// The CTA's pieces in order, found by one warp. prefix[r]: units of the ranges before r.
template <int RB>
struct Sched {
  const Params& p;
  const int64_t* prefix;
  const Range* ranges;
  int64_t each, at, p0, p1;  // units a run; the current item's first unit; the CTA's run [p0, p1)
  int more;                  // the first so many runs have one unit more
  int r, hk, k, nb;
  Range x;

  __device__ __forceinline__ int64_t cut(int c) const { return c * each + min(c, more); }
  // The run of a unit.
  __device__ __forceinline__ int run_of(int64_t u) const {
    const int64_t first = more * (each + 1);
    return int(u < first ? div(u, each + 1) : more + div(u - first, each));
  }
  // (64-bit divisions take a few hundred clocks: they are kept for calls that need them)
  static __device__ __forceinline__ int64_t div(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
  }

  __device__ __noinline__ Sched(const Params& p_, const int64_t* prefix_, const Range* ranges_) : p(p_), prefix(prefix_), ranges(ranges_) {
    const int NR = p.c.a.B + 2, lane = threadIdx.x & 31;
    const int64_t total = prefix[NR];
    const int runs = int(max(int64_t(1), min(int64_t(gridDim.x), div(total, p.min_units)))), c = blockIdx.x;
    each = div(total, runs);
    more = int(total - each * runs);
    p0 = c < runs ? cut(c) : 0;
    p1 = c < runs ? cut(c + 1) : 0;
    r = hk = k = nb = 0;
    at = 0;
    if (p0 >= p1) return;
    int lo = 0, hi = NR;  // the last range with prefix <= p0 that is not empty
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= p0) lo = mid; else hi = mid;
    }
    enter(lo);
    const int64_t of_head = div(prefix[r + 1] - prefix[r], p.c.a.Hkv);
    hk = int(div(p0 - at, of_head));
    at += hk * of_head;
    for (int k0 = 0; k0 < nb; k0 += 32) {  // 32 blocks at a time
      const int own = k0 + lane < nb ? block_of<RB>(p, x, k0 + lane).units : 0;
      int64_t sum = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, k0 + lane < nb && at + sum > p0);
      if (past) {
        const int l = __ffs(past) - 1;
        at += __shfl_sync(0xffffffffu, sum - own, l);
        k = k0 + l;
        break;
      }
      at += __shfl_sync(0xffffffffu, sum, 31);
    }
  }

  __device__ __forceinline__ void enter(int range) {
    r = range;
    x = ranges[r];
    nb = (x.n * p.G + RB - 1) / RB;
    at = prefix[r];
  }

  __device__ __noinline__ bool next(Piece& w) {
    while (at < p1) {
      const Block b = block_of<RB>(p, x, k);
      int64_t a = max(p0 - at, int64_t(0)), z = min(p1 - at, int64_t(b.units));
      if (b.pair) a &= ~int64_t(1), z &= ~int64_t(1);  // (runs are two units at least: a cut parts no pair)
      w.b = r - 1, w.lo = x.lo, w.n = x.n, w.len = x.len, w.hk = hk;
      w.f0 = k * RB, w.rows = b.rows, w.horizon = b.horizon, w.pair = b.pair;
      w.kt0 = int(b.pair ? a >> 1 : a);
      w.units = int(z - a);
      w.nt = b.pair ? w.units >> 1 : w.units;
      w.whole = a == 0 && z == b.units;
      w.slot = 2 * int(blockIdx.x) + (a == 0 ? 1 : 0);
      w.nparts = 0;
      if (a == 0 && !w.whole) w.nparts = run_of(at + b.units - 1) - int(blockIdx.x) + 1;
      at += b.units;
      if (++k == nb) {
        k = 0;
        if (++hk == p.c.a.Hkv) {
          hk = 0;
          int rr = r + 1;
          while (rr < p.c.a.B + 2 && prefix[rr + 1] == prefix[rr]) ++rr;
          if (rr < p.c.a.B + 2) enter(rr);
        }
      }
      if (w.units > 0) return true;
    }
    return false;
  }
};

// Entry e of a piece's 2 nt fills of the operand ring: which (V or K) and key tile. The order is the products': with pairs
// K_0 V_0 K_1 V_1 .., else K_0 K_1 V_0 K_2 V_1 .. V_{nt-1}.
__device__ __forceinline__ void entry(bool pair, int nt, int e, int& kind, int& t) {
  if (pair) kind = e & 1, t = e >> 1;
  else if (e == 0) kind = 0, t = 0;
  else if (e == 2 * nt - 1) kind = 1, t = nt - 1;
  else kind = 1 - (e & 1), t = kind ? (e - 2) >> 1 : (e + 1) >> 1;
}
__device__ __forceinline__ int k_entry(bool pair, int t) { return pair ? 2 * t : t == 0 ? 0 : 2 * t - 1; }
__device__ __forceinline__ int v_entry(bool pair, int nt, int t) { return pair ? 2 * t + 1 : t == nt - 1 ? 2 * nt - 1 : 2 * t + 2; }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

// Waits for the loads from tensor memory so far; the values of one of them pass through, so that no use of them moves ahead.
__device__ __forceinline__ void wait_ld32(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                 "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
                 "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]),
                 "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}

// The products and commits of attn_prefill.cuh, issued by the lane whose `lead` is set; a, b: the descriptors' low words, HI
// the high word that all operands here share (stride 1024 bytes, version 1, 128-byte swizzle).
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 x, {%1, %6};\n\tmov.b64 y, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(lead), "n"(DESC_HI));
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 y, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(lead), "n"(DESC_HI));
}
__device__ __forceinline__ void mma_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}

// l 2^x, x <= 0, in two steps: l reaches 2^115 where V scales are far apart, and 2^x alone may be 0.
__device__ __forceinline__ float shrink(float l, float x) {
  const float h = prefill::ex2f(0.5f * x);
  return l * h * h;
}

// A row whose maximum is so large that the roundings of the maximum and of a weight's exponent, each half a step between fp32
// numbers of that size, could lift weights past f16's range, or all of them out of it. (The look for such rows takes 1 % of 2048
// new of 32768 tokens, 1.21 -> 1.23 ms; a branch in the loop of the weights instead, or their loop twice, 3 to 5 %.)
__device__ __forceinline__ bool is_loud(float m) { return fabsf(m) >= LOUD && m != -FLT_MAX; }

// The weights of a unit with loud rows, out of line: exponents are the scores as the maximum saw them, each rounded once, less the
// maximum, so that none is above what the maximum may lag by. P takes the place of S; l with the weights' sum.
__device__ __noinline__ float loud_weights(uint32_t s_col, const float4* sc, uint32_t marked, float fac, float m, float l) {
#pragma unroll 1
  for (int c = 0; c < BH; c += 32) {
    float x[32];
    uint32_t pk[16];
    prefill::tmem_ld32(s_col + c, x);
    prefill::tmem_wait_ld();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 f = sc[c / 16 + q];
      const float mul = fmaxf(fac * f.x, FLT_MIN);
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float a = x[16 * q + e], b = x[16 * q + e + 1];
        const float y = prefill::ex2f(fmaf(a, mul, f.w) - m), z = prefill::ex2f(fmaf(b, mul, f.w) - m);
        sum += y + z;
        pk[8 * q + e / 2] = pack2<__half>(y, z);
        if (marked >> (c / 16 + q) & 1u)
          l += prefill::ex2f(fmaf(a, mul, f.y) - m - f.y) + prefill::ex2f(fmaf(b, mul, f.y) - m - f.y);
      }
      l = fmaf(sum, f.z, l);
    }
    prefill::tmem_st16(s_col + c / 2, pk);
    prefill::tmem_wait_st();
  }
  return l;
}

// 16 bytes of codes. (volatile: the loads stay ahead of the wait behind them)
__device__ __forceinline__ uint4 ld_codes(const uint8_t* p) {
  uint4 x;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p));
  return x;
}

// 16 bytes, or zeros where they are not wanted, without a branch.
__device__ __forceinline__ uint4 load_if(const uint8_t* p, bool want) {
  uint4 x;
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@q ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(x.x), "=&r"(x.y), "=&r"(x.z), "=&r"(x.w)
      : "l"(p), "r"(uint32_t(want)));
  return x;
}

// Registers a thread: 640 are launched with 96 each, of which the softmax warps take more. (Once a warp: a second change would
// need a barrier of its warpgroup first.)
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
static_assert(256 * 128 + 384 * 72 <= THREADS * 96, "a split above what was launched would wait forever");

// A wait's look at the clock, out of line, as the roles' loops together should stay small (an SM's instruction cache holds
// some thousand instructions near the schedulers, and five roles share it). since: 0 at a wait's first look, then what this
// returned; 1: give up, some role has or the wait's time is over.
__device__ __noinline__ uint32_t wait_check(uint32_t since, volatile int* abort_flag, int where) {
  if (*abort_flag) return 1;
  // (the list's warp waits for whole pieces of work: its bound is for the others to have failed to end theirs)
  since = wait_look(since, globaltimer_ns(), kWaitNs * (where == STATUS_PLAN ? 64u : 1u));
  if (since != 1u) return since;
  report_timeout(where);
  *abort_flag = 1;
  return 1;
}

// A bounded wait that gives up at once when some role of the CTA has. With HINT the waiting thread sleeps between polls.
template <uint32_t HINT = 1000>
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int where) {
  uint32_t since = 0, n = 0;
  while (!(HINT ? mbar_try_wait_hint(bar, parity, HINT) : mbar_try_wait(bar, parity)))
    if ((++n & 63u) == 0 && (since = wait_check(since, abort_flag, where)) == 1u) return false;
  return true;
}

// The second look at folded row f of an item, by one warp: where its output has NaN columns and one of the keys behind it that
// its item's products took holds a NaN there, the row again, reading only what it sees.
template <typename T, int D>
__device__ __noinline__ void row_again(const Params& p, int b, int lo, int n, int len, int hk, int f, int horizon, int c0, int c1) {
  constexpr int E = D / 32;
  const arows::PagedParams& a = p.c.a;
  const int lane = threadIdx.x & 31, t = f / p.G, h = hk * p.G + f % p.G;
  const bool mine = lane * E >= c0 && lane * E < c1;  // columns c0 .. c1 - 1
  const int seen = a.causal ? max(len - (n - 1 - t), 0) : len;
  T* o = static_cast<T*>(a.o) + h * a.o_st[1] + int64_t(lo + t) * a.o_st[2] + lane * E;
  bool bad[E], any = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float x = to_f<T>(o[e]);
    any |= bad[e] = mine && x != x;
  }
  if (!__any_sync(0xffffffffu, any)) return;
  arows::PagedKeys<E> keys{a.pages, a.scales, a.table + b * a.table_st, a.Hkv, hk, a.page, a.num_pages, lane * E};
  any = false;
  for (int i = seen; i < horizon; ++i) {
    float k[E], v[E];
    keys.load(i, k, v);
#pragma unroll
    for (int e = 0; e < E; ++e) any |= bad[e] && v[e] != v[e];
  }
  if (!__any_sync(0xffffffffu, any)) return;
  const T* q = static_cast<const T*>(a.q) + h * a.q_st[1] + int64_t(lo + t) * a.q_st[2] + lane * E;
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = to_f<T>(q[e]);
  arows::attend_row<E>(keys, seen, a.scale, x);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (mine) o[e] = from_f<T>(x[e]);
}

// 32 output values of a row, in the widest stores that its alignment allows.
template <typename T>
__device__ __forceinline__ void store32(T* o, const float* v, float f, int wide) {
  if (wide) {
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = pack2<T>(v[2 * e] * f, v[2 * e + 1] * f);
    if (wide == 32) {
#pragma unroll
      for (int e = 0; e < 16; e += 8)
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(o + 2 * e), "r"(w[e]), "r"(w[e + 1]),
                     "r"(w[e + 2]), "r"(w[e + 3]), "r"(w[e + 4]), "r"(w[e + 5]), "r"(w[e + 6]), "r"(w[e + 7])
                     : "memory");
    } else {
#pragma unroll
      for (int e = 0; e < 16; e += 4) *reinterpret_cast<uint4*>(o + 2 * e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = from_f<T>(v[e] * f);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1) chunk_kernel(const Params p) {
  using C = Cfg<D>;
  constexpr int RB = C::RB, NS = C::NS, SPT = C::SPT;
  constexpr uint32_t IDESC_S = prefill::idesc_f16(0, 0, 0, BM, BH);
  constexpr uint32_t IDESC_PV = prefill::idesc_f16(0, 0, 1, BM, D);

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float4* tab = reinterpret_cast<float4*>(sm + C::TAB_OFF);
  int64_t* at_s = reinterpret_cast<int64_t*>(sm + C::ID_OFF);
  uint32_t* far_s = reinterpret_cast<uint32_t*>(sm + C::FAR_OFF);
  float* fac_s = reinterpret_cast<float*>(sm + C::FAC_OFF);
  float2* ml_s = reinterpret_cast<float2*>(sm + C::ML_OFF);
  volatile float* m_sh = reinterpret_cast<volatile float*>(sm + C::MSH_OFF);
  int64_t* prefix = reinterpret_cast<int64_t*>(sm + C::PREFIX_OFF);
  Range* ranges = reinterpret_cast<Range*>(sm + C::RANGE_OFF);
  Piece* list = reinterpret_cast<Piece*>(sm + C::PIECE_OFF);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);  // [NS] a stage's operand is in
  uint64_t* empty = full + NS;           // [NS] its products are done
  uint64_t* q_full = empty + NS;
  uint64_t* q_empty = q_full + 1;        // the item's last S has read Q
  uint64_t* s_full = q_empty + 1;        // [4] the unit's S is complete
  uint64_t* p_full = s_full + 4;         // [4]
  uint64_t* o_done = p_full + 4;         // [4] its P V is complete
  uint64_t* o_free = o_done + 4;         // the epilogue has read O
  uint64_t* tab_full = o_free + 1;       // [TABLES]
  uint64_t* tab_empty = tab_full + TABLES;
  uint64_t* token = tab_empty + TABLES;  // [2 warpgroups][4 quarters]: the shared maximum after the group's unit
  uint64_t* piece_full = token + 8;      // [PIECES]
  uint64_t* piece_empty = piece_full + PIECES;
  uint64_t* meet = piece_empty + PIECES;  // [4 quarters]: the two softmax warps of the same rows
  uint64_t* written = meet + 4;          // the softmax warps are done
  uint64_t* drain = written + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* again = abort_flag + 1;
  static_assert((2 * NS + 2 + 12 + 1 + 2 * TABLES + 8 + 2 * PIECES + 4 + 3) * 8 + 12 <= C::BAR_BYTES, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 4);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, CONV_WARPS);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(o_free, 8);
    for (int i = 0; i < TABLES; ++i) {
      mbar_init(&tab_full[i], 1);
      mbar_init(&tab_empty[i], 4 * SPT + 8);  // the V loads and the softmax warps
    }
    for (int i = 0; i < 8; ++i) mbar_init(&token[i], 1);
    for (int i = 0; i < PIECES; ++i) {
      mbar_init(&piece_full[i], 1);
      mbar_init(&piece_empty[i], CONV_WARPS + 11);  // eight softmax warps, the products' two, the tables'
    }
    for (int i = 0; i < 4; ++i) mbar_init(&meet[i], 2);
    mbar_init(written, 8);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    *abort_flag = 0;
    *again = 0;
    fence_barrier_init();
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // A programmatic dependent of the stream's previous kernel: global memory is read only past this point.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  {
    const int NR = p.c.a.B + 2;
    for (int r = warp; r < NR; r += THREADS / 32) {
      const Range x = range_of(p, r);
      if (blockIdx.x == 0 && lane == 0 && r > 0 && r <= p.c.a.B) arows::chunk_range(p.c, r - 1, STATUS, true);
      const int nb = (x.n * p.G + RB - 1) / RB;
      int64_t s = 0;
      for (int k = lane; k < nb; k += 32) s += block_of<RB>(p, x, k).units;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) prefix[r + 1] = s * p.c.a.Hkv, ranges[r] = x;
    }
    __syncthreads();
    if (warp == 0) {
      int64_t run = 0;
      for (int r0 = 0; r0 < NR; r0 += 32) {
        int64_t x = r0 + lane < NR ? prefix[r0 + lane + 1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        if (r0 + lane < NR) prefix[r0 + lane + 1] = run + x;
        run += __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) prefix[0] = 0;
    }
  }
  prefill::tc_fence_before();
  __syncthreads();
  prefill::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // Piece number i of the list (the end of it, or a wait that gave up: false); done with, its place is free.
  auto piece = [&](int i) {
    bool ok = wait_or_abort(&piece_full[i % PIECES], (i / PIECES) & 1, abort_flag, 157);
    ok = __all_sync(0xffffffffu, ok);
    return ok && list[i % PIECES].units > 0;
  };
  auto piece_done = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&piece_empty[i % PIECES]);
  };

  if (warp >= CONV_WARP + CONV_WARPS) {
    reg_dec<72>();
    if (warp == PLAN_WARP) {
      // ---------------------------------------------------------------------------------- the list of pieces
      Sched<RB> sched(p, prefix, ranges);
      Piece w;
      bool more = true;
      for (int i = 0; more; ++i) {
        more = sched.next(w);
        if (!more) w.units = 0;
        bool ok = i < PIECES || wait_or_abort(&piece_empty[i % PIECES], ((i / PIECES) - 1) & 1, abort_flag, STATUS_PLAN);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) {
          list[i % PIECES] = w;
          mbar_arrive(&piece_full[i % PIECES]);
        }
        __syncwarp();
      }
    } else if (warp == MMA_WARP || warp == SCORE_WARP) {
      // ---------------------------------------------------------------------------------- MMA issuers
      // One warp issues the S products, one the P V, so that neither's waits hold up the other's. Each walks the units as a
      // whole, with values that are the same in all lanes; one lane's predicate issues.
      const bool scores = warp == SCORE_WARP;
      const uint32_t lead = elect_one();
      auto uni = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
      auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
        return __all_sync(0xffffffffu, wait_or_abort<0>(bar, parity, abort_flag, where)) != 0;
      };
      const uint32_t tm = uni(tmem);
      int pieces = 0, base = 0, g01 = 0, g23 = 0;  // pieces and ring entries so far; units of each buffer so far
      bool ok = true;
      while (ok && piece(pieces)) {
        const bool pair = uni(list[pieces % PIECES].pair) != 0;
        const int nt = uni(list[pieces % PIECES].nt), units = (pair ? 4 : 2) * nt;
        // operands' descriptors: the K-major tiles' (Q, K) and the MN-major V's; tiles differ in the low word's address
        const uint32_t q_desc = smem_u32(sm) >> 4 | 1u << 16;
        const uint32_t s_desc = smem_u32(sm + C::K_OFF) >> 4 | uint32_t(scores ? 16 >> 4 : C::BOX >> 4) << 16;
        if (scores) {
          ok = wait(q_full, pieces & 1, 141);
        } else if (pieces > 0) {
          ok = wait(o_free, (pieces - 1) & 1, 144);
        }
#pragma unroll 1
        for (int i = 0; ok && i < units; ++i) {
          const int ht = pair ? i >> 1 : i, half = ht & 1, buf = i & 3, nth = (i & 2 ? g23 : g01) + (i >> 2);
          const int e = (base + (scores ? k_entry(pair, ht >> 1) : v_entry(pair, nt, ht >> 1))) * SPT + (C::WIDE ? half : 0);
          // whether the unit is its stage's first, its last
          const bool begins = C::WIDE || (half == 0 && (!pair || !(i & 1))), ends = C::WIDE || (half && (!pair || (i & 1)));
          if (scores) {  // S overwrites the buffer's last P: its P V is done
            if (nth > 0) ok = wait(&o_done[buf], (nth - 1) & 1, 161);
          } else {
            ok = wait(&p_full[buf], nth & 1, 143);
          }
          const uint32_t q = q_desc + (pair && (i & 1) ? C::QTILE >> 4 : 0);
          const bool own = !C::WIDE;  // each warpgroup its O
          const uint32_t o = tm + C::O_COL + (own && (i & 1) ? D : 0);
          const int st = e % NS;
          if (begins && ok) ok = wait(&full[st], (e / NS) & 1, 142);
          if (!ok) break;
          prefill::tc_fence_after();
          const uint32_t x = s_desc + st * (C::STAGE >> 4) + (C::WIDE ? 0 : half * (BH * 128 >> 4));
          if (scores) {
#pragma unroll 1
            for (uint32_t bx = 0; bx < D / 64; ++bx)
#pragma unroll
              for (uint32_t kk = 0; kk < 4; ++kk)
                mma_ss(lead, tm + buf * BH, q + ((bx * BM * 128 + kk * 32) >> 4), x + ((bx * C::BOX + kk * 32) >> 4), IDESC_S,
                       bx + kk > 0 ? 1u : 0u);
          } else {
#pragma unroll
            for (int kk = 0; kk < BH / 16; ++kk)
              mma_ts(lead, o, tm + buf * BH + kk * 8, x + ((kk * 16 * 128) >> 4), IDESC_PV,
                     (own ? i > 1 : i > 0) || kk > 0 ? 1u : 0u);
          }
          if (ends) mma_commit(lead, &empty[st]);
          mma_commit(lead, scores ? &s_full[buf] : &o_done[buf]);
          if (scores && i == units - 1) mma_commit(lead, q_empty);
        }
        ok = ok && __all_sync(0xffffffffu, !*abort_flag);
        piece_done(pieces);
        ++pieces;
        base += 2 * nt;
        g01 += (units + 2) >> 2;
        g23 += units >> 2;
      }
      if (lead) {
        prefill::umma_commit(&drain[scores]);
        mbar_wait(&drain[scores], 0, 146);
      }
      __syncwarp();
    } else if (warp == TABLE_WARP) {
      // ---------------------------------------------------------------------------------- page ids and scales, ahead
      // A slice of 16 keys: its K scale; its V scale's logarithm, for the maximum not below -100; the factor that takes a sum
      // of its weights to l's scale, 1 / s_v; and the logarithm itself. Where s_v is so small, or so far below a scale
      // before it in the piece, that weights of fp32's full range times 1 / s_v could miss keys that count in l, the
      // factor is 0 and the slice is marked: its sum is formed apart.
      // Four tiles at a time, a lane a slice, the next four asked for while these wait for their places.
      int g = 0;
      bool ok = true;
      const int per = min(8, BN >> p.lpage);  // pages a tile
      for (int i = 0; ok && piece(i); ++i) {
        const Piece& w = list[i % PIECES];
        const int32_t* row = p.c.a.table + int64_t(max(w.b, 0)) * p.c.a.table_st;
        const int key0 = w.kt0 * BN, horizon = w.horizon, hk = w.hk, nt = w.nt;
        float most = -INFINITY;
        auto fetch = [&](int t, int& id, float& ks, float& vs) {
          const int key = key0 + t * BN + lane * 16;
          id = -1, ks = 0.f, vs = 0.f;
          if (key < horizon && t + (lane >> 3) < nt) {
            id = row[key >> p.lpage];
            if (id < 0 || id >= p.c.a.num_pages) {
              report_bad_index(STATUS);
              id = -1;
            } else {
              const float* sc = p.c.a.scales + int64_t(id) * 2 * p.c.a.Hkv + hk;
              ks = sc[0], vs = sc[p.c.a.Hkv];
            }
          }
        };
        int id;
        float ks, vs;
        fetch(0, id, ks, vs);
        for (int t = 0; ok && t < nt; t += 4) {
          const int cid = id;
          const float cks = ks, vl = log2f(vs);
          const bool held = cid >= 0, there = key0 + t * BN + lane * 16 < horizon && t + (lane >> 3) < nt;
          fetch(t + 4, id, ks, vs);
          // the largest scale up to each tile
          float hi = vl;
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
#pragma unroll
          for (int o = 8; o < 32; o <<= 1) {
            const float y = __shfl_up_sync(0xffffffffu, hi, o);
            if (lane >= o) hi = fmaxf(hi, y);
          }
          hi = fmaxf(hi, most);
          most = __shfl_sync(0xffffffffu, hi, 31);
          const bool apart = there && vl < fmaxf(-100.f, hi - 64.f);  // (also a page that is none: it counts as zeros)
          const float4 f = make_float4(cks, fmaxf(vl, -100.f), apart ? 0.f : exp2f(-fmaxf(vl, -100.f)), vl);
          const uint32_t marked = __ballot_sync(0xffffffffu, apart);
          const uint32_t whole = __ballot_sync(0xffffffffu, held && key0 + t * BN + lane * 16 + 15 < horizon);
          const int pg = __shfl_sync(0xffffffffu, cid, (lane & 24) | ((lane & 7) * 8 / per & 7));  // the tile's page lane % 8
          for (int j = 0; j < min(4, nt - t); ++j, ++g) {
            const int s = g % TABLES;
            if (g >= TABLES) ok = wait_or_abort(&tab_empty[s], ((g / TABLES) - 1) & 1, abort_flag, 147);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (lane >> 3 == j) {
              tab[s * 8 + (lane & 7)] = f;
              if ((lane & 7) < per) at_s[s * 8 + (lane & 7)] = pg < 0 ? -1 : (int64_t(pg) * 2 * p.c.a.Hkv + hk) * (D << p.lpage);
              if ((lane & 7) == 0) far_s[s] = (marked >> (8 * j) & 255u) | ((whole >> (8 * j) & 255u) == 255u ? WHOLE : 0u);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&tab_full[s]);
          }
        }
        piece_done(i);
      }
    }
  } else if (warp >= CONV_WARP) {
    // ------------------------------------------------------------------------------------ codes into operand tiles
    reg_dec<72>();
    // A thread takes units of 16 codes: unit ul + 4 h of keys r0, r0 + 32, .. Eight lanes that store 16 bytes each then fill 128:
    // four units of two keys, whose swizzles are apart.
    constexpr int UH = D / 64, KP = C::SK / 32, LD = KP * UH;  // 64-dim boxes, keys and units a thread and stage
    const int tid = threadIdx.x - CONV_WARP * 32, ul = tid & 3, r0 = (tid & 127) >> 2;
    const int group = tid >> 7;  // the two warpgroups take the stages in turn
    const int page = 1 << p.lpage;
    const int64_t kv_off = int64_t(p.c.a.Hkv) * (D << p.lpage);  // from a page's K to its V
    const uint32_t dst0 = r0 * 128 + ((2 * ul ^ (r0 & 7)) << 4), dst1 = r0 * 128 + (((2 * ul + 1) ^ (r0 & 7)) << 4);
    int pieces = 0, g = 0, gt = 0;  // pieces, stages and tiles so far
    bool ok = true;
    while (ok && piece(pieces)) {
      const Piece& w = list[pieces % PIECES];
      const int horizon = w.horizon, hk = w.hk, nt = w.nt, kt0 = w.kt0;
      const bool pair = w.pair;
      // ---- queries: rows as they lie, f16, K-major swizzled; and the rows' score factors
      if (pieces > 0) ok = wait_or_abort(q_empty, (pieces - 1) & 1, abort_flag, 148);
      if (!__all_sync(0xffffffffu, ok)) break;
      {
        constexpr int LPR = D / 8;          // lanes a row
        constexpr int RPP = CT / LPR;       // rows a pass
        constexpr int HOLD = 4;             // passes whose loads are in flight
        const int qr = tid / LPR, qc = tid % LPR;
        const int rows = w.rows, tiles = pair ? 2 * BM : BM;
        const uint32_t dq = uint32_t(qc >> 3) * (BM * 128) + (((qc & 7) ^ (qr & 7)) << 4);  // (RPP is a multiple of 8)
        // the thread's row as (token, query head), stepped from pass to pass
        const int st = RPP / p.G, sg = RPP % p.G;
        int tq = (w.f0 + qr) / p.G, gq = (w.f0 + qr) % p.G;
        const T* qh = static_cast<const T*>(p.c.a.q) + int64_t(hk) * p.G * p.c.a.q_st[1] + int64_t(w.lo) * p.c.a.q_st[2] + qc * 8;
        float* fac = fac_s + (pieces & 1) * RB;
#pragma unroll 1
        for (int b0 = qr; b0 < tiles; b0 += RPP * HOLD) {
          uint4 raw[HOLD];
#pragma unroll
          for (int i = 0; i < HOLD; ++i) {
            raw[i] = make_uint4(0, 0, 0, 0);
            if (b0 + i * RPP < rows) {
              const T* src = qh + gq * p.c.a.q_st[1] + tq * p.c.a.q_st[2];
              if (p.wide_q) {
                raw[i] = *reinterpret_cast<const uint4*>(src);
              } else {
                for (int e = 0; e < 8; e += 2) {
                  const uint32_t lo = reinterpret_cast<const uint16_t*>(src)[e], hi = reinterpret_cast<const uint16_t*>(src)[e + 1];
                  (e == 0 ? raw[i].x : e == 2 ? raw[i].y : e == 4 ? raw[i].z : raw[i].w) = lo | hi << 16;
                }
              }
            }
            tq += st, gq += sg;
            if (gq >= p.G) gq -= p.G, ++tq;
          }
          [[maybe_unused]] uint32_t mx[HOLD];
          if constexpr (!std::is_same<T, __half>::value) {  // the rows' largest magnitudes (bits of bf16 values rise with them)
#pragma unroll
            for (int i = 0; i < HOLD; ++i) {
              const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&raw[i]);
              const __nv_bfloat162 m2 = __hmax2(__hmax2(__habs2(h2[0]), __habs2(h2[1])), __hmax2(__habs2(h2[2]), __habs2(h2[3])));
              const uint32_t m = *reinterpret_cast<const uint32_t*>(&m2);  // (NaN is passed over, unless both are)
              mx[i] = max(m >> 16, m & 0xffffu);
              mx[i] = mx[i] > 0x7f80u ? 0u : mx[i];
            }
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1)
#pragma unroll
              for (int i = 0; i < HOLD; ++i) mx[i] = max(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
          }
#pragma unroll
          for (int i = 0; i < HOLD; ++i) {
            const int r = b0 + i * RPP;
            uint4 x = raw[i];
            float f = p.scale_log2;
            if constexpr (!std::is_same<T, __half>::value) {
              // times 2^(14 - ex), the largest value's exponent to 14; undone by the factor, in two powers
              const int ex = mx[i] ? min(max(int(mx[i] >> 7) - 127, -112), 127) : 14;
              const float up = __uint_as_float(uint32_t(127 + 14 - ex) << 23);
              uint32_t* wx = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                wx[e] = pack2<__half>(__uint_as_float(wx[e] << 16) * up, __uint_as_float(wx[e] & 0xffff0000u) * up);
              const int d = ex - 14;
              f = f * __uint_as_float(uint32_t(127 + d / 2) << 23) * __uint_as_float(uint32_t(127 + d - d / 2) << 23);
            }
            if (p.flip) x.x ^= 0x80008000u, x.y ^= 0x80008000u, x.z ^= 0x80008000u, x.w ^= 0x80008000u;
            if (r < tiles) {
              *reinterpret_cast<uint4*>(sm + (r / BM) * C::QTILE + dq + (r % BM) * 128) = x;
              if (qc == 0) fac[r] = f;
            }
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      // ---- codes: a stage's loads, and behind the other group's stage its operand
      const int fills = 2 * nt * SPT;  // (even: each group's turns go on from piece to piece)
      int tabs = 0;  // tiles of the piece whose places are known to be in
#pragma unroll 1
      for (int s = group; s < fills; s += 2) {
        int kind, t;
        entry(pair, nt, s / SPT, kind, t);
        const int slot = (gt + t) % TABLES;
        if (t >= tabs) {
          if (ok) ok = wait_or_abort(&tab_full[slot], ((gt + t) / TABLES) & 1, abort_flag, 149);
          tabs = t + 1;
        }
        const int end = ok ? horizon - (kt0 + t) * BN : 0;  // keys of the tile that some row sees
        const uint8_t* from = p.c.a.pages + kind * kv_off + ul * 16;
        const int r1 = r0 + (s % SPT) * C::SK;  // the thread's first key in the tile
        const int64_t* at = at_s + slot * 8;
        const uint8_t* x0[KP];
#pragma unroll
        for (int k = 0; k < KP; ++k) {
          const int r = r1 + 32 * k;
          x0[k] = from + at[r >> p.lpage] + (r & (page - 1)) * D;
        }
        uint4 x[LD];
        if (ok && (far_s[slot] & WHOLE)) {
#pragma unroll
          for (int k = 0; k < KP; ++k)
#pragma unroll
            for (int h = 0; h < UH; ++h) x[k * UH + h] = ld_codes(x0[k] + 64 * h);
        } else {  // the tile's last keys, or a page that is none, are zeros
#pragma unroll
          for (int k = 0; k < KP; ++k)
#pragma unroll
            for (int h = 0; h < UH; ++h)
              x[k * UH + h] = load_if(x0[k] + 64 * h, r1 + 32 * k < end && at[(r1 + 32 * k) >> p.lpage] >= 0);
        }
        if (kind == 1) {  // the tile's places have been used
          __syncwarp();
          if (lane == 0) mbar_arrive(&tab_empty[slot]);
        }
        const int gs = g + s, st = gs % NS;
        if (ok && gs >= NS) ok = wait_or_abort(&empty[st], ((gs / NS) - 1) & 1, abort_flag, 150);
        uint8_t* d = sm + C::K_OFF + st * C::STAGE;
#pragma unroll
        for (int k = 0; k < KP; ++k)
#pragma unroll
          for (int h = 0; h < UH; ++h) {
            const uint4 c = x[k * UH + h];
            uint4 a, b;
            kv8::dec4(c.x, a.x, a.y);
            kv8::dec4(c.y, a.z, a.w);
            kv8::dec4(c.z, b.x, b.y);
            kv8::dec4(c.w, b.z, b.w);
            *reinterpret_cast<uint4*>(d + dst0 + h * C::BOX + k * (32 * 128)) = a;
            *reinterpret_cast<uint4*>(d + dst1 + h * C::BOX + k * (32 * 128)) = b;
          }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
      }
      g += fills;
      ok = __all_sync(0xffffffffu, ok);
      piece_done(pieces);
      ++pieces;
      gt += nt;
    }
    if (!ok) *abort_flag = 1;
  } else {
    // ------------------------------------------------------------------------------------ softmax, epilogue
    reg_inc<128>();
    const int wg = warp >> 2, quarter = warp & 3, r = 32 * quarter + lane;
    const uint32_t lane_base = tmem + (uint32_t(32 * quarter) << 16);
    const uint32_t o_col = lane_base + C::O_COL + (C::WIDE ? 0 : wg * D);
    int pieces = 0, gt = 0, g01 = 0, g23 = 0, met = 0;  // pieces, tiles, units of each buffer so far; meetings
    auto meet_other = [&](bool& ok) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&meet[quarter]);
      if (ok) ok = wait_or_abort(&meet[quarter], met & 1, abort_flag, 159);
      ++met;
    };
    bool ok = true;
    int4 rec0 = make_int4(0, 0, 0, 0), rec1 = rec0;
    while (piece(pieces)) {
      const Piece& w = list[pieces % PIECES];
      const bool pair = w.pair;
      const int units = (pair ? 4 : 2) * w.nt, kt0 = w.kt0;
      const int done = g01 + g23;  // each warpgroup's units before the piece's
      const int row = r + (pair ? wg * BM : 0);  // in the item
      const bool live = row < w.rows;
      const int tok = (w.f0 + row) / p.G;
      // the last key that the row sees (rows past the item's are zeros; nothing of them is kept)
      const int lim = !live ? w.horizon - 1 : (p.c.a.causal ? w.len - (w.n - 1 - tok) : w.len) - 1;
      float m = -FLT_MAX, l = 0.f, fac = 0.f;
      bool far = false;  // the row is loud
      // Waits for the P V of the piece's unit n. (Barriers are waited for within one phase of where they are: S_i comes after
      // the P V of unit i - 4, the buffer's last.)
      auto pv_done = [&](int n) {
        return wait_or_abort(&o_done[n & 3], ((n & 2 ? g23 : g01) + (n >> 2)) & 1, abort_flag, 153);
      };
      for (int i = wg; i < units; i += 2) {
        const int ht = pair ? i >> 1 : i, t = ht >> 1, half = ht & 1, slot = (gt + t) % TABLES;
        const uint32_t s_col = lane_base + (i & 3) * BH;
        if (ok) ok = wait_or_abort(&s_full[i & 3], ((i & 2 ? g23 : g01) + (i >> 2)) & 1, abort_flag, 151);
        ok = __all_sync(0xffffffffu, ok);
        prefill::tc_fence_after();
        const int over = lim - (kt0 + t) * BN - half * BH;  // the last column that the row sees
        // Masked tiles are few: their scores are masked in place, so that all tiles share one short piece of code.
        for (int c = max(__reduce_min_sync(0xffffffffu, over + 1), 0) & ~15; c < BH; c += 16) {
          float x[16];
          prefill2::tmem_ld16(s_col + c, x);
          prefill::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = c + e > over ? -INFINITY : x[e];
          prefill::tmem_st16(s_col + c, reinterpret_cast<const uint32_t*>(x));
          prefill::tmem_wait_st();
        }
        if (i < 2) fac = fac_s[(pieces & 1) * RB + row];
        const float4* sc = tab + slot * 8 + half * 4;
        float s[BH];
        prefill::tmem_ld32(s_col, s);
        prefill::tmem_ld32(s_col + 32, s + 32);
        wait_ld32(s);
        wait_ld32(s + 32);
        // The row's largest score with the values' scale (a factor is never 0: -inf times it stays -inf).
        auto largest = [&] {
          float top = -INFINITY;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 f = *reinterpret_cast<const float2*>(sc + q);
            const float* x = s + 16 * q;
            float a = max3(x[0], x[1], x[2]), b = max3(x[3], x[4], x[5]);
            a = max3(a, x[6], x[7]), b = max3(b, x[8], x[9]);
            a = max3(a, x[10], x[11]), b = max3(b, x[12], x[13]);
            a = max3(a, x[14], x[15]);
            top = fmaxf(top, fmaf(fmaxf(a, b), fmaxf(fac * f.x, FLT_MIN), f.y));
          }
          return top;
        };
        // The maximum moves to `now`: what was summed against the old one follows. `prev`: the unit whose P V must be done.
        auto move_to = [&](float now, int prev) {
          const float corr = prefill::ex2f(m - now);
          if (prev >= 0) {  // O holds something
            if (ok) ok = pv_done(prev);
            ok = __all_sync(0xffffffffu, ok);
            prefill::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float ov[16];
              prefill2::tmem_ld16(o_col + c, ov);
              prefill::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) ov[e] *= corr;
              prefill::tmem_st16(o_col + c, reinterpret_cast<const uint32_t*>(ov));
            }
            prefill::tmem_wait_st();
          }
          l = shrink(l, m - now);
          m = now;
        };
        const float top = largest();
        if (C::WIDE && i > 0) {  // the maximum after the unit before
          if (ok) ok = wait_or_abort(&token[(1 - wg) * 4 + quarter], (done + ((i - 1) >> 1)) & 1, abort_flag, 152);
          const float now = m_sh[r];
          if (now != m) {
            l = shrink(l, m - now);
            m = now;
            far = is_loud(m);
          }
        }
        const bool move = top - m > TOP + 8.f;
        bool loud = false;  // of some of the warp's rows
        if (__any_sync(0xffffffffu, move || far)) {
          move_to(move ? top - TOP : m, i - (C::WIDE ? 1 : 2));
          far = is_loud(m);
          loud = __any_sync(0xffffffffu, far);
          if (loud) l = loud_weights(s_col, sc, far_s[slot] >> (4 * half), fac, m, l);
        }
        if (C::WIDE) {
          m_sh[r] = m;
          __syncwarp();
          if (lane == 0) mbar_arrive(&token[wg * 4 + quarter]);
        }
        // weights; P_i takes the place of S_i
        if (!loud) {
          uint32_t pk[32];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 f = sc[q];
            const float mul = fmaxf(fac * f.x, FLT_MIN), add = f.w - m;
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float2 y = kv8::fma2(make_float2(s[16 * q + e], s[16 * q + e + 1]), make_float2(mul, mul), make_float2(add, add));
              y.x = prefill::ex2f(y.x), y.y = prefill::ex2f(y.y);
              sum = add2(sum, y);
              pk[8 * q + e / 2] = pack2<__half>(y.x, y.y);
            }
            l = fmaf(sum.x + sum.y, f.z, l);
          }
          for (uint32_t marked = far_s[slot] >> (4 * half) & 15u; marked; marked &= marked - 1) {  // (rare)
            const int q = __ffs(marked) - 1;
            const float mul = fmaxf(fac * sc[q].x, FLT_MIN);
            float x[16];
            prefill2::tmem_ld16(s_col + 16 * q, x);
            prefill::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) l += prefill::ex2f(fmaf(x[e], mul, -m));
          }
          prefill::tmem_st32(s_col, reinterpret_cast<const float*>(pk));
        }
        prefill::tmem_wait_st();
        prefill::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&p_full[i & 3]);
          if (half || !pair) mbar_arrive(&tab_empty[slot]);
        }
      }
      // -------------------------------------------------------------------------------- the piece's end
      float f0 = 1.f, f1 = 0.f;  // factors of this group's O, or of O 0 and O 1
      if (pair) {
        if (ok) ok = pv_done(units - 2 + wg);
      } else {
        ml_s[wg * BM + r] = make_float2(m, l);
        meet_other(ok);
        const float2 x = ml_s[r], y = ml_s[BM + r];
        m = fmaxf(x.x, y.x);  // (a shared maximum never falls, so it is the later one)
        f0 = prefill::ex2f(x.x - m);
        f1 = prefill::ex2f(y.x - m);
        l = shrink(x.y, x.x - m) + shrink(y.y, y.x - m);
        if (C::WIDE) f0 = 1.f;
        meet_other(ok);  // (read before the next piece's are written)
        if (ok) ok = pv_done(units - 2);
        if (ok) ok = pv_done(units - 1);
      }
      ok = __all_sync(0xffffffffu, ok);
      prefill::tc_fence_after();
      const int first = pair ? 0 : wg * (D / 2), count = pair ? D : D / 2;  // this thread's columns of O
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      const uint32_t oc = pair ? o_col : lane_base + C::O_COL;
      T* out = static_cast<T*>(p.c.a.o) + int64_t(w.hk * p.G + (w.f0 + row) % p.G) * p.c.a.o_st[1] + int64_t(w.lo + tok) * p.c.a.o_st[2];
      float* part = p.ws_o + int64_t(w.slot) * (D * RB) + 4 * row;
#pragma unroll 1
      for (int c = first; c < first + count; c += 32) {
        float ov[32];
        prefill::tmem_ld32(oc + c, ov);
        prefill::tmem_wait_ld();
        if (!C::WIDE && !pair) {
          float o1[32];
          prefill::tmem_ld32(oc + D + c, o1);
          prefill::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) ov[e] = ov[e] * f0 + o1[e] * f1;
        }
        if (!live || !ok) continue;
        if (w.whole) {
          float sum = 0.f;  // (finite unless some value is not)
#pragma unroll
          for (int e = 0; e < 32; ++e) sum = fmaf(ov[e], 0.f, sum);
          if (sum != sum && l == l) *again = 1;
          store32<T>(out + c, ov, inv, p.wide_o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(part + (c + e) * RB) = make_float4(ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
        }
      }
      prefill::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      if (!w.whole && (pair || wg == 0)) {
        p.ws_ml[int64_t(w.slot) * 2 * RB + row] = m;
        p.ws_ml[int64_t(w.slot) * 2 * RB + RB + row] = l;
      }
      if (w.nparts) rec0 = make_int4(w.nparts, w.b, w.lo, w.n), rec1 = make_int4(w.len, w.hk, w.f0, w.rows);
      piece_done(pieces);
      ++pieces;
      gt += w.nt;
      g01 += (units + 2) >> 2;
      g23 += units >> 2;
    }
    if (!ok) *abort_flag = 1, rec0.x = 0;
    if (threadIdx.x == 0) {
      p.rec[2 * blockIdx.x] = rec0;
      p.rec[2 * blockIdx.x + 1] = rec1;
    }
    // The second look (rare), when all of the CTA's rows are written: its whole items' rows, a warp a row.
    __syncwarp();
    if (lane == 0) mbar_arrive(written);
    if (ok) ok = wait_or_abort(written, 0, abort_flag, 160);
    if (__all_sync(0xffffffffu, ok) && *again) {
      Sched<RB> sched(p, prefix, ranges);
      Piece y;
      while (sched.next(y))
        for (int x = warp; y.whole && x < y.rows; x += CONV_WARP)
          row_again<T, D>(p, y.b, y.lo, y.n, y.len, y.hk, y.f0 + x, y.horizon, 0, D);
    }
  }

  prefill::tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    prefill::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512));
  }
}

// Merges an item's parts: a block for the CTA that begins it and 16 pieces of 32 rows x 32 columns, a warp each, a lane a row.
// Two parts' loads are in flight at once. (A block a piece, with the parts shared by its warps, took 18 to 40 us a call: most
// of the many blocks have nothing to do.)
constexpr int COMBINE_WARPS = 16;

template <typename T, int D>
__global__ void __launch_bounds__(COMBINE_WARPS * 32) combine_kernel(const Params p) {
  constexpr int RB = Cfg<D>::RB;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 a = p.rec[2 * blockIdx.x], e4 = p.rec[2 * blockIdx.x + 1];
  const int lane = threadIdx.x & 31, task = blockIdx.y * COMBINE_WARPS + (threadIdx.x >> 5);
  const int parts = a.x, r0 = task / (D / 32) * 32, c0 = task % (D / 32) * 32, rows = e4.w, row = r0 + lane;
  if (parts == 0 || r0 >= rows) return;
  const float* ml = p.ws_ml + row;
  const float* ws = p.ws_o + int64_t(c0) * RB + 4 * row;
  auto slot = [&](int i) { return i == 0 ? 2 * int64_t(blockIdx.x) + 1 : 2 * (int64_t(blockIdx.x) + i); };
  float M = -FLT_MAX, L = 0.f, x[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) x[e] = 0.f;
  for (int i = 0; i < parts; i += 2) {
    float y[2][32], m[2], l[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t s = slot(min(i + k, parts - 1));
      m[k] = ml[s * 2 * RB], l[k] = ml[s * 2 * RB + RB];
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const float4 v = *reinterpret_cast<const float4*>(ws + s * (D * RB) + e * RB);
        y[k][e] = v.x, y[k][e + 1] = v.y, y[k][e + 2] = v.z, y[k][e + 3] = v.w;
      }
    }
    if (i + 1 == parts) m[1] = -FLT_MAX, l[1] = 0.f;
    const float now = fmaxf(M, fmaxf(m[0], m[1]));
    const float f = prefill::ex2f(M - now), g0 = prefill::ex2f(m[0] - now);
    const float g1 = i + 1 == parts ? 0.f : prefill::ex2f(m[1] - now);
    L = shrink(L, M - now) + shrink(l[0], m[0] - now) + shrink(l[1], m[1] - now);
    M = now;
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = fmaf(y[0][e], g0, x[e] * f);
    if (i + 1 < parts)
#pragma unroll
      for (int e = 0; e < 32; ++e) x[e] = fmaf(y[1][e], g1, x[e]);
  }
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
  const int f = e4.z + row, tok = f / p.G;
  float sum = 0.f;  // (finite unless some value is not)
#pragma unroll
  for (int e = 0; e < 32; ++e) sum = fmaf(x[e], 0.f, sum);
  if (row < rows)
    store32<T>(static_cast<T*>(p.c.a.o) + int64_t(e4.y * p.G + f % p.G) * p.c.a.o_st[1] + int64_t(a.z + tok) * p.c.a.o_st[2] + c0, x,
               inv, p.wide_o);
  uint32_t nan = __ballot_sync(0xffffffffu, row < rows && sum != sum && L == L);
  if (nan == 0) return;
  __syncwarp();
  const Block b = block_of<RB>(p, Range{a.z, a.w, e4.x}, e4.z / RB);
  for (; nan; nan &= nan - 1)
    row_again<T, D>(p, a.y, a.z, a.w, e4.x, e4.y, e4.z + r0 + __ffs(nan) - 1, b.horizon, c0, c0 + 32);
}

}  // namespace kv8chunk
}  // namespace lb2
