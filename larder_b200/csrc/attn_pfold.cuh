// Packed prompts on one CTA (tcgen05): blocks of 128 rows, a row being a (token, query head) of one KV head, so that the
// F = G query heads that share K and V fill a block with 128 / F tokens (F = 1 for more than 64 heads a KV head). A short
// prompt then leaves little of its last block empty, and a block reads few key tiles past its own tokens.
//
// What bounds a block is the chain load -> S -> softmax -> P V (-> epilogue) and the softmax's instructions, not the
// products. So the kernel is persistent, each CTA walking the plan's blocks (heaviest first) in rounds, with Q, K and V of
// the next block on their way and its first S computed while this one's O is written; and at head dims 64 and 128 a CTA
// takes half an SM's tensor memory and shared memory, so that two share the SM, one's products under the other's softmax.
// Measured (bf16, 32 / 8 heads x 128): 33 prompts of 8 to 441 rows, 4001 in all, 34 us on the device with the plan's launch
// (128 us with a CTA a block of one head, 55 us not persistent); 982 TFLOP/s at prompts of 4096 rows.
//
// A value that is infinite or NaN spoils the rows before it that share its tiles (0 times NaN): the epilogue only notes that
// a row came out non-finite, and at its end, when no warp waits for another any more, the CTA looks at its rows again
// (packed_row_again). That costs calls without such values nothing. One prompt of 4096 rows takes 0.15 ms; 0.33 ms with an
// infinity in its first row, which all rows see; 7.7 ms with a NaN in its last, where a block's rows are taken again.
//
// Roles (320 threads): warps 0-7 softmax and epilogue (warp w: TMEM lanes of quarter w % 4, key / O column half w / 4),
// warp 8 TMA (lane 0 Q and K, lane 1 V), warp 9 issues the MMAs. S_j = Q K_j^T and O += P_j V_j as in attn_prefill.cuh;
// rings and barriers run on counters that continue across blocks, and two barriers hand resources on: q_empty (the
// block's last S has read Q), o_free (the epilogue has read O).
#pragma once

#include "attn_prefill.cuh"
#include "attn_prefill2.cuh"

namespace lb2 {
namespace pfold {

using prefill::BM;
using prefill::Params;

constexpr int SOFTMAX_WARPS = 8;
constexpr int PRODUCER_WARP = 8;
constexpr int MMA_WARP = 9;
constexpr int THREADS = 320;

template <int D>
struct Cfg {
  static constexpr int BN = 64;                  // keys a tile
  static constexpr int CTAS = D == 256 ? 1 : 2;  // an SM
  static constexpr int TCOLS = 512 / CTAS;       // TMEM columns
  static constexpr int ST = 2;                   // K stages, V stages
  static constexpr int QBYTES = BM * D * 2;
  static constexpr int KBYTES = BN * D * 2;      // one K (or V) tile
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = Q_OFF + QBYTES;
  static constexpr int V_OFF = K_OFF + ST * KBYTES;
  static constexpr int BAR_OFF = V_OFF + ST * KBYTES;
  static constexpr int RED_OFF = BAR_OFF + 256;  // [2 halves][128 rows] fp32
  static constexpr int SMEM_BYTES = RED_OFF + 2 * BM * 4 + 1024;
  static constexpr int S_COL = 0;                // S (fp32)
  static constexpr int P_COL = BN;               // P (16-bit, BN / 2 columns)
  static constexpr int O_COL = 2 * BN;           // O
  static_assert(O_COL + D <= TCOLS, "TMEM budget");
  static_assert(SMEM_BYTES <= 232448 / CTAS - 1024, "shared memory budget");
};

// 32 bytes of one row in one store.
__device__ __forceinline__ void st_global32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Item (block, heads) r of CTA c of n: the heaviest-first list dealt in a snake, so that the CTAs' totals even out.
__device__ __forceinline__ int item_at(int r) {
  const int n = gridDim.x, c = blockIdx.x;
  return r * n + ((r & 1) ? n - 1 - c : c);
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, Cfg<D>::CTAS) pfold_kernel(const __grid_constant__ CUtensorMap qmap,
                                                                      const __grid_constant__ CUtensorMap kmap,
                                                                      const __grid_constant__ CUtensorMap vmap,
                                                                      const Params p) {
  using C = Cfg<D>;
  constexpr int BN = C::BN, ST = C::ST;
  constexpr int AB = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  constexpr uint32_t IDESC_S = prefill::idesc_f16(AB, 0, 0, BM, BN);
  constexpr uint32_t IDESC_PV = prefill::idesc_f16(AB, 0, 1, BM, D);

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;    // [ST]
  uint64_t* k_empty = k_full + ST;   // [ST]
  uint64_t* v_full = k_empty + ST;   // [ST]
  uint64_t* v_empty = v_full + ST;   // [ST]
  uint64_t* s_full = v_empty + ST;   // S_j complete
  uint64_t* s_free = s_full + 1;     // the softmax warps have loaded S_j
  uint64_t* p_full = s_free + 1;     // P_j written
  uint64_t* o_done = p_full + 1;     // P_j V_j complete
  uint64_t* o_free = o_done + 1;     // the softmax warps have read the block's O
  uint64_t* drain = o_free + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* again = abort_flag + 1;  // some row came out non-finite with a finite sum of weights
  static_assert((4 * ST + 8) * 8 + 12 <= 256, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, SOFTMAX_WARPS);
    mbar_init(p_full, SOFTMAX_WARPS);
    mbar_init(o_done, 1);
    mbar_init(o_free, SOFTMAX_WARPS);
    mbar_init(drain, 1);
    *abort_flag = 0;
    *again = 0;
    fence_barrier_init();
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TCOLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  prefill::tc_fence_before();
  __syncthreads();
  prefill::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the plan
  const int F = p.fold, heads = p.Hq / F, tpb = p.tpb;
  const int total = *p.pk_n * heads;

  if (warp == PRODUCER_WARP) {
    // ------------------------------------------------------------------------------------ TMA producers
    if (lane < 2) {
      if (lane == 0) {
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&kmap);
      } else {
        prefetch_tensormap(&vmap);
      }
      uint64_t* fullb = lane == 0 ? k_full : v_full;
      uint64_t* emptyb = lane == 0 ? k_empty : v_empty;
      const CUtensorMap* map = lane == 0 ? &kmap : &vmap;
      const int off = lane == 0 ? C::K_OFF : C::V_OFF;
      int jg = 0, qi = 0, q_issued = -1;
      bool stop = false;
      for (int r = 0, it; r * int(gridDim.x) < total && !stop; ++r) {
        if ((it = item_at(r)) >= total) continue;
        const int4 blk = p.pk[it / heads];
        const int h = it % heads * F, hk = h / p.G;
        if (blk.w == 0) continue;
        if (lane == 0) {
          if (qi > 0 && !mbar_wait(q_empty, (qi - 1) & 1, 121)) {
            *abort_flag = 1;
            break;
          }
          mbar_arrive_expect_tx(q_full, tpb * F * D * 2);
#pragma unroll
          for (int db = 0; db < D / 64; ++db)  // (64, F heads, tpb tokens) boxes: row = token F + head
            tma_load_4d(sm + C::Q_OFF + db * BM * 128, &qmap, db * 64, h, blk.x + blk.z * tpb, 0, q_full);
          q_issued = qi;
        }
        for (int j = 0; j < blk.w; ++j, ++jg) {
          const int st = jg % ST;
          if (*abort_flag || (jg >= ST && !mbar_wait(&emptyb[st], ((jg / ST) - 1) & 1, 122 + lane))) {
            *abort_flag = 1;
            stop = true;
            break;
          }
          mbar_arrive_expect_tx(&fullb[st], C::KBYTES);
#pragma unroll
          for (int db = 0; db < D / 64; ++db)
            tma_load_4d(sm + off + st * C::KBYTES + db * BN * 128, map, db * 64, blk.x + j * BN, hk, 0, &fullb[st]);
        }
        ++qi;
      }
      // Drain: everything this lane issued has landed before the CTA may end.
      if (lane == 0 && q_issued >= 0) mbar_wait(q_full, q_issued & 1, 124);
      for (int g = max(0, jg - ST); g < jg; ++g) mbar_wait(&fullb[g % ST], (g / ST) & 1, 125);
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      const uint32_t q_addr = smem_u32(sm + C::Q_OFF);
      bool ok = true;
      int js_g = 0, jp_g = 0, qi = 0;  // S and PV tiles issued; blocks with keys so far
      for (int r = 0, it; ok && r * int(gridDim.x) < total; ++r) {
        if ((it = item_at(r)) >= total) continue;
        const int nt = p.pk[it / heads].w;
        if (nt == 0) continue;
        ok = mbar_wait(q_full, qi & 1, 126);
        bool o_ok = qi == 0;  // O may be overwritten by this block's first PV
        int js = 0, jp = 0;
        uint64_t t0 = 0;
        for (uint32_t n = 1; ok && jp < nt; ++n) {
          if (jp < js && (jp > 0 || o_ok || (o_ok = mbar_test_wait(o_free, (qi - 1) & 1))) &&
              mbar_test_wait(&v_full[jp_g % ST], (jp_g / ST) & 1) && mbar_test_wait(p_full, jp_g & 1)) {
            const int st = jp_g % ST;
            prefill::tc_fence_after();
            const uint32_t v_addr = smem_u32(sm + C::V_OFF + st * C::KBYTES);
#pragma unroll
            for (int kk = 0; kk < BN / 16; ++kk)
              prefill::umma_ts(tmem + C::O_COL, tmem + C::P_COL + kk * 8,
                               prefill::sdesc(v_addr + kk * 16 * 128, BN * 128, 1024), IDESC_PV, (jp > 0 || kk > 0) ? 1u : 0u);
            prefill::umma_commit(o_done);
            prefill::umma_commit(&v_empty[st]);
            ++jp_g, ++jp;
            t0 = 0;
            continue;
          }
          if (js < nt && mbar_test_wait(&k_full[js_g % ST], (js_g / ST) & 1) &&
              (js_g == 0 || mbar_test_wait(s_free, (js_g - 1) & 1))) {
            const int st = js_g % ST;
            prefill::tc_fence_after();
            const uint32_t k_addr = smem_u32(sm + C::K_OFF + st * C::KBYTES);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              prefill::umma_ss(tmem + C::S_COL, prefill::sdesc(q_addr + (kk >> 2) * BM * 128 + (kk & 3) * 32, 16, 1024),
                               prefill::sdesc(k_addr + (kk >> 2) * BN * 128 + (kk & 3) * 32, 16, 1024), IDESC_S,
                               kk > 0 ? 1u : 0u);
            prefill::umma_commit(s_full);
            prefill::umma_commit(&k_empty[st]);
            ++js_g;
            if (++js == nt) prefill::umma_commit(q_empty);  // the block's S are done with Q
            t0 = 0;
            continue;
          }
          // Nothing ready: sleep on the barrier that gates the next product in the usual order.
          if (jp < js)
            mbar_try_wait_hint(p_full, jp_g & 1, 500);
          else if (js_g > 0 && !mbar_test_wait(s_free, (js_g - 1) & 1))
            mbar_try_wait_hint(s_free, (js_g - 1) & 1, 500);
          else
            mbar_try_wait_hint(&k_full[js_g % ST], (js_g / ST) & 1, 500);
          if ((n & 15) == 0) {
            if (*abort_flag) {
              ok = false;
              break;
            }
            const uint64_t now = globaltimer_ns();
            if (t0 == 0) {
              t0 = now;
            } else if (now - t0 > kWaitNs) {
              report_timeout(127);
              ok = false;
              break;
            }
          }
        }
        ++qi;
      }
      if (!ok) *abort_flag = 1;
      prefill::umma_commit(drain);
      mbar_wait(drain, 0, 128);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------------------------ softmax warps
    constexpr int HC = BN / 2;  // S columns (keys) a thread owns
    constexpr int HD = D / 2;   // O columns a thread owns
    constexpr float TOP = prefill::packed_top<T>();
    const int r = 32 * (warp & 3) + lane, half = warp >> 2;
    const uint32_t lane_base = tmem + (uint32_t(32 * (warp & 3)) << 16);
    const uint32_t pair_bar = 2 + (warp & 3);  // named barrier of the two warps of a lane quarter
    float* red = reinterpret_cast<float*>(sm + C::RED_OFF);
    const int tok = r / F, head = r - tok * F;  // the row's token in the block, and head
    bool ok = true;
    int jg = 0;
    for (int rr = 0, it; ok && rr * int(gridDim.x) < total; ++rr) {
      if ((it = item_at(rr)) >= total) continue;
      const int4 blk = p.pk[it / heads];
      const int h = it % heads * F + head, nt = blk.w;
      const int row = blk.z * tpb + tok;  // in its prompt
      const bool live = tok < tpb && row < blk.y;
      const int last = live ? row : -1;  // the last key that the row sees (rows of nothing see none)
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < nt; ++j) {
        const int g = jg + j;
        bool okj = ok && !*abort_flag && mbar_wait(s_full, g & 1, 129);
        okj = __all_sync(0xffffffffu, okj);
        float s[HC];
        if (okj) {
          prefill::tc_fence_after();
          prefill::tmem_ld32(lane_base + C::S_COL + half * HC, s);
          prefill::tmem_wait_ld();
          prefill::tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_free);
        } else {
#pragma unroll
          for (int c = 0; c < HC; ++c) s[c] = -INFINITY;
        }
        const int key0 = j * BN + half * HC;
        if (j * BN + BN - 1 > last) {
#pragma unroll
          for (int c = 0; c < HC; ++c)
            if (key0 + c > last) s[c] = -INFINITY;
        }
        // P with the running maximum, which moves only when a weight would pass 2^(TOP + 8) (or at the row's first key): one
        // barrier of the two warps asks whether any of their rows wants that (or a wait failed).
        float nm = m_run == -INFINITY ? 0.f : TOP - m_run;
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[HC / 2];
        auto weights = [&] {
#pragma unroll
          for (int c = 0; c < 4; ++c) ls[c] = 0.f;
#pragma unroll
          for (int c = 0; c < HC; c += 2) {
            const float e0 = prefill::ex2f(fmaf(s[c], p.scale_log2, nm)), e1 = prefill::ex2f(fmaf(s[c + 1], p.scale_log2, nm));
            ls[c & 3] += e0;
            ls[(c + 1) & 3] += e1;
            pk[c / 2] = pack2<T>(e0, e1);
          }
        };
        weights();
        const bool want = !okj || (live && (m_run == -INFINITY || !((ls[0] + ls[1]) + (ls[2] + ls[3]) <= 256.f)));
        uint32_t any_want;
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
            "bar.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
            : "=r"(any_want)
            : "r"(uint32_t(want)), "r"(pair_bar)
            : "memory");
        if (any_want) {
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < HC; ++c) mx[c & 3] = fmaxf(mx[c & 3], s[c]);
          float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          red[half * BM + r] = tmax;
          uint32_t all_ok;
          asm volatile(
              "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
              "bar.red.and.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
              : "=r"(all_ok)
              : "r"(uint32_t(okj)), "r"(pair_bar)
              : "memory");
          tmax = fmaxf(tmax, red[(1 - half) * BM + r]);
          asm volatile("bar.sync %0, 64;" ::"r"(pair_bar));
          if (!all_ok) {
            ok = false;
            break;
          }
          const float tmax2 = tmax * p.scale_log2;
          const bool move = tmax2 > m_run + 8.f;
          const float factor = move ? prefill::ex2f(m_run - tmax2) : 1.f;
          // (the maximum is the row's; l_run, this half's share of the sum, may be 0 where O is not)
          if (__any_sync(0xffffffffu, move && m_run != -INFINITY)) {
            if (!mbar_wait(o_done, (g - 1) & 1, 130)) ok = false;
            prefill::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              float ov[16];
              prefill2::tmem_ld16(lane_base + C::O_COL + half * HD + c, ov);
              prefill::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) ov[e] *= factor;
              prefill::tmem_st16(lane_base + C::O_COL + half * HD + c, reinterpret_cast<const uint32_t*>(ov));
            }
            prefill::tmem_wait_st();
          }
          if (move) {
            l_run *= factor;
            m_run = tmax2;
            nm = TOP - m_run;
            weights();
          }
        }
        if (j > 0 && !mbar_wait(o_done, (g - 1) & 1, 131)) ok = false;  // PV_{j-1} has read P
        prefill::tc_fence_after();
        prefill::tmem_st16(lane_base + C::P_COL + half * (HC / 2), pk);
        l_run += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        prefill::tmem_wait_st();
        prefill::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      if (ok && nt > 0) {
        if (!mbar_wait(o_done, (jg + nt - 1) & 1, 132)) ok = false;
        prefill::tc_fence_after();
      }
      // -------------------------------------------------------------------------------- epilogue of the block
      ok = __all_sync(0xffffffffu, ok);
      float l_tot = 0.f;
      if (nt > 0) {
        red[half * BM + r] = l_run;
        uint32_t all_ok;  // both warps leave the loop together or neither does
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
            "bar.red.and.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
            : "=r"(all_ok)
            : "r"(uint32_t(ok)), "r"(pair_bar)
            : "memory");
        ok = all_ok != 0;
        l_tot = red[r] + red[BM + r];
      }
      const bool have_o = nt > 0 && ok;
      T* orow = reinterpret_cast<T*>(p.o) + int64_t(h) * p.o_st[1] + int64_t(blk.x + row) * p.o_st[2] + half * HD;
      const float inv = (have_o && (l_tot > 0.f || l_tot != l_tot)) ? 1.f / l_tot : 0.f;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float ov[32];
        if (have_o) {
          prefill::tmem_ld32(lane_base + C::O_COL + half * HD + c, ov);
          prefill::tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) ov[e] = 0.f;
        }
        if (c + 32 >= HD && nt > 0) {  // O is read: the next block's first PV may overwrite it
          prefill::tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(o_free);
        }
        if (!live) continue;
        float sum = 0.f;  // (finite unless some value is not)
#pragma unroll
        for (int e = 0; e < 32; ++e) sum = fmaf(ov[e], 0.f, sum);
        if (sum != sum && l_tot == l_tot) *again = 1;
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = pack2<T>(ov[2 * e] * inv, ov[2 * e + 1] * inv);
        if (p.wide_o) {
          st_global32(orow + c, w);
          st_global32(orow + c + 16, w + 8);
        } else {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<uint4*>(orow + c + 2 * e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
        }
      }
      jg += nt;
    }
    if (!ok) *abort_flag = 1;
  }

  prefill::tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    prefill::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TCOLS));
  }
  // The second look (rare), when nothing waits for this CTA any more: its items' rows again, a warp a row.
  if (*again && !*abort_flag) {
    for (int r = 0, it; r * int(gridDim.x) < total; ++r) {
      if ((it = item_at(r)) >= total) continue;
      const int4 blk = p.pk[it / heads];
      const int first = blk.z * tpb, rows = min(tpb, blk.y - first) * F, end = min(blk.w * BN, p.T - blk.x);
      for (int x = warp; x < rows; x += THREADS / 32)
        prefill::packed_row_again<T, D>(p, blk.x, first + x / F, end, it % heads * F + x % F);
    }
  }
}

}  // namespace pfold
}  // namespace lb2
