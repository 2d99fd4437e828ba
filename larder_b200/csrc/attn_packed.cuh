// Packed prompts: the list of row blocks that the kernels take (attn_pfold.cuh, attn_prefill2.cuh's PK form).
//
// Prompt s is rows [cu[s], cu[s + 1]) of one row axis; its blocks of RB rows (256 on CTA pairs, 128 over the folded heads on one CTA) read
// its key tiles from the first up to the block's last row. The lengths are known on the device only, so the list is made
// there, by one block of threads: blocks in falling order of their index m in their prompt (the work of block m grows with
// m, so this is heaviest first but for prompts' last, partial blocks), prompts in order within an m. Each warp takes the
// values of m in turn: ballots over the prompts count those that reach m and place their blocks. Bounds that fall or
// pass T are clamped, so that no row is addressed outside the tensors whatever cu holds. Rows before the first prompt and
// past the last are listed as blocks without keys, whose outputs are zeros: ranges 0 and S + 1 of the plan, prompt s
// being range s + 1.
#pragma once

#include "common.cuh"

namespace lb2 {
namespace packed {

constexpr int THREADS = 256;

struct PlanParams {
  const int32_t* cu;
  int32_t* n;    // blocks listed
  int32_t* cnt;  // [T / rb + 2] ranges that reach m, then (after the scan) where m's blocks begin
  int32_t* at;   // [S + 3] where the ranges begin and the last one's end
  int4* out;
  int S, T, rb, bn;
};

__global__ void __launch_bounds__(THREADS) plan_kernel(const PlanParams p) {
  constexpr int HELD = 2048;  // bounds and counts up to so many stay in shared memory
  __shared__ int s_w[32], s_max, s_at[HELD], s_cnt[HELD];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the attention kernel waits for this one's end)
  int* const at = p.S + 3 <= HELD ? s_at : p.at;
  int* const cnt = p.T / p.rb + 2 <= HELD ? s_cnt : p.cnt;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_max = 0;
  __syncthreads();
  // bounds: 0, the running maximum of cu within [0, T], T
  int carry = 0;
  for (int b0 = 0; b0 <= p.S; b0 += THREADS) {
    const int s = b0 + tid;
    int x = s <= p.S ? min(max(p.cu[s], 0), p.T) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = max(x, y);
    }
    if (lane == 31) s_w[warp] = x;
    __syncthreads();
    int pre = carry, all = carry;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) pre = max(pre, s_w[w]);
      all = max(all, s_w[w]);
    }
    if (s <= p.S) at[s + 1] = max(x, pre);
    carry = all;
    __syncthreads();
  }
  if (tid == 0) at[0] = 0, at[p.S + 2] = p.T;
  __syncthreads();
  int mx = 0;
  for (int s = tid; s <= p.S + 1; s += THREADS) mx = max(mx, (at[s + 1] - at[s] + p.rb - 1) / p.rb);
  atomicMax(&s_max, mx);
  __syncthreads();
  const int M = s_max;  // m runs over 0 .. M - 1
  for (int m = warp; m < M; m += THREADS / 32) {
    int c = 0;
    for (int s0 = 0; s0 <= p.S + 1; s0 += 32) {
      const int s = s0 + lane;
      c += __popc(__ballot_sync(0xffffffffu, s <= p.S + 1 && at[s + 1] - at[s] > m * p.rb));
    }
    if (lane == 0) cnt[m] = c;
  }
  __syncthreads();
  // where m's blocks begin: the blocks of all larger m come first
  int run = 0;
  for (int b0 = 0; b0 < M; b0 += THREADS) {
    const int m = M - 1 - b0 - tid;
    const int own = m >= 0 ? cnt[m] : 0;
    int x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_w[warp] = x;
    __syncthreads();
    int pre = run, all = run;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) pre += s_w[w];
      all += s_w[w];
    }
    if (m >= 0) cnt[m] = pre + x - own;
    run = all;
    __syncthreads();
  }
  for (int m = warp; m < M; m += THREADS / 32) {
    int c = cnt[m];
    for (int s0 = 0; s0 <= p.S + 1; s0 += 32) {
      const int s = s0 + lane;
      const int a = s <= p.S + 1 ? at[s] : 0, n = s <= p.S + 1 ? at[s + 1] - a : 0;
      const uint32_t has = __ballot_sync(0xffffffffu, n > m * p.rb);
      if (n > m * p.rb)
        p.out[c + __popc(has & ((1u << lane) - 1))] =
            make_int4(a, n, m, s == 0 || s == p.S + 1 ? 0 : (min(n, (m + 1) * p.rb) + p.bn - 1) / p.bn);
      c += __popc(has);
    }
  }
  if (tid == 0) *p.n = run;
}

}  // namespace packed
}  // namespace lb2
