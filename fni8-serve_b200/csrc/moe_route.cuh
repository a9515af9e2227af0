// Routing of one token by one warp (fni8serve/models/moe.py:65-95): shared by the routing
// kernel (moe.cu) and the few-token layer (moe_few.cu), so both choose alike.
#pragma once
#include "fni8_common.cuh"

namespace fni8b {
namespace moe {

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// Order-preserving key of a float that is no NaN (-0 and +0 alike).
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
// warp-wide arg-max over indexes >= 0: the larger value wins, ties go to the lower index (two
// warp reductions; a shuffle tree over value and index took three times as long)
__device__ __forceinline__ void warp_argmax(float& v, int& i) {
  const uint32_t key = order_key(v);
  const uint32_t top = __reduce_max_sync(0xffffffffu, key);
  i = static_cast<int>(__reduce_min_sync(0xffffffffu, key == top ? static_cast<uint32_t>(i) : 0x7fffffffu));
  v = __uint_as_float((top & 0x80000000u) ? top & 0x7FFFFFFFu : ~top);
}

// Scores of logits row `lr` [E] and the top k of them: lane j < k returns slot j's expert in
// `out_i` and its weight in `out_w`. VPL = experts per lane (E <= 32 * VPL). The inputs are read
// from L2: few_down routes before its own wait, where a line of an older call in L1 may be stale.
template <int VPL>
__device__ __forceinline__ void route_token(const float* __restrict__ lr, int E, int k, int scoring,
                                            const float* __restrict__ sel_bias, int n_groups, int topk_group,
                                            int norm_topk, float scaling, int wdtype, int lane, int& out_i,
                                            float& out_w) {
  const float NEG = -INFINITY;
  float sc[VPL], sel[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = lane + 32 * i;
    sc[i] = e < E ? __ldcg(lr + e) : NEG;
  }
  if (scoring == FNI8_SCORE_SOFTMAX) {
    float mx = NEG;
#pragma unroll
    for (int i = 0; i < VPL; ++i) mx = fmaxf(mx, sc[i]);
    mx = warp_max(mx);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 32 * i;
      sc[i] = e < E ? expf(__fadd_rn(sc[i], -mx)) : 0.0f;
      sum = __fadd_rn(sum, sc[i]);
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      sc[i] = __fdiv_rn(sc[i], sum);
      sel[i] = (lane + 32 * i) < E ? sc[i] : NEG;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 32 * i;
      sc[i] = e < E ? __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-sc[i]))) : 0.0f;
      sel[i] = e < E ? (sel_bias ? __fadd_rn(sc[i], __ldcg(sel_bias + e)) : sc[i]) : NEG;
    }
  }
  if (n_groups > 0 && topk_group > 0) {
    // keep only the topk_group groups with the largest max score: lane g takes group g's
    // maximum, then one arg-max per kept group (a group without a score above -inf is none)
    const int epg = E / n_groups;
    int group[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) group[i] = (lane + 32 * i) / epg;
    float mine = NEG;
    for (int g = 0; g < n_groups; ++g) {
      float gm = NEG;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (lane + 32 * i < E && group[i] == g) gm = fmaxf(gm, sel[i]);
      gm = warp_max(gm);
      if (lane == g) mine = gm;
    }
    unsigned keep = 0;  // bitmask over groups (n_groups <= 32)
    for (int r = 0; r < topk_group; ++r) {
      const bool open = lane < n_groups && !(keep & (1u << lane)) && mine > NEG;
      float best = open ? mine : NEG;
      int bg = open ? lane : 0x7fffffff;
      warp_argmax(best, bg);
      if (bg != 0x7fffffff) keep |= 1u << bg;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 32 * i;
      if (e < E && !(keep & (1u << group[i]))) sel[i] = NEG;
    }
  }
  float my_w = 0.0f;
  int my_i = 0;
  float wsum = 0.0f;
  for (int j = 0; j < k; ++j) {
    float v = NEG;
    int idx = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 32 * i;
      if (e < E && (sel[i] > v || (sel[i] == v && e < idx))) {
        v = sel[i];
        idx = e;
      }
    }
    warp_argmax(v, idx);
    float w = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      if (lane + 32 * i == idx) {
        w = sc[i];
        sel[i] = NEG;  // taken
        // a -inf entry can only be re-picked if everything left is -inf; mark it below E
      }
    }
    w = __shfl_sync(0xffffffffu, w, idx & 31);
    if (lane == j) {  // slot j stays in lane j (k <= 32)
      my_w = w;
      my_i = idx;
    }
    wsum = __fadd_rn(wsum, w);  // in slot order, as the reference's sum over k
  }
  if (lane < k) {
    const float denom = fmaxf(wsum, 1e-9f);
    float w = norm_topk ? __fdiv_rn(my_w, denom) : my_w;
    w = __fmul_rn(w, scaling);
    if (wdtype == FNI8_F16) w = __half2float(__float2half_rn(w));
    else if (wdtype == FNI8_BF16) w = __bfloat162float(__float2bfloat16_rn(w));
    out_i = my_i;
    out_w = w;
  }
}

}  // namespace moe
}  // namespace fni8b
