// The routed-expert layer for a few tokens (T <= 16) in two kernels:
//
//   few_gate_up  logits -> top-k (optional), int8 rows of x, then per active expert e and slot
//                (t, j) routed to it   h[slot] = T(T(act(g)) u),
//                g | u = T((q_t . Wgu[e]) a_t s_gu[e])
//   few_down     int8 rows of h, y[slot] = T((p . Wdn[e]) b s_dn[e]), and
//                out[t] = T(sum_j w[t, j] y[(t, j)]) in slot order
//
// with every rounding where the composed path of moe.cu has it, so the results are the same
// bit for bit (the int32 sums are exact, whatever their order).
//
// What bounds it: the active experts' weights, read once (3 H I bytes each). A token or two
// per expert leave a 128-row tcgen05 tile empty, so the products run on mma.sync m16n8k32:
// 16 weight rows are the M side, up to 8 slots of an expert the N side (16 in two steps).
// At one MMA for 512 weight bytes the SM's share of HBM asks for one in 22 cycles.
//
//  * Every warp is on its own: it takes (expert, 16 weight rows) units, and lane 0 streams
//    them through the warp's private ring of 4 KB stages by TMA (16 rows x 256 bytes,
//    128-byte swizzle). There is no producer warp and no barrier between warps.
//  * In few_gate_up the 16 rows are 8 gate rows and the 8 matching up rows: an accumulator
//    fragment holds gate and up of the same column and slot in one lane, so act(g) * u needs
//    no exchange. In few_down a CTA owns 16 output columns through all experts, keeps their
//    y in shared memory and sums each token's k slots there: no atomics, no third kernel.
//  * Each CTA routes, quantises the rows and lists the experts for itself (T rows of x, the
//    T k rows of h): cheaper than a launch that would hand them over. few_down does its
//    routing and starts its weight loads before it waits for few_gate_up.
//  * Lane (g, q) of a warp reads the 16-byte pieces 2 q + j (j = 0, 1) of row g of a 128-byte
//    column: with the swizzle, eight neighbouring lanes then touch all 32 banks. The order of
//    K inside a piece is the same on both sides of the product, so it needs no shuffle.
#include <type_traits>

#include "fni8_common.cuh"
#include "gemm_internal.h"
#include "moe_route.cuh"

namespace fni8b {
namespace few {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kStage = 4096;  // 16 weight rows x 256 bytes
constexpr int kEntry = 16;    // slots of one expert in one entry (two n8 tiles)
constexpr int kMaxTokens = 16;
constexpr int kMaxSlots = 512;

static __device__ int g_status;
enum : int { kCodeGateUp = 0x801, kCodeDown = 0x802 };

struct Layer {
  const void* x;
  const float* logits;  // null: topi, topw are given
  const int32_t* topi;
  const float* topw;
  const float* sel_bias;
  int T, H, E, I, k;
  int scoring, n_groups, topk_group, norm_topk, wdtype;
  float scaling;
  const float* s_gu;  // [E, 2I]
  const float* s_dn;  // [E, H]
  void* h;            // [T k, I]
  void* out;          // [T, H]
  int stages;
};

// Shared-memory plan of either kernel: `row` bytes of codes per row (odd multiple of 16 modulo
// 128, so that rows fall on different banks).
struct Plan {
  int row, codes, slot_e, slot_w, scale, ent_e, ent_n, list, extra, bars, total;
};
__host__ __device__ inline Plan make_plan(int stages, int rows, int k_len, int slots, int extra_bytes) {
  Plan p;
  int o = kWarps * stages * kStage;
  auto take = [&](int bytes) {
    const int at = o;
    o += (bytes + 15) & ~15;
    return at;
  };
  p.row = (k_len + 127) / 128 * 128 + 16;
  p.codes = take(rows * p.row);
  p.slot_e = take(slots * 4);
  p.slot_w = take(slots * 4);
  p.scale = take(rows * 4);
  p.ent_e = take(slots * 4);
  p.ent_n = take(slots * 4);
  p.list = take(slots * kEntry * 2);
  p.extra = take(extra_bytes);
  p.bars = take(kWarps * 4 * 8);
  p.total = o + 1024;  // the ring is aligned to 1024 bytes
  return p;
}

__device__ __forceinline__ void imma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const T* v = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(v[i]);
}

// One warp: int8 row of src[K] (K a multiple of 16) into dst, zeros up to a multiple of 128;
// returns the scale. The row is read twice, the second time from L1.
template <typename T>
__device__ __forceinline__ float quant_row(const T* __restrict__ src, int K, uint8_t* dst, int lane) {
  const uint4* s = reinterpret_cast<const uint4*>(src);
  const int n = K >> 3;
  float amax = 0.0f;
#pragma unroll 4
  for (int c = lane; c < n; c += 32) {
    float f[8];
    unpack8<T>(s[c], f);
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[i]));
  }
  amax = moe::warp_max(amax);
  const float inv = quant_inv(amax);
  const int padded = (K + 127) / 128 * 16;
#pragma unroll 4
  for (int c = lane; c < padded; c += 32) {
    uint32_t w[2] = {0u, 0u};
    if (c < n) {
      float f[8];
      unpack8<T>(s[c], f);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(quant_one(f[i], inv))) << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(dst + c * 8) = make_uint2(w[0], w[1]);
  }
  return quant_scale(amax);
}

__device__ __forceinline__ void route_one(const Layer& p, int t, int lane, int* slot_e, float* slot_w) {
  const float* lr = p.logits + static_cast<int64_t>(t) * p.E;
  int e = 0;
  float w = 0.0f;
  auto go = [&](auto vpl) {
    moe::route_token<decltype(vpl)::value>(lr, p.E, p.k, p.scoring, p.sel_bias, p.n_groups, p.topk_group, p.norm_topk,
                                           p.scaling, p.wdtype, lane, e, w);
  };
  if (p.E <= 32) go(std::integral_constant<int, 1>{});
  else if (p.E <= 64) go(std::integral_constant<int, 2>{});
  else if (p.E <= 128) go(std::integral_constant<int, 4>{});
  else if (p.E <= 256) go(std::integral_constant<int, 8>{});
  else go(std::integral_constant<int, 16>{});
  if (lane < p.k) {
    slot_e[t * p.k + lane] = e;
    slot_w[t * p.k + lane] = w;
  }
}

// Entries: the slots of each expert, at most kEntry to an entry (an id that appears more often
// has several), slots in order. A slot whose id is outside [0, E) is in none. Returns their
// number; every thread of the CTA takes part. Quadratic in the slots, which are few.
__device__ int list_entries(const int* slot_e, int n, int E, int* ent_e, int* ent_n, uint16_t* list) {
  __shared__ int warp_sum[2 * kWarps];
  __shared__ int16_t ent_of[kMaxSlots];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int base = 0, rank[2], start[2];
  for (int r = 0; r < 2; ++r) {
    const int i = r * kThreads + threadIdx.x;
    const int e = i < n ? slot_e[i] : -1;
    const bool valid = e >= 0 && e < E;
    int before = 0, first = i, all = 0;
    if (valid) {
      for (int j = 0; j < n; ++j) {
        if (slot_e[j] == e) {
          if (j < i) {
            if (before % kEntry == 0) first = j;
            ++before;
          }
          ++all;
        }
      }
      if (before % kEntry == 0) first = i;
    }
    rank[r] = valid ? before : -1;
    start[r] = first;
    const bool opens = valid && before % kEntry == 0;
    const unsigned m = __ballot_sync(0xffffffffu, opens);
    if (lane == 0) warp_sum[r * kWarps + warp] = __popc(m);
    __syncthreads();
    int at = base;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) at += warp_sum[r * kWarps + w];
      base += warp_sum[r * kWarps + w];
    }
    if (opens) {
      const int a = at + __popc(m & ((1u << lane) - 1u));
      ent_of[i] = static_cast<int16_t>(a);
      ent_e[a] = e;
      ent_n[a] = min(kEntry, all - before);
    }
    if (n <= kThreads) break;
  }
  __syncthreads();
  for (int r = 0; r < 2; ++r) {
    const int i = r * kThreads + threadIdx.x;
    if (i < n && rank[r] >= 0) list[ent_of[start[r]] * kEntry + rank[r] % kEntry] = static_cast<uint16_t>(i);
    if (n <= kThreads) break;
  }
  __syncthreads();
  return base;
}

// One stage (16 weight rows x 256 bytes from k0 on, in two 128-byte columns; none behind K)
// times up to 8 NT slots, whose code rows lane (g, q) reads at x[.].
template <int NT>
__device__ __forceinline__ void stage_product(int (&acc)[NT][4], const uint8_t* st, int g, int q,
                                              const uint8_t* const (&x)[NT], int k0, int K) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (k0 + c * 128 >= K) break;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int piece = 2 * q + j;
      const uint8_t* wp = st + c * 2048 + g * 128 + ((piece ^ g) << 4);
      const uint4 lo = *reinterpret_cast<const uint4*>(wp);
      const uint4 hi = *reinterpret_cast<const uint4*>(wp + 1024);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 b = *reinterpret_cast<const uint4*>(x[n] + k0 + c * 128 + piece * 16);
        imma(acc[n], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
        imma(acc[n], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
      }
    }
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) few_gate_up(const __grid_constant__ CUtensorMap tmW, Layer p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int n = p.T * p.k;
  const Plan pl = make_plan(p.stages, p.T, p.H, n, 0);
  uint8_t* codes = smem + pl.codes;
  int* slot_e = reinterpret_cast<int*>(smem + pl.slot_e);
  float* slot_w = reinterpret_cast<float*>(smem + pl.slot_w);
  float* a_s = reinterpret_cast<float*>(smem + pl.scale);
  int* ent_e = reinterpret_cast<int*>(smem + pl.ent_e);
  int* ent_n = reinterpret_cast<int*>(smem + pl.ent_n);
  uint16_t* list = reinterpret_cast<uint16_t*>(smem + pl.list);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + pl.bars) + warp * 4;
  uint8_t* ring = smem + warp * p.stages * kStage;
  if (threadIdx.x == 0) tma_prefetch_desc(&tmW);
  if (lane == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  pdl_wait();
  const int routes = p.logits != nullptr ? p.T : 0;
  if (routes == 0)
    for (int i = threadIdx.x; i < n; i += kThreads) slot_e[i] = p.topi[i];
  for (int job = warp; job < routes + p.T; job += kWarps) {
    if (job < routes) {
      route_one(p, job, lane, slot_e, slot_w);
    } else {
      const int t = job - routes;
      const float s = quant_row<T>(static_cast<const T*>(p.x) + static_cast<int64_t>(t) * p.H, p.H, codes + t * pl.row, lane);
      if (lane == 0) a_s[t] = s;
    }
  }
  __syncthreads();
  const int n_ent = list_entries(slot_e, n, p.E, ent_e, ent_n, list);

  const int U = p.I >> 3, KC = (p.H + 255) >> 8;
  const int first = warp * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);
  const int stride = kWarps * static_cast<int>(gridDim.x);
  const int total = n_ent * U;
  const int units = total > first ? (total - first - 1) / stride + 1 : 0;
  const int steps = units * KC;
  int pu = first, pk = 0, ps = 0;  // the next stage to load (lane 0)
  auto issue = [&]() {
    uint8_t* dst = ring + ps * kStage;
    uint64_t* bar = &full[ps];
    const int e = ent_e[pu / U], c = pu % U * 8;
    mbar_arrive_expect_tx(bar, kStage);
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      tma_load_3d(&tmW, bar, dst + hh * 2048, pk * 256 + hh * 128, c, e);
      tma_load_3d(&tmW, bar, dst + hh * 2048 + 1024, pk * 256 + hh * 128, p.I + c, e);
    }
    if (++pk == KC) {
      pk = 0;
      pu += stride;
    }
    if (++ps == p.stages) ps = 0;
  };
  int issued = min(steps, p.stages), consumed = 0;
  if (lane == 0)
    for (int i = 0; i < issued; ++i) issue();
  pdl_launch_dependents();

  int s = 0;
  uint32_t ph = 0;
  bool ok = true;
  for (int u = first; u < total && ok; u += stride) {
    const int a = u / U, c = u % U;
    const int cnt = ent_n[a];
    const int64_t srow = static_cast<int64_t>(ent_e[a]) * 2 * p.I + c * 8 + g;
    const float sg = __ldg(p.s_gu + srow), su = __ldg(p.s_gu + srow + p.I);
    int acc[2][4] = {};
    auto run = [&](auto nt) {
      constexpr int NT = decltype(nt)::value;
      const uint8_t* x[NT];
      int part[NT][4] = {};
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int at = min(i * 8 + g, cnt - 1);  // columns behind the last slot repeat it and are not stored
        x[i] = codes + list[a * kEntry + at] / p.k * pl.row;
      }
      for (int kc = 0; kc < KC && ok; ++kc) {
        ok = mbar_wait(&full[s], ph, &g_status, kCodeGateUp);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        stage_product<NT>(part, ring + s * kStage, g, q, x, kc * 256, p.H);
        ++consumed;
        __syncwarp();
        if (lane == 0 && issued < steps) issue();
        if (issued < steps) ++issued;
        if (++s == p.stages) {
          s = 0;
          ph ^= 1u;
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] = part[i][r];
    };
    if (cnt <= 8) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 2>{});
    if (!ok) break;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int at = i * 8 + 2 * q + r;
        if (at < cnt) {
          const int slot = list[a * kEntry + at];
          const float as = a_s[slot / p.k];
          const float gate = round_trip<T>(__fmul_rn(__fmul_rn(__int2float_rn(acc[i][r]), as), sg));
          const float up = round_trip<T>(__fmul_rn(__fmul_rn(__int2float_rn(acc[i][2 + r]), as), su));
          static_cast<T*>(p.h)[static_cast<int64_t>(slot) * p.I + c * 8 + g] = act_mul_one<T, ACT>(gate, up);
        }
      }
    }
  }
  // after a wait that gave up: the loads still in flight land before the CTA leaves
  for (; consumed < issued; ++consumed) {
    mbar_wait(&full[s], ph, &g_status, kCodeGateUp);
    if (++s == p.stages) {
      s = 0;
      ph ^= 1u;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) few_down(const __grid_constant__ CUtensorMap tmW, Layer p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int n = p.T * p.k;
  const Plan pl = make_plan(p.stages, n, p.I, n, n * 64);
  uint8_t* codes = smem + pl.codes;
  int* slot_e = reinterpret_cast<int*>(smem + pl.slot_e);
  float* slot_w = reinterpret_cast<float*>(smem + pl.slot_w);
  float* h_s = reinterpret_cast<float*>(smem + pl.scale);
  int* ent_e = reinterpret_cast<int*>(smem + pl.ent_e);
  int* ent_n = reinterpret_cast<int*>(smem + pl.ent_n);
  uint16_t* list = reinterpret_cast<uint16_t*>(smem + pl.list);
  float* y = reinterpret_cast<float*>(smem + pl.extra);  // [slots][16]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + pl.bars) + warp * 4;
  uint8_t* ring = smem + warp * p.stages * kStage;
  if (threadIdx.x == 0) tma_prefetch_desc(&tmW);
  if (lane == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  // The routing's inputs are older than few_gate_up, which released this kernel after its own
  // wait for them: they are read before this kernel waits for few_gate_up.
  if (p.logits != nullptr) {
    for (int t = warp; t < p.T; t += kWarps) route_one(p, t, lane, slot_e, slot_w);
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      slot_e[i] = p.topi[i];
      slot_w[i] = p.topw[i];
    }
  }
  __syncthreads();
  const int n_ent = list_entries(slot_e, n, p.E, ent_e, ent_n, list);

  const int KC = (p.I + 255) >> 8, tiles = p.H >> 4;
  const int my_tiles = (tiles - static_cast<int>(blockIdx.x) - 1) / static_cast<int>(gridDim.x) + 1;
  const int my_ents = n_ent > warp ? (n_ent - warp - 1) / kWarps + 1 : 0;
  const int steps = my_tiles * my_ents * KC;
  int pt = static_cast<int>(blockIdx.x), pa = warp, pk = 0, ps = 0;
  auto issue = [&]() {
    uint8_t* dst = ring + ps * kStage;
    uint64_t* bar = &full[ps];
    mbar_arrive_expect_tx(bar, kStage);
    tma_load_3d(&tmW, bar, dst, pk * 256, pt * 16, ent_e[pa]);
    tma_load_3d(&tmW, bar, dst + 2048, pk * 256 + 128, pt * 16, ent_e[pa]);
    if (++pk == KC) {
      pk = 0;
      if ((pa += kWarps) >= n_ent) {
        pa = warp;
        pt += static_cast<int>(gridDim.x);
      }
    }
    if (++ps == p.stages) ps = 0;
  };
  int issued = min(steps, p.stages), consumed = 0;
  if (lane == 0)
    for (int i = 0; i < issued; ++i) issue();
  pdl_wait();
  for (int i = warp; i < n; i += kWarps) {
    const float sc = quant_row<T>(static_cast<const T*>(p.h) + static_cast<int64_t>(i) * p.I, p.I, codes + i * pl.row, lane);
    if (lane == 0) h_s[i] = sc;
  }
  __syncthreads();
  pdl_launch_dependents();

  int s = 0;
  uint32_t ph = 0;
  bool ok = true;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    for (int a = warp; a < n_ent && ok; a += kWarps) {
      const int cnt = ent_n[a];
      const float* sd = p.s_dn + static_cast<int64_t>(ent_e[a]) * p.H + tile * 16 + g;
      const float s0 = __ldg(sd), s1 = __ldg(sd + 8);
      int acc[2][4] = {};
      auto run = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        const uint8_t* x[NT];
        int part[NT][4] = {};
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] = codes + list[a * kEntry + min(i * 8 + g, cnt - 1)] * pl.row;
        for (int kc = 0; kc < KC; ++kc) {
          ok = mbar_wait(&full[s], ph, &g_status, kCodeDown);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          stage_product<NT>(part, ring + s * kStage, g, q, x, kc * 256, p.I);
          ++consumed;
          __syncwarp();
          if (lane == 0 && issued < steps) issue();
          if (issued < steps) ++issued;
          if (++s == p.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][r] = part[i][r];
      };
      if (cnt <= 8) run(std::integral_constant<int, 1>{});
      else run(std::integral_constant<int, 2>{});
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int at = i * 8 + 2 * q + r;
          if (at < cnt) {
            const int slot = list[a * kEntry + at];
            const float hs = h_s[slot];
            y[slot * 16 + g] = round_trip<T>(__fmul_rn(__fmul_rn(__int2float_rn(acc[i][r]), hs), s0));
            y[slot * 16 + g + 8] = round_trip<T>(__fmul_rn(__fmul_rn(__int2float_rn(acc[i][2 + r]), hs), s1));
          }
        }
      }
    }
    __syncthreads();
    {
      const int t = threadIdx.x >> 4, col = threadIdx.x & 15;
      if (t < p.T) {
        float sum = 0.0f;
        for (int j = 0; j < p.k; ++j) {
          const int slot = t * p.k + j, e = slot_e[slot];
          if (e >= 0 && e < p.E) sum = __fadd_rn(sum, __fmul_rn(slot_w[slot], y[slot * 16 + col]));
        }
        static_cast<T*>(p.out)[static_cast<int64_t>(t) * p.H + tile * 16 + col] = from_f32<T>(sum);
      }
    }
    __syncthreads();  // y is read before the next tile writes it
  }
  for (; consumed < issued; ++consumed) {
    mbar_wait(&full[s], ph, &g_status, kCodeDown);
    if (++s == p.stages) {
      s = 0;
      ph ^= 1u;
    }
  }
}

}  // namespace few
}  // namespace fni8b

namespace fni8h {

using namespace fni8b;

int few_status_read_and_clear(int* code) {
  int v = 0, z = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, few::g_status, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "read few-token watchdog");
  e = cudaMemcpyToSymbol(few::g_status, &z, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "clear few-token watchdog");
  *code = v;
  return FNI8_OK;
}

namespace {

constexpr int kSmemMax = 226 * 1024;  // static shared memory (the entry list's) beside it

// Ring depth of a kernel: three stages a warp, two where the codes leave no room; 0: none fits.
int few_stages(int rows, int64_t k_len, int slots, int extra) {
  for (int st = 3; st >= 2; --st)
    if (few::make_plan(st, rows, (int)k_len, slots, extra).total + 2048 <= kSmemMax) return st;
  return 0;
}

template <typename Kern>
int configure(Kern kern, std::atomic<bool>* done) {
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices) return fail(FNI8_ERR_CUDA, "no current CUDA device");
  if (done[dev]) return FNI8_OK;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax - 2048);
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(few-token layer)");
  done[dev] = true;
  return FNI8_OK;
}

template <typename T, int ACT>
int launch_few(few::Layer& p, const CUtensorMap& gu, const CUtensorMap& dn, cudaStream_t st) {
  static std::atomic<bool> done_a[kMaxDevices] = {}, done_b[kMaxDevices] = {};
  if (int s = configure(few::few_gate_up<T, ACT>, done_a)) return s;
  if (int s = configure(few::few_down<T>, done_b)) return s;
  const int sms = num_sms(current_device());
  const int slots = p.T * p.k;
  p.stages = few_stages(p.T, p.H, slots, 0);
  const int64_t most = (int64_t)slots * (p.I / 8);  // units, if every slot had its own expert
  launch_pdl(few::few_gate_up<T, ACT>, dim3((unsigned)(most < sms ? most : sms)), dim3(few::kThreads),
             few::make_plan(p.stages, p.T, p.H, slots, 0).total, st, gu, p);
  p.stages = few_stages(slots, p.I, slots, slots * 64);
  const int tiles = p.H / 16;
  launch_pdl(few::few_down<T>, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(few::kThreads),
             few::make_plan(p.stages, slots, p.I, slots, slots * 64).total, st, dn, p);
  FNI8_CHECK_LAUNCH("moe few-token layer");
  return FNI8_OK;
}

}  // namespace

bool few_supported(int64_t T, int64_t H, int64_t k, int64_t E, int64_t I) {
  if (T < 1 || T > few::kMaxTokens || k < 1 || k > 32 || T * k > few::kMaxSlots || E < 1 || E > 512) return false;
  if (H % 16 != 0 || I % 16 != 0 || H > (1 << 17) || I > (1 << 17)) return false;
  const int n = (int)(T * k);
  return few_stages((int)T, H, n, 0) > 0 && few_stages(n, I, n, n * 64) > 0;
}

int few_moe(const FewMoe& m, cudaStream_t st) {
  CUtensorMap gu, dn;
  if (int s = encode_tmap_3d_i8(&gu, m.w_gu, (uint64_t)m.H, (uint64_t)(2 * m.I), (uint64_t)m.E, (uint64_t)m.H,
                                (uint64_t)(2 * m.I * m.H), 128, 8))
    return s;
  if (int s = encode_tmap_3d_i8(&dn, m.w_dn, (uint64_t)m.I, (uint64_t)m.H, (uint64_t)m.E, (uint64_t)m.I,
                                (uint64_t)(m.H * m.I), 128, 16))
    return s;
  few::Layer p{m.x, m.logits, m.topi, m.topw, m.sel_bias, (int)m.T, (int)m.H, (int)m.E, (int)m.I, (int)m.k, m.scoring,
               (int)m.n_groups, (int)m.topk_group, m.norm_topk, m.dtype, m.scaling, m.s_gu, m.s_dn, m.h, m.out, 0};
  if (m.dtype == FNI8_F16) {
    if (m.act == FNI8_ACT_SILU) return launch_few<__half, FNI8_ACT_SILU>(p, gu, dn, st);
    return launch_few<__half, FNI8_ACT_GELU_TANH>(p, gu, dn, st);
  }
  if (m.act == FNI8_ACT_SILU) return launch_few<__nv_bfloat16, FNI8_ACT_SILU>(p, gu, dn, st);
  return launch_few<__nv_bfloat16, FNI8_ACT_GELU_TANH>(p, gu, dn, st);
}

}  // namespace fni8h
