// The routed-expert layer for a few tokens (T <= 16, as long as the int8 rows of x and of every
// slot's h fit into shared memory beside the rings) in two kernels, or three:
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
//    them through the warp's private ring of stages by TMA (16 rows x 256 or 512 bytes,
//    128-byte swizzle). There is no producer warp and no barrier between warps.
//  * In few_gate_up the 16 rows are 8 gate rows and the 8 matching up rows: an accumulator
//    fragment holds gate and up of the same column and slot in one lane, so act(g) * u needs
//    no exchange. In few_down a CTA owns 16 output columns through all experts, keeps their
//    int32 sums in shared memory and joins each token's k slots there: no atomics in global
//    memory, no third kernel. With fewer experts than warps it splits their K.
//  * Each CTA, or each cluster of four where there are many values, routes, quantises the
//    rows and lists the experts for itself: cheaper than a launch that would hand them over.
//    Where both kernels fit on an SM few_down does that too, and starts its weight loads, before
//    it waits for few_gate_up. Where they do not, it reads the lists that few_gate_up leaves, and
//    h is quantised once by the row kernel of quant.cu, launched between the two (16 tokens
//    through 8 of 128 experts 56 -> 51 us).
//  * A CTA runs most of its code once, and an instruction line that is not in its SM's caches
//    costs 0.1 us and more; so the preparation is short loops, not unrolled ones (listing the
//    experts of one token: 4.9 us at first sight, 0.8 us the second time), and the weights pass
//    through L2 with an evict-first policy, which leaves the instructions there.
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
// A stage: 16 weight rows x 2 or 4 128-byte columns of K. Four stream faster (512 contiguous
// bytes of a row; 4 tokens through large experts 74 -> 65 us), two let both kernels share an SM.
__host__ __device__ constexpr int stage_bytes(int cols) { return 16 * 128 * cols; }
constexpr int kEntry = 16;    // slots of one expert in one entry (two n8 tiles)
constexpr int kMaxTokens = 16;
constexpr int kMaxSlots = 512;
constexpr int kMaxExperts = 512;

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
  // few_down begins before few_gate_up has ended (both fit on an SM) and lists the experts for
  // itself; else it reads few_gate_up's lists: entries, n, slots' experts and weights.
  int early;
  int32_t* t_count;  // [1]
  int32_t* t_slot_e;
  float* t_slot_w;
  int32_t* t_ent_e;
  int32_t* t_ent_n;
  uint16_t* t_list;  // [T k][kEntry]
  // not early: the int8 rows of h and their scales, quantised by a kernel between the two
  const int8_t* hq;
  const float* hs;
};

// Shared-memory plan of either kernel: `row` bytes of codes per row (odd multiple of 16 modulo
// 128, so that rows fall on different banks).
struct Plan {
  int row, codes, slot_e, slot_w, scale, top, ent_e, ent_n, list, masks, extra, bars, total;
};
__host__ __device__ inline Plan make_plan(int cols, int stages, int rows, int k_len, int slots, int E, int extra_bytes) {
  Plan p;
  int o = kWarps * stages * stage_bytes(cols);
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
  p.top = take(rows * 4);
  p.ent_e = take(slots * 4);
  p.ent_n = take(slots * 4);
  p.list = take(slots * kEntry * 2);
  p.masks = take(E * ((slots + 31) / 32) * 4);
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

// Absmax of eight values, NaNs left out (as fmaxf leaves them out).
template <typename T>
__device__ __forceinline__ float abs_max8(const uint4& u);
template <>
__device__ __forceinline__ float abs_max8<__half>(const uint4& u) {
  const __half2* h = reinterpret_cast<const __half2*>(&u);
  const __half2 m = __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
  return __half2float(__hmax(__low2half(m), __high2half(m)));
}
template <>
__device__ __forceinline__ float abs_max8<__nv_bfloat16>(const uint4& u) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
  return __bfloat162float(__hmax(__low2bfloat16(m), __high2bfloat16(m)));
}

// quant_one of four values, packed: the clamp comes before the rounding (the same, its bounds
// are whole), which is an addition of 1.5 * 2^23: the low byte then holds the code.
__device__ __forceinline__ uint32_t quant4(const float* f, float inv) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = fminf(fmaxf(__fmul_rn(f[i], inv), -127.0f), 127.0f);
    b[i] = __float_as_uint(__fadd_rn(t, 12582912.0f));
  }
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// A value into this CTA's shared memory and the same place in its cluster peers'.
template <typename V>
__device__ __forceinline__ void share(V* at, V v, int peers) {
  static_assert(sizeof(V) == 4 || sizeof(V) == 8, "words");
  if (peers == 1) {
    *at = v;
    return;
  }
  const uint32_t local = smem_u32(at);
  for (int p = 0; p < peers; ++p) {
    const uint32_t to = mapa_shared(local, static_cast<uint32_t>(p));
    if constexpr (sizeof(V) == 8) {
      const uint2 w = *reinterpret_cast<const uint2*>(&v);
      asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(to), "r"(w.x), "r"(w.y) : "memory");
    } else {
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(*reinterpret_cast<const uint32_t*>(&v)) : "memory");
    }
  }
}

// Every thread of the CTA, or of the cluster: what they shared before is seen after.
__device__ __forceinline__ void join(int peers) {
  __syncwarp();
  if (peers > 1) cluster_sync_all();
  else __syncthreads();
}

// int8 rows of src [n, K] (K a multiple of 16) into dst [n][row_bytes], zeros up to a multiple
// of 128, and their scales, here and in the cluster's other CTAs: this CTA's part are rows
// rank, rank + peers, ... The last `threads` threads of the CTA take part, eight values each
// at a time; they meet at named barrier 1. top: [n] scratch.
template <typename T>
__device__ void quant_rows(const T* __restrict__ src, int n, int K, int rank, int peers, int threads, uint8_t* dst,
                           int row_bytes, float* scale, uint32_t* top) {
  const int nc = K >> 3, padded = (K + 127) / 128 * 16;
  const int t0 = static_cast<int>(threadIdx.x) - (kThreads - threads);
  if (t0 < 0) return;
  for (int i = rank + t0 * peers; i < n; i += threads * peers) top[i] = 0u;
  named_bar_sync(1, threads);
  const uint4* rows = reinterpret_cast<const uint4*>(src);
  // Piece c of row i: this thread's pieces in turn, `per` to a row (zeros behind K), with the
  // loads of the next four in flight. (A queue, not an unrolled loop: short code.)
  auto each = [&](int per, auto&& f) {
    const int di = threads / per * peers, dc = threads % per;
    struct Pos {
      int i, c;
    };
    auto advance = [&](Pos& p) {
      p.i += di;
      if ((p.c += dc) >= per) {
        p.c -= per;
        p.i += peers;
      }
    };
    Pos at{rank + t0 / per * peers, t0 % per}, ahead = at;
    auto fetch = [&]() {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (ahead.i < n && ahead.c < nc) u = rows[static_cast<int64_t>(ahead.i) * nc + ahead.c];
      advance(ahead);
      return u;
    };
    uint4 q0 = fetch(), q1 = fetch(), q2 = fetch(), q3 = fetch();
#pragma unroll 1
    for (; at.i < n; advance(at)) {
      const uint4 u = q0;
      q0 = q1;
      q1 = q2;
      q2 = q3;
      q3 = fetch();
      f(at.i, at.c, u);
    }
  };
  each(nc, [&](int i, int, const uint4& u) {
    // (a NaN is no maximum)
    atomicMax(&top[i], __float_as_uint(fmaxf(abs_max8<T>(u), 0.0f)));
  });
  named_bar_sync(1, threads);
  each(padded, [&](int i, int c, const uint4& u) {
    const float amax = __uint_as_float(top[i]), inv = quant_inv(amax);
    float f[8];
    unpack8<T>(u, f);
    uint2 w = make_uint2(quant4(f, inv), quant4(f + 4, inv));
    if (c >= nc) w = make_uint2(0u, 0u);  // (an infinite or NaN factor makes no zero of a zero)
    share(reinterpret_cast<uint2*>(dst + i * row_bytes + c * 8), w, peers);
    if (c == 0) share(scale + i, quant_scale(amax), peers);
  });
}

__device__ __forceinline__ void route_one(const Layer& p, int t, int lane, int* slot_e, float* slot_w, int peers) {
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
    share(slot_e + t * p.k + lane, e, peers);
    share(slot_w + t * p.k + lane, w, peers);
  }
}

// Entries: the slots of each expert, at most kEntry to an entry (an id that appears more often
// has several), by expert, slots in order. A slot whose id is outside [0, E) is in none. masks:
// zeroed, for each expert the slots that name it, a bit each. Returns the number of entries;
// every thread of the CTA takes part.
__device__ int list_entries(const int* slot_e, int n, int E, int* ent_e, int* ent_n, uint16_t* list, uint32_t* masks) {
  __shared__ int total;
  __shared__ int16_t first[kMaxExperts];  // entry of an expert's first slots
  const int lane = threadIdx.x & 31, words = (n + 31) >> 5;
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int e = slot_e[i];
    if (e >= 0 && e < E) atomicOr(&masks[e * words + (i >> 5)], 1u << (i & 31));
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int at = 0;
#pragma unroll 1
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      int c = 0;
      if (e < E) {
#pragma unroll 1
        for (int w = 0; w < words; ++w) c += __popc(masks[e * words + w]);
      }
      const int ne = (c + kEntry - 1) / kEntry;
      int sum = ne;
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const int a = at + sum - ne;
      if (ne > 0) first[e] = static_cast<int16_t>(a);
#pragma unroll 1
      for (int j = 0; j < ne; ++j) {
        ent_e[a + j] = e;
        ent_n[a + j] = min(kEntry, c - j * kEntry);
      }
      at += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) total = at;
  }
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int e = slot_e[i];
    if (e >= 0 && e < E) {
      int before = __popc(masks[e * words + (i >> 5)] & ((1u << (i & 31)) - 1u));
#pragma unroll 1
      for (int w = 0; w < i >> 5; ++w) before += __popc(masks[e * words + w]);
      list[(first[e] + before / kEntry) * kEntry + before % kEntry] = static_cast<uint16_t>(i);
    }
  }
  __syncthreads();
  return total;
}

// One stage (16 weight rows x COLS 128-byte columns from k0 on; none behind K)
// times up to 8 NT slots, whose code rows lane (g, q) reads at x[.].
template <int NT, int COLS>
__device__ __forceinline__ void stage_product(int (&acc)[NT][4], const uint8_t* st, int g, int q,
                                              const uint8_t* const (&x)[NT], int k0, int K) {
#pragma unroll 1
  for (int c = 0; c < COLS; ++c) {
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

template <typename T, int ACT, bool WIDE, int COLS>
__global__ void __launch_bounds__(kThreads) few_gate_up(const __grid_constant__ CUtensorMap tmW, Layer p) {
  constexpr int kStageK = 128 * COLS, kStage = stage_bytes(COLS);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int n = p.T * p.k;
  const Plan pl = make_plan(COLS, p.stages, p.T, p.H, n, p.E, 0);
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
  for (int i = threadIdx.x; i < p.E * ((n + 31) >> 5); i += kThreads) reinterpret_cast<uint32_t*>(smem + pl.masks)[i] = 0u;
  const int rank = static_cast<int>(cluster_ctarank()), peers = static_cast<int>(cluster_nctarank());
  if (peers > 1) cluster_sync_all();  // the peers have started
  pdl_wait();
  // the first warps route this CTA's tokens, the others quantise its rows meanwhile
  int routers = 0;
  if (p.logits != nullptr) {
    routers = min(kWarps / 2, (p.T - rank + peers - 1) / peers);
    if (warp < routers)
      for (int t = warp * peers + rank; t < p.T; t += routers * peers) route_one(p, t, lane, slot_e, slot_w, peers);
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads) slot_e[i] = p.topi[i];
  }
  quant_rows<T>(static_cast<const T*>(p.x), p.T, p.H, rank, peers, 32 * (kWarps - routers), codes, pl.row, a_s,
                reinterpret_cast<uint32_t*>(smem + pl.top));
  join(peers);
  const int n_ent = list_entries(slot_e, n, p.E, ent_e, ent_n, list, reinterpret_cast<uint32_t*>(smem + pl.masks));

  if (!p.early && blockIdx.x == 0) {  // hand the lists over
    if (threadIdx.x == 0) *p.t_count = n_ent;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      p.t_slot_e[i] = slot_e[i];
      p.t_slot_w[i] = p.logits != nullptr ? slot_w[i] : p.topw[i];
      p.t_ent_e[i] = ent_e[i];
      p.t_ent_n[i] = ent_n[i];
    }
    for (int i = threadIdx.x; i < n * kEntry / 2; i += kThreads)
      reinterpret_cast<uint32_t*>(p.t_list)[i] = reinterpret_cast<const uint32_t*>(list)[i];
  }
  pdl_launch_dependents();

  const int U = p.I >> 3, KC = (p.H + kStageK - 1) / kStageK;
  const int first = warp * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);
  const int stride = kWarps * static_cast<int>(gridDim.x);
  const int total = n_ent * U;
  const int units = total > first ? (total - first - 1) / stride + 1 : 0;
  const int steps = units * KC;
  // the next stage to load (lane 0): unit pu = entry pa, column block pc
  int pu = first, pa = first / U, pc = first % U, pk = 0, ps = 0;
  const int stride_a = stride / U, stride_c = stride % U;
  const uint64_t policy = evict_first_policy();
  auto issue = [&]() {
    uint8_t* dst = ring + ps * kStage;
    uint64_t* bar = &full[ps];
    const int e = ent_e[pa], c = pc * 8;
    mbar_arrive_expect_tx(bar, kStage);
    if constexpr (WIDE) {  // 128 bytes x 8 rows x {gate, up} x COLS columns
      tma_load_5d(&tmW, bar, dst, 0, c, 0, pk * COLS, e, policy);
    } else {
#pragma unroll
      for (int hh = 0; hh < COLS; ++hh) {
        tma_load_3d(&tmW, bar, dst + hh * 2048, pk * kStageK + hh * 128, c, e, policy);
        tma_load_3d(&tmW, bar, dst + hh * 2048 + 1024, pk * kStageK + hh * 128, p.I + c, e, policy);
      }
    }
    if (++pk == KC) {
      pk = 0;
      pu += stride;
      pa += stride_a;
      if ((pc += stride_c) >= U) {
        pc -= U;
        ++pa;
      }
    }
    if (++ps == p.stages) ps = 0;
  };
  int issued = min(steps, p.stages), consumed = 0;
  if (lane == 0)
    for (int i = 0; i < issued; ++i) issue();

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
        stage_product<NT, COLS>(part, ring + s * kStage, g, q, x, kc * kStageK, p.H);
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
    // column c * 8 + g of this lane's slots 2 q, 2 q + 1 (and 8 + those)
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      const int at = (j >> 1) * 8 + 2 * q + (j & 1);
      if (at < cnt) {
        const int slot = list[a * kEntry + at];
        const float as = a_s[slot / p.k];
        const float gate = round_trip<T>(__fmul_rn(__fmul_rn(__int2float_rn(acc[0][0]), as), sg));
        const float up = round_trip<T>(__fmul_rn(__fmul_rn(__int2float_rn(acc[0][2]), as), su));
        static_cast<T*>(p.h)[static_cast<int64_t>(slot) * p.I + c * 8 + g] = act_mul_one<T, ACT>(gate, up);
      }
      if (j == 1 && cnt <= 8) break;
      const bool odd = (j & 1) != 0;  // the next slot's accumulators to the front
      acc[0][0] = odd ? acc[1][0] : acc[0][1];
      acc[0][2] = odd ? acc[1][2] : acc[0][3];
      acc[0][1] = acc[1][1];
      acc[0][3] = acc[1][3];
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

template <typename T, bool WIDE, int COLS>
__global__ void __launch_bounds__(kThreads) few_down(const __grid_constant__ CUtensorMap tmW, Layer p) {
  constexpr int kStageK = 128 * COLS, kStage = stage_bytes(COLS);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int n = p.T * p.k;
  const Plan pl = make_plan(COLS, p.stages, n, p.I, n, p.E, n * 64);
  uint8_t* codes = smem + pl.codes;
  int* slot_e = reinterpret_cast<int*>(smem + pl.slot_e);
  float* slot_w = reinterpret_cast<float*>(smem + pl.slot_w);
  float* h_s = reinterpret_cast<float*>(smem + pl.scale);
  int* ent_e = reinterpret_cast<int*>(smem + pl.ent_e);
  int* ent_n = reinterpret_cast<int*>(smem + pl.ent_n);
  uint16_t* list = reinterpret_cast<uint16_t*>(smem + pl.list);
  int* y = reinterpret_cast<int*>(smem + pl.extra);  // [slots][16] sums of the tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + pl.bars) + warp * 4;
  uint8_t* ring = smem + warp * p.stages * kStage;
  if (threadIdx.x == 0) tma_prefetch_desc(&tmW);
  if (lane == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  const int rank = static_cast<int>(cluster_ctarank()), peers = static_cast<int>(cluster_nctarank());
  if (peers > 1) cluster_sync_all();  // the peers have started
  for (int i = threadIdx.x; i < n * 16; i += kThreads) y[i] = 0;
  int n_ent;
  if (p.early) {
    for (int i = threadIdx.x; i < p.E * ((n + 31) >> 5); i += kThreads) reinterpret_cast<uint32_t*>(smem + pl.masks)[i] = 0u;
    // The routing's inputs (and the weights that the ring loads) are older than few_gate_up, which
    // released this kernel after its own wait for them: what wrote them had ended, its stores were in
    // L2. So they are read before this kernel waits for few_gate_up, and from L2.
    if (p.logits != nullptr) {
      for (int t = warp * peers + rank; t < p.T; t += kWarps * peers) route_one(p, t, lane, slot_e, slot_w, peers);
    } else {
      for (int i = threadIdx.x; i < n; i += kThreads) {
        slot_e[i] = __ldcg(p.topi + i);
        slot_w[i] = __ldcg(p.topw + i);
      }
    }
    join(peers);
    n_ent = list_entries(slot_e, n, p.E, ent_e, ent_n, list, reinterpret_cast<uint32_t*>(smem + pl.masks));
  } else {
    pdl_wait();
    n_ent = *p.t_count;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      slot_e[i] = p.t_slot_e[i];
      slot_w[i] = p.t_slot_w[i];
      ent_e[i] = p.t_ent_e[i];
      ent_n[i] = p.t_ent_n[i];
    }
    for (int i = threadIdx.x; i < n * kEntry / 2; i += kThreads)
      reinterpret_cast<uint32_t*>(list)[i] = reinterpret_cast<const uint32_t*>(p.t_list)[i];
    __syncthreads();
  }

  const int KC = (p.I + kStageK - 1) / kStageK, tiles = p.H >> 4;
  const int my_tiles = (tiles - static_cast<int>(blockIdx.x) - 1 + static_cast<int>(gridDim.x)) / static_cast<int>(gridDim.x);
  // Fewer entries than warps: an entry's K range is cut into 2^lg parts, so that no warp idles
  // (one token through 2 experts of 4096 x 4096: 40 -> 32 us).
  int lg = 0;
  while (n_ent << (lg + 1) <= kWarps && 2 << lg <= KC) ++lg;
  const int items = n_ent << lg;
  auto k_begin = [&](int part) { return (part * KC) >> lg; };
  auto part_of = [&](int item) { return item & ((1 << lg) - 1); };
  // the next stage to load (lane 0): item pi of tile pt, step pk of [.., pe)
  int pt = static_cast<int>(blockIdx.x), pi = warp, ps = 0;
  int pk = k_begin(part_of(warp)), pe = k_begin(part_of(warp) + 1);
  if (items <= warp) pt = tiles;
  const uint64_t policy = evict_first_policy();
  auto issue = [&]() {
    uint8_t* dst = ring + ps * kStage;
    uint64_t* bar = &full[ps];
    mbar_arrive_expect_tx(bar, kStage);
    if constexpr (WIDE) {  // 128 bytes x 16 rows x COLS columns
      tma_load_4d(&tmW, bar, dst, 0, pt * 16, pk * COLS, ent_e[pi >> lg], policy);
    } else {
#pragma unroll
      for (int hh = 0; hh < COLS; ++hh)
        tma_load_3d(&tmW, bar, dst + hh * 2048, pk * kStageK + hh * 128, pt * 16, ent_e[pi >> lg], policy);
    }
    if (++pk == pe) {
      if ((pi += kWarps) >= items) {
        pi = warp;
        pt += static_cast<int>(gridDim.x);
      }
      pk = k_begin(part_of(pi));
      pe = k_begin(part_of(pi) + 1);
    }
    if (++ps == p.stages) ps = 0;
  };
  int steps = 0;
#pragma unroll 1
  for (int i = warp; i < items; i += kWarps) steps += k_begin(part_of(i) + 1) - k_begin(part_of(i));
  steps *= my_tiles;
  int issued = min(steps, p.stages), consumed = 0;
  if (lane == 0)
    for (int i = 0; i < issued; ++i) issue();
  if (p.early) {
    pdl_wait();
    quant_rows<T>(static_cast<const T*>(p.h), n, p.I, rank, peers, kThreads, codes, pl.row, h_s,
                  reinterpret_cast<uint32_t*>(smem + pl.top));
  } else {
    const int per = p.I >> 4, di = kThreads / per, dc = kThreads % per;
    int c = threadIdx.x % per;
#pragma unroll 1
    for (int i = threadIdx.x / per; i < n; i += di) {
      cp_async_16(codes + i * pl.row + c * 16, p.hq + static_cast<int64_t>(i) * p.I + c * 16);
      if ((c += dc) >= per) {
        c -= per;
        ++i;
      }
    }
    cp_async_commit();
    for (int i = threadIdx.x; i < n; i += kThreads) h_s[i] = p.hs[i];
    cp_async_wait_group<0>();
  }
  join(peers);
  pdl_launch_dependents();

  int s = 0;
  uint32_t ph = 0;
  bool ok = true;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    // Thread (t, col) has the tile's column col of token t; what its first eight slots need is
    // loaded while the products run (zeros for a slot without an expert).
    const int t = threadIdx.x >> 4, col = threadIdx.x & 15, first = t * p.k;
    auto scales_of = [&](int j, float& b, float& s_dn, float& w) {
      const int e = t < p.T && j < p.k ? slot_e[first + j] : -1;
      const bool live = e >= 0 && e < p.E;
      b = live ? h_s[first + j] : 0.0f;
      s_dn = live ? __ldg(p.s_dn + static_cast<int64_t>(e) * p.H + tile * 16 + col) : 0.0f;
      w = live ? slot_w[first + j] : 0.0f;
    };
    float b[8], s_dn[8], w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) scales_of(j, b[j], s_dn[j], w[j]);
#pragma unroll 1
    for (int item = warp; item < items && ok; item += kWarps) {
      const int a = item >> lg, k_end = k_begin(part_of(item) + 1);
      const int cnt = ent_n[a];
      int acc[2][4] = {};
      auto run = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        const uint8_t* x[NT];
        int sum[NT][4] = {};
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] = codes + list[a * kEntry + min(i * 8 + g, cnt - 1)] * pl.row;
#pragma unroll 1
        for (int kc = k_begin(part_of(item)); kc < k_end; ++kc) {
          ok = mbar_wait(&full[s], ph, &g_status, kCodeDown);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          stage_product<NT, COLS>(sum, ring + s * kStage, g, q, x, kc * kStageK, p.I);
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
          for (int r = 0; r < 4; ++r) acc[i][r] = sum[i][r];
      };
      if (cnt <= 8) run(std::integral_constant<int, 1>{});
      else run(std::integral_constant<int, 2>{});
      // the parts' sums meet as integers: their order does not matter
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int at = i * 8 + 2 * q + r;
          if (at < cnt) {
            int* ys = y + list[a * kEntry + at] * 16 + g;
            atomicAdd(ys, acc[i][r]);
            atomicAdd(ys + 8, acc[i][2 + r]);
          }
        }
      }
    }
    __syncthreads();
    if (t < p.T) {
      // y = T(float(sum) b s_dn) of each slot, the token's weighted sum, zeros for the next tile
      int* ys = y + first * 16 + col;
      int part[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) part[j] = j < p.k ? ys[j * 16] : 0;
      float sum = 0.0f;
      auto add = [&](int v, float b_j, float s_j, float w_j) {
        sum = __fadd_rn(sum, __fmul_rn(w_j, round_trip<T>(__fmul_rn(__fmul_rn(__int2float_rn(v), b_j), s_j))));
      };
#pragma unroll
      for (int j = 0; j < 8; ++j) add(part[j], b[j], s_dn[j], w[j]);
#pragma unroll 1
      for (int j = 8; j < p.k; ++j) {
        float b_j, s_j, w_j;
        scales_of(j, b_j, s_j, w_j);
        add(ys[j * 16], b_j, s_j, w_j);
      }
#pragma unroll 1
      for (int j = 0; j < p.k; ++j) ys[j * 16] = 0;
      static_cast<T*>(p.out)[static_cast<int64_t>(t) * p.H + tile * 16 + col] = from_f32<T>(sum);
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

// Ring of a kernel: three stages a warp, two where the codes leave no room; 0: none fits.
int few_stages(int cols, int rows, int64_t k_len, int slots, int E, int extra) {
  for (int st = 3; st >= 2; --st)
    if (few::make_plan(cols, st, rows, (int)k_len, slots, E, extra).total + 2048 <= kSmemMax) return st;
  return 0;
}

// CTAs per cluster that share the preparation. Four, where the rows have 16384 values in all: 4
// tokens of 8 large experts 59 us when this was chosen (56 now), 63 in pairs, 64 in clusters of eight,
// which leave 28 of the 148 SMs idle; fewer values are sooner quantised than shared (one token of
// 2048: 20.9 us, in clusters 21.1).
int few_cluster(int64_t rows, int64_t k_len) { return rows * k_len >= 16384 ? 4 : 1; }

// Grid of `want` CTAs at most, in clusters of cs that are resident at once.
int few_grid(int64_t want, int smem, int cs) {
  const int sms = num_sms(current_device());
  int64_t n = want < sms ? want : sms;
  if (cs > 1) {
    int most = max_active_clusters(few::kThreads, smem, cs);
    if (most < 1) most = sms / cs;
    n = (n + cs - 1) / cs;
    n = (n < most ? n : most) * cs;
  }
  return (int)n;
}

template <typename... KArgs, typename... Args>
void launch_cluster(void (*kern)(KArgs...), int grid, int cs, int smem, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(few::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cs;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
  if (e != cudaSuccess && t_launch_error == cudaSuccess) t_launch_error = e;
}

template <typename Kern>
int configure(Kern kern, std::atomic<bool>* done) {
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices) return fail(FNI8_ERR_CUDA, "no current CUDA device");
  if (done[dev]) return FNI8_OK;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax - 2048);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(few-token layer)");
  done[dev] = true;
  return FNI8_OK;
}

template <typename T, int ACT, bool WIDE, int COLS>
int launch_gate_up(const few::Layer& p, const CUtensorMap& map, int smem, cudaStream_t st) {
  static std::atomic<bool> done[kMaxDevices] = {};
  if (int s = configure(few::few_gate_up<T, ACT, WIDE, COLS>, done)) return s;
  const int cs = few_cluster(p.T, p.H);
  // units at most: every slot its own expert
  const int grid = few_grid((int64_t)p.T * p.k * (p.I / 8), smem, cs);
  launch_cluster(few::few_gate_up<T, ACT, WIDE, COLS>, grid, cs, smem, st, map, p);
  return FNI8_OK;
}

template <typename T, bool WIDE, int COLS>
int launch_down(const few::Layer& p, const CUtensorMap& map, int smem, cudaStream_t st) {
  static std::atomic<bool> done[kMaxDevices] = {};
  if (int s = configure(few::few_down<T, WIDE, COLS>, done)) return s;
  const int cs = p.early ? few_cluster(p.T * p.k, p.I) : 1;
  launch_cluster(few::few_down<T, WIDE, COLS>, few_grid(p.H / 16, smem, cs), cs, smem, st, map, p);
  return FNI8_OK;
}

// Columns per stage, ring and shared memory of both kernels.
struct FewPlan {
  int cols_g, cols_d, stages_g, stages_d, smem_g, smem_d, early;
};
bool few_plan(int64_t T, int64_t H, int64_t k, int64_t E, int64_t I, FewPlan* p) {
  const int n = (int)(T * k);
  auto gate_up = [&](int cols) {
    p->cols_g = cols;
    p->stages_g = few_stages(cols, (int)T, H, n, (int)E, 0);
    p->smem_g = few::make_plan(cols, p->stages_g, (int)T, (int)H, n, (int)E, 0).total;
    return p->stages_g > 0;
  };
  auto down = [&](int cols) {
    p->cols_d = cols;
    p->stages_d = few_stages(cols, n, I, n, (int)E, n * 64);
    p->smem_d = few::make_plan(cols, p->stages_d, n, (int)I, n, (int)E, n * 64).total;
    return p->stages_d > 0;
  };
  // Both kernels on an SM where they fit and the weights are few: one token through 8 of 128
  // experts (38 MB) 21.7 us, 24 with wide stages; through 2 of 4096 x 4096 (101 MB) 32 and 34, two
  // tokens (201 MB) 57 and 48.
  p->early = 0;
  if ((int64_t)n * 3 * H * I <= (128 << 20) && gate_up(2) && down(2) && p->smem_g + p->smem_d + 2 * 2048 <= kSmemMax) {
    p->early = 1;
    return true;
  }
  return (gate_up(4) || gate_up(2)) && (down(4) || down(2));
}

template <typename T, int ACT>
int gate_up_any(const few::Layer& p, const FewPlan& f, const CUtensorMap& map, cudaStream_t st) {
  if (p.H % 128 == 0)
    return f.cols_g == 4 ? launch_gate_up<T, ACT, true, 4>(p, map, f.smem_g, st)
                         : launch_gate_up<T, ACT, true, 2>(p, map, f.smem_g, st);
  return f.cols_g == 4 ? launch_gate_up<T, ACT, false, 4>(p, map, f.smem_g, st)
                       : launch_gate_up<T, ACT, false, 2>(p, map, f.smem_g, st);
}

template <typename T>
int launch_few(const few::Layer& layer, const FewPlan& f, int act, const CUtensorMap& gu, const CUtensorMap& dn,
               cudaStream_t st) {
  few::Layer p = layer, d = layer;
  p.stages = f.stages_g;
  d.stages = f.stages_d;
  p.early = d.early = f.early;
  int s = act == FNI8_ACT_SILU ? gate_up_any<T, FNI8_ACT_SILU>(p, f, gu, st)
                               : gate_up_any<T, FNI8_ACT_GELU_TANH>(p, f, gu, st);
  if (s) return s;
  if (!f.early) {
    const int dtype = std::is_same<T, __half>::value ? FNI8_F16 : FNI8_BF16;
    s = fni8_quantize_rows_i8(p.h, dtype, (int64_t)p.T * p.k, p.I, const_cast<int8_t*>(d.hq), const_cast<float*>(d.hs), st);
    if (s) return s;
  }
  if (d.I % 128 == 0)
    s = f.cols_d == 4 ? launch_down<T, true, 4>(d, dn, f.smem_d, st) : launch_down<T, true, 2>(d, dn, f.smem_d, st);
  else
    s = f.cols_d == 4 ? launch_down<T, false, 4>(d, dn, f.smem_d, st) : launch_down<T, false, 2>(d, dn, f.smem_d, st);
  if (s) return s;
  FNI8_CHECK_LAUNCH("moe few-token layer");
  return FNI8_OK;
}

}  // namespace

bool few_supported(int64_t T, int64_t H, int64_t k, int64_t E, int64_t I) {
  if (T < 1 || T > few::kMaxTokens || k < 1 || k > 32 || T * k > few::kMaxSlots || E < 1 || E > few::kMaxExperts) return false;
  if (H % 16 != 0 || I % 16 != 0 || H > (1 << 17) || I > (1 << 17)) return false;
  FewPlan p;
  return few_plan(T, H, k, E, I, &p);
}

int few_moe(const FewMoe& m, cudaStream_t st) {
  FewPlan f;
  if (!few_plan(m.T, m.H, m.k, m.E, m.I, &f)) return fail(FNI8_ERR_UNSUPPORTED, "few-token layer: sizes");
  // One load per stage where K is whole 128-byte columns (they become a dimension of the map);
  // small loads are issued at one in some 35 cycles, four to a stage took the first ring 1.7 us.
  CUtensorMap gu, dn;
  const uint64_t H = (uint64_t)m.H, I = (uint64_t)m.I, E = (uint64_t)m.E;
  if (m.H % 128 == 0) {
    const uint64_t dims[5] = {128, I, 2, H / 128, E}, strides[4] = {H, I * H, 128, 2 * I * H};
    const uint32_t box[5] = {128, 8, 2, (uint32_t)f.cols_g, 1};
    if (int s = encode_tmap_i8(&gu, m.w_gu, 5, dims, strides, box)) return s;
  } else if (int s = encode_tmap_3d_i8(&gu, m.w_gu, H, 2 * I, E, H, 2 * I * H, 128, 8)) {
    return s;
  }
  if (m.I % 128 == 0) {
    const uint64_t dims[4] = {128, H, I / 128, E}, strides[3] = {I, 128, H * I};
    const uint32_t box[4] = {128, 16, (uint32_t)f.cols_d, 1};
    if (int s = encode_tmap_i8(&dn, m.w_dn, 4, dims, strides, box)) return s;
  } else if (int s = encode_tmap_3d_i8(&dn, m.w_dn, I, H, E, I, H * I, 128, 16)) {
    return s;
  }
  few::Layer p{m.x, m.logits, m.topi, m.topw, m.sel_bias, (int)m.T, (int)m.H, (int)m.E, (int)m.I, (int)m.k, m.scoring,
               (int)m.n_groups, (int)m.topk_group, m.norm_topk, m.dtype, m.scaling, m.s_gu, m.s_dn, m.h, m.out, 0, 0, m.t_count, m.t_slot_e, m.t_slot_w, m.t_ent_e,
               m.t_ent_n, m.t_list, m.hq, m.hs};
  return m.dtype == FNI8_F16 ? launch_few<__half>(p, f, m.act, gu, dn, st)
                              : launch_few<__nv_bfloat16>(p, f, m.act, gu, dn, st);
}

}  // namespace fni8h
