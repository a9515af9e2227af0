// GEMM of 4-bit floating point operands on the block-scaled tensor core (sm_100a).
//
//   out[m, n] = dtype((sum_k a[m,k] sa[m,k/g] w[n,k] sw[n,k/g]) * ra[m] * rw[n] (+ bias[n]))
//
// a, w: e2m1 codes, sa, sw: their block scales (fp4_common.cuh), ra, rw: the row scales of
// nvfp4. tcgen05.mma kind::mxf4 / kind::mxf4nvf4 applies the block scales, so the fp32
// accumulator holds the finished sum and the epilogue only multiplies by the row scales.
//
// Structure of the int8 tile kernel (gemm_tile.cu): one persistent CTA per SM, a TMA warp,
// an MMA warp, eight epilogue warps. A stage is 128 bytes of K (256 values) of 128 rows of a
// and BN rows of w with the 128-byte swizzle, plus their scale tiles as they lie in memory
// (512 bytes each, no swizzle); tcgen05.cp brings those into tensor memory.
//
// What bounds it (8192 rows): a stage of a pair takes some 835 cycles where its MMAs take 512, and
// a tile 2350 more (K = 4096: 350 us at the full clock, 370 to 430 in long runs under the power cap;
// tensor pipe busy half the time, L2 a third; K = 12288: 160).
// Neither the bytes of the feed (256 x 384 tiles, a sixth fewer, took 347 and 169 us) nor the
// power (operands of zeros 347 and 150) holds it there, the scale copies do in part. Measured on
// B200: one thread issues one in 45 cycles, whatever its shape, so the 12 of an nvfp4 stage of 256
// columns take 540; issued by the MMAs' thread they overlap neither the MMAs before its last
// commit nor those behind them (8192 x 4096 x 16384: mxfp4 256 us, nvfp4 358, without the copies
// 183 and 189). From other threads they leave the MMAs alone, but a stage's copies then complete
// some 1400 cycles after their issue. So two more warps issue them (211 and 274 us with one, 209
// and 232 with two, 219 and 236 with three), and the scales run ahead: their ring is kLead stages
// deeper than the operands', their tiles are loaded before the operands of earlier stages, and
// SETS sets of tensor-memory columns take turns.
#include "fp4_common.cuh"
#include "gemm_internal.h"

namespace fni8b {
namespace fp4 {

constexpr int BM = 128;
constexpr int BK = 128;  // bytes of K per stage: 256 values
constexpr int kEpiWarps = 8;
constexpr int kEpiThreads = 32 * kEpiWarps;
constexpr int kScaleWarps = 2;
constexpr int kTileThreads = 64 + kEpiThreads + 32 * kScaleWarps;
constexpr int kLead = 2;  // stages that the scales run ahead of their operands
constexpr int kBand = 16;  // m-tiles per band of the tile order: a wave reuses its rows and columns from L2

static __device__ int g_status;

enum : int { kCodeProducer = 0x701, kCodeMma = 0x702, kCodeEpilogue = 0x703, kCodeDrain = 0x704, kCodeScales = 0x705 };

struct Epi {
  const float* a_rs;  // [M] or null (mxfp4)
  const float* w_rs;  // [N] or null
  const void* bias;   // [N] or null
  void* out;          // [M, N]
  int bf16;
  int tma_store;  // rows 16-byte aligned: slabs leave by TMA
};

template <int FMT, int BN, bool PAIR>
struct Cfg {
  static constexpr int BMT = PAIR ? 2 * BM : BM;  // rows of a tile
  static constexpr int BNL = PAIR ? BN / 2 : BN;  // weight rows this CTA loads per stage
  static constexpr int TILES = Fmt<FMT>::kStageTiles;
  static constexpr int A_BYTES = BM * BK;
  static constexpr int B_BYTES = BNL * BK;
  static constexpr int SFA_BYTES = TILES * 512;
  static constexpr int SFB_BYTES = BN / 128 * TILES * 512;  // of all BN columns, in both CTAs of a pair
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int SF = SFA_BYTES + SFB_BYTES;
  static constexpr int STG_BUF = 32 * 32 * 2;  // one output slab of an epilogue warp
  static constexpr int FIXED = 1024 + 1024 + kEpiWarps * STG_BUF + 2 * BN * 4 + kLead * SF;
  static constexpr int STAGES = (227 * 1024 - FIXED) / (STAGE + SF);
  static constexpr int SLOTS = STAGES + kLead;  // scale ring
  static constexpr int SF_OFF = STAGES * STAGE;
  static constexpr int BAR_OFF = SF_OFF + SLOTS * SF;
  static constexpr int STG_OFF = BAR_OFF + 1024;  // 1024-aligned
  static constexpr int SMEM = FIXED + STAGES * (STAGE + SF);
  // accumulators in columns [0, 256), then the sets of scale columns
  static constexpr int NACC = 256 / BN;
  static constexpr int SFA_COLS = TILES * 4;
  static constexpr int SF_COLS = SFA_COLS + BN / 128 * TILES * 4;
  static constexpr int SETS = 4;
  static_assert(256 + SETS * SF_COLS <= 512 && SETS < STAGES, "tensor memory");
  static_assert(STAGES >= 3 && STAGES <= 8, "ring");
  static_assert(STG_OFF % 1024 == 0, "the store's swizzle follows address bits");
};

template <int BMT>
__device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int& m_blk, int& n_blk) {
  const int band_tiles = kBand * n_tiles;
  const int b = t / band_tiles;
  const int first = b * kBand;
  const int gm = min(kBand, m_tiles - first);
  const int local = t - b * band_tiles;
  m_blk = first + local % gm;
  n_blk = local / gm;
}

// 32 accumulators of one row, scaled, biased and rounded: four 16-byte pieces.
template <typename T, int FMT>
__device__ __forceinline__ void finish_chunk(const uint32_t (&r)[32], float ra, const float* rw, const float* bs,
                                             bool has_bias, uint4 (&o)[4]) {
#pragma unroll
  for (int j8 = 0; j8 < 4; ++j8) {
    T* oo = reinterpret_cast<T*>(&o[j8]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = j8 * 8 + j;
      float v = __uint_as_float(r[c]);
      if constexpr (FMT == FNI8_NVFP4) v = __fmul_rn(__fmul_rn(v, ra), rw[c]);
      if (has_bias) v = __fadd_rn(v, bs[c]);
      oo[j] = from_f32<T>(v);
    }
  }
}

// A warp's 32 x 32 slab (lane = row) through its staging buffer: one TMA store, or, where
// the rows are not 16-byte aligned, 64 contiguous bytes of a row per store instruction.
__device__ __forceinline__ void store_slab(uint8_t* buf, const uint4 (&o)[4], int lane, const CUtensorMap* map,
                                           bool tma, uint16_t* out, int n0, int N, int64_t row0, int rows) {
  if (tma && lane == 0) bulk_wait_group_read<0>();
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = o[j];
  if (tma) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(map, buf, n0, static_cast<int>(row0));
      bulk_commit_group();
    }
  } else {
    __syncwarp();
    const int n = n0 + lane;
    for (int r = 0; r < rows; ++r) {
      const uint16_t v =
          *reinterpret_cast<const uint16_t*>(buf + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
      if (n < N) out[(row0 + r) * N + n] = v;
    }
    __syncwarp();
  }
}

template <int FMT, int BN, bool PAIR>
__global__ void __launch_bounds__(kTileThreads, 1)
    fp4_tile_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                    const __grid_constant__ CUtensorMap tmOut, Epi epi, int M, int N, int Kp, int ktiles) {
  using C = Cfg<FMT, BN, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* empty = full + C::STAGES;
  uint64_t* sfull = empty + C::STAGES;
  uint64_t* sready = sfull + C::SLOTS;
  uint64_t* tfull = sready + C::SETS;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1 + kScaleWarps);
  uint8_t* stg = smem + C::STG_OFF;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t half = PAIR ? (cluster_ctarank() & 1u) : 0u;
  const int t0 = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int tstep = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < C::SLOTS; ++s) mbar_init(&sfull[s], 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], PAIR ? 2 * kEpiWarps : kEpiWarps);
    }
    for (int s = 0; s < C::SETS; ++s) mbar_init(&sready[s], kScaleWarps);
    mbar_init(drain, 1);
    for (int s = 0; s < kScaleWarps; ++s) mbar_init(drain + 1 + s, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
    tc_fence_before();
  }
  // Of every thread, before any load: the kernel in front writes the rows, and may have written the weights
  // or their scales. (What the CTA does ahead of it is the set-up above.)
  pdl_wait();
  const int n_tiles = (N + BN - 1) / BN;
  const int m_tiles = (M + C::BMT - 1) / C::BMT;
  const int total = m_tiles * n_tiles;
  const int kb = (Kp + 255) / 256;
  if constexpr (PAIR) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      tma_prefetch_desc(&tmSA);
      tma_prefetch_desc(&tmSB);
      constexpr int kCtas = PAIR ? 2 : 1;  // a pair's loads complete on the even CTA's barriers
      auto load = [&](const CUtensorMap* map, uint64_t* bar, int off, int cx, int cy) {
        if constexpr (PAIR) tma_load_2d_pair(map, mapa_shared(smem_u32(bar), 0), smem + off, cx, cy);
        else tma_load_2d(map, bar, smem + off, cx, cy);
      };
      // this CTA's 128 rows of an m-tile
      auto row_tile = [&](int m_blk) { return PAIR ? 2 * m_blk + static_cast<int>(half) : m_blk; };
      // (tile, stage of it) that a load is for; two of them walk the same sequence
      struct Pos {
        int t, k, mb, nb;
      };
      auto start = [&](Pos& p) {
        p = Pos{t0, 0, 0, 0};
        if (p.t < total) tile_at<C::BMT>(p.t, m_tiles, n_tiles, p.mb, p.nb);
      };
      auto advance = [&](Pos& p) {
        if (++p.k == kb) {
          p.k = 0;
          p.t += tstep;
          if (p.t < total) tile_at<C::BMT>(p.t, m_tiles, n_tiles, p.mb, p.nb);
        }
      };
      auto load_a = [&](int s, const Pos& p) {
        load(&tmA, &full[s], s * C::STAGE, p.k * BK, row_tile(p.mb) * BM);
      };
      auto load_b = [&](int s, const Pos& p) {
        if (half == 0) mbar_arrive_expect_tx(&full[s], kCtas * C::STAGE);
        load(&tmB, &full[s], s * C::STAGE + C::A_BYTES, p.k * BK, p.nb * BN + static_cast<int>(half) * C::BNL);
      };
      auto load_sa = [&](int u, const Pos& p) {
        load(&tmSA, &sfull[u], C::SF_OFF + u * C::SF, 0, (row_tile(p.mb) * ktiles + p.k * C::TILES) * 4);
      };
      auto load_sb = [&](int u, const Pos& p) {
        if (half == 0) mbar_arrive_expect_tx(&sfull[u], kCtas * C::SF);
#pragma unroll
        for (int i = 0; i < BN / 128; ++i)
          load(&tmSB, &sfull[u], C::SF_OFF + u * C::SF + C::SFA_BYTES + i * C::TILES * 512, 0,
               ((p.nb * (BN / 128) + i) * ktiles + p.k * C::TILES) * 4);
      };
      Pos x, y;  // next operand stage, next scale slot (kLead ahead)
      start(x);
      start(y);
      int slot = 0, stage = 0, issued = 0;
      uint32_t ph = 0, armed = 0, slot_ph = 0, slot_armed = 0;
      auto next_slot = [&]() {
        slot_armed = (slot_armed & ~(1u << slot)) | (slot_ph << slot);
        advance(y);
        if (++slot == C::SLOTS) {
          slot = 0;
          slot_ph ^= 1u;
        }
      };
      // The first ring: the weights' part of all its stages, then the rows' part. Stage by stage, as below,
      // the loop behind runs slower (8192 x 4096 x 16384 mxfp4 242 -> 265 us, nvfp4 260 -> 283; 8192 x 24576
      // x 4096 nvfp4 436 -> 454; short products gain, 300 x 6144 x 4096 12.1 -> 10.7).
      Pos first_x[C::STAGES], first_y[C::SLOTS];
      int nx = 0, ny = 0;
      for (; ny < C::SLOTS && y.t < total; ++ny) {
        load_sb(slot, y);
        first_y[ny] = y;
        next_slot();
      }
      for (; nx < C::STAGES && x.t < total; ++nx, advance(x)) {
        load_b(nx, x);
        first_x[nx] = x;
      }
      for (int i = 0; i < ny; ++i) load_sa(i, first_y[i]);
      for (int i = 0; i < nx; ++i) load_a(i, first_x[i]);
      issued = nx;
      stage = nx % C::STAGES;
      ph = nx == C::STAGES ? 1u : 0u;
      for (; x.t < total; advance(x)) {
        // frees the operands of the stage, and the scale slot behind it
        if (!mbar_wait(&empty[stage], ph ^ 1u, &g_status, kCodeProducer)) break;
        if (y.t < total) {
          load_sb(slot, y);
          load_sa(slot, y);
          next_slot();
        }
        load_b(stage, x);
        load_a(stage, x);
        armed = (armed & ~(1u << stage)) | (ph << stage);
        ++issued;
        if (++stage == C::STAGES) {
          stage = 0;
          ph ^= 1u;
        }
      }
      pdl_launch_dependents();
      // Every load lands before the CTA may exit (normally all have: the MMAs consumed them).
      // The odd CTA of a pair sees its loads land through the release of their stages.
      uint64_t* done = half == 0 ? full : empty;
      const int pending = issued < C::STAGES ? issued : C::STAGES;
      for (int i = 0; i < pending; ++i) {
        const int s = (stage - 1 - i + 2 * C::STAGES) % C::STAGES;
        mbar_wait(&done[s], (armed >> s) & 1u, &g_status, kCodeDrain);
      }
      const int used = slot_ph != 0u || slot_armed != 0u ? C::SLOTS : slot;
      if (half == 0)
        for (int u = 0; u < used; ++u) mbar_wait(&sfull[u], (slot_armed >> u) & 1u, &g_status, kCodeDrain);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && half == 0) {
      int stage = 0, acc = 0, set = 0;
      uint32_t ph = 0, aph = 0, sph = 0;
      bool ok = true;
      for (int t = t0; t < total && ok; t += tstep) {
        if (!mbar_wait(&tempty[acc], aph ^ 1u, &g_status, kCodeMma)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int k = 0; k < kb; ++k) {
          if (!mbar_wait(&sready[set], sph, &g_status, kCodeMma) || !mbar_wait(&full[stage], ph, &g_status, kCodeMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint8_t* sa = smem + stage * C::STAGE;
          const int steps = min(4, (Kp - k * 256 + 63) / 64);
          const uint32_t sc = tmem_base + 256u + static_cast<uint32_t>(set * C::SF_COLS);
          stage_mmas<FMT, PAIR, C::BMT, BN>(d, sa, sa + C::A_BYTES, sc, sc + C::SFA_COLS, steps, k == 0);
          if constexpr (PAIR) umma_commit_pair_to(&empty[stage], 3);
          else umma_commit(&empty[stage]);
          if (++stage == C::STAGES) {
            stage = 0;
            ph ^= 1u;
          }
          if (++set == C::SETS) {
            set = 0;
            sph ^= 1u;
          }
        }
        if (!ok) break;
        if constexpr (PAIR) umma_commit_pair_to(&tfull[acc], 3);
        else umma_commit(&tfull[acc]);
        if (++acc == C::NACC) {
          acc = 0;
          aph ^= 1u;
        }
      }
      if constexpr (PAIR) umma_commit_pair(drain);
      else umma_commit(drain);
      mbar_wait(drain, 0, &g_status, kCodeDrain);
    }
    __syncwarp();
  } else if (warp >= 2 + kEpiWarps) {
    // ------------------------------------------------------------ scales into tensor memory
    if (lane == 0 && half == 0) {
      const int part = warp - 2 - kEpiWarps;
      int slot = 0, set = 0, freed = 0;  // freed: the operand stage whose release frees the set
      uint32_t ph = 0, fph = 0;
      const int per = t0 < total ? (total - t0 - 1) / tstep + 1 : 0;
      const int64_t stages = static_cast<int64_t>(per) * kb;
      for (int64_t j = 0; j < stages; ++j) {
        if (!mbar_wait(&sfull[slot], ph, &g_status, kCodeScales)) break;
        if (j >= C::SETS) {
          if (!mbar_wait(&empty[freed], fph, &g_status, kCodeScales)) break;
          if (++freed == C::STAGES) {
            freed = 0;
            fph ^= 1u;
          }
        }
        tc_fence_after();
        const uint8_t* sf = smem + C::SF_OFF + slot * C::SF;
        const uint32_t sc = tmem_base + 256u + static_cast<uint32_t>(set * C::SF_COLS);
        if (part == 0) stage_scales<FMT, PAIR, BN, 0, 2>(sf, sf + C::SFA_BYTES, sc, sc + C::SFA_COLS);
        else stage_scales<FMT, PAIR, BN, 1, 2>(sf, sf + C::SFA_BYTES, sc, sc + C::SFA_COLS);
        if constexpr (PAIR) umma_commit_pair(&sready[set]);
        else umma_commit(&sready[set]);
        if (++set == C::SETS) set = 0;
        if (++slot == C::SLOTS) {
          slot = 0;
          ph ^= 1u;
        }
      }
      if constexpr (PAIR) umma_commit_pair(drain + 1 + part);
      else umma_commit(drain + 1 + part);
      mbar_wait(drain + 1 + part, 0, &g_status, kCodeDrain);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    // Warp w reads the TMEM lanes [32 q, 32 q + 32), q = w % 4, and half of the columns, all of
    // them before anything else is done: the next tile's MMAs wait for the accumulator.
    const int q = warp & 3, ew = warp - 2, et = threadIdx.x - 64;
    const int c_beg = (ew >> 2) * (BN / 2);
    float* s_rw = reinterpret_cast<float*>(stg + kEpiWarps * C::STG_BUF);
    float* s_bias = s_rw + BN;
    int acc = 0;
    uint32_t aph = 0;
    if (epi.tma_store && lane == 0) tma_prefetch_desc(&tmOut);
    for (int t = t0; t < total; t += tstep) {
      int mb, nb;
      tile_at<C::BMT>(t, m_tiles, n_tiles, mb, nb);
      const int64_t row0 = static_cast<int64_t>(mb) * C::BMT + static_cast<int>(half) * BM + q * 32;
      const int64_t row = row0 + lane;
      const int rows = static_cast<int>(M - row0 < 32 ? (M > row0 ? M - row0 : 0) : 32);
      float ra = 1.0f, rw = 1.0f, bs = 0.0f;
      if (et < BN && nb * BN + et < N) {
        const int n = nb * BN + et;
        if constexpr (FMT == FNI8_NVFP4) rw = __ldg(epi.w_rs + n);
        if (epi.bias != nullptr)
          bs = epi.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(epi.bias)[n])
                        : __half2float(static_cast<const __half*>(epi.bias)[n]);
      }
      if constexpr (FMT == FNI8_NVFP4)
        if (row < M) ra = __ldg(epi.a_rs + row);
      int ok = 0;
      if (lane == 0) ok = mbar_wait(&tfull[acc], aph, &g_status, kCodeEpilogue) ? 1 : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!named_bar_and(2, kEpiThreads, ok)) break;  // also: the previous tile's scales are read
      tc_fence_after();
      if (et < BN) {
        s_rw[et] = rw;
        s_bias[et] = bs;
      }
      named_bar_sync(2, kEpiThreads);
      const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * BN + c_beg);
      constexpr int kChunks = BN / 64;
      uint32_t r[kChunks][32];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) tmem_ld32(tb + c * 32, r[c]);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < kChunks; ++c) tmem_regs_ready(r[c]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (half == 0) mbar_arrive(&tempty[acc]);
        else mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0));
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int n0 = nb * BN + c_beg + c * 32;
        if (rows > 0 && n0 < N) {
          const float* w = s_rw + c_beg + c * 32;
          const float* b = s_bias + c_beg + c * 32;
          uint4 o[4];
          if (epi.bf16) finish_chunk<__nv_bfloat16, FMT>(r[c], ra, w, b, epi.bias != nullptr, o);
          else finish_chunk<__half, FMT>(r[c], ra, w, b, epi.bias != nullptr, o);
          store_slab(stg + ew * C::STG_BUF, o, lane, &tmOut, epi.tma_store != 0, static_cast<uint16_t*>(epi.out), n0,
                     N, row0, rows);
        }
      }
      if (++acc == C::NACC) {
        acc = 0;
        aph ^= 1u;
      }
    }
    if (epi.tma_store && lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }

  if constexpr (PAIR) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace fp4
}  // namespace fni8b

namespace fni8h {

using namespace fni8b;

int fp4_status_read_and_clear(int* code) {
  int v = 0, z = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, fp4::g_status, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "read fp4 watchdog");
  e = cudaMemcpyToSymbol(fp4::g_status, &z, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "clear fp4 watchdog");
  *code = v;
  return FNI8_OK;
}

namespace {

template <int FMT, int BN, bool PAIR>
int launch_tile(const Fp4Gemm& g, cudaStream_t st) {
  using C = fp4::Cfg<FMT, BN, PAIR>;
  auto kern = fp4::fp4_tile_kernel<FMT, BN, PAIR>;
  static std::atomic<bool> configured[kMaxDevices] = {};
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices) return fail(FNI8_ERR_CUDA, "no current CUDA device");
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(fp4 gemm)");
    configured[dev] = true;
  }
  const uint64_t row = (uint64_t)fp4::padded_k(g.K) / 2;
  CUtensorMap ta, tb, tsa, tsb, to = {};
  if (int s = encode_tmap_2d_i8(&ta, g.a, row, (uint64_t)g.M, row, 128, 128)) return s;
  if (int s = encode_tmap_2d_i8(&tb, g.w, row, (uint64_t)g.N, row, 128, (uint32_t)C::BNL)) return s;
  if (int s = encode_scale_map(&tsa, g.a_sf, FMT, g.M, g.K, C::TILES)) return s;
  if (int s = encode_scale_map(&tsb, g.w_sf, FMT, g.N, g.K, C::TILES)) return s;
  fp4::Epi epi{g.a_rs, g.w_rs, g.bias, g.out, g.bf16 ? 1 : 0, 0};
  if (g.N % 8 == 0 && (reinterpret_cast<uintptr_t>(g.out) & 15u) == 0) {
    if (int s = encode_tmap_2d_16_sw(&to, g.out, g.bf16, (uint64_t)g.N, (uint64_t)g.M, (uint64_t)g.N * 2, 32, 32, true))
      return s;
    epi.tma_store = 1;
  }
  const int64_t tiles = ((g.M + C::BMT - 1) / C::BMT) * ((g.N + BN - 1) / BN);
  if (tiles >= (1LL << 31)) return fail(FNI8_ERR_UNSUPPORTED, "fp4 GEMM: too many tiles");
  const int64_t ctas = PAIR ? 2 * tiles : tiles;
  const int sms = num_sms(dev), cap = PAIR ? (sms & ~1) : sms;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas < cap ? ctas : cap));
  cfg.blockDim = dim3(fp4::kTileThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, ta, tb, tsa, tsb, to, epi, (int)g.M, (int)g.N,
                                           (int)fp4::padded_k(g.K), (int)fp4::k_tiles(FMT, g.K));
  if (e != cudaSuccess) return cuda_status(e, "launch fp4 gemm");
  return FNI8_OK;
}

// 128 x 128 tiles of one CTA each where they take no more waves than 256 x 256 tiles of a pair,
// whose waves last longer: 192 x 4096 x 4096 mxfp4 11.6 us (pairs 13.1), 333 x 12288 x 4096 18.8
// (22.6), 512 x 1024 x 4096 nvfp4 11.3 (14.3), two waves against one 1024 x 4096 x 4096 19.0 (14.9).
template <int FMT>
int pick_tile(const Fp4Gemm& g, cudaStream_t st) {
  const int64_t sms = num_sms(current_device()), pairs = sms > 1 ? sms / 2 : 1;
  const int64_t small = ((g.M + 127) / 128) * ((g.N + 127) / 128), large = ((g.M + 255) / 256) * ((g.N + 255) / 256);
  if ((small + sms - 1) / sms <= (large + pairs - 1) / pairs) return launch_tile<FMT, 128, false>(g, st);
  return launch_tile<FMT, 256, true>(g, st);
}

// Up to 64 tokens the split-K kernel. Above, it takes over where the tiles leave SMs idle and
// the cut shortens the K loop by more than eight stages (0.4 us each): the partial sums' way
// through shared memory costs about as much. 128 x 4096 x 12288 nvfp4 16.3 us (tiles 24), 128 x
// 6144 x 4096 (8 of 16 stages) 14.9 (12.0), 128 x 2048 x 768 9.5 (5.7).
int run_gemm(const Fp4Gemm& g, cudaStream_t st) {
  if (g.M <= 64) return fp4_splitk(g, st);
  const int64_t kb = (fp4::padded_k(g.K) + 255) / 256;
  if (kb > 8 && ((g.M + 127) / 128) * ((g.N + 127) / 128) <= num_sms(current_device())) {
    const int parts = fp4_splitk_parts(g);
    if (kb - (kb + parts - 1) / parts > 8) return fp4_splitk(g, st);
  }
  if (g.format == FNI8_MXFP4) return pick_tile<FNI8_MXFP4>(g, st);
  return pick_tile<FNI8_NVFP4>(g, st);
}

int check_gemm_fp4(const Fp4Gemm& g, int out_dtype) {
  if (g.format != FNI8_MXFP4 && g.format != FNI8_NVFP4)
    return fail(FNI8_ERR_INVALID, "fp4 GEMM: format %d: expected MXFP4 or NVFP4", g.format);
  if (out_dtype != FNI8_F16 && out_dtype != FNI8_BF16)
    return fail(FNI8_ERR_INVALID, "out_dtype %d: expected F16 or BF16", out_dtype);
  if (g.M < 0 || g.N <= 0 || g.K <= 0)
    return fail(FNI8_ERR_INVALID, "bad GEMM shape M=%lld N=%lld K=%lld", (long long)g.M, (long long)g.N, (long long)g.K);
  // the scale maps address four rows of 128 bytes per tile with 32-bit coordinates
  const int64_t lim = 1LL << 31;
  if (g.M >= lim || g.N >= lim || g.K >= lim ||
      (fp4::row_tiles(g.M) + 2) * fp4::k_tiles(g.format, g.K) * 4 >= lim ||
      (fp4::row_tiles(g.N) + 2) * fp4::k_tiles(g.format, g.K) * 4 >= lim)
    return fail(FNI8_ERR_UNSUPPORTED, "fp4 GEMM: sizes too large");
  if (g.M == 0) return FNI8_OK;
  if (!g.w || !g.w_sf || !g.out) return fail(FNI8_ERR_INVALID, "null GEMM operand");
  if (g.format == FNI8_NVFP4 && !g.w_rs) return fail(FNI8_ERR_INVALID, "nvfp4 GEMM: null row scale");
  if ((reinterpret_cast<uintptr_t>(g.w) | reinterpret_cast<uintptr_t>(g.w_sf)) & 15u)
    return fail(FNI8_ERR_ALIGN, "fp4 GEMM: codes and scales must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(g.out) | reinterpret_cast<uintptr_t>(g.bias)) & 1u)
    return fail(FNI8_ERR_ALIGN, "fp4 GEMM: out and bias must be 2-byte aligned");
  return FNI8_OK;
}

// Scratch of fni8_linear_fp4: scale tiles, codes, row scales.
struct Fp4Scratch {
  size_t q, rs, total;
};
Fp4Scratch fp4_scratch(int format, int64_t M, int64_t K) {
  Fp4Scratch s;
  s.q = fni8_fp4_scale_bytes(format, M, K);
  s.rs = s.q + static_cast<size_t>(M) * (fp4::padded_k(K) / 2);
  s.total = s.rs + static_cast<size_t>(M) * 4;
  return s;
}

}  // namespace
}  // namespace fni8h

using namespace fni8h;

extern "C" int fni8_gemm_fp4(const uint8_t* a, const uint8_t* a_sf, const float* a_row_scale, const uint8_t* w,
                             const uint8_t* w_sf, const float* w_row_scale, const void* bias, void* out, int out_dtype,
                             int format, int64_t M, int64_t N, int64_t K, void* stream) {
  const Fp4Gemm g{a, a_sf, a_row_scale, w, w_sf, w_row_scale, bias, out, out_dtype == FNI8_BF16, format, M, N, K};
  if (int s = check_gemm_fp4(g, out_dtype)) return s;
  if (M == 0) return FNI8_OK;
  if (!a || !a_sf) return fail(FNI8_ERR_INVALID, "null GEMM operand");
  if (format == FNI8_NVFP4 && !a_row_scale) return fail(FNI8_ERR_INVALID, "nvfp4 GEMM: null row scale");
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(a_sf)) & 15u)
    return fail(FNI8_ERR_ALIGN, "fp4 GEMM: codes and scales must be 16-byte aligned");
  return run_gemm(g, static_cast<cudaStream_t>(stream));
}

extern "C" size_t fni8_linear_fp4_scratch_bytes(int format, int64_t M, int64_t N, int64_t K) {
  if ((format != FNI8_MXFP4 && format != FNI8_NVFP4) || M <= 0 || N <= 0 || K <= 0) return 0;
  return fp4_fused_supported(format, M, N, K) ? 0 : fp4_scratch(format, M, K).total;
}

extern "C" int fni8_linear_fp4(const void* x, int dtype, const uint8_t* w, const uint8_t* w_sf, const float* w_row_scale,
                               const void* bias, void* out, int format, int64_t M, int64_t N, int64_t K, void* scratch,
                               size_t scratch_bytes, void* stream) {
  Fp4Gemm g{nullptr, nullptr, nullptr, w, w_sf, w_row_scale, bias, out, dtype == FNI8_BF16, format, M, N, K};
  if (int s = check_gemm_fp4(g, dtype)) return s;
  if (M == 0) return FNI8_OK;
  if (!x) return fail(FNI8_ERR_INVALID, "null linear input");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
  if (aligned && fp4_fused_supported(format, M, N, K)) return fp4_fused(g, x, st);
  const Fp4Scratch sc = fp4_scratch(format, M, K);
  if (!scratch || scratch_bytes < sc.total) {
    if (!aligned && fp4_fused_supported(format, M, N, K))
      return fail(FNI8_ERR_ALIGN, "fp4 linear: x must be 16-byte aligned to run without scratch");
    return fail(FNI8_ERR_WORKSPACE, "fp4 linear needs %zu scratch bytes (got %zu)", sc.total, scratch_bytes);
  }
  uint8_t* b = static_cast<uint8_t*>(scratch);
  g.a_sf = b;
  g.a = b + sc.q;
  g.a_rs = reinterpret_cast<float*>(b + sc.rs);
  if (int s = fp4_check_rows(x, dtype, format, M, K, b + sc.q, b, reinterpret_cast<float*>(b + sc.rs))) return s;
  if (int s = fp4_quantize(x, dtype, format, M, K, false, b + sc.q, b, reinterpret_cast<float*>(b + sc.rs), st)) return s;
  return run_gemm(g, st);
}
