// GEMM of 4-bit floating point operands for few tokens or few tiles: every SM streams weights.
//
//   acc^T[n, m] = sum_k w[n,k] sw[n,k/g] a[m,k] sa[m,k/g]   (tcgen05.mma kind::mxf4 / mxf4nvf4)
//   out[m, n]   = dtype(acc * ra[m] * rw[n] (+ bias[n]))
//
// Bound: HBM, N K (1/2 + 1/g) bytes of weights read once. As in gemm_splitk.cu the operands
// are swapped (128 weight rows = MMA M, NT tokens = MMA N) and a cluster of S CTAs splits the
// K range of a weight tile (and of a block of 128 tokens, where there are more), S chosen so that the grid fills the GPU
// once; the first weights enter L2 while the kernel in front still runs. Here the S partial accumulators meet in shared memory:
// CTA r owns a share of the token columns, every CTA stores the columns of the others into
// their landing areas (distributed shared memory, 16-byte pieces of four tokens, the weight row
// innermost), and the owner adds the S parts in rank order, so the result does not depend on
// timing and there is no workspace.
//
// FUSED (fni8_linear_fp4, up to 16 tokens): the epilogue warps quantise the CTA's K slice of
// the 16-bit rows themselves, straight into the swizzled operand tiles and scale tiles, while
// the weights are on their way; the ring then holds weights only. It saves the quantiser's
// launch and its scratch, and up to 1.6 us on the device (fused_chunks). An nvfp4 row's maximum
// goes through the cluster's shared memory: each CTA posts its slice's.
#include "fp4_common.cuh"
#include "gemm_internal.h"

namespace fni8b {
namespace fp4s {

using namespace fp4;

constexpr int kThreads = 192;
constexpr int kMaxStages = 8;

static __device__ int g_status;
enum : int { kCodeProducer = 0x711, kCodeMma = 0x712, kCodeEpilogue = 0x713, kCodeDrain = 0x714 };

struct Epi {
  const void* x;  // FUSED: [M, K], 16-byte aligned rows of the output type
  int64_t K;
  const float* a_rs;
  const float* w_rs;
  const void* bias;
  void* out;
  int bf16;
};

template <int FMT, int NT, bool FUSED>
struct Cfg {
  static constexpr int TILES = Fmt<FMT>::kStageTiles;
  static constexpr int W_BYTES = 128 * 128;
  static constexpr int X_BYTES = NT * 128;
  static constexpr int SF_BYTES = TILES * 512;
  static constexpr int X_STAGE = X_BYTES + SF_BYTES;
  static constexpr int STAGE = W_BYTES + SF_BYTES + (FUSED ? 0 : X_STAGE);  // of the ring
  static constexpr int ACC_COLS = NT;
  static constexpr int SF_COLS = 8 * TILES;  // weights', then tokens' scales of a stage
  static constexpr int COLS = ACC_COLS + 2 * SF_COLS;
  static constexpr int TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : 256;
  // A CTA holds its columns while it waits for its cluster, and another's allocation waits for columns: clusters of
  // two streams could wait for each other for good. So no CTA takes a larger share of an SM's 512 columns than of
  // its 228 KB of shared memory (1 KB of them the system's, for each CTA): what is resident together always fits.
  static constexpr int MIN_SMEM = TMEM_COLS * (228 * 1024 / 512) - 1024;
  static_assert(STAGE % 1024 == 0, "stages keep the 1024-byte alignment of the swizzle");
};

// token columns that rank r of S owns: [r share, (r + 1) share) of the first mcols
__host__ __device__ __forceinline__ int column_share(int mcols, int S) { return ((mcols + S - 1) / S + 3) & ~3; }

// Chunks of eight values that a thread of FUSED takes at most. Measured against the two
// kernels at M = 1, in a graph: 4096 x 12288 mxfp4 10.3 / 11.9 us, nvfp4 12.7 / 13.7; 6144 x 4096
// mxfp4 7.3 / 7.9, nvfp4 9.6 / 8.0 (called eagerly one launch less counts for more); 24576 x 4096
// mxfp4 14.7 / 14.8 (4 chunks); nvfp4, which reads twice through its maxima, lost 1.7 us there.
__host__ __device__ constexpr int fused_chunks(int fmt) { return fmt == FNI8_MXFP4 ? 4 : 2; }

// FUSED: the epilogue warps' part before the product. 128 threads; xs: nk stages of X_STAGE
// bytes; s_top: [16] row maxima of this CTA's slice, tops: [S][16] of all; s_ra: row scales.
template <int FMT, int NT, typename T>
__device__ __forceinline__ void quantise_slice(const Epi& epi, int M, int kbeg, int nk, int rank, int S, uint8_t* xs,
                                               uint32_t* s_top, uint32_t* tops, float* s_ra, uint64_t* posted) {
  using C = Cfg<FMT, NT, true>;
  constexpr int kLanes = Fmt<FMT>::kBlock / 8;  // threads that share a block
  constexpr int kFusedChunks = fused_chunks(FMT);
  const int et = threadIdx.x - 64, lane = threadIdx.x & 31;
  const int per_row = nk * 32;  // chunks of eight values; a warp's 32 are one row's
  const int items = M * per_row;
  const T* x = static_cast<const T*>(epi.x) + static_cast<int64_t>(kbeg) * 256;
  const int left = static_cast<int>(epi.K - static_cast<int64_t>(kbeg) * 256);  // values of a row from kbeg on
  uint4 raw[kFusedChunks];  // this thread's chunks et, et + 128, ...; a warp has the same number of them
#pragma unroll
  for (int b = 0; b < kFusedChunks; ++b) {
    const int i = et + 128 * b;
    if (i >= items) break;
    const int m = i / per_row, c = i - m * per_row;
    raw[b] = make_uint4(0, 0, 0, 0);
    if (c * 8 < left) raw[b] = __ldg(reinterpret_cast<const uint4*>(x + m * epi.K + c * 8));  // K % 8 == 0
  }
  auto block_top = [&](int b) {
    uint32_t m = pattern_max(raw[b]);
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return pattern_bits<T>(m);
  };
  if constexpr (FMT == FNI8_NVFP4) {
    if (et < 16) s_top[et] = 0;
    named_bar_sync(1, 128);
#pragma unroll
    for (int b = 0; b < kFusedChunks; ++b) {
      if (et + 128 * b >= items) break;
      uint32_t top = block_top(b);
      if (top >= kInfBits) top = 0;  // a block with an infinity or NaN stands for itself alone
#pragma unroll
      for (int o = kLanes; o < 32; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) atomicMax(&s_top[(et + 128 * b) / per_row], top);
    }
    named_bar_sync(1, 128);
  }
  if (S > 1) {
    // the peers have started (every thread waits here or before the exchange); the first warp
    // posts the maxima to all of them
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if constexpr (FMT == FNI8_NVFP4) {
      if (et < 32) {
        for (int i = et; i < S * 16; i += 32) {
          const uint32_t to = mapa_shared(smem_u32(tops), static_cast<uint32_t>(i >> 4));
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + static_cast<uint32_t>((rank * 16 + (i & 15)) * 4)),
                       "r"(s_top[i & 15])
                       : "memory");
        }
        __syncwarp();
        if (et < S) mbar_arrive_cluster(mapa_shared(smem_u32(posted), static_cast<uint32_t>(et)));
      }
      mbar_wait_cluster(posted, 0, &g_status, kCodeEpilogue);
    }
  }
  if constexpr (FMT == FNI8_NVFP4) {
    if (et < M) {
      uint32_t top = S > 1 ? 0 : s_top[et];
      if (S > 1)
        for (int s = 0; s < S; ++s) top = max(top, tops[s * 16 + et]);
      s_ra[et] = pow2f(row_exponent(top));
    }
    named_bar_sync(1, 128);
  }
#pragma unroll
  for (int b = 0; b < kFusedChunks; ++b) {
    const int i = et + 128 * b;
    if (i >= items) break;
    const int m = i / per_row, c = i - m * per_row;
    const uint32_t top = block_top(b);
    const int row_exp = FMT == FNI8_NVFP4 ? static_cast<int>(__float_as_uint(s_ra[m]) >> 23) - 127 : 0;
    const BlockScale<FMT> scale(top, row_exp);
    const uint32_t codes = scale.template codes<T>(raw[b]);
    uint8_t* st = xs + (c >> 5) * C::X_STAGE;
    *reinterpret_cast<uint32_t*>(st + m * 128 + ((((c & 31) >> 2) ^ (m & 7)) << 4) + (c & 3) * 4) = codes;
    const int s = (c & 31) / kLanes;
    if (lane % kLanes == 0) st[C::X_BYTES + (s >> 2) * 512 + m * 16 + (s & 3)] = static_cast<uint8_t>(scale.byte);
  }
  fence_proxy_async_smem();  // read by the tensor core
}

template <int FMT, int NT, bool FUSED>
__global__ void __launch_bounds__(kThreads, 2)
    fp4_splitk_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                      const __grid_constant__ CUtensorMap tmSW, const __grid_constant__ CUtensorMap tmSX, Epi epi, int rows,
                      int N, int Kp, int ktiles, int stages, int xstages) {
  using C = Cfg<FMT, NT, FUSED>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* xs = smem + stages * C::STAGE;  // FUSED: the slice's quantised rows
  uint8_t* rest = xs + (FUSED ? xstages * C::X_STAGE : 0);
  uint64_t* full = reinterpret_cast<uint64_t*>(rest);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;
  uint64_t* drain = tfull + 1;
  uint64_t* xready = drain + 1;
  uint64_t* posted = xready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(posted + 1);
  float* s_ra = reinterpret_cast<float*>(rest + 256);                          // [NT]
  uint32_t* tops = reinterpret_cast<uint32_t*>(rest + 256 + NT * 4);           // FUSED: [9][16]
  uint4* land = reinterpret_cast<uint4*>(rest + 256 + NT * 4 + (FUSED ? 9 * 64 : 0));  // [S][share / 4][128]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank()), S = static_cast<int>(cluster_nctarank());
  const int tile = static_cast<int>(blockIdx.x) / S;
  const int m0 = static_cast<int>(blockIdx.y) * NT, M = min(rows - m0, NT);  // this CTA's tokens
  const int kb = (Kp + 255) / 256;
  const int kbeg = static_cast<int>(static_cast<int64_t>(rank) * kb / S);
  const int nk = static_cast<int>(static_cast<int64_t>(rank + 1) * kb / S) - kbeg;

  // The kernel in front may be the one that writes the weights or their scales, and what a grid wrote is
  // promised to be seen only behind the wait; so ahead of it the first ring's weights only enter L2, where
  // a line that is written later stays right.
  const int pre = nk < stages ? nk : stages;
  if (warp == 2 && lane == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmSW);
    if constexpr (!FUSED) {
      tma_prefetch_desc(&tmX);
      tma_prefetch_desc(&tmSX);
    }
    for (int i = 0; i < pre; ++i) {
      tma_prefetch_l2_2d(&tmW, (kbeg + i) * 128, tile * 128);
      tma_prefetch_l2_2d(&tmSW, 0, (tile * ktiles + (kbeg + i) * C::TILES) * 4);
    }
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_init(drain, 1);
    mbar_init(xready, 4);
    mbar_init(posted, static_cast<uint32_t>(S));
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // the peers have started before anything is stored into their shared memory
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_wait();  // of every thread, before any operand is read

  int okt = 0;
  float rw = 1.0f, bias = 0.0f;  // of this epilogue thread's weight row
  const int row = (warp & 3) * 32 + lane;  // epilogue warps 2-5 read the TMEM lanes of quarters 2, 3, 0, 1
  const int n = tile * 128 + row;
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      auto load_w = [&](int s, int k) {
        uint8_t* dst = smem + s * C::STAGE;
        mbar_arrive_expect_tx(&full[s], C::STAGE);
        tma_load_2d(&tmW, &full[s], dst, k * 128, tile * 128);
        tma_load_2d(&tmSW, &full[s], dst + C::W_BYTES, 0, (tile * ktiles + k * C::TILES) * 4);
      };
      auto load_x = [&](int s, int k) {
        if constexpr (!FUSED) {
          uint8_t* dst = smem + s * C::STAGE + C::W_BYTES + C::SF_BYTES;
          tma_load_2d(&tmSX, &full[s], dst, 0, (static_cast<int>(blockIdx.y) * ktiles + k * C::TILES) * 4);
          tma_load_2d(&tmX, &full[s], dst + C::SF_BYTES, k * 128, m0);
        }
      };
      for (int i = 0; i < pre; ++i) {
        load_w(i, kbeg + i);
        load_x(i, kbeg + i);
      }
      int stage = pre % stages, issued = pre;
      uint32_t ph = pre == stages ? 1u : 0u, armed = 0;
      for (int i = pre; i < nk; ++i) {
        if (!mbar_wait(&empty[stage], ph ^ 1u, &g_status, kCodeProducer)) break;
        load_w(stage, kbeg + i);
        load_x(stage, kbeg + i);
        armed = (armed & ~(1u << stage)) | (ph << stage);
        ++issued;
        if (++stage == stages) {
          stage = 0;
          ph ^= 1u;
        }
      }
      const int pending = issued < stages ? issued : stages;
      for (int i = 0; i < pending; ++i) {
        const int s = (stage - 1 - i + 2 * stages) % stages;
        mbar_wait(&full[s], (armed >> s) & 1u, &g_status, kCodeDrain);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int stage = 0;
      uint32_t ph = 0;
      bool ok = !FUSED || mbar_wait(xready, 0, &g_status, kCodeMma);
      for (int i = 0; i < nk && ok; ++i) {
        if (!mbar_wait(&full[stage], ph, &g_status, kCodeMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint8_t* sw = smem + stage * C::STAGE;
        const uint8_t* sx = FUSED ? xs + i * C::X_STAGE : sw + C::W_BYTES + 2 * C::SF_BYTES;
        const uint8_t* sfx = FUSED ? sx + C::X_BYTES : sw + C::W_BYTES + C::SF_BYTES;
        const uint32_t ta = tmem_base + C::ACC_COLS + static_cast<uint32_t>((i & 1) * C::SF_COLS);
        const uint32_t tb = ta + 4 * C::TILES;
        const int steps = min(4, (Kp - (kbeg + i) * 256 + 63) / 64);
        stage_scales<FMT, false, NT>(sw + C::W_BYTES, sfx, ta, tb);
        stage_mmas<FMT, false, 128, NT>(tmem_base, sw, sx, ta, tb, steps, i == 0);
        umma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          ph ^= 1u;
        }
      }
      if (ok) umma_commit(tfull);
      umma_commit(drain);
      mbar_wait(drain, 0, &g_status, kCodeDrain);
    }
  } else {
    if constexpr (FMT == FNI8_NVFP4)
      if (n < N) rw = __ldg(epi.w_rs + n);
    if (n < N && epi.bias != nullptr)
      bias = epi.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(epi.bias)[n])
                      : __half2float(static_cast<const __half*>(epi.bias)[n]);
    if constexpr (FUSED) {
      if (epi.bf16) quantise_slice<FMT, NT, __nv_bfloat16>(epi, M, kbeg, nk, rank, S, xs, tops + 128, tops, s_ra, posted);
      else quantise_slice<FMT, NT, __half>(epi, M, kbeg, nk, rank, S, xs, tops + 128, tops, s_ra, posted);
      __syncwarp();
      if (lane == 0) mbar_arrive(xready);
    } else if constexpr (FMT == FNI8_NVFP4) {
      for (int m = threadIdx.x - 64; m < M; m += 128) s_ra[m] = __ldg(epi.a_rs + m0 + m);
      named_bar_sync(1, 128);
    }
    if (lane == 0) okt = mbar_wait(tfull, 0, &g_status, kCodeEpilogue) ? 1 : 0;
    okt = __shfl_sync(0xffffffffu, okt, 0);
    tc_fence_after();
    pdl_launch_dependents();  // (at the start, here and after the exchange measured within 3 %)
  }
  __syncwarp();
  if (!(FUSED && S > 1 && warp >= 2))  // (those have waited already)
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  const uint32_t taddr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
  const int mcols = (M + 3) & ~3;
  const int share = S > 1 ? column_share(mcols, S) : mcols;
  if (S > 1) {
    if (warp >= 2 && okt) {
      const int g4 = share >> 2;
      int owner = 0, first = 0;  // of the column at hand
      uint32_t peer = mapa_shared(smem_u32(land), 0);
#pragma unroll 1
      for (int c0 = 0; c0 < mcols; c0 += 16) {
        uint32_t r[16];
        tmem_ld16(taddr + static_cast<uint32_t>(c0), r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const int c = c0 + j;
          if (c < mcols) {
            if (c == first + share) {
              first = c;
              peer = mapa_shared(smem_u32(land), static_cast<uint32_t>(++owner));
            }
            if (owner != rank)
              st_dsmem_v4(peer + static_cast<uint32_t>(((rank * g4 + ((c - first) >> 2)) * 128 + row) * 16),
                          make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]));
          }
        }
      }
    }
    __syncwarp();
    cluster_sync_all();
  }
  if (warp >= 2 && okt) {
    const int own0 = rank * share, end = min(own0 + share, M), g4 = share >> 2;
#pragma unroll 1
    for (int c0 = own0; c0 < end; c0 += 16) {
      uint32_t r[16];
      tmem_ld16(taddr + static_cast<uint32_t>(c0), r);  // columns behind the accumulator are not used
      tmem_ld_wait();
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = rank == 0 ? __uint_as_float(r[j]) : 0.0f;
      for (int s = 0; s < S; ++s) {
        if (s == 0 && rank == 0) continue;
        const uint4* part = land + (s * g4 + ((c0 - own0) >> 2)) * 128 + row;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          if (c0 + j < end) {
            uint4 p = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
            if (s != rank) p = part[(j >> 2) * 128];
            v[j] = __fadd_rn(v[j], __uint_as_float(p.x));
            v[j + 1] = __fadd_rn(v[j + 1], __uint_as_float(p.y));
            v[j + 2] = __fadd_rn(v[j + 2], __uint_as_float(p.z));
            v[j + 3] = __fadd_rn(v[j + 3], __uint_as_float(p.w));
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int m = c0 + j;
        if (m < end && n < N) {
          float o = v[j];
          if constexpr (FMT == FNI8_NVFP4) o = __fmul_rn(__fmul_rn(o, s_ra[m]), rw);
          if (epi.bias != nullptr) o = __fadd_rn(o, bias);
          const int64_t at = static_cast<int64_t>(m0 + m) * N + n;
          if (epi.bf16) static_cast<__nv_bfloat16*>(epi.out)[at] = __float2bfloat16_rn(o);
          else static_cast<__half*>(epi.out)[at] = __float2half_rn(o);
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

}  // namespace fp4s
}  // namespace fni8b

namespace fni8h {

using namespace fni8b;

int fp4s_status_read_and_clear(int* code) {
  int v = 0, z = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, fp4s::g_status, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "read fp4 split-K watchdog");
  e = cudaMemcpyToSymbol(fp4s::g_status, &z, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "clear fp4 split-K watchdog");
  *code = v;
  return FNI8_OK;
}

namespace {

constexpr int kMinRing = 2;

struct Plan {
  int S, stages, xstages, smem;
  bool fits;
};

// Ring: half an SM's shared memory where that holds kMinRing stages beside the rest (two CTAs
// per SM), else a whole SM's. S: as many CTAs per tile as are resident at once, less an eighth
// where the quantiser's last CTAs are still there: a cluster that finds no room waits for a whole
// other one to end (32 x 4096 x 12288 nvfp4 19.7 -> 13.9 us; the longer products of 64 tokens
// and more lose as much by the smaller S).
template <int FMT, int NT, bool FUSED>
Plan plan_splitk(int64_t rows, int64_t N, int64_t K) {
  using C = fp4s::Cfg<FMT, NT, FUSED>;
  const int64_t tiles = (N + 127) / 128 * ((rows + NT - 1) / NT), M = rows < NT ? rows : NT;
  const int kb = (int)((fp4::padded_k(K) + 255) / 256);
  auto plan = [&](int S) {
    const int land = S > 1 ? S * fp4s::column_share(((int)M + 3) & ~3, S) * 128 * 4 : 0;
    const int per = (kb + S - 1) / S;
    const int64_t fixed = 1024 + 256 + NT * 4 + land + (FUSED ? 9 * 64 + (int64_t)per * C::X_STAGE : 0);
    int64_t n = (113 * 1024 - fixed) / C::STAGE;
    if (n < kMinRing && n < per) n = (225 * 1024 - fixed) / C::STAGE;
    n = n < fp4s::kMaxStages ? n : fp4s::kMaxStages;
    n = n < per ? n : per;
    const bool slice = !FUSED || M * per * 32 <= 128 * fp4s::fused_chunks(FMT);
    const int64_t smem = fixed + n * C::STAGE;
    return Plan{S, (int)n, per, (int)(smem < C::MIN_SMEM ? C::MIN_SMEM : smem), slice && n >= (per < kMinRing ? per : kMinRing)};
  };
  if constexpr (NT == 16 && !FUSED) {
    // split as the fused form does, so that both give the same sums
    const Plan f = K % 8 == 0 ? plan_splitk<FMT, NT, true>(M, N, K) : Plan{};
    if (f.fits) return plan(f.S);
  }
  int64_t most = 2 * (int64_t)num_sms(current_device()) / tiles;
  most = most < 1 ? 1 : most > 8 ? 8 : most;
  Plan p = plan((int)(most > kb ? kb : most));
  while (p.S > 1) {
    const int n = p.fits ? max_active_clusters(fp4s::kThreads, p.smem, p.S) : -1;
    if (p.fits && (n < 0 || tiles <= (!FUSED && NT <= 32 ? n - n / 8 : n))) break;
    p = plan(p.S - 1);
  }
  return p;
}

template <int FMT, int NT, bool FUSED>
int launch_splitk(const Fp4Gemm& g, const void* x, cudaStream_t st) {
  using C = fp4s::Cfg<FMT, NT, FUSED>;
  auto kern = fp4s::fp4_splitk_kernel<FMT, NT, FUSED>;
  static std::atomic<bool> configured[kMaxDevices] = {};
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices) return fail(FNI8_ERR_CUDA, "no current CUDA device");
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(fp4 split-K)");
    configured[dev] = true;
  }
  const Plan p = plan_splitk<FMT, NT, FUSED>(g.M, g.N, g.K);
  if (!p.fits) return fail(FNI8_ERR_UNSUPPORTED, "fp4 split-K GEMM: K=%lld does not fit", (long long)g.K);
  const uint64_t row = (uint64_t)fp4::padded_k(g.K) / 2;
  CUtensorMap tw, tx = {}, tsw, tsx = {};
  if (int s = encode_tmap_2d_i8(&tw, g.w, row, (uint64_t)g.N, row, 128, 128)) return s;
  if (int s = encode_scale_map(&tsw, g.w_sf, FMT, g.N, g.K, C::TILES)) return s;
  if constexpr (!FUSED) {
    if (int s = encode_tmap_2d_i8(&tx, g.a, row, (uint64_t)g.M, row, 128, NT)) return s;
    if (int s = encode_scale_map(&tsx, g.a_sf, FMT, g.M, g.K, C::TILES)) return s;
  }
  const fp4s::Epi epi{x, g.K, g.a_rs, g.w_rs, g.bias, g.out, g.bf16 ? 1 : 0};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((g.N + 127) / 128 * p.S), (unsigned)((g.M + NT - 1) / NT));
  cfg.blockDim = dim3(fp4s::kThreads);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled();
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tw, tx, tsw, tsx, epi, (int)g.M, (int)g.N,
                                           (int)fp4::padded_k(g.K), (int)fp4::k_tiles(FMT, g.K), p.stages, p.xstages);
  if (e != cudaSuccess) return cuda_status(e, "launch fp4 split-K gemm");
  return FNI8_OK;
}

template <int FMT>
int splitk_any(const Fp4Gemm& g, cudaStream_t st) {
  if (g.M <= 16) return launch_splitk<FMT, 16, false>(g, nullptr, st);
  if (g.M <= 32) return launch_splitk<FMT, 32, false>(g, nullptr, st);
  if (g.M <= 64) return launch_splitk<FMT, 64, false>(g, nullptr, st);
  return launch_splitk<FMT, 128, false>(g, nullptr, st);
}

}  // namespace

int fp4_splitk(const Fp4Gemm& g, cudaStream_t st) {
  return g.format == FNI8_MXFP4 ? splitk_any<FNI8_MXFP4>(g, st) : splitk_any<FNI8_NVFP4>(g, st);
}

int fp4_splitk_parts(const Fp4Gemm& g) {
  const Plan p = g.format == FNI8_MXFP4 ? plan_splitk<FNI8_MXFP4, 128, false>(g.M, g.N, g.K)
                                        : plan_splitk<FNI8_NVFP4, 128, false>(g.M, g.N, g.K);
  return p.fits ? p.S : 1;
}

bool fp4_fused_supported(int format, int64_t M, int64_t N, int64_t K) {
  if (M < 1 || M > 16 || K % 8 != 0) return false;
  return format == FNI8_MXFP4 ? plan_splitk<FNI8_MXFP4, 16, true>(M, N, K).fits
                              : plan_splitk<FNI8_NVFP4, 16, true>(M, N, K).fits;
}

int fp4_fused(const Fp4Gemm& g, const void* x, cudaStream_t st) {
  return g.format == FNI8_MXFP4 ? launch_splitk<FNI8_MXFP4, 16, true>(g, x, st)
                                : launch_splitk<FNI8_NVFP4, 16, true>(g, x, st);
}

}  // namespace fni8h
