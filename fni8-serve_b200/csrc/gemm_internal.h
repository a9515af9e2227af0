// Host-side functions shared between the translation units of libfni8_b200.so. Not part
// of the public C ABI (include/fni8_b200.h).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "tuning.h"

namespace fni8h {

constexpr int kMaxDevices = 64;
constexpr int kTileMaxSeg = 512;  // segments of one grouped launch

// tcgen05 tile GEMM (gemm_tile.cu). out_mode: 0 fp16, 1 bf16, 2 int32 accumulators.
// pair: 256-row tiles on CTA pairs (tcgen05.mma.cta_group::2).
int tile_gemm(const int8_t* a, const float* a_scale, const int8_t* w, const float* w_scale, const void* bias,
              const void* residual, void* out, int out_mode, int64_t M, int64_t N, int64_t K, int bn, bool pair,
              cudaStream_t st);
int tile_gemm_grouped(const int8_t* a, const float* a_scale, int64_t R, const int8_t* w, const float* w_scale,
                      int64_t E, int64_t N, int64_t K, const int32_t* seg_expert, const int32_t* seg_off,
                      const int32_t* seg_cnt, int64_t S, void* out, int out_mode, int bn, bool pair,
                      cudaStream_t st, const int32_t* row_tag = nullptr, void* const* peer_out = nullptr,
                      int n_peers = 0, int64_t peer_rows = 0);
// (row_tag set: output row r goes to row (row_tag[r] & 0xFFFFFF) of the [peer_rows, N]
// buffer peer_out[row_tag[r] >> 24] instead of out; 16-bit out_mode, N % 64 == 0, buffers
// 16-byte aligned, checked by the caller.)
// Dense tile GEMM whose epilogue writes output element (m, n) to element
// (m, col_off + n) of each of the n_peers (<= 8) buffers peer_out[p] (row stride ld
// elements; this GPU's memory or an NVLink peer's mapped into this process): a column
// shard's part of an all-gather. 16-bit out_mode, no residual; the caller validates
// alignment (buffers, ld and col_off 16-byte multiples, N % 64 == 0).
int tile_gemm_peer_cols(const int8_t* a, const float* a_scale, const int8_t* w, const float* w_scale, const void* bias,
                        int out_mode, int64_t M, int64_t N, int64_t K, void* const* peer_out, int n_peers, int64_t ld,
                        int64_t col_off, int bn, bool pair, cudaStream_t st);
// Tile GEMM over a merged gate_up weight (gate rows [0, I), up rows [I, 2I)) whose
// epilogue applies act_and_mul: out[M, I] in fp16/bf16 (out_mode 0/1), I % 128 == 0.
// Dense when seg_expert is null; grouped over S segments of a [E, 2I, K] stack otherwise.
int tile_gemm_act(const int8_t* a, const float* a_scale, int64_t M, const int8_t* w, const float* w_scale, int64_t E,
                  int64_t I, int64_t K, const int32_t* seg_expert, const int32_t* seg_off, const int32_t* seg_cnt,
                  int64_t S, int act, void* out, int out_mode, bool pair, cudaStream_t st);
// Whether dense (prefill-size) and grouped tile GEMMs run on CTA pairs.
bool tile_pair_enabled();
bool grouped_pair_enabled();
int tile_status_read_and_clear(int* code);

// Swap-AB stream-K GEMM for skinny M (gemm_stream.cu).
size_t stream_workspace_bytes(int64_t M, int64_t N, int64_t K);
int stream_gemm(const int8_t* a, const float* a_scale, const int8_t* w, const float* w_scale, const void* bias,
                const void* residual, void* out, int out_mode, int64_t M, int64_t N, int64_t K, void* ws,
                size_t ws_bytes, cudaStream_t st);
int stream_status_read_and_clear(int* code);
constexpr int64_t kStreamMaxM = 256;
// Re-zero the allocation-free GEMM's built-in scratch on the current device (synchronous).
int noalloc_scratch_reset();


// Cluster split-K swap-AB GEMM for decode (gemm_splitk.cu): int8 activations; partial sums
// of a split K range cross the zero-maintained GEMM workspace and are zeroed again.
constexpr int64_t kSplitkMaxM = 256;
bool splitk_supported(int64_t M, int64_t N, int64_t K);
// Clusters of S CTAs (`threads` threads, `smem` bytes of dynamic shared memory) that can
// be resident at once; -1 when the runtime cannot tell.
int max_active_clusters(int threads, int smem, int S);

// The split-K plan for this shape splits K (S > 1) and every one of its clusters can be
// resident at once.
bool splitk_split_one_wave(int64_t M, int64_t N, int64_t K);
size_t splitk_workspace_bytes(int64_t M, int64_t N, int64_t K);
int splitk_gemm(const int8_t* a, const float* a_scale, const int8_t* w, const float* w_scale, const void* bias,
                const void* residual, void* out, int out_mode, int64_t M, int64_t N, int64_t K, void* ws,
                size_t ws_bytes, cudaStream_t st);
int splitk_status_read_and_clear(int* code);

// W4A8 decode-shaped GEMM (gemm_w4a8.cu): packed int4 weights [N, K/2] with fp32 scales
// per 128-channel group [N, K/128]; 64 tokens per launch.
constexpr int64_t kW4ChunkM = 64;
size_t w4a8_workspace_bytes(int64_t M, int64_t N, int64_t K);
int w4a8_gemm(const int8_t* a, const float* a_scale, const uint8_t* w4, const float* w_scale, const void* bias,
              void* out, int out_mode, int64_t M, int64_t N, int64_t K, void* ws, size_t ws_bytes, cudaStream_t st);
int w4a8_status_read_and_clear(int* code);

// 4-bit floating point (fp4.cu: row kernels; gemm_fp4.cu: block-scaled GEMM). Formats and
// layouts as include/fni8_b200.h documents them.
struct Fp4Gemm {
  const uint8_t* a;
  const uint8_t* a_sf;
  const float* a_rs;
  const uint8_t* w;
  const uint8_t* w_sf;
  const float* w_rs;
  const void* bias;
  void* out;
  bool bf16;
  int format;
  int64_t M, N, K;
};
int fp4_check_rows(const void* x, int dtype, int format, int64_t M, int64_t K, const uint8_t* q, const uint8_t* sf,
                   const float* row_scale);
// pad: the scales of the rows behind M in the last tile are zeroed, and the next kernel starts when this one
// has ended; else (the rows of a GEMM that follows at once) it may start early.
int fp4_quantize(const void* x, int dtype, int format, int64_t M, int64_t K, bool pad, uint8_t* q, uint8_t* sf,
                 float* row_scale, cudaStream_t st);
// The swap-AB split-K kernel (gemm_fp4_splitk.cu), and into how many parts it would cut K at M > 64.
int fp4_splitk(const Fp4Gemm& g, cudaStream_t st);
int fp4_splitk_parts(const Fp4Gemm& g);
// Its form that quantises the 16-bit rows x itself (16-byte aligned; a, a_sf and a_rs unused).
bool fp4_fused_supported(int format, int64_t M, int64_t N, int64_t K);
int fp4_fused(const Fp4Gemm& g, const void* x, cudaStream_t st);
int fp4_status_read_and_clear(int* code);
int fp4s_status_read_and_clear(int* code);

// The routed-expert layer for a few tokens in two kernels (moe_few.cu). logits null: the
// routing topi / topw is given. h: scratch [T k, I] of the activations' type, 16-byte aligned,
// as x is.
struct FewMoe {
  const void* x;
  int dtype;
  int64_t T, H, E, I, k;
  const float* logits;
  const int32_t* topi;
  const float* topw;
  int scoring;
  const float* sel_bias;
  int64_t n_groups, topk_group;
  int norm_topk;
  float scaling;
  const int8_t* w_gu;
  const float* s_gu;
  const int8_t* w_dn;
  const float* s_dn;
  int act;
  void* h;
  void* out;
  // scratch for the lists that pass from one kernel to the other: [1], 4 x [T k], [T k][16]
  int32_t* t_count;
  int32_t* t_slot_e;
  float* t_slot_w;
  int32_t* t_ent_e;
  int32_t* t_ent_n;
  uint16_t* t_list;
  int8_t* hq;  // [T k, I]
  float* hs;   // [T k]
};
bool few_supported(int64_t T, int64_t H, int64_t k, int64_t E, int64_t I);
int few_moe(const FewMoe& m, cudaStream_t st);
int few_status_read_and_clear(int* code);

// Expert-parallel exchange kernels (ep_p2p.cu): capacity-overflow status word.
int ep_status_read_and_clear(int* code);
// src [M, N] 16-bit rows (row stride N) to columns [col_off, col_off + N) of each of the
// n_peers buffers peer_out[p] (row stride ld elements): the all-gather step of a column
// shard whose GEMM wrote a local buffer. Same alignment rules as tile_gemm_peer_cols.
int push_cols(const void* src, int64_t M, int64_t N, void* const* peer_out, int n_peers, int64_t ld, int64_t col_off,
              cudaStream_t st);

}  // namespace fni8h
