// Row kernels of the 4-bit floating point path: 16-bit rows to e2m1 codes with block scales
// (the activation stage of fni8_linear_fp4, and the weights' conversion) and back.
//
// Both formats are defined by real quotients (x / 2^e, max / 6, x / sf), and the kernels
// produce exactly their roundings:
//   * dividing by a power of two is exact (a float holds every quotient that matters: a
//     denormal one rounds to code 0 either way);
//   * max / 6 and x / sf are products with the reciprocal, corrected once by their fused
//     remainders (BlockScale), which leaves the quotient's own rounding, or its neighbour in
//     rare cases. max has at most 11 significant bits, so max / 6 either is a midpoint of e4m3
//     (then the quotient is a float and exact) or is at least 2^-17 of itself away from one,
//     further than any rounding here. With 11 bits in x and 4 in sf the same holds for x / sf
//     and the midpoints of e2m1.
// Nothing of a row depends on another row.
//
// A row belongs to 32, 128, 256 or 512 threads, sixteen values to a thread and step (an nvfp4
// block, half of an mxfp4 one: with eight, the scale's arithmetic was done twice as often and
// an nvfp4 8192 x 4096 took 25 us, 80 % of the issue slots). An nvfp4 row stays in registers
// while its maximum is found, so it is read once, up to 16384 values.
// Bound: HBM, 2 bytes read and 1/2 + 1/g written per value; the issue rate comes next.
#include "fp4_common.cuh"
#include "gemm_internal.h"

namespace fni8b {
namespace fp4 {

struct Raw16 {  // sixteen 16-bit values
  uint4 lo, hi;
};

// The values of a row from k on, zeros behind K. VW values to a load (the largest power of two
// that the rows' alignment allows).
template <typename T, int VW>
__device__ __forceinline__ Raw16 load16(const T* __restrict__ row, int64_t k, int64_t K) {
  alignas(16) T v[16];
  if (k + 16 <= K) {
#pragma unroll
    for (int i = 0; i < 16; i += VW) {
      if constexpr (VW == 8) *reinterpret_cast<uint4*>(v + i) = __ldg(reinterpret_cast<const uint4*>(row + k + i));
      else if constexpr (VW == 4) *reinterpret_cast<uint2*>(v + i) = __ldg(reinterpret_cast<const uint2*>(row + k + i));
      else if constexpr (VW == 2) *reinterpret_cast<uint32_t*>(v + i) = __ldg(reinterpret_cast<const uint32_t*>(row + k + i));
      else v[i] = row[k + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = k + i < K ? row[k + i] : from_f32<T>(0.0f);
  }
  return Raw16{*reinterpret_cast<const uint4*>(v), *reinterpret_cast<const uint4*>(v + 8)};
}

template <typename T>
__device__ __forceinline__ uint32_t raw_max(const Raw16& r) {
  return pattern_bits<T>(max(pattern_max(r.lo), pattern_max(r.hi)));
}

// GROUP threads per row. KEEP: chunks of a row that each thread holds in registers (0: the
// row is read a second time, for longer ones). Rows [M, pad_rows) only get zero scales. early:
// the next kernel may start at once, where that is the GEMM of these rows, which sets itself up meanwhile.
// Other kernels only take room from this one (1024 x 12288 mxfp4 back to back 7.7 us, with it 10.1).
template <typename T, int FMT, int VW, int GROUP, int KEEP>
__global__ void __launch_bounds__(GROUP < 128 ? 128 : GROUP) quant_rows(const T* __restrict__ x, int64_t M, int64_t K,
                                                                        int64_t pad_rows, uint8_t* __restrict__ q,
                                                                        uint8_t* __restrict__ sf,
                                                                        float* __restrict__ row_scale, bool early) {
  constexpr int kThreads = GROUP < 128 ? 128 : GROUP;
  constexpr int kLanes = Fmt<FMT>::kBlock / 16;  // threads that share a block
  constexpr int kWordLanes = 4 * kLanes;         // threads that share a cell of four scales
  __shared__ uint32_t red[kThreads / 32];
  if (early) pdl_launch_dependents();
  pdl_wait();
  const int g = threadIdx.x / GROUP, t = threadIdx.x % GROUP, lane = threadIdx.x & 31;
  const int64_t tiles = k_tiles(FMT, K);
  const int chunks = static_cast<int>(tiles * kWordLanes);  // with the last cell's zero scales
  const int code_chunks = static_cast<int>(padded_k(K) / 16);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (kThreads / GROUP);
  const Raw16 zero{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  // a CTA's groups take the same number of rounds (they meet at barriers)
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kThreads / GROUP); row0 < pad_rows; row0 += stride) {
    const int64_t row = row0 + g;
    const bool real = row < M;
    const T* xr = x + row * K;
    uint2* qr = reinterpret_cast<uint2*>(q + row * (padded_k(K) / 2));
    uint8_t* sr = sf + (row >> 7) * tiles * 512 + row_byte(static_cast<int>(row & 127));
    int row_exp = 0;
    Raw16 kept[KEEP > 0 ? KEEP : 1];
    uint32_t tops[KEEP > 0 ? KEEP : 1];
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        kept[i] = real ? load16<T, VW>(xr, static_cast<int64_t>(t + i * GROUP) * 16, K) : zero;
#pragma unroll
      for (int i = 0; i < KEEP; ++i) tops[i] = raw_max<T>(kept[i]);
    }
    if constexpr (FMT == FNI8_NVFP4) {
      // the row's largest finite block: a block with an infinity or NaN stands for itself alone
      uint32_t top = 0;
      auto enter = [&](uint32_t m) {
        if (m < kInfBits) top = max(top, m);
      };
      if constexpr (KEEP > 0) {
#pragma unroll
        for (int i = 0; i < KEEP; ++i) enter(tops[i]);
      } else {
#pragma unroll 2
        for (int c0 = 0; c0 < chunks; c0 += GROUP)
          enter(raw_max<T>(real ? load16<T, VW>(xr, static_cast<int64_t>(c0 + t) * 16, K) : zero));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if constexpr (GROUP > 32) {
        __syncthreads();  // the previous row's maxima are read
        if (lane == 0) red[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < GROUP / 32; ++w) top = max(top, red[w]);
      }
      row_exp = row_exponent(top);
      if (real && t == 0) row_scale[row] = pow2f(row_exp);
    }
    auto emit = [&](int c, const Raw16& r, uint32_t top) {
      if constexpr (kLanes == 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      const BlockScale<FMT> scale(top, row_exp);
      const uint32_t lo = scale.template codes<T>(r.lo), hi = scale.template codes<T>(r.hi);
      // the cell's four scale bytes, from its blocks' lanes
      uint32_t word = real ? scale.byte << (8 * ((lane / kLanes) & 3)) : 0u;
#pragma unroll
      for (int o = kLanes; o < kWordLanes; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
      if (real && c < code_chunks) qr[c] = make_uint2(lo, hi);
      if (row < pad_rows && c < chunks && (lane & (kWordLanes - 1)) == 0)
        *reinterpret_cast<uint32_t*>(sr + static_cast<int64_t>(c / kWordLanes) * 512) = word;
    };
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (i * GROUP < chunks) emit(t + i * GROUP, kept[i], tops[i]);
    } else {
#pragma unroll 2
      for (int c0 = 0; c0 < chunks; c0 += GROUP) {
        const Raw16 r = real ? load16<T, VW>(xr, static_cast<int64_t>(c0 + t) * 16, K) : zero;
        emit(c0 + t, r, raw_max<T>(r));
      }
    }
  }
}

// Eight values per thread and step: their codes (4 bytes), the block's scale byte, stores of VB
// bytes (the largest power of two up to 16 that the output rows' alignment allows). Bound:
// HBM, 1/2 + 1/g bytes read and the output written per value.
template <typename T, int FMT, int VB>
__global__ void __launch_bounds__(256) dequant_rows(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sf,
                                                    const float* __restrict__ row_scale, int64_t M, int64_t K,
                                                    T* __restrict__ out) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kChunks = Fmt<FMT>::kBlock / 8;  // threads that share a block
  const int64_t tiles = k_tiles(FMT, K), row_bytes = padded_k(K) / 2;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; row < M;
       row += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    const float rs = FMT == FNI8_NVFP4 ? __ldg(row_scale + row) : 1.0f;
    const uint8_t* sr = sf + (row >> 7) * tiles * 512 + row_byte(static_cast<int>(row & 127));
    // of this thread's steps, `blockDim.x` (a power of two >= 32) chunks apart
    const uint32_t* qp = reinterpret_cast<const uint32_t*>(q + row * row_bytes) + threadIdx.x;
    const int s0 = threadIdx.x / kChunks;  // its block of the row
    const uint8_t* sp = sr + (s0 >> 2) * 512 + (s0 & 3);
    const int s_step = blockDim.x / (4 * kChunks) * 512;
    T* o = out + row * K + threadIdx.x * 8;
    auto step = [&](int c, auto whole) {
      uint32_t h[4];
      e2m1x8_values(__ldg(qp), h);
      const uint32_t sb = __ldg(sp);
      Pair sc;
      if constexpr (FMT == FNI8_MXFP4) {
        const float f = sb == 0xFF ? __uint_as_float(0x7FC00000u) : pow2f(static_cast<int>(sb) - 127);
        sc = pair(f, f);
      } else {  // code * scale is exact in halves: 2 + 4 significant bits, between 2^-10 and 2688
        const __half2 s2 = __half2half2(__float2half_rn(e4m3_value(sb)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), s2);
          h[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
        sc = pair(rs, rs);
      }
      alignas(16) T v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        float lo, hi;
        unpair(mul2(pair(f.x, f.y), sc), lo, hi);
        if constexpr (sizeof(T) == 4) {
          v[2 * i] = lo;
          v[2 * i + 1] = hi;
        } else if constexpr (std::is_same<T, __half>::value) {
          *reinterpret_cast<__half2*>(v + 2 * i) = __floats2half2_rn(lo, hi);
        } else {
          *reinterpret_cast<__nv_bfloat162*>(v + 2 * i) = __floats2bfloat162_rn(lo, hi);
        }
      }
      if constexpr (decltype(whole)::value) {
        char* ob = reinterpret_cast<char*>(o);
        const char* vb = reinterpret_cast<const char*>(v);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(v)); i += VB) {
          if constexpr (VB == 16) *reinterpret_cast<uint4*>(ob + i) = *reinterpret_cast<const uint4*>(vb + i);
          else if constexpr (VB == 8) *reinterpret_cast<uint2*>(ob + i) = *reinterpret_cast<const uint2*>(vb + i);
          else if constexpr (VB == 4) *reinterpret_cast<uint32_t*>(ob + i) = *reinterpret_cast<const uint32_t*>(vb + i);
          else *reinterpret_cast<uint16_t*>(ob + i) = *reinterpret_cast<const uint16_t*>(vb + i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c * 8 + i < K) o[i] = v[i];
      }
      qp += blockDim.x;
      sp += s_step;
      o += blockDim.x * 8;
    };
    int c = threadIdx.x;
#pragma unroll 4
    for (; c < K >> 3; c += blockDim.x) step(c, std::true_type{});
    if (c * 8 < K) step(c, std::false_type{});
  }
}

}  // namespace fp4
}  // namespace fni8b

using namespace fni8b;
using namespace fni8h;

namespace {

int check_fp4_rows(int format, int64_t M, int64_t K, const char* what) {
  if (format != FNI8_MXFP4 && format != FNI8_NVFP4)
    return fail(FNI8_ERR_INVALID, "%s: format %d: expected MXFP4 or NVFP4", what, format);
  if (M < 0 || K <= 0) return fail(FNI8_ERR_INVALID, "%s: bad size M=%lld K=%lld", what, (long long)M, (long long)K);
  if (M >= (1LL << 31) || K >= (1LL << 31)) return fail(FNI8_ERR_UNSUPPORTED, "%s: sizes must be < 2^31", what);
  return FNI8_OK;
}

template <typename T, int FMT, int VW>
void launch_quant(const T* x, int64_t M, int64_t K, int64_t pad_rows, bool early, uint8_t* q, uint8_t* sf, float* rs,
                  cudaStream_t st) {
  const int64_t chunks = fp4::k_tiles(FMT, K) * 4 * (fp4::Fmt<FMT>::kBlock / 16);
  const int64_t blocks = chunks <= 64 ? (pad_rows + 3) / 4 : pad_rows;
  // four to ten waves; an nvfp4 row's barriers like CTAs that go on to a next row (8192 x 4096
  // 21.3 -> 18.4 us), mxfp4 rows do not (24576 x 4096 45.5 -> 46.6)
  const int64_t cap = 148 * (FMT == FNI8_NVFP4 ? 24 : 64);
  const dim3 grid((unsigned)(blocks < cap ? blocks : cap));
#define FNI8_QUANT_FP4(G, KEEP)                                                                                     \
  launch_pdl(fp4::quant_rows<T, FMT, VW, G, KEEP>, grid, dim3(G < 128 ? 128 : G), 0, st, x, M, K, pad_rows, q, sf, rs, early)
  // few long rows: more threads to each (1 x 12288 nvfp4 2.9 us with 512, 7.7 with 128)
  const bool few = M < 4 * 148;
  if constexpr (FMT == FNI8_MXFP4) {  // no row maximum: nothing to keep
    if (chunks <= 64) FNI8_QUANT_FP4(32, 0);
    else if (few && chunks > 256) FNI8_QUANT_FP4(512, 0);
    else FNI8_QUANT_FP4(128, 0);
  } else {
    if (chunks <= 32) FNI8_QUANT_FP4(32, 1);
    else if (chunks <= 64) FNI8_QUANT_FP4(32, 2);
    else if (chunks <= 128) FNI8_QUANT_FP4(128, 1);
    else if (chunks <= 256) FNI8_QUANT_FP4(128, 2);
    else if (few && chunks <= 1024) FNI8_QUANT_FP4(512, 2);
    else if (chunks <= 512) FNI8_QUANT_FP4(256, 2);
    else if (chunks <= 1024) FNI8_QUANT_FP4(256, 4);
    else FNI8_QUANT_FP4(512, 0);
  }
#undef FNI8_QUANT_FP4
}

template <typename T, int FMT>
void launch_quant_vw(const void* x, int64_t M, int64_t K, int64_t pad_rows, bool early, uint8_t* q, uint8_t* sf, float* rs,
                     cudaStream_t st) {
  const T* xt = static_cast<const T*>(x);
  const uintptr_t a = reinterpret_cast<uintptr_t>(x) | (M > 1 ? static_cast<uintptr_t>(K) * 2 : 0);
  if (a % 16 == 0) launch_quant<T, FMT, 8>(xt, M, K, pad_rows, early, q, sf, rs, st);
  else if (a % 8 == 0) launch_quant<T, FMT, 4>(xt, M, K, pad_rows, early, q, sf, rs, st);
  else if (a % 4 == 0) launch_quant<T, FMT, 2>(xt, M, K, pad_rows, early, q, sf, rs, st);
  else launch_quant<T, FMT, 1>(xt, M, K, pad_rows, early, q, sf, rs, st);
}

}  // namespace

namespace fni8h {

int fp4_quantize(const void* x, int dtype, int format, int64_t M, int64_t K, bool pad, uint8_t* q, uint8_t* sf,
                 float* row_scale, cudaStream_t st) {
  const int64_t pad_rows = pad ? fp4::row_tiles(M) * 128 : M;
  if (format == FNI8_MXFP4) {
    if (dtype == FNI8_F16) launch_quant_vw<__half, FNI8_MXFP4>(x, M, K, pad_rows, !pad, q, sf, row_scale, st);
    else launch_quant_vw<__nv_bfloat16, FNI8_MXFP4>(x, M, K, pad_rows, !pad, q, sf, row_scale, st);
  } else {
    if (dtype == FNI8_F16) launch_quant_vw<__half, FNI8_NVFP4>(x, M, K, pad_rows, !pad, q, sf, row_scale, st);
    else launch_quant_vw<__nv_bfloat16, FNI8_NVFP4>(x, M, K, pad_rows, !pad, q, sf, row_scale, st);
  }
  FNI8_CHECK_LAUNCH("quantize_rows_fp4");
  return FNI8_OK;
}

int fp4_check_rows(const void* x, int dtype, int format, int64_t M, int64_t K, const uint8_t* q, const uint8_t* sf,
                   const float* row_scale) {
  if (dtype != FNI8_F16 && dtype != FNI8_BF16) return fail(FNI8_ERR_INVALID, "dtype %d: expected F16 or BF16", dtype);
  if (int s = check_fp4_rows(format, M, K, "quantize_rows_fp4")) return s;
  if (M == 0) return FNI8_OK;
  if (!x || !q || !sf || (format == FNI8_NVFP4 && !row_scale))
    return fail(FNI8_ERR_INVALID, "quantize_rows_fp4: null pointer");
  if (reinterpret_cast<uintptr_t>(x) & 1u) return fail(FNI8_ERR_ALIGN, "quantize_rows_fp4: x must be 2-byte aligned");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(sf)) & 15u)
    return fail(FNI8_ERR_ALIGN, "quantize_rows_fp4: q and sf must be 16-byte aligned");
  return FNI8_OK;
}

}  // namespace fni8h

extern "C" size_t fni8_fp4_scale_bytes(int format, int64_t M, int64_t K) {
  if ((format != FNI8_MXFP4 && format != FNI8_NVFP4) || M <= 0 || K <= 0) return 0;
  return static_cast<size_t>(fp4::row_tiles(M) * fp4::k_tiles(format, K)) * 512;
}

extern "C" int fni8_quantize_rows_fp4(const void* x, int dtype, int format, int64_t M, int64_t K, uint8_t* q,
                                      uint8_t* sf, float* row_scale, void* stream) {
  if (int s = fp4_check_rows(x, dtype, format, M, K, q, sf, row_scale)) return s;
  if (M == 0) return FNI8_OK;
  return fp4_quantize(x, dtype, format, M, K, true, q, sf, row_scale, static_cast<cudaStream_t>(stream));
}

extern "C" int fni8_dequantize_rows_fp4(const uint8_t* q, const uint8_t* sf, const float* row_scale, int format,
                                        int64_t M, int64_t K, void* out, int out_dtype, void* stream) {
  if (out_dtype != FNI8_F16 && out_dtype != FNI8_BF16 && out_dtype != FNI8_F32)
    return fail(FNI8_ERR_INVALID, "dequantize_rows_fp4: out_dtype %d", out_dtype);
  if (int s = check_fp4_rows(format, M, K, "dequantize_rows_fp4")) return s;
  if (M == 0) return FNI8_OK;
  if (!q || !sf || !out || (format == FNI8_NVFP4 && !row_scale))
    return fail(FNI8_ERR_INVALID, "dequantize_rows_fp4: null pointer");
  if (reinterpret_cast<uintptr_t>(q) & 3u) return fail(FNI8_ERR_ALIGN, "dequantize_rows_fp4: q must be 4-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int esz = out_dtype == FNI8_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(out) % esz != 0) return fail(FNI8_ERR_ALIGN, "dequantize_rows_fp4: misaligned out");
  const uintptr_t a = reinterpret_cast<uintptr_t>(out) | (M > 1 ? static_cast<uintptr_t>(K) * esz : 0);
  const int64_t per_row = (K + 7) / 8;
  // four steps of a row to a thread, so that their loads are in flight together, and 256
  // threads to a CTA
  int threads = 32;
  while (threads < 256 && threads * 4 < per_row) threads *= 2;
  const int rows = 256 / threads;
  const int64_t ctas = (M + rows - 1) / rows;
  const dim3 grid((unsigned)(ctas < 148 * 64 ? ctas : 148 * 64)), block(threads, rows);
#define FNI8_DEQUANT_FP4(T, FMT, VB) \
  launch_pdl(fp4::dequant_rows<T, FMT, VB>, grid, block, 0, st, q, sf, row_scale, M, K, static_cast<T*>(out))
#define FNI8_DEQUANT_VB(T, FMT)                          \
  do {                                                   \
    if (a % 16 == 0) FNI8_DEQUANT_FP4(T, FMT, 16);       \
    else if (a % 8 == 0) FNI8_DEQUANT_FP4(T, FMT, 8);    \
    else if (a % 4 == 0) FNI8_DEQUANT_FP4(T, FMT, 4);    \
    else FNI8_DEQUANT_FP4(T, FMT, 2);                    \
  } while (0)
  if (format == FNI8_MXFP4) {
    if (out_dtype == FNI8_F16) FNI8_DEQUANT_VB(__half, FNI8_MXFP4);
    else if (out_dtype == FNI8_BF16) FNI8_DEQUANT_VB(__nv_bfloat16, FNI8_MXFP4);
    else FNI8_DEQUANT_VB(float, FNI8_MXFP4);
  } else {
    if (out_dtype == FNI8_F16) FNI8_DEQUANT_VB(__half, FNI8_NVFP4);
    else if (out_dtype == FNI8_BF16) FNI8_DEQUANT_VB(__nv_bfloat16, FNI8_NVFP4);
    else FNI8_DEQUANT_VB(float, FNI8_NVFP4);
  }
#undef FNI8_DEQUANT_VB
#undef FNI8_DEQUANT_FP4
  FNI8_CHECK_LAUNCH("dequantize_rows_fp4");
  return FNI8_OK;
}
