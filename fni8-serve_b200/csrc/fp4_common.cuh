// 4-bit floating point (e2m1) with block scales: the layout shared by the row kernels
// (fp4.cu) and the block-scaled GEMMs (gemm_fp4.cu, gemm_fp4_splitk.cu).
//
//   FNI8_MXFP4  one e8m0 scale (a power of two) for every 32 values
//   FNI8_NVFP4  one e4m3 scale for every 16 values, and one fp32 scale for each row
//
// Codes: two to a byte, the even element in the low half, rows of Kp / 2 bytes with
// Kp = K rounded up to 32 (zero codes behind K). Scales: tiles of 128 rows x 4 scales, 512
// bytes each, tile (r / 128, s / 4) at index (r / 128) * ceil(S / 4) + s / 4, where row r
// and scale s are at byte (r % 32) * 16 + (r % 128 / 32) * 4 + s % 4: the order in which
// tcgen05.cp.32x128b.warpx4 brings a tile into tensor memory, four scales of a row in one
// 32-bit cell. Scales behind K are zero, so the padded part of a tile adds nothing.
#pragma once
#include <type_traits>

#include "fni8_common.cuh"

namespace fni8b {
namespace fp4 {

template <int FMT>
struct Fmt;
template <>
struct Fmt<FNI8_MXFP4> {
  static constexpr int kBlock = 32;
  static constexpr int kStageTiles = 2;  // scale tiles of a 256-value (128-byte) stage
};
template <>
struct Fmt<FNI8_NVFP4> {
  static constexpr int kBlock = 16;
  static constexpr int kStageTiles = 4;
};

__host__ __device__ __forceinline__ int64_t padded_k(int64_t K) { return (K + 31) / 32 * 32; }
// scale tiles along K
__host__ __device__ __forceinline__ int64_t k_tiles(int fmt, int64_t K) {
  return fmt == FNI8_MXFP4 ? (K + 127) / 128 : (K + 63) / 64;
}
__host__ __device__ __forceinline__ int64_t row_tiles(int64_t M) { return (M + 127) / 128; }
// byte of row r within its column of tiles (add tile * 512 and s % 4)
__device__ __forceinline__ int row_byte(int r) { return (r & 31) * 16 + ((r & 127) >> 5) * 4; }

// Instruction descriptor of tcgen05.mma kind::mxf4 / kind::mxf4nvf4: A = B = e2m1, both
// K-major, dense, K = 64, shape M x N; sf_id: which two of a cell's four scales (0 or 2)
// an mxfp4 step takes (nvfp4 takes all four, sf_id 0).
__host__ __device__ constexpr uint32_t idesc_fp4(int fmt, int M, int N, int sf_id) {
  return (static_cast<uint32_t>(sf_id) << 4)                      // B scales
         | (1u << 7) | (1u << 10)                                 // A, B: e2m1
         | (static_cast<uint32_t>(N >> 3) << 17)                  // N / 8
         | ((fmt == FNI8_MXFP4 ? 1u : 0u) << 23)                  // scales: e8m0 (1) or e4m3 (0)
         | (static_cast<uint32_t>(M >> 7) << 27)                  // M / 128
         | (static_cast<uint32_t>(sf_id) << 29);                  // A scales
}

// Shared-memory descriptor of one 512-byte scale tile for tcgen05.cp: 32 rows of 16 bytes,
// no swizzle, 128 bytes from one group of 8 rows to the next.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128u >> 4) << 32) |
         (static_cast<uint64_t>(1u) << 46);
}

template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D[tmem] (+)= (A * SFA)[smem] * (B * SFB)[smem]^T over 64 values of K, issued by one thread.
#define FNI8_MMA_FP4(GROUP, KIND, VEC)                                                             \
  asm volatile(                                                                                    \
      "{\n\t.reg .pred p;\n\t"                                                                     \
      "setp.ne.b32 p, %6, 0;\n\t"                                                                  \
      "tcgen05.mma.cta_group::" GROUP ".kind::" KIND ".block_scale.scale_vec::" VEC                \
      " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),                                           \
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                      \
      : "memory")
template <int FMT, bool PAIR>
__device__ __forceinline__ void umma_fp4(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                         uint32_t sfb, uint32_t accumulate) {
  if constexpr (FMT == FNI8_MXFP4) {
    if constexpr (PAIR) FNI8_MMA_FP4("2", "mxf4", "2X");
    else FNI8_MMA_FP4("1", "mxf4", "2X");
  } else {
    if constexpr (PAIR) FNI8_MMA_FP4("2", "mxf4nvf4", "4X");
    else FNI8_MMA_FP4("1", "mxf4nvf4", "4X");
  }
}
#undef FNI8_MMA_FP4

// Every PARTS-th (from PART on) of a 256-value stage's scale tiles, from shared memory (sfa;
// sfb, the tiles of B's second 128 rows behind all of the first's) to the tensor-memory columns
// ta and tb. Copies and MMAs of one thread execute in order: a copy needs no wait before the
// MMA that reads it, nor after the one that read its columns before.
template <int FMT, bool PAIR, int N, int PART = 0, int PARTS = 1>
__device__ __forceinline__ void stage_scales(const uint8_t* sfa, const uint8_t* sfb, uint32_t ta, uint32_t tb) {
  constexpr int kTiles = Fmt<FMT>::kStageTiles;
  constexpr int kRowTiles = (N + 127) / 128;  // of B
  const uint64_t da = scale_desc(smem_u32(sfa)), db = scale_desc(smem_u32(sfb));
#pragma unroll
  for (int c = PART; c < kTiles * (1 + kRowTiles); c += PARTS) {
    if (c < kTiles) {
      copy_scales<PAIR>(ta + c * 4, da + static_cast<uint64_t>(c * 512 >> 4));
    } else {
      const int i = (c - kTiles) / kRowTiles, j = (c - kTiles) % kRowTiles;
      copy_scales<PAIR>(tb + (i * kRowTiles + j) * 4, db + static_cast<uint64_t>((j * kTiles + i) * 512 >> 4));
    }
  }
}

// The stage's MMAs: `steps` (1 to 4) of 64 values each. sa, sb: the operands' stage (128-byte
// swizzle).
template <int FMT, bool PAIR, int M, int N>
__device__ __forceinline__ void stage_mmas(uint32_t d, const void* sa, const void* sb, uint32_t ta, uint32_t tb,
                                           int steps, bool first) {
  constexpr int kRowTiles = (N + 127) / 128;
  const uint64_t adesc = sw128_kmajor_desc(smem_u32(sa)), bdesc = sw128_kmajor_desc(smem_u32(sb));
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    if (kk < steps) {
      const int tile = FMT == FNI8_MXFP4 ? kk >> 1 : kk;
      const uint32_t idesc = idesc_fp4(FMT, M, N, FMT == FNI8_MXFP4 ? (kk & 1) * 2 : 0);
      umma_fp4<FMT, PAIR>(d, adesc + static_cast<uint64_t>(kk * 2), bdesc + static_cast<uint64_t>(kk * 2), idesc,
                          ta + static_cast<uint32_t>(tile * 4), tb + static_cast<uint32_t>(tile * kRowTiles * 4),
                          (kk != 0 || !first) ? 1u : 0u);
    }
  }
}

// ---------------------------------------------------------------- quantisation of a chunk
// Largest magnitude of eight 16-bit values as a 16-bit pattern (an infinity or NaN wins): the
// order of the patterns without their signs.
__device__ __forceinline__ uint32_t pattern_max(const uint4& u) {
  const uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu),
                              __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
  return max(m & 0xFFFFu, m >> 16);
}
// ... as the bits of the float
template <typename T>
__device__ __forceinline__ uint32_t pattern_bits(uint32_t pattern) {
  const unsigned short top = static_cast<unsigned short>(pattern);
  return __float_as_uint(to_f32<T>(*reinterpret_cast<const T*>(&top)));
}

// 2^e of a float, e in [-127, 127]
__device__ __forceinline__ float pow2f(int e) {
  return __uint_as_float(e > -127 ? static_cast<uint32_t>(e + 127) << 23 : 0x00400000u);
}

// floor(log2(v)) of a positive float given by its bits
__device__ __forceinline__ int floor_log2(uint32_t bits) {
  const int e = static_cast<int>(bits >> 23);
  return e > 0 ? e - 127 : -118 - __clz(bits);  // denormal: 2^-149 has one bit, 31 leading zeros
}

// Two floats in one register pair: the pair's product and fused multiply-add are one instruction.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void unpair(Pair p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

__device__ __forceinline__ uint32_t e2m1x8(const Pair (&v)[4]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpair(v[i], f[2 * i], f[2 * i + 1]);
  uint32_t out;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(out)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return out;
}

// Eight codes (a register) as halves: exact.
__device__ __forceinline__ void e2m1x8_values(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

__device__ __forceinline__ uint32_t e4m3_bits(float v) {
  uint16_t b;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(0.0f), "f"(v));
  return b & 0xFF;
}
__device__ __forceinline__ float e4m3_value(uint32_t bits) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(bits)));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h2 & 0xFFFF)));
}

constexpr uint32_t kInfBits = 0x7F800000u;

// The scale of a block with the maximum `top` (the bits of a float; an infinity or NaN makes it
// NaN), and what eight values of it need for their codes. nvfp4: row_exp is the exponent of
// the row scale; f / (2^row_exp sf) is formed without dividing by the row scale first, but
// for rows so small that 1 / (2^row_exp sf) might not be a float.
template <int FMT>
struct BlockScale {
  uint32_t byte;
  float inv, d, pre;

  __device__ __forceinline__ BlockScale(uint32_t top, int row_exp) {
    if constexpr (FMT == FNI8_MXFP4) {
      const int e = max(top == 0 ? -127 : floor_log2(top) - 2, -127);
      byte = top >= kInfBits ? 0xFFu : static_cast<uint32_t>(e + 127);
      inv = pow2f(-e);  // e <= 125
    } else {
      // max / 6, corrected like the quotients below
      const float t = __fmul_rn(__uint_as_float(top), pow2f(-row_exp)), sixth = 1.0f / 6.0f;
      const float q = __fmul_rn(t, sixth);
      byte = top >= kInfBits ? 0x7Fu : e4m3_bits(__fmaf_rn(__fmaf_rn(-q, 6.0f, t), sixth, q));
      d = top >= kInfBits ? 0.0f : e4m3_value(byte);  // 2^-9 .. 448, or 0
      float r;
      asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(d));
      inv = d > 0.0f ? r : 0.0f;
      pre = 1.0f;
      if (row_exp < -100) {
        pre = pow2f(-row_exp);
      } else {
        d = __fmul_rn(d, pow2f(row_exp));  // exact, as is the next line
        inv = __fmul_rn(inv, pow2f(-row_exp));
      }
    }
  }

  // The codes of eight 16-bit values f. nvfp4: q = f inv is the quotient but for a few units in
  // the last place; its fused remainder f - q d is exact and corrects it to the quotient's rounding
  // (Markstein's step, as in div_by_ge1). All from -f and -inv: so a zero keeps its sign.
  template <typename T>
  __device__ __forceinline__ uint32_t codes(const uint4& raw) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    const Pair inv2 = pair(-inv, -inv), d2 = pair(d, d);
    Pair v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t n = w[i] ^ 0x80008000u;
      Pair f;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f = pair(__uint_as_float(n << 16), __uint_as_float(n & 0xFFFF0000u));
      } else {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&n));
        f = pair(h.x, h.y);
      }
      if constexpr (FMT == FNI8_NVFP4) {
        if (pre != 1.0f) f = mul2(f, pair(pre, pre));
        const Pair q = mul2(f, inv2);
        v[i] = fma2(fma2(q, d2, f), inv2, q);
      } else {
        v[i] = mul2(f, inv2);
      }
    }
    return e2m1x8(v);
  }
};

// Exponent of an nvfp4 row's scale from the bits of its largest magnitude: the least power of
// two >= top / 2688, 2688 = 1.3125 * 2^11.
__device__ __forceinline__ int row_exponent(uint32_t top) {
  if (top == 0) return -126;
  const int e = floor_log2(top);
  return max(-126, (top >> 23) > 0 && (top & 0x7FFFFFu) > 0x280000u ? e - 10 : e - 11);
}

}  // namespace fp4
}  // namespace fni8b

namespace fni8h {
// The scale tiles as a 2-D map of 128-byte rows (four to a tile); a box is `tiles` of them.
inline int encode_scale_map(CUtensorMap* map, const uint8_t* sf, int fmt, int64_t M, int64_t K, int tiles) {
  const int64_t rows = fni8b::fp4::row_tiles(M) * fni8b::fp4::k_tiles(fmt, K) * 4;
  return encode_tmap_2d_u8(map, sf, 128, (uint64_t)rows, 128, 128, (uint32_t)(tiles * 4));
}
}  // namespace fni8h
