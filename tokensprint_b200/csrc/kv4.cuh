// The 4-bit cache: how its rows lie in memory and how they become numbers again.
//
// A pool of pages is a uint8 array [pages][kv heads][page size / 16][18 D].  The last dimension is the
// record of 16 tokens of one head, contiguous and on a 16-byte boundary:
//
//   key codes     16 rows of D/2 bytes    channel c in the low (c even) or high half of byte c/2
//   key scales    16 rows of D/16 bytes   one byte for 16 channels
//   value codes   16 rows of D/2 bytes
//   value scales  16 rows of D/16 bytes
//
// A value is (code - 8) * s.  The scale byte holds 5 bits of exponent and 3 of mantissa, no sign: it is
// the upper byte but for the sign of a half, so that (byte << 7) read as a half IS the scale.  The code
// has three bits and a sign, the scale four significant bits: their product has seven and is exact in half and in
// bfloat16.  Storing: s = amax / 7 rounded to the nearest such number (ties to even mantissa, at most
// 8192), code = 8 + round(x / s) between 1 and 15.  NaN is stored as 0, infinities as +-7 * 8192: no row
// makes an attention over it anything but finite.
#pragma once

#include "common.cuh"

#define KV4_BLOCK 16  // tokens of a record; channels of a group

template <int D>
struct Kv4Record {
  static constexpr int kRow = D / 2;           // bytes of one row's codes
  static constexpr int kScales = D / 16;       // bytes of one row's scales
  static constexpr int kKeyScales = 8 * D;     // offsets within the record
  static constexpr int kValues = 9 * D;
  static constexpr int kValueScales = 17 * D;
  static constexpr int kBytes = 18 * D;
};

// Two codes that stand at bits 3..6 and 19..22 of `x`, minus 8, times the scales, in bfloat16: 0x3f80 | code << 3 is
// 1 + code / 16, and with f = 16 s and c = -24 s one multiply-add gives (code - 8) s; all of it is exact.
__device__ __forceinline__ uint32_t kv4_pair(uint32_t x, __nv_bfloat162 f, __nv_bfloat162 c) {
  uint32_t h;
  asm("lop3.b32 %0, %1, 0x00780078, 0x3f803f80, 0xea;" : "=r"(h) : "r"(x));  // (x & mask) | one
  __nv_bfloat162 v = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&h), f, c);
  return *reinterpret_cast<uint32_t*>(&v);
}

// f and c of two scale bytes a, b.  A scale byte at the mantissa's top and the exponent's end of a bfloat16 is its
// number times 2^-112, small exponents (subnormal there as here) included.
__device__ __forceinline__ void kv4_factors(uint32_t a, uint32_t b, __nv_bfloat162& f, __nv_bfloat162& c) {
  const uint32_t u = (a << 4) | (b << 20);
  const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&u);
  f = __hmul2(v, __float2bfloat162_rn(8.307674973655724e+34f));    // 2^116
  c = __hmul2(v, __float2bfloat162_rn(-1.2461512460483586e+35f));  // -1.5 * 2^116
}

// Eight codes with their scale as values: bfloat16 in order.
__device__ __forceinline__ uint4 kv4_unpack(uint32_t x, uint32_t scale) {
  __nv_bfloat162 f, c;
  kv4_factors(scale, scale, f, c);
  const uint32_t p0 = kv4_pair(x << 3, f, c), p1 = kv4_pair(x >> 1, f, c), p2 = kv4_pair(x >> 5, f, c), p3 = kv4_pair(x >> 9, f, c);
  return make_uint4(__byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632), __byte_perm(p2, p3, 0x7632));
}

// D (float32) += A (bfloat16, 16 x 16, row major) * B (bfloat16, 16 x 8).
__device__ __forceinline__ void kv4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float kv4_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// kParts bfloat16 pairs whose sum is (a, b) up to 2^(-8 kParts - 1) of it.
template <int kParts>
__device__ __forceinline__ void kv4_split(float a, float b, uint32_t (&out)[kParts]) {
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    out[i] = *reinterpret_cast<const uint32_t*>(&v);
    if (i + 1 < kParts) {
      a -= __uint_as_float(out[i] << 16);
      b -= __uint_as_float(out[i] & 0xffff0000u);
    }
  }
}

// One query row as the MMA's B operand.  Lane (g, t) = (lane / 4, lane % 4) holds of row g the channels
// [t D/4, (t+1) D/4), in the order in which the keys' words give theirs: word w of 8 channels feeds the k-steps 2w
// with the pairs (0,4) (1,5) and 2w+1 with (2,6) (3,7).  A bfloat16 row is one part, a float32 row three.
// `p`: the lane's channels, on a 16-byte boundary, or null for a row of zeros.
template <int D, int kParts>
__device__ __forceinline__ void kv4_query_row(const __nv_bfloat16* p, uint32_t (&frag)[kParts][D / 16][2]) {
  static_assert(kParts == 1, "bfloat16 rows are one part");
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    const uint4 v = p != nullptr ? reinterpret_cast<const uint4*>(p)[w] : make_uint4(0u, 0u, 0u, 0u);
    frag[0][2 * w][0] = __byte_perm(v.x, v.z, 0x5410);
    frag[0][2 * w][1] = __byte_perm(v.x, v.z, 0x7632);
    frag[0][2 * w + 1][0] = __byte_perm(v.y, v.w, 0x5410);
    frag[0][2 * w + 1][1] = __byte_perm(v.y, v.w, 0x7632);
  }
}
template <int D, int kParts>
__device__ __forceinline__ void kv4_query_row(const float* p, uint32_t (&frag)[kParts][D / 16][2]) {
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 a = p != nullptr ? reinterpret_cast<const float4*>(p)[2 * w] : zero, b = p != nullptr ? reinterpret_cast<const float4*>(p)[2 * w + 1] : zero;
    const float lo[4] = {a.x, a.y, a.z, a.w}, hi[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t out[kParts];
      kv4_split<kParts>(lo[j], hi[j], out);
#pragma unroll
      for (int i = 0; i < kParts; ++i) frag[i][2 * w + j / 2][j % 2] = out[i];
    }
  }
}

// Keys 16 x D of a record times query rows: S[token][row] of tiles of 8 rows.  Lane (g, t) has of the rows g and g + 8 the words of a quarter of
// their channels and those channels' scale bytes.  `q(tile, part, word)` gives the lane's four registers of a query tile for the word's
// two k-steps.
template <int D, int kTiles, int kParts, typename Query>
__device__ __forceinline__ void kv4_scores_of(const uint32_t (&w)[2][D / 32], const uint32_t (&sc)[2], Query q, float (&s)[kTiles][4]) {
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; i += 2) {  // 16 channels: one group
    __nv_bfloat162 f[2], c[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) kv4_factors((sc[r] >> (4 * i)) & 0xffu, (sc[r] >> (4 * i)) & 0xffu, f[r], c[r]);
#pragma unroll
    for (int k = i; k < i + 2; ++k) {
      const uint32_t a00 = kv4_pair(w[0][k] << 3, f[0], c[0]), a01 = kv4_pair(w[1][k] << 3, f[1], c[1]);
      const uint32_t a02 = kv4_pair(w[0][k] >> 1, f[0], c[0]), a03 = kv4_pair(w[1][k] >> 1, f[1], c[1]);
      const uint32_t a10 = kv4_pair(w[0][k] >> 5, f[0], c[0]), a11 = kv4_pair(w[1][k] >> 5, f[1], c[1]);
      const uint32_t a12 = kv4_pair(w[0][k] >> 9, f[0], c[0]), a13 = kv4_pair(w[1][k] >> 9, f[1], c[1]);
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          const uint4 b = q(n, part, k);
          kv4_mma(s[n], a00, a01, a02, a03, b.x, b.y);
          kv4_mma(s[n], a10, a11, a12, a13, b.z, b.w);
        }
    }
  }
}

// The same from where the record's key codes and scales lie.
template <int D, int kTiles, int kParts, typename Query>
__device__ __forceinline__ void kv4_scores(const uint8_t* codes, const uint8_t* scales, Query q, float (&s)[kTiles][4], int g, int t) {
  constexpr int kWords = D / 32;  // of 8 codes, per lane and row
  uint32_t w[2][kWords], sc[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint8_t* p = codes + (g + 8 * r) * (D / 2) + t * (D / 8);
    const uint8_t* ps = scales + (g + 8 * r) * (D / 16) + t * (D / 64);
    if constexpr (kWords == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[r][0] = v.x, w[r][1] = v.y;
      sc[r] = *ps;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
        w[r][i] = v.x, w[r][i + 1] = v.y, w[r][i + 2] = v.z, w[r][i + 3] = v.w;
      }
      if constexpr (kWords == 4) sc[r] = *reinterpret_cast<const uint16_t*>(ps);
      else sc[r] = *reinterpret_cast<const uint32_t*>(ps);
    }
  }
  kv4_scores_of<D, kTiles, kParts>(w, sc, q, s);
}
