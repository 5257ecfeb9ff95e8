// Matrices of microscaled 4-bit floats: layout, scales, and the checks of the entry points (see cr_mx4).
#pragma once
#include "common.cuh"

namespace cr {

// Offset of the scale byte of (row, block) in tiles of 128 rows x 4 blocks; groups = ceil(inner / 128).
__host__ __device__ __forceinline__ size_t mx4_scale_at(int row, int block, int groups) {
  return ((size_t)(row >> 7) * groups + (block >> 2)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (block & 3);
}
__host__ __device__ __forceinline__ int mx4_groups(int inner) { return (inner + 127) >> 7; }

// 2^(b - 127) of an e8m0 byte: the byte is the exponent field, but for 0 (a subnormal number) and 255 (NaN).
__device__ __forceinline__ float e8m0(uint32_t b) {
  return __uint_as_float(b == 0 ? 0x00400000u : (b == 255 ? 0x7fc00000u : b << 23));
}

// The largest magnitude of eight numbers as bits, three at a time; a NaN is above infinity.
__device__ __forceinline__ uint32_t largest8(const float (&v)[8]) {
  uint32_t m[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) m[k] = __float_as_uint(v[k]) & 0x7fffffffu;
  const uint32_t a = __vimax3_u32(m[0], m[1], m[2]), b = __vimax3_u32(m[3], m[4], m[5]);
  return __vimax3_u32(__vimax3_u32(a, b, m[6]), m[7], 0u);
}

// Eight numbers times `by` as e2m1 codes: nearest, ties to even, 6 at most.
__device__ __forceinline__ uint32_t pack_e2m1(const float (&v)[8], float by) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0] * by), "f"(v[1] * by), "f"(v[2] * by), "f"(v[3] * by), "f"(v[4] * by), "f"(v[5] * by), "f"(v[6] * by), "f"(v[7] * by));
  return r;
}

// Eight consecutive elements of a row buffer as floats.  `wide`: the address is a multiple of 16 bytes.
template <int TYPE>
__device__ __forceinline__ void load_row8(const void* p, size_t i, bool wide, float (&v)[8]) {
  if constexpr (TYPE == CR_ROW_F32) {
    const float* f = reinterpret_cast<const float*>(p) + i;
    if (wide) {
      const float4 a = *reinterpret_cast<const float4*>(f), b = *reinterpret_cast<const float4*>(f + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = f[k];
    }
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + i;
    uint32_t u[4];
    if (wide) {
      const uint4 a = *reinterpret_cast<const uint4*>(h);
      u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = (uint32_t)h[2 * k] | ((uint32_t)h[2 * k + 1] << 16);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (TYPE == CR_ROW_BF16) {
        v[2 * k] = __uint_as_float(u[k] << 16);
        v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
        v[2 * k] = f.x; v[2 * k + 1] = f.y;
      }
    }
  }
}

inline cr_status check_mx4(const cr_mx4* m, const char* who, const char* what) {
  CR_REQUIRE(m && m->codes && m->scales, "%s: null %s", who, what);
  CR_REQUIRE(m->rows >= 1 && m->rows < (1 << 24) && m->inner >= 64 && m->inner % 64 == 0 && m->inner < (1 << 24),
             "%s: %s of %d x %d: at least one row, inner a multiple of 64, both below 2^24", who, what, m->rows, m->inner);
  CR_REQUIRE(((uintptr_t)m->codes & 15) == 0 && ((uintptr_t)m->scales & 15) == 0, "%s: %s must be 16-byte aligned", who, what);
  return CR_OK;
}
inline cr_status check_rows(const void* x, int dtype, long long ld, int inner, const char* who) {
  CR_REQUIRE(x, "%s: null rows", who);
  CR_REQUIRE(dtype == CR_ROW_F32 || dtype == CR_ROW_BF16 || dtype == CR_ROW_F16, "%s: unknown element type %d", who, dtype);
  CR_REQUIRE(((uintptr_t)x & (dtype == CR_ROW_F32 ? 3 : 1)) == 0, "%s: rows off the alignment of their type", who);
  CR_REQUIRE(ld >= inner, "%s: row pitch %lld below the %d elements of a row", who, ld, inner);
  return CR_OK;
}
// Whether eight elements from a multiple of eight on can be read or written 16 bytes at a time.
inline bool wide_rows(const void* p, int dtype, long long ld) { return ((uintptr_t)p & 15) == 0 && ld * (dtype == CR_ROW_F32 ? 4 : 2) % 16 == 0; }
// Calls f with an integral constant of the element type.
template <typename F>
inline cr_status by_dtype(int dtype, F&& f) {
  if (dtype == CR_ROW_F32) return f(std::integral_constant<int, CR_ROW_F32>());
  if (dtype == CR_ROW_BF16) return f(std::integral_constant<int, CR_ROW_BF16>());
  return f(std::integral_constant<int, CR_ROW_F16>());
}

}  // namespace cr
