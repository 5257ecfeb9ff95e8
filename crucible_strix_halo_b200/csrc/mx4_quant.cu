// Rows to microscaled 4-bit floats and back (see cr_mx4 for the format).
//   s = clamp(floor(log2 max |x|) - 2, -127, 127),  code = e2m1(x 2^-s), round to nearest even, saturating
// The exponent field of the largest magnitude is floor(log2) + 127 (0 for a subnormal one, whose s is held to -127 either way), and
// x 2^-s is exact: both steps have the definition's own bits.  A thread takes 8 elements, four threads a block.
// HBM-bound: an element's bytes in, 17/32 of a byte out.
#include "mx4.cuh"

namespace cr {

template <int TYPE>
__global__ void __launch_bounds__(256) mx4_quant_kernel(const void* __restrict__ x, long long ld, bool wide, uint8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ scales, int rows, int inner) {
  pdl_release();
  pdl_wait();
  const int per_row = inner / 8, groups = mx4_groups(inner);
  const long long units = (long long)rows * per_row;
  for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256) {
    const int row = (int)(u / per_row), i = (int)(u - (long long)row * per_row);     // units is a multiple of 8: blocks of four threads are whole
    float v[8];
    load_row8<TYPE>(x, (size_t)row * ld + (size_t)i * 8, wide, v);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
    const unsigned four = 0xfu << (threadIdx.x & 28);
    top = max(top, __shfl_xor_sync(four, top, 1));
    top = max(top, __shfl_xor_sync(four, top, 2));
    const int field = (int)(top >> 23);                                              // 255: an infinity or a NaN is among them
    const int s = max(field - 129, -127);
    const uint32_t packed = field == 255 ? 0u : pack_e2m1(v, __uint_as_float((uint32_t)(127 - s) << 23));
    reinterpret_cast<uint32_t*>(codes)[u] = packed;
    if ((threadIdx.x & 3) == 0) scales[mx4_scale_at(row, i >> 2, groups)] = field == 255 ? 255 : (uint8_t)(s + 127);
  }
}

template <int TYPE>
__global__ void __launch_bounds__(256) mx4_dequant_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int inner,
                                                          void* __restrict__ y, long long ld, bool wide) {
  pdl_release();
  pdl_wait();
  const int per_row = inner / 8, groups = mx4_groups(inner);
  const long long units = (long long)rows * per_row;
  for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256) {
    const int row = (int)(u / per_row), i = (int)(u - (long long)row * per_row);
    const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[u];
    const float scale = e8m0(scales[mx4_scale_at(row, i >> 2, groups)]);
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // The low and the high nibble of byte k as fp16 numbers times 2^-14: sign to bit 15, e2m1's other bits to bits 11..9.
      const uint32_t b = (w >> (8 * k)) & 0xffu, h = ((b & 8) << 12 | (b & 7) << 9) | ((b & 0x80) << 24 | (b & 0x70) << 21);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      v[2 * k] = f.x * 16384.f * scale;
      v[2 * k + 1] = f.y * 16384.f * scale;
    }
    const size_t at = (size_t)row * ld + (size_t)i * 8;
    if constexpr (TYPE == CR_ROW_F32) {
      float* p = reinterpret_cast<float*>(y) + at;
      if (wide) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] = v[k];
      }
    } else {
      uint16_t* p = reinterpret_cast<uint16_t*>(y) + at;
      uint32_t o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (TYPE == CR_ROW_BF16) { const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]); o[k] = *reinterpret_cast<const uint32_t*>(&t); }
        else { const __half2 t = __floats2half2_rn(v[2 * k], v[2 * k + 1]); o[k] = *reinterpret_cast<const uint32_t*>(&t); }
      }
      if (wide) *reinterpret_cast<uint4*>(p) = make_uint4(o[0], o[1], o[2], o[3]);
      else {
#pragma unroll
        for (int k = 0; k < 4; ++k) { p[2 * k] = (uint16_t)o[k]; p[2 * k + 1] = (uint16_t)(o[k] >> 16); }
      }
    }
  }
}

static dim3 unit_grid(int rows, int inner) {
  const long long blocks = ((long long)rows * (inner / 8) + 255) / 256, most = (long long)sm_count() * 8;
  return dim3((unsigned)(blocks < most ? blocks : most));
}

}  // namespace cr

extern "C" size_t cr_mx4_code_bytes(int rows, int inner) { return rows < 1 || inner < 1 ? 0 : (size_t)rows * inner / 2; }
extern "C" size_t cr_mx4_scale_bytes(int rows, int inner) {
  return rows < 1 || inner < 1 ? 0 : ((size_t)rows + 127) / 128 * (((size_t)inner + 127) / 128) * 512;
}

extern "C" cr_status cr_mx4_quant(const void* x, cr_row_dtype dtype, long long ld, const cr_mx4* to, void* stream_) {
  using namespace cr;
  if (cr_status s = check_mx4(to, "cr_mx4_quant", "destination")) return s;
  if (cr_status s = check_rows(x, dtype, ld, to->inner, "cr_mx4_quant")) return s;
  cudaStream_t stream = (cudaStream_t)stream_;
  use_stream(stream);
  return by_dtype(dtype, [&](auto type) -> cr_status {
    CR_CUDA(launch_pdl(mx4_quant_kernel<decltype(type)::value>, unit_grid(to->rows, to->inner), dim3(256), 0, stream, x, ld, wide_rows(x, dtype, ld),
                       to->codes, to->scales, to->rows, to->inner));
    CR_LAUNCH_CHECK("mx4_quant_kernel");
    return CR_OK;
  });
}

extern "C" cr_status cr_mx4_dequant(const cr_mx4* m, void* y, cr_row_dtype dtype, long long ld, void* stream_) {
  using namespace cr;
  if (cr_status s = check_mx4(m, "cr_mx4_dequant", "matrix")) return s;
  if (cr_status s = check_rows(y, dtype, ld, m->inner, "cr_mx4_dequant")) return s;
  cudaStream_t stream = (cudaStream_t)stream_;
  use_stream(stream);
  return by_dtype(dtype, [&](auto type) -> cr_status {
    CR_CUDA(launch_pdl(mx4_dequant_kernel<decltype(type)::value>, unit_grid(m->rows, m->inner), dim3(256), 0, stream, m->codes, m->scales, m->rows, m->inner,
                       y, ld, wide_rows(y, dtype, ld)));
    CR_LAUNCH_CHECK("mx4_dequant_kernel");
    return CR_OK;
  });
}
