// Products with 4-bit weights: Y[R][N] = X[R][K] W[N][K]^T, W microscaled 4-bit floats, X rows as they are.
//
// mx4_simple_kernel: 64 x 64 tiles, both operands as fp32 numbers in shared memory, 4 x 4 products a thread.  A row's sums run over
// K in order, whatever the tile.
#include "mx4.cuh"
#include "proj.cuh"

namespace cr {

__device__ __forceinline__ float mx4_value(const uint8_t* codes, const uint8_t* scales, int row, int k, int K, int groups) {
  const uint32_t b = codes[(size_t)row * (K / 2) + k / 2] >> (4 * (k & 1));
  const uint16_t h = (uint16_t)((b & 8) << 12 | (b & 7) << 9);
  return __half2float(*reinterpret_cast<const __half*>(&h)) * 16384.f * e8m0(scales[mx4_scale_at(row, k / 32, groups)]);
}

template <int TYPE>
__global__ void __launch_bounds__(256) mx4_simple_kernel(const __grid_constant__ ProjParams P, const void* __restrict__ x, long long ld, const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws) {
  __shared__ float A[32][65], B[32][65];
  pdl_release();
  pdl_wait();
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, t = threadIdx.x, tr = t / 16, tc = t % 16, groups = mx4_groups(P.K);
  float acc[4][4] = {};
  for (int k0 = 0; k0 < P.K; k0 += 32) {
    for (int i = t; i < 64 * 32; i += 256) {
      const int r = i / 32, k = i % 32;
      float a = 0.f, b = 0.f;
      if (m0 + r < P.R) {
        const size_t at = (size_t)(m0 + r) * ld + k0 + k;
        if constexpr (TYPE == CR_ROW_F32) a = reinterpret_cast<const float*>(x)[at];
        else if constexpr (TYPE == CR_ROW_BF16) a = bf16_bits_to_float(reinterpret_cast<const uint16_t*>(x)[at]);
        else a = __half2float(reinterpret_cast<const __half*>(x)[at]);
      }
      if (n0 + r < P.N) b = mx4_value(w, ws, n0 + r, k0 + k, P.K, groups);
      A[k][r] = a;
      B[k][r] = b;
    }
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < 32; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(A[k][tr * 4 + i], B[k][tc * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (m0 + tr * 4 + i < P.R && n0 + tc * 4 < P.N) store_quad(P, m0 + tr * 4 + i, n0 + tc * 4, make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]));
}

}  // namespace cr

extern "C" cr_status cr_mx4_rows(const void* x, cr_row_dtype dtype, long long ld, int R, const cr_mx4* w, const cr_proj_out* outs, int n_outs, void* stream_) {
  using namespace cr;
  if (cr_status s = check_mx4(w, "cr_mx4_rows", "W")) return s;
  CR_REQUIRE(R >= 1 && R < (1 << 24), "cr_mx4_rows: R=%d rows", R);
  if (cr_status s = check_rows(x, dtype, ld, w->inner, "cr_mx4_rows")) return s;
  ProjParams P;
  if (cr_status s = list_outs(P, "cr_mx4_rows", R, w->inner, w->rows, outs, n_outs)) return s;
  cudaStream_t stream = (cudaStream_t)stream_;
  use_stream(stream);
  return by_dtype(dtype, [&](auto type) -> cr_status {
    CR_CUDA(launch_pdl(mx4_simple_kernel<decltype(type)::value>, dim3((P.N + 63) / 64, (P.R + 63) / 64), dim3(256), 0, stream, P, x, ld,
                       w->codes, w->scales));
    CR_LAUNCH_CHECK("mx4_simple_kernel");
    return CR_OK;
  });
}
