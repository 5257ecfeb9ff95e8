// Rows to microscaled 4-bit floats and back (see cr_mx4 for the format).
//   s = clamp(floor(log2 max |x|) - 2, -127, 127),  code = e2m1(x 2^-s), round to nearest even, saturating
// The exponent field of the largest magnitude is floor(log2) + 127 (0 for a subnormal one, whose s is held to -127 either way), and
// x 2^-s is exact: both steps have the definition's own bits.
//
// Fp32 rows are HBM-bound (16,001 x 6,144: 71 us in, 76 us back, 6.1 and 5.0 TB/s); with 16-bit rows the 110 instructions for a lane's eight
// elements take as long as their bytes (56 and 46 us).  A warp takes 256 elements of a row, so that all that depends on the row is
// computed once for the warp, and four such pieces at a time, asked for before it works on the first.  With pieces that cross rows each
// lane found its own row and addresses: 70 us for bf16 rows; with 32 bytes of bf16 a lane 86; fp32 rows stored 32 bytes a lane in two
// stores instead of a warp's 512 bytes side by side: 110.
#include "mx4.cuh"

namespace cr {

constexpr int kPieces = 4, kQuantThreads = 256, kQuantPerSm = 16;      // pieces of a warp at a time; CTAs per SM at most

// A piece: elements 256 seg .. of a row.  The warp's pieces lie a grid apart and are stepped through, without a division for each.
struct Piece {
  int row, seg;
  __device__ __forceinline__ Piece(unsigned i, unsigned segs) : row((int)(i / segs)), seg((int)(i % segs)) {}
  __device__ __forceinline__ void step(const Piece& by, int segs) {
    row += by.row;
    seg += by.seg;
    if (seg >= segs) { seg -= segs; ++row; }
  }
};

// The warp's first; by a shuffle, which tells the compiler that it is one number for the warp.
__device__ __forceinline__ unsigned first_piece() { return blockIdx.x * (kQuantThreads / 32) + __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0); }

template <int TYPE>
__global__ void __launch_bounds__(kQuantThreads) mx4_quant_kernel(const void* __restrict__ x, long long ld, bool wide, uint8_t* __restrict__ codes,
                                                                  uint8_t* __restrict__ scales, int rows, int inner) {
  pdl_release();
  pdl_wait();
  const int l = threadIdx.x & 31, segs = (inner + 255) / 256, groups = mx4_groups(inner);
  const Piece apart(gridDim.x * (kQuantThreads / 32), segs);
  for (Piece at(first_piece(), segs); at.row < rows;) {
    float v[kPieces][8];
    Piece piece[kPieces] = {at, at, at, at};
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      piece[k] = at;
      const int col = at.seg * 256 + l * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
      if (at.row < rows && col < inner) load_row8<TYPE>(x, (size_t)at.row * ld + col, wide, v[k]);
      at.step(apart, segs);
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const Piece p = piece[k];
      if (p.row >= rows) break;
      const int col = p.seg * 256 + l * 8;
      uint32_t top = largest8(v[k]);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int field = (int)(top >> 23);                            // 255: an infinity or a NaN is among them
      const int s = max(field - 129, -127);
      const uint32_t packed = field == 255 ? 0u : pack_e2m1(v[k], __uint_as_float((uint32_t)(127 - s) << 23));
      if (col < inner) {
        *reinterpret_cast<uint32_t*>(codes + (size_t)p.row * (inner / 2) + col / 2) = packed;
        if ((l & 3) == 0) scales[mx4_scale_at(p.row, p.seg * 8, groups) + (l >> 4) * 512 + (l >> 2 & 3)] = field == 255 ? 255 : (uint8_t)(s + 127);
      }
    }
  }
}

template <int TYPE>
__global__ void __launch_bounds__(kQuantThreads) mx4_dequant_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int inner,
                                                                    void* __restrict__ y, long long ld, bool wide) {
  constexpr int PER = TYPE == CR_ROW_F32 ? 4 : 8, PARTS = 8 / PER;   // elements of a lane that lie together: 16 bytes of the row
  pdl_release();
  pdl_wait();
  const int l = threadIdx.x & 31, segs = (inner + 255) / 256, groups = mx4_groups(inner);
  const Piece apart(gridDim.x * (kQuantThreads / 32), segs);
  for (Piece at(first_piece(), segs); at.row < rows;) {
    uint32_t w[kPieces][PARTS], byte[kPieces][PARTS];
    Piece piece[kPieces] = {at, at, at, at};
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      piece[k] = at;
#pragma unroll
      for (int h = 0; h < PARTS; ++h) {
        const int in = h * 128 + l * PER, col = at.seg * 256 + in, block = in / 32;
        w[k][h] = byte[k][h] = 0;
        if (at.row < rows && col < inner) {
          const uint8_t* c = codes + (size_t)at.row * (inner / 2) + col / 2;
          w[k][h] = PER == 8 ? *reinterpret_cast<const uint32_t*>(c) : *reinterpret_cast<const uint16_t*>(c);
          byte[k][h] = scales[mx4_scale_at(at.row, at.seg * 8, groups) + (block >> 2) * 512 + (block & 3)];
        }
      }
      at.step(apart, segs);
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const Piece p = piece[k];
      if (p.row >= rows) break;
#pragma unroll
      for (int h = 0; h < PARTS; ++h) {
        const int col = p.seg * 256 + h * 128 + l * PER;
        if (col >= inner) continue;
        const float scale = e8m0(byte[k][h]);
        float v[PER];
#pragma unroll
        for (int j = 0; j < PER / 2; ++j) {
          uint32_t two;
          asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}\n" : "=r"(two) : "r"(w[k][h] >> (8 * j)));
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
          v[2 * j] = f.x * scale;
          v[2 * j + 1] = f.y * scale;
        }
        const size_t to = (size_t)p.row * ld + col;
        if constexpr (TYPE == CR_ROW_F32) {
          float* q = reinterpret_cast<float*>(y) + to;
          if (wide) {
            *reinterpret_cast<float4*>(q) = make_float4(v[0], v[1], v[2], v[3]);
          } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) q[j] = v[j];
          }
        } else {
          uint16_t* q = reinterpret_cast<uint16_t*>(y) + to;
          uint32_t o[PER / 2];
#pragma unroll
          for (int j = 0; j < PER / 2; ++j) {
            if constexpr (TYPE == CR_ROW_BF16) { const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]); o[j] = *reinterpret_cast<const uint32_t*>(&t); }
            else { const __half2 t = __floats2half2_rn(v[2 * j], v[2 * j + 1]); o[j] = *reinterpret_cast<const uint32_t*>(&t); }
          }
          if (wide) *reinterpret_cast<uint4*>(q) = make_uint4(o[0], o[1], o[2], o[3]);
          else {
#pragma unroll
            for (int j = 0; j < PER / 2; ++j) { q[2 * j] = (uint16_t)o[j]; q[2 * j + 1] = (uint16_t)(o[j] >> 16); }
          }
        }
      }
    }
  }
}

// The CTAs that take a matrix.
static cr_status quant_grid(const cr_mx4* m, const char* who, dim3* grid) {
  const long long all = (long long)m->rows * ((m->inner + 255) / 256);
  CR_REQUIRE(all < (1ll << 31), "%s: %d x %d elements are too many for a call", who, m->rows, m->inner);
  const long long ctas = (all + kQuantThreads / 32 - 1) / (kQuantThreads / 32), most = (long long)sm_count() * kQuantPerSm;
  *grid = dim3((unsigned)(ctas < most ? ctas : most));
  return CR_OK;
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
  dim3 grid;
  if (cr_status s = quant_grid(to, "cr_mx4_quant", &grid)) return s;
  cudaStream_t stream = (cudaStream_t)stream_;
  use_stream(stream);
  return by_dtype(dtype, [&](auto type) -> cr_status {
    CR_CUDA(launch_pdl(mx4_quant_kernel<decltype(type)::value>, grid, dim3(kQuantThreads), 0, stream, x, ld, wide_rows(x, dtype, ld), to->codes, to->scales, to->rows,
                       to->inner));
    CR_LAUNCH_CHECK("mx4_quant_kernel");
    return CR_OK;
  });
}

extern "C" cr_status cr_mx4_dequant(const cr_mx4* m, void* y, cr_row_dtype dtype, long long ld, void* stream_) {
  using namespace cr;
  if (cr_status s = check_mx4(m, "cr_mx4_dequant", "matrix")) return s;
  if (cr_status s = check_rows(y, dtype, ld, m->inner, "cr_mx4_dequant")) return s;
  dim3 grid;
  if (cr_status s = quant_grid(m, "cr_mx4_dequant", &grid)) return s;
  cudaStream_t stream = (cudaStream_t)stream_;
  use_stream(stream);
  return by_dtype(dtype, [&](auto type) -> cr_status {
    CR_CUDA(launch_pdl(mx4_dequant_kernel<decltype(type)::value>, grid, dim3(kQuantThreads), 0, stream, m->codes, m->scales, m->rows, m->inner, y, ld,
                       wide_rows(y, dtype, ld)));
    CR_LAUNCH_CHECK("mx4_dequant_kernel");
    return CR_OK;
  });
}
