// What the projection GEMMs share: the outputs that the columns of a product are scattered into, and the tensor-map copies of
// two-dimensional boxes.
#pragma once
#include "common.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace cr {

constexpr int kMaxOuts = 6;

struct ProjParams {
  int R, K, N, n_outs;
  void* ptr[kMaxOuts];
  int col0[kMaxOuts], cols[kMaxOuts], ld[kMaxOuts], f32[kMaxOuts];
};

// Checks the outputs of a product of R rows and N columns and lists them in P; `who` is the entry point.
inline cr_status list_outs(ProjParams& P, const char* who, int R, int K, int N, const cr_proj_out* outs, int n_outs) {
  CR_REQUIRE(outs && n_outs >= 1 && n_outs <= kMaxOuts, "%s: 1..%d outputs", who, kMaxOuts);
  P.R = R; P.K = K; P.N = N; P.n_outs = n_outs;
  int next = 0;
  for (int i = 0; i < n_outs; ++i) {
    const cr_proj_out& o = outs[i];
    CR_REQUIRE(o.ptr && o.col0 == next && o.cols >= 32 && o.cols % 32 == 0, "%s: output %d must start at column %d and hold a multiple of 32 columns", who, i, next);
    CR_REQUIRE(o.ld >= o.cols && (o.ld * (o.f32 ? 4 : 2)) % 16 == 0 && ((uintptr_t)o.ptr & 15) == 0, "%s: output %d: row pitch and base must keep 16-byte alignment", who, i);
    P.ptr[i] = o.ptr; P.col0[i] = o.col0; P.cols[i] = o.cols; P.ld[i] = o.ld; P.f32[i] = o.f32 ? 1 : 0;
    next += o.cols;
  }
  CR_REQUIRE(next == N, "%s: the outputs cover %d columns, the product has %d", who, next, N);
  return CR_OK;
}

__device__ __forceinline__ void load_box_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
                   umma::smem_u32(dst)),
               "l"(map), "r"(c0), "r"(c1), "r"(umma::smem_u32(bar))
               : "memory");
}
// A box into this CTA's shared memory whose bytes complete on a barrier of either CTA of the pair.
__device__ __forceinline__ void pair_load_box_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
                   umma::smem_u32(dst)),
               "l"(map), "r"(c0), "r"(c1), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory"); }

// Columns col .. col + 31 of one row to the output that owns them.
__device__ __forceinline__ void store_chunk(const ProjParams& P, int row, int col, const float (&v)[32]) {
  int o = 0;
  while (o < P.n_outs - 1 && col >= P.col0[o] + P.cols[o]) ++o;       // outputs are ordered by column; chunks do not straddle them
  const size_t at = (size_t)row * P.ld[o] + (col - P.col0[o]);
  if (P.f32[o]) {
    float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(P.ptr[o]) + at);
#pragma unroll
    for (int k = 0; k < 8; ++k) dst[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
  } else {
    uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(P.ptr[o]) + at);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      unsigned pk[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 b2 = __floats2bfloat162_rn(v[8 * k + 2 * j], v[8 * k + 2 * j + 1]);
        pk[j] = *reinterpret_cast<const unsigned*>(&b2);
      }
      dst[k] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
    }
  }
}
// Four columns of one row.
__device__ __forceinline__ void store_quad(const ProjParams& P, int row, int col, const float4 v) {
  int o = 0;
  while (o < P.n_outs - 1 && col >= P.col0[o] + P.cols[o]) ++o;
  const size_t at = (size_t)row * P.ld[o] + (col - P.col0[o]);
  if (P.f32[o]) *reinterpret_cast<float4*>(reinterpret_cast<float*>(P.ptr[o]) + at) = v;
  else {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(P.ptr[o]) + at) =
        make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
  }
}

}  // namespace cr
