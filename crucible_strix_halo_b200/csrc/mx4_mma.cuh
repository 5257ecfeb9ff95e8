// Block-scaled 4-bit products on tcgen05 (kind::mxf4): tensor maps of the operands, scales to tensor memory, issue of a stage of
// 256 elements of K.
//
// The unit multiplies 64 elements of K per step, each block of 32 by its operands' two powers of two, on the codes as they lie
// (packed, K-major, 128-byte-swizzled tiles of 256 elements).  The scales of 128 rows x 4 blocks are one 512-byte tile of the matrix,
// which tcgen05.cp.32x128b.warpx4 spreads over the lanes of tensor memory as the unit reads it: row r in lane r % 32 and column
// r / 32, its four blocks in the bytes of that word.  tcgen05.cp is ordered before the products issued after it, but not behind those
// issued before it: the columns that it writes must have been read.
#pragma once
#include "mx4.cuh"
#include "proj.cuh"

namespace cr {

constexpr int kXM = 128, kXK = 256;                               // rows of a tile, K elements of a stage
constexpr int kXTile = kXM * kXK / 2;                             // codes of 128 rows of a stage
constexpr int kXScale = 2 * 512;                                  // their scales

// Instruction descriptor for kind::mxf4: e2m1 operands (format 1), e8m0 scales, both operands K-major.
__host__ __device__ constexpr uint32_t idesc_mx4(int M, int N) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27);
}
// The two blocks of a step of 64 lie in the low (0) or the high (1) half of the scale words.
__host__ __device__ constexpr uint32_t idesc_half(uint32_t idesc, int half) { return idesc | ((uint32_t)half << 5) | ((uint32_t)half << 30); }

template <int GROUP>
__device__ __forceinline__ void mx4_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  if constexpr (GROUP == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}
// One 512-byte scale tile to four columns of tensor memory (of both CTAs of a pair, each from its own shared memory).
template <int GROUP>
__device__ __forceinline__ void scales_to_tmem(uint32_t col, uint64_t tile) {
  if constexpr (GROUP == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(col), "l"(tile) : "memory");
  else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(col), "l"(tile) : "memory");
}
// Descriptors of what a stage holds, as 16-byte steps behind the first stage's: the address is the low 14 bits of the low word, and
// shared memory ends below their range, so that one 32-bit sum moves a descriptor.
struct Desc {
  uint32_t lo, hi;
  __device__ __forceinline__ explicit Desc(uint64_t d) : lo((uint32_t)d), hi((uint32_t)(d >> 32)) {}
  __device__ __forceinline__ uint64_t at(uint32_t bytes16) const { return (uint64_t)hi << 32 | (lo + bytes16); }
};
// One thread of a warp whose lanes all run the loop: the operands of the instructions stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}\n" : "=r"(p));
  return p != 0;
}

// The scales of one stage: tiles [k group] of A, [row group][k group] of B in shared memory; four columns of tensor memory per tile,
// those of A first, then B's row groups side by side.  aoff, boff: 16-byte steps from the first stage.
template <int GROUP, int NG>
__device__ __forceinline__ void issue_scales(uint32_t cols, const Desc& as, uint32_t aoff, const Desc& bs, uint32_t boff, int steps) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (2 * k >= steps) break;
    scales_to_tmem<GROUP>(cols + 4 * k, as.at(aoff + 32 * k));
#pragma unroll
    for (int g = 0; g < NG; ++g) scales_to_tmem<GROUP>(cols + 8 + (k * NG + g) * 4, bs.at(boff + (2 * g + k) * 32));
  }
}
// The products of one stage.  sb0: columns from the first of B's scales to the tile's own first row.
template <int GROUP, int NG>
__device__ __forceinline__ void issue_products(uint32_t d, const Desc& ac, uint32_t aoff, const Desc& bc, uint32_t boff, uint32_t cols, int sb0, uint32_t idesc, int steps, bool first) {
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    if (ks >= steps) break;
    mx4_mma<GROUP>(d, ac.at(aoff + ks * 2), bc.at(boff + ks * 2), idesc_half(idesc, ks & 1), cols + 4 * (ks >> 1), cols + 8 + (ks >> 1) * NG * 4 + sb0,
                   first && ks == 0 ? 0u : 1u);
  }
}

// After a wait has given up, by the thread that issued the copies: no CTA ends before its last copies have landed, for a millisecond
// each at most.  `issued` stages went into a ring of `ring`.
__device__ __forceinline__ void drain_copies(uint64_t* full, int issued, int ring) {
  for (int i = issued > ring ? issued - ring : 0; i < issued; ++i) umma::mbar_wait_timed(&full[i % ring], (i / ring) & 1, nullptr, 1000000);
}

// Codes as a tensor map of bytes with boxes of box_rows x 128 bytes, 128-byte swizzle; scales as words, a row of the map for a row
// group, boxes of two tiles by box_groups.  Past the edges the copy engine fills in zeros.
inline cr_status map_mx4(CUtensorMap* codes, CUtensorMap* scales, const cr_mx4* m, int box_rows, int box_groups) {
  tma::EncodeFn enc;
  if (cr_status s = tma::encoder(&enc)) return s;
  const cuuint32_t unit[2] = {1, 1};
  const cuuint64_t dims[2] = {(cuuint64_t)m->inner / 2, (cuuint64_t)m->rows}, pitch[1] = {(cuuint64_t)m->inner / 2};
  const cuuint32_t box[2] = {kXK / 2, (cuuint32_t)box_rows};
  CUresult r = enc(codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, m->codes, dims, pitch, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) {
    const cuuint64_t groups = mx4_groups(m->inner);
    const cuuint64_t sdims[2] = {groups * 128, ((cuuint64_t)m->rows + 127) / 128}, spitch[1] = {groups * 512};
    const cuuint32_t sbox[2] = {256, (cuuint32_t)box_groups};
    r = enc(scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, m->scales, sdims, spitch, sbox, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed with code %d", (int)r);
    return CR_ERR_CUDA;
  }
  return CR_OK;
}

}  // namespace cr
