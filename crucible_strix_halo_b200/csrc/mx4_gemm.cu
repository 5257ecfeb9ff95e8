// Product of two matrices of microscaled 4-bit floats for sm_100a: Y[R][N] = X[R][K] W[N][K]^T, fp32 accumulation, the columns
// scattered into the outputs as cr_proj_gemm does (mx4_mma.cuh: how the operands and scales reach the tensor cores).
//
// A step of 64 moves the bytes of a bf16 step of 16 in the same cycles, so the kernels are shaped as those of cr_proj_gemm.
//
// mx4_gemm_pair_kernel<PARTS> (many rows): CTA pairs on 256 x 256 tiles.  Two accumulators of 256 columns would fill tensor memory and
// leave the scales no room: they share 128 columns, which the epilogue reads first and hands over before it stores.  The issuing warp
// decides the pace: with one lane in a branch of its own its descriptors went through vector registers and 32,768 x 2,048 x 12,352
// took 566 us (no stores: 496); with all lanes in the loop and one elected for the instructions 442 (296).  Rows turned through shared
// memory before they are stored 381, sixteen epilogue warps instead of eight 361: 4.6 PFLOP/s, 0.69 of four times the measured bf16
// rate.  What bounds it now is the power cap: block after block of calls runs at 1.3 GHz and takes 416 us (the same products without
// stores 332 us at 1.57 GHz); short K the stores (16,384 x 64 x 12,800: 5.1 TB/s).  Taken back: two whole accumulators on 256 x 192
// tiles (384 us: more bytes a product), stores by the copy engine (387), stores of 32 bytes a lane from
// registers (16,384 x 512 x 9,856, fp32: 125 -> 134), waits that spin (K = 6,144: 103 -> 109 us).
// The few tiles of a last wave are cut into PARTS = 2 or 4, of 128 or 64 columns: 2,048 x 2,048 x 9,856 (312 tiles for 74 pairs) 28.8 -> 27.7 us,
// 2,500 x 512 x 6,144 (240) 19.6 -> 17.7, 8,192 x 2,048 x 2,048 (256) 21.4 -> 20.6.
//
// mx4_gemm_split_kernel<TN> (few rows): 128 x TN tiles, K split over a cluster of up to eight CTAs, bound by latencies: 333 x 4,096 x 2,048
// takes 7.9 us, 1 x 64 x 32 2.1 us.
//
// Every stage has scale columns of its own in tensor memory: they are free when the stage is.  (Two sets, and a wait for the products
// of the stage before the last: 10.3 us for 333 x 4,096 x 2,048.)
// Every wait is bounded; a wait that gives up raises bit 5 of the device status word.
#include <cooperative_groups.h>
#include "mx4_mma.cuh"

namespace cg = cooperative_groups;

namespace cr {

CR_DEFINE_STATUS_WORD(mx4_gemm)

// ---- epilogue: rows of a warp's 32 accumulator lanes to the outputs -----------------------------------------------------
// A lane holds a row; stored from there, an instruction would touch 32 lines for 512 bytes.  The warp turns its rows through 2 KB of
// shared memory, 64 bytes of every row at a time (16-byte chunks exchanged by row, free of bank conflicts).
constexpr int kTurnBytes = 2048;
__device__ __forceinline__ void store_turned(unsigned char* buf, const uint4 (&v)[4], char* to, size_t pitch, int live) {
  const int l = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(buf + l * 64 + ((c ^ (l >> 1 & 3)) << 4)) = v[c];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + l / 4, c = l % 4;
    if (r < live) *reinterpret_cast<uint4*>(to + r * pitch + c * 16) = *reinterpret_cast<const uint4*>(buf + r * 64 + ((c ^ (r >> 1 & 3)) << 4));
  }
  __syncwarp();
}
// Columns col .. col + 31 (which no output divides) of `live` rows from row0 on.
__device__ __forceinline__ void store_columns(const ProjParams& P, unsigned char* buf, int row0, int col, const float (&v)[32], int live) {
  int o = 0;
  while (o < P.n_outs - 1 && col >= P.col0[o] + P.cols[o]) ++o;
  const size_t at = (size_t)row0 * P.ld[o] + (col - P.col0[o]), pitch = P.ld[o];
  uint4 p[4];
  if (P.f32[o]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float* f = v + 16 * h + 4 * c;
        p[c] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      }
      store_turned(buf, p, reinterpret_cast<char*>(reinterpret_cast<float*>(P.ptr[o]) + at + 16 * h), pitch * 4, live);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      unsigned k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 b2 = __floats2bfloat162_rn(v[8 * c + 2 * j], v[8 * c + 2 * j + 1]);
        k[j] = *reinterpret_cast<const unsigned*>(&b2);
      }
      p[c] = make_uint4(k[0], k[1], k[2], k[3]);
    }
    store_turned(buf, p, reinterpret_cast<char*>(reinterpret_cast<__nv_bfloat16*>(P.ptr[o]) + at), pitch * 2, live);
  }
}

// ---- CTA pairs on 256 x 256 tiles ------------------------------------------------------------------------------------
constexpr int kQStages = 5, kQStageBytes = 2 * kXTile + 3 * kXScale, kQBand = 16;
constexpr int kQWarps = 16, kQThreads = 64 + 32 * kQWarps;                // producer, issuer, epilogue warps
constexpr int kQShared = 128, kQScaleCols = 512 - kQShared;               // columns that both accumulators use; first scale column
static_assert(kQStages * 24 <= kQShared, "every stage has scale columns of its own");
constexpr int kQTurn = kQStages * kQStageBytes;                            // room of the epilogue warps behind the stages
constexpr size_t kQSmem = (size_t)kQTurn + kQWarps * kTurnBytes + (2 * kQStages + 4) * 8 + 16;

// Tiles that are left after the last full wave are cut into this many, of as many columns each, while every part finds a pair.
constexpr int pair_parts(long long left, int pairs) { return left == 0 ? 1 : 4 * left <= pairs ? 4 : 2 * left <= pairs ? 2 : 1; }

// whole: tiles that are not cut; cmap: codes of W in boxes for the parts of the others.
template <int PARTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kQThreads, 1)
mx4_gemm_pair_kernel(const __grid_constant__ ProjParams P, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                     const __grid_constant__ CUtensorMap cmap, const __grid_constant__ CUtensorMap xsmap, const __grid_constant__ CUtensorMap wsmap, int whole) {
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + kQTurn + kQWarps * kTurnBytes);
  uint64_t *full = bars, *empty = bars + kQStages, *accFull = bars + 2 * kQStages, *handed = bars + 2 * kQStages + 2;
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bars + 2 * kQStages + 4);
  volatile int& dead = *reinterpret_cast<volatile int*>(&tmem_slot + 1);
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank();                          // 0 leads
  const int t = threadIdx.x, w = t >> 5, l = t & 31;
  const int mt = (P.R + 255) / 256, nt = (P.N + 255) / 256, kb_n = (P.K + kXK - 1) / kXK, tiles = mt * nt;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, units = PARTS == 1 ? tiles : whole + (tiles - whole) * PARTS;
  // Unit i: a tile, or columns from..from + width - 1 of one.
  auto unit_at = [&](int i, int& m0, int& n0, int& from, int& width) {
    from = 0;
    width = 256;
    if (PARTS > 1 && i >= whole) {
      width = 256 / PARTS;
      from = (i - whole) % PARTS * width;
      i = whole + (i - whole) / PARTS;
    }
    const int per_band = mt * kQBand, band = i / per_band, in = i - band * per_band;
    const int tiles_wide = min(kQBand, nt - band * kQBand);
    m0 = (in / tiles_wide) * 256;
    n0 = (band * kQBand + in % tiles_wide) * 256;
  };
  if (t == 0) {
    for (int i = 0; i < kQStages; ++i) { umma::mbar_init(&full[i], 1); umma::mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) umma::mbar_init(&accFull[i], 1);
    umma::mbar_init(handed, 2 * kQWarps);                                 // the epilogue warps of both CTAs
    umma::mbar_fence_init();
    dead = (umma::smem_u32(sm) & 1023u) != 0;                           // the swizzled tiles need 1 KB boundaries
    if (dead) g_mx4_gemm_status = 1;
    prefetch_map(&xmap); prefetch_map(&wmap); prefetch_map(&xsmap); prefetch_map(&wsmap);
  }
  if (w == 1) umma::pair_tmem_alloc(&tmem_slot, 512);
  umma::fence_before_sync();
  cluster.sync();                                                       // both CTAs' barriers are ready
  umma::fence_after_sync();
  pdl_release();
  pdl_wait();
  const uint32_t tm = tmem_slot;
  bool gave_up = dead;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (gave_up) return;
    if (!umma::mbar_wait_timed(bar, parity, &dead)) { gave_up = true; dead = 1; g_mx4_gemm_status = 1; }
  };

  int issued = 0;
  if (w == 0) {
    // ---------------------------------------------------------------- producer (each CTA its own rows of X and of W, all of W's scales)
    if (l == 0) {
      int s = 0, phase = 1;
      for (int i = pair; i < units && !gave_up; i += pairs) {
        int m0, n0, from, width;
        unit_at(i, m0, n0, from, width);
        const uint32_t bytes = 2 * kQStageBytes - (256 - width) * (kXK / 2);
        const CUtensorMap* codes = PARTS == 1 || width == 256 ? &wmap : &cmap;
        const int wrow = n0 + from + width / 2 * (int)rank;
        for (int kb = 0; kb < kb_n; ++kb, ++issued) {
          if (issued >= kQStages) wait(&empty[s], phase);
          if (gave_up) break;
          unsigned char* st = sm + s * kQStageBytes;
          if (rank == 0) umma::mbar_expect_tx(&full[s], bytes);
          const uint32_t bar = umma::cluster_addr(&full[s], 0);
          pair_load_box_2d(st, &xmap, kb * (kXK / 2), m0 + 128 * (int)rank, bar);
          pair_load_box_2d(st + kXTile, codes, kb * (kXK / 2), wrow, bar);
          pair_load_box_2d(st + 2 * kXTile, &xsmap, kb * 256, m0 / 128 + (int)rank, bar);
          pair_load_box_2d(st + 2 * kXTile + kXScale, &wsmap, kb * 256, n0 / 128, bar);
          if (++s == kQStages) { s = 0; phase ^= 1; }
        }
      }
    }
  } else if (w == 1) {
    // ---------------------------------------------------------------- issuer
    if (rank == 0) {
      const bool one = elect_one();
      const Desc xc(tma::desc_sw128(sm, 16, 1024)), wc(tma::desc_sw128(sm + kXTile, 16, 1024));
      const Desc xs(umma::smem_desc(sm + 2 * kXTile, 0, 128)), ws(umma::smem_desc(sm + 2 * kXTile + kXScale, 0, 128));
      int s = 0, phase = 0, local = 0;
      for (int i = pair; i < units && !gave_up; i += pairs, ++local) {
        int m0, n0, from, width;
        unit_at(i, m0, n0, from, width);
        const uint32_t idesc = idesc_mx4(256, width);
        const uint32_t acc = tm + (local & 1) * (256 - kQShared);
        if (local >= 1) wait(handed, (local - 1) & 1);                     // the other accumulator's shared columns, and all of this one, have been read
        for (int kb = 0; kb < kb_n; ++kb) {
          wait(&full[s], phase);
          if (gave_up) break;
          umma::fence_after_sync();
          const uint32_t off = s * (kQStageBytes / 16), cols = tm + kQScaleCols + s * 24;
          const int steps = P.K / 64 - kb * 4;
          if (one) {
            issue_scales<2, 2>(cols, xs, off, ws, off, steps);
            issue_products<2, 2>(acc, xc, off, wc, off, cols, from / 32, idesc, steps, kb == 0);
            umma::pair_commit(&empty[s]);                                         // the stage is free in both CTAs once these products have read it
            if (kb == kb_n - 1) umma::pair_commit(&accFull[local & 1]);
          }
          if (++s == kQStages) { s = 0; phase ^= 1; }
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue: four warps to each quarter of the lanes
    const int q = w & 3, h = (w - 2) >> 2;
    int local = 0;
    for (int i = pair; i < units; i += pairs, ++local) {
      int m0, n0, from, width;
      unit_at(i, m0, n0, from, width);
      n0 += from;
      const int odd = local & 1;
      if (l == 0) wait(&accFull[odd], (local >> 1) & 1);
      __syncwarp();
      if (dead) break;
      umma::fence_after_sync();
      const int row0 = m0 + 128 * (int)rank + 32 * q, live = min(32, P.R - row0);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // the shared columns are the last half of the even accumulator and the first half of the odd one
        const int c = ((odd + j) & 1 ? 0 : 4) + h;
        float v[32];
        umma::tmem_ld32(umma::tmem_addr(tm, q, odd * (256 - kQShared) + 32 * c), v);     // warp-collective
        if (j == 0) {
          umma::fence_before_sync();
          __syncwarp();
          if (l == 0) umma::pair_arrive_relaxed(umma::cluster_addr(handed, 0));
        }
        if (live > 0 && 32 * c < width && n0 + 32 * c < P.N) store_columns(P, sm + kQTurn + (w - 2) * kTurnBytes, row0, n0 + 32 * c, v, live);
      }
    }
  }
  if (dead && rank == 0 && w == 0 && l == 0) drain_copies(full, issued, kQStages);     // both CTAs' copies complete on the leader's barriers
  umma::fence_before_sync();
  __syncwarp();
  cluster.sync();                                                          // neither CTA leaves while the other may still use its memory
  if (w == 1) umma::pair_tmem_dealloc(tm, 512);
}

// ---- few rows: 128 x TN tiles, K split over a cluster ------------------------------------------------------------------
// As in cr_proj_gemm: a stage holds the rows of X that exist (a multiple of 8), the MMA reads 128 all the same, and kVRing keeps a
// whole tile behind the last stage's start.
constexpr int kVRing = 212992, kVMaxStages = 16;
template <int TN> constexpr int kVLd = TN + 4;                           // floats per row of a partial tile in shared memory
constexpr size_t kVSmem = (size_t)kVRing + (2 * kVMaxStages + 1) * 8 + 16;
constexpr int kVThreads = 64 + 256;
template <int TN> constexpr int kVGroups = TN > 128 ? 2 : 1;             // row groups of W's scales
template <int TN> constexpr int kVScaleCols = 8 + 8 * kVGroups<TN>;
template <int TN> constexpr int kVStages = (512 - TN) / kVScaleCols<TN> < kVMaxStages ? (512 - TN) / kVScaleCols<TN> : kVMaxStages;   // as many as have scale columns

// grid: tiles x splits, cluster = splits (along x).
template <int TN>
__global__ void __launch_bounds__(kVThreads, 1)
mx4_gemm_split_kernel(const __grid_constant__ ProjParams P, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                      const __grid_constant__ CUtensorMap xsmap, const __grid_constant__ CUtensorMap wsmap, int splits, int xrows, int ST) {
  static_assert(128 * kVLd<TN> * 4 <= kVRing, "the partial tile takes the place of the stages");
  extern __shared__ __align__(1024) unsigned char sm[];
  constexpr int NG = kVGroups<TN>;
  const int xbytes = xrows * (kXK / 2), stage = xbytes + TN * (kXK / 2) + (1 + NG) * kXScale;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + kVRing);
  uint64_t *full = bars, *empty = bars + kVMaxStages, *accFull = bars + 2 * kVMaxStages;
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bars + 2 * kVMaxStages + 1);
  volatile int& dead = *reinterpret_cast<volatile int*>(&tmem_slot + 1);
  const int t = threadIdx.x, w = t >> 5, l = t & 31;
  const int mt = (P.R + kXM - 1) / kXM, tile = blockIdx.x / splits, split = blockIdx.x % splits;
  const int m0 = (tile % mt) * kXM, n0 = (tile / mt) * TN;                // row tiles of one W tile side by side
  const int kb_all = (P.K + kXK - 1) / kXK, kb0 = kb_all * split / splits, kb_n = kb_all * (split + 1) / splits - kb0;
  if (t == 0) {
    for (int i = 0; i < ST; ++i) { umma::mbar_init(&full[i], 1); umma::mbar_init(&empty[i], 1); }
    umma::mbar_init(accFull, 1);
    umma::mbar_fence_init();
    dead = (umma::smem_u32(sm) & 1023u) != 0;
    if (dead) g_mx4_gemm_status = 1;
    prefetch_map(&xmap); prefetch_map(&wmap); prefetch_map(&xsmap); prefetch_map(&wsmap);
  }
  if (w == 1) umma::tmem_alloc(&tmem_slot, 512);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  pdl_release();
  pdl_wait();
  const uint32_t tm = tmem_slot;
  bool gave_up = dead;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (gave_up) return;
    if (!umma::mbar_wait_timed(bar, parity, &dead)) { gave_up = true; dead = 1; g_mx4_gemm_status = 1; }
  };
  int issued = 0;
  if (w == 0) {
    if (l == 0) {
      for (int it = 0, s = 0, phase = 1; it < kb_n; ++it, ++issued) {
        if (it >= ST) wait(&empty[s], phase);
        if (gave_up) break;
        unsigned char* st = sm + s * stage;
        umma::mbar_expect_tx(&full[s], stage);
        load_box_2d(st + xbytes, &wmap, (kb0 + it) * (kXK / 2), n0, &full[s]);
        load_box_2d(st, &xmap, (kb0 + it) * (kXK / 2), m0, &full[s]);
        load_box_2d(st + xbytes + TN * (kXK / 2), &xsmap, (kb0 + it) * 256, m0 / 128, &full[s]);
        load_box_2d(st + xbytes + TN * (kXK / 2) + kXScale, &wsmap, (kb0 + it) * 256, n0 / 128, &full[s]);
        if (++s == ST) { s = 0; phase ^= 1; }
      }
    }
  } else if (w == 1) {
    const bool one = elect_one();
    const Desc xc(tma::desc_sw128(sm, 16, 1024)), wc(tma::desc_sw128(sm + xbytes, 16, 1024));
    const Desc xs(umma::smem_desc(sm + xbytes + TN * (kXK / 2), 0, 128)), ws(umma::smem_desc(sm + xbytes + TN * (kXK / 2) + kXScale, 0, 128));
    for (int it = 0, s = 0, phase = 0; it < kb_n; ++it) {
      wait(&full[s], phase);
      if (gave_up) break;
      umma::fence_after_sync();
      const uint32_t off = s * (stage / 16), cols = tm + TN + s * kVScaleCols<TN>;
      const int steps = P.K / 64 - (kb0 + it) * 4;
      if (one) {
        issue_scales<1, NG>(cols, xs, off, ws, off, steps);
        issue_products<1, NG>(tm, xc, off, wc, off, cols, (n0 & 127) / 32, idesc_mx4(kXM, TN), steps, it == 0);
        umma::commit(&empty[s]);
        if (it == kb_n - 1) umma::commit(accFull);
      }
      if (++s == ST) { s = 0; phase ^= 1; }
    }
  } else {
    const int q = w & 3, r = 32 * q + l;
    if (l == 0) wait(accFull, 0);
    __syncwarp();
    umma::fence_after_sync();
    if (!dead) {
#pragma unroll 1
      for (int c = (w - 2) >> 2; c < TN / 32; c += 2) {                     // the two warps of a lane quarter take every other chunk
        float v[32];
        umma::tmem_ld32(umma::tmem_addr(tm, q, 32 * c), v);                 // warp-collective
        if (splits == 1) {
          const int row0 = m0 + 32 * q;                                     // the stages have been read: their place serves to turn the rows
          if (row0 < P.R && n0 + 32 * c < P.N) store_columns(P, sm + (w - 2) * kTurnBytes, row0, n0 + 32 * c, v, min(32, P.R - row0));
        } else {                                                            // the stages have been read: the partial tile goes over them
          float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(sm) + (size_t)r * kVLd<TN> + 32 * c);
#pragma unroll
          for (int k = 0; k < 8; ++k) dst[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        }
      }
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  if (dead && w == 0 && l == 0) drain_copies(full, issued, ST);
  if (w == 1) umma::tmem_dealloc(tm, 512);
  if (splits == 1) return;
  // Every CTA of the cluster sums a slice of the rows over all partial tiles, in the order of K.
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int live = min(kXM, P.R - m0), r0 = live * split / splits, r1 = live * (split + 1) / splits;
  constexpr int kQuads = TN / 4, kFlight = 3;
  const float* part[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) part[k] = cluster.map_shared_rank(reinterpret_cast<float*>(sm), k < splits ? k : 0);
  for (int i0 = t; i0 < (r1 - r0) * kQuads; i0 += kFlight * kVThreads) {
    float4 x[kFlight][8];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int i = i0 + f * kVThreads;
      const size_t at = (size_t)(r0 + i / kQuads) * kVLd<TN> + (i % kQuads) * 4;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < splits && i < (r1 - r0) * kQuads) x[f][k] = *reinterpret_cast<const float4*>(part[k] + at);
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int i = i0 + f * kVThreads, c = (i % kQuads) * 4;
      if (i >= (r1 - r0) * kQuads || n0 + c >= P.N) continue;
      float4 sum = x[f][0];
#pragma unroll
      for (int k = 1; k < 8; ++k)
        if (k < splits) { sum.x += x[f][k].x; sum.y += x[f][k].y; sum.z += x[f][k].z; sum.w += x[f][k].w; }
      store_quad(P, m0 + r0 + i / kQuads, n0 + c, sum);
    }
  }
  cluster.sync();                                                          // the partial tiles stay until everybody has read them
}

// How a product is cut.  Costs in cycles, from eighteen shapes of 1 to 8,192 rows timed with every cut: a step of 64, what a tile takes
// beside its steps (its first loads and its epilogue; a pair starts later but overlaps them from its second tile on), and the sum over a
// cluster.  The choice is within 5 % of the fastest cut on all of them (128 x 6,144 x 2,560: 7.7 us on three CTAs a tile of 64 columns,
// 8.5 on five of 128, 12.9 on pairs; 2,048 x 4,096 x 2,048: 10.6 on 128 x 256, 11.7 on pairs; 4,096 rows: 20.6, 18.2).
// A split has to fit in one wave of the clusters that the device holds at once, which the runtime is asked for.
struct Mx4Shape { int tn, splits; };                                       // tn 0: CTA pairs
static cr_status mx4_cluster_slots(const int (**slots)[9]) {
  static PerDeviceOnce looked_up;
  static int table[64][9];
  int dev = 0;
  CR_CUDA(cudaGetDevice(&dev));
  if (cr_status st = once_per_device(looked_up, [dev] {
        CR_CUDA(cudaFuncSetAttribute(mx4_gemm_split_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kVSmem));
        for (int s = 1; s <= 8; ++s) {
          cudaLaunchConfig_t cfg = {};
          cfg.gridDim = dim3(s); cfg.blockDim = dim3(kVThreads); cfg.dynamicSmemBytes = kVSmem;
          cudaLaunchAttribute attr[1];
          attr[0].id = cudaLaunchAttributeClusterDimension;
          attr[0].val.clusterDim.x = s; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
          cfg.attrs = attr; cfg.numAttrs = 1;
          CR_CUDA(cudaOccupancyMaxActiveClusters(&table[dev & 63][s], mx4_gemm_split_kernel<128>, &cfg));
        }
        return CR_OK;
      })) return st;
  *slots = &table[dev & 63];
  return CR_OK;
}
static Mx4Shape mx4_shape(int R, int K, int N, int sms, const int (&slots)[9]) {
  auto up = [](long long a, long long b) { return (a + b - 1) / b; };
  const long long stages = up(K, kXK);
  Mx4Shape best{0, 1};
  double cost = (double)up(up(R, 256) * up(N, 256), sms / 2) * (up(K, 64) * 125 + 1500) + 9900;
  const int tns[3] = {64, 128, 256};
  const double step[3] = {75, 100, 140};
  for (int i = 0; i < 3; ++i) {
    const long long tiles = up(R, kXM) * up(N, tns[i]);
    for (int s = 1; s <= 8 && s <= stages; ++s) {
      if (s > 1 && tiles > slots[s]) break;                                 // splitting pays only while SMs would idle
      const double c = (double)up(tiles * s, sms) * ((s > 1 ? up(stages, s) * 4 : up(K, 64)) * step[i] + 6000 + tns[i] * 10 + (s > 1 ? 500 + tns[i] * 18 : 0));
      if (c < cost) { cost = c; best = Mx4Shape{tns[i], s}; }
    }
  }
  return best;
}

template <int TN>
static cr_status mx4_split_launch(const ProjParams& P, const cr_mx4* x, const cr_mx4* w, int splits, cudaStream_t stream) {
  static PerDeviceOnce configured;
  if (cr_status st = once_per_device(configured, [] {
        CR_CUDA(cudaFuncSetAttribute(mx4_gemm_split_kernel<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kVSmem));
        return CR_OK;
      })) return st;
  const int xrows = P.R < kXM ? (P.R + 7) / 8 * 8 : kXM;
  CUtensorMap xmap, wmap, xsmap, wsmap;
  if (cr_status st = map_mx4(&xmap, &xsmap, x, xrows, 1)) return st;
  if (cr_status st = map_mx4(&wmap, &wsmap, w, TN, kVGroups<TN>)) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((P.R + kXM - 1) / kXM) * ((P.N + TN - 1) / TN) * splits));
  cfg.blockDim = dim3(kVThreads);
  cfg.dynamicSmemBytes = kVSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (pdl_enabled()) { attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[na++].val.programmaticStreamSerializationAllowed = 1; }
  if (splits > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = splits; attr[na].val.clusterDim.y = 1; attr[na++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr; cfg.numAttrs = na;
  const int stage = (xrows + TN) * (kXK / 2) + (1 + kVGroups<TN>) * kXScale, fit = (kVRing - (stage < kXTile ? kXTile - stage : 0)) / stage;
  CR_CUDA(cudaLaunchKernelEx(&cfg, mx4_gemm_split_kernel<TN>, P, xmap, wmap, xsmap, wsmap, splits, xrows, fit < kVStages<TN> ? fit : kVStages<TN>));
  CR_LAUNCH_CHECK("mx4_gemm_split_kernel");
  return CR_OK;
}

template <int PARTS>
static cr_status mx4_pair_launch(const ProjParams& P, const cr_mx4* x, const cr_mx4* w, long long tiles, int pairs, cudaStream_t stream) {
  static PerDeviceOnce configured;
  if (cr_status st = once_per_device(configured, [] {
        CR_CUDA(cudaFuncSetAttribute(mx4_gemm_pair_kernel<PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kQSmem));
        return CR_OK;
      })) return st;
  const long long whole = tiles / pairs * pairs, units = whole + (tiles - whole) * PARTS;
  CUtensorMap xmap, wmap, cmap, xsmap, wsmap;
  if (cr_status st = map_mx4(&xmap, &xsmap, x, 128, 1)) return st;
  if (cr_status st = map_mx4(&wmap, &wsmap, w, 128, 2)) return st;
  if (PARTS == 1) cmap = wmap;
  else if (cr_status st = map_mx4(&cmap, &wsmap, w, 128 / PARTS, 2)) return st;
  CR_CUDA(launch_pdl(mx4_gemm_pair_kernel<PARTS>, dim3(2 * (unsigned)(units < pairs ? units : pairs)), dim3(kQThreads), kQSmem, stream, P, xmap, wmap, cmap, xsmap,
                     wsmap, (int)whole));
  CR_LAUNCH_CHECK("mx4_gemm_pair_kernel");
  return CR_OK;
}
}  // namespace cr

extern "C" cr_status cr_mx4_gemm(const cr_mx4* x, const cr_mx4* w, const cr_proj_out* outs, int n_outs, void* stream_) {
  using namespace cr;
  if (cr_status s = check_mx4(x, "cr_mx4_gemm", "X")) return s;
  if (cr_status s = check_mx4(w, "cr_mx4_gemm", "W")) return s;
  CR_REQUIRE(x->inner == w->inner, "cr_mx4_gemm: X has %d elements a row, W %d", x->inner, w->inner);
  ProjParams P;
  if (cr_status s = list_outs(P, "cr_mx4_gemm", x->rows, w->inner, w->rows, outs, n_outs)) return s;
  const int(*slots)[9];
  if (cr_status st = mx4_cluster_slots(&slots)) return st;
  const Mx4Shape shape = mx4_shape(P.R, P.K, P.N, sm_count(), *slots);
  cudaStream_t stream = (cudaStream_t)stream_;
  use_stream(stream);
  if (shape.tn == 64) return mx4_split_launch<64>(P, x, w, shape.splits, stream);
  if (shape.tn == 128) return mx4_split_launch<128>(P, x, w, shape.splits, stream);
  if (shape.tn == 256) return mx4_split_launch<256>(P, x, w, shape.splits, stream);
  const long long tiles = (long long)((P.R + 255) / 256) * ((P.N + 255) / 256);
  const int pairs = sm_count() / 2, parts = pair_parts(tiles % pairs, pairs);
  if (parts == 4) return mx4_pair_launch<4>(P, x, w, tiles, pairs, stream);
  if (parts == 2) return mx4_pair_launch<2>(P, x, w, tiles, pairs, stream);
  return mx4_pair_launch<1>(P, x, w, tiles, pairs, stream);
}
