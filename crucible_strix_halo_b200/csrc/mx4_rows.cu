// Products of a few rows with 4-bit weights for sm_100a: Y[R][N] = X[R][K] W[N][K]^T, W microscaled 4-bit floats, X fp32, bf16 or
// fp16 rows as they are: the projections of decode and verify rows, and the head.  W's bytes set the time.
//
// Turning the weights into numbers that X could be multiplied with costs more instructions than an SM has while it receives them:
// with mma.sync on unpacked weights 131,072 x 2,048 took 72 us for one row and 114 for nine, 3 to 5 times the weights' own 22.  Here
// X is turned into 4-bit numbers instead, without loss, and the tensor cores multiply the weights as they lie:
//   x = sum over j = 0.. of d_j 2^(E - 2 - 3 j),  d_j = the whole number in -4..4 nearest to what the digits before it left,
// with 2^E above the largest of x's block of 32.  A digit is an e2m1 number and its weight an e8m0 scale, so that the digits of a row
// are rows of a 4-bit matrix.  Ten of them for bf16 and fp16 rows, twelve for fp32 rows: an element is off by at most 2^(E - 30) or
// 2^(E - 36), and exact where it has no bits below twice that, so that a channel a thousand times the others' size takes
// nothing from them.  No weight is below 2^-127, the smallest scale: where that comes first an element is off by at most 2^-128.  (E = 128,
// the range's last octave: twice the bound.)  The sums of an output's digits, each in fp32, are added from the smallest up.  The order
// of all sums depends on N and K alone: a row has the same bits in every call.
//
// mx4_rows_kernel: 128 rows of W are the M side, up to 256 digit rows the N side; persistent over W (up to 128 digit rows), or one tile
// per cluster of CTAs that share K where there are few tiles.  With few elements of X for a CTA it makes their digits itself, into the tiles that the
// tensor cores read, while the first stages of W arrive: one launch.  Otherwise mx4_digits_kernel writes them into the workspace, a
// block of 256 rows for each pass over W, from where they come with every stage, and the first stages of W are asked for while it runs.
// The line between the two is at 2,048 elements: 1 x 2,048 x 12,352 takes 6.1 us this way and 7.9 that way, 1 x 4,096 x 2,048 (eight CTAs
// to a row) 6.5 and 7.2; 2 x 2,048 x 131,072 29.3 and 29.0, 4 x 2,048 x 12,352 11.5 and 8.4, since every CTA makes all digits.
//
// mx4_rows_pair_kernel, for more than 128 digit rows where nothing shares K: CTA pairs, 256 rows of W to a tile, each CTA with half of the
// digits' codes, which come from L2 once for 256 rows of W and not for 128.  At 131,072 x 2,048, against one CTA: 16 rows 30.9 and 32.8 us,
// 20 rows 33.7 and 47.9, 24 rows 35.3 and 52.9, 72 rows (three passes) 79.6 and 131.7.
//
// Taken back: X's digits kept in shared memory beside a shorter ring (13 rows 30.3 -> 31.7 us); a digits kernel that lets this one in
// before it waits, so that both start sooner and the weights are asked for later (4 rows 29.5 -> 31.4).
//
// What bounds it: W at 131,072 x 2,048 is 142.6 MB, 21.8 us at the copy bandwidth and 22.6 us for the same copies without products.  One row
// takes 26.3 us, 9 rows 30.5, 13 rows 30.1 (4.9 TB/s): the launches, the first stage's and the last tile's latency, 4 to 7 us.  The
// copying thread's divisions had cost 4 us; one accumulator for 11 to 19 rows 13 us, since the epilogue stands between two tiles then.
// Calls over few weights are latencies: 1 x 64 x 32 3.6 us.
//
// Every wait is bounded (bit 6 of the device status word), and the bound is the kernel's own time: under a programmatic launch the kernel
// ahead may run for as long as it likes, so every role waits for its end before its first bounded wait.
#include <cooperative_groups.h>
#include "mx4_mma.cuh"

namespace cg = cooperative_groups;

namespace cr {

CR_DEFINE_STATUS_WORD(mx4_rows)

constexpr int kDigitsMost = 12, kPassRows = 256;                 // digit rows of a pass over W
constexpr int kRowsEnd = 1 << 20;                                // rows of X: fewer
__host__ __device__ constexpr int digits_of(int dtype) { return dtype == CR_ROW_F32 ? 12 : 10; }
// Digit rows come in halves of 128: so many rows of X fill one, twice as many make a pass.
__host__ __device__ constexpr int half_rows(int digits) { return 128 / digits; }
constexpr int kHalfMost = half_rows(10);
__host__ __device__ constexpr int digit_row(int r, int digits) { return r / half_rows(digits) * 128 + r % half_rows(digits) * digits; }
constexpr int kStream = -1;                                      // digits from the workspace, instead of from rows of a type
// producer, issuer, four epilogue warps; eight where they make digits before
__host__ __device__ constexpr int rows_threads(int from) { return from == kStream ? 192 : 320; }
constexpr int kOwnElements = 2048;                               // elements of X that a CTA turns into digits itself
constexpr int kNMaxStages = 8;
constexpr size_t kNRing = 212992;
constexpr size_t kNSmem = kNRing + (2 * kNMaxStages + 6) * 8 + 16;

// ---- digits ----------------------------------------------------------------------------------------------------------
// The digits of eight elements of a block, whose other elements are with three neighbouring threads (`quad`: the four lanes): for each
// j the word of codes and the scale byte go to `put`.
template <int D, typename F>
__device__ __forceinline__ void make_digits(float (&v)[8], unsigned quad, F&& put) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(quad, top, 1));
  top = max(top, __shfl_xor_sync(quad, top, 2));
  int field = max((int)(top >> 23), 1);                            // 2^(field - 126) is above every element; 255: not finite
  if (field <= 3 * D - 2) field = (field + 1) / 3 * 3 + 1;         // where the weights go below 2^-127, the last one is 2^-127 itself
  // In the range's last octave a first digit of 4 would stand for 2^128, with sums that overflow where the product does not: it is
  // held to 3, and the next digit's weight is a quarter of its.
  const bool last_octave = field == 254;
  const float up = __uint_as_float((uint32_t)(field == 255 ? 1 : 255 - field) << 23);
  f2 x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = mul2(pack2(v[2 * k], v[2 * k + 1]), pack2(up, up));       // below 4
  const f2 whole = pack2(12582912.f, 12582912.f), back = pack2(-12582912.f, -12582912.f), minus = pack2(-1.f, -1.f), eight = pack2(8.f, 8.f);
  const f2 second = last_octave ? pack2(4.f, 4.f) : eight;
#pragma unroll
  for (int j = 0; j < D; ++j) {
    float d[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f2 n = add2(add2(x[k], whole), back);                        // 1.5 2^23 leaves no room behind the point: the nearest whole number
      float2 f = unpack2(n);
      if (j == 0) {
        const float most = last_octave ? 3.f : 4.f;
        f = make_float2(fminf(fmaxf(f.x, -most), most), fminf(fmaxf(f.y, -most), most));
        n = pack2(f.x, f.y);
      }
      x[k] = mul2(fma2(n, minus, x[k]), j == 0 ? second : eight);
      d[2 * k] = f.x;
      d[2 * k + 1] = f.y;
    }
    const int scale = field - 1 - 3 * j + (j > 0 && last_octave);  // below 0: what is left, 2^-128 at most, is left out
    put(j, field == 255 || scale < 0 ? 0u : pack_e2m1(d, 1.f), field == 255 ? 255 : (uint8_t)max(scale, 0));
  }
}

template <int TYPE>
__global__ void __launch_bounds__(128) mx4_digits_kernel(const void* __restrict__ x, long long ld, bool wide, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                         int rows, int inner, int pass_rows) {
  // What stands before this kernel on the stream has ended when the kernel behind it is let in: that one reads the weights at once.
  pdl_wait();
  pdl_release();
  const int per_row = inner / 8, groups = mx4_groups(inner);
  const long long u = (long long)blockIdx.x * 128 + threadIdx.x;
  if (u >= (long long)rows * per_row) return;                      // a multiple of eight threads
  const int row = (int)(u / per_row), i = (int)(u - (long long)row * per_row);
  float v[8];
  load_row8<TYPE>(x, (size_t)row * ld + (size_t)i * 8, wide, v);
  const int at = row / pass_rows * kPassRows + digit_row(row % pass_rows, digits_of(TYPE));
  uint32_t* to = reinterpret_cast<uint32_t*>(codes) + (size_t)at * per_row + i;
  make_digits<digits_of(TYPE)>(v, 0xfu << (threadIdx.x & 28), [&](int j, uint32_t word, uint8_t scale) {
    to[(size_t)j * per_row] = word;
    if ((threadIdx.x & 3) == 0) scales[mx4_scale_at(at + j, i >> 2, groups)] = scale;
  });
}

// ---- product ----------------------------------------------------------------------------------------------------------------
struct RowsShape {
  int splits, tiles, passes, pass_rows;                            // CTAs that share K; tiles of W; passes over W, rows of X in each
  int digits, cols;                                                // digits of an element; digit rows of a pass, a multiple of 8
  int stages, stage, accs;                                         // the ring and its stages' bytes; accumulators
  const void* x;                                                   // rows whose digits the CTAs make, their pitch, and whether they come 16 bytes at a time
  long long ld;
  int wide;
};

// Columns of tensor memory: an accumulator's (read 16 at a time from a row's first digit on) and the scales' of a stage.
__host__ __device__ inline int acc_columns(int cols) { return (cols + 31) / 32 * 32; }
__host__ __device__ inline int scale_columns(int cols) { return cols > 128 ? 24 : 16; }

// The same for CTA pairs: from one accumulator to the other, and the first scale column.
__host__ __device__ inline bool pair_shares(int cols) { return cols > 192; }
__host__ __device__ inline int pair_acc_step(int cols) { return pair_shares(cols) ? 128 : acc_columns(cols); }
__host__ __device__ inline int pair_scale_column(int cols) { return pair_shares(cols) ? 384 : 2 * acc_columns(cols); }

template <int FROM>
__global__ void __launch_bounds__(rows_threads(FROM), 1)
mx4_rows_kernel(const __grid_constant__ ProjParams P, const __grid_constant__ RowsShape S, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                const __grid_constant__ CUtensorMap wsmap, const __grid_constant__ CUtensorMap xsmap) {
  constexpr bool OWN = FROM != kStream;
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + kNRing);
  uint64_t *full = bars, *empty = bars + kNMaxStages, *accFull = bars + 2 * kNMaxStages, *accEmpty = bars + 2 * kNMaxStages + 2, *ready = bars + 2 * kNMaxStages + 4;
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bars + 2 * kNMaxStages + 5);
  volatile int& dead = *reinterpret_cast<volatile int*>(&tmem_slot + 1);
  const int t = threadIdx.x, w = t >> 5, l = t & 31;
  const int split = blockIdx.x % S.splits, first = blockIdx.x / S.splits, step = gridDim.x / S.splits, units = S.tiles * S.passes;
  const int kb_all = (P.K + kXK - 1) / kXK, kb0 = kb_all * split / S.splits, kb_n = kb_all * (split + 1) / S.splits - kb0;
  const int ST = S.stages, two = !OWN && S.cols > 128;
  const int accs = S.accs, acc_cols = acc_columns(S.cols), scale_cols = scale_columns(S.cols);
  // The CTA's own digits behind the ring: codes of every stage of K, then their scales.
  unsigned char *own_codes = sm + ST * S.stage, *own_scales = own_codes + kb_n * S.cols * (kXK / 2);
  if (t == 0) {
    for (int i = 0; i < ST; ++i) { umma::mbar_init(&full[i], 1); umma::mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { umma::mbar_init(&accFull[i], 1); umma::mbar_init(&accEmpty[i], 4); }
    umma::mbar_init(ready, 8);                                        // the warps that make digits
    umma::mbar_fence_init();
    dead = (umma::smem_u32(sm) & 1023u) != 0;                        // the swizzled tiles need 1 KB boundaries
    if (dead) g_mx4_rows_status = 1;
    prefetch_map(&wmap); prefetch_map(&wsmap);
    if constexpr (!OWN) { prefetch_map(&xmap); prefetch_map(&xsmap); }
  }
  if (w == 1) umma::tmem_alloc(&tmem_slot, 512);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  pdl_release();
  const uint32_t tm = tmem_slot;
  bool gave_up = dead;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (gave_up) return;
    if (!umma::mbar_wait_timed(bar, parity, &dead)) { gave_up = true; dead = 1; g_mx4_rows_status = 1; }
  };
  int issued = 0;
  // A unit is a tile of W and a pass; the passes of a tile follow one another.  Stage: codes of W, scales of W; scales and codes of X.
  if (w == 0) {
    if (l == 0) {
      // Where a stage comes from and goes to, moved on without a division per stage: they set the pace of the copies otherwise.
      struct Cursor {
        int unit, left, kb, n0, pass, s = 0, phase = 0;
        __device__ __forceinline__ void seek(int passes) { n0 = unit / passes; pass = unit - n0 * passes; n0 *= 128; }
      };
      const int own = first < units ? (units - first + step - 1) / step : 0;
      auto begin = [&] { Cursor c; c.unit = first; c.left = own * kb_n; c.kb = 0; c.seek(S.passes); return c; };
      auto advance = [&](Cursor& c) {
        --c.left;
        if (++c.kb == kb_n) { c.kb = 0; c.unit += step; c.seek(S.passes); }
        if (++c.s == ST) { c.s = 0; c.phase ^= 1; }
      };
      auto load_w = [&](const Cursor& c) {
        unsigned char* st = sm + c.s * S.stage;
        umma::mbar_expect_tx(&full[c.s], S.stage);
        load_box_2d(st, &wmap, (kb0 + c.kb) * (kXK / 2), c.n0, &full[c.s]);
        load_box_2d(st + kXTile, &wsmap, (kb0 + c.kb) * 256, c.n0 / 128, &full[c.s]);
      };
      auto load_x = [&](const Cursor& c) {
        unsigned char* st = sm + c.s * S.stage + kXTile + kXScale;
        load_box_2d(st + kXScale * (1 + two), &xmap, (kb0 + c.kb) * (kXK / 2), c.pass * kPassRows, &full[c.s]);
        load_box_2d(st, &xsmap, (kb0 + c.kb) * 256, c.pass * (kPassRows / 128), &full[c.s]);
      };
      Cursor cw = begin(), cx = cw;
      if constexpr (OWN) pdl_wait();                                   // the kernel ahead is the caller's: it may be writing the weights
      for (int i = 0; i < ST && cw.left > 0; ++i) { load_w(cw); advance(cw); }
      if constexpr (!OWN) {
        pdl_wait();
        for (int i = 0; i < ST && cx.left > 0; ++i) { load_x(cx); advance(cx); }
      }
      while (cw.left > 0) {
        wait(&empty[cw.s], cw.phase ^ 1);
        if (gave_up) break;
        load_w(cw);
        if constexpr (!OWN) load_x(cw);
        advance(cw);
      }
      issued = own * kb_n - cw.left;
    }
  } else if (w == 1) {
    const bool one = elect_one();
    const Desc wc(tma::desc_sw128(sm, 16, 1024)), xc(tma::desc_sw128(OWN ? own_codes : sm + kXTile + kXScale * (2 + two), 16, 1024));
    const Desc ws(umma::smem_desc(sm + kXTile, 0, 128)), xs(umma::smem_desc(OWN ? own_scales : sm + kXTile + kXScale, 0, 128));
    const uint32_t idesc = idesc_mx4(kXM, S.cols), scales = tm + accs * acc_cols;
    int s = 0, phase = 0, local = 0;
    pdl_wait();
    if constexpr (OWN) wait(ready, 0);
    for (int u = first; u < units && !gave_up; u += step, ++local) {
      const int a = accs == 2 ? local & 1 : 0, use = accs == 2 ? local >> 1 : local;
      if (use >= 1) wait(&accEmpty[a], (use - 1) & 1);
      for (int kb = 0; kb < kb_n; ++kb) {
        wait(&full[s], phase);
        if (gave_up) break;
        umma::fence_after_sync();
        const uint32_t off = s * (S.stage / 16), cols = scales + s * scale_cols;
        const uint32_t xoff = OWN ? kb * (S.cols * (kXK / 2) / 16) : off, xsoff = OWN ? kb * (kXScale / 16) : off;
        const int steps = P.K / 64 - (kb0 + kb) * 4;
        if (one) {
          if (two) {
            issue_scales<1, 2>(cols, ws, off, xs, xsoff, steps);
            issue_products<1, 2>(tm + a * acc_cols, wc, off, xc, xoff, cols, 0, idesc, steps, kb == 0);
          } else {
            issue_scales<1, 1>(cols, ws, off, xs, xsoff, steps);
            issue_products<1, 1>(tm + a * acc_cols, wc, off, xc, xoff, cols, 0, idesc, steps, kb == 0);
          }
          umma::commit(&empty[s]);
          if (kb == kb_n - 1) umma::commit(&accFull[a]);
        }
        if (++s == ST) { s = 0; phase ^= 1; }
      }
    }
  } else {
    pdl_wait();
    if constexpr (OWN) {
      // Eight elements a thread, in the places that a 128-byte-swizzled copy would give them: the 16-byte chunk of a row changes
      // places with its number xor the row's.
      const int D = digits_of(FROM), eights = kb_n * (kXK / 8), k0 = kb0 * kXK;
      for (int i = t - 64; i < S.pass_rows * eights; i += 256) {
        const int r = i / eights, e = i - r * eights, kb = e / 32, word = e % 32, b = word / 4;     // b: block of the stage
        float v[8] = {};
        if (k0 + e * 8 < P.K) load_row8<FROM>(S.x, (size_t)r * S.ld + k0 + e * 8, S.wide, v);
        make_digits<digits_of(FROM)>(v, 0xfu << (t & 28), [&](int j, uint32_t codes, uint8_t scale) {
          const int row = r * D + j;
          *reinterpret_cast<uint32_t*>(own_codes + kb * S.cols * (kXK / 2) + row * 128 + ((b ^ (row & 7)) << 4) + word % 4 * 4) = codes;
          if ((t & 3) == 0) own_scales[kb * kXScale + b / 4 * 512 + row % 32 * 16 + row / 32 * 4 + b % 4] = scale;
        });
      }
      umma::fence_async_smem();
      __syncwarp();
      if (l == 0) umma::mbar_arrive(ready);
    }
    const int q = w & 3;
    int local = 0;
    for (int u = first; u < units && w < 6; u += step, ++local) {
      const int a = accs == 2 ? local & 1 : 0, use = accs == 2 ? local >> 1 : local;
      const int n0 = u / S.passes * 128 + 32 * q, r0 = u % S.passes * S.pass_rows, live = min(S.pass_rows, P.R - r0);
      if (l == 0) wait(&accFull[a], use & 1);
      __syncwarp();
      if (dead) break;
      umma::fence_after_sync();
      int o = 0;
      while (o < P.n_outs - 1 && n0 >= P.col0[o] + P.cols[o]) ++o;     // 32 columns never straddle outputs
      const int half = 128 / S.digits;
      float y[2 * kHalfMost];
#pragma unroll
      for (int r = 0; r < 2 * kHalfMost; ++r) {
        if (r >= live) break;
        float v[16];
        const int col = r < half ? r * S.digits : 128 + (r - half) * S.digits;
        umma::tmem_ld16(umma::tmem_addr(tm, q, a * acc_cols + col), v);     // warp-collective
        y[r] = 0.f;
#pragma unroll
        for (int j = kDigitsMost - 1; j >= 0; --j)
          if (j < S.digits) y[r] += v[j];
      }
      umma::fence_before_sync();
      __syncwarp();
      if (l == 0) umma::mbar_arrive_relaxed(&accEmpty[a]);                  // the next tile's products may come
#pragma unroll
      for (int r = 0; r < 2 * kHalfMost; ++r) {
        if (r >= live) break;
        if (S.splits > 1) {
          reinterpret_cast<float*>(sm)[r * 128 + 32 * q + l] = y[r];                  // every stage has been read
        } else if (n0 < P.N) {
          const size_t at = (size_t)(r0 + r) * P.ld[o] + (n0 + l - P.col0[o]);
          if (P.f32[o]) reinterpret_cast<float*>(P.ptr[o])[at] = y[r];
          else reinterpret_cast<__nv_bfloat16*>(P.ptr[o])[at] = __float2bfloat16_rn(y[r]);
        }
      }
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  if (dead && w == 0 && l == 0) drain_copies(full, issued, ST);
  if (w == 1) umma::tmem_dealloc(tm, 512);
  if (S.splits == 1) return;
  // One unit per cluster: each CTA adds a part of the outputs over all shares of K, in their order.
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int n0 = first / S.passes * 128, r0 = first % S.passes * S.pass_rows, outs = min(S.pass_rows, P.R - r0) * 128;
  for (int i = outs * split / S.splits + t; i < outs * (split + 1) / S.splits; i += rows_threads(FROM)) {
    float y = 0.f;
    for (int k = 0; k < S.splits; ++k) y += *cluster.map_shared_rank(reinterpret_cast<float*>(sm) + i, k);
    const int col = n0 + i % 128;
    if (col >= P.N) continue;
    int o = 0;
    while (o < P.n_outs - 1 && col >= P.col0[o] + P.cols[o]) ++o;
    const size_t at = (size_t)(r0 + i / 128) * P.ld[o] + (col - P.col0[o]);
    if (P.f32[o]) reinterpret_cast<float*>(P.ptr[o])[at] = y;
    else reinterpret_cast<__nv_bfloat16*>(P.ptr[o])[at] = __float2bfloat16_rn(y);
  }
  cluster.sync();                                                       // the parts stay until everybody has read them
}

// ---- many digit rows: CTA pairs over two tiles of W ---------------------------------------------------------------------
// With more than 128 digit rows a CTA's shared memory sets the pace (see mx4_gemm_pair_kernel): a pair multiplies 256 rows of W, each CTA
// its 128, with all digit rows, each CTA half of them.  Whole accumulators in turn up to 192 digit rows; above, two that share 128
// columns, which are free once the warps of that half have read them.  Stage: codes of W, half of X's codes, scales of W, all of X's
// scales.  D: digits of an element.
constexpr int kPairThreads = 64 + 256;                           // producer, issuer, four epilogue warps to each half of the digit rows
template <int D>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
mx4_rows_pair_kernel(const __grid_constant__ ProjParams P, const __grid_constant__ RowsShape S, const __grid_constant__ CUtensorMap wmap,
                     const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wsmap, const __grid_constant__ CUtensorMap xsmap) {
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + kNRing);
  uint64_t *full = bars, *empty = bars + kNMaxStages, *accFull = bars + 2 * kNMaxStages, *handed = bars + 2 * kNMaxStages + 2;     // handed: [accumulator][half]
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bars + 2 * kNMaxStages + 6);
  volatile int& dead = *reinterpret_cast<volatile int*>(&tmem_slot + 1);
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank();                          // 0 leads
  const int t = threadIdx.x, w = t >> 5, l = t & 31;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1, units = S.tiles * S.passes, kb_n = (P.K + kXK - 1) / kXK, ST = S.stages;
  const bool shared = pair_shares(S.cols);
  const int xcodes = S.cols / 2 * (kXK / 2);
  if (t == 0) {
    for (int i = 0; i < ST; ++i) { umma::mbar_init(&full[i], 1); umma::mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) umma::mbar_init(&accFull[i], 1);
    for (int i = 0; i < 4; ++i) umma::mbar_init(&handed[i], 8);           // four epilogue warps in each CTA
    umma::mbar_fence_init();
    dead = (umma::smem_u32(sm) & 1023u) != 0;                           // the swizzled tiles need 1 KB boundaries
    if (dead) g_mx4_rows_status = 1;
    prefetch_map(&wmap); prefetch_map(&xmap); prefetch_map(&wsmap); prefetch_map(&xsmap);
  }
  if (w == 1) umma::pair_tmem_alloc(&tmem_slot, 512);
  umma::fence_before_sync();
  cluster.sync();                                                       // both CTAs' barriers are ready
  umma::fence_after_sync();
  pdl_release();
  const uint32_t tm = tmem_slot;
  bool gave_up = dead;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (gave_up) return;
    if (!umma::mbar_wait_timed(bar, parity, &dead)) { gave_up = true; dead = 1; g_mx4_rows_status = 1; }
  };
  int issued = 0;
  if (w == 0) {
    if (l == 0) {
      struct Cursor {
        int unit, left, kb, n0, pass, s, phase;
        __device__ __forceinline__ void seek(int passes) { n0 = unit / passes; pass = unit - n0 * passes; n0 *= 256; }
      };
      const int all = first < units ? (units - first + step - 1) / step * kb_n : 0;
      auto advance = [&](Cursor& c) {
        --c.left;
        if (++c.kb == kb_n) { c.kb = 0; c.unit += step; c.seek(S.passes); }
        if (++c.s == ST) { c.s = 0; c.phase ^= 1; }
      };
      auto load_w = [&](const Cursor& c) {
        unsigned char* st = sm + c.s * S.stage;
        if (rank == 0) umma::mbar_expect_tx(&full[c.s], 2 * S.stage);
        const uint32_t bar = umma::cluster_addr(&full[c.s], 0);
        pair_load_box_2d(st, &wmap, c.kb * (kXK / 2), c.n0 + 128 * (int)rank, bar);
        pair_load_box_2d(st + kXTile + xcodes, &wsmap, c.kb * 256, c.n0 / 128 + (int)rank, bar);
      };
      auto load_x = [&](const Cursor& c) {
        unsigned char* st = sm + c.s * S.stage + kXTile;
        const uint32_t bar = umma::cluster_addr(&full[c.s], 0);
        pair_load_box_2d(st, &xmap, c.kb * (kXK / 2), c.pass * kPassRows + S.cols / 2 * (int)rank, bar);
        pair_load_box_2d(st + xcodes + kXScale, &xsmap, c.kb * 256, c.pass * (kPassRows / 128), bar);
      };
      Cursor cw{first, all, 0, 0, 0, 0, 0};
      cw.seek(S.passes);
      Cursor cx = cw;
      for (int i = 0; i < ST && cw.left > 0; ++i) { load_w(cw); advance(cw); }
      pdl_wait();
      for (int i = 0; i < ST && cx.left > 0; ++i) { load_x(cx); advance(cx); }
      while (cw.left > 0) {
        wait(&empty[cw.s], cw.phase ^ 1);
        if (gave_up) break;
        load_w(cw);
        load_x(cw);
        advance(cw);
      }
      issued = all - cw.left;
    }
  } else if (w == 1) {
    if (rank == 0) {
      const bool one = elect_one();
      const Desc wc(tma::desc_sw128(sm, 16, 1024)), xc(tma::desc_sw128(sm + kXTile, 16, 1024));
      const Desc ws(umma::smem_desc(sm + kXTile + xcodes, 0, 128)), xs(umma::smem_desc(sm + kXTile + xcodes + kXScale, 0, 128));
      const uint32_t idesc = idesc_mx4(256, S.cols), scales = tm + pair_scale_column(S.cols);
      int s = 0, phase = 0, local = 0;
      pdl_wait();
      for (int u = first; u < units && !gave_up; u += step, ++local) {
        const int odd = local & 1;
        const uint32_t acc = tm + odd * pair_acc_step(S.cols);
        if (local >= 2) {                                                  // this accumulator has been read
          wait(&handed[2 * odd], ((local - 2) >> 1) & 1);
          wait(&handed[2 * odd + 1], ((local - 2) >> 1) & 1);
        }
        // and the shared columns of the other one: the second half of the even accumulator, the first half of the odd one
        if (shared && local >= 1) wait(&handed[2 * (odd ^ 1) + odd], ((local - 1) >> 1) & 1);
        for (int kb = 0; kb < kb_n; ++kb) {
          wait(&full[s], phase);
          if (gave_up) break;
          umma::fence_after_sync();
          const uint32_t off = s * (S.stage / 16), cols = scales + s * 24;
          const int steps = P.K / 64 - kb * 4;
          if (one) {
            issue_scales<2, 2>(cols, ws, off, xs, off, steps);
            issue_products<2, 2>(acc, wc, off, xc, off, cols, 0, idesc, steps, kb == 0);
            umma::pair_commit(&empty[s]);                                         // the stage is free in both CTAs once these products have read it
            if (kb == kb_n - 1) umma::pair_commit(&accFull[odd]);
          }
          if (++s == ST) { s = 0; phase ^= 1; }
        }
      }
    }
  } else {
    constexpr int HALF = half_rows(D), GROUP = HALF / 2;                 // rows of X of a half; of one read of 64 columns
    static_assert(GROUP * D <= 64 && 2 * GROUP == HALF, "");
    const int q = w & 3, h = (w - 2) >> 2;
    int local = 0;
    pdl_wait();
    for (int u = first; u < units; u += step, ++local) {
      const int odd = local & 1, n0 = u / S.passes * 256 + 128 * (int)rank + 32 * q;
      const int r0 = u % S.passes * S.pass_rows + h * HALF, live = min(HALF, min(S.pass_rows - h * HALF, P.R - r0));   // rows of this half
      if (l == 0) wait(&accFull[odd], (local >> 1) & 1);
      __syncwarp();
      if (dead) break;
      umma::fence_after_sync();
      float y[HALF];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (g * GROUP >= live) break;
        float v[64];
        umma::tmem_ld64(umma::tmem_addr(tm, q, odd * pair_acc_step(S.cols) + 128 * h + g * GROUP * D), v);     // warp-collective
#pragma unroll
        for (int i = 0; i < GROUP; ++i) {
          y[g * GROUP + i] = 0.f;
#pragma unroll
          for (int j = D - 1; j >= 0; --j) y[g * GROUP + i] += v[i * D + j];
        }
      }
      umma::fence_before_sync();
      __syncwarp();
      if (l == 0) umma::pair_arrive_relaxed(umma::cluster_addr(&handed[2 * odd + h], 0));
      if (n0 >= P.N) continue;
      int o = 0;
      while (o < P.n_outs - 1 && n0 >= P.col0[o] + P.cols[o]) ++o;       // 32 columns never straddle outputs
#pragma unroll
      for (int i = 0; i < HALF; ++i) {
        if (i >= live) break;
        const size_t at = (size_t)(r0 + i) * P.ld[o] + (n0 + l - P.col0[o]);
        if (P.f32[o]) reinterpret_cast<float*>(P.ptr[o])[at] = y[i];
        else reinterpret_cast<__nv_bfloat16*>(P.ptr[o])[at] = __float2bfloat16_rn(y[i]);
      }
    }
  }
  if (dead && rank == 0 && w == 0 && l == 0) drain_copies(full, issued, ST);     // both CTAs' copies complete on the leader's barriers
  umma::fence_before_sync();
  __syncwarp();
  cluster.sync();                                                          // neither CTA leaves while the other may still use its memory
  if (w == 1) umma::pair_tmem_dealloc(tm, 512);
}

// CTAs that share K: as many as give every SM a tile, while all clusters run at once.  R has no part in it.
static cr_status rows_splits(int N, int K, int* splits) {
  static PerDeviceOnce configured;
  static int slots[64][9];
  int dev = 0;
  CR_CUDA(cudaGetDevice(&dev));
  if (cr_status st = once_per_device(configured, [dev] {
        CR_CUDA(cudaFuncSetAttribute(mx4_rows_kernel<kStream>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kNSmem));
        CR_CUDA(cudaFuncSetAttribute(mx4_rows_kernel<CR_ROW_F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kNSmem));
        CR_CUDA(cudaFuncSetAttribute(mx4_rows_kernel<CR_ROW_BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kNSmem));
        CR_CUDA(cudaFuncSetAttribute(mx4_rows_kernel<CR_ROW_F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kNSmem));
        CR_CUDA(cudaFuncSetAttribute(mx4_rows_pair_kernel<10>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kNSmem));
        CR_CUDA(cudaFuncSetAttribute(mx4_rows_pair_kernel<12>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kNSmem));
        for (int s = 1; s <= 8; ++s) {
          cudaLaunchConfig_t cfg = {};
          cfg.gridDim = dim3(s); cfg.blockDim = dim3(rows_threads(kStream)); cfg.dynamicSmemBytes = kNSmem;
          cudaLaunchAttribute attr[1];
          attr[0].id = cudaLaunchAttributeClusterDimension;
          attr[0].val.clusterDim.x = s; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
          cfg.attrs = attr; cfg.numAttrs = 1;
          CR_CUDA(cudaOccupancyMaxActiveClusters(&slots[dev & 63][s], mx4_rows_kernel<kStream>, &cfg));
        }
        return CR_OK;
      })) return st;
  const int tiles = (N + 127) / 128, stages = (K + kXK - 1) / kXK;
  *splits = 1;
  for (int s = 2; s <= 8 && s <= stages; ++s)
    if (tiles <= slots[dev & 63][s]) *splits = s;
  return CR_OK;
}

template <int FROM>
static cr_status rows_launch(const ProjParams& P, const RowsShape& S, const CUtensorMap (&maps)[4], cudaStream_t stream) {
  const long long units = (long long)S.tiles * S.passes;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(S.splits > 1 ? units * S.splits : (units < sm_count() ? units : sm_count())));
  cfg.blockDim = dim3(rows_threads(FROM));
  cfg.dynamicSmemBytes = kNSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (pdl_enabled()) { attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[na++].val.programmaticStreamSerializationAllowed = 1; }
  if (S.splits > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = S.splits; attr[na].val.clusterDim.y = 1; attr[na++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr; cfg.numAttrs = na;
  CR_CUDA(cudaLaunchKernelEx(&cfg, mx4_rows_kernel<FROM>, P, S, maps[0], maps[1], maps[2], maps[3]));
  CR_LAUNCH_CHECK("mx4_rows_kernel");
  return CR_OK;
}

}  // namespace cr

// Passes over W of R rows: as few as hold them, with about as many rows in each.
static int rows_passes(int R, int digits) {
  const int most = 2 * cr::half_rows(digits);
  return (R + most - 1) / most;
}
extern "C" size_t cr_mx4_rows_workspace_bytes(int R, int inner) {
  if (R < 1 || R >= cr::kRowsEnd || inner < 1) return 0;
  const int rows = rows_passes(R, cr::kDigitsMost) * cr::kPassRows;
  return cr_mx4_code_bytes(rows, inner) + cr_mx4_scale_bytes(rows, inner);
}

extern "C" cr_status cr_mx4_rows(const void* x, cr_row_dtype dtype, long long ld, int R, const cr_mx4* w, void* workspace, size_t workspace_bytes,
                                 const cr_proj_out* outs, int n_outs, void* stream_) {
  using namespace cr;
  if (cr_status s = check_mx4(w, "cr_mx4_rows", "W")) return s;
  CR_REQUIRE(R >= 1 && R < kRowsEnd, "cr_mx4_rows: R=%d rows", R);
  if (cr_status s = check_rows(x, dtype, ld, w->inner, "cr_mx4_rows")) return s;
  CR_REQUIRE((long long)R * w->inner < (1ll << 35) && (long long)R * w->rows < (1ll << 40), "cr_mx4_rows: %d rows of %d x %d are too many for a call", R, w->rows, w->inner);
  CR_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= cr_mx4_rows_workspace_bytes(R, w->inner),
             "cr_mx4_rows: the workspace must hold %zu bytes at a 16-byte boundary", cr_mx4_rows_workspace_bytes(R, w->inner));
  ProjParams P;
  if (cr_status s = list_outs(P, "cr_mx4_rows", R, w->inner, w->rows, outs, n_outs)) return s;
  RowsShape S{};
  if (cr_status s = rows_splits(P.N, P.K, &S.splits)) return s;
  S.tiles = (P.N + 127) / 128;
  S.digits = digits_of(dtype);
  S.passes = rows_passes(R, S.digits);
  S.pass_rows = (R + S.passes - 1) / S.passes;
  // A multiple of 16 above 128: a pair halves it.
  S.cols = S.pass_rows <= half_rows(S.digits) ? (S.digits * S.pass_rows + 7) / 8 * 8 : (digit_row(S.pass_rows - 1, S.digits) + S.digits + 15) / 16 * 16;
  const bool pairs = S.splits == 1 && S.cols > 128;
  cr_mx4 d{static_cast<uint8_t*>(workspace), nullptr, S.passes * kPassRows, w->inner};
  d.scales = d.codes + cr_mx4_code_bytes(d.rows, d.inner);
  const int kb_most = ((w->inner + kXK - 1) / kXK + S.splits - 1) / S.splits;
  const bool own = S.passes == 1 && S.cols <= 128 && (long long)R * kb_most * kXK <= kOwnElements;
  S.stage = kXTile + kXScale + (own ? 0 : S.cols / (pairs ? 2 : 1) * (kXK / 2) + (S.cols > 128 ? 2 : 1) * kXScale);
  const size_t room = kNRing - (own ? (size_t)kb_most * (S.cols * (kXK / 2) + kXScale) : 0);
  // Two accumulators while they leave columns for the scales of four stages: the epilogue of a tile beside the products of the next.
  S.accs = 2 * acc_columns(S.cols) + 4 * scale_columns(S.cols) <= 512 ? 2 : 1;
  const int columned = (512 - (pairs ? pair_scale_column(S.cols) : S.accs * acc_columns(S.cols))) / scale_columns(S.cols);
  const int most = columned < kNMaxStages ? columned : kNMaxStages;
  S.stages = (int)(room / S.stage) < most ? (int)(room / S.stage) : most;
  S.x = x;
  S.ld = ld;
  S.wide = wide_rows(x, dtype, ld);
  CUtensorMap maps[4];                                               // W, X, scales of W, scales of X
  if (cr_status s = map_mx4(&maps[0], &maps[2], w, 128, 1)) return s;
  cudaStream_t stream = (cudaStream_t)stream_;
  use_stream(stream);
  if (own) {
    maps[1] = maps[0];                                               // not used
    maps[3] = maps[2];
    return by_dtype(dtype, [&](auto type) { return rows_launch<decltype(type)::value>(P, S, maps, stream); });
  }
  if (cr_status s = map_mx4(&maps[1], &maps[3], &d, S.cols / (pairs ? 2 : 1), S.cols > 128 ? 2 : 1)) return s;
  if (cr_status s = by_dtype(dtype, [&](auto type) -> cr_status {
        const long long threads = (long long)R * (w->inner / 8);
        CR_CUDA(launch_pdl(mx4_digits_kernel<decltype(type)::value>, dim3((unsigned)((threads + 127) / 128)), dim3(128), 0, stream, x, ld, (bool)S.wide, d.codes, d.scales,
                           R, w->inner, S.pass_rows));
        CR_LAUNCH_CHECK("mx4_digits_kernel");
        return CR_OK;
      })) return s;
  if (!pairs) return rows_launch<kStream>(P, S, maps, stream);
  S.tiles = (P.N + 255) / 256;
  const long long units = (long long)S.tiles * S.passes;
  const int most_pairs = sm_count() / 2;
  CR_CUDA(launch_pdl(S.digits == 10 ? mx4_rows_pair_kernel<10> : mx4_rows_pair_kernel<12>, dim3(2 * (unsigned)(units < most_pairs ? units : most_pairs)), dim3(kPairThreads), kNSmem, stream, P, S, maps[0], maps[1],
                     maps[2], maps[3]));
  CR_LAUNCH_CHECK("mx4_rows_pair_kernel");
  return CR_OK;
}
