// Penalties, biases and grammar masks on the logits of spans, and the greedy choice (see cr_logits_choose for the formula).
// Every product, quotient and sum is rounded by itself (no contraction), so that a choice is the definition's own.
//
// A cluster of eight CTAs takes a row, its warps 256 tokens at a time: four and four of a lane lie together where the addresses allow
// it, else a run of 32 after another, so that rows of any pitch and address are read whole lines at a time.  The next 256 logits are
// asked for while these are worked on.  Counts and biases come from L2 after the first row; a span's drafts stay in a register of a lane
// each.  The division by the repetition penalty is left to the pieces that hold a repeated token.  The best token goes from thread to warp
// to CTA, and the CTAs' are gathered through distributed shared memory: one launch, no scratch.
//
// What bounds it: with many rows the chain of a piece's loads and some 40 instructions a token (16 x 13 rows of 131,072, fp32, mask and
// processed logits: 58 us, 4.0 TB/s; 8 x 9 rows of 100,352 in bf16: 26 us); with one row latency (5.7 us at 131,071 tokens).  CTAs of 1,024
// threads while one wave holds all rows, of 256 otherwise (82 us for the first call with 512).  Drafts read from memory for every piece
// and runs of 32 alone: 70 us.  Taken back: all rows of a span in one cluster, with counts, biases and keys of twelve rows in registers
// (8 x 9 rows 90 us); one comparison for the eight tokens of a lane with a search behind it (85 us for 16 x 13: in every piece some lane
// finds a better token); pieces of 128 tokens (94 us); fewer registers and five CTAs on an SM (8 x 9 rows 25 us, 16 x 13 rows 79 us); the
// division as a 64-bit product corrected by its exact remainder, without a call (one row 5.9 us, all tokens of a lane at once 6.5).
#include <cooperative_groups.h>
#include "mx4.cuh"

namespace cg = cooperative_groups;

namespace cr {

constexpr int kChooseCluster = 8;

struct LogitsTable { cr_logits_args s[kMaxSpans]; };

// Larger value = larger key, above 0.  The sum makes one number of both zeros and of all NaN (0x7fffffff: above infinity).
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(__fadd_rn(v, 0.f));
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

template <int TYPE>
__device__ __forceinline__ uint32_t logit_bits(const char* p) {
  if constexpr (TYPE == CR_ROW_F32) return __ldcs(reinterpret_cast<const unsigned*>(p));
  else return __ldcs(reinterpret_cast<const unsigned short*>(p));
}
template <int TYPE>
__device__ __forceinline__ float logit_value(uint32_t u) {
  if constexpr (TYPE == CR_ROW_F32) return __uint_as_float(u);
  else if constexpr (TYPE == CR_ROW_BF16) return __uint_as_float(u << 16);
  else return __half2float(__ushort_as_half((unsigned short)u));
}

// What a warp has found: key and index of its lanes' best tokens.
struct Best { uint32_t key = 0; int at = 0; };

// A lane's eight of 256 tokens: one of each run of 32, or (WIDE, where every address allows it) four and four that lie together.
template <bool WIDE>
__device__ __forceinline__ int token_of(int k, int l) { return WIDE ? (k >> 2) * 128 + 4 * l + (k & 3) : 32 * k + l; }

// Eight 32-bit values of a lane's tokens from p (the piece's first); FULL: all of them below `left`.
template <bool FULL, bool WIDE, typename T>
__device__ __forceinline__ void load_tokens(const T* p, int left, T (&v)[8]) {
  static_assert(sizeof(T) == 4, "");
  const int l = threadIdx.x & 31;
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int4 u = *reinterpret_cast<const int4*>(p + 128 * j + 4 * l);
      v[4 * j] = reinterpret_cast<const T&>(u.x); v[4 * j + 1] = reinterpret_cast<const T&>(u.y);
      v[4 * j + 2] = reinterpret_cast<const T&>(u.z); v[4 * j + 3] = reinterpret_cast<const T&>(u.w);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = FULL || 32 * k + l < left ? p[32 * k + l] : T(0);
  }
}

// 256 tokens from v0 on; FULL: all of them below V.
template <bool FULL, bool WIDE>
__device__ __forceinline__ void choose_piece(const cr_logits_args& a, int r, int v0, int draft, float (&x)[8], const uint32_t* mask, float* out, Best& best) {
  const int l = threadIdx.x & 31, left = a.V - v0;
  int n[8];
  bool said = false;
#pragma unroll
  for (int k = 0; k < 8; ++k) n[k] = 0;
  if (a.counts) load_tokens<FULL, WIDE>(a.counts + v0, left, n);
  uint32_t word = 0xffffffffu;                                            // lane k < 8 has the words of tokens 32 k on
  if (mask && l < 8 && (FULL || 32 * l < left)) word = mask[(v0 >> 5) + l];
  float add[8];
  if (a.bias) load_tokens<FULL, WIDE>(a.bias + v0, left, add);
  // Drafts that lie in the piece: lane j has the j-th of them.
  for (int j0 = 0;;) {
    for (uint32_t hits = __ballot_sync(0xffffffffu, (unsigned)(draft - v0) < 256u); hits; hits &= hits - 1) {
      const int d = __shfl_sync(0xffffffffu, draft, __ffs(hits) - 1) - v0;
#pragma unroll
      for (int k = 0; k < 8; ++k) n[k] += d == token_of<WIDE>(k, l);
    }
    if ((j0 += 32) >= r || !a.drafts) break;
    draft = j0 + l < r ? a.drafts[j0 + l] : -1;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) said |= n[k] > 0;
  if (__any_sync(0xffffffffu, said)) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (n[k] > 0) {
        x[k] = x[k] > 0.f ? __fdiv_rn(x[k], a.repetition) : __fmul_rn(x[k], a.repetition);
        x[k] = __fsub_rn(__fsub_rn(x[k], __fmul_rn((float)n[k], a.frequency)), a.presence);
      }
  }
  if (a.bias) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __fadd_rn(x[k], add[k]);
  }
  if (mask) {
    uint32_t mine = 0;                                                    // bit k: the lane's token k is allowed
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < 2; ++j) mine |= (__shfl_sync(0xffffffffu, word, 4 * j + (l >> 3)) >> (4 * (l & 7)) & 15) << (4 * j);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) mine |= (__shfl_sync(0xffffffffu, word, k) >> l & 1) << k;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool allowed = mine >> k & 1;
      const uint32_t o = order_key(x[k]);
      x[k] = allowed ? x[k] : -INFINITY;
      if (allowed && (FULL || 32 * k + l < left) && o > best.key) { best.key = o; best.at = v0 + token_of<WIDE>(k, l); }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t o = order_key(x[k]);
      if ((FULL || 32 * k + l < left) && o > best.key) { best.key = o; best.at = v0 + token_of<WIDE>(k, l); }
    }
  }
  if (out) {
    float* p = out + v0;
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < 2; ++j) __stcs(reinterpret_cast<float4*>(p + 128 * j + 4 * l), make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (FULL || 32 * k + l < left) __stcs(p + 32 * k + l, x[k]);
    }
  }
}

// Row r, the tokens of this warp out of `warps`.  Returns the warp's best: key and complement of the index, so that the larger number
// is the better token and the lower index among equals; 0 where none is allowed.
template <int TYPE, bool WIDE>
__device__ __forceinline__ uint64_t choose_row(const cr_logits_args& a, int r, int warp, int warps) {
  constexpr int SIZE = TYPE == CR_ROW_F32 ? 4 : 2;
  const int l = threadIdx.x & 31, step = warps * 256;
  const char* row = static_cast<const char*>(a.logits) + (size_t)r * a.ld * SIZE;
  float* out = a.out ? a.out + (size_t)r * a.out_ld : nullptr;
  const uint32_t* mask = a.mask ? a.mask + (size_t)r * a.mask_ld : nullptr;
  const int draft = a.drafts && l < r ? a.drafts[l] : -1;
  Best best;
  uint32_t ahead[8];                                                       // of 16-bit logits two to a word where they are loaded so
  auto fetch = [&](int v0) {
    const char* p = row + (size_t)v0 * SIZE;
    if (WIDE && v0 + 256 <= a.V) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (SIZE == 4) {
          const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p) + 32 * j + l);
          ahead[4 * j] = u.x; ahead[4 * j + 1] = u.y; ahead[4 * j + 2] = u.z; ahead[4 * j + 3] = u.w;
        } else {
          const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p) + 32 * j + l);
          ahead[4 * j] = u.x & 0xffffu; ahead[4 * j + 1] = u.x >> 16; ahead[4 * j + 2] = u.y & 0xffffu; ahead[4 * j + 3] = u.y >> 16;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) ahead[k] = v0 + 32 * k + l < a.V ? logit_bits<TYPE>(p + (32 * k + l) * SIZE) : 0;
    }
  };
  if (warp * 256 < a.V) fetch(warp * 256);
#pragma unroll 1
  for (int v0 = warp * 256; v0 < a.V; v0 += step) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = logit_value<TYPE>(ahead[k]);
    if (v0 + step < a.V) fetch(v0 + step);
    if (v0 + 256 <= a.V) choose_piece<true, WIDE>(a, r, v0, draft, x, mask, out, best);
    else choose_piece<false, false>(a, r, v0, draft, x, mask, out, best);
  }
  const uint32_t top = __reduce_max_sync(0xffffffffu, best.key);
  const uint32_t low = __reduce_min_sync(0xffffffffu, best.key == top ? (uint32_t)best.at : 0xffffffffu);
  return top ? (uint64_t)top << 32 | (uint32_t)~low : 0;
}
template <int TYPE>
__device__ __forceinline__ uint64_t choose_row(const cr_logits_args& a, int r, int warp, int warps) {
  constexpr size_t SIZE = TYPE == CR_ROW_F32 ? 4 : 2;
  const uintptr_t row = (uintptr_t)a.logits + (size_t)r * a.ld * SIZE, out = (uintptr_t)a.out + (a.out ? (size_t)r * a.out_ld * 4 : 0);
  const bool wide = ((row & (4 * SIZE - 1)) | (out & 15) | ((uintptr_t)a.counts & 15) | ((uintptr_t)a.bias & 15)) == 0;
  return wide ? choose_row<TYPE, true>(a, r, warp, warps) : choose_row<TYPE, false>(a, r, warp, warps);
}

// grid: (8 CTAs x rows, spans).
template <int THREADS>
__global__ void __cluster_dims__(kChooseCluster, 1, 1) __launch_bounds__(THREADS, 1024 / THREADS) logits_choose_kernel(const __grid_constant__ LogitsTable T) {
  constexpr int WARPS = THREADS / 32;
  __shared__ uint64_t warp_best[WARPS], cta_best[kChooseCluster];
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();                                             // this CTA's shared memory may be written from now on
  const cr_logits_args& a = T.s[blockIdx.y];
  const int rank = (int)cluster.block_rank(), t = threadIdx.x, r = blockIdx.x / kChooseCluster, warp = rank * WARPS + (t >> 5);
  pdl_release();
  pdl_wait();
  uint64_t best = 0;
  if (r < a.R) {
    if (a.dtype == CR_ROW_F32) best = choose_row<CR_ROW_F32>(a, r, warp, kChooseCluster * WARPS);
    else if (a.dtype == CR_ROW_BF16) best = choose_row<CR_ROW_BF16>(a, r, warp, kChooseCluster * WARPS);
    else best = choose_row<CR_ROW_F16>(a, r, warp, kChooseCluster * WARPS);
  }
  if ((t & 31) == 0) warp_best[t >> 5] = best;
  __syncthreads();
  cluster.barrier_wait();
  if (t < 32) {                                                         // the CTA's best to the first CTA of the cluster
    best = t < WARPS ? warp_best[t] : 0;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, m));
    if (t == 0) *cluster.map_shared_rank(&cta_best[rank], 0) = best;
  }
  cluster.barrier_arrive();
  if (rank != 0) return;                                                // arrived: nobody writes here
  cluster.barrier_wait();
  if (t < 32 && r < a.R) {
    best = t < kChooseCluster ? cta_best[t] : 0;
#pragma unroll
    for (int m = kChooseCluster / 2; m > 0; m >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, m));
    if (t == 0 && a.choice) a.choice[r] = best ? (int)~(uint32_t)best : -1;
  }
}

__global__ void __launch_bounds__(256) token_count_kernel(const int* __restrict__ tokens, int n, int delta, int* counts, int V) {
  pdl_release();
  pdl_wait();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int v = tokens[i];
    if (v >= 0 && v < V) atomicAdd(counts + v, delta);          // whole numbers: any order gives the same sums
  }
}

}  // namespace cr

extern "C" cr_status cr_logits_choose(const cr_logits_args* spans, int n_spans, void* stream_) {
  using namespace cr;
  CR_REQUIRE(spans && n_spans >= 1, "cr_logits_choose: no spans");
  for (int i = 0; i < n_spans; ++i) {
    const cr_logits_args& a = spans[i];
    CR_REQUIRE(a.R >= 1 && a.R < (1 << 20) && a.V >= 1 && a.V < (1 << 30), "cr_logits_choose: span %d: R=%d V=%d", i, a.R, a.V);
    if (cr_status s = check_rows(a.logits, a.dtype, a.ld, a.V, "cr_logits_choose")) return s;
    CR_REQUIRE(a.out || a.choice, "cr_logits_choose: span %d asks for nothing", i);
    CR_REQUIRE(!a.out || a.out_ld >= a.V, "cr_logits_choose: span %d: pitch %lld of the processed logits below V=%d", i, a.out_ld, a.V);
    CR_REQUIRE((const void*)a.out != a.logits || (a.dtype == CR_ROW_F32 && a.out_ld == a.ld), "cr_logits_choose: span %d: in place only for fp32 rows of the same pitch", i);
    CR_REQUIRE(!a.mask || a.mask_ld == 0 || a.mask_ld >= (a.V + 31) / 32, "cr_logits_choose: span %d: mask pitch %lld below %d words", i, a.mask_ld, (a.V + 31) / 32);
    CR_REQUIRE(a.repetition > 0.f && a.repetition < INFINITY && fabsf(a.frequency) < INFINITY && fabsf(a.presence) < INFINITY,
               "cr_logits_choose: span %d: penalties must be finite, the repetition penalty positive", i);
  }
  cudaStream_t stream = (cudaStream_t)stream_;
  use_stream(stream);
  for (int i0 = 0; i0 < n_spans; i0 += kMaxSpans) {
    LogitsTable T;
    const int n = n_spans - i0 < kMaxSpans ? n_spans - i0 : kMaxSpans;
    int rows = 1;
    for (int i = 0; i < n; ++i) { T.s[i] = spans[i0 + i]; rows = rows > T.s[i].R ? rows : T.s[i].R; }
    const dim3 grid((unsigned)(kChooseCluster * rows), n);
    if (rows * n * kChooseCluster <= sm_count()) CR_CUDA(launch_pdl(logits_choose_kernel<1024>, grid, dim3(1024), 0, stream, T));
    else CR_CUDA(launch_pdl(logits_choose_kernel<256>, grid, dim3(256), 0, stream, T));
    CR_LAUNCH_CHECK("logits_choose_kernel");
  }
  return CR_OK;
}

extern "C" cr_status cr_token_count(const int* tokens, int n, int delta, int* counts, int V, void* stream_) {
  using namespace cr;
  CR_REQUIRE(n >= 0 && (n == 0 || tokens) && counts && V >= 1, "cr_token_count: null buffer, or n=%d V=%d", n, V);
  if (n == 0) return CR_OK;
  cudaStream_t stream = (cudaStream_t)stream_;
  use_stream(stream);
  const int blocks = n / 256 + 1;
  CR_CUDA(launch_pdl(token_count_kernel, dim3(blocks < 1024 ? blocks : 1024), dim3(256), 0, stream, tokens, n, delta, counts, V));
  CR_LAUNCH_CHECK("token_count_kernel");
  return CR_OK;
}
