// Penalties, biases and grammar masks on the logits of spans, and the greedy choice (see cr_logits_choose for the formula).
// Every product, quotient and sum is rounded by itself (no contraction), so that a choice is the definition's own.
//
// HBM-bound with many rows, latency-bound with one: a cluster of eight CTAs takes some rows of a span, its warps 256 tokens at a time in
// eight runs of 32, so that rows of any pitch and address are read a line at a time.  Counts and biases are read once for all rows
// of the cluster; a draft raises its token's count from the next row on.  The best token of a row goes from thread to warp to CTA, and
// the CTAs' are gathered through distributed shared memory: one launch, no scratch.
#include <cooperative_groups.h>
#include "mx4.cuh"

namespace cg = cooperative_groups;

namespace cr {

constexpr int kChooseCluster = 8;
constexpr int kChooseRows = 12;                    // rows of a span that a cluster takes at most

struct LogitsTable { cr_logits_args s[kMaxSpans]; };

// Larger value = larger key, above 0.  The sum makes one number of both zeros and of all NaN (0x7fffffff: above infinity).
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(__fadd_rn(v, 0.f));
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

__device__ __forceinline__ float processed(float l, int n, float bias, const cr_logits_args& a) {
  if (n > 0) {
    l = l > 0.f ? __fdiv_rn(l, a.repetition) : __fmul_rn(l, a.repetition);
    l = __fsub_rn(__fsub_rn(l, __fmul_rn((float)n, a.frequency)), a.presence);
  }
  return a.bias ? __fadd_rn(l, bias) : l;
}

template <int TYPE>
__device__ __forceinline__ float load_logit(const void* p, size_t i) {
  if constexpr (TYPE == CR_ROW_F32) return __ldcs(reinterpret_cast<const float*>(p) + i);
  else if constexpr (TYPE == CR_ROW_BF16) return bf16_bits_to_float(__ldcs(reinterpret_cast<const unsigned short*>(p) + i));
  else return __half2float(__ushort_as_half(__ldcs(reinterpret_cast<const unsigned short*>(p) + i)));
}

// Rows r0 .. r0 + n - 1 of a span, the tokens of this CTA; the best of every warp to warp_best[warp][row]: key and complement of the
// index, so that the larger number is the better token and the lower index among equals.  0: none allowed.
template <int TYPE, int ROWS, int THREADS>
__device__ __forceinline__ void choose_rows(const cr_logits_args& a, int r0, int n, int rank, uint64_t (*warp_best)[ROWS]) {
  const int t = threadIdx.x, l = t & 31, warp = rank * (THREADS / 32) + (t >> 5);
  uint32_t key[ROWS];
  int at[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) { key[r] = 0; at[r] = 0; }
  const int earlier = a.drafts ? r0 : 0;
  for (int v0 = warp * 256; v0 < a.V; v0 += kChooseCluster * (THREADS / 32) * 256) {
    int count[8];
    float bias[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int v = v0 + 32 * k + l;
      count[k] = a.counts && v < a.V ? a.counts[v] : 0;
      bias[k] = a.bias && v < a.V ? a.bias[v] : 0.f;
    }
    for (int j = 0; j < earlier; ++j) {
      const int d = a.drafts[j] - v0 - l;
#pragma unroll
      for (int k = 0; k < 8; ++k) count[k] += d == 32 * k;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (r >= n) break;
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int v = v0 + 32 * k + l;
        x[k] = v < a.V ? load_logit<TYPE>(a.logits, (size_t)(r0 + r) * a.ld + v) : 0.f;
      }
      // lane k < 8 has the words of the piece
      uint32_t word = 0xffffffffu;
      if (a.mask && l < 8 && v0 + 32 * l < a.V) word = a.mask[(size_t)(r0 + r) * a.mask_ld + (v0 >> 5) + l];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int v = v0 + 32 * k + l;
        const bool allowed = (__shfl_sync(0xffffffffu, word, k) >> l & 1) && v < a.V;
        const float y = processed(x[k], count[k], bias[k], a);
        const uint32_t o = order_key(y);
        if (allowed && o > key[r]) { key[r] = o; at[r] = v; }
        if (a.out && v < a.V) __stcs(a.out + (size_t)(r0 + r) * a.out_ld + v, allowed ? y : -INFINITY);
      }
      if (a.drafts && r + 1 < n) {                                  // the row's draft counts from the next row on
        const int d = a.drafts[r0 + r] - v0 - l;
#pragma unroll
        for (int k = 0; k < 8; ++k) count[k] += d == 32 * k;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (r >= n) break;
    const uint32_t top = __reduce_max_sync(0xffffffffu, key[r]);
    const uint32_t low = __reduce_min_sync(0xffffffffu, key[r] == top ? (uint32_t)at[r] : 0xffffffffu);
    if (l == 0) warp_best[t >> 5][r] = top ? (uint64_t)top << 32 | ~low : 0;
  }
}

// grid: (8 CTAs x row groups, spans).
template <int ROWS, int THREADS>
__global__ void __cluster_dims__(kChooseCluster, 1, 1) __launch_bounds__(THREADS)
logits_choose_kernel(const __grid_constant__ LogitsTable T, int group_rows) {
  __shared__ uint64_t warp_best[THREADS / 32][ROWS], cta_best[ROWS];
  cg::cluster_group cluster = cg::this_cluster();
  const cr_logits_args& a = T.s[blockIdx.y];
  const int rank = (int)cluster.block_rank(), t = threadIdx.x;
  const int r0 = blockIdx.x / kChooseCluster * group_rows, n = min(group_rows, a.R - r0);
  pdl_release();
  pdl_wait();
  if (n <= 0) return;                                                // the same for the whole cluster
  if (a.dtype == CR_ROW_F32) choose_rows<CR_ROW_F32, ROWS, THREADS>(a, r0, n, rank, warp_best);
  else if (a.dtype == CR_ROW_BF16) choose_rows<CR_ROW_BF16, ROWS, THREADS>(a, r0, n, rank, warp_best);
  else choose_rows<CR_ROW_F16, ROWS, THREADS>(a, r0, n, rank, warp_best);
  if (!a.choice) return;
  __syncthreads();
  for (int r = t >> 5; r < n; r += THREADS / 32) {                    // a warp per row
    uint64_t best = (t & 31) < THREADS / 32 ? warp_best[t & 31][r] : 0;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, m));
    if ((t & 31) == 0) cta_best[r] = best;
  }
  cluster.sync();
  if (rank == 0 && t < n) {
    uint64_t best = 0;
#pragma unroll
    for (int k = 0; k < kChooseCluster; ++k) best = max(best, *cluster.map_shared_rank(&cta_best[t], k));
    a.choice[r0 + t] = best ? (int)~(uint32_t)best : -1;
  }
  cluster.sync();                                                    // a CTA stays until its best tokens have been read
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
    CR_REQUIRE(a.R >= 1 && a.V >= 1, "cr_logits_choose: span %d: R=%d V=%d", i, a.R, a.V);
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
    // One row per cluster while all clusters run at once, else as many rows as that takes: the counts and biases are read once for them.
    const int room = sm_count() / kChooseCluster / n, want = room > 0 ? (rows + room - 1) / room : rows;
    const int group = want < kChooseRows ? want : kChooseRows;
    const dim3 grid((unsigned)(kChooseCluster * ((rows + group - 1) / group)), n);
    if (group == 1) CR_CUDA(launch_pdl(logits_choose_kernel<1, 1024>, grid, dim3(1024), 0, stream, T, group));
    else CR_CUDA(launch_pdl(logits_choose_kernel<kChooseRows, 512>, grid, dim3(512), 0, stream, T, group));
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
  const int blocks = (n + 255) / 256;
  CR_CUDA(launch_pdl(token_count_kernel, dim3(blocks < 1024 ? blocks : 1024), dim3(256), 0, stream, tokens, n, delta, counts, V));
  CR_LAUNCH_CHECK("token_count_kernel");
  return CR_OK;
}
