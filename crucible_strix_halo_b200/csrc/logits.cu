// Penalties, biases and grammar masks on the logits of spans, and the greedy choice (see cr_logits_choose for the formula).
// Every product, quotient and sum is rounded by itself (no contraction), so that a choice is the definition's own.
// One CTA per (row, span).
#include "mx4.cuh"

namespace cr {

constexpr int kChooseThreads = 512;

struct LogitsTable { cr_logits_args s[kMaxSpans]; };

// Larger value = larger key; every NaN is one key above infinity, both zeros are one key.  0 is below every allowed token.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return v != v ? 0xffffffffu : (u >> 31 ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ uint64_t best_of(float v, int index) { return (uint64_t)order_key(v) << 32 | (uint32_t)~index; }

__device__ __forceinline__ float processed(float l, int n, float bias, const cr_logits_args& a) {
  if (n > 0) {
    l = l > 0.f ? __fdiv_rn(l, a.repetition) : __fmul_rn(l, a.repetition);
    l = __fsub_rn(__fsub_rn(l, __fmul_rn((float)n, a.frequency)), a.presence);
  }
  return a.bias ? __fadd_rn(l, bias) : l;
}

__global__ void __launch_bounds__(kChooseThreads) logits_choose_kernel(const __grid_constant__ LogitsTable T) {
  __shared__ uint64_t warp_best[kChooseThreads / 32];
  pdl_release();
  pdl_wait();
  const cr_logits_args& a = T.s[blockIdx.y];
  const int t = threadIdx.x;
  for (int r = blockIdx.x; r < a.R; r += gridDim.x) {
    uint64_t best = 0;
    for (int v = t; v < a.V; v += kChooseThreads) {
      const size_t at = (size_t)r * a.ld + v;
      float l = a.dtype == CR_ROW_F32 ? reinterpret_cast<const float*>(a.logits)[at]
                                      : (a.dtype == CR_ROW_BF16 ? bf16_bits_to_float(reinterpret_cast<const uint16_t*>(a.logits)[at])
                                                                : __half2float(reinterpret_cast<const __half*>(a.logits)[at]));
      int n = a.counts ? a.counts[v] : 0;
      if (a.drafts)
        for (int j = 0; j < r; ++j) n += a.drafts[j] == v;
      l = processed(l, n, a.bias ? a.bias[v] : 0.f, a);
      const bool allowed = !a.mask || (a.mask[(size_t)r * a.mask_ld + (v >> 5)] >> (v & 31) & 1);
      if (allowed) best = max(best, best_of(l, v));
      if (a.out) a.out[(size_t)r * a.out_ld + v] = allowed ? l : -INFINITY;
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, m));
    if ((t & 31) == 0) warp_best[t >> 5] = best;
    __syncthreads();
    if (t == 0 && a.choice) {
      for (int i = 1; i < kChooseThreads / 32; ++i) best = max(best, warp_best[i]);
      a.choice[r] = best ? (int)~(uint32_t)best : -1;
    }
    __syncthreads();
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
    CR_CUDA(launch_pdl(logits_choose_kernel, dim3(rows < 65535 ? rows : 65535, n), dim3(kChooseThreads), 0, stream, T));
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
