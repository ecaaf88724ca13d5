// What a row of logits says about tokens: the log probability of a given one, its rank, the row's entropy, and the most likely
// alternatives with their log probabilities.
//
//   lse = log sum_j exp(x_j),   log p_t = x_t - lse,   H = -sum_j p_j log p_j = log s - (sum_j d_j exp(d_j)) / s
//   with d_j = x_j - max, s = sum_j exp(d_j);   rank of t = how many columns come before it (larger, or equal with a lower id).
//
// Both terms of H are >= 0, so nothing cancels.  A row whose every column is -inf has no distribution: its log probabilities
// are -inf and its entropy 0.  A row that holds NaN or +inf gives NaN.  NaN ranks behind -inf among the alternatives.
#include "common.cuh"

namespace {

constexpr int TOP_MAX = 64;

// (order-preserving image of the value) << 32 | ~id: a larger key comes first, no two are equal, zero is none of them
__device__ __forceinline__ unsigned long long rank_key(float v, unsigned id) {
  unsigned b = __float_as_uint(v == 0.f ? 0.f : v);
  b = v != v ? 0u : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
  return ((unsigned long long)b << 32) | (unsigned long long)(0xFFFFFFFFu - id);
}
__device__ __forceinline__ float rank_value(unsigned long long key) {
  const unsigned o = (unsigned)(key >> 32);
  return o == 0u ? __int_as_float(0x7fffffff) : __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__global__ void __launch_bounds__(256)
token_logprobs_kernel(const T* __restrict__ logits, long ld, int V, const int* __restrict__ tokens, float* __restrict__ logprob,
                      float* __restrict__ entropy, int* __restrict__ rank, int top, int* __restrict__ top_ids,
                      float* __restrict__ top_logprobs) {
  kf_pdl_trigger();
  kf_pdl_wait();
  __shared__ float red[33];
  __shared__ unsigned long long best[8];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int token = tokens ? tokens[row] : 0;
  if (token < 0) return;                                    // a row of padding
  const T* x = logits + (size_t)row * ld;
  const bool inside = token < V;
  float m = -INFINITY;
  for (int i = tid; i < V; i += 256) m = max_nan(m, kf_load(x, i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[warp] = m;
  __syncthreads();
  for (int w = 0; w < 8; ++w) m = max_nan(m, red[w]);
  const float given = inside ? kf_load(x, token) : 0.f;
  float s = 0.f, u = 0.f, before = 0.f;
  for (int i = tid; i < V; i += 256) {
    const float v = kf_load(x, i), d = v - m;
    const float e = m == -INFINITY ? 0.f : expf(d);
    s += e;
    if (e > 0.f) u += d * e;
    before += (v > given || (v == given && i < token)) ? 1.f : 0.f;
  }
  s = kf_block_sum(s, red);
  u = kf_block_sum(u, red);
  const float n_before = kf_block_sum(before, red);
  const bool empty = m == -INFINITY;
  const float log_s = logf(s);
  if (tid == 0) {
    if (logprob) logprob[row] = !inside ? __int_as_float(0x7fffffff) : (empty ? -INFINITY : (given - m) - log_s);
    if (entropy) entropy[row] = empty ? 0.f : log_s - u / s;
    if (rank) rank[row] = inside ? (int)n_before : -1;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long b = 0ull;
    for (int i = tid; i < V; i += 256) {
      const unsigned long long key = rank_key(kf_load(x, i), (unsigned)i);
      if (key < last && key > b) b = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, b, o);
      b = other > b ? other : b;
    }
    __syncthreads();
    if (lane == 0) best[warp] = b;
    __syncthreads();
    for (int w = 0; w < 8; ++w) b = best[w] > b ? best[w] : b;
    last = b;
    if (tid == 0) {
      const float v = rank_value(b);
      if (top_ids) top_ids[(size_t)row * top + k] = (int)(0xFFFFFFFFu - (unsigned)b);
      if (top_logprobs) top_logprobs[(size_t)row * top + k] = (empty && v == v) ? -INFINITY : (v - m) - log_s;
    }
  }
}

}  // namespace

// logits [R, V] of element type dt (KF_F32, KF_BF16), rows ld elements apart; tokens [R] (null: only entropy and alternatives;
// a negative one: the row's outputs stay as they are; one >= V: NaN and rank -1); every output may be null; top <= 64, <= V.
KF_API int kf_token_logprobs(const void* logits, int dt, long ld, int R, int V, const int* tokens, float* logprob, float* entropy,
                             int* rank, int top, int* top_ids, float* top_logprobs, cudaStream_t stream) {
  if (R <= 0) return KF_OK;
  if (V <= 0 || top < 0 || top > TOP_MAX || top > V || (!tokens && (logprob || rank))) return KF_ERR_SIZE;
  if (dt == KF_F32)
    kf_launch(token_logprobs_kernel<float>, dim3(R), dim3(256), 0, stream, (const float*)logits, ld, V, tokens, logprob, entropy,
              rank, top, top_ids, top_logprobs);
  else if (dt == KF_BF16)
    kf_launch(token_logprobs_kernel<__nv_bfloat16>, dim3(R), dim3(256), 0, stream, (const __nv_bfloat16*)logits, ld, V, tokens,
              logprob, entropy, rank, top, top_ids, top_logprobs);
  else
    return KF_ERR_DTYPE;
  KF_CHECK_LAUNCH();
  return KF_OK;
}
