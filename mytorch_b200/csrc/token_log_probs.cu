// Log probabilities of given tokens, the entropy and the most likely alternatives of every row of logits z [n, v], and their gradient.
//   m = max z,  S = sum exp(z - m),  T = sum exp(z - m) (z - m),  log p_j = z_j - m - log S,  H = log S - T / S  (two terms of one sign: nothing cancels).
//   dz_j = -p_j (g + sum of the alternatives' g) - g_H p_j (log p_j + H), and g, or an alternative's g, added at its token.
// A logit of -inf has probability 0 and adds nothing to the entropy or its gradient; a row of nothing else, or with a NaN or +inf, is NaN.
// Alternatives are in the order of their logits, NaN before everything, equal ones by place, which one whole number holds (`key_of`).
#include "common.cuh"

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

__device__ __forceinline__ unsigned ordered(float z) {
  const unsigned b = __float_as_uint(z + 0.f);  // -0 is 0
  return z != z ? 0xFFFFFFFFu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Larger: a larger logit, or of equal ones the earlier.
__device__ __forceinline__ unsigned long long key_of(float z, int place) { return (unsigned long long)ordered(z) << 32 | (0xFFFFFFFFu - (unsigned)place); }

__device__ __forceinline__ long long token_at(const void* tokens, int wide, long long row) {
  return wide ? ((const long long*)tokens)[row] : ((const int*)tokens)[row];
}

template <class T, class F>
__device__ __forceinline__ T over_cta(T x, F f, T* shared) {
  for (int o = 16; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
  __syncthreads();
  x = shared[0];
  for (int w = 1; w < kWarps; ++w) x = f(x, shared[w]);
  return x;
}

__global__ void __launch_bounds__(kThreads) log_probs_kernel(int v, const float* __restrict__ logits, int wide, const void* __restrict__ tokens, int ignores, long long ignore_index, int top,
                                                             float* __restrict__ log_probs, float* __restrict__ entropy, float* __restrict__ stats,
                                                             float* __restrict__ top_log_probs, long long* __restrict__ top_tokens) {
  __shared__ float sf[kWarps];
  __shared__ double sd[kWarps];
  __shared__ unsigned long long sk[kWarps];
  mtb_launch_dependents();
  mtb_wait_prior();
  const long long row = blockIdx.x;
  const float* z = logits + row * v;
  const auto sum = [](double a, double b) { return a + b; };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < v; i += kThreads) m = z[i] != z[i] || m != m ? NAN : fmaxf(m, z[i]);
  m = over_cta(m, [](float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); }, sf);
  double sum_e = 0, sum_ed = 0;  // rows are long
  for (int i = threadIdx.x; i < v; i += kThreads) {
    const float d = z[i] - m, e = expf(d);
    sum_e += e;
    if (e != 0.f) sum_ed += e * d;
  }
  const float s = (float)over_cta(sum_e, sum, sd), t = (float)over_cta(sum_ed, sum, sd);
  const float log_s = logf(s);
  if (threadIdx.x == 0) {
    const long long token = token_at(tokens, wide, row);
    log_probs[row] = ignores && token == ignore_index ? 0.f : token < 0 || token >= v ? NAN : z[token] - m - log_s;
    const float h = log_s - t / s;
    entropy[row] = h;
    if (stats) {
      stats[3 * row] = m;
      stats[3 * row + 1] = s;
      stats[3 * row + 2] = h;
    }
  }
  unsigned long long below = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < v; i += kThreads) {
      const unsigned long long key = key_of(z[i], i);
      if (key < below && key > best) best = key;
    }
    below = over_cta(best, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; }, sk);
    if (threadIdx.x == 0) {
      const int place = (int)(0xFFFFFFFFu - (unsigned)below);
      top_tokens[row * top + k] = place;
      top_log_probs[row * top + k] = z[place] - m - log_s;
    }
  }
}

__global__ void __launch_bounds__(kThreads) log_probs_backward_kernel(int v, const float* __restrict__ logits, int wide, const void* __restrict__ tokens, int ignores, long long ignore_index,
                                                                      int top, const float* __restrict__ dlog_probs, const float* __restrict__ dentropy, const float* __restrict__ dtop,
                                                                      const float* __restrict__ stats, const long long* __restrict__ top_tokens, float* __restrict__ dlogits) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const long long row = blockIdx.x, token = token_at(tokens, wide, row);
  const float* z = logits + row * v;
  float* dz = dlogits + row * v;
  const float m = stats[3 * row], s = stats[3 * row + 1], h = stats[3 * row + 2], log_s = logf(s);
  const float g = !dlog_probs || (ignores && token == ignore_index) ? 0.f : dlog_probs[row], gh = dentropy ? dentropy[row] : 0.f;
  float all = g;
  for (int k = 0; dtop && k < top; ++k) all += dtop[row * top + k];
  for (int i = threadIdx.x; i < v; i += kThreads) {
    const float d = z[i] - m, p = expf(d) / s;
    float x = -p * all;
    if (p != 0.f && gh != 0.f) x -= gh * p * (d - log_s + h);
    if (i == token) x += g;
    for (int k = 0; dtop && k < top; ++k)
      if (top_tokens[row * top + k] == i) x += dtop[row * top + k];
    dz[i] = x;
  }
}

}  // namespace

MTB_API int mtb_token_log_probs_forward_f32(long long n, int v, const float* logits, int token_kind, const void* tokens, int ignores, long long ignore_index, int top,
                                            float* log_probs, float* entropy, float* stats, float* top_log_probs, long long* top_tokens, void* stream) {
  MTB_REQUIRE(n >= 0 && n < (1LL << 31) && v > 0 && top >= 0 && top <= 32 && top <= v && (token_kind == 0 || token_kind == 1), "token_log_probs_forward: bad sizes");
  if (n == 0) return MTB_OK;
  MTB_REQUIRE(logits && tokens && log_probs && entropy && (top == 0 || (top_log_probs && top_tokens)), "token_log_probs_forward: bad arguments");
  MTB_LAUNCH(log_probs_kernel, (unsigned)n, kThreads, 0, (cudaStream_t)stream, v, logits, token_kind, tokens, ignores, ignore_index, top, log_probs, entropy, stats, top_log_probs,
             top_tokens);
  MTB_LAUNCH_CHECK("log_probs_kernel");
  return MTB_OK;
}

MTB_API int mtb_token_log_probs_backward_f32(long long n, int v, const float* logits, int token_kind, const void* tokens, int ignores, long long ignore_index, int top,
                                             const float* dlog_probs, const float* dentropy, const float* dtop, const float* stats, const long long* top_tokens, float* dlogits,
                                             void* stream) {
  MTB_REQUIRE(n >= 0 && n < (1LL << 31) && v > 0 && top >= 0 && top <= 32 && top <= v && (token_kind == 0 || token_kind == 1), "token_log_probs_backward: bad sizes");
  if (n == 0) return MTB_OK;
  MTB_REQUIRE(logits && tokens && stats && dlogits && (top == 0 || !dtop || top_tokens), "token_log_probs_backward: bad arguments");
  MTB_LAUNCH(log_probs_backward_kernel, (unsigned)n, kThreads, 0, (cudaStream_t)stream, v, logits, token_kind, tokens, ignores, ignore_index, top, dlog_probs, dentropy, dtop, stats,
             top_tokens, dlogits);
  MTB_LAUNCH_CHECK("log_probs_backward_kernel");
  return MTB_OK;
}
