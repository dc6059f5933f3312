// The norm of all gradients together, sqrt(sum over every tensor of g^2), and clipping: g *= min(1, max_norm / (norm + 1e-6)).
//
// Squares and sums are held in 64 bits: a square of a float32 is then exact, none overflows or vanishes, and a conversion and
// an FMA for each 4 bytes are far below what memory allows.  Each CTA adds up chunks of the tensors in a fixed order, and the
// sums of the CTAs are added in a fixed order too: the norm has the same bits every time.
//
// Bound by memory, each gradient read once for the norm; what comes next goes through the chunks backwards and finds the last of them in L2.  Norm and
// update of 161 tensors, 25.6 M elements: 93.5 us with three CTAs of 512 threads and four float4 a thread on an SM, 97.7 with two or four; the
// norm by itself 19.5, 5.2 TB/s.  20 tensors of 0.19 M elements in all: norm and clipping in place 14 us, the host's time for two launches.
#include "clip.cuh"

namespace {

constexpr int kTensors = 192;
constexpr int kChunk = 8192;  // elements of one tensor that a CTA takes at a time: four vectors a thread, all on their way at once
constexpr int kThreads = 512;
template <class T>
struct Table {
  T* g[kTensors];
  long long n[kTensors];
  int chunk_start[kTensors + 1];  // chunk c is one of tensor k with chunk_start[k] <= c < chunk_start[k + 1]
  int count;
};

template <class T>
__device__ __forceinline__ int tensor_of(const Table<T>& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {  // last k with chunk_start[k] <= chunk
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunk_start[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double square(float v) { return (double)v * (double)v; }

// The squares of p[0 .. n), n <= kChunk, by all threads of the CTA.
__device__ __forceinline__ void sum_squares(const float* p, int n, double& a, double& b) {
  int head = (16 - (int)(reinterpret_cast<uintptr_t>(p) & 15)) / 4 % 4;
  if (head > n) head = n;
  if ((int)threadIdx.x < head) a += square(p[threadIdx.x]);
  p += head;
  n -= head;
  float4 f[kChunk / 4 / kThreads];
#pragma unroll
  for (int u = 0; u < kChunk / 4 / kThreads; ++u) {
    const int v = threadIdx.x + u * kThreads;
    f[u] = v < n / 4 ? ld4(p + 4 * v) : make_float4(0, 0, 0, 0);
  }
#pragma unroll
  for (int u = 0; u < kChunk / 4 / kThreads; ++u) {
    a += square(f[u].x) + square(f[u].y);
    b += square(f[u].z) + square(f[u].w);
  }
  if ((int)threadIdx.x < n % 4) b += square(p[n / 4 * 4 + threadIdx.x]);
}

// The CTAs go through the chunks side by side, so that what was read last is what the next kernel, which goes through them backwards, begins with.
__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const __grid_constant__ Table<const float> t, double* __restrict__ sums) {
  mtb_wait_prior();
  mtb_launch_dependents();
  double a = 0, b = 0;
  for (int c = blockIdx.x; c < t.chunk_start[t.count]; c += gridDim.x) {
    const int k = tensor_of(t, c);
    const long long e = (long long)(c - t.chunk_start[k]) * kChunk, left = t.n[k] - e;
    sum_squares(t.g[k] + e, left < kChunk ? (int)left : kChunk, a, b);
  }
  __shared__ double part[kThreads / 32];
  a += b;
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x < 32) {
    a = threadIdx.x < kThreads / 32 ? part[threadIdx.x] : 0;
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (threadIdx.x == 0) sums[blockIdx.x] = a;
  }
}

// Writes nothing where the gradients are under the limit: a factor of one changes no value.
__global__ void __launch_bounds__(kThreads) scale_grads_kernel(const __grid_constant__ Table<float> t, MtbClip clip) {
  mtb_wait_prior();
  mtb_launch_dependents();
  const float factor = mtb_clip_factor<kThreads>(clip);
  if (factor == 1.f) return;
  for (int c = t.chunk_start[t.count] - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
    const int k = tensor_of(t, c);
    const long long e = (long long)(c - t.chunk_start[k]) * kChunk, left = t.n[k] - e;
    int n = left < kChunk ? (int)left : kChunk;
    float* p = t.g[k] + e;
    int head = (16 - (int)(reinterpret_cast<uintptr_t>(p) & 15)) / 4 % 4;
    if (head > n) head = n;
    if ((int)threadIdx.x < head) p[threadIdx.x] *= factor;
    p += head;
    n -= head;
    float4 f[kChunk / 4 / kThreads];
#pragma unroll
    for (int u = 0; u < kChunk / 4 / kThreads; ++u) {
      const int v = threadIdx.x + u * kThreads;
      if (v < n / 4) f[u] = ld4(p + 4 * v);
    }
#pragma unroll
    for (int u = 0; u < kChunk / 4 / kThreads; ++u) {
      const int v = threadIdx.x + u * kThreads;
      f[u].x *= factor; f[u].y *= factor; f[u].z *= factor; f[u].w *= factor;
      if (v < n / 4) st4(p + 4 * v, f[u]);
    }
    if ((int)threadIdx.x < n % 4) p[n / 4 * 4 + threadIdx.x] *= factor;
  }
}

template <class T>
int fill(Table<T>& t, int count, T* const* grads, const long long* sizes, const char* name) {
  long long chunks = 0;
  t.count = count < kTensors ? count : kTensors;
  for (int k = 0; k < t.count; ++k) {
    MTB_REQUIRE(sizes[k] >= 0 && (grads[k] || sizes[k] == 0), "%s: null tensor %d", name, k);
    t.g[k] = grads[k];
    t.n[k] = sizes[k];
    t.chunk_start[k] = (int)chunks;
    chunks += (sizes[k] + kChunk - 1) / kChunk;
    MTB_REQUIRE(chunks < 1LL << 30, "%s: too many elements in one call", name);
  }
  t.chunk_start[t.count] = (int)chunks;
  return MTB_OK;
}

int norm_blocks() { return 3 * mtb_sm_count(); }

}  // namespace

// How many partial sums mtb_grad_norm_f32 leaves for `count` tensors.
MTB_API int mtb_grad_norm_sums(int count) { return count <= 0 ? 0 : mtb_div_up(count, kTensors) * norm_blocks(); }

MTB_API int mtb_grad_norm_f32(int count, const float* const* grads, const long long* sizes, double* sums, void* stream) {
  MTB_REQUIRE(count >= 0 && (count == 0 || (grads && sizes && sums)), "grad_norm: bad arguments");
  for (int base = 0; base < count; base += kTensors) {
    Table<const float> t;
    if (int rc = fill(t, count - base, grads + base, sizes + base, "grad_norm")) return rc;
    MTB_LAUNCH(grad_norm_kernel, norm_blocks(), kThreads, 0, (cudaStream_t)stream, t, sums + base / kTensors * norm_blocks());
  }
  return MTB_OK;
}

MTB_API int mtb_clip_grads_f32(int count, float* const* grads, const long long* sizes, const double* sums, int nsums, double max_norm, float* norm,
                               void* stream) {
  MTB_REQUIRE(count > 0 && grads && sizes && sums && nsums > 0 && norm, "clip_grads: bad arguments");
  for (int base = (count - 1) / kTensors * kTensors; base >= 0; base -= kTensors) {
    Table<float> t;
    if (int rc = fill(t, max_norm < 0 ? 0 : count - base, grads + base, sizes + base, "clip_grads")) return rc;
    const MtbClip clip{sums, nsums, 1.0, max_norm, norm};
    const int chunks = t.chunk_start[t.count], most = 4 * mtb_sm_count();
    MTB_LAUNCH(scale_grads_kernel, chunks < 1 ? 1 : chunks < most ? chunks : most, kThreads, 0, (cudaStream_t)stream, t, clip);
    if (max_norm < 0) break;
    norm = nullptr;  // left by the first launch
  }
  return MTB_OK;
}
