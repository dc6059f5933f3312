// The norm of all gradients together, sqrt(sum over every tensor of g^2), and clipping: g *= min(1, max_norm / (norm + 1e-6)).
//
// Squares and sums are held in 64 bits: a square of a float32 is then exact, none overflows or vanishes, and a conversion and
// an FMA for each 4 bytes are far below what memory allows.  Each CTA adds up one stretch of all elements laid end to end, in
// a fixed order, and the sums of the CTAs are added in a fixed order too: the norm has the same bits every time.
#include "clip.cuh"

namespace {

constexpr int kNormTensors = 192;
struct NormTable {
  const float* g[kNormTensors];
  long long start[kNormTensors + 1];  // of each tensor, among all elements of the table
  int count;
};

__device__ __forceinline__ int tensor_of(const NormTable& t, long long e) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {  // last k with start[k] <= e
    const int mid = (lo + hi + 1) >> 1;
    if (t.start[mid] <= e) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double square(float v) { return (double)v * (double)v; }

// f(pointer to four values on a 16-byte boundary) and f1(pointer to one) over p[0 .. n), THREADS at a time.
template <int THREADS, int AHEAD>
__device__ __forceinline__ void sum_squares(const float* p, long long n, double& a, double& b) {
  long long head = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) / 4 % 4;
  if (head > n) head = n;
  if (threadIdx.x < head) a += square(p[threadIdx.x]);
  p += head;
  n -= head;
  const long long n4 = n / 4;
  long long v = threadIdx.x;
  for (; v + (AHEAD - 1) * THREADS < n4; v += AHEAD * THREADS) {
    float4 f[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) f[u] = ld4(p + 4 * (v + u * THREADS));
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      a += square(f[u].x) + square(f[u].y);
      b += square(f[u].z) + square(f[u].w);
    }
  }
  for (; v < n4; v += THREADS) {
    const float4 f = ld4(p + 4 * v);
    a += square(f.x) + square(f.y);
    b += square(f.z) + square(f.w);
  }
  if (threadIdx.x < n - 4 * n4) b += square(p[4 * n4 + threadIdx.x]);
}

__global__ void __launch_bounds__(1024) grad_norm_kernel(const __grid_constant__ NormTable t, double* __restrict__ sums) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const long long total = t.start[t.count], each = (total + gridDim.x - 1) / gridDim.x;
  long long e = blockIdx.x * each;
  const long long end = e + each < total ? e + each : total;
  double a = 0, b = 0;
  for (int k = e < end ? tensor_of(t, e) : 0; e < end; ++k) {
    const long long stop = t.start[k + 1] < end ? t.start[k + 1] : end;
    sum_squares<1024, 4>(t.g[k] + (e - t.start[k]), stop - e, a, b);
    e = stop;
  }
  __shared__ double part[32];
  a += b;
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x < 32) {
    a = part[threadIdx.x];
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (threadIdx.x == 0) sums[blockIdx.x] = a;
  }
}

constexpr int kScaleTensors = 192;
struct ScaleTable {
  float* g[kScaleTensors];
  long long start[kScaleTensors + 1];
  int count;
};

// Writes nothing where the gradients are under the limit: a factor of one changes no value.
__global__ void __launch_bounds__(512) scale_grads_kernel(const __grid_constant__ ScaleTable t, MtbClip clip) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const float factor = mtb_clip_factor<512>(clip);
  if (factor == 1.f) return;
  const long long total = t.start[t.count], each = (total + gridDim.x - 1) / gridDim.x;
  long long e = blockIdx.x * each;
  const long long end = e + each < total ? e + each : total;
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.start[mid] <= e) lo = mid; else hi = mid - 1;
  }
  for (int k = lo; e < end; ++k) {
    const long long stop = t.start[k + 1] < end ? t.start[k + 1] : end;
    float* p = t.g[k] + (e - t.start[k]);
    long long n = stop - e, head = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) / 4 % 4;
    if (head > n) head = n;
    if (threadIdx.x < head) p[threadIdx.x] *= factor;
    p += head;
    n -= head;
    for (long long v = threadIdx.x; v < n / 4; v += 512) {
      float4 f = ld4(p + 4 * v);
      f.x *= factor; f.y *= factor; f.z *= factor; f.w *= factor;
      st4(p + 4 * v, f);
    }
    if (threadIdx.x < n % 4) p[n / 4 * 4 + threadIdx.x] *= factor;
    e = stop;
  }
}

int norm_blocks() { return mtb_sm_count(); }

}  // namespace

// How many partial sums mtb_grad_norm_f32 leaves for `count` tensors.
MTB_API int mtb_grad_norm_sums(int count) { return count <= 0 ? 0 : mtb_div_up(count, kNormTensors) * norm_blocks(); }

MTB_API int mtb_grad_norm_f32(int count, const float* const* grads, const long long* sizes, double* sums, void* stream) {
  MTB_REQUIRE(count >= 0 && (count == 0 || (grads && sizes && sums)), "grad_norm: bad arguments");
  for (int base = 0; base < count; base += kNormTensors) {
    NormTable t;
    t.count = count - base < kNormTensors ? count - base : kNormTensors;
    t.start[0] = 0;
    for (int k = 0; k < t.count; ++k) {
      MTB_REQUIRE(sizes[base + k] >= 0 && (grads[base + k] || sizes[base + k] == 0), "grad_norm: null tensor %d", base + k);
      t.g[k] = grads[base + k];
      t.start[k + 1] = t.start[k] + sizes[base + k];
    }
    MTB_LAUNCH(grad_norm_kernel, norm_blocks(), 1024, 0, (cudaStream_t)stream, t, sums + base / kNormTensors * norm_blocks());
  }
  return MTB_OK;
}

MTB_API int mtb_clip_grads_f32(int count, float* const* grads, const long long* sizes, const double* sums, int nsums, double max_norm, float* norm,
                               void* stream) {
  MTB_REQUIRE(count > 0 && grads && sizes && sums && nsums > 0 && norm, "clip_grads: bad arguments");
  for (int base = 0; base < count; base += kScaleTensors) {
    ScaleTable t;
    t.count = max_norm < 0 ? 0 : count - base < kScaleTensors ? count - base : kScaleTensors;
    t.start[0] = 0;
    for (int k = 0; k < t.count; ++k) {
      MTB_REQUIRE(sizes[base + k] >= 0 && (grads[base + k] || sizes[base + k] == 0), "clip_grads: null tensor %d", base + k);
      t.g[k] = grads[base + k];
      t.start[k + 1] = t.start[k] + sizes[base + k];
    }
    const MtbClip clip{sums, nsums, 1.0, max_norm, base == 0 ? norm : nullptr};
    MTB_LAUNCH(scale_grads_kernel, mtb_stream_grid((t.start[t.count] + 3) / 4, 512, 4), 512, 0, (cudaStream_t)stream, t, clip);
    if (max_norm < 0) break;
  }
  return MTB_OK;
}
