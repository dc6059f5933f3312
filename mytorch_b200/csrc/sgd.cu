// SGD with momentum / dampening / Nesterov / weight decay / maximize, per tensor and as a
// multi-tensor launch (pointer table passed by value in kernel parameters, so a whole model
// updates in a few launches and the launch can be captured in a CUDA graph).
#include "clip.cuh"

namespace {

struct SgdHyper {
  float lr, weight_decay, momentum, one_minus_dampening, grad_scale;
  int nesterov, maximize, first;
};

__device__ __forceinline__ void sgd_update(float& p, float g, float& buf, const SgdHyper& h) {
  g = (h.maximize ? -g : g) * h.grad_scale + h.weight_decay * p;
  buf = h.first ? g : (h.momentum * buf + h.one_minus_dampening * g);
  g = h.nesterov ? (g + h.momentum * buf) : buf;
  p -= g * h.lr;
}

__device__ __forceinline__ void sgd_span(float* p, const float* g, float* buf, long long n, const SgdHyper& h, long long tid, long long nthreads) {
  bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(buf)) & 15u) == 0;
  long long n4 = vec ? n / 4 : 0;
  for (long long v = tid; v < n4; v += nthreads) {
    float4 pp = ld4(p + 4 * v), gg = ld4(g + 4 * v), bb = h.first ? make_float4(0, 0, 0, 0) : ld4(buf + 4 * v);
    sgd_update(pp.x, gg.x, bb.x, h);
    sgd_update(pp.y, gg.y, bb.y, h);
    sgd_update(pp.z, gg.z, bb.z, h);
    sgd_update(pp.w, gg.w, bb.w, h);
    st4(p + 4 * v, pp);
    st4(buf + 4 * v, bb);
  }
  for (long long t = 4 * n4 + tid; t < n; t += nthreads) {
    float pp = p[t], bb = h.first ? 0.f : buf[t];
    sgd_update(pp, g[t], bb, h);
    p[t] = pp;
    buf[t] = bb;
  }
}

// sgd_span over at most VECTORS * 4 * 256 elements, the gradients times the factor that clips them (CTAs of 256 threads): everything is on its way
// while the CTA adds up the norm.  The gradients were read just now, and some are still in L2: what is used once is marked to leave it first.
// Bound by memory.  Norm and update of 161 tensors, 25.6 M elements, one step after the other: 93.5 us, 5.5 TB/s of the 20 bytes an element that an update
// must move; the update without a norm 81 us.  Measured when the norm took 4 us longer: 97.7; without the marks 100.9; chunks of 4096 elements 99.0, of 1024
// 103.9; the factor before the loads and the chunks forwards 104.
template <int VECTORS>
__device__ __forceinline__ void sgd_span_clipped(float* p, const float* g, float* buf, int n, SgdHyper h, const MtbClip& clip) {
  if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(buf)) & 15u) != 0) {
    h.grad_scale *= mtb_clip_factor<256>(clip);
    sgd_span(p, g, buf, n, h, threadIdx.x, 256);
    return;
  }
  float4 pp[VECTORS], gg[VECTORS], bb[VECTORS];
#pragma unroll
  for (int u = 0; u < VECTORS; ++u) {
    const int v = threadIdx.x + u * 256;
    bb[u] = make_float4(0, 0, 0, 0);
    if (v < n / 4) {
      gg[u] = __ldcs((const float4*)g + v);
      pp[u] = __ldcs((const float4*)p + v);
      if (!h.first) bb[u] = __ldcs((const float4*)buf + v);
    }
  }
  h.grad_scale *= mtb_clip_factor<256>(clip);
#pragma unroll
  for (int u = 0; u < VECTORS; ++u) {
    const int v = threadIdx.x + u * 256;
    if (v < n / 4) {
      sgd_update(pp[u].x, gg[u].x, bb[u].x, h);
      sgd_update(pp[u].y, gg[u].y, bb[u].y, h);
      sgd_update(pp[u].z, gg[u].z, bb[u].z, h);
      sgd_update(pp[u].w, gg[u].w, bb[u].w, h);
      __stcs((float4*)p + v, pp[u]);
      __stcs((float4*)buf + v, bb[u]);
    }
  }
  for (int t = n / 4 * 4 + threadIdx.x; t < n; t += 256) {
    float q = p[t], b = h.first ? 0.f : buf[t];
    sgd_update(q, g[t], b, h);
    p[t] = q;
    buf[t] = b;
  }
}

__global__ void __launch_bounds__(256) sgd_kernel(float* p, const float* g, float* buf, long long n, SgdHyper h) {
  mtb_launch_dependents();
  mtb_wait_prior();
  sgd_span(p, g, buf, n, h, blockIdx.x * (long long)blockDim.x + threadIdx.x, (long long)gridDim.x * blockDim.x);
}

constexpr int kMaxTensors = 96;
constexpr int kSgdChunk = 4096;  // elements per CTA: four float4 per thread and array in flight
constexpr int kClipChunk = 2048;  // of the clipped update: two float4 per thread and array
struct SgdTable {
  float* p[kMaxTensors];
  const float* g[kMaxTensors];
  float* buf[kMaxTensors];
  long long n[kMaxTensors];
  int first[kMaxTensors];
  int chunk_start[kMaxTensors + 1];  // CTA b works on tensor k with chunk_start[k] <= b < chunk_start[k + 1]
  int count;
};

// One CTA per chunk of kSgdChunk elements of one tensor (a model has a few large tensors and dozens of
// tiny ones: a grid of tensors x the largest tensor's chunks would be mostly empty CTAs).
// CLIP: the gradients are multiplied by the factor that clips them, which nothing writes back; the chunks are taken backwards.
template <bool CLIP>
__global__ void __launch_bounds__(256) sgd_multi_kernel(const __grid_constant__ SgdTable t, SgdHyper h, MtbClip clip) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int chunk = CLIP ? t.chunk_start[t.count] - 1 - (int)blockIdx.x : (int)blockIdx.x;
  if (CLIP && chunk < 0) {  // nothing to update: one CTA leaves the norm
    mtb_clip_factor<256>(clip);
    return;
  }
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {  // last k with chunk_start[k] <= chunk
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunk_start[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  const int k = lo;
  const long long e0 = (long long)(chunk - t.chunk_start[k]) * (CLIP ? kClipChunk : kSgdChunk);
  const long long left = t.n[k] - e0;
  h.first = t.first[k];
  if (CLIP) sgd_span_clipped<kClipChunk / 1024>(t.p[k] + e0, t.g[k] + e0, t.buf[k] + e0, left < kClipChunk ? (int)left : kClipChunk, h, clip);
  else sgd_span(t.p[k] + e0, t.g[k] + e0, t.buf[k] + e0, left < kSgdChunk ? left : kSgdChunk, h, threadIdx.x, blockDim.x);
}

// Gather `count` gradient tensors into one flat buffer, scaling on the way.
struct PackTable {
  const float* src[kMaxTensors];
  long long off[kMaxTensors];
  long long n[kMaxTensors];
  int count;
};
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackTable t, float* dst, float scale) {
  mtb_launch_dependents();
  mtb_wait_prior();
  int k = blockIdx.y;
  if (k >= t.count) return;
  long long n = t.n[k];
  const float* s = t.src[k];
  float* d = dst + t.off[k];
  long long stride = (long long)gridDim.x * blockDim.x;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += stride) d[i] = s[i] * scale;
}

}  // namespace

// One parameter tensor. grad_scale multiplies the gradient first (1/world_size under data
// parallelism, 1 otherwise). is_first != 0: the momentum buffer is initialised to g.
MTB_API int mtb_sgd_f32(float* param, const float* grad, float* momentum_buffer, long long n, int is_first, double lr, double weight_decay,
                        double momentum, double dampening, int nesterov, int maximize, double grad_scale, void* stream) {
  MTB_REQUIRE(n >= 0 && ((param && grad && momentum_buffer) || n == 0), "sgd: bad arguments");
  if (n == 0) return MTB_OK;
  SgdHyper h{(float)lr, (float)weight_decay, (float)momentum, (float)(1.0 - dampening), (float)grad_scale, nesterov, maximize, is_first};
  MTB_LAUNCH(sgd_kernel, mtb_stream_grid((n + 3) / 4, 256), 256, 0, (cudaStream_t)stream, param, grad, momentum_buffer, n, h);
  MTB_LAUNCH_CHECK("sgd_kernel");
  return MTB_OK;
}

static int sgd_multi(int count, float* const* params, const float* const* grads, float* const* momentum_buffers, const long long* sizes, const int* is_first,
                     double lr, double weight_decay, double momentum, double dampening, int nesterov, int maximize, double grad_scale, MtbClip clip,
                     void* stream) {
  MTB_REQUIRE(count >= 0 && (count == 0 || (params && grads && momentum_buffers && sizes && is_first)), "sgd_multi: bad arguments");
  SgdHyper h{(float)lr, (float)weight_decay, (float)momentum, (float)(1.0 - dampening), (float)grad_scale, nesterov, maximize, 0};
  const int chunk = clip.sums ? kClipChunk : kSgdChunk, last = count > 0 ? (count - 1) / kMaxTensors * kMaxTensors : -1;
  for (int turn = 0; turn <= last; turn += kMaxTensors) {
    const int base = clip.sums ? last - turn : turn;
    SgdTable t;
    t.count = count - base < kMaxTensors ? count - base : kMaxTensors;
    long long chunks = 0;
    for (int k = 0; k < t.count; ++k) {
      MTB_REQUIRE(sizes[base + k] >= 0 && params[base + k] && grads[base + k] && momentum_buffers[base + k], "sgd_multi: null tensor %d", base + k);
      t.p[k] = params[base + k];
      t.g[k] = grads[base + k];
      t.buf[k] = momentum_buffers[base + k];
      t.n[k] = sizes[base + k];
      t.first[k] = is_first[base + k];
      t.chunk_start[k] = (int)chunks;
      chunks += (t.n[k] + chunk - 1) / chunk;
      MTB_REQUIRE(chunks < (1LL << 30), "sgd_multi: too many elements in one call");
    }
    t.chunk_start[t.count] = (int)chunks;
    if (chunks == 0 && clip.norm) chunks = 1;  // for the norm
    if (chunks == 0) continue;
    dim3 grid((unsigned int)chunks);
    MTB_LAUNCH(clip.sums ? sgd_multi_kernel<true> : sgd_multi_kernel<false>, grid, 256, 0, (cudaStream_t)stream, t, h, clip);
    MTB_LAUNCH_CHECK("sgd_multi_kernel");
    clip.norm = nullptr;  // left by the first launch
  }
  return MTB_OK;
}

// `count` parameter tensors with shared hyper-parameters. Host arrays of device pointers.
MTB_API int mtb_sgd_multi_f32(int count, float* const* params, const float* const* grads, float* const* momentum_buffers, const long long* sizes,
                              const int* is_first, double lr, double weight_decay, double momentum, double dampening, int nesterov,
                              int maximize, double grad_scale, void* stream) {
  return sgd_multi(count, params, grads, momentum_buffers, sizes, is_first, lr, weight_decay, momentum, dampening, nesterov, maximize, grad_scale, MtbClip{}, stream);
}

// The same with the gradients clipped to max_norm on the way, by the sums that mtb_grad_norm_f32 left of all gradients.
MTB_API int mtb_sgd_multi_clipped_f32(int count, float* const* params, const float* const* grads, float* const* momentum_buffers, const long long* sizes,
                                      const int* is_first, double lr, double weight_decay, double momentum, double dampening, int nesterov, int maximize,
                                      double grad_scale, const double* sums, int nsums, double max_norm, float* norm, void* stream) {
  MTB_REQUIRE(sums && nsums > 0 && max_norm >= 0, "sgd_multi_clipped: bad arguments");
  return sgd_multi(count, params, grads, momentum_buffers, sizes, is_first, lr, weight_decay, momentum, dampening, nesterov, maximize, grad_scale,
                   MtbClip{sums, nsums, grad_scale, max_norm, norm}, stream);
}

// dst[offsets[k] : offsets[k] + sizes[k]] = scale * srcs[k][:] for k < count.
MTB_API int mtb_pack_scale_f32(int count, const float* const* srcs, const long long* offsets, const long long* sizes, float* dst, double scale,
                               void* stream) {
  MTB_REQUIRE(count >= 0 && (count == 0 || (srcs && offsets && sizes && dst)), "pack_scale: bad arguments");
  for (int base = 0; base < count; base += kMaxTensors) {
    PackTable t;
    t.count = count - base < kMaxTensors ? count - base : kMaxTensors;
    long long maxn = 1;
    for (int k = 0; k < t.count; ++k) {
      t.src[k] = srcs[base + k];
      t.off[k] = offsets[base + k];
      t.n[k] = sizes[base + k];
      if (t.n[k] > maxn) maxn = t.n[k];
    }
    int gx = mtb_div_up(maxn, 256 * 4);
    int cap = mtb_sm_count() * 4;
    if (gx > cap) gx = cap;
    if (gx < 1) gx = 1;
    MTB_LAUNCH(pack_kernel, dim3(gx, t.count), 256, 0, (cudaStream_t)stream, t, dst, (float)scale);
    MTB_LAUNCH_CHECK("pack_kernel");
  }
  return MTB_OK;
}
