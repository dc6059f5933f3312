// AdamW over many tensors at once, with moments in 32 or in 8 bits:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps).
// The step t lies in device memory, so that a captured update counts on when it is replayed.
//
// Moments in 8 bits.  A block of 256 values of one tensor shares a scale, the exponent of its largest value (one byte, that of a float32: 0 a block of
// zeros, 255 a block that a value which is not finite entered, all of which reads NaN).  A first moment is a sign, 4 bits of exponent and 3 of fraction, a
// second moment 5 bits of exponent and 3 of fraction; the highest exponent stands for twice the scale, so that rounding up the largest value needs no care, and
// what lies under the lowest is in equal steps, as in any float.  Scaled so that the lowest exponents meet, a code is the upper bits of a float32.  A code is rounded up as often as
// the value is near the upper neighbour, by 16 random bits: to the nearest, the thousandth part by which a step moves a second moment would never
// leave a step of an eighth.  The bits follow from seed, tensor, step and place.  A second moment that is not zero never becomes zero, which would
// make the next update a division by eps.
// So that every path rounds alike: b1 and b2 have 20 bits, their product with a moment (4 bits) is then a float32, and one FMA rounds the new moment once;
// v adds the square of h = sqrt(1 - b2) g, rounded to float32.  The update takes the moments as they are before they are rounded to 8 bits.
#include <cmath>
#include <vector>

#include "clip.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 192;
constexpr int kChunk = 2048;   // elements of a CTA with moments in 32 bits
constexpr int kChunk8 = 4096;  // and in 8: two blocks a warp
constexpr int kBlock = 256;
constexpr int kSteps = 256;

struct Hyper {
  float lr, b1, b2, c1, c2, eps, keep, grad_scale;  // c1 = 1 - b1, c2 = 1 - b2 (8 bits: its root), keep = 1 - lr wd
};

// What a step makes of t, for every counter of a call.
struct Corrections {
  float step_size, root;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  unsigned t, unused;
};

struct StepTable {
  long long* step[kSteps];
  int count;
};
__global__ void __launch_bounds__(256) adamw_begin_kernel(const __grid_constant__ StepTable t, double lr, double b1, double b2, Corrections* __restrict__ out) {
  mtb_launch_dependents();
  mtb_wait_prior();
  if ((int)threadIdx.x >= t.count) return;
  const long long step = *t.step[threadIdx.x] + 1;
  *t.step[threadIdx.x] = step;
  out[threadIdx.x] = Corrections{(float)(lr / (1.0 - pow(b1, (double)step))), (float)(1.0 / sqrt(1.0 - pow(b2, (double)step))), (unsigned)step, 0u};
}

template <class M>
struct Table {
  float* p[kTensors];
  const float* g[kTensors];
  M* m[kTensors];  // 32 bits: the first moments; 8 bits: [block][first 256 | second 256]
  M* v[kTensors];  // 32 bits: the second moments; 8 bits: [block][scale of the first, of the second]
  long long n[kTensors];
  int chunk_start[kTensors + 1];  // CTA b works on tensor k with chunk_start[k] <= b < chunk_start[k + 1]
  unsigned short slot[kTensors];  // which corrections
  unsigned key[kTensors];
  int count;
};

template <class M>
__device__ __forceinline__ int tensor_of(const Table<M>& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {  // last k with chunk_start[k] <= chunk
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunk_start[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void update(float& p, float m, float v, const Hyper& h, const Corrections& c) {
  p = p * h.keep - c.step_size * m / (sqrtf(v) * c.root + h.eps);
}

__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<float> t, Hyper h, const Corrections* __restrict__ corrections, MtbClip clip) {
  mtb_launch_dependents();
  mtb_wait_prior();
  if (clip.sums) h.grad_scale *= mtb_clip_factor<kThreads>(clip);
  const int k = tensor_of(t, blockIdx.x);
  const long long e = (long long)((int)blockIdx.x - t.chunk_start[k]) * kChunk, left = t.n[k] - e;
  const int n = left < kChunk ? (int)left : kChunk;
  const Corrections c = corrections[t.slot[k]];
  float *p = t.p[k] + e, *m = t.m[k] + e, *v = t.v[k] + e;
  const float* g = t.g[k] + e;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float gg = g[i] * h.grad_scale;
    m[i] = h.b1 * m[i] + h.c1 * gg;
    v[i] = h.b2 * v[i] + h.c2 * gg * gg;
    update(p[i], m[i], v[i], h, c);
  }
}

// 32 bits to 32 bits, each of which depends on all: multiplications by fractions of square roots (of 2 and of 3), the upper bits folded into the lower ones.
__host__ __device__ __forceinline__ unsigned mix(unsigned x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
constexpr unsigned kGolden = 0x9E3779B1u;

// What a block's scale stands for, and its reciprocal.
__device__ __forceinline__ float unit_of(unsigned scale) { return scale == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float(scale << 23); }
__device__ __forceinline__ float per_unit(unsigned scale) { return __uint_as_float(scale >= 254 ? 0x00400000u : (254u - scale) << 23); }
// The scale for values of which the largest has these bits.
__device__ __forceinline__ unsigned scale_of(unsigned bits) { return bits == 0 ? 0u : bits < 0x00800000u ? 1u : bits >> 23; }

__device__ __forceinline__ float decode_first(unsigned code, float unit) {
  return __uint_as_float((code & 0x7Fu) << 20 | (code & 0x80u) << 24) * 0x1p113f * unit;
}
__device__ __forceinline__ float decode_second(unsigned code, float unit) { return __uint_as_float(code << 20) * 0x1p97f * unit; }
// random: 16 bits.  The reciprocal's product with a value is exact where it is not far under the lowest code.
__device__ __forceinline__ unsigned encode_first(float m, float per, unsigned random) {
  return (__float_as_uint(fabsf(m) * per * 0x1p-113f) + (random << 4) + 8u) >> 20 | (__float_as_uint(m) >> 31) << 7;
}
__device__ __forceinline__ unsigned encode_second(float v, float per, unsigned random) {
  const unsigned code = (__float_as_uint(v * per * 0x1p-97f) + (random << 4) + 8u) >> 20;
  return v > 0.f && code == 0 ? 1u : code;
}

// A warp a block, 8 values a lane: 4 at 4 lane, 4 at 128 + 4 lane.
__global__ void __launch_bounds__(kThreads) adamw8_kernel(const __grid_constant__ Table<unsigned char> t, Hyper h, const Corrections* __restrict__ corrections, MtbClip clip) {
  mtb_launch_dependents();
  mtb_wait_prior();
  if (clip.sums) h.grad_scale *= mtb_clip_factor<kThreads>(clip);
  const int k = tensor_of(t, blockIdx.x), lane = threadIdx.x & 31;
  const Corrections c = corrections[t.slot[k]];
  const unsigned key = mix(t.key[k] + c.t);
  for (int turn = threadIdx.x >> 5; turn < kChunk8 / kBlock; turn += kThreads / 32) {
    const long long block = (long long)((int)blockIdx.x - t.chunk_start[k]) * (kChunk8 / kBlock) + turn, e = block * kBlock, left = t.n[k] - e;
    if (left <= 0) return;
    const int n = left < kBlock ? (int)left : kBlock;
    float* p = t.p[k] + e;
    const float* g = t.g[k] + e;
    unsigned char *codes = t.m[k] + block * 2 * kBlock, *scales = t.v[k] + block * 2;
    const float unit_m = unit_of(scales[0]), unit_v = unit_of(scales[1]);
    float m[8], v[8];
    unsigned most_m = 0, most_v = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const unsigned cm = *(const unsigned*)(codes + 128 * u + 4 * lane), cv = *(const unsigned*)(codes + kBlock + 128 * u + 4 * lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 128 * u + 4 * lane + j;
        float &mm = m[4 * u + j], &vv = v[4 * u + j];
        mm = vv = 0.f;
        if (i < n) {
          const float gg = g[i] * h.grad_scale, root = h.c2 * gg;
          mm = __fmaf_rn(h.c1, gg, __fmul_rn(h.b1, decode_first(cm >> 8 * j & 0xFFu, unit_m)));
          vv = __fmaf_rn(root, root, __fmul_rn(h.b2, decode_second(cv >> 8 * j & 0xFFu, unit_v)));
          update(p[i], mm, vv, h, c);
        }
        most_m = max(most_m, __float_as_uint(mm) & 0x7FFFFFFFu);
        most_v = max(most_v, __float_as_uint(vv) & 0x7FFFFFFFu);
      }
    }
    const unsigned scale_m = scale_of(__reduce_max_sync(0xFFFFFFFFu, most_m)), scale_v = scale_of(__reduce_max_sync(0xFFFFFFFFu, most_v));
    const float per_m = per_unit(scale_m), per_v = per_unit(scale_v);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      unsigned cm = 0, cv = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned r = mix(key + ((unsigned)e + 128 * u + 4 * lane + j) * kGolden);
        cm |= encode_first(m[4 * u + j], per_m, r >> 16) << 8 * j;
        cv |= encode_second(v[4 * u + j], per_v, r & 0xFFFFu) << 8 * j;
      }
      *(unsigned*)(codes + 128 * u + 4 * lane) = scale_m == 255 ? 0u : cm;
      *(unsigned*)(codes + kBlock + 128 * u + 4 * lane) = scale_v == 255 ? 0u : cv;
    }
    if (lane == 0) *(unsigned short*)scales = (unsigned short)(scale_m | scale_v << 8);
  }
}

struct MomentsTable {
  const unsigned char *codes[kTensors], *scales[kTensors];
  float *m[kTensors], *v[kTensors];
  long long n[kTensors];
  int chunk_start[kTensors + 1];
  int count;
};
__global__ void __launch_bounds__(kThreads) adamw8_moments_kernel(const __grid_constant__ MomentsTable t) {
  mtb_launch_dependents();
  mtb_wait_prior();
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunk_start[mid] <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const int k = lo;
  const long long e = (long long)((int)blockIdx.x - t.chunk_start[k]) * kChunk8;
  for (long long i = e + threadIdx.x; i < e + kChunk8 && i < t.n[k]; i += kThreads) {
    const long long block = i / kBlock;
    const unsigned char *codes = t.codes[k] + block * 2 * kBlock + i % kBlock, *scales = t.scales[k] + 2 * block;
    t.m[k][i] = decode_first(codes[0], unit_of(scales[0]));
    t.v[k][i] = decode_second(codes[kBlock], unit_of(scales[1]));
  }
}

// What `params` says of a tensor.
struct Tensor {
  float* p;
  const float* g;
  void *m, *v;
  long long* step;
};
Tensor tensor_at(void* const* params, int k) {
  void* const* a = params + 5 * (long long)k;
  return Tensor{(float*)a[0], (const float*)a[1], a[2], a[3], (long long*)a[4]};
}

// Counts the steps of the call's tensors, each counter once, and leaves which of the corrections a tensor takes.
int begin(int count, void* const* params, double lr, double b1, double b2, Corrections* out, std::vector<unsigned short>& slots, cudaStream_t st) {
  std::vector<long long*> distinct;
  slots.resize(count);
  for (int k = 0; k < count; ++k) {
    long long* step = tensor_at(params, k).step;
    size_t at = k ? slots[k - 1] : 0;  // mostly the one before
    if (k == 0 || distinct[at] != step)
      for (at = 0; at < distinct.size() && distinct[at] != step;) ++at;
    if (at == distinct.size()) distinct.push_back(step);
    MTB_REQUIRE(at < 65536, "adamw: more than 65536 step counters in one call");
    slots[k] = (unsigned short)at;
  }
  for (size_t base = 0; base < distinct.size(); base += kSteps) {
    StepTable t;
    t.count = (int)(distinct.size() - base < kSteps ? distinct.size() - base : kSteps);
    for (int i = 0; i < t.count; ++i) t.step[i] = distinct[base + i];
    MTB_LAUNCH(adamw_begin_kernel, 1, 256, 0, st, t, lr, b1, b2, out + base);
  }
  return MTB_OK;
}

bool moments_aligned(const void* codes, const void* scales) { return mtb_aligned16(codes) && (reinterpret_cast<uintptr_t>(scales) & 1u) == 0; }

bool fine(double lr, double b1, double b2, double eps, double weight_decay) {
  return lr >= 0 && b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1 && eps >= 0 && weight_decay >= 0;
}

// stride: numbers in `sizes` a tensor.
template <class M, class K>
int run(const char* name, K kernel, int count, void* const* params, const long long* sizes, int stride, const std::vector<unsigned short>& slots, int chunk, const Hyper& h,
        const Corrections* corrections, MtbClip clip, cudaStream_t st) {
  for (int base = (count - 1) / kTensors * kTensors; base >= 0; base -= kTensors) {  // backwards: what the norm read last is still in L2
    Table<M> t;
    t.count = count - base < kTensors ? count - base : kTensors;
    long long chunks = 0;
    for (int k = 0; k < t.count; ++k) {
      const Tensor a = tensor_at(params, base + k);
      const long long* size = sizes + (long long)stride * (base + k);
      t.p[k] = a.p;
      t.g[k] = a.g;
      t.m[k] = (M*)a.m;
      t.v[k] = (M*)a.v;
      t.n[k] = size[0];
      t.slot[k] = slots[base + k];
      t.key[k] = stride > 1 ? mix((unsigned)size[1]) : 0;
      t.chunk_start[k] = (int)chunks;
      chunks += (t.n[k] + chunk - 1) / chunk;
      MTB_REQUIRE(chunks < (1LL << 30), "%s: too many elements in one call", name);
    }
    t.chunk_start[t.count] = (int)chunks;
    if (chunks == 0 && clip.norm) chunks = 1;  // for the norm
    if (chunks == 0) continue;
    MTB_LAUNCH(kernel, dim3((unsigned)chunks), kThreads, 0, st, t, h, corrections, clip);
    MTB_LAUNCH_CHECK(name);
    clip.norm = nullptr;  // left by the first launch
  }
  return MTB_OK;
}

}  // namespace

MTB_API long long mtb_adamw_scratch_bytes(int count) { return (long long)(count < 1 ? 1 : count) * (long long)sizeof(Corrections); }

MTB_API int mtb_adamw_f32(int count, void* const* params, const long long* sizes, double lr, double beta1, double beta2, double eps, double weight_decay, double grad_scale,
                          const double* sums, int nsums, double max_norm, float* norm, void* scratch, void* stream) {
  MTB_REQUIRE(count >= 0 && (count == 0 || (params && sizes && scratch)), "adamw: bad arguments");
  MTB_REQUIRE(fine(lr, beta1, beta2, eps, weight_decay), "adamw: bad hyper-parameters");
  MTB_REQUIRE(!sums || (nsums > 0 && max_norm >= 0), "adamw: bad sums of squares");
  for (int k = 0; k < count; ++k) {
    const Tensor a = tensor_at(params, k);
    MTB_REQUIRE(a.step && sizes[k] >= 0 && (sizes[k] == 0 || (a.p && a.g && a.m && a.v)), "adamw: null tensor %d", k);
  }
  std::vector<unsigned short> slots;
  if (int rc = begin(count, params, lr, beta1, beta2, (Corrections*)scratch, slots, (cudaStream_t)stream)) return rc;
  const Hyper h{(float)lr, (float)beta1, (float)beta2, (float)(1 - beta1), (float)(1 - beta2), (float)eps, (float)(1 - lr * weight_decay), (float)grad_scale};
  return run<float>("adamw_kernel", adamw_kernel, count, params, sizes, 1, slots, kChunk, h, (const Corrections*)scratch, MtbClip{sums, nsums, grad_scale, max_norm, norm},
                    (cudaStream_t)stream);
}

MTB_API int mtb_adamw8_f32(int count, void* const* params, const long long* sizes, double lr, double beta1, double beta2, double eps, double weight_decay, double grad_scale,
                           const double* sums, int nsums, double max_norm, float* norm, void* scratch, void* stream) {
  MTB_REQUIRE(count >= 0 && (count == 0 || (params && sizes && scratch)), "adamw8: bad arguments");
  const double b1 = std::round(beta1 * (1 << 20)) / (1 << 20), b2 = std::round(beta2 * (1 << 20)) / (1 << 20);
  MTB_REQUIRE(fine(lr, beta1, beta2, eps, weight_decay) && b1 < 1 && b2 < 1, "adamw8: bad hyper-parameters (betas count with 20 bits)");
  MTB_REQUIRE(!sums || (nsums > 0 && max_norm >= 0), "adamw8: bad sums of squares");
  for (int k = 0; k < count; ++k) {
    const Tensor a = tensor_at(params, k);
    MTB_REQUIRE(a.step && sizes[2 * k] >= 0 && (sizes[2 * k] == 0 || (a.p && a.g && a.m && a.v)), "adamw8: null tensor %d", k);
    MTB_REQUIRE(moments_aligned(a.m, a.v), "adamw8: moments of tensor %d begin off 16 bytes, or scales off 2", k);
  }
  std::vector<unsigned short> slots;
  if (int rc = begin(count, params, lr, b1, b2, (Corrections*)scratch, slots, (cudaStream_t)stream)) return rc;
  const Hyper h{(float)lr, (float)b1, (float)b2, (float)(1 - b1), (float)std::sqrt(1 - b2), (float)eps, (float)(1 - lr * weight_decay), (float)grad_scale};
  return run<unsigned char>("adamw8_kernel", adamw8_kernel, count, params, sizes, 2, slots, kChunk8, h, (const Corrections*)scratch,
                            MtbClip{sums, nsums, grad_scale, max_norm, norm}, (cudaStream_t)stream);
}

MTB_API int mtb_adamw8_moments_f32(int count, void* const* params, const long long* sizes, void* stream) {
  MTB_REQUIRE(count >= 0 && (count == 0 || (params && sizes)), "adamw8_moments: bad arguments");
  for (int base = 0; base < count; base += kTensors) {
    MomentsTable t;
    t.count = count - base < kTensors ? count - base : kTensors;
    long long chunks = 0;
    for (int k = 0; k < t.count; ++k) {
      void* const* a = params + 4 * (long long)(base + k);
      const long long size = sizes[base + k];
      MTB_REQUIRE(size >= 0 && (size == 0 || (a[0] && a[1] && a[2] && a[3])), "adamw8_moments: null tensor %d", base + k);
      MTB_REQUIRE(moments_aligned(a[0], a[1]), "adamw8_moments: moments of tensor %d begin off 16 bytes, or scales off 2", base + k);
      t.codes[k] = (const unsigned char*)a[0];
      t.scales[k] = (const unsigned char*)a[1];
      t.m[k] = (float*)a[2];
      t.v[k] = (float*)a[3];
      t.n[k] = size;
      t.chunk_start[k] = (int)chunks;
      chunks += (size + kChunk8 - 1) / kChunk8;
      MTB_REQUIRE(chunks < (1LL << 30), "adamw8_moments: too many elements in one call");
    }
    t.chunk_start[t.count] = (int)chunks;
    if (chunks == 0) continue;
    MTB_LAUNCH(adamw8_moments_kernel, dim3((unsigned)chunks), kThreads, 0, (cudaStream_t)stream, t);
    MTB_LAUNCH_CHECK("adamw8_moments_kernel");
  }
  return MTB_OK;
}
