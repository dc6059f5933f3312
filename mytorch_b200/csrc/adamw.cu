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
constexpr int kBlock = 256;
constexpr int kChunk = 2048;  // elements of a CTA: eight a thread, all of whose loads are on their way at once; of 8 bits a block a warp
constexpr int kSteps = 256;

struct Hyper {
  float b1, b2, c1, c2, eps, decay;  // c1 = 1 - b1, c2 = 1 - b2 (8 bits: its root), decay = lr wd: as 1 - lr wd it would lose all but a bit or two where it is a millionth
};

// What a step makes of t, for every counter of a call, and what multiplies the gradients.
struct alignas(16) Corrections {
  float step_size, root;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  unsigned t;
  float grad_scale;
};

struct StepTable {
  long long* step[kSteps];
  int count;
};
// One CTA in front of the update: no CTA of that waits for a sum.
__global__ void __launch_bounds__(256) adamw_begin_kernel(const __grid_constant__ StepTable t, double lr, double b1, double b2, float grad_scale, MtbClip clip,
                                                          Corrections* __restrict__ out) {
  mtb_launch_dependents();
  mtb_wait_prior();
  if (clip.sums) grad_scale *= mtb_clip_factor<256>(clip);
  if ((int)threadIdx.x >= t.count) return;
  const long long step = *t.step[threadIdx.x] + 1;
  *t.step[threadIdx.x] = step;
  out[threadIdx.x] = Corrections{(float)(lr / (1.0 - pow(b1, (double)step))), (float)(1.0 / sqrt(1.0 - pow(b2, (double)step))), (unsigned)step, grad_scale};
}

// Which tensor a CTA's chunk of elements is of: chunk b is one of tensor k with start[k] <= b < start[k + 1].  `near` says where to look from: bisection took a
// tenth of the instructions of the update in 8 bits.
template <int N>
struct Chunks {
  static constexpr int kNear = 128;
  int start[N + 1], count, shift;
  unsigned char near[kNear];  // of chunk j << shift

  int fill(int tensors, const long long* sizes, long long stride) {  // the number of chunks
    count = tensors;
    start[0] = 0;
    for (int k = 0; k < count; ++k) start[k + 1] = start[k] + (int)((sizes[stride * k] + kChunk - 1) / kChunk);
    shift = 0;
    while (start[count] >> shift >= kNear) ++shift;
    for (int j = 0, k = 0; j < kNear; ++j) {
      while (k + 1 < count && start[k + 1] <= (long long)j << shift) ++k;
      near[j] = (unsigned char)k;
    }
    return start[count];
  }
  __device__ __forceinline__ int tensor(int chunk) const {
    int k = near[chunk >> shift];
    while (start[k + 1] <= chunk) ++k;
    return k;
  }
};

// N tensors: a table of a few costs its launch less.
template <class M, int N>
struct Table {
  float* p[N];
  const float* g[N];
  M* m[N];  // 32 bits: the first moments; 8 bits: [block][first 256 | second 256]
  M* v[N];  // 32 bits: the second moments; 8 bits: [block][scale of the first, of the second]
  long long n[N];
  unsigned short slot[N];  // which corrections
  unsigned key[N];
  Chunks<N> chunks;
};

// What a parameter loses: decay and step, added up.  An infinite parameter counts as the largest, whose product with a decay of 0 is no NaN, and from which the difference stays infinite.
__device__ __forceinline__ float loss_of(float p, float decay, float step) {
  float finite;
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(finite) : "f"(p), "f"(3.402823466e38f));
  return fmaf(decay, finite, step);
}
// Root and quotient to 2^-22 of themselves, the step's share of which is far under a parameter's last place.  Decay and step are added up first, so that only their sum is
// rounded against the parameter.
__device__ __forceinline__ void update(float& p, float m, float v, const Hyper& h, const Corrections& c) {
  float root;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
  p -= loss_of(p, h.decay, __fdividef(c.step_size * m, fmaf(root, c.root, h.eps)));
}
__device__ __forceinline__ void moments(float g, float& m, float& v, const Hyper& h) {
  m = fmaf(h.b1, m, h.c1 * g);
  v = fmaf(h.b2, v, h.c2 * g * g);
}

// The chunks are taken backwards: what the norm read last is still in L2.  What is used once is marked to leave it first.
template <int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<float, N> t, Hyper h, const Corrections* __restrict__ corrections) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int chunk = (int)(gridDim.x - 1 - blockIdx.x), k = t.chunks.tensor(chunk);
  const long long e = (long long)(chunk - t.chunks.start[k]) * kChunk, left = t.n[k] - e;
  const int n = left < kChunk ? (int)left : kChunk;
  float *p = t.p[k] + e, *m = t.m[k] + e, *v = t.v[k] + e;
  const float* g = t.g[k] + e;
  const bool vectors = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0;
  if (vectors && n == kChunk) {
    float4 pp[2], gg[2], mm[2], vv[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = threadIdx.x + u * kThreads;
      gg[u] = __ldcs((const float4*)g + i);
      pp[u] = __ldcs((const float4*)p + i);
      mm[u] = __ldcs((const float4*)m + i);
      vv[u] = __ldcs((const float4*)v + i);
    }
    const Corrections c = corrections[t.slot[k]];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = threadIdx.x + u * kThreads;
      float* const ps[4] = {&pp[u].x, &pp[u].y, &pp[u].z, &pp[u].w};
      float* const ms[4] = {&mm[u].x, &mm[u].y, &mm[u].z, &mm[u].w};
      float* const vs[4] = {&vv[u].x, &vv[u].y, &vv[u].z, &vv[u].w};
      const float gs[4] = {gg[u].x, gg[u].y, gg[u].z, gg[u].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        moments(gs[j] * c.grad_scale, *ms[j], *vs[j], h);
        update(*ps[j], *ms[j], *vs[j], h, c);
      }
      __stcs((float4*)p + i, pp[u]);
      __stcs((float4*)m + i, mm[u]);
      __stcs((float4*)v + i, vv[u]);
    }
    return;
  }
  float pp[8], gg[8], mm[8], vv[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = threadIdx.x + u * kThreads;
    if (i < n) {
      gg[u] = __ldcs(g + i);
      pp[u] = __ldcs(p + i);
      mm[u] = __ldcs(m + i);
      vv[u] = __ldcs(v + i);
    }
  }
  const Corrections c = corrections[t.slot[k]];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = threadIdx.x + u * kThreads;
    if (i < n) {
      moments(gg[u] * c.grad_scale, mm[u], vv[u], h);
      update(pp[u], mm[u], vv[u], h, c);
      __stcs(p + i, pp[u]);
      __stcs(m + i, mm[u]);
      __stcs(v + i, vv[u]);
    }
  }
}

// 32 bits to 32 bits, each of which depends on all: multiplications by fractions of square roots (of 2 and of 3), the upper bits folded into the lower ones.
__host__ __device__ __forceinline__ unsigned mix(unsigned x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
constexpr unsigned kGolden = 0x9E3779B1u;

// What a block's scale stands for.
__device__ __forceinline__ float unit_of(unsigned scale) { return scale == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float(scale << 23); }
__device__ __forceinline__ float per_unit(unsigned scale) { return __uint_as_float(scale >= 254 ? 0x00400000u : (254u - scale) << 23); }  // its reciprocal
// The scale for values of which the largest is this; NaN where one is.
__device__ __forceinline__ unsigned scale_of(float most) {
  const unsigned bits = __float_as_uint(most) & 0x7FFFFFFFu;
  return bits == 0 ? 0u : bits < 0x00800000u ? 1u : bits >> 23;
}

// The float32 whose upper bits the code in byte B of a word is.
template <int B>
__device__ __forceinline__ float first_bits(unsigned w) { return __uint_as_float((unsigned)((int)(w << (24 - 8 * B)) >> 4) & 0x87F00000u); }
template <int B>
__device__ __forceinline__ float second_bits(unsigned w) { return __uint_as_float((B == 3 ? w >> 4 : w << (20 - 8 * B)) & 0x0FF00000u); }

// Power of two by which such a float is multiplied to be what the code stands for, or the other way; two products where one power does not fit a float32, which is
// the same for all of a block.  A scale of 0 stands for zeros, whatever they are multiplied by.
struct Powers {
  unsigned scale;
  int by;  // in one product: 2^(scale - 127 + by), or 2^(127 - scale - by)

  __device__ __forceinline__ bool two() const { return scale + by > 253; }
  __device__ __forceinline__ float up() const { return __uint_as_float((scale + by) << 23); }
  __device__ __forceinline__ float down() const { return __uint_as_float((254u - scale - by) << 23); }
  __device__ __forceinline__ float up_twice(float x) const { return x * __uint_as_float((unsigned)(127 + by) << 23) * unit_of(scale); }
  __device__ __forceinline__ float down_twice(float x) const { return x * per_unit(scale) * __uint_as_float((unsigned)(127 - by) << 23); }
};
constexpr int kFirst = 113, kSecond = 97;  // the highest exponents, 15 and 31 in a float32, are that of twice the unit

// A lane's eight values of a block, and their codes, a byte each in four words.  VECTORS: four at 4 lane and four at 128 + 4 lane, where parameters and gradients
// begin at 16 bytes; else at lane + 32 j, a value or a byte a load, which is as many bytes of memory.
template <bool VECTORS>
struct Lane {
  int lane;
  __device__ __forceinline__ int at(int j) const { return VECTORS ? 128 * (j / 4) + 4 * lane + j % 4 : lane + 32 * j; }
  __device__ __forceinline__ void values(const float* from, int n, float (&x)[8]) const {
    if (VECTORS && n == kBlock) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float4 f = __ldcs((const float4*)(from + 128 * u) + lane);
        x[4 * u] = f.x; x[4 * u + 1] = f.y; x[4 * u + 2] = f.z; x[4 * u + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = at(j) < n ? __ldcs(from + at(j)) : 0.f;
    }
  }
  __device__ __forceinline__ void put(float* to, int n, const float (&x)[8]) const {
    if (VECTORS && n == kBlock) {
#pragma unroll
      for (int u = 0; u < 2; ++u) __stcs((float4*)(to + 128 * u) + lane, make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at(j) < n) __stcs(to + at(j), x[j]);
    }
  }
  // Of VECTORS two words of four codes, else eight words of one.
  static constexpr int kWords = VECTORS ? 2 : 8;
  __device__ __forceinline__ void codes(const unsigned char* from, unsigned (&w)[8]) const {
#pragma unroll
    for (int u = 0; u < kWords; ++u) w[u] = VECTORS ? __ldcs((const unsigned*)(from + 128 * u) + lane) : (unsigned)__ldcs(from + at(u));
  }
  __device__ __forceinline__ void decode(const unsigned (&w)[8], unsigned scale, float (&x)[8], bool second) const {
    if (VECTORS) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        x[4 * u] = second ? second_bits<0>(w[u]) : first_bits<0>(w[u]);
        x[4 * u + 1] = second ? second_bits<1>(w[u]) : first_bits<1>(w[u]);
        x[4 * u + 2] = second ? second_bits<2>(w[u]) : first_bits<2>(w[u]);
        x[4 * u + 3] = second ? second_bits<3>(w[u]) : first_bits<3>(w[u]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = second ? second_bits<0>(w[j]) : first_bits<0>(w[j]);
    }
    const Powers power{scale, second ? kSecond : kFirst};
    if (power.two()) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = power.up_twice(x[j]);
    } else {
      const float up = power.up();
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= up;
    }
  }
  // t: codes above 20 bits of fraction; signs: values with the codes' signs, or NULL.
  __device__ __forceinline__ void put_codes(unsigned char* to, const unsigned (&t)[8], const float* signs, bool none) const {
    if (VECTORS) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        unsigned w = t[4 * u] >> 20 | t[4 * u + 1] >> 20 << 8 | t[4 * u + 2] >> 20 << 16 | t[4 * u + 3] >> 20 << 24;
        if (signs) {
          const unsigned a = __byte_perm(__float_as_uint(signs[4 * u]), __float_as_uint(signs[4 * u + 1]), 0x0073);
          const unsigned b = __byte_perm(__float_as_uint(signs[4 * u + 2]), __float_as_uint(signs[4 * u + 3]), 0x0073);
          w |= __byte_perm(a, b, 0x5410) & 0x80808080u;
        }
        __stcs((unsigned*)(to + 128 * u) + lane, none ? 0u : w);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) __stcs(to + at(j), (unsigned char)(none ? 0u : t[j] >> 20 | (signs ? __float_as_uint(signs[j]) >> 31 << 7 : 0u)));
    }
  }
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The same as update() where eps hides what becomes of a root of a value under the smallest normal number: in 1e-10 it is under 2^-24.
__device__ __forceinline__ void update_quickly(float& p, float m, float v, const Hyper& h, const Corrections& c) {
  float root, per;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(v));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(per) : "f"(fmaf(root, c.root, h.eps)));
  p -= loss_of(p, h.decay, c.step_size * m * per);
}

// A block by a warp.  What bounds it is the number of instructions, 532 a warp with its eight values a lane (41 us of the integer pipe, 46 of issue slots and 54 of HBM in 73 us for 25.6 M
// values): words of codes are taken apart and put together whole, and everything that a scale decides is decided once a block.  Two to eight blocks a warp: 5 to 60 us more; 48
// registers instead of 64, five CTAs an SM: no difference.
template <bool VECTORS>
__device__ __forceinline__ void update_block(const Lane<VECTORS> l, float* p, const float* g, int n, unsigned char* codes, unsigned char* scales, unsigned first, unsigned key,
                                             const Hyper& h, const Corrections* corrections) {
  float pp[8], gg[8], m[8], v[8];
  unsigned cm[8], cv[8];
  l.values(g, n, gg);
  l.codes(codes, cm);
  l.codes(codes + kBlock, cv);
  l.values(p, n, pp);
  const unsigned scale = *(const unsigned short*)scales;
  const Corrections c = *corrections;
  l.decode(cm, scale & 0xFFu, m, false);
  l.decode(cv, scale >> 8, v, true);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = gg[j] * c.grad_scale, root = h.c2 * x;
    m[j] = __fmaf_rn(h.c1, x, __fmul_rn(h.b1, m[j]));
    v[j] = __fmaf_rn(root, root, __fmul_rn(h.b2, v[j]));
  }
  if (n < kBlock) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (l.at(j) >= n) m[j] = v[j] = 0.f;
  }
  float most_m = 0, most_v = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    most_m = max_nan(most_m, fabsf(m[j]));
    most_v = max_nan(most_v, v[j]);
  }
  if (h.eps >= 1e-10f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) update_quickly(pp[j], m[j], v[j], h, c);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) update(pp[j], m[j], v[j], h, c);
  }
  l.put(p, n, pp);
  // a NaN's bits are above infinity's, and scale_of takes both for 255
  const unsigned scale_m = scale_of(__uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most_m))));
  const unsigned scale_v = scale_of(__uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most_v))));
  // To codes with 20 bits of fraction, of which 16 are compared with a random number: it and a half are added.
  const Powers to_m{scale_m, kFirst}, to_v{scale_v, kSecond};
  float x[8], y[8];
  if (to_m.two()) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = to_m.down_twice(fabsf(m[j]));
  } else {
    const float down = to_m.down();
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fabsf(m[j]) * down;
  }
  if (to_v.two()) {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = to_v.down_twice(v[j]);
  } else {
    const float down = to_v.down();
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = v[j] * down;
  }
  key = mix(key + c.t) + (first + l.at(0)) * kGolden;
  bool zero = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned r = mix(key + (unsigned)(l.at(j) - l.at(0)) * kGolden);
    cm[j] = __float_as_uint(x[j]) + ((r >> 12 & 0xFFFF0u) | 8u);
    cv[j] = max(__float_as_uint(y[j]) + ((r << 4 & 0xFFFF0u) | 8u), 1u << 20);  // not to zero
    zero |= v[j] == 0.f;
  }
  if (__any_sync(0xFFFFFFFFu, zero)) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (v[j] == 0.f) cv[j] = 0;
  }
  l.put_codes(codes, cm, m, scale_m == 255);
  l.put_codes(codes + kBlock, cv, nullptr, scale_v == 255);
  if (l.lane == 0) *(unsigned short*)scales = (unsigned short)(scale_m | scale_v << 8);
}

template <int N>
__global__ void __launch_bounds__(kThreads) adamw8_kernel(const __grid_constant__ Table<unsigned char, N> t, Hyper h, const Corrections* __restrict__ corrections) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int chunk = (int)(gridDim.x - 1 - blockIdx.x), k = t.chunks.tensor(chunk), lane = threadIdx.x & 31;
  const long long block = (long long)(chunk - t.chunks.start[k]) * (kChunk / kBlock) + (threadIdx.x >> 5), e = block * kBlock, left = t.n[k] - e;
  if (left <= 0) return;
  const int n = left < kBlock ? (int)left : kBlock;
  float* p = t.p[k] + e;
  const float* g = t.g[k] + e;
  unsigned char *codes = t.m[k] + block * 2 * kBlock, *scales = t.v[k] + block * 2;
  if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) & 15u) == 0)
    update_block(Lane<true>{lane}, p, g, n, codes, scales, (unsigned)e, t.key[k], h, corrections + t.slot[k]);
  else
    update_block(Lane<false>{lane}, p, g, n, codes, scales, (unsigned)e, t.key[k], h, corrections + t.slot[k]);
}

template <int N>
struct MomentsTable {
  const unsigned char *codes[N], *scales[N];
  float *m[N], *v[N];
  long long n[N];
  Chunks<N> chunks;
};
template <bool VECTORS>
__device__ __forceinline__ void write_block(const Lane<VECTORS> l, const unsigned char* codes, const unsigned char* scales, float* m, float* v, int n) {
  unsigned cm[8], cv[8];
  float x[8], y[8];
  l.codes(codes, cm);
  l.codes(codes + kBlock, cv);
  const unsigned scale = *(const unsigned short*)scales;
  l.decode(cm, scale & 0xFFu, x, false);
  l.decode(cv, scale >> 8, y, true);
  l.put(m, n, x);
  l.put(v, n, y);
}
// A whole block to where values begin `past` ones behind 16 bytes: a lane takes its codes from two words, so that it still stores 16 bytes at a time.  161 tensors packed side by side
// 47 -> 41 us, 6.1 TB/s.
__device__ __forceinline__ void write_shifted(const Lane<true> l, const unsigned char* codes, const unsigned char* scales, float* m, float* v, int past) {
  const int skip = 4 - past, lane = l.lane;
  const unsigned scale = *(const unsigned short*)scales;
#pragma unroll
  for (int second = 0; second < 2; ++second) {
    unsigned w[8], q[8];
    l.codes(codes + second * kBlock, w);
    float* const to = second ? v : m;
    float x[8], head[8];
    const unsigned behind = __shfl_sync(0xFFFFFFFFu, w[1], 0);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      unsigned next = __shfl_down_sync(0xFFFFFFFFu, w[u], 1);
      if (u == 0 && lane == 31) next = behind;
      q[u] = __funnelshift_r(w[u], next, 8 * skip);
    }
    l.decode(q, second ? scale >> 8 : scale & 0xFFu, x, second);
    st4(to + skip + 4 * lane, make_float4(x[0], x[1], x[2], x[3]));
    if (lane < 31) {
      st4(to + skip + 128 + 4 * lane, make_float4(x[4], x[5], x[6], x[7]));
    } else {  // the last ones
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < past) to[skip + 252 + j] = x[4 + j];
    }
    if (lane == 0) {  // the first ones
      l.decode(w, second ? scale >> 8 : scale & 0xFFu, head, second);
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < skip) to[j] = head[j];
    }
  }
}
template <int N>
__global__ void __launch_bounds__(kThreads) adamw8_moments_kernel(const __grid_constant__ MomentsTable<N> t) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int k = t.chunks.tensor(blockIdx.x), lane = threadIdx.x & 31;
  const long long block = (long long)((int)blockIdx.x - t.chunks.start[k]) * (kChunk / kBlock) + (threadIdx.x >> 5), e = block * kBlock, left = t.n[k] - e;
  if (left <= 0) return;
  const int n = left < kBlock ? (int)left : kBlock;
  float *m = t.m[k] + e, *v = t.v[k] + e;
  const unsigned char *codes = t.codes[k] + block * 2 * kBlock, *scales = t.scales[k] + block * 2;
  const int past = (int)(reinterpret_cast<uintptr_t>(m) >> 2 & 3);
  if (((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0) write_block(Lane<true>{lane}, codes, scales, m, v, n);
  else if (n == kBlock && past && ((reinterpret_cast<uintptr_t>(m) ^ reinterpret_cast<uintptr_t>(v)) & 15u) == 0) write_shifted(Lane<true>{lane}, codes, scales, m, v, past);
  else write_block(Lane<false>{lane}, codes, scales, m, v, n);
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
int begin(int count, void* const* params, double lr, double b1, double b2, double grad_scale, MtbClip clip, Corrections* out, std::vector<unsigned short>& slots, cudaStream_t st) {
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
    MTB_LAUNCH(adamw_begin_kernel, 1, 256, 0, st, t, lr, b1, b2, (float)grad_scale, clip, out + base);
    clip.norm = nullptr;  // left by the first launch
  }
  return MTB_OK;
}

bool moments_aligned(const void* codes, const void* scales) { return mtb_aligned16(codes) && (reinterpret_cast<uintptr_t>(scales) & 1u) == 0; }

bool fine(double lr, double b1, double b2, double eps, double weight_decay) {
  return lr >= 0 && b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1 && eps >= 0 && weight_decay >= 0;
}

constexpr int kFew = 24, kMany = 192;

// stride: numbers in `sizes` a tensor.
template <class M, int N, class K>
int run(const char* name, K kernel, int count, void* const* params, const long long* sizes, int stride, const std::vector<unsigned short>& slots, const Hyper& h,
        const Corrections* corrections, cudaStream_t st) {
  for (int base = (count - 1) / N * N; count > 0 && base >= 0; base -= N) {
    Table<M, N> t;
    const int tensors = count - base < N ? count - base : N, chunks = t.chunks.fill(tensors, sizes + (long long)stride * base, stride);
    for (int k = 0; k < tensors; ++k) {
      const Tensor a = tensor_at(params, base + k);
      const long long* size = sizes + (long long)stride * (base + k);
      t.p[k] = a.p;
      t.g[k] = a.g;
      t.m[k] = (M*)a.m;
      t.v[k] = (M*)a.v;
      t.n[k] = size[0];
      t.slot[k] = slots[base + k];
      t.key[k] = stride > 1 ? mix((unsigned)size[1]) : 0;
    }
    if (chunks == 0) continue;
    MTB_LAUNCH(kernel, dim3((unsigned)chunks), kThreads, 0, st, t, h, corrections);
    MTB_LAUNCH_CHECK(name);
  }
  return MTB_OK;
}

// Before anything is counted: no launch of the call has too many chunks.
bool fits(int count, const long long* sizes, int stride) {
  long long chunks = 0;
  for (int k = 0; k < count; ++k) chunks += sizes[(long long)stride * k] / kChunk + 1;
  return chunks < 1LL << 30;
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
  MTB_REQUIRE(fits(count, sizes, 1), "adamw: too many elements in one call");
  cudaStream_t st = (cudaStream_t)stream;
  Corrections* corrections = (Corrections*)scratch;
  if (int rc = begin(count, params, lr, beta1, beta2, grad_scale, MtbClip{sums, nsums, grad_scale, max_norm, norm}, corrections, slots, st)) return rc;
  const Hyper h{(float)beta1, (float)beta2, (float)(1 - beta1), (float)(1 - beta2), (float)eps, (float)(lr * weight_decay)};
  return count <= kFew ? run<float, kFew>("adamw_kernel", adamw_kernel<kFew>, count, params, sizes, 1, slots, h, corrections, st)
                       : run<float, kMany>("adamw_kernel", adamw_kernel<kMany>, count, params, sizes, 1, slots, h, corrections, st);
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
  MTB_REQUIRE(fits(count, sizes, 2), "adamw8: too many elements in one call");
  cudaStream_t st = (cudaStream_t)stream;
  Corrections* corrections = (Corrections*)scratch;
  if (int rc = begin(count, params, lr, b1, b2, grad_scale, MtbClip{sums, nsums, grad_scale, max_norm, norm}, corrections, slots, st)) return rc;
  const Hyper h{(float)b1, (float)b2, (float)(1 - b1), (float)std::sqrt(1 - b2), (float)eps, (float)(lr * weight_decay)};
  return count <= kFew ? run<unsigned char, kFew>("adamw8_kernel", adamw8_kernel<kFew>, count, params, sizes, 2, slots, h, corrections, st)
                       : run<unsigned char, kMany>("adamw8_kernel", adamw8_kernel<kMany>, count, params, sizes, 2, slots, h, corrections, st);
}

template <int N>
static int moments_of(int count, void* const* params, const long long* sizes, cudaStream_t st) {
  for (int base = 0; base < count; base += N) {
    MomentsTable<N> t;
    const int tensors = count - base < N ? count - base : N, chunks = t.chunks.fill(tensors, sizes + base, 1);
    for (int k = 0; k < tensors; ++k) {
      void* const* a = params + 4 * (long long)(base + k);
      t.codes[k] = (const unsigned char*)a[0];
      t.scales[k] = (const unsigned char*)a[1];
      t.m[k] = (float*)a[2];
      t.v[k] = (float*)a[3];
      t.n[k] = sizes[base + k];
    }
    if (chunks == 0) continue;
    MTB_LAUNCH(adamw8_moments_kernel<N>, dim3((unsigned)chunks), kThreads, 0, st, t);
    MTB_LAUNCH_CHECK("adamw8_moments_kernel");
  }
  return MTB_OK;
}

MTB_API int mtb_adamw8_moments_f32(int count, void* const* params, const long long* sizes, void* stream) {
  MTB_REQUIRE(count >= 0 && (count == 0 || (params && sizes)), "adamw8_moments: bad arguments");
  for (int k = 0; k < count; ++k) {
    void* const* a = params + 4 * (long long)k;
    MTB_REQUIRE(sizes[k] >= 0 && (sizes[k] == 0 || (a[0] && a[1] && a[2] && a[3])), "adamw8_moments: null tensor %d", k);
    MTB_REQUIRE(moments_aligned(a[0], a[1]), "adamw8_moments: moments of tensor %d begin off 16 bytes, or scales off 2", k);
  }
  MTB_REQUIRE(fits(count, sizes, 1), "adamw8_moments: too many elements in one call");
  return count <= kFew ? moments_of<kFew>(count, params, sizes, (cudaStream_t)stream) : moments_of<kMany>(count, params, sizes, (cudaStream_t)stream);
}
