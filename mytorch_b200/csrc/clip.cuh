// What turns the partial sums of squares that mtb_grad_norm_f32 left into the norm of all gradients and the factor that clips them.
#pragma once
#include "common.cuh"

struct MtbClip {
  const double* sums;  // NULL: no clipping
  int count;
  double grad_scale, max_norm;  // max_norm < 0: the norm only
  float* norm;                  // where the first CTA leaves the norm; may be NULL
};

// min(1, max_norm / (norm + 1e-6)), the norm that of grad_scale times the gradients.  Every CTA of a kernel that needs the factor
// adds the sums up for itself, all in the same order: a few hundred values that are in L2, while its own data is on its
// way, instead of a launch of one CTA in between that everything would wait for.  A norm that is no number makes the factor none, an infinite
// one makes it 0, as the formula has it.  All threads of the CTA call this; THREADS is their number.
template <int THREADS>
__device__ __forceinline__ float mtb_clip_factor(const MtbClip& clip) {
  __shared__ double part[THREADS / 32];
  double s = 0;
  for (int i = threadIdx.x; i < clip.count; i += THREADS) s += clip.sums[i];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) s += part[i];
  const double norm = sqrt(s) * fabs(clip.grad_scale);
  if (clip.norm && blockIdx.x == 0 && threadIdx.x == 0) *clip.norm = (float)norm;
  if (clip.max_norm < 0) return 1.f;
  const double q = clip.max_norm / (norm + 1e-6);
  return q > 1 ? 1.f : (float)q;
}
