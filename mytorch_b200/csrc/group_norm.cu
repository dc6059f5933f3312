// GroupNorm over channels-last activations [n][hw][c], with an activation behind it, forward and backward.
//
// A group is M = (c / groups) * hw values of one image.  Forward: mean, r = 1 / sqrt(var + eps) over the group,
// xh = (x - mean) r, z = gamma xh + beta, y = f(z).  Backward, from the saved mean and r: dz = dy f'(z),
// dbeta = sum dz, dgamma = sum dz xh over images and positions, and dx = r (gamma dz - (A + xh B) / M) with
// A = sum gamma dz, B = sum gamma dz xh over the group.
#include "common.cuh"

namespace {

enum Activation { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2 };

__device__ __forceinline__ float activate(float z, int act) {
  if (act == ACT_RELU) return fmaxf(z, 0.f);
  if (act == ACT_SILU) return z / (1.f + expf(-z));
  return z;
}
// dy f'(z); a ReLU passes what is at zero, as ReLU's own backward does
__device__ __forceinline__ float activate_grad(float dy, float z, int act) {
  if (act == ACT_RELU) return z < 0.f ? 0.f : dy;
  if (act == ACT_SILU) {
    const float s = 1.f / (1.f + expf(-z));
    return dy * (s * (1.f + z * (1.f - s)));
  }
  return dy;
}

template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* sm) {
  __syncthreads();
  sm[threadIdx.x] = v;
  __syncthreads();
  for (int w = THREADS / 2; w > 0; w >>= 1) {
    if (threadIdx.x < w) sm[threadIdx.x] += sm[threadIdx.x + w];
    __syncthreads();
  }
  return sm[0];
}

// One CTA a group, two passes: the mean, then the squares of what differs from it.
__global__ void __launch_bounds__(256) gn_stats_kernel(const float* __restrict__ x, int hw, int c, int groups, float eps, float* __restrict__ mean_out,
                                                        float* __restrict__ rstd_out) {
  mtb_launch_dependents();
  mtb_wait_prior();
  __shared__ float sm[256];
  const int cg = c / groups, g = blockIdx.x % groups;
  const long long n = blockIdx.x / groups, m = (long long)cg * hw;
  const float* base = x + n * hw * c + (long long)g * cg;
  float s = 0.f;
  for (long long i = threadIdx.x; i < m; i += 256) s += base[i / cg * c + i % cg];
  const float mean = block_sum<256>(s, sm) / (float)m;
  s = 0.f;
  for (long long i = threadIdx.x; i < m; i += 256) {
    const float d = base[i / cg * c + i % cg] - mean;
    s += d * d;
  }
  const float var = block_sum<256>(s, sm) / (float)m;
  if (threadIdx.x == 0) {
    mean_out[blockIdx.x] = mean;
    rstd_out[blockIdx.x] = 1.f / sqrtf(var + eps);
  }
}

__global__ void __launch_bounds__(256) gn_apply_kernel(const float* __restrict__ x, long long total, long long hw, int c, int groups, const float* __restrict__ gamma,
                                                        const float* __restrict__ beta, int act, const float* __restrict__ mean,
                                                        const float* __restrict__ rstd, float* __restrict__ y) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int cg = c / groups;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int ch = (int)(i % c);
    const long long k = i / c / hw * groups + ch / cg;
    const float z = (x[i] - mean[k]) * rstd[k] * (gamma ? gamma[ch] : 1.f) + (beta ? beta[ch] : 0.f);
    y[i] = activate(z, act);
  }
}

// Per image and channel: the sums of dz and of dz xh over the positions, to sums[n][2][c].
__global__ void __launch_bounds__(256) gn_bwd_sums_kernel(const float* __restrict__ dy, const float* __restrict__ x, int hw, int c, int groups,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ sums) {
  mtb_launch_dependents();
  mtb_wait_prior();
  __shared__ float sa[8][33], sb[8][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, ch = blockIdx.x * 32 + lane;
  const long long n = blockIdx.y;
  float a = 0.f, b = 0.f;
  if (ch < c) {
    const long long k = n * groups + ch / (c / groups);
    const float mu = mean[k], r = rstd[k], ga = gamma ? gamma[ch] : 1.f, be = beta ? beta[ch] : 0.f;
    for (int s = row; s < hw; s += 8) {
      const long long i = (n * hw + s) * c + ch;
      const float xh = (x[i] - mu) * r;
      const float dz = activate_grad(dy[i], xh * ga + be, act);
      a += dz;
      b += dz * xh;
    }
  }
  sa[row][lane] = a;
  sb[row][lane] = b;
  __syncthreads();
  if (row == 0 && ch < c) {
    for (int k = 1; k < 8; ++k) { a += sa[k][lane]; b += sb[k][lane]; }
    sums[(n * 2) * c + ch] = a;
    sums[(n * 2 + 1) * c + ch] = b;
  }
}

__global__ void __launch_bounds__(256) gn_bwd_params_kernel(const float* __restrict__ sums, int n, int c, float* __restrict__ dgamma, float* __restrict__ dbeta) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int ch = blockIdx.x * 256 + threadIdx.x;
  if (ch >= c) return;
  float a = 0.f, b = 0.f;
  for (int i = 0; i < n; ++i) { a += sums[(long long)i * 2 * c + ch]; b += sums[((long long)i * 2 + 1) * c + ch]; }
  if (dbeta) dbeta[ch] = a;
  if (dgamma) dgamma[ch] = b;
}

__global__ void __launch_bounds__(256) gn_bwd_groups_kernel(const float* __restrict__ sums, int n, int c, int groups, const float* __restrict__ gamma, float inv_m,
                                                             float* __restrict__ of_group) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const long long k = blockIdx.x * 256LL + threadIdx.x;
  if (k >= (long long)n * groups) return;
  const int cg = c / groups, g = (int)(k % groups);
  const float* s = sums + k / groups * 2 * c + (long long)g * cg;
  float a = 0.f, b = 0.f;
  for (int j = 0; j < cg; ++j) {
    const float ga = gamma ? gamma[g * cg + j] : 1.f;
    a += ga * s[j];
    b += ga * s[c + j];
  }
  of_group[2 * k] = a * inv_m;
  of_group[2 * k + 1] = b * inv_m;
}

__global__ void __launch_bounds__(256) gn_bwd_dx_kernel(const float* __restrict__ dy, const float* __restrict__ x, long long total, long long hw, int c, int groups,
                                                         const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd,
                                                         const float* __restrict__ of_group, float* __restrict__ dx) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int cg = c / groups;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int ch = (int)(i % c);
    const long long k = i / c / hw * groups + ch / cg;
    const float ga = gamma ? gamma[ch] : 1.f, be = beta ? beta[ch] : 0.f, r = rstd[k];
    const float xh = (x[i] - mean[k]) * r;
    const float dz = activate_grad(dy[i], xh * ga + be, act);
    dx[i] = r * (ga * dz - (of_group[2 * k] + xh * of_group[2 * k + 1]));
  }
}

}  // namespace

// Scratch of the backward: per image and channel two sums, per image and group two.
MTB_API long long mtb_group_norm_workspace_bytes(int n, int c, int hw, int groups) {
  (void)hw;
  return 8LL * n * c + 8LL * n * groups + 256;
}

MTB_API int mtb_group_norm_forward_f32(int n, int c, int hw, int groups, const float* x, const float* gamma, const float* beta, double eps, int activation,
                                       float* y, float* mean, float* rstd, void* stream) {
  MTB_REQUIRE(n >= 0 && c > 0 && hw >= 0 && groups > 0 && c % groups == 0, "group_norm_forward: %d channels in %d groups", c, groups);
  MTB_REQUIRE(activation >= ACT_NONE && activation <= ACT_SILU, "group_norm_forward: unknown activation %d", activation);
  const long long total = (long long)n * hw * c;
  if (total == 0) return MTB_OK;
  MTB_REQUIRE(x && y && mean && rstd, "group_norm_forward: null tensor");
  MTB_REQUIRE((long long)n * groups < (1LL << 31), "group_norm_forward: too many groups");
  cudaStream_t st = (cudaStream_t)stream;
  MTB_LAUNCH(gn_stats_kernel, n * groups, 256, 0, st, x, hw, c, groups, (float)eps, mean, rstd);
  MTB_LAUNCH(gn_apply_kernel, mtb_stream_grid(total, 256), 256, 0, st, x, total, (long long)hw, c, groups, gamma, beta, activation, mean, rstd, y);
  return MTB_OK;
}

MTB_API int mtb_group_norm_backward_f32(int n, int c, int hw, int groups, const float* dy, const float* mean, const float* rstd, const float* x,
                                        const float* gamma, const float* beta, int activation, float* dx, float* dgamma, float* dbeta, void* workspace,
                                        long long workspace_bytes, void* stream) {
  const MtbScratchTurn turn;
  MTB_REQUIRE(n >= 0 && c > 0 && hw >= 0 && groups > 0 && c % groups == 0, "group_norm_backward: %d channels in %d groups", c, groups);
  MTB_REQUIRE(activation >= ACT_NONE && activation <= ACT_SILU, "group_norm_backward: unknown activation %d", activation);
  cudaStream_t st = (cudaStream_t)stream;
  const long long total = (long long)n * hw * c;
  if (total == 0) {  // sums over nothing
    if (dgamma) MTB_CUDA(cudaMemsetAsync(dgamma, 0, 4LL * c, st));
    if (dbeta) MTB_CUDA(cudaMemsetAsync(dbeta, 0, 4LL * c, st));
    return MTB_OK;
  }
  MTB_REQUIRE(dy && mean && rstd && x && workspace, "group_norm_backward: null tensor");
  MTB_REQUIRE(n < 65536, "group_norm_backward: %d images", n);
  MTB_REQUIRE(workspace_bytes >= mtb_group_norm_workspace_bytes(n, c, hw, groups), "group_norm_backward: workspace too small");
  float *sums = (float*)workspace, *of_group = sums + 2LL * n * c;
  MTB_LAUNCH(gn_bwd_sums_kernel, dim3(mtb_div_up(c, 32), n), 256, 0, st, dy, x, hw, c, groups, gamma, beta, activation, mean, rstd, sums);
  if (dgamma || dbeta) MTB_LAUNCH(gn_bwd_params_kernel, mtb_div_up(c, 256), 256, 0, st, sums, n, c, dgamma, dbeta);
  if (dx) {
    MTB_LAUNCH(gn_bwd_groups_kernel, mtb_div_up((long long)n * groups, 256), 256, 0, st, sums, n, c, groups, gamma,
               (float)(1.0 / ((double)(c / groups) * hw)), of_group);
    MTB_LAUNCH(gn_bwd_dx_kernel, mtb_stream_grid(total, 256), 256, 0, st, dy, x, total, (long long)hw, c, groups, gamma, beta, activation, mean, rstd,
               of_group, dx);
  }
  return MTB_OK;
}
