// GroupNorm over channels-last activations [n][hw][c], with an activation behind it, forward and backward.
//
// A group is M = (c / groups) * hw values of one image.  Forward: mean, r = 1 / sqrt(var + eps) over the group,
// xh = (x - mean) r, z = gamma xh + beta, y = f(z).  Backward, from the saved mean and r: dz = dy f'(z),
// dbeta = sum dz, dgamma = sum dz xh over images and positions, and dx = r (gamma dz - (A + xh B) / M) with
// A = sum gamma dz, B = sum gamma dz xh over the group.
//
// HBM-bound: 8 bytes a value forward, 12 backward, if the values stay on the chip between the sums and what is made of them.  So a cluster of CTAs holds
// a slab, some whole groups of one image (32 channels or more: a line of memory), in its shared memory, each CTA a stretch of positions.  A thread copies (cp.async) and later
// reads its own vectors only, so the copies need no barrier; the CTAs exchange their sums through distributed shared memory.  A slab that no
// cluster can hold goes through memory twice instead, see the kernels at the end.
#include "colreduce.cuh"
#include <cooperative_groups.h>

namespace {

namespace cg = cooperative_groups;

enum Activation { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2 };

// SiLU by the fast exponential and quotient: a relative error of about 2^-21 of a value whose input carries the error of a normalisation
__device__ __forceinline__ float activate(float z, int act) {
  if (act == ACT_RELU) return z < 0.f ? 0.f : z;
  if (act == ACT_SILU) return __fdividef(z, 1.f + __expf(-z));
  return z;
}
// dy f'(z); a ReLU passes what is at zero, as ReLU's own backward does
__device__ __forceinline__ float activate_grad(float dy, float z, int act) {
  if (act == ACT_RELU) return z < 0.f ? 0.f : dy;
  if (act == ACT_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-z));
    return dy * (s * (1.f + z * (1.f - s)));
  }
  return dy;
}

__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int V>
__device__ __forceinline__ void copy_async(float* to, const float* from) {
  const unsigned at = (unsigned)__cvta_generic_to_shared(to);
  if (V == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else if (V == 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <int V> struct alignas(4 * V) Vec { float v[V]; };
template <int V> __device__ __forceinline__ Vec<V>& vec(float* p) { return *reinterpret_cast<Vec<V>*>(p); }

// ---------------------------------------------------------------- a slab on the chip

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct Slabs {
  int hw, c, groups, each;  // channels of a group
  int wide, slabs;          // channels of a slab (the last one may have fewer), slabs of an image
  int ctas, stretch;        // CTAs of a cluster, positions of a CTA
  int steps;                // positions of a thread at most
  int sums;                 // floats of shared memory between the values and what the other CTAs read
  PoolDiv by_each;
};

// What a CTA and a thread of it have to do.
struct Share {
  int n, c0, width, vectors, rows;  // image, first channel, channels; vectors of a position, positions a step
  int row, col, positions, steps;   // a thread's position within a step and its channels' offset; positions of the CTA, steps of the thread
  long long first;                  // of the thread's values
  template <int V>
  __device__ __forceinline__ void of(const Slabs& p, int unit, int rank) {
    n = unit / p.slabs;
    c0 = (unit - n * p.slabs) * p.wide;
    width = p.wide < p.c - c0 ? p.wide : p.c - c0;
    vectors = width / V;
    rows = kThreads / vectors;
    row = threadIdx.x / vectors;
    col = (threadIdx.x - row * vectors) * V;
    const int p0 = rank * p.stretch;
    positions = p.stretch < p.hw - p0 ? p.stretch : p.hw - p0;
    steps = row < rows && row < positions ? (positions - row - 1) / rows + 1 : 0;
    first = ((long long)n * p.hw + p0 + row) * p.c + c0 + col;
  }
};

// The sum of `part` [rows][width] over a group's channels, by a warp.
__device__ __forceinline__ float sum_group(const float* part, const Share& s, const Slabs& p, int g) {
  float sum = 0.f;
  for (unsigned q = threadIdx.x & 31; q < (unsigned)(s.rows * p.each); q += 32) {
    unsigned ch;
    const unsigned row = p.by_each.divmod(q, ch);
    sum += part[row * s.width + g * p.each + ch];
  }
  return warp_sum(sum);
}

template <int V, int ACT>
__global__ void __launch_bounds__(kThreads) gn_forward_kernel(const __grid_constant__ Slabs p, const float* __restrict__ x, const float* __restrict__ gamma,
                                                               const float* __restrict__ beta, float eps, float* __restrict__ y,
                                                               float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  extern __shared__ __align__(16) float held[];  // [steps][kThreads][V], then the threads' sums and the groups' statistics
  mtb_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = p.ctas > 1 ? (int)cluster.block_rank() : 0;
  Share s;
  s.of<V>(p, blockIdx.x / p.ctas, rank);
  float *mine = held + threadIdx.x * V, *part = held + p.steps * kThreads * V, *mean_of = part + p.sums, *m2_of = mean_of + p.wide;
  const int groups = s.width / p.each, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool active = s.row < s.rows;
  mtb_wait_prior();
  const float* from = x + s.first;
  const long long step = (long long)s.rows * p.c;
  for (int j = 0; j < s.steps; ++j) copy_async<V>(mine + j * kThreads * V, from + j * step);
  int of[V];  // group
  float scale[V], shift[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    of[i] = (s.col + i) / p.each;
    scale[i] = active && gamma ? gamma[s.c0 + s.col + i] : 1.f;
    shift[i] = active && beta ? beta[s.c0 + s.col + i] : 0.f;
  }
  copies_done();

  // the CTA's mean, then the squares of what differs from it
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.f;
  for (int j = 0; j < s.steps; ++j) {
    const Vec<V> v = vec<V>(mine + j * kThreads * V);
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] += v.v[i];
  }
  if (active)
#pragma unroll
    for (int i = 0; i < V; ++i) part[threadIdx.x * V + i] = sum[i];
  __syncthreads();
  const float inv = 1.f / ((float)p.each * s.positions);
  for (int g = warp; g < groups; g += kWarps) {
    const float t = sum_group(part, s, p, g);
    if (lane == 0) mean_of[g] = t * inv;
  }
  __syncthreads();
  float mu[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    mu[i] = active ? mean_of[of[i]] : 0.f;
    sum[i] = 0.f;
  }
  for (int j = 0; j < s.steps; ++j) {
    const Vec<V> v = vec<V>(mine + j * kThreads * V);
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] += (v.v[i] - mu[i]) * (v.v[i] - mu[i]);
  }
  if (active)
#pragma unroll
    for (int i = 0; i < V; ++i) part[threadIdx.x * V + i] = sum[i];
  __syncthreads();
  for (int g = warp; g < groups; g += kWarps) {
    const float t = sum_group(part, s, p, g);
    if (lane == 0) m2_of[g] = t;
  }

  // the group's, from the CTAs' (Chan): sum of n_k mean_k / N, then M2_k + n_k (mean_k - mean)^2
  if (p.ctas > 1) cluster.sync(); else __syncthreads();
  float *group_mean = part, *group_rstd = part + p.wide;
  const float whole = (float)p.hw;
  for (int g = threadIdx.x; g < groups; g += kThreads) {
    float mean = mean_of[g], m2 = m2_of[g];
    if (p.ctas > 1) {
      mean = 0.f;
      for (int r = 0; r < p.ctas; ++r) {
        const int count = r + 1 < p.ctas ? p.stretch : p.hw - r * p.stretch;
        mean += (float)count / whole * cluster.map_shared_rank(mean_of, r)[g];
      }
      m2 = 0.f;
      for (int r = 0; r < p.ctas; ++r) {
        const int count = r + 1 < p.ctas ? p.stretch : p.hw - r * p.stretch;
        const float d = cluster.map_shared_rank(mean_of, r)[g] - mean;
        m2 += cluster.map_shared_rank(m2_of, r)[g] + (float)count * p.each * (d * d);
      }
    }
    const float rstd = 1.f / sqrtf(m2 / ((float)p.each * whole) + eps);
    group_mean[g] = mean;
    group_rstd[g] = rstd;
    if (rank == 0) {
      const long long k = (long long)s.n * p.groups + s.c0 / p.each + g;
      mean_out[k] = mean;
      rstd_out[k] = rstd;
    }
  }
  if (p.ctas > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");  // this CTA has read the others'
  __syncthreads();
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (active) {
      mu[i] = group_mean[of[i]];
      scale[i] *= group_rstd[of[i]];
    }
  }
  float* to = y + s.first;
  for (int j = 0; j < s.steps; ++j) {
    Vec<V> v = vec<V>(mine + j * kThreads * V);
#pragma unroll
    for (int i = 0; i < V; ++i) v.v[i] = activate((v.v[i] - mu[i]) * scale[i] + shift[i], ACT);
    *reinterpret_cast<Vec<V>*>(to + j * step) = v;
  }
  if (p.ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the others have read this CTA's
}

// sums (may be NULL): per image and channel the sums of dz and of dz xh, [n][2][c].  dx may be NULL.
template <int V, int ACT>
__global__ void __launch_bounds__(kThreads) gn_backward_kernel(const __grid_constant__ Slabs p, const float* __restrict__ dy, const float* __restrict__ x,
                                                                const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ dx,
                                                                float* __restrict__ sums) {
  extern __shared__ __align__(16) float held[];  // [2][steps][kThreads][V], then the threads' sums, the CTA's and the groups'
  mtb_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = p.ctas > 1 ? (int)cluster.block_rank() : 0;
  Share s;
  s.of<V>(p, blockIdx.x / p.ctas, rank);
  const int plane = p.steps * kThreads * V;
  float *mine = held + threadIdx.x * V, *part = held + 2 * plane, *part2 = part + kThreads * V, *sum_of = part + p.sums, *sum2_of = sum_of + p.wide;
  const int groups = s.width / p.each, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool active = s.row < s.rows;
  mtb_wait_prior();
  const long long step = (long long)s.rows * p.c;
  for (int j = 0; j < s.steps; ++j) {
    copy_async<V>(mine + j * kThreads * V, x + s.first + j * step);
    copy_async<V>(mine + plane + j * kThreads * V, dy + s.first + j * step);
  }
  int of[V];
  float mu[V], r[V], ga[V], be[V], a[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    of[i] = (s.col + i) / p.each;
    const long long k = (long long)s.n * p.groups + s.c0 / p.each + of[i];
    mu[i] = active ? mean[k] : 0.f;
    r[i] = active ? rstd[k] : 0.f;
    ga[i] = active && gamma ? gamma[s.c0 + s.col + i] : 1.f;
    be[i] = active && beta ? beta[s.c0 + s.col + i] : 0.f;
    a[i] = b[i] = 0.f;
  }
  copies_done();
  for (int j = 0; j < s.steps; ++j) {  // xh and dz take the places of x and dy
    Vec<V> v = vec<V>(mine + j * kThreads * V), d = vec<V>(mine + plane + j * kThreads * V);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v.v[i] = (v.v[i] - mu[i]) * r[i];
      d.v[i] = activate_grad(d.v[i], v.v[i] * ga[i] + be[i], ACT);
      a[i] += d.v[i];
      b[i] += d.v[i] * v.v[i];
    }
    vec<V>(mine + j * kThreads * V) = v;
    if (ACT != ACT_NONE) vec<V>(mine + plane + j * kThreads * V) = d;
  }
  if (active) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      part[threadIdx.x * V + i] = a[i];
      part2[threadIdx.x * V + i] = b[i];
    }
  }
  __syncthreads();
  for (int k = warp; k < 2 * s.width; k += kWarps) {  // a channel's sums over the CTA's rows
    const float* from = k < s.width ? part + k : part2 + k - s.width;
    float t = 0.f;
    for (int row = lane; row < s.rows; row += 32) t += from[row * s.width];
    t = warp_sum(t);
    if (lane == 0) (k < s.width ? sum_of[k] : sum2_of[k - s.width]) = t;
  }
  if (p.ctas > 1) cluster.sync(); else __syncthreads();
  // over the cluster
  for (int k = threadIdx.x; k < 2 * s.width; k += kThreads) {
    float* from = k < s.width ? sum_of + k : sum2_of + k - s.width;
    float t = 0.f;
    if (p.ctas > 1) {
      for (int q = 0; q < p.ctas; ++q) t += *cluster.map_shared_rank(from, q);
    } else {
      t = *from;
    }
    part[k] = t;
    if (rank == 0 && sums) sums[((long long)s.n * 2 + (k < s.width ? 0 : 1)) * p.c + s.c0 + (k < s.width ? k : k - s.width)] = t;
  }
  if (p.ctas > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  if (dx) {
    __syncthreads();
    float* of_group = part + 2 * p.wide;  // A / M, B / M
    const float inv = 1.f / ((float)p.each * p.hw);
    for (int k = warp; k < 2 * groups; k += kWarps) {
      const int g = k >> 1, base = g * p.each;
      float t = 0.f;
      for (int ch = lane; ch < p.each; ch += 32) t += (gamma ? gamma[s.c0 + base + ch] : 1.f) * part[(k & 1) * s.width + base + ch];
      t = warp_sum(t);
      if (lane == 0) of_group[k] = t * inv;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] = active ? of_group[2 * of[i]] * r[i] : 0.f;
      b[i] = active ? of_group[2 * of[i] + 1] * r[i] : 0.f;
      ga[i] *= r[i];
    }
    float* to = dx + s.first;
    for (int j = 0; j < s.steps; ++j) {
      Vec<V> v = vec<V>(mine + j * kThreads * V);
      const Vec<V> d = vec<V>(mine + plane + j * kThreads * V);
#pragma unroll
      for (int i = 0; i < V; ++i) v.v[i] = ga[i] * d.v[i] - (a[i] + v.v[i] * b[i]);
      *reinterpret_cast<Vec<V>*>(to + j * step) = v;
    }
  }
  if (p.ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// dgamma and dbeta: the sums over the images, 32 columns of [n][2 c] a CTA, in a fixed order.
__global__ void __launch_bounds__(256) gn_params_kernel(const float* __restrict__ sums, int n, int c, float* __restrict__ dgamma, float* __restrict__ dbeta) {
  mtb_launch_dependents();
  mtb_wait_prior();
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (col < 2 * c)
#pragma unroll 8
    for (int i = row; i < n; i += 8) t += sums[(long long)i * 2 * c + col];
  part[row][lane] = t;
  __syncthreads();
  if (row != 0 || col >= 2 * c) return;
  for (int k = 1; k < 8; ++k) t += part[k][lane];
  if (col < c) { if (dbeta) dbeta[col] = t; }
  else if (dgamma) dgamma[col - c] = t;
}

// ---------------------------------------------------------------- a slab through memory

// Images that no cluster can hold, and groups of more channels than a CTA has threads' vectors: partial statistics of stretches of positions,
// statistics, result.

// partial[group][split][3]: count, mean, M2, of shifted sums
__global__ void __launch_bounds__(256) gn_stats_kernel(const float* __restrict__ x, int hw, int c, int groups, int splits, float* __restrict__ partial) {
  mtb_launch_dependents();
  mtb_wait_prior();
  __shared__ float sm[3][8];
  const int each = c / groups, g = blockIdx.y % groups, n = blockIdx.y / groups, stretch = (hw + splits - 1) / splits;
  const int p0 = blockIdx.x * stretch, p1 = p0 + stretch < hw ? p0 + stretch : hw;
  const float* base = x + ((long long)n * hw + p0) * c + (long long)g * each;
  const int lanes = each < 256 ? each : 256, rows = 256 / lanes, row = threadIdx.x / lanes, lane = threadIdx.x - row * lanes;
  float count = 0.f, s1 = 0.f, s2 = 0.f, pivot = 0.f;
  if (row < rows && p0 + row < p1) {
    pivot = base[(long long)row * c + lane];
    for (int pos = row; pos < p1 - p0; pos += rows) {
#pragma unroll 4
      for (int ch = lane; ch < each; ch += lanes) {
        const float d = base[(long long)pos * c + ch] - pivot;
        s1 += d;
        s2 += d * d;
        count += 1.f;
      }
    }
  }
  float mean = count > 0.f ? pivot + s1 / count : 0.f, m2 = count > 0.f ? s2 - s1 * s1 / count : 0.f;
  auto merge = [&](float nb, float mb, float qb) {
    if (nb == 0.f) return;
    const float total = count + nb, d = mb - mean;
    mean += d * (nb / total);
    m2 += qb + d * d * count * (nb / total);
    count = total;
  };
  for (int o = 16; o > 0; o >>= 1) {
    const float nb = __shfl_down_sync(0xffffffffu, count, o), mb = __shfl_down_sync(0xffffffffu, mean, o), qb = __shfl_down_sync(0xffffffffu, m2, o);
    merge(nb, mb, qb);
  }
  if ((threadIdx.x & 31) == 0) { sm[0][threadIdx.x >> 5] = count; sm[1][threadIdx.x >> 5] = mean; sm[2][threadIdx.x >> 5] = m2; }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 8; ++w) merge(sm[0][w], sm[1][w], sm[2][w]);
  float* to = partial + ((long long)blockIdx.y * splits + blockIdx.x) * 3;
  to[0] = count;
  to[1] = mean;
  to[2] = m2;
}

__global__ void __launch_bounds__(128) gn_stats_final_kernel(const float* __restrict__ partial, int count, int splits, float eps, float* __restrict__ mean_out,
                                                              float* __restrict__ rstd_out) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int k = blockIdx.x * 128 + threadIdx.x;
  if (k >= count) return;
  float n = 0.f, mean = 0.f, m2 = 0.f;
  for (int i = 0; i < splits; ++i) {
    const float* q = partial + ((long long)k * splits + i) * 3;
    if (q[0] == 0.f) continue;
    const float total = n + q[0], d = q[1] - mean;
    mean += d * (q[0] / total);
    m2 += q[2] + d * d * n * (q[0] / total);
    n = total;
  }
  mean_out[k] = mean;
  rstd_out[k] = 1.f / sqrtf(m2 / n + eps);
}

__global__ void __launch_bounds__(256) gn_apply_kernel(const float* __restrict__ x, long long image, PoolDiv by_c, PoolDiv by_each, int groups,
                                                        const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                        const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ y) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const long long first = blockIdx.y * image;
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < image; i += gridDim.x * 256) {
    unsigned ch, unused;
    by_c.divmod(i, ch);
    const int k = blockIdx.y * groups + by_each.divmod(ch, unused);
    const float z = (x[first + i] - mean[k]) * rstd[k] * (gamma ? gamma[ch] : 1.f) + (beta ? beta[ch] : 0.f);
    y[first + i] = activate(z, act);
  }
}

// partial[split][n][2][c]: the sums of dz and of dz xh over a stretch of positions
__global__ void __launch_bounds__(256) gn_bwd_sums_kernel(const float* __restrict__ dy, const float* __restrict__ x, int hw, int c, int groups, int splits,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ partial) {
  mtb_launch_dependents();
  mtb_wait_prior();
  __shared__ float sa[8][33], sb[8][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, ch = blockIdx.x * 32 + lane, n = blockIdx.y, stretch = (hw + splits - 1) / splits;
  const int p0 = blockIdx.z * stretch, p1 = p0 + stretch < hw ? p0 + stretch : hw;
  float a = 0.f, b = 0.f;
  if (ch < c) {
    const int k = n * groups + ch / (c / groups);
    const float mu = mean[k], r = rstd[k], ga = gamma ? gamma[ch] : 1.f, be = beta ? beta[ch] : 0.f;
#pragma unroll 4
    for (int s = p0 + row; s < p1; s += 8) {
      const long long i = ((long long)n * hw + s) * c + ch;
      const float xh = (x[i] - mu) * r, dz = activate_grad(dy[i], xh * ga + be, act);
      a += dz;
      b += dz * xh;
    }
  }
  sa[row][lane] = a;
  sb[row][lane] = b;
  __syncthreads();
  if (row == 0 && ch < c) {
    for (int k = 1; k < 8; ++k) { a += sa[k][lane]; b += sb[k][lane]; }
    float* to = partial + ((long long)blockIdx.z * gridDim.y + n) * 2 * c + ch;
    to[0] = a;
    to[c] = b;
  }
}

// sums[n][2][c] over the splits, in place of the first; then A / M and B / M of each group.  A warp a group.
__global__ void __launch_bounds__(128) gn_bwd_groups_kernel(float* __restrict__ sums, int n, int c, int groups, int splits, const float* __restrict__ gamma,
                                                             float inv_m, float* __restrict__ of_group) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int k = blockIdx.x * 4 + (threadIdx.x >> 5), each = c / groups;
  if (k >= n * groups) return;
  float* s = sums + (long long)(k / groups) * 2 * c + (k % groups) * each;
  float a = 0.f, b = 0.f;
  for (int ch = threadIdx.x & 31; ch < each; ch += 32) {
    float u = 0.f, v = 0.f;
    for (int i = 0; i < splits; ++i) {
      u += s[(long long)i * n * 2 * c + ch];
      v += s[(long long)i * n * 2 * c + c + ch];
    }
    s[ch] = u;
    s[c + ch] = v;
    const float ga = gamma ? gamma[k % groups * each + ch] : 1.f;
    a += ga * u;
    b += ga * v;
  }
  a = warp_sum(a);
  b = warp_sum(b);
  if ((threadIdx.x & 31) == 0) {
    of_group[2 * k] = a * inv_m;
    of_group[2 * k + 1] = b * inv_m;
  }
}

__global__ void __launch_bounds__(256) gn_bwd_dx_kernel(const float* __restrict__ dy, const float* __restrict__ x, long long image, PoolDiv by_c, PoolDiv by_each,
                                                         int groups, const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd,
                                                         const float* __restrict__ of_group, float* __restrict__ dx) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const long long first = blockIdx.y * image;
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < image; i += gridDim.x * 256) {
    unsigned ch, unused;
    by_c.divmod(i, ch);
    const int k = blockIdx.y * groups + by_each.divmod(ch, unused);
    const float ga = gamma ? gamma[ch] : 1.f, r = rstd[k], xh = (x[first + i] - mean[k]) * r;
    const float dz = activate_grad(dy[first + i], xh * ga + (beta ? beta[ch] : 0.f), act);
    dx[first + i] = r * (ga * dz - (of_group[2 * k] + xh * of_group[2 * k + 1]));
  }
}

// ---------------------------------------------------------------- host

struct Plan {
  bool on_chip;
  int v, units, smem;
  Slabs s;
};

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// planes: tensors that the cluster holds (1 forward, 2 backward).
Plan plan_slabs(int n, int c, int hw, int groups, int planes, int alignment) {
  Plan t{};
  const int each = c / groups;
  t.v = c % 4 == 0 && alignment % 16 == 0 ? 4 : c % 2 == 0 && alignment % 8 == 0 ? 2 : 1;
  const int unit = t.v / gcd(each, t.v);  // groups whose channels are whole vectors
  // a line of memory a position; with few positions enough channels that every thread has a vector
  int want = kThreads * t.v / hw;
  want = want < 32 ? 32 : want > kThreads * t.v ? kThreads * t.v : want;
  for (int attempt = 0; attempt < 2; ++attempt) {
    int of_slab = attempt ? unit : ((want + each - 1) / each + unit - 1) / unit * unit;
    if (of_slab * each > kThreads * t.v && of_slab > unit) of_slab = kThreads * t.v / each / unit * unit;
    if (of_slab < unit) of_slab = unit;
    if (of_slab > groups) of_slab = groups;
    const int wide = of_slab * each;
    if (wide > kThreads * t.v) return t;
    const int rows = kThreads / (wide / t.v), slabs = (groups + of_slab - 1) / of_slab;
    auto steps_of = [&](int ctas) { const int stretch = (hw + ctas - 1) / ctas; return (stretch + rows - 1) / rows; };
    auto bytes_of = [&](int ctas) { return 4LL * planes * kThreads * t.v * steps_of(ctas); };
    // The fewest CTAs that leave an SM room for four of them, or two, or one.
    int ctas = 0;
    for (int most : {48, 100, 200}) {
      for (int k = 1; k <= 8 && !ctas; ++k)
        if (bytes_of(k) <= most * 1024LL) ctas = k;
      if (!ctas && most > 48 && bytes_of(16) <= most * 1024LL) ctas = 16;
      if (ctas) break;
    }
    if (!ctas) continue;
    // few slabs: more CTAs each, as long as a thread has several positions
    while (ctas < 8 && (long long)n * slabs * ctas < mtb_sm_count() && steps_of(ctas) > 2) ++ctas;
    const int stretch = (hw + ctas - 1) / ctas;
    ctas = (hw + stretch - 1) / stretch;
    // the threads' sums, and then a slab's and its groups'
    const int sums = planes * kThreads * t.v > 4 * wide ? planes * kThreads * t.v : 4 * wide;
    t.s = Slabs{hw, c, groups, each, wide, slabs, ctas, stretch, steps_of(ctas), sums, PoolDiv((unsigned)each)};
    t.smem = (int)bytes_of(ctas) + 4 * (sums + 2 * wide);
    if ((long long)n * slabs * ctas >= 1LL << 31) return t;
    t.units = n * slabs;
    t.on_chip = true;
    return t;
  }
  return t;
}

template <class... P, class... A>
int launch_slabs(unsigned long long* opted, unsigned long long* wide, const Plan& t, cudaStream_t st, void (*kernel)(P...), A... args) {
  if (int rc = mtb_opt_in_smem((const void*)kernel, 227 * 1024, opted)) return rc;
  if (t.s.ctas > 8) {
    int device = 0;
    MTB_CUDA(cudaGetDevice(&device));
    if (device >= 64 || !((__atomic_load_n(wide, __ATOMIC_ACQUIRE) >> device) & 1ull)) {
      MTB_CUDA(cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      if (device < 64) __atomic_fetch_or(wide, 1ull << device, __ATOMIC_RELEASE);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(t.units * t.s.ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = t.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = t.s.ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = t.s.ctas > 1 ? 2 : 1;
  MTB_CUDA(cudaLaunchKernelEx(&cfg, kernel, (P)args...));
  return MTB_OK;
}

template <int V, int ACT, class... A>
int forward_on_chip(const Plan& t, cudaStream_t st, A... args) {
  static unsigned long long opted, wide;
  return launch_slabs(&opted, &wide, t, st, gn_forward_kernel<V, ACT>, t.s, args...);
}
template <int V, int ACT, class... A>
int backward_on_chip(const Plan& t, cudaStream_t st, A... args) {
  static unsigned long long opted, wide;
  return launch_slabs(&opted, &wide, t, st, gn_backward_kernel<V, ACT>, t.s, args...);
}

#define MTB_GN_PICK(f, t, act, ...)                                                                                                               \
  ((t).v == 4 ? (act == ACT_SILU ? f<4, ACT_SILU>(t, __VA_ARGS__) : act == ACT_RELU ? f<4, ACT_RELU>(t, __VA_ARGS__) : f<4, ACT_NONE>(t, __VA_ARGS__)) \
   : (t).v == 2 ? (act == ACT_SILU ? f<2, ACT_SILU>(t, __VA_ARGS__) : act == ACT_RELU ? f<2, ACT_RELU>(t, __VA_ARGS__) : f<2, ACT_NONE>(t, __VA_ARGS__)) \
                : (act == ACT_SILU ? f<1, ACT_SILU>(t, __VA_ARGS__) : act == ACT_RELU ? f<1, ACT_RELU>(t, __VA_ARGS__) : f<1, ACT_NONE>(t, __VA_ARGS__)))

// Stretches that the positions of an image are cut into where slabs go through memory.
int splits_of(int n, int hw, int parts) {
  long long want = (4LL * mtb_sm_count() + (long long)n * parts - 1) / ((long long)n * parts);
  if (want > hw / 64) want = hw / 64;
  return want < 1 ? 1 : want > 256 ? 256 : (int)want;
}

// The largest power of two up to 16 that all of them are a multiple of.
int alignment_of(const void* a, const void* b, const void* c) {
  const int m = (int)(((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15);
  return m ? m & -m : 16;
}

}  // namespace

// Scratch of both directions: what slabs that go through memory leave of their stretches, and the backward's sums.
MTB_API long long mtb_group_norm_workspace_bytes(int n, int c, int hw, int groups) {
  if (n <= 0 || c <= 0 || hw <= 0 || groups <= 0) return 256;
  const long long forward = 12LL * n * groups * splits_of(n, hw, groups), backward = 8LL * n * c * splits_of(n, hw, mtb_div_up(c, 32)) + 8LL * n * groups;
  return (forward > backward ? forward : backward) + 256;
}

MTB_API int mtb_group_norm_forward_f32(int n, int c, int hw, int groups, const float* x, const float* gamma, const float* beta, double eps, int activation,
                                       float* y, float* mean, float* rstd, void* workspace, long long workspace_bytes, void* stream) {
  const MtbScratchTurn turn;
  MTB_REQUIRE(n >= 0 && c > 0 && hw >= 0 && groups > 0 && c % groups == 0, "group_norm_forward: %d channels in %d groups", c, groups);
  MTB_REQUIRE(activation >= ACT_NONE && activation <= ACT_SILU, "group_norm_forward: unknown activation %d", activation);
  if (n == 0 || hw == 0) return MTB_OK;
  MTB_REQUIRE(x && y && mean && rstd, "group_norm_forward: null tensor");
  MTB_REQUIRE((long long)n * groups < 1LL << 31 && (long long)hw * c < 1LL << 31, "group_norm_forward: too many values");
  cudaStream_t st = (cudaStream_t)stream;
  const Plan t = plan_slabs(n, c, hw, groups, 1, alignment_of(x, y, nullptr));
  if (t.on_chip) return MTB_GN_PICK(forward_on_chip, t, activation, st, x, gamma, beta, (float)eps, y, mean, rstd);
  MTB_REQUIRE(workspace && workspace_bytes >= mtb_group_norm_workspace_bytes(n, c, hw, groups), "group_norm_forward: workspace too small");
  MTB_REQUIRE((long long)n * groups < 65536 && n < 65536, "group_norm_forward: %d images of %d groups", n, groups);
  const int splits = splits_of(n, hw, groups);
  float* partial = (float*)workspace;
  const long long image = (long long)hw * c;
  MTB_LAUNCH(gn_stats_kernel, dim3(splits, n * groups), 256, 0, st, x, hw, c, groups, splits, partial);
  MTB_LAUNCH(gn_stats_final_kernel, mtb_div_up((long long)n * groups, 128), 128, 0, st, partial, n * groups, splits, (float)eps, mean, rstd);
  MTB_LAUNCH(gn_apply_kernel, dim3(mtb_stream_grid(image, 256), n), 256, 0, st, x, image, PoolDiv(c), PoolDiv(c / groups), groups, gamma, beta, activation, mean, rstd, y);
  return MTB_OK;
}

MTB_API int mtb_group_norm_backward_f32(int n, int c, int hw, int groups, const float* dy, const float* mean, const float* rstd, const float* x,
                                        const float* gamma, const float* beta, int activation, float* dx, float* dgamma, float* dbeta, void* workspace,
                                        long long workspace_bytes, void* stream) {
  const MtbScratchTurn turn;
  MTB_REQUIRE(n >= 0 && c > 0 && hw >= 0 && groups > 0 && c % groups == 0, "group_norm_backward: %d channels in %d groups", c, groups);
  MTB_REQUIRE(activation >= ACT_NONE && activation <= ACT_SILU, "group_norm_backward: unknown activation %d", activation);
  cudaStream_t st = (cudaStream_t)stream;
  if (n == 0 || hw == 0) {  // sums over nothing
    if (dgamma) MTB_CUDA(cudaMemsetAsync(dgamma, 0, 4LL * c, st));
    if (dbeta) MTB_CUDA(cudaMemsetAsync(dbeta, 0, 4LL * c, st));
    return MTB_OK;
  }
  MTB_REQUIRE(dy && mean && rstd && x && workspace, "group_norm_backward: null tensor");
  MTB_REQUIRE((long long)n * groups < 1LL << 31 && (long long)hw * c < 1LL << 31, "group_norm_backward: too many values");
  MTB_REQUIRE(workspace_bytes >= mtb_group_norm_workspace_bytes(n, c, hw, groups), "group_norm_backward: workspace too small");
  float* sums = (float*)workspace;
  const bool params = dgamma || dbeta;
  const Plan t = plan_slabs(n, c, hw, groups, 2, alignment_of(dy, x, dx));
  if (t.on_chip) {
    if (int rc = MTB_GN_PICK(backward_on_chip, t, activation, st, dy, x, gamma, beta, mean, rstd, dx, params ? sums : nullptr)) return rc;
  } else {
    MTB_REQUIRE((long long)n * groups < 65536 && n < 65536, "group_norm_backward: %d images of %d groups", n, groups);
    const int blocks = mtb_div_up(c, 32), splits = splits_of(n, hw, blocks);
    float* of_group = sums + 2LL * n * c * splits;
    const long long image = (long long)hw * c;
    MTB_LAUNCH(gn_bwd_sums_kernel, dim3(blocks, n, splits), 256, 0, st, dy, x, hw, c, groups, splits, gamma, beta, activation, mean, rstd, sums);
    MTB_LAUNCH(gn_bwd_groups_kernel, mtb_div_up((long long)n * groups, 4), 128, 0, st, sums, n, c, groups, splits, gamma,
               (float)(1.0 / ((double)(c / groups) * hw)), of_group);
    if (dx) MTB_LAUNCH(gn_bwd_dx_kernel, dim3(mtb_stream_grid(image, 256), n), 256, 0, st, dy, x, image, PoolDiv(c), PoolDiv(c / groups), groups, gamma, beta,
                       activation, mean, rstd, of_group, dx);
  }
  if (params) MTB_LAUNCH(gn_params_kernel, mtb_div_up(2LL * c, 32), 256, 0, st, sums, n, c, dgamma, dbeta);
  return MTB_OK;
}
