// GroupNorm over channels-last activations [n][hw][c], with an activation behind it, forward and backward.
//
// A group is M = (c / groups) * hw values of one image.  Forward: mean, r = 1 / sqrt(var + eps) over the group,
// xh = (x - mean) r, z = gamma xh + beta, y = f(z).  Backward, from the saved mean and r: dz = dy f'(z),
// dbeta = sum dz, dgamma = sum dz xh over images and positions, and dx = r (gamma dz - (A + xh B) / M) with
// A = sum gamma dz, B = sum gamma dz xh over the group.
//
// HBM-bound: 8 bytes a value forward, 12 backward, if the values stay on the chip between the sums and what is made of them.  So a cluster of CTAs holds
// a slab, some whole groups of one image, in its shared memory, each CTA a stretch of the positions; four CTAs or so on an SM, one of which loads
// while another one adds up or stores.  A thread copies (cp.async) and later reads its own vectors only, so the copies need no barrier; the CTAs exchange their sums
// through distributed shared memory.
// 256 x 128 x 56 x 56 with SiLU: forward 147 us (5.6 TB/s, 86 % of a copy), backward 252 to 260 (4.8 TB/s, 74 %; with ReLU 246).  What bounds the backward now: a CTA's time
// from its last value to its first store, in which the cluster waits for its slowest, and an SM has four of them to overlap (backward without the exchange 190 us).
// Its steps, each measured when it was made, took instructions and waits out of that time: 292 us at first, xh recomputed instead of written back 275, sums over
// rows all at once 258 and by halves 250, gamma from shared memory 247; what SiLU's exponent leaves (see sigmoid) costs 3.  The 64 registers of four CTAs are
// what it may not pass: 12 bytes spilled cost 20 us.  Tried: clusters that stay and fetch
// the next slab meanwhile (forward 155 us, backward 337), sums sent with st.async (152, 319), two readings from the L2 cache by tickets or by launches (backward
// 377), adding up while copies are on their way (+1 % to +11 %), marks for L2 (no change), CTAs that begin one after another (no change).
// A slab that no cluster can hold goes through memory twice instead, see the kernels at the end.
#include "colreduce.cuh"
#include <cooperative_groups.h>
#include <type_traits>

namespace {

namespace cg = cooperative_groups;

enum Activation { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2 };

__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int V>
__device__ __forceinline__ void copy_async(unsigned at, const float* from) {
  if (V == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else if (V == 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A CTA's shared memory is there for the others of its cluster once it has started.  So each arrives first of all and waits for the others just before it
// writes to them; its own values are on their way meanwhile.  A CTA without a cluster is one of one: the backward asks it too, since a branch here costs it
// registers that it has not (12 bytes spilled).
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

template <int V> struct alignas(4 * V) Vec { float v[V]; };
template <int V> __device__ __forceinline__ Vec<V>& vec(float* p) { return *reinterpret_cast<Vec<V>*>(p); }
template <int V> __device__ __forceinline__ Vec<V> all(float x) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = x;
  return r;
}
// Two values an instruction: arithmetic would otherwise take as long as memory does.
#define MTB_PAIRS(name, op, scalar)                                                                                                     \
  template <int V> __device__ __forceinline__ Vec<V> name(Vec<V> a, Vec<V> b) {                                                         \
    Vec<V> r;                                                                                                                           \
    if constexpr (V == 1) r.v[0] = scalar(a.v[0], b.v[0]);                                                                              \
    else                                                                                                                                \
      for (int i = 0; i < V; i += 2)                                                                                                    \
        asm("{.reg .b64 a, b, r; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; " op ".rn.f32x2 r, a, b; mov.b64 {%0, %1}, r;}"              \
            : "=f"(r.v[i]), "=f"(r.v[i + 1]) : "f"(a.v[i]), "f"(a.v[i + 1]), "f"(b.v[i]), "f"(b.v[i + 1]));                             \
    return r;                                                                                                                           \
  }
MTB_PAIRS(add, "add", __fadd_rn)
MTB_PAIRS(mul, "mul", __fmul_rn)
#undef MTB_PAIRS
template <int V> __device__ __forceinline__ Vec<V> fma(Vec<V> a, Vec<V> b, Vec<V> c) {
  Vec<V> r;
  if constexpr (V == 1) r.v[0] = fmaf(a.v[0], b.v[0], c.v[0]);
  else
#pragma unroll
    for (int i = 0; i < V; i += 2)
      asm("{.reg .b64 a, b, c, r; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7}; fma.rn.f32x2 r, a, b, c; mov.b64 {%0, %1}, r;}"
          : "=f"(r.v[i]), "=f"(r.v[i + 1])
          : "f"(a.v[i]), "f"(a.v[i + 1]), "f"(b.v[i]), "f"(b.v[i + 1]), "f"(c.v[i]), "f"(c.v[i + 1]));
  return r;
}
// 1 / (1 + e^-z).  e^-z = 2^h e^-r with h = -z log2 e as 32 bits have it and r = z + h ln 2 what that leaves, so small that e^-r = 1 - r; without r the error would
// grow with z, to 2^-18 of the result at -80.  By the approximate power and reciprocal of the hardware: under 2^-20 of itself.  Where e^-z overflows or vanishes, r
// may be anything and counts nothing: it is cut to 1/16, a NaN too.
template <int V> __device__ __forceinline__ Vec<V> sigmoid(Vec<V> z) {
  Vec<V> e = mul(z, all<V>(-1.4426950408889634f)), r = fma(e, all<V>(0.6931471805599453f), z);
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = __saturatef(fmaf(r.v[i], 8.f, 0.5f));
#pragma unroll
  for (int i = 0; i < V; ++i) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.v[i]));
  e = fma(e, fma(r, all<V>(-0.125f), all<V>(1.0625f)), all<V>(1.f));
#pragma unroll
  for (int i = 0; i < V; ++i) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e.v[i]));
  return e;
}
template <int V, int ACT> __device__ __forceinline__ Vec<V> activated(Vec<V> z) {
  if (ACT == ACT_SILU) return mul(z, sigmoid(z));
  if (ACT == ACT_RELU)
#pragma unroll
    for (int i = 0; i < V; ++i) z.v[i] = z.v[i] < 0.f ? 0.f : z.v[i];
  return z;
}
template <int V, int ACT> __device__ __forceinline__ Vec<V> activated_grad(Vec<V> dy, Vec<V> z) {
  if (ACT == ACT_SILU) {
    const Vec<V> s = sigmoid(z);
    return mul(dy, fma(mul(s, z), fma(s, all<V>(-1.f), all<V>(1.f)), s));
  }
  if (ACT == ACT_RELU)
#pragma unroll
    for (int i = 0; i < V; ++i) dy.v[i] = z.v[i] < 0.f ? 0.f : dy.v[i];
  return dy;
}

// The same of one value, the activation an argument.
__device__ __forceinline__ float activate(float z, int act) {
  const Vec<1> v{{z}};
  return (act == ACT_SILU ? activated<1, ACT_SILU>(v) : act == ACT_RELU ? activated<1, ACT_RELU>(v) : v).v[0];
}
// dy f'(z); a ReLU passes what is at zero, as ReLU's own backward does
__device__ __forceinline__ float activate_grad(float dy, float z, int act) {
  const Vec<1> d{{dy}}, v{{z}};
  return (act == ACT_SILU ? activated_grad<1, ACT_SILU>(d, v) : act == ACT_RELU ? activated_grad<1, ACT_RELU>(d, v) : d).v[0];
}

// ---------------------------------------------------------------- a slab on the chip

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct Slabs {
  int hw, c, groups, each;  // channels of a group
  int wide, slabs, units;   // channels of a slab (the last of an image may have fewer), slabs of an image, of all images
  int of_slab;              // groups of a slab
  int ctas, stretch;        // CTAs of a cluster, positions of a CTA
  int lanes, rows;          // threads to a position (its vectors, up to a power of two), positions that the CTA's threads take at a time
  int lane_bits, row_bits;  // of the two
  int steps;                // positions of a thread at most
  // A slot is what a warp makes of its rows, or a row of more than a warp.  Where a thread's channels are of several groups it has several entries in it; `merged`
  // lanes' entries are made one, and a group has `entries` of them.
  int of_vector, entries, merged, slots, slot_rows, slot_stride;
  bool vectors;                    // gamma and beta can be read as the values are
  float inv_positions, inv_group;  // 1 / hw, 1 / M
  PoolDiv by_slabs, by_each;
};

// What a thread has to do.
template <int V>
struct Share {
  int rank, row, col, full, more;  // CTA of the cluster; position within a step, first channel; steps of all rows, rows with one more
  int positions, steps;            // of the CTA, of the thread
  int group[V];                    // of each channel, within the slab
  __device__ __forceinline__ Share(const Slabs& p, int rank_) : rank(rank_) {
    row = threadIdx.x >> p.lane_bits;
    col = (threadIdx.x & (p.lanes - 1)) * V;
    const int left = p.hw - rank * p.stretch;
    positions = p.stretch < left ? p.stretch : left;
    full = positions >> p.row_bits;
    more = positions & (p.rows - 1);
    steps = full + (row < more ? 1 : 0);
    unsigned in;
    group[0] = (int)p.by_each.divmod((unsigned)col, in);
#pragma unroll
    for (int i = 1; i < V; ++i) {
      const bool next = ++in == (unsigned)p.each;
      group[i] = group[i - 1] + (next ? 1 : 0);
      if (next) in = 0;
    }
  }
  __device__ __forceinline__ int slot(const Slabs& p) const { return p.lanes < 32 ? threadIdx.x >> 5 : row; }
  __device__ __forceinline__ int of_slot(const Slabs& p, int slot) const {  // positions
    const int extra = more - slot * p.slot_rows;
    return full * p.slot_rows + (extra < 0 ? 0 : extra < p.slot_rows ? extra : p.slot_rows);
  }
};
struct Unit {
  int n, c0, width, groups;  // image, first channel, channels, their groups
  __device__ __forceinline__ Unit(const Slabs& p, int unit) {
    unsigned slab;
    n = (int)p.by_slabs.divmod((unsigned)unit, slab);
    c0 = (int)slab * p.wide;
    width = p.wide < p.c - c0 ? p.wide : p.c - c0;
    groups = p.of_slab < p.groups - (int)slab * p.of_slab ? p.of_slab : p.groups - (int)slab * p.of_slab;
  }
  // of the thread's first value
  template <int V>
  __device__ __forceinline__ long long first(const Slabs& p, const Share<V>& s) const {
    return ((long long)n * p.hw + s.rank * p.stretch + s.row) * p.c + c0 + s.col;
  }
};

// f(j) for the thread's steps, U at a time; `full` is the same for all threads that have any.
template <int U = 4, class F>
__device__ __forceinline__ void each_step(int full, int steps, F f) {
  int j = 0;
  for (; j + U <= full; j += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) f(j + u);
  }
  for (; j < full; ++j) f(j);
  if (j < steps) f(j);
}

// V values of gamma or beta, or as many of `otherwise`.
template <int V>
__device__ __forceinline__ Vec<V> parameter(const float* from, bool there, bool vectors, float otherwise) {
  Vec<V> r = all<V>(otherwise);
  if (from && there) {
    if (vectors) r = *reinterpret_cast<const Vec<V>*>(from);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) r.v[i] = from[i];
  }
  return r;
}

// Adds up over the lanes of a warp that hold the same channels.
__device__ __forceinline__ float sum_rows(float t, const Slabs& p) {
  for (int o = p.lanes; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// A warp's mean and M2 of each of its entries, to slots [slots][lanes * E / merged]; E: entries of a thread.
template <int V, int E>
__device__ __forceinline__ void slot_statistics(float* mine, int full, int steps, const Slabs& p, const Share<V>& s, float2* slots) {
  constexpr int N = V / E;  // channels of an entry
  Vec<V> sum = all<V>(0.f), m2 = sum, off = sum;
  each_step(full, steps, [&](int j) { sum = add(sum, vec<V>(mine + j * kThreads * V)); });
  const int count = s.of_slot(p, s.slot(p)) * p.merged * N;
  const float inv = count ? __frcp_rn((float)count) : 0.f;
  float mean[E];
#pragma unroll
  for (int k = 0; k < E; ++k) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) t += sum.v[k * N + i];
    for (int o = 1; o < p.merged; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    mean[k] = sum_rows(t, p) * inv;
#pragma unroll
    for (int i = 0; i < N; ++i) off.v[k * N + i] = -mean[k];
  }
  each_step(full, steps, [&](int j) {
    const Vec<V> d = add(vec<V>(mine + j * kThreads * V), off);
    m2 = fma(d, d, m2);
  });
  const int in_row = threadIdx.x & (p.lanes - 1);
  float2* to = slots + s.slot(p) * (p.lanes * E / p.merged) + in_row / p.merged * E;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) t += m2.v[k * N + i];
    for (int o = 1; o < p.merged; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    t = sum_rows(t, p);
    if ((threadIdx.x & 31) < p.lanes && (in_row & (p.merged - 1)) == 0) to[k] = make_float2(mean[k], t);
  }
}

template <int V, int ACT>
__global__ void __launch_bounds__(kThreads, 4) gn_forward_kernel(const __grid_constant__ Slabs p, const float* __restrict__ x, const float* __restrict__ gamma,
                                                                  const float* __restrict__ beta, float eps, float* __restrict__ y,
                                                                  float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  extern __shared__ __align__(16) float held[];  // [positions][lanes][V]; the warps' (mean, M2); the CTAs' [ctas][groups of a slab]
  cg::cluster_group cluster = cg::this_cluster();
  if (p.ctas > 1) cluster_arrive();
  const Share<V> s(p, p.ctas > 1 ? (int)cluster.block_rank() : 0);
  const Unit u(p, blockIdx.x / p.ctas);
  const int per_slot = p.lanes * p.of_vector / p.merged;
  float* mine = held + threadIdx.x * V;
  float2 *slots = (float2*)(held + (p.stretch * p.lanes * V + 1) / 2 * 2), *of_cta = slots + p.slots * per_slot;
  const bool active = s.col < u.width;
  const int full = active ? s.full : 0, steps = active ? s.steps : 0;
  const unsigned step = p.rows * p.c;  // of an image's values
  mtb_wait_prior();
  mtb_launch_dependents();  // not before: the next kernel's CTAs would take places from this one's
  const float* from = x + u.first(p, s);
  const unsigned at = (unsigned)__cvta_generic_to_shared(mine);
  each_step(full, steps, [&](int j) { copy_async<V>(at + j * kThreads * V * 4, from + j * step); });
  Vec<V> scale = parameter<V>(gamma + u.c0 + s.col, gamma && active, p.vectors, 1.f);
  const Vec<V> shift = parameter<V>(beta + u.c0 + s.col, beta && active, p.vectors, 0.f);
  copies_done();
  if (V >= 4 && p.of_vector == 4) slot_statistics<V, V >= 4 ? 4 : 1>(mine, full, steps, p, s, slots);
  else if (V >= 2 && p.of_vector == 2) slot_statistics<V, V >= 2 ? 2 : 1>(mine, full, steps, p, s, slots);
  else slot_statistics<V, 1>(mine, full, steps, p, s, slots);
  __syncthreads();
  if (p.ctas > 1) cluster_wait();
  // Chan's update for several: the mean of the means, and M2_k + n_k (mean_k - mean)^2 added up.  The CTA's of a group by eight lanes, a slot each, who give it to
  // each CTA of the cluster ...
  const float share = (float)(V / p.of_vector * p.merged), inv = __frcp_rn((float)(s.positions * p.each));
  const int w = threadIdx.x & 7;
  for (int g = threadIdx.x >> 3; g < (p.of_slab + 3) / 4 * 4; g += kThreads / 8) {  // whole warps
    const float2* entry = slots + w * per_slot + g * p.entries;
    const bool in = w < p.slots && g < u.groups;
    const float count = in ? (float)s.of_slot(p, w) * share : 0.f;
    float mean = 0.f, m2 = 0.f;
    if (in)
      for (int q = 0; q < p.entries; ++q) mean += entry[q].x;
    mean *= count;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
    mean *= inv;
    if (in)
      for (int q = 0; q < p.entries; ++q) {
        const float d = entry[q].x - mean;
        m2 += entry[q].y + count * (d * d);
      }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, o);
    float2* to = of_cta + s.rank * p.of_slab + g;
    if (g < u.groups) {
      if (p.ctas == 1) *to = make_float2(mean, m2);  // by eight lanes alike
      else
        for (int r = w; r < p.ctas; r += 8) *cluster.map_shared_rank(to, r) = make_float2(mean, m2);
    }
  }
  if (p.ctas > 1) cluster.sync(); else __syncthreads();
  // ... and the group's
  Vec<V> minus = all<V>(0.f);
  float mean = 0.f, rstd = 0.f;
  const float one = p.ctas > 1 ? (float)p.stretch * p.inv_positions : 1.f, end = 1.f - one * (float)(p.ctas - 1), n_one = (float)(p.stretch * p.each),
              n_end = (float)((p.hw - (p.ctas - 1) * p.stretch) * p.each);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (active && (i == 0 || s.group[i] != s.group[i - 1 < 0 ? 0 : i - 1])) {
      const float2* theirs = of_cta + s.group[i];
      mean = 0.f;
      float m2 = 0.f;
#pragma unroll 8
      for (int r = 0; r < p.ctas; ++r) mean += theirs[r * p.of_slab].x * (r + 1 < p.ctas ? one : end);
#pragma unroll 8
      for (int r = 0; r < p.ctas; ++r) {
        const float2 e = theirs[r * p.of_slab];
        const float d = e.x - mean;
        m2 += e.y + (r + 1 < p.ctas ? n_one : n_end) * (d * d);
      }
      rstd = rsqrtf(m2 * p.inv_group + eps);
      if (s.rank == 0 && s.row == 0 && s.group[i] * p.each == s.col + i) {
        const long long k = (long long)u.n * p.groups + u.c0 / p.each + s.group[i];
        mean_out[k] = mean;
        rstd_out[k] = rstd;
      }
    }
    minus.v[i] = -mean;
    scale.v[i] *= rstd;
  }
  float* to = y + u.first(p, s);
  each_step(full, steps, [&](int j) {
    *reinterpret_cast<Vec<V>*>(to + j * step) = activated<V, ACT>(fma(add(vec<V>(mine + j * kThreads * V), minus), scale, shift));
  });
}

// Sums of a and b over the lanes of a warp that hold the same channels, to `to` and to [lanes * V] behind.  While a lane has several values, it gives half of them
// to the lane opposite for half of its own: 7 shuffles for 8 values of 8 rows instead of 24.
template <int V>
__device__ __forceinline__ void add_rows(Vec<V> a, Vec<V> b, int lane, int lanes, float* to) {
  if (lanes >= 32) {
    vec<V>(to) = a;
    vec<V>(to + lanes * V) = b;
    return;
  }
  bool upper = lane & 16;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float give = upper ? a.v[i] : b.v[i], keep = upper ? b.v[i] : a.v[i];
    a.v[i] = keep + __shfl_xor_sync(0xffffffffu, give, 16);
  }
  if (upper) to += lanes * V;
  int o = 8;
  if (V == 4) {
    if (lanes > 8) { vec<V>(to) = a; return; }
    upper = lane & 8;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float give = upper ? a.v[i] : a.v[V / 2 + i], keep = upper ? a.v[V / 2 + i] : a.v[i];
      a.v[i] = keep + __shfl_xor_sync(0xffffffffu, give, 8);
    }
    if (upper) to += 2;
    o = 4;
  }
  if (V >= 2) {
    if (lanes > o) { vec<2>(to) = Vec<2>{{a.v[0], a.v[1 % V]}}; return; }
    upper = lane & o;
    const float give = upper ? a.v[0] : a.v[1 % V], keep = upper ? a.v[1 % V] : a.v[0];
    a.v[0] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    if (upper) to += 1;
    o >>= 1;
  }
  float t = a.v[0];
  int first = 0;  // of the lanes that differ in these bits one writes
  for (; o >= lanes; o >>= 1) {
    t += __shfl_xor_sync(0xffffffffu, t, o);
    first |= o;
  }
  if ((lane & first) == 0) *to = t;
}

// sums (may be NULL): per image and channel the sums of dz and of dz xh, [n][2][c].  dx may be NULL.
template <int V, int ACT>
__global__ void __launch_bounds__(kThreads, 4) gn_backward_kernel(const __grid_constant__ Slabs p, const float* __restrict__ dy, const float* __restrict__ x,
                                                                   const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                   const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ dx,
                                                                   float* __restrict__ sums) {
  extern __shared__ __align__(16) float held[];  // [2][positions][lanes][V]; the warps' sums; the CTAs' of channels and of groups
  cg::cluster_group cluster = cg::this_cluster();
  cluster_arrive();
  const Share<V> s(p, p.ctas > 1 ? (int)cluster.block_rank() : 0);
  const Unit u(p, blockIdx.x / p.ctas);
  const int plane = p.stretch * p.lanes * V, both = 2 * p.lanes * V;  // two sums of each channel
  float *mine = held + threadIdx.x * V, *of_warp = held + 2 * plane, *weights = of_warp + p.slots * p.slot_stride, *of_channel = weights + (p.lanes * V + 3 & ~3);
  float2* of_cta = (float2*)(of_channel + p.ctas * both);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool active = s.col < u.width;
  const int full = active ? s.full : 0, steps = active ? s.steps : 0;
  const unsigned step = p.rows * p.c;
  mtb_wait_prior();
  mtb_launch_dependents();  // not before: the next kernel's CTAs would take places from this one's
  {
    const float *from = x + u.first(p, s), *from2 = dy + u.first(p, s);
    const unsigned at = (unsigned)__cvta_generic_to_shared(mine);
    each_step(full, steps, [&](int j) {
      copy_async<V>(at + j * kThreads * V * 4, from + j * step);
      copy_async<V>(at + plane * 4 + j * kThreads * V * 4, from2 + j * step);
    });
  }
  for (int ch = threadIdx.x; ch < u.width; ch += kThreads) {  // for the groups' sums
    if (gamma) copy_async<1>((unsigned)__cvta_generic_to_shared(weights + ch), gamma + u.c0 + ch); else weights[ch] = 1.f;
  }
  Vec<V> ga = parameter<V>(gamma + u.c0 + s.col, gamma && active, p.vectors, 1.f);
  const Vec<V> be = parameter<V>(beta + u.c0 + s.col, beta && active, p.vectors, 0.f);
  Vec<V> minus = all<V>(0.f), r = minus, a = minus, b = minus;
  if (active) {
    const long long k = (long long)u.n * p.groups + u.c0 / p.each;
    if (p.of_vector == 1) {
      minus = all<V>(-mean[k + s.group[0]]);
      r = all<V>(rstd[k + s.group[0]]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        minus.v[i] = -mean[k + s.group[i]];
        r.v[i] = rstd[k + s.group[i]];
      }
    }
  }
  ga = mul(ga, r);
  copies_done();
  each_step<6>(full, steps, [&](int j) {  // dz takes the place of dy
    const Vec<V> v = add(vec<V>(mine + j * kThreads * V), minus);
    const Vec<V> d = activated_grad<V, ACT>(vec<V>(mine + plane + j * kThreads * V), fma(v, ga, be));
    a = add(a, d);
    b = fma(d, v, b);
    if (ACT != ACT_NONE) vec<V>(mine + plane + j * kThreads * V) = d;
  });
  b = mul(b, r);
  add_rows<V>(a, b, lane, p.lanes, of_warp + s.slot(p) * p.slot_stride + s.col);
  __syncthreads();
  cluster_wait();
  if (dx) {
    const int entries = p.each * p.slots;
    for (int g = warp; g < u.groups; g += kWarps) {  // the group's in the CTA, given to each CTA of the cluster
      float t = 0.f, t2 = 0.f;
      for (int e = lane; e < entries; e += 32) {
        unsigned in;
        const float* from = of_warp + p.by_each.divmod((unsigned)e, in) * p.slot_stride + g * p.each;
        const float weight = weights[g * p.each + in];
        t = fmaf(weight, from[in], t);
        t2 = fmaf(weight, from[p.lanes * V + in], t2);
      }
      const float2 both_sums = make_float2(warp_sum(t) * p.inv_group, warp_sum(t2) * p.inv_group);
      float2* to = of_cta + s.rank * p.of_slab + g;
      if (lane < p.ctas) *(p.ctas > 1 ? cluster.map_shared_rank(to, lane) : to) = both_sums;
    }
  }
  if (sums) {
    for (int k = kThreads - 1 - threadIdx.x; k < both; k += kThreads) {  // the CTA's of its channels, by the warps without a group
      const int second = k >= p.lanes * V, ch = k - (second ? p.lanes * V : 0);
      if (ch >= u.width) continue;
      float t = 0.f;
#pragma unroll 8
      for (int w = 0; w < p.slots; ++w) t += of_warp[w * p.slot_stride + k];
      if (p.ctas > 1) cluster.map_shared_rank(of_channel, 0)[s.rank * both + k] = t;
      else sums[((long long)u.n * 2 + second) * p.c + u.c0 + ch] = t;
    }
  }
  if (p.ctas > 1) cluster.sync(); else __syncthreads();
  if (p.ctas > 1 && sums && s.rank == 0) {
    for (int k = threadIdx.x; k < both; k += kThreads) {
      const int second = k >= p.lanes * V, ch = k - (second ? p.lanes * V : 0);
      if (ch >= u.width) continue;
      float t = 0.f;
#pragma unroll 8
      for (int q = 0; q < p.ctas; ++q) t += of_channel[q * both + k];
      sums[((long long)u.n * 2 + second) * p.c + u.c0 + ch] = t;
    }
  }
  if (!dx) return;
  float group_a = 0.f, group_b = 0.f;  // -A / M, -B / M
  auto add_up = [&](int group) {
    group_a = group_b = 0.f;
#pragma unroll 8
    for (int q = 0; q < p.ctas; ++q) {
      const float2 e = of_cta[q * p.of_slab + group];
      group_a -= e.x;
      group_b -= e.y;
    }
  };
  if (p.of_vector == 1) {
    if (active) add_up(s.group[0]);
    a = all<V>(group_a);
    b = all<V>(group_b);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (active && (i == 0 || s.group[i] != s.group[i - 1 < 0 ? 0 : i - 1])) add_up(s.group[i]);
      a.v[i] = group_a;
      b.v[i] = group_b;
    }
  }
  a = mul(a, r);
  b = mul(mul(b, r), r);  // of x - mean; finite for every r below 1.8e19, as any eps of 1e-38 makes it
  float* to = dx + u.first(p, s);
  each_step<2>(full, steps, [&](int j) {
    *reinterpret_cast<Vec<V>*>(to + j * step) = fma(add(vec<V>(mine + j * kThreads * V), minus), b, fma(ga, vec<V>(mine + plane + j * kThreads * V), a));
  });
}

// dgamma and dbeta: the sums over the images, 32 columns of [n][2 c] a CTA, in a fixed order; of many images first those of stretches of them, to
// stretches[gridDim.y][2 c].  Backward of 2000 images of 64 x 8 x 8 28 us, 37 with one stretch; of 70001 rows of 96 channels 438, not 1007.
constexpr int kStretches = 128;
int stretches_of(int n) { return n < 1024 ? 1 : n / 256 < kStretches ? n / 256 : kStretches; }

__global__ void __launch_bounds__(256) gn_params_kernel(const float* __restrict__ sums, int n, int c, float* __restrict__ stretches, float* __restrict__ dgamma,
                                                         float* __restrict__ dbeta) {
  mtb_wait_prior();
  mtb_launch_dependents();
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  const int each = (n + gridDim.y - 1) / gridDim.y, first = blockIdx.y * each, end = first + each < n ? first + each : n;
  double sum = 0;  // of sums of eight in 32 bits
  if (col < 2 * c)
    for (unsigned i = first + row; i < (unsigned)end; i += 64) {
      float v[8], t = 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i + 8 * u < (unsigned)end ? sums[(long long)(i + 8 * u) * 2 * c + col] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) t += v[u];
      sum += t;
    }
  part[row][lane] = (float)sum;
  __syncthreads();
  if (row != 0 || col >= 2 * c) return;
  for (int k = 1; k < 8; ++k) sum += part[k][lane];
  const float t = (float)sum;
  if (gridDim.y > 1) stretches[(long long)blockIdx.y * 2 * c + col] = t;
  else if (col < c) { if (dbeta) dbeta[col] = t; }
  else if (dgamma) dgamma[col - c] = t;
}

// ---------------------------------------------------------------- a slab through memory

// Images that no cluster can hold, and groups of more channels than a CTA has threads' vectors: partial statistics of stretches of positions,
// statistics, result.  Bound by latency and by reading twice: 2 x 64 x 400 x 400 in 2 groups forward 82 us (25 is HBM's time for 8 bytes a value; 170 with a value a thread
// on its way instead of kAhead), backward 114.  Rare among images that are trained on, so simple.

constexpr int kAhead = 8;

// z of `v`, a value less the mean, with the roundings of the kernels above: a backward that goes through memory finds each ReLU on the side of zero on
// which a forward on the chip left it.
__device__ __forceinline__ float scaled(float v, float gamma, float rstd, float beta) { return fmaf(v, __fmul_rn(gamma, rstd), beta); }

// Chan's update of (count, mean, M2) by another such.
__device__ __forceinline__ void merge(float& count, float& mean, float& m2, float nb, float mb, float qb) {
  if (nb == 0.f) return;
  const float total = count + nb, d = mb - mean;
  mean += d * (nb / total);
  m2 += qb + d * d * count * (nb / total);
  count = total;
}
// Those of a warp, to its first lane.
__device__ __forceinline__ void merge_lanes(float& count, float& mean, float& m2) {
  for (int o = 16; o > 0; o >>= 1) {
    const float nb = __shfl_down_sync(0xffffffffu, count, o), mb = __shfl_down_sync(0xffffffffu, mean, o), qb = __shfl_down_sync(0xffffffffu, m2, o);
    merge(count, mean, m2, nb, mb, qb);
  }
}

// partial[group][split][3]: count, mean, M2.  A thread's values, less the first of them, kAhead at a time: their sum, and their squares about their own mean, in 32
// bits; what comes of kAhead is added up in 64, so that the error does not grow with the image.  (Where there are no more than kAhead that is left out: 65600
// rows of 1028 channels forward 473 us instead of 492.)
__global__ void __launch_bounds__(256) gn_stats_kernel(const float* __restrict__ x, int hw, int c, int groups, int splits, PoolDiv by_each,
                                                        float* __restrict__ partial) {
  mtb_wait_prior();
  mtb_launch_dependents();
  __shared__ float sm[3][8];
  const int each = c / groups, g = blockIdx.x % groups, n = blockIdx.x / groups, stretch = (hw + splits - 1) / splits;
  const int p0 = blockIdx.y * stretch, p1 = p0 + stretch < hw ? p0 + stretch : hw;
  const float* base = x + ((long long)n * hw + p0) * c + (long long)g * each;
  const unsigned total = p1 > p0 ? (unsigned)(p1 - p0) * each : 0;  // the stretch's values of the group, 256 a step, kAhead steps at once
  const bool more = total > 256 * kAhead;
  double sum = 0, about = 0, between = 0;  // of all, of the squares about the means of kAhead, of those means' squares times kAhead
  float pivot = 0.f, mean = 0.f, m2 = 0.f;
  if (threadIdx.x < total) {
    unsigned ch;
    const unsigned pos = by_each.divmod(threadIdx.x, ch);
    pivot = base[(long long)pos * c + ch];
  }
  for (unsigned e = threadIdx.x; e < total; e += 256 * kAhead) {
    float v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      v[u] = pivot;
      if (e + 256 * u < total) {
        unsigned ch;
        const unsigned pos = by_each.divmod(e + 256 * u, ch);
        v[u] = base[(long long)pos * c + ch];
      }
    }
    const unsigned left = (total - e + 255) / 256;
    const float inv = left < kAhead ? __frcp_rn((float)left) : 1.f / kAhead;
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) s += v[u] -= pivot;
    const float own = s * inv;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float d = u < left ? v[u] - own : 0.f;
      q += d * d;
    }
    if (more) {
      sum += s;
      about += q;
      between += (double)s * s * inv;
    }
    mean = pivot + own;
    m2 = q;
  }
  float count = threadIdx.x < total ? (float)((total - threadIdx.x + 255) / 256) : 0.f;
  if (more) {  // each thread has some
    const double shift = sum / count;
    mean = (float)(pivot + shift);
    m2 = (float)(about + (between - sum * shift));
  }
  merge_lanes(count, mean, m2);
  if ((threadIdx.x & 31) == 0) { sm[0][threadIdx.x >> 5] = count; sm[1][threadIdx.x >> 5] = mean; sm[2][threadIdx.x >> 5] = m2; }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 8; ++w) merge(count, mean, m2, sm[0][w], sm[1][w], sm[2][w]);
  float* to = partial + ((long long)blockIdx.x * splits + blockIdx.y) * 3;
  to[0] = count;
  to[1] = mean;
  to[2] = m2;
}

__global__ void __launch_bounds__(128) gn_stats_final_kernel(const float* __restrict__ partial, int count, int splits, float eps, float* __restrict__ mean_out,
                                                              float* __restrict__ rstd_out) {
  mtb_wait_prior();
  mtb_launch_dependents();
  const int k = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;  // a warp a group
  if (k >= count) return;
  float n = 0.f, mean = 0.f, m2 = 0.f;
  for (int i = lane; i < splits; i += 32) {
    const float* q = partial + ((long long)k * splits + i) * 3;
    merge(n, mean, m2, q[0], q[1], q[2]);
  }
  merge_lanes(n, mean, m2);
  if (lane != 0) return;
  mean_out[k] = mean;
  rstd_out[k] = 1.f / sqrtf(m2 / n + eps);
}

__global__ void __launch_bounds__(256) gn_apply_kernel(const float* __restrict__ x, long long image, PoolDiv by_c, PoolDiv by_each, int groups,
                                                        const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                        const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ y) {
  mtb_wait_prior();
  mtb_launch_dependents();
  const long long first = blockIdx.x * image;
  const unsigned values = (unsigned)image;
  for (unsigned i0 = blockIdx.y * 256 * kAhead + threadIdx.x; i0 < values; i0 += gridDim.y * 256 * kAhead) {
    float v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u] = i0 + 256 * u < values ? x[first + i0 + 256 * u] : 0.f;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const unsigned i = i0 + 256 * u;
      if (i >= values) break;
      unsigned ch, unused;
      by_c.divmod(i, ch);
      const int k = blockIdx.x * groups + by_each.divmod(ch, unused);
      y[first + i] = activate(scaled(__fadd_rn(v[u], -mean[k]), gamma ? gamma[ch] : 1.f, rstd[k], beta ? beta[ch] : 0.f), act);
    }
  }
}

// A sum of more than kChain terms is one of 64 bits, so that its error does not grow with the image.  Fewer have no use for it: 65600 rows of 1028 channels
// backward 4.3 ms, 5.3 with 64 bits everywhere.
constexpr int kChain = 64;
template <bool LONG> using SumOf = std::conditional_t<LONG, double, float>;

// partial[split][n][2][c]: the sums of dz and of dz xh over a stretch of positions.  A CTA has 32 channels, of an image's `blocks`.  LONG: more than kChain rows a
// thread.
template <bool LONG>
__global__ void __launch_bounds__(256) gn_bwd_sums_kernel(const float* __restrict__ dy, const float* __restrict__ x, int hw, int c, int groups, int splits, int blocks,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ partial) {
  mtb_wait_prior();
  mtb_launch_dependents();
  __shared__ float sa[8][33], sb[8][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, n = blockIdx.x / blocks, ch = (blockIdx.x - n * blocks) * 32 + lane, stretch = (hw + splits - 1) / splits;
  const int p0 = blockIdx.y * stretch, p1 = p0 + stretch < hw ? p0 + stretch : hw;
  SumOf<LONG> a = 0, b = 0;
  if (ch < c) {
    const int k = n * groups + ch / (c / groups);
    const float mu = mean[k], r = rstd[k], ga = gamma ? gamma[ch] : 1.f, be = beta ? beta[ch] : 0.f;
    if constexpr (LONG) {  // sums of kRows in 32 bits
      constexpr int kRows = 4;
      for (int s = p0 + row; s < p1; s += 8 * kRows) {
        float v[kRows], d[kRows], ta = 0.f, tb = 0.f;
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          const long long i = ((long long)n * hw + s + 8 * u) * c + ch;
          v[u] = s + 8 * u < p1 ? x[i] : 0.f;
          d[u] = s + 8 * u < p1 ? dy[i] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          if (s + 8 * u >= p1) break;
          const float less = __fadd_rn(v[u], -mu), dz = activate_grad(d[u], scaled(less, ga, r, be), act);
          ta += dz;
          tb += dz * (less * r);
        }
        a += ta;
        b += tb;
      }
    } else {
#pragma unroll 4
      for (int s = p0 + row; s < p1; s += 8) {
        const long long i = ((long long)n * hw + s) * c + ch;
        const float v = __fadd_rn(x[i], -mu), xh = v * r, dz = activate_grad(dy[i], scaled(v, ga, r, be), act);
        a += dz;
        b += dz * xh;
      }
    }
  }
  sa[row][lane] = (float)a;
  sb[row][lane] = (float)b;
  __syncthreads();
  if (row == 0 && ch < c) {
    for (int k = 1; k < 8; ++k) { a += sa[k][lane]; b += sb[k][lane]; }
    float* to = partial + ((long long)blockIdx.y * (gridDim.x / blocks) + n) * 2 * c + ch;
    to[0] = (float)a;
    to[c] = (float)b;
  }
}

// sums[n][2][c] over the splits, in place of the first; then A / M and B / M of each group.  A warp a group.  LONG: more than kChain splits, or channels a lane.
template <bool LONG>
__global__ void __launch_bounds__(128) gn_bwd_groups_kernel(float* __restrict__ sums, int n, int c, int groups, int splits, const float* __restrict__ gamma,
                                                             float inv_m, float* __restrict__ of_group) {
  mtb_wait_prior();
  mtb_launch_dependents();
  const int k = blockIdx.x * 4 + (threadIdx.x >> 5), each = c / groups;
  if (k >= n * groups) return;
  float* s = sums + (long long)(k / groups) * 2 * c + (k % groups) * each;
  SumOf<LONG> a = 0, b = 0;
  for (int ch = threadIdx.x & 31; ch < each; ch += 32) {
    SumOf<LONG> u = 0, v = 0;
    for (int i = 0; i < splits; ++i) {
      u += s[(long long)i * n * 2 * c + ch];
      v += s[(long long)i * n * 2 * c + c + ch];
    }
    s[ch] = (float)u;
    s[c + ch] = (float)v;
    const float ga = gamma ? gamma[k % groups * each + ch] : 1.f;
    a += ga * u;
    b += ga * v;
  }
  const float both[2] = {warp_sum((float)a), warp_sum((float)b)};
  if ((threadIdx.x & 31) == 0) {
    of_group[2 * k] = both[0] * inv_m;
    of_group[2 * k + 1] = both[1] * inv_m;
  }
}

__global__ void __launch_bounds__(256) gn_bwd_dx_kernel(const float* __restrict__ dy, const float* __restrict__ x, long long image, PoolDiv by_c, PoolDiv by_each,
                                                         int groups, const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd,
                                                         const float* __restrict__ of_group, float* __restrict__ dx) {
  mtb_wait_prior();
  mtb_launch_dependents();
  const long long first = blockIdx.x * image;
  const unsigned values = (unsigned)image;
  for (unsigned i0 = blockIdx.y * 256 * kAhead + threadIdx.x; i0 < values; i0 += gridDim.y * 256 * kAhead) {
    float v[kAhead], d[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool in = i0 + 256 * u < values;
      v[u] = in ? x[first + i0 + 256 * u] : 0.f;
      d[u] = in ? dy[first + i0 + 256 * u] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const unsigned i = i0 + 256 * u;
      if (i >= values) break;
      unsigned ch, unused;
      by_c.divmod(i, ch);
      const int k = blockIdx.x * groups + by_each.divmod(ch, unused);
      const float ga = gamma ? gamma[ch] : 1.f, r = rstd[k], less = __fadd_rn(v[u], -mean[k]), xh = less * r;
      const float dz = activate_grad(d[u], scaled(less, ga, r, beta ? beta[ch] : 0.f), act);
      dx[first + i] = r * (ga * dz - (of_group[2 * k] + xh * of_group[2 * k + 1]));
    }
  }
}

// ---------------------------------------------------------------- host

struct Plan {
  bool on_chip;
  int v, smem;
  Slabs s;
};

constexpr int kMostShared = 225 * 1024, kShared = 227 * 1024;  // of a CTA, of an SM for CTAs that take 1 KB more than they ask for

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// planes: tensors that the cluster holds (1 forward, 2 backward).  Of slabs of several widths (the widest for so many lanes) and clusters of several sizes the pair is
// taken that is done first.  A turn of all SMs takes 6.5 us, 0.015 us for each value of each thread of an SM's CTAs and 0.01 for one thread's, fitted to the forward:
// hardly more if four CTAs share an SM than if two do (256 x 128 x 56 x 56 forward: 13.8 turns of two CTAs of 100 KB or four of 51, 147 and 145 us), so the number of
// turns decides, and what fills the shared memory wins.  The backward is priced the same, by its two tensors: of 256 x 128 x 56 x 56 it takes clusters of eight
// CTAs of 53 KB.  Measured beside that: a single CTA on an SM, with nobody beside it while it loads, 2.4 us; pieces of 32 bytes 3.7 (of 64 bytes 0.15);
// 16 CTAs wait 2 us longer for one another, one CTA for nobody.  What the price does not see: 30 x 150 x 37 x 41 backward takes clusters of eight for 30 channels,
// 1200 CTAs, 30 us; 71 such clusters fit the GPU at once, so the last few have a third turn to themselves.
Plan plan_slabs(int n, int c, int hw, int groups, int planes, int alignment) {
  Plan t{};
  const int each = c / groups;
  t.v = c % 4 == 0 && alignment % 16 == 0 ? 4 : c % 2 == 0 && alignment % 8 == 0 ? 2 : 1;
  const int unit = t.v / gcd(each, t.v);  // groups whose channels are whole vectors
  const int sms = mtb_sm_count(), of_vector = t.v / gcd(each, t.v);
  double best = 0;
  for (int lanes = 1, before = 0; lanes <= kThreads; lanes *= 2) {
    int of_slab = lanes * t.v / each / unit * unit;
    if (of_slab > groups) of_slab = groups;
    if (of_slab == before) continue;
    before = of_slab;
    const int wide = of_slab * each, rows = kThreads / lanes, slabs = (groups + of_slab - 1) / of_slab;
    const long long units = (long long)n * slabs;
    // a group's lanes become one where they are a power of two of whole vectors
    int merged = 1;
    if (of_vector == 1 && ((each / t.v) & (each / t.v - 1)) == 0) merged = each / t.v < 32 ? each / t.v : 32;
    const int entries = each * of_vector / t.v / merged, slots = lanes < 32 ? kWarps : rows, slot_stride = 2 * lanes * t.v + 4;
    for (int ctas = 1; ctas <= 16; ctas = ctas == 8 ? 16 : ctas + 1) {
      const int stretch = (hw + ctas - 1) / ctas, steps = (stretch + rows - 1) / rows;
      if ((ctas > 1 && (hw + stretch - 1) / stretch != ctas) || units * ctas >= 1LL << 31) continue;
      const long long sums = planes == 1 ? 2 * (slots * (lanes * of_vector / merged) + ctas * of_slab) + 1 : slots * slot_stride + (lanes * t.v + 3 & ~3) + ctas * (2 * lanes * t.v + 2 * of_slab);
      const long long smem = 4 * ((long long)planes * stretch * lanes * t.v + sums);
      if (smem > kMostShared) continue;
      int at_once = (int)(kShared / (smem + 1024));  // CTAs on an SM
      if (at_once > 4) at_once = 4;
      double turns = (double)units * ctas / ((double)sms * at_once);
      turns = turns > 1 ? turns + 0.25 : 1;
      const long long there = (units * ctas + sms - 1) / sms;
      if (there < at_once) at_once = (int)there;
      const double values = (double)steps * t.v * planes;
      const double cost = turns * (6.5 + 0.015 * at_once * values + 0.01 * values + (at_once == 1 && turns > 1 ? 2.4 : 0.0) +
                                   (wide < 16 ? 3.7 : wide < 32 ? 0.15 : 0.0) + (ctas == 16 ? 2.0 : ctas == 1 ? -1.5 : 0.0));
      if (t.on_chip && cost >= best) continue;
      best = cost;
      t.on_chip = true;
      t.smem = (int)smem;
      t.s = Slabs{hw, c, groups, each, wide, slabs, (int)units, of_slab, ctas, stretch, lanes, rows, __builtin_ctz(lanes), __builtin_ctz(rows), steps,
                  of_vector, entries, merged, slots, lanes < 32 ? 32 / lanes : 1, slot_stride, false, 1.f / (float)hw, (float)(1.0 / ((double)each * hw)),
                  PoolDiv((unsigned)slabs), PoolDiv((unsigned)each)};
    }
    if (of_slab == groups) break;
  }
  return t;
}

template <class... P, class... A>
int launch_slabs(unsigned long long* opted, unsigned long long* large, const Plan& t, cudaStream_t st, void (*kernel)(P...), A... args) {
  if (int rc = mtb_opt_in_smem((const void*)kernel, kMostShared, opted)) return rc;
  if (t.s.ctas > 8) {
    int device = 0;
    MTB_CUDA(cudaGetDevice(&device));
    if (device >= 64 || !((__atomic_load_n(large, __ATOMIC_ACQUIRE) >> device) & 1ull)) {
      MTB_CUDA(cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      if (device < 64) __atomic_fetch_or(large, 1ull << device, __ATOMIC_RELEASE);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(t.s.units * t.s.ctas));
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
  static unsigned long long opted, large;
  return launch_slabs(&opted, &large, t, st, gn_forward_kernel<V, ACT>, t.s, args...);
}
template <int V, int ACT, class... A>
int backward_on_chip(const Plan& t, cudaStream_t st, A... args) {
  static unsigned long long opted, large;
  return launch_slabs(&opted, &large, t, st, gn_backward_kernel<V, ACT>, t.s, args...);
}

#define MTB_GN_PICK(f, t, act, ...)                                                                                                               \
  ((t).v == 4 ? (act == ACT_SILU ? f<4, ACT_SILU>(t, __VA_ARGS__) : act == ACT_RELU ? f<4, ACT_RELU>(t, __VA_ARGS__) : f<4, ACT_NONE>(t, __VA_ARGS__)) \
   : (t).v == 2 ? (act == ACT_SILU ? f<2, ACT_SILU>(t, __VA_ARGS__) : act == ACT_RELU ? f<2, ACT_RELU>(t, __VA_ARGS__) : f<2, ACT_NONE>(t, __VA_ARGS__)) \
                : (act == ACT_SILU ? f<1, ACT_SILU>(t, __VA_ARGS__) : act == ACT_RELU ? f<1, ACT_RELU>(t, __VA_ARGS__) : f<1, ACT_NONE>(t, __VA_ARGS__)))

// Stretches that the positions of an image are cut into where slabs go through memory: of 64 positions at least, or of 4096 values of a part whose threads take
// whatever there is.
int splits_of(int n, int hw, int parts, int values = 64) {
  long long want = (4LL * mtb_sm_count() + (long long)n * parts - 1) / ((long long)n * parts);
  const long long most = (long long)hw * values / 4096;
  if (want > most) want = most;
  if (want > hw) want = hw;
  return want < 1 ? 1 : want > 256 ? 256 : (int)want;
}

// The largest power of two up to 16 that all of them are a multiple of.
int alignment_of(const void* a, const void* b, const void* c) {
  const int m = (int)(((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15);
  return m ? m & -m : 16;
}

}  // namespace

// Values of an image: an int counts them and the positions that the last steps and stretches reach for beyond them.
constexpr long long kMostValues = (1LL << 31) - (1 << 16);

// Scratch of both directions: what slabs that go through memory leave of their stretches, and the backward's sums.
MTB_API long long mtb_group_norm_workspace_bytes(int n, int c, int hw, int groups) {
  if (n <= 0 || c <= 0 || hw <= 0 || groups <= 0) return 256;
  const long long forward = 12LL * n * groups * splits_of(n, hw, groups, c / groups), backward = 8LL * n * c * splits_of(n, hw, mtb_div_up(c, 32)) + 8LL * n * groups + 8LL * c * kStretches;
  return (forward > backward ? forward : backward) + 256;
}

MTB_API int mtb_group_norm_forward_f32(int n, int c, int hw, int groups, const float* x, const float* gamma, const float* beta, double eps, int activation,
                                       float* y, float* mean, float* rstd, void* workspace, long long workspace_bytes, void* stream) {
  const MtbScratchTurn turn;
  MTB_REQUIRE(n >= 0 && c > 0 && hw >= 0 && groups > 0 && c % groups == 0, "group_norm_forward: %d channels in %d groups", c, groups);
  MTB_REQUIRE(activation >= ACT_NONE && activation <= ACT_SILU, "group_norm_forward: unknown activation %d", activation);
  if (n == 0 || hw == 0) return MTB_OK;
  MTB_REQUIRE(x && y && mean && rstd, "group_norm_forward: null tensor");
  MTB_REQUIRE((long long)n * groups < 1LL << 31 && (long long)hw * c <= kMostValues, "group_norm_forward: too many values");
  cudaStream_t st = (cudaStream_t)stream;
  Plan t = plan_slabs(n, c, hw, groups, 1, alignment_of(x, y, nullptr));
  t.s.vectors = alignment_of(gamma, beta, nullptr) % (4 * t.v) == 0;
  if (t.on_chip) return MTB_GN_PICK(forward_on_chip, t, activation, st, x, gamma, beta, (float)eps, y, mean, rstd);
  MTB_REQUIRE(workspace && workspace_bytes >= mtb_group_norm_workspace_bytes(n, c, hw, groups), "group_norm_forward: workspace too small");
  const int splits = splits_of(n, hw, groups, c / groups);
  float* partial = (float*)workspace;
  const long long image = (long long)hw * c;
  MTB_LAUNCH(gn_stats_kernel, dim3(n * groups, splits), 256, 0, st, x, hw, c, groups, splits, PoolDiv(c / groups), partial);
  MTB_LAUNCH(gn_stats_final_kernel, mtb_div_up((long long)n * groups, 4), 128, 0, st, partial, n * groups, splits, (float)eps, mean, rstd);
  MTB_LAUNCH(gn_apply_kernel, dim3(n, mtb_stream_grid((image + kAhead - 1) / kAhead, 256)), 256, 0, st, x, image, PoolDiv(c), PoolDiv(c / groups), groups, gamma, beta, activation, mean, rstd, y);
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
  MTB_REQUIRE((long long)n * groups < 1LL << 31 && (long long)hw * c <= kMostValues, "group_norm_backward: too many values");
  MTB_REQUIRE(workspace_bytes >= mtb_group_norm_workspace_bytes(n, c, hw, groups), "group_norm_backward: workspace too small");
  float *sums = (float*)workspace, *after = sums + 2LL * n * c;  // what is left of the scratch
  const bool params = dgamma || dbeta;
  if (!params && !dx) return MTB_OK;
  Plan t = plan_slabs(n, c, hw, groups, 2, alignment_of(dy, x, dx));
  t.s.vectors = alignment_of(gamma, beta, nullptr) % (4 * t.v) == 0;
  if (t.on_chip) {
    if (int rc = MTB_GN_PICK(backward_on_chip, t, activation, st, dy, x, gamma, beta, mean, rstd, dx, params ? sums : nullptr)) return rc;
  } else {
    const int blocks = mtb_div_up(c, 32), splits = splits_of(n, hw, blocks);
    MTB_REQUIRE((long long)n * blocks < 1LL << 31, "group_norm_backward: %d images of %d channels", n, c);
    float* of_group = sums + 2LL * n * c * splits;
    after = of_group + 2LL * n * groups;
    const long long image = (long long)hw * c;
    const int each = c / groups;
    MTB_LAUNCH(mtb_div_up(hw, splits) > 8 * kChain ? gn_bwd_sums_kernel<true> : gn_bwd_sums_kernel<false>, dim3(n * blocks, splits), 256, 0, st, dy, x, hw, c, groups, splits, blocks, gamma, beta, activation, mean, rstd, sums);
    MTB_LAUNCH(splits > kChain || each > 32 * kChain ? gn_bwd_groups_kernel<true> : gn_bwd_groups_kernel<false>, mtb_div_up((long long)n * groups, 4), 128, 0, st, sums, n, c, groups, splits, gamma,
               (float)(1.0 / ((double)each * hw)), of_group);
    if (dx) MTB_LAUNCH(gn_bwd_dx_kernel, dim3(n, mtb_stream_grid((image + kAhead - 1) / kAhead, 256)), 256, 0, st, dy, x, image, PoolDiv(c), PoolDiv(c / groups), groups, gamma, beta,
                       activation, mean, rstd, of_group, dx);
  }
  if (params) {
    const int columns = mtb_div_up(2LL * c, 32), stretches = stretches_of(n);
    if (stretches > 1) {
      MTB_LAUNCH(gn_params_kernel, dim3(columns, stretches), 256, 0, st, sums, n, c, after, nullptr, nullptr);
      MTB_LAUNCH(gn_params_kernel, columns, 256, 0, st, after, stretches, c, nullptr, dgamma, dbeta);
    } else {
      MTB_LAUNCH(gn_params_kernel, columns, 256, 0, st, sums, n, c, nullptr, dgamma, dbeta);
    }
  }
  return MTB_OK;
}
