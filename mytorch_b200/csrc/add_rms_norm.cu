// What lies between two blocks of a residual network, and the norm by itself.  For every row of c values (the channels of a position):
//   b_hat = block r_b with r_b = 1 / sqrt(mean(block^2) + eps),  inner = b_hat post_weight  (without post_weight: inner = block),
//   new = scale residual + gate inner,  y = new rho weight with rho = 1 / sqrt(mean(new^2) + eps).
// Backward, for dnew and dy:  u = dy weight,  x_hat = new rho,  D = dnew + rho (u - x_hat mean(u x_hat)),
//   dresidual = scale D,  dgate = D inner,  dinner = gate D,  t = dinner post_weight,  dblock = r_b (t - b_hat mean(t b_hat)),
//   dweight = sum of dy x_hat,  dpost_weight = sum of dinner b_hat  over rows; dgate is summed over the rows that share a row of the gate.
//
// Bound by memory: 16 bytes a value forward, 24 backward, each once, if a row stays in registers between its sums and what is made of them.  So a group of W warps holds
// a row, PER vectors a thread and tensor, and goes on to its next one; W is 1 where a row fits a warp, which then waits for no other, and narrow rows lie side by side in
// a warp, LANES lanes each.
#include <cooperative_groups.h>

#include <algorithm>

#include "colreduce.cuh"

namespace cg = cooperative_groups;

namespace {

struct Operands {
  const float *x, *block, *weight, *post_weight, *gate;  // x: the residual (backward: the sum, new)
  long long rows;
  int c;
  long long rows_per_gate;
  float scale, eps;
};

constexpr int kMostCtas = 8;  // of a row

// Sums over the threads that share a row, W warps or LANES lanes of one, in all of them.  Two buffers taken in turn: a third sum writes where the first was read before
// the second.  JOINED: those of a cluster's CTAs, each of which gives its own to all of them.
template <int W, int LANES = 32, bool JOINED = false>
struct GroupSum {
  static constexpr int kThreads = W == 1 ? 256 : 32 * W;
  static constexpr int kGroups = W == 1 ? 256 / LANES : 1, kShare = W == 1 ? LANES : 32 * W;
  float (*part)[W];
  float (*given)[kMostCtas] = nullptr;
  int ctas = 1, rank = 0;
  int turn = 0;

  __device__ __forceinline__ float operator()(float x) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (W == 1) return x;
    if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) x += part[turn][w];
    if (JOINED) {
      cg::cluster_group cluster = cg::this_cluster();
      if ((int)threadIdx.x < ctas) cluster.map_shared_rank(&given[turn][0], threadIdx.x)[rank] = x;
      cluster.sync();
      x = 0;
      for (int r = 0; r < ctas; ++r) x += given[turn][r];
    }
    turn ^= 1;
    return x;
  }
};

template <int V>
__device__ __forceinline__ VecF<V> load(const float* p) {
  if constexpr (V == 2) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    return VecF<V>{{t.x, t.y}};
  } else {
    return vload<V>(p);
  }
}
template <int V>
__device__ __forceinline__ void store(float* p, const VecF<V>& r) {
  if constexpr (V == 2) *reinterpret_cast<float2*>(p) = make_float2(r.v[0], r.v[1]);
  else vstore<V>(p, r);
}
// A thread's own values come to shared memory while it works on those before them: nobody else reads them there, so nothing waits but the thread for its copies.
template <int V>
__device__ __forceinline__ void fetch(float* to, const float* from) {
  const unsigned at = (unsigned)__cvta_generic_to_shared(to);
  if constexpr (V == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(4 * V) : "memory");
}
__device__ __forceinline__ void fetched() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <int V>
__device__ __forceinline__ VecF<V> filled(float x) {
  VecF<V> r;
#pragma unroll
  for (int j = 0; j < V; ++j) r.v[j] = x;
  return r;
}

template <int V, int PER, int W, int LANES>
__global__ void __launch_bounds__(GroupSum<W, LANES>::kThreads) add_rms_norm_kernel(const __grid_constant__ Operands a, float* __restrict__ out, float* __restrict__ y, float* __restrict__ rstd,
                                                                             float* __restrict__ block_rstd) {
  __shared__ float part[2][W];
  GroupSum<W, LANES> sum{part};
  constexpr int kShare = GroupSum<W, LANES>::kShare, kGroups = GroupSum<W, LANES>::kGroups;
  mtb_launch_dependents();
  mtb_wait_prior();
  const int id = threadIdx.x % kShare, beside = W == 1 ? (threadIdx.x & 31) / LANES : 0;
  const long long groups = (long long)gridDim.x * kGroups;
  // all lanes of a warp go on as long as one of them has a row
  for (long long first = blockIdx.x * (long long)kGroups + (W == 1 ? threadIdx.x / 32 * (32 / LANES) : 0); first < a.rows; first += groups) {
    const long long row = LANES == 32 || first + beside < a.rows ? first + beside : first;
    const int c = LANES == 32 || first + beside < a.rows ? a.c : 0;
    const long long at = row * a.c;
    const float* gate = a.gate ? a.gate + (long long)((unsigned)row / (unsigned)a.rows_per_gate) * a.c : nullptr;
    VecF<V> x[PER], b[PER], g[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = (id + k * kShare) * V;
      x[k] = b[k] = filled<V>(0);
      g[k] = filled<V>(1);
      if (i < c) {
        if (a.block) b[k] = load<V>(a.block + at + i);
        x[k] = load<V>(a.x + at + i);
        if (gate) g[k] = load<V>(gate + i);
      }
    }
    if (a.block) {
      float rb = 1.f;
      if (a.post_weight) {
        float s = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) s = fmaf(b[k].v[j], b[k].v[j], s);
        rb = 1.f / sqrtf(sum(s) / a.c + a.eps);
        if (block_rstd && id == 0 && c) block_rstd[row] = rb;
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * kShare) * V;
        if (i < c) {
          const VecF<V> w = a.post_weight ? load<V>(a.post_weight + i) : filled<V>(1);
#pragma unroll
          for (int j = 0; j < V; ++j) x[k].v[j] = fmaf(a.scale, x[k].v[j], b[k].v[j] * rb * w.v[j] * g[k].v[j]);
          store<V>(out + at + i, x[k]);
        }
      }
    }
    float s = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(x[k].v[j], x[k].v[j], s);
    const float rho = 1.f / sqrtf(sum(s) / a.c + a.eps);
    if (rstd && id == 0 && c) rstd[row] = rho;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = (id + k * kShare) * V;
      if (i < c) {
        const VecF<V> w = a.weight ? load<V>(a.weight + i) : filled<V>(1);
        VecF<V> r;
#pragma unroll
        for (int j = 0; j < V; ++j) r.v[j] = x[k].v[j] * rho * w.v[j];
        store<V>(y + at + i, r);
      }
    }
  }
}

// What the backward makes beside the rows: sums of groups' rows, which a last kernel adds up.
struct Gradients {
  const float *dnew, *dy, *rstd, *block_rstd;
  float *dresidual, *dblock;
  float* partial;     // [CTA or cluster][3][c]: dweight, dpost_weight, dgate of a gate that all rows share; NULL: nobody asks
  float* gate_rows;   // a row for every row (a gate like the block), or for every stretch; NULL: neither
  int gate_each;      // 1: of every row
  // Rows come in stretches, none of which goes past a row of the gate: `parts` for each of its rows, `stretch` rows each but for the last.
  long long stretches, parts, stretch, rows_of_gate;
};

// AHEAD: the next row's values come to shared memory meanwhile.  That pays where many warps wait for one another at a row's sums (16384 x 2048 with post norm and gate 153 -> 136 us,
// 8192 x 4096 167 -> 142), not where rows of other groups are under way on the SM (32768 x 1024 135 -> 146), nor by copies of 4 bytes (32768 x 1023 158 -> 215).
// Where it is not 0: registers for so many on an SM; what else the compiler takes leaves a third of the warps (32768 x 750 by six values a thread and 4 warps 125 -> 111 us,
// 12672 x 2601 by eight and 12 warps 302 -> 207).  Kernels that lose more by spilling have none (16384 x 2047 by eight and 8 warps 171 -> 190).  With it spill: groups of 12 and 24 warps of
// pairs or single values 8 to 24 bytes a thread, six values of a warp 16, clusters by 8 and 12 warps of fours 20, by 12 of pairs 52 and of single values 136.  Without it: pairs by 2 and 5 warps
// 4, and, as 32 warps a CTA have 64 registers each at most, these 108 of fours, 140 of pairs, 152 of single values.
template <int V, int PER, int W, int LANES, bool JOINED>
constexpr int kBackwardCtas = JOINED ? (W == 8 && V != 4 ? 2 : 24 / W) : V * PER == 6 ? (W == 1 ? 3 : 24 / W) : W == 24 ? 1 : V != 4 && W == 12 ? 2 : V != 4 && V * PER == 4 && W == 1 && LANES == 32 ? 4 : 0;

template <int V, int PER, int W, int LANES, bool AHEAD, bool JOINED = false>
__global__ void __launch_bounds__(GroupSum<W, LANES, JOINED>::kThreads, kBackwardCtas<V, PER, W, LANES, JOINED>) add_rms_norm_backward_kernel(const __grid_constant__ Operands a, const __grid_constant__ Gradients d) {
  constexpr int kGroups = GroupSum<W, LANES, JOINED>::kGroups, kShare = GroupSum<W, LANES, JOINED>::kShare;
  extern __shared__ __align__(16) float shared[];  // AHEAD: [x, dy, dnew, block][PER][thread][V]; W 1: [3][c]
  __shared__ float part[2][W], given[JOINED ? 2 : 1][JOINED ? kMostCtas : 1];
  GroupSum<W, LANES, JOINED> sum{part};
  mtb_launch_dependents();
  mtb_wait_prior();
  if constexpr (JOINED) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();  // all of them have started: their shared memory is there
    sum.given = given;
    sum.ctas = (int)cluster.num_blocks();
    sum.rank = (int)cluster.block_rank();
  }
  const int share = JOINED ? sum.ctas * kShare : kShare;
  const long long unit = JOINED ? blockIdx.x / sum.ctas : blockIdx.x;  // the CTA, or the cluster
  const int id = (JOINED ? sum.rank * kShare : 0) + threadIdx.x % kShare, beside = W == 1 ? (threadIdx.x & 31) / LANES : 0;
  const long long groups = (long long)(JOINED ? gridDim.x / sum.ctas : gridDim.x) * kGroups;
  const float per_c = 1.f / a.c;
  VecF<V> dw[PER], dpw[PER], dg[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) dw[k] = dpw[k] = dg[k] = filled<V>(0);
  // where a row's values of this thread lie
  const auto slot = [&](int tensor, int j) { return shared + ((tensor * PER + j) * GroupSum<W, LANES, JOINED>::kThreads + (int)threadIdx.x) * V; };
  const auto fetch_row = [&](long long row) {
    const long long at = row * a.c;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = (id + j * share) * V;
      if (i < a.c) {
        fetch<V>(slot(0, j), a.x + at + i);
        if (d.dy) fetch<V>(slot(1, j), d.dy + at + i);
        if (d.dnew) fetch<V>(slot(2, j), d.dnew + at + i);
        if (a.block) fetch<V>(slot(3, j), a.block + at + i);
      }
    }
  };
  const auto first_of = [&](long long stretch) { const long long g = stretch / d.parts; return g * d.rows_of_gate + (stretch - g * d.parts) * d.stretch; };
  long long begin = unit * kGroups + (W == 1 ? threadIdx.x / 32 * (32 / LANES) : 0);
  if (AHEAD && begin < d.stretches) fetch_row(first_of(begin));
  for (; begin < d.stretches; begin += groups) {
    const long long stretch = LANES == 32 || begin + beside < d.stretches ? begin + beside : begin;
    const bool there = LANES == 32 || begin + beside < d.stretches;
    const long long first = first_of(stretch), limit = (stretch / d.parts + 1) * d.rows_of_gate, last = first + d.stretch < limit ? first + d.stretch : limit;
    for (long long next = first; next < (LANES == 32 ? last : first + d.stretch); ++next) {
      // all lanes of a warp go on as long as one of them has a row
      const bool on = LANES == 32 || (there && next < last);
      const long long row = on ? next : first, at = row * a.c;
      const int c = on ? a.c : 0;
      const float rho = d.rstd[row], rb = d.block_rstd ? d.block_rstd[row] : 1.f;
      const float* gate = a.gate ? a.gate + (long long)((unsigned)row / (unsigned)a.rows_per_gate) * a.c : nullptr;
      VecF<V> x[PER], dy[PER], D[PER], b[PER], g[PER];
      if (AHEAD) fetched();
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * share) * V;
        x[k] = dy[k] = D[k] = b[k] = filled<V>(0);
        g[k] = filled<V>(1);
        if (i < c) {
          const auto value = [&](int tensor, const float* from) { return AHEAD ? load<V>(slot(tensor, k)) : load<V>(from + at + i); };
          if (d.dnew) D[k] = value(2, d.dnew);
          if (a.block) b[k] = value(3, a.block);
          x[k] = value(0, a.x);
          if (d.dy) dy[k] = value(1, d.dy);
          if (gate) g[k] = load<V>(gate + i);
        }
      }
      const long long then = !AHEAD ? -1 : row + 1 < last ? row + 1 : begin + groups < d.stretches ? first_of(begin + groups) : -1;
      if (!d.dy && then >= 0) {
        __syncthreads();  // all values have been read, as below
        fetch_row(then);
      }
      if (d.dy) {
        float s = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int i = (id + k * share) * V;
          const VecF<V> w = a.weight && i < c ? load<V>(a.weight + i) : filled<V>(1);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            x[k].v[j] *= rho;
            dw[k].v[j] = fmaf(dy[k].v[j], x[k].v[j], dw[k].v[j]);
            dy[k].v[j] *= w.v[j];
            s = fmaf(dy[k].v[j], x[k].v[j], s);
          }
        }
        const float mean = sum(s) * per_c;
        if (then >= 0) fetch_row(then);  // all values have been read: the sum has a barrier
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) D[k].v[j] = fmaf(rho, dy[k].v[j] - x[k].v[j] * mean, D[k].v[j]);
      }
      if (d.dresidual) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int i = (id + k * share) * V;
          if (i < c) {
            VecF<V> r;
#pragma unroll
            for (int j = 0; j < V; ++j) r.v[j] = a.scale * D[k].v[j];
            store<V>(d.dresidual + at + i, r);
          }
        }
      }
      if (!a.block) continue;
      float s = 0;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * share) * V;
        const VecF<V> w = a.post_weight && i < c ? load<V>(a.post_weight + i) : filled<V>(1);
        VecF<V> each;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          b[k].v[j] *= rb;
          each.v[j] = D[k].v[j] * b[k].v[j] * w.v[j];
          dg[k].v[j] += each.v[j];
          D[k].v[j] *= g[k].v[j];
          dpw[k].v[j] = fmaf(D[k].v[j], b[k].v[j], dpw[k].v[j]);
          D[k].v[j] *= w.v[j];
          s = fmaf(D[k].v[j], b[k].v[j], s);
        }
        if (d.gate_each && d.gate_rows && i < c) store<V>(d.gate_rows + at + i, each);
      }
      if (!d.dblock) continue;
      const float mean = a.post_weight ? sum(s) * per_c : 0.f;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * share) * V;
        if (i < c) {
          VecF<V> r;
#pragma unroll
          for (int j = 0; j < V; ++j) r.v[j] = a.post_weight ? rb * (D[k].v[j] - b[k].v[j] * mean) : D[k].v[j];  // of an infinite block too
          store<V>(d.dblock + at + i, r);
        }
      }
    }
    if (d.gate_rows && !d.gate_each) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * share) * V;
        if (i < a.c && there) store<V>(d.gate_rows + stretch * a.c + i, dg[k]);
        dg[k] = filled<V>(0);
      }
    }
  }
  if (!d.partial) return;
  const int c = a.c;
  float* mine = d.partial + unit * 3 * c;
  if (W == 1) {  // the CTA's groups one after the other: the same order every time
    float* joined = shared;
    for (int w = 0; w < kGroups; ++w) {
      if ((int)threadIdx.x / LANES == w) {
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int i = (id + k * share) * V + j;
            if (i < c) {
              joined[i] = w ? joined[i] + dw[k].v[j] : dw[k].v[j];
              joined[c + i] = w ? joined[c + i] + dpw[k].v[j] : dpw[k].v[j];
              joined[2 * c + i] = w ? joined[2 * c + i] + dg[k].v[j] : dg[k].v[j];
            }
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 3 * c; i += 256) mine[i] = joined[i];
  } else {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = (id + k * share) * V;
      if (i < c) {
        store<V>(mine + i, dw[k]);
        store<V>(mine + c + i, dpw[k]);
        store<V>(mine + 2 * c + i, dg[k]);
      }
    }
  }
}

// Sums over rows of scratch.  The first CTAs add up three rows of c columns, 32 columns a CTA by 32 warps: dweight, dpost_weight, the gate that all rows share; the others
// the gate's rows from their stretches', a column a thread.  Latency bounds it: by eight warps a CTA the gradient of 32768 x 1024 takes 140 us instead of 135, of 65536 x 300 106 instead of 97.
struct Columns {
  const float *partial, *gate_rows;
  float *dweight, *dpost_weight, *dgate;
  int rows, c, blocks;  // CTAs of one of the three
  int parts, gates;     // gates 0: one that all rows share
};
constexpr int kColumnThreads = 1024, kColumnWarps = kColumnThreads / 32;
__global__ void __launch_bounds__(kColumnThreads) add_rms_norm_columns_kernel(const __grid_constant__ Columns t) {
  __shared__ float part[kColumnWarps][33];
  mtb_wait_prior();
  const int c = t.c;
  if ((int)blockIdx.x >= 3 * t.blocks) {
    const long long count = (long long)t.gates * c, step = (gridDim.x - 3LL * t.blocks) * kColumnThreads;
    for (long long n = (blockIdx.x - 3LL * t.blocks) * kColumnThreads + threadIdx.x; n < count; n += step) {
      const float* from = t.gate_rows + n / c * (t.parts - 1) * c + n;
      float s = 0;
#pragma unroll 8
      for (int r = 0; r < t.parts; ++r) s += from[(long long)r * c];
      t.dgate[n] = s;
    }
    return;
  }
  const int which = blockIdx.x / t.blocks, lane = threadIdx.x & 31, row = threadIdx.x >> 5, i = (blockIdx.x - which * t.blocks) * 32 + lane;
  float* out = which == 0 ? t.dweight : which == 1 ? t.dpost_weight : t.gates ? nullptr : t.dgate;
  if (!out) return;
  const long long stride = 3LL * c;
  const float* from = t.partial + (long long)which * c + i;
  float s[4] = {0, 0, 0, 0};
  if (i < c) {
    int r = row;
    for (; r + 3 * kColumnWarps < t.rows; r += 4 * kColumnWarps) {
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += from[(r + kColumnWarps * u) * stride];
    }
    for (; r < t.rows; r += kColumnWarps) s[0] += from[r * stride];
  }
  part[row][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  // a warp a column: 32 of them, one value a lane
  float x = part[lane][row];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  const int column = i - lane + row;
  if (lane == 0 && column < c) out[column] = x;
}

// ------------------------------------------------------------------ rows that no group holds: through memory, a CTA a row

constexpr int kLongThreads = 1024;

__device__ __forceinline__ float over_cta(float x, float* shared) {
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0;
  for (int w = 0; w < kLongThreads / 32; ++w) x += shared[w];
  return x;
}

__global__ void __launch_bounds__(kLongThreads) add_rms_norm_long_kernel(const __grid_constant__ Operands a, float* __restrict__ out, float* __restrict__ y, float* __restrict__ rstd,
                                                                         float* __restrict__ block_rstd) {
  __shared__ float shared[kLongThreads / 32];
  mtb_launch_dependents();
  mtb_wait_prior();
  const long long row = blockIdx.x;
  const float *x = a.x + row * a.c, *b = a.block ? a.block + row * a.c : nullptr, *gate = a.gate ? a.gate + (long long)((unsigned)row / (unsigned)a.rows_per_gate) * a.c : nullptr;
  float rb = 1.f;
  if (b && a.post_weight) {
    float s = 0;
    for (int i = threadIdx.x; i < a.c; i += kLongThreads) s += b[i] * b[i];
    rb = 1.f / sqrtf(over_cta(s, shared) / a.c + a.eps);
    if (block_rstd && threadIdx.x == 0) block_rstd[row] = rb;
  }
  float s = 0;
  for (int i = threadIdx.x; i < a.c; i += kLongThreads) {
    float v = x[i];
    if (b) {
      v = a.scale * v + b[i] * rb * (a.post_weight ? a.post_weight[i] : 1.f) * (gate ? gate[i] : 1.f);
      out[row * a.c + i] = v;
    }
    s += v * v;
  }
  const float rho = 1.f / sqrtf(over_cta(s, shared) / a.c + a.eps);
  if (rstd && threadIdx.x == 0) rstd[row] = rho;
  const float* from = b ? out + row * a.c : x;  // each thread what it wrote itself
  for (int i = threadIdx.x; i < a.c; i += kLongThreads) y[row * a.c + i] = from[i] * rho * (a.weight ? a.weight[i] : 1.f);
}

// The stretches of the kernel above; the sums over rows lie in scratch.
__global__ void __launch_bounds__(kLongThreads) add_rms_norm_backward_long_kernel(const __grid_constant__ Operands a, const __grid_constant__ Gradients d) {
  __shared__ float shared[kLongThreads / 32];
  mtb_launch_dependents();
  mtb_wait_prior();
  const int c = a.c;
  float* mine = d.partial ? d.partial + (long long)blockIdx.x * 3 * c : nullptr;
  if (mine)
    for (int i = threadIdx.x; i < c; i += kLongThreads) mine[i] = mine[c + i] = mine[2 * c + i] = 0;
  for (long long stretch = blockIdx.x; stretch < d.stretches; stretch += gridDim.x) {
    const long long of_gate = stretch / d.parts, first = of_gate * d.rows_of_gate + (stretch - of_gate * d.parts) * d.stretch;
    const long long limit = (of_gate + 1) * d.rows_of_gate, last = first + d.stretch < limit ? first + d.stretch : limit;
    for (long long row = first; row < last; ++row) {
      const long long at = row * c;
      const float* gate = a.gate ? a.gate + (long long)((unsigned)row / (unsigned)a.rows_per_gate) * c : nullptr;
      const float rho = d.rstd[row], rb = d.block_rstd ? d.block_rstd[row] : 1.f;
      float s = 0;
      for (int i = threadIdx.x; d.dy && i < c; i += kLongThreads) s += d.dy[at + i] * (a.weight ? a.weight[i] : 1.f) * a.x[at + i] * rho;
      const float c1 = over_cta(s, shared) / c;
      const auto total = [&](int i) {
        const float D = d.dnew ? d.dnew[at + i] : 0.f;
        return d.dy ? D + rho * (d.dy[at + i] * (a.weight ? a.weight[i] : 1.f) - a.x[at + i] * rho * c1) : D;
      };
      float c2 = 0;
      if (a.block && a.post_weight) {
        s = 0;
        for (int i = threadIdx.x; i < c; i += kLongThreads) s += total(i) * (gate ? gate[i] : 1.f) * a.post_weight[i] * a.block[at + i] * rb;
        c2 = over_cta(s, shared) / c;
      }
      for (int i = threadIdx.x; i < c; i += kLongThreads) {
        const float D = total(i);
        if (mine && d.dy) mine[i] += d.dy[at + i] * a.x[at + i] * rho;
        if (d.dresidual) d.dresidual[at + i] = a.scale * D;
        if (!a.block) continue;
        const float hat = a.block[at + i] * rb, w = a.post_weight ? a.post_weight[i] : 1.f, dinner = D * (gate ? gate[i] : 1.f), each = D * hat * w;
        if (mine) {
          mine[c + i] += dinner * hat;
          mine[2 * c + i] += each;
        }
        if (d.gate_rows) {
          float* to = d.gate_rows + (d.gate_each ? at : stretch * c) + i;
          *to = d.gate_each || row == first ? each : *to + each;
        }
        if (d.dblock) d.dblock[at + i] = a.post_weight ? rb * (dinner * w - hat * c2) : dinner;
      }
    }
  }
}

// ------------------------------------------------------------------ which kernel

struct Plan {
  int v, per, warps, lanes;  // warps 0: through memory
  int groups;         // of a CTA
  int ctas;           // the most that the grid has, or clusters
  bool ahead;
  int joined = 1;     // CTAs of a row: a cluster
};

// How many CTAs of a kernel an SM holds: the grid is no larger, so that none waits for another to end.
template <class K>
int resident(K kernel, int threads, int smem, int* known) {
  if (!*known && cudaOccupancyMaxActiveBlocksPerMultiprocessor(known, kernel, threads, smem) != cudaSuccess) *known = 0;
  return *known > 0 ? *known : 1;
}

// The same of clusters.
template <class... P>
int resident_clusters(void (*kernel)(P...), int ctas, int threads, int smem, int* known) {
  if (!*known) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(known, kernel, &cfg) != cudaSuccess) *known = 0;
  }
  return *known > 0 ? *known : 1;
}
template <class... P, class... A>
cudaError_t launch_clusters(void (*kernel)(P...), int clusters, int ctas, int threads, int smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * ctas));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// What holds a row: values a thread and tensor, warps.  Taken is the first of a table that is large enough.
struct Share {
  int values, warps;
};
template <int N>
Share share_of(const Share (&table)[N], int c) {
  for (const Share s : table)
    if (c <= 32 * s.warps * s.values) return s;
  return Share{0, 0};
}

// Vectors of four, of two where rows or operands begin at 8 bytes, else single values; the smallest group that holds a row, of few values a thread, so that other rows are under
// way meanwhile.  Of few rows eight warps a row.  Measured with post norm and gate, us: 33 million values in rows of 256 by 1 warp 93, by 2 with four values 86, but of 192 90 and 106;
// of 520 by 3 92, by 2 with 32 values 131; of 1200 by 5 85, by 8 110; of 2400 by 10 85, by 16 124; of 4096 by 8 98, by 16 95, by 32 164; in vectors of two, of 750 by 3 86, by 4 93; in
// single values, of 575 by 3 with six 96, by 4 with eight 118; of 2301 by 10 112, by 16 143; of 8185 by 16 with sixteen values 147, by 32 with eight 180.
constexpr Share kForwardSharesOfFour[] = {{8, 1}, {16, 1}, {8, 3}, {8, 4}, {8, 5}, {8, 6}, {8, 8}, {8, 10}, {8, 12}, {8, 16}, {16, 16}, {16, 32}};
constexpr Share kForwardShares[] = {{8, 1}, {6, 2}, {8, 2}, {6, 3}, {8, 3}, {8, 4}, {8, 5}, {8, 6}, {8, 8}, {8, 10}, {8, 12}, {8, 16}, {16, 16}, {16, 32}};
Plan forward_plan(long long rows, int c, int align) {
  const int v = align >= 4 && c % 4 == 0 ? 4 : align >= 2 && c % 2 == 0 ? 2 : 1;
  const auto plan = [&](int per, int warps, int lanes = 32) { return Plan{v, per, warps, lanes, warps == 1 ? 256 / lanes : 1, 0, false}; };
  if (rows <= 8LL * mtb_sm_count() && c > 256)
    for (const int per : {1, 2, 4})
      if (c <= 256 * per * v) return plan(per, 8);
  if (c <= 128) return plan(4 / v, 1, c <= 32 ? 8 : c <= 64 ? 16 : 32);
  const Share s = v == 4 ? share_of(kForwardSharesOfFour, c) : share_of(kForwardShares, c);
  return plan(s.values / v, s.warps);
}

// The smallest group that holds a row: what idles costs as what works does.  With post norm and gate, us: 65536 x 300 by 3 warps with four values a thread 98, by 2 with
// eight 104; 43840 x 752 by 3 with eight 141, by 4 155; 13696 x 2400 by 12 151, by 16 176; 5440 x 6000 by 24 162, by 32 216; in single values 65536 x 575 by 3 with six 179, by 4
// with eight 220; 27456 x 1201 by 5 158, by 8 with six 183, with eight 217; 8192 x 4601 by 24 with six 271, by 32 with eight 383.  Not in between: 22720 x 1450 in vectors of two by 12
// with six 194, by 8 with six 156.
constexpr Share kSharesOfFour[] = {{4, 2}, {4, 3}, {8, 2}, {8, 3}, {8, 4}, {8, 5}, {8, 8}, {8, 12}, {8, 16}, {8, 24}, {8, 32}};
constexpr Share kShares[] = {{6, 1}, {4, 2}, {4, 3}, {8, 2}, {6, 3}, {6, 4}, {8, 4}, {8, 5}, {6, 8}, {8, 8}, {6, 12}, {8, 10}, {8, 12}, {8, 16}, {6, 24}, {8, 24}, {8, 32}};
// A longer row by as many CTAs of eight values a thread as hold it, by 8 warps each as long as that is no more than eight: others of the SM's go on while a cluster waits for one of its
// own.  1984 x 16384 by eight CTAs of 8 warps 237, by six of 12 288, by four of 16 317, through memory 765.
constexpr int kJoinedWarps[] = {8, 12, 16};
Plan backward_plan(int c, int align) {
  const int v = align >= 4 && c % 4 == 0 ? 4 : align >= 2 && c % 2 == 0 ? 2 : 1, sms = mtb_sm_count();
  const auto plan = [&](int per, int warps, int per_sm, bool ahead = false, int lanes = 32) { return Plan{v, per, warps, lanes, warps == 1 ? 256 / lanes : 1, sms * per_sm, ahead}; };
  if (c <= 128) return plan(4 / v, 1, 5, false, c <= 32 ? 8 : c <= 64 ? 16 : 32);
  const Share s = v == 4 ? share_of(kSharesOfFour, c) : share_of(kShares, c);
  if (s.warps) return plan(s.values / v, s.warps, s.warps == 1 ? 3 : 32 / s.warps, v == 4 && s.warps >= 8);
  for (const int warps : kJoinedWarps) {
    const int ctas = (c + 256 * warps - 1) / (256 * warps);
    if (ctas <= kMostCtas) {
      Plan p = plan(8 / v, warps, 24 / warps, v == 4);
      p.ctas /= ctas;  // clusters
      p.joined = ctas;
      return p;
    }
  }
  return plan(0, 0, 1);
}

// How rows come in stretches (see Gradients): as many as there are groups, or more where the gate has more rows.
struct Stretches {
  long long stretches, parts, stretch, rows_of_gate;
  int ctas;
};
Stretches stretches_of(const Plan& p, int ctas, long long rows, long long rows_of_gate) {
  // as many stretches as there are groups, or up to four times as many: what leaves the group with the most rows the fewest
  const long long gates = rows / rows_of_gate, groups = (long long)ctas * p.groups;
  Stretches best{};
  long long least = 0;
  for (int turns = 1; turns <= 4; ++turns) {
    long long parts = turns * groups / gates;
    if (parts > (rows_of_gate + 1) / 2) parts = (rows_of_gate + 1) / 2;  // two rows at least
    if (parts < 1) parts = 1;
    const long long stretch = (rows_of_gate + parts - 1) / parts;
    parts = (rows_of_gate + stretch - 1) / stretch;
    const long long all = gates * parts, most = (all + groups - 1) / groups * stretch, needed = (all + p.groups - 1) / p.groups;
    if (turns == 1 || most < least) {
      best = {all, parts, stretch, rows_of_gate, (int)(needed < ctas ? needed : ctas)};
      least = most;
    }
  }
  return best;
}

bool sizes_fine(long long rows, int c, long long rows_per_gate) { return rows >= 0 && rows < 1LL << 31 && c > 0 && c <= 1 << 30 && rows_per_gate > 0 && rows % rows_per_gate == 0; }

// At how many floats all of them begin: 4, 2 or 1.
template <class... P>
int alignment(P... p) {
  const uintptr_t all = (reinterpret_cast<uintptr_t>(p) | ... | 0);
  return all % 16 == 0 ? 4 : all % 8 == 0 ? 2 : 1;
}

}  // namespace

MTB_API int mtb_add_rms_norm_forward_f32(long long rows, int c, const float* residual, const float* block, const float* weight, const float* post_weight, const float* gate,
                                         long long rows_per_gate, double scale, double eps, float* out, float* y, float* rstd, float* block_rstd, void* stream) {
  MTB_REQUIRE(sizes_fine(rows, c, gate ? rows_per_gate : 1) && eps >= 0, "add_rms_norm_forward: bad sizes");
  if (rows == 0) return MTB_OK;
  MTB_REQUIRE(residual && y && (block ? out != nullptr : !post_weight && !gate), "add_rms_norm_forward: bad arguments");
  cudaStream_t st = (cudaStream_t)stream;
  const Operands a{residual, block, weight, post_weight, gate, rows, c, gate ? rows_per_gate : 1, (float)scale, (float)eps};
  const Plan p = forward_plan(rows, c, alignment(residual, block, weight, post_weight, gate, out, y));
  const long long needed = (rows + p.groups - 1) / p.groups;
#define MTB_CASE(V, PER, W, LANES) \
  if (p.v == V && p.per == PER && p.warps == W && p.lanes == LANES) { \
    static int known; \
    const long long most = (long long)mtb_sm_count() * resident(add_rms_norm_kernel<V, PER, W, LANES>, GroupSum<W>::kThreads, 0, &known); \
    MTB_LAUNCH((add_rms_norm_kernel<V, PER, W, LANES>), (unsigned)(needed < most ? needed : most), GroupSum<W>::kThreads, 0, st, a, out, y, rstd, block_rstd); \
  } else
#define MTB_EIGHT(V, W) MTB_CASE(V, 8 / V, W, 32)
#define MTB_OF(V) \
  MTB_CASE(V, 4 / V, 1, 8) MTB_CASE(V, 4 / V, 1, 16) MTB_CASE(V, 4 / V, 1, 32) MTB_EIGHT(V, 1) MTB_EIGHT(V, 3) MTB_EIGHT(V, 4) MTB_EIGHT(V, 5) MTB_EIGHT(V, 6) MTB_EIGHT(V, 8) MTB_EIGHT(V, 10) \
  MTB_EIGHT(V, 12) MTB_EIGHT(V, 16) MTB_CASE(V, 16 / V, 16, 32) MTB_CASE(V, 16 / V, 32, 32) MTB_CASE(V, 1, 8, 32) MTB_CASE(V, 2, 8, 32) MTB_CASE(V, 4, 8, 32)
#define MTB_BESIDE(V) MTB_OF(V) MTB_EIGHT(V, 2) MTB_CASE(V, 6 / V, 2, 32) MTB_CASE(V, 6 / V, 3, 32)
  MTB_OF(4) MTB_CASE(4, 4, 1, 32) MTB_BESIDE(2) MTB_BESIDE(1) {
    MTB_LAUNCH(add_rms_norm_long_kernel, (unsigned)rows, kLongThreads, 0, st, a, out, y, rstd, block_rstd);
  }
#undef MTB_BESIDE
#undef MTB_OF
#undef MTB_EIGHT
#undef MTB_CASE
  MTB_LAUNCH_CHECK("add_rms_norm_kernel");
  return MTB_OK;
}

MTB_API long long mtb_add_rms_norm_workspace_bytes(long long rows, int c) {
  // whichever kernel it will be: a row of three sums for each CTA that has rows, and one for each stretch that does not fill a row of the gate (four a group at most)
  long long most = 4;  // what begins at 16 bytes
  for (const int align : {1, 2, 4}) {
    const Plan p = backward_plan(c, align);
    const long long ctas = std::min<long long>(p.ctas, (rows + p.groups - 1) / p.groups), stretches = std::min(rows, 4LL * p.ctas * p.groups);
    most = std::max(most, (3 * ctas + stretches) * c);
  }
  return 4 * most;
}

// The kernels that backward_plan names, each as a case of whatever MTB_CASE is.
#define MTB_EIGHT(V, W, AHEAD) MTB_CASE(V, 8 / V, W, 32, AHEAD)
#define MTB_SIX(V, W) MTB_CASE(V, 6 / V, W, 32, false)
#define MTB_OF(V, AHEAD) \
  MTB_CASE(V, 4 / V, 1, 8, false) MTB_CASE(V, 4 / V, 1, 16, false) MTB_CASE(V, 4 / V, 1, 32, false) MTB_CASE(V, 4 / V, 2, 32, false) MTB_CASE(V, 4 / V, 3, 32, false) MTB_EIGHT(V, 2, false) \
  MTB_EIGHT(V, 4, false) MTB_EIGHT(V, 5, false) MTB_EIGHT(V, 8, AHEAD) MTB_EIGHT(V, 12, AHEAD) MTB_EIGHT(V, 16, AHEAD) MTB_EIGHT(V, 24, AHEAD) MTB_EIGHT(V, 32, AHEAD)
#define MTB_BESIDE(V) MTB_OF(V, false) MTB_EIGHT(V, 10, false) MTB_SIX(V, 1) MTB_SIX(V, 3) MTB_SIX(V, 4) MTB_SIX(V, 8) MTB_SIX(V, 12) MTB_SIX(V, 24)
#define MTB_KERNELS MTB_OF(4, true) MTB_EIGHT(4, 3, false) MTB_BESIDE(2) MTB_BESIDE(1)
#define MTB_CLUSTERS MTB_JOINED(4, 8) MTB_JOINED(4, 12) MTB_JOINED(4, 16) MTB_JOINED(2, 8) MTB_JOINED(2, 12) MTB_JOINED(2, 16) MTB_JOINED(1, 8) MTB_JOINED(1, 12) MTB_JOINED(1, 16)

MTB_API int mtb_add_rms_norm_backward_f32(long long rows, int c, const float* dnew, const float* dy, const float* x, const float* rstd, const float* block,
                                          const float* block_rstd, const float* weight, const float* post_weight, const float* gate, long long rows_per_gate, double scale,
                                          float* dresidual, float* dblock, float* dweight, float* dpost_weight, float* dgate, void* workspace, long long workspace_bytes, void* stream) {
  const MtbScratchTurn turn;
  MTB_REQUIRE(sizes_fine(rows, c, gate ? rows_per_gate : 1), "add_rms_norm_backward: bad sizes");
  MTB_REQUIRE(x && rstd && (!post_weight || block_rstd) && (block || (!post_weight && !gate)), "add_rms_norm_backward: bad arguments");
  MTB_REQUIRE(workspace && mtb_aligned16(workspace) && workspace_bytes >= mtb_add_rms_norm_workspace_bytes(rows, c), "add_rms_norm_backward: workspace too small or off 16 bytes");
  cudaStream_t st = (cudaStream_t)stream;
  if (!post_weight) block_rstd = nullptr;
  if (!block) dblock = nullptr;
  if (!post_weight) dpost_weight = nullptr;
  if (!gate) dgate = nullptr;
  const Operands a{x, block, weight, post_weight, gate, rows, c, gate ? rows_per_gate : 1, block ? (float)scale : 1.f, 0.f};
  const Plan p = backward_plan(c, alignment(dnew, dy, x, block, weight, post_weight, gate, dresidual, dblock, dgate));
  const bool each = dgate && rows_per_gate == 1 && rows > 0, of_gate = dgate && !each && rows_per_gate < rows;
  Stretches s{0, 1, 1, 1, 0};
  float *partial = (float*)workspace, *gate_rows = nullptr;
  const bool summed = dweight || dpost_weight || (dgate && !each && !of_gate);
  if (rows > 0) {
    int ctas = p.ctas;
#define MTB_CASE(V, PER, W, LANES, AHEAD) \
  if (p.v == V && p.per == PER && p.warps == W && p.lanes == LANES && p.ahead == AHEAD && p.joined == 1) { \
    static unsigned long long opted; \
    static int known; \
    constexpr int kAhead = 16 * V * PER * GroupSum<W>::kThreads; \
    if (AHEAD) \
      if (int rc = mtb_opt_in_smem((const void*)add_rms_norm_backward_kernel<V, PER, W, LANES, AHEAD>, kAhead, &opted)) return rc; \
    const int most = mtb_sm_count() * resident(add_rms_norm_backward_kernel<V, PER, W, LANES, AHEAD>, GroupSum<W>::kThreads, AHEAD ? kAhead : W == 1 ? 12 * 256 : 0, &known); \
    ctas = most < ctas ? most : ctas; \
  } else
    MTB_KERNELS {}
#undef MTB_CASE
#define MTB_JOINED(V, W) \
  if (p.v == V && p.warps == W && p.joined > 1) { \
    static unsigned long long opted; \
    static int known[kMostCtas + 1]; \
    const auto kernel = add_rms_norm_backward_kernel<V, 8 / V, W, 32, V == 4, true>; \
    if (V == 4) \
      if (int rc = mtb_opt_in_smem((const void*)kernel, 16 * 8 * 32 * W, &opted)) return rc; \
    ctas = std::min(ctas, resident_clusters(kernel, p.joined, 32 * W, V == 4 ? 16 * 8 * 32 * W : 0, &known[p.joined])); \
  }
    MTB_CLUSTERS
#undef MTB_JOINED
    s = stretches_of(p, ctas, rows, of_gate ? rows_per_gate : rows);
    gate_rows = each || (of_gate && s.parts == 1) ? dgate : of_gate ? partial + (long long)s.ctas * 3 * c : nullptr;
    const Gradients d{dnew, dy, rstd, block_rstd, dresidual, dblock, summed ? partial : nullptr, gate_rows, each ? 1 : 0, s.stretches, s.parts, s.stretch, s.rows_of_gate};
#define MTB_CASE(V, PER, W, LANES, AHEAD) \
  if (p.v == V && p.per == PER && p.warps == W && p.lanes == LANES && p.ahead == AHEAD && p.joined == 1) { \
    MTB_LAUNCH((add_rms_norm_backward_kernel<V, PER, W, LANES, AHEAD>), (unsigned)s.ctas, GroupSum<W>::kThreads, AHEAD ? 16 * V * PER * GroupSum<W>::kThreads : W == 1 ? 12 * c : 0, st, a, d); \
  } else
#define MTB_JOINED(V, W) \
  if (p.v == V && p.warps == W && p.joined > 1) { \
    MTB_CUDA(launch_clusters(add_rms_norm_backward_kernel<V, 8 / V, W, 32, V == 4, true>, s.ctas, p.joined, 32 * W, V == 4 ? 16 * 8 * 32 * W : 0, st, a, d)); \
  } else
    MTB_KERNELS MTB_CLUSTERS {
      MTB_LAUNCH(add_rms_norm_backward_long_kernel, (unsigned)s.ctas, kLongThreads, 0, st, a, d);
    }
#undef MTB_JOINED
#undef MTB_CASE
    MTB_LAUNCH_CHECK("add_rms_norm_backward_kernel");
  }
  // a gate of every row is written; one of several rows is unless its stretches are shorter
  const bool shared_gate = dgate && !each && !of_gate, by_parts = of_gate && s.parts > 1;
  if (dweight || dpost_weight || shared_gate || by_parts) {
    const long long gates = by_parts ? rows / rows_per_gate : 0;
    const Columns t{partial, gate_rows, dweight, dpost_weight, shared_gate || by_parts ? dgate : nullptr, s.ctas, c, mtb_div_up(c, 32), (int)s.parts, (int)gates};
    MTB_LAUNCH(add_rms_norm_columns_kernel, 3 * t.blocks + (by_parts ? mtb_stream_grid(gates * c, kColumnThreads, 2) : 0), kColumnThreads, 0, st, t);
    MTB_LAUNCH_CHECK("add_rms_norm_columns_kernel");
  }
  return MTB_OK;
}
