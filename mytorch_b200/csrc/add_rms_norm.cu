// What lies between two blocks of a residual network, and the norm by itself.  For every row of c values (the channels of a position):
//   b_hat = block r_b with r_b = 1 / sqrt(mean(block^2) + eps),  inner = b_hat post_weight  (without post_weight: inner = block),
//   new = scale residual + gate inner,  y = new rho weight with rho = 1 / sqrt(mean(new^2) + eps).
// Backward, for dnew and dy:  u = dy weight,  x_hat = new rho,  D = dnew + rho (u - x_hat mean(u x_hat)),
//   dresidual = scale D,  dgate = D inner,  dinner = gate D,  t = dinner post_weight,  dblock = r_b (t - b_hat mean(t b_hat)),
//   dweight = sum of dy x_hat,  dpost_weight = sum of dinner b_hat  over rows; dgate is summed over the rows that share a row of the gate.
//
// Bound by memory: 16 bytes a value forward, 24 backward, each once, if a row stays in registers between its sums and what is made of them.  So a group of W warps holds
// a row, PER vectors a thread and tensor, and goes on to its next one; W is 1 where a row fits a warp, which then waits for no other.
#include <utility>

#include "colreduce.cuh"

namespace {

struct Operands {
  const float *x, *block, *weight, *post_weight, *gate;  // x: the residual (backward: the sum, new)
  long long rows;
  int c;
  long long rows_per_gate;
  float scale, eps;
};

// Sums over the W warps that share a row, in all their threads.  Two buffers taken in turn: a third sum writes where the first was read before the second.
template <int W>
struct GroupSum {
  static constexpr int kThreads = W == 1 ? 256 : 32 * W, kGroups = W == 1 ? 8 : 1;
  float (*part)[W];
  int turn = 0;

  __device__ __forceinline__ float operator()(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (W == 1) return x;
    if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) x += part[turn][w];
    turn ^= 1;
    return x;
  }
};

template <int V>
__device__ __forceinline__ VecF<V> filled(float x) {
  VecF<V> r;
#pragma unroll
  for (int j = 0; j < V; ++j) r.v[j] = x;
  return r;
}

template <int V, int PER, int W>
__global__ void __launch_bounds__(GroupSum<W>::kThreads) add_rms_norm_kernel(const __grid_constant__ Operands a, float* __restrict__ out, float* __restrict__ y, float* __restrict__ rstd,
                                                                             float* __restrict__ block_rstd) {
  __shared__ float part[2][W];
  GroupSum<W> sum{part};
  mtb_launch_dependents();
  mtb_wait_prior();
  const int id = W == 1 ? threadIdx.x & 31 : threadIdx.x;
  const long long groups = (long long)gridDim.x * GroupSum<W>::kGroups;
  for (long long row = W == 1 ? blockIdx.x * 8LL + (threadIdx.x >> 5) : blockIdx.x; row < a.rows; row += groups) {
    const long long at = row * a.c;
    VecF<V> x[PER], b[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = (id + k * 32 * W) * V;
      x[k] = b[k] = filled<V>(0);
      if (i < a.c) {
        x[k] = vload<V>(a.x + at + i);
        if (a.block) b[k] = vload<V>(a.block + at + i);
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
        if (block_rstd && id == 0) block_rstd[row] = rb;
      }
      const float* gate = a.gate ? a.gate + (long long)((unsigned)row / (unsigned)a.rows_per_gate) * a.c : nullptr;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * 32 * W) * V;
        if (i < a.c) {
          const VecF<V> w = a.post_weight ? vload<V>(a.post_weight + i) : filled<V>(1), g = gate ? vload<V>(gate + i) : filled<V>(1);
#pragma unroll
          for (int j = 0; j < V; ++j) x[k].v[j] = fmaf(a.scale, x[k].v[j], b[k].v[j] * rb * w.v[j] * g.v[j]);
          vstore<V>(out + at + i, x[k]);
        }
      }
    }
    float s = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(x[k].v[j], x[k].v[j], s);
    const float rho = 1.f / sqrtf(sum(s) / a.c + a.eps);
    if (rstd && id == 0) rstd[row] = rho;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = (id + k * 32 * W) * V;
      if (i < a.c) {
        const VecF<V> w = a.weight ? vload<V>(a.weight + i) : filled<V>(1);
        VecF<V> r;
#pragma unroll
        for (int j = 0; j < V; ++j) r.v[j] = x[k].v[j] * rho * w.v[j];
        vstore<V>(y + at + i, r);
      }
    }
  }
}

// What the backward makes beside the rows: sums of groups' rows, which a last kernel adds up.
struct Gradients {
  const float *dnew, *dy, *rstd, *block_rstd;
  float *dresidual, *dblock;
  float* partial;     // [CTA][3][c]: dweight, dpost_weight, dgate of a gate that all rows share; NULL: nobody asks
  float* gate_rows;   // a row for every row (a gate like the block), or for every stretch; NULL: neither
  int gate_each;      // 1: of every row
  // Rows come in stretches, none of which goes past a row of the gate: `parts` for each of its rows, `stretch` rows each but for the last.
  long long stretches, parts, stretch, rows_of_gate;
};

template <int V, int PER, int W>
__global__ void __launch_bounds__(GroupSum<W>::kThreads) add_rms_norm_backward_kernel(const __grid_constant__ Operands a, const __grid_constant__ Gradients d) {
  constexpr int kGroups = GroupSum<W>::kGroups;
  extern __shared__ float joined[];  // W 1: [3][c]
  __shared__ float part[2][W];
  GroupSum<W> sum{part};
  mtb_launch_dependents();
  mtb_wait_prior();
  const int id = W == 1 ? threadIdx.x & 31 : threadIdx.x, c = a.c;
  const long long groups = (long long)gridDim.x * kGroups;
  const float per_c = 1.f / c;
  VecF<V> dw[PER], dpw[PER], dg[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) dw[k] = dpw[k] = dg[k] = filled<V>(0);
  for (long long stretch = W == 1 ? blockIdx.x * 8LL + (threadIdx.x >> 5) : blockIdx.x; stretch < d.stretches; stretch += groups) {
    const long long of_gate = stretch / d.parts, first = of_gate * d.rows_of_gate + (stretch - of_gate * d.parts) * d.stretch;
    const long long limit = (of_gate + 1) * d.rows_of_gate, last = first + d.stretch < limit ? first + d.stretch : limit;
    for (long long row = first; row < last; ++row) {
      const long long at = row * c;
      const float rho = d.rstd[row], rb = d.block_rstd ? d.block_rstd[row] : 1.f;
      const float* gate = a.gate ? a.gate + (long long)((unsigned)row / (unsigned)a.rows_per_gate) * c : nullptr;
      VecF<V> x[PER], dy[PER], D[PER], b[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * 32 * W) * V;
        x[k] = dy[k] = D[k] = b[k] = filled<V>(0);
        if (i < c) {
          x[k] = vload<V>(a.x + at + i);
          if (d.dy) dy[k] = vload<V>(d.dy + at + i);
          if (d.dnew) D[k] = vload<V>(d.dnew + at + i);
          if (a.block) b[k] = vload<V>(a.block + at + i);
        }
      }
      if (d.dy) {
        float s = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int i = (id + k * 32 * W) * V;
          const VecF<V> w = a.weight && i < c ? vload<V>(a.weight + i) : filled<V>(1);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            x[k].v[j] *= rho;
            dw[k].v[j] = fmaf(dy[k].v[j], x[k].v[j], dw[k].v[j]);
            dy[k].v[j] *= w.v[j];
            s = fmaf(dy[k].v[j], x[k].v[j], s);
          }
        }
        const float mean = sum(s) * per_c;
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) D[k].v[j] = fmaf(rho, dy[k].v[j] - x[k].v[j] * mean, D[k].v[j]);
      }
      if (d.dresidual) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int i = (id + k * 32 * W) * V;
          if (i < c) {
            VecF<V> r;
#pragma unroll
            for (int j = 0; j < V; ++j) r.v[j] = a.scale * D[k].v[j];
            vstore<V>(d.dresidual + at + i, r);
          }
        }
      }
      if (!a.block) continue;
      float s = 0;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * 32 * W) * V;
        const VecF<V> w = a.post_weight && i < c ? vload<V>(a.post_weight + i) : filled<V>(1), g = gate && i < c ? vload<V>(gate + i) : filled<V>(1);
        VecF<V> each;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          b[k].v[j] *= rb;
          each.v[j] = D[k].v[j] * b[k].v[j] * w.v[j];
          dg[k].v[j] += each.v[j];
          D[k].v[j] *= g.v[j];
          dpw[k].v[j] = fmaf(D[k].v[j], b[k].v[j], dpw[k].v[j]);
          D[k].v[j] *= w.v[j];
          s = fmaf(D[k].v[j], b[k].v[j], s);
        }
        if (d.gate_each && d.gate_rows && i < c) vstore<V>(d.gate_rows + at + i, each);
      }
      if (!d.dblock) continue;
      const float mean = a.post_weight ? sum(s) * per_c : 0.f;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * 32 * W) * V;
        if (i < c) {
          VecF<V> r;
#pragma unroll
          for (int j = 0; j < V; ++j) r.v[j] = rb * (D[k].v[j] - b[k].v[j] * mean);
          vstore<V>(d.dblock + at + i, r);
        }
      }
    }
    if (d.gate_rows && !d.gate_each) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = (id + k * 32 * W) * V;
        if (i < c) vstore<V>(d.gate_rows + stretch * c + i, dg[k]);
        dg[k] = filled<V>(0);
      }
    }
  }
  if (!d.partial) return;
  float* mine = d.partial + (long long)blockIdx.x * 3 * c;
  if (W == 1) {  // the CTA's eight warps one after the other: the same order every time
    for (int w = 0; w < kGroups; ++w) {
      if ((int)(threadIdx.x >> 5) == w) {
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int i = (id + k * 32) * V + j;
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
      const int i = (id + k * 32 * W) * V;
      if (i < c) {
        vstore<V>(mine + i, dw[k]);
        vstore<V>(mine + c + i, dpw[k]);
        vstore<V>(mine + 2 * c + i, dg[k]);
      }
    }
  }
}

// Sums over rows of scratch, 32 columns a CTA by eight lanes each: task 0 dweight, 1 dpost_weight, 2 the gate that all rows share, or from 2 on a row of the gate each.
struct Columns {
  const float *partial, *gate_rows;
  float *dweight, *dpost_weight, *dgate;
  int c, ctas, shared_gate, first;  // first: the first task of the launch
  long long parts;
};
__global__ void __launch_bounds__(256) add_rms_norm_columns_kernel(const __grid_constant__ Columns t) {
  __shared__ float part[8][33];
  mtb_wait_prior();
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, i = blockIdx.x * 32 + lane, task = blockIdx.y + t.first;
  const bool of_gate = task >= 2 && !t.shared_gate;
  float* out = task == 0 ? t.dweight : task == 1 ? t.dpost_weight : t.dgate ? t.dgate + (of_gate ? (long long)(task - 2) * t.c : 0) : nullptr;
  if (!out) return;
  const float* from = of_gate ? t.gate_rows + (task - 2) * t.parts * t.c : t.partial + (long long)task * t.c;
  const long long rows = of_gate ? t.parts : t.ctas, stride = of_gate ? t.c : 3LL * t.c;
  float s[4] = {0, 0, 0, 0};
  if (i < t.c) {
    long long r = row;
    for (; r + 24 < rows; r += 32) {
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += from[(r + 8 * u) * stride + i];
    }
    for (; r < rows; r += 8) s[0] += from[r * stride + i];
  }
  part[row][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (row == 0 && i < t.c) {
    float x = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) x += part[k][lane];
    out[i] = x;
  }
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
        const float u = d.dy ? d.dy[at + i] * (a.weight ? a.weight[i] : 1.f) : 0.f;
        return (d.dnew ? d.dnew[at + i] : 0.f) + rho * (u - a.x[at + i] * rho * c1);
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
        if (d.dblock) d.dblock[at + i] = rb * (dinner * w - hat * c2);
      }
    }
  }
}

// ------------------------------------------------------------------ which kernel

struct Plan {
  int v, per, warps;  // warps 0: through memory
  int groups;         // of a CTA
  int ctas;           // the most that the grid has
};

Plan forward_plan(long long rows, int c, bool vectors) {
  const int v = vectors && c % 4 == 0 ? 4 : 1, n = (c + v - 1) / v, sms = mtb_sm_count();
  const bool many = rows > 8LL * sms;
  for (const auto [per, warps] : {std::pair{1, 1}, {2, 1}, {4, 1}, {8, 1}, {1, 8}, {2, 8}, {4, 8}, {8, 8}, {v == 4 ? 4 : 8, 32}})
    if (n <= 32 * warps * per && (warps > 1 || many || per <= 2)) return Plan{v, per, warps, warps == 1 ? 8 : 1, sms * (warps == 32 ? 2 : 8)};
  return Plan{v, 0, 0, 1, 0};
}

Plan backward_plan(long long rows, int c, bool vectors) {
  const int v = vectors && c % 4 == 0 ? 4 : 1, n = (c + v - 1) / v, sms = mtb_sm_count();
  if (v == 4) {
    for (const auto [per, warps] : {std::pair{1, 1}, {2, 1}, {1, 4}, {2, 4}, {2, 8}, {2, 16}, {4, 16}})
      if (n <= 32 * warps * per) return Plan{v, per, warps, warps == 1 ? 8 : 1, sms * (warps == 16 ? 1 : warps == 4 ? 6 : 3)};
  } else {
    for (const auto [per, warps] : {std::pair{1, 1}, {2, 1}, {4, 1}, {8, 1}, {4, 4}, {8, 4}, {8, 8}, {8, 16}})
      if (n <= 32 * warps * per) return Plan{v, per, warps, warps == 1 ? 8 : 1, sms * (warps == 16 ? 1 : warps == 4 ? 6 : 3)};
  }
  return Plan{v, 0, 0, 1, sms};
}

// How rows come in stretches (see Gradients): as many as there are groups, or more where the gate has more rows.
struct Stretches {
  long long stretches, parts, stretch, rows_of_gate;
  int ctas;
};
Stretches stretches_of(const Plan& p, long long rows, long long rows_of_gate) {
  const long long gates = rows / rows_of_gate, groups = (long long)p.ctas * p.groups;
  long long parts = groups / gates;
  if (parts > (rows_of_gate + 1) / 2) parts = (rows_of_gate + 1) / 2;  // two rows at least
  if (parts < 1) parts = 1;
  const long long stretch = (rows_of_gate + parts - 1) / parts;
  parts = (rows_of_gate + stretch - 1) / stretch;
  const long long all = gates * parts, needed = (all + p.groups - 1) / p.groups;
  return {all, parts, stretch, rows_of_gate, (int)(needed < p.ctas ? needed : p.ctas)};
}

bool sizes_fine(long long rows, int c, long long rows_per_gate) { return rows >= 0 && rows < 1LL << 31 && c > 0 && c <= 1 << 30 && rows_per_gate > 0 && rows % rows_per_gate == 0; }

template <class... P>
bool aligned(P... p) { return ((reinterpret_cast<uintptr_t>(p) | ... | 0) & 15u) == 0; }

}  // namespace

MTB_API int mtb_add_rms_norm_forward_f32(long long rows, int c, const float* residual, const float* block, const float* weight, const float* post_weight, const float* gate,
                                         long long rows_per_gate, double scale, double eps, float* out, float* y, float* rstd, float* block_rstd, void* stream) {
  MTB_REQUIRE(sizes_fine(rows, c, gate ? rows_per_gate : 1) && eps >= 0, "add_rms_norm_forward: bad sizes");
  if (rows == 0) return MTB_OK;
  MTB_REQUIRE(residual && y && (block ? out != nullptr : !post_weight && !gate), "add_rms_norm_forward: bad arguments");
  cudaStream_t st = (cudaStream_t)stream;
  const Operands a{residual, block, weight, post_weight, gate, rows, c, gate ? rows_per_gate : 1, (float)scale, (float)eps};
  const Plan p = forward_plan(rows, c, aligned(residual, block, weight, post_weight, gate, out, y));
  const long long needed = (rows + p.groups - 1) / p.groups;
#define MTB_CASE(V, PER, W) \
  if (p.v == V && p.per == PER && p.warps == W) { \
    MTB_LAUNCH((add_rms_norm_kernel<V, PER, W>), (unsigned)(needed < p.ctas ? needed : p.ctas), GroupSum<W>::kThreads, 0, st, a, out, y, rstd, block_rstd); \
  } else
#define MTB_BOTH(PER, W) MTB_CASE(4, PER, W) MTB_CASE(1, PER, W)
  MTB_BOTH(1, 1) MTB_BOTH(2, 1) MTB_BOTH(4, 1) MTB_BOTH(8, 1) MTB_BOTH(1, 8) MTB_BOTH(2, 8) MTB_BOTH(4, 8) MTB_BOTH(8, 8) MTB_CASE(4, 4, 32) MTB_CASE(1, 8, 32) {
    MTB_LAUNCH(add_rms_norm_long_kernel, (unsigned)rows, kLongThreads, 0, st, a, out, y, rstd, block_rstd);
  }
#undef MTB_BOTH
#undef MTB_CASE
  MTB_LAUNCH_CHECK("add_rms_norm_kernel");
  return MTB_OK;
}

MTB_API long long mtb_add_rms_norm_workspace_bytes(long long rows, int c) {
  // whichever kernel it will be: a row of three sums for each CTA, and one for each stretch that does not fill a row of the gate
  long long most = 0;
  for (const bool vectors : {false, true}) {
    const Plan p = backward_plan(rows, c, vectors);
    const long long floats = (long long)p.ctas * (3 + p.groups) * c;
    if (floats > most) most = floats;
  }
  return 4 * most;
}

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
  const Plan p = backward_plan(rows, c, aligned(dnew, dy, x, block, weight, post_weight, gate, dresidual, dblock, dgate));
  const bool each = dgate && rows_per_gate == 1 && rows > 0, of_gate = dgate && !each && rows_per_gate < rows;
  Stretches s{0, 1, 1, 1, 0};
  float *partial = (float*)workspace, *gate_rows = nullptr;
  const bool summed = dweight || dpost_weight || (dgate && !each && !of_gate);
  if (rows > 0) {
    s = stretches_of(p, rows, of_gate ? rows_per_gate : rows);
    gate_rows = each || (of_gate && s.parts == 1) ? dgate : of_gate ? partial + (long long)p.ctas * 3 * c : nullptr;
    const Gradients d{dnew, dy, rstd, block_rstd, dresidual, dblock, summed ? partial : nullptr, gate_rows, each ? 1 : 0, s.stretches, s.parts, s.stretch, s.rows_of_gate};
#define MTB_CASE(V, PER, W) \
  if (p.v == V && p.per == PER && p.warps == W) { \
    MTB_LAUNCH((add_rms_norm_backward_kernel<V, PER, W>), (unsigned)s.ctas, GroupSum<W>::kThreads, W == 1 ? 12 * c : 0, st, a, d); \
  } else
    MTB_CASE(4, 1, 1) MTB_CASE(4, 2, 1) MTB_CASE(4, 1, 4) MTB_CASE(4, 2, 4) MTB_CASE(4, 2, 8) MTB_CASE(4, 2, 16) MTB_CASE(4, 4, 16)
    MTB_CASE(1, 1, 1) MTB_CASE(1, 2, 1) MTB_CASE(1, 4, 1) MTB_CASE(1, 8, 1) MTB_CASE(1, 4, 4) MTB_CASE(1, 8, 4) MTB_CASE(1, 8, 8) MTB_CASE(1, 8, 16) {
      MTB_LAUNCH(add_rms_norm_backward_long_kernel, (unsigned)s.ctas, kLongThreads, 0, st, a, d);
    }
#undef MTB_CASE
    MTB_LAUNCH_CHECK("add_rms_norm_backward_kernel");
  }
  // a gate of every row is written; one of several rows is unless its stretches are shorter
  const bool parts = of_gate && s.parts > 1, shared_gate = dgate && !each && !of_gate;
  const long long tasks = 2 + (shared_gate ? 1 : parts ? rows / rows_per_gate : 0);
  if (!dweight && !dpost_weight && tasks == 2) return MTB_OK;
  for (long long first = 0; first < tasks; first += 65535) {
    const Columns t{partial, gate_rows, dweight, dpost_weight, dgate, c, s.ctas, shared_gate ? 1 : 0, (int)first, s.parts};
    MTB_LAUNCH(add_rms_norm_columns_kernel, dim3(mtb_div_up(c, 32), (unsigned)(tasks - first < 65535 ? tasks - first : 65535)), 256, 0, st, t);
    MTB_LAUNCH_CHECK("add_rms_norm_columns_kernel");
  }
  return MTB_OK;
}
