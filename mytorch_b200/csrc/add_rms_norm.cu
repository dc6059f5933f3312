// What lies between two blocks of a residual network, and the norm by itself.  For every row of c values (the channels of a position):
//   b_hat = block r_b with r_b = 1 / sqrt(mean(block^2) + eps),  inner = b_hat post_weight  (without post_weight: inner = block),
//   new = scale residual + gate inner,  y = new rho weight with rho = 1 / sqrt(mean(new^2) + eps).
// Backward, for dnew and dy:  u = dy weight,  x_hat = new rho,  D = dnew + rho (u - x_hat mean(u x_hat)),
//   dresidual = scale D,  dgate = D inner,  dinner = gate D,  t = dinner post_weight,  dblock = r_b (t - b_hat mean(t b_hat)),
//   dweight = sum of dy x_hat,  dpost_weight = sum of dinner b_hat  over rows; dgate is summed over the rows that share a row of the gate.
#include "common.cuh"

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

__device__ __forceinline__ float over_cta(float x, float* shared) {
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0;
  for (int w = 0; w < kWarps; ++w) x += shared[w];
  return x;
}

struct Operands {
  const float *x, *block, *weight, *post_weight, *gate;  // x: the residual (backward: the sum, new)
  long long rows;
  int c;
  long long rows_per_gate;
  float scale, eps;
};

__global__ void __launch_bounds__(kThreads) add_rms_norm_kernel(Operands a, float* __restrict__ out, float* __restrict__ y, float* __restrict__ rstd, float* __restrict__ block_rstd) {
  __shared__ float shared[kWarps];
  mtb_launch_dependents();
  mtb_wait_prior();
  const long long row = blockIdx.x;
  const float *x = a.x + row * a.c, *b = a.block ? a.block + row * a.c : nullptr, *gate = a.gate ? a.gate + row / a.rows_per_gate * a.c : nullptr;
  float rb = 1.f;
  if (b && a.post_weight) {
    float s = 0;
    for (int i = threadIdx.x; i < a.c; i += kThreads) s += b[i] * b[i];
    rb = 1.f / sqrtf(over_cta(s, shared) / a.c + a.eps);
    if (block_rstd && threadIdx.x == 0) block_rstd[row] = rb;
  }
  float s = 0;
  for (int i = threadIdx.x; i < a.c; i += kThreads) {
    float v = x[i];
    if (b) {
      v = a.scale * v + b[i] * rb * (a.post_weight ? a.post_weight[i] : 1.f) * (gate ? gate[i] : 1.f);
      out[row * a.c + i] = v;
    }
    s += v * v;
  }
  const float rho = 1.f / sqrtf(over_cta(s, shared) / a.c + a.eps);
  if (rstd && threadIdx.x == 0) rstd[row] = rho;
  const float* from = b ? out + row * a.c : x;
  for (int i = threadIdx.x; i < a.c; i += kThreads) y[row * a.c + i] = from[i] * rho * (a.weight ? a.weight[i] : 1.f);
}

// A CTA takes every gridDim-th row; what it adds up over rows lies in its own row of `partial` [grid][3][c]: dweight, dpost_weight, dgate.
__global__ void __launch_bounds__(kThreads) add_rms_norm_backward_kernel(Operands a, const float* __restrict__ dnew, const float* __restrict__ dy, const float* __restrict__ rstd,
                                                                         const float* __restrict__ block_rstd, float* __restrict__ dresidual, float* __restrict__ dblock,
                                                                         float* __restrict__ dgate_rows, float* __restrict__ partial) {
  __shared__ float shared[kWarps];
  mtb_launch_dependents();
  mtb_wait_prior();
  const int c = a.c;
  float* mine = partial ? partial + (long long)blockIdx.x * 3 * c : nullptr;
  if (mine)
    for (int i = threadIdx.x; i < 3 * c; i += kThreads) mine[i] = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const long long at = row * c;
    const float *gate = a.gate ? a.gate + row / a.rows_per_gate * c : nullptr;
    const float rho = rstd[row], rb = block_rstd ? block_rstd[row] : 1.f;
    float s = 0;
    for (int i = threadIdx.x; i < c; i += kThreads)
      if (dy) s += dy[at + i] * (a.weight ? a.weight[i] : 1.f) * a.x[at + i] * rho;
    const float c1 = over_cta(s, shared) / c;
    const auto total = [&](int i) {
      const float u = dy ? dy[at + i] * (a.weight ? a.weight[i] : 1.f) : 0.f;
      return (dnew ? dnew[at + i] : 0.f) + rho * (u - a.x[at + i] * rho * c1);
    };
    float c2 = 0;
    if (a.block && a.post_weight) {
      s = 0;
      for (int i = threadIdx.x; i < c; i += kThreads) s += total(i) * (gate ? gate[i] : 1.f) * a.post_weight[i] * a.block[at + i] * rb;
      c2 = over_cta(s, shared) / c;
    }
    for (int i = threadIdx.x; i < c; i += kThreads) {
      const float D = total(i);
      if (mine && dy) mine[i] += dy[at + i] * a.x[at + i] * rho;
      if (dresidual) dresidual[at + i] = a.block ? a.scale * D : D;
      if (!a.block) continue;
      const float hat = a.block[at + i] * rb, w = a.post_weight ? a.post_weight[i] : 1.f, dinner = D * (gate ? gate[i] : 1.f);
      if (mine) {
        mine[c + i] += dinner * hat;
        mine[2 * c + i] += D * hat * w;
      }
      if (dgate_rows) dgate_rows[at + i] = D * hat * w;
      if (dblock) dblock[at + i] = a.post_weight ? rb * (dinner * w - hat * c2) : dinner;
    }
  }
}

// out[i] = sum over `rows` of from[row * stride + i]
__global__ void __launch_bounds__(256) sum_rows_kernel(const float* __restrict__ from, long long rows, long long stride, int c, float* __restrict__ out, long long from_step, long long out_step) {
  mtb_wait_prior();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= c) return;
  from += blockIdx.y * from_step;
  double s = 0;
  for (long long r = 0; r < rows; ++r) s += from[r * stride + i];
  out[blockIdx.y * out_step + i] = (float)s;
}

int partial_rows(long long rows) {
  const int most = 4 * mtb_sm_count();
  return (int)(rows < most ? rows : most);
}

int sizes_fine(long long rows, int c, long long rows_per_gate) { return rows >= 0 && rows < (1LL << 31) && c > 0 && rows_per_gate > 0 && rows % rows_per_gate == 0; }

}  // namespace

MTB_API int mtb_add_rms_norm_forward_f32(long long rows, int c, const float* residual, const float* block, const float* weight, const float* post_weight, const float* gate,
                                         long long rows_per_gate, double scale, double eps, float* out, float* y, float* rstd, float* block_rstd, void* stream) {
  MTB_REQUIRE(sizes_fine(rows, c, gate ? rows_per_gate : 1) && eps >= 0, "add_rms_norm_forward: bad sizes");
  if (rows == 0) return MTB_OK;
  MTB_REQUIRE(residual && y && (block ? out != nullptr : !post_weight && !gate), "add_rms_norm_forward: bad arguments");
  const Operands a{residual, block, weight, post_weight, gate, rows, c, rows_per_gate, (float)scale, (float)eps};
  MTB_LAUNCH(add_rms_norm_kernel, (unsigned)rows, kThreads, 0, (cudaStream_t)stream, a, out, y, rstd, block_rstd);
  MTB_LAUNCH_CHECK("add_rms_norm_kernel");
  return MTB_OK;
}

MTB_API long long mtb_add_rms_norm_workspace_bytes(long long rows, int c) { return 4LL * 3 * c * (partial_rows(rows) + (rows > 0 ? rows : 0)); }

MTB_API int mtb_add_rms_norm_backward_f32(long long rows, int c, const float* dnew, const float* dy, const float* x, const float* rstd, const float* block,
                                          const float* block_rstd, const float* weight, const float* post_weight, const float* gate, long long rows_per_gate, double scale,
                                          float* dresidual, float* dblock, float* dweight, float* dpost_weight, float* dgate, void* workspace, long long workspace_bytes, void* stream) {
  const MtbScratchTurn turn;
  MTB_REQUIRE(sizes_fine(rows, c, gate ? rows_per_gate : 1), "add_rms_norm_backward: bad sizes");
  MTB_REQUIRE(x && rstd && (!post_weight || block_rstd) && (block || (!post_weight && !gate)), "add_rms_norm_backward: bad arguments");
  MTB_REQUIRE(workspace && workspace_bytes >= mtb_add_rms_norm_workspace_bytes(rows, c), "add_rms_norm_backward: workspace too small");
  cudaStream_t st = (cudaStream_t)stream;
  const Operands a{x, block, weight, post_weight, gate, rows, c, rows_per_gate, (float)scale, 0.f};
  const int grid = partial_rows(rows);
  float *partial = (float*)workspace, *each = dgate && gate && rows_per_gate < rows ? (rows_per_gate == 1 ? dgate : partial + 3LL * c * grid) : nullptr;
  if (grid > 0) {
    MTB_LAUNCH(add_rms_norm_backward_kernel, grid, kThreads, 0, st, a, dnew, dy, rstd, block_rstd, dresidual, dblock, each, partial);
    MTB_LAUNCH_CHECK("add_rms_norm_backward_kernel");
  }
  const auto add_up = [&](const float* from, long long n, long long stride, float* to, int many, long long from_step, long long out_step) {
    MTB_LAUNCH(sum_rows_kernel, dim3(mtb_div_up(c, 256), many), 256, 0, st, from, n, stride, c, to, from_step, out_step);
    return (int)MTB_OK;
  };
  if (dweight)
    if (int rc = add_up(partial, grid, 3LL * c, dweight, 1, 0, 0)) return rc;
  if (dpost_weight)
    if (int rc = add_up(partial + c, grid, 3LL * c, dpost_weight, 1, 0, 0)) return rc;
  if (dgate && gate) {
    if (each && each != dgate) {
      for (long long first = 0; first < rows / rows_per_gate; first += 32768) {
        const long long many = rows / rows_per_gate - first < 32768 ? rows / rows_per_gate - first : 32768;
        if (int rc = add_up(each + first * rows_per_gate * c, rows_per_gate, c, dgate + first * c, (int)many, rows_per_gate * c, c)) return rc;
      }
    } else if (!each) {
      if (int rc = add_up(partial + 2 * c, grid, 3LL * c, dgate, 1, 0, 0)) return rc;
    }
  }
  return MTB_OK;
}
