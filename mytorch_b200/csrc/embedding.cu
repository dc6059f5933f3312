// Embedding: out[i] = scale * table[token[i]], and the table's gradient: dtable[v] = scale * the sum of dy[i] over the tokens
// that are v.  A token outside the table reads nothing: its row of the result is NaN, and the gradient leaves it out.
#include "common.cuh"

namespace {

template <class T>
__device__ __forceinline__ long long token_at(const void* tokens, long long i) { return (long long)static_cast<const T*>(tokens)[i]; }

template <class T>
__global__ void __launch_bounds__(256) embedding_rows_kernel(const void* __restrict__ tokens, long long count, int rows, int width, const float* __restrict__ table,
                                                              float scale, float* __restrict__ out) {
  mtb_launch_dependents();
  mtb_wait_prior();
  for (long long k = blockIdx.x * 256LL + threadIdx.x; k < count * width; k += gridDim.x * 256LL) {
    const long long t = token_at<T>(tokens, k / width);
    out[k] = t >= 0 && t < rows ? table[t * width + k % width] * scale : __int_as_float(0x7fc00000);
  }
}

// One warp a row of the table and 128 columns: it looks through all tokens for its own.
template <class T>
__global__ void __launch_bounds__(128) embedding_grad_kernel(const void* __restrict__ tokens, long long count, int rows, int width, const float* __restrict__ dy,
                                                              float scale, long long padding, float* __restrict__ dtable) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const int lane = threadIdx.x & 31, c0 = blockIdx.y * 128 + lane;
  const long long v = blockIdx.x * 4LL + (threadIdx.x >> 5);
  if (v >= rows) return;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (long long i = 0; v != padding && i < count; i += 32) {
    unsigned mine = __ballot_sync(0xffffffffu, i + lane < count && token_at<T>(tokens, i + lane) == v);
    for (; mine; mine &= mine - 1) {
      const float* row = dy + (i + __ffs(mine) - 1) * width;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c0 + 32 * k < width) acc[k] += row[c0 + 32 * k];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (c0 + 32 * k < width) dtable[v * width + c0 + 32 * k] = acc[k] * scale;
}

}  // namespace

MTB_API int mtb_embedding_forward_f32(int kind, const void* tokens, long long count, int rows, int width, const float* table, double scale, float* out,
                                      void* stream) {
  MTB_REQUIRE((kind == 0 || kind == 1) && count >= 0 && rows > 0 && width > 0, "embedding_forward: bad arguments");
  if (count == 0) return MTB_OK;
  MTB_REQUIRE(tokens && table && out, "embedding_forward: null tensor");
  cudaStream_t st = (cudaStream_t)stream;
  const int grid = mtb_stream_grid(count * width, 256);
  if (kind == 0) MTB_LAUNCH(embedding_rows_kernel<int>, grid, 256, 0, st, tokens, count, rows, width, table, (float)scale, out);
  else MTB_LAUNCH(embedding_rows_kernel<long long>, grid, 256, 0, st, tokens, count, rows, width, table, (float)scale, out);
  return MTB_OK;
}

MTB_API long long mtb_embedding_backward_workspace_bytes(long long count, int rows, int width) {
  (void)count, (void)rows, (void)width;
  return 256;
}

MTB_API int mtb_embedding_backward_f32(int kind, const void* tokens, long long count, int rows, int width, const float* dy, double scale, long long padding,
                                       float* dtable, void* workspace, long long workspace_bytes, void* stream) {
  const MtbScratchTurn turn;
  MTB_REQUIRE((kind == 0 || kind == 1) && count >= 0 && rows > 0 && width > 0 && dtable, "embedding_backward: bad arguments");
  MTB_REQUIRE(count == 0 || (tokens && dy), "embedding_backward: null tensor");
  MTB_REQUIRE(workspace && workspace_bytes >= mtb_embedding_backward_workspace_bytes(count, rows, width), "embedding_backward: workspace too small");
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid(mtb_div_up(rows, 4), mtb_div_up(width, 128));
  MTB_REQUIRE(grid.y < 65536, "embedding_backward: rows of %d values", width);
  if (kind == 0) MTB_LAUNCH(embedding_grad_kernel<int>, grid, 128, 0, st, tokens, count, rows, width, dy, (float)scale, padding, dtable);
  else MTB_LAUNCH(embedding_grad_kernel<long long>, grid, 128, 0, st, tokens, count, rows, width, dy, (float)scale, padding, dtable);
  return MTB_OK;
}
