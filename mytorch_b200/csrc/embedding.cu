// Embedding: out[i] = scale * table[token[i]], and the table's gradient: dtable[v] = scale * the sum of dy[i] over the tokens
// that are v.  A token outside the table reads nothing: its row of the result is NaN, and the gradient leaves it out.
#include "colreduce.cuh"
#include <cooperative_groups.h>

namespace {

namespace cg = cooperative_groups;

template <class T>
__device__ __forceinline__ long long token_at(const void* tokens, long long i) { return (long long)static_cast<const T*>(tokens)[i]; }

// ---------------------------------------------------------------- lookup

constexpr int kLookupAhead = 4;

// One value or four a thread and step, kLookupAhead steps at a time: tokens, then rows, then results.
template <class T, int V, class I>
__global__ void __launch_bounds__(256) embedding_rows_kernel(const void* __restrict__ tokens, I total, int rows, int width, PoolDiv by_row, const float* __restrict__ table,
                                                              float scale, float* __restrict__ out) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const I per = (I)gridDim.x * 256, vectors = width / V;
  for (I k0 = (I)blockIdx.x * 256 + threadIdx.x; k0 < total; k0 += per * kLookupAhead) {
    long long t[kLookupAhead];
    unsigned col[kLookupAhead];
    VecF<V> v[kLookupAhead];
#pragma unroll
    for (int u = 0; u < kLookupAhead; ++u) {
      const I k = k0 + per * u;
      t[u] = -1;
      col[u] = 0;
      if (k < total) {
        I row;
        if (sizeof(I) == 4) row = by_row.divmod((unsigned)k, col[u]);
        else { row = k / vectors; col[u] = (unsigned)(k - row * vectors); }
        t[u] = token_at<T>(tokens, row);
      }
    }
#pragma unroll
    for (int u = 0; u < kLookupAhead; ++u) {
      if (t[u] >= 0 && t[u] < rows) v[u] = vload<V>(table + t[u] * width + (long long)col[u] * V);
      else
#pragma unroll
        for (int i = 0; i < V; ++i) v[u].v[i] = __int_as_float(0x7fc00000);
    }
#pragma unroll
    for (int u = 0; u < kLookupAhead; ++u) {
      const I k = k0 + per * u;
      if (k >= total) break;
#pragma unroll
      for (int i = 0; i < V; ++i) v[u].v[i] *= scale;
      vstore<V>(out + (long long)k * V, v[u]);
    }
  }
}

template <class T>
int lookup(const void* tokens, long long count, int rows, int width, const float* table, float scale, float* out, cudaStream_t st) {
  const bool four = width % 4 == 0 && mtb_aligned16(table) && mtb_aligned16(out);
  const long long total = count * (four ? width / 4 : width);
  const int grid = mtb_stream_grid((total + kLookupAhead - 1) / kLookupAhead, 256);
  const PoolDiv by_row((unsigned)(four ? width / 4 : width));
  const bool wide = total + (long long)grid * 256 * kLookupAhead >= 1LL << 31;
#define MTB_LOOKUP(V, I) MTB_LAUNCH((embedding_rows_kernel<T, V, I>), grid, 256, 0, st, tokens, (I)total, rows, width, by_row, table, scale, out)
  if (four && wide) MTB_LOOKUP(4, long long);
  else if (four) MTB_LOOKUP(4, int);
  else if (wide) MTB_LOOKUP(1, long long);
  else MTB_LOOKUP(1, int);
#undef MTB_LOOKUP
  return MTB_OK;
}

// ---------------------------------------------------------------- gradient: order the tokens

// Least digits first, by one cluster of CTAs, so that a pass costs two barriers of the cluster and no launch.  A warp owns a stretch of
// tokens and a row of counters, one for each digit; a token's place is what all smaller digits take, what its digit takes in the stretches before, and
// its rank in its own.  The order among equal tokens is kept, so the sums below have the same bits every time.
// The clusters behind the first clear the gradient meanwhile: rows that no token names stay so.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortAhead = 4;

struct SortPlan {
  int count, rows, passes, bits;  // bits of a digit
  long long padding;
  int *keys[2], *places[2];  // scratch; the last pass leaves its result in the first of each
  int* runs;                 // cleared: how many long runs there are
  float* dtable;
  long long cells;
};

// The table's row of token i, or `rows` for those that count nothing.
template <class T>
__device__ __forceinline__ int key_of(const void* tokens, int i, const SortPlan& p) {
  const long long t = token_at<T>(tokens, i);
  return t >= 0 && t < p.rows && t != p.padding ? (int)t : p.rows;
}

__device__ __forceinline__ void clear_cells(float* p, long long n, int block, int blocks) {
  long long head = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) / 4 % 4;
  if (head > n) head = n;
  const long long tid = (long long)block * kSortThreads + threadIdx.x, step = (long long)blocks * kSortThreads;
  if (tid < head) p[tid] = 0.f;
  p += head;
  n -= head;
  for (long long v = tid; v < n / 4; v += step) st4(p + 4 * v, make_float4(0.f, 0.f, 0.f, 0.f));
  if (tid < n % 4) p[n / 4 * 4 + tid] = 0.f;
}

template <class T>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const void* __restrict__ tokens, SortPlan p) {
  extern __shared__ int counters[];  // [kSortWarps][kDigits], then the digits' totals and first places
  mtb_launch_dependents();
  mtb_wait_prior();
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  if (blockIdx.x >= ctas) {
    clear_cells(p.dtable, p.cells, (int)blockIdx.x - ctas, (int)gridDim.x - ctas);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int *mine = counters + warp * kDigits, *totals = counters + kSortWarps * kDigits, *first = totals + kDigits, *sums = first + kDigits;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.runs = 0;
  const int each = ((p.count + ctas * kSortWarps - 1) / (ctas * kSortWarps) + 31) / 32 * 32;
  const long long begin = (long long)(cta * kSortWarps + warp) * each;
  const int lo = (int)(begin < p.count ? begin : p.count), hi = begin + each < p.count ? (int)(begin + each) : p.count;
  const unsigned below = (1u << lane) - 1;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int to = (p.passes - 1 - pass) & 1, from = to ^ 1, shift = pass * p.bits, digits = 1 << p.bits;
    for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) counters[i] = 0;
    __syncthreads();
    // what other CTAs wrote is read past the L1 cache
    auto key = [&](int i) { return pass ? __ldcg(p.keys[from] + i) : key_of<T>(tokens, i, p); };
    for (int i0 = lo; i0 < hi; i0 += 32 * kSortAhead) {
      int d[kSortAhead];
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        const int i = i0 + 32 * u + lane;
        d[u] = i < hi ? key(i) >> shift & (digits - 1) : digits;
      }
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        const unsigned same = __match_any_sync(0xffffffffu, d[u]);
        if (d[u] < digits && !(same & below)) mine[d[u]] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    if (threadIdx.x < digits) {
      int sum = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const int n = counters[w * kDigits + threadIdx.x];
        counters[w * kDigits + threadIdx.x] = sum;
        sum += n;
      }
      totals[threadIdx.x] = sum;
    }
    cluster.sync();
    int before = 0, all = 0;
    if (threadIdx.x < digits) {
      for (int r = 0; r < ctas; ++r) {
        const int n = cluster.map_shared_rank(totals, r)[threadIdx.x];
        if (r < cta) before += n;
        all += n;
      }
    }
    int upto = all;  // inclusive over the digits
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += n;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int offset = 0;
    for (int w = 0; w < warp; ++w) offset += sums[w];
    if (threadIdx.x < digits) first[threadIdx.x] = offset + upto - all + before;
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += 32 * kSortAhead) {
      int k[kSortAhead], at[kSortAhead];
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        const int i = i0 + 32 * u + lane;
        k[u] = i < hi ? key(i) : 0;
        at[u] = i < hi && pass ? __ldcg(p.places[from] + i) : i;
      }
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        const int d = i0 + 32 * u + lane < hi ? k[u] >> shift & (digits - 1) : digits;
        const unsigned same = __match_any_sync(0xffffffffu, d);
        int taken = 0;
        if (d < digits) taken = mine[d];
        __syncwarp();
        if (d < digits) {
          const int place = first[d] + taken + __popc(same & below);
          p.keys[to][place] = k[u];
          p.places[to][place] = at[u];
          if (!(same & below)) mine[d] = taken + __popc(same);
        }
        __syncwarp();
      }
    }
    cluster.sync();  // also makes this pass's places visible to the others
  }
}

// ---------------------------------------------------------------- gradient: add up

// The ordered tokens are cut into tiles of `tile`.  A run of equal tokens of up to kRun is added up by the tile it begins in, past the tile's end if need be,
// and goes to the table; a longer one is added up piece by piece, each tile its own, and the pieces are added by the kernel behind, in
// their order.  Frequent tokens thus keep no tile waiting, and the rest has no second step.
constexpr int kRun = 32, kMaxTile = kRun, kSumAhead = 8;  // a longer tile could hold a whole long run

struct SumPlan {
  const int *keys, *places;
  int count, rows, width, tile, lanes, groups;  // threads to a tile, tiles to a CTA
  float scale;
  const float* dy;
  float* dtable;
  float* pieces;  // [tiles][2][width]: of the long run that begins before the tile, of the one that begins in it
  int *runs, *run_tiles;
};

template <int V>
__global__ void __launch_bounds__(128) embedding_sum_kernel(SumPlan p) {
  // keys from kRun before a tile to kRun behind it; one more on either side tells where a run ends
  constexpr int kSpan = kMaxTile + 2 * kRun + 2;
  extern __shared__ int shared[];
  mtb_launch_dependents();
  mtb_wait_prior();
  const int group = threadIdx.x / p.lanes, lane = threadIdx.x - group * p.lanes;
  const int t0 = (blockIdx.x * p.groups + group) * p.tile;
  int *keys = shared + group * 2 * kSpan, *places = keys + kSpan;
  if (t0 < p.count) {
    for (int j = lane; j < p.tile + 2 * kRun + 2; j += p.lanes) {
      const int i = t0 - kRun - 1 + j;
      const bool in = i >= 0 && i < p.count;
      keys[j] = in ? p.keys[i] : -1;
      places[j] = in ? p.places[i] : 0;
    }
  }
  __syncthreads();
  if (t0 >= p.count) return;
  const int col = (blockIdx.y * p.lanes + lane) * V;
  const bool in_row = col < p.width;
  constexpr int kFirst = kRun + 1;  // where the tile begins
  const int end = kFirst + (p.tile < p.count - t0 ? p.tile : p.count - t0);
  float* pieces = p.pieces + 2LL * (t0 / p.tile) * p.width + col;
  int e = kFirst;
  while (e < end) {
    const int k = keys[e];
    if (k >= p.rows) break;  // those that count nothing are last
    int s = e, stop = e;  // the run's ends, as far as kRun from the tile's
    if (e == kFirst)
      while (s > 0 && keys[s - 1] == k) --s;
    while (stop < end && keys[stop] == k) ++stop;
    const int inside = stop;
    if (inside == end)
      while (stop - s <= kRun && keys[stop] == k) ++stop;
    const bool whole = stop - s <= kRun;
    if (whole && s < e) { e = inside; continue; }  // the tile before has it
    const int last = whole ? stop : inside;
    VecF<V> sum;
#pragma unroll
    for (int i = 0; i < V; ++i) sum.v[i] = 0.f;
    if (in_row) {
      for (int j0 = e; j0 < last; j0 += kSumAhead) {
        VecF<V> v[kSumAhead];
#pragma unroll
        for (int u = 0; u < kSumAhead; ++u)
          if (j0 + u < last) v[u] = vload<V>(p.dy + (long long)places[j0 + u] * p.width + col);
#pragma unroll
        for (int u = 0; u < kSumAhead; ++u)
          if (j0 + u < last)
#pragma unroll
            for (int i = 0; i < V; ++i) sum.v[i] += v[u].v[i];
      }
      if (whole) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum.v[i] *= p.scale;
        vstore<V>(p.dtable + (long long)k * p.width + col, sum);
      } else {
        vstore<V>(pieces + (s < e ? 0 : p.width), sum);
      }
    }
    if (!whole && s == e && lane == 0 && blockIdx.y == 0) p.run_tiles[atomicAdd(p.runs, 1)] = t0 / p.tile;
    e = inside;
  }
}

constexpr int kJoinThreads = 512;

// One CTA a long run and 32 lanes' columns: its warps add up a part of the pieces each, and those sums are added in their order.
template <int V>
__global__ void __launch_bounds__(kJoinThreads) embedding_join_kernel(SumPlan p) {
  mtb_launch_dependents();
  mtb_wait_prior();
  __shared__ float sums[kJoinThreads / 32][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kJoinThreads / 32;
  const int columns = (p.width + 32 * V - 1) / (32 * V), tiles = (p.count + p.tile - 1) / p.tile;
  const int items = *p.runs * columns;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int t = p.run_tiles[item / columns], col = (item % columns * 32 + lane) * V;
    const int last = t + 1 < tiles ? (t + 1) * p.tile - 1 : p.count - 1, k = p.keys[last];  // the run that begins in the tile and ends behind it
    int a = t, b = tiles;  // tile a begins within the run (or is t), tile b does not: 32 probes at a time
    while (b - a > 1) {
      const int step = (b - a + 31) / 32, probe = a + 1 + lane * step;
      const unsigned yes = __ballot_sync(0xffffffffu, probe < b && p.keys[(long long)probe * p.tile] == k);
      const int n = __popc(yes);
      if (n == 0) { b = a + 1; break; }
      const int na = a + 1 + (n - 1) * step, nb = na + step;
      a = na;
      b = nb < b ? nb : b;
    }
    const int count = a - t + 1;  // pieces
    const int lo = (int)((long long)count * warp / warps), hi = (int)((long long)count * (warp + 1) / warps);
    VecF<V> sum;
#pragma unroll
    for (int i = 0; i < V; ++i) sum.v[i] = 0.f;
    if (col < p.width) {
      for (int j0 = lo; j0 < hi; j0 += kSumAhead) {
        VecF<V> v[kSumAhead];
#pragma unroll
        for (int u = 0; u < kSumAhead; ++u)
          if (j0 + u < hi) v[u] = vload<V>(p.pieces + (2LL * (t + j0 + u) + (j0 + u == 0 ? 1 : 0)) * p.width + col);
#pragma unroll
        for (int u = 0; u < kSumAhead; ++u)
          if (j0 + u < hi)
#pragma unroll
            for (int i = 0; i < V; ++i) sum.v[i] += v[u].v[i];
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sums[warp][lane * V + i] = sum.v[i];
    __syncthreads();
    if (warp == 0 && col < p.width) {
      for (int w = 1; w < warps; ++w)
#pragma unroll
        for (int i = 0; i < V; ++i) sum.v[i] += sums[w][lane * V + i];
#pragma unroll
      for (int i = 0; i < V; ++i) sum.v[i] *= p.scale;
      vstore<V>(p.dtable + (long long)k * p.width + col, sum);
    }
    __syncthreads();
  }
}

struct GradPlan {
  int passes, bits, ctas, tile, tiles, lanes, groups, columns;
  long long bytes;
};

// Scratch: two sets of keys and places, the list of long runs, the pieces.
GradPlan plan_gradient(long long count, int rows, int width, bool four) {
  GradPlan g{};
  int bits = 1;
  while ((1LL << bits) <= rows) ++bits;  // the largest key is `rows`
  g.passes = (bits + kDigitBits - 1) / kDigitBits;
  g.bits = (bits + g.passes - 1) / g.passes;
  g.ctas = 1;
  while (g.ctas < 16 && count > (long long)g.ctas * kSortThreads * 4) g.ctas *= 2;
  const int vectors = four ? width / 4 : width;
  g.lanes = 4;
  while (g.lanes < vectors && g.lanes < 32) g.lanes *= 2;
  if (vectors > 32) g.lanes = vectors > 128 ? 128 : (vectors + 31) / 32 * 32;
  g.groups = 128 / g.lanes;
  g.columns = (vectors + g.lanes - 1) / g.lanes;
  // tiles as large as leaves every SM some CTAs
  g.tile = 8;
  while (g.tile < kMaxTile && count / (2LL * g.tile * g.groups) * g.columns >= mtb_sm_count() * 16LL) g.tile *= 2;
  g.tiles = (int)((count + g.tile - 1) / g.tile);
  g.bytes = 16 * count + 4LL * g.tiles + 512 + 8LL * g.tiles * width;
  return g;
}

template <class T>
int sort_tokens(const void* tokens, const SortPlan& p, int ctas, cudaStream_t st) {
  static unsigned long long opted;
  constexpr int smem = (kSortWarps * kDigits + 2 * kDigits + kSortWarps) * 4;
  if (int rc = mtb_opt_in_smem((const void*)embedding_sort_kernel<T>, smem, &opted)) return rc;
  static unsigned long long wide;
  int device = 0;
  MTB_CUDA(cudaGetDevice(&device));
  if (device >= 64 || !((__atomic_load_n(&wide, __ATOMIC_ACQUIRE) >> device) & 1ull)) {
    MTB_CUDA(cudaFuncSetAttribute((const void*)embedding_sort_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (device < 64) __atomic_fetch_or(&wide, 1ull << device, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t cfg = {};
  const long long clear = (p.cells + 4LL * kSortThreads * 4 - 1) / (4LL * kSortThreads * 4);  // four vectors a thread
  long long blocks = mtb_sm_count() / ctas * ctas - ctas;
  if (clear < blocks) blocks = (clear + ctas - 1) / ctas * ctas;
  cfg.gridDim = dim3((unsigned)(ctas + (blocks < ctas ? ctas : blocks)));
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  MTB_CUDA(cudaLaunchKernelEx(&cfg, embedding_sort_kernel<T>, tokens, p));
  return MTB_OK;
}

template <int V>
int add_up(const SumPlan& p, const GradPlan& g, cudaStream_t st) {
  const int smem = g.groups * 2 * (kMaxTile + 2 * kRun + 2) * 4;
  MTB_LAUNCH(embedding_sum_kernel<V>, dim3(mtb_div_up(g.tiles, g.groups), g.columns), g.lanes * g.groups, smem, st, p);
  if (p.count > kRun) MTB_LAUNCH(embedding_join_kernel<V>, mtb_sm_count() * 2, kJoinThreads, 0, st, p);
  return MTB_OK;
}

}  // namespace

MTB_API int mtb_embedding_forward_f32(int kind, const void* tokens, long long count, int rows, int width, const float* table, double scale, float* out,
                                      void* stream) {
  MTB_REQUIRE((kind == 0 || kind == 1) && count >= 0 && rows > 0 && width > 0, "embedding_forward: bad arguments");
  if (count == 0) return MTB_OK;
  MTB_REQUIRE(tokens && table && out, "embedding_forward: null tensor");
  return kind == 0 ? lookup<int>(tokens, count, rows, width, table, (float)scale, out, (cudaStream_t)stream)
                   : lookup<long long>(tokens, count, rows, width, table, (float)scale, out, (cudaStream_t)stream);
}

MTB_API long long mtb_embedding_backward_workspace_bytes(long long count, int rows, int width) {
  if (count <= 0 || rows <= 0 || width <= 0) return 256;
  const long long a = plan_gradient(count, rows, width, false).bytes, b = width % 4 == 0 ? plan_gradient(count, rows, width, true).bytes : 0;
  return a > b ? a : b;
}

MTB_API int mtb_embedding_backward_f32(int kind, const void* tokens, long long count, int rows, int width, const float* dy, double scale, long long padding,
                                       float* dtable, void* workspace, long long workspace_bytes, void* stream) {
  const MtbScratchTurn turn;
  MTB_REQUIRE((kind == 0 || kind == 1) && count >= 0 && rows > 0 && width > 0 && dtable, "embedding_backward: bad arguments");
  MTB_REQUIRE(count == 0 || (tokens && dy), "embedding_backward: null tensor");
  MTB_REQUIRE(count <= 1LL << 30 && rows <= 1 << 30, "embedding_backward: %lld tokens, %d rows", count, rows);
  MTB_REQUIRE(workspace && workspace_bytes >= mtb_embedding_backward_workspace_bytes(count, rows, width), "embedding_backward: workspace too small");
  cudaStream_t st = (cudaStream_t)stream;
  if (count == 0) {
    MTB_CUDA(cudaMemsetAsync(dtable, 0, 4LL * rows * width, st));
    return MTB_OK;
  }
  const bool four = width % 4 == 0 && mtb_aligned16(dy) && mtb_aligned16(dtable) && mtb_aligned16(workspace);
  const GradPlan g = plan_gradient(count, rows, width, four);
  MTB_REQUIRE(g.columns < 65536, "embedding_backward: rows of %d values", width);
  float* pieces = (float*)workspace;  // first: read and written four at a time
  int* ints = (int*)(pieces + 2LL * g.tiles * width);
  int* keys[2] = {ints, ints + count};
  int* places[2] = {ints + 2 * count, ints + 3 * count};
  int *run_tiles = ints + 4 * count, *runs = run_tiles + g.tiles;
  SortPlan s{(int)count, rows, g.passes, g.bits, padding, {keys[0], keys[1]}, {places[0], places[1]}, runs, dtable, (long long)rows * width};
  if (int rc = kind == 0 ? sort_tokens<int>(tokens, s, g.ctas, st) : sort_tokens<long long>(tokens, s, g.ctas, st)) return rc;
  const SumPlan p{keys[0], places[0], (int)count, rows, width, g.tile, g.lanes, g.groups, (float)scale, dy, dtable, pieces, runs, run_tiles};
  return four ? add_up<4>(p, g, st) : add_up<1>(p, g, st);
}
