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
// What bounds it: latency, and scattered stores, of which an SM takes one line a cycle.  So a token and its place travel as one 8-byte entry, and a CTA puts its
// share in order in shared memory first and writes stretches of a digit.  SORTED_FIGURES
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortAhead = 8, kSortCtas = 16, kStaged = 8192;

struct SortPlan {
  int count, rows, passes, bits;  // bits of a digit
  long long padding;
  int2* entries[2];  // scratch, (token, place); the last pass leaves its result in the first
  int* runs;         // cleared: how many long runs there are
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
  extern __shared__ int2 staged[];  // [kStaged], then counters [kSortWarps][kDigits], the CTA's totals of the digits, where they go
  mtb_launch_dependents();
  mtb_wait_prior();
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  if (blockIdx.x >= ctas) {
    clear_cells(p.dtable, p.cells, (int)blockIdx.x - ctas, (int)gridDim.x - ctas);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int *counters = (int*)(staged + kStaged), *mine = counters + warp * kDigits, *totals = counters + kSortWarps * kDigits;
  int *local = totals + kDigits, *shift_to = local + kDigits, *sums = shift_to + kDigits;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.runs = 0;
  const int each = ((p.count + ctas * kSortWarps - 1) / (ctas * kSortWarps) + 31) / 32 * 32;
  auto bounded = [&](long long i) { return (int)(i < p.count ? i : p.count); };
  const int lo = bounded((long long)(cta * kSortWarps + warp) * each), hi = bounded((long long)(cta * kSortWarps + warp + 1) * each);
  const int share = bounded((long long)(cta + 1) * kSortWarps * each) - bounded((long long)cta * kSortWarps * each);
  const unsigned below = (1u << lane) - 1;
  const bool held = each <= 32 * kSortAhead, stage = share <= kStaged;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int to = (p.passes - 1 - pass) & 1, shift = pass * p.bits, digits = 1 << p.bits;
    for (int i = threadIdx.x; i < kSortWarps * kDigits / 4; i += kSortThreads) ((int4*)counters)[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    int2 entry[kSortAhead];
    auto load = [&](int i0) {
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        const int i = i0 + 32 * u + lane;
        // what other CTAs wrote is read past the L1 cache
        if (i < hi) entry[u] = pass ? __ldcg(p.entries[to ^ 1] + i) : make_int2(key_of<T>(tokens, i, p), i);
      }
    };
    for (int i0 = lo; i0 < hi; i0 += 32 * kSortAhead) {
      load(i0);
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u)
        if (i0 + 32 * u + lane < hi) atomicAdd(mine + (entry[u].x >> shift & (digits - 1)), 1);
    }
    __syncthreads();
    int total = 0;
    if (threadIdx.x < digits) {
      for (int w0 = 0; w0 < kSortWarps; w0 += 16) {
        int n[16];
#pragma unroll
        for (int w = 0; w < 16; ++w) n[w] = counters[(w0 + w) * kDigits + threadIdx.x];
#pragma unroll
        for (int w = 0; w < 16; ++w) {
          counters[(w0 + w) * kDigits + threadIdx.x] = total;
          total += n[w];
        }
      }
      totals[threadIdx.x] = total;
    }
    cluster.sync();
    int before = 0, all = 0;
    if (threadIdx.x < digits) {
#pragma unroll
      for (int r = 0; r < kSortCtas; ++r) {
        const int n = r < ctas ? cluster.map_shared_rank(totals, r)[threadIdx.x] : 0;
        if (r < cta) before += n;
        all += n;
      }
    }
    int upto_all = all, upto_total = total;  // inclusive over the digits
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, upto_all, o), b = __shfl_up_sync(0xffffffffu, upto_total, o);
      if (lane >= o) { upto_all += a; upto_total += b; }
    }
    if (lane == 31) { sums[warp] = upto_all; sums[kSortWarps + warp] = upto_total; }
    __syncthreads();
    if (threadIdx.x < digits) {
      int offset = upto_all - all + before, here = upto_total - total;
      for (int w = 0; w < warp; ++w) { offset += sums[w]; here += sums[kSortWarps + w]; }
      local[threadIdx.x] = here;
      shift_to[threadIdx.x] = offset - here;
    }
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += 32 * kSortAhead) {
      if (!held) load(i0);
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        if (i0 + 32 * u >= hi) break;
        const bool in = i0 + 32 * u + lane < hi;
        const int d = entry[u].x >> shift & (digits - 1);
        // the lanes with the same digit, bit by bit (__match_any_sync took some 500 cycles for 32 different ones)
        unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
        for (int b = 0; b < kDigitBits; ++b) {
          const unsigned set = __ballot_sync(0xffffffffu, d >> b & 1);
          same &= d >> b & 1 ? set : ~set;
        }
        int taken = 0;
        if (in) taken = mine[d];
        __syncwarp();
        if (in) {
          const int place = local[d] + taken + __popc(same & below);
          if (stage) staged[place] = entry[u];
          else p.entries[to][place + shift_to[d]] = entry[u];
          if (!(same & below)) mine[d] = taken + __popc(same);
        }
        __syncwarp();
      }
    }
    if (stage) {
      __syncthreads();
      for (int i = threadIdx.x; i < share; i += kSortThreads) {
        const int2 e = staged[i];
        p.entries[to][i + shift_to[e.x >> shift & (digits - 1)]] = e;
      }
    }
    cluster.sync();  // also makes this pass's entries visible to the others
  }
}

// ---------------------------------------------------------------- gradient: add up

// The ordered tokens are cut into tiles of `tile`.  A run of equal tokens of up to kRun is added up by the tile it begins in, past the tile's end if need be,
// and goes to the table; a longer one is added up piece by piece, each tile its own, and the pieces are added by the kernel behind, in
// their order.  Frequent tokens thus keep no tile waiting, and the rest has no second step.
constexpr int kRun = 32, kMaxTile = kRun, kSumAhead = 8;  // a longer tile could hold a whole long run

struct SumPlan {
  const int2* entries;
  int count, rows, width, tile, lanes, groups;  // threads to a tile, tiles to a CTA
  float scale;
  const float* dy;
  float* dtable;
  float* pieces;  // [tiles][2][width]: of the long run that begins before the tile, of the one that begins in it
  int* runs;              // how many long runs there are,
  int2* run_starts;       // of each, the tile that it begins in and its token
  int* run_ends;          // [rows]: the tile that a long run of this token ends in
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
      const int2 entry = in ? p.entries[i] : make_int2(-1, 0);
      keys[j] = entry.x;
      places[j] = entry.y;
    }
  }
  __syncthreads();
  if (t0 >= p.count) return;
  const int col = (blockIdx.y * p.lanes + lane) * V;
  if (col >= p.width) return;
  // the entries [e, to) are this tile's: without the end of a short run that began before it, with the rest of one that begins in it
  int e = kRun + 1, to = e + (p.tile < p.count - t0 ? p.tile : p.count - t0);
  while (to > e && keys[to - 1] >= p.rows) --to;  // those that count nothing are last
  if (e == to) return;
  bool begun = keys[e - 1] == keys[e], left = false;  // long runs that began before, that go on behind
  if (begun) {
    const int k = keys[e];
    int s = e - 1, stop = e + 1;
    while (s > 0 && keys[s - 1] == k) --s;
    while (stop - s <= kRun && keys[stop] == k) ++stop;
    if (stop - s <= kRun) {
      begun = false;
      e = stop < to ? stop : to;
      if (e == to) return;
    } else if (keys[to] != k && blockIdx.y == 0 && lane == 0) {
      p.run_ends[k] = t0 / p.tile;
    }
  }
  if (keys[to] == keys[to - 1] && !(begun && keys[e] == keys[to - 1])) {
    const int k = keys[to];
    int s = to - 1, stop = to + 1;
    while (s > e && keys[s - 1] == k) --s;
    while (stop - s <= kRun && keys[stop] == k) ++stop;
    left = stop - s > kRun;
    if (!left) to = stop;
    else if (blockIdx.y == 0 && lane == 0) p.run_starts[atomicAdd(p.runs, 1)] = make_int2(t0 / p.tile, k);
  }
  float* pieces = p.pieces + 2LL * (t0 / p.tile) * p.width + col;
  const float* dy = p.dy + col;
  VecF<V> sum;
#pragma unroll
  for (int i = 0; i < V; ++i) sum.v[i] = 0.f;
  int k = keys[e];
  auto flush = [&](bool is_last) {
    float* to_row = begun ? pieces : is_last && left ? pieces + p.width : p.dtable + (long long)k * p.width + col;
    if (!begun && !(is_last && left)) {
#pragma unroll
      for (int i = 0; i < V; ++i) sum.v[i] *= p.scale;
    }
    vstore<V>(to_row, sum);
    begun = false;
#pragma unroll
    for (int i = 0; i < V; ++i) sum.v[i] = 0.f;
  };
  // rows are loaded kSumAhead at a time, whichever runs they belong to
  for (; e < to; e += kSumAhead) {
    VecF<V> v[kSumAhead];
#pragma unroll
    for (int u = 0; u < kSumAhead; ++u)
      if (e + u < to) v[u] = vload<V>(dy + (long long)places[e + u] * p.width);
#pragma unroll
    for (int u = 0; u < kSumAhead; ++u) {
      if (e + u >= to) break;
      if (keys[e + u] != k) {
        flush(false);
        k = keys[e + u];
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum.v[i] += v[u].v[i];
    }
  }
  flush(true);
}

constexpr int kJoinThreads = 256, kJoinAhead = 4;

// One CTA a long run and 32 lanes' columns: its warps add up a part of the pieces each, and those sums are added in their order.
template <int V>
__global__ void __launch_bounds__(kJoinThreads, 5) embedding_join_kernel(SumPlan p) {
  mtb_launch_dependents();
  mtb_wait_prior();
  __shared__ float sums[kJoinThreads / 32][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kJoinThreads / 32;
  const int columns = (p.width + 32 * V - 1) / (32 * V);
  const int items = *p.runs * columns;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int2 start = p.run_starts[item / columns];
    const int t = start.x, k = start.y, col = (item % columns * 32 + lane) * V;
    const int count = p.run_ends[k] - t + 1;  // pieces
    const int lo = (int)((long long)count * warp / warps), hi = (int)((long long)count * (warp + 1) / warps);
    VecF<V> sum;
#pragma unroll
    for (int i = 0; i < V; ++i) sum.v[i] = 0.f;
    if (col < p.width) {
      for (int j0 = lo; j0 < hi; j0 += kJoinAhead) {
        VecF<V> v[kJoinAhead];
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u)
          if (j0 + u < hi) v[u] = vload<V>(p.pieces + (2LL * (t + j0 + u) + (j0 + u == 0 ? 1 : 0)) * p.width + col);
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u)
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

// Scratch: two sets of entries, the long runs' starts and ends, the pieces.
GradPlan plan_gradient(long long count, int rows, int width, bool four) {
  GradPlan g{};
  int bits = 1;
  while ((1LL << bits) <= rows) ++bits;  // the largest key is `rows`
  g.passes = (bits + kDigitBits - 1) / kDigitBits;
  g.bits = (bits + g.passes - 1) / g.passes;
  g.ctas = 1;
  while (g.ctas < kSortCtas && count > (long long)g.ctas * kSortThreads) g.ctas *= 2;
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
  g.bytes = 16 * count + 4LL * rows + 8LL * g.tiles + 512 + 8LL * g.tiles * width;
  return g;
}

template <class T>
int sort_tokens(const void* tokens, const SortPlan& p, int ctas, cudaStream_t st) {
  static unsigned long long opted;
  constexpr int smem = kStaged * 8 + (kSortWarps * kDigits + 3 * kDigits + 2 * kSortWarps) * 4;
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
  if (p.count > kRun) MTB_LAUNCH(embedding_join_kernel<V>, mtb_sm_count() * 5, kJoinThreads, 0, st, p);
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
  int2* entries = (int2*)(pieces + 2LL * g.tiles * width);
  int2* run_starts = entries + 2 * count;
  int *run_ends = (int*)(run_starts + g.tiles), *runs = run_ends + rows;
  SortPlan s{(int)count, rows, g.passes, g.bits, padding, {entries, entries + count}, runs, dtable, (long long)rows * width};
  if (int rc = kind == 0 ? sort_tokens<int>(tokens, s, g.ctas, st) : sort_tokens<long long>(tokens, s, g.ctas, st)) return rc;
  const SumPlan p{entries, (int)count, rows, width, g.tile, g.lanes, g.groups, (float)scale, dy, dtable, pieces, runs, run_starts, run_ends};
  return four ? add_up<4>(p, g, st) : add_up<1>(p, g, st);
}
