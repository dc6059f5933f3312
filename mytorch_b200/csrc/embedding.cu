// Embedding: out[i] = scale * table[token[i]], and the table's gradient: dtable[v] = scale * the sum of dy[i] over the tokens
// that are v.  A token outside the table reads nothing: its row of the result is NaN, and the gradient leaves it out.
#include "colreduce.cuh"

namespace {

template <class T>
__device__ __forceinline__ long long token_at(const void* tokens, long long i) { return (long long)static_cast<const T*>(tokens)[i]; }

// ---------------------------------------------------------------- lookup

// Bound by memory: 131072 rows of 512 values out of 50000, 318 MB read and written at least: 50.3 us, 6.3 TB/s.  Two steps ahead 53.7 us, eight (fewer threads) 58.7;
// a result that is not marked 53.2; steps a grid apart instead of side by side 55.2; as many CTAs as fit the SMs, with a loop, 57.4.  Eight
// tokens: a launch.
constexpr int kLookupAhead = 4;
constexpr long long kStreamed = 64 << 20;  // bytes: half of L2

// One value or four a thread and step, kLookupAhead steps at once: tokens, then rows, then results.  STREAM: the result is more than L2 holds, and is
// marked to leave it first, so that rows which are read again stay.
template <class T, int V, class I, bool STREAM>
__global__ void __launch_bounds__(256) embedding_rows_kernel(const void* __restrict__ tokens, I total, int rows, int width, PoolDiv by_row, const float* __restrict__ table,
                                                              float scale, float* __restrict__ out) {
  mtb_launch_dependents();
  mtb_wait_prior();
  const I k0 = (I)blockIdx.x * 256 * kLookupAhead + threadIdx.x, per = 256, vectors = width / V;
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
    float* to = out + (long long)k * V;
    if (!STREAM) vstore<V>(to, v[u]);
    else if (V == 4) __stcs((float4*)to, make_float4(v[u].v[0], v[u].v[1 % V], v[u].v[2 % V], v[u].v[3 % V]));
    else __stcs(to, v[u].v[0]);
  }
}

template <class T>
int lookup(const void* tokens, long long count, int rows, int width, const float* table, float scale, float* out, cudaStream_t st) {
  const bool four = width % 4 == 0 && mtb_aligned16(table) && mtb_aligned16(out);
  const long long total = count * (four ? width / 4 : width);
  const long long grid = (total + 256 * kLookupAhead - 1) / (256 * kLookupAhead);
  MTB_REQUIRE(grid < 1LL << 31, "embedding_forward: too many values");
  const PoolDiv by_row((unsigned)(four ? width / 4 : width));
  const bool wide = total + 256 * kLookupAhead >= 1LL << 31, stream = 4 * count * width > kStreamed;
#define MTB_LOOKUP(V, I)                                                                                                              \
  do {                                                                                                                                \
    if (stream) MTB_LAUNCH((embedding_rows_kernel<T, V, I, true>), (int)grid, 256, 0, st, tokens, (I)total, rows, width, by_row, table, scale, out); \
    else MTB_LAUNCH((embedding_rows_kernel<T, V, I, false>), (int)grid, 256, 0, st, tokens, (I)total, rows, width, by_row, table, scale, out);       \
  } while (0)
  if (four && wide) MTB_LOOKUP(4, long long);
  else if (four) MTB_LOOKUP(4, int);
  else if (wide) MTB_LOOKUP(1, long long);
  else MTB_LOOKUP(1, int);
#undef MTB_LOOKUP
  return MTB_OK;
}

// ---------------------------------------------------------------- gradient: order the tokens

// The gradient's kernels let the next one come once they have waited themselves, not before: else kernels of several calls are on the SMs at once, waiting, and
// those that work find too few places (23 tokens to 48423 rows of 458, call after call: 57 us, 24 this way).

// Least digits first.  A CTA has a share of the tokens, a warp of it a stretch and a row of counters, one for each digit; a token's place is what all
// smaller digits take, what its digit takes in the shares and stretches before, and its rank in its own.  The order among equal tokens is
// kept, so the sums below have the same bits every time.  Up to kOneCta tokens are ordered by one CTA in one launch; more by a launch that counts
// the first digits and one for each pass, which counts the next pass's digits where it puts the tokens.
// What bounds it: latency, the ranking's instructions (on the 16 SMs of one cluster, with barriers instead of
// launches, 131072 tokens took 35 us) and scattered stores, of which an SM takes one line a cycle.  So all SMs take part, a token and its place
// travel as one 8-byte entry, and a CTA puts its share in order in shared memory first and writes stretches of a digit.
// kOneAhead: 2049 tokens 17.8 us of the whole gradient instead of 20.1, 4096 (rows of 512) 17.2 instead of 19.0; sixteen a thread lose: 8191 tokens 26.7, not 21.4.
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kDigitBits = 8, kDigits = 1 << kDigitBits;
constexpr int kSortAhead = 4, kOneAhead = 8, kOneCta = kSortThreads * kOneAhead, kStaged = 8192;

struct SortPlan {
  int count, rows, passes, bits;  // bits of a digit
  int share_bits, ctas;           // tokens to a CTA: 1 << share_bits
  long long padding;
  int2 *from, *to;  // scratch, (token, place)
  int* table;       // scratch, [passes][ctas][digits]: how many of each digit a CTA's share has in each pass
  int* runs;        // cleared: how many long runs there are
};

// The table's row of token i, or `rows` for those that count nothing.
template <class T>
__device__ __forceinline__ int key_of(const void* tokens, int i, const SortPlan& p) {
  const long long t = token_at<T>(tokens, i);
  return t >= 0 && t < p.rows && t != p.padding ? (int)t : p.rows;
}

struct alignas(16) SortShared {
  int counters[kSortWarps][kDigits];
  unsigned lanes[kSortWarps][kDigits];  // 0 between two uses
  int local[kDigits];     // where a digit begins in the CTA's own order
  int shift_to[kDigits];  // from there to its place among all
  int sums[2][kSortWarps];
};
static_assert(alignof(SortShared) % 16 == 0 && offsetof(SortShared, lanes) % 16 == 0, "counters and lanes are cleared, and take sums, 16 bytes at a time");

// Exclusive sums over the digits of `a` and `b`, one digit a thread.  All threads call it; `sums` is free again after the next barrier.
__device__ __forceinline__ void scan_digits(int& a, int& b, SortShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int ua = a, ub = b;
  for (int o = 1; o < 32; o <<= 1) {
    const int na = __shfl_up_sync(0xffffffffu, ua, o), nb = __shfl_up_sync(0xffffffffu, ub, o);
    if (lane >= o) { ua += na; ub += nb; }
  }
  if (lane == 31) { sh.sums[0][warp] = ua; sh.sums[1][warp] = ub; }
  __syncthreads();
  ua -= a;
  ub -= b;
  for (int w = 0; w < warp; ++w) { ua += sh.sums[0][w]; ub += sh.sums[1][w]; }
  a = ua;
  b = ub;
}

// Turns the warps' counts of a digit into what the warps before have of it; the whole CTA's count.
__device__ __forceinline__ int sum_warps(SortShared& sh, int digits) {
  int total = 0;
  if (threadIdx.x < digits) {
    int n[kSortWarps];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) n[w] = sh.counters[w][threadIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      sh.counters[w][threadIdx.x] = total;
      total += n[w];
    }
  }
  return total;
}

// An entry's place in its CTA's order; advances the warp's counters.  All lanes call it; `in`: the lane has an entry.  The lanes with the same digit find one
// another in a word of shared memory: 20 instructions, against 40 and more bit by bit with ballots, and some 500 cycles of __match_any_sync.
__device__ __forceinline__ int place_of(bool in, int digit, int* mine, unsigned* lanes, const int* local) {
  const int lane = threadIdx.x & 31;
  if (in) atomicOr(lanes + digit, 1u << lane);
  __syncwarp();
  unsigned same = 0;
  int place = 0;
  if (in) {
    same = lanes[digit];
    place = mine[digit];
  }
  __syncwarp();
  const int rank = __popc(same & ((1u << lane) - 1));
  if (in && rank == 0) {
    mine[digit] = place + __popc(same);
    lanes[digit] = 0;
  }
  __syncwarp();
  return in ? local[digit] + place + rank : 0;
}

template <class T>
__global__ void __launch_bounds__(kSortThreads) embedding_order_kernel(const void* __restrict__ tokens, SortPlan p) {
  __shared__ SortShared sh;
  extern __shared__ int2 staged[];  // [kOneCta]
  mtb_wait_prior();
  mtb_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << p.bits;
  const int ahead = (p.count + kSortThreads - 1) / kSortThreads, lo = warp * 32 * ahead + lane;  // a warp's stretch: as short as the count allows
  if (threadIdx.x == 0) *p.runs = 0;
  for (int i = threadIdx.x; i < kSortWarps * kDigits / 4; i += kSortThreads) ((int4*)sh.lanes)[i] = make_int4(0, 0, 0, 0);
  int2 entry[kOneAhead];
#pragma unroll
  for (int u = 0; u < kOneAhead; ++u)
    if (u < ahead && lo + 32 * u < p.count) entry[u] = make_int2(key_of<T>(tokens, lo + 32 * u, p), lo + 32 * u);
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    for (int i = threadIdx.x; i < kSortWarps * kDigits / 4; i += kSortThreads) ((int4*)sh.counters)[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kOneAhead; ++u)
      if (u < ahead && lo + 32 * u < p.count) atomicAdd(&sh.counters[warp][entry[u].x >> shift & (digits - 1)], 1);
    __syncthreads();
    int total = sum_warps(sh, digits), unused = 0;
    scan_digits(total, unused, sh);
    if (threadIdx.x < digits) sh.local[threadIdx.x] = total;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kOneAhead; ++u) {
      if (u < ahead && lo - lane + 32 * u < p.count) {
        const bool in = lo + 32 * u < p.count;
        const int place = place_of(in, entry[u].x >> shift & (digits - 1), sh.counters[warp], sh.lanes[warp], sh.local);
        if (in) staged[place] = entry[u];
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kOneAhead; ++u)
      if (u < ahead && lo + 32 * u < p.count) entry[u] = staged[lo + 32 * u];
  }
#pragma unroll
  for (int u = 0; u < kOneAhead; ++u)
    if (u < ahead && lo + 32 * u < p.count) p.to[lo + 32 * u] = entry[u];
}

template <class T>
__global__ void __launch_bounds__(kSortThreads) embedding_count_kernel(const void* __restrict__ tokens, SortPlan p) {
  __shared__ int counts[kDigits];
  mtb_wait_prior();
  mtb_launch_dependents();
  const int digits = 1 << p.bits, lo = blockIdx.x << p.share_bits, stop = lo + (1 << p.share_bits), hi = stop < p.count ? stop : p.count;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.runs = 0;
  if (threadIdx.x < digits) counts[threadIdx.x] = 0;
  __syncthreads();
  for (int i0 = lo + threadIdx.x; i0 < hi; i0 += kSortThreads * kSortAhead) {
    int k[kSortAhead];
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u)
      if (i0 + u * kSortThreads < hi) k[u] = key_of<T>(tokens, i0 + u * kSortThreads, p);
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u)
      if (i0 + u * kSortThreads < hi) atomicAdd(counts + (k[u] & (digits - 1)), 1);
  }
  __syncthreads();
  if (threadIdx.x < digits) {
    int* row = p.table + blockIdx.x * digits + threadIdx.x;
    *row = counts[threadIdx.x];
    for (int pass = 1; pass < p.passes; ++pass) row[pass * p.ctas * digits] = 0;
  }
}

template <class T>
__global__ void __launch_bounds__(kSortThreads) embedding_place_kernel(const void* __restrict__ tokens, SortPlan p, int pass) {
  __shared__ SortShared sh;
  extern __shared__ int2 staged[];
  mtb_wait_prior();
  mtb_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << p.bits, shift = pass * p.bits;
  const int first = blockIdx.x << p.share_bits, each = 1 << p.share_bits >> 4;  // a warp's stretch
  static_assert(kSortWarps == 16, "a stretch is a sixteenth of a share");
  auto bounded = [&](int i) { return i < p.count ? i : p.count; };
  const int lo = bounded(first + warp * each), hi = bounded(first + (warp + 1) * each), share = bounded(first + (1 << p.share_bits)) - first;
  const bool held = each <= 32 * kSortAhead, stage = 1 << p.share_bits <= kStaged;  // of all CTAs, whose shared memory the launch sized
  for (int i = threadIdx.x; i < kSortWarps * kDigits / 4; i += kSortThreads) ((int4*)sh.counters)[i] = make_int4(0, 0, 0, 0);
  __syncthreads();
  int2 entry[kSortAhead];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      const int i = i0 + 32 * u + lane;
      if (i < hi) entry[u] = pass ? p.from[i] : make_int2(key_of<T>(tokens, i, p), i);
    }
  };
  for (int i0 = lo; i0 < hi; i0 += 32 * kSortAhead) {
    load(i0);
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u)
      if (i0 + 32 * u + lane < hi) atomicAdd(&sh.counters[warp][entry[u].x >> shift & (digits - 1)], 1);
  }
  // The shares before, and all of them: four digits a thread, an eighth of the shares each.  A CTA begins at its own, since all of them at
  // the same lines wait for one another.
  constexpr int kParts = kSortThreads * 4 / kDigits;
  static_assert(2 * kParts == kSortWarps, "the parts' sums take the place of the lanes' words");
  int(*of_part)[kDigits] = (int(*)[kDigits])sh.lanes;
  const int quad = threadIdx.x % (kDigits / 4), part = threadIdx.x / (kDigits / 4);
  const int* table = p.table + pass * p.ctas * digits;
  if (quad * 4 < digits) {
    int4 before = make_int4(0, 0, 0, 0), all = before;
    for (int i0 = part; i0 < p.ctas; i0 += kParts * 8) {
      int4 n[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        int c = i0 + kParts * u + blockIdx.x;
        if (c >= p.ctas) c -= p.ctas;
        n[u] = i0 + kParts * u < p.ctas ? *(const int4*)(table + c * digits + 4 * quad) : make_int4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        all.x += n[u].x; all.y += n[u].y; all.z += n[u].z; all.w += n[u].w;
        if (i0 + kParts * u + blockIdx.x >= p.ctas) { before.x += n[u].x; before.y += n[u].y; before.z += n[u].z; before.w += n[u].w; }
      }
    }
    *(int4*)(of_part[part] + 4 * quad) = before;
    *(int4*)(of_part[kParts + part] + 4 * quad) = all;
  }
  __syncthreads();
  int total = sum_warps(sh, digits), begin = total, before = 0, all = 0;
  if (threadIdx.x < digits) {
#pragma unroll
    for (int u = 0; u < kParts; ++u) {
      before += of_part[u][threadIdx.x];
      all += of_part[kParts + u][threadIdx.x];
    }
  }
  scan_digits(all, begin, sh);  // the parts' sums are read
  for (int i = threadIdx.x; i < kSortWarps * kDigits / 4; i += kSortThreads) ((int4*)sh.lanes)[i] = make_int4(0, 0, 0, 0);
  if (threadIdx.x < digits) {
    sh.local[threadIdx.x] = begin;
    sh.shift_to[threadIdx.x] = all + before - begin;
  }
  __syncthreads();
  int* next = p.table + (pass + 1) * p.ctas * digits;
  auto put = [&](int2 e, int place) {
    const int at = place + sh.shift_to[e.x >> shift & (digits - 1)];
    p.to[at] = e;
    if (pass + 1 < p.passes) atomicAdd(next + (at >> p.share_bits) * digits + (e.x >> (shift + p.bits) & (digits - 1)), 1);
  };
  for (int i0 = lo; i0 < hi; i0 += 32 * kSortAhead) {
    if (!held) load(i0);
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      if (i0 + 32 * u < hi) {
        const bool in = i0 + 32 * u + lane < hi;
        const int place = place_of(in, entry[u].x >> shift & (digits - 1), sh.counters[warp], sh.lanes[warp], sh.local);
        if (in) {
          if (stage) staged[place] = entry[u];
          else put(entry[u], place);
        }
      }
    }
  }
  if (!stage) return;
  __syncthreads();
  for (int i = threadIdx.x; i < share; i += kSortThreads) put(staged[i], i);
}

// ---------------------------------------------------------------- gradient: add up

// Rows of the table that no token names are cleared by CTAs of their own, 32 rows a warp.  (Clearing the whole table while the tokens are put in order costs more:
// 102 MB of it take longer than that, and half of them are written again: 131072 tokens, 50000 x 512: 115 us, 104 this way.)
//
// The ordered tokens are cut into tiles of `tile`.  A run of equal tokens of up to kRun is added up by the tile it begins in, past the tile's end if need be,
// and goes to the table; a longer one is added up piece by piece, each tile its own, and the pieces are added by the kernel behind, in
// their order.  Frequent tokens thus keep no tile waiting, and the rest has no second step.
//
// Bound by memory: 131072 tokens of 512 values to 50000 rows 64 us, 5.8 TB/s of the 371 MB of gradients read and rows written; 90 us with the ordering (19) and the
// joining (12, the pieces of the most frequent token one after another).  Sixteen rows ahead 94 us in all, runs of 16 96; 4096 tokens are 2 us faster
// with runs of 16.
constexpr int kRun = 32, kMaxTile = kRun, kSumAhead = 8;  // a longer tile could hold a whole long run

struct SumPlan {
  const int2* entries;
  int count, rows, width, tile, lanes, groups;  // threads to a tile, tiles to a CTA
  int clearing;                                 // CTAs that clear rows, in front of the others
  float scale;
  const float* dy;
  float* dtable;
  float* pieces;  // [tiles][2][width]: of the long run that begins before the tile, of the one that begins in it
  int* runs;              // how many long runs there are,
  int2* run_starts;       // of each, the tile that it begins in and its token
  int* run_ends;          // [rows]: the tile that a long run of this token ends in
};

// Whether an ordered entry names `row`.
__device__ __forceinline__ bool is_named(const SumPlan& p, int row) {
  int lo = 0, hi = p.count;  // the first entry not below `row` is in [lo, hi]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.entries[mid].x < row) lo = mid + 1; else hi = mid;
  }
  return lo < p.count && p.entries[lo].x == row;
}

template <int V>
__device__ __forceinline__ void clear_rows(const SumPlan& p, int block) {
  const int lane = threadIdx.x & 31, warps = blockDim.x / 32, row = (block * warps + threadIdx.x / 32) * 32 + lane;
  VecF<V> zero;
#pragma unroll
  for (int i = 0; i < V; ++i) zero.v[i] = 0.f;
  unsigned bare = __ballot_sync(0xffffffffu, row < p.rows && !is_named(p, row));
  for (; bare; bare &= bare - 1) {
    float* to = p.dtable + (long long)(row - lane + __ffs(bare) - 1) * p.width;
    for (int col = lane * V; col < p.width; col += 32 * V) vstore<V>(to + col, zero);
  }
}

// A load that L2 need not keep.
template <int V>
__device__ __forceinline__ VecF<V> vload_once(const float* p) {
  VecF<V> r;
  if (V == 4) {
    const float4 t = __ldcs((const float4*)p);
    r.v[0] = t.x; r.v[1 % V] = t.y; r.v[2 % V] = t.z; r.v[3 % V] = t.w;
  } else {
    r.v[0] = __ldcs(p);
  }
  return r;
}

template <int V>
__global__ void __launch_bounds__(128) embedding_sum_kernel(SumPlan p) {
  // keys from kRun before a tile to kRun behind it; one more on either side tells where a run ends
  constexpr int kSpan = kMaxTile + 2 * kRun + 2;
  extern __shared__ int shared[];
  mtb_wait_prior();
  mtb_launch_dependents();
  if (blockIdx.x < p.clearing) {
    if (blockIdx.y == 0) clear_rows<V>(p, blockIdx.x);
    return;
  }
  const int group = threadIdx.x / p.lanes, lane = threadIdx.x - group * p.lanes;
  const int t0 = ((blockIdx.x - p.clearing) * p.groups + group) * p.tile;
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
      if (e + u < to) v[u] = vload_once<V>(dy + (long long)places[e + u] * p.width);
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

constexpr int kJoinThreads = 256, kJoinAhead = 4;  // eight ahead spill: 102 us of the whole gradient above instead of 91; 512 threads 95

// One CTA a long run and 32 lanes' columns: its warps add up a part of the pieces each, and those sums are added in their order.
template <int V>
__global__ void __launch_bounds__(kJoinThreads, 5) embedding_join_kernel(SumPlan p) {
  mtb_wait_prior();
  mtb_launch_dependents();
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
  int passes, bits, ctas, share_bits, tile, tiles, lanes, groups, columns;
  long long bytes;
};

// Scratch: two sets of entries, the digits' counts, the long runs' starts and ends, the pieces.
GradPlan plan_gradient(long long count, int rows, int width, bool four) {
  GradPlan g{};
  int bits = 2;  // digits are read four at a time
  while ((1LL << bits) <= rows) ++bits;  // the largest key is `rows`
  g.passes = (bits + kDigitBits - 1) / kDigitBits;
  g.bits = (bits + g.passes - 1) / g.passes;
  g.ctas = g.share_bits = 0;
  if (count > kOneCta) {
    for (g.share_bits = 9; (count >> g.share_bits) >= mtb_sm_count();) ++g.share_bits;
    g.ctas = (int)((count + (1LL << g.share_bits) - 1) >> g.share_bits);
  }
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
  g.bytes = 16 * count + 4LL * g.passes * g.ctas * kDigits + 4LL * rows + 8LL * g.tiles + 512 + 8LL * g.tiles * width;
  return g;
}

template <class T>
int sort_tokens(const void* tokens, SortPlan p, int2* entries, cudaStream_t st) {
  if (p.ctas == 0) {
    static unsigned long long opted;
    if (int rc = mtb_opt_in_smem((const void*)embedding_order_kernel<T>, kOneCta * 8, &opted)) return rc;
    p.to = entries;
    MTB_LAUNCH(embedding_order_kernel<T>, 1, kSortThreads, kOneCta * 8, st, tokens, p);
    return MTB_OK;
  }
  static unsigned long long opted;
  if (int rc = mtb_opt_in_smem((const void*)embedding_place_kernel<T>, kStaged * 8, &opted)) return rc;
  MTB_LAUNCH(embedding_count_kernel<T>, p.ctas, kSortThreads, 0, st, tokens, p);
  const int smem = (1 << p.share_bits) <= kStaged ? 8 << p.share_bits : 0;
  for (int pass = 0; pass < p.passes; ++pass) {  // the last one's result is the first set
    const bool second = (p.passes - 1 - pass) & 1;
    p.to = entries + (second ? p.count : 0);
    p.from = entries + (second ? 0 : p.count);
    MTB_LAUNCH(embedding_place_kernel<T>, p.ctas, kSortThreads, smem, st, tokens, p, pass);
  }
  return MTB_OK;
}

template <int V>
int add_up(const SumPlan& p, const GradPlan& g, cudaStream_t st) {
  const int smem = g.groups * 2 * (kMaxTile + 2 * kRun + 2) * 4;
  MTB_LAUNCH(embedding_sum_kernel<V>, dim3(p.clearing + mtb_div_up(g.tiles, g.groups), g.columns), g.lanes * g.groups, smem, st, p);
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
  MTB_REQUIRE(mtb_aligned16(workspace), "embedding_backward: the workspace does not begin at a 16-byte boundary");
  cudaStream_t st = (cudaStream_t)stream;
  if (count == 0) {
    MTB_CUDA(cudaMemsetAsync(dtable, 0, 4LL * rows * width, st));
    return MTB_OK;
  }
  const bool four = width % 4 == 0 && mtb_aligned16(dy) && mtb_aligned16(dtable);
  const GradPlan g = plan_gradient(count, rows, width, four);
  MTB_REQUIRE(g.columns < 65536, "embedding_backward: rows of %d values", width);
  int* table = (int*)workspace;  // read four at a time, like the pieces
  float* pieces = (float*)(table + g.passes * g.ctas * (1 << g.bits));
  int2* entries = (int2*)(pieces + 2LL * g.tiles * width);
  int2* run_starts = entries + 2 * count;
  int *run_ends = (int*)(run_starts + g.tiles), *runs = run_ends + rows;
  const SortPlan s{(int)count, rows, g.passes, g.bits, g.share_bits, g.ctas, padding, nullptr, nullptr, table, runs};
  if (int rc = kind == 0 ? sort_tokens<int>(tokens, s, entries, st) : sort_tokens<long long>(tokens, s, entries, st)) return rc;
  const SumPlan p{entries, (int)count, rows, width, g.tile, g.lanes, g.groups, mtb_div_up(rows, g.lanes * g.groups), (float)scale, dy, dtable, pieces, runs, run_starts, run_ends};
  return four ? add_up<4>(p, g, st) : add_up<1>(p, g, st);
}
