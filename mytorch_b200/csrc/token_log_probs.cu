// Log probabilities of given tokens, the entropy and the most likely alternatives of every row of logits z [n, v], and their gradient.
//   m = max z,  S = sum exp(z - m),  T = sum exp(z - m) (z - m),  log p_j = z_j - m - log S,  H = log S - T / S  (two terms of one sign: nothing cancels).
//   dz_j = -p_j (g + sum of the alternatives' g) - g_H p_j (log p_j + H), and g, or an alternative's g, added at its token.
// A logit of -inf has probability 0 and adds nothing to the entropy or its gradient; a row of nothing else, or with a NaN or +inf, is NaN.
// Alternatives are in the order of their logits, NaN before everything, equal ones by place, which one whole number holds (`key_of`).
//
// Bound by memory: forward reads a row once, backward reads and writes it once.  4096 rows of 50000, logits out of HBM: forward 130 us without alternatives, 6.3 TB/s, 150 with 8,
// 5.5; backward 255 us, 6.4 TB/s.  Each thread keeps a running maximum and both sums of its share of the row, four loads of 16 bytes on their way at a time.  What counts is
// how many warps are under way (40 an SM): a second set of loads ahead of use costs a quarter of them, 146 us, reloading each register as soon as it is used 162, copies
// through shared memory two batches ahead and across rows 149, CTAs whose warps go on to the next row while one of them looks for the last one's alternatives 146, with 8 of them 174.
//
// Alternatives.  A thread also keeps the maxima of the four groups that its quads fall into, nothing else.  When the row is through, the top-th largest of the maxima of 64 parts
// of it is a bound that `top` values reach, and only groups whose maximum reaches it can hold an alternative: little more than `top` of the row's 1024 (512, 128) groups, whose values
// are read again, and what reaches the bound is put in order by counting.  The bound takes a third of the 20 us that 8 alternatives cost, the second reading the rest.  An
// exact bound by sorting all groups' maxima: 180 us; the r-th largest of each warp's: 163; one group a thread, which reads four times as much again out of HBM, as the
// rows under way are more than the L2 holds: 170; candidates picked while the row comes by would cost every batch of values an insertion at first.  Where very many
// values equal the bound, as where a mask leaves fewer than `top`, those above it are taken and then the first of the row that equal it; rows with a NaN, and more candidates
// than there is room for, take `top` passes that find one each.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMostTop = 32;
constexpr int kMostCtas = 8;  // of a row
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -200.f;  // exp of it is 0 in 32 bits
constexpr float kLowest = -3.402823466e38f;
typedef unsigned long long Key;

__device__ __forceinline__ unsigned ordered(float z) {
  const unsigned b = __float_as_uint(z + 0.f);  // -0 is 0
  return z != z ? 0xFFFFFFFFu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Larger: a larger logit, or of equal ones the earlier.  No key is 0.
__device__ __forceinline__ Key key_of(float z, int place) { return (Key)ordered(z) << 32 | (0xFFFFFFFFu - (unsigned)place); }
__device__ __forceinline__ int place_of(Key k) { return (int)(0xFFFFFFFFu - (unsigned)k); }
__device__ __forceinline__ float value_of(Key k) {
  const unsigned o = (unsigned)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_of(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// a - b, which is at most 0, and finite where it counts: beside -inf and the type's lowest value exp of it is 0 and its product with that is, too.
__device__ __forceinline__ float gap(float a, float b) { return fmaxf(a - b, kFar); }

// The sums of some values, relative to `ref`, as a value and what its rounding left (a row may be long).
struct Sums {
  float most = -INFINITY, ref = kLowest, s = 0, s_low = 0, t = 0, t_low = 0;  // most: NaN where there is one

  static __device__ __forceinline__ void add(float& hi, float& low, float x) {
    x += low;
    const float y = hi + x;
    low = x - (y - hi);
    hi = y;
  }
  __device__ __forceinline__ void raise(float to) {  // a new `most`
    most = to;
    const float r = fmaxf(to, kLowest), d = gap(ref, r), f = exp2_of(d * kLog2e);
    t = f * (t + s * d);
    t_low = f * (t_low + s_low * d);
    s *= f;
    s_low *= f;
    ref = r;
  }
  // Over the warp, in all its lanes.  RUN: to `runs` the largest value of each run of so many lanes.
  // LANES: over each of so many, which hold the same as the others.
  template <int RUN = 32, int LANES = 32>
  __device__ __forceinline__ void reduce(float* runs = nullptr) {
    float to = most;
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) {
      if (RUN < 32 && o == RUN && (threadIdx.x & (RUN - 1)) == 0) runs[(threadIdx.x & 31) / RUN] = to;
      to = max_nan(to, __shfl_xor_sync(0xFFFFFFFFu, to, o));
    }
    raise(to);
    s += s_low;
    t += t_low;
    s_low = t_low = 0;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
      t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    }
  }
};

// A row in quads of four values, the first of which begins at a 16-byte boundary at or before the row: `lead` values lie before it.
struct Row {
  const float* z;  // of the first quad
  int lead, v, quads;

  __device__ __forceinline__ Row(const float* row, int v) : lead((int)(reinterpret_cast<uintptr_t>(row) >> 2 & 3)), v(v) {
    z = row - lead;
    quads = (int)(((unsigned)v + lead + 3) / 4);
  }
  __device__ __forceinline__ int place(int q) const { return 4 * q - lead; }
  __device__ __forceinline__ float4 quad(int q, int end) const {  // -inf where there is nothing, and from quad `end` on
    const int i = place(q);
    if (q < end && i >= 0 && i + 3 < v) return ld4(z + 4LL * q);
    float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (q < end) {
      const float* p = z + 4LL * q;
      if (i >= 0 && i < v) f.x = p[0];
      if (i + 1 >= 0 && i + 1 < v) f.y = p[1];
      if (i + 2 >= 0 && i + 2 < v) f.z = p[2];
      if (i + 3 < v) f.w = p[3];
    }
    return f;
  }
};

// Over the warp, the largest first.
template <class T>
__device__ __forceinline__ T sorted(T k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int j = size / 2; j > 0; j /= 2) {
      const T o = __shfl_xor_sync(0xFFFFFFFFu, k, j);
      if (((lane & j) == 0) == ((lane & size) == 0 || size == 32) ? o > k : o < k) k = o;
    }
  return k;
}
// The 32 largest of two sorted lists, `other` backwards.
template <class T>
__device__ __forceinline__ T merged(T k, T other, int lane) {
  if (other > k) k = other;
#pragma unroll
  for (int j = 16; j > 0; j /= 2) {
    const T o = __shfl_xor_sync(0xFFFFFFFFu, k, j);
    if ((lane & j) == 0 ? o > k : o < k) k = o;
  }
  return k;
}
template <class T>
__device__ __forceinline__ T merged_across(T k, T other, int lane) { return merged(k, __shfl_xor_sync(0xFFFFFFFFu, other, 31), lane); }

// What W warps that share a row exchange.
template <int W>
struct Shared {
  static constexpr int kCandidates = W == 1 ? 256 : 512, kGroups = W == 1 ? 128 : 256;
  alignas(16) float part[W][4];
  float runs[64];
  Key candidate[kCandidates], list[W];
  int group[kGroups], groups, candidates, taken;  // taken: a word of its own, `candidates` may still be read by a warp that comes late
};
constexpr int kSplit = 4;  // a thread's quads fall into groups by their number modulo this
template <int W>
__device__ __forceinline__ void meet() {
  if (W == 1) __syncwarp(); else __syncthreads();
}

// The keys of the groups' values that reach the bound (`above`: that are above it) to the candidates, which are counted beyond what there is room for.
template <int W>
__device__ __forceinline__ void take(const Row& row, int begin, int end, Shared<W>& shared, int groups, int id, float bound, bool above = false) {
  constexpr int T = 32 * W, kStride = kSplit * T;
  if (groups <= 0) return;
  const int each = (end - begin + kStride - 1) / kStride;  // quads of a group, rounded up
  int g = id / each, k = id - g * each;
  const int step_g = T / each, step_k = T - step_g * each;
  while (g < groups) {
    const int q = begin + shared.group[g] + k * kStride;
    const float4 f = row.quad(q, end);
    const int i = row.place(q);
    const float x[4] = {f.x, f.y, f.z, f.w};
    if (q < end) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((above ? x[j] > bound : x[j] >= bound) && i + j >= 0 && i + j < row.v) {
          const int at = atomicAdd(&shared.candidates, 1);
          if (at < Shared<W>::kCandidates) shared.candidate[at] = key_of(x[j], i + j);
        }
    }
    g += step_g;
    k += step_k;
    if (k >= each) { k -= each; ++g; }
  }
}
// The r-th largest of the values that the lanes of a warp hold, two each, the larger first, in all lanes.
__device__ __forceinline__ float largest_but(int r, const float (&m)[2]) {
  unsigned o[2] = {ordered(m[0]), ordered(m[1])}, most = 0;
  for (int k = 0; k < r; ++k) {
    most = __reduce_max_sync(0xFFFFFFFFu, o[0]);
    if ((threadIdx.x & 31) == __ffs(__ballot_sync(0xFFFFFFFFu, o[0] == most)) - 1) {
      o[0] = o[1];
      o[1] = 0;
    }
  }
  return value_of((Key)most << 32);
}
__device__ __forceinline__ void exchange(float& a, float& b) {
  const float x = fmaxf(a, b);
  b = fminf(a, b);
  a = x;
}

// By a warp: the first places of a value to the candidates, up to `top` of these; their number.
template <int W>
__device__ __forceinline__ int take_equal(const Row& row, int begin, int end, Shared<W>& shared, int lane, float value, int count, int top) {
  for (int from = begin; from < end && count < top; from += 32) {
    const int q = from + lane, i = row.place(q);
    const float4 f = row.quad(q, end);
    const float x[4] = {f.x, f.y, f.z, f.w};
    int mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) mine += q < end && x[j] == value && i + j >= 0 && i + j < row.v;
    int at = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int other = __shfl_up_sync(0xFFFFFFFFu, at, o);
      if (lane >= o) at += other;
    }
    const int all = __shfl_sync(0xFFFFFFFFu, at, 31);
    at += count - mine;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (q < end && x[j] == value && i + j >= 0 && i + j < row.v) {
        if (at < top) shared.candidate[at] = key_of(x[j], i + j);
        ++at;
      }
    count = min(top, count + all);
    __syncwarp();
  }
  return count;
}

// Of the quads [begin, end) of a row: the sums, in all threads, and in `out` the `top` largest keys in their order, 0 where there are fewer.  given: loads
// what the caller wants besides, called once while the row comes.
template <int W, class F>
__device__ __forceinline__ Sums look(const Row& row, int begin, int end, int top, Shared<W>& shared, Key* out, F given) {
  constexpr int T = 32 * W;
  const int lane = threadIdx.x & 31, warp = W == 1 ? 0 : threadIdx.x >> 5, id = W == 1 ? lane : threadIdx.x;
  Sums sums;
  constexpr int G = kSplit;
  float most[G];  // of the thread's groups
#pragma unroll
  for (int u = 0; u < G; ++u) most[u] = -INFINITY;
  for (int q = begin; q < end; q += 4 * T) {
    float4 f[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) f[u] = row.quad(q + id + u * T, end);
    if (q == begin) given();
#pragma unroll
    for (int u = 0; u < 4; ++u) most[u % G] = max_nan(most[u % G], max_nan(max_nan(f[u].x, f[u].y), max_nan(f[u].z, f[u].w)));
    float to = most[0];
#pragma unroll
    for (int u = 1; u < G; ++u) to = max_nan(to, most[u]);
    if (to != sums.most) sums.raise(to);
    float s[4], t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float x[4] = {f[u].x, f[u].y, f[u].z, f[u].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = gap(x[j], sums.ref), e = exp2_of(d * kLog2e);
        s[j] = u ? s[j] + e : e;
        t[j] = u ? fmaf(e, d, t[j]) : e * d;
      }
    }
    Sums::add(sums.s, sums.s_low, (s[0] + s[1]) + (s[2] + s[3]));
    Sums::add(sums.t, sums.t_low, (t[0] + t[1]) + (t[2] + t[3]));
  }
  // a bound that `top` values reach: of 64 parts of the row, the top-th largest of their maxima
  constexpr int kRun = W == 1 ? 32 : W / 2;  // threads of a part
  float m[2] = {fmaxf(most[0], most[1]), fmaxf(most[2], most[3])};
  sums.reduce<kRun>(&shared.runs[warp * (32 / kRun)]);
  if (W > 1 && lane == 0) { shared.part[warp][0] = sums.most; shared.part[warp][1] = sums.s; shared.part[warp][2] = sums.t; }
  if (id == 0) shared.groups = shared.candidates = 0;
  meet<W>();
  if (W > 1) {
    const float4 p = *(const float4*)shared.part[lane % W];
    if (top) {
      m[0] = shared.runs[lane];
      m[1] = shared.runs[32 + lane];
    }
    sums = Sums();
    sums.most = p.x;
    sums.ref = fmaxf(p.x, kLowest);
    sums.s = p.y;
    sums.t = p.z;
    sums.reduce<32, W>();
  }
  float bound = sums.most;
  if (top > 1) {
    exchange(m[0], m[1]);
    bound = largest_but(top, m);
  }
  if (!top) return sums;
  bool slow = sums.most != sums.most;
  if (!slow) {
#pragma unroll
    for (int u = 0; u < G; ++u)
      if (most[u] >= bound) {  // some more than `top`, many where some are equal
        const int at = atomicAdd(&shared.groups, 1);
        if (at < Shared<W>::kGroups) shared.group[at] = id + u * T;
      }
    meet<W>();
    const int groups = shared.groups;
    const bool equal = groups > Shared<W>::kGroups;
    take(row, begin, end, shared, equal ? 0 : groups, id, bound);
    meet<W>();
    int count = shared.candidates;
    if (equal || count > Shared<W>::kCandidates) {
      // many values equal the bound: those above it, and of those that equal it the first of the row
      meet<W>();
      if (id == 0) shared.groups = shared.candidates = 0;
      meet<W>();
#pragma unroll
      for (int u = 0; u < G; ++u)
        if (most[u] > bound) {
          const int at = atomicAdd(&shared.groups, 1);
          if (at < Shared<W>::kGroups) shared.group[at] = id + u * T;
        }
      meet<W>();
      count = shared.groups;
      if (count <= Shared<W>::kGroups) {
        take(row, begin, end, shared, count, id, bound, true);
        meet<W>();
        count = shared.candidates;
      } else {
        count = Shared<W>::kCandidates + 1;
      }
      if (count < top) {
        if (warp == 0) count = take_equal(row, begin, end, shared, lane, bound, count, top);
        if (W > 1) {
          if (id == 0) shared.taken = count;
          __syncthreads();
          count = shared.taken;
        }
      }
    }
    slow = count > Shared<W>::kCandidates;
    if (!slow && count <= T) {
      if (id < count || id < top) {
        const Key best = id < count ? shared.candidate[id] : 0;
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < count; ++j) place += shared.candidate[j] > best;
        if (id >= count) out[id] = 0;
        else if (place < top) out[place] = best;
      }
    } else if (!slow) {
      if (warp == 0) {
        Key best = sorted(shared.candidate[lane], lane);
        for (int from = 32; from < count; from += 32) best = merged_across(best, sorted(from + lane < count ? shared.candidate[from + lane] : 0, lane), lane);
        if (lane < top) out[lane] = best;
      }
    }
  }
  if (slow) {
    Key below = ~0ull;
    for (int k = 0; k < top; ++k) {
      Key best = 0;
      for (int q = begin + id; q < end; q += T) {
        const float4 f = row.quad(q, end);
        const int i = row.place(q);
        const float x[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const Key one = key_of(x[j], i + j);
          if (one < below && one > best && i + j >= 0 && i + j < row.v) best = one;
        }
      }
      for (int o = 16; o > 0; o >>= 1) {
        const Key other = __shfl_xor_sync(0xFFFFFFFFu, best, o);
        if (other > best) best = other;
      }
      if (W > 1) {
        __syncthreads();
        if (lane == 0) shared.list[warp] = best;
        __syncthreads();
        for (int w = 0; w < W; ++w)
          if (shared.list[w] > best) best = shared.list[w];
      }
      if (id == 0) out[k] = best;
      below = best;
    }
  }
  meet<W>();
  return sums;
}

struct Forward {
  long long n;
  int v, wide, ignores, top;
  long long ignore_index;
  const float* logits;
  const void* tokens;
  float *log_probs, *entropy, *stats, *top_log_probs;
  long long* top_tokens;
};

__device__ __forceinline__ long long token_at(const void* tokens, int wide, long long row) { return wide ? ((const long long*)tokens)[row] : ((const int*)tokens)[row]; }

// The row's token and its logit, which come while the row does; in thread 0 of those that share the row.
struct Given {
  const Forward& a;
  long long row;
  int id;
  long long token;
  float z = 0;

  __device__ __forceinline__ Given(const Forward& a, long long row, int id) : a(a), row(row), id(id), token(id == 0 ? token_at(a.tokens, a.wide, row) : -1) {}
  __device__ __forceinline__ void operator()() { if (token >= 0 && token < a.v) z = a.logits[row * a.v + token]; }
};

// By thread `id` of those that share the row.
__device__ __forceinline__ void leave(const Forward& a, long long row, int id, const Given& given, const Sums& sums, const Key* found) {
  const bool none = !(sums.most >= kLowest && sums.most < INFINITY);  // a NaN, +inf, or nothing but -inf
  const float s = none ? NAN : sums.s + sums.s_low, log_s = logf(s);
  if (id == 0) {
    a.log_probs[row] = a.ignores && given.token == a.ignore_index ? 0.f : given.token < 0 || given.token >= a.v ? NAN : given.z - sums.most - log_s;
    const float h = log_s - (sums.t + sums.t_low) / s;
    a.entropy[row] = h;
    if (a.stats) {
      a.stats[3 * row] = sums.most;
      a.stats[3 * row + 1] = s;
      a.stats[3 * row + 2] = h;
    }
  }
  if (id < a.top) {
    a.top_tokens[row * a.top + id] = place_of(found[id]);
    a.top_log_probs[row * a.top + id] = value_of(found[id]) - sums.most - log_s;
  }
}

// A row by W warps: 1 (eight rows a CTA) or a whole CTA.
template <int W>
__global__ void __launch_bounds__(W == 1 ? kThreads : 32 * W) log_probs_kernel(const __grid_constant__ Forward a) {
  constexpr int kRows = W == 1 ? kWarps : 1;
  __shared__ Shared<W> shared[kRows];
  __shared__ Key found[kRows][kMostTop];
  mtb_launch_dependents();
  mtb_wait_prior();
  const int part = W == 1 ? threadIdx.x >> 5 : 0;
  const long long index = W == 1 ? blockIdx.x * (long long)kWarps + part : blockIdx.x;
  if (index >= a.n) return;
  const Row row(a.logits + index * a.v, a.v);
  const int id = W == 1 ? threadIdx.x & 31 : threadIdx.x;
  Given given(a, index, id);
  const Sums sums = look<W>(row, 0, row.quads, a.top, shared[part], found[part], [&] { given(); });
  leave(a, index, id, given, sums, found[part]);
}

// A row by a cluster of CTAs, each of which finds the alternatives of its part; the first puts them together.  Its shared memory is there for the others once it has started: each
// arrives first of all and waits for the others before it writes to it.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

__global__ void __launch_bounds__(kThreads) log_probs_cluster_kernel(const __grid_constant__ Forward a) {
  __shared__ Shared<kWarps> shared;
  __shared__ Key found[kMostTop], all[kMostCtas][kMostTop];
  __shared__ float parts[kMostCtas][3];
  mtb_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  cluster_arrive();
  mtb_wait_prior();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const long long index = blockIdx.x / ctas;
  const Row row(a.logits + index * a.v, a.v);
  const int each = (row.quads + ctas - 1) / ctas, begin = rank * each < row.quads ? rank * each : row.quads, end = begin + each < row.quads ? begin + each : row.quads;
  Given given(a, index, rank == 0 ? threadIdx.x : 1);
  const Sums mine = look<kWarps>(row, begin, end, a.top, shared, found, [&] { given(); });
  cluster_wait();
  if (a.top && threadIdx.x < kMostTop) cluster.map_shared_rank(&all[0][0], 0)[rank * kMostTop + threadIdx.x] = threadIdx.x < a.top ? found[threadIdx.x] : 0;
  if (threadIdx.x == 0) {
    float* to = cluster.map_shared_rank(&parts[0][0], 0) + 3 * rank;
    to[0] = mine.most;
    to[1] = mine.s + mine.s_low;
    to[2] = mine.t + mine.t_low;
  }
  cluster.sync();
  if (rank != 0) return;
  Sums sums;
  const int r = (threadIdx.x & 31) < ctas ? threadIdx.x & 31 : 0;
  sums.most = parts[r][0];
  sums.ref = fmaxf(sums.most, kLowest);
  sums.s = (threadIdx.x & 31) < ctas ? parts[r][1] : 0.f;
  sums.t = (threadIdx.x & 31) < ctas ? parts[r][2] : 0.f;
  sums.reduce();
  if (a.top && threadIdx.x < 32) {  // sorted lists
    Key best = all[0][threadIdx.x];
    for (int r = 1; r < ctas; ++r) best = merged(best, all[r][31 - threadIdx.x], threadIdx.x);
    found[threadIdx.x] = best;
    __syncwarp();
  }
  leave(a, index, threadIdx.x, given, sums, found);
}

struct Backward {
  long long n;
  int v, wide, ignores, top;
  long long ignore_index;
  const float* logits;
  const void* tokens;
  const float *dlog_probs, *dentropy, *dtop, *stats;
  const long long* top_tokens;
  float* dlogits;
  int parts;  // CTAs of a row
};

// What a row's gradient is made with.
struct RowGradient {
  float m, per_s, log_s, h, g, gh, all;

  // Where no gradient reaches the row: zero for a value of 0, which stands for each of the row's, as these may make everything NaN.
  __device__ __forceinline__ void clear() { m = per_s = log_s = h = 0; }
  // exp here by the function, whose error does not grow with its argument: an element moves 8 bytes, there is time.
  __device__ __forceinline__ float at(float z) const {
    const float d = z - m, p = expf(d) * per_s;
    return -p * (all + gh * (fmaxf(d, kFar) - log_s + h));
  }
};

// A row by W warps: 1, or `parts` CTAs, U vectors a thread.
template <int W, int U>
__global__ void __launch_bounds__(kThreads) log_probs_backward_kernel(const __grid_constant__ Backward a) {
  constexpr int T = 32 * W;
  mtb_launch_dependents();
  mtb_wait_prior();
  const int lane = threadIdx.x & 31, id = W == 1 ? lane : threadIdx.x;
  const long long index = W == 1 ? blockIdx.x * (long long)kWarps + (threadIdx.x >> 5) : blockIdx.x / a.parts;
  if (index >= a.n) return;
  const Row row(a.logits + index * a.v, a.v);
  float* to = a.dlogits + index * a.v - row.lead;
  const bool together = ((reinterpret_cast<uintptr_t>(to) ^ reinterpret_cast<uintptr_t>(row.z)) & 15u) == 0;
  const int begin = W == 1 ? 0 : (int)(blockIdx.x % a.parts) * (U * kThreads), end = W == 1 ? row.quads : min(begin + U * kThreads, row.quads);
  float4 f[U];
#pragma unroll
  for (int u = 0; u < U; ++u) f[u] = row.quad(begin + id + u * T, end);
  // every warp for itself: the row's numbers, an alternative a lane
  const long long token = token_at(a.tokens, a.wide, index);
  RowGradient r;
  r.m = a.stats[3 * index];
  const float s = a.stats[3 * index + 1];
  r.h = a.stats[3 * index + 2];
  r.per_s = 1.f / s;
  r.log_s = logf(s);
  r.g = !a.dlog_probs || (a.ignores && token == a.ignore_index) || token < 0 || token >= a.v ? 0.f : a.dlog_probs[index];
  r.gh = a.dentropy ? a.dentropy[index] : 0.f;
  const bool mine = a.dtop && lane < a.top;
  const float extra = mine ? a.dtop[index * a.top + lane] : 0.f;
  const long long other = mine ? a.top_tokens[index * a.top + lane] : -1;
  r.all = extra;
  for (int o = 16; o > 0; o >>= 1) r.all += __shfl_xor_sync(0xFFFFFFFFu, r.all, o);
  r.all += r.g;
  const bool none = !__any_sync(0xFFFFFFFFu, extra != 0.f) && r.g == 0.f && r.gh == 0.f;
  if (none) r.clear();
  for (int q = begin; q < end; q += U * T) {
    if (W == 1 && q > begin) {
#pragma unroll
      for (int u = 0; u < U; ++u) f[u] = row.quad(q + id + u * T, end);
    }
    if (none) {
#pragma unroll
      for (int u = 0; u < U; ++u) f[u] = make_float4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = q + id + u * T, i = row.place(at);
      if (at >= end) continue;
      const float4 d = make_float4(r.at(f[u].x), r.at(f[u].y), r.at(f[u].z), r.at(f[u].w));
      if (together && i >= 0 && i + 3 < a.v) {
        st4(to + 4LL * at, d);
      } else {
        float* p = to + 4LL * at;
        if (i >= 0) p[0] = d.x;
        if (i + 1 >= 0 && i + 1 < a.v) p[1] = d.y;
        if (i + 2 >= 0 && i + 2 < a.v) p[2] = d.z;
        if (i + 3 < a.v) p[3] = d.w;
      }
    }
  }
  // what is added at the tokens, by one warp, over what the others have stored
  meet<W>();
  if (W > 1 && threadIdx.x >= 32) return;
  const long long first = row.place(begin), last = row.place(end);  // the places of this part
  if (mine && other >= first && other < last && other >= 0 && other < a.v) to[row.lead + other] = r.at(none ? 0.f : row.z[row.lead + other]) + (other == token ? extra + r.g : extra);
  if (!__any_sync(0xFFFFFFFFu, mine && other == token) && lane == 0 && token >= first && token < last && token >= 0 && token < a.v)
    to[row.lead + token] = r.at(none ? 0.f : row.z[row.lead + token]) + r.g;
}

void describe(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], long long rows, int ctas) {
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
}
// How many clusters of so many CTAs are resident at a time.
int resident_clusters(int ctas) {
  static int known[kMostCtas + 1];
  if (!known[ctas]) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    describe(cfg, attr, 1, ctas);
    cfg.numAttrs = 1;
    int most = 0;
    if (cudaOccupancyMaxActiveClusters(&most, log_probs_cluster_kernel, &cfg) != cudaSuccess || most < 1) {
      cudaGetLastError();  // not of the launch that follows
      most = 1;
    }
    known[ctas] = most;
  }
  return known[ctas];
}

bool sizes_fine(long long n, int v, int token_kind, int top) {
  return n >= 0 && n < 1LL << 31 && v > 0 && v <= 1 << 30 && top >= 0 && top <= kMostTop && top <= v && (token_kind == 0 || token_kind == 1);
}

}  // namespace

MTB_API int mtb_token_log_probs_forward_f32(long long n, int v, const float* logits, int token_kind, const void* tokens, int ignores, long long ignore_index, int top,
                                            float* log_probs, float* entropy, float* stats, float* top_log_probs, long long* top_tokens, void* stream) {
  MTB_REQUIRE(sizes_fine(n, v, token_kind, top), "token_log_probs_forward: bad sizes (at most 2^30 values a row, 32 alternatives)");
  if (n == 0) return MTB_OK;
  MTB_REQUIRE(logits && tokens && log_probs && entropy && (top == 0 || (top_log_probs && top_tokens)), "token_log_probs_forward: bad arguments");
  cudaStream_t st = (cudaStream_t)stream;
  const Forward a{n, v, token_kind, ignores, top, ignore_index, logits, tokens, log_probs, entropy, stats, top_log_probs, top_tokens};
  // Few rows: CTAs side by side on each, as long as each has enough of it and all clusters are resident: where some wait, rows by one CTA each take less, but for long ones, where
  // up to six CTAs an SM, some of which wait, still take less than whole rows.  With 8 alternatives, by clusters of 2 and by one CTA each, 370 rows (all resident) of 33000 17.0 and 16.0
  // us, of 50000 20.5 and 21.0, of 131072 38 and 45; 400 rows of 16384 15.2 and 12.2, of 33000 23.0 and 21.0, of 50000 28.1 and 27.9, of 65536 32.2 and 33.3, of 131072 53.7 and 60.9.  By
  // clusters of 8 and of 4, 100 rows of 33000 15.3 and 12.8, of 65536 16.0 and 14.5, of 131072 21.8 and 21.7, of 262144 33.1 and 36.5; one row of 50000 6.7 and 7.2, by one CTA 10.5.
  int ctas = 1;
  const int sms = mtb_sm_count();
  const bool many = n > 8LL * sms;
  while (ctas < kMostCtas && v / (2 * ctas) >= 4096 && n <= (v < 1 << 16 ? resident_clusters(2 * ctas) : 6 * sms / (2 * ctas))) ctas *= 2;
  // Otherwise a row by so many warps that there are enough of them under way, and few as long as the CTAs that an SM holds take turns anyway: then one's search for
  // alternatives is the others' time for loads.  On both sides of each limit, with 8 alternatives, us, by 1 and 4 warps: 16384 x 1024 22.7, 54.6; 800 x 1025 5.5, 6.6, but 300 x 1025
  // 5.0, 4.2; 3000 x 2048 12.7, 13.7; 3000 x 4096 20.1, 18.0; 4000 x 4096 20.7, 21.6; 4000 x 6000 29.3, 26.7.  By 4 and 8: 800 x 2048 6.6, 8.1; 592 x 4096 8.0, 6.9; 1000 x 16384
  // 19.8, 19.8; 1184 x 16384 20.6, 22.0; of all counts from 1185 to 3000, in whose last turns the SMs have more or less to do, x 28000 0.94 to 1.06 of the time, x 32768 0.98 to 1.09; 3400 x 50000
  // 130.8, 129.8; 4096 x 50000 151.0, 159.1; 4096 x 56000 170.1, 171.0; 4096 x 65536 195, 194; with 12 alternatives 4096 x 50000 158, 162, x 56000 177, 175, with 16 165, 166 and 184, 179.
  const bool most = n >= 25LL * sms;
  if (ctas > 1) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    describe(cfg, attr, n, ctas);
    cfg.stream = st;
    cfg.numAttrs = 2;
    MTB_CUDA(cudaLaunchKernelEx(&cfg, log_probs_cluster_kernel, a));
  } else if (v <= 1024 || (v <= 2048 && many) || (v <= 4096 && most)) {
    MTB_LAUNCH(log_probs_kernel<1>, (unsigned)mtb_div_up(n, kWarps), kThreads, 0, st, a);
  } else if (v <= 2048 || (v <= 28000 && many) || (v <= 56000 && top <= 12 && most)) {
    MTB_LAUNCH(log_probs_kernel<4>, (unsigned)n, 128, 0, st, a);
  } else {
    MTB_LAUNCH(log_probs_kernel<kWarps>, (unsigned)n, kThreads, 0, st, a);
  }
  MTB_LAUNCH_CHECK("log_probs_kernel");
  return MTB_OK;
}

MTB_API int mtb_token_log_probs_backward_f32(long long n, int v, const float* logits, int token_kind, const void* tokens, int ignores, long long ignore_index, int top,
                                             const float* dlog_probs, const float* dentropy, const float* dtop, const float* stats, const long long* top_tokens, float* dlogits,
                                             void* stream) {
  MTB_REQUIRE(sizes_fine(n, v, token_kind, top), "token_log_probs_backward: bad sizes (at most 2^30 values a row, 32 alternatives)");
  if (n == 0) return MTB_OK;
  MTB_REQUIRE(logits && tokens && stats && dlogits && (top == 0 || !dtop || top_tokens), "token_log_probs_backward: bad arguments");
  // By one warp 16384 x 1500 takes 34 us, by CTAs of two vectors a thread 46, of four 54; 8192 x 3000 35, 45, 38; eight vectors a thread: 4096 x 10007 58 instead
  // of 56, 4096 x 50000 246 instead of 262.
  const bool warps = v <= 1024 || (v <= 4096 && n > 8LL * mtb_sm_count());
  const int vectors = v <= 2048 ? 2 : v <= 16384 ? 4 : 8, parts = warps ? 1 : mtb_div_up((long long)v + 3, 4 * vectors * kThreads);  // a row may begin three values into its first quad
  const long long ctas = warps ? mtb_div_up(n, kWarps) : n * parts;
  MTB_REQUIRE(ctas < 1LL << 31, "token_log_probs_backward: too many values in one call");
  const Backward a{n, v, token_kind, ignores, top, ignore_index, logits, tokens, dlog_probs, dentropy, dtop, stats, top_tokens, dlogits, parts};
  const auto kernel = warps ? log_probs_backward_kernel<1, 4> : vectors == 2 ? log_probs_backward_kernel<kWarps, 2>
                      : vectors == 4 ? log_probs_backward_kernel<kWarps, 4> : log_probs_backward_kernel<kWarps, 8>;
  MTB_LAUNCH(kernel, (unsigned)ctas, kThreads, 0, (cudaStream_t)stream, a);
  MTB_LAUNCH_CHECK("log_probs_backward_kernel");
  return MTB_OK;
}
