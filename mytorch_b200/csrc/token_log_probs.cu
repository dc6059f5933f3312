// Log probabilities of given tokens, the entropy and the most likely alternatives of every row of logits z [n, v], and their gradient.
//   m = max z,  S = sum exp(z - m),  T = sum exp(z - m) (z - m),  log p_j = z_j - m - log S,  H = log S - T / S  (two terms of one sign: nothing cancels).
//   dz_j = -p_j (g + sum of the alternatives' g) - g_H p_j (log p_j + H), and g, or an alternative's g, added at its token.
// A logit of -inf has probability 0 and adds nothing to the entropy or its gradient; a row of nothing else, or with a NaN or +inf, is NaN.
// Alternatives are in the order of their logits, NaN before everything, equal ones by place, which one whole number holds (`key_of`).
//
// Bound by memory: forward reads a row once, backward reads and writes it once.  Each thread keeps a running maximum and both sums for its sixteenths of a row, and for
// the alternatives only in which of its batches the maximum lies.  When the row is through, the top-th largest of the threads' own largest keys is a bound that no
// alternative is under (so many keys reach it), and only the threads whose largest key reaches it, `top` of them, can hold one: their values are looked at again, out of
// L2, and what reaches the bound, mostly little more than `top` keys, is put in order by counting.  Nothing of this depends on how the values are distributed but the number of keys that reach the
// bound; above kCandidates of them, and for rows with a NaN, `top` passes find one each.
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
  __device__ __forceinline__ void join(float most2, float s2, float t2) {
    const float to = max_nan(most, most2);
    if (to != most) raise(to);
    const float d = gap(fmaxf(most2, kLowest), ref), f = exp2_of(d * kLog2e);
    add(s, s_low, f * s2);
    add(t, t_low, f * (t2 + s2 * d));
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

__device__ __forceinline__ Key sorted(Key k, int lane) {  // over the warp, the largest first
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int j = size / 2; j > 0; j /= 2) {
      const Key o = __shfl_xor_sync(0xFFFFFFFFu, k, j);
      if (((lane & j) == 0) == ((lane & size) == 0 || size == 32) ? o > k : o < k) k = o;
    }
  return k;
}
__device__ __forceinline__ Key merged(Key k, Key other_backwards, int lane) {  // the 32 largest of two sorted lists
  if (other_backwards > k) k = other_backwards;
#pragma unroll
  for (int j = 16; j > 0; j /= 2) {
    const Key o = __shfl_xor_sync(0xFFFFFFFFu, k, j);
    if ((lane & j) == 0 ? o > k : o < k) k = o;
  }
  return k;
}

// What W warps that share a row exchange.
template <int W>
struct Shared {
  static constexpr int kCandidates = W == 1 ? 256 : 1024;
  Key list[W][32], candidate[kCandidates], bound;
  float part[W][3];
  int chosen[kMostTop], chosen_count, candidate_count;
};
template <int W>
__device__ __forceinline__ void meet() {
  if (W == 1) __syncwarp(); else __syncthreads();
}

// Of the quads [begin, end) of a row: the sums, in all threads, and in `out` (not shared.candidate) the `top` largest keys in their order, 0 where there are fewer.
template <int W>
__device__ __forceinline__ Sums look(const Row& row, int begin, int end, int top, Shared<W>& shared, Key* out) {
  constexpr int T = 32 * W;
  const int lane = threadIdx.x & 31, warp = W == 1 ? 0 : threadIdx.x >> 5, id = W == 1 ? lane : threadIdx.x;
  Sums sums;
  int where = -1;  // the first quad of the batch with the largest value
  float4 next[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) next[u] = row.quad(begin + id + u * T, end);
  for (int q = begin; q < end; q += 4 * T) {
    float x[16];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      x[4 * u] = next[u].x; x[4 * u + 1] = next[u].y; x[4 * u + 2] = next[u].z; x[4 * u + 3] = next[u].w;
    }
    if (q + 4 * T < end) {
#pragma unroll
      for (int u = 0; u < 4; ++u) next[u] = row.quad(q + 4 * T + id + u * T, end);
    }
    float most = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) most = max_nan(most, x[i]);
    most = max_nan(most, sums.most);
    if (most != sums.most) {
      where = q;
      sums.raise(most);
    }
    float s[4] = {0, 0, 0, 0}, t[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float d = gap(x[i], sums.ref), e = exp2_of(d * kLog2e);
      s[i % 4] += e;
      t[i % 4] = fmaf(e, d, t[i % 4]);
    }
    Sums::add(sums.s, sums.s_low, (s[0] + s[1]) + (s[2] + s[3]));
    Sums::add(sums.t, sums.t_low, (t[0] + t[1]) + (t[2] + t[3]));
  }
  const float mine = sums.most;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_xor_sync(0xFFFFFFFFu, sums.most, o), s = __shfl_xor_sync(0xFFFFFFFFu, sums.s, o), t = __shfl_xor_sync(0xFFFFFFFFu, sums.t, o);
    sums.join(m, s, t);
  }
  if (W > 1) {
    if (lane == 0) { shared.part[warp][0] = sums.most; shared.part[warp][1] = sums.s; shared.part[warp][2] = sums.t; }
  }
  if (id == 0) shared.chosen_count = shared.candidate_count = 0;
  // the thread's largest key
  Key key = 0;
  if (top) {
    if (where >= 0 && mine == mine) {
#pragma unroll
      for (int u = 3; u >= 0; --u) {
        const int q = where + id + u * T, i = row.place(q);
        const float4 f = row.quad(q, end);
        if (f.w == mine) key = key_of(mine, i + 3);
        if (f.z == mine) key = key_of(mine, i + 2);
        if (f.y == mine) key = key_of(mine, i + 1);
        if (f.x == mine) key = key_of(mine, i);
      }
    } else if (begin + id < end && row.place(begin + id) < row.v) {  // nothing but -inf
      const int i = row.place(begin + id);
      key = key_of(-INFINITY, i < 0 ? 0 : i);
    }
    Key best = sorted(key, lane);
    if (W > 1) {
      shared.list[warp][lane] = best;
#pragma unroll
      for (int step = 1; step < W; step *= 2) {
        __syncthreads();
        if (warp % (2 * step) == 0) {
          best = merged(best, shared.list[warp + step][31 - lane], lane);
          shared.list[warp][lane] = best;
        }
      }
    }
    if (warp == 0 && lane == top - 1) shared.bound = best;
  }
  meet<W>();
  if (W > 1) {
    sums = Sums();
    for (int w = 0; w < W; ++w) sums.join(shared.part[w][0], shared.part[w][1], shared.part[w][2]);
  }
  if (!top) return sums;
  bool slow = sums.most != sums.most;
  if (!slow) {
    const Key bound = shared.bound;
    if (key != 0 && key >= bound) shared.chosen[atomicAdd(&shared.chosen_count, 1)] = id;  // at most `top` of them, or all that have a key where fewer have
    meet<W>();
    const int chosen = shared.chosen_count;
    for (int c = warp; c < chosen; c += W) {
      for (int q = begin + shared.chosen[c] + lane * T; q < end; q += 32 * T) {
        const float4 f = row.quad(q, end);
        const int i = row.place(q);
        const float x[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const Key k = key_of(x[j], i + j);
          if (k >= bound && i + j >= 0 && i + j < row.v) {
            const int at = atomicAdd(&shared.candidate_count, 1);
            if (at < Shared<W>::kCandidates) shared.candidate[at] = k;
          }
        }
      }
    }
    meet<W>();
    const int count = shared.candidate_count;
    slow = count > Shared<W>::kCandidates;
    if (!slow) {
      for (int i = id; i < top; i += T)
        if (i >= count) out[i] = 0;
      for (int i = id; i < count; i += T) {
        const Key k = shared.candidate[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += shared.candidate[j] > k;
        if (rank < top) out[rank] = k;
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
        if (lane == 0) shared.list[warp][0] = best;
        __syncthreads();
        for (int w = 0; w < W; ++w)
          if (shared.list[w][0] > best) best = shared.list[w][0];
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

// By thread `id` of those that share the row.
__device__ __forceinline__ void leave(const Forward& a, long long row, int id, const Sums& sums, const Key* found) {
  const bool none = !(sums.most >= kLowest && sums.most < INFINITY);  // a NaN, +inf, or nothing but -inf
  const float s = none ? NAN : sums.s + sums.s_low, log_s = logf(s);
  if (id == 0) {
    const long long token = token_at(a.tokens, a.wide, row);
    a.log_probs[row] = a.ignores && token == a.ignore_index ? 0.f : token < 0 || token >= a.v ? NAN : a.logits[row * a.v + token] - sums.most - log_s;
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
__global__ void __launch_bounds__(kThreads) log_probs_kernel(const __grid_constant__ Forward a) {
  __shared__ Shared<W> shared[kWarps / W];
  __shared__ Key found[kWarps / W][kMostTop];
  mtb_launch_dependents();
  mtb_wait_prior();
  const int part = W == 1 ? threadIdx.x >> 5 : 0;
  const long long index = W == 1 ? blockIdx.x * (long long)kWarps + part : blockIdx.x;
  if (index >= a.n) return;
  const Row row(a.logits + index * a.v, a.v);
  const Sums sums = look<W>(row, 0, row.quads, a.top, shared[part], found[part]);
  leave(a, index, W == 1 ? threadIdx.x & 31 : threadIdx.x, sums, found[part]);
}

// A row by a cluster of CTAs, each of which finds the alternatives of its part; the first puts them together.
__global__ void __launch_bounds__(kThreads) log_probs_cluster_kernel(const __grid_constant__ Forward a) {
  __shared__ Shared<kWarps> shared;
  __shared__ Key found[kMostTop], all[kMostCtas][kMostTop];
  __shared__ float parts[kMostCtas][3];
  mtb_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // the first CTA's shared memory is there once it has started
  mtb_wait_prior();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const long long index = blockIdx.x / ctas;
  const Row row(a.logits + index * a.v, a.v);
  const int each = (row.quads + ctas - 1) / ctas, begin = rank * each < row.quads ? rank * each : row.quads, end = begin + each < row.quads ? begin + each : row.quads;
  const Sums mine = look<kWarps>(row, begin, end, a.top, shared, found);
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (threadIdx.x < a.top) cluster.map_shared_rank(&all[0][0], 0)[rank * kMostTop + threadIdx.x] = found[threadIdx.x];
  if (threadIdx.x == 0) {
    float* to = cluster.map_shared_rank(&parts[0][0], 0) + 3 * rank;
    to[0] = mine.most;
    to[1] = mine.s + mine.s_low;
    to[2] = mine.t + mine.t_low;
  }
  cluster.sync();
  if (rank != 0) return;
  Sums sums;
  for (int r = 0; r < ctas; ++r) sums.join(parts[r][0], parts[r][1], parts[r][2]);
  if (a.top) {
    for (int i = threadIdx.x; i < ctas * a.top; i += kThreads) {
      const Key k = all[i / a.top][i % a.top];
      int place = i % a.top;  // in its own list
      for (int r = 0; r < ctas; ++r)
        for (int j = 0; r != i / a.top && j < a.top && all[r][j] > k; ++j) ++place;
      if (k != 0 && place < a.top) found[place] = k;
    }
    __syncthreads();
  }
  leave(a, index, threadIdx.x, sums, found);
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

  // exp here by the function, whose error does not grow with its argument: an element moves 8 bytes, there is time.
  __device__ __forceinline__ float at(float z) const {
    const float d = z - m, p = expf(d) * per_s;
    return -p * (all + gh * (fmaxf(d, kFar) - log_s + h));
  }
};

constexpr int kPart = 16 * kThreads;  // values of a CTA

// A row by W warps: 1, or `parts` CTAs, four vectors a thread.
template <int W>
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
  const int begin = W == 1 ? 0 : (int)(blockIdx.x % a.parts) * (kPart / 4), end = W == 1 ? row.quads : min(begin + kPart / 4, row.quads);
  float4 f[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) f[u] = row.quad(begin + id + u * T, end);
  // every warp for itself: the row's numbers, an alternative a lane
  const long long token = token_at(a.tokens, a.wide, index);
  RowGradient r;
  r.m = a.stats[3 * index];
  const float s = a.stats[3 * index + 1];
  r.h = a.stats[3 * index + 2];
  r.per_s = 1.f / s;
  r.log_s = logf(s);
  r.g = !a.dlog_probs || (a.ignores && token == a.ignore_index) ? 0.f : a.dlog_probs[index];
  r.gh = a.dentropy ? a.dentropy[index] : 0.f;
  const bool mine = a.dtop && lane < a.top;
  const float extra = mine ? a.dtop[index * a.top + lane] : 0.f;
  const long long other = mine ? a.top_tokens[index * a.top + lane] : -1;
  r.all = extra;
  for (int o = 16; o > 0; o >>= 1) r.all += __shfl_xor_sync(0xFFFFFFFFu, r.all, o);
  r.all += r.g;
  for (int q = begin; q < end; q += 4 * T) {
    if (W == 1 && q > begin) {
#pragma unroll
      for (int u = 0; u < 4; ++u) f[u] = row.quad(q + id + u * T, end);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
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
  if (mine && other >= first && other < last && other >= 0 && other < a.v) to[row.lead + other] = r.at(row.z[row.lead + other]) + (other == token ? extra + r.g : extra);
  if (!__any_sync(0xFFFFFFFFu, mine && other == token) && lane == 0 && token >= first && token < last && token >= 0 && token < a.v)
    to[row.lead + token] = r.at(row.z[row.lead + token]) + r.g;
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
  // few rows: CTAs side by side on each, as long as all fit and each has enough of it
  int ctas = 1;
  while (ctas < kMostCtas && n * ctas * 2 <= 2 * mtb_sm_count() && v / (2 * ctas) >= 2048) ctas *= 2;
  if (ctas > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    MTB_CUDA(cudaLaunchKernelEx(&cfg, log_probs_cluster_kernel, a));
  } else if (v <= 1024) {
    MTB_LAUNCH(log_probs_kernel<1>, (unsigned)mtb_div_up(n, kWarps), kThreads, 0, st, a);
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
  const int parts = mtb_div_up((long long)v + 3, kPart);  // a row may begin three values into its first quad
  const Backward a{n, v, token_kind, ignores, top, ignore_index, logits, tokens, dlog_probs, dentropy, dtop, stats, top_tokens, dlogits, parts};
  if (v <= 1024) {
    MTB_LAUNCH(log_probs_backward_kernel<1>, (unsigned)mtb_div_up(n, kWarps), kThreads, 0, (cudaStream_t)stream, a);
  } else {
    MTB_REQUIRE(n * parts < 1LL << 31, "token_log_probs_backward: too many values in one call");
    MTB_LAUNCH(log_probs_backward_kernel<kWarps>, (unsigned)(n * parts), kThreads, 0, (cudaStream_t)stream, a);
  }
  MTB_LAUNCH_CHECK("log_probs_backward_kernel");
  return MTB_OK;
}
