// Log probabilities of given tokens, the entropy and the likeliest alternatives of rows of logits x under p = softmax(x / T):
//   log p_i = (x_i - M) / T - ln S,   M = max x,  S = sum_i e^((x_i - M) / T)
//   entropy = -sum_i p_i ln p_i = ln S - (sum_i d_i e^d_i) / S,   d_i = (x_i - M) / T
// One pass: a thread keeps M, S and the third sum of what it has seen, rescaled when M rises, 16 values at a time; these meet over
// lanes, warps, the CTAs of a cluster that share a row, and the ranks that share a vocabulary. Differences are taken before they
// are scaled, so that a row of the type's lowest value is the uniform distribution that it stands for. The logarithm of a token that is
// nearly certain is kept to its own last bits (log1p of the others' sum): the warp that has it sums its values once more, 62.1 -> 63.5 us
// for 1500 x 100003 with such a token in each row. To sum them apart in the one pass, at each rise of M, took 103 for all rows.
//
// The `top` largest ride along: a CTA's first 4096 values give a bound below which none of them is, what lies above is noted in shared
// memory (a test of each thread's maximum of 16, which the sums need anyway), and only those few are ranked. Values are compared as
// they came, ties by the token, through one 64-bit key; NaN counts as -inf there.
// Without alternatives the reading bounds it: 2048 x 32768 in fp32 47 us (5.7 TB/s), 1500 x 100003 in bf16 62 (4.8 TB/s). With them noting and ranking do: 75
// with top = 20 and 95 with top = 2; one row of 32768 6.5 us, 3.5 without. Rows that rise from token to token (read again) or are constant (all
// values reach the bound) are the slowest: 256 x 32768 in bf16 265 and 190 us, 20 otherwise.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ivb_common.h"
#include "ivb_device.cuh"
#include "ivb_kv4.cuh"

namespace ivb {
namespace {

namespace cg = cooperative_groups;

constexpr int kLogThreads = 256, kMostTop = 256, kBatch = 16;  // values of a thread at a time
constexpr int kWarps = kLogThreads / 32, kSpan = kLogThreads * kBatch;
constexpr int kSlack = 96, kRoom = 32 * kBatch + kSlack;  // a warp's list: one turn's values and what it had before
constexpr int kFewTop = 64;
// So many keys are ranked each against all; of more the largest `top` are found first, bit by bit (against all, 256 x 32768 with top = 128 took 164 us).
constexpr int kRankAll = 384;
// Above it logf of the sum has three bits fewer than its own at most, and two lanes cannot have the largest.
constexpr float kSure = 1.125f;
constexpr int kHead = 4;  // words of a slice's statistics
constexpr unsigned kAbsent = 0x7fffffffu;  // of a slice that does not hold the token
constexpr float kLeast = -200.0f;  // 2^-200 is zero in fp32: keeps -inf * 0 out of the third sum

typedef unsigned long long Key;

struct LogProbs {
  const void* logits;
  const int64_t* tokens;
  int64_t stride;
  int vocab, given, top, v0;
  float inv_t;
  float* token_lp;
  float* entropy;
  float* top_lp;
  int64_t* top_ids;
  uint32_t* parts;  // of a slice, in place of the others: its statistics, tokens' logits, keys, ids
};

// The largest logit, the sum of e^(x - largest), and the third sum in units of log2. Where one token has nearly all of the probability its own 1
// would cut the others' sum, of which its logarithm and the entropy are made, at 2^-24: a warp whose sum is below kSure sums the others
// apart, and n = 1 stands for the largest. Else n = 0.
struct Stats {
  float m, n, s, t;
};

// Ascending with x; -0 as +0 and NaN as -inf.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x == x ? x + 0.0f : -INFINITY);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
// The next float above x; of infinity NaN, which none reaches.
__device__ __forceinline__ float above(float x) { return unordered(ordered(x) + 1); }
__device__ __forceinline__ Key key_of(uint32_t value, uint32_t id) { return static_cast<Key>(value) << 32 | (0xffffffffu - id); }
__device__ __forceinline__ uint32_t id_of(Key k) { return 0xffffffffu - static_cast<uint32_t>(k); }

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two parts' sums over the larger maximum; NaN in either stays.
__device__ __forceinline__ Stats join(Stats a, Stats b, float c) {
  Stats r;
  r.m = fmaxf(a.m, b.m);
  const bool top_a = a.m == r.m, top_b = b.m == r.m;
  const float da = top_a ? 0.0f : fmaxf((a.m - r.m) * c, kLeast), db = top_b ? 0.0f : fmaxf((b.m - r.m) * c, kLeast);
  const float fa = exp2_of(da), fb = exp2_of(db), sa = top_a ? a.s : a.s + a.n, sb = top_b ? b.s : b.s + b.n;
  r.n = (top_a ? a.n : 0.0f) + (top_b ? b.n : 0.0f);
  r.s = fmaf(sa, fa, sb * fb);
  r.t = fmaf(fmaf(sa, da, a.t), fa, fmaf(sb, db, b.t) * fb);
  return r;
}
__device__ __forceinline__ Stats from_lane(Stats a, int other) {
  return {__shfl_sync(0xFFFFFFFFu, a.m, other), __shfl_sync(0xFFFFFFFFu, a.n, other), __shfl_sync(0xFFFFFFFFu, a.s, other), __shfl_sync(0xFFFFFFFFu, a.t, other)};
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// The largest keys so far in order (`have` of them, zeros behind), and what each warp has noted since.
struct Shared {
  Key noted[kWarps][kRoom];
  alignas(16) Key list[kRankAll];
  Key best[kMostTop];
  Stats warps[kWarps], all;
  float bounds[kWarps];
  int counts[kWarps], have, found, over, reached[3];
};

// The `top` largest of the best and all that is noted become the best, in order if `in_order`; nothing is noted then. Returns a key
// that `top` keys at least reach, 0 where there are fewer. All threads; barriers on both sides. kDistinct: a token is there once, as within a
// row; slices that were handed in may overlap.
template <bool kDistinct>
__device__ Key rank_keys(Shared& sh, int top, bool in_order) {
  const int tid = threadIdx.x;
  __syncthreads();
  const int have = sh.have;
  int n = have, before = have;
  Key at = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    before += w < (tid >> 5) ? sh.counts[w] : 0;
    n += sh.counts[w];
  }
  auto each = [&](auto f) {
    for (int i = tid; i < have; i += kLogThreads) f(sh.best[i]);
    for (int w = 0; w < kWarps; ++w)
      for (int i = tid; i < sh.counts[w]; i += kLogThreads) f(sh.noted[w][i]);
  };
  if (n <= kRankAll) {
    for (int i = tid; i < have; i += kLogThreads) sh.list[i] = sh.best[i];
    for (int i = tid & 31; i < sh.counts[tid >> 5]; i += 32) sh.list[before + i] = sh.noted[tid >> 5][i];
  } else {
    // the largest value that at least `top` keys reach, until just these do. A thread keeps its first keys.
    constexpr int kKept = 5;
    Key kept[kKept];
    auto key_at = [&](int i) {
      if (i < have) return sh.best[i];
      i -= have;
      int w = 0;
      while (i >= sh.counts[w]) i -= sh.counts[w++];
      return sh.noted[w][i];
    };
#pragma unroll
    for (int i = 0; i < kKept; ++i) kept[i] = i * kLogThreads + tid < n ? key_at(i * kLogThreads + tid) : 0;
    const bool all_kept = n <= kKept * kLogThreads;
    if (tid < 3) sh.reached[tid] = 0;
    if (tid == 3) sh.found = 0;
    __syncthreads();
    for (int bit = 63; bit >= 0; --bit) {
      const Key trial = at | Key(1) << bit;
      int mine = 0;
      if (all_kept) {
#pragma unroll
        for (int i = 0; i < kKept; ++i) mine += kept[i] >= trial;
      } else {
        each([&](Key k) { mine += k >= trial; });
      }
      mine = __reduce_add_sync(0xFFFFFFFFu, mine);
      if ((tid & 31) == 0 && mine != 0) atomicAdd(&sh.reached[bit % 3], mine);
      __syncthreads();
      const int reached = sh.reached[bit % 3];
      if (reached >= top) at = trial;
      if (reached == top) break;
      if (tid == 0) sh.reached[(bit + 1) % 3] = 0;  // read before the barrier, and next used after another one
    }
    __syncthreads();
    each([&](Key k) {
      if (kDistinct ? k >= at : k > at) sh.list[atomicAdd(&sh.found, 1)] = k;  // `top` of them, or fewer and all others the same
    });
    n = top;
    __syncthreads();
    if constexpr (!kDistinct) {
      for (int i = sh.found + tid; i < top; i += kLogThreads) sh.list[i] = at;
      __syncthreads();
    }
    if (!in_order) {
      for (int i = tid; i < top; i += kLogThreads) sh.best[i] = sh.list[i];
      if (tid < kWarps) sh.counts[tid] = 0;
      if (tid == kWarps) sh.have = top;
      __syncthreads();
      return at;
    }
  }
  __syncthreads();
  // each key against all, by 1 to 8 neighbouring lanes
  const int lanes = n <= 32 ? 8 : n <= 64 ? 4 : n <= 128 ? 2 : 1, l = tid & (lanes - 1);
  for (int i0 = 0; i0 < n; i0 += kLogThreads / lanes) {
    const int i = i0 + tid / lanes;
    const Key k = i < n ? sh.list[i] : 0;
    int above = 0;
#pragma unroll 4
    for (int j = 2 * l; j + 1 < n; j += 2 * lanes) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(sh.list + j);
      above += (two.x > k) + (two.y > k);
      if constexpr (!kDistinct) above += (two.x == k && j < i) + (two.y == k && j + 1 < i);
    }
    if ((n & 1) != 0 && l == 0) above += sh.list[n - 1] > k;  // of equal ones it is the last
    for (int d = 1; d < lanes; d <<= 1) above += __shfl_xor_sync(0xFFFFFFFFu, above, d);
    if (i < n && l == 0 && above < top) sh.best[above] = k;
  }
  for (int i = n + tid; i < top; i += kLogThreads) sh.best[i] = 0;
  if (tid < kWarps) sh.counts[tid] = 0;
  if (tid == kWarps) sh.have = min(n, top);
  __syncthreads();
  return n < top ? 0 : sh.best[top - 1];
}

// Notes up to `top` keys of an ordered list that ends in zeros; a whole warp, its own list is empty.
__device__ __forceinline__ void note_list(Shared& sh, int warp, int top, Key key_at(const void*, int, int), const void* from) {
  const int lane = threadIdx.x & 31;
  int count = 0;
  for (int i0 = 0; i0 < top; i0 += 32) {
    const Key k = i0 + lane < top ? key_at(from, i0 + lane, top) : 0;
    if (k != 0) sh.noted[warp][i0 + lane] = k;
    count += __popc(__ballot_sync(0xFFFFFFFFu, k != 0));
  }
  if (lane == 0) sh.counts[warp] = count;
}

// What one row's sums and largest keys say; all threads of a CTA.
template <typename F>
__device__ __forceinline__ void finish(const LogProbs& p, const Shared& sh, Stats all, int64_t row, F token_logit) {
  const int tid = threadIdx.x;
  const float sum = all.n + all.s;
  const float ln_s = !(sum > 0.0f) ? __uint_as_float(0x7fffffffu) : all.n == 1.0f ? log1pf(all.s) : logf(sum);  // nothing but -inf: no distribution
  if (tid == 0) p.entropy[row] = ln_s - all.t / sum * 0.6931471805599453f;
  auto log_p = [&](float x) {
    const float d = x - all.m;
    if (d > -INFINITY || x == -INFINITY) return fmaf(d, p.inv_t, -ln_s);
    return x * p.inv_t - all.m * p.inv_t - ln_s;  // further apart than fp32 reaches, which their quotients by T need not be
  };
  for (int i = tid; i < p.given; i += kLogThreads) p.token_lp[row * p.given + i] = log_p(token_logit(i));
  for (int i = tid; i < p.top; i += kLogThreads) {
    p.top_lp[row * p.top + i] = log_p(unordered(static_cast<uint32_t>(sh.best[i] >> 32)));
    p.top_ids[row * p.top + i] = sh.best[i] == 0 ? -1 : static_cast<int64_t>(id_of(sh.best[i]));  // none: slices of fewer tokens than that
  }
}

template <typename T>
__device__ float logit_of_token(const LogProbs& p, int64_t row, int i) {
  const int64_t token = p.tokens[row * p.given + i] - p.v0;
  return token >= 0 && token < p.vocab ? to_f32<T>(static_cast<const T*>(p.logits)[row * p.stride + token]) : __uint_as_float(kAbsent);
}

template <typename T, bool kTop>
__global__ void __launch_bounds__(kLogThreads, 4) log_probs_kernel(LogProbs p) {
  constexpr int E = 16 / static_cast<int>(sizeof(T)), U = kBatch / E;
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / static_cast<unsigned>(C);
  pdl_enter();
  // 16-byte chunks from the one that holds the row's first value on; value i of chunk k is the row's value k E + i - shift
  const T* const x = static_cast<const T*>(p.logits) + row * p.stride;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int chunks = static_cast<int>((static_cast<int64_t>(shift) + p.vocab + E - 1) / E), per = (chunks + C - 1) / C;
  const int c0 = min(rank * per, chunks), c1 = min(c0 + per, chunks), turns = (c1 - c0 + kLogThreads * U - 1) / (kLogThreads * U);
  const float c = p.inv_t * 1.4426950408889634f;
  // Chunk c0 + (256 u + tid) of a turn; chunks from `whole0` to `whole1` lie in the row with all their values, as those of nearly all turns do.
  const uint4* at = reinterpret_cast<const uint4*>(x - shift) + c0 + tid;
  const int whole0 = shift > 0 ? 1 : 0, whole1 = min(c1, static_cast<int>((static_cast<int64_t>(shift) + p.vocab) / E));
  constexpr int kTurn = kLogThreads * U;
  auto load = [&](int turn, int thread, uint4 (&to)[U]) {
    const int first = c0 + turn * kTurn;
    if (first >= whole0 && first + kTurn <= whole1) {
#pragma unroll
      for (int u = 0; u < U; ++u) to[u] = __ldcs(at + u * kLogThreads);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int chunk = first + u * kLogThreads + thread;
        union {
          uint4 w;
          T t[E];
        } e;
        if (chunk >= whole0 && chunk < whole1) {
          e.w = __ldcs(at + u * kLogThreads);
        } else {
          const int64_t i0 = static_cast<int64_t>(chunk) * E - shift;
#pragma unroll
          for (int i = 0; i < E; ++i) e.t[i] = chunk < c1 && i0 + i >= 0 && i0 + i < p.vocab ? x[i0 + i] : from_f32<T>(-INFINITY);
        }
        to[u] = e.w;
      }
    }
    at += kTurn;
  };
  auto unpack = [](const uint4 (&from)[U], float (&v)[kBatch]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const uint32_t w[4] = {from[u].x, from[u].y, from[u].z, from[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[u * E + 2 * i] = __uint_as_float(w[i] << 16);
          v[u * E + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      } else {
        union {
          uint4 w;
          T t[E];
        } e;
        e.w = from[u];
#pragma unroll
        for (int i = 0; i < E; ++i) v[u * E + i] = to_f32<T>(e.t[i]);
      }
    }
  };
  // the row's first 256 tokens' logits are on their way meanwhile
  const float first_logit = rank == 0 && tid < p.given ? logit_of_token<T>(p, row, tid) : 0.0f;
  float m = -INFINITY;
  float2 s2 = make_float2(0.0f, 0.0f), t2 = s2;  // of even and of odd values
  float edge = -INFINITY;  // the first value that is noted: above the bound, as later tokens as large as it are too late
  int noted = 0;  // by this warp, since the last ranking
  if (kTop && tid == 0) sh.have = sh.over = 0;
  uint4 next[U];
  // What is noted is ranked, and the bound raised to the top-th largest, after the turns 0, 3, 15, ...: between them warps need not wait
  // for one another. A row that notes more than there is room for (one in ascending order does) is read again, and ranked after every turn.
  bool careful = false;
  const uint4* const begin = at;
scan:
  if (turns > 0) load(0, tid, next);
  for (int turn = 0; turn < turns; ++turn) {
    float v[kBatch];
    uint4 now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = next[u];
    unpack(now, v);
    if (turn + 1 < turns) load(turn + 1, tid, next);
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kBatch; i += 2) most = max3(most, v[i], v[i + 1]);
    if (most > m) {
      const float d = fmaxf((m - most) * c, kLeast), f = exp2_of(d);  // from nothing: sums of zero
      t2 = make_float2(fmaf(s2.x, d, t2.x) * f, fmaf(s2.y, d, t2.y) * f);
      s2 = make_float2(s2.x * f, s2.y * f);
      m = most;
    }
    const float minus = m == -INFINITY ? 0.0f : -m;
    const float2 minus2 = make_float2(minus, minus), c2 = make_float2(c, c);
#pragma unroll
    for (int i = 0; i < kBatch; i += 2) {
      const float2 d = __fmul2_rn(__fadd2_rn(make_float2(v[i], v[i + 1]), minus2), c2), e = make_float2(exp2_of(d.x), exp2_of(d.y));
      s2 = __fadd2_rn(s2, e);
      t2 = __ffma2_rn(make_float2(fmaxf(d.x, kLeast), fmaxf(d.y, kLeast)), e, t2);
    }
    if constexpr (kTop) {
      const uint32_t first = static_cast<uint32_t>((static_cast<int64_t>(c0) + turn * kTurn + tid) * E - shift);  // value 0's place; wraps below zero
      auto again = [&] {
#pragma unroll
        for (int u = 0; u < U; ++u) asm volatile("" : "+r"(now[u].x), "+r"(now[u].y), "+r"(now[u].z), "+r"(now[u].w));
        unpack(now, v);
      };
      auto place = [&](int i) { return first + i / E * (kLogThreads * E) + i % E; };
      auto keep = [&](bool in, unsigned who, float value, uint32_t id) {
        const int to = noted + __popc(who & ((1u << lane) - 1));
        if (in && to < kRoom) sh.noted[warp][to] = key_of(ordered(value), id + static_cast<uint32_t>(p.v0));
        noted += __popc(who);
      };
      // Notes the values from `edge` on: all lanes' first ones, then their second ones, as they seldom have more than one (the 16 values in turn, a
      // vote and a branch apiece: 76.9 us for 74.6 with 2048 x 32768 in fp32, top = 20).
      auto note = [&](float edge) {
        // unpacked again: values kept for this in each turn took 91 us there
        again();
        unsigned mine = 0;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) mine |= v[i] >= edge ? 1u << i : 0u;
        for (unsigned who; (who = __ballot_sync(0xFFFFFFFFu, mine != 0)) != 0; mine &= mine - 1) {
          const int at_hand = __ffs(mine) - 1;
          float value = v[0];
#pragma unroll
          for (int i = 1; i < kBatch; ++i) value = at_hand == i ? v[i] : value;
          keep(mine != 0, who, value, place(at_hand));
        }
        if (noted > kRoom) {
          noted = kRoom;
          if (lane == 0) sh.over = 1;
        }
      };
      if (turn == 0) {
        float bound = -INFINITY;
        if (p.top <= kFewTop) {
          // Each warp's r-th largest of its lanes' maxima, with r = top / 8 rounded up: `top` values at least reach the least of these.
          // (The top-th largest of all 256, each ranked against all, is a closer bound, but took 1.6 us of each CTA.)
          uint32_t own = ordered(most), reached = 0;
          for (int r = 0; r < p.top; r += kWarps) {
            reached = __reduce_max_sync(0xFFFFFFFFu, own);
            const unsigned who = __ballot_sync(0xFFFFFFFFu, own == reached);
            if (lane == __ffs(who) - 1) own = 0;
          }
          if (lane == 0) sh.bounds[warp] = unordered(reached);
          __syncthreads();
          bound = sh.bounds[0];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) bound = fminf(bound, sh.bounds[w]);
        }
        if (bound == -INFINITY) {
          // Of more, and where a mask leaves warps nothing: the upper 16 bits of the top-th largest value's key, bit by bit (with as many maxima the bound would pass a third of all values:
          // 338 us for 256 x 32768 with top = 256).
          again();
          if (tid < 3) sh.reached[tid] = 0;
          __syncthreads();
          uint32_t key = 0;
          for (int bit = 31; bit >= 16; --bit) {
            const float trial = unordered(key | 1u << bit);  // a NaN above all: reached by none
            int mine = 0;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) mine += v[i] >= trial;
            mine = __reduce_add_sync(0xFFFFFFFFu, mine);
            if (lane == 0 && mine != 0) atomicAdd(&sh.reached[bit % 3], mine);
            __syncthreads();
            if (sh.reached[bit % 3] >= p.top) key |= 1u << bit;
            if (tid == 0) sh.reached[(bit + 1) % 3] = 0;
          }
          bound = key > ordered(-INFINITY) ? unordered(key) : -INFINITY;
        }
        if (bound == -INFINITY) {
          // Fewer than `top` values above -inf, which are noted, and of those that count as -inf the `top` tokens the CTA begins with: what
          // comes behind these is less than all of them (all noted, a row with 100 tokens allowed took 115 us in place of 9).
          again();
          const uint32_t begins = static_cast<uint32_t>(max(static_cast<int64_t>(c0) * E - shift, static_cast<int64_t>(0)));
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const bool in = c0 + i / E * kLogThreads + tid < c1 && place(i) < static_cast<uint32_t>(p.vocab) &&
                            (v[i] > -INFINITY || place(i) - begins < static_cast<uint32_t>(p.top));
            const unsigned who = __ballot_sync(0xFFFFFFFFu, in);
            if (who != 0) keep(in, who, v[i], place(i));
          }
        } else if (__any_sync(0xFFFFFFFFu, most >= bound)) note(bound);
        edge = above(bound);
      } else if (__any_sync(0xFFFFFFFFu, most >= edge)) {
        note(edge);
      }
      if (turn + 1 < turns && (careful || ((turn & (turn + 1)) == 0 && (turn + 1 & 0x55555555) != 0))) {
        if (lane == 0) sh.counts[warp] = noted;
        noted = 0;
        const Key least = rank_keys<true>(sh, p.top, false);
        if (least != 0) edge = fmaxf(edge, above(unordered(static_cast<uint32_t>(least >> 32))));
      }
    }
  }
  if constexpr (kTop) {
    if (lane == 0) sh.counts[warp] = noted;
    __syncthreads();
    const bool again = sh.over != 0;  // never when careful: a turn's values find room
    __syncthreads();
    if (again) {
      if (tid == 0) sh.over = sh.have = 0;
      careful = true;
      noted = 0;
      at = begin;
      m = -INFINITY;
      s2 = t2 = make_float2(0.0f, 0.0f);
      __syncthreads();
      goto scan;
    }
  }
  const Stats own = {m, 0.0f, s2.x + s2.y, t2.x + t2.y};
  Stats mine = own;
  // over lanes, warps and the cluster
#pragma unroll
  for (int d = 1; d < 32; d <<= 1)
    mine = join(mine, {__shfl_xor_sync(0xFFFFFFFFu, mine.m, d), 0.0f, __shfl_xor_sync(0xFFFFFFFFu, mine.s, d), __shfl_xor_sync(0xFFFFFFFFu, mine.t, d)}, c);
  // By one lane's sum, as the lanes' own may differ in their last bits and what follows needs the whole warp; all have the same maximum.
  if (__shfl_sync(0xFFFFFFFFu, mine.s, 0) < kSure && mine.m > -INFINITY) {  // NaN: not
    // one lane has the largest, once: the warp's lanes take a turn of that lane's each again, and sum what is not it
    const int sure = __ffs(__ballot_sync(0xFFFFFFFFu, m == mine.m)) - 1;
    float others = 0.0f;
    for (int turn = lane; turn < turns; turn += 32) {
      at = begin + (sure - lane) + turn * kTurn;
      load(turn, tid - lane + sure, next);
      float v[kBatch];
      unpack(next, v);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) others += v[i] == mine.m ? 0.0f : exp2_of((v[i] - mine.m) * c);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) others += __shfl_xor_sync(0xFFFFFFFFu, others, d);
    mine = lane == sure ? Stats{m, 1.0f, others, own.t} : own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) mine = join(mine, from_lane(mine, lane ^ d), c);
  }
  if (lane == 0) sh.warps[warp] = mine;
  __syncthreads();
  Stats all = sh.warps[lane & (kWarps - 1)];
#pragma unroll
  for (int d = 1; d < kWarps; d <<= 1)
    all = join(all, from_lane(all, lane ^ d), c);
  // one lane's, as the lanes' sums may differ in their last bits
  all = from_lane(all, 0);
  if constexpr (kTop) rank_keys<true>(sh, p.top, true);
  if (C > 1) {
    if (tid == 0) sh.all = all;
    cluster.sync();
    if (rank == 0) {
      for (int k = 1; k < C; ++k) all = join(all, cluster.map_shared_rank(&sh, k)->all, c);
      if constexpr (kTop) {
        if (warp > 0 && warp < C)
          note_list(sh, warp, p.top, [](const void* from, int i, int) { return static_cast<const Key*>(from)[i]; }, cluster.map_shared_rank(&sh, warp)->best);
        rank_keys<true>(sh, p.top, true);
      }
    }
    cluster.sync();  // no CTA leaves while another reads its shared memory
    if (rank != 0) return;
  }
  if (p.parts == nullptr) {
    finish(p, sh, all, row, [&](int i) { return i == tid ? first_logit : logit_of_token<T>(p, row, i); });
    return;
  }
  uint32_t* const out = p.parts + row * (kHead + p.given + 2 * p.top);
  if (tid == 0) {
    out[0] = __float_as_uint(all.m);
    out[1] = __float_as_uint(all.n);
    out[2] = __float_as_uint(all.s);
    out[3] = __float_as_uint(all.t);
  }
  for (int i = tid; i < p.given; i += kLogThreads) out[kHead + i] = __float_as_uint(i == tid ? first_logit : logit_of_token<T>(p, row, i));
  for (int i = tid; i < p.top; i += kLogThreads) {
    out[kHead + p.given + i] = static_cast<uint32_t>(sh.best[i] >> 32);
    out[kHead + p.given + p.top + i] = id_of(sh.best[i]);
  }
}

// The slices' parts [world][rows][4 + given + 2 top] of a row.
__global__ void __launch_bounds__(kLogThreads) log_probs_merge_kernel(LogProbs p, int world, int rows) {
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x, words = kHead + p.given + 2 * p.top, step = rows * words;
  pdl_enter();
  const uint32_t* const part = p.parts + row * words;
  const float c = p.inv_t * 1.4426950408889634f;
  Stats all = {-INFINITY, 0.0f, 0.0f, 0.0f};
  for (int w = 0; w < world; ++w)
    all = join(all, {__uint_as_float(part[w * step]), __uint_as_float(part[w * step + 1]), __uint_as_float(part[w * step + 2]),
                     __uint_as_float(part[w * step + 3])}, c);
  if (p.top > 0) {
    const int warp = tid >> 5;
    if (tid == 0) sh.have = 0;
    for (int w0 = 0; w0 < world; w0 += kWarps) {  // a warp a slice's list
      if (w0 + warp < world)
        note_list(sh, warp, p.top, [](const void* from, int i, int top) {
          const uint32_t* const list = static_cast<const uint32_t*>(from);
          return list[i] == 0 ? Key(0) : key_of(list[i], list[top + i]);
        }, part + (w0 + warp) * step + kHead + p.given);
      else if ((tid & 31) == 0) sh.counts[warp] = 0;
      rank_keys<false>(sh, p.top, true);
    }
  }
  finish(p, sh, all, row, [&](int i) {
    uint32_t logit = kAbsent;
    for (int w = 0; w < world; ++w) {
      const uint32_t theirs = part[w * step + kHead + i];
      if (theirs != kAbsent) logit = theirs;
    }
    return __uint_as_float(logit);
  });
}

int32_t check_log_probs(const char* who, int32_t rows, int32_t vocab, int32_t given, int32_t top, float temperature, const void* tokens) {
  if (rows < 0 || given < 0 || vocab <= 0) return fail(IVB_EINVAL, "%s: rows %d, vocabulary %d, %d tokens a row", who, rows, vocab, given);
  if (top < 0 || top > kMostTop) return fail(IVB_EINVAL, "%s: top %d (0 to %d)", who, top, kMostTop);
  if (!(temperature >= 1e-30f) || !(temperature <= 1e30f)) return fail(IVB_EINVAL, "%s: temperature %g", who, temperature);
  if (given > 0 && rows > 0 && tokens == nullptr) return fail(IVB_EINVAL, "%s: null tokens", who);
  return IVB_OK;
}

template <typename T, bool kTop>
int32_t launch(const LogProbs& p, int rows, cudaStream_t stream) {
  // a cluster a row where the rows alone leave places on the GPU's SMs, four CTAs each, and the parts are a turn at least
  int C = 1;
  while (C < 8 && static_cast<int64_t>(rows) * C * 2 <= 148 * 4 && static_cast<int64_t>(C) * kSpan < p.vocab) C *= 2;
  if (static_cast<int64_t>(rows) * C > 0x7fffffff) return fail(IVB_EINVAL, "ivb_log_probs: %d rows in one call", rows);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * C));
  cfg.blockDim = dim3(kLogThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(C);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  IVB_CUDA(cudaLaunchKernelEx(&cfg, log_probs_kernel<T, kTop>, p));
  return IVB_OK;
}

template <typename T>
int32_t launch(const LogProbs& p, int rows, cudaStream_t stream) {
  return p.top > 0 ? launch<T, true>(p, rows, stream) : launch<T, false>(p, rows, stream);
}

int32_t log_probs_call(const char* who, LogProbs p, int32_t dtype, int32_t rows, cudaStream_t stream) {
  if (dtype != IVB_F32 && dtype != IVB_F16 && dtype != IVB_BF16) return fail(IVB_EINVAL, "%s: type %d", who, dtype);
  if (p.stride < 0) return fail(IVB_EINVAL, "%s: stride %lld", who, static_cast<long long>(p.stride));
  if (rows == 0) return IVB_OK;
  if (p.logits == nullptr) return fail(IVB_EINVAL, "%s: null logits", who);
  if (dtype == IVB_F32) return launch<float>(p, rows, stream);
  if (dtype == IVB_F16) return launch<__half>(p, rows, stream);
  return launch<__nv_bfloat16>(p, rows, stream);
}

}  // namespace
}  // namespace ivb

extern "C" {

int32_t ivb_log_probs(const void* logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t stride, const int64_t* tokens, int32_t given,
                      float temperature, int32_t top, float* token_lp, float* entropy, float* top_lp, int64_t* top_ids, void* stream) {
  using namespace ivb;
  if (int32_t rc = check_log_probs("ivb_log_probs", rows, vocab, given, top, temperature, tokens)) return rc;
  if (top > vocab) return fail(IVB_EINVAL, "ivb_log_probs: top %d of a vocabulary of %d", top, vocab);
  if (rows > 0 && (entropy == nullptr || (given > 0 && token_lp == nullptr) || (top > 0 && (top_lp == nullptr || top_ids == nullptr))))
    return fail(IVB_EINVAL, "ivb_log_probs: null output");
  return log_probs_call("ivb_log_probs", {logits, tokens, stride, vocab, given, top, 0, 1.0f / temperature, token_lp, entropy, top_lp, top_ids, nullptr},
                        dtype, rows, static_cast<cudaStream_t>(stream));
}

int32_t ivb_log_probs_slice(const void* logits, int32_t dtype, int32_t rows, int32_t vloc, int32_t v0, int64_t stride, const int64_t* tokens,
                            int32_t given, float temperature, int32_t top, uint32_t* parts, void* stream) {
  using namespace ivb;
  if (int32_t rc = check_log_probs("ivb_log_probs_slice", rows, vloc, given, top, temperature, tokens)) return rc;
  if (v0 < 0 || v0 > 0x7fffffff - vloc) return fail(IVB_EINVAL, "ivb_log_probs_slice: %d tokens from %d on", vloc, v0);
  if (rows > 0 && parts == nullptr) return fail(IVB_EINVAL, "ivb_log_probs_slice: null output");
  return log_probs_call("ivb_log_probs_slice", {logits, tokens, stride, vloc, given, top, v0, 1.0f / temperature, nullptr, nullptr, nullptr, nullptr, parts},
                        dtype, rows, static_cast<cudaStream_t>(stream));
}

int32_t ivb_log_probs_merge(const uint32_t* parts, int32_t world, int32_t rows, int32_t given, float temperature, int32_t top, float* token_lp,
                            float* entropy, float* top_lp, int64_t* top_ids, void* stream) {
  using namespace ivb;
  if (int32_t rc = check_log_probs("ivb_log_probs_merge", rows, 1, given, top, temperature, reinterpret_cast<const void*>(1))) return rc;
  if (world <= 0) return fail(IVB_EINVAL, "ivb_log_probs_merge: %d slices", world);
  if (rows == 0) return IVB_OK;
  if (parts == nullptr || entropy == nullptr || (given > 0 && token_lp == nullptr) || (top > 0 && (top_lp == nullptr || top_ids == nullptr)))
    return fail(IVB_EINVAL, "ivb_log_probs_merge: null argument");
  const LogProbs p = {nullptr, nullptr, 0, 0, given, top, 0, 1.0f / temperature, token_lp, entropy, top_lp, top_ids, const_cast<uint32_t*>(parts)};
  IVB_CUDA(launch_pdl(log_probs_merge_kernel, dim3(static_cast<unsigned>(rows)), dim3(kLogThreads), 0, static_cast<cudaStream_t>(stream), p,
                      static_cast<int>(world), static_cast<int>(rows)));
  return IVB_OK;
}

}  // extern "C"
