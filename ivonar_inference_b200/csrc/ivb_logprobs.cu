// Log probabilities of given tokens, the entropy and the likeliest alternatives of rows of logits x under p = softmax(x / T):
//   log p_i = (x_i - M) / T - ln S,   M = max x,  S = sum_i e^((x_i - M) / T)
//   entropy = -sum_i p_i ln p_i = ln S - (sum_i d_i e^d_i) / S,   d_i = (x_i - M) / T
// One pass: a thread keeps M, S and the third sum of what it has seen, rescaled when M rises, 16 values at a time; these meet over
// lanes, warps, the CTAs of a cluster that share a row, and the ranks that share a vocabulary. Differences are taken before they
// are scaled, so that a row of the type's lowest value is the uniform distribution that it stands for.
//
// The `top` largest ride along: after a CTA's first 4096 values the top-th largest of its threads' maxima bounds them from
// below, what lies above is noted in shared memory (a test of each thread's maximum of 16, which the sums need anyway), and only
// those few are ranked. Values are compared as they came, ties by the token, through one 64-bit key; NaN counts as -inf there.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "ivb_common.h"
#include "ivb_device.cuh"
#include "ivb_kv4.cuh"

namespace ivb {
namespace {

namespace cg = cooperative_groups;

constexpr int kLogThreads = 256, kMostTop = 256, kBatch = 16;  // values of a thread at a time
constexpr int kSpan = kLogThreads * kBatch, kNoted = kSpan + 1024;
constexpr int kRankAll = 512;  // so many are ranked each against all; more are first cut to the largest `top`
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
  uint32_t* parts;  // of a slice, in place of the others: M, S, sum, tokens' logits, keys, ids
};

struct Stats {
  float m, s, t;  // t in units of log2
};

// Ascending with x; -0 as +0 and NaN as -inf.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x == x ? x + 0.0f : -INFINITY);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
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
  const float da = a.m == r.m ? 0.0f : fmaxf((a.m - r.m) * c, kLeast), db = b.m == r.m ? 0.0f : fmaxf((b.m - r.m) * c, kLeast);
  const float fa = exp2_of(da), fb = exp2_of(db);
  r.s = fmaf(a.s, fa, b.s * fb);
  r.t = fmaf(fmaf(a.s, da, a.t), fa, fmaf(b.s, db, b.t) * fb);
  return r;
}

struct Shared {
  Key noted[kNoted];
  Key best[kMostTop], cut[kMostTop];
  uint32_t maxima[kLogThreads];
  Stats warps[kLogThreads / 32], all;
  int count, found;
  float bound;
  int counts[2];
};

// The `top` largest of noted[0, n) into best[0, top), descending, zeros behind them. All threads; barriers on both sides.
__device__ void rank_keys(Shared& sh, int n, int top) {
  const int tid = threadIdx.x;
  const Key* from = sh.noted;
  __syncthreads();
  if (n > kRankAll) {
    // the top-th largest key, bit by bit: the largest value that at least `top` keys reach
    Key at = 0;
    if (tid < 2) sh.counts[tid] = 0;
    __syncthreads();
    for (int bit = 63; bit >= 0; --bit) {
      const Key trial = at | Key(1) << bit;
      int mine = 0;
      for (int i = tid; i < n; i += kLogThreads) mine += sh.noted[i] >= trial;
      mine = __reduce_add_sync(0xFFFFFFFFu, mine);
      if ((tid & 31) == 0 && mine != 0) atomicAdd(&sh.counts[bit & 1], mine);
      __syncthreads();
      if (sh.counts[bit & 1] >= top) at = trial;
      if (tid == 0) sh.counts[(bit & 1) ^ 1] = 0;
      __syncthreads();
    }
    if (tid == 0) sh.found = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kLogThreads)
      if (sh.noted[i] >= at) sh.cut[atomicAdd(&sh.found, 1)] = sh.noted[i];  // keys differ: `top` of them
    __syncthreads();
    from = sh.cut;
    n = top;
  }
  for (int i = tid; i < n; i += kLogThreads) {
    const Key k = from[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += from[j] > k;
    if (above < top) sh.best[above] = k;
  }
  for (int i = n + tid; i < top; i += kLogThreads) sh.best[i] = 0;
  __syncthreads();
}

// What one row's sums and largest keys say; all threads of a CTA.
template <typename F>
__device__ __forceinline__ void finish(const LogProbs& p, const Shared& sh, Stats all, int64_t row, F token_logit) {
  const int tid = threadIdx.x;
  const float ln_s = all.s > 0.0f ? logf(all.s) : __uint_as_float(0x7fffffffu);  // nothing but -inf: no distribution
  if (tid == 0) p.entropy[row] = ln_s - all.t / all.s * 0.6931471805599453f;
  for (int i = tid; i < p.given; i += kLogThreads) p.token_lp[row * p.given + i] = fmaf(token_logit(i) - all.m, p.inv_t, -ln_s);
  for (int i = tid; i < p.top; i += kLogThreads) {
    p.top_lp[row * p.top + i] = fmaf(unordered(static_cast<uint32_t>(sh.best[i] >> 32)) - all.m, p.inv_t, -ln_s);
    p.top_ids[row * p.top + i] = id_of(sh.best[i]);
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
  auto first_of = [&](int chunk) { return static_cast<int64_t>(chunk) * E - shift; };
  auto load = [&](int turn, uint4 (&to)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t chunk = static_cast<int64_t>(c0) + (static_cast<int64_t>(turn) * U + u) * kLogThreads + tid;
      const int64_t i0 = chunk * E - shift;
      if (chunk < c1 && i0 >= 0 && i0 + E <= p.vocab) {
        to[u] = __ldcs(reinterpret_cast<const uint4*>(x + i0));
      } else {
        union {
          uint4 w;
          T t[E];
        } e;
#pragma unroll
        for (int i = 0; i < E; ++i) e.t[i] = chunk < c1 && i0 + i >= 0 && i0 + i < p.vocab ? x[i0 + i] : from_f32<T>(-INFINITY);
        to[u] = e.w;
      }
    }
  };
  Stats mine = {-INFINITY, 0.0f, 0.0f};
  float bound = -INFINITY;
  if (kTop && tid == 0) sh.count = 0;
  uint4 next[U];
  if (turns > 0) load(0, next);
  for (int turn = 0; turn < turns; ++turn) {
    float v[kBatch];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      union {
        uint4 w;
        T t[E];
      } e;
      e.w = next[u];
#pragma unroll
      for (int i = 0; i < E; ++i) v[u * E + i] = to_f32<T>(e.t[i]);
    }
    if (turn + 1 < turns) load(turn + 1, next);
    float most = v[0];
#pragma unroll
    for (int i = 1; i < kBatch; ++i) most = fmaxf(most, v[i]);
    most = fmaxf(most, -INFINITY);  // 16 NaN
    if (most > mine.m) mine = join(mine, {most, 0.0f, 0.0f}, c);
    const float m = mine.m == -INFINITY ? 0.0f : mine.m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float d = (v[i] - m) * c, e = exp2_of(d);
      mine.s += e;
      mine.t = fmaf(fmaxf(d, kLeast), e, mine.t);
    }
    if constexpr (kTop) {
      auto note = [&](bool all) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const int chunk = c0 + (turn * U + u) * kLogThreads + tid;
            const int64_t id = first_of(chunk) + i;
            const float y = v[u * E + i] == v[u * E + i] ? v[u * E + i] : -INFINITY;
            if (chunk < c1 && id >= 0 && id < p.vocab && (all ? y >= bound : y > bound))
              sh.noted[atomicAdd(&sh.count, 1)] = key_of(ordered(y), static_cast<uint32_t>(id + p.v0));
          }
      };
      if (turn == 0) {
        sh.maxima[tid] = ordered(most);
        __syncthreads();
        int above = 0;
        const uint32_t own = sh.maxima[tid];
        for (int j = 0; j < kLogThreads; j += 4) {
          const uint4 o = *reinterpret_cast<const uint4*>(sh.maxima + j);
          above += (o.x > own || (o.x == own && j < tid)) + (o.y > own || (o.y == own && j + 1 < tid)) + (o.z > own || (o.z == own && j + 2 < tid)) +
                   (o.w > own || (o.w == own && j + 3 < tid));
        }
        if (above == p.top - 1) sh.bound = most;
        __syncthreads();
        bound = sh.bound;
        if (most >= bound) note(true);
      } else if (most > bound) {
        note(false);  // later tokens: as large as the bound is too late
      }
      if (turn + 1 < turns) {
        __syncthreads();
        const int n = sh.count;
        if (n > kNoted - kSpan) {  // the next turn could note more than there is room for
          rank_keys(sh, n, p.top);
          for (int i = tid; i < p.top; i += kLogThreads) sh.noted[i] = sh.best[i];
          bound = unordered(static_cast<uint32_t>(sh.best[p.top - 1] >> 32));
          if (tid == 0) sh.count = p.top;
          __syncthreads();
        }
      }
    }
  }
  // over lanes, warps and the cluster
#pragma unroll
  for (int d = 1; d < 32; d <<= 1)
    mine = join(mine, {__shfl_xor_sync(0xFFFFFFFFu, mine.m, d), __shfl_xor_sync(0xFFFFFFFFu, mine.s, d), __shfl_xor_sync(0xFFFFFFFFu, mine.t, d)}, c);
  if (lane == 0) sh.warps[warp] = mine;
  __syncthreads();
  Stats all = sh.warps[0];
#pragma unroll
  for (int w = 1; w < kLogThreads / 32; ++w) all = join(all, sh.warps[w], c);
  if constexpr (kTop) rank_keys(sh, sh.count, p.top);
  if (C > 1) {
    if (tid == 0) sh.all = all;
    cluster.sync();
    if (rank == 0) {
      for (int k = 1; k < C; ++k) all = join(all, cluster.map_shared_rank(&sh, k)->all, c);
      if constexpr (kTop) {
        if (tid == 0) sh.count = 0;
        __syncthreads();
        for (int i = tid; i < C * p.top; i += kLogThreads) {
          const Key k = cluster.map_shared_rank(&sh, i / p.top)->best[i % p.top];
          if (k != 0) sh.noted[atomicAdd(&sh.count, 1)] = k;
        }
        __syncthreads();
        rank_keys(sh, sh.count, p.top);
      }
    }
    cluster.sync();  // no CTA leaves while another reads its shared memory
    if (rank != 0) return;
  }
  if (p.parts == nullptr) {
    finish(p, sh, all, row, [&](int i) { return logit_of_token<T>(p, row, i); });
    return;
  }
  uint32_t* const out = p.parts + row * (3 + p.given + 2 * p.top);
  if (tid == 0) {
    out[0] = __float_as_uint(all.m);
    out[1] = __float_as_uint(all.s);
    out[2] = __float_as_uint(all.t);
  }
  for (int i = tid; i < p.given; i += kLogThreads) out[3 + i] = __float_as_uint(logit_of_token<T>(p, row, i));
  for (int i = tid; i < p.top; i += kLogThreads) {
    out[3 + p.given + i] = static_cast<uint32_t>(sh.best[i] >> 32);
    out[3 + p.given + p.top + i] = id_of(sh.best[i]);
  }
}

// The slices' parts [world][rows][3 + given + 2 top] of a row.
__global__ void __launch_bounds__(kLogThreads) log_probs_merge_kernel(LogProbs p, int world, int rows) {
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x, words = 3 + p.given + 2 * p.top, step = rows * words;
  pdl_enter();
  const uint32_t* const part = p.parts + row * words;
  const float c = p.inv_t * 1.4426950408889634f;
  Stats all = {-INFINITY, 0.0f, 0.0f};
  for (int w = 0; w < world; ++w)
    all = join(all, {__uint_as_float(part[w * step]), __uint_as_float(part[w * step + 1]), __uint_as_float(part[w * step + 2])}, c);
  if (p.top > 0) {
    int have = 0;
    for (int w0 = 0; w0 < world;) {
      const int n = min(world - w0, (kNoted - have) / p.top);
      if (tid == 0) sh.count = have;
      __syncthreads();
      for (int i = tid; i < n * p.top; i += kLogThreads) {
        const uint32_t* from = part + (w0 + i / p.top) * step + 3 + p.given + i % p.top;
        if (from[0] != 0) sh.noted[atomicAdd(&sh.count, 1)] = key_of(from[0], from[p.top]);
      }
      __syncthreads();
      have = min(sh.count, p.top);
      rank_keys(sh, sh.count, p.top);
      for (int i = tid; i < p.top; i += kLogThreads) sh.noted[i] = sh.best[i];
      w0 += n;
      __syncthreads();
    }
  }
  finish(p, sh, all, row, [&](int i) {
    uint32_t logit = kAbsent;
    for (int w = 0; w < world; ++w) {
      const uint32_t theirs = part[w * step + 3 + i];
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
  while (C < 8 && static_cast<int64_t>(rows) * C < 148 * 4 && static_cast<int64_t>(C) * kSpan < p.vocab) C *= 2;
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
