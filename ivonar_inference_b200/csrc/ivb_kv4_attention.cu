// Causal attention over the 4-bit key/value cache, with a sliding window and visible first tokens (sinks): few rows a sequence
// (the prompts are in ivb_kv4_prompt.cu), and the entry point.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "ivb_kv4_attention.cuh"

namespace ivb {

int32_t check_kv4(const IvbKv4Cache* c, const char* who);
int32_t check_kv4_rows(const IvbKv4Cache* c, const int32_t* starts, const int64_t* positions, int32_t rows, int32_t dtype, const char* who);

namespace {

namespace cg = cooperative_groups;

// Sequences of up to so many items (tokens x query heads of a group) are for the kernel of few rows, which splits a history over
// more of the GPU; the others for the prompts' one, which reads it once for 256 items. Measured (rows / prompts): where the
// prompts' tiles are many, 32 items 57 / 84 us and 42 / 67 (16 sequences, 16 heads x 64, 2000 positions, fp32 and fp16), 44 / 53 (8
// sequences, 8 heads x 128, 4000 positions, bf16), 48 items 60 / 67 and 64 / 54 (those two in 16 bits), 116 / 101 (64 sequences, 8 heads
// x 128, 1000 positions); where they are few, 64 items 111 / 138 and 96 items 177 / 138 (2 sequences, 8 heads x 128, 30000 positions,
// bf16), 64 items 86 / 163 and 100 items 195 / 165 (8 heads x 64, fp32).
constexpr int kFewItems = 32, kFewItemsSparse = 64;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<unsigned>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}
// ---- few rows: one token per sequence, a few drafted ones, or any number in tiles -----------------------------------------
// One cluster of C CTAs of W warps per (sequence, key/value head, tile of rows); row i of a sequence's head group is token
// i / group, query head i % group of the group. The 32-position groups of the cache that a row of the tile sees are dealt
// out to the cluster's warps in turn; each warp streams its own through a ring of cp.async stages and joins what it found
// with the others' in shared memory, then over the cluster's.
//
// The codes are the A operands, 16 positions (keys) or 16 channels (values) a product, and the rows are the columns of B: with
// one to four rows half the products of the other order are needed, and half its accumulators. Scores leave the
// first product as positions x rows in the C layout; an 8x8 transposition (movmatrix) makes them the second one's B.
// Columns hold, per tile of 8: kSplit 4 rows, each as the fp16 of its values and next to it the remainder's; else 8 rows.
// fp32 outputs: the tensor cores cut what they add to an accumulator towards zero, so every 16 groups (512 positions) it is added to
// its sums in shared memory, rounding to nearest, and begins anew.
constexpr int kFoldSteps = 16;

template <int D, typename T, bool kSplit, int kTiles>
struct RowsGeometry {
  static constexpr bool fold = std::is_same<T, float>::value;
  static constexpr int rows = (kSplit ? 4 : 8) * kTiles;
  static constexpr int stages = D == 128 ? 2 : 3;
  static constexpr int group_bytes = kKv4Group * (D + 8);
  static constexpr int warp_bytes = stages * group_bytes;
  static constexpr int comb_floats = rows * D + 3 * rows;
  static constexpr int term_bytes = kKv4Group * 24;  // a float4 and a float2 for each position
  static constexpr int fold_bytes = fold ? rows * D * 4 : 0;
  static constexpr int smem(int warps) { return warps * (warp_bytes + term_bytes + rows * 12 + fold_bytes) + comb_floats * 4; }
};

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int D, typename T, bool kSplit, int kTiles, bool kShared>
__device__ __forceinline__ void kv4_rows(const Kv4Attention& A, int tiles_per_sequence) {
  using G = RowsGeometry<D, T, kSplit, kTiles>;
  constexpr int R = G::rows, kSteps = D / 16, kTile = kv4_tile_bytes(D);
  constexpr int kPer = kSplit ? 1 : 2;        // rows of a lane in a column tile
  constexpr int kSets = kPer * kTiles;        // rows of a lane
  constexpr int kOut = D / 16;                // 16-channel tiles of the output
  extern __shared__ __align__(128) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank()), W = blockDim.x >> 5;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  unsigned char* const ring = smem + warp * G::warp_bytes;
  float4* const terms4 = reinterpret_cast<float4*>(smem + W * G::warp_bytes + warp * G::term_bytes);
  float2* const terms2 = reinterpret_cast<float2*>(terms4 + kKv4Group);
  float* const comb = reinterpret_cast<float*>(smem + W * (G::warp_bytes + G::term_bytes));  // [R][D], then ref, sum, offset [R]
  float* const stats = comb + G::comb_floats;                                               // [W][R][3]
  float* const folded = stats + W * R * 3 + warp * R * D;                                    // [R][D], fp32 outputs only

  if (A.beside_prompts) __threadfence();
  else pdl_wait();
  pdl_trigger();
  // which rows (rows x heads is below 2^31)
  const unsigned cluster_id = blockIdx.x / static_cast<unsigned>(C), group_size = static_cast<unsigned>(A.group);
  const int tile = static_cast<int>(cluster_id % static_cast<unsigned>(tiles_per_sequence));
  const unsigned sh = cluster_id / static_cast<unsigned>(tiles_per_sequence);
  const int b = static_cast<int>(sh / static_cast<unsigned>(A.cache.kv_heads)), kvh = static_cast<int>(sh) - b * A.cache.kv_heads;
  int row0 = b, count = 1;
  int64_t before = 0;  // rows of the sequence that the call does not have
  if (A.starts != nullptr) {
    row0 = max(0, A.starts[b]);
    before = static_cast<int64_t>(row0) - A.starts[b];
    count = min(A.rows, A.starts[b + 1]) - row0;
  }
  const int items = max(count, 0) * A.group, i0 = tile * R;
  if (i0 >= items || items > A.few) return;  // the whole cluster
  const int live = min(R, items - i0);
  const int64_t base = kv4_position(A.positions, b) + before;
  const int max_len = A.cache.max_len;
  // a beginning that the sequence shares: joined from its parts at the end, or walked here, at positions below zero
  int prefix_group = 0;
  const int shared_length = kShared ? kv4_prefix(A, b, prefix_group) : 0, sinks = kShared ? A.sinks - shared_length : A.sinks;
  const bool joined = kShared && shared_length > 0 && A.part_stats != nullptr, walked = kShared && shared_length > 0 && !joined;
  // token and query head of an item of the sequence's head group
  auto token_of = [&](int i) { return static_cast<int>(static_cast<unsigned>(i) / group_size); };
  // positions of the tile's first and last rows, -1 where idle and max_len where beyond the capacity
  auto clamp_position = [&](int64_t p) { return static_cast<int>(max(static_cast<int64_t>(-1), min(p, static_cast<int64_t>(max_len)))); };
  const int first = clamp_position(base + token_of(i0)), last = clamp_position(base + token_of(i0 + live - 1));
  // row of the tile that set s of this lane holds, and its position (-1: sees nothing)
  auto row_of = [&](int s) { return kSplit ? 4 * s + c : 8 * (s >> 1) + 2 * c + (s & 1); };
  int at[kSets];
#pragma unroll
  for (int s = 0; s < kSets; ++s) {
    const int p = clamp_position(base + token_of(i0 + row_of(s)));
    at[s] = row_of(s) < live && p < max_len ? p : -1;
  }
  if (last >= max_len && threadIdx.x == 0 && rank == 0 && A.error != nullptr) atomicCAS(A.error, 0u, static_cast<unsigned>(IVB_ECAPACITY));
  // the groups of 32 positions that some row sees: the sinks' below the window, then the window's
  const int high = min(last, max_len - 1);  // negative: none
  const int low = A.window > 0 ? max(0, max(first, 0) - A.window + 1) : 0;
  const int window_group = low / kKv4Group;
  const int sink_groups = A.window > 0 ? min((min(kShared ? max(0, sinks) : sinks, low) + kKv4Group - 1) / kKv4Group, window_group) : 0;
  const int own_groups = high < 0 ? 0 : sink_groups + high / kKv4Group - window_group + 1;
  int shared_groups = 0, shared_sinks = 0, shared_window = 0;  // of the beginning, before these
  if (walked && own_groups > 0) {
    const int all = (shared_length + kKv4Group - 1) / kKv4Group, from = A.window > 0 ? max(0, max(first, 0) + shared_length - A.window + 1) : 0;
    shared_window = min(from / kKv4Group, all);
    shared_sinks = A.window > 0 ? min((min(A.sinks, from) + kKv4Group - 1) / kKv4Group, shared_window) : 0;
    shared_groups = shared_sinks + all - shared_window;
  }
  const int groups = shared_groups + own_groups;
  const int lanes_in = C * W, mine = rank * W + warp;
  const int steps = groups > mine ? (groups - mine + lanes_in - 1) / lanes_in : 0;

  const unsigned char* const codes = static_cast<const unsigned char*>(A.cache.data) +
                                     (static_cast<int64_t>(b) * A.cache.kv_heads + kvh) * kv4_tiles(max_len) * kTile + lane * 16;
  const unsigned char* const shared_codes = static_cast<const unsigned char*>(A.prefix.data) +
                                            (static_cast<int64_t>(prefix_group) * A.cache.kv_heads + kvh) * kv4_tiles(A.prefix.max_len) * kTile + lane * 16;
  auto of_prefix = [&](int step) { return kShared && mine + step * lanes_in < shared_groups; };
  auto group_of = [&](int step) {  // in its cache
    int i = mine + step * lanes_in;
    if (of_prefix(step)) return i < shared_sinks ? i : shared_window + i - shared_sinks;
    if constexpr (kShared) i -= shared_groups;
    return i < sink_groups ? i : window_group + i - sink_groups;
  };
  auto issue = [&](int step, int stage) {
    if (step < steps) {
      const unsigned char* src = (of_prefix(step) ? shared_codes : codes) + static_cast<int64_t>(group_of(step)) * G::group_bytes;
      unsigned char* dst = ring + stage * G::group_bytes + lane * 16;
#pragma unroll
      for (int o = 0; o < G::group_bytes; o += 512)
        if (o + 512 <= G::group_bytes || lane * 16 < G::group_bytes - o) cp_async16(dst + o, src + o);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < G::stages - 1; ++s) issue(s, s);

  // queries as B fragments (this lane: column r, channels D/4 c .. of its row), each row scaled by the power of two that brings its
  // largest to 2^13, so that no row's bits depend on its neighbours; row_unit undoes it. Idle rows' queries are not read.
  uint32_t qf[kTiles][kSteps][2];
  float sum_q[kSets], row_unit[kSets];
  {
    float total[kTiles], unit[kTiles];
    const float scale = A.scale * kLog2e;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      const int row = kSplit ? 4 * n + (r >> 1) : 8 * n + r;
      float qv[D / 4];
#pragma unroll
      for (int j = 0; j < D / 4; ++j) qv[j] = 0.0f;
      const int t = token_of(i0 + row), p = clamp_position(base + t);
      if (row < live && p >= 0 && p < max_len)
        load_values<T, D / 4>(static_cast<const T*>(A.q) + (row0 + t) * A.q_row + (kvh * A.group + i0 + row - t * A.group) * A.q_head + D / 4 * c,
                              A.q_vec, qv);
      float amax = 0.0f;
#pragma unroll
      for (int j = 0; j < D / 4; ++j) amax = fmaxf(amax, finite_size(qv[j]));
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
      const int up = query_power(amax);
      const float q_unit = power_of_two(up);
      unit[n] = power_of_two(-up) * scale;
      total[n] = 0.0f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x0 = qv[4 * s + 2 * e] * q_unit, x1 = qv[4 * s + 2 * e + 1] * q_unit;
          total[n] = total[n] + x0 + x1;
          uint32_t w = pack_f16(x0, x1);
          if (kSplit && (r & 1)) {
            const float2 hi = unpack_f16(w);
            w = pack_f16(x0 - hi.x, x1 - hi.y);
          }
          qf[n][s][e] = w;
        }
      total[n] += __shfl_xor_sync(0xFFFFFFFFu, total[n], 1);
      total[n] += __shfl_xor_sync(0xFFFFFFFFu, total[n], 2);
    }
#pragma unroll
    for (int s = 0; s < kSets; ++s) {  // from the lanes that hold the row as a column
      const int from = kSplit ? 8 * c : 4 * (2 * c + (s & 1));
      row_unit[s] = __shfl_sync(0xFFFFFFFFu, unit[kSplit ? s : s >> 1], from);
      sum_q[s] = __shfl_sync(0xFFFFFFFFu, total[kSplit ? s : s >> 1], from) * row_unit[s];
    }
  }

  float acc[kTiles][kOut][4];
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int i = 0; i < kOut; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.0f;
  float ref[kSets], sum[kSets], off[kSets];
#pragma unroll
  for (int s = 0; s < kSets; ++s) {
    ref[s] = -INFINITY;
    sum[s] = off[s] = 0.0f;
  }

  constexpr int kPlanes = D == 128 ? 2 : 1, kRun = D == 32 ? 4 : 8;  // channels of a lane in a plane of 64 (or 32)
  // channel of value j: D = 32: 8 (r / 2) + r % 2 + 2 j, else 64 plane + 8 r + j
  auto channel = [&](int h, int j) { return D == 32 ? 8 * (r >> 1) + (r & 1) + 2 * j : 64 * h + 8 * r + j; };
  float o[kSets][kPlanes][kRun];
  float folded_ref[kSets];  // the reference that the sums in shared memory stand at, -inf: none yet
#pragma unroll
  for (int s = 0; s < kSets; ++s) folded_ref[s] = -INFINITY;
  bool any_folded = false;
  // the accumulators joined with what was folded before: into o at the end, into shared memory (each lane its own places) else
  auto fold = [&](bool last) {
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      const float f = folded_ref[s] == -INFINITY ? 0.0f : ex2(folded_ref[s] - ref[s]);
#pragma unroll
      for (int h = 0; h < kPlanes; ++h)
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          const int i = 4 * h + (j >> 1), e = 2 * (j & 1);
          float v;
          if constexpr (kSplit) v = acc[s][i][e] + acc[s][i][e + 1];
          else v = acc[s >> 1][i][e + (s & 1)];
          v *= 0.00006103515625f;  // the weights' 2^14
          if (any_folded) v = fmaf(folded[row_of(s) * D + channel(h, j)], f, v);
          if (last) o[s][h][j] = v;
          else folded[row_of(s) * D + channel(h, j)] = v;
        }
      folded_ref[s] = ref[s];
    }
    if (last) return;
    any_folded = true;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < kOut; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.0f;
  };

  const CodeMiddle key_middle = code_middle(8.0f, 8.0f), value_middle = code_middle(8.0f, 7.0f);  // halves: channels, positions
  int at_stage = 0, to_stage = G::stages - 1;
  for (int step = 0; step < steps; ++step) {
    cp_async_wait<G::stages - 2>();
    __syncwarp();
    const unsigned char* const stage = ring + at_stage * G::group_bytes;
    const bool shared = of_prefix(step);
    const int p0 = group_of(step) * kKv4Group - (shared ? shared_length : 0);
    {
      const uint2 par = *reinterpret_cast<const uint2*>(stage + (lane >> 4) * kTile + 16 * D + (lane & 15) * 8);
      const PositionTerms t = position_terms(par, 1.0f, 16384.0f, lane);
      terms4[lane] = make_float4(t.key_scale, t.key_offset, t.bias, t.mantissa);
      terms2[lane] = make_float2(t.unbias, t.value_offset);
    }
    __syncwarp();
    // scores: x[set][2 tile + half] is position p0 + 16 tile + 4 (r / 2) + r % 2 + 2 half
    const int mine_of = 4 * (r >> 1) + (r & 1);
    float x[kSets][4], mantissa[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float s2[kTiles][4];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) s2[n][0] = s2[n][1] = s2[n][2] = s2[n][3] = 0.0f;
      uint32_t w[2][D / 32];
      const uint32_t* kw = reinterpret_cast<const uint32_t*>(stage + t * kTile);
      if constexpr (D == 32) {
        const uint2 v = reinterpret_cast<const uint2*>(kw)[lane];
        w[0][0] = v.x;
        w[1][0] = v.y;
      } else if constexpr (D == 64) {
        const uint4 v = reinterpret_cast<const uint4*>(kw)[lane];
        w[0][0] = v.x;
        w[0][1] = v.y;
        w[1][0] = v.z;
        w[1][1] = v.w;
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 v = reinterpret_cast<const uint4*>(kw)[32 * h + lane];
          w[h][0] = v.x;
          w[h][1] = v.y;
          w[h][2] = v.z;
          w[h][3] = v.w;
        }
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t v0 = s & 1 ? w[0][s >> 1] >> 8 : w[0][s >> 1], v1 = s & 1 ? w[1][s >> 1] >> 8 : w[1][s >> 1];
        const uint32_t a0 = codes_low(v0, key_middle), a1 = codes_low(v1, key_middle), a2 = codes_high(v0, key_middle), a3 = codes_high(v1, key_middle);
#pragma unroll
        for (int n = 0; n < kTiles; ++n) mma_f16(s2[n], a0, a1, a2, a3, qf[n][s][0], qf[n][s][1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 pt = terms4[16 * t + mine_of + 2 * h];
        mantissa[2 * t + h] = pt.w;
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
          const float dot = kSplit ? s2[s][2 * h] + s2[s][2 * h + 1] : s2[s >> 1][2 * h + (s & 1)];
          x[s][2 * t + h] = fmaf(dot, row_unit[s] * pt.x, fmaf(sum_q[s], pt.y, pt.z));  // (dot * row_unit could overflow)
        }
      }
    }
    // a group that every row sees whole needs no masks
    const bool whole = (shared ? first >= 0 && p0 + kKv4Group <= 0 : first >= p0 + kKv4Group - 1) && last < max_len && (A.window <= 0 || p0 > last - A.window || p0 <= sinks - kKv4Group);
    if (!whole) {
#pragma unroll
      for (int s = 0; s < kSets; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int p = p0 + 16 * (i >> 1) + mine_of + 2 * (i & 1);
          const bool seen = (shared ? p < 0 && at[s] >= 0 : p <= at[s]) && (A.window <= 0 || p > at[s] - A.window || p < sinks);
          if (!seen) x[s][i] = -INFINITY;
        }
    }
    bool raise = false;
    float next[kSets];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      float m = fmaxf(fmaxf(x[s][0], x[s][1]), fmaxf(x[s][2], x[s][3]));
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
      next[s] = fmaxf(ref[s], m);
      raise |= next[s] > ref[s];
    }
    if (__any_sync(0xFFFFFFFFu, raise)) {
#pragma unroll
      for (int s = 0; s < kSets; ++s) {
        const float corr = next[s] > ref[s] ? ex2(ref[s] - next[s]) : 1.0f;
        ref[s] = next[s];
        sum[s] *= corr;
        off[s] *= corr;
#pragma unroll
        for (int i = 0; i < kOut; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if constexpr (kSplit) {
              acc[s][i][2 * j] *= corr;
              acc[s][i][2 * j + 1] *= corr;
            } else {
              acc[s >> 1][i][2 * j + (s & 1)] *= corr;
            }
          }
      }
    }
    float from[kSets];  // a row that has seen nothing yet: any number, so that its weights are 2^-inf
#pragma unroll
    for (int s = 0; s < kSets; ++s) from[s] = ref[s] == -INFINITY ? 0.0f : ref[s];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t bw[kTiles][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 pt = terms2[16 * t + mine_of + 2 * h];
        float wgt[kSets];
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
          const float pw = ex2(x[s][2 * t + h] - from[s]);
          sum[s] = fmaf(pw, pt.x, sum[s]);
          off[s] = fmaf(pw, pt.y, off[s]);
          wgt[s] = pw * mantissa[2 * t + h];
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          if constexpr (kSplit) {
            const __half hi = __float2half_rn(wgt[n]);
            const __half2 both = __halves2half2(hi, __float2half_rn(wgt[n] - __half2float(hi)));
            bw[n][h] = transpose8(*reinterpret_cast<const uint32_t*>(&both));
          } else {
            bw[n][h] = transpose8(pack_f16(wgt[2 * n], wgt[2 * n + 1]));
          }
        }
      }
      const uint4* vw = reinterpret_cast<const uint4*>(stage + t * kTile + 8 * D);
      if constexpr (D == 32) {
        const uint4 v = vw[4 * (r >> 1) + c];
        const unsigned sel = r & 1 ? 0x7632u : 0x5410u;
        const uint32_t x01 = __byte_perm(v.x, v.y, sel), x23 = __byte_perm(v.z, v.w, sel);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t y01 = i ? x01 >> 8 : x01, y23 = i ? x23 >> 8 : x23;
          const uint32_t a0 = codes_low(y01, value_middle), a1 = codes_high(y01, value_middle);
          const uint32_t a2 = codes_low(y23, value_middle), a3 = codes_high(y23, value_middle);
#pragma unroll
          for (int n = 0; n < kTiles; ++n) mma_f16(acc[n][i], a0, a1, a2, a3, bw[n][0], bw[n][1]);
        }
      } else {
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          const uint4 v = vw[32 * h + lane];
          uint32_t l01 = __byte_perm(v.x, v.y, 0x5410u), l23 = __byte_perm(v.z, v.w, 0x5410u);
          uint32_t h01 = __byte_perm(v.x, v.y, 0x7632u), h23 = __byte_perm(v.z, v.w, 0x7632u);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i == 2) {
              l01 >>= 8;
              l23 >>= 8;
              h01 >>= 8;
              h23 >>= 8;
            }
            const uint32_t a0 = i & 1 ? codes_high(l01, value_middle) : codes_low(l01, value_middle), a1 = i & 1 ? codes_high(h01, value_middle) : codes_low(h01, value_middle);
            const uint32_t a2 = i & 1 ? codes_high(l23, value_middle) : codes_low(l23, value_middle), a3 = i & 1 ? codes_high(h23, value_middle) : codes_low(h23, value_middle);
#pragma unroll
            for (int n = 0; n < kTiles; ++n) mma_f16(acc[n][4 * h + i], a0, a1, a2, a3, bw[n][0], bw[n][1]);
          }
        }
      }
    }
    __syncwarp();
    if constexpr (G::fold)
      if (step % kFoldSteps == kFoldSteps - 1 && step + 1 < steps) fold(false);
    issue(step + G::stages - 1, to_stage);
    at_stage = at_stage + 1 == G::stages ? 0 : at_stage + 1;
    to_stage = to_stage + 1 == G::stages ? 0 : to_stage + 1;
  }
  cp_async_wait<0>();
  __syncwarp();

  // the lane's rows: their sums over the 8 lanes that hold other positions, and 8 neighbouring channels a plane of 64 (or 32)
#pragma unroll
  for (int s = 0; s < kSets; ++s)
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      sum[s] += __shfl_xor_sync(0xFFFFFFFFu, sum[s], d);
      off[s] += __shfl_xor_sync(0xFFFFFFFFu, off[s], d);
    }
  fold(true);
  auto place = [&](int row) {
    const int t = token_of(i0 + row);
    return static_cast<T*>(A.out) + (row0 + t) * A.o_row + (kvh * A.group + i0 + row - t * A.group) * A.o_head;
  };
  if (C * W == 1 && !joined) {
#pragma unroll
    for (int s = 0; s < kSets; ++s)
      if (row_of(s) < live) {
        T* out = place(row_of(s));
        const float inv = sum[s] == 0.0f ? 0.0f : 1.0f / sum[s];
#pragma unroll
        for (int h = 0; h < kPlanes; ++h) {
          float y[kRun];
#pragma unroll
          for (int j = 0; j < kRun; ++j) y[j] = sum[s] == 0.0f ? 0.0f : (o[s][h][j] + off[s]) * inv;
          if constexpr (D == 32) {
#pragma unroll
            for (int j = 0; j < kRun; ++j) out[channel(h, j)] = from_f32<T>(y[j]);
          } else {
            store_values<T, kRun>(out + channel(h, 0), A.o_vec, y);
          }
        }
      }
    return;
  }
  float* const part = reinterpret_cast<float*>(ring);  // the warp's ring is free
#pragma unroll
  for (int s = 0; s < kSets; ++s)
    if (row_of(s) < live) {
      if (r == 0) {
        float* st = stats + (warp * R + row_of(s)) * 3;
        st[0] = ref[s];
        st[1] = sum[s];
        st[2] = off[s];
      }
#pragma unroll
      for (int h = 0; h < kPlanes; ++h)
#pragma unroll
        for (int j = 0; j < kRun; ++j) part[row_of(s) * D + channel(h, j)] = o[s][h][j];
    }
  __syncthreads();
  // what the CTA's warps found for a row and n of its channels: values with their offset, reference and sum
  auto of_warps = [&](int row, int c0, auto& v, float& top, float& l) {
    constexpr int n = sizeof(v) / sizeof(float);
    top = -INFINITY;
    l = 0.0f;
    for (int w = 0; w < W; ++w) top = fmaxf(top, stats[(w * R + row) * 3]);
#pragma unroll
    for (int j = 0; j < n; ++j) v[j] = 0.0f;
    for (int w = 0; w < W; ++w) {
      const float* st = stats + (w * R + row) * 3;
      if (st[1] == 0.0f) continue;  // the warp saw nothing for this row
      const float f = ex2(st[0] - top);
      l = fmaf(st[1], f, l);
#pragma unroll
      for (int j = 0; j < n; ++j) v[j] = fmaf(reinterpret_cast<const float*>(smem + w * G::warp_bytes)[row * D + c0 + j] + st[2], f, v[j]);
    }
  };
  if (kShared && joined) {
    // a warp a row, D / 32 neighbouring channels a lane
    constexpr int n = D / 32;
    float* const cref = comb + R * D;
    if (C > 1) {
      for (int row = warp; row < live; row += W) {
        float v[n], top, l;
        of_warps(row, n * lane, v, top, l);
#pragma unroll
        for (int j = 0; j < n; ++j) comb[row * D + n * lane + j] = v[j];
        if (lane == 0) {
          cref[row] = top;
          cref[R + row] = l;
        }
      }
      cluster.sync();
    }
    pdl_wait();  // for the parts
    for (int row = rank + C * warp; row < live; row += C * W) {
      float v[n], top = -INFINITY, l = 0.0f;
      if (C == 1) {
        of_warps(row, n * lane, v, top, l);
      } else {
        for (int k = 0; k < C; ++k) top = fmaxf(top, cluster.map_shared_rank(comb, k)[R * D + row]);
#pragma unroll
        for (int j = 0; j < n; ++j) v[j] = 0.0f;
        for (int k = 0; k < C; ++k) {
          const float* other = cluster.map_shared_rank(comb, k);
          const float theirs = other[R * D + R + row];
          if (theirs == 0.0f) continue;
          const float f = ex2(other[R * D + row] - top);
          l = fmaf(theirs, f, l);
#pragma unroll
          for (int j = 0; j < n; ++j) v[j] = fmaf(other[row * D + n * lane + j], f, v[j]);
        }
      }
      const int p = clamp_position(base + token_of(i0 + row));
      if (p >= 0 && p < max_len) {
        const int t = token_of(i0 + row);
        kv4_join_parts<D>(A, static_cast<int64_t>(row0 + t) * A.heads + kvh * A.group + i0 + row - t * A.group, top, l, v);
      }  // an idle row: zeros
      store_values<T, n>(place(row) + n * lane, A.o_vec && n > 1, v);
    }
    if (C > 1) cluster.sync();  // no CTA leaves while another reads its shared memory
    return;
  }
  float* const cref = comb + R * D;
  for (int i = threadIdx.x; i < live * D; i += 32 * W) {
    const int row = i / D;
    float top = -INFINITY;
    for (int w = 0; w < W; ++w) top = fmaxf(top, stats[(w * R + row) * 3]);
    float v = 0.0f, l = 0.0f, m = 0.0f;
    for (int w = 0; w < W; ++w) {
      const float* st = stats + (w * R + row) * 3;
      if (st[1] != 0.0f) {  // zero: the warp saw nothing for this row
        const float f = ex2(st[0] - top);
        v = fmaf(reinterpret_cast<const float*>(smem + w * G::warp_bytes)[i], f, v);
        l = fmaf(st[1], f, l);
        m = fmaf(st[2], f, m);
      }
    }
    if (C == 1) {
      place(row)[i - row * D] = from_f32<T>(l == 0.0f ? 0.0f : (v + m) / l);
    } else {
      comb[i] = v;
      if (i - row * D == 0) {
        cref[row] = top;
        cref[R + row] = l;
        cref[2 * R + row] = m;
      }
    }
  }
  if (C == 1) return;
  cluster.sync();
  // the cluster's parts: every CTA writes its share of the rows' values
  for (int i = rank * 32 * W + threadIdx.x; i < live * D; i += C * 32 * W) {
    const int row = i / D;
    float top = -INFINITY;
    for (int k = 0; k < C; ++k) top = fmaxf(top, cluster.map_shared_rank(comb, k)[R * D + row]);
    float v = 0.0f, l = 0.0f;
    for (int k = 0; k < C; ++k) {
      const float* other = cluster.map_shared_rank(comb, k);
      const float part_sum = other[R * D + R + row];
      if (part_sum != 0.0f) {
        const float f = ex2(other[R * D + row] - top);
        v = fmaf(other[i] + other[R * D + 2 * R + row], f, v);
        l = fmaf(part_sum, f, l);
      }
    }
    place(row)[i - row * D] = from_f32<T>(l == 0.0f ? 0.0f : v / l);
  }
  cluster.sync();  // no CTA leaves while another reads its shared memory
}

// kShared: behind beginnings that the sequences share. (Told apart as it runs, 39.4 us where 38.7 are kept for 256 sequences.)
template <int D, typename T, bool kSplit, int kTiles, bool kShared>
__global__ void __launch_bounds__(256, 2) kv4_rows_kernel(Kv4Attention A, int tiles_per_sequence) {
  kv4_rows<D, T, kSplit, kTiles, kShared>(A, tiles_per_sequence);
  // whichever way the rows took: this grid does not end before the ones that it runs beside
  if (A.beside_prompts && blockIdx.x == 0) pdl_wait();
}

// Opt-in shared memory, once per device and kernel.
template <typename K>
int32_t allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  IVB_CUDA(cudaGetDevice(&device));
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if ((done.load(std::memory_order_relaxed) & bit) != 0 && bit != 0) return IVB_OK;
  IVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return IVB_OK;
}

template <int D, typename T, bool kSplit, int kTiles, bool kShared>
int32_t launch_rows_attention(const Kv4Attention& A, cudaStream_t stream) {
  using G = RowsGeometry<D, T, kSplit, kTiles>;
  constexpr int kMostWarps = 8;
  static std::atomic<uint64_t> done{0};
  if (int32_t rc = allow_smem(kv4_rows_kernel<D, T, kSplit, kTiles, kShared>, G::smem(kMostWarps), done)) return rc;
  const int64_t most = std::min<int64_t>(A.few, static_cast<int64_t>(A.starts == nullptr ? 1 : A.rows) * A.group);
  const int64_t tiles = (most + G::rows - 1) / G::rows;
  const int64_t grid = tiles * A.cache.kv_heads * A.cache.batch;
  // the tiles with rows in them, if the call's rows are spread evenly: the grid has places for each sequence's most
  const int64_t even = (static_cast<int64_t>(A.rows) * A.group + G::rows - 1) / G::rows;
  const int64_t base = std::min(tiles * A.cache.batch, std::max<int64_t>(std::min(A.rows, A.cache.batch), even)) * A.cache.kv_heads;
  // Warps a row tile by what fills the GPU twice over, then clusters where eight do not fill it once and leave each warp more than
  // four groups at the cache's capacity (a cluster costs 1.4 us). Measured with 1, 2, 4, 8 warps: 4096 tiles at positions
  // 128-640 51, 41, 49, 74 us; 1024 tiles at 300-1900 51, 36, 34, 38; 256 tiles of 1028 positions x 128 50, 30, 21, 17; 32 tiles
  // of 30000 x 128 with 8 warps, clusters of 1 and 8: 203 and 42.
  const int64_t slots = 148 * 16;  // warps of this kernel that the GPU holds
  const int64_t reach = A.cache.max_len + (kShared && A.part_stats == nullptr ? static_cast<int64_t>(A.prefix.max_len) : 0);
  int W = 1, C = 1;
  // Joined behind short histories of their own, a CTA has a warp for each row and head of its tile at least, up to four, and else so many
  // that all CTAs are on the GPU at once. How long the histories are is known by the cache's capacity alone. Brief / not, the same content: 64
  // sequences x 16 heads x 64 of 10-500 positions behind 8192 37.7 us (2 warps) / 48.7 (8), in bf16 35.6 / 45.7, 128 of them 52.7 / 57.3; 96 x
  // 8 heads x 4 of 17-900 behind 30,000 118 (4 warps) / 123; but 64 x 16 heads of 1,000-4,000 behind 8192 99 / 91.
  const bool joined = kShared && A.part_stats != nullptr, brief = joined && A.cache.max_len <= 1024;
  const int64_t fill = brief ? slots / 2 + 1 : 2 * slots;
  while (W < kMostWarps && ((base * W < fill && reach > W * kKv4Group) || (joined && W < std::min(4, A.group)))) W *= 2;
  while (C < 8 && W == kMostWarps && base * W * C * 2 <= slots && reach > 4 * C * W * kKv4Group) C *= 2;
  if (grid * C > 0x7fffffff) return fail(IVB_EINVAL, "ivb_kv4_attention: %lld tiles of rows in one call", static_cast<long long>(grid));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid * C));
  cfg.blockDim = dim3(32 * W);
  cfg.dynamicSmemBytes = G::smem(W);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = kv4_attributes(C, attr);
  IVB_CUDA(cudaLaunchKernelEx(&cfg, kv4_rows_kernel<D, T, kSplit, kTiles, kShared>, A, static_cast<int>(tiles)));
  return IVB_OK;
}

// Rows of a tile by what a sequence can have: four as pairs of fp16 (for every type: no less exact, and as fast), then
// eight; 16-bit queries with more in columns of their own.
template <int D, typename T, bool kShared>
int32_t launch_rows_of(const Kv4Attention& A, cudaStream_t stream) {
  const bool one = A.starts == nullptr;
  if (keeps_rest(A)) return launch_rows_attention<D, T, true, 1, kShared>(A, stream);
  if constexpr (std::is_same<T, float>::value) {
    return launch_rows_attention<D, T, true, 2, kShared>(A, stream);
  } else {
    if (one && A.group <= 8) return launch_rows_attention<D, T, false, 1, kShared>(A, stream);
    return launch_rows_attention<D, T, false, 2, kShared>(A, stream);
  }
}

template <int D, typename T>
int32_t launch_dim(const Kv4Attention& A, cudaStream_t stream) {
  return A.prefix.data == nullptr ? launch_rows_of<D, T, false>(A, stream) : launch_rows_of<D, T, true>(A, stream);
}

template <typename T>
int32_t launch_attention(const Kv4Attention& A, cudaStream_t stream) {
  switch (A.cache.head_dim) {
    case 32: return launch_dim<32, T>(A, stream);
    case 64: return launch_dim<64, T>(A, stream);
    default: return launch_dim<128, T>(A, stream);
  }
}

// Which sequences are few rows' (those with so many items at most).
int few_items(const IvbKv4Cache& c, int group, const int32_t* starts, int rows) {
  const int64_t items = static_cast<int64_t>(rows) * group;
  const int64_t tiles = items / 256 + std::min<int64_t>(c.batch, items / (kFewItems + 1));
  const int few = tiles * c.kv_heads * 4 >= 148 ? kFewItems : kFewItemsSparse;
  // a lone sequence that can have more takes the prompts' kernel however many it has: one launch
  return starts == nullptr || items <= few ? 0x7fffffff : c.batch == 1 ? 0 : few;
}

// Whether few rows walk the beginning that they share each on their own, in one kernel, where that is less than a pass over it (whose
// kernel takes 9 us at least): by row tiles x heads x its positions. Measured, walked / passed, us: 16 sequences x 16 heads x 64 in fp32,
// 256k 10 / 18, 640k 17 / 18, 1,536k 33 / 22; 64 x 16 x 64 in bf16, 410k 20 / 19, 1,024k 30 / 18; 8 x 8 heads x 4 x 128, 160k 14 / 21,
// 384k 19 / 22; 64 x 8 x 4 x 128, 204k 19 / 29, 512k 29 / 31, 1,280k 50 / 33; 32 x 8 x 32, 640k 13 / 16, 1,536k 24 / 17.
constexpr int64_t kWalkReach = 500000;
bool walks_prefix(const IvbKv4Cache& c, const IvbKv4Cache& prefix, int group, int rows) {
  const int64_t tiles = std::max<int64_t>(std::min(rows, c.batch), static_cast<int64_t>(rows) * group / 8);
  return tiles * c.kv_heads * prefix.max_len <= kWalkReach;
}

// Bytes of the parts of a shared beginning: for each split, row and head its statistics and its values.
uint64_t part_bytes(int splits, int rows, int heads, int dim) { return static_cast<uint64_t>(splits) * rows * heads * (8 + 4 * static_cast<uint64_t>(dim)); }

int32_t check_heads(const IvbKv4Cache* c, int32_t heads, int32_t rows) {
  if (heads <= 0 || heads % c->kv_heads != 0) return fail(IVB_EINVAL, "ivb_kv4_attention: %d query heads over %d key/value heads", heads, c->kv_heads);
  if (static_cast<int64_t>(rows) * heads > 0x7fffffff - 1024) return fail(IVB_EINVAL, "ivb_kv4_attention: %d rows of %d heads", rows, heads);
  return IVB_OK;
}

int32_t check_prefix(const IvbKv4Cache* c, const IvbKv4Prefix* prefix) {
  if (prefix == nullptr) return fail(IVB_EINVAL, "ivb_kv4_attention_prefix: null prefix");
  if (int32_t rc = check_kv4(&prefix->cache, "ivb_kv4_attention_prefix")) return rc;
  if (prefix->cache.kv_heads != c->kv_heads || prefix->cache.head_dim != c->head_dim)
    return fail(IVB_EINVAL, "ivb_kv4_attention_prefix: %d heads x %d behind a prefix of %d x %d", c->kv_heads, c->head_dim, prefix->cache.kv_heads,
                prefix->cache.head_dim);
  if (prefix->lengths == nullptr) return fail(IVB_EINVAL, "ivb_kv4_attention_prefix: null lengths");
  if (prefix->groups == nullptr && prefix->cache.batch != 1)
    return fail(IVB_EINVAL, "ivb_kv4_attention_prefix: %d prefixes without groups", prefix->cache.batch);
  if (static_cast<int64_t>(prefix->cache.max_len) + c->max_len > 0x7fffffff - 256)
    return fail(IVB_EINVAL, "ivb_kv4_attention_prefix: %d positions behind %d", c->max_len, prefix->cache.max_len);
  return IVB_OK;
}

int32_t attention_call(const IvbKv4Cache* c, const IvbKv4Prefix* prefix, const void* q, int32_t dtype, int64_t q_row, int64_t q_head, int32_t heads,
                       const int32_t* starts, const int64_t* positions, int32_t rows, float scale, int32_t window, int32_t sinks, void* out,
                       int64_t o_row, int64_t o_head, void* workspace, uint64_t workspace_bytes, uint32_t* error, void* stream, bool withhold) {
  if (int32_t rc = check_kv4(c, "ivb_kv4_attention")) return rc;
  if (int32_t rc = check_kv4_rows(c, starts, positions, rows, dtype, "ivb_kv4_attention")) return rc;
  if (int32_t rc = check_heads(c, heads, rows)) return rc;
  if (window < 0 || sinks < 0) return fail(IVB_EINVAL, "ivb_kv4_attention: window %d, sinks %d", window, sinks);
  if (rows == 0) return IVB_OK;
  if (q == nullptr || out == nullptr) return fail(IVB_EINVAL, "ivb_kv4_attention: null queries or output");
  Kv4Attention A{};
  A.cache = *c;
  A.q = q;
  A.out = out;
  A.q_row = q_row;
  A.q_head = q_head;
  A.o_row = o_row;
  A.o_head = o_head;
  A.starts = starts;
  A.positions = positions;
  A.error = error;
  A.scale = scale;
  A.heads = heads;
  A.group = heads / c->kv_heads;
  A.rows = rows;
  A.window = window;
  A.sinks = sinks;
  A.wait_ns = withhold ? kKv4ProbeNs : kKv4WaitNs;
  A.withhold = withhold;
  const int size = dtype == IVB_F32 ? 4 : 2;
  auto aligned = [&](const void* p, int64_t row, int64_t head) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row * size % 16 == 0 && head * size % 16 == 0;
  };
  A.q_vec = aligned(q, q_row, q_head);
  A.o_vec = aligned(out, o_row, o_head);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  A.few = few_items(*c, A.group, starts, rows);
  if (prefix != nullptr) {
    A.prefix = prefix->cache;
    A.prefix_lengths = prefix->lengths;
    A.prefix_groups = prefix->groups;
    if (A.few != 0 && !walks_prefix(*c, prefix->cache, A.group, rows)) {
      A.splits = kv4_prefix_splits(*c, prefix->cache, A.group, rows);
      if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < part_bytes(A.splits, rows, heads, c->head_dim))
        return fail(IVB_EINVAL, "ivb_kv4_attention_prefix: a workspace of %llu bytes at %p, not 16-byte aligned or too small",
                    static_cast<unsigned long long>(workspace_bytes), workspace);
      A.part_values = static_cast<float*>(workspace);
      A.part_stats = reinterpret_cast<float2*>(A.part_values + static_cast<int64_t>(A.splits) * rows * heads * c->head_dim);
    }
  }
  A.beside_prompts = A.few != 0x7fffffff;
  if (A.beside_prompts)
    if (int32_t rc = launch_kv4_prompts(A, dtype, A.few, s)) return rc;
  if (A.few == 0) return IVB_OK;
  if (A.part_stats != nullptr) {
    if (int32_t rc = launch_kv4_prefix(A, dtype, A.few, s)) return rc;
    A.beside_prompts = true;  // beside the pass, and what that is beside
  }
  if (dtype == IVB_F32) return launch_attention<float>(A, s);
  if (dtype == IVB_F16) return launch_attention<__half>(A, s);
  return launch_attention<__nv_bfloat16>(A, s);
}

}  // namespace
}  // namespace ivb

extern "C" {

int32_t ivb_kv4_attention(const IvbKv4Cache* c, const void* q, int32_t dtype, int64_t q_row, int64_t q_head, int32_t heads,
                          const int32_t* starts, const int64_t* positions, int32_t rows, float scale, int32_t window, int32_t sinks, void* out,
                          int64_t o_row, int64_t o_head, uint32_t* error, void* stream) {
  return ivb::attention_call(c, nullptr, q, dtype, q_row, q_head, heads, starts, positions, rows, scale, window, sinks, out, o_row, o_head, nullptr, 0,
                             error, stream, false);
}

uint64_t ivb_kv4_prefix_workspace_bytes(const IvbKv4Cache* c, const IvbKv4Prefix* prefix, int32_t dtype, int32_t heads, const int32_t* starts,
                                        int32_t rows) {
  if (ivb::check_kv4(c, "ivb_kv4_prefix_workspace_bytes") || rows <= 0 || ivb::check_heads(c, heads, rows) || ivb::check_prefix(c, prefix)) return 0;
  const int group = heads / c->kv_heads;
  if (ivb::few_items(*c, group, starts, rows) == 0 || ivb::walks_prefix(*c, prefix->cache, group, rows)) return 0;
  return ivb::part_bytes(ivb::kv4_prefix_splits(*c, prefix->cache, group, rows), rows, heads, c->head_dim);
}

int32_t ivb_kv4_attention_prefix(const IvbKv4Cache* c, const IvbKv4Prefix* prefix, const void* q, int32_t dtype, int64_t q_row, int64_t q_head,
                                 int32_t heads, const int32_t* starts, const int64_t* positions, int32_t rows, float scale, int32_t window,
                                 int32_t sinks, void* out, int64_t o_row, int64_t o_head, void* workspace, uint64_t workspace_bytes, uint32_t* error,
                                 void* stream) {
  if (int32_t rc = ivb::check_kv4(c, "ivb_kv4_attention_prefix")) return rc;
  if (int32_t rc = ivb::check_prefix(c, prefix)) return rc;
  return ivb::attention_call(c, prefix, q, dtype, q_row, q_head, heads, starts, positions, rows, scale, window, sinks, out, o_row, o_head, workspace,
                             workspace_bytes, error, stream, false);
}

int32_t ivb_probe_kv4_prefix_timeout(const IvbKv4Cache* c, const IvbKv4Prefix* prefix, const void* q, int32_t dtype, int64_t q_row, int64_t q_head,
                                     int32_t heads, const int32_t* starts, const int64_t* positions, int32_t rows, float scale, int32_t window,
                                     int32_t sinks, void* out, int64_t o_row, int64_t o_head, void* workspace, uint64_t workspace_bytes,
                                     uint32_t* error, void* stream) {
  if (int32_t rc = ivb::check_kv4(c, "ivb_kv4_attention_prefix")) return rc;
  if (int32_t rc = ivb::check_prefix(c, prefix)) return rc;
  return ivb::attention_call(c, prefix, q, dtype, q_row, q_head, heads, starts, positions, rows, scale, window, sinks, out, o_row, o_head, workspace,
                             workspace_bytes, error, stream, true);
}

int32_t ivb_probe_kv4_timeout(const IvbKv4Cache* c, const void* q, int32_t dtype, int64_t q_row, int64_t q_head, int32_t heads,
                              const int32_t* starts, const int64_t* positions, int32_t rows, float scale, int32_t window, int32_t sinks,
                              void* out, int64_t o_row, int64_t o_head, uint32_t* error, void* stream) {
  return ivb::attention_call(c, nullptr, q, dtype, q_row, q_head, heads, starts, positions, rows, scale, window, sinks, out, o_row, o_head, nullptr, 0,
                             error, stream, true);
}

}  // extern "C"
