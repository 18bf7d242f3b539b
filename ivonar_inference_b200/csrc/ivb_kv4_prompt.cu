// Causal attention over the 4-bit key/value cache for prompts: many rows a sequence, on the 5th-generation tensor cores.
//
// One CTA per (sequence, key/value head, 256 rows), 12 warps. Row i of a sequence's head group is token i / group, query head
// i % group; rows 0..127 and 128..255 are two tiles X of the tensor cores' 128 lanes. Per tile of 128 positions:
//   warps 8..10 (producers) read the codes, expand them to fp16 in shared memory (keys as a K-major operand, values as an
//     MN-major one: both are position rows of 16-byte channel chunks, so neither is transposed) and compute each
//     position's terms (scales and offsets; ivb_kv4_attention.cuh);
//   warp 11 (whose instructions come slowly beside the softmax's: no more of them than needed) issues S_X = Q_X U^T and
//     O_X += P_X U'^T, fp32 in tensor memory;
//   warps 0..7 (32 rows each, their tensor-memory lanes) turn S_X into weights: online softmax in 32 bits, the
//     reference raised only when the maximum passes it by 2^8, and O_X rescaled in tensor memory then. The weights P_X take
//     S_X's place as the fp16 A operand, so S_X(it + 1) follows P_X(it)'s product; while one X waits for it the other computes.
// fp32 queries and weights are hi + lo fp16 pairs: two products each. The scores come 64 positions at a time (48 cycles a product
// where 128 columns take 65), so that the next half's are there when a half's weights are done. With few CTAs a cluster of C shares
// the rows: each takes every C-th tile, and they join what they found through one another's shared memory.
// What takes the time is the softmax: 2048 rows at 6144 under a window of 4096, 32 heads x 128 in bf16, take 230 us (0.60 PFLOP/s). Measured
// when it was 228: 47 % of the issue slots used; without the exponentials 203, with a sixth of the products 222, without the
// producers' stores 226, without any of these and without the terms 168.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "ivb_decode.cuh"
#include "ivb_kv4_attention.cuh"
#include "ivb_tc.cuh"

namespace ivb {
namespace {

namespace cg = cooperative_groups;

constexpr int kRowsX = 128, kRowsCta = 256, kPos = 128;
// 12 warps: three on each of the SM's four parts have 168 registers a thread, for the scores of four rows at a time
constexpr int kSoftmaxWarps = 8, kSoftmaxThreads = 32 * kSoftmaxWarps, kProducerWarps = 3, kProducers = 32 * kProducerWarps;
constexpr int kIssueWarp = kSoftmaxWarps + kProducerWarps, kPromptThreads = 32 * (kIssueWarp + 1);
constexpr int kTermSets = 3;  // terms(it + 2) are written when S(it) is done, so when nobody reads terms(it - 1) any more
constexpr float kWeightUnit = 64.0f;  // weights are at most 2 * 64 * 2^8 in fp16
constexpr float kRaise = 8.0f;
// A tile's rows share the queries' power of two (no multiplication of the scores by a row's own) unless one's largest is so far below
// another's: to there hi + lo keep 2^-23 of a row's largest, and fp16 as many bits as bf16 or fp16 queries have.
constexpr float kEven = 0.000244140625f;
// The tensor cores cut what they add to an accumulator towards zero, a bias that grows with its length (1.6e-6 of the output after
// 1024 positions). fp32 outputs keep a second one, to which the threads add the first every so many tiles, rounding to nearest.
constexpr int kFoldTiles = 2;

template <int D, bool kSplit>
struct PromptGeometry {
  static constexpr int parts = kSplit ? 2 : 1;
  static constexpr int stages = kSplit && D == 128 ? 1 : 2;  // of keys and of values
  static constexpr int q_bytes = kRowsX * D * 2;             // one part of one row tile
  static constexpr int kv_bytes = kPos * D * 2;              // keys or values of a stage
  static constexpr int term_bytes = kPos * 24;
  static constexpr int q_at = 0, k_at = (kSplit && D == 128 ? 1 : 2) * parts * q_bytes, v_at = k_at + stages * kv_bytes, terms_at = v_at + stages * kv_bytes;
  // over half of an SM's at least: of two clusters sharing two SMs each could hold the tensor memory that the other waits for
  static constexpr int used = terms_at + kTermSets * term_bytes, smem = used < 118 * 1024 ? 118 * 1024 : used;
  // row tiles of a CTA: at fp32 and D = 128 tensor memory holds the accumulators of one
  static constexpr int row_tiles = kSplit && D == 128 ? 1 : 2, rows = row_tiles * kRowsX;
  // tensor memory columns: S_X, then P_X in its place (of every 64 columns 32 hi, 32 lo), O_X, and O_X's sums (fp32)
  static constexpr int s_at = 0, o_at = row_tiles * kPos, fold_at = o_at + row_tiles * D, columns = 512;
  static_assert(fold_at + (kSplit ? row_tiles * D : 0) <= columns, "tensor memory");
};

// kind::f16, fp32 result, A K-major, B MN-major.
__host__ __device__ constexpr uint32_t idesc_f16_bt(int m, int n) { return idesc_f16(m, n) | (1u << 16); }

// Descriptor of an MN-major operand without swizzle: core matrices of 8 K rows x 8 channels (16 bytes a row), the next 8
// channels 128 bytes on, the next 8 K rows `k_step` bytes on.
__device__ __forceinline__ uint64_t smem_desc_mn(unsigned addr, unsigned k_step) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((k_step >> 4) & 0x3FFFu) << 16) |
         (static_cast<uint64_t>(128 >> 4) << 32) | (1ull << 46);
}

// Byte offset of channel chunk i (8 channels) of row p in core matrices of 8 rows x 16 bytes, D / 8 chunks a row.
template <int D>
__device__ __forceinline__ int chunk_at(int p, int i) {
  return ((p >> 3) * (D / 8) + i) * 128 + (p & 7) * 16;
}

__device__ __forceinline__ uint4 expand(uint32_t w, CodeMiddle m) {
  return make_uint4(codes_low(w, m), codes_high(w, m), codes_low(w >> 8, m), codes_high(w >> 8, m));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Two fp32 operations in one instruction.
typedef float2 f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) { return make_float2(a, b); }
__device__ __forceinline__ float2 unpair(f32x2 a) { return a; }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { return __fadd2_rn(a, b); }

template <typename T>
__device__ __forceinline__ void values_of_chunk(uint4 w, float (&v)[16 / sizeof(T)]) {
  union {
    uint4 w;
    T t[16 / sizeof(T)];
  } u;
  u.w = w;
#pragma unroll
  for (int j = 0; j < static_cast<int>(16 / sizeof(T)); ++j) v[j] = to_f32<T>(u.t[j]);
}

struct PromptBarriers {
  unsigned long long k_full[2], k_free[2], v_full[2], v_free[2], terms_full[kTermSets], s_full[2][2], p_full[2][2], p_free[2][2], drain;
};

// What a lane of a producer warp holds of the keys or values of one tile of 16 positions (D = 32: values in lanes 0..15), dealt
// out so that 8 neighbouring lanes write the 8 rows of a core matrix, without bank conflicts.
template <int D>
struct RawChunks {
  static constexpr int n = D == 128 ? 2 : 1;
  uint4 v[n];
};

template <int D>
__device__ __forceinline__ void load_keys(const unsigned char* tile, bool in, int lane, RawChunks<D>& raw) {
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (D == 128) {
    const int h = (lane >> 2) & 1, c = lane >> 3;
#pragma unroll
    for (int k = 0; k < 2; ++k) raw.v[k] = in ? *reinterpret_cast<const uint4*>(tile + 512 * h + (((lane & 3) + 4 * k) * 4 + c) * 16) : zero;
  } else {
    const int r = lane & 7, c = lane >> 3;
    if constexpr (D == 64) {
      raw.v[0] = in ? *reinterpret_cast<const uint4*>(tile + (r * 4 + c) * 16) : zero;
    } else {
      const uint2 v = in ? *reinterpret_cast<const uint2*>(tile + (r * 4 + c) * 8) : make_uint2(0u, 0u);
      raw.v[0] = make_uint4(v.x, v.y, 0u, 0u);
    }
  }
}
template <int D>
__device__ __forceinline__ void load_codes_of_values(const unsigned char* tile, bool in, int lane, RawChunks<D>& raw) {
  const int r = D == 32 ? lane & 3 : (lane & 3) + 4 * (lane >> 4), c = (lane >> 2) & 3;
  in = in && (D != 32 || lane < 16);
#pragma unroll
  for (int k = 0; k < RawChunks<D>::n; ++k)
    raw.v[k] = in ? *reinterpret_cast<const uint4*>(tile + 8 * D + 512 * k + (r * 4 + c) * 16) : make_uint4(0u, 0u, 0u, 0u);
}

// `keys`, `values`: the tile's 16 position rows.
template <int D>
__device__ __forceinline__ void store_keys(const RawChunks<D>& raw, int lane, unsigned char* keys) {
  const CodeMiddle m = code_middle(8.0f, 8.0f);
  if constexpr (D == 128) {
    const int h = (lane >> 2) & 1, c = lane >> 3;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = (lane & 3) + 4 * k, p = 4 * (r >> 1) + (r & 1) + 2 * h;
      const uint32_t w[4] = {raw.v[k].x, raw.v[k].y, raw.v[k].z, raw.v[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(keys + chunk_at<D>(p, 4 * c + i)) = expand(w[i], m);
    }
  } else {
    const int r = lane & 7, c = lane >> 3, other = r >> 2;  // the upper four rows' lanes take their two positions in the other order
    const int p = 4 * (r >> 1) + (r & 1);
    if constexpr (D == 64) {
      const uint2 a = other ? make_uint2(raw.v[0].z, raw.v[0].w) : make_uint2(raw.v[0].x, raw.v[0].y);
      const uint2 b = other ? make_uint2(raw.v[0].x, raw.v[0].y) : make_uint2(raw.v[0].z, raw.v[0].w);
      *reinterpret_cast<uint4*>(keys + chunk_at<D>(p + 2 * other, 2 * c)) = expand(a.x, m);
      *reinterpret_cast<uint4*>(keys + chunk_at<D>(p + 2 * other, 2 * c + 1)) = expand(a.y, m);
      *reinterpret_cast<uint4*>(keys + chunk_at<D>(p + 2 - 2 * other, 2 * c)) = expand(b.x, m);
      *reinterpret_cast<uint4*>(keys + chunk_at<D>(p + 2 - 2 * other, 2 * c + 1)) = expand(b.y, m);
    } else {
      *reinterpret_cast<uint4*>(keys + chunk_at<D>(p + 2 * other, c)) = expand(other ? raw.v[0].y : raw.v[0].x, m);
      *reinterpret_cast<uint4*>(keys + chunk_at<D>(p + 2 - 2 * other, c)) = expand(other ? raw.v[0].x : raw.v[0].y, m);
    }
  }
}
template <int D>
__device__ __forceinline__ void store_codes_of_values(const RawChunks<D>& raw, int lane, unsigned char* values) {
  if (D == 32 && lane >= 16) return;
  const float mine = lane & 1 ? 7.0f : 8.0f, other = 15.0f - mine;  // by the parity of the positions 4 c + (i + turn) % 4
  const CodeMiddle middle[2] = {code_middle(mine, mine), code_middle(other, other)};
  const int turn = lane & 3, c = (lane >> 2) & 3, r = D == 32 ? lane & 3 : (lane & 3) + 4 * (lane >> 4);
#pragma unroll
  for (int k = 0; k < RawChunks<D>::n; ++k) {
    uint4 v = raw.v[k];  // word i of the lane is position 4 c + i: each lane begins with another one
    if (turn & 1) v = make_uint4(v.y, v.z, v.w, v.x);
    if (turn & 2) v = make_uint4(v.z, v.w, v.x, v.y);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(values + chunk_at<D>(4 * c + ((i + turn) & 3), 8 * k + r)) = expand(w[i], middle[i & 1]);
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(kPromptThreads, 1) kv4_prompt_kernel(Kv4Attention A, int few) {
  constexpr bool kSplit = std::is_same<T, float>::value;
  using G = PromptGeometry<D, kSplit>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ PromptBarriers bar;
  __shared__ unsigned tmem_base;
  __shared__ float largest[kSoftmaxWarps], smallest[kSoftmaxWarps], sums[kRowsCta], row_units[kRowsCta], refs_of[kRowsCta], totals[kRowsCta], offsets[kRowsCta];
  __shared__ int which[3];  // sequence, tile of its rows; and whether a wait ran out
  const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;

  pdl_wait();
  // which rows: the call's tiles of 256 items in the order of the sequences, the last ones (the longest rows) first
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int unit = static_cast<int>(blockIdx.x) / C, units = static_cast<int>(gridDim.x) / C;
  const int kvh = unit % A.cache.kv_heads, order = units / A.cache.kv_heads - 1 - unit / A.cache.kv_heads;
  if (warp == 0) {
    int seen = 0, found = -1, tile = 0;
    for (int b0 = 0; b0 < A.cache.batch && found < 0; b0 += 32) {
      const int b = b0 + lane;
      int n = 0;
      if (b < A.cache.batch) {
        int count = 1;
        if (A.starts != nullptr) count = max(0, min(A.rows, A.starts[b + 1]) - max(0, A.starts[b]));
        const int items = count * A.group;
        n = items > few ? (items + G::rows - 1) / G::rows : 0;
      }
      int upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += o;
      }
      const unsigned hit = __ballot_sync(0xFFFFFFFFu, seen + upto > order);
      if (hit != 0u) {
        const int l = __ffs(hit) - 1;
        found = b0 + l;
        tile = order - (seen + __shfl_sync(0xFFFFFFFFu, upto, l) - __shfl_sync(0xFFFFFFFFu, n, l));
      }
      seen += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    if (lane == 0) {
      which[0] = found;
      which[1] = tile;
      which[2] = 0;
    }
  }
  if (tid == 32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.k_full[i], kProducers);
      mbar_init(&bar.k_free[i], 1);
      mbar_init(&bar.v_full[i], kProducers);
      mbar_init(&bar.v_free[i], 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bar.p_full[i][h], kSoftmaxThreads / 2);
        mbar_init(&bar.p_free[i][h], 1);
        mbar_init(&bar.s_full[i][h], 1);
      }
    }
#pragma unroll
    for (int i = 0; i < kTermSets; ++i) mbar_init(&bar.terms_full[i], kProducers);
    mbar_init(&bar.drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const int b = which[0];
  if (b < 0) return;
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)), "r"(G::columns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    pdl_trigger();  // not before this CTA has its tensor memory: the next grid may take some too, and waits for this one
  }
  int row0 = b, count = 1;
  int64_t before = 0;  // rows of the sequence that the call does not have
  if (A.starts != nullptr) {
    row0 = max(0, A.starts[b]);
    before = static_cast<int64_t>(row0) - A.starts[b];
    count = min(A.rows, A.starts[b + 1]) - row0;
  }
  const int i0 = which[1] * G::rows, live = min(G::rows, count * A.group - i0), row_tiles = live > kRowsX ? 2 : 1;
  const int64_t base = kv4_position(A.positions, b) + before;
  const int max_len = A.cache.max_len;
  const unsigned group_size = static_cast<unsigned>(A.group);
  auto token_of = [&](int i) { return static_cast<int>(static_cast<unsigned>(i) / group_size); };
  auto clamp_position = [&](int64_t p) { return static_cast<int>(max(static_cast<int64_t>(-1), min(p, static_cast<int64_t>(max_len)))); };
  const int first = clamp_position(base + token_of(i0)), last = clamp_position(base + token_of(i0 + live - 1));
  if (last >= max_len && tid == 0 && rank == 0 && A.error != nullptr) atomicCAS(A.error, 0u, static_cast<unsigned>(IVB_ECAPACITY));
  // the tiles of 128 positions that some row sees: the sinks' below the window, then the window's
  const int high = min(last, max_len - 1);
  const int low = A.window > 0 ? max(0, max(first, 0) - A.window + 1) : 0;
  const int window_tile = low / kPos;
  const int sink_tiles = A.window > 0 ? min((min(A.sinks, low) + kPos - 1) / kPos, window_tile) : 0;
  const int all_tiles = high < 0 ? 0 : sink_tiles + high / kPos - window_tile + 1;
  const int tiles = all_tiles > rank ? (all_tiles - rank + C - 1) / C : 0;  // this CTA's
  auto tile_of = [&](int it) {
    const int i = rank + it * C;
    return i < sink_tiles ? i : window_tile + i - sink_tiles;
  };

  // queries: a warp takes 32 rows in 16-byte chunks, 8 rows and 4 chunks at a time (64 contiguous bytes of a row, and no bank
  // conflicts); the rows' largest first, then hi (and lo) parts as K-major operands, scaled by a power of two that brings the largest of
  // all rows to 2^13, or each row's own where they are uneven. Idle rows' queries are not read.
  constexpr int kPer = 16 / static_cast<int>(sizeof(T)), L = D / kPer, kQuads = L / 4;  // values of a chunk, chunks of a row
  const int row8 = lane & 7, chunk4 = lane >> 3;
  const int x = warp >> 2;  // row tile of a softmax warp
  auto item_row = [&](const void* array, int i, int64_t row_stride, int64_t head_stride) {
    const int t = token_of(i), h = kvh * A.group + i - t * A.group;
    return static_cast<const T*>(array) + (row0 + t) * row_stride + h * head_stride;
  };
  uint4 raw[4][kQuads];
  if (tid < kSoftmaxThreads) {
    const T* q[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r = 32 * warp + 8 * g + row8;
      const int p = clamp_position(base + token_of(i0 + r));
      q[g] = r < live && p >= 0 && p < max_len ? item_row(A.q, i0 + r, A.q_row, A.q_head) + chunk4 * kPer : nullptr;
    }
    if (A.q_vec) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int k = 0; k < kQuads; ++k)
          raw[g][k] = q[g] != nullptr ? reinterpret_cast<const uint4*>(q[g])[4 * k] : make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int k = 0; k < kQuads; ++k) {
          union {
            uint4 w;
            T t[kPer];
          } u;
          u.w = make_uint4(0u, 0u, 0u, 0u);
          if (q[g] != nullptr)
#pragma unroll
            for (int j = 0; j < kPer; ++j) u.t[j] = q[g][4 * k * kPer + j];
          raw[g][k] = u.w;
        }
    }
    float most = 0.0f, least = INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float top = 0.0f;
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        float v[kPer];
        values_of_chunk<T>(raw[g][k], v);
#pragma unroll
        for (int j = 0; j < kPer; ++j) top = fmaxf(top, finite_size(v[j]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
      if (chunk4 == 0) row_units[32 * warp + 8 * g + row8] = top;
      most = fmaxf(most, top);
      if (top > 0.0f) least = fminf(least, top);
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
      most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
      least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, d));
    }
    if (lane == 0) {
      largest[warp] = most;
      smallest[warp] = least;
    }
  }
  __syncthreads();
  float most = 0.0f, least = INFINITY;
#pragma unroll
  for (int w = 0; w < kSoftmaxWarps; ++w) {
    most = fmaxf(most, largest[w]);
    least = fminf(least, smallest[w]);
  }
  const bool even = least >= most * kEven;
  const int up = query_power(most);
  const float score_unit = power_of_two(-up) * (A.scale * kLog2e);  // in the positions' terms
  if (tid < kSoftmaxThreads && x < row_tiles) {
    unsigned char* dst = smem + G::q_at + x * G::parts * G::q_bytes;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int row = 32 * warp + 8 * g + row8, own = even ? up : min(query_power(row_units[row]), up + 126);
      const float q_unit = power_of_two(own);
      float total = 0.0f;
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        const int r = 32 * (warp & 3) + 8 * g + row8, i = 4 * k + chunk4;
        float v[kPer];
        values_of_chunk<T>(raw[g][k], v);
        uint32_t hi[kPer / 2], lo[kPer / 2];
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j) {
          const float a = v[2 * j] * q_unit, c = v[2 * j + 1] * q_unit;
          total = total + a + c;
          hi[j] = pack_f16(a, c);
          const float2 h = unpack_f16(hi[j]);
          lo[j] = pack_f16(a - h.x, c - h.y);
        }
        if constexpr (kSplit) {
          unsigned char* to = dst + chunk_at<D>(r, i / 2) + 8 * (i & 1);
          *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2*>(to + G::q_bytes) = make_uint2(lo[0], lo[1]);
        } else {
          *reinterpret_cast<uint4*>(dst + chunk_at<D>(r, i)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        }
      }
      total += __shfl_xor_sync(0xFFFFFFFFu, total, 8);
      total += __shfl_xor_sync(0xFFFFFFFFu, total, 16);  // the lanes of the row have read row_units[row]
      const float unit = power_of_two(up - own);  // what is left to undo for the row
      if (chunk4 == 0) {
        row_units[row] = unit;
        sums[row] = total * unit;
      }
    }
  }
  fence_proxy_async();  // the tensor cores read what the threads wrote
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xFFFFFFFFu, tmem_base, 0);
  auto keys_of = [&](int it) { return smem + G::k_at + it % G::stages * G::kv_bytes; };
  auto values_of = [&](int it) { return smem + G::v_at + it % G::stages * G::kv_bytes; };
  auto terms_of = [&](int it) { return reinterpret_cast<float*>(smem + G::terms_at + it % kTermSets * G::term_bytes); };
  auto turn_of = [&](int it) { return static_cast<unsigned>(it / G::stages) & 1u; };  // parity of a stage's use
  bool ok = true;
  auto wait_for = [&](unsigned long long* at, unsigned turn) { return mbar_wait_bounded(at, turn, A.wait_ns); };

  if (warp >= kSoftmaxWarps && warp < kIssueWarp) {
    // ---- producers: 16-position tiles in turn ----
    constexpr int kTile = kv4_tile_bytes(D), kUnits = kPos / 16, kMine = (kUnits + kProducerWarps - 1) / kProducerWarps;
    const int unit0 = warp - kSoftmaxThreads / 32;
    const int64_t tiles16 = kv4_tiles(max_len);
    const unsigned char* codes = static_cast<const unsigned char*>(A.cache.data) + (static_cast<int64_t>(b) * A.cache.kv_heads + kvh) * tiles16 * kTile;
    RawChunks<D> key[kMine], value[kMine];
    uint2 par[kMine];
    auto fetch = [&](int it, bool keys) {
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int u = unit0 + k * kProducerWarps;
        const int64_t t = static_cast<int64_t>(tile_of(it)) * kUnits + u;
        const bool in = u < kUnits && t < tiles16;
        const unsigned char* tile = codes + (in ? t : 0) * kTile;
        if (keys) {
          load_keys<D>(tile, in, lane, key[k]);
          par[k] = in && lane < 16 ? *reinterpret_cast<const uint2*>(tile + 16 * D + lane * 8) : make_uint2(0u, 0u);
        } else {
          load_codes_of_values<D>(tile, in, lane, value[k]);
        }
      }
    };
    if (tiles > 0) fetch(0, true);
    for (int it = 0; it < tiles; ++it) {
      fetch(it, false);
      if (it >= G::stages && !wait_for(&bar.k_free[it % G::stages], turn_of(it) ^ 1u)) {
        ok = false;
        break;
      }
      if (lane < 16) {
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
          const int u = unit0 + k * kProducerWarps;
          if (u < kUnits) {
            const PositionTerms p = position_terms(par[k], score_unit, kWeightUnit, lane);
            float* at_terms = terms_of(it) + 12 * (8 * u + (lane >> 1)) + (lane & 1);
            at_terms[0] = p.key_scale;
            at_terms[2] = p.key_offset;
            at_terms[4] = p.bias;
            at_terms[6] = p.mantissa;
            at_terms[8] = p.unbias;
            at_terms[10] = p.value_offset;
          }
        }
      }
      mbar_arrive(&bar.terms_full[it % kTermSets]);
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int u = unit0 + k * kProducerWarps;
        if (u < kUnits) store_keys<D>(key[k], lane, keys_of(it) + u * 16 * D * 2);
      }
      fence_proxy_async();
      mbar_arrive(&bar.k_full[it % G::stages]);
      if (it + 1 < tiles) fetch(it + 1, true);
      if (it >= G::stages && !wait_for(&bar.v_free[it % G::stages], turn_of(it) ^ 1u)) {
        ok = false;
        break;
      }
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int u = unit0 + k * kProducerWarps;
        if (u < kUnits) store_codes_of_values<D>(value[k], lane, values_of(it) + u * 16 * D * 2);
      }
      fence_proxy_async();
      mbar_arrive(&bar.v_full[it % G::stages]);
    }
  } else if (warp >= kIssueWarp) {
    // ---- the warp that issues the products: all its lanes take the same way (ok is the same in each) ----
    auto wait = [&](unsigned long long* at, unsigned turn) { return __all_sync(0xFFFFFFFFu, wait_for(at, turn)) != 0; };
    const uint64_t q0 = smem_desc(smem_addr(smem + G::q_at), D / 8 * 128);
    const uint64_t k0 = smem_desc(smem_addr(smem + G::k_at), D / 8 * 128), v0 = smem_desc_mn(smem_addr(smem + G::v_at), D / 8 * 128);
    // Half h of tile it: its 64 columns of S_X, and with P_X in their place its 64 positions' part of O_X. Descriptors count
    // in 16 bytes.
    auto issue_s = [&](int it, int h) {
      const uint64_t k = k0 + (it % G::stages * G::kv_bytes + h * (G::kv_bytes / 2)) / 16;
      for (int xx = 0; xx < row_tiles; ++xx) {
        if (it > 0) {  // S takes the place of P
          ok = ok && wait(&bar.p_free[xx][h], (it - 1) & 1);
          if (!ok) return;
        }
        tc_fence_after();
        const uint64_t q = q0 + xx * (G::parts * G::q_bytes / 16);
        const unsigned t_s = tmem + G::s_at + xx * kPos + h * (kPos / 2);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int part = 0; part < G::parts; ++part)
            umma_f16_ss_warp(t_s, q + (part * G::q_bytes + kk * 256) / 16, k + kk * 16, idesc_f16(kRowsX, kPos / 2), kk + part > 0);
        umma_commit_warp(&bar.s_full[xx][h]);
      }
      if (h == 1) umma_commit_warp(&bar.k_free[it % G::stages]);
    };
    auto issue_o = [&](int it, int h) {
      const uint64_t v = v0 + (it % G::stages * G::kv_bytes + h * (G::kv_bytes / 2)) / 16;
      for (int xx = 0; xx < row_tiles; ++xx) {
        ok = ok && wait(&bar.p_full[xx][h], it & 1);
        if (!ok) return;
        tc_fence_after();
        const unsigned t_p = tmem + G::s_at + xx * kPos + h * (kPos / 2), t_o = tmem + G::o_at + xx * D;
#pragma unroll
        for (int kk = 0; kk < kPos / 32; ++kk)
#pragma unroll
          for (int part = 0; part < G::parts; ++part)
            umma_f16_ts_warp(t_o, t_p + part * (kPos / 4) + kk * 8, v + kk * 2 * (D / 8) * 8, idesc_f16_bt(kRowsX, D), kk + part > 0 || h > 0 || (kSplit ? it % kFoldTiles != 0 : it > 0));
        umma_commit_warp(&bar.p_free[xx][h]);
      }
      if (h == 1) umma_commit_warp(&bar.v_free[it % G::stages]);
    };
    if (tiles > 0) {
      ok = wait(&bar.k_full[0], 0) && !A.withhold;
      if (ok) {
        issue_s(0, 0);
        issue_s(0, 1);
      }
    }
    // both row tiles' weights of a half, then, while they are used up, their next scores in that half's place
    for (int it = 0; it < tiles && ok; ++it) {
      ok = wait(&bar.v_full[it % G::stages], turn_of(it));
      if (ok) issue_o(it, 0);
      if (it + 1 < tiles) {
        ok = ok && wait(&bar.k_full[(it + 1) % G::stages], turn_of(it + 1));
        if (ok) issue_s(it + 1, 0);
      }
      if (ok) issue_o(it, 1);
      if (ok && it + 1 < tiles) issue_s(it + 1, 1);
    }
    // what was issued ends before shared and tensor memory go, also where another warp's wait ran out
    umma_commit_warp(&bar.drain);
    ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&bar.drain, 0, kKv4WaitNs)) != 0 && ok;
  } else if (x < row_tiles) {
    // ---- softmax: a warp has 32 rows, a thread in each 8-row set the row r and every fourth pair of positions, so that a
    // position's terms are loaded once for four rows (loaded for each row they bound the kernel: 12 cycles of the SM's
    // shared memory pipe for 64 scores)
    const int r = lane >> 2, c = lane & 3, row0x = 32 * (warp & 3);
    const unsigned lanes = static_cast<unsigned>(row0x) << 16;
    const unsigned ts = tmem + lanes + G::s_at + x * kPos, to = tmem + lanes + G::o_at + x * D, tf = tmem + lanes + G::fold_at + x * D;
    float sum_q[4], refs[4];
    int at[4];
    f32x2 sum2[4], off2[4];
    bool live_rows = false;
    int first_at = 0x7fffffff, last_at = -1;  // of the warp's rows
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = kRowsX * x + row0x + 8 * i + r;
      sum_q[i] = sums[n];
      at[i] = -1;
      if (n < live) {
        const int p = clamp_position(base + token_of(i0 + n));
        at[i] = p < max_len ? p : -1;
        live_rows = true;
        first_at = min(first_at, at[i]);
        last_at = max(last_at, at[i]);
      }
      refs[i] = -INFINITY;
      sum2[i] = off2[i] = pair(0.0f, 0.0f);
    }
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      first_at = min(first_at, __shfl_xor_sync(0xFFFFFFFFu, first_at, d));
      last_at = max(last_at, __shfl_xor_sync(0xFFFFFFFFu, last_at, d));
    }
    live_rows = __any_sync(0xFFFFFFFFu, live_rows);
    // a copy for each kind of rows: the test within costs a chunk 235 us in place of 230
    auto walk = [&](auto evenly) {
      bool stop = false;  // the same in all lanes, where `ok` is each lane's own between two votes
      for (int it = 0; it < tiles && !stop; ++it) {
        const int p0 = tile_of(it) * kPos;
        const float* terms = terms_of(it);
        ok = ok && wait_for(&bar.terms_full[it % kTermSets], static_cast<unsigned>(it / kTermSets) & 1u);
        // what the warp's rows see of the tile: all of it, or nothing (first_at, last_at: the lowest and highest, -1 among them)
        const bool whole = live_rows && first_at >= p0 + kPos - 1 && (A.window <= 0 || p0 > last_at - A.window || p0 <= A.sinks - kPos);
        const bool none = last_at < p0 || (A.window > 0 && p0 + kPos - 1 <= first_at - A.window && p0 >= A.sinks);
        // 64 positions at a time: the next ones' scores and the last ones' product are computed meanwhile
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          ok = ok && wait_for(&bar.s_full[x][h], it & 1);
          if (!__all_sync(0xFFFFFFFFu, ok)) {
            ok = false;
            stop = true;
            break;
          }
          tc_fence_after();
          const unsigned th = ts + h * (kPos / 2);
          if (kSplit && h == 0 && it > 0 && it % kFoldTiles == 0) {  // the next product begins anew
            ok = wait_for(&bar.p_free[x][1], (it - 1) & 1);
            tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < 2 * D; c0 += 32) {
              const unsigned at_c = static_cast<unsigned>(c0 / 64 * 32) + (static_cast<unsigned>(c0 / 32 % 2 * 16) << 16);  // 32 columns of 16 rows
              uint32_t o[16], f[16];
              tmem_ld_16x256b_x4(to + at_c, o);
              if (it > kFoldTiles) {
                tmem_ld_16x256b_x4(tf + at_c, f);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float(f[j]));
              }
              tmem_st_16x256b_x4(tf + at_c, o);
            }
          }
          const float4* const t4 = reinterpret_cast<const float4*>(terms) + 3 * (32 * h + c);  // of the pair c; every fourth is ours
          if (none) {
            uint32_t zero[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) zero[i] = 0u;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              tmem_st_16x128b_x8(th + (static_cast<unsigned>(16 * g) << 16), zero);
              if constexpr (kSplit) tmem_st_16x128b_x8(th + kPos / 4 + (static_cast<unsigned>(16 * g) << 16), zero);
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bar.p_full[x][h]);
            continue;
          }
          uint32_t s[2][32];  // [16 rows][4 pair + 2 (8 rows) + position], scores in place
#pragma unroll
          for (int g = 0; g < 2; ++g) tmem_ld_16x256b_x8_begin(th + (static_cast<unsigned>(16 * g) << 16), s[g]);
          tmem_ld_end(s[0], s[1]);
          if constexpr (!decltype(evenly)::value) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const float unit = row_units[kRowsX * x + row0x + 8 * n + r];
#pragma unroll
              for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int j = 4 * i + 2 * (n & 1) + e;
                  s[n >> 1][j] = __float_as_uint(__uint_as_float(s[n >> 1][j]) * unit);
                }
            }
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 k = t4[12 * i];
            const float2 e = *reinterpret_cast<const float2*>(&t4[12 * i + 1]);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int j = 4 * i + 2 * (n & 1);
              const float2 y = unpair(fma2(pair(__uint_as_float(s[n >> 1][j]), __uint_as_float(s[n >> 1][j + 1])), pair(k.x, k.y),
                                           fma2(pair(sum_q[n], sum_q[n]), pair(k.z, k.w), pair(e.x, e.y))));
              s[n >> 1][j] = __float_as_uint(y.x);
              s[n >> 1][j + 1] = __float_as_uint(y.y);
            }
          }
          if (!whole) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int from = A.window > 0 ? at[n] - A.window : -1;
#pragma unroll
              for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int p = p0 + h * (kPos / 2) + 8 * i + 2 * c + e;
                  if (p > at[n] || (p <= from && p >= A.sinks)) s[n >> 1][4 * i + 2 * (n & 1) + e] = 0xff800000u;
                }
            }
          }
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              top[n] = max3(top[n], __uint_as_float(s[n >> 1][4 * i + 2 * (n & 1)]), __uint_as_float(s[n >> 1][4 * i + 2 * (n & 1) + 1]));
          bool raise = false;
#pragma unroll
          for (int n = 0; n < 4; ++n) raise |= top[n] > refs[n] + kRaise;  // the first seen position too: the reference is -inf
          if (__any_sync(0xFFFFFFFFu, raise)) {
            float corr[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              top[n] = fmaxf(top[n], __shfl_xor_sync(0xFFFFFFFFu, top[n], 1));
              top[n] = fmaxf(top[n], __shfl_xor_sync(0xFFFFFFFFu, top[n], 2));
              const float next = fmaxf(refs[n], top[n]);
              corr[n] = next > refs[n] ? ex2(refs[n] - next) : 1.0f;
              refs[n] = next;
              sum2[n] = mul2(sum2[n], pair(corr[n], corr[n]));
              off2[n] = mul2(off2[n], pair(corr[n], corr[n]));
            }
            if (it + h > 0) {  // the last 64 positions' product may be under way
              ok = ok && wait_for(&bar.p_free[x][h ^ 1], (it - (h ^ 1)) & 1);
              tc_fence_after();
            }
            auto rescale = [&](unsigned from) {
#pragma unroll 1
              for (int c0 = 0; c0 < D; c0 += 32)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                  uint32_t o[16];
                  const unsigned at_o = from + c0 + (static_cast<unsigned>(16 * g) << 16);
                  tmem_ld_16x256b_x4(at_o, o);
#pragma unroll
                  for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr[2 * g + ((j >> 1) & 1)]);
                  tmem_st_16x256b_x4(at_o, o);
                }
            };
            if (h > 0 || (kSplit ? it % kFoldTiles != 0 : it > 0)) rescale(to);
            if (kSplit && it >= kFoldTiles) {
              tmem_wait_st();
              rescale(tf);
            }
          }
          f32x2 minus[4];  // a row that has seen nothing yet: its weights are 2^-inf
#pragma unroll
          for (int n = 0; n < 4; ++n) minus[n] = refs[n] == -INFINITY ? pair(0.0f, 0.0f) : pair(-refs[n], -refs[n]);
          uint32_t hi[2][16], lo[2][16];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 mu = reinterpret_cast<const float2*>(t4)[24 * i + 3];
            const float4 uo = t4[12 * i + 2];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int j = 4 * i + 2 * (n & 1);
              const float2 d = unpair(add2(pair(__uint_as_float(s[n >> 1][j]), __uint_as_float(s[n >> 1][j + 1])), minus[n]));
              const f32x2 pw = pair(ex2(d.x), ex2(d.y));
              sum2[n] = fma2(pw, pair(uo.x, uo.y), sum2[n]);
              off2[n] = fma2(pw, pair(uo.z, uo.w), off2[n]);
              const float2 w = unpair(mul2(pw, pair(mu.x, mu.y)));
              hi[n >> 1][2 * i + (n & 1)] = pack_f16(w.x, w.y);
              if constexpr (kSplit) {
                const float2 f = unpack_f16(hi[n >> 1][2 * i + (n & 1)]);
                lo[n >> 1][2 * i + (n & 1)] = pack_f16(w.x - f.x, w.y - f.y);
              }
            }
          }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            tmem_st_16x128b_x8(th + (static_cast<unsigned>(16 * g) << 16), hi[g]);
            if constexpr (kSplit) tmem_st_16x128b_x8(th + kPos / 4 + (static_cast<unsigned>(16 * g) << 16), lo[g]);
          }
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&bar.p_full[x][h]);
        }
      }
    };
    if (even) walk(std::true_type{});
    else walk(std::false_type{});
    if (tiles > 0) ok = __all_sync(0xFFFFFFFFu, ok && wait_for(&bar.p_free[x][1], (tiles - 1) & 1)) != 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float2 s = unpair(sum2[n]), f = unpair(off2[n]);
      float l = s.x + s.y, o = f.x + f.y;
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
      o += __shfl_xor_sync(0xFFFFFFFFu, o, 1);
      o += __shfl_xor_sync(0xFFFFFFFFu, o, 2);
      if (c == 0) {
        const int row = kRowsX * x + row0x + 8 * n + r;
        refs_of[row] = refs[n];
        totals[row] = ok ? l : __uint_as_float(0x7fffffffu);  // a row whose wait ran out becomes NaN, in all of a cluster
        offsets[row] = o;
      }
    }
  }
  tc_fence_before();
  __syncthreads();  // all products are done: the operands' place is free
  tc_fence_after();
  // now a thread has a row of its own: tensor-memory lane tid % 128 of row tile x
  const int row = tid & (kRowsCta - 1);
  const unsigned to = tmem + (static_cast<unsigned>(32 * (warp & 3)) << 16) + G::o_at + x * D;
  const bool mine = tid < kSoftmaxThreads && x < row_tiles;
  auto load_o = [&](int c0, uint32_t (&o)[16]) {  // 16 channels of the row
    tmem_ld16(to + c0, o);
    if (kSplit && tiles > kFoldTiles) {
      uint32_t f[16];
      tmem_ld16(to + (G::fold_at - G::o_at) + c0, f);
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float(f[j]));
    }
  };
  if (C == 1) {
    if (mine) {
      // through the place of its tile's queries, to leave in whole 16-byte chunks: 32 rows a warp
      const float total = totals[row], offset = offsets[row], inv = total == 0.0f ? 0.0f : 1.0f / total;
      uint4* const stage = reinterpret_cast<uint4*>(smem + G::q_at) + (32 * warp) * L;
      auto chunk_of = [&](int r, int c) { return stage + r * L + (c ^ (r & (L < 8 ? L - 1 : 7))); };
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 16) {
        uint32_t o[16];
        if (tiles > 0 && ok) load_o(c0, o);
        else
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = 0u;
#pragma unroll
        for (int c = 0; c < 16 / kPer; ++c) {
          union {
            uint4 w;
            T t[kPer];
          } u;
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            u.t[j] = from_f32<T>(total == 0.0f ? 0.0f : fmaf(__uint_as_float(o[kPer * c + j]), 1.0f / kWeightUnit, offset) * inv);
          *chunk_of(lane, c0 / kPer + c) = u.w;
        }
      }
      __syncwarp();
#pragma unroll
      for (int k = 0; k < L; ++k) {
        const int r = (32 / L) * k + lane / L, c = lane % L;
        const int n = kRowsX * x + 32 * (warp & 3) + r;
        if (n < live) {
          T* out = const_cast<T*>(item_row(A.out, i0 + n, A.o_row, A.o_head)) + c * kPer;
          union {
            uint4 w;
            T t[kPer];
          } u;
          u.w = *chunk_of(r, c);
          if (A.o_vec) {
            *reinterpret_cast<uint4*>(out) = u.w;
          } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) out[j] = u.t[j];
          }
        }
      }
    }
  } else {
    // every CTA leaves its O [channel][row], and finishes D / C channels of all rows
    float* const part = reinterpret_cast<float*>(smem);
    static_assert(D * kRowsCta * 4 <= G::smem, "shared memory");
    if (mine) {
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 16) {
        uint32_t o[16];
        if (tiles > 0 && ok) load_o(c0, o);
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c0 + j) * kRowsCta + row] = tiles > 0 && ok ? __uint_as_float(o[j]) : 0.0f;
      }
    }
    cluster.sync();
    if (mine && row < live) {
      T* out = const_cast<T*>(item_row(A.out, i0 + row, A.o_row, A.o_head));
      float top = -INFINITY, l = 0.0f, off = 0.0f, scale[4];
      for (int k = 0; k < C; ++k) top = fmaxf(top, cluster.map_shared_rank(refs_of, k)[row]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        scale[k] = 0.0f;
        if (k < C) {
          const float theirs = cluster.map_shared_rank(totals, k)[row];
          if (theirs != 0.0f) {  // zero: the CTA saw nothing for this row
            scale[k] = ex2(cluster.map_shared_rank(refs_of, k)[row] - top);
            l = fmaf(theirs, scale[k], l);
            off = fmaf(cluster.map_shared_rank(offsets, k)[row], scale[k], off);
          }
        }
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      for (int c = rank * (D / C); c < (rank + 1) * (D / C); c += 8) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < C && scale[k] != 0.0f) {
            const float* other = cluster.map_shared_rank(part, k) + c * kRowsCta + row;
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = fmaf(other[j * kRowsCta], scale[k], y[j]);
          }
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = l == 0.0f ? 0.0f : fmaf(y[j], 1.0f / kWeightUnit, off) * inv;
        store_values<T, 8>(out + c, A.o_vec, y);
      }
    }
    cluster.sync();  // no CTA leaves while another reads its shared memory
  }
  if (!ok) which[2] = 1;
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && which[2] != 0 && A.error != nullptr) atomicCAS(A.error, 0u, static_cast<unsigned>(IVB_ETIMEOUT));
  if (warp == kIssueWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::columns));
  }
}

template <int D, typename T>
int32_t launch_prompts(const Kv4Attention& A, int few, cudaStream_t stream) {
  using G = PromptGeometry<D, std::is_same<T, float>::value>;
  static std::atomic<uint64_t> done{0};
  int device = 0;
  IVB_CUDA(cudaGetDevice(&device));
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if ((done.load(std::memory_order_relaxed) & bit) == 0) {
    IVB_CUDA(cudaFuncSetAttribute(kv4_prompt_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::smem));
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  // as many tiles as the rows can make: each sequence of the call may leave one unfilled
  const int64_t items = static_cast<int64_t>(A.rows) * A.group;
  const int64_t sequences = std::min<int64_t>(A.cache.batch, items / (few + 1));
  const int64_t tiles = items / G::rows + sequences;
  if (tiles * A.cache.kv_heads > 0x1fffffff) return fail(IVB_EINVAL, "ivb_kv4_attention: %lld tiles of rows in one call", static_cast<long long>(tiles));
  // a cluster where one CTA each would leave SMs without work (128 CTAs of a 2048-row causal prompt: 68 us, in pairs 56, in fours
  // 88; 256 CTAs of a chunk under a window: 228, in pairs 275; each pair measured on one day's kernel)
  int C = 1;
  while (C < 4 && tiles * A.cache.kv_heads * C < 148 && A.cache.max_len > 2 * C * kPos) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * A.cache.kv_heads * C));
  cfg.blockDim = dim3(kPromptThreads);
  cfg.dynamicSmemBytes = G::smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = kv4_attributes(C, attr);
  IVB_CUDA(cudaLaunchKernelEx(&cfg, kv4_prompt_kernel<D, T>, A, few));
  return IVB_OK;
}

template <typename T>
int32_t launch_dim(const Kv4Attention& A, int few, cudaStream_t stream) {
  switch (A.cache.head_dim) {
    case 32: return launch_prompts<32, T>(A, few, stream);
    case 64: return launch_prompts<64, T>(A, few, stream);
    default: return launch_prompts<128, T>(A, few, stream);
  }
}

}  // namespace

int32_t launch_kv4_prompts(const Kv4Attention& A, int32_t dtype, int few, cudaStream_t stream) {
  if (dtype == IVB_F32) return launch_dim<float>(A, few, stream);
  if (dtype == IVB_F16) return launch_dim<__half>(A, few, stream);
  return launch_dim<__nv_bfloat16>(A, few, stream);
}

}  // namespace ivb
