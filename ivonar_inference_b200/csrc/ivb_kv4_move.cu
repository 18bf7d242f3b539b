// The 4-bit key/value cache: sequences that begin as others do (fork), and rows that move up (compact). What is moved is the words
// of a tile (layout: ivb_kv4.cuh), each of which belongs to one position.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "ivb_common.h"
#include "ivb_device.cuh"
#include "ivb_kv4.cuh"

namespace ivb {

int32_t check_kv4(const IvbKv4Cache* c, const char* who);
int32_t check_kv4_rows(const IvbKv4Cache* c, const int32_t* starts, const int64_t* positions, int32_t rows, int32_t dtype, const char* who);

namespace {

namespace cg = cooperative_groups;

// The position (0..15) that word `w` of a tile belongs to.
template <int D>
__device__ __forceinline__ int kv4_position_of_word(int w) {
  if (w < 2 * D) {  // keys (kv4_key_word)
    const int lane = D == 128 ? (w & 127) >> 2 : D == 64 ? w >> 2 : w >> 1;
    const int half = D == 128 ? w >> 7 : D == 64 ? (w >> 1) & 1 : w & 1;
    const int r = lane >> 2;
    return 4 * (r >> 1) + (r & 1) + 2 * half;
  }
  if (w < 4 * D) return w & 15;  // values (kv4_value_word): word 16 i + p of theirs
  return (w - 4 * D) >> 1;
}

constexpr int kForkThreads = 512, kForkPer = 8;  // 16-byte pieces of a thread at a time

// A CTA takes pieces of a run of `across` x 16 bytes of one head at the same place of every sequence, kForkThreads * kForkPer
// at a time: read all, a barrier, write all. In one cache `batch` x `across` pieces fit that, so whatever sequence another's
// beginning comes from is read before any of its bytes at that place is written, in any permutation and without a copy elsewhere.
template <int D>
__global__ void __launch_bounds__(kForkThreads) kv4_fork_kernel(IvbKv4Cache to, IvbKv4Cache from, const int64_t* sources,
                                                                const int64_t* lengths, int across, uint32_t* error) {
  constexpr int kTile = kv4_tile_bytes(D), kPieces = kTile / 16;  // of a tile
  __shared__ int longest_of[kForkThreads / 32];
  const int tid = threadIdx.x;
  pdl_enter();
  const int64_t most = min(to.max_len, from.max_len);
  // what a sequence takes: its source (-1: nothing) and its length
  auto taken = [&](int b, int& source) {
    const int64_t s = sources[b], n = lengths[b];
    const bool there = s >= 0 && n > 0 && (s != b || to.data != from.data);
    source = there && s < from.batch && n <= most ? static_cast<int>(s) : -1;
    if (there && source < 0 && blockIdx.x == 0 && error != nullptr) atomicCAS(error, 0u, static_cast<unsigned>(n > most ? IVB_ECAPACITY : IVB_EINVAL));
    return source < 0 ? 0 : static_cast<int>(n);
  };
  int longest = 0;
  for (int b = tid; b < to.batch; b += kForkThreads) {
    int source;
    longest = max(longest, taken(b, source));
  }
  longest = __reduce_max_sync(0xFFFFFFFFu, longest);
  if ((tid & 31) == 0) longest_of[tid >> 5] = longest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kForkThreads / 32; ++w) longest = max(longest, longest_of[w]);
  const int64_t to_step = kv4_tiles(to.max_len) * kPieces, from_step = kv4_tiles(from.max_len) * kPieces;  // of a head
  const int runs = static_cast<int>(((longest + 15) / 16 * static_cast<int64_t>(kPieces) + across - 1) / across);
  const int together = kForkThreads * kForkPer / across;  // sequences
  const int blocks = (to.batch + together - 1) / together;
  const int64_t items = static_cast<int64_t>(runs) * to.kv_heads * blocks;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int b0 = static_cast<int>(item % blocks) * together;
    const int64_t rest = item / blocks;
    const int run = static_cast<int>(rest % runs), head = static_cast<int>(rest / runs);
    uint4 v[kForkPer];
    uint4* at[kForkPer];
    int left[kForkPer];  // positions taken, from the piece's tile's first on
#pragma unroll
    for (int i = 0; i < kForkPer; ++i) {
      const int n = i * kForkThreads + tid, b = b0 + n / across;
      const int64_t piece = static_cast<int64_t>(run) * across + n % across;
      left[i] = 0;
      if (n < together * across && b < to.batch) {
        int source;
        const int length = taken(b, source);
        left[i] = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(16), length - piece / kPieces * 16)));
        if (left[i] > 0) {
          v[i] = __ldcg(static_cast<const uint4*>(from.data) + (static_cast<int64_t>(source) * from.kv_heads + head) * from_step + piece);
          at[i] = static_cast<uint4*>(to.data) + (static_cast<int64_t>(b) * to.kv_heads + head) * to_step + piece;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kForkPer; ++i) {
      if (left[i] == 16) {
        *at[i] = v[i];
      } else if (left[i] > 0) {  // the positions behind stay as they are
        const int n = i * kForkThreads + tid;
        const int word = static_cast<int>((static_cast<int64_t>(run) * across + n % across) % kPieces) * 4;
        uint32_t* w = reinterpret_cast<uint32_t*>(at[i]);
        if (kv4_position_of_word<D>(word) < left[i]) w[0] = v[i].x;
        if (kv4_position_of_word<D>(word + 1) < left[i]) w[1] = v[i].y;
        if (kv4_position_of_word<D>(word + 2) < left[i]) w[2] = v[i].z;
        if (kv4_position_of_word<D>(word + 3) < left[i]) w[3] = v[i].w;
      }
    }
  }
}

constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32;

// One cluster per (sequence, head), a tile of 16 destinations a warp at a time. A row comes from its own place or behind, so a turn's
// destinations are no later turn's sources: a turn's reads come before its writes (a barrier of the cluster), and the next
// turn's reads may come before these too.
template <int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_compact_kernel(IvbKv4Cache C, const int64_t* index, const int64_t* positions,
                                                                   const int32_t* starts, int rows, uint32_t* error) {
  constexpr int kTile = kv4_tile_bytes(D), kWords = kTile / 4, kPer = kWords / 32;  // words of a lane: 5, 9 or 17
  static_assert(kWords % 32 == 0, "words of a tile");
  cg::cluster_group cluster = cg::this_cluster();
  const int N = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int unit = blockIdx.x / static_cast<unsigned>(N), b = unit / C.kv_heads, head = unit - b * C.kv_heads;
  pdl_enter();
  int row0 = b, count = 1;
  int64_t before = 0;  // rows of the sequence that the call does not have
  if (starts != nullptr) {
    row0 = max(0, starts[b]);
    before = static_cast<int64_t>(row0) - starts[b];
    count = max(0, min(rows, starts[b + 1]) - row0);
  }
  const int64_t base = kv4_position(positions, b) + before;  // of the first row
  unsigned char* const data = static_cast<unsigned char*>(C.data) + (static_cast<int64_t>(b) * C.kv_heads + head) * kv4_tiles(C.max_len) * kTile;
  // destinations lo .. hi - 1, a tile of them a warp
  const int64_t lo = max(base, static_cast<int64_t>(0)), hi = min(base + count, static_cast<int64_t>(C.max_len));
  if (base + count > C.max_len && head == 0 && rank == 0 && error != nullptr) {  // rows beyond the capacity, but for idle ones
    for (int64_t i = max(static_cast<int64_t>(0), C.max_len - base) + threadIdx.x; i < count; i += kMoveThreads)
      if (index[row0 + i] >= 0) atomicCAS(error, 0u, static_cast<unsigned>(IVB_ECAPACITY));
  }
  const int64_t tile0 = lo >> 4, tiles = hi > lo ? ((hi + 15) >> 4) - tile0 : 0, turns = (tiles + N * kMoveWarps - 1) / (N * kMoveWarps);
  // lane l < 16 has the source of the tile's position l, -1 where nothing is written
  auto source_of = [&](int64_t turn) {
    const int64_t t = turn * N * kMoveWarps + rank * kMoveWarps + warp, p = ((tile0 + t) << 4) + lane;
    if (t >= tiles || lane >= 16 || p < lo || p >= hi) return static_cast<int64_t>(-1);
    const int64_t s = index[row0 + (p - base)];
    if (s < 0 || s == p) return static_cast<int64_t>(-1);
    if (s < p || s >= C.max_len) {
      if (head == 0 && error != nullptr) atomicCAS(error, 0u, static_cast<unsigned>(s < p ? IVB_EINVAL : IVB_ECAPACITY));
      return static_cast<int64_t>(-1);
    }
    return s;
  };
  auto read = [&](int64_t source, uint32_t (&v)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int w = 32 * i + lane, p = kv4_position_of_word<D>(w);
      const int64_t s = __shfl_sync(0xFFFFFFFFu, source, p);
      if (s >= 0) {
        const int q = static_cast<int>(s & 15);
        // the same word of position q (kv4_key_word, kv4_value_word, scales and offsets)
        int from;
        if (w < 2 * D) from = kv4_key_word<D>(q, (w >> (D == 32 ? 1 : 2) & 3) * (D / 32) + (w & (D / 32 - 1)));
        else if (w < 4 * D) from = (w & ~15) | q;
        else from = 4 * D + 2 * q + (w & 1);
        v[i] = __ldcg(reinterpret_cast<const uint32_t*>(data + (s >> 4) * kTile) + from);
      }
    }
  };
  uint32_t next[kPer];
  int64_t source = source_of(0);
  read(source, next);
  for (int64_t turn = 0; turn < turns; ++turn) {
    uint32_t v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = next[i];
    const int64_t mine = source;
    // the words have to be there before another warp of the cluster writes: used, not only asked for
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) any |= v[i];
    asm volatile("" ::"r"(any) : "memory");
    if (turn + 1 < turns) {
      source = source_of(turn + 1);
      read(source, next);
    }
    cluster.sync();
    const int64_t t = turn * N * kMoveWarps + rank * kMoveWarps + warp;
    uint32_t* const to = reinterpret_cast<uint32_t*>(data + (tile0 + t) * kTile);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int w = 32 * i + lane;
      const int64_t s = __shfl_sync(0xFFFFFFFFu, mine, kv4_position_of_word<D>(w));
      if (s >= 0) to[w] = v[i];
    }
  }
}

// The storage's bytes; sizes are checked before.
int64_t bytes_of(const IvbKv4Cache& c) { return static_cast<int64_t>(c.batch) * c.kv_heads * kv4_tiles(c.max_len) * kv4_tile_bytes(c.head_dim); }

template <int D>
int32_t launch_fork(const IvbKv4Cache& to, const IvbKv4Cache& from, const int64_t* sources, const int64_t* lengths, uint32_t* error,
                    cudaStream_t stream) {
  constexpr int kPieces = kForkThreads * kForkPer;
  int across = 64;
  if (to.data == from.data)
    while (across * static_cast<int64_t>(to.batch) > kPieces) across /= 2;
  const int64_t pieces = kv4_tiles(std::min(to.max_len, from.max_len)) * (kv4_tile_bytes(D) / 16), together = kPieces / across;
  const int64_t items = (pieces + across - 1) / across * to.kv_heads * ((to.batch + together - 1) / together);
  IVB_CUDA(launch_pdl(kv4_fork_kernel<D>, dim3(static_cast<unsigned>(std::min<int64_t>(items, 148 * 2))), dim3(kForkThreads), 0, stream, to, from,
                      sources, lengths, across, error));
  return IVB_OK;
}

template <int D>
int32_t launch_compact(const IvbKv4Cache& c, const int64_t* index, const int64_t* positions, const int32_t* starts, int32_t rows, uint32_t* error,
                       cudaStream_t stream) {
  const int64_t units = static_cast<int64_t>(c.batch) * c.kv_heads;
  // a cluster where a sequence may have more rows than a CTA moves at a time and the sequences alone leave SMs without work
  int N = 1;
  while (N < 8 && units * N < 148 * 4 && rows / c.batch > N * kMoveWarps * 16) N *= 2;
  if (units * N > 0x7fffffff) return fail(IVB_EINVAL, "ivb_kv4_compact: %d sequences of %d heads", c.batch, c.kv_heads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(units * N));
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(N);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = N > 1 ? 2 : 1;
  IVB_CUDA(cudaLaunchKernelEx(&cfg, kv4_compact_kernel<D>, c, index, positions, starts, static_cast<int>(rows), error));
  return IVB_OK;
}

}  // namespace
}  // namespace ivb

extern "C" {

int32_t ivb_kv4_fork(const IvbKv4Cache* c, const IvbKv4Cache* source, const int64_t* sources, const int64_t* lengths, uint32_t* error,
                     void* stream) {
  using namespace ivb;
  if (int32_t rc = check_kv4(c, "ivb_kv4_fork")) return rc;
  if (source == nullptr) source = c;
  if (int32_t rc = check_kv4(source, "ivb_kv4_fork")) return rc;
  if (source->kv_heads != c->kv_heads || source->head_dim != c->head_dim)
    return fail(IVB_EINVAL, "ivb_kv4_fork: %d heads x %d from a cache of %d x %d", c->kv_heads, c->head_dim, source->kv_heads, source->head_dim);
  if (sources == nullptr || lengths == nullptr) return fail(IVB_EINVAL, "ivb_kv4_fork: null sources or lengths");
  const bool same = source->data == c->data && source->batch == c->batch && source->max_len == c->max_len;
  const char *a = static_cast<const char*>(c->data), *b = static_cast<const char*>(source->data);
  if (!same && a < b + bytes_of(*source) && b < a + bytes_of(*c)) return fail(IVB_EINVAL, "ivb_kv4_fork: the caches share memory");
  if (same && c->batch > kForkThreads * kForkPer)
    return fail(IVB_EINVAL, "ivb_kv4_fork: %d sequences within one cache (%d at most)", c->batch, kForkThreads * kForkPer);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->head_dim == 32) return launch_fork<32>(*c, *source, sources, lengths, error, s);
  if (c->head_dim == 64) return launch_fork<64>(*c, *source, sources, lengths, error, s);
  return launch_fork<128>(*c, *source, sources, lengths, error, s);
}

int32_t ivb_kv4_compact(const IvbKv4Cache* c, const int64_t* index, const int32_t* starts, const int64_t* positions, int32_t rows, uint32_t* error,
                        void* stream) {
  using namespace ivb;
  if (int32_t rc = check_kv4(c, "ivb_kv4_compact")) return rc;
  if (int32_t rc = check_kv4_rows(c, starts, positions, rows, IVB_F32, "ivb_kv4_compact")) return rc;
  if (rows == 0) return IVB_OK;
  if (index == nullptr) return fail(IVB_EINVAL, "ivb_kv4_compact: null index");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->head_dim == 32) return launch_compact<32>(*c, index, positions, starts, rows, error, s);
  if (c->head_dim == 64) return launch_compact<64>(*c, index, positions, starts, rows, error, s);
  return launch_compact<128>(*c, index, positions, starts, rows, error, s);
}

}  // extern "C"
