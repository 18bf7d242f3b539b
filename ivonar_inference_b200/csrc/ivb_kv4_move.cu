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
constexpr int kForkPieces = kForkThreads * kForkPer;

// A CTA takes runs of `across` (a power of two) pieces of one head at the same place of every sequence, kForkPieces at a time: read all,
// a barrier, write all. In one cache `batch` x `across` pieces fit that, so whatever sequence another's beginning comes from is read
// before any of its bytes at that place is written, in any permutation and without a copy elsewhere. Two CTAs an SM: one reads while
// the other writes. Bound by the writes: 64 x 2048 positions x 8 heads x 128 from one sequence 27.7 us (145 MB, 5.2 TB/s), 96 of 128 sequences of
// 300-700 x 16 x 64 in place 22.6 (74 MB, 3.3 TB/s: runs of 512 bytes there, and sequences that end early).
template <int D>
__global__ void __launch_bounds__(kForkThreads, 2) kv4_fork_kernel(IvbKv4Cache to, IvbKv4Cache from, const int64_t* sources,
                                                                   const int64_t* lengths, int across_log, uint32_t* error) {
  constexpr int kPieces = kv4_tile_bytes(D) / 16;  // of a tile
  __shared__ int longest_of[kForkThreads / 32];
  __shared__ int2 takes[kForkPieces];  // of the sequences at hand: source and length, 0 where nothing is taken
  const int tid = threadIdx.x;
  pdl_enter();
  const int64_t most = min(to.max_len, from.max_len);
  auto taken = [&](int b) {
    const int64_t s = sources[b], n = lengths[b];
    const bool wanted = s >= 0 && n > 0 && (s != b || to.data != from.data), there = wanted && s < from.batch && n <= most;
    if (wanted && !there && blockIdx.x == 0 && error != nullptr) atomicCAS(error, 0u, static_cast<unsigned>(n > most ? IVB_ECAPACITY : IVB_EINVAL));
    return there ? make_int2(static_cast<int>(s), static_cast<int>(n)) : make_int2(0, 0);
  };
  const int across = 1 << across_log, together = kForkPieces >> across_log;  // sequences at a time
  const int blocks = (to.batch + together - 1) / together;
  int longest = 0;
  for (int b = tid; b < to.batch; b += kForkThreads) {
    const int2 t = taken(b);
    longest = max(longest, t.y);
    if (blocks == 1) takes[b] = t;
  }
  longest = __reduce_max_sync(0xFFFFFFFFu, longest);
  if ((tid & 31) == 0) longest_of[tid >> 5] = longest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kForkThreads / 32; ++w) longest = max(longest, longest_of[w]);
  const int64_t to_step = kv4_tiles(to.max_len) * kPieces, from_step = kv4_tiles(from.max_len) * kPieces;  // of a head
  const unsigned runs = static_cast<unsigned>(((longest + 15) / 16 * static_cast<int64_t>(kPieces) + across - 1) >> across_log);
  const unsigned items = runs * static_cast<unsigned>(to.kv_heads) * static_cast<unsigned>(blocks);  // of 1 KB at least: below 2^32
  for (unsigned item = blockIdx.x; item < items; item += gridDim.x) {
    const unsigned rest = item / static_cast<unsigned>(blocks);
    const int b0 = static_cast<int>(item - rest * blocks) * together;
    const int head = static_cast<int>(rest / runs), run = static_cast<int>(rest - head * runs);
    if (blocks > 1) {
      __syncthreads();  // the last item's are no longer read
      for (int i = tid; i < together && b0 + i < to.batch; i += kForkThreads) takes[i] = taken(b0 + i);
      __syncthreads();
    }
    // A thread's pieces stand at one place of sequences kForkThreads / across apart; what has the last one's source, as the answers to one
    // prompt have, is not read again.
    const int64_t piece = (static_cast<int64_t>(run) << across_log) + (tid & (across - 1));
    const int first = static_cast<int>(piece / kPieces) * 16;  // position of the piece's tile
    const int i0 = tid >> across_log, step = kForkThreads >> across_log;
    const int64_t from_stride = from.kv_heads * from_step, to_stride = to.kv_heads * to_step;  // of a sequence
    const uint4* const source = static_cast<const uint4*>(from.data) + head * from_step + piece;
    uint4* at = static_cast<uint4*>(to.data) + (b0 + i0) * to_stride + head * to_step + piece;
    const int there = min(together, to.batch - b0);
    uint4 v[kForkPer], held = make_uint4(0u, 0u, 0u, 0u);
    unsigned reads = 0;  // which of them are read
    int last = -1;       // the source at hand
#pragma unroll
    for (int i = 0; i < kForkPer; ++i) {
      const int b = i0 + i * step;
      if (b >= there) break;
      const int2 t = takes[b];
      if (first < t.y && t.x != last) {
        last = t.x;
        reads |= 1u << i;
        v[i] = __ldcg(source + last * from_stride);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kForkPer; ++i, at += step * to_stride) {
      const int b = i0 + i * step;
      if (b >= there) break;
      const int left = takes[b].y - first;  // positions taken from the tile's first on
      if (reads >> i & 1) held = v[i];
      if (left <= 0) continue;
      if (left >= 16) {
        *at = held;
      } else {  // the positions behind stay as they are
        const int word = static_cast<int>(piece % kPieces) * 4;
        uint32_t* const w = reinterpret_cast<uint32_t*>(at);
        if (kv4_position_of_word<D>(word) < left) w[0] = held.x;
        if (kv4_position_of_word<D>(word + 1) < left) w[1] = held.y;
        if (kv4_position_of_word<D>(word + 2) < left) w[2] = held.z;
        if (kv4_position_of_word<D>(word + 3) < left) w[3] = held.w;
      }
    }
  }
}

constexpr int kMoveWarps = 16;  // at most: so many tiles a CTA moves at a time

// One cluster per (sequence, head), a tile of 16 destinations a warp at a time. A row comes from its own place or behind, so a turn's
// destinations are no later turn's sources: a turn's reads come before its writes (a barrier with release and acquire), and the next
// turn's reads may come before these too, as the index of the one after that does. Lane l < 16 holds the source of the tile's position l;
// a word finds its row's by a shuffle, and moves to the same word of another position: the keys' words are 4 c + w plus what depends on
// the position alone (kv4_key_word), the values' 16 i + p, the scales' 2 p + w. Bound by a turn's latency where sequences x heads are few: 54,800
// rows of four sequences x 8 heads x 128 27.9 us (118 MB, 4.2 TB/s), 64 sequences x 16 heads x 64 of 1-6 rows 2.9.
template <int D>
__global__ void __launch_bounds__(32 * kMoveWarps) kv4_compact_kernel(IvbKv4Cache C, const int64_t* index, const int64_t* positions,
                                                                   const int32_t* starts, int rows, uint32_t* error) {
  constexpr int kTile = kv4_tile_bytes(D), kWords = kTile / 4, kPer = kWords / 32;  // words of a lane: 5, 9 or 17
  static_assert(kWords % 32 == 0, "words of a tile");
  cg::cluster_group cluster = cg::this_cluster();
  const int N = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
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
  if (base + count > C.max_len && head == 0 && rank == 0 && error != nullptr) {  // rows beyond the capacity, but for idle ones
    for (int64_t i = max(static_cast<int64_t>(0), C.max_len - base) + threadIdx.x; i < count; i += 32 * W)
      if (index[row0 + i] >= 0) atomicCAS(error, 0u, static_cast<unsigned>(IVB_ECAPACITY));
  }
  // destinations lo .. hi - 1, a tile of them a warp
  const int64_t lo64 = max(base, static_cast<int64_t>(0)), hi64 = min(base + count, static_cast<int64_t>(C.max_len));
  const int lo = static_cast<int>(min(lo64, static_cast<int64_t>(C.max_len))), hi = static_cast<int>(max(hi64, static_cast<int64_t>(0)));
  const int tile0 = lo >> 4, tiles = hi > lo ? ((hi + 15) >> 4) - tile0 : 0, each = N * W, turns = (tiles + each - 1) / each;
  auto tile_of = [&](int turn) { return turn * each + rank * W + warp; };
  // -1: nothing is written; what index holds is checked when it is there
  auto ask = [&](int turn) {
    const int t = tile_of(turn), p = ((tile0 + t) << 4) + lane;
    return t < tiles && lane < 16 && p >= lo && p < hi ? index[row0 + (p - base)] : static_cast<int64_t>(-1);
  };
  auto source_of = [&](int turn, int64_t s) {
    const int p = ((tile0 + tile_of(turn)) << 4) + lane;
    if (s < 0 || s == p) return -1;
    if (s < p || s >= C.max_len) {
      if (head == 0 && error != nullptr) atomicCAS(error, 0u, static_cast<unsigned>(s < p ? IVB_EINVAL : IVB_ECAPACITY));
      return -1;
    }
    return static_cast<int>(s);
  };
  auto read = [&](int source, uint32_t (&v)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int w = 32 * i + lane, s = __shfl_sync(0xFFFFFFFFu, source, kv4_position_of_word<D>(w)), q = s & 15;
      if (s >= 0) {
        int from;
        if (w < 2 * D) from = kv4_key_word<D>(q, (w >> (D == 32 ? 1 : 2) & 3) * (D / 32) + (w & (D / 32 - 1)));
        else if (w < 4 * D) from = (w & ~15) | q;
        else from = 4 * D + 2 * q + (w & 1);
        v[i] = __ldcg(reinterpret_cast<const uint32_t*>(data + static_cast<int64_t>(s >> 4) * kTile) + from);
      }
    }
  };
  if (turns == 0) return;  // the whole cluster
  uint32_t next[kPer];
  int source = source_of(0, ask(0));
  int64_t asked = ask(1);
  read(source, next);
  for (int turn = 0; turn < turns; ++turn) {
    uint32_t v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = next[i];
    const int mine = source;
    // This turn's reads are ordered before all of its writes, other warps' and CTAs' too: by a barrier with release and acquire, on the two
    // sides of what the next turn asks and reads.
    if (N > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (turn + 1 < turns) {
      source = source_of(turn + 1, asked);
      asked = ask(turn + 2);
      read(source, next);
    }
    if (N > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
    uint32_t* const to = reinterpret_cast<uint32_t*>(data + static_cast<int64_t>(tile0 + tile_of(turn)) * kTile);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int w = 32 * i + lane;
      if (__shfl_sync(0xFFFFFFFFu, mine, kv4_position_of_word<D>(w)) >= 0) to[w] = v[i];
    }
  }
}

// The storage's bytes; sizes are checked before.
int64_t bytes_of(const IvbKv4Cache& c) { return static_cast<int64_t>(c.batch) * c.kv_heads * kv4_tiles(c.max_len) * kv4_tile_bytes(c.head_dim); }

template <int D>
int32_t launch_fork(const IvbKv4Cache& to, const IvbKv4Cache& from, const int64_t* sources, const int64_t* lengths, uint32_t* error,
                    cudaStream_t stream) {
  // runs of 1 KB, shorter ones where a cache's many sequences would not fit otherwise
  int across_log = 6;
  if (to.data == from.data)
    while ((static_cast<int64_t>(to.batch) << across_log) > kForkPieces) --across_log;
  const int64_t pieces = kv4_tiles(std::min(to.max_len, from.max_len)) * (kv4_tile_bytes(D) / 16), together = kForkPieces >> across_log;
  const int64_t items = ((pieces + (1 << across_log) - 1) >> across_log) * to.kv_heads * ((to.batch + together - 1) / together);
  IVB_CUDA(launch_pdl(kv4_fork_kernel<D>, dim3(static_cast<unsigned>(std::min<int64_t>(items, 148 * 2))), dim3(kForkThreads), 0, stream, to, from,
                      sources, lengths, across_log, error));
  return IVB_OK;
}

template <int D>
int32_t launch_compact(const IvbKv4Cache& c, const int64_t* index, const int64_t* positions, const int32_t* starts, int32_t rows, uint32_t* error,
                       cudaStream_t stream) {
  const int64_t units = static_cast<int64_t>(c.batch) * c.kv_heads;
  // Warps by the rows of a sequence, if they are spread evenly (64 x 16 heads of 1-6 rows: 10 us with 16 warps); a cluster where these are
  // more than a CTA moves at a time and the sequences alone leave SMs without work.
  const int64_t tiles = rows / c.batch / 16 + 2;
  int W = 1, N = 1;
  while (W < kMoveWarps && W < tiles) W *= 2;
  while (N < 8 && units * N < 148 * 4 && tiles > N * W) N *= 2;
  if (units * N > 0x7fffffff) return fail(IVB_EINVAL, "ivb_kv4_compact: %d sequences of %d heads", c.batch, c.kv_heads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(units * N));
  cfg.blockDim = dim3(static_cast<unsigned>(32 * W));
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
  if (same && c->batch > kForkPieces)
    return fail(IVB_EINVAL, "ivb_kv4_fork: %d sequences within one cache (%d at most)", c->batch, kForkPieces);
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
