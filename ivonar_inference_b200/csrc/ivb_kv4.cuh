// Layout and row lookup of the 4-bit key/value cache, shared by its kernels (ivb_kv4.cu, ivb_kv4_attention.cu, ivb_kv4_prompt.cu).
//
// A row x of D values (one position of one key/value head) is kept as codes u in 0..15 with one fp16 scale s and
// one fp16 offset m, x ~ m + s u. Sixteen positions of one head form a tile of 16 (D + 8) bytes:
//   [key codes, 8 D bytes][value codes, 8 D bytes][16 x (key scale, key offset, value scale, value offset) fp16]
// The order of the 32-bit code words inside a tile is that of the B operands of mma.m16n8k16, lane by lane, so that
// the attention kernels read whole 16-byte chunks and need no transposition:
//   keys    lane 4 r + c holds the channels D/4 c .. D/4 (c + 1) - 1 of the positions 4 (r / 2) + r % 2 and that + 2
//   values  lane 4 r + c holds the channel word r (and r + 8 at D = 128) of the positions 4 c .. 4 c + 3
// A word holds 8 channels, channel 2 j in nibble j and channel 2 j + 1 in nibble j + 4: masking (w >> 8 i) with
// 0x000f000f or 0x00f000f0 leaves two neighbouring channels in the two halves of a word, as an fp16 operand has them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace ivb {

constexpr int kKv4Tile = 16;   // positions of a tile
constexpr int kKv4Group = 32;  // positions are allocated in groups of two tiles

__host__ __device__ constexpr int kv4_tile_bytes(int dim) { return 16 * (dim + 8); }
__host__ __device__ constexpr int64_t kv4_tiles(int max_len) { return 2 * ((static_cast<int64_t>(max_len) + 31) / 32); }

// Word number, from the start of the tile, of channels 8 i .. 8 i + 7 of position p (0..15) of the tile.
template <int D>
__device__ __forceinline__ int kv4_key_word(int p, int i) {
  constexpr int n = D / 32;
  const int lane = (2 * (p >> 2) + (p & 1)) * 4 + i / n, half = (p >> 1) & 1;
  return D == 128 ? 128 * half + 4 * lane + i % n : (n * 2) * lane + n * half + i % n;
}
template <int D>
__device__ __forceinline__ int kv4_value_word(int p, int i) {
  return 2 * D + 128 * (i >> 3) + (4 * (i & 7) + (p >> 2)) * 4 + (p & 3);
}

// The sequence that row `row` belongs to (starts [batch + 1] ascending; nullptr: row b is sequence b's only row),
// found by the whole warp: the number of sequences that end at or before it. `batch` where there is none.
__device__ __forceinline__ int kv4_sequence(const int32_t* starts, int batch, int row) {
  if (starts == nullptr) return row;
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0; b0 < batch; b0 += 32) {
    const int b = b0 + lane;
    before += __popc(__ballot_sync(0xFFFFFFFFu, b < batch && starts[b + 1] <= row));
  }
  return row < *starts ? batch : before;
}

// The position of a sequence's first row; far beyond any capacity it stays so for all of its rows.
__device__ __forceinline__ int64_t kv4_position(const int64_t* positions, int b) { return min(positions[b], static_cast<int64_t>(1) << 62); }

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// n values from p, in 16- or 8-byte loads where `vec` says that the address allows it (n * sizeof(T) a power of two).
template <typename T, int n>
__device__ __forceinline__ void load_values(const T* p, bool vec, float (&v)[n]) {
  constexpr int bytes = n * static_cast<int>(sizeof(T));
  constexpr int step = bytes >= 16 ? 16 : bytes;
  if (vec) {
#pragma unroll
    for (int i = 0; i < bytes / step; ++i) {
      union {
        uint4 q;
        uint2 d;
        uint32_t w;
        T t[step / sizeof(T)];
      } u;
      const char* at = reinterpret_cast<const char*>(p) + i * step;
      if constexpr (step == 16) u.q = *reinterpret_cast<const uint4*>(at);
      else if constexpr (step == 8) u.d = *reinterpret_cast<const uint2*>(at);
      else u.w = *reinterpret_cast<const uint32_t*>(at);
#pragma unroll
      for (int j = 0; j < step / static_cast<int>(sizeof(T)); ++j) v[i * (step / static_cast<int>(sizeof(T))) + j] = to_f32<T>(u.t[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = to_f32<T>(p[i]);
  }
}

template <typename T, int n>
__device__ __forceinline__ void store_values(T* p, bool vec, const float (&v)[n]) {
  constexpr int bytes = n * static_cast<int>(sizeof(T));
  constexpr int step = bytes >= 16 ? 16 : bytes;
  if (vec) {
#pragma unroll
    for (int i = 0; i < bytes / step; ++i) {
      union {
        uint4 q;
        uint2 d;
        uint32_t w;
        T t[step / sizeof(T)];
      } u;
#pragma unroll
      for (int j = 0; j < step / static_cast<int>(sizeof(T)); ++j) u.t[j] = from_f32<T>(v[i * (step / static_cast<int>(sizeof(T))) + j]);
      char* at = reinterpret_cast<char*>(p) + i * step;
      if constexpr (step == 16) *reinterpret_cast<uint4*>(at) = u.q;
      else if constexpr (step == 8) *reinterpret_cast<uint2*>(at) = u.d;
      else *reinterpret_cast<uint32_t*>(at) = u.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) p[i] = from_f32<T>(v[i]);
  }
}

}  // namespace ivb
