// The 4-bit key/value cache: quantising rows as they are written, and reading them back (layout: ivb_kv4.cuh).
//
// Per row x of D values: m = fp16(min x), s = fp16((max x - m) / 15), u = round((x - m) / s) clipped to 0..15. The offset
// and the scale are what is stored, and the codes are taken against the stored ones, so that their rounding costs no more
// than the clip. fp16 for both: 4 bytes beside D / 2 bytes of codes, and a rounding of 2^-12 of the offset, far below the
// half step s / 2 that the codes leave (the row's range over 30) unless the row's offset is over 100 times its range.
#include <cuda_runtime.h>

#include "ivb_common.h"
#include "ivb_device.cuh"
#include "ivb_kv4.cuh"

namespace ivb {
namespace {

constexpr int kKv4Threads = 256;  // 8 warps, a row of one or four heads each

// The codes of n values by the real quotients (x - m) / s, value i at bit shift(i) of the result. The 32-bit products with the
// reciprocal are within 2^-18 of them; where that could change a rounding (2e-4 of all values) the quotients are taken in 64
// bits. Adding 1.5 2^23 rounds to an integer in the low bits; the constants' sum comes off at the end.
template <int n, typename Shift>
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[n], float m, float s, float rs, Shift shift) {
  constexpr float kMagic = 12582912.0f;
  uint32_t word = 0;
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const float t = fminf(fmaxf((x[i] - m) * rs, 0.0f), 15.0f), u = t + kMagic;
    off = fmaxf(off, fabsf(t - (u - kMagic)));
    word += (__float_as_uint(u) - 0x4b400000u) << shift(i);
  }
  if (off > 0.4999f) {
    word = 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const double u = rint((static_cast<double>(x[i]) - static_cast<double>(m)) / static_cast<double>(s));
      word |= static_cast<uint32_t>(fmin(fmax(u, 0.0), 15.0)) << shift(i);
    }
  }
  return word;
}

// fp16 of the real quotient d / 15, rounded to 32 bits and then to 16, with d = hi - m. The 32-bit product is within 2^-22 of it;
// where that could change the rounding to 16 bits (1 of 250 rows, and scales below fp16's normal range) it is taken in 64.
__device__ __forceinline__ __half kv4_scale(float hi, float m) {
  float wide = (hi - m) * (1.0f / 15.0f);
  const int to_border = static_cast<int>(__float_as_uint(wide) & 0x1fffu) - 0x1000;
  if (!(wide >= 6.2e-5f) || abs(to_border) < 16) wide = static_cast<float>((static_cast<double>(hi) - static_cast<double>(m)) / 15.0);
  return __float2half_rn(fminf(fmaxf(wide, 0.0f), 65504.0f));
}

// The row's sequence and position; false where there is nothing to do.
__device__ __forceinline__ bool kv4_place(const IvbKv4Cache& C, const int32_t* starts, const int64_t* positions, int row, uint32_t* error,
                                          int& b, int64_t& pos) {
  b = kv4_sequence(starts, C.batch, row);
  if (b >= C.batch) return false;
  pos = kv4_position(positions, b) + (starts == nullptr ? 0 : row - starts[b]);
  if (pos >= C.max_len && (threadIdx.x & 31) == 0 && error != nullptr) atomicCAS(error, 0u, static_cast<unsigned>(IVB_ECAPACITY));
  return pos >= 0 && pos < C.max_len;
}

// One warp per row and kHeads heads: lanes 0..15 the key rows, lanes 16..31 the value rows, D / 16 channels each. Four heads a
// warp share the look-up of the row and keep their loads in flight together; one is for calls too small to fill the GPU with
// the others (2048 rows of 32 heads x 128 in bf16: written in 25 us and read in 11 with four, 32 and 17 with one; in fp32 written in 23
// and read in 21. The writing takes 140 instructions a row, at 57 % of the issue slots; the reading 4 bytes a lane and load, each
// from a sector of its own).
template <int D, typename T, int kHeads>
__global__ void __launch_bounds__(kKv4Threads) kv4_append_kernel(IvbKv4Cache C, const T* k, const T* v, int64_t k_row, int64_t k_head,
                                                                 int64_t v_row, int64_t v_head, const int32_t* starts,
                                                                 const int64_t* positions, int rows, bool vec, uint32_t* error) {
  pdl_enter();
  constexpr int n = D / 16;
  const int row = blockIdx.x * (kKv4Threads / 32) + (threadIdx.x >> 5), h0 = blockIdx.y * kHeads;
  if (row >= rows) return;
  const int lane = threadIdx.x & 31, l = lane & 15;
  const bool value = lane >= 16;
  const T* src = (value ? v + row * v_row + h0 * v_head : k + row * k_row + h0 * k_head) + l * n;
  float x[kHeads][n];
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
    if (h0 + h < C.kv_heads) load_values<T, n>(src + h * (value ? v_head : k_head), vec, x[h]);
  int b;
  int64_t pos;
  if (!kv4_place(C, starts, positions, row, error, b, pos)) return;
  const int p = static_cast<int>(pos & 15);
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (h0 + h >= C.kv_heads) break;
    float lo = x[h][0], hi = x[h][0], zero = 0.0f;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      lo = fminf(lo, x[h][i]);
      hi = fmaxf(hi, x[h][i]);
      zero = fmaf(x[h][i], 0.0f, zero);  // NaN where a value is none or infinite
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d));
      hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
    }
    const unsigned all = __ballot_sync(0xFFFFFFFFu, zero == 0.0f);
    const bool row_finite = (value ? all >> 16 : all & 0xFFFFu) == 0xFFFFu;
    const __half mh = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
    const float m = __half2float(mh);
    const __half sh = kv4_scale(hi, m);
    const float s = __half2float(sh);
    const float rs = __fdividef(1.0f, s);  // within 2 ulp; of no use where s is zero
    uint32_t word = 0;
    if (s > 0.0f && row_finite)
      word = kv4_codes<n>(x[h], m, s, rs, [&](int i) {
        const int ch = (l * n + i) & 7;
        return 4 * (ch >> 1) + 16 * (ch & 1);
      });
    // the D / 16 lanes' parts of each word meet in the first of them
#pragma unroll
    for (int d = 1; d < 8 / n; d <<= 1) word |= __shfl_xor_sync(0xFFFFFFFFu, word, d);
    const int64_t tile = (static_cast<int64_t>(b) * C.kv_heads + h0 + h) * kv4_tiles(C.max_len) + (pos >> 4);
    uint32_t* words = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(C.data) + tile * kv4_tile_bytes(D));
    if (l % (8 / n) == 0) {
      const int i = l / (8 / n);
      words[value ? kv4_value_word<D>(p, i) : kv4_key_word<D>(p, i)] = word;
    }
    if (l == 0) {
      // a row that holds an infinity or a NaN reads back as NaN
      const uint32_t par = row_finite ? static_cast<uint32_t>(__half_as_ushort(sh)) | static_cast<uint32_t>(__half_as_ushort(mh)) << 16
                                      : 0x7fff7fffu;
      words[4 * D + 2 * p + (value ? 1 : 0)] = par;
    }
  }
}

template <int D, typename T, int kHeads>
__global__ void __launch_bounds__(kKv4Threads) kv4_read_kernel(IvbKv4Cache C, T* k, T* v, int64_t k_row, int64_t k_head, int64_t v_row,
                                                               int64_t v_head, const int32_t* starts, const int64_t* positions, int rows,
                                                               bool vec, uint32_t* error) {
  pdl_enter();
  constexpr int n = D / 16;
  const int row = blockIdx.x * (kKv4Threads / 32) + (threadIdx.x >> 5), h0 = blockIdx.y * kHeads;
  if (row >= rows) return;
  const int lane = threadIdx.x & 31, l = lane & 15;
  int b;
  int64_t pos;
  if (!kv4_place(C, starts, positions, row, error, b, pos)) return;
  const bool value = lane >= 16;
  const int p = static_cast<int>(pos & 15), i = l * n / 8;
  const int64_t step = kv4_tiles(C.max_len) * kv4_tile_bytes(D);
  const unsigned char* tile = static_cast<const unsigned char*>(C.data) + (static_cast<int64_t>(b) * C.kv_heads + h0) * step + (pos >> 4) * kv4_tile_bytes(D);
  uint32_t word[kHeads], par[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
    if (h0 + h < C.kv_heads) {
      const uint32_t* words = reinterpret_cast<const uint32_t*>(tile + h * step);
      word[h] = words[value ? kv4_value_word<D>(p, i) : kv4_key_word<D>(p, i)];
      par[h] = words[4 * D + 2 * p + (value ? 1 : 0)];
    }
  T* dst = (value ? v + row * v_row + h0 * v_head : k + row * k_row + h0 * k_head) + l * n;
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (h0 + h >= C.kv_heads) break;
    const float s = __half2float(__ushort_as_half(static_cast<uint16_t>(par[h]))), m = __half2float(__ushort_as_half(static_cast<uint16_t>(par[h] >> 16)));
    float x[n];
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const int ch = (l * n + j) & 7;
      x[j] = fmaf(s, static_cast<float>((word[h] >> (4 * (ch >> 1) + 16 * (ch & 1))) & 15u), m);
    }
    store_values<T, n>(dst + h * (value ? v_head : k_head), vec, x);
  }
}

// Whether rows at `p` with these strides (in values of `size` bytes) can be read in chunks of `chunk` bytes.
bool aligned(const void* p, int64_t row, int64_t head, int size, int chunk) {
  return reinterpret_cast<uintptr_t>(p) % chunk == 0 && row * size % chunk == 0 && head * size % chunk == 0;
}

}  // namespace

// Bytes of a cache with sizes above zero; 0 where 63 bits do not count them.
static uint64_t kv4_bytes(int32_t batch, int32_t kv_heads, int32_t head_dim, int32_t max_len) {
  const unsigned __int128 bytes = static_cast<unsigned __int128>(static_cast<uint64_t>(batch) * static_cast<uint64_t>(kv_heads)) *
                                  static_cast<uint64_t>(kv4_tiles(max_len) * kv4_tile_bytes(head_dim));
  return bytes >> 63 == 0 ? static_cast<uint64_t>(bytes) : 0;
}

int32_t check_kv4(const IvbKv4Cache* c, const char* who) {
  if (c == nullptr || c->data == nullptr) return fail(IVB_EINVAL, "%s: null cache", who);
  if (c->batch <= 0 || c->kv_heads <= 0 || c->max_len <= 0) return fail(IVB_EINVAL, "%s: batch %d, kv_heads %d, max_len %d", who, c->batch, c->kv_heads, c->max_len);
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return fail(IVB_EINVAL, "%s: head_dim %d (32, 64 or 128)", who, c->head_dim);
  if (kv4_bytes(c->batch, c->kv_heads, c->head_dim, c->max_len) == 0) return fail(IVB_EINVAL, "%s: a cache of over 2^63 bytes", who);
  if (reinterpret_cast<uintptr_t>(c->data) % 16 != 0) return fail(IVB_EINVAL, "%s: the cache must be 16-byte aligned", who);
  return IVB_OK;
}

int32_t check_kv4_rows(const IvbKv4Cache* c, const int32_t* starts, const int64_t* positions, int32_t rows, int32_t dtype, const char* who) {
  if (positions == nullptr || rows < 0) return fail(IVB_EINVAL, "%s: positions %p, rows %d", who, static_cast<const void*>(positions), rows);
  if (starts == nullptr && rows != c->batch) return fail(IVB_EINVAL, "%s: %d rows for %d sequences without starts", who, rows, c->batch);
  if (dtype != IVB_F32 && dtype != IVB_F16 && dtype != IVB_BF16) return fail(IVB_EINVAL, "%s: type %d", who, dtype);
  return IVB_OK;
}

namespace {

template <int D, typename T>
int32_t launch_rows(bool append, const IvbKv4Cache& c, void* k, void* v, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head,
                    const int32_t* starts, const int64_t* positions, int32_t rows, uint32_t* error, cudaStream_t stream) {
  constexpr int size = sizeof(T), chunk = D / 16 * size >= 16 ? 16 : D / 16 * size, kWarps = kKv4Threads / 32;
  const bool vec = aligned(k, k_row, k_head, size, chunk) && aligned(v, v_row, v_head, size, chunk);
  const int heads = static_cast<int64_t>(rows) * c.kv_heads > 148 * 64 ? 4 : 1;
  const int by = (c.kv_heads + heads - 1) / heads;
  if (by > 65535) return fail(IVB_EINVAL, "ivb_kv4: %d key/value heads", c.kv_heads);
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(rows) + kWarps - 1) / kWarps), static_cast<unsigned>(by));
  auto go = [&](auto append_kernel, auto read_kernel) {
    return append ? launch_pdl(append_kernel, grid, dim3(kKv4Threads), 0, stream, c, static_cast<const T*>(k), static_cast<const T*>(v), k_row,
                               k_head, v_row, v_head, starts, positions, static_cast<int>(rows), vec, error)
                  : launch_pdl(read_kernel, grid, dim3(kKv4Threads), 0, stream, c, static_cast<T*>(k), static_cast<T*>(v), k_row, k_head, v_row,
                               v_head, starts, positions, static_cast<int>(rows), vec, error);
  };
  if (heads == 4) IVB_CUDA(go(kv4_append_kernel<D, T, 4>, kv4_read_kernel<D, T, 4>));
  else IVB_CUDA(go(kv4_append_kernel<D, T, 1>, kv4_read_kernel<D, T, 1>));
  return IVB_OK;
}

template <typename T, typename... A>
int32_t launch_dim(int dim, A... a) {
  return dim == 32 ? launch_rows<32, T>(a...) : dim == 64 ? launch_rows<64, T>(a...) : launch_rows<128, T>(a...);
}

int32_t rows_call(bool append, const char* who, const IvbKv4Cache* c, void* k, void* v, int32_t dtype, int64_t k_row, int64_t k_head,
                  int64_t v_row, int64_t v_head, const int32_t* starts, const int64_t* positions, int32_t rows, uint32_t* error,
                  void* stream) {
  if (int32_t rc = check_kv4(c, who)) return rc;
  if (int32_t rc = check_kv4_rows(c, starts, positions, rows, dtype, who)) return rc;
  if (rows == 0) return IVB_OK;
  if (k == nullptr || v == nullptr) return fail(IVB_EINVAL, "%s: null keys or values", who);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == IVB_F32) return launch_dim<float>(c->head_dim, append, *c, k, v, k_row, k_head, v_row, v_head, starts, positions, rows, error, s);
  if (dtype == IVB_F16) return launch_dim<__half>(c->head_dim, append, *c, k, v, k_row, k_head, v_row, v_head, starts, positions, rows, error, s);
  return launch_dim<__nv_bfloat16>(c->head_dim, append, *c, k, v, k_row, k_head, v_row, v_head, starts, positions, rows, error, s);
}

}  // namespace
}  // namespace ivb

extern "C" {

uint64_t ivb_kv4_bytes(int32_t batch, int32_t kv_heads, int32_t head_dim, int32_t max_len) {
  if (batch <= 0 || kv_heads <= 0 || max_len <= 0 || (head_dim != 32 && head_dim != 64 && head_dim != 128)) return 0;
  return ivb::kv4_bytes(batch, kv_heads, head_dim, max_len);
}

int32_t ivb_kv4_append(const IvbKv4Cache* c, const void* k, const void* v, int32_t dtype, int64_t k_row, int64_t k_head, int64_t v_row,
                       int64_t v_head, const int32_t* starts, const int64_t* positions, int32_t rows, uint32_t* error, void* stream) {
  return ivb::rows_call(true, "ivb_kv4_append", c, const_cast<void*>(k), const_cast<void*>(v), dtype, k_row, k_head, v_row, v_head, starts,
                        positions, rows, error, stream);
}

int32_t ivb_kv4_read(const IvbKv4Cache* c, void* k, void* v, int32_t dtype, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head,
                     const int32_t* starts, const int64_t* positions, int32_t rows, uint32_t* error, void* stream) {
  return ivb::rows_call(false, "ivb_kv4_read", c, k, v, dtype, k_row, k_head, v_row, v_head, starts, positions, rows, error, stream);
}

}  // extern "C"
