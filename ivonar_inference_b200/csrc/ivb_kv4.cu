// The 4-bit key/value cache: quantising rows as they are written, and reading them back (layout: ivb_kv4.cuh).
//
// Per row x of D values: m = fp16(min x), s = fp16((max x - m) / 15), u = round((x - m) / s) clipped to 0..15. The offset
// and the scale are what is stored, and the codes are taken against the stored ones, so that their rounding costs no more
// than the clip. fp16 for both: 4 bytes beside D / 2 bytes of codes, and a rounding of 2^-12 of the offset, far below the
// half step s / 2 that the codes leave (the row's range over 30) unless the row's offset is over 100 times its range.
#include <cuda_runtime.h>

#include "ivb_common.h"
#include "ivb_kv4.cuh"

namespace ivb {
namespace {

constexpr int kKv4Threads = 256;  // 8 warps, one row of one head each

// The code of x by the real quotient (x - m) / s. The 32-bit product with the reciprocal is within 2^-18 of it; where that
// could change the rounding (2e-4 of all values) the quotient is taken in 64 bits.
__device__ __forceinline__ int kv4_code(float x, float m, float s, float rs) {
  const float t = (x - m) * rs;
  float u = rintf(t);
  if (fabsf(t - u) > 0.4999f) u = static_cast<float>(rint((static_cast<double>(x) - static_cast<double>(m)) / static_cast<double>(s)));
  return static_cast<int>(fminf(fmaxf(u, 0.0f), 15.0f));
}

// One warp per (row, head): lanes 0..15 the key row, lanes 16..31 the value row, D / 16 channels each.
template <int D, typename T>
__global__ void __launch_bounds__(kKv4Threads) kv4_append_kernel(IvbKv4Cache C, const T* k, const T* v, int64_t k_row, int64_t k_head,
                                                                 int64_t v_row, int64_t v_head, const int32_t* starts,
                                                                 const int64_t* positions, int rows, bool vec, uint32_t* error) {
  constexpr int n = D / 16;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kKv4Threads + threadIdx.x) >> 5;
  if (item >= static_cast<int64_t>(rows) * C.kv_heads) return;
  const int lane = threadIdx.x & 31, l = lane & 15;
  const int row = static_cast<int>(item / C.kv_heads), h = static_cast<int>(item - static_cast<int64_t>(row) * C.kv_heads);
  const int b = kv4_sequence(starts, C.batch, row);
  if (b >= C.batch) return;
  const int64_t pos = __ldg(positions + b) + (starts == nullptr ? 0 : row - __ldg(starts + b));
  if (pos < 0) return;
  if (pos >= C.max_len) {
    if (lane == 0 && error != nullptr) atomicCAS(error, 0u, static_cast<unsigned>(IVB_ECAPACITY));
    return;
  }
  const bool value = lane >= 16;
  const T* src = value ? v + row * v_row + h * v_head : k + row * k_row + h * k_head;
  float x[n];
  load_values<T, n>(src + l * n, vec, x);
  float lo = x[0], hi = x[0];
  bool finite = fabsf(x[0]) <= 3.402823466e38f;
#pragma unroll
  for (int i = 1; i < n; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    finite = finite && fabsf(x[i]) <= 3.402823466e38f;
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d));
    hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
  }
  const unsigned all = __ballot_sync(0xFFFFFFFFu, finite);
  const bool row_finite = (value ? all >> 16 : all & 0xFFFFu) == 0xFFFFu;
  const __half mh = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
  const float m = __half2float(mh);
  // to 32 bits first, then to 16
  const float wide = static_cast<float>((static_cast<double>(hi) - static_cast<double>(m)) / 15.0);
  const __half sh = __float2half_rn(fminf(fmaxf(wide, 0.0f), 65504.0f));
  const float s = __half2float(sh);
  const float rs = s > 0.0f ? 1.0f / s : 0.0f;
  uint32_t word = 0;
  if (s > 0.0f && row_finite) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int ch = (l * n + i) & 7;
      word |= static_cast<uint32_t>(kv4_code(x[i], m, s, rs)) << (4 * (ch >> 1) + 16 * (ch & 1));
    }
  }
  // the D / 16 lanes' parts of each word meet in the first of them
#pragma unroll
  for (int d = 1; d < 8 / n; d <<= 1) word |= __shfl_xor_sync(0xFFFFFFFFu, word, d);
  const int64_t tile = (static_cast<int64_t>(b) * C.kv_heads + h) * kv4_tiles(C.max_len) + (pos >> 4);
  const int p = static_cast<int>(pos & 15);
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

template <int D, typename T>
__global__ void __launch_bounds__(kKv4Threads) kv4_read_kernel(IvbKv4Cache C, T* k, T* v, int64_t k_row, int64_t k_head, int64_t v_row,
                                                               int64_t v_head, const int32_t* starts, const int64_t* positions, int rows,
                                                               bool vec, uint32_t* error) {
  constexpr int n = D / 16;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kKv4Threads + threadIdx.x) >> 5;
  if (item >= static_cast<int64_t>(rows) * C.kv_heads) return;
  const int lane = threadIdx.x & 31, l = lane & 15;
  const int row = static_cast<int>(item / C.kv_heads), h = static_cast<int>(item - static_cast<int64_t>(row) * C.kv_heads);
  const int b = kv4_sequence(starts, C.batch, row);
  if (b >= C.batch) return;
  const int64_t pos = __ldg(positions + b) + (starts == nullptr ? 0 : row - __ldg(starts + b));
  if (pos < 0) return;
  if (pos >= C.max_len) {
    if (lane == 0 && error != nullptr) atomicCAS(error, 0u, static_cast<unsigned>(IVB_ECAPACITY));
    return;
  }
  const bool value = lane >= 16;
  const int64_t tile = (static_cast<int64_t>(b) * C.kv_heads + h) * kv4_tiles(C.max_len) + (pos >> 4);
  const int p = static_cast<int>(pos & 15);
  const uint32_t* words = reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(C.data) + tile * kv4_tile_bytes(D));
  const int i = l * n / 8;
  const uint32_t word = words[value ? kv4_value_word<D>(p, i) : kv4_key_word<D>(p, i)];
  const uint32_t par = words[4 * D + 2 * p + (value ? 1 : 0)];
  const float s = __half2float(__ushort_as_half(static_cast<uint16_t>(par))), m = __half2float(__ushort_as_half(static_cast<uint16_t>(par >> 16)));
  float x[n];
#pragma unroll
  for (int j = 0; j < n; ++j) {
    const int ch = (l * n + j) & 7;
    x[j] = fmaf(s, static_cast<float>((word >> (4 * (ch >> 1) + 16 * (ch & 1))) & 15u), m);
  }
  T* dst = value ? v + row * v_row + h * v_head : k + row * k_row + h * k_head;
  store_values<T, n>(dst + l * n, vec, x);
}

// Whether rows at `p` with these strides (in values of `size` bytes) can be read in chunks of `chunk` bytes.
bool aligned(const void* p, int64_t row, int64_t head, int size, int chunk) {
  return reinterpret_cast<uintptr_t>(p) % chunk == 0 && row * size % chunk == 0 && head * size % chunk == 0;
}

}  // namespace

int32_t check_kv4(const IvbKv4Cache* c, const char* who) {
  if (c == nullptr || c->data == nullptr) return fail(IVB_EINVAL, "%s: null cache", who);
  if (c->batch <= 0 || c->kv_heads <= 0 || c->max_len <= 0) return fail(IVB_EINVAL, "%s: batch %d, kv_heads %d, max_len %d", who, c->batch, c->kv_heads, c->max_len);
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return fail(IVB_EINVAL, "%s: head_dim %d (32, 64 or 128)", who, c->head_dim);
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
  const int64_t items = static_cast<int64_t>(rows) * c.kv_heads, blocks = (items + kKv4Threads / 32 - 1) / (kKv4Threads / 32);
  if (blocks > 0x7fffffff) return fail(IVB_EINVAL, "ivb_kv4: %lld rows of heads in one call", static_cast<long long>(items));
  constexpr int size = sizeof(T), chunk = D / 16 * size >= 16 ? 16 : D / 16 * size;
  const bool vec = aligned(k, k_row, k_head, size, chunk) && aligned(v, v_row, v_head, size, chunk);
  if (append)
    kv4_append_kernel<D, T><<<static_cast<unsigned>(blocks), kKv4Threads, 0, stream>>>(
        c, static_cast<const T*>(k), static_cast<const T*>(v), k_row, k_head, v_row, v_head, starts, positions, rows, vec, error);
  else
    kv4_read_kernel<D, T><<<static_cast<unsigned>(blocks), kKv4Threads, 0, stream>>>(
        c, static_cast<T*>(k), static_cast<T*>(v), k_row, k_head, v_row, v_head, starts, positions, rows, vec, error);
  IVB_CUDA(cudaGetLastError());
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
  return static_cast<uint64_t>(batch) * kv_heads * ivb::kv4_tiles(max_len) * ivb::kv4_tile_bytes(head_dim);
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
