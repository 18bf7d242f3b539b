// Causal attention over the 4-bit key/value cache, with a sliding window and visible first tokens (sinks).
//
// With k_j = m_j + s_j u_j (codes u_j) the score is  a q.k_j = a s_j (q.u_j) + a m_j sum(q), and with v_j = m'_j + s'_j u'_j the
// output is  sum_j p_j v_j = sum_j (p_j s'_j) u'_j + sum_j p_j m'_j : both products run on the codes themselves, and scales and
// offsets are applied to scores and weights in 32 bits, one multiply-add per score. The operands are u - 8, exact in
// fp16, with m + 8 s in the offsets' place: the tensor cores cut their sums towards zero, which adds up over a long axis
// where all terms have one sign (3e-6 of the output at 2000 positions with u, 5e-7 with u - 8). fp32 queries and weights are split in two fp16 (x = hi + lo, 22 bits); fp16 and bf16
// queries are exact in fp16 after a common power of two, and weights are rounded once to fp16.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "ivb_common.h"
#include "ivb_kv4.cuh"

namespace ivb {

int32_t check_kv4(const IvbKv4Cache* c, const char* who);
int32_t check_kv4_rows(const IvbKv4Cache* c, const int32_t* starts, const int64_t* positions, int32_t rows, int32_t dtype, const char* who);

namespace {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.4426950408889634f;

struct Kv4Attention {
  IvbKv4Cache cache;
  const void* q;
  void* out;
  int64_t q_row, q_head, o_row, o_head;
  const int32_t* starts;
  const int64_t* positions;
  uint32_t* error;
  float scale;
  int heads, group;  // query heads, query heads per key/value head
  int rows, window, sinks;
  bool q_vec, o_vec;
};

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
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two nibbles of a word as fp16 values u - 8: the bits under 0x6400 give 1024 + u and 1024 + 16 u, the rest is exact. The
// bare bits, fp16 subnormals u 2^-24, would save this instruction, but the tensor cores align products by the operands'
// exponent fields and cut 7 to 10 bits more of a subnormal's: 5e-5 of the output, measured.
__device__ __forceinline__ uint32_t codes_low(uint32_t w) {
  const uint32_t x = (w & 0x000f000fu) | 0x64006400u;
  const __half2 y = __hadd2(*reinterpret_cast<const __half2*>(&x), __floats2half2_rn(-1032.0f, -1032.0f));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t codes_high(uint32_t w) {
  const uint32_t x = (w & 0x00f000f0u) | 0x64006400u;
  const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&x), __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.0f, -72.0f));
  return *reinterpret_cast<const uint32_t*>(&y);
}

// What the softmax needs of one position: x = S key_scale + sum(q) key_offset + bias, with bias the exponent of the value
// scale, so that the running reference is the maximum of weight times value scale and neither overflows fp16, whatever the
// scales; the weight is then 2^(x - ref) = p 2^bias, its product with the mantissa the A operand of the value product, and
// p = weight * unbias enters the sum.
struct PositionTerms {
  float key_scale, key_offset, bias, mantissa;  // mantissa of the value scale, times 2^14
  float unbias, value_offset;                   // 2^-bias, value offset times 2^-bias (offsets are of u - 8)
};

__device__ __forceinline__ PositionTerms position_terms(uint2 par, float score_unit, float offset_unit) {
  const float2 key = unpack_f16(par.x), value = unpack_f16(par.y);
  PositionTerms t;
  t.key_scale = key.x * score_unit;
  t.key_offset = fmaf(8.0f, key.x, key.y) * offset_unit;
  const uint32_t bits = __float_as_uint(value.x) & 0x7f800000u;
  const uint32_t e = bits == 0x7f800000u ? 0x3f800000u : max(bits, 0x33800000u);  // 2^-24 is the least scale above zero
  t.bias = static_cast<float>(static_cast<int>(e >> 23) - 127);
  t.unbias = __uint_as_float(0x7f000000u - e);
  t.mantissa = value.x * t.unbias * 16384.0f;
  t.value_offset = fmaf(8.0f, value.x, value.y) * t.unbias;
  return t;
}

// ---- few rows: one token per sequence, a few drafted ones, or any number in tiles of 16 (8 for fp32) rows -----------------
// One cluster of C CTAs per (sequence, key/value head, tile of rows); row i of a sequence's head group is token i / group,
// query head i % group of the group. The 32-position groups of the cache that a row of the tile sees are dealt out to the
// cluster's warps in turn; each warp streams its own through a ring of cp.async stages, holds its scores and its online
// softmax in registers (scores in the C fragment's layout are weights in the A fragment's), and the partial (reference,
// sum, output) join in shared memory, then over the cluster's.
template <int D, typename T>
struct RowsGeometry {
  static constexpr bool split = std::is_same<T, float>::value;
  static constexpr int rows = split ? 8 : 16;
  static constexpr int warps = 8;
  static constexpr int stages = D == 128 ? 2 : 4;
  static constexpr int group_bytes = kKv4Group * (D + 8);

  static constexpr int ring_bytes = warps * stages * group_bytes;
  static constexpr int comb_floats = rows * D + 3 * rows;
  static constexpr int smem = ring_bytes + warps * kKv4Group * 24 + comb_floats * 4 + warps * rows * 3 * 4;
};

template <int D, typename T>
__global__ void __launch_bounds__(256, D == 128 ? 2 : 2) kv4_rows_kernel(Kv4Attention A, int tiles_per_sequence) {
  using G = RowsGeometry<D, T>;
  constexpr int R = G::rows, W = G::warps, kSteps = D / 16, kTile = kv4_tile_bytes(D), kSets = G::split ? 1 : 2;
  constexpr int kOut = D / 8;  // column tiles of the output
  extern __shared__ __align__(128) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  unsigned char* const ring = smem + warp * G::stages * G::group_bytes;
  float4* const terms4 = reinterpret_cast<float4*>(smem + G::ring_bytes) + warp * kKv4Group;
  float2* const terms2 = reinterpret_cast<float2*>(smem + G::ring_bytes + W * kKv4Group * 16) + warp * kKv4Group;
  float* const comb = reinterpret_cast<float*>(smem + G::ring_bytes + W * kKv4Group * 24);  // [R][D], then ref, sum, offset [R]
  float* const stats = comb + G::comb_floats;                                              // [W][R][3]

  // which rows
  const int64_t cluster_id = blockIdx.x / C;
  const int tile = static_cast<int>(cluster_id % tiles_per_sequence);
  const int64_t sh = cluster_id / tiles_per_sequence;
  const int kvh = static_cast<int>(sh % A.cache.kv_heads), b = static_cast<int>(sh / A.cache.kv_heads);
  int row0 = b, count = 1;
  if (A.starts != nullptr) {
    row0 = max(0, __ldg(A.starts + b));
    count = min(A.rows, __ldg(A.starts + b + 1)) - row0;
  }
  const int64_t items = static_cast<int64_t>(max(count, 0)) * A.group;
  const int64_t i0 = static_cast<int64_t>(tile) * R;
  if (i0 >= items) return;  // the whole cluster
  const int live = static_cast<int>(min(static_cast<int64_t>(R), items - i0));
  const int64_t base = __ldg(A.positions + b);
  const int64_t first = base + i0 / A.group, last = base + (i0 + live - 1) / A.group;
  const int max_len = A.cache.max_len;
  // position of this lane's rows (-1: sees nothing)
  int at[kSets], sum_row[kSets];
#pragma unroll
  for (int s = 0; s < kSets; ++s) {
    const int64_t p = base + (i0 + r + 8 * s) / A.group;
    at[s] = r + 8 * s < live && p >= 0 && p < max_len ? static_cast<int>(p) : -1;
    sum_row[s] = r + 8 * s;
  }
  if (last >= max_len && threadIdx.x == 0 && rank == 0 && A.error != nullptr) atomicCAS(A.error, 0u, static_cast<unsigned>(IVB_ECAPACITY));
  // the groups of 32 positions that some row sees: the sinks' below the window, then the window's
  const int high = static_cast<int>(min(last, static_cast<int64_t>(max_len) - 1));  // negative: none
  const int lowest = static_cast<int>(min(max(first, static_cast<int64_t>(0)), static_cast<int64_t>(max_len)));
  const int low = A.window > 0 ? max(0, lowest - A.window + 1) : 0;
  const int window_group = low / kKv4Group;
  const int sink_groups = A.window > 0 ? min((min(A.sinks, low) + kKv4Group - 1) / kKv4Group, window_group) : 0;
  const int groups = high < 0 ? 0 : sink_groups + high / kKv4Group - window_group + 1;
  const int lanes_in = C * W, mine = rank * W + warp;
  const int steps = groups > mine ? (groups - mine + lanes_in - 1) / lanes_in : 0;

  const unsigned char* const codes = static_cast<const unsigned char*>(A.cache.data) +
                                     (static_cast<int64_t>(b) * A.cache.kv_heads + kvh) * kv4_tiles(max_len) * kTile;
  auto group_of = [&](int step) {
    const int i = mine + step * lanes_in;
    return i < sink_groups ? i : window_group + i - sink_groups;
  };
  auto issue = [&](int step) {
    if (step < steps) {
      const unsigned char* src = codes + static_cast<int64_t>(group_of(step)) * G::group_bytes;
      unsigned char* dst = ring + step % G::stages * G::group_bytes;
#pragma unroll
      for (int o = 0; o < G::group_bytes; o += 512)
        if (o + lane * 16 < G::group_bytes) cp_async16(dst + o + lane * 16, src + o + lane * 16);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < G::stages - 1; ++s) issue(s);

  // queries as A fragments, scaled by a power of two that brings the largest to 2^13: channels D/4 c + 4 s + {0, 1} and
  // {2, 3}
  float amax = 0.0f, sum_q[kSets];
  float qv[kSets][D / 4];
#pragma unroll
  for (int s = 0; s < kSets; ++s) {
    sum_q[s] = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 4; ++j) qv[s][j] = 0.0f;
    const int64_t i = i0 + sum_row[s];
    if (sum_row[s] < live) {
      const int64_t t = i / A.group;
      const int h = kvh * A.group + static_cast<int>(i - t * A.group);
      load_values<T, D / 4>(static_cast<const T*>(A.q) + (row0 + t) * A.q_row + h * A.q_head + D / 4 * c, A.q_vec, qv[s]);
    }
#pragma unroll
    for (int j = 0; j < D / 4; ++j) {
      sum_q[s] += qv[s][j];
      const float m = fabsf(qv[s][j]);
      if (m <= 3.402823466e38f) amax = fmaxf(amax, m);
    }
    sum_q[s] += __shfl_xor_sync(0xFFFFFFFFu, sum_q[s], 1);
    sum_q[s] += __shfl_xor_sync(0xFFFFFFFFu, sum_q[s], 2);
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
  int up = 13 - (static_cast<int>(__float_as_uint(amax) >> 23) - 127);
  up = amax == 0.0f ? 0 : min(max(up, -100), 100);
  const float q_unit = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
  const float score_unit = __uint_as_float(static_cast<uint32_t>(127 - up) << 23) * A.scale * kLog2e;
  const float offset_unit = A.scale * kLog2e;
  uint32_t qf[kSteps][4];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x0 = qv[0][4 * s + 2 * e] * q_unit, x1 = qv[0][4 * s + 2 * e + 1] * q_unit;
      qf[s][2 * e] = pack_f16(x0, x1);
      if constexpr (G::split) {
        const float2 hi = unpack_f16(qf[s][2 * e]);
        qf[s][2 * e + 1] = pack_f16(x0 - hi.x, x1 - hi.y);
      } else {
        qf[s][2 * e + 1] = pack_f16(qv[kSets - 1][4 * s + 2 * e] * q_unit, qv[kSets - 1][4 * s + 2 * e + 1] * q_unit);
      }
    }
  }

  float acc[kOut][4];
#pragma unroll
  for (int i = 0; i < kOut; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
  float ref[kSets], sum[kSets], off[kSets];
#pragma unroll
  for (int s = 0; s < kSets; ++s) {
    ref[s] = -INFINITY;
    sum[s] = off[s] = 0.0f;
  }

  for (int step = 0; step < steps; ++step) {
    cp_async_wait<G::stages - 2>();
    __syncwarp();
    const unsigned char* const stage = ring + step % G::stages * G::group_bytes;
    const int p0 = group_of(step) * kKv4Group;
    {
      const uint2 par = *reinterpret_cast<const uint2*>(stage + (lane >> 4) * kTile + 16 * D + (lane & 15) * 8);
      const PositionTerms t = position_terms(par, score_unit, offset_unit);
      terms4[lane] = make_float4(t.key_scale, t.key_offset, t.bias, t.mantissa);
      terms2[lane] = make_float2(t.unbias, t.value_offset);
    }
    __syncwarp();
    // scores of 8 positions per lane and set: x[set][4 tile + i] is position p0 + 16 tile + 4 c + i
    float x[kSets][8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float s2[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) s2[h][0] = s2[h][1] = s2[h][2] = s2[h][3] = 0.0f;
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
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t v = s & 1 ? w[h][s >> 1] >> 8 : w[h][s >> 1];
          mma_f16(s2[h], qf[s][0], qf[s][1], qf[s][2], qf[s][3], codes_low(v), codes_high(v));
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 pt = terms4[16 * t + 4 * c + i];
        const int h = i >> 1, e = i & 1;
        if constexpr (G::split) {
          x[0][4 * t + i] = fmaf(s2[h][e] + s2[h][e + 2], pt.x, fmaf(sum_q[0], pt.y, pt.z));
        } else {
          x[0][4 * t + i] = fmaf(s2[h][e], pt.x, fmaf(sum_q[0], pt.y, pt.z));
          x[kSets - 1][4 * t + i] = fmaf(s2[h][e + 2], pt.x, fmaf(sum_q[kSets - 1], pt.y, pt.z));
        }
      }
    }
    // a group that every row sees whole needs no masks
    const bool whole = first >= p0 + kKv4Group - 1 && last < max_len && (A.window <= 0 || p0 > last - A.window || p0 + kKv4Group <= A.sinks);
    if (!whole) {
#pragma unroll
      for (int s = 0; s < kSets; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int p = p0 + 16 * (i >> 2) + 4 * c + (i & 3);
          const bool seen = p <= at[s] && (A.window <= 0 || p > at[s] - A.window || p < A.sinks);
          if (!seen) x[s][i] = -INFINITY;
        }
    }
    bool raise = false;
    float next[kSets];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      float m = fmaxf(fmaxf(fmaxf(x[s][0], x[s][1]), fmaxf(x[s][2], x[s][3])), fmaxf(fmaxf(x[s][4], x[s][5]), fmaxf(x[s][6], x[s][7])));
      m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
      next[s] = fmaxf(ref[s], m);
      raise |= next[s] > ref[s];
    }
    if (__any_sync(0xFFFFFFFFu, raise)) {
      float corr[kSets];
#pragma unroll
      for (int s = 0; s < kSets; ++s) {
        corr[s] = next[s] > ref[s] ? ex2(ref[s] - next[s]) : 1.0f;
        ref[s] = next[s];
        sum[s] *= corr[s];
        off[s] *= corr[s];
      }
#pragma unroll
      for (int i = 0; i < kOut; ++i) {
        acc[i][0] *= corr[0];
        acc[i][1] *= corr[0];
        acc[i][2] *= corr[kSets - 1];
        acc[i][3] *= corr[kSets - 1];
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float wgt[kSets][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float mantissa = terms4[16 * t + 4 * c + i].w;
        const float2 pt = terms2[16 * t + 4 * c + i];
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
          const float xi = x[s][4 * t + i];
          const float pw = ex2(xi - ref[s]);
          if (whole) {
            sum[s] = fmaf(pw, pt.x, sum[s]);
            off[s] = fmaf(pw, pt.y, off[s]);
            wgt[s][i] = pw * mantissa;
          } else {  // a masked position's terms may hold anything
            const bool seen = xi != -INFINITY;
            sum[s] = seen ? fmaf(pw, pt.x, sum[s]) : sum[s];
            off[s] = seen ? fmaf(pw, pt.y, off[s]) : off[s];
            wgt[s][i] = seen ? pw * mantissa : 0.0f;
          }
        }
      }
      uint32_t a[4];
      a[0] = pack_f16(wgt[0][0], wgt[0][1]);
      a[2] = pack_f16(wgt[0][2], wgt[0][3]);
      if constexpr (G::split) {
        const float2 h0 = unpack_f16(a[0]), h1 = unpack_f16(a[2]);
        a[1] = pack_f16(wgt[0][0] - h0.x, wgt[0][1] - h0.y);
        a[3] = pack_f16(wgt[0][2] - h1.x, wgt[0][3] - h1.y);
      } else {
        a[1] = pack_f16(wgt[kSets - 1][0], wgt[kSets - 1][1]);
        a[3] = pack_f16(wgt[kSets - 1][2], wgt[kSets - 1][3]);
      }
      const uint4* vw = reinterpret_cast<const uint4*>(stage + t * kTile + 8 * D);
      constexpr int planes = D == 128 ? 2 : 1;
#pragma unroll
      for (int h = 0; h < planes; ++h) {
        if constexpr (D == 32) {
          const uint4 v = vw[4 * (r >> 1) + c];
          const unsigned sel = r & 1 ? 0x7632u : 0x5410u;
          const uint32_t x01 = __byte_perm(v.x, v.y, sel), x23 = __byte_perm(v.z, v.w, sel);
          mma_f16(acc[0], a[0], a[1], a[2], a[3], codes_low(x01), codes_low(x23));
          mma_f16(acc[1], a[0], a[1], a[2], a[3], codes_high(x01), codes_high(x23));
          mma_f16(acc[2], a[0], a[1], a[2], a[3], codes_low(x01 >> 8), codes_low(x23 >> 8));
          mma_f16(acc[3], a[0], a[1], a[2], a[3], codes_high(x01 >> 8), codes_high(x23 >> 8));
        } else {
          const uint4 v = vw[32 * h + lane];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const unsigned sel = e ? 0x7632u : 0x5410u;
            const uint32_t x01 = __byte_perm(v.x, v.y, sel), x23 = __byte_perm(v.z, v.w, sel);
            float(&o)[4] = acc[8 * h + 4 * e];
            mma_f16(o, a[0], a[1], a[2], a[3], codes_low(x01), codes_low(x23));
            mma_f16(acc[8 * h + 4 * e + 1], a[0], a[1], a[2], a[3], codes_high(x01), codes_high(x23));
            mma_f16(acc[8 * h + 4 * e + 2], a[0], a[1], a[2], a[3], codes_low(x01 >> 8), codes_low(x23 >> 8));
            mma_f16(acc[8 * h + 4 * e + 3], a[0], a[1], a[2], a[3], codes_high(x01 >> 8), codes_high(x23 >> 8));
          }
        }
      }
    }
    __syncwarp();
    issue(step + G::stages - 1);
  }
  cp_async_wait<0>();
  __syncwarp();

  // this warp's part: reference, sum and offset sum per row, and its output over the ring it no longer needs
  float* const part = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int s = 0; s < kSets; ++s) {
    sum[s] += __shfl_xor_sync(0xFFFFFFFFu, sum[s], 1);
    sum[s] += __shfl_xor_sync(0xFFFFFFFFu, sum[s], 2);
    off[s] += __shfl_xor_sync(0xFFFFFFFFu, off[s], 1);
    off[s] += __shfl_xor_sync(0xFFFFFFFFu, off[s], 2);
    if (c == 0) {
      float* st = stats + (warp * R + r + 8 * s) * 3;
      st[0] = ref[s];
      st[1] = sum[s];
      st[2] = off[s];
    }
    if (r + 8 * s < live) {
#pragma unroll
      for (int i = 0; i < kOut; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // column 2 c + e of column tile i
          const int j = i & 3;
          const int ch = D == 32 ? 8 * c + 2 * j + e : 64 * (i >> 3) + 8 * (2 * c + e) + 2 * j + ((i >> 2) & 1);
          const float v = G::split ? acc[i][e] + acc[i][e + 2] : acc[i][2 * s + e];
          part[(r + 8 * s) * D + ch] = v * 0.00006103515625f;  // the weights' 2^14
        }
    }
  }
  __syncthreads();
  float* const cref = comb + R * D;
  for (int i = threadIdx.x; i < live * D; i += 32 * W) {
    const int row = i / D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, stats[(w * R + row) * 3]);
    float o = 0.0f, l = 0.0f, m = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* st = stats + (w * R + row) * 3;
      if (st[1] != 0.0f) {  // zero: the warp saw nothing for this row
        const float f = ex2(st[0] - top);
        o = fmaf(reinterpret_cast<const float*>(smem + w * G::stages * G::group_bytes)[i], f, o);
        l = fmaf(st[1], f, l);
        m = fmaf(st[2], f, m);
      }
    }
    comb[i] = o;
    if (i - row * D == 0) {
      cref[row] = top;
      cref[R + row] = l;
      cref[2 * R + row] = m;
    }
  }
  if (C > 1) cluster.sync();
  else __syncthreads();
  // the cluster's parts: every CTA writes its share of the rows' values
  for (int i = rank * 32 * W + threadIdx.x; i < live * D; i += C * 32 * W) {
    const int row = i / D;
    float top = -INFINITY;
    for (int k = 0; k < C; ++k) top = fmaxf(top, cluster.map_shared_rank(comb, k)[R * D + row]);
    float o = 0.0f, l = 0.0f;
    for (int k = 0; k < C; ++k) {
      const float* other = cluster.map_shared_rank(comb, k);
      const float part_sum = other[R * D + R + row];
      if (part_sum != 0.0f) {
        const float f = ex2(other[R * D + row] - top);
        o = fmaf(other[i] + other[R * D + 2 * R + row], f, o);
        l = fmaf(part_sum, f, l);
      }
    }
    const int64_t item = i0 + row, t = item / A.group;
    const int h = kvh * A.group + static_cast<int>(item - t * A.group);
    static_cast<T*>(A.out)[(row0 + t) * A.o_row + h * A.o_head + (i - row * D)] = from_f32<T>(l == 0.0f ? 0.0f : o / l);
  }
  if (C > 1) cluster.sync();  // no CTA leaves while another reads its shared memory
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

template <int D, typename T>
int32_t launch_rows_attention(const Kv4Attention& A, cudaStream_t stream) {
  using G = RowsGeometry<D, T>;
  static std::atomic<uint64_t> done{0};
  if (int32_t rc = allow_smem(kv4_rows_kernel<D, T>, G::smem, done)) return rc;
  const int64_t most = static_cast<int64_t>(A.starts == nullptr ? 1 : A.rows) * A.group;
  const int64_t tiles = (most + G::rows - 1) / G::rows;
  const int64_t base = tiles * A.cache.kv_heads * A.cache.batch;
  int C = 1;
  while (C < 8 && base * C * 2 <= 2 * 148 && A.cache.max_len > C * G::warps * kKv4Group) C *= 2;
  if (base * C > 0x7fffffff) return fail(IVB_EINVAL, "ivb_kv4_attention: %lld tiles of rows in one call", static_cast<long long>(base));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(base * C));
  cfg.blockDim = dim3(32 * G::warps);
  cfg.dynamicSmemBytes = G::smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  IVB_CUDA(cudaLaunchKernelEx(&cfg, kv4_rows_kernel<D, T>, A, static_cast<int>(tiles)));
  return IVB_OK;
}

template <typename T>
int32_t launch_attention(Kv4Attention& A, cudaStream_t stream) {
  const int size = static_cast<int>(sizeof(T)), chunk = std::min(16, A.cache.head_dim / 4 * size);
  A.q_vec = reinterpret_cast<uintptr_t>(A.q) % chunk == 0 && A.q_row * size % chunk == 0 && A.q_head * size % chunk == 0;
  switch (A.cache.head_dim) {
    case 32: return launch_rows_attention<32, T>(A, stream);
    case 64: return launch_rows_attention<64, T>(A, stream);
    default: return launch_rows_attention<128, T>(A, stream);
  }
}

}  // namespace
}  // namespace ivb

extern "C" int32_t ivb_kv4_attention(const IvbKv4Cache* c, const void* q, int32_t dtype, int64_t q_row, int64_t q_head, int32_t heads,
                                     const int32_t* starts, const int64_t* positions, int32_t rows, float scale, int32_t window,
                                     int32_t sinks, void* out, int64_t o_row, int64_t o_head, uint32_t* error, void* stream) {
  using namespace ivb;
  if (int32_t rc = check_kv4(c, "ivb_kv4_attention")) return rc;
  if (int32_t rc = check_kv4_rows(c, starts, positions, rows, dtype, "ivb_kv4_attention")) return rc;
  if (heads <= 0 || heads % c->kv_heads != 0) return fail(IVB_EINVAL, "ivb_kv4_attention: %d query heads over %d key/value heads", heads, c->kv_heads);
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == IVB_F32) return launch_attention<float>(A, s);
  if (dtype == IVB_F16) return launch_attention<__half>(A, s);
  return launch_attention<__nv_bfloat16>(A, s);
}
