// What the kernels of the attention over the 4-bit cache share.
//
// With k_j = m_j + s_j u_j (codes u_j) the score is  a q.k_j = a s_j (q.u_j) + a m_j sum(q), and with v_j = m'_j + s'_j u'_j the
// output is  sum_j p_j v_j = sum_j (p_j s'_j) u'_j + sum_j p_j m'_j : both products run on the codes themselves, and scales and
// offsets are applied to scores and weights in 32 bits, one multiply-add per score. The operands are the codes less their
// middle, exact in fp16, with m + 8 s in the offsets' place: the tensor cores cut their sums towards zero, which adds up over a
// long axis where the terms have one sign (with u itself 3e-6 of the output at 2000 positions). Values take u - 8 at even
// positions and u - 7 at odd ones, since the 0.5 that is left of either mean is what all of a long history has in
// common (with u - 8 throughout 1.3e-5 at 100000 positions, where the values average out to little).
// fp32 queries and weights are split in two fp16 (x = hi + lo, 22 bits). fp16 and bf16 queries have no more bits than fp16 after their
// row's power of two (what lies 2^27 and more below the row's largest is cut at that), and their weights are rounded once to fp16, by
// 2^-11 of each at most (the sums that divide them are not), but for the few rows' tiles of four, which hold the remainder anyway. With it
// the prompts' fp16 calls would be as near as fp32 ones before the output's rounding, but take a second product: a causal prompt of
// 2048 x 16 heads x 64 53 us in place of 49, a chunk of 2048 under a window of 4096 x 32 heads x 128 267 in place of 230, a mixed call 74
// in place of 67; for few rows it would take the columns of other rows. Who needs the bits hands in fp32 queries.
#pragma once

#include "ivb_common.h"
#include "ivb_device.cuh"
#include "ivb_kv4.cuh"

namespace ivb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr unsigned long long kKv4WaitNs = 2000000000ull, kKv4ProbeNs = 1000000ull;

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
  int few;             // sequences with more items (tokens x group) are prompts
  bool q_vec, o_vec;   // rows begin on 16 bytes
  // The few rows' kernel runs beside the prompts', which is the grid before it, and does not wait before it reads. It is launched
  // once every CTA of that one has triggered or ended, which each does only after its own wait for the grids before both: these
  // had ended then, with their writes in device memory, and a fence at its start keeps it from what an SM's cache may have from before.
  // The two write different rows. The first CTA waits at its end instead, so that who waits for this grid has waited for both.
  bool beside_prompts;
  unsigned long long wait_ns;  // the longest wait within the prompts' kernel
  bool withhold;               // issue no products, so that the waits for them run out (ivb_probe_kv4_timeout)
};

// Launch attributes: beside the end of the grid before, and clusters of C CTAs.
inline int kv4_attributes(int C, cudaLaunchAttribute (&attr)[2]) {
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  return C > 1 ? 2 : 1;
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

// Queries become fp16 by a power of two that brings the largest finite value of their row to 2^13 (a row's values below 2^-87 stay small).
__device__ __forceinline__ float finite_size(float x) {
  const float m = fabsf(x);
  return m <= 3.402823466e38f ? m : 0.0f;
}
__device__ __forceinline__ int query_power(float largest) {
  const int up = 13 - (static_cast<int>(__float_as_uint(largest) >> 23) - 127);
  return largest == 0.0f ? 0 : min(max(up, -114), 100);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// (a & b) | c in one instruction (two constants keep the compiler from it).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(a), "r"(b), "r"(c));
  return y;
}

// Two nibbles of a word as fp16 values u - lo (low half) and u - hi: the bits under 0x6400 give 1024 + u and 1024 + 16 u, the rest
// is exact. The bare bits, fp16 subnormals u 2^-24, would save this instruction, but the tensor cores align products by
// the operands' exponent fields and cut 7 to 10 bits more of a subnormal's: 5e-5 of the output, measured.
struct CodeMiddle {
  __half2 low, high;  // to add to 1024 + u, and to 64 + u
};
__device__ __forceinline__ CodeMiddle code_middle(float lo, float hi) {
  return {__floats2half2_rn(-1024.0f - lo, -1024.0f - hi), __floats2half2_rn(-64.0f - lo, -64.0f - hi)};
}
__device__ __forceinline__ uint32_t codes_low(uint32_t w, CodeMiddle m) {
  const uint32_t x = and_or(w, 0x000f000fu, 0x64006400u);
  const __half2 y = __hadd2(*reinterpret_cast<const __half2*>(&x), m.low);
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t codes_high(uint32_t w, CodeMiddle m) {
  const uint32_t x = and_or(w, 0x00f000f0u, 0x64006400u);
  const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&x), __floats2half2_rn(0.0625f, 0.0625f), m.high);
  return *reinterpret_cast<const uint32_t*>(&y);
}

// What the softmax needs of one position: x = S key_scale + sum(q) key_offset + bias (S and sum(q) of the queries as the operands hold
// them, a power of two apart, which score_unit undoes together with the scale, or 1 where the rows have units of their own), with bias the exponent of the value
// scale, so that the running reference is the maximum of weight times value scale and neither overflows fp16, whatever the
// scales; the weight is then 2^(x - ref) = p 2^bias, its product with the mantissa the A operand of the value product, and
// p = weight * unbias enters the sum. A position whose value scale or offset is no number has a score that is none, and
// value terms of zero: it makes the rows that see it NaN, and a masked one's weight of zero stays zero whatever it holds.
struct PositionTerms {
  float key_scale, key_offset, bias, mantissa;  // mantissa of the value scale, times weight_unit
  float unbias, value_offset;                   // 2^-bias, value offset times 2^-bias (offsets are of the middle)
};

__device__ __forceinline__ PositionTerms position_terms(uint2 par, float score_unit, float weight_unit, int position) {
  const float2 key = unpack_f16(par.x), value = unpack_f16(par.y);
  PositionTerms t;
  t.key_scale = key.x * score_unit;
  t.key_offset = fmaf(8.0f, key.x, key.y) * score_unit;
  const bool number = (par.y & 0x7c00u) != 0x7c00u && (par.y & 0x7c000000u) != 0x7c000000u;
  const uint32_t e = max(__float_as_uint(value.x) & 0x7f800000u, 0x33800000u);  // 2^-24 is the least scale above zero
  t.bias = number ? static_cast<float>(static_cast<int>(e >> 23) - 127) : __uint_as_float(0x7fffffffu);
  t.unbias = number ? __uint_as_float(0x7f000000u - e) : 0.0f;
  t.mantissa = number ? value.x * t.unbias * weight_unit : 0.0f;
  t.value_offset = number ? fmaf(position & 1 ? 7.0f : 8.0f, value.x, value.y) * t.unbias : 0.0f;
  return t;
}

// Prompts: every sequence of the call with more than `few` items (tokens x query heads of a group).
int32_t launch_kv4_prompts(const Kv4Attention& A, int32_t dtype, int few, cudaStream_t stream);

}  // namespace ivb
