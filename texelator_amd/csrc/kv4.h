// The paged 4-bit KV cache (gfx950): layout and conversions shared by the kernels that write, read and attend to it.
//
// A pool holds pages of `page` positions (a power of two, 16 to 1024). A page holds for each KV head its keys,
// then its values; a row (one key or value of dim elements, dim 64 or 128) is stored as dim/32 groups of 32
// elements: packed E2M1 codes, dim/2 bytes (even element in the low nibble), and one E8M0 scale a group. The
// codes of a head's rows come first, [page][dim/2], then their scales, [page][dim/32]: every 16 bytes of codes
// are one group, aligned, and codes and scales of consecutive rows are contiguous.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tx {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Kv4Pool {
  uint8_t *pages;
  int64_t num_pages;
  int page_shift;  // log2 of the positions a page holds
  int kv_heads;
  const int *table;      // [sequences][max_pages] page ids, rows table_stride apart
  int64_t table_stride;
  int max_pages;
  const int *lengths;  // [sequences] positions in use
  int sequences;
};

struct Kv4Attention {
  Kv4Pool pool;
  const uint16_t *q;  // query h of sequence s at q + s * q_sequence + h * q_head (elements)
  int64_t q_sequence, q_head;
  uint16_t *out;
  int64_t out_sequence, out_head;
  int group;  // query heads per KV head
  // exp2(sl2 * q . k) is exp(scale * q . k): sl2 is above zero, the scale's sign is put into the queries' bits
  // ((bits & q_and) ^ q_xor), which are cleared for a scale of zero.
  float sl2;
  uint32_t q_and, q_xor;
  float *pieces;        // results of heads that several workgroups share
  int64_t piece_bytes;  // bytes of them
  int piece_floats;     // of each: per query its output [dim], then max and sum of all queries; whole vectors of four
  int workgroups;
  bool whole;  // a workgroup for each head: no pieces
};

// Bytes of one head's keys (or values) in a page.
__host__ __device__ inline int64_t kv4_half_bytes(int page_shift, int dim) { return ((int64_t)dim * 17 / 32) << page_shift; }

// A sequence's length, kept within what its table row can hold.
__device__ __forceinline__ int kv4_length(const Kv4Pool &pool, int sequence) {
  const int64_t room = (int64_t)pool.max_pages << pool.page_shift;
  return (int)min((int64_t)max(pool.lengths[sequence], 0), room);
}

// Two elements of a packed word (byte SEL) times 2^(e - 127), where the exponent field of `scale` is e: exact in
// bf16; in fp16 rounded to nearest where it is subnormal. v_cvt_scalef32_pk_*_fp4 reads the exponent field alone
// (sign and mantissa are ignored, 0 means 2^-127, and 255 gives NaN whatever the codes: the E8M0 rule), checked
// for all of these.
template <bool F16, int SEL>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t word, float scale) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, SEL));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, SEL));
}
template <bool F16>
__device__ __forceinline__ u32x4 kv4_octet(uint32_t word, float scale) {
  return u32x4{kv4_pair<F16, 0>(word, scale), kv4_pair<F16, 1>(word, scale), kv4_pair<F16, 2>(word, scale),
               kv4_pair<F16, 3>(word, scale)};
}

}  // namespace tx
