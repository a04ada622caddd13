// Causal attention of several packed prompts (gfx950): the queries of all sequences one behind the other, their keys and
// values likewise, grouped heads, head_dim 64 or 128, bf16 or fp16.
//
// No reference counterpart: the reference runs attention as the Hugging Face module's sdpa call on one prompt.
//
//   out[i][h] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale * q_i . k_j - max_i),  j <= i + keys - queries
// within a sequence: its last query sees its last key (keys of earlier turns come first); a query that sees none gets zeros.
//
// A workgroup takes 32 * QW queries of one head of one sequence with QW * KW waves; it finds its sequence from cu_q
// by itself, so the grid needs the totals only. Wave (kw, qw) owns 32 queries and every KW-th block of KB keys (KW > 1
// shortens the chain of dependent key blocks where there are few workgroups; the KW shares meet in LDS at the end).
//   * scores are computed transposed, S^T = K q^T (v_mfma_f32_32x32x16: A = 32 keys, B = the wave's 32 queries, held in
//     registers): a lane holds 16 scores of ONE query, so the row maximum is in-lane but for one lane swap, the rescale
//     factor is a scalar of the lane, and the probabilities, rounded to 16 bits in place, are the B operand of
//     O^T = V^T P^T: none of them passes through LDS;
//   * keys and values reach LDS by direct buffer loads one block ahead, as they lie in memory; the descriptors end at
//     the sequence's last row, rows past it read as zeros. 16-byte chunks of a row are permuted by its number so
//     that operand reads hit distinct banks; the values' transpose is done by the read (ds_read_b64_tr_b16).
// Online softmax in fp32 with exp2; the sum runs over the probabilities as rounded. In fp16 they are held times 2^15, so
// that small ones keep their bits.
#include <math.h>

#include <type_traits>

#include "elementwise.h"
#include "kernels.h"
#include "ragged.h"

namespace tx {

namespace {

constexpr int kXcds = 8;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <bool F16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b, float &sum) {
  if constexpr (F16) {
    const f16x2 p = {(_Float16)a, (_Float16)b};
    sum = __builtin_amdgcn_fdot2(p, f16x2{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
    return __builtin_bit_cast(uint32_t, p);
  } else {
    const bf16x2 p = {(__bf16)a, (__bf16)b};
    sum = __builtin_amdgcn_fdot2_f32_bf16(p, bf16x2{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
    return __builtin_bit_cast(uint32_t, p);
  }
}

template <bool F16>
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  else return (uint32_t)to_bf(a) | (uint32_t)to_bf(b) << 16;
}

// The larger (or the sum) of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// First row and rows of a sequence, kept within the array whatever cu holds.
struct Rows {
  int begin, count;
};
__device__ __forceinline__ Rows rows_of(const int *cu, int sequence, int total) {
  const int begin = min(max(cu[sequence], 0), total);
  return {begin, min(max(cu[sequence + 1], begin), total) - begin};
}

// Two waves per SIMD, but for <1, 4, 32>, whose four waves have a CU's LDS to themselves.
template <bool F16, int DIM, int QW, int KW, int KB>
__global__ __launch_bounds__(64 * QW * KW, QW * KW * KB == 128 ? 1 : 2) __attribute__((amdgpu_num_vgpr(256))) void packed_attention_kernel(
    PackedAttention a) {
  constexpr int kRow = DIM * 2;                 // bytes of a key or value
  constexpr int kTile = KB * kRow;              // bytes of a key (or value) block
  constexpr int kLoads = kTile / 1024;          // 1 KiB direct loads per block and array
  constexpr int kPer = kLoads / QW;             // of them this wave issues
  constexpr int kChunks = DIM / 8;              // 16-byte chunks of a row = lanes that bring it
  constexpr int kLoadRows = 64 / kChunks;       // rows of a load
  constexpr int kSubs = KB / 32;
  constexpr int kSteps = DIM / 16, kOut = DIM / 32;
  constexpr float kLift = F16 ? 15.f : 0.f;
  static_assert(kPer * QW == kLoads, "loads divide among the waves");
  // Two buffers, separate LDS objects (the compiler then knows that reads of one do not wait for the
  // direct loads that fill the other): per key group its key block, then its value block.
  __shared__ __attribute__((aligned(1024))) char buf0[KW * 2 * kTile];
  __shared__ __attribute__((aligned(1024))) char buf1[KW * 2 * kTile];
  __shared__ float stats[KW][QW][2][KW > 1 ? 64 : 1];  // (m, l) of every wave, for the merge

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qw = wave % QW, kw = wave / QW;
  const int n = lane & 31, h = lane >> 5;
  // Heads fastest; where the head count allows, an XCD (workgroups arrive round-robin) gets neighbouring heads, which
  // share keys.
  const int hx = blockIdx.x % a.heads;
  const int head = a.heads % kXcds == 0 ? (hx % kXcds) * (a.heads / kXcds) + hx / kXcds : hx;
  auto tiles_of = [&](int s) { return (rows_of(a.cu_q, s, a.total_q).count + 32 * QW - 1) / (32 * QW); };
  const int wanted = blockIdx.x / a.heads;
  const RaggedPlace place = ragged_place(a.sequences, tiles_of, [&](int) { return wanted; });
  if (wanted >= place.total) return;
  const int sequence = place.sequence;
  const Rows qs = rows_of(a.cu_q, sequence, a.total_q), ks = rows_of(a.cu_k, sequence, a.total_k);
  const int queries = __builtin_amdgcn_readfirstlane(qs.count), keys = __builtin_amdgcn_readfirstlane(ks.count);
  // The heaviest tiles of a sequence (the last) first.
  const int tile = (queries + 32 * QW - 1) / (32 * QW) - 1 - place.local;
  const int shift = keys - queries;            // query i sees the keys up to i + shift
  const int q0 = (tile * QW + qw) * 32;        // this wave's first query

  // q as MFMA B operands: column n = query q0 + n (clamped into the sequence), dimensions 16 st + 8 h ...
  const float sl2 = a.scale * 1.44269504088896340736f;  // scores in log2 units
  u32x4 qb[kSteps];
  {
    const uint16_t *qr = a.q + (qs.begin + min(q0 + n, queries - 1)) * a.q_token + head * a.q_head;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) qb[st] = *reinterpret_cast<const u32x4 *>(qr + 16 * st + 8 * h);
  }

  const int kv = head / a.group;
  const char *kg = reinterpret_cast<const char *>(a.k + ks.begin * a.k_token + kv * a.k_head);
  const char *vg = reinterpret_cast<const char *>(a.v + ks.begin * a.v_token + kv * a.v_head);
  const uint32_t k_bytes = (uint32_t)a.k_token * 2, v_bytes = (uint32_t)a.v_token * 2;  // between rows
  // Load i of a block brings rows kLoadRows * i .., lane l landing in chunk l % kChunks of the load's row l / kChunks,
  // which holds the row's chunk (l % kChunks) ^ turn(row): the row's number mod 16 for keys (mod 16 of its
  // pair for rows of 128 bytes, two of which make a pass over the banks), 4 times it mod 4 (mod 2 of its pair) for values.
  const uint32_t load_row = lane / kChunks;
  const uint32_t k_chunk = 16u * (uint32_t)((lane % kChunks) ^ (lane >> 4));  // but for the load's number
  const uint32_t v_chunk = 16u * (uint32_t)((lane % kChunks) ^ (DIM == 128 ? 4 * (lane >> 4) : 4 * ((lane >> 4) & 1)));
  auto stage = [&](char *buf, int kb) __attribute__((always_inline)) {
    const int first = kb * KB, rows = min(KB, keys - first);
    char *kd = buf + kw * 2 * kTile, *vd = kd + kTile;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char *>(kg) + (int64_t)first * k_bytes, (short)0, rows > 0 ? (rows - 1) * k_bytes + kRow : 0, 0x00020000);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char *>(vg) + (int64_t)first * v_bytes, (short)0, rows > 0 ? (rows - 1) * v_bytes + kRow : 0, 0x00020000);
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = qw + QW * u;
      const uint32_t row = i * kLoadRows + load_row, turn = 64u * (uint32_t)(DIM == 128 ? i & 3 : i & 1);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (__attribute__((address_space(3))) void *)(kd + i * 1024), 16,
                                               row * k_bytes + (k_chunk ^ turn), 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (__attribute__((address_space(3))) void *)(vd + i * 1024), 16,
                                               row * v_bytes + v_chunk, 0, 0, 0);
    }
  };

  float m = -INFINITY, l = 0.f;  // running maximum (log2 units) and this lane's share of the sum, query q0 + n
  f32x16 o[kOut];                // o[t][r] = O[query q0 + n][dimension 32 t + 8 (r / 4) + 4 h + r % 4]
#pragma unroll
  for (int t = 0; t < kOut; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;

  // Byte offsets of this lane's operands in a tile: of key row n, dimensions 16 st + 8 h (chunk 2 st + h) at
  // k_at ^ 32 st; and, for the transposing reads, of key 4 h + (lane % 16) / 4, dimensions
  // 32 t + 16 ((lane / 16) % 2) + 4 (lane % 4) at v_at ^ 64 t.
  const uint32_t x4 = (lane >> 2) & 3;
  const uint32_t k_at = (uint32_t)n * kRow + 16u * (uint32_t)(h ^ (DIM == 128 ? n & 15 : (n >> 1) & 7));
  const uint32_t v_at = (4u * h + x4) * kRow + 32u * ((lane >> 4) & 1) + 8u * (lane & 3) + 64u * (DIM == 128 ? x4 : x4 >> 1);
  const int limit = min(q0 + n, queries - 1) + shift;  // the last key this lane's query sees

  // NS sub-blocks of 32 keys at once (their score chains are independent); MASK: some keys are past some query's limit.
  auto block = [&](const char *buf, int k0, auto ns_c, auto mask_c) __attribute__((always_inline)) {
    constexpr int NS = decltype(ns_c)::value;
    constexpr bool MASK = decltype(mask_c)::value;
    const char *kt = buf + kw * 2 * kTile, *vt = kt + kTile;
    f32x16 sc[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[s][r] = 0.f;
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const u32x4 b = *reinterpret_cast<const u32x4 *>(kt + 32 * s * kRow + (k_at ^ (32u * st)));
        sc[s] = mfma32<F16>(b, qb[st], sc[s]);
      }
    // sc[s][r] = score of key 32 s + 8 (r / 4) + 4 h + r % 4 of the block and query q0 + n
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sc[s][r] *= sl2;
        if (MASK) sc[s][r] = k0 + 32 * s + 8 * (r >> 2) + 4 * h + (r & 3) > limit ? -INFINITY : sc[s][r];
      }
    float mx = fmaxf(sc[0][0], sc[0][1]);
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int r = s == 0 ? 2 : 0; r < 16; r += 2) mx = fmaxf(fmaxf(mx, sc[s][r]), sc[s][r + 1]);
    // The running maximum is each query's own: its output does not depend on which others share the wave. It is
    // finite from the first block on in which the query sees a key (in unmasked blocks all do).
    const float mnew = fmaxf(m, halves_max(mx));
    if (__builtin_amdgcn_ballot_w64(mnew > m) != 0) {
      const float alpha = !MASK || mnew > m ? __builtin_amdgcn_exp2f(m - mnew) : 1.f;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < kOut; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] *= alpha;
      m = mnew;
    }
    const float base = MASK && m == -INFINITY ? 0.f : m - kLift;
    uint32_t pb[NS][8];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int r = 0; r < 16; r += 2)
        pb[s][r / 2] = pack2<F16>(__builtin_amdgcn_exp2f(sc[s][r] - base), __builtin_amdgcn_exp2f(sc[s][r + 1] - base), l);
    // O^T += V^T P^T, sixteen keys at a time: slots 0-3 of half h are keys 4 h .. + 3, slots 4-7 the keys 8 on
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4 b = {pb[s][4 * j], pb[s][4 * j + 1], pb[s][4 * j + 2], pb[s][4 * j + 3]};
#pragma unroll
        for (int t = 0; t < kOut; ++t) {
          const char *at = vt + (32 * s + 16 * j) * kRow + (v_at ^ (64u * t));
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(at + 8 * kRow));
          const u32x2 lw = __builtin_bit_cast(u32x2, lo), hw = __builtin_bit_cast(u32x2, hi);
          o[t] = mfma32<F16>(u32x4{lw[0], lw[1], hw[0], hw[1]}, b, o[t]);
        }
      }
  };
  // A key block against this wave's queries: nothing to do for a wave without queries or whose last query ends before it.
  const int reach = q0 < queries ? min(q0 + 31, queries - 1) + shift : -1;
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  auto visit = [&](const char *buf, int kb) __attribute__((always_inline)) {
    const int k0 = kb * KB;
    if (k0 > reach) return;
    if constexpr (kSubs == 2) {
      if (k0 + 63 <= q0 + shift) block(buf, k0, Two{}, std::false_type{});
      else if (k0 + 32 <= reach) block(buf, k0, Two{}, std::true_type{});
      else block(buf, k0, One{}, std::true_type{});
    } else {
      if (k0 + 31 <= q0 + shift) block(buf, k0, One{}, std::false_type{});
      else block(buf, k0, One{}, std::true_type{});
    }
  };

  // Blocks of this key group: kw, kw + KW, ... up to the workgroup's last key; every wave runs every
  // turn (the barriers are workgroup-wide). A turn's loads were issued a turn before; the barrier
  // that ends their wait also says that the other buffer is no longer read.
  const int last_key = min((tile + 1) * QW * 32, queries) - 1 + shift;
  const int last = last_key < 0 ? -1 : last_key / KB;
  const int turns = last < 0 ? 0 : last / KW + 1;
  auto turn = [&](int it, char *cur, char *next) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int kb = it * KW + kw;
    if (kb + KW <= last) stage(next, kb + KW);
    if (kb <= last) visit(cur, kb);
  };
  if (kw <= last) stage(buf0, kw);
  int it = 0;
  for (; it + 2 <= turns; it += 2) {
    turn(it, buf0, buf1);
    turn(it + 1, buf1, buf0);
  }
  if (it < turns) turn(it, buf0, buf1);

  l = halves_sum(l);
  if constexpr (KW > 1) {
    // The groups' (m, l) meet in LDS; with M = max m, every group scales its O by exp2(m - M), and group
    // t % KW sums the output tile t of all. A group whose blocks a query does not see has m = -inf, l = 0, O = 0
    // for it and weighs nothing (or NaN, where its scores were).
    constexpr int kHalf = kOut / 2;  // output tiles that go through a buffer
    static_assert(KW * QW * kHalf * 4096 <= KW * 2 * kTile, "half the output tiles of every wave fit a buffer");
    stats[kw][qw][0][lane] = m;
    stats[kw][qw][1][lane] = l;
    __syncthreads();  // every tile read is done, too
    float mm = m, total = 0.f;
#pragma unroll
    for (int g = 0; g < KW; ++g) mm = fmaxf(mm, stats[g][qw][0][lane]);
    auto weight = [&](float mine) { return mine == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mine - mm); };
#pragma unroll
    for (int g = 0; g < KW; ++g) total += stats[g][qw][1][lane] * weight(stats[g][qw][0][lane]);
    l = total;
    const float alpha = weight(m);
    auto at = [&](int g, int t) {
      return reinterpret_cast<float *>(t < kHalf ? buf0 : buf1) + ((g * QW + qw) * kHalf + t % kHalf) * 1024 + lane;
    };
#pragma unroll
    for (int t = 0; t < kOut; ++t) {
      float *mine = at(kw, t);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        o[t][r] *= alpha;
        if (t % KW != kw) mine[r * 64] = o[t][r];
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kOut; ++t) {
      if (t % KW != kw) continue;
#pragma unroll
      for (int g = 0; g < KW; ++g) {
        if (g == kw) continue;
        const float *theirs = at(g, t);
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] += theirs[r * 64];
      }
    }
  }
  const int query = q0 + n;
  if (query >= queries) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint16_t *dst = a.out + (qs.begin + query) * a.out_token + head * a.out_head + 4 * h;
#pragma unroll
  for (int t = 0; t < kOut; ++t) {
    if (KW > 1 && t % KW != kw) continue;
#pragma unroll
    for (int rq = 0; rq < 4; ++rq)
      *reinterpret_cast<u32x2 *>(dst + 32 * t + 8 * rq) = u32x2{half2_bits<F16>(o[t][4 * rq] * inv, o[t][4 * rq + 1] * inv),
                                                                half2_bits<F16>(o[t][4 * rq + 2] * inv, o[t][4 * rq + 3] * inv)};
  }
}

template <bool F16, int DIM>
hipError_t launch_typed(const PackedAttention &a, int cus, hipStream_t stream) {
  auto launch = [&](auto kernel, int queries, int waves) {
    const int64_t tiles = a.total_q / queries + a.sequences;  // at least what the sequences' partial tiles make it
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles * a.heads)), dim3(64 * waves), 0, stream, a);
  };
  const int64_t tokens = a.total_q;
  const int64_t tiles128 = (tokens + 127) / 128 * a.heads, tiles64 = (tokens + 63) / 64 * a.heads,
                tiles32 = (tokens + 31) / 32 * a.heads;
  if (4 * tiles128 >= 9 * (int64_t)cus) launch(packed_attention_kernel<F16, DIM, 4, 1, 64>, 128, 4);
  else if (5 * tiles64 >= 8 * (int64_t)cus) launch(packed_attention_kernel<F16, DIM, 4, 2, 64>, 128, 8);
  else if (tiles32 <= cus) launch(packed_attention_kernel<F16, DIM, 1, 4, 32>, 32, 4);
  else launch(packed_attention_kernel<F16, DIM, 2, 4, 32>, 64, 8);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_packed_attention(const PackedAttention &a, bool f16, int dim, int cus, hipStream_t stream) {
  if (f16) return dim == 128 ? launch_typed<true, 128>(a, cus, stream) : launch_typed<true, 64>(a, cus, stream);
  return dim == 128 ? launch_typed<false, 128>(a, cus, stream) : launch_typed<false, 64>(a, cus, stream);
}

}  // namespace tx
