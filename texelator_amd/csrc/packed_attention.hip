// Causal attention of several packed prompts (gfx950): the queries of all sequences one behind the other, their keys and
// values likewise, grouped heads, head_dim 64 or 128, bf16 or fp16.
//
// No reference counterpart: the reference runs attention as the Hugging Face module's sdpa call on one prompt.
//
//   out[i][h] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale * q_i . k_j - max_i),  j <= i + keys - queries
// within a sequence: its last query sees its last key (keys of earlier turns come first); a query that sees none gets zeros.
//
// A workgroup takes 32 * QW queries of one head of one sequence with QW * KW waves; it finds its place from cu_q by
// itself, so the grid needs the totals only. Wave (kw, qw) owns 32 queries and every KW-th block of KB keys (KW > 1
// shortens the chain of dependent key blocks where there are few workgroups; the KW shares meet in LDS at the end).
//   * scores are computed transposed, S^T = K q^T (v_mfma_f32_32x32x16: A = 32 keys, B = the wave's 32 queries, held in
//     registers): a lane holds 16 scores of ONE query, so the row maximum is in-lane but for one lane swap, the rescale
//     factor is a scalar of the lane, and the probabilities, rounded to 16 bits in place, are the B operand of
//     O^T = V^T P^T: none of them passes through LDS;
//   * the next 32 keys' scores are computed while these 32 keys' exponentials are, woven by hand: a wave that ran its
//     products and its exponentials one after the other kept the matrix cores 44% busy, woven 54%;
//   * a query's running maximum follows its scores only where they pass it by 2^4: rescaling the outputs had been a third of
//     the vector instructions, since some of a wave's queries almost always finds a new maximum;
//   * keys and values reach LDS by direct buffer loads one block ahead, as they lie in memory; the descriptors end at
//     the sequence's last row, rows past it read as zeros. 16-byte chunks of a row are permuted by its number so
//     that operand reads hit distinct banks; the values' transpose is done by the read (ds_read_b64_tr_b16).
// Online softmax in fp32 with exp2; the sum runs over the probabilities as rounded. In fp16 they are held times 2^11, so
// that small ones keep their bits and large ones (2^4 more while a maximum lags) stay below fp16's largest; in bf16 times a power
// of two below 1 / (2^4 keys), so that sums of the type's largest values stay finite (in turn values below 2^-110, at 8190 keys, lose
// bits to fp32's smallest; held unscaled, sums of values above 2^111 overflowed).
//
// Bound: power. At 8190 tokens and 40/8 heads 1.22 M cycles a SIMD, 54% of them with products, at 1.83 GHz, 650 to 669 us by card (1030
// to 1060 TFLOP/s; a plain 16384^3 product of the library reaches 1370); on zeros as many cycles at 2.4 GHz, 494 us. At 64 dimensions
// 0.73 M cycles, 45% of them with products, 68% with vector instructions, 372 us, on zeros 296. Two waves a SIMD: vector
// instructions take 2.6 cycles each there against 5 of a wave alone. 64 queries a wave (half the LDS reads per product, one wave a
// SIMD) took 1.73 M cycles, 718 us.
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

// This wave's loads (to LDS too) and LDS accesses are done, then every wave's. Builtins: the compiler has to know
// that nothing is under way any more, or it waits again before the reads that follow.
__device__ __forceinline__ void drain_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// First row and rows of a sequence, kept within the array whatever cu holds.
struct Rows {
  int begin, count;
};
__device__ __forceinline__ Rows rows_of(const int *cu, int sequence, int total) {
  const int begin = min(max(cu[sequence], 0), total);
  return {begin, min(max(cu[sequence + 1], begin), total) - begin};
}

// Bits of a count: it is below 2^bits.
__device__ __forceinline__ float bits_of(int count) { return (float)(32 - __builtin_clz(count | 1)); }

// Whether values of the rows first .. last hold an infinity or a NaN: asked by a whole wave.
template <bool F16, int DIM>
__device__ __forceinline__ bool unseen_odd_value(const PackedAttention &a, const char *vg, int first, int last, int lane) {
  constexpr uint32_t kExponent = F16 ? 0x7C00 : 0x7F80;
  bool odd = false;
#pragma unroll 1
  for (int row = first; row <= last; ++row) {
    const uint16_t *v = reinterpret_cast<const uint16_t *>(vg) + row * a.v_token + lane;
    for (int e = 0; e < DIM; e += 64) odd |= (v[e] & kExponent) == kExponent;
  }
  return __builtin_amdgcn_ballot_w64(odd) != 0;
}

// One query's attention over the keys 0 .. limit and no other, by one wave, in fp32 throughout: 64 scores at a time, a key a
// lane, then the values one row after the other. Writes the output tiles t % KW == kw. Slow (about 1500 cycles for 64 keys): for
// the few queries that lie before a value that is not finite.
template <bool F16, int DIM, int KW>
__device__ __forceinline__ void seen_keys_alone(const PackedAttention &a, const uint16_t *q, const char *kg, const char *vg, int limit,
                                                uint16_t *out, int kw, int lane) {
  const uint16_t *k = reinterpret_cast<const uint16_t *>(kg), *v = reinterpret_cast<const uint16_t *>(vg);
  auto score = [&](int key) {
    if (key > limit) return -INFINITY;
    float s = 0.f;
#pragma unroll 1
    for (int d = 0; d < DIM; d += 8) {
      u32x4 x = *reinterpret_cast<const u32x4 *>(q + d);
      const u32x4 y = *reinterpret_cast<const u32x4 *>(k + key * a.k_token + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = (x[j] & a.q_and) ^ a.q_xor;
        s = __builtin_fmaf(half_bits_to_float<F16>((uint16_t)x[j]), half_bits_to_float<F16>((uint16_t)y[j]), s);
        s = __builtin_fmaf(half_bits_to_float<F16>((uint16_t)(x[j] >> 16)), half_bits_to_float<F16>((uint16_t)(y[j] >> 16)), s);
      }
    }
    return s;
  };
  float m = -INFINITY;
#pragma unroll 1
  for (int k0 = 0; k0 <= limit; k0 += 64) m = fmaxf(m, score(k0 + lane));
#pragma unroll
  for (int w = 1; w < 64; w *= 2) m = fmaxf(m, __shfl_xor(m, w));
  const float base = m == -INFINITY ? 0.f : -bits_of(limit + 1) - m * a.sl2;  // the sum of the largest values stays finite
  float l = 0.f, o[DIM / 64] = {};
#pragma unroll 1
  for (int k0 = 0; k0 <= limit; k0 += 64) {
    const float mine = __builtin_amdgcn_exp2f(__builtin_fmaf(score(k0 + lane), a.sl2, base));
    const int many = min(64, limit + 1 - k0);
#pragma unroll 1
    for (int j = 0; j < many; ++j) {
      const float p = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), j));
      l += p;
#pragma unroll
      for (int e = 0; e < DIM / 64; ++e) o[e] = __builtin_fmaf(p, half_bits_to_float<F16>(v[(k0 + j) * a.v_token + 64 * e + lane]), o[e]);
    }
  }
  const float inv = limit < 0 ? 0.f : 1.0f / l;
#pragma unroll
  for (int e = 0; e < DIM / 64; ++e)
    if (KW == 1 || (2 * e + (lane >> 5)) % KW == kw) out[64 * e + lane] = (uint16_t)half2_bits<F16>(o[e] * inv, 0.f);
}

// Two waves per SIMD at least, but for <1, 4, 32>, whose four waves have a CU's LDS to themselves (at 128 dimensions).
template <bool F16, int DIM, int QW, int KW, int KB>
__global__ __launch_bounds__(64 * QW * KW, QW == 1 ? 1 : 2) void packed_attention_kernel(PackedAttention a) {
  constexpr int kRow = DIM * 2;                 // bytes of a key or value
  constexpr int kTile = KB * kRow;              // bytes of a key group's keys (or values) of a turn
  constexpr int kSub = 32 * kRow;               // of 32 of them
  constexpr int kSubs = KB / 32;
  constexpr int kChunks = DIM / 8;              // 16-byte chunks of a row = lanes that bring it
  constexpr int kLoadRows = 64 / kChunks;       // rows of a 1 KiB load
  constexpr int kPer = kSub / 1024 / QW;        // loads of this wave for 32 rows
  constexpr int kSteps = DIM / 16, kOut = DIM / 32;
  static_assert(kPer * QW * 1024 == kSub, "loads divide among the waves");
  // Two buffers of each, separate LDS objects: the compiler then knows that reads of one do not wait for the direct
  // loads that fill the other.
  __shared__ __attribute__((aligned(1024))) char k_even[KW * kTile];
  __shared__ __attribute__((aligned(1024))) char k_odd[KW * kTile];
  __shared__ __attribute__((aligned(1024))) char v_even[KW * kTile];
  __shared__ __attribute__((aligned(1024))) char v_odd[KW * kTile];
  __shared__ float stats[KW][QW][2][KW > 1 ? 64 : 1];  // (m, l) of every wave, for the merge

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qw = wave % QW, kw = wave / QW;
  const int n = lane & 31, h = lane >> 5;
  // The heaviest tiles of all sequences first. Where two workgroups a CU are all there are, the second of a CU come in
  // reverse order, so that the heaviest meets the lightest (by eights: the order of the XCDs, which workgroups reach
  // round-robin, stays): 4096 tokens of 16/2 heads 95.1 -> 89.8 us; with more than that 2048 tokens of 40/8 58.4 -> 61.5.
  // Heads fastest; where the head count allows, an XCD gets neighbouring heads, which share keys.
  constexpr int kQueries = 32 * QW;
  int hx = 0;
  // Up to 64 sequences, lane s keeps the rows of sequence s: they are loaded once.
  const bool few = a.sequences <= 64;
  Rows lane_q = {0, 0}, lane_k = {0, 0};
  if (few && lane < a.sequences) lane_q = rows_of(a.cu_q, lane, a.total_q), lane_k = rows_of(a.cu_k, lane, a.total_k);
  auto queries_of = [&](int s) { return few ? lane_q.count : rows_of(a.cu_q, s, a.total_q).count; };
  auto tiles_of = [&](int count) { return (count + kQueries - 1) / kQueries; };
  auto before_of = [&](int) { return (lane_k.count - lane_q.count) / kQueries; };
  const RaggedPlace place = ragged_heaviest(a.sequences, queries_of, tiles_of, before_of, [&](int total) {
    int index = blockIdx.x;
    const int64_t all = (int64_t)total * a.heads;
    const int first = a.cus & ~7, end = (int)min((int64_t)2 * first, all) & ~7;
    if (index >= first && index < end && all <= 2 * first) index = first + (end - 8 - (index & ~7)) + (index & 7);
    hx = index % a.heads;
    return index / a.heads;
  });
  if (blockIdx.x >= (int64_t)place.total * a.heads) return;
  const int head = a.heads % kXcds == 0 ? (hx % kXcds) * (a.heads / kXcds) + hx / kXcds : hx;
  const int tile = place.local;
  const int sequence = place.sequence;
  auto rows_at = [&](Rows of_lane, const int *cu, int total) {
    const Rows r = few ? Rows{__builtin_amdgcn_readlane(of_lane.begin, sequence), __builtin_amdgcn_readlane(of_lane.count, sequence)}
                       : rows_of(cu, sequence, total);
    return Rows{__builtin_amdgcn_readfirstlane(r.begin), __builtin_amdgcn_readfirstlane(r.count)};
  };
  const Rows qs = rows_at(lane_q, a.cu_q, a.total_q), ks = rows_at(lane_k, a.cu_k, a.total_k);
  const int queries = qs.count, keys = ks.count;
  const int shift = keys - queries;      // query i sees the keys up to i + shift
  const float lift = F16 ? 15.f - kPackedLag : -kPackedLag - 1.f - bits_of(keys);  // probabilities are held times 2^lift
  const int q0 = tile * kQueries + qw * 32;  // this wave's first query

  // q as MFMA B operands: column n = query q0 + n (clamped into the sequence), dimensions 16 st + 8 h ...
  u32x4 qb[kSteps];
  {
    const uint16_t *qr = a.q + (qs.begin + min(q0 + n, queries - 1)) * a.q_token + head * a.q_head;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      qb[st] = *reinterpret_cast<const u32x4 *>(qr + 16 * st + 8 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) qb[st][j] = (qb[st][j] & a.q_and) ^ a.q_xor;
    }
  }

  const int kv = head / a.group;
  const char *kg = reinterpret_cast<const char *>(a.k + ks.begin * a.k_token + kv * a.k_head);
  const char *vg = reinterpret_cast<const char *>(a.v + ks.begin * a.v_token + kv * a.v_head);
  const uint32_t k_bytes = (uint32_t)a.k_token * 2, v_bytes = (uint32_t)a.v_token * 2;  // between rows
  // 32 rows from `first` on into LDS. Load i brings rows kLoadRows * i .., lane l landing in chunk l % kChunks of the
  // load's row l / kChunks, which holds the row's chunk (l % kChunks) ^ turn(row): the row's number mod 16 for keys (mod 16
  // of its pair for rows of 128 bytes, two of which make a pass over the banks), 4 times it mod 4 (mod 2 of its pair) for values.
  const uint32_t load_row = lane / kChunks;
  const uint32_t k_chunk = 16u * (uint32_t)((lane % kChunks) ^ (lane >> 4));  // but for the load's number
  const uint32_t v_chunk = 16u * (uint32_t)((lane % kChunks) ^ (DIM == 128 ? 4 * (lane >> 4) : 4 * ((lane >> 4) & 1)));
  auto stage = [&](const char *from, uint32_t bytes, uint32_t chunk, bool turned, char *to, int first) __attribute__((always_inline)) {
    const int rows = min(32, keys - first);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char *>(from) + (int64_t)first * bytes, (short)0, rows > 0 ? (rows - 1) * bytes + kRow : 0, 0x00020000);
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = qw + QW * u;
      const uint32_t turn = turned ? 64u * (uint32_t)(DIM == 128 ? i & 3 : i & 1) : 0u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(to + i * 1024), 16,
                                               (i * kLoadRows + load_row) * bytes + (chunk ^ turn), 0, 0, 0);
    }
  };

  // Byte offsets of this lane's operands in a tile: of key row n, dimensions 16 st + 8 h (chunk 2 st + h) at
  // k_at ^ 32 st; and, for the transposing reads, of key 4 h + (lane % 16) / 4, dimensions
  // 32 t + 16 ((lane / 16) % 2) + 4 (lane % 4) at v_at ^ 64 t.
  const uint32_t x4 = (lane >> 2) & 3;
  const uint32_t k_at = (uint32_t)n * kRow + 16u * (uint32_t)(h ^ (DIM == 128 ? n & 15 : (n >> 1) & 7));
  const uint32_t v_at = (4u * h + x4) * kRow + 32u * ((lane >> 4) & 1) + 8u * (lane & 3) + 64u * (DIM == 128 ? x4 : x4 >> 1);
  const int limit = min(q0 + n, queries - 1) + shift;  // the last key this lane's query sees

  float m = -INFINITY, l = 0.f;  // running maximum (before the scale) and this lane's share of the sum, query q0 + n
  float mx = -INFINITY;          // the largest of the scores at hand
  f32x16 o[kOut];                // o[t][r] = O[query q0 + n][dimension 32 t + 8 (r / 4) + 4 h + r % 4]
#pragma unroll
  for (int t = 0; t < kOut; ++t) o[t] = f32x16{};

  auto largest = [&](const f32x16 &sc) __attribute__((always_inline)) {
    mx = fmaxf(sc[0], sc[1]);
#pragma unroll
    for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, sc[r]), sc[r + 1]);
  };
  // Before the scores of keys k0 .. k0 + 31 are used (sc[r]: key k0 + 8 (r / 4) + 4 h + r % 4, query q0 + n): hides those
  // past each query's limit and moves the running maximum. Whether it moves depends on the query's own scores alone,
  // and one that stays is scaled by exactly 1: a query's output does not depend on which others share the wave.
  auto settle = [&](f32x16 &sc, int k0) __attribute__((always_inline)) {
    if (k0 + 31 > q0 + shift) {
      asm volatile("" ::: "memory");  // stays a branch: few blocks are hidden in part
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = k0 + 8 * (r >> 2) + 4 * h + (r & 3) > limit ? -INFINITY : sc[r];
      largest(sc);
    }
    const float mnew = halves_max(mx);
    const bool grow = mnew > m + a.lag;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float alpha = grow ? __builtin_amdgcn_exp2f((m - mnew) * a.sl2) : 1.f;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < kOut; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] *= alpha;
      m = grow ? mnew : m;
    }
  };
  // The next 32 keys' scores, and these 32 keys' share of the outputs: O^T += V^T P^T, sixteen keys at a time (slots 0-3 of half h
  // are keys 4 h .. + 3, slots 4-7 the keys 8 on). The order here is the order of issue (the scheduling barriers hold the
  // compiler to it): the exponentials in the time of the products, operands read two products ahead, the next scores'
  // maximum last.
  // The first two of a step's key operands set out before its scores' maxima are settled.
  auto first_keys = [&](const char *kt, u32x4 &x, u32x4 &y) __attribute__((always_inline)) {
    x = *reinterpret_cast<const u32x4 *>(kt + k_at);
    y = *reinterpret_cast<const u32x4 *>(kt + (k_at ^ 32u));
    __builtin_amdgcn_sched_barrier(0);
  };
  auto step = [&](const f32x16 &cur, f32x16 &next, const char *vt, const char *kt_next, u32x4 x, u32x4 y) __attribute__((always_inline)) {
    const float base = m == -INFINITY ? 0.f : lift - m * a.sl2;  // no key yet: every score is -infinity
    uint32_t pb[8];
    auto pair = [&](int p) __attribute__((always_inline)) {  // probabilities 2 p and 2 p + 1
      pb[p] = pack2<F16>(__builtin_amdgcn_exp2f(__builtin_fmaf(cur[2 * p], a.sl2, base)),
                         __builtin_amdgcn_exp2f(__builtin_fmaf(cur[2 * p + 1], a.sl2, base)), l);
      asm volatile("" : "+v"(pb[p]));
    };
    auto key = [&](int st) __attribute__((always_inline)) { return *reinterpret_cast<const u32x4 *>(kt_next + (k_at ^ (32u * st))); };
    auto value = [&](int i) __attribute__((always_inline)) {
      const char *at = vt + 16 * (i / kOut) * kRow + (v_at ^ (64u * (i % kOut)));
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(at + 8 * kRow)));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    constexpr int kGroups = kSteps + kOut;  // products before the second sixteen keys' probabilities are needed
    int done = 0;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const u32x4 z = st + 2 < kSteps ? key(st + 2) : value(st + 2 - kSteps);
      next = mfma32<F16>(x, qb[st], st == 0 ? f32x16{} : next);
#pragma unroll
      for (; done < max(8 * (st + 1) / kGroups, 4 * (st + 1) / kSteps); ++done) pair(done);
      x = y;
      y = z;
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < 2 * kOut; ++i) {
      const u32x4 z = i + 2 < 2 * kOut ? value(i + 2) : x;
      const int j = i / kOut, t = i % kOut;
      o[t] = mfma32<F16>(x, u32x4{pb[4 * j], pb[4 * j + 1], pb[4 * j + 2], pb[4 * j + 3]}, o[t]);
#pragma unroll
      for (; i < kOut && done < 8 * (kSteps + i + 1) / kGroups; ++done) pair(done);
      x = y;
      y = z;
      if (i == kOut) {
        largest(next);
        asm volatile("" : "+v"(mx));  // here, not where it is used
      }
      if (i < kOut) __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  // Blocks of this key group: kw, kw + KW, ... up to the workgroup's last key; every wave runs every turn (the barriers
  // are workgroup-wide). In turn `it` the values of block b = it * KW + kw are in LDS, and the keys 32 further on: b's but for
  // its first 32, then the first 32 of the group's next block. Those of the next turn set out behind the barrier, which also says
  // that their buffers are no longer read. Scores past the wave's last key are computed from whatever lies there and dropped.
  const int last_key = min((tile + 1) * kQueries, queries) - 1 + shift;
  const int blocks = last_key < 0 ? 0 : last_key / KB + 1, turns = (blocks + KW - 1) / KW;
  const int reach = q0 < queries ? min(q0 + 31, queries - 1) + shift : -1;  // this wave's last key
  f32x16 s0, s1;
  auto stage_keys = [&](char *to, int b) __attribute__((always_inline)) {  // those of the turn of block b
    to += kw * kTile;
    if (kSubs == 2 && b * KB + 32 <= last_key) stage(kg, k_bytes, k_chunk, true, to, b * KB + 32);
    if ((b + KW) * KB <= last_key) stage(kg, k_bytes, k_chunk, true, to + (kSubs - 1) * kSub, (b + KW) * KB);
  };
  auto stage_values = [&](char *to, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < kSubs; ++s)
      if (b * KB + 32 * s <= last_key) stage(vg, v_bytes, v_chunk, false, to + kw * kTile + s * kSub, b * KB + 32 * s);
  };
  auto turn = [&](int it, const char *k_cur, char *k_next, const char *v_cur, char *v_next) __attribute__((always_inline)) {
    drain_barrier();
    const int b = it * KW + kw, k0 = b * KB;
    u32x4 x, y;
    first_keys(k_cur + kw * kTile, x, y);
    stage_values(v_next, b + KW);
    stage_keys(k_next, b + KW);
    k_cur += kw * kTile;
    v_cur += kw * kTile;
    if (k0 > reach) return;
    if constexpr (kSubs == 2) {
      step(s0, s1, v_cur, k_cur, x, y);
      if (k0 + 32 > reach) return;
      first_keys(k_cur + kSub, x, y);
      settle(s1, k0 + 32);
      step(s1, s0, v_cur + kSub, k_cur + kSub, x, y);
    } else {
      step(s0, s1, v_cur, k_cur, x, y);
      s0 = s1;
    }
    if (k0 + KW * KB <= reach) settle(s0, k0 + KW * KB);
  };
  if (turns > 0) {
    if (kw * KB <= last_key) stage(kg, k_bytes, k_chunk, true, k_odd + kw * kTile, kw * KB);
    stage_keys(k_even, kw);
    stage_values(v_even, kw);
    drain_barrier();
    if (kw * KB <= reach) {
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
        s0 = mfma32<F16>(*reinterpret_cast<const u32x4 *>(k_odd + kw * kTile + (k_at ^ (32u * st))), qb[st], st == 0 ? f32x16{} : s0);
      largest(s0);
      settle(s0, kw * KB);
    }
  }
  int it = 0;
  for (; it + 2 <= turns; it += 2) {
    turn(it, k_even, k_odd, v_even, v_odd);
    turn(it + 1, k_odd, k_even, v_odd, v_even);
  }
  if (it < turns) turn(it, k_even, k_odd, v_even, v_odd);

  l = halves_sum(l);
  if constexpr (KW > 1) {
    // The groups' (m, l) meet in LDS; with M = max m, every group scales its O by exp(m - M), and group
    // t % KW sums the output tile t of all. A group whose blocks a query does not see has m = -inf, l = 0, O = 0
    // for it and weighs nothing (or NaN, where its scores were).
    constexpr int kHalf = kOut / 2;  // output tiles that go through the keys' buffers; the others through the values'
    static_assert(kHalf * QW * KW * 4096 <= 2 * KW * kTile, "half the output tiles of every wave fit two buffers");
    stats[kw][qw][0][lane] = m;
    stats[kw][qw][1][lane] = l;
    __syncthreads();  // every tile read is done, too
    float mm = m, total = 0.f;
#pragma unroll
    for (int g = 0; g < KW; ++g) mm = fmaxf(mm, stats[g][qw][0][lane]);
    auto weight = [&](float mine) { return mine == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mine - mm) * a.sl2); };
#pragma unroll
    for (int g = 0; g < KW; ++g) total += stats[g][qw][1][lane] * weight(stats[g][qw][0][lane]);
    l = total;
    const float alpha = weight(m);
    // Tile t of wave (g, qw): 4 KiB; those of a half in the even buffer first, then in the odd one.
    auto at = [&](int g, int t) {
      const int index = (g * QW + qw) * kHalf + t % kHalf, half = KW * kTile / 4096;
      char *even = t < kHalf ? k_even : v_even, *odd = t < kHalf ? k_odd : v_odd;
      return reinterpret_cast<float *>(index < half ? even + index * 4096 : odd + (index - half) * 4096) + lane;
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
  // A value that is not finite also meets the zero probabilities of queries that do not see its key (0 * inf is NaN). Outputs
  // that are not finite are looked at again where such a value lies among the keys that a query of this wave met unseen. The
  // look costs 0.2 us a call (12 prompts of up to 60 tokens 6.4 -> 6.6).
  const int query = q0 + n;
  float probe = 0.f;
#pragma unroll
  for (int t = 0; t < kOut; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (KW == 1 || t % KW == kw) probe = __builtin_fmaf(o[t][r], 0.f, probe);
  const uint64_t odd = __builtin_amdgcn_ballot_w64(query < queries && __builtin_isnan(probe));
  uint32_t again = (uint32_t)(odd | odd >> 32);
  if (again != 0 && !unseen_odd_value<F16, DIM>(a, vg, max(q0 + shift + 1, 0), min(reach | 31, keys - 1), lane)) again = 0;
  // A query that sees no key gets zeros; one whose scores are all -infinity has l = 0 and O = 0 as well, and gets NaN.
  const float inv = limit < 0 ? 0.f : 1.0f / l;
  uint16_t *dst = a.out + (qs.begin + query) * a.out_token + head * a.out_head + 4 * h;
  if (query < queries && !(again >> n & 1)) {
#pragma unroll
    for (int t = 0; t < kOut; ++t) {
      if (KW > 1 && t % KW != kw) continue;
#pragma unroll
      for (int rq = 0; rq < 4; ++rq)
        *reinterpret_cast<u32x2 *>(dst + 32 * t + 8 * rq) = u32x2{half2_bits<F16>(o[t][4 * rq] * inv, o[t][4 * rq + 1] * inv),
                                                                  half2_bits<F16>(o[t][4 * rq + 2] * inv, o[t][4 * rq + 3] * inv)};
    }
  }
  for (; again != 0; again &= again - 1) {
    const int i = q0 + __builtin_ctz(again);
    seen_keys_alone<F16, DIM, KW>(a, a.q + (qs.begin + i) * a.q_token + head * a.q_head, kg, vg, i + shift,
                                  a.out + (qs.begin + i) * a.out_token + head * a.out_head, kw, lane);
  }
}

template <bool F16, int DIM>
hipError_t launch_typed(const PackedAttention &a, hipStream_t stream) {
  auto launch = [&](auto kernel, int queries, int waves) {
    const int64_t tiles = a.total_q / queries + a.sequences;  // at least what the sequences' partial tiles make it
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles * a.heads)), dim3(64 * waves), 0, stream, a);
  };
  // Which split of the waves, by how many tiles of 32 and 64 queries the rows can make and how many keys a sequence has on
  // average (us, graph replays, at 40/8 heads of 128 where no others are named):
  //   <1, 4, 32> where its workgroups fit the CUs at once and there is a chain of key blocks to shorten: 128 tokens 7.6
  //              against 8.1 of <4, 1, 64>, 256 tokens of 16/2 heads 8.5 against 10.1; but 12 prompts of up to 60 tokens at
  //              32/8 heads 12.7 against 6.6, whose chains are short;
  //   <2, 4, 32> likewise: 1024 tokens of 16/2 heads 17.5 against 23.9; but 512 tokens (320 workgroups) 18.8 against 15.5;
  //   <2, 2, KB> where the longest chain still outlasts the others' work. Heads of 64: KB 64 up to two and a half
  //              workgroups a CU, which holds two (3 turns of up to 400 behind up to 6000 keys 39 against 62 of <4, 1, 64>, 2500
  //              tokens of 16/2 heads 27 against 37), beyond KB 32, of which a CU holds four (9 turns of up to 777 behind up to 2500 of
  //              28/4 heads 34.5 against 40 of KB 64 and of <4, 1, 64>, 2048 tokens of 28/4 30 against 34; but 1477 tokens of
  //              64/8, 1600 workgroups, 30 against 26). Heads of 128: KB 32 and longer chains (3000 tokens of 16/2 heads 54
  //              against 60, those 3 turns 60 against 82; but 2048 tokens, 1280 workgroups, 70 against 60, and 3 prompts of up
  //              to 300 tokens 12.6 against 11.5). The lengths themselves, on the device, decide as much: of 13 shapes of 128
  //              that the rule sends here three got slower, by 2 to 16%, ten faster, by up to 27%;
  //   <4, 1, 64> for all else: 1024 tokens 28.1 against 34.2 of <2, 4, 32>, 8190 tokens 650 against 756 of <2, 2, 32>.
  const int64_t tiles32 = (a.total_q + (int64_t)31 * a.sequences) / 32 * a.heads,
                tiles64 = (a.total_q + (int64_t)63 * a.sequences) / 64 * a.heads;
  const bool some_keys = a.total_k >= (int64_t)96 * a.sequences, many_keys = a.total_k >= (int64_t)256 * a.sequences;
  if (tiles32 <= a.cus && some_keys) launch(packed_attention_kernel<F16, DIM, 1, 4, 32>, 32, 4);
  else if (tiles64 <= a.cus && some_keys) launch(packed_attention_kernel<F16, DIM, 2, 4, 32>, 64, 8);
  else if (DIM == 64 ? tiles64 <= 5 * (int64_t)a.cus && some_keys : tiles64 < 3 * (int64_t)a.cus && many_keys) {
    if (DIM == 64 && 2 * tiles64 <= 5 * (int64_t)a.cus) launch(packed_attention_kernel<F16, DIM, 2, 2, DIM == 64 ? 64 : 32>, 64, 4);
    else launch(packed_attention_kernel<F16, DIM, 2, 2, 32>, 64, 4);
  } else launch(packed_attention_kernel<F16, DIM, 4, 1, 64>, 128, 4);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_packed_attention(const PackedAttention &a, bool f16, int dim, hipStream_t stream) {
  if (f16) return dim == 128 ? launch_typed<true, 128>(a, stream) : launch_typed<true, 64>(a, stream);
  return dim == 128 ? launch_typed<false, 128>(a, stream) : launch_typed<false, 64>(a, stream);
}

}  // namespace tx
