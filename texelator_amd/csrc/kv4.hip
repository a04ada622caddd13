// Writing, reading and moving the rows of a paged 4-bit KV cache (gfx950; layout in kv4.h).
//
// No reference counterpart: the reference's Hugging Face path keeps its caches in 16 bits.
//
// A group of 32 elements is stored as MXFP4, the rule of the activation quantizer (fp4.hip): scale exponent
// e = max(floor(log2(amax)) - 2 + 127, 0), each code the E2M1 value nearest to v * 2^(127 - e), ties to the even code,
// saturated at 6. A group that holds an infinity or a NaN gets e = 255 and reads back as NaN.
//
// All are copies with arithmetic on the way, bound by memory.
#include "elementwise.h"
#include "kernels.h"
#include "kv4.h"

namespace tx {

namespace {

constexpr int kThreads = 256;
constexpr int kCuEntries = 2048;  // sequence starts held in LDS: 8 KiB

// Where the token rows of a call lie in the cache. cu [sequences + 1]: sequence s has the tokens cu[s] .. cu[s + 1] - 1,
// which are the last ones of its lengths[s] positions; null: token s is the last one of sequence s.
// Returns the byte offset of the row's half page (its keys or values of one head) and the position in it, or a
// negative page where the token has no row in the cache.
struct Row {
  int64_t page;
  int offset;
};

// The sequence that has a token and the token's position in it, which may be below zero; sequence -1: no sequence has it.
struct Place {
  int sequence, position;
};

__device__ __forceinline__ Place place_of(const Kv4Pool &pool, const int *cu, const int *starts, int token) {
  int sequence = token, back = 1;  // `back`: how far before the sequence's end the token lies
  if (cu) {
    if (token < cu[0] || token >= cu[pool.sequences]) return {-1, 0};
    int low = 0, high = pool.sequences;  // cu[low] <= token < cu[high]
    while (high - low > 1) {
      const int mid = (low + high) >> 1;
      if (starts[mid] <= token) low = mid;
      else high = mid;
    }
    sequence = low;
    back = cu[low + 1] - token;
  }
  if (back <= 0 || (cu == nullptr && token >= pool.sequences)) return {-1, 0};
  return {sequence, kv4_length(pool, sequence) - back};
}

__device__ __forceinline__ Row row_at(const Kv4Pool &pool, const Place &place) {
  if (place.sequence < 0 || place.position < 0) return {-1, 0};
  const int page = pool.table[place.sequence * pool.table_stride + (place.position >> pool.page_shift)];
  if ((uint32_t)page >= (uint64_t)pool.num_pages) return {-1, 0};
  return {page, place.position & ((1 << pool.page_shift) - 1)};
}

__device__ __forceinline__ Row locate(const Kv4Pool &pool, const int *cu, const int *starts, int token) {
  return row_at(pool, place_of(pool, cu, starts, token));
}

// Sequence starts into LDS where they fit, for the binary search.
__device__ __forceinline__ const int *stage_starts(const int *cu, int sequences, int *lds) {
  if (!cu || sequences > kCuEntries) return cu;
  for (int i = threadIdx.x; i < sequences; i += kThreads) lds[i] = cu[i];
  __syncthreads();
  return lds;
}

__device__ __forceinline__ uint32_t e2m1_octet(const float *v) {
  uint32_t word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], 1.0f, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], 1.0f, 1);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], 1.0f, 3);
}

// Grid: x token blocks, y = kv head * 2 + (0 keys, 1 values). A thread has one group of one row; the groups of a row
// are neighbours and the rows follow each other, so a wave's codes are 1 KiB of consecutive bytes within a page.
template <bool F16, int DIM>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(const uint16_t *k, int64_t k_token, int64_t k_head,
                                                              const uint16_t *v, int64_t v_token, int64_t v_head,
                                                              int tokens, const int *cu, Kv4Pool pool) {
  constexpr int kGroups = DIM / 32;
  __shared__ int lds[kCuEntries];
  const int *starts = stage_starts(cu, pool.sequences, lds);
  const int group = threadIdx.x % kGroups;
  const int64_t index = (int64_t)blockIdx.x * (kThreads / kGroups) + threadIdx.x / kGroups;
  if (index >= tokens) return;
  const int token = (int)index, head = blockIdx.y >> 1;
  const bool values = blockIdx.y & 1;
  const Row row = locate(pool, cu, starts, token);
  if (row.page < 0) return;
  const uint16_t *src = (values ? v + token * v_token + head * v_head : k + token * k_token + head * k_head) + 32 * group;
  float x[32];
  uint32_t top = 0;  // the largest magnitude's bits; as integers they order like the magnitudes, infinities and NaN last
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32x4 u = reinterpret_cast<const u32x4 *>(src)[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[8 * i + 2 * j] = half_bits_to_float<F16>((uint16_t)(u[j] & 0xFFFFu));
      x[8 * i + 2 * j + 1] = half_bits_to_float<F16>((uint16_t)(u[j] >> 16));
    }
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  const uint32_t field = top >> 23;
  const uint32_t e = field == 255 ? 255 : (uint32_t)max((int)field - 2, 0);
  const float inverse = __uint_as_float((254u - min(e, 254u)) << 23);  // 2^(127 - e), exact
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] *= inverse;
  uint8_t *half = pool.pages + ((row.page * pool.kv_heads + head) * 2 + values) * kv4_half_bytes(pool.page_shift, DIM);
  u32x4 codes = {e2m1_octet(x), e2m1_octet(x + 8), e2m1_octet(x + 16), e2m1_octet(x + 24)};
  if (e == 255) codes = u32x4{0, 0, 0, 0};
  *reinterpret_cast<u32x4 *>(half + row.offset * (DIM / 2) + 16 * group) = codes;
  half[((int64_t)(DIM / 2) << pool.page_shift) + row.offset * kGroups + group] = (uint8_t)e;
}

// The same the other way: k_out and v_out [tokens][kv_heads][DIM], row strides as given. A workgroup finds the places of
// its kReadRows rows first, one a thread; then a thread turns four bytes of codes into 16 bytes of output, so that a wave stores
// 1 KiB of consecutive bytes: 20291 tokens of 8 heads of 128 17.7 us (5.9 TB/s), with a group a thread, 64 bytes each, 29.8.
template <int DIM>
constexpr int kReadRows = 8192 / DIM;
template <bool F16, int DIM>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(uint16_t *k, int64_t k_token, int64_t k_head, uint16_t *v,
                                                            int64_t v_token, int64_t v_head, int tokens, const int *cu,
                                                            Kv4Pool pool) {
  constexpr int kGroups = DIM / 32, kOctets = DIM / 8, kPasses = kReadRows<DIM> * kOctets / kThreads;
  __shared__ int lds[kCuEntries];
  __shared__ int pages[kReadRows<DIM>], offsets[kReadRows<DIM>];
  const int *starts = stage_starts(cu, pool.sequences, lds);
  const int64_t first = (int64_t)blockIdx.x * kReadRows<DIM>;
  if (threadIdx.x < kReadRows<DIM>) {
    Row row = {-1, 0};
    if (first + threadIdx.x < tokens) row = locate(pool, cu, starts, (int)first + threadIdx.x);
    pages[threadIdx.x] = (int)row.page;
    offsets[threadIdx.x] = row.offset;
  }
  __syncthreads();
  const int head = blockIdx.y >> 1;
  const bool values = blockIdx.y & 1;
  const int64_t half_bytes = kv4_half_bytes(pool.page_shift, DIM), scales_at = (int64_t)(DIM / 2) << pool.page_shift;
  const int octet = threadIdx.x % kOctets;
  uint16_t *out = (values ? v + head * v_head : k + head * k_head) + 8 * octet;
  const int64_t stride = values ? v_token : k_token;
  uint32_t codes[kPasses], scale[kPasses];
  int page[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = threadIdx.x / kOctets + i * (kThreads / kOctets);
    page[i] = pages[r];
    const uint8_t *half = pool.pages + (((int64_t)max(page[i], 0) * pool.kv_heads + head) * 2 + values) * half_bytes;
    codes[i] = *reinterpret_cast<const uint32_t *>(half + offsets[r] * (DIM / 2) + 4 * octet);
    scale[i] = half[scales_at + offsets[r] * kGroups + octet / 4];
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int64_t token = first + threadIdx.x / kOctets + i * (kThreads / kOctets);
    if (page[i] >= 0) *reinterpret_cast<u32x4 *>(out + token * stride) = kv4_octet<F16>(codes[i], __uint_as_float(scale[i] << 23));
  }
}

// A value of two 16-bit numbers turned: a cos - b sin in 64 bits, rounded to 32 so that no comparison of the quantizer comes out
// otherwise: towards an odd last bit where it does not fit (borders of codes and scales are even by many bits). The products are exact in
// 64 bits, and so is their difference but where one is below 2^-18 of the other. One below 2^-53 of the other is not seen, though on
// a border it would decide: to bring back what the sum leaves out took 141 us instead of 137 for 21,447 tokens of 56 heads.
__device__ __forceinline__ float turned_to_odd(float a, float cos, float b, float sin) {
  const double exact = __builtin_fma((double)a, (double)cos, -((double)b * (double)sin));
  const float near = (float)exact;
  const double back = (double)near;
  uint32_t bits = __float_as_uint(near);
  const bool moves = (back != exact) & !(bits & 1) & ((bits & 0x7F800000u) != 0x7F800000u);
  const uint32_t step = fabs(exact) > fabs(back) ? 1u : ~0u;
  return __uint_as_float(bits + (moves ? step : 0u));
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

// kv4_append with the rotary embedding on the way, and the queries' rotation in the same launch. Dimensions below `rotary` of
// every query and key head are turned in pairs (i, i + rotary / 2), or (2i, 2i + 1) where INTERLEAVED, by the angle that the tables'
// row of the token's position has for pair i; the others pass. Grid: x token blocks, y blocks of `per` heads of [q | k | v]. A
// thread has eight elements of one token, loads their cosines and sines once for all its heads and has the next head's elements
// under way while it turns one's; a pair's other element comes from another lane where it is not its own; four neighbours share a
// group's scale. Queries are computed in 32 bits, two products and their sum (off by 2^-23 (|a cos| + |b sin|) at most, which may be
// much of a result that cancels), then rounded. Keys are stored and returned (k_out, where given) from the value in 64 bits
// (turned_to_odd), rounded once: a slowly turning key stays so near the 16-bit value that it was that 32 bits put it midway
// between two codes. Bound by memory: 136 us for 21,447 tokens of 40 + 2 * 8 heads of 128, 4.05 TB/s.
template <bool F16, int DIM, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void kv4_append_rope_kernel(Kv4Rope a, Kv4Pool pool) {
  constexpr int kChunks = DIM / 8, kGroups = DIM / 32;
  __shared__ int lds[kCuEntries];
  const int *starts = stage_starts(a.cu, pool.sequences, lds);
  const int chunk = threadIdx.x % kChunks;
  const int64_t index = (int64_t)blockIdx.x * (kThreads / kChunks) + threadIdx.x / kChunks;
  if (index >= a.tokens) return;
  const int token = (int)index;
  const Place place = place_of(pool, a.cu, starts, token);
  if (place.sequence < 0) return;
  const Row row = row_at(pool, place);
  const int position = a.positions ? a.positions[token] : place.position;
  const bool turns = 8 * chunk < a.rotary;
  // Pairs of this thread: eight where the halves pair up (its elements' partners are another chunk), else four.
  const int half = a.rotary / 2;
  const bool second = !INTERLEAVED && 8 * chunk >= half;  // of the half layout: b cos + a sin
  const int pair = INTERLEAVED ? 4 * chunk : 8 * chunk - (second ? half : 0);
  const int partner = second ? -half : half;
  constexpr int kPairs = INTERLEAVED ? 4 : 8;
  float cs[kPairs], sn[kPairs];  // sn with the sign that it has for this thread's (or the even) elements
  if (turns) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) cs[i] = sn[i] = NAN;
    if ((uint32_t)position < (uint64_t)a.table_rows) {
      const float *cos = a.cos + position * a.cos_row + pair, *sin = a.sin + position * a.sin_row + pair;
      if (a.wide) {
#pragma unroll
        for (int i = 0; i < kPairs; i += 4) {
          const f32x4 c = *reinterpret_cast<const f32x4 *>(cos + i), s = *reinterpret_cast<const f32x4 *>(sin + i);
#pragma unroll
          for (int j = 0; j < 4; ++j) cs[i + j] = c[j], sn[i + j] = s[j];
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) cs[i] = cos[i], sn[i] = sin[i];
      }
#pragma unroll
      for (int i = 0; i < kPairs; ++i) sn[i] = second ? -sn[i] : sn[i];
    }
  }
  const int heads = a.heads + 2 * pool.kv_heads, first = blockIdx.y * a.per, last = min(first + a.per, heads);
  const uint16_t *const q = a.q + token * a.q_token + 8 * chunk;
  uint16_t *const q_out = a.q_out + token * a.q_out_token + 8 * chunk;
  auto load = [&](int h) __attribute__((always_inline)) {
    const uint16_t *src = h < a.heads ? q + h * a.q_head
                          : 8 * chunk + (h < a.heads + pool.kv_heads ? a.k + token * a.k_token + (h - a.heads) * a.k_head
                                                                     : a.v + token * a.v_token + (h - a.heads - pool.kv_heads) * a.v_head);
    return *reinterpret_cast<const u32x4 *>(src);
  };
  // The partners' elements: this chunk's own, or another lane's of the same token.
  const int partner_lane = 4 * ((threadIdx.x & 63) + (turns ? partner / 8 : 0));
  auto partners_of = [&](u32x4 mine) __attribute__((always_inline)) {
    if constexpr (!INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(partner_lane, (int)mine[i]);
    }
    return mine;
  };
  u32x4 next = load(first);
#pragma unroll 1
  for (int h = first; h < last; ++h) {
    const u32x4 mine = next;
    if (h + 1 < last) next = load(h + 1);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = half_bits_to_float<F16>((uint16_t)(mine[i / 2] >> (16 * (i % 2))));
    if (h < a.heads + pool.kv_heads) {
      const u32x4 theirs = partners_of(mine);
      u32x4 packed = mine;
      if (turns) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int from = INTERLEAVED ? i ^ 1 : i;
          y[i] = half_bits_to_float<F16>((uint16_t)(theirs[from / 2] >> (16 * (from % 2))));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int p = INTERLEAVED ? i / 2 : i;
          const float s = INTERLEAVED && i % 2 == 1 ? -sn[p] : sn[p];
          x[i] = h < a.heads ? x[i] * cs[p] - y[i] * s : turned_to_odd(x[i], cs[p], y[i], s);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) packed[i] = to_half_bits<F16>(x[2 * i]) | (uint32_t)to_half_bits<F16>(x[2 * i + 1]) << 16;
      }
      if (h < a.heads) {
        *reinterpret_cast<u32x4 *>(q_out + h * a.q_out_head) = packed;
        continue;
      }
      if (a.k_out) *reinterpret_cast<u32x4 *>(a.k_out + token * a.k_out_token + (h - a.heads) * a.k_out_head + 8 * chunk) = packed;
    }
    if (row.page < 0) continue;  // all four threads of a group alike
    const int which = h < a.heads + pool.kv_heads ? 1 : 2, head = h - a.heads - (which - 1) * pool.kv_heads;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));  // quad_perm [1,0,3,2]
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));  // quad_perm [2,3,0,1]
    const uint32_t field = top >> 23;
    const uint32_t e = field == 255 ? 255 : (uint32_t)max((int)field - 2, 0);
    const float inverse = __uint_as_float((254u - min(e, 254u)) << 23);  // 2^(127 - e), exact
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= inverse;
    uint8_t *cache = pool.pages + ((row.page * pool.kv_heads + head) * 2 + (which - 1)) * kv4_half_bytes(pool.page_shift, DIM);
    *reinterpret_cast<uint32_t *>(cache + row.offset * (DIM / 2) + 4 * chunk) = e == 255 ? 0u : e2m1_octet(x);
    if (chunk % 4 == 0) cache[((int64_t)(DIM / 2) << pool.page_shift) + row.offset * kGroups + chunk / 4] = (uint8_t)e;
  }
}

// The rows of an accepted path moved together: of sequence s, whose last cu[s + 1] - cu[s] positions are drafted rows, row path[cu[s] + j]
// moves to the place of row j, j = 1 .. accepted[s]. A wave has one head's keys or values of one sequence, in `per` layers: it holds
// every piece of a layer that moves before it stores the first, so paths may run in any order, and finds their places once for all
// layers. Bound by the latency of its dependent loads. Grid: x sequences, y heads and halves by kKeepWaves, z layers by `per`.
constexpr int kKeepWaves = 4;
template <int DIM>
__global__ __launch_bounds__(64 * kKeepWaves) void kv4_keep_path_kernel(Kv4Pool pool, int layers, int per, int64_t layer_bytes,
                                                                        const int *cu, int tokens, const int *path,
                                                                        const int *accepted, int *lengths_out) {
  constexpr int kGroups = DIM / 32, kHeld = kMostDrafts * kGroups / 64;
  const int sequence = blockIdx.x, lane = threadIdx.x & 63, half = blockIdx.y * kKeepWaves + (threadIdx.x >> 6);
  const int begin = min(max(cu[sequence], 0), tokens), count = min(max(cu[sequence + 1], begin), tokens) - begin;
  const int rows = min(count, kMostDrafts);
  const int length = kv4_length(pool, sequence), context = length - count;
  const int kept = min(max(accepted[sequence], -1), rows - 1);
  if (half == 0 && lane == 0 && blockIdx.z == 0) lengths_out[sequence] = context + kept + 1;
  if (half >= 2 * pool.kv_heads || kept < 1) return;
  const int64_t half_bytes = kv4_half_bytes(pool.page_shift, DIM), scales_at = (int64_t)(DIM / 2) << pool.page_shift;
  const int group = lane % kGroups;
  // A group's place: of its codes in a layer (below 0: none), and how far behind them its scale is.
  struct Group {
    int64_t codes;
    int scale;
  };
  auto group_at = [&](int position) -> Group {
    const Row row = row_at(pool, {sequence, position});
    if (row.page < 0) return {-1, 0};
    const int codes = row.offset * (DIM / 2) + 16 * group;
    return {(row.page * pool.kv_heads * 2 + half) * half_bytes + codes, (int)scales_at + row.offset * kGroups + group - codes};
  };
  Group from[kHeld], to[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int j = 1 + (64 * i + lane) / kGroups;
    from[i] = to[i] = {-1, 0};
    if (j > kept) continue;
    const int row = path[begin + j];
    if (row < 0 || row >= rows || row == j) continue;
    from[i] = group_at(context + row);
    to[i] = group_at(context + j);
    if (to[i].codes < 0) from[i].codes = -1;
  }
  struct Held {
    u32x4 codes[kHeld];
    uint8_t scale[kHeld];
  };
  auto load = [&](int layer, Held &held) __attribute__((always_inline)) {
    const uint8_t *pages = pool.pages + layer * layer_bytes;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (from[i].codes >= 0) {
        held.codes[i] = *reinterpret_cast<const u32x4 *>(pages + from[i].codes);
        held.scale[i] = pages[from[i].codes + from[i].scale];
      }
  };
  const int first = blockIdx.z * per, end = min(first + per, layers);
  Held held;
  load(first, held);
#pragma unroll 1
  for (int layer = first; layer < end; ++layer) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // everything of this layer is held
    const Held now = held;
    if (layer + 1 < end) load(layer + 1, held);
    uint8_t *pages = pool.pages + layer * layer_bytes;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (from[i].codes >= 0) {
        *reinterpret_cast<u32x4 *>(pages + to[i].codes) = now.codes[i];
        pages[to[i].codes + to[i].scale] = now.scale[i];
      }
  }
}

// Page pairs travel as kernel arguments: no copy to the device, nothing to keep alive.
struct Kv4Pairs {
  uint32_t src[kKv4Pairs], dst[kKv4Pairs];
};

// Grid: x parts of a page, y pair, z layer; a thread moves kCopyLoads 16-byte pieces.
constexpr int kCopyLoads = 4;
__global__ __launch_bounds__(kThreads) void kv4_copy_kernel(uint8_t *pool, int64_t layer_bytes, int64_t page_bytes,
                                                            Kv4Pairs pairs) {
  const int64_t pieces = page_bytes / 16;
  uint8_t *layer = pool + blockIdx.z * layer_bytes;
  const u32x4 *src = reinterpret_cast<const u32x4 *>(layer + pairs.src[blockIdx.y] * page_bytes);
  u32x4 *dst = reinterpret_cast<u32x4 *>(layer + pairs.dst[blockIdx.y] * page_bytes);
  const int64_t first = (int64_t)blockIdx.x * (kThreads * kCopyLoads) + threadIdx.x;
  u32x4 held[kCopyLoads];
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i)
    if (first + i * kThreads < pieces) held[i] = src[first + i * kThreads];
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i)
    if (first + i * kThreads < pieces) dst[first + i * kThreads] = held[i];
}

template <typename Launch>
void by_type(bool f16, int dim, Launch launch) {
  using std::integral_constant;
  auto with_dim = [&](auto type) {
    if (dim == 128) launch(type, integral_constant<int, 128>{});
    else launch(type, integral_constant<int, 64>{});
  };
  if (f16) with_dim(integral_constant<bool, true>{});
  else with_dim(integral_constant<bool, false>{});
}

}  // namespace

hipError_t launch_kv4_append(const uint16_t *k, int64_t k_token, int64_t k_head, const uint16_t *v, int64_t v_token,
                             int64_t v_head, int tokens, bool f16, int dim, const int *cu, const Kv4Pool &pool,
                             hipStream_t stream) {
  const int rows = kThreads / (dim / 32);
  by_type(f16, dim, [&](auto type, auto d) {
    hipLaunchKernelGGL((kv4_append_kernel<decltype(type)::value, decltype(d)::value>),
                       dim3((unsigned)((tokens + (int64_t)rows - 1) / rows), (unsigned)pool.kv_heads * 2), dim3(kThreads), 0,
                       stream, k, k_token, k_head, v, v_token, v_head, tokens, cu, pool);
  });
  return hipGetLastError();
}

hipError_t launch_kv4_read(uint16_t *k, int64_t k_token, int64_t k_head, uint16_t *v, int64_t v_token, int64_t v_head,
                           int tokens, bool f16, int dim, const int *cu, const Kv4Pool &pool, hipStream_t stream) {
  const int rows = dim == 128 ? kReadRows<128> : kReadRows<64>;
  by_type(f16, dim, [&](auto type, auto d) {
    hipLaunchKernelGGL((kv4_read_kernel<decltype(type)::value, decltype(d)::value>),
                       dim3((unsigned)((tokens + (int64_t)rows - 1) / rows), (unsigned)pool.kv_heads * 2), dim3(kThreads), 0,
                       stream, k, k_token, k_head, v, v_token, v_head, tokens, cu, pool);
  });
  return hipGetLastError();
}

hipError_t launch_kv4_append_rope(Kv4Rope a, bool interleaved, bool f16, int dim, const Kv4Pool &pool, int cus, hipStream_t stream) {
  const int heads = a.heads + 2 * pool.kv_heads, rows = kThreads / (dim / 8);
  const int64_t blocks = (a.tokens + (int64_t)rows - 1) / rows;
  // Heads of a workgroup, which loads their angles once: as many as leave eight workgroups a CU, up to 16 in even shares. For 21,447
  // tokens of 56 heads: 432 us with one, 165 with 4, 141 with 8, 137 with 14.
  const int64_t full = blocks * heads / (8 * cus), most = full < 1 ? 1 : full > 16 ? 16 : full, shares = (heads + most - 1) / most;
  a.per = (int)((heads + shares - 1) / shares);
  a.wide = a.cos_row % 4 == 0 && a.sin_row % 4 == 0 && ((uintptr_t)a.cos | (uintptr_t)a.sin) % 16 == 0;
  by_type(f16, dim, [&](auto type, auto d) {
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)((heads + a.per - 1) / a.per)), dim3(kThreads), 0, stream, a, pool);
    };
    constexpr bool kF16 = decltype(type)::value;
    constexpr int kDim = decltype(d)::value;
    if (interleaved) launch(kv4_append_rope_kernel<kF16, kDim, true>);
    else launch(kv4_append_rope_kernel<kF16, kDim, false>);
  });
  return hipGetLastError();
}

hipError_t launch_kv4_keep_path(const Kv4Pool &pool, int dim, int layers, int64_t layer_bytes, const int *cu, int tokens,
                                const int *path, const int *accepted, int *lengths_out, int cus, hipStream_t stream) {
  // Layers of a wave: as many as leave four workgroups a CU. 32 sequences of up to 26 rows, 16 heads and halves, 64 layers: 8.3 us with
  // 8 layers (14.4 with one, 10.8 with 2, 9.4 with 4, 11.0 with 16).
  const int64_t quads = (2 * pool.kv_heads + kKeepWaves - 1) / kKeepWaves, most = (int64_t)pool.sequences * quads * layers / (4 * cus);
  const int per = (int)(most < 1 ? 1 : most > layers ? layers : most);
  const dim3 grid((unsigned)pool.sequences, (unsigned)quads, (unsigned)((layers + per - 1) / per));
  if (dim == 128) hipLaunchKernelGGL(kv4_keep_path_kernel<128>, grid, dim3(64 * kKeepWaves), 0, stream, pool, layers, per, layer_bytes, cu,
                                     tokens, path, accepted, lengths_out);
  else hipLaunchKernelGGL(kv4_keep_path_kernel<64>, grid, dim3(64 * kKeepWaves), 0, stream, pool, layers, per, layer_bytes, cu, tokens, path,
                                     accepted, lengths_out);
  return hipGetLastError();
}

hipError_t launch_kv4_copy_pages(uint8_t *pool, int layers, int64_t layer_bytes, int64_t page_bytes, const int64_t *src,
                                 const int64_t *dst, int64_t count, hipStream_t stream) {
  const unsigned parts = (unsigned)((page_bytes / 16 + kThreads * kCopyLoads - 1) / (kThreads * kCopyLoads));
  for (int64_t first = 0; first < count; first += kKv4Pairs) {
    Kv4Pairs pairs;
    const int n = (int)(count - first < kKv4Pairs ? count - first : kKv4Pairs);
    for (int i = 0; i < n; ++i) {
      pairs.src[i] = (uint32_t)src[first + i];
      pairs.dst[i] = (uint32_t)dst[first + i];
    }
    hipLaunchKernelGGL(kv4_copy_kernel, dim3(parts, (unsigned)n, (unsigned)layers), dim3(kThreads), 0, stream, pool, layer_bytes,
                       page_bytes, pairs);
    const hipError_t error = hipGetLastError();
    if (error != hipSuccess) return error;
  }
  return hipSuccess;
}

}  // namespace tx
