// Attention of drafted rows over a paged 4-bit KV cache (gfx950; layout in kv4.h), grouped heads.
//
// No reference counterpart: the reference decodes one token at a time.
//
//   out[i][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[i][h] . k_j - max),  j over the positions that row i sees:
// of a sequence's `length` positions the last `rows` are its drafted rows; row i sees every position before them (the context)
// and the rows that its parents lead to, itself included.
//
// A KV head's queries are columns, row by row and query head by query head: rows * group of them, in blocks of 32, up to four blocks
// a pass. Work: a part is one (sequence, KV head, pass); a tile is kTile positions of it, and weighs as many ticks as its blocks take
// time. A part of about as many ticks as an even share of the grid, or fewer, is one workgroup's, which writes its output; a longer
// one is cut into even pieces, a workgroup each, that leave (max, sum, unnormalised output) for the combine kernel. Every workgroup
// finds its piece from the lengths itself, so that a captured call serves any; pieces of cut parts come first in the grid, and parts
// of a sequence are cut alike.
//
// A workgroup converts a tile's codes once, into LDS, each thread a scale group of keys and one of values: the conversion is what
// single tokens' attention spends most on, and what the columns share. A wave then has one column block and, where there are
// fewer blocks than waves, a share of the positions:
//   * S^T = K q^T (v_mfma_f32_32x32x16: A = 32 keys, B = the block's queries, held in registers): a lane holds 16 scores of one
//     query, the maximum is in-lane but for one lane swap, and the probabilities, rounded to 16 bits in place, are the B operand of
//     O^T = V^T P^T, whose A operand the transposing LDS reads give;
//   * a query's running maximum follows its scores only where they pass it by 2^4: rescaling is 64 multiplications;
//   * the next tile's codes are under way while this one is multiplied, from pages whose ids are scalar loads a tile earlier.
// Positions past the length, and those of pages outside the pool, become zeros before they are converted and their scores
// -infinity. A draft's values that are not finite become zeros too and are added, for the rows that see them, at the end: zero
// probabilities of the others would make them NaN.
// Statistics and sums in fp32; sums run over the probabilities as rounded. In fp16 they are held times 2^11, in bf16 times a power
// of two below 1 / (2^4 length), so that sums of the largest values stay finite.
//
// Bound by instruction issue where contexts are long: 80 columns over 262,144 positions of 8 heads of 128 take 150 us and 9 to combine
// (1.9 TB/s of codes, 560 TFLOP/s), a tile as long as the two 32-position steps of its busiest wave: scores, maximum, exponentials and
// value products one behind the other, beside one wave of another workgroup. Short contexts are
// a chain of dependent steps: 24 trees of 130 columns over up to 8,191 positions 30 us and 13, of which 5 find the place, 6 fetch and
// convert the first tile and 1 to 2 are each tile behind.
// Columns in units of 16 (v_mfma_f32_16x16x32), each wave converting for itself, took 145 us for the one and 54 for the other;
// 64 positions a step with joined maxima (spills) 174 and 34; one buffer, two barriers a tile 174 and 28.

#include <math.h>

#include <type_traits>

#include "elementwise.h"
#include "kernels.h"
#include "kv4.h"
#include "ragged.h"

namespace tx {

namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kCols = 32;      // columns of a block
constexpr int kPass = kWaves;  // blocks of a pass

// Positions of a tile: a thread converts one group of 32 elements of its keys and one of its values.
template <int DIM>
constexpr int kTile = kThreads / (DIM / 32);
// Workgroups that a CU holds. Three of head dimension 128 have 168 registers a thread and spill 37: 173 us instead of 175 for 80
// columns and 262,144 positions, but 35 instead of 28 for 24 trees, whose runs are short.
template <int DIM>
constexpr int kResident = 2;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <bool F16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The two values rounded to 16 bits, packed, and the sum of what they were rounded to.
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

// Over the two lanes that hold one query (lane, + 32).
__device__ __forceinline__ float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// All of the workgroup's LDS accesses so far are done; loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Ticks: what starting and ending a piece costs, and a tile of up to two blocks, whose waves share its positions, or more.
constexpr int kStart = 6, kMostWeight = 3;
constexpr int kLeast = 3;  // of a share: a tile a piece, 9.4 us for one tree behind 700 positions, where a share of 6 takes 11.0 and of 9 12.0
__device__ __forceinline__ int weight_of(int blocks) { return blocks <= 2 ? 2 : kMostWeight; }

// A value that all lanes have, in a scalar register.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A sequence as the grid sees it.
struct Drafts {
  int begin, rows;  // its first row, and how many: at most kMostDrafts
  int length, context;
  int columns, passes, blocks;  // column blocks of every pass but the last, which may have fewer
};
__host__ __device__ __forceinline__ int pieces_of(int count, int most) { return (count + most - 1) / most; }
__device__ __forceinline__ Drafts drafts_of(const Kv4Tree &a, int first, int end, int length) {
  Drafts d;
  first = min(max(first, 0), a.tokens);
  end = min(max(end, first), a.tokens);
  d.begin = first;
  d.length = length;
  d.context = length - (end - first);
  d.rows = min(end - first, kMostDrafts);
  d.columns = d.rows * a.group;
  const int blocks = pieces_of(d.columns, kCols);
  d.passes = pieces_of(blocks, kPass);
  d.blocks = d.passes <= 1 ? blocks : pieces_of(blocks, d.passes);
  return d;
}
// Of a sequence that all lanes ask for, in scalar registers: page ids then stay scalar.
__device__ __forceinline__ Drafts scalar_drafts(const Kv4Tree &a, int sequence) {
  return drafts_of(a, scalar(a.cu[sequence]), scalar(a.cu[sequence + 1]), scalar(kv4_length(a.pool, sequence)));
}

template <int TILE>
__device__ __forceinline__ int tiles_of(int length) { return max(1, (length + TILE - 1) / TILE); }
// Ticks of a part, the start among them, in units of 2^shift: passes count alike, whatever their blocks.
template <int TILE>
__device__ __forceinline__ int part_ticks(const Kv4Tree &a, const Drafts &d) {
  return ((kStart + weight_of(d.blocks) * tiles_of<TILE>(d.length)) >> a.shift) + (a.shift > 0);
}

// How the parts are cut: into as many pieces as they have even shares of the grid, rounded; the pieces of cut parts are at most
// four thirds of the grid's even shares.
struct Cut {
  Drafts d;  // in scalar registers
  int sequence, part, piece, pieces;  // part: head * passes + pass
  int before;                         // pieces of cut parts before this part
};
// Piece `wanted` of all (`wanted` >= 0), or with wanted = ~sequence the first piece of that sequence. sequence < 0: there is none.
template <int TILE>
__device__ __forceinline__ Cut cut_at(const Kv4Tree &a, int wanted) {
  const int lane = threadIdx.x & 63, sequences = a.pool.sequences;
  int parts = 0, ticks = 0, tiles = 0, begin = 0, end = 0, length = 0;  // of the lane's sequence
  auto load = [&](int first) {
    parts = ticks = tiles = 0;
    if (first + lane < sequences) {
      begin = a.cu[first + lane];
      end = a.cu[first + lane + 1];
      length = kv4_length(a.pool, first + lane);
      const Drafts d = drafts_of(a, begin, end, length);
      parts = a.pool.kv_heads * d.passes;
      tiles = tiles_of<TILE>(d.length);
      ticks = part_ticks<TILE>(a, d);
    }
  };
  int total = 0;
  for (int first = 0; first < sequences; first += 64) {
    load(first);
    total += __builtin_amdgcn_readlane(wave_scan(parts * ticks), 63);
  }
  const int share = max((total + a.workgroups - 1) / a.workgroups, max(kLeast >> a.shift, 1));
  auto pieces_now = [&] { return max(min((int)((2u * ticks + share) / (2u * share)), tiles), 1); };
  int before = 0;
#pragma unroll 1
  for (int cut = 1; cut >= 0; --cut) {  // the cut parts, then the others
    for (int first = 0; first < sequences; first += 64) {
      if (sequences > 64) load(first);
      const int pieces = pieces_now(), n = (pieces > 1) == (cut != 0) ? pieces * parts : 0, sum = wave_scan(n);
      uint64_t past;
      if (wanted >= 0)
        past = __builtin_amdgcn_ballot_w64(before + sum > wanted);
      else
        past = __builtin_amdgcn_ballot_w64(first + lane == ~wanted);
      if (past) {
        const int at = __builtin_ctzll(past), each = __builtin_amdgcn_readlane(pieces, at);
        const int start = before + __builtin_amdgcn_readlane(sum - n, at), local = scalar(max(wanted, start)) - start;
        const int part = scalar(local / each);
        const Drafts d = drafts_of(a, __builtin_amdgcn_readlane(begin, at), __builtin_amdgcn_readlane(end, at), __builtin_amdgcn_readlane(length, at));
        return {d, first + at, part, local - part * each, each, start + part * each};
      }
      before += __builtin_amdgcn_readlane(sum, 63);
    }
  }
  return {{}, -1, 0, 0, 1, 0};
}

// The row of a column, and its query head in the KV head's group: column / a.group by the host's ceil(2^32 / group), exact for
// columns times group below 2^32.
struct Query {
  int row, head;
};
__device__ __forceinline__ Query query_of(const Kv4Tree &a, int column) {
  const int row = a.group == 1 ? column : (int)__umulhi((uint32_t)column, a.group_inverse);
  return {row, column - row * a.group};
}

__device__ __forceinline__ int parent_of(const Kv4Tree &a, const Drafts &d, int row) {
  const int parent = a.parents ? a.parents[d.begin + row] : row - 1;
  return (uint32_t)parent < (uint32_t)d.rows ? parent : -1;
}

// A query's sum where all its scores are -infinity: above zero, so that it is told from a query without a position, whose outputs are
// zeros; next to any other share's sum it is nothing.
constexpr float kNoScore = 1e-30f;
__device__ __forceinline__ float inverse_of(float top, float sum) {
  return top == -INFINITY ? (sum == 0.f ? 0.f : NAN) : 1.f / sum;
}

// Whether a word of two 16-bit values holds an infinity or a NaN.
template <bool F16>
__device__ __forceinline__ bool not_finite(uint32_t word) {
  constexpr uint32_t kExponent = F16 ? 0x7C00u : 0x7F80u;
  return (word & kExponent) == kExponent || (word >> 16 & kExponent) == kExponent;
}

// Elements e and e + 1 of a cached row in the rows' type: `half` its head's keys or values in its page, `at` its place there.
template <bool F16, int DIM>
__device__ __forceinline__ uint32_t cached_pair(const uint8_t *half, int64_t scales_at, int at, int e) {
  return kv4_pair<F16, 0>(half[at * (DIM / 2) + e / 2], __uint_as_float((uint32_t)half[scales_at + at * (DIM / 32) + e / 32] << 23));
}
// A query's score of a cached key, before the scale.
template <bool F16, int DIM>
__device__ __forceinline__ float cached_score(const Kv4Tree &a, const uint16_t *q, const uint8_t *half, int64_t scales_at, int at) {
  float score = 0.f;
#pragma unroll 1
  for (int e = 0; e < DIM; e += 2) {
    const uint32_t k = cached_pair<F16, DIM>(half, scales_at, at, e), x = (*reinterpret_cast<const uint32_t *>(q + e) & a.q_and) ^ a.q_xor;
    score = __builtin_fmaf(half_bits_to_float<F16>((uint16_t)x), half_bits_to_float<F16>((uint16_t)k), score);
    score = __builtin_fmaf(half_bits_to_float<F16>((uint16_t)(x >> 16)), half_bits_to_float<F16>((uint16_t)(k >> 16)), score);
  }
  return score;
}

// Of a block's piece: its outputs in the order of the registers, [DIM / 8][64 lanes][4], then the columns' maxima and sums.
template <int DIM>
constexpr int kPieceFloats = kCols * DIM + 2 * kCols;

template <bool F16, int DIM>
__global__ __launch_bounds__(kThreads, kResident<DIM>) void kv4_tree_kernel(Kv4Tree a) {
  constexpr int kTile = tx::kTile<DIM>, kSubs = kTile / 32, kGroups = DIM / 32;
  constexpr int kRow = DIM * 2;  // bytes of a converted row
  constexpr int kSteps = DIM / 16, kOut = DIM / 32;
  __shared__ __attribute__((aligned(1024))) char keys[2][kTile * kRow];
  __shared__ __attribute__((aligned(1024))) char values[2][kTile * kRow];
  __shared__ float stats[kWaves][2][64];
  __shared__ uint64_t sees[kMostDrafts];  // the rows that each row sees, a bit each
  __shared__ uint64_t mads;               // drafted rows of whose values a group was left out
  __shared__ __attribute__((aligned(8))) uint8_t known[2][8];  // whether each 16 positions of the tile lie in the pool

  const Kv4Pool &pool = a.pool;
  const int lane = threadIdx.x & 63;
  const int wave = scalar(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;

  Drafts d;
  int sequence, head, pass, piece = 0, pieces = 1;
  if (a.whole) {  // a workgroup for each part
    pass = blockIdx.x % a.most_passes;
    head = blockIdx.x / a.most_passes % pool.kv_heads;
    sequence = blockIdx.x / a.most_passes / pool.kv_heads;
    d = scalar_drafts(a, sequence);
    if (pass >= d.passes) return;
  } else {
    const Cut cut = cut_at<kTile>(a, blockIdx.x);
    if (cut.sequence < 0) return;
    sequence = cut.sequence;
    d = cut.d;
    head = scalar(cut.part / d.passes);
    pass = cut.part - head * d.passes;
    piece = cut.piece;
    pieces = cut.pieces;
  }
  const int tiles = tiles_of<kTile>(d.length);
  // Products pass 32 bits.
  const int first = (int)((uint64_t)tiles * piece / pieces), until = (int)((uint64_t)tiles * (piece + 1) / pieces);

  // This thread's part of a conversion: position `row` of its wave's kTile / kWaves, elements 32 g .. 32 g + 31.
  const int row = lane / kGroups, g = lane % kGroups;
  const int64_t half_bytes = kv4_half_bytes(pool.page_shift, DIM), scales_at = (int64_t)(DIM / 2) << pool.page_shift;
  const int64_t head_bytes = 2 * half_bytes, page_bytes = head_bytes * pool.kv_heads;
  const int page_mask = (1 << pool.page_shift) - 1;
  // 16-byte chunk c of row r lies at chunk c ^ turn: operand reads and these stores hit distinct banks.
  const int k_turn = DIM == 128 ? row & 15 : (row >> 1) & 7;
  const int v_turn = DIM == 128 ? 5 * (row & 3) : 4 * ((row >> 1) & 1) ^ ((row >> 1) & 3);
  // Operands: key row n, dimensions 16 st + 8 h at k_at ^ 32 st; by the transposing reads key 4 h + (lane % 16) / 4,
  // dimensions 32 t + 16 ((lane / 16) % 2) + 4 (lane % 4) at v_at ^ 64 t.
  const uint32_t k_at = (uint32_t)n * kRow + 16u * (uint32_t)(h ^ (DIM == 128 ? n & 15 : (n >> 1) & 7));
  const uint32_t v_row = 4u * h + ((lane >> 2) & 3), v_chunk = 2u * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_at = v_row * kRow + 8u * (lane & 1) +
                        16u * (v_chunk ^ (DIM == 128 ? 5 * (v_row & 3) : 4 * ((v_row >> 1) & 1) ^ ((v_row >> 1) & 3)));

  const int col0 = pass * d.blocks * kCols;
  const int blocks = min(d.blocks, pieces_of(d.columns - col0, kCols));
  // Waves that share a block's positions: all of them for one block (at dim 128 two), pairs for two. Of three blocks two waves have one
  // each and two share the third.
  const int shares = blocks >= 4 ? 1 : blocks == 3 ? (wave >= 2 ? 2 : 1) : blocks == 2 ? 2 : min(kWaves, kSubs);
  const int block = blocks >= 4 ? wave : blocks == 3 ? min(wave, 2) : blocks == 2 ? wave & 1 : 0;
  const int share = blocks >= 4 ? 0 : blocks == 3 ? (wave == 3 ? 1 : 0) : blocks == 2 ? wave >> 1 : wave;
  const bool works = block < blocks && share < shares;
  const int stop = min(until * kTile, d.length);

  // Quarters of a tile that this wave converts: its own; where two waves have less to multiply, or nothing, they convert for all. 80
  // columns and 262,144 positions 150 us (165 where all convert), 32 columns and 100,000 positions of 2 heads 17.1 (19.2), of 16 heads
  // in 8 sequences of up to as many 18.7 (21.6).
  const bool apart = blocks == 3 || (blocks == 1 && kSubs < kWaves);
  const int quarters = !apart ? 1 : wave >= 2 ? 2 : 0, quarter = !apart ? wave : 2 * (wave & 1);
  // Page ids of a quarter's positions (at dim 64 twice 16 of them), a tile before its codes.
  constexpr int kIds = kTile / kWaves / 16;
  struct Ids {
    int page[kIds];
  };
  auto ids_of = [&](int tile, int k) __attribute__((always_inline)) {
    // Constant for the whole launch: scalar loads.
    const auto *table = (const __attribute__((address_space(4))) int *)(pool.table + sequence * pool.table_stride);
    Ids ids;
#pragma unroll
    for (int i = 0; i < kIds; ++i)
      ids.page[i] = table[min(tile * kTile + (quarter + k) * (kTile / kWaves) + 16 * i, max(d.length - 1, 0)) >> pool.page_shift];
    return ids;
  };
  struct Codes {
    u32x4 k, v;
    uint32_t k_scale, v_scale;
    int there;  // whether the position's page is known
  };
  auto codes_of = [&](int tile, int k, const Ids &ids) __attribute__((always_inline)) {
    const int position = tile * kTile + (quarter + k) * (kTile / kWaves) + row, at = position & page_mask;
    const uint8_t *half[kIds];
    int known_page[kIds];
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      known_page[i] = (uint32_t)ids.page[i] < (uint64_t)pool.num_pages;
      half[i] = pool.pages + (known_page[i] ? ids.page[i] : 0) * page_bytes + head * head_bytes;
    }
    const bool second = kIds == 2 && lane >= 32;
    const uint8_t *mine = second ? half[kIds - 1] : half[0];
    Codes c;
    c.there = second ? known_page[kIds - 1] : known_page[0];
    c.k = *reinterpret_cast<const u32x4 *>(mine + at * (DIM / 2) + 16 * g);
    c.v = *reinterpret_cast<const u32x4 *>(mine + half_bytes + at * (DIM / 2) + 16 * g);
    c.k_scale = mine[scales_at + at * kGroups + g];
    c.v_scale = mine[half_bytes + scales_at + at * kGroups + g];
    return c;
  };
  Codes codes[2] = {};
  Ids ids[2] = {};
  // The codes of `tile`, whose ids are here, and the ids of the one behind.
  auto load = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (k < quarters) {
        codes[k] = codes_of(tile, k, ids[k]);
        ids[k] = ids_of(tile + 1, k);
      }
  };
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (k < quarters) ids[k] = ids_of(first, k);
  load(first);

  const int column = col0 + block * kCols + n;  // this lane's query
  const Query query = query_of(a, min(column, d.columns - 1));
  u32x4 qb[kSteps];
  {
    const uint16_t *q = a.q + (int64_t)(d.begin + query.row) * a.q_token + (head * a.group + query.head) * a.q_head + 8 * h;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      qb[st] = *reinterpret_cast<const u32x4 *>(q + 16 * st);
#pragma unroll
      for (int j = 0; j < 4; ++j) qb[st][j] = (qb[st][j] & a.q_and) ^ a.q_xor;
    }
  }
  if (wave == 0 && until * kTile > d.context) {
    uint64_t seen = ((uint64_t)2 << lane) - 1;
    if (a.parents) {  // pointers doubled, so that any parents end
      int up = lane < d.rows ? parent_of(a, d, lane) : -1;
      seen = (uint64_t)1 << lane;
#pragma unroll 1
      for (int i = 0; i < 6; ++i) {
        const int from_lane = max(up, 0);
        const uint64_t theirs = __shfl(seen, from_lane);
        const int further = __shfl(up, from_lane);
        seen |= up >= 0 ? theirs : 0;
        up = up >= 0 ? further : -1;
      }
    }
    sees[lane] = seen;  // the others read it behind a barrier
  }
  if (threadIdx.x == 0) mads = 0;
  const float lift = F16 ? 15.f - kPackedLag : -kPackedLag - 1.f - (float)(32 - __builtin_clz(d.length | 1));
  float m = -INFINITY, l = 0.f;  // running maximum of the query (before the scale), this lane's share of the sum
  bool any = false;              // whether the query sees a position of this wave's
  f32x16 o[kOut];                // o[t][r] = O[query][dimension 32 t + 8 (r / 4) + 4 h + r % 4]
#pragma unroll
  for (int t = 0; t < kOut; ++t) o[t] = f32x16{};

  // The codes in registers, converted into the buffers of their tile.
  auto convert_one = [&](int tile, int k, Codes c) __attribute__((always_inline)) {
    const int p = (quarter + k) * (kTile / kWaves) + row, position = tile * kTile + p;
    char *const kb = keys[tile & 1] + p * kRow, *const vb = values[tile & 1] + p * kRow;
    const bool counts = c.there && position < d.length;
    if (tile * kTile + kTile > min(d.context, d.length)) {
      asm volatile("" ::: "memory");  // stays a branch: the last tiles of a sequence
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 x = kv4_octet<F16>(c.v[i], __uint_as_float(c.v_scale << 23));
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= not_finite<F16>(x[j]);
      }
      odd = odd && counts && position >= d.context;
      const int draft = position - d.context;
      if (odd && draft < kMostDrafts) atomicOr((unsigned long long *)&mads, 1ull << draft);
      c.v_scale = odd ? 127u : c.v_scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) c.v[i] = odd ? 0u : c.v[i];
    }
    const uint32_t ks = counts ? c.k_scale : 127u, vs = counts ? c.v_scale : 127u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t kc = counts ? c.k[i] : 0u, vc = counts ? c.v[i] : 0u;
      *reinterpret_cast<u32x4 *>(kb + 16 * ((4 * g + i) ^ k_turn)) = kv4_octet<F16>(kc, __uint_as_float(ks << 23));
      *reinterpret_cast<u32x4 *>(vb + 16 * ((4 * g + i) ^ v_turn)) = kv4_octet<F16>(vc, __uint_as_float(vs << 23));
    }
    if (g == 0 && p % 16 == 0) known[tile & 1][p / 16] = (uint8_t)c.there;
  };
  auto convert = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (k < quarters) convert_one(tile, k, codes[k]);
  };
  lds_barrier();  // `mads` is clear
  convert(first);
  if (first + 1 < until) load(first + 1);

#pragma unroll 1
  for (int tile = first; tile < until; ++tile) {
    const int base0 = tile * kTile;
    lds_barrier();  // this tile is converted, the last one read
    if (tile + 1 < until) {
      convert(tile + 1);
      if (tile + 2 < until) load(tile + 2);
    }
    if (!works) continue;
#pragma unroll 1
    for (int sub = share; sub < kSubs; sub += shares) {
      const int base = base0 + 32 * sub;
      if (base >= stop) break;
      const char *kt = keys[tile & 1] + 32 * sub * kRow, *vt = values[tile & 1] + 32 * sub * kRow;
      const uint32_t pages = *reinterpret_cast<const uint16_t *>(known[tile & 1] + 2 * sub);
      f32x16 sc;
      {
        constexpr int kAhead = kSteps < 4 ? kSteps : 4;
        auto key = [&](int st) __attribute__((always_inline)) { return *reinterpret_cast<const u32x4 *>(kt + (k_at ^ (32u * st))); };
        u32x4 x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) x[i] = key(i);
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          sc = mfma32<F16>(x[st % kAhead], qb[st], st == 0 ? f32x16{} : sc);
          if (st + kAhead < kSteps) x[st % kAhead] = key(st + kAhead);
        }
      }
      // sc[r]: position base + 8 (r / 4) + 4 h + r % 4
      if (scalar(pages) != 0x0101 || base + 32 > min(stop, d.context)) {
        asm volatile("" ::: "memory");
        uint32_t bits = (pages & 1 ? 0xFFFFu : 0u) | (pages >> 8 ? 0xFFFF0000u : 0u);
        if (stop - base < 32) bits &= (1u << (stop - base)) - 1u;
        const int ahead = d.context - base;  // where the first drafted row lies, counted from the base
        if (ahead < 32) {
          const uint64_t rows = sees[query.row];
          bits &= ahead >= 0 ? (uint32_t)(rows << ahead) | ((1u << ahead) - 1u) : ahead > -64 ? (uint32_t)(rows >> -ahead) : 0u;
        }
        any |= bits != 0;
        bits >>= 4 * h;
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = bits >> (8 * (r >> 2) + (r & 3)) & 1 ? sc[r] : -INFINITY;
      } else {
        any = true;
      }
      float mx = fmaxf(sc[0], sc[1]);
#pragma unroll
      for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, sc[r]), sc[r + 1]);
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
      const float zero = m == -INFINITY ? 0.f : lift - m * a.sl2;  // no position yet: every score is -infinity
      uint32_t pb[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        pb[i] = pack2<F16>(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * i], a.sl2, zero)),
                           __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * i + 1], a.sl2, zero)), l);
      {
        constexpr int kAhead = 3;
        auto value = [&](int i) __attribute__((always_inline)) {
          const char *at = vt + 16 * (i / kOut) * kRow + (v_at ^ (64u * (i % kOut)));
          const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at));
          const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(at + 8 * kRow)));
          return u32x4{lo[0], lo[1], hi[0], hi[1]};  // slots 0-3: positions 4 h .., 4-7: the 8 behind
        };
        u32x4 x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) x[i] = value(i);
#pragma unroll
        for (int i = 0; i < 2 * kOut; ++i) {
          const int j = i / kOut, t = i % kOut;
          o[t] = mfma32<F16>(x[i % kAhead], u32x4{pb[4 * j], pb[4 * j + 1], pb[4 * j + 2], pb[4 * j + 3]}, o[t]);
          if (i + kAhead < 2 * kOut) x[i % kAhead] = value(i + kAhead);
        }
      }
    }
  }

  // The shares of a block meet in LDS, in the tiles' place. A share without a score above -infinity has l = 0 and O = 0 (or NaN,
  // where scores were).
  l = halves_sum(l);
  if (m == -INFINITY && any) l += kNoScore;
  lds_barrier();  // the last tile is read
  const uint64_t lost = mads;
  if (blocks < 4) {
    // Share s of a block: 4 KiB for each 32 dimensions, of which the keys' place has 8.
    auto region = [&](int s) { return reinterpret_cast<f32x4 *>(keys[0] + (blocks == 3 ? 0 : (s - 1) * blocks + block) * kOut * 4096) + lane; };
    if (works && share > 0) {
      stats[wave][0][lane] = m;
      stats[wave][1][lane] = l;
      f32x4 *put = region(share);
#pragma unroll
      for (int t = 0; t < kOut; ++t)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) put[64 * (4 * t + rq)] = f32x4{o[t][4 * rq], o[t][4 * rq + 1], o[t][4 * rq + 2], o[t][4 * rq + 3]};
    }
    lds_barrier();
    if (works && share == 0) {
#pragma unroll 1
      for (int s = 1; s < shares; ++s) {
        const int theirs = blocks == 3 ? 3 : blocks == 2 ? 2 * s + block : s;
        const float m2 = stats[theirs][0][lane], l2 = stats[theirs][1][lane], top = fmaxf(m, m2);
        const float w1 = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - top) * a.sl2);
        const float w2 = m2 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m2 - top) * a.sl2);
        const f32x4 *from_share = region(s);
#pragma unroll
        for (int t = 0; t < kOut; ++t)
#pragma unroll
          for (int rq = 0; rq < 4; ++rq) {
            const f32x4 x = from_share[64 * (4 * t + rq)];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][4 * rq + r] = o[t][4 * rq + r] * w1 + x[r] * w2;
          }
        l = l * w1 + l2 * w2;
        m = top;
      }
    }
  }
  if (works && share == 0) {
    // Groups of value rows that the products left out, for the queries that see them: slow, and seldom.
    uint64_t rows = lost;
#pragma unroll 1
    for (; __builtin_expect(rows != 0, 0); rows &= rows - 1) {
      const int row = __builtin_ctzll(rows), at = (d.context + row) & page_mask;
      const int page = pool.table[sequence * pool.table_stride + ((d.context + row) >> pool.page_shift)];
      const uint8_t *k_half = pool.pages + page * page_bytes + head * head_bytes, *v_half = k_half + half_bytes;
      uint32_t out = 0;  // a bit for each group
#pragma unroll 1
      for (int e = 0; e < DIM; e += 2) out |= (uint32_t)not_finite<F16>(cached_pair<F16, DIM>(v_half, scales_at, at, e)) << (e / 32);
      const uint16_t *q = a.q + (int64_t)(d.begin + query.row) * a.q_token + (head * a.group + query.head) * a.q_head;
      const float prob = __builtin_amdgcn_exp2f((cached_score<F16, DIM>(a, q, k_half, scales_at, at) - m) * a.sl2 + lift);
      const bool does = sees[query.row] >> row & 1;
#pragma unroll
      for (int t = 0; t < kOut; ++t) {
        if (!does || !(out >> t & 1)) continue;
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const uint32_t v = cached_pair<F16, DIM>(v_half, scales_at, at, 32 * t + 8 * (r >> 2) + 4 * h + (r & 3));
          o[t][r] = __builtin_fmaf(prob, half_bits_to_float<F16>((uint16_t)v), o[t][r]);
          o[t][r + 1] = __builtin_fmaf(prob, half_bits_to_float<F16>((uint16_t)(v >> 16)), o[t][r + 1]);
        }
      }
    }
    if (pieces == 1) {
      const float inverse = inverse_of(m, l);
      uint16_t *out = a.out + (int64_t)(d.begin + query.row) * a.out_token + (head * a.group + query.head) * a.out_head + 4 * h;
      if (column < d.columns) {
#pragma unroll
        for (int t = 0; t < kOut; ++t)
#pragma unroll
          for (int rq = 0; rq < 4; ++rq) {
            const f32x4 v = f32x4{o[t][4 * rq], o[t][4 * rq + 1], o[t][4 * rq + 2], o[t][4 * rq + 3]} * inverse;
            *reinterpret_cast<u32x2 *>(out + 32 * t + 8 * rq) =
                u32x2{to_half_bits<F16>(v[0]) | (uint32_t)to_half_bits<F16>(v[1]) << 16,
                      to_half_bits<F16>(v[2]) | (uint32_t)to_half_bits<F16>(v[3]) << 16};
          }
      }
    } else {
      float *piece = a.pieces + (int64_t)blockIdx.x * a.piece_floats + block * kPieceFloats<DIM>;
#pragma unroll
      for (int t = 0; t < kOut; ++t)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq)
          reinterpret_cast<f32x4 *>(piece)[64 * (4 * t + rq) + lane] = f32x4{o[t][4 * rq], o[t][4 * rq + 1], o[t][4 * rq + 2], o[t][4 * rq + 3]};
      if (h == 0) {
        piece[kCols * DIM + n] = m;
        piece[kCols * DIM + kCols + n] = l;
      }
    }
  }
}

// Joins the pieces of the parts that were cut. Grid: x = parts, y = block of the pass. SHARED: z = slices of 1 KiB of a block's
// outputs, of which the waves each take every fourth piece; else each wave has a quarter of the slices.
template <bool F16, int DIM, bool SHARED>
__global__ __launch_bounds__(kThreads) void kv4_tree_combine_kernel(Kv4Tree a) {
  constexpr int kTile = tx::kTile<DIM>, kHeld = 4, kStride = SHARED ? kWaves : 1, kSlices = SHARED ? 1 : DIM / 8 / kWaves;
  __shared__ f32x4 sums[SHARED ? kWaves : 1][64];
  __shared__ float stats[SHARED ? kWaves : 1][2][64];
  const Kv4Pool &pool = a.pool;
  const int lane = threadIdx.x & 63, wave = scalar(threadIdx.x >> 6);
  const int pass = blockIdx.x % a.most_passes, head = blockIdx.x / a.most_passes % pool.kv_heads;
  const int sequence = blockIdx.x / a.most_passes / pool.kv_heads, block = blockIdx.y;
  const Cut cut = cut_at<kTile>(a, ~sequence);
  const Drafts &d = cut.d;
  const int col0 = (pass * d.blocks + block) * kCols;
  if (pass >= d.passes || block >= d.blocks || col0 >= d.columns) return;
  const int w1 = cut.pieces - 1, slice0 = SHARED ? blockIdx.z : wave * kSlices;
  if (w1 == 0) return;  // one workgroup had it all and wrote the output
  const float *pieces = a.pieces + (int64_t)(cut.before + (head * d.passes + pass) * cut.pieces) * a.piece_floats + block * kPieceFloats<DIM>;
  const int n = lane & 31, column = col0 + n;
  const Query query = query_of(a, min(column, d.columns - 1));
  auto put = [&](int slice, f32x4 sum, float top, float ll) __attribute__((always_inline)) {
    sum *= inverse_of(top, ll);
    if (column < d.columns)
      *reinterpret_cast<u32x2 *>(a.out + (int64_t)(d.begin + query.row) * a.out_token + (head * a.group + query.head) * a.out_head +
                                 8 * slice + 4 * (lane >> 5)) =
          u32x2{to_half_bits<F16>(sum[0]) | (uint32_t)to_half_bits<F16>(sum[1]) << 16,
                to_half_bits<F16>(sum[2]) | (uint32_t)to_half_bits<F16>(sum[3]) << 16};
  };
  f32x4 sum[kSlices] = {};
  float l = 0.f, m = -INFINITY;
  for (int w = SHARED ? wave : 0; w <= w1; w += kStride * kHeld) {
    f32x4 value[kHeld][kSlices];
    float pm[kHeld], pl[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const float *at = pieces + (int64_t)min(w + i * kStride, w1) * a.piece_floats;
      pm[i] = at[kCols * DIM + n];
      pl[i] = at[kCols * DIM + kCols + n];
#pragma unroll
      for (int j = 0; j < kSlices; ++j) value[i][j] = *reinterpret_cast<const f32x4 *>(at + 256 * (slice0 + j) + 4 * lane);
    }
    float mnew = m;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) mnew = w + i * kStride <= w1 ? fmaxf(mnew, pm[i]) : mnew;
    const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mnew) * a.sl2);
#pragma unroll
    for (int j = 0; j < kSlices; ++j) sum[j] *= alpha;
    l *= alpha;
    m = mnew;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (w + i * kStride > w1) continue;
      const float weight = pm[i] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((pm[i] - m) * a.sl2);  // an empty piece holds zeros (or NaN)
#pragma unroll
      for (int j = 0; j < kSlices; ++j) sum[j] += value[i][j] * weight;
      l += pl[i] * weight;
    }
  }
  if constexpr (!SHARED) {
#pragma unroll
    for (int j = 0; j < kSlices; ++j) put(slice0 + j, sum[j], m, l);
  } else {
    sums[wave][lane] = sum[0];
    stats[wave][0][lane] = m;
    stats[wave][1][lane] = l;
    __syncthreads();
    if (wave != 0) return;
    float top = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][0][lane]);
    f32x4 total = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float weight = stats[w][0][lane] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((stats[w][0][lane] - top) * a.sl2);
      total += sums[w][lane] * weight;
      ll += stats[w][1][lane] * weight;
    }
    put(slice0, total, top, ll);
  }
}

// Upper bounds of a call from what the host knows.
int64_t most_blocks(const Kv4Tree &a) { return ((int64_t)(a.tokens < kMostDrafts ? a.tokens : kMostDrafts) * a.group + kCols - 1) / kCols; }
int64_t most_passes(const Kv4Tree &a) { return (most_blocks(a) + kPass - 1) / kPass; }
int64_t most_parts(const Kv4Tree &a) { return (int64_t)a.pool.sequences * a.pool.kv_heads * most_passes(a); }
int64_t most_ticks(const Kv4Tree &a, int tile) {
  const int64_t room = (int64_t)a.pool.max_pages << a.pool.page_shift, tiles = (room + tile - 1) / tile;
  return most_parts(a) * (kStart + kMostWeight * tiles);
}

}  // namespace

// What single tokens' attention takes; a launch has fewer than 2^32 threads, 256 for each (head, pass).
bool kv4_tree_fits(const Kv4Tree &a) { return kv4_attention_fits(a.pool) && most_parts(a) < (int64_t)1 << 23; }

void kv4_tree_plan(Kv4Tree &a, int dim, int cus) {
  const int64_t room = (int64_t)a.pool.max_pages << a.pool.page_shift;
  a.most_passes = (int)most_passes(a);
  // Ticks are 32-bit: where tables have room for more of them than 2^30 (64 rows a sequence, all as long as the table), in coarser units, so
  // that their sum holds whatever cu and the lengths are. Cuts are then as fine as 2^-30 of that most.
  a.shift = 0;
  while (most_ticks(a, dim == 128 ? kTile<128> : kTile<64>) >> a.shift > (int64_t)1 << 30) ++a.shift;
  const int64_t shares = most_ticks(a, dim == 128 ? kTile<128> : kTile<64>) / kLeast + 1;
  const int64_t fill = (dim == 128 ? kResident<128> : kResident<64>) * (int64_t)cus;
  // Where tables hold at most 512 positions and the parts, were all sequences as wide as they may be, fill the grid, none is cut. That
  // many are seldom there, but a second launch costs more than uneven workgroups: up to 400 positions, 8 heads of 16 * 5
  // rows, 32 sequences take 20.6 us, cut and combined 27.5; up to 512, 64 of 6 rows and 16/2 heads 21.5 and 23.6, 90 of 4 rows
  // and 12/1 heads 16.6 and 23.5. Others lose: 26 of 3 rows and 40/1 heads 20.9 and 19.7; where half the workgroups have no part
  // (64 of 5 rows and 32/8 heads) 31.5 and 24.3. Below the bound 1 sequence of 16 * 5 rows takes 15.7 whole and 12.9 cut, 2 11.0 and
  // 15.3, 4 14.1 and 21.4, 8 17.4 and 18.6. 32 of up to 1,000 positions: 26 and 22.
  a.whole = room <= 512 && most_parts(a) >= fill;
  a.workgroups = (int)(shares < fill ? shares : fill);
  const int64_t blocks = most_blocks(a) < kPass ? most_blocks(a) : kPass;
  a.piece_floats = (int)blocks * (dim == 128 ? kPieceFloats<128> : kPieceFloats<64>);
  // A part is cut where it has one and a half shares: into at most four thirds of them.
  a.piece_bytes = a.whole ? 0 : ((int64_t)a.workgroups * 4 / 3 + 1) * a.piece_floats * (int64_t)sizeof(float);
}

hipError_t launch_kv4_tree(const Kv4Tree &a, bool f16, int dim, hipStream_t stream) {
  auto launch = [&](auto type, auto dims) {
    constexpr bool kF16 = decltype(type)::value;
    constexpr int kDim = decltype(dims)::value;
    const int64_t parts = most_parts(a);
    const unsigned in_pass = (unsigned)(most_blocks(a) < kPass ? most_blocks(a) : kPass);
    hipLaunchKernelGGL((kv4_tree_kernel<kF16, kDim>), dim3((unsigned)(parts + (a.whole ? 0 : a.workgroups))), dim3(kThreads), 0, stream, a);
    if (a.whole) return;
    // Few parts have many pieces. 24 parts: 8.7 us shared, 21 not; 96: 11.6 and 14.3; 192: 13.0 and 7.5; 576: 35 and 14.
    if (parts <= 128)
      hipLaunchKernelGGL((kv4_tree_combine_kernel<kF16, kDim, true>), dim3((unsigned)parts, in_pass, kDim / 8), dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((kv4_tree_combine_kernel<kF16, kDim, false>), dim3((unsigned)parts, in_pass), dim3(kThreads), 0, stream, a);
  };
  using std::integral_constant;
  if (f16 && dim == 128) launch(integral_constant<bool, true>{}, integral_constant<int, 128>{});
  else if (f16) launch(integral_constant<bool, true>{}, integral_constant<int, 64>{});
  else if (dim == 128) launch(integral_constant<bool, false>{}, integral_constant<int, 128>{});
  else launch(integral_constant<bool, false>{}, integral_constant<int, 64>{});
  return hipGetLastError();
}

}  // namespace tx
