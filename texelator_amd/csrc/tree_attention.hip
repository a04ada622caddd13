// Attention of drafted rows over a paged 4-bit KV cache (gfx950; layout in kv4.h), grouped heads.
//
// No reference counterpart: the reference decodes one token at a time.
//
//   out[i][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[i][h] . k_j - max),  j over the positions that row i sees:
// of a sequence's `length` positions the last `rows` are its drafted rows; row i sees every position before them (the context)
// and the rows that its parents lead to, itself included.
//
// A KV head's queries are columns, row by row and query head by query head: rows * group of them, in blocks of 32. Work: a unit
// is kTile positions of one sequence, KV head and pass (of up to four column blocks); the units of all lie in one row, and every
// workgroup takes an equal run of them, whatever the lengths (it finds its place from the lengths itself, so that a captured call serves
// any). A run that covers a whole (sequence, head, pass) writes its output; the others leave (max, sum, unnormalised
// output) for the combine kernel, at most two such pieces a workgroup.
//
// A workgroup converts a unit's codes once, into LDS (each thread one scale group of keys and one of values); a wave then has one
// column block and, where there are fewer blocks than waves, a share of the positions:
//   * S^T = K q^T (v_mfma_f32_32x32x16: A = 32 keys, B = the block's queries, held in registers): a lane holds 16 scores of one
//     query, the maximum is in-lane but for one lane swap, and the probabilities, rounded to 16 bits in place, are the B operand of
//     O^T = V^T P^T, whose A operand the transposing LDS reads give;
//   * a query's running maximum follows its scores only where they pass it by 2^4;
//   * the next unit's codes are under way while this one is multiplied.
// Positions past the length, and those of pages outside the pool, are stored as zeros and their scores hidden. A draft's values that are
// not finite are stored as zeros too and reach the rows that see them by themselves: zero probabilities of the others would
// make them NaN.
// Statistics and sums in fp32; sums run over the probabilities as rounded. In fp16 they are held times 2^11, in bf16 times a power
// of two below 1 / (2^4 length), so that sums of the largest values stay finite.
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

// Positions of a unit: a thread converts one group of 32 elements of its keys and one of its values.
template <int DIM>
constexpr int kTile = kThreads / (DIM / 32);
constexpr int kResident = 3;  // workgroups that a CU holds

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

// What starting and ending a (head, pass) costs, in units.
constexpr int kStart = 1;

// A sequence as the grid sees it.
struct Drafts {
  int begin, rows;  // its first row, and how many: at most kMostDrafts
  int length, context;
  int columns, passes;
};
__device__ __forceinline__ Drafts drafts_of(const Kv4Tree &a, int sequence) {
  Drafts d;
  const int first = min(max(a.cu[sequence], 0), a.tokens), end = min(max(a.cu[sequence + 1], first), a.tokens);
  d.begin = first;
  d.length = kv4_length(a.pool, sequence);
  d.context = d.length - (end - first);
  d.rows = min(end - first, kMostDrafts);
  d.columns = d.rows * a.group;
  d.passes = (d.columns + kCols * kPass - 1) / (kCols * kPass);
  return d;
}
template <int TILE>
__device__ __forceinline__ int tiles_of(int length) { return max(1, (length + TILE - 1) / TILE); }
template <int TILE>
__device__ __forceinline__ int units_of(const Kv4Tree &a, const Drafts &d) {
  return a.pool.kv_heads * d.passes * (kStart + tiles_of<TILE>(d.length));
}
__device__ __forceinline__ int run_units(int total, const Kv4Tree &a) { return (total + a.workgroups - 1) / a.workgroups; }

// Column blocks are shared out evenly over the passes.
__device__ __forceinline__ int blocks_a_pass(const Drafts &d) {
  const int blocks = (d.columns + kCols - 1) / kCols;
  return (blocks + d.passes - 1) / d.passes;
}

__device__ __forceinline__ bool known_position(const Kv4Pool &pool, int sequence, int position) {
  if (position < 0) return false;
  return (uint32_t)pool.table[sequence * pool.table_stride + (position >> pool.page_shift)] < (uint64_t)pool.num_pages;
}

__device__ __forceinline__ int parent_of(const Kv4Tree &a, const Drafts &d, int row) {
  const int parent = a.parents ? a.parents[d.begin + row] : row - 1;
  return (uint32_t)parent < (uint32_t)d.rows ? parent : -1;
}

// Whether row `row` of a sequence sees any position in the pool. Asked only where no score was above -infinity, to tell zeros (none)
// from a softmax that is undefined (NaN).
__device__ __forceinline__ bool sees_any(const Kv4Tree &a, const Drafts &d, int sequence, int row) {
  for (int64_t position = 0; position < d.context; position += (int64_t)1 << a.pool.page_shift)
    if (known_position(a.pool, sequence, (int)position)) return true;
  for (int step = 0; step < kMostDrafts && row >= 0; ++step, row = parent_of(a, d, row))
    if (known_position(a.pool, sequence, d.context + row)) return true;
  return false;
}

template <bool F16, int DIM>
__global__ __launch_bounds__(kThreads, kResident) void kv4_tree_kernel(Kv4Tree a) {
  constexpr int kTile = tx::kTile<DIM>, kSubs = kTile / 32, kGroups = DIM / 32;
  constexpr int kRow = DIM * 2;  // bytes of a converted row
  constexpr int kSteps = DIM / 16, kOut = DIM / 32;
  __shared__ __attribute__((aligned(1024))) char lds[2 * kTile * kRow];  // keys, then values; later the shares' outputs
  __shared__ float stats[kWaves][2][64];
  __shared__ uint8_t known[kTile / 16], odd[kTile];
  char *const keys = lds, *const values = lds + kTile * kRow;

  const Kv4Pool &pool = a.pool;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;

  // The run: units [unit, end) of the row of all; a part is what of one (head, pass) lies in it.
  Drafts d;
  int unit, end, sequence, head, pass, from, slot = 0;
  if (a.whole) {  // a workgroup for each (sequence, head, pass)
    pass = blockIdx.x % a.most_passes;
    head = blockIdx.x / a.most_passes % pool.kv_heads;
    sequence = blockIdx.x / a.most_passes / pool.kv_heads;
    d = drafts_of(a, sequence);
    if (pass >= d.passes) return;
    unit = from = 0;
    end = tiles_of<kTile>(d.length);
  } else {
    const RaggedPlace place = ragged_place(
        pool.sequences, [](int s) { return s; }, [&](int s) { return units_of<kTile>(a, drafts_of(a, s)); },
        [&](int total) { return (int)blockIdx.x * run_units(total, a); });
    const int run = run_units(place.total, a);
    unit = blockIdx.x * run;
    end = min(unit + run, place.total);
    if (unit >= end) return;
    sequence = place.sequence;
    d = drafts_of(a, sequence);
    const int share = kStart + tiles_of<kTile>(d.length), index = place.local / share;
    head = index / d.passes;
    pass = index % d.passes;
    from = place.local - index * share - kStart;  // below 0: units without work
  }

  // This thread's part of a conversion: position p of the unit, elements 32 g .. 32 g + 31.
  const int p = threadIdx.x / kGroups, g = threadIdx.x % kGroups;
  const int64_t half_bytes = kv4_half_bytes(pool.page_shift, DIM), scales_at = (int64_t)(DIM / 2) << pool.page_shift;
  const int page_mask = (1 << pool.page_shift) - 1;
  // 16-byte chunk c of row r lies at chunk c ^ turn: operand reads and these stores hit distinct banks.
  const int k_turn = DIM == 128 ? p & 15 : (p >> 1) & 7;
  const int v_turn = DIM == 128 ? 5 * (p & 3) : 4 * ((p >> 1) & 1) ^ ((p >> 1) & 3);
  // Operands: key row n, dimensions 16 st + 8 h at k_at ^ 32 st; by the transposing reads key 4 h + (lane % 16) / 4,
  // dimensions 32 t + 16 ((lane / 16) % 2) + 4 (lane % 4) at v_at ^ 64 t.
  const uint32_t x4 = (lane >> 2) & 3;
  const uint32_t k_at = (uint32_t)n * kRow + 16u * (uint32_t)(h ^ (DIM == 128 ? n & 15 : (n >> 1) & 7));
  const uint32_t v_row = 4u * h + x4, v_chunk = 2u * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_at = v_row * kRow + 8u * (lane & 1) +
                        16u * (v_chunk ^ (DIM == 128 ? 5 * (v_row & 3) : 4 * ((v_row >> 1) & 1) ^ ((v_row >> 1) & 3)));

  struct Codes {
    u32x4 k, v;
    uint32_t ks, vs;
    bool valid;
  };
  Codes codes;

  while (unit < end) {
    const int share_tiles = tiles_of<kTile>(d.length);
    const int first = max(from, 0), until = min(share_tiles, from + end - unit);
    const bool any = until > first;
    if (any) {
      const int per_pass = blocks_a_pass(d), col0 = pass * per_pass * kCols;
      const int columns = min(per_pass * kCols, d.columns - col0);  // above zero
      const int blocks = (columns + kCols - 1) / kCols;
      const int shares = blocks >= 3 ? 1 : min(kWaves / blocks, kSubs);  // waves that share a block's positions
      const int block = wave % blocks, share = wave / blocks;
      const bool works = share < shares;
      const int column = col0 + block * kCols + n;  // this lane's query
      const int row = min(column, d.columns - 1) / a.group;
      const bool mine = column < d.columns && column < col0 + columns;

      const int stop = min(until * kTile, d.length);
      auto load = [&](int tile) {
        const int position = tile * kTile + p;
        int page = -1;
        if (position < d.length) page = pool.table[sequence * pool.table_stride + (position >> pool.page_shift)];
        codes.valid = (uint32_t)page < (uint64_t)pool.num_pages;
        codes.k = codes.v = u32x4{0, 0, 0, 0};
        codes.ks = codes.vs = 127;
        if (codes.valid) {
          const uint8_t *half = pool.pages + ((int64_t)page * pool.kv_heads + head) * 2 * half_bytes;
          const int at = position & page_mask;
          codes.k = *reinterpret_cast<const u32x4 *>(half + at * (DIM / 2) + 16 * g);
          codes.v = *reinterpret_cast<const u32x4 *>(half + half_bytes + at * (DIM / 2) + 16 * g);
          codes.ks = half[scales_at + at * kGroups + g];
          codes.vs = half[half_bytes + scales_at + at * kGroups + g];
        }
      };
      load(first);

      u32x4 qb[kSteps];
      {
        const int c = min(column, d.columns - 1);
        const uint16_t *q = a.q + (int64_t)(d.begin + row) * a.q_token + (head * a.group + c % a.group) * a.q_head + 8 * h;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          qb[st] = *reinterpret_cast<const u32x4 *>(q + 16 * st);
#pragma unroll
          for (int j = 0; j < 4; ++j) qb[st][j] = (qb[st][j] & a.q_and) ^ a.q_xor;
        }
      }
      // The rows that this lane's row sees, a bit each: pointers doubled, so that any parents end.
      uint64_t seen = 0;
      if (until * kTile > d.context) {
        if (a.parents) {
          int up = lane < d.rows ? parent_of(a, d, lane) : -1;
          seen = (uint64_t)1 << lane;
#pragma unroll
          for (int i = 0; i < 6; ++i) {
            const int from_lane = max(up, 0);
            const uint64_t theirs = __shfl(seen, from_lane);
            const int further = __shfl(up, from_lane);
            seen |= up >= 0 ? theirs : 0;
            up = up >= 0 ? further : -1;
          }
          seen = __shfl(seen, row);
        } else {
          seen = ((uint64_t)2 << row) - 1;
        }
      }

      const float lift = F16 ? 15.f - kPackedLag : -kPackedLag - 1.f - (float)(32 - __builtin_clz(d.length | 1));
      float m = -INFINITY, l = 0.f;  // running maximum of the query (before the scale), this lane's share of the sum
      f32x16 o[kOut];                // o[t][r] = O[query][dimension 32 t + 8 (r / 4) + 4 h + r % 4]
#pragma unroll
      for (int t = 0; t < kOut; ++t) o[t] = f32x16{};

      for (int tile = first; tile < until; ++tile) {
        const bool drafts = (tile + 1) * kTile > d.context;  // some positions are drafted rows
        lds_barrier();  // the last unit is read
        {
          const float ks = __uint_as_float(codes.ks << 23), vs = __uint_as_float(codes.vs << 23);
          u32x4 x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = kv4_octet<F16>(codes.v[i], vs);
          if (drafts) {
            constexpr uint32_t kExponent = F16 ? 0x7C00u : 0x7F80u;
            bool mad = false;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                mad |= (x[i][j] & kExponent) == kExponent || (x[i][j] >> 16 & kExponent) == kExponent;
            const uint64_t all = __builtin_amdgcn_ballot_w64(mad);
            const bool out = tile * kTile + p >= d.context && (all >> (lane - g) & ((1 << kGroups) - 1)) != 0;
            if (g == 0) odd[p] = out;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) x[i][j] = out ? 0u : x[i][j];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            *reinterpret_cast<u32x4 *>(keys + p * kRow + 16 * ((4 * g + i) ^ k_turn)) = kv4_octet<F16>(codes.k[i], ks);
            *reinterpret_cast<u32x4 *>(values + p * kRow + 16 * ((4 * g + i) ^ v_turn)) = x[i];
          }
          if (g == 0 && p % 16 == 0) known[p / 16] = codes.valid;
        }
        if (tile + 1 < until) load(tile + 1);
        lds_barrier();
        if (!works) continue;
#pragma unroll 1
        for (int sub = share; sub < kSubs; sub += shares) {
          const int base = tile * kTile + 32 * sub;
          if (base >= stop) break;
          const char *kt = keys + 32 * sub * kRow, *vt = values + 32 * sub * kRow;
          f32x16 sc = {};
#pragma unroll
          for (int st = 0; st < kSteps; ++st) sc = mfma32<F16>(*reinterpret_cast<const u32x4 *>(kt + (k_at ^ (32u * st))), qb[st], sc);
          // sc[r]: position base + 8 (r / 4) + 4 h + r % 4
          uint32_t there = (known[2 * sub] ? 0xFFFFu : 0u) | (known[2 * sub + 1] ? 0xFFFF0000u : 0u);
          if (stop - base < 32) there &= (1u << (stop - base)) - 1u;
          there = __builtin_amdgcn_readfirstlane(there);
          uint32_t sees = there;  // a bit for each of the 32 positions
          if (base + 32 > d.context) {
            const int ahead = d.context - base;  // of the rows: the first of them, above or below the base
            sees &= ahead >= 0 ? (uint32_t)(seen << ahead) | ((1u << ahead) - 1u) : ahead > -64 ? (uint32_t)(seen >> -ahead) : 0u;
          }
          if (there != ~0u || base + 32 > d.context) {
            const uint32_t bits = sees >> (4 * h);
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = bits >> (8 * (r >> 2) + (r & 3)) & 1 ? sc[r] : -INFINITY;
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
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const u32x4 pr = {pb[4 * j], pb[4 * j + 1], pb[4 * j + 2], pb[4 * j + 3]};  // slots 0-3: positions 16 j + 4 h .., 4-7: the 8 behind
#pragma unroll
            for (int t = 0; t < kOut; ++t) {
              const char *at = vt + 16 * j * kRow + (v_at ^ (64u * t));
              const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at));
              const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(at + 8 * kRow)));
              o[t] = mfma32<F16>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pr, o[t]);
            }
          }
          if (drafts) {
            // Drafts whose values are not finite: their share, for the queries that see them alone.
            uint32_t mad = (uint32_t)__builtin_amdgcn_ballot_w64(h == 0 && odd[32 * sub + n]);
            for (; mad != 0; mad &= mad - 1) {
              const int j = __builtin_ctz(mad), position = base + j;
              uint32_t word = 0;
#pragma unroll
              for (int i = 0; i < 8; ++i) word = i == 2 * (j >> 3) + ((j & 3) >> 1) ? pb[i] : word;
              word = __shfl(word, n + 32 * (j >> 2 & 1));
              const float pj = half_bits_to_float<F16>((uint16_t)(j & 1 ? word >> 16 : word));
              const bool does = sees >> j & 1;
              const int page = pool.table[sequence * pool.table_stride + (position >> pool.page_shift)];
              const uint8_t *half = pool.pages + (((int64_t)page * pool.kv_heads + head) * 2 + 1) * half_bytes;
              const int at = position & page_mask;
#pragma unroll
              for (int t = 0; t < kOut; ++t) {
                const float scale = __uint_as_float((uint32_t)half[scales_at + at * kGroups + t] << 23);
#pragma unroll
                for (int rq = 0; rq < 4; ++rq) {
                  const uint32_t word4 = *reinterpret_cast<const uint16_t *>(half + at * (DIM / 2) + 16 * t + 4 * rq + 2 * h);
                  const uint32_t pair[2] = {kv4_pair<F16, 0>(word4, scale), kv4_pair<F16, 1>(word4, scale)};
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float v = half_bits_to_float<F16>((uint16_t)(pair[e / 2] >> (16 * (e % 2))));
                    o[t][4 * rq + e] = does ? __builtin_fmaf(pj, v, o[t][4 * rq + e]) : o[t][4 * rq + e];
                  }
                }
              }
            }
          }
        }
      }

      // The shares of a block meet in LDS. A share without a score above -infinity has l = 0 and O = 0 (or NaN, where scores were).
      l = halves_sum(l);
      if (shares > 1) {
        lds_barrier();  // the last unit is read
        if (works && share > 0) {
          stats[wave][0][lane] = m;
          stats[wave][1][lane] = l;
          float *to = reinterpret_cast<float *>(lds) + ((share - 1) * blocks + block) * kOut * 1024 + lane;
#pragma unroll
          for (int t = 0; t < kOut; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) to[(16 * t + r) * 64] = o[t][r];
        }
        lds_barrier();
        if (share == 0) {
          for (int s = 1; s < shares; ++s) {
            const float m2 = stats[s * blocks + block][0][lane], l2 = stats[s * blocks + block][1][lane];
            const float top = fmaxf(m, m2);
            const float w1 = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - top) * a.sl2);
            const float w2 = m2 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m2 - top) * a.sl2);
            const float *theirs = reinterpret_cast<const float *>(lds) + ((s - 1) * blocks + block) * kOut * 1024 + lane;
#pragma unroll
            for (int t = 0; t < kOut; ++t)
#pragma unroll
              for (int r = 0; r < 16; ++r) o[t][r] = o[t][r] * w1 + theirs[(16 * t + r) * 64] * w2;
            l = l * w1 + l2 * w2;
            m = top;
          }
        }
      }
      if (share == 0) {
        if (first == 0 && until == share_tiles) {
          if (mine) {
            const float inverse = m == -INFINITY && !sees_any(a, d, sequence, row) ? 0.f : 1.f / l;
            uint16_t *out = a.out + (int64_t)(d.begin + row) * a.out_token + (head * a.group + column % a.group) * a.out_head + 4 * h;
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
          // A block's piece: its outputs four registers at a time [4 kOut][64 lanes][4], then max and sum of its queries.
          float *piece = a.pieces + ((int64_t)blockIdx.x * 2 + slot) * a.piece_floats + block * (kOut * 1024 + 64);
#pragma unroll
          for (int t = 0; t < kOut; ++t)
#pragma unroll
            for (int rq = 0; rq < 4; ++rq)
              *reinterpret_cast<f32x4 *>(piece + (4 * t + rq) * 256 + 4 * lane) =
                  f32x4{o[t][4 * rq], o[t][4 * rq + 1], o[t][4 * rq + 2], o[t][4 * rq + 3]};
          if (h == 0) {
            piece[kOut * 1024 + n] = m;
            piece[kOut * 1024 + 32 + n] = l;
          }
        }
      }
    }
    unit += until - from;
    from = -kStart;
    slot = 1;
    if (unit < end && ++pass == d.passes) {
      pass = 0;
      if (++head == pool.kv_heads) {
        head = 0;
        do d = drafts_of(a, ++sequence);
        while (d.rows == 0);  // one with work follows: unit < end
      }
    }
  }
}

// Joins the pieces of (head, pass)es that several workgroups shared. Grid: x = (sequence * kv_heads + head) * most_passes + pass, y =
// column block, z = four output registers of a lane; a wave takes every fourth piece.
template <bool F16, int DIM>
__global__ __launch_bounds__(kThreads) void kv4_tree_combine_kernel(Kv4Tree a) {
  constexpr int kTile = tx::kTile<DIM>, kOut = DIM / 32, kHeld = 4;
  __shared__ f32x4 sums[kWaves][64];
  __shared__ float stats[kWaves][2][32];
  const Kv4Pool &pool = a.pool;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const int pass = blockIdx.x % a.most_passes, head = blockIdx.x / a.most_passes % pool.kv_heads;
  const int sequence = blockIdx.x / a.most_passes / pool.kv_heads, block = blockIdx.y, quad = blockIdx.z;
  const Drafts d = drafts_of(a, sequence);
  if (pass >= d.passes) return;
  const int per_pass = blocks_a_pass(d);
  const int column = (pass * per_pass + block) * kCols + n;
  if (block >= per_pass || (pass * per_pass + block) * kCols >= d.columns) return;
  const RaggedPlace place = ragged_before(
      pool.sequences, [](int s) { return s; }, [&](int s) { return units_of<kTile>(a, drafts_of(a, s)); }, sequence);
  const int run = run_units(place.total, a);
  const int tiles = tiles_of<kTile>(d.length);
  const int begin = place.local + (head * d.passes + pass) * (kStart + tiles), work = begin + kStart;  // units with work from here on
  const int w0 = work / run, w1 = (work + tiles - 1) / run;
  if (w0 == w1) return;  // one workgroup had it all and wrote the output
  // Only the first workgroup can have had another part before this one.
  auto piece = [&](int w) {
    return a.pieces + ((int64_t)w * 2 + (w == w0 && begin > w0 * run ? 1 : 0)) * a.piece_floats + block * (kOut * 1024 + 64);
  };
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f, m = -INFINITY;
  for (int w = w0 + wave; w <= w1; w += kWaves * kHeld) {
    f32x4 value[kHeld];
    float pm[kHeld], pl[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const float *at = piece(min(w + i * kWaves, w1));
      value[i] = *reinterpret_cast<const f32x4 *>(at + quad * 256 + 4 * lane);
      pm[i] = at[kOut * 1024 + n];
      pl[i] = at[kOut * 1024 + 32 + n];
    }
    float mnew = m;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) mnew = w + i * kWaves <= w1 ? fmaxf(mnew, pm[i]) : mnew;
    const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mnew) * a.sl2);
    sum *= alpha;
    l *= alpha;
    m = mnew;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (w + i * kWaves > w1) continue;
      const float weight = pm[i] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((pm[i] - m) * a.sl2);  // an empty piece holds zeros (or NaN)
      sum += value[i] * weight;
      l += pl[i] * weight;
    }
  }
  sums[wave][lane] = sum;
  if (h == 0) {
    stats[wave][0][n] = m;
    stats[wave][1][n] = l;
  }
  __syncthreads();
  if (wave != 0 || column >= d.columns) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][0][n]);
  f32x4 total = {0.f, 0.f, 0.f, 0.f};
  float ll = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float weight = stats[w][0][n] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((stats[w][0][n] - top) * a.sl2);
    total += sums[w][lane] * weight;
    ll += stats[w][1][n] * weight;
  }
  const int row = column / a.group;
  total *= top == -INFINITY && !sees_any(a, d, sequence, row) ? 0.f : 1.f / ll;
  uint16_t *out = a.out + (int64_t)(d.begin + row) * a.out_token + (head * a.group + column % a.group) * a.out_head + 4 * h;
  *reinterpret_cast<u32x2 *>(out + 32 * (quad / 4) + 8 * (quad % 4)) =
      u32x2{to_half_bits<F16>(total[0]) | (uint32_t)to_half_bits<F16>(total[1]) << 16,
            to_half_bits<F16>(total[2]) | (uint32_t)to_half_bits<F16>(total[3]) << 16};
}

// Upper bounds of a call from what the host knows.
int64_t most_columns(const Kv4Tree &a) { return (int64_t)(a.tokens < kMostDrafts ? a.tokens : kMostDrafts) * a.group; }
int64_t most_passes(const Kv4Tree &a) { return (most_columns(a) + kCols * kPass - 1) / (kCols * kPass); }
int64_t most_units(const Kv4Tree &a, int tile) {
  const int64_t room = (int64_t)a.pool.max_pages << a.pool.page_shift, tiles = (room + tile - 1) / tile;
  return (int64_t)a.pool.sequences * a.pool.kv_heads * most_passes(a) * (kStart + tiles);
}

}  // namespace

// Unit numbers are 32-bit; a launch has fewer than 2^32 threads, 256 for each (head, pass).
bool kv4_tree_fits(const Kv4Tree &a) {
  return most_units(a, kTile<128>) <= (int64_t)1 << 30 && (int64_t)a.pool.sequences * a.pool.kv_heads * most_passes(a) < (int64_t)1 << 24;
}

void kv4_tree_plan(Kv4Tree &a, int dim, int cus) {
  const int64_t room = (int64_t)a.pool.max_pages << a.pool.page_shift;
  const int64_t parts = (int64_t)a.pool.sequences * a.pool.kv_heads * most_passes(a);
  a.most_passes = (int)most_passes(a);
  a.whole = room <= 512;
  const int64_t most = most_units(a, dim == 128 ? kTile<128> : kTile<64>), fill = kResident * (int64_t)cus;
  a.workgroups = (int)(a.whole ? parts : most < fill ? most : fill);
  const int64_t blocks = (most_columns(a) + kCols - 1) / kCols;
  a.piece_floats = (int)(blocks < kPass ? blocks : kPass) * (kCols * dim + 64);
  a.piece_bytes = a.whole ? 0 : (int64_t)a.workgroups * 2 * a.piece_floats * (int64_t)sizeof(float);
}

hipError_t launch_kv4_tree(const Kv4Tree &a, bool f16, int dim, hipStream_t stream) {
  auto launch = [&](auto type, auto dims) {
    constexpr bool kF16 = decltype(type)::value;
    constexpr int kDim = decltype(dims)::value;
    hipLaunchKernelGGL((kv4_tree_kernel<kF16, kDim>), dim3((unsigned)a.workgroups), dim3(kThreads), 0, stream, a);
    if (a.whole) return;
    const int64_t blocks = (most_columns(a) + kCols - 1) / kCols;
    hipLaunchKernelGGL((kv4_tree_combine_kernel<kF16, kDim>),
                       dim3((unsigned)(a.pool.sequences * a.pool.kv_heads * a.most_passes), (unsigned)(blocks < kPass ? blocks : kPass), kDim / 8),
                       dim3(kThreads), 0, stream, a);
  };
  using std::integral_constant;
  if (f16 && dim == 128) launch(integral_constant<bool, true>{}, integral_constant<int, 128>{});
  else if (f16) launch(integral_constant<bool, true>{}, integral_constant<int, 64>{});
  else if (dim == 128) launch(integral_constant<bool, false>{}, integral_constant<int, 128>{});
  else launch(integral_constant<bool, false>{}, integral_constant<int, 64>{});
  return hipGetLastError();
}

}  // namespace tx
