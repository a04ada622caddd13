// Attention of one query token per sequence over a paged 4-bit KV cache (gfx950; layout in kv4.h), grouped heads.
//
// No reference counterpart: the reference's attention is the Hugging Face module's sdpa over a 16-bit cache.
//
//   out[s][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[s][h] . k_j - max),  j < lengths[s]
//
// Work: a unit is kUnit positions of one sequence and KV head; the units of all sequences lie in one row, and every
// workgroup takes an equal run of them, whatever the lengths (it finds its place from the lengths itself, so that a captured
// call serves any). A run that covers a whole (sequence, head) writes its output; the others leave (max, sum,
// unnormalised output) for the combine kernel, at most two such pieces a workgroup, so the workspace does not grow with the lengths.
//
// A wave takes kTile positions (4.25 KiB of cache) at a time and shares nothing with the other waves until its run of a head ends:
//   * S^T = K q^T (v_mfma_f32_16x16x32: A = 16 keys, B = the head's queries, up to 16): a lane's 16 bytes of codes
//     (8 at dim 64) lie in one scale group and become MFMA operands by v_cvt_scalef32_pk_*_fp4 alone: the scale rides
//     along. The queries' dimensions are laid out to match the codes;
//   * a lane then holds 4 scores of one query for every 16 keys: running maximum by two lane swaps, the probabilities,
//     rounded to 16 bits in place, are the B operand of O^T = V^T P^T;
//   * values are converted the same way and pass through the wave's own LDS, whose transposing reads
//     (ds_read_b64_tr_b16) give the A operand. 32-byte pieces lie at piece ^ f(row): the reads hit distinct banks;
//   * the next step's codes set out before these are multiplied, by buffer loads whose page is scalar, and the page ids of the one
//     after by scalar loads (as vector loads their wait had taken in the codes just set out: 54.8 against 45.4 us below);
//   * the next head's first codes set out before this head's sums are joined.
// Positions past the length (the rest of a page is stale) are loaded where they lie and replaced by zeros before they
// are converted, their scores by -infinity; a page id outside the pool counts as such.
// Statistics and sums in fp32; sums run over the probabilities as rounded. In fp16 probabilities are held times 2^15,
// so that small ones keep their bits (p <= 2^15 stays below fp16's largest); in bf16 times a power of two below 1 / (2 length), so
// that sums of the largest values stay finite (in turn values below 2^-110, at 8191 positions, lose bits to fp32's smallest).
//
// Bound: memory for long contexts, 262144 positions of 8 heads of 128 (285 MB) 44 to 47 us, 6.0 to 6.5 TB/s with a part of it still cached, and 5
// for the combine kernel and the gap before it; at dim 64 instruction issue (half the bytes for the same scores), 163 MB at 31 us, 5.3
// TB/s. A few thousand positions in all: the chain of dependent loads (lengths, page ids, codes), the merge and the second
// launch, 8 us; a codes' step further ahead, more workgroups a CU and 16-wave workgroups were all slower.
#include <math.h>

#include <type_traits>

#include "elementwise.h"
#include "kernels.h"
#include "kv4.h"
#include "ragged.h"

namespace tx {

namespace {

constexpr int kCols = 16;  // queries of an MFMA tile

constexpr int kWaves = 4;  // of a workgroup

// Positions of a wave's step (4.25 KiB of cache) and of a workgroup's: a unit.
template <int DIM>
constexpr int kTile = 4096 / DIM;
template <int DIM>
constexpr int kUnit = kTile<DIM> * kWaves;
// Workgroups that a CU holds: their registers (and, at dim 64, their LDS) set it. At dim 128 four would spill.
template <int DIM>
constexpr int kResident = DIM == 128 ? 3 : 4;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <bool F16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
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

template <bool F16>
__device__ __forceinline__ uint16_t to_half_bits(float v) {
  if constexpr (F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
  else return to_bf(v);
}

// Over the four lanes that hold one query (lane, + 16, + 32, + 48).
__device__ __forceinline__ float quarters_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quarters_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Units of a sequence's KV head: one even if it is empty, whose output is zeros.
template <int UNIT>
__device__ __forceinline__ int head_units(int length) { return max(1, (length + UNIT - 1) / UNIT); }

// What starting and ending a head costs, in units: a head's share of the row of units begins with as many without work (96
// sequences of 1 to 16384 positions, 16 heads of 64: 42.9 us, with none 50.8, with two 44.0).
constexpr int kStart = 1;

// Units of every workgroup.
__device__ __forceinline__ int run_units(int total, const Kv4Attention &a) {
  return (total + a.workgroups - 1) / a.workgroups;
}

// All of the workgroup's LDS accesses so far are done; loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Whether any position of a sequence lies in the pool, by LANES lanes that ask together. Asked only where no score was above
// -infinity, to tell zeros (no position) from a softmax that is undefined (NaN): carried along with the maxima it cost 1% at dim 64.
template <int LANES>
__device__ __forceinline__ bool any_position(const Kv4Pool &pool, int sequence, int length) {
  const int lane = threadIdx.x % LANES;
  for (int64_t first = 0; first << pool.page_shift < length; first += LANES) {
    const bool inside = (first + lane) << pool.page_shift < length;
    const bool known = inside && (uint32_t)pool.table[sequence * pool.table_stride + first + lane] < (uint64_t)pool.num_pages;
    if (LANES == 1 ? known : __builtin_amdgcn_ballot_w64(known) != 0) return true;
  }
  return false;
}

// SHARE: 16-position groups of a step that lie in one page: a page's, or all of the step's.
template <bool F16, int DIM, int SHARE>
__global__ __launch_bounds__(64 * kWaves, kResident<DIM>) void kv4_attention_kernel(Kv4Attention a) {
  constexpr int kUnit = tx::kUnit<DIM>, kTile = tx::kTile<DIM>;
  constexpr int kSubs = kTile / 16;       // 16 positions make an MFMA tile of scores
  constexpr int kWords = DIM / 32;        // words of codes a lane holds of a row: 4 or 2
  constexpr int kRow = DIM * 2;           // bytes of a converted row
  constexpr int kMergeRow = DIM + 4;      // floats of a query's output in the merge
  constexpr int kWaveBytes = kCols * kMergeRow * 4 > kTile * kRow ? kCols * kMergeRow * 4 : kTile * kRow;
  using Codes = std::conditional_t<DIM == 128, u32x4, u32x2>;
  __shared__ __attribute__((aligned(256))) char lds[kWaves][kWaveBytes];
  __shared__ float stats[kWaves][2][kCols];

  const Kv4Pool &pool = a.pool;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quarter = lane >> 4;
  const int col0 = blockIdx.y * kCols;                 // first query (of the group) of this workgroup
  const int cols = min(kCols, a.group - col0);

  // The run: units [unit, end) of the row of all; the part of one head that lies in it.
  struct Part {
    int sequence, head, length, units;
    int first, until;  // the head's units
    int slot;          // where its piece goes: 0 for the head in which the run begins
    bool any;
  };
  int unit, end, sequence, head, from, length;
  if (a.whole) {  // a workgroup for each head
    sequence = blockIdx.x / pool.kv_heads;
    head = blockIdx.x % pool.kv_heads;
    length = __builtin_amdgcn_readfirstlane(kv4_length(pool, sequence));
    unit = from = 0;
    end = head_units<kUnit>(length);
  } else {
    auto length_of = [&](int s) { return kv4_length(pool, s); };
    auto units_of = [&](int l) { return pool.kv_heads * (kStart + head_units<kUnit>(l)); };
    const RaggedPlace place = ragged_place(pool.sequences, length_of, units_of, [&](int total) { return (int)blockIdx.x * run_units(total, a); });
    const int run = run_units(place.total, a);
    unit = blockIdx.x * run;
    end = min(unit + run, place.total);
    if (unit >= end) return;
    sequence = place.sequence;
    length = place.length;
    head = place.local / (kStart + head_units<kUnit>(length));
    from = place.local - head * (kStart + head_units<kUnit>(length)) - kStart;  // below 0: units without work
  }
  int slot = 0;
  auto take = [&]() {
    const int units = head_units<kUnit>(length);
    const int until = min(units, from + end - unit);
    const Part part = {sequence, head, length, units, max(from, 0), until, slot, unit < end && until > max(from, 0)};
    unit += until - from;
    from = -kStart;
    slot = 1;
    if (++head == pool.kv_heads && unit < end) {
      head = 0;
      length = __builtin_amdgcn_readfirstlane(kv4_length(pool, ++sequence));
    }
    return part;
  };

  const int64_t half_bytes = kv4_half_bytes(pool.page_shift, DIM);
  const int64_t scales_at = (int64_t)(DIM / 2) << pool.page_shift;
  const float sl2 = a.sl2;  // above zero; the scale's sign is in the queries

  char *mine = lds[wave];
  // A converted row's 32-byte pieces lie at piece ^ turn(row): rows that one transposing read takes hit distinct banks.
  auto piece_at = [](int row, int piece) { return row * kRow + 32 * (piece ^ (DIM == 128 ? row & 7 : (row >> 1) & 3)); };

  // Page ids of a step's positions, fetched a step before its codes are.
  constexpr int kPages = kSubs / SHARE;
  struct Ids {
    int page[kPages];
  };
  auto ids_of = [&](const Part &part, int position) __attribute__((always_inline)) {
    // Constant for the whole launch: scalar loads, whose wait leaves the codes under way alone.
    const auto *table = (const __attribute__((address_space(4))) int *)(pool.table + part.sequence * pool.table_stride);
    Ids ids;
#pragma unroll
    for (int i = 0; i < kPages; ++i) ids.page[i] = table[min(position + 16 * SHARE * i, max(part.length - 1, 0)) >> pool.page_shift];
    return ids;
  };
  struct Tile {
    Codes k[kSubs], v[kSubs];
    uint32_t ks[kSubs], vs[kSubs];
    int valid[kSubs];  // positions of each 16 that count
  };
  // A lane's share of row n of each 16 positions.
  const uint32_t code_lane = n * (DIM / 2) + quarter * (DIM / 8), scale_lane = n * kWords + (DIM == 128 ? quarter : quarter >> 1);
  auto load = [&](Tile &t, const Part &part, int position, const Ids &ids) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < kPages; ++p) {
      const int at = position + 16 * SHARE * p;
      const bool known = (uint32_t)ids.page[p] < (uint64_t)pool.num_pages;
      const int page = known ? ids.page[p] : 0;
      const int row = at & ((1 << pool.page_shift) - 1);
      // Buffer loads: the page's place is scalar, the lane's share one register for all of them.
      const __amdgpu_buffer_rsrc_t half2 = __builtin_amdgcn_make_buffer_rsrc(
          pool.pages + ((int64_t)page * pool.kv_heads + part.head) * 2 * half_bytes, (short)0, (int)(2 * half_bytes), 0x00020000);
      const int codes = row * (DIM / 2), scales = (int)scales_at + row * kWords;
#pragma unroll
      for (int j = 0; j < SHARE; ++j) {
        const int i = p * SHARE + j;
        t.valid[i] = known ? min(max(part.length - at - 16 * j, 0), 16) : 0;
        const uint32_t code = code_lane + 16 * j * (DIM / 2), scale = scale_lane + 16 * j * kWords;
        if constexpr (DIM == 128) {
          t.k[i] = __builtin_amdgcn_raw_buffer_load_b128(half2, code, codes, 0);
          t.v[i] = __builtin_amdgcn_raw_buffer_load_b128(half2, code, codes + (int)half_bytes, 0);
        } else {
          t.k[i] = __builtin_amdgcn_raw_buffer_load_b64(half2, code, codes, 0);
          t.v[i] = __builtin_amdgcn_raw_buffer_load_b64(half2, code, codes + (int)half_bytes, 0);
        }
        t.ks[i] = __builtin_amdgcn_raw_buffer_load_b8(half2, scale, scales, 0);
        t.vs[i] = __builtin_amdgcn_raw_buffer_load_b8(half2, scale, scales + (int)half_bytes, 0);
      }
    }
  };
  // This wave's steps of a part: every unit's `wave`-th.
  Tile cur, next;
  Ids ids;
  auto start_of = [&](const Part &part) { return part.first * kUnit + wave * kTile; };
  auto stop_of = [&](const Part &part) { return min(part.until * kUnit, part.length); };
  auto begin = [&](const Part &part) __attribute__((always_inline)) {
    const int position = start_of(part);
    if (!part.any || position >= stop_of(part)) return;
    ids = ids_of(part, position);
    load(cur, part, position, ids);
    ids = ids_of(part, position + kUnit);
  };

  Part part = take();
  begin(part);
  while (part.any) {
    int position = start_of(part);
    const int last = stop_of(part);
    // B operands: query n, dimensions DIM/4 * quarter + 8 st ..
    u32x4 qb[kWords];
    {
      const uint16_t *q = a.q + part.sequence * a.q_sequence + (part.head * a.group + col0 + min(n, cols - 1)) * a.q_head + DIM / 4 * quarter;
#pragma unroll
      for (int st = 0; st < kWords; ++st) {
        qb[st] = reinterpret_cast<const u32x4 *>(q)[st];
#pragma unroll
        for (int j = 0; j < 4; ++j) qb[st][j] = (qb[st][j] & a.q_and) ^ a.q_xor;
      }
    }

    float m = -INFINITY, l = 0.f;  // running maximum of query n (before the scale), this lane's share of the sum
    f32x4 o[DIM / 16];             // o[t][r] = O[query n][dimension 16 t + 4 quarter + r]
#pragma unroll
    for (int t = 0; t < DIM / 16; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto multiply = [&](Tile &t) __attribute__((always_inline)) {
      int valid = 0;
#pragma unroll
      for (int i = 0; i < kSubs; ++i) valid += t.valid[i];
      const bool whole = valid == kTile;
      if (!whole) {
#pragma unroll
        for (int i = 0; i < kSubs; ++i) {
          const bool out = n >= t.valid[i];
#pragma unroll
          for (int st = 0; st < kWords; ++st) {
            t.k[i][st] = out ? 0u : t.k[i][st];
            t.v[i][st] = out ? 0u : t.v[i][st];
          }
          t.ks[i] = out ? 127u : t.ks[i];
          t.vs[i] = out ? 127u : t.vs[i];
        }
      }
      f32x4 sc[kSubs];
#pragma unroll
      for (int i = 0; i < kSubs; ++i) {
        sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float scale = __uint_as_float(t.ks[i] << 23);
#pragma unroll
        for (int st = 0; st < kWords; ++st) sc[i] = mfma16<F16>(kv4_octet<F16>(t.k[i][st], scale), qb[st], sc[i]);
      }
      // Values: converted rows into LDS while the scores finish.
#pragma unroll
      for (int i = 0; i < kSubs; ++i) {
        const float scale = __uint_as_float(t.vs[i] << 23);
#pragma unroll
        for (int st = 0; st < kWords; ++st) {
          const int d = DIM / 4 * quarter + 8 * st;  // first dimension of these eight
          *reinterpret_cast<u32x4 *>(mine + piece_at(16 * i + n, d / 16) + 2 * (d & 8)) = kv4_octet<F16>(t.v[i][st], scale);
        }
      }
      // sc[i][r]: position 16 i + 4 quarter + r, query n
      if (!whole) {
#pragma unroll
        for (int i = 0; i < kSubs; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[i][r] = 4 * quarter + r < t.valid[i] ? sc[i][r] : -INFINITY;
      }
      float mx = fmaxf(sc[0][0], sc[0][1]);
#pragma unroll
      for (int i = 0; i < kSubs; ++i)
#pragma unroll
        for (int r = i == 0 ? 2 : 0; r < 4; r += 2) mx = fmaxf(fmaxf(mx, sc[i][r]), sc[i][r + 1]);
      const float mnew = fmaxf(m, quarters_max(mx));
      if (__builtin_amdgcn_ballot_w64(mnew > m) != 0) {
        const float alpha = mnew > m ? __builtin_amdgcn_exp2f((m - mnew) * sl2) : 1.f;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < DIM / 16; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[t][r] *= alpha;
        m = mnew;
      }
      // Probabilities are held times 2^lift: in bf16 below 1 / (2 length), worked out at every step: kept, it spilled
      // registers (16 sequences of 8192 positions, 16 heads of 64: 14.5 us against 14.1).
      float lift = 15.f;
      if constexpr (!F16) {
        int length = part.length;
        asm volatile("" : "+s"(length));
        lift = (float)(__builtin_clz(length | 1) - 33);
      }
      const float base = m == -INFINITY ? 0.f : lift - m * sl2;  // no position yet: every score is -infinity
      uint32_t pb[2 * kSubs];
#pragma unroll
      for (int i = 0; i < kSubs; ++i)
#pragma unroll
        for (int r = 0; r < 4; r += 2)
          pb[2 * i + r / 2] = pack2<F16>(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][r], sl2, base)),
                                         __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][r + 1], sl2, base)), l);
      // The wave's own writes, then its reads: LDS runs a wave's operations in order, the fence holds the compiler to it.
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < kSubs / 2; ++j) {
        const u32x4 p = {pb[4 * j], pb[4 * j + 1], pb[4 * j + 2], pb[4 * j + 3]};  // slots 0-3: positions 4 quarter .., 4-7: the 16 behind
        const int row = 32 * j + 4 * quarter + (n >> 2);
#pragma unroll
        for (int t = 0; t < DIM / 16; ++t) {
          const char *lo_at = mine + piece_at(row, t) + 8 * (n & 3), *hi_at = mine + piece_at(row + 16, t) + 8 * (n & 3);
          const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)lo_at));
          const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)hi_at));
          o[t] = mfma16<F16>(u32x4{lo[0], lo[1], hi[0], hi[1]}, p, o[t]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
    while (position < last) {
      if (position + kUnit < last) {
        load(next, part, position + kUnit, ids);
        ids = ids_of(part, position + 2 * kUnit);
      }
      multiply(cur);
      cur = next;
      position += kUnit;
    }

    // The next part's first codes set out before this part's sums are joined.
    const Part after = take();
    begin(after);

    // The waves' shares meet in LDS. M is -infinity where no position counted or no score was above it: then l = 0 and O = 0
    // everywhere (or NaN, where scores were).
    l = quarters_sum(l);
    if (quarter == 0) {
      stats[wave][0][n] = m;
      stats[wave][1][n] = l;
    }
    lds_barrier();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][0][n]);
    const float weight = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - top) * sl2);
    float *merge = reinterpret_cast<float *>(mine);
#pragma unroll
    for (int t = 0; t < DIM / 16; ++t)
      *reinterpret_cast<f32x4 *>(merge + n * kMergeRow + 16 * t + 4 * quarter) = o[t] * weight;
    lds_barrier();
    const bool complete = part.first == 0 && part.until == part.units;
    float *piece = a.pieces + ((int64_t)(blockIdx.x * 2 + part.slot)) * a.piece_floats;
    for (int i = threadIdx.x; i < cols * (DIM / 4); i += 64 * kWaves) {
      const int q = i / (DIM / 4), d = 4 * (i % (DIM / 4));
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        sum += *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(lds[w]) + q * kMergeRow + d);
        mm = fmaxf(mm, stats[w][0][q]);
      }
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        ll += stats[w][0][q] == -INFINITY ? stats[w][1][q] : stats[w][1][q] * __builtin_amdgcn_exp2f((stats[w][0][q] - mm) * sl2);
      if (complete) {
        // A lane each: a head that one workgroup has to itself has few pages.
        const float inverse = mm == -INFINITY && !any_position<1>(pool, part.sequence, part.length) ? 0.f : 1.f / ll;
        uint16_t *out = a.out + part.sequence * a.out_sequence + (part.head * a.group + col0 + q) * a.out_head + d;
        const uint32_t lo = to_half_bits<F16>(sum[0] * inverse) | (uint32_t)to_half_bits<F16>(sum[1] * inverse) << 16;
        const uint32_t hi = to_half_bits<F16>(sum[2] * inverse) | (uint32_t)to_half_bits<F16>(sum[3] * inverse) << 16;
        *reinterpret_cast<u32x2 *>(out) = u32x2{lo, hi};
      } else {
        *reinterpret_cast<f32x4 *>(piece + (int64_t)(col0 + q) * DIM + d) = sum;
        if (d == 0) {
          float *s = piece + (int64_t)a.group * DIM + 2 * (col0 + q);
          s[0] = mm;
          s[1] = ll;
        }
      }
    }
    lds_barrier();  // before the buffers are written again
    part = after;
  }
}

// Joins the pieces of heads that several workgroups shared. Grid: x = sequence * kv_heads + head, y = query of the group,
// z = 4 * LANES dimensions of its output.
template <bool F16, int DIM, int LANES>
__global__ __launch_bounds__(256) void kv4_combine_kernel(Kv4Attention a) {
  constexpr int kUnit = tx::kUnit<DIM>;
  constexpr int kLanes = LANES, kGroups = 256 / kLanes, kHeld = 4;  // a thread holds kHeld pieces' values at once
  __shared__ f32x4 lds[kGroups][kLanes];
  __shared__ float sums[kGroups], tops[4];
  const Kv4Pool &pool = a.pool;
  const int sequence = blockIdx.x / pool.kv_heads, head = blockIdx.x % pool.kv_heads, q = blockIdx.y;
  auto length_of = [&](int s) { return kv4_length(pool, s); };
  auto units_of = [&](int l) { return pool.kv_heads * (kStart + head_units<kUnit>(l)); };
  const RaggedPlace place = ragged_before(pool.sequences, length_of, units_of, sequence);
  const int run = run_units(place.total, a);
  const int units = head_units<kUnit>(place.length);
  const int begin = place.local + head * (kStart + units), work = begin + kStart;  // units with work: work .. work + units - 1
  const int w0 = work / run, w1 = (work + units - 1) / run;
  if (w0 == w1) return;  // one workgroup had it all and wrote the output
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, d = 4 * (kLanes * blockIdx.z + lane);
  const int64_t floats = a.piece_floats, stats_at = (int64_t)a.group * DIM + 2 * q;
  // Only the first workgroup can have had another head before this one.
  auto piece = [&](int w) { return a.pieces + ((int64_t)w * 2 + (w == w0 && begin > w0 * run ? 1 : 0)) * floats; };
  // Each thread keeps its own running maximum over its pieces; the threads' sums meet under the largest.
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f, m = -INFINITY;
  for (int w = w0 + group; w <= w1; w += kGroups * kHeld) {
    f32x4 value[kHeld];
    float pm[kHeld], pl[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const float *p = piece(min(w + i * kGroups, w1));
      value[i] = *reinterpret_cast<const f32x4 *>(p + (int64_t)q * DIM + d);
      pm[i] = p[stats_at];
      pl[i] = p[stats_at + 1];
    }
    float mnew = m;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) mnew = w + i * kGroups <= w1 ? fmaxf(mnew, pm[i]) : mnew;
    const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mnew) * a.sl2);
    sum *= alpha;
    l *= alpha;
    m = mnew;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (w + i * kGroups > w1) continue;
      const float weight = pm[i] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((pm[i] - m) * a.sl2);  // an empty piece holds zeros (or NaN)
      sum += value[i] * weight;
      l += pl[i] * weight;
    }
  }
  float top = wave_max(m);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const bool none = top == -INFINITY && !any_position<64>(pool, sequence, place.length);
  const float weight = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - top) * a.sl2);
  lds[group][lane] = sum * weight;
  if (lane == 0) sums[group] = l * weight;
  __syncthreads();
  if (threadIdx.x < 4 * kLanes) {
    const float *column = reinterpret_cast<const float *>(&lds[0][0]) + threadIdx.x;
    float total = 0.f, ll = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      total += column[g * 4 * kLanes];
      ll += sums[g];
    }
    a.out[sequence * a.out_sequence + (head * a.group + q) * a.out_head + 4 * kLanes * blockIdx.z + threadIdx.x] =
        to_half_bits<F16>(none ? 0.f : total / ll);
  }
}

// An upper bound on a call's units, from what the host knows.
int64_t most_units(const Kv4Pool &pool, int unit) {
  const int64_t room = (int64_t)pool.max_pages << pool.page_shift;
  const int64_t units = (room + unit - 1) / unit;
  return (int64_t)pool.sequences * pool.kv_heads * (kStart + (units > 1 ? units : 1));
}

}  // namespace

// Unit numbers are 32-bit; a launch has fewer than 2^32 threads, 256 for each head.
bool kv4_attention_fits(const Kv4Pool &pool) {
  return most_units(pool, kUnit<128>) <= (int64_t)1 << 30 && (int64_t)pool.sequences * pool.kv_heads < (int64_t)1 << 24;
}

void kv4_attention_plan(Kv4Attention &a, int dim, int cus) {
  const int64_t room = (int64_t)a.pool.max_pages << a.pool.page_shift, heads = (int64_t)a.pool.sequences * a.pool.kv_heads;
  // A workgroup for each head, and no combine kernel, where no head can be long: always up to 512 positions (128
  // sequences of 500, 4 heads of 64: 7.3 us against 13.3), up to 1024 where the heads fill the chip by themselves (1024 heads
  // of 64 at 600 positions 14.3 against 16.8; 2 heads of 128 at 700: 9.4 against 8.7).
  a.whole = room <= 512 || (room <= 1024 && heads >= cus);
  const int64_t most = most_units(a.pool, dim == 128 ? kUnit<128> : kUnit<64>);
  const int64_t fill = (dim == 128 ? kResident<128> : kResident<64>) * (int64_t)cus;
  a.workgroups = (int)(a.whole ? heads : most < fill ? most : fill);
  a.piece_floats = (a.group * (dim + 2) + 3) & ~3;
  a.piece_bytes = a.whole ? 0 : (int64_t)a.workgroups * 2 * a.piece_floats * (int64_t)sizeof(float);
}

hipError_t launch_kv4_attention(const Kv4Attention &a, bool f16, int dim, hipStream_t stream) {
  const dim3 grid((unsigned)a.workgroups, (unsigned)((a.group + kCols - 1) / kCols));
  const unsigned heads = (unsigned)(a.pool.sequences * a.pool.kv_heads);
  auto launch = [&](auto type, auto d) {
    constexpr bool kF16 = decltype(type)::value;
    constexpr int kDim = decltype(d)::value;
    const int groups = 1 << (a.pool.page_shift - 4);  // of 16 positions, in a page
    if (groups >= kTile<kDim> / 16) hipLaunchKernelGGL((kv4_attention_kernel<kF16, kDim, kTile<kDim> / 16>), grid, dim3(64 * kWaves), 0, stream, a);
    else if (groups >= 2) hipLaunchKernelGGL((kv4_attention_kernel<kF16, kDim, 2>), grid, dim3(64 * kWaves), 0, stream, a);
    else hipLaunchKernelGGL((kv4_attention_kernel<kF16, kDim, 1>), grid, dim3(64 * kWaves), 0, stream, a);
    if (a.whole) return;
    // Few outputs are spread over more workgroups, 32 dimensions each (40 heads' queries of 1024 pieces: 5.2 us against
    // 6.7); many are not (1280 of them 5.2 against 8.0).
    if ((int64_t)heads * a.group * (kDim / 32) <= 1024)
      hipLaunchKernelGGL((kv4_combine_kernel<kF16, kDim, 8>), dim3(heads, (unsigned)a.group, kDim / 32), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((kv4_combine_kernel<kF16, kDim, kDim / 4>), dim3(heads, (unsigned)a.group), dim3(256), 0, stream, a);
  };
  using std::integral_constant;
  if (f16 && dim == 128) launch(integral_constant<bool, true>{}, integral_constant<int, 128>{});
  else if (f16) launch(integral_constant<bool, true>{}, integral_constant<int, 64>{});
  else if (dim == 128) launch(integral_constant<bool, false>{}, integral_constant<int, 128>{});
  else launch(integral_constant<bool, false>{}, integral_constant<int, 64>{});
  return hipGetLastError();
}

}  // namespace tx
