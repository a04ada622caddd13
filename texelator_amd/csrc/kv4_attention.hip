// Attention of one query token per sequence over a paged 4-bit KV cache (gfx950; layout in kv4.h), grouped heads.
//
// No reference counterpart: the reference's attention is the Hugging Face module's sdpa over a 16-bit cache.
//
//   out[s][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[s][h] . k_j - max),  j < lengths[s]
//
// Work: a unit is kUnit positions of one sequence and KV head; the units of all sequences lie in one row, and every
// workgroup takes an equal run of them, whatever the lengths (it finds its place from the lengths itself). A run
// that covers a whole (sequence, head) writes its output; the others leave (max, sum, unnormalised output) for the
// combine kernel, at most two such pieces a workgroup, so the workspace does not grow with the lengths.
//
// A wave takes 32 positions at a time and shares nothing with the other waves until its run of a head ends:
//   * S^T = K q^T (v_mfma_f32_16x16x32: A = 16 keys, B = the head's queries, up to 16): a lane's 16 bytes of codes
//     (8 at dim 64) lie in one scale group and become MFMA operands by v_cvt_scalef32_pk_*_fp4 alone: the scale rides
//     along. The queries' dimensions are laid out to match the codes;
//   * a lane then holds 8 scores of one query: running maximum by two lane swaps, the probabilities, rounded to 16
//     bits in place, are the B operand of O^T = V^T P^T;
//   * values are converted the same way and pass through the wave's own LDS, whose transposing reads
//     (ds_read_b64_tr_b16) give the A operand. 32-byte pieces lie at piece ^ f(row): the reads hit distinct banks;
//   * the next 32 positions' codes are loaded while these are multiplied.
// Positions past the length (the rest of a page is stale) are loaded where they lie and replaced by zeros before they
// are converted, their scores by -infinity; a page id outside the pool counts as such.
// Statistics and sums in fp32; sums run over the probabilities as rounded. In fp16 probabilities are held times 2^15,
// so that small ones keep their bits (p <= 2^15 stays below fp16's largest).
#include <math.h>

#include <type_traits>

#include "elementwise.h"
#include "kernels.h"
#include "kv4.h"
#include "ragged.h"

namespace tx {

namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;               // positions of a wave's step
constexpr int kUnit = kWaves * kTile;   // positions of a workgroup's step
constexpr int kCols = 16;               // queries of an MFMA tile

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
__device__ __forceinline__ int head_units(int length) { return max(1, (length + kUnit - 1) / kUnit); }

// Units of every workgroup.
__device__ __forceinline__ int run_units(int total, const Kv4Attention &a) {
  return max((total + a.workgroups - 1) / a.workgroups, a.least_units);
}

// Floats of a piece: per query its output [dim], then max and sum of all queries.
__device__ __host__ inline int64_t piece_floats(int group, int dim) { return (int64_t)group * (dim + 2); }

template <bool F16, int DIM>
__global__ __launch_bounds__(64 * kWaves, 4) void kv4_attention_kernel(Kv4Attention a) {
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

  auto units_of = [&](int s) { return pool.kv_heads * head_units(kv4_length(pool, s)); };
  const int total = ragged_total(pool.sequences, units_of);
  const int run = run_units(total, a);
  int unit = blockIdx.x * run;
  if (unit >= total) return;
  const int end = min(unit + run, total);
  int sequence, local;
  ragged_find(pool.sequences, unit, units_of, sequence, local);
  sequence = __builtin_amdgcn_readfirstlane(sequence);
  int length = __builtin_amdgcn_readfirstlane(kv4_length(pool, sequence));
  int units = head_units(length);
  int head = __builtin_amdgcn_readfirstlane(local / units);
  int first = __builtin_amdgcn_readfirstlane(local) - head * units;  // first unit of this head to do
  int slot = 0;                                        // 0: the run's first piece

  const int64_t half_bytes = kv4_half_bytes(pool.page_shift, DIM);
  const int64_t scales_at = (int64_t)(DIM / 2) << pool.page_shift;
  const float sl2 = a.scale * 1.44269504088896340736f;  // scores in log2 units
  constexpr float kLift = F16 ? 15.f : 0.f;

  char *mine = lds[wave];
  // A converted row's 32-byte pieces lie at piece ^ turn(row): rows that one transposing read takes hit distinct banks.
  auto piece_at = [](int row, int piece) { return row * kRow + 32 * (piece ^ (DIM == 128 ? row & 7 : (row >> 1) & 3)); };

  while (unit < end) {
    const int count = min(units - first, end - unit);
    const int sequence_pages = (length + (1 << pool.page_shift) - 1) >> pool.page_shift;
    const int *table = pool.table + sequence * pool.table_stride;

    // B operands: query n, dimensions DIM/4 * quarter + 8 st ..
    u32x4 qb[kWords];
    {
      const uint16_t *q = a.q + sequence * a.q_sequence + (head * a.group + col0 + min(n, cols - 1)) * a.q_head + DIM / 4 * quarter;
#pragma unroll
      for (int st = 0; st < kWords; ++st) qb[st] = reinterpret_cast<const u32x4 *>(q)[st];
    }

    struct Tile {
      Codes k[2], v[2];
      uint32_t ks[2], vs[2];
      int valid[2];
    };
    // The 16 positions from `position` on: a lane's share of row n.
    auto load = [&](Tile &t, int position) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = position + 16 * i, index = at >> pool.page_shift;
        int page = index < sequence_pages ? table[index] : -1;
        int valid = min(max(length - at, 0), 16);
        if ((uint32_t)page >= (uint64_t)pool.num_pages) page = 0, valid = 0;
        t.valid[i] = valid;
        const uint8_t *keys = pool.pages + ((int64_t)page * pool.kv_heads + head) * 2 * half_bytes;
        const uint8_t *values = keys + half_bytes;
        const uint32_t row = (uint32_t)(at & ((1 << pool.page_shift) - 1)) + n;
        const uint32_t codes = row * (DIM / 2) + quarter * (DIM / 8), scale = row * kWords + (DIM == 128 ? quarter : quarter >> 1);
        t.k[i] = *reinterpret_cast<const Codes *>(keys + codes);
        t.v[i] = *reinterpret_cast<const Codes *>(values + codes);
        t.ks[i] = (keys + scales_at)[scale];
        t.vs[i] = (values + scales_at)[scale];
      }
    };

    float m = -INFINITY, l = 0.f;  // running maximum of query n (log2 units), this lane's share of the sum
    f32x4 o[DIM / 16];             // o[t][r] = O[query n][dimension 16 t + 4 quarter + r]
#pragma unroll
    for (int t = 0; t < DIM / 16; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto step = [&](const Tile &t) __attribute__((always_inline)) {
      const bool whole = t.valid[0] + t.valid[1] == kTile;
      f32x4 sc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        const bool out = !whole && n >= t.valid[i];
        const float scale = __uint_as_float((out ? 127u : t.ks[i]) << 23);
#pragma unroll
        for (int st = 0; st < kWords; ++st)
          sc[i] = mfma16<F16>(kv4_octet<F16>(out ? 0u : t.k[i][st], scale), qb[st], sc[i]);
      }
      // sc[i][r]: position 16 i + 4 quarter + r, query n
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sc[i][r] *= sl2;
          if (!whole) sc[i][r] = 4 * quarter + r < t.valid[i] ? sc[i][r] : -INFINITY;
        }
      // Values: converted rows into LDS while the scores finish.
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool out = !whole && n >= t.valid[i];
        const float scale = __uint_as_float((out ? 127u : t.vs[i]) << 23);
#pragma unroll
        for (int st = 0; st < kWords; ++st) {
          const int d = DIM / 4 * quarter + 8 * st;  // first dimension of these eight
          *reinterpret_cast<u32x4 *>(mine + piece_at(16 * i + n, d / 16) + 2 * (d & 8)) =
              kv4_octet<F16>(out ? 0u : t.v[i][st], scale);
        }
      }
      float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                       fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
      const float mnew = fmaxf(m, quarters_max(mx));
      if (__builtin_amdgcn_ballot_w64(mnew > m) != 0) {
        const float alpha = mnew > m ? __builtin_amdgcn_exp2f(m - mnew) : 1.f;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < DIM / 16; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[t][r] *= alpha;
        m = mnew;
      }
      const float base = m == -INFINITY ? 0.f : m - kLift;  // no position yet: every score is -infinity
      uint32_t pb[4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; r += 2)
          pb[2 * i + r / 2] = pack2<F16>(__builtin_amdgcn_exp2f(sc[i][r] - base), __builtin_amdgcn_exp2f(sc[i][r + 1] - base), l);
      const u32x4 p = {pb[0], pb[1], pb[2], pb[3]};  // slots 0-3: positions 4 quarter .., slots 4-7: the 16 behind
      // The wave's own writes, then its reads: LDS runs a wave's operations in order, the fence holds the compiler to it.
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < DIM / 16; ++t) {
        const int row = 4 * quarter + (n >> 2);
        const char *lo_at = mine + piece_at(row, t) + 8 * (n & 3), *hi_at = mine + piece_at(row + 16, t) + 8 * (n & 3);
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)lo_at));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)hi_at));
        o[t] = mfma16<F16>(u32x4{lo[0], lo[1], hi[0], hi[1]}, p, o[t]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };

    // This wave's tiles: every unit's `wave`-th 32 positions, the next ones loaded before these are used.
    const int last = min((first + count) * kUnit, length);
    int position = first * kUnit + wave * kTile;
    if (position < last) {
      Tile cur, next;
      load(cur, position);
      for (; position + kUnit < last; position += kUnit) {
        load(next, position + kUnit);
        step(cur);
        cur = next;
      }
      step(cur);
    }

    // The waves' shares meet in LDS. M is -infinity where no position counted: then l = 0 and O = 0 everywhere.
    l = quarters_sum(l);
    if (quarter == 0) {
      stats[wave][0][n] = m;
      stats[wave][1][n] = l;
    }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][0][n]);
    const float weight = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    float *merge = reinterpret_cast<float *>(mine);
#pragma unroll
    for (int t = 0; t < DIM / 16; ++t)
      *reinterpret_cast<f32x4 *>(merge + n * kMergeRow + 16 * t + 4 * quarter) = o[t] * weight;
    __syncthreads();
    const bool complete = first == 0 && count == units;
    float *piece = a.pieces + ((int64_t)(blockIdx.x * 2 + slot)) * piece_floats(a.group, DIM);
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
        ll += stats[w][0][q] == -INFINITY ? stats[w][1][q] : stats[w][1][q] * __builtin_amdgcn_exp2f(stats[w][0][q] - mm);
      if (complete) {
        const float inverse = ll == 0.f ? 0.f : 1.f / ll;
        uint16_t *out = a.out + sequence * a.out_sequence + (head * a.group + col0 + q) * a.out_head + d;
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
    __syncthreads();  // before the buffers are written again
    unit += count;
    first = 0;
    slot = 1;
    if (++head == pool.kv_heads) {
      head = 0;
      ++sequence;
      if (unit < end) {
        length = __builtin_amdgcn_readfirstlane(kv4_length(pool, sequence));
        units = head_units(length);
      }
    }
  }
}

// Joins the pieces of heads that several workgroups shared. Grid: x = sequence * kv_heads + head, y = query of the group.
template <bool F16, int DIM>
__global__ __launch_bounds__(256) void kv4_combine_kernel(Kv4Attention a) {
  constexpr int kLanes = DIM / 4, kGroups = 256 / kLanes;
  __shared__ float lds[kGroups][DIM + 1];
  __shared__ float sums[kGroups];
  const Kv4Pool &pool = a.pool;
  auto units_of = [&](int s) { return pool.kv_heads * head_units(kv4_length(pool, s)); };
  const int sequence = blockIdx.x / pool.kv_heads, head = blockIdx.x % pool.kv_heads, q = blockIdx.y;
  const int run = run_units(ragged_total(pool.sequences, units_of), a);
  const int units = head_units(kv4_length(pool, sequence));
  const int begin = ragged_total(sequence, units_of) + head * units;  // this head's units: begin .. begin + units - 1
  const int w0 = begin / run, w1 = (begin + units - 1) / run;
  if (w0 == w1) return;  // one workgroup had it all and wrote the output
  const int group = threadIdx.x / kLanes, d = 4 * (threadIdx.x % kLanes);
  const int64_t floats = piece_floats(a.group, DIM);
  // Only the first workgroup can have had another head before this one.
  auto piece = [&](int w) { return a.pieces + ((int64_t)w * 2 + (w == w0 && begin > w0 * run ? 1 : 0)) * floats; };
  float top = -INFINITY;
  for (int w = w0 + (threadIdx.x & 63); w <= w1; w += 64) top = fmaxf(top, piece(w)[(int64_t)a.group * DIM + 2 * q]);
  top = wave_max(top);
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int w = w0 + group; w <= w1; w += kGroups) {
    const float *p = piece(w);
    const float *s = p + (int64_t)a.group * DIM + 2 * q;
    const float m = s[0];
    const float weight = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);  // an empty piece holds zeros (or NaN)
    sum += *reinterpret_cast<const f32x4 *>(p + (int64_t)q * DIM + d) * weight;
    l += s[1] * weight;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) lds[group][d + j] = sum[j];
  if (d == 0) sums[group] = l;
  __syncthreads();
  if (threadIdx.x < DIM) {
    float total = 0.f, ll = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      total += lds[g][threadIdx.x];
      ll += sums[g];
    }
    a.out[sequence * a.out_sequence + (head * a.group + q) * a.out_head + threadIdx.x] =
        to_half_bits<F16>(ll == 0.f ? 0.f : total / ll);
  }
}

// Workgroups of a call, from what the host knows: an upper bound on its units.
int64_t most_units(const Kv4Pool &pool) {
  const int64_t room = (int64_t)pool.max_pages << pool.page_shift;
  const int64_t units = (room + kUnit - 1) / kUnit;
  return (int64_t)pool.sequences * pool.kv_heads * (units > 1 ? units : 1);
}

}  // namespace

bool kv4_attention_fits(const Kv4Pool &pool) { return most_units(pool) <= (int64_t)1 << 30; }

void kv4_attention_plan(Kv4Attention &a, int dim, int cus) {
  const int64_t most = most_units(a.pool);
  const int64_t fill = 4 * (int64_t)cus;  // four workgroups a CU are resident
  a.workgroups = (int)(most < fill ? most : fill);
  a.least_units = 1;
  a.piece_bytes = (int64_t)a.workgroups * 2 * piece_floats(a.group, dim) * (int64_t)sizeof(float);
}

hipError_t launch_kv4_attention(const Kv4Attention &a, bool f16, int dim, hipStream_t stream) {
  const dim3 grid((unsigned)a.workgroups, (unsigned)((a.group + kCols - 1) / kCols));
  const dim3 combine((unsigned)(a.pool.sequences * a.pool.kv_heads), (unsigned)a.group);
  auto launch = [&](auto type, auto d) {
    constexpr bool kF16 = decltype(type)::value;
    constexpr int kDim = decltype(d)::value;
    hipLaunchKernelGGL((kv4_attention_kernel<kF16, kDim>), grid, dim3(64 * kWaves), 0, stream, a);
    if (a.pool.max_pages > kUnit >> a.pool.page_shift)  // else no head has more than one unit
      hipLaunchKernelGGL((kv4_combine_kernel<kF16, kDim>), combine, dim3(256), 0, stream, a);
  };
  using std::integral_constant;
  if (f16 && dim == 128) launch(integral_constant<bool, true>{}, integral_constant<int, 128>{});
  else if (f16) launch(integral_constant<bool, true>{}, integral_constant<int, 64>{});
  else if (dim == 128) launch(integral_constant<bool, false>{}, integral_constant<int, 128>{});
  else launch(integral_constant<bool, false>{}, integral_constant<int, 64>{});
  return hipGetLastError();
}

}  // namespace tx
