// Verification of drafted tokens against the target model's probabilities (gfx950), from given random numbers.
//
// No reference counterpart: the reference decodes one token at a time.
//
// A sequence's rows are a tree: row 0 its last token, row i a draft behind row parents[i]. p_v = softmax(logits[v] / T). From
// row 0 on, the drafts behind the row v that is reached are tried in the order of their rows:
//   * given drafts: draft i is accepted where u_i (1 - sum of the earlier drafts' p_v) < p_v(token i), a token that an earlier one
//     of them has never; where none is, the closing token is drawn from p_v without their tokens;
//   * chains sampled from a draft model, q_v = softmax(draft_logits[v] / T): accepted where u_i q_v(token i) < p_v(token i); else the
//     closing token is drawn from max(p_v - q_v, 0);
//   * T = 0: accepted where the token is the largest logit's (of equal ones the first), which is the closing token too.
// A token is drawn as the first whose running sum in the vocabulary's order exceeds u_0 times the whole sum.
//
// Two launches. The first reads all logits once, a wave 64 * kLoads * 16 bytes of a row, and leaves the maximum and the sum
// of exponentials of each such span, in 32 bits: enough for the tests (sums of thousands of terms that count are off by some 1e-8, of a
// few by up to 1e-7, half a unit of the last bit of each). In the second every workgroup of a sequence
// finds its path: a lane has a row, all drafts are tested at once and a row is reached where all rows that lead to it are taken. The
// workgroups then share the last row reached and sum its weights in 64 bits, a wave 512 tokens: a draw is as exact as those
// sums are, and 150 thousand borders lie close. The one that ends last finds the 512 tokens, then the token in them; who that is
// changes no result. For the residual max(p - q, 0) the sums of p and q are only known then: the weights of p and q are summed over the
// tokens where p > q by the first launch's sums; a token that those put on the wrong side adds at most what they are off by, of its own
// probability.
//
// Measured, first and second launch: 16 chains of up to 8 rows sampled from a draft's logits of 151,936 bf16 tokens 14 us (the
// logits' 55 MB at 3.9 TB/s) and 23 us, 24 trees of up to 64 rows of 32,003 fp32 tokens 26 us (5.5 TB/s) and 17 us, one
// tree of 6 rows 4 us and 15 us. The second is bound by its steps' latency: 6 us to the path, 5 to 10 for the sums, 5 to 7 for the token.
// With a launch of its own for the token and a wave for each row's statistics they took 64, 69 and 26 us in all; with a fence by every
// thread behind the sums, not one, the second launch takes 84, 32 and 19 us.
#include <math.h>

#include "elementwise.h"
#include "kernels.h"
#include "kv4.h"
#include "ragged.h"

namespace tx {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kLoads = 4;  // 16-byte loads of a lane

// Elements of a lane's load, and of a wave's span.
template <typename T>
constexpr int kVector = 16 / (int)sizeof(T);
template <typename T>
constexpr int kSpan = 64 * kLoads * kVector<T>;

struct Bf16 {
  uint16_t bits;
};
struct Fp16 {
  uint16_t bits;
};
__device__ __forceinline__ float widen(Bf16 v) { return bf(v.bits); }
__device__ __forceinline__ float widen(Fp16 v) { return hf(v.bits); }
__device__ __forceinline__ float widen(float v) { return v; }

// 16 bytes at any element's address: rows of odd widths begin anywhere.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <typename T>
__device__ __forceinline__ void widen_all(u32x4 raw, float *x) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = widen(T{(uint16_t)(raw[i / 2] >> (16 * (i % 2)))});
  }
}

// ln(2)^k / k!: 2^f is the sum of these times f^k.
constexpr double power_of_ln2(int k) { return k == 0 ? 1.0 : power_of_ln2(k - 1) * 0.693147180559945309417232121458 / k; }

// 2^y of y <= 1 in 64 bits: the Taylor sum of 2^f, |f| <= 1/2, to the twelfth power (off by 2e-16). NaN stays.
__device__ __forceinline__ double exp2_64(double y) {
  y = y < -1100.0 ? -1100.0 : y;  // 2^-1100 is zero
  constexpr double kTerm[13] = {power_of_ln2(0), power_of_ln2(1), power_of_ln2(2),  power_of_ln2(3),  power_of_ln2(4),
                                power_of_ln2(5), power_of_ln2(6), power_of_ln2(7),  power_of_ln2(8),  power_of_ln2(9),
                                power_of_ln2(10), power_of_ln2(11), power_of_ln2(12)};
  const double whole = rint(y), f = y - whole;
  double sum = kTerm[12];
#pragma unroll
  for (int i = 11; i >= 0; --i) sum = __builtin_fma(sum, f, kTerm[i]);
  return ldexp(sum, (int)whole);
}

// log2(e) / T; finite for every T above zero, of which those that fp32 holds with fewer bits count as the least that it holds with all.
__device__ __forceinline__ double rate_of(float temperature) { return 1.44269504088896340736 / fmax((double)temperature, 0x1p-126); }

// The exponents of a span's terms, x * rate - shift. The rate is the sum of two floats: rounded to one it would put all terms of a row off
// alike, the more the farther they are below the maximum (sums of 151,936 tokens at a temperature of 2.5 by 1.3e-7, so by 1e-8). The
// larger has 12 bits, or the smaller's products would be lost behind its products' last bits, again all one way. The shift is the
// largest exponent, rounded, so that no subtraction comes before the products; where that rounding would tell, or a part of the rate
// is zero (no factor for -infinity), it is (x - maximum) * rate. Neither part is below zero.
struct Exponents {
  float high, low, shift;
  bool shifted;
};
__device__ __forceinline__ Exponents exponents_of(float top, double rate) {
  const float near = (float)rate;
  const float high = __uint_as_float((__float_as_uint(near) - ((double)near > rate)) & 0xFFFFF000u), low = (float)(rate - (double)high);
  const float shift = (float)((double)top * rate);
  return {high, low, shift, high > 0.f && low > 0.f && fabsf(shift) < 1024.f};
}

struct Rows {
  int begin, count;  // a sequence's rows: at most kMostDrafts
};
__device__ __forceinline__ Rows rows_of(const Verify &a, int sequence) {
  const int begin = min(max(a.cu[sequence], 0), a.tokens);
  return {begin, min(min(max(a.cu[sequence + 1], begin), a.tokens) - begin, kMostDrafts)};
}
__device__ __forceinline__ float temperature_of(const Verify &a, int sequence) {
  return a.temperatures ? a.temperatures[sequence] : a.temperature;
}
__device__ __forceinline__ int wave_min_int(int v) { return -wave_max_int(-v); }

// Grid: x spans by kWaves, y rows, z target and draft logits. Partial of a span: (maximum, sum of 2^(x / T * log2(e) - shift)), or
// at T = 0 (maximum, its first index); a NaN among the logits makes the sum (at T = 0 the maximum) NaN.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(Verify a) {
  const int lane = threadIdx.x & 63, span = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.y;
  if (blockIdx.x == 0 && blockIdx.z == 0)  // the second launch counts in them
    for (int64_t s = (int64_t)row * kThreads + threadIdx.x; s < a.sequences; s += (int64_t)a.tokens * kThreads) a.counters[s] = 0;
  if (span >= a.spans) return;
  const bool draft = blockIdx.z != 0;
  const T *logits = reinterpret_cast<const T *>(draft ? a.draft : a.target) + row * (draft ? a.draft_row : a.target_row);
  // The row's sequence: as many starts behind the first lie at or before it.
  int sequence = 0;
  for (int first = 0; first < a.sequences; first += 64) {
    const bool before = first + lane < a.sequences && a.cu[first + lane + 1] <= row;
    sequence += __builtin_popcountll(__builtin_amdgcn_ballot_w64(before));
  }
  if (sequence >= a.sequences || row < a.cu[0]) return;
  const Rows rows = rows_of(a, sequence);
  const int local = row - rows.begin;
  if (local < 0 || local >= rows.count || (draft && local + 1 >= rows.count)) return;  // a chain's last row has no draft behind it
  const float temperature = temperature_of(a, sequence);
  if (draft && !(temperature > 0.f)) return;

  constexpr int kVector = tx::kVector<T>;
  const int first = span * kSpan<T> + lane * kVector;
  float x[kLoads][kVector];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = first + i * 64 * kVector;
    if (at + kVector <= a.vocab) {
      widen_all<T>(*reinterpret_cast<const u32x4_any *>(logits + at), x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < kVector; ++j) x[i][j] = at + j < a.vocab ? widen(logits[at + j]) : -INFINITY;
    }
  }
  float top = -INFINITY;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
#pragma unroll
    for (int j = 0; j < kVector; ++j) top = fmaxf(top, x[i][j]);
  top = wave_max(top);
  float2 *partial = a.partials + ((int64_t)(draft ? a.tokens : 0) + row) * a.spans + span;
  if (!(temperature > 0.f)) {
    int index = 0x7FFFFFFF;
#pragma unroll
    for (int i = kLoads - 1; i >= 0; --i)
#pragma unroll
      for (int j = kVector - 1; j >= 0; --j) {
        if (x[i][j] == top) index = first + i * 64 * kVector + j;
        odd |= x[i][j] != x[i][j];
      }
    index = wave_min_int(index);
    if (__builtin_amdgcn_ballot_w64(odd) != 0) top = NAN;
    if (lane == 0) *partial = make_float2(top, __int_as_float(index));
    return;
  }
  const float base = top == -INFINITY ? 0.f : top;
  const Exponents e = exponents_of(base, rate_of(temperature));
  float sum = 0.f;
  if (e.shifted) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int j = 0; j < kVector; ++j) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][j], e.low, __builtin_fmaf(x[i][j], e.high, -e.shift)));
  } else {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int j = 0; j < kVector; ++j) {
        const float below = 0.5f * x[i][j] - 0.5f * base;  // halves: finite for all that are
        sum += x[i][j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(2.f * __builtin_fmaf(below, e.high, below * e.low));
      }
  }
  sum = wave_sum(sum);
  if (lane == 0) *partial = make_float2(top, sum);
}

// How a sequence's last token is drawn.
struct Closing {
  int row;       // the last row reached, in the packed rows; -1: nothing to draw
  int first;     // the sequence's first row
  int slot;      // where the token goes
  int residual;  // drawn from max(p - q, 0)
  float top, draft_top;
  double scale_p, scale_q;  // 1 / sums of the row's p and q, by the first launch
  int removed;              // tokens that are left out
  int64_t tokens[kMostDrafts];
};

// Sums of a chunk of the last row: all weights of p and of q; of the tokens that may be drawn, those of p and of q.
struct Sums {
  double p, q, rest_p, rest_q;
};

template <typename T>
__device__ __forceinline__ float logit(const void *logits, int64_t row_stride, int64_t row, int64_t token) {
  return widen(reinterpret_cast<const T *>(logits)[row * row_stride + token]);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int w = 1; w < 64; w *= 2) v += __shfl_xor(v, w);
  return v;
}

// Tokens that a wave sums at once, eight neighbours a lane.
constexpr int kEight = 8, kChunk = 64 * kEight;
constexpr int kWalkWaves = 16;  // waves of a workgroup of the second launch

// The eight logits from `at` on, -infinity behind the last.
template <typename T>
__device__ __forceinline__ void eight_logits(const void *logits, int64_t row_stride, int64_t row, int at, int vocab, float *x) {
  const T *from = reinterpret_cast<const T *>(logits) + row * row_stride + at;
  if (at + kEight <= vocab) {
#pragma unroll
    for (int i = 0; i < kEight; i += kVector<T>) widen_all<T>(*reinterpret_cast<const u32x4_any *>(from + i), x + i);
  } else {
#pragma unroll
    for (int i = 0; i < kEight; ++i) x[i] = at + i < vocab ? widen(from[i]) : -INFINITY;
  }
}

// exp((x - top) / T) in 64 bits.
__device__ __forceinline__ double weight_of(float x, float top, double rate) {
  const double w = exp2_64(((double)x - (double)top) * rate);
  return x == -INFINITY ? 0.0 : w;
}

// Eight tokens of the last row: take(i, weight of p, weight of q, whether it may be drawn); scale_p and scale_q say where p > q.
template <typename T, typename Take>
__device__ __forceinline__ void eight_weights(const Verify &a, const Closing &c, double rate, int at, double scale_p, double scale_q, Take take) {
  float x[kEight], y[kEight];
  eight_logits<T>(a.target, a.target_row, c.row, at, a.vocab, x);
  const bool residual = __builtin_amdgcn_readfirstlane(c.residual);
  if (residual) eight_logits<T>(a.draft, a.draft_row, c.row, at, a.vocab, y);
  uint32_t out = 0;
  for (int i = 0; i < c.removed; ++i) {
    const int64_t distance = c.tokens[i] - at;
    out |= (uint64_t)distance < kEight ? 1u << distance : 0u;
  }
  // Without branches: the eight are then under way together.
  double p[kEight], q[kEight];
#pragma unroll
  for (int i = 0; i < kEight; ++i) p[i] = weight_of(x[i], c.top, rate), q[i] = 0.0;
  if (residual) {
#pragma unroll
    for (int i = 0; i < kEight; ++i) q[i] = weight_of(y[i], c.draft_top, rate);
  }
#pragma unroll
  for (int i = 0; i < kEight; ++i) {
    const bool some = !residual | (p[i] * scale_p > q[i] * scale_q);
    take(i, p[i], q[i], !(out >> i & 1) & some);
  }
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ double wave_scan64(double v, int lane) {
#pragma unroll
  for (int w = 1; w < 64; w *= 2) {
    const double other = __shfl_up(v, w);
    v += lane >= w ? other : 0.0;
  }
  return v;
}

// The first lane whose running sum exceeds `target`, the sums before it added to `before`; else the last lane with a weight, else -1.
__device__ __forceinline__ int crossing(double v, double target, double &before, int lane) {
  const double sum = before + wave_scan64(v, lane);
  const uint64_t past = __builtin_amdgcn_ballot_w64(sum > target && v > 0.0), some = __builtin_amdgcn_ballot_w64(v > 0.0);
  if (some == 0) return -1;
  const int at = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  before = __shfl(sum - v, at);
  return at;
}

// Lanes that have this lane's `bits` low bits of v.
__device__ __forceinline__ uint64_t same_lanes(int v, int bits) {
  uint64_t same = ~(uint64_t)0;
  for (int b = 0; b < bits; ++b) {
    const bool mine = v >> b & 1;
    const uint64_t set = __builtin_amdgcn_ballot_w64(mine);
    same &= mine ? set : ~set;
  }
  return same;
}

// Draws the closing token by one wave: the 512 tokens of the last row in which the running sum passes, then the token in them.
template <typename T>
__device__ __forceinline__ int64_t closing_token(const Verify &a, const Closing &closing, double rate, const Sums *sums, float uniform) {
  const int lane = threadIdx.x & 63;
  // Lane l has the chunks l * each .. of the row.
  const int each = (a.chunks + 63) / 64, first = lane * each, last = min(first + each, a.chunks);
  Sums mine = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
  for (int i = first; i < last; ++i) {
    mine.p += sums[i].p;
    mine.q += sums[i].q;
    mine.rest_p += sums[i].rest_p;
    mine.rest_q += sums[i].rest_q;
  }
  const bool residual = __builtin_amdgcn_readfirstlane(closing.residual);
  const double all_p = wave_sum64(mine.p), all_q = residual ? wave_sum64(mine.q) : 0.0;
  const double scale_p = 1.0 / all_p, scale_q = residual ? 1.0 / all_q : 0.0;
  // What counts of a sum, and whether anything does: else it is drawn from all of p.
  auto rest_of = [&](const Sums &s) { return residual ? fmax(s.rest_p * scale_p - s.rest_q * scale_q, 0.0) : s.rest_p; };
  const bool all = !(wave_sum64(rest_of(mine)) > 0.0);
  auto value_of = [&](const Sums &s) { return all ? s.p : rest_of(s); };
  // A lane's sum of the chunks from `at` on, of `run` that end before `stop`.
  auto value_from = [&](int at, int run, int stop) {
    double value = 0.0;
#pragma unroll 4
    for (int i = at; i < min(at + run, stop); ++i) value += value_of(sums[i]);
    return value;
  };
  double value = value_from(first, each, a.chunks);
  const double total = wave_sum64(value);
  if (!(total > 0.0) || (residual && !(all_q > 0.0))) return -1;
  const double target = (double)uniform * total;
  // The run of chunks in which the sum passes, then 64 runs of that, down to one chunk.
  double before = 0.0;
  int chunk = 0, run = each, stop = a.chunks;
  while (true) {
    chunk += run * max(crossing(value, target, before, lane), 0);
    if (run == 1) break;
    stop = min(chunk + run, stop);
    run = (run + 63) / 64;
    value = value_from(chunk + lane * run, run, stop);
  }
  int64_t token = -1;
  // Once more with all of p where a chunk's rest was nothing but rounding.
  for (int turn = 0; turn < 2 && token < 0; ++turn) {
    double weight[kEight], held = 0.0;
    eight_weights<T>(a, closing, rate, chunk * kChunk + lane * kEight, scale_p, scale_q, [&](int i, double p, double q, bool rest) {
      weight[i] = all || turn ? p : !rest ? 0.0 : residual ? p * scale_p - q * scale_q : p;
      held += weight[i];
    });
    double sum = before;
    const int at = crossing(held, target, sum, lane);
    bool past = false;
#pragma unroll
    for (int i = 0; i < kEight; ++i) {
      sum += weight[i];
      if (weight[i] > 0.0 && !past) {
        token = chunk * kChunk + lane * kEight + i;
        past = sum > target;
      }
    }
    token = at >= 0 ? __shfl(token, max(at, 0)) : -1;
  }
  return token;
}

// Grid: x workgroups of a sequence, y sequences.
template <typename T>
__global__ __launch_bounds__(64 * kWalkWaves) void verify_walk_kernel(Verify a) {
  __shared__ float tops[2][kMostDrafts];   // maxima of the rows; of the draft's
  __shared__ double sums[2][kMostDrafts];  // sums of their weights; at T = 0 the target's first largest token
  __shared__ Closing closing;
  __shared__ int order[kMostDrafts];  // the path's rows
  __shared__ bool ends;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sequence = blockIdx.y;
  const Rows rows = rows_of(a, sequence);
  const bool writes = blockIdx.x == 0;
  if (rows.count <= 0) {
    if (writes && threadIdx.x == 0) a.accepted[sequence] = -1;
    return;
  }
  const float temperature = temperature_of(a, sequence);
  const bool greedy = !(temperature > 0.f);
  const double rate = greedy ? 0.0 : rate_of(temperature);
  // The first wave's lane i is row i; its logits are under way while the statistics are joined.
  const bool row = wave == 0 && lane < rows.count;
  int parent = -1;
  int64_t token = -1;
  float u = 0.f, x = -INFINITY, y = -INFINITY;
  if (row) {
    parent = a.parents ? a.parents[rows.begin + lane] : lane - 1;
    token = a.ids[rows.begin + lane];
    u = a.uniforms[rows.begin + lane];
  }
  if (lane == 0 || (uint32_t)parent >= (uint32_t)rows.count) parent = -1;
  const bool child = row && parent >= 0, known = child && token >= 0 && token < a.vocab;
  if (known && !greedy) {
    x = logit<T>(a.target, a.target_row, rows.begin + parent, token);
    if (a.draft) y = logit<T>(a.draft, a.draft_row, rows.begin + parent, token);
  }
  // The rows' statistics from their spans', by 16, 32 or 64 lanes a row.
  const int kinds = a.draft && !greedy ? 2 : 1, width = a.spans <= 16 ? 16 : a.spans <= 32 ? 32 : 64;
  for (int i = threadIdx.x / width; i < rows.count * kinds; i += 64 * kWalkWaves / width) {
    const int kind = i >= rows.count, local = i - kind * rows.count, mine = lane & (width - 1);
    if (kind == 1 && local + 1 >= rows.count) continue;
    const float2 *partial = a.partials + ((int64_t)(kind ? a.tokens : 0) + rows.begin + local) * a.spans;
    constexpr int kHeld = 4;
    float2 held[kHeld];
#pragma unroll
    for (int s = 0; s < kHeld; ++s) held[s] = mine + s * width < a.spans ? partial[mine + s * width] : make_float2(-INFINITY, 0.f);
    // The rest of a vocabulary of more spans is read twice.
    auto each = [&](auto take) __attribute__((always_inline)) {
#pragma unroll
      for (int s = 0; s < kHeld; ++s) take(held[s]);
      for (int s = mine + kHeld * width; s < a.spans; s += width) take(partial[s]);
    };
    float top = -INFINITY;
    int odd = 0;
    each([&](float2 v) {
      odd |= v.x != v.x;
      top = fmaxf(top, v.x);
    });
    for (int w = 1; w < width; w *= 2) {
      top = fmaxf(top, __shfl_xor(top, w));
      odd |= __shfl_xor(odd, w);
    }
    if (greedy) {
      int index = 0x7FFFFFFF;
      each([&](float2 v) { index = v.x == top ? min(index, __float_as_int(v.y)) : index; });
      for (int w = 1; w < width; w *= 2) index = min(index, __shfl_xor(index, w));
      if (mine == 0) sums[0][local] = odd || top == -INFINITY ? -1.0 : (double)index;
    } else {
      double sum = 0.0;
      each([&](float2 v) {
        const Exponents e = exponents_of(v.x, rate);
        const double exponent = (e.shifted ? (double)e.shift : (double)v.x * rate) - (double)top * rate;
        sum += v.x == -INFINITY ? (double)v.y : (double)v.y * exp2_64(exponent);
      });
      for (int w = 1; w < width; w *= 2) sum += __shfl_xor(sum, w);
      if (mine == 0) {
        tops[kind][local] = top;
        sums[kind][local] = sum;
      }
    }
  }
  __syncthreads();
  if (wave == 0) {
    double p = 0.0, q = 0.0;
    if (known) {
      if (greedy) {
        p = sums[0][parent] == (double)token ? 1.0 : 0.0;
      } else {
        p = weight_of(x, tops[0][parent], rate) / sums[0][parent];
        if (a.draft) q = weight_of(y, tops[1][parent], rate) / sums[1][parent];
      }
    }
    // Earlier drafts behind the same row: whether one has this token, and their probabilities' sum.
    const uint64_t earlier = child ? same_lanes(parent, 7) & __builtin_amdgcn_ballot_w64(child) & (((uint64_t)1 << lane) - 1) : 0;
    const uint64_t twins = same_lanes((int)token, 31) & __builtin_amdgcn_ballot_w64(known);
    const bool again = known && (earlier & twins) != 0;
    double before = 0.0;
    uint64_t left = earlier & __builtin_amdgcn_ballot_w64(known && !again);
    while (__builtin_amdgcn_ballot_w64(left != 0) != 0) {
      const double theirs = __shfl(p, left ? __builtin_ctzll(left) : 0);
      before += left ? theirs : 0.0;
      left &= left - 1;
    }
    bool accept = p > 0.0 && !again;
    if (!greedy) accept = accept && (a.draft ? (double)u * q < p : (double)u * (1.0 - before) < p);
    // The first accepted draft behind a row is taken.
    const bool taken = accept && (earlier & __builtin_amdgcn_ballot_w64(accept)) == 0;
    const uint64_t fine = __builtin_amdgcn_ballot_w64(taken) | 1;
    // The rows that lead to each, by doubled pointers; reached: row 0 is among them and all are taken.
    uint64_t leads = (uint64_t)1 << lane;
    int up = parent;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const int from = max(up, 0);
      const uint64_t theirs = __shfl(leads, from);
      const int further = __shfl(up, from);
      leads |= up >= 0 ? theirs : 0;
      up = up >= 0 ? further : -1;
    }
    const bool reached = row && (leads & 1) && (leads & ~fine) == 0;
    const int depth = __builtin_popcountll(leads) - 1;
    const int count = __builtin_popcountll(__builtin_amdgcn_ballot_w64(reached)) - 1;  // accepted drafts
    const int last = __builtin_ctzll(__builtin_amdgcn_ballot_w64(reached && depth == count));
    const uint64_t followers = __builtin_amdgcn_ballot_w64(child && parent == last);
    if (writes) {
      order[lane] = -1;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (reached) order[depth] = lane;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const int at = order[lane], behind = order[min(lane + 1, kMostDrafts - 1)];
      const int64_t theirs = __shfl(token, max(behind, 0));
      if (row) a.path[rows.begin + lane] = at;
      if (row && lane != count) a.next[rows.begin + lane] = lane < count ? theirs : -1;
      if (lane == 0) a.accepted[sequence] = count;
    }
    if (lane == 0) {
      closing.row = greedy ? -1 : rows.begin + last;
      closing.first = rows.begin;
      closing.slot = rows.begin + count;
      closing.residual = a.draft && followers != 0;
      closing.removed = a.draft ? 0 : __builtin_popcountll(followers);
      if (!greedy) {
        closing.top = tops[0][last];
        closing.scale_p = 1.0 / sums[0][last];
        closing.draft_top = closing.residual ? tops[1][last] : 0.f;
        closing.scale_q = closing.residual ? 1.0 / sums[1][last] : 0.0;
      } else if (writes) {
        a.next[rows.begin + count] = (int64_t)sums[0][last];
      }
    }
    if (!a.draft && (followers >> lane & 1)) closing.tokens[__builtin_popcountll(followers & (((uint64_t)1 << lane) - 1))] = token;
  }
  __syncthreads();
  if (closing.row < 0) return;
  Sums *kept = reinterpret_cast<Sums *>(a.sums) + (int64_t)sequence * a.chunks;
  // Neighbouring chunks go to different workgroups: what is left for a second round is spread over all of them.
  for (int chunk = wave * a.groups + blockIdx.x; chunk < a.chunks; chunk += a.groups * kWalkWaves) {
    Sums mine = {0.0, 0.0, 0.0, 0.0};
    eight_weights<T>(a, closing, rate, chunk * kChunk + lane * kEight, closing.scale_p, closing.scale_q, [&](int, double p, double q, bool rest) {
      mine.p += p;
      mine.q += q;
      mine.rest_p += rest ? p : 0.0;
      mine.rest_q += rest ? q : 0.0;
    });
    mine.p = wave_sum64(mine.p);
    mine.rest_p = wave_sum64(mine.rest_p);
    if (closing.residual) {
      mine.q = wave_sum64(mine.q);
      mine.rest_q = wave_sum64(mine.rest_q);
    }
    if (lane == 0) kept[chunk] = mine;
  }
  // Every wave's sums have reached the cache of its die before the barrier, which does not wait for stores by itself; one thread's fence
  // behind it makes them visible to the other dies.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    ends = atomicAdd(a.counters + sequence, 1) == a.groups - 1;
  }
  __syncthreads();
  if (!ends || wave != 0) return;
  __threadfence();
  const int64_t drawn = closing_token<T>(a, closing, rate, kept, a.uniforms[closing.first]);
  if (lane == 0) a.next[closing.slot] = drawn;
}

}  // namespace

void verify_plan(Verify &a, int dtype_bytes, int cus) {
  const int span = 64 * kLoads * 16 / dtype_bytes;
  a.spans = (a.vocab + span - 1) / span;
  // Workgroups that share a sequence's last row: one a CU in all, with work for every wave.
  a.chunks = (a.vocab + kChunk - 1) / kChunk;
  const int64_t full = (int64_t)cus / (a.sequences > 0 ? a.sequences : 1), most = (a.chunks + kWalkWaves - 1) / kWalkWaves;
  a.groups = (int)(full < 1 ? 1 : full < most ? full : most);
  auto whole = [](int64_t bytes) { return (bytes + 15) & ~(int64_t)15; };
  a.counters_at = whole((int64_t)a.tokens * (a.draft ? 2 : 1) * a.spans * sizeof(float2));
  a.sums_at = a.counters_at + whole((int64_t)a.sequences * sizeof(int));
  a.workspace_bytes = a.sums_at + (int64_t)a.sequences * a.chunks * sizeof(Sums);
}

hipError_t launch_verify(Verify a, int dtype, char *workspace, hipStream_t stream) {
  a.partials = reinterpret_cast<float2 *>(workspace);
  a.counters = reinterpret_cast<int *>(workspace + a.counters_at);
  a.sums = workspace + a.sums_at;
  const dim3 stats((unsigned)((a.spans + kWaves - 1) / kWaves), (unsigned)a.tokens, a.draft ? 2 : 1);
  auto launch = [&](auto type) {
    using T = decltype(type);
    if (a.tokens > 0) hipLaunchKernelGGL(verify_stats_kernel<T>, stats, dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL(verify_walk_kernel<T>, dim3((unsigned)a.groups, (unsigned)a.sequences), dim3(64 * kWalkWaves), 0, stream, a);
  };
  if (dtype == kVerifyF32) launch(0.f);
  else if (dtype == kVerifyF16) launch(Fp16{});
  else launch(Bf16{});
  return hipGetLastError();
}

}  // namespace tx
