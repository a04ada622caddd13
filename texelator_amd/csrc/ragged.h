// Device helpers for batches of sequences of different lengths whose lengths lie in device memory: a workgroup
// finds its share of the work by itself, so that a launch (or a captured graph) serves any lengths.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tx {

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// All sequences' items in one row: how many there are, and where one of them lies.
struct RaggedPlace {
  int total;     // items of all sequences
  int sequence;  // the sequence that holds the item asked for (the last one's number past the end)
  int local;     // the item's number in it
  int length;    // that sequence's length
};

// The item `target(total)`, where sequence s has count(length(s)) items. Every wave finds it alone; up to 64 sequences
// each length is loaded once.
template <typename Length, typename Count, typename Target>
__device__ __forceinline__ RaggedPlace ragged_place(int sequences, Length length, Count count, Target target) {
  const int lane = threadIdx.x & 63;
  auto length_at = [&](int s) { return s < sequences ? length(s) : 0; };
  auto count_at = [&](int s, int l) { return s < sequences ? count(l) : 0; };
  const int l0 = length_at(lane), n0 = count_at(lane, l0);
  const int sum0 = wave_scan(n0);
  int total = __builtin_amdgcn_readlane(sum0, 63);
  for (int first = 64; first < sequences; first += 64)
    total += __builtin_amdgcn_readlane(wave_scan(count_at(first + lane, length_at(first + lane))), 63);
  const int wanted = target(total);
  RaggedPlace place = {total, sequences - 1, 0, 0};
  int before = 0;
  for (int first = 0; first < sequences; first += 64) {
    const int l = first == 0 ? l0 : length_at(first + lane);
    const int n = first == 0 ? n0 : count_at(first + lane, l);
    const int sum = first == 0 ? sum0 : wave_scan(n);
    const uint64_t past = __builtin_amdgcn_ballot_w64(sum > wanted - before);
    if (past) {
      const int at = __builtin_ctzll(past);
      place.sequence = first + at;
      place.local = wanted - before - __builtin_amdgcn_readlane(sum - n, at);
      place.length = __builtin_amdgcn_readlane(l, at);
      break;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return place;
}

// Largest value of the lanes of a wave.
__device__ __forceinline__ int wave_max_int(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(v, 63);
}

// The item at rank target(total), heaviest first, where item i of sequence s weighs i + offset(s); up to 64 sequences
// (beyond, the sequences keep their order and each its heaviest items first).
template <typename Length, typename Count, typename Offset, typename Target>
__device__ __forceinline__ RaggedPlace ragged_heaviest(int sequences, Length length, Count count, Offset offset, Target target) {
  if (sequences > 64) {
    RaggedPlace place = ragged_place(sequences, length, count, target);
    place.local = count(place.length) - 1 - place.local;
    return place;
  }
  const int lane = threadIdx.x & 63;
  const int l = lane < sequences ? length(lane) : 0;
  const int n = lane < sequences ? count(l) : 0, o = lane < sequences ? offset(lane) : 0;
  const int total = __builtin_amdgcn_readlane(wave_scan(n), 63);
  const int rank = target(total);
  if (sequences == 1) return {total, 0, total - 1 - rank, __builtin_amdgcn_readlane(l, 0)};
  // Weights of at least `low` belong to more than `rank` items, of at least `high` to `heavier` <= rank of them.
  int low = -wave_max_int(n > 0 ? -o : -(1 << 30)), high = wave_max_int(n > 0 ? n + o : -(1 << 30)), heavier = 0;
  if (rank >= total) return {total, 0, 0, 0};
  while (high - low > 1) {
    const int mid = low + ((high - low) >> 1);
    const int items = __builtin_amdgcn_readlane(wave_scan(min(max(n + o - mid, 0), n)), 63);
    if (items > rank) low = mid;
    else high = mid, heavier = items;
  }
  const bool has = low >= o && low < n + o;
  const int among = wave_scan(has ? 1 : 0);  // with every lane: a lane left out would break the sums
  const uint64_t here = __builtin_amdgcn_ballot_w64(has && among == rank - heavier + 1);
  const int sequence = here ? __builtin_ctzll(here) : 0;
  return {total, sequence, low - __builtin_amdgcn_readlane(o, sequence), __builtin_amdgcn_readlane(l, sequence)};
}

// The items in all, and in `local` those before sequence `s`.
template <typename Length, typename Count>
__device__ __forceinline__ RaggedPlace ragged_before(int sequences, Length length, Count count, int s) {
  const int lane = threadIdx.x & 63;
  RaggedPlace place = {0, s, 0, 0};
  for (int first = 0; first < sequences; first += 64) {
    const int l = first + lane < sequences ? length(first + lane) : 0;
    const int n = first + lane < sequences ? count(l) : 0;
    const int sum = wave_scan(n);
    if (s >= first && s < first + 64) {
      place.local = place.total + __builtin_amdgcn_readlane(sum - n, s - first);
      place.length = __builtin_amdgcn_readlane(l, s - first);
    }
    place.total += __builtin_amdgcn_readlane(sum, 63);
  }
  return place;
}

}  // namespace tx
