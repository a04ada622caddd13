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

// Sum of count(s) over all sequences; every wave computes it alone.
template <typename Count>
__device__ __forceinline__ int ragged_total(int sequences, Count count) {
  const int lane = threadIdx.x & 63;
  int total = 0;
  for (int first = 0; first < sequences; first += 64) {
    const int n = first + lane < sequences ? count(first + lane) : 0;
    total += __builtin_amdgcn_readlane(wave_scan(n), 63);
  }
  return total;
}

// The sequence that holds item `target` of all sequences' items in order, and the item's number within it;
// false past the last one. `before`: items of the earlier sequences.
template <typename Count>
__device__ __forceinline__ bool ragged_find(int sequences, int target, Count count, int &sequence, int &local) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int first = 0; first < sequences; first += 64) {
    const int n = first + lane < sequences ? count(first + lane) : 0;
    const int sum = wave_scan(n);
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (target < before + total) {
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > target - before));
      sequence = first + at;
      local = target - before - __builtin_amdgcn_readlane(sum - n, at);
      return true;
    }
    before += total;
  }
  return false;
}

}  // namespace tx
