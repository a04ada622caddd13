// Writing, reading and moving the rows of a paged 4-bit KV cache (gfx950; layout in kv4.h).
//
// No reference counterpart: the reference's Hugging Face path keeps its caches in 16 bits.
//
// A group of 32 elements is stored as MXFP4, the rule of the activation quantizer (fp4.hip): scale exponent
// e = max(floor(log2(amax)) - 2 + 127, 0), each code the E2M1 value nearest to v * 2^(127 - e), ties to the even code,
// saturated at 6. A group that holds an infinity or a NaN gets e = 255 and reads back as NaN.
//
// All three are copies with arithmetic on the way, bound by memory; the scale and the codes of a group never leave its thread.
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

__device__ __forceinline__ Row locate(const Kv4Pool &pool, const int *cu, const int *starts, int token) {
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
  const int position = kv4_length(pool, sequence) - back;
  if (position < 0 || back <= 0 || (cu == nullptr && token >= pool.sequences)) return {-1, 0};
  const int page = pool.table[sequence * pool.table_stride + (position >> pool.page_shift)];
  if ((uint32_t)page >= (uint64_t)pool.num_pages) return {-1, 0};
  return {page, position & ((1 << pool.page_shift) - 1)};
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
