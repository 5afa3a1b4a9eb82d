// The MXFP4 KV cache's writer and reader (format: mxfp4.h).
//
// Store: every group of 32 elements x of a K or V row becomes codes
// rne(x / 2^e) and the byte e + 127, where 2^e is the smallest power of two
// with max|x| <= 7 * 2^e: the largest element is then off by at most one unit
// 2^e (half its step), where the smallest 2^e with max|x| < 8 * 2^e would cut
// values up to 7.99 down to 6.  Division by a power of two is exact, so a code
// depends on one rounding only.  e stops at 125 (bf16) or 13 (fp16), which
// keeps every value read back finite in the row's type.  A group that holds an
// infinity or a NaN becomes byte 255 (NaN) with codes 0.
//
// Both are bound by memory (324 bytes a row of one KV head): 16 lanes take a
// row, 16 bytes of bf16/fp16 and 4 bytes of codes a lane; a group's maximum is
// two lane exchanges away.  A workgroup takes 16 or 64 tokens of one head, so the
// codes of consecutive tokens leave as whole lines.
//
// Measured, kernels, 8 KV heads, K and V, microseconds, with all data in memory / in the
// 256 MB last-level cache (one set of rows and results again and again): 16384 tokens (85
// MB) in runs of 1024 slots stored in 18.9 / 15.5 and read back in 21.5 / 14.7, at random slots
// 25.9 / 16.8 and 28.2 / 18.2; 30001 of one sequence (156 MB) 30.3 / 24.5 and 34.9 / 24.2: 4.5
// TB/s from memory, where a large copy reaches 4.7.  61 tokens 2.7 and 2.8, launch latency.
#include "mva_capi.h"
#include "mxfp4.h"

namespace mva {
namespace {

constexpr int kRowLanes = 16;
constexpr int kRowsPerBlock = 16;

// Maximum of both 16-bit halves over the four lanes of a group.
__device__ inline uint32_t group_max(uint32_t m) {
  m = max(m, (uint32_t)__shfl_xor((int)m, 1));
  return max(m, (uint32_t)__shfl_xor((int)m, 2));
}

// Where a slot's row of one head lies, or false: a negative slot or one past the cache.
template <typename SlotT>
__device__ inline bool slot_block(SlotT slot, int64_t num_pages, int64_t page_stride, int64_t head_stride, int head,
                                  int64_t& block, int& token) {
  const int64_t page = (int64_t)slot >> 4;
  token = (int)slot & (kFp4PageTokens - 1);
  block = page * page_stride + head * head_stride;
  return (int64_t)slot >= 0 && page < num_pages;
}

// The tokens of a workgroup, kRows times 16, of one head of K or V: consecutive
// workgroups take the K heads and the V heads of the same tokens, whose rows lie
// side by side.
struct RowBlock {
  int64_t token;  // this thread's first
  int head;
  bool is_v;
};
template <int kRows>
__device__ inline RowBlock row_block(int num_heads) {
  const int which = (int)(blockIdx.x % (uint32_t)(2 * num_heads));
  const int64_t chunk = blockIdx.x / (uint32_t)(2 * num_heads);
  return {chunk * (kRows * kRowsPerBlock) + threadIdx.x / kRowLanes, which >= num_heads ? which - num_heads : which,
          which >= num_heads};
}

template <typename T, typename SlotT, int kRows>
__global__ __launch_bounds__(kRowLanes* kRowsPerBlock) void kv_store_mxfp4_kernel(
    const T* __restrict__ key, int64_t key_stride, int64_t key_head_stride, const T* __restrict__ value,
    int64_t value_stride, int64_t value_head_stride, uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache,
    int64_t num_pages, int64_t page_stride, int64_t head_stride, const SlotT* __restrict__ slots, int64_t num_tokens,
    int num_heads) {
  typedef Fp4<T> F;
  const int sub = threadIdx.x & (kRowLanes - 1);
  const RowBlock at = row_block<kRows>(num_heads);
  const T* rows = (at.is_v ? value + at.head * value_head_stride : key + at.head * key_head_stride) + 8 * sub;
  const int64_t stride = at.is_v ? value_stride : key_stride;
  uint8_t* const cache = at.is_v ? v_cache : k_cache;
  u32x4 x[kRows];
  int64_t slot[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    // The 16 lanes of a row agree; past the last token it is read again.
    const int64_t t = at.token + r * kRowsPerBlock;
    const int64_t in = t < num_tokens ? t : num_tokens - 1;
    x[r] = ld16<u32x4>(rows + in * stride);
    slot[r] = t < num_tokens ? (int64_t)slots[in] : -1;
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    int64_t block;
    int token;
    const bool kept = slot_block(slot[r], num_pages, page_stride, head_stride, at.head, block, token);
    // Magnitudes order as their bits do, in both halves of a word.
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max((x[r][i] >> 16) & 0x7fffu, x[r][i] & 0x7fffu));
    m = group_max(m);
    const bool finite = m < F::kInfBits;
    // The exponent of the maximum, one more where its mantissa is above 1.75;
    // 4 and 7 lie two binades above 1.
    const int e = (int)((F::f32_bits(m) + 0x1fffffu) >> 23) - 2;
    const uint32_t byte = finite ? (uint32_t)min(max(e, 0), F::kMaxScale) : 255u;
    const float scale = byte == 0 ? 0x1p-127f : fp4_scale(byte);
    uint32_t codes = 0;
    if (finite) {
      codes = F::template pack<0>(codes, x[r][0], scale);
      codes = F::template pack<1>(codes, x[r][1], scale);
      codes = F::template pack<2>(codes, x[r][2], scale);
      codes = F::template pack<3>(codes, x[r][3], scale);
    }
    if (!kept) continue;
    uint8_t* dst = cache + block;
    *(uint32_t*)(dst + token * kFp4RowBytes + 4 * sub) = codes;
    if ((sub & 3) == 0) dst[kFp4ScaleOffset + token * kFp4RowScales + (sub >> 2)] = (uint8_t)byte;
  }
}

template <typename T, typename SlotT, int kRows>
__global__ __launch_bounds__(kRowLanes* kRowsPerBlock) void kv_load_mxfp4_kernel(
    T* __restrict__ key, int64_t key_stride, int64_t key_head_stride, T* __restrict__ value, int64_t value_stride,
    int64_t value_head_stride, const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
    int64_t num_pages, int64_t page_stride, int64_t head_stride, const SlotT* __restrict__ slots, int64_t num_tokens,
    int num_heads) {
  const int sub = threadIdx.x & (kRowLanes - 1);
  const RowBlock at = row_block<kRows>(num_heads);
  T* rows = (at.is_v ? value + at.head * value_head_stride : key + at.head * key_head_stride) + 8 * sub;
  const int64_t stride = at.is_v ? value_stride : key_stride;
  const uint8_t* const cache = at.is_v ? v_cache : k_cache;
  int64_t slot[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t t = at.token + r * kRowsPerBlock;
    slot[r] = t < num_tokens ? (int64_t)slots[t] : -1;
  }
  uint32_t codes[kRows], byte[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    int64_t block;
    int token;
    codes[r] = 0;
    byte[r] = 127;
    if (slot_block(slot[r], num_pages, page_stride, head_stride, at.head, block, token)) {
      const uint8_t* src = cache + block;
      codes[r] = *(const uint32_t*)(src + token * kFp4RowBytes + 4 * sub);
      byte[r] = src[kFp4ScaleOffset + token * kFp4RowScales + (sub >> 2)];
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t t = at.token + r * kRowsPerBlock;
    if (t < num_tokens) st16(rows + t * stride, fp4_unpack8<T>(codes[r], fp4_scale(byte[r])));
  }
}

// Rows a thread takes: four in flight where that leaves enough workgroups to
// fill the chip, one otherwise.  8 KV heads, microseconds, one / four: 8192 tokens (2048
// workgroups of four) stored 10.8 / 9.9, read back 10.1 / 8.9; 2048 tokens 4.0 / 4.5 and
// 4.5 / 4.4; 61 tokens 2.7 / 3.4 and 2.4 / 2.8.
constexpr int kManyRows = 4;
constexpr int64_t kManyBlocks = 2048;

// Launches `go(rows a thread, blocks, first token, tokens)` for all tokens: one
// launch has fewer than 2^32 threads.
template <typename Go>
void launch_rows(int64_t num_tokens, int num_heads, Go go) {
  const int64_t wide = (num_tokens + kManyRows * kRowsPerBlock - 1) / (kManyRows * kRowsPerBlock) * 2 * num_heads;
  const int rows = wide >= kManyBlocks ? kManyRows : 1;
  const int64_t per_block = rows * kRowsPerBlock;
  const int64_t most = (int64_t(0xffffff) / (2 * num_heads)) * per_block;  // tokens of one launch
  for (int64_t first = 0; first < num_tokens; first += most) {
    const int64_t tokens = num_tokens - first < most ? num_tokens - first : most;
    go(rows, (uint32_t)((tokens + per_block - 1) / per_block * 2 * num_heads), first, tokens);
  }
}

// The checks that both directions share; *rc is set when the call ends here.
bool rows_ready(const void* key, int64_t ks, int64_t khs, const void* value, int64_t vs, int64_t vhs,
                const void* k_cache, const void* v_cache, int64_t num_pages, int64_t page_stride, int64_t head_stride,
                const void* slots, int64_t num_tokens, int num_kv_heads, int head_dim, int dtype, int* rc) {
  *rc = 0;
  auto fail = [&](const char* what) {
    *rc = set_error(what);
    return false;
  };
  if (num_tokens < 0 || num_kv_heads <= 0 || num_pages < 0) return fail("kv cache mxfp4: invalid sizes");
  if (head_dim != 4 * kFp4Group) return fail("kv cache mxfp4: head_dim must be 128");
  if (dtype != kBF16 && dtype != kF16) return fail("kv cache mxfp4: dtype must be bf16 or fp16");
  if (num_tokens == 0) return false;
  if (num_kv_heads > 32767) return fail("kv cache mxfp4: at most 32767 KV heads");
  if (num_tokens > (int64_t(1) << 40)) return fail("kv cache mxfp4: too many tokens");
  if (!key || !value || !slots || (num_pages > 0 && (!k_cache || !v_cache)))
    return fail("kv cache mxfp4: null buffer");
  if (((uint64_t)(uintptr_t)key | (uint64_t)(uintptr_t)value | (uint64_t)(ks * 2) | (uint64_t)(khs * 2) |
       (uint64_t)(vs * 2) | (uint64_t)(vhs * 2)) % 16)
    return fail("kv cache mxfp4: key / value rows must be 16-byte aligned");
  if (((uint64_t)(uintptr_t)k_cache | (uint64_t)(uintptr_t)v_cache | (uint64_t)page_stride | (uint64_t)head_stride) % 16)
    return fail("kv cache mxfp4: cache buffers and strides must be 16-byte aligned");
  if (page_stride < 0 || head_stride < 0) return fail("kv cache mxfp4: cache strides must not be negative");
  return true;
}

}  // namespace
}  // namespace mva

extern "C" int mva_kv_store_mxfp4(const void* key, int64_t key_token_stride, int64_t key_head_stride,
                                  const void* value, int64_t value_token_stride, int64_t value_head_stride,
                                  void* k_cache, void* v_cache, int64_t num_pages, int64_t page_stride_bytes,
                                  int64_t head_stride_bytes, const void* slot_mapping, int slot_is_int64,
                                  int64_t num_tokens, int num_kv_heads, int head_dim, int dtype, void* stream) {
  using namespace mva;
  int rc;
  if (!rows_ready(key, key_token_stride, key_head_stride, value, value_token_stride, value_head_stride, k_cache,
                  v_cache, num_pages, page_stride_bytes, head_stride_bytes, slot_mapping, num_tokens, num_kv_heads,
                  head_dim, dtype, &rc))
    return rc;
  if (num_pages == 0) return 0;
  auto go = [&](auto type, auto slot) {
    typedef decltype(type) T;
    typedef decltype(slot) S;
    launch_rows(num_tokens, num_kv_heads, [&](int rows, uint32_t blocks, int64_t first, int64_t tokens) {
      auto kernel = rows == 1 ? kv_store_mxfp4_kernel<T, S, 1> : kv_store_mxfp4_kernel<T, S, kManyRows>;
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kRowLanes * kRowsPerBlock), 0, (hipStream_t)stream,
                         (const T*)key + first * key_token_stride, key_token_stride, key_head_stride,
                         (const T*)value + first * value_token_stride, value_token_stride, value_head_stride,
                         (uint8_t*)k_cache, (uint8_t*)v_cache, num_pages, page_stride_bytes, head_stride_bytes,
                         (const S*)slot_mapping + first, tokens, num_kv_heads);
    });
  };
  if (dtype == kBF16) slot_is_int64 ? go(__bf16{}, int64_t{}) : go(__bf16{}, int32_t{});
  else slot_is_int64 ? go(_Float16{}, int64_t{}) : go(_Float16{}, int32_t{});
  return check_launch("kv_store_mxfp4");
}

extern "C" int mva_kv_load_mxfp4(void* key, int64_t key_token_stride, int64_t key_head_stride, void* value,
                                 int64_t value_token_stride, int64_t value_head_stride, const void* k_cache,
                                 const void* v_cache, int64_t num_pages, int64_t page_stride_bytes,
                                 int64_t head_stride_bytes, const void* slot_mapping, int slot_is_int64,
                                 int64_t num_tokens, int num_kv_heads, int head_dim, int dtype, void* stream) {
  using namespace mva;
  int rc;
  if (!rows_ready(key, key_token_stride, key_head_stride, value, value_token_stride, value_head_stride, k_cache,
                  v_cache, num_pages, page_stride_bytes, head_stride_bytes, slot_mapping, num_tokens, num_kv_heads,
                  head_dim, dtype, &rc))
    return rc;
  auto go = [&](auto type, auto slot) {
    typedef decltype(type) T;
    typedef decltype(slot) S;
    launch_rows(num_tokens, num_kv_heads, [&](int rows, uint32_t blocks, int64_t first, int64_t tokens) {
      auto kernel = rows == 1 ? kv_load_mxfp4_kernel<T, S, 1> : kv_load_mxfp4_kernel<T, S, kManyRows>;
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kRowLanes * kRowsPerBlock), 0, (hipStream_t)stream,
                         (T*)key + first * key_token_stride, key_token_stride, key_head_stride,
                         (T*)value + first * value_token_stride, value_token_stride, value_head_stride,
                         (const uint8_t*)k_cache, (const uint8_t*)v_cache, num_pages, page_stride_bytes, head_stride_bytes,
                         (const S*)slot_mapping + first, tokens, num_kv_heads);
    });
  };
  if (dtype == kBF16) slot_is_int64 ? go(__bf16{}, int64_t{}) : go(__bf16{}, int32_t{});
  else slot_is_int64 ? go(_Float16{}, int64_t{}) : go(_Float16{}, int32_t{});
  return check_launch("kv_load_mxfp4");
}
