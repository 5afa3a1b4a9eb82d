// C-ABI entry points of the paged GQA decode over an MXFP4 cache (kernel body
// in paged_decode_mxfp4.h).
#include "mva_capi.h"
#include "paged_decode_mxfp4.h"

namespace mva {

int fill_decode_params(DecodeParams& p, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                       const void* k_cache, const void* v_cache, int64_t num_pages, int64_t page_stride,
                       int64_t token_stride, const int32_t* block_tables, int64_t block_table_stride,
                       const int32_t* seq_lens, const int32_t* items, int64_t num_items, int64_t num_waves,
                       const int32_t* wave_extra, const int32_t* merges, int64_t num_merges, int64_t num_part_slots,
                       void* out, int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                       int64_t workspace_bytes, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                       float softmax_scale);
int launch_decode_merge(const DecodeParams& p, const int32_t* merges, int64_t num_merges, int64_t num_part_slots,
                        int dtype, hipStream_t stream);

namespace {

// kWaves wavefronts per workgroup, each with private LDS buffers; wavefront w of
// workgroup b is decode wavefront b * kWaves + w.
template <typename T, int kWaves>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(3))) void paged_decode_mxfp4_kernel(
    Fp4DecodeParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves * kFp4WaveLdsBytes];
  // Tiles done by the wavefronts; one without work reads as far ahead.
  __shared__ int progress[kWaves];
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wave = (int)blockIdx.x * kWaves + w;
  if (kWaves == 12 && (threadIdx.x & 63) == 0) progress[w] = 0x3fffffff;
  if (wave >= p.num_waves) return;
  decode_wave_mxfp4<T>(p, wave, (lds_u8*)lds, kWaves == 12 ? progress : nullptr, w);
}

template <typename T>
int launch(const Fp4DecodeParams& p, int waves_per_group, hipStream_t s) {
  if (p.num_waves > (int)(0xffffffffu / 64) - 12)  // a launch has fewer than 2^32 threads
    return set_error("paged attention mxfp4: too many wavefronts");
  const uint32_t blocks = ((uint32_t)p.num_waves + waves_per_group - 1) / waves_per_group;
  switch (waves_per_group) {
    case 4: hipLaunchKernelGGL((paged_decode_mxfp4_kernel<T, 4>), dim3(blocks), dim3(256), 0, s, p); break;
    case 12: hipLaunchKernelGGL((paged_decode_mxfp4_kernel<T, 12>), dim3(blocks), dim3(768), 0, s, p); break;
    default: return set_error("paged attention mxfp4: waves_per_group must be 4 or 12");
  }
  return check_launch("paged_decode_mxfp4");
}

}  // namespace
}  // namespace mva

extern "C" int mva_paged_decode_mxfp4(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                      const void* k_cache, const void* v_cache, int64_t num_pages,
                                      int64_t page_stride_bytes, int64_t head_stride_bytes,
                                      const int32_t* block_tables, int64_t block_table_stride,
                                      const int32_t* seq_lens, const int32_t* counts, const int32_t* items,
                                      int64_t num_items, int64_t num_waves, const int32_t* wave_extra,
                                      int waves_per_group, const int32_t* merges, int64_t num_merges,
                                      int64_t num_part_slots, void* out, int64_t out_token_stride,
                                      int64_t out_head_stride, void* workspace, int64_t workspace_bytes,
                                      int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                      float softmax_scale, int dtype, void* stream) {
  using namespace mva;
  if (wave_extra == nullptr && num_items > 0) return set_error("paged attention mxfp4: piece lists (wave_extra) needed");
  if (((uint64_t)page_stride_bytes | (uint64_t)head_stride_bytes) % 16)
    return set_error("paged attention mxfp4: cache strides must be 16-byte aligned");
  if (page_stride_bytes < 0 || head_stride_bytes < 0)
    return set_error("paged attention mxfp4: cache strides must not be negative");
  if (page_stride_bytes > 0xffffffffLL)
    return set_error("paged attention mxfp4: pages must lie less than 4 GiB apart");
  if (dtype != kBF16 && dtype != kF16) return set_error("paged attention: dtype must be bf16 or fp16");
  Fp4DecodeParams p;
  const int rc = fill_decode_params(p, q, q_token_stride, q_head_stride, k_cache, v_cache, num_pages, 0, 0,
                                    block_tables, block_table_stride, seq_lens, items, num_items, num_waves,
                                    wave_extra, merges, num_merges, num_part_slots, out, out_token_stride,
                                    out_head_stride, workspace, workspace_bytes, num_q_heads, num_kv_heads, head_dim,
                                    page_size, softmax_scale);
  if (rc) return rc;
  if (num_items == 0) return 0;
  p.page_stride = page_stride_bytes;
  p.head_stride = head_stride_bytes;
  p.counts = counts;
  hipStream_t s = (hipStream_t)stream;
  const int rc_launch = dtype == kBF16 ? launch<__bf16>(p, waves_per_group, s)
                                       : launch<_Float16>(p, waves_per_group, s);
  if (rc_launch) return rc_launch;
  return launch_decode_merge(p, merges, num_merges, num_part_slots, dtype, s);
}
