// Decode attention over selected pages of a 16-bit cache.
//
//   o = sum_j softmax_j(scale * q . K[j]) V[j]
// over the lens[s] tokens of the pages tables[s][h][0 .. ceil(lens[s] / 16)),
// a list for each row s and KV head h; all pages but the last are full.
#include "mva_capi.h"
#include "paged_decode.h"
#include "page_selection.h"

namespace mva {
namespace {

struct SelectedParams {
  const void* q;
  int64_t q_tok_stride;
  int64_t q_head_stride;
  const void* k_cache;
  const void* v_cache;
  int64_t num_pages;
  int64_t page_stride;
  int64_t tok_stride;
  const int32_t* tables;  // [S][Hkv][table_stride]
  int64_t seq_table_stride;
  int64_t head_table_stride;
  const int32_t* lens;
  int num_selected;
  int parts;
  void* out;
  int64_t out_tok_stride;
  int64_t out_head_stride;
  float* part_lse;  // [S][Hkv][parts][G]
  float* part_o;    // [S][Hkv][parts][G][128]
  int num_kv_heads;
  int group;
  float scale_log2;
};

constexpr int kSelWaves = 8;
constexpr int kSelWaveLds = 2 * kDecodePageBytes;

// One workgroup per (row, KV head, part); its wavefronts take the part's pages
// in turns, each with a running maximum and sum of its own, and join in LDS.
template <typename T>
__global__ __launch_bounds__(64 * kSelWaves) void selected_decode_kernel(SelectedParams p) {
  typedef typename Elem<T>::v8 V8;
  typedef typename Elem<T>::v4 V4;
  __shared__ __attribute__((aligned(16))) uint8_t lds_all[kSelWaves * kSelWaveLds];
  __shared__ float join_m[kSelWaves][16], join_l[kSelWaves][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int q4 = lane >> 4, c = lane & 15;
  const int h = (int)(blockIdx.x % p.num_kv_heads);
  const int part = (int)(blockIdx.x / p.num_kv_heads % p.parts);
  const int64_t s = blockIdx.x / p.num_kv_heads / p.parts;
  const int G = p.group;
  const int len = sload(p.lens, s);
  const int pages = len <= 0 ? 0 : min((int)(((int64_t)len + kPageSize - 1) / kPageSize), p.num_selected);
  const int begin = (int)((int64_t)pages * part / p.parts), end = (int)((int64_t)pages * (part + 1) / p.parts);
  const int32_t* table = p.tables + s * p.seq_table_stride + h * p.head_table_stride;

  V8 qf[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    qf[j] = V8{};
    if (c < G)
      qf[j] = ld16<V8>((const T*)p.q + s * p.q_tok_stride + (int64_t)(h * G + c) * p.q_head_stride + 32 * q4 + 8 * j);
  }
  f32x4 o[8];
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  for (int i = begin + wave; i < end; i += kSelWaves) {
    int id = sload(table, i);
    if (id < 0 || id >= p.num_pages) id = 0;
    const int64_t base = (int64_t)id * p.page_stride + h * kHeadDim;
    const int left = len - i * kPageSize;  // tokens from this page on
    // K rows as the A operand, straight from memory: lane (q4, c) token c.
    f32x4 sc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const V8 k = ld16<V8>((const T*)p.k_cache + base + c * p.tok_stride + 32 * q4 + 8 * j);
      sc = Elem<T>::mfma16(k, qf[j], sc);
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (4 * q4 + r >= left) sc[r] = -INFINITY;
      tmax = fmaxf(tmax, sc[r]);
    }
    tmax = wave_max16(tmax) * p.scale_log2;
    const float m_new = fmaxf(m, tmax);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = fast_exp2(m - m_use);
    m = m_new;
    l *= alpha;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[mt] *= alpha;
    V4 pf;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float pr = fast_exp2(sc[r] * p.scale_log2 - m_use);
      l += pr;
      pf[r] = (T)pr;
    }
    // V^T operands element by element: lane (q4, c) tokens 4 q4 .. + 3, channel 16 mt + c.
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      V4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 4 * q4 + e;
        v[e] = t < left ? ((const T*)p.v_cache)[base + t * p.tok_stride + 16 * mt + c] : (T)0.f;
      }
      o[mt] = Elem<T>::mfma16k16(v, pf, o[mt]);
    }
  }

  // Join the wavefronts: o[mt][r] = O[g = c][d = 16 mt + 4 q4 + r].
  const float l_tot = wave_sum16(l);
  if (q4 == 0) {
    join_m[wave][c] = m;
    join_l[wave][c] = l_tot;
  }
  float* mine = (float*)(lds_all + wave * kSelWaveLds);  // [g][128]
#pragma unroll
  for (int mt = 0; mt < 8; ++mt)
    if (c < G) *(f32x4*)(mine + c * kHeadDim + 16 * mt + 4 * q4) = o[mt];
  __syncthreads();
  for (int v = threadIdx.x; v < G * (kHeadDim / 4); v += 64 * kSelWaves) {
    const int g = v / (kHeadDim / 4), d = v % (kHeadDim / 4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) top = fmaxf(top, join_m[w][g]);
    const float use = top == -INFINITY ? 0.f : top;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) {
      const float f = fast_exp2(join_m[w][g] - use);
      sum += f * join_l[w][g];
      acc += f * *(const f32x4*)((const float*)(lds_all + w * kSelWaveLds) + g * kHeadDim + d);
    }
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
    if (p.parts == 1) {
      V4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(acc[e] * inv);
      *(V4*)((T*)p.out + s * p.out_tok_stride + (int64_t)(h * G + g) * p.out_head_stride + d) = y;
    } else {
      const int64_t slot = ((s * p.num_kv_heads + h) * p.parts + part) * G + g;
      *(f32x4*)(p.part_o + slot * kHeadDim + d) = acc * inv;
      if (d == 0) p.part_lse[slot] = sum > 0.f ? use + fast_log2(sum) : -INFINITY;
    }
  }
}

// One wavefront per (row, query head): the parts of a row joined.
template <typename T>
__global__ __launch_bounds__(256) void selected_merge_kernel(SelectedParams p, int64_t rows) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // (s, h, g)
  if (row >= rows) return;
  const int g = (int)(row % p.group);
  const int64_t sh = row / p.group;
  float top = -INFINITY;
  for (int k = 0; k < p.parts; ++k) top = fmaxf(top, p.part_lse[(sh * p.parts + k) * p.group + g]);
  const float use = top == -INFINITY ? 0.f : top;
  float sum = 0.f, a = 0.f, b = 0.f;
  for (int k = 0; k < p.parts; ++k) {
    const int64_t slot = (sh * p.parts + k) * p.group + g;
    const float f = fast_exp2(p.part_lse[slot] - use);
    sum += f;
    a += f * p.part_o[slot * kHeadDim + 2 * lane];
    b += f * p.part_o[slot * kHeadDim + 2 * lane + 1];
  }
  const float inv = sum > 0.f ? 1.0f / sum : 0.f;
  T* out = (T*)p.out + sh / p.num_kv_heads * p.out_tok_stride +
           (sh % p.num_kv_heads * p.group + g) * p.out_head_stride + 2 * lane;
  out[0] = (T)(a * inv);
  out[1] = (T)(b * inv);
}

// Parts a row's pages are cut into, one workgroup each: enough workgroups for
// 256 CUs, as long as every wavefront has a page.
int selected_parts(int64_t num_seqs, int hkv, int64_t num_selected) {
  const int64_t rows = num_seqs * hkv;
  const int64_t most = (num_selected + kSelWaves - 1) / kSelWaves;
  const int64_t want = rows > 0 ? (256 + rows - 1) / rows : 1;
  return (int)(want < most ? want : most);
}

}  // namespace

int64_t selection_part_bytes(int64_t num_seqs, int hq, int hkv, int64_t num_selected) {
  const int64_t slots = num_seqs * hq * selected_parts(num_seqs, hkv, num_selected);
  return align_up256(slots * 4) + align_up256(slots * kHeadDim * 4);
}

}  // namespace mva

extern "C" int mva_paged_decode_selected(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                         const void* k_cache, const void* v_cache, int64_t num_pages,
                                         int64_t page_stride, int64_t token_stride, const int32_t* tables,
                                         int64_t seq_table_stride, int64_t head_table_stride, const int32_t* lens,
                                         int64_t num_seqs, int64_t num_selected, void* out, int64_t out_token_stride,
                                         int64_t out_head_stride, void* workspace, int64_t workspace_bytes,
                                         int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                         float softmax_scale, int dtype, void* stream) {
  using namespace mva;
  if (head_dim != kHeadDim || page_size != kPageSize)
    return set_error("selected attention: head_dim must be 128, page_size 16");
  if (dtype != kBF16 && dtype != kF16) return set_error("selected attention: dtype must be bf16 or fp16");
  if (!selection_sizes_ok(num_seqs, num_q_heads, num_kv_heads, num_selected) || seq_table_stride < 0 ||
      head_table_stride < 0)
    return set_error("selected attention: invalid sizes");
  if (num_pages <= 0 || num_pages > 0x7fffffffLL) return set_error("selected attention: empty or oversized KV cache");
  if (num_seqs == 0) return 0;
  if (!q || !k_cache || !v_cache || !tables || !lens || !out) return set_error("selected attention: null buffer");
  if (((uint64_t)(uintptr_t)q | (uint64_t)(uintptr_t)k_cache | (uint64_t)(uintptr_t)v_cache |
       (uint64_t)(q_token_stride * 2) | (uint64_t)(q_head_stride * 2) | (uint64_t)(page_stride * 2) |
       (uint64_t)(token_stride * 2)) % 16)
    return set_error("selected attention: q / cache buffers and strides must be 16-byte aligned");
  if (((uint64_t)(uintptr_t)out | (uint64_t)(out_token_stride * 2) | (uint64_t)(out_head_stride * 2)) % 8)
    return set_error("selected attention: output buffer and strides must be 8-byte aligned");
  const int parts = selected_parts(num_seqs, num_kv_heads, num_selected);
  if (parts > 1 && (workspace == nullptr || (uint64_t)(uintptr_t)workspace % 16 ||
                    workspace_bytes < selection_part_bytes(num_seqs, num_q_heads, num_kv_heads, num_selected)))
    return set_error("selected attention: workspace missing, too small or unaligned");
  const int64_t blocks = num_seqs * num_kv_heads * parts;
  if (blocks > 0xffffffffLL / (64 * kSelWaves)) return set_error("selected attention: too many rows for one launch");
  const int64_t slots = num_seqs * num_q_heads * parts;
  SelectedParams p = {q, q_token_stride, q_head_stride, k_cache, v_cache, num_pages, page_stride, token_stride, tables,
                      seq_table_stride, head_table_stride, lens, (int)num_selected, parts, out, out_token_stride,
                      out_head_stride, (float*)workspace, (float*)((uint8_t*)workspace + align_up256(slots * 4)),
                      num_kv_heads, num_q_heads / num_kv_heads, softmax_scale * 1.4426950408889634f};
  const hipStream_t st = (hipStream_t)stream;
  const int64_t rows = num_seqs * num_q_heads;
  if (dtype == kBF16) {
    hipLaunchKernelGGL(selected_decode_kernel<__bf16>, dim3((uint32_t)blocks), dim3(64 * kSelWaves), 0, st, p);
    if (parts > 1)
      hipLaunchKernelGGL(selected_merge_kernel<__bf16>, dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, st, p, rows);
  } else {
    hipLaunchKernelGGL(selected_decode_kernel<_Float16>, dim3((uint32_t)blocks), dim3(64 * kSelWaves), 0, st, p);
    if (parts > 1)
      hipLaunchKernelGGL(selected_merge_kernel<_Float16>, dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, st, p, rows);
  }
  return check_launch("selected_decode");
}
