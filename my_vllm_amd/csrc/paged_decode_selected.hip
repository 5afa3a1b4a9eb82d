// Decode attention over selected pages of a 16-bit cache.
//
//   o = sum_j softmax_j(scale * q . K[j]) V[j]
// over the lens[s] tokens of the pages tables[s][h][0 .. ceil(lens[s] / 16)),
// a list for each row s and KV head h; all pages but the last are full.
//
// Bound by the reads of K and V: 64 rows of 256 pages at 64 / 8 heads (1.07 GB)
// take 170 us, 6.3 TB/s.  Few pages are a chain of latencies: 1.8 us of launch, then
// lengths, page ids, pages, the join of a row's parts through memory; 128 pages of
// one row at 32 / 8 heads (8.4 MB) 7.8 us.
//
// Unlike the dense decode's ragged batches, lists are at most num_selected pages
// long, so equal parts of them need no plan: a launch is fixed by its shapes, which
// a captured graph can keep.
#include "mva_capi.h"
#include "paged_decode.h"
#include "page_selection.h"

#include <algorithm>

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
  int* counters;    // [S][Hkv], zero between launches
  int num_kv_heads;
  int group;
  float scale_log2;
};

constexpr int kSelWaves = 4;       // wavefronts of a workgroup
constexpr int kSelGroupsPerCu = 3;  // workgroups that a CU holds
// Pages of a part, at least.  A part more costs the join more than the pages it
// takes off the others' streams: 128 pages of one row at 32 / 8 heads in parts of
// 4, 8, 16 and 32 pages take 10.4, 7.9, 7.6 and 9.8 us.
constexpr int kPartPages = 16;
constexpr int kJoinRow = kHeadDim + 4;  // floats of a joined row in LDS: its 16 rows start in different banks

// Lanes 0-31 of a, then of b; and lanes 32-63 of a, then of b.
__device__ inline float lower_halves(float a, float b) {
  return __uint_as_float(__builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false)[0]);
}
__device__ inline float upper_halves(float a, float b) {
  return __uint_as_float(__builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false)[1]);
}

// A page of one KV head in registers, every load whole 128-byte lines.
// k[i]: of token 8 (i % 2) + c % 8 the channels 64 (i / 2) + 32 (c / 8) + 8 q4 .. + 7,
// an A operand of S^T = K Q^T whose rows 0-7 and 8-15 are the same tokens, over
// the channels of one half of a line and of the other.
// v[e]: channels 8 c .. 8 c + 7 of token 4 q4 + e, so that halves of v[0 .. 3] make
// the A operand of O^T += V^T P^T whose rows are the channels 8 m + i, m the row of
// the matrix instruction.
template <typename T>
struct PageRegs {
  typename Elem<T>::v8 k[4];
  u32x4 v[4];
};

// One workgroup per (row, part of its pages, KV head).  Its wavefronts take the
// part's pages in turns, each with a running maximum and sum of its own, and
// join in LDS; the row's last workgroup joins the parts.
//
// Pages come straight into registers, the next one while one is computed (150
// registers, so three wavefronts a SIMD); through LDS, 16 KB a wavefront, a CU
// would hold fewer.  A first form of eight wavefronts that loaded V element by
// element, with the joins in a second launch, took 286 us for the 1.07 GB and 21.9
// us for the one row; loads of K over half lines 173 us with V non-temporal, 188
// with both.
template <typename T>
__global__ __launch_bounds__(64 * kSelWaves, kSelGroupsPerCu) void selected_decode_kernel(SelectedParams p) {
  typedef typename Elem<T>::v8 V8;
  typedef typename Elem<T>::v4 V4;
  __shared__ __attribute__((aligned(16))) float join_o[kSelWaves][16][kJoinRow];
  __shared__ float join_m[kSelWaves][16], join_l[kSelWaves][16];
  __shared__ int join_last;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int q4 = lane >> 4, c = lane & 15;
  const int h = (int)(blockIdx.x % p.num_kv_heads);
  const int part = (int)(blockIdx.x / p.num_kv_heads % p.parts);
  const int64_t s = blockIdx.x / p.num_kv_heads / p.parts;
  const int G = p.group;
  const int len = sload(p.lens, s);
  const int pages = len <= 0 ? 0 : min((int)(((int64_t)len + kPageSize - 1) / kPageSize), p.num_selected);
  const int parts = min(p.parts, max(1, (pages + kPartPages - 1) / kPartPages));  // fewer for a row of few pages
  if (part >= parts) return;
  const int begin = (int)((int64_t)pages * part / parts), end = (int)((int64_t)pages * (part + 1) / parts);
  const int32_t* table = p.tables + s * p.seq_table_stride + h * p.head_table_stride;

  V8 qf[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    qf[j] = V8{};
    if (c < G)
      qf[j] = ld16<V8>((const T*)p.q + s * p.q_tok_stride + (int64_t)(h * G + c) * p.q_head_stride + 32 * j + 8 * q4);
  }
  f32x4 o[8];  // o[i][r] = O[g = c][channel 32 q4 + 8 r + i]
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY;  // reference maximum of the scaled scores (log2), per g = c
  float l = 0.f;        // this lane's share of the running sum

  // Byte offsets in a page, one register each beside the page's address in scalar ones.
  const uint32_t tok = (uint32_t)p.tok_stride * 2;
  const uint32_t k_off[2] = {(c & 7) * tok + 64 * (c >> 3) + 16 * q4, (8 + (c & 7)) * tok + 64 * (c >> 3) + 16 * q4};
  uint32_t v_off[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v_off[e] = (4 * q4 + e) * tok + 16 * c;
  auto load = [&](PageRegs<T>& r, int id) __attribute__((always_inline)) {
    const int64_t base = ((int64_t)id * p.page_stride + h * kHeadDim) * 2;
    const uint8_t* const k = (const uint8_t*)p.k_cache + base;
    const uint8_t* const v = (const uint8_t*)p.v_cache + base;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.k[i] = ld16_once<V8>(k + 128 * (i >> 1) + (size_t)k_off[i & 1]);
#pragma unroll
    for (int e = 0; e < 4; ++e) r.v[e] = ld16_once<u32x4>(v + (size_t)v_off[e]);
  };
  // `left`: tokens of the row from this page on (16 or more unless it is the last one).
  auto compute = [&](PageRegs<T>& r, int left, auto may_end) __attribute__((always_inline)) {
    // Rows 0-7 of near[u] and 8-15 of far[u] are the two halves of the scores of tokens 8 u .. 8 u + 7.
    f32x4 near[2] = {}, far[2] = {}, sc;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      near[i & 1] = Elem<T>::mfma16(r.k[i], qf[i & 2], near[i & 1]);
      far[i & 1] = Elem<T>::mfma16(r.k[i], qf[(i & 2) + 1], far[i & 1]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sc[e] = lower_halves(near[0][e], near[1][e]) + upper_halves(far[0][e], far[1][e]);
    // sc[e] = S[token 4 q4 + e][g = c].  Rows behind the last token, whatever they hold, do not count.
    if (decltype(may_end)::value && left < kPageSize) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (4 * q4 + e >= left) {
          sc[e] = -INFINITY;
          r.v[e] = u32x4{0u, 0u, 0u, 0u};
        }
      }
    }
    const float tmax = wave_max16(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]))) * p.scale_log2;
    // The reference is the maximum so far: the largest P are near 1, where the operand's type rounds them least.
    if (__any(tmax > m)) {
      const float m_new = fmaxf(m, tmax);
      const float alpha = fast_exp2(m - (m_new == -INFINITY ? 0.f : m_new));
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] *= alpha;
    }
    const float m_use = m == -INFINITY ? 0.f : m;
    V4 pf;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float pr = fast_exp2(sc[e] * p.scale_log2 - m_use);
      l += pr;
      pf[e] = (T)pr;  // the operand's type; the sum takes the value before it is rounded
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const u32x2 lo = {__builtin_amdgcn_perm(r.v[1][w], r.v[0][w], 0x05040100u),
                        __builtin_amdgcn_perm(r.v[3][w], r.v[2][w], 0x05040100u)};
      const u32x2 hi = {__builtin_amdgcn_perm(r.v[1][w], r.v[0][w], 0x07060302u),
                        __builtin_amdgcn_perm(r.v[3][w], r.v[2][w], 0x07060302u)};
      o[2 * w] = Elem<T>::mfma16k16(__builtin_bit_cast(V4, lo), pf, o[2 * w]);
      o[2 * w + 1] = Elem<T>::mfma16k16(__builtin_bit_cast(V4, hi), pf, o[2 * w + 1]);
    }
  };

  // This wavefront's pages begin + wave + kSelWaves * k, 64 ids at a time.
  const int mine = end - begin > wave ? (end - begin - wave + kSelWaves - 1) / kSelWaves : 0;
  for (int k0 = 0; k0 < mine; k0 += 64) {
    const int n = min(64, mine - k0);
    const int at = begin + wave + kSelWaves * k0;
    int ids = table[at + kSelWaves * min(lane, n - 1)];
    if (ids < 0 || ids >= p.num_pages) ids = 0;
    PageRegs<T> a, b;
    load(a, __builtin_amdgcn_readlane(ids, 0));
    for (int k = 1; k < n; ++k) {
      load(b, __builtin_amdgcn_readlane(ids, k));
      compute(a, kPageSize, std::false_type{});
      a = b;
    }
    compute(a, len - (at + kSelWaves * (n - 1)) * kPageSize, std::true_type{});
  }

  const float l_tot = wave_sum16(l);
  if (q4 == 0) {
    join_m[wave][c] = m;
    join_l[wave][c] = l_tot;
  }
  if (c < G) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int i = 0; i < 8; i += 4)
        *(f32x4*)&join_o[wave][c][32 * q4 + 8 * r + i] = f32x4{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
    }
  }
  __syncthreads();
  // Four channels of a query a thread, kSelWaves * 2 queries at a time.
  const int g0 = threadIdx.x / (kHeadDim / 4), d = threadIdx.x % (kHeadDim / 4) * 4;
  const int64_t slot0 = (s * p.num_kv_heads + h) * p.parts * G;
  auto write = [&](int g, f32x4 acc, float inv) {
    V4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(acc[e] * inv);
    *(V4*)((T*)p.out + s * p.out_tok_stride + (int64_t)(h * G + g) * p.out_head_stride + d) = y;
  };
  for (int g = g0; g < G; g += 2 * kSelWaves) {
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
      acc += f * *(const f32x4*)&join_o[w][g][d];
    }
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
    if (parts == 1) {
      write(g, acc, inv);
    } else {
      const int64_t slot = slot0 + part * G + g;
      store16_device_untracked(p.part_o + slot * kHeadDim + d, __builtin_bit_cast(u32x4, acc * inv));
      if (d == 0) store4_device_untracked(p.part_lse + slot, sum > 0.f ? use + fast_log2(sum) : -INFINITY);
    }
  }
  if (parts == 1) return;
  // Parts meet in memory: stores that reach it, counted in once they have, and
  // loads that come from there.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    int* counter = p.counters + s * p.num_kv_heads + h;
    const bool last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    join_last = last;
  }
  __syncthreads();
  if (!join_last) return;
  constexpr int kAtOnce = 8;
  for (int g = g0; g < G; g += 2 * kSelWaves) {
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, sum = 0.f;
    for (int k = 0; k < parts; k += kAtOnce) {
      float lse[kAtOnce];
      f32x4 rows[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int64_t slot = slot0 + min(k + i, parts - 1) * G + g;
        lse[i] = part_load<true>(p.part_lse + slot);
        rows[i] = part_load4<true>(p.part_o + slot * kHeadDim + d);
      }
      float most = top;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (k + i >= parts) lse[i] = -INFINITY;
        most = fmaxf(most, lse[i]);
      }
      const float use = most == -INFINITY ? 0.f : most;
      const float alpha = fast_exp2(top - use);
      top = most;
      sum *= alpha;
      acc *= alpha;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const float f = fast_exp2(lse[i] - use);
        sum += f;
        acc += f * rows[i];
      }
    }
    write(g, acc, sum > 0.f ? 1.0f / sum : 0.f);
  }
}

static_assert(256 * kSelGroupsPerCu <= kSelectionCounters, "a row in several parts has a counter");

// Parts a row's pages are cut into, one workgroup each: as many workgroups as
// the GPU holds, as long as a part has kPartPages pages.
int selected_parts(int64_t num_seqs, int hkv, int64_t num_selected) {
  const int64_t rows = num_seqs * hkv;
  const int64_t most = (num_selected + kPartPages - 1) / kPartPages;
  const int64_t want = rows > 0 ? 256 * kSelGroupsPerCu / rows : 1;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

}  // namespace

// Rows are cut into more parts the fewer they are, so that 64 rows can need less than
// 48.  The bytes are therefore those of a bound that does not fall as any size grows:
// in several parts a row, `parts` * rows is at most the workgroups that the GPU
// holds, each of kMaxQueryGroup queries at most.
int64_t selection_part_bytes(int64_t num_seqs, int hq, int64_t num_selected) {
  const int64_t queries = num_seqs * hq;
  const int64_t in_parts = queries * ((num_selected + kPartPages - 1) / kPartPages);
  const int64_t resident = std::max(queries, (int64_t)256 * kSelGroupsPerCu * kMaxQueryGroup);
  const int64_t slots = std::min(in_parts, resident);
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
      head_table_stride < 0 || page_stride < 0)
    return set_error("selected attention: invalid sizes");
  if (num_pages <= 0 || num_pages > 0x7fffffffLL) return set_error("selected attention: empty or oversized KV cache");
  if (!(softmax_scale > 0.f && softmax_scale < INFINITY))
    return set_error("selected attention: softmax_scale must be positive and finite");
  if (num_seqs == 0) return 0;
  if (!q || !k_cache || !v_cache || !tables || !lens || !out) return set_error("selected attention: null buffer");
  if (((uint64_t)(uintptr_t)q | (uint64_t)(uintptr_t)k_cache | (uint64_t)(uintptr_t)v_cache |
       (uint64_t)(q_token_stride * 2) | (uint64_t)(q_head_stride * 2) | (uint64_t)(page_stride * 2) |
       (uint64_t)(token_stride * 2)) % 16)
    return set_error("selected attention: q / cache buffers and strides must be 16-byte aligned");
  if (token_stride < 0 || token_stride >= (1 << 26))
    return set_error("selected attention: a page's tokens must lie less than 2^26 elements apart");
  if (((uint64_t)(uintptr_t)out | (uint64_t)(out_token_stride * 2) | (uint64_t)(out_head_stride * 2)) % 8)
    return set_error("selected attention: output buffer and strides must be 8-byte aligned");
  const int parts = selected_parts(num_seqs, num_kv_heads, num_selected);
  if (parts > 1 && (workspace == nullptr || (uint64_t)(uintptr_t)workspace % 16 ||
                    workspace_bytes < kSelectionHeaderBytes + selection_part_bytes(num_seqs, num_q_heads, num_selected)))
    return set_error("selected attention: workspace missing, too small or unaligned");
  const int64_t blocks = num_seqs * num_kv_heads * parts;
  if (blocks > 0xffffffffLL / (64 * kSelWaves)) return set_error("selected attention: too many rows for one launch");
  const int64_t slots = num_seqs * num_q_heads * parts;
  uint8_t* const ws = (uint8_t*)workspace;
  float* const part_lse = (float*)(ws + kSelectionHeaderBytes);
  const SelectedParams p = {q, q_token_stride, q_head_stride, k_cache, v_cache, num_pages, page_stride, token_stride,
                            tables, seq_table_stride, head_table_stride, lens, (int)num_selected, parts, out,
                            out_token_stride, out_head_stride, part_lse,
                            (float*)((uint8_t*)part_lse + align_up256(slots * 4)), (int*)ws + kSelectionCounters,
                            num_kv_heads, num_q_heads / num_kv_heads, softmax_scale * 1.4426950408889634f};
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == kBF16)
    hipLaunchKernelGGL(selected_decode_kernel<__bf16>, dim3((uint32_t)blocks), dim3(64 * kSelWaves), 0, st, p);
  else
    hipLaunchKernelGGL(selected_decode_kernel<_Float16>, dim3((uint32_t)blocks), dim3(64 * kSelWaves), 0, st, p);
  return check_launch("selected_decode");
}
