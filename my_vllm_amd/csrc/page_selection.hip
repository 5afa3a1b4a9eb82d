// Page bounds and page selection for decode over a part of a 16-bit cache.
//
// page_bounds [P][Hkv][2][128] holds, for every full page, the smallest and
// the largest value of each channel of its 16 keys, in the keys' own type (no
// rounding).  For the G queries that share KV head h of row s, the score
//   score[s, h, j] = sum_d P[d] hi[j, h, d] + N[d] lo[j, h, d],
//   P = sum_g max(q_g, 0),  N = sum_g min(q_g, 0),
// is at least sum_g q_g . k for every key k of page j, and costs one dot
// product of length 256 whatever G is.  Selected are the first `sink` pages,
// the last `recent` and, of those between, the ones of the highest score.
#include "mva_capi.h"
#include "mva_common.h"
#include "page_selection.h"

namespace mva {
namespace {

typedef short s16x8v __attribute__((ext_vector_type(8)));

// ---- bounds --------------------------------------------------------------------

struct BoundsParams {
  const uint8_t* k_cache;
  int64_t num_pages;
  int64_t page_stride;  // bytes
  int64_t tok_stride;   // bytes
  uint8_t* bounds;
  const int32_t* block_tables;
  int64_t bt_stride;
  int64_t width;
  const int32_t* seq_lens;
  const int32_t* query_start_loc;  // nullptr: one token a sequence
  int64_t num_seqs;
  int64_t num_tokens;
  int num_kv_heads;
};

// The order of the values as that of signed 16-bit integers: an involution.
__device__ inline s16x8v ordered(s16x8v b) { return b ^ ((b >> 15) & (short)0x7fff); }

// Whether the 16-bit pattern is a NaN of a type whose infinity is `kInf`.
template <int kInf>
__device__ inline s16x8v nan_mask(s16x8v b) {
  return (b & (short)0x7fff) > (short)kInf;
}

constexpr int kBoundsTokens = 16;  // tokens whose pages one wavefront looks after

// One wavefront per (16 tokens of the step, KV head).  Lane t finds the page
// that token t completes, if any; then, page by page, lane (r, c) = (lane / 16,
// lane % 16) reads channels 8c .. 8c + 7 of rows r, r + 4, r + 8 and r + 12.
template <int kInf>
__global__ __launch_bounds__(256) void page_bounds_kernel(BoundsParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t chunk = unit / p.num_kv_heads;
  const int h = (int)(unit % p.num_kv_heads);
  if (chunk * kBoundsTokens >= p.num_tokens) return;
  int64_t page = -1;
  const int64_t t = chunk * kBoundsTokens + lane;
  if (lane < kBoundsTokens && t < p.num_tokens) {
    int64_t s = t, place = 0, count = 1;
    if (p.query_start_loc != nullptr) {
      // The last sequence that starts at or before token t.
      int64_t lo = 0, hi = p.num_seqs;
      while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (p.query_start_loc[mid] <= t) lo = mid;
        else hi = mid;
      }
      s = lo;
      place = t - p.query_start_loc[s];
      count = (int64_t)p.query_start_loc[s + 1] - p.query_start_loc[s];
    }
    if (place >= 0 && place < count) {
      const int64_t pos = (int64_t)p.seq_lens[s] - count + place;
      if (pos >= 0 && pos % kPageTokens == kPageTokens - 1 && pos / kPageTokens < p.width) {
        page = p.block_tables[s * p.bt_stride + pos / kPageTokens];
        if (page >= p.num_pages) page = -1;
      }
    }
  }
  for (uint64_t todo = __ballot(page >= 0); todo != 0; todo &= todo - 1) {
    const int from = __builtin_ctzll(todo);
    const int64_t id = __shfl((int)page, from);
    const int r = lane >> 4, c = lane & 15;
    const uint8_t* src = p.k_cache + id * p.page_stride + r * p.tok_stride + h * 256 + c * 16;
    s16x8v rows[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rows[i] = ld16<s16x8v>(src + 4 * i * p.tok_stride);
    s16x8v lo = ordered(rows[0]), hi = lo;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      const s16x8v v = ordered(rows[i]);
      lo = __builtin_elementwise_min(lo, v);
      hi = __builtin_elementwise_max(hi, v);
    }
#pragma unroll
    for (int x = 16; x <= 32; x += 16) {
      u32x4 a = __builtin_bit_cast(u32x4, lo), b = __builtin_bit_cast(u32x4, hi);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = __shfl_xor(a[e], x);
        b[e] = __shfl_xor(b[e], x);
      }
      lo = __builtin_elementwise_min(lo, __builtin_bit_cast(s16x8v, a));
      hi = __builtin_elementwise_max(hi, __builtin_bit_cast(s16x8v, b));
    }
    lo = ordered(lo);
    hi = ordered(hi);
    // A NaN is the largest or the smallest of its column by its sign: both bounds become NaN.
    const s16x8v bad = nan_mask<kInf>(lo) | nan_mask<kInf>(hi);
    lo |= bad & (short)0x7fff;
    hi |= bad & (short)0x7fff;
    if (lane < 32) st16(p.bounds + ((id * p.num_kv_heads + h) * 2 + r) * 256 + c * 16, r == 0 ? lo : hi);
  }
}

// ---- scores --------------------------------------------------------------------

struct SelectParams {
  const void* q;
  int64_t q_tok_stride;
  int64_t q_head_stride;
  const uint8_t* bounds;
  int64_t num_pages;
  const int32_t* block_tables;
  int64_t bt_stride;
  int64_t width;
  const int32_t* seq_lens;
  int64_t num_seqs;
  int num_selected;
  int sink;
  int recent;
  int32_t* tables;
  int32_t* lens;
  uint64_t* keys;  // [S][Hkv][width]
  int* counters;   // [S][Hkv], zero between launches
  int num_kv_heads;
  int group;
};

// Tokens of row s, within what its block table holds.
__device__ inline int64_t row_tokens(const SelectParams& p, int64_t s) {
  const int64_t len = p.seq_lens[s];
  return len < 0 ? 0 : min(len, p.width * kPageTokens);
}

// Keys of the order in which pages are taken: a score's order as an unsigned
// integer, the two zeros alike, NaN above everything.
__device__ inline uint64_t order_key(double score) {
  if (score != score) return ~uint64_t(0);
  const uint64_t b = __builtin_bit_cast(uint64_t, score + 0.0);
  return (int64_t)b < 0 ? ~b : b | (uint64_t(1) << 63);
}

constexpr int kSelectThreads = 256;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kBatch = 16;       // pages that a wavefront scores at a time
constexpr int kShortKeys = 512;  // keys held in LDS where one workgroup scores a row
constexpr int kKeyRegs = 8;      // keys that a thread of the choice holds in registers

// Workgroup state of the choice.
struct ChoiceLds {
  uint64_t keys[kShortKeys];
  int hist[256];
  int found[3];
  uint32_t differ[kSelectWaves][2];
  int last;
  int counts[kSelectWaves * kKeyRegs];
};

// Keys go from the workgroups that score a row to the one that chooses, in any
// XCD: stores that reach memory and loads that come from there.
__device__ inline void key_store(uint64_t* a, uint64_t key) {
  __hip_atomic_store(a, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline uint64_t key_load(const uint64_t* a) {
  return __hip_atomic_load(a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Adds up eight values of 32 lanes each: of v[i] the sum over the lanes of this
// half, in the lanes of index i = lane / 4 % 8 (bits 4, 3, 2 from the top).
__device__ inline double sums_of_8(double (&v)[8], int lane) {
#pragma unroll
  for (int step = 0; step < 3; ++step) {
    const int x = 16 >> step, n = 4 >> step;
    const bool up = lane & x;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const double send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor(send, x);
    }
  }
  v[0] += __shfl_xor(v[0], 2);
  return v[0] + __shfl_xor(v[0], 1);
}

// The place-th key and page of the pages between the ends.
struct Scored {
  const uint64_t* keys;  // in memory, or nullptr: in LDS
  const int32_t* row;    // page ids from the first one between the ends on
  int64_t count;
};

// The threshold of the `want` largest keys: a key is taken if key >> shift is
// above `top`, and the first `want` (as returned) of those that equal it.
// each(f) calls f(key) for every key of this thread.
//
// Digit by digit from the highest bit in which keys differ, each by a histogram
// of the keys that agree with the digits before, until a digit's keys are all
// taken.
template <typename Each>
__device__ inline void threshold(Each each, uint64_t some, ChoiceLds& lds, int& want, uint64_t& top, int& shift) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint64_t differ = 0;
  each([&](uint64_t key) { differ |= key ^ some; });
  uint32_t lo = (uint32_t)differ, hi = (uint32_t)(differ >> 32);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    lo |= __shfl_xor(lo, x);
    hi |= __shfl_xor(hi, x);
  }
  if (lane == 0) {
    lds.differ[wave][0] = lo;
    lds.differ[wave][1] = hi;
  }
  lds.hist[tid] = 0;
  __syncthreads();
  differ = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) differ |= (uint64_t)lds.differ[w][1] << 32 | lds.differ[w][0];
  int end = differ ? 64 - __builtin_clzll(differ) : 0;  // bits from here up are the same in all keys
  shift = end;
  top = end == 64 ? 0 : some >> end;
  bool all = false;
  while (shift > 0 && !all) {
    end = shift;
    shift = end > 8 ? end - 8 : 0;
    const uint64_t mask = (uint64_t(1) << (end - shift)) - 1;
    each([&](uint64_t key) {
      if (end == 64 || key >> end == top) atomicAdd(&lds.hist[(int)(key >> shift & mask)], 1);
    });
    __syncthreads();
    if (wave == 0) {
      // Lane l holds digits 255 - 4l down to 252 - 4l.
      int mine[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += mine[i] = lds.hist[255 - 4 * lane - i];
      int before = sum;
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) {
        const int other = __shfl_up(before, x);
        if (lane >= x) before += other;
      }
      before -= sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < want && before + mine[i] >= want) {
          lds.found[0] = 255 - 4 * lane - i;
          lds.found[1] = want - before;
          lds.found[2] = mine[i];
        }
        before += mine[i];
      }
    }
    __syncthreads();
    top = top << (end - shift) | (uint64_t)lds.found[0];
    want = lds.found[1];
    all = lds.found[2] == want;
    lds.hist[tid] = 0;
    __syncthreads();
  }
}

// Chooses `want` of the scored pages and lists them in the order of their
// places; all threads of the workgroup, the keys visible to them.
__device__ inline void choose(const Scored& r, int want, int32_t* out, ChoiceLds& lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  uint64_t top;
  int shift;
  if (r.count <= kKeyRegs * kSelectThreads) {
    uint64_t key[kKeyRegs];
    int32_t id[kKeyRegs];
#pragma unroll
    for (int i = 0; i < kKeyRegs; ++i) {
      const int64_t j = i * kSelectThreads + tid;
      key[i] = 0;
      id[i] = 0;
      if (j < r.count) {
        key[i] = r.keys == nullptr ? lds.keys[j & (kShortKeys - 1)] : key_load(r.keys + j);
        id[i] = r.row[j];
      }
    }
    const uint64_t some = r.keys == nullptr ? lds.keys[0] : key_load(r.keys);
    threshold(
        [&](auto f) {
#pragma unroll
          for (int i = 0; i < kKeyRegs; ++i)
            if (i * kSelectThreads + tid < r.count) f(key[i]);
        },
        some, lds, want, top, shift);
    // Keys above and at the threshold, low and high half: first of each 64 places, then before each.
    uint64_t gts[kKeyRegs], eqs[kKeyRegs];
#pragma unroll
    for (int i = 0; i < kKeyRegs; ++i) {
      const bool in = i * kSelectThreads + tid < r.count;
      const uint64_t k = key[i] >> shift;
      gts[i] = __ballot(in && k > top);
      eqs[i] = __ballot(in && k == top);
      if (lane == 0) lds.counts[i * kSelectWaves + wave] = __popcll(gts[i]) | __popcll(eqs[i]) << 16;
    }
    __syncthreads();
    int mine = lane < kSelectWaves * kKeyRegs ? lds.counts[lane] : 0;
    const int own = mine;
#pragma unroll
    for (int x = 1; x < kSelectWaves * kKeyRegs; x <<= 1) {
      const int other = __shfl_up(mine, x);
      if (lane >= x) mine += other;
    }
    mine -= own;
#pragma unroll
    for (int i = 0; i < kKeyRegs; ++i) {
      const int before = __builtin_amdgcn_readlane(mine, i * kSelectWaves + wave);
      const int a = (before & 0xffff) + __popcll(gts[i] & below), b = (before >> 16) + __popcll(eqs[i] & below);
      if ((gts[i] >> lane & 1) || ((eqs[i] >> lane & 1) && b < want)) out[a + min(b, want)] = id[i];
    }
    return;
  }
  threshold(
      [&](auto f) {
        for (int64_t j = tid; j < r.count; j += kSelectThreads) f(key_load(r.keys + j));
      },
      key_load(r.keys), lds, want, top, shift);
  int above = 0, equal = 0;  // over the places before this block
  for (int64_t base = 0; base < r.count; base += kSelectThreads) {
    const int64_t j = base + tid;
    const uint64_t key = j < r.count ? key_load(r.keys + j) >> shift : 0;
    const uint64_t gts = __ballot(j < r.count && key > top), eqs = __ballot(j < r.count && key == top);
    if (lane == 0) {
      lds.counts[2 * wave] = __popcll(gts);
      lds.counts[2 * wave + 1] = __popcll(eqs);
    }
    __syncthreads();
    int a = above + __popcll(gts & below), b = equal + __popcll(eqs & below);
#pragma unroll
    for (int w = 0; w < kSelectWaves; ++w) {
      if (w < wave) {
        a += lds.counts[2 * w];
        b += lds.counts[2 * w + 1];
      }
      above += lds.counts[2 * w];
      equal += lds.counts[2 * w + 1];
    }
    if ((gts >> lane & 1) || ((eqs >> lane & 1) && b < want)) out[a + min(b, want)] = r.row[j];
    __syncthreads();
  }
}

// One workgroup per (row, `chunk` pages between the ends, KV head): its
// wavefronts score 16 pages at a time; the row's last workgroup to have scored
// its pages chooses.
//
// Lanes 0-31 take one page's 512 bytes and lanes 32-63 the next one's, 16 bytes
// a lane: lane % 32 / 16 the minima or the maxima, lane % 16 the channels.
// Products and sums are in 64 bits: products of 16-bit values are exact there
// and sums of them nearly so, so that which page is taken does not hang on the
// order of a sum.
template <typename T>
__global__ __launch_bounds__(kSelectThreads) void page_select_kernel(SelectParams p, int chunk, int chunks) {
  typedef typename Elem<T>::v8 V8;
  __shared__ ChoiceLds lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = (int)(blockIdx.x % p.num_kv_heads);
  const int part = (int)(blockIdx.x / p.num_kv_heads % chunks);
  const int64_t s = blockIdx.x / p.num_kv_heads / chunks;
  const int64_t len = row_tokens(p, s);
  const int64_t n = (len + kPageTokens - 1) / kPageTokens;
  const int taken = (int)min(n, (int64_t)p.num_selected);
  const int32_t* row = p.block_tables + s * p.bt_stride;
  int32_t* out = p.tables + (s * p.num_kv_heads + h) * (int64_t)p.num_selected;
  const bool whole = n <= p.num_selected;
  if (part == 0) {
    if (h == 0 && tid == 0) p.lens[s] = (int32_t)(len - kPageTokens * (n - taken));
    const int first = whole ? taken : p.sink;
    for (int i = tid; i < first; i += kSelectThreads) out[i] = row[i];
    for (int i = taken + tid; i < p.num_selected; i += kSelectThreads) out[i] = -1;
    if (!whole)
      for (int i = tid; i < p.recent; i += kSelectThreads) out[taken - p.recent + i] = row[n - p.recent + i];
  }
  const int want = p.num_selected - p.sink - p.recent;
  if (whole || want <= 0) return;
  const int64_t count = n - p.sink - p.recent;
  const int64_t parts = (count + chunk - 1) / chunk;
  if (part >= parts) return;
  const int64_t first = (int64_t)part * chunk, last = min(first + chunk, count);
  const bool in_lds = parts == 1 && count <= kShortKeys;
  uint64_t* keys = p.keys + (s * p.num_kv_heads + h) * p.width;
  row += p.sink;

  const int piece = lane & 31, half = lane >> 5;
  double w[8] = {};
  for (int g = 0; g < p.group; ++g) {
    const V8 q = ld16<V8>((const T*)p.q + s * p.q_tok_stride + (int64_t)(h * p.group + g) * p.q_head_stride +
                          8 * (piece & 15));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = (float)q[e];
      // A NaN stays in both parts.
      w[e] += (double)(piece < 16 ? (x > 0.f ? 0.f : x) : (x < 0.f ? 0.f : x));
    }
  }
  const uint8_t* bounds = p.bounds + h * 512 + piece * 16;
  for (int64_t base = first + wave * kBatch; base < last; base += kSelectWaves * kBatch) {
    int id = row[min(base + (lane & 15), last - 1)];
    if (id < 0 || id >= p.num_pages) id = 0;
    V8 box[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t a = __builtin_amdgcn_readlane(id, 2 * i), b = __builtin_amdgcn_readlane(id, 2 * i + 1);
      box[i] = ld16<V8>(bounds + (half ? b : a) * ((int64_t)p.num_kv_heads * 512));
    }
    double sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum[i] = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[i] = __builtin_fma((double)(float)box[i][e], w[e], sum[i]);
    }
    const uint64_t key = order_key(sums_of_8(sum, lane));
    const int64_t place = base + 2 * (piece >> 2) + half;
    if ((lane & 3) == 0 && place < last) {
      if (in_lds) lds.keys[place] = key;
      else key_store(keys + place, key);
    }
  }
  if (parts > 1) {
    // This wavefront's keys have reached memory before the workgroup counts itself in.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      int* counter = p.counters + s * p.num_kv_heads + h;
      const bool is_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
      if (is_last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      lds.last = is_last;
    }
    __syncthreads();
    if (!lds.last) return;
  } else {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }
  choose({in_lds ? nullptr : keys, row, count}, want, out + p.sink, lds);
}

}  // namespace

int64_t selection_keys_bytes(int64_t num_seqs, int hkv, int64_t width) { return align_up256(num_seqs * hkv * width * 8); }

}  // namespace mva

extern "C" int mva_update_page_bounds(const void* k_cache, int64_t num_pages, int64_t page_stride,
                                      int64_t token_stride, void* page_bounds, const int32_t* block_tables,
                                      int64_t block_table_stride, int64_t table_width, const int32_t* seq_lens,
                                      const int32_t* query_start_loc, int64_t num_seqs, int64_t num_tokens,
                                      int num_kv_heads, int head_dim, int page_size, int dtype, void* stream) {
  using namespace mva;
  if (head_dim != 128 || page_size != kPageTokens) return set_error("page bounds: head_dim must be 128, page_size 16");
  if (dtype != kBF16 && dtype != kF16) return set_error("page bounds: dtype must be bf16 or fp16");
  if (num_kv_heads <= 0 || num_pages < 0 || num_pages > 0x7fffffffLL || num_seqs < 0 || num_tokens < 0 ||
      table_width < 0 || block_table_stride < 0)
    return set_error("page bounds: invalid sizes");
  if (query_start_loc == nullptr && num_tokens != num_seqs)
    return set_error("page bounds: without query_start_loc every sequence has one token");
  if (num_seqs == 0 || num_tokens == 0 || num_pages == 0 || table_width == 0) return 0;
  if (!k_cache || !page_bounds || !block_tables || !seq_lens) return set_error("page bounds: null buffer");
  if (((uint64_t)(uintptr_t)k_cache | (uint64_t)(uintptr_t)page_bounds | (uint64_t)(page_stride * 2) |
       (uint64_t)(token_stride * 2)) % 16)
    return set_error("page bounds: cache and bounds must be 16-byte aligned");
  const int64_t blocks = ((num_tokens + kBoundsTokens - 1) / kBoundsTokens * num_kv_heads + 3) / 4;
  if (blocks > 0xffffffffLL / 256) return set_error("page bounds: too many tokens for one launch");
  const BoundsParams p = {(const uint8_t*)k_cache, num_pages, page_stride * 2, token_stride * 2, (uint8_t*)page_bounds,
                          block_tables, block_table_stride, table_width, seq_lens, query_start_loc, num_seqs,
                          num_tokens, num_kv_heads};
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == kBF16) hipLaunchKernelGGL(page_bounds_kernel<0x7f80>, dim3((uint32_t)blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(page_bounds_kernel<0x7c00>, dim3((uint32_t)blocks), dim3(256), 0, st, p);
  return check_launch("page_bounds");
}

extern "C" int64_t mva_selection_workspace_bytes(int64_t num_seqs, int num_q_heads, int num_kv_heads,
                                                 int64_t table_width, int64_t num_selected) {
  using namespace mva;
  if (!selection_sizes_ok(num_seqs, num_q_heads, num_kv_heads, num_selected) || table_width < 0 ||
      table_width > 0x7fffffffLL / kPageTokens)
    return -1;
  return kSelectionHeaderBytes + selection_part_bytes(num_seqs, num_q_heads, num_kv_heads, num_selected) +
         selection_keys_bytes(num_seqs, num_kv_heads, table_width);
}

extern "C" int mva_select_pages(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* page_bounds,
                                int64_t num_pages, const int32_t* block_tables, int64_t block_table_stride,
                                int64_t table_width, const int32_t* seq_lens, int64_t num_seqs, int64_t num_selected,
                                int64_t sink_pages, int64_t recent_pages, int32_t* tables, int32_t* lens,
                                void* workspace, int64_t workspace_bytes, int num_q_heads, int num_kv_heads,
                                int head_dim, int page_size, int dtype, void* stream) {
  using namespace mva;
  if (head_dim != 128 || page_size != kPageTokens) return set_error("page selection: head_dim must be 128, page_size 16");
  if (dtype != kBF16 && dtype != kF16) return set_error("page selection: dtype must be bf16 or fp16");
  const int64_t need = mva_selection_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, table_width, num_selected);
  if (need < 0) return set_error("page selection: invalid sizes");
  if (sink_pages < 0 || recent_pages < 1 || sink_pages > num_selected || recent_pages > num_selected - sink_pages)
    return set_error("page selection: needs recent_pages >= 1 and sink_pages + recent_pages <= num_selected");
  if (block_table_stride < 0 || num_pages < 0 || num_pages > 0x7fffffffLL)
    return set_error("page selection: invalid sizes");
  if (num_seqs == 0) return 0;
  if (!q || !page_bounds || !block_tables || !seq_lens || !tables || !lens)
    return set_error("page selection: null buffer");
  if (num_pages == 0 || table_width == 0) return set_error("page selection: empty KV cache");
  if (workspace == nullptr || workspace_bytes < need) return set_error("page selection: workspace too small");
  if (((uint64_t)(uintptr_t)q | (uint64_t)(uintptr_t)page_bounds | (uint64_t)(uintptr_t)workspace |
       (uint64_t)(q_token_stride * 2) | (uint64_t)(q_head_stride * 2)) % 16)
    return set_error("page selection: q, bounds, workspace and strides must be 16-byte aligned");
  const int64_t rows = num_seqs * num_kv_heads;
  uint8_t* const ws = (uint8_t*)workspace;
  const SelectParams p = {
      q, q_token_stride, q_head_stride, (const uint8_t*)page_bounds, num_pages, block_tables, block_table_stride,
      table_width, seq_lens, num_seqs, (int)num_selected, (int)sink_pages, (int)recent_pages, tables, lens,
      (uint64_t*)(ws + kSelectionHeaderBytes + selection_part_bytes(num_seqs, num_q_heads, num_kv_heads, num_selected)),
      (int*)ws, num_kv_heads, num_q_heads / num_kv_heads};
  // Chunks: as small as 64 pages (16 a wavefront) as long as that makes no more
  // workgroups than the GPU holds at a time; one a row beyond the counters.
  const int64_t most = table_width - sink_pages - recent_pages;
  int64_t chunk = 64;
  while (chunk < most && (rows > kSelectionCounters || rows * ((most + chunk - 1) / chunk) > 2048)) chunk *= 2;
  const int64_t chunks = most > chunk && table_width > num_selected ? (most + chunk - 1) / chunk : 1;
  const int64_t blocks = rows * chunks;
  if (blocks > 0xffffffffLL / kSelectThreads) return set_error("page selection: too many rows for one launch");
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == kBF16)
    hipLaunchKernelGGL(page_select_kernel<__bf16>, dim3((uint32_t)blocks), dim3(kSelectThreads), 0, st, p, (int)chunk,
                       (int)chunks);
  else
    hipLaunchKernelGGL(page_select_kernel<_Float16>, dim3((uint32_t)blocks), dim3(kSelectThreads), 0, st, p,
                       (int)chunk, (int)chunks);
  return check_launch("page_select");
}
