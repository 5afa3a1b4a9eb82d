// Page bounds and page selection for decode over a part of a 16-bit cache.
//
// page_bounds [P][Hkv][2][128] holds, for every full page, the smallest and
// the largest value of each channel of its 16 keys, in the keys' own type (no
// rounding).  For the G queries that share KV head h of row s, the score
//   score[s, h, j] = sum_d P[d] hi[j, h, d] + N[d] lo[j, h, d],
//   P = sum_g max(q_g, 0),  N = sum_g min(q_g, 0),
// is at least sum_g q_g . k for every key k of page j, and costs one dot
// product of length 256 whatever G is.  It stands for sum_g sum_d of the larger of
// q_g lo and q_g hi; where a bound or a query is infinite, 0 of P or N times it would
// not, and such pages are scored again.  Selected are the first `sink` pages,
// the last `recent` and, of those between, the ones of the highest score.
#include "mva_capi.h"
#include "mva_common.h"
#include "page_selection.h"

#include <type_traits>

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

constexpr int kInfBF16 = 0x7f80, kInfF16 = 0x7c00;  // bits of the infinities
constexpr int kBoundsTokens = 16;  // tokens whose pages one wavefront looks after

// The sequence of each token first + lane (lanes below kBoundsTokens), the
// token's place in it and the sequence's new tokens, from starts [S + 1] that do
// not fall; all lanes.
struct TokenOf {
  int64_t seq;
  int place, count;
};
__device__ inline TokenOf token_of(const int32_t* starts, int64_t num_seqs, int64_t first, int lane) {
  // A sequence that starts at or before `first`, less than 62 from the last one
  // that does: 64 starts a step.
  int64_t lo = 0, hi = num_seqs;
  while (hi - lo > 62) {
    const int64_t step = (hi - lo + 63) / 64;
    const int64_t at = lo + lane * step;
    const int below = __popcll(__ballot(at < hi && starts[min(at, hi - 1)] <= first));
    lo += max(below - 1, 0) * step;
    hi = min(hi, lo + step);
  }
  // The starts from there on tell each token's sequence.
  const int mine = starts[min(lo + lane, num_seqs)];
  int later = 0;
#pragma unroll
  for (int k = 0; k < kBoundsTokens; ++k) {
    const int n = __popcll(__ballot(lane > 0 && lo + lane < num_seqs && mine <= first + k));
    if (lane == k) later = n;
  }
  if (__any(lane < kBoundsTokens && later >= 62)) {
    // It may lie beyond the starts that were read: each lane searches for itself.
    lo = 0, hi = num_seqs;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (starts[mid] <= first + lane) lo = mid;
      else hi = mid;
    }
    return {lo, (int)(first + lane - starts[lo]), starts[lo + 1] - starts[lo]};
  }
  const int start = __shfl(mine, later), end = __shfl(mine, later + 1);
  return {lo + later, (int)(first + lane - start), end - start};
}

// One wavefront per (16 tokens of the step, KV head).  Lane t finds the page
// that token t completes, if any; then, page by page, lane (r, c) = (lane / 16,
// lane % 16) reads channels 8c .. 8c + 7 of rows r, r + 4, r + 8 and r + 12.
//
// Bound by the reads of K where many pages are completed (16384 tokens at 8 KV
// heads, 38 MB: 9.9 us, of them 1.8 of launch), by the chain starts - length - page id
// - rows - bounds where few are (61 sequences of one token: 5.1 us).  16 tokens a
// wavefront: of consecutive positions exactly one page's end.  Values are compared
// as integers, two a lane's register; a search of the starts lane by lane took
// 0.2 us longer at 61 sequences.
template <int kInf>
__device__ inline void bounds_of_tokens(const BoundsParams& p, int64_t unit, int lane) {
  const int64_t first = unit / p.num_kv_heads * kBoundsTokens;
  const int h = (int)(unit % p.num_kv_heads);
  if (first >= p.num_tokens) return;
  TokenOf of = {first + lane, 0, 1};
  if (p.query_start_loc != nullptr) of = token_of(p.query_start_loc, p.num_seqs, first, lane);
  int page = -1;
  if (lane < kBoundsTokens && first + lane < p.num_tokens && of.place >= 0 && of.place < of.count) {
    const int64_t pos = (int64_t)p.seq_lens[of.seq] - of.count + of.place;
    if (pos >= 0 && pos % kPageTokens == kPageTokens - 1 && pos / kPageTokens < p.width) {
      page = p.block_tables[of.seq * p.bt_stride + pos / kPageTokens];
      if (page >= p.num_pages) page = -1;
    }
  }
  for (uint64_t todo = __ballot(page >= 0); todo != 0; todo &= todo - 1) {
    const int from = __builtin_ctzll(todo);
    const int64_t id = __builtin_amdgcn_readlane(page, from);
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

template <int kInf>
__global__ __launch_bounds__(256) void page_bounds_kernel(BoundsParams p) {
  bounds_of_tokens<kInf>(p, (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
                         threadIdx.x & 63);
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

constexpr int kSelectThreads = 512;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kSelectGroups = 2 * 256;  // workgroups that the GPU holds, two on each of its CUs
static_assert(kSelectGroups <= kSelectionCounters, "a row in several workgroups has a counter");
constexpr int kBatch = 16;        // pages that a wavefront scores at a time
constexpr int kShortKeys = 8192;  // keys held in LDS where one workgroup scores a row
constexpr int kKeyRegs = 4;       // keys that a thread of the choice holds in registers

// Workgroup state of the choice.
struct ChoiceLds {
  uint64_t keys[kShortKeys];
  int hist[3][256];  // in turns
  uint64_t differ[kSelectWaves];
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

// The value of the lane whose number differs in bit X (within 32 lanes).
template <int X>
__device__ inline double across(double v) {
  const u32x2 b = __builtin_bit_cast(u32x2, v);
  u32x2 r;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if constexpr (X == 1) r[e] = __builtin_amdgcn_update_dpp(0, b[e], 0xb1, 0xf, 0xf, true);       // quad_perm 1 0 3 2
    else if constexpr (X == 2) r[e] = __builtin_amdgcn_update_dpp(0, b[e], 0x4e, 0xf, 0xf, true);  // quad_perm 2 3 0 1
    else if constexpr (X == 8) r[e] = __builtin_amdgcn_update_dpp(0, b[e], 0x128, 0xf, 0xf, true);  // row_ror 8
    else r[e] = __builtin_amdgcn_ds_swizzle(b[e], X << 10 | 0x1f);
  }
  return __builtin_bit_cast(double, r);
}
template <int X>
__device__ inline double halves(double a, double b, bool up) {
  return (up ? b : a) + across<X>(up ? a : b);
}

// Adds up eight values of 32 lanes each: of v[i] the sum over the lanes of this
// half, in the lanes of index i = lane / 4 % 8 (bits 4, 3, 2 from the top).
__device__ inline double sums_of_8(const double (&v)[8], int lane) {
  const bool b4 = lane & 16, b3 = lane & 8, b2 = lane & 4;
  const double x0 = halves<16>(v[0], v[4], b4), x1 = halves<16>(v[1], v[5], b4);
  const double x2 = halves<16>(v[2], v[6], b4), x3 = halves<16>(v[3], v[7], b4);
  const double y0 = halves<8>(x0, x2, b3), y1 = halves<8>(x1, x3, b3);
  double z = halves<4>(y0, y1, b2);
  z += across<2>(z);
  return z + across<1>(z);
}

// Within a wavefront by DPP: of lane l the value of lane l - 1, 2, 4, 8 of its row of
// 16, then of the rows before; 0 where there is none.
template <int Ctrl, int Rows>
__device__ inline int from_before(int x) {
  return __builtin_amdgcn_update_dpp(0, x, Ctrl, Rows, 0xf, true);
}
template <typename Op>
__device__ inline int wave_scan(int x, Op op) {
  x = op(x, from_before<0x111, 0xf>(x));
  x = op(x, from_before<0x112, 0xf>(x));
  x = op(x, from_before<0x114, 0xf>(x));
  x = op(x, from_before<0x118, 0xf>(x));
  x = op(x, from_before<0x142, 0xa>(x));  // the last lane of the row before, into rows 1 and 3
  return op(x, from_before<0x143, 0xc>(x));  // lane 31, into rows 2 and 3
}
__device__ inline int wave_scan_add(int x) {
  return wave_scan(x, [](int a, int b) { return a + b; });
}
__device__ inline uint32_t wave_or(uint32_t x) {
  return __builtin_amdgcn_readlane(wave_scan((int)x, [](int a, int b) { return a | b; }), 63);
}

// The pages between the ends: their keys, in memory or (nullptr) in LDS, and ids.
struct Scored {
  const uint64_t* keys;
  const int32_t* row;
  int64_t count;
  __device__ uint64_t key(const ChoiceLds& lds, int64_t j) const {
    return keys == nullptr ? lds.keys[j] : key_load(keys + j);
  }
};

// The threshold of the `want` largest keys: a key is taken if key >> shift is
// above `top`, and the first `want` (as returned) of those that equal it.
// each(f) calls f(key) for every key of this thread; `some` is any of the keys.
//
// Digit by digit from the highest bit in which keys differ, each by a histogram
// of the keys that agree with the digits before, until a digit's keys are all
// taken.  Every wavefront reads the histogram for itself, so a digit costs one
// barrier; the next one's is cleared meanwhile.
template <typename Each>
__device__ inline void threshold(Each each, uint64_t some, ChoiceLds& lds, int& want, uint64_t& top, int& shift) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint64_t differ = 0;
  each([&](uint64_t key) { differ |= key ^ some; });
  differ = (uint64_t)wave_or((uint32_t)(differ >> 32)) << 32 | wave_or((uint32_t)differ);
  if (lane == 0) lds.differ[wave] = differ;
  if (tid < 256) lds.hist[0][tid] = 0;
  __syncthreads();
  differ = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) differ |= lds.differ[w];
  int end = differ ? 64 - __builtin_clzll(differ) : 0;  // bits from here up are the same in all keys
  shift = end;
  top = end == 64 ? 0 : some >> end;
  bool all = false;
  for (int turn = 0; shift > 0 && !all; turn = turn == 2 ? 0 : turn + 1) {
    int* const hist = lds.hist[turn];
    end = shift;
    shift = end > 8 ? end - 8 : 0;
    const uint64_t mask = (uint64_t(1) << (end - shift)) - 1;
    each([&](uint64_t key) {
      if (end == 64 || key >> end == top) atomicAdd(&hist[(int)(key >> shift & mask)], 1);
    });
    if (tid < 256) lds.hist[turn == 2 ? 0 : turn + 1][tid] = 0;  // last read two barriers ago
    __syncthreads();
    // Lane l holds digits 252 - 4l .. 255 - 4l; `before`: keys of larger digits.
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const i32x4 mine = *(const i32x4*)&hist[252 - 4 * lane];
    const int sum = mine[0] + mine[1] + mine[2] + mine[3];
    int before = wave_scan_add(sum) - sum;
    const uint64_t holds = __ballot(before < want && before + sum >= want);
    int digit = 255 - 4 * lane, keys = mine[3];
#pragma unroll
    for (int i = 2; i >= 0; --i) {
      if (before + keys < want) {
        before += keys;
        digit = 252 - 4 * lane + i;
        keys = mine[i];
      }
    }
    const int from = __builtin_ctzll(holds);
    want -= __builtin_amdgcn_readlane(before, from);
    top = top << (end - shift) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(digit, from);
    all = __builtin_amdgcn_readlane(keys, from) == want;
  }
}

// Chooses `want` of the scored pages and lists them in the order of their
// places; all threads of the workgroup, the keys visible to them.  Nothing is
// written beyond `want` entries, whatever a launch that should not overlap does
// to keys in memory.
__device__ inline void choose(const Scored& r, int want, int32_t* out, ChoiceLds& lds) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const int room = want;
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
        key[i] = r.key(lds, j);
        id[i] = r.row[j];
      }
    }
    threshold(
        [&](auto f) {
#pragma unroll
          for (int i = 0; i < kKeyRegs; ++i)
            if (i * kSelectThreads + tid < r.count) f(key[i]);
        },
        r.key(lds, 0), lds, want, top, shift);
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
    mine = wave_scan_add(mine) - mine;
#pragma unroll
    for (int i = 0; i < kKeyRegs; ++i) {
      const int before = __builtin_amdgcn_readlane(mine, i * kSelectWaves + wave);
      const int a = (before & 0xffff) + __popcll(gts[i] & below), b = (before >> 16) + __popcll(eqs[i] & below);
      const int at = a + min(b, want);
      if (((gts[i] >> lane & 1) || ((eqs[i] >> lane & 1) && b < want)) && at < room) out[at] = id[i];
    }
    return;
  }
  threshold(
      [&](auto f) {
        for (int64_t j = tid; j < r.count; j += kSelectThreads) f(r.key(lds, j));
      },
      r.key(lds, 0), lds, want, top, shift);
  int above = 0, equal = 0;  // over the places before this block
  for (int64_t base = 0; base < r.count; base += kSelectThreads) {
    const int64_t j = base + tid;
    const uint64_t key = j < r.count ? r.key(lds, j) >> shift : 0;
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
    const int at = a + min(b, want);
    if (((gts >> lane & 1) || ((eqs >> lane & 1) && b < want)) && at < room) out[at] = r.row[j];
    __syncthreads();
  }
}

// One workgroup per (row, `chunk` pages between the ends, KV head): its
// wavefronts score 16 pages at a time; the row's last workgroup to have scored
// its pages chooses.
//
// Bound by the reads of the bounds on large batches (56 rows of 8192-32768 tokens at
// 64 / 8 heads, 324 MB: 69 us, 4.7 TB/s over the launch; its reads alone 62).  Small
// ones are a chain of latencies (one row of 30001 tokens at 32 / 8 heads, 7.7 MB:
// 9.7 us): launch and length 2.0, page ids 0.5, bounds 2.7, keys counted in 1.4,
// choice 2.8.  Two launches with the keys in memory between them and one page at a
// time took 132 and 35.5 us.
//
// Workgroups from `blocks` on write the bounds of the pages that the rows' last
// tokens complete.  Such a page is its row's last and is not scored, so a decode
// step of different sequences needs no launch before this one for them.
//
// Lanes 0-31 take one page's 512 bytes and lanes 32-63 the next one's, 16 bytes
// a lane: lane % 32 / 16 the minima or the maxima, lane % 16 the channels.
// Products and sums are in 64 bits and round there (P and N are sums of up to 16
// queries, a score of 256 products), all in one order: pages of equal bounds have equal
// scores wherever they lie, and scores whose sums are exact, as those of whole numbers
// are, tie where they are equal.  Other scores may round apart by 2^-48 of the sum of
// their terms' sizes (at most 28 roundings of 2^-53).  Sums in 32 bits instead take 67.2 us of the 69.9 and 11.4 of 13.0 at 37 rows.
template <typename T>
__global__ __launch_bounds__(kSelectThreads) void page_select_kernel(SelectParams p, int chunk, int chunks,
                                                                    uint32_t blocks, BoundsParams update) {
  typedef typename Elem<T>::v8 V8;
  __shared__ ChoiceLds lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (blockIdx.x >= blocks) {
    constexpr int kInf = std::is_same<T, __bf16>::value ? kInfBF16 : kInfF16;
    bounds_of_tokens<kInf>(update, (int64_t)(blockIdx.x - blocks) * kSelectWaves + wave, lane);
    return;
  }
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
  auto weights = [&]() __attribute__((always_inline)) {
    const float sign = piece < 16 ? -1.f : 1.f;  // the negative or the positive parts
    const T* q = (const T*)p.q + s * p.q_tok_stride + (int64_t)h * p.group * p.q_head_stride + 8 * (piece & 15);
    for (int g = 0; g < p.group; g += 4) {
      V8 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = ld16<V8>(q + min(g + i, p.group - 1) * p.q_head_stride);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (g + i >= p.group) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = (float)v[i][e] * sign;
          w[e] += (double)(x <= 0.f ? 0.f : x);  // a NaN stays in both parts
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] *= sign;
  };
  // This wavefront's pages, 16 at a time, the next ones loaded before the
  // present ones are scored; their ids 256 at a time.
  const uint8_t* bounds = p.bounds + h * 512 + piece * 16;
  const int64_t begin = first + wave * (int64_t)(chunk / kSelectWaves);
  const int64_t mine = min(begin + chunk / kSelectWaves, last);
  bool odd = false;  // an infinity or a NaN among this lane's scores
  auto put = [&](int64_t place, double score, bool writes) __attribute__((always_inline)) {
    if (!writes || place >= mine) return;
    if (in_lds) lds.keys[place] = order_key(score);
    else key_store(keys + place, order_key(score));
  };
  for (int64_t base = begin; base < mine; base += 4 * 64) {
    uint32_t ids[4];  // times the heads: pages' first rows of 512 bytes
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = row[min(base + 64 * i + lane, mine - 1)];
      ids[i] = (uint32_t)(id < 0 || id >= p.num_pages ? 0 : id) * (uint32_t)p.num_kv_heads;
    }
    const int batches = (int)((min(mine - base, (int64_t)256) + kBatch - 1) / kBatch);
    auto load = [&](V8 (&box)[8], int t) __attribute__((always_inline)) {
      const int of = t >> 2, at = (t & 3) * kBatch;
      const uint32_t id = of == 0 ? ids[0] : of == 1 ? ids[1] : of == 2 ? ids[2] : ids[3];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = __builtin_amdgcn_readlane(id, at + 2 * i), b = __builtin_amdgcn_readlane(id, at + 2 * i + 1);
        box[i] = ld16_once<V8>(bounds + ((uint64_t)(half ? b : a) << 9));
      }
    };
    auto score = [&](const V8 (&box)[8], int t) __attribute__((always_inline)) {
      double sum[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum[i] = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[i] = __builtin_fma((double)(float)box[i][e], w[e], sum[i]);
      }
      const double total = sums_of_8(sum, lane);
      odd |= !__builtin_isfinite(total);
      put(base + t * kBatch + 2 * (piece >> 2) + half, total, (lane & 3) == 0);
    };
    V8 box[8], next[8];
    load(box, 0);
    if (base == begin) weights();
    for (int t = 1; t < batches; ++t) {
      load(next, t);
      score(box, t - 1);
#pragma unroll
      for (int i = 0; i < 8; ++i) box[i] = next[i];
    }
    score(box, batches - 1);
  }
  if (__any(odd)) {
    // Again, two pages at a time, for what an infinity makes of a weight that stands for no
    // query: 0 times it is NaN above and nothing here, where it is a NaN only if a query or
    // a bound is that 0.  Scores without infinities come out as they were, bit for bit.
    __builtin_amdgcn_s_waitcnt(0);  // other lanes' keys at these places have been written
    uint32_t part = 0, zero = 0, infinite = 0;  // a bit a channel: queries that have this part, are 0, are infinite
    const T* q = (const T*)p.q + s * p.q_tok_stride + (int64_t)h * p.group * p.q_head_stride + 8 * (piece & 15);
#pragma unroll 1
    for (int g = 0; g < p.group; ++g) {
      const V8 v = ld16<V8>(q + g * p.q_head_stride);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = (float)v[e];
        part |= (uint32_t)(piece < 16 ? !(x >= 0.f) : !(x <= 0.f)) << e;
        zero |= (uint32_t)(x == 0.f) << e;
        infinite |= (uint32_t)__builtin_isinf(x) << e;
      }
    }
#pragma unroll 1
    for (int64_t place = begin + half; place - half < mine; place += 2) {
      const int id = row[min(place, mine - 1)];
      const V8 box = ld16<V8>(bounds + ((uint64_t)((uint32_t)(id < 0 || id >= p.num_pages ? 0 : id) *
                                                    (uint32_t)p.num_kv_heads) << 9));
      double sum = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float x = (float)box[e];
        const bool inf = __builtin_isinf(x), has = part >> e & 1;
        if (inf ? zero >> e & 1 : x == 0.f && (infinite >> e & 1)) x = __builtin_nanf("");
        else if (inf && !has) x = 0.f;
        sum = __builtin_fma((double)x, w[e], sum);
      }
      sum += across<16>(sum);
      sum += across<8>(sum);
      sum += across<4>(sum);
      sum += across<2>(sum);
      sum += across<1>(sum);
      put(place, sum, piece == 0);
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

namespace mva {
namespace {

// The parameters of an update of the bounds, or an error; p.num_tokens 0: nothing to do.
int bounds_params(BoundsParams& p, const void* k_cache, int64_t num_pages, int64_t page_stride, int64_t token_stride,
                  const void* page_bounds, const int32_t* block_tables, int64_t block_table_stride,
                  int64_t table_width, const int32_t* seq_lens, const int32_t* query_start_loc, int64_t num_seqs,
                  int64_t num_tokens, int num_kv_heads) {
  if (num_kv_heads <= 0 || num_pages < 0 || num_pages > 0x7fffffffLL || num_seqs < 0 || num_tokens < 0 ||
      table_width < 0 || block_table_stride < 0 || page_stride < 0 || token_stride < 0)
    return set_error("page bounds: invalid sizes");
  if (query_start_loc == nullptr && num_tokens != num_seqs)
    return set_error("page bounds: without query_start_loc every sequence has one token");
  p = {(const uint8_t*)k_cache, num_pages, page_stride * 2, token_stride * 2, (uint8_t*)page_bounds, block_tables,
       block_table_stride, table_width, seq_lens, query_start_loc, num_seqs, num_tokens, num_kv_heads};
  if (num_seqs == 0 || num_pages == 0 || table_width == 0) p.num_tokens = 0;
  if (p.num_tokens == 0) return 0;
  if (!k_cache || !page_bounds || !block_tables || !seq_lens) return set_error("page bounds: null buffer");
  if (((uint64_t)(uintptr_t)k_cache | (uint64_t)(uintptr_t)page_bounds | (uint64_t)(page_stride * 2) |
       (uint64_t)(token_stride * 2)) % 16)
    return set_error("page bounds: cache and bounds must be 16-byte aligned");
  return 0;
}

// Workgroups of `waves` wavefronts for an update.
int64_t bounds_blocks(const BoundsParams& p, int waves) {
  return ((p.num_tokens + kBoundsTokens - 1) / kBoundsTokens * p.num_kv_heads + waves - 1) / waves;
}

}  // namespace
}  // namespace mva

extern "C" int mva_update_page_bounds(const void* k_cache, int64_t num_pages, int64_t page_stride,
                                      int64_t token_stride, void* page_bounds, const int32_t* block_tables,
                                      int64_t block_table_stride, int64_t table_width, const int32_t* seq_lens,
                                      const int32_t* query_start_loc, int64_t num_seqs, int64_t num_tokens,
                                      int num_kv_heads, int head_dim, int page_size, int dtype, void* stream) {
  using namespace mva;
  if (head_dim != 128 || page_size != kPageTokens) return set_error("page bounds: head_dim must be 128, page_size 16");
  if (dtype != kBF16 && dtype != kF16) return set_error("page bounds: dtype must be bf16 or fp16");
  BoundsParams p;
  if (const int rc = bounds_params(p, k_cache, num_pages, page_stride, token_stride, page_bounds, block_tables,
                                   block_table_stride, table_width, seq_lens, query_start_loc, num_seqs, num_tokens,
                                   num_kv_heads))
    return rc;
  if (p.num_tokens == 0) return 0;
  // (Starts are 32-bit.  A product with the heads passes 64 bits for counts near 2^63.)
  if (num_tokens > 0x7fffffffLL) return set_error("page bounds: too many tokens for one launch");
  const int64_t blocks = bounds_blocks(p, 4);
  if (blocks > 0xffffffffLL / 256) return set_error("page bounds: too many tokens for one launch");
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == kBF16) hipLaunchKernelGGL(page_bounds_kernel<kInfBF16>, dim3((uint32_t)blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(page_bounds_kernel<kInfF16>, dim3((uint32_t)blocks), dim3(256), 0, st, p);
  return check_launch("page_bounds");
}

extern "C" int64_t mva_selection_workspace_bytes(int64_t num_seqs, int num_q_heads, int num_kv_heads,
                                                 int64_t table_width, int64_t num_selected) {
  using namespace mva;
  if (!selection_sizes_ok(num_seqs, num_q_heads, num_kv_heads, num_selected) || table_width < 0 ||
      table_width > 0x7fffffffLL / kPageTokens)
    return -1;
  return kSelectionHeaderBytes + selection_part_bytes(num_seqs, num_q_heads, num_selected) +
         selection_keys_bytes(num_seqs, num_kv_heads, table_width);
}

extern "C" int mva_select_pages(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* page_bounds,
                                int64_t num_pages, const int32_t* block_tables, int64_t block_table_stride,
                                int64_t table_width, const int32_t* seq_lens, int64_t num_seqs, int64_t num_selected,
                                int64_t sink_pages, int64_t recent_pages, int32_t* tables, int32_t* lens,
                                const void* k_cache, int64_t page_stride, int64_t token_stride, void* workspace,
                                int64_t workspace_bytes, int num_q_heads, int num_kv_heads, int head_dim,
                                int page_size, int dtype, void* stream) {
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
  if (num_pages * num_kv_heads > 0xffffffffLL) return set_error("page selection: too many pages");
  const int64_t rows = num_seqs * num_kv_heads;
  uint8_t* const ws = (uint8_t*)workspace;
  const SelectParams p = {
      q, q_token_stride, q_head_stride, (const uint8_t*)page_bounds, num_pages, block_tables, block_table_stride,
      table_width, seq_lens, num_seqs, (int)num_selected, (int)sink_pages, (int)recent_pages, tables, lens,
      (uint64_t*)(ws + kSelectionHeaderBytes + selection_part_bytes(num_seqs, num_q_heads, num_selected)),
      (int*)ws, num_kv_heads, num_q_heads / num_kv_heads};
  // Chunks: as small as 128 pages (16 a wavefront) as long as that makes no more
  // workgroups than the GPU holds at a time.  In microseconds, chunks of 128, 256 and
  // 512 pages: one row of 30001 tokens at 8 KV heads 9.7, 10.4 and 13.1; 8 rows of
  // 1024-4096 at 8 heads 8.1, 8.5 and 9.1; 37 of 300-6000 at 4 heads (at most 3, 2 and 1
  // workgroups a row) 13.0, 14.8 and 12.6.  448 (row, KV head) pairs of 512-2048 pages
  // in one workgroup each 70, in chunks of 1024 pages 83, of 512 86.
  const int64_t most = table_width - sink_pages - recent_pages;
  int64_t chunk = kBatch * kSelectWaves;
  while (chunk < most && rows * ((most + chunk - 1) / chunk) > kSelectGroups) chunk *= 2;
  const int64_t chunks = most > chunk && table_width > num_selected ? (most + chunk - 1) / chunk : 1;
  const int64_t blocks = rows * chunks;
  BoundsParams update = {};
  if (k_cache != nullptr) {
    if (const int rc = bounds_params(update, k_cache, num_pages, page_stride, token_stride, page_bounds, block_tables,
                                     block_table_stride, table_width, seq_lens, nullptr, num_seqs, num_seqs,
                                     num_kv_heads))
      return rc;
  }
  const int64_t all = blocks + (k_cache != nullptr ? bounds_blocks(update, kSelectWaves) : 0);
  if (all > 0xffffffffLL / kSelectThreads) return set_error("page selection: too many rows for one launch");
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == kBF16)
    hipLaunchKernelGGL(page_select_kernel<__bf16>, dim3((uint32_t)all), dim3(kSelectThreads), 0, st, p, (int)chunk,
                       (int)chunks, (uint32_t)blocks, update);
  else
    hipLaunchKernelGGL(page_select_kernel<_Float16>, dim3((uint32_t)all), dim3(kSelectThreads), 0, st, p, (int)chunk,
                       (int)chunks, (uint32_t)blocks, update);
  return check_launch("page_select");
}
