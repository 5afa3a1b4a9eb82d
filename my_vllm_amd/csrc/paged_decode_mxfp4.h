// Paged GQA decode over an MXFP4 cache (format: mxfp4.h): the work split, the
// partials and the merge kernel of paged_decode.h, with another page stream.
//
//   o = sum_j softmax_j(scale * q . K[j]) V[j],  K, V = code * 2^(byte - 127)
//
// A wavefront streams its pieces (sequence, KV head, page range) in tiles of two
// pages, 32 tokens: 2 KB of codes and 128 bytes of scales of K, as much of V.
// Both go from memory into LDS by global_load_lds, in three buffers: two tiles in
// flight while one is computed, up to twelve wavefronts per CU.  (Tiles of four pages in
// two buffers, eight wavefronts: 275 us for the largest batch below.)
//
// Measured: 56 sequences of 8192-32768 tokens at 64 / 8 heads 249 us a call with its merge
// (1.38 GB, 5.5 TB/s; a stream of the same pages into LDS without arithmetic reaches
// 6.1), 64 of 128-2048 at 16 / 8 18.6 us (74 MB, 4.0 TB/s), 8 of 256-1024 9.1 us.  The small
// ones are bound by a chain of latencies: launch, piece, page table, pages, and 0.75 us a
// tile of a wavefront alone on its SIMD (155 vector instructions, V through LDS).
//
//  * K: a lane reads the 16 bytes of one token's 32-element group, which is
//    also what one scale covers, and converts them to the query's type with
//    that scale in one instruction a pair, exactly.  The contraction may take
//    the 128 dimensions in any order, so lane group j holds dimensions 32j..
//    and Q is loaded to match: S^T = K Q^T by 16x16x32 MFMAs, fp32.
//  * V: O^T += V^T P^T wants a lane to hold one dimension of eight tokens, and a
//    token's scales run along its dimensions.  So a lane takes one group of one
//    token from LDS, converts it with its scale, exactly, and writes the rows
//    back to LDS (over the codes, which every lane has read by then), from where
//    ds_read_b64_tr_b16 transposes them.  Transposing the codes instead
//    (ds_read_b64_tr_b4) leaves the scales to P, four scaled copies of it: 32
//    more conversions and 128 more multiplies and byte extracts a tile, and P
//    times a scale leaves fp16's range.
// Tokens past a sequence's end or its piece get S = -inf and V = 0: nothing of a
// stale row, whose scales may be NaN, can reach the result.
#pragma once

#include "mxfp4.h"
#include "paged_decode.h"

namespace mva {

// page_stride counts bytes here, and tok_stride is unused.
struct Fp4DecodeParams : DecodeParams {
  int64_t head_stride;  // bytes between the blocks of a page's KV heads
};

constexpr int kFp4TilePages = 2;
constexpr int kFp4TileTokens = kFp4TilePages * kPageSize;
// A tile in LDS: K codes, V codes, then the scales of both pages of K and of V.
constexpr int kFp4TileV = kFp4TilePages * kFp4ScaleOffset;
constexpr int kFp4TileKScales = 2 * kFp4TileV;
constexpr int kFp4TileVScales = kFp4TileKScales + kFp4TileTokens * kFp4RowScales;
constexpr int kFp4TileBytes = kFp4TileVScales + kFp4TileTokens * kFp4RowScales;  // 4352
constexpr int kFp4TileBufs = 3;
constexpr int kFp4WaveLdsBytes = kFp4TileBufs * kFp4TileBytes;  // 13056: twelve wavefronts in 160 KB
// Wavefronts that share a piece, and where each leaves its m and l of 16 heads,
// after its 16 rows of o.
constexpr int kFp4ShareWaves = 4;  // as the planner's
constexpr int kFp4ShareMax = 16 * kHeadDim * 4;
constexpr int kFp4ShareSum = kFp4ShareMax + 64;
static_assert(kFp4ShareSum + 64 <= kFp4WaveLdsBytes, "a share fits its wavefront's LDS");
typedef __attribute__((address_space(3))) float lds_f32;
constexpr int kFp4TileLoads = 2 * kFp4TilePages + 1;
// Pages whose ids a wavefront holds at a time, four table words a lane.
constexpr int kFp4RunPages = 256;

// A tile's copies into LDS at byte address `lds`: the codes of its pages of K and
// of V, 16 bytes a lane, 1 KB each, from a[0] .. a[3], and its scales, 4 bytes a
// lane, from w (lane group j: K pages 0 and 1, V pages 0 and 1).  One asm
// statement (see paged_decode.h), which first waits for this wavefront's LDS
// reads of the buffer.
struct Fp4Copy {
  const uint8_t* a[4];
  const uint8_t* w;
};

static_assert(kFp4TileV == 0x800 && kFp4TileKScales == 0x1000 && kFp4TileVScales == 0x1080, "the copies' LDS layout");

__device__ inline void fp4_copy_tile(const Fp4Copy& c, uint32_t lds) {
  uint32_t m0_saved;
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile(
      "s_mov_b32 %[m0s], m0\n\t"
      "s_mov_b32 m0, %[l]\n\t"
      "s_waitcnt lgkmcnt(0)\n\t"
      "global_load_lds_dwordx4 %[a0], off\n\t"
      "s_add_u32 m0, %[l], 0x400\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %[a1], off\n\t"
      "s_add_u32 m0, %[l], 0x800\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %[a2], off\n\t"
      "s_add_u32 m0, %[l], 0xc00\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %[a3], off\n\t"
      "s_add_u32 m0, %[l], 0x1000\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %[w], off\n\t"
      "s_mov_b32 m0, %[m0s]"
      : [m0s] "=&s"(m0_saved)
      : [l] "s"(lds), [a0] "v"(c.a[0]), [a1] "v"(c.a[1]), [a2] "v"(c.a[2]), [a3] "v"(c.a[3]), [w] "v"(c.w)
      : "memory", "scc");
}

// Maximum and sum over the four lane groups of a wavefront, without LDS.
__device__ inline float groups_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float groups_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// One wavefront, number `slot` of its workgroup, of a decode launch over piece
// lists (see decode_wave); `group_lds` is kFp4WaveLdsBytes for each wavefront of the workgroup.
//
// Wavefronts 4 i .. 4 i + 3 of a launch may instead share a piece: each has one
// descriptor, with a quarter of the pages and the complement of part_base, and the four
// join in LDS, with one partial for them, or none and no merge kernel where the piece is
// a whole segment.  Either all pieces of a launch are shared or none.
//
// A piece goes in runs of up to 256 pages.  A run loads its queries and page table
// words, copies its first three tiles, and then computes tile after tile, copying
// into each buffer the tile three further on.  Nothing of the next run is
// requested before the run has ended: its wavefront waits for that, the others of
// the CU do not, and the loop stays short (at the start of a launch fetching its
// code counts: a form with the next piece's first tiles in flight was twice the
// code and 1-2 us slower on small batches, level on large ones).
//
// `progress` (LDS, one int per wavefront of the workgroup, or nullptr): the
// wavefronts of one `slot` % 4 share a SIMD, whose issue favours the oldest.  Each
// publishes the tiles it has done and runs at the higher priority the fewer of
// its two partners are behind it, so the three stay level.
template <typename T>
__device__ void decode_wave_mxfp4(const Fp4DecodeParams& p, int wave, lds_u8* group_lds, int* progress, int slot) {
  lds_u8* const lds = group_lds + slot * kFp4WaveLdsBytes;
  typedef typename Elem<T>::v8 V8;
  typedef typename Elem<T>::v4 V4;
  const int lane = threadIdx.x & 63;
  const int q4 = lane >> 4;
  const int c = lane & 15;
  const int G = p.group;
  const int Hkv = p.num_kv_heads;
  // Graph launches read this step's counts; wavefronts past them have no work.
  const int W = p.counts ? min(sload(p.counts, 1), p.num_waves) : p.num_waves;
  const int N = p.counts ? min(sload(p.counts, 0), p.num_items) : p.num_items;
  if (wave >= W || wave >= N) return;
  const bool q_lane = c < G;

  // Descriptor fields: {seq, page_begin, page_end, chunk, n_chunks, part_base, q_row, kv_head}.
  auto desc_at = [&](int idx) -> i32x8 { return ((const_i32x8*)p.items)[idx]; };
  // Lane (q4, c) of the B operand holds Q[g = c][32 q4 + 8 j .. +8]; lanes
  // c >= G read head 0 of the group (in bounds) and are zeroed.
  auto q_addr = [&](const i32x8& d) -> const T* {
    int g = d[7] * G + (q_lane ? c : 0);
    asm volatile("" : "+v"(g));  // made for each piece, not held in registers
    return (const T*)p.q + (int64_t)d[6] * p.q_tok_stride + (int64_t)g * p.q_head_stride + 32 * q4;
  };
  // This wavefront's list: piece `wave`, then entries [nx, nx_end), clamped to
  // the item array.
  int nx = max(sload(p.wave_extra, wave), 0);
  const int nx_end = min(sload(p.wave_extra, wave + 1), N);

  // Per-lane offsets.  K codes lie in LDS token by token, 64 bytes each, with
  // 16-byte chunk ch of token t at slot ch ^ (t / 4): the 16 tokens that a read
  // takes at one chunk then fall on different banks.  V codes lie in lane order.
  const uint32_t koff = (uint32_t)((lane >> 2) * kFp4RowBytes + (((lane & 3) ^ (lane >> 4)) << 4));
  const uint32_t voff = (uint32_t)(lane << 4);
  const int kread = c * kFp4RowBytes + ((q4 ^ (c >> 2)) << 4);
  const int ksread = kFp4TileKScales + c * kFp4RowScales + q4;
  // Converted V rows of one page, 256 bytes a token, 16-byte chunk ch of token t
  // at slot ch ^ vswz(t): 16 lanes of a write take 16 slots, 32 lanes of a
  // transposed read take all 256 bytes of banks.  This lane writes chunks 4 (lane % 4) + u of token
  // lane / 4, and supplies token 4 q4 + c / 4, dimensions 16 mt + 4 (c % 4) .. + 3
  // to a transposed read, which gives it dimension 16 mt + c of tokens 4 q4 .. + 3.
  auto vswz = [](int t) { return (t & 3) | (t & 1) << 2 | (t & 4) << 1; };
  const int vtok = lane >> 2;
  const int rtok = 4 * q4 + (c >> 2);
  const int vwrite = vtok * 256 + ((4 * (lane & 3)) ^ vswz(vtok)) * 16;            // chunk u: ^ 16 u
  const int vread = rtok * 256 + (((c >> 1) & 1) ^ vswz(rtok)) * 16 + (c & 1) * 8;  // d-tile mt: ^ 32 mt

  i32x8 X = desc_at(wave);  // the piece being computed
  i32x8 N_ = X;             // the one after it
  int seq_len = sload(p.seq_lens, X[0]);
  auto good_id = [&](int id) { return (uint32_t)id < (uint32_t)p.num_pages ? id : 0; };
  // This lane's addresses in page 0 of head X[7]; a page id adds page_stride,
  // below 2^32 bytes.
  const uint8_t *k_lane, *v_lane, *sc_lane;
  auto tile_at = [&](int id0, int id1) {
    auto page = [&](const uint8_t* lane_base, int id) {
      return lane_base + (uint64_t)(uint32_t)id * (uint32_t)p.page_stride;
    };
    return Fp4Copy{{page(k_lane, id0), page(k_lane, id1), page(v_lane, id0), page(v_lane, id1)},
                   page(sc_lane, (q4 & 1) ? id1 : id0)};
  };
  V8 qf[4];
  f32x4 o[8];  // o[mt][r] = O^T[d = 16 mt + 4 q4 + r][g = c]
  float m, l;  // reference max (log2 domain) of g = c; this lane's share of the denominator
  // `valid`: tokens of the tile that count; below 32 on an edge tile.
  auto compute = [&](lds_u8* buf, int valid) __attribute__((always_inline)) {
    const bool edge = valid < kFp4TileTokens;  // wave-uniform
    u32x4 vw[2];  // page i's codes of token lane / 4, group lane % 4
    uint32_t vs[2];
    u32x4 kw[2];
    float ks[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kw[i] = lds_ld16<u32x4>(buf + kread + i * kFp4ScaleOffset);
      ks[i] = fp4_scale((uint32_t)buf[ksread + 64 * i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      vw[i] = lds_ld16<u32x4>(buf + kFp4TileV + i * kFp4ScaleOffset + voff);
      vs[i] = buf[kFp4TileVScales + 64 * i + lane];
    }
    // A branch, not selects (the asm keeps it one).
    if (edge) {
      int end = valid;
      asm volatile("" : "+s"(end));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool live = kPageSize * i + vtok < end;
        vs[i] = live ? vs[i] : 127u;
#pragma unroll
        for (int u = 0; u < 4; ++u) vw[i][u] = live ? vw[i][u] : 0u;
      }
    }
    // Rows of page i over the tile's codes, and their transposed reads.  LDS works
    // in order for a wavefront: the reads of codes above come before the first
    // page's writes, its transposed reads before the second page's writes.
    auto write_v = [&](int i) __attribute__((always_inline)) {
      const float scale = fp4_scale(vs[i]);
#pragma unroll
      for (int u = 0; u < 4; ++u) lds_st16(buf + (vwrite ^ (16 * u)), fp4_unpack8<T>(vw[i][u], scale));
    };
    // v[mt]: dimension 16 mt + c of tokens 4 q4 .. + 3 of the page.
    auto read_v = [&](s16x4 (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) v[mt] = lds_ld_tr16(buf + (vread ^ (32 * mt)));
    };
    // The first page's rows are on their way while the scores are computed (after them:
    // 0.05 us a tile more for a wavefront alone on its SIMD, 200 sequences of 128-4096 at
    // 40 / 8 heads 100 against 97 us).  A second place for the other page's, so that both
    // are on their way, was slower: two workgroups a CU instead of three.
    s16x4 v0[8], v1[8];
    wave_lds_fence();
    write_v(0);
    wave_lds_fence();
    f32x4 sc[2];  // sc[i][r] = S[token 4 q4 + r of page i][g = c]
#pragma unroll
    for (int i = 0; i < 2; ++i) sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // The two pages' sums in turn: one alone is a chain of dependent MFMAs.
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) sc[i] = Elem<T>::mfma16(fp4_unpack8<T>(kw[i][j], ks[i]), qf[j], sc[i]);
      if (j & 1) __builtin_amdgcn_sched_barrier(0);  // not all conversions at once: registers
    }
    read_v(v0);
    wave_lds_fence();
    write_v(1);
    wave_lds_fence();
    read_v(v1);
    if (edge) {
      int end = valid;
      asm volatile("" : "+s"(end));
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (kPageSize * i + 4 * q4 + r >= end) sc[i][r] = -INFINITY;
    }
    // P = 2^(S * scale - m), packed, and this lane's sum of it.
    V8 pf;
    auto exponentials = [&](float m_use) __attribute__((always_inline)) {
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float pr = fast_exp2(sc[i][r] * p.scale_log2 - m_use);
          sum[r & 1] += pr;
          pf[4 * i + r] = (T)pr;
        }
      return sum[0] + sum[1];
    };
    // The reference maximum moves only when a score exceeds it by more than 8
    // (P stays <= 2^8).  A sum below 128 shows that none does, as every P is
    // below 128 then (2^7.01 covers the rounding of S * scale and m + 8 while
    // |m| < 2^20), so most tiles take no maximum.
    float sum = exponentials(m);
    if (__any(!(sum < 128.f && __builtin_fabsf(m) < 0x1p20f))) {
      float tmax = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, sc[i][r]);
      tmax = groups_max(tmax) * p.scale_log2;  // scale > 0 commutes with max
      const bool grow = tmax > m + 8.0f;
      const float m_new = grow ? tmax : m;
      const float alpha = grow ? fast_exp2(m - m_new) : 1.0f;  // m = -inf -> 0
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) o[mt] *= alpha;
      sum = exponentials(m == -INFINITY ? 0.f : m);
    }
    l += sum;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt)
      o[mt] = Elem<T>::mfma16(
          __builtin_bit_cast(V8, __builtin_shufflevector(v0[mt], v1[mt], 0, 1, 2, 3, 4, 5, 6, 7)), pf, o[mt]);
  };

  // A quarter of a shared piece: its four wavefronts leave their o, m and l in LDS,
  // over their tiles, and join them together, into the output or a partial.
  auto join_share = [&](float l_tot) __attribute__((always_inline)) {
    // Row c of this wavefront, 16-byte chunk ch at slot ch ^ c: 16 lanes of a
    // write take 16 slots.
    int row = c, part = q4;
    asm volatile("" : "+v"(row), "+v"(part));  // addresses made here, not held in registers through the stream
    if (q_lane) {
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) lds_st16(lds + row * 4 * kHeadDim + (((4 * mt + part) ^ row) << 4), o[mt]);
      if (part == 0) {
        *(lds_f32*)(lds + kFp4ShareMax + 4 * row) = m;
        *(lds_f32*)(lds + kFp4ShareSum + 4 * row) = l_tot;
      }
    }
    __syncthreads();
    lds_u8* const first = group_lds + (slot & ~(kFp4ShareWaves - 1)) * kFp4WaveLdsBytes;
    int thread = lane;
    asm volatile("" : "+v"(thread));
    for (int i = (slot & (kFp4ShareWaves - 1)) * 64 + thread; i < G * (kHeadDim / 4); i += 64 * kFp4ShareWaves) {
      const int g = i >> 5, ch = i & 31;
      float mw[kFp4ShareWaves], top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFp4ShareWaves; ++w) {
        mw[w] = *(lds_f32*)(first + w * kFp4WaveLdsBytes + kFp4ShareMax + 4 * g);
        top = fmaxf(top, mw[w]);
      }
      const float m_use = top == -INFINITY ? 0.f : top;
      f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < kFp4ShareWaves; ++w) {
        const float a = fast_exp2(mw[w] - m_use);  // a wavefront without pages: m = -inf -> 0
        den += a * *(lds_f32*)(first + w * kFp4WaveLdsBytes + kFp4ShareSum + 4 * g);
        sum += a * lds_ld16<f32x4>(first + w * kFp4WaveLdsBytes + g * 4 * kHeadDim + ((ch ^ g) << 4));
      }
      const float inv = den > 0.f ? 1.0f / den : 0.f;
      if (X[4] > 1) {
        const int64_t at = ((int64_t)(~X[5] + X[3]) * Hkv + X[7]) * G + g;
        store16_device_untracked(p.part_o + at * kHeadDim + 4 * ch, __builtin_bit_cast(u32x4, sum * inv));
        if (ch == 0) store4_device_untracked(&p.part_lse[at], den > 0.f ? m_use + fast_log2(den) : -INFINITY);
        continue;
      }
      V4 y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = (T)(sum[r] * inv);
      store8_untracked((T*)p.out + (int64_t)X[6] * p.out_tok_stride + (int64_t)(X[7] * G + g) * p.out_head_stride +
                           4 * ch,
                       __builtin_bit_cast(u32x2, y));
    }
  };
  // End of piece X: the final output, its share of one, or its split-K partial
  // (normalised o and log2-sum-exp) for the merge kernel.
  auto finish_piece = [&]() __attribute__((always_inline)) {
    const float l_tot = groups_sum(l);
    if (X[5] < 0) {
      join_share(l_tot);
      return;
    }
    const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;
    const int h = X[7];
    if (!q_lane) return;
    int hc = h * G + c, part = q4;
    asm volatile("" : "+v"(hc), "+v"(part));  // as above
    if (X[4] == 1) {
      T* op = (T*)p.out + (int64_t)X[6] * p.out_tok_stride + (int64_t)hc * p.out_head_stride + 4 * part;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        V4 w;
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = (T)(o[mt][r] * inv);
        store8_untracked(op + 16 * mt, __builtin_bit_cast(u32x2, w));
      }
      return;
    }
    const int64_t row = (int64_t)(X[5] + X[3]) * Hkv * G + hc;
    float* po = p.part_o + row * kHeadDim + 4 * part;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) store16_device_untracked(po + 16 * mt, __builtin_bit_cast(u32x4, o[mt] * inv));
    if (part == 0) store4_device_untracked(&p.part_lse[row], l_tot > 0.f ? m + fast_log2(l_tot) : -INFINITY);
  };

  int done = 0;
  const int mate1 = slot < 8 ? slot + 4 : slot - 8, mate2 = slot < 4 ? slot + 8 : slot - 4;
  auto keep_level = [&]() {
    if (!progress) return;
    if (lane == 0) progress[slot] = done;
    const int a = __builtin_amdgcn_readfirstlane(*(volatile int*)&progress[mate1]);
    const int b = __builtin_amdgcn_readfirstlane(*(volatile int*)&progress[mate2]);
    const int behind = (a < done ? 1 : 0) + (b < done ? 1 : 0);
    if (behind == 0) __builtin_amdgcn_s_setprio(2);
    else if (behind == 1) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
    ++done;
  };

  // ---- piece by piece, run by run -------------------------------------------
  static_assert(kFp4TileBufs == 3 && kFp4TilePages == 2, "the run's copies and waits");
  for (;;) {
    const bool more = nx < nx_end;
    if (more) N_ = desc_at(nx);
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
    const int64_t head = (int64_t)X[7] * p.head_stride;
    k_lane = (const uint8_t*)p.k_cache + head + koff;
    v_lane = (const uint8_t*)p.v_cache + head + voff;
    sc_lane = (const uint8_t*)(q4 < 2 ? p.k_cache : p.v_cache) + head + kFp4ScaleOffset + c * kFp4RowScales;
    for (int first = X[1]; first < X[2]; first += kFp4RunPages) {
      const int pages = min(X[2] - first, kFp4RunPages);
      const int tiles = (pages + 1) >> 1;
      const int32_t* const row = p.block_tables + (int64_t)X[0] * p.bt_stride + first;
      int words[kFp4RunPages / 64];  // lane L of words[k]: page 64 k + L of the run
#pragma unroll
      for (int k = 0; k < kFp4RunPages / 64; ++k) words[k] = row[min(64 * k + lane, pages - 1)];
      const T* const q = q_addr(X);
#pragma unroll
      for (int j = 0; j < 4; ++j) qf[j] = ld16<V8>(q + 8 * j);
#pragma unroll
      for (int k = 0; k < kFp4RunPages / 64; ++k) words[k] = good_id(words[k]);
#pragma unroll
      for (int j = 0; j < 4; ++j) qf[j] = q_lane ? qf[j] : V8{};
      const int tokens = min(seq_len, X[2] * kPageSize) - first * kPageSize;  // of the run on
      lds_u8* buf = lds;
      int t = -kFp4TileBufs;
      asm volatile("" : "+s"(t));  // one copy of the loop's code: no peeled first turns
#pragma unroll 1
      for (; t < tiles; ++t) {
        if (t >= 0) {
          if (t + 2 < tiles) __builtin_amdgcn_s_waitcnt(waitcnt_vm(2 * kFp4TileLoads));
          else if (t + 1 < tiles) __builtin_amdgcn_s_waitcnt(waitcnt_vm(kFp4TileLoads));
          else __builtin_amdgcn_s_waitcnt(kVmcnt0);
          wave_lds_fence();
          compute(buf, tokens - t * kFp4TileTokens);
          wave_lds_fence();
        }
        const int page = kFp4TilePages * (t + kFp4TileBufs);
        if (page < pages) {
          const int word = page < 128 ? (page < 64 ? words[0] : words[1]) : (page < 192 ? words[2] : words[3]);
          fp4_copy_tile(
              tile_at(__builtin_amdgcn_readlane(word, page & 63), __builtin_amdgcn_readlane(word, (page & 63) + 1)),
              (uint32_t)(uintptr_t)buf);
        }
        buf = buf == lds + (kFp4TileBufs - 1) * kFp4TileBytes ? lds : buf + kFp4TileBytes;
        keep_level();
      }
    }
    finish_piece();
    if (!more) break;
    X = N_;
    ++nx;
    seq_len = sload(p.seq_lens, X[0]);
  }
  if (progress && lane == 0) progress[slot] = 0x3fffffff;  // no longer in the way
  __builtin_amdgcn_s_waitcnt(kVmcnt0);
}

}  // namespace mva
