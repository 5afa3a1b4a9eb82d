// Paged GQA decode over an MXFP4 cache (format: mxfp4.h): the work split, the
// partials and the merge kernel of paged_decode.h, with another page stream.
//
//   o = sum_j softmax_j(scale * q . K[j]) V[j],  K, V = code * 2^(byte - 127)
//
// A wavefront streams its pieces (sequence, KV head, page range) in tiles of
// four pages, 64 tokens: 4 KB of codes and 256 bytes of scales of K, as much of
// V.  Both go from memory into LDS by global_load_lds, double-buffered, the
// next tile in flight while this one is computed.
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

constexpr int kFp4TilePages = 4;
constexpr int kFp4TileTokens = kFp4TilePages * kPageSize;
// A tile in LDS: K codes, V codes, K scales, V scales.
constexpr int kFp4TileV = kFp4TilePages * kFp4ScaleOffset;
constexpr int kFp4TileKScales = 2 * kFp4TileV;
constexpr int kFp4TileVScales = kFp4TileKScales + kFp4TileTokens * kFp4RowScales;
constexpr int kFp4TileBytes = kFp4TileVScales + kFp4TileTokens * kFp4RowScales;  // 8704
constexpr int kFp4WaveLdsBytes = 2 * kFp4TileBytes;

// One tile's copies into LDS at byte address `lds`, ten loads, then a wait for
// everything before them: page j's codes of K and V, 16 bytes a lane, from k[j]
// and v[j], and both scale blocks, 4 bytes a lane, from ks and vs.
struct Fp4Copy {
  const uint8_t* k[kFp4TilePages];
  const uint8_t* v[kFp4TilePages];
  const uint8_t* ks;
  const uint8_t* vs;
};

#define MVA_FP4_TILE_DMA                   \
  "s_mov_b32 %[m0s], m0\n\t"               \
  "s_mov_b32 m0, %[l]\n\t"                 \
  "s_nop 0\n\t"                            \
  "global_load_lds_dwordx4 %[k0], off\n\t" \
  "s_add_u32 m0, %[l], 0x400\n\t"          \
  "s_nop 0\n\t"                            \
  "global_load_lds_dwordx4 %[k1], off\n\t" \
  "s_add_u32 m0, %[l], 0x800\n\t"          \
  "s_nop 0\n\t"                            \
  "global_load_lds_dwordx4 %[k2], off\n\t" \
  "s_add_u32 m0, %[l], 0xc00\n\t"          \
  "s_nop 0\n\t"                            \
  "global_load_lds_dwordx4 %[k3], off\n\t" \
  "s_add_u32 m0, %[l], 0x1000\n\t"         \
  "s_nop 0\n\t"                            \
  "global_load_lds_dwordx4 %[v0], off\n\t" \
  "s_add_u32 m0, %[l], 0x1400\n\t"         \
  "s_nop 0\n\t"                            \
  "global_load_lds_dwordx4 %[v1], off\n\t" \
  "s_add_u32 m0, %[l], 0x1800\n\t"         \
  "s_nop 0\n\t"                            \
  "global_load_lds_dwordx4 %[v2], off\n\t" \
  "s_add_u32 m0, %[l], 0x1c00\n\t"         \
  "s_nop 0\n\t"                            \
  "global_load_lds_dwordx4 %[v3], off\n\t" \
  "s_add_u32 m0, %[l], 0x2000\n\t"         \
  "s_nop 0\n\t"                            \
  "global_load_lds_dword %[ks], off\n\t"   \
  "s_add_u32 m0, %[l], 0x2100\n\t"         \
  "s_nop 0\n\t"                            \
  "global_load_lds_dword %[vs], off\n\t"   \
  "s_mov_b32 m0, %[m0s]\n\t"               \
  "s_waitcnt vmcnt(10)"

static_assert(kFp4TileV == 0x1000 && kFp4TileKScales == 0x2000 && kFp4TileVScales == 0x2100, "the copies' LDS layout");

#define MVA_FP4_TILE_IN                                                                                          \
  [l] "s"(lds), [k0] "v"(c.k[0]), [k1] "v"(c.k[1]), [k2] "v"(c.k[2]), [k3] "v"(c.k[3]), [v0] "v"(c.v[0]),        \
      [v1] "v"(c.v[1]), [v2] "v"(c.v[2]), [v3] "v"(c.v[3]), [ks] "v"(c.ks), [vs] "v"(c.vs)

__device__ inline void fp4_tile_copy(const Fp4Copy& c, uint32_t lds) {
  uint32_t m0_saved;
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile(MVA_FP4_TILE_DMA : [m0s] "=&s"(m0_saved) : MVA_FP4_TILE_IN : "memory", "scc");
}

// The first tile of a piece: also requests, ahead of the tile, so that the wait
// covers them, the query fragments at `q` (4 x 16 bytes) and the piece's page
// table words at t0 and t1.
struct Fp4Piece {
  u32x4 q[4];
  int lo, hi;
};
__device__ inline void fp4_tile_copy_first(const Fp4Copy& c, uint32_t lds, const void* q, const int32_t* t0,
                                           const int32_t* t1, Fp4Piece& out) {
  uint32_t m0_saved;
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile(
      "global_load_dword %[lo], %[t0], off\n\t"
      "global_load_dword %[hi], %[t1], off\n\t"
      "global_load_dwordx4 %[q0], %[qp], off\n\t"
      "global_load_dwordx4 %[q1], %[qp], off offset:16\n\t"
      "global_load_dwordx4 %[q2], %[qp], off offset:32\n\t"
      "global_load_dwordx4 %[q3], %[qp], off offset:48\n\t" MVA_FP4_TILE_DMA
      : [m0s] "=&s"(m0_saved), [lo] "=&v"(out.lo), [hi] "=&v"(out.hi), [q0] "=&v"(out.q[0]), [q1] "=&v"(out.q[1]),
        [q2] "=&v"(out.q[2]), [q3] "=&v"(out.q[3])
      : MVA_FP4_TILE_IN, [qp] "v"(q), [t0] "v"(t0), [t1] "v"(t1)
      : "memory", "scc");
}

#undef MVA_FP4_TILE_DMA
#undef MVA_FP4_TILE_IN

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

// One wavefront of a decode launch over piece lists (see decode_wave); `lds` is
// its kFp4WaveLdsBytes of LDS.
template <typename T>
__device__ void decode_wave_mxfp4(const Fp4DecodeParams& p, int wave, lds_u8* lds) {
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
    const int g = q_lane ? c : 0;
    return (const T*)p.q + (int64_t)d[6] * p.q_tok_stride + (int64_t)(d[7] * G + g) * p.q_head_stride + 32 * q4;
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
  // Converted V rows of two pages, 256 bytes a token, 16-byte chunk ch of token t
  // at slot ch ^ vswz(t).  This lane writes chunks 4 (lane % 4) + u of token
  // lane / 4, and supplies token 4 q4 + c / 4, dimensions 16 mt + 4 (c % 4) .. + 3
  // to a transposed read, which gives it dimension 16 mt + c of tokens 4 q4 .. + 3.
  auto vswz = [](int t) { return 2 * (t & 3) | ((t >> 2) & 1) << 3; };
  const int vtok = lane >> 2;
  int vwrite[4], vread[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) vwrite[u] = vtok * 256 + ((4 * (lane & 3) + u) ^ vswz(vtok)) * 16;
  const int rtok = 4 * q4 + (c >> 2);
#pragma unroll
  for (int u = 0; u < 4; ++u) vread[u] = rtok * 256 + ((2 * u + ((c >> 1) & 1)) ^ vswz(rtok)) * 16 + (c & 1) * 8;

  // The tile to copy next: tile ft of piece F, its page ids, and whether it
  // opens a piece.  A piece's first page ids come by scalar loads, one piece
  // ahead; the others from its table words, lane L of lo / hi holding page L and
  // 64 + L, which arrive with its first tile.
  i32x8 F = desc_at(wave);
  int ft = 0;
  bool fvalid = true, fnew = true;
  int id0, id1, id2, id3;
  Fp4Piece piece;
  auto good_id = [&](int id) { return (uint32_t)id < (uint32_t)p.num_pages ? id : 0; };
  auto bt_row = [&]() { return p.block_tables + (int64_t)F[0] * p.bt_stride + F[1]; };
  auto open_ids = [&]() {
    const int last = max(F[2] - F[1] - 1, 0);
    id0 = good_id(sload(bt_row(), 0));
    id1 = good_id(sload(bt_row(), min(1, last)));
    id2 = good_id(sload(bt_row(), min(2, last)));
    id3 = good_id(sload(bt_row(), min(3, last)));
  };
  open_ids();
  auto advance = [&]() {
    ++ft;
    fnew = kFp4TilePages * ft >= F[2] - F[1];
    if (!fnew) {
      const int words = kFp4TilePages * ft < 64 ? piece.lo : piece.hi;
      const int at = (kFp4TilePages * ft) & 63;
      id0 = __builtin_amdgcn_readlane(words, at);
      id1 = __builtin_amdgcn_readlane(words, at + 1);
      id2 = __builtin_amdgcn_readlane(words, at + 2);
      id3 = __builtin_amdgcn_readlane(words, at + 3);
      return;
    }
    fvalid = nx < nx_end;
    if (!fvalid) return;
    F = desc_at(nx);
    ++nx;
    ft = 0;
    open_ids();
  };
  // This lane's addresses in page 0 of head F[7]; a page id adds page_stride,
  // below 2^32 bytes.
  const uint8_t *k_lane, *v_lane, *ks_lane, *vs_lane;
  auto copy_tile = [&](lds_u8* buf) {
    if (fnew) {
      const int64_t head = (int64_t)F[7] * p.head_stride;
      k_lane = (const uint8_t*)p.k_cache + head + koff;
      v_lane = (const uint8_t*)p.v_cache + head + voff;
      ks_lane = (const uint8_t*)p.k_cache + head + kFp4ScaleOffset + c * kFp4RowScales;
      vs_lane = (const uint8_t*)p.v_cache + head + kFp4ScaleOffset + c * kFp4RowScales;
    }
    Fp4Copy cp;
    const uint32_t stride = (uint32_t)p.page_stride;
    auto page = [&](const uint8_t* lane_base, int id) { return lane_base + (uint64_t)(uint32_t)id * stride; };
    cp.k[0] = page(k_lane, id0), cp.k[1] = page(k_lane, id1), cp.k[2] = page(k_lane, id2), cp.k[3] = page(k_lane, id3);
    cp.v[0] = page(v_lane, id0), cp.v[1] = page(v_lane, id1), cp.v[2] = page(v_lane, id2), cp.v[3] = page(v_lane, id3);
    int mine = id0;  // the page whose scales this lane copies
    mine = q4 == 1 ? id1 : mine;
    mine = q4 == 2 ? id2 : mine;
    mine = q4 == 3 ? id3 : mine;
    cp.ks = page(ks_lane, mine), cp.vs = page(vs_lane, mine);
    const uint32_t at = (uint32_t)(uintptr_t)buf;
    if (fnew) {
      const int last = max(F[2] - F[1] - 1, 0);
      fp4_tile_copy_first(cp, at, q_addr(F), bt_row() + min(lane, last), bt_row() + min(64 + lane, last), piece);
      piece.lo = good_id(piece.lo);
      piece.hi = good_id(piece.hi);
    } else {
      fp4_tile_copy(cp, at);
    }
  };

  i32x8 X = F;  // the piece being computed
  int seq_len = sload(p.seq_lens, X[0]);
  int xt = 0;
  V8 qf[4];
  f32x4 o[8];  // o[mt][r] = O^T[d = 16 mt + 4 q4 + r][g = c]
  float m, l;  // reference max (log2 domain) of g = c; this lane's share of the denominator
  auto open_piece = [&]() {
#pragma unroll
    for (int j = 0; j < 4; ++j) qf[j] = q_lane ? __builtin_bit_cast(V8, piece.q[j]) : V8{};
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  };

  // `valid`: tokens of the tile that count; below 64 on an edge tile.
  auto compute = [&](lds_u8* buf, int valid) __attribute__((always_inline)) {
    const bool edge = valid < kFp4TileTokens;  // wave-uniform
    u32x4 vw[4];  // page i's codes of token lane / 4, group lane % 4
    uint32_t vs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      vw[i] = lds_ld16<u32x4>(buf + kFp4TileV + i * kFp4ScaleOffset + voff);
      vs[i] = buf[kFp4TileVScales + 64 * i + lane];
    }
    u32x4 kw[4];
    float ks[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kw[i] = lds_ld16<u32x4>(buf + kread + i * kFp4ScaleOffset);
      ks[i] = fp4_scale((uint32_t)buf[ksread + 64 * i]);
    }
    f32x4 sc[4];  // sc[i][r] = S[token 4 q4 + r of page i][g = c]
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // The four pages' sums in turn: one alone is a chain of dependent MFMAs.
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[i] = Elem<T>::mfma16(fp4_unpack8<T>(kw[i][j], ks[i]), qf[j], sc[i]);
      __builtin_amdgcn_sched_barrier(0);  // not all conversions at once: registers
    }
    // Rows of pages 2 half and 2 half + 1 over the tile's codes.  LDS works in
    // order for a wavefront: reads before these writes see the codes, and the
    // second half's writes come after the first half's reads.
    auto write_v = [&](int half) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = 2 * half + k;
        u32x4 w = vw[i];
        uint32_t byte = vs[i];
        if (edge) {
          const bool live = kPageSize * i + vtok < valid;
          byte = live ? byte : 127u;
#pragma unroll
          for (int u = 0; u < 4; ++u) w[u] = live ? w[u] : 0u;
        }
        const float scale = fp4_scale(byte);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          lds_st16(buf + k * kDecodePageBytes + vwrite[u], fp4_unpack8<T>(w[u], scale));
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    wave_lds_fence();
    write_v(0);
    if (edge) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (kPageSize * i + 4 * q4 + r >= valid) sc[i][r] = -INFINITY;
    }
    // P = 2^(S * scale - m), packed, and this lane's sum of it.
    V8 pf[2];
    auto exponentials = [&](float m_use) __attribute__((always_inline)) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float pr = fast_exp2(sc[i][r] * p.scale_log2 - m_use);
          sum[r] += pr;
          pf[i >> 1][4 * (i & 1) + r] = (T)pr;
        }
      return (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };
    // The reference maximum moves only when a score exceeds it by more than 8
    // (P stays <= 2^8).  A sum below 128 shows that none does, as every P is
    // below 128 then (2^7.01 covers the rounding of S * scale and m + 8 while
    // |m| < 2^20), so most tiles take no maximum.
    float sum = exponentials(m);
    if (__any(!(sum < 128.f && __builtin_fabsf(m) < 0x1p20f))) {
      float tmax = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
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
    // d-tile mt: tokens 4 q4 .. + 3 of the half's two pages.
    auto read_v = [&](V8 (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        // Chunks of d-tile mt lie 8 chunks, one bit of the slot, from those of mt - 4.
        const lds_u8* a = buf + (mt < 4 ? vread[mt] : vread[mt - 4] ^ 128);
        v[mt] = __builtin_bit_cast(
            V8, __builtin_shufflevector(lds_ld_tr16(a), lds_ld_tr16(a + kDecodePageBytes), 0, 1, 2, 3, 4, 5, 6, 7));
      }
    };
    V8 v[8];
    __builtin_amdgcn_sched_barrier(0);
    wave_lds_fence();
    read_v(v);
    wave_lds_fence();
    __builtin_amdgcn_sched_barrier(0);
    write_v(1);
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[mt] = Elem<T>::mfma16(v[mt], pf[0], o[mt]);
    __builtin_amdgcn_sched_barrier(0);
    wave_lds_fence();
    read_v(v);
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[mt] = Elem<T>::mfma16(v[mt], pf[1], o[mt]);
  };

  // End of piece X: the final output, or its split-K partial (normalised o and
  // log2-sum-exp) for the merge kernel.
  auto finish_piece = [&]() __attribute__((always_inline)) {
    const float l_tot = groups_sum(l);
    const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;
    const int h = X[7];
    if (!q_lane) return;
    if (X[4] == 1) {
      T* op = (T*)p.out + (int64_t)X[6] * p.out_tok_stride + (int64_t)(h * G + c) * p.out_head_stride + 4 * q4;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        V4 w;
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = (T)(o[mt][r] * inv);
        store8_untracked(op + 16 * mt, __builtin_bit_cast(u32x2, w));
      }
      return;
    }
    const int64_t slot = (int64_t)(X[5] + X[3]) * Hkv + h;
    float* po = p.part_o + (slot * G + c) * kHeadDim + 4 * q4;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) store16_device_untracked(po + 16 * mt, __builtin_bit_cast(u32x4, o[mt] * inv));
    if (q4 == 0) store4_device_untracked(&p.part_lse[slot * G + c], l_tot > 0.f ? m + fast_log2(l_tot) : -INFINITY);
  };

  // ---- tile stream: tile k + 1 is copied while tile k is computed -----------
  copy_tile(lds);
  advance();
  open_piece();
  int buf = 0;
  for (;;) {
    lds_u8* const cur = lds + buf * kFp4TileBytes;
    lds_u8* const nxt = lds + (buf ^ 1) * kFp4TileBytes;
    const bool more = fvalid, piece_ends = fnew || !fvalid;
    const i32x8 Y = F;
    const int y_len = sload(p.seq_lens, Y[0]);
    if (more) {
      copy_tile(nxt);
      advance();
    } else {
      __builtin_amdgcn_s_waitcnt(kVmcnt0);
    }
    wave_lds_fence();
    const int begin = X[1] + kFp4TilePages * xt;
    const int valid = min(seq_len, X[2] * kPageSize) - begin * kPageSize;
    compute(cur, valid);
    wave_lds_fence();
    buf ^= 1;
    ++xt;
    if (!piece_ends) continue;
    finish_piece();
    if (!more) break;
    X = Y;
    xt = 0;
    seq_len = y_len;
    open_piece();
  }
  __builtin_amdgcn_s_waitcnt(kVmcnt0);
}

}  // namespace mva
