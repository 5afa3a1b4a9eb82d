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
//  * V: ds_read_b64_tr_b4 turns 16 tokens x 16 dimensions of codes, so that a
//    lane holds one dimension of 16 tokens, the A operand of O^T += V^T P^T.
//    Its scales run along tokens there, so the codes convert with scale 1 and
//    P takes the scales: P_g[t] = P[t] * 2^(b[t][g] - 127) for the four groups
//    g of dimensions.
//  * The tokens of the S^T tiles are dealt so that lane group j gets the 16
//    tokens of page j of the tile, in order: tile i of four takes rows 4i..4i+3
//    of each page.  P then lies as the PV MFMA wants it, without a shuffle.
//  * P is rounded to bf16 for the product, whatever the query's type: its
//    products with the scales need bf16's exponents, and 2^-9 relative is far
//    below the cache's own rounding (up to 2^-3).  Row sums stay in fp32.
//
// Tokens past a sequence's end or its piece get S = -inf and P_g = 0; codes are
// always finite, so nothing else of a stale row can reach the result.
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
// everything before them: page j's codes of K and V from kb[j] / vb[j] (uniform)
// + the lane's offset koff[j] / voff, and both tiles' scales, 4 bytes a lane,
// from ks / vs.  With kQ the query fragments at `q` (4 x 16 bytes) are requested
// first, so the wait covers them too.  One asm statement: see paged_decode.h.
struct Fp4Copy {
  const uint8_t* kb[kFp4TilePages];
  const uint8_t* vb[kFp4TilePages];
  const uint8_t* ks;
  const uint8_t* vs;
};

#define MVA_FP4_TILE_DMA                          \
  "s_mov_b32 %[m0s], m0\n\t"                      \
  "s_mov_b32 m0, %[l]\n\t"                        \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dwordx4 %[ko0], %[k0]\n\t"     \
  "s_add_u32 m0, %[l], 0x400\n\t"                 \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dwordx4 %[ko1], %[k1]\n\t"     \
  "s_add_u32 m0, %[l], 0x800\n\t"                 \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dwordx4 %[ko2], %[k2]\n\t"     \
  "s_add_u32 m0, %[l], 0xc00\n\t"                 \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dwordx4 %[ko3], %[k3]\n\t"     \
  "s_add_u32 m0, %[l], 0x1000\n\t"                \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dwordx4 %[vo], %[v0]\n\t"      \
  "s_add_u32 m0, %[l], 0x1400\n\t"                \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dwordx4 %[vo], %[v1]\n\t"      \
  "s_add_u32 m0, %[l], 0x1800\n\t"                \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dwordx4 %[vo], %[v2]\n\t"      \
  "s_add_u32 m0, %[l], 0x1c00\n\t"                \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dwordx4 %[vo], %[v3]\n\t"      \
  "s_add_u32 m0, %[l], 0x2000\n\t"                \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dword %[ks], off\n\t"          \
  "s_add_u32 m0, %[l], 0x2100\n\t"                \
  "s_nop 0\n\t"                                   \
  "global_load_lds_dword %[vs], off\n\t"          \
  "s_mov_b32 m0, %[m0s]\n\t"                      \
  "s_waitcnt vmcnt(10)"

static_assert(kFp4TileV == 0x1000 && kFp4TileKScales == 0x2000 && kFp4TileVScales == 0x2100, "the copies' LDS layout");

#define MVA_FP4_TILE_IN                                                                                         \
  [l] "s"(lds), [ko0] "v"(koff[0]), [ko1] "v"(koff[1]), [ko2] "v"(koff[2]), [ko3] "v"(koff[3]), [vo] "v"(voff), \
      [k0] "s"(c.kb[0]), [k1] "s"(c.kb[1]), [k2] "s"(c.kb[2]), [k3] "s"(c.kb[3]), [v0] "s"(c.vb[0]),            \
      [v1] "s"(c.vb[1]), [v2] "s"(c.vb[2]), [v3] "s"(c.vb[3]), [ks] "v"(c.ks), [vs] "v"(c.vs)

__device__ inline void fp4_tile_copy(const Fp4Copy& c, const uint32_t (&koff)[4], uint32_t voff, uint32_t lds) {
  uint32_t m0_saved;
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile(MVA_FP4_TILE_DMA : [m0s] "=&s"(m0_saved) : MVA_FP4_TILE_IN : "memory", "scc");
}

__device__ inline void fp4_tile_copy_q(const Fp4Copy& c, const uint32_t (&koff)[4], uint32_t voff, uint32_t lds,
                                       const void* q, u32x4 (&qv)[4]) {
  uint32_t m0_saved;
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile(
      "global_load_dwordx4 %[q0], %[qp], off\n\t"
      "global_load_dwordx4 %[q1], %[qp], off offset:16\n\t"
      "global_load_dwordx4 %[q2], %[qp], off offset:32\n\t"
      "global_load_dwordx4 %[q3], %[qp], off offset:48\n\t" MVA_FP4_TILE_DMA
      : [m0s] "=&s"(m0_saved), [q0] "=&v"(qv[0]), [q1] "=&v"(qv[1]), [q2] "=&v"(qv[2]), [q3] "=&v"(qv[3])
      : MVA_FP4_TILE_IN, [qp] "v"(q)
      : "memory", "scc");
}

#undef MVA_FP4_TILE_DMA
#undef MVA_FP4_TILE_IN

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

  // Per-lane offsets.  A page's codes lie in LDS token by token, 64 bytes each,
  // with 16-byte chunk ch of a token at slot ch ^ j (K, page j of the tile) or
  // ch ^ (token / 4) (V): then the 16 tokens that a K read takes (four of each
  // page) and the 16 of a V read fall on different banks.
  uint32_t koff[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) koff[j] = (uint32_t)((lane >> 2) * kFp4RowBytes + (((lane & 3) ^ j) << 4));
  const uint32_t voff = (uint32_t)((lane >> 2) * kFp4RowBytes + (((lane & 3) ^ (lane >> 4)) << 4));
  const int kread = (c >> 2) * kFp4ScaleOffset + (c & 3) * kFp4RowBytes + ((q4 ^ (c >> 2)) << 4);
  const int ksread = kFp4TileKScales + (c >> 2) * 64 + (c & 3) * 4 + q4;
  int vread[4];
#pragma unroll
  for (int g = 0; g < 4; ++g)
    vread[g] = kFp4TileV + q4 * kFp4ScaleOffset + c * kFp4RowBytes + ((g ^ (c >> 2)) << 4);
  const int vsread = kFp4TileVScales + q4 * 64;

  // The tile to copy next: tile ft of piece F, its page ids, and whether it
  // opens a piece.
  i32x8 F = desc_at(wave);
  int ft = 0;
  bool fvalid = true, fnew = true;
  int ids[kFp4TilePages];
  auto load_ids = [&]() {
    const int32_t* row = p.block_tables + (int64_t)F[0] * p.bt_stride + F[1];
    const int last = max(F[2] - F[1] - 1, 0);
#pragma unroll
    for (int j = 0; j < kFp4TilePages; ++j) ids[j] = sload(row, min(kFp4TilePages * ft + j, last));
  };
  load_ids();
  auto advance = [&]() {
    ++ft;
    fnew = false;
    if (kFp4TilePages * ft >= F[2] - F[1]) {
      fvalid = nx < nx_end;
      if (!fvalid) return;
      F = desc_at(nx);
      ++nx;
      ft = 0;
      fnew = true;
    }
    load_ids();
  };
  u32x4 qn[4];
  const int scale_off = kFp4ScaleOffset + c * kFp4RowScales;
  auto copy_tile = [&](lds_u8* buf) {
    Fp4Copy cp;
    int64_t scale_page = 0;
#pragma unroll
    for (int j = 0; j < kFp4TilePages; ++j) {
      const int id = (ids[j] >= 0 && ids[j] < p.num_pages) ? ids[j] : 0;
      const int64_t off = (int64_t)id * p.page_stride + (int64_t)F[7] * p.head_stride;
      cp.kb[j] = (const uint8_t*)p.k_cache + off;
      cp.vb[j] = (const uint8_t*)p.v_cache + off;
      if (q4 == j) scale_page = off;
    }
    cp.ks = (const uint8_t*)p.k_cache + scale_page + scale_off;
    cp.vs = (const uint8_t*)p.v_cache + scale_page + scale_off;
    const uint32_t at = (uint32_t)(uintptr_t)buf;
    if (fnew) fp4_tile_copy_q(cp, koff, voff, at, q_addr(F), qn);
    else fp4_tile_copy(cp, koff, voff, at);
  };

  i32x8 X = F;  // the piece being computed
  int seq_len = sload(p.seq_lens, X[0]);
  int xt = 0;
  V8 qf[4];
  f32x4 o[8];  // o[mt][r] = O^T[d = 16 mt + 4 q4 + r][g = c]
  float m, l;  // reference max (log2 domain) of g = c; this lane's share of the denominator
  auto open_piece = [&]() {
#pragma unroll
    for (int j = 0; j < 4; ++j) qf[j] = q_lane ? __builtin_bit_cast(V8, qn[j]) : V8{};
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  };

  // `valid`: tokens of the tile that count; below 64 on an edge tile.
  auto compute = [&](const lds_u8* buf, int valid, auto edge_tag) __attribute__((always_inline)) {
    constexpr bool edge = decltype(edge_tag)::value;
    f32x4 sc[4];  // sc[i][r] = S[token 4 i + r of page q4][g = c]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 w = lds_ld16<u32x4>(buf + kread + i * 4 * kFp4RowBytes);
      const float ks = fp4_scale((uint32_t)buf[ksread + 16 * i]);
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j) acc = Elem<T>::mfma16(fp4_unpack8<T>(w[j], ks), qf[j], acc);
      sc[i] = acc;
    }
    const int mine = valid - kPageSize * q4;  // valid tokens of this lane's page
    float tmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (edge) {
          if (4 * i + r >= mine) sc[i][r] = -INFINITY;
        }
        tmax = fmaxf(tmax, sc[i][r]);
      }
    tmax = wave_max16(tmax) * p.scale_log2;  // scale > 0 commutes with max
    // Move the reference max only when it grows by > 8 (p stays <= 2^8).
    const bool grow = tmax > m + 8.0f;
    if (__any(grow)) {
      const float m_new = grow ? tmax : m;
      const float alpha = grow ? fast_exp2(m - m_new) : 1.0f;  // m = -inf -> 0
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) o[mt] *= alpha;
    }
    const float m_use = (m == -INFINITY) ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sc[i][r] = fast_exp2(sc[i][r] * p.scale_log2 - m_use);
        l += sc[i][r];
      }
    u32x4 vs[4];  // vs[i][r]: the four scale bytes of token 4 i + r
#pragma unroll
    for (int i = 0; i < 4; ++i) vs[i] = lds_ld16<u32x4>(buf + vsread + 16 * i);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      bf16x8 pg[2];  // tokens 0-7 and 8-15
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = sc[i][r] * fp4_scale((vs[i][r] >> (8 * g)) & 0xffu);
          if constexpr (edge) {
            if (4 * i + r >= mine) x = 0.f;  // a stale scale may be NaN
          }
          pg[i >> 1][4 * (i & 1) + r] = (__bf16)x;
        }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)(buf + vread[g] + 8 * half));
        f32x4& acc = o[2 * g + half];
        acc = Elem<__bf16>::mfma16(fp4_unpack8<__bf16>((uint32_t)v[0], 1.f), pg[0], acc);
        acc = Elem<__bf16>::mfma16(fp4_unpack8<__bf16>((uint32_t)v[1], 1.f), pg[1], acc);
      }
    }
  };

  // End of piece X: the final output, or its split-K partial (normalised o and
  // log2-sum-exp) for the merge kernel.
  auto finish_piece = [&]() __attribute__((always_inline)) {
    const float l_tot = wave_sum16(l);
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
    if (valid < kFp4TileTokens) compute(cur, valid, std::true_type{});
    else compute(cur, valid, std::false_type{});
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
