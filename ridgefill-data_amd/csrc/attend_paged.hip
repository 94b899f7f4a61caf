// Attention of new tokens of many sequences over a paged K / V cache (bf16 or 4-bit codes), gfx950.
//
// k_paged_few: a few query rows a sequence (one token of each, or some drafted ones). The keys are read once from HBM and
// that read is the bound, so a wave streams them from memory straight into the registers of its products, with no LDS on
// the way: a block takes one K / V head and up to 16 MT query rows (queries x the query heads of the K / V head, query by
// query) of one sequence, its four waves take turns at the key tiles (32 keys) of the block's split. Per tile and wave:
//   S^T = K Q^T on v_mfma_f32_16x16x32_bf16. A's row m of key half kb is key 8 (m / 4) + 4 kb + m % 4 of the tile, so that
//       lane (n, g) (n = lane % 16, g = lane / 16) holds, for query row n, the scores of keys 8 g .. 8 g + 7: the order in
//       which A of the second product wants them. The contraction's order over d is free, too: a lane takes its share of d
//       as memory gives it (bf16: 16-byte chunk 4 s + g in step s; 4 bits: codes of d / 4 consecutive values).
//   Softmax in fp32 base 2, the running maximum raised only when a score exceeds it by 2^8 (lazily: O is rescaled rarely).
//   O += P V on the same MFMA: B's column n of product nb is d = n (D / 16) + nb, so a lane reads D / 16 consecutive values
//       of each of its 8 keys and transposes 2 x 2 with v_perm (half an instruction a value); O's columns of a lane are
//       consecutive in memory again.
// 4-bit codes become bf16 by v_cvt_scalef32_pk_bf16_fp4, scale included, exactly: the arithmetic after it is that of bf16
// pages. The waves' parts are merged through LDS in wave order.
#include <stdint.h>

#include <algorithm>

#include "attend_tile.h"
#include "paged.h"

namespace rf {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int KT = 32;                     // keys a tile of k_paged_few
constexpr int NW = 4;                      // its waves a block

struct PagedArgs {
  const uint16_t* q;
  int64_t ldq, T;
  PagesDev pg;
  const int32_t* table;
  int64_t ld_table;
  int width;                               // pages of a sequence at most
  const int32_t* lens;
  const int32_t* cu;
  int n_seq, hq, hkv, rep, qb;             // qb: queries a block
  int max_rows, max_keys;
  float c;                                 // scale log2(e)
  uint16_t* out;
  int64_t ldo;
  float* part;                             // partials of the splits
  int* length;                             // behind them: the split length, from the splits' launch to the merge
  int fit;                                 // units a head that one round of blocks holds (0: no splits)
  bool once;                               // as many as that at most
  float ov;                                // what a unit costs besides its tiles, in tiles
  int64_t units;                           // units a head that the launch has blocks and the workspace partials for
  int kt, wmin;                            // keys a tile, key tiles a split at least
};

struct Seq {
  int rows, keys, first;                   // new rows, tokens with them, the first row of q
};

// Sequence b, its sizes brought into what the caller's bounds, the table and q hold.
__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int b) {
  const int64_t c0 = a.cu[b], c1 = a.cu[b + 1];
  const int64_t held = min(static_cast<int64_t>(a.width) << a.pg.shift, static_cast<int64_t>(a.max_keys));
  Seq s;
  s.first = static_cast<int>(max<int64_t>(c0, 0));
  s.rows = static_cast<int>(max<int64_t>(0, min(min(c1, a.T) - s.first, static_cast<int64_t>(a.max_rows))));
  s.keys = static_cast<int>(max<int64_t>(0, min<int64_t>(a.lens[b], held)));
  return s;
}

__device__ __forceinline__ int tiles_of(int keys, int kt) { return max(1, (keys + kt - 1) / kt); }

struct Unit {
  int b, rb, sp, ns;                       // sequence (-1: none), row block, split, splits of the sequence
  int W;                                   // key tiles a split
  int64_t part;                            // index of the row block's first split's partial; the next ones are nrb apart
  int nrb;
  Seq s;
};

// Inclusive scan of a wave by data-parallel moves (within rows of 16 lanes, then across them); lane 63 has the total.
template <class F>
__device__ __forceinline__ int wave_scan(int v, int none, F&& f) {
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x111, 0xf, 0xf, false));      // row_shr:1, 2, 4, 8
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x112, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x114, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x118, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xa, 0xf, false));      // row_bcast:15, 31
  return f(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xc, 0xf, false));
}

__device__ __forceinline__ int wave_sum_below(int v, int& total) {              // exclusive prefix sum over 64 lanes
  const int s = wave_scan(v, 0, [](int x, int y) { return x + y; });
  total = __builtin_amdgcn_readlane(s, 63);
  return s - v;
}

__device__ __forceinline__ float wave_sum(float v) {
  return __uint_as_float(__builtin_amdgcn_readlane(
      wave_scan(__float_as_uint(v), 0, [](int x, int y) { return static_cast<int>(__float_as_uint(__uint_as_float(x) + __uint_as_float(y))); }), 63));
}

__device__ __forceinline__ int wave_max(int v) {                                // v >= 0
  return __builtin_amdgcn_readlane(wave_scan(v, 0, [](int x, int y) { return max(x, y); }), 63);
}

// The key tiles of a split. Blocks of one length that fill the GPU once are best; a few more than fill it wait for a second
// round, so splits are as short as one round of blocks allows (fit: its units a head). Where the row blocks alone nearly fill
// it, the length of the least estimated time: all tiles and what each unit costs besides (ov) over the round's blocks, and a
// third of a split for the end (or one round's longest split). 32 sequences of 500 to 8000 keys (bf16, 8 heads): 80 us
// as one round, 85 at 1.25; 48 of 1500 to 24000 in 4 bits 98 against 107; 1499-row chunks of three prompts 521 at three
// rounds, 599 at 1.6. Up to 64 sequences the lanes try 64 lengths each; more of them take a length that
// surely fits. Every block does the same arithmetic on the same sizes: no launch has to plan before this one, and a captured
// graph follows its lens.
__device__ int split_length(const PagedArgs& a, float work, float blocks, int tmax, int nrb0, int tiles0, int lane) {
  const float fit = static_cast<float>(a.fit);
  const bool once = a.once;
  if (a.n_seq > 64) {
    const float W = once ? work / fmaxf(fit - blocks, 1.f) : work / (2.f * fit);
    return max(a.wmin, static_cast<int>(ceilf(W)));
  }
  const float lo = fmaxf(static_cast<float>(a.wmin), ceilf(work / (once ? fit : 3.f * fit)));
  const float hi = fmaxf(static_cast<float>(tmax), lo);
  const float W = ceilf(lo * __builtin_amdgcn_exp2f(__builtin_amdgcn_logf(hi / lo) * (static_cast<float>(lane) / 63.f)));
  const float inv = 1.f / W;
  float units = 0.f;
  for (int b = 0; b < a.n_seq; ++b)
    units += static_cast<float>(__builtin_amdgcn_readlane(nrb0, b)) *
             ceilf(static_cast<float>(__builtin_amdgcn_readlane(tiles0, b)) * inv);
  const float longest = fminf(W, static_cast<float>(tmax));
  float cost = units <= fit ? fmaxf(longest, work / fit) : (work + a.ov * units) / fit + 0.35f * longest;
  // (lane 63's length is every tile: one unit a row block, which always fits)
  if (once && units > fit + 0.5f && lane != 63) cost = 3e38f;
  // the least cost, the shorter length among equals (the bits of positive floats are in order)
  const int bits = static_cast<int>(__float_as_uint(cost)), least = 0x7f800000 - wave_max(0x7f800000 - bits);
  const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(__ballot(bits == least))) - 1);
  return __builtin_amdgcn_readlane(static_cast<int>(W), l);
}

// Unit `want` of the call: units are the (sequence, split, row block)s in that order, row blocks fastest; merging:
// the (sequence, row block)s. (A wave looks at 64 sequences at once.)
__device__ Unit find_unit(const PagedArgs& a, int want, bool merging) {
  const int lane = threadIdx.x & 63;
  int W = 1 << 30;
  Seq s0{0, 0, 0};
  if (lane < a.n_seq) s0 = seq_of(a, lane);
  if (a.fit && merging) {
    W = *a.length;                         // as the launch before this one found it
  } else if (a.fit) {
    float work = 0.f, blocks = 0.f;        // (only the split length depends on them; the same sums in every block)
    int tmax = 1;
    for (int b0 = 0; b0 < a.n_seq; b0 += 64) {
      const Seq s = b0 == 0 ? s0 : b0 + lane < a.n_seq ? seq_of(a, b0 + lane) : Seq{0, 0, 0};
      const float r = static_cast<float>((s.rows + a.qb - 1) / a.qb);
      work += wave_sum(r * static_cast<float>(tiles_of(s.keys, a.kt)));
      blocks += wave_sum(r);
      tmax = max(tmax, wave_max(s.rows ? tiles_of(s.keys, a.kt) : 1));
    }
    W = split_length(a, work, blocks, tmax, (s0.rows + a.qb - 1) / a.qb, tiles_of(s0.keys, a.kt), lane);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.length = W;
  }
  Unit u;
  u.b = -1;
  int before = 0, parts = 0;
  for (int b0 = 0; b0 < a.n_seq; b0 += 64) {
    const Seq s = b0 == 0 ? s0 : b0 + lane < a.n_seq ? seq_of(a, b0 + lane) : Seq{0, 0, 0};
    const int nrb = (s.rows + a.qb - 1) / a.qb, ns = nrb ? (tiles_of(s.keys, a.kt) + W - 1) / W : 0;
    const int n = merging ? nrb : nrb * ns;
    int total, ptotal;
    const int pre = wave_sum_below(n, total);
    const int ppre = merging ? wave_sum_below(nrb * ns, ptotal) : pre;
    if (!merging) ptotal = total;
    if (want < before + total) {
      // (scalar from here on: what follows from a unit is uniform over its block)
      const uint64_t hit = __ballot(n > 0 && before + pre <= want && want < before + pre + n);
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(hit)) - 1);
      const int at = want - before - __builtin_amdgcn_readlane(pre, l);
      u.b = b0 + l;
      u.nrb = __builtin_amdgcn_readlane(nrb, l);
      u.ns = __builtin_amdgcn_readlane(ns, l);
      u.s = Seq{__builtin_amdgcn_readlane(s.rows, l), __builtin_amdgcn_readlane(s.keys, l), __builtin_amdgcn_readlane(s.first, l)};
      u.sp = at / u.nrb;
      u.rb = at - u.sp * u.nrb;
      u.W = W;
      u.part = parts + __builtin_amdgcn_readlane(ppre, l) + u.rb;
      return u;
    }
    before += total;
    parts += ptotal;
  }
  return u;
}

// Key half kb's registers of a tile: the lane's share of d of its key.
template <int D, bool MX>
struct KTile {
  static constexpr int NS = D / 32;                          // 32-deep steps over d
  uint4 x[MX ? 1 : 2][MX ? 1 : NS];                          // bf16
  uint32_t c[MX ? 2 : 1][MX ? D / 32 : 1];                   // codes of D / 4 values
  uint2 sc[MX ? (D == 256 ? 2 : 1) : 1];                     // scales of the 8 keys that the lane's two keys are among
};

template <int D, bool MX>
struct VTile {
  static constexpr int VL = D / 16;                          // consecutive values a lane takes of a key
  uint32_t x[MX ? 1 : 8][MX ? 1 : VL / 2];                   // bf16 pairs of 8 keys
  uint32_t c[MX ? 8 * VL / 8 : 1];                           // codes of 8 keys, key by key
  uint2 sc;
};

template <int D, bool MX>
__device__ __forceinline__ void load_k(KTile<D, MX>& kt, const PagesDev& pg, int64_t id, int head, int tok0, int m, int g) {
  // tok0: the page's token of the 16-key half of the tile that key row m lies in
  const int key = 8 * ((m >> 2) & 1) + (m & 3);              // of that half, for kb = 0
  const char* base = pg.k + id * pg.page_stride + static_cast<int64_t>(head) * pg.head_bytes;
  if constexpr (!MX) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const char* row = base + (tok0 + key + 4 * kb) * (D * 2) + g * 16;
#pragma unroll
      for (int s = 0; s < KTile<D, MX>::NS; ++s) kt.x[kb][s] = *reinterpret_cast<const uint4*>(row + s * 64);
    }
  } else {
    constexpr int LB = D / 8;                                // bytes a lane takes of a key
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const char* row = base + (tok0 + key + 4 * kb) * (D / 2) + g * LB;
      if constexpr (D == 64) {
        const uint2 w = *reinterpret_cast<const uint2*>(row);
        kt.c[kb][0] = w.x;
        kt.c[kb][1] = w.y;
      } else {
#pragma unroll
        for (int i = 0; i < LB / 16; ++i) {
          const uint4 w = *reinterpret_cast<const uint4*>(row + 16 * i);
          kt.c[kb][4 * i] = w.x;
          kt.c[kb][4 * i + 1] = w.y;
          kt.c[kb][4 * i + 2] = w.z;
          kt.c[kb][4 * i + 3] = w.w;
        }
      }
    }
    const uint8_t* sc = pg.ks + id * pg.scale_stride + static_cast<int64_t>(head) * pg.head_scales +
                        ((tok0 + 8 * ((m >> 2) & 1)) >> 3) * (D / 4);
    if constexpr (D == 256) {
      kt.sc[0] = *reinterpret_cast<const uint2*>(sc + (2 * g) * 8);
      kt.sc[1] = *reinterpret_cast<const uint2*>(sc + (2 * g + 1) * 8);
    } else {
      kt.sc[0] = *reinterpret_cast<const uint2*>(sc + (D == 128 ? g : g >> 1) * 8);
    }
  }
}

template <int D, bool MX>
__device__ __forceinline__ void load_v(VTile<D, MX>& vt, const PagesDev& pg, int64_t id, int head, int tok0, int n, int g) {
  const int key = 8 * (g & 1);                               // first of the lane's 8 keys within the 16-key half
  const char* base = pg.v + id * pg.page_stride + static_cast<int64_t>(head) * pg.head_bytes;
  constexpr int VL = D / 16;
  if constexpr (!MX) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const char* row = base + (tok0 + key + e) * (D * 2) + n * (VL * 2);
      if constexpr (VL == 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(row);
        vt.x[e][0] = w.x;
        vt.x[e][1] = w.y;
      } else {
#pragma unroll
        for (int i = 0; i < VL / 8; ++i) {
          const uint4 w = *reinterpret_cast<const uint4*>(row + 16 * i);
          vt.x[e][4 * i] = w.x;
          vt.x[e][4 * i + 1] = w.y;
          vt.x[e][4 * i + 2] = w.z;
          vt.x[e][4 * i + 3] = w.w;
        }
      }
    }
  } else {
    const char* run = base + ((tok0 + key) >> 3) * (4 * D) + n * (VL * 4);    // 8 keys x VL / 2 bytes
#pragma unroll
    for (int i = 0; i < VL / 4; ++i) {
      const uint4 w = *reinterpret_cast<const uint4*>(run + 16 * i);
      vt.c[4 * i] = w.x;
      vt.c[4 * i + 1] = w.y;
      vt.c[4 * i + 2] = w.z;
      vt.c[4 * i + 3] = w.w;
    }
    const uint8_t* sc = pg.vs + id * pg.scale_stride + static_cast<int64_t>(head) * pg.head_scales +
                        ((tok0 + key) >> 3) * (D / 4) + (n * VL / 32) * 8;
    vt.sc = *reinterpret_cast<const uint2*>(sc);
  }
}

// The 32-deep step s of key half kb as an MFMA operand.
template <int D, bool MX>
__device__ __forceinline__ bf16x8 k_frag(const KTile<D, MX>& kt, const float (&scale)[2][2], int kb, int s) {
  if constexpr (!MX) return as_frag(kt.x[kb][s]);
  const uint32_t w = kt.c[kb][s];
  const float f = scale[kb][D == 256 ? s / 4 : 0];
  return as_frag(make_uint4(fp4_pair<0>(w, f), fp4_pair<1>(w, f), fp4_pair<2>(w, f), fp4_pair<3>(w, f)));
}

__device__ __forceinline__ float byte_scale(const uint2& w, int i) {       // i in 0 .. 7, known when inlined or not
  const uint32_t v = i < 4 ? w.x : w.y;
  return __uint_as_float(((v >> (8 * (i & 3))) & 255u) << 23);
}

// V's bf16 pairs of the lane's 8 keys at pair j (d = n VL + 2 j, 2 j + 1), one dword a key.
template <int D, bool MX>
__device__ __forceinline__ void v_pairs(const VTile<D, MX>& vt, const float (&vs)[8], int j, uint32_t (&p)[8]) {
  if constexpr (!MX) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = vt.x[e][j];
  } else {
    constexpr int VB = D / 32;                               // bytes a key
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int byte = e * VB + j;
      const uint32_t w = vt.c[byte / 4];
      switch (byte & 3) {
        case 0: p[e] = fp4_pair<0>(w, vs[e]); break;
        case 1: p[e] = fp4_pair<1>(w, vs[e]); break;
        case 2: p[e] = fp4_pair<2>(w, vs[e]); break;
        default: p[e] = fp4_pair<3>(w, vs[e]); break;
      }
    }
  }
}

__device__ __forceinline__ uint32_t both_low(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t both_high(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

__device__ __forceinline__ bool not_finite(uint32_t pair) {  // either bf16 half is NaN or infinite
  return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}

__device__ __forceinline__ float inverse_sum(float sum) {    // no key seen: zeros (a NaN stays one)
  return sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
}

// N columns from d0 of row r of a row block (query q0 + r / rep): the output, or the partial of a split.
template <int D, int N>
__device__ __forceinline__ void finish_row(const PagedArgs& a, const Unit& u, int64_t part, int rpb, int r, int head, int q0,
                                           int d0, const float (&acc)[N], float top, float sum) {
  if (u.ns > 1) {
    float* p = a.part + part * (static_cast<int64_t>(rpb) * (D + 2));
#pragma unroll
    for (int b = 0; b < N; b += 4)
      *reinterpret_cast<float4*>(p + r * D + d0 + b) = make_float4(acc[b], acc[b + 1], acc[b + 2], acc[b + 3]);
    if (d0 == 0) {
      p[rpb * D + r] = top;
      p[rpb * (D + 1) + r] = sum;
    }
    return;
  }
  const float inv = inverse_sum(sum);
  const int qi = r / a.rep;
  uint16_t* dst = a.out + static_cast<int64_t>(u.s.first + q0 + qi) * a.ldo + (head * a.rep + r - qi * a.rep) * D + d0;
#pragma unroll
  for (int b = 0; b < N; b += 4)
    *reinterpret_cast<uint2*>(dst + b) =
        make_uint2(bf16_pair(acc[b] * inv, acc[b + 1] * inv), bf16_pair(acc[b + 2] * inv, acc[b + 3] * inv));
}

template <int D>
constexpr int merge_floats() { return NW * 16 * (D + 4) + 2 * NW * 16; }

// One tile's registers and what its pages are.
template <int D, bool MX>
struct Tile {
  KTile<D, MX> k;
  VTile<D, MX> v;
  int k0;                                  // first key
  uint32_t bad;                            // bits: a 16-key half on a page that is none
};

// The wave's running state: O [rows 16 mt + 4 g + j][d = n NB + b], and of row 16 mt + n the reference maximum m (raw
// scores; the same in the four lanes of a row) and the lane's share of the row sum.
template <int D, int MT>
struct Rows {
  f32x4 o[MT][D / 16];
  float m[MT], l[MT];
};

__device__ __forceinline__ uint32_t finite_pair(uint32_t p) {  // with zeros for the halves that are NaN or infinite
  p = (p & 0x7f80u) == 0x7f80u ? p & 0xffff0000u : p;
  return (p & 0x7f800000u) == 0x7f800000u ? p & 0xffffu : p;
}

// V's fragments of pair j; CUT: with zeros for the lane's keys past `last` and for what is not finite.
template <int D, bool MX, bool CUT>
__device__ __forceinline__ void v_frags(const VTile<D, MX>& vt, const float (&vs)[8], int j, int last, bf16x8& f0, bf16x8& f1) {
  uint32_t p[8];
  v_pairs<D, MX>(vt, vs, j, p);
  if constexpr (CUT) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = e <= last ? finite_pair(p[e]) : 0u;
  }
  f0 = as_frag(make_uint4(both_low(p[0], p[1]), both_low(p[2], p[3]), both_low(p[4], p[5]), both_low(p[6], p[7])));
  f1 = as_frag(make_uint4(both_high(p[0], p[1]), both_high(p[2], p[3]), both_high(p[4], p[5]), both_high(p[6], p[7])));
}

// What a row meets of V that is not finite, kept apart from the products (there, 0 x infinity would reach rows that do not
// see the key): marks of (row, column), one byte each (1 infinity, 2 -infinity, 4 NaN).
__device__ __forceinline__ uint32_t mark_of(uint32_t half) {
  return (half & 0x7f80u) != 0x7f80u ? 0u : (half & 0x7fu) ? 4u : (half & 0x8000u) ? 2u : 1u;
}

__device__ __forceinline__ float marked(uint32_t m) {
  return (m & 4u) || (m & 3u) == 3u ? NAN : (m & 1u) ? INFINITY : (m & 2u) ? -INFINITY : 0.f;
}

// S^T of a tile: sc[mt][kb][j] = the raw score of key 8 g + 4 kb + j for query row 16 mt + n.
template <int D, bool MX, int MT>
__device__ __forceinline__ void scores(const KTile<D, MX>& kt, const bf16x8 (&qf)[MT][D / 32], f32x4 (&sc)[MT][2], int n) {
  constexpr int NS = D / 32;
  float ks[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
  if constexpr (MX) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int x = 0; x < (D == 256 ? 2 : 1); ++x)
        ks[kb][x] = __uint_as_float((((kb ? kt.sc[x].y : kt.sc[x].x) >> (8 * (n & 3))) & 255u) << 23);
  }
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) sc[mt][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const bf16x8 kf = k_frag<D, MX>(kt, ks, kb, s);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) sc[mt][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[mt][s], sc[mt][kb], 0, 0, 0);
    }
  }
}

__device__ __forceinline__ float lane_max(const f32x4 (&s)[2]) {
  return fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
}

// Raise row block mt's reference maxima to what its rows' four lanes have seen (tmax), and rescale their sums and O.
template <int D, int MT>
__device__ __forceinline__ void raise(Rows<D, MT>& st, int mt, float tmax, float c, int g) {
  tmax = fmaxf(tmax, __shfl_xor(tmax, 16, 64));
  tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
  const float top = fmaxf(st.m[mt], tmax);
  const float alpha = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((st.m[mt] - top) * c);
  st.m[mt] = top;
  st.l[mt] *= alpha;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float al = __shfl(alpha, 4 * g + j, 64);           // O's rows of a lane are 4 g + j
#pragma unroll
    for (int b = 0; b < D / 16; ++b) st.o[mt][b][j] *= al;
  }
}

// The probabilities of a tile as the product's operand; their sum goes to l.
__device__ __forceinline__ bf16x8 probabilities(const f32x4 (&s)[2], float m, float c, float& l) {
  const float mc = m == -INFINITY ? 0.f : m * c;             // (no key seen yet)
  float p[8];
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int j = 0; j < 4; ++j) p[4 * kb + j] = __builtin_amdgcn_exp2f(fmaf(s[kb][j], c, -mc));
  l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
  return as_frag(make_uint4(bf16_pair(p[0], p[1]), bf16_pair(p[2], p[3]), bf16_pair(p[4], p[5]), bf16_pair(p[6], p[7])));
}

// O += P V. CUT: as v_frags.
template <int D, bool MX, int MT, bool CUT>
__device__ __forceinline__ void product(const VTile<D, MX>& vt, const bf16x8 (&pf)[MT], int last, Rows<D, MT>& st) {
  float vs[8];
  if constexpr (MX) {
#pragma unroll
    for (int e = 0; e < 8; ++e) vs[e] = byte_scale(vt.sc, e);
  }
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    bf16x8 f0, f1;
    v_frags<D, MX, CUT>(vt, vs, j, last, f0, f1);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      st.o[mt][2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[mt], f0, st.o[mt][2 * j], 0, 0, 0);
      st.o[mt][2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[mt], f1, st.o[mt][2 * j + 1], 0, 0, 0);
    }
  }
}

// A tile of which some row does not see some key. Keys are hidden from rows by their scores (-infinity); of V, what no row
// sees and what is not finite enters the product as zero, and the latter leaves its marks in the rows that see it.
template <int D, bool MX, int MT>
__device__ __forceinline__ void edge_step(const Tile<D, MX>& tl, const bf16x8 (&qf)[MT][D / 32], const int (&pos)[MT],
                                          Rows<D, MT>& st, float c, int p0, int plast, int rep, int lane, uint32_t* marks) {
  constexpr int NB = D / 16;
  const int n = lane & 15, g = lane >> 4, k0 = tl.k0;
  f32x4 sc[MT][2];
  scores<D, MX, MT>(tl.k, qf, sc, n);
  const bool hidden = (tl.bad >> (g >> 1)) & 1u;             // the lane's 8 keys lie on a page that is none
  bf16x8 pf[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (hidden || k0 + 8 * g + 4 * kb + j > pos[mt]) sc[mt][kb][j] = -INFINITY;
    const float tmax = lane_max(sc[mt]);
    if (__any(tmax > st.m[mt] + RESCALE_LOG2 / c)) raise<D, MT>(st, mt, tmax, c, g);
    pf[mt] = probabilities(sc[mt], st.m[mt], c, st.l[mt]);
  }
  const int last = hidden ? -1 : plast - k0 - 8 * g;         // of the lane's keys, the last that any row sees
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int j = 0; j < NB / 2; ++j) {
      uint32_t two;
      if constexpr (MX) {                                    // 4 bits: only a scale can make values NaN
        if (j) continue;
        two = (((e < 4 ? tl.v.sc.x : tl.v.sc.y) >> (8 * (e & 3))) & 255u) == 255u ? 0x7fff7fffu : 0u;
      } else {
        two = tl.v.x[e][j];
      }
      if (e <= last && not_finite(two)) {
        const uint32_t m2 = mark_of(two & 0xffffu) | mark_of(two >> 16) << 8;
        const int first = max(0, k0 + 8 * g + e - p0) * rep;            // rows from the key's own query on
        for (int r = first; r < min(16 * MT, (plast - p0 + 1) * rep); ++r) {
          if constexpr (MX) {
#pragma unroll
            for (int x = 0; x < NB / 4; ++x) atomicOr(marks + (r * D + n * NB) / 4 + x, 0x04040404u);
          } else {
            atomicOr(marks + (r * D + n * NB + 2 * j) / 4, m2 << (j & 1 ? 16 : 0));
          }
        }
        marks[4 * MT * D] = 1u;
      }
    }
  }
  product<D, MX, MT, true>(tl.v, pf, last, st);
}

// Blocks a CU that the registers of a kernel hold.
constexpr int few_blocks(int d, bool mx, int mt) {
  return d == 64 ? (mt <= 2 ? 3 : mt == 3 ? 2 : 1) : d == 128 ? (mt == 1 && mx ? 3 : mt <= 2 ? 2 : 1) : 1;
}

template <int D, bool MX, int MT>
__global__ __launch_bounds__(64 * NW, (few_blocks(D, MX, MT))) void k_paged_few(PagedArgs a) {
  constexpr int NS = D / 32, NB = D / 16;
  __shared__ float lds[merge_floats<D>() + 4 * MT * D + 1];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), n = lane & 15, g = lane >> 4;
  const int head = blockIdx.x % a.hkv;
  const Unit u = find_unit(a, blockIdx.x / a.hkv, false);
  if (u.b < 0) return;                                       // (uniform over the block: before any barrier)
  const int q0 = u.rb * a.qb, nq = min(a.qb, u.s.rows - q0); // the block's queries
  const int p0 = u.s.keys - u.s.rows + q0;                   // position of the first of them (may lie before 0)
  const int plast = p0 + nq - 1;                             // keys 0 .. plast are read
  const int ntiles = plast < 0 ? 0 : plast / KT + 1;
  const int it0 = u.sp * u.W, it1 = min(ntiles, it0 + u.W);  // (it0 < 2^31: ns W is below tiles + W)

  // The wave's tiles are it0 + w + NW i, i < mine. Lane l holds the page of 16-key half l % 2 of tile i0 + l / 2 of a window
  // of 32 tiles (0 for pages that are none, whose keys `bad` then hides), and the next window's entry on its way.
  const int mine = it0 + w < it1 ? (it1 - it0 - w + NW - 1) / NW : 0;
  const int32_t* row = a.table + static_cast<int64_t>(u.b) * a.ld_table;
  auto entry = [&](int i0) {
    const int it = it0 + w + NW * (i0 + (lane >> 1));
    const int at = (it * 2 + (lane & 1)) >> (a.pg.shift - 4);
    return it < it1 && at < a.width ? row[at] : -1;
  };
  int ids = entry(0), coming = entry(32);
  uint64_t bad;
  auto settle = [&]() {
    const bool out = ids < 0 || ids >= a.pg.n_pages;
    ids = out ? 0 : ids;
    bad = __ballot(out);
  };
  settle();
  const int mask = (1 << a.pg.shift) - 1;
  auto window = [&](int i) {                                 // before the loads of tile i
    if ((i & 31) == 0) {
      ids = coming;
      settle();
      coming = entry(i + 32);
    }
  };
  auto get_k = [&](Tile<D, MX>& tl, int i) {                 // i < mine; windows in order
    const int x = 2 * (i & 31), id0 = __builtin_amdgcn_readlane(ids, x), id1 = __builtin_amdgcn_readlane(ids, x + 1);
    const int k0 = (it0 + w + NW * i) * KT;
    load_k<D, MX>(tl.k, a.pg, n >= 8 ? id1 : id0, head, (k0 + (n >= 8 ? 16 : 0)) & mask, n, g);
  };
  auto get_v = [&](Tile<D, MX>& tl, int i) {
    const int x = 2 * (i & 31), id0 = __builtin_amdgcn_readlane(ids, x), id1 = __builtin_amdgcn_readlane(ids, x + 1);
    tl.k0 = (it0 + w + NW * i) * KT;
    tl.bad = static_cast<uint32_t>(bad >> x) & 3u;
    load_v<D, MX>(tl.v, a.pg, g >= 2 ? id1 : id0, head, (tl.k0 + (g >= 2 ? 16 : 0)) & mask, n, g);
  };

  constexpr int NT = MX || D == 64 ? 2 : 1;                  // tiles at once
  Tile<D, MX> tl[NT];
  if (mine) {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      get_k(tl[x], min(x, mine - 1));
      get_v(tl[x], min(x, mine - 1));
    }
  }
  uint32_t* marks = reinterpret_cast<uint32_t*>(lds + merge_floats<D>());
  for (int x = t; x <= 4 * MT * D; x += 64 * NW) marks[x] = 0u;
  __syncthreads();
  // queries: row 16 mt + n
  bf16x8 qf[MT][NS];
  int pos[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = 16 * mt + n, qi = r / a.rep;
    const bool live = qi < nq;
    pos[mt] = live ? p0 + qi : -1;
    const uint16_t* qrow = a.q + static_cast<int64_t>(u.s.first + q0 + (live ? qi : 0)) * a.ldq +
                           (head * a.rep + (live ? r - qi * a.rep : 0)) * D;
#pragma unroll
    for (int s = 0; s < NS; ++s)
      qf[mt][s] = as_frag(*reinterpret_cast<const uint4*>(qrow + (MX ? g * (D / 4) + 8 * s : 32 * s + 8 * g)));
  }
  Rows<D, MT> st;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    st.m[mt] = -INFINITY;
    st.l[mt] = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) st.o[mt][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Whole tiles first (NT at once; the keys' registers are reloaded behind the scores, the values' behind the product, so
  // that loads are always in flight), then the tiles that some row sees in part; from the first page that is none on all of
  // them are taken as such. A maximum that has to rise leaves the inner loop: with the rescale inside it the compiler moves
  // all of O at every tile (16 to 48 rows of head_dim 256 in 4 bits). Tiles past the last are loaded as the last one again:
  // no load of the loop is conditional.
  const int whole = p0 >= KT - 1 ? min(mine, ((p0 + 1) / KT - it0 - w + NW - 1) / NW) : 0;
  int i = 0;
  bool none = false;
  while (!none && i + NT <= whole) {
    f32x4 sc[NT][MT][2];
    float tmax[MT];
    for (; i + NT <= whole; i += NT) {
      uint32_t bads = 0;
#pragma unroll
      for (int x = 0; x < NT; ++x) bads |= tl[x].bad;
      none = bads != 0;
      if (none) break;
      bool up = false;
#pragma unroll
      for (int x = 0; x < NT; ++x) scores<D, MX, MT>(tl[x].k, qf, sc[x], n);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        tmax[mt] = lane_max(sc[0][mt]);
        if constexpr (NT > 1) tmax[mt] = fmaxf(tmax[mt], lane_max(sc[NT - 1][mt]));
        up |= tmax[mt] > st.m[mt] + RESCALE_LOG2 / a.c;
      }
      if (__any(up)) break;
      const int i1 = min(i + NT, mine - 1);
      if (i1 == i + NT) window(i1);
#pragma unroll
      for (int x = 0; x < NT; ++x) get_k(tl[x], min(i1 + x, mine - 1));
      bf16x8 pf[NT][MT];
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) pf[x][mt] = probabilities(sc[x][mt], st.m[mt], a.c, st.l[mt]);
#pragma unroll
      for (int x = 0; x < NT; ++x) product<D, MX, MT, false>(tl[x].v, pf[x], 8, st);
#pragma unroll
      for (int x = 0; x < NT; ++x) get_v(tl[x], min(i1 + x, mine - 1));
    }
    if (!none && i + NT <= whole) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) raise<D, MT>(st, mt, tmax[mt], a.c, g);
    }
  }
  for (; i < mine; ++i) {
    edge_step<D, MX, MT>(tl[0], qf, pos, st, a.c, p0, plast, a.rep, lane, marks);
    if (i + 1 < mine) {
      window(i + 1);
      get_k(tl[0], i + 1);
      get_v(tl[0], i + 1);
    }
  }

  // merge the waves: thread t takes row t / 16 of each 16 rows and D / 16 columns
  const int64_t part = (u.part + static_cast<int64_t>(u.sp) * u.nrb) * a.hkv + head;
  float* ml = lds + NW * 16 * (D + 4);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (mt) __syncthreads();
    float ls = st.l[mt];
    ls += __shfl_xor(ls, 16, 64);
    ls += __shfl_xor(ls, 32, 64);
    if (g == 0) {
      ml[w * 16 + n] = st.m[mt] == -INFINITY ? st.m[mt] : st.m[mt] * a.c;  // base 2
      ml[(NW + w) * 16 + n] = ls;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int b = 0; b < NB; b += 4)
        *reinterpret_cast<float4*>(lds + (w * 16 + 4 * g + j) * (D + 4) + n * NB + b) =
            make_float4(st.o[mt][b][j], st.o[mt][b + 1][j], st.o[mt][b + 2][j], st.o[mt][b + 3][j]);
    __syncthreads();
    const int rw = t >> 4, d0 = (t & 15) * NB;
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < NW; ++x) top = fmaxf(top, ml[x * 16 + rw]);
    float sum = 0.f, acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float mx = ml[x * 16 + rw];
      const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - top);
      sum += ml[(NW + x) * 16 + rw] * f;
#pragma unroll
      for (int b = 0; b < NB; b += 4) {
        const float4 v = *reinterpret_cast<const float4*>(lds + (x * 16 + rw) * (D + 4) + d0 + b);
        acc[b] += v.x * f;
        acc[b + 1] += v.y * f;
        acc[b + 2] += v.z * f;
        acc[b + 3] += v.w * f;
      }
    }
    const int r = 16 * mt + rw, qi = r / a.rep;
    if (marks[4 * MT * D]) {
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] += marked((marks[(r * D + d0 + b) / 4] >> (8 * (b & 3))) & 255u);
    }
    if (qi < nq) finish_row<D, NB>(a, u, part, 16 * MT, r, head, q0, d0, acc, top, sum);
  }
}

// k_paged_many: many query rows a sequence (a chunk of a prompt). A block takes 256 query rows (queries x the query heads of
// a K / V head) of one sequence, 32 a wave, and the key tiles of its split through LDS, each read by all eight waves:
// attend_causal.hip's tile (S^T = K Q^T, P^T straight from the score registers, V^T by transpose reads), with rows of any
// query and head side by side in a wave, so that any group size fills it. Tiles come from pages: bf16 by direct loads, three
// tiles in flight, the page of each load's rows (never more than 16) read off a lane; 4 bits through registers, a tile's
// codes loaded while the one before it is converted into LDS, once for all eight waves (160 of a tile's 2000 cycles).
// Bound by the products and the softmax beside them (64 keys: 1024 cycles of MFMA a wave, two waves a SIMD).
template <int AD, bool MX>
struct ManyCodes {
  uint2 k, v;                              // codes of 16 values (8 at head_dim 64)
  uint32_t ks, vs;                         // their scale bytes
};

// The wave's 16-key half of a tile that it loads: rows of one page.
template <int AD>
__device__ __forceinline__ int half_of_wave(int w) { return AD == 256 ? w >> 2 : w >> 1; }

// A thread's codes of a tile whose half lies at token tok0 of page id.
template <int AD>
__device__ __forceinline__ void load_codes(ManyCodes<AD, true>& c, const PagesDev& pg, int id, int head, int tok0, int w, int lane) {
  const int64_t at = static_cast<int64_t>(id) * pg.page_stride + static_cast<int64_t>(head) * pg.head_bytes;
  const int64_t sat = static_cast<int64_t>(id) * pg.scale_stride + static_cast<int64_t>(head) * pg.head_scales;
  constexpr int TPR = AD == 256 ? 16 : 8;                    // threads a key row (8 bytes each; 4 at head_dim 64)
  const int row = (AD == 256 ? 4 * (w & 3) : 8 * (w & 1)) + lane / TPR, part = lane % TPR;
  const char* kp = pg.k + at + (tok0 + row) * (AD / 2) + part * (AD / 2 / TPR);
  if constexpr (AD == 64) c.k.x = *reinterpret_cast<const uint32_t*>(kp);
  else c.k = *reinterpret_cast<const uint2*>(kp);
  c.ks = pg.ks[sat + ((tok0 + row) >> 3) * (AD / 4) + (part * (AD / TPR) / 32) * 8 + (row & 7)];
  // values: 8 tokens' runs; d 128: two tokens of a run of 8 values, 256: one of 16, 64: one of two runs of 4
  const int grp = AD == 256 ? (w >> 1) & 1 : w & 1;
  const char* vp = pg.v + at + ((tok0 >> 3) + grp) * (4 * AD);
  const uint8_t* sp = pg.vs + sat + ((tok0 >> 3) + grp) * (AD / 4);
  if constexpr (AD == 128) {
    c.v = *reinterpret_cast<const uint2*>(vp + lane * 8);
    c.vs = *reinterpret_cast<const uint16_t*>(sp + ((lane >> 2) / 4) * 8 + 2 * (lane & 3));
  } else if constexpr (AD == 256) {
    const int x = 64 * (w & 1) + lane;
    c.v = *reinterpret_cast<const uint2*>(vp + x * 8);
    c.vs = sp[((x >> 3) / 2) * 8 + (x & 7)];
  } else {
    const int cc = lane >> 3, key = lane & 7;
    c.v.x = *reinterpret_cast<const uint16_t*>(vp + (2 * cc) * 16 + 2 * key) |
            static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(vp + (2 * cc + 1) * 16 + 2 * key)) << 16;
    c.vs = sp[(cc / 4) * 8 + key];
  }
}

__device__ __forceinline__ uint4 eight_values(uint32_t w, float s) {
  return make_uint4(fp4_pair<0>(w, s), fp4_pair<1>(w, s), fp4_pair<2>(w, s), fp4_pair<3>(w, s));
}

// ... as bf16 into a stage.
template <int AD>
__device__ __forceinline__ void store_codes(const ManyCodes<AD, true>& c, char* st, int w, int lane) {
  using L = Layout<AD>;
  constexpr int TPR = AD == 256 ? 16 : 8;
  const int row = (AD == 256 ? 4 : 8) * w + lane / TPR, part = lane % TPR;
  uint4* s4 = reinterpret_cast<uint4*>(st);
  const float ks = scale_of<0>(c.ks), vs = scale_of<0>(c.vs);
  if constexpr (AD == 64) {
    s4[L::kslot(row, part)] = eight_values(c.k.x, ks);
    s4[L::vslot(8 * w + (lane & 7), lane >> 3)] = eight_values(c.v.x, vs);
  } else {
    s4[L::kslot(row, 2 * part)] = eight_values(c.k.x, ks);
    s4[L::kslot(row, 2 * part + 1)] = eight_values(c.k.y, ks);
    if constexpr (AD == 128) {
      const int r = 8 * w + 2 * (lane & 3);
      s4[L::vslot(r, lane >> 2)] = eight_values(c.v.x, vs);
      s4[L::vslot(r + 1, lane >> 2)] = eight_values(c.v.y, scale_of<1>(c.vs));
    } else {
      const int x = 64 * (w & 1) + lane, r = 8 * (w >> 1) + (x & 7);
      s4[L::vslot(r, 2 * (x >> 3))] = eight_values(c.v.x, vs);
      s4[L::vslot(r, 2 * (x >> 3) + 1)] = eight_values(c.v.y, vs);
    }
  }
}

// tile_step for a tile of which some row does not see some key, without the next tile's scores: bad has a bit a 16-key half
// on a page that is none. Of V, what is not finite enters the product as zero; a row that sees such a value takes it
// from LDS afterwards (0 x infinity must not reach the rows that do not).
template <int AD>
__device__ __forceinline__ void edge_tile(const char* __restrict__ st, f32x16 (&sc)[Cfg<AD>::KB], f32x16 (&o)[AD / 32],
                                          float& mref, float& lsum, int k0, uint32_t bad, int mypos, int hh, float c,
                                          const FragOffsets<AD>& fo) {
  using L = Layout<AD>;
  constexpr int NB = AD / 32, KB = Cfg<AD>::KB, KTL = Cfg<AD>::KT, NP = 8 * KB;
  const int rel = min(max(mypos - k0, -1), KTL) - 4 * hh;
  float tmax = -INFINITY;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const bool gone = (bad >> (2 * kb + (j >> 3))) & 1u;   // keys 32 kb + 8 (j / 4) + ..
      if (gone || 32 * kb + 8 * (j >> 2) + (j & 3) > rel) sc[kb][j] = -INFINITY;
      tmax = fmaxf(tmax, sc[kb][j]);
    }
  float lo, hi;
  lane_pair(tmax, lo, hi);
  tmax = fmaxf(lo, hi);
  if (tmax > mref + RESCALE_LOG2 / c) {
    const float alpha = __builtin_amdgcn_exp2f((mref - tmax) * c);
    mref = tmax;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][r] *= alpha;
    lsum *= alpha;
  }
  const float mc = mref == -INFINITY ? 0.f : mref * c;
  float psum = 0.f;
  uint32_t pk[NP];
#pragma unroll
  for (int e = 0; e < NP; ++e) {
    const float q0 = __builtin_amdgcn_exp2f(fmaf(sc[e / 8][2 * (e % 8)], c, -mc));
    const float q1 = __builtin_amdgcn_exp2f(fmaf(sc[e / 8][2 * (e % 8) + 1], c, -mc));
    psum += q0 + q1;
    pk[e] = bf16_pair(q0, q1);
  }
  lsum += psum;
  bool odd = false;
#pragma unroll
  for (int stp = 0; stp < KTL / 16; ++stp) {
    const bf16x8 pf = __builtin_bit_cast(bf16x8, make_uint4(pk[4 * stp], pk[4 * stp + 1], pk[4 * stp + 2], pk[4 * stp + 3]));
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const char* vp = st + fo.v(b) + 16 * stp * L::KCPR * 16;
      uint2 vl = read_tr(vp), vh = read_tr(vp + 8 * L::KCPR * 16);
      odd |= not_finite(vl.x) || not_finite(vl.y) || not_finite(vh.x) || not_finite(vh.y);
      vl = make_uint2(finite_pair(vl.x), finite_pair(vl.y));
      vh = make_uint2(finite_pair(vh.x), finite_pair(vh.y));
      o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_frag(make_uint4(vl.x, vl.y, vh.x, vh.y)), pf, o[b], 0, 0, 0);
    }
  }
  if (!__any(odd)) return;
  for (int kk = 0; kk < KTL; ++kk) {
    if (((bad >> (kk >> 4)) & 1u) || k0 + kk > mypos) continue;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {                          // d = 32 b + 8 g + 4 hh + 0 .. 3
        const uint2 v = *reinterpret_cast<const uint2*>(st + L::vslot(kk, 4 * b + g) * 16 + 8 * hh);
        o[b][4 * g] += marked(mark_of(v.x & 0xffffu));
        o[b][4 * g + 1] += marked(mark_of(v.x >> 16));
        o[b][4 * g + 2] += marked(mark_of(v.y & 0xffffu));
        o[b][4 * g + 3] += marked(mark_of(v.y >> 16));
      }
  }
}

template <int AD, bool MX>
__global__ __launch_bounds__(Cfg<AD>::NTHR, 1) void k_paged_many(PagedArgs a) {
  using L = Layout<AD>;
  constexpr int NS = AD / 16, NB = AD / 32, KTL = Cfg<AD>::KT, QROWS = Cfg<AD>::QROWS, KB = Cfg<AD>::KB;
  constexpr int HPT = KTL / 16, WIN = 64 / HPT;              // 16-key halves a tile, tiles a window of table entries
  __shared__ uint4 lds[NSTAGE * L::STAGE_U4];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), n = lane & 31, hh = lane >> 5;
  // heads fastest within a unit's row blocks: a head's row blocks of one split lie hkv blocks apart
  const int head = blockIdx.x % a.hkv;
  const Unit u = find_unit(a, blockIdx.x / a.hkv, false);
  if (u.b < 0) return;                                       // (uniform over the block: before any barrier)
  const int q0 = u.rb * a.qb, nq = min(a.qb, u.s.rows - q0), rows = nq * a.rep;
  const int p0 = u.s.keys - u.s.rows + q0, plast = p0 + nq - 1;
  const int ntiles = plast < 0 ? 0 : plast / KTL + 1;
  const int it0 = u.sp * u.W, it1 = min(ntiles, it0 + u.W);

  // row 32 w + n: query r / rep, head r % rep; lanes past the last row repeat it and write nothing
  const int r = min(32 * w + n, rows - 1), qi = r / a.rep;
  const bool live = 32 * w + n < rows;
  const int mypos = p0 + qi;
  const int wave_last = 32 * w < rows ? p0 + min(32 * w + 31, rows - 1) / a.rep : -1;
  bf16x8 qf[NS];
  {
    const uint16_t* qrow = a.q + static_cast<int64_t>(u.s.first + q0 + qi) * a.ldq + (head * a.rep + r - qi * a.rep) * AD + 8 * hh;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = as_frag(*reinterpret_cast<const uint4*>(qrow + 16 * s));
  }

  // pages: lane l holds the entry of half l % HPT of tile l / HPT of a window of WIN tiles (0 for none, with its bit of bad)
  const int32_t* row = a.table + static_cast<int64_t>(u.b) * a.ld_table;
  auto entry = [&](int win) {
    const int it = it0 + win * WIN + lane / HPT;
    const int at = (it * HPT + lane % HPT) >> (a.pg.shift - 4);
    return it < it1 && at < a.width ? row[at] : -1;
  };
  int ids = entry(0), coming = entry(1), window = 0;
  uint64_t bad = 0, bad_before = 0;
  auto settle = [&]() {
    const bool out = ids < 0 || ids >= a.pg.n_pages;
    ids = out ? 0 : ids;
    bad_before = bad;
    bad = __ballot(out);
  };
  settle();
  wait_vm_lgkm0<0>();        // queries and entries are in registers before any tile load is in flight
  auto advance = [&](int it) {                               // before tile it is loaded; tiles in order
    if ((it - it0) / WIN != window) {
      ++window;
      ids = coming;
      settle();
      coming = entry(window + 1);
    }
  };
  auto bad_of = [&](int it) {
    const int win = (it - it0) / WIN, x = ((it - it0) % WIN) * HPT;
    return static_cast<uint32_t>((win == window ? bad : bad_before) >> x) & ((1u << HPT) - 1u);
  };
  const int mask = (1 << a.pg.shift) - 1;
  char* base = reinterpret_cast<char*>(lds);
  auto stage = [&](int it) { return base + ((it - it0) % NSTAGE) * L::STAGE_U4 * 16; };
  auto id_of = [&](int it, int half) { return __builtin_amdgcn_readlane(ids, ((it - it0) % WIN) * HPT + half); };

  // bf16: instruction i of wave w fills 64 consecutive 16-byte slots, rows row0 .. of one half; the lane's slot gives the row
  // and the chunk it fetches
  [[maybe_unused]] auto issue = [&](int it) {
    advance(it);
    char* st = stage(it);
#pragma unroll
    for (int i = 0; i < L::KLOADS; ++i) {
      constexpr int RPI = 64 / L::KCPR;
      const int row0 = (w * L::KLOADS + i) * RPI, half = row0 >> 4;
      const int tok = (it * KTL + row0) & mask;
      const int64_t at = static_cast<int64_t>(id_of(it, half)) * a.pg.page_stride + static_cast<int64_t>(head) * a.pg.head_bytes +
                         static_cast<int64_t>(tok) * (AD * 2);
      const int rl = lane / L::KCPR, pc = lane % L::KCPR;
      const uint32_t ko = static_cast<uint32_t>(rl * (AD * 2) + (pc ^ ((row0 + rl) & (L::KCPR - 1))) * 16);
      const uint32_t vo = static_cast<uint32_t>(rl * (AD * 2) + (pc ^ (4 * L::vsw(row0 + rl))) * 16);
      const __amdgpu_buffer_rsrc_t rk = buffer_rsrc(a.pg.k + at, 1024u), rv = buffer_rsrc(a.pg.v + at, 1024u);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_ptr)(st + (w * L::KLOADS + i) * 1024), 16, ko, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_ptr)(st + (L::K_U4 + (w * L::VLOADS + i) * 64) * 16), 16, vo, 0, 0, 0);
    }
  };
  // 4 bits: the tile's codes into registers
  [[maybe_unused]] ManyCodes<AD, true> codes;
  [[maybe_unused]] auto fetch = [&](int it) {
    advance(it);
    const int half = half_of_wave<AD>(w);
    load_codes<AD>(codes, a.pg, id_of(it, half), head, (it * KTL + 16 * half) & mask, w, lane);
  };

  f32x16 o[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int x = 0; x < 16; ++x) o[b][x] = 0.f;
  float m = -INFINITY, lsum = 0.f;
  const float c = a.c;
  const FragOffsets<AD> fo(lane);
  f32x16 sc[KB], sn[KB];
  // Turn it, then softmax and product of tile it, with the scores of tile it + 1 in the same block. bf16: tile it + 3 is
  // loaded into the stage of tile it - 1, whose last reads ended before this iteration's barrier. 4 bits: the codes of tile
  // it + 2 go to its stage (tile it - 2's) and those of tile it + 3 to registers; the next barrier makes the stage visible.
  if constexpr (MX) {
    for (int i = 0; i < 2; ++i)
      if (it0 + i < it1) {
        fetch(it0 + i);
        store_codes<AD>(codes, stage(it0 + i), w, lane);
      }
    if (it0 + 2 < it1) fetch(it0 + 2);
    __syncthreads();
  } else {
    for (int i = 0; i < 3; ++i)
      if (it0 + i < it1) issue(it0 + i);
    if (it0 + 2 < it1) wait_vm_lgkm0<2 * L::LOADS>();        // tile it0 landed
    else if (it0 + 1 < it1) wait_vm_lgkm0<L::LOADS>();
    else wait_vm_lgkm0<0>();
    __builtin_amdgcn_s_barrier();
  }
  if (it0 < it1) tile_scores<AD>(stage(it0), qf, sc, fo);
  auto turn = [&](int it) {
    if constexpr (MX) {
      __syncthreads();
      if (it + 2 < it1) store_codes<AD>(codes, stage(it + 2), w, lane);
      if (it + 3 < it1) fetch(it + 3);
    } else {
      if (it + 2 < it1) wait_vm_lgkm0<L::LOADS>();           // tile it + 1 landed, tile it + 2 may fly
      else wait_vm_lgkm0<0>();
      __builtin_amdgcn_s_barrier();                          // every wave's share of it has landed and every
      if (it + 3 < it1) issue(it + 3);                       // wave is done with the stage reloaded here
    }
  };
  // Tiles that every row of the block sees whole, in pairs (the scores' buffers swap roles), up to the first page that is
  // none (uniform over the block, as the barriers need); then the others, whose code stays out of this loop's registers.
  if (32 * w >= rows) {                                      // a wave without rows: its share of the loads and the barriers
    for (int it = it0; it < it1; ++it) turn(it);
    return;
  }
  const int full = p0 >= KTL - 1 ? min(it1, (p0 + 1) / KTL) : it0;
  int it = it0;
  if constexpr (AD == 256) {                                 // (one buffer's copy each: in pairs it spills)
    for (; it < full; ++it) {
      if (bad_of(it)) break;
      turn(it);
      tile_step<AD>(stage(it), stage(it + 1), qf, sc, sn, o, m, lsum, it * KTL, false, mypos, hh, c, fo);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) sc[kb] = sn[kb];
    }
  } else {
    for (; it + 1 < full; it += 2) {
      if (bad_of(it) | bad_of(it + 1)) break;
      turn(it);
      tile_step<AD>(stage(it), stage(it + 1), qf, sc, sn, o, m, lsum, it * KTL, false, mypos, hh, c, fo);
      turn(it + 1);
      tile_step<AD>(stage(it + 1), stage(it + 2), qf, sn, sc, o, m, lsum, it * KTL + KTL, false, mypos, hh, c, fo);
    }
  }
  for (; it < it1; ++it) {
    turn(it);
    if (it * KTL > wave_last) continue;                      // this and every later tile lie past the wave's rows
    edge_tile<AD>(stage(it), sc, o, m, lsum, it * KTL, bad_of(it), mypos, hh, c, fo);
    tile_scores<AD>(stage(it + 1), qf, sc, fo);
  }
  wait_vm_lgkm0<0>();

  // lane holds O[row n][d = 32 b + 8 (j / 4) + 4 hh + j % 4]
  float llo, lhi;
  lane_pair(lsum, llo, lhi);
  const float ltot = llo + lhi;
  if (!live) return;
  if (u.ns > 1) {
    const int64_t part = (u.part + static_cast<int64_t>(u.sp) * u.nrb) * a.hkv + head;
    float* pb = a.part + part * (static_cast<int64_t>(QROWS) * (AD + 2));
    float* orow = pb + r * AD + 4 * hh;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(orow + 32 * b + 8 * g) = make_float4(o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2],
                                                                        o[b][4 * g + 3]);
    if (hh == 0) {
      pb[QROWS * AD + r] = m == -INFINITY ? m : m * c;
      pb[QROWS * (AD + 1) + r] = ltot;
    }
    return;
  }
  const float inv = inverse_sum(ltot);
  uint16_t* dst = a.out + static_cast<int64_t>(u.s.first + q0 + qi) * a.ldo + (head * a.rep + r - qi * a.rep) * AD + 4 * hh;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2*>(dst + 32 * b + 8 * g) =
          make_uint2(bf16_pair(o[b][4 * g] * inv, o[b][4 * g + 1] * inv), bf16_pair(o[b][4 * g + 2] * inv, o[b][4 * g + 3] * inv));
}

// Merges the splits of a row block and head: D / 4 lanes a row (4 columns each); the block's lanes beyond its rows make G
// groups a row, group i takes splits i, i + G, .. (eight in flight) with a running maximum, and the groups are joined in
// order through LDS. The order depends on the sizes alone. blockIdx.y takes a share of the rows where few row blocks leave
// CUs idle.
constexpr int MERGE_THREADS = 1024;
template <int D>
__global__ __launch_bounds__(MERGE_THREADS) void k_paged_merge(PagedArgs a, int rpb) {
  constexpr int LPR = D / 4, U = 8;
  __shared__ float4 ls[MERGE_THREADS];
  __shared__ float lm[MERGE_THREADS / LPR], ll[MERGE_THREADS / LPR];
  const int t = threadIdx.x, head = blockIdx.x % a.hkv, slots = blockDim.x / LPR, slot = t / LPR, col = 4 * (t % LPR);
  const Unit u = find_unit(a, blockIdx.x / a.hkv, true);
  // (partials past the last unit: only with a cu that does not rise, whose units the launch does not hold)
  if (u.b < 0 || u.ns == 1 || u.part + static_cast<int64_t>(u.ns - 1) * u.nrb >= a.units) return;
  const int q0 = u.rb * a.qb, rows = min(a.qb, u.s.rows - q0) * a.rep;
  const int per = (rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
  if (r0 >= r1) return;
  int G = 1;
  while (2 * G * (r1 - r0) <= slots && 2 * G <= u.ns) G *= 2;
  const int grp = slot % G;
  const float* p0 = a.part + (u.part * a.hkv + head) * (static_cast<int64_t>(rpb) * (D + 2));
  const int64_t step = static_cast<int64_t>(u.nrb) * a.hkv * (static_cast<int64_t>(rpb) * (D + 2));
  for (int rb = r0; rb < r1; rb += slots / G) {              // (uniform)
    const int r = rb + slot / G, rc = min(r, r1 - 1);
    const float* pv = p0 + static_cast<int64_t>(rc) * D + col;
    const float* ms = p0 + static_cast<int64_t>(rpb) * D + rc;
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = grp; s0 < u.ns; s0 += U * G) {
      float4 v[U];
      float m[U], l[U];
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int64_t s = min(s0 + x * G, u.ns - 1);
        m[x] = ms[s * step];
        l[x] = ms[s * step + rpb];
        v[x] = *reinterpret_cast<const float4*>(pv + s * step);
      }
      float now = top;
#pragma unroll
      for (int x = 0; x < U; ++x) now = fmaxf(now, s0 + x * G < u.ns ? m[x] : -INFINITY);
      const float f0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
      top = now;
      sum *= f0;
      acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
#pragma unroll
      for (int x = 0; x < U; ++x) {
        if (s0 + x * G >= u.ns) break;                       // (uniform over a group)
        const float f = m[x] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[x] - top);
        sum += l[x] * f;
        acc.x += v[x].x * f;
        acc.y += v[x].y * f;
        acc.z += v[x].z * f;
        acc.w += v[x].w * f;
      }
    }
    if (G > 1) {
      __syncthreads();                                       // the last rows' groups were read
      ls[t] = acc;
      if (col == 0) {
        lm[slot] = top;
        ll[slot] = sum;
      }
      __syncthreads();
      if (grp == 0) {
        const int first = slot;
        for (int x = 0; x < G; ++x) top = fmaxf(top, lm[first + x]);
        sum = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int x = 0; x < G; ++x) {
          const float m = lm[first + x], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
          const float4 v = ls[t + x * LPR];
          sum += ll[first + x] * f;
          acc.x += v.x * f;
          acc.y += v.y * f;
          acc.z += v.z * f;
          acc.w += v.w * f;
        }
      }
    }
    if (grp == 0 && r < r1) {
      const float inv = inverse_sum(sum);
      const int qi = r / a.rep;
      uint16_t* dst = a.out + static_cast<int64_t>(u.s.first + q0 + qi) * a.ldo + (head * a.rep + r - qi * a.rep) * D + col;
      *reinterpret_cast<uint2*>(dst) = make_uint2(bf16_pair(acc.x * inv, acc.y * inv), bf16_pair(acc.z * inv, acc.w * inv));
    }
  }
}

// 16-row blocks a wave takes: as few as hold a sequence's rows (their state and queries live in registers: up to 4, 3 at
// head_dim 256).
int row_tiles(int rep, int d, int64_t max_rows) {
  return static_cast<int>(std::min<int64_t>(d == 256 ? 3 : 4, (max_rows * rep + 15) / 16));
}

struct Plan {
  bool many, once;
  int mt, qb, fit, kt;                     // mt: 16-row blocks of k_paged_few
  int64_t blocks, units;                   // (sequence, row block)s at most, and with their splits
  size_t bytes;
  int rows() const { return many ? Cfg<128>::QROWS : 16 * mt; }
};

// The launch for these sizes: a sequence's rows in the registers of k_paged_few's waves, or more of them through
// k_paged_many. Row blocks: sum of ceil(rows / qb) <= T / qb + n_seq. With splits of W tiles at most work / W units more
// (split_length: one round of blocks, or W >= work / 3 fit).
Plan plan_of(int64_t T, int hq, int hkv, int d, bool mx, int n_seq, int64_t max_rows, int64_t max_keys) {
  Plan p{};
  const int rep = hq / hkv;
  p.many = std::min<int64_t>(max_rows, T) * rep > (d == 256 ? 48 : 64);
  p.mt = p.many ? 0 : row_tiles(rep, d, std::min<int64_t>(max_rows, T));
  p.qb = p.rows() / rep;
  p.kt = p.many ? (d == 256 ? Cfg<256>::KT : Cfg<128>::KT) : KT;
  p.blocks = std::min<int64_t>(T, T / p.qb + n_seq);
  const int round = p.many ? 256 : 256 * few_blocks(d, mx, p.mt);
  p.fit = max_keys <= 16 * NW * KT ? 0 : std::max(1, round / hkv);
  p.once = p.blocks * 4 <= static_cast<int64_t>(p.fit) * 3;
  p.units = !p.fit ? p.blocks : p.once ? p.fit : 3 * p.fit + 1 + p.blocks;
  p.bytes = p.fit ? static_cast<size_t>(p.units) * hkv * (p.rows() * (d + 2)) * 4 + 16 : 0;
  return p;
}

int attend_sizes(const char* fn, int64_t T, int hq, int hkv, int d, int kind, int n_seq, int64_t max_rows, int64_t max_keys) {
  if (d != 64 && d != 128 && d != 256) return fail(RF_EUNSUPPORTED, "%s: head_dim %d (the kernels take 64, 128, 256)", fn, d);
  if (hq <= 0 || hkv <= 0 || hkv > 4096 || hq % hkv || hq / hkv > 64)
    return fail(RF_EUNSUPPORTED, "%s: %d query heads over %d K / V heads (groups of up to 64)", fn, hq, hkv);
  if (kind != RF_PAGES_BF16 && kind != RF_PAGES_MX4) return fail(RF_EINVAL_ARG, "%s: kind of pages %d", fn, kind);
  if (T < 0 || T > (1 << 24) || n_seq < 0 || n_seq > (1 << 20) || max_rows < 0 || max_keys < 0 || max_keys > (1 << 27))
    return fail(RF_EINVAL_SHAPE, "%s: %lld rows of %d sequences, at most %lld rows and %lld keys each", fn, (long long)T, n_seq,
                (long long)max_rows, (long long)max_keys);
  return RF_OK;
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" int rf_attend_paged_workspace_bytes(int64_t T, int hq, int hkv, int d, int kind, int n_seq, int64_t max_rows,
                                               int64_t max_keys, size_t* bytes) {
  const char* fn = "rf_attend_paged_workspace_bytes";
  if (!bytes) return fail(RF_EINVAL_ARG, "%s: null pointer", fn);
  if (int rc = attend_sizes(fn, T, hq, hkv, d, kind, n_seq, max_rows, max_keys)) return rc;
  *bytes = T && n_seq && max_rows ? plan_of(T, hq, hkv, d, kind == RF_PAGES_MX4, n_seq, max_rows, max_keys).bytes : 0;
  return RF_OK;
}

extern "C" int rf_attend_paged(const uint16_t* q, int64_t ldq, int64_t T, int hq, const rf_pages* pages,
                               const int32_t* table, int64_t ld_table, int64_t table_width, const int32_t* lens,
                               const int32_t* cu, int n_seq, int64_t max_rows, int64_t max_keys, float scale, uint16_t* out,
                               int64_t ldo, void* workspace, size_t ws_bytes, hipStream_t stream) {
  const char* fn = "rf_attend_paged";
  PagesDev pg;
  if (int rc = check_pages(fn, pages, &pg)) return rc;
  const int d = pages->d, hkv = pages->hkv;
  if (!q || !table || !lens || !cu || !out) return fail(RF_EINVAL_ARG, "%s: null pointer", fn);
  if (int rc = attend_sizes(fn, T, hq, hkv, d, pages->kind, n_seq, max_rows, max_keys)) return rc;
  if (ldq < static_cast<int64_t>(hq) * d || ldo < static_cast<int64_t>(hq) * d || ldq % 8 || ldo % 4 || table_width < 0 ||
      table_width > (1 << 26) || ld_table < table_width)
    return fail(RF_EINVAL_SHAPE, "%s: strides (q %lld, out %lld) or a table %lld wide (row stride %lld)", fn, (long long)ldq,
                (long long)ldo, (long long)table_width, (long long)ld_table);
  if (!aligned16(q) || (reinterpret_cast<uintptr_t>(out) & 7u) || (workspace && !aligned16(workspace)))
    return fail(RF_EINVAL_SHAPE, "%s: alignment", fn);
  if (!(scale > 0.f) || !(scale < 1e30f))
    return fail(RF_EINVAL_ARG, "%s: scale %g (must be positive)", fn, static_cast<double>(scale));
  if (T == 0 || n_seq == 0 || max_rows == 0) return RF_OK;
  Plan p = plan_of(T, hq, hkv, d, pages->kind == RF_PAGES_MX4, n_seq, max_rows, max_keys);
  if (p.fit && (!workspace || ws_bytes < p.bytes)) {
    p.fit = 0;
    p.units = p.blocks;
  }
  const PagedArgs a{q, ldq, T, pg, table, ld_table, static_cast<int>(table_width), lens, cu, n_seq, hq, hkv, hq / hkv, p.qb,
                    static_cast<int>(std::min<int64_t>(max_rows, T)), static_cast<int>(max_keys),
                    scale * 1.4426950408889634f, out, ldo, static_cast<float*>(workspace),
                    p.fit ? reinterpret_cast<int*>(static_cast<char*>(workspace) + p.bytes) - 4 : nullptr, p.fit, p.once, p.many ? 3.f : 1.f, p.units, p.kt,
                    p.many ? 4 : 2 * NW};
  const dim3 grid(static_cast<unsigned>(p.units * hkv));
  // the merge: a block a row block and head, or a share of its rows; wide blocks where they are few
  const int64_t pairs = p.blocks * hkv, rows = std::min<int64_t>(static_cast<int64_t>(a.max_rows) * a.rep, p.rows());
  const dim3 grid2(static_cast<unsigned>(pairs), static_cast<unsigned>(std::min<int64_t>(p.many ? (rows + 15) / 16 : rows, ((p.many ? 2047 : 511) + pairs) / pairs)));
  const dim3 merge(grid2.x * grid2.y <= 256 ? MERGE_THREADS : 256);
  const bool mx = pages->kind == RF_PAGES_MX4;
#define RF_FEW(D, MT)                                                                                    \
  do {                                                                                                   \
    if (mx) hipLaunchKernelGGL((k_paged_few<D, true, MT>), grid, dim3(64 * NW), 0, stream, a);           \
    else hipLaunchKernelGGL((k_paged_few<D, false, MT>), grid, dim3(64 * NW), 0, stream, a);             \
  } while (0)
#define RF_ATTEND(D)                                                                                     \
  do {                                                                                                   \
    if (p.many && mx) hipLaunchKernelGGL((k_paged_many<D, true>), grid, dim3(Cfg<D>::NTHR), 0, stream, a); \
    else if (p.many) hipLaunchKernelGGL((k_paged_many<D, false>), grid, dim3(Cfg<D>::NTHR), 0, stream, a); \
    else if (p.mt == 1) RF_FEW(D, 1);                                                                    \
    else if (p.mt == 2) RF_FEW(D, 2);                                                                    \
    else if (p.mt == 3) RF_FEW(D, 3);                                                                    \
    else if constexpr (D != 256) RF_FEW(D, 4);                                                           \
    if (p.fit) {                                                                                         \
      if (int rc = check_launch(fn)) return rc;                                                          \
      hipLaunchKernelGGL(k_paged_merge<D>, grid2, merge, 0, stream, a, p.rows());                        \
    }                                                                                                    \
  } while (0)
  if (d == 64) RF_ATTEND(64);
  else if (d == 128) RF_ATTEND(128);
  else RF_ATTEND(256);
#undef RF_ATTEND
#undef RF_FEW
  return check_launch(fn);
}
