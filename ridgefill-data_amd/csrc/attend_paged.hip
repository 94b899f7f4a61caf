// Attention of new tokens of many sequences over a paged K / V cache (bf16 or 4-bit codes), gfx950.
//
// k_paged_few: a few query rows a sequence (one token of each, or some drafted ones). The keys are read once from HBM and
// that read is the bound: a block takes one K / V head and 16 query rows (queries x the query heads of the K / V head, query
// by query) of one sequence, its four waves take turns at the key tiles (32 keys) of the block's run, with no barrier until
// they join. bf16 tiles go straight from memory into the registers of the products; 4-bit ones, a quarter of the bytes a
// product, through a ring in LDS a wave, which keeps enough of them in flight. Per tile and wave:
//   S^T = K Q^T. A's row m of key half kb is key 8 (m / 4) + 4 kb + m % 4 of the tile, so that lane (n, g) (n = lane % 16,
//       g = lane / 16) holds, for query row n, the scores of keys 8 g .. 8 g + 7: the order in which A of the second product
//       wants them. bf16: v_mfma_f32_16x16x32_bf16, the contraction's order over d as memory gives it (16-byte chunk 4 s + g
//       in step s). 4 bits: v_mfma_scale_f32_16x16x128_f8f6f4, which takes codes and scales as they are; the queries as two
//       E4M3 terms (split_queries).
//   Softmax in fp32 base 2, the running maximum raised only when a score exceeds it by 2^8 (lazily: O is rescaled rarely).
//   O += P V on v_mfma_f32_16x16x32_bf16: B's column n of product nb is d = n (D / 16) + nb, so a lane reads D / 16 consecutive
//       values of each of its 8 keys and transposes 2 x 2 with v_perm (half an instruction a value); O's columns of a lane are
//       consecutive in memory again. 4-bit values become bf16 by v_cvt_scalef32_pk_bf16_fp4, scale included, exactly. (P in
//       8 bits or less would round the probabilities by 2^-4 and more; they keep bf16's 2^-8.)
// The waves' parts are merged through LDS in wave order. Measured, merge included: 32 sequences of 500 to 8111 keys, 8 heads of
// 128, bf16, 79 us for the 377 MB they hold (4.8 TB/s); 48 of 1500 to 24001 in 4 bits 91 us for 405 MB; one of 122880 keys in 4
// bits, 2 heads of 256, 30 us for 67 MB: of that 9 are the merge and 10 the launch, the first tiles' way and the end.
// The bf16 kernels' addresses take more scalar registers than there are: 115, 210 and 406 of them at head_dim 64, 128 and 256 lie
// in lanes of vector registers (4 bits: 45 to 51); no vector register spills.
#include <stdint.h>

#include <algorithm>

#include "attend_tile.h"
#include "paged.h"

namespace rf {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

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
  int n_seq, hq, hkv, rep, rpb;            // rpb: query rows a block
  int max_rows, max_keys;
  float c;                                 // scale log2(e)
  uint16_t* out;
  int64_t ldo;
  float* part;                             // partials of the splits
  int* length;                             // behind them: the split length, from the splits' launch to the merge
  int fit;                                 // blocks a head that one round holds (0: no splits)
  bool once;                               // k_paged_many: as many units as that at most
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

// Query rows are a sequence's (query, head of the K / V head)s, query by query; row blocks take rpb of them.
__device__ __forceinline__ int row_blocks(const PagedArgs& a, const Seq& s) { return (s.rows * a.rep + a.rpb - 1) / a.rpb; }

struct RowBlock {
  int q0, off, rows;                       // query and head of its first row, its rows
  __device__ RowBlock(const PagedArgs& a, const Seq& s, int rb) {
    const int r0 = rb * a.rpb;
    q0 = r0 / a.rep;
    off = r0 - q0 * a.rep;
    rows = min(a.rpb, s.rows * a.rep - r0);
  }
};

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

// k_paged_many: the key tiles of a split. Where the row blocks leave a quarter of the GPU idle (once), splits are as short as
// one round of blocks allows (fit: its units a head): a few more than fill it wait for a second round. Otherwise the length of
// the least estimated time: all tiles and what each unit costs besides over the round's blocks, and a third of a split for the
// end (or one round's longest split): 1499-row chunks of three prompts 521 us at three rounds, 599 at 1.6; a unit's cost as 6,
// 10 or 16 tiles instead of 3 changed nothing that stood out. Without the end's third three chunks of 1499 rows in 4 bits took
// 905 us for 802 and three of 700 in bf16 250 for 240, but five of 500 over 5000 keys 154 for 187; with a whole split all as
// with a third. Up to 64 sequences the lanes try 64 lengths each; more of them take a length that surely fits. Every block does
// the same arithmetic on the same sizes: no launch has to plan before this one, and a captured graph follows its lens.
constexpr float UNIT_TILES = 3.f;
__device__ int split_length(const PagedArgs& a, float work, float blocks, int tmax, int nrb0, int tiles0, int lane) {
  const float fit = static_cast<float>(a.fit);
  const bool once = a.once;
  if (a.n_seq > 64) {
    const float W = once ? work / fmaxf(fit - blocks, 1.f) : work / (2.f * fit);
    return max(a.wmin, static_cast<int>(ceilf(W)));
  }
  const float lo = fmaxf(static_cast<float>(a.wmin), ceilf(work / (once ? fit : 3.f * fit)));
  const float hi = fmaxf(static_cast<float>(tmax), lo);
  const float step = __builtin_amdgcn_exp2f(__builtin_amdgcn_logf(hi / lo) * (static_cast<float>(lane) / 63.f));
  const float W = lane == 63 ? hi : ceilf(lo * step);        // (hi itself: past 4 million tiles the rounded power may fall short of it)
  const float inv = 1.f / W;
  float units = 0.f;
  for (int b = 0; b < a.n_seq; ++b)
    units += static_cast<float>(__builtin_amdgcn_readlane(nrb0, b)) *
             ceilf(static_cast<float>(__builtin_amdgcn_readlane(tiles0, b)) * inv);
  const float longest = fminf(W, static_cast<float>(tmax));
  float cost = units <= fit ? fmaxf(longest, work / fit) : (work + UNIT_TILES * units) / fit + 0.35f * longest;
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
      const float r = static_cast<float>(row_blocks(a, s));
      work += wave_sum(r * static_cast<float>(tiles_of(s.keys, a.kt)));
      blocks += wave_sum(r);
      tmax = max(tmax, wave_max(s.rows ? tiles_of(s.keys, a.kt) : 1));
    }
    W = split_length(a, work, blocks, tmax, row_blocks(a, s0), tiles_of(s0.keys, a.kt), lane);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.length = W;
  }
  Unit u;
  u.b = -1;
  int before = 0, parts = 0;
  for (int b0 = 0; b0 < a.n_seq; b0 += 64) {
    const Seq s = b0 == 0 ? s0 : b0 + lane < a.n_seq ? seq_of(a, b0 + lane) : Seq{0, 0, 0};
    const int nrb = row_blocks(a, s), ns = nrb ? (tiles_of(s.keys, a.kt) + W - 1) / W : 0;
    const int n = merging ? nrb : nrb * ns;
    int total, ptotal;
    const int pre = wave_sum_below(n, total);
    const int ppre = merging ? wave_sum_below(nrb * ns, ptotal) : pre;
    if (!merging) ptotal = total;
    if (want < before + total) {
      // (scalar from here on: what follows from a unit is uniform over its block)
      const uint64_t hit = __ballot(n > 0 && before + pre <= want && want < before + pre + n);
      if (!hit) return u;                 // (sums past 31 bits: only with a cu that does not rise)
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

// k_paged_few's shares: the key tiles of all (sequence, row block)s in a row, cut into equal runs, one a block of a round
// (a run may end inside a row block and begin the next one's: its parts are then two pieces or more). 48 sequences of 1500
// to 24000 keys in 4 bits, in 96 splits of one length at most: a quarter of the blocks idle, 107 us where equal runs took 97.
struct Piece {
  int b, rb, t0, nt;                       // sequence (-1: none), row block, tile that the position falls on, its tiles
  int begin;                               // position of its first tile
  Seq s;
};

// The piece at position `want` of the tiles in a row; by_block: the want-th (sequence, row block), from its first tile.
__device__ __forceinline__ Piece piece_at(const PagedArgs& a, const Seq& s0, int want, bool by_block, int lane) {
  Piece pc;
  pc.b = -1;
  int before = 0, tiles_before = 0;
  for (int b0 = 0; b0 < a.n_seq; b0 += 64) {
    const Seq s = b0 == 0 ? s0 : b0 + lane < a.n_seq ? seq_of(a, b0 + lane) : Seq{0, 0, 0};
    const int nrb = row_blocks(a, s), nt = tiles_of(s.keys, a.kt);
    int total, tiles;
    const int tpre = wave_sum_below(nrb * nt, tiles), pre = by_block ? wave_sum_below(nrb, total) : tpre, n = by_block ? nrb : nrb * nt;
    if (!by_block) total = tiles;
    if (want < before + total) {
      const uint64_t hit = __ballot(n > 0 && before + pre <= want && want < before + pre + n);
      if (!hit) return pc;                 // (sums past 31 bits: only with a cu that does not rise)
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(hit)) - 1);
      const int off = want - before - __builtin_amdgcn_readlane(pre, l);
      pc.b = b0 + l;
      pc.nt = __builtin_amdgcn_readlane(nt, l);
      pc.rb = by_block ? off : off / pc.nt;
      pc.t0 = by_block ? 0 : off - pc.rb * pc.nt;
      pc.begin = tiles_before + __builtin_amdgcn_readlane(tpre, l) + pc.rb * pc.nt;
      pc.s = Seq{__builtin_amdgcn_readlane(s.rows, l), __builtin_amdgcn_readlane(s.keys, l), __builtin_amdgcn_readlane(s.first, l)};
      return pc;
    }
    before += total;
    tiles_before += tiles;
  }
  return pc;
}

// The length of a run: every block's own sum of the tiles.
__device__ __forceinline__ int run_length(const PagedArgs& a, const Seq& s0, int lane, int& total) {
  total = 0;
  for (int b0 = 0; b0 < a.n_seq; b0 += 64) {
    const Seq s = b0 == 0 ? s0 : b0 + lane < a.n_seq ? seq_of(a, b0 + lane) : Seq{0, 0, 0};
    int n;
    wave_sum_below(row_blocks(a, s) * tiles_of(s.keys, a.kt), n);
    total += n;
  }
  return max(a.wmin, (total + a.fit - 1) / a.fit);
}

// Key half kb's registers of a tile: the lane's share of d of its key.
template <int D, bool MX>
struct KTile {
  static constexpr int NS = D / 32;                          // 32-deep steps over d
  uint4 x[MX ? 1 : 2][MX ? 1 : NS];                          // bf16
  uint32_t c[MX ? 2 : 1][MX ? (D == 256 ? 8 : 4) : 1];       // codes: of 32 values from d = 128 s + 32 g on, 4 dwords each
  uint2 sc[MX ? (D == 256 ? 2 : 1) : 1];                     // scales of the 8 keys that the lane's two keys are among
};

template <int D, bool MX>
struct VTile {
  static constexpr int VL = D / 16;                          // consecutive values a lane takes of a key
  uint32_t x[MX ? 1 : 8][MX ? 1 : VL / 2];                   // bf16 pairs of 8 keys
  uint32_t c[MX ? 8 * VL / 8 : 1];                           // codes of 8 keys, key by key
  uint2 sc;
};

// bf16: a tile's registers from memory. tok0: the page's token of the 16-key half of the tile that key row m (load_k), or
// lane group g's 8 keys (load_v), lie in.
template <int D>
__device__ __forceinline__ void load_k(KTile<D, false>& kt, const PagesDev& pg, int64_t id, int head, int tok0, int m, int g) {
  const int key = 8 * ((m >> 2) & 1) + (m & 3);              // of that half, for kb = 0
  const char* base = pg.k + id * pg.page_stride + static_cast<int64_t>(head) * pg.head_bytes;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const char* row = base + (tok0 + key + 4 * kb) * (D * 2) + g * 16;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) kt.x[kb][s] = *reinterpret_cast<const uint4*>(row + s * 64);
  }
}

template <int D>
__device__ __forceinline__ void load_v(VTile<D, false>& vt, const PagesDev& pg, int64_t id, int head, int tok0, int n, int g) {
  constexpr int VL = D / 16;
  const char* base = pg.v + id * pg.page_stride + static_cast<int64_t>(head) * pg.head_bytes;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const char* row = base + (tok0 + 8 * (g & 1) + e) * (D * 2) + n * (VL * 2);
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
}

// 4 bits: a wave's ring of tiles in LDS, as they lie in memory, keys and values apart: 32 keys' codes (16 D bytes) and their
// scales (D; 256 bytes at least, as their load writes). Two turns of T tiles: while one is computed the other is on its way,
// and each half is loaded again as soon as it has been read. (head_dim 256: with two tiles a turn the LDS holds four waves, one
// a SIMD; with one tile two a SIMD: 9 sequences of 5 new tokens and up to 30011 keys 49 -> 43 us, 1024 rows of 8007 keys 285 ->
// 232. There the vector pipe is 51 % busy, the matrix pipe 21 %, and a third of the waves' time is waits: two waves a SIMD, all
// that the LDS and the registers hold, do not cover more. An order of the 16-byte chunks that spreads every read over all banks
// changed nothing.)
template <int D>
struct Ring {
  static constexpr int T = D == 256 ? 1 : 2, R = 2 * T;      // tiles a turn, tiles
  static constexpr int HALF = 16 * D + (D < 256 ? 256 : D), SLOT = 2 * HALF;
  static constexpr int L = (D == 64 ? 1 : D / 64) + 1;       // load instructions a half
  static constexpr int BYTES = R * SLOT + 256;               // and the coming window's table entries
};

template <int D>
__device__ __forceinline__ void read_k(KTile<D, true>& kt, const char* slot, int n, int g) {
  const int gd = D == 64 ? g & 1 : g;                        // (head_dim 64: lanes of d past 64 repeat; their queries are zero)
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int s = 0; s < (D == 256 ? 2 : 1); ++s) {
      const uint4 w = *reinterpret_cast<const uint4*>(slot + (8 * (n >> 2) + 4 * kb + (n & 3)) * (D / 2) + s * 64 + gd * 16);
      kt.c[kb][4 * s] = w.x;
      kt.c[kb][4 * s + 1] = w.y;
      kt.c[kb][4 * s + 2] = w.z;
      kt.c[kb][4 * s + 3] = w.w;
    }
#pragma unroll
  for (int s = 0; s < (D == 256 ? 2 : 1); ++s)
    kt.sc[s] = *reinterpret_cast<const uint2*>(slot + 16 * D + (n >> 2) * (D / 4) + (4 * s + gd) * 8);
}

template <int D>
__device__ __forceinline__ void read_v(VTile<D, true>& vt, const char* slot, int n, int g) {
  constexpr int VL = D / 16;
  slot += Ring<D>::HALF;
#pragma unroll
  for (int i = 0; i < VL / 4; ++i) {
    const uint4 w = *reinterpret_cast<const uint4*>(slot + g * (4 * D) + n * (VL * 4) + 16 * i);       // 8 keys x VL / 2 bytes
    vt.c[4 * i] = w.x;
    vt.c[4 * i + 1] = w.y;
    vt.c[4 * i + 2] = w.z;
    vt.c[4 * i + 3] = w.w;
  }
  vt.sc = *reinterpret_cast<const uint2*>(slot + 16 * D + g * (D / 4) + (n * VL / 32) * 8);
}

// Loads from memory into LDS (64 lanes side by side from lds on), without destination registers: the kernel's own waits
// order them. (As builtins the compiler makes every LDS read wait for all of them.)
__device__ __forceinline__ void to_lds16(uint32_t lds, const char* base, uint32_t off) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const uint64_t s = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b >> 32)))) << 32 |
                     static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds)),
               "v"(off), "s"(s) : "memory", "m0");
}
__device__ __forceinline__ void to_lds16(uint32_t lds, const char* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)),
               "v"(at) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(uint32_t lds, const void* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)),
               "v"(at) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A tile's keys or values into the half slot at lds: its 16-key halves' codes lie o0, o1 bytes into the pool (keys' rows and
// values' runs alike), their scales s0, s1.
template <int D>
__device__ __forceinline__ void issue_half(uint32_t lds, const char* codes, const uint8_t* scales, int64_t o0, int64_t o1, int64_t s0,
                                           int64_t s1, int lane) {
  if constexpr (D == 64) {                                   // 512 bytes a 16-key half: lanes 0 .. 31 and 32 .. 63
    to_lds16(lds, codes + (lane < 32 ? o0 : o1) + (lane & 31) * 16);
  } else {
    constexpr int I = D / 128;                               // 1 KB instructions a 16-key half
#pragma unroll
    for (int x = 0; x < 2 * I; ++x) to_lds16(lds + 1024 * x, codes + (x < I ? o0 : o1) + 1024 * (x % I), 16 * lane);
  }
  constexpr int H = D / 8;                                   // dwords of a 16-key half's scales; past both they are repeated
  to_lds4(lds + 16 * D, scales + (((lane / H) & 1) ? s1 : s0) + (lane % H) * 4);
}

// A row block's queries as the products' operands. bf16: 32-deep steps. 4 bits: the matrix instruction takes codes and scales
// as they are when the other side has 8 bits, so a query's 32 values are split as q = 2^e (hi + lo / 16) with hi, lo in E4M3
// (4 significant bits each, a bf16 value has 8) and 128 <= max |q| / 2^e < 256: exact for values down to 2^-14 of
// the largest of their 32, and off by less than 2^-22 of that below. An operand holds d 128 s + 16 g .. + 15 and 64 more
// on in its two halves.
template <int D, bool MX>
struct Queries {
  bf16x8 x[MX ? 1 : D / 32];
  i32x8 hi[MX ? (D == 256 ? 2 : 1) : 1], lo[MX ? (D == 256 ? 2 : 1) : 1];
  int eh[MX ? (D == 256 ? 2 : 1) : 1], el[MX ? (D == 256 ? 2 : 1) : 1];       // scale bytes of block 4 s + g
};

__device__ __forceinline__ uint32_t fp8x4(float a, float b, float c, float d) {
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// The values of a lane: 16 of each 128, and 16 more 64 on.
template <int D>
struct RawQueries {
  uint4 x[D / 128 + (D == 64)][D > 64 ? 2 : 1][2];
};

template <int D>
__device__ __forceinline__ void load_queries(RawQueries<D>& q, const uint16_t* row, int g) {
#pragma unroll
  for (int s = 0; s < (D == 256 ? 2 : 1); ++s)
#pragma unroll
    for (int h = 0; h < (D > 64 ? 2 : 1); ++h)
#pragma unroll
      for (int x = 0; x < 2; ++x) q.x[s][h][x] = *reinterpret_cast<const uint4*>(row + 128 * s + 64 * h + 16 * g + 8 * x);
}

// (here, and not behind the loads into LDS that follow, which the compiler does not count)
template <int D>
__device__ __forceinline__ void arrived(RawQueries<D>& q) {
#pragma unroll
  for (int s = 0; s < (D == 256 ? 2 : 1); ++s)
#pragma unroll
    for (int h = 0; h < (D > 64 ? 2 : 1); ++h)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint4& v = q.x[s][h][x];
        asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
      }
}

template <int D>
__device__ __forceinline__ void split_queries(Queries<D, true>& q, const RawQueries<D>& raw, int g, int lane) {
#pragma unroll
  for (int s = 0; s < (D == 256 ? 2 : 1); ++s) {
    int e[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};              // 16 values
      if (D > 64 || h == 0) {
        const uint4 a = raw.x[s][D > 64 ? h : 0][0], b = raw.x[s][D > 64 ? h : 0][1];
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
      }
      int top = 0;
#pragma unroll
      for (int x = 0; x < 8; ++x) top = max(top, max(static_cast<int>(w[x] & 0x7fffu), static_cast<int>((w[x] >> 16) & 0x7fffu)));
      top = max(top, __shfl_xor(top, 16, 64));               // of the block of 32
      const bool odd = top >= 0x7f80;                        // a NaN or an infinity: the block is NaN
      e[h] = min(max(top >> 7, 20), 254) - 7;                // biased; tiny values keep a scale in range
      const float up = __uint_as_float(static_cast<uint32_t>(254 - e[h]) << 23);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float v0 = bf_lo(w[2 * x]) * up, v1 = bf_hi(w[2 * x]) * up, v2 = bf_lo(w[2 * x + 1]) * up, v3 = bf_hi(w[2 * x + 1]) * up;
        const uint32_t hi = fp8x4(v0, v1, v2, v3);
        const auto h01 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), h23 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
        const uint32_t lo = fp8x4((v0 - h01[0]) * 16.f, (v1 - h01[1]) * 16.f, (v2 - h23[0]) * 16.f, (v3 - h23[1]) * 16.f);
        q.hi[s][4 * h + x] = odd ? 0x7f7f7f7f : hi;
        q.lo[s][4 * h + x] = odd ? 0x7f7f7f7f : lo;
      }
    }
    // block 4 s + g's scale: d 32 g .. are the first halves of lanes 2 g, 2 g + 1 for g < 2, else second halves
    const int from = (lane & 15) + 32 * (g & 1), e0 = __shfl(e[0], from, 64), e1 = __shfl(e[1], from, 64);
    q.eh[s] = g < 2 ? e0 : e1;
    q.el[s] = q.eh[s] - 4;
  }
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

// N columns from d0 of row r of a 16-row block that begins at head off of row `first` of q: the output, or a part's partial.
template <int D, int N>
__device__ __forceinline__ void finish_row(const PagedArgs& a, int first, int off, bool whole, int64_t part, int r, int head,
                                           int d0, const float (&acc)[N], float top, float sum) {
  if (!whole) {
    float* p = a.part + part * (16 * (D + 2));
#pragma unroll
    for (int b = 0; b < N; b += 4)
      *reinterpret_cast<float4*>(p + r * D + d0 + b) = make_float4(acc[b], acc[b + 1], acc[b + 2], acc[b + 3]);
    if (d0 == 0) {
      p[16 * D + r] = top;
      p[16 * (D + 1) + r] = sum;
    }
    return;
  }
  const float inv = inverse_sum(sum);
  const int qi = (off + r) / a.rep;
  uint16_t* dst = a.out + static_cast<int64_t>(first + qi) * a.ldo + (head * a.rep + off + r - qi * a.rep) * D + d0;
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

// The wave's running state: O [rows 4 g + j][d = n NB + b], and of row n the reference maximum m (raw
// scores; the same in the four lanes of a row) and the lane's share of the row sum.
template <int D>
struct Rows {
  f32x4 o[D / 16];
  float m, l;
};

__device__ __forceinline__ uint32_t finite_pair(uint32_t p) {  // with zeros for the halves that are NaN or infinite
  p = (p & 0x7f80u) == 0x7f80u ? p & 0xffff0000u : p;
  return (p & 0x7f800000u) == 0x7f800000u ? p & 0xffffu : p;
}

// V's fragments of pair j; CUT, if cut: with zeros for the lane's keys past `last` and for what is not finite.
template <int D, bool MX, bool CUT>
__device__ __forceinline__ void v_frags(const VTile<D, MX>& vt, const float (&vs)[8], int j, int last, bool cut,
                                        bf16x8& f0, bf16x8& f1) {
  uint32_t p[8];
  v_pairs<D, MX>(vt, vs, j, p);
  if (CUT && cut) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = e <= last ? finite_pair(p[e]) : 0u;
  }
  f0 = as_frag(make_uint4(both_low(p[0], p[1]), both_low(p[2], p[3]), both_low(p[4], p[5]), both_low(p[6], p[7])));
  f1 = as_frag(make_uint4(both_high(p[0], p[1]), both_high(p[2], p[3]), both_high(p[4], p[5]), both_high(p[6], p[7])));
}

// What a row meets of V that is not finite, kept apart from the products (there, 0 x infinity would reach rows that do not
// see the key): marks of (row, column), two bits each (1 infinity, 2 -infinity, 3 NaN, also of both).
__device__ __forceinline__ uint32_t mark_of(uint32_t half) {
  return (half & 0x7f80u) != 0x7f80u ? 0u : (half & 0x7fu) ? 3u : (half & 0x8000u) ? 2u : 1u;
}

__device__ __forceinline__ float marked(uint32_t m) { return m == 3u ? NAN : m == 1u ? INFINITY : m == 2u ? -INFINITY : 0.f; }

// S^T of a tile: sc[kb][j] = the raw score of key 8 g + 4 kb + j for query row n.
template <int D, bool MX>
__device__ __forceinline__ void scores(const KTile<D, MX>& kt, const Queries<D, MX> &qf, f32x4 (&sc)[2], int n) {
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    sc[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (MX) {
#pragma unroll
      for (int s = 0; s < (D == 256 ? 2 : 1); ++s) {
        const i32x8 k = {static_cast<int>(kt.c[kb][4 * s]), static_cast<int>(kt.c[kb][4 * s + 1]), static_cast<int>(kt.c[kb][4 * s + 2]),
                         static_cast<int>(kt.c[kb][4 * s + 3]), 0, 0, 0, 0};
        const int e = static_cast<int>((kb ? kt.sc[s].y : kt.sc[s].x) >> (8 * (n & 3)));        // (its low byte counts)
        sc[kb] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, qf.lo[s], sc[kb], 4, 0, 0, e, 0, qf.el[s]);
        sc[kb] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, qf.hi[s], sc[kb], 4, 0, 0, e, 0, qf.eh[s]);
      }
    } else {
#pragma unroll
      for (int s = 0; s < D / 32; ++s)
        sc[kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_frag(kt.x[kb][s]), qf.x[s], sc[kb], 0, 0, 0);
    }
  }
}

__device__ __forceinline__ float lane_max(const f32x4 (&s)[2]) {
  return fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
}

__device__ __forceinline__ float row_max(float v) {          // of a row's four lanes
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}

// Raise the reference maxima to what the rows' four lanes have seen (tmax), and rescale their sums and O.
template <int D>
__device__ __forceinline__ void raise(Rows<D>& st, float tmax, float c, int g) {
  const float top = fmaxf(st.m, row_max(tmax));
  const float alpha = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((st.m - top) * c);
  st.m = top;
  st.l *= alpha;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float al = __shfl(alpha, 4 * g + j, 64);           // O's rows of a lane are 4 g + j
#pragma unroll
    for (int b = 0; b < D / 16; ++b) st.o[b][j] *= al;
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
template <int D, bool MX, bool CUT>
__device__ __forceinline__ void product(const VTile<D, MX>& vt, const bf16x8 &pf, int last, bool cut, Rows<D>& st) {
  float vs[8];
  if constexpr (MX) {
#pragma unroll
    for (int e = 0; e < 8; ++e) vs[e] = byte_scale(vt.sc, e);
  }
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    bf16x8 f0, f1;
    if constexpr (CUT) __builtin_amdgcn_sched_barrier(0);    // (all pairs at once would not fit the registers)
    v_frags<D, MX, CUT>(vt, vs, j, last, cut, f0, f1);
    st.o[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf, f0, st.o[2 * j], 0, 0, 0);
    st.o[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf, f1, st.o[2 * j + 1], 0, 0, 0);
  }
}

// A tile of which some row does not see some key. Keys are hidden from rows by their scores (-infinity). Where the tile's V is not
// all finite, what no row sees of it and what is not finite enters the product as zero, and the latter leaves its marks in the
// rows that see it. slot: the tile in LDS (4 bits). (Zeros in any case: 8 sequences of up to 2000 keys in 4 bits 20 us for 18, 48
// of up to 24001 94 for 91.)
template <int D, bool MX>
__device__ __forceinline__ void edge_step(Tile<D, MX>& tl, const Queries<D, MX> &qf, int pos,
                                          Rows<D>& st, float c, int p0, int plast, const RowBlock& rows, int rep, int lane,
                                          uint32_t* marks, [[maybe_unused]] const char* slot) {
  constexpr int NB = D / 16;
  const int n = lane & 15, g = lane >> 4, k0 = tl.k0;
  f32x4 sc[2];
  scores<D, MX>(tl.k, qf, sc, n);
  const bool hidden = (tl.bad >> (g >> 1)) & 1u;             // the lane's 8 keys lie on a page that is none
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (hidden || k0 + 8 * g + 4 * kb + j > pos) sc[kb][j] = -INFINITY;
  const float tmax = lane_max(sc);
  if (__any(tmax > st.m + headroom(c))) raise<D>(st, tmax, c, g);
  const bf16x8 pf = probabilities(sc, st.m, c, st.l);
  if constexpr (MX) read_v<D>(tl.v, slot, n, g);
  // (4 bits: the scales 253 and 254 take some codes past bf16, 255 makes NaN of all)
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (MX) {
      odd |= (((e < 4 ? tl.v.sc.x : tl.v.sc.y) >> (8 * (e & 3))) & 255u) >= 253u;
    } else {
#pragma unroll
      for (int j = 0; j < NB / 2; ++j) odd |= not_finite(tl.v.x[e][j]);
    }
  }
  const bool cut = __any(odd);                               // (else what is hidden counts for nothing by its probability)
  const int last = hidden ? -1 : plast - k0 - 8 * g;         // of the lane's keys, the last that any row sees
  // marks of key e's columns from `from` on, which lie in one word of a row's, in the rows from the key's own query on
  auto mark = [&](int e, int g, int from, uint32_t m) {
    const int first = max(0, (k0 + 8 * g + e - p0) * rep - rows.off);
    for (int r = first; r < rows.rows; ++r) {
      const int at = r * D + from;
      atomicOr(marks + at / 16, m << (2 * (at % 16)));
    }
    marks[D] = 1u;
  };
  if constexpr (!MX) {
    if (cut) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int j = 0; j < NB / 2; ++j) {
          const uint32_t two = tl.v.x[e][j];
          if (e <= last && not_finite(two)) mark(e, g, n * NB + 2 * j, mark_of(two & 0xffffu) | mark_of(two >> 16) << 2);
        }
      }
    }
  }
  product<D, MX, true>(tl.v, pf, last, cut, st);
  if constexpr (MX) {
    if (cut) {                                               // (a value at a time from LDS: the registers hold no more)
      int here = lane;                                       // (nor what follows from it, kept through the tiles)
      asm volatile("" : "+v"(here));
      const int m = here & 15, h = here >> 4;
      const char* values = slot + Ring<D>::HALF + h * (4 * D) + m * (4 * NB);
      const char* scales = slot + Ring<D>::HALF + 16 * D + h * (D / 4) + (m * NB / 32) * 8;
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        if (e > last) continue;
        const float s = scale_of<0>(*reinterpret_cast<const uint8_t*>(scales + e));
        uint32_t all = 0;
#pragma unroll 1
        for (int j = 0; j < NB / 2; ++j) {
          const uint32_t two = fp4_pair<0>(*reinterpret_cast<const uint8_t*>(values + e * (NB / 2) + j), s);
          all |= (mark_of(two & 0xffffu) | mark_of(two >> 16) << 2) << (4 * j);
        }
        if (all) mark(e, h, m * NB, all);
      }
    }
  }
}

// Blocks a CU that the registers of a kernel hold (4 bits: and its rings the LDS).
constexpr int few_blocks(int d, bool mx) { return d == 256 && !mx ? 1 : 2; }

template <int D, bool MX>
struct FewLds {
  static constexpr int RINGS = MX ? NW * Ring<D>::BYTES : 0;
  static constexpr int MARKS = RINGS > merge_floats<D>() * 4 ? RINGS : merge_floats<D>() * 4;   // (the merge takes the rings' place)
  static constexpr int BYTES = MARKS + 4 * D + 16;
};

template <int D, bool MX>
__global__ __launch_bounds__(64 * NW, (few_blocks(D, MX))) void k_paged_few(PagedArgs a) {
  constexpr int NB = D / 16;
  using F = FewLds<D, MX>;
  __shared__ uint4 lds4[F::BYTES / 16];
  float* lds = reinterpret_cast<float*>(lds4);
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), n = lane & 15, g = lane >> 4;
  // (heads slowest: the blocks of an XCD then read all heads' parts of the pages. With heads fastest and 8 of them each XCD
  // reads one head's, which all lie at the same offset of a page, and in 4 bits, 4 KB of 32, 4 % slower)
  const int blocks = gridDim.x / a.hkv, head = blockIdx.x / blocks, mask = (1 << a.pg.shift) - 1;
  uint32_t* marks = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(lds4) + F::MARKS);
  for (int x = t; x <= D; x += 64 * NW) marks[x] = 0u;
  __syncthreads();
  Seq s0{0, 0, 0};
  if (lane < a.n_seq) s0 = seq_of(a, lane);
  // the block's run of tiles [at, end), or (unsplit) its row block
  const int x0 = blockIdx.x - head * blocks;
  int at = 0, end = 1, run = 0;
  if (a.fit) {
    int total;
    run = run_length(a, s0, lane, total);
    at = x0 * run;
    end = min(total, at + run);
    if (blockIdx.x == 0 && t == 0) *a.length = run;          // for the merge
  }
  for (bool once = true; at < end; once = false) {           // (uniform over the block)
    const Piece u = a.fit ? piece_at(a, s0, at, false, lane) : piece_at(a, s0, x0, true, lane);
    if (u.b < 0) return;
    const int it0 = u.t0, itn = a.fit ? min(u.nt, it0 + end - at) : u.nt;
    const bool whole_block = it0 == 0 && itn == u.nt;
    const int64_t part = static_cast<int64_t>(2 * x0 + (once ? 0 : 1)) * a.hkv + head;    // (only the first and last pieces are parts)
    at += a.fit ? itn - it0 : 1;
    const RowBlock r(a, u.s, u.rb);
    const int p0 = u.s.keys - u.s.rows + r.q0;                 // position of its first query (may lie before 0)
    const int plast = p0 + (r.off + r.rows - 1) / a.rep;       // keys 0 .. plast are read
    const int it1 = min(itn, plast < 0 ? 0 : plast / KT + 1);

    // The wave's tiles are it0 + w + NW i, i < mine. Lane l holds the page of 16-key half l % 2 of tile i0 + l / 2 of a window
    // of 32 tiles (0 for pages that are none, whose keys `bad` then hides), and the next window's entry on its way.
    const int mine = it0 + w < it1 ? (it1 - it0 - w + NW - 1) / NW : 0;
    const int32_t* row = a.table + static_cast<int64_t>(u.b) * a.ld_table;
    auto entry = [&](int i0) {
      const int it = it0 + w + NW * (i0 + (lane >> 1));
      const int at = (it * 2 + (lane & 1)) >> (a.pg.shift - 4);
      return it < it1 && at < a.width ? row[at] : -1;
    };
    int ids = entry(0);
    // queries: row n. Their loads go before the tiles', which wait for the table's entries (behind them, 2 us later a piece)
    Queries<D, MX> qf;
    [[maybe_unused]] RawQueries<D> raw;
    const int qx = r.off + min(n, r.rows - 1), qi = qx / a.rep;            // (rows past the last repeat it, and see nothing)
    const int pos = n < r.rows ? p0 + qi : -1;
    const uint16_t* qrow = a.q + static_cast<int64_t>(u.s.first + r.q0 + qi) * a.ldq + (head * a.rep + qx - qi * a.rep) * D;
    if constexpr (MX) {
      load_queries<D>(raw, qrow, g);
    } else {
#pragma unroll
      for (int s = 0; s < D / 32; ++s) qf.x[s] = as_frag(*reinterpret_cast<const uint4*>(qrow + 32 * s + 8 * g));
    }
    [[maybe_unused]] int coming = MX ? 0 : entry(32);
    uint64_t bad;
    auto settle = [&]() {
      const bool out = ids < 0 || ids >= a.pg.n_pages;
      ids = out ? 0 : ids;
      bad = __ballot(out);
    };
    settle();
    if constexpr (MX) arrived<D>(raw);
    Rows<D> st;
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) st.o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Whole tiles first, then the tiles that some row sees in part; from the first page that is none on all of them are taken as
    // such. A maximum that has to rise leaves the inner loop: with the rescale inside it the compiler moves all of O at every tile.
    // (Not the first of a piece, which 13 sequences at head_dim 256, two tiles a wave, took 2 us longer for.)
    const int whole = p0 >= KT - 1 ? min(mine, ((p0 + 1) / KT - it0 - w + NW - 1) / NW) : 0;
    int i = 0;
    bool none = false, fresh = true;                           // fresh: O is zero, nothing to rescale
    if constexpr (MX) {
      // Tiles come through the wave's ring. (A wave that loaded its next two tiles into registers behind their last use had one
      // product's time for a latency of 2 us: 8500 cycles a turn at head_dim 256 for 3000 of work; one 122880-key sequence
      // took 23 us.)
      using G = Ring<D>;
      constexpr int TT = G::T, LG = G::L * TT;                 // loads of a turn's keys, or values
      char* ring = reinterpret_cast<char*>(lds4) + w * G::BYTES;
      const uint32_t ring_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)ring));
      uint32_t bads = 0;                                       // two bits a slot
      // a lane's entry as byte offsets of its half's codes and scales, once a window
      int64_t code_at = 0, scale_at = 0;
      auto place = [&](int i0) {
        const int tok = ((it0 + w + NW * (i0 + (lane >> 1))) * KT + 16 * (lane & 1)) & mask;
        code_at = ids * a.pg.page_stride + static_cast<int64_t>(head) * a.pg.head_bytes + tok * (D / 2);
        scale_at = ids * a.pg.scale_stride + static_cast<int64_t>(head) * a.pg.head_scales + (tok >> 3) * (D / 4);
      };
      auto lane64 = [](int64_t v, int l) {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), l), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), l);
        return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
      };
      place(0);
      auto fetch_entries = [&](int i0) {                       // table entries of the window that begins at tile i0
        const int at = ((it0 + w + NW * (i0 + (lane >> 1))) * 2 + (lane & 1)) >> (a.pg.shift - 4);
        to_lds4(ring_at + G::R * G::SLOT, row + min(at, a.width - 1));
      };
      // tile x < mine, a turn's keys before its values, turns in order; the slot's reads have returned
      auto issue_k = [&](int x) {
        if ((x & 31) == 0 && x) {
          const int it = it0 + w + NW * (x + (lane >> 1)), at = (it * 2 + (lane & 1)) >> (a.pg.shift - 4);
          ids = reinterpret_cast<const int32_t*>(ring + G::R * G::SLOT)[lane];     // landed turns ago
          wait_lds_reads();
          ids = it < it1 && at < a.width ? ids : -1;
          settle();
          place(x);
          fetch_entries(x + 32);
        }
        const int y = 2 * (x & 31), s = x % G::R;
        bads = (bads & ~(3u << (2 * s))) | (static_cast<uint32_t>(bad >> y) & 3u) << (2 * s);
        issue_half<D>(ring_at + s * G::SLOT, a.pg.k, a.pg.ks, lane64(code_at, y), lane64(code_at, y + 1), lane64(scale_at, y),
                      lane64(scale_at, y + 1), lane);
      };
      auto issue_v = [&](int x) {
        const int y = 2 * (x & 31), s = x % G::R;
        issue_half<D>(ring_at + s * G::SLOT + G::HALF, a.pg.v, a.pg.vs, lane64(code_at, y), lane64(code_at, y + 1),
                      lane64(scale_at, y), lane64(scale_at, y + 1), lane);
      };
      auto issue_turn = [&](auto&& issue, int x) {
#pragma unroll
        for (int y = 0; y < TT; ++y)
          if (x + y < mine) issue(x + y);
      };
      if (mine) {
        fetch_entries(32);
        for (int x = 0; x < G::R; x += TT) {
          issue_turn(issue_k, x);
          issue_turn(issue_v, x);
        }
      }
      split_queries<D>(qf, raw, g, lane);
      while (!none && i + TT <= whole) {
        f32x4 sc[TT][2];
        float tmax;
        for (; i + TT <= whole; i += TT) {
          none = ((bads >> (2 * (i % G::R))) & ((1u << (2 * TT)) - 1u)) != 0;       // (a turn's slots lie side by side)
          if (none) break;
          // its keys have landed when no more than the loads after them are on their way: its values, the next turn
          if (i + 2 * TT <= mine) wait_loads<3 * LG>();
          else wait_loads<LG>();
          const char* slot = ring + (i % G::R) * G::SLOT;
          tmax = -INFINITY;
#pragma unroll
          for (int x = 0; x < TT; ++x) {
            KTile<D, true> kt;
            read_k<D>(kt, slot + x * G::SLOT, n, g);
            scores<D, true>(kt, qf, sc[x], n);
            tmax = fmaxf(tmax, lane_max(sc[x]));
          }
          if (__any(tmax > st.m + headroom(a.c))) {
            if (!fresh) break;
            fresh = false;
            st.m = row_max(tmax);
          }
          wait_lds_reads();
          issue_turn(issue_k, i + G::R);
          bf16x8 pf[TT];
#pragma unroll
          for (int x = 0; x < TT; ++x) pf[x] = probabilities(sc[x], st.m, a.c, st.l);
          // its values: the next turn, and the keys of the one after it
          if (i + 3 * TT <= mine) wait_loads<3 * LG>();
          else if (i + 2 * TT <= mine) wait_loads<2 * LG>();
          else wait_loads<0>();
          VTile<D, true> vt[TT];
#pragma unroll
          for (int x = 0; x < TT; ++x) read_v<D>(vt[x], slot + x * G::SLOT, n, g);
          wait_lds_reads();
          issue_turn(issue_v, i + G::R);
#pragma unroll
          for (int x = 0; x < TT; ++x) product<D, true, false>(vt[x], pf[x], 8, false, st);
        }
        if (!none && i + TT <= whole) raise<D>(st, tmax, a.c, g);
      }
      for (; i < mine; ++i) {                                  // (few: every load is waited for)
        wait_loads<0>();
        const char* slot = ring + (i % G::R) * G::SLOT;
        Tile<D, true> tl;
        read_k<D>(tl.k, slot, n, g);
        tl.k0 = (it0 + w + NW * i) * KT;
        tl.bad = (bads >> (2 * (i % G::R))) & 3u;
        edge_step<D, true>(tl, qf, pos, st, a.c, p0, plast, r, a.rep, lane, marks, slot);
        wait_lds_reads();
        if (i + G::R < mine) {
          issue_k(i + G::R);
          issue_v(i + G::R);
        }
      }
      wait_loads<0>();                                         // nothing in flight into the rings:
      __syncthreads();                                         // the merge takes their place
    } else {
      // A tile takes D / 2 registers: one (two at head_dim 64), the keys' reloaded behind the scores and the values' behind the
      // product. Tiles past the last are loaded as the last one again: no load of the loop is conditional.
      constexpr int NT = D == 64 ? 2 : 1;
      auto window = [&](int x) {                               // before the loads of tile x
        if ((x & 31) == 0) {
          ids = coming;
          settle();
          coming = entry(x + 32);
        }
      };
      auto get_k = [&](Tile<D, false>& tl, int x) {            // x < mine; windows in order
        const int y = 2 * (x & 31), id0 = __builtin_amdgcn_readlane(ids, y), id1 = __builtin_amdgcn_readlane(ids, y + 1);
        const int k0 = (it0 + w + NW * x) * KT;
        load_k<D>(tl.k, a.pg, n >= 8 ? id1 : id0, head, (k0 + (n >= 8 ? 16 : 0)) & mask, n, g);
      };
      auto get_v = [&](Tile<D, false>& tl, int x) {
        const int y = 2 * (x & 31), id0 = __builtin_amdgcn_readlane(ids, y), id1 = __builtin_amdgcn_readlane(ids, y + 1);
        tl.k0 = (it0 + w + NW * x) * KT;
        tl.bad = static_cast<uint32_t>(bad >> y) & 3u;
        load_v<D>(tl.v, a.pg, g >= 2 ? id1 : id0, head, (tl.k0 + (g >= 2 ? 16 : 0)) & mask, n, g);
      };
      Tile<D, false> tl[NT];
      if (mine) {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          get_k(tl[x], min(x, mine - 1));
          get_v(tl[x], min(x, mine - 1));
        }
      }
      while (!none && i + NT <= whole) {
        f32x4 sc[NT][2];
        float tmax;
        for (; i + NT <= whole; i += NT) {
          uint32_t bads = 0;
#pragma unroll
          for (int x = 0; x < NT; ++x) bads |= tl[x].bad;
          none = bads != 0;
          if (none) break;
#pragma unroll
          for (int x = 0; x < NT; ++x) scores<D, false>(tl[x].k, qf, sc[x], n);
          tmax = lane_max(sc[0]);
          if constexpr (NT > 1) tmax = fmaxf(tmax, lane_max(sc[NT - 1]));
          if (__any(tmax > st.m + headroom(a.c))) {
            if (!fresh) break;
            fresh = false;
            st.m = row_max(tmax);
          }
          const int i1 = min(i + NT, mine - 1);
          if (i1 == i + NT) window(i1);
#pragma unroll
          for (int x = 0; x < NT; ++x) get_k(tl[x], min(i1 + x, mine - 1));
          bf16x8 pf[NT];
#pragma unroll
          for (int x = 0; x < NT; ++x) pf[x] = probabilities(sc[x], st.m, a.c, st.l);
#pragma unroll
          for (int x = 0; x < NT; ++x) product<D, false, false>(tl[x].v, pf[x], 8, false, st);
#pragma unroll
          for (int x = 0; x < NT; ++x) get_v(tl[x], min(i1 + x, mine - 1));
        }
        if (!none && i + NT <= whole) raise<D>(st, tmax, a.c, g);
      }
      for (; i < mine; ++i) {
        edge_step<D, false>(tl[0], qf, pos, st, a.c, p0, plast, r, a.rep, lane, marks, nullptr);
        if constexpr (NT > 1) {                                // the next one is here, the one after it on its way
          tl[0] = tl[1];
          if (i + 2 < mine) {
            window(i + 2);
            get_k(tl[1], i + 2);
            get_v(tl[1], i + 2);
          }
        } else if (i + 1 < mine) {
          window(i + 1);
          get_k(tl[0], i + 1);
          get_v(tl[0], i + 1);
        }
      }
    }

    // merge the waves: thread t takes row t / 16 and D / 16 columns
    float* ml = lds + NW * 16 * (D + 4);
    float ls = st.l;
    ls += __shfl_xor(ls, 16, 64);
    ls += __shfl_xor(ls, 32, 64);
    if (g == 0) {
      ml[w * 16 + n] = st.m == -INFINITY ? st.m : st.m * a.c;  // base 2
      ml[(NW + w) * 16 + n] = ls;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int b = 0; b < NB; b += 4)
        *reinterpret_cast<float4*>(lds + (w * 16 + 4 * g + j) * (D + 4) + n * NB + b) =
            make_float4(st.o[b][j], st.o[b + 1][j], st.o[b + 2][j], st.o[b + 3][j]);
    __syncthreads();
    const int rw = t >> 4, d0 = (t & 15) * NB;
    const bool odd = marks[D] != 0;                            // (read between barriers: a wave ahead may mark the next piece)
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
    if (odd) {
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] += marked((marks[(rw * D + d0 + b) / 16] >> (2 * ((d0 + b) % 16))) & 3u);
    }
    if (rw < r.rows) finish_row<D, NB>(a, u.s.first + r.q0, r.off, whole_block, part, rw, head, d0, acc, top, sum);
    __syncthreads();                                           // the next piece takes the LDS
    if (odd) {
      for (int x = t; x <= D; x += 64 * NW) marks[x] = 0u;
      __syncthreads();
    }
  }
}

// k_paged_many: many query rows a sequence (a chunk of a prompt). A block takes 256 query rows (queries x the query heads of
// a K / V head) of one sequence, 32 a wave, and the key tiles of its split through LDS, each read by all eight waves:
// attend_causal.hip's tile (S^T = K Q^T, P^T straight from the score registers, V^T by transpose reads), with rows of any
// query and head side by side in a wave, so that any group size fills it. Tiles come from pages: bf16 by direct loads, three
// tiles in flight, the page of each load's rows (never more than 16) read off a lane; 4 bits through registers, a tile's
// codes loaded while the one before it is converted into LDS, once for all eight waves (160 of a tile's 2000 cycles).
// Bound by the products and the softmax beside them (64 keys: 1024 cycles of MFMA a wave, two waves a SIMD): 2048 rows of 32768
// keys, 8 heads of 128 in groups of 4, bf16, 960 to 1040 us (1.0 to 1.1 PFLOP/s), the same heads in 4 bits, 3 x 1499 rows of up
// to 12011 keys, 510 to 540 us with the merge's 29 (0.9 PFLOP/s). head_dim 256, 1024 rows of 8007 keys: 520 us, LDS reads as long
// as the products and one wave a SIMD.
template <int AD, bool MX>
struct ManyCodes {
  uint2 k, v;                              // codes of 16 values (8 at head_dim 64)
  uint32_t ks, vs;                         // their scale bytes
};

// The wave's 16-key half of a tile that it loads: rows of one page.
__device__ __forceinline__ int half_of_wave(int w) { return w >> 1; }

// A thread's codes of a tile whose half lies at token tok0 of page id.
template <int AD>
__device__ __forceinline__ void load_codes(ManyCodes<AD, true>& c, const PagesDev& pg, int id, int head, int tok0, int w, int lane) {
  const int64_t at = static_cast<int64_t>(id) * pg.page_stride + static_cast<int64_t>(head) * pg.head_bytes;
  const int64_t sat = static_cast<int64_t>(id) * pg.scale_stride + static_cast<int64_t>(head) * pg.head_scales;
  const int row = 8 * (w & 1) + lane / 8, part = lane % 8;   // eight threads a key row
  const char* kp = pg.k + at + (tok0 + row) * (AD / 2) + part * (AD / 16);
  if constexpr (AD == 64) c.k.x = *reinterpret_cast<const uint32_t*>(kp);
  else c.k = *reinterpret_cast<const uint2*>(kp);
  c.ks = pg.ks[sat + ((tok0 + row) >> 3) * (AD / 4) + (part * (AD / 8) / 32) * 8 + (row & 7)];
  // values: 8 tokens' runs; d 128: two tokens of a run of 8 values, 64: one of two runs of 4
  const char* vp = pg.v + at + ((tok0 >> 3) + (w & 1)) * (4 * AD);
  const uint8_t* sp = pg.vs + sat + ((tok0 >> 3) + (w & 1)) * (AD / 4);
  if constexpr (AD == 128) {
    c.v = *reinterpret_cast<const uint2*>(vp + lane * 8);
    c.vs = *reinterpret_cast<const uint16_t*>(sp + ((lane >> 2) / 4) * 8 + 2 * (lane & 3));
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
  const int row = 8 * w + lane / 8, part = lane % 8;
  uint4* s4 = reinterpret_cast<uint4*>(st);
  const float ks = scale_of<0>(c.ks), vs = scale_of<0>(c.vs);
  if constexpr (AD == 64) {
    s4[L::kslot(row, part)] = eight_values(c.k.x, ks);
    s4[L::vslot(8 * w + (lane & 7), lane >> 3)] = eight_values(c.v.x, vs);
  } else {
    s4[L::kslot(row, 2 * part)] = eight_values(c.k.x, ks);
    s4[L::kslot(row, 2 * part + 1)] = eight_values(c.k.y, ks);
    const int r = 8 * w + 2 * (lane & 3);
    s4[L::vslot(r, lane >> 2)] = eight_values(c.v.x, vs);
    s4[L::vslot(r + 1, lane >> 2)] = eight_values(c.v.y, scale_of<1>(c.vs));
  }
}

// The largest of a row's scores of a tile.
template <int AD>
__device__ __forceinline__ float top_score(const f32x16 (&sc)[Cfg<AD>::KB]) {
  float tmax = -INFINITY, lo, hi;
#pragma unroll
  for (int kb = 0; kb < Cfg<AD>::KB; ++kb)
#pragma unroll
    for (int j = 0; j < 16; ++j) tmax = fmaxf(tmax, sc[kb][j]);
  lane_pair(tmax, lo, hi);
  return fmaxf(lo, hi);
}

template <int AD>
__device__ __forceinline__ void raise_tile(f32x16 (&o)[AD / 32], float& mref, float& lsum, float tmax, float c) {
  const float top = fmaxf(mref, tmax);
  const float alpha = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mref - top) * c);
  mref = top;
#pragma unroll
  for (int b = 0; b < AD / 32; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] *= alpha;
  lsum *= alpha;
}

// The probabilities of a tile, in pairs as the product takes them; their sum goes to lsum.
template <int AD>
__device__ __forceinline__ void tile_probabilities(const f32x16 (&sc)[Cfg<AD>::KB], uint32_t (&pk)[8 * Cfg<AD>::KB], float mref,
                                                   float& lsum, float c) {
  const float mc = mref == -INFINITY ? 0.f : mref * c;
  float psum = 0.f;
#pragma unroll
  for (int e = 0; e < 8 * Cfg<AD>::KB; ++e) {
    const float q0 = __builtin_amdgcn_exp2f(fmaf(sc[e / 8][2 * (e % 8)], c, -mc));
    const float q1 = __builtin_amdgcn_exp2f(fmaf(sc[e / 8][2 * (e % 8) + 1], c, -mc));
    psum += q0 + q1;
    pk[e] = bf16_pair(q0, q1);
  }
  lsum += psum;
}

// tile_step for a tile of which some row does not see some key, without the next tile's scores: bad has a bit a 16-key half
// on a page that is none. Of V, what is not finite enters the product as zero; a row that sees such a value takes it
// from LDS afterwards (0 x infinity must not reach the rows that do not).
template <int AD>
__device__ __forceinline__ void edge_tile(const char* __restrict__ st, f32x16 (&sc)[Cfg<AD>::KB], f32x16 (&o)[AD / 32],
                                          float& mref, float& lsum, int k0, uint32_t bad, int mypos, int hh, float c,
                                          const FragOffsets<AD>& fo) {
  using L = Layout<AD>;
  constexpr int NB = AD / 32, KB = Cfg<AD>::KB, KTL = Cfg<AD>::KT;
  const int rel = min(max(mypos - k0, -1), KTL) - 4 * hh;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const bool gone = (bad >> (2 * kb + (j >> 3))) & 1u;   // keys 32 kb + 8 (j / 4) + ..
      if (gone || 32 * kb + 8 * (j >> 2) + (j & 3) > rel) sc[kb][j] = -INFINITY;
    }
  const float tmax = top_score<AD>(sc);
  if (__any(tmax > mref + headroom(c))) raise_tile<AD>(o, mref, lsum, tmax, c);
  uint32_t pk[8 * KB];
  tile_probabilities<AD>(sc, pk, mref, lsum, c);
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

// Its waves (32 rows each): 8, two a SIMD. head_dim 256: 4, with the 512 registers that O^T (128), the queries (64), two tiles'
// scores and the edge tiles' code want, and 59 more that spill (236 bytes a lane of scratch; 8 waves of 256 spilled 360 registers,
// and 13 sequences of 256 rows took 350 us instead of 157).
constexpr int many_waves(int d) { return d == 256 ? 4 : 8; }
constexpr int many_rows(int d) { return 32 * many_waves(d); }

template <int AD, bool MX>
__global__ __launch_bounds__(64 * many_waves(AD), 1) void k_paged_many(PagedArgs a) {
  using L = Layout<AD>;
  constexpr int NS = AD / 16, NB = AD / 32, KTL = Cfg<AD>::KT, QROWS = many_rows(AD), KB = Cfg<AD>::KB;
  constexpr int NWM = many_waves(AD), SHARES = Cfg<AD>::NW / NWM;      // shares of a tile's loads a wave takes
  constexpr int KLOADS = L::KLOADS * SHARES, LOADS = L::LOADS * SHARES;
  constexpr int HPT = KTL / 16, WIN = 64 / HPT;              // 16-key halves a tile, tiles a window of table entries
  __shared__ uint4 lds[NSTAGE * L::STAGE_U4];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), n = lane & 31, hh = lane >> 5;
  // heads fastest within a unit's row blocks: a head's row blocks of one split lie hkv blocks apart
  const int head = blockIdx.x % a.hkv;
  const Unit u = find_unit(a, blockIdx.x / a.hkv, false);
  if (u.b < 0) return;                                       // (uniform over the block: before any barrier)
  const RowBlock rb(a, u.s, u.rb);
  const int q0 = rb.q0, rows = rb.rows;
  const int p0 = u.s.keys - u.s.rows + q0, plast = p0 + (rb.off + rows - 1) / a.rep;
  const int ntiles = plast < 0 ? 0 : plast / KTL + 1;
  const int it0 = u.sp * u.W, it1 = min(ntiles, it0 + u.W);

  // row 32 w + n of the block; lanes past the last row repeat it and write nothing
  const int r = min(32 * w + n, rows - 1), qi = (rb.off + r) / a.rep, hd = head * a.rep + rb.off + r - qi * a.rep;
  const bool live = 32 * w + n < rows;
  const int mypos = p0 + qi;
  const int wave_last = 32 * w < rows ? p0 + (rb.off + min(32 * w + 31, rows - 1)) / a.rep : -1;
  bf16x8 qf[NS];
  {
    const uint16_t* qrow = a.q + static_cast<int64_t>(u.s.first + q0 + qi) * a.ldq + hd * AD + 8 * hh;
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
    for (int i = 0; i < KLOADS; ++i) {
      constexpr int RPI = 64 / L::KCPR;
      const int row0 = (w * KLOADS + i) * RPI, half = row0 >> 4;
      const int tok = (it * KTL + row0) & mask;
      const int64_t at = static_cast<int64_t>(id_of(it, half)) * a.pg.page_stride + static_cast<int64_t>(head) * a.pg.head_bytes +
                         static_cast<int64_t>(tok) * (AD * 2);
      const int rl = lane / L::KCPR, pc = lane % L::KCPR;
      const uint32_t ko = static_cast<uint32_t>(rl * (AD * 2) + (pc ^ ((row0 + rl) & (L::KCPR - 1))) * 16);
      const uint32_t vo = static_cast<uint32_t>(rl * (AD * 2) + (pc ^ (4 * L::vsw(row0 + rl))) * 16);
      const __amdgpu_buffer_rsrc_t rk = buffer_rsrc(a.pg.k + at, 1024u), rv = buffer_rsrc(a.pg.v + at, 1024u);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_ptr)(st + (w * KLOADS + i) * 1024), 16, ko, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_ptr)(st + (L::K_U4 + (w * KLOADS + i) * 64) * 16), 16, vo, 0, 0, 0);
    }
  };
  // 4 bits: the tile's codes into registers
  [[maybe_unused]] ManyCodes<AD, true> codes;
  [[maybe_unused]] auto fetch = [&](int it) {
    advance(it);
    const int half = half_of_wave(w);
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
    if (it0 + 2 < it1) wait_vm_lgkm0<2 * LOADS>();        // tile it0 landed
    else if (it0 + 1 < it1) wait_vm_lgkm0<LOADS>();
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
      if (it + 2 < it1) wait_vm_lgkm0<LOADS>();           // tile it + 1 landed, tile it + 2 may fly
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
  for (; it + 1 < full; it += 2) {
    if (bad_of(it) | bad_of(it + 1)) break;
    turn(it);
    tile_step<AD>(stage(it), stage(it + 1), qf, sc, sn, o, m, lsum, it * KTL, false, mypos, hh, c, fo);
    turn(it + 1);
    tile_step<AD>(stage(it + 1), stage(it + 2), qf, sn, sc, o, m, lsum, it * KTL + KTL, false, mypos, hh, c, fo);
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
  uint16_t* dst = a.out + static_cast<int64_t>(u.s.first + q0 + qi) * a.ldo + hd * AD + 4 * hh;
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
template <int D, bool RUNS>
__global__ __launch_bounds__(MERGE_THREADS) void k_paged_merge(PagedArgs a) {
  const int rpb = a.rpb;
  constexpr int LPR = D / 4, U = 8;
  __shared__ float4 ls[MERGE_THREADS];
  __shared__ float lm[MERGE_THREADS / LPR], ll[MERGE_THREADS / LPR];
  const int t = threadIdx.x, head = blockIdx.x % a.hkv, slots = blockDim.x / LPR, slot = t / LPR, col = 4 * (t % LPR);
  const int64_t size = static_cast<int64_t>(rpb) * (D + 2);
  // the parts: ns of them, the first at `first`, part s > 0 at rest + s step
  int ns, rows, row0, off;
  const float *first, *rest;
  int64_t step;
  if constexpr (RUNS) {                                      // runs of tiles: its own run's last piece (or first), then first pieces
    const int run = *a.length;
    Seq s0{0, 0, 0};
    if ((t & 63) < a.n_seq) s0 = seq_of(a, t & 63);
    const Piece u = piece_at(a, s0, blockIdx.x / a.hkv, true, t & 63);
    if (u.b < 0) return;
    const int x0 = u.begin / run;
    ns = (u.begin + u.nt - 1) / run - x0 + 1;
    if (u.begin < 0 || x0 + ns > a.fit) return;              // (only with a cu that does not rise: more tiles than 31 bits count)
    const RowBlock r(a, u.s, u.rb);
    off = r.off;
    rows = r.rows;
    row0 = u.s.first + r.q0;
    step = 2 * a.hkv * size;
    rest = a.part + (2 * static_cast<int64_t>(x0) * a.hkv + head) * size;
    first = u.begin == x0 * run ? rest : rest + a.hkv * size;
  } else {
    const Unit u = find_unit(a, blockIdx.x / a.hkv, true);
    // (partials past the last unit: only with a cu that does not rise, whose units the launch does not hold)
    if (u.b < 0 || u.part + static_cast<int64_t>(u.ns - 1) * u.nrb >= a.units) return;
    ns = u.ns;
    const RowBlock r(a, u.s, u.rb);
    off = r.off;
    rows = r.rows;
    row0 = u.s.first + r.q0;
    step = static_cast<int64_t>(u.nrb) * a.hkv * size;
    first = rest = a.part + (u.part * a.hkv + head) * size;
  }
  if (ns == 1) return;
  const int per = (rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
  if (r0 >= r1) return;
  int G = 1;
  while (2 * G * (r1 - r0) <= slots && 2 * G <= ns) G *= 2;
  const int grp = slot % G;
  for (int rb = r0; rb < r1; rb += slots / G) {              // (uniform)
    const int r = rb + slot / G, rc = min(r, r1 - 1);
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = grp; s0 < ns; s0 += U * G) {
      float4 v[U];
      float m[U], l[U];
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int s = min(s0 + x * G, ns - 1);
        const float* p = s ? rest + s * step : first;
        m[x] = p[static_cast<int64_t>(rpb) * D + rc];
        l[x] = p[static_cast<int64_t>(rpb) * (D + 1) + rc];
        v[x] = *reinterpret_cast<const float4*>(p + static_cast<int64_t>(rc) * D + col);
      }
      float now = top;
#pragma unroll
      for (int x = 0; x < U; ++x) now = fmaxf(now, s0 + x * G < ns ? m[x] : -INFINITY);
      const float f0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
      top = now;
      sum *= f0;
      acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
#pragma unroll
      for (int x = 0; x < U; ++x) {
        if (s0 + x * G >= ns) break;                       // (uniform over a group)
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
        for (int x = 0; x < G; ++x) top = fmaxf(top, lm[slot + x]);
        sum = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int x = 0; x < G; ++x) {
          const float m = lm[slot + x], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
          const float4 v = ls[t + x * LPR];
          sum += ll[slot + x] * f;
          acc.x += v.x * f;
          acc.y += v.y * f;
          acc.z += v.z * f;
          acc.w += v.w * f;
        }
      }
    }
    if (grp == 0 && r < r1) {
      const float inv = inverse_sum(sum);
      const int qi = (off + r) / a.rep;
      uint16_t* dst = a.out + static_cast<int64_t>(row0 + qi) * a.ldo + (head * a.rep + off + r - qi * a.rep) * D + col;
      *reinterpret_cast<uint2*>(dst) = make_uint2(bf16_pair(acc.x * inv, acc.y * inv), bf16_pair(acc.z * inv, acc.w * inv));
    }
  }
}

struct Plan {
  bool many, once;
  int fit, kt;
  int64_t blocks, units;                   // (sequence, row block)s at most, and with their splits
  size_t bytes;
  int d;
  int rows() const { return many ? many_rows(d) : 16; }
};

// The most rows a sequence that k_paged_few takes in blocks of 16. 13 sequences of 2000 to 8000 keys, few against many (us):
// bf16, d 128, 12 rows 52 / 55, 28 64 / 58, 64 108 / 63; d 64, 16 rows 22 / 22, 64 28 / 22; d 256, 64 rows 66 / 96, 128
// 105 / 110, 256 185 / 157. 4 bits, d 128, 64 rows 45 / 65, 128 71 / 67, 256 121 / 92; d 64, 64 rows 23 / 23, 128 26 / 25;
// d 256, 256 rows 81 / 146, 512 138 / 239: there k_paged_many is not built (its products take bf16, those of k_paged_few the
// keys' codes at four times the rate, and a wave's 256 columns leave no registers to convert the codes beside them).
constexpr int64_t few_rows(int d, bool mx) { return d == 256 ? (mx ? INT64_MAX : 128) : mx ? 96 : 16; }

// The launch for these sizes: k_paged_few or k_paged_many. Row blocks: sum of ceil(rows rep / rpb) <= T rep / rpb + n_seq.
// k_paged_few: `fit` runs a head, two parts each; k_paged_many: with splits of W tiles at most work / W units more
// (split_length: one round of blocks, or W >= work / 3 fit).
Plan plan_of(int64_t T, int hq, int hkv, int d, bool mx, int n_seq, int64_t max_rows, int64_t max_keys) {
  Plan p{};
  p.d = d;
  const int rep = hq / hkv;
  p.many = std::min<int64_t>(max_rows, T) * rep > few_rows(d, mx);
  p.kt = p.many ? (d == 256 ? Cfg<256>::KT : Cfg<128>::KT) : KT;
  p.blocks = std::min<int64_t>(T * rep, T * rep / p.rows() + n_seq);
  const int round = p.many ? 256 : 256 * few_blocks(d, mx);
  // No splits up to 2048 keys (or where the tiles would not count in 31 bits). One number for all: at most 1000 keys, split against
  // not, 8 sequences of 8 heads of 128 20 / 16 us, one of 2 heads of 64 15 / 11; 2000 keys 8 of 2 heads of 64 18 / 16, of 8 heads of
  // 128 21 / 25, of 2 heads of 256 24 / 46, in 4 bits 18 / 17 and 26 / 27, a chunk of 200 rows 32 / 62; 4000 keys 26 / 43, 4 bits
  // 19 / 28, a chunk 40 / 111. By the number of blocks as well it could begin earlier for chunks and head_dim 256.
  const bool split = max_keys > 16 * NW * KT && static_cast<double>(p.blocks) * static_cast<double>(max_keys / p.kt + 1) < 1e9;
  p.fit = split ? std::max(1, round / hkv) : 0;
  p.once = p.blocks * 4 <= static_cast<int64_t>(p.fit) * 3;
  p.units = !p.fit ? p.blocks : !p.many || p.once ? p.fit : 3 * p.fit + 1 + p.blocks;
  p.bytes = p.fit ? static_cast<size_t>(p.many ? p.units : 2 * p.units) * hkv * (p.rows() * (d + 2)) * 4 + 16 : 0;
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
  if (std::max(p.units, p.blocks) * hkv > INT32_MAX)
    return fail(RF_EINVAL_SHAPE, "%s: %lld blocks of query rows over %d K / V heads", fn, (long long)p.blocks, hkv);
  if (p.fit && (!workspace || ws_bytes < p.bytes)) {
    p.fit = 0;
    p.units = p.blocks;
  }
  const PagedArgs a{q, ldq, T, pg, table, ld_table, static_cast<int>(table_width), lens, cu, n_seq, hq, hkv, hq / hkv, p.rows(),
                    static_cast<int>(std::min<int64_t>(max_rows, T)), static_cast<int>(max_keys),
                    scale * 1.4426950408889634f, out, ldo, static_cast<float*>(workspace),
                    p.fit ? reinterpret_cast<int*>(static_cast<char*>(workspace) + p.bytes) - 4 : nullptr, p.fit, p.once, p.units, p.kt,
                    // key tiles a split at least (a quarter or half of it, this, four times it): one sequence of 4000 keys 16 / 17 /
                    // 33 us, of 6000 in 4 bits 15 / 14 / 20; chunks of 200 rows over 4000 keys 38 / 38 / 46, 2 of 64 over 3000 33 / 36 / 47
                    p.many ? 4 : 2 * NW};
  const dim3 grid(static_cast<unsigned>(p.units * hkv));
  // the merge: a block a row block and head, or a share of its rows; wide blocks where they are few
  const int64_t pairs = p.blocks * hkv, rows = std::min<int64_t>(static_cast<int64_t>(a.max_rows) * a.rep, p.rows());
  const dim3 grid2(static_cast<unsigned>(pairs), static_cast<unsigned>(std::min<int64_t>(p.many ? (rows + 15) / 16 : rows, ((p.many ? 2047 : 511) + pairs) / pairs)));
  const dim3 merge(grid2.x * grid2.y <= 256 ? MERGE_THREADS : 256);
  const bool mx = pages->kind == RF_PAGES_MX4;
#define RF_ATTEND(D)                                                                                     \
  do {                                                                                                   \
    if (p.many && mx) {                                                                                  \
      if constexpr (D != 256) hipLaunchKernelGGL((k_paged_many<D, true>), grid, dim3(64 * many_waves(D)), 0, stream, a); \
    } else if (p.many) hipLaunchKernelGGL((k_paged_many<D, false>), grid, dim3(64 * many_waves(D)), 0, stream, a); \
    else if (mx) hipLaunchKernelGGL((k_paged_few<D, true>), grid, dim3(64 * NW), 0, stream, a);          \
    else hipLaunchKernelGGL((k_paged_few<D, false>), grid, dim3(64 * NW), 0, stream, a);                 \
    if (p.fit) {                                                                                         \
      if (int rc = check_launch(fn)) return rc;                                                          \
      if (p.many) hipLaunchKernelGGL((k_paged_merge<D, false>), grid2, merge, 0, stream, a);   \
      else hipLaunchKernelGGL((k_paged_merge<D, true>), grid2, merge, 0, stream, a);           \
    }                                                                                                    \
  } while (0)
  if (d == 64) RF_ATTEND(64);
  else if (d == 128) RF_ATTEND(128);
  else RF_ATTEND(256);
#undef RF_ATTEND
  return check_launch(fn);
}
