// The key tile of the many-query attentions (attend_causal.hip, attend_paged.hip): its LDS layout, fragment reads, scores and
// softmax step. attend_causal.hip's head describes the arithmetic.
#pragma once
#include "rf_common.h"

namespace rf {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Per head_dim: keys per tile KT; 8 waves per block (two per SIMD), 32 query rows each. d 64 / 128:
// 64-key tiles. d 256: 32-key tiles keep four 32 KB stages in LDS; a wave's queries take 64 registers and
// its O^T 128 of the 256 two waves per SIMD leave it, so the tile loads' per-lane offsets are recomputed
// at each issue instead of held, and a few values still spill (outside the key loop but for one query
// fragment and the edge tiles' lane offset).
template <int AD>
struct Cfg {
  static constexpr int KT = AD == 256 ? 32 : 64;
  static constexpr int NW = 8;
  static constexpr int NTHR = 64 * NW;
  static constexpr int QROWS = 32 * NW;  // query rows (query, head) per block: 32 per wave
  static constexpr int KB = KT / 32;     // 32-key halves of a tile
};
constexpr int NSTAGE = 4;              // LDS stages: three tiles in flight, one still read

__device__ __forceinline__ bf16x8 as_frag(const uint4& u) { return __builtin_bit_cast(bf16x8, u); }

typedef __attribute__((address_space(3))) void* lds_ptr;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0), static_cast<int>(bytes),
                                           0x00020000);
}

// s_waitcnt with vmcnt <= n and lgkmcnt = 0 (expcnt not waited), gfx9 encoding.
template <int n>
__device__ __forceinline__ void wait_vm_lgkm0() {
  static_assert(n >= 0 && n < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((n & 15) | (7 << 4) | (0 << 8) | ((n >> 4) << 14));
}

// LDS layout of one stage: the K tile then the V tile, each 64 keys x AD row-major in 16-byte chunks. K row
// r's chunk c sits at r * KCPR + (c ^ (r % KCPR)): the score fragment reads (32 rows, one chunk per lane)
// hit distinct banks. V row r's chunk c sits at K_U4 + r * KCPR + (c ^ (4 vsw(r))): a transpose read takes
// 8 bytes in each of 4 consecutive rows over 4 chunks per row per 32 lanes, and the swizzle moves the four
// rows onto four different 64-byte bank ranges.
template <int AD, int KEYS = Cfg<AD>::KT, int WAVES = Cfg<AD>::NW>
struct Layout {
  static constexpr int KT = KEYS, NW = WAVES;
  static constexpr int KCPR = AD / 8;
  static constexpr int K_U4 = KT * KCPR;
  static constexpr int V_U4 = KT * KCPR;
  static constexpr int STAGE_U4 = K_U4 + V_U4;
  static constexpr int KLOADS = K_U4 / 64 / NW;     // direct-load instructions per wave per tile
  static constexpr int VLOADS = V_U4 / 64 / NW;
  static constexpr int LOADS = KLOADS + VLOADS;
  static_assert(KLOADS * 64 * NW == K_U4 && VLOADS * 64 * NW == V_U4, "tile loads must split evenly");
  static_assert(NSTAGE * STAGE_U4 * 16 <= 160 * 1024, "stages fit the LDS");
  __device__ static int kslot(int row, int c) { return row * KCPR + (c ^ (row & (KCPR - 1))); }
  // d 128 / 256: a row is 256 / 512 bytes, rows r .. r + 3 shift by 0, 64, 128, 192 bytes; d 64: rows are
  // 128 bytes, row parity already picks the half of a 256-byte bank line, and rows r, r + 2 shift by 0 and 64
  __device__ static int vsw(int row) { return AD >= 128 ? (row & 3) : ((row >> 1) & 1); }
  __device__ static int vslot(int row, int c) { return K_U4 + row * KCPR + (c ^ (4 * vsw(row))); }
};

// Headroom of the lazy softmax rescale: the running reference maximum is raised only when a score
// exceeds it by more than this (in base 2), so probabilities stay below 2^8 and the O rescale runs
// only on the tiles that raise it.
constexpr float RESCALE_LOG2 = 8.0f;

// That headroom in raw scores (c = scale log2(e)), a float still where c is tiny: from a maximum of -infinity any score rises.
__device__ __forceinline__ float headroom(float c) { return fminf(RESCALE_LOG2 / c, 3e38f); }

// Per-lane LDS byte offsets of the fragments within a stage, the same for every tile. K fragment (key
// half kb, d step s): row 32 kb + n, chunk 2 s + hh, at k(s) + kb * 32 KCPR 16 (row 32 kb + n has the
// swizzle of row n). V^T fragment (d block b, 16-key step stp): lane l = 16 g + t takes, in each of two
// transpose reads, row 16 stp + 8 i + 4 (g / 2) + t / 4 (i = 0, 1) at d 32 b + 16 (g % 2) + 4 (t % 4)
// (8 bytes), and receives keys 16 stp + 8 i + 4 (g / 2) + 0 .. 3 of d 32 b + 16 (g % 2) + t: the fragment
// order {0..3, 8..11} + 4 hh. Its byte offset is v(b) + (16 stp + 8 i) KCPR 16 (rows 16 stp + 8 i + r have
// the swizzle of row r).
// Both are one XOR per read: the K chunk 2 s + hh = 2 s ^ hh, so its swizzled byte offset within row n is
// 32 s ^ 16 (hh ^ (n % KCPR)), and the row's base n KCPR 16 has no bits in common with it; the V^T block
// offset 64 (b ^ vsw) = 64 b ^ 64 vsw sits in bits 6 .. 8, which the rest of the V offset leaves clear.
template <int AD>
struct FragOffsets {
  uint32_t kz, vz;
  __device__ FragOffsets(int lane, int k_u4 = Layout<AD>::K_U4) {          // (the tile's keys, in 16-byte chunks)
    using L = Layout<AD>;
    const int n = lane & 31, hh = lane >> 5, g = lane >> 4, t = lane & 15;
    kz = static_cast<uint32_t>(n * L::KCPR * 16) | static_cast<uint32_t>(16 * (hh ^ (n & (L::KCPR - 1))));
    const int r0 = 4 * (g >> 1) + (t >> 2), cl = 2 * (g & 1) + ((t & 3) >> 1);
    vz = static_cast<uint32_t>((k_u4 + r0 * L::KCPR + cl) * 16 + 8 * (t & 1)) |
         static_cast<uint32_t>(64 * L::vsw(r0));
  }
  __device__ uint32_t k(int s) const { return kz ^ static_cast<uint32_t>(32 * s); }
  __device__ uint32_t v(int b) const { return vz ^ static_cast<uint32_t>(64 * b); }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Four keys of one d column per lane out of the row-major V tile (ds_read_b64_tr_b16).
__device__ __forceinline__ uint2 read_tr(const char* p) {
  const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
  return __builtin_bit_cast(uint2, v);
}

// The two lane halves' values of a lane pair (l, l ^ 32), the same in both lanes: v of the lower lane
// and v of the upper lane (one v_permlane32_swap).
__device__ __forceinline__ void lane_pair(float v, float& lo, float& hi) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  lo = __uint_as_float(r[0]);
  hi = __uint_as_float(r[1]);
}

// S^T = K Q^T for one key tile (KB halves of 32 keys) and the wave's 32 queries: sc[kb][j] = the raw
// score of key 32 kb + 8 (j / 4) + 4 hh + j % 4 of the tile for query n. (The stage pointers are
// __restrict__: the LDS reads then carry alias information, and the compiler does not make them wait for
// the direct loads in flight into the other stages; the kernel's own waits order them.)
template <int AD, int KB = Cfg<AD>::KB>
__device__ __forceinline__ void tile_scores(const char* __restrict__ st, const bf16x8 (&qf)[AD / 16],
                                            f32x16 (&sc)[KB], const FragOffsets<AD>& fo) {
  using L = Layout<AD>;
  constexpr int NS = AD / 16;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[kb][r] = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s)
      sc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          as_frag(*reinterpret_cast<const uint4*>(st + fo.k(s) + kb * 32 * L::KCPR * 16)), qf[s], sc[kb], 0, 0, 0);
  }
}

// One tile's softmax and products, with the next tile's scores interleaved: mask the scores sc of the
// tile at key k0 when some key lies past some query of the wave (edge), raise the lane's reference
// maximum mref (raw-score units, -inf until a key is visible) lazily, then in one block the base-2
// probabilities exp2(fma(s, c, -mref c)) of sc (c = scale * log2(e) > 0) beside the MFMAs of the next
// tile's scores sn (from stage sn_st), and O^T += V^T P^T from this tile's stage st.
template <int AD, int KB = Cfg<AD>::KB>
__device__ __forceinline__ void tile_step(const char* __restrict__ st, const char* __restrict__ sn_st,
                                          const bf16x8 (&qf)[AD / 16], f32x16 (&sc)[KB],
                                          f32x16 (&sn)[KB], f32x16 (&o)[AD / 32], float& mref, float& lsum,
                                          int k0, bool edge, int mypos, int hh, float c,
                                          const FragOffsets<AD>& fo) {
  using L = Layout<AD>;
  constexpr int NB = AD / 32, NS = AD / 16, KT = 32 * KB;
  constexpr int NP = 8 * KB;                            // probability pairs per lane
  if (edge) {
    // key 32 kb + 8 (j / 4) + 4 hh + j % 4 of the tile is past the query when its offset exceeds rel
    const int rel = min(max(mypos - k0, -1), KT) - 4 * hh;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (32 * kb + 8 * (j >> 2) + (j & 3) > rel) sc[kb][j] = -INFINITY;
  }
  float tmax = -INFINITY;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int j = 0; j < 16; ++j) tmax = fmaxf(tmax, sc[kb][j]);
  float lo, hi;
  lane_pair(tmax, lo, hi);
  tmax = fmaxf(lo, hi);
  if (tmax > mref + headroom(c)) {                 // raise the reference (always on the first visible key)
    const float alpha = __builtin_amdgcn_exp2f((mref - tmax) * c);    // 0 while mref is -inf
    mref = tmax;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][r] *= alpha;
    lsum *= alpha;
  }
  const float mc = mref == -INFINITY ? 0.f : mref * c;  // every key so far masked (a split past the query)
  // the next tile's KB NS score MFMAs, the NP probability pairs spread between them
  float psum = 0.f;
  uint32_t pk[NP];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int r = 0; r < 16; ++r) sn[kb][r] = 0.f;
#pragma unroll
  for (int q = 0; q < KB * NS; ++q) {
    const int kb = q / NS, s = q % NS;
    sn[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        as_frag(*reinterpret_cast<const uint4*>(sn_st + fo.k(s) + kb * 32 * L::KCPR * 16)), qf[s], sn[kb], 0, 0, 0);
#pragma unroll
    for (int e = q * NP / (KB * NS); e < (q + 1) * NP / (KB * NS); ++e) {
      const int pkb = e / 8, pj = 2 * (e % 8);
      const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[pkb][pj], c, -mc));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[pkb][pj + 1], c, -mc));
      psum += p0 + p1;
      pk[e] = bf16_pair(p0, p1);
    }
  }
  lsum += psum;
  // O^T[d, query] += V^T[d, keys] P^T[keys, query] over the tile's 16-key steps (keys 16 stp ..: chunks
  // 2 stp and 2 stp + 1; P^T step stp = the lane's probabilities 8 stp .. 8 stp + 7)
#pragma unroll
  for (int stp = 0; stp < KT / 16; ++stp) {
    const bf16x8 pf = __builtin_bit_cast(bf16x8, make_uint4(pk[4 * stp], pk[4 * stp + 1], pk[4 * stp + 2],
                                                             pk[4 * stp + 3]));
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const char* vp = st + fo.v(b) + 16 * stp * L::KCPR * 16;
      const uint2 vl = read_tr(vp), vh = read_tr(vp + 8 * L::KCPR * 16);
      o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_frag(make_uint4(vl.x, vl.y, vh.x, vh.y)), pf, o[b], 0, 0, 0);
    }
  }
}

}  // namespace
}  // namespace rf
