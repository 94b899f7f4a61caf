// The paged cache's row kernels for gfx950: slots of new rows, their K / V into pages (bf16 or 4-bit codes) with norm and
// rotation on the way, and rows read back. All are bound by HBM on many rows and by launch latency on a step's few.
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace rf {
namespace {

// Sequence of row t: the last b with cu[b] <= t (empty sequences share a start, the last of them wins, which holds row t
// if any does). cu need not rise for the search to stay inside [0, n_seq).
__global__ __launch_bounds__(256) void k_paged_slots(const int32_t* __restrict__ table, int64_t ld_table, int64_t width,
                                                     const int32_t* __restrict__ lens, const int32_t* __restrict__ cu,
                                                     int n_seq, int64_t n_pages, int shift, int64_t T,
                                                     int64_t* __restrict__ slots, int64_t* __restrict__ pos) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t >= T) return;
  int lo = 0, hi = n_seq;                                    // cu[lo] <= t (or lo = 0), hi past it
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  int64_t slot = -1, p = 0;
  if (n_seq > 0 && t >= cu[lo] && t < cu[lo + 1]) {
    p = static_cast<int64_t>(lens[lo]) - cu[lo + 1] + t;
    const int64_t at = p >> shift;
    if (p >= 0 && at < width) {
      const int64_t pg = table[lo * ld_table + at];
      if (pg >= 0 && pg < n_pages) slot = (pg << shift) + (p & ((1 << shift) - 1));
    }
    if (p < 0) p = 0;
  }
  slots[t] = slot;
  pos[t] = p;
}

struct AppendArgs {
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  int64_t ld_k, head_k, ld_v, head_v, ld_q, ld_qo, T;
  const int64_t* slots;
  PagesDev pg;
  const uint16_t* cs;
  int rot, hq, hkv;
  uint16_t* q_out;
  const uint16_t* qnorm;
  const uint16_t* knorm;
  int norm_kind;
  float eps;
};

// x g r of 8 values with the gain's 8 entries; the products round one after the other.
__device__ __forceinline__ void normed(float (&f)[8], const uint4& gain, int kind, float r) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float g = bf2f(lane_of(gain, e));
    f[e] = (f[e] * r) * (kind ? 1.0f + g : g);
  }
}

__device__ __forceinline__ void unpack8(float (&f)[8], const uint4& u) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = bf2f(lane_of(u, e));
}

// 4-bit codes of the 8 values a lane holds of a block of 32 (4 lanes side by side); `byte`: the block's scale.
// With a = m 2^n the largest magnitude (1 <= m < 2), the scale is 2^(n - 2), twice that when m > 1.75 (it would round past
// 6): both are read off the bits of a. The bits of NaN and infinity are the largest, so they win the integer maximum.
__device__ __forceinline__ uint32_t encode8(const float (&f)[8], uint32_t& byte) {
  uint32_t a = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) a = max(a, __float_as_uint(f[e]) & 0x7fffffffu);
  a = max(a, static_cast<uint32_t>(__shfl_xor(static_cast<int>(a), 1, 64)));
  a = max(a, static_cast<uint32_t>(__shfl_xor(static_cast<int>(a), 2, 64)));
  const int n = static_cast<int>(a >> 23) - 2 + ((a & 0x7fffffu) > 0x600000u ? 1 : 0);
  byte = a >= 0x7f800000u ? 255u : static_cast<uint32_t>(min(max(n, 1), 254));
  const float s = __uint_as_float((byte == 255u ? 127u : byte) << 23);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], s, 3);
  return byte == 255u ? 0u : c;
}

// Sum over the D / 8 lanes of a head vector, by data-parallel moves within rows of 16 (a sum's two sides in either order).
template <int CTRL>
__device__ __forceinline__ double moved(double v) {
  const uint64_t b = __double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, 0xf, 0xf, true);
  return __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo));
}

template <int D>
__device__ __forceinline__ double vector_sum(double s) {
  s += moved<0xb1>(s);                                       // lanes ^ 1, ^ 2, mirrored in 8, in 16
  s += moved<0x4e>(s);
  s += moved<0x141>(s);
  if constexpr (D > 64) s += moved<0x140>(s);
  if constexpr (D > 128) s += __shfl_xor(s, 16, 64);
  return s;
}

// 1 / sqrt(mean of squares + eps) from the lane's 8 values: the squares of bf16 values and nearly always their sum are exact
// in fp64; the instruction's root gets one step of Newton's. (With the library's root and quotient, sums through LDS and every
// partner normed twice, 6200 rows of 32 query and 8 K / V heads into 4 bits took 38 us, then 35; their 134 MB take 26.)
template <int D>
__device__ __forceinline__ float inverse_rms(const float (&f)[8], float eps) {
  double s = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) s = fma(static_cast<double>(f[e]), static_cast<double>(f[e]), s);
  const double m = vector_sum<D>(s) * (1.0 / D) + static_cast<double>(eps), y = __builtin_amdgcn_rsq(m);
  return static_cast<float>(m < 1e300 ? y * fma(-0.5 * m * y, y, 1.5) : y);       // (an infinity's root is 0)
}

// D / 8 lanes a head vector, 8 values a lane; blockIdx.x is a run of rows, blockIdx.y the head of [queries | keys | values]:
// the rows of one head lie side by side in a block, so that the codes of a page's tokens, side by side in memory, are written
// together. Queries: four heads a block, whose gains and rotation are then loaded once (6200 rows of 32 of them 35 -> 29 us,
// 4.6 TB/s). Heads that stay bf16: a lane takes 4 values and their rotation partners. Keys that become codes: 8 values side by
// side, for a block's scale comes from 4 lanes, and their partners once more (d / 2 apart or less, in L1).
constexpr int HG = 4;
template <int D, bool MX>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
  constexpr int LPR = D / 8, RPB = 256 / LPR;
  const int t = threadIdx.x, c = t % LPR, j0 = 8 * c;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + t / LPR;
  const bool in = row < a.T;
  const int64_t rr = in ? row : a.T - 1;                     // (lanes past the end follow along: the shuffles take all)
  const int groups = (a.hq + HG - 1) / HG, head = static_cast<int>(blockIdx.y) - groups;        // queries: below 0
  const bool is_q = head < 0, is_v = head >= a.hkv;
  const int h = is_q ? static_cast<int>(blockIdx.y) * HG : is_v ? head - a.hkv : head;
  const uint16_t* src = is_q ? a.q + rr * a.ld_q + h * D
                             : is_v ? a.v + rr * a.ld_v + h * a.head_v : a.k + rr * a.ld_k + h * a.head_k;
  const int64_t slot = is_q ? 0 : a.slots[rr];
  const uint16_t* gain = is_q ? a.qnorm : a.knorm;
  const int half = a.cs ? a.rot >> 1 : 0;
  const bool turn = j0 < 2 * half;
  float f[8];
  if (is_q || (!MX && !is_v)) {
    const int ja = turn ? 4 * c : j0, jb = turn ? half + 4 * c : j0 + 4;
    const int64_t page = slot >> a.pg.shift;
    const bool out = !in || slot < 0 || page >= a.pg.n_pages;            // (queries: slot 0)
    uint16_t* dst;
    if (is_q) {
      dst = a.q_out + row * a.ld_qo + h * D;
    } else {
      const int tok = static_cast<int>(slot) & ((1 << a.pg.shift) - 1);
      dst = reinterpret_cast<uint16_t*>(a.pg.k + page * a.pg.page_stride + static_cast<int64_t>(h) * a.pg.head_bytes) + tok * D;
    }
    auto heads = [&](auto count, int n) {                    // n <= count heads side by side
      constexpr int N = decltype(count)::value;
      uint4 raw[N];
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const uint16_t* from = src + min(x, n - 1) * D;
        const uint2 xa = *reinterpret_cast<const uint2*>(from + ja), xb = *reinterpret_cast<const uint2*>(from + jb);
        raw[x] = make_uint4(xa.x, xa.y, xb.x, xb.y);
      }
      uint4 gains = make_uint4(0u, 0u, 0u, 0u), cs = gains;
      if (gain) {
        const uint2 ga = *reinterpret_cast<const uint2*>(gain + ja), gb = *reinterpret_cast<const uint2*>(gain + jb);
        gains = make_uint4(ga.x, ga.y, gb.x, gb.y);
      }
      if (turn) {
        const uint16_t* tab = a.cs + rr * a.rot + 4 * c;
        const uint2 cv = *reinterpret_cast<const uint2*>(tab), sv = *reinterpret_cast<const uint2*>(tab + half);
        cs = make_uint4(cv.x, cv.y, sv.x, sv.y);
      }
#pragma unroll
      for (int x = 0; x < N; ++x) {
        unpack8(f, raw[x]);
        if (gain) normed(f, gains, a.norm_kind, inverse_rms<D>(f, a.eps));
        if (turn) {
#pragma clang fp contract(off)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float co = bf2f(lane_of(cs, e)), si = bf2f(lane_of(cs, e + 4)), y = f[e], z = f[e + 4];
            const float yc = y * co, zs = z * si, zc = z * co, ys = y * si;
            f[e] = yc - zs;
            f[e + 4] = zc + ys;
          }
        }
        if (gain || turn)
          raw[x] = make_uint4(bf16_pair(f[0], f[1]), bf16_pair(f[2], f[3]), bf16_pair(f[4], f[5]), bf16_pair(f[6], f[7]));
        if (!out && x < n) {
          *reinterpret_cast<uint2*>(dst + x * D + ja) = make_uint2(raw[x].x, raw[x].y);
          *reinterpret_cast<uint2*>(dst + x * D + jb) = make_uint2(raw[x].z, raw[x].w);
        }
      }
    };
    if (is_q) heads(std::integral_constant<int, HG>{}, min(HG, a.hq - h));
    else heads(std::integral_constant<int, 1>{}, 1);
    return;
  }
  const uint4 raw = *reinterpret_cast<const uint4*>(src + j0);
  if (MX && !is_v) {
    const bool low = j0 < half;
    const int jp = half == 4 || !turn ? j0 : low ? j0 + half : j0 - half;
    uint4 rawp = raw;
    if (turn) rawp = *reinterpret_cast<const uint4*>(src + jp);
    float p[8];
    unpack8(f, raw);
    unpack8(p, rawp);
    if (gain) {
      const float r = inverse_rms<D>(f, a.eps);
      normed(f, *reinterpret_cast<const uint4*>(gain + j0), a.norm_kind, r);
      normed(p, *reinterpret_cast<const uint4*>(gain + jp), a.norm_kind, r);
    }
    if (turn) {
#pragma clang fp contract(off)
      const uint16_t* tab = a.cs + rr * a.rot;
      if (half >= 8) {
        const uint4 cv = *reinterpret_cast<const uint4*>(tab + (low ? j0 : jp));
        const uint4 sv = *reinterpret_cast<const uint4*>(tab + half + (low ? j0 : jp));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float m = f[e] * bf2f(lane_of(cv, e)), n = p[e] * bf2f(lane_of(sv, e));
          f[e] = low ? m - n : m + n;
        }
      } else {                                               // rot == 8: the lane holds both halves
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float m = p[e] * bf2f(tab[e & 3]), n = p[e ^ 4] * bf2f(tab[4 + (e & 3)]);
          f[e] = e < 4 ? m - n : m + n;
        }
      }
    }
  }
  if (!MX) {                                                 // values as they came
    const int64_t page = slot >> a.pg.shift;
    if (!in || slot < 0 || page >= a.pg.n_pages) return;
    const int tok = static_cast<int>(slot) & ((1 << a.pg.shift) - 1);
    *reinterpret_cast<uint4*>(a.pg.v + page * a.pg.page_stride + static_cast<int64_t>(h) * a.pg.head_bytes + (tok * D + j0) * 2) = raw;
    return;
  }
  if (is_v) unpack8(f, raw);
  uint32_t byte;
  const uint32_t code = encode8(f, byte);
  const int64_t page = slot >> a.pg.shift;
  if (!in || slot < 0 || page >= a.pg.n_pages) return;
  const int tok = static_cast<int>(slot) & ((1 << a.pg.shift) - 1);
  char* dst = (is_v ? a.pg.v : a.pg.k) + page * a.pg.page_stride + static_cast<int64_t>(h) * a.pg.head_bytes;
  if (!is_v) {
    *reinterpret_cast<uint32_t*>(dst + tok * (D / 2) + j0 / 2) = code;
  } else {
    char* run = dst + (tok >> 3) * (4 * D);                  // 8 tokens: 16 runs of 8 x D / 32 bytes
    if (D == 64) {                                           // two runs of 4 values
      *reinterpret_cast<uint16_t*>(run + (2 * c) * 16 + (tok & 7) * 2) = static_cast<uint16_t>(code);
      *reinterpret_cast<uint16_t*>(run + (2 * c + 1) * 16 + (tok & 7) * 2) = static_cast<uint16_t>(code >> 16);
    } else {
      constexpr int RB = D / 32;                             // bytes of a token in a run: 4, or 8 (two lanes)
      *reinterpret_cast<uint32_t*>(run + (j0 / (D / 16)) * (8 * RB) + (tok & 7) * RB + (j0 % (D / 16)) / 2) = code;
    }
  }
  if ((c & 3) == 0) {
    uint8_t* sc = (is_v ? a.pg.vs : a.pg.ks) + page * a.pg.scale_stride + static_cast<int64_t>(h) * a.pg.head_scales;
    sc[(tok >> 3) * (D / 4) + (c >> 2) * 8 + (tok & 7)] = static_cast<uint8_t>(byte);
  }
}

// One lane takes 8 values of one head vector: rows of pages as bf16.
template <int D, bool MX>
__global__ __launch_bounds__(256) void k_paged_read(PagesDev pg, const int64_t* __restrict__ slots, int64_t T, int hkv,
                                                    uint16_t* __restrict__ k_out, int64_t ld_k,
                                                    uint16_t* __restrict__ v_out, int64_t ld_v) {
  constexpr int LPR = D / 8, RPB = 256 / LPR;
  const int t = threadIdx.x, c = t % LPR, j0 = 8 * c;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + t / LPR;
  if (row >= T) return;
  const int h = static_cast<int>(blockIdx.y) % hkv;
  const bool is_v = static_cast<int>(blockIdx.y) >= hkv;
  const int64_t slot = slots[row], page = slot >> pg.shift;
  uint4 x = make_uint4(0u, 0u, 0u, 0u);
  if (slot >= 0 && page < pg.n_pages) {
    const int tok = static_cast<int>(slot) & ((1 << pg.shift) - 1);
    const char* src = (is_v ? pg.v : pg.k) + page * pg.page_stride + static_cast<int64_t>(h) * pg.head_bytes;
    if (!MX) {
      x = *reinterpret_cast<const uint4*>(src + (tok * D + j0) * 2);
    } else {
      uint32_t w;
      if (!is_v) {
        w = *reinterpret_cast<const uint32_t*>(src + tok * (D / 2) + j0 / 2);
      } else {
        const char* run = src + (tok >> 3) * (4 * D);
        if (D == 64) {
          w = *reinterpret_cast<const uint16_t*>(run + (2 * c) * 16 + (tok & 7) * 2) |
              static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(run + (2 * c + 1) * 16 + (tok & 7) * 2)) << 16;
        } else {
          constexpr int RB = D / 32;
          w = *reinterpret_cast<const uint32_t*>(run + (j0 / (D / 16)) * (8 * RB) + (tok & 7) * RB + (j0 % (D / 16)) / 2);
        }
      }
      const uint8_t* sc = (is_v ? pg.vs : pg.ks) + page * pg.scale_stride + static_cast<int64_t>(h) * pg.head_scales;
      const float s = scale_of<0>(sc[(tok >> 3) * (D / 4) + (c >> 2) * 8 + (tok & 7)]);
      x = make_uint4(fp4_pair<0>(w, s), fp4_pair<1>(w, s), fp4_pair<2>(w, s), fp4_pair<3>(w, s));
    }
  }
  uint16_t* dst = is_v ? v_out + row * ld_v : k_out + row * ld_k;
  *reinterpret_cast<uint4*>(dst + h * D + j0) = x;
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" int rf_paged_slots(const int32_t* table, int64_t ld_table, int64_t table_width, const int32_t* lens,
                              const int32_t* cu, int n_seq, int64_t n_pages, int page, int64_t T, int64_t* slots,
                              int64_t* pos, hipStream_t stream) {
  if (!table || !lens || !cu || !slots || !pos) return fail(RF_EINVAL_ARG, "rf_paged_slots: null pointer");
  if (T < 0 || T > INT32_MAX || n_seq < 0 || table_width < 0 || ld_table < table_width || n_pages < 0 || page < 16 ||
      page > 1024 || (page & (page - 1)))
    return fail(RF_EINVAL_SHAPE, "rf_paged_slots: %lld rows, %d sequences, table %lld wide (row stride %lld), %lld pages of "
                "%d tokens (a power of two from 16 to 1024)", (long long)T, n_seq, (long long)table_width,
                (long long)ld_table, (long long)n_pages, page);
  if (T == 0) return RF_OK;
  hipLaunchKernelGGL(k_paged_slots, dim3(static_cast<unsigned>((T + 255) / 256)), dim3(256), 0, stream, table, ld_table,
                     table_width, lens, cu, n_seq, n_pages, log2_of(page), T, slots, pos);
  return check_launch("rf_paged_slots");
}

extern "C" int rf_paged_append(const uint16_t* k, int64_t ld_k, int64_t head_k, const uint16_t* v, int64_t ld_v,
                               int64_t head_v, int64_t T, const int64_t* slots, const rf_pages* pages,
                               const uint16_t* cs, int rot, const uint16_t* q, int64_t ld_q, int hq, uint16_t* q_out,
                               int64_t ld_qo, const uint16_t* qnorm, const uint16_t* knorm, int norm_kind, float eps,
                               hipStream_t stream) {
  const char* fn = "rf_paged_append";
  PagesDev pg;
  if (int rc = check_pages(fn, pages, &pg)) return rc;
  const int d = pages->d, hkv = pages->hkv;
  if (!k || !v || !slots || hq < 0 || (hq > 0) != (q != nullptr) || (q && !q_out))
    return fail(RF_EINVAL_ARG, "%s: null pointer, or queries without heads or an output", fn);
  if ((qnorm && !q) || ((qnorm || knorm) && norm_kind != 0 && norm_kind != 1) || !(eps >= 0.f) || !(eps < 1e30f))
    return fail(RF_EINVAL_ARG, "%s: norm (kind %d, eps %g)", fn, norm_kind, static_cast<double>(eps));
  if (T < 0 || T > INT32_MAX || ld_k % 8 || ld_v % 8 || head_k % 8 || head_v % 8 || head_k < d || head_v < d || ld_k < d ||
      ld_v < d || hq > 4096 || (q && (ld_q < static_cast<int64_t>(hq) * d || ld_qo < static_cast<int64_t>(hq) * d ||
      ld_q % 8 || ld_qo % 8)))
    return fail(RF_EINVAL_SHAPE, "%s: %lld rows, strides (K %lld / %lld, V %lld / %lld, q %lld, out %lld)", fn, (long long)T,
                (long long)ld_k, (long long)head_k, (long long)ld_v, (long long)head_v, (long long)ld_q, (long long)ld_qo);
  if (cs && (rot <= 0 || rot > d || rot % 2 || ((rot / 2) % 8 && rot / 2 != 4)))
    return fail(RF_EUNSUPPORTED, "%s: rotary dims %d of head_dim %d", fn, rot, d);
  if (!aligned16(k) || !aligned16(v) || !aligned16(cs) || !aligned16(q) || !aligned16(q_out) || !aligned16(qnorm) ||
      !aligned16(knorm))
    return fail(RF_EINVAL_SHAPE, "%s: pointers must be 16-byte aligned", fn);
  if (T == 0) return RF_OK;
  const AppendArgs a{k, v, q, ld_k, head_k, ld_v, head_v, ld_q, ld_qo, T, slots, pg, cs, cs ? rot : 0, hq, hkv, q_out,
                     qnorm, knorm, norm_kind, eps};
  const int rpb = 256 / (d / 8);
  const bool mx = pages->kind == RF_PAGES_MX4;
  const dim3 grid(static_cast<unsigned>((T + rpb - 1) / rpb), static_cast<unsigned>((hq + HG - 1) / HG + 2 * hkv));
#define RF_APPEND(D)                                                                                     \
  if (mx) hipLaunchKernelGGL((k_paged_append<D, true>), grid, dim3(256), 0, stream, a);                  \
  else hipLaunchKernelGGL((k_paged_append<D, false>), grid, dim3(256), 0, stream, a)
  if (d == 64) { RF_APPEND(64); }
  else if (d == 128) { RF_APPEND(128); }
  else { RF_APPEND(256); }
#undef RF_APPEND
  return check_launch(fn);
}

extern "C" int rf_paged_read(const rf_pages* pages, const int64_t* slots, int64_t T, uint16_t* k_out, int64_t ld_k,
                             uint16_t* v_out, int64_t ld_v, hipStream_t stream) {
  const char* fn = "rf_paged_read";
  PagesDev pg;
  if (int rc = check_pages(fn, pages, &pg)) return rc;
  const int d = pages->d, hkv = pages->hkv;
  if (!slots || !k_out || !v_out) return fail(RF_EINVAL_ARG, "%s: null pointer", fn);
  if (T < 0 || T > INT32_MAX || ld_k < static_cast<int64_t>(hkv) * d || ld_v < static_cast<int64_t>(hkv) * d || ld_k % 8 ||
      ld_v % 8 || !aligned16(k_out) || !aligned16(v_out))
    return fail(RF_EINVAL_SHAPE, "%s: %lld rows, strides %lld / %lld or alignment", fn, (long long)T, (long long)ld_k,
                (long long)ld_v);
  if (T == 0) return RF_OK;
  const int rpb = 256 / (d / 8);
  const dim3 grid(static_cast<unsigned>((T + rpb - 1) / rpb), static_cast<unsigned>(2 * hkv));
  const bool mx = pages->kind == RF_PAGES_MX4;
#define RF_READ(D)                                                                                                         \
  if (mx) hipLaunchKernelGGL((k_paged_read<D, true>), grid, dim3(256), 0, stream, pg, slots, T, hkv, k_out, ld_k, v_out, ld_v); \
  else hipLaunchKernelGGL((k_paged_read<D, false>), grid, dim3(256), 0, stream, pg, slots, T, hkv, k_out, ld_k, v_out, ld_v)
  if (d == 64) { RF_READ(64); }
  else if (d == 128) { RF_READ(128); }
  else { RF_READ(256); }
#undef RF_READ
  return check_launch(fn);
}
