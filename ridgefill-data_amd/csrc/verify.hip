// Verification of drafted tokens against the target's probabilities, gfx950: from given random numbers, which path of a tree of
// drafted tokens is accepted and which token follows it.
//
// With p the softmax of a row's logits over its temperature and w = e^((x - top) / T) its weights:
//   no draft probabilities: a child's token is accepted if u Z < w(token), Z the weight of the tokens that are not rejected yet.
//   draft probabilities q (the children of a row were drawn from them): after a rejection what is left is
//       p' = max(p - q, 0) / sum max(p - q, 0). With c_0 = 0, Z_0 = 1 and c_{k+1} = c_k + Z_k the k-th of them is
//       max(p - c_k q, 0) / Z_k, Z_k = sum max(p - c_k q, 0): max(max(a, 0) - b, 0) = max(a - b, 0) for b >= 0. So a rejection
//       takes one pass over a row and no memory; a child's token is accepted if u q Z_k < max(p - c_k q, 0).
//   the next token: the first at which the running sum of what is left exceeds r times its total.
// The answers are whole numbers and a draw may lie next to a border (there are as many as tokens), so weights and sums are in
// 64 bits: the vector pipe's 64-bit products run at the rate of 32-bit ones. Without a draft the walk begins with sums of whole rows
// from 32-bit weights (k_verify_rows) and takes a test that they leave open again with a 64-bit sum of what is left (walk).
//
// Three launches. k_verify_rows: every row with children gets its largest logit and weight sum by chunks (which rows a path meets
// is known row by row only, and a launch a row costs more than reading the others; a row without children is read only where a
// path ends). k_verify_sums: the blocks of a sequence, one a chunk, gather its rows' numbers into LDS, take the walk, each the
// same, up to the first sums that it needs (what a rejection leaves, or the last row's weights), and sum their own chunk.
// k_verify_draw: a block a sequence draws, or, where a draft's token was rejected before its last sibling or a test was left open,
// walks on alone.
// (The last two as one, its last block going on: the fences before and behind the count of blocks that are done take 50 ns a
// block, one after the other: 60 us for 32 sequences over 32 chunks.)
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "rf_common.h"

namespace rf {
namespace {

constexpr int CHUNK = 4096;                // logits a share of a row has at least, and a block of k_verify_sums at once
constexpr int MAX_CHUNKS = 128;
constexpr int MAX_ROWS = 1024;             // of a sequence
constexpr int NT = 256;                    // threads of k_verify_rows
constexpr int NW = 512;                    // of k_verify_sums
constexpr int ND = 1024;                   // of k_verify_draw

struct Part {                              // of some of a row's logits: the largest logit, where it first is (-1: nowhere), and the
  float top;                               // sum of the weights relative to it (0 for greedy rows)
  int best;
  double sum;
};

struct Stop;

struct VerifyArgs {
  const char* logits;
  int64_t ld, T;
  int V, chunks, shares;                   // chunks of a row; the waves that read one in k_verify_rows
  const int64_t* tokens;
  const int32_t* parents;
  const int32_t* cu;
  int n_seq;
  const float* u;
  const float* r;
  const float* temperature;
  const char* draft;
  int64_t ld_draft;
  int rows, depth;                         // of a sequence at most
  int32_t* path;
  int64_t ld_path;
  int32_t* count;
  int64_t* next;
  Part* parts;                             // [T, shares]
  Part* ends;                              // [n_seq, chunks * RUNS]: of the row whose sums a walk wants first, by runs
  Stop* stops;                             // [n_seq]
  int32_t* gone;                           // [n_seq, rows]
};

// N values from element e on, of which n are there (the others: 0, not read). Rows begin at any element.
template <class E, int N>
__device__ __forceinline__ void load(float (&f)[N], const E* p, int n) {
  if (n >= N) {
    E w[N];
    __builtin_memcpy(w, p, sizeof(w));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (sizeof(E) == 2) f[i] = bf2f(w[i]);
      else f[i] = w[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f[i] = 0.f;
      if (i < n) {
        if constexpr (sizeof(E) == 2) f[i] = bf2f(p[i]);
        else f[i] = p[i];
      }
    }
  }
}

template <class E>
__device__ __forceinline__ float load1(const E* p) {
  float f[1];
  load<E, 1>(f, p, 1);
  return f[0];
}

__device__ __forceinline__ float logit(float x) { return x == x ? x : -INFINITY; }        // NaN: never taken
__device__ __forceinline__ float share(float q) { return q > 0.f ? q : 0.f; }             // (of a draft; NaN: none)

typedef uint32_t words2 __attribute__((ext_vector_type(2)));

// 2^t for -1022 <= t <= 0, to 3e-12: n = t to the nearest whole by adding 1.5 2^52 (n is then in the low word), 2^(t - n) =
// 1 + f g(f) with g interpolated at the 8 Chebyshev nodes of [-1/2, 1/2] (2^0 is 1 exactly), and n added to the exponent. The
// coefficients are kept in scalar registers: as literals each is two moves beside its product.
struct Exp2 {
  double g[8];
  __device__ Exp2() : g{0x1.62e42fef9cc69p-1, 0x1.ebfbdff82a734p-3, 0x1.c6b08da70cce3p-5, 0x1.3b2ab70ad2565p-7,
                        0x1.5d877598350eap-10, 0x1.4308c7183d8ecp-13, 0x1.00c0e4e1528e6p-16, 0x1.63b2d796dd1efp-20} {
#pragma unroll
    for (int i = 0; i < 8; ++i) asm("" : "+s"(g[i]));
  }
  __device__ __forceinline__ double operator()(double t) const {
    constexpr double WHOLE = 6755399441055744.0;
    const double n = t + WHOLE, f = t - (n - WHOLE);
    double p = g[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) p = __builtin_fma(p, f, g[i]);
    p = __builtin_fma(p, f, 1.0);
    words2 w = __builtin_bit_cast(words2, p);                // (low, high)
    w.y += __builtin_bit_cast(words2, n).x << 20;
    return __builtin_bit_cast(double, w);
  }
};

// The weight of a logit x <= top relative to top: 2^((x - top) c), c = log2(e) / T; nothing below 2^-1022, for -infinity and
// NaN. An infinite top is shared by the logits like it (any c), c = 0 by all above -infinity.
__device__ __forceinline__ double weight(const Exp2& e, float x, float top, double c) {
  const double t = x == top ? 0.0 : __builtin_fmax((static_cast<double>(x) - static_cast<double>(top)) * c, -1022.0);
  const double w = e(t);
  return t > -1022.0 && x > -INFINITY ? w : 0.0;
}

__device__ __forceinline__ double slope(float t) { return 1.4426950408889634 / static_cast<double>(t); }

__device__ __forceinline__ double shfl_xor64(double v, int m) { return __shfl_xor(v, m, 64); }

// The sequence that row t may lie in (as rf_paged_slots): the last b with cu[b] <= t. A wave looks at 64 offsets at once.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int n_seq, int64_t t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n_seq;                                    // cu[lo] <= t (or lo = 0), hi past it
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const uint64_t below = __ballot(at < hi && (lane == 0 || cu[min(at, n_seq)] <= t));
    const int k = 63 - __clzll(static_cast<long long>(below));
    hi = min(hi, lo + (k + 1) * step);
    lo += k * step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Largest of a block's THREADS values; every thread gets it. (lds: a value a wave; the barrier before its next use is the caller's)
template <int THREADS>
__device__ __forceinline__ float block_top(float v, float* lds) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int x = 1; x < THREADS / 64; ++x) v = fmaxf(v, lds[x]);
  return v;
}

// A wave's 1024 logits from element e0 on, 16 a lane in loads of 16 bytes; past the vocabulary -infinity.
template <class E>
struct Step {
  static constexpr int N = 16 / sizeof(E), I = 16 / N, SIZE = 1024;
  float f[16];
  __device__ __forceinline__ static int at(int e0, int k) { return e0 + (k / N) * 64 * N + static_cast<int>(threadIdx.x & 63) * N + k % N; }
  __device__ __forceinline__ void fetch(const E* row, int e0, int V) {
    if (e0 + SIZE <= V) {                                    // (uniform)
#pragma unroll
      for (int i = 0; i < I; ++i) load<E, N>(reinterpret_cast<float(&)[N]>(f[i * N]), row + at(e0, i * N), N);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) f[k] = at(e0, k) < V ? load1(row + at(e0, k)) : -INFINITY;
    }
  }
};

// How far, of themselves, sums without a draft may be off: those of k_verify_rows, and 64-bit ones (weights 3e-12, scaled twice).
constexpr double ROW_ERROR = 1e-5, SUM_ERROR = 2e-11;

// A wave a share of a row: chunks share, share + shares .. Sums are relative to the first step's largest logit as long as the
// others stay near it, so a step has no more to do than its maximum and its weights.
// EXACT (with a draft: p - c q, and with it every border of what is left, moves with the row's sum): weights in 64 bits, 16
// instructions a logit (none of them at a quarter of the rate), as 2^(x c - ref c) of logits not below ref - 1000 / c (those, NaN
// and -infinity count 2^-1000). Without a draft a row's sum decides only whether u Z < w, and the draw sums its row again: there
// weights are in 32 bits, 16 of them a sum in 32 bits and those in 64. A weight 2^t is off by three roundings of its exponent (the
// difference, c, the product), t 3 2^-24 ln 2 of itself, by 2^-23 of v_exp_f32 and 5 2^-24 of the sum; no t is above 64 (the reference
// is raised), and weights below 2^-64 are nothing beside the reference's 1: a sum is within 8.4e-6 of itself, ROW_ERROR with room.
// (527 rows of 151936 in bf16, of which 374 have children: 52 us in 64 bits, 35 in 32; their bytes take 22.)
// Where reference and slope allow neither, weight by weight.
template <class E, bool EXACT>
__global__ __launch_bounds__(NT) void k_verify_rows(VerifyArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * (NT / 64) + (threadIdx.x >> 6);
  const int shares = a.shares;
  const int64_t row = __builtin_amdgcn_readfirstlane(static_cast<int>(task / shares));
  const int share = __builtin_amdgcn_readfirstlane(static_cast<int>(task - row * shares));
  if (row >= a.T) return;
  const int b = sequence_of(a.cu, a.n_seq, row);
  const int64_t c0 = a.cu[b], c1 = min<int64_t>(a.cu[b + 1], a.T);
  if (row < c0 || row >= c1) return;                         // a row of no sequence
  const float temp = a.temperature ? a.temperature[b] : 0.f;
  const bool drawn = temp > 0.f;
  if (a.temperature) {                                       // has it children? (without temperatures nothing reads a path's end again)
    bool any = false;
    for (int64_t i = row + 1; i < c1 && !any; i += 64) any = __any(i + lane < c1 && a.parents[min(i + lane, c1 - 1)] == row - c0);
    if (!any) return;
  }
  const E* src = reinterpret_cast<const E*>(a.logits) + row * a.ld;
  const Exp2 e2;
  const double c = drawn ? slope(temp) : 0.0;
  const float reach = EXACT ? static_cast<float>(1000.0 / c) : 0.f, c32 = static_cast<float>(c);
  constexpr int STEPS = CHUNK / 1024;
  const int chunks = (a.chunks - share + shares - 1) / shares, steps = chunks * STEPS;
  auto begin = [&](int i) { return (share + i / STEPS * shares) * CHUNK + i % STEPS * 1024; };
  Step<E> now, coming;
  now.fetch(src, begin(0), a.V);
  float top = -INFINITY, ref = -INFINITY, lo = 0.f;          // the lane's largest logit, the sums' reference
  double sum = 0, k = 0;
  bool fast = false;
  int best = INT32_MAX;
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    if (i + 1 < steps) coming.fetch(src, begin(i + 1), a.V);
    float own = now.f[0];
#pragma unroll
    for (int x = 1; x < 16; ++x) own = fmaxf(own, now.f[x]);   // (NaN is left out by the maximum)
    if (own > top) {
      top = own;
#pragma unroll
      for (int x = 15; x >= 0; --x)
        if (now.f[x] == own) best = now.at(begin(i), x);
    }
    if (drawn) {
      if (!__all(fast ? (static_cast<double>(top) - ref) * c < (EXACT ? 500 : 64) : top == -INFINITY)) {
        float high = top;                                    // the first reference, or a new one
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) high = fmaxf(high, __shfl_xor(high, m, 64));
        if (high > ref) {
          sum = ref > -INFINITY ? sum * weight(e2, ref, high, c) : 0.0;
          ref = high;
          if constexpr (EXACT) {
            lo = ref - reach;
            k = -ref * c;
            const double far = (static_cast<double>(ref) - lo) * c;
            fast = far > 100 && far < 1020 && k > -1024 && k < 1024;
          } else {
            fast = ref < INFINITY && ref > -1e30f && c > 1e-25 && c < 1e25;            // (-3e38 is then nothing)
          }
        }
      }
      if (__builtin_expect(fast, 1)) {                       // (uniform; the median of three is its smallest where one is NaN)
        std::conditional_t<EXACT, double, float> s[4] = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          if constexpr (EXACT) s[x & 3] += e2(__builtin_fma(static_cast<double>(__builtin_amdgcn_fmed3f(now.f[x], lo, INFINITY)), c, k));
          else s[x & 3] += __builtin_amdgcn_exp2f((__builtin_amdgcn_fmed3f(now.f[x], -3e38f, INFINITY) - ref) * c32);
        }
        sum += (s[0] + s[1]) + (s[2] + s[3]);
      } else if (ref > -INFINITY) {
#pragma unroll
        for (int x = 0; x < 16; ++x) sum += weight(e2, now.f[x], ref, c);
      }
    }
    now = coming;
  }
  float high = top;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) high = fmaxf(high, __shfl_xor(high, m, 64));
  int first = top == high ? best : INT32_MAX;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    first = min(first, __shfl_xor(first, m, 64));
    sum += shfl_xor64(sum, m);
  }
  if (lane == 0)
    a.parts[row * shares + share] = Part{high, high > -INFINITY ? first : -1, drawn && high > -INFINITY ? sum * weight(e2, ref, high, c) : 0.0};
}

// What a block knows of its sequence's rows, in LDS. Of rows without children in a sequence that is not greedy: no sums.
struct Rows {
  double* sum;                             // of the weights
  double* w;                               // its token's weight in its parent's row
  float* top;
  int* best;
  int* parent;
  int* token;                              // -1: none of the vocabulary's
  float* q;                                // its share of its parent's row of the draft
  float* u;
  __device__ Rows(char* lds, int rows) {
    sum = reinterpret_cast<double*>(lds);
    w = sum + rows;
    top = reinterpret_cast<float*>(w + rows);
    best = reinterpret_cast<int*>(top + rows);
    parent = best + rows;
    token = parent + rows;
    q = reinterpret_cast<float*>(token + rows);
    u = q + rows;
  }
};
constexpr int ROW_BYTES = 40;

struct Block {                             // a block's sequence
  int b, n;                                // its rows
  int64_t first;
  double slope;
  bool greedy;
};

__device__ __forceinline__ Block block_of(const VerifyArgs& a, int b) {
  const int64_t c0 = max(a.cu[b], 0), c1 = min<int64_t>(a.cu[b + 1], a.T);
  Block s;
  s.b = b;
  s.first = c0;
  s.n = static_cast<int>(max<int64_t>(0, min<int64_t>(c1 - c0, a.rows)));
  const float temp = a.temperature ? a.temperature[b] : 0.f;
  s.greedy = !(temp > 0.f);
  s.slope = s.greedy ? 0.0 : slope(temp);
  return s;
}

template <class E, class Q, int THREADS>
__device__ __forceinline__ void gather(const VerifyArgs& a, const Block& s, const Rows& l, const Exp2& e2) {
  const int t = threadIdx.x, j = t & 15;
  const E* logits = reinterpret_cast<const E*>(a.logits) + s.first * a.ld;
  // a row's parts by 16 lanes (their first loads go before those of the rows, which wait for one another)
#pragma unroll 1
  for (int i0 = 0; i0 < s.n; i0 += THREADS / 16) {
    const int i = i0 + t / 16;
    const Part* parts = a.parts + (s.first + min(i, s.n - 1)) * a.shares;
    const Part p0 = parts[min(j, a.shares - 1)], p1 = parts[min(j + 16, a.shares - 1)];
    if (i0 == 0) {
#pragma unroll 1
      for (int r = t; r < s.n; r += THREADS) {
        const int p = r ? a.parents[s.first + r] : -1;
        const int64_t tok = a.tokens[s.first + r];
        const int par = p >= 0 && p < r ? p : -1, id = tok >= 0 && tok < a.V ? static_cast<int>(tok) : -1;
        l.parent[r] = par;
        l.token[r] = id;
        l.u[r] = a.u ? a.u[s.first + r] : 0.f;
        const bool in = par >= 0 && id >= 0;
        l.w[r] = in && !s.greedy ? logit(load1(logits + par * a.ld + id)) : -INFINITY;       // (its logit first)
        l.q[r] = in && a.draft ? share(load1(reinterpret_cast<const Q*>(a.draft) + (s.first + par) * a.ld_draft + id)) : 0.f;
      }
    }
    float top = j < a.shares ? p0.top : -INFINITY;
    int best = top > -INFINITY ? p0.best : INT32_MAX;
    auto larger = [&](const Part& p) {
      if (p.top > top || (p.top == top && p.best < best)) {
        top = p.top;
        best = p.best;
      }
    };
    if (j + 16 < a.shares) larger(p1);
#pragma unroll 1
    for (int x = j + 32; x < a.shares; x += 16) larger(parts[x]);
    float all = top;
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) all = fmaxf(all, __shfl_xor(all, m, 64));
    if (top != all) best = INT32_MAX;
    double sum = 0;
    if (!s.greedy && all > -INFINITY) {
      Part p = p0;
#pragma unroll 1
      for (int x = j; x < a.shares; x += 16) {
        if (x >= 32) p = parts[x];
        if (p.top > -INFINITY) sum += p.sum * weight(e2, p.top, all, s.slope);               // (rows without sums: left out)
        p = p1;
      }
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) {
      best = min(best, __shfl_xor(best, m, 64));
      sum += shfl_xor64(sum, m);
    }
    if (j == 0 && i < s.n) {
      l.top[i] = all;
      l.best[i] = all > -INFINITY ? best : -1;
      l.sum[i] = sum;
    }
  }
  __syncthreads();
  if (!s.greedy) {
#pragma unroll 1
    for (int r = t; r < s.n; r += THREADS)
      l.w[r] = l.parent[r] >= 0 && l.token[r] >= 0 ? weight(e2, static_cast<float>(l.w[r]), l.top[l.parent[r]], s.slope) : 0.0;
    __syncthreads();
  }
}

// Where a sequence's path has come to.
struct State {
  int node, count, next;                   // next: the row from which on the node's children are still to be tested
  double c, Z;                             // what is left of the node's distribution (without a draft Z in weights, off by up to c)
  bool cut;                                // a draft's token was rejected here
  bool fresh;                              // without a draft: Z was summed for the next test
};

// ... when its first sums are wanted, for k_verify_draw.
struct Stop {
  State st;
  double sum;                              // of the node's weights (cut)
  float top;
  int more, n_gone;                        // whether the walk goes on, the tokens rejected at its last row (without a draft)
};

// The walk from st on, by every wave with the same numbers. True: Z of the node is wanted for the next child, of a drawn token's
// rejection sum max(p - c q, 0), without a draft the weights left, because u Z lies nearer to w than Z is known (the row's sum is off
// by up to ROW_ERROR, and what a rejection leaves by as much as the whole: where little is left of a row, nearly every test); false:
// the path has ended (cut: with a rejected token, and c is new).
__device__ __forceinline__ bool walk(const VerifyArgs& a, const Block& s, const Rows& l, State& st) {
  const int lane = threadIdx.x & 63;
  const bool drawn = a.draft != nullptr && !s.greedy;
  auto child = [&](int from) {                               // the next row below the node; -1: none
#pragma unroll 1
    for (int i0 = from; i0 < s.n; i0 += 64) {
      const uint64_t hit = __ballot(i0 + lane < s.n && l.parent[min(i0 + lane, s.n - 1)] == st.node);
      if (hit) return i0 + __ffsll(static_cast<unsigned long long>(hit)) - 1;
    }
    return -1;
  };
#pragma unroll 1
  while (st.count < a.depth) {
    const int at = __builtin_amdgcn_readfirstlane(child(st.next));
    if (at < 0) return false;
    st.next = at + 1;
    const int tok = l.token[at];
    bool yes;
    if (s.greedy) {
      yes = tok >= 0 && tok == l.best[st.node];
    } else if (!drawn) {
      if (st.Z < 0) {                                        // (the node's first child)
        st.Z = l.sum[st.node];
        st.c = ROW_ERROR * st.Z;
      }
      bool gone = tok < 0;                                   // rejected before, or no token at all
      for (int k0 = st.node + 1; k0 < at; k0 += 64) {
        const int k = min(k0 + lane, at - 1);
        gone |= __any(k0 + lane < at && l.parent[k] == st.node && l.token[k] == tok);
      }
      const double own = gone ? 0.0 : l.w[at], mark = l.u[at] * st.Z;
      if (own > 0 && !st.fresh && __builtin_fabs(mark - own) <= l.u[at] * st.c + SUM_ERROR * own) {
        st.next = at;
        return true;
      }
      st.fresh = false;
      yes = mark < own;
      if (!yes) st.Z = __builtin_fmax(st.Z - own, 0.0);
    } else {
      const double q = l.q[at], total = l.sum[st.node];
      const double p = total > 0 ? __builtin_fmax(l.w[at] / total - st.c * q, 0.0) : 0.0;
      yes = tok >= 0 && l.u[at] * q * st.Z < p;
      if (!yes) {
        st.c += st.Z;
        st.cut = true;
        return child(st.next) >= 0;
      }
    }
    if (yes) {
      st.node = at;
      st.c = 0.0;
      st.Z = drawn ? 1.0 : -1.0;
      st.cut = false;
      ++st.count;
    }
  }
  return false;
}

// 1 / S once a row: as p of the walk's tests but for its last bit. (0 for a row of nothing)
__device__ __forceinline__ double inverse(double s) { return s > 0 ? 1.0 / s : 0.0; }

// What is left of a row: its weights without the tokens in `gone`, or max(p - c q, 0).
template <class E, class Q>
struct Left {
  const E* src;
  const Q* from;                           // null: weights
  double slope, inv, c;
  const int* gone;
  int n_gone;
};

// The tokens rejected at the node without a draft, each once, in the rows' order, by one wave: of the children before the next one to be
// tested. Returns how many.
__device__ __forceinline__ int rejected(const Block& s, const Rows& l, const State& st, int* gone) {
  const int lane = threadIdx.x & 63, end = min(st.next, s.n);
  int m = 0;
#pragma unroll 1
  for (int k0 = st.node + 1; k0 < end; k0 += 64) {
    const int k = min(k0 + lane, end - 1), tok = l.token[k];
    bool here = k0 + lane < end && l.parent[k] == st.node && tok >= 0;
#pragma unroll 1
    for (int y = st.node + 1; here && y < k; ++y) here = !(l.parent[y] == st.node && l.token[y] == tok);
    const uint64_t mask = __ballot(here);
    if (here) gone[m + __popcll(mask & ((1ull << lane) - 1))] = tok;
    m += __popcll(mask);
  }
  return m;
}

// A lane's four elements e .. e + 3: logits (NaN, what is gone and what lies past the vocabulary as -infinity) and shares.
template <class E, class Q>
__device__ __forceinline__ void fetch4(const Left<E, Q>& left, float (&f)[4], float (&q)[4], int e, int V) {
  load<E, 4>(f, left.src + min(e, V), V - e);
  if (left.from) load<Q, 4>(q, left.from + min(e, V), V - e);
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = e + k < V ? logit(f[k]) : -INFINITY;
#pragma unroll 1
  for (int g = 0; g < left.n_gone; ++g) {
    const int at = left.gone[g] - e;
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = at == k ? -INFINITY : f[k];
  }
}

template <class E, class Q>
__device__ __forceinline__ double left4(const Left<E, Q>& left, const Exp2& e2, double (&w)[4], const float (&f)[4],
                                        const float (&q)[4], float top) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k] = weight(e2, f[k], top, left.slope);
    if (left.from) w[k] = __builtin_fmax(w[k] * left.inv - left.c * share(q[k]), 0.0);
  }
  return (w[0] + w[1]) + (w[2] + w[3]);
}

// A wave's run of RUN elements, four a lane of its first half and four of its second: its sum and its largest logit (of what is
// left by a draft: relative to the row's).
constexpr int RUN = 512, RUNS = CHUNK / RUN;
static_assert(RUNS == NW / 64, "a wave a run of a chunk");
template <class E, class Q>
__device__ __forceinline__ Part sum_run(const Left<E, Q>& left, const Exp2& e2, int run, int V, float top) {
  const int lane = threadIdx.x & 63;
  float f[2][4], q[2][4] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) fetch4(left, f[k], q[k], run * RUN + 256 * k + 4 * lane, V);
  if (!left.from) {
    top = fmaxf(fmaxf(fmaxf(f[0][0], f[0][1]), fmaxf(f[0][2], f[0][3])), fmaxf(fmaxf(f[1][0], f[1][1]), fmaxf(f[1][2], f[1][3])));
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  }
  double sum = 0, w[4];
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    sum += left4(left, e2, w, f[0], q[0], top);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[0][i] = f[1][i], q[0][i] = q[1][i];
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sum += shfl_xor64(sum, m);
  return Part{top, 0, sum};
}

// The path of a sequence from its last row up, and its length.
__device__ __forceinline__ void write_path(const VerifyArgs& a, int b, const int* parent, const State& st) {
  int32_t* path = a.path + b * a.ld_path;
#pragma unroll 1
  for (int j = st.count + threadIdx.x; j < a.depth; j += blockDim.x) path[j] = -1;
  if (threadIdx.x) return;
  int at = st.node;
#pragma unroll 1
  for (int j = st.count - 1; j >= 0; --j) {
    path[j] = at;
    at = parent[at];
  }
  a.count[b] = st.count;
}

template <class E, class Q>
__device__ __forceinline__ Left<E, Q> left_of(const VerifyArgs& a, const Block& s, const State& st, double sum, const int* gone, int n_gone) {
  return Left<E, Q>{reinterpret_cast<const E*>(a.logits) + (s.first + st.node) * a.ld,
                    st.cut ? reinterpret_cast<const Q*>(a.draft) + (s.first + st.node) * a.ld_draft : nullptr, s.slope,
                    st.cut ? inverse(sum) : 1.0, st.c, gone, n_gone};
}

// `blocks` blocks a sequence; without temperatures one, which has the answers.
template <class E, class Q>
__global__ __launch_bounds__(NW) void k_verify_sums(VerifyArgs a, int blocks) {
  extern __shared__ double lds[];
  __shared__ int n_gone;
  const int b = blockIdx.x / blocks, x = blockIdx.x - b * blocks, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const Block s = block_of(a, b);
  if ((s.n == 0 || !a.temperature) && x) return;             // (uniform)
  const Rows l(reinterpret_cast<char*>(lds), a.rows);
  State st{0, 0, 1, 0.0, a.draft != nullptr ? 1.0 : -1.0, false, false};
  if (s.n == 0) {
    write_path(a, b, l.parent, st);
    if (t == 0) a.next[b] = -1;
    return;
  }
  st.count = 1;
  const Exp2 e2;
  gather<E, Q, NW>(a, s, l, e2);
  const bool more = walk(a, s, l, st);
  if (x == 0) write_path(a, b, l.parent, st);
  if (!a.temperature) {
    if (t == 0) a.next[b] = l.best[st.node];
    return;
  }
  // the tokens rejected at the last row, each once, in the rows' order; they take the place of the rows' u
  int* gone = reinterpret_cast<int*>(l.u);
  int dropped = 0;
  if (a.draft == nullptr && !s.greedy) {
    __syncthreads();
    if (wave == 0) {
      const int m = rejected(s, l, st, gone);
      if (lane == 0) n_gone = m;
    }
    __syncthreads();
    dropped = n_gone;
  }
  const Left<E, Q> left = left_of<E, Q>(a, s, st, l.sum[st.node], gone, dropped);
#pragma unroll 1
  for (int run = x * RUNS + wave; run * RUN < a.V; run += blocks * RUNS) {
    const Part p = sum_run(left, e2, run, a.V, l.top[st.node]);
    if (lane == 0) a.ends[static_cast<int64_t>(b) * a.chunks * RUNS + run] = p;
  }
  if (x) return;
  if (t == 0) a.stops[b] = Stop{st, l.sum[st.node], l.top[st.node], more, dropped};
#pragma unroll 1
  for (int g = t; g < dropped; g += NW) a.gone[static_cast<int64_t>(b) * a.rows + g] = gone[g];
}

// A block a sequence.
template <class E, class Q>
__global__ __launch_bounds__(ND) void k_verify_draw(VerifyArgs a) {
  extern __shared__ double lds[];
  __shared__ float tops[ND / 64];
  __shared__ int found, n_gone;
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, runs = (a.V + RUN - 1) / RUN;
  const Part* ends = a.ends + static_cast<int64_t>(b) * a.chunks * RUNS;
  const Part mine = ends[min(t, runs - 1)];
  const Stop stop = a.stops[b];
  const Block s = block_of(a, b);
  if (s.n == 0) return;                                      // (uniform)
  const Rows l(reinterpret_cast<char*>(lds), a.rows);
  double* cs = reinterpret_cast<double*>(reinterpret_cast<char*>(lds) + static_cast<size_t>((a.rows + 1) & ~1) * ROW_BYTES);    // the runs' sums
  float* ct = reinterpret_cast<float*>(cs + runs);           // ... and largest logits
  int* gone = reinterpret_cast<int*>(ct + runs);
  const Exp2 e2;
  State st = stop.st;
  bool more = stop.more;
#pragma unroll 1
  for (int g = t; g < stop.n_gone; g += ND) gone[g] = a.gone[static_cast<int64_t>(b) * a.rows + g];
  Left<E, Q> left = left_of<E, Q>(a, s, st, stop.sum, gone, stop.n_gone);
  float top = stop.top;                                      // what the sums are relative to
#pragma unroll 1
  for (int y = t; y < runs; y += ND) {
    const Part p = y < ND ? mine : ends[y];
    ct[y] = p.top;
    cs[y] = p.sum;
  }
  if (more) gather<E, Q, ND>(a, s, l, e2);
  while (true) {
    if (!st.cut) {                                           // (runs' sums are relative to their own)
      float own = -INFINITY;
#pragma unroll 1
      for (int y = t; y < runs; y += ND) own = fmaxf(own, ct[y]);
      top = block_top<ND>(own, tops);
      if (s.greedy) break;
#pragma unroll 1
      for (int y = t; y < runs; y += ND) cs[y] = ct[y] > -INFINITY ? cs[y] * weight(e2, ct[y], top, s.slope) : 0.0;
    }
    __syncthreads();
    if (!more) break;
    double z = 0;                                            // (every wave the same)
#pragma unroll 1
    for (int y = lane; y < runs; y += 64) z += cs[y];
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) z += shfl_xor64(z, m);
    if (st.cut) {
      st.Z = z;
    } else {                                                 // (as the children's weights, relative to the row's largest logit)
      st.Z = z * weight(e2, top, l.top[st.node], s.slope);
      st.c = SUM_ERROR * st.Z;
      st.fresh = true;
    }
    more = walk(a, s, l, st);
    __syncthreads();                                         // then further sums, of another test or the last row
    int dropped = 0;
    if (a.draft == nullptr) {
      if (wave == 0) {
        const int m = rejected(s, l, st, gone);
        if (lane == 0) n_gone = m;
      }
      __syncthreads();
      dropped = n_gone;
    }
    top = l.top[st.node];
    left = left_of<E, Q>(a, s, st, l.sum[st.node], gone, dropped);
#pragma unroll 1
    for (int run = wave; run < runs; run += ND / 64) {
      const Part p = sum_run(left, e2, run, a.V, top);
      if (lane == 0) {
        ct[run] = p.top;
        cs[run] = p.sum;
      }
    }
    __syncthreads();
  }
  if (stop.more) write_path(a, b, l.parent, st);
  if (s.greedy) {                                            // the first of the row's largest logits, in the first run that has it
    __syncthreads();
    if (t == 0) found = INT32_MAX;
    __syncthreads();
#pragma unroll 1
    for (int y = t; y < runs; y += ND)
      if (ct[y] == top) atomicMin(&found, y);                // (whole numbers: in any order)
    __syncthreads();
    const int e = found * RUN + t;
    __syncthreads();
    if (t == 0) found = INT32_MAX;
    __syncthreads();
    if (top > -INFINITY && t < RUN && e < a.V && load1(left.src + e) == top) atomicMin(&found, e);
    __syncthreads();
    if (t == 0) a.next[b] = found == INT32_MAX ? -1 : found;
    return;
  }
  // the draw, by one wave: the run, then the token in it, at which the running sum first exceeds r times the total
  if (wave == 0) {
    int next = -1;
    const int per = (runs + 63) / 64, y0 = min(lane * per, runs), y1 = min(y0 + per, runs);
    double own = 0;
#pragma unroll 1
    for (int y = y0; y < y1; ++y) own += cs[y];
    auto scan_of = [&](double v) {                           // inclusive sums over the lanes
#pragma unroll 1
      for (int m = 1; m < 64; m <<= 1) {
        const double y = __shfl_up(v, m, 64);
        if (lane >= m) v += y;
      }
      return v;
    };
    const double upto = scan_of(own), total = __shfl(upto, 63, 64), want = a.r[b] * total;
    double before = upto - own, base = 0;
    int run = -1, end = -1;
#pragma unroll 1
    for (int y = y0; y < y1; ++y) {
      if (cs[y] > 0) {
        end = y;
        if (run < 0 && before + cs[y] > want) {
          run = y;
          base = before;
        }
      }
      before += cs[y];
    }
    const uint64_t hit = __ballot(run >= 0), some = __ballot(end >= 0);
    if (some) {
      if (hit) {
        const int at = __ffsll(static_cast<unsigned long long>(hit)) - 1;
        run = __shfl(run, at, 64);
        base = __shfl(base, at, 64);
      } else {                                               // r of 1 or more, or a rounding: the last token there is
        run = __shfl(end, 63 - __clzll(static_cast<long long>(some)), 64);
        base = -INFINITY;
      }
      int tail = -1;
#pragma unroll 1
      for (int k = 0; k < 2 && next < 0; ++k) {
        const int e = run * RUN + 256 * k + 4 * lane;
        float f[4], q[4] = {};
        double w[4];
        fetch4(left, f, q, e, a.V);
        const double four = left4(left, e2, w, f, q, top), sums = scan_of(four);
        double at = base + (sums - four);
        int first = -1, some_last = -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          at += w[i];
          if (w[i] > 0) {
            some_last = e + i;
            if (first < 0 && at > want) first = e + i;
          }
        }
        const uint64_t here = __ballot(first >= 0), any = __ballot(some_last >= 0);
        if (here) next = __shfl(first, __ffsll(static_cast<unsigned long long>(here)) - 1, 64);
        if (any) tail = __shfl(some_last, 63 - __clzll(static_cast<long long>(any)), 64);
        base += __shfl(sums, 63, 64);
      }
      if (next < 0) next = tail;
    }
    if (lane == 0) found = next >= 0 ? next : INT32_MAX;
  }
  __syncthreads();
  if (found == INT32_MAX) {                                  // nothing is left: the row's largest logit
    float own = -INFINITY;
#pragma unroll 1
    for (int e = t; e < a.V; e += ND) own = fmaxf(own, load1(left.src + e));
    own = block_top<ND>(own, tops);
    if (own > -INFINITY)
#pragma unroll 1
      for (int e = t; e < a.V; e += ND)
        if (load1(left.src + e) == own) atomicMin(&found, e);        // (whole numbers: in any order)
    __syncthreads();
  }
  if (t == 0) a.next[b] = found == INT32_MAX ? -1 : found;
}

int sizes(const char* fn, int64_t T, int64_t V, int n_seq, int64_t max_rows, int* chunks) {
  if (V < 1 || V > static_cast<int64_t>(MAX_CHUNKS) * CHUNK)
    return fail(RF_EUNSUPPORTED, "%s: a vocabulary of %lld (up to %d)", fn, (long long)V, MAX_CHUNKS * CHUNK);
  if (max_rows < 0 || max_rows > MAX_ROWS)
    return fail(RF_EUNSUPPORTED, "%s: %lld rows a sequence (up to %d)", fn, (long long)max_rows, MAX_ROWS);
  *chunks = static_cast<int>((V + CHUNK - 1) / CHUNK);
  if (T < 0 || n_seq < 0 || n_seq > (1 << 20) || T > (1 << 30) || static_cast<int64_t>(n_seq) * *chunks > INT32_MAX)
    return fail(RF_EINVAL_SHAPE, "%s: %lld rows of %d sequences over a vocabulary of %lld", fn, (long long)T, n_seq, (long long)V);
  return RF_OK;
}

// Waves a row in k_verify_rows: 8192 in all (a CU holds 28), a chunk each at least.
int shares_of(int64_t T, int chunks) { return static_cast<int>(std::min<int64_t>(chunks, std::max<int64_t>(1, 8192 / std::max<int64_t>(T, 1)))); }

// The workspace: parts, ends, stops, gone.
struct Space {
  size_t ends, stops, gone, bytes;
  Space(int64_t T, int n_seq, int chunks, int64_t max_rows)
      : ends(static_cast<size_t>(T) * shares_of(T, chunks) * sizeof(Part)),
        stops(ends + static_cast<size_t>(n_seq) * chunks * RUNS * sizeof(Part)), gone(stops + static_cast<size_t>(n_seq) * sizeof(Stop)),
        bytes(gone + static_cast<size_t>(n_seq) * std::min(max_rows, T) * 4) {}
};

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" int rf_verify_drafts_workspace_bytes(int64_t T, int64_t vocab, int n_seq, int64_t max_rows, size_t* bytes) {
  const char* fn = "rf_verify_drafts_workspace_bytes";
  int chunks;
  if (!bytes) return fail(RF_EINVAL_ARG, "%s: null pointer", fn);
  if (int rc = sizes(fn, T, vocab, n_seq, max_rows, &chunks)) return rc;
  *bytes = T && n_seq ? Space(T, n_seq, chunks, max_rows).bytes : 0;
  return RF_OK;
}

extern "C" int rf_verify_drafts(const void* logits, int logits_kind, int64_t ld, int64_t vocab, int64_t T, const int64_t* tokens,
                                const int32_t* parents, const int32_t* cu, int n_seq, const float* u, const float* r,
                                const float* temperature, const void* draft, int draft_kind, int64_t ld_draft, int64_t max_rows,
                                int64_t depth, int32_t* path, int64_t ld_path, int32_t* count, int64_t* next, void* workspace,
                                size_t ws_bytes, hipStream_t stream) {
  const char* fn = "rf_verify_drafts";
  int chunks;
  if (int rc = sizes(fn, T, vocab, n_seq, max_rows, &chunks)) return rc;
  if (n_seq == 0) return RF_OK;
  if (!cu || !path || !count || !next || (T && (!logits || !tokens || !parents || !workspace)) || (temperature && T && (!u || !r)))
    return fail(RF_EINVAL_ARG, "%s: null pointer", fn);
  if ((logits_kind != RF_F32 && logits_kind != RF_BF16) || (draft && draft_kind != RF_F32 && draft_kind != RF_BF16))
    return fail(RF_EINVAL_ARG, "%s: kinds %d, %d of logits and draft", fn, logits_kind, draft_kind);
  if (ld < vocab || (draft && ld_draft < vocab) || depth < 1 || depth > MAX_ROWS || ld_path < depth)
    return fail(RF_EINVAL_SHAPE, "%s: row strides %lld, %lld for a vocabulary of %lld, paths of %lld rows (row stride %lld)", fn,
                (long long)ld, (long long)ld_draft, (long long)vocab, (long long)depth, (long long)ld_path);
  const int size = logits_kind == RF_F32 ? 4 : 2, dsize = draft_kind == RF_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size || (draft && reinterpret_cast<uintptr_t>(draft) % dsize) || !aligned16(workspace))
    return fail(RF_EINVAL_SHAPE, "%s: alignment", fn);
  const Space space(T, n_seq, chunks, max_rows);
  if (T && ws_bytes < space.bytes)
    return fail(RF_EINVAL_ARG, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, space.bytes);
  const bool drawn = temperature && T;
  char* ws = static_cast<char*>(workspace);
  const VerifyArgs a{static_cast<const char*>(logits), ld, T, static_cast<int>(vocab), chunks, shares_of(T, chunks), tokens, parents, cu, n_seq, u, r,
                     T ? temperature : nullptr, drawn ? static_cast<const char*>(draft) : nullptr, ld_draft,
                     static_cast<int>(std::min<int64_t>(max_rows, T)), static_cast<int>(depth), path, ld_path, count, next,
                     reinterpret_cast<Part*>(ws), reinterpret_cast<Part*>(ws + space.ends), reinterpret_cast<Stop*>(ws + space.stops),
                     reinterpret_cast<int32_t*>(ws + space.gone)};
  const size_t rows = static_cast<size_t>((a.rows + 1) & ~1) * ROW_BYTES, sums = static_cast<size_t>((vocab + RUN - 1) / RUN) * 12 + static_cast<size_t>(a.rows) * 4;
  // k_verify_sums: a block a chunk, fewer where that is more than a round of blocks (two a CU): 32 sequences over 32 chunks
  // 19 us with a block a chunk, 15 with 16 blocks each
  const dim3 grid(static_cast<unsigned>((T * a.shares + NT / 64 - 1) / (NT / 64)));
  const int blocks = drawn ? std::min(chunks, std::max(1, 512 / n_seq)) : 1;
#define RF_VERIFY(E, Q)                                                                                                       \
  do {                                                                                                                        \
    if (T && a.draft) hipLaunchKernelGGL((k_verify_rows<E, true>), grid, dim3(NT), 0, stream, a);                             \
    else if (T) hipLaunchKernelGGL((k_verify_rows<E, false>), grid, dim3(NT), 0, stream, a);                                  \
    hipLaunchKernelGGL((k_verify_sums<E, Q>), dim3(static_cast<unsigned>(n_seq * blocks)), dim3(NW), rows + 16, stream, a, blocks); \
    if (drawn) hipLaunchKernelGGL((k_verify_draw<E, Q>), dim3(static_cast<unsigned>(n_seq)), dim3(ND), rows + sums, stream, a); \
  } while (0)
  if (logits_kind == RF_F32) {
    if (!a.draft || draft_kind == RF_F32) RF_VERIFY(float, float);
    else RF_VERIFY(float, uint16_t);
  } else {
    if (a.draft && draft_kind == RF_F32) RF_VERIFY(uint16_t, float);
    else RF_VERIFY(uint16_t, uint16_t);
  }
#undef RF_VERIFY
  return check_launch(fn);
}
