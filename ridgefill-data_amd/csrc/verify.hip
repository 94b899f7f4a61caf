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
// 64 bits: the vector pipe's 64-bit products run at the rate of 32-bit ones, and 17 instructions a logit stay below what HBM
// takes to bring four bytes of it.
//
// Which rows a path meets is known row by row only, and a launch a row costs more than reading the others: the first launch
// takes every row's largest logit and weight sums by chunks (HBM's rate is its bound), the last walks (a block a sequence; its
// rows' numbers are gathered at once into LDS) and finds the next token in one chunk. With draft probabilities a launch between
// them has the sums of the first row in which a token is rejected, on as many blocks as the row has chunks; later rejections
// the walking block sums by itself.
#include <stdint.h>

#include <algorithm>

#include "rf_common.h"

namespace rf {
namespace {

constexpr int CHUNK = 4096;                // logits a block of the passes over rows
constexpr int MAX_CHUNKS = 256;
constexpr int MAX_ROWS = 1024;             // of a sequence
constexpr int NT = 256;                    // threads of the passes
constexpr int NW = 1024;                   // of the walk

struct Part {                              // of a chunk of a row: its largest logit, where it first is (-1: nowhere), and the
  float top;                               // sum of the weights relative to it (0 for greedy rows)
  int best;
  double sum;
};

struct VerifyArgs {
  const char* logits;
  int64_t ld, T;
  int V, chunks;
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
  Part* parts;                             // [T, chunks]
  double* rest;                            // [n_seq, chunks]
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

// 2^t for t <= 0 (below -1075: 0; NaN likewise), to 3e-12: n = t to the nearest whole, 2^(t - n) = 1 + f g(f) with g
// interpolated at the 8 Chebyshev nodes of [-1/2, 1/2] (2^0 is 1 exactly).
__device__ __forceinline__ double exp2_64(double t) {
  t = __builtin_fmax(t, -1100.0);
  const double n = __builtin_rint(t), f = t - n;
  double g = 0x1.63b2d796dd1efp-20;
  g = __builtin_fma(g, f, 0x1.00c0e4e1528e6p-16);
  g = __builtin_fma(g, f, 0x1.4308c7183d8ecp-13);
  g = __builtin_fma(g, f, 0x1.5d877598350eap-10);
  g = __builtin_fma(g, f, 0x1.3b2ab70ad2565p-7);
  g = __builtin_fma(g, f, 0x1.c6b08da70cce3p-5);
  g = __builtin_fma(g, f, 0x1.ebfbdff82a734p-3);
  g = __builtin_fma(g, f, 0x1.62e42fef9cc69p-1);
  return __builtin_amdgcn_ldexp(__builtin_fma(g, f, 1.0), static_cast<int>(n));
}

// A row's weights relative to its largest logit: log2(e) / T, or (odd) an infinite logit or temperature, where the largest
// logits or all that are not -infinity share alike.
struct Scale {
  double c;
  float top;
  bool odd;
  __device__ Scale(double c, float top) : c(c), top(top), odd(!(top < INFINITY) || !(c > 0)) {}
  __device__ __forceinline__ double even(float x) const { return exp2_64((static_cast<double>(x) - top) * c); }
  __device__ __forceinline__ double weight(float x) const {
    if (odd) return top < INFINITY ? (x > -INFINITY ? 1.0 : 0.0) : (x == top ? 1.0 : 0.0);
    return x > -INFINITY ? even(x) : 0.0;                    // (a row of nothing: top is -infinity too)
  }
};

__device__ __forceinline__ double slope(float t) { return 1.4426950408889634 / static_cast<double>(t); }

__device__ __forceinline__ double shfl_xor64(double v, int m) { return __shfl_xor(v, m, 64); }

// The sequence that row t may lie in (as rf_paged_slots): the last b with cu[b] <= t.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int n_seq, int64_t t) {
  int lo = 0, hi = n_seq;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A block a (row, chunk): 256 threads x 16 logits, all loaded before the first is used.
template <class E>
__global__ __launch_bounds__(NT) void k_verify_rows(VerifyArgs a) {
  constexpr int N = 16 / sizeof(E), I = CHUNK / NT / N;      // values a load, loads
  const int64_t row = blockIdx.x / a.chunks;
  const int x = static_cast<int>(blockIdx.x - row * a.chunks), t = threadIdx.x, lane = t & 63;
  __shared__ float tops[NT / 64];
  __shared__ int bests[NT / 64];
  __shared__ double sums[NT / 64];
  const int b = sequence_of(a.cu, a.n_seq, row);
  if (row < a.cu[b] || row >= a.cu[b + 1]) return;           // a row of no sequence (uniform)
  const E* src = reinterpret_cast<const E*>(a.logits) + row * a.ld;
  float f[I][N];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int e = x * CHUNK + (i * NT + t) * N;
    load<E, N>(f[i], src + e, a.V - e);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      f[i][k] = e + k < a.V ? logit(f[i][k]) : -INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) top = fmaxf(top, f[i][k]);
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  if (lane == 0) tops[t >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  int best = INT32_MAX;
#pragma unroll
  for (int i = I - 1; i >= 0; --i)
#pragma unroll
    for (int k = N - 1; k >= 0; --k)
      if (f[i][k] == top) best = x * CHUNK + (i * NT + t) * N + k;
  const float temp = a.temperature ? a.temperature[b] : 0.f;
  double sum = 0;
  if (temp > 0.f && top > -INFINITY) {                       // (uniform)
    const Scale s(slope(temp), top);
    if (s.odd) {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) sum += s.weight(f[i][k]);
    } else {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) sum += s.even(f[i][k]);
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    best = min(best, __shfl_xor(best, m, 64));
    sum += shfl_xor64(sum, m);
  }
  if (lane == 0) {
    bests[t >> 6] = best;
    sums[t >> 6] = sum;
  }
  __syncthreads();
  if (t == 0) {
    best = min(min(bests[0], bests[1]), min(bests[2], bests[3]));
    a.parts[blockIdx.x] = Part{top, top > -INFINITY ? best : -1, (sums[0] + sums[1]) + (sums[2] + sums[3])};
  }
}

// What a block knows of its sequence's rows, in LDS.
struct Rows {
  double* sum;                             // of the weights
  float* top;
  int* best;
  int* parent;
  int* token;                              // -1: none of the vocabulary's
  float* x;                                // its logit in its parent's row
  float* q;                                // its share of its parent's row of the draft
  float* u;
  __device__ Rows(char* lds, int rows) {
    sum = reinterpret_cast<double*>(lds);
    top = reinterpret_cast<float*>(sum + rows);
    best = reinterpret_cast<int*>(top + rows);
    parent = best + rows;
    token = parent + rows;
    x = reinterpret_cast<float*>(token + rows);
    q = x + rows;
    u = q + rows;
  }
};
constexpr int ROW_BYTES = 36;

// Where a sequence's path has come to.
struct State {
  int node, count;
  double c, Z;                             // what is left of the node's distribution (Z in weights without a draft)
  bool cut;                                // a draft's token was rejected here
};

struct Block {                             // a block of `threads` threads on sequence b
  int b, n;                                // its rows
  int64_t first;
  double slope;
  bool greedy;
};

template <class E, class Q>
__device__ void gather(const VerifyArgs& a, const Block& s, const Rows& l, int threads) {
  const int t = threadIdx.x;
  const E* logits = reinterpret_cast<const E*>(a.logits);
  for (int i = t; i < s.n; i += threads) {
    const int p = i ? a.parents[s.first + i] : -1;
    const int64_t tok = a.tokens[s.first + i];
    const int par = p >= 0 && p < i ? p : -1, id = tok >= 0 && tok < a.V ? static_cast<int>(tok) : -1;
    l.parent[i] = par;
    l.token[i] = id;
    l.u[i] = a.u ? a.u[s.first + i] : 0.f;
    const bool in = par >= 0 && id >= 0;
    l.x[i] = in ? logit(load1(logits + (s.first + par) * a.ld + id)) : -INFINITY;
    l.q[i] = in && a.draft ? share(load1(reinterpret_cast<const Q*>(a.draft) + (s.first + par) * a.ld_draft + id)) : 0.f;
  }
  // a row's chunks by 16 lanes
  const int j = t & 15;
  for (int i0 = 0; i0 < s.n; i0 += threads / 16) {
    const int i = i0 + t / 16;
    const Part* parts = a.parts + (s.first + min(i, s.n - 1)) * a.chunks;
    float top = -INFINITY;
    int best = INT32_MAX;
    for (int x = j; x < a.chunks; x += 16) {
      const float m = parts[x].top;
      if (m > top) {
        top = m;
        best = parts[x].best;
      }
    }
    float all = top;
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) all = fmaxf(all, __shfl_xor(all, m, 64));
    if (top != all) best = INT32_MAX;
    double sum = 0;
    if (!s.greedy && all > -INFINITY) {
      const Scale sc(s.slope, all);
      for (int x = j; x < a.chunks; x += 16) sum += parts[x].sum * sc.weight(parts[x].top);
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
}

// The walk: every wave takes it with the same numbers. rest(node, c) gives sum max(p - c q, 0) of a row, or NaN for "stop here".
template <class F>
__device__ State walk(const VerifyArgs& a, const Block& s, const Rows& l, bool write, F&& rest) {
  const int lane = threadIdx.x & 63;
  const bool drawn = a.draft != nullptr && !s.greedy;
  State st{0, 1, 0.0, drawn ? 1.0 : l.sum[0], false};
  if (write) a.path[s.b * a.ld_path] = 0;
  int i = 1;
  while (st.count < a.depth) {
    // the next row below the node
    int at = -1;
    for (int i0 = i; i0 < s.n; i0 += 64) {
      const uint64_t hit = __ballot(i0 + lane < s.n && l.parent[min(i0 + lane, s.n - 1)] == st.node);
      if (hit) {
        at = i0 + __ffsll(static_cast<unsigned long long>(hit)) - 1;
        break;
      }
    }
    if (at < 0) break;
    at = __builtin_amdgcn_readfirstlane(at);
    i = at + 1;
    const int tok = l.token[at];
    bool yes;
    if (s.greedy) {
      yes = tok >= 0 && tok == l.best[st.node];
    } else {
      const Scale sc(s.slope, l.top[st.node]);
      const double w = sc.weight(l.x[at]), u = l.u[at];
      if (!drawn) {
        bool gone = tok < 0;                                 // rejected before, or no token at all
        for (int k0 = st.node + 1; k0 < at; k0 += 64) {
          const int k = min(k0 + lane, at - 1);
          gone |= __any(k0 + lane < at && l.parent[k] == st.node && l.token[k] == tok);
        }
        const double own = gone ? 0.0 : w;
        yes = u * st.Z < own;
        if (!yes) st.Z = __builtin_fmax(st.Z - own, 0.0);
      } else {
        const double q = l.q[at], total = l.sum[st.node];
        const double p = total > 0 ? __builtin_fmax(w / total - st.c * q, 0.0) : 0.0;
        yes = tok >= 0 && u * q * st.Z < p;
        if (!yes) {
          st.c += st.Z;
          st.cut = true;
          const double z = rest(st.node, st.c);
          if (!(z == z)) return st;
          st.Z = z;
        }
      }
    }
    if (yes) {
      st.node = at;
      st.c = 0.0;
      st.Z = drawn ? 1.0 : l.sum[at];
      st.cut = false;
      if (write) a.path[s.b * a.ld_path + st.count] = at;
      ++st.count;
    }
  }
  return st;
}

// sum max(p - c q, 0) of up to N logits and shares.
template <int N>
__device__ __forceinline__ double rest_of(const float (&x)[N], const float (&q)[N], const Scale& sc, double inv, double c, int n) {
  double s = 0;
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (k < n) s += __builtin_fmax(sc.weight(logit(x[k])) * inv - c * share(q[k]), 0.0);
  return s;
}

// 1 / S once a row: as p of the walk's tests but for its last bit. (fp64; 0 for a row of nothing)
__device__ __forceinline__ double inverse(double s) { return s > 0 ? 1.0 / s : 0.0; }

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

// The sums of the first row in which a drawn token is rejected: a block a (sequence, chunk).
template <class E, class Q>
__global__ __launch_bounds__(NT) void k_verify_rest(VerifyArgs a) {
  extern __shared__ double lds[];
  __shared__ double sums[NT / 64];
  const int b = blockIdx.x / a.chunks, x = blockIdx.x - b * a.chunks, t = threadIdx.x;
  const Block s = block_of(a, b);
  if (s.n == 0 || s.greedy) return;                          // (uniform)
  const Rows l(reinterpret_cast<char*>(lds), a.rows);
  gather<E, Q>(a, s, l, NT);
  const State st = walk(a, s, l, false, [](int, double) { return static_cast<double>(NAN); });
  if (!st.cut) return;
  const Scale sc(s.slope, l.top[st.node]);
  const double inv = inverse(l.sum[st.node]);
  const E* src = reinterpret_cast<const E*>(a.logits) + (s.first + st.node) * a.ld;
  const Q* from = reinterpret_cast<const Q*>(a.draft) + (s.first + st.node) * a.ld_draft;
  constexpr int N = 4, I = CHUNK / NT / N;
  float f[I][N], q[I][N];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int e = x * CHUNK + (i * NT + t) * N;
    load<E, N>(f[i], src + e, a.V - e);
    load<Q, N>(q[i], from + e, a.V - e);
  }
  double sum = 0;
#pragma unroll
  for (int i = 0; i < I; ++i) sum += rest_of<N>(f[i], q[i], sc, inv, st.c, a.V - (x * CHUNK + (i * NT + t) * N));
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sum += shfl_xor64(sum, m);
  if ((t & 63) == 0) sums[t >> 6] = sum;
  __syncthreads();
  if (t == 0) a.rest[blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// A row's weights, or what is left of it, by elements.
template <class E, class Q>
struct Left {
  const E* src;
  const Q* from;                           // null: weights without the tokens in `gone`
  Scale sc;
  double inv, c;
  const int* gone;
  int n_gone;
  __device__ __forceinline__ void weights(double (&w)[4], int e, int V) const {
    float f[4], q[4];
    load<E, 4>(f, src + e, V - e);
    if (from) load<Q, 4>(q, from + e, V - e);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = e + k < V ? sc.weight(logit(f[k])) : 0.0;
      if (from) w[k] = __builtin_fmax(w[k] * inv - c * (e + k < V ? share(q[k]) : 0.f), 0.0);
    }
    for (int g = 0; g < n_gone; ++g) {
      const int at = gone[g] - e;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at == k) w[k] = 0.0;
    }
  }
};

// All chunks' sums by one block of NW threads, a wave a chunk; returns their total (every thread).
__device__ __forceinline__ double total_of(const double* cs, int chunks) {
  double z = 0;
  for (int x = threadIdx.x & 63; x < chunks; x += 64) z += cs[x];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) z += shfl_xor64(z, m);
  return z;
}

template <class E, class Q>
__device__ double sum_chunks(const Left<E, Q>& left, double* cs, int chunks, int V) {
  const int lane = threadIdx.x & 63;
  __syncthreads();                                           // the last sums were read
  for (int x = threadIdx.x >> 6; x < chunks; x += NW / 64) {
    double s = 0;
    const int end = min(V, (x + 1) * CHUNK);
#pragma unroll 4
    for (int e = x * CHUNK + 4 * lane; e < end; e += 256) {
      double w[4];
      left.weights(w, e, V);
      s += (w[0] + w[1]) + (w[2] + w[3]);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) s += shfl_xor64(s, m);
    if (lane == 0) cs[x] = s;
  }
  __syncthreads();
  return total_of(cs, chunks);
}

// The first token at which the running sum exceeds r times the total, from the chunks' sums; -1: there is none to take.
template <class E, class Q>
__device__ int draw(const Left<E, Q>& left, const double* cs, int chunks, int V, double r, double* scan, int* found) {
  const int t = threadIdx.x, lane = t & 63;
  const double total = total_of(cs, chunks);
  if (!(total > 0)) return -1;                               // (uniform)
  const double want = r * total;
  // the chunk: lane l has chunks 4 l .. 4 l + 3
  double c4[4], own = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    c4[k] = 4 * lane + k < chunks ? cs[4 * lane + k] : 0.0;
    own += c4[k];
  }
  double run = own;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double y = __shfl_up(run, m, 64);
    if (lane >= m) run += y;
  }
  double before = run - own;
  int at = -1, last = -1;
  double base = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (at < 0 && c4[k] > 0 && before + c4[k] > want) {
      at = 4 * lane + k;
      base = before;
    }
    if (c4[k] > 0) last = 4 * lane + k;
    before += c4[k];
  }
  const uint64_t hit = __ballot(at >= 0), some = __ballot(last >= 0);
  int chunk;
  if (hit) {
    const int from = __ffsll(static_cast<unsigned long long>(hit)) - 1;
    chunk = __shfl(at, from, 64);
    base = __shfl(base, from, 64);
  } else {                                                   // r of 1 or more, or a rounding: the last token there is
    chunk = __shfl(last, 63 - __clzll(static_cast<long long>(some)), 64);
    base = -INFINITY;
  }
  // its elements: thread t has 4 side by side
  const int e = chunk * CHUNK + 4 * t;
  double w[4];
  left.weights(w, min(e, V), V);
  own = (w[0] + w[1]) + (w[2] + w[3]);
  run = own;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double y = __shfl_up(run, m, 64);
    if (lane >= m) run += y;
  }
  __syncthreads();                                           // (scan, found of an earlier call)
  if (lane == 63) scan[t >> 6] = run;
  if (t == 0) found[0] = INT32_MAX, found[1] = -1;
  __syncthreads();
  double upto = base;
  for (int x = 0; x < t >> 6; ++x) upto += scan[x];
  upto += run - own;
  int first = INT32_MAX, end = -1;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    upto += w[k];
    if (w[k] > 0) {
      if (first == INT32_MAX && upto > want) first = e + k;
      end = e + k;
    }
  }
  if (first != INT32_MAX) atomicMin(&found[0], first);       // (whole numbers: in any order)
  if (end >= 0) atomicMax(&found[1], end);
  __syncthreads();
  return found[0] != INT32_MAX ? found[0] : found[1];
}

// A block a sequence.
template <class E, class Q>
__global__ __launch_bounds__(NW) void k_verify_walk(VerifyArgs a) {
  extern __shared__ double lds[];
  __shared__ double cs[MAX_CHUNKS], scan[NW / 64];
  __shared__ int found[2], n_gone;
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const Block s = block_of(a, b);
  if (s.n == 0) {                                            // (uniform)
    for (int j = t; j < a.depth; j += NW) a.path[b * a.ld_path + j] = -1;
    if (t == 0) {
      a.count[b] = 0;
      a.next[b] = -1;
    }
    return;
  }
  const Rows l(reinterpret_cast<char*>(lds), a.rows);
  gather<E, Q>(a, s, l, NW);
  const E* logits = reinterpret_cast<const E*>(a.logits) + s.first * a.ld;
  const Q* draft = reinterpret_cast<const Q*>(a.draft) + s.first * a.ld_draft;
  bool ready = a.draft != nullptr;                           // k_verify_rest has the first rejection's sums
  const State st = walk(a, s, l, t == 0, [&](int node, double c) {
    if (ready) {
      ready = false;
      for (int x = t; x < a.chunks; x += NW) cs[x] = a.rest[static_cast<int64_t>(b) * a.chunks + x];
      __syncthreads();
      return total_of(cs, a.chunks);
    }
    return sum_chunks(Left<E, Q>{logits + node * a.ld, draft + node * a.ld_draft, Scale(s.slope, l.top[node]), inverse(l.sum[node]), c,
                                 nullptr, 0}, cs, a.chunks, a.V);
  });
  for (int j = st.count + t; j < a.depth; j += NW) a.path[b * a.ld_path + j] = -1;
  int next = l.best[st.node];
  if (!s.greedy && next >= 0) {
    Left<E, Q> left{logits + st.node * a.ld, st.cut ? draft + st.node * a.ld_draft : nullptr, Scale(s.slope, l.top[st.node]),
                    inverse(l.sum[st.node]), st.c, nullptr, 0};
    if (!st.cut) {
      // the tokens rejected here, each once, in the rows' order; they take the place of the rows' u
      __syncthreads();
      int* gone = reinterpret_cast<int*>(l.u);
      if (t < 64) {
        int m = 0;
        for (int k0 = st.node + 1; a.draft == nullptr && st.count < a.depth && k0 < s.n; k0 += 64) {
          const int k = min(k0 + lane, s.n - 1), tok = l.token[k];
          bool here = k0 + lane < s.n && l.parent[k] == st.node && tok >= 0;
          for (int y = st.node + 1; here && y < k; ++y) here = !(l.parent[y] == st.node && l.token[y] == tok);
          const uint64_t mask = __ballot(here);
          if (here) gone[m + __popcll(mask & ((1ull << lane) - 1))] = tok;
          m += __popcll(mask);
        }
        if (lane == 0) n_gone = m;
      }
      __syncthreads();
      left.gone = gone;
      left.n_gone = n_gone;
      const Part* parts = a.parts + (s.first + st.node) * a.chunks;
      for (int x = t; x < a.chunks; x += NW) {
        double z = parts[x].sum * left.sc.weight(parts[x].top);
        for (int g = 0; g < left.n_gone; ++g)
          if (gone[g] / CHUNK == x) z -= left.sc.weight(logit(load1(left.src + gone[g])));
        cs[x] = __builtin_fmax(z, 0.0);
      }
      __syncthreads();
    }
    int at = draw(left, cs, a.chunks, a.V, a.r ? a.r[b] : 0.f, scan, found);
    if (at < 0 && left.n_gone) {                             // (a chunk's difference that was only rounding)
      sum_chunks(left, cs, a.chunks, a.V);
      at = draw(left, cs, a.chunks, a.V, a.r ? a.r[b] : 0.f, scan, found);
    }
    if (at >= 0) next = at;
  }
  if (t == 0) {
    a.count[b] = st.count;
    a.next[b] = next;
  }
}

int sizes(const char* fn, int64_t T, int64_t V, int n_seq, int64_t max_rows, int* chunks) {
  if (V < 1 || V > static_cast<int64_t>(MAX_CHUNKS) * CHUNK)
    return fail(RF_EUNSUPPORTED, "%s: a vocabulary of %lld (up to %d)", fn, (long long)V, MAX_CHUNKS * CHUNK);
  if (max_rows < 0 || max_rows > MAX_ROWS)
    return fail(RF_EUNSUPPORTED, "%s: %lld rows a sequence (up to %d)", fn, (long long)max_rows, MAX_ROWS);
  *chunks = static_cast<int>((V + CHUNK - 1) / CHUNK);
  if (T < 0 || n_seq < 0 || n_seq > (1 << 20) || T > (INT32_MAX / *chunks) || static_cast<int64_t>(n_seq) * *chunks > INT32_MAX)
    return fail(RF_EINVAL_SHAPE, "%s: %lld rows of %d sequences over a vocabulary of %lld", fn, (long long)T, n_seq, (long long)V);
  return RF_OK;
}

size_t bytes_of(int64_t T, int n_seq, int chunks, bool draft) {
  return static_cast<size_t>(T) * chunks * sizeof(Part) + (draft ? static_cast<size_t>(n_seq) * chunks * sizeof(double) : 0);
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" int rf_verify_drafts_workspace_bytes(int64_t T, int64_t vocab, int n_seq, int64_t max_rows, int draft, size_t* bytes) {
  const char* fn = "rf_verify_drafts_workspace_bytes";
  int chunks;
  if (!bytes) return fail(RF_EINVAL_ARG, "%s: null pointer", fn);
  if (int rc = sizes(fn, T, vocab, n_seq, max_rows, &chunks)) return rc;
  *bytes = n_seq ? bytes_of(T, n_seq, chunks, draft != 0) : 0;
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
  if (T && ws_bytes < bytes_of(T, n_seq, chunks, draft != nullptr))
    return fail(RF_EINVAL_ARG, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, bytes_of(T, n_seq, chunks, draft != nullptr));
  const bool drawn = draft && temperature && T;
  const VerifyArgs a{static_cast<const char*>(logits), ld, T, static_cast<int>(vocab), chunks, tokens, parents, cu, n_seq, u, r,
                     temperature, drawn ? static_cast<const char*>(draft) : nullptr, ld_draft,
                     static_cast<int>(std::min<int64_t>(max_rows, T)), static_cast<int>(depth), path, ld_path, count,
                     next, static_cast<Part*>(workspace),
                     reinterpret_cast<double*>(static_cast<char*>(workspace) + static_cast<size_t>(T) * chunks * sizeof(Part))};
  const size_t shared = static_cast<size_t>(std::max(1, a.rows)) * ROW_BYTES;
#define RF_VERIFY(E, Q)                                                                                                       \
  do {                                                                                                                        \
    if (T) hipLaunchKernelGGL((k_verify_rows<E>), dim3(static_cast<unsigned>(T * chunks)), dim3(NT), 0, stream, a);           \
    if (drawn) hipLaunchKernelGGL((k_verify_rest<E, Q>), dim3(static_cast<unsigned>(n_seq * chunks)), dim3(NT), shared, stream, a); \
    hipLaunchKernelGGL((k_verify_walk<E, Q>), dim3(static_cast<unsigned>(n_seq)), dim3(NW), shared, stream, a);               \
  } while (0)
  if (logits_kind == RF_F32) {
    if (!drawn || draft_kind == RF_F32) RF_VERIFY(float, float);
    else RF_VERIFY(float, uint16_t);
  } else {
    if (!drawn || draft_kind == RF_F32) RF_VERIFY(uint16_t, float);
    else RF_VERIFY(uint16_t, uint16_t);
  }
#undef RF_VERIFY
  return check_launch(fn);
}
