// One token per row of logits from one given number per row, with a temperature, top-k, min-p and top-p of the row's own.
//
// Order the tokens by logit descending, then by index ascending, with weights w_i = exp((x_i - max) / T). Keep the first k;
// of these the ones with w >= min_p; of these the ones in front of which less than top_p of their whole weight stands (the
// first always). The token is the one on whose stretch of the kept weight u falls. T <= 0 takes the largest logit, lowest
// index first. The log-probability is that of the kept, renormalised distribution.
//
// No row is sorted. A token's weight depends on its value alone, so everything above is a search in the histogram of the
// row's values: counts per value, weights per value in 64 bits, prefix sums over values. Where 150,000 weights are summed in
// 32 bits, u falls on the wrong side of a border of two tokens often enough to be seen; here a bf16 row's sums are good to
// 2^-45 of themselves (what the weights' series is), an fp32 row's to 2^-34 of the largest weight and 2^-45 of themselves.
// Only values within kWindow T of the maximum count: what lies below weighs less than 2^-41 of the row together, 2^-17 of
// the distance between two neighbouring numbers u.
//
// bf16 rows (sample_bf16_kernel): 16 binades of values below the largest magnitude are 4096 counters in shared memory, one
// atomic a token. Values closer to zero (a thousandth of a row) share one more, whose weight is summed apart; a row whose
// search ends there is marked and left to the second kernel. fp32 rows and marked ones (sample_any_kernel): 2048 equal
// steps below the maximum with counts and weights, then the step in question digit by digit.
//
// A row is read for the histogram and for the token's place, the second time from L2 or shared memory. Measured: one bf16 row of
// 151936 19 us, 67 rows of 128256 27 us, of which 17 are the latency of their steps; 512 rows of 151936 106 us: a turn of 296 rows
// takes 50 us, 27 of them reading and counting (a warp's 32 atomics 1.5 ns, 14 us in all, beside 14 of reading), 9 looking for
// the token, and the rest the look ahead, sums in 64 bits and waiting on each other. 24 fp32 rows of 248320 with 3 % of the
// tokens left 49 us, 256 full ones of 151936 299 us: there every token's weight is computed in 64 bits (6 ns for a warp's), by a
// kernel that spills (two CTAs a multiprocessor hold it to 64 registers).
#include "bw_common.cuh"
#include "host_util.h"

#include <cfloat>

#include <cooperative_groups.h>

namespace {
using namespace bw;
namespace cg = cooperative_groups;

constexpr float kWindow = 42.f;       // e^-42 * 2^19 tokens < 2^-41
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;

struct Args {
  const void* logits;
  long long ld;
  int V;
  const float* u;
  const float* temperature;           // each may be null: 1, off, off, off
  const int* top_k;
  const float* top_p;
  const float* min_p;
  long long* tokens;
  float* logprobs;
  int* marked;                        // rows the first kernel leaves to the second (null: all rows are the second's)
  int cached;                         // a CTA's pieces stay in shared memory after the first pass
  int kept;                           // room for them, in pieces
};

template <typename T>
__device__ __forceinline__ float value_of(T x);
template <>
__device__ __forceinline__ float value_of<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float value_of<float>(float x) { return x; }

// A CTA's share of a row: 16-byte pieces [lo, hi) behind an unaligned head (rank 0) and before a tail (the last rank).
extern __shared__ __align__(16) uint4 kept_pieces[];
template <typename T>
struct Share {
  static constexpr int kPer = 16 / sizeof(T);
  const T* row;
  const uint4* vec;
  int head, lo, hi, tail0, tail1;
  int first;                          // index of the first element of piece 0
  bool cached;
  __device__ __forceinline__ Share(const Args& a, int r, int rank, int c) {
    row = static_cast<const T*>(a.logits) + static_cast<long long>(r) * a.ld;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T));
    first = head = min(a.V, off ? kPer - off : 0);
    vec = reinterpret_cast<const uint4*>(row + head);
    const int n = (a.V - head) / kPer;
    lo = static_cast<int>(static_cast<long long>(n) * rank / c), hi = static_cast<int>(static_cast<long long>(n) * (rank + 1) / c);
    tail0 = head + n * kPer, tail1 = rank == c - 1 ? a.V : tail0;
    if (rank != 0) head = 0;
    cached = a.cached;
  }
  // f(element) for what is not in whole pieces
  template <typename F>
  __device__ __forceinline__ void edges(F&& f) const {
    if (static_cast<int>(threadIdx.x) < head) f(row[threadIdx.x]);
    if (tail0 + static_cast<int>(threadIdx.x) < tail1) f(row[tail0 + threadIdx.x]);
  }
  // f(piece) for every piece, in no particular order; FILL: the first pass, which leaves them in shared memory
  template <bool FILL, typename F>
  __device__ __forceinline__ void pieces(F&& f) const {
    int i = lo + threadIdx.x;
    if (!FILL && cached) {
      for (; i < hi; i += kThreads) f(kept_pieces[i - lo]);
      return;
    }
    for (; i + 3 * kThreads < hi; i += 4 * kThreads) {
      uint4 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = vec[i + q * kThreads];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (FILL && cached) kept_pieces[i + q * kThreads - lo] = w[q];
        f(w[q]);
      }
    }
    uint4 w[3];
#pragma unroll
    for (int q = 0; q < 3; ++q)
      if (i + q * kThreads < hi) w[q] = vec[i + q * kThreads];
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      if (i + q * kThreads < hi) {
        if (FILL && cached) kept_pieces[i + q * kThreads - lo] = w[q];
        f(w[q]);
      }
    }
  }
  __device__ __forceinline__ uint4 piece(int i) const { return cached ? kept_pieces[i - lo] : vec[i]; }
  // f(value) for every element
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    edges([&](T x) { f(value_of<T>(x)); });
    pieces<false>([&](const uint4& w) {
      const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int q = 0; q < kPer; ++q) f(value_of<T>(x[q]));
    });
  }
  // bit q: element q of the piece equals `value`
  __device__ __forceinline__ unsigned equal(const uint4& w, float value) const {
    unsigned m = 0;
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 v = __float2bfloat162_rn(value);
      const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&w);
      const unsigned e0 = __heq2_mask(x[0], v), e1 = __heq2_mask(x[1], v), e2 = __heq2_mask(x[2], v), e3 = __heq2_mask(x[3], v);
      if (e0 | e1 | e2 | e3) m = (e0 & 1u) | (e0 >> 16 & 1u) << 1 | (e1 & 1u) << 2 | (e1 >> 16 & 1u) << 3 | (e2 & 1u) << 4 | (e2 >> 16 & 1u) << 5 | (e3 & 1u) << 6 | (e3 >> 16 & 1u) << 7;
    } else {
      const float* x = reinterpret_cast<const float*>(&w);
#pragma unroll
      for (int q = 0; q < kPer; ++q) m |= (x[q] == value ? 1u : 0u) << q;
    }
    return m;
  }
};

template <typename T, typename Op>
__device__ __forceinline__ T warp_all(T v, Op op) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
using u64 = unsigned long long;
struct Add {
  template <typename T>
  __device__ T operator()(T a, T b) const { return a + b; }
};

// exclusive prefix over the block of a pair, in a fixed order; all[0..1] the totals
template <typename A, typename B>
__device__ __forceinline__ void block_prefix(A& x, B& y, A* sx, B* sy, A& all_x, B& all_y) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  A ix = x;
  B iy = y;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const A ox = __shfl_up_sync(0xffffffffu, ix, d);
    const B oy = __shfl_up_sync(0xffffffffu, iy, d);
    if (lane >= d) ix += ox, iy += oy;
  }
  if (lane == 31) sx[warp] = ix, sy[warp] = iy;
  __syncthreads();
  A bx = 0;
  B by = 0;
  all_x = 0, all_y = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) bx = all_x, by = all_y;
    all_x += sx[w], all_y += sy[w];
  }
  ix = __shfl_up_sync(0xffffffffu, ix, 1), iy = __shfl_up_sync(0xffffffffu, iy, 1);
  x = bx + (lane ? ix : A(0)), y = by + (lane ? iy : B(0));
  __syncthreads();
}

struct Row {                          // what a row asks for
  double T, top_p, min_p, u;
  int k;
  bool greedy;
  __device__ __forceinline__ Row(const Args& a, int r) {
    const float t = a.temperature ? a.temperature[r] : 1.f;
    greedy = !(t > 0.f);
    T = t;
    k = a.top_k ? a.top_k[r] : 0;
    if (k <= 0 || k > a.V) k = a.V;
    const float p = a.top_p ? a.top_p[r] : 1.f, m = a.min_p ? a.min_p[r] : 0.f;
    top_p = p < 1.f ? static_cast<double>(p) : 2.0;     // 2: off (so is what is not a number)
    min_p = m > 0.f ? static_cast<double>(m) : 0.0;
    const float v = a.u[r];
    u = v > 0.f ? fminf(v, 0.99999994f) : 0.f;          // the numbers are of [0, 1): what is not, or is no number, is moved there
  }
};

__device__ __forceinline__ double weight(float x, float top, double T) { return x == top ? 1.0 : exp((static_cast<double>(x) - static_cast<double>(top)) / T); }

// 2^-t for t > -1/64: 2^-(n / 64) from a table, the rest by its series, six terms (Tang, "Table-driven implementation of the
// exponential function in IEEE floating-point arithmetic", 1989); a third of exp's work in 64 bits, good to 2e-14 (t itself is
// rounded to 2^-47)
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = exp2(threadIdx.x * (-1.0 / 64.0));
}
__device__ __forceinline__ double two_to_minus(double t, const double* table) {
  if (!(t < 900.0)) return 0.0;
  const int n = static_cast<int>(t * 64.0);
  const double f = (t - n * (1.0 / 64.0)) * -0.69314718055994530942;
  const double e = 1.0 + f * (1.0 + f * (1.0 / 2 + f * (1.0 / 6 + f * (1.0 / 24 + f * (1.0 / 120)))));
  return e * __longlong_as_double(__double_as_longlong(table[n & 63]) - (static_cast<long long>(n >> 6) << 52));
}

struct Shared {                       // of one CTA; rank 0's copy is the cluster's
  float top[kWarps], low[kWarps];
  float cta_top, cta_low;
  double sd[kWarps];
  u64 su[kWarps];
  unsigned sc[kWarps];
  u64 cta_mass;
  unsigned cta_count, cta_zero, cta_match;
  // outcome
  float value;
  unsigned nth, ties;
  int state;                          // 1: the nth token of this value, 0: no token left, -1: marked
  // the search's steps
  double f0, f1;
  unsigned c0, c1, i0;
  // what place() finds
  unsigned found_n, found_min;
};

// The threads' largest and smallest values over the cluster.
__device__ __forceinline__ void over_cluster(float hi, float lo, Shared& sh, int c, float& top, float& low) {
  hi = warp_all(hi, [](float a, float b) { return fmaxf(a, b); });
  lo = warp_all(lo, [](float a, float b) { return fminf(a, b); });
  if ((threadIdx.x & 31) == 0) sh.top[threadIdx.x >> 5] = hi, sh.low[threadIdx.x >> 5] = lo;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) hi = fmaxf(hi, sh.top[w]), lo = fminf(lo, sh.low[w]);
  if (c > 1) {
    if (threadIdx.x == 0) sh.cta_top = hi, sh.cta_low = lo;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
#pragma unroll
    for (int q = 0; q < kMaxCluster; ++q) {
      if (q < c) {
        const Shared* o = cl.map_shared_rank(&sh, q);
        hi = fmaxf(hi, o->cta_top), lo = fminf(lo, o->cta_low);
      }
    }
  }
  top = hi, low = lo;
}

// The row's largest value and its smallest one, over the cluster, without NaN; fills the kept pieces.
template <typename T>
__device__ __forceinline__ void extremes(const Share<T>& s, Shared& sh, int c, float& top, float& low) {
  float hi = -INFINITY, lo = INFINITY;
  s.edges([&](T x) { hi = fmaxf(hi, value_of<T>(x)), lo = fminf(lo, value_of<T>(x)); });
  if constexpr (sizeof(T) == 2) {                       // two values an instruction; the number wins over NaN
    __nv_bfloat162 h = __float2bfloat162_rn(-INFINITY), l = __float2bfloat162_rn(INFINITY);
    s.template pieces<true>([&](const uint4& w) {
      const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
      for (int q = 0; q < 4; ++q) h = __hmax2(h, x[q]), l = __hmin2(l, x[q]);
    });
    hi = fmaxf(hi, fmaxf(__low2float(h), __high2float(h))), lo = fminf(lo, fminf(__low2float(l), __high2float(l)));
  } else {
    s.template pieces<true>([&](const uint4& w) {
      const float* x = reinterpret_cast<const float*>(&w);
#pragma unroll
      for (int q = 0; q < 4; ++q) hi = fmaxf(hi, x[q]), lo = fminf(lo, x[q]);
    });
  }
  over_cluster(hi, lo, sh, c, top, low);
}

// Index of the nth (from 0) element that equals `value`, for any number of them: warps own neighbouring pieces, so counts in
// order of warp and rank are counts in order of index. Out of line: rows with that many equal values are rare.
template <typename T>
__device__ __noinline__ void place_among_many(const Share<T>& s, Shared& sh, const Args& a, int r, int c, int rank, float value, unsigned nth) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = s.hi - s.lo;
  const int w0 = s.lo + static_cast<int>(static_cast<long long>(n) * warp / kWarps), w1 = s.lo + static_cast<int>(static_cast<long long>(n) * (warp + 1) / kWarps);
  auto matches = [&](int i) { return s.equal(s.piece(i), value); };
  unsigned mine = 0;
  if (s.cached) {
    for (int i = w0 + lane; i < w1; i += 32) mine += __popc(s.equal(kept_pieces[i - s.lo], value));
  } else {
    int i = w0 + lane;
    for (; i + 7 * 32 < w1; i += 8 * 32) {
      uint4 w[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) w[q] = s.vec[i + q * 32];
#pragma unroll
      for (int q = 0; q < 8; ++q) mine += __popc(s.equal(w[q], value));
    }
    for (; i < w1; i += 32) mine += __popc(s.equal(s.vec[i], value));
  }
  const bool is_head = warp == 0 && lane < s.head, is_tail = warp == kWarps - 1 && s.tail0 + lane < s.tail1;
  const unsigned mh = __ballot_sync(0xffffffffu, is_head && value_of<T>(s.row[is_head ? lane : 0]) == value);
  const unsigned mt = __ballot_sync(0xffffffffu, is_tail && value_of<T>(s.row[is_tail ? s.tail0 + lane : 0]) == value);
  mine = warp_all(mine, Add());
  if (lane == 0) sh.sc[warp] = mine + __popc(mh) + __popc(mt);
  __syncthreads();
  unsigned before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before = all;
    all += sh.sc[w];
  }
  if (c > 1) {
    if (threadIdx.x == 0) sh.cta_match = all;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    unsigned v[kMaxCluster];
#pragma unroll
    for (int q = 0; q < kMaxCluster; ++q)
      if (q < rank) v[q] = cl.map_shared_rank(&sh, q)->cta_match;
#pragma unroll
    for (int q = 0; q < kMaxCluster; ++q)
      if (q < rank) before += v[q];
    cl.sync();                        // nobody reaches into a peer after this
  }
  const unsigned here = mine + __popc(mh) + __popc(mt);
  if (nth < before || nth >= before + here) return;
  unsigned left = nth - before;       // of this warp's matches
  auto nth_bit = [](unsigned m, unsigned k) {
    for (; k; --k) m &= m - 1;
    return __ffs(m) - 1;
  };
  int found = -1;
  if (left < __popc(mh)) {
    found = nth_bit(mh, left);
  } else {
    left -= __popc(mh);
    for (int i0 = w0; i0 < w1 && found < 0; i0 += 8 * 32) {
      unsigned m[8], all8 = 0;        // 8 x 32 pieces at a time: one wait for all of them
#pragma unroll
      for (int q = 0; q < 8; ++q) m[q] = i0 + q * 32 + lane < w1 ? matches(i0 + q * 32 + lane) : 0u;
#pragma unroll
      for (int q = 0; q < 8; ++q) all8 += __popc(m[q]);
      all8 = warp_all(all8, Add());
      if (left >= all8) {
        left -= all8;
        continue;
      }
      unsigned mine8 = 0;             // the eighth that has it
      int eighth = 0;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const unsigned whole = warp_all(static_cast<unsigned>(__popc(m[q])), Add());
        if (eighth == q) {
          mine8 = m[q];
          if (left >= whole) left -= whole, ++eighth;
        }
      }
      unsigned upto = __popc(mine8);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
      }
      const unsigned front = upto - __popc(mine8);
      const bool me = left >= front && left < upto;
      const int at = me ? s.first + (i0 + eighth * 32 + lane) * Share<T>::kPer + nth_bit(mine8, left - front) : 0;
      const unsigned who = __ballot_sync(0xffffffffu, me);
      found = __shfl_sync(0xffffffffu, at, __ffs(who) - 1);
    }
    if (found < 0) found = s.tail0 + nth_bit(mt, left);
  }
  if (lane == 0) a.tokens[r] = found;
}

// Writes the row's outcome: the index of the nth (from 0) of `ties` elements that equal `value`, and the log-probability
// (value - top) / T - log(kept), with per = log2(e) / T. The first is a minimum over the cluster; of a few, the indices are
// collected in rank 0's `list` (kTies places) and each looks how many stand in front of it.
constexpr unsigned kTies = 1024;
template <typename T>
__device__ __forceinline__ void place(const Share<T>& s, Shared& sh, const Args& a, int r, int c, int rank, float value, unsigned nth, unsigned ties,
                                      unsigned* list, float top, double per, double kept, const double* table) {
  const auto outcome = [&]() {
    // log(kept) = y + log(kept e^-y) with y the logarithm in 32 bits: the second one is its argument less 1
    const double y = logf(static_cast<float>(kept));
    const double fine = kept * two_to_minus(y * 1.4426950408889634, table) - 1.0;
    const double distance = value == top ? 0.0 : (static_cast<double>(top) - static_cast<double>(value)) * per * 0.69314718055994530942;
    a.logprobs[r] = static_cast<float>(-distance - (y + fine));
  };
  if (nth > 0 && ties > kTies) {
    if (rank == 0 && threadIdx.x == kThreads - 1) outcome();
    place_among_many(s, sh, a, r, c, rank, value, nth);
    return;
  }
  cg::cluster_group cl = cg::this_cluster();
  unsigned* const lead_n = c > 1 ? cl.map_shared_rank(&sh.found_n, 0) : &sh.found_n;
  unsigned* const lead_min = c > 1 ? cl.map_shared_rank(&sh.found_min, 0) : &sh.found_min;
  unsigned* const lead_list = c > 1 ? cl.map_shared_rank(list, 0) : list;
  unsigned least = 0xffffffffu;
  const auto hit = [&](unsigned at) {
    if (nth == 0) least = min(least, at);
    else lead_list[atomicAdd(lead_n, 1u)] = at;
  };
  if (static_cast<int>(threadIdx.x) < s.head && value_of<T>(s.row[threadIdx.x]) == value) hit(threadIdx.x);
  if (s.tail0 + static_cast<int>(threadIdx.x) < s.tail1 && value_of<T>(s.row[s.tail0 + threadIdx.x]) == value) hit(s.tail0 + threadIdx.x);
  const auto look = [&](const uint4& w, int i) {
    for (unsigned m = s.equal(w, value); m; m &= m - 1) hit(s.first + i * Share<T>::kPer + __ffs(m) - 1);
  };
  int i = s.lo + threadIdx.x;
  if (s.cached) {
    for (; i < s.hi; i += kThreads) look(kept_pieces[i - s.lo], i);
  } else {
    for (; i + 3 * kThreads < s.hi; i += 4 * kThreads) {
      uint4 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = s.vec[i + q * kThreads];
#pragma unroll
      for (int q = 0; q < 4; ++q) look(w[q], i + q * kThreads);
    }
    for (; i < s.hi; i += kThreads) look(s.vec[i], i);
  }
  if (nth == 0) {
    least = warp_all(least, [](unsigned x, unsigned y) { return min(x, y); });
    if ((threadIdx.x & 31) == 0 && least != 0xffffffffu) atomicMin(lead_min, least);
  }
  if (c > 1) cl.sync();               // the last time that anybody reaches into a peer
  else __syncthreads();
  if (rank != 0) return;
  if (threadIdx.x == kThreads - 1) outcome();
  if (nth == 0) {
    if (threadIdx.x == 0) a.tokens[r] = sh.found_min;
    return;
  }
  for (unsigned t = threadIdx.x; t < ties; t += kThreads) {
    const unsigned at = list[t];
    unsigned front = 0;
    for (unsigned j = 0; j < ties; ++j) front += list[j] < at;
    if (front == nth) a.tokens[r] = at;
  }
}

// ------------------------------------------------------------------------------------------------ bf16
constexpr int kBinades = 16, kHalf = kBinades * 128;                           // what a row is searched in
constexpr int kRoom = (kBinades + 1) * 128, kBins = 2 * kRoom + 1;             // negative values | around zero | positive ones
constexpr int kEach = 2 * kHalf / kThreads;                                    // bins a thread searches
static_assert(kEach * kThreads == 2 * kHalf, "bins are shared out evenly; the middle one goes to a thread of its own place");

__global__ void __launch_bounds__(kThreads, 2) sample_bf16_kernel(const __grid_constant__ Args a) {
  __shared__ unsigned bins[kBins + 3];
  __shared__ double table[64];
  __shared__ Shared sh;
  const int c = gridDim.x, rank = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  pdl_launch_dependents();
  const Share<__nv_bfloat16> s(a, r, rank, c);
  const Row row(a, r);
  for (int i = tid; i < kBins; i += kThreads) bins[i] = 0u;
  fill_table(table);
  if (tid == 0) sh.found_n = 0u, sh.found_min = 0xffffffffu;
  // The bins are the 16 binades from the widest magnitude of the window down: a function of the row, so that its sums are. A
  // row's first 4096 tokens suggest them, and one pass finds the extremes and counts, in a binade more, of which either
  // end may be the one too many; where the row then says otherwise, it is counted again.
  const auto mag = [](float x) { return static_cast<int>((__float_as_uint(x) >> 16) & 0x7fffu); };   // compared as integers
  const double per = 1.4426950408889634 / row.T;
  int base, first;                    // magnitudes: the lowest binade's first, and the first that has a bin
  unsigned some;                      // how many have one
  unsigned *up, *downward;            // bins of distance 0 from `first`, and one past the first negative one (-d is ~d + 1)
  const auto lay_out = [&](int widest, int binades) {
    base = max(0, (widest - (binades - 1)) << 7), first = max(1, base);
    some = binades * 128 + base - first;
    up = bins + kRoom + 1 + (first - base), downward = bins + kRoom - (first - base);
  };
  unsigned zeros = 0, tiny = 0;       // tokens that are zero, or closer to it than the bins reach
  u64 tiny_mass = 0;                  // weight of the latter, relative to that of a zero, in 2^-44
  const auto around_zero = [&](unsigned bits, unsigned n) {
    if (bits & 0x7fffu) {
      // where zero is in the window, T is at least a 42nd of the widest magnitude, and this is next to 1; elsewhere it counts for nothing
      const double t = static_cast<double>(__uint_as_float(bits << 16)) * -per;
      tiny += n;
      if (fabs(t) < 1.0 / 64.0) tiny_mass += n * static_cast<u64>(two_to_minus(t, table) * 17592186044416.0 + 0.5);
    } else {
      zeros += n;
    }
  };
  const auto add = [&](unsigned bits, unsigned n) {
    const int d = static_cast<int>(bits & 0x7fffu) - first;
    const int sign = -static_cast<int>(bits >> 15 & 1u);
    if (static_cast<unsigned>(d) < some) atomicAdd((sign ? downward : up) + (d ^ sign), n);
    return d;
  };
  const auto count_edges = [&]() {
    s.edges([&](__nv_bfloat16 x) {
      const unsigned bits = __bfloat16_as_ushort(x);
      if (add(bits, 1u) < 0) around_zero(bits, 1u);
    });
  };
  const auto count = [&](const uint4& w) {
    if (w.x == w.y && w.z == w.w && w.x == w.z && (w.x >> 16) == (w.x & 0xffffu)) {          // a mask's run: one atomic, not eight
      if (add(w.x & 0xffffu, 8u) < 0) around_zero(w.x & 0xffffu, 8u);
      return;
    }
    int below = add(w.x & 0xffffu, 1u) | add(w.x >> 16, 1u) | add(w.y & 0xffffu, 1u) | add(w.y >> 16, 1u);
    below |= add(w.z & 0xffffu, 1u) | add(w.z >> 16, 1u) | add(w.w & 0xffffu, 1u) | add(w.w >> 16, 1u);
    if (below < 0) {
#pragma unroll 1
      for (int q = 0; q < 8; ++q) {
        const unsigned word = q < 4 ? (q < 2 ? w.x : w.y) : (q < 6 ? w.z : w.w), bits = q & 1 ? word >> 16 : word & 0xffffu;
        if (static_cast<int>(bits & 0x7fffu) < first) around_zero(bits, 1u);
      }
    }
  };
  float top, low;
  int guess = -1;
  if (!row.greedy && !s.cached) {                       // (a second pass over shared memory is no more than the look ahead)
    __nv_bfloat162 h = __float2bfloat162_rn(-INFINITY), l = __float2bfloat162_rn(INFINITY);
    if (tid < (a.V - s.first) / 8) {
      const uint4 w = s.vec[tid];
      const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
      for (int q = 0; q < 4; ++q) h = __hmax2(h, x[q]), l = __hmin2(l, x[q]);
    }
    const float hi = warp_all(fmaxf(__low2float(h), __high2float(h)), [](float x, float y) { return fmaxf(x, y); });
    const float lo = warp_all(fminf(__low2float(l), __high2float(l)), [](float x, float y) { return fminf(x, y); });
    if ((tid & 31) == 0) sh.top[tid >> 5] = hi, sh.low[tid >> 5] = lo;
    __syncthreads();                                    // (the bins are zero, too)
    top = -INFINITY, low = INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh.top[w]), low = fminf(low, sh.low[w]);
    __syncthreads();
    low = fmaxf(low, top - kWindow * static_cast<float>(row.T));
    if (top > -INFINITY && top < INFINITY) guess = min(254, (max(mag(top), mag(low)) >> 7) + 1);
  }
  if (guess >= 0) {
    lay_out(guess, kBinades + 1);
    float hi = -INFINITY, lo = INFINITY;
    count_edges();
    s.edges([&](__nv_bfloat16 x) { hi = fmaxf(hi, __bfloat162float(x)), lo = fminf(lo, __bfloat162float(x)); });
    __nv_bfloat162 h = __float2bfloat162_rn(-INFINITY), l = __float2bfloat162_rn(INFINITY);
    s.pieces<true>([&](const uint4& w) {
      const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
      for (int q = 0; q < 4; ++q) h = __hmax2(h, x[q]), l = __hmin2(l, x[q]);
      count(w);
    });
    hi = fmaxf(hi, fmaxf(__low2float(h), __high2float(h))), lo = fminf(lo, fminf(__low2float(l), __high2float(l)));
    over_cluster(hi, lo, sh, c, top, low);
  } else {
    extremes(s, sh, c, top, low);
  }
  cg::cluster_group cl = cg::this_cluster();
  if (top == -INFINITY || row.greedy) {                 // the same for the whole cluster
    if (c > 1) cl.sync();                               // peers have read this CTA's extremes
    if (top == -INFINITY) {
      if (rank == 0 && tid == 0) a.tokens[r] = 0, a.logprobs[r] = -INFINITY, a.marked[r] = 0;
      return;
    }
    if (rank == 0 && tid == 0) a.marked[r] = 0;
    place(s, sh, a, r, c, rank, top, 0u, 1u, bins, top, 1.0, 1.0, table);
    return;
  }
  low = fmaxf(low, top - kWindow * static_cast<float>(row.T));
  // What is larger than the widest magnitude is negative and below the window, or no number; where the widest is infinite the
  // row is marked
  const int widest = max(mag(top), mag(low)) >> 7;
  const auto weigh_value = [&](float x) { return x == top ? 1.0 : two_to_minus((static_cast<double>(top) - static_cast<double>(x)) * per, table); };
  int shift = 0;                                        // magnitudes with bins below the lowest of the 16 binades
  if (widest == guess || widest + 1 == guess) {
    const int low_base = base;
    base = max(0, (widest - (kBinades - 1)) << 7), shift = base - low_base;
    const int i = tid & 127;                            // their tokens belong to what is around zero
    if (tid < 256 && i < shift) {
      const unsigned bits = static_cast<unsigned>(low_base + i) | (tid >> 7) << 15, n = bins[tid >> 7 ? kRoom - 1 - i : kRoom + 1 + i];
      if (n) around_zero(bits, n);
    }
  } else {
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) bins[i] = 0u;
    __syncthreads();
    zeros = 0, tiny = 0, tiny_mass = 0;
    lay_out(widest, kBinades);
    count_edges();
    s.pieces<false>(count);
  }
  // what lies around zero, summed over the CTA
  zeros = warp_all(zeros, Add()), tiny = warp_all(tiny, Add()), tiny_mass = warp_all(tiny_mass, Add());
  __shared__ unsigned s_zero[kWarps], s_tiny[kWarps];
  if ((tid & 31) == 0) s_zero[tid >> 5] = zeros, s_tiny[tid >> 5] = tiny, sh.su[tid >> 5] = tiny_mass;
  __syncthreads();
  if (tid == 0) {
    unsigned z = 0, t = 0;
    u64 m = 0;
    for (int w = 0; w < kWarps; ++w) z += s_zero[w], t += s_tiny[w], m += sh.su[w];
    sh.cta_zero = z, sh.cta_count = t, sh.cta_mass = m;
  }
  if (c > 1) {
    cl.sync();
    // each CTA adds up its share of the bins and puts it into rank 0's
    unsigned* lead_bins = cl.map_shared_rank(bins, 0);
    const int from = kRoom - kHalf - shift, all = 2 * (kHalf + shift) + 1;
    for (int i = from + all * rank / c + tid; i < from + all * (rank + 1) / c; i += kThreads) {
      unsigned v[kMaxCluster], sum = 0;
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q)
        if (q < c) v[q] = *cl.map_shared_rank(bins + i, q);
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q)
        if (q < c) sum += v[q];
      lead_bins[i] = sum;
    }
    cl.sync();
  } else {
    __syncthreads();
  }

  if (rank == 0) {
    // bins in descending order of value: thread t has places kEach t .. of the 2 kHalf bins of their own; the middle one
    // stands in front of the first negative bin, at a thread's edge
    unsigned n[kEach];
    double w[kEach];
    unsigned zc = 0, tc = 0;
    u64 tm = 0;
    {
      unsigned vz[kMaxCluster], vt[kMaxCluster];
      u64 vm[kMaxCluster];
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) {
        if (q < c) {
          const Shared* o = cl.map_shared_rank(&sh, q);
          vz[q] = o->cta_zero, vt[q] = o->cta_count, vm[q] = o->cta_mass;
        }
      }
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q)
        if (q < c) zc += vz[q], tc += vt[q], tm += vm[q];
    }
    const unsigned mid = zc + tc;
    const double mid_mass = mid ? (static_cast<double>(tm) * (1.0 / 17592186044416.0) + zc) * two_to_minus(static_cast<double>(top) * per, table) : 0.0;
    const int place0 = tid * kEach;
    const bool after_mid = place0 == kHalf;
    const auto value_at = [&](int j) {
      const int at = place0 + j;
      return at < kHalf ? __uint_as_float(static_cast<unsigned>(base + kHalf - 1 - at) << 16)
                        : __uint_as_float((0x8000u | static_cast<unsigned>(base + at - kHalf)) << 16);
    };
    unsigned count = after_mid ? mid : 0u, any = 0u;
    double mass = after_mid ? mid_mass : 0.0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int at = place0 + j;
      n[j] = bins[at < kHalf ? kRoom + shift + kHalf - at : kRoom - shift + kHalf - 1 - at];
      any |= n[j];
    }
    // the thread's values are equally spaced (a binade has 128), so their weights are a geometric series
    {
      const float v0 = value_at(0);
      const int e = max(1, static_cast<int>((__float_as_uint(v0) >> 23) & 255u));
      const double ratio = any ? two_to_minus(__longlong_as_double(static_cast<long long>(e - 134 + 1023) << 52) * per, table) : 0.0;
      double run = any && v0 <= top ? weigh_value(v0) : 0.0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (j) run = value_at(j) == top ? 1.0 : run * ratio;
        w[j] = n[j] ? run : 0.0;
        count += n[j], mass += n[j] * w[j];
      }
    }
    unsigned c_all;
    double m_all;
    block_prefix(count, mass, sh.sc, sh.sd, c_all, m_all);
    // now (count, mass): what stands before this thread's stretch, the middle included in front of the thread that has it.
    // Each search ends in a number of tokens (the largest that any bin gives), and the bin that this number ends in says
    // the weight: whole numbers, so that no rounding of a prefix leaves a search without an end, or with two
    const unsigned c_mid = count;
    const double m_mid = mass;
    if (after_mid) count += mid, mass += mid_mass;
    __shared__ int s_marked;
    if (tid == 0) s_marked = 0, sh.c0 = 0u, sh.c1 = 1u, sh.f0 = m_all, sh.nth = 0u;
    __syncthreads();
    const auto weigh = [&](unsigned upto) {             // sh.f0 = weight of the first `upto` tokens
      unsigned cc = count;
      double mm = mass;
      if (after_mid && mid && upto == c_mid + mid) sh.f0 = m_mid + mid_mass;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (upto > cc && upto <= cc + n[j]) sh.f0 = mm + (upto - cc) * w[j];
        cc += n[j], mm += n[j] * w[j];
      }
      __syncthreads();
      return sh.f0;
    };

    // how many tokens are kept by k and min_p, and their weight
    unsigned keep = min(static_cast<unsigned>(row.k), c_all);
    if (row.min_p > 0.0) {                              // tokens with w >= min_p are a prefix of the order
      unsigned some = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) some += n[j] && w[j] >= row.min_p ? n[j] : 0u;
      if (after_mid && mid) {
        const float edge = __uint_as_float(static_cast<unsigned>(max(1, base)) << 16);
        if (weigh_value(-edge) >= row.min_p) some += mid;
        else if ((edge >= top || weigh_value(edge) >= row.min_p) && keep > c_mid) s_marked = 1;
      }
      some = warp_all(some, Add());
      if ((tid & 31) == 0) atomicAdd(&sh.c0, some);
      __syncthreads();
      keep = max(1u, min(keep, sh.c0));
    }
    if (after_mid && keep > c_mid && keep < c_mid + mid) s_marked = 1;
    const double total = keep < c_all ? weigh(keep) : m_all;
    // top-p: tokens in front of which less than top_p of the total stands, the first always
    unsigned last = keep;
    double kept = total;
    if (row.top_p < 1.0) {
      const double limit = row.top_p * total;
      unsigned cc = count, upto = 1u;
      double mm = mass;
      if (after_mid && mid && keep > c_mid && m_mid < limit) {
        if (m_mid + mid_mass < limit && keep >= c_mid + mid) upto = max(upto, c_mid + mid);
        else s_marked = 1;
      }
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const unsigned have = keep > cc ? min(n[j], keep - cc) : 0u;
        if (have && mm < limit) {
          const bool through = mm + have * w[j] < limit;
          upto = max(upto, cc + (through ? have : static_cast<unsigned>(fmin(static_cast<double>(have), fmax(ceil((limit - mm) / w[j]), 1.0)))));
        }
        cc += n[j], mm += n[j] * w[j];
      }
      upto = warp_all(upto, [](unsigned x, unsigned y) { return max(x, y); });
      if ((tid & 31) == 0) atomicMax(&sh.c1, upto);
      __syncthreads();
      last = sh.c1;
      kept = weigh(last);
    }
    // the token: as many stand in front of it as end at or before u of the kept weight
    {
      if (tid == 0) sh.f1 = kept;
      const double target = row.u * kept;
      unsigned cc = count, before = 0u;
      double mm = mass;
      if (after_mid && mid && last > c_mid && target >= m_mid) {
        if (target >= m_mid + mid_mass) before = c_mid + mid;
        else s_marked = 1;
      }
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const unsigned have = last > cc ? min(n[j], last - cc) : 0u;
        if (have && mm <= target) {
          const bool past = mm + have * w[j] <= target;
          before = max(before, cc + (past ? have : static_cast<unsigned>(fmin(static_cast<double>(have), floor((target - mm) / w[j])))));
        }
        cc += n[j], mm += n[j] * w[j];
      }
      before = warp_all(before, [](unsigned x, unsigned y) { return max(x, y); });
      if ((tid & 31) == 0) atomicMax(&sh.nth, before);
      __syncthreads();
      before = min(sh.nth, last - 1u);
      if (tid == 0) sh.state = -1;
      __syncthreads();                                  // everybody has read sh.nth
      cc = count;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (before >= cc && before < cc + n[j]) {
          sh.nth = before - cc;
          sh.ties = n[j];
          sh.value = value_at(j);
          sh.state = 1;
        }
        cc += n[j];
      }
      __syncthreads();
      if (tid == 0) {
        if (s_marked || widest == 255) sh.state = -1;
        a.marked[r] = sh.state < 0;
      }
    }
    __syncthreads();
  }
  if (c > 1) cl.sync();
  const Shared* lead = c > 1 ? cl.map_shared_rank(&sh, 0) : &sh;
  const int state = lead->state;
  const float value = lead->value;
  const unsigned nth = lead->nth;
  const double kept_mass = lead->f1;
  if (state < 0) {
    if (c > 1) cl.sync();               // peers have read this CTA's outcome
    return;
  }
  place(s, sh, a, r, c, rank, value, nth, lead->ties, bins, top, per, kept_mass, table);
}

// ------------------------------------------------------------------------------------------------ any type
constexpr int kSteps = 2048, kStepsEach = kSteps / kThreads;
// A row's weights are whole numbers of 2^-44 of the largest, so 2^19 tokens fit into 64 bits. A step's are counted in units
// smaller by its own power of two (2^-44 of the weight at its beginning, give or take a factor of 2) and rounded once, as
// their sum: many tokens far below the largest keep their weight.
constexpr double kUnit = 17592186044416.0;
__device__ __forceinline__ u64 to_row_units(u64 q, int e) { return e ? (q + (1ull << (e - 1))) >> e : q; }

__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned b = __float_as_uint(x + 0.f);         // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Step {                         // what rank 0 tells the cluster
  int go;                             // 0: this search is not needed
  int bin;
  int few;                            // the bin's tokens fit into the list
  unsigned prefix;
};
constexpr int kList = 1024;
constexpr int kAlive = 512;           // a warp's places for tokens in the window
// Whether a search ends in the n tokens that stand behind cc others (weights in the row's units: mm before them, next behind
// them). 0: the end-th token. 1: the last that begin in front of the aim and among the first `end`. 2: the last that begin at
// or in front of it. Exactly one of a row's bins, or of a bin's values, says yes: the sums are whole numbers, a bin's in smaller
// units until they are rounded, which never falls as the sum grows and ends where the bin ends.
__device__ __forceinline__ bool here(int what, unsigned cc, unsigned n, u64 mm, u64 next, double aim, unsigned end) {
  if (what == 0) return cc < end && end <= cc + n;
  if (what == 1) return (cc == 0 || static_cast<double>(mm) < aim) && cc < end && (!(static_cast<double>(next) < aim) || cc + n >= end);
  return (cc == 0 || static_cast<double>(mm) <= aim) && cc < end && (static_cast<double>(next) > aim || cc + n >= end);
}

__device__ __forceinline__ u64 units_of(double t, const double* table) {
  return t < 64.0 ? static_cast<u64>(two_to_minus(t, table) * kUnit + 0.5) : 0ull;      // nothing in units of 2^-44
}

// A 64-bit sum in two words of shared memory: whoever carries the low one over adds the carry to the high one. (An atomic
// on 64 bits there is a loop of compare and swap: 14 ns for a warp's, against 3 for these.)
__device__ __forceinline__ void add_units(unsigned* low, unsigned* high, u64 q) {
  const unsigned ql = static_cast<unsigned>(q), old = atomicAdd(low, ql), qh = static_cast<unsigned>(q >> 32) + (old + ql < ql ? 1u : 0u);
  if (qh) atomicAdd(high, qh);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_any_kernel(const __grid_constant__ Args a) {
  __shared__ unsigned cnt[kSteps], low_half[kSteps], high_half[kSteps];       // tokens, and their weight in two words
  __shared__ unsigned dcnt[256], dlow[256], dhigh[256];
  __shared__ Shared sh;
  __shared__ Step step[3][5];
  float* const alive = reinterpret_cast<float*>(kept_pieces + a.kept);        // behind the row's pieces
  __shared__ unsigned list[kList], list_n;
  __shared__ u64 list_units[kList];
  __shared__ double table[64];
  const int c = gridDim.x, rank = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  if (a.marked != nullptr) {
    pdl_wait();
    if (a.marked[r] == 0) return;                      // the same for the whole cluster
  }
  cg::cluster_group cl = cg::this_cluster();
  const Share<T> s(a, r, rank, c);
  const Row row(a, r);
  for (int i = tid; i < kSteps; i += kThreads) cnt[i] = 0u, low_half[i] = 0u, high_half[i] = 0u;
  fill_table(table);
  if (tid == 0) sh.found_n = 0u, sh.found_min = 0xffffffffu;
  float top, low;
  extremes(s, sh, c, top, low);
  if (top == -INFINITY || row.greedy) {
    cl.sync();
    if (top == -INFINITY) {
      if (rank == 0 && tid == 0) a.tokens[r] = 0, a.logprobs[r] = -INFINITY;
      return;
    }
    place(s, sh, a, r, c, rank, top, 0u, 1u, list, top, 1.0, 1.0, table);
    return;
  }
  low = top == INFINITY ? top : fmaxf(fmaxf(low, -FLT_MAX), top - kWindow * static_cast<float>(row.T));
  // equal steps; the product is rounded but never falls as the distance grows
  const float inv = top > low ? static_cast<float>(kSteps) / (top - low) : 0.f;
  const auto bin_of = [&](float x) {
    const float q = (top - x) * inv;
    return q < static_cast<float>(kSteps - 1) ? static_cast<int>(q) : q >= static_cast<float>(kSteps - 1) ? kSteps - 1 : 0;
  };
  const double per = 1.4426950408889634 / row.T;
  // a step's power of two: the binary logarithm of the weight at its beginning, a little less so that rounded steps keep below it
  const float fall = inv > 0.f ? static_cast<float>(per / inv * 0.9999) : 0.f;
  // (60 is 42 log2(e); where T is next to the logits' own rounding, top - low is rounded to more than 42 T)
  const auto power_of = [&](int bin) { return min(60, static_cast<int>(bin * fall)); };
  const auto units = [&](float x, int e) { return x == top ? static_cast<u64>(kUnit) : units_of((static_cast<double>(top) - static_cast<double>(x)) * per - e, table); };
  const double floor_units = row.min_p * kUnit;
  unsigned some = 0;
  const auto count_in = [&](float x) {
    const int b = bin_of(x), e = power_of(b);
    const u64 q = units(x, e);
    atomicAdd(&cnt[b], 1u);
    add_units(&low_half[b], &high_half[b], q);
    // on the border itself (a unit is 2^-44) the weight decides
    if (row.min_p > 0.0) {
      const double edge = floor_units * static_cast<double>(1ull << e);
      some += fabs(static_cast<double>(q) - edge) > 2.0 ? static_cast<double>(q) > edge : weight(x, top, row.T) >= row.min_p;
    } else {
      ++some;
    }
  };
  // A warp gathers what lies in the window and counts it in full groups of 32: a masked row's work in 64 bits is that of the
  // tokens its mask leaves. Where all of them fit, the searches look at these instead of at the row again.
  float* const mine = alive + (tid >> 5) * kAlive;
  const int lane = tid & 31;
  int have = 0, done = 0, seen_tokens = 0;
  bool all_kept = true, dense = false;
  s.edges([&](T x) {
    if (value_of<T>(x) >= low) count_in(value_of<T>(x));
  });
  for (int i0 = s.lo + (tid & ~31); i0 < s.hi; i0 += 2 * kThreads) {
    uint4 w[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (i0 + u * kThreads + lane < s.hi) w[u] = s.piece(i0 + u * kThreads + lane);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool in = i0 + u * kThreads + lane < s.hi;
      const T* x = reinterpret_cast<const T*>(&w[u]);
      if (dense) {                                      // most tokens are in the window: gathering them costs more than it saves
#pragma unroll
        for (int q = 0; q < Share<T>::kPer; ++q)
          if (in && value_of<T>(x[q]) >= low) count_in(value_of<T>(x[q]));
        continue;
      }
      seen_tokens += 32 * Share<T>::kPer;
#pragma unroll
      for (int q = 0; q < Share<T>::kPer; ++q) {
        const float v = in ? value_of<T>(x[q]) : 0.f;
        const bool ok = in && v >= low;
        const unsigned m = __ballot_sync(0xffffffffu, ok);
        if (ok) mine[have + __popc(m & ((1u << lane) - 1u))] = v;
        have += __popc(m);
      }
      __syncwarp();
      for (; have - done >= 32; done += 32) count_in(mine[done + lane]);
      if (have > kAlive - 32 * Share<T>::kPer) {        // no room for another piece: only what is not counted yet stays
        const float v = done + lane < have ? mine[done + lane] : 0.f;
        __syncwarp();
        if (done + lane < have) mine[lane] = v;
        __syncwarp();
        if (all_kept) dense = 2 * have > seen_tokens;
        have -= done, done = 0, all_kept = false;
      }
    }
  }
  if (done + lane < have) count_in(mine[done + lane]);
  const auto each_alive = [&](auto&& f) {
    if (!all_kept) {
      s.each([&](float x) {
        if (x >= low) f(x);
      });
      return;
    }
    s.edges([&](T x) {
      if (value_of<T>(x) >= low) f(value_of<T>(x));
    });
    for (int j = lane; j < have; j += 32) f(mine[j]);
  };
  some = warp_all(some, Add());
  if ((tid & 31) == 0) sh.sc[tid >> 5] = some;
  __syncthreads();
  if (tid == 0) {
    unsigned t = 0;
    for (int w = 0; w < kWarps; ++w) t += sh.sc[w];
    sh.cta_count = t;
  }
  cl.sync();
  if (c > 1) {                                         // each CTA adds up its share of the steps and puts it into rank 0's
    unsigned* lead_cnt = cl.map_shared_rank(cnt, 0);
    unsigned* lead_low = cl.map_shared_rank(low_half, 0);
    unsigned* lead_high = cl.map_shared_rank(high_half, 0);
    for (int i = kSteps / c * rank + tid; i < kSteps / c * (rank + 1); i += kThreads) {
      unsigned v[kMaxCluster], l[kMaxCluster], h[kMaxCluster], x = 0;
      u64 y = 0;
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q)
        if (q < c) v[q] = *cl.map_shared_rank(cnt + i, q), l[q] = *cl.map_shared_rank(low_half + i, q), h[q] = *cl.map_shared_rank(high_half + i, q);
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q)
        if (q < c) x += v[q], y += (static_cast<u64>(h[q]) << 32) + l[q];
      lead_cnt[i] = x, lead_low[i] = static_cast<unsigned>(y), lead_high[i] = static_cast<unsigned>(y >> 32);
    }
    cl.sync();
  }
  // rank 0 holds the cluster's histogram and its prefix sums in registers
  unsigned n[kStepsEach], count = 0, c_all = 0, keep = 0, last = 0;
  u64 m[kStepsEach], mass = 0, m_all = 0;
  double total = 0.0, kept = 0.0;
  if (rank == 0) {
#pragma unroll
    for (int j = 0; j < kStepsEach; ++j) {
      const int b = tid * kStepsEach + j;
      n[j] = cnt[b], m[j] = to_row_units((static_cast<u64>(high_half[b]) << 32) + low_half[b], power_of(b));
      count += n[j], mass += m[j];
    }
    unsigned fine = 0;
#pragma unroll
    for (int q = 0; q < kMaxCluster; ++q)
      if (q < c) fine += cl.map_shared_rank(&sh, q)->cta_count;
    block_prefix(count, mass, sh.sc, sh.su, c_all, m_all);
    keep = max(1u, min(min(static_cast<unsigned>(row.k), c_all), fine));
  }
  // three searches: the kept tokens' weight (by their number), the end of top-p, the token
  for (int what = 0; what < 3; ++what) {
    double aim = 0.0;                                  // in units
    if (rank == 0) {
      if (tid == 0) step[what][0].go = what == 0 ? keep < c_all : what == 1 ? row.top_p < 1.0 : 1;
      if (what == 0 && !(keep < c_all)) total = static_cast<double>(m_all);
      if (what == 1) {
        aim = row.top_p * total;
        if (!(row.top_p < 1.0)) kept = total, last = keep;
      }
      if (what == 2) aim = row.u * kept;
      __syncthreads();
      if (step[what][0].go) {
        unsigned cc = count;
        u64 mm = mass;
#pragma unroll
        for (int j = 0; j < kStepsEach; ++j) {
          if (n[j]) {
            if (here(what, cc, n[j], mm, mm + m[j], aim, what == 2 ? last : keep)) {
              step[what][0].bin = tid * kStepsEach + j;
              step[what][0].few = n[j] <= kList;
              sh.c0 = cc, sh.su[0] = mm;
            }
          }
          cc += n[j], mm += m[j];
        }
        if (tid == 0) list_n = 0u;
      }
      __syncthreads();
    }
    cl.sync();
    const Step first = *cl.map_shared_rank(&step[what][0], 0);
    if (!first.go) continue;
    unsigned prefix = 0, seen = 0;
    u64 weighed = 0, inside = 0;                       // what stands in front of the bin in the row's units, and behind that in the bin's
    const int power = power_of(first.bin);
    if (rank == 0) seen = sh.c0, weighed = sh.su[0];
    if (first.few) {
      // the bin's tokens in a list of rank 0; each finds what stands in front of it by looking at all the others
      unsigned* to = cl.map_shared_rank(list, 0);
      unsigned* at = cl.map_shared_rank(&list_n, 0);
      each_alive([&](float x) {
        if (bin_of(x) == first.bin) to[atomicAdd(at, 1u)] = order_key(x);
      });
      cl.sync();
      if (rank == 0) {
        const unsigned many = list_n;
        for (unsigned i = tid; i < many; i += kThreads) list_units[i] = units(key_value(list[i]), power);
        __syncthreads();
        for (unsigned i = tid; i < many; i += kThreads) {
          const unsigned k = list[i];
          unsigned dc = seen, dn = 0u;
          u64 dw = 0;
          const u64 q = list_units[i];
#pragma unroll 4
          for (unsigned j = 0; j < many; ++j) {
            const unsigned o = list[j];
            const u64 oq = list_units[j];
            if (o > k) ++dc, dw += oq;
            dn += o == k;
          }
          if (here(what, dc, dn, weighed + to_row_units(dw, power), weighed + to_row_units(dw + dn * q, power), aim, what == 2 ? last : keep))
            sh.i0 = k, sh.c0 = dc, sh.c1 = dn, sh.cta_mass = dw;
        }
        __syncthreads();
        prefix = sh.i0, seen = sh.c0, inside = sh.cta_mass;
      }
    }
    for (int level = 0; level < 4 && !first.few; ++level) {
      const int shift = 24 - 8 * level;
      if (tid < 256) dcnt[tid] = 0u, dlow[tid] = 0u, dhigh[tid] = 0u;
      __syncthreads();
      each_alive([&](float x) {
        if (bin_of(x) != first.bin) return;
        const unsigned k = order_key(x);
        if (level > 0 && (k >> (shift + 8)) != prefix) return;
        atomicAdd(&dcnt[(k >> shift) & 255u], 1u);
        add_units(&dlow[(k >> shift) & 255u], &dhigh[(k >> shift) & 255u], units(x, power));
      });
      cl.sync();
      if (rank == 0) {
        // digits in descending order, one a thread
        unsigned dn = 0, dc = 0, da;
        u64 dm = 0, dw = 0, db;
        if (tid < 256) {
          unsigned v[kMaxCluster], l[kMaxCluster], h[kMaxCluster];
#pragma unroll
          for (int q = 0; q < kMaxCluster; ++q)
            if (q < c) v[q] = *cl.map_shared_rank(dcnt + 255 - tid, q), l[q] = *cl.map_shared_rank(dlow + 255 - tid, q), h[q] = *cl.map_shared_rank(dhigh + 255 - tid, q);
#pragma unroll
          for (int q = 0; q < kMaxCluster; ++q)
            if (q < c) dn += v[q], dm += (static_cast<u64>(h[q]) << 32) + l[q];
        }
        dc = dn, dw = dm;
        block_prefix(dc, dw, sh.sc, sh.su, da, db);
        dc += seen, dw += inside;
        if (dn) {
          if (here(what, dc, dn, weighed + to_row_units(dw, power), weighed + to_row_units(dw + dm, power), aim, what == 2 ? last : keep)) {
            step[what][level + 1].prefix = (prefix << 8) | static_cast<unsigned>(255 - tid);
            sh.c0 = dc, sh.c1 = dn, sh.cta_mass = dw;
          }
        }
        __syncthreads();
        seen = sh.c0, inside = sh.cta_mass;
      }
      cl.sync();
      prefix = cl.map_shared_rank(&step[what][level + 1], 0)->prefix;
    }
    if (rank == 0) {
      // all tokens of one value: seen, weighed and inside stand before them, sh.c1 is their number
      const float x = key_value(prefix);
      const double w = weight(x, top, row.T) * kUnit, front = static_cast<double>(weighed) + static_cast<double>(inside) / static_cast<double>(1ull << power);
      const unsigned have = min(sh.c1, (what == 2 ? last : keep) - seen);
      if (what == 0) {
        total = front + (keep - seen) * w;
      } else if (what == 1) {
        const double fit = ceil((aim - front) / w);
        const unsigned take = static_cast<unsigned>(fmin(static_cast<double>(have), fmax(fit, 1.0)));
        last = seen + take, kept = front + take * w;
      } else {
        const double at = floor((aim - front) / w);
        if (tid == 0) {
          sh.nth = at < 0.0 ? 0u : at < have ? static_cast<unsigned>(at) : have - 1u;
          sh.value = x;
          sh.ties = sh.c1;
          sh.f1 = kept / kUnit;
        }
      }
      __syncthreads();
    }
  }
  cl.sync();
  const Shared* lead = cl.map_shared_rank(&sh, 0);
  const float value = lead->value;
  const unsigned nth = lead->nth;
  const double kept_mass = lead->f1;
  place(s, sh, a, r, c, rank, value, nth, lead->ties, list, top, per, kept_mass, table);
}

template <auto Kern>
int launch(const Args& args, int rows, int cluster, int smem, int most, bool early, cudaStream_t s) {
  return ixh::launch_cluster<Kern>(args, dim3(cluster, rows), kThreads, cluster, smem, most, early, s);
}

}  // namespace

IX_API int ix_sample_rows_max_vocab() { return 1 << 19; }

// logits [rows, V] with row stride ld, dtype 0 = bf16, 1 = fp32; u fp32 [rows] in [0, 1), others are clamped; temperature / top_p / min_p fp32
// [rows], top_k int32 [rows] (each may be null); tokens int64 [rows], logprobs fp32 [rows]; marked int32 [rows] scratch (bf16).
IX_API int ix_sample_rows(const void* logits, long long ld, int rows, int V, int dtype, const void* u, const void* temperature, const void* top_k,
                          const void* top_p, const void* min_p, void* tokens, void* logprobs, void* marked, void* stream) {
  if (rows <= 0) return 0;
  if (rows > 65535) return ixh::fail(ixh::IX_ESIZE, "sample_rows: %d rows, at most 65535 in a call", rows);
  if (V < 1 || V > ix_sample_rows_max_vocab()) return ixh::fail(ixh::IX_ESIZE, "sample_rows: a vocabulary of 1 to %d, not %d", ix_sample_rows_max_vocab(), V);
  if (dtype != 0 && dtype != 1) return ixh::fail(ixh::IX_EARG, "sample_rows: dtype must be 0 (bf16) or 1 (fp32)");
  if (dtype == 0 && marked == nullptr) return ixh::fail(ixh::IX_EARG, "sample_rows: bf16 rows need the scratch for marks");
  Args a;
  a.logits = logits, a.ld = ld, a.V = V;
  a.u = static_cast<const float*>(u);
  a.temperature = static_cast<const float*>(temperature);
  a.top_k = static_cast<const int*>(top_k);
  a.top_p = static_cast<const float*>(top_p);
  a.min_p = static_cast<const float*>(min_p);
  a.tokens = static_cast<long long*>(tokens);
  a.logprobs = static_cast<float*>(logprobs);
  a.marked = dtype == 0 ? static_cast<int*>(marked) : nullptr;
  // CTAs a row: as many as leave all rows' CTAs resident together (two a multiprocessor), but not beyond a few thousand
  // tokens each. Where its pieces then fit beside another CTA's, they stay in shared memory after the first pass
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= 148 * 2 && V > c * 8192) c *= 2;
  const int pieces = static_cast<int>(static_cast<long long>(V) * (dtype == 0 ? 2 : 4) / c / 16 + 2);
  const bool alone = static_cast<long long>(rows) * c <= 148;          // one CTA a multiprocessor
  constexpr int kAnyStatic = 44 * 1024, kFew = kWarps * kAlive * 4, kBf16Static = 20 * 1024, kAll = 220 * 1024;
  const auto keep = [&](int other) {
    a.cached = pieces * 16 <= (alone ? kAll : 106 * 1024) - other;
    a.kept = a.cached ? pieces : 0;
    return a.kept * 16;
  };
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == 1) return launch<sample_any_kernel<float>>(a, rows, c, keep(kAnyStatic + kFew) + kFew, kAll - kAnyStatic, false, s);
  const int rc = launch<sample_bf16_kernel>(a, rows, c, keep(kBf16Static), kAll - kBf16Static, false, s);
  if (rc) return rc;
  // started while the first one drains: it waits for its marks, and nearly always ends there
  return launch<sample_any_kernel<__nv_bfloat16>>(a, rows, c, keep(kAnyStatic + kFew) + kFew, kAll - kAnyStatic, true, s);
}
