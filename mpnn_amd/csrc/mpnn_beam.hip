// Beam search: the choice of the next hypotheses over beams x vocabulary, and the beams' states following it.
//
//   mpnn_beam_select   c[w][v] = score[w] + x[w][v] - log sum_u exp x[w][u],  x = logits + bias;  the best n_out of a
//                      group's W V candidates, ties to the lowest beam, then the lowest token
//   mpnn_beam_reorder  x[b][j] <- x[b][parent[b][j]] for several state tensors, in place
//
// The choice compares candidates of different beams, whose scores lie close together: the log-sum-exp and the candidates
// are held in fp64 (CDNA's fp64 vector rate is its fp32 rate without packed instructions), so that the order does not
// hang on the order of a sum.  Only the scores handed back are rounded, to fp32.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <stdint.h>

#include "mpnn_common.h"
#include "mpnn_hip.h"
#include "mpnn_reduce.h"

namespace {

constexpr int SEL_MAX_N = 256;       // hypotheses kept of a group
constexpr int SEL_U = 32;            // logits a thread of a long slice holds
constexpr int SEL_CAP = 1024;        // candidates a workgroup ranks in LDS
constexpr int SEL_LONG = 300;        // long slices from this many on: about one a CU
constexpr long long KEY_NONE = (long long)0x8000000000000000ull;  // below every candidate
constexpr long long KEY_NAN = 0x7fffffffffffffffll;               // NaN ranks first: a broken beam shows at once

// ---- order of candidates: signed 64-bit keys that sort like the values (-0 as +0) ----
__device__ __forceinline__ long long key_of(double c) {
  if (c != c) return KEY_NAN;
  const long long b = __double_as_longlong(c + 0.0);
  return b ^ ((b >> 63) & 0x7fffffffffffffffll);
}
__device__ __forceinline__ double value_of(long long k) {
  return k == KEY_NAN ? __longlong_as_double(0x7ff8000000000000ll) : __longlong_as_double(k ^ ((k >> 63) & 0x7fffffffffffffffll));
}
__device__ __forceinline__ bool better(long long ka, int ia, long long kb, int ib) { return ka > kb || (ka == kb && ia < ib); }

// A NaN or +inf among a beam's logits makes its log-sum-exp NaN; so may its score be NaN or +inf.  Such a beam offers one
// candidate, token 0 with the score NaN: the failure stands in the first slot and takes no more than one.
__device__ __forceinline__ bool broken(double score, double lse) { return lse != lse || !(score < INFINITY); }

// exp(d) for d <= 0 to 1.1e-12 relative (2^f by a degree-8 polynomial, tools/fit_exp2.py; exactly 1 at 0).  d below -700 and
// NaN count as -700: 1e-304, nothing beside a sum that holds a 1.  15 instructions: adding 1.5 * 2^52 rounds to the nearest
// integer and leaves it in the low word, which goes straight into the exponent.
__device__ __forceinline__ double exp_neg(double d) {
  d = fmax(d, -700.0);
  const double t = fma(d, 1.4426950408889634, 6755399441055744.0), n = t - 6755399441055744.0;
  const double f = fma(d, 1.4426950408889634, -n);
  double p = 1.32552248847991267e-06;
  p = fma(p, f, 1.53100794023831035e-05);
  p = fma(p, f, 1.54034558524190164e-04);
  p = fma(p, f, 1.33334505680000079e-03);
  p = fma(p, f, 9.61812915940261914e-03);
  p = fma(p, f, 5.55041094120593409e-02);
  p = fma(p, f, 2.40226506958129887e-01);
  p = fma(p, f, 6.93147180545933494e-01);
  p = fma(p, f, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}

template <typename T>
__device__ __forceinline__ float to_f(T x) { return (float)x; }
template <>
__device__ __forceinline__ float to_f<__hip_bfloat16>(__hip_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }

// 32 bits that order values (NaN above all), and the least value that has at least those bits; fp64 by its high word
template <typename X>
struct Order;
template <>
struct Order<float> {
  static __device__ __forceinline__ unsigned bits(float x, bool nan) {
    const int b = __float_as_int(x + 0.0f);
    return nan ? 0xffffffffu : (unsigned)(b ^ ((b >> 31) & 0x7fffffff)) ^ 0x80000000u;
  }
  static __device__ __forceinline__ float least(unsigned u) {
    const int k = (int)(u ^ 0x80000000u), b = k ^ ((k >> 31) & 0x7fffffff);
    return u <= 0x007fffffu ? -3.4028234663852886e38f : u >= 0xff800000u ? INFINITY : __int_as_float(b);
  }
};
template <>
struct Order<double> {
  static __device__ __forceinline__ unsigned bits(double x, bool nan) {
    return nan ? 0xffffffffu : (unsigned)(key_of(x) >> 32) ^ 0x80000000u;
  }
  static __device__ __forceinline__ double least(unsigned u) {   // u <= -inf's: everything but -inf
    return u <= 0x000fffffu   ? -1.7976931348623157e308
           : u >= 0xfff00000u ? INFINITY
                              : value_of((long long)((unsigned long long)(u ^ 0x80000000u) << 32));
  }
};

// the least X that is not below d
template <typename X>
__device__ __forceinline__ X at_least(double d) {
  const X x = (X)d;
  if (std::is_same<X, double>::value || !((double)x < d)) return x;
  const int b = __float_as_int((float)x);
  return (X)__int_as_float((float)x == 0.f ? 1 : b < 0 ? b - 1 : b + 1);
}

// largest and least value of the wave, uniform: rotations within rows of 16 lanes, then one lane of each row
__device__ __forceinline__ unsigned wave_max_u(unsigned x) {
#define MPNN_ROR(n)                                                                               \
  {                                                                                               \
    const unsigned y = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + n, 0xf, 0xf, false); \
    x = y > x ? y : x;                                                                            \
  }
  MPNN_ROR(8) MPNN_ROR(4) MPNN_ROR(2) MPNN_ROR(1)
#undef MPNN_ROR
  unsigned m = (unsigned)__builtin_amdgcn_readlane((int)x, 0);
#pragma unroll
  for (int l = 16; l < 64; l += 16) {
    const unsigned y = (unsigned)__builtin_amdgcn_readlane((int)x, l);
    m = y > m ? y : m;
  }
  return m;
}
__device__ __forceinline__ unsigned wave_min_u(unsigned x) { return ~wave_max_u(~x); }

// Bisection starts at the first bit in which values between least and largest differ: T with the bits they share, and that
// bit's place (-1: they are equal).  Scores share a sign and most of an exponent.
__device__ __forceinline__ int common_prefix(unsigned least, unsigned largest, unsigned& T) {
  const unsigned differ = least ^ largest;
  const int bit = 31 - __clz((int)differ);     // -1 for 0
  // (as `bit < 0 ? largest : largest & mask` hipcc 7.2 selects by an SCC that the mask's shift has overwritten)
  T = largest & (unsigned)(~0ull << (bit + 1));
  return bit;
}

// some T that at least q of the wave's values u reach, and seldom half as many more, 0 if fewer than q are above 0 (uniform):
// bisection over ballots
template <int E>
__device__ __forceinline__ unsigned wave_kth(const unsigned (&u)[E], int q) {
  unsigned largest = 0, least = 0xffffffffu;
  int some = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    largest = u[i] > largest ? u[i] : largest;
    least = u[i] && u[i] < least ? u[i] : least;
    some += __popcll(__ballot(u[i] != 0));
  }
  if (some < q) return 0;
  unsigned T;
  int bit = common_prefix(wave_min_u(least), wave_max_u(largest), T);
#pragma unroll 1
  for (; bit >= 0; --bit) {
    const unsigned t = T | (1u << bit);
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) cnt += __popcll(__ballot(u[i] >= t));
    if (cnt >= q) {
      T = t;
      if (cnt <= (E > 1 && q > 42 ? (q <= 64 ? 64 : q + (q >> 2)) : q + (q >> 1))) break;   // 64 are ranked in one turn
    }
  }
  return T;
}

// a bound that the n-th best of a workgroup's values is no worse than, from each thread's best (u, 0 = none): the least of
// the four waves' ceil(n / 4)-th best threads where every thread has values (they share a row: close to the n-th best), else the
// best of the waves' n-th best threads, which threads without values do not spoil.  ru: 4 words of LDS, written here; the
// caller's barrier follows, then block_bound reads them.
__device__ __forceinline__ void wave_bounds(unsigned u, int n, bool full, unsigned* ru) {
  const unsigned each[1] = {u}, q = wave_kth(each, full || n > 64 ? (n + 3) / 4 : n);
  if ((threadIdx.x & 63) == 0) ru[threadIdx.x >> 6] = q;
}
__device__ __forceinline__ unsigned block_bound(int n, bool full, const unsigned* ru) {
  unsigned lo = ru[0], hi = ru[0];
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    lo = ru[i] < lo ? ru[i] : lo;
    hi = ru[i] > hi ? ru[i] : hi;
  }
  return full || n > 64 ? lo : hi;
}

struct SelectArgs {
  const void* logits;
  long long sb, sw;          // strides of a group and of a beam, in elements
  const float* scores;       // [B][W]
  const float* bias;         // NULL or element (b, w, v) at bias[b * bb + w * bw + v]
  long long bb, bw;
  const long long* forced;   // NULL or [B][W]; negative = free
  int B, W, V, n;
  float* out_scores;
  long long* parent;
  long long* token;
};

__device__ __forceinline__ void write_slot(const SelectArgs& a, int b, int slot, long long key, int flat) {
  const long long o = (long long)b * a.n + slot;
  a.out_scores[o] = (float)value_of(key);
  a.parent[o] = flat / a.V;
  a.token[o] = flat % a.V;
}
// a slot that no candidate is left for keeps its beam: nothing has to move for it
__device__ __forceinline__ void write_dead_slot(const SelectArgs& a, int b, int slot) {
  const long long o = (long long)b * a.n + slot;
  const int w = slot % a.W;
  const long long f = a.forced ? a.forced[(long long)b * a.W + w] : -1;
  a.out_scores[o] = -INFINITY;
  a.parent[o] = w;
  a.token[o] = f < 0 ? 0 : (f < a.V ? f : a.V - 1);
}

// Rank the `cnt` collected candidates and hand the n best to put(slot, key, place): each is compared with every other one, by 2, 4
// or 8 neighbouring lanes where there are lanes enough, eight at a time (they are in LDS: one by one, each waits for its read).
// lk and li have RANK_PAD places behind the candidates.
constexpr int RANK_PAD = 64;
template <int WAVES = 4, typename Put>
__device__ __forceinline__ void rank_collected(long long* lk, const int* li, int cnt, int n, Put put) {
  constexpr int T = 64 * WAVES;
  if (threadIdx.x < RANK_PAD) lk[cnt + threadIdx.x] = KEY_NONE;
  int lp = 0;
  auto sum = [&](int v) {
    if (lp > 0) v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false);    // lane ^ 1
    if (lp > 1) v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false);    // lane ^ 2
    if (lp > 2) v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false);   // mirrored in 8 lanes
    return v;
  };
  __syncthreads();
  for (int e0 = 0; e0 < cnt; e0 += T >> lp) {
    lp = 0;
    while (cnt > 32 && lp < 3 && (cnt - e0) << (lp + 1) <= T) ++lp;
    const int part = threadIdx.x & ((1 << lp) - 1), step = 1 << lp;
    const int e = e0 + ((int)threadIdx.x >> lp);
    const bool in = e < cnt;                 // the same in all lanes of an entry
    if (!__any(in)) break;
    const long long ke = lk[in ? e : 0];
    const int ie = li[in ? e : 0];
    int r = 0;
    for (int q0 = 0; q0 < cnt; q0 += 8 * step) {
      long long kq[8];
      int iq[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        kq[i] = lk[q0 + i * step + part];
        iq[i] = li[q0 + i * step + part];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) r += better(kq[i], iq[i], ke, ie);
    }
    r = sum(r);
    if (in && part == 0 && r < n) put(r, ke, ie);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Small groups: one wave holds all W V candidates of a group in registers (M per lane).  Lanes are split into W
// subgroups of g = 64 / (W rounded up to a power of two); lane j of a subgroup has tokens j, j + g, ...  No LDS
// exchange before the winners are ranked, no barrier: at the model's 21 letters the call is bound by its own latency.
// ---------------------------------------------------------------------------------------------------------------
constexpr int SMALL_CAP = 512;   // candidates a wave ranks in LDS

// The candidates of lane j of the g = 2^g_log2 lanes that share beam w: keys of tokens j, j + g, ...; the best of them
template <typename T, int M>
__device__ __forceinline__ long long lane_candidates(const SelectArgs& a, int b, int w, int j, int g_log2, long long (&k)[M]) {
  const int g = 1 << g_log2;
  const bool live = w < a.W;
  const long long row = (long long)b * a.W + (live ? w : 0);
  const double s = (double)a.scores[row];
  const long long f = a.forced ? a.forced[row] : -1;
  const T* logits = (const T*)a.logits + (long long)b * a.sb + (live ? w : 0) * a.sw;
  const float* bias = a.bias ? a.bias + (long long)b * a.bb + (live ? w : 0) * a.bw : nullptr;
  T raw[M];
  float add[M];
#pragma unroll
  for (int i = 0; i < M; ++i) {      // every load is in flight before the first is used; places beyond V read the last one
    const int v = j + (i << g_log2);
    raw[i] = logits[v < a.V ? v : a.V - 1];
    add[i] = bias ? bias[v < a.V ? v : a.V - 1] : 0.f;
  }
  double x[M];
  double top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int v = j + (i << g_log2);
    x[i] = live && v < a.V && add[i] != -INFINITY ? (double)to_f(raw[i]) + (double)add[i] : -INFINITY;
    top = fmax(top, x[i]);
    nan |= x[i] != x[i];
  }
  top = group_max(top, g);
  double sum = nan || top == INFINITY ? (double)NAN : 0.0;
  const double base = top == -INFINITY ? 0.0 : top;
#pragma unroll
  for (int i = 0; i < M; ++i) sum += exp_neg(x[i] - base);
  sum = group_sum(sum, g);
  const double lse = base + log(sum);   // of no use where nothing is left of the row: no candidate below
  const bool bad = broken(s, lse);
  long long best = KEY_NONE;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int v = j + (i << g_log2);
    double c = x[i] == -INFINITY ? -INFINITY : s + (x[i] - lse);
    if (bad) c = v == 0 ? (double)NAN : -INFINITY;
    if (f >= 0) c = v == (int)(f < a.V ? f : a.V - 1) ? s : -INFINITY;
    k[i] = live && v < a.V && !(c == -INFINITY) ? key_of(c) : KEY_NONE;
    best = k[i] > best ? k[i] : best;
  }
  return best;
}

template <typename T, int M>
__global__ void __launch_bounds__(64)
k_select_small(SelectArgs a, int g_log2) {
  __shared__ long long lk[SMALL_CAP];
  __shared__ int li[SMALL_CAP];
  const int b = blockIdx.x, lane = threadIdx.x, w = lane >> g_log2, j = lane & ((1 << g_log2) - 1);
  long long k[M];
  const long long best = lane_candidates<T, M>(a, b, w, j, g_log2, k);
  // at least n candidates reach the bound that n lanes' best ones do, seldom many more
  int cnt = SMALL_CAP + 1;
  if (a.n <= 64) {
    const unsigned each[1] = {(unsigned)(best >> 32) ^ 0x80000000u}, T32 = wave_kth(each, a.n);
    const long long bound = T32 ? (long long)((unsigned long long)(T32 ^ 0x80000000u) << 32) : KEY_NONE + 1;
    cnt = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const bool in = k[i] >= bound && k[i] != KEY_NONE;
      const unsigned long long m = __ballot(in);
      const int p = cnt + __popcll(m & ((1ull << lane) - 1));
      if (in && p < SMALL_CAP) {
        lk[p] = k[i];
        li[p] = w * a.V + j + (i << g_log2);
      }
      cnt += __popcll(m);
    }
  }
  if (cnt > SMALL_CAP) {
    // many kept, or many equal ones: the n best exactly, by bisection over the keys and then over places of equal ones
    int total = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) total += __popcll(__ballot(k[i] != KEY_NONE));
    const int n = total < a.n ? total : a.n;
    unsigned long long cut = 1;            // as unsigned words: KEY_NONE is 0
    int last = 0x7fffffff;                 // of the candidates that equal cut, those up to this place
    if (total > n) {
      cut = 0;
      int reach = total;
      for (int bit = 63; bit >= 0 && reach != n; --bit) {
        const unsigned long long t = cut | (1ull << bit);
        int c = 0;
#pragma unroll
        for (int i = 0; i < M; ++i) c += __popcll(__ballot(((unsigned long long)k[i] ^ (unsigned long long)KEY_NONE) >= t));
        if (c >= n) {
          cut = t;
          reach = c;
        }
      }
      if (reach > n) {
        int above = 0;
#pragma unroll
        for (int i = 0; i < M; ++i)
          above += __popcll(__ballot(((unsigned long long)k[i] ^ (unsigned long long)KEY_NONE) > cut));
        int lo = 0, hi = a.W * a.V - 1;    // the smallest place p with above + #(equal, place <= p) >= n
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          int c = above;
#pragma unroll
          for (int i = 0; i < M; ++i)
            c += __popcll(__ballot(((unsigned long long)k[i] ^ (unsigned long long)KEY_NONE) == cut &&
                                   w * a.V + j + (i << g_log2) <= mid));
          if (c >= n) hi = mid; else lo = mid + 1;
        }
        last = lo;
      }
    }
    cnt = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const unsigned long long u = (unsigned long long)k[i] ^ (unsigned long long)KEY_NONE;
      const int place = w * a.V + j + (i << g_log2);
      const bool in = u > cut || (u == cut && place <= last);
      const unsigned long long m = __ballot(in);
      if (in) {
        const int p = cnt + __popcll(m & ((1ull << lane) - 1));
        lk[p] = k[i];
        li[p] = place;
      }
      cnt += __popcll(m);
    }
  }
  __syncthreads();
  for (int e = lane; e < cnt; e += 64) {
    const long long ke = lk[e];
    const int ie = li[e];
    int r = 0;
#pragma unroll 8
    for (int q = 0; q < cnt; ++q) r += better(lk[q], li[q], ke, ie);
    if (r < a.n) write_slot(a, b, r, ke, ie);
  }
  for (int e = cnt + lane; e < a.n; e += 64) write_dead_slot(a, b, e);
}

// ---------------------------------------------------------------------------------------------------------------
// Large vocabularies, first pass: a workgroup reads a slice of 256 U logits of one beam once, keeps it in registers,
// and leaves the slice's maximum, its sum of exponentials and its `depth` best logits, n + 1 of them where n < 256.  (One
// more than can be kept: logits that differ may become equal scores, of which the lowest tokens are wanted.  By the entry
// behind the n-th the second pass sees whether the slice may hold such tokens beside its list.)
// ---------------------------------------------------------------------------------------------------------------
struct SlicePart {
  double top, sum;
};

// some T that at least q of the workgroup's values u reach, and seldom a quarter more; 0 if fewer than q are above 0
template <int E, int WAVES = 4>
__device__ __forceinline__ unsigned block_kth(const unsigned (&u)[E], int q, unsigned (*cnt)[WAVES]) {
  unsigned largest = 0, least = 0xffffffffu;
  int some = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    largest = u[i] > largest ? u[i] : largest;
    least = u[i] && u[i] < least ? u[i] : least;
    some += __popcll(__ballot(u[i] != 0));
  }
  largest = wave_max_u(largest);
  least = wave_min_u(least);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    cnt[0][wave] = largest;
    cnt[1][wave] = least;
    cnt[2][wave] = some;
  }
  __syncthreads();
  some = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    largest = cnt[0][i] > largest ? cnt[0][i] : largest;
    least = cnt[1][i] < least ? cnt[1][i] : least;
    some += cnt[2][i];
  }
  if (some < q) return 0;
  unsigned T;
  int bit = common_prefix(least, largest, T), turn = 3;
#pragma unroll 1
  for (; bit >= 0; --bit) {
    const unsigned t = T | (1u << bit);
    int c = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) c += __popcll(__ballot(u[i] >= t));
    if ((threadIdx.x & 63) == 0) cnt[turn][wave] = c;
    __syncthreads();
    c = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) c += (int)cnt[turn][i];
    turn ^= 7;             // 3, 4, 3 ...: written again two barriers from here
    if (c >= q) {
      T = t;
      if (c <= q + (q >> 2)) break;
    }
  }
  return T;
}

// Ranking compares every collected candidate with every other one.  Where the first bound let many through, the best of
// those in the list give a closer one: collect(least) puts what is not below `least` into the list again, counting in rc.
// Returns the list's length; more than CAP where too many are equal.  (256 x 60 beams x 1000 tokens, 60 kept: lists of 600 and
// 1136 us before; 82 with one wave a row.)
template <int CAP, int WAVES, typename Collect>
__device__ __forceinline__ int collect_fewer(int q, const long long* lk, int* rc, unsigned (*ct)[WAVES], Collect collect) {
  constexpr int T = 64 * WAVES;
  unsigned last = 0;
  int cnt = *rc;
#pragma unroll 1
  while (cnt > 256 && cnt > 2 * q) {
    unsigned u[CAP / T];
#pragma unroll
    for (int i = 0; i < CAP / T; ++i) {
      const int e = threadIdx.x + T * i;
      u[i] = e < cnt ? (unsigned)(lk[e] >> 32) ^ 0x80000000u : 0u;
    }
    const unsigned bound = block_kth<CAP / T, WAVES>(u, q, ct);
    if (bound <= last) break;
    last = bound;
    __syncthreads();                         // everybody has read the list
    if (threadIdx.x == 0) *rc = 0;
    __syncthreads();
    collect(value_of((long long)((unsigned long long)(bound ^ 0x80000000u) << 32)), bound);
    __syncthreads();
    cnt = *rc;
  }
  return cnt;
}

// best of the workgroup's (key, place) pairs; every thread gets it
template <int WAVES = 4>
__device__ __forceinline__ void block_best(long long& k, int& p, long long* sk, int* sp) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const long long ok = __shfl_xor(k, o);
    const int op = __shfl_xor(p, o);
    if (better(ok, op, k, p)) { k = ok; p = op; }
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { sk[threadIdx.x >> 6] = k; sp[threadIdx.x >> 6] = p; }
  __syncthreads();
  k = sk[0];
  p = sp[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i)
    if (better(sk[i], sp[i], k, p)) { k = sk[i]; p = sp[i]; }
}

// Middling groups: 4 to 16 waves hold a group's candidates in registers, as one wave does for small ones, and rank those that
// reach the bound in LDS.  64 beams x 21 letters, 64 kept: 6.2 us with 4, where one wave took 16-21; 21 x 9 x 468, 18 kept: 13
// us with 16, 18 with 4; 205 x 61 x 131, 64 kept: 20 us, as slices 69.
template <typename T, int M, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
k_select_group(SelectArgs a, int g_log2) {
  __shared__ unsigned ct[5][WAVES];
  __shared__ int rc;
  __shared__ long long lk[SEL_CAP + RANK_PAD];
  __shared__ int li[SEL_CAP + RANK_PAD];
  const int b = blockIdx.x, tid = threadIdx.x, w = tid >> g_log2, j = tid & ((1 << g_log2) - 1);
  long long k[M];
  const unsigned best[1] = {(unsigned)(lane_candidates<T, M>(a, b, w, j, g_log2, k) >> 32) ^ 0x80000000u};   // 0: none
  if (tid == 0) rc = 0;
  const unsigned first = block_kth<1, WAVES>(best, a.n, ct);   // the n-th best thread, or 0
  auto collect = [&](double, unsigned bound) {
#pragma unroll
    for (int i = 0; i < M; ++i) {
      if (k[i] != KEY_NONE && ((unsigned)(k[i] >> 32) ^ 0x80000000u) >= bound) {
        const int q = atomicAdd(&rc, 1);
        if (q < SEL_CAP) {
          lk[q] = k[i];
          li[q] = w * a.V + j + (i << g_log2);
        }
      }
    }
  };
  collect(0.0, first);
  __syncthreads();
  const int cnt = collect_fewer<SEL_CAP, WAVES>(a.n, lk, &rc, ct, collect);
  if (cnt <= SEL_CAP) {
    rank_collected<WAVES>(lk, li, cnt, a.n, [&](int r, long long ke, int pe) { write_slot(a, b, r, ke, pe); });
    for (int r = cnt + tid; r < a.n; r += 64 * WAVES) write_dead_slot(a, b, r);
    return;
  }
  // more ties than the list holds: one after the other
  long long prev = KEY_NAN;
  int place = -1;
  __shared__ long long sk[WAVES];
  __shared__ int sp[WAVES];
  for (int r = 0; r < a.n; ++r) {
    long long kb = KEY_NONE;
    int pb = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int pe = w * a.V + j + (i << g_log2);
      if (k[i] != KEY_NONE && better(prev, place, k[i], pe) && better(k[i], pe, kb, pb)) { kb = k[i]; pb = pe; }
    }
    block_best<WAVES>(kb, pb, sk, sp);
    if (tid == 0) {
      if (kb != KEY_NONE) write_slot(a, b, r, kb, pb); else write_dead_slot(a, b, r);
    }
    prev = kb;
    place = pb;
  }
}

__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }

// U logits of a thread on their way: 16-byte loads, VE = 16 / sizeof(T) neighbours each, THREADS VE apart.  They stay packed as
// they come until they are used: unpacking at the load would wait for each before the next is requested.
template <typename T, int U, bool BIAS, int THREADS>
struct Logits {
  static constexpr int VE = 16 / (int)sizeof(T), WORDS = U * (int)sizeof(T) / 4, PER = 4 / (int)sizeof(T);
  typedef typename std::conditional<BIAS, double, float>::type X;
  unsigned q[WORDS];
  float add[BIAS ? U : 1];
  // elements base .. base + THREADS U of a row; what is outside counts as -inf
  __device__ __forceinline__ void load(const T* row, const float* bias, int base, int V) {
#pragma unroll
    for (int it = 0; it < U / VE; ++it) {
      const int c0 = base + it * THREADS * VE, e0 = c0 + (int)threadIdx.x * VE;   // of the turn, of this thread
      if (c0 + THREADS * VE <= V) {
        __builtin_memcpy(q + 4 * it, row + e0, 16);                               // of any alignment
        if (BIAS) __builtin_memcpy(add + it * VE, bias + e0, 4 * VE);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          q[4 * it + i] = 0;
#pragma unroll
          for (int h = 0; h < PER; ++h) {
            const int e = e0 + PER * i + h;
            q[4 * it + i] |= (e < V ? bits_of(row[e]) : minus_inf()) << (16 * h);
            if (BIAS) add[BIAS ? it * VE + PER * i + h : 0] = e < V ? bias[e] : 0.f;
          }
        }
      }
    }
  }
  static __device__ __forceinline__ unsigned bits_of(float x) { return __float_as_uint(x); }
  static __device__ __forceinline__ unsigned bits_of(__hip_bfloat16 x) { return __bfloat16_as_ushort(x); }
  static __device__ __forceinline__ unsigned bits_of(__half x) { return __half_as_ushort(x); }
  static __device__ __forceinline__ unsigned minus_inf() {
    return std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
  }
  __device__ __forceinline__ X value(int i) const {
    float x;
    if (std::is_same<T, float>::value) x = __uint_as_float(q[i / PER]);
    else if (std::is_same<T, __hip_bfloat16>::value) x = __uint_as_float(i % PER ? q[i / PER] & 0xffff0000u : q[i / PER] << 16);
    else x = __half2float(__ushort_as_half((unsigned short)(q[i / PER] >> (i % PER * 16))));
    if (!BIAS) return (X)x;
    return add[BIAS ? i : 0] == -INFINITY ? (X)-INFINITY : (X)x + (X)add[BIAS ? i : 0];
  }
  static __device__ __forceinline__ int place(int base, int i) {
    return base + (i / VE * THREADS + (int)threadIdx.x) * VE + i % VE;
  }
};

// Four waves a SIMD leave 128 registers: with U = 32 and no bias 2 of them are spilled (12 bytes of scratch a lane), 14 (60 bytes)
// for fp16; the other instances spill none.
template <typename T, int U, bool BIAS, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, U > 8 ? 4 : 1)
k_select_slice(SelectArgs a, int splits, int depth, SlicePart* __restrict__ part, long long* __restrict__ pk,
               int* __restrict__ pi) {
  constexpr int THREADS = 64 * WAVES, CAP = WAVES == 1 ? 512 : SEL_CAP;
  __shared__ double rd[2 * WAVES];
  __shared__ unsigned ru[4], ct[5][WAVES];
  __shared__ int rc;
  __shared__ long long lk[CAP + RANK_PAD];
  __shared__ int li[CAP + RANK_PAD];
  typedef Logits<T, U, BIAS, THREADS> In;
  typedef typename In::X X;
  const int row = blockIdx.x / splits, split = blockIdx.x % splits;
  const int b = row / a.W, w = row % a.W, tid = threadIdx.x, wave = tid >> 6;
  // a group's lists lie side by side: entry r of its list l at r * lists + l
  const int lists = a.W * splits;
  const long long mine = (long long)b * lists * depth + w * splits + split;
  if (a.forced && a.forced[row] >= 0) return;     // the second pass knows the row's one candidate
  const T* lrow = (const T*)a.logits + (long long)b * a.sb + (long long)w * a.sw;
  const float* brow = BIAS ? a.bias + (long long)b * a.bb + (long long)w * a.bw : nullptr;
  // slices are cut by the row's tokens, not by memory's 16 bytes: beams of equal logits have equal sums, bit for bit, and tie
  const int base = split * (THREADS * U);
  In in;
  in.load(lrow, brow, base, a.V);
  X x[U], tmax = (X)-INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    x[i] = in.value(i);
    tmax = max_of(tmax, x[i]);
    nan |= x[i] != x[i];
  }
  const bool full = base + THREADS * U <= a.V;
  unsigned bound = 0;
  if (WAVES == 1) {
    unsigned u[U];
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = x[i] == -INFINITY ? 0u : Order<X>::bits(x[i], x[i] != x[i]);
    bound = wave_kth(u, depth);
  } else if (full || depth <= 16) {
    wave_bounds(Order<X>::bits(tmax, nan), depth, full, ru);
  } else {
    const unsigned each[1] = {Order<X>::bits(tmax, nan)};
    bound = block_kth<1>(each, depth, ct);
  }
  double top = group_max((double)tmax, 64);
  if ((tid & 63) == 0) rd[wave] = top;
  if (tid == 0) rc = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) top = fmax(top, rd[i]);
  if (WAVES > 1 && (full || depth <= 16)) bound = block_bound(depth, full, ru);
  const X least = Order<X>::least(bound);
  const double from = top == -INFINITY ? 0.0 : top;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int i = 0; i < U; ++i) s[i & 3] += exp_neg((double)x[i] - from);
  double sum = nan || top == INFINITY ? (double)NAN : (s[0] + s[1]) + (s[2] + s[3]);
  auto put = [&](X xi, int place) {
    const int p = atomicAdd(&rc, 1);
    if (p < CAP) {
      lk[p] = key_of((double)xi);
      li[p] = place;
    }
  };
  if (!(tmax < least) || nan) {            // few threads: one look at the largest instead of one at each
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (!(x[i] < least)) put(x[i], In::place(base, i));
  }
  sum = group_sum(sum, 64);
  if ((tid & 63) == 0) rd[WAVES + wave] = sum;
  __syncthreads();                         // the list is complete too
  if (tid == 0) {
    double all = rd[WAVES];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) all += rd[WAVES + i];
    part[blockIdx.x].top = top;            // -inf with a NaN for the sum where the slice holds nothing but NaN
    part[blockIdx.x].sum = top == -INFINITY && all == all ? 0.0 : all;
  }
  // (a second time from memory: a second use of the logits in registers costs the main path a wave or two a SIMD)
  const int cnt = collect_fewer<CAP, WAVES>(depth, lk, &rc, ct, [&](double lowest, unsigned) {
    const X bound = at_least<X>(lowest);
#pragma unroll 4
    for (int e = base + tid; e < base + THREADS * U; e += THREADS) {
      if (e >= a.V) break;
      X xe = (X)to_f(lrow[e]);
      if (BIAS) xe = brow[e] == -INFINITY ? (X)-INFINITY : xe + (X)brow[e];
      if (!(xe < bound)) put(xe, e);
    }
  });
  if (cnt <= CAP) {
    rank_collected<WAVES>(lk, li, cnt, depth, [&](int r, long long k, int p) {
      pk[mine + (long long)r * lists] = k;
      pi[mine + (long long)r * lists] = p;
    });
    for (int r = cnt + tid; r < depth; r += THREADS) pk[mine + (long long)r * lists] = KEY_NONE;
    return;
  }
  // more equal logits than the list holds: one after the other
  long long prev = KEY_NAN;
  int place = -1;
  __shared__ long long sk[4];
  __shared__ int sp[4];
  for (int r = 0; r < depth; ++r) {
    long long k = KEY_NONE;
    int p = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const double xi = (double)x[i];
      const long long ki = xi == -INFINITY ? KEY_NONE : key_of(xi);
      const int q = In::place(base, i);
      if (ki != KEY_NONE && better(prev, place, ki, q) && better(ki, q, k, p)) { k = ki; p = q; }
    }
    block_best<WAVES>(k, p, sk, sp);
    if (tid == 0) {
      pk[mine + (long long)r * lists] = k;
      pi[mine + (long long)r * lists] = p;
    }
    prev = k;
    place = p;
  }
}

// The last score kept, `kth`, may belong to more candidates than the slices' lists hold.  From slot `slot` on (those before it
// hold larger scores): the group's candidates of exactly this score, in order, from the logits, up to the last slot.  found: 4
// words of LDS.
template <typename T>
__device__ __forceinline__ void repair_ties(const SelectArgs& a, int b, long long kth, int slot, const double* lse,
                                            const float* sc, const int* fc, int* found) {
  constexpr int R = 4;                       // tokens of a thread's turn
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int w = 0; w < a.W && slot < a.n; ++w) {
    if (fc[w] >= 0 || broken((double)sc[w], lse[w])) {   // one candidate
      const long long key = fc[w] < 0 ? KEY_NAN : sc[w] == -INFINITY ? KEY_NONE : key_of((double)sc[w]);
      if (key == kth) {
        if (tid == 0) write_slot(a, b, slot, key, w * a.V + (fc[w] < 0 ? 0 : fc[w]));
        ++slot;
      }
      continue;
    }
    const T* row = (const T*)a.logits + (long long)b * a.sb + (long long)w * a.sw;
    const float* bias = a.bias ? a.bias + (long long)b * a.bb + (long long)w * a.bw : nullptr;
    for (int v0 = 0; v0 < a.V && slot < a.n; v0 += 256 * R) {
      float raw[R], add[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int v = v0 + 256 * i + tid;
        raw[i] = to_f(row[v < a.V ? v : a.V - 1]);
        add[i] = bias ? bias[v < a.V ? v : a.V - 1] : 0.f;
      }
      unsigned hits = 0;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const double x = add[i] == -INFINITY ? -INFINITY : (double)raw[i] + (double)add[i];
        const bool in = v0 + 256 * i + tid < a.V && !(x == -INFINITY);
        hits |= in && key_of((double)sc[w] + (x - lse[w])) == kth ? 1u << i : 0u;
      }
      if (!__syncthreads_or((int)hits)) continue;
      for (int i = 0; i < R; ++i) {
        const bool hit = hits >> i & 1;
        const unsigned long long m = __ballot(hit);
        if (lane == 0) found[wave] = __popcll(m);
        __syncthreads();
        int at = slot + __popcll(m & ((1ull << lane) - 1)), all = 0;
        for (int q = 0; q < 4; ++q) {
          at += q < wave ? found[q] : 0;
          all += found[q];
        }
        if (hit && at < a.n) write_slot(a, b, at, kth, w * a.V + v0 + 256 * i + tid);
        slot += all;
        __syncthreads();
      }
    }
  }
}

// Second pass, one workgroup a group: the beams' log-sum-exps from the slices', then the n best of the slices' lists.  The
// lists are sorted; the first 256 E entries by depth (all lists' best, all lists' second ...) are in registers before
// anything else is done and give the bound, and lists go on beyond them only where their entries still reach it.  A chain
// of latencies, 7-8 us (with the lists' heads alone as the bound 120 us at 32 beams x 2 slices, 32 kept).
template <typename T>
__global__ void __launch_bounds__(256)
k_select_merge(SelectArgs a, int splits, int depth, int g_log2, const SlicePart* __restrict__ part, const long long* __restrict__ pk,
               const int* __restrict__ pi) {
  constexpr int E = 4;
  __shared__ double lse[SEL_MAX_N];
  __shared__ float sc[SEL_MAX_N];
  __shared__ int fc[SEL_MAX_N];
  __shared__ unsigned ct[5][4];
  __shared__ int live[SEL_MAX_N];
  __shared__ short open[256 * E];            // lists that go on beyond the registers
  __shared__ int rc, above, n_open, reach;   // reach: the last entry collected there
  __shared__ long long deep, kth;            // best of the lists' last entries; the last score kept
  __shared__ long long lk[SEL_CAP + RANK_PAD];
  __shared__ int li[SEL_CAP + RANK_PAD];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int lists = a.W * splits, total = lists * depth;
  const long long* keys = pk + (long long)b * total;
  const int* places = pi + (long long)b * total;
  long long k[E];
  int p[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int e = tid + 256 * i;
    k[i] = keys[e < total ? e : 0];
    p[i] = places[e < total ? e : 0];
  }
  // 2^g_log2 lanes a beam
  const int g = 1 << g_log2, j = tid & (g - 1);
  for (int w0 = 0; w0 < a.W; w0 += 256 >> g_log2) {
    const int w = w0 + (tid >> g_log2);
    const bool in = w < a.W;
    const long long row = (long long)b * a.W + (in ? w : 0);
    const long long f = a.forced ? a.forced[row] : -1;
    const float score = a.scores[row];
    double top = -INFINITY, sum = 0.0;
    const SlicePart* q = part + row * splits;
    if (f < 0)
      for (int i = j; i < splits; i += g) top = fmax(top, q[i].top);
    top = group_max(top, g);
    if (f < 0)
      for (int i = j; i < splits; i += g) sum += q[i].top == -INFINITY ? q[i].sum : q[i].sum * exp_neg(q[i].top - top);
    sum = group_sum(sum, g);
    if (in && j == 0) {
      lse[w] = top + log(sum);
      sc[w] = score;
      fc[w] = f < 0 ? -1 : (f < a.V ? (int)f : a.V - 1);
    }
  }
  if (tid == 0) {
    rc = above = n_open = 0;
    reach = -1;
    deep = kth = KEY_NONE;
  }
  __syncthreads();
  // beams whose lists count: not dead, no other candidate in place of the list's.  Where the registers do not hold all entries the
  // other beams' are left out (at a search's first step one beam is alive): else live[w] = w, or -1.
  const bool listed = tid < a.W && fc[tid] < 0 && !(sc[tid] == -INFINITY) && !broken((double)sc[tid], lse[tid]);
  int in_use = lists;                        // lists
  bool all = true;
  if (total > 256 * E) {
    const unsigned long long m = __ballot(listed);
    if ((tid & 63) == 0) ct[0][tid >> 6] = __popcll(m);
    __syncthreads();
    int at = __popcll(m & ((1ull << (tid & 63)) - 1));
    for (int i = 0; i < tid >> 6; ++i) at += ct[0][i];
    if (listed) live[at] = tid;
    in_use = (int)(ct[0][0] + ct[0][1] + ct[0][2] + ct[0][3]) * splits;
    all = in_use == lists;
  } else if (tid < a.W) {
    live[tid] = listed ? tid : -1;
  }
  __syncthreads();
  const int used = in_use * depth;           // entries
  // the entry at depth r of list l; e = r in_use + l
  auto fetch = [&](int r, int l, bool load, long long& kx, int& px, int& w) {
    const int i = l / splits;
    w = live[i];
    if (!load) return;
    const int o = r * lists + w * splits + (l - i * splits);
    kx = keys[o];
    px = places[o];
  };
  auto candidate = [&](int w, long long& kx, int& px) {
    if (w < 0) kx = KEY_NONE;
    if (kx == KEY_NONE) return;
    const double c = (double)sc[w] + (value_of(kx) - lse[w]);
    kx = c == -INFINITY ? KEY_NONE : key_of(c);
    px += w * a.V;
  };
  unsigned u[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int e = tid + 256 * i;
    int w = -1;
    if (e < used) fetch(e / in_use, e % in_use, !all, k[i], p[i], w);
    candidate(w, k[i], p[i]);
    u[i] = k[i] == KEY_NONE ? 0u : (unsigned)(k[i] >> 32) ^ 0x80000000u;
  }
  const unsigned first_bound = block_kth<E>(u, a.n, ct);
  // Entries beyond the registers: of the lists whose entry in the registers' last whole row reaches the bound (of all lists, if
  // there is no whole row), row by row as far as one of them does.  (One thread walking down a list: 40 us where one beam of 60
  // has most of the best; all lists row by row: 50 us for 16 x 64 x 20000, 64 kept.)
  const int rows = used > 256 * E ? 256 * E / in_use : 0;
  if (rows) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = tid + 256 * i - (rows - 1) * in_use;
      if (e >= 0 && e < in_use && u[i] && u[i] >= first_bound) open[atomicAdd(&n_open, 1)] = (short)e;
    }
    __syncthreads();
  }
  const int wide = rows ? n_open : in_use, more = used > 256 * E ? wide * (depth - rows) : 0;
  // e: place among the entries beyond the registers, -1 for others
  auto take = [&](int e, bool at_end, long long kx, int px, unsigned bound) {
    if (kx == KEY_NONE || ((unsigned)(kx >> 32) ^ 0x80000000u) < bound) return;
    if (at_end) atomicMax(&deep, kx);
    if (e >= 0) atomicMax(&reach, e);
    const int q = atomicAdd(&rc, 1);
    if (q < SEL_CAP) { lk[q] = kx; li[q] = px; }
  };
  auto alone = [&]() {                       // the one candidate of a forced or broken beam
    if (fc[tid] < 0) return broken((double)sc[tid], lse[tid]) ? KEY_NAN : KEY_NONE;
    return sc[tid] == -INFINITY ? KEY_NONE : key_of((double)sc[tid]);
  };
  auto collect = [&](double, unsigned bound) {
#pragma unroll
    for (int i = 0; i < E; ++i) take(-1, tid + 256 * i >= used - in_use, k[i], p[i], bound);
    if (tid < a.W && !listed) take(-1, false, alone(), tid * a.V + (fc[tid] < 0 ? 0 : fc[tid]), bound);
    for (int base = 0; base < more; base += 256 * E) {
      __syncthreads();
      if (base > reach + wide) break;
      __syncthreads();
      long long kx[E];
      int px[E], w[E], r[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int e = base + tid + 256 * i < more ? base + tid + 256 * i : base, l = rows ? open[e % wide] : e % wide;
        r[i] = rows + e / wide;
        fetch(r[i], l, true, kx[i], px[i], w[i]);
        if (base + tid + 256 * i >= more) kx[i] = KEY_NONE;
        else if (r[i] * in_use + l < 256 * E) {      // is in the registers
          kx[i] = KEY_NONE;
          atomicMax(&reach, e);
        }
      }
#pragma unroll
      for (int i = 0; i < E; ++i) {
        candidate(w[i], kx[i], px[i]);
        take(base + tid + 256 * i, r[i] == depth - 1, kx[i], px[i], bound);
      }
    }
  };
  collect(0.0, first_bound);
  __syncthreads();
  const int cnt = collect_fewer<SEL_CAP, 4>(a.n, lk, &rc, ct, collect);
  long long last = KEY_NONE;                 // the last score kept and the first slot that holds it
  int first = 0;
  if (cnt <= SEL_CAP) {
    rank_collected(lk, li, cnt, a.n, [&](int r, long long ke, int pe) {
      write_slot(a, b, r, ke, pe);
      if (r == a.n - 1) kth = ke;
    });
    for (int r = cnt + tid; r < a.n; r += 256) write_dead_slot(a, b, r);
    if (deep == KEY_NONE) return;
    __syncthreads();
    last = kth;
    if (deep < last) return;
    for (int e = tid; e < cnt; e += 256)
      if (lk[e] > last) atomicAdd(&above, 1);
    __syncthreads();
    first = above;
  } else {
    // more ties than the list holds: one after the other
    long long prev = KEY_NAN;
    int place = -1;
    __shared__ long long sk[4];
    __shared__ int sp[4];
    for (int r = 0; r < a.n; ++r) {
      long long kb = KEY_NONE;
      int pb = 0x7fffffff;
      auto look = [&](long long ke, int pe) {
        if (ke != KEY_NONE && better(prev, place, ke, pe) && better(ke, pe, kb, pb)) { kb = ke; pb = pe; }
      };
      for (int e = tid; e < used; e += 256) {
        long long ke;
        int pe, w;
        fetch(e / in_use, e % in_use, true, ke, pe, w);
        candidate(w, ke, pe);
        look(ke, pe);
      }
      if (tid < a.W && !listed) look(alone(), tid * a.V + (fc[tid] < 0 ? 0 : fc[tid]));
      block_best(kb, pb, sk, sp);
      if (tid == 0) {
        if (kb != KEY_NONE) write_slot(a, b, r, kb, pb); else write_dead_slot(a, b, r);
      }
      first = kb == prev ? first : r;
      prev = kb;
      place = pb;
    }
    last = prev;
  }
  if (last != KEY_NONE && deep >= last) repair_ties<T>(a, b, last, first, lse, sc, fc, (int*)ct);
}

inline int list_depth(int n) { return n < SEL_MAX_N ? n + 1 : SEL_MAX_N; }   // entries of a slice's list

// How a call is split.  One wave a group up to 8 candidates a lane (64 x 16 x 21).  A beam's lanes are at most a wave: three or
// four beams take one workgroup of four waves, up to 32 a lane; more of them four waves up to 8, else 8 or (more than eight beams)
// 16 waves up to 16 (8 x 6 x 882: 12 us with 8 waves, 15 with 16, 14 with 4).  Else slices and a second pass: a row of up to 512 or
// 1024 logits for one wave (250 x 20 x 700 and more; 250 x 16 x 700 took 28 us so, with four waves 33), or 256 u logits for four:
// u = 32 where rows hold two such slices and there are 300 (512 rows of 31839 fp32: 33 us with 32, 44 with 8; 32 rows: 15.6 and
// 14.0; 2048 rows of 9000 bf16: 75 and 53).
struct SelectPlan {
  int waves, g_log2, m;  // waves a group, 0 = slices; 2^g_log2 lanes a beam; candidates a lane
  int u, per, splits;    // slices: values a thread holds, waves a slice, slices a beam
};
inline SelectPlan select_plan(long long B, int W, int V) {
  SelectPlan p = {};
  for (int waves : {1, 4, 8, 16}) {
    int gl = 6;
    while (gl > 0 && ((64 * waves) >> gl) < W) --gl;
    const int m = (V + (1 << gl) - 1) >> gl, most = waves == 1 ? 8 : waves == 4 ? (W <= 2 ? 0 : W <= 4 ? 32 : 8) : W <= waves / 2 ? 0 : 16;
    if (((64 * waves) >> gl) >= W && m <= most) {
      p.waves = waves;
      p.g_log2 = gl;
      p.m = m;
      return p;
    }
  }
  p.per = V <= 1024 ? 1 : 4;
  if (p.per == 1) p.u = V <= 512 ? 8 : 16;
  else p.u = V >= 2 * 256 * SEL_U && B * W * (V / (256 * SEL_U)) >= SEL_LONG ? SEL_U : 8;
  p.splits = (V + 64 * p.per * p.u - 1) / (64 * p.per * p.u);
  return p;
}

template <typename T>
int launch_select(const SelectArgs& a, const SelectPlan& p, void* ws, hipStream_t st) {
  if (p.waves == 1) {
    const dim3 grid(a.B), block(64);
    if (p.m <= 2) hipLaunchKernelGGL((k_select_small<T, 2>), grid, block, 0, st, a, p.g_log2);
    else if (p.m <= 4) hipLaunchKernelGGL((k_select_small<T, 4>), grid, block, 0, st, a, p.g_log2);
    else hipLaunchKernelGGL((k_select_small<T, 8>), grid, block, 0, st, a, p.g_log2);
    MPNN_LAUNCH_CHECK();
  }
  if (p.waves) {
    const dim3 grid(a.B), block(64 * p.waves);
    if (p.waves == 16 && p.m <= 8) hipLaunchKernelGGL((k_select_group<T, 8, 16>), grid, block, 0, st, a, p.g_log2);
    else if (p.waves == 8 && p.m <= 8) hipLaunchKernelGGL((k_select_group<T, 8, 8>), grid, block, 0, st, a, p.g_log2);
    else if (p.waves == 8) hipLaunchKernelGGL((k_select_group<T, 16, 8>), grid, block, 0, st, a, p.g_log2);
    else if (p.waves == 16) hipLaunchKernelGGL((k_select_group<T, 16, 16>), grid, block, 0, st, a, p.g_log2);
    else if (p.m <= 8) hipLaunchKernelGGL((k_select_group<T, 8, 4>), grid, block, 0, st, a, p.g_log2);
    else if (p.m <= 16) hipLaunchKernelGGL((k_select_group<T, 16, 4>), grid, block, 0, st, a, p.g_log2);
    else hipLaunchKernelGGL((k_select_group<T, 32, 4>), grid, block, 0, st, a, p.g_log2);
    MPNN_LAUNCH_CHECK();
  }
  const long long parts = (long long)a.B * a.W * p.splits;
  SlicePart* part = (SlicePart*)ws;
  long long* pk = (long long*)(part + parts);
  const int depth = list_depth(a.n);
  int* pi = (int*)(pk + parts * depth);
  const dim3 grid((unsigned)parts), block(256);
#define MPNN_SLICE(U, WAVES)                                                                                             \
  do {                                                                                                                   \
    if (a.bias)                                                                                                          \
      hipLaunchKernelGGL((k_select_slice<T, U, true, WAVES>), grid, dim3(64 * WAVES), 0, st, a, p.splits, depth, part,   \
                         pk, pi);                                                                                        \
    else                                                                                                                 \
      hipLaunchKernelGGL((k_select_slice<T, U, false, WAVES>), grid, dim3(64 * WAVES), 0, st, a, p.splits, depth, part,  \
                         pk, pi);                                                                                        \
  } while (0)
  if (p.per == 1 && p.u == 8) MPNN_SLICE(8, 1);
  else if (p.per == 1) MPNN_SLICE(16, 1);
  else if (p.u == 8) MPNN_SLICE(8, 4);
  else MPNN_SLICE(SEL_U, 4);
#undef MPNN_SLICE
  int gl = 0;                               // lanes that share a beam's slices
  while (gl < 6 && (1 << gl) < p.splits && (long long)a.W << (gl + 1) <= 256) ++gl;
  hipLaunchKernelGGL((k_select_merge<T>), dim3(a.B), block, 0, st, a, p.splits, depth, gl, part, pk, pi);
  MPNN_LAUNCH_CHECK();
}

// ---------------------------------------------------------------------------------------------------------------
// States: a wave owns 64 columns of up to 16 bytes of one group - the same bytes of all its beams.  It reads the columns of
// the rows that another row becomes, all of them before the first write, then writes each row that changes.  A column belongs
// to one lane from first read to last write, so the update is in place without a barrier.  Bound by the bytes of the rows
// that move: a row that stays is not written, one that nobody else becomes is not read.  Up to 64 beams the rows wait in
// registers (all reads in flight at once, and more waves a CU than when they wait in LDS: 36 us against 56 for 16 structures
// x 16 beams x 512 residues, half of them decided), beyond that in LDS.  234 us for 1.05 GB of caches of four beams; of 1.6 GB of
// rows that move 309-350 us with 16 to 64 beams (5.3 to 4.9 TB/s), but 868, 1440 and 2566 us with 65, 128 and 256: 33 to 64 KB
// of LDS a wave leave two to four waves a CU, with eight rows of 4 or 8 bytes a lane in flight each.
// ---------------------------------------------------------------------------------------------------------------
constexpr int RO_MAX = 32;
struct ReorderTable {
  mpnn_beam_state s[RO_MAX];
  unsigned char vec_log2[RO_MAX];   // bytes of a column
};

// OR over the wave, uniform: rotations within rows of 16 lanes, then one lane of each row
__device__ __forceinline__ unsigned wave_or(unsigned x) {
  x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false);
  x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, false);
  x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, false);
  x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, false);
  return (unsigned)(__builtin_amdgcn_readlane((int)x, 0) | __builtin_amdgcn_readlane((int)x, 16) |
                    __builtin_amdgcn_readlane((int)x, 32) | __builtin_amdgcn_readlane((int)x, 48));
}

// up to R <= 64 beams.  from: lane w holds the row that row w becomes, -1 where it stays
template <typename V, int R>
__device__ __forceinline__ void reorder_in_registers(char* data, long long sw, bool live, int from) {
  V r[R];
#pragma unroll
  for (int p = 0; p < R; ++p)
    if (__ballot(from == p) && live) r[p] = *(const V*)(data + p * sw);
#pragma unroll
  for (int p = 0; p < R; ++p)
#pragma unroll 1
    for (unsigned long long kids = __ballot(from == p); kids; kids &= kids - 1)
      if (live) *(V*)(data + __builtin_ctzll(kids) * sw) = r[p];
}

// any number of beams.  from[k]: lane w holds the row that row 64 k + w becomes
template <typename V>
__device__ __forceinline__ void reorder_through_lds(char* data, long long sw, int W, bool live, const int (&from)[4], V* lds) {
  const int lane = threadIdx.x;
  unsigned long long needed[4] = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (64 * k >= W) break;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (64 * m >= W) break;
      const unsigned lo = wave_or(from[k] >> 5 == 2 * m ? 1u << (from[k] & 31) : 0u);
      const unsigned hi = wave_or(from[k] >> 5 == 2 * m + 1 ? 1u << (from[k] & 31) : 0u);
      needed[m] |= (unsigned long long)lo | (unsigned long long)hi << 32;
    }
  }
  // a lane without a column (or whose position stays) goes on with the others: it holds parents that they ask it for
#pragma unroll
  for (int k = 0; k < 4; ++k)
    for (int w0 = 64 * k; w0 < W && w0 < 64 * k + 64; w0 += 8) {   // eight rows in flight
      const unsigned bits = (unsigned)(needed[k] >> (w0 & 63)) & 0xff;
      if (!bits) continue;
      V r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((bits >> i & 1) && live) r[i] = *(const V*)(data + (w0 + i) * sw);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((bits >> i & 1) && live) lds[(w0 + i) * 64 + lane] = r[i];
    }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    for (int w0 = 64 * k; w0 < W && w0 < 64 * k + 64; w0 += 8) {
      V r[8];
      int f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = __builtin_amdgcn_readlane(from[k], (w0 + i) & 63);
        r[i] = lds[(f[i] < 0 ? 0 : f[i]) * 64 + lane];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (f[i] >= 0 && live) *(V*)(data + (w0 + i) * sw) = r[i];
    }
}

// R: rows held in registers; 0: through LDS
template <int R>
__global__ void __launch_bounds__(64)
k_beam_reorder(ReorderTable t, const long long* __restrict__ parent, int W, int length_all, const int* __restrict__ length,
               const int* __restrict__ rank) {
  extern __shared__ char lds[];
  const mpnn_beam_state s = t.s[blockIdx.z];
  const int b = blockIdx.y, vl = t.vec_log2[blockIdx.z];
  const unsigned per = (unsigned)(s.run >> vl);
  const unsigned long long col = (unsigned long long)blockIdx.x * 64 + threadIdx.x;
  const unsigned mid = (unsigned)(col / per), off = (unsigned)(col % per);
  bool live = col < (unsigned long long)per * s.n_mid;
  if (live && (length || length_all >= 0)) {
    const int len = length ? length[b] : length_all;
    live = (rank ? rank[(long long)b * s.n_mid + mid] : (int)mid) < len;
  }
  if (!__any(live)) return;
  const long long* p = parent + (long long)b * W;
  int from[4] = {-1, -1, -1, -1};
#pragma unroll
  for (int k = 0; k < (R ? 1 : 4); ++k) {
    const int w = 64 * k + threadIdx.x;
    const long long q = w < W ? p[w] : -1;
    from[k] = q == w || q < 0 || q >= W ? -1 : (int)q;
  }
  char* data = (char*)s.data + b * s.stride_group + mid * s.stride_mid + ((long long)off << vl);
#define MPNN_COLUMNS(V)                                                            \
  do {                                                                             \
    if (R) reorder_in_registers<V, R ? R : 1>(data, s.stride_beam, live, from[0]); \
    else reorder_through_lds(data, s.stride_beam, W, live, from, (V*)lds);         \
  } while (0)
  if (vl == 4 && R <= 32) MPNN_COLUMNS(f32x4);
  else if (vl == 3) MPNN_COLUMNS(unsigned long long);
  else if (vl == 2) MPNN_COLUMNS(unsigned);
  else if (vl == 1) MPNN_COLUMNS(unsigned short);
  else MPNN_COLUMNS(unsigned char);
#undef MPNN_COLUMNS
}

// widest access every row of the state allows (its address, strides and run are multiples of it), as a power of two
inline int state_vec_log2(const mpnn_beam_state& s, int W) {
  unsigned long long bits = (unsigned long long)(uintptr_t)s.data | (unsigned long long)s.stride_group |
                            (unsigned long long)s.stride_beam | (unsigned long long)s.run;
  if (s.n_mid > 1) bits |= (unsigned long long)s.stride_mid;
  int vl = 4;
  while (vl > 0 && (bits & ((1u << vl) - 1))) --vl;
  if (W > 32 && W <= 64 && vl > 3) vl = 3;                   // 64 rows of 16 bytes are all the registers a lane has
  while (vl > 0 && W > 64 && (64 << vl) * W > 65536) --vl;   // the LDS a wave may hold
  return vl;
}

// ---------------------------------------------------------------------------------------------------------------
// The model's own search: logits of the residues of a step, and the chosen letters' way into the decoder's rows.
// ---------------------------------------------------------------------------------------------------------------

// logits[q][v] = W_out hV[list[q]] + b for the listed residues: 16 of them a wave, one column each
__global__ void __launch_bounds__(64)
k_beam_logits(const float* __restrict__ hV, const f32x4* __restrict__ Wp, const float* __restrict__ bias, int n_letters,
              const int* __restrict__ list, int n_list, float* __restrict__ logits) {
  const int lane = threadIdx.x, g = lane >> 4, q = blockIdx.x * 16 + (lane & 15);
  const bool live = q < n_list;
  const int nd = list[live ? q : n_list - 1];
  f32x4 h[MPNN_NT][1], y[2][1];
#pragma unroll
  for (int t = 0; t < MPNN_NT; ++t) h[t][0] = *reinterpret_cast<const f32x4*>(hV + (size_t)nd * MPNN_H + 16 * t + 4 * g);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int letter = 16 * t + 4 * g + r;
      y[t][0][r] = letter < n_letters ? bias[letter] : 0.f;
    }
  tile_gemm<1, MPNN_NT, 0, 2>(Wp, lane, h, y);
  if (!live) return;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int letter = 16 * t + 4 * g + r;
      if (letter < n_letters) logits[(size_t)q * n_letters + letter] = y[t][0][r];
    }
}

struct PlaceArgs {
  const int* list;             // residue id of (group, beam)
  const long long* parent;
  const long long* token;
  const float* logits;         // [group][beam][n_letters]
  int W, n_letters, n_layers;
  float* A[4];                 // gathered rows of each decoder layer
  int lda[4], offA[4];
  const float* TS;             // letters' terms, 128 columns a layer
  int ld_ts;
  long long* S;
  float* log_probs;
};

// The residue just decided, beam by beam: its gathered rows become the parent's plus the letter's term (block y < n_layers),
// its letter and log-probs are written down (the last block).  Four waves share a layer's rows, sixteen at a time each, so
// that up to 64 beams cost two round trips to memory; every row is in LDS before the first is written.
__global__ void __launch_bounds__(256)
k_beam_place(PlaceArgs a) {
  extern __shared__ char lds[];
  const int b = blockIdx.x, l = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, W = a.W;
  const long long* parent = a.parent + (long long)b * W;
  const long long* token = a.token + (long long)b * W;
  const int* list = a.list + b * W;
  const int mine = lane < W ? lane : 0;          // W <= 64: a lane's beam
  const int at = list[mine], from = (int)parent[mine], letter = (int)token[mine];
  if (l < a.n_layers) {
    float2* row = reinterpret_cast<float2*>(lds);
    float* A = a.A[l] + a.offA[l] + 2 * lane;
    const float* T = a.TS + l * MPNN_H + 2 * lane;
    float2 v[16], t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int w = wave + 4 * i;
      if (w < W) {
        v[i] = *reinterpret_cast<const float2*>(A + (size_t)__builtin_amdgcn_readlane(at, w) * a.lda[l]);
        t[i] = *reinterpret_cast<const float2*>(T + (size_t)__builtin_amdgcn_readlane(letter, w) * a.ld_ts);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (wave + 4 * i < W) row[(wave + 4 * i) * 64 + lane] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int w = wave + 4 * i;
      if (w < W) {
        float2 x = row[__builtin_amdgcn_readlane(from, w) * 64 + lane];
        x.x += t[i].x;
        x.y += t[i].y;
        *reinterpret_cast<float2*>(A + (size_t)__builtin_amdgcn_readlane(at, w) * a.lda[l]) = x;
      }
    }
    return;
  }
  // four lanes a beam: 64 beams at once
  const int w = threadIdx.x >> 2, q = threadIdx.x & 3;
  const bool live = w < W;
  const int p = live ? (int)parent[w] : 0;
  const float* x = a.logits + ((long long)b * W + p) * a.n_letters;
  float y[8], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = q + 4 * i < a.n_letters ? x[q + 4 * i] : -INFINITY;
    top = fmaxf(top, y[i]);
  }
  top = fmaxf(top, __shfl_xor(top, 1));
  top = fmaxf(top, __shfl_xor(top, 2));
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += expf(y[i] - top);
  sum += __shfl_xor(sum, 1);
  sum += __shfl_xor(sum, 2);
  if (!live) return;
  const float lse = top + logf(sum);
  float* lp = a.log_probs + (size_t)list[w] * a.n_letters;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (q + 4 * i < a.n_letters) lp[q + 4 * i] = y[i] - lse;
  if (q == 0) a.S[list[w]] = token[w];
}

}  // namespace

extern "C" long long mpnn_beam_select_workspace(int dtype, int n_groups, int n_beams, int n_tokens, int n_out) {
  if (dtype < 0 || dtype > 2 || n_groups <= 0 || n_beams <= 0 || n_tokens <= 0 || n_out <= 0 || n_out > SEL_MAX_N) return -1;
  const SelectPlan p = select_plan(n_groups, n_beams, n_tokens);
  if (p.waves) return 0;
  return (long long)n_groups * n_beams * p.splits * ((long long)sizeof(SlicePart) + 12LL * list_depth(n_out));
}

extern "C" int mpnn_beam_select(const void* logits, int dtype, long long stride_group, long long stride_beam,
                                const float* scores, const float* bias, long long bias_group, long long bias_beam,
                                const int64_t* forced, int n_groups, int n_beams, int n_tokens, int n_out,
                                float* out_scores, int64_t* parent, int64_t* token, void* workspace,
                                long long workspace_bytes, void* stream) {
  MPNN_CHECK_ARG(logits && scores && out_scores && parent && token, "mpnn_beam_select: null pointer");
  MPNN_CHECK_ARG(dtype >= 0 && dtype <= 2, "mpnn_beam_select: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
  MPNN_CHECK_ARG(n_groups > 0 && n_beams > 0 && n_beams <= SEL_MAX_N && n_out > 0 && n_out <= SEL_MAX_N && n_tokens > 0 &&
                     n_tokens <= (1 << 22),
                 "mpnn_beam_select: bad sizes (at most 256 beams and hypotheses kept, at most 2^22 tokens)");
  MPNN_CHECK_ARG(((uintptr_t)logits & (dtype == 0 ? 3 : 1)) == 0, "mpnn_beam_select: logits are not aligned to their type");
  const long long need = mpnn_beam_select_workspace(dtype, n_groups, n_beams, n_tokens, n_out);
  MPNN_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                 "mpnn_beam_select: workspace missing, too small (mpnn_beam_select_workspace) or not 16-byte aligned");
  const SelectPlan p = select_plan(n_groups, n_beams, n_tokens);
  // a launch has less than 2^32 threads; entries of a group's lists are counted in 32 bits
  MPNN_CHECK_ARG((long long)n_groups < (1LL << 32) / (p.waves ? 64 * p.waves : 256) &&
                     (p.waves || (long long)n_groups * n_beams * p.splits < (1LL << 24)) &&
                     (long long)n_beams * (p.waves ? 1 : p.splits) * list_depth(n_out) < (1LL << 31),
                 "mpnn_beam_select: too many groups for one launch");
  SelectArgs a = {logits, stride_group, stride_beam, scores, bias, bias_group, bias_beam, (const long long*)forced,
                  n_groups, n_beams, n_tokens, n_out, out_scores, (long long*)parent, (long long*)token};
  if (dtype == 0) return launch_select<float>(a, p, workspace, (hipStream_t)stream);
  if (dtype == 1) return launch_select<__hip_bfloat16>(a, p, workspace, (hipStream_t)stream);
  return launch_select<__half>(a, p, workspace, (hipStream_t)stream);
}

extern "C" int mpnn_beam_reorder(int n, const mpnn_beam_state* states, const int64_t* parent, int n_groups, int n_beams,
                                 int length_all, const int32_t* length, const int32_t* rank, void* stream) {
  MPNN_CHECK_ARG(n > 0 && states && parent, "mpnn_beam_reorder: null pointer");
  MPNN_CHECK_ARG(n_groups > 0 && n_groups <= 65535 && n_beams > 0 && n_beams <= 256,
                 "mpnn_beam_reorder: bad sizes (at most 65535 groups and 256 beams)");
  MPNN_CHECK_ARG(!rank || length || length_all >= 0, "mpnn_beam_reorder: rank needs a length");
  for (int i = 0; i < n; ++i) {
    const mpnn_beam_state& s = states[i];
    MPNN_CHECK_ARG(s.data && s.n_mid > 0 && s.run > 0 && (n_beams == 1 || s.stride_beam != 0) &&
                       (n_groups == 1 || s.stride_group != 0) && (s.n_mid == 1 || s.stride_mid != 0),
                   "mpnn_beam_reorder: a state is empty or its rows share memory");
    const int vl = state_vec_log2(s, n_beams);
    MPNN_CHECK_ARG((s.run >> vl) < (1LL << 32) && ((unsigned long long)(s.run >> vl) * s.n_mid + 63) / 64 < (1ULL << 26),
                   "mpnn_beam_reorder: a state is too large for one launch");
  }
  for (int i0 = 0; i0 < n; i0 += RO_MAX) {
    ReorderTable t;
    const int m = n - i0 < RO_MAX ? n - i0 : RO_MAX;
    unsigned long long cols = 0;
    int widest = 0;
    for (int i = 0; i < m; ++i) {
      const mpnn_beam_state& s = states[i0 + i];
      const int vl = state_vec_log2(s, n_beams);
      t.s[i] = s;
      t.vec_log2[i] = (unsigned char)vl;
      widest = vl > widest ? vl : widest;
      const unsigned long long c = (unsigned long long)(s.run >> vl) * (unsigned long long)s.n_mid;
      cols = c > cols ? c : cols;
    }
    const dim3 grid((unsigned)((cols + 63) / 64), (unsigned)n_groups, (unsigned)m), block(64);
#define MPNN_REORDER(R)                                                                                                  \
  hipLaunchKernelGGL((k_beam_reorder<R>), grid, block, R ? 0 : (size_t)(64 << widest) * n_beams, (hipStream_t)stream, t, \
                     (const long long*)parent, n_beams, length_all, length, rank)
    if (n_beams <= 4) MPNN_REORDER(4);
    else if (n_beams <= 16) MPNN_REORDER(16);
    else if (n_beams <= 32) MPNN_REORDER(32);
    else if (n_beams <= 64) MPNN_REORDER(64);
    else MPNN_REORDER(0);
#undef MPNN_REORDER
  }
  MPNN_LAUNCH_CHECK();
}

// The whole search in one call: per position of the decoding order the decoder layers on the groups' current residues, their
// logits, the choice, the states of the residues decided earlier following their parents, and the chosen letters' terms.
static int beam_run(bool f16, const float* hE_frag, const float* PVenc, int ldenc, const int32_t* rank,
                    const int32_t* E_idx32, const float* mask, const float* edge_mask, const int32_t* node_list,
                    const int64_t* forced, int n_groups, int n_beams, int L, int K, const mpnn_level_layer* layers,
                    int n_layers, const float* Wlogit_packed, const float* blogit, const float* logit_bias, int n_letters,
                    const float* TS, int ld_ts, float* gsum, float* logits, float* scores, int64_t* parent, int64_t* token,
                    int64_t* S, float* log_probs, void* stream) {
  MPNN_CHECK_ARG(hE_frag && PVenc && rank && E_idx32 && mask && node_list && forced && layers && Wlogit_packed && blogit && TS &&
                     logits && scores && parent && token && S && log_probs,
                 "mpnn_beam_run: null pointer");
  MPNN_CHECK_ARG(n_groups > 0 && n_groups <= 65535 && n_beams > 0 && n_beams <= 64 && L > 0 && K >= 1 && K <= 64 &&
                     n_layers >= 1 && n_layers <= 4 && n_letters >= 1 && n_letters <= 32 && (K <= 48 || gsum) &&
                     (long long)n_groups * n_beams * L < (1LL << 31),
                 "mpnn_beam_run: bad sizes (at most 64 beams, K <= 64, 1..4 layers, 32 letters; gsum for K > 48)");
  const long long N = (long long)n_groups * L;
  const int n_list = n_groups * n_beams;
  PlaceArgs place = {};
  mpnn_beam_state states[6];
  for (int l = 0; l < n_layers; ++l) {
    const mpnn_level_layer& y = layers[l];
    MPNN_CHECK_ARG(l == 0 || (y.hV_in == layers[l - 1].hV_out && layers[l - 1].nproj >= 2),
                   "mpnn_beam_run: layer l must read the hV rows (and Pa | A projections) layer l-1 writes");
    MPNN_CHECK_ARG((y.lda & 3) == 0 && (y.offA & 3) == 0, "mpnn_beam_run: row strides and offsets are multiples of 4 floats");
    place.A[l] = y.RowA;
    place.lda[l] = y.lda;
    place.offA[l] = y.offA;
    // residue (w, b, i) is row w N + b L + i
    states[l] = {y.RowA + y.offA, 4LL * y.lda * L, 4LL * y.lda * N, 4LL * y.lda, 4 * MPNN_H, L};
  }
  MPNN_CHECK_ARG(layers[n_layers - 1].nproj == 0, "mpnn_beam_run: the last decoder layer carries no projections");
  states[n_layers] = {S, 8LL * L, 8LL * N, 8, 8, L};
  states[n_layers + 1] = {log_probs, 4LL * n_letters * L, 4LL * n_letters * N, 4LL * n_letters, 4LL * n_letters, L};
  place.parent = (const long long*)parent;
  place.token = (const long long*)token;
  place.logits = logits;
  place.W = n_beams;
  place.n_letters = n_letters;
  place.n_layers = n_layers;
  place.TS = TS;
  place.ld_ts = ld_ts;
  place.S = (long long*)S;
  place.log_probs = log_probs;
  float* now = scores;                      // the scores alternate between the two halves of their buffer
  float* next = scores + n_list;
  hipStream_t st = (hipStream_t)stream;
  for (int t = 0; t < L; ++t) {
    const int32_t* list = node_list + (long long)t * n_list;
    for (int l = 0; l < n_layers; ++l) {
      const mpnn_level_layer& y = layers[l];
      int rc;
      if (K <= 48) {
        rc = (f16 ? mpnn_dec_layer_subset_f16 : mpnn_dec_layer_subset)(
            hE_frag, y.P, y.ldp, y.offP, y.RowA, y.lda, y.offA, PVenc, ldenc, y.offEnc, rank, E_idx32, mask, edge_mask,
            y.W1b_packed, y.W2_packed, y.b2, list, n_list, (int)N, L, K, y.hV_in, (float)K, y.W3_packed, y.b3, y.ln1_w,
            y.ln1_b, y.Win_packed, y.b_in, y.Wout8_packed, y.b_out, y.ln2_w, y.ln2_b, y.scale, y.Wproj_packed, y.bproj,
            y.nproj, y.hV_out, y.PQ, stream);
      } else {
        rc = (f16 ? mpnn_dec_message_subset_f16 : mpnn_dec_message_subset)(
            hE_frag, y.P, y.ldp, y.offP, y.RowA, y.lda, y.offA, PVenc, ldenc, y.offEnc, rank, E_idx32, mask, edge_mask,
            y.W1b_packed, y.W2_packed, y.b2, list, n_list, (int)N, L, K, gsum, stream);
        if (!rc)
          rc = (f16 ? mpnn_node_update_subset_f16 : mpnn_node_update_subset)(
              y.hV_in, gsum, (K + 15) / 16, (float)K, mask, y.W3_packed, y.b3, y.ln1_w, y.ln1_b, y.Win_packed, y.b_in,
              y.Wout8_packed, y.b_out, y.ln2_w, y.ln2_b, y.scale, y.Wproj_packed, y.bproj, y.nproj, list, n_list, y.hV_out,
              y.PQ, stream);
      }
      if (rc) return rc;
    }
    hipLaunchKernelGGL(k_beam_logits, dim3((n_list + 15) / 16), dim3(64), 0, st, layers[n_layers - 1].hV_out,
                       (const f32x4*)Wlogit_packed, blogit, n_letters, list, n_list, logits);
    int rc = mpnn_beam_select(logits, 0, (long long)n_beams * n_letters, n_letters, now, logit_bias, 0, 0,
                              forced + (long long)t * n_list, n_groups, n_beams, n_letters, n_beams, next, parent, token,
                              nullptr, 0, stream);
    if (!rc && t > 0)
      rc = mpnn_beam_reorder(n_layers + 2, states, parent, n_groups, n_beams, t, nullptr, rank, stream);
    if (rc) return rc;
    place.list = list;
    hipLaunchKernelGGL(k_beam_place, dim3(n_groups, n_layers + 1), dim3(256), (size_t)n_beams * 512, st, place);
    float* s = now;
    now = next;
    next = s;
  }
  MPNN_LAUNCH_CHECK();
}

#define MPNN_BEAM_RUN(name, f16)                                                                                          \
  extern "C" int name(const float* hE_frag, const float* PVenc, int ldenc, const int32_t* rank, const int32_t* E_idx32,   \
                      const float* mask, const float* edge_mask, const int32_t* node_list, const int64_t* forced,         \
                      int n_groups, int n_beams, int L, int K, const mpnn_level_layer* layers, int n_layers,              \
                      const float* Wlogit_packed, const float* blogit, const float* logit_bias, int n_letters,            \
                      const float* TS, int ld_ts, float* gsum, float* logits, float* scores, int64_t* parent,             \
                      int64_t* token, int64_t* S, float* log_probs, void* stream) {                                       \
    return beam_run(f16, hE_frag, PVenc, ldenc, rank, E_idx32, mask, edge_mask, node_list, forced, n_groups, n_beams, L,  \
                    K, layers, n_layers, Wlogit_packed, blogit, logit_bias, n_letters, TS, ld_ts, gsum, logits, scores,   \
                    parent, token, S, log_probs, stream);                                                                 \
  }
MPNN_BEAM_RUN(mpnn_beam_run, false)
MPNN_BEAM_RUN(mpnn_beam_run_f16, true)
