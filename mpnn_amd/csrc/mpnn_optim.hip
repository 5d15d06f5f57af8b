// AdamW over many tensors with the moments of each in 8 bits or in 32.
//
//   g = coef * grad,  coef = min(1, max_norm / (|grad| + 1e-6)) over all tensors
//   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit moments are e4m3 codes with a power of two for each 64 elements (the largest of them lies in [128, 256) scales) and
// are rounded STOCHASTICALLY: with b2 = 0.999 a step moves v by 0.1 %, a fiftieth of half a step of a 3-bit mantissa, so
// rounding to nearest would freeze it; rounded up with the probability of the part cut off, the stored moment follows the
// exact one in the mean.  The bits come from a hash of (seed, step, tensor, element): a step is the same on every run.  v
// above zero is never stored as zero (m / eps would follow).  A power of two scales without a rounding of its own, so the
// stored value has one error only, and moments are fp64 up to it (the fp64 vector rate is the fp32 one): which code an element
// gets does not hang on the order of operations.  Memory-bound: 16.25 bytes an element of an 8-bit tensor (28 with 32-bit moments), and 4 more
// where the norm is needed.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "mpnn_common.h"
#include "mpnn_hip.h"
#include "mpnn_reduce.h"

namespace {

constexpr int AW_MAX = 120;      // tensors of a launch: the table travels as a kernel argument of less than 4 KB
constexpr int AW_CHUNK = 1024;   // elements of a workgroup's turn: four a thread
constexpr int AW_WGS = 16384;    // workgroups of a launch at most (100 M parameters: 429 us with 8192 or 16384, 457 with 2048)
constexpr int AW_BLOCK = 64;     // elements that share a scale: 16 lanes of four elements
constexpr int AW_PARTS = 256;    // workgroups (and partial sums) of the norm, over all launches of a call
constexpr int NT_THREADS = 1024;
constexpr int NT_CHUNK = 4 * NT_THREADS * 4;   // elements of a workgroup's turn in the norm
constexpr int NT_MAX = 128;      // tensors of a launch of the norm, by pointers
constexpr int NT_NEAR = 320;     // by distances
constexpr int FEW = 16;          // tensors whose table is a launch's smallest: 3.1 us a launch with 640 bytes of arguments, 2.7 with
                                 // 64, 4.1-4.9 with 1.5 to 4 KB

// A tensor's six addresses as distances from those of the first tensor of its kind, in units of four bytes: 32 bytes a
// tensor, where pointers take 56 and two launches for the model's 118 tensors.  A tensor that lies 8 GB away from the first
// (or whose codes have another residue modulo four) opens the next table.
struct Origin {
  char *p, *g, *m, *v, *ms, *vs;
};
template <int N>
struct AdamTable {
  static constexpr int MAX = N;
  Origin origin[2];              // of 32-bit moments, of 8-bit ones
  int p[N], g[N], m[N], v[N], ms[N], vs[N];   // ms: NO_SCALE for 32-bit moments
  unsigned numel[N];
  int chunk0[N + 1];             // first chunk of each tensor
  int n;
};
constexpr int NO_SCALE = (int)0x80000000;

// the norm's: distances in units of four bytes from the first, as above, or pointers where those do not reach
template <int N>
struct NearTable {
  static constexpr int MAX = N;
  const float* origin;
  int at[N];
  unsigned numel[N];
  int chunk0[N + 1];
  int n;
  __device__ const float* grad(int i) const { return origin + at[i]; }
};
struct FarTable {
  static constexpr int MAX = NT_MAX;
  const float* at[NT_MAX];
  unsigned numel[NT_MAX];
  int chunk0[NT_MAX + 1];
  int n;
  __device__ const float* grad(int i) const { return at[i]; }
};

struct AdamHyper {
  double b1, c1, b2, c2;         // c = 1 - b
  float decay, rate, root, eps;  // 1 - lr wd;  lr / (1 - b1^t);  1 / sqrt(1 - b2^t);  eps
  double max_norm;
  const double* parts;           // AW_PARTS partial sums of squares, NULL without clipping
  float* sumsq;                  // the sum, for the caller
  unsigned key, tensor0;
};

// 32 bits of a counter and a seed, as dropout_keep's (mpnn_edge_common.h)
__host__ __device__ __forceinline__ unsigned mix_bits(unsigned h) {
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  h ^= h >> 13;
  h *= 0xC2B2AE35u;
  h ^= h >> 16;
  return h;
}
__host__ __device__ __forceinline__ unsigned hash_bits(unsigned id, unsigned seed) { return mix_bits((id * 0x9E3779B1u) ^ seed); }

// tensor of a chunk: each lane compares an entry of the table (or two)
template <typename Table>
__device__ __forceinline__ int tensor_of(const Table& t, int chunk) {
  int at = -1;
#pragma unroll
  for (int o = 0; o < (int)(sizeof(t.chunk0) / 4) - 1; o += 64) {
    const int e = (threadIdx.x & 63) + o;
    at += __popcll(__ballot(e < t.n && t.chunk0[e < t.n ? e : 0] <= chunk));
  }
  return __builtin_amdgcn_readfirstlane(at);
}

// sum over the workgroup, in every thread
template <int WAVES>
__device__ __forceinline__ double block_sum(double s, double* sh) {
  s = group_sum(s, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) s += sh[i];
  return s;
}

template <typename Table>
__global__ void __launch_bounds__(NT_THREADS)
k_grad_sumsq_parts(Table t, double* __restrict__ parts) {
  __shared__ double sh[NT_THREADS / 64];
  double s = 0.0;
  for (int chunk = blockIdx.x; chunk < t.chunk0[t.n]; chunk += gridDim.x) {
    const int ti = tensor_of(t, chunk);
    const float* __restrict__ g = t.grad(ti);
    const long long n = t.numel[ti], i = (long long)(chunk - t.chunk0[ti]) * NT_CHUNK + threadIdx.x * 4;
    constexpr int ROW = 4 * NT_THREADS;
    if (((uintptr_t)g & 15) == 0 && i + NT_CHUNK - ROW + 4 <= n) {   // this thread's last four included
      f32x4 x[NT_CHUNK / ROW];
#pragma unroll
      for (int k = 0; k < NT_CHUNK / ROW; ++k) x[k] = *reinterpret_cast<const f32x4*>(g + i + ROW * k);
#pragma unroll
      for (int k = 0; k < NT_CHUNK / ROW; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) s += (double)x[k][j] * (double)x[k][j];
    } else {
      for (int k = 0; k < NT_CHUNK; k += ROW)
        for (int j = 0; j < 4; ++j)
          if (i + k + j < n) s += (double)g[i + k + j] * (double)g[i + k + j];
    }
  }
  s = block_sum<NT_THREADS / 64>(s, sh);
  if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

__device__ __forceinline__ unsigned hi_word(double x) { return (unsigned)__double2hiint(x); }
__device__ __forceinline__ double pow2(int e) { return __hiloint2double((1023 + e) << 20, 0); }

// largest of 16 lanes (a DPP row): the 64 elements that share a scale
__device__ __forceinline__ unsigned row_max(unsigned x) {
#define MPNN_ROR(n)                                                                                   \
  {                                                                                                   \
    const unsigned y = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + n, 0xf, 0xf, false);  \
    x = y > x ? y : x;                                                                                \
  }
  MPNN_ROR(8) MPNN_ROR(4) MPNN_ROR(2) MPNN_ROR(1)
#undef MPNN_ROR
  return x;
}

// What turns a block's moments into codes, from the high word of the largest: the scale's exponent e puts that one into
// [128, 256) scales.  A moment's code is floor(y / step + r / 65536), y = |x| / scale, r 16 random bits.  Above 2^-6 the
// step is an eighth of y's power of two: r added to the mantissa's high word 17 bits down, what is left above them is the
// code (the floor depends on the 19 leading mantissa bits only, the high word has 20).  Below, the step is 2^-9 and y a
// fixed-point number.
struct Encoder {
  bool finite;
  unsigned rebias, normal;    // from the high word to e4m3's exponent; the least high word of a code above 2^-6
  double fixed;               // 2^25 / scale
  float scale;
  __device__ __forceinline__ explicit Encoder(unsigned top) {
    int e = (int)(top >> 20) - 1023 - 7;
    e = e < -126 ? -126 : e;
    if (top == 0) e = 0;
    finite = (top >> 20) < 1023 + 128;    // else infinite, NaN or beyond fp32
    rebias = (unsigned)(-e - 1016) << 20;
    normal = (unsigned)(1023 - 6 + e) << 20;
    fixed = pow2(25 - e);
    scale = finite ? __int_as_float((127 + e) << 23) : NAN;
  }
  __device__ __forceinline__ unsigned code(double x, unsigned r) const {
    const unsigned hi = hi_word(x) & 0x7fffffffu;
    const unsigned above = (hi + rebias + (r << 1)) >> 17;
    const unsigned below = ((unsigned)__double2uint_rz(fabs(x) * fixed) + r) >> 16;
    const unsigned c = hi >= normal ? above : below;
    return finite ? c : 0u;
  }
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void decode4(unsigned codes, double (&x)[4]) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  x[0] = (double)a.x;
  x[1] = (double)a.y;
  x[2] = (double)b.x;
  x[3] = (double)b.y;
}

// The update in fp32.  The square root and the reciprocal are the hardware's (within one step of the last place; the move
// they scale is a small part of p): correctly rounded ones are a third of the kernel's instructions.  They count fp32
// denormals as zero, which shows where eps does not cover sqrt(2^-126) only: then the exact ones run.
__device__ __forceinline__ float adam_update(float p, double m, double v, const AdamHyper& h) {
  if (h.eps >= 1e-12f) {
    const float d = fmaf(__builtin_amdgcn_sqrtf((float)v), h.root, h.eps);
    return fmaf(p, h.decay, -h.rate * ((float)m * __builtin_amdgcn_rcpf(d)));
  }
  return p * h.decay - h.rate * ((float)m / (sqrtf((float)v) * h.root + h.eps));
}

// four elements of a thread on their way through the step
struct Four {
  float* p;
  void *m, *v;
  float *ms, *vs;                // of the block; NULL: 32-bit moments
  unsigned key, id;
  int left;                      // of the four that exist
  bool wide;                     // moved as vectors
  f32x4 pv, gv, mv, vv;          // 8-bit moments: four codes in mv[0], vv[0], the scale in mv[1], vv[1]
};

template <typename Table>
__device__ __forceinline__ void load_four(const Table& t, const AdamHyper& h, int chunk, Four& c) {
  const int ti = tensor_of(t, chunk);
  const long long n = t.numel[ti], i = (long long)(chunk - t.chunk0[ti]) * AW_CHUNK + threadIdx.x * 4;
  const bool eight = t.ms[ti] != NO_SCALE;
  const Origin& o = t.origin[eight];
  const float* g = (const float*)(o.g + 4LL * t.g[ti]);
  char *m = o.m + 4LL * t.m[ti], *v = o.v + 4LL * t.v[ti];
  c.left = i >= n ? 0 : n - i < 4 ? (int)(n - i) : 4;
  c.p = (float*)(o.p + 4LL * t.p[ti]) + i;
  c.pv = c.gv = c.mv = c.vv = f32x4{0.f, 0.f, 0.f, 0.f};
  c.id = (unsigned)i * 0x9E3779B1u;
  c.key = h.tensor0 + ti;
  if (eight) {
    c.m = m + i;
    c.v = v + i;
    c.ms = (float*)(o.ms + 4LL * t.ms[ti]) + i / AW_BLOCK;
    c.vs = (float*)(o.vs + 4LL * t.vs[ti]) + i / AW_BLOCK;
    c.wide = c.left == 4 && (((uintptr_t)c.p | (uintptr_t)(g + i)) & 15) == 0 && (((uintptr_t)c.m | (uintptr_t)c.v) & 3) == 0;
    unsigned mc = 0, vc = 0;
    if (c.wide) {
      mc = *(const unsigned*)c.m;
      vc = *(const unsigned*)c.v;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < c.left) {
          mc |= (unsigned)((const unsigned char*)c.m)[j] << (8 * j);
          vc |= (unsigned)((const unsigned char*)c.v)[j] << (8 * j);
        }
    }
    c.mv[0] = __uint_as_float(mc);
    c.vv[0] = __uint_as_float(vc);
    c.mv[1] = c.left ? *c.ms : 1.f;
    c.vv[1] = c.left ? *c.vs : 1.f;
  } else {
    c.m = (float*)m + i;
    c.v = (float*)v + i;
    c.ms = c.vs = nullptr;
    c.wide = c.left == 4 && (((uintptr_t)c.p | (uintptr_t)(g + i) | (uintptr_t)c.m | (uintptr_t)c.v) & 15) == 0;
    if (c.wide) {
      c.mv = *(const f32x4*)c.m;
      c.vv = *(const f32x4*)c.v;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < c.left) {
          c.mv[j] = ((const float*)c.m)[j];
          c.vv[j] = ((const float*)c.v)[j];
        }
    }
  }
  if (c.wide) {
    c.pv = *(const f32x4*)c.p;
    c.gv = *(const f32x4*)(g + i);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < c.left) {
        c.pv[j] = c.p[j];
        c.gv[j] = g[i + j];
      }
  }
}

__device__ __forceinline__ void finish_four(const AdamHyper& h, double coef, Four& c) {
  if (c.ms) {
    // a power of two multiplies exactly: b * (code * scale) = (b * scale) * code
    const double b1 = h.b1 * (double)c.mv[1], b2 = h.b2 * (double)c.vv[1];
    const unsigned key = hash_bits(c.key, h.key);
    double md[4], vd[4];
    decode4(__float_as_uint(c.mv[0]), md);
    decode4(__float_as_uint(c.vv[0]), vd);
    unsigned mtop = 0, vtop = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {                // elements past the end are zeros and stay so
      const double gi = (double)c.gv[j] * coef;
      md[j] = b1 * md[j] + h.c1 * gi;
      vd[j] = b2 * vd[j] + h.c2 * (gi * gi);
      const unsigned a = hi_word(md[j]) & 0x7fffffffu, b = hi_word(vd[j]) & 0x7fffffffu;
      mtop = a > mtop ? a : mtop;
      vtop = b > vtop ? b : vtop;
      c.pv[j] = adam_update(c.pv[j], md[j], vd[j], h);
    }
    const Encoder me(row_max(mtop)), ve(row_max(vtop));
    unsigned mc = 0, vc = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned r = mix_bits((c.id + j * 0x9E3779B1u) ^ key);
      const unsigned a = me.code(md[j], r & 0xffffu), b = ve.code(vd[j], r >> 16);
      const unsigned least = vd[j] > 0.0 ? 1u : 0u;
      mc |= (a | (a ? (hi_word(md[j]) >> 24) & 0x80u : 0u)) << (8 * j);
      vc |= (b > least ? b : least) << (8 * j);
    }
    if (c.wide) {
      *(unsigned*)c.m = mc;
      *(unsigned*)c.v = vc;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < c.left) {
          ((unsigned char*)c.m)[j] = (unsigned char)(mc >> (8 * j));
          ((unsigned char*)c.v)[j] = (unsigned char)(vc >> (8 * j));
        }
    }
    if (c.left && (threadIdx.x & 15) == 0) {
      *c.ms = me.scale;
      *c.vs = ve.scale;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double gi = (double)c.gv[j] * coef;
      const double mi = h.b1 * (double)c.mv[j] + h.c1 * gi, vi = h.b2 * (double)c.vv[j] + h.c2 * (gi * gi);
      c.mv[j] = (float)mi;
      c.vv[j] = (float)vi;
      c.pv[j] = adam_update(c.pv[j], mi, vi, h);
    }
    if (c.wide) {
      *(f32x4*)c.m = c.mv;
      *(f32x4*)c.v = c.vv;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < c.left) {
          ((float*)c.m)[j] = c.mv[j];
          ((float*)c.v)[j] = c.vv[j];
        }
    }
  }
  if (c.wide) {
    *(f32x4*)c.p = c.pv;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < c.left) c.p[j] = c.pv[j];
  }
}

template <typename Table>
__global__ void __launch_bounds__(256)
k_adamw_mixed(Table t, AdamHyper h) {
  __shared__ double sh[4];
  const int total = t.chunk0[t.n];
  int chunk = blockIdx.x;
  const double part = h.parts ? h.parts[threadIdx.x] : 0.0;   // requested first: loads return in order
  Four c;
  load_four(t, h, chunk, c);                     // under way while the norm is added up
  double coef = 1.0;
  if (h.parts) {
    static_assert(AW_PARTS == 256, "one partial sum a thread");
    const double s = block_sum<4>(part, sh);
    if (blockIdx.x == 0 && threadIdx.x == 0 && h.sumsq) *h.sumsq = (float)s;
    const double f = h.max_norm / (sqrt(s) + 1e-6);
    coef = f < 1.0 || f != f ? f : 1.0;          // a NaN norm reaches every parameter, as in clip_coef (mpnn_loss.hip)
  }
  for (;;) {   // (the next elements requested before these are finished: 472 us instead of 429, too many registers)
    finish_four(h, coef, c);
    chunk += gridDim.x;
    if (chunk >= total) return;
    load_four(t, h, chunk, c);
  }
}

}  // namespace

static void place(FarTable& t, int j, const float* const* grads, int k0) { t.at[j] = grads[k0 + j]; }
template <int N>
static void place(NearTable<N>& t, int j, const float* const* grads, int k0) {
  t.origin = grads[0];
  t.at[j] = (int)(grads[k0 + j] - grads[0]);
}

template <typename Table>
static void launch_parts(int n, const float* const* grads, const long long* numel, double* parts, hipStream_t st) {
  const int launches = (n + Table::MAX - 1) / Table::MAX, share = AW_PARTS / launches;
  for (int l = 0; l < launches; ++l) {
    Table t;
    const int k0 = l * Table::MAX;
    t.n = n - k0 < Table::MAX ? n - k0 : Table::MAX;
    long long chunks = 0;                            // at most 320 * 2^18
    for (int j = 0; j < t.n; ++j) {
      place(t, j, grads, k0);
      t.numel[j] = (unsigned)numel[k0 + j];
      t.chunk0[j] = (int)chunks;
      chunks += (numel[k0 + j] + NT_CHUNK - 1) / NT_CHUNK;
    }
    t.chunk0[t.n] = (int)chunks;
    const int wgs = l + 1 < launches ? share : AW_PARTS - share * (launches - 1);   // every part is written
    hipLaunchKernelGGL((k_grad_sumsq_parts<Table>), dim3(wgs), dim3(NT_THREADS), 0, st, t, parts + (long long)share * l);
  }
}

extern "C" int mpnn_grad_sumsq_parts(int n, const float* const* grads, const long long* numel, double* parts, void* stream) {
  MPNN_CHECK_ARG(n > 0 && n <= AW_PARTS * NT_MAX && grads && numel && parts, "mpnn_grad_sumsq_parts: bad arguments");
  bool near = true;
  for (int j = 0; j < n; ++j) {
    MPNN_CHECK_ARG(grads[j] && ((uintptr_t)grads[j] & 3) == 0 && numel[j] > 0 && numel[j] < (1LL << 32),
                   "mpnn_grad_sumsq_parts: null, misaligned, empty or oversized tensor");
    const long long d = ((const char*)grads[j] - (const char*)grads[0]) / 4;
    near &= d > -(1LL << 31) && d < (1LL << 31);
  }
  hipStream_t st = (hipStream_t)stream;
  if (!near) launch_parts<FarTable>(n, grads, numel, parts, st);
  else if (n <= FEW) launch_parts<NearTable<FEW>>(n, grads, numel, parts, st);
  else launch_parts<NearTable<NT_NEAR>>(n, grads, numel, parts, st);
  MPNN_LAUNCH_CHECK();
}

// distance of x from the table's origin in units of four bytes, if it has one (NO_SCALE is none)
static bool offset(const void* x, const char* origin, int& out) {
  const long long d = (const char*)x - origin;
  out = (int)(d / 4);
  return d % 4 == 0 && d / 4 > -(1LL << 31) && d / 4 < (1LL << 31);
}

struct AdamLists {
  int n, first;
  float* const* params;
  const float* const* grads;
  void* const* exp_avg;
  void* const* exp_avg_sq;
  float* const* exp_avg_scale;
  float* const* exp_avg_sq_scale;
  const long long* numel;
};

template <typename Table>
static void launch_adamw(const AdamLists& q, AdamHyper h, hipStream_t st) {
  for (int k0 = 0; k0 < q.n;) {
    Table t;
    t.origin[0] = t.origin[1] = Origin{};
    long long chunks = 0;
    int j = 0;
    for (; j < Table::MAX && k0 + j < q.n; ++j) {
      const int k = k0 + j;
      const bool eight = q.exp_avg_scale[k] != nullptr;
      Origin& o = t.origin[eight];
      if (!o.p)
        o = Origin{(char*)q.params[k], (char*)q.grads[k], (char*)q.exp_avg[k], (char*)q.exp_avg_sq[k], (char*)q.exp_avg_scale[k],
                   (char*)q.exp_avg_sq_scale[k]};
      const long long more = (q.numel[k] + AW_CHUNK - 1) / AW_CHUNK;
      t.ms[j] = t.vs[j] = NO_SCALE;
      if (!offset(q.params[k], o.p, t.p[j]) || !offset(q.grads[k], o.g, t.g[j]) || !offset(q.exp_avg[k], o.m, t.m[j]) ||
          !offset(q.exp_avg_sq[k], o.v, t.v[j]) ||
          (eight && (!offset(q.exp_avg_scale[k], o.ms, t.ms[j]) || !offset(q.exp_avg_sq_scale[k], o.vs, t.vs[j]))) ||
          chunks + more >= (1LL << 31) - 65536)
        break;                                       // never the first: it is an origin
      t.numel[j] = (unsigned)q.numel[k];
      t.chunk0[j] = (int)chunks;
      chunks += more;
    }
    t.n = j;
    t.chunk0[j] = (int)chunks;
    h.tensor0 = (unsigned)(q.first + k0);
    hipLaunchKernelGGL((k_adamw_mixed<Table>), dim3((unsigned)(chunks < AW_WGS ? chunks : AW_WGS)), dim3(256), 0, st, t, h);
    h.sumsq = nullptr;
    k0 += j;
  }
}

extern "C" int mpnn_adamw_mixed(int n, float* const* params, const float* const* grads, void* const* exp_avg,
                                void* const* exp_avg_sq, float* const* exp_avg_scale, float* const* exp_avg_sq_scale,
                                const long long* numel, double lr, double beta1, double beta2, double eps,
                                double weight_decay, int step, uint32_t seed, int first, const double* sumsq_parts,
                                double max_norm, float* grad_sumsq, void* stream) {
  MPNN_CHECK_ARG(n > 0 && params && grads && exp_avg && exp_avg_sq && exp_avg_scale && exp_avg_sq_scale && numel && first >= 0,
                 "mpnn_adamw_mixed: bad arguments");
  MPNN_CHECK_ARG(step >= 1 && lr >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && weight_decay >= 0,
                 "mpnn_adamw_mixed: bad hyper-parameters");
  for (int j = 0; j < n; ++j) {
    MPNN_CHECK_ARG(params[j] && grads[j] && exp_avg[j] && exp_avg_sq[j] && numel[j] > 0 && numel[j] < (1LL << 32),
                   "mpnn_adamw_mixed: null, empty or oversized tensor");
    const uintptr_t moments = exp_avg_scale[j] ? 0 : (uintptr_t)exp_avg[j] | (uintptr_t)exp_avg_sq[j];
    MPNN_CHECK_ARG((((uintptr_t)params[j] | (uintptr_t)grads[j] | (uintptr_t)exp_avg_scale[j] | (uintptr_t)exp_avg_sq_scale[j] |
                     moments) & 3) == 0,
                   "mpnn_adamw_mixed: fp32 tensors are aligned to four bytes");
    MPNN_CHECK_ARG(!exp_avg_scale[j] == !exp_avg_sq_scale[j], "mpnn_adamw_mixed: both moments of a tensor have scales, or none");
  }
  AdamHyper h = {};
  h.b1 = beta1;
  h.c1 = 1.0 - beta1;
  h.b2 = beta2;
  h.c2 = 1.0 - beta2;
  h.decay = (float)(1.0 - lr * weight_decay);
  h.rate = (float)(lr / (1.0 - pow(beta1, (double)step)));
  h.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
  h.eps = (float)eps;
  h.max_norm = max_norm;
  h.parts = max_norm > 0 ? sumsq_parts : nullptr;
  h.key = hash_bits((unsigned)step, seed);
  h.sumsq = grad_sumsq;
  const AdamLists lists = {n, first, params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, numel};
  if (n <= FEW) launch_adamw<AdamTable<FEW>>(lists, h, (hipStream_t)stream);
  else launch_adamw<AdamTable<AW_MAX>>(lists, h, (hipStream_t)stream);
  MPNN_LAUNCH_CHECK();
}
