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
// stored value has one error only, and moments are fp64 up to it (the fp64 vector rate is the fp32 one): which code an element gets does not hang
// on the order of operations.  Memory-bound: 16.25 bytes an element of an 8-bit tensor (28 with 32-bit moments), and 4 more
// where the norm is needed.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "mpnn_common.h"
#include "mpnn_hip.h"

namespace {

constexpr int AW_MAX = 60;       // tensors of a launch: the table travels as a kernel argument of less than 4 KB
constexpr int AW_CHUNK = 2048;   // elements of a workgroup's turn
constexpr int AW_BLOCK = 64;     // elements that share a scale: 16 lanes of four elements
constexpr int AW_PARTS = 1024;   // workgroups (and partial sums) of the norm, over all launches of a call
constexpr int NT_MAX = 128;      // tensors of a launch of the norm

struct AdamTable {
  float* p[AW_MAX];
  const float* g[AW_MAX];
  void* m[AW_MAX];
  void* v[AW_MAX];
  float* ms[AW_MAX];             // scales; NULL = 32-bit moments
  float* vs[AW_MAX];
  long long numel[AW_MAX];
  int chunk0[AW_MAX + 1];        // first chunk of each tensor
  int n;
};

struct NormTable {
  const float* g[NT_MAX];
  long long numel[NT_MAX];
  int chunk0[NT_MAX + 1];
  int n;
};

struct AdamHyper {
  double b1, c1, b2, c2;         // c = 1 - b
  float decay, rate, root, eps;  // 1 - lr wd;  lr / (1 - b1^t);  1 / sqrt(1 - b2^t);  eps
  double max_norm;
  const double* parts;           // AW_PARTS partial sums of squares, NULL without clipping
  float* sumsq;                  // the sum, for the caller
  unsigned key, tensor0;
};

__host__ __device__ __forceinline__ unsigned hash_bits(unsigned id, unsigned seed) {  // as dropout_keep's (mpnn_edge_common.h)
  unsigned h = (id * 0x9E3779B1u) ^ seed;
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  h ^= h >> 13;
  h *= 0xC2B2AE35u;
  h ^= h >> 16;
  return h;
}

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

__device__ __forceinline__ double block_sum(double s, double* sh) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

__global__ void __launch_bounds__(256)
k_grad_sumsq_parts(NormTable t, double* __restrict__ parts) {
  __shared__ double sh[4];
  double s = 0.0;
  for (int chunk = blockIdx.x; chunk < t.chunk0[t.n]; chunk += gridDim.x) {
    const int ti = tensor_of(t, chunk);
    const float* __restrict__ g = t.g[ti];
    const long long n = t.numel[ti], i0 = (long long)(chunk - t.chunk0[ti]) * AW_CHUNK;
    const bool wide = ((uintptr_t)g & 15) == 0 && i0 + AW_CHUNK <= n;
    if (wide) {
#pragma unroll
      for (int it = 0; it < AW_CHUNK / 1024; ++it) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(g + i0 + it * 1024 + threadIdx.x * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) s += (double)x[i] * (double)x[i];
      }
    } else {
      for (long long i = i0 + threadIdx.x; i < n && i < i0 + AW_CHUNK; i += 256) s += (double)g[i] * (double)g[i];
    }
  }
  s = block_sum(s, sh);
  if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

__device__ __forceinline__ unsigned hi_word(double x) { return (unsigned)(__double_as_longlong(x) >> 32); }
__device__ __forceinline__ double pow2(int e) { return __longlong_as_double((long long)(1023 + e) << 52); }

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

// exponent of a block's scale from the high word of its largest magnitude: the largest lands in [128, 256)
__device__ __forceinline__ bool scale_exponent(unsigned top, int& e) {
  e = (int)(top >> 20) - 1023 - 7;
  e = e < -126 ? -126 : e;
  if (top == 0) e = 0;
  return (top >> 20) < 1023 + 128;    // else infinite, NaN or beyond fp32: the block's scale becomes NaN
}

// |x| / scale as an e4m3 code, rounded up with probability r / 65536 of the part cut off.  floor(y / step + u) with u a
// multiple of 2^-16 needs the 19 leading mantissa bits of y only: the high word has 20.
__device__ __forceinline__ unsigned to_code(double x, double inv, unsigned r) {
  const double y = fabs(x) * inv;
  const unsigned normal = ((hi_word(y) + (r << 1)) >> 17) - (1016u << 3);
  const unsigned small = (unsigned)(int)floor(fma(y, 512.0, (double)r * 0x1p-16));   // below 2^-6 the step is 2^-9
  return y >= 0x1p-6 ? normal : small;
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void decode4(unsigned codes, float scale, double (&x)[4]) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  const double s = (double)scale;
  x[0] = (double)a.x * s;
  x[1] = (double)a.y * s;
  x[2] = (double)b.x * s;
  x[3] = (double)b.y * s;
}

__device__ __forceinline__ float adam_update(float p, double m, double v, const AdamHyper& h) {
  return p * h.decay - h.rate * ((float)m / (sqrtf((float)v) * h.root + h.eps));
}

__global__ void __launch_bounds__(256)
k_adamw_mixed(AdamTable t, AdamHyper h) {
  __shared__ double sh[4];
  double coef = 1.0;
  if (h.parts) {
    double s = 0.0;
    for (int i = threadIdx.x; i < AW_PARTS; i += 256) s += h.parts[i];
    s = block_sum(s, sh);
    if (blockIdx.x == 0 && threadIdx.x == 0 && h.sumsq) *h.sumsq = (float)s;
    const double c = h.max_norm / (sqrt(s) + 1e-6);
    coef = c < 1.0 || c != c ? c : 1.0;          // a NaN norm reaches every parameter, as in clip_coef (mpnn_loss.hip)
  }
  for (int chunk = blockIdx.x; chunk < t.chunk0[t.n]; chunk += gridDim.x) {
    const int ti = tensor_of(t, chunk);
    float* __restrict__ p = t.p[ti];
    const float* __restrict__ g = t.g[ti];
    const long long n = t.numel[ti], i0 = (long long)(chunk - t.chunk0[ti]) * AW_CHUNK;
    if (!t.ms[ti]) {
      float* __restrict__ m = (float*)t.m[ti];
      float* __restrict__ v = (float*)t.v[ti];
      for (long long i = i0 + threadIdx.x; i < n && i < i0 + AW_CHUNK; i += 256) {
        const double gi = (double)g[i] * coef;
        const double mi = h.b1 * (double)m[i] + h.c1 * gi, vi = h.b2 * (double)v[i] + h.c2 * (gi * gi);
        m[i] = (float)mi;
        v[i] = (float)vi;
        p[i] = adam_update(p[i], mi, vi, h);
      }
      continue;
    }
    unsigned char* __restrict__ m = (unsigned char*)t.m[ti];
    unsigned char* __restrict__ v = (unsigned char*)t.v[ti];
    const unsigned key = hash_bits(h.tensor0 + ti, h.key);
    const bool wide = (((uintptr_t)p | (uintptr_t)g) & 15) == 0 && (((uintptr_t)m | (uintptr_t)v) & 3) == 0;
    for (int it = 0; it < AW_CHUNK / 1024; ++it) {
      const long long i = i0 + it * 1024 + threadIdx.x * 4;
      if (i0 + it * 1024 >= n) break;
      const long long blk = i / AW_BLOCK;
      const int left = i >= n ? 0 : n - i < 4 ? (int)(n - i) : 4;
      f32x4 pv = {0.f, 0.f, 0.f, 0.f}, gv = pv;
      unsigned mc = 0, vc = 0;
      float ms = 1.f, vs = 1.f;
      if (left) {
        ms = t.ms[ti][blk];
        vs = t.vs[ti][blk];
      }
      if (wide && left == 4) {
        pv = *reinterpret_cast<const f32x4*>(p + i);
        gv = *reinterpret_cast<const f32x4*>(g + i);
        mc = *reinterpret_cast<const unsigned*>(m + i);
        vc = *reinterpret_cast<const unsigned*>(v + i);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < left) {
            pv[j] = p[i + j];
            gv[j] = g[i + j];
            mc |= (unsigned)m[i + j] << (8 * j);
            vc |= (unsigned)v[i + j] << (8 * j);
          }
      }
      double md[4], vd[4];
      decode4(mc, ms, md);
      decode4(vc, vs, vd);
      unsigned mtop = 0, vtop = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double gi = (double)gv[j] * coef;
        md[j] = h.b1 * md[j] + h.c1 * gi;
        vd[j] = h.b2 * vd[j] + h.c2 * (gi * gi);
        if (j >= left) md[j] = vd[j] = 0.0;
        const unsigned a = hi_word(md[j]) & 0x7fffffffu, b = hi_word(vd[j]) & 0x7fffffffu;
        mtop = a > mtop ? a : mtop;
        vtop = b > vtop ? b : vtop;
        pv[j] = adam_update(pv[j], md[j], vd[j], h);
      }
      int me, ve;
      const bool mfin = scale_exponent(row_max(mtop), me), vfin = scale_exponent(row_max(vtop), ve);
      const double minv = pow2(-me), vinv = pow2(-ve);
      mc = vc = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned r = hash_bits((unsigned)(i + j), key);
        const unsigned a = mfin ? to_code(md[j], minv, r & 0xffffu) : 0u;
        unsigned b = vfin ? to_code(vd[j], vinv, r >> 16) : 0u;
        if (b == 0 && vd[j] > 0.0) b = 1;
        mc |= (a | (a && md[j] < 0.0 ? 0x80u : 0u)) << (8 * j);
        vc |= b << (8 * j);
      }
      if (wide && left == 4) {
        *reinterpret_cast<f32x4*>(p + i) = pv;
        *reinterpret_cast<unsigned*>(m + i) = mc;
        *reinterpret_cast<unsigned*>(v + i) = vc;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < left) {
            p[i + j] = pv[j];
            m[i + j] = (unsigned char)(mc >> (8 * j));
            v[i + j] = (unsigned char)(vc >> (8 * j));
          }
      }
      if (left && (threadIdx.x & 15) == 0) {
        t.ms[ti][blk] = mfin ? (float)pow2(me) : NAN;
        t.vs[ti][blk] = vfin ? (float)pow2(ve) : NAN;
      }
    }
  }
}

template <typename Table>
bool place_chunks(Table& t, const long long* numel) {
  long long chunks = 0;
  for (int j = 0; j < t.n; ++j) {
    t.numel[j] = numel[j];
    t.chunk0[j] = (int)chunks;
    chunks += (numel[j] + AW_CHUNK - 1) / AW_CHUNK;
    if (chunks >= (1LL << 31) - 65536) return false;
  }
  t.chunk0[t.n] = (int)chunks;
  return true;
}

}  // namespace

extern "C" int mpnn_grad_sumsq_parts(int n, const float* const* grads, const long long* numel, double* parts, void* stream) {
  MPNN_CHECK_ARG(n > 0 && n <= AW_PARTS * NT_MAX && grads && numel && parts, "mpnn_grad_sumsq_parts: bad arguments");
  for (int j = 0; j < n; ++j)
    MPNN_CHECK_ARG(grads[j] && numel[j] > 0 && numel[j] < (1LL << 40), "mpnn_grad_sumsq_parts: null, empty or oversized tensor");
  const int launches = (n + NT_MAX - 1) / NT_MAX, share = AW_PARTS / launches;
  for (int l = 0; l < launches; ++l) {
    NormTable t;
    const int k0 = l * NT_MAX;
    t.n = n - k0 < NT_MAX ? n - k0 : NT_MAX;
    for (int j = 0; j < t.n; ++j) t.g[j] = grads[k0 + j];
    MPNN_CHECK_ARG(place_chunks(t, numel + k0), "mpnn_grad_sumsq_parts: too many elements for one launch");
    const int wgs = l + 1 < launches ? share : AW_PARTS - share * (launches - 1);   // every part is written
    hipLaunchKernelGGL(k_grad_sumsq_parts, dim3(wgs), dim3(256), 0, (hipStream_t)stream, t, parts + (long long)share * l);
  }
  MPNN_LAUNCH_CHECK();
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
    MPNN_CHECK_ARG(params[j] && grads[j] && exp_avg[j] && exp_avg_sq[j] && numel[j] > 0 && numel[j] < (1LL << 40),
                   "mpnn_adamw_mixed: null, empty or oversized tensor");
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
  for (int k0 = 0; k0 < n; k0 += AW_MAX) {
    AdamTable t;
    t.n = n - k0 < AW_MAX ? n - k0 : AW_MAX;
    for (int j = 0; j < t.n; ++j) {
      t.p[j] = params[k0 + j];
      t.g[j] = grads[k0 + j];
      t.m[j] = exp_avg[k0 + j];
      t.v[j] = exp_avg_sq[k0 + j];
      t.ms[j] = exp_avg_scale[k0 + j];
      t.vs[j] = exp_avg_sq_scale[k0 + j];
    }
    MPNN_CHECK_ARG(place_chunks(t, numel + k0), "mpnn_adamw_mixed: too many elements for one launch");
    h.tensor0 = (unsigned)(first + k0);
    const int wgs = t.chunk0[t.n] < 2048 ? t.chunk0[t.n] : 2048;
    hipLaunchKernelGGL(k_adamw_mixed, dim3(wgs), dim3(256), 0, (hipStream_t)stream, t, h);
    h.sumsq = nullptr;
  }
  MPNN_LAUNCH_CHECK();
}
