// AdamW over many tensors in one launch, with the two moments in 32 or 8 bits.
//
//   g = grad * grad_scale
//   m = beta1 m + (1 - beta1) g            v = beta2 v + (1 - beta2) g^2
//   p = (1 - lr wd) p - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// and, where asked for, the bf16 copy of p that the next step's cast reads and
// its amax per tensor.  Moments, p's update and every sum are computed in 32
// bits from the values read; only what is stored is rounded.
//
// 8-bit moments: blocks of 128 consecutive elements share one scale byte s,
// which stands for 2^(s - 127) (255: the block holds a value that is not
// finite, and every value reads as NaN).  s = max(exponent(block amax) - 7, 1),
// so scaled magnitudes are below 256 and a power of two costs no rounding of
// its own.  exp_avg is a sign and E4M3; exp_avg_sq, which has no sign, spends
// that bit on a fourth mantissa bit (E4M4, bias 7).  Both are rounded
// stochastically: with beta2 near 1 a moment moves by less than half a step
// of any 8-bit format in one update, and rounding to nearest would never move
// it at all.  16 random bits a value (Philox4x32-10, one call for four
// elements' two moments) leave a bias below 2^-16 of a step.  A second moment
// above zero never becomes zero: its element's next update would divide by
// eps alone.
//
// Memory-bound: each byte of the parameters, gradients and states moves once.
#include <cmath>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "element_io.cuh"
#include "launch_common.h"
#include "nvfp4_b200.h"
#include "nvfp4_device.cuh"

namespace nvfp4 {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 4;                              // elements a thread takes at once
constexpr int kUnroll = 4;
constexpr uint32_t kChunk = kThreads * kVec * kUnroll;  // elements per thread block
constexpr int kStateBlock = 128;                     // = 32 lanes x kVec: one warp's share
static_assert(kStateBlock == 32 * kVec, "a warp holds whole state blocks");

struct Tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  uint8_t* ms;
  uint8_t* vs;
  __nv_bfloat16* copy;
  uint64_t n;
  uint64_t offset;
  float decay;           // lr * weight_decay, or weight_decay alone where lr comes from the device
  uint32_t first_chunk;  // number of this tensor's first chunk in the launch
};

// The tensors of one launch travel as a kernel parameter: no device table to
// allocate, copy or keep.  The short form keeps the parameter block small for
// the usual small call.
template <int CAP>
struct Args {
  Tensor t[CAP];
  int count;
  uint32_t vec[(CAP + 31) / 32];  // bit t: tensor t takes vector accesses
  float beta1, beta2, omb1, omb2, eps;
  float step_size, rsqrt_bc2;
  const float* grad_scale;
  const float* scalars;
  uint32_t* amax;
  const size_t* rng;
  uint64_t step;
};

// The value of a scale byte: 2^(s - 127); 0 of the zero state; NaN of 255.
__device__ __forceinline__ float scale_value(uint32_t s) {
  return __uint_as_float((s << 23) | (s == 255u ? 0x400000u : 0u));
}

template <int DROP, uint32_t LOW>
__device__ __forceinline__ float unpack8(uint32_t code, float scale) {
  // `code` above LOW carries its own exponent (bias 7); below it counts steps
  // of the lowest binade: 2^-6 (1 + f) - 2^-6.
  const bool low = code < LOW;
  const float t = __uint_as_float((code << DROP) + ((low ? 121u : 120u) << 23));
  return (low ? t - 0.015625f : t) * scale;
}
// |x| scaled into [0, 256), rounded by 16 random bits at the top of the DROP
// bits that are cut.
template <int DROP>
__device__ __forceinline__ uint32_t pack8(float mag, float inv_scale, uint32_t r16) {
  const float y = __fmul_rn(mag, inv_scale);
  const bool low = y < 0.015625f;
  const uint32_t t = __float_as_uint(low ? __fadd_rn(y, 0.015625f) : y) + (r16 << (DROP - 16));
  return (t >> DROP) - ((low ? 121u : 120u) << (23 - DROP));
}

template <typename P, typename G, bool EIGHT, int CAP>
__global__ void __launch_bounds__(kThreads) k_adamw(const __grid_constant__ Args<CAP> a) {
  // The tensor of this block's chunk: the last one whose first chunk is not
  // behind it.
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.t[mid].first_chunk <= blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const Tensor& t = a.t[lo];
  const bool vec = (a.vec[lo >> 5] >> (lo & 31)) & 1u;
  const uint64_t n = t.n;
  const uint64_t base = (uint64_t)(blockIdx.x - t.first_chunk) * kChunk + threadIdx.x * kVec;

  const float gs = a.grad_scale ? *a.grad_scale : 1.0f;
  float keep = 1.0f - t.decay, step_size = a.step_size, rbc2 = a.rsqrt_bc2;
  if (a.scalars) {
    const float lr = a.scalars[0];
    step_size = __fdiv_rn(lr, a.scalars[1]);
    rbc2 = __fdiv_rn(1.0f, __fsqrt_rn(a.scalars[2]));
    keep = 1.0f - lr * t.decay;
  }
  uint64_t seed = 0, roff = 0;
  if constexpr (EIGHT) {
    seed = a.rng[0];
    roff = a.rng[1] + a.step;
  }

  P* pp = reinterpret_cast<P*>(t.p);
  const G* pg = reinterpret_cast<const G*>(t.g);
  float p[kUnroll][kVec], g[kUnroll][kVec];
  float m[kUnroll][kVec], v[kUnroll][kVec];
  uint32_t mc[kUnroll], vc[kUnroll];
  uint8_t msb[kUnroll], vsb[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint64_t i = base + (uint64_t)u * (kThreads * kVec);
    const bool full = vec && i + kVec <= n;
    load4(pp, i, n, full, p[u]);
    load4(pg, i, n, full, g[u]);
    if constexpr (EIGHT) {
      mc[u] = load4_bytes(reinterpret_cast<const uint8_t*>(t.m), i, n, full);
      vc[u] = load4_bytes(reinterpret_cast<const uint8_t*>(t.v), i, n, full);
      msb[u] = i < n ? t.ms[i / kStateBlock] : 0;
      vsb[u] = i < n ? t.vs[i / kStateBlock] : 0;
    } else {
      load4(reinterpret_cast<const float*>(t.m), i, n, full, m[u]);
      load4(reinterpret_cast<const float*>(t.v), i, n, full, v[u]);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint64_t i = base + (uint64_t)u * (kThreads * kVec);
    const bool full = vec && i + kVec <= n;
    if constexpr (EIGHT) {
      const float ms = scale_value(msb[u]);
      const float vs = scale_value(vsb[u]);
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const uint32_t cm = (mc[u] >> (8 * k)) & 0xFFu;
        const float x = unpack8<20, 8u>(cm & 127u, ms);
        m[u][k] = (cm & 128u) ? -x : x;
        v[u][k] = unpack8<19, 16u>((vc[u] >> (8 * k)) & 0xFFu, vs);
      }
    }
    // The roundings of each operation are kept apart (no contraction): the
    // stochastic rounding below then depends on the formula alone, not on how
    // a compiler fuses it.
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const float gk = __fmul_rn(g[u][k], gs);
      m[u][k] = __fadd_rn(__fmul_rn(m[u][k], a.beta1), __fmul_rn(gk, a.omb1));
      v[u][k] = __fadd_rn(__fmul_rn(v[u][k], a.beta2), __fmul_rn(__fmul_rn(gk, gk), a.omb2));
      const float den = __fadd_rn(__fmul_rn(__fsqrt_rn(v[u][k]), rbc2), a.eps);
      p[u][k] = __fadd_rn(__fmul_rn(p[u][k], keep),
                          -__fmul_rn(__fdiv_rn(m[u][k], den), step_size));
    }
    store4(pp, i, n, full, p[u]);
    if (t.copy != nullptr) store4(t.copy, i, n, full, p[u]);
    if (a.amax != nullptr) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        // the amax of what the cast will read: p rounded to bf16
        const float b = __bfloat162float(__float2bfloat16_rn(p[u][k]));
        if (i + k < n) top = max(top, __float_as_uint(b) & 0x7FFFFFFFu);
      }
    }
    if constexpr (EIGHT) {
      uint32_t am = 0, av = 0;
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        if (i + k >= n) m[u][k] = v[u][k] = 0.0f;
        am = max(am, __float_as_uint(m[u][k]) & 0x7FFFFFFFu);
        av = max(av, __float_as_uint(v[u][k]) & 0x7FFFFFFFu);
      }
      // NaN patterns are above infinity's, so the unsigned maximum keeps them.
      am = __reduce_max_sync(0xFFFFFFFFu, am) >> 23;
      av = __reduce_max_sync(0xFFFFFFFFu, av) >> 23;
      const uint32_t sm = am == 255u ? 255u : max((int)am - 7, 1);
      const uint32_t sv = av == 255u ? 255u : max((int)av - 7, 1);
      const float im = __uint_as_float((254u - min(sm, 254u)) << 23);
      const float iv = __uint_as_float((254u - min(sv, 254u)) << 23);
      Philox ph;
      ph.init(seed, (t.offset + i) / kVec, roff, 0);
      const uint4 r4 = ph.generate4();
      const uint32_t r[kVec] = {r4.x, r4.y, r4.z, r4.w};
      uint32_t om = 0, ov = 0;
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        uint32_t cm = sm == 255u ? 0u : pack8<20>(fabsf(m[u][k]), im, r[k] & 0xFFFFu);
        cm |= m[u][k] < 0.0f ? 128u : 0u;
        uint32_t cv = sv == 255u ? 0u : pack8<19>(v[u][k], iv, r[k] >> 16);
        if (sv != 255u && v[u][k] > 0.0f) cv = max(cv, 1u);
        om |= cm << (8 * k);
        ov |= cv << (8 * k);
      }
      store4_bytes(reinterpret_cast<uint8_t*>(t.m), i, n, full, om);
      store4_bytes(reinterpret_cast<uint8_t*>(t.v), i, n, full, ov);
      if ((threadIdx.x & 31) == 0 && i < n) {
        t.ms[i / kStateBlock] = (uint8_t)sm;
        t.vs[i / kStateBlock] = (uint8_t)sv;
      }
    } else {
      store4(reinterpret_cast<float*>(t.m), i, n, full, m[u]);
      store4(reinterpret_cast<float*>(t.v), i, n, full, v[u]);
    }
  }
  if (a.amax != nullptr) {
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    // The word only grows: a stale read costs an atomic, never a result.
    if ((threadIdx.x & 31) == 0 && top > *(volatile uint32_t*)(a.amax + lo))
      atomicMax(a.amax + lo, top);
  }
}

template <typename OUT, int DROP, uint32_t LOW, bool SIGNED>
__global__ void __launch_bounds__(kThreads) k_unpack_state(const uint8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales,
                                                           size_t n, bool vec,
                                                           OUT* __restrict__ out) {
  const size_t stride = (size_t)gridDim.x * kThreads * kVec;
  for (size_t i = ((size_t)blockIdx.x * kThreads + threadIdx.x) * kVec; i < n; i += stride) {
    const bool full = vec && i + kVec <= n;
    const uint32_t c = load4_bytes(codes, i, n, full);
    const float s = scale_value(scales[i / kStateBlock]);
    float x[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const uint32_t b = (c >> (8 * k)) & 0xFFu;
      const float y = unpack8<DROP, LOW>(SIGNED ? b & 127u : b, s);
      x[k] = SIGNED && (b & 128u) ? -y : y;
    }
    store4(out, i, n, full, x);
  }
}

template <typename P, typename G, bool EIGHT, int CAP>
int launch_group(const nvfp4_adamw_tensor* tensors, int count, double lr, Args<CAP>& a,
                 cudaStream_t stream) {
  // As many launches as the tensors' chunks and the parameter block need.
  for (int at = 0; at < count;) {
    uint64_t chunks = 0;
    int k = 0;
    for (uint32_t& w : a.vec) w = 0;
    const int begin = at;
    for (; at < count && k < CAP; ++at) {
      const nvfp4_adamw_tensor& t = tensors[at];
      const uint64_t need = (t.n + kChunk - 1) / kChunk;
      if (chunks + need > 0x7FFFFFFFull) break;   // need alone is below: checked on entry
      Tensor& d = a.t[k];
      d.p = t.param; d.g = t.grad; d.m = t.exp_avg; d.v = t.exp_avg_sq;
      d.ms = t.exp_avg_scale; d.vs = t.exp_avg_sq_scale;
      d.copy = reinterpret_cast<__nv_bfloat16*>(t.copy);
      d.n = t.n;
      d.offset = t.offset;
      d.decay = a.scalars ? (float)t.weight_decay : (float)(lr * t.weight_decay);
      d.first_chunk = (uint32_t)chunks;
      const uintptr_t state = EIGHT ? (uintptr_t)t.exp_avg % 4 | (uintptr_t)t.exp_avg_sq % 4
                                    : (uintptr_t)t.exp_avg % 16 | (uintptr_t)t.exp_avg_sq % 16;
      if (((uintptr_t)t.param % (4 * sizeof(P)) | (uintptr_t)t.grad % (4 * sizeof(G)) | state |
           (uintptr_t)t.copy % 8) == 0)
        a.vec[k >> 5] |= 1u << (k & 31);
      chunks += need;
      ++k;
    }
    if (chunks == 0) continue;
    a.count = k;
    uint32_t* amax = a.amax;
    if (amax) a.amax = amax + begin;
    k_adamw<P, G, EIGHT, CAP><<<(unsigned)chunks, kThreads, 0, stream>>>(a);
    a.amax = amax;
    if (cudaError_t e = cudaGetLastError()) return cuda_status(e);
  }
  return NVFP4_OK;
}

template <typename P, typename G, bool EIGHT>
int launch_all(const nvfp4_adamw_tensor* tensors, int count, double lr, double beta1, double beta2,
               double eps, int64_t step, const float* grad_scale, const float* scalars,
               float* amax, const size_t* rng, cudaStream_t stream) {
  auto go = [&](auto& a) {
    a.beta1 = (float)beta1;
    a.beta2 = (float)beta2;
    a.omb1 = (float)(1.0 - beta1);
    a.omb2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.step_size = scalars ? 0.0f : (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    a.rsqrt_bc2 = scalars ? 0.0f : (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    a.grad_scale = grad_scale;
    a.scalars = scalars;
    a.amax = reinterpret_cast<uint32_t*>(amax);
    a.rng = rng;
    a.step = (uint64_t)step;
    return launch_group<P, G, EIGHT>(tensors, count, lr, a, stream);
  };
  // Kernel parameters are copied on every launch: a call of a few tensors
  // takes the short parameter block.
  if (count <= 32) {
    Args<32> a;
    return go(a);
  }
  Args<384> a;
  return go(a);
}

template <typename P, bool EIGHT, typename... Rest>
int launch_grad(int grad_dtype, Rest... rest) {
  if (grad_dtype == NVFP4_DTYPE_F32) return launch_all<P, float, EIGHT>(rest...);
  if (grad_dtype == NVFP4_DTYPE_BF16) return launch_all<P, __nv_bfloat16, EIGHT>(rest...);
  return launch_all<P, __half, EIGHT>(rest...);
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

NVFP4_API int nvfp4_adamw_step(const nvfp4_adamw_tensor* tensors, int count, int param_dtype,
                               int grad_dtype, int state_format, double lr, double beta1,
                               double beta2, double eps, int64_t step, const float* grad_scale,
                               const float* scalars, float* amax_out, const size_t* rng_state,
                               nvfp4_stream_t stream) {
  if (count < 0) return NVFP4_ERR_INVALID_SHAPE;
  if (count == 0) return NVFP4_OK;
  if (!tensors) return NVFP4_ERR_INVALID_ARGUMENT;
  if (param_dtype != NVFP4_DTYPE_F32 && param_dtype != NVFP4_DTYPE_BF16)
    return NVFP4_ERR_INVALID_ARGUMENT;
  if (grad_dtype < NVFP4_DTYPE_F32 || grad_dtype > NVFP4_DTYPE_F16)
    return NVFP4_ERR_INVALID_ARGUMENT;
  if (state_format != NVFP4_STATE_F32 && state_format != NVFP4_STATE_8BIT)
    return NVFP4_ERR_INVALID_ARGUMENT;
  const bool eight = state_format == NVFP4_STATE_8BIT;
  // Written so that a NaN is refused too.
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0))
    return NVFP4_ERR_INVALID_ARGUMENT;
  if (!scalars && (step < 1 || !std::isfinite(lr))) return NVFP4_ERR_INVALID_ARGUMENT;
  if (eight && !rng_state) return NVFP4_ERR_INVALID_ARGUMENT;
  if ((uintptr_t)grad_scale % 4 || (uintptr_t)scalars % 4 || (uintptr_t)amax_out % 4 ||
      (uintptr_t)rng_state % 8)
    return NVFP4_ERR_MISALIGNED;
  const uintptr_t psize = param_dtype == NVFP4_DTYPE_F32 ? 4 : 2;
  const uintptr_t gsize = grad_dtype == NVFP4_DTYPE_F32 ? 4 : 2;
  const uintptr_t ssize = eight ? 1 : 4;
  for (int i = 0; i < count; ++i) {
    const nvfp4_adamw_tensor& t = tensors[i];
    if (t.n > (1ull << 42)) return NVFP4_ERR_INVALID_SHAPE;
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return NVFP4_ERR_INVALID_ARGUMENT;
    if (eight && (!t.exp_avg_scale || !t.exp_avg_sq_scale || t.offset % kStateBlock != 0))
      return NVFP4_ERR_INVALID_ARGUMENT;
    if (t.copy && param_dtype != NVFP4_DTYPE_F32) return NVFP4_ERR_INVALID_ARGUMENT;
    if (!std::isfinite(t.weight_decay)) return NVFP4_ERR_INVALID_ARGUMENT;
    if ((uintptr_t)t.param % psize || (uintptr_t)t.grad % gsize || (uintptr_t)t.exp_avg % ssize ||
        (uintptr_t)t.exp_avg_sq % ssize || (uintptr_t)t.copy % 2)
      return NVFP4_ERR_MISALIGNED;
  }
  int sms = 0;
  if (int e = device_sm_count(&sms)) return e;
  cudaStream_t st = (cudaStream_t)stream;
  if (amax_out)
    if (cudaError_t e = cudaMemsetAsync(amax_out, 0, sizeof(float) * (size_t)count, st))
      return cuda_status(e);
  if (param_dtype == NVFP4_DTYPE_F32)
    return eight ? launch_grad<float, true>(grad_dtype, tensors, count, lr, beta1, beta2, eps,
                                            step, grad_scale, scalars, amax_out, rng_state, st)
                 : launch_grad<float, false>(grad_dtype, tensors, count, lr, beta1, beta2, eps,
                                             step, grad_scale, scalars, amax_out, rng_state, st);
  return eight ? launch_grad<__nv_bfloat16, true>(grad_dtype, tensors, count, lr, beta1, beta2,
                                                  eps, step, grad_scale, scalars, amax_out,
                                                  rng_state, st)
               : launch_grad<__nv_bfloat16, false>(grad_dtype, tensors, count, lr, beta1, beta2,
                                                   eps, step, grad_scale, scalars, amax_out,
                                                   rng_state, st);
}

NVFP4_API int nvfp4_adamw_unpack_state(const void* codes, const uint8_t* scales, size_t n,
                                       int moment, void* out, int out_dtype,
                                       nvfp4_stream_t stream) {
  if (moment != NVFP4_EXP_AVG && moment != NVFP4_EXP_AVG_SQ) return NVFP4_ERR_INVALID_ARGUMENT;
  if (out_dtype != NVFP4_DTYPE_F32 && out_dtype != NVFP4_DTYPE_BF16)
    return NVFP4_ERR_INVALID_ARGUMENT;
  if (n == 0) return NVFP4_OK;
  if (!codes || !scales || !out) return NVFP4_ERR_INVALID_ARGUMENT;
  const uintptr_t osize = out_dtype == NVFP4_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)out % osize) return NVFP4_ERR_MISALIGNED;
  int sms = 0;
  if (int e = device_sm_count(&sms)) return e;
  size_t blocks = (n + kThreads * kVec - 1) / (kThreads * kVec);
  if (blocks > (size_t)sms * 32) blocks = (size_t)sms * 32;
  const bool vec = (uintptr_t)codes % 4 == 0 && (uintptr_t)out % (4 * osize) == 0;
  const uint8_t* c = reinterpret_cast<const uint8_t*>(codes);
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)blocks;
  if (out_dtype == NVFP4_DTYPE_F32) {
    float* o = reinterpret_cast<float*>(out);
    if (moment == NVFP4_EXP_AVG)
      k_unpack_state<float, 20, 8u, true><<<grid, kThreads, 0, st>>>(c, scales, n, vec, o);
    else
      k_unpack_state<float, 19, 16u, false><<<grid, kThreads, 0, st>>>(c, scales, n, vec, o);
  } else {
    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(out);
    if (moment == NVFP4_EXP_AVG)
      k_unpack_state<__nv_bfloat16, 20, 8u, true><<<grid, kThreads, 0, st>>>(c, scales, n, vec, o);
    else
      k_unpack_state<__nv_bfloat16, 19, 16u, false><<<grid, kThreads, 0, st>>>(c, scales, n, vec,
                                                                               o);
  }
  return cuda_status(cudaGetLastError());
}

}  // extern "C"
