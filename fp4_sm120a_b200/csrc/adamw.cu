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
// Each byte of the parameters, gradients and states moves once.  With fp32 moments
// the step is bound by memory: 147 M parameters in 605 us (6.8 TB/s).  With 8-bit
// moments it is bound by issue slots (72 % taken; some 75 instructions a parameter, of
// which Philox and the rounding are most): 294 M parameters in 880 us (5.3 TB/s).
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
constexpr uint32_t kTopScale = 247;                  // of a block of finite values
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
  uint32_t vec;          // takes vector accesses
};

// The tensors of one launch travel as a kernel parameter: no device table to
// allocate, copy or keep.  The short form keeps the parameter block small for
// the usual small call.  The chunk numbers lie side by side for the search.
template <int CAP>
struct Args {
  Tensor t[CAP];
  uint32_t first_chunk[CAP];   // number of a tensor's first chunk in the launch
  int count;
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

// Four 8-bit moments.  A code moved to the top of an fp16's exponent and
// mantissa is the code's value times 2^-8 exactly, subnormals included (both
// formats have a bias of 8 less than fp16's 15), so fp16's conversion decodes it.
template <bool SIGNED>
__device__ __forceinline__ void unpack8x4(uint32_t codes, uint32_t scale, float (&x)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t w = __byte_perm(codes, 0u, h ? 0x4342 : 0x4140);   // bytes 2h, 2h + 1 in halves
    const uint32_t bits =
        SIGNED ? ((w << 7) & 0x3F803F80u) | ((w << 8) & 0x80008000u) : w << 6;
    unpack2<__half>(bits, x[2 * h], x[2 * h + 1]);
  }
  // 2^(s - 127 + 8); the largest scale takes its last binade in a second step.
  const float f = scale == 0u ? 0.0f : scale_value(scale >= 247u && scale < 255u ? 254u
                                                   : scale == 255u               ? 255u
                                                                                 : scale + 8u);
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] *= f;
  if (scale >= 247u && scale < 255u) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] *= __uint_as_float((scale - 246u + 127u) << 23);
  }
}
// Moments of four elements as the step reads them: exp_avg through E4M3's own
// conversion.  (A block that is not finite holds zero codes, and 0 times the
// scale's infinity is NaN.)
__device__ __forceinline__ void read_avg(uint32_t codes, uint32_t scale, float (&x)[4]) {
  uint32_t lo, hi;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
  unpack2<__half>(lo, x[0], x[1]);
  unpack2<__half>(hi, x[2], x[3]);
  const float f = __uint_as_float(scale << 23);
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] *= f;
}
__device__ __forceinline__ void read_avg_sq(uint32_t codes, uint32_t scale, float (&x)[4]) {
  unpack2<__half>(__byte_perm(codes, 0u, 0x4140) << 6, x[0], x[1]);
  unpack2<__half>(__byte_perm(codes, 0u, 0x4342) << 6, x[2], x[3]);
  const float f = __uint_as_float(scale << 23);
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = x[k] * f * 256.0f;
}

// Stochastic rounding of x, scaled below 256 in magnitude by `inv`: times 2^-120
// the 8-bit formats' lowest binade (from 2^-6 down, equal steps) is fp32's own
// subnormal range, so that the fp32 bits of every value count steps of 2^-DROP
// of a code; 16 random bits below the code's last place carry into it.
template <int DROP>
__device__ __forceinline__ uint32_t rounded_bits(float x, float inv, uint32_t r16) {
  return __float_as_uint(x * inv * 7.52316384526264e-37f) + (r16 << (DROP - 16));
}
// Byte 3 of four words in one.
__device__ __forceinline__ uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
__device__ __forceinline__ float max4_nan(float a, float b, float c, float d) {
  float r;
  asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, %2, %3;\n\tmax.NaN.f32 %0, t, %4;\n\t}"
      : "=f"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// x / y and sqrt(x) to a few 2^-23: p's update is rounded to p's precision
// afterwards, and the moments do not depend on it.
__device__ __forceinline__ float fast_sqrt(float x) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

struct Rates {
  float keep, step_size, rbc2, gs;
  uint64_t seed, offset;
};

// One chunk.  FULL: every element exists and all accesses are vectors.
template <typename P, typename G, bool EIGHT, bool FULL, int CAP>
__device__ __forceinline__ uint32_t adamw_chunk(const Args<CAP>& a, const Tensor& t,
                                                const Rates& r, uint64_t base) {
  const uint64_t n = t.n;
  P* pp = reinterpret_cast<P*>(t.p);
  const G* pg = reinterpret_cast<const G*>(t.g);
  float p[kUnroll][kVec], g[kUnroll][kVec];
  float m[EIGHT ? 1 : kUnroll][kVec], v[EIGHT ? 1 : kUnroll][kVec];
  uint32_t mc[kUnroll], vc[kUnroll], sb[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint64_t i = base + (uint64_t)u * (kThreads * kVec);
    const bool full = FULL || (t.vec && i + kVec <= n);
    load4(pp, i, n, full, p[u]);
    load4(pg, i, n, full, g[u]);
    if constexpr (EIGHT) {
      mc[u] = load4_bytes(reinterpret_cast<const uint8_t*>(t.m), i, n, full);
      vc[u] = load4_bytes(reinterpret_cast<const uint8_t*>(t.v), i, n, full);
      sb[u] = FULL || i < n ? (uint32_t)t.ms[i / kStateBlock] |
                                  ((uint32_t)t.vs[i / kStateBlock] << 8)
                            : 0u;
    } else {
      load4(reinterpret_cast<const float*>(t.m), i, n, full, m[u]);
      load4(reinterpret_cast<const float*>(t.v), i, n, full, v[u]);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint64_t i = base + (uint64_t)u * (kThreads * kVec);
    const bool full = FULL || (t.vec && i + kVec <= n);
    constexpr int kKeep = EIGHT ? 0 : 1;
    float(&mu)[kVec] = m[u * kKeep];
    float(&vu)[kVec] = v[u * kKeep];
    if constexpr (EIGHT) {
      read_avg(mc[u], sb[u] & 0xFFu, mu);
      read_avg_sq(vc[u], sb[u] >> 8, vu);
    }
    // The roundings of each operation on the moments are kept apart (no
    // contraction): the stochastic rounding below then depends on the formula
    // alone, not on how a compiler fuses it.  The sums are scalar for that: a
    // pair's product and sum were seen to be fused in spite of their .rn.
    const uint64_t b1 = pair(a.beta1, a.beta1), b2 = pair(a.beta2, a.beta2);
    const uint64_t o1 = pair(a.omb1, a.omb1), o2 = pair(a.omb2, a.omb2), gs = pair(r.gs, r.gs);
#pragma unroll
    for (int k = 0; k < kVec; k += 2) {
      const uint64_t gk = mul2(pair(g[u][k], g[u][k + 1]), gs);
      float x0, x1, y0, y1;
      split(mul2(pair(mu[k], mu[k + 1]), b1), x0, x1);
      split(mul2(gk, o1), y0, y1);
      mu[k] = __fadd_rn(x0, y0);
      mu[k + 1] = __fadd_rn(x1, y1);
      split(mul2(pair(vu[k], vu[k + 1]), b2), x0, x1);
      split(mul2(mul2(gk, gk), o2), y0, y1);
      vu[k] = __fadd_rn(x0, y0);
      vu[k + 1] = __fadd_rn(x1, y1);
    }
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      // (The root of a subnormal number is far above them; an eps below 2^-126
      // counts as zero.)
      const float update = mu[k] * fast_rcp(fmaf(fast_sqrt(vu[k]), r.rbc2, a.eps));
      p[u][k] = fmaf(-update, r.step_size, p[u][k] * r.keep);
    }
    store4(pp, i, n, full, p[u]);
    if (t.copy != nullptr) store4(t.copy, i, n, full, p[u]);
    if (a.amax != nullptr) {
      // the amax of what the cast will read: p rounded to bf16
      if (FULL || i + kVec <= n) {
        top = max_abs2<__nv_bfloat16>(top, pack2<__nv_bfloat16>(p[u][0], p[u][1]));
        top = max_abs2<__nv_bfloat16>(top, pack2<__nv_bfloat16>(p[u][2], p[u][3]));
      } else {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (i + k < n) top = max_abs2<__nv_bfloat16>(top, pack2<__nv_bfloat16>(p[u][k], 0.0f));
      }
    }
    if constexpr (EIGHT) {
      if (!FULL) {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (i + k >= n) mu[k] = vu[k] = 0.0f;
      }
      // NaN patterns are above infinity's, so the unsigned maximum keeps them.
      const uint32_t am =
          __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(max4_nan(fabsf(mu[0]), fabsf(mu[1]),
                                                                  fabsf(mu[2]), fabsf(mu[3])))) >> 23;
      const uint32_t av =
          __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(max4_nan(vu[0], vu[1], vu[2], vu[3]))) >> 23;
      const uint32_t sm = am == 255u ? 255u : max((int)am - 7, 1);
      const uint32_t sv = av == 255u ? 255u : max((int)av - 7, 1);
      const float im = __uint_as_float((254u - min(sm, 254u)) << 23);
      const float iv = __uint_as_float((254u - min(sv, 254u)) << 23);
      Philox ph;
      ph.init(r.seed, (t.offset + i) / kVec, r.offset, 0);
      const uint4 r4 = ph.generate4();
      const uint32_t w[kVec] = {r4.x, r4.y, r4.z, r4.w};
      uint32_t bm[kVec], bv[kVec];
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        // The code to the top byte; a sign only below zero (-0 + 0 is +0).
        const uint32_t tm = rounded_bits<20>(mu[k] + 0.0f, im, w[k] & 0xFFFFu);
        bm[k] = (tm << 4) | (tm & 0x80000000u);
        uint32_t tv = rounded_bits<19>(vu[k], iv, w[k] >> 16);
        if (vu[k] > 0.0f) tv = max(tv, 1u << 19);
        bv[k] = tv << 5;
      }
      uint32_t om = top_bytes(bm[0], bm[1], bm[2], bm[3]);
      uint32_t ov = top_bytes(bv[0], bv[1], bv[2], bv[3]);
      // Under the largest scale the code of 256 stands for 2^128, which is not
      // finite: the code below takes its place.
      if (sm >= kTopScale) {
        om = (om & 0x80808080u) | __vminu4(om & 0x7F7F7F7Fu, 0x77777777u);
        if (sm == 255u) {
          // No code has a value here; the signs stay.
          om = 0u;
#pragma unroll
          for (int k = 0; k < kVec; ++k) om |= mu[k] < 0.0f ? 0x80u << (8 * k) : 0u;
        }
      }
      if (sv >= kTopScale) ov = sv == 255u ? 0u : __vminu4(ov, 0xEFEFEFEFu);
      store4_bytes(reinterpret_cast<uint8_t*>(t.m), i, n, full, om);
      store4_bytes(reinterpret_cast<uint8_t*>(t.v), i, n, full, ov);
      if ((threadIdx.x & 31) == 0 && (FULL || i < n)) {
        t.ms[i / kStateBlock] = (uint8_t)sm;
        t.vs[i / kStateBlock] = (uint8_t)sv;
      }
    } else {
      store4(reinterpret_cast<float*>(t.m), i, n, full, mu);
      store4(reinterpret_cast<float*>(t.v), i, n, full, vu);
    }
  }
  return top;
}

template <typename P, typename G, bool EIGHT, int CAP>
__global__ void __launch_bounds__(kThreads, 3) k_adamw(const __grid_constant__ Args<CAP> a) {
  // The tensor of this block's chunk: the last one whose first chunk is not
  // behind it.
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first_chunk[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const Tensor& t = a.t[lo];
  const uint64_t chunk = (uint64_t)(blockIdx.x - a.first_chunk[lo]) * kChunk;
  Rates r;
  r.gs = a.grad_scale ? *a.grad_scale : 1.0f;
  r.keep = 1.0f - t.decay;
  r.step_size = a.step_size;
  r.rbc2 = a.rsqrt_bc2;
  if (a.scalars) {
    const float lr = a.scalars[0];
    r.step_size = __fdiv_rn(lr, a.scalars[1]);
    r.rbc2 = __fdiv_rn(1.0f, __fsqrt_rn(a.scalars[2]));
    r.keep = 1.0f - lr * t.decay;
  }
  if constexpr (EIGHT) {
    // Through a warp reduction, whose result the compiler knows to be the same
    // in all lanes: the key schedule then costs the lanes nothing.
    const uint64_t seed = a.rng[0];
    r.seed = (uint64_t)__reduce_or_sync(0xFFFFFFFFu, (uint32_t)(seed >> 32)) << 32 |
             __reduce_or_sync(0xFFFFFFFFu, (uint32_t)seed);
    r.offset = a.rng[1] + a.step;
  }
  const uint64_t base = chunk + threadIdx.x * kVec;
  uint32_t top = t.vec && chunk + kChunk <= t.n
                     ? adamw_chunk<P, G, EIGHT, true, CAP>(a, t, r, base)
                     : adamw_chunk<P, G, EIGHT, false, CAP>(a, t, r, base);
  if (a.amax != nullptr) {
    top &= 0x7FFF7FFFu;
    top = __reduce_max_sync(0xFFFFFFFFu, max(top & 0xFFFFu, top >> 16)) << 16;
    // The word only grows: a stale read costs an atomic, never a result.
    if ((threadIdx.x & 31) == 0 && top > *(volatile uint32_t*)(a.amax + lo))
      atomicMax(a.amax + lo, top);
  }
}

// N values a thread, which leave as one 16-byte vector (FULL), four times over;
// else four values element by element.  Bound by memory: both moments of 294 M
// parameters to bf16 in 264 us (6.7 TB/s).
template <typename OUT, bool SIGNED, bool FULL>
__global__ void __launch_bounds__(kThreads) k_unpack_state(const uint8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales,
                                                           size_t n, OUT* __restrict__ out) {
  constexpr int N = FULL ? 16 / (int)sizeof(OUT) : 4, U = 4;
  const size_t base = (size_t)blockIdx.x * (kThreads * N * U) + threadIdx.x * N;
  uint32_t c[U][N / 4], s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = base + (size_t)u * (kThreads * N);
    const bool in = FULL && i + N <= n;
    if (in && N == 8) {
      const uint2 q = *reinterpret_cast<const uint2*>(codes + i);
      c[u][0] = q.x;
      c[u][N / 4 - 1] = q.y;
    } else {
#pragma unroll
      for (int j = 0; j < N / 4; ++j) c[u][j] = load4_bytes(codes, i + 4 * j, n, in);
    }
    s[u] = i < n ? scales[i / kStateBlock] : 0u;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = base + (size_t)u * (kThreads * N);
    float x[N / 4][4];
#pragma unroll
    for (int j = 0; j < N / 4; ++j) unpack8x4<SIGNED>(c[u][j], s[u], x[j]);
    if (FULL && i + N <= n && N == 8) {
      *reinterpret_cast<uint4*>(out + i) =
          make_uint4(pack2<__nv_bfloat16>(x[0][0], x[0][1]), pack2<__nv_bfloat16>(x[0][2], x[0][3]),
                     pack2<__nv_bfloat16>(x[N / 4 - 1][0], x[N / 4 - 1][1]),
                     pack2<__nv_bfloat16>(x[N / 4 - 1][2], x[N / 4 - 1][3]));
    } else {
#pragma unroll
      for (int j = 0; j < N / 4; ++j)
        store4(out, i + 4 * j, n, FULL && i + N <= n, x[j]);
    }
  }
}

template <typename OUT, bool SIGNED>
int launch_unpack(const void* codes, const uint8_t* scales, size_t n, void* out, cudaStream_t st) {
  const uint8_t* c = reinterpret_cast<const uint8_t*>(codes);
  OUT* o = reinterpret_cast<OUT*>(out);
  constexpr size_t kFull = 16 / sizeof(OUT);
  const bool full = (uintptr_t)c % kFull == 0 && (uintptr_t)o % 16 == 0;
  const size_t per = (full ? kFull : 4) * 4 * kThreads, blocks = (n + per - 1) / per;
  if (blocks > 0x7FFFFFFF) return NVFP4_ERR_INVALID_SHAPE;
  if (full)
    k_unpack_state<OUT, SIGNED, true><<<(unsigned)blocks, kThreads, 0, st>>>(c, scales, n, o);
  else
    k_unpack_state<OUT, SIGNED, false><<<(unsigned)blocks, kThreads, 0, st>>>(c, scales, n, o);
  return cuda_status(cudaGetLastError());
}

template <typename P, typename G, bool EIGHT, int CAP>
int launch_group(const nvfp4_adamw_tensor* tensors, int count, double lr, Args<CAP>& a,
                 cudaStream_t stream) {
  // As many launches as the tensors' chunks and the parameter block need.
  for (int at = 0; at < count;) {
    uint64_t chunks = 0;
    int k = 0;
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
      a.first_chunk[k] = (uint32_t)chunks;
      const uintptr_t state = EIGHT ? (uintptr_t)t.exp_avg % 4 | (uintptr_t)t.exp_avg_sq % 4
                                    : (uintptr_t)t.exp_avg % 16 | (uintptr_t)t.exp_avg_sq % 16;
      d.vec = ((uintptr_t)t.param % (4 * sizeof(P)) | (uintptr_t)t.grad % (4 * sizeof(G)) | state |
               (uintptr_t)t.copy % 8) == 0;
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
  if (count <= 112) {
    Args<112> a;
    return go(a);
  }
  Args<368> a;
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
  // amax_out is cleared before the scalars are read.
  auto in_amax = [&](const float* p, int words) {
    return amax_out && p && p < amax_out + count && p + words > amax_out;
  };
  if (in_amax(grad_scale, 1) || in_amax(scalars, 3)) return NVFP4_ERR_INVALID_ARGUMENT;
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
  cudaStream_t st = (cudaStream_t)stream;
  if (out_dtype == NVFP4_DTYPE_F32)
    return moment == NVFP4_EXP_AVG
               ? launch_unpack<float, true>(codes, scales, n, out, st)
               : launch_unpack<float, false>(codes, scales, n, out, st);
  return moment == NVFP4_EXP_AVG
             ? launch_unpack<__nv_bfloat16, true>(codes, scales, n, out, st)
             : launch_unpack<__nv_bfloat16, false>(codes, scales, n, out, st);
}

}  // extern "C"
