// Layer norm, forward and backward, with the reduction of the weights'
// gradients.
//
//   forward    mean_r, rstd_r = 1 / sqrt(var_r + eps);  h = (x - mean) rstd
//              y = h gamma + beta, and the amax of y that the cast of y needs
//   backward   u = dy gamma
//              dx = rstd (u - mean_c(u) - h mean_c(u h)) [+ residual]
//              dgamma_c = sum_r dy h,  dbeta_c = sum_r dy
//
// Memory-bound: every row is read once, kept in registers between its
// reduction and its output, and written once.  Where the rows are 16-byte
// aligned (k_fwd_rows, k_bwd_rows) they arrive through a ring of bulk copies
// (one thread, one mbarrier a stage), so the bytes in flight do not depend on
// how many registers a row's arithmetic leaves free; one barrier a row serves
// the reduction and, because every thread has taken its part of the stage by
// then, frees the stage.  Blocks are persistent: gamma and beta stay in
// registers, and the backward pass adds its rows' weight gradients in
// registers and writes one partial row a block, which k_bwd_reduce sums in a
// fixed order (no atomics: results repeat bit for bit).  Odd widths and
// unaligned rows take the same arithmetic with element-wise loads; rows wider
// than the registers hold are read again instead (k_fwd_wide, k_bwd_wide).
//
// The statistics come from two passes over registers: each warp's mean, then
// its sum of squares about that mean, combined over warps by
//   M2 = sum_w M2_w + n_w (mean_w - mean)^2,
// so a large common offset or an outlier costs no digits.
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

__device__ uint32_t g_layernorm_error_word;

constexpr int kMaxThreads = 512;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxStages = 8;
constexpr uint32_t kRingBytes = 96 * 1024;     // per block: two blocks fit one SM
constexpr uint64_t kWaitLimitNs = 1000000000ull;
constexpr int kMaxPartials = 296;              // partial rows of dgamma and dbeta
constexpr int kWideThreads = 256;

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
  return x;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack_one(float x) {
  if constexpr (sizeof(T) == 4) return __float_as_uint(x);
  else return pack2<T>(x, 0.0f);
}

// VEC consecutive elements: 16 bytes, or one element.
template <typename T, int VEC>
struct Pack {
  static constexpr int kWords = VEC == 1 ? 1 : 4;
  uint32_t w[kWords];
};
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& p, float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(T) == 4) {
      x[0] = __uint_as_float(p.w[0]);
    } else {
      float hi;
      unpack2<T>(p.w[0], x[0], hi);
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(p.w[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) unpack2<T>(p.w[k], x[2 * k], x[2 * k + 1]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_global(const T* p) {
  Pack<T, VEC> r;
  if constexpr (VEC == 1) {
    if constexpr (sizeof(T) == 4) r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    else r.w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
  }
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> zero_pack() {
  Pack<T, VEC> r;
#pragma unroll
  for (int k = 0; k < Pack<T, VEC>::kWords; ++k) r.w[k] = 0u;
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const float (&x)[VEC]) {
  Pack<T, VEC> r;
  if constexpr (VEC == 1) {
    r.w[0] = pack_one<T>(x[0]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) r.w[k] = __float_as_uint(x[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) r.w[k] = pack2<T>(x[2 * k], x[2 * k + 1]);
  }
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_global(T* p, const Pack<T, VEC>& r) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = r.w[0];
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)r.w[0];
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  }
}
// Unsigned maximum of the magnitudes' bit patterns, per 16-bit half or per
// word (NaN patterns are above infinity's), and its value as fp32 bits.
template <typename T, int VEC>
__device__ __forceinline__ uint32_t pack_top(uint32_t m, const Pack<T, VEC>& r) {
#pragma unroll
  for (int k = 0; k < Pack<T, VEC>::kWords; ++k)
    m = sizeof(T) == 4 ? max(m, r.w[k] & 0x7FFFFFFFu) : __vmaxu2(m, r.w[k] & 0x7FFF7FFFu);
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m;
  else {
    float lo, hi;
    unpack2<T>(m, lo, hi);
    return max(__float_as_uint(lo), __float_as_uint(hi));
  }
}

// The ring of bulk copies: ARRAYS rows a stage (x, dy, residual).
struct Ring {
  uint32_t base, bar, stage_bytes, row_bytes;
  int stages;
};

struct Shared {
  uint64_t bar[kMaxStages];
  float2 red[2][kMaxWarps];
  uint32_t abort_flag;
  uint32_t pad[3];
};

// Position of a row in the ring: its stage and the parity its barrier completes
// with.
struct RingAt {
  uint32_t stage = 0, parity = 0;
  __device__ __forceinline__ void next(const Ring& r) {
    if (++stage == (uint32_t)r.stages) { stage = 0; parity ^= 1u; }
  }
};
__device__ __forceinline__ bool ring_wait(const Ring& r, const RingAt& at,
                                          volatile uint32_t* abort_flag) {
  return mbar_wait_bounded(r.bar + 8 * at.stage, at.parity, abort_flag, kWaitLimitNs,
                           kErrTimeoutProducer, &g_layernorm_error_word);
}
// A launch that gave up: the loads in flight land before the block ends.
__device__ __forceinline__ void ring_drain(const Ring& r, RingAt at, int64_t rows_left) {
  volatile uint32_t never = 0u;
  for (int j = 0; j < r.stages && j < rows_left; ++j, at.next(r)) ring_wait(r, at, &never);
}

// Eight weights or one as fp32.
template <typename W, int VEC>
__device__ __forceinline__ void load_weights(const W* w, float (&x)[VEC]) {
#pragma unroll
  for (int k = 0; k < VEC; ++k) x[k] = to_f32(w[k]);
}

struct FwdArgs {
  const void* x;
  const void* gamma;
  const void* beta;
  void* y;
  float* mean;
  float* rstd;
  uint32_t* amax;
  int64_t rows, ldx, ldy;
  int cols, stages;
  float eps;
};

// One row per block at a time; thread t holds the vectors t, t + blockDim, ...
// BULK: the row arrives through the ring; otherwise by element-wise loads.
template <typename T, typename W, int VEC, int ITEMS, bool BULK>
__global__ void __launch_bounds__(kMaxThreads) k_fwd_rows(const FwdArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Shared sh;
  const int tid = threadIdx.x, nthr = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int nwarps = nthr >> 5, nvec = a.cols / VEC;
  const T* x = reinterpret_cast<const T*>(a.x);
  T* y = reinterpret_cast<T*>(a.y);
  Ring ring;
  ring.row_bytes = ring.stage_bytes = (uint32_t)a.cols * sizeof(T);
  ring.base = smem_addr(smem);
  ring.bar = smem_addr(sh.bar);
  ring.stages = BULK ? a.stages : 1;
  const int64_t mine = (a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x;
  auto issue = [&](int64_t k, uint32_t stage) {
    mbar_arrive_expect_tx(ring.bar + 8 * stage, ring.row_bytes);
    bulk_load(ring.base + stage * ring.stage_bytes, x + (blockIdx.x + k * gridDim.x) * a.ldx,
              ring.row_bytes, ring.bar + 8 * stage);
  };
  if constexpr (BULK) {
    if (tid == 0) {
      for (int s = 0; s < ring.stages; ++s) mbar_init(ring.bar + 8 * s, 1);
      sh.abort_flag = 0u;
      fence_barrier_init();
      for (int64_t k = 0; k < ring.stages && k < mine; ++k) issue(k, (uint32_t)k);
    }
  }
  const W* wg = reinterpret_cast<const W*>(a.gamma);
  const W* wb = reinterpret_cast<const W*>(a.beta);
  // Weights stay in registers while there is room for them.
  constexpr bool kKeep = ITEMS * VEC <= 16;
  float gamma[kKeep ? ITEMS : 1][VEC], beta[kKeep ? ITEMS : 1][VEC];
  auto weights = [&](int v, float (&g)[VEC], float (&b)[VEC]) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) g[k] = b[k] = 0.0f;
    if (v < nvec) {
      load_weights<W, VEC>(wg + v * VEC, g);
      if (wb) load_weights<W, VEC>(wb + v * VEC, b);
    }
  };
  if constexpr (kKeep) {
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) weights(tid + it * nthr, gamma[it], beta[it]);
  }
  if constexpr (BULK) __syncthreads();
  // Elements that warp `lane` holds of a row (0 for lanes without a warp).
  float nw = 0.0f;
  if (lane < nwarps) {
#pragma unroll
    for (int it = 0; it < ITEMS; ++it)
      nw += (float)(min(max(nvec - lane * 32 - it * nthr, 0), 32) * VEC);
  }
  const float own = __shfl_sync(0xFFFFFFFFu, nw, warp);
  const float inv_own = own > 0.0f ? 1.0f / own : 0.0f;
  const float inv_n = 1.0f / (float)a.cols;
  uint32_t top = 0;
  int64_t k = 0;
  RingAt at;
  for (; k < mine; ++k, at.next(ring)) {
    const int64_t row = blockIdx.x + k * gridDim.x;
    Pack<T, VEC> raw[ITEMS];
    bool ok = true;
    if constexpr (BULK) ok = ring_wait(ring, at, &sh.abort_flag);
    if (ok) {
      const T* src = BULK ? reinterpret_cast<const T*>(smem + at.stage * ring.stage_bytes)
                          : x + row * a.ldx;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        const int v = tid + it * nthr;
        raw[it] = v < nvec ? load_global<T, VEC>(src + v * VEC) : zero_pack<T, VEC>();
      }
      float s = 0.0f;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        float f[VEC];
        unpack<T, VEC>(raw[it], f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += f[j];
      }
      const float mw = warp_sum(s) * inv_own;
      float q = 0.0f;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        if (tid + it * nthr < nvec) {
          float f[VEC];
          unpack<T, VEC>(raw[it], f);
#pragma unroll
          for (int j = 0; j < VEC; ++j) q += (f[j] - mw) * (f[j] - mw);
        }
      }
      q = warp_sum(q);
      if (lane == 0) sh.red[k & 1][warp] = make_float2(mw, q);
    }
    // Everybody has taken its part of the stage and written its sums.  (The
    // sums alternate between two copies: those written next were last read
    // before this barrier.)
    __syncthreads();
    if constexpr (BULK) {
      if (*(volatile uint32_t*)&sh.abort_flag) break;
      if (tid == 0 && k + ring.stages < mine) issue(k + ring.stages, at.stage);
    }
    // Lane w joins warp w's share; every warp does so by itself.
    const float2 part = lane < nwarps ? sh.red[k & 1][lane] : make_float2(0.0f, 0.0f);
    const float mean = warp_sum(part.x * (nw * inv_n));
    const float m2 = warp_sum(part.y + nw * (part.x - mean) * (part.x - mean));
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(m2 * inv_n + a.eps));
    if (tid == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int v = tid + it * nthr;
      if (!kKeep) weights(v, gamma[0], beta[0]);
      const int w = kKeep ? it : 0;
      if (v < nvec) {
        float f[VEC];
        unpack<T, VEC>(raw[it], f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = (f[j] - mean) * rstd * gamma[w][j] + beta[w][j];
        const Pack<T, VEC> o = pack<T, VEC>(f);
        if (a.amax) top = pack_top<T, VEC>(top, o);
        store_global<T, VEC>(y + row * a.ldy + v * VEC, o);
      }
    }
  }
  if constexpr (BULK) {
    if (k < mine && tid == 0) ring_drain(ring, at, mine - k);
  }
  if (a.amax) {
    const uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, top_bits<T>(top));
    if (lane == 0 && bits) atomicMax(a.amax, bits);
  }
}

// Rows wider than the registers hold: three passes over a row, the second and
// third mostly from cache.
template <typename T, typename W>
__global__ void __launch_bounds__(kWideThreads) k_fwd_wide(const FwdArgs a) {
  __shared__ float red[2][kWideThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float inv_n = 1.0f / (float)a.cols;
  uint32_t top = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    T* y = reinterpret_cast<T*>(a.y) + row * a.ldy;
    float s = 0.0f;
    for (int c = tid; c < a.cols; c += kWideThreads) s += to_f32(x[c]);
    s = warp_sum(s);
    if (lane == 0) red[0][warp] = s;
    __syncthreads();
    float mean = 0.0f;
#pragma unroll
    for (int w = 0; w < kWideThreads / 32; ++w) mean += red[0][w];
    mean *= inv_n;
    float q = 0.0f;
    for (int c = tid; c < a.cols; c += kWideThreads) {
      const float d = to_f32(x[c]) - mean;
      q += d * d;
    }
    q = warp_sum(q);
    if (lane == 0) red[1][warp] = q;
    __syncthreads();
    float m2 = 0.0f;
#pragma unroll
    for (int w = 0; w < kWideThreads / 32; ++w) m2 += red[1][w];
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(m2 * inv_n + a.eps));
    if (tid == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    for (int c = tid; c < a.cols; c += kWideThreads) {
      const float b = a.beta ? to_f32(reinterpret_cast<const W*>(a.beta)[c]) : 0.0f;
      const float f =
          (to_f32(x[c]) - mean) * rstd * to_f32(reinterpret_cast<const W*>(a.gamma)[c]) + b;
      const T o = from_f32<T>(f);
      top = max(top, __float_as_uint(to_f32(o)) & 0x7FFFFFFFu);
      y[c] = o;
    }
  }
  if (a.amax) {
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if (lane == 0 && top) atomicMax(a.amax, top);
  }
}

struct BwdArgs {
  const void* dy;
  const void* x;
  const float* mean;
  const float* rstd;
  const void* gamma;
  const void* res;
  void* dx;
  float* partial;       // [partials][2][cols]: sums of dy h, sums of dy
  int64_t rows, lddy, ldx, ldr, lddx;
  int cols, stages, partials;
};

template <typename T, typename W, int VEC, int ITEMS, bool BULK, bool RES>
__global__ void __launch_bounds__(kMaxThreads) k_bwd_rows(const BwdArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Shared sh;
  constexpr int kArrays = RES ? 3 : 2;
  const int tid = threadIdx.x, nthr = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int nwarps = nthr >> 5, nvec = a.cols / VEC;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* dy = reinterpret_cast<const T*>(a.dy);
  const T* res = reinterpret_cast<const T*>(a.res);
  T* dx = reinterpret_cast<T*>(a.dx);
  Ring ring;
  ring.row_bytes = (uint32_t)a.cols * sizeof(T);
  ring.stage_bytes = kArrays * ring.row_bytes;
  ring.base = smem_addr(smem);
  ring.bar = smem_addr(sh.bar);
  ring.stages = BULK ? a.stages : 1;
  const int64_t mine = (a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x;
  auto issue = [&](int64_t k, uint32_t stage) {
    const uint32_t bar = ring.bar + 8 * stage, dst = ring.base + stage * ring.stage_bytes;
    const int64_t row = blockIdx.x + k * gridDim.x;
    mbar_arrive_expect_tx(bar, ring.stage_bytes);
    bulk_load(dst, x + row * a.ldx, ring.row_bytes, bar);
    bulk_load(dst + ring.row_bytes, dy + row * a.lddy, ring.row_bytes, bar);
    if constexpr (RES)
      bulk_load(dst + 2 * ring.row_bytes, res + row * a.ldr, ring.row_bytes, bar);
  };
  if constexpr (BULK) {
    if (tid == 0) {
      for (int s = 0; s < ring.stages; ++s) mbar_init(ring.bar + 8 * s, 1);
      sh.abort_flag = 0u;
      fence_barrier_init();
      for (int64_t k = 0; k < ring.stages && k < mine; ++k) issue(k, (uint32_t)k);
    }
  }
  const W* wg = reinterpret_cast<const W*>(a.gamma);
  constexpr bool kKeep = ITEMS * VEC <= 16;      // gamma stays in registers
  float gamma[kKeep ? ITEMS : 1][VEC], dg[ITEMS][VEC], db[ITEMS][VEC];
  auto weights = [&](int v, float (&g)[VEC]) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) g[k] = 0.0f;
    if (v < nvec) load_weights<W, VEC>(wg + v * VEC, g);
  };
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    if constexpr (kKeep) weights(tid + it * nthr, gamma[it]);
#pragma unroll
    for (int k = 0; k < VEC; ++k) dg[it][k] = db[it][k] = 0.0f;
  }
  if constexpr (BULK) __syncthreads();
  const float inv_n = 1.0f / (float)a.cols;
  int64_t k = 0;
  RingAt at;
  // A row's statistics are fetched a row ahead.
  float next_mean = mine > 0 ? a.mean[blockIdx.x] : 0.0f;
  float next_rstd = mine > 0 ? a.rstd[blockIdx.x] : 0.0f;
  for (; k < mine; ++k, at.next(ring)) {
    const int64_t row = blockIdx.x + k * gridDim.x;
    const float mean = next_mean, rstd = next_rstd;
    if (k + 1 < mine) {
      next_mean = a.mean[row + gridDim.x];
      next_rstd = a.rstd[row + gridDim.x];
    }
    Pack<T, VEC> px[ITEMS], pd[ITEMS], pr[RES ? ITEMS : 1];
    bool ok = true;
    if constexpr (BULK) ok = ring_wait(ring, at, &sh.abort_flag);
    if (ok) {
      const unsigned char* st = smem + at.stage * ring.stage_bytes;
      const T* sx = BULK ? reinterpret_cast<const T*>(st) : x + row * a.ldx;
      const T* sd = BULK ? reinterpret_cast<const T*>(st + ring.row_bytes) : dy + row * a.lddy;
      const T* sr = BULK ? reinterpret_cast<const T*>(st + 2 * ring.row_bytes) : res + row * a.ldr;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        const int v = tid + it * nthr;
        const bool in = v < nvec;
        px[it] = in ? load_global<T, VEC>(sx + v * VEC) : zero_pack<T, VEC>();
        pd[it] = in ? load_global<T, VEC>(sd + v * VEC) : zero_pack<T, VEC>();
        if constexpr (RES) pr[it] = in ? load_global<T, VEC>(sr + v * VEC) : zero_pack<T, VEC>();
      }
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        const int v = tid + it * nthr;
        if (!kKeep) weights(v, gamma[0]);
        const int w = kKeep ? it : 0;
        if (v < nvec) {
          float fx[VEC], fd[VEC];
          unpack<T, VEC>(px[it], fx);
          unpack<T, VEC>(pd[it], fd);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float h = (fx[j] - mean) * rstd;
            const float u = fd[j] * gamma[w][j];
            s1 += u;
            s2 += u * h;
            dg[it][j] += fd[j] * h;
            db[it][j] += fd[j];
          }
        }
      }
      s1 = warp_sum(s1);
      s2 = warp_sum(s2);
      if (lane == 0) sh.red[k & 1][warp] = make_float2(s1, s2);
    }
    __syncthreads();
    if constexpr (BULK) {
      if (*(volatile uint32_t*)&sh.abort_flag) break;
      if (tid == 0 && k + ring.stages < mine) issue(k + ring.stages, at.stage);
    }
    const float2 part = lane < nwarps ? sh.red[k & 1][lane] : make_float2(0.0f, 0.0f);
    const float c1 = warp_sum(part.x) * inv_n, c2 = warp_sum(part.y) * inv_n;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int v = tid + it * nthr;
      if (!kKeep) weights(v, gamma[0]);
      const int w = kKeep ? it : 0;
      if (v < nvec) {
        float fx[VEC], fd[VEC], fr[VEC];
        unpack<T, VEC>(px[it], fx);
        unpack<T, VEC>(pd[it], fd);
        if constexpr (RES) unpack<T, VEC>(pr[it], fr);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float h = (fx[j] - mean) * rstd;
          fx[j] = rstd * (fd[j] * gamma[w][j] - c1 - h * c2);
          if constexpr (RES) fx[j] += fr[j];
        }
        store_global<T, VEC>(dx + row * a.lddx + v * VEC, pack<T, VEC>(fx));
      }
    }
  }
  if constexpr (BULK) {
    if (k < mine && tid == 0) ring_drain(ring, at, mine - k);
  }
  float* out = a.partial + (size_t)blockIdx.x * 2 * a.cols;
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const int v = tid + it * nthr;
    if (v < nvec) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        out[v * VEC + j] = dg[it][j];
        out[a.cols + v * VEC + j] = db[it][j];
      }
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kWideThreads) k_bwd_wide_dx(const BwdArgs a) {
  __shared__ float red[2][kWideThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float inv_n = 1.0f / (float)a.cols;
  const W* gamma = reinterpret_cast<const W*>(a.gamma);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.lddy;
    const T* res = a.res ? reinterpret_cast<const T*>(a.res) + row * a.ldr : nullptr;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.lddx;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = tid; c < a.cols; c += kWideThreads) {
      const float u = to_f32(dy[c]) * to_f32(gamma[c]);
      s1 += u;
      s2 += u * (to_f32(x[c]) - mean) * rstd;
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    __syncthreads();   // the previous row's sums have been read
    if (lane == 0) {
      red[0][warp] = s1;
      red[1][warp] = s2;
    }
    __syncthreads();
    float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
    for (int w = 0; w < kWideThreads / 32; ++w) {
      c1 += red[0][w];
      c2 += red[1][w];
    }
    c1 *= inv_n;
    c2 *= inv_n;
    for (int c = tid; c < a.cols; c += kWideThreads) {
      const float h = (to_f32(x[c]) - mean) * rstd;
      float f = rstd * (to_f32(dy[c]) * to_f32(gamma[c]) - c1 - h * c2);
      if (res) f += to_f32(res[c]);
      dx[c] = from_f32<T>(f);
    }
  }
}

// Weight-gradient partials of the wide rows: block (bx, by) sums the rows by,
// by + partials, ... of its columns.
template <typename T>
__global__ void __launch_bounds__(kWideThreads) k_bwd_wide_w(const BwdArgs a) {
  const int64_t c = (int64_t)blockIdx.x * kWideThreads + threadIdx.x;
  if (c >= a.cols) return;
  float dg = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float d = to_f32(reinterpret_cast<const T*>(a.dy)[row * a.lddy + c]);
    const float h = (to_f32(reinterpret_cast<const T*>(a.x)[row * a.ldx + c]) - a.mean[row]) *
                    a.rstd[row];
    dg += d * h;
    db += d;
  }
  float* out = a.partial + (size_t)blockIdx.y * 2 * a.cols;
  out[c] = dg;
  out[a.cols + c] = db;
}

// dgamma, dbeta: the partial rows summed in a fixed order.  32 columns of one
// of the two outputs a block; 8 warps take every eighth partial row.
template <typename W>
__global__ void __launch_bounds__(256) k_bwd_reduce(const float* __restrict__ partial,
                                                    int partials, int cols, W* dgamma, W* dbeta) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float v = 0.0f;
  if (c < cols) {
    const float* p = partial + (size_t)which * cols + c;
    for (int r = warp; r < partials; r += 8) v += p[(size_t)r * 2 * cols];
  }
  s[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < cols) {
#pragma unroll
    for (int w = 1; w < 8; ++w) v += s[w][lane];
    W* out = which == 0 ? dgamma : dbeta;
    if (out) out[c] = from_f32<W>(v);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// How a row is laid over threads: `items` vectors a thread, few enough threads
// that none is idle for most of the row.
struct Shape {
  int items, threads;
};
// items are 1, 2 or 4; false: the row is wider than the registers hold.
bool row_shape(int64_t nvec, int want, Shape* s) {
  for (int items : {want, 4}) {
    while (items > 1 && nvec <= (int64_t)items / 2 * 32) items /= 2;
    const int64_t threads = ((nvec + items - 1) / items + 31) / 32 * 32;
    if (threads <= kMaxThreads) {
      *s = {items, (int)threads};
      return true;
    }
  }
  return false;
}

template <typename K>
int set_smem(K kernel, size_t bytes) {
  // 48 KB is the default limit of static and dynamic memory together.
  if (bytes + sizeof(Shared) > 48 * 1024)
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)bytes))
      return cuda_status(e);
  return NVFP4_OK;
}

int ring_stages(size_t stage_bytes) {
  const size_t s = kRingBytes / stage_bytes;
  return (int)(s < 2 ? 2 : s > kMaxStages ? kMaxStages : s);
}

// Blocks of a persistent grid: as many as fit at once, at most one a row.
template <typename K>
int grid_of(K kernel, int threads, size_t smem, int64_t rows, int sms, int64_t most,
            unsigned* grid) {
  int per_sm = 0;
  if (cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem))
    return cuda_status(e);
  int64_t g = (int64_t)(per_sm < 1 ? 1 : per_sm) * sms;
  if (g > most) g = most;
  *grid = (unsigned)(g < rows ? g : rows);
  return NVFP4_OK;
}

template <typename T, typename W, int VEC, int ITEMS, bool BULK>
int launch_fwd_rows(FwdArgs a, int threads, int sms, cudaStream_t st) {
  auto kernel = k_fwd_rows<T, W, VEC, ITEMS, BULK>;
  size_t smem = 0;
  if constexpr (BULK) {
    a.stages = ring_stages((size_t)a.cols * sizeof(T));
    smem = (size_t)a.stages * a.cols * sizeof(T);
    if (int e = set_smem(kernel, smem)) return e;
  }
  unsigned grid;
  if (int e = grid_of(kernel, threads, smem, a.rows, sms, INT32_MAX, &grid)) return e;
  kernel<<<grid, threads, smem, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename T, typename W>
int launch_fwd(const FwdArgs& a, int sms, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool bulk = ((uintptr_t)a.x % 16 | (uintptr_t)a.y % 16 | (uintptr_t)(a.ldx % V) |
                     (uintptr_t)(a.ldy % V) | (uintptr_t)(a.cols % V)) == 0;
  Shape s;
  if (bulk && row_shape(a.cols / V, 2, &s)) {
    switch (s.items) {
      case 1: return launch_fwd_rows<T, W, V, 1, true>(a, s.threads, sms, st);
      case 2: return launch_fwd_rows<T, W, V, 2, true>(a, s.threads, sms, st);
      default: return launch_fwd_rows<T, W, V, 4, true>(a, s.threads, sms, st);
    }
  }
  if (a.cols <= 16 * kMaxThreads) {
    const int threads = ((a.cols + 15) / 16 + 31) / 32 * 32;
    return launch_fwd_rows<T, W, 1, 16, false>(a, threads, sms, st);
  }
  const int64_t most = (int64_t)sms * 8;
  k_fwd_wide<T, W><<<(unsigned)(a.rows < most ? a.rows : most), kWideThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename T, typename W, int VEC, int ITEMS, bool BULK, bool RES>
int launch_bwd_rows(BwdArgs& a, int threads, int sms, cudaStream_t st) {
  auto kernel = k_bwd_rows<T, W, VEC, ITEMS, BULK, RES>;
  size_t smem = 0;
  if constexpr (BULK) {
    const size_t stage = (size_t)a.cols * sizeof(T) * (RES ? 3 : 2);
    a.stages = ring_stages(stage);
    smem = a.stages * stage;
    if (int e = set_smem(kernel, smem)) return e;
  }
  unsigned grid;
  if (int e = grid_of(kernel, threads, smem, a.rows, sms, kMaxPartials, &grid)) return e;
  a.partials = (int)grid;
  kernel<<<grid, threads, smem, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename T, typename W, bool RES>
int launch_bwd(BwdArgs& a, int sms, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool bulk = ((uintptr_t)a.x % 16 | (uintptr_t)a.dy % 16 | (uintptr_t)a.dx % 16 |
                     (uintptr_t)a.res % 16 | (uintptr_t)(a.ldx % V) | (uintptr_t)(a.lddy % V) |
                     (uintptr_t)(a.lddx % V) | (uintptr_t)(RES ? a.ldr % V : 0) |
                     (uintptr_t)(a.cols % V)) == 0;
  Shape s;
  if (bulk && row_shape(a.cols / V, 2, &s)) {
    switch (s.items) {
      case 1: return launch_bwd_rows<T, W, V, 1, true, RES>(a, s.threads, sms, st);
      case 2: return launch_bwd_rows<T, W, V, 2, true, RES>(a, s.threads, sms, st);
      default: return launch_bwd_rows<T, W, V, 4, true, RES>(a, s.threads, sms, st);
    }
  }
  if (a.cols <= 16 * kMaxThreads) {
    const int threads = ((a.cols + 15) / 16 + 31) / 32 * 32;
    return launch_bwd_rows<T, W, 1, 16, false, RES>(a, threads, sms, st);
  }
  // The weights' partial sums first: dx may overwrite dy.
  a.partials = (int)(a.rows < kMaxPartials ? a.rows : kMaxPartials);
  const dim3 grid((unsigned)((a.cols + kWideThreads - 1) / kWideThreads), (unsigned)a.partials);
  k_bwd_wide_w<T><<<grid, kWideThreads, 0, st>>>(a);
  if (cudaError_t e = cudaGetLastError()) return cuda_status(e);
  const int64_t most = (int64_t)sms * 8;
  k_bwd_wide_dx<T, W><<<(unsigned)(a.rows < most ? a.rows : most), kWideThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename W>
int launch_reduce(const BwdArgs& a, void* dgamma, void* dbeta, cudaStream_t st) {
  k_bwd_reduce<W><<<dim3((unsigned)((a.cols + 31) / 32), 2), 256, 0, st>>>(
      a.partial, a.partials, a.cols, reinterpret_cast<W*>(dgamma), reinterpret_cast<W*>(dbeta));
  return cuda_status(cudaGetLastError());
}

size_t elem_size(int dtype) { return dtype == NVFP4_DTYPE_F32 ? 4 : 2; }
bool known_dtype(int d) { return d >= NVFP4_DTYPE_F32 && d <= NVFP4_DTYPE_F16; }

}  // namespace

int layernorm_device_error(uint32_t* code, int clear) {
  if (cudaError_t e = cudaMemcpyFromSymbol(code, g_layernorm_error_word, sizeof(uint32_t)))
    return cuda_status(e);
  if (clear && *code) {
    const uint32_t zero = 0;
    if (cudaError_t e = cudaMemcpyToSymbol(g_layernorm_error_word, &zero, sizeof(uint32_t)))
      return cuda_status(e);
  }
  return NVFP4_OK;
}

}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

NVFP4_API int nvfp4_layernorm_fwd(int64_t rows, int64_t cols, const void* x, int64_t ldx,
                                  const void* gamma, const void* beta, int dtype,
                                  int weight_dtype, float eps, void* y, int64_t ldy, float* mean,
                                  float* rstd, float* amax_out, nvfp4_stream_t stream) {
  if (rows < 0 || cols < 0 || cols > (1 << 24) || rows > ((int64_t)1 << 31) || ldx < cols ||
      ldy < cols)
    return NVFP4_ERR_INVALID_SHAPE;
  if (!known_dtype(dtype) || (weight_dtype != dtype && weight_dtype != NVFP4_DTYPE_F32) ||
      !(eps >= 0.0f))
    return NVFP4_ERR_INVALID_ARGUMENT;
  const uintptr_t es = elem_size(dtype), ws = elem_size(weight_dtype);
  const bool empty = rows == 0 || cols == 0;
  if (!empty && (!x || !gamma || !y)) return NVFP4_ERR_INVALID_ARGUMENT;
  if ((uintptr_t)x % es || (uintptr_t)y % es || (uintptr_t)gamma % ws || (uintptr_t)beta % ws ||
      (uintptr_t)mean % 4 || (uintptr_t)rstd % 4 || (uintptr_t)amax_out % 4)
    return NVFP4_ERR_MISALIGNED;
  if (empty && !amax_out) return NVFP4_OK;
  int sms = 0;
  if (int e = device_sm_count(&sms)) return e;
  cudaStream_t st = (cudaStream_t)stream;
  if (amax_out)
    if (cudaError_t e = cudaMemsetAsync(amax_out, 0, sizeof(float), st)) return cuda_status(e);
  if (empty) return NVFP4_OK;
  FwdArgs a = {x, gamma, beta, y, mean, rstd, reinterpret_cast<uint32_t*>(amax_out),
               rows, ldx, ldy, (int)cols, 1, eps};
  if (dtype == NVFP4_DTYPE_F32) return launch_fwd<float, float>(a, sms, st);
  if (dtype == NVFP4_DTYPE_BF16)
    return weight_dtype == NVFP4_DTYPE_F32 ? launch_fwd<__nv_bfloat16, float>(a, sms, st)
                                           : launch_fwd<__nv_bfloat16, __nv_bfloat16>(a, sms, st);
  return weight_dtype == NVFP4_DTYPE_F32 ? launch_fwd<__half, float>(a, sms, st)
                                         : launch_fwd<__half, __half>(a, sms, st);
}

NVFP4_API size_t nvfp4_layernorm_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)(rows < kMaxPartials ? rows : kMaxPartials) * 2 * (size_t)cols * sizeof(float);
}

NVFP4_API int nvfp4_layernorm_bwd(int64_t rows, int64_t cols, const void* dy, int64_t lddy,
                                  const void* x, int64_t ldx, const float* mean,
                                  const float* rstd, const void* gamma, const void* residual,
                                  int64_t ldr, int dtype, int weight_dtype, void* dx,
                                  int64_t lddx, void* dgamma, void* dbeta, void* workspace,
                                  size_t workspace_bytes, nvfp4_stream_t stream) {
  if (rows < 0 || cols < 0 || cols > (1 << 24) || rows > ((int64_t)1 << 31) || lddy < cols ||
      ldx < cols || lddx < cols || (residual && ldr < cols))
    return NVFP4_ERR_INVALID_SHAPE;
  if (!known_dtype(dtype) || (weight_dtype != dtype && weight_dtype != NVFP4_DTYPE_F32))
    return NVFP4_ERR_INVALID_ARGUMENT;
  const uintptr_t es = elem_size(dtype), ws = elem_size(weight_dtype);
  if (cols == 0) return NVFP4_OK;
  if (rows > 0 && (!dy || !x || !mean || !rstd || !gamma || !dx || !workspace ||
                   workspace_bytes < nvfp4_layernorm_bwd_workspace_bytes(rows, cols)))
    return NVFP4_ERR_INVALID_ARGUMENT;
  if ((uintptr_t)dy % es || (uintptr_t)x % es || (uintptr_t)residual % es || (uintptr_t)dx % es ||
      (uintptr_t)gamma % ws || (uintptr_t)dgamma % ws || (uintptr_t)dbeta % ws ||
      (uintptr_t)mean % 4 || (uintptr_t)rstd % 4 || (uintptr_t)workspace % 4)
    return NVFP4_ERR_MISALIGNED;
  int sms = 0;
  if (int e = device_sm_count(&sms)) return e;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    // No rows: the weights' gradients are empty sums.
    if (dgamma)
      if (cudaError_t e = cudaMemsetAsync(dgamma, 0, cols * ws, st)) return cuda_status(e);
    if (dbeta)
      if (cudaError_t e = cudaMemsetAsync(dbeta, 0, cols * ws, st)) return cuda_status(e);
    return NVFP4_OK;
  }
  BwdArgs a = {dy, x, mean, rstd, gamma, residual, dx, reinterpret_cast<float*>(workspace),
               rows, lddy, ldx, ldr, lddx, (int)cols, 1, 0};
  auto rows_of = [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    const int e = residual ? launch_bwd<T, W, true>(a, sms, st) : launch_bwd<T, W, false>(a, sms, st);
    if (e || (!dgamma && !dbeta)) return e;
    return launch_reduce<W>(a, dgamma, dbeta, st);
  };
  if (dtype == NVFP4_DTYPE_F32) return rows_of(float(), float());
  if (dtype == NVFP4_DTYPE_BF16)
    return weight_dtype == NVFP4_DTYPE_F32 ? rows_of(__nv_bfloat16(), float())
                                           : rows_of(__nv_bfloat16(), __nv_bfloat16());
  return weight_dtype == NVFP4_DTYPE_F32 ? rows_of(__half(), float())
                                         : rows_of(__half(), __half());
}

}  // extern "C"
