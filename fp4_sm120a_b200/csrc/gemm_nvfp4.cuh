// Parts shared by the two product kernels: parameters, bounded waits, tcgen05
// block-scaled wrappers, activations.
#pragma once

#include <cstdint>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "element_io.cuh"
#include "launch_common.h"
#include "nvfp4_b200.h"
#include "nvfp4_device.cuh"

namespace nvfp4 {
namespace gemm {

constexpr int kTileF = 128;                  // n side of a CTA's tile: TMEM lanes
constexpr int kSliceK = 256;                 // codes per k-slice (128 bytes)
constexpr int kSteps = kSliceK / 64;         // MMAs per k-slice
constexpr int kEpiWarps = 8;
constexpr int kEpiThreads = 32 * kEpiWarps;
constexpr uint32_t kAtomBytes = 512;         // scales of 128 rows x one MMA step
constexpr uint32_t kSmemMax = 227 * 1024;
constexpr uint64_t kWaitLimitNs = 1000000000ull;

enum Activation : int { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

struct Params {
  int m, n, k;
  int slices;                 // ceil(k / 256)
  int tiles_f, tiles_t;
  const uint8_t* sf_f;        // scales of the n side (B), pitch k / 16
  const uint8_t* sf_t;        // scales of the m side (A)
  int sf_pitch;
  int sf_width_f, sf_width_t;   // bytes per scale load: 16, 4 or 1
  const float* amax_f;
  const float* amax_t;
  void* d;
  int64_t ldd;
  const void* bias;
  int bias_dtype;
  const void* res;            // forward: residual; backward: the activation's argument
  int64_t ldr;
  void* aux;
  int64_t ldaux;
  int act;
  float* dbias_partial;       // [partial rows][n]
  uint32_t* amax;
  int vec;                    // rows of D, residual / argument and aux are 16-byte aligned (wide kernel)
};

// Launch of the wide kernel (tiles of 256 (n) x tn (m) by pairs of CTAs); the
// scales first go to `scale_ws` in the order the kernel copies them.
size_t wide_scale_bytes(int64_t m, int64_t n, int64_t k);
int launch_wide(int dtype, bool dact, int tn, const Params& p, const void* a, const void* b,
                void* scale_ws, int sms, cudaStream_t st);
int wide_device_error(uint32_t* code, int clear);

// Tensor map of packed codes [rows, k / 2], box 128 bytes x `box_rows`,
// 128-byte swizzle; and of 32-bit words [rows, 256], box 256 x 2.
int encode_codes_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t k, int box_rows);
int encode_words_map(CUtensorMap* map, const void* ptr, int64_t rows);

namespace {
// Error word of the kernels of one source file (see nvfp4_device_error).
__device__ uint32_t g_gemm_error_word;
}  // namespace

// Reads (and with clear resets) the word of the including source file.
static inline int read_error_word(uint32_t* code, int clear) {
  if (cudaError_t e = cudaMemcpyFromSymbol(code, g_gemm_error_word, sizeof(uint32_t)))
    return cuda_status(e);
  if (clear && *code) {
    const uint32_t zero = 0;
    if (cudaError_t e = cudaMemcpyToSymbol(g_gemm_error_word, &zero, sizeof(uint32_t)))
      return cuda_status(e);
  }
  return NVFP4_OK;
}

template <bool RELAXED = false>
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                     uint32_t err) {
  return mbar_wait_bounded<RELAXED>(bar, parity, abort_flag, kWaitLimitNs, err,
                                    &g_gemm_error_word);
}

// The same by a whole warp, which stays together.
template <bool RELAXED = false>
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity,
                                          volatile uint32_t* abort_flag, uint32_t err) {
  return __all_sync(0xFFFFFFFFu, wait<RELAXED>(bar, parity, abort_flag, err));
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(r));
  return r != 0;
}

// tcgen05.mma, block-scaled: D (+)= (A sfa) (B sfb)^T, one E4M3 scale for each
// 16 elements of a row.
__device__ __forceinline__ void mma_nvfp4(uint32_t d, uint64_t a_desc, uint64_t b_desc,
                                          uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X "
      "[%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 32 rows of 16 bytes to 32 lanes x 4 columns, repeated for the four warps' lanes.
__device__ __forceinline__ void cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z,
                                       uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z),
               "r"(w)
               : "memory");
}
__device__ __forceinline__ void sts_f32(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// 16 scale bytes (one k-slice) of a row (null: zeros); bytes behind the row's
// end are zero.
__device__ __forceinline__ uint4 load_scales(const uint8_t* row, int pitch, int width, int slice) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  if (row != nullptr) {
    const uint8_t* p = row + slice * 16;
    const int left = pitch - slice * 16;
    if (width == 16) return *reinterpret_cast<const uint4*>(p);
    if (width == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * i < left) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < left) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Widest load that a scale matrix's address and pitch allow: 16, 4 or 1 bytes.
static inline int scale_width(const void* sf, int64_t pitch) {
  if ((uintptr_t)sf % 16 == 0 && pitch % 16 == 0) return 16;
  if ((uintptr_t)sf % 4 == 0 && pitch % 4 == 0) return 4;
  return 1;
}

// COLS consecutive fp32 columns of this thread's TMEM lane.
template <int COLS>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, float (&v)[COLS]) {
  if constexpr (COLS == 16) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
  } else {
    static_assert(COLS == 8, "8 or 16 columns");
    uint32_t r[8];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
  }
}

// 1 / (1 + exp(-x)).  Where 2^-126 is the difference, 1 + exp(-x) does not show it.
__device__ __forceinline__ float sigmoid(float x) {
  return fast_rcp(1.0f + fast_exp2(-1.4426950408889634f * x));
}

constexpr float kGeluC = 1.5957691216057308f;    // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// 0.5 z (1 + tanh(c z (1 + a z^2))) = z sigmoid(2 c z (1 + a z^2))
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == kRelu) return z > 0.0f ? z : (z != z ? z : 0.0f);
  if constexpr (ACT == kGelu) return z * sigmoid(kGeluC * z * (1.0f + kGeluA * z * z));
  if constexpr (ACT == kSilu) return z * sigmoid(z);
  return z;
}
template <int ACT>
__device__ __forceinline__ float slope(float z) {
  if constexpr (ACT == kRelu) return z > 0.0f ? 1.0f : 0.0f;
  // Beyond |z| = 64 both slopes are 0 or 1 to the last bit; the clamp keeps
  // powers of a huge argument from overflowing (and lets NaN through).
  const float c = fmax_nan(fmin_nan(z, 64.0f), -64.0f);
  if constexpr (ACT == kGelu) {
    const float q = sigmoid(kGeluC * c * (1.0f + kGeluA * c * c));
    return q + c * q * (1.0f - q) * kGeluC * (1.0f + 3.0f * kGeluA * c * c);
  }
  if constexpr (ACT == kSilu) {
    const float q = sigmoid(c);
    return q + c * q * (1.0f - q);
  }
  return 1.0f;
}

__device__ __forceinline__ float load_bias(const Params& p, int f) {
  if (!p.bias) return 0.0f;
  if (p.bias_dtype == NVFP4_DTYPE_F32) return reinterpret_cast<const float*>(p.bias)[f];
  if (p.bias_dtype == NVFP4_DTYPE_BF16)
    return to_f32(reinterpret_cast<const __nv_bfloat16*>(p.bias)[f]);
  return to_f32(reinterpret_cast<const __half*>(p.bias)[f]);
}

// Tiles in an order that keeps a wave's tiles near a square: groups of
// kGroup column tiles, walked feature tile by feature tile.
constexpr int kGroup = 8;
__device__ __forceinline__ void tile_at(const Params& p, int i, int& tf, int& tt) {
  const int per = kGroup * p.tiles_f;
  const int g = i / per, in = i - g * per;
  const int wide = min(kGroup, p.tiles_t - g * kGroup);
  tf = in / wide;
  tt = g * kGroup + in - tf * wide;
}

}  // namespace gemm
}  // namespace nvfp4
