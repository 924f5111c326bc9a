// Product of two NVFP4 matrices with a fused epilogue, for B200 (sm_100a).
//
//   z[i, j] = S_a S_b sum_k (a[i, k] sfa[i, k / 16]) (b[j, k] sfb[j, k / 16]) + bias[j]
//   nvfp4_gemm        D = act(z) + residual, aux = z
//   nvfp4_gemm_dact   D = z act'(aux), dbias[j] = sum_i D[i, j]
//
// with S = 1 / global_encode_scale(amax) of each operand, the scale that the
// casts of this library divide out.  Both operands are what the casts write:
// packed E2M1 rows along k and row-major E4M3 scales of 16-element blocks.
//
// The products run on the tensor cores' block-scaled form (kind::mxf4nvf4,
// one E4M3 scale per 16 elements, fp32 accumulators in TMEM): code products
// and scales are exact there, only the accumulation rounds.
//
// Orientation: the n side (weights) lies along the 128 TMEM lanes and the m
// side (tokens) along the accumulator's columns.  A short m then costs a
// narrow column tile rather than an empty lane tile, bias is one register a
// thread, a warp's stores cover 32 consecutive elements of a row of D, and a
// column sum of D (the bias gradient) never leaves a thread.
//
// Products of many tiles take the kernel in gemm_nvfp4_wide_sm100.cu.  Here:
// output tiles of 128 (n) x TN (m), warp-specialised:
//   warps 0-7   epilogue: two groups of four warps, each half of the columns
//   warp  8     TMA producer: 128-byte k-slices (256 codes) of both operands
//               into a ring of 128-byte-swizzled stages
//   warp  9     MMA issuer: copies a stage's scales to TMEM (tcgen05.cp),
//               issues four K = 64 MMAs; owns the TMEM columns
//   warps 10-11 scale loaders: the casts' row-major scales into the 32 x 16
//               byte atoms that tcgen05.cp spreads over the lanes.  A lane
//               takes 16 bytes (one k-slice) of rows l, l + 32, l + 64, l + 96,
//               so the transpose is a choice of registers.
// Few tiles (short m): the k range is split over a cluster of up to 8 CTAs,
// whose partial tiles meet in distributed shared memory and are added in rank
// order (no atomics: results repeat bit for bit).
// Measured, on the device: 1 x 5120 x 5120 7.7 us (14.8 MB; a launch, the first
// loads' latency and the cluster's join are most of it), 37 x 5000 x 8192 11.2 us
// (24 MB), 64 x 5120 x 5120 10.8 us.  The bytes alone would take 2.3, 3.7 and
// 2.4 us.
// Every wait is bounded; a kernel that gives up records an error word, waits
// for its own copies and MMAs, frees TMEM and returns.
#include <cstdint>
#include <mutex>

#include <cudaTypedefs.h>

#include "gemm_nvfp4.cuh"

namespace nvfp4 {
namespace gemm {

constexpr int kWarpTma = 8, kWarpMma = 9, kWarpScales = 10;
constexpr int kMaxSplit = 8;

// Tile widths and what follows from them.
template <int TN>
struct Tile {
  static constexpr uint32_t kBytesF = kTileF * 128;
  static constexpr uint32_t kBytesT = TN * 128;
  static constexpr uint32_t kBytesSf = kSteps * 2 * kAtomBytes;
  static constexpr uint32_t kStageBytes = kBytesF + kBytesT + kBytesSf;
  static constexpr uint32_t kPlaceBytes = 2 * 128 * 16;      // scales in flight, a stage
  // Two CTAs an SM: a split that does not divide the SMs evenly still runs in
  // one wave, and one CTA's epilogue meets the other's products.
  static constexpr int kCtasPerSm = 2;
  static constexpr uint32_t kBudget = kSmemMax / kCtasPerSm - 2048;
  static constexpr int kStagesRaw = (int)(kBudget / (kStageBytes + kPlaceBytes));
  static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;
  static constexpr int kAccStages = 2;
  static constexpr uint32_t kSfCols = kSteps * 4 * 2;      // TMEM columns of a slice's scales
  static constexpr uint32_t kColsUsed = kAccStages * TN + 2 * kSfCols;
  static constexpr uint32_t kTmemCols = kColsUsed <= 128 ? 128 : kColsUsed <= 256 ? 256 : 512;
  static constexpr uint32_t kSmemBytes = kStages * (kStageBytes + kPlaceBytes) + 1024;
  static constexpr int kThreads = 32 * (kWarpScales + 2);
  static_assert(kStages >= 3, "the scale columns of slice g - 2 are checked through its stage");
  static_assert(kColsUsed <= 512, "TMEM");
  static_assert(kTmemCols * kCtasPerSm <= 512, "TMEM of all CTAs of an SM");
  // Instruction descriptor, kind::mxf4nvf4: E2M1 operands, both K-major,
  // UE4M3 scales, N = TN, M = 128.
  static constexpr uint32_t kIdesc =
      (1u << 7) | (1u << 10) | ((uint32_t)(TN / 8) << 17) | ((uint32_t)(kTileF / 16) << 24);
};

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// 16 scale bytes (one k-slice) of a row (null: zeros) on their way to shared
// memory; bytes behind the row's end become zero.
__device__ __forceinline__ void fetch_scales(uint32_t dst, const uint8_t* row,
                                             const uint8_t* any, int pitch, int width, int slice) {
  const uint8_t* p = row ? row + slice * 16 : any;
  const int left = row ? pitch - slice * 16 : 0;
  if (width == 16) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p),
                 "r"(left > 0 ? 16 : 0)
                 : "memory");
  } else if (width == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = 4 * i < left;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * i),
                   "l"(in ? p + 4 * i : any), "r"(in ? 4 : 0)
                   : "memory");
    }
  } else {
    const uint4 v = load_scales(row, pitch, width, slice);
    sts128(dst, v.x, v.y, v.z, v.w);
  }
}

// A thread's share of a tile: one feature (lane) and COLS columns from
// column c0 on, the accumulator's values in v.
struct Out {
  float alpha, bias;
  float dbias;
  uint32_t top;
};

template <typename T, bool DACT, int ACT, int COLS>
__device__ __forceinline__ void finish_act(const Params& p, Out& o, float (&v)[COLS],
                                           const float (&r)[COLS], int f, int t0, int step,
                                           int count) {
  T* d = reinterpret_cast<T*>(p.d) + f;
#pragma unroll
  for (int j = 0; j < COLS; ++j) {
    if (j < count) {
      const int64_t t = t0 + (int64_t)j * step;
      float x;
      if constexpr (DACT) {
        x = v[j] * o.alpha * slope<ACT>(r[j]);
        o.dbias += x;
      } else {
        const float z = v[j] * o.alpha + o.bias;
        if (p.aux) reinterpret_cast<T*>(p.aux)[t * p.ldaux + f] = from_f32<T>(z);
        x = activate<ACT>(z) + r[j];
      }
      const T s = from_f32<T>(x);
      d[t * p.ldd] = s;
      o.top = max(o.top, __float_as_uint(to_f32(s)) & 0x7FFFFFFFu);
    }
  }
}

// Epilogue of COLS columns (tokens t0, t0 + step, ...; the first `count` are real).
template <typename T, bool DACT, int COLS>
__device__ __forceinline__ void finish(const Params& p, Out& o, float (&v)[COLS], int f, int t0,
                                       int step, int count) {
  float r[COLS];
  const T* res = reinterpret_cast<const T*>(p.res) + f;
#pragma unroll
  for (int j = 0; j < COLS; ++j)
    r[j] = (DACT || p.res) && j < count ? to_f32(res[(t0 + (int64_t)j * step) * p.ldr]) : 0.0f;
  switch (p.act) {
    case kRelu: finish_act<T, DACT, kRelu, COLS>(p, o, v, r, f, t0, step, count); break;
    case kGelu: finish_act<T, DACT, kGelu, COLS>(p, o, v, r, f, t0, step, count); break;
    case kSilu: finish_act<T, DACT, kSilu, COLS>(p, o, v, r, f, t0, step, count); break;
    default: finish_act<T, DACT, kNone, COLS>(p, o, v, r, f, t0, step, count); break;
  }
}

template <int TN, typename T, bool DACT, bool SPLIT>
__global__ void __launch_bounds__(Tile<TN>::kThreads, Tile<TN>::kCtasPerSm)
    k_gemm(const __grid_constant__ CUtensorMap tm_f, const __grid_constant__ CUtensorMap tm_t,
           const Params p) {
  using C = Tile<TN>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * C::kStages + 2 * C::kAccStages + 1];
  __shared__ uint32_t tmem_holder;
  __shared__ uint32_t abort_word;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar0 = smem_addr(bars);
  auto full = [&](uint32_t s) { return bar0 + 8 * s; };
  auto empty = [&](uint32_t s) { return bar0 + 8 * (C::kStages + s); };
  auto acc_full = [&](uint32_t a) { return bar0 + 8 * (2 * C::kStages + a); };
  auto acc_empty = [&](uint32_t a) { return bar0 + 8 * (2 * C::kStages + C::kAccStages + a); };
  const uint32_t drain = bar0 + 8 * (2 * C::kStages + 2 * C::kAccStages);
  volatile uint32_t* abort_flag = &abort_word;

  // This CTA's tiles and k-slices.
  const uint32_t split = SPLIT ? cluster_size() : 1u, rank = SPLIT ? cluster_rank() : 0u;
  const int first = SPLIT ? (int)(blockIdx.x / split) : (int)blockIdx.x;
  const int tiles = p.tiles_f * p.tiles_t;
  const int stride = SPLIT ? tiles : (int)gridDim.x;
  const int s_begin = SPLIT ? (int)((int64_t)p.slices * rank / split) : 0;
  const int s_end = SPLIT ? (int)((int64_t)p.slices * (rank + 1) / split) : p.slices;

  // The one barrier of all warps: behind it barriers and TMEM stand.  Each role
  // comes to it after what it can do alone, so that the first loads are under way
  // while TMEM is being allocated (one token, 5120 x 5120: 7.7 us against 8.4).
  auto start = [&] {
    __syncwarp();
    tc_fence_before();
    asm volatile("barrier.cta.sync.aligned 0, %0;" ::"n"(C::kThreads) : "memory");
    tc_fence_after();
  };
  float alpha = 0.0f, bias = 0.0f;      // of the epilogue's threads; the bias with SPLIT

  if (warp == kWarpTma) {
    uint32_t stage = 0, phase = 0, issued = 0;
    int tile = first, slice = s_begin;
    // Loads until `most` have been issued; false: given up.
    auto produce = [&](uint32_t most) {
      while (tile < tiles && issued < most) {
        // (The first kStages find their stages empty.)
        if (issued >= (uint32_t)C::kStages &&
            !wait(empty(stage), phase ^ 1u, abort_flag, kErrTimeoutProducer))
          return false;
        int tf, tt;
        tile_at(p, tile, tf, tt);
        const uint32_t dst = ring + stage * C::kStageBytes;
        mbar_arrive_expect_tx(full(stage), C::kBytesF + C::kBytesT);
        tma_load_2d(dst, &tm_f, full(stage), slice * 128, tf * kTileF);
        tma_load_2d(dst + C::kBytesF, &tm_t, full(stage), slice * 128, tt * TN);
        ++issued;
        if (++stage == (uint32_t)C::kStages) { stage = 0; phase ^= 1u; }
        if (++slice == s_end) { slice = s_begin; tile += stride; }
      }
      return true;
    };
    if (lane == 0) {
      for (int s = 0; s < C::kStages; ++s) {
        mbar_init(full(s), 1 + 2);
        mbar_init(empty(s), 1);
      }
      for (int a = 0; a < C::kAccStages; ++a) {
        mbar_init(acc_full(a), 1);
        mbar_init(acc_empty(a), kEpiThreads);
      }
      mbar_init(drain, 1);
      abort_word = 0u;
      fence_barrier_init();
      fence_proxy_async_smem();
      produce(C::kStages);
    }
    start();
    if (lane == 0) {
      const bool ok = produce(0xFFFFFFFFu);
      if (!ok) {
        // Given up: the loads in flight land before the CTA ends.  (A stage
        // whose scale loader gave up too never completes: its wait runs to the
        // limit, far longer than a load takes.)
        const uint32_t n = issued < (uint32_t)C::kStages ? issued : (uint32_t)C::kStages;
        volatile uint32_t never = 0u;
        for (uint32_t j = 0; j < n; ++j) {
          if (stage == 0) { stage = C::kStages - 1; phase ^= 1u; } else { --stage; }
          wait(full(stage), phase, &never, kErrTimeoutDrain);
        }
      }
    }
    __syncwarp();
  } else if (warp == kWarpMma) {
    tmem_alloc(smem_addr(&tmem_holder), C::kTmemCols);
    tmem_relinquish();
    start();
    const uint32_t tmem = tmem_holder, tmem_sf = tmem + C::kAccStages * TN;
    // The whole warp walks the loop, so that addresses and descriptors stay
    // uniform; one elected lane issues.
    const bool leader = elect_one();
    uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0, set = 0;
    uint32_t old_stage = 0, old_phase = 0, g = 0;     // of slice g - 2
    bool ok = true;
    for (int i = first; i < tiles && ok; i += stride) {
      if (!wait_warp(acc_empty(acc), acc_phase ^ 1u, abort_flag, kErrTimeoutMma)) break;
      tc_fence_after();
      const uint32_t d = tmem + acc * TN;
      for (int s = s_begin; s < s_end; ++s, ++g) {
        ok = wait_warp(full(stage), phase, abort_flag, kErrTimeoutMma);
        // The scale columns alternate between two sets: the MMAs of slice
        // g - 2 are done with this one when they have freed their stage.
        // (That stage's next phase needs a commit still to come, so the parity
        // cannot have moved on.)
        if (ok && g >= 2) {
          ok = wait_warp(empty(old_stage), old_phase, abort_flag, kErrTimeoutMma);
          if (++old_stage == (uint32_t)C::kStages) { old_stage = 0; old_phase ^= 1u; }
        }
        if (!ok) break;
        tc_fence_after();
        const uint32_t base = ring + stage * C::kStageBytes;
        const uint32_t sf_f = tmem_sf + set * C::kSfCols, sf_t = sf_f + kSteps * 4;
        const uint64_t desc_f = umma_smem_desc(base, 16, 1024, 2);
        const uint64_t desc_t = umma_smem_desc(base + C::kBytesF, 16, 1024, 2);
        const uint64_t desc_s = umma_smem_desc(base + C::kBytesF + C::kBytesT, 128, 128, 0);
        const int steps = min(kSteps, (p.k - s * kSliceK + 63) / 64);
        if (leader) {
          // Addresses within a stage add to the descriptors' address field
          // (16-byte units; the ring ends below its 18 bits).
#pragma unroll
          for (int q = 0; q < kSteps; ++q) {
            cp_scales(sf_f + 4 * q, desc_s + q * (kAtomBytes / 16));
            cp_scales(sf_t + 4 * q, desc_s + (kSteps + q) * (kAtomBytes / 16));
          }
#pragma unroll
          for (int q = 0; q < kSteps; ++q)
            if (q < steps)
              mma_nvfp4(d, desc_f + 2 * q, desc_t + 2 * q, C::kIdesc, sf_f + 4 * q,
                        sf_t + 4 * q, s > s_begin || q > 0);
          tc_commit(empty(stage));
        }
        __syncwarp();
        set ^= 1u;
        if (++stage == (uint32_t)C::kStages) { stage = 0; phase ^= 1u; }
      }
      if (!ok) break;
      if (leader) tc_commit(acc_full(acc));
      __syncwarp();
      if (++acc == (uint32_t)C::kAccStages) { acc = 0; acc_phase ^= 1u; }
    }
    // All issued work completes before TMEM is released.
    if (leader) tc_commit(drain);
    __syncwarp();
    volatile uint32_t never = 0u;
    wait_warp(drain, 0, &never, kErrTimeoutDrain);
  } else if (warp >= kWarpScales) {
    // One warp a part (0: n side, 1: m side).  A lane looks after the rows
    // l, l + 32, l + 64, l + 96: it fetches their 16 bytes of a k-slice
    // asynchronously into a place of its own, as many slices ahead as the ring
    // has stages, and later reads them back in the order of the atoms.  Nobody
    // else touches that place, so its own wait is all the synchronization.
    const int part = warp - kWarpScales;
    const bool f_side = part == 0;
    const uint8_t* sf = f_side ? p.sf_f : p.sf_t;
    const int width = f_side ? p.sf_width_f : p.sf_width_t;
    const int rows = f_side ? p.n : p.m;
    const int tile_rows = f_side ? kTileF : TN;
    const uint32_t place = ring + C::kStages * C::kStageBytes +
                           (uint32_t)(part * C::kStages * 4 * 32 + lane) * 16;
    struct Cursor {
      int tile, slice;
    };
    auto next = [&](Cursor& c) {
      if (++c.slice == s_end) { c.slice = s_begin; c.tile += stride; }
    };
    const uint8_t* row[4];                          // this lane's rows, null behind the end
    int row_tile = -1;
    auto fetch = [&](const Cursor& c, uint32_t slot) {
      if (c.tile < tiles) {
        if (c.tile != row_tile) {
          row_tile = c.tile;
          int tf, tt;
          tile_at(p, c.tile, tf, tt);
          const int row0 = f_side ? tf * kTileF : tt * TN;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = q * 32 + lane;
            row[q] = r < tile_rows && row0 + r < rows ? sf + (int64_t)(row0 + r) * p.sf_pitch
                                                      : nullptr;
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          fetch_scales(place + (slot * 4 + q) * 512, row[q], sf, p.sf_pitch, width, c.slice);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");   // empty behind the last tile
    };
    uint32_t stage = 0, phase = 0;
    Cursor in = {first, s_begin}, out = in;
    for (int j = 0; j < C::kStages; ++j, next(in)) fetch(in, j);
    start();
    bool ok = true;
    while (out.tile < tiles) {
      asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
      uint4 b[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) b[q] = lds128(place + (stage * 4 + q) * 512);
      fetch(in, stage);
      next(in);
      ok = wait_warp(empty(stage), phase ^ 1u, abort_flag, kErrTimeoutProducer);
      if (!ok) break;
      const uint32_t dst = ring + stage * C::kStageBytes + C::kBytesF + C::kBytesT +
                           part * kSteps * kAtomBytes + lane * 16;
      sts128(dst, b[0].x, b[1].x, b[2].x, b[3].x);
      sts128(dst + kAtomBytes, b[0].y, b[1].y, b[2].y, b[3].y);
      sts128(dst + 2 * kAtomBytes, b[0].z, b[1].z, b[2].z, b[3].z);
      sts128(dst + 3 * kAtomBytes, b[0].w, b[1].w, b[2].w, b[3].w);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full(stage));
      next(out);
      if (++stage == (uint32_t)C::kStages) { stage = 0; phase ^= 1u; }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
  } else {
    // ------------------------------- epilogue -------------------------------
    const int group = warp >> 2, quad = warp & 3;
    constexpr int kHalf = TN / 2;
    constexpr int kChunk = kHalf < 16 ? kHalf : 16;   // what the registers hold
    Out o;
    o.top = 0u;
    {
      const float ea = global_encode_scale(*p.amax_f), eb = global_encode_scale(*p.amax_t);
      o.alpha = alpha = __fdiv_rn(1.0f, ea) * __fdiv_rn(1.0f, eb);
    }
    if constexpr (SPLIT) {
      int tf, tt;
      tile_at(p, first, tf, tt);
      const int f = tf * kTileF + quad * 32 + lane;
      if (f < p.n) bias = load_bias(p, f);
    }
    start();
    const uint32_t tmem = tmem_holder;
    uint32_t acc = 0, acc_phase = 0;
    for (int i = first; i < tiles; i += stride) {
      int tf, tt;
      tile_at(p, i, tf, tt);
      const int f = tf * kTileF + quad * 32 + lane;
      if (!wait_warp(acc_full(acc), acc_phase, abort_flag, kErrTimeoutEpilogue)) break;
      tc_fence_after();
      const uint32_t src = tmem + ((uint32_t)(quad * 32) << 16) + acc * TN + group * kHalf;
      if constexpr (SPLIT) {
        // The partial tile to shared memory, column by column (the ring is
        // free: every load has been consumed).
        for (int c = 0; c < kHalf; c += kChunk) {
          float v[kChunk];
          tmem_ld_cols<kChunk>(src + c, v);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < kChunk; ++j)
            sts_f32(ring + (uint32_t)((group * kHalf + c + j) * kTileF + quad * 32 + lane) * 4,
                    v[j]);
        }
      } else {
        o.dbias = 0.0f;
        if (f < p.n) o.bias = load_bias(p, f);
        for (int c = 0; c < kHalf; c += kChunk) {
          const int t0 = tt * TN + group * kHalf + c;
          float v[kChunk];
          tmem_ld_cols<kChunk>(src + c, v);
          tc_wait_ld();
          if (c + kChunk >= kHalf) {
            // The last of this warp's columns are in registers.
            tc_fence_before();
            mbar_arrive(acc_empty(acc));
          }
          if (f < p.n) finish<T, DACT, kChunk>(p, o, v, f, t0, 1, p.m - t0);
        }
        if (DACT && p.dbias_partial && f < p.n)
          p.dbias_partial[(int64_t)(tt * 2 + group) * p.n + f] = o.dbias;
        if (++acc == (uint32_t)C::kAccStages) { acc = 0; acc_phase ^= 1u; }
      }
    }
    if constexpr (!SPLIT) {
      if (p.amax) {
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, o.top);
        if (lane == 0 && top) atomicMax(p.amax, top);
      }
    }
    tc_fence_before();
  }
  if constexpr (SPLIT) {
    // Rank r adds the partial tiles' columns r, r + split, ... over the ranks
    // in order.  A CTA that gave up still comes here (its values are void and
    // the error word says so).
    cluster_sync();
    if (warp < kEpiWarps) {
      int tf, tt;
      tile_at(p, first, tf, tt);
      const int group = warp >> 2, quad = warp & 3;
      const int l = quad * 32 + lane, f = tf * kTileF + l;
      Out o;
      o.top = 0u;
      o.dbias = 0.0f;
      o.alpha = alpha;
      o.bias = bias;
      if (f < p.n) {
        const int c0 = (int)rank + group * (int)split;     // this group's first column
        const int step = 2 * (int)split;
        const int have = min(TN, p.m - tt * TN);
        for (int c = c0; c < have; c += 4 * step) {
          // All loads first: a remote one takes as long as several hundred adds.
          float w[kMaxSplit][4], v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (uint32_t r = 0; r < kMaxSplit; ++r) {
            if (r < split) {
              const uint32_t src = map_rank(ring + (uint32_t)(c * kTileF + l) * 4, r);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                w[r][j] = c + j * step < have
                              ? ld_cluster_f32(src + (uint32_t)(j * step * kTileF) * 4)
                              : 0.0f;
            }
          }
#pragma unroll
          for (uint32_t r = 0; r < kMaxSplit; ++r) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (r < split) v[j] += w[r][j];
          }
          finish<T, DACT, 4>(p, o, v, f, tt * TN + c, step, (have - c + step - 1) / step);
        }
        if (DACT && p.dbias_partial)
          p.dbias_partial[(int64_t)((tt * (int)split + (int)rank) * 2 + group) * p.n + f] = o.dbias;
      }
      if (p.amax) {
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, o.top);
        if (lane == 0 && top) atomicMax(p.amax, top);
      }
    }
    cluster_sync();   // the others have read this CTA's partial tile
  }
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem_holder, C::kTmemCols);
  }
}

// dbias: the partial rows summed in a fixed order, 32 columns a block.
__global__ void __launch_bounds__(256) k_dbias(const float* partial, int rows, int n, float* out) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (c < n)
    for (int r = warp; r < rows; r += 8) v += partial[(int64_t)r * n + c];
  s[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < n) {
#pragma unroll
    for (int w = 1; w < 8; ++w) v += s[w][lane];
    out[c] = v;
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

int encode_map(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, int64_t d0, int64_t d1,
               int64_t pitch, int b0, int b1, CUtensorMapSwizzle swizzle) {
  auto fn = encode_fn();
  if (!fn) return cuda_status(cudaErrorNotSupported);
  const cuuint64_t dims[2] = {(cuuint64_t)d0, (cuuint64_t)d1};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(cuuint32_t)b0, (cuuint32_t)b1};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = fn(map, type, 2, const_cast<void*>(ptr), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? NVFP4_OK : cuda_status(cudaErrorInvalidValue);
}

}  // namespace

int encode_codes_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t k, int box_rows) {
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, ptr, k / 2, rows, k / 2, 128, box_rows,
                    CU_TENSOR_MAP_SWIZZLE_128B);
}
int encode_words_map(CUtensorMap* map, const void* ptr, int64_t rows) {
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, ptr, 256, rows, 1024, 256, 2,
                    CU_TENSOR_MAP_SWIZZLE_NONE);
}

namespace {

// Tile width and split, from the sizes alone (148 SMs), so that a workspace
// can be sized without a device.
struct Plan {
  bool wide;
  int tn, split;
  int64_t tiles_f, tiles_t;
  int64_t partial_rows() const { return tiles_t * (wide ? 3 : 2 * split); }
};
constexpr int kSms = 148;

Plan make_plan(int64_t m, int64_t n, int64_t k) {
  Plan p;
  const int64_t slices = (k + kSliceK - 1) / kSliceK;
  // Few tiles: one launch, k split over clusters.  Many: pairs of CTAs behind the
  // kernel that orders the scales, which a short k does not repay while every SM
  // has one tile.  (m n k = 512 512 512, 32 tiles: 7.0 us against 7.9; 128 6400 512,
  // 100 tiles: 7.0 against 8.2; 128 7000 1280, 110 tiles: 8.8 against 9.0; 400 2560
  // 4096, 140 tiles: 13.5 against 12.1; 200 5120 1280, 160 tiles: 10.2 against 9.0.)
  const int64_t few = slices <= 5 ? kSms : 96;
  p.wide = m > 64 && ((m + 63) / 64) * ((n + 127) / 128) > few;
  if (p.wide) {
    // The narrower tile where it takes no more waves of pairs: it is done
    // sooner, but not twice as soon.  (200 5120 5120: 14.0 us against 15.1; 512
    // 5120 5120, two waves against one: 19.5 against 16.4.)
    p.tiles_f = (n + 255) / 256;
    auto waves = [&](int64_t tn) {
      return (p.tiles_f * ((m + tn - 1) / tn) + kSms / 2 - 1) / (kSms / 2);
    };
    p.tn = waves(128) <= waves(256) ? 128 : 256;
    p.tiles_t = (m + p.tn - 1) / p.tn;
    p.split = 1;
    return p;
  }
  p.tiles_f = (n + kTileF - 1) / kTileF;
  p.tn = m <= 16 ? 16 : m <= 32 ? 32 : 64;
  p.tiles_t = (m + p.tn - 1) / p.tn;
  // Split k while all clusters run at once and every part keeps at least four
  // slices.  A cluster lives within one GPC: 148 SMs are counted as nine of 16,
  // each SM with room for two CTAs.  (5120 x 5120, one token: 11.5 us whole, 8.5
  // in four parts, 8.0 in five or six; in seven, whose clusters take two waves, 11.5.)
  p.split = 1;
  for (int s = 2; s <= kMaxSplit && 4 * s <= slices; ++s)
    if (p.tiles_f * p.tiles_t <= 9 * (32 / s)) p.split = s;
  return p;
}

// Workspace: the bias gradient's partial rows, then the ordered scales.
size_t align256(size_t x) { return (x + 255) / 256 * 256; }
size_t partial_bytes(const Plan& p, int64_t n, bool dbias) {
  return dbias ? align256((size_t)p.partial_rows() * (size_t)n * sizeof(float)) : 0;
}
size_t workspace_bytes(int64_t m, int64_t n, int64_t k, bool dbias) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const Plan p = make_plan(m, n, k);
  return partial_bytes(p, n, dbias) + (p.wide ? wide_scale_bytes(m, n, k) : 0);
}

template <int TN, typename T, bool DACT>
int launch_tile(const Plan& plan, const Params& p, const CUtensorMap& f, const CUtensorMap& t,
                int sms, cudaStream_t st) {
  using C = Tile<TN>;
  const int64_t tiles = plan.tiles_f * plan.tiles_t;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)plan.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  if (plan.split > 1) {
    constexpr auto kernel = k_gemm<TN, T, DACT, true>;
    if (int e = allow_smem<kernel>((int)C::kSmemBytes)) return e;
    cfg.gridDim = dim3((unsigned)(tiles * plan.split));
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, f, t, p));
  }
  constexpr auto kernel = k_gemm<TN, T, DACT, false>;
  if (int e = allow_smem<kernel>((int)C::kSmemBytes)) return e;
  const int64_t slots = (int64_t)sms * C::kCtasPerSm;
  cfg.gridDim = dim3((unsigned)(tiles < slots ? tiles : slots));
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, f, t, p));
}

template <typename T, bool DACT>
int launch_type(const Plan& plan, const Params& p, const CUtensorMap& f, const CUtensorMap& t,
                int sms, cudaStream_t st) {
  switch (plan.tn) {
    case 16: return launch_tile<16, T, DACT>(plan, p, f, t, sms, st);
    case 32: return launch_tile<32, T, DACT>(plan, p, f, t, sms, st);
    default: return launch_tile<64, T, DACT>(plan, p, f, t, sms, st);
  }
}

struct Call {
  int64_t m, n, k;
  const void *a, *sfa, *b, *sfb;
  const float *amax_a, *amax_b;
  void* d;
  int64_t ldd;
  int dtype;
  const void* bias;
  int bias_dtype;
  const void* res;
  int64_t ldr;
  int act;
  void* aux;
  int64_t ldaux;
  bool dact;
  float* dbias;
  float* amax_out;
  void* ws;
  size_t ws_bytes;
  uint32_t sm_count;
  cudaStream_t st;
};

bool known_dtype(int d) { return d >= NVFP4_DTYPE_F32 && d <= NVFP4_DTYPE_F16; }

int run(const Call& c) {
  constexpr int64_t kMaxDim = 1 << 30;
  if (c.m < 0 || c.n < 0 || c.k < 0 || c.m > kMaxDim || c.n > kMaxDim || c.k > kMaxDim ||
      c.k % 32 != 0 || c.ldd < c.n || (c.res && c.ldr < c.n) || (c.aux && c.ldaux < c.n))
    return NVFP4_ERR_INVALID_SHAPE;
  if (!known_dtype(c.dtype) || (c.bias && !known_dtype(c.bias_dtype)) || c.act < kNone ||
      c.act > kSilu)
    return NVFP4_ERR_INVALID_ARGUMENT;
  const uintptr_t es = c.dtype == NVFP4_DTYPE_F32 ? 4 : 2;
  const uintptr_t bs = c.bias_dtype == NVFP4_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)c.a % 16 || (uintptr_t)c.b % 16 || (uintptr_t)c.d % es ||
      (uintptr_t)c.res % es || (uintptr_t)c.aux % es || (c.bias && (uintptr_t)c.bias % bs) ||
      (uintptr_t)c.amax_a % 4 || (uintptr_t)c.amax_b % 4 || (uintptr_t)c.amax_out % 4 ||
      (uintptr_t)c.dbias % 4)
    return NVFP4_ERR_MISALIGNED;
  const bool empty = c.m == 0 || c.n == 0;
  // k = 0 would be an empty sum; no cast writes such an operand.
  if (!empty && c.k == 0) return NVFP4_ERR_INVALID_SHAPE;
  if (!empty) {
    if (!c.a || !c.sfa || !c.b || !c.sfb || !c.amax_a || !c.amax_b || !c.d || (c.dact && !c.res))
      return NVFP4_ERR_INVALID_ARGUMENT;
    auto partly = [&](const void* x, int64_t ldx, const void* y, int64_t ldy) {
      return partly_over(x, ldx, y, ldy, c.m, c.n, (int64_t)es);
    };
    if (partly(c.d, c.ldd, c.res, c.ldr) || partly(c.aux, c.ldaux, c.res, c.ldr) ||
        partly(c.d, c.ldd, c.aux, c.ldaux) || (c.aux && c.aux == c.d))
      return NVFP4_ERR_INVALID_ARGUMENT;
    // amax_out is cleared before the operands' amax are read.
    if (c.amax_out && (c.amax_out == c.amax_a || c.amax_out == c.amax_b))
      return NVFP4_ERR_INVALID_ARGUMENT;
    const Plan plan = make_plan(c.m, c.n, c.k);
    if (plan.tiles_f * plan.tiles_t > (1ll << 28)) return NVFP4_ERR_INVALID_SHAPE;
    const size_t need = workspace_bytes(c.m, c.n, c.k, c.dbias != nullptr);
    if (need && (!c.ws || c.ws_bytes < need)) return NVFP4_ERR_INVALID_ARGUMENT;
    if (need && (uintptr_t)c.ws % 256) return NVFP4_ERR_MISALIGNED;
  }
  if (empty && !c.amax_out && !(c.dbias && c.n)) return NVFP4_OK;
  int sms = 0;
  if (int e = device_sm_count(&sms)) return e;
  if (c.sm_count && (int)c.sm_count < sms) sms = (int)c.sm_count;
  // (The wide kernel's first launch clears the word itself.)
  if (c.amax_out && (empty || !make_plan(c.m, c.n, c.k).wide))
    if (cudaError_t e = cudaMemsetAsync(c.amax_out, 0, sizeof(float), c.st)) return cuda_status(e);
  if (empty) {
    if (c.dbias && c.n)
      if (cudaError_t e = cudaMemsetAsync(c.dbias, 0, sizeof(float) * (size_t)c.n, c.st))
        return cuda_status(e);
    return NVFP4_OK;
  }
  const Plan plan = make_plan(c.m, c.n, c.k);
  Params p = {};
  p.m = (int)c.m;
  p.n = (int)c.n;
  p.k = (int)c.k;
  p.slices = (int)((c.k + kSliceK - 1) / kSliceK);
  p.tiles_f = (int)plan.tiles_f;
  p.tiles_t = (int)plan.tiles_t;
  p.sf_f = reinterpret_cast<const uint8_t*>(c.sfb);
  p.sf_t = reinterpret_cast<const uint8_t*>(c.sfa);
  p.sf_pitch = (int)(c.k / 16);
  p.sf_width_f = scale_width(c.sfb, c.k / 16);
  p.sf_width_t = scale_width(c.sfa, c.k / 16);
  p.amax_f = c.amax_b;
  p.amax_t = c.amax_a;
  p.d = c.d;
  p.ldd = c.ldd;
  p.bias = c.bias;
  p.bias_dtype = c.bias_dtype;
  p.res = c.res;
  p.ldr = c.ldr;
  p.aux = c.aux;
  p.ldaux = c.ldaux;
  p.act = c.act;
  p.dbias_partial = c.dbias ? reinterpret_cast<float*>(c.ws) : nullptr;
  p.amax = reinterpret_cast<uint32_t*>(c.amax_out);
  const int64_t per16 = 16 / (int64_t)es;
  p.vec = ((uintptr_t)c.d % 16 | (uintptr_t)c.res % 16 | (uintptr_t)c.aux % 16 |
           (uintptr_t)(c.ldd % per16) | (uintptr_t)(c.res ? c.ldr % per16 : 0) |
           (uintptr_t)(c.aux ? c.ldaux % per16 : 0)) == 0;
  CUtensorMap map_f, map_t;
  auto typed = [&](auto t) {
    using T = decltype(t);
    return c.dact ? launch_type<T, true>(plan, p, map_f, map_t, sms, c.st)
                  : launch_type<T, false>(plan, p, map_f, map_t, sms, c.st);
  };
  int e;
  if (plan.wide) {
    e = launch_wide(c.dtype, c.dact, plan.tn, p, c.a, c.b,
                    reinterpret_cast<unsigned char*>(c.ws) +
                        partial_bytes(plan, c.n, c.dbias != nullptr),
                    sms, c.st);
  } else {
    if (int r = encode_codes_map(&map_f, c.b, c.n, c.k, kTileF)) return r;
    if (int r = encode_codes_map(&map_t, c.a, c.m, c.k, plan.tn)) return r;
    e = c.dtype == NVFP4_DTYPE_F32    ? typed(float())
        : c.dtype == NVFP4_DTYPE_BF16 ? typed(__nv_bfloat16())
                                      : typed(__half());
  }
  if (e || !c.dbias) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((c.n + 31) / 32));
  cfg.blockDim = dim3(256);
  cfg.stream = c.st;
  // Launched while the product is still running; waits for it.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, k_dbias, (const float*)p.dbias_partial,
                                        (int)plan.partial_rows(), p.n, c.dbias));
}

}  // namespace
}  // namespace gemm

int gemm_device_error(uint32_t* code, int clear) {
  uint32_t wide = 0;
  if (int e = gemm::read_error_word(code, clear)) return e;
  if (int e = gemm::wide_device_error(&wide, clear)) return e;
  if (*code == 0) *code = wide;
  return NVFP4_OK;
}

}  // namespace nvfp4

extern "C" {

NVFP4_API int nvfp4_gemm(int64_t m, int64_t n, int64_t k, const void* A, const void* SFA,
                         const float* amax_a, const void* B, const void* SFB, const float* amax_b,
                         void* D, int64_t ldd, int out_dtype, const void* bias, int bias_dtype,
                         const void* residual, int64_t ldr, int activation, void* aux,
                         int64_t ldaux, float* amax_out, void* workspace, size_t workspace_bytes,
                         uint32_t sm_count, nvfp4_stream_t stream) {
  nvfp4::gemm::Call c = {};
  c.m = m; c.n = n; c.k = k;
  c.a = A; c.sfa = SFA; c.amax_a = amax_a;
  c.b = B; c.sfb = SFB; c.amax_b = amax_b;
  c.d = D; c.ldd = ldd; c.dtype = out_dtype;
  c.bias = bias; c.bias_dtype = bias_dtype;
  c.res = residual; c.ldr = ldr;
  c.act = activation;
  c.aux = aux; c.ldaux = ldaux;
  c.amax_out = amax_out;
  c.ws = workspace; c.ws_bytes = workspace_bytes;
  c.sm_count = sm_count;
  c.st = (cudaStream_t)stream;
  return nvfp4::gemm::run(c);
}

NVFP4_API size_t nvfp4_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  return nvfp4::gemm::workspace_bytes(m, n, k, false);
}

NVFP4_API size_t nvfp4_gemm_dact_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  return nvfp4::gemm::workspace_bytes(m, n, k, true);
}

NVFP4_API int nvfp4_gemm_dact(int64_t m, int64_t n, int64_t k, const void* A, const void* SFA,
                              const float* amax_a, const void* B, const void* SFB,
                              const float* amax_b, const void* aux, int64_t ldaux, int activation,
                              void* D, int64_t ldd, int out_dtype, float* dbias, float* amax_out,
                              void* workspace, size_t workspace_bytes, uint32_t sm_count,
                              nvfp4_stream_t stream) {
  nvfp4::gemm::Call c = {};
  c.m = m; c.n = n; c.k = k;
  c.a = A; c.sfa = SFA; c.amax_a = amax_a;
  c.b = B; c.sfb = SFB; c.amax_b = amax_b;
  c.d = D; c.ldd = ldd; c.dtype = out_dtype;
  c.res = aux; c.ldr = ldaux;
  c.act = activation;
  c.dact = true;
  c.dbias = dbias;
  c.amax_out = amax_out;
  c.ws = workspace; c.ws_bytes = workspace_bytes;
  c.sm_count = sm_count;
  c.st = (cudaStream_t)stream;
  return nvfp4::gemm::run(c);
}

}  // extern "C"
