// The product of two NVFP4 matrices for large m: tiles of 256 (n) x TN (m) by
// pairs of CTAs (tcgen05 cta_group::2).
//
// A pair's tensor cores work on one tile: each CTA holds 128 rows of the n side
// and half of the m side's rows, and each half serves both.  That is what the
// kernel is bound by: one CTA alone must read 12 KB of operands from shared
// memory for an M128 N256 K64 product and write as much for the next ones,
// more than the 128 bytes a cycle of that memory; in a pair it is 8 KB.
//
// The scales arrive by TMA like the codes.  The casts' row-major order would
// have to be gathered 16 bytes a row, which costs a cycle of the shared-memory
// port for each row; so a first kernel (k_order_scales, a few microseconds for
// 1/9 of the operands' bytes) writes them as the 512-byte atoms that tcgen05.cp
// spreads over the TMEM lanes, one contiguous 2 KB of four atoms for each 128
// rows and k-slice.
//
// TMEM: two accumulators and two sets of scale columns.  At TN = 256 that is
// more than 512 columns, so the accumulators overlap by kOverlap columns: the
// epilogue of a tile takes the shared columns first, and the next tile's
// products start when these (not the whole accumulator) have been read.
//
// Warps: 0-11 epilogue, 12 TMA producer, 13 MMA issuer (of the pair's first
// CTA).  Epilogue: a warp's 32 lanes (features) x 32 columns (tokens) are turned
// around through 2 KB of shared memory, after which a thread holds eight
// consecutive features of a token: bias, activation, residual and the stores
// work on 16-byte vectors.
//
// Measured: 8192 x 14336 x 5120 230-237 us without an epilogue (5.1-5.2 PFLOP/s; k =
// 20480: 5.7-6.1), 260-286 us with GELU, aux and amax; odd rows, 4099 x 14335 x 5120,
// 150 us.  Those are bursts: in a stream of such calls the board reaches its power
// limit, the clock falls below 1.5 GHz, and the same take 273 and 314-336 us.  A
// 256 x 256 x 256 slice of a pair takes 0.415 us; its products and scale copies
// alone 0.32, its loads alone 0.26.
#include "gemm_nvfp4.cuh"

namespace nvfp4 {
namespace gemm {
namespace {

// Twelve epilogue warps: three column groups of four warps (TMEM lane quarters),
// as many as 128 registers a thread allow.
constexpr int kPairEpiWarps = 12, kGroups = kPairEpiWarps / 4;
constexpr int kWarpTma = kPairEpiWarps, kWarpMma = kPairEpiWarps + 1;
constexpr int kThreads = 32 * (kPairEpiWarps + 2);
constexpr int kTurnRows = 16;                                // tokens turned around at once
constexpr uint32_t kTurnWarp = kTurnRows * 128;

template <int TN>
struct Wide {
  static constexpr int kAtomsT = TN / 128;
  static constexpr uint32_t kBytesF = kTileF * 128;
  static constexpr uint32_t kBytesT = TN / 2 * 128;          // this CTA's half
  static constexpr uint32_t kBytesSf = kSteps * (1 + kAtomsT) * kAtomBytes;
  static constexpr uint32_t kStageBytes = kBytesF + kBytesT + kBytesSf;
  static constexpr uint32_t kTurnBytes = kPairEpiWarps * kTurnWarp;
  static constexpr int kStagesRaw = (int)((kSmemMax - 2048 - kTurnBytes) / kStageBytes);
  static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + kTurnBytes + 1024;
  static constexpr uint32_t kSfCols = kSteps * 4 * (1 + kAtomsT);
  static constexpr int kFree = 512 - 2 * (int)kSfCols;       // columns for accumulators
  static constexpr int kOverlap = 2 * TN > kFree ? 2 * TN - kFree : 0;
  static constexpr int kAcc1 = TN - kOverlap;                // second accumulator's first column
  static constexpr int kChunks = TN / 32;
  static constexpr int kTurns = (kChunks + kGroups - 1) / kGroups;   // per column group
  // Turns whose columns the next tile's products overwrite.
  static constexpr int kEarly = (kOverlap + 32 * kGroups - 1) / (32 * kGroups);
  static constexpr uint32_t kIdesc =
      (1u << 7) | (1u << 10) | ((uint32_t)(TN / 8) << 17) | ((uint32_t)(256 / 16) << 24);
  static_assert(kStages >= 3, "the scale columns of slice g - 2 are checked through its stage");
  static_assert(kEarly <= 1, "columns held in registers");
};

// TMA load by a CTA of a pair into its own shared memory, completing on the
// first CTA's barrier.  No multicast: each CTA fetches its own rows.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const void* tmap, uint32_t bar,
                                              int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes."
      "cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a_desc, uint64_t b_desc,
                                         uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X "
      "[%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void cp_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}
// Arrive on the barrier at this address in both CTAs when all tcgen05 work
// issued so far has completed.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}
// Tells the pair's issuer that TMEM reads are done (they are: tcgen05.wait::ld).  What
// orders them before the next products are the two tcgen05 fences, before_thread_sync
// ahead of this arrive and after_thread_sync behind the issuer's wait; between the
// two the PTX manual asks for no more than relaxed operations at cluster scope, and
// that the wait is too (RELAXED).  No other memory is handed over.  A release would
// wait for this thread's stores: 348 us against 336 for 8192 x 14336 x 5120 with GELU
// and aux, 201 against 194 for the backward product of 4099 x 14336 x 5120.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// Eight consecutive elements of T as loaded from memory.
template <typename T>
struct Raw8 {
  static constexpr int kVecs = sizeof(T) / 2;
  uint4 q[kVecs];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) q[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[kVecs - 1].x, q[kVecs - 1].y,
                           q[kVecs - 1].z, q[kVecs - 1].w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) unpack2<T>(w[i], x[2 * i], x[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
      q[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                        __float_as_uint(x[3]));
      q[kVecs - 1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]),
                                __float_as_uint(x[6]), __float_as_uint(x[7]));
    } else {
      q[0] = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                        pack2<T>(x[6], x[7]));
    }
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) reinterpret_cast<uint4*>(p)[i] = q[i];
  }
  // Maximum of the magnitudes, NaN if one is: of fp32 words as an unsigned
  // maximum of their bits (above every finite value comes infinity, above that
  // NaN), of 16-bit halves with signs that mean nothing.
  __device__ __forceinline__ uint32_t top(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      if constexpr (sizeof(T) == 4) {
        m = max(max(m, q[i].x & 0x7FFFFFFFu), q[i].y & 0x7FFFFFFFu);
        m = max(max(m, q[i].z & 0x7FFFFFFFu), q[i].w & 0x7FFFFFFFu);
      } else {
        m = max_abs2<T>(max_abs2<T>(m, q[i].x), q[i].y);
        m = max_abs2<T>(max_abs2<T>(m, q[i].z), q[i].w);
      }
    }
    return m;
  }
};
// Such a maximum as fp32 bits.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m;
  float lo, hi;
  unpack2<T>(m & 0x7FFF7FFFu, lo, hi);
  return max(__float_as_uint(lo), __float_as_uint(hi));
}

// What a thread keeps over a tile: eight features from f on.
struct Acc {
  float alpha;
  float bias[8], dbias[8];
  uint32_t top, some;   // maximum over whole vectors (packed) and the others (fp32 bits)
  int f;
};

// One token's eight features, all of them in D and in whole vectors: x holds
// the accumulators.
template <typename T, bool DACT, int ACT>
__device__ __forceinline__ void finish8(const Params& p, Acc& o, float (&x)[8], const Raw8<T>& r,
                                        int64_t t) {
  float e[8];
  Raw8<T> w;
  if (DACT || p.res) r.get(e);
  if constexpr (DACT) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = x[j] * o.alpha * slope<ACT>(e[j]);
      o.dbias[j] += x[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] * o.alpha + o.bias[j];
    if (p.aux) {
      w.set(x);
      w.store(reinterpret_cast<T*>(p.aux) + t * p.ldaux + o.f);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = activate<ACT>(x[j]);
    if (p.res) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] += e[j];
    }
  }
  w.set(x);
  if (p.amax) o.top = w.top(o.top);
  w.store(reinterpret_cast<T*>(p.d) + t * p.ldd + o.f);
}

// The same element by element, for the features that exist: ragged borders.  A
// function of its own, since the instruction cache holds little more than the
// loop that calls it.  In: accumulators in x, the scaled
// bias beside them; out: what D holds (0 outside), for the bias gradient.
template <typename T, bool DACT>
__device__ __noinline__ uint32_t finish_some(const Params& p, float alpha, const float* bias,
                                             float* x, int f, int64_t t) {
  uint32_t top = 0;
#pragma unroll 1
  for (int j = 0; j < 8; ++j) {
    if (f + j >= p.n) {
      x[j] = 0.0f;
      continue;
    }
    const float e = DACT || p.res
                        ? to_f32(reinterpret_cast<const T*>(p.res)[t * p.ldr + f + j])
                        : 0.0f;
    float z = x[j] * alpha;
    if constexpr (DACT) {
      z *= p.act == kRelu   ? slope<kRelu>(e)
           : p.act == kGelu ? slope<kGelu>(e)
           : p.act == kSilu ? slope<kSilu>(e)
                            : 1.0f;
    } else {
      z += bias[j];
      if (p.aux) reinterpret_cast<T*>(p.aux)[t * p.ldaux + f + j] = from_f32<T>(z);
      z = (p.act == kRelu   ? activate<kRelu>(z)
           : p.act == kGelu ? activate<kGelu>(z)
           : p.act == kSilu ? activate<kSilu>(z)
                            : z) + e;
    }
    const T s = from_f32<T>(z);
    reinterpret_cast<T*>(p.d)[t * p.ldd + f + j] = s;
    x[j] = z;
    top = max(top, __float_as_uint(to_f32(s)) & 0x7FFFFFFFu);
  }
  return top;
}

// A warp's chunk: lane l holds feature l's accumulators of the tokens t0 ..
// t0 + 31 in v.  `turn` is the warp's 2 KB: row = token, 16-byte units of a
// row swapped by the token's parity so that neither side meets a bank twice.
template <typename T, bool DACT, int ACT>
__device__ __forceinline__ void finish_chunk(const Params& p, Acc& o, const float (&v)[32],
                                             float* turn, int lane, int t0) {
  constexpr int kRows = kTurnRows / 8;         // tokens of a thread at a time
  const T* res = reinterpret_cast<const T*>(p.res);
  const bool whole = o.f + 8 <= p.n;
#pragma unroll
  for (int h = 0; h < 32; h += kTurnRows) {
    Raw8<T> r[kRows];
    const int row0 = lane >> 2;
    if (DACT || p.res) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t t = t0 + h + row0 + 8 * i;
        if (t < p.m && whole) r[i].load(res + t * p.ldr + o.f);
      }
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kTurnRows; ++j)
      turn[j * 32 + ((((lane >> 2) ^ (j & 1)) << 2) | (lane & 3))] = v[h + j];
    __syncwarp();
    float x[kRows][8];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = row0 + 8 * i, u = (lane & 3) * 2;
      const float4 a = *reinterpret_cast<const float4*>(turn + row * 32 + ((u ^ (row & 1)) << 2));
      const float4 b =
          *reinterpret_cast<const float4*>(turn + row * 32 + (((u + 1) ^ (row & 1)) << 2));
      x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w;
      x[i][4] = b.x; x[i][5] = b.y; x[i][6] = b.z; x[i][7] = b.w;
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t t = t0 + h + row0 + 8 * i;
        if (t < p.m && o.f < p.n) {
          float y[8], b[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            y[j] = x[i][j];
            b[j] = o.bias[j];
          }
          o.some = max(o.some, finish_some<T, DACT>(p, o.alpha, b, y, o.f, t));
#pragma unroll
          for (int j = 0; j < 8; ++j) o.dbias[j] += y[j];
        }
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (t0 + h + row0 + 8 * i < p.m)
        finish8<T, DACT, ACT>(p, o, x[i], r[i], t0 + h + row0 + 8 * i);
  }
}

// Rows that take no vectors (an odd stride or address): a lane keeps its feature
// f, and a warp's access of one token covers 32 neighbours.  The chunk's tokens
// are t0 .. t0 + 31.
template <typename T, bool DACT, int ACT>
__device__ __forceinline__ void finish_lanes(const Params& p, Acc& o, const float (&v)[32], int f,
                                             int t0, float bias, float& sum) {
  const int count = f < p.n ? p.m - t0 : 0;
  const T* res = reinterpret_cast<const T*>(p.res) + (int64_t)t0 * p.ldr + f;
  T* d = reinterpret_cast<T*>(p.d) + (int64_t)t0 * p.ldd + f;
  T* aux = reinterpret_cast<T*>(p.aux) + (int64_t)t0 * p.ldaux + f;
#pragma unroll
  for (int h = 0; h < 32; h += 8) {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = (DACT || p.res) && h + j < count ? to_f32(*res) : 0.0f;
      res += p.ldr;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (h + j < count) {
        float z = v[h + j] * o.alpha;
        if constexpr (DACT) {
          z *= slope<ACT>(e[j]);
          sum += z;
        } else {
          z += bias;
          if (p.aux) *aux = from_f32<T>(z);
          z = activate<ACT>(z) + e[j];
        }
        const T s = from_f32<T>(z);
        *d = s;
        o.some = max(o.some, __float_as_uint(to_f32(s)) & 0x7FFFFFFFu);
      }
      d += p.ldd;
      aux += p.ldaux;
    }
  }
}

// VEC: rows of D, residual / argument and aux take 16-byte vectors.  (Kernels of
// their own: with both epilogues in one the vector form lost a fifth.)
template <int TN, typename T, bool DACT, bool VEC, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_gemm_pair(const __grid_constant__ CUtensorMap tm_f, const __grid_constant__ CUtensorMap tm_t,
                const __grid_constant__ CUtensorMap tm_sf, const __grid_constant__ CUtensorMap tm_st,
                const Params p) {
  using C = Wide<TN>;
  // k_dbias may be scheduled; it waits for this kernel to complete.  (Only when it
  // follows: a caller's own programmatic dependent must not start this early.)
  if (DACT && p.dbias_partial) asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * C::kStages + 5];
  __shared__ uint32_t tmem_holder;
  __shared__ uint32_t abort_word;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar0 = smem_addr(bars);
  auto full = [&](uint32_t s) { return bar0 + 8 * s; };
  auto empty = [&](uint32_t s) { return bar0 + 8 * (C::kStages + s); };
  auto acc_full = [&](uint32_t a) { return bar0 + 8 * (2 * C::kStages + a); };
  auto acc_free = [&](uint32_t a) { return bar0 + 8 * (2 * C::kStages + 2 + a); };
  const uint32_t drain = bar0 + 8 * (2 * C::kStages + 4);
  volatile uint32_t* abort_flag = &abort_word;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full(a), 1);
      mbar_init(acc_free(a), 2 * kPairEpiWarps);   // both CTAs' epilogue warps
    }
    mbar_init(drain, 1);
    abort_word = 0u;
    fence_barrier_init();
  }
  if (warp == kWarpTma && lane == 0) {
    prefetch_tmap(&tm_f);
    prefetch_tmap(&tm_t);
    prefetch_tmap(&tm_sf);
    prefetch_tmap(&tm_st);
  }
  if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&tmem_holder)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();     // the other CTA's barriers and TMEM stand too
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  const uint32_t tmem_sf = tmem + (uint32_t)C::kFree;
  auto acc_col = [&](uint32_t a) { return a ? (uint32_t)C::kAcc1 : 0u; };

  const int tiles = p.tiles_f * p.tiles_t;
  const int first = (int)(blockIdx.x >> 1), stride = (int)(gridDim.x >> 1);

  if (warp == kWarpTma) {
    const bool leader = elect_one();
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    const uint32_t first_full = map_rank(full(0), 0);     // the first CTA's barriers
    grid_dependency_wait();     // the scales in their order, the amax cleared
    for (int i = first; i < tiles && ok; i += stride) {
      int tf, tt;
      tile_at(p, i, tf, tt);
      const int yf = tf * 256 + (int)rank * 128, yt = tt * TN + (int)rank * (TN / 2);
      // 2 KB (two 1 KB rows of the words map) for each 128 rows and k-slice.
      const int bf = (tf * 2 + (int)rank) * p.slices * 2, bt = tt * C::kAtomsT * p.slices * 2;
      for (int s = 0; s < p.slices; ++s) {
        ok = wait_warp(empty(stage), phase ^ 1u, abort_flag, kErrTimeoutProducer);
        if (!ok) break;
        if (leader) {
          const uint32_t dst = ring + stage * C::kStageBytes;
          const uint32_t sf = dst + C::kBytesF + C::kBytesT;
          const uint32_t bar = first_full + 8 * stage;
          if (rank == 0) mbar_arrive_expect_tx(full(stage), 2 * C::kStageBytes);
          tma_load_pair(dst, &tm_f, bar, s * 128, yf);
          tma_load_pair(dst + C::kBytesF, &tm_t, bar, s * 128, yt);
          tma_load_pair(sf, &tm_sf, bar, 0, bf + 2 * s);
#pragma unroll
          for (int b = 0; b < C::kAtomsT; ++b)
            tma_load_pair(sf + kSteps * (1 + b) * kAtomBytes, &tm_st, bar, 0,
                          bt + 2 * (b * p.slices + s));
        }
        __syncwarp();
        if (++stage == (uint32_t)C::kStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok) {
      // Given up.  This CTA's loads complete on the first CTA's barrier; what
      // is in flight has landed long before 10 ms are over.
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 10000000ull) __nanosleep(1000);
    }
  } else if (warp == kWarpMma) {
    if (rank == 0) {
      const bool leader = elect_one();
      uint32_t stage = 0, phase = 0, set = 0, n = 0;       // n: tiles begun
      uint32_t old_stage = 0, old_phase = 0, g = 0;        // of slice g - 2
      bool ok = true;
      for (int i = first; i < tiles && ok; i += stride, ++n) {
        // Columns to be overwritten: with an overlap the previous tile's
        // shared ones (its warps have then drained the tile before, too),
        // otherwise those of the tile before the previous.
        if (C::kOverlap > 0) {
          if (n >= 1) ok = wait_warp<true>(acc_free((n - 1) & 1u), ((n - 1) >> 1) & 1u,
                                           abort_flag, kErrTimeoutMma);
        } else {
          if (n >= 2) ok = wait_warp<true>(acc_free(n & 1u), ((n - 2) >> 1) & 1u, abort_flag,
                                           kErrTimeoutMma);
        }
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + acc_col(n & 1u);
        for (int s = 0; s < p.slices; ++s, ++g) {
          ok = wait_warp(full(stage), phase, abort_flag, kErrTimeoutMma);
          // Scale columns alternate between two sets: slice g - 2's products
          // are done with this one when they have freed their stage.
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
#pragma unroll
            for (int q = 0; q < kSteps; ++q) {
              cp_scales_pair(sf_f + 4 * q, desc_s + q * (kAtomBytes / 16));
#pragma unroll
              for (int b = 0; b < C::kAtomsT; ++b)
                cp_scales_pair(sf_t + 4 * (q * C::kAtomsT + b),
                               desc_s + (kSteps * (1 + b) + q) * (kAtomBytes / 16));
            }
#pragma unroll
            for (int q = 0; q < kSteps; ++q)
              if (q < steps)
                mma_pair(d, desc_f + 2 * q, desc_t + 2 * q, C::kIdesc, sf_f + 4 * q,
                         sf_t + 4 * q * C::kAtomsT, s > 0 || q > 0);
            commit_pair(empty(stage));
          }
          __syncwarp();
          set ^= 1u;
          if (++stage == (uint32_t)C::kStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if (leader) commit_pair(acc_full(n & 1u));
        __syncwarp();
      }
      // All issued work completes before TMEM is released.
      if (leader)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                drain)
            : "memory");
      __syncwarp();
      volatile uint32_t never = 0u;
      wait_warp(drain, 0, &never, kErrTimeoutDrain);
    }
  } else {
    const int group = warp >> 2, quad = warp & 3;
    float* turn = reinterpret_cast<float*>(smem_raw + (ring - smem_addr(smem_raw)) +
                                           C::kStages * C::kStageBytes + warp * kTurnWarp);
    Acc o;
    o.top = o.some = 0u;
    {
      const float ea = global_encode_scale(*p.amax_f), eb = global_encode_scale(*p.amax_t);
      o.alpha = __fdiv_rn(1.0f, ea) * __fdiv_rn(1.0f, eb);
    }
    uint32_t n = 0;
    for (int i = first; i < tiles; i += stride, ++n) {
      int tf, tt;
      tile_at(p, i, tf, tt);
      o.f = tf * 256 + (int)rank * 128 + quad * 32 + (lane & 3) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        o.bias[j] = VEC && !DACT && o.f + j < p.n ? load_bias(p, o.f + j) : 0.0f;
        o.dbias[j] = 0.0f;
      }
      // Without vectors a lane keeps one feature instead.
      const int lane_f = tf * 256 + (int)rank * 128 + quad * 32 + lane;
      const float lane_bias = !DACT && !VEC && lane_f < p.n ? load_bias(p, lane_f) : 0.0f;
      float lane_sum = 0.0f;
      const uint32_t a = n & 1u;
      if (!wait_warp(acc_full(a), (n >> 1) & 1u, abort_flag, kErrTimeoutEpilogue)) break;
      tc_fence_after();
      const uint32_t src = tmem + ((uint32_t)(quad * 32) << 16) + acc_col(a);
      // Chunk of this group's turn u: the first accumulator shares its last
      // columns with the second, the second its first ones.
      auto chunk = [&](int u) {
        const int c = kGroups * u + group;
        return a ? c : C::kChunks - 1 - c;
      };
      // The accumulator's columns are free for the next products once the last
      // turn (or, with an overlap, the last shared one) is in registers.
      constexpr int kLast = C::kEarly > 0 ? C::kEarly - 1 : C::kTurns - 1;
#pragma unroll 1
      for (int u = 0; u < C::kTurns; ++u) {
        const bool have = kGroups * u + group < C::kChunks;
        float v[32];
        if (have) {
          tmem_ld_32cols(src + 32 * chunk(u), v);
          tc_wait_ld();
        }
        if (u == kLast) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(map_rank(acc_free(a), 0));
        }
        if (!have) break;
        const int t0 = tt * TN + 32 * chunk(u);
        if constexpr (VEC)
          finish_chunk<T, DACT, ACT>(p, o, v, turn, lane, t0);
        else
          finish_lanes<T, DACT, ACT>(p, o, v, lane_f, t0, lane_bias, lane_sum);
      }
      if (!VEC && DACT && p.dbias_partial) {
        if (lane_f < p.n) p.dbias_partial[(int64_t)(tt * kGroups + group) * p.n + lane_f] = lane_sum;
      } else if (DACT && p.dbias_partial) {
        // A feature's tokens are spread over the eight lanes l, l + 4, ...
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int k = 4; k < 32; k <<= 1)
            o.dbias[j] += __shfl_xor_sync(0xFFFFFFFFu, o.dbias[j], k);
          if (lane < 4 && o.f + j < p.n)
            p.dbias_partial[(int64_t)(tt * kGroups + group) * p.n + o.f + j] = o.dbias[j];
        }
      }
    }
    if (p.amax) {
      const uint32_t top =
          __reduce_max_sync(0xFFFFFFFFu, max(top_bits<T>(o.top), o.some));
      if (lane == 0 && top) atomicMax(p.amax, top);
    }
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync();     // nobody leaves while the other still signals or reads here
  if (warp == kWarpMma) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u)
                 : "memory");
  }
}

// ---------------------------------------------------------------------------
// Scales into copy order: for each 128 rows and k-slice four atoms; atom q
// holds, 16 bytes for each l < 32, step q's four scales of the rows l, l + 32,
// l + 64, l + 96.  A block takes 128 rows x 8 slices: 128-byte row pieces in,
// 16 KB in a run out.
// ---------------------------------------------------------------------------
struct OrderArgs {
  const uint8_t* sf[2];
  uint32_t* out[2];
  int rows[2], width[2];
  int blocks0;          // row blocks of operand 0
  int pitch, slices;
  uint32_t* amax;       // cleared for the product's epilogue, may be null
};

__global__ void __launch_bounds__(256) k_order_scales(const OrderArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  if (a.amax && blockIdx.x == 0 && threadIdx.x == 0) *a.amax = 0u;
  __shared__ uint32_t tile[128][33];                     // 8 slices x 4 words, padded
  const int groups = (a.slices + 7) / 8;
  const int at = (int)blockIdx.x / groups, which = at >= a.blocks0;
  const int block = at - (which ? a.blocks0 : 0);
  const int s0 = ((int)blockIdx.x - at * groups) * 8;
  const int rows = which ? a.rows[1] : a.rows[0], width = which ? a.width[1] : a.width[0];
  const uint8_t* sf = which ? a.sf[1] : a.sf[0];
  uint32_t* out = which ? a.out[1] : a.out[0];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int idx = (int)threadIdx.x + 256 * i, r = idx >> 3, s = idx & 7;
    const int row = block * 128 + r;
    const bool in = row < rows && s0 + s < a.slices;
    const uint4 v = load_scales(in ? sf + (int64_t)row * a.pitch : nullptr, a.pitch, width, s0 + s);
    tile[r][4 * s] = v.x;
    tile[r][4 * s + 1] = v.y;
    tile[r][4 * s + 2] = v.z;
    tile[r][4 * s + 3] = v.w;
  }
  __syncthreads();
  const int have = min(8, a.slices - s0);
  uint4* dst = reinterpret_cast<uint4*>(out) + ((int64_t)block * a.slices + s0) * 128;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int idx = (int)threadIdx.x + 256 * i, s = idx >> 7, q = (idx >> 5) & 3, l = idx & 31;
    if (s < have)
      dst[idx] = make_uint4(tile[l][4 * s + q], tile[l + 32][4 * s + q], tile[l + 64][4 * s + q],
                            tile[l + 96][4 * s + q]);
  }
}

template <int TN, typename T, bool DACT, bool VEC, int ACT>
int launch_act(const Params& p, const CUtensorMap (&maps)[4], int sms, cudaStream_t st) {
  using C = Wide<TN>;
  constexpr auto kernel = k_gemm_pair<TN, T, DACT, VEC, ACT>;
  if (int e = allow_smem<kernel>((int)C::kSmemBytes)) return e;
  const int64_t tiles = (int64_t)p.tiles_f * p.tiles_t;
  const int64_t pairs = sms / 2 > 0 ? sms / 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (tiles < pairs ? tiles : pairs)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  // Starts while the scales are being ordered; the producer waits for them.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], maps[3], p))
    return cuda_status(e);
  return cuda_status(cudaGetLastError());
}

template <int TN, typename T, bool DACT, bool VEC>
int launch(const Params& p, const CUtensorMap (&maps)[4], int sms, cudaStream_t st) {
  switch (p.act) {
    case kRelu: return launch_act<TN, T, DACT, VEC, kRelu>(p, maps, sms, st);
    case kGelu: return launch_act<TN, T, DACT, VEC, kGelu>(p, maps, sms, st);
    case kSilu: return launch_act<TN, T, DACT, VEC, kSilu>(p, maps, sms, st);
    default: return launch_act<TN, T, DACT, VEC, kNone>(p, maps, sms, st);
  }
}
template <typename T, bool DACT>
int launch_tile(int tn, const Params& p, const CUtensorMap (&maps)[4], int sms, cudaStream_t st) {
  if (tn == 128)
    return p.vec ? launch<128, T, DACT, true>(p, maps, sms, st)
                 : launch<128, T, DACT, false>(p, maps, sms, st);
  return p.vec ? launch<256, T, DACT, true>(p, maps, sms, st)
               : launch<256, T, DACT, false>(p, maps, sms, st);
}
template <typename T>
int launch_type(bool dact, int tn, const Params& p, const CUtensorMap (&maps)[4], int sms,
                cudaStream_t st) {
  return dact ? launch_tile<T, true>(tn, p, maps, sms, st)
              : launch_tile<T, false>(tn, p, maps, sms, st);
}

int64_t row_blocks(int64_t rows) { return (rows + 127) / 128; }

}  // namespace

size_t wide_scale_bytes(int64_t m, int64_t n, int64_t k) {
  const int64_t slices = (k + kSliceK - 1) / kSliceK;
  return (size_t)((row_blocks(m) + row_blocks(n)) * slices) * kSteps * kAtomBytes;
}

int wide_device_error(uint32_t* code, int clear) { return read_error_word(code, clear); }

int launch_wide(int dtype, bool dact, int tn, const Params& p, const void* a, const void* b,
                void* scale_ws, int sms, cudaStream_t st) {
  const int64_t rows_f = row_blocks(p.n) * p.slices, rows_t = row_blocks(p.m) * p.slices;
  unsigned char* ws_f = reinterpret_cast<unsigned char*>(scale_ws);
  unsigned char* ws_t = ws_f + rows_f * kSteps * kAtomBytes;
  CUtensorMap maps[4];
  if (int e = encode_codes_map(&maps[0], b, p.n, p.k, kTileF)) return e;
  if (int e = encode_codes_map(&maps[1], a, p.m, p.k, tn / 2)) return e;
  if (int e = encode_words_map(&maps[2], ws_f, 2 * rows_f)) return e;
  if (int e = encode_words_map(&maps[3], ws_t, 2 * rows_t)) return e;
  OrderArgs o = {};
  o.sf[0] = p.sf_f;
  o.sf[1] = p.sf_t;
  o.out[0] = reinterpret_cast<uint32_t*>(ws_f);
  o.out[1] = reinterpret_cast<uint32_t*>(ws_t);
  o.rows[0] = p.n;
  o.rows[1] = p.m;
  o.pitch = p.sf_pitch;
  o.slices = p.slices;
  o.width[0] = p.sf_width_f;
  o.width[1] = p.sf_width_t;
  o.blocks0 = (int)row_blocks(p.n);
  o.amax = p.amax;
  // One-dimensional: more than 65535 blocks of rows are a long m, no error.
  const int64_t blocks = (row_blocks(p.n) + row_blocks(p.m)) * ((p.slices + 7) / 8);
  if (blocks > INT32_MAX) return NVFP4_ERR_INVALID_SHAPE;
  k_order_scales<<<(unsigned)blocks, 256, 0, st>>>(o);
  if (cudaError_t e = cudaGetLastError()) return cuda_status(e);
  if (dtype == NVFP4_DTYPE_F32) return launch_type<float>(dact, tn, p, maps, sms, st);
  if (dtype == NVFP4_DTYPE_BF16) return launch_type<__nv_bfloat16>(dact, tn, p, maps, sms, st);
  return launch_type<__half>(dact, tn, p, maps, sms, st);
}

}  // namespace gemm
}  // namespace nvfp4
