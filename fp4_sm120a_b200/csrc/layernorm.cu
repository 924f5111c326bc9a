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
// reduction and its output, and written once.  Rows arrive through a ring of bulk
// copies (one thread, one mbarrier a stage), so the bytes in flight do not depend
// on how many registers a row's arithmetic leaves free; one barrier a row serves
// the reduction and, because every thread has taken its part of the stage by
// then, frees the stage.  Blocks are persistent: gamma and beta stay in
// registers, and the backward pass adds its rows' weight gradients in
// registers and writes one partial row a block, which k_bwd_reduce sums in a
// fixed order (no atomics: results repeat bit for bit).  Unaligned rows take the
// same arithmetic with vectors that are partly the row's (kPhased) or element by
// element (kOdd); rows wider than the registers hold (16384 columns, unaligned 8192)
// are read again instead (k_fwd_wide; k_bwd_wide_w and k_bwd_wide_dx).
//
// The statistics come from two passes over registers: each warp's mean, then
// its sum of squares about that mean, and of what the first pass's rounding left
// in the mean; combined over warps by
//   mean = mean_0 + sum_w n_w (mean_w - mean_0) / n,  M2 = sum_w M2_w + n_w (mean_w - mean)^2.
// Every sum but the first is of differences (or exact), so the mean is off by its own last
// rounding and by little of the spread, however large a common offset is, and the
// mean of a constant row is its value exactly: x - mean is zero there, which an
// rstd of 1 / sqrt(eps) would otherwise blow up.
//
// Measured on the device, inputs from memory, fp32 weights: forward with the amax bf16
// 16384 x 8192 103 us (5.2 TB/s), 16384 x 5120 74 us; backward with a residual 16384 x
// 5120 121 us (5.5 TB/s), 16384 x 8192 171 us (6.3 TB/s), fp32 16384 x 4096 160 us (6.7
// TB/s).  The forward pass is bound by issue slots (72 % taken) and the latency of a
// row's two reductions at the 32 warps an SM that the registers allow, the backward pass
// by memory.
// Unaligned rows: bf16 8192 x 5121 forward 60 us, backward with a residual 93; fp32
// 10000 x 5001 76 us (5.3 TB/s) and 123 us (6.5 TB/s); fp32 1003 x 4099 backward 20.8 us
// (18.6 with the inputs in L2).  Weights that do not stay in registers: bf16 4096 x
// 16384 forward 91 us (2.9 TB/s), backward 198.  Rows wider than the registers: bf16
// 2048 x 18432 75-82 us and 240.
#include <atomic>
#include <cstdint>
#include <type_traits>
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

constexpr int kMaxStages = 8;
constexpr size_t kRingBytes = 200 * 1024;      // of an SM, over its blocks
constexpr size_t kSmBytes = 228 * 1024;        // of an SM
constexpr size_t kBlockBytes = 2048;           // of a block beside its ring: 1 KB reserved, statics
constexpr size_t kRingMost = 226 * 1024;       // dynamic shared memory a block may ask for
constexpr uint64_t kWaitLimitNs = 1000000000ull;
constexpr int kWideThreads = 256;

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
  return x;
}
// The sum over 16 lanes (a half warp each), for the joint of at most 16 warps.
template <int WARPS>
__device__ __forceinline__ float join_sum(float x) {
#pragma unroll
  for (int o = WARPS > 16 ? 16 : 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
  return x;
}

// Mean and sum of squares about it (times `scale`), of n values whose sums about a
// rounded mean `m` are q (of squares) and `left`; fix = left / n.  Values that are
// not finite leave m as it is and the squares not finite.
__device__ __forceinline__ float2 centred(float m, float q, float left, float fix, float scale) {
  const float m2 = (q - left * fix) * scale;
  return make_float2(fix == fix ? m + fix : m, m2 < 0.0f ? 0.0f : m2);
}
// Two sums over 16 lanes, for the joint of at most 16 warps: the lower half warp
// joins a, the upper one b, of the same warps.  And over 32 lanes.  In all lanes.
__device__ __forceinline__ float2 halves_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  const float other = __shfl_xor_sync(0xFFFFFFFFu, v, 16);
  return threadIdx.x & 16 ? make_float2(other, v) : make_float2(v, other);
}
__device__ __forceinline__ float2 warp_sum2(float a, float b) {
  const bool upper = threadIdx.x & 16;
  const float give = upper ? a : b, keep = upper ? b : a;
  return halves_sum(keep + __shfl_xor_sync(0xFFFFFFFFu, give, 16));
}
__device__ __forceinline__ float finite_or_zero(float x) {
  return fabsf(x) <= 3.402823466e38f ? x : 0.0f;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

__device__ __forceinline__ float sum2(uint64_t p) {
  float a, b;
  split(p, a, b);
  return a + b;
}

// A row over the threads.  kWhole: every row of every array is whole aligned
// 16-byte vectors, and thread t holds the vectors t, t + threads, ...  kPhased: the
// same with the vectors of 16-byte aligned memory, of which a row's first and last
// hold only part; a row starts `shift` elements into its first vector in all
// arrays, and a block takes rows of the same shift only, so that its columns stay
// with their threads.  kOdd: the elements t, t + threads, ...
enum Mode : int { kOdd = 0, kWhole = 1, kPhased = 2 };
template <typename T, int MODE>
struct Layout {
  static constexpr int kVec = MODE != kOdd ? 16 / (int)sizeof(T) : 1;
};

// 16 bytes as fp32.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& q, float* x) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) x[k] = __uint_as_float(w[k]);
    else unpack2<T>(w[k], x[2 * k], x[2 * k + 1]);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* x) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                      __float_as_uint(x[3]));
  else
    return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                      pack2<T>(x[6], x[7]));
}
// Maximum of the magnitudes, NaN if one is: of fp32 words as an unsigned maximum
// of their bits (NaN patterns are above infinity's), of 16-bit halves with signs
// that mean nothing.  And its value as fp32 bits.
template <typename T>
__device__ __forceinline__ uint32_t max_bits(uint32_t m, uint32_t w) {
  if constexpr (sizeof(T) == 4) return max(m, w & 0x7FFFFFFFu);
  else return max_abs2<T>(m, w);
}
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) {
    return m;
  } else {
    float lo, hi;
    unpack2<T>(m & 0x7FFF7FFFu, lo, hi);
    return max(__float_as_uint(lo), __float_as_uint(hi));
  }
}

// A row's bytes in whole 16-byte units, which is what bulk copies move.  The first
// and last unit of an unaligned row hold its neighbours' bytes too: they are read
// and left unused, whatever is being written to them meanwhile.  Loading the row's
// share of them apart, a row ahead, made the first warp late for every barrier (fp32
// backward 10000 x 4097: 151 us against 102).
template <int MODE>
__device__ __forceinline__ uint32_t span_bytes(const void* row, uint32_t row_bytes) {
  if constexpr (MODE == kWhole) return row_bytes;
  return (((uint32_t)(uintptr_t)row & 15u) + row_bytes + 15u) & ~15u;
}
template <int MODE>
__device__ __forceinline__ void span_load(uint32_t slot, const void* row, uint32_t row_bytes,
                                          uint32_t bar) {
  bulk_load(slot, reinterpret_cast<const void*>((uintptr_t)row & ~(uintptr_t)15),
            span_bytes<MODE>(row, row_bytes), bar);
}
// Only the unit before the first row's start and the one behind the last row's end
// reach outside the caller's rows.  Those two rows are edges: their copies leave such
// units out (`lo`, `bytes`: of the row's whole units), and EdgeElement adds the
// elements in them.  They are the rows that a block asks for first, before its loop, which knows
// nothing of them: the block of the last row takes that one before its others (and the
// host sees to it that it is not the first row's block too).  (Looked for row by row
// instead: fp32 backward 10000 x 4097 124 us against 103.  That block's rows all
// backwards: 108; it then reads far from the others all the time.)
template <int MODE>
struct Order {
  int start, base;        // the block's first row, and the others less j * gridDim.x
  bool first, last;       // whether that row is the first, the last of all
  __device__ __forceinline__ Order(int64_t rows, int64_t mine)
      : start((int)blockIdx.x), base((int)blockIdx.x), first(blockIdx.x == 0), last(false) {
    if constexpr (MODE != kWhole) {
      last = start + (mine - 1) * gridDim.x == rows - 1;
      if (last) {
        start = (int)(rows - 1);
        base -= (int)gridDim.x;
      }
    }
  }
  template <typename I>
  __device__ __forceinline__ int64_t row(I j) const {
    if constexpr (MODE == kWhole) return blockIdx.x + (int64_t)j * gridDim.x;
    return j == 0 ? start : base + (int64_t)j * gridDim.x;
  }
};
struct Span {
  uint32_t lo, bytes;
};
__device__ __forceinline__ Span edge_span(const void* row, uint32_t row_bytes, bool first,
                                          bool last) {
  const uint32_t lead = (uint32_t)(uintptr_t)row & 15u, end = lead + row_bytes;
  const uint32_t lo = first && lead ? 16u : 0u, hi = (last ? end : end + 15u) & ~15u;
  return {lo, hi > lo ? hi - lo : 0u};
}
__device__ __forceinline__ void edge_load(uint32_t slot, const void* row, const Span& s,
                                          uint32_t bar) {
  if (s.bytes)
    bulk_load(slot + s.lo,
              reinterpret_cast<const unsigned char*>((uintptr_t)row & ~(uintptr_t)15) + s.lo,
              s.bytes, bar);
}
// The elements that an edge's copy leaves out, one a lane of a warp: asked for before
// the weights, put into the slot (whose other bytes the copy fills) after them, so that
// one latency serves all.
template <typename T>
struct EdgeElement {
  T value;
  int at = -1;              // place in the slot, -1: none
  __device__ __forceinline__ void load(const T* row, int cols, bool first, bool last) {
    constexpr int kUnit = 16 / (int)sizeof(T);
    const int lead = (int)((uintptr_t)row & 15u) / (int)sizeof(T), lane = (int)threadIdx.x & 31;
    const int head = first && lead ? min(kUnit - lead, cols) : 0;
    const int tail = last ? min((lead + cols) % kUnit, cols) : 0;
    const int l = lane & 15, c = lane < 16 ? l : cols - tail + l;
    if (l < (lane < 16 ? head : tail)) {
      value = row[c];
      at = lead + c;
    }
  }
  __device__ __forceinline__ void store(unsigned char* slot) const {
    if (at >= 0) reinterpret_cast<T*>(slot)[at] = value;
  }
};
// A thread's items (vectors or elements) within the row: the first `count`.
template <typename T, int MODE, int ITEMS>
struct Mine {
  static constexpr int kVec = Layout<T, MODE>::kVec;
  int total;        // the row's items
  int count;
  int shift;        // kPhased: elements of the first vector before the row
  int last, hi;     // this thread's item that is the row's last (-1: none), its elements
  __device__ __forceinline__ Mine(int cols, const T* row) : shift(0), last(-1), hi(kVec) {
    const int tid = (int)threadIdx.x, nthr = (int)blockDim.x;
    total = cols / kVec;
    if constexpr (MODE == kPhased) {
      shift = (int)((uintptr_t)row & 15u) / (int)sizeof(T);
      total = (shift + cols + kVec - 1) / kVec;
      hi = shift + cols - (total - 1) * kVec;
    }
    const int n = total - tid;
    count = n > 0 ? (n + nthr - 1) / nthr : 0;
    if (MODE == kPhased && n > 0 && (n - 1) % nthr == 0) last = (n - 1) / nthr;
  }
  __device__ __forceinline__ bool has(int it) const { return it < count; }
  // Column of an item's element k.
  __device__ __forceinline__ int column(int it, int k) const {
    return ((int)threadIdx.x + it * (int)blockDim.x) * kVec + k - shift;
  }
  // A vector that is only partly the row's, and whether its element k is.
  __device__ __forceinline__ bool part(int it) const {
    return MODE == kPhased && ((it == 0 && threadIdx.x == 0 && shift > 0) ||
                               (it == last && hi < kVec));
  }
  __device__ __forceinline__ bool in(int it, int k) const {
    return k >= (it == 0 && threadIdx.x == 0 ? shift : 0) && k < (it == last ? hi : kVec);
  }
};
// This thread's elements of a row that has arrived in `slot`.
template <typename T, int MODE, int ITEMS>
__device__ __forceinline__ void fetch(const Mine<T, MODE, ITEMS>& my, const unsigned char* slot,
                                      const T* row, float* f) {
  constexpr int VEC = Layout<T, MODE>::kVec;
  const int tid = threadIdx.x, nthr = blockDim.x;
  if constexpr (MODE != kOdd) {
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const uint4 q = my.has(it) ? reinterpret_cast<const uint4*>(slot)[tid + it * nthr]
                                 : make_uint4(0, 0, 0, 0);
      unpack16<T>(q, f + it * VEC);
      if (my.part(it)) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          if (!my.in(it, k)) f[it * VEC + k] = 0.0f;
      }
    }
  } else {
    // Loads without branches: what lies behind the row's end reads its first element.
    const T* in = reinterpret_cast<const T*>(slot + ((uint32_t)(uintptr_t)row & 15u));
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const T v = in[my.has(it) ? tid + it * nthr : 0];
      f[it] = my.has(it) ? to_f32(v) : 0.0f;
    }
  }
}
// Stores this thread's elements; with TOP returns the magnitudes' maximum
// joined to `top`.
template <bool TOP, typename T>
__device__ __forceinline__ uint32_t put_one(T* at, float f, uint32_t top) {
  *at = from_f32<T>(f);
  if constexpr (!TOP) return top;
  else if constexpr (sizeof(T) == 4) return max_bits<T>(top, __float_as_uint(f));
  else return max_bits<T>(top, pack2<T>(f, 0.0f));
}
template <bool TOP, typename T, int MODE, int ITEMS>
__device__ __forceinline__ uint32_t put(const Mine<T, MODE, ITEMS>& my, T* row, const float* f,
                                        uint32_t top) {
  constexpr int VEC = Layout<T, MODE>::kVec;
  const int nthr = blockDim.x;
  if constexpr (MODE != kOdd) {
    uint4* out = reinterpret_cast<uint4*>(row - my.shift) + threadIdx.x;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      if (my.part(it)) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          if (my.in(it, k)) top = put_one<TOP>(row + my.column(it, k), f[it * VEC + k], top);
      } else {
        const uint4 q = pack16<T>(f + it * VEC);
        if (my.has(it)) out[it * nthr] = q;
        if (TOP && my.has(it)) {
          top = max_bits<T>(max_bits<T>(top, q.x), q.y);
          top = max_bits<T>(max_bits<T>(top, q.z), q.w);
        }
      }
    }
  } else {
    T* out = row + threadIdx.x;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it)
      if (my.has(it)) top = put_one<TOP>(out + it * nthr, f[it], top);
  }
  return top;
}
// This thread's weights, zero behind the row's end: as 16-byte vectors where
// they are aligned (a launch of few rows waits for them).
template <typename T, typename W, int MODE, int ITEMS>
__device__ __forceinline__ void fetch_weights(const Mine<T, MODE, ITEMS>& my, const W* w, int cols,
                                              float* f) {
  constexpr int VEC = Layout<T, MODE>::kVec;
  const bool vectors = MODE == kWhole && (uintptr_t)w % 16 == 0;
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[it * VEC + k] = 0.0f;
    if (w != nullptr && my.has(it)) {
      if (vectors) {
        constexpr int N = 16 / (int)sizeof(W);       // VEC or half of it
#pragma unroll
        for (int k = 0; k + N <= VEC; k += N)
          unpack16<W>(*reinterpret_cast<const uint4*>(w + my.column(it, k)), f + it * VEC + k);
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          if (!my.part(it) || my.in(it, k)) f[it * VEC + k] = to_f32(w[my.column(it, k)]);
      }
    }
  }
}

// The ring of rows in flight: ARRAYS slots a stage (x, dy, residual).
struct Ring {
  uint32_t base, bar, stage_bytes, slot_bytes;
  int stages;
};

struct Shared {
  uint64_t bar[kMaxStages];
  float2 red[2][32];
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
  uint32_t slot_bytes;
  float eps;
};

// One row per block at a time; two blocks or more share an SM and hide each
// other's reductions.
template <typename T, typename W, int MODE, int ITEMS, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) k_fwd_rows(const FwdArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Shared sh;
  // Of each warp: the elements n it holds of a row, 1 / n (0 for none), n / cols and
  // 1 / cols.  In shared memory, since registers that do not change over the rows
  // are the ones that get spilled, and a spilled one costs more than these reads
  // (16384 x 8192 bf16: 108 us with four words spilled, 104 with none).
  __shared__ float4 counts[16];
  constexpr int VEC = Layout<T, MODE>::kVec, E = ITEMS * VEC;
  const int tid = threadIdx.x, nthr = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t row_bytes = (uint32_t)a.cols * sizeof(T);
  const T* x = reinterpret_cast<const T*>(a.x);
  const Mine<T, MODE, ITEMS> my(a.cols, x + blockIdx.x * a.ldx);
  T* y = reinterpret_cast<T*>(a.y);
  Ring ring;
  ring.slot_bytes = ring.stage_bytes = a.slot_bytes;
  ring.base = smem_addr(smem);
  ring.bar = smem_addr(sh.bar);
  ring.stages = a.stages;
  const int mine = (int)((a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);
  const Order<MODE> order(a.rows, mine);
  auto issue = [&](int j, uint32_t stage) {
    const T* row = x + order.row(j) * a.ldx;
    const uint32_t bar = ring.bar + 8 * stage;
    mbar_arrive_expect_tx(bar, span_bytes<MODE>(row, row_bytes));
    span_load<MODE>(ring.base + stage * ring.stage_bytes, row, row_bytes, bar);
  };
  const bool edge = MODE != kWhole && (order.first || order.last);
  if (tid == 0) {
    for (int s = 0; s < ring.stages; ++s) mbar_init(ring.bar + 8 * s, 1);
    sh.abort_flag = 0u;
    fence_barrier_init();
    if (edge) {
      const T* row = x + order.row(0) * a.ldx;
      const Span span = edge_span(row, row_bytes, order.first, order.last);
      mbar_arrive_expect_tx(ring.bar, span.bytes);
      edge_load(ring.base, row, span, ring.bar);
    }
    for (int j = edge; j < ring.stages && j < mine; ++j) issue(j, (uint32_t)j);
  }
  const bool edge_warp = edge && warp == (nthr >> 5) - 1;
  EdgeElement<T> ex;
  if (edge_warp) ex.load(x + order.row(0) * a.ldx, a.cols, order.first, order.last);
  const W* wg = reinterpret_cast<const W*>(a.gamma);
  const W* wb = reinterpret_cast<const W*>(a.beta);
  // Weights stay in registers while there is room for them.
  constexpr bool kKeep = E <= 16;
  constexpr bool kSumLeft = sizeof(T) == 4;
  float gamma[E], beta[E];
  if constexpr (kKeep) {
    fetch_weights<T, W, MODE, ITEMS>(my, wg, a.cols, gamma);
    fetch_weights<T, W, MODE, ITEMS>(my, wb, a.cols, beta);
  }
  if (edge_warp) {
    ex.store(smem);
    if (mine > ring.stages) fence_proxy_async_smem();   // a later copy writes these bytes
  }
  static_assert(THREADS <= 512, "a half warp joins all warps");
  const int share = lane & 15;        // the warp whose sums this lane joins
  if (warp == 0 && lane < 16) {
    float n = 0.0f;
    if (lane >= nthr >> 5) {
      sh.red[0][lane] = sh.red[1][lane] = make_float2(0.0f, 0.0f);
    } else {
#pragma unroll
      for (int it = 0; it < ITEMS; ++it)
        n += (float)(min(max(my.total - lane * 32 - it * nthr, 0), 32) * VEC);
      if constexpr (MODE == kPhased) {
        if (lane == 0) n -= (float)my.shift;
        if ((my.total - 1) % nthr >> 5 == lane) n -= (float)(VEC - my.hi);
      }
    }
    const float inv_n = 1.0f / (float)a.cols;
    counts[lane] = make_float4(n, n > 0.0f ? 1.0f / n : 0.0f, n * inv_n, inv_n);
  }
  __syncthreads();
  uint32_t top = 0;
  int k = 0;
  RingAt at;
  for (; k < mine; ++k, at.next(ring)) {
    const int64_t row = order.row(k);
    float f[E];
    if (ring_wait(ring, at, &sh.abort_flag)) {
      fetch<T, MODE, ITEMS>(my, smem + at.stage * ring.stage_bytes, x + row * a.ldx, f);
      uint64_t s = pair(0.0f, 0.0f);
#pragma unroll
      for (int e = 0; e < E; e += 2) s = add2(s, pair(f[e], f[e + 1]));
      const float4 own = counts[warp];
      const float sum = warp_sum(sum2(s));
      float mw = sum * own.y;
      // What the rounding of mw leaves.  In 16 bits the difference of the sums: a
      // warp's 1024 values of similar size at most (8 or 11 digits and 10 more) add up
      // without rounding.  In 32 bits sum (f - mw), taken along with the squares.
      // (16384 x 8192 bf16: 104 us, with the second sum 118.)
      if constexpr (!kSumLeft) mw += finite_or_zero(fmaf(-own.x, mw, sum) * own.y);
      const uint64_t minus = pair(-mw, -mw);
      uint64_t r = pair(0.0f, 0.0f);
      s = pair(0.0f, 0.0f);
      if constexpr (MODE != kOdd) {
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
          if (my.part(it)) {
            // What is not the row's counts as the mean.
#pragma unroll
            for (int k = 0; k < VEC; ++k)
              if (!my.in(it, k)) f[it * VEC + k] = mw;
          }
          if (my.has(it)) {
#pragma unroll
            for (int e = it * VEC; e < (it + 1) * VEC; e += 2) {
              const uint64_t d = add2(pair(f[e], f[e + 1]), minus);
              s = fma2(d, d, s);
              if constexpr (kSumLeft) r = add2(r, d);
            }
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          // What lies behind the row's end counts as the mean.
          const float u = my.has(e) ? f[e] : mw, v = my.has(e + 1) ? f[e + 1] : mw;
          const uint64_t d = add2(pair(u, v), minus);
          s = fma2(d, d, s);
          if constexpr (kSumLeft) r = add2(r, d);
        }
      }
      if constexpr (kSumLeft) {
        const float2 t = warp_sum2(sum2(s), sum2(r));
        if (lane == 0) sh.red[k & 1][warp] = centred(mw, t.x, t.y, t.y * own.y, own.w);
      } else {
        const float q = warp_sum(sum2(s)) * own.w;
        if (lane == 0) sh.red[k & 1][warp] = make_float2(mw, q);
      }
    }
    // Everybody has taken its part of the stage and written its sums.  (The
    // sums alternate between two copies: those written next were last read
    // before this barrier.)
    __syncthreads();
    if (*(volatile uint32_t*)&sh.abort_flag) break;
    if (tid == 0 && k + ring.stages < mine) issue(k + ring.stages, at.stage);
    // A lane joins one warp's share; every warp does so by itself.  Both sums are
    // taken about the first warp's mean, so that neither waits for the other: with
    // v = mean - about, M2 = sum (M2_w + n_w (mean_w - about)^2) - n v^2.  The first
    // warp's own deviation is in M2, so the difference loses four digits of 24 at
    // the most.
    const float2 part = sh.red[k & 1][share];       // zeros where there is no such warp
    const float about = finite_or_zero(sh.red[k & 1][0].x);
    const float d = part.x - about, v = d * counts[share].z;
    const float2 joint = halves_sum(lane < 16 ? v : fmaf(v, d, part.y));
    const float mean = about + joint.x;
    const float var = joint.y - joint.x * joint.x;
    const float rstd = rsqrtf((var < 0.0f ? 0.0f : var) + a.eps);
    if (tid == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    if constexpr (!kKeep) {
      fetch_weights<T, W, MODE, ITEMS>(my, wg, a.cols, gamma);
      fetch_weights<T, W, MODE, ITEMS>(my, wb, a.cols, beta);
    }
    // (x - mean) first: a constant row's difference is zero exactly, and stays so
    // whatever rstd is.
    const uint64_t scale = pair(rstd, rstd), minus = pair(-mean, -mean);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const uint64_t h = mul2(add2(pair(f[e], f[e + 1]), minus), scale);
      split(fma2(h, pair(gamma[e], gamma[e + 1]), pair(beta[e], beta[e + 1])), f[e], f[e + 1]);
    }
    if (a.amax)
      top = put<true, T, MODE, ITEMS>(my, y + row * a.ldy, f, top);
    else
      put<false, T, MODE, ITEMS>(my, y + row * a.ldy, f, 0u);
  }
  if (k < mine && tid == 0) ring_drain(ring, at, mine - k);
  if (a.amax) {
    const uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, top_bits<T>(top));
    if (lane == 0 && bits) atomicMax(a.amax, bits);
  }
}

// Sums of f(c, a, b) over a thread's columns, in runs of 32 that are added
// afterwards: the error of a sum of a long row does not grow with its length.
template <typename F>
__device__ __forceinline__ float2 wide_sums(int cols, const F& f) {
  constexpr int kRun = 32, kStep = kRun * kWideThreads;
  float a = 0.0f, b = 0.0f;
  int c = threadIdx.x;
  for (; c < cols - (kStep - kWideThreads); c += kStep) {
    float ra = 0.0f, rb = 0.0f;
#pragma unroll 16
    for (int j = 0; j < kRun; ++j) f(c + j * kWideThreads, ra, rb);
    a += ra;
    b += rb;
  }
  float ra = 0.0f, rb = 0.0f;
#pragma unroll 4
  for (; c < cols; c += kWideThreads) f(c, ra, rb);
  return make_float2(warp_sum(a + ra), warp_sum(b + rb));
}
// Rows wider than the registers hold: three passes over a row, the second and
// third mostly from cache.
template <typename T, typename W>
__global__ void __launch_bounds__(kWideThreads) k_fwd_wide(const FwdArgs a) {
  __shared__ float first[kWideThreads / 32];
  __shared__ float2 second[kWideThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float inv_n = 1.0f / (float)a.cols;
  uint32_t top = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    T* y = reinterpret_cast<T*>(a.y) + row * a.ldy;
    const float2 s = wide_sums(a.cols, [&](int c, float& sum, float&) { sum += to_f32(x[c]); });
    if (lane == 0) first[warp] = s.x;
    __syncthreads();
    float m = 0.0f;
#pragma unroll
    for (int w = 0; w < kWideThreads / 32; ++w) m += first[w];
    m *= inv_n;
    const float2 t = wide_sums(a.cols, [&](int c, float& squares, float& left) {
      const float d = to_f32(x[c]) - m;
      squares += d * d;
      left += d;
    });
    if (lane == 0) second[warp] = t;
    __syncthreads();
    float q = 0.0f, left = 0.0f;
#pragma unroll
    for (int w = 0; w < kWideThreads / 32; ++w) {
      q += second[w].x;
      left += second[w].y;
    }
    const float2 stat = centred(m, q, left, left * inv_n, inv_n);
    const float mean = stat.x, rstd = __fdiv_rn(1.0f, __fsqrt_rn(stat.y + a.eps));
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
  uint32_t slot_bytes;
  int reduce;           // k_bwd_reduce follows
};

template <typename T, typename W, int MODE, int ITEMS, int THREADS, bool RES>
__global__ void __launch_bounds__(THREADS, 1) k_bwd_rows(const BwdArgs a) {
  // k_bwd_reduce may be scheduled; it waits for this kernel to complete.  (Only
  // when it follows: a caller's own programmatic dependent must not start this
  // early.)
  if (a.reduce) asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Shared sh;
  constexpr int VEC = Layout<T, MODE>::kVec, E = ITEMS * VEC;
  constexpr int kArrays = RES ? 3 : 2;
  const int tid = threadIdx.x, nthr = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int nwarps = nthr >> 5;
  const uint32_t row_bytes = (uint32_t)a.cols * sizeof(T);
  const T* x = reinterpret_cast<const T*>(a.x);
  const Mine<T, MODE, ITEMS> my(a.cols, x + blockIdx.x * a.ldx);
  const T* dy = reinterpret_cast<const T*>(a.dy);
  const T* res = reinterpret_cast<const T*>(a.res);
  T* dx = reinterpret_cast<T*>(a.dx);
  Ring ring;
  ring.slot_bytes = a.slot_bytes;
  ring.stage_bytes = kArrays * a.slot_bytes;
  ring.base = smem_addr(smem);
  ring.bar = smem_addr(sh.bar);
  ring.stages = a.stages;
  // 64 bits for whole rows, 32 for the others: what the compiler made the faster loop of
  // (bf16 16384 x 5120 120 us against 124, 16000 x 1001 42.6 against 43.3).
  using Index = std::conditional_t<MODE == kWhole, int64_t, int>;
  const Index mine = (Index)((a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);
  const Order<MODE> order(a.rows, mine);
  auto issue = [&](Index j, uint32_t stage) {
    const uint32_t bar = ring.bar + 8 * stage, dst = ring.base + stage * ring.stage_bytes;
    const int64_t row = order.row(j);
    const T *rx = x + row * a.ldx, *rdy = dy + row * a.lddy;
    const T* rr = RES ? res + row * a.ldr : nullptr;
    mbar_arrive_expect_tx(bar, span_bytes<MODE>(rx, row_bytes) + span_bytes<MODE>(rdy, row_bytes) +
                                   (RES ? span_bytes<MODE>(rr, row_bytes) : 0u));
    span_load<MODE>(dst, rx, row_bytes, bar);
    span_load<MODE>(dst + ring.slot_bytes, rdy, row_bytes, bar);
    if constexpr (RES) span_load<MODE>(dst + 2 * ring.slot_bytes, rr, row_bytes, bar);
  };
  const bool edge = MODE != kWhole && (order.first || order.last);
  if (tid == 0) {
    for (int s = 0; s < ring.stages; ++s) mbar_init(ring.bar + 8 * s, 1);
    sh.abort_flag = 0u;
    fence_barrier_init();
    if (edge) {
      const int64_t row = order.row(0);
      const T *rx = x + row * a.ldx, *rdy = dy + row * a.lddy;
      const T* rr = RES ? res + row * a.ldr : nullptr;
      const Span sx = edge_span(rx, row_bytes, order.first, order.last),
                 sdy = edge_span(rdy, row_bytes, order.first, order.last),
                 sr = RES ? edge_span(rr, row_bytes, order.first, order.last) : Span{0u, 0u};
      mbar_arrive_expect_tx(ring.bar, sx.bytes + sdy.bytes + sr.bytes);
      edge_load(ring.base, rx, sx, ring.bar);
      edge_load(ring.base + ring.slot_bytes, rdy, sdy, ring.bar);
      if constexpr (RES) edge_load(ring.base + 2 * ring.slot_bytes, rr, sr, ring.bar);
    }
    for (Index j = edge; j < ring.stages && j < mine; ++j) issue(j, (uint32_t)j);
  }
  const bool edge_warp = edge && warp == (nthr >> 5) - 1;
  EdgeElement<T> ex, edy, er;
  if (edge_warp) {
    const int64_t row = order.row(0);
    ex.load(x + row * a.ldx, a.cols, order.first, order.last);
    edy.load(dy + row * a.lddy, a.cols, order.first, order.last);
    if constexpr (RES) er.load(res + row * a.ldr, a.cols, order.first, order.last);
  }
  const W* wg = reinterpret_cast<const W*>(a.gamma);
  constexpr bool kKeep = E <= 16;      // gamma stays in registers
  float gamma[E], dg[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dg[e] = db[e] = 0.0f;
  if constexpr (kKeep) fetch_weights<T, W, MODE, ITEMS>(my, wg, a.cols, gamma);
  if (edge_warp) {
    ex.store(smem);
    edy.store(smem + ring.slot_bytes);
    if constexpr (RES) er.store(smem + 2 * ring.slot_bytes);
    if (mine > ring.stages) fence_proxy_async_smem();   // later copies write these bytes
  }
  __syncthreads();
  const float inv_n = 1.0f / (float)a.cols;
  Index k = 0;
  RingAt at;
  // A row's statistics are fetched a row ahead.
  float next_mean = a.mean[order.row(0)];
  float next_rstd = a.rstd[order.row(0)];
  for (; k < mine; ++k, at.next(ring)) {
    const int64_t row = order.row(k);
    const float mean = next_mean, rstd = next_rstd;
    if (k + 1 < mine) {
      const int64_t next = order.row(k + 1);
      next_mean = a.mean[next];
      next_rstd = a.rstd[next];
    }
    float h[E], u[E], fr[RES ? E : 2];
    const bool ok = ring_wait(ring, at, &sh.abort_flag);
    if (ok) {
      const unsigned char* st = smem + at.stage * ring.stage_bytes;
      fetch<T, MODE, ITEMS>(my, st, x + row * a.ldx, h);
      fetch<T, MODE, ITEMS>(my, st + ring.slot_bytes, dy + row * a.lddy, u);
      if constexpr (RES)
        fetch<T, MODE, ITEMS>(my, st + 2 * ring.slot_bytes, res + row * a.ldr, fr);
      if constexpr (!kKeep) fetch_weights<T, W, MODE, ITEMS>(my, wg, a.cols, gamma);
      const uint64_t scale = pair(rstd, rstd), minus = pair(-mean, -mean);
      uint64_t t1 = pair(0.0f, 0.0f), t2 = pair(0.0f, 0.0f);
      // Behind the row's end dy and gamma are zero: nothing is added there.
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const uint64_t hh = mul2(add2(pair(h[e], h[e + 1]), minus), scale);
        const uint64_t d = pair(u[e], u[e + 1]);
        const uint64_t uu = mul2(d, pair(gamma[e], gamma[e + 1]));
        t1 = add2(t1, uu);
        t2 = fma2(uu, hh, t2);
        split(fma2(d, hh, pair(dg[e], dg[e + 1])), dg[e], dg[e + 1]);
        split(add2(d, pair(db[e], db[e + 1])), db[e], db[e + 1]);
        split(hh, h[e], h[e + 1]);
        split(uu, u[e], u[e + 1]);
      }
      const float s1 = warp_sum(sum2(t1)), s2 = warp_sum(sum2(t2));
      if (lane == 0) sh.red[k & 1][warp] = make_float2(s1, s2);
    }
    __syncthreads();
    if (*(volatile uint32_t*)&sh.abort_flag) break;
    if (tid == 0 && k + ring.stages < mine) issue(k + ring.stages, at.stage);
    const int share = THREADS > 512 ? lane : lane & 15;
    const float2 part = share < nwarps ? sh.red[k & 1][share] : make_float2(0.0f, 0.0f);
    const float c1 = join_sum<THREADS / 32>(part.x) * inv_n * rstd;
    const float c2 = join_sum<THREADS / 32>(part.y) * inv_n * rstd;
    const uint64_t scale = pair(rstd, rstd), n1 = pair(-c1, -c1), n2 = pair(-c2, -c2);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      uint64_t o = fma2(pair(u[e], u[e + 1]), scale, n1);
      o = fma2(pair(h[e], h[e + 1]), n2, o);
      if constexpr (RES) o = add2(o, pair(fr[e], fr[e + 1]));
      split(o, h[e], h[e + 1]);
    }
    put<false, T, MODE, ITEMS>(my, dx + row * a.lddx, h, 0u);
  }
  if (k < mine && tid == 0) ring_drain(ring, at, mine - k);
  float* out = a.partial + (size_t)blockIdx.x * 2 * a.cols;
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = my.column(it, j);
      if (c >= 0 && c < a.cols) {
        out[c] = dg[it * VEC + j];
        out[a.cols + c] = db[it * VEC + j];
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
// of the two outputs a block; warp w takes the partial rows w, w + 16, ...
constexpr int kReduceWarps = 16;
template <typename W>
__global__ void __launch_bounds__(32 * kReduceWarps) k_bwd_reduce(const float* partial,
                                                                  int partials, int cols,
                                                                  W* dgamma, W* dbeta) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float s[kReduceWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float v = 0.0f;
  if (c < cols) {
    const float* p = partial + (size_t)which * cols + c;
    float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int r = warp;
    for (; r + 3 * kReduceWarps < partials; r += 4 * kReduceWarps) {
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] += p[(size_t)(r + j * kReduceWarps) * 2 * cols];
    }
    for (; r < partials; r += kReduceWarps) t[0] += p[(size_t)r * 2 * cols];
    v = (t[0] + t[1]) + (t[2] + t[3]);
  }
  s[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < cols) {
#pragma unroll
    for (int w = 1; w < kReduceWarps; ++w) v += s[w][lane];
    W* out = which == 0 ? dgamma : dbeta;
    if (out) out[c] = from_f32<W>(v);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// Threads for a row of `n` vectors (or elements) at `items` a thread.
int row_threads(int64_t n, int items) { return (int)(((n + items - 1) / items + 31) / 32 * 32); }

// Blocks of `kernel` that an SM's registers and threads take, before shared
// memory (kept: the query costs more than a launch).
template <auto KERNEL>
int blocks_of(int threads, int* blocks) {
  static std::atomic<int> kept[33];
  if (int e = allow_smem<KERNEL>((int)kRingMost)) return e;
  int n = kept[threads / 32].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, 0))
      return cuda_status(e);
    if (n < 1) n = 1;
    kept[threads / 32].store(n, std::memory_order_relaxed);
  }
  *blocks = n;
  return NVFP4_OK;
}

// Ring and grid of a launch: the SM's shared memory over the blocks that fit it
// otherwise, two stages a block at least (fewer blocks then) while they fit.  A
// block's rows, `grid` apart, start at the same phase of 16 bytes.  Of unaligned rows
// the first and the last are not one block's, unless it is the only row.  (There is
// such a grid for all sizes that fit the memory: rows - 1 would have to be a multiple of
// all grids down to 0, and the launch is refused then.)
constexpr int kTooWide = -1;          // rows for the kernels of the widest
struct Launch {
  int stages;
  size_t smem;
  unsigned grid;
};
Launch launch_shape(int blocks, size_t stage_bytes, int sms, int64_t rows, int64_t most,
                    int phases, bool unaligned) {
  Launch l;
  const size_t least = 2 * stage_bytes <= kRingMost ? 2 : 1;
  // (Small rings: what the block holds beside them counts, or not all the blocks that
  // the grid is made for run at once.)
  auto room = [](int n) {
    const size_t all = kSmBytes / n - kBlockBytes;
    return all < kRingBytes / n ? all : kRingBytes / n;
  };
  while (blocks > 1 && room(blocks) < least * stage_bytes) --blocks;
  const size_t fit = room(blocks) / stage_bytes;
  l.stages = (int)(fit < least ? least : fit > (size_t)kMaxStages ? kMaxStages : fit);
  l.smem = l.stages * stage_bytes;
  int64_t g = (int64_t)blocks * sms;
  if (g > most) g = most;
  if (g >= rows) {
    g = rows;
  } else {
    g -= g % phases;
    while (unaligned && g > 0 && (rows - 1) % g == 0) g -= phases;
  }
  l.grid = (unsigned)g;
  return l;
}
// Partial rows of the weights' gradients: enough blocks to fill the SMs, more
// of them where a row takes few threads.
int64_t most_partials(int64_t rows, int64_t cols) {
  const int64_t narrow = 2048 / cols;
  const int64_t p = 296 * (narrow < 1 ? 1 : narrow > 4 ? 4 : narrow);
  return rows < p ? rows : p;
}
// Rows after which a row stride comes back to the same phase of 16 bytes.
int phases_of(int64_t stride_bytes) {
  return stride_bytes % 16 == 0 ? 1 : stride_bytes % 8 == 0 ? 2 : stride_bytes % 4 == 0 ? 4 : 8;
}
// Whether an array's rows start at the same phases as x's.
bool in_phase(const void* x, int64_t ldx, const void* p, int64_t ld, int64_t es) {
  return ((uintptr_t)x - (uintptr_t)p) % 16 == 0 && (ldx - ld) * es % 16 == 0;
}
// Unaligned rows of at least so many columns, and in the backward pass of at
// least so many elements, go by vectors with partial ends (kPhased); the others
// element by element, which starts sooner.  Forward, bf16: 16000 x 1001 32 us against
// 41, 4000 x 4099 31 against 47, 16000 x 777 32 against 38, but fp32 16000 x 501 29
// against 26 and 16000 x 201 25 against 23.  Backward with a residual, bf16: 4000 x
// 4099 50 us against 55, 16000 x 1001 45 against 49, but 1200 x 4099 24.7 against 24.2
// and 4000 x 777 20 against 19.
constexpr int64_t kPhasedCols = 700, kPhasedSize = 1 << 23;
uint32_t slot_of(size_t row_bytes, bool aligned) {
  return (uint32_t)(aligned ? row_bytes : (row_bytes + 15) / 16 * 16 + 16);
}

template <typename T, typename W, int MODE, int ITEMS, int THREADS, int BLOCKS>
int launch_fwd_rows(FwdArgs a, int threads, int sms, cudaStream_t st) {
  constexpr auto kernel = k_fwd_rows<T, W, MODE, ITEMS, THREADS, BLOCKS>;
  int blocks;
  if (int e = blocks_of<kernel>(threads, &blocks)) return e;
  a.slot_bytes = slot_of((size_t)a.cols * sizeof(T), MODE == kWhole);
  const Launch l = launch_shape(blocks, a.slot_bytes, sms, a.rows, INT32_MAX,
                                phases_of(a.ldx * (int64_t)sizeof(T)), MODE != kWhole);
  a.stages = l.stages;
  kernel<<<l.grid, threads, l.smem, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename T, typename W>
int launch_fwd_unaligned(const FwdArgs& a, int sms, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (a.cols >= kPhasedCols && in_phase(a.x, a.ldx, a.y, a.ldy, sizeof(T))) {
    const int64_t n = (a.cols + 2 * V - 2) / V;        // with the largest shift
    if (int t = row_threads(n, 16 / V); t <= 512)
      return launch_fwd_rows<T, W, kPhased, 16 / V, 512, 2>(a, t, sms, st);
  }
  // Element-wise addressing takes more registers: 80 at two blocks of 384.
  if (a.cols <= 32 * 4) return launch_fwd_rows<T, W, kOdd, 4, 32, 16>(a, 32, sms, st);
  const int t = row_threads(a.cols, 16);
  if (t <= 384) return launch_fwd_rows<T, W, kOdd, 16, 384, 2>(a, t, sms, st);
  if (t <= 512) return launch_fwd_rows<T, W, kOdd, 16, 512, 1>(a, t, sms, st);
  return kTooWide;
}

template <typename T, typename W>
int launch_fwd(const FwdArgs& a, int sms, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool aligned = ((uintptr_t)a.x % 16 | (uintptr_t)a.y % 16 | (uintptr_t)(a.ldx % V) |
                        (uintptr_t)(a.ldy % V) | (uintptr_t)(a.cols % V)) == 0;
  // 16 columns a thread (its gamma and beta fill half of the 64 registers that
  // two blocks of 512 threads leave), 8 for a row of one warp, 32 for the widest.
  if (aligned) {
    const int64_t n = a.cols / V;
    if (n <= 32 * (8 / V)) return launch_fwd_rows<T, W, kWhole, 8 / V, 32, 16>(a, 32, sms, st);
    if (int t = row_threads(n, 16 / V); t <= 512)
      return launch_fwd_rows<T, W, kWhole, 16 / V, 512, 2>(a, t, sms, st);
    if (int t = row_threads(n, 32 / V); t <= 512)
      return launch_fwd_rows<T, W, kWhole, 32 / V, 512, 1>(a, t, sms, st);
  } else if (int e = launch_fwd_unaligned<T, W>(a, sms, st); e != kTooWide) {
    return e;
  }
  const int64_t most = (int64_t)sms * 8;
  k_fwd_wide<T, W><<<(unsigned)(a.rows < most ? a.rows : most), kWideThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename T, typename W, int MODE, int ITEMS, int THREADS, bool RES>
int launch_bwd_rows(BwdArgs& a, int threads, int sms, cudaStream_t st) {
  constexpr auto kernel = k_bwd_rows<T, W, MODE, ITEMS, THREADS, RES>;
  int blocks;
  if (int e = blocks_of<kernel>(threads, &blocks)) return e;
  a.slot_bytes = slot_of((size_t)a.cols * sizeof(T), MODE == kWhole);
  const Launch l = launch_shape(blocks, (RES ? 3 : 2) * (size_t)a.slot_bytes, sms, a.rows,
                                most_partials(a.rows, a.cols),
                                phases_of(a.ldx * (int64_t)sizeof(T)), MODE != kWhole);
  a.stages = l.stages;
  a.partials = (int)l.grid;
  kernel<<<l.grid, threads, l.smem, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename T, typename W, bool RES>
int launch_bwd_unaligned(BwdArgs& a, int sms, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (a.cols >= kPhasedCols && a.rows * a.cols >= kPhasedSize &&
      in_phase(a.x, a.ldx, a.dy, a.lddy, sizeof(T)) &&
      in_phase(a.x, a.ldx, a.dx, a.lddx, sizeof(T)) &&
      (!RES || in_phase(a.x, a.ldx, a.res, a.ldr, sizeof(T)))) {
    const int64_t n = (a.cols + 2 * V - 2) / V;
    if (int t = row_threads(n, 8 / V); t <= 704)
      return launch_bwd_rows<T, W, kPhased, 8 / V, 704, RES>(a, t, sms, st);
    if (int t = row_threads(n, 16 / V); t <= 512)
      return launch_bwd_rows<T, W, kPhased, 16 / V, 512, RES>(a, t, sms, st);
  }
  if (int t = row_threads(a.cols, 8); t <= 704)
    return launch_bwd_rows<T, W, kOdd, 8, 704, RES>(a, t, sms, st);
  if (int t = row_threads(a.cols, 16); t <= 512)
    return launch_bwd_rows<T, W, kOdd, 16, 512, RES>(a, t, sms, st);
  return kTooWide;
}

template <typename T, typename W, bool RES>
int launch_bwd(BwdArgs& a, int sms, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool aligned = ((uintptr_t)a.x % 16 | (uintptr_t)a.dy % 16 | (uintptr_t)a.dx % 16 |
                        (uintptr_t)a.res % 16 | (uintptr_t)(a.ldx % V) | (uintptr_t)(a.lddy % V) |
                        (uintptr_t)(a.lddx % V) | (uintptr_t)(RES ? a.ldr % V : 0) |
                        (uintptr_t)(a.cols % V)) == 0;
  // 8 columns a thread while a row then takes at most 512 threads (its warps, or
  // those of several blocks, fill an SM), then 16, then 32.  Unaligned rows stay
  // with 8 up to 704 threads: their addressing leaves 16 too few registers.
  if (aligned) {
    const int64_t n = a.cols / V;
    if (int t = row_threads(n, 8 / V); t <= 512)
      return launch_bwd_rows<T, W, kWhole, 8 / V, 512, RES>(a, t, sms, st);
    if (int t = row_threads(n, 16 / V); t <= 512)
      return launch_bwd_rows<T, W, kWhole, 16 / V, 512, RES>(a, t, sms, st);
    if (int t = row_threads(n, 32 / V); t <= 512)
      return launch_bwd_rows<T, W, kWhole, 32 / V, 512, RES>(a, t, sms, st);
  } else if (int e = launch_bwd_unaligned<T, W, RES>(a, sms, st); e != kTooWide) {
    return e;
  }
  // The weights' partial sums first: dx may overwrite dy.
  a.partials = (int)most_partials(a.rows, a.cols);
  const dim3 grid((unsigned)((a.cols + kWideThreads - 1) / kWideThreads), (unsigned)a.partials);
  k_bwd_wide_w<T><<<grid, kWideThreads, 0, st>>>(a);
  if (cudaError_t e = cudaGetLastError()) return cuda_status(e);
  const int64_t most = (int64_t)sms * 8;
  k_bwd_wide_dx<T, W><<<(unsigned)(a.rows < most ? a.rows : most), kWideThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename W>
int launch_reduce(const BwdArgs& a, void* dgamma, void* dbeta, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.cols + 31) / 32), 2);
  cfg.blockDim = dim3(32 * kReduceWarps);
  cfg.stream = st;
  // Launched while the rows are still being worked on; waits for them.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, k_bwd_reduce<W>, (const float*)a.partial,
                                         a.partials, a.cols, reinterpret_cast<W*>(dgamma),
                                         reinterpret_cast<W*>(dbeta)))
    return cuda_status(e);
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
  if (partly_over(y, ldy, x, ldx, rows, cols, (int64_t)es)) return NVFP4_ERR_INVALID_ARGUMENT;
  int sms = 0;
  if (int e = device_sm_count(&sms)) return e;
  cudaStream_t st = (cudaStream_t)stream;
  if (amax_out)
    if (cudaError_t e = cudaMemsetAsync(amax_out, 0, sizeof(float), st)) return cuda_status(e);
  if (empty) return NVFP4_OK;
  FwdArgs a = {x, gamma, beta, y, mean, rstd, reinterpret_cast<uint32_t*>(amax_out),
               rows, ldx, ldy, (int)cols, 1, 0u, eps};
  if (dtype == NVFP4_DTYPE_F32) return launch_fwd<float, float>(a, sms, st);
  if (dtype == NVFP4_DTYPE_BF16)
    return weight_dtype == NVFP4_DTYPE_F32 ? launch_fwd<__nv_bfloat16, float>(a, sms, st)
                                           : launch_fwd<__nv_bfloat16, __nv_bfloat16>(a, sms, st);
  return weight_dtype == NVFP4_DTYPE_F32 ? launch_fwd<__half, float>(a, sms, st)
                                         : launch_fwd<__half, __half>(a, sms, st);
}

NVFP4_API size_t nvfp4_layernorm_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)most_partials(rows, cols) * 2 * (size_t)cols * sizeof(float);
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
  if (partly_over(dx, lddx, dy, lddy, rows, cols, (int64_t)es) ||
      partly_over(dx, lddx, residual, ldr, rows, cols, (int64_t)es) ||
      partly_over(dx, lddx, x, ldx, rows, cols, (int64_t)es))
    return NVFP4_ERR_INVALID_ARGUMENT;
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
               rows, lddy, ldx, ldr, lddx, (int)cols, 1, 0, 0u, dgamma || dbeta};
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
