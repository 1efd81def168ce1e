// experts_mxfp4.cu -- routed-expert SwiGLU over MXFP4 expert rows: a grouped
// GEMM on the 5th-generation tensor cores with block-scaled operands
// (tcgen05.mma kind::mxf8f6f4), so that 4-bit weights go from memory into the
// MMA without a single instruction spent on expanding them.
//
// The operator beside execute_experts (ferry/csrc/expert_ops.cpp:16-45): per
// group of routes, y = (silu(x Wg^T) * (x Wu^T)) Wd^T * w with W = code *
// 2^(scale - 127).
//
// Operands.  A = weights: e2m1 codes, one scale byte for 32 columns, exactly as
// they lie in the cache row ([gate I x H | up I x H | down H x I] codes, two a
// byte, then their scale bytes in the same order).  B = routes: a bf16 number
// has 8 significant bits and an e4m3 number 4, so a row is stored as two e4m3
// parts, hi (the value rounded to e4m3) and lo (what is left of it), each with
// a power-of-two scale for 32 columns, the lo scale 2^-4 of the hi one; both
// parts are multiplied and summed into the same float32 accumulator.  A block's
// largest value is brought to [2^7, 2^8); hi + lo is then the bf16 number itself
// down to 2^-6 (2^-13 of the largest) and within 2^-14 (2^-21 of the largest)
// below that, half the lo part's smallest step of 2^-9 * 2^-4.  The activation,
// operand of the second product, is stored the same way: hi + lo rounds it to
// within 2^-9 of its value (bf16: 2^-9), or 2^-21 of its block's largest.  Gate, up and silu stay in float32, the result is rounded
// to bf16 once.
//
// Orientation as in experts.cu: 128 weight rows are the MMA's M side (64 gate
// rows above the 64 up rows of the same features, or 128 down rows), the routes
// its N side.  Groups are split into sub-groups of at most 32, 64 or 128 routes
// (by the mean of the groups: small groups need no wide tiles, and narrow ones
// leave shared memory to the weights), each with its own work items, so that a
// popular expert is spread over the GPU.
//
// Data flow of a step (128 columns): TMA unpacks the codes of 128 weight rows
// into 16 KB of shared memory (4-bit data in 8-bit places, 128-byte swizzle, as
// the MMA reads them) and brings the routes' hi and lo parts; cp.async brings
// the weight rows' scale bytes, 4 a step, in pieces of 16, 8 or 4 as the rows are
// aligned (no padding of the scale rows); four warps move the scales of both sides into tensor memory
// (row r in lane r % 32 of every 32-lane quarter, column r / 32, one byte for
// each 32 columns of the step); one thread issues the 8 MMAs of K = 32, hi and
// lo for each scale byte.
//
// CTA roles (512 threads): warp 0 claims work and loads codes; warp 1 issues the
// MMAs; warps 2-5 and 6-9 drain the two accumulators; warp 10 loads the routes;
// warp 15 brings the weights' scales, warps 11-14 move all scales on.  Codes do not depend on phase
// 1, so warp 0 runs ahead into phase 2 while the routes' warps wait for the
// activations.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"
#include "experts.cuh"

namespace ferryb {

constexpr int kMxWarps = 16;
constexpr int kMxThreads = kMxWarps * 32;
constexpr int kFirstEpi = 2, kRouteWarp = 10, kFirstScale = 11, kScaleLoad = 15;
constexpr int kMxM = 128;          // weight rows per tile
constexpr int kMxN = 128;          // most routes of a sub-group
constexpr int kStepK = 128;        // columns per step
constexpr int kSpan = 2;           // steps per load and barrier
constexpr int kMxFeatures = 64;    // gate (= up) rows per phase-1 tile
constexpr int kBars = 8;           // barriers of the spans' pipeline, more than any buffer's depth
constexpr int kBlock = 4;          // steps whose scales come in one piece and are arranged by one warp
constexpr int kPieces = 4;         // places for a block's scales as they are in memory
constexpr uint32_t kStepCodes = kMxM * kStepK;  // a step's codes, unpacked
constexpr uint32_t kCodeBytes = kSpan * kStepCodes;
constexpr uint32_t kPieceBytes = kMxM * 16;  // of up to four steps
constexpr uint32_t kScalePool = 24 * 1024;  // scales as they are in memory, and arranged
constexpr uint32_t kTmemScale = 256;  // first TMEM column of the scales: four places of 16 columns
constexpr int kRing = 4;           // claimed items in flight
constexpr int kXStride = 9;        // floats a feature of the gate/up exchange (padded)
constexpr uint32_t kXchgBytes = 2 * kMxFeatures * kXStride * 4;  // an epilogue group's
constexpr uint32_t kPoolBytes = 12 * 16384;  // codes and routes
constexpr uint32_t kMxSmem = kPoolBytes + kScalePool + 1024 + 1024;
constexpr uint64_t kMxWaitNs = 2000000000ull;  // bound on any wait

// Up to 128 routes of one group.
struct MxGroup {
  int32_t slot;   // cache slot (0 where the caller's is out of range)
  int32_t start;  // first route
  int32_t count;  // routes
  int32_t bad;    // slot out of range: the routes' outputs are NaN
};

// Written by the prepare kernel.
struct MxHeader {
  int queue;     // claim counter
  int n_groups;  // sub-groups
  int box;       // 0..3: sub-groups of at most 16, 32, 64, 128 routes
};

struct MxParams {
  const MxGroup* groups;
  MxHeader* header;
  int mt1, mt2;         // items per sub-group: I / 64 phase 1, H / 128 phase 2
  int tma1, tma2;       // weight scales of phase 1 (2) through s1 (s2): rows of 16-byte multiples
  int hidden, inter;
  const uint8_t* scales;  // slot 0's scale bytes
  int64_t row_bytes;      // bytes of a cache row
  uint8_t* act;           // [routes, 2 * I]: hi, lo
  uint8_t* as;            // hi scale bytes of the activations [routes, pitch2]
  int pitch2;
  __nv_bfloat16* out;
  const float* route_w;
  int* dep;    // [sub-groups] phase-1 epilogue-warp completions, zero at launch
  int* err;
};

struct MxMaps {
  CUtensorMap w1, w2;      // codes of gate and up rows, of down rows
  CUtensorMap x[4], a[4];  // routes and activations, 16, 32, 64, 128 rows at once
  CUtensorMap xs, as;      // their scale bytes [routes, pitch], 16 rows x 16 bytes at once
  CUtensorMap s1, s2;      // scale bytes of gate and up rows, of down rows, 16 bytes of 128 rows
};

// A claimed work item, handed from warp 0 to the other roles.
struct MxItem {
  int phase;  // 1, 2 or 0 = no more work
  int group, tile;
  int start, count, bad;  // of the sub-group
  int slot, pad;
};

__device__ __forceinline__ MxItem mx_item(const MxParams& p, int n_groups, int item) {
  MxItem it{};
  const int n1 = n_groups * p.mt1;
  if (item < n1) {
    it.phase = 1; it.group = item / p.mt1; it.tile = item - it.group * p.mt1;
  } else if (item < n1 + n_groups * p.mt2) {
    const int i = item - n1;
    it.phase = 2; it.group = i / p.mt2; it.tile = i - it.group * p.mt2;
  } else {
    return it;
  }
  const MxGroup g = p.groups[it.group];
  it.start = g.start; it.count = g.count; it.bad = g.bad; it.slot = g.slot;
  return it;
}

// One wait of at most about 20 us: the hint lets the hardware suspend the warp,
// which otherwise polls and takes issue slots from the warps that expand.
__device__ __forceinline__ bool mx_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
// Wait for an mbarrier phase, bounded in time; on time-out the CTA's abort flag
// and the error word are set.  The clock is read only once a wait has become
// long.
__device__ __noinline__ bool mx_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          int* err) {
  const uint64_t t0 = globaltimer_ns();
  for (;;) {
    for (int i = 0; i < 16; ++i)
      if (mx_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (globaltimer_ns() - t0 > kMxWaitNs) {
      *abort_flag = 1;
      atomicCAS(err, 0, DEV_WAIT_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ bool mx_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                        int* err) {
  for (int i = 0; i < 8; ++i)
    if (mx_try_wait(bar, parity)) return true;
  return mx_wait_long(bar, parity, abort_flag, err);
}
// The same for a whole warp: all lanes agree on the outcome.
__device__ __forceinline__ bool mx_wait_warp(uint64_t* bar, uint32_t parity,
                                             volatile int* abort_flag, int* err) {
  return __all_sync(0xffffffffu, mx_wait(bar, parity, abort_flag, err));
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int32_t c0,
                                            int32_t c1, int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int32_t c0,
                                            int32_t c1, int32_t c2, int32_t c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int32_t c0,
                                            int32_t c1, int32_t c2, int32_t c3, int32_t c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3),
      "r"(c4)
      : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_async(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES)
               : "memory");
}
// Arrive on `bar` once this thread's cp.async copies so far have landed (the
// barrier's count includes this arrival).
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// 32 rows of 16 bytes of shared memory (rows one after the other) into 4 columns
// of every 32-lane quarter of tensor memory.  Ordered before the MMAs that the
// same thread issues after it.  Descriptor: address >> 4, 8-row groups 128 bytes
// apart (bits 32-45), version 1 (bits 46-47), no swizzle.
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFF) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(128 >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// 32 lanes x 8 consecutive columns of 32 bits.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float* v) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                 "=r"(r[7])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}

// D[tmem] (+)= (A[smem] * scales) x (B[smem] * scales)^T, 32 columns: e2m1 codes
// in 8-bit places times e4m3, float32 accumulate, one UE8M0 scale for the 32.
__device__ __forceinline__ void umma_mxf8f6f4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                              uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], "
      "p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// Instruction descriptor of kind::mxf8f6f4: A e2m1 (5 in bits 7-9), B e4m3 (0 in
// bits 10-12), both K-major, N >> 3 in bits 17-22, UE8M0 scales (bit 23), M >> 7
// in bits 27-28; the scale byte a K-block takes from its 32-bit columns is in
// bits 4-5 for B and 29-30 for A.
__device__ __forceinline__ uint32_t mx_idesc(uint32_t n, uint32_t byte) {
  return (5u << 7) | ((n >> 3) << 17) | (1u << 23) | (1u << 27) | (byte << 4) | (byte << 29);
}

// A step: its scales into tensor memory, then four K = 32 MMAs (eight with WIDE:
// hi, then lo into the same columns).  Descriptors count in 16 bytes: 32 columns
// are 2, 512 bytes of scales 32, the 128 rows of a wide hi part 1024.
template <bool WIDE>
__device__ __forceinline__ void issue_step(uint32_t d, uint64_t a, uint64_t b, uint32_t b_off, uint32_t sa,
                                           uint64_t from, uint32_t idesc, bool accumulate) {
  tmem_copy_scales(sa, from);
  tmem_copy_scales(sa + 4, from + 32);
  if (WIDE) tmem_copy_scales(sa + 8, from + 64);
  b += b_off;
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    const uint32_t id = idesc | (k << 4) | (k << 29);
    umma_mxf8f6f4(d, a + 2 * k, b + 2 * k, id, sa, sa + 4, accumulate || k > 0 ? 1u : 0u);
    if (WIDE) umma_mxf8f6f4(d, a + 2 * k, b + 1024 + 2 * k, id, sa, sa + 8, 1u);
  }
}

// ---- hi and lo parts of values ----
// Scale byte of a block whose largest magnitude has the float32 exponent field
// `field`: the block's values times 2^(127 - byte) stay below 2^8.  At least 4,
// so that the lo scale (byte - 4) exists; 255 (NaN) if a value is not finite.
__device__ __forceinline__ int mx_block_byte(uint32_t field) {
  return field == 255u ? 255 : max(static_cast<int>(field) - 7, 4);
}
__device__ __forceinline__ float mx_block_mult(int byte) {
  return byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
}
// Two values (already times 2^(127 - byte)) -> two hi bytes and two lo bytes.
__device__ __forceinline__ void mx_split2(float a, float b, uint32_t* hi, uint32_t* lo) {
  const __nv_fp8x2_storage_t h = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3)));
  const __nv_fp8x2_storage_t l = __nv_cvt_float2_to_fp8x2(
      make_float2((a - back.x) * 16.0f, (b - back.y) * 16.0f), __NV_SATFINITE, __NV_E4M3);
  *hi = h;
  *lo = l;
}

// The four warps of epilogue group g (0 or 1) meet at named barrier 1 + g, and
// leave their loop together: every decision goes through a barrier that ANDs
// it.
__device__ __forceinline__ void mx_epilogue_sync(int g) {
  asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");
}
__device__ __forceinline__ bool mx_epilogue_all(int g, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(v)), "r"(1 + g)
      : "memory");
  return r != 0;
}

// The pool of shared memory, by the sub-groups' size: places of codes first, then
// places of routes (hi and lo parts of `box` rows), a span each.  Many places
// for codes where routes are few (memory-bound), as many of both where they
// are many.
__host__ __device__ __forceinline__ int mx_code_stages(int box) {
  return box == 0 ? 5 : box == 1 ? 4 : box == 2 ? 3 : 2;
}
__host__ __device__ __forceinline__ int mx_route_stages(int box) {
  return box == 0 ? 4 : box == 1 ? 4 : box == 2 ? 3 : 2;
}
__host__ __device__ __forceinline__ uint32_t mx_route_bytes(int box) {
  return (16u << box) * kStepK * 2 * kSpan;
}

// Rows of routes that a sub-group's tile holds: 16, 32, 64 or 128.
__device__ __forceinline__ int mx_class(int count) {
  return count <= 16 ? 0 : count <= 32 ? 1 : count <= 64 ? 2 : 3;
}
__device__ __forceinline__ int mx_rows(int count) { return 16 << mx_class(count); }

// A span is two steps: loads, barriers and commits cost the one thread that
// issues them 100 to 300 cycles each (a TMA load alone 290, the next one behind
// it 50), which by the step was more than the step's 375 cycles of HBM time.
// Spans are numbered from 0 over all items of a CTA (an item's last span may be
// half empty: zeros).  Span t uses barrier t % 8 of each pipeline; a buffer of S
// places may be refilled for span t once span t - S is done, and S < 8 keeps the
// parity unambiguous.
__device__ __forceinline__ bool mx_wait_span(uint64_t* bars, uint32_t t, volatile int* abort_flag,
                                             int* err) {
  return mx_wait(bars + t % kBars, (t / kBars) & 1, abort_flag, err);
}

// Wait until the sub-group's activations are written: four epilogue warps for
// each of its phase-1 tiles.
__device__ __forceinline__ bool mx_wait_dep(const int* dep, uint32_t want, volatile int* abort_flag,
                                            int* err) {
  const uint32_t* cnt = reinterpret_cast<const uint32_t*>(dep);
  if (ld_acquire_gpu_u32(cnt) >= want) return true;
  const uint64_t t0 = globaltimer_ns();
  while (ld_acquire_gpu_u32(cnt) < want) {
    __nanosleep(32);
    if (*abort_flag) return false;
    if (globaltimer_ns() - t0 > kMxWaitNs) {
      *abort_flag = 1;
      atomicCAS(err, 0, DEV_WAIT_TIMEOUT);
      return false;
    }
  }
  return true;
}

__global__ void __launch_bounds__(kMxThreads, 1)
    mxfp4_swiglu_kernel(const __grid_constant__ MxMaps maps, const MxParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* scale = smem + kPoolBytes;  // places of weights' scales [128 rows] 16 bytes
  uint64_t* full = reinterpret_cast<uint64_t*>(scale + kScalePool);
  uint64_t* done = full + kBars;     // the MMAs of a step are complete
  uint64_t* kfull = done + kBars;    // [kPieces] a block's scales landed
  uint64_t* kempty = kfull + kPieces;
  uint64_t* tfull = kempty + kPieces;  // [2] accumulators
  uint64_t* tempty = tfull + 2;
  uint64_t* ifull = tempty + 2;      // [kRing] claimed items
  uint64_t* iempty = ifull + kRing;
  uint64_t* drain = iempty + kRing;
  uint32_t* tmem_smem = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_smem + 1);
  MxItem* ring = reinterpret_cast<MxItem*>(drain + 2);  // [kRing]
  __shared__ float xchg_all[2][kXchgBytes / 4];

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kBars; ++s) {
      mbar_init(&full[s], 3);  // codes, routes and scales
      mbar_init(&done[s], 1);
    }
    for (int s = 0; s < kPieces; ++s) {
      mbar_init(&kfull[s], 33);  // TMA, and the lanes' cp.async
      mbar_init(&kempty[s], 1);
    }
    for (int b = 0; b < 2; ++b) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], 4); }
    for (int q = 0; q < kRing; ++q) { mbar_init(&ifull[q], 1); mbar_init(&iempty[q], 11 + (p.header->box == 3 ? 2 : 4)); }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(tmem_smem, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_smem;
  const int box = p.header->box;
  const uint32_t code_stages = mx_code_stages(box), route_stages = mx_route_stages(box);
  const uint32_t route_bytes = mx_route_bytes(box);
  uint8_t* const routes = smem + code_stages * kCodeBytes;
  // Blocks go around the scale warps, each of which has a place of its own for
  // the weights' and for the routes' bytes.  Arranged, a step has 512 bytes of
  // weights' scales, 512 of routes' and, for 128 routes, 512 of lo scales: more,
  // and two warps (and places) instead of four.
  const uint32_t places = box == 3 ? 2 : 4, tile_bytes = box == 3 ? 1536 : 1024;
  const uint32_t place_bytes = box == 3 ? kPieceBytes : kPieceBytes / 2;  // of the routes
  uint8_t* const rscale = scale + places * kPieceBytes;
  uint8_t* const tiles = rscale + places * place_bytes;
  const uint32_t tile_spans = box == 3 ? 5 : 6;
  int q = 0;            // this role's place in the item ring
  uint32_t qphase = 0;

  if (warp == 0) {
    // ---------------- claims and codes ----------------
    if (elect_one()) {
      uint32_t t = 0, stage = 0;
      bool ok = true;
      const int n_groups = p.header->n_groups;
      auto publish = [&](const MxItem& it) {
        if (!mx_wait(&iempty[q], qphase ^ 1, abort_flag, p.err)) return false;
        ring[q] = it;
        mbar_arrive(&ifull[q]);
        if (++q == kRing) { q = 0; qphase ^= 1; }
        return true;
      };
      MxItem it = mx_item(p, n_groups, atomicAdd(&p.header->queue, 1));
      ok = publish(it);
      while (ok && it.phase != 0) {
        // the next item is claimed now and published a few loads on, before this
        // one's last: its scales and routes are under way in time
        const int id = atomicAdd(&p.header->queue, 1);
        MxItem next{};
        const int K = it.phase == 1 ? p.hidden : p.inter;
        const int row0 = it.tile * (it.phase == 1 ? kMxFeatures : kMxM);
        const int steps = K / kStepK, ahead = steps > kSpan ? kSpan : 0;
        for (int kb = 0; kb < steps; kb += kSpan, ++t) {
          if (t >= code_stages && !mx_wait_span(done, t - code_stages, abort_flag, p.err)) {
            ok = false;
            break;
          }
          uint64_t* bar = full + t % kBars;
          uint8_t* cs = smem + stage * kCodeBytes;
          mbar_expect_tx(bar, kCodeBytes / 2);  // the copy counts its 4-bit data, not the gaps
          if (it.phase == 1) tma_load_5d(cs, &maps.w1, bar, 0, row0, 0, kb, it.slot);
          else tma_load_4d(cs, &maps.w2, bar, 0, row0, kb, it.slot);
          if (++stage == code_stages) stage = 0;
          if (kb == ahead) {
            next = mx_item(p, n_groups, id);
            if (!publish(next)) { ok = false; break; }
          }
        }
        it = next;
      }
      if (!ok) {
        // the other roles stop at the abort flag; this CTA's loads get a bounded
        // time to land (a step's barrier may lack another role's arrival now)
        *abort_flag = 1;
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000) {}
      }
    }
  } else if (warp == kScaleLoad) {
    // ---------------- scales into shared memory ----------------
    // Its own warp: the scales of a block go through more hands than the codes
    // and routes of its steps, and start their way earlier.
    uint32_t place = 0, ph = 0;
    bool ok = true;
    while (ok) {
      if (!mx_wait_warp(&ifull[q], qphase, abort_flag, p.err)) break;
      const int phase = ring[q].phase, tile = ring[q].tile, slot = ring[q].slot, group = ring[q].group;
      const int start = ring[q].start, rows = mx_rows(ring[q].count);
      __syncwarp();
      if (lane == 0) mbar_arrive(&iempty[q]);
      if (++q == kRing) { q = 0; qphase ^= 1; }
      if (phase == 0) break;
      const int K = phase == 1 ? p.hidden : p.inter;
      // 16 bytes (four steps) of each tile row: one TMA load where the rows are
      // 16-byte multiples (K a multiple of 512), else cp.async of 8 or 4 bytes, rows
      // lane + 32 * i
      const bool tma = (phase == 1 ? p.tma1 : p.tma2) != 0;
      const int pitch = K / 32;
      const uint8_t* src = p.scales + slot * p.row_bytes +
                           (phase == 1 ? 0 : 2 * static_cast<int64_t>(p.inter) * (p.hidden / 32)) +
                           static_cast<int64_t>(tile * (phase == 1 ? kMxFeatures : kMxM) + lane) * pitch;
      const int64_t d1 = 32 * pitch;
      const int64_t d2 = phase == 1 ? static_cast<int64_t>(p.inter) * pitch : 2 * d1;  // up rows
      if (phase == 2) {
        bool there = true;
        if (lane == 0) there = mx_wait_dep(p.dep + group, 4 * p.mt1, abort_flag, p.err);
        if (!__shfl_sync(0xffffffffu, there, 0)) break;
        asm volatile("fence.proxy.async.global;" ::: "memory");
      }
      for (int b = 0; b < pitch; b += 16) {
        if (!mx_wait_warp(&kempty[place], ph ^ 1, abort_flag, p.err)) { ok = false; break; }
        uint8_t* to = scale + place * kPieceBytes;
        if (lane == 0) {
          mbar_expect_tx(&kfull[place], rows * 16 + (tma ? kPieceBytes : 0));
          if (tma && phase == 1) tma_load_4d(to, &maps.s1, &kfull[place], b, tile * kMxFeatures, 0, slot);
          else if (tma) tma_load_3d(to, &maps.s2, &kfull[place], b, tile * kMxM, slot);
          for (int i = 0; i < rows; i += 16)
            tma_load_2d(rscale + place * place_bytes + i * 16, phase == 1 ? &maps.xs : &maps.as, &kfull[place], b,
                        start + i);
        }
        __syncwarp();
        to += lane * 16;
        const uint8_t* from = src + b;
        if (tma) {
        } else if (pitch % 8 == 0) {
          for (int i = 0; i < min(16, pitch - b); i += 8) {
            cp_async<8>(to + i, from + i);
            cp_async<8>(to + 512 + i, from + d1 + i);
            cp_async<8>(to + 1024 + i, from + d2 + i);
            cp_async<8>(to + 1536 + i, from + d2 + d1 + i);
          }
        } else {
          for (int i = 0; i < min(16, pitch - b); i += 4) {
            cp_async<4>(to + i, from + i);
            cp_async<4>(to + 512 + i, from + d1 + i);
            cp_async<4>(to + 1024 + i, from + d2 + i);
            cp_async<4>(to + 1536 + i, from + d2 + d1 + i);
          }
        }
        cp_async_arrive(&kfull[place]);
        if (++place == places) { place = 0; ph ^= 1; }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kRouteWarp) {
    // ---------------- routes ----------------
    if (elect_one()) {
      uint32_t t = 0, stage = 0;
      bool ok = true;
      while (ok) {
        if (!mx_wait(&ifull[q], qphase, abort_flag, p.err)) { ok = false; break; }
        const MxItem it = ring[q];
        mbar_arrive(&iempty[q]);
        if (++q == kRing) { q = 0; qphase ^= 1; }
        if (it.phase == 0) break;
        if (it.phase == 2) {
          if (!mx_wait_dep(p.dep + it.group, 4 * p.mt1, abort_flag, p.err)) { ok = false; break; }
          asm volatile("fence.proxy.async.global;" ::: "memory");
        }
        const int steps = (it.phase == 1 ? p.hidden : p.inter) / kStepK;
        const int cls = mx_class(it.count);
        const CUtensorMap* map = it.phase == 1 ? &maps.x[cls] : &maps.a[cls];
        for (int kb = 0; kb < steps; kb += kSpan, ++t) {
          if (t >= route_stages && !mx_wait_span(done, t - route_stages, abort_flag, p.err)) {
            ok = false;
            break;
          }
          uint64_t* bar = full + t % kBars;
          mbar_expect_tx(bar, (16u << cls) * kStepK * 2 * kSpan);
          // per step the rows' hi parts, then their lo parts
          tma_load_4d(routes + stage * route_bytes, map, bar, 0, it.start, 0, kb);
          if (++stage == route_stages) stage = 0;
        }
      }
      if (!ok) {
        *abort_flag = 1;
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000) {}
      }
    }
  } else if (warp >= kFirstScale) {
    // ---------------- scales arranged ----------------
    // Into the MMA's order: row r's four bytes of a step at (r % 32) * 16 + r / 32
    // * 4.
    const uint32_t me = warp - kFirstScale;
    uint32_t t = 0, turn = 0, ph = 0;  // spans and blocks of all items
    bool ok = me < places;
    while (ok) {
      if (!mx_wait_warp(&ifull[q], qphase, abort_flag, p.err)) break;
      const int phase = ring[q].phase, rows = mx_rows(ring[q].count);
      __syncwarp();
      if (lane == 0) mbar_arrive(&iempty[q]);
      if (++q == kRing) { q = 0; qphase ^= 1; }
      if (phase == 0) break;
      const int steps = (phase == 1 ? p.hidden : p.inter) / kStepK;
      for (int k = 0; k < steps; k += kBlock) {
        const int n = min(kBlock, steps - k);
        const uint32_t spans = (n + kSpan - 1) / kSpan;
        const bool mine = turn == me;
        if (++turn == places) turn = 0;
        if (!mine) { t += spans; continue; }
        if (!mx_wait_warp(&kfull[me], ph, abort_flag, p.err)) { ok = false; break; }
        ph ^= 1;
        // four steps of weight rows lane + 32 * c, and of routes
        const uint4* rs = reinterpret_cast<const uint4*>(rscale + me * place_bytes);
        const uint4* ws = reinterpret_cast<const uint4*>(scale + me * kPieceBytes);
        uint4 b4[4], a4[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          a4[c] = ws[lane + 32 * c];
          b4[c] = make_uint4(0, 0, 0, 0);
          if (c == 0) b4[c] = rs[rows == 16 ? lane & 15 : lane];
          else if (rows > 32 * c) b4[c] = rs[lane + 32 * c];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&kempty[me]);
        // the tiles' last users are done
        if (t + spans > tile_spans &&
            !__all_sync(0xffffffffu, mx_wait_span(done, t + spans - 1 - tile_spans, abort_flag, p.err))) {
          ok = false;
          break;
        }
#pragma unroll
        for (int i = 0; i < kBlock; ++i) {
          if (i < n) {
            auto part = [&](const uint4& v) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; };
            // the lo scales are 2^-4 of the hi ones (every byte is at least 4)
            constexpr uint32_t kLo = 0x04040404u;
            uint4 b = make_uint4(part(b4[0]), part(b4[1]), part(b4[2]), part(b4[3]));
            uint4* to = reinterpret_cast<uint4*>(
                            tiles + (((t + i / kSpan) % tile_spans) * kSpan + i % kSpan) * tile_bytes) + lane;
            if (rows == 16) {
              if (lane >= 16) b.x -= kLo;
            } else if (rows == 32) {
              b.y = b.x - kLo;
            } else if (rows == 64) {
              b.z = b.x - kLo;
              b.w = b.y - kLo;
            } else {
              to[64] = make_uint4(b.x - kLo, b.y - kLo, b.z - kLo, b.w - kLo);
            }
            to[0] = make_uint4(part(a4[0]), part(a4[1]), part(a4[2]), part(a4[3]));
            to[32] = b;
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane < static_cast<int>(spans)) mbar_arrive(&full[(t + lane) % kBars]);
        t += spans;
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA ----------------
    if (elect_one()) {
      uint32_t t = 0, cstage = 0, rstage = 0, tspan = 0;
      const uint64_t a0 = smem_desc_sw128(smem_u32(smem)), b0 = smem_desc_sw128(smem_u32(routes));
      const uint64_t s0 = smem_desc_scales(smem_u32(tiles));
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      while (ok) {
        if (!mx_wait(&ifull[q], qphase, abort_flag, p.err)) break;
        const int kind = ring[q].phase;
        const uint32_t rows = mx_rows(ring[q].count);
        mbar_arrive(&iempty[q]);
        if (++q == kRing) { q = 0; qphase ^= 1; }
        if (kind == 0) break;
        // up to 64 routes: hi and lo side by side in one MMA of twice the columns
        // (added up in the epilogue), so that the weights are read once; 128: one
        // after the other into the same columns
        const bool wide = rows == 128;
        const uint32_t idesc = mx_idesc(wide ? 128 : 2 * rows, 0);
        const int steps = (kind == 1 ? p.hidden : p.inter) / kStepK;
        if (!mx_wait(&tempty[acc], acc_phase ^ 1, abort_flag, p.err)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * kMxN;
        for (int kb = 0; kb < steps; kb += kSpan, ++t) {
          if (!mx_wait_span(full, t, abort_flag, p.err)) { ok = false; break; }
          tc_fence_after();
          const uint64_t a = a0 + cstage * (kCodeBytes >> 4), b = b0 + rstage * (route_bytes >> 4);
          const uint32_t sa = tmem + kTmemScale + (t & 1) * (kSpan * 16);
          const uint64_t from = s0 + tspan * (kSpan * tile_bytes >> 4);
          if (wide) {
            issue_step<true>(d, a, b, 0, sa, from, idesc, kb > 0);
            if (kb + 1 < steps)
              issue_step<true>(d, a + (kStepCodes >> 4), b, 256 * kStepK >> 4, sa + 16, from + (1536 >> 4), idesc, true);
          } else {
            issue_step<false>(d, a, b, 0, sa, from, idesc, kb > 0);
            if (kb + 1 < steps)
              issue_step<false>(d, a + (kStepCodes >> 4), b, rows * (2 * kStepK >> 4), sa + 16, from + (tile_bytes >> 4),
                                idesc, true);
          }
          umma_commit(&done[t % kBars]);
          if (++cstage == code_stages) cstage = 0;
          if (++rstage == route_stages) rstage = 0;
          if (++tspan == tile_spans) tspan = 0;
        }
        if (!ok) break;
        umma_commit(&tfull[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      // no MMA may still be writing tensor memory when the CTA frees it
      umma_commit(drain);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < kMxWaitNs) {}
    }
  } else {
    // ---------------- epilogue (warps 2..9) ----------------
    // group 0 drains accumulator 0, group 1 accumulator 1: every other item.
    // TMEM lanes 32 * (warp % 4)..: quarters 0, 1 hold gate rows of a phase-1
    // tile, 2, 3 the up rows of the same features
    const int eg = (warp - kFirstEpi) >> 2;
    const int qd = warp & 3;
    const bool up_rows = qd >= 2;
    const int f_local = (qd & 1) * 32 + lane;
    float* xchg = xchg_all[eg];
    float* give = xchg + (up_rows ? kMxFeatures * kXStride : 0) + f_local * kXStride;
    const float* take = xchg + (up_rows ? 0 : kMxFeatures * kXStride) + f_local * kXStride;
    uint32_t acc_phase = 0;
    for (int turn = 0;; turn ^= 1) {
      if (!mx_epilogue_all(eg, mx_wait(&ifull[q], qphase, abort_flag, p.err))) break;
      const MxItem it = ring[q];
      __syncwarp();
      if (lane == 0) mbar_arrive(&iempty[q]);
      if (++q == kRing) { q = 0; qphase ^= 1; }
      if (it.phase == 0) break;  // the same entry for all four warps
      if (turn != eg) continue;
      // routing weights of routes lane, lane + 32, ... (phase 2)
      float w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        w[c] = it.bad ? __uint_as_float(0x7fc00000u)
               : it.phase == 2 && lane + 32 * c < it.count ? p.route_w[it.start + lane + 32 * c] : 0.0f;
      if (!mx_epilogue_all(eg, mx_wait(&tfull[eg], acc_phase, abort_flag, p.err))) break;
      acc_phase ^= 1;
      tc_fence_after();
      const uint32_t d = tmem + (static_cast<uint32_t>(qd * 32) << 16) + eg * kMxN;
      // 8 columns from c0 on: the hi part's sums, plus the lo part's where they
      // have columns of their own
      const int lo_at = it.count > 64 ? 0 : mx_rows(it.count);
      auto columns = [&](int c0, float* v) {
        tmem_ld8(d + c0, v);
        if (lo_at) {
          float more[8];
          tmem_ld8(d + lo_at + c0, more);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] += more[j];
        }
      };
      if (it.phase == 1) {
        // 16 routes at a time: gate warps finish the first 8, up warps the rest
        const int block = it.tile * 2 + (qd & 1);  // of 32 features
        for (int c0 = 0; c0 < it.count; c0 += 16) {
          float lo[8], hi[8];
          columns(c0, lo);
          columns(c0 + 8, hi);
#pragma unroll
          for (int j = 0; j < 8; ++j) give[j] = up_rows ? lo[j] : hi[j];
          mx_epilogue_sync(eg);
          const int first = c0 + (up_rows ? 8 : 0);
          const int n = it.count - first;  // of these 8 routes
          if (n > 0) {
            // no branches between the routes: 8 independent chains
            float a[8];
            uint32_t top[8], h[4], l[4];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float gate = up_rows ? take[j] : lo[j];
              const float up = up_rows ? hi[j] : take[j];
              a[j] = __fdividef(gate, 1.0f + __expf(-gate)) * up;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              top[j] = __reduce_max_sync(0xffffffffu, __float_as_uint(a[j]) & 0x7fffffffu);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              top[j] = mx_block_byte(top[j] >> 23);
              a[j] *= mx_block_mult(top[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) mx_split2(a[2 * j], a[2 * j + 1], &h[j], &l[j]);
            uint8_t* to = p.act + static_cast<int64_t>(it.start + first) * (2 * p.inter) +
                          it.tile * kMxFeatures + f_local;
            uint8_t* sb = p.as + static_cast<int64_t>(it.start + first) * p.pitch2 + block;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (j < n) {
                to[0] = static_cast<uint8_t>(j & 1 ? h[j / 2] >> 8 : h[j / 2]);
                to[p.inter] = static_cast<uint8_t>(j & 1 ? l[j / 2] >> 8 : l[j / 2]);
                if (lane == 0) sb[0] = static_cast<uint8_t>(top[j]);
              }
              to += 2 * p.inter;
              sb += p.pitch2;
            }
          }
          mx_epilogue_sync(eg);
        }
      } else {
        __nv_bfloat16* to = p.out + static_cast<int64_t>(it.start) * p.hidden + it.tile * kMxM + qd * 32 + lane;
        for (int c0 = 0; c0 < it.count; c0 += 8) {
          float v[8];
          columns(c0, v);
          const float ws = c0 < 32 ? w[0] : c0 < 64 ? w[1] : c0 < 96 ? w[2] : w[3];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float wj = __shfl_sync(0xffffffffu, ws, (c0 & 24) + j);
            if (c0 + j < it.count) *to = __float2bfloat16_rn(v[j] * wj);
            to += p.hidden;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[eg]);
      if (it.phase == 1) {
        // publish this warp's activations to the sub-group's phase-2 items
        __threadfence();
        __syncwarp();
        if (lane == 0) atomicAdd(p.dep + it.group, 1);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// Before the GEMM, one launch: block 0 turns the groups into sub-groups and
// zeroes the counters; the other blocks gather the routes' rows as hi and lo
// parts, their scales and weights, a warp per route.
struct MxPrepare {
  const int64_t* slots;
  const int64_t* starts;
  int n_groups;
  int64_t cache_slots, routes;
  const int64_t* rows;
  const int64_t* cols;
  const __nv_bfloat16* input;
  int64_t n_input, input_stride;
  const void* weights;
  int weights_type;
  int64_t topk;
  int hidden, pitch1;
  uint8_t* x;   // [routes, 2 * hidden]
  uint8_t* xs;  // [routes, pitch1]
  float* route_w;
  MxGroup* groups;
  MxHeader* header;
  int* dep;
  int* err;
};

constexpr int kPrepThreads = 256;

__global__ void __launch_bounds__(kPrepThreads) mxfp4_prepare_kernel(const MxPrepare a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x == 0) {
    __shared__ int warp_sum[kPrepThreads / 32];
    __shared__ int base;
    // ascending starts inside [0, routes], or no group at all: the tables below
    // are sized for groups that do not overlap
    bool ordered = true;
    int active = 0;
    for (int g = threadIdx.x; g <= a.n_groups; g += kPrepThreads) {
      const int64_t s0 = a.starts[g], before = g == 0 ? 0 : a.starts[g - 1];
      ordered &= s0 >= before && s0 <= a.routes;
      active += g > 0 && s0 > before;
    }
    if (threadIdx.x == 0) { base = 0; a.header->queue = 0; }
    ordered = __syncthreads_and(ordered);
    if (!ordered) {
      if (threadIdx.x == 0) { a.header->n_groups = 0; a.header->box = 0; atomicCAS(a.err, 0, DEV_BAD_INPUT); }
      return;
    }
    atomicAdd(&base, active);
    __syncthreads();
    active = base;
    __syncthreads();
    if (threadIdx.x == 0) base = 0;
    // sub-groups no wider than the mean group asks for, in one of four sizes
    const int64_t all = a.starts[a.n_groups] - a.starts[0];
    const int64_t mean = active ? (all + active - 1) / active : 0;
    const int cap = mean <= 4 ? 16 : mean <= 24 ? 32 : mean <= 48 ? 64 : 128;
    __syncthreads();
    for (int g0 = 0; g0 < a.n_groups; g0 += kPrepThreads) {
      const int g = g0 + threadIdx.x;
      int s0 = 0, count = 0;
      int64_t slot = 0;
      if (g < a.n_groups) {
        s0 = static_cast<int>(a.starts[g]);
        count = static_cast<int>(a.starts[g + 1]) - s0;
        slot = a.slots[g];
      }
      const bool bad = count > 0 && (slot < 0 || slot >= a.cache_slots);
      if (bad) { slot = 0; atomicCAS(a.err, 0, DEV_BAD_INPUT); }
      const int n = (count + cap - 1) / cap;
      int scan = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
      }
      if (lane == 31) warp_sum[warp] = scan;
      __syncthreads();
      int before = base;
      for (int w = 0; w < warp; ++w) before += warp_sum[w];
      const int at = before + scan - n;
      // parts of count / n routes, the first count % n of them one longer
      for (int i = 0, r = s0; i < n; ++i) {
        const int len = count / n + (i < count % n);
        a.groups[at + i] = MxGroup{static_cast<int>(slot), r, len, bad ? 1 : 0};
        a.dep[at + i] = 0;
        r += len;
      }
      __syncthreads();
      if (threadIdx.x == kPrepThreads - 1) base = before + scan;
      __syncthreads();
    }
    if (threadIdx.x == 0) {
      a.header->n_groups = base;
      a.header->box = cap == 16 ? 0 : cap == 32 ? 1 : cap == 64 ? 2 : 3;
    }
    return;
  }
  // routes outside [starts[0], starts[n_groups]) belong to no group
  int64_t lo = a.starts[0], hi = a.starts[a.n_groups];
  lo = lo < 0 ? 0 : lo;
  hi = hi > a.routes ? a.routes : hi;
  const int64_t step = static_cast<int64_t>(gridDim.x - 1) * (kPrepThreads / 32);
  for (int64_t i = lo + static_cast<int64_t>(blockIdx.x - 1) * (kPrepThreads / 32) + warp; i < hi; i += step) {
    const int64_t row = a.rows[i], col = a.cols[i];
    const bool good = row >= 0 && row < a.n_input && col >= 0 && col < a.topk;
    if (lane == 0) {
      float w = __uint_as_float(0x7fc00000u);
      if (good) {
        const int64_t k = row * a.topk + col;
        w = a.weights_type == FERRYB_FP32   ? static_cast<const float*>(a.weights)[k]
            : a.weights_type == FERRYB_FP16 ? __half2float(static_cast<const __half*>(a.weights)[k])
                                            : __bfloat162float(static_cast<const __nv_bfloat16*>(a.weights)[k]);
      } else {
        atomicCAS(a.err, 0, DEV_BAD_INPUT);
      }
      a.route_w[i] = w;
    }
    const uint4* from = reinterpret_cast<const uint4*>(a.input + (good ? row : 0) * a.input_stride);
    uint2* to = reinterpret_cast<uint2*>(a.x + i * 2 * a.hidden);
    uint8_t* sb = a.xs + i * a.pitch1;
    // 8 values a lane, a block of 32 in four neighbours (hidden is a multiple of
    // 128: whole blocks, and the lanes of a block are all in or all out)
    for (int v0 = 0; v0 < a.hidden / 8; v0 += 32) {
      const int v = v0 + lane;
      const bool in = v < a.hidden / 8;
      uint4 e = make_uint4(0, 0, 0, 0);
      if (in && good) e = from[v];
      const uint32_t m = __vmaxu2(__vmaxu2(e.x & 0x7fff7fffu, e.y & 0x7fff7fffu),
                                  __vmaxu2(e.z & 0x7fff7fffu, e.w & 0x7fff7fffu));
      uint32_t top = max(m & 0xffffu, m >> 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int byte = mx_block_byte(top >> 7);
      const float mult = mx_block_mult(byte);
      const uint32_t in8[4] = {e.x, e.y, e.z, e.w};
      uint32_t h[4], l[4];
#pragma unroll
      for (int i2 = 0; i2 < 4; ++i2)
        mx_split2(__uint_as_float(in8[i2] << 16) * mult, __uint_as_float(in8[i2] & 0xffff0000u) * mult,
                  &h[i2], &l[i2]);
      if (in) {
        to[v] = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        to[a.hidden / 8 + v] = make_uint2(l[0] | (l[1] << 16), l[2] | (l[3] << 16));
        if ((v & 3) == 0) sb[v >> 2] = static_cast<uint8_t>(byte);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
static int make_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base,
                    const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box, bool swizzle) {
  PFN_encodeTiled enc = encode_tiled_fn();
  if (!enc) return fail(FERRYB_ECUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint32_t elem[5] = {1, 1, 1, 1, 1};
  CUresult r = enc(map, type, rank, const_cast<void*>(base), dims, strides, box, elem,
                   CU_TENSOR_MAP_INTERLEAVE_NONE,
                   swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(FERRYB_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return FERRYB_OK;
}

// All maps of a call.  Codes are 4-bit elements, unpacked on the way (16 codes
// to 16 bytes of shared memory, 8 of them data).  A column index is split into
// steps of 128 and the column inside, so that one load brings a span: for
// each of its steps the tile's rows (gate rows, then up rows; for routes the hi
// parts, then the lo parts), 128 columns each.
static int make_maps(MxMaps* m, const ferryb_mxfp4_experts_args* e, const uint8_t* x, const uint8_t* act,
                     const uint8_t* xs, const uint8_t* as, int64_t pitch1, int64_t pitch2) {
  const cuuint64_t H = e->hidden, I = e->intermediate, slots = e->cache_slots, routes = e->routes;
  const cuuint64_t row_bytes = 3 * H * I / 32 * 17;
  const uint8_t* cache = static_cast<const uint8_t*>(e->cache);
  constexpr auto k4 = CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B;
  constexpr auto k8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int s;
  {
    const cuuint64_t dims[5] = {kStepK, I, 2, H / kStepK, slots};
    const cuuint64_t strides[4] = {H / 2, I * H / 2, kStepK / 2, row_bytes};
    const cuuint32_t box[5] = {kStepK, kMxFeatures, 2, kSpan, 1};
    if ((s = make_map(&m->w1, k4, 5, cache, dims, strides, box, true))) return s;
  }
  {
    const cuuint64_t dims[4] = {kStepK, H, I / kStepK, slots};
    const cuuint64_t strides[3] = {I / 2, kStepK / 2, row_bytes};
    const cuuint32_t box[4] = {kStepK, kMxM, kSpan, 1};
    if ((s = make_map(&m->w2, k4, 4, cache + H * I, dims, strides, box, true))) return s;
  }
  // weight scales of rows that are 16-byte multiples (the strides' unit)
  const uint8_t* scales = cache + 3 * H * I / 2;
  if (H % 512 == 0) {
    const cuuint64_t dims[4] = {H / 32, I, 2, slots};
    const cuuint64_t strides[3] = {H / 32, I * (H / 32), row_bytes};
    const cuuint32_t box[4] = {16, kMxFeatures, 2, 1};
    if ((s = make_map(&m->s1, k8, 4, scales, dims, strides, box, false))) return s;
  }
  if (I % 512 == 0) {
    const cuuint64_t dims[3] = {I / 32, H, slots};
    const cuuint64_t strides[2] = {I / 32, row_bytes};
    const cuuint32_t box[3] = {16, kMxM, 1};
    if ((s = make_map(&m->s2, k8, 3, scales + 2 * I * (H / 32), dims, strides, box, false))) return s;
  }
  for (int c = 0; c < 4; ++c) {
    const cuuint32_t box[4] = {kStepK, 16u << c, 2, kSpan};
    for (int phase = 0; phase < 2; ++phase) {
      const cuuint64_t K = phase ? I : H;
      const cuuint64_t dims[4] = {kStepK, routes, 2, K / kStepK};
      const cuuint64_t strides[3] = {2 * K, K, kStepK};
      if ((s = make_map(phase ? &m->a[c] : &m->x[c], k8, 4, phase ? act : x, dims, strides, box, true)))
        return s;
    }
  }
  for (int phase = 0; phase < 2; ++phase) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(phase ? pitch2 : pitch1), routes};
    const cuuint64_t strides[1] = {dims[0]};
    const cuuint32_t box[2] = {16, 16};
    if ((s = make_map(phase ? &m->as : &m->xs, k8, 2, phase ? as : xs, dims, strides, box, false))) return s;
  }
  return FERRYB_OK;
}

static int64_t mx_align(int64_t b) { return (b + 255) & ~int64_t(255); }

struct MxWs {
  int64_t x, xs, act, as, w, groups, header, total;
  int64_t pitch1, pitch2, max_sub;
};
static MxWs mx_ws(int64_t routes, int64_t n_groups, int64_t hidden, int64_t inter) {
  MxWs w{};
  w.max_sub = n_groups + routes / 16 + 1;
  w.pitch1 = (hidden / 32 + 15) & ~int64_t(15);
  w.pitch2 = (inter / 32 + 15) & ~int64_t(15);
  w.x = 0;
  w.xs = w.x + mx_align(routes * hidden * 2);
  w.act = w.xs + mx_align(routes * w.pitch1);
  w.as = w.act + mx_align(routes * inter * 2);
  w.w = w.as + mx_align(routes * w.pitch2);
  w.groups = w.w + mx_align(routes * 4);
  w.header = w.groups + mx_align(w.max_sub * (int64_t)sizeof(MxGroup));
  w.total = w.header + 256 + mx_align(w.max_sub * 4);  // then the dependency counters
  return w;
}

}  // namespace ferryb

using namespace ferryb;

static int mx_sizes(int64_t routes, int64_t n_groups, int64_t hidden, int64_t inter) {
  FB_CHECK_ARG(hidden > 0 && inter > 0 && hidden % 128 == 0 && inter % 128 == 0 &&
                   hidden <= 65536 && inter <= 65536,
               "execute_experts_mxfp4: hidden (%lld) and intermediate (%lld) must be multiples of 128, "
               "at most 65536", (long long)hidden, (long long)inter);
  FB_CHECK_ARG(routes >= 0 && routes <= (int64_t(1) << 30) && n_groups >= 0 &&
                   n_groups <= (int64_t(1) << 20),
               "execute_experts_mxfp4: %lld routes in %lld groups", (long long)routes,
               (long long)n_groups);
  // the work counter is 32 bits
  FB_CHECK_ARG((n_groups + routes / 16 + 1) * (inter / 64 + hidden / 128) < (int64_t(1) << 30),
               "execute_experts_mxfp4: too many work items");
  return FERRYB_OK;
}

extern "C" int64_t ferryb_execute_experts_mxfp4_workspace(int64_t routes, int64_t n_groups,
                                                          int64_t hidden, int64_t intermediate) {
  if (mx_sizes(routes, n_groups, hidden, intermediate)) return -1;
  return mx_ws(routes, n_groups, hidden, intermediate).total;
}

extern "C" int ferryb_execute_experts_mxfp4(const ferryb_mxfp4_experts_args* e, cudaStream_t stream) {
  FB_CHECK_ARG(e, "execute_experts_mxfp4: null argument");
  int s = mx_sizes(e->routes, e->n_groups, e->hidden, e->intermediate);
  if (s) return s;
  if (e->routes == 0 || e->n_groups == 0) return FERRYB_OK;
  FB_CHECK_ARG(e->cache && e->input && e->routing_weights && e->slots && e->starts && e->rows &&
                   e->cols && e->out && e->err, "execute_experts_mxfp4: null pointer");
  FB_CHECK_ARG(e->cache_slots >= 1 && e->cache_slots <= 0x7fffffff,
               "execute_experts_mxfp4: %lld cache slots", (long long)e->cache_slots);
  FB_CHECK_ARG(e->n_input >= 0 && e->topk >= 0, "execute_experts_mxfp4: bad input sizes");
  FB_CHECK_ARG(e->weights_type >= FERRYB_BF16 && e->weights_type <= FERRYB_FP32,
               "execute_experts_mxfp4: unknown weights type %d", e->weights_type);
  FB_CHECK_ARG(reinterpret_cast<uintptr_t>(e->cache) % 32 == 0 &&
                   reinterpret_cast<uintptr_t>(e->input) % 16 == 0 &&
                   (e->n_input <= 1 || (e->input_stride % 8 == 0 && e->input_stride >= e->hidden)),
               "execute_experts_mxfp4: the cache must be 32-byte, input rows 16-byte aligned");
  const MxWs ws = mx_ws(e->routes, e->n_groups, e->hidden, e->intermediate);
  FB_CHECK_ARG(e->workspace && reinterpret_cast<uintptr_t>(e->workspace) % 256 == 0 &&
                   e->workspace_bytes >= ws.total,
               "execute_experts_mxfp4: workspace too small (%lld < %lld) or misaligned",
               (long long)e->workspace_bytes, (long long)ws.total);
  uint8_t* base = static_cast<uint8_t*>(e->workspace);

  MxPrepare pr{};
  pr.slots = e->slots;
  pr.starts = e->starts;
  pr.n_groups = static_cast<int>(e->n_groups);
  pr.cache_slots = e->cache_slots;
  pr.routes = e->routes;
  pr.rows = e->rows;
  pr.cols = e->cols;
  pr.input = static_cast<const __nv_bfloat16*>(e->input);
  pr.n_input = e->n_input;
  pr.input_stride = e->input_stride;
  pr.weights = e->routing_weights;
  pr.weights_type = e->weights_type;
  pr.topk = e->topk;
  pr.hidden = static_cast<int>(e->hidden);
  pr.pitch1 = static_cast<int>(ws.pitch1);
  pr.x = base + ws.x;
  pr.xs = base + ws.xs;
  pr.route_w = reinterpret_cast<float*>(base + ws.w);
  pr.groups = reinterpret_cast<MxGroup*>(base + ws.groups);
  pr.header = reinterpret_cast<MxHeader*>(base + ws.header);
  pr.dep = reinterpret_cast<int*>(base + ws.header + 256);
  pr.err = e->err;

  int device = 0;
  FB_CUDA(cudaGetDevice(&device));
  const int sms = num_sms(device);
  MxMaps maps{};
  if ((s = make_maps(&maps, e, pr.x, base + ws.act, pr.xs, base + ws.as, ws.pitch1, ws.pitch2))) return s;
  MxParams p{};
  p.groups = pr.groups;
  p.header = pr.header;
  p.mt1 = static_cast<int>(e->intermediate / kMxFeatures);
  p.mt2 = static_cast<int>(e->hidden / kMxM);
  p.tma1 = e->hidden % 512 == 0;
  p.tma2 = e->intermediate % 512 == 0;
  p.hidden = static_cast<int>(e->hidden);
  p.inter = static_cast<int>(e->intermediate);
  p.scales = static_cast<const uint8_t*>(e->cache) + 3 * e->hidden * e->intermediate / 2;
  p.row_bytes = 3 * e->hidden * e->intermediate / 32 * 17;
  p.act = base + ws.act;
  p.as = base + ws.as;
  p.pitch2 = static_cast<int>(ws.pitch2);
  p.out = static_cast<__nv_bfloat16*>(e->out);
  p.route_w = pr.route_w;
  p.dep = pr.dep;
  p.err = e->err;

  const int64_t gather = (e->routes + kPrepThreads / 32 - 1) / (kPrepThreads / 32);
  const int64_t most = 8 * static_cast<int64_t>(sms);
  mxfp4_prepare_kernel<<<1 + static_cast<int>(gather < most ? gather : most), kPrepThreads, 0, stream>>>(pr);
  FB_LAUNCH_CHECK();
  static std::atomic<bool> attr_set[64];
  if (device >= 64 || !attr_set[device].load(std::memory_order_acquire)) {
    FB_CUDA(cudaFuncSetAttribute(mxfp4_swiglu_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)kMxSmem));
    if (device < 64) attr_set[device].store(true, std::memory_order_release);
  }
  const int64_t subs = e->n_groups < e->routes ? e->n_groups + e->routes / 16 : e->routes;
  const int64_t items = subs * (p.mt1 + p.mt2);
  mxfp4_swiglu_kernel<<<static_cast<int>(items < sms ? items : sms), kMxThreads, kMxSmem, stream>>>(maps, p);
  FB_LAUNCH_CHECK();
  return FERRYB_OK;
}
