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
// below that, half the lo part's smallest step of 2^-9 * 2^-4.  (Of 2^-115 where the
// block's largest is less: scale bytes have an end.)  The activation times its route's
// weight, operand of the second product, is stored the same way: hi + lo rounds it to
// within 2^-9 of its value, half of what bf16's rounding may take (2^-8), or 2^-21 of
// its block's largest.  It is the one rounding below 32 bits before the result's: two
// e4m3 parts are what keeps the weights as they are (a third would be half as many
// bytes and MMAs again in the second product), and an error of 0.0018 of the result's
// norm against 0.0017 from its rounding to bf16 alone.  Gate, up and silu stay in
// float32, the result is rounded to bf16 once.
//
// Orientation as in experts.cu: 128 weight rows are the MMA's M side (four times
// 16 gate rows and the 16 up rows of the same features, so that a feature's gate
// and up meet in one warp; or 128 down rows), the routes its N side.  An item is
// two such tiles, which share the routes, by a sub-group of up to 16, 32, 48, 64 or
// 112 routes (by the mean of the groups: few routes leave shared memory to the
// weights; 112 is what two accumulators of two tiles leave room for beside the
// scales).  A popular expert is many items, spread over the GPU.  One tile an
// item, with two CTAs on an SM instead, loads the routes twice as often: 64 decode
// tokens 44 us against 36, 4096 prompt tokens 429 against 342.
//
// Data flow of a step (128 columns): one TMA load unpacks the codes of 256 weight
// rows into 32 KB of shared memory (4-bit data in 8-bit places, 128-byte swizzle, as
// the MMA reads them), one brings the routes' hi and lo parts; the scale bytes of
// four steps come in pieces of 16 bytes a row, by TMA or, where K is no multiple of
// 512, by cp.async; two warps arrange them and tcgen05.cp copies them into tensor
// memory (row r's bytes in lane r % 32 of every 32-lane quarter, column r / 32, a byte
// for each 32 columns).  Up to 48 routes: hi and lo side by side in N, added up in the
// epilogue, so that the weights are read once (four MMAs a tile); more: hi, then lo
// into the same columns, the weights kept in the tensor core's buffer in between.
//
// CTA roles (512 threads): warp 0 claims work and loads codes; warps 1 and 2 issue a
// tile's MMAs each; warps 3-10 drain the accumulators, four a tile; warp 11 loads the
// routes; warps 12 and 13 arrange scales, warps 14 and 15 bring the weights' and the
// routes'.  Codes do not depend on phase 1, so warps 0 and 14 run ahead into phase 2
// while the routes' warps wait for the activations.
//
// What bounds it.  2048 x 768 experts, GPU time: 8 experts of one token 15.6 us, of
// which the chain prepare - claim - load - phase 1 - phase 2 without queueing is about
// 11 (32 experts of 256 x 128 take 11.5); 64 tokens (43 experts, 110 MB) 32.5 us: 8
// before the first load and after the last store, phase 1 at 5.6 TB/s, about 5 lost in
// the change of phase and with the last items; 4096 tokens of 8 routes 310 us (367 to 377 when
// it runs on and the power limit brings the clock to 1.5 GHz): 36 for the routes' hi and
// lo parts (134 MB written), then 1,220 cycles a step whose MMAs take 750: loads are
// under way for 1,900 cycles (850 alone), 33 bytes a cycle into the SM where tiles that
// all lie in a corner of L2 come at 40 to 55.  Half the route bytes, or half the MMAs,
// change a step by 3 to 6 %.
// Tried and left out: prefetching the next item into L2 (64 tokens 34 -> 38 to 40 us:
// the loads of the item at hand wait behind it), routes gathered by cp.async in the
// kernel (no prepared copies, but 36 -> 42, and 342 -> 335), 16 epilogue warps (34 ->
// 39), scales copied a step ahead (321 -> 350), four stages of 80 routes for three of
// 112 (321 -> 343), one tile an item where groups are few (8 experts 16.1 -> 17.2).
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"
#include "experts.cuh"

namespace ferryb {

constexpr int kMxM = 128;          // weight rows per tile
constexpr int kStepK = 128;        // columns per step
constexpr int kMxFeatures = 64;    // gate (= up) rows per phase-1 tile
constexpr int kBars = 8;           // barriers of the step pipeline, more than any buffer's depth
constexpr int kBlock = 4;          // steps whose scales come in one piece and are arranged by one warp
constexpr int kPlaces = 2;         // such pieces in shared memory, one for each of two warps
constexpr uint32_t kTileCodes = kMxM * kStepK;  // a step's codes of one tile, unpacked
constexpr uint32_t kPieceBytes = kMxM * 16;     // scale bytes of four steps of 128 rows
constexpr int kRing = 4;           // claimed items in flight
constexpr uint32_t kXchgBytes = 2 * 4 * 32;  // magnitudes of 16 routes from four warps, twice
constexpr uint32_t kBarBytes = 512;

constexpr int kTiles = 2;          // tiles of weight rows per item
// warps: 0 claims and codes, 1 and 2 MMAs of a tile each, then
constexpr int kFirstEpi = 3, kEpiWarps = 4 * kTiles, kRouteWarp = kFirstEpi + kEpiWarps, kFirstScale = kRouteWarp + 1,
              kScaleLoad = kFirstScale + 2, kRouteScale = kScaleLoad + 1;
constexpr int kMxThreads = (kRouteScale + 1) * 32;
constexpr int kItemReaders = 2 + kEpiWarps + 5;
constexpr uint32_t kCodeBytes = kTiles * kTileCodes;
constexpr uint32_t kPoolBytes = 196 * 1024;        // codes and routes
constexpr uint32_t kTilePool = 12 * 1024;          // arranged scales
// tensor memory: two accumulators of two tiles of 112 columns, then the scales: two
// places of two times 12 columns (weights', hi, lo) where hi and lo are apart,
// else four of two times 8
constexpr uint32_t kTmemCols = 512, kTileCols = 112, kAccCols = kTiles * kTileCols, kTmemScale = 2 * kAccCols;
constexpr uint32_t kMxSmem =
    kPoolBytes + kPlaces * (kTiles + 1) * kPieceBytes + kTilePool + kTiles * kXchgBytes + kBarBytes;
static_assert(kMxSmem <= 227 * 1024, "shared memory");
// one wrap at most when a block of steps is passed over in the ring of arranged scales
static_assert(kTilePool / ((kTiles + 2) * 512) >= kBlock, "ring of arranged scales");
constexpr uint64_t kMxWaitNs = 2000000000ull;  // bound on any wait

// Up to 112 routes of one group (kTileCols, MxHeader's cap).
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
  int cap;       // most routes of a sub-group: 16, 32, 48, 64 or 112
};

struct MxParams {
  const MxGroup* groups;
  MxHeader* header;
  int mt1, mt2;         // items per sub-group, each of two tiles: I / 64 tiles phase 1, H / 128 phase 2
  int t1, t2;           // those tiles
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
  CUtensorMap x[7], a[7];  // routes and activations: 16, 32, ... 112 rows at once
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
// which otherwise polls and takes issue slots from the warps that work.
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
// 32 lanes x 16 consecutive columns of 32 bits; tmem_ld_wait before they are used.
__device__ __forceinline__ void tmem_ld16_start(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32"
      " {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
        "=f"(v[14]), "=f"(v[15])
      : "r"(taddr));
}
// The values pass through, so that no use of them moves before the wait.
__device__ __forceinline__ void tmem_ld_wait(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
                 "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]),
                 "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}

// D[tmem] (+)= (A[smem] * scales) x (B[smem] * scales)^T, 32 columns: e2m1 codes
// in 8-bit places times e4m3, float32 accumulate, one UE8M0 scale for the 32.
// KEEP 1 leaves A in the tensor core's buffer, for the next MMA with the same A,
// KEEP 2, which does not read it from shared memory again.
template <int KEEP>
__device__ __forceinline__ void umma_mxf8f6f4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                              uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                              uint32_t accumulate) {
#define FB_UMMA(collector)                                                                              \
  asm volatile(                                                                                         \
      "{\n\t.reg .pred p;\n\t"                                                                          \
      "setp.ne.b32 p, %6, 0;\n\t"                                                                       \
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X" collector                     \
      " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),                                           \
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                           \
      : "memory")
  if (KEEP == 0) FB_UMMA("");
  else if (KEEP == 1) FB_UMMA(".collector::a::fill");
  else FB_UMMA(".collector::a::lastuse");
#undef FB_UMMA
}
// Instruction descriptor of kind::mxf8f6f4: A e2m1 (5 in bits 7-9), B e4m3 (0 in
// bits 10-12), both K-major, N >> 3 in bits 17-22, UE8M0 scales (bit 23), M >> 7
// in bits 27-28; the scale byte a K-block takes from its 32-bit columns is in
// bits 4-5 for B and 29-30 for A.
__device__ __forceinline__ uint32_t mx_idesc(uint32_t n, uint32_t byte) {
  return (5u << 7) | ((n >> 3) << 17) | (1u << 23) | (1u << 27) | (byte << 4) | (byte << 29);
}

// A tile's step: its scales into tensor memory, then four K = 32 MMAs (eight where
// hi and lo go into the same columns, one after the other).  Descriptors count in
// 16 bytes: 32 columns are 2, 512 bytes of scales 32; `lo` is the distance of the
// lo part, `bs` the routes' scales.
template <bool SPLIT>
__device__ __forceinline__ void issue_step(uint32_t d, uint64_t a, uint64_t b, uint64_t lo, uint32_t sa,
                                           uint64_t as, uint64_t bs, uint32_t idesc, bool accumulate) {
  tmem_copy_scales(sa, as);
  tmem_copy_scales(sa + 4, bs);
  if (SPLIT) tmem_copy_scales(sa + 8, bs + 32);
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    const uint32_t id = idesc | (k << 4) | (k << 29);
    umma_mxf8f6f4<SPLIT ? 1 : 0>(d, a + 2 * k, b + 2 * k, id, sa, sa + 4, accumulate || k > 0 ? 1u : 0u);
    if (SPLIT) umma_mxf8f6f4<2>(d, a + 2 * k, b + lo + 2 * k, id, sa, sa + 8, 1u);
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

// The same through half precision, which holds a bf16 number times the power of two
// exactly down to 2^-17 and within 2^-25 below (the lo part's step is 2^-13): fewer
// conversions.
__device__ __forceinline__ void mx_split2_bf16(float a, float b, uint32_t* hi, uint32_t* lo) {
  const __half2 v = __floats2half2_rn(a, b);
  const __nv_fp8x2_storage_t h = __nv_cvt_halfraw2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
  const __half2 rest = __hsub2(v, __half2(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3)));
  *hi = h;
  *lo = __nv_cvt_halfraw2_to_fp8x2(__hmul2(rest, __float2half2_rn(16.0f)), __NV_SATFINITE, __NV_E4M3);
}

// A tile's four epilogue warps meet at their named barrier, and leave their loop
// together: every decision goes through a barrier that ANDs it.
__device__ __forceinline__ void mx_epilogue_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool mx_epilogue_all(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(v)), "r"(id)
      : "memory");
  return r != 0;
}

// The pool of shared memory, by the sub-groups' size: places of codes first, then
// places of routes (hi and lo parts of `cap` rows), a step each.  More places
// for codes where routes are few (memory-bound), as many of both where they
// are many.
__device__ __forceinline__ uint32_t mx_code_stages(int cap) { return cap <= 48 ? 5 : cap == 64 ? 4 : 3; }
__device__ __forceinline__ uint32_t mx_route_stages(int cap) { return cap <= 32 || cap == 64 ? 4 : 3; }

// Rows of routes that a sub-group's tile holds: the next multiple of 16.
__device__ __forceinline__ int mx_rows(int count) { return (count + 15) & ~15; }
// Hi and lo side by side in one MMA of twice the columns (added up in the
// epilogue), so that the weights are read once, as far as the accumulators have
// room; else one after the other into the same columns.
__device__ __forceinline__ bool mx_split(int rows) { return rows > 48; }

// Steps are numbered from 0 over all items of a CTA.  Step t uses barrier t % 8
// of each pipeline; a buffer of S places may be refilled for step t once step t
// - S is done, and S < 8 keeps the parity unambiguous.
__device__ __forceinline__ bool mx_wait_step(uint64_t* bars, uint32_t t, volatile int* abort_flag,
                                             int* err) {
  return mx_wait(bars + t % kBars, (t / kBars) & 1, abort_flag, err);
}

// Count one up, after everything the warp wrote before its last __syncwarp.
__device__ __forceinline__ void red_release_gpu(int* p) {
  asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(p) : "memory");
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
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) % 1024 != 0) {  // the swizzled tiles rely on it
    if (threadIdx.x == 0) atomicCAS(p.err, 0, DEV_LAYOUT_OVERFLOW);
    return;
  }
  uint8_t* scale = smem + kPoolBytes;  // [kPlaces] weights' scales, 16 bytes of 128 * kTiles rows
  uint8_t* rscale = scale + kPlaces * kTiles * kPieceBytes;  // [kPlaces] the same of the routes
  uint8_t* tiles = rscale + kPlaces * kPieceBytes;  // a step's arranged scales each
  uint8_t* xchg = tiles + kTilePool;
  uint64_t* full = reinterpret_cast<uint64_t*>(xchg + kTiles * kXchgBytes);
  uint64_t* done = full + kBars;     // the MMAs of a step are complete
  uint64_t* kfull = done + kBars;    // [kPlaces] a block's scales landed
  uint64_t* kempty = kfull + kPlaces;
  uint64_t* tfull = kempty + kPlaces;  // [tile][2] accumulators
  uint64_t* tempty = tfull + 2 * kTiles;
  uint64_t* ifull = tempty + 2 * kTiles;      // [kRing] claimed items
  uint64_t* iempty = ifull + kRing;
  uint64_t* drain = iempty + kRing;
  uint32_t* tmem_smem = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_smem + 1);
  MxItem* ring = reinterpret_cast<MxItem*>(drain + 2);  // [kRing]

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kBars; ++s) {
      mbar_init(&full[s], 3);  // codes, routes and scales
      mbar_init(&done[s], kTiles);
    }
    for (int s = 0; s < kPlaces; ++s) {
      mbar_init(&kfull[s], 34);  // both loaders' TMA, and the lanes' cp.async
      mbar_init(&kempty[s], 1);
    }
    for (int b = 0; b < 2 * kTiles; ++b) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], 4); }
    for (int q = 0; q < kRing; ++q) { mbar_init(&ifull[q], 1); mbar_init(&iempty[q], kItemReaders); }
    mbar_init(drain, kTiles);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(tmem_smem, kTmemCols); tmem_relinquish(); }
  if (warp == 0 && lane < 4) {
    tma_prefetch_desc(lane == 0 ? &maps.w1 : lane == 1 ? &maps.w2 : lane == 2 ? &maps.xs : &maps.as);
    tma_prefetch_desc(&maps.x[lane]);
    tma_prefetch_desc(&maps.a[lane]);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_smem;
  pdl_wait();  // what follows reads the prepare kernel's tables
  const int cap = p.header->cap;
  const uint32_t code_stages = mx_code_stages(cap), route_stages = mx_route_stages(cap);
  const uint32_t route_bytes = cap * kStepK * 2;
  uint8_t* const routes = smem + code_stages * kCodeBytes;
  // arranged, a step has 512 bytes of scales for each tile, 512 for the routes and,
  // where hi and lo are apart, 512 of lo scales
  const uint32_t tile_bytes = (kTiles + 1 + mx_split(cap)) * 512;
  const uint32_t n_tiles = min(kTilePool / tile_bytes, 6u);
  int q = 0;            // this role's place in the item ring
  uint32_t qphase = 0;

  if (warp == 0) {
    // ---------------- claims and codes ----------------
    if (elect_one()) {
      uint32_t t = 0, stage = 0;
      bool ok = true;
      const int first = atomicAdd(&p.header->queue, 1), n_groups = p.header->n_groups;
      auto publish = [&](const MxItem& it) {
        if (!mx_wait(&iempty[q], qphase ^ 1, abort_flag, p.err)) return false;
        ring[q] = it;
        mbar_arrive(&ifull[q]);
        if (++q == kRing) { q = 0; qphase ^= 1; }
        return true;
      };
      MxItem it = mx_item(p, n_groups, first);
      ok = publish(it);
      while (ok && it.phase != 0) {
        // the next item is claimed now and published a few loads on, before this
        // one's last: its scales and routes are under way in time
        const int id = atomicAdd(&p.header->queue, 1);
        MxItem next{};
        const int K = it.phase == 1 ? p.hidden : p.inter;
        const int steps = K / kStepK, ahead = min(steps - 1, 3);
        for (int kb = 0; kb < steps; ++kb, ++t) {
          if (t >= code_stages && !mx_wait_step(done, t - code_stages, abort_flag, p.err)) {
            ok = false;
            break;
          }
          uint64_t* bar = full + t % kBars;
          uint8_t* cs = smem + stage * kCodeBytes;
          mbar_expect_tx(bar, kCodeBytes / 2);  // the copy counts its 4-bit data, not the gaps
          if (it.phase == 1) tma_load_5d(cs, &maps.w1, bar, kb * kStepK, 0, 0, it.tile * 4 * kTiles, it.slot);
          else tma_load_3d(cs, &maps.w2, bar, kb * kStepK, it.tile * kMxM * kTiles, it.slot);
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
    // ---------------- weights' scales into shared memory ----------------
    uint32_t place = 0, ph = 0;
    bool ok = true;
    while (ok) {
      if (!mx_wait_warp(&ifull[q], qphase, abort_flag, p.err)) break;
      const int phase = ring[q].phase, tile = ring[q].tile, slot = ring[q].slot;
      __syncwarp();
      if (lane == 0) mbar_arrive(&iempty[q]);
      if (++q == kRing) { q = 0; qphase ^= 1; }
      if (phase == 0) break;
      const int K = phase == 1 ? p.hidden : p.inter;
      // 16 bytes (four steps) of each tile row: one TMA load where the rows are
      // 16-byte multiples (K a multiple of 512), else cp.async of 8 or 4 bytes, rows
      // lane + 32 * i (16 gate rows, 16 up rows, ...)
      const bool tma = (phase == 1 ? p.tma1 : p.tma2) != 0;
      const int pitch = K / 32;
      const int row = phase == 1 ? (lane < 16 ? 0 : p.inter) + tile * kMxFeatures * kTiles + (lane & 15)
                                 : tile * kMxM * kTiles + lane;
      const int parts = min(4 * kTiles, 4 * ((phase == 1 ? p.t1 : p.t2) - tile * kTiles));  // of 32 rows
      const uint8_t* src = p.scales + slot * p.row_bytes +
                           (phase == 1 ? 0 : 2 * static_cast<int64_t>(p.inter) * (p.hidden / 32)) +
                           static_cast<int64_t>(row) * pitch;
      const int64_t d1 = (phase == 1 ? 16 : 32) * pitch;
      for (int b = 0; b < pitch; b += 16) {
        if (!mx_wait_warp(&kempty[place], ph ^ 1, abort_flag, p.err)) { ok = false; break; }
        uint8_t* to = scale + place * kTiles * kPieceBytes;
        if (lane == 0) {
          mbar_expect_tx(&kfull[place], tma ? kTiles * kPieceBytes : 0);
          if (tma && phase == 1) tma_load_5d(to, &maps.s1, &kfull[place], b, 0, 0, tile * 4 * kTiles, slot);
          else if (tma) tma_load_3d(to, &maps.s2, &kfull[place], b, tile * kMxM * kTiles, slot);
        }
        __syncwarp();
        to += lane * 16;
        const uint8_t* from = src + b;
        if (!tma) {
          const int n = min(16, pitch - b);
          for (int c = 0; c < parts; ++c, to += 512, from += d1) {
            if (pitch % 8 == 0) {
              for (int i = 0; i < n; i += 8) cp_async<8>(to + i, from + i);
            } else {
              for (int i = 0; i < n; i += 4) cp_async<4>(to + i, from + i);
            }
          }
        }
        cp_async_arrive(&kfull[place]);
        if (++place == kPlaces) { place = 0; ph ^= 1; }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kRouteScale) {
    // ---------------- routes' scales into shared memory ----------------
    // Apart from the routes: a block's scales go through more hands than the
    // codes and routes of its steps, and start their way earlier.
    if (elect_one()) {
      uint32_t place = 0, ph = 0;
      bool ok = true;
      while (ok) {
        if (!mx_wait(&ifull[q], qphase, abort_flag, p.err)) break;
        const int phase = ring[q].phase, group = ring[q].group, start = ring[q].start;
        const int rows = mx_rows(ring[q].count);
        mbar_arrive(&iempty[q]);
        if (++q == kRing) { q = 0; qphase ^= 1; }
        if (phase == 0) break;
        if (phase == 2) {
          if (!mx_wait_dep(p.dep + group, 4 * p.t1, abort_flag, p.err)) break;
          asm volatile("fence.proxy.async.global;" ::: "memory");
        }
        const int pitch = (phase == 1 ? p.hidden : p.inter) / 32;
        const CUtensorMap* map = phase == 1 ? &maps.xs : &maps.as;
        for (int b = 0; b < pitch; b += 16) {
          if (!mx_wait(&kempty[place], ph ^ 1, abort_flag, p.err)) { ok = false; break; }
          mbar_expect_tx(&kfull[place], rows * 16);
          for (int i = 0; i < rows; i += 16)
            tma_load_2d(rscale + place * kPieceBytes + i * 16, map, &kfull[place], b, start + i);
          if (++place == kPlaces) { place = 0; ph ^= 1; }
        }
      }
    }
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
          if (!mx_wait_dep(p.dep + it.group, 4 * p.t1, abort_flag, p.err)) { ok = false; break; }
          asm volatile("fence.proxy.async.global;" ::: "memory");
        }
        const int steps = (it.phase == 1 ? p.hidden : p.inter) / kStepK;
        const int rows = mx_rows(it.count), cls = rows / 16 - 1;
        const CUtensorMap* map = it.phase == 1 ? &maps.x[cls] : &maps.a[cls];
        for (int kb = 0; kb < steps; ++kb, ++t) {
          if (t >= route_stages && !mx_wait_step(done, t - route_stages, abort_flag, p.err)) {
            ok = false;
            break;
          }
          uint64_t* bar = full + t % kBars;
          mbar_expect_tx(bar, rows * kStepK * 2);
          // the rows' hi parts, then their lo parts
          tma_load_3d(routes + stage * route_bytes, map, bar, kb * kStepK, it.start, 0);
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
    uint32_t t = 0, turn = 0, tile = 0, ph = 0;  // steps and blocks of all items
    bool ok = true;
    while (ok) {
      if (!mx_wait_warp(&ifull[q], qphase, abort_flag, p.err)) break;
      const int phase = ring[q].phase, rows = mx_rows(ring[q].count);
      const bool split = mx_split(rows);
      __syncwarp();
      if (lane == 0) mbar_arrive(&iempty[q]);
      if (++q == kRing) { q = 0; qphase ^= 1; }
      if (phase == 0) break;
      const int steps = (phase == 1 ? p.hidden : p.inter) / kStepK;
      for (int k = 0; k < steps && ok; k += kBlock, turn ^= 1) {
        const int n = min(kBlock, steps - k);
        if (turn != me) {
          t += n;
          tile = tile + n >= n_tiles ? tile + n - n_tiles : tile + n;
          continue;
        }
        if (!mx_wait_warp(&kfull[me], ph, abort_flag, p.err)) { ok = false; break; }
        ph ^= 1;
        // four steps of weight rows lane + 32 * c, and of routes
        const uint4* rs = reinterpret_cast<const uint4*>(rscale + me * kPieceBytes);
        const uint4* ws = reinterpret_cast<const uint4*>(scale + me * kTiles * kPieceBytes);
        uint4 b4[4], a4[kTiles][4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int i = 0; i < kTiles; ++i) a4[i][c] = ws[i * 128 + lane + 32 * c];
          // columns of the MMA: the rows' hi parts and, side by side, their lo parts
          const int r = lane + 32 * c;
          b4[c] = make_uint4(0, 0, 0, 0);
          if (r < rows) b4[c] = rs[r];
          else if (!split && r < 2 * rows) b4[c] = rs[r - rows];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&kempty[me]);
#pragma unroll
        for (int i = 0; i < kBlock; ++i) {
          if (i < n && ok) {
            auto part = [&](const uint4& v) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; };
            // the lo scales are 2^-4 of the hi ones (every byte is at least 4)
            constexpr uint32_t kLo = 0x04040404u;
            uint4 b = make_uint4(part(b4[0]), part(b4[1]), part(b4[2]), part(b4[3]));
            const uint4 low = make_uint4(b.x - kLo, b.y - kLo, b.z - kLo, b.w - kLo);
            if (!split) {
              if (lane >= rows) b.x = low.x;
              if (lane + 32 >= rows) b.y = low.y;
              if (lane + 64 >= rows) b.z = low.z;
              if (lane + 96 >= rows) b.w = low.w;
            }
            // the tile's last user is done
            if (t >= n_tiles &&
                !__all_sync(0xffffffffu, mx_wait_step(done, t - n_tiles, abort_flag, p.err))) {
              ok = false;
            } else {
              uint4* to = reinterpret_cast<uint4*>(tiles + tile * tile_bytes) + lane;
#pragma unroll
              for (int u = 0; u < kTiles; ++u)
                to[32 * u] = make_uint4(part(a4[u][0]), part(a4[u][1]), part(a4[u][2]), part(a4[u][3]));
              to[32 * kTiles] = b;
              if (split) to[32 * kTiles + 32] = low;
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) mbar_arrive(&full[t % kBars]);
              ++t;
              if (++tile == n_tiles) tile = 0;
            }
          }
        }
      }
    }
  } else if (warp < kFirstEpi) {
    // ---------------- MMA ----------------
    // One warp for each tile: the thread that waits, issues and commits would
    // bound a step that had both.
    if (elect_one()) {
      const uint32_t part = warp - 1;
      uint32_t t = 0, cstage = 0, rstage = 0, tile = 0;
      const uint64_t a0 = smem_desc_sw128(smem_u32(smem + part * kTileCodes)), b0 = smem_desc_sw128(smem_u32(routes));
      const uint64_t s0 = smem_desc_scales(smem_u32(tiles));
      const bool apart = mx_split(cap);
      uint32_t acc = 0, acc_phase = 0;
      tfull += 2 * part;
      tempty += 2 * part;
      bool ok = true;
      while (ok) {
        if (!mx_wait(&ifull[q], qphase, abort_flag, p.err)) break;
        const int kind = ring[q].phase;
        const uint32_t rows = mx_rows(ring[q].count);
        mbar_arrive(&iempty[q]);
        if (++q == kRing) { q = 0; qphase ^= 1; }
        if (kind == 0) break;
        const bool split = mx_split(rows);
        const uint32_t idesc = mx_idesc(split ? rows : 2 * rows, 0);
        const int steps = (kind == 1 ? p.hidden : p.inter) / kStepK;
        if (!mx_wait(&tempty[acc], acc_phase ^ 1, abort_flag, p.err)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * kAccCols + part * kTileCols;
        for (int kb = 0; kb < steps; ++kb, ++t) {
          if (!mx_wait_step(full, t, abort_flag, p.err)) { ok = false; break; }
          tc_fence_after();
          const uint64_t a = a0 + cstage * (kCodeBytes >> 4), b = b0 + rstage * (route_bytes >> 4);
          const uint32_t sa = tmem + kTmemScale + (apart ? (t & 1) * 24 + part * 12 : (t & 3) * 16 + part * 8);
          const uint64_t from = s0 + tile * (tile_bytes >> 4);
          if (split) issue_step<true>(d, a, b, rows * 8, sa, from + part * 32, from + kTiles * 32, idesc, kb > 0);
          else issue_step<false>(d, a, b, 0, sa, from + part * 32, from + kTiles * 32, idesc, kb > 0);
          umma_commit(&done[t % kBars]);
          if (++cstage == code_stages) cstage = 0;
          if (++rstage == route_stages) rstage = 0;
          if (++tile == n_tiles) tile = 0;
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
    // ---------------- epilogue (four warps for each tile) ----------------
    // TMEM lanes 32 * (warp % 4)..: 16 gate rows of a phase-1 tile and the 16 up
    // rows of the same features, or 32 down rows
    const int qd = warp & 3, part = (warp - kFirstEpi) / 4, bar = 1 + part;
    tfull += 2 * part;
    tempty += 2 * part;
    xchg += part * kXchgBytes;
    const bool low = lane < 16;
    uint32_t turn = 0;
    uint32_t acc = 0, acc_phase = 0;
    for (;;) {
      if (!mx_epilogue_all(bar, mx_wait(&ifull[q], qphase, abort_flag, p.err))) break;
      const MxItem it = ring[q];
      __syncwarp();
      if (lane == 0) mbar_arrive(&iempty[q]);
      if (++q == kRing) { q = 0; qphase ^= 1; }
      if (it.phase == 0) break;  // the same entry for all four warps
      const int tile = it.tile * kTiles + part;
      const bool mine = tile < (it.phase == 1 ? p.t1 : p.t2);  // the last item may lack a tile
      // routing weights of routes lane, lane + 32, ..., with which the activations
      // are multiplied before they are rounded
      float w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        w[c] = it.bad ? __uint_as_float(0x7fc00000u)
               : it.phase == 1 && lane + 32 * c < it.count ? p.route_w[it.start + lane + 32 * c] : 0.0f;
      if (!mx_epilogue_all(bar, mx_wait(&tfull[acc], acc_phase, abort_flag, p.err))) break;
      tc_fence_after();
      const uint32_t d = tmem + (static_cast<uint32_t>(qd * 32) << 16) + acc * kAccCols + part * kTileCols;
      // 16 columns from c0 on: the hi part's sums, plus the lo part's where they
      // have columns of their own
      const int lo_at = mx_split(mx_rows(it.count)) ? 0 : mx_rows(it.count);
      auto columns = [&](int c0, float* v) {
        tmem_ld16_start(d + c0, v);
        if (lo_at) {
          float more[16];
          tmem_ld16_start(d + lo_at + c0, more);
          tmem_ld_wait(more);
          tmem_ld_wait(v);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] += more[j];
        } else {
          tmem_ld_wait(v);
        }
      };
      if (!mine) {
      } else if (it.phase == 1) {
        // 16 routes at a time, in pairs: a feature's gate lane takes the even one, its
        // up lane the odd one, each handing the other the value it needs: eight
        // activations of one feature a lane.
        const int f = lane & 15, odd = lane >> 4;
        // byte selectors of the 4 x 4 transposes below
        const uint32_t swap1 = f & 1 ? 0x3715u : 0x6240u, swap2 = f & 2 ? 0x3276u : 0x5410u;
        uint8_t* const to = p.act + (static_cast<int64_t>(it.start) + 2 * (f & 3) + odd) * (2 * p.inter) +
                            tile * kMxFeatures + qd * 16 + (f & ~3);
        uint8_t* const sb = p.as + (static_cast<int64_t>(it.start) + 2 * (f & 7) + odd) * p.pitch2 + tile * 2 + (qd >> 1);
        for (int c0 = 0; c0 < it.count; c0 += 16, turn ^= 1) {
          float v[16], a[8];
          uint32_t m[4], hi[2], lo[2];
          columns(c0, v);
          const float ws = c0 < 32 ? w[0] : c0 < 64 ? w[1] : c0 < 96 ? w[2] : w[3];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float own = low ? v[2 * j] : v[2 * j + 1];
            const float other = __shfl_xor_sync(0xffffffffu, low ? v[2 * j + 1] : v[2 * j], 16);
            const float gate = low ? own : other, up = low ? other : own;
            a[j] = __fdividef(gate, 1.0f + __expf(-gate)) * up *
                   __shfl_sync(0xffffffffu, ws, (c0 & 16) + 2 * j + odd);
          }
          // The scale of 32 features is two warps'.  Largest magnitudes (their upper 16
          // bits, two routes a register) of the warp's 16 features: a butterfly in which
          // a lane keeps two registers, then one; then exchanged with the other warp, by
          // turns in two places, so that one barrier does.
#pragma unroll
          for (int i = 0; i < 4; ++i)
            m[i] = __byte_perm(__float_as_uint(a[2 * i]), __float_as_uint(a[2 * i + 1]), 0x7632) & 0x7fff7fffu;
          const bool b0 = f & 1, b1 = f & 2;
          uint32_t k0 = __vmaxu2(b0 ? m[2] : m[0], __shfl_xor_sync(0xffffffffu, b0 ? m[0] : m[2], 1));
          const uint32_t k1 = __vmaxu2(b0 ? m[3] : m[1], __shfl_xor_sync(0xffffffffu, b0 ? m[1] : m[3], 1));
          k0 = __vmaxu2(b1 ? k1 : k0, __shfl_xor_sync(0xffffffffu, b1 ? k0 : k1, 2));
          k0 = __vmaxu2(k0, __shfl_xor_sync(0xffffffffu, k0, 4));
          k0 = __vmaxu2(k0, __shfl_xor_sync(0xffffffffu, k0, 8));
          uint8_t* ex = xchg + turn * (4 * 32) + odd * 16;  // [warp][odd][route] of 16 bits
          if (f < 4) *reinterpret_cast<uint32_t*>(ex + qd * 32 + ((f & 1) * 2 + (f >> 1)) * 4) = k0;
          mx_epilogue_sync(bar);
          const uint4 e0 = *reinterpret_cast<const uint4*>(ex + qd * 32);
          const uint4 e1 = *reinterpret_cast<const uint4*>(ex + (qd ^ 1) * 32);
          m[0] = __vmaxu2(e0.x, e1.x);
          m[1] = __vmaxu2(e0.y, e1.y);
          m[2] = __vmaxu2(e0.z, e1.z);
          m[3] = __vmaxu2(e0.w, e1.w);
          // times 2^(127 - byte), byte = max(exponent field - 7, 4); what a block that is
          // not finite (byte 255) holds does not matter
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t z = __vminu2(0x01050105u - ((m[i] >> 7) & 0x00ff00ffu), 0x00fa00fau);
            uint32_t h, l;
            mx_split2(a[2 * i] * __uint_as_float(z << 23), a[2 * i + 1] * __uint_as_float((z & 0x00ff0000u) << 7),
                      &h, &l);
            hi[i / 2] = i & 1 ? hi[i / 2] | h << 16 : h;
            lo[i / 2] = i & 1 ? lo[i / 2] | l << 16 : l;
          }
          // four routes of one feature -> four features of one route
          auto transpose = [&](uint32_t x) {
            x = __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 1), swap1);
            return __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 2), swap2);
          };
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            hi[i] = transpose(hi[i]);
            lo[i] = transpose(lo[i]);
            if (c0 + 8 * i + 2 * (f & 3) + odd < it.count) {
              uint8_t* at = to + static_cast<int64_t>(c0 + 8 * i) * (2 * p.inter);
              *reinterpret_cast<uint32_t*>(at) = hi[i];
              *reinterpret_cast<uint32_t*>(at + p.inter) = lo[i];
            }
          }
          if ((qd & 1) == 0 && f < 8 && c0 + 2 * f + odd < it.count) {
            const uint32_t top = max(*reinterpret_cast<const uint16_t*>(ex + qd * 32 + f * 2),
                                     *reinterpret_cast<const uint16_t*>(ex + (qd ^ 1) * 32 + f * 2));
            sb[static_cast<int64_t>(c0) * p.pitch2] = static_cast<uint8_t>(mx_block_byte(top >> 7));
          }
        }
      } else {
        // 16 routes at a time, in pairs: an even lane takes the first one's two
        // neighbouring features, an odd lane the second one's
        const bool odd = lane & 1;
        __nv_bfloat16* to = p.out + static_cast<int64_t>(it.start + odd) * p.hidden + tile * kMxM + qd * 32 + (lane & ~1);
        for (int c0 = 0; c0 < it.count; c0 += 16) {
          float v[16];
          columns(c0, v);
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
            const __nv_bfloat162 y = odd ? __floats2bfloat162_rn(other, v[j + 1]) : __floats2bfloat162_rn(v[j], other);
            if (c0 + j + odd < it.count) *reinterpret_cast<__nv_bfloat162*>(to) = y;
            to += 2 * p.hidden;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      if (it.phase == 1 && mine) {
        // publish this warp's activations to the sub-group's phase-2 items
        __syncwarp();
        if (lane == 0) red_release_gpu(p.dep + it.group);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
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
  int sort_from;  // active groups from which sub-groups are ordered by size
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
  // First wait for what the stream ran before, then let the GEMM's CTAs set up and wait:
  // they fill the SMs, and must not while an earlier kernel may need another stream's.
  pdl_wait();
  pdl_launch_dependents();
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
      if (threadIdx.x == 0) { a.header->n_groups = 0; a.header->cap = 16; atomicCAS(a.err, 0, DEV_BAD_INPUT); }
      return;
    }
    atomicAdd(&base, active);
    __syncthreads();
    active = base;
    __syncthreads();
    if (threadIdx.x == 0) base = 0;
    // sub-groups no wider than the mean group asks for: narrow ones leave shared memory
    // to more loads under way, wide ones read the weights less often (128 experts of
    // 2048 x 768, routes of a group in the mean: 16: 32 at most 36.2 us, 48 36.0, 112
    // 40.2; 24: 50.2, 47.7, 53.2; 43: 72.9, 65.0, 65.9 and 64 63.4; 55: 87.2, 77.9, 74.1
    // and 64 73.8; groups of uneven sizes, 3: 16 49.9, 32 49.7, 112 60.4; 7: 64.6, 64.1,
    // 76.9).  Of 64 experts of 2048 x 1408 and 16 of 4096 x 1792 the rule is within 3 % of
    // the best width for means of 1 to 128, of 64 of 512 x 512 within 5 % but for means
    // of 3 and 80 (18.7 against 16.2, 32.9 against 30.1).  Experts of a step or two of K
    // would take narrower ones, their items being latency: 128 of 512 x 128 at 24 19.5
    // against 16.7 with 32, 32 of 256 x 128 at 56 15.6 against 13.4 with 16.
    const int64_t all = a.starts[a.n_groups] - a.starts[0];
    const int64_t mean = active ? (all + active - 1) / active : 0;
    const int cap = mean <= 4 ? 16 : mean <= 16 ? 32 : mean <= 32 ? 48 : mean <= 56 ? 64 : 112;
    __syncthreads();
    // Sub-groups in descending order of their rows, so that the long epilogues of the
    // first product are over early and the work left at the end comes in small items:
    // a pass over the groups for each number of rows (up to 256 groups stay in
    // registers).  Not where every CTA has an item or two at most: there the passes are
    // what a call waits for (32 experts of 256 x 128: 12.0 -> 12.8 us).
    int s0 = 0, count = 0, slot = 0;
    bool bad = false;
    auto read = [&](int g) {
      s0 = count = slot = 0;
      bad = false;
      if (g >= a.n_groups) return;
      s0 = static_cast<int>(a.starts[g]);
      count = static_cast<int>(a.starts[g + 1]) - s0;
      const int64_t wanted = a.slots[g];
      bad = count > 0 && (wanted < 0 || wanted >= a.cache_slots);
      if (bad) atomicCAS(a.err, 0, DEV_BAD_INPUT);
      else slot = static_cast<int>(wanted);
    };
    read(threadIdx.x);
    const bool by_size = active >= a.sort_from;
    for (int rows = by_size ? cap : 16; rows > 0; rows -= 16) {
      for (int g0 = 0; g0 < a.n_groups; g0 += kPrepThreads) {
        if (a.n_groups > kPrepThreads) read(g0 + threadIdx.x);
        int n = (count + cap - 1) / cap;
        if (by_size && n > 0 && mx_rows((count + n - 1) / n) != rows) n = 0;
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
          a.groups[at + i] = MxGroup{slot, r, len, bad ? 1 : 0};
          a.dep[at + i] = 0;
          r += len;
        }
        __syncthreads();
        if (threadIdx.x == kPrepThreads - 1) base = before + scan;
        __syncthreads();
      }
    }
    if (threadIdx.x == 0) {
      a.header->n_groups = base;
      a.header->cap = cap;
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
    uint4* to = reinterpret_cast<uint4*>(a.x + i * 2 * a.hidden);
    uint8_t* sb = a.xs + i * a.pitch1;
    // 16 values a lane, a block of 32 in two neighbours (hidden is a multiple of 128:
    // whole blocks, and the lanes of a block are all in or all out); eight loads in flight
    const int n16 = a.hidden / 16;
    for (int v0 = 0; v0 < n16; v0 += 4 * 32) {
      uint4 e[4][2];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int v = v0 + u * 32 + lane;
        e[u][0] = e[u][1] = make_uint4(0, 0, 0, 0);
        if (good && v < n16) {
          e[u][0] = from[2 * v];
          e[u][1] = from[2 * v + 1];
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int v = v0 + u * 32 + lane;
        const uint32_t in[8] = {e[u][0].x, e[u][0].y, e[u][0].z, e[u][0].w, e[u][1].x, e[u][1].y, e[u][1].z, e[u][1].w};
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = __vmaxu2(m, in[j] & 0x7fff7fffu);
        uint32_t top = max(m & 0xffffu, m >> 16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        const int byte = mx_block_byte(top >> 7);
        const float mult = mx_block_mult(byte);
        uint32_t h[8], l[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          mx_split2_bf16(__uint_as_float(in[j] << 16) * mult, __uint_as_float(in[j] & 0xffff0000u) * mult, &h[j],
                         &l[j]);
        if (v < n16) {
          to[v] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
          to[n16 + v] = make_uint4(l[0] | l[1] << 16, l[2] | l[3] << 16, l[4] | l[5] << 16, l[6] | l[7] << 16);
          if ((v & 1) == 0) sb[v >> 1] = static_cast<uint8_t>(byte);
        }
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
// to 16 bytes of shared memory, 8 of them data).  One load brings a step's tile:
// four times 16 gate rows and their 16 up rows, or 128 down rows; for routes the
// hi parts, then the lo parts.
static int make_maps(MxMaps* m, const ferryb_mxfp4_experts_args* e, const uint8_t* x, const uint8_t* act,
                     const uint8_t* xs, const uint8_t* as, int64_t pitch1, int64_t pitch2) {
  const cuuint64_t H = e->hidden, I = e->intermediate, slots = e->cache_slots, routes = e->routes;
  const cuuint64_t row_bytes = 3 * H * I / 32 * 17;
  const uint8_t* cache = static_cast<const uint8_t*>(e->cache);
  constexpr auto k4 = CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B;
  constexpr auto k8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int s;
  {
    const cuuint64_t dims[5] = {H, 16, 2, I / 16, slots};
    const cuuint64_t strides[4] = {H / 2, I * H / 2, 16 * H / 2, row_bytes};
    const cuuint32_t box[5] = {kStepK, 16, 2, kTiles * kMxFeatures / 16, 1};
    if ((s = make_map(&m->w1, k4, 5, cache, dims, strides, box, true))) return s;
  }
  {
    const cuuint64_t dims[3] = {I, H, slots};
    const cuuint64_t strides[2] = {I / 2, row_bytes};
    const cuuint32_t box[3] = {kStepK, kTiles * kMxM, 1};
    if ((s = make_map(&m->w2, k4, 3, cache + H * I, dims, strides, box, true))) return s;
  }
  // weight scales of rows that are 16-byte multiples (the strides' unit)
  const uint8_t* scales = cache + 3 * H * I / 2;
  if (H % 512 == 0) {
    const cuuint64_t dims[5] = {H / 32, 16, 2, I / 16, slots};
    const cuuint64_t strides[4] = {H / 32, I * (H / 32), 16 * (H / 32), row_bytes};
    const cuuint32_t box[5] = {16, 16, 2, kTiles * kMxFeatures / 16, 1};
    if ((s = make_map(&m->s1, k8, 5, scales, dims, strides, box, false))) return s;
  }
  if (I % 512 == 0) {
    const cuuint64_t dims[3] = {I / 32, H, slots};
    const cuuint64_t strides[2] = {I / 32, row_bytes};
    const cuuint32_t box[3] = {16, kTiles * kMxM, 1};
    if ((s = make_map(&m->s2, k8, 3, scales + 2 * I * (H / 32), dims, strides, box, false))) return s;
  }
  for (unsigned c = 0; c < 7; ++c) {
    const cuuint32_t box[3] = {kStepK, 16 * (c + 1), 2};
    for (int phase = 0; phase < 2; ++phase) {
      const cuuint64_t K = phase ? I : H;
      const cuuint64_t dims[3] = {K, routes, 2};
      const cuuint64_t strides[2] = {2 * K, K};
      if ((s = make_map(phase ? &m->a[c] : &m->x[c], k8, 3, phase ? act : x, dims, strides, box, true)))
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

static int launch_experts(const MxMaps& maps, const MxParams& p, const ferryb_mxfp4_experts_args* e, int device,
                          cudaStream_t stream) {
  static std::atomic<bool> attr_set[64];
  if (device >= 64 || !attr_set[device].load(std::memory_order_acquire)) {
    FB_CUDA(cudaFuncSetAttribute(mxfp4_swiglu_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)kMxSmem));
    if (device < 64) attr_set[device].store(true, std::memory_order_release);
  }
  const int64_t subs = e->n_groups < e->routes ? e->n_groups + e->routes / 16 : e->routes;
  const int64_t items = subs * (p.mt1 + p.mt2), most = num_sms(device);
  // the CTAs set up while the routes are prepared
  return launch_behind(mxfp4_swiglu_kernel, static_cast<unsigned>(items < most ? items : most), kMxThreads, kMxSmem,
                       stream, maps, p);
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
  // the epilogue stores pairs of bf16
  FB_CHECK_ARG(reinterpret_cast<uintptr_t>(e->out) % 4 == 0, "execute_experts_mxfp4: out must be 4-byte aligned");
  FB_CHECK_ARG((reinterpret_cast<uintptr_t>(e->slots) | reinterpret_cast<uintptr_t>(e->starts) |
                reinterpret_cast<uintptr_t>(e->rows) | reinterpret_cast<uintptr_t>(e->cols)) % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(e->err) % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(e->routing_weights) % (e->weights_type == FERRYB_FP32 ? 4 : 2) == 0,
               "execute_experts_mxfp4: slots, starts, rows, cols, err and routing_weights must be aligned to "
               "their elements");
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
  p.t1 = static_cast<int>(e->intermediate / kMxFeatures);
  p.t2 = static_cast<int>(e->hidden / kMxM);
  p.mt1 = (p.t1 + kTiles - 1) / kTiles;
  p.mt2 = (p.t2 + kTiles - 1) / kTiles;
  pr.sort_from = 2 * sms / (p.mt1 + p.mt2) + 1;
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
  if ((s = launch_behind(mxfp4_prepare_kernel, 1 + static_cast<unsigned>(gather < most ? gather : most),
                         kPrepThreads, 0, stream, pr)))
    return s;
  return launch_experts(maps, p, e, device, stream);
}
