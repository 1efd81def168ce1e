// experts_mxfp4.cu -- routed-expert SwiGLU over MXFP4 expert rows: a grouped
// GEMM on the 5th-generation tensor cores whose weight operand is expanded from
// 4 bits on its way into tensor memory.
//
// The operator beside execute_experts (ferry/csrc/expert_ops.cpp:16-45): per
// group of routes, y = (silu(x Wg^T) * (x Wu^T)) Wd^T * w with W = code *
// 2^(scale - 127).  Every such weight is a bf16 number, so the products are the
// exact ones of bf16 operands; sums, gate, up and silu stay in float32, and two
// roundings to bf16 remain: the activation (it is the second product's tensor-
// core operand) and the result.
//
// Data layout.  A cache row is [gate I x H | up I x H | down H x I] codes, two
// a byte, then their scale bytes in the same order, one for 32 codes.  Groups
// of more than 128 routes are split into sub-groups of nearly equal size, each
// with its own work items, so that a popular expert is spread over the GPU.
//
// Orientation as in experts.cu: 128 weight rows are the MMA's M side (64 gate
// rows above the 64 up rows of the same features, or 128 down rows), the routes
// its N side.  The weight operand comes from tensor memory (tcgen05.mma takes A
// from there): a thread expands one row's codes in registers and stores them
// with tcgen05.st, so expanded weights touch neither shared memory nor a
// swizzle, and shared memory carries codes and routes only.
//
// Expansion.  Of a 32-bit word of 8 codes, shifts and masks put code j into the
// sign, the two low exponent bits and the top mantissa bit of a bf16, and code
// j + 4 into the upper half: as a bf16 that pattern is the e2m1 value times
// 2^-126 (subnormals included), and one bf16x2 multiply by 2^(scale - 1) makes
// both weights exactly.  The order (0 4 1 5 2 6 3 7) of every 8 columns is met
// by storing the routes' columns in the same order.
//
// CTA roles (480 threads): warp 0 claims work and loads codes (TMA) and scales
// (cp.async, whose 4-byte pieces need no padding of the scale rows); warp 14
// loads the routes (TMA); warps 6-13 expand, four on even and four on odd
// k-steps (warp w owns TMEM lanes 32 * (w % 4)..+31); warp 1 issues the MMAs;
// warps 2-5 drain the accumulators.  Codes do not depend on phase 1, so warp 0
// runs ahead into phase 2 while warp 14 waits for the activations.
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "experts.cuh"

namespace ferryb {

constexpr int kMxWarps = 15;
constexpr int kMxThreadsG = kMxWarps * 32;
constexpr int kMxM = 128;          // weight rows per tile
constexpr int kMxN = 128;          // routes per sub-group
constexpr int kMxStepK = 64;       // columns per MMA step (one swizzled 128-byte row of routes)
constexpr int kMxChunkK = 256;     // columns per code stage (128 bytes of codes a row)
constexpr int kMxFeatures = 64;    // gate (= up) rows per phase-1 tile
constexpr int kCodeStages = 4;
constexpr int kSteps = 8;          // route stages = expanded-weight stages
constexpr uint32_t kCodeBytes = kMxM * 128;
constexpr uint32_t kScaleBytes = kMxM * 8;
constexpr uint32_t kRouteBytes = kMxN * kMxStepK * 2;
constexpr uint32_t kTmemW = 256;   // first TMEM column of the expanded weights
constexpr int kRing = 4;           // claimed items in flight
constexpr int kXStride = 17;       // floats a feature of the gate/up exchange (padded)
constexpr uint32_t kXchgBytes = 2 * kMxFeatures * kXStride * 4;
constexpr uint32_t kMxSmem = kCodeStages * (kCodeBytes + kScaleBytes) + kSteps * kRouteBytes +
                             kXchgBytes + 512 + 1024;
constexpr uint64_t kMxWaitNs = 2000000000ull;  // bound on any wait

// Up to 128 routes of one group.
struct MxGroup {
  int32_t slot;   // cache slot (0 where the caller's is out of range)
  int32_t start;  // first route
  int32_t count;  // routes
  int32_t bad;    // slot out of range: the routes' outputs are NaN
};

struct MxParams {
  const MxGroup* groups;
  const int* n_groups;  // [1] sub-groups, written by the prepare kernel
  int mt1, mt2;         // items per sub-group: I / 64 phase 1, H / 128 phase 2
  int hidden, inter;
  const uint8_t* scales;  // slot 0's scale bytes
  int64_t row_bytes;      // bytes of a cache row
  __nv_bfloat16* act;
  __nv_bfloat16* out;
  const float* route_w;
  int* queue;  // [1] claim counter, zero at launch
  int* dep;    // [sub-groups] phase-1 epilogue-warp completions, zero at launch
  int* err;
};

struct MxItem {
  int phase, group, tile;
};

__device__ __forceinline__ MxItem mx_item(const MxParams& p, int n_groups, int item) {
  MxItem it;
  const int n1 = n_groups * p.mt1;
  if (item < n1) {
    it.phase = 1; it.group = item / p.mt1; it.tile = item - it.group * p.mt1;
  } else {
    const int i = item - n1;
    it.phase = 2; it.group = i / p.mt2; it.tile = i - it.group * p.mt2;
  }
  return it;
}

// Wait for an mbarrier phase, bounded in time; on time-out the CTA's abort flag
// and the error word are set.
__device__ __forceinline__ bool mx_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                        int* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255) == 0) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > kMxWaitNs) {
        *abort_flag = 1;
        atomicCAS(err, 0, DEV_WAIT_TIMEOUT);
        return false;
      }
    }
  }
}
// The same for a whole warp: all lanes agree on the outcome.
__device__ __forceinline__ bool mx_wait_warp(uint64_t* bar, uint32_t parity,
                                             volatile int* abort_flag, int* err) {
  return __all_sync(0xffffffffu, mx_wait(bar, parity, abort_flag, err));
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Arrive on `bar` once this thread's cp.async copies so far have landed (the
// barrier's count includes this arrival).
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// 32 lanes x 32 columns of 32 bits into tensor memory.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// D[tmem] (+)= A[tmem] x B[smem]^T, bf16 inputs, float32 accumulate.
__device__ __forceinline__ void umma_bf16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// 8 codes of a word -> 4 x bf16x2 (codes j and j + 4) times 2^-126.
__device__ __forceinline__ void spread8(uint32_t w, uint32_t* o) {
  constexpr uint32_t kMag = 0x01C001C0u, kSign = 0x80008000u;
  o[0] = ((w << 6) & kMag) | ((w << 12) & kSign);
  o[1] = ((w << 2) & kMag) | ((w << 8) & kSign);
  o[2] = ((w >> 2) & kMag) | ((w << 4) & kSign);
  o[3] = ((w >> 6) & kMag) | (w & kSign);
}

// 32 codes and their scale byte -> 16 x bf16x2.  2^(s - 127) * 2^126 is a bf16
// up to s = 128 (blocks whose largest value is below 16); beyond, the factor is
// applied in two steps.  s = 255 stands for NaN.
__device__ __forceinline__ void expand32(const uint4& c, uint32_t s, uint32_t* o) {
  const uint32_t m = min(s + 126u, 254u) * 0x00800080u;
  spread8(c.x, o);
  spread8(c.y, o + 4);
  spread8(c.z, o + 8);
  spread8(c.w, o + 12);
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = mul_bf16x2(o[i], m);
  if (s > 128u) {
    const uint32_t m2 = s == 255u ? 0x7FC07FC0u : (s - 1u) * 0x00800080u;
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = mul_bf16x2(o[i], m2);
  }
}

__device__ __forceinline__ void mx_epilogue_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// The four epilogue warps leave their loop together: every decision goes
// through a barrier that ANDs it.
__device__ __forceinline__ bool mx_epilogue_all(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(v))
      : "memory");
  return r != 0;
}

__device__ __forceinline__ int mx_box(int n) { return n <= 16 ? 0 : n <= 32 ? 1 : n <= 64 ? 2 : 3; }

// Column of feature f in the stored order of every 8 columns.
__device__ __forceinline__ int mx_column(int f) {
  const int e = f & 7;
  return (f & ~7) | (e < 4 ? 2 * e : 2 * e - 7);
}

__global__ void __launch_bounds__(kMxThreadsG, 1)
    mxfp4_swiglu_kernel(const __grid_constant__ CUtensorMap w1, const __grid_constant__ CUtensorMap w2,
                        const __grid_constant__ BMaps bx, const __grid_constant__ BMaps ba,
                        const MxParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* codes = smem;
  uint8_t* routes = codes + kCodeStages * kCodeBytes;
  uint8_t* scale = routes + kSteps * kRouteBytes;
  float* xchg = reinterpret_cast<float*>(scale + kCodeStages * kScaleBytes);
  uint64_t* cfull = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(xchg) + kXchgBytes);
  uint64_t* cempty = cfull + kCodeStages;
  uint64_t* rfull = cempty + kCodeStages;  // routes landed
  uint64_t* wfull = rfull + kSteps;        // weights expanded
  uint64_t* sempty = wfull + kSteps;       // step consumed by the MMA
  uint64_t* tfull = sempty + kSteps;       // [2] accumulators
  uint64_t* tempty = tfull + 2;
  uint64_t* ifull = tempty + 2;            // [kRing] claimed items
  uint64_t* iempty = ifull + kRing;
  uint64_t* drain = iempty + kRing;
  int* ring = reinterpret_cast<int*>(drain + 1);
  uint32_t* tmem_smem = reinterpret_cast<uint32_t*>(ring + kRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_smem + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kCodeStages; ++s) { mbar_init(&cfull[s], 33); mbar_init(&cempty[s], 8); }
    for (int s = 0; s < kSteps; ++s) {
      mbar_init(&rfull[s], 1);
      mbar_init(&wfull[s], 4);
      mbar_init(&sempty[s], 1);
    }
    for (int b = 0; b < 2; ++b) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], 4); }
    for (int q = 0; q < kRing; ++q) { mbar_init(&ifull[q], 1); mbar_init(&iempty[q], 14); }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(tmem_smem, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_smem;
  const int n_groups = *p.n_groups;
  const int n_items = n_groups * (p.mt1 + p.mt2);
  int q = 0;            // this role's place in the item ring
  uint32_t qphase = 0;

  if (warp == 0) {
    // ---------------- claims, codes and scales ----------------
    int stage = 0;
    uint32_t phase = 0, pending = 0, pend_parity = 0;
    bool ok = true;
    while (ok) {
      if (!mx_wait_warp(&iempty[q], qphase ^ 1, abort_flag, p.err)) { ok = false; break; }
      int item = 0;
      if (lane == 0) {
        item = atomicAdd(p.queue, 1);
        if (item >= n_items || *abort_flag) item = -1;
        ring[q] = item;
        mbar_arrive(&ifull[q]);
      }
      item = __shfl_sync(0xffffffffu, item, 0);
      if (++q == kRing) { q = 0; qphase ^= 1; }
      if (item < 0) break;
      const MxItem it = mx_item(p, n_groups, item);
      const MxGroup g = p.groups[it.group];
      const int K = it.phase == 1 ? p.hidden : p.inter;
      // first scale byte of the rows this lane copies: tile rows lane + 32 * i
      const uint8_t* src = p.scales + static_cast<int64_t>(g.slot) * p.row_bytes;
      const int64_t pitch = K / 32;
      int64_t row0;  // matrix row of tile row 0
      if (it.phase == 1) {
        row0 = static_cast<int64_t>(it.tile) * kMxFeatures;
      } else {
        src += 2 * static_cast<int64_t>(p.inter) * (p.hidden / 32);
        row0 = static_cast<int64_t>(it.tile) * kMxM;
      }
      for (int k0 = 0; k0 < K; k0 += kMxChunkK) {
        if (!mx_wait_warp(&cempty[stage], phase ^ 1, abort_flag, p.err)) { ok = false; break; }
        uint8_t* cs = codes + stage * kCodeBytes;
        if (lane == 0) {
          mbar_expect_tx(&cfull[stage], kCodeBytes);
          if (it.phase == 1) {
            tma_load_3d(cs, &w1, &cfull[stage], k0 / 2, static_cast<int>(row0), g.slot);
            tma_load_3d(cs + kCodeBytes / 2, &w1, &cfull[stage], k0 / 2, p.inter + static_cast<int>(row0),
                        g.slot);
          } else {
            tma_load_3d(cs, &w2, &cfull[stage], k0 / 2, static_cast<int>(row0), g.slot);
          }
        }
        uint8_t* ss = scale + stage * kScaleBytes;
        const bool whole = K - k0 >= kMxChunkK;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = lane + 32 * i;
          const int64_t row = it.phase == 1 && r >= kMxFeatures ? p.inter + row0 + r - kMxFeatures
                                                                : row0 + r;
          const uint8_t* from = src + row * pitch + k0 / 32;
          cp_async4(ss + r * 8, from);
          if (whole) cp_async4(ss + r * 8 + 4, from + 4);
        }
        cp_async_arrive(&cfull[stage]);
        pending |= 1u << stage;
        pend_parity = (pend_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == kCodeStages) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok) {
      // the other roles stop at the abort flag; let this CTA's loads land first
      *abort_flag = 1;
      asm volatile("cp.async.wait_all;" ::: "memory");
      const uint64_t t0 = globaltimer_ns();
      for (int s = 0; s < kCodeStages; ++s)
        if (pending & (1u << s))
          while (!mbar_try_wait(&cfull[s], (pend_parity >> s) & 1) && globaltimer_ns() - t0 < kMxWaitNs) {}
    }
  } else if (warp == 14) {
    // ---------------- routes ----------------
    int stage = 0;
    uint32_t phase = 0, pending = 0, pend_parity = 0;
    bool ok = true;
    if (elect_one()) {
      while (ok) {
        if (!mx_wait(&ifull[q], qphase, abort_flag, p.err)) { ok = false; break; }
        const int item = ring[q];
        mbar_arrive(&iempty[q]);
        if (++q == kRing) { q = 0; qphase ^= 1; }
        if (item < 0) break;
        const MxItem it = mx_item(p, n_groups, item);
        const MxGroup g = p.groups[it.group];
        if (it.phase == 2) {
          // the sub-group's activations: four epilogue warps for each phase-1 tile
          const uint32_t want = 4 * p.mt1;
          const uint32_t* cnt = reinterpret_cast<const uint32_t*>(p.dep + it.group);
          const uint64_t t0 = globaltimer_ns();
          while (ld_acquire_gpu_u32(cnt) < want) {
            __nanosleep(64);
            if (*abort_flag) { ok = false; break; }
            if (globaltimer_ns() - t0 > kMxWaitNs) {
              *abort_flag = 1;
              atomicCAS(p.err, 0, DEV_WAIT_TIMEOUT);
              ok = false;
              break;
            }
          }
          if (!ok) break;
          asm volatile("fence.proxy.async.global;" ::: "memory");
        }
        const BMaps* bm = it.phase == 1 ? &bx : &ba;
        const int bi = mx_box(g.count);
        const uint32_t bytes = (16u << bi) * kMxStepK * 2;
        const int steps = (it.phase == 1 ? p.hidden : p.inter) / kMxStepK;
        for (int kb = 0; kb < steps; ++kb) {
          if (!mx_wait(&sempty[stage], phase ^ 1, abort_flag, p.err)) { ok = false; break; }
          mbar_expect_tx(&rfull[stage], bytes);
          tma_load_2d(routes + stage * kRouteBytes, &bm->m[bi], &rfull[stage], kb * kMxStepK, g.start);
          pending |= 1u << stage;
          pend_parity = (pend_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == kSteps) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) {
        *abort_flag = 1;
        const uint64_t t0 = globaltimer_ns();
        for (int s = 0; s < kSteps; ++s)
          if (pending & (1u << s))
            while (!mbar_try_wait(&rfull[s], (pend_parity >> s) & 1) && globaltimer_ns() - t0 < kMxWaitNs) {}
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA ----------------
    if (elect_one()) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      while (ok) {
        if (!mx_wait(&ifull[q], qphase, abort_flag, p.err)) break;
        const int item = ring[q];
        mbar_arrive(&iempty[q]);
        if (++q == kRing) { q = 0; qphase ^= 1; }
        if (item < 0) break;
        const MxItem it = mx_item(p, n_groups, item);
        const uint32_t n = static_cast<uint32_t>(p.groups[it.group].count + 15) & ~15u;
        const uint32_t idesc = idesc_bf16_f32(kMxM, n);
        const int steps = (it.phase == 1 ? p.hidden : p.inter) / kMxStepK;
        if (!mx_wait(&tempty[acc], acc_phase ^ 1, abort_flag, p.err)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * kMxN;
        for (int kb = 0; kb < steps; ++kb) {
          if (!mx_wait(&rfull[stage], phase, abort_flag, p.err) ||
              !mx_wait(&wfull[stage], phase, abort_flag, p.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t b = smem_u32(routes + stage * kRouteBytes);
          const uint32_t a = tmem + kTmemW + stage * 32;
#pragma unroll
          for (int k = 0; k < kMxStepK / 16; ++k)
            umma_bf16_ta(d, a + k * 8, smem_desc_sw128(b + k * 32), idesc, (kb > 0 || k > 0) ? 1u : 0u);
          umma_commit(&sempty[stage]);
          if (++stage == kSteps) { stage = 0; phase ^= 1; }
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
  } else if (warp >= 6) {
    // ---------------- expansion (warps 6..13) ----------------
    const int set = warp >= 10;            // even or odd steps
    const int r = (warp & 3) * 32 + lane;  // weight row of the tile = TMEM lane
    const uint32_t lanes = tmem + kTmemW + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    int cstage = 0, stage = set;
    uint32_t cphase = 0, phase = 0;
    bool ok = true;
    while (ok) {
      if (!mx_wait_warp(&ifull[q], qphase, abort_flag, p.err)) break;
      const int item = ring[q];
      __syncwarp();
      if (lane == 0) mbar_arrive(&iempty[q]);
      if (++q == kRing) { q = 0; qphase ^= 1; }
      if (item < 0) break;
      const int K = item < n_groups * p.mt1 ? p.hidden : p.inter;
      for (int k0 = 0; k0 < K && ok; k0 += kMxChunkK) {
        if (!mx_wait_warp(&cfull[cstage], cphase, abort_flag, p.err)) { ok = false; break; }
        const uint8_t* cs = codes + cstage * kCodeBytes + r * 128;
        const uint2 sc = *reinterpret_cast<const uint2*>(scale + cstage * kScaleBytes + r * 8);
        // this warp's one or two steps of the chunk: steps set and set + 2
        const int n = K - k0 >= kMxChunkK ? 2 : 1;
        uint4 c[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i < n) {
            const int at = 2 * (set + 2 * i);
            c[2 * i] = *reinterpret_cast<const uint4*>(cs + ((at ^ (r & 7)) << 4));
            c[2 * i + 1] = *reinterpret_cast<const uint4*>(cs + (((at + 1) ^ (r & 7)) << 4));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&cempty[cstage]);  // the codes are in registers
        if (++cstage == kCodeStages) { cstage = 0; cphase ^= 1; }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i < n) {
            const uint32_t two = (i ? sc.y : sc.x) >> (16 * set);
            uint32_t o[32];
            expand32(c[2 * i], two & 255u, o);
            expand32(c[2 * i + 1], (two >> 8) & 255u, o + 16);
            if (!mx_wait_warp(&sempty[stage], phase ^ 1, abort_flag, p.err)) { ok = false; break; }
            tc_fence_after();
            tmem_st32(lanes + stage * 32, o);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&wfull[stage]);
            stage += 2;
            if (stage >= kSteps) { stage -= kSteps; phase ^= 1; }
          }
        }
      }
    }
  } else {
    // ---------------- epilogue (warps 2..5) ----------------
    // TMEM lanes 32 * (warp % 4)..: quarters 0, 1 hold gate rows of a phase-1
    // tile, 2, 3 the up rows of the same features
    const int qd = warp & 3;
    const bool up_rows = qd >= 2;
    const int f_local = (qd & 1) * 32 + lane;
    float* give = xchg + (up_rows ? kMxFeatures * kXStride : 0) + f_local * kXStride;
    const float* take = xchg + (up_rows ? 0 : kMxFeatures * kXStride) + f_local * kXStride;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (;;) {
      if (!mx_epilogue_all(mx_wait(&ifull[q], qphase, abort_flag, p.err))) break;
      const int item = ring[q];
      __syncwarp();
      if (lane == 0) mbar_arrive(&iempty[q]);
      if (++q == kRing) { q = 0; qphase ^= 1; }
      if (item < 0) break;  // the same entry for all four warps
      const MxItem it = mx_item(p, n_groups, item);
      const MxGroup g = p.groups[it.group];
      if (!mx_epilogue_all(mx_wait(&tfull[acc], acc_phase, abort_flag, p.err))) break;
      tc_fence_after();
      const uint32_t d = tmem + (static_cast<uint32_t>(qd * 32) << 16) + acc * kMxN;
      if (it.phase == 1) {
        // 32 routes at a time: gate warps finish the first 16, up warps the rest
        const int column = mx_column(it.tile * kMxFeatures + f_local);
        for (int c0 = 0; c0 < g.count; c0 += 32) {
          float lo[16], hi[16];
          tmem_ld16(d + c0, lo);
          tmem_ld16(d + c0 + 16, hi);
#pragma unroll
          for (int j = 0; j < 16; ++j) give[j] = up_rows ? lo[j] : hi[j];
          mx_epilogue_sync();
          const int first = c0 + (up_rows ? 16 : 0);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (first + j < g.count) {
              const float gate = up_rows ? take[j] : lo[j];
              const float up = up_rows ? hi[j] : take[j];
              const float a = __fdividef(gate, 1.0f + __expf(-gate)) * up;
              p.act[static_cast<size_t>(g.start + first + j) * p.inter + column] = __float2bfloat16_rn(a);
            }
          }
          mx_epilogue_sync();
        }
      } else {
        const int feature = it.tile * kMxM + qd * 32 + lane;
        for (int c0 = 0; c0 < g.count; c0 += 16) {
          float v[16];
          tmem_ld16(d + c0, v);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (c0 + j < g.count) {
              const size_t row = static_cast<size_t>(g.start + c0 + j);
              const float w = g.bad ? __uint_as_float(0x7fc00000u) : p.route_w[row];
              p.out[row * p.hidden + feature] = __float2bfloat16_rn(v[j] * w);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
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
// zeroes the counters; the other blocks gather the routes' rows (columns in the
// stored order) and weights, a warp per route.
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
  int hidden;
  __nv_bfloat16* x;
  float* route_w;
  MxGroup* groups;
  int* n_sub;
  int* queue;
  int* dep;
  int* err;
};

constexpr int kPrepThreads = 256;

__global__ void __launch_bounds__(kPrepThreads) mxfp4_prepare_kernel(const MxPrepare a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x == 0) {
    __shared__ int warp_sum[kPrepThreads / 32];
    __shared__ int base;
    if (threadIdx.x == 0) { base = 0; *a.queue = 0; }
    // ascending starts inside [0, routes], or no group at all: the tables below
    // are sized for groups that do not overlap
    bool ordered = true;
    for (int g = threadIdx.x; g <= a.n_groups; g += kPrepThreads) {
      const int64_t s0 = a.starts[g];
      ordered &= s0 >= 0 && s0 <= a.routes && (g == 0 || a.starts[g - 1] <= s0);
    }
    if (!__syncthreads_and(ordered)) {
      if (threadIdx.x == 0) { *a.n_sub = 0; atomicCAS(a.err, 0, DEV_BAD_INPUT); }
      return;
    }
    for (int g0 = 0; g0 < a.n_groups; g0 += kPrepThreads) {
      const int g = g0 + threadIdx.x;
      int64_t s0 = 0, count = 0, slot = 0;
      if (g < a.n_groups) {
        s0 = a.starts[g];
        count = a.starts[g + 1] - s0;
        slot = a.slots[g];
      }
      const bool bad = count > 0 && (slot < 0 || slot >= a.cache_slots);
      if (bad) { slot = 0; atomicCAS(a.err, 0, DEV_BAD_INPUT); }
      const int n = static_cast<int>((count + kMxN - 1) / kMxN);
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
      for (int i = 0; i < n; ++i) {
        const int64_t r0 = count * i / n, r1 = count * (i + 1) / n;
        a.groups[at + i] = MxGroup{static_cast<int>(slot), static_cast<int>(s0 + r0),
                                   static_cast<int>(r1 - r0), bad ? 1 : 0};
        a.dep[at + i] = 0;
      }
      __syncthreads();
      if (threadIdx.x == kPrepThreads - 1) base = before + scan;
      __syncthreads();
    }
    if (threadIdx.x == 0) *a.n_sub = base;
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
    uint4* to = reinterpret_cast<uint4*>(a.x + i * a.hidden);
    for (int v = lane; v < a.hidden / 8; v += 32) {
      uint4 e = make_uint4(0, 0, 0, 0);
      if (good) e = from[v];
      to[v] = make_uint4(__byte_perm(e.x, e.z, 0x5410), __byte_perm(e.x, e.z, 0x7632),
                         __byte_perm(e.y, e.w, 0x5410), __byte_perm(e.y, e.w, 0x7632));
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
static int make_map_codes(CUtensorMap* map, const void* base, uint64_t row_codes, uint64_t rows,
                          uint64_t slots, uint64_t slot_bytes, uint32_t box_rows) {
  PFN_encodeTiled enc = encode_tiled_fn();
  if (!enc) return fail(FERRYB_ECUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {row_codes, rows, slots};
  cuuint64_t strides[2] = {row_codes, slot_bytes};
  cuuint32_t box[3] = {128, box_rows, 1};
  cuuint32_t elem[3] = {1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box,
                   elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(FERRYB_ECUDA, "cuTensorMapEncodeTiled failed (%d) for %llu x %llu codes", (int)r,
                (unsigned long long)rows, (unsigned long long)row_codes);
  return FERRYB_OK;
}

static int64_t mx_align(int64_t b) { return (b + 255) & ~int64_t(255); }

struct MxWs {
  int64_t x, act, w, groups, counters, total;
  int64_t max_sub;
};
static MxWs mx_ws(int64_t routes, int64_t n_groups, int64_t hidden, int64_t inter) {
  MxWs w{};
  w.max_sub = n_groups + routes / kMxN + 1;
  w.x = 0;
  w.act = w.x + mx_align(routes * hidden * 2);
  w.w = w.act + mx_align(routes * inter * 2);
  w.groups = w.w + mx_align(routes * 4);
  w.counters = w.groups + mx_align(w.max_sub * (int64_t)sizeof(MxGroup));
  w.total = w.counters + mx_align((2 + w.max_sub) * 4);
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
  FB_CHECK_ARG((n_groups + routes / kMxN + 1) * (inter / 64 + hidden / 128) < (int64_t(1) << 30),
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
  FB_CHECK_ARG(reinterpret_cast<uintptr_t>(e->cache) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(e->input) % 16 == 0 &&
                   (e->n_input <= 1 || (e->input_stride % 8 == 0 && e->input_stride >= e->hidden)),
               "execute_experts_mxfp4: cache and input rows must be 16-byte aligned");
  const MxWs ws = mx_ws(e->routes, e->n_groups, e->hidden, e->intermediate);
  FB_CHECK_ARG(e->workspace && reinterpret_cast<uintptr_t>(e->workspace) % 256 == 0 &&
                   e->workspace_bytes >= ws.total,
               "execute_experts_mxfp4: workspace too small (%lld < %lld) or misaligned",
               (long long)e->workspace_bytes, (long long)ws.total);
  uint8_t* base = static_cast<uint8_t*>(e->workspace);
  int* counters = reinterpret_cast<int*>(base + ws.counters);

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
  pr.x = reinterpret_cast<__nv_bfloat16*>(base + ws.x);
  pr.route_w = reinterpret_cast<float*>(base + ws.w);
  pr.groups = reinterpret_cast<MxGroup*>(base + ws.groups);
  pr.queue = counters;
  pr.n_sub = counters + 1;
  pr.dep = counters + 2;
  pr.err = e->err;

  int device = 0;
  FB_CUDA(cudaGetDevice(&device));
  const int sms = num_sms(device);
  CUtensorMap w1, w2;
  BMaps bx, ba;
  const int64_t hi = e->hidden * e->intermediate, row_bytes = 3 * hi / 32 * 17;
  const uint8_t* cache = static_cast<const uint8_t*>(e->cache);
  if ((s = make_map_codes(&w1, cache, e->hidden / 2, 2 * e->intermediate, e->cache_slots, row_bytes,
                          kMxFeatures)))
    return s;
  if ((s = make_map_codes(&w2, cache + hi, e->intermediate / 2, e->hidden, e->cache_slots, row_bytes,
                          kMxM)))
    return s;
  for (int i = 0; i < 4; ++i) {
    if ((s = make_map_2d_bf16(&bx.m[i], base + ws.x, e->routes, e->hidden, e->hidden * 2, 16u << i,
                              kMxStepK)))
      return s;
    if ((s = make_map_2d_bf16(&ba.m[i], base + ws.act, e->routes, e->intermediate,
                              e->intermediate * 2, 16u << i, kMxStepK)))
      return s;
  }
  MxParams p{};
  p.groups = pr.groups;
  p.n_groups = pr.n_sub;
  p.mt1 = static_cast<int>(e->intermediate / kMxFeatures);
  p.mt2 = static_cast<int>(e->hidden / kMxM);
  p.hidden = static_cast<int>(e->hidden);
  p.inter = static_cast<int>(e->intermediate);
  p.scales = cache + 3 * hi / 2;
  p.row_bytes = row_bytes;
  p.act = reinterpret_cast<__nv_bfloat16*>(base + ws.act);
  p.out = static_cast<__nv_bfloat16*>(e->out);
  p.route_w = pr.route_w;
  p.queue = pr.queue;
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
  const int64_t subs = e->n_groups < e->routes ? e->n_groups + e->routes / kMxN : e->routes;
  const int64_t items = subs * (p.mt1 + p.mt2);
  mxfp4_swiglu_kernel<<<static_cast<int>(items < sms ? items : sms), kMxThreadsG, kMxSmem, stream>>>(
      w1, w2, bx, ba, p);
  FB_LAUNCH_CHECK();
  return FERRYB_OK;
}
