// mxfp4.cu -- MXFP4 quantisation of weight rows and its inverse: e2m1 codes in
// blocks of 32 along a row, one power-of-two scale byte a block.
//
// No counterpart in the reference, whose experts are bf16.  A quantised expert
// is 17 bytes where a bf16 one is 64, and the host link bounds decode, so a
// pool of quantised rows is fetched 3.76 times as fast; execute_experts_mxfp4
// (experts_mxfp4.cu) reads the rows as they are.
//
// A thread takes 8 consecutive values (one 16-byte load of a 16-bit type), four
// neighbouring lanes hold a block: its largest magnitude is two shuffles away.
// The scale is the exponent field of that magnitude minus 2 (the largest e2m1
// value is 6 = 1.5 * 2^2), so x * 2^(127 - s) lies below 8, is exact, and the
// conversion instruction rounds it half to even and holds it at 6.
#include <cuda_fp16.h>
#include <cuda_fp4.h>

#include "common.cuh"

namespace ferryb {

constexpr int kMxThreads = 256;
constexpr int kMxUnroll = 4;  // loads in flight a thread

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }

// 8 values at p, which is aligned to ALIGN bytes (0: to a value).  8 floats go as one
// 32-byte access where they may: two of 16 bytes with 32 between lanes leave half
// sectors to each (1.4e8 values there and back: 194 us, at the
// copy rate, against 229).
template <typename T, int ALIGN>
__device__ __forceinline__ void load8(const T* p, float* v) {
  if constexpr (ALIGN == 32 && sizeof(T) == 4) {
    asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(p));
  } else if constexpr (ALIGN && sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else if constexpr (ALIGN != 0) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(p[i]);
  }
}

struct MxShape {
  int64_t units;          // groups of 8 values in all
  int64_t units_per_row;
  int64_t stride, codes_stride, scales_stride;  // elements, bytes, bytes
};

__device__ __forceinline__ void unit_place(const MxShape& s, int64_t u, int64_t* row, int64_t* in_row) {
  if (s.units == s.units_per_row) { *row = 0; *in_row = u; return; }  // one row (or rows without gaps)
  if (s.units <= 0xffffffffll) {
    const uint32_t r = static_cast<uint32_t>(u) / static_cast<uint32_t>(s.units_per_row);
    *row = r;
    *in_row = u - static_cast<int64_t>(r) * s.units_per_row;
  } else {
    *row = u / s.units_per_row;
    *in_row = u - *row * s.units_per_row;
  }
}

template <typename T, int ALIGN>
__global__ void __launch_bounds__(kMxThreads)
    quantize_mxfp4_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                          uint8_t* __restrict__ scales, const MxShape s) {
  pdl_wait();
  const int64_t u0 = static_cast<int64_t>(blockIdx.x) * (kMxThreads * kMxUnroll) + threadIdx.x;
  float v[kMxUnroll][8];
  int64_t row[kMxUnroll], in_row[kMxUnroll];
#pragma unroll
  for (int k = 0; k < kMxUnroll; ++k) {
    const int64_t u = u0 + k * kMxThreads;
    if (u < s.units) {
      unit_place(s, u, &row[k], &in_row[k]);
      load8<T, ALIGN>(x + row[k] * s.stride + in_row[k] * 8, v[k]);
    } else {
      row[k] = -1;
    }
  }
#pragma unroll
  for (int k = 0; k < kMxUnroll; ++k) {
    // units is a multiple of 4 (a block), so a block's four lanes are all in or all out
    uint32_t top = 0;
    if (row[k] >= 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[k][i]) & 0x7fffffffu);
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (row[k] < 0) continue;
    const int field = static_cast<int>(top >> 23);
    const bool bad = field == 255;
    const int byte = bad ? 255 : max(field - 2, 0);
    const float mult = bad ? 0.0f : __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
    uint32_t packed = 0;
    if (!bad) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 pair = make_float2(v[k][2 * i] * mult, v[k][2 * i + 1] * mult);
        packed |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(pair, __NV_E2M1, cudaRoundNearest))
                  << (8 * i);
      }
    }
    uint8_t* c = codes + row[k] * s.codes_stride + in_row[k] * 4;
    if constexpr (ALIGN != 0) {
      *reinterpret_cast<uint32_t*>(c) = packed;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = static_cast<uint8_t>(packed >> (8 * i));
    }
    if ((in_row[k] & 3) == 0) scales[row[k] * s.scales_stride + (in_row[k] >> 2)] = static_cast<uint8_t>(byte);
  }
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v, int align) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  if (align) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
  else
    for (int i = 0; i < 8; ++i) p[i] = reinterpret_cast<const __nv_bfloat16*>(h)[i];
}
__device__ __forceinline__ void store8(__half* p, const float* v, int align) {
  __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  if (align) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
  else
    for (int i = 0; i < 8; ++i) p[i] = reinterpret_cast<const __half*>(h)[i];
}
__device__ __forceinline__ void store8(float* p, const float* v, int align) {
  if (align == 32) {
    asm volatile("st.global.v8.f32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                 "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "l"(p)
                 : "memory");
  } else if (align) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = v[i];
  }
}

template <typename T, int ALIGN>
__global__ void __launch_bounds__(kMxThreads)
    dequantize_mxfp4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                            T* __restrict__ y, const MxShape s) {
  pdl_wait();
  const int64_t u0 = static_cast<int64_t>(blockIdx.x) * (kMxThreads * kMxUnroll) + threadIdx.x;
  uint32_t packed[kMxUnroll];
  int byte[kMxUnroll];
  T* out[kMxUnroll];
#pragma unroll
  for (int k = 0; k < kMxUnroll; ++k) {
    const int64_t u = u0 + k * kMxThreads;
    out[k] = nullptr;
    if (u < s.units) {
      int64_t row, in_row;
      unit_place(s, u, &row, &in_row);
      const uint8_t* c = codes + row * s.codes_stride + in_row * 4;
      if constexpr (ALIGN != 0) packed[k] = *reinterpret_cast<const uint32_t*>(c);
      else packed[k] = c[0] | (c[1] << 8) | (c[2] << 16) | (static_cast<uint32_t>(c[3]) << 24);
      byte[k] = scales[row * s.scales_stride + (in_row >> 2)];
      out[k] = y + row * s.stride + in_row * 8;
    }
  }
#pragma unroll
  for (int k = 0; k < kMxUnroll; ++k) {
    if (!out[k]) continue;
    // 2^(byte - 127): byte 0 is the subnormal 2^-127, byte 255 NaN
    const float scale = byte[k] == 255 ? __uint_as_float(0x7fc00000u)
                        : byte[k] == 0 ? __uint_as_float(0x00400000u)
                                       : __uint_as_float(static_cast<uint32_t>(byte[k]) << 23);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(
          static_cast<__nv_fp4x2_storage_t>(packed[k] >> (8 * i)), __NV_E2M1);
      const float2 f = __half22float2(__half2(h));
      v[2 * i] = f.x * scale;
      v[2 * i + 1] = f.y * scale;
    }
    store8(out[k], v, ALIGN);
  }
}

// Rows without gaps on either side are one long row: no division a unit.
static MxShape mx_shape(int64_t rows, int64_t width, int64_t stride, int64_t codes_stride,
                        int64_t scales_stride) {
  MxShape s{};
  s.units = rows * (width / 8);
  const bool dense = stride == width && codes_stride == width / 2 && scales_stride == width / 32;
  s.units_per_row = dense ? s.units : width / 8;
  s.stride = stride;
  s.codes_stride = codes_stride;
  s.scales_stride = scales_stride;
  return s;
}

static bool aligned(const void* p, int64_t stride_bytes, int64_t to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && stride_bytes % to == 0;
}

static int mx_check(const char* what, const void* x, int32_t type, int64_t rows, int64_t width,
                    int64_t stride, const void* codes, int64_t codes_stride, const void* scales,
                    int64_t scales_stride) {
  FB_CHECK_ARG(rows >= 0 && width >= 0 && width % 32 == 0,
               "%s: width %lld must be a multiple of 32", what, (long long)width);
  FB_CHECK_ARG(type >= FERRYB_BF16 && type <= FERRYB_FP32, "%s: unknown type %d", what, type);
  if (rows == 0 || width == 0) return FERRYB_OK;
  FB_CHECK_ARG(x && codes && scales, "%s: null pointer", what);
  FB_CHECK_ARG(reinterpret_cast<uintptr_t>(x) % (type == FERRYB_FP32 ? 4 : 2) == 0,
               "%s: misaligned values", what);
  FB_CHECK_ARG(rows <= (int64_t(1) << 42) / width, "%s: more than 2^42 values", what);
  FB_CHECK_ARG(rows == 1 || (stride >= width && codes_stride >= width / 2 &&
                             scales_stride >= width / 32), "%s: rows overlap", what);
  return FERRYB_OK;
}

template <typename T>
static int quantize_typed(const void* x, void* codes, void* scales, const MxShape& s, int align,
                          cudaStream_t stream) {
  const int64_t per = kMxThreads * kMxUnroll;
  const unsigned grid = static_cast<unsigned>((s.units + per - 1) / per);
  auto kernel = align == 0 ? quantize_mxfp4_kernel<T, 0> : quantize_mxfp4_kernel<T, 16>;
  if (sizeof(T) == 4 && align == 32) kernel = quantize_mxfp4_kernel<T, sizeof(T) == 4 ? 32 : 16>;
  return launch_behind(kernel, grid, kMxThreads, 0, stream, static_cast<const T*>(x), static_cast<uint8_t*>(codes),
                       static_cast<uint8_t*>(scales), s);
}

template <typename T>
static int dequantize_typed(const void* codes, const void* scales, void* y, const MxShape& s, int align,
                            cudaStream_t stream) {
  const int64_t per = kMxThreads * kMxUnroll;
  const unsigned grid = static_cast<unsigned>((s.units + per - 1) / per);
  auto kernel = align == 0 ? dequantize_mxfp4_kernel<T, 0> : dequantize_mxfp4_kernel<T, 16>;
  if (sizeof(T) == 4 && align == 32) kernel = dequantize_mxfp4_kernel<T, sizeof(T) == 4 ? 32 : 16>;
  return launch_behind(kernel, grid, kMxThreads, 0, stream, static_cast<const uint8_t*>(codes),
                       static_cast<const uint8_t*>(scales), static_cast<T*>(y), s);
}

}  // namespace ferryb

using namespace ferryb;

extern "C" int ferryb_quantize_mxfp4(const void* x, int32_t x_type, int64_t rows, int64_t width,
                                     int64_t x_stride, void* codes, int64_t codes_stride,
                                     void* scales, int64_t scales_stride, cudaStream_t stream) {
  int st = mx_check("quantize_mxfp4", x, x_type, rows, width, x_stride, codes, codes_stride, scales,
                    scales_stride);
  if (st || rows == 0 || width == 0) return st;
  const MxShape s = mx_shape(rows, width, x_stride, codes_stride, scales_stride);
  const int64_t size = x_type == FERRYB_FP32 ? 4 : 2;
  const int64_t step = rows > 1 ? x_stride * size : 0;
  const int align = !aligned(codes, rows > 1 ? codes_stride : 0, 4) ? 0
                    : aligned(x, step, 32) ? 32 : aligned(x, step, 16) ? 16 : 0;
  switch (x_type) {
    case FERRYB_BF16: return quantize_typed<__nv_bfloat16>(x, codes, scales, s, align, stream);
    case FERRYB_FP16: return quantize_typed<__half>(x, codes, scales, s, align, stream);
    default: return quantize_typed<float>(x, codes, scales, s, align, stream);
  }
}

extern "C" int ferryb_dequantize_mxfp4(const void* codes, int64_t codes_stride, const void* scales,
                                       int64_t scales_stride, int64_t rows, int64_t width, void* y,
                                       int32_t y_type, int64_t y_stride, cudaStream_t stream) {
  int st = mx_check("dequantize_mxfp4", y, y_type, rows, width, y_stride, codes, codes_stride, scales,
                    scales_stride);
  if (st || rows == 0 || width == 0) return st;
  const MxShape s = mx_shape(rows, width, y_stride, codes_stride, scales_stride);
  const int64_t size = y_type == FERRYB_FP32 ? 4 : 2;
  const int64_t step = rows > 1 ? y_stride * size : 0;
  const int align = !aligned(codes, rows > 1 ? codes_stride : 0, 4) ? 0
                    : aligned(y, step, 32) ? 32 : aligned(y, step, 16) ? 16 : 0;
  switch (y_type) {
    case FERRYB_BF16: return dequantize_typed<__nv_bfloat16>(codes, scales, y, s, align, stream);
    case FERRYB_FP16: return dequantize_typed<__half>(codes, scales, y, s, align, stream);
    default: return dequantize_typed<float>(codes, scales, y, s, align, stream);
  }
}
