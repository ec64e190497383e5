// Rows of a matrix in signed 8-bit integers, one FP32 scale a row.
//
//   top = max |x_j|,   scale = top / 127,   q_j = round to even( x_j * (127 / top) )
//
// all in FP32.  A row whose top is below 2^-100 (127 / top would leave the FP32 range) is taken as
// zero: q = 0, scale = 0.  A row that holds a NaN or an infinity gets q = 0 and scale = NaN, so that a
// product with it is NaN in that row and in no other.
// The pass is bound by memory (the input is read once, a byte an element written): a row is held in
// registers between the maximum and the rounding, up to kHeld vectors a thread; what a longer row has
// beyond that is read again, from L2.  A warp takes a row where that holds all of it (16 vectors a lane: 8 KiB
// of row in flight for a warp and no block-wide barrier), a block the longer ones.  8192 x 4096 bf16: 15.2 us,
// 6.6 TB/s; with a conversion instruction an element and single maxima it took 22.9.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "ptx_sm100.cuh"

namespace fnn {

constexpr int kQuantThreads = 256;
constexpr int kQuantHeld = 4;         // vectors a thread holds of a short row, or of one a block shares
constexpr int kQuantManyRows = 1184;  // eight warps for each SM
constexpr int kQuantHeldLong = 16;    // of a row of up to 16 * 512 bytes that a warp takes alone

template <typename T>
__device__ __forceinline__ void quant_unpack(const uint4& w, float (&v)[16 / sizeof(T)]) {
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(q[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q[i]));
      v[2 * i] = f.x; v[2 * i + 1] = f.y;
    } else {
      v[2 * i] = __uint_as_float(q[i] << 16);
      v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
    }
  }
}

// The integer nearest to the FP32 product x * inv, ties to even, in the low byte: |x * inv| <= 127.5, so
// adding 1.5 * 2^23 leaves it in the last bits of the sum.  (The product is rounded first, as the
// definition says: no fused multiply-add.)  A conversion instruction runs at a quarter of this rate.
__device__ __forceinline__ uint32_t quant_one(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.0f));
}
__device__ __forceinline__ uint32_t quant_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// The largest magnitude of a vector as a bit pattern; 16-bit types two at a time, in the upper and the
// lower half of `top` (quant_top joins them).
template <typename T>
__device__ __forceinline__ uint32_t quant_max(uint32_t top, const uint4& w) {
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) top = max(top, q[i] & 0x7fffffffu);
    else top = __vmaxu2(top, q[i] & 0x7fff7fffu);
  }
  return top;
}
template <typename T>
__device__ __forceinline__ uint32_t quant_top(uint32_t top) {
  if constexpr (sizeof(T) == 4) return top;
  const uint32_t m = max(top >> 16, top & 0xffffu);
  if constexpr (std::is_same<T, __half>::value)
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m)))) & 0x7fffffffu;
  else return m << 16;
}

// kPerRow threads share a row (32: a warp, kQuantThreads: the block).  kVec: rows and outputs in whole
// 16-byte vectors of the input.
template <typename T, int kPerRow, bool kVec, int kHeld>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const T* __restrict__ x, long long ld,
                                                                      int8_t* __restrict__ q,
                                                                      float* __restrict__ scale, int rows, int cols) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();
  constexpr int kV = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
  const int part = threadIdx.x % kPerRow;
  const long long row = static_cast<long long>(blockIdx.x) * (kQuantThreads / kPerRow) + threadIdx.x / kPerRow;
  if (kPerRow == 32 && row >= rows) return;            // whole warps leave
  const T* src = x + row * ld;
  int8_t* dst = q + row * cols;
  const int vecs = cols / kV;

  // the magnitudes' bit patterns order as the magnitudes do, NaN above infinity
  uint32_t top = 0;
  uint4 held[kHeld];
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int v = part + i * kPerRow;
      held[i] = v < vecs ? __ldg(reinterpret_cast<const uint4*>(src) + v) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) top = quant_max<T>(top, held[i]);
    for (int v = part + kHeld * kPerRow; v < vecs; v += kPerRow)
      top = quant_max<T>(top, __ldg(reinterpret_cast<const uint4*>(src) + v));
    top = quant_top<T>(top);
  } else {
    for (int c = part; c < cols; c += kPerRow)
      top = max(top, __float_as_uint(static_cast<float>(src[c])) & 0x7fffffffu);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (kPerRow > 32) {
    __shared__ uint32_t warp_top[kQuantThreads / 32];
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerRow / 32; ++i) top = max(top, warp_top[i]);
  }
  const float t = __uint_as_float(top);
  const bool finite = top < 0x7f800000u;
  const bool live = finite && t >= 7.888609052210118e-31f;      // 2^-100
  const float inv = live ? __fdiv_rn(127.0f, t) : 0.0f;
  if (part == 0) scale[row] = finite ? (live ? __fdiv_rn(t, 127.0f) : 0.0f) : __uint_as_float(0x7fffffffu);
  if constexpr (kVec) {
    auto put = [&](const uint4& w, int v) {
      float f[kVec ? 16 / sizeof(T) : 1];
      quant_unpack<T>(w, f);
      uint32_t b[2] = {0, 0};
      if (live) {
#pragma unroll
        for (int j = 0; j < kV; j += 4)
          b[j >> 2] = quant_pack4(quant_one(f[j], inv), quant_one(f[j + 1], inv), quant_one(f[j + 2], inv),
                                  quant_one(f[j + 3], inv));
      }
      if constexpr (kV == 8) reinterpret_cast<uint2*>(dst)[v] = make_uint2(b[0], b[1]);
      else reinterpret_cast<uint32_t*>(dst)[v] = b[0];
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int v = part + i * kPerRow;
      if (v < vecs) put(held[i], v);
    }
    for (int v = part + kHeld * kPerRow; v < vecs; v += kPerRow)
      put(__ldg(reinterpret_cast<const uint4*>(src) + v), v);
  } else {
    for (int c = part; c < cols; c += kPerRow)
      dst[c] = static_cast<int8_t>(live ? quant_one(static_cast<float>(src[c]), inv) & 0xffu : 0u);
  }
}

}  // namespace fnn
