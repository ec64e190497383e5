// Products of 16-bit, 8-bit and TF32 operands on CTA pairs, with the epilogues of a gated
// feed-forward block and of a product in scaled 8-bit integers.
//
//   C = epilogue( A (m x k) . B (k x n) ),  accumulated in tensor memory (FP32; INT32 for 8 bits)
//
// The pair scheme of gemm_tcgen05_pair.cuh: two CTAs on neighbouring SMs compute one
// 256 x block_n tile with tcgen05.mma cta_group::2, each loading its own 128 rows of A and half of
// the B tile.  What is different:
//   * every operand kind uses the same stage: 128 bytes of K per row, i.e. 64 elements of 16 bits,
//     128 of 8 bits or 32 of 32 bits, and four MMAs of 32 bytes of K each;
//   * a launch holds up to four products (the gradients of one block, which all depend on the same
//     launch before them), so their tiles share the machine's waves instead of ending in four tails;
//   * a gated product takes its B tile from two matrices: the leader's half of the 256 columns from
//     the gate's weight, the peer's from the up projection's.  Columns [0, block_n/2) of the
//     accumulator are then gate and the others up for the SAME outputs, in the same CTA's tensor
//     memory, and act(gate) * up is formed in the epilogue without either leaving the chip.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "gemm_tcgen05.cuh"

namespace fnn {

// Operand kinds.  16-bit operands of one launch are all bf16 or all fp16.
enum : int { kKindF16 = 0, kKindI8 = 1, kKindTf32 = 2 };
// Epilogues.
enum : int {
  kEpiStore = 0,      // C = acc
  kEpiGated = 1,      // out0 = act(gate) * up, optionally out1 = gate, out2 = up
  kEpiGatedGrad = 2,  // acc = dh: out0 = dh * up * act'(gate), out1 = dh * act(gate), out2 = act(gate) * up
  kEpiScaled = 3,     // C = act(acc * row_scale * col_scale + bias)
  kEpiScaledGated = 4 // C = act(gate * row_scale * col_scale) * (up * row_scale * col_scale2)
};
// Activations of this file's epilogues (the public codes, kActSilu beyond the GEMM epilogue's own).
constexpr int kActSilu = 5;

constexpr int kNarrowEpiWarps = 8;
constexpr int kNarrowThreads = 64 + 32 * kNarrowEpiWarps;
constexpr int kNarrowMaxProblems = 4;
constexpr int kNarrowMaxStages = 8;
constexpr int kNarrowTile = 4096;                    // one staging tile: 32 rows x 128 bytes
constexpr int kNarrowABytes = 128 * 128;             // 128 rows x 128 bytes of K

struct NarrowProblem {
  CUtensorMap a[2], b[2];      // [1]: second K range (C = A0.B0 + A1.B1), or the up weight of a gated product
  CUtensorMap out[3];
  void* out_ptr[3];            // the same outputs for stores TMA cannot make; null: not wanted
  long long out_ld[3];         // their row strides in elements
  const void* gate;            // saved projections of kEpiGatedGrad, row stride aux_ld elements
  const void* up;
  long long aux_ld;
  int m, n;                    // n: columns of ONE output
  int tiles_m, tiles_n;
  int num_kb, num_kb1;         // 128-byte k-blocks in all, and those of the first operand pair
  int split_k, kb_per_split;   // split_k > 1: partial sums, FP32, one [m, n] block per slice in out[0]
  int first_unit;
  int a_mn, b_mn;              // operand stored with M (N) contiguous
  int tma_out[3];              // outputs are TMA-addressable
};

struct NarrowParams {
  NarrowProblem pr[kNarrowMaxProblems];
  int count, total_units, block_n, num_stages, group_m;
  int act, is_bf16;
  const float* row_scale;
  const float* col_scale;
  const float* col_scale2;
  const float* bias;
  unsigned int* status;
  long long spin_budget;
};

namespace ptx {
template <int kKind>
__device__ __forceinline__ void mma_narrow_2cta(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                                uint32_t accumulate) {
  if constexpr (kKind == kKindF16)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
                 "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
                 : "memory");
  else if constexpr (kKind == kKindI8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
                 "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
                 : "memory");
  else
    mma_tf32_2cta(tmem_d, desc_a, desc_b, idesc, accumulate);
}
// Instruction descriptor.  Formats of kind::f16: 0 = fp16, 1 = bf16; of kind::i8: 1 = signed; of
// kind::tf32: 2.  D: 1 = F32, 2 = S32.
template <int kKind>
__device__ __forceinline__ uint32_t idesc_narrow(int m, int n, int a_mn, int b_mn, int is_bf16) {
  const uint32_t d = kKind == kKindI8 ? 2u : 1u;
  const uint32_t f = kKind == kKindF16 ? (is_bf16 ? 1u : 0u) : (kKind == kKindI8 ? 1u : 2u);
  return (d << 4) | (f << 7) | (f << 10) | (static_cast<uint32_t>(a_mn & 1) << 15) |
         (static_cast<uint32_t>(b_mn & 1) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
}  // namespace ptx

// Bytes of an element, elements of one 128-byte k-block.
template <int kKind>
struct NarrowKind {
  static constexpr int kBytes = kKind == kKindF16 ? 2 : (kKind == kKindI8 ? 1 : 4);
  static constexpr int kBlock = 128 / kBytes;
  // MN-major operands: chunks of 128 bytes along M (N), one row per k, kBlock rows per chunk;
  // 16-bit ones in the 16-byte swizzle with 8-row groups, TF32 in the 32-byte swizzle with 4-row groups.
  static constexpr uint32_t kChunkElems = kBlock;
  static constexpr uint32_t kChunkBytes = kBlock * 128;
  static constexpr uint32_t kMnSbo = kKind == kKindTf32 ? 512 : 1024;
  static constexpr uint32_t kMnStep = kKind == kKindTf32 ? 1024 : 2048;   // bytes per MMA's K
  static constexpr uint32_t kMnLayout = kKind == kKindTf32 ? ptx::kLayoutSw128Base32 : ptx::kLayoutSw128;
};

template <int kKind>
__device__ __forceinline__ uint64_t narrow_desc(uint32_t addr, int mn_major) {
  using K = NarrowKind<kKind>;
  return mn_major ? ptx::smem_desc_sw128(addr, K::kChunkBytes, K::kMnSbo, K::kMnLayout)
                  : ptx::smem_desc_sw128(addr, 16u, 1024u, ptx::kLayoutSw128);
}

// ------------------------------------------------------------------ activations ---
// x / (1 + e^-x) on the special-function unit: __expf and __fdividef are good to a few units in
// the last place of FP32 where the result is a normal number.
__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

template <int kAct>
__device__ __forceinline__ float gate_act(float x) {
  if constexpr (kAct == kActRelu) return x < 0.0f ? 0.0f : x;        // NaN stays NaN
  else if constexpr (kAct == kActGelu) return gelu_erf(x);
  else if constexpr (kAct == kActSilu) return silu(x);
  else return x;
}
// act(x) and its derivative together
template <int kAct>
__device__ __forceinline__ void gate_act_grad(float x, float& a, float& da) {
  if constexpr (kAct == kActRelu) {
    a = x < 0.0f ? 0.0f : x;
    da = x > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (kAct == kActGelu) {
    const float cdf = 0.5f * (1.0f + erff(x * 0.7071067811865475f));
    a = x * cdf;
    da = fmaf(x, __expf(-0.5f * x * x) * 0.3989422804014327f, cdf);
  } else if constexpr (kAct == kActSilu) {
    const float s = __fdividef(1.0f, 1.0f + __expf(-x));
    a = x * s;
    da = s * fmaf(x, 1.0f - s, 1.0f);
  } else {
    a = x;
    da = 1.0f;
  }
}

// ---------------------------------------------------------------- output helpers ---
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// 32 consecutive columns of this lane's row into a staging tile (32 rows x 128 bytes, 16-byte unit j
// of row r at unit j ^ (r & 7)).  16-bit outputs fill the lower (half = 0) or upper half of the row.
template <typename T>
__device__ __forceinline__ void stage_put(uint8_t* tile, int lane, int half, const float (&v)[32]) {
  uint8_t* row = tile + lane * 128;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<float4*>(row + ((j ^ (lane & 7)) << 4)) =
          make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4*>(row + (((half * 4 + j) ^ (lane & 7)) << 4)) =
          make_uint4(pack2<T>(v[8 * j], v[8 * j + 1]), pack2<T>(v[8 * j + 2], v[8 * j + 3]),
                     pack2<T>(v[8 * j + 4], v[8 * j + 5]), pack2<T>(v[8 * j + 6], v[8 * j + 7]));
  }
}

// The staging tile to output rows [m0, m0 + 32), columns from col0: one TMA store, which clips at the
// matrix's edges, or row by row (row strides that are no multiple of 16 bytes, unaligned bases).
template <typename T>
__device__ __forceinline__ void stage_flush(const CUtensorMap* map, void* out, long long ld, int tma, uint8_t* tile,
                                            uint32_t tile_addr, int m0, int col0, int z, int m, int n, int lane) {
  if (tma) {
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      ptx::tma_store_3d(map, tile_addr, col0, m0, z);
      ptx::tma_store_commit();
    }
  } else {
    __syncwarp();
    const int rows = min(32, m - m0);
    for (int r = 0; r < rows; ++r) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) +
                                                            ((lane & 3) << 2));
      T* dst = static_cast<T*>(out) + (static_cast<long long>(z) * m + m0 + r) * ld + col0;
      if constexpr (sizeof(T) == 4) {
        if (col0 + lane < n) reinterpret_cast<uint32_t*>(dst)[lane] = w;
      } else {
        uint16_t* d16 = reinterpret_cast<uint16_t*>(dst);
        if (col0 + 2 * lane < n) d16[2 * lane] = static_cast<uint16_t>(w & 0xffffu);
        if (col0 + 2 * lane + 1 < n) d16[2 * lane + 1] = static_cast<uint16_t>(w >> 16);
      }
    }
    __syncwarp();
  }
}

// 32 columns of this lane's row of a saved projection (16-byte aligned rows; zero outside)
template <typename T>
__device__ __forceinline__ void load_row32(const void* base, long long ld, int row, int col0, int m, int n,
                                           float (&v)[32]) {
  constexpr int kPer = 16 / sizeof(T);
  const T* src = static_cast<const T*>(base) + static_cast<long long>(row) * ld + col0;
#pragma unroll
  for (int j = 0; j < 32 / kPer; ++j) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (row < m && col0 + j * kPer < n) w = __ldg(reinterpret_cast<const uint4*>(src + j * kPer));
    if constexpr (sizeof(T) == 4) {
      v[4 * j] = __uint_as_float(w.x); v[4 * j + 1] = __uint_as_float(w.y);
      v[4 * j + 2] = __uint_as_float(w.z); v[4 * j + 3] = __uint_as_float(w.w);
    } else {
      const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(q[i]);
        v[8 * j + 2 * i] = f.x; v[8 * j + 2 * i + 1] = f.y;
      }
    }
  }
}

// The activation is chosen outside the unrolled loops over columns: body(std::integral_constant<int, act>).
template <typename Body>
__device__ __forceinline__ void for_act(int act, const Body& body) {
  if (act == kActSilu) body(std::integral_constant<int, kActSilu>());
  else if (act == kActGelu) body(std::integral_constant<int, kActGelu>());
  else if (act == kActRelu) body(std::integral_constant<int, kActRelu>());
  else body(std::integral_constant<int, kActNone>());
}

template <typename Params>
__device__ __forceinline__ bool narrow_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                            const Params& p, unsigned int code) {
  if (ptx::mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  int it = 0;
  while (true) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if ((++it & 63) == 0) {
      if (*abort_flag) return false;
      if (clock64() - t0 > p.spin_budget) {
        atomicCAS(p.status, 0u, code);
        *abort_flag = 1;
        __threadfence_block();
        return false;
      }
    }
  }
}

struct NarrowUnit {
  int pr, s, mt, nt, kb0, kb1;
};
__device__ __forceinline__ NarrowUnit narrow_unit(const NarrowParams& p, int u) {
  NarrowUnit w;
  int i = 0;
  while (i + 1 < p.count && u >= p.pr[i + 1].first_unit) ++i;
  const NarrowProblem& q = p.pr[i];
  int t = u - q.first_unit;
  w.pr = i;
  w.s = t % q.split_k;
  t /= q.split_k;
  const int group_sz = p.group_m * q.tiles_n;
  const int g = t / group_sz;
  const int first_m = g * p.group_m;
  const int gm = min(q.tiles_m - first_m, p.group_m);
  const int r = t - g * group_sz;
  w.mt = first_m + r % gm;
  w.nt = r / gm;
  w.kb0 = w.s * q.kb_per_split;
  w.kb1 = min(q.num_kb, w.kb0 + q.kb_per_split);
  return w;
}

template <int kKind, int kEpi, typename OutT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNarrowThreads, 1)
narrow_pair_kernel(const __grid_constant__ NarrowParams p) {
  using K = NarrowKind<kKind>;
  constexpr bool kTwoB = kEpi == kEpiGated || kEpi == kEpiScaledGated;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const int cluster_id = blockIdx.x >> 1;
  const int num_clusters = gridDim.x >> 1;
  const int half_n = p.block_n >> 1;                     // B columns this CTA loads
  const uint32_t stage_bytes = kNarrowABytes + static_cast<uint32_t>(half_n) * 128u;
  const uint32_t staging_base = smem_base + p.num_stages * stage_bytes;
  const uint32_t bar_base = staging_base + kNarrowEpiWarps * kNarrowTile;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 64u + 8u * s; };
  auto tfull_bar = [&](int a) { return bar_base + 128u + 8u * a; };
  auto tempty_bar = [&](int a) { return bar_base + 144u + 8u * a; };
  const uint32_t tmem_slot = bar_base + 160u;
  uint8_t* bar_gen = smem_gen + (bar_base - smem_base);
  volatile uint32_t* tmem_slot_gen = reinterpret_cast<volatile uint32_t*>(bar_gen + 160);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_gen + 168);
  float* scale_gen = reinterpret_cast<float*>(bar_gen + 256);     // 96 floats per epilogue warp (8-bit kinds)

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.num_stages; ++s) {
      ptx::mbar_init(full_bar(s), 2);          // one arrive.expect_tx from each CTA's producer
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(tfull_bar(a), 1);
      ptx::mbar_init(tempty_bar(a), 2 * kNarrowEpiWarps);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  if (warp == 1) {
    ptx::tmem_alloc_2cta(tmem_slot, kTmemCols);
    ptx::tmem_relinquish_2cta();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_arrive_release();               // the peer's barriers exist before anything arrives on them
  ptx::cluster_wait_acquire();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot_gen;

  if (warp == 0) {
    // ------------------------------------------------------------- producer ---
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t pol = ptx::make_l2_policy(3);
      for (int u = cluster_id; u < p.total_units && ok; u += num_clusters) {
        const NarrowUnit w = narrow_unit(p, u);
        const NarrowProblem& q = p.pr[w.pr];
        const int m0 = w.mt * 256 + static_cast<int>(rank) * 128;
        // a gated tile: this CTA's columns are all gate (leader) or all up (peer) columns of the same outputs
        const int n0 = kTwoB ? w.nt * half_n : w.nt * p.block_n + static_cast<int>(rank) * half_n;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          ok = narrow_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, kStatusProducerTimeout);
          if (!ok) break;
          const uint32_t fb = ptx::mapa_shared(full_bar(stage), 0);
          ptx::mbar_expect_tx_cluster(fb, stage_bytes);
          const uint32_t sa = smem_base + stage * stage_bytes;
          const uint32_t sb = sa + kNarrowABytes;
          const bool second = kb >= q.num_kb1;
          const int k0 = (second ? kb - q.num_kb1 : kb) * K::kBlock;
          const CUtensorMap* mA = &q.a[second ? 1 : 0];
          const CUtensorMap* mB = &q.b[kTwoB ? static_cast<int>(rank) : (second ? 1 : 0)];
          if (!q.a_mn) {
            ptx::tma_load_3d_pair(sa, mA, fb, k0, m0, 0, pol);
          } else {
#pragma unroll
            for (int c = 0; c < 128 / static_cast<int>(K::kChunkElems); ++c)
              ptx::tma_load_3d_pair(sa + c * K::kChunkBytes, mA, fb, m0 + c * K::kChunkElems, k0, 0, pol);
          }
          if (!q.b_mn) {
            ptx::tma_load_3d_pair(sb, mB, fb, k0, n0, 0, pol);
          } else {
            for (int c = 0; c < half_n / static_cast<int>(K::kChunkElems); ++c)
              ptx::tma_load_3d_pair(sb + c * K::kChunkBytes, mB, fb, n0 + c * K::kChunkElems, k0, 0, pol);
          }
          if (++stage == p.num_stages) { stage = 0; phase ^= 1u; }
        }
      }
      // every release the leader's commits still owe this CTA must land before exit
      for (int i = 0; i < p.num_stages && ok; ++i) {
        ok = narrow_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, kStatusProducerTimeout);
        if (++stage == p.num_stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (leader only) ---
    if (lane == 0 && rank == 0) {
      const uint64_t stage_step = stage_bytes >> 4;
      const uint32_t bar0 = ptx::mapa_shared(bar_base, 0);
      const uint32_t bar1 = ptx::mapa_shared(bar_base, 1);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int u = cluster_id; u < p.total_units && ok; u += num_clusters) {
        const NarrowUnit w = narrow_unit(p, u);
        const NarrowProblem& q = p.pr[w.pr];
        const uint32_t idesc = ptx::idesc_narrow<kKind>(256, p.block_n, q.a_mn, q.b_mn, p.is_bf16);
        const uint64_t a_desc0 = narrow_desc<kKind>(smem_base, q.a_mn);
        const uint64_t b_desc0 = narrow_desc<kKind>(smem_base + kNarrowABytes, q.b_mn);
        const uint64_t a_step = (q.a_mn ? K::kMnStep : 32u) >> 4;
        const uint64_t b_step = (q.b_mn ? K::kMnStep : 32u) >> 4;
        ok = narrow_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, p, kStatusMmaTmemTimeout);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * kMaxBlockN);
        uint32_t accumulate = 0u;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          ok = narrow_wait(full_bar(stage), phase, abort_flag, p, kStatusMmaTimeout);
          if (!ok) break;
          const uint64_t da = a_desc0 + stage * stage_step;
          const uint64_t db = b_desc0 + stage * stage_step;
          ptx::mma_narrow_2cta<kKind>(tmem_d, da, db, idesc, accumulate);
          accumulate = 1u;
#pragma unroll
          for (int ks = 1; ks < 4; ++ks)
            ptx::mma_narrow_2cta<kKind>(tmem_d, da + ks * a_step, db + ks * b_step, idesc, 1u);
          ptx::mma_commit_2cta(bar0 + 64u + 8u * stage);    // empty[stage], leader
          ptx::mma_commit_2cta(bar1 + 64u + 8u * stage);    // empty[stage], peer
          if (++stage == p.num_stages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        ptx::mma_commit_2cta(bar0 + 128u + 8u * acc);       // accumulator full, both CTAs
        ptx::mma_commit_2cta(bar1 + 128u + 8u * acc);
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
    }
  } else {
    // -------------------------------------------------------------- epilogue ---
    // Two warps per TMEM lane quadrant take alternate chunks of the tile; a chunk is what fills a
    // staging tile, 128 bytes of a row: 64 columns of 16 bits, 32 of 32.
    const int ew = warp - 2;
    const int q4 = warp & 3;
    const int group = ew >> 2;
    const uint32_t tile_addr = staging_base + ew * kNarrowTile;
    uint8_t* tile = smem_gen + (tile_addr - smem_base);
    float* scales = scale_gen + ew * 96;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int u = cluster_id; u < p.total_units && ok; u += num_clusters) {
      const NarrowUnit w = narrow_unit(p, u);
      const NarrowProblem& q = p.pr[w.pr];
      const int m0 = w.mt * 256 + static_cast<int>(rank) * 128 + q4 * 32;
      const int row = m0 + lane;
      const bool raw = q.split_k > 1;
      ok = narrow_wait(tfull_bar(acc), acc_phase, abort_flag, p, kStatusEpilogueTimeout);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ptx::tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q4 * 32) << 16) +
                             static_cast<uint32_t>(acc * kMaxBlockN);
      auto load32 = [&](int col, float (&v)[32]) {           // 32 accumulator columns as floats
        uint32_t r[32];
        ptx::tmem_ld_32x32(taddr + col, r);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j)
          v[j] = kKind == kKindI8 ? static_cast<float>(static_cast<int>(r[j])) : __uint_as_float(r[j]);
      };
      auto tile_free = [&]() {                               // the staging tile may be overwritten
        if (lane == 0) ptx::tma_store_wait_read<0>();
        __syncwarp();
      };
      const bool rows_live = m0 < q.m;                       // warp-uniform
      if (rows_live) {
      if constexpr (kEpi == kEpiStore) {
        const int n0 = w.nt * p.block_n;
        if (raw) {                                           // FP32 partial sums of one K slice
          for (int c = group; c < p.block_n / 32; c += 2) {
            const int col0 = n0 + c * 32;
            if (col0 >= q.n) break;
            float v[32];
            load32(c * 32, v);
            tile_free();
            stage_put<float>(tile, lane, 0, v);
            stage_flush<float>(&q.out[0], q.out_ptr[0], q.out_ld[0], true, tile, tile_addr, m0, col0, w.s, q.m, q.n, lane);
          }
        } else {
          constexpr int kCols = 128 / sizeof(OutT);
          for (int c = group; c < p.block_n / kCols; c += 2) {
            const int col0 = n0 + c * kCols;
            if (col0 >= q.n) break;
            tile_free();
#pragma unroll
            for (int h = 0; h < kCols / 32; ++h) {
              float v[32];
              load32(c * kCols + h * 32, v);
              stage_put<OutT>(tile, lane, h, v);
            }
            stage_flush<OutT>(&q.out[0], q.out_ptr[0], q.out_ld[0], q.tma_out[0], tile, tile_addr, m0, col0, 0, q.m, q.n, lane);
          }
        }
      } else if constexpr (kEpi == kEpiGated) {
        constexpr int kCols = 128 / sizeof(OutT);
        const int n0 = w.nt * half_n;
        for (int c = group; c < half_n / kCols; c += 2) {
          const int col0 = n0 + c * kCols;
          if (col0 >= q.n) break;
          tile_free();
#pragma unroll
          for (int h = 0; h < kCols / 32; ++h) {
            float g[32], v[32];
            load32(c * kCols + h * 32, g);
            load32(half_n + c * kCols + h * 32, v);
            for_act(p.act, [&](auto tag) {
                constexpr int kAct = decltype(tag)::value;
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] *= gate_act<kAct>(g[j]);
            });
            stage_put<OutT>(tile, lane, h, v);
          }
          stage_flush<OutT>(&q.out[0], q.out_ptr[0], q.out_ld[0], q.tma_out[0], tile, tile_addr, m0, col0, 0, q.m, q.n, lane);
          // the projections themselves, for the backward pass: read again, so that no thread holds three rows
          for (int i = 1; i <= 2; ++i) {
            if (q.out_ptr[i] == nullptr) continue;
            tile_free();
#pragma unroll
            for (int h = 0; h < kCols / 32; ++h) {
              float v[32];
              load32((i - 1) * half_n + c * kCols + h * 32, v);
              stage_put<OutT>(tile, lane, h, v);
            }
            stage_flush<OutT>(&q.out[i], q.out_ptr[i], q.out_ld[i], q.tma_out[i], tile, tile_addr, m0, col0, 0, q.m, q.n, lane);
          }
        }
      } else if constexpr (kEpi == kEpiGatedGrad) {
        constexpr int kCols = 128 / sizeof(OutT);
        const int n0 = w.nt * p.block_n;
        for (int c = group; c < p.block_n / kCols; c += 2) {
          const int col0 = n0 + c * kCols;
          if (col0 >= q.n) break;
#pragma unroll 1
          for (int i = 0; i < 3; ++i) {
            tile_free();
#pragma unroll 1
            for (int h = 0; h < kCols / 32; ++h) {
              float dh[32], g[32], up[32];
              load_row32<OutT>(q.gate, q.aux_ld, row, col0 + h * 32, q.m, q.n, g);
              if (i != 1) load_row32<OutT>(q.up, q.aux_ld, row, col0 + h * 32, q.m, q.n, up);
              if (i != 2) load32(c * kCols + h * 32, dh);
              for_act(p.act, [&](auto tag) {
                constexpr int kAct = decltype(tag)::value;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  float a, da;
                  gate_act_grad<kAct>(g[j], a, da);
                  dh[j] = i == 0 ? dh[j] * up[j] * da : (i == 1 ? dh[j] * a : a * up[j]);
                }
              });
              stage_put<OutT>(tile, lane, h, dh);
            }
            stage_flush<OutT>(&q.out[i], q.out_ptr[i], q.out_ld[i], q.tma_out[i], tile, tile_addr, m0, col0, 0, q.m, q.n, lane);
          }
        }
      } else {
        // 8-bit products: the scale of this lane's row, the scales (and bias) of 32 columns through a
        // few bytes of shared memory, read back as broadcasts
        constexpr int kCols = 128 / sizeof(OutT);
        constexpr bool kGated = kEpi == kEpiScaledGated;
        const float rs = row < q.m ? __ldg(p.row_scale + row) : 0.0f;
        const int width = kGated ? half_n : p.block_n;
        const int n0 = w.nt * width;
        for (int c = group; c < width / kCols; c += 2) {
          const int col0 = n0 + c * kCols;
          if (col0 >= q.n) break;
          tile_free();
#pragma unroll
          for (int h = 0; h < kCols / 32; ++h) {
            const int cl = col0 + h * 32 + lane;
            const bool in = cl < q.n;
            scales[lane] = in ? __ldg(p.col_scale + cl) : 0.0f;
            if constexpr (kGated) scales[32 + lane] = in ? __ldg(p.col_scale2 + cl) : 0.0f;
            else scales[64 + lane] = (in && p.bias != nullptr) ? __ldg(p.bias + cl) : 0.0f;
            __syncwarp();
            float v[32];
            load32(c * kCols + h * 32, v);
            if constexpr (kGated) {
              float up[32];
              load32(half_n + c * kCols + h * 32, up);
              for_act(p.act, [&](auto tag) {
                constexpr int kAct = decltype(tag)::value;
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  v[j] = gate_act<kAct>(v[j] * (rs * scales[j])) * (up[j] * (rs * scales[32 + j]));
              });
            } else {
              for_act(p.act, [&](auto tag) {
                constexpr int kAct = decltype(tag)::value;
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = gate_act<kAct>(fmaf(v[j], rs * scales[j], scales[64 + j]));
              });
            }
            __syncwarp();
            stage_put<OutT>(tile, lane, h, v);
          }
          stage_flush<OutT>(&q.out[0], q.out_ptr[0], q.out_ld[0], q.tma_out[0], tile, tile_addr, m0, col0, 0, q.m, q.n, lane);
        }
      }
      }
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(tempty_bar(acc), 0));
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
    if (lane == 0) ptx::tma_store_wait_all<0>();
  }

  // ---------------------------------------------------------------- teardown ---
  __syncwarp();
  if (*abort_flag) {
    // give loads that are still in flight towards this CTA's shared memory time to land
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000) { }
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_arrive_release();
  ptx::cluster_wait_acquire();
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_2cta(tmem_base, kTmemCols);
  }
}

constexpr int kNarrowTailBytes = 256 + kNarrowEpiWarps * 96 * 4;     // barriers, then the column scales
inline size_t narrow_pair_smem_bytes(int block_n, int num_stages) {
  return 1024 + static_cast<size_t>(num_stages) * (kNarrowABytes + block_n / 2 * 128) +
         kNarrowEpiWarps * kNarrowTile + kNarrowTailBytes;
}

// ------------------------------------------------------------- K-split reduction ---
// Partial products of up to four problems of one launch, added in slice order and rounded once.
struct NarrowReduceItem {
  const float* partials;       // [slices][rows][ld]
  void* out;                   // [rows, cols], row stride out_ld
  long long ld, slice, out_ld;
  int rows, cols, slices, first_block;
};
struct NarrowReduceParams {
  NarrowReduceItem it[kNarrowMaxProblems];
  int count;
};
constexpr int kReduceCols = 4;                     // columns per thread
template <typename T>
__global__ void __launch_bounds__(256) narrow_reduce_kernel(const __grid_constant__ NarrowReduceParams p) {
  int i = 0;
  while (i + 1 < p.count && static_cast<int>(blockIdx.x) >= p.it[i + 1].first_block) ++i;
  const NarrowReduceItem& q = p.it[i];
  const int per_row = (q.cols + kReduceCols - 1) / kReduceCols;
  const long long idx = static_cast<long long>(blockIdx.x - q.first_block) * 256 + threadIdx.x;
  const long long r = idx / per_row;
  if (r >= q.rows) return;
  const int c = static_cast<int>(idx - r * per_row) * kReduceCols;
  const float* src = q.partials + r * q.ld + c;    // ld is a multiple of 4: aligned, and the padding is readable
  float4 s = *reinterpret_cast<const float4*>(src);
  for (int k = 1; k < q.slices; ++k) {
    const float4 t = *reinterpret_cast<const float4*>(src + k * q.slice);
    s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
  }
  T* dst = static_cast<T*>(q.out) + r * q.out_ld + c;
  const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j < q.cols) dst[j] = static_cast<T>(v[j]);
}

// ------------------------------------------------------------------- row packing ---
// Copies rows that TMA cannot address (a base or a row stride that is no multiple of 16 bytes) into a
// buffer whose rows are.  Every destination word is put together from the two aligned source words it
// straddles, so reads and writes are whole 32-bit words whatever the offset.
struct PackItem {
  const uint8_t* src;
  uint8_t* dst;
  long long src_pitch, dst_pitch;    // bytes; dst_pitch a multiple of 16
  int rows, row_bytes, first_block;
};
constexpr int kMaxPack = 8;
struct PackParams {
  PackItem it[kMaxPack];
  int count;
};
constexpr int kPackWords = 4 * 256;                  // destination words of one block (rows are not shared)
__global__ void __launch_bounds__(256) pack_rows_kernel(const __grid_constant__ PackParams p) {
  int i = 0;
  while (i + 1 < p.count && static_cast<int>(blockIdx.x) >= p.it[i + 1].first_block) ++i;
  const PackItem& q = p.it[i];
  const int words = static_cast<int>(q.dst_pitch >> 2);
  const long long total = static_cast<long long>(q.rows) * words;
  const long long base = static_cast<long long>(blockIdx.x - q.first_block) * kPackWords + threadIdx.x;
  const uintptr_t last = (reinterpret_cast<uintptr_t>(q.src) + (q.rows - 1) * q.src_pitch + q.row_bytes - 1) & ~uintptr_t(3);
#pragma unroll
  for (int k = 0; k < kPackWords / 256; ++k) {
    const long long idx = base + k * 256;
    if (idx >= total) break;
    const long long r = idx / words;
    const int w = static_cast<int>(idx - r * words);
    uint32_t v = 0;
    if (w * 4 < q.row_bytes) {
      const uintptr_t s = reinterpret_cast<uintptr_t>(q.src) + r * q.src_pitch + w * 4;
      const uintptr_t lo = s & ~uintptr_t(3);
      // words that hold at least one byte of the matrix: the aligned word below an allocation's first
      // byte, or the one that ends past its last, lies in the same 4-byte word as that byte
      const uint32_t a = *reinterpret_cast<const uint32_t*>(lo);
      const uint32_t b = (lo + 4 <= last) ? *reinterpret_cast<const uint32_t*>(lo + 4) : 0u;
      v = __funnelshift_r(a, b, static_cast<uint32_t>(s & 3) * 8);
      const int left = q.row_bytes - w * 4;
      if (left < 4) v &= (1u << (left * 8)) - 1u;
    }
    *reinterpret_cast<uint32_t*>(q.dst + r * q.dst_pitch + w * 4) = v;
  }
}

}  // namespace fnn
