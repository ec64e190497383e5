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
// What bounds it: with many tokens the 1 kW power cap (8192 x 4096 x 16384 in bf16: the block's forward
// 1.38 PFLOP/s over 0.3 s, 1.53 in a burst, where cuBLAS's products of these shapes alone run at 1.30-1.37;
// backward 1.25; 8-bit 2.3-2.5 Pop/s).  Which tile: 256 x 512 (two MMA groups over one A tile) where K is deep,
// since at 256 x 256 an SM has to take in 64 bytes a clock, all that it can (2.64 ms against 2.40); 256 x 256
// where the epilogue of a short K has to hide under the next tile.  With a short K (the character model's
// block, K = 256) the epilogue: 1.9 us a 256-column tile gated, 2.9 in 8 bits, 8.2 for the gradient's, whose
// 48 MB of saved and formed rows a wave of tiles are 5.9 TB/s of memory traffic.
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
  kEpiScaledGated = 4,// C = act(gate * row_scale * col_scale) * (up * row_scale * col_scale2)
  kEpiGatedGradDeep = 5  // CTA pairs: kEpiGatedGrad with less staging and deeper stages
};
constexpr bool epi_grad(int epi) { return epi == kEpiGatedGrad || epi == kEpiGatedGradDeep; }
// Activations of this file's epilogues (the public codes, kActSilu beyond the GEMM epilogue's own).
constexpr int kActSilu = 5;

// Epilogue warps, four for each TMEM lane quadrant: what an epilogue waits for (tensor memory, staging
// tiles, fixed latencies) is covered by other warps, and with two for each quadrant a tile's drain took
// 1.5 to 2 times as long (7.2 against 4 k clocks for 256 columns of 8-bit products).  The gradient
// epilogue is bound by its memory traffic and has two with more tiles each.
template <int kEpi>
constexpr int kEpiWarps = kEpi == kEpiGatedGrad || kEpi == kEpiGatedGradDeep ? 8 : 16;
template <int kEpi>
constexpr int kNarrowThreads = 32 * (kEpiWarps<kEpi> + 4);    // + two producers and two MMA issuers
constexpr int kNarrowMaxProblems = 4;
constexpr int kNarrowMaxStages = 8;
constexpr int kNarrowABytes = 128 * 128;             // 128 rows x 128 bytes of K
constexpr int kNarrowBarBytes = 512;
constexpr int kNarrowGroupM = 8;                     // tile rows of a rasterisation group: 2048 rows
// A staging tile is 32 rows of 64 bytes (in the 64-byte swizzle): 32 columns of 16 bits, 16 of 32.  An
// epilogue warp owns one; a gradient epilogue's owns two sets of (gate, up, h),
// or two tiles where K is deep.
constexpr int kTile = 32 * 64;
template <typename T>
constexpr int kTileCols = 64 / static_cast<int>(sizeof(T));
// Staging of one epilogue warp. kEpiGatedGrad has two sets of (gate, up, h) tiles, so that a chunk's loads
// run under the chunk before it. kEpiGatedGradDeep has two tiles, and h goes through the first one once that
// is stored: a chunk's loads and stores then wait for one another, which a long main loop covers, and the
// room holds three stages of two k-blocks instead of four of one (256 columns).
// Whole backward in bf16, two sets / deep, in turn on one GPU: 8192 tokens, d 4096, f 16384 5663 / 5515 us;
// 2048 tokens of it 1401 / 1372; 8192 tokens, d 2048, f 8192 1429 / 1403; d 1536 (24 k-blocks), f 6144 907 / 907.
// Below that the two sets win (both forms in one kernel with a branch): d 1280, f 5120 644 / 648; d 1024,
// f 8192 831 / 849; d 256, f 1024 51.5 / 58.4.  They are kernels of their own because that branch cost 18
// registers, and the 8192-token d 256 case 53.9 in place of 52.1 us.
template <int kEpi>
constexpr int kStagingWarp = kEpi == kEpiGatedGrad ? 6 * kTile : (kEpi == kEpiGatedGradDeep ? 2 * kTile : kTile);
constexpr int kGradDeepMinKb = 24;

// n / d for 0 <= n < 2^31 without a division (Granlund and Montgomery): every epilogue warp decodes every
// tile, and four integer divisions were a third of a short-K tile's instructions.
struct FastDiv {
  uint32_t mul, shift, d;
};
inline FastDiv fast_div(int d) {
  FastDiv f;
  f.d = static_cast<uint32_t>(d);
  f.shift = 0;
  while ((1ull << f.shift) < f.d) ++f.shift;
  f.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.shift) - f.d)) / f.d + 1);
  return f;
}
__device__ __forceinline__ int div_by(int n, const FastDiv& f) {
  return static_cast<int>((__umulhi(static_cast<uint32_t>(n), f.mul) + static_cast<uint32_t>(n)) >> f.shift);
}

struct NarrowProblem {
  CUtensorMap a[2], b[2];      // [1]: second K range (C = A0.B0 + A1.B1), or the up weight of a gated product
  CUtensorMap out[3];
  CUtensorMap aux[2];          // kEpiGatedGrad: the saved gate and up projections
  void* out_ptr[3];            // the outputs for stores TMA cannot make; null: not wanted
  long long out_ld[3];         // their row strides in elements
  int tma_out[3];              // outputs are TMA-addressable
  int m, n;                    // n: columns of ONE output
  int tiles_m, tiles_n;
  int num_kb, num_kb1;         // 128-byte k-blocks in all, and those of the first operand pair
  int full_tiles;              // tiles done whole; the others in split_k slices of K, whose FP32 sums go to
  int split_k, kb_per_split;   // partial: one 256 x block_n block for each (tile, slice), stacked
  CUtensorMap partial;
  int first_unit;
  int full_groups;             // rasterisation groups of group_m tile rows
  FastDiv by_split, by_group, by_rows, by_last;   // K slices; tiles of a full group; tile rows of a group, of the last
  int a_mn, b_mn;              // operand stored with M (N) contiguous
};

template <int kProblems>
struct NarrowParams {
  NarrowProblem pr[kProblems];
  int count, total_units;
  int groups;                  // 256-column MMA groups of a tile: 2 for wide tiles
  int mma_n;                   // columns of one group's MMA; a tile has groups * mma_n
  int num_stages, group_m;
  int kb_per_stage;            // k-blocks of a stage: two where the MMA thread's issue would set the pace
  int act, is_bf16;
  const float* row_scale;
  const float* col_scale;
  const float* col_scale2;
  const float* bias;
  int vec_scale;               // the column vectors are 16-byte aligned
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
// These run over every output of a tile while the next tile's main loop wants to start, so they are
// written for few instructions: the special-function unit's 2^x and 1/x (a unit or two in the last
// place of FP32) and no range handling beyond what the formulas need.
constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + e^-x).  e^-x overflows to infinity below x = -88, where 1 / inf = 0 stands for e^x < 1e-38.
__device__ __forceinline__ float sigmoid_fast(float x) {
  return ptx::rcp_approx(1.0f + ptx::ex2_approx(x * -kLog2e));
}

// The normal distribution's Phi(x) = 0.5 erfc(-x / sqrt 2), and e^(-x^2 / 2) beside it.  erfc by
// Abramowitz & Stegun 7.1.26, erfc(z) = (a1 t + ... + a5 t^5) e^(-z^2) with t = 1 / (1 + 0.3275911 z),
// z >= 0: off by at most 1.5e-7.  The tail is computed as itself, not as 1 - erf, so Phi keeps that
// accuracy's size for negative x.  About half the instructions of erff.
__device__ __forceinline__ float normal_cdf(float x, float& gauss) {
  const float t = ptx::rcp_approx(fmaf(fabsf(x), 0.3275911f * 0.7071067811865475f, 1.0f));
  gauss = ptx::ex2_approx(x * x * (-0.5f * kLog2e));
  float q = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  q = fmaf(t, q, 0.5f * 1.421413741f);
  q = fmaf(t, q, 0.5f * -0.284496736f);
  q = fmaf(t, q, 0.5f * 0.254829592f);
  q *= t * gauss;
  return x >= 0.0f ? 1.0f - q : q;
}

template <int kAct>
__device__ __forceinline__ float gate_act(float x) {
  if constexpr (kAct == kActRelu) return x < 0.0f ? 0.0f : x;        // NaN stays NaN
  else if constexpr (kAct == kActGelu) { float e; return x * normal_cdf(x, e); }
  else if constexpr (kAct == kActSilu) return x * sigmoid_fast(x);
  else return x;
}
// act(x) and its derivative together
template <int kAct>
__device__ __forceinline__ void gate_act_grad(float x, float& a, float& da) {
  if constexpr (kAct == kActRelu) {
    a = x < 0.0f ? 0.0f : x;
    da = x > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (kAct == kActGelu) {
    float e;
    const float cdf = normal_cdf(x, e);
    a = x * cdf;
    da = fmaf(x * 0.3989422804014327f, e, cdf);
  } else if constexpr (kAct == kActSilu) {
    const float s = sigmoid_fast(x);
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

// Byte offset of 16-byte unit j of row r in a staging tile: unit j at j ^ ((r >> 1) & 3).
__device__ __forceinline__ uint32_t tile_unit(int r, int j) {
  return static_cast<uint32_t>(r * 64 + ((j ^ ((r >> 1) & 3)) << 4));
}

// 8 columns of this lane's row to and from a staging tile: the j-th eight (a unit of 16 bits, two of 32).
template <typename T>
__device__ __forceinline__ void tile_get8(const uint8_t* tile, int lane, int j, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 f = *reinterpret_cast<const float4*>(tile + tile_unit(lane, 2 * j + i));
      v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
    }
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(tile + tile_unit(lane, j));
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(q[i]);
      v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void tile_put8(uint8_t* tile, int lane, int j, const float* v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<float4*>(tile + tile_unit(lane, 2 * j + i)) =
          make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
    *reinterpret_cast<uint4*>(tile + tile_unit(lane, j)) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}
// 16 columns, the h-th sixteen
template <typename T>
__device__ __forceinline__ void tile_put16(uint8_t* tile, int lane, int h, const float (&v)[16]) {
  tile_put8<T>(tile, lane, 2 * h, v);
  tile_put8<T>(tile, lane, 2 * h + 1, v + 8);
}

// A staging tile to output rows [m0, m0 + 32), columns from col0: one TMA store, which clips at the
// matrix's edges, or row by row (row strides that are no multiple of 16 bytes, unaligned bases).
template <typename T>
__device__ __forceinline__ void tile_flush(const CUtensorMap* map, void* out, long long ld, int tma, uint8_t* tile,
                                           uint32_t tile_addr, int m0, int col0, int m, int n, int lane) {
  if (tma) {
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      ptx::tma_store_3d(map, tile_addr, col0, m0, 0);
      ptx::tma_store_commit();
    }
  } else {
    __syncwarp();
    const int rows = min(32, m - m0);
    constexpr int kPer = 16 / static_cast<int>(sizeof(T));
    // lanes over the columns of as many rows at once as fit the warp
    constexpr int kRowsAtOnce = 32 / kTileCols<T>;
    const int cl = lane % kTileCols<T>;
    T* dst = static_cast<T*>(out) + static_cast<long long>(m0) * ld + col0 + cl;
    if (col0 + cl < n)
      for (int r = lane / kTileCols<T>; r < rows; r += kRowsAtOnce)
        dst[r * ld] = *reinterpret_cast<const T*>(tile + tile_unit(r, cl / kPer) + (cl % kPer) * sizeof(T));
    __syncwarp();
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
  int pr, slot, mt, nt, kb0, kb1;      // slot: block of partial sums, -1 for a whole tile
};
template <int kProblems>
__device__ __forceinline__ NarrowUnit narrow_unit(const NarrowParams<kProblems>& p, int u) {
  NarrowUnit w;
  int i = 0;
  if constexpr (kProblems > 1)
    while (i + 1 < p.count && u >= p.pr[i + 1].first_unit) ++i;
  const NarrowProblem& q = p.pr[i];
  int t = u - q.first_unit;
  w.pr = i;
  int tile = t;
  w.slot = -1;
  w.kb0 = 0;
  w.kb1 = q.num_kb;
  if (t >= q.full_tiles) {
    w.slot = t - q.full_tiles;
    const int k = div_by(w.slot, q.by_split);
    const int slice = w.slot - k * q.split_k;
    tile = q.full_tiles + k;
    w.kb0 = slice * q.kb_per_split;
    w.kb1 = min(q.num_kb, w.kb0 + q.kb_per_split);
  }
  const int g = div_by(tile, q.by_group);
  const int r = tile - g * static_cast<int>(q.by_group.d);
  const FastDiv& rows = g < q.full_groups ? q.by_rows : q.by_last;
  w.nt = div_by(r, rows);
  w.mt = g * p.group_m + r - w.nt * static_cast<int>(rows.d);
  return w;
}

template <int kKind, int kEpi, typename OutT, int kProblems>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNarrowThreads<kEpi>, 1)
narrow_pair_kernel(const __grid_constant__ NarrowParams<kProblems> p) {
  using K = NarrowKind<kKind>;
  constexpr bool kTwoB = kEpi == kEpiGated || kEpi == kEpiScaledGated;
  constexpr bool kDeep = kEpi == kEpiGatedGradDeep;      // see kStagingWarp
  constexpr bool kGrad = kEpi == kEpiGatedGrad || kDeep;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const int cluster_id = blockIdx.x >> 1;
  const int num_clusters = gridDim.x >> 1;
  const int groups = p.groups;
  const int half_n = p.mma_n >> 1;                       // B columns of one MMA group this CTA loads
  const int block_n = groups * p.mma_n;
  const uint32_t half_bytes = static_cast<uint32_t>(half_n) * 128u;
  const uint32_t kb_bytes = kNarrowABytes + static_cast<uint32_t>(groups) * half_bytes;
  const uint32_t stage_bytes = static_cast<uint32_t>(p.kb_per_stage) * kb_bytes;
  const uint32_t staging_base = smem_base + p.num_stages * stage_bytes;
  constexpr int kWarps = kEpiWarps<kEpi>;
  constexpr int kMmaWarpB = 2 + kWarps;                  // second MMA-issuing warp (wide tiles)
  constexpr int kLoadWarpB = 3 + kWarps;                 // loads B while warp 0 loads A
  const uint32_t bar_base = staging_base + kWarps * kStagingWarp<kEpi>;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 64u + 8u * s; };
  auto tfull_bar = [&](int a) { return bar_base + 128u + 8u * a; };
  auto tempty_bar = [&](int a) { return bar_base + 144u + 8u * a; };
  const uint32_t tmem_slot = bar_base + 160u;
  uint8_t* bar_gen = smem_gen + (bar_base - smem_base);
  volatile uint32_t* tmem_slot_gen = reinterpret_cast<volatile uint32_t*>(bar_gen + 160);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_gen + 168);
  auto aux_bar = [&](int ew, int set) { return bar_base + 256u + 16u * ew + 8u * set; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.num_stages; ++s) {
      ptx::mbar_init(full_bar(s), 2);          // one arrive.expect_tx from each CTA's producer
      ptx::mbar_init(empty_bar(s), groups);    // one commit per MMA-issuing thread
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(tfull_bar(a), 1);
      ptx::mbar_init(tempty_bar(a), 2 * kWarps);
    }
    if constexpr (kGrad)
      for (int i = 0; i < 2 * kWarps; ++i) ptx::mbar_init(bar_base + 256u + 8u * i, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
    ptx::prefetch_tensormap(&p.pr[0].a[0]);
    ptx::prefetch_tensormap(&p.pr[0].b[kTwoB ? rank : 0]);
    ptx::prefetch_tensormap(&p.pr[0].out[0]);
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
  // Launched as a programmatic dependent: everything above overlaps the end of the kernel before, whose
  // writes are complete only from here on.  The next kernel may in turn be placed on SMs this grid leaves
  // (never beside one of its CTAs, which take a whole SM's shared memory and tensor memory).
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();

  if (warp == 0 || warp == kLoadWarpB) {
    // ------------------------------------------------------------ producers ---
    // One thread loads A, another B: one thread's wait, announcement and boxes took 600 to 1000 clocks a
    // k-block, more than the tensor cores (B with two boxes a group: 985 -> 750).  What a unit's loop
    // needs is in registers; a k-block is `boxes` boxes of each group, `x_step` apart in the matrix.
    const bool for_a = warp == 0;
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t pol = ptx::make_l2_policy(3);
      const uint32_t full0 = ptx::mapa_shared(full_bar(0), 0);       // the leader's barriers
      const int n_step = kTwoB ? half_n : p.mma_n;                   // to the next group's columns
      const int my_groups = for_a ? 1 : groups;
      const int stages = p.num_stages, per_stage = p.kb_per_stage;
      const uint32_t my_base = smem_base + (for_a ? 0u : static_cast<uint32_t>(kNarrowABytes));
      uint32_t ready = 0;
      for (int u = cluster_id; u < p.total_units && ok; u += num_clusters) {
        const NarrowUnit w = narrow_unit(p, u);
        const NarrowProblem& q = p.pr[w.pr];
        // a gated tile: this CTA's columns are all gate (leader) or all up (peer) columns of the same outputs
        const int x0 = for_a ? w.mt * 256 + static_cast<int>(rank) * 128
                             : (kTwoB ? w.nt * (block_n >> 1) : w.nt * block_n + static_cast<int>(rank) * half_n);
        const bool mn = (for_a ? q.a_mn : q.b_mn) != 0;
        const int boxes = mn ? (for_a ? 128 : half_n) / static_cast<int>(K::kChunkElems) : 1;
        const CUtensorMap* map1 = for_a ? &q.a[0] : &q.b[kTwoB ? static_cast<int>(rank) : 0];
        const CUtensorMap* map2 = for_a ? &q.a[1] : &q.b[1];
        const int kb1 = w.kb1, num_kb1 = q.num_kb1;
        for (int kb = w.kb0; kb < kb1; kb += per_stage) {
          if (!ready) {
            ok = narrow_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, kStatusProducerTimeout);
            if (!ok) break;
          }
          const uint32_t fb = full0 + 8u * stage;
          uint32_t dst = my_base + stage * stage_bytes;
          const int count = min(per_stage, kb1 - kb);
          if (for_a) ptx::mbar_expect_tx_cluster(fb, count * kb_bytes);
          if (++stage == stages) { stage = 0; phase ^= 1u; }
          ready = ptx::mbar_test_wait(empty_bar(stage), phase ^ 1u);
          for (int i = kb; i < kb + count; ++i, dst += kb_bytes) {
            const bool second = !kTwoB && i >= num_kb1;
            const int k0 = (second ? i - num_kb1 : i) * K::kBlock;
            const CUtensorMap* map = second ? map2 : map1;
            if (!mn) {
              ptx::tma_load_3d_pair(dst, map, fb, k0, x0, 0, pol);
              if (my_groups == 2) ptx::tma_load_3d_pair(dst + half_bytes, map, fb, k0, x0 + n_step, 0, pol);
            } else {
              for (int g = 0; g < my_groups; ++g)
                for (int c = 0; c < boxes; ++c)
                  ptx::tma_load_3d_pair(dst + g * half_bytes + c * K::kChunkBytes, map, fb,
                                        x0 + g * n_step + c * static_cast<int>(K::kChunkElems), k0, 0, pol);
            }
          }
        }
      }
      // every release the leader's commits still owe this CTA must land before exit
      for (int i = 0; i < p.num_stages && ok; ++i) {
        ok = narrow_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, kStatusProducerTimeout);
        if (++stage == p.num_stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1 || warp == kMmaWarpB) {
    // ----------------------------------------------- MMA issuers (leader only) ---
    // One thread per MMA group.  The two accumulator slots of 256 columns hold alternate tiles of a
    // one-group launch, or the two groups of a wide tile; either way a slot is filled again as soon as
    // the epilogue has drained it, so a wide tile's first group starts while its second is being read.
    const int my_group = warp == 1 ? 0 : 1;
    if (lane == 0 && rank == 0 && my_group < groups) {
      const uint64_t stage_step = stage_bytes >> 4;
      const uint64_t kb_step = kb_bytes >> 4;
      uint32_t ready = 0;
      int stage = 0;
      uint32_t phase = 0;
      int slot = my_group;
      uint32_t slot_phase = 0;
      bool ok = true;
      for (int u = cluster_id; u < p.total_units && ok; u += num_clusters) {
        const NarrowUnit w = narrow_unit(p, u);
        const NarrowProblem& q = p.pr[w.pr];
        const uint32_t idesc = ptx::idesc_narrow<kKind>(256, p.mma_n, q.a_mn, q.b_mn, p.is_bf16);
        const uint64_t a_desc0 = narrow_desc<kKind>(smem_base, q.a_mn);
        const uint64_t b_desc0 = narrow_desc<kKind>(smem_base + kNarrowABytes + my_group * half_bytes, q.b_mn);
        const uint64_t a_step = (q.a_mn ? K::kMnStep : 32u) >> 4;
        const uint64_t b_step = (q.b_mn ? K::kMnStep : 32u) >> 4;
        ok = narrow_wait(tempty_bar(slot), slot_phase ^ 1u, abort_flag, p, kStatusMmaTmemTimeout);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(slot * kMaxBlockN);
        uint32_t accumulate = 0u;
        for (int kb = w.kb0; kb < w.kb1; kb += p.kb_per_stage) {
          // `ready`: the probe of this stage's barrier made a stage ago, its latency hidden behind the
          // MMAs between
          if (!ready) {
            ok = narrow_wait(full_bar(stage), phase, abort_flag, p, kStatusMmaTimeout);
            if (!ok) break;
          }
          const int count = min(p.kb_per_stage, w.kb1 - kb);
          uint64_t da = a_desc0 + stage * stage_step;
          uint64_t db = b_desc0 + stage * stage_step;
          const uint32_t freed = stage;
          if (++stage == p.num_stages) { stage = 0; phase ^= 1u; }
          ready = ptx::mbar_test_wait(full_bar(stage), phase);
          for (int i = 0; i < count; ++i, da += kb_step, db += kb_step) {
            ptx::mma_narrow_2cta<kKind>(tmem_d, da, db, idesc, accumulate);
            accumulate = 1u;
#pragma unroll
            for (int ks = 1; ks < 4; ++ks)
              ptx::mma_narrow_2cta<kKind>(tmem_d, da + ks * a_step, db + ks * b_step, idesc, 1u);
          }
          ptx::mma_commit_2cta_mask(empty_bar(freed), 3);   // the stage is free, in both CTAs
        }
        if (!ok) break;
        ptx::mma_commit_2cta_mask(tfull_bar(slot), 3);      // the accumulator is complete, in both CTAs
        if (groups == 2) slot_phase ^= 1u;
        else if (++slot == 2) { slot = 0; slot_phase ^= 1u; }
      }
    }
  } else {
    // -------------------------------------------------------------- epilogue ---
    // The warps of a TMEM lane quadrant take the column chunks of a slot in turn; a chunk fills a tile.
    const int ew = warp - 2;
    const int q4 = warp & 3;
    const int group = ew >> 2;
    constexpr int kStep = kWarps / 4;
    constexpr int kCols = kTileCols<OutT>;
    const uint32_t my_addr = staging_base + ew * kStagingWarp<kEpi>;
    uint8_t* my_gen = smem_gen + (my_addr - smem_base);
    int slot = 0;
    uint32_t slot_phase = 0;
    bool ok = true;

    // kGrad: the (gate, up) tiles of the next chunk are fetched while this one is computed
    int set = 0;
    uint32_t set_phase = 0;                                  // a bit for each set
    bool fetched = false;                                    // the current set's tiles are on their way
    auto set_addr = [&](int s) { return my_addr + s * 3 * kTile; };
    auto fetch_aux = [&](const NarrowUnit& w, int c, int s) {          // lane 0
      if constexpr (kGrad) {
        const NarrowProblem& q = p.pr[w.pr];
        const int m0 = w.mt * 256 + static_cast<int>(rank) * 128 + q4 * 32;
        const int col0 = w.nt * block_n + c * kCols;
        const uint32_t bar = aux_bar(ew, s);
        ptx::mbar_expect_tx(bar, 2 * kTile);
        ptx::tma_load_3d(set_addr(s), &q.aux[0], bar, col0, m0, 0);
        ptx::tma_load_3d(set_addr(s) + kTile, &q.aux[1], bar, col0, m0, 0);
      }
    };
    // whether chunk c of unit u exists for this warp (its rows and columns reach into the matrix)
    auto live = [&](const NarrowUnit& w, int c) {
      const NarrowProblem& q = p.pr[w.pr];
      return w.mt * 256 + static_cast<int>(rank) * 128 + q4 * 32 < q.m && w.nt * block_n + c * kCols < q.n;
    };
    if constexpr (kGrad) {
      const NarrowUnit w = narrow_unit(p, cluster_id);       // the grid has no more pairs than units
      fetched = live(w, group);
      if (fetched && lane == 0) fetch_aux(w, group, 0);
    }

    for (int u = cluster_id; u < p.total_units && ok; u += num_clusters) {
      const NarrowUnit w = narrow_unit(p, u);
      const NarrowProblem& q = p.pr[w.pr];
      const int m0 = w.mt * 256 + static_cast<int>(rank) * 128 + q4 * 32;
      const int row = m0 + lane;
      const bool rows_live = m0 < q.m;                       // warp-uniform
      for (int g = 0; g < groups && ok; ++g) {
        ok = narrow_wait(tfull_bar(slot), slot_phase, abort_flag, p, kStatusEpilogueTimeout);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q4 * 32) << 16) +
                               static_cast<uint32_t>(slot * kMaxBlockN);
        auto load16 = [&](int col, uint32_t (&r)[16]) { ptx::tmem_ld_32x16(taddr + col, r); };
        auto value = [&](uint32_t r) {
          return kKind == kKindI8 ? static_cast<float>(static_cast<int>(r)) : __uint_as_float(r);
        };
        auto tile_free = [&]() {                             // the staging tile may be overwritten
          if (lane == 0) ptx::tma_store_wait_read<0>();
          __syncwarp();
        };
        auto flush = [&](int i, int col0) {
          tile_flush<OutT>(&q.out[i], q.out_ptr[i], q.out_ld[i], q.tma_out[i], my_gen, my_addr, m0, col0, q.m, q.n, lane);
        };
        if (rows_live) {
          if constexpr (kEpi == kEpiStore) {
            const int n0 = w.nt * block_n + g * p.mma_n;
            if (w.slot >= 0) {                               // FP32 partial sums of one K slice
              for (int c = group; c < p.mma_n / 16; c += kStep) {
                const int col0 = n0 + c * 16;
                if (col0 >= q.n) break;
                uint32_t r[16];
                load16(c * 16, r);
                tile_free();
                ptx::tmem_ld_wait();
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                tile_put16<float>(my_gen, lane, 0, v);
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                  ptx::tma_store_3d(&q.partial, my_addr, g * p.mma_n + c * 16, w.slot * 256 + (m0 - w.mt * 256), 0);
                  ptx::tma_store_commit();
                }
              }
            } else {
              for (int c = group; c < p.mma_n / kCols; c += kStep) {
                const int col0 = n0 + c * kCols;
                if (col0 >= q.n) break;
                uint32_t r[kCols / 16][16];
#pragma unroll
                for (int h = 0; h < kCols / 16; ++h) load16(c * kCols + h * 16, r[h]);
                tile_free();
                ptx::tmem_ld_wait();
#pragma unroll
                for (int h = 0; h < kCols / 16; ++h) {
                  float v[16];
#pragma unroll
                  for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[h][j]);
                  tile_put16<OutT>(my_gen, lane, h, v);
                }
                flush(0, col0);
              }
            }
          } else if constexpr (kEpi == kEpiGated) {
            const int n0 = w.nt * (block_n >> 1) + g * half_n;
            for (int c = group; c < half_n / kCols; c += kStep) {
              const int col0 = n0 + c * kCols;
              if (col0 >= q.n) break;
              if (q.out_ptr[1] != nullptr) {                 // the projections themselves, for the backward pass
                for (int i = 0; i < 2; ++i) {
                  tile_free();
#pragma unroll
                  for (int h = 0; h < kCols / 16; ++h) {
                    uint32_t r[16];
                    load16(i * half_n + c * kCols + h * 16, r);
                    ptx::tmem_ld_wait();
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                    tile_put16<OutT>(my_gen, lane, h, v);
                  }
                  flush(1 + i, col0);
                }
              }
              tile_free();
#pragma unroll
              for (int h = 0; h < kCols / 16; ++h) {
                uint32_t rg[16], ru[16];
                load16(c * kCols + h * 16, rg);
                load16(half_n + c * kCols + h * 16, ru);
                ptx::tmem_ld_wait();
                float v[16];
                for_act(p.act, [&](auto tag) {
                  constexpr int kAct = decltype(tag)::value;
#pragma unroll
                  for (int j = 0; j < 16; ++j)
                    v[j] = gate_act<kAct>(__uint_as_float(rg[j])) * __uint_as_float(ru[j]);
                });
                tile_put16<OutT>(my_gen, lane, h, v);
              }
              flush(0, col0);
            }
          } else if constexpr (kGrad) {
            // dgate and dup take the places of gate and up in the set's tiles (a lane reads and writes
            // its own row), h a third tile; all three rows are addressable by construction
            const int n0 = w.nt * block_n;
            for (int c = group; c < block_n / kCols; c += kStep) {
              const int col0 = n0 + c * kCols;
              if (col0 >= q.n) break;
              uint32_t r[kCols / 16][16];
#pragma unroll
              for (int h = 0; h < kCols / 16; ++h) load16(c * kCols + h * 16, r[h]);
              uint8_t* tiles = my_gen + set * 3 * kTile;
              NarrowUnit wn = w;                             // the chunk this warp comes to next
              int cn = c + kStep;
              bool more = cn * kCols < block_n && live(wn, cn);
              if (!more && u + num_clusters < p.total_units) {
                wn = narrow_unit(p, u + num_clusters);
                cn = group;
                more = live(wn, cn);
              }
              if (lane == 0) {
                if (!kDeep || !fetched) ptx::tma_store_wait_read<0>();     // every store so far has read its tiles
                if (!fetched) fetch_aux(w, c, set);
                if (!kDeep && more) fetch_aux(wn, cn, set ^ 1);
              }
              __syncwarp();
              ok = narrow_wait(aux_bar(ew, set), (set_phase >> set) & 1u, abort_flag, p, kStatusEpilogueTimeout);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              set_phase ^= 1u << set;
              ptx::tmem_ld_wait();
              [[maybe_unused]] uint32_t kept[16];            // kDeep: this lane's row of h, as stored
              for_act(p.act, [&](auto tag) {
                constexpr int kAct = decltype(tag)::value;
#pragma unroll
                for (int j = 0; j < kCols / 8; ++j) {
                  float gv[8], uv[8], hv[8];
                  tile_get8<OutT>(tiles, lane, j, gv);
                  tile_get8<OutT>(tiles + kTile, lane, j, uv);
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    float a, da;
                    gate_act_grad<kAct>(gv[i], a, da);
                    const float dh = __uint_as_float(r[j >> 1][(j & 1) * 8 + i]);
                    hv[i] = a * uv[i];
                    gv[i] = dh * uv[i] * da;
                    uv[i] = dh * a;
                  }
                  tile_put8<OutT>(tiles, lane, j, gv);
                  tile_put8<OutT>(tiles + kTile, lane, j, uv);
                  if constexpr (!kDeep) {
                    tile_put8<OutT>(tiles + 2 * kTile, lane, j, hv);
                  } else if constexpr (sizeof(OutT) == 4) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) kept[8 * j + i] = __float_as_uint(hv[i]);
                  } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) kept[4 * j + i] = pack2<OutT>(hv[2 * i], hv[2 * i + 1]);
                  }
                }
              });
              ptx::fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                const uint32_t ta = set_addr(set);
                ptx::tma_store_3d(&q.out[0], ta, col0, m0, 0);
                ptx::tma_store_3d(&q.out[1], ta + kTile, col0, m0, 0);
                if constexpr (!kDeep) ptx::tma_store_3d(&q.out[2], ta + 2 * kTile, col0, m0, 0);
                ptx::tma_store_commit();
                if constexpr (kDeep) ptx::tma_store_wait_read<0>();
              }
              if constexpr (kDeep) {                         // h follows through the first tile
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  *reinterpret_cast<uint4*>(tiles + tile_unit(lane, j)) =
                      make_uint4(kept[4 * j], kept[4 * j + 1], kept[4 * j + 2], kept[4 * j + 3]);
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                  ptx::tma_store_3d(&q.out[2], set_addr(0), col0, m0, 0);
                  ptx::tma_store_commit();
                  ptx::tma_store_wait_read<0>();
                  if (more) fetch_aux(wn, cn, 0);
                }
              } else {
                set ^= 1;
              }
              fetched = more;
            }
          } else {
            // 8-bit products: the scale of this lane's row, and the scales (and bias) of the columns,
            // which all lanes read from the same addresses
            constexpr bool kGated = kEpi == kEpiScaledGated;
            const float rs = row < q.m ? __ldg(p.row_scale + row) : 0.0f;
            const int width = kGated ? half_n : p.mma_n;
            auto columns16 = [&](const float* src, int col0, float (&to)[16]) {
              if (src != nullptr && p.vec_scale && col0 + 16 <= q.n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float4 f = __ldg(reinterpret_cast<const float4*>(src + col0) + j);
                  to[4 * j] = f.x; to[4 * j + 1] = f.y; to[4 * j + 2] = f.z; to[4 * j + 3] = f.w;
                }
              } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) to[j] = src != nullptr && col0 + j < q.n ? __ldg(src + col0 + j) : 0.0f;
              }
            };
            const int n0 = w.nt * (kGated ? block_n >> 1 : block_n) + g * width;
            for (int c = group; c < width / kCols; c += kStep) {
              const int col0 = n0 + c * kCols;
              if (col0 >= q.n) break;
              tile_free();
#pragma unroll
              for (int h = 0; h < kCols / 16; ++h) {
                uint32_t r[16], ru[16];
                load16(c * kCols + h * 16, r);
                if constexpr (kGated) load16(half_n + c * kCols + h * 16, ru);
                float cs[16], more[16];                      // scales; the other scales, or the bias
                columns16(p.col_scale, col0 + h * 16, cs);
                columns16(kGated ? p.col_scale2 : p.bias, col0 + h * 16, more);
                ptx::tmem_ld_wait();
                float v[16];
                for_act(p.act, [&](auto tag) {
                  constexpr int kAct = decltype(tag)::value;
#pragma unroll
                  for (int j = 0; j < 16; ++j) {
                    if constexpr (kGated)
                      v[j] = gate_act<kAct>(value(r[j]) * (rs * cs[j])) * (value(ru[j]) * (rs * more[j]));
                    else
                      v[j] = gate_act<kAct>(fmaf(value(r[j]), rs * cs[j], more[j]));
                  }
                });
                tile_put16<OutT>(my_gen, lane, h, v);
              }
              flush(0, col0);
            }
          }
        }
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(tempty_bar(slot), 0));
        if (++slot == 2) { slot = 0; slot_phase ^= 1u; }
      }
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

// Shared memory beside the stages.
inline size_t narrow_fixed_bytes(int epi) {
  const int staging = epi == kEpiGatedGrad       ? kEpiWarps<kEpiGatedGrad> * kStagingWarp<kEpiGatedGrad>
                      : epi == kEpiGatedGradDeep ? kEpiWarps<kEpiGatedGradDeep> * kStagingWarp<kEpiGatedGradDeep>
                                                 : kEpiWarps<kEpiStore> * kStagingWarp<kEpiStore>;
  return 1024 + static_cast<size_t>(staging) + kNarrowBarBytes;
}

// ------------------------------------------------------------- K-split reduction ---
// The partial sums of up to four problems' split tiles, added in slice order and rounded once.
struct NarrowReduceItem {
  const float* partials;       // [tile - first_tile][slice][256][block_n]
  void* out;                   // [rows, cols], row stride out_ld
  long long out_ld;
  int rows, cols, slices, first_tile, tiles_m, tiles_n, first_block;
  int vec;                     // rows of out may be written four columns at a time
};
struct NarrowReduceParams {
  NarrowReduceItem it[kNarrowMaxProblems];
  int count, block_n, group_m;
};
constexpr int kReduceRows = 4;                     // rows of a tile one block adds up
template <typename T>
__global__ void __launch_bounds__(256) narrow_reduce_kernel(const __grid_constant__ NarrowReduceParams p) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();
  int i = 0;
  while (i + 1 < p.count && static_cast<int>(blockIdx.x) >= p.it[i + 1].first_block) ++i;
  const NarrowReduceItem& q = p.it[i];
  const int b = static_cast<int>(blockIdx.x) - q.first_block;
  const int k = b / (256 / kReduceRows);                       // split tile
  const int tile = q.first_tile + k;
  // the tile's place, as narrow_unit finds it
  const int group_sz = p.group_m * q.tiles_n;
  const int first_m = tile / group_sz * p.group_m;
  const int gm = min(q.tiles_m - first_m, p.group_m);
  const int r = tile % group_sz;
  const int row0 = b % (256 / kReduceRows) * kReduceRows;
  const int m0 = (first_m + r % gm) * 256 + row0, n0 = r / gm * p.block_n;
  const int quads = p.block_n >> 2;
  const float* src = q.partials + (static_cast<long long>(k) * q.slices * 256 + row0) * p.block_n;
  const long long slice = 256ll * p.block_n;
  for (int e = threadIdx.x; e < kReduceRows * quads; e += 256) {
    const int rr = e / quads, c = (e - rr * quads) * 4;
    if (m0 + rr >= q.rows || n0 + c >= q.cols) continue;
    const float* at = src + rr * p.block_n + c;
    float4 s = *reinterpret_cast<const float4*>(at);
    for (int j = 1; j < q.slices; ++j) {
      const float4 t = *reinterpret_cast<const float4*>(at + j * slice);
      s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
    T* dst = static_cast<T*>(q.out) + static_cast<long long>(m0 + rr) * q.out_ld + n0 + c;
    if (q.vec && n0 + c + 4 <= q.cols) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = s;
      else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + c + j < q.cols) dst[j] = static_cast<T>(v[j]);
    }
  }
}

// ------------------------------------------------------------------- row packing ---
// Copies rows that TMA cannot address (a base or a row stride that is no multiple of 16 bytes) into a
// buffer whose rows are.  A thread puts 16 destination bytes together from the two aligned 16-byte blocks
// they straddle, so reads and writes are whole vectors whatever the offset.  A block is read only if it
// holds a byte of the matrix; what else it holds lies in the same 256-byte granule of device memory.
struct PackItem {
  const uint8_t* src;
  uint8_t* dst;
  long long src_pitch;               // bytes
  int rows, row_bytes, first_block;
  FastDiv by_vecs;                   // 16-byte vectors of a destination row
};
constexpr int kMaxPack = 8;
struct PackParams {
  PackItem it[kMaxPack];
  int count;
};
constexpr int kPackVecs = 2;                         // vectors of one thread
__global__ void __launch_bounds__(256) pack_rows_kernel(const __grid_constant__ PackParams p) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch_dependents();
  int i = 0;
  while (i + 1 < p.count && static_cast<int>(blockIdx.x) >= p.it[i + 1].first_block) ++i;
  const PackItem& q = p.it[i];
  const int vecs = static_cast<int>(q.by_vecs.d);
  const int first = (static_cast<int>(blockIdx.x) - q.first_block) * 256 * kPackVecs + static_cast<int>(threadIdx.x);
  const uintptr_t last = reinterpret_cast<uintptr_t>(q.src) + static_cast<long long>(q.rows - 1) * q.src_pitch +
                         q.row_bytes - 1;            // the matrix's last byte
#pragma unroll
  for (int k = 0; k < kPackVecs; ++k) {
    const int idx = first + k * 256;
    const int r = div_by(idx, q.by_vecs);
    if (r >= q.rows) break;
    const int v = idx - r * vecs;
    const uintptr_t s = reinterpret_cast<uintptr_t>(q.src) + r * q.src_pitch + v * 16;
    const uintptr_t lo = s & ~uintptr_t(15);
    const uint32_t off = static_cast<uint32_t>(s & 15);
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (lo <= last) a = __ldg(reinterpret_cast<const uint4*>(lo));
    if (off != 0 && lo + 16 <= last) b = __ldg(reinterpret_cast<const uint4*>(lo + 16));
    // the words from the first that holds a wanted byte on
    const bool two = (off & 8) != 0, one = (off & 4) != 0;
    const uint32_t t[6] = {two ? a.z : a.x, two ? a.w : a.y, two ? b.x : a.z, two ? b.y : a.w, two ? b.z : b.x,
                           two ? b.w : b.y};
    uint32_t w[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = one ? t[j + 1] : t[j];
    const uint32_t shift = (off & 3) * 8;
    const int left = q.row_bytes - v * 16;           // bytes of the row from here on
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[j] = __funnelshift_r(w[j], w[j + 1], shift);
      const int mine = left - 4 * j;
      if (mine < 4) o[j] = mine <= 0 ? 0u : o[j] & ((1u << (mine * 8)) - 1u);
    }
    *reinterpret_cast<uint4*>(q.dst + (static_cast<long long>(r) * vecs + v) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

}  // namespace fnn
