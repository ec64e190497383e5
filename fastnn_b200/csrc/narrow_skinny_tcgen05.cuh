// The same products for few tokens (decoding): the weight's rows on the tensor core's M side.
//
//   out[t, r] = epilogue( sum_k x[t, k] * W[r, k] )         W stored [r, k], or [k, r] (the gradients')
//
// With up to 128 tokens the time is that of reading the weights once, so the form is chosen for bytes in
// flight and for even shares of them; a few hundred are cut into equal tiles of at most 128, whose CTAs
// stand side by side in the grid and meet the weights in L2.  A CTA takes 128 rows of W (a gated product: 64 rows of the gate's
// weight and the same 64 of the up projection's) and one slice of K, and streams them through a ring of
// TMA stages; the tokens are the MMA's N (rounded up to 16, rows past the last one read as zero), so one
// tcgen05.mma per 32 bytes of K covers all of them and the tensor core is never what is waited for.
// The slices of a row tile are the CTAs of one cluster: each leaves its accumulator in its own shared
// memory as [token][row], and after a cluster barrier the CTAs add the slices in ascending order over
// distributed shared memory, apply the epilogue and write -- no workspace, no second kernel, the same
// bits every time.  A CTA asks for at most half of an SM, so that a CTA's start and end lie under its
// neighbour's stream, and so that the next kernel's CTAs find room while this one's last are running.
//
// Between the two products of a block of at most 32 tokens the hidden rows are kept as a sum of two
// 16-bit values, h = hi + lo: the second product takes both as tokens of their own and adds their results,
// at no weight byte more, so that the only rounding of the block that counts is its output's.  (With many
// tokens that would be twice the tensor work; there h is rounded once.)
//
// Measured: 1 token through a bf16 block of 4096 x 16384 in 67 us, 6.0 TB/s of weights (0.91 of the copy rate);
// 24 tokens, 1024 x 4096 in 12.5 us, of which the bytes are 3.9 and the rest two launches' start, cluster
// meeting and end; 57 tokens, 8-bit gated 4096 x 11009 in 23.5 us (14.1 of bytes).
#pragma once
#include "narrow_gemm_tcgen05.cuh"

namespace fnn {

constexpr int kSkinnyTokens = 128;                  // tokens of a tile, at most
constexpr int kSkinnyFoldTokens = 32;               // tokens whose hidden rows are kept in two parts; twice that fits a tile
// Producer, MMA issuer, and four to sixteen warps that drain the accumulator and apply the epilogue: at
// 128 tokens and a short K the epilogue is most of a CTA's life, with a few tokens more warps only start
// and meet later.
constexpr int kSkinnyMaxEpiWarps = 16;
constexpr int kSkinnyMaxThreads = 32 * (2 + kSkinnyMaxEpiWarps);
constexpr int kSkinnyMaxStages = 8;
constexpr int kSkinnyBarBytes = 256;

struct SkinnyParams {
  CUtensorMap w[2], x[2];    // [1]: the up weight of a gated product, or a second K range of both operands
  void* out[3];              // as NarrowProblem: the product, and for a gated one optionally gate and up
  long long out_ld[3];
  int vec_out[3];            // rows may be written four columns at a time
  const void* aux[2];        // kEpiGatedGrad: the saved gate and up projections
  long long aux_ld;
  int vec_aux;
  int tokens, n;             // n: columns of one output
  int t_tiles;               // token tiles
  int n_mma;                 // tokens of a tile, a multiple of 16
  int num_kb, num_kb1, split, num_stages, tmem_cols;    // num_kb1: k-blocks of the first range
  int fold;                  // > 0: a gated epilogue writes the low parts of its outputs this many rows on, a
                             // plain one adds the rows this far on to its own
  int early_w;               // the weights may be read before the kernel ahead of this one has finished
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
__device__ __forceinline__ void mma_narrow_1cta(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                                uint32_t accumulate) {
  if constexpr (kKind == kKindF16)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
                 "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
                 : "memory");
  else if constexpr (kKind == kKindI8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
                 "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
                 : "memory");
  else
    mma_tf32_1cta(tmem_d, desc_a, desc_b, idesc, accumulate);
}
}  // namespace ptx

// Four sums over the slices of one token's consecutive rows, in slice order.
template <int kKind>
__device__ __forceinline__ void skinny_sum(const uint8_t* own, uint32_t local, int split, float (&v)[4]) {
  if (split == 1) {
    const uint4 t = *reinterpret_cast<const uint4*>(own);
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = kKind == kKindI8 ? static_cast<float>(static_cast<int>(w[j])) : __uint_as_float(w[j]);
  } else if constexpr (kKind == kKindI8) {
    int s[4] = {0, 0, 0, 0};
#pragma unroll 4
    for (int r = 0; r < split; ++r) {
      const float4 t = ptx::ld_shared_cluster_f4(ptx::mapa_shared(local, static_cast<uint32_t>(r)));
      s[0] += __float_as_int(t.x); s[1] += __float_as_int(t.y); s[2] += __float_as_int(t.z); s[3] += __float_as_int(t.w);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = static_cast<float>(s[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = 0.0f;
#pragma unroll 4
    for (int r = 0; r < split; ++r) {
      const float4 t = ptx::ld_shared_cluster_f4(ptx::mapa_shared(local, static_cast<uint32_t>(r)));
      v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
    }
  }
}

template <typename T>
__device__ __forceinline__ void skinny_put(void* out, long long ld, int vec, int t, int c, int n, const float (&v)[4]) {
  T* dst = static_cast<T*>(out) + static_cast<long long>(t) * ld + c;
  if (vec && c + 4 <= n) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < n) dst[j] = static_cast<T>(v[j]);
  }
}

// Four values of a saved projection's row.
template <typename T>
__device__ __forceinline__ void skinny_get(const void* src, long long ld, int vec, int t, int c, int n, float (&v)[4]) {
  const T* at = static_cast<const T*>(src) + static_cast<long long>(t) * ld + c;
  if (vec && c + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(at));
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(at));
      const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
      v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c + j < n ? static_cast<float>(at[j]) : 0.0f;
  }
}

// v as a 16-bit value, in v's place the rest: nothing to add to an overflow or a NaN.
template <typename T>
__device__ __forceinline__ void skinny_rest(float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float hi = static_cast<float>(static_cast<T>(v[j]));
    v[j] = isfinite(hi) ? v[j] - hi : 0.0f;
  }
}

template <int kKind, int kEpi, typename OutT, bool kWMn>
__global__ void __launch_bounds__(kSkinnyMaxThreads, 2) narrow_skinny_kernel(const __grid_constant__ SkinnyParams p) {
  using K = NarrowKind<kKind>;
  constexpr bool kTwo = kEpi == kEpiGated || kEpi == kEpiScaledGated;
  constexpr int kRows = kTwo ? 64 : 128;              // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int epi_warps = static_cast<int>(blockDim.x >> 5) - 2;
  const uint32_t x_bytes = static_cast<uint32_t>(p.n_mma) * 128u;
  const uint32_t stage_bytes = kNarrowABytes + x_bytes;       // x_bytes is a multiple of 2048
  const uint32_t bar_base = smem_base + p.num_stages * stage_bytes;
  uint8_t* bar_gen = smem_gen + (bar_base - smem_base);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 64u + 8u * s; };
  const uint32_t done_bar = bar_base + 128u;
  const uint32_t tmem_slot = bar_base + 136u;
  volatile uint32_t* tmem_slot_gen = reinterpret_cast<volatile uint32_t*>(bar_gen + 136);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_gen + 140);

  const int slice = static_cast<int>(blockIdx.x) % p.split;   // = rank in the cluster
  const int unit = static_cast<int>(blockIdx.x) / p.split;
  const int r0 = unit / p.t_tiles * kRows;
  const int t0 = unit % p.t_tiles * p.n_mma;
  const int kb0 = static_cast<int>(static_cast<long long>(slice) * p.num_kb / p.split);
  const int kb1 = static_cast<int>(static_cast<long long>(slice + 1) * p.num_kb / p.split);

  auto load_w = [&](int kb, int s, uint64_t pol) {
    const uint32_t sa = smem_base + s * stage_bytes;
    const uint32_t fb = full_bar(s);
    ptx::mbar_expect_tx(fb, stage_bytes);
    if constexpr (kTwo) {
      ptx::tma_load_3d_hint(sa, &p.w[0], fb, kb * K::kBlock, r0, 0, pol);
      ptx::tma_load_3d_hint(sa + 64 * 128, &p.w[1], fb, kb * K::kBlock, r0, 0, pol);
    } else {
      const bool second = kb >= p.num_kb1;
      const CUtensorMap* map = &p.w[second ? 1 : 0];
      const int k0 = (second ? kb - p.num_kb1 : kb) * K::kBlock;
      if constexpr (kWMn) {
#pragma unroll
        for (int c = 0; c < 128 / static_cast<int>(K::kChunkElems); ++c)
          ptx::tma_load_3d_hint(sa + c * K::kChunkBytes, map, fb, r0 + c * static_cast<int>(K::kChunkElems), k0, 0, pol);
      } else {
        ptx::tma_load_3d_hint(sa, map, fb, k0, r0, 0, pol);
      }
    }
  };
  auto load_x = [&](int kb, int s) {
    const bool second = !kTwo && kb >= p.num_kb1;
    ptx::tma_load_3d(smem_base + s * stage_bytes + kNarrowABytes, &p.x[second ? 1 : 0], full_bar(s),
                     (second ? kb - p.num_kb1 : kb) * K::kBlock, t0, 0);
  };

  int pre = 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.num_stages; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(done_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
    const uint64_t pol = ptx::make_l2_policy(3);
    pre = min(p.num_stages, kb1 - kb0);
    // weights that nothing ahead in the stream can still be writing start before that kernel has ended
    if (!p.early_w) ptx::grid_dep_wait();
    for (int i = 0; i < pre; ++i) load_w(kb0 + i, i, pol);
    if (p.early_w) ptx::grid_dep_wait();
    for (int i = 0; i < pre; ++i) load_x(kb0 + i, i);
  }
  if (warp == 1) {
    ptx::tmem_alloc_1cta(tmem_slot, static_cast<uint32_t>(p.tmem_cols));
    ptx::tmem_relinquish_1cta();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot_gen;
  // The next kernel's CTAs may come once every CTA of this grid holds its tensor memory and has seen the
  // kernels before it finish (thread 0 waited above): what the next kernel reads early is then final.
  ptx::grid_dep_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol = ptx::make_l2_policy(3);
      int stage = pre % p.num_stages;
      uint32_t phase = pre == p.num_stages ? 1u : 0u;
      for (int kb = kb0 + pre; kb < kb1; ++kb) {
        if (!narrow_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, kStatusProducerTimeout)) break;
        load_w(kb, stage, pol);
        load_x(kb, stage);
        if (++stage == p.num_stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = ptx::idesc_narrow<kKind>(128, p.n_mma, kWMn ? 1 : 0, 0, p.is_bf16);
      const uint64_t a_desc0 = narrow_desc<kKind>(smem_base, kWMn ? 1 : 0);
      constexpr uint64_t kAStep = (kWMn ? K::kMnStep : 32u) >> 4;
      const uint64_t b_desc0 = narrow_desc<kKind>(smem_base + kNarrowABytes, 0);
      const uint64_t stage_step = stage_bytes >> 4;
      int stage = 0;
      uint32_t phase = 0;
      uint32_t accumulate = 0u;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = narrow_wait(full_bar(stage), phase, abort_flag, p, kStatusMmaTimeout);
        if (!ok) break;
        const uint64_t da = a_desc0 + stage * stage_step;
        const uint64_t db = b_desc0 + stage * stage_step;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          ptx::mma_narrow_1cta<kKind>(tmem_base, da + ks * kAStep, db + ks * 2, idesc, accumulate);
          accumulate = 1u;
        }
        ptx::mma_commit_1cta(empty_bar(stage));
        if (++stage == p.num_stages) { stage = 0; phase ^= 1u; }
      }
      if (ok) ptx::mma_commit_1cta(done_bar);
    }
  } else {
    // The accumulator to shared memory as [token][row], over the ring: every stage has been consumed.
    bool ok = narrow_wait(done_bar, 0u, abort_flag, p, kStatusEpilogueTimeout);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      ptx::tc_fence_after_sync();
      const int q = warp & 3;
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
      uint32_t* part = reinterpret_cast<uint32_t*>(smem_gen) + q * 32 + lane;
      for (int c = ((warp - 2) >> 2) * 16; c < p.n_mma; c += 4 * epi_warps) {
        uint32_t r[16];
        ptx::tmem_ld_32x16(taddr + c, r);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * 128] = r[j];
      }
      ptx::tc_fence_before_sync();
    }
  }

  // Every thread of every CTA of the cluster passes both barriers, aborting or not.
  ptx::grid_dep_wait();                               // before any thread reads or writes other global data
  __syncwarp();
  ptx::cluster_arrive_release();
  ptx::cluster_wait_acquire();
  if (!*abort_flag && warp >= 2) {
    // A thread keeps its four columns and walks over the tokens; the cluster's CTAs take tokens in turn.
    constexpr int kQuads = kRows / 4;
    const int at_once = 32 * epi_warps / kQuads;               // tokens one CTA covers per step
    const int tid = static_cast<int>(threadIdx.x) - 64;
    const int r = tid % kQuads * 4;
    const int c = r0 + r;
    const int tokens = c < p.n ? min((kEpi == kEpiStore && p.fold > 0 ? p.fold : p.tokens) - t0, p.n_mma) : 0;
    float cs[4], more[4];
    if constexpr (kEpi == kEpiScaled || kEpi == kEpiScaledGated) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = c + j < p.n;
        cs[j] = in ? __ldg(p.col_scale + c + j) : 0.0f;
        if constexpr (kEpi == kEpiScaledGated) more[j] = in ? __ldg(p.col_scale2 + c + j) : 0.0f;
        else more[j] = in && p.bias != nullptr ? __ldg(p.bias + c + j) : 0.0f;
      }
    }
    // the saved projections of a token come from memory while the one before it is computed
    float g[4], gu[4];
    auto load_aux = [&](int tl) {
      if constexpr (kEpi == kEpiGatedGrad) {
        if (tl < tokens) {
          skinny_get<OutT>(p.aux[0], p.aux_ld, p.vec_aux, t0 + tl, c, p.n, g);
          skinny_get<OutT>(p.aux[1], p.aux_ld, p.vec_aux, t0 + tl, c, p.n, gu);
        }
      }
    };
    const int step = p.split * at_once;
    load_aux(slice * at_once + tid / kQuads);
    for (int tl = slice * at_once + tid / kQuads; tl < tokens; tl += step) {
      const int t = t0 + tl;
      const uint32_t off = static_cast<uint32_t>(tl * 128 + r) * 4u;
      float v[4], u[4];
      skinny_sum<kKind>(smem_gen + off, smem_base + off, p.split, v);
      if constexpr (kTwo) skinny_sum<kKind>(smem_gen + off + 256, smem_base + off + 256, p.split, u);
      if constexpr (kEpi == kEpiStore) {
        if (p.fold > 0) {                              // one token tile: the row is in this CTA's reach
          const uint32_t low = off + static_cast<uint32_t>(p.fold) * 512u;
          skinny_sum<kKind>(smem_gen + low, smem_base + low, p.split, u);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += u[j];
        }
      }
      if constexpr (kEpi == kEpiGated) {
        if (p.out[1] != nullptr) {
          skinny_put<OutT>(p.out[1], p.out_ld[1], p.vec_out[1], t, c, p.n, v);
          skinny_put<OutT>(p.out[2], p.out_ld[2], p.vec_out[2], t, c, p.n, u);
        }
        for_act(p.act, [&](auto tag) {
          constexpr int kAct = decltype(tag)::value;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = gate_act<kAct>(v[j]) * u[j];
        });
        if (p.fold > 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) u[j] = v[j];
          skinny_rest<OutT>(u);
          skinny_put<OutT>(p.out[0], p.out_ld[0], p.vec_out[0], t + p.fold, c, p.n, u);
        }
      } else if constexpr (kEpi == kEpiGatedGrad) {
        // v is dh: dgate = dh * up * act'(gate), dup = dh * act(gate), h = act(gate) * up
        float o[3][4], here[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) { here[j] = g[j]; u[j] = gu[j]; }
        load_aux(tl + step);
        for_act(p.act, [&](auto tag) {
          constexpr int kAct = decltype(tag)::value;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float a, da;
            gate_act_grad<kAct>(here[j], a, da);
            o[0][j] = v[j] * u[j] * da;
            o[1][j] = v[j] * a;
            o[2][j] = a * u[j];
          }
        });
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          skinny_put<OutT>(p.out[i], p.out_ld[i], p.vec_out[i], t, c, p.n, o[i]);
          if (p.fold > 0) {
            skinny_rest<OutT>(o[i]);
            skinny_put<OutT>(p.out[i], p.out_ld[i], p.vec_out[i], t + p.fold, c, p.n, o[i]);
          }
        }
      } else if constexpr (kEpi != kEpiStore) {
        const float rs = __ldg(p.row_scale + t);
        for_act(p.act, [&](auto tag) {
          constexpr int kAct = decltype(tag)::value;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (kEpi == kEpiScaledGated)
              v[j] = gate_act<kAct>(v[j] * (rs * cs[j])) * (u[j] * (rs * more[j]));
            else
              v[j] = gate_act<kAct>(fmaf(v[j], rs * cs[j], more[j]));
          }
        });
      }
      if constexpr (kEpi != kEpiGatedGrad) skinny_put<OutT>(p.out[0], p.out_ld[0], p.vec_out[0], t, c, p.n, v);
    }
  }
  __syncwarp();
  ptx::cluster_arrive_release();                      // no CTA leaves while its shared memory is being read
  ptx::cluster_wait_acquire();

  if (*abort_flag) {
    const long long began = clock64();
    while (clock64() - began < 2000000) { }
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_1cta(tmem_base, static_cast<uint32_t>(p.tmem_cols));
  }
}

inline size_t skinny_smem_bytes(int n_mma, int num_stages) {
  return 1024 + static_cast<size_t>(num_stages) * (kNarrowABytes + n_mma * 128) + kSkinnyBarBytes;
}

}  // namespace fnn
