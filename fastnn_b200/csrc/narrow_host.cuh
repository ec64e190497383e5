// Host side of the gated feed-forward block and the 8-bit products: argument checks, the plan of each
// launch, workspace layout, tensor maps.  Included once, by fastnn_api.cu.
#pragma once

namespace {

constexpr size_t kSkinnyMinSmem = 73 * 1024;
constexpr size_t kSkinnySmem = 115712;     // half of an SM's 228 KiB, less the 1 KiB reserved per CTA
constexpr int kDefaultClusters = 74;       // CTA pairs of a B200, for size queries without a device

struct DType {
  int code;            // FASTNN_B200_F32 / F16 / BF16, or -1: signed 8-bit
  int bytes;
  int kind;            // fnn::kKind*
  CUtensorMapDataType map;
};
bool dtype_of(int code, DType* d) {
  switch (code) {
    case FASTNN_B200_F32: *d = DType{code, 4, fnn::kKindTf32, CU_TENSOR_MAP_DATA_TYPE_FLOAT32}; return true;
    case FASTNN_B200_F16: *d = DType{code, 2, fnn::kKindF16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16}; return true;
    case FASTNN_B200_BF16: *d = DType{code, 2, fnn::kKindF16, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16}; return true;
    default: return false;
  }
}
const DType kInt8 = {-1, 1, fnn::kKindI8, CU_TENSOR_MAP_DATA_TYPE_UINT8};

bool gate_act_ok(int act) {
  return act == FASTNN_B200_ACT_NONE || act == FASTNN_B200_ACT_RELU || act == FASTNN_B200_ACT_GELU ||
         act == FASTNN_B200_ACT_SILU;
}

enum MapSwizzle : uint32_t { kSwz128 = 0, kSwz128Atom32 = 1, kSwz64 = 2 };
// Tensor map of a row-major [d1, d0] matrix (x `d2` slices), zero outside.
bool encode_narrow(CUtensorMap* map, const DType& t, const void* base, uint64_t d0, uint64_t d1, uint64_t d2,
                   uint64_t pitch, uint64_t slice, uint32_t box0, uint32_t box1, MapSwizzle swz) {
  const EncodeTiledFn encode = g_encode.load(std::memory_order_acquire);
  if (encode == nullptr) return false;
  MapKey key;
  std::memset(&key, 0, sizeof(key));
  key.base = base;
  key.d[0] = d0; key.d[1] = d1; key.d[2] = d2;
  key.s[0] = pitch; key.s[1] = slice;
  key.box[0] = box0; key.box[1] = box1; key.box[2] = 1;
  key.kind = 16u + 4u * static_cast<uint32_t>(t.map) + swz;
  if (map_cache_get(key, map)) return true;
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {pitch, slice};
  cuuint32_t box[3] = {box0, box1, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = encode(map, t.map, 3, const_cast<void*>(base), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swz == kSwz64 ? CU_TENSOR_MAP_SWIZZLE_64B
                            : (swz == kSwz128Atom32 ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B : CU_TENSOR_MAP_SWIZZLE_128B),
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) map_cache_put(key, *map);
  return r == CUDA_SUCCESS;
}

// A launch that may be placed while the kernel before it is finishing (the kernels wait for it before they
// touch global memory).
template <typename... Params, typename... Args>
int launch_dependent(void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream,
                     const Args&... args) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = tunables().pdl ? 1 : 0;
  FNN_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args...));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return 0;
}

// A row-major matrix as a call gives it; `ld` in elements.
struct Mat {
  const void* p;
  long long ld;
  int rows, cols;
};
inline long long round_up(long long v, long long to) { return (v + to - 1) / to * to; }
inline bool rows_addressable(const void* p, long long ld, int bytes) {
  return aligned16(p) && ((ld * bytes) & 15) == 0 && ld * bytes < (1ll << 40);
}

// Carves a call's workspace.  A dry one only adds up, which is how the size queries work: both
// run the same code, so they cannot disagree.
struct Carver {
  uint8_t* base;
  size_t bytes;
  bool dry;
  size_t used = 0;
  void* take(size_t want) {
    void* p = dry || base == nullptr ? nullptr : base + used;
    used += (want + 255) & ~size_t(255);
    return p;
  }
  // Whether the caller's buffer holds what was taken; asked once everything is, before the first launch.
  bool fits() const {
    if (used <= bytes && (used == 0 || (base != nullptr && aligned16(base)))) return true;
    std::fprintf(stderr, "fastnn_b200: a workspace of %zu bytes on a 16-byte boundary is needed, %zu were given at %p\n",
                 used, bytes, static_cast<void*>(base));
    return false;
  }
};

struct Packer {
  fnn::PackParams p;
  long long blocks = 0;
  bool too_large = false;
  Packer() { std::memset(&p, 0, sizeof(p)); }
  // m as TMA can address it: itself, or a copy in the workspace with rows padded to 16 bytes
  Mat fit(Carver& ws, const Mat& m, int bytes, bool pack) {
    if (!pack) return m;
    const long long pitch = round_up(1ll * m.cols * bytes, 16);
    Mat out{ws.take(static_cast<size_t>(pitch) * m.rows), pitch / bytes, m.rows, m.cols};
    if (!ws.dry) {
      fnn::PackItem& it = p.it[p.count++];
      it.src = static_cast<const uint8_t*>(m.p);
      it.dst = static_cast<uint8_t*>(const_cast<void*>(out.p));
      it.src_pitch = m.ld * bytes;
      it.rows = m.rows;
      it.row_bytes = m.cols * bytes;
      it.by_vecs = fnn::fast_div(static_cast<int>(pitch >> 4));
      it.first_block = static_cast<int>(blocks);
      const long long vecs = m.rows * (pitch >> 4);
      if (vecs > 0x7fffffffll - 256 * fnn::kPackVecs) too_large = true;      // 32 GiB of one operand
      blocks += (vecs + 256 * fnn::kPackVecs - 1) / (256 * fnn::kPackVecs);
    }
    return out;
  }
  int launch(cudaStream_t s) {
    if (too_large || blocks > 0x7fffffffll) return -1;
    if (blocks == 0) return 0;
    return launch_dependent(fnn::pack_rows_kernel, static_cast<unsigned>(blocks), 256, 0, s, p);
  }
};

// One product of a launch before its maps are made.
struct NarrowTask {
  Mat a[2], b[2];            // as stored; second pair optional (rows = 0), or b[1] = the up weight
  bool a_mn = false, b_mn = false;
  int m = 0, n = 0, k = 0, k2 = 0;
  void* out[3] = {nullptr, nullptr, nullptr};
  long long out_ld[3] = {0, 0, 0};
  const void* aux[2] = {nullptr, nullptr};     // kEpiGatedGrad: gate and up
  long long aux_ld = 0;
  // plan
  int full = 0, split = 1, kb_per_split = 0, num_kb1 = 0, num_kb = 0;   // whole tiles; slices of the others
  float* partials = nullptr;
};

struct NarrowPlan {
  int block_n;
};

// Tile width and K split of a launch: the least time of the busiest CTA pair, in SM clocks.  Units go
// round robin over the pairs, so their sums are exact; what a unit takes is a model of measured parts:
// clocks of a 128-byte k-block by tile width (512 columns: two MMA groups over one A tile, the fewest
// bytes an SM takes in per product; 128 and less are bound by the loads), the drain of an accumulator
// (under the next main loop, except a wide tile's, of which a part shows), the pipeline's fill, and for a
// K split the reduction's launch and bytes.
inline bool epi_gated(int epi) { return epi == fnn::kEpiGated || epi == fnn::kEpiScaledGated; }
struct PlanChoice {
  int block_n, len;          // len: k-blocks of a unit, at most
  bool keep_full;            // a problem's whole waves of tiles stay uncut, only its last tiles are split
};
inline int tiles_of(const NarrowTask& t, int bn, int epi) {
  return ceil_div(t.m, 256) * ceil_div(t.n, epi_gated(epi) ? bn / 2 : bn);
}
PlanChoice choose_narrow(const NarrowTask* t, int count, int kblock, int clusters, int epi, bool may_split,
                         int want_bn, int want_split) {
  int max_kb = 1;
  for (int i = 0; i < count; ++i)
    if (t[i].num_kb > max_kb) max_kb = t[i].num_kb;
  double best = 1e300;
  int best_bn = 256, best_len = max_kb;
  bool best_keep = false;
  // a CTA's half of an MN-major B tile is whole 128-byte chunks of N
  int min_bn = epi_gated(epi) ? 128 : 64;
  for (int i = 0; i < count; ++i)
    if (t[i].b_mn && min_bn < 2 * kblock) min_bn = 2 * kblock;
  const int max_bn = epi == fnn::kEpiGatedGrad ? 256 : 512;
  for (int bn = min_bn; bn <= max_bn; bn *= 2) {
    if (want_bn >= min_bn && want_bn <= max_bn && bn != want_bn) continue;
    const double per_kb = bn == 512 ? 1130.0 : (bn == 256 ? 620.0 : (bn == 128 ? 465.0 : 410.0));
    // a tile's fixed part, and for 256 accumulator columns: a plain store is memory traffic, the others
    // mostly arithmetic
    static const double kDrain[5] = {1000.0, 2200.0, 13500.0, 6500.0, 3500.0};        // by kEpi*
    const double drain = 1500.0 + kDrain[epi] * bn / 256.0;
    for (int parts = 1; parts <= (may_split ? 64 : 1); parts += parts < 8 ? 1 : (parts < 16 ? 2 : 8)) {
      const int len = ceil_div(max_kb, parts);                  // k-blocks of a unit, at most
      if (parts > 1 && len < 4) break;
      if (may_split && want_split > 0 && parts != want_split) continue;
      for (int keep = 0; keep < (parts > 1 ? 2 : 1); ++keep) {
        double most = 0.0, partial = 0.0;
        double whole[fnn::kNarrowMaxProblems], part[fnn::kNarrowMaxProblems];
        long long full[fnn::kNarrowMaxProblems], units[fnn::kNarrowMaxProblems];
        auto clocks = [&](int kb) {
          const double main = kb * per_kb;
          return (main > drain ? main : drain) + 300.0 + (bn == 512 ? 0.3 * drain : 0.0);
        };
        for (int i = 0; i < count; ++i) {
          const int split = ceil_div(t[i].num_kb, len);
          const long long tiles = tiles_of(t[i], bn, epi);
          full[i] = split == 1 ? tiles : (keep ? tiles / clusters * clusters : 0);
          units[i] = full[i] + (tiles - full[i]) * split;
          whole[i] = clocks(t[i].num_kb);
          part[i] = clocks(ceil_div(t[i].num_kb, split));
          if (split > 1) partial += 4.0 * 256 * bn * (tiles - full[i]) * split;
        }
        // units go round robin: those u in [first, first + units) with u % clusters == c are pair c's
        for (int c = 0; c < clusters; ++c) {
          double sum = 0.0;
          long long first = 0;
          for (int i = 0; i < count; ++i) {
            const long long lo = (c - first + clusters) % clusters;
            auto below = [&](long long n) { return lo < n ? (n - lo + clusters - 1) / clusters : 0; };
            const long long mine = below(full[i]);
            sum += mine * whole[i] + (below(units[i]) - mine) * part[i];
            first = (first + units[i]) % clusters;
          }
          if (sum > most) most = sum;
        }
        // partial sums are written and read once, at about half the cost while they stay in L2
        const double reduce = partial > 0.0 ? 5000.0 + 2.0 * partial / (partial < 48e6 ? 6000.0 : 3400.0) : 0.0;
        const double cost = most + drain + reduce;
        if (cost < best) { best = cost; best_bn = bn; best_len = len; best_keep = keep != 0; }
      }
    }
  }
  return PlanChoice{best_bn, best_len, best_keep};
}

// The choice walks some ten thousand combinations; programs repeat a handful of shapes, so answers are
// remembered by shape.
NarrowPlan plan_narrow(NarrowTask* t, int count, int kblock, int clusters, int epi, bool may_split) {
  struct Slot {
    int key[24];
    PlanChoice choice;
    bool valid;
  };
  constexpr int kSlots = 512;
  static Slot memo[kSlots];
  static std::mutex memo_mutex;
  int key[24] = {kblock, clusters, epi, may_split ? 1 : 0, count, t_policy.block_n, t_policy.split_k};
  uint64_t h = 0x9E3779B97F4A7C15ull;
  for (int i = 0; i < count; ++i) {
    t[i].num_kb1 = ceil_div(t[i].k, kblock);
    t[i].num_kb = t[i].num_kb1 + (t[i].k2 > 0 ? ceil_div(t[i].k2, kblock) : 0);
    int* q = key + 7 + 4 * i;
    q[0] = t[i].m; q[1] = t[i].n; q[2] = t[i].num_kb; q[3] = t[i].b_mn ? 1 : 0;
  }
  for (int v : key) h = (h ^ static_cast<uint32_t>(v)) * 0x100000001B3ull;
  PlanChoice c;
  {
    std::lock_guard<std::mutex> lock(memo_mutex);
    Slot& slot = memo[(h >> 24) % kSlots];
    if (!slot.valid || std::memcmp(slot.key, key, sizeof(key)) != 0) {
      slot.choice = choose_narrow(t, count, kblock, clusters, epi, may_split, t_policy.block_n, t_policy.split_k);
      std::memcpy(slot.key, key, sizeof(key));
      slot.valid = true;
    }
    c = slot.choice;
  }
  for (int i = 0; i < count; ++i) {
    const int tiles = tiles_of(t[i], c.block_n, epi);
    t[i].split = ceil_div(t[i].num_kb, c.len);
    t[i].kb_per_split = ceil_div(t[i].num_kb, t[i].split);
    t[i].split = ceil_div(t[i].num_kb, t[i].kb_per_split);
    t[i].full = t[i].split == 1 ? tiles : (c.keep_full ? tiles / clusters * clusters : 0);
    if (t[i].full == tiles) t[i].split = 1;
  }
  return NarrowPlan{c.block_n};
}

// Room for the partial sums of split tiles (of a launch without a gated epilogue).
void reserve_partials(Carver& ws, NarrowTask* t, int count, const NarrowPlan& plan) {
  for (int i = 0; i < count; ++i)
    if (t[i].split > 1)
      t[i].partials = static_cast<float*>(ws.take(sizeof(float) * 256 * static_cast<size_t>(plan.block_n) * t[i].split *
                                                  (tiles_of(t[i], plan.block_n, fnn::kEpiStore) - t[i].full)));
}

template <int N>
using NarrowKernel = void (*)(fnn::NarrowParams<N>);
// The instantiation for an operand kind, epilogue and output type; null where there is none.  Only the
// gradients' products share a launch.
template <int N>
NarrowKernel<N> pair_kernel(int kind, int epi, int out_code) {
  using namespace fnn;
  const bool bf = out_code == FASTNN_B200_BF16;
  if (kind == kKindF16) {
    if (epi == kEpiStore) return bf ? &narrow_pair_kernel<kKindF16, kEpiStore, __nv_bfloat16, N> : &narrow_pair_kernel<kKindF16, kEpiStore, __half, N>;
    if constexpr (N == 1) {
      if (epi == kEpiGated) return bf ? &narrow_pair_kernel<kKindF16, kEpiGated, __nv_bfloat16, N> : &narrow_pair_kernel<kKindF16, kEpiGated, __half, N>;
      if (epi == kEpiGatedGradDeep) return bf ? &narrow_pair_kernel<kKindF16, kEpiGatedGradDeep, __nv_bfloat16, N> : &narrow_pair_kernel<kKindF16, kEpiGatedGradDeep, __half, N>;
      if (epi == kEpiGatedGrad) return bf ? &narrow_pair_kernel<kKindF16, kEpiGatedGrad, __nv_bfloat16, N> : &narrow_pair_kernel<kKindF16, kEpiGatedGrad, __half, N>;
    }
  } else if (kind == kKindTf32) {
    if (epi == kEpiStore) return &narrow_pair_kernel<kKindTf32, kEpiStore, float, N>;
    if constexpr (N == 1) {
      if (epi == kEpiGated) return &narrow_pair_kernel<kKindTf32, kEpiGated, float, N>;
      if (epi == kEpiGatedGradDeep) return &narrow_pair_kernel<kKindTf32, kEpiGatedGradDeep, float, N>;
      if (epi == kEpiGatedGrad) return &narrow_pair_kernel<kKindTf32, kEpiGatedGrad, float, N>;
    }
  } else if constexpr (N == 1) {
    if (epi == kEpiScaled)
      return out_code == FASTNN_B200_F32 ? &narrow_pair_kernel<kKindI8, kEpiScaled, float, N>
             : (bf ? &narrow_pair_kernel<kKindI8, kEpiScaled, __nv_bfloat16, N> : &narrow_pair_kernel<kKindI8, kEpiScaled, __half, N>);
    if (epi == kEpiScaledGated)
      return out_code == FASTNN_B200_F32 ? &narrow_pair_kernel<kKindI8, kEpiScaledGated, float, N>
             : (bf ? &narrow_pair_kernel<kKindI8, kEpiScaledGated, __nv_bfloat16, N> : &narrow_pair_kernel<kKindI8, kEpiScaledGated, __half, N>);
  }
  return nullptr;
}

typedef void (*SkinnyKernel)(fnn::SkinnyParams);
// w_mn: the weights are stored [k, rows] (the gradients' products).
SkinnyKernel skinny_kernel(int kind, int epi, int out_code, bool w_mn) {
  using namespace fnn;
  const bool bf = out_code == FASTNN_B200_BF16;
  if (kind == kKindF16) {
    if (epi == kEpiStore && !w_mn) return bf ? &narrow_skinny_kernel<kKindF16, kEpiStore, __nv_bfloat16, false> : &narrow_skinny_kernel<kKindF16, kEpiStore, __half, false>;
    if (epi == kEpiStore) return bf ? &narrow_skinny_kernel<kKindF16, kEpiStore, __nv_bfloat16, true> : &narrow_skinny_kernel<kKindF16, kEpiStore, __half, true>;
    if (epi == kEpiGated && !w_mn) return bf ? &narrow_skinny_kernel<kKindF16, kEpiGated, __nv_bfloat16, false> : &narrow_skinny_kernel<kKindF16, kEpiGated, __half, false>;
    if (epi == kEpiGatedGrad && w_mn) return bf ? &narrow_skinny_kernel<kKindF16, kEpiGatedGrad, __nv_bfloat16, true> : &narrow_skinny_kernel<kKindF16, kEpiGatedGrad, __half, true>;
  } else if (kind == kKindTf32) {
    if (epi == kEpiStore) return w_mn ? &narrow_skinny_kernel<kKindTf32, kEpiStore, float, true> : &narrow_skinny_kernel<kKindTf32, kEpiStore, float, false>;
    if (epi == kEpiGated && !w_mn) return &narrow_skinny_kernel<kKindTf32, kEpiGated, float, false>;
    if (epi == kEpiGatedGrad && w_mn) return &narrow_skinny_kernel<kKindTf32, kEpiGatedGrad, float, true>;
  } else if (!w_mn) {
    if (epi == kEpiScaled)
      return out_code == FASTNN_B200_F32 ? &narrow_skinny_kernel<kKindI8, kEpiScaled, float, false>
             : (bf ? &narrow_skinny_kernel<kKindI8, kEpiScaled, __nv_bfloat16, false> : &narrow_skinny_kernel<kKindI8, kEpiScaled, __half, false>);
    if (epi == kEpiScaledGated)
      return out_code == FASTNN_B200_F32 ? &narrow_skinny_kernel<kKindI8, kEpiScaledGated, float, false>
             : (bf ? &narrow_skinny_kernel<kKindI8, kEpiScaledGated, __nv_bfloat16, false> : &narrow_skinny_kernel<kKindI8, kEpiScaledGated, __half, false>);
  }
  return nullptr;
}

// Called once per device by fastnn_cuda_init.
int narrow_init() {
  const int codes[3] = {FASTNN_B200_F32, FASTNN_B200_F16, FASTNN_B200_BF16};
  for (int kind = 0; kind <= 2; ++kind)
    for (int epi = 0; epi <= 5; ++epi)
      for (int c : codes) {
        if (auto k = pair_kernel<1>(kind, epi, c))
          FNN_CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMaxDynSmem)));
        if (auto k = pair_kernel<fnn::kNarrowMaxProblems>(kind, epi, c))
          FNN_CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMaxDynSmem)));
        for (bool mn : {false, true})
          if (SkinnyKernel k = skinny_kernel(kind, epi, c, mn))
            FNN_CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSkinnySmem)));
      }
  return 0;
}

struct NarrowLaunch {
  DType in;
  int out_code;
  int epi;
  int act = 0;
  const float* row_scale = nullptr;
  const float* col_scale = nullptr;
  const float* col_scale2 = nullptr;
  const float* bias = nullptr;
};

template <int N>
int launch_pair(DeviceState* st, const NarrowLaunch& l, const NarrowTask* t, int count, const NarrowPlan& plan,
                cudaStream_t stream) {
  using namespace fnn;
  NarrowParams<N> p;
  std::memset(&p, 0, sizeof(p));
  const bool gated = epi_gated(l.epi);
  const int kblock = 128 / l.in.bytes;
  p.groups = plan.block_n > kMaxBlockN ? 2 : 1;
  p.mma_n = plan.block_n / p.groups;
  const uint32_t half_n = p.mma_n / 2;
  DType out, f32;
  if (!dtype_of(l.out_code, &out) || !dtype_of(FASTNN_B200_F32, &f32)) return -1;
  const uint32_t out_cols = 64 / out.bytes;           // a staging tile: 32 rows of 64 bytes
  const int group_m = tunables().group_m >= 1 && tunables().group_m <= 1024 ? tunables().group_m
                      : (l.in.bytes == 1 ? 2 * kNarrowGroupM : kNarrowGroupM);    // 16 MiB of A rows at K = 4096
  bool ok = true;
  long long units = 0;
  for (int i = 0; i < count; ++i) {
    const NarrowTask& q = t[i];
    NarrowProblem& d = p.pr[i];
    d.m = q.m; d.n = q.n;
    d.tiles_m = ceil_div(q.m, 256);
    d.tiles_n = ceil_div(q.n, gated ? plan.block_n / 2 : plan.block_n);
    d.num_kb = q.num_kb; d.num_kb1 = q.num_kb1;
    d.split_k = q.split; d.kb_per_split = q.kb_per_split;
    d.first_unit = static_cast<int>(units);
    const long long tiles = 1ll * d.tiles_m * d.tiles_n;
    d.full_tiles = q.full;
    units += q.full + (tiles - q.full) * q.split;
    if (units > 0x3fffffffll) return -1;
    d.full_groups = d.tiles_m / group_m;
    const int last = d.tiles_m - d.full_groups * group_m;
    d.by_split = fast_div(d.split_k);
    d.by_group = fast_div(group_m * d.tiles_n);
    d.by_rows = fast_div(group_m);
    d.by_last = fast_div(last > 0 ? last : 1);
    d.a_mn = q.a_mn ? 1 : 0; d.b_mn = q.b_mn ? 1 : 0;
    const MapSwizzle mn_swz = l.in.kind == kKindTf32 ? kSwz128Atom32 : kSwz128;
    for (int j = 0; j < 2; ++j) {
      if (q.a[j].rows > 0)
        ok = ok && encode_narrow(&d.a[j], l.in, q.a[j].p, q.a[j].cols, q.a[j].rows, 1, q.a[j].ld * l.in.bytes,
                                 q.a[j].ld * l.in.bytes * q.a[j].rows, kblock, q.a_mn ? kblock : 128,
                                 q.a_mn ? mn_swz : kSwz128);
      if (q.b[j].rows > 0)
        ok = ok && encode_narrow(&d.b[j], l.in, q.b[j].p, q.b[j].cols, q.b[j].rows, 1, q.b[j].ld * l.in.bytes,
                                 q.b[j].ld * l.in.bytes * q.b[j].rows, kblock, q.b_mn ? kblock : half_n,
                                 q.b_mn ? mn_swz : kSwz128);
      if (q.aux[j] != nullptr)
        ok = ok && encode_narrow(&d.aux[j], out, q.aux[j], q.n, q.m, 1, q.aux_ld * out.bytes,
                                 q.aux_ld * out.bytes * q.m, out_cols, 32, kSwz64);
    }
    if (q.split > 1) {
      const uint64_t blocks = static_cast<uint64_t>(tiles - q.full) * q.split;
      ok = ok && encode_narrow(&d.partial, f32, q.partials, plan.block_n, blocks * 256, 1, plan.block_n * 4ull,
                               blocks * 256 * plan.block_n * 4ull, 16, 32, kSwz64);
    }
    for (int j = 0; j < 3; ++j) {
      if (q.out[j] == nullptr) continue;
      d.out_ptr[j] = q.out[j];
      d.out_ld[j] = q.out_ld[j];
      d.tma_out[j] = rows_addressable(q.out[j], q.out_ld[j], out.bytes) ? 1 : 0;
      if (d.tma_out[j])
        ok = ok && encode_narrow(&d.out[j], out, q.out[j], q.n, q.m, 1, q.out_ld[j] * out.bytes,
                                 q.out_ld[j] * out.bytes * q.m, out_cols, 32, kSwz64);
    }
  }
  if (!ok) return -1;
  p.count = count;
  p.total_units = static_cast<int>(units);
  // one thread issues a group's MMAs, and a stage's wait and commit cost it as much as an MMA or two: two
  // k-blocks a stage, except for wide tiles, whose two threads have twice the clocks for the same work, and
  // beside the gradient's two staging sets
  const int epi = l.epi == kEpiGatedGrad && t[0].num_kb >= kGradDeepMinKb ? kEpiGatedGradDeep : l.epi;
  const int want_kb = tunables().kb_per_stage >= 1 && tunables().kb_per_stage <= 4 ? tunables().kb_per_stage : 2;
  p.kb_per_stage = p.groups == 2 || epi == kEpiGatedGrad ? 1 : want_kb;
  const size_t stage = p.kb_per_stage * (kNarrowABytes + static_cast<size_t>(p.groups) * half_n * 128);
  const size_t fixed = narrow_fixed_bytes(epi);
  const int stages = static_cast<int>((kMaxDynSmem - fixed) / stage);
  if (stages < 1) return -1;
  p.num_stages = stages > kNarrowMaxStages ? kNarrowMaxStages : stages;
  p.group_m = group_m;
  p.act = l.act;
  p.is_bf16 = l.in.code == FASTNN_B200_BF16 ? 1 : 0;
  p.row_scale = l.row_scale; p.col_scale = l.col_scale; p.col_scale2 = l.col_scale2; p.bias = l.bias;
  p.vec_scale = aligned16(l.col_scale) && aligned16(l.col_scale2) && aligned16(l.bias) ? 1 : 0;
  p.status = st->status;
  p.spin_budget = st->spin_budget;
  const int clusters = p.total_units < st->max_clusters ? p.total_units : st->max_clusters;
  const NarrowKernel<N> k = pair_kernel<N>(l.in.kind, epi, l.out_code);
  if (k == nullptr || clusters < 1) return -1;
  // All of the SM's shared memory, whatever the stages need: the kernel takes all of tensor memory, and no
  // CTA that wants columns too may come to wait for them beside it.
  if (launch_dependent(k, 2 * clusters, epi_grad(epi) ? kNarrowThreads<kEpiGatedGrad> : kNarrowThreads<kEpiStore>, kMaxDynSmem, stream, p) != 0) return -1;
  t_last = LastCall{12, plan.block_n, t[0].split, 2 * clusters};

  NarrowReduceParams r;
  std::memset(&r, 0, sizeof(r));
  long long blocks = 0;
  for (int i = 0; i < count; ++i) {
    if (t[i].split <= 1) continue;
    NarrowReduceItem& it = r.it[r.count++];
    it.partials = t[i].partials;
    it.out = t[i].out[0];
    it.out_ld = t[i].out_ld[0];
    it.rows = t[i].m; it.cols = t[i].n; it.slices = t[i].split;
    it.first_tile = t[i].full;
    it.tiles_m = p.pr[i].tiles_m; it.tiles_n = p.pr[i].tiles_n;
    it.vec = reinterpret_cast<uintptr_t>(it.out) % (4 * out.bytes) == 0 && it.out_ld % 4 == 0 ? 1 : 0;
    it.first_block = static_cast<int>(blocks);
    blocks += (1ll * it.tiles_m * it.tiles_n - it.first_tile) * (256 / kReduceRows);
  }
  r.block_n = plan.block_n;
  r.group_m = group_m;
  if (blocks > 0) {
    if (blocks > 0x7fffffffll) return -1;
    const unsigned g = static_cast<unsigned>(blocks);
    auto* k = l.out_code == FASTNN_B200_F32 ? narrow_reduce_kernel<float>
              : (l.out_code == FASTNN_B200_BF16 ? narrow_reduce_kernel<__nv_bfloat16> : narrow_reduce_kernel<__half>);
    if (launch_dependent(k, g, 256, 0, stream, r) != 0) return -1;
  }
  return 0;
}

// Few tokens take the form with the weights on the M side, and so do a few hundred while its tiles fit the
// machine once: CTA pairs then have fewer tiles than SMs and cannot cut K under a gated epilogue (200
// tokens, 1024 x 1024 block: 12 against 18 us; 2048 x 2048: 20 / 26; 4096 x 16384, 512 tiles: 120 / 97).
// set_policy(3) and (4) force it and CTA pairs.
// The gradients' products can share a launch on CTA pairs, whose K splits have no limit and whose epilogue
// reads the saved projections ahead.  There (`grad`) this form is for tokens whose parts are kept in two,
// and for weights that are worth streaming on their own, over enough CTAs (200 tokens, 1024 x 1024: 21.9
// against 24.9 us; 59 tokens, 4085 x 14336: 281 / 306; 127 tokens,
// 3336 x 768: 27 / 44; but 140 tokens, 320 x 2496: 38 / 29, and 500 tokens, 512 x 2048: 30 / 25).
bool use_skinny(int tokens, int n, int k, int epi, bool grad) {
  if (t_policy.policy == 3 || t_policy.policy == 4) return t_policy.policy == 3;
  if (grad && tokens > fnn::kSkinnyFoldTokens) {
    const long long ctas = 1ll * ceil_div(n, 128) * ceil_div(tokens, fnn::kSkinnyTokens) * (tokens > 64 ? 4 : 8);
    const bool long_k = epi == fnn::kEpiGatedGrad && k >= 1024;      // the pairs' gated epilogue cannot split it
    if (!long_k && (tokens > 320 || 1ll * n * k < (1 << 20) || ctas < 64)) return false;
  }
  if (tokens <= fnn::kSkinnyTokens) return true;
  return tokens <= 512 && 1ll * ceil_div(n, epi_gated(epi) ? 64 : 128) * ceil_div(tokens, fnn::kSkinnyTokens) <= 256;
}

// K slices of a row tile, the CTAs of one cluster: enough for most of the SMs to have a CTA, twice that
// while every slice keeps eight k-blocks (bytes in flight against meeting costs: 8-bit 4096 x 4096, 1
// token: 13.1 / 9.1 / 7.2 / 7.5 us with 1 / 2 / 4 / 8 slices), and no more than four for many tokens,
// whose partial sums cross the cluster (1024 x 1024 block, 128 tokens: 11.7 us with four, 13.9 with eight).
int skinny_split(long long tiles, int num_kb, int n_mma) {
  int want = t_policy.split_k;
  if (want == 0) {
    want = 1;
    while (want < 8 && tiles * want < 120) want *= 2;
    if (want < 8 && num_kb / want >= 16 && tiles * want * 2 <= 296) want *= 2;
    if (n_mma > 64 && want > 4) want = 4;
  }
  int split = 8;
  while (split > 1 && (split > want || num_kb < 2 * split)) split /= 2;
  return split;
}

// Operands as launch_pair's; t.a[0] holds the tokens, t.b the weights.
// fold: see SkinnyParams.
int launch_skinny(DeviceState* st, const NarrowLaunch& l, const NarrowTask& t, bool early_w, int fold,
                  cudaStream_t stream) {
  using namespace fnn;
  SkinnyParams p;
  std::memset(&p, 0, sizeof(p));
  const bool two = l.epi == kEpiGated || l.epi == kEpiScaledGated;
  const int kblock = 128 / l.in.bytes;
  const int tile_rows = two ? 64 : 128;
  p.tokens = t.m; p.n = t.n;
  p.t_tiles = ceil_div(t.m, kSkinnyTokens);
  p.n_mma = ceil_div(ceil_div(t.m, p.t_tiles), 16) * 16;
  p.t_tiles = ceil_div(t.m, p.n_mma);
  p.num_kb1 = ceil_div(t.k, kblock);
  p.num_kb = p.num_kb1 + (t.k2 > 0 ? ceil_div(t.k2, kblock) : 0);
  const int tiles = ceil_div(t.n, tile_rows);
  p.split = skinny_split(1ll * tiles * p.t_tiles, p.num_kb, p.n_mma);
  bool ok = true;
  auto operand = [&](CUtensorMap* map, const Mat& m, uint32_t box1, MapSwizzle swz) {
    const uint64_t pitch = m.ld * l.in.bytes;
    return m.rows == 0 || encode_narrow(map, l.in, m.p, m.cols, m.rows, 1, pitch, pitch * m.rows, kblock, box1, swz);
  };
  for (int j = 0; j < 2; ++j) {
    ok = ok && operand(&p.x[j], t.a[j], p.n_mma, kSwz128);
    // t.b as launch_pair takes it: [rows, k], or [k, rows] when b_mn
    ok = ok && operand(&p.w[j], t.b[j], t.b_mn ? kblock : tile_rows,
                       t.b_mn && l.in.kind == kKindTf32 ? kSwz128Atom32 : kSwz128);
  }
  if (!ok) return -1;
  DType out;
  if (!dtype_of(l.out_code, &out)) return -1;
  for (int j = 0; j < 3; ++j) {
    p.out[j] = t.out[j];
    p.out_ld[j] = t.out_ld[j];
    p.vec_out[j] = (reinterpret_cast<uintptr_t>(t.out[j]) % (4 * out.bytes) == 0 && t.out_ld[j] % 4 == 0) ? 1 : 0;
  }
  p.aux[0] = t.aux[0]; p.aux[1] = t.aux[1]; p.aux_ld = t.aux_ld;
  p.vec_aux = (reinterpret_cast<uintptr_t>(t.aux[0]) | reinterpret_cast<uintptr_t>(t.aux[1])) % (4 * out.bytes) == 0 &&
              t.aux_ld % 4 == 0 ? 1 : 0;
  const int slice_kb = ceil_div(p.num_kb, p.split);
  const size_t stage = kNarrowABytes + static_cast<size_t>(p.n_mma) * 128;
  int stages = static_cast<int>((kSkinnySmem - skinny_smem_bytes(p.n_mma, 0)) / stage);
  if (stages > kSkinnyMaxStages) stages = kSkinnyMaxStages;
  if (stages > slice_kb) stages = slice_kb;
  const int for_partial = static_cast<int>((p.n_mma * 512 + stage - 1) / stage);    // the ring holds the partial tile
  if (stages < for_partial) stages = for_partial;
  p.num_stages = stages;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.n_mma) p.tmem_cols *= 2;
  p.early_w = early_w ? 1 : 0;
  p.fold = fold;
  p.act = l.act;
  p.is_bf16 = l.in.code == FASTNN_B200_BF16 ? 1 : 0;
  p.row_scale = l.row_scale; p.col_scale = l.col_scale; p.col_scale2 = l.col_scale2; p.bias = l.bias;
  p.status = st->status;
  p.spin_budget = st->spin_budget;
  // Tensor memory is 512 columns.  A CTA that waits for columns while its cluster waits for it, beside
  // another such, would never get them, so CTAs that fit an SM together must never want more than 512
  // together: at 73 KiB three of these share an SM, and beside the CTAs of the cluster split-K GEMM, which
  // ask for 228 KiB / (512 / columns + 1) each, no mix that fits wants more.
  size_t smem = skinny_smem_bytes(p.n_mma, stages);
  if (smem < kSkinnyMinSmem) smem = kSkinnyMinSmem;
  SkinnyKernel k = skinny_kernel(l.in.kind, l.epi, l.out_code, t.b_mn);
  if (k == nullptr || smem > kSkinnySmem) return -1;
  const long long grid = 1ll * tiles * p.t_tiles * p.split;
  if (grid > 0x7fffffffll) return -1;
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  const int epi_warps = p.n_mma <= 16 ? 4 : (p.n_mma <= 64 ? 8 : kSkinnyMaxEpiWarps);
  cfg.blockDim = dim3(32 * (2 + epi_warps), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = static_cast<unsigned>(p.split);
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = tunables().pdl ? 2 : 1;
  FNN_CUDA_OK(cudaLaunchKernelEx(&cfg, k, p));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  t_last = LastCall{13, p.n_mma, p.split, static_cast<int>(grid)};
  return 0;
}

// ------------------------------------------------------------- gated feed-forward ---
struct FfnArgs {
  DType t;
  int rows, d, f, act;
  Mat x, wg, wu, wd, dy;
  Mat gate, up;              // backward: saved; forward: outputs or null
  void* y = nullptr;
  void *dx = nullptr, *dwg = nullptr, *dwu = nullptr, *dwd = nullptr;
};

int clusters_of(const DeviceState* st) { return st != nullptr && st->max_clusters > 0 ? st->max_clusters : kDefaultClusters; }

// Forward.  With ws.dry only the workspace is added up (pack_all: as if no operand were
// addressable).
int ffn_forward(DeviceState* st, const FfnArgs& a, Carver& ws, bool pack_all, cudaStream_t s) {
  const int e = a.t.bytes;
  const bool dry = ws.dry;
  auto must_pack = [&](const Mat& m) { return dry ? pack_all || ((m.ld * e) & 15) != 0 : !rows_addressable(m.p, m.ld, e); };
  Packer pk;
  const Mat x = pk.fit(ws, a.x, e, must_pack(a.x));
  const Mat wg = pk.fit(ws, a.wg, e, must_pack(a.wg));
  const Mat wu = pk.fit(ws, a.wu, e, must_pack(a.wu));
  const Mat wd = pk.fit(ws, a.wd, e, must_pack(a.wd));
  const bool skinny1 = use_skinny(a.rows, a.f, a.d, fnn::kEpiGated, false);
  const bool skinny2 = use_skinny(a.rows, a.d, a.f, fnn::kEpiStore, false);
  // Hidden rows in two parts for up to 32 tokens, where it costs no more than the second product's tokens
  // (24 tokens, 1024 x 4096: 11.9 -> 12.5 us; 64 tokens: 13.5 -> 16.8).
  const int fold = skinny1 && skinny2 && e == 2 && a.rows <= fnn::kSkinnyFoldTokens ? a.rows : 0;
  const int h_rows = a.rows + fold;
  const long long h_ld = round_up(1ll * a.f * e, 16) / e;
  void* h = ws.take(static_cast<size_t>(h_ld) * h_rows * e);
  const int kblock = 128 / e;

  NarrowTask t1;
  t1.a[0] = x; t1.a[1] = Mat{nullptr, 0, 0, 0};
  t1.b[0] = wg; t1.b[1] = wu;
  t1.m = a.rows; t1.n = a.f; t1.k = a.d;
  t1.out[0] = h; t1.out[1] = const_cast<void*>(a.gate.p); t1.out[2] = const_cast<void*>(a.up.p);
  t1.out_ld[0] = h_ld; t1.out_ld[1] = t1.out_ld[2] = a.f;
  NarrowTask t2;
  t2.a[0] = Mat{h, h_ld, h_rows, a.f}; t2.a[1] = Mat{nullptr, 0, 0, 0};
  t2.b[0] = wd; t2.b[1] = Mat{nullptr, 0, 0, 0};
  t2.m = h_rows; t2.n = a.d; t2.k = a.f;
  t2.out[0] = a.y; t2.out_ld[0] = a.d;
  const int cl = clusters_of(st);
  NarrowPlan p1{0}, p2{0};
  if (!skinny1) p1 = plan_narrow(&t1, 1, kblock, cl, fnn::kEpiGated, false);
  if (!skinny2) {
    p2 = plan_narrow(&t2, 1, kblock, cl, fnn::kEpiStore, true);
    reserve_partials(ws, &t2, 1, p2);
  }
  if (dry) return 0;
  if (!ws.fits()) return -1;
  if (pk.launch(s) != 0) return -1;
  NarrowLaunch l{a.t, a.t.code, fnn::kEpiGated, a.act};
  if ((skinny1 ? launch_skinny(st, l, t1, false, fold, s) : launch_pair<1>(st, l, &t1, 1, p1, s)) != 0) return -1;
  l.epi = fnn::kEpiStore;
  // Wd may be read early: the launch ahead writes only h, gate and up, and lets this one start only after
  // it has itself seen everything before it finish
  return skinny2 ? launch_skinny(st, l, t2, true, fold, s) : launch_pair<1>(st, l, &t2, 1, p2, s);
}

int ffn_backward(DeviceState* st, const FfnArgs& a, Carver& ws, bool pack_all, cudaStream_t s) {
  const int e = a.t.bytes;
  const bool dry = ws.dry;
  auto must_pack = [&](const Mat& m) { return dry ? pack_all || ((m.ld * e) & 15) != 0 : !rows_addressable(m.p, m.ld, e); };
  Packer pk;
  const Mat dy = pk.fit(ws, a.dy, e, must_pack(a.dy));
  const Mat x = pk.fit(ws, a.x, e, must_pack(a.x));
  const Mat wg = pk.fit(ws, a.wg, e, must_pack(a.wg));
  const Mat wu = pk.fit(ws, a.wu, e, must_pack(a.wu));
  const Mat wd = pk.fit(ws, a.wd, e, must_pack(a.wd));
  const bool skinny1 = use_skinny(a.rows, a.f, a.d, fnn::kEpiGatedGrad, true);
  const bool skinny2 = use_skinny(a.rows, a.d, a.f, fnn::kEpiStore, true);
  // dgate, dup and h in two parts each, as the forward pass keeps its hidden rows
  const int fold = skinny1 && skinny2 && e == 2 && a.rows <= fnn::kSkinnyFoldTokens ? a.rows : 0;
  const int h_rows = a.rows + fold;
  // CTA pairs read the saved projections by TMA, with one stride for both
  const bool pack_aux = !skinny1 && (must_pack(a.gate) || must_pack(a.up));
  const Mat gate = pk.fit(ws, a.gate, e, pack_aux);
  const Mat up = pk.fit(ws, a.up, e, pack_aux);
  const long long h_ld = round_up(1ll * a.f * e, 16) / e;
  const size_t h_bytes = static_cast<size_t>(h_ld) * h_rows * e;
  void* dg = ws.take(h_bytes);
  void* du = ws.take(h_bytes);
  void* h = ws.take(h_bytes);
  const int kblock = 128 / e;
  const Mat none{nullptr, 0, 0, 0};
  // rows of the high parts, or all rows; and the low parts' rows, none without them
  auto part = [&](void* p, int first, int rows) {
    if (rows == 0) return none;
    return Mat{p == nullptr ? nullptr : static_cast<uint8_t*>(p) + static_cast<size_t>(h_ld) * first * e, h_ld, rows, a.f};
  };

  NarrowTask t1;                                   // dh = dy . Wd, never stored
  t1.a[0] = dy; t1.a[1] = none; t1.b[0] = wd; t1.b[1] = none;
  t1.b_mn = true;
  t1.m = a.rows; t1.n = a.f; t1.k = a.d;
  t1.out[0] = dg; t1.out[1] = du; t1.out[2] = h;
  for (long long& ld : t1.out_ld) ld = h_ld;
  t1.aux[0] = gate.p; t1.aux[1] = up.p; t1.aux_ld = gate.ld;

  // dx, then dWg, dWu, dWd; with low parts a second range of K adds their products
  NarrowTask g[4];
  g[0].a[0] = part(dg, 0, h_rows); g[0].a[1] = part(du, 0, h_rows); g[0].b[0] = wg; g[0].b[1] = wu;
  g[0].b_mn = true;
  g[0].m = h_rows; g[0].n = a.d; g[0].k = a.f; g[0].k2 = a.f;
  g[0].out[0] = a.dx; g[0].out_ld[0] = a.d;
  for (int i = 1; i <= 2; ++i) {
    void* d = i == 1 ? dg : du;
    g[i].a[0] = part(d, 0, a.rows); g[i].a[1] = part(d, a.rows, fold);
    g[i].b[0] = x; g[i].b[1] = fold > 0 ? x : none;
    g[i].a_mn = g[i].b_mn = true;
    g[i].m = a.f; g[i].n = a.d; g[i].k = a.rows; g[i].k2 = fold;
    g[i].out[0] = i == 1 ? a.dwg : a.dwu; g[i].out_ld[0] = a.d;
  }
  g[3].a[0] = dy; g[3].a[1] = fold > 0 ? dy : none; g[3].b[0] = part(h, 0, a.rows); g[3].b[1] = part(h, a.rows, fold);
  g[3].a_mn = g[3].b_mn = true;
  g[3].m = a.d; g[3].n = a.f; g[3].k = a.rows; g[3].k2 = fold;
  g[3].out[0] = a.dwd; g[3].out_ld[0] = a.f;
  NarrowTask* group = skinny2 ? g + 1 : g;             // the products of the last launch
  const int count = skinny2 ? 3 : 4;
  const int cl = clusters_of(st);
  NarrowPlan p1{0};
  if (!skinny1) p1 = plan_narrow(&t1, 1, kblock, cl, fnn::kEpiGatedGrad, false);
  const NarrowPlan p2 = plan_narrow(group, count, kblock, cl, fnn::kEpiStore, true);
  reserve_partials(ws, group, count, p2);
  if (dry) return 0;
  if (!ws.fits()) return -1;
  if (pk.launch(s) != 0) return -1;
  NarrowLaunch l{a.t, a.t.code, fnn::kEpiGatedGrad, a.act};
  if ((skinny1 ? launch_skinny(st, l, t1, false, fold, s) : launch_pair<1>(st, l, &t1, 1, p1, s)) != 0) return -1;
  l.epi = fnn::kEpiStore;
  // Wg and Wu may be read early, as Wd in the forward pass
  if (skinny2 && launch_skinny(st, l, g[0], true, fold, s) != 0) return -1;
  return launch_pair<fnn::kNarrowMaxProblems>(st, l, group, count, p2, s);
}

bool ffn_sizes_ok(int rows, int d, int f) { return rows >= 0 && d >= 1 && f >= 1; }

FfnArgs ffn_shape(const DType& t, int rows, int d, int f) {
  FfnArgs a;
  a.t = t; a.rows = rows; a.d = d; a.f = f; a.act = 0;
  a.x = Mat{nullptr, d, rows, d};
  a.dy = a.x;
  a.wg = Mat{nullptr, d, f, d}; a.wu = a.wg;
  a.wd = Mat{nullptr, f, d, f};
  a.gate = Mat{nullptr, f, rows, f}; a.up = a.gate;
  return a;
}

// ------------------------------------------------------------------ 8-bit products ---
struct Int8Args {
  Mat x, w, w2;              // w2: the up weight, or null
  const float *xs, *ws, *ws2, *bias;
  void* y;
  int out_code, rows, k, n, act;
  bool gated;
};

int int8_product(DeviceState* st, const Int8Args& a, Carver& ws, bool pack_all, cudaStream_t s) {
  const bool dry = ws.dry;
  auto must_pack = [&](const Mat& m) { return dry ? pack_all || (m.ld & 15) != 0 : !rows_addressable(m.p, m.ld, 1); };
  Packer pk;
  NarrowTask t;
  t.a[0] = pk.fit(ws, a.x, 1, must_pack(a.x)); t.a[1] = Mat{nullptr, 0, 0, 0};
  t.b[0] = pk.fit(ws, a.w, 1, must_pack(a.w));
  t.b[1] = a.gated ? pk.fit(ws, a.w2, 1, must_pack(a.w2)) : Mat{nullptr, 0, 0, 0};
  t.m = a.rows; t.n = a.n; t.k = a.k;
  t.out[0] = a.y; t.out_ld[0] = a.n;
  if (dry) return 0;
  if (!ws.fits()) return -1;
  if (pk.launch(s) != 0) return -1;
  NarrowLaunch l{kInt8, a.out_code, a.gated ? fnn::kEpiScaledGated : fnn::kEpiScaled, a.act};
  l.row_scale = a.xs; l.col_scale = a.ws; l.col_scale2 = a.ws2; l.bias = a.bias;
  if (use_skinny(a.rows, a.n, a.k, l.epi, false)) return launch_skinny(st, l, t, false, 0, s);
  const NarrowPlan p = plan_narrow(&t, 1, 128, clusters_of(st), l.epi, false);
  return launch_pair<1>(st, l, &t, 1, p, s);
}

// INT32 accumulators hold sums of k products of magnitude at most 128 * 128.
constexpr int kInt8MaxK = 131071;

template <typename T>
int quantize_launch(const void* x, long long ld, int8_t* q, float* scale, int rows, int cols, cudaStream_t s) {
  using namespace fnn;
  const int v = 16 / static_cast<int>(sizeof(T));
  const bool vec = rows_addressable(x, ld, sizeof(T)) && cols % v == 0 && (reinterpret_cast<uintptr_t>(q) & (v - 1)) == 0;
  const T* src = static_cast<const T*>(x);
  // rows that a warp holds whole take a warp each, longer ones a block, and so do a few rows, whose loads a
  // block has in flight all at once (1 row of 4096: 1.4 against 2.9 us)
  const bool shorter = cols <= 32 * kQuantHeld * v;
  const bool warp = shorter || (vec && rows >= kQuantManyRows && cols <= 32 * kQuantHeldLong * v);
  const int per = kQuantThreads / 32;
  const int grid = warp ? (rows + per - 1) / per : rows;
  auto* k = quantize_rows_kernel<T, kQuantThreads, false, kQuantHeld>;
  if (vec) k = !warp ? quantize_rows_kernel<T, kQuantThreads, true, kQuantHeld>
                     : (shorter ? quantize_rows_kernel<T, 32, true, kQuantHeld> : quantize_rows_kernel<T, 32, true, kQuantHeldLong>);
  else if (warp) k = quantize_rows_kernel<T, 32, false, kQuantHeld>;
  return launch_dependent(k, static_cast<unsigned>(grid), kQuantThreads, 0, s, src, ld, q, scale, rows, cols);
}

}  // namespace

extern "C" size_t fastnn_b200_gated_ffn_workspace(int dtype, int rows, int d_model, int d_ff, int backward,
                                                  int unaligned) {
  DType t;
  if (!dtype_of(dtype, &t) || !ffn_sizes_ok(rows, d_model, d_ff) || rows == 0) return 0;
  Carver ws{nullptr, 0, true};
  const FfnArgs a = ffn_shape(t, rows, d_model, d_ff);
  if (backward) ffn_backward(current_state(), a, ws, unaligned != 0, nullptr);
  else ffn_forward(current_state(), a, ws, unaligned != 0, nullptr);
  return ws.used;
}

extern "C" int fastnn_b200_gated_ffn_forward(int dtype, const void* x, long long ld_x, const void* w_gate,
                                             const void* w_up, const void* w_down, void* y, void* gate, void* up,
                                             int rows, int d_model, int d_ff, int act, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  DType t;
  if (!dtype_of(dtype, &t) || !ffn_sizes_ok(rows, d_model, d_ff) || !gate_act_ok(act) || ld_x < d_model) return -1;
  if ((gate == nullptr) != (up == nullptr)) return -1;
  if (rows == 0) return 0;
  if (x == nullptr || w_gate == nullptr || w_up == nullptr || w_down == nullptr || y == nullptr) return -1;
  DeviceState* st = current_state();
  if (st == nullptr) return -1;
  FfnArgs a = ffn_shape(t, rows, d_model, d_ff);
  a.act = act;
  a.x.p = x; a.x.ld = ld_x;
  a.wg.p = w_gate; a.wu.p = w_up; a.wd.p = w_down;
  a.gate.p = gate; a.up.p = up;
  a.y = y;
  Carver ws{static_cast<uint8_t*>(workspace), workspace_bytes, false};
  return ffn_forward(st, a, ws, false, static_cast<cudaStream_t>(stream));
}

extern "C" int fastnn_b200_gated_ffn_backward(int dtype, const void* dy, long long ld_dy, const void* x, long long ld_x,
                                              const void* gate, const void* up, const void* w_gate, const void* w_up,
                                              const void* w_down, void* dx, void* dw_gate, void* dw_up, void* dw_down,
                                              int rows, int d_model, int d_ff, int act, void* workspace,
                                              size_t workspace_bytes, void* stream) {
  DType t;
  if (!dtype_of(dtype, &t) || !ffn_sizes_ok(rows, d_model, d_ff) || !gate_act_ok(act)) return -1;
  if (ld_x < d_model || ld_dy < d_model) return -1;
  if (dw_gate == nullptr || dw_up == nullptr || dw_down == nullptr) return -1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {                                   // no tokens: the weights' gradients are zero
    const size_t bytes = static_cast<size_t>(d_model) * d_ff * t.bytes;
    void* outs[3] = {dw_gate, dw_up, dw_down};
    for (void* o : outs) FNN_CUDA_OK(cudaMemsetAsync(o, 0, bytes, s));
    return 0;
  }
  if (dy == nullptr || x == nullptr || gate == nullptr || up == nullptr || w_gate == nullptr || w_up == nullptr ||
      w_down == nullptr || dx == nullptr)
    return -1;
  DeviceState* st = current_state();
  if (st == nullptr) return -1;
  FfnArgs a = ffn_shape(t, rows, d_model, d_ff);
  a.act = act;
  a.x.p = x; a.x.ld = ld_x;
  a.dy.p = dy; a.dy.ld = ld_dy;
  a.wg.p = w_gate; a.wu.p = w_up; a.wd.p = w_down;
  a.gate.p = gate; a.up.p = up;
  a.dx = dx; a.dwg = dw_gate; a.dwu = dw_up; a.dwd = dw_down;
  Carver ws{static_cast<uint8_t*>(workspace), workspace_bytes, false};
  return ffn_backward(st, a, ws, false, s);
}

extern "C" int fastnn_b200_quantize_rows(int dtype, const void* x, long long ld_x, signed char* q, float* scale,
                                         int rows, int cols, void* stream) {
  DType t;
  if (!dtype_of(dtype, &t) || rows < 0 || cols < 1 || ld_x < cols) return -1;
  if (rows == 0) return 0;
  if (x == nullptr || q == nullptr || scale == nullptr || current_state() == nullptr) return -1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == FASTNN_B200_F32) return quantize_launch<float>(x, ld_x, q, scale, rows, cols, s);
  if (dtype == FASTNN_B200_F16) return quantize_launch<__half>(x, ld_x, q, scale, rows, cols, s);
  return quantize_launch<__nv_bfloat16>(x, ld_x, q, scale, rows, cols, s);
}

namespace {
int int8_entry(Int8Args a, void* workspace, size_t workspace_bytes, void* stream) {
  DType t;
  if (!dtype_of(a.out_code, &t) || a.rows < 0 || a.k < 1 || a.n < 1 || a.k > kInt8MaxK || !gate_act_ok(a.act)) return -1;
  if (a.rows == 0) return 0;
  if (a.x.p == nullptr || a.w.p == nullptr || a.xs == nullptr || a.ws == nullptr || a.y == nullptr) return -1;
  if (a.gated && (a.w2.p == nullptr || a.ws2 == nullptr)) return -1;
  DeviceState* st = current_state();
  if (st == nullptr) return -1;
  Carver ws{static_cast<uint8_t*>(workspace), workspace_bytes, false};
  return int8_product(st, a, ws, false, static_cast<cudaStream_t>(stream));
}
Int8Args int8_shape(int rows, int k, int n, bool gated) {
  Int8Args a;
  std::memset(static_cast<void*>(&a), 0, sizeof(a));
  a.x = Mat{nullptr, k, rows, k};
  a.w = Mat{nullptr, k, n, k};
  a.w2 = a.w;
  a.rows = rows; a.k = k; a.n = n; a.gated = gated;
  return a;
}
}  // namespace

extern "C" size_t fastnn_b200_int8_workspace(int rows, int in_features, int out_features, int gated, int unaligned) {
  if (rows < 1 || in_features < 1 || out_features < 1) return 0;
  Carver ws{nullptr, 0, true};
  int8_product(current_state(), int8_shape(rows, in_features, out_features, gated != 0), ws, unaligned != 0, nullptr);
  return ws.used;
}

extern "C" int fastnn_b200_int8_linear_forward(const signed char* xq, const float* x_scale, const signed char* wq,
                                               const float* w_scale, const float* bias, void* y, int out_dtype,
                                               int rows, int in_features, int out_features, int act, void* workspace,
                                               size_t workspace_bytes, void* stream) {
  Int8Args a = int8_shape(rows, in_features, out_features, false);
  a.x.p = xq; a.xs = x_scale; a.w.p = wq; a.ws = w_scale; a.bias = bias;
  a.y = y; a.out_code = out_dtype; a.act = act;
  return int8_entry(a, workspace, workspace_bytes, stream);
}

extern "C" int fastnn_b200_int8_gated_forward(const signed char* xq, const float* x_scale, const signed char* wq_gate,
                                              const float* gate_scale, const signed char* wq_up, const float* up_scale,
                                              void* h, int out_dtype, int rows, int in_features, int out_features,
                                              int act, void* workspace, size_t workspace_bytes, void* stream) {
  Int8Args a = int8_shape(rows, in_features, out_features, true);
  a.x.p = xq; a.xs = x_scale; a.w.p = wq_gate; a.ws = gate_scale; a.w2.p = wq_up; a.ws2 = up_scale;
  a.y = h; a.out_code = out_dtype; a.act = act;
  return int8_entry(a, workspace, workspace_bytes, stream);
}
