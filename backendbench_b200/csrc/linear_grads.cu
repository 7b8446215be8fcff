// Both gradients of a linear layer y = x w^T in one launch, bf16 / f16:
//
//   dx[m, k] = sum_j g[m, j] w[j, k]        g: [M, J], the gradient of y
//   dw[j, k] = sum_m g[m, j] x[m, k]
//
// Two products of the same size: the first has few tiles with a long contraction (J), the second many with a short one (M).
// One after the other, each ends with SMs that have nothing left to do (M 4096, J 22016, K 4096: dx has 256 tiles for
// 74 pairs of CTAs, 3.5 rounds that take four); here the pairs walk the long tiles first and then fill up with the short ones.
//
// A pair of CTAs to a tile of 256 x 256 (tcgen05.mma, cta_group::2, fp32 sums in tensor memory, one rounding), loads, products
// and stores as in the other kernels here. No operand is turned: g lies along the contraction for dx and across it for dw, x and w lie across it,
// and the descriptors say so.
//
// f16 holds 2^-24 to 65504, which a gradient of the projections need not keep to although dx and dw do: there g comes twice, its rows scaled by powers
// of two for dx and its columns for dw, and the sums take the factors back before they are rounded.
//
// bf16 2048 x 8192 x 4096: 158 us, 1.74 PFLOP/s, the tensor pipe 85 % busy, which is what bounds it; 4096 x 22016 x 4096 in a loop 1073 (under the power cap),
// one product after the other 1178; 512 x 2048 x 1024 15.3 and 24.5.
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "linear_common.cuh"

namespace b200 {

namespace {

constexpr int kGradStage = 32 * 1024, kGradStages = kLinRing / kGradStage, kGradAccs = 2;
constexpr size_t kGradSmem = static_cast<size_t>(kLinRing) + kLinEpiWarps * kLinEpiBytes + 1024 /*align*/ + 256 /*barriers*/;

struct GradParams {
  int64_t M, J, K;
  int nt;                       // tiles across
  TwoParts two;                 // 0 is dx, 1 is dw
  const uint32_t* most[2];      // f16: largest magnitudes of g's rows and columns before they were scaled, as fp32 bits, or NULL
  int group_m;
};

// Groups of row blocks, the row block fastest inside one
__device__ __forceinline__ void grad_block(const GradParams& p, int part, int t, int& mb, int& nb) {
  const unsigned mt = static_cast<unsigned>(((part ? p.J : p.M) + 255) / 256), group_m = static_cast<unsigned>(p.group_m), per_group = group_m * static_cast<unsigned>(p.nt);
  const unsigned g = static_cast<unsigned>(t) / per_group, in_g = static_cast<unsigned>(t) - g * per_group, left = mt - g * group_m, gm = left < group_m ? left : group_m, n = in_g / gm;
  nb = static_cast<int>(n);
  mb = static_cast<int>(g * group_m + in_g - n * gm);
}

template <typename T>
__global__ void __launch_bounds__(kLinThreads, 1)
linear_grads(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_gt, const __grid_constant__ CUtensorMap map_x,
             T* __restrict__ dx, T* __restrict__ dw, GradParams p, uint32_t* __restrict__ status) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* epi_stage = smem + kLinRing;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kLinRing + kLinEpiWarps * kLinEpiBytes);
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(bars + 2 * kGradStages + 2 * kGradAccs);
  volatile uint32_t* abort_flag = tmem_base_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem), bar_base = smem_u32(bars);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kGradStages + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * kGradStages + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * kGradStages + kGradAccs + a); };
  const uint32_t rank = cluster_ctarank();
  const int pair = static_cast<int>(blockIdx.x >> 1);

  if (threadIdx.x == 64) {
    for (const CUtensorMap* m : {&map_g, &map_w, &map_gt, &map_x}) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kGradStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < kGradAccs; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 16);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_slot)), "r"(kGradAccs * 256) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  after_grids_before();
  constexpr bool kScaledRows = std::is_same<T, __half>::value;
  const uint32_t *const most_dx = waited(p.most[0]), *const most_dw = waited(p.most[1]);
  T *const to_dx = waited(dx), *const to_dw = waited(dw);  // (the copy engine reads, and nothing is written before)

  const int slabs_j = static_cast<int>((p.J + 63) / 64), slabs_m = static_cast<int>((p.M + 63) / 64);
  int part, tile;
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int n = 0; ok && two_parts_tile(p.two, pair, n, part, tile); ++n) {
        int mb, nb;
        grad_block(p, part, tile, mb, nb);
        const int slabs = part ? slabs_m : slabs_j;
        const int m0 = mb * 256 + static_cast<int>(rank) * 128, n0 = nb * 256 + static_cast<int>(rank) * 128;
        const CUtensorMap* map_b = part ? &map_x : &map_w;
        for (int kb = 0; kb < slabs; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, kLinWaitNs)) { ok = false; break; }
          const uint32_t a_dst = smem_base + stage * kGradStage, b_dst = a_dst + 128 * kSlabBytes;
          const uint32_t bar = map_to_cta(full_bar(stage), 0u);
          if (rank == 0u) mbar_expect_tx(full_bar(stage), 2 * kGradStage);  // both CTAs' bytes
          if (part == 0) {
            tma_load_3d_pair(a_dst, &map_g, bar, kb * 64, m0, 0);  // box [128 m][64 j]
          } else {
            tma_load_3d_pair(a_dst, &map_gt, bar, m0, kb * 64, 0);  // boxes [64 m][64 j]
            tma_load_3d_pair(a_dst + 64 * kSlabBytes, &map_gt, bar, m0 + 64, kb * 64, 0);
          }
          tma_load_3d_pair(b_dst, map_b, bar, n0, kb * 64, 0);  // boxes [64 of the contraction][64 k]
          tma_load_3d_pair(b_dst + 64 * kSlabBytes, map_b, bar, n0 + 64, kb * 64, 0);
          if (++stage == kGradStages) { stage = 0; phase ^= 1u; }
        }
      }
      // the even CTA's commits arrive here from afar: none may land after this CTA's shared memory is gone
      for (int i = 0; i < kGradStages && ok; ++i) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, kLinWaitNs)) ok = false;
        if (++stage == kGradStages) { stage = 0; phase ^= 1u; }
      }
      if (!ok) {
        *abort_flag = 1;
        if (status) atomicOr(status, B200_DEV_WAIT_TIMEOUT);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (the whole warp walks, one lane issues)
    if (rank == 0u) {
      // fp32 sums; operands' type; B across the contraction, A (dw, bit 15) as well; N >> 3, M >> 4
      constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      const uint32_t idesc0 = (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | (32u << 17) | (16u << 24);
      const uint32_t empty0 = map_to_cta(empty_bar(0), 0u), empty1 = map_to_cta(empty_bar(0), 1u);
      auto warp_wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, kLinWaitNs)) != 0; };
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int n = 0; ok && two_parts_tile(p.two, pair, n, part, tile); ++n) {
        if (!warp_wait(tempty_bar(acc), acc_phase ^ 1u)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * 256), idesc = part ? idesc0 | 1u << 15 : idesc0;
        const uint32_t a_adv = part ? 2048u : 32u, a_lbo = part ? 8192u : 16u;
        const int slabs = part ? slabs_m : slabs_j;
        for (int kb = 0; kb < slabs; ++kb) {
          if (!warp_wait(full_bar(stage), phase)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_base + stage * kGradStage, b_addr = a_addr + 128 * kSlabBytes;
          uint64_t da[4], db[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            da[k] = smem_desc(a_addr + k * a_adv, a_lbo, 1024u);
            db[k] = smem_desc(b_addr + k * 2048u, 8192u, 1024u);
          }
          const uint32_t e0 = empty0 + 8u * stage, e1 = empty1 + 8u * stage;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) tc_mma_f16_pair(d_tmem, da[k], db[k], idesc, (kb | k) != 0 ? 1u : 0u);
            tc_commit_pair(e0);
            tc_commit_pair(e1);
          }
          __syncwarp();
          if (++stage == kGradStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if (elect_one()) {
          tc_commit_pair(map_to_cta(tfull_bar(acc), 0u));
          tc_commit_pair(map_to_cta(tfull_bar(acc), 1u));
        }
        __syncwarp();
        if (++acc == kGradAccs) { acc = 0; acc_phase ^= 1u; }
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        if (status) atomicOr(status, B200_DEV_WAIT_TIMEOUT);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue: 64 columns at a time, two warps to a lane quarter
    const int q = warp & 3, half = (warp - 2) >> 2;
    unsigned char* mine = epi_stage + (warp - 2) * kLinEpiBytes;
    const bool vec = p.K % 8 == 0 && ((reinterpret_cast<uintptr_t>(to_dx) | reinterpret_cast<uintptr_t>(to_dw)) & 15u) == 0;
    const uint32_t tempty_target = map_to_cta(tempty_bar(0), 0u);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int n = 0; ok && two_parts_tile(p.two, pair, n, part, tile); ++n) {
      T* out = part ? to_dw : to_dx;
      int mb, nb;
      grad_block(p, part, tile, mb, nb);
      const int64_t r0 = static_cast<int64_t>(mb) * 256 + static_cast<int64_t>(rank) * 128 + q * 32, n0 = static_cast<int64_t>(nb) * 256 + half * 128, rows = part ? p.J : p.M;
      const int left = p.K - n0 < 128 ? static_cast<int>(p.K - n0) : 128, nrows = rows - r0 < 32 ? static_cast<int>(rows - r0) : 32;  // (0 or less: none)
      const int count = (left + 63) / 64;
      float factor = 1.f;
      if (kScaledRows && most_dx && lane < nrows) factor = row_factor((part ? most_dw : most_dx)[r0 + lane]);
      int got = 0;
      if (lane == 0) got = mbar_wait(tfull_bar(acc), acc_phase, abort_flag, kLinWaitNs) ? 1 : 0;
      got = __shfl_sync(0xffffffffu, got, 0);
      if (!got) { ok = false; break; }
      tc_fence_after();
      const uint32_t t_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * 256 + half * 128);
      T* to = out + r0 * p.K + n0;
      uint32_t r[64];
      auto fetch = [&](int i) {
        tc_ld_32x32(t_base + static_cast<uint32_t>(i * 64), r);
        tc_ld_32x32(t_base + static_cast<uint32_t>(i * 64 + 32), r + 32);
      };
      // the values are out of the registers: the next ones are on their way while these are stored, or, behind the last, the
      // accumulator goes back to the MMA warp
      auto next = [&](int i) {
        if (i + 1 < count) {
          fetch(i + 1);
          return;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty_target + 8u * acc);
      };
      if (count > 0) fetch(0);
      else next(0);
#pragma unroll 1
      for (int i = 0; i < count; ++i, to += 64) {
        const int ncols = left - i * 64 < 64 ? left - i * 64 : 64;
        float* v = reinterpret_cast<float*>(r);
        tc_ld_wait();
        if constexpr (kScaledRows) {
#pragma unroll
          for (int e = 0; e < 64; ++e) v[e] *= factor;
        }
        if (vec) {
          __syncwarp();  // what was staged has been read out
#pragma unroll
          for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(mine + lane * 128 + ((j ^ (lane & 7)) << 4)) = narrow<T>(v + j * 8);
          __syncwarp();
          next(i);
          const int j = lane & 7, row = lane >> 3;
          T* o = to + row * p.K + j * 8;
          if (j * 8 < ncols) {
#pragma unroll
            for (int k = 0; k < 32; k += 4, o += 4 * p.K)
              if (row + k < nrows) *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(mine + (row + k) * 128 + ((j ^ ((row + k) & 7)) << 4));
          }
        } else {
          if (nrows > 0) {
            lin_store<T>(v, mine, to, p.K, nrows, ncols < 32 ? ncols : 32, false, lane);
            if (ncols > 32) lin_store<T>(v + 32, mine, to + 32, p.K, nrows, ncols - 32, false, lane);
          }
          next(i);
        }
      }
      if (++acc == kGradAccs) { acc = 0; acc_phase ^= 1u; }
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      if (status) atomicOr(status, B200_DEV_WAIT_TIMEOUT);
    }
    __syncwarp();
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the shared memory goes away
    __syncthreads();
  }
  cluster_sync_all();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kGradAccs * 256) : "memory");
}

// ------------------------------------------------------------------ host side
bool encode_grad(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, bool bf16, int box_rows) {
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), 1};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(pitch * 2), static_cast<cuuint64_t>(pitch * 2) * static_cast<cuuint64_t>(rows)};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return encode_fn()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// x and w as the copy engine takes them; every tile of the other part's rows reads them once
LinOperand grad_operand(const void* base, int64_t rows, int64_t others, int64_t K, int64_t s_r) { return LinOperand{base, rows, K, s_r, 1, 2, (others + 255) / 256}; }

// us: a tile of 256 x 256, a start and its slabs
struct GradTimes : TwoTimes {
  GradTimes(int64_t M, int64_t J, int64_t K)
      : TwoTimes((M + 255) / 256 * ((K + 255) / 256), (J + 255) / 256 * ((K + 255) / 256), 1.5 + static_cast<double>((J + 63) / 64) * 0.31, 1.5 + static_cast<double>((M + 63) / 64) * 0.31) {}
};

template <typename T>
int launch_grads(const CUtensorMap* maps, void* dx, void* dw, const GradParams& p, int launches, uint32_t* status, cudaStream_t st) {
  const auto kernel = linear_grads<T>;
  static std::atomic<uint64_t> allowed{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kGradSmem));
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) { set_last_cuda_error(e); return B200_ELAUNCH; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * p.two.pairs), 1, 1);
  cfg.blockDim = dim3(kLinThreads, 1, 1);
  cfg.dynamicSmemBytes = kGradSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // (see launch_after)
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], maps[3], static_cast<T*>(dx), static_cast<T*>(dw), p, status);
  if (e != cudaSuccess) {  // (a refused cluster launch: the caller has other products)
    set_last_cuda_error(e);
    (void)cudaGetLastError();
    return B200_ELAUNCH;
  }
  return check_launch(launches);
}

}  // namespace

}  // namespace b200

using namespace b200;

namespace {
int64_t grads_need(const void* g, const void* x, const void* w, int64_t M, int64_t J, int64_t K, int64_t sgm, int64_t sxm, int64_t sxk, int64_t swj, int64_t swk, bool f16) {
  if (M < 1 || J <= 128 || K <= 64 || M > 0x7ffffeffLL || J > 0x7ffffeffLL || K > 0x7ffffeffLL || !encode_fn()) return -1;
  if (sxk != 1 || swk != 1 || !aligned16(g) || sgm < J || sgm % 8) return -1;
  const GradTimes t(M, J, K);
  if (t.tiles[0] > (1 << 29) || t.tiles[1] > (1 << 29)) return -1;  // (they are counted in 32 bits)
  // One tile to a pair is a poor way through a long contraction (28672: 140 us, where a product by itself shares it and takes 25). 1,062 sizes of 136 to 8192
  // rows that this lets through: 19 % faster than one product after the other on average, slower by more than 3 % for 38; up to 128 rows, which are half a
  // tile, 27 to 39 % faster for J up to 1400, even at 2048.
  // f16 has other products to weigh against (b200_linear_scaled), which turn dP, x and w first, 2.6e-6 us an element: 17 x 22016 x 4096 363 us with
  // them, 134 here; 1024 x 4096 x 1024 95 and 50.
  const double turned = 2.6e-6 * (static_cast<double>(J) * static_cast<double>(K) + static_cast<double>(M) * static_cast<double>(J + K));
  const double most = f16 ? 20. + turned : M <= 128 ? 10. : 20.;
  if (t.longest >= most && ((M <= 128 && !f16) || t.longest > 1.75 * t.even)) return -1;
  const int64_t need = grad_operand(x, M, J, K, sxm).packed_bytes() + grad_operand(w, J, M, K, swj).packed_bytes();
  return need ? need + 256 : 0;
}
}  // namespace

extern "C" int64_t b200_linear_grads_scratch_bytes(const void* g, const void* x, const void* w, int64_t M, int64_t J, int64_t K, int64_t sgm, int64_t sxm, int64_t sxk, int64_t swj, int64_t swk) {
  return grads_need(g, x, w, M, J, K, sgm, sxm, sxk, swj, swk, false);
}
extern "C" int64_t b200_linear_grads_scaled_scratch_bytes(const void* g, const void* x, const void* w, int64_t M, int64_t J, int64_t K, int64_t sgm, int64_t sxm, int64_t sxk, int64_t swj, int64_t swk) {
  return grads_need(g, x, w, M, J, K, sgm, sxm, sxk, swj, swk, true);
}

namespace {
// g by rows (for dx) and by columns (for dw), the same where neither is scaled (`most` is NULL)
int run_linear_grads(const void* g, const void* g_columns, const uint32_t* most, const void* x, const void* w, void* dx, void* dw, int64_t M, int64_t J, int64_t K, int64_t sgm, int64_t sxm, int64_t swj,
                     int dtype, void* scratch, int64_t scratch_bytes, uint32_t* status, void* stream) {
  if (!dx) g = g_columns;  // (the one that nobody wants need not be there)
  if (!dw) g_columns = g;
  if (!g || !g_columns || !aligned16(g_columns) || !x || !w || (!dx && !dw)) return B200_EINVAL;
  const int64_t need = grads_need(g, x, w, M, J, K, sgm, sxm, 1, swj, 1, most != nullptr);
  if (need < 0) return B200_EINVAL;
  if (need && (!scratch || scratch_bytes < need)) return B200_ESCRATCH;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LinOperand ox = grad_operand(x, M, J, K, sxm), ow = grad_operand(w, J, M, K, swj);
  // one of them alone comes from the same tiles, so that it does not depend on whether the other is wanted
  const LinOperand as_it_is{g, M, J, sgm, 1, 2, 0};
  if (!dw) ox = as_it_is;
  if (!dx) ow = as_it_is;
  int launches = 1;
  lin_pack(ox, ow, reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(scratch) + 255) & ~static_cast<uintptr_t>(255)), st, launches);
  const bool bf16 = dtype == B200_BF16;
  alignas(64) CUtensorMap maps[4];
  if (!encode_grad(&maps[0], g, M, J, sgm, bf16, 128) || !encode_grad(&maps[2], g_columns, M, J, sgm, bf16, 64)) return B200_EDRIVER;
  maps[1] = maps[3] = maps[2];
  if ((dx && !encode_grad(&maps[1], ow.base, J, K, ow.s_r, bf16, 64)) || (dw && !encode_grad(&maps[3], ox.base, M, K, ox.s_r, bf16, 64)))
    return B200_EDRIVER;
  GradParams p{};
  p.M = M;
  p.J = J;
  p.K = K;
  p.nt = static_cast<int>((K + 255) / 256);
  p.group_m = 8;
  p.most[0] = most;
  p.most[1] = most ? most + M : nullptr;
  const GradTimes t(M, J, K);
  p.two = two_parts(t.first, dx ? t.tiles[0] : 0, dw ? t.tiles[1] : 0, t.tile);
  return bf16 ? launch_grads<__nv_bfloat16>(maps, dx, dw, p, launches, status, st) : launch_grads<__half>(maps, dx, dw, p, launches, status, st);
}
}  // namespace

extern "C" int b200_linear_grads(const void* g, const void* x, const void* w, void* dx, void* dw, int64_t M, int64_t J, int64_t K, int64_t sgm, int64_t sxm, int64_t swj, int dtype, void* scratch,
                                 int64_t scratch_bytes, uint32_t* status, void* stream) {
  if (dtype != B200_BF16 && dtype != B200_F16) return B200_EDTYPE;
  return run_linear_grads(g, g, nullptr, x, w, dx, dw, M, J, K, sgm, sxm, swj, dtype, scratch, scratch_bytes, status, stream);
}
extern "C" int b200_linear_grads_scaled(const void* g, const void* g_columns, const uint32_t* most, const void* x, const void* w, void* dx, void* dw, int64_t M, int64_t J, int64_t K, int64_t sgm,
                                        int64_t sxm, int64_t swj, void* scratch, int64_t scratch_bytes, uint32_t* status, void* stream) {
  if (!most) return B200_EINVAL;
  return run_linear_grads(g, g_columns, most, x, w, dx, dw, M, J, K, sgm, sxm, swj, B200_F16, scratch, scratch_bytes, status, stream);
}
