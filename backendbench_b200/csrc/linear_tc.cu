// The linear layers of a feed-forward block on the 5th-generation tensor cores:
//
//   gated   h[m, n] = act(g[m, n]) * u[m, n],  g = x Wg^T, u = x Wu^T   (bf16 / f16, W = [Wg; Wu], 2 N x K)
//   int8    y[m, n] = (sum_k a[m, k] b[n, k]) * sa[m] * sb[n] + bias[n]   (int8 operands, exact 32-bit sums)
//   scaled  y[m, n] = (sum_k a[m, k] b[n, k]) * 2^e[m]                    (f16, rows of a scaled by powers of two: see row_factor)
//
// All read operands whose rows lie along K, in slabs of 128 bytes, and all need the whole accumulator of a tile
// before anything is written, so they share one kernel: a TMA producer warp, a warp that issues tcgen05.mma
// (kind::f16 or kind::i8, four steps of 32 bytes of K to a slab), two accumulators of 256 columns in tensor memory and eight
// epilogue warps that empty one while the other fills.
//
// Gated: a tile of w outputs takes w rows of Wg and the same w rows of Wu as ONE B operand of 2 w rows, so that gate
// and up land side by side in the accumulator of the same lane: x crosses into shared memory once for both,
// and act(g) * u is formed from the fp32 sums with one rounding (training: the sums g and u are written beside it as
// they are; rounded to bf16 they would cost the gradients a third of their exactness: 3.0e-3 against 2.4e-3 of the norm, 1.7e-3
// of which is their own rounding). A pair of CTAs (cta_group::2, 256 rows) splits it the natural way: the even CTA loads the
// gate rows, the odd one the up rows.
//
// Few rows (decoding): what counts is that every SM streams its share of the weights without a pause. A tile's width is
// any multiple of 8 (16) columns, chosen so that the tiles come out even over the SMs, and the A slab has as many
// rows as there are; the MMA's other rows multiply whatever lies behind it and are never stored.
#include <cuda.h>

#include <atomic>
#include <cmath>
#include <type_traits>
#include <utility>

#include "gate_act.cuh"
#include "linear_common.cuh"

namespace b200 {

namespace {

constexpr int kLinMaxStages = 16;
constexpr int kLinAccs = 2;  // at most
constexpr int kLinHalfRing = 108 * 1024;                // half an SM's shared memory: 110 KB a CTA (never three of them, which would be more tensor memory than there is)
constexpr size_t lin_smem(int ring) { return static_cast<size_t>(ring) + (ring == kLinRing ? kLinEpiWarps * kLinEpiBytes : 0) + 1024 /*align*/ + 512 /*barriers*/; }

enum : int { kGated = 0, kInt8 = 1, kScaled = 2 };

struct LinParams {
  int64_t M, N, K;        // outputs M x N; K in elements
  int w;                  // output columns of a tile
  int a_rows, b_rows;     // rows of the A box; rows of one B box
  int b_boxes;            // boxes of B in this CTA's stage (gated on a single CTA: gate and up)
  int k_step;             // elements of K to a slab
  int group_m;            // row blocks per rasterisation group
  int splits;             // kSplit: CTAs that share a tile's K
  int ring, stages;       // bytes of shared memory for the slabs, and how many that is (see ring_stages)
  int acc_cols, accs;     // accumulators in tensor memory: columns of one, how many
  int early, ahead;       // the next grid may start beside this one; slabs of weights that it brings into L2 then
  uint32_t idesc;
  int act;                // gated: activation
  float* side;            // gated: the projections [M, 2 N], or NULL
  const float* a_scale;   // int8
  const float* b_scale;
  const void* bias;       // int8: [N] of the output type, or NULL
  const uint32_t* a_most; // scaled: largest magnitude of every row of a before it was scaled, as fp32 bits
};

__device__ __forceinline__ void lin_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, bool i8) {
  if (i8) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  } else {
    tc_mma_f16(d, a, b, idesc, accumulate);
  }
}
__device__ __forceinline__ void lin_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, bool i8) {
  if (i8) {
    const uint32_t z = 0u;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(z)
        : "memory");
  } else {
    tc_mma_f16_pair(d, a, b, idesc, accumulate);
  }
}

// Four outputs of a row, from sums (gated: of both projections), and where they go
template <int MODE, typename TO>
__device__ __forceinline__ void lin_out(const LinParams& p, TO* out, const float* a_scale, const float* b_scale, const TO* bias, const uint32_t* a_most, int64_t m, int64_t n, const float* g, const float* u, bool vec) {
  float v[4];
  const int left = p.N - n < 4 ? static_cast<int>(p.N - n) : 4;
  if constexpr (MODE == kInt8) {
    const float sa = a_scale[m];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = e < left ? g[e] * sa * b_scale[n + e] : 0.f;
      if (bias && e < left) v[e] += to_f32(bias[n + e]);
    }
  } else if constexpr (MODE == kScaled) {
    const float factor = row_factor(a_most[m]);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = g[e] * factor;
  } else {
    gate_act_each(p.act, [&](auto act) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = act.fast(g[e]) * u[e];
    });
    if (p.side) {
      float* to = p.side + m * 2 * p.N + n;
      if (vec) {
        *reinterpret_cast<uint4*>(to) = narrow<float>(g);
        *reinterpret_cast<uint4*>(to + p.N) = narrow<float>(u);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < left) {
            to[e] = g[e];
            to[p.N + e] = u[e];
          }
      }
    }
  }
  TO* to = out + m * p.N + n;
  if (vec) {
    if constexpr (sizeof(TO) == 4) {
      *reinterpret_cast<uint4*>(to) = narrow<float>(v);
    } else {
      const float w[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
      const uint4 r = narrow<TO>(w);
      *reinterpret_cast<uint2*>(to) = make_uint2(r.x, r.y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) to[e] = from_f32<TO>(v[e]);
  }
}

template <int MODE, typename TO, int SHARE>
__global__ void __launch_bounds__(kLinThreads, 1) linear_tc(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, TO* __restrict__ out, LinParams p, uint32_t* __restrict__ status) {
  constexpr bool kI8 = MODE == kInt8, kTwice = MODE == kGated /* two accumulators' columns to an output */, kPair = SHARE == kPaired;
  constexpr int kTileM = kPair ? 256 : 128;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  // (a CTA with one tile has multiplied all of its slabs when it stores: it stages where they were)
  unsigned char* epi_stage = smem + (p.ring == kLinRing ? kLinRing : 0);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.ring + (p.ring == kLinRing ? kLinEpiWarps * kLinEpiBytes : 0));
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(bars + 2 * kLinMaxStages + 2 * kLinAccs);
  volatile uint32_t* abort_flag = tmem_base_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem), bar_base = smem_u32(bars);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kLinMaxStages + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * kLinMaxStages + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * kLinMaxStages + kLinAccs + a); };
  const uint32_t a_bytes = static_cast<uint32_t>(p.a_rows) * kSlabBytes, b_bytes = static_cast<uint32_t>(p.b_rows) * kSlabBytes;
  const uint32_t stage_bytes = a_bytes + static_cast<uint32_t>(p.b_boxes) * b_bytes;
  const int stages = p.stages;
  const uint32_t rank = SHARE != kSingle ? cluster_ctarank() : 0u, cta_rank = kPair ? rank : 0u;

  if (threadIdx.x == 64) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_a)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_b)) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < p.accs; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), kPair ? 16 : 8);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_slot)), "r"(p.accs * p.acc_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_slot)), "r"(p.accs * p.acc_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (kPair) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  if constexpr (!kPair) {
    // Beside this grid there may be room for the next one's CTAs (which start here, where every CTA has its tensor memory), see half_an_sm: they set
    // themselves up and bring the first of their weights into L2, which holds whatever this grid writes all the same.
    if (p.early) next_grid_may_start();
    if (p.early && warp == 0 && lane == 0) {
      const int64_t t = SHARE == kSplit ? blockIdx.x / p.splits : blockIdx.x, mt = (p.M + 127) / 128, nt = (p.N + p.w - 1) / p.w;
      const int all = static_cast<int>((p.K + p.k_step - 1) / p.k_step), k0 = SHARE == kSplit ? static_cast<int>(static_cast<int64_t>(all) * rank / p.splits) : 0,
                k1 = SHARE == kSplit ? static_cast<int>(static_cast<int64_t>(all) * (rank + 1) / p.splits) : all;
      int mb, nb;
      lin_tile(t, mt, nt, p.group_m, mb, nb);
      for (int s = 0; s < p.ahead && k0 + s < k1; ++s) {
        prefetch_l2_3d(&map_b, (k0 + s) * p.k_step, nb * p.w, 0);
        if (kTwice) prefetch_l2_3d(&map_b, (k0 + s) * p.k_step, nb * p.w + static_cast<int>(p.N), 0);
      }
    }
  }
  after_grids_before();
  const float *a_scale = waited(p.a_scale), *b_scale = waited(p.b_scale);
  const TO* bias = waited(static_cast<const TO*>(p.bias));
  const uint32_t* a_most = waited(p.a_most);

  const int64_t mt = (p.M + kTileM - 1) / kTileM, nt = (p.N + p.w - 1) / p.w, tiles = mt * nt;
  const int64_t tile_first = kPair ? (blockIdx.x >> 1) : SHARE == kSplit ? blockIdx.x / p.splits : blockIdx.x, tile_step = kPair ? (gridDim.x >> 1) : SHARE == kSplit ? tiles : gridDim.x;
  const int all_slabs = static_cast<int>((p.K + p.k_step - 1) / p.k_step);
  const int slab0 = SHARE == kSplit ? static_cast<int>(static_cast<int64_t>(all_slabs) * rank / p.splits) : 0;
  const int slabs = SHARE == kSplit ? static_cast<int>(static_cast<int64_t>(all_slabs) * (rank + 1) / p.splits) - slab0 : all_slabs;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int64_t t = tile_first; t < tiles && ok; t += tile_step) {
        int mb, nb;
        lin_tile(t, mt, nt, p.group_m, mb, nb);
        const int m0 = mb * kTileM + static_cast<int>(cta_rank) * 128;
        // gated: the gate rows n0.., then the up rows N + n0..; a pair has a box of B to each CTA
        int n0 = nb * p.w, n1 = n0 + static_cast<int>(p.N);
        if (kPair && cta_rank == 1u) n0 = kTwice ? n1 : n0 + p.b_rows;
        for (int kb = 0; kb < slabs; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, kLinWaitNs)) { ok = false; break; }
          const uint32_t a_dst = smem_base + stage * stage_bytes, b_dst = a_dst + a_bytes;
          const int k = (slab0 + kb) * p.k_step;
          if (kPair) {
            const uint32_t fbar = map_to_cta(full_bar(stage), 0u);
            if (cta_rank == 0u) mbar_expect_tx(full_bar(stage), 2 * stage_bytes);
            tma_load_3d_pair(a_dst, &map_a, fbar, k, m0, 0);
            tma_load_3d_pair(b_dst, &map_b, fbar, k, n0, 0);
          } else {
            mbar_expect_tx(full_bar(stage), stage_bytes);
            tma_load_3d(b_dst, &map_b, full_bar(stage), k, n0, 0);
            if (kTwice) tma_load_3d(b_dst + b_bytes, &map_b, full_bar(stage), k, n1, 0);
            tma_load_3d(a_dst, &map_a, full_bar(stage), k, m0, 0);
          }
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
      }
      if (kPair && ok) {
        // the even CTA's commits arrive here from afar: none may land after this CTA's shared memory is gone
        for (int i = 0; i < stages && ok; ++i) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, kLinWaitNs)) ok = false;
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {
        *abort_flag = 1;
        if (status) atomicOr(status, B200_DEV_WAIT_TIMEOUT);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (the whole warp walks, one lane issues)
    if (cta_rank == 0u) {
      const uint32_t empty0 = kPair ? map_to_cta(empty_bar(0), 0u) : 0u, empty1 = kPair ? map_to_cta(empty_bar(0), 1u) : 0u;
      auto warp_wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, kLinWaitNs)) != 0; };
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int64_t t = tile_first; t < tiles && ok; t += tile_step) {
        if (!warp_wait(tempty_bar(acc), acc_phase ^ 1u)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * p.acc_cols);
        for (int kb = 0; kb < slabs; ++kb) {
          if (!warp_wait(full_bar(stage), phase)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_base + stage * stage_bytes, b_addr = a_addr + a_bytes;
          uint64_t da[4], db[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            da[k] = smem_desc(a_addr + k * 32u, 16u, 1024u);
            db[k] = smem_desc(b_addr + k * 32u, 16u, 1024u);
          }
          const uint32_t e0 = kPair ? empty0 + 8u * stage : empty_bar(stage), e1 = empty1 + 8u * stage;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (kPair) lin_mma_pair(d_tmem, da[k], db[k], p.idesc, (kb | k) != 0 ? 1u : 0u, kI8);
              else lin_mma(d_tmem, da[k], db[k], p.idesc, (kb | k) != 0 ? 1u : 0u, kI8);
            }
            if (kPair) {
              tc_commit_pair(e0);
              tc_commit_pair(e1);
            } else {
              tc_commit(e0);
            }
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if (elect_one()) {
          if (kPair) {
            tc_commit_pair(map_to_cta(tfull_bar(acc), 0u));
            tc_commit_pair(map_to_cta(tfull_bar(acc), 1u));
          } else {
            tc_commit(tfull_bar(acc));
          }
        }
        __syncwarp();
        if (++acc == p.accs) { acc = 0; acc_phase ^= 1u; }
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        if (status) atomicOr(status, B200_DEV_WAIT_TIMEOUT);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue: 32 columns at a time, two warps to a lane quarter
    const int q = warp & 3, half = (warp - 2) >> 2;
    unsigned char* mine = epi_stage + (warp - 2) * kLinEpiBytes;
    constexpr int kPer = 16 / static_cast<int>(sizeof(TO)), kRegs = kTwice ? 64 : 32;
    const bool vec = p.N % kPer == 0 && ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(p.side)) & 15u) == 0;
    const uint32_t tempty_target = kPair ? map_to_cta(tempty_bar(0), 0u) : 0u;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int64_t t = tile_first; t < tiles && ok; t += tile_step) {
      int mb, nb;
      lin_tile(t, mt, nt, p.group_m, mb, nb);
      const int64_t mr0 = static_cast<int64_t>(mb) * kTileM + static_cast<int64_t>(cta_rank) * 128 + q * 32, n0 = static_cast<int64_t>(nb) * p.w;
      const int wide = p.N - n0 < p.w ? static_cast<int>(p.N - n0) : p.w;  // columns of this tile that exist
      const int nrows = p.M - mr0 < 32 ? static_cast<int>(p.M - mr0) : 32;  // <= 0: none
      const int chunks = (wide + 31) / 32, count = (chunks + 1 - half) / 2;  // this warp takes chunks half, half + 2, ...
      float scale_next = 0.f, bias_next = 0.f;
      auto ahead = [&](int64_t n, int left) {
        if constexpr (kI8) {
          scale_next = lane < left ? b_scale[n + lane] : 0.f;
          bias_next = bias && lane < left ? to_f32(bias[n + lane]) : 0.f;
        }
      };
      ahead(n0 + half * 32, wide - half * 32);
      float sa = 0.f;
      if (!kTwice && lane < nrows) sa = kI8 ? a_scale[mr0 + lane] : row_factor(a_most[mr0 + lane]);
      int got = 0;
      if (lane == 0) got = mbar_wait(tfull_bar(acc), acc_phase, abort_flag, kLinWaitNs) ? 1 : 0;
      got = __shfl_sync(0xffffffffu, got, 0);
      if (!got) { ok = false; break; }
      tc_fence_after();
      const uint32_t t_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * p.acc_cols);
      if constexpr (SHARE == kSplit) {
        // this CTA's sums to its own shared memory (everything that was in the ring has been multiplied), a row to a lane
        const int columns = p.w * (kTwice ? 2 : 1);
        if (q * 32 < p.a_rows) {
          for (int c = half * 32; c < columns; c += 64) {
            uint32_t r[32];
            tc_ld_32x32(t_base + static_cast<uint32_t>(c), r);
            tc_ld_wait();
            unsigned char* row = smem + (q * 32 + lane) * (columns * 4 + 16) + c * 4;
            if (q * 32 + lane < p.a_rows) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                if (c + e < columns) *reinterpret_cast<uint4*>(row + e * 4) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
            }
          }
        }
        break;
      }
      uint32_t r[kRegs];
      auto fetch = [&](int i) {
        const uint32_t col = static_cast<uint32_t>((half + 2 * i) * 32);
        tc_ld_32x32(t_base + col, r);
        if constexpr (kTwice) tc_ld_32x32(t_base + static_cast<uint32_t>(p.w) + col, r + 32);
      };
      // the chunk's values are in `v`: the next chunk is on its way while they are rounded and stored, or, behind the last,
      // the accumulator goes back to the MMA warp
      auto next = [&](int i) {
        if (i + 1 < count) {
          fetch(i + 1);
          return;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (kPair) mbar_arrive_cluster(tempty_target + 8u * acc);
          else mbar_arrive(tempty_bar(acc));
        }
      };
      if (count > 0) fetch(0);
      else next(0);
#pragma unroll 1
      for (int i = 0; i < count; ++i) {
        const int c0 = (half + 2 * i) * 32, ncols = wide - c0 < 32 ? wide - c0 : 32;
        const int64_t n = n0 + c0;
        float v[32];
        tc_ld_wait();
        if constexpr (kI8) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = static_cast<float>(static_cast<int>(r[e])) * sa;
          next(i);
          // this chunk's scales and bias, a column to a lane since the chunk before, to every lane by way of the staging buffer
          float* shared = reinterpret_cast<float*>(mine);
          __syncwarp();
          shared[lane] = scale_next;
          shared[32 + lane] = bias_next;
          __syncwarp();
          ahead(n + 64, wide - c0 - 64);
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 b = *reinterpret_cast<const float4*>(shared + e), c = *reinterpret_cast<const float4*>(shared + 32 + e);
            v[e] = v[e] * b.x + c.x;
            v[e + 1] = v[e + 1] * b.y + c.y;
            v[e + 2] = v[e + 2] * b.z + c.z;
            v[e + 3] = v[e + 3] * b.w + c.w;
          }
        } else if constexpr (MODE == kScaled) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]) * sa;
          next(i);
        } else {
          const float *g = reinterpret_cast<const float*>(r), *u = reinterpret_cast<const float*>(r + 32);
          if (p.side && nrows > 0) {
            float* side = p.side + mr0 * (2 * p.N) + n;
            lin_store<float>(g, mine, side, 2 * p.N, nrows, ncols, vec, lane);
            lin_store<float>(u, mine, side + p.N, 2 * p.N, nrows, ncols, vec, lane);
          }
          gate_act_each(p.act, [&](auto act) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = act.fast(g[e]) * u[e];
          });
          next(i);
        }
        if (nrows > 0) lin_store<TO>(v, mine, out + mr0 * p.N + n, p.N, nrows, ncols, vec, lane);
      }
      if (++acc == p.accs) { acc = 0; acc_phase ^= 1u; }
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      if (status) atomicOr(status, B200_DEV_WAIT_TIMEOUT);
    }
    __syncwarp();
  }

  if constexpr (SHARE == kSplit) {
    // Every CTA of the cluster puts together its share of the tile: four columns to a thread, the CTAs' sums added in the order of
    // their ranges of K.
    cluster_sync_all();
    const int columns = p.w * (kTwice ? 2 : 1), quads = p.w / 4;
    const uint32_t pitch = static_cast<uint32_t>(columns) * 4 + 16;
    int mb, nb;
    lin_tile(tile_first, mt, nt, p.group_m, mb, nb);
    const int64_t mr0 = static_cast<int64_t>(mb) * 128, n0 = static_cast<int64_t>(nb) * p.w;
    const bool quad_vec = p.N % 4 == 0 && ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(p.side)) & 15u) == 0;
    const int rows = p.M - mr0 < p.a_rows ? static_cast<int>(p.M - mr0) : p.a_rows, units = rows * quads;
    for (int i = static_cast<int>(rank) * kLinThreads + static_cast<int>(threadIdx.x); i < units; i += p.splits * kLinThreads) {
      const int r = i / quads, c = (i - r * quads) * 4;
      const uint32_t at = smem_base + static_cast<uint32_t>(r) * pitch + static_cast<uint32_t>(c) * 4;
      float g[4] = {}, u[4] = {};
      int s[4] = {};
      for (int k = 0; k < p.splits; ++k) {
        const uint32_t from = map_to_cta(at, static_cast<uint32_t>(k));
        if constexpr (kI8) {
          const int4 v = ld_cluster<int4>(from);
          s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
        } else {
          const float4 v = ld_cluster<float4>(from);
          g[0] += v.x; g[1] += v.y; g[2] += v.z; g[3] += v.w;
          if constexpr (kTwice) {
            const float4 w = ld_cluster<float4>(from + static_cast<uint32_t>(p.w) * 4);
            u[0] += w.x; u[1] += w.y; u[2] += w.z; u[3] += w.w;
          }
        }
      }
      if (n0 + c >= p.N) continue;
      if constexpr (kI8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = static_cast<float>(s[e]);
      }
      lin_out<MODE, TO>(p, out, a_scale, b_scale, bias, a_most, mr0 + r, n0 + c, g, u, quad_vec);
    }
    cluster_sync_all();  // nobody leaves while another reads its sums
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the shared memory goes away
    __syncthreads();
  }
  if (kPair) cluster_sync_all();
  if (warp == 1) {
    if (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(p.accs * p.acc_cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(p.accs * p.acc_cols) : "memory");
  }
}

// ------------------------------------------------------------------ operands off the grid
// A matrix [rows, K] of any strides into rows along K for the copy engine, which wants a pitch that is a multiple of 16 bytes, and is
// faster where no slab of a row lies across two lines.
//
// Rows that lie along K, off the 16-byte grid: a thread to 16 bytes of the result, from the one or two aligned blocks that its bytes
// lie in, shifted into place. A block holds a byte of the matrix or is not read, so that no load leaves the
// 16-byte granules of the matrix itself. What lands behind a row's end is padding that the tensor map leaves out.
// Both operands of a call that need it go in one launch, the first `blocks0` CTAs taking the one.
struct PackRows {
  const unsigned char* x;
  unsigned char* to;
  int64_t rows, row_bytes, s_bytes, pitch;  // (the last: bytes)
  uint32_t pieces;  // of sixteen bytes that a row's elements take
};
__global__ void __launch_bounds__(256) pack_rows_shifted(PackRows A, PackRows B, unsigned blocks0) {
  next_grid_may_start();  // (the product's CTAs set themselves up meanwhile)
  const bool second = blockIdx.x >= blocks0;
  const PackRows& P = second ? B : A;
  const unsigned char* x = P.x;
  unsigned char* to = P.to;
  const int64_t s_bytes = P.s_bytes, total = P.rows * P.pieces, step = static_cast<int64_t>(second ? gridDim.x - blocks0 : blocks0) * 256;
  const uint32_t pieces = P.pieces;
  const unsigned char* end = x + (P.rows - 1) * s_bytes + P.row_bytes;
  for (int64_t i = static_cast<int64_t>(second ? blockIdx.x - blocks0 : blockIdx.x) * 256 + threadIdx.x; i < total; i += step) {
    const int64_t r = total <= 0xffffffffll ? static_cast<uint32_t>(i) / pieces : i / pieces;
    const int64_t j = i - r * pieces;
    const unsigned char* from = x + r * s_bytes + j * 16;
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from)) & 15u;
    const unsigned char* block = from - off;
    const uint4 lo = ld_keep(block);
    uint4 hi = make_uint4(0u, 0u, 0u, 0u);
    if (off && block + 16 < end) hi = ld_keep(block + 16);
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    const uint32_t skip = off >> 2, bits = (off & 3u) * 8u;
    uint32_t v[5];  // the five words that the sixteen bytes lie in
#pragma unroll
    for (int k = 0; k < 5; ++k) {
      const uint32_t a = skip & 1u ? w[k + 1 < 8 ? k + 1 : 7] : w[k], b = skip & 1u ? w[k + 3 < 8 ? k + 3 : 7] : w[k + 2 < 8 ? k + 2 : 7];
      v[k] = skip & 2u ? b : a;
    }
    *reinterpret_cast<uint4*>(to + r * P.pitch + j * 16) = make_uint4(__funnelshift_r(v[0], v[1], bits), __funnelshift_r(v[1], v[2], bits), __funnelshift_r(v[2], v[3], bits), __funnelshift_r(v[3], v[4], bits));
  }
}

// Any other strides: 32 x 32 tiles through shared memory, read along whichever dimension is contiguous.
template <typename E>
__global__ void __launch_bounds__(256) pack_rows(const E* x, E* __restrict__ to, int64_t rows, int64_t K, int64_t s_r, int64_t s_k, int64_t pitch) {
  __shared__ E tile[32][33];
  next_grid_may_start();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t kt = (K + 31) / 32, tiles = ((rows + 31) / 32) * kt;
  const bool along_k = s_r != 1;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t r0 = t / kt * 32, k0 = (t % kt) * 32;
    __syncthreads();
    for (int i = ty; i < 32; i += 8) {
      const int64_t r = r0 + (along_k ? i : tx), k = k0 + (along_k ? tx : i);
      if (r < rows && k < K) tile[along_k ? i : tx][along_k ? tx : i] = x[r * s_r + k * s_k];
    }
    __syncthreads();
    for (int i = ty; i < 32; i += 8)
      if (r0 + i < rows && k0 + tx < K) to[(r0 + i) * pitch + k0 + tx] = tile[i][tx];
  }
}

}  // namespace

void lin_pack(LinOperand& a, LinOperand& b, unsigned char* at, cudaStream_t st, int& launches) {
  const int64_t most = kNumSMs * 8;
  PackRows rows[2] = {};
  unsigned blocks[2] = {};
  int n = 0;
  for (LinOperand* o : {&a, &b}) {
    if (o->ready()) {
      if (o->rows == 1) o->s_r = o->pitch();  // never used
      continue;
    }
    const int64_t pitch = o->pitch(), bytes = o->packed_bytes();
    if (o->s_k == 1 || o->K == 1) {
      const int64_t pieces = (o->K * o->esize + 15) / 16, needed = (o->rows * pieces + 255) / 256;
      rows[n] = PackRows{static_cast<const unsigned char*>(o->base), at, o->rows, o->K * o->esize, o->s_r * o->esize, pitch * o->esize, static_cast<uint32_t>(pieces)};
      blocks[n++] = static_cast<unsigned>(needed < most ? needed : most);
    } else {
      const int64_t tiles = ((o->rows + 31) / 32) * ((o->K + 31) / 32);
      const int grid = static_cast<int>(tiles < most ? tiles : most);
      if (o->esize == 2) pack_rows<uint16_t><<<grid, 256, 0, st>>>(static_cast<const uint16_t*>(o->base), reinterpret_cast<uint16_t*>(at), o->rows, o->K, o->s_r, o->s_k, pitch);
      else pack_rows<uint8_t><<<grid, 256, 0, st>>>(static_cast<const uint8_t*>(o->base), at, o->rows, o->K, o->s_r, o->s_k, pitch);
      ++launches;
    }
    o->s_r = pitch;
    o->s_k = 1;
    o->base = at;
    at += bytes;
  }
  if (n) {
    pack_rows_shifted<<<blocks[0] + blocks[1], 256, 0, st>>>(rows[0], rows[1], blocks[0]);
    ++launches;
  }
}

namespace {

bool encode_rows(CUtensorMap* map, const LinOperand& o, CUtensorMapDataType dt, int box_rows) {
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(o.K), static_cast<cuuint64_t>(o.rows), 1};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(o.s_r * o.esize), static_cast<cuuint64_t>(o.s_r * o.esize) * static_cast<cuuint64_t>(o.rows)};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(kSlabBytes / o.esize), static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return encode_fn()(map, dt, 3, const_cast<void*>(o.base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Slabs that fit into `ring` bytes. The MMA reads 128 rows of A whatever the box holds, so the last slab has that much room too.
constexpr int kMmaABytes = 128 * kSlabBytes;
int ring_stages(int ring, int stage_bytes) {
  const int last = stage_bytes > kMmaABytes ? stage_bytes : kMmaABytes, fit = 1 + (ring - last) / stage_bytes;
  return fit < kLinMaxStages ? fit : kLinMaxStages;
}

struct LinPlan {
  int share, w, a_rows, splits;
};
int lin_stage_bytes(int per, int w, int a_rows) { return (a_rows + per * w) * kSlabBytes; }  // (a CTA of a pair: half of them)
// A tile to a CTA, room for four slabs and for its sums: half an SM's shared memory is enough, and the next grid may start early. Clusters' CTAs (56 to 72
// registers a thread) share an SM two by two. A CTA without a cluster keeps what it stores in 166 to 168 registers and has its SM to itself: there the
// next grid starts on the SMs that this one leaves free. 110 sizes of up to 1024 rows, calls in a row: without the early start of single CTAs up to 28 % slower
// where they are few (int8 24 x 128 x 120 3.0 us, 3.9 without; bf16 40 x 64 x 512 3.9 and 4.6), up to 13 % faster where the next call packs an
// operand (bf16 144 x 265 x 896 8.7 and 7.6: weights are brought into L2 while they are written), 0.6 % slower on average; with the whole ring and the
// early start as fast as with half of it (0.2 %); with plans that give single CTAs the whole SM 0.8 % slower.
bool half_an_sm(int per, int w, int a_rows, int splits) {
  return 4 * lin_stage_bytes(per, w, a_rows) <= kLinHalfRing && (splits == 1 || a_rows * (w * per * 4 + 16) <= kLinHalfRing);
}

// What a plan takes, in us, with `per` rows of B to an output column (gated 2, int8 1) and slabs of 128 bytes of K. The terms: what
// starting, handing over and storing take; the weights out of HBM; every CTA's bytes over the fabric; the latency of the loads
// (longer for B, which comes from HBM, than for A, which comes from L2) over the bytes that are in flight; the issue of a
// slab. Their constants were fitted to 1,500 timings of 68 products (1 to 8192 rows, K 160 to 11008, 128 to 11008 columns, both
// types); the plan with the least of these is 2 % slower than the best one that was timed, on average, and at most 16 %.
double time_of(const LinPlan& q, int64_t M, int64_t N, int64_t slabs, int per) {
  const double k = static_cast<double>(slabs), cols = q.w * per;
  const int64_t across = (N + q.w - 1) / q.w;
  if (q.share == kPaired) {
    const int64_t tiles = ((M + 255) / 256) * across, rounds = (tiles + kNumSMs / 2 - 1) / (kNumSMs / 2);
    return 6.8 + static_cast<double>(rounds) * (2.16 + k * (cols == 256 ? 0.31 : cols == 192 ? 0.242 : 0.192));
  }
  const int64_t tiles = ((M + 127) / 128) * across;
  const bool half = half_an_sm(per, q.w, q.a_rows, q.splits) && tiles * q.splits <= 2 * kResident[q.splits];
  const int64_t room = (half ? 2 : 1) * kResident[q.splits];
  double ctas = static_cast<double>(tiles * q.splits), rounds = 1;
  if (tiles * q.splits > room) {
    if (q.splits > 1) return 1e30;  // a cluster has one tile
    rounds = static_cast<double>((tiles + kNumSMs - 1) / kNumSMs);
    ctas = kNumSMs;
  }
  const double each = static_cast<double>((slabs + q.splits - 1) / q.splits) * rounds, a = each * kSlabBytes * q.a_rows * ctas, b = each * kSlabBytes * cols * ctas;
  const double deep = ctas > kNumSMs ? 2. : 1.;  // CTAs to an SM (of clusters beside each other, single ones after each other)
  double t = k * kSlabBytes * static_cast<double>(N * per) / 11e6;
  t = fmax(t, (a + b) / 16.8e6);
  t = fmax(t, (1.98 * b + 0.6 * a) / (ctas * (half ? kLinHalfRing : kLinRing)));
  t = fmax(t, each * (0.225 * (deep > 1. ? 1.44 : 1.) + 0.000225 * cols * deep));
  return 3.64 + (half ? 0. : 0.12) + t + 1.29 * rounds + 0.007 * cols * deep + (q.splits > 1 ? 0.68 + q.a_rows * cols / 3.9e3 : 0.);
}
LinPlan best_plan(int64_t M, int64_t N, int64_t slabs, int per) {
  const int most = 256 / per, grain = 16 / per, a_rows = M >= 128 ? 128 : static_cast<int>((M + 7) / 8 * 8);
  LinPlan best{kSingle, most, a_rows, 1};
  double least = 1e30;
  auto offer = [&](const LinPlan& q) {
    const double t = time_of(q, M, N, slabs, per);
    if (t < least) { least = t; best = q; }
  };
  if (M > 128)
    for (int w : {most, most * 3 / 4, most / 2}) offer(LinPlan{kPaired, w, 128, 1});
  for (int s : {1, 2, 3, 4, 6, 8})
    for (int w : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16})
      if (s <= slabs) offer(LinPlan{s > 1 ? kSplit : kSingle, w * grain, a_rows, s});
  return best;
}
// (a look at some seventy plans takes longer than a launch: each thread keeps those of the sizes it saw last)
LinPlan plan_linear(int64_t M, int64_t N, int64_t K, int per, int k_step) {
  struct Seen {
    int64_t M, N, slabs;
    int per;
    LinPlan plan;
  };
  static thread_local Seen seen[64] = {};
  const int64_t slabs = (K + k_step - 1) / k_step;
  Seen& s = seen[(static_cast<uint64_t>(M) * 31 + static_cast<uint64_t>(N) * 7 + static_cast<uint64_t>(slabs) * 3 + per) % 64];
  if (s.M != M || s.N != N || s.slabs != slabs || s.per != per) s = Seen{M, N, slabs, per, best_plan(M, N, slabs, per)};
  return s.plan;
}

template <int MODE, typename TO, int SHARE>
int launch_linear(int cluster, int64_t ctas, cudaStream_t st, const CUtensorMap& map_a, const CUtensorMap& map_b, TO* out, const LinParams& p, uint32_t* status) {
  const auto kernel = linear_tc<MODE, TO, SHARE>;
  static std::atomic<uint64_t> allowed{0};  // devices on which this kernel may have that much shared memory (0.4 us a call to say so each time)
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lin_smem(kLinRing)));
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) { set_last_cuda_error(e); return B200_ELAUNCH; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(kLinThreads, 1, 1);
  cfg.dynamicSmemBytes = lin_smem(p.ring);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // (see launch_after)
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t le = cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, out, p, status);
  if (le != cudaSuccess) { set_last_cuda_error(le); return B200_ELAUNCH; }
  return B200_OK;
}

struct LinOperands {
  LinOperand a, b;
  LinPlan plan;
  // a is [M, K], b [per N, K]
  LinOperands(const void* A, const void* B, int64_t M, int64_t N, int64_t K, int64_t sAm, int64_t sAk, int64_t sBn, int64_t sBk, int per, int esize)
      : a{A, M, K, sAm, sAk, esize, 0}, b{B, per * N, K, sBn, sBk, esize, 0}, plan(plan_linear(M, N, K, per, kSlabBytes / esize)) {
    const int tile_m = plan.share == kPaired ? 256 : 128;
    a.reads = (N + plan.w - 1) / plan.w;
    b.reads = (M + tile_m - 1) / tile_m;
  }
  int64_t packed_bytes() const { return a.packed_bytes() + b.packed_bytes(); }
};

template <int MODE>
int run_linear(LinOperands ops, void* out, int64_t M, int64_t N, int64_t K, int dtype_out, bool is_bf16, LinParams& p, void* scratch, int64_t scratch_bytes, uint32_t* status, cudaStream_t st) {
  constexpr int per = MODE == kGated ? 2 : 1;
  LinOperand &a = ops.a, &b = ops.b;
  if (!encode_fn()) return B200_EDRIVER;
  const int64_t need = ops.packed_bytes();
  if (need && (!scratch || scratch_bytes < need + 256)) return B200_ESCRATCH;
  unsigned char* at = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(scratch) + 255) & ~static_cast<uintptr_t>(255));
  int launches = 1;
  lin_pack(a, b, at, st, launches);
  p.M = M;
  p.N = N;
  p.K = K;
  p.k_step = kSlabBytes / a.esize;
  int64_t rows = (32ll << 20) / (K * a.esize) / 256 * 256;  // a group's panel of A stays in L2 while B goes by
  rows = rows < 2048 ? 2048 : rows > 65536 ? 65536 : rows;
  const uint32_t fmt = MODE == kInt8 ? 1u /* signed */ : is_bf16 ? 1u : 0u, sums = MODE == kInt8 ? 2u /* s32 */ : 1u /* f32 */;
  const CUtensorMapDataType dt = MODE == kInt8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto run = [&](const LinPlan& plan) -> int {
    const bool pair = plan.share == kPaired;
    const int tile_m = pair ? 256 : 128;
    p.w = plan.w;
    p.a_rows = plan.a_rows;
    p.b_rows = MODE == kGated ? plan.w : pair ? plan.w / 2 : plan.w;
    p.b_boxes = MODE == kGated && !pair ? 2 : 1;
    p.splits = plan.splits;
    p.group_m = static_cast<int>(rows / tile_m);
    p.idesc = (sums << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(plan.w * per >> 3) << 17) | (static_cast<uint32_t>(tile_m >> 4) << 24);
    alignas(64) CUtensorMap map_a, map_b;
    if (!encode_rows(&map_a, a, dt, p.a_rows) || !encode_rows(&map_b, b, dt, p.b_rows)) return B200_EDRIVER;
    const int64_t tiles = ((M + tile_m - 1) / tile_m) * ((N + plan.w - 1) / plan.w);
    // (see half_an_sm)
    const bool half = !pair && half_an_sm(per, plan.w, p.a_rows, plan.splits) && tiles * plan.splits <= 2 * kResident[plan.splits];
    const int64_t slots = pair ? kNumSMs / 2 : half ? 2 * kNumSMs : kNumSMs, resident = tiles < slots ? tiles : slots;
    p.ring = half ? kLinHalfRing : kLinRing;
    p.stages = ring_stages(p.ring, (p.a_rows + p.b_boxes * p.b_rows) * kSlabBytes);
    p.acc_cols = 256;
    p.accs = half ? 1 : 2;
    p.early = half ? 1 : 0;
    p.ahead = kLinHalfRing / (p.b_boxes * p.b_rows * kSlabBytes);  // (two or three times as much is no faster, and much more slower: bf16 1 x 4096 x 11008 31.1 us, 36.6 with 500 KB a CTA)
    auto go = [&](auto* o) {
      using TO = std::remove_pointer_t<decltype(o)>;
      if (pair) return launch_linear<MODE, TO, kPaired>(2, 2 * resident, st, map_a, map_b, o, p, status);
      if (plan.share == kSplit) return launch_linear<MODE, TO, kSplit>(plan.splits, tiles * plan.splits, st, map_a, map_b, o, p, status);
      return launch_linear<MODE, TO, kSingle>(1, resident, st, map_a, map_b, o, p, status);
    };
    if (dtype_out == B200_F16) return go(static_cast<__half*>(out));
    if constexpr (MODE != kScaled)
      if (dtype_out == B200_BF16) return go(static_cast<__nv_bfloat16*>(out));
    if constexpr (MODE == kInt8) return go(static_cast<float*>(out));
    return B200_EDTYPE;
  };
  int rc = run(ops.plan);
  if (rc == B200_ELAUNCH && ops.plan.share != kSingle) {
    // the cluster launch was refused (a device or a partition without thread-block clusters): the same on single CTAs
    (void)cudaGetLastError();
    rc = run(LinPlan{kSingle, 256 / per, M >= 128 ? 128 : static_cast<int>((M + 7) / 8 * 8), 1});
  }
  if (rc) return rc;
  return check_launch(launches);
}

// y = bias, for an empty contraction
template <typename TO> __global__ void __launch_bounds__(256) bias_rows(const TO* bias, TO* __restrict__ out, int64_t M, int64_t N) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < M * N; i += static_cast<int64_t>(gridDim.x) * 256) out[i] = bias ? bias[i % N] : from_f32<TO>(0.f);
}

constexpr int64_t kMostExtent = 0x7fffffff;

}  // namespace

}  // namespace b200

using namespace b200;

extern "C" int64_t b200_gated_linear_scratch_bytes(const void* x, const void* w, int64_t M, int64_t N, int64_t K, int64_t sxm, int64_t sxk, int64_t swn, int64_t swk) {
  if (M < 1 || N < 1 || K < 1) return 0;
  const int64_t need = LinOperands(x, w, M, N, K, sxm, sxk, swn, swk, 2, 2).packed_bytes();
  return need ? need + 256 : 0;
}

extern "C" int b200_gated_linear(const void* x, const void* w, void* out, float* projections, int64_t M, int64_t N, int64_t K, int64_t sxm, int64_t sxk, int64_t swn, int64_t swk, int activation,
                                 int dtype, void* scratch, int64_t scratch_bytes, uint32_t* status, void* stream) {
  if (M < 0 || N < 0 || K < 0 || activation < 0 || activation >= B200_ACT_COUNT) return B200_EINVAL;
  if (dtype != B200_BF16 && dtype != B200_F16) return B200_EDTYPE;
  if (M == 0 || N == 0) return B200_OK;
  if (!out || M > kMostExtent || N > kMostExtent / 2 || K > kMostExtent) return B200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (K == 0) {  // both projections are zero, and so is their product
    cudaError_t e = cudaMemsetAsync(out, 0, static_cast<size_t>(M * N * 2), st);
    if (e == cudaSuccess && projections) e = cudaMemsetAsync(projections, 0, static_cast<size_t>(M * N * 8), st);
    if (e != cudaSuccess) { set_last_cuda_error(e); return B200_ELAUNCH; }
    return B200_OK;
  }
  if (!x || !w) return B200_EINVAL;
  LinParams p{};
  p.act = activation;
  p.side = projections;
  return run_linear<kGated>(LinOperands(x, w, M, N, K, sxm, sxk, swn, swk, 2, 2), out, M, N, K, dtype, dtype == B200_BF16, p, scratch, scratch_bytes, status, st);
}

extern "C" int64_t b200_linear_scaled_scratch_bytes(const void* A, const void* B, int64_t M, int64_t N, int64_t K, int64_t sAm, int64_t sAk, int64_t sBk, int64_t sBn) {
  if (M < 1 || N < 1 || K < 1) return 0;
  const int64_t need = LinOperands(A, B, M, N, K, sAm, sAk, sBn, sBk, 1, 2).packed_bytes();
  return need ? need + 256 : 0;
}

extern "C" int b200_linear_scaled(const void* A, const uint32_t* a_most, const void* B, void* out, int64_t M, int64_t N, int64_t K, int64_t sAm, int64_t sAk, int64_t sBk, int64_t sBn, void* scratch,
                                  int64_t scratch_bytes, uint32_t* status, void* stream) {
  if (M < 0 || N < 0 || K < 1) return B200_EINVAL;
  if (M == 0 || N == 0) return B200_OK;
  if (!A || !a_most || !B || !out || M > kMostExtent || N > kMostExtent || K > kMostExtent) return B200_EINVAL;
  LinParams p{};
  p.a_most = a_most;
  return run_linear<kScaled>(LinOperands(A, B, M, N, K, sAm, sAk, sBn, sBk, 1, 2), out, M, N, K, B200_F16, false, p, scratch, scratch_bytes, status, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t b200_mm_int8_scratch_bytes(const void* A, const void* B, int64_t M, int64_t N, int64_t K, int64_t sAm, int64_t sAk, int64_t sBk, int64_t sBn) {
  if (M < 1 || N < 1 || K < 1) return 0;
  const int64_t need = LinOperands(A, B, M, N, K, sAm, sAk, sBn, sBk, 1, 1).packed_bytes();
  return need ? need + 256 : 0;
}

extern "C" int b200_mm_int8(const void* A, const void* B, const float* a_scale, const float* b_scale, const void* bias, void* out, int64_t M, int64_t N, int64_t K, int64_t sAm, int64_t sAk,
                            int64_t sBk, int64_t sBn, int dtype_out, void* scratch, int64_t scratch_bytes, uint32_t* status, void* stream) {
  if (M < 0 || N < 0 || K < 0 || K > B200_INT8_MAX_K) return B200_EINVAL;
  if (!is_float_dtype(dtype_out)) return B200_EDTYPE;
  if (M == 0 || N == 0) return B200_OK;
  if (!out || M > kMostExtent || N > kMostExtent) return B200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (K == 0) {
    const int grid = static_cast<int>((M * N + 255) / 256 < kNumSMs * 8 ? (M * N + 255) / 256 : kNumSMs * 8);
    if (dtype_out == B200_F32) bias_rows<<<grid, 256, 0, st>>>(static_cast<const float*>(bias), static_cast<float*>(out), M, N);
    else if (dtype_out == B200_BF16) bias_rows<<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(bias), static_cast<__nv_bfloat16*>(out), M, N);
    else bias_rows<<<grid, 256, 0, st>>>(static_cast<const __half*>(bias), static_cast<__half*>(out), M, N);
    return check_launch();
  }
  if (!A || !B || !a_scale || !b_scale) return B200_EINVAL;
  LinParams p{};
  p.a_scale = a_scale;
  p.b_scale = b_scale;
  p.bias = bias;
  return run_linear<kInt8>(LinOperands(A, B, M, N, K, sAm, sAk, sBn, sBk, 1, 1), out, M, N, K, dtype_out, false, p, scratch, scratch_bytes, status, st);
}
