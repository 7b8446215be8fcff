// fp32 products of the linear layers on the tensor cores: C = A B, and the gated projection pair.
//
// A row of an operand (its K elements) is scaled by a power of two so that its largest magnitude lies in [2^14, 2^15), and every
// element is split into two f16 values, y = h + l: h the nearest one, l the nearest to what is left. That resolves an element to
// 2^-22 of itself, or to 2^-39 of the row's largest, whichever is more (l is subnormal below 2^-14, where half a step is 2^-25). Three f16 products, h h + h l + l h,
// exact in the tensor cores' fp32 sums, are then the fp32 product; what l l would add is below 2^-22 of it. Half the products
// that three bf16 planes take, and as those have no exponents to spare, the scales come back with the result.
//
// The tensor cores truncate when they add, half a unit in the last place of the running sum each time and always towards zero: over a K of
// 1000 to 1500 that was 2 to 3e-6 of the norm, more than everything else together. So no sum runs longer than one slab here: of
// 64 k, smallest products first, and the epilogue warps add the slabs' sums up in registers, rounded to nearest, while the
// tensor cores are at the next ones (four accumulators of 128 columns).
//
// Tiles of 128 or (pairs of CTAs) 256 rows by 128 rows of B: gated, 64 gate and 64 up rows, which the halves of a pair bring one
// kind each. Clusters share a tile's K where tiles are few. An operand whose K elements are not contiguous is turned on its way into the planes.
//
// 1531 x 1027 x 1365 gated: 43 us with the split (10), 2.9e-7 of the norm off 64 bits; three bf16 planes and a gate of its own took 74, 2.8e-6 off.
// The training step of that size 236 -> 142 (operands across K read once, not twice: 9 less; both gradients' products in one launch: 10 less, 3 of them left when
// inputs come from memory). What bounds it: shared memory, which a product of 128 columns waits for (the
// tensor pipe is 43 % busy), and 256 columns would want 128 sums to a thread.
#include <atomic>
#include <utility>

#include "gate_act.cuh"
#include "linear_common.cuh"

namespace b200 {

namespace {

constexpr int kF32Cols = 128, kF32Accs = 4, kF32MaxStages = 8;
constexpr size_t kF32Smem = static_cast<size_t>(kLinRing) + kLinEpiWarps * kLinEpiBytes + 1024 /*align*/ + 512 /*barriers*/;

// The accumulator is handed back through tensor memory's own fence; nothing in memory goes with it, so the arrival is ordered within
// the CTA alone. (With a release to the cluster each of these waited for a memory barrier: a slab took four times as long.)
__device__ __forceinline__ void mbar_arrive_of_pair(uint32_t bar_cluster) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory"); }

struct F32Params {
  int64_t M, N, kp;       // outputs; K rounded up to whole slabs of 64: planes are kp apart
  int a_rows;             // rows of the A box
  int splits, group_m, stages;
  uint32_t idesc;
  int act;
  float* side;            // gated: the projections [M, 2 N], or NULL
  const uint32_t *a_max, *b_max;  // largest magnitude of every row, as fp32 bits
};

// 2^exponent of a row or column as two factors, its halves (one cannot hold all of them); of row and column the halves are multiplied
// with each other first: powers of two, so that a sum is rounded once at most, where the result itself is subnormal
__device__ __forceinline__ float2 halves_of(uint32_t bits) {
  const int e = scale_exponent(bits), h = e >> 1;
  return make_float2(__int_as_float((h + 127) << 23), __int_as_float((e - h + 127) << 23));
}
__device__ __forceinline__ float scaled(float v, float2 row, float2 col) { return v * (row.x * col.x) * (row.y * col.y); }

// The gate of eight outputs: a call, since the exact activations are long and a tile's 32 to a thread would not fit the instruction cache
struct Eight {
  float v[8];
};
__device__ __noinline__ Eight gate_eight(int act, Eight g, Eight u) {
  gate_act_each(act, [&](auto a) {
#pragma unroll
    for (int e = 0; e < 8; ++e) g.v[e] = a.exact(g.v[e]) * u.v[e];
  });
  return g;
}

template <bool GATED> __device__ __forceinline__ void f32_out(const F32Params& p, float* out, int64_t m, int64_t n, const float* first, const float* second, bool vec) {
  const int left = p.N - n < 4 ? static_cast<int>(p.N - n) : 4;
  const float2 row = halves_of(p.a_max[m]);
  float g[4], u[4], v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    g[e] = e < left ? scaled(first[e], row, halves_of(p.b_max[n + e])) : 0.f;
    if constexpr (GATED) u[e] = e < left ? scaled(second[e], row, halves_of(p.b_max[p.N + n + e])) : 0.f;
    v[e] = g[e];
  }
  auto put = [&](float* to, const float* f) {
    if (vec) {
      *reinterpret_cast<uint4*>(to) = narrow<float>(f);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) to[e] = f[e];
    }
  };
  if constexpr (GATED) {
    if (p.side) {
      put(p.side + m * 2 * p.N + n, g);
      put(p.side + m * 2 * p.N + p.N + n, u);
    }
    gate_act_each(p.act, [&](auto act) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = act.exact(g[e]) * u[e];
    });
  }
  put(out + m * p.N + n, v);
}

constexpr int kTwo = 3;  // pairs, with two products to deal out (part 1: map_a1, map_b1, out1, p1)
template <bool GATED, int SHARE>
__device__ __forceinline__ void linear_f32_body(const CUtensorMap& map_a, const CUtensorMap& map_b, const CUtensorMap& map_a1, const CUtensorMap& map_b1, float* __restrict__ out, float* __restrict__ out1,
                                                F32Params p, F32Params p1, const TwoParts& two, uint32_t* __restrict__ status) {
  constexpr bool kPair = SHARE == kPaired || SHARE == kTwo;
  constexpr int kTileM = kPair ? 256 : 128, kW = GATED ? kF32Cols / 2 : kF32Cols;  // output columns of a tile
  constexpr uint32_t kBPlane = (kPair ? kF32Cols / 2 : kF32Cols) * kSlabBytes;      // of B in this CTA
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* epi_stage = smem + kLinRing;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kLinRing + kLinEpiWarps * kLinEpiBytes);
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(bars + 2 * kF32MaxStages + 2 * kF32Accs);
  volatile uint32_t* abort_flag = tmem_base_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem), bar_base = smem_u32(bars);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kF32MaxStages + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * kF32MaxStages + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * kF32MaxStages + kF32Accs + a); };
  const uint32_t a_plane = static_cast<uint32_t>(p.a_rows) * kSlabBytes, stage_bytes = 2 * (a_plane + kBPlane);
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
    for (int a = 0; a < kF32Accs; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), kPair ? 16 : 8);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_slot)), "r"(kF32Accs * kF32Cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_slot)), "r"(kF32Accs * kF32Cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (kPair) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  after_grids_before();
  p.a_max = waited(p.a_max);
  p.b_max = waited(p.b_max);
  p1.a_max = waited(p1.a_max);
  p1.b_max = waited(p1.b_max);

  const int64_t mt = (p.M + kTileM - 1) / kTileM, nt = (p.N + kW - 1) / kW, tiles = mt * nt;
  const int64_t tile_first = kPair ? (blockIdx.x >> 1) : SHARE == kSplit ? blockIdx.x / p.splits : blockIdx.x, tile_step = kPair ? (gridDim.x >> 1) : SHARE == kSplit ? tiles : gridDim.x;
  const int all_slabs = static_cast<int>(p.kp / 64);
  const int slabs1 = static_cast<int>(p1.kp / 64);
  const int64_t mt1 = (p1.M + kTileM - 1) / kTileM, nt1 = (p1.N + kW - 1) / kW;
  // this CTA's (pair's) n-th tile
  auto next_tile = [&](int n, int& part, int64_t& t) {
    if constexpr (SHARE == kTwo) {
      int tile = 0;
      const bool is = two_parts_tile(two, static_cast<int>(blockIdx.x >> 1), n, part, tile);
      t = tile;
      return is;
    } else {
      part = 0;
      t = tile_first + n * tile_step;
      return t < tiles;
    }
  };
  auto block_of = [&](int part, int64_t t, int& mb, int& nb) {
    if (SHARE == kTwo && part) lin_tile(t, mt1, nt1, p1.group_m, mb, nb);
    else lin_tile(t, mt, nt, p.group_m, mb, nb);
  };
  int part = 0;
  int64_t t = 0;
  const int slab0 = SHARE == kSplit ? static_cast<int>(static_cast<int64_t>(all_slabs) * rank / p.splits) : 0;
  const int slabs = SHARE == kSplit ? static_cast<int>(static_cast<int64_t>(all_slabs) * (rank + 1) / p.splits) - slab0 : all_slabs;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer: both planes of a slab of A and of B
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int n = 0; ok && next_tile(n, part, t); ++n) {
        int mb, nb;
        block_of(part, t, mb, nb);
        const bool other = SHARE == kTwo && part;
        const CUtensorMap *ma = other ? &map_a1 : &map_a, *mapb = other ? &map_b1 : &map_b;
        const int plane = static_cast<int>(other ? p1.kp : p.kp), tile_slabs = other ? slabs1 : slabs;
        const int m0 = mb * kTileM + static_cast<int>(cta_rank) * 128;
        int n0 = nb * kW;
        const int n1 = n0 + static_cast<int>(p.N);  // gated: the up rows
        if (kPair && cta_rank == 1u) n0 = GATED ? n1 : n0 + kF32Cols / 2;
        for (int kb = 0; kb < tile_slabs; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, kLinWaitNs)) { ok = false; break; }
          const uint32_t a_dst = smem_base + stage * stage_bytes, b_dst = a_dst + 2 * a_plane;
          const uint32_t bar = kPair ? map_to_cta(full_bar(stage), 0u) : full_bar(stage);
          if (!kPair) mbar_expect_tx(full_bar(stage), stage_bytes);
          else if (cta_rank == 0u) mbar_expect_tx(full_bar(stage), 2 * stage_bytes);
          for (int q = 0; q < 2; ++q) {
            const int k = (slab0 + kb) * 64 + q * plane;
            if (kPair) {
              tma_load_3d_pair(a_dst + q * a_plane, ma, bar, k, m0, 0);
              tma_load_3d_pair(b_dst + q * kBPlane, mapb, bar, k, n0, 0);
            } else {
              tma_load_3d(a_dst + q * a_plane, &map_a, bar, k, m0, 0);
              tma_load_3d(b_dst + q * kBPlane, &map_b, bar, k, n0, 0);
              if (GATED) tma_load_3d(b_dst + q * kBPlane + kBPlane / 2, &map_b, bar, k, n1, 0);
            }
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
    // ------------------------------------------------------------ MMA issuer: an accumulator to a slab
    if (cta_rank == 0u) {
      auto warp_wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, kLinWaitNs)) != 0; };
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int n = 0; ok && next_tile(n, part, t); ++n) {
        const int tile_slabs = SHARE == kTwo && part ? slabs1 : slabs;
        for (int kb = 0; kb < tile_slabs; ++kb) {
          if (!warp_wait(tempty_bar(acc), acc_phase ^ 1u) || !warp_wait(full_bar(stage), phase)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kF32Cols);
          const uint32_t a_addr = smem_base + stage * stage_bytes, b_addr = a_addr + 2 * a_plane;
          uint64_t da[2][4], db[2][4];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              da[q][k] = smem_desc(a_addr + q * a_plane + k * 32u, 16u, 1024u);
              db[q][k] = smem_desc(b_addr + q * kBPlane + k * 32u, 16u, 1024u);
            }
          }
          if (elect_one()) {
#pragma unroll
            for (int pr = 0; pr < 3; ++pr) {  // h l, l h, h h
              const int qa = pr == 1 ? 1 : 0, qb = pr == 0 ? 1 : 0;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (kPair) tc_mma_f16_pair(d_tmem, da[qa][k], db[qb][k], p.idesc, (pr | k) != 0 ? 1u : 0u);
                else tc_mma_f16(d_tmem, da[qa][k], db[qb][k], p.idesc, (pr | k) != 0 ? 1u : 0u);
              }
            }
            if (kPair) {
#pragma unroll
              for (uint32_t c = 0; c < 2; ++c) {
                tc_commit_pair(map_to_cta(empty_bar(stage), c));
                tc_commit_pair(map_to_cta(tfull_bar(acc), c));
              }
            } else {
              tc_commit(empty_bar(stage));
              tc_commit(tfull_bar(acc));
            }
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1u; }
          if (++acc == kF32Accs) { acc = 0; acc_phase ^= 1u; }
        }
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        if (status) atomicOr(status, B200_DEV_WAIT_TIMEOUT);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue: a warp has 32 rows by 64 of the 128 columns (gated: 32 gates and their 32 ups)
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t col0 = static_cast<uint32_t>(GATED ? half * 32 : half * 64), col1 = static_cast<uint32_t>(GATED ? 64 + half * 32 : half * 64 + 32);
    unsigned char* mine = epi_stage + (warp - 2) * kLinEpiBytes;
    const uint32_t tempty_target = kPair ? map_to_cta(tempty_bar(0), 0u) : 0u;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int n = 0; ok && next_tile(n, part, t); ++n) {
      int mb, nb;
      block_of(part, t, mb, nb);
      const bool other = SHARE == kTwo && part;
      const int64_t M = other ? p1.M : p.M, N = other ? p1.N : p.N;
      float* to = other ? out1 : out;
      const uint32_t *a_max = other ? p1.a_max : p.a_max, *b_max = other ? p1.b_max : p.b_max;
      const int tile_slabs = other ? slabs1 : slabs;
      const bool vec = N % 4 == 0 && ((reinterpret_cast<uintptr_t>(to) | reinterpret_cast<uintptr_t>(p.side)) & 15u) == 0;
      const int64_t mr0 = static_cast<int64_t>(mb) * kTileM + static_cast<int64_t>(cta_rank) * 128 + q * 32, n0 = static_cast<int64_t>(nb) * kW;
      const int nrows = M - mr0 < 32 ? static_cast<int>(M - mr0) : 32;
      const int64_t na = n0 + (GATED ? half * 32 : half * 64), nbb = GATED ? na : na + 32;  // first output columns of the two chunks
      const float2 row = halves_of(lane < nrows ? a_max[mr0 + lane] : 0u);
      const float2 c0 = halves_of(na + lane < N ? b_max[na + lane] : 0u), c1 = halves_of(nbb + lane < N ? b_max[(GATED ? N : 0) + nbb + lane] : 0u);
      float sum[64];
#pragma unroll
      for (int e = 0; e < 64; ++e) sum[e] = 0.f;
#pragma unroll 1
      for (int kb = 0; kb < tile_slabs; ++kb) {
        int got = 0;
        if (lane == 0) got = mbar_wait(tfull_bar(acc), acc_phase, abort_flag, kLinWaitNs) ? 1 : 0;
        got = __shfl_sync(0xffffffffu, got, 0);
        if (!got) { ok = false; break; }
        tc_fence_after();
        const uint32_t t_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * kF32Cols);
        uint32_t r[64];
        tc_ld_32x32(t_base + col0, r);
        tc_ld_32x32(t_base + col1, r + 32);
        tc_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (kPair) mbar_arrive_of_pair(tempty_target + 8u * acc);
          else mbar_arrive(tempty_bar(acc));
        }
#pragma unroll
        for (int e = 0; e < 64; ++e) sum[e] += __uint_as_float(r[e]);
        if (++acc == kF32Accs) { acc = 0; acc_phase ^= 1u; }
      }
      if (!ok) break;
      if constexpr (SHARE == kSplit) {
        // to this CTA's shared memory, where its slabs were (all of them have been multiplied)
        if (q * 32 + lane < p.a_rows) {
          unsigned char* row = smem + (q * 32 + lane) * (kF32Cols * 4 + 16);
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            *reinterpret_cast<float4*>(row + (col0 + e) * 4) = make_float4(sum[e], sum[e + 1], sum[e + 2], sum[e + 3]);
            *reinterpret_cast<float4*>(row + (col1 + e) * 4) = make_float4(sum[32 + e], sum[33 + e], sum[34 + e], sum[35 + e]);
          }
        }
        break;
      }
      // the columns' factors, one to a lane so far, to every lane by way of the staging buffer
      float2* shared = reinterpret_cast<float2*>(mine);
      __syncwarp();
      shared[lane] = c0;
      shared[32 + lane] = c1;
      __syncwarp();
#pragma unroll
      for (int e = 0; e < 64; e += 2) {
        const float4 c = *reinterpret_cast<const float4*>(shared + e);
        sum[e] = scaled(sum[e], row, make_float2(c.x, c.y));
        sum[e + 1] = scaled(sum[e + 1], row, make_float2(c.z, c.w));
      }
      if (nrows <= 0) continue;
      const int wide0 = N - na < 32 ? static_cast<int>(N - na) : 32, wide1 = N - nbb < 32 ? static_cast<int>(N - nbb) : 32;
      if constexpr (GATED) {
        if (wide0 <= 0) continue;
        if (p.side) {
          float* side = p.side + mr0 * (2 * N) + na;
          lin_store<float>(sum, mine, side, 2 * N, nrows, wide0, vec, lane);
          lin_store<float>(sum + 32, mine, side + N, 2 * N, nrows, wide0, vec, lane);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          Eight g, u;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            g.v[i] = sum[e + i];
            u.v[i] = sum[32 + e + i];
          }
          g = gate_eight(p.act, g, u);
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[e + i] = g.v[i];
        }
        lin_store<float>(sum, mine, to + mr0 * N + na, N, nrows, wide0, vec, lane);
      } else {
        if (wide0 > 0) lin_store<float>(sum, mine, to + mr0 * N + na, N, nrows, wide0, vec, lane);
        if (wide1 > 0) lin_store<float>(sum + 32, mine, to + mr0 * N + nbb, N, nrows, wide1, vec, lane);
      }
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      if (status) atomicOr(status, B200_DEV_WAIT_TIMEOUT);
    }
    __syncwarp();
  }

  if constexpr (SHARE == kSplit) {
    // every CTA of the cluster puts together its share of the tile, the CTAs' sums added in the order of their ranges of K
    cluster_sync_all();
    constexpr int kQuads = kW / 4;
    constexpr uint32_t kPitch = kF32Cols * 4 + 16;
    int mb, nb;
    lin_tile(tile_first, mt, nt, p.group_m, mb, nb);
    const int64_t mr0 = static_cast<int64_t>(mb) * 128, n0 = static_cast<int64_t>(nb) * kW;
    const bool vec = p.N % 4 == 0 && ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(p.side)) & 15u) == 0;
    const int rows = p.M - mr0 < p.a_rows ? static_cast<int>(p.M - mr0) : p.a_rows, units = rows * kQuads;
    for (int i = static_cast<int>(rank) * kLinThreads + static_cast<int>(threadIdx.x); i < units; i += p.splits * kLinThreads) {
      const int r = i / kQuads, c = (i - r * kQuads) * 4;
      if (n0 + c >= p.N) continue;
      const uint32_t at = smem_base + static_cast<uint32_t>(r) * kPitch + static_cast<uint32_t>(c) * 4;
      float g[4] = {}, u[4] = {};
      for (int k = 0; k < p.splits; ++k) {
        const uint32_t from = map_to_cta(at, static_cast<uint32_t>(k));
        const float4 v = ld_cluster<float4>(from);
        g[0] += v.x; g[1] += v.y; g[2] += v.z; g[3] += v.w;
        if constexpr (GATED) {
          const float4 w = ld_cluster<float4>(from + 64 * 4);
          u[0] += w.x; u[1] += w.y; u[2] += w.z; u[3] += w.w;
        }
      }
      f32_out<GATED>(p, out, mr0 + r, n0 + c, g, u, vec);
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
    if (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kF32Accs * kF32Cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kF32Accs * kF32Cols) : "memory");
  }
}

template <bool GATED, int SHARE>
__global__ void __launch_bounds__(kLinThreads, 1) linear_f32(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, float* __restrict__ out, F32Params p, uint32_t* __restrict__ status) {
  linear_f32_body<GATED, SHARE>(map_a, map_b, map_a, map_b, out, out, p, p, TwoParts{}, status);
}
// Two products in one launch: C = A B and C1 = A1 B1
__global__ void __launch_bounds__(kLinThreads, 1)
linear_f32_two(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_b1,
               float* __restrict__ out, float* __restrict__ out1, F32Params p, F32Params p1, TwoParts two, uint32_t* __restrict__ status) {
  linear_f32_body<false, kTwo>(map_a, map_b, map_a1, map_b1, out, out1, p, p1, two, status);
}

// ------------------------------------------------------------------ planes
struct F32Operand {
  const float* x;
  __half* to;             // [rows, 2 kp]: h, then l
  uint32_t* most;         // [rows]
  int64_t rows, K, kp, s_r, s_k;
};
// 2^-exponent as two factors (one cannot hold all of them)
struct ToScale {
  float a, b;
  bool finite;  // the whole row
  __device__ __forceinline__ explicit ToScale(uint32_t most) : finite(most < 0x7f800000u) {
    const int e = -scale_exponent(most), h = e >> 1;
    a = __int_as_float((h + 127) << 23);
    b = __int_as_float((e - h + 127) << 23);
  }
};
// A row that holds an infinity or a NaN makes no finite output, so of its elements only signs count, and which are zero or not finite: h is 1, -1 or 0, l is
// the infinity (or NaN) itself, else 0. In h h + h l + l h an infinity meets the other operand's h alone, as it would meet the element in fp32; with h infinite
// it would meet l too, which is as often zero or of the other sign, and every output of its row would be NaN.
__device__ __forceinline__ void planes_of(float x0, float x1, const ToScale& s, __half2& h, __half2& l) {
  if (!s.finite) {
    h = __floats2half2_rn(x0 == 0.f ? 0.f : copysignf(1.f, x0), x1 == 0.f ? 0.f : copysignf(1.f, x1));
    l = __floats2half2_rn(isfinite(x0) ? 0.f : x0, isfinite(x1) ? 0.f : x1);
    return;
  }
  const float y0 = x0 * s.a * s.b, y1 = x1 * s.a * s.b;
  h = __floats2half2_rn(y0, y1);
  const float2 f = __half22float2(h);
  l = __floats2half2_rn(y0 - f.x, y1 - f.y);
}

// Rows along K: a CTA to a row, read once where it fits into registers (NV pairs of elements to a thread), twice else (NV = 0). Both
// operands in one launch, the first `rows0` CTAs taking the one. UNIT: the elements of every row are contiguous.
template <int NV, bool UNIT> __global__ void __launch_bounds__(256) split_rows(F32Operand A, F32Operand B, unsigned rows0) {
  __shared__ uint32_t part[8];
  next_grid_may_start();
  after_grids_before();
  const bool second = blockIdx.x >= rows0;
  const F32Operand& P = second ? B : A;
  const int64_t r = second ? blockIdx.x - rows0 : blockIdx.x, s_k = UNIT ? 1 : P.s_k;
  const int K = static_cast<int>(P.K), kp = static_cast<int>(P.kp), first = 2 * static_cast<int>(threadIdx.x);
  const float* x = P.x + r * P.s_r;
  __half* to = P.to + r * 2 * P.kp;
  float v[NV ? NV : 1][2];
  uint32_t m = 0u;
  auto fetch = [&](int j, float* f) {
    f[0] = j < K ? x[j * s_k] : 0.f;
    f[1] = j + 1 < K ? x[(j + 1) * s_k] : 0.f;
  };
  auto look = [&](const float* f) { m = max(m, max(__float_as_uint(f[0]) & 0x7fffffffu, __float_as_uint(f[1]) & 0x7fffffffu)); };
  if constexpr (NV) {
#pragma unroll
    for (int k = 0; k < NV; ++k) fetch(first + k * 512, v[k]);
#pragma unroll
    for (int k = 0; k < NV; ++k) look(v[k]);
  } else {
    for (int j = first; j < K; j += 512) {
      fetch(j, v[0]);
      look(v[0]);
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  m = __reduce_max_sync(0xffffffffu, part[threadIdx.x & 7]);
  if (threadIdx.x == 0) P.most[r] = m;
  const ToScale scale(m);
  auto store = [&](int j, const float* f) {
    __half2 h, l;
    planes_of(f[0], f[1], scale, h, l);
    *reinterpret_cast<__half2*>(to + j) = h;
    *reinterpret_cast<__half2*>(to + kp + j) = l;
  };
  if constexpr (NV) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (first + k * 512 < kp) store(first + k * 512, v[k]);
  } else {
    for (int j = first; j < kp; j += 512) {
      fetch(j, v[0]);
      store(j, v[0]);
    }
  }
}

// Operands whose rows are contiguous across K, read once: a cluster to 32 rows, each of its CTAs with a range of `slabs` times 64 k in
// shared memory, where the largest magnitudes are found, exchanged, and the planes written from.
constexpr int kOncePitch = 33, kOnceMost = 26;  // slabs of 64 x 33 values that fit into an SM's shared memory
__global__ void __launch_bounds__(256) split_columns_once(F32Operand A, F32Operand B, unsigned tiles0, int ctas, int slabs) {
  extern __shared__ float once_tile[];
  __shared__ uint32_t part[8][32], largest[32];
  next_grid_may_start();
  after_grids_before();
  const unsigned t = blockIdx.x / static_cast<unsigned>(ctas), rank = blockIdx.x % static_cast<unsigned>(ctas);
  const bool second = t >= tiles0;
  const F32Operand& P = second ? B : A;
  const int64_t r0 = static_cast<int64_t>(second ? t - tiles0 : t) * 32, k0 = static_cast<int64_t>(rank) * slabs * 64;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int count = static_cast<int>(P.kp - k0 < slabs * 64 ? P.kp - k0 : slabs * 64);  // (a multiple of 64; 0 or less: none)
  const int64_t left = r0 + tx < P.rows ? P.K - k0 : 0;
  const float* x = P.x + (r0 + tx) * P.s_r + (k0 + ty) * P.s_k;
  uint32_t m = 0u;
  for (int base = ty; base < count; base += 128) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i, x += 8 * P.s_k) v[i] = base + 8 * i < left && base + 8 * i < count ? *x : 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
      if (base + 8 * i < count) once_tile[(base + 8 * i) * kOncePitch + tx] = v[i];
    }
  }
  part[ty][tx] = m;
  __syncthreads();
  if (ty == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max(m, part[i][tx]);
    largest[tx] = m;
  }
  const int c = threadIdx.x >> 3;
  const int64_t r = r0 + c;
  if (ctas > 1) {
    cluster_sync_all();
    m = 0u;
    for (int i = 0; i < ctas; ++i) {
      uint32_t of;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(of) : "r"(map_to_cta(smem_u32(&largest[c]), static_cast<uint32_t>(i))) : "memory");
      m = max(m, of);
    }
  } else {
    __syncthreads();
    m = largest[c];
  }
  if (r < P.rows) {
    if (rank == 0 && (threadIdx.x & 7) == 0) P.most[r] = m;
    const ToScale scale(m);
    __half* to = P.to + r * 2 * P.kp + k0;
    for (int kk = (threadIdx.x & 7) * 8; kk < count; kk += 64) {
      __half2 h[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) planes_of(once_tile[(kk + 2 * i) * kOncePitch + c], once_tile[(kk + 2 * i + 1) * kOncePitch + c], scale, h[i], l[i]);
      *reinterpret_cast<uint4*>(to + kk) = *reinterpret_cast<const uint4*>(h);
      *reinterpret_cast<uint4*>(to + P.kp + kk) = *reinterpret_cast<const uint4*>(l);
    }
  }
  if (ctas > 1) cluster_sync_all();  // nobody leaves while another reads its largest
}

// Longer ones, read twice: the largest magnitudes first (most[] is zero before; a maximum does not
// depend on its order), then tiles of 32 rows by 64 k turned in shared memory.
constexpr int kLookRows = 128;
__global__ void __launch_bounds__(256) largest_of_columns(F32Operand A, F32Operand B, unsigned blocks0) {
  __shared__ uint32_t part[8][32];
  next_grid_may_start();
  after_grids_before();
  const bool second = blockIdx.x >= blocks0;
  const F32Operand& P = second ? B : A;
  const uint32_t across = static_cast<uint32_t>((P.rows + 31) / 32), block = second ? blockIdx.x - blocks0 : blockIdx.x;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t r = static_cast<int64_t>(block % across) * 32 + tx, k0 = static_cast<int64_t>(block / across) * kLookRows + ty;
  uint32_t m = 0u;
  if (r < P.rows) {
    const float* x = P.x + r * P.s_r + k0 * P.s_k;
    const int64_t step = 8 * P.s_k;
    const int left = static_cast<int>(P.K - k0 < kLookRows ? P.K - k0 : kLookRows);
    float v[kLookRows / 8];
#pragma unroll
    for (int i = 0; i < kLookRows / 8; ++i, x += step) v[i] = 8 * i < left ? *x : 0.f;
#pragma unroll
    for (int i = 0; i < kLookRows / 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  part[ty][tx] = m;
  __syncthreads();
  if (ty == 0 && r < P.rows) {
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max(m, part[i][tx]);
    atomicMax(P.most + r, m);
  }
}
__global__ void __launch_bounds__(256) split_columns(F32Operand A, F32Operand B, unsigned blocks0) {
  __shared__ float tile[64][33];
  next_grid_may_start();
  after_grids_before();
  const bool second = blockIdx.x >= blocks0;
  const F32Operand& P = second ? B : A;
  const uint32_t across = static_cast<uint32_t>((P.rows + 31) / 32), block = second ? blockIdx.x - blocks0 : blockIdx.x;
  const int64_t r0 = static_cast<int64_t>(block % across) * 32, k0 = static_cast<int64_t>(block / across) * 64;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t left = P.K - k0 - ty;  // of K, from this thread's first row on
  const float* x = P.x + (r0 + tx) * P.s_r + (k0 + ty) * P.s_k;
  const bool in = r0 + tx < P.rows;
#pragma unroll
  for (int i = 0; i < 8; ++i, x += 8 * P.s_k) tile[ty + 8 * i][tx] = in && 8 * i < left ? *x : 0.f;
  __syncthreads();
  const int c = threadIdx.x >> 3, kk = (threadIdx.x & 7) * 8;
  const int64_t r = r0 + c;
  if (r >= P.rows) return;
  const ToScale scale(P.most[r]);
  __half2 h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) planes_of(tile[kk + 2 * i][c], tile[kk + 2 * i + 1][c], scale, h[i], l[i]);
  __half* to = P.to + r * 2 * P.kp + k0 + kk;  // (kp is a multiple of 64)
  *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(h);
  *reinterpret_cast<uint4*>(to + P.kp) = *reinterpret_cast<const uint4*>(l);
}

// ------------------------------------------------------------------ host side
int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
struct F32Plan {
  int share, splits;
  double us;
};
// us: splitting and starting 9, a slab 0.62 in a pair and 0.88 on a CTA of its own. Pairs or ranges, both measured: 500 x 2000 x 700 31.8 in pairs, 28.7 in two
// ranges; 1024 x 1024 x 1024 22.1 in pairs, 25.6 on single CTAs; 200 x 4096 x 300 43.7, 63.6, 19.0 in eight ranges.
F32Plan plan_f32(int64_t M, int64_t N, int64_t kp, bool gated) {
  const int64_t w = gated ? kF32Cols / 2 : kF32Cols, nt = (N + w - 1) / w, slabs = kp / 64;
  F32Plan best{kSingle, 1, 0.};
  double least = 1e30;
  auto offer = [&](int share, int splits, double t) {
    if (t < least) { least = t; best = F32Plan{share, splits, t}; }
  };
  if (M > 128) {
    const int64_t tiles = (M + 255) / 256 * nt, rounds = (tiles + kNumSMs / 2 - 1) / (kNumSMs / 2);
    offer(kPaired, 1, 9. + static_cast<double>(rounds) * (1.5 + 0.62 * static_cast<double>(slabs)));
  }
  const int64_t tiles = (M + 127) / 128 * nt;
  for (int s : {1, 2, 3, 4, 6, 8}) {
    if (s > slabs || (s > 1 && tiles * s > kResident[s])) continue;
    const int64_t rounds = s > 1 ? 1 : (tiles + kNumSMs - 1) / kNumSMs;
    offer(s > 1 ? kSplit : kSingle, s, 9. + static_cast<double>(rounds) * (1.5 + 0.88 * static_cast<double>((slabs + s - 1) / s)) + (s > 1 ? 1.5 : 0.));
  }
  return best;
}

bool encode_planes(CUtensorMap* map, const __half* planes, int64_t rows, int64_t kp, int box_rows) {
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(2 * kp), static_cast<cuuint64_t>(rows), 1};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(4 * kp), static_cast<cuuint64_t>(4 * kp) * static_cast<cuuint64_t>(rows)};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(planes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool GATED, int SHARE>
int launch_f32(int cluster, int64_t ctas, cudaStream_t st, const CUtensorMap& map_a, const CUtensorMap& map_b, float* out, const F32Params& p, uint32_t* status) {
  const auto kernel = linear_f32<GATED, SHARE>;
  static std::atomic<uint64_t> allowed{0};  // devices on which this kernel may have that much shared memory
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kF32Smem));
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) { set_last_cuda_error(e); return B200_ELAUNCH; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(kLinThreads, 1, 1);
  cfg.dynamicSmemBytes = kF32Smem;
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

// Eight slabs to a CTA, or fewer where that makes fewer than two CTAs to an SM. `done` stays false where the columns are too long for a
// cluster, or the cluster is refused.
cudaError_t launch_once(const F32Operand* across, int64_t tiles0, int64_t tiles, int64_t slabs, cudaStream_t st, bool& done) {
  int64_t ctas = (slabs + 7) / 8;
  if (tiles * ctas < 2 * kNumSMs) ctas = (2 * kNumSMs + tiles - 1) / tiles;
  ctas = ctas < slabs ? ctas : slabs;
  ctas = ctas < 8 ? ctas : 8;
  const int64_t each = (slabs + ctas - 1) / ctas;
  if (each > kOnceMost || tiles * ctas > 0x7fffffff) return cudaSuccess;
  static std::atomic<uint64_t> allowed{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(split_columns_once, cudaFuncAttributeMaxDynamicSharedMemorySize, kOnceMost * 64 * kOncePitch * 4);
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * ctas));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = static_cast<size_t>(each) * 64 * kOncePitch * 4;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // (see launch_after)
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  done = cudaLaunchKernelEx(&cfg, split_columns_once, across[0], across[1], static_cast<unsigned>(tiles0), static_cast<int>(ctas), static_cast<int>(each)) == cudaSuccess;
  if (!done) (void)cudaGetLastError();
  return cudaSuccess;
}

// The planes of both operands of a product, whose magnitudes lie side by side
int make_planes(const F32Operand& a, const F32Operand& b, cudaStream_t st, int& launches) {
  // rows that lie along K, and those that lie across it
  F32Operand along[2], across[2];
  int n_along = 0, n_across = 0;
  const int64_t K = a.K, kp = a.kp;
  cudaError_t le = cudaSuccess;
  for (const F32Operand* o : {&a, &b}) {
    if (o->s_k == 1 || (o->s_r != 1 && o->rows > 1)) along[n_along++] = *o;
    else across[n_across++] = *o;
  }
  bool once = false;
  if (n_across) {
    if (n_across == 1) across[1] = F32Operand{};
    const int64_t tiles0 = (across[0].rows + 31) / 32, tiles = tiles0 + (across[1].rows + 31) / 32;
    const cudaError_t e = launch_once(across, tiles0, tiles, kp / 64, st, once);
    if (e != cudaSuccess) { set_last_cuda_error(e); return B200_ELAUNCH; }
    if (once) ++launches;
  }
  if (n_across && !once) {
    const cudaError_t e = cudaMemsetAsync(across[0].most, 0, static_cast<size_t>((n_across == 2 ? a.rows + b.rows : across[0].rows) * 4), st);
    if (e != cudaSuccess) { set_last_cuda_error(e); return B200_ELAUNCH; }
    auto blocks = [&](int i, int64_t step, int64_t k) { return i < n_across ? (across[i].rows + 31) / 32 * ((k + step - 1) / step) : 0; };
    le = launch_after(largest_of_columns, blocks(0, kLookRows, K) + blocks(1, kLookRows, K), 256, 0, st, across[0], across[1], static_cast<unsigned>(blocks(0, kLookRows, K)));
    if (le == cudaSuccess) le = launch_after(split_columns, blocks(0, 64, kp) + blocks(1, 64, kp), 256, 0, st, across[0], across[1], static_cast<unsigned>(blocks(0, 64, kp)));
    launches += 2;
  }
  if (n_along) {
    if (n_along == 1) along[1] = F32Operand{};
    const unsigned grid = static_cast<unsigned>(along[0].rows + along[1].rows), rows0 = static_cast<unsigned>(along[0].rows);
    const bool unit = along[0].s_k == 1 && (n_along == 1 || along[1].s_k == 1);
    auto go = [&](auto kernel) {
      if (le == cudaSuccess) le = launch_after(kernel, grid, 256, 0, st, along[0], along[1], rows0);
    };
    if (kp <= 1024) unit ? go(split_rows<2, true>) : go(split_rows<2, false>);
    else if (kp <= 2048) unit ? go(split_rows<4, true>) : go(split_rows<4, false>);
    else if (kp <= 4096) unit ? go(split_rows<8, true>) : go(split_rows<8, false>);
    else unit ? go(split_rows<0, true>) : go(split_rows<0, false>);
    ++launches;
  }
  if (le != cudaSuccess) { set_last_cuda_error(le); return B200_ELAUNCH; }
  return B200_OK;
}

template <bool GATED>
int run_f32(const float* A, const float* B, float* out, int64_t M, int64_t N, int64_t K, int64_t sAm, int64_t sAk, int64_t sBn, int64_t sBk, int act, float* side, void* scratch, uint32_t* status, cudaStream_t st) {
  if (!encode_fn()) return B200_EDRIVER;
  const int64_t rows_b = GATED ? 2 * N : N, kp = up_to(K, 64);
  unsigned char* at = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(scratch) + 255) & ~static_cast<uintptr_t>(255));
  uint32_t* most = reinterpret_cast<uint32_t*>(at);
  __half* planes = reinterpret_cast<__half*>(at + up_to((M + rows_b) * 4, 256));
  const F32Operand a{A, planes, most, M, K, kp, sAm, sAk}, b{B, planes + M * 2 * kp, most + M, rows_b, K, kp, sBn, sBk};
  int launches = 1;
  const int planes_rc = make_planes(a, b, st, launches);
  if (planes_rc) return planes_rc;
  F32Params p{};
  p.M = M;
  p.N = N;
  p.kp = kp;
  p.act = act;
  p.side = side;
  p.a_max = a.most;
  p.b_max = b.most;
  int64_t rows = (32ll << 20) / (4 * kp) / 256 * 256;  // a group's panel of A stays in L2 while B goes by
  rows = rows < 2048 ? 2048 : rows > 65536 ? 65536 : rows;
  auto run = [&](const F32Plan& plan) -> int {
    const bool pair = plan.share == kPaired;
    const int tile_m = pair ? 256 : 128;
    const int64_t w = GATED ? kF32Cols / 2 : kF32Cols, tiles = (M + tile_m - 1) / tile_m * ((N + w - 1) / w), slots = pair ? kNumSMs / 2 : kNumSMs, resident = tiles < slots ? tiles : slots;
    p.a_rows = pair || M >= 128 ? 128 : static_cast<int>(up_to(M, 8));
    p.splits = plan.splits;
    p.group_m = static_cast<int>(rows / tile_m);
    const int stage = 2 * (p.a_rows + (pair ? kF32Cols / 2 : kF32Cols)) * kSlabBytes, fit = kLinRing / stage;
    p.stages = fit < kF32MaxStages ? fit : kF32MaxStages;
    p.idesc = (1u << 4) | (static_cast<uint32_t>(kF32Cols >> 3) << 17) | (static_cast<uint32_t>(tile_m >> 4) << 24);  // f16 operands, fp32 sums
    alignas(64) CUtensorMap map_a, map_b;
    if (!encode_planes(&map_a, a.to, M, kp, p.a_rows) || !encode_planes(&map_b, b.to, rows_b, kp, pair || GATED ? kF32Cols / 2 : kF32Cols)) return B200_EDRIVER;
    if (pair) return launch_f32<GATED, kPaired>(2, 2 * resident, st, map_a, map_b, out, p, status);
    if (plan.share == kSplit) return launch_f32<GATED, kSplit>(plan.splits, tiles * plan.splits, st, map_a, map_b, out, p, status);
    return launch_f32<GATED, kSingle>(1, resident, st, map_a, map_b, out, p, status);
  };
  const F32Plan plan = plan_f32(M, N, kp, GATED);
  int rc = run(plan);
  if (rc == B200_ELAUNCH && plan.share != kSingle) {  // the cluster launch was refused: the same on single CTAs
    (void)cudaGetLastError();
    rc = run(F32Plan{kSingle, 1, 0.});
  }
  if (rc) return rc;
  return check_launch(launches);
}

int64_t f32_scratch(int64_t M, int64_t rows_b, int64_t K) { return 256 + up_to((M + rows_b) * 4, 256) + (M + rows_b) * up_to(K, 64) * 4; }
bool f32_sizes(int64_t M, int64_t rows_b, int64_t K) { return M >= 1 && rows_b >= 1 && K >= 1 && M <= 0x7fffffff && rows_b <= 0x7fffffff && K <= (1ll << 29) && M + rows_b <= 0x7fffffff; }

// Both gradients of y = x w^T, dx = g w and dw = g^T x: four sets of planes (g's rows for the one are its columns for the other), one launch for the
// products (see TwoParts; fp32 1531 x 2730 x 1027: 54 tiles of 43 slabs and 99 of 24).
bool grads_pay(int64_t M, int64_t J, int64_t K) {
  if (!f32_sizes(M, K, J) || !f32_sizes(J, K, M) || M <= 128 || J <= 128) return false;
  const int64_t kx = up_to(J, 64), kw = up_to(M, 64), nt = (K + kF32Cols - 1) / kF32Cols;
  const TwoTimes t((M + 255) / 256 * nt, (J + 255) / 256 * nt, 1. + 0.62 * static_cast<double>(kx / 64), 1. + 0.62 * static_cast<double>(kw / 64));
  if (t.tiles[0] > (1 << 29) || t.tiles[1] > (1 << 29)) return false;  // (they are counted in 32 bits)
  const double shorter = t.tile[1 - t.first], together = 9. + (t.longest > t.even + 0.5 * shorter ? t.longest : t.even + 0.5 * shorter);
  // (0.8: a slab takes longer where every pair is at work. 206 sizes that this lets through: 16 % faster on average, 4 % slower at most)
  return together < 0.8 * (plan_f32(M, K, kx, false).us + plan_f32(J, K, kw, false).us);
}
int run_grads(const float* g, const float* x, const float* w, float* dx, float* dw, int64_t M, int64_t J, int64_t K, const int64_t* s, void* scratch, uint32_t* status, cudaStream_t st) {
  if (!encode_fn()) return B200_EDRIVER;
  unsigned char* at = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(scratch) + 255) & ~static_cast<uintptr_t>(255));
  int launches = 1;
  alignas(64) CUtensorMap maps[4];
  F32Params p[2] = {};
  for (int i = 0; i < 2; ++i) {
    const int64_t rows = i ? J : M, contraction = i ? M : J, kp = up_to(contraction, 64);
    p[i].M = rows;
    p[i].N = K;
    p[i].kp = kp;
    p[i].a_rows = 128;
    p[i].splits = 1;
    const int64_t group = (32ll << 20) / (4 * kp) / 256 * 256;  // (see run_f32)
    p[i].group_m = static_cast<int>((group < 2048 ? 2048 : group > 65536 ? 65536 : group) / 256);
    p[i].stages = kLinRing / (2 * (128 + kF32Cols / 2) * kSlabBytes);
    p[i].idesc = (1u << 4) | (static_cast<uint32_t>(kF32Cols >> 3) << 17) | (16u << 24);  // f16 operands, fp32 sums
    if (!(i ? dw : dx)) continue;
    uint32_t* most = reinterpret_cast<uint32_t*>(at);
    __half* planes = reinterpret_cast<__half*>(at + up_to((rows + K) * 4, 256));
    const F32Operand a{g, planes, most, rows, contraction, kp, i ? s[1] : s[0], i ? s[0] : s[1]};
    const F32Operand b{i ? x : w, planes + rows * 2 * kp, most + rows, K, contraction, kp, i ? s[3] : s[5], i ? s[2] : s[4]};
    const int rc = make_planes(a, b, st, launches);
    if (rc) return rc;
    if (!encode_planes(&maps[2 * i], a.to, rows, kp, 128) || !encode_planes(&maps[2 * i + 1], b.to, K, kp, kF32Cols / 2)) return B200_EDRIVER;
    p[i].a_max = a.most;
    p[i].b_max = b.most;
    at += up_to(f32_scratch(rows, K, contraction) - 256, 256);
  }
  for (int i = 0; i < 2; ++i) {  // a gradient that nobody wants has no tiles
    if (i ? dw : dx) continue;
    maps[2 * i] = maps[2 - 2 * i];
    maps[2 * i + 1] = maps[3 - 2 * i];
    p[i].a_max = p[1 - i].a_max;
    p[i].b_max = p[1 - i].b_max;
  }
  const int64_t nt = (K + kF32Cols - 1) / kF32Cols;
  const double tile[2] = {1. + 0.62 * static_cast<double>(p[0].kp / 64), 1. + 0.62 * static_cast<double>(p[1].kp / 64)};
  const TwoParts two = two_parts(tile[1] > tile[0] ? 1 : 0, dx ? (M + 255) / 256 * nt : 0, dw ? (J + 255) / 256 * nt : 0, tile);
  static std::atomic<uint64_t> allowed{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(linear_f32_two, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kF32Smem));
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) { set_last_cuda_error(e); return B200_ELAUNCH; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * two.pairs), 1, 1);
  cfg.blockDim = dim3(kLinThreads, 1, 1);
  cfg.dynamicSmemBytes = kF32Smem;
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
  e = cudaLaunchKernelEx(&cfg, linear_f32_two, maps[0], maps[1], maps[2], maps[3], dx, dw, p[0], p[1], two, status);
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

// Splitting costs a pass over both operands, and a tile has 128 rows: it pays where there is work enough for each of them
// (below, the package's other fp32 products take the call).
extern "C" int64_t b200_linear_f32_scratch_bytes(int64_t M, int64_t N, int64_t K) {
  if (!f32_sizes(M, N, K) || !encode_fn()) return 0;
  if (M <= 32 || N <= 32 || K < 32 || static_cast<double>(M) * static_cast<double>(N) * static_cast<double>(K) < 67108864.) return 0;
  return f32_scratch(M, N, K);
}

extern "C" int b200_linear_f32(const float* A, const float* B, float* C, int64_t M, int64_t N, int64_t K, int64_t sAm, int64_t sAk, int64_t sBk, int64_t sBn, void* scratch, int64_t scratch_bytes,
                               uint32_t* status, void* stream) {
  if (!f32_sizes(M, N, K) || !A || !B || !C) return B200_EINVAL;
  if (!scratch || scratch_bytes < f32_scratch(M, N, K)) return B200_ESCRATCH;
  return run_f32<false>(A, B, C, M, N, K, sAm, sAk, sBn, sBk, 0, nullptr, scratch, status, static_cast<cudaStream_t>(stream));
}

extern "C" int b200_gated_linear_f32(const float* x, const float* w, float* out, float* projections, int64_t M, int64_t N, int64_t K, int64_t sxm, int64_t sxk, int64_t swn, int64_t swk, int activation,
                                     void* scratch, int64_t scratch_bytes, uint32_t* status, void* stream) {
  if (N < 1 || N > 0x3fffffff || !f32_sizes(M, 2 * N, K) || activation < 0 || activation >= B200_ACT_COUNT || !x || !w || !out) return B200_EINVAL;
  if (!scratch || scratch_bytes < f32_scratch(M, 2 * N, K)) return B200_ESCRATCH;
  return run_f32<true>(x, w, out, M, N, K, sxm, sxk, swn, swk, activation, projections, scratch, status, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t b200_linear_f32_grads_scratch_bytes(int64_t M, int64_t J, int64_t K) {
  if (M < 1 || J < 1 || K < 1 || b200_linear_f32_scratch_bytes(M, K, J) <= 0 || b200_linear_f32_scratch_bytes(J, K, M) <= 0 || !grads_pay(M, J, K)) return -1;
  return f32_scratch(M, K, J) + 256 + f32_scratch(J, K, M);
}

extern "C" int b200_linear_f32_grads(const float* g, const float* x, const float* w, float* dx, float* dw, int64_t M, int64_t J, int64_t K, int64_t sgm, int64_t sgj, int64_t sxm, int64_t sxk, int64_t swj,
                                     int64_t swk, void* scratch, int64_t scratch_bytes, uint32_t* status, void* stream) {
  if (!g || !x || !w || (!dx && !dw)) return B200_EINVAL;
  const int64_t need = b200_linear_f32_grads_scratch_bytes(M, J, K), s[6] = {sgm, sgj, sxm, sxk, swj, swk};
  if (need < 0) return B200_EINVAL;
  if (!scratch || scratch_bytes < need) return B200_ESCRATCH;
  return run_grads(g, x, w, dx, dw, M, J, K, s, scratch, status, static_cast<cudaStream_t>(stream));
}
