// What the kernels of linear_tc.cu, linear_f32.cu and linear_grads.cu share: sizes, the order of tiles, two products in one launch, stores of
// 32 x 32 values, shared memory of a cluster, operands copied to lines.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "b200_common.cuh"
#include "tc_common.cuh"

namespace b200 {

constexpr int kLinThreads = 320;                        // TMA warp, MMA warp, 8 epilogue warps
constexpr int kSlabBytes = 128;                         // of K to a slab: one row of the 128-byte swizzle
constexpr int kLinRing = 192 * 1024;
constexpr int kLinEpiWarps = 8, kLinEpiBytes = 4096;    // staging: 32 rows x 128 bytes per epilogue warp
constexpr uint64_t kLinWaitNs = 2000000000ull;          // every mbarrier wait gives up after 2 s
enum : int { kSingle = 0, kPaired = 1, kSplit = 2 };  // a CTA to a tile; a pair to a tile of 256 rows; a cluster that shares a tile's K

// CTAs of a whole SM's shared memory that are resident at once in clusters of 1 .. 8 (cudaOccupancyMaxActiveClusters on a B200)
constexpr int kResident[9] = {0, 148, 148, 135, 132, 130, 132, 105, 120};

__device__ __forceinline__ void prefetch_l2_3d(const CUtensorMap* map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(map), "r"(c0), "r"(c1), "r"(c2) : "memory");
}

__device__ __forceinline__ void lin_tile(int64_t t, int64_t mt, int64_t nt, int group_m, int& mb, int& nb) {
  const int64_t per_group = static_cast<int64_t>(group_m) * nt;
  const int64_t g = t / per_group, in_g = t - g * per_group;
  const int64_t left = mt - g * group_m, gm = left < group_m ? left : group_m;
  mb = static_cast<int>(g * group_m + in_g % gm);
  nb = static_cast<int>(in_g / gm);
}

// Two products in one launch, dealt to pairs of CTAs. The tiles of the one with the longer contraction (`first`, 0 or 1) go round; the pairs that
// have one less (all but the first `late`) take `head` tiles of the other each meanwhile, and the rest of its `tiles` goes round again, so that
// pairs at work at one time have neighbouring tiles.
struct TwoParts {
  int pairs, first, rounds, late, head, tiles;
};
__device__ __forceinline__ bool two_parts_tile(const TwoParts& p, int pair, int n, int& part, int& tile) {  // the n-th of a pair
  const int mine = p.rounds + (pair < p.late ? 1 : 0), early = p.late ? p.pairs - p.late : 0;
  if (n < mine) {
    part = p.first;
    tile = n * p.pairs + pair;
    return true;
  }
  part = 1 - p.first;
  n -= mine;
  if (early && pair >= p.late) {
    if (n < p.head) {
      tile = n * early + (pair - p.late);
      return tile < p.tiles;
    }
    n -= p.head;
  }
  tile = p.head * early + n * p.pairs + pair;
  return tile < p.tiles;
}
// us, by what a tile of each takes: the one with the longer tiles by itself; both dealt out evenly
struct TwoTimes {
  int64_t tiles[2];
  double tile[2], longest, even;
  int first;
  TwoTimes(int64_t tiles0, int64_t tiles1, double tile0, double tile1) : tiles{tiles0, tiles1}, tile{tile0, tile1}, first(tile1 > tile0 ? 1 : 0) {
    const int pairs = kNumSMs / 2;
    longest = static_cast<double>((tiles[first] + pairs - 1) / pairs) * tile[first];
    even = (static_cast<double>(tiles[0]) * tile[0] + static_cast<double>(tiles[1]) * tile[1]) / pairs;
  }
};
inline TwoParts two_parts(int first, int64_t tiles0, int64_t tiles1, const double* tile) {
  TwoParts p{};
  const int64_t tiles[2] = {tiles0, tiles1};
  p.pairs = kNumSMs / 2;
  p.first = first;
  p.rounds = static_cast<int>(tiles[first] / p.pairs);
  p.late = static_cast<int>(tiles[first] % p.pairs);
  p.head = p.late ? static_cast<int>(tile[first] / tile[1 - first] + 0.5) : 0;
  p.tiles = static_cast<int>(tiles[1 - first]);
  return p;
}

// Rows scaled by a power of two for f16, so that their largest magnitude (as fp32 bits) lies in [2^14, 2^15): its exponent, 2^-exponent being the scale
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
  const int e = static_cast<int>(bits >> 23);
  return bits == 0u ? 0 : (e == 255 ? 254 : e) - 141;
}
// 2^exponent, and 2^-exponent, in one float each: exponents below -100 count as that, which takes rows whose largest is below 2^-86 (times f16
// operands they make no f16 result but zero)
__device__ __forceinline__ int bounded_exponent(uint32_t bits) { return max(scale_exponent(bits), -100); }
__device__ __forceinline__ float row_factor(uint32_t bits) { return __int_as_float((127 + bounded_exponent(bits)) << 23); }
__device__ __forceinline__ float row_scale(uint32_t bits) { return __int_as_float((127 - bounded_exponent(bits)) << 23); }

// 16 bytes of a cluster CTA's shared memory
template <typename V> __device__ __forceinline__ V ld_cluster(uint32_t from) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
  return *reinterpret_cast<const V*>(&v);
}

// What is staged (see lin_store) to rows off the grid: a column to a lane, eight rows on their way together. (A call, so that
// its registers are not the epilogue's.)
template <typename TO> __device__ __noinline__ void lin_copy_ragged(const unsigned char* mine, TO* out, int64_t pitch, int nrows, int ncols, int lane) {
  constexpr int kRow = 32 * static_cast<int>(sizeof(TO)), kPieces = kRow / 16, kPer = 16 / static_cast<int>(sizeof(TO)), kShift = sizeof(TO) == 2 ? 1 : 0;
  const unsigned char* from = mine + lane % kPer * static_cast<int>(sizeof(TO));
  const int j = lane / kPer;
  out += lane;
  auto rows = [&](int r0, auto whole) {
    TO w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const TO*>(from + i * kRow + ((j ^ ((i >> kShift) & (kPieces - 1))) << 4));
#pragma unroll
    for (int i = 0; i < 8; ++i, out += pitch)
      if (decltype(whole)::value || (lane < ncols && r0 + i < nrows)) *out = w[i];
  };
  if (nrows >= 32 && ncols >= 32) {
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 8, from += 8 * kRow) rows(r0, std::true_type{});
  } else {
#pragma unroll 1
    for (int r0 = 0; r0 < nrows; r0 += 8, from += 8 * kRow) rows(r0, std::false_type{});
  }
}

// 32 values of a lane's row to 32 columns of `out` (row pitch `pitch`, column 0 at `col`): rounded once into the warp's
// staging buffer (16-byte pieces swizzled so that neither side meets a bank twice), then out in 16-byte pieces of
// eight (fp32: four) rows at a time, or element by element where rows are off the grid.
template <typename TO>
__device__ __forceinline__ void lin_store(const float* v, unsigned char* mine, TO* out, int64_t pitch, int nrows, int ncols, bool vec, int lane) {
  constexpr int kRow = 32 * static_cast<int>(sizeof(TO)), kPieces = kRow / 16, kPer = 16 / static_cast<int>(sizeof(TO)), kShift = sizeof(TO) == 2 ? 1 : 0;
  __syncwarp();  // what was there has been read out
#pragma unroll
  for (int j = 0; j < kPieces; ++j) *reinterpret_cast<uint4*>(mine + lane * kRow + ((j ^ ((lane >> kShift) & (kPieces - 1))) << 4)) = narrow<TO>(v + j * kPer);
  __syncwarp();
  if (vec) {
    constexpr int kRowsAt = 32 / kPieces;
    const int j = lane % kPieces, r0 = lane / kPieces;
    if (j * kPer < ncols) {
#pragma unroll 4
      for (int i = 0; i < kPieces; ++i) {
        const int r = r0 + i * kRowsAt;
        if (r < nrows) *reinterpret_cast<uint4*>(out + static_cast<int64_t>(r) * pitch + j * kPer) = *reinterpret_cast<const uint4*>(mine + r * kRow + ((j ^ ((r >> kShift) & (kPieces - 1))) << 4));
      }
    }
  } else {
    lin_copy_ragged<TO>(mine, out, pitch, nrows, ncols, lane);
  }
}

// An operand [rows, K] that the copy engine reads along K
struct LinOperand {
  const void* base;
  int64_t rows, K, s_r, s_k;
  int esize;
  int64_t reads;  // how many tiles read a row
  bool ready() const {  // as the copy engine takes it, and a copy would not pay
    return aligned16(base) && (s_k == 1 || K == 1) && (rows == 1 || (s_r >= K && s_r * esize % 16 == 0)) && !better_copied();
  }
  // Rows on the 16-byte grid but across lines of 128: every slab of a row that a tile reads takes a second line, 4.5 ps of the whole device
  // each time (2.9 to 6.7 over nine sizes); a copy takes 3e-5 us a slab once, more where it does not fit into L2, and a launch. bf16 gated 8192 x 4088 x 11008:
  // 1345 us as they are, 1046 copied, 914 with rows on lines; 512 x 4088 x 11008 107, 87 with the input alone copied, 76; 128 x 2040 x 5504 stays at 17 (14), where copies
  // would make it 29.
  bool better_copied() const {
    const bool lines = (reinterpret_cast<uintptr_t>(base) & 127u) == 0 && (rows == 1 || s_r * esize % 128 == 0);
    if (lines || rows == 1 || K * esize <= 128) return false;
    const double slabs = static_cast<double>(rows) * static_cast<double>((K * esize + kSlabBytes - 1) / kSlabBytes);
    return slabs * (4.5e-6 * static_cast<double>(reads) - (slabs * kSlabBytes > 64e6 ? 4.5e-5 : 3e-5)) > 1.5;
  }
  int64_t pitch() const { return K * esize > 128 ? (K * esize + 127) / 128 * 128 / esize : (K * esize + 15) / 16 * 16 / esize; }
  int64_t packed_bytes() const { return ready() ? 0 : (rows * pitch() * esize + 255) / 256 * 256; }
};
// The operands that are not ready are copied behind `at`, and become their copies.
void lin_pack(LinOperand& a, LinOperand& b, unsigned char* at, cudaStream_t st, int& launches);

}  // namespace b200
