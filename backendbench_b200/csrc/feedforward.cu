// What stands around the products of a feed-forward block: the gate of a projection pair and its gradient, dropout
// whose mask is drawn from a counter, and the quantisation of rows to 8 bits. All are one pass over their data.
#include <type_traits>

#include "b200_common.cuh"
#include "gate_act.cuh"
#include "linear_common.cuh"

namespace b200 {

namespace {

constexpr int kFfThreads = 256;

// ------------------------------------------------------------------ the gate
// h = act(g) * u of fp32 projections P = [g | u] (M x 2 N). The tensor-core products form the gate on their sums; small fp32 ones (b200_linear_f32_scratch_bytes
// gives 0) are the package's other fp32 products, which know no gate, so it has a kernel of its own for them.
// Backward: dP = [dh * u * act'(g) | dh * act(g)], rounded to the type of the operands it is multiplied by next, in rows of any pitch.
template <int N> __device__ __forceinline__ void load_f32(const float* p, float* v) {
#pragma unroll
  for (int e = 0; e < N; e += 4) widen<float>(ld_stream(p + e), v + e);
}
__device__ __forceinline__ int64_t row_of(int64_t i, int64_t per_row, int64_t total) {
  return total <= 0xffff0000ll ? static_cast<uint32_t>(i) / static_cast<uint32_t>(per_row) : i / per_row;  // (i may run past total, by less than four CTAs' worth)
}

// Rows off the grid: four single elements to a thread, a CTA's width apart and all on their way together (backward, bf16 4096 x 5501:
// 64 us, 48 for 5504 columns).
// The row of element span + offset of a matrix of N columns, when element `span` is in row m0 and column c0: past the row's
// end a wide matrix has one more row to go, a narrow one takes a division of small numbers.
__device__ __forceinline__ int64_t row_behind(int offset, int64_t m0, int64_t c0, int64_t N) {
  const int64_t past = c0 + offset;
  return m0 + (N >= 4 * kFfThreads ? (past >= N ? 1 : 0) : static_cast<uint32_t>(past) / static_cast<uint32_t>(N));
}

template <typename ACT, bool VECTOR>
__global__ void __launch_bounds__(kFfThreads) gate_forward(const float* p, float* __restrict__ h, int64_t M, int64_t N) {
  if constexpr (VECTOR) {
    const int64_t per_row = N / 4, total = M * per_row;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kFfThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kFfThreads) {
      const int64_t m = row_of(i, per_row, total);
      const float* row = p + i * 4 + m * N;  // m rows of 2 N, not N, lie before
      float g[4], u[4];
      load_f32<4>(row, g);
      load_f32<4>(row + N, u);
#pragma unroll
      for (int e = 0; e < 4; ++e) g[e] = ACT::template f<false>(g[e]) * u[e];
      *reinterpret_cast<uint4*>(h + i * 4) = narrow<float>(g);
    }
  } else {
    const int64_t total = M * N;
    for (int64_t span = static_cast<int64_t>(blockIdx.x) * (4 * kFfThreads); span < total; span += static_cast<int64_t>(gridDim.x) * (4 * kFfThreads)) {
      const int64_t m0 = row_of(span, N, total), c0 = span - m0 * N, i0 = span + threadIdx.x;
      float g[4], u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t i = i0 + e * kFfThreads, at = i + row_behind(static_cast<int>(threadIdx.x) + e * kFfThreads, m0, c0, N) * N;  // (m rows of 2 N, not N, lie before)
        g[e] = i < total ? p[at] : 0.f;
        u[e] = i < total ? p[at + N] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i0 + e * kFfThreads < total) h[i0 + e * kFfThreads] = ACT::template f<false>(g[e]) * u[e];
    }
  }
}

// Four elements of a row on the grid of four
template <typename T> __device__ __forceinline__ void load_four_floats(const T* p, float* v) {
  if constexpr (sizeof(T) == 4) {
    widen<float>(ld_stream(p), v);
  } else {
    uint2 w;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "l"(p));
    float out[8];
    widen<T>(make_uint4(w.x, w.y, 0u, 0u), out);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = out[e];
  }
}
template <typename T> __device__ __forceinline__ void store_four(T* p, const float* v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<uint4*>(p) = narrow<float>(v);
  } else {
    const float w[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
    const uint4 r = narrow<T>(w);
    *reinterpret_cast<uint2*>(p) = make_uint2(r.x, r.y);
  }
}
template <typename T, typename ACT, bool VECTOR>
__global__ void __launch_bounds__(kFfThreads) gate_backward(const T* dh, const float* p, T* __restrict__ dp, int64_t M, int64_t N, int64_t pitch) {
  auto slope = [](float& d, float& g, float& u) {
    float a, s;
    ACT::template both<sizeof(T) == 2>(g, a, s);
    g = d * u * s;
    u = d * a;
  };
  if constexpr (VECTOR) {
    // Four elements to a thread whatever the type: 16 bytes of a projection, so that a warp's loads are whole lines (bf16 4096 x 11008: 133 us with
    // eight, whose loads are every second 16 bytes, 96 so: the memory's own time).
    const int64_t per_row = N / 4, total = M * per_row;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kFfThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kFfThreads) {
      const int64_t m = row_of(i, per_row, total), at = i * 4 + m * N, to = i * 4 + m * (pitch - N);
      float d[4], g[4], u[4];
      load_four_floats<T>(dh + i * 4, d);
      load_f32<4>(p + at, g);
      load_f32<4>(p + at + N, u);
#pragma unroll
      for (int e = 0; e < 4; ++e) slope(d[e], g[e], u[e]);
      store_four<T>(dp + to, g);  // (both products read it next: not streamed past L2)
      store_four<T>(dp + to + N, u);
    }
  } else {
    const int64_t total = M * N;
    for (int64_t span = static_cast<int64_t>(blockIdx.x) * (4 * kFfThreads); span < total; span += static_cast<int64_t>(gridDim.x) * (4 * kFfThreads)) {
      const int64_t m0 = row_of(span, N, total), c0 = span - m0 * N, i0 = span + threadIdx.x;
      float d[4], g[4], u[4];
      int64_t to[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t i = i0 + e * kFfThreads, m = row_behind(static_cast<int>(threadIdx.x) + e * kFfThreads, m0, c0, N), at = i + m * N;
        to[e] = i + m * (pitch - N);
        d[e] = i < total ? to_f32(dh[i]) : 0.f;
        g[e] = i < total ? p[at] : 0.f;
        u[e] = i < total ? p[at + N] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (i0 + e * kFfThreads >= total) break;
        slope(d[e], g[e], u[e]);
        dp[to[e]] = from_f32<T>(g[e]);
        dp[to[e] + N] = from_f32<T>(u[e]);
      }
    }
  }
}

// f16: dP = dh * u * act'(g) may leave what f16 holds (2^-24 to 65504) where neither of its two products does. So its rows are scaled by powers of two for the
// one, dP W, and its columns for the other, dP^T x, and written twice: an element is resolved to 2^-11 of itself or to 2^-39 of the largest of its row
// (column), whichever is more, and the products take the factors back from their fp32 sums. Two passes over dh and P: the largest magnitudes of
// rows and columns (most[] is zero before; a maximum does not depend on its order), then dP.
// A CTA has 32 rows by 128 of the N columns of each half, a warp four rows, a lane four columns side by side, or, off the grid (VECTOR false), every 32nd.
// What bounds it is memory: 4096 x 11008 takes 103 us for the magnitudes and 148 us to write (4.4 and 5.5 TB/s), where bf16, in one pass, takes 96.
constexpr int kScaledRows = 32, kScaledCols = 128;
template <typename ACT, bool WRITE, bool VECTOR>
__global__ void __launch_bounds__(kFfThreads)
gate_backward_scaled(const __half* dh, const float* p, __half* __restrict__ by_rows, __half* __restrict__ by_cols, uint32_t* row_most, uint32_t* col_most, int64_t M, int64_t N, int64_t pitch) {
  __shared__ uint32_t part[WRITE ? 1 : 8][2 * kScaledCols];
  next_grid_may_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t across = (N + kScaledCols - 1) / kScaledCols, tiles = (M + kScaledRows - 1) / kScaledRows * across;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t m0 = t / across * kScaledRows + warp * 4, tile_n = t % across * kScaledCols, n0 = tile_n + (VECTOR ? 4 * lane : lane);
    constexpr int kStep = VECTOR ? 1 : 32;  // from a lane's column to its next
    float d[4][4], g[4][4], u[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + i;
      if constexpr (VECTOR) {
        if (m < M && n0 < N) {
          load_four_floats<__half>(dh + m * N + n0, d[i]);
          load_f32<4>(p + m * 2 * N + n0, g[i]);
          load_f32<4>(p + m * 2 * N + N + n0, u[i]);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) d[i][c] = g[i][c] = u[i][c] = 0.f;
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int64_t n = n0 + 32 * c;
          const bool in = m < M && n < N;
          d[i][c] = in ? to_f32(dh[m * N + n]) : 0.f;
          g[i][c] = in ? p[m * 2 * N + n] : 0.f;
          u[i][c] = in ? p[m * 2 * N + N + n] : 0.f;
        }
      }
    }
    float col[4][2];
    if constexpr (WRITE) {
      after_grids_before();  // (dh and P were complete before the first pass, which is launched the ordinary way)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool in = n0 + kStep * c < N;
        col[c][0] = by_cols && in ? row_scale(col_most[n0 + kStep * c]) : 0.f;
        col[c][1] = by_cols && in ? row_scale(col_most[N + n0 + kStep * c]) : 0.f;
      }
    }
    uint32_t most[4][2] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float dg[4], du[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float a, s;
        ACT::template both<true>(g[i][c], a, s);
        dg[c] = d[i][c] * u[i][c] * s;
        du[c] = d[i][c] * a;
      }
      if constexpr (WRITE) {
        if (m0 + i >= M) continue;
        const int64_t to = (m0 + i) * pitch + n0;
        auto put = [&](__half* out, float gate, const float (&cols)[4][2], bool of_cols) {
          float v[4], w[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            v[c] = dg[c] * (of_cols ? cols[c][0] : gate);
            w[c] = du[c] * (of_cols ? cols[c][1] : gate);
          }
          if constexpr (VECTOR) {
            if (n0 >= N) return;
            store_four<__half>(out + to, v);  // (both products read it next: not streamed past L2)
            store_four<__half>(out + to + N, w);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (n0 + 32 * c >= N) break;
              out[to + 32 * c] = __float2half_rn(v[c]);
              out[to + N + 32 * c] = __float2half_rn(w[c]);
            }
          }
        };
        if (by_rows) put(by_rows, row_scale(row_most[m0 + i]), col, false);
        if (by_cols) put(by_cols, 0.f, col, true);
      } else {
        uint32_t of_row = 0u;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t bg = __float_as_uint(dg[c]) & 0x7fffffffu, bu = __float_as_uint(du[c]) & 0x7fffffffu;
          most[c][0] = max(most[c][0], bg);
          most[c][1] = max(most[c][1], bu);
          of_row = max(of_row, max(bg, bu));
        }
        of_row = __reduce_max_sync(0xffffffffu, of_row);
        if (lane == 0 && m0 + i < M) atomicMax(row_most + m0 + i, of_row);
      }
    }
    if constexpr (!WRITE) {
      __syncthreads();  // what was there has been read
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int at = static_cast<int>(n0 - tile_n) + kStep * c;
        part[warp][at] = most[c][0];
        part[warp][kScaledCols + at] = most[c][1];
      }
      __syncthreads();
      uint32_t of_col = 0u;
#pragma unroll
      for (int w = 0; w < 8; ++w) of_col = max(of_col, part[w][threadIdx.x]);
      const int up = static_cast<int>(threadIdx.x) >= kScaledCols ? 1 : 0;
      const int64_t n = tile_n + static_cast<int>(threadIdx.x) - up * kScaledCols;
      if (n < N) atomicMax(col_most + up * N + n, of_col);
    }
  }
}

inline int ff_grid(int64_t items) {
  const int64_t b = (items + kFfThreads - 1) / kFfThreads, most = kNumSMs * 64LL;
  return static_cast<int>(b < 1 ? 1 : b < most ? b : most);
}

int launch_gate(const float* p, float* out, int64_t M, int64_t N, int act, cudaStream_t st) {
  const bool vec = N % 4 == 0 && aligned16(p) && aligned16(out);
  const int grid = ff_grid(M * N / 4);
  gate_act_each(act, [&](auto a) {
    if (vec) gate_forward<decltype(a), true><<<grid, kFfThreads, 0, st>>>(p, out, M, N);
    else gate_forward<decltype(a), false><<<grid, kFfThreads, 0, st>>>(p, out, M, N);
  });
  return check_launch();
}

template <typename T> int launch_gate_backward(const void* dh, const float* p, void* out, int64_t M, int64_t N, int64_t pitch, int act, cudaStream_t st) {
  const bool vec = N % 4 == 0 && pitch % 4 == 0 && aligned16(p) && ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(dh)) & (4 * sizeof(T) - 1)) == 0;
  const int grid = ff_grid(M * N / 4);
  gate_act_each(act, [&](auto a) {
    if (vec) gate_backward<T, decltype(a), true><<<grid, kFfThreads, 0, st>>>(static_cast<const T*>(dh), p, static_cast<T*>(out), M, N, pitch);
    else gate_backward<T, decltype(a), false><<<grid, kFfThreads, 0, st>>>(static_cast<const T*>(dh), p, static_cast<T*>(out), M, N, pitch);
  });
  return check_launch();
}

int launch_gate_backward_scaled(const __half* dh, const float* p, __half* by_rows, __half* by_cols, uint32_t* most, int64_t M, int64_t N, int64_t pitch, int act, cudaStream_t st) {
  const bool vec = N % 4 == 0 && pitch % 4 == 0 && aligned16(p) && ((reinterpret_cast<uintptr_t>(dh) | reinterpret_cast<uintptr_t>(by_rows) | reinterpret_cast<uintptr_t>(by_cols)) & 7u) == 0;
  const int64_t tiles = (M + kScaledRows - 1) / kScaledRows * ((N + kScaledCols - 1) / kScaledCols), room = kNumSMs * 16LL;
  const int grid = static_cast<int>(tiles < room ? tiles : room);
  cudaError_t e = cudaMemsetAsync(most, 0, static_cast<size_t>(M + 2 * N) * 4, st);
  if (e != cudaSuccess) { set_last_cuda_error(e); return B200_ELAUNCH; }
  gate_act_each(act, [&](auto a) {
    auto go = [&](auto look, auto write) {
      look<<<grid, kFfThreads, 0, st>>>(dh, p, by_rows, by_cols, most, most + M, M, N, pitch);
      e = launch_after(write, grid, kFfThreads, 0, st, dh, p, by_rows, by_cols, most, most + M, M, N, pitch);
    };
    if (vec) go(gate_backward_scaled<decltype(a), false, true>, gate_backward_scaled<decltype(a), true, true>);
    else go(gate_backward_scaled<decltype(a), false, false>, gate_backward_scaled<decltype(a), true, false>);
  });
  if (e != cudaSuccess) { set_last_cuda_error(e); return B200_ELAUNCH; }
  return check_launch(2);
}

// ------------------------------------------------------------------ dropout
// y_i = residual_i + (word_i >= threshold ? x_i * scale : 0), word_i = word i % 4 of Philox-4x32 with ten rounds
// (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) for the 128-bit counter
// (offset + i / 4, subsequence) under the 64-bit key `seed`. Nothing but the counter goes into an element's
// word, so the backward pass draws the same mask again instead of reading one, whatever the launch shape.
// What is dropped is not multiplied: an infinity or a NaN in a dropped place leaves nothing.
//
// What bounds it is the generator's multiplications as much as memory: 20 of 32 x 32 bits to four elements. The counter's upper three
// words hardly ever change, so the products of the first two rounds that depend on them alone are kept (18 remain), and
// the next elements are on their way while the words of these are worked out. 8192 x 4096 in bf16: 33.4 us, 37.2 with a residual (4.0 and
// 5.4 TB/s; with p = 0, where nothing is drawn, 21.9), fp32 47 and 64 us (5.7 and 6.3 TB/s). The words of that many elements
// alone take 20.6 us: a 32-bit multiplication keeps its pipe for four cycles, wide or not.
struct Philox {
  uint32_t k[20];                  // the rounds' keys
  uint32_t sub0, sub1;             // the counter's words 2 and 3
  uint32_t hi, a1, b1, c2, d2;     // word 1, and what the first two rounds make of words 1 to 3 alone
  __device__ __forceinline__ Philox(uint64_t seed, uint64_t subsequence) : sub0(static_cast<uint32_t>(subsequence)), sub1(static_cast<uint32_t>(subsequence >> 32)) {
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      k[2 * r] = k0;
      k[2 * r + 1] = k1;
      k0 += 0x9E3779B9u;
      k1 += 0xBB67AE85u;
    }
    upper(0u);
  }
  __device__ __forceinline__ void upper(uint32_t word1) {
    hi = word1;
    const uint64_t q = static_cast<uint64_t>(sub0) * 0xCD9E8D57u;
    a1 = static_cast<uint32_t>(q >> 32) ^ hi ^ k[0];
    b1 = static_cast<uint32_t>(q) ^ k[2];
    const uint64_t p = static_cast<uint64_t>(a1) * 0xD2511F53u;
    c2 = static_cast<uint32_t>(p >> 32) ^ k[3];
    d2 = static_cast<uint32_t>(p);
  }
  // (word 1 of the counter is `hi`)
  __device__ __forceinline__ void words(uint32_t word0, uint32_t* w) const {
    const uint64_t p1 = static_cast<uint64_t>(word0) * 0xD2511F53u;
    const uint64_t q2 = static_cast<uint64_t>(static_cast<uint32_t>(p1 >> 32) ^ sub1 ^ k[1]) * 0xCD9E8D57u;
    uint32_t a = static_cast<uint32_t>(q2 >> 32) ^ b1, b = static_cast<uint32_t>(q2), c = c2 ^ static_cast<uint32_t>(p1), d = d2;
#pragma unroll
    for (int r = 2; r < 10; ++r) {
      const uint64_t p = static_cast<uint64_t>(a) * 0xD2511F53u, q = static_cast<uint64_t>(c) * 0xCD9E8D57u;
      a = static_cast<uint32_t>(q >> 32) ^ b ^ k[2 * r];
      c = static_cast<uint32_t>(p >> 32) ^ d ^ k[2 * r + 1];
      b = static_cast<uint32_t>(q);
      d = static_cast<uint32_t>(p);
    }
    w[0] = a;
    w[1] = b;
    w[2] = c;
    w[3] = d;
  }
};

struct DropoutArgs {
  int64_t n;
  uint64_t subsequence;
  const int64_t* state;  // seed, offset
  uint32_t threshold;
  float scale;
};
enum : int { kKeepAll = 0, kByWords = 1, kDropAll = 2 };

// Said so that it stays a byte permutation: a shift may become a multiplication, and these are what there is too much of (8192 x 4096
// in bf16 35.1 -> 33.4 us, with a residual 39.3 -> 37.2).
__device__ __forceinline__ uint32_t byte_order(uint32_t v, uint32_t order) {
  uint32_t r;
  asm volatile("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(v), "r"(order));
  return r;
}
// Two elements of a 16-bit word, or an fp32 pair, as fp32 bits: what is dropped becomes zero here, before any arithmetic
template <typename T> __device__ __forceinline__ void kept_pair(uint32_t lo, uint32_t hi, bool keep0, bool keep1, float& a, float& b) {
  if constexpr (sizeof(T) == 4) {
    a = keep0 ? __uint_as_float(lo) : 0.f;
    b = keep1 ? __uint_as_float(hi) : 0.f;
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    a = __uint_as_float(keep0 ? byte_order(lo, 0x1044u) : 0u);
    b = __uint_as_float(keep1 ? byte_order(lo, 0x3244u) : 0u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    a = keep0 ? f.x : 0.f;
    b = keep1 ? f.y : 0.f;
  }
}

__device__ __forceinline__ void copy_async(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ uint4 ld_shared(uint32_t from) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
  return v;
}

// Sixteen bytes of elements to a thread and step, the next ones on their way to its own slot in shared memory; whatever is behind the last whole sixteen, or all of them where the operands are off
// the grid (VECTOR false), goes four elements to a thread.
template <typename T, int MODE, bool RESIDUAL, bool VECTOR>
__global__ void __launch_bounds__(kFfThreads, 4) dropout_kernel(const T* x, const T* residual, T* __restrict__ y, DropoutArgs A) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T)), kWords = sizeof(T) == 4 ? 2 : 1;
  Philox gen(static_cast<uint64_t>(A.state[0]), A.subsequence);
  const uint64_t offset = static_cast<uint64_t>(A.state[1]);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kFfThreads + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * kFfThreads;
  const int64_t vecs = VECTOR ? A.n / kPer : 0;
  if constexpr (VECTOR) {
    __shared__ uint4 slots[2][RESIDUAL ? 2 : 1][kFfThreads];
    int trips = first < vecs ? static_cast<int>((vecs - first + step - 1) / step) : 0;
    const uint4 *px = reinterpret_cast<const uint4*>(x) + first, *pr = reinterpret_cast<const uint4*>(residual) + first;
    uint4* py = reinterpret_cast<uint4*>(y) + first;
    uint64_t count = offset + static_cast<uint64_t>(first) * (kPer / 4);
    const uint64_t counts = static_cast<uint64_t>(step) * (kPer / 4);
    const F2 scale = F2::of(A.scale, A.scale);
    const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(&slots[0][0][threadIdx.x]));
    constexpr uint32_t kOther = kFfThreads * 16, kSlot = (RESIDUAL ? 2 : 1) * kOther;
    auto load = [&](uint32_t slot) {
      if constexpr (MODE != kDropAll) copy_async(mine + slot, px);
      if constexpr (RESIDUAL) copy_async(mine + slot + kOther, pr);
      px += step;
      pr += step;
    };
    auto take = [&](uint32_t slot, uint32_t next) {
      if (trips > 1) load(next);
      asm volatile("cp.async.commit_group;" ::: "memory");
      uint32_t w[kPer];
      if constexpr (MODE == kByWords) {
        const uint32_t word0 = static_cast<uint32_t>(count);
        if (static_cast<uint32_t>(count >> 32) != gen.hi) gen.upper(static_cast<uint32_t>(count >> 32));
        gen.words(word0, w);
        if constexpr (kPer == 8) {
          if (word0 == 0xffffffffu) gen.upper(gen.hi + 1);
          gen.words(word0 + 1, w + 4);
        }
        count += counts;
      }
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      const uint4 rx = MODE != kDropAll ? ld_shared(mine + slot) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t in[4] = {rx.x, rx.y, rx.z, rx.w};
      float v[kPer], r[kPer];
      if constexpr (RESIDUAL) widen<T>(ld_shared(mine + slot + kOther), r);
#pragma unroll
      for (int e = 0; e < kPer; e += 2) {
        auto keep = [&](int k) { return MODE == kKeepAll || (MODE == kByWords && w[k] >= A.threshold); };
        kept_pair<T>(in[e / 2 * kWords], in[e / 2 * kWords + kWords - 1], keep(e), keep(e + 1), v[e], v[e + 1]);
        const F2 of = F2::of(v[e], v[e + 1]);
        p_parts(RESIDUAL ? p_fma(of, scale, F2::of(r[e], r[e + 1])) : p_mul(of, scale), v[e], v[e + 1]);
      }
      __stcs(py, narrow<T>(v));
      py += step;
    };
    if (trips) load(0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    while (trips > 0) {
      take(0, kSlot);
      if (--trips == 0) break;
      take(kSlot, 0);
      --trips;
    }
  }
  const int64_t groups = (A.n + 3) / 4;
  for (int64_t i = vecs * (kPer / 4) + first; i < groups; i += step) {
    uint32_t w[4];
    const uint64_t count = offset + static_cast<uint64_t>(i);
    if constexpr (MODE == kByWords) {
      if (static_cast<uint32_t>(count >> 32) != gen.hi) gen.upper(static_cast<uint32_t>(count >> 32));
      gen.words(static_cast<uint32_t>(count), w);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t at = 4 * i + e;
      if (at >= A.n) break;
      const float v = MODE == kKeepAll || (MODE == kByWords && w[e] >= A.threshold) ? to_f32(x[at]) : 0.f;
      y[at] = from_f32<T>(RESIDUAL ? fmaf(v, A.scale, to_f32(residual[at])) : v * A.scale);
    }
  }
}

template <typename T> int launch_dropout(const void* x, const void* residual, void* y, int mode, const DropoutArgs& A, cudaStream_t st) {
  const bool vec = aligned16(x) && aligned16(y) && (!residual || aligned16(residual));
  const int64_t per = vec ? 16 / static_cast<int>(sizeof(T)) : 4, blocks = (A.n + per * kFfThreads - 1) / (per * kFfThreads), most = kNumSMs * 8LL;
  const int grid = static_cast<int>(blocks < most ? blocks : most);
  const T *tx = static_cast<const T*>(x), *tr = static_cast<const T*>(residual);
  T* ty = static_cast<T*>(y);
  auto go = [&](auto kernel) { kernel<<<grid, kFfThreads, 0, st>>>(tx, tr, ty, A); };
  auto by_mode = [&](auto r, auto v) {
    constexpr bool kR = decltype(r)::value, kV = decltype(v)::value;
    if (mode == kKeepAll) go(dropout_kernel<T, kKeepAll, kR, kV>);
    else if (mode == kByWords) go(dropout_kernel<T, kByWords, kR, kV>);
    else go(dropout_kernel<T, kDropAll, kR, kV>);
  };
  if (residual) vec ? by_mode(std::true_type{}, std::true_type{}) : by_mode(std::true_type{}, std::false_type{});
  else vec ? by_mode(std::false_type{}, std::true_type{}) : by_mode(std::false_type{}, std::false_type{});
  return check_launch();
}

// ------------------------------------------------------------------ rows to 8 bits
// scale = max|x| / 127, q = x * (127 / max|x|) rounded to even; a row of zeros (or of values below 2^-118, whose
// reciprocal scale would overflow) has scale 0 and zeros, a row with an infinity or a NaN has that as its scale and zeros.
// A row is read once and stays in registers: NV pieces to a thread, a piece being 16 bytes of elements, or, off the grid (VECTOR
// false), the four elements of an aligned word of the result; NV = 0 takes rows of any length, read twice. Where rows are
// many a warp takes one by itself (WARP) and nobody waits for another. The largest magnitude is found on the bit patterns
// (as whole numbers they order like the magnitudes, NaN above all), and a code is the low byte of v + 1.5 * 2^23, whose addition
// rounds to even: a conversion instruction for each took longer than the memory. (Product and sum are two instructions: packed in
// pairs they came out fused, which rounds a product next to a tie the other way.) 8192 x 4096 in bf16: 15.5 us, the memory's own
// time; 46.7 with a CTA to a row and conversions, 30.4 with a warp to a row and conversions; 8192 x 4095 52.9 (78.9 element by element).
constexpr uint32_t kLeastMax = 0x04800000u;  // 2^-118
constexpr uint32_t kInfinity = 0x7f800000u;
constexpr float kToInteger = 12582912.f;

template <typename T> __device__ __forceinline__ uint32_t magnitudes(uint32_t m, uint32_t w) {  // of a word: one, or two side by side
  if constexpr (sizeof(T) == 4) return max(m, w & 0x7fffffffu);
  else return __vmaxu2(m, w & 0x7fff7fffu);
}
template <typename T> __device__ __forceinline__ uint32_t widest(uint32_t m) {  // the largest of a lane's, as fp32 bits
  if constexpr (sizeof(T) == 4) {
    return m;
  } else {
    const uint32_t h = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return h << 16;
    else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h)))) & 0x7fffffffu;
  }
}
__device__ __forceinline__ uint32_t codes(float a, float b, float c, float d, float inv) {
  auto code = [&](float v) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), kToInteger)); };
  return __byte_perm(__byte_perm(code(a), code(b), 0x0040), __byte_perm(code(c), code(d), 0x0040), 0x5410);
}
// Four elements from any address: 16-bit ones from the one or two aligned blocks of eight bytes that they lie in (each holds a byte of
// them or is not read)
template <typename T> __device__ __forceinline__ void load_four(const T* p, uint32_t* w) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(p[e]);
  } else {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 7u;
    const uint2* block = reinterpret_cast<const uint2*>(reinterpret_cast<uintptr_t>(p) - off);
    const uint2 lo = __ldg(block);
    const uint2 hi = off ? __ldg(block + 1) : make_uint2(0u, 0u);
    const uint32_t a = off & 4u ? lo.y : lo.x, b = off & 4u ? hi.x : lo.y, c = off & 4u ? hi.y : hi.x, bits = (off & 3u) * 8u;
    w[0] = __funnelshift_r(a, b, bits);
    w[1] = __funnelshift_r(b, c, bits);
  }
}
template <typename T> __device__ __forceinline__ void four_floats(const uint32_t* w, float* v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(w[e]);
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      v[2 * e] = __uint_as_float(w[e] << 16);
      v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      v[2 * e] = f.x;
      v[2 * e + 1] = f.y;
    }
  }
}

template <typename T, int NV, bool VECTOR, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) quantize_rows_kernel(const T* x, int8_t* __restrict__ q, float* __restrict__ scale, int64_t rows, int64_t cols, int64_t pitch) {
  constexpr int kPer = VECTOR ? 16 / static_cast<int>(sizeof(T)) : 4, kWords = kPer * static_cast<int>(sizeof(T)) / 4;
  __shared__ uint32_t part[32];
  next_grid_may_start();  // (the product's CTAs set themselves up meanwhile)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;
  if (WARP && r >= rows) return;
  const int at = WARP ? lane : static_cast<int>(threadIdx.x), step = WARP ? 32 : static_cast<int>(blockDim.x);
  const T* row = x + r * pitch;
  int8_t* qrow = q + r * cols;
  // off the grid, piece 0 is what lies before the first aligned word of the result
  const int head = VECTOR ? kPer : static_cast<int>(-reinterpret_cast<intptr_t>(qrow) & 3);
  const int64_t pieces = cols > head ? (cols - head + kPer - 1) / kPer + 1 : 1;
  uint32_t m = 0u;
  uint32_t raw[NV ? NV : 1][kWords];
  auto fetch = [&](int64_t j, uint32_t* w) {
    const int64_t c = head + (j - 1) * kPer;
#pragma unroll
    for (int e = 0; e < kWords; ++e) w[e] = 0u;
    if (j >= pieces) return;
    if constexpr (VECTOR) {
      const uint4 v = ld_stream(row + c);
      w[0] = v.x;
      w[1] = v.y;
      w[2] = v.z;
      w[3] = v.w;
    } else if (c >= 0 && c + 4 <= cols) {
      load_four<T>(row + c, w);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e >= 0 && c + e < cols) {
          if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(row[c + e]);
          else w[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[c + e]) << (e % 2 * 16);
        }
    }
  };
  auto look = [&](const uint32_t* w) {
#pragma unroll
    for (int e = 0; e < kWords; ++e) m = magnitudes<T>(m, w[e]);
  };
  if constexpr (NV == 0) {
    for (int64_t j = at; j < pieces; j += step) {
      fetch(j, raw[0]);
      look(raw[0]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) fetch(at + static_cast<int64_t>(k) * step, raw[k]);
#pragma unroll
    for (int k = 0; k < NV; ++k) look(raw[k]);
  }
  m = __reduce_max_sync(0xffffffffu, widest<T>(m));
  if constexpr (!WARP) {
    if (lane == 0) part[warp] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, lane < static_cast<int>((blockDim.x + 31) >> 5) ? part[lane] : 0u);
  }
  const bool some = m >= kLeastMax && m < kInfinity;
  const float most = __uint_as_float(m), inv = some ? __fdiv_rn(127.f, most) : 0.f;
  if (at == 0) scale[r] = m < kLeastMax ? 0.f : __fdiv_rn(most, 127.f);
  auto store = [&](int64_t j, const uint32_t* w) {
    const int64_t c = head + (j - 1) * kPer;
    uint32_t code[kPer / 4];
#pragma unroll
    for (int e = 0; e < kPer / 4; ++e) {
      float v[4];
      four_floats<T>(w + e * static_cast<int>(sizeof(T)), v);
      code[e] = some ? codes(v[0], v[1], v[2], v[3], inv) : 0u;
    }
    if constexpr (kPer == 8) {
      *reinterpret_cast<uint2*>(qrow + c) = make_uint2(code[0], code[1]);
    } else if (VECTOR || (c >= 0 && c + 4 <= cols)) {
      *reinterpret_cast<uint32_t*>(qrow + c) = code[0];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e >= 0 && c + e < cols) qrow[c + e] = static_cast<int8_t>(code[0] >> (8 * e));
    }
  };
  if constexpr (NV == 0) {
    for (int64_t j = at; j < pieces; j += step) {
      fetch(j, raw[0]);
      store(j, raw[0]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t j = at + static_cast<int64_t>(k) * step;
      if (j < pieces) store(j, raw[k]);
    }
  }
}

template <typename T> void launch_quantize(const void* x, void* q, void* scale, int64_t rows, int64_t cols, int64_t pitch, cudaStream_t st) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  const T* tx = static_cast<const T*>(x);
  int8_t* tq = static_cast<int8_t*>(q);
  float* ts = static_cast<float*>(scale);
  const bool vec = cols && aligned16(x) && cols % kPer == 0 && (rows == 1 || pitch % kPer == 0) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
  const int64_t pieces = vec ? cols / kPer : (cols + 3) / 4 + 1;  // at most
  const bool many = rows >= kNumSMs * 4;  // warps enough for every SM
  auto go = [&](auto kernel, int64_t grid, int64_t t) { kernel<<<static_cast<unsigned>(grid), static_cast<int>(t <= 32 ? 32 : (t + 31) / 32 * 32), 0, st>>>(tx, tq, ts, rows, cols, pitch); };
  auto by = [&](auto v) {
    constexpr bool kV = decltype(v)::value;
    auto by_warps = [&](auto kernel) { go(kernel, (rows + 7) / 8, 256); };
    if (many && pieces <= 32) by_warps(quantize_rows_kernel<T, 1, kV, true>);
    else if (many && pieces <= 128) by_warps(quantize_rows_kernel<T, 4, kV, true>);
    else if (many && pieces <= 512) by_warps(quantize_rows_kernel<T, 16, kV, true>);
    else if (pieces <= 512) go(quantize_rows_kernel<T, 1, kV, false>, rows, pieces);
    else if (pieces <= 4096) go(quantize_rows_kernel<T, 4, kV, false>, rows, (pieces + 3) / 4);
    else go(quantize_rows_kernel<T, 0, kV, false>, rows, 1024);
  };
  vec ? by(std::true_type{}) : by(std::false_type{});
}

}  // namespace

}  // namespace b200

using namespace b200;

extern "C" int b200_gate(const float* projections, float* out, int64_t M, int64_t N, int activation, void* stream) {
  if (M < 0 || N < 0 || activation < 0 || activation >= B200_ACT_COUNT) return B200_EINVAL;
  if (M == 0 || N == 0) return B200_OK;
  if (!projections || !out) return B200_EINVAL;
  return launch_gate(projections, out, M, N, activation, static_cast<cudaStream_t>(stream));
}

extern "C" int b200_gate_backward_rows(const void* grad, const float* projections, void* grad_projections, int64_t row_stride, int64_t M, int64_t N, int activation, int dtype, void* stream) {
  if (M < 0 || N < 0 || row_stride < 2 * N || activation < 0 || activation >= B200_ACT_COUNT) return B200_EINVAL;
  if (!is_float_dtype(dtype)) return B200_EDTYPE;
  if (M == 0 || N == 0) return B200_OK;
  if (!grad || !projections || !grad_projections) return B200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200_F32: return launch_gate_backward<float>(grad, projections, grad_projections, M, N, row_stride, activation, st);
    case B200_BF16: return launch_gate_backward<__nv_bfloat16>(grad, projections, grad_projections, M, N, row_stride, activation, st);
    default: return launch_gate_backward<__half>(grad, projections, grad_projections, M, N, row_stride, activation, st);
  }
}

extern "C" int b200_gate_backward_scaled(const void* grad, const float* projections, void* by_rows, void* by_columns, uint32_t* most, int64_t row_stride, int64_t M, int64_t N, int activation, void* stream) {
  if (M < 0 || N < 0 || row_stride < 2 * N || activation < 0 || activation >= B200_ACT_COUNT) return B200_EINVAL;
  if (M == 0 || N == 0) return B200_OK;
  if (!grad || !projections || !most || (!by_rows && !by_columns)) return B200_EINVAL;
  return launch_gate_backward_scaled(static_cast<const __half*>(grad), projections, static_cast<__half*>(by_rows), static_cast<__half*>(by_columns), most, M, N, row_stride, activation,
                                     static_cast<cudaStream_t>(stream));
}

extern "C" int b200_gate_backward(const void* grad, const float* projections, void* grad_projections, int64_t M, int64_t N, int activation, int dtype, void* stream) {
  return b200_gate_backward_rows(grad, projections, grad_projections, N < 0 ? 0 : 2 * N, M, N, activation, dtype, stream);
}

extern "C" int b200_dropout(const void* x, const void* residual, void* out, int64_t n, double p, const int64_t* state, int64_t subsequence, int dtype, void* stream) {
  if (n < 0 || !(p >= 0. && p <= 1.)) return B200_EINVAL;
  if (!is_float_dtype(dtype)) return B200_EDTYPE;
  if (n == 0) return B200_OK;
  if (!x || !out || !state) return B200_EINVAL;
  const double words = p * 4294967296.;
  DropoutArgs A;
  A.n = n;
  A.subsequence = static_cast<uint64_t>(subsequence);
  A.state = state;
  const uint64_t threshold = static_cast<uint64_t>(nearbyint(words));
  const int mode = threshold == 0 ? kKeepAll : threshold > 0xffffffffull ? kDropAll : kByWords;
  A.threshold = static_cast<uint32_t>(threshold);
  A.scale = p < 1. ? static_cast<float>(1. / (1. - p)) : 0.f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200_F32: return launch_dropout<float>(x, residual, out, mode, A, st);
    case B200_BF16: return launch_dropout<__nv_bfloat16>(x, residual, out, mode, A, st);
    default: return launch_dropout<__half>(x, residual, out, mode, A, st);
  }
}

extern "C" int b200_quantize_rows(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t row_stride, int dtype, void* stream) {
  if (rows < 0 || cols < 0 || rows > 0x7fffffffLL) return B200_EINVAL;
  if (!is_float_dtype(dtype)) return B200_EDTYPE;
  if (rows == 0) return B200_OK;
  if (!scale || (cols && (!x || !q))) return B200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200_F32) launch_quantize<float>(x, q, scale, rows, cols, row_stride, st);
  else if (dtype == B200_BF16) launch_quantize<__nv_bfloat16>(x, q, scale, rows, cols, row_stride, st);
  else launch_quantize<__half>(x, q, scale, rows, cols, row_stride, st);
  return check_launch();
}
