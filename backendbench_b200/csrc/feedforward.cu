// What stands around the products of a feed-forward block: the gate of a projection pair and its gradient, dropout
// whose mask is drawn from a counter, and the quantisation of rows to 8 bits. All are one pass over their data.
#include <type_traits>

#include "b200_common.cuh"
#include "gate_act.cuh"

namespace b200 {

namespace {

constexpr int kFfThreads = 256;

// ------------------------------------------------------------------ the gate
// h = act(g) * u of fp32 projections P = [g | u] (M x 2 N). fp32 products come in two steps (their sums are
// put together from six plane products over several launches), so the gate has a kernel of its own there.
// Backward: dP = [dh * u * act'(g) | dh * act(g)], rounded to the type of the operands it is multiplied by next.
// VEC elements to a thread: whole vectors of every operand where rows are on the grid, else one.
template <int N> __device__ __forceinline__ void load_f32(const float* p, float* v) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 4) widen<float>(ld_stream(p + e), v + e);
  } else {
    v[0] = p[0];
  }
}

template <typename ACT, int VEC>
__global__ void __launch_bounds__(kFfThreads) gate_forward(const float* p, float* __restrict__ h, int64_t M, int64_t N) {
  const int64_t per_row = N / VEC, total = M * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kFfThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kFfThreads) {
    const int64_t m = total <= 0xffffffffll ? static_cast<uint32_t>(i) / static_cast<uint32_t>(per_row) : i / per_row;
    const float* row = p + i * VEC + m * N;  // m rows of 2 N, not N, lie before
    float g[VEC], u[VEC];
    load_f32<VEC>(row, g);
    load_f32<VEC>(row + N, u);
#pragma unroll
    for (int e = 0; e < VEC; ++e) g[e] = ACT::template f<false>(g[e]) * u[e];
    if constexpr (VEC > 1) *reinterpret_cast<uint4*>(h + i * VEC) = narrow<float>(g);
    else h[i] = g[0];
  }
}

template <typename T, typename ACT, int VEC>
__global__ void __launch_bounds__(kFfThreads) gate_backward(const T* dh, const float* p, T* __restrict__ dp, int64_t M, int64_t N) {
  const int64_t per_row = N / VEC, total = M * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kFfThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kFfThreads) {
    const int64_t m = total <= 0xffffffffll ? static_cast<uint32_t>(i) / static_cast<uint32_t>(per_row) : i / per_row;
    const int64_t at = i * VEC + m * N;
    float d[VEC], g[VEC], u[VEC];
    if constexpr (VEC > 1) widen<T>(ld_stream(dh + i * VEC), d);
    else d[0] = to_f32(dh[i]);
    load_f32<VEC>(p + at, g);
    load_f32<VEC>(p + at + N, u);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float a, s;
      ACT::template both<sizeof(T) == 2>(g[e], a, s);
      g[e] = d[e] * u[e] * s;
      u[e] = d[e] * a;
    }
    if constexpr (VEC > 1) {  // (both products read it next: not streamed past L2)
      *reinterpret_cast<uint4*>(dp + at) = narrow<T>(g);
      *reinterpret_cast<uint4*>(dp + at + N) = narrow<T>(u);
    } else {
      dp[at] = from_f32<T>(g[0]);
      dp[at + N] = from_f32<T>(u[0]);
    }
  }
}

inline int ff_grid(int64_t items) {
  const int64_t b = (items + kFfThreads - 1) / kFfThreads, most = kNumSMs * 16LL;
  return static_cast<int>(b < most ? b : most);
}

int launch_gate(const float* p, float* out, int64_t M, int64_t N, int act, cudaStream_t st) {
  const bool vec = N % 4 == 0 && aligned16(p) && aligned16(out);
  const int grid = ff_grid(M * N / (vec ? 4 : 1));
  gate_act_each(act, [&](auto a) {
    if (vec) gate_forward<decltype(a), 4><<<grid, kFfThreads, 0, st>>>(p, out, M, N);
    else gate_forward<decltype(a), 1><<<grid, kFfThreads, 0, st>>>(p, out, M, N);
  });
  return check_launch();
}

template <typename T> int launch_gate_backward(const void* dh, const float* p, void* out, int64_t M, int64_t N, int act, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);
  const bool vec = N % kVec == 0 && aligned16(p) && aligned16(out) && aligned16(dh);
  const int grid = ff_grid(M * N / (vec ? kVec : 1));
  gate_act_each(act, [&](auto a) {
    if (vec) gate_backward<T, decltype(a), kVec><<<grid, kFfThreads, 0, st>>>(static_cast<const T*>(dh), p, static_cast<T*>(out), M, N);
    else gate_backward<T, decltype(a), 1><<<grid, kFfThreads, 0, st>>>(static_cast<const T*>(dh), p, static_cast<T*>(out), M, N);
  });
  return check_launch();
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
// NV vectors of 16 bytes to a thread: the row is read once and stays in registers. NV = 0: any length
// and alignment, read twice.
constexpr float kLeastMax = 3.0092655e-36f;  // 2^-118

__device__ __forceinline__ float abs_max_nan(float m, float v) {  // a NaN stays
  const float a = fabsf(v);
  return a > m || a != a ? a : m;
}

template <typename T, int NV>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const T* x, int8_t* __restrict__ q, float* __restrict__ scale, int64_t cols, int64_t pitch) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  __shared__ float part[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  next_grid_may_start();  // (the product's CTAs set themselves up meanwhile)
  const T* row = x + blockIdx.x * pitch;
  int8_t* qrow = q + blockIdx.x * cols;
  float m = 0.f;
  uint4 raw[NV ? NV : 1];
  if constexpr (NV) {
    const int64_t vecs = cols / kPer;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t j = tid + static_cast<int64_t>(k) * blockDim.x;
      raw[k] = j < vecs ? ld_stream(row + j * kPer) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float v[kPer];
      widen<T>(raw[k], v);
#pragma unroll
      for (int e = 0; e < kPer; ++e) m = abs_max_nan(m, v[e]);
    }
  } else {
    for (int64_t j = tid; j < cols; j += blockDim.x) m = abs_max_nan(m, to_f32(row[j]));
  }
  auto all = [&](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = abs_max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  m = all(m);
  if (lane == 0) part[warp] = m;
  __syncthreads();
  m = all(lane < static_cast<int>((blockDim.x + 31) >> 5) ? part[lane] : 0.f);
  const bool some = m >= kLeastMax && m <= 3.402823466e38f;
  const float inv = some ? __fdiv_rn(127.f, m) : 0.f;
  if (tid == 0) scale[blockIdx.x] = m < kLeastMax ? 0.f : __fdiv_rn(m, 127.f);
  auto one = [&](float v) { return some ? __float2int_rn(v * inv) : 0; };
  if constexpr (NV) {
    const int64_t vecs = cols / kPer;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t j = tid + static_cast<int64_t>(k) * blockDim.x;
      if (j >= vecs) break;
      float v[kPer];
      widen<T>(raw[k], v);
      uint32_t w[kPer / 4];
#pragma unroll
      for (int e = 0; e < kPer / 4; ++e)
        w[e] = (one(v[4 * e]) & 0xff) | (one(v[4 * e + 1]) & 0xff) << 8 | (one(v[4 * e + 2]) & 0xff) << 16 | static_cast<uint32_t>(one(v[4 * e + 3])) << 24;
      if constexpr (kPer == 8) *reinterpret_cast<uint2*>(qrow + j * 8) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(qrow + j * 4) = w[0];
    }
  } else {
    for (int64_t j = tid; j < cols; j += blockDim.x) qrow[j] = static_cast<int8_t>(one(to_f32(row[j])));
  }
}

template <typename T> void launch_quantize(const void* x, void* q, void* scale, int64_t rows, int64_t cols, int64_t pitch, cudaStream_t st) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  const T* tx = static_cast<const T*>(x);
  int8_t* tq = static_cast<int8_t*>(q);
  float* ts = static_cast<float*>(scale);
  const bool vec = aligned16(x) && cols % kPer == 0 && (rows == 1 || pitch % kPer == 0) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
  const int64_t vecs = cols / kPer;
  auto threads = [](int64_t n) { return static_cast<int>(n >= 1024 ? 1024 : n <= 32 ? 32 : (n + 31) / 32 * 32); };
  auto go = [&](auto kernel, int t) { kernel<<<static_cast<unsigned>(rows), t, 0, st>>>(tx, tq, ts, cols, pitch); };
  if (vec && vecs <= 512) return go(quantize_rows_kernel<T, 1>, threads(vecs));
  if (vec && vecs <= 1024) return go(quantize_rows_kernel<T, 2>, threads((vecs + 1) / 2));
  if (vec && vecs <= 4096) return go(quantize_rows_kernel<T, 4>, threads((vecs + 3) / 4));
  return go(quantize_rows_kernel<T, 0>, threads((cols + 3) / 4));
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

extern "C" int b200_gate_backward(const void* grad, const float* projections, void* grad_projections, int64_t M, int64_t N, int activation, int dtype, void* stream) {
  if (M < 0 || N < 0 || activation < 0 || activation >= B200_ACT_COUNT) return B200_EINVAL;
  if (!is_float_dtype(dtype)) return B200_EDTYPE;
  if (M == 0 || N == 0) return B200_OK;
  if (!grad || !projections || !grad_projections) return B200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200_F32: return launch_gate_backward<float>(grad, projections, grad_projections, M, N, activation, st);
    case B200_BF16: return launch_gate_backward<__nv_bfloat16>(grad, projections, grad_projections, M, N, activation, st);
    default: return launch_gate_backward<__half>(grad, projections, grad_projections, M, N, activation, st);
  }
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
