// Dropout from a counter-based generator: the mask is a function of (key, index) and is computed
// where it is used, forward and backward alike, so it is never stored.
//
//   word(i)  = word i % 4 of Philox4x32-10 at counter (i / 4, offset) under the key seed
//   y[i]     = word(j) >= floor(p * 2^32) ? x[i] / (1 - p) : 0
//
// with j = i (each value for itself) or j = i / T (a whole neuron for all of its steps, what the
// reference's neuron dropout does, src/lava/lib/dl/slayer/neuron/dropout.py).  The generator is the
// one published in J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as
// 1, 2, 3" (SC 2011), section 3.2: multipliers, Weyl increments and round function from there.
//
// Bound: 8 bytes per value at copy bandwidth.  Ten rounds are 20 wide multiplies per four values.
#include "api_util.cuh"

using namespace sb;

namespace {

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t counter, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32);
  uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

constexpr int kThreads = 256;

// Four consecutive values per thread and trip: exactly one counter.  VEC needs 16-byte bases.
template <bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_values_kernel(const float* __restrict__ x, float* __restrict__ y, const int64_t* __restrict__ key, int64_t n,
                      uint32_t threshold, float scale) {
  const uint64_t seed = (uint64_t)key[0], offset = (uint64_t)key[1];
  const int64_t quads = (n + 3) / 4;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < quads; i += (int64_t)gridDim.x * kThreads) {
    const int64_t base = i * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const bool whole = VEC && base + 4 <= n;
    if (whole) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(x + base));
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (base + e < n) v[e] = __ldg(x + base + e);
    }
    const Words w = philox((uint64_t)i, offset, seed);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = w.w[e] >= threshold ? v[e] * scale : 0.f;   // a select: NaN does not pass a drop
    if (whole) {
      *reinterpret_cast<float4*>(y + base) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (base + e < n) y[base + e] = v[e];
    }
  }
}

// Whole rows of T values: a thread's four values lie in one row or straddle rows.
template <bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_rows_kernel(const float* __restrict__ x, float* __restrict__ y, const int64_t* __restrict__ key, int64_t n,
                    int64_t T, uint32_t threshold, float scale) {
  const uint64_t seed = (uint64_t)key[0], offset = (uint64_t)key[1];
  const int64_t quads = (n + 3) / 4;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < quads; i += (int64_t)gridDim.x * kThreads) {
    const int64_t base = i * 4;
    int64_t row = base / T, pos = base - row * T, have = -1;
    Words w{};
    bool keep[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (pos >= T) { ++row; pos = 0; }
      if (row / 4 != have) { have = row / 4; w = philox((uint64_t)have, offset, seed); }
      const int s = (int)(row & 3);
      const uint32_t word = s == 0 ? w.w[0] : s == 1 ? w.w[1] : s == 2 ? w.w[2] : w.w[3];
      keep[e] = word >= threshold;
      ++pos;
    }
    const bool any = keep[0] || keep[1] || keep[2] || keep[3];
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const bool whole = VEC && base + 4 <= n;
    if (whole) {
      if (any) {   // a dropped row is not read at all
        const float4 a = __ldg(reinterpret_cast<const float4*>(x + base));
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (keep[e] && base + e < n) v[e] = __ldg(x + base + e);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = keep[e] ? v[e] * scale : 0.f;
    if (whole) {
      *reinterpret_cast<float4*>(y + base) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (base + e < n) y[base + e] = v[e];
    }
  }
}

// One step of the generator's state: the key of this call is handed out, the offset moves on.
__global__ void dropout_next_kernel(int64_t* state, int64_t* key) {
  key[0] = state[0];
  key[1] = state[1];
  state[1] = (int64_t)((uint64_t)state[1] + 1u);
}

}  // namespace

extern "C" {

int sb_dropout(const float* x, float* y, const int64_t* key, int64_t rows, int64_t T, double p, int per_step,
               void* stream) {
  SB_REQUIRE(rows >= 0 && T >= 0, "negative geometry");
  SB_REQUIRE(p >= 0.0 && p <= 1.0, "dropout probability %g outside 0..1", p);
  SB_REQUIRE(T == 0 || rows <= INT64_MAX / 8 / T, "geometry too large");
  const int64_t n = rows * T;
  if (n == 0) return SB_OK;
  SB_REQUIRE(x && y && key, "null tensor pointer");
  const cudaStream_t s = (cudaStream_t)stream;
  if (p >= 1.0) {                                     // the threshold 2^32 does not fit a word: nothing is kept
    SB_CUDA(cudaMemsetAsync(y, 0, (size_t)n * sizeof(float), s));
    return SB_OK;
  }
  const uint32_t threshold = (uint32_t)(uint64_t)(p * 4294967296.0);
  const float scale = (float)(1.0 / (1.0 - p));
  const bool vec = ((((uintptr_t)x) | ((uintptr_t)y)) & 15u) == 0;
  const int64_t blocks = (n + 4 * kThreads - 1) / (4 * kThreads);
  const int64_t most = (int64_t)sm_count() * 16;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  if (per_step) {
    if (vec) dropout_values_kernel<true><<<grid, kThreads, 0, s>>>(x, y, key, n, threshold, scale);
    else dropout_values_kernel<false><<<grid, kThreads, 0, s>>>(x, y, key, n, threshold, scale);
  } else {
    if (vec) dropout_rows_kernel<true><<<grid, kThreads, 0, s>>>(x, y, key, n, T, threshold, scale);
    else dropout_rows_kernel<false><<<grid, kThreads, 0, s>>>(x, y, key, n, T, threshold, scale);
  }
  SB_CUDA(cudaGetLastError());
  return SB_OK;
}

int sb_dropout_next(int64_t* state, int64_t* key, void* stream) {
  SB_REQUIRE(state && key, "null tensor pointer");
  dropout_next_kernel<<<1, 1, 0, (cudaStream_t)stream>>>(state, key);
  SB_CUDA(cudaGetLastError());
  return SB_OK;
}

}  // extern "C"
