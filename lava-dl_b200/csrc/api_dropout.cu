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

// A block takes spans of 4096 values: four groups of four consecutive ones per thread, all loaded before
// the first is used (262 M values: 0.33 ms, 6.3 TB/s; with one group in flight per thread 0.39 ms).
constexpr int kThreads = 256, kGroups = 4, kSpan = kThreads * kGroups * 4;

struct Group {
  float v[4];
};
// n: values of the tensor from `at` on (4 or more: a whole group)
template <bool VEC>
__device__ __forceinline__ Group load_group(const float* x, int64_t n) {
  Group g{{0.f, 0.f, 0.f, 0.f}};
  if (VEC && n >= 4) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(x));
    g.v[0] = a.x; g.v[1] = a.y; g.v[2] = a.z; g.v[3] = a.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) g.v[e] = __ldcs(x + e);
  }
  return g;
}
template <bool VEC>
__device__ __forceinline__ void store_group(float* y, int64_t n, const Group& g) {
  if (VEC && n >= 4) {
    __stcs(reinterpret_cast<float4*>(y), make_float4(g.v[0], g.v[1], g.v[2], g.v[3]));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) __stcs(y + e, g.v[e]);
  }
}

// Each value for itself: a group is exactly one counter.  VEC needs 16-byte bases.
template <bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_values_kernel(const float* __restrict__ x, float* __restrict__ y, const int64_t* __restrict__ key, int64_t n,
                      uint32_t threshold, float scale) {
  const uint64_t seed = (uint64_t)key[0], offset = (uint64_t)key[1];
  for (int64_t span = (int64_t)blockIdx.x * kSpan; span < n; span += (int64_t)gridDim.x * kSpan) {
    const int64_t first = span + threadIdx.x * 4;
    Group g[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) g[i] = load_group<VEC>(x + first + i * kThreads * 4, n - (first + i * kThreads * 4));
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int64_t at = first + i * kThreads * 4;
      const Words w = philox((uint64_t)at / 4, offset, seed);
#pragma unroll
      for (int e = 0; e < 4; ++e) g[i].v[e] = w.w[e] >= threshold ? g[i].v[e] * scale : 0.f;   // a select: NaN does not pass
      store_group<VEC>(y + at, n - at, g[i]);
    }
  }
}

// Whole rows of T values.  The rows a span touches are drawn once, into shared memory.
template <bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_rows_kernel(const float* __restrict__ x, float* __restrict__ y, const int64_t* __restrict__ key, int64_t n,
                    int64_t T, uint32_t threshold, float scale) {
  __shared__ uint8_t keep_s[kSpan + 12];
  __shared__ int64_t row_s;
  const uint64_t seed = (uint64_t)key[0], offset = (uint64_t)key[1];
  const float inv = 1.0f / (float)T;
  for (int64_t span = (int64_t)blockIdx.x * kSpan; span < n; span += (int64_t)gridDim.x * kSpan) {
    if (threadIdx.x == 0) row_s = span / T;
    __syncthreads();
    const int64_t row0 = row_s;
    const int64_t pos0 = span - row0 * T;                        // within the first row
    const int64_t left = n - span < kSpan ? n - span : kSpan;
    // rows of the span behind the first (T < 4096 only: a longer row ends at most once in it)
    auto row_of = [&](int i) {
      if (T >= kSpan) return pos0 + i >= T ? 1 : 0;
      // whole numbers below 8192: half a unit from the next multiple is more than the rounding of the product
      return (int)(((float)((int)pos0 + i) + 0.5f) * inv);
    };
    // (one row more than the span has: a group that ends with the span may look at it)
    const int rows = row_of((int)left - 1) + 2, head = (int)(row0 & 3);
    for (int r = threadIdx.x * 4; r < rows + head; r += kThreads * 4) {
      const Words w = philox((uint64_t)((row0 - head + r) >> 2), offset, seed);
#pragma unroll
      for (int e = 0; e < 4; ++e) keep_s[r + e] = w.w[e] >= threshold ? 1 : 0;
    }
    __syncthreads();
    Group g[kGroups];
    uint32_t keep[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int at = (threadIdx.x + i * kThreads) * 4;
      keep[i] = 0;
      if (at < left) {
        if (T >= 4) {                            // the group ends in its first row or in the next
          const int r = row_of(at);
          const int64_t here = T - (pos0 + at - r * T);           // values of the first row, 1 or more
          const uint32_t first = here >= 4 ? 15u : (1u << here) - 1u;
          keep[i] = keep_s[head + r] ? first : 0u;
          if (here < 4 && keep_s[head + r + 1]) keep[i] |= 15u & ~first;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (at + e < left) keep[i] |= (uint32_t)keep_s[head + row_of(at + e)] << e;
        }
        if (keep[i]) g[i] = load_group<VEC>(x + span + at, left - at);   // a dropped row is not read at all
      }
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int at = (threadIdx.x + i * kThreads) * 4;
      if (at < left) {
#pragma unroll
        for (int e = 0; e < 4; ++e) g[i].v[e] = (keep[i] >> e & 1) ? g[i].v[e] * scale : 0.f;
        store_group<VEC>(y + span + at, left - at, g[i]);
      }
    }
    __syncthreads();
  }
}

// One step of the generator's state: the key of this call is handed out, the offset moves on.  Atomic, so that
// calls on several streams get keys of their own (which gets which is open).
__global__ void dropout_next_kernel(int64_t* state, int64_t* key) {
  key[0] = state[0];
  key[1] = (int64_t)atomicAdd(reinterpret_cast<unsigned long long*>(state + 1), 1ull);
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
  const int64_t blocks = (n + kSpan - 1) / kSpan;
  const int64_t most = (int64_t)sm_count() * 32;
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
