// Dense synapse in 8-bit integers.
//
//   p[n, t]      = smallest p >= -126 with 127 * 2^p >= max_k |x[n, k, t]|
//   xq[n, k, t]  = round(x[n, k, t] / 2^p)                        (half to even; |xq| <= 127)
//   y[n, o, t]   = (sum_k wq[o, k] xq[n, k, t]) * ws[o] * 2^p     (whole-number sum, then two products)
//
// A power of two as the step of a time step costs at most one bit against max / 127, and buys that
// spikes and graded spikes on a binary grid are held exactly: with weights on the neurons' 8-bit grid
// the product is then the float synapse's, bit for bit.  A time step with a value that is not finite
// gives NaN for all of its outputs.
#include "api_util.cuh"

using namespace sb;

namespace {

constexpr int kMaxK = 131072;   // 127 * 128 * 131072 < 2^31

// The step 2^p of a largest magnitude (given as its bits) and the factor 2^-p; both normal numbers.
__device__ __forceinline__ void step_of(uint32_t top_bits, float* step, float* inv) {
  if (top_bits >= 0x7f800000u) {
    *step = *inv = __int_as_float(0x7fffffff);
    return;
  }
  // 127 * 2^p with p = e - 6 is the float of exponent e and mantissa 127 / 64
  int p = (int)(top_bits >> 23) - 127 - 6 + ((top_bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  if (p < -126) p = -126;
  *step = __int_as_float((p + 127) << 23);
  *inv = __int_as_float((127 - p) << 23);
}

// ---------------------------------------------------------------------------
// Few tokens: the weights are what there is to read.  A block takes the step of each of its (up to TK)
// tokens, quantises them into shared memory, and every warp walks weight rows with four-byte dot
// products, 16 bytes of weights per lane and trip.
// ---------------------------------------------------------------------------
template <int TK>
__global__ void __launch_bounds__(256)
qdense_few_kernel(const float* __restrict__ x, const int8_t* __restrict__ w, const float* __restrict__ ws,
                  float* __restrict__ y, int64_t tokens, int K, int Kp, int O, int64_t T) {
  extern __shared__ int4 smem_few[];
  int8_t* xq = reinterpret_cast<int8_t*>(smem_few);          // [TK][Kp]
  __shared__ uint32_t top[TK];
  __shared__ float step[TK];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t m0 = (int64_t)blockIdx.x * TK;
  if (tid < TK) top[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int m = 0; m < TK; ++m) {
    if (m0 + m >= tokens) break;
    const int64_t n = (m0 + m) / T, t = (m0 + m) - n * T;
    const float* src = x + n * K * T + t;
    uint32_t b = 0;
    for (int k = tid; k < K; k += 256) b = max(b, __float_as_uint(src[(int64_t)k * T]) & 0x7fffffffu);
    b = __reduce_max_sync(0xffffffffu, b);
    if (lane == 0) atomicMax(&top[m], b);
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < TK; ++m) {
    float st = 0.f, inv = 0.f;
    const bool in = m0 + m < tokens;
    if (in) step_of(top[m], &st, &inv);
    const int64_t n = in ? (m0 + m) / T : 0, t = in ? (m0 + m) - n * T : 0;
    const float* src = x + n * K * T + t;
    for (int k = tid; k < Kp; k += 256)
      xq[m * Kp + k] = (in && k < K) ? (int8_t)__float2int_rn(src[(int64_t)k * T] * inv) : (int8_t)0;
    if (tid == 0) step[m] = st;
  }
  __syncthreads();
  for (int o = blockIdx.y * 8 + warp; o < O; o += gridDim.y * 8) {
    int acc[TK];
#pragma unroll
    for (int m = 0; m < TK; ++m) acc[m] = 0;
    const int4* row = reinterpret_cast<const int4*>(w + (int64_t)o * Kp);
    for (int c = lane; c < Kp / 16; c += 32) {
      const int4 a = __ldg(row + c);
#pragma unroll
      for (int m = 0; m < TK; ++m) {
        const int4 b = *reinterpret_cast<const int4*>(xq + m * Kp + c * 16);
        acc[m] = __dp4a(a.x, b.x, acc[m]);
        acc[m] = __dp4a(a.y, b.y, acc[m]);
        acc[m] = __dp4a(a.z, b.z, acc[m]);
        acc[m] = __dp4a(a.w, b.w, acc[m]);
      }
    }
    const float scale = __ldg(ws + o);
#pragma unroll
    for (int m = 0; m < TK; ++m) {
      const int sum = __reduce_add_sync(0xffffffffu, acc[m]);
      if (lane == 0 && m0 + m < tokens) {
        const int64_t n = (m0 + m) / T, t = (m0 + m) - n * T;
        y[(n * O + o) * T + t] = (float)sum * scale * step[m];
      }
    }
  }
}

template <int TK>
int launch_few(const float* x, const int8_t* w, const float* ws, float* y, int64_t tokens, int K, int Kp, int O,
               int64_t T, cudaStream_t s) {
  const size_t bytes = (size_t)TK * Kp;
  SB_CUDA(cudaFuncSetAttribute(qdense_few_kernel<TK>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 1024));
  const int64_t groups = (tokens + TK - 1) / TK;
  int64_t by = (O + 7) / 8;
  const int64_t most = (int64_t)sm_count() * 8;
  if (by * groups > most) by = most / groups > 1 ? most / groups : 1;
  SB_REQUIRE(groups < (1LL << 31), "geometry too large");
  qdense_few_kernel<TK><<<dim3((unsigned)groups, (unsigned)by), 256, bytes, s>>>(x, w, ws, y, tokens, K, Kp, O, T);
  SB_CUDA(cudaGetLastError());
  return SB_OK;
}

}  // namespace

extern "C" {

int64_t sb_qdense_scratch_bytes(int64_t tokens, int64_t Kp) {
  (void)tokens; (void)Kp;
  return 0;
}

int sb_qdense_fwd(const float* x, const signed char* w, const float* w_scale, float* y, int64_t N, int64_t K,
                  int64_t Kp, int64_t O, int64_t T, void* scratch, void* stream) {
  SB_REQUIRE(N >= 0 && K >= 0 && O >= 0 && T >= 0, "negative geometry");
  SB_REQUIRE(K >= 1 && K <= kMaxK, "%lld inputs outside 1..%d (the sums are 32-bit integers)", (long long)K, kMaxK);
  SB_REQUIRE(Kp >= K && Kp % 16 == 0 && Kp - K < 16, "weight rows of %lld bytes for %lld inputs", (long long)Kp, (long long)K);
  SB_REQUIRE(O < (1LL << 31) && T < (1LL << 31) && (T == 0 || N <= (1LL << 40) / T), "geometry too large");
  if (N * O * T == 0) return SB_OK;
  SB_REQUIRE(x && w && w_scale && y, "null tensor pointer");
  SB_REQUIRE(((uintptr_t)w & 15u) == 0, "weights must be 16-byte aligned");
  (void)scratch;
  const cudaStream_t s = (cudaStream_t)stream;
  const int64_t tokens = N * T;
  const int8_t* w8 = (const int8_t*)w;
  const int k = (int)K, kp = (int)Kp, o = (int)O;
  if (tokens > 4 && 8 * Kp <= 200 * 1024) return launch_few<8>(x, w8, w_scale, y, tokens, k, kp, o, T, s);
  if (tokens > 2 && 4 * Kp <= 200 * 1024) return launch_few<4>(x, w8, w_scale, y, tokens, k, kp, o, T, s);
  if (tokens > 1 && 2 * Kp <= 200 * 1024) return launch_few<2>(x, w8, w_scale, y, tokens, k, kp, o, T, s);
  return launch_few<1>(x, w8, w_scale, y, tokens, k, kp, o, T, s);
}

}  // extern "C"
