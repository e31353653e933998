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
#include "tc.cuh"

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
// Few tokens: the weights are what there is to read.  A block takes the step of each of the (up to TK)
// tokens, quantises them into shared memory, and every warp walks weight rows with four-byte dot
// products, 16 bytes of weights per lane and trip.
// ---------------------------------------------------------------------------
template <int TK>
__global__ void __launch_bounds__(256)
qdense_few_kernel(const float* __restrict__ x, const int8_t* __restrict__ w, const float* __restrict__ ws,
                  float* __restrict__ y, int tokens, int K, int Kp, int O, int64_t T) {
  extern __shared__ int4 smem_few[];
  int8_t* xq = reinterpret_cast<int8_t*>(smem_few);          // [TK][Kp]
  __shared__ uint32_t top[TK];
  __shared__ float step[TK];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < TK) top[tid] = 0;
  __syncthreads();
  const float* src[TK];
#pragma unroll
  for (int m = 0; m < TK; ++m) {       // a token past the last reads the last again and is not written
    const int64_t i = m < tokens ? m : tokens - 1, n = i / T;
    src[m] = x + n * K * T + (i - n * T);
  }
  uint32_t b[TK];
#pragma unroll
  for (int m = 0; m < TK; ++m) b[m] = 0;
#pragma unroll 4
  for (int k = tid; k < K; k += 256) {
#pragma unroll
    for (int m = 0; m < TK; ++m) b[m] = max(b[m], __float_as_uint(__ldg(src[m] + (int64_t)k * T)) & 0x7fffffffu);
  }
#pragma unroll
  for (int m = 0; m < TK; ++m) {
    b[m] = __reduce_max_sync(0xffffffffu, b[m]);
    if (lane == 0) atomicMax(&top[m], b[m]);
  }
  __syncthreads();
  float inv[TK];
#pragma unroll
  for (int m = 0; m < TK; ++m) {
    float st;
    step_of(top[m], &st, &inv[m]);
    if (tid == 0) step[m] = st;
  }
#pragma unroll 4
  for (int k = tid; k < Kp; k += 256) {
#pragma unroll
    for (int m = 0; m < TK; ++m)
      xq[m * Kp + k] = k < K ? (int8_t)__float2int_rn(__ldg(src[m] + (int64_t)k * T) * inv[m]) : (int8_t)0;
  }
  __syncthreads();
  for (int o = blockIdx.x * 8 + warp; o < O; o += gridDim.x * 8) {
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
      if (lane == 0 && m < tokens) {
        const int64_t n = m / T, t = m - n * T;
        y[(n * O + o) * T + t] = (float)sum * scale * step[m];
      }
    }
  }
}

template <int TK>
int launch_few(const float* x, const int8_t* w, const float* ws, float* y, int64_t tokens, int K, int Kp, int O,
               int64_t T, cudaStream_t s) {
  int64_t blocks = (O + 7) / 8;
  const int64_t most = (int64_t)sm_count() * 8;
  if (blocks > most) blocks = most;
  qdense_few_kernel<TK><<<(unsigned)blocks, 256, (size_t)TK * Kp, s>>>(x, w, ws, y, (int)tokens, K, Kp, O, T);
  SB_CUDA(cudaGetLastError());
  return SB_OK;
}

// ---------------------------------------------------------------------------
// Many tokens, first pass: x [n][k][t] -> xq [token][k] (rows of Kp bytes, zeros past K) and the steps.
// A block owns TT consecutive time steps of a sample.  A thread is a time step and holds 32 neighbouring
// inputs of it, so that loads are coalesced along time and a rounded row is written in whole sectors; as
// long as the block's threads hold all inputs (K <= 1024 with 32 steps, 2048 with 8), x is read once.
// Beyond that it is walked twice, the second time out of L2.  [64, 2048, 300]: 85 us walked twice in blocks
// of 32 steps, 60 us held by 1024 threads and 16 steps, 50 us by 512 threads and 8 steps, of which two
// blocks share an SM (197 MB, 30 us at copy bandwidth).
// ---------------------------------------------------------------------------
template <int TT>
__global__ void __launch_bounds__(1024, 1)
qdense_quantize_kernel(const float* __restrict__ x, int8_t* __restrict__ xq, float* __restrict__ steps, int K, int Kp,
                       int64_t T, int64_t tiles_t) {
  __shared__ uint32_t top_s[32][TT];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int64_t n = blockIdx.x / tiles_t, t = (blockIdx.x - n * tiles_t) * TT + lane % TT;
  const bool in = t < T;
  const float* src = x + n * K * T + (in ? t : 0);
  const int group = warp * (32 / TT) + lane / TT, stride = warps * (32 / TT) * 32;   // inputs 32 group ...
  const bool once = stride >= Kp;
  float v[32];
  auto load = [&](int k0) {
    const float* p = src + (int64_t)k0 * T;
    if (k0 + 32 <= K) {
#pragma unroll
      for (int e = 0; e < 32; ++e) { v[e] = __ldg(p); p += T; }
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) { v[e] = k0 + e < K ? __ldg(p) : 0.f; p += T; }
    }
  };
  uint32_t top = 0;
#pragma unroll 1
  for (int k0 = group * 32; k0 < Kp; k0 += stride) {
    load(k0);
#pragma unroll
    for (int e = 0; e < 32; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  }
  if (TT <= 16) top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
  if (TT <= 8) top = max(top, __shfl_xor_sync(0xffffffffu, top, 8));
  top_s[warp][lane % TT] = top;
  __syncthreads();
  for (int w = 0; w < warps; ++w) top = max(top, top_s[w][lane % TT]);
  float step, inv;
  step_of(top, &step, &inv);
  const int64_t token = n * T + t;
  if (group == 0 && in) steps[token] = step;
#pragma unroll 1
  for (int k0 = group * 32; k0 < Kp; k0 += stride) {
    if (!once) load(k0);
    uint32_t p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int a = __float2int_rn(v[4 * e] * inv), b = __float2int_rn(v[4 * e + 1] * inv),
                c = __float2int_rn(v[4 * e + 2] * inv), d = __float2int_rn(v[4 * e + 3] * inv);
      p[e] = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    }
    if (in) {
      uint4* dst = reinterpret_cast<uint4*>(xq + token * Kp + k0);
      dst[0] = make_uint4(p[0], p[1], p[2], p[3]);
      if (k0 + 16 < Kp) dst[1] = make_uint4(p[4], p[5], p[6], p[7]);
    }
  }
}

template <int TT>
int launch_quantize(const float* x, int8_t* xq, float* steps, int64_t N, int K, int Kp, int64_t T, cudaStream_t s) {
  const int64_t tiles_t = (T + TT - 1) / TT;
  SB_REQUIRE(N * tiles_t < (1LL << 31), "geometry too large");
  int threads = (Kp + 31) / 32 * TT;
  const int most = TT == 8 ? 512 : 1024;
  threads = threads > most ? most : (threads + 31) / 32 * 32;
  qdense_quantize_kernel<TT><<<(unsigned)(N * tiles_t), threads, 0, s>>>(x, xq, steps, K, Kp, T, tiles_t);
  SB_CUDA(cudaGetLastError());
  return SB_OK;
}

// The same for samples of few time steps: a block per token, its threads along the inputs.
__global__ void __launch_bounds__(256)
qdense_quantize_short_kernel(const float* __restrict__ x, int8_t* __restrict__ xq, float* __restrict__ steps, int K, int Kp,
                             int T) {
  __shared__ uint32_t top_s;
  const int tid = threadIdx.x;
  const int64_t token = blockIdx.x, n = token / T;
  const float* src = x + n * K * T + (token - n * T);
  if (tid == 0) top_s = 0;
  __syncthreads();
  uint32_t top = 0;
#pragma unroll 8
  for (int k = tid; k < K; k += 256) top = max(top, __float_as_uint(__ldg(src + (int64_t)k * T)) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) atomicMax(&top_s, top);
  __syncthreads();
  float step, inv;
  step_of(top_s, &step, &inv);
  if (tid == 0) steps[token] = step;
  for (int k0 = tid * 4; k0 < Kp; k0 += 1024) {
    int q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = k0 + e < K ? __float2int_rn(__ldg(src + (int64_t)(k0 + e) * T) * inv) : 0;
    *reinterpret_cast<uint32_t*>(xq + token * Kp + k0) =
        __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  }
}

// ---------------------------------------------------------------------------
// Second pass: D[token][o] = xq w^T on the tensor cores (kind::i8, 32-bit sums in tensor memory).
// Tokens are the rows of a tile, so that a warp's 32 lanes write 32 neighbouring time steps of one output
// neuron.  One persistent CTA per SM: a thread fetches 128-byte-wide boxes of both operands into a ring of
// stages, a thread issues the MMAs (32 inputs each), eight warps take a finished tile out of one half of
// tensor memory while the next one is summed in the other.  19200 tokens x 2048 -> 2048: 78 us, 2.1 PFLOP/s
// in 8-bit terms; what bounds it is the 12 TB/s at which the SMs fetch their tiles out of L2 (48 KB for every
// 128 x 256 x 128 products).
// ---------------------------------------------------------------------------
constexpr int kGThreads = 320, kTM = 128, kTK = 128;
__host__ __device__ constexpr int stages_of(int nt) { return nt == 256 ? 4 : (nt == 128 ? 6 : 8); }   // narrow tiles: more boxes in flight

__device__ __forceinline__ void mma_i8(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %4};\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(acc)
      : "memory");
}
// signed 8-bit operands, both K-major, 32-bit integer accumulator
__host__ __device__ constexpr uint32_t idesc_i8(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTM >> 4) << 24);
}

template <int NT>
__global__ void __launch_bounds__(kGThreads, 1)
qdense_gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                   const float* __restrict__ steps, const float* __restrict__ ws, float* __restrict__ y, int64_t tokens,
                   int kblocks, int O, int64_t T, int tiles_n, int64_t tiles, unsigned int* status) {
  constexpr int kStageBytes = (kTM + NT) * kTK, kStages = stages_of(NT);
  constexpr uint32_t kCols = 2 * NT < 32 ? 32 : 2 * NT;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 4];
  __shared__ int dead_s;
  __shared__ uint32_t tmem_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  volatile int* dead = &dead_s;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kStages, done = empty + 8 * kStages, taken = done + 16;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(done + 8 * i, 1);
      mbar_init(taken + 8 * i, 256);
    }
    fence_mbar_init();
    dead_s = 0;
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_s)), "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;

  if (warp == 8) {
    if (lane == 0) {
      uint32_t it = 0;
      for (int64_t tile = blockIdx.x; tile < tiles && !*dead; tile += gridDim.x) {
        const int m0 = (int)(tile / tiles_n) * kTM, n0 = (int)(tile % tiles_n) * NT;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const uint32_t s = it % kStages;
          if (it >= kStages && !wait_or_dead(empty + 8 * s, (it / kStages - 1u) & 1u, dead)) break;
          mbar_expect_tx(full + 8 * s, kStageBytes);
          tma_load_2d(base + s * kStageBytes, &amap, kb * (kTK / 4), m0, full + 8 * s);
          tma_load_2d(base + s * kStageBytes + kTM * kTK, &bmap, kb * (kTK / 4), n0, full + 8 * s);
        }
      }
      if (*dead)   // boxes in flight land before the memory is given back
        for (uint32_t j = it > kStages ? it - kStages : 0; j < it; ++j) mbar_wait(full + 8 * (j % kStages), (j / kStages) & 1u);
    }
  } else if (warp == 9) {
    if (lane == 0) {
      uint32_t it = 0, nt = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++nt) {
        const uint32_t acc = nt & 1u, d = tmem + acc * NT;
        if (nt >= 2) ok = wait_or_dead(taken + 8 * acc, (nt / 2 - 1u) & 1u, dead);
        tc_fence_after();
        for (int kb = 0; kb < kblocks && ok; ++kb, ++it) {
          const uint32_t s = it % kStages;
          ok = wait_or_dead(full + 8 * s, (it / kStages) & 1u, dead);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = desc_lo(base + s * kStageBytes), b = desc_lo(base + s * kStageBytes + kTM * kTK);
#pragma unroll
          for (uint32_t k = 0; k < kTK / 32; ++k) mma_i8(d, a + 2 * k, b + 2 * k, idesc_i8(NT), (uint32_t)(kb > 0 || k > 0));
          umma_commit(empty + 8 * s);
        }
        umma_commit(done + 8 * acc);
      }
      if (nt > 0) mbar_wait(done + 8 * ((nt - 1) & 1u), ((nt - 1) / 2) & 1u);
    }
  } else {
    // eight warps: lanes 32 (warp % 4) ... of the tile, columns by halves
    const int quarter = warp & 3, half = warp >> 2;
    constexpr int kMine = NT / 2, kStep = kMine < 32 ? kMine : 32;   // columns of this warp, of one load
    uint32_t nt = 0;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++nt) {
      const uint32_t acc = nt & 1u;
      const int64_t m = (tile / tiles_n) * kTM + quarter * 32 + lane;
      const int n0 = (int)(tile % tiles_n) * NT + half * kMine;
      const bool live = m < tokens;
      const int64_t n = live ? m / T : 0;
      float* out = y + (n * O + n0) * T + (live ? m - n * T : 0);
      const float step = live ? __ldg(steps + m) : 0.f;
      const bool ok = wait_or_dead(done + 8 * acc, (nt / 2) & 1u, dead);
      tc_fence_after();
      const uint32_t src = tmem + ((uint32_t)(quarter * 32) << 16) + acc * NT + half * kMine;
#pragma unroll 1
      for (int c = 0; c < kMine; c += kStep) {
        uint32_t r[kStep];
        if constexpr (kStep == 32) tmem_ld32(src + c, r);
        else tmem_ld16(src + c, r);
        tmem_ld_wait();
        if (c + kStep >= kMine) {
          tc_fence_before();
          mbar_arrive(taken + 8 * acc);
        }
        if (!ok || !live) continue;
        const int left = O - (n0 + c);
        const float* scale = ws + n0 + c;
        if (left >= kStep) {
#pragma unroll
          for (int e = 0; e < kStep; ++e) {
            *out = (float)(int)r[e] * __ldg(scale + e) * step;
            out += T;
          }
        } else {
#pragma unroll
          for (int e = 0; e < kStep; ++e) {
            if (e < left) *out = (float)(int)r[e] * __ldg(scale + e) * step;
            out += T;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*dead && tid == 0) dev_flag(status, SB_DEV_TMA_TIMEOUT);
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

template <int NT>
int launch_gemm(const int8_t* xq, const float* steps, const int8_t* w, const float* ws, float* y, int64_t tokens, int Kp,
                int O, int64_t T, cudaStream_t s) {
  CUtensorMap amap, bmap;
  SB_TRY(make_row_map_box(&amap, xq, tokens, Kp / 4, 32, kTM));
  SB_TRY(make_row_map_box(&bmap, w, O, Kp / 4, 32, NT));
  unsigned int* status = status_ptr();
  if (!status) return SB_ERR_CUDA;
  const int tiles_n = (O + NT - 1) / NT;
  const int64_t tiles = (tokens + kTM - 1) / kTM * tiles_n;
  constexpr int smem = 1024 + stages_of(NT) * (kTM + NT) * kTK;
  SB_CUDA(cudaFuncSetAttribute(qdense_gemm_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int64_t grid = tiles < sm_count() ? tiles : sm_count();
  qdense_gemm_kernel<NT><<<(unsigned)grid, kGThreads, smem, s>>>(amap, bmap, steps, ws, y, tokens, (Kp + kTK - 1) / kTK, O,
                                                                T, tiles_n, tiles, status);
  SB_CUDA(cudaGetLastError());
  return SB_OK;
}

// Every block of the few-token kernel rounds all of its tokens again, so it is for 8 KB of them: 2048 inputs
// and 1 / 2 / 4 / 8 tokens take 3.7 / 4.8 / 8.1 / 12.4 us on it, 9 take 11.1 on the two passes; with 4096
// inputs 8 take 52 against 19.
constexpr int64_t kFewBytes = 8192;
bool few_tokens(int64_t tokens, int64_t Kp) { return tokens <= 8 && tokens * Kp <= kFewBytes; }

// Below this many time steps a lane per step leaves lanes idle.
constexpr int64_t kShort = 16;

int64_t steps_at(int64_t tokens, int64_t Kp) { return (tokens * Kp + 127) / 128 * 128; }

}  // namespace

extern "C" {

int64_t sb_qdense_scratch_bytes(int64_t tokens, int64_t Kp) {
  if (tokens <= 0 || Kp < 16 || tokens > (1LL << 40) || Kp > kMaxK || few_tokens(tokens, Kp)) return 0;
  return steps_at(tokens, Kp) + tokens * (int64_t)sizeof(float);
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
  const cudaStream_t s = (cudaStream_t)stream;
  const int64_t tokens = N * T;
  const int8_t* w8 = (const int8_t*)w;
  const int k = (int)K, kp = (int)Kp, o = (int)O;
  if (!few_tokens(tokens, Kp)) {
    SB_REQUIRE(scratch && ((uintptr_t)scratch & 15u) == 0, "scratch must be given and 16-byte aligned");
    SB_REQUIRE(tokens < (1LL << 31) - kTM, "geometry too large");
    int8_t* xq = (int8_t*)scratch;
    float* steps = (float*)(xq + steps_at(tokens, Kp));
    if (T < kShort) {
      qdense_quantize_short_kernel<<<(unsigned)tokens, 256, 0, s>>>(x, xq, steps, k, kp, (int)T);
      SB_CUDA(cudaGetLastError());
    } else if (kp <= 1024) {
      SB_TRY(launch_quantize<32>(x, xq, steps, N, k, kp, T, s));
    } else {
      SB_TRY(launch_quantize<8>(x, xq, steps, N, k, kp, T, s));
    }
    // the tile width whose waves cost least: a tile takes its columns and about 64 more to fill and empty
    const int64_t rows = (tokens + kTM - 1) / kTM, sms = sm_count();
    int best = 32;
    int64_t best_cost = INT64_MAX;
    for (int nt = 256; nt >= 32; nt /= 2) {
      const int64_t cost = (rows * ((O + nt - 1) / nt) + sms - 1) / sms * (nt + 64);
      if (cost < best_cost) { best = nt; best_cost = cost; }
    }
    if (best == 256) return launch_gemm<256>(xq, steps, w8, w_scale, y, tokens, kp, o, T, s);
    if (best == 128) return launch_gemm<128>(xq, steps, w8, w_scale, y, tokens, kp, o, T, s);
    if (best == 64) return launch_gemm<64>(xq, steps, w8, w_scale, y, tokens, kp, o, T, s);
    return launch_gemm<32>(xq, steps, w8, w_scale, y, tokens, kp, o, T, s);
  }
  if (tokens > 4) return launch_few<8>(x, w8, w_scale, y, tokens, k, kp, o, T, s);
  if (tokens > 2) return launch_few<4>(x, w8, w_scale, y, tokens, k, kp, o, T, s);
  if (tokens > 1) return launch_few<2>(x, w8, w_scale, y, tokens, k, kp, o, T, s);
  return launch_few<1>(x, w8, w_scale, y, tokens, k, kp, o, T, s);
}

}  // extern "C"
