// Linear attention with a decay for each head: the leaky integrator whose input is an outer product.
//
//   S[t] = r S[t-1] + k[t] v[t]^T        (Dk x Dv, r = 1 - decay / 4096)
//   o[t] = S[t]^T q[t]
//
// q, k: [heads, Dk, T], v, o: [heads, Dv, T], time contiguous like every tensor of this library.
// With G[t] = r G[t+1] + q[t] go[t]^T the gradients are
//
//   gq[t] = S[t] go[t]      gk[t] = G[t] v[t]      gv[t] = G[t]^T k[t]      gS[-1] = r G[0],
//
// i.e. the same operator three more times: gq is the walk with (q, k, v) <- (go, v, k) on the
// transposed state, gk and gv are walks back in time with (v, go, q) and (k, q, go).  A walk back in
// time hands its state on already decayed (the first step must see G[T-1] = gS[T-1] + q go^T).
// So every kernel here takes a direction and an `after` flag and serves all four walks.
#include "linear_attention.cuh"

using namespace sb;
using namespace sb::la;

namespace {

// r is applied as the sum of two floats: over the thousand steps a slow head remembers, half an ulp of
// r would grow a thousandfold.  decay / 4096 is exact, and so is what 1 - decay / 4096 loses to rounding.
struct Keep {
  float r, lo;
};
__device__ __forceinline__ Keep keep_of(float decay) {
  const float delta = decay * (1.0f / 4096.0f), r = __fsub_rn(1.0f, delta);
  return Keep{r, __fsub_rn(__fsub_rn(1.0f, r), delta)};
}

// ---------------------------------------------------------------------------
// Walk step by step: any size, any length.
// A block of 128 threads owns one head and 64 columns of its state; a thread holds NI x 4 elements of
// it (rows dg + 8 i, four neighbouring columns).  The row sums of a tile of steps are joined through
// shared memory at the end of the tile.
// ---------------------------------------------------------------------------
constexpr int kTile = 8;

struct Walks {
  Walk w[3];
};

// MANY: one walk per blockIdx.z, copied out of the parameters (indexed, they would be read in the loops);
// a single walk reads them as constants, which saves the registers (66 against 94 us at [64, 16, 64, 48]).
template <int NI, bool MANY>
__global__ void __launch_bounds__(128) walk_kernel(const __grid_constant__ Walks walks) {
  Walk copy;
  if (MANY) copy = walks.w[blockIdx.z];
  const Walk& w = MANY ? copy : walks.w[0];
  __shared__ float qs[kTile][8 * NI], ks[kTile][8 * NI], vs[kTile][64];
  __shared__ float part[kTile][8][64];
  const int tid = threadIdx.x, ec = (tid & 15) * 4, dg = tid >> 4;
  const int64_t head = blockIdx.x;
  const int e0 = blockIdx.y * 64;
  if (e0 >= w.Dv) return;
  const int ne = min(64, w.Dv - e0);
  const Keep keep = keep_of(w.decay[w.n_decay > 1 ? head % w.n_decay : 0]);
  const float r = keep.r, r_lo = keep.lo;
  const float* q = w.q + head * w.Dk * w.T;
  const float* k = w.k + head * w.Dk * w.T;
  const float* v = w.v + (head * w.Dv + e0) * w.T;
  float* o = w.o + (head * w.Dv + e0) * w.T;

  float S[NI][4];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = dg + 8 * i;
      S[i][e] = (w.s_in && d < w.Dk && ec + e < ne)
                    ? w.s_in[head * w.Dk * w.Dv + (int64_t)d * w.s_row + (int64_t)(e0 + ec + e) * w.s_col]
                    : 0.f;
    }

  for (int64_t t0 = 0; t0 < w.T; t0 += kTile) {
    const int nt = (int)min((int64_t)kTile, w.T - t0);
    __syncthreads();
    for (int i = tid; i < kTile * 8 * NI; i += 128) {
      const int d = i / kTile, s = i % kTile;
      const int64_t t = w.reverse ? w.T - 1 - (t0 + s) : t0 + s;
      const bool in = d < w.Dk && s < nt;
      qs[s][d] = in ? q[d * w.T + t] : 0.f;
      ks[s][d] = in ? k[d * w.T + t] : 0.f;
    }
    for (int i = tid; i < kTile * 64; i += 128) {
      const int e = i / kTile, s = i % kTile;
      const int64_t t = w.reverse ? w.T - 1 - (t0 + s) : t0 + s;
      vs[s][e] = (e < ne && s < nt) ? v[e * w.T + t] : 0.f;
    }
    __syncthreads();
    for (int s = 0; s < nt; ++s) {
      const float4 vv = *reinterpret_cast<const float4*>(&vs[s][ec]);
      const float ve[4] = {vv.x, vv.y, vv.z, vv.w};
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const float kd = ks[s][dg + 8 * i], qd = qs[s][dg + 8 * i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = S[i][e];
          if (w.after) {
            x = fmaf(r, x, fmaf(r_lo, x, kd * ve[e]));
            acc[e] = fmaf(qd, x, acc[e]);
          } else {
            x = fmaf(kd, ve[e], x);
            acc[e] = fmaf(qd, x, acc[e]);
            x = fmaf(r, x, r_lo * x);
          }
          S[i][e] = x;
        }
      }
      *reinterpret_cast<float4*>(&part[s][dg][ec]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    }
    __syncthreads();
    for (int i = tid; i < kTile * 64; i += 128) {
      const int e = i / kTile, s = i % kTile;
      if (e >= ne || s >= nt) continue;
      float sum = 0.f;
#pragma unroll
      for (int g = 0; g < 8; ++g) sum += part[s][g][e];
      const int64_t t = w.reverse ? w.T - 1 - (t0 + s) : t0 + s;
      o[e * w.T + t] = sum;
    }
  }
  if (w.s_out) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = dg + 8 * i;
        if (d < w.Dk && ec + e < ne)
          w.s_out[head * w.Dk * w.Dv + (int64_t)d * w.s_row + (int64_t)(e0 + ec + e) * w.s_col] = S[i][e];
      }
  }
}

int launch_walks(const Walk* walks, int n, cudaStream_t s) {
  Walks a{};
  int dk = 0, dv = 0;
  for (int i = 0; i < n; ++i) {
    a.w[i] = walks[i];
    dk = walks[i].Dk > dk ? walks[i].Dk : dk;
    dv = walks[i].Dv > dv ? walks[i].Dv : dv;
  }
  const unsigned heads = (unsigned)walks[0].heads, tiles = (unsigned)((dv + 63) / 64);
  if (n > 1 && walks[0].heads * tiles <= sm_count()) {      // few heads: side by side in one launch
    const dim3 grid(heads, tiles, (unsigned)n);
    if (dk <= 64) walk_kernel<8, true><<<grid, 128, 0, s>>>(a);
    else walk_kernel<16, true><<<grid, 128, 0, s>>>(a);
    SB_CUDA(cudaGetLastError());
    return SB_OK;
  }
  for (int i = 0; i < n; ++i) {
    a.w[0] = walks[i];
    const dim3 grid(heads, (unsigned)((walks[i].Dv + 63) / 64));
    if (walks[i].Dk <= 64) walk_kernel<8, false><<<grid, 128, 0, s>>>(a);
    else walk_kernel<16, false><<<grid, 128, 0, s>>>(a);
    SB_CUDA(cudaGetLastError());
  }
  return SB_OK;
}

// Whether sequences shorter than a chunk walk step by step, in us.  The chunked kernel takes 1.5 and 9.6 (Dk > 64:
// 13.2) for every wave of items whatever their length; a launch of walks takes 3 and for each step 0.48 or, with
// many blocks, 1.3 ns for each of them (twice that for Dk > 64).  Steps against chunks: [1, 8, 64, T] 9.5 and 11.4
// at T = 16, 17.4 and 11.2 at 32; [64, 16, 64, T] 67 and 72 at T = 48, 90 and 70 at 64; their gradients 72 and 212
// at T = 16, 199 and 213 at 48; [16, 16, 128, T] 49 and 52 at T = 32, their gradients 150 and 144 (the rule takes
// steps).  At T = 48 and 1024 heads that is 9 times what the bytes need (7.7): a block has 128 threads, three
// barriers for eight steps and loads of 32 bytes a row, and a chunk is 128 steps whatever the length.
bool walks_by_steps(const Walk* w, int n) {
  const int64_t T = w[0].T;
  if (T >= 128) return false;
  int64_t items = 0;
  bool wide = false, few = n > 1;                // few heads: the walks side by side in one launch
  double steps = 0.0;
  for (int i = 0; i < n; ++i) {
    const int64_t blocks = w[i].heads * ((w[i].Dv + 63) / 64);
    items += blocks;
    wide = wide || w[i].Dk > 64;
    few = few && blocks <= sm_count();
  }
  for (int i = 0; i < (few ? 1 : n); ++i) {
    const double blocks = few ? (double)items : (double)(w[i].heads * ((w[i].Dv + 63) / 64));
    const double many = (few ? 2.0e-3 : 1.3e-3) * blocks, per_step = many > 0.48 ? many : 0.48;
    steps += 3.0 + (double)T * per_step * (w[i].Dk > 64 ? 2.0 : 1.0);
  }
  return steps < 1.5 + (wide ? 13.2 : 9.6) * (double)((items + sm_count() - 1) / sm_count());
}

// Splits walks into the two widths of the chunked kernel; returns how many come first.
int by_width(const Walk* in, int n, Walk* out) {
  int k = 0;
  for (int i = 0; i < n; ++i)
    if (in[i].Dk <= 64) out[k++] = in[i];
  const int narrow = k;
  for (int i = 0; i < n; ++i)
    if (in[i].Dk > 64) out[k++] = in[i];
  return narrow;
}

int run_walks(const Walk* walks, int n, bool fp32, void* scratch, cudaStream_t s) {
  if (fp32 || walks_by_steps(walks, n)) return launch_walks(walks, n, s);
  Walk w[3];
  const int narrow = by_width(walks, n, w);
  float* f = static_cast<float*>(scratch);
  if (narrow) {
    const int64_t need = tc_scratch_floats(w, narrow);
    SB_REQUIRE(need == 0 || f, "null scratch pointer");
    SB_TRY(tc_walks(w, narrow, f, s));
    f += need;
  }
  if (narrow < n) {
    SB_REQUIRE(tc_scratch_floats(w + narrow, n - narrow) == 0 || scratch, "null scratch pointer");
    SB_TRY(tc_walks(w + narrow, n - narrow, f, s));
  }
  return SB_OK;
}

// The walks of a forward or backward pass, without tensors: what the scratch size is computed from.
int shape_walks(int64_t heads, int dk, int dv, int64_t T, bool backward, Walk* w) {
  Walk f{}, b{};
  f.heads = b.heads = heads;
  f.T = b.T = T;
  f.Dk = b.Dv = dk;
  f.Dv = b.Dk = dv;
  w[0] = backward ? b : f;
  w[1] = b;
  w[2] = f;
  return backward ? 3 : 1;
}

// ---------------------------------------------------------------------------
// One step on a kept state: reads and writes the state once, Dk x Dv floats each way.
// Threads lie over the columns of a state row (four each) and over groups of rows; a thread's NI rows are
// all loaded before the first is written back (they are the same memory, so the compiler would wait for one
// after the other).
// ---------------------------------------------------------------------------
template <bool VEC, int NI>
__global__ void __launch_bounds__(256)
step_kernel(const float* __restrict__ q, const float* __restrict__ k, const float* __restrict__ v,
            const float* __restrict__ decay, int n_decay, float* state, float* __restrict__ o, int Dk, int Dv, int lanes) {
  __shared__ float part[256 * 4];
  const int64_t head = blockIdx.x;
  const int tid = threadIdx.x, col = (tid % lanes) * 4, group = tid / lanes, groups = 256 / lanes;
  float* S = state + head * Dk * Dv + col;
  float x[NI][4], kd[NI], qd[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int d = group + i * groups;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
    kd[i] = qd[i] = 0.f;
    if (d < Dk && col < Dv) {
      if (VEC) {
        const float4 a = *reinterpret_cast<const float4*>(S + (int64_t)d * Dv);
        x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < Dv) x[i][e] = S[(int64_t)d * Dv + e];
      }
      kd[i] = __ldg(k + head * Dk + d);
      qd[i] = __ldg(q + head * Dk + d);
    }
  }
  const Keep keep = keep_of(decay[n_decay > 1 ? head % n_decay : 0]);
  float ve[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) ve[e] = col + e < Dv ? __ldg(v + head * Dv + col + e) : 0.f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int d = group + i * groups;
    if (d < Dk && col < Dv) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[i][e] = fmaf(keep.r, x[i][e], fmaf(keep.lo, x[i][e], kd[i] * ve[e]));
        acc[e] = fmaf(qd[i], x[i][e], acc[e]);
      }
      if (VEC) {
        *reinterpret_cast<float4*>(S + (int64_t)d * Dv) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < Dv) S[(int64_t)d * Dv + e] = x[i][e];
      }
    }
  }
  *reinterpret_cast<float4*>(&part[tid * 4]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (tid < Dv) {
    float sum = 0.f;
    for (int g = 0; g < groups; ++g) sum += part[g * lanes * 4 + tid];
    o[head * Dv + tid] = sum;
  }
}

template <bool VEC>
void launch_step(const float* q, const float* k, const float* v, const float* decay, int n_decay, float* state, float* o,
                 int64_t heads, int Dk, int Dv, cudaStream_t s) {
  int lanes = 1;
  while (lanes * 4 < Dv) lanes *= 2;
  const int rows = (Dk * lanes + 255) / 256;             // per thread: 1 to 16
  const unsigned g = (unsigned)heads;
  if (rows <= 1) step_kernel<VEC, 1><<<g, 256, 0, s>>>(q, k, v, decay, n_decay, state, o, Dk, Dv, lanes);
  else if (rows <= 2) step_kernel<VEC, 2><<<g, 256, 0, s>>>(q, k, v, decay, n_decay, state, o, Dk, Dv, lanes);
  else if (rows <= 4) step_kernel<VEC, 4><<<g, 256, 0, s>>>(q, k, v, decay, n_decay, state, o, Dk, Dv, lanes);
  else if (rows <= 8) step_kernel<VEC, 8><<<g, 256, 0, s>>>(q, k, v, decay, n_decay, state, o, Dk, Dv, lanes);
  else step_kernel<VEC, 16><<<g, 256, 0, s>>>(q, k, v, decay, n_decay, state, o, Dk, Dv, lanes);
}

int check_shape(int64_t heads, int64_t H, int64_t n_decay, int64_t Dk, int64_t Dv, int64_t T) {
  SB_REQUIRE(heads >= 0 && T >= 0 && H >= 1, "negative geometry");
  SB_REQUIRE(Dk >= 1 && Dk <= kMaxDim && Dv >= 1 && Dv <= kMaxDim, "head widths %lld, %lld outside 1..%d",
             (long long)Dk, (long long)Dv, kMaxDim);
  SB_REQUIRE(heads % H == 0, "%lld heads are no multiple of %lld heads a sample", (long long)heads, (long long)H);
  SB_REQUIRE(n_decay == 1 || n_decay == H, "decay has %lld elements, expected 1 or %lld", (long long)n_decay,
             (long long)H);
  SB_REQUIRE(T < (1LL << 31) - 256 && heads < (1LL << 31), "geometry too large");
  return SB_OK;
}

int forward(const float* q, const float* k, const float* v, const float* decay, int64_t n_decay, const float* state,
            float* out, float* final_state, int64_t heads, int64_t H, int64_t Dk, int64_t Dv, int64_t T, bool fp32,
            void* scratch, void* stream) {
  SB_TRY(check_shape(heads, H, n_decay, Dk, Dv, T));
  if (heads == 0) return SB_OK;
  SB_REQUIRE(decay && (T == 0 || (q && k && v && out)), "null tensor pointer");
  const Walk w{q, k, v, out, decay, state, final_state, (int)n_decay, heads, (int)Dk, (int)Dv, T, Dv, 1, 0, 1};
  return run_walks(&w, 1, fp32, scratch, (cudaStream_t)stream);
}

int backward(const float* q, const float* k, const float* v, const float* decay, int64_t n_decay, const float* state,
             const float* grad_out, const float* grad_final, float* grad_q, float* grad_k, float* grad_v,
             float* grad_state, int64_t heads, int64_t H, int64_t Dk, int64_t Dv, int64_t T, bool fp32, void* scratch,
             void* stream) {
  SB_TRY(check_shape(heads, H, n_decay, Dk, Dv, T));
  if (heads == 0) return SB_OK;
  SB_REQUIRE(decay && (T == 0 || (q && k && v && grad_out && grad_q && grad_k && grad_v)), "null tensor pointer");
  const int nd = (int)n_decay, dk = (int)Dk, dv = (int)Dv;
  const Walk w[3] = {{grad_out, v, k, grad_q, decay, state, nullptr, nd, heads, dv, dk, T, 1, Dv, 0, 1},
                     {v, grad_out, q, grad_k, decay, grad_final, nullptr, nd, heads, dv, dk, T, 1, Dv, 1, 0},
                     {k, q, grad_out, grad_v, decay, grad_final, grad_state, nd, heads, dk, dv, T, Dv, 1, 1, 0}};
  return run_walks(w, 3, fp32, scratch, (cudaStream_t)stream);
}

}  // namespace

extern "C" {

int64_t sb_linear_attention_scratch_bytes(int64_t heads, int64_t Dk, int64_t Dv, int64_t T, int backward) {
  if (check_shape(heads, 1, 1, Dk, Dv, T) != SB_OK || heads == 0 || T < 128) return 0;   // (one chunk is not cut)
  Walk all[3], w[3];
  const int n = shape_walks(heads, (int)Dk, (int)Dv, T, backward != 0, all);
  const int narrow = by_width(all, n, w);
  int64_t floats = 0;
  if (narrow) floats += tc_scratch_floats(w, narrow);
  if (narrow < n) floats += tc_scratch_floats(w + narrow, n - narrow);
  return floats * (int64_t)sizeof(float);
}

int sb_linear_attention_fwd(const float* q, const float* k, const float* v, const float* decay, int64_t n_decay,
                            const float* state, float* out, float* final_state, int64_t heads, int64_t H, int64_t Dk,
                            int64_t Dv, int64_t T, void* scratch, void* stream) {
  return forward(q, k, v, decay, n_decay, state, out, final_state, heads, H, Dk, Dv, T, false, scratch, stream);
}

int sb_linear_attention_fwd_fp32(const float* q, const float* k, const float* v, const float* decay, int64_t n_decay,
                                 const float* state, float* out, float* final_state, int64_t heads, int64_t H,
                                 int64_t Dk, int64_t Dv, int64_t T, void* stream) {
  return forward(q, k, v, decay, n_decay, state, out, final_state, heads, H, Dk, Dv, T, true, nullptr, stream);
}

int sb_linear_attention_bwd(const float* q, const float* k, const float* v, const float* decay, int64_t n_decay,
                            const float* state, const float* grad_out, const float* grad_final, float* grad_q,
                            float* grad_k, float* grad_v, float* grad_state, int64_t heads, int64_t H, int64_t Dk,
                            int64_t Dv, int64_t T, void* scratch, void* stream) {
  return backward(q, k, v, decay, n_decay, state, grad_out, grad_final, grad_q, grad_k, grad_v, grad_state, heads, H, Dk,
                  Dv, T, false, scratch, stream);
}

int sb_linear_attention_bwd_fp32(const float* q, const float* k, const float* v, const float* decay, int64_t n_decay,
                                 const float* state, const float* grad_out, const float* grad_final, float* grad_q,
                                 float* grad_k, float* grad_v, float* grad_state, int64_t heads, int64_t H, int64_t Dk,
                                 int64_t Dv, int64_t T, void* stream) {
  return backward(q, k, v, decay, n_decay, state, grad_out, grad_final, grad_q, grad_k, grad_v, grad_state, heads, H, Dk,
                  Dv, T, true, nullptr, stream);
}

int sb_linear_attention_step(const float* q, const float* k, const float* v, const float* decay, int64_t n_decay,
                             float* state, float* out, int64_t heads, int64_t H, int64_t Dk, int64_t Dv,
                             void* stream) {
  SB_TRY(check_shape(heads, H, n_decay, Dk, Dv, 1));
  if (heads == 0) return SB_OK;
  SB_REQUIRE(q && k && v && decay && state && out, "null tensor pointer");
  const bool vec = Dv % 4 == 0 && ((uintptr_t)state & 15u) == 0;
  const cudaStream_t s = (cudaStream_t)stream;
  const auto launch = vec ? launch_step<true> : launch_step<false>;
  launch(q, k, v, decay, (int)n_decay, state, out, heads, (int)Dk, (int)Dv, s);
  SB_CUDA(cudaGetLastError());
  return SB_OK;
}

}  // extern "C"
