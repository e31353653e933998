// Linear attention on the tensor cores: the walk of api_linear_attention.cu in chunks of 128 steps.
//
// With i, j the steps of a chunk, S the state before it and a = 1 (the state decays before a step is
// added) or 0 (after it has been read),
//
//   o_i  = sum_{j <= i} r^(i-j) (q_i . k_j) v_j  +  r^(i+a) S^T q_i
//   S'   = r^L S + sum_j r^(L-a-j) k_j v_j^T                        (L = 128, or what is left of T)
//
// i.e. four products per chunk and 64 columns of v: scores q k^T [128 x Dk x 128], read-out P v
// [128 x 128 x 64], the state's part q S [128 x Dk x 64] and its growth v^T k [64 x 128 x Dk].
//
// Precision.  The operands are fp32.  Each is split into two fp16 numbers, x 2^-f = hi + lo, 22 bits
// together, and a product is hi hi + lo hi + hi lo with fp32 accumulators: what is dropped is below
// 2^-22 of a term.  fp16 rather than TF32 pairs because an MMA step then takes 16 elements of the
// contraction instead of 8 and a tile half the shared memory, which is what leaves room to stage the
// next chunk.  fp16 has no range, so the powers of two travel beside the mantissas: q, k and v have one
// exponent per step, the state one per column of v, and a row of P one per step i: |q_i . k_j| is at most
// Dk times the two largest elements, so the largest of 2^(f + g) over j <= i (a running maximum that
// decays with r) bounds the row without looking at it, and no outlier costs the accuracy of a step that
// does not read it.  A vector's largest element has 2^13 or more and an fp16 pair steps of 2^-24.
//
// Values that are not finite must not meet a zero of the causal mask in an MMA (0 * NaN): the loader
// zeroes them and notes from which step on a column of the output is spoilt.
//
// Layout.  Time is contiguous in memory, so a thread that owns one step reads 64 rows with coalesced
// loads and holds that step's whole vector: its exponent needs no exchange, and its hi and lo halves are
// written as one 128-byte row of a [step][channel] tile each.  That one tile of k is the K-major B
// operand of the scores and the MN-major B operand of the growth; v is MN-major in the read-out, and a
// copy weighted by r^(L-a-j) is the MN-major A operand of the growth (64 rows, repeated to M = 128: each
// half of the lanes keeps half of the columns).  q goes to tensor memory (it is A of two products) and so does P,
// converted in place of the scores.
//
// Roles of a CTA (one per SM, six warpgroups): k, v and q are each converted by a warpgroup (one step per
// thread) out of raw tiles that TMA has landed, in place for k and v; one turns scores into P, one keeps the
// state (32 elements per thread and 64 of Dk in registers, fp32) and writes the output; of the last, three
// single threads issue the MMAs and the TMA loads.  Tensors that TMA cannot describe (T % 4 != 0, unaligned)
// are loaded by the converting threads themselves.
//
// What bounds it is the instruction stream.  A chunk of 128 steps and 64 channels a side (131 KB, 3.0 us of
// an SM's share of copy bandwidth; 0.65 us of MMA time at the bf16 rate) takes 6.5 us, 12,000 cycles, in which
// a scheduler issues 4,500 instructions, mostly the splitting into fp16 pairs, at 0.38 per cycle with a
// sixth of the fetches missing the instruction cache.  Steps on the way: one loading warpgroup with two
// operands in registers 15.3 us, a warpgroup per operand 8.9, the same code for the three 7.7, TMA with
// raw tiles 7.7, waits that hold the warp in hardware instead of polling 6.4.
//
// A head with T steps is one CTA, or several when there are fewer heads than SMs: the axis is then cut
// into segments, a first launch takes each segment's growth from zero, a small one joins them, and the
// walk starts every segment from its own state.
#include <string.h>

#include "linear_attention.cuh"
#include "tc.cuh"

namespace sb {

int make_map_5d(CUtensorMap* out, const void* base, const uint64_t (&dims)[5], const uint64_t (&strides)[4],
                const uint32_t (&box)[5], int swizzle);

namespace la {
namespace {

constexpr int kL = 128;                      // steps per chunk
constexpr int kTileB = kL * 128;             // bytes of a [128 steps][64 channels] fp16 tile
constexpr int kThreads = 768;
// Registers per thread of the six warpgroups: 80 at launch (65536 / 768, in steps of 8), moved to where
// the vectors live.  Each row adds up to 6 * 80.
template <int KT>
struct Regs {
  static constexpr int load = KT == 1 ? 96 : 88, p = KT == 1 ? 72 : 64, s = KT == 1 ? 80 : 112, mma = 40;
  static_assert(3 * load + p + s + mma <= 480, "more registers than the block was launched with");
};
constexpr int kMaxSub = 6;

struct TcArgs {
  CUtensorMap map[3][3];   // q, k, v of each walk in boxes of 64 rows and 128 steps, when `boxes`
  Walk w[3];
  float* seg[3];        // [nseg][heads][Dk * Dv]: states after each segment
  int nsub;             // CTAs per head and segment: (walk, 64 columns of v)
  int sub_walk[kMaxSub], sub_e0[kMaxSub];
  int64_t heads;
  int nseg, seg_chunks;
  int boxes;            // TMA can describe the tensors: 16-byte bases, T % 4 == 0
  unsigned int* status;
};

template <int KT>
struct Shape {
  static constexpr int stages = KT == 1 ? 2 : 1;      // KT = 2 has room for one
  static constexpr int nq = KT == 1 ? 2 : 1;          // q's of chunks in tensor memory
  static constexpr int score = KT == 1 ? 34 : 35;     // scores of the scaled vectors are below 2^score: 2^14 2^14 Dk
  // shared memory: k, v (hi and lo tile of each 64 channels; the raw fp32 tile they are converted from lies
  // in the same 32 KB), weighted v, raw q (64 channels at a time), state
  static constexpr int k_bytes = 2 * KT * kTileB, v_at = stages * k_bytes, v_bytes = 2 * kTileB,
                       vw_at = v_at + stages * v_bytes, q_at = vw_at + v_bytes, s_at = q_at + v_bytes;
  static constexpr int smem = 1024 + s_at + 2 * KT * 64 * 128;
  // tensor memory columns
  static constexpr uint32_t q = 0, sp = 128, oi = sp + 128, ox = oi + 64, ds = ox + 64;
};

// Bounded wait of this kernel.  The hardware holds the warp until the phase completes or the hinted time is
// over, so that waiting warps do not fetch and issue polls between the instructions of the working ones.
// Gives up after two seconds, or when another thread has.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile int* dead) {
  uint64_t start = 0;
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
    if (ok) return true;
    uint64_t now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    if (start == 0) start = now;
    if (*dead) return false;
    if (now - start > 2000000000ull) {
      *dead = 1;
      return false;
    }
  }
}

__device__ __forceinline__ float p2(int n) { return __int_as_float((n + 127) << 23); }   // -126 <= n <= 127
struct Factors {
  float a, b;
};
// 2^n as two factors, so that n may leave the range of a float's exponent
__device__ __forceinline__ Factors p2_wide(int n) {
  n = max(-252, min(n, 254));
  return Factors{p2(n >> 1), p2(n - (n >> 1))};
}
// largest magnitude of three, NaN if one is NaN
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// pairs of floats in one 64-bit register: two products or sums per instruction
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// hi = fp16(x), lo = fp16(x - hi) of two neighbours, packed
__device__ __forceinline__ void split2(uint64_t x, uint32_t* hi, uint32_t* lo) {
  const float2 v = unpair(x);
  float h0, h1;
  uint32_t h;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(v.y), "f"(v.x));
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
      : "=f"(h0), "=f"(h1) : "r"(h));
  const float2 d = unpair(fma2(pair(h0, h1), pair(-1.f, -1.f), x));
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(*lo) : "f"(d.y), "f"(d.x));
  *hi = h;
}
// D (+)= A B^T, fp16 operands, fp32 accumulator: A in tensor memory or shared memory, B in shared memory
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %4};\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(acc)
      : "memory");
}
// fp16 x fp16 -> fp32, M = 128; bits 15 and 16 mark an MN-major A and B
__host__ __device__ constexpr uint32_t idesc_f16(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kL >> 4) << 24);
}
constexpr uint32_t kAMajorMN = 1u << 15, kBMajorMN = 1u << 16;
// Low descriptor word: K-major (the leading offset is unused with the 128-byte swizzle), or MN-major
// with the next 64 channels two tiles further on; groups of eight rows lie 1024 bytes apart either way.
__device__ __forceinline__ uint32_t desc_mn(uint32_t saddr) {
  return ((saddr & 0x3ffffu) >> 4) | ((uint32_t)(2 * kTileB >> 4) << 16);
}

// MN-major, the rows 64-127 a repetition of the rows 0-63
__device__ __forceinline__ uint32_t desc_twice(uint32_t saddr) { return (saddr & 0x3ffffu) >> 4; }

// 64 rows of one step.  volatile: the loads stay where they are issued, in one batch ahead of the waits
// and conversions (left to itself the compiler sinks them to their use).
__device__ __forceinline__ void load64(uint64_t (&x)[32], const float* p, int64_t T, int rows, bool in, bool whole) {
  if (whole && rows >= 64) {
#pragma unroll
    for (int d = 0; d < 64; d += 2) {
      float a, b;
      asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(a) : "l"(p));
      p += T;
      asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(b) : "l"(p));
      p += T;
      x[d / 2] = pair(a, b);
    }
  } else {
    const int n = in ? rows : 0;
#pragma unroll
    for (int d = 0; d < 64; d += 2) {
      float a, b;
      asm volatile(
          "{\n\t.reg .pred p;\n\tsetp.gt.s32 p, %2, %3;\n\tmov.f32 %0, 0f00000000;\n\t@p ld.global.nc.f32 %0, [%1];\n\t}"
          : "=f"(a) : "l"(p), "r"(n), "r"(d));
      p += T;
      asm volatile(
          "{\n\t.reg .pred p;\n\tsetp.gt.s32 p, %2, %3;\n\tmov.f32 %0, 0f00000000;\n\t@p ld.global.nc.f32 %0, [%1];\n\t}"
          : "=f"(b) : "l"(p), "r"(n), "r"(d + 1));
      p += T;
      x[d / 2] = pair(a, b);
    }
  }
}
// the same out of a raw tile [64][128] in shared memory (rows and steps outside the tensor are zeros)
__device__ __forceinline__ void load64_shared(uint64_t (&x)[32], uint32_t p) {
#pragma unroll
  for (int d = 0; d < 32; ++d) {
    float a, b;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(a) : "r"(p + d * 1024));
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(b) : "r"(p + d * 1024 + 512));
    x[d] = pair(a, b);
  }
}
__device__ __forceinline__ float top64_shared(uint32_t p, float m) {
#pragma unroll
  for (int d = 0; d < 32; ++d) {
    float a, b;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(a) : "r"(p + d * 1024));
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(b) : "r"(p + d * 1024 + 512));
    m = max_abs3(m, a, b);
  }
  return m;
}
__device__ __forceinline__ void tma_load_box(uint32_t dst, const CUtensorMap* map, int t, int row, int head, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(t), "r"(row), "r"(head), "r"(0), "r"(bar)
      : "memory");
}
__device__ __forceinline__ float top64(const uint64_t (&x)[32], float m = 0.f) {
#pragma unroll
  for (int d = 0; d < 32; ++d) {
    const float2 v = unpair(x[d]);
    m = max_abs3(m, v.x, v.y);
  }
  return m;
}
// Exponent that brings a largest magnitude into [2^13, 2^14); a zero vector gets one that no sum prefers.
constexpr int kNoTerm = -400;
__device__ __forceinline__ int fit_exponent(float top) {
  const int e = (int)(__float_as_uint(top) >> 23) - 127;
  return max(e, -113) - 13;
}
__device__ __forceinline__ bool not_finite(float top) { return __float_as_uint(top) >= 0x7f800000u; }
template <int R>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

// KT: 64-wide tiles of Dk.  FULL: the walk itself; otherwise only the state after each segment but the last.
template <int KT, bool FULL>
__global__ void __launch_bounds__(kThreads, 1) attention_tc_kernel(const __grid_constant__ TcArgs args) {
  using S_ = Shape<KT>;
  constexpr int NS = S_::stages;
  extern __shared__ uint8_t raw[];
  // What travels beside the mantissas.  A slot of two is rewritten for chunk c + 2 once the read-out of
  // chunk c has ended, a slot of four once the output of chunk c + 1 has been written.
  __shared__ int f_s[2][kL];                                        // k's exponent
  __shared__ int fg_s[2][kL];                                       // k's and v's exponents together
  __shared__ __align__(16) float col_s[kL];                         // of a column of P: 2^(fg - largest fg)
  __shared__ int m_s[4][kL], qe_s[4][kL], mw_s[4];
  __shared__ float scan_s[4];
  __shared__ int fmax_s[4], kmax_s[2][4];
  __shared__ float pow_pad[32 + kL + 1];       // r^n at 32 + n; zeros before it are the causal mask
  __shared__ __align__(16) float scale_s[2][64];
  __shared__ float top_s[kL];
  __shared__ int poison_s[64];
  __shared__ int any_poison_s, dead_s;
  __shared__ uint32_t tmem_s;
  __shared__ __align__(8) uint64_t bars[30];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, role = tid >> 7, th = tid & 127, tw = warp & 3;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t sbase = base + S_::s_at;
  volatile int* dead = &dead_s;
  volatile int* any_poison = &any_poison_s;
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  // by stage or chunk parity: two each
  const uint32_t bar_k = bar(0), bar_v = bar(2), bar_free = bar(4), bar_kx = bar(6), bar_kraw = bar(8), bar_vraw = bar(10),
                 bar_q = bar(12), bar_qfree = bar(14);
  const uint32_t bar_sp = bar(16), bar_p = bar(17), bar_ds = bar(18), bar_s = bar(19), bar_o = bar(20), bar_ofree = bar(21),
                 bar_qraw = bar(22), bar_qread = bar(23), bar_end = bar(24), bar_dsfree = bar(25);
  const uint32_t bar_kfree = bar(26), bar_vw = bar(28);    // two each

  // which head, segment, walk and columns
  const int64_t bid = blockIdx.x;
  const int sub = (int)(bid % args.nsub);
  const int64_t head = (bid / args.nsub) % args.heads;
  const int seg = (int)(bid / args.nsub / args.heads);
  const int wi = args.sub_walk[sub], e0 = args.sub_e0[sub];
  const Walk& w = args.w[wi];
  const int64_t T = w.T;
  const int Dk = w.Dk, ne = min(64, w.Dv - e0);
  const int64_t c0 = (int64_t)seg * args.seg_chunks;
  const int nc = (int)min((int64_t)args.seg_chunks, (T + kL - 1) / kL - c0);
  const int after = w.after;
  const bool boxes = args.boxes != 0;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_k + 8 * i, 128);
      mbar_init(bar_v + 8 * i, 128);
      mbar_init(bar_free + 8 * i, 1);
      mbar_init(bar_kfree + 8 * i, 1);
      mbar_init(bar_vw + 8 * i, 128);
      mbar_init(bar_q + 8 * i, 128);
      mbar_init(bar_qfree + 8 * i, 2);
      mbar_init(bar_kx + 8 * i, 128);
      mbar_init(bar_kraw + 8 * i, 1);
      mbar_init(bar_vraw + 8 * i, 1);
    }
    mbar_init(bar_qraw, 1);
    mbar_init(bar_qread, 128);
    mbar_init(bar_sp, 2);
    mbar_init(bar_p, 128);
    mbar_init(bar_ds, 2);
    mbar_init(bar_s, 128);
    mbar_init(bar_dsfree, 128);
    mbar_init(bar_o, 2);
    mbar_init(bar_ofree, 128);
    mbar_init(bar_end, 1);
    fence_mbar_init();
    dead_s = 0;
    any_poison_s = 0;
  }
  if (tid < 64) poison_s[tid] = 0x7fffffff;
  if (tid < 32) pow_pad[tid] = 0.f;
  if (tid <= kL) {
    // r^n by squaring in 64 bits: r itself does not fit 32 (a slow head multiplies it a thousandfold)
    double b = 1.0 - (double)w.decay[w.n_decay > 1 ? head % w.n_decay : 0] / 4096.0, p = 1.0;
    for (int n = tid; n; n >>= 1) {
      if (n & 1) p *= b;
      b *= b;
    }
    pow_pad[32 + tid] = (float)p;
  }
  if (role == 5 && tw == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_s)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  const uint32_t trow = tmem + ((uint32_t)(tw * 32) << 16);   // this warp's lanes of tensor memory

  if (role < 3) {
    // ---------------- k, v, q: load, convert, hand on ----------------
    regs_inc<Regs<KT>::load>();
    const int j = th;
    const bool is_k = role == 0, is_v = role == 1, is_q = role == 2;
    const float* src = is_k ? w.k + head * (int64_t)Dk * T
                            : (is_v ? w.v + (head * (int64_t)w.Dv + e0) * T : w.q + head * (int64_t)Dk * T);
    const int rows = is_v ? ne : Dk;
    // Passes over an operand.  Dk > 64 needs the largest magnitude of both halves before either is converted:
    // k's raw tiles are looked through first; otherwise the first half is loaded, the second, which is
    // converted while it is there, and the first again.  v: weighted, and as it is.
    const bool ahead = KT == 2 && is_k && boxes;
    const int passes = is_v ? (FULL ? 2 : 1) : (KT == 1 ? 1 : (ahead ? 2 : 3));
    const int mid = is_v || ahead ? 0 : KT - 1;  // the pass after whose load the exponent is known
#pragma unroll 1
    for (int c = (FULL || !is_q) ? 0 : nc; c < nc; ++c) {
      const uint32_t slot = base + (is_k ? (uint32_t)(c % NS) * S_::k_bytes
                                         : (is_v ? S_::v_at + (uint32_t)(c % NS) * S_::v_bytes : S_::q_at));
      const int64_t t = (c0 + c) * kL + j;
      const int len = (int)min((int64_t)kL, T - (c0 + c) * kL);
      const bool in = j < len, whole = len == kL;
      const float* at = src + (w.reverse ? T - 1 - t : t);
      uint64_t x[32];
      float top = 0.f, scale = 0.f, scale_w = 0.f;
      bool zero = false;                         // the whole vector is left out
#pragma unroll 1
      for (int pass = 0; pass < passes; ++pass) {
        const int half = (KT == 2 && !is_v && pass == 1) ? 1 : 0;
        if (!is_v || pass == 0) {
          if (boxes) {
            // the raw tile, a step earlier or later in memory by direction; its place is free to be written
            // (k, v) or to receive the next tile (q) once the whole warpgroup has read it
            const uint32_t raw_at = slot + (uint32_t)(w.reverse ? kL - 1 - j : j) * 4;
            if (is_q) {
              const uint32_t n = (uint32_t)(KT == 1 ? c : 3 * c + pass);
              wait_phase(bar_qraw, n & 1u, dead);
            } else if (pass == 0) {
              wait_phase((is_k ? bar_kraw : bar_vraw) + 8 * (c % NS), (uint32_t)(c / NS) & 1u, dead);
              if (ahead) top = top64_shared(raw_at + 2 * kTileB, top);
            }
            load64_shared(x, raw_at + (is_k ? (uint32_t)half * 2 * kTileB : 0u));
            if (is_q) mbar_arrive(bar_qread);
            else bar_sync(3 + role, 128);
          } else {
            load64(x, at + (int64_t)half * 64 * T, T, rows - half * 64, in, whole);
          }
        }
        if (pass <= mid) top = top64(x, top);
        if (pass == mid) {
          const bool bad = not_finite(top);
          if (is_k) {
            if (bad) {                           // every column of the output is spoilt from this step on
              for (int e = 0; e < 64; ++e) atomicMin(&poison_s[e], (int)t);
              any_poison_s = 1;
              zero = true;
            }
            const int f = fit_exponent(bad ? 0.f : top);
            scale = p2(-f);
            if (!boxes && c >= NS) wait_phase(bar_kfree + 8 * (c % NS), (uint32_t)(c / NS - 1) & 1u, dead);
            f_s[c & 1][j] = bad ? kNoTerm - 1 : (top > 0.f ? f : kNoTerm);
            mbar_arrive(bar_kx + 8 * (c & 1));
          } else if (is_q) {
            zero = bad;
            const int qe = bad ? 0 : fit_exponent(top);
            scale = p2(-qe);
            if (c >= S_::nq)
              wait_phase(bar_qfree + 8 * ((c - S_::nq) & 1), (uint32_t)((c - S_::nq) >> 1) & 1u, dead);
            tc_fence_after();
            qe_s[c & 3][j] = bad ? 0x7fffffff : qe;
          } else {
            // v, and what P and the growth need to know of the steps
            wait_phase(bar_kx + 8 * (c & 1), (uint32_t)(c >> 1) & 1u, dead);
            const int f = f_s[c & 1][j];
            zero = f == kNoTerm - 1;
            if (bad && !zero) {                  // single columns are spoilt; the rest of the vector counts
              for (int e = 0; e < ne; ++e)
                if (not_finite(fabsf(at[(int64_t)e * T]))) atomicMin(&poison_s[e], (int)t);
              any_poison_s = 1;
            }
            if (bad || zero) {
              top = 0.f;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                float2 v = unpair(x[e]);
                if (zero || not_finite(fabsf(v.x))) v.x = 0.f;
                if (zero || not_finite(fabsf(v.y))) v.y = 0.f;
                top = max_abs3(top, v.x, v.y);
                x[e] = pair(v.x, v.y);
              }
            }
            const int g = fit_exponent(top);
            const int fg = (top > 0.f && f > kNoTerm) ? f + g : kNoTerm;
            // weight of the step in the state, and the largest exponent of the weighted steps
            const float wt = in ? pow_pad[32 + len - after - j] : 0.f;
            const int we = (int)((__float_as_uint(wt) >> 23) & 0xff) - 127;
            const int key = wt != 0.f && fg != kNoTerm ? fg + we : kNoTerm;
            const int kmax = __reduce_max_sync(0xffffffffu, key);
            if (lane == 0) kmax_s[c & 1][tw] = kmax;
            bar_sync(1, 128);
            const int mw = max(max(kmax_s[c & 1][0], kmax_s[c & 1][1]), max(kmax_s[c & 1][2], kmax_s[c & 1][3]));
            if (!boxes && c >= NS) wait_phase(bar_free + 8 * (c % NS), (uint32_t)(c / NS - 1) & 1u, dead);
            if (FULL) fg_s[c & 1][j] = fg;
            if (j == 0) mw_s[c & 3] = mw;
            scale = p2(-g);
            // 2^-g r^(..) 2^(fg - mw): the two powers of two together, the weight's mantissa first.  What this
            // takes below a float's range is nothing in fp16 either.
            scale_w = key != kNoTerm ? (wt * p2(max(-we, -126))) * p2(max(fg + we - mw, -100)) * scale : 0.f;
          }
        }
        if (pass < mid) continue;
        if (__any_sync(0xffffffffu, zero)) {
          if (zero) {
#pragma unroll
            for (int d = 0; d < 32; ++d) x[d] = 0;
          }
        }
        // the weighted rows first where the growth waits for them (Dk > 64: 18.2 against 20.2 us per chunk of both
        // halves of v; Dk <= 64: 6.9 against 6.5)
        const bool weighted = is_v && (!FULL || pass == (KT == 2 ? 0 : 1));
        const float by = weighted ? scale_w : scale;
        const uint64_t sc = pair(by, by);
        if (is_q) {
          // 16 channels of q (one step of an MMA) are 8 columns of hi and 8 of lo, side by side: one store
#pragma unroll
          for (int b = 0; b < 32; b += 8) {
            uint32_t r[16];
#pragma unroll
            for (int e = 0; e < 8; ++e) split2(mul2(x[b + e], sc), &r[e], &r[8 + e]);
            tmem_st16(trow + S_::q + (uint32_t)(c % S_::nq) * 64 + half * 64 + 2 * b, r);
          }
          if constexpr (KT == 1) break;          // (x is not carried on)
          continue;
        }
        // one row of a hi and a lo tile (128-byte swizzle)
        if (weighted && c >= 1) wait_phase(bar_ds, (uint32_t)(c - 1) & 1u, dead);    // read by the growth before
        const uint32_t tile = (weighted ? base + S_::vw_at : slot + (uint32_t)half * 2 * kTileB) + (uint32_t)(j * 128);
#pragma unroll
        for (int q8 = 0; q8 < 8; ++q8) {
          uint32_t h[4], l[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            split2(mul2(x[4 * q8 + e], sc), &h[e], &l[e]);
          }
          const uint32_t to = tile + (uint32_t)((q8 ^ (j & 7)) << 4);
          sts128(to, h[0], h[1], h[2], h[3]);
          sts128(to + kTileB, l[0], l[1], l[2], l[3]);
        }
        if (is_v || pass == passes - 1) {
          fence_proxy_async();
          mbar_arrive((is_k ? bar_k : (weighted ? bar_vw : bar_v)) + 8 * (c % NS));
        }
      }
      if (is_q) {
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar_q + 8 * (c & 1));
      }
    }
  } else if (role == 3) {
    // ---------------- scores -> P: thread = row i ----------------
    if constexpr (Regs<KT>::p < 80) regs_dec<Regs<KT>::p>();
    if constexpr (FULL) {
      const int l = th;
      // log2 r, for exponents only; a head that forgets everything at once gets a steep slope
      const float slope = fminf(fmaxf(log2f(fabsf(pow_pad[33])), -250.f), 250.f);
#pragma unroll 1
      for (int c = 0; c < nc; ++c) {
        const uint32_t sp = trow + S_::sp;
        wait_phase(bar_vw + 8 * (c % NS), (uint32_t)(c / NS) & 1u, dead);     // the steps' exponents
        // running maximum of fg_j + (i - j) log2 r: the scan runs on that less i log2 r
        const int fg = fg_s[c & 1][l];
        float mk = fg == kNoTerm ? -1e30f : (float)fg - (float)l * slope;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float up = __shfl_up_sync(0xffffffffu, mk, o);
          if (lane >= o) mk = fmaxf(mk, up);
        }
        const int fmax = __reduce_max_sync(0xffffffffu, fg);
        if (lane == 31) {
          scan_s[tw] = mk;
          fmax_s[tw] = fmax;
        }
        bar_sync(6, 128);
        const int mc = max(max(fmax_s[0], fmax_s[1]), max(fmax_s[2], fmax_s[3]));
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (i < tw) mk = fmaxf(mk, scan_s[i]);
        const int m = max(kNoTerm, (int)floorf(fmaxf(mk + (float)l * slope, (float)kNoTerm)) + 1);
        m_s[c & 3][l] = m;
        col_s[l] = fg == kNoTerm ? 0.f : p2(max(fg - mc, -126));
        bar_sync(6, 128);
        wait_phase(bar_sp, (uint32_t)c & 1u, dead);
        tc_fence_after();
        // |q_i . k_j| <= 2^score of the scaled vectors: P is held as its multiple of 2^(m + score - 15)
        const float rowf = p2(max(-126, min(mc - m - (S_::score - 15), 127)));
        const uint64_t rf = pair(rowf, rowf);
        const float* pw = &pow_pad[32 + l];      // r^(i - j), zero for j > i: the mask
        const float* col = col_s;
#pragma unroll 1
        for (int g = 0; g < 128; g += 32, pw -= 32, col += 32) {
          uint32_t s[32];                        // 16 columns of hi and 16 of lo, in the place of 32 scores
          if (g <= tw * 32) {
            uint32_t r[32];
            tmem_ld32(sp + g, r);
            tmem_ld_wait();
#pragma unroll
            for (int jj = 0; jj < 32; jj += 4) {
              const float4 cf = *reinterpret_cast<const float4*>(col + jj);
              // the power first: its zeros take whatever the steps after i hold
              const uint64_t x = mul2(pair(__uint_as_float(r[jj]), __uint_as_float(r[jj + 1])), pair(pw[-jj], pw[-jj - 1]));
              const uint64_t y = mul2(pair(__uint_as_float(r[jj + 2]), __uint_as_float(r[jj + 3])), pair(pw[-jj - 2], pw[-jj - 3]));
              split2(mul2(mul2(x, pair(cf.x, cf.y)), rf), &s[jj / 2], &s[16 + jj / 2]);
              split2(mul2(mul2(y, pair(cf.z, cf.w)), rf), &s[jj / 2 + 1], &s[17 + jj / 2]);
            }
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) s[x] = 0u;
          }
          tmem_st32(sp + g, s);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar_p);
      }
    }
  } else if (role == 4) {
    // ---------------- state (thread = column e, half of Dk) and output (thread = step i) ----------------
    if constexpr (Regs<KT>::s > 80) regs_inc<Regs<KT>::s>();
    const int l = th, e = l & 63, half = l >> 6;
    constexpr int NSt = 32 * KT;                 // state elements per thread: d = half * NSt ...
    float St[NSt];
    {
      const float* src = nullptr;
      int64_t rs = 0, cs = 0;
      if (seg == 0) {
        if (w.s_in) { src = w.s_in + head * (int64_t)Dk * w.Dv; rs = w.s_row; cs = w.s_col; }
      } else if (FULL) {
        src = args.seg[wi] + ((int64_t)(seg - 1) * args.heads + head) * Dk * w.Dv; rs = w.Dv; cs = 1;
      }
#pragma unroll
      for (int i = 0; i < NSt; ++i) {
        const int d = half * NSt + i;
        St[i] = (src && d < Dk && e < ne) ? src[d * rs + (int64_t)(e0 + e) * cs] : 0.f;
      }
    }
    // the state as the B operand [e][d] of the read-out, one exponent per row
    auto publish = [&](int slot) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < NSt; ++i) top = fmaxf(top, fabsf(St[i]));
      top_s[l] = top;
      bar_sync(2, 128);
      top = fmaxf(top, top_s[l ^ 64]);
      const int se = min(fit_exponent(top), 113);
      const uint64_t ss = pair(p2(-se), p2(-se));
      if (half == 0) scale_s[slot][e] = p2(se);
      const uint32_t tile = sbase + (KT == 2 ? half * 8192 : 0);
#pragma unroll
      for (int c = 0; c < NSt / 8; ++c) {
        uint32_t h[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) split2(mul2(pair(St[8 * c + 2 * x], St[8 * c + 2 * x + 1]), ss), &h[x], &lo[x]);
        const int chunk = (KT == 1 ? half * 4 : 0) + c;
        const uint32_t at = tile + (uint32_t)(e * 128 + ((chunk ^ (e & 7)) << 4));
        sts128(at, h[0], h[1], h[2], h[3]);
        sts128(at + KT * 8192, lo[0], lo[1], lo[2], lo[3]);
      }
      fence_proxy_async();
    };
    // Trip c writes the output of chunk c - 1, then takes the state over chunk c.  Trip -1 publishes what the
    // walk starts from.
#pragma unroll 1
    for (int c = -1; c <= (FULL ? nc : nc - 1); ++c) {
      if (FULL && c >= 1) {
        const int p = c - 1;                     // the chunk whose output this is
        const int64_t t = (c0 + p) * kL + l;
        float* out = w.o + (head * (int64_t)w.Dv + e0) * T + (w.reverse ? T - 1 - t : t);
        const bool live = t < T, plain = (c0 + p + 1) * kL <= T && ne == 64;
        wait_phase(bar_o, (uint32_t)p & 1u, dead);
        tc_fence_after();
        const int qe = qe_s[p & 3][l], m = m_s[p & 3][l] + S_::score - 15;
        const bool bad = qe == 0x7fffffff;
        const Factors fi = p2_wide((bad ? 0 : qe) + m), fx = p2_wide(bad ? 0 : qe);
        const float nan = __int_as_float(0x7fffffff), rowx = fx.b * pow_pad[32 + l + after];
        const uint64_t ia = pair(bad ? nan : fi.a, bad ? nan : fi.a), ib = pair(fi.b, fi.b), xa = pair(fx.a, fx.a),
                       xb = pair(rowx, rowx);
#pragma unroll 1
        for (int b = 0; b < 64; b += 16) {
          uint32_t ri[16], rx[16];
          tmem_ld16(trow + S_::oi + b, ri);
          tmem_ld16(trow + S_::ox + b, rx);
          tmem_ld_wait();
          if (b == 48) {
            tc_fence_before();
            mbar_arrive(bar_ofree);
          }
          const float* sc = &scale_s[p & 1][b];
          float y[16];
#pragma unroll
          for (int x = 0; x < 16; x += 2) {
            const uint64_t inter = mul2(mul2(pair(__uint_as_float(rx[x]), __uint_as_float(rx[x + 1])), xa),
                                        mul2(pair(sc[x], sc[x + 1]), xb));
            const float2 v = unpair(fma2(mul2(pair(__uint_as_float(ri[x]), __uint_as_float(ri[x + 1])), ia), ib, inter));
            y[x] = v.x;
            y[x + 1] = v.y;
          }
          if (plain) {
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              *out = y[x];
              out += T;
            }
          } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              if (live && b + x < ne) *out = y[x];
              out += T;
            }
          }
        }
        if (*any_poison != 0 && live) {          // spoilt columns
          out -= 64 * T;
          for (int x = 0; x < ne; ++x)
            if (poison_s[x] <= (int)t) out[(int64_t)x * T] = nan;
        }
      }
      if (c == nc) break;
      if (c >= 0) {
        // the state after chunk c
        const int len = (int)min((int64_t)kL, T - (c0 + c) * kL);
        wait_phase(bar_ds, (uint32_t)c & 1u, dead);
        tc_fence_after();
        const Factors mw = p2_wide(mw_s[c & 3]);
        const float carry = pow_pad[32 + len];
        const uint64_t ma = pair(mw.a, mw.a), mb = pair(mw.b, mw.b), cy = pair(carry, carry);
        // (rows 64-127 of the accumulator repeat rows 0-63)
#pragma unroll
        for (int b = 0; b < NSt; b += 32) {
          uint32_t r[32];
          tmem_ld32(trow + S_::ds + (uint32_t)(half * NSt + b), r);
          tmem_ld_wait();
          if (b + 32 == NSt) {
            tc_fence_before();
            mbar_arrive(bar_dsfree);
          }
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            const uint64_t grown = mul2(mul2(pair(__uint_as_float(r[x]), __uint_as_float(r[x + 1])), ma), mb);
            const float2 v = unpair(fma2(cy, pair(St[b + x], St[b + x + 1]), grown));
            St[b + x] = v.x;
            St[b + x + 1] = v.y;
          }
        }
      }
      if (FULL && c + 1 < nc) {
        // the published state is replaced once the MMAs of the chunk have read it
        if (c >= 0) wait_phase(bar_qfree + 8 * (c & 1), (uint32_t)(c >> 1) & 1u, dead);
        publish((c + 1) & 1);
        mbar_arrive(bar_s);
      }
    }
    // the state after the last chunk
    float* dst = nullptr;
    int64_t rs = 0, cs = 0;
    if (!FULL) {
      dst = args.seg[wi] + ((int64_t)seg * args.heads + head) * Dk * w.Dv; rs = w.Dv; cs = 1;
    } else if (seg == args.nseg - 1 && w.s_out) {
      dst = w.s_out + head * (int64_t)Dk * w.Dv; rs = w.s_row; cs = w.s_col;
    }
    if (dst && e < ne) {
      const bool bad = poison_s[e] != 0x7fffffff;
#pragma unroll
      for (int i = 0; i < NSt; ++i) {
        const int d = half * NSt + i;
        if (d < Dk) dst[d * rs + (int64_t)(e0 + e) * cs] = bad ? __int_as_float(0x7fffffff) : St[i];
      }
    }
  } else {
    regs_dec<Regs<KT>::mma>();
    if (th == 0) {
      // ---------------- MMAs ----------------
      constexpr uint32_t id_scores = idesc_f16(kL), id_inter = idesc_f16(64), id_intra = idesc_f16(64) | kBMajorMN,
                         id_grow = idesc_f16(64 * KT) | kAMajorMN | kBMajorMN;
      const uint32_t tq = tmem + S_::q, toi = tmem + S_::oi, tox = tmem + S_::ox, tds = tmem + S_::ds;
      bool ok = true;
      // The barriers that count to two take an arrival of this thread beside the commit: it hands on what
      // the loaders wrote beside the operands.
      auto scores = [&](int c) {
        ok = wait_phase(bar_q + 8 * (c & 1), (uint32_t)(c >> 1) & 1u, dead) && ok;
        ok = wait_phase(bar_k + 8 * (c % NS), (uint32_t)(c / NS) & 1u, dead) && ok;
        if (!ok) return;
        tc_fence_after();
        const uint32_t k_hi = base + (uint32_t)(c % NS) * S_::k_bytes, d = tmem + S_::sp;
#pragma unroll 1
        for (int s = 0; s < 4 * KT; ++s) {
          const uint32_t bh = desc_lo(k_hi + (uint32_t)((s >> 2) * 2 * kTileB + (s & 3) * 32));
          const uint32_t q_hi = tq + (uint32_t)(c % S_::nq) * 64 + (uint32_t)s * 16;
          mma_f16_ts(d, q_hi, bh, id_scores, s > 0);
          mma_f16_ts(d, q_hi + 8, bh, id_scores, 1u);
          mma_f16_ts(d, q_hi, bh + (kTileB >> 4), id_scores, 1u);
        }
        umma_commit(bar_sp);
        mbar_arrive(bar_sp);
      };
      if (FULL) scores(0);
      // Growth first, it waits for nothing but the state's warps; then the state's part of the output, for
      // which the output before has to be taken away, the read-out, and the next chunk's scores.
#pragma unroll 1
      for (int c = 0; c < nc && ok; ++c) {
        const uint32_t k_hi = base + (uint32_t)(c % NS) * S_::k_bytes,
                       v_hi = base + S_::v_at + (uint32_t)(c % NS) * S_::v_bytes, vw_hi = base + S_::vw_at;
        if (!FULL) ok = wait_phase(bar_k + 8 * (c % NS), (uint32_t)(c / NS) & 1u, dead) && ok;
        ok = wait_phase(bar_vw + 8 * (c % NS), (uint32_t)(c / NS) & 1u, dead) && ok;
        if (c >= 1) ok = wait_phase(bar_dsfree, (uint32_t)(c - 1) & 1u, dead) && ok;
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int s = 0; s < 8; ++s) {
          const uint32_t a = desc_twice(vw_hi + s * 2048), b = desc_mn(k_hi + s * 2048);
          mma_f16_ss(tds, a, b, id_grow, s > 0);
          mma_f16_ss(tds, a + (kTileB >> 4), b, id_grow, 1u);
          mma_f16_ss(tds, a, b + (kTileB >> 4), id_grow, 1u);
        }
        umma_commit(bar_ds);
        mbar_arrive(bar_ds);
        umma_commit(bar_kfree + 8 * (c % NS));
        if (!FULL) {
          umma_commit(bar_free + 8 * (c % NS));
          continue;
        }
        ok = wait_phase(bar_s, (uint32_t)c & 1u, dead) && ok;
        if (c >= 1) ok = wait_phase(bar_ofree, (uint32_t)(c - 1) & 1u, dead) && ok;
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int s = 0; s < 4 * KT; ++s) {
          const uint32_t bh = desc_lo(sbase + (uint32_t)((s >> 2) * 8192 + (s & 3) * 32));
          const uint32_t q_hi = tq + (uint32_t)(c % S_::nq) * 64 + (uint32_t)s * 16;
          mma_f16_ts(tox, q_hi, bh, id_inter, s > 0);
          mma_f16_ts(tox, q_hi + 8, bh, id_inter, 1u);
          mma_f16_ts(tox, q_hi, bh + (KT * 8192 >> 4), id_inter, 1u);
        }
        umma_commit(bar_qfree + 8 * (c & 1));
        mbar_arrive(bar_qfree + 8 * (c & 1));
        ok = wait_phase(bar_v + 8 * (c % NS), (uint32_t)(c / NS) & 1u, dead) && ok;
        ok = wait_phase(bar_p, (uint32_t)c & 1u, dead) && ok;
        if (!ok) break;
        tc_fence_after();
        const uint32_t sp = tmem + S_::sp;
#pragma unroll 1
        for (int s = 0; s < 8; ++s) {
          const uint32_t p_hi = sp + (uint32_t)((s >> 1) * 32 + (s & 1) * 8), bh = desc_mn(v_hi + s * 2048);
          mma_f16_ts(toi, p_hi, bh, id_intra, s > 0);
          mma_f16_ts(toi, p_hi + 16, bh, id_intra, 1u);
          mma_f16_ts(toi, p_hi, bh + (kTileB >> 4), id_intra, 1u);
        }
        umma_commit(bar_o);
        mbar_arrive(bar_o);
        umma_commit(bar_free + 8 * (c % NS));
        if (c + 1 < nc) scores(c + 1);
      }
      umma_commit(bar_end);          // everything issued has landed before tensor memory is given back
      if (!mbar_wait(bar_end, 0)) *dead = 1;
    } else if (th == 32 && boxes) {
      // ---------------- raw k and v, a TMA box for 64 channels ----------------
      const CUtensorMap* maps = args.map[wi];
      int k_issued = 0, v_issued = 0;
#pragma unroll 1
      for (int c = 0; c < nc; ++c) {
        const int64_t t = (c0 + c) * kL;
        const int from = (int)(w.reverse ? T - t - kL : t);      // walking back, the last box may start before 0
        const uint32_t bk = bar_kraw + 8 * (c % NS), bv = bar_vraw + 8 * (c % NS), again = (uint32_t)(c / NS - 1) & 1u;
        if (c >= NS) wait_phase(bar_kfree + 8 * (c % NS), again, dead);
        if (*dead) break;
        mbar_expect_tx(bk, S_::k_bytes);
        for (int h = 0; h < KT; ++h)
          tma_load_box(base + (uint32_t)(c % NS) * S_::k_bytes + h * 2 * kTileB, &maps[1], from, 64 * h, (int)head, bk);
        k_issued = c + 1;
        if (c >= NS) wait_phase(bar_free + 8 * (c % NS), again, dead);
        if (*dead) break;
        mbar_expect_tx(bv, S_::v_bytes);
        tma_load_box(base + S_::v_at + (uint32_t)(c % NS) * S_::v_bytes, &maps[2], from, e0, (int)head, bv);
        v_issued = c + 1;
      }
      if (*dead) {   // nobody may have waited for the boxes in flight: not before they have landed
        for (int c = max(k_issued - NS, 0); c < k_issued; ++c) mbar_wait(bar_kraw + 8 * (c % NS), (uint32_t)(c / NS) & 1u);
        for (int c = max(v_issued - NS, 0); c < v_issued; ++c) mbar_wait(bar_vraw + 8 * (c % NS), (uint32_t)(c / NS) & 1u);
      }
    } else if (FULL && th == 64 && boxes) {
      // ---------------- raw q, 64 channels at a time ----------------
      constexpr int per = KT == 1 ? 1 : 3;       // the halves in the order they are asked for: 0, 1, 0
      int n = 0;
#pragma unroll 1
      for (; n < per * nc; ++n) {
        const int64_t t = (c0 + n / per) * kL;
        if (n >= 1) wait_phase(bar_qread, (uint32_t)(n - 1) & 1u, dead);
        if (*dead) break;
        mbar_expect_tx(bar_qraw, 2 * kTileB);
        tma_load_box(base + S_::q_at, &args.map[wi][0], (int)(w.reverse ? T - t - kL : t), n % per == 1 ? 64 : 0,
                     (int)head, bar_qraw);
      }
      if (*dead && n > 0) mbar_wait(bar_qraw, (uint32_t)(n - 1) & 1u);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (*dead && tid == 0) dev_flag(args.status, SB_DEV_TMA_TIMEOUT);
  if (role == 5 && tw == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// States after each segment from their growths: seg[s] += r^(steps of segment s) seg[s - 1].
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ TcArgs args, int nwalks) {
  for (int wi = 0; wi < nwalks; ++wi) {
    const Walk& w = args.w[wi];
    const int64_t per = (int64_t)w.Dk * w.Dv, total = per * args.heads;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
      const int64_t head = i / per;
      double b = 1.0 - (double)w.decay[w.n_decay > 1 ? head % w.n_decay : 0] / 4096.0, p = 1.0;
      for (int64_t n = (int64_t)args.seg_chunks * kL; n; n >>= 1) {
        if (n & 1) p *= b;
        b *= b;
      }
      const float r = (float)p;
      float* s = args.seg[wi] + i;
      float x = *s;
      for (int g = 1; g < args.nseg - 1; ++g) {
        s += total;
        x = fmaf(r, x, *s);
        *s = x;
      }
    }
  }
}

}  // namespace

// Segments the axis is cut into: `ctas` CTAs per segment walk `chunks` chunks.  The fewest waves of
// (segments x chunks) win; a cut axis is walked by the first launch too, at about half the cost of a
// chunk, and every CTA pays about two chunks to fill and drain.
int plan_segments(int64_t ctas, int64_t chunks) {
  const int64_t sms = sm_count();
  int best = 1;
  double best_cost = 0;
  for (int64_t n = 1; n <= chunks && n <= 256; ++n) {
    const int64_t per = (chunks + n - 1) / n;
    if ((chunks + per - 1) / per != n) continue;       // the same cut as a smaller n
    double cost = (double)((ctas * n + sms - 1) / sms) * (double)(per + 2);
    if (n > 1) cost += (double)((ctas * (n - 1) + sms - 1) / sms) * (0.5 * (double)per + 2) + 4;
    if (n == 1 || cost < best_cost) { best = (int)n; best_cost = cost; }
    if (ctas * n > 16 * sms) break;
  }
  return best;
}

int64_t tc_scratch_floats(const Walk* walks, int n) {
  int64_t ctas = 0, floats = 0;
  for (int i = 0; i < n; ++i) ctas += walks[i].heads * ((walks[i].Dv + 63) / 64);
  const int nseg = plan_segments(ctas, (walks[0].T + kL - 1) / kL);
  if (nseg > 1)
    for (int i = 0; i < n; ++i) floats += (int64_t)(nseg - 1) * walks[i].heads * walks[i].Dk * walks[i].Dv;
  return floats;
}

template <int KT>
static int go(const TcArgs& a, cudaStream_t s) {
  constexpr int smem = Shape<KT>::smem;
  SB_CUDA(cudaFuncSetAttribute(attention_tc_kernel<KT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int64_t ctas = a.heads * a.nsub;
  SB_REQUIRE(ctas * a.nseg < (1LL << 31), "geometry too large");
  if (a.nseg > 1) {
    SB_CUDA(cudaFuncSetAttribute(attention_tc_kernel<KT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attention_tc_kernel<KT, false><<<(unsigned)(ctas * (a.nseg - 1)), kThreads, smem, s>>>(a);
    SB_CUDA(cudaGetLastError());
  }
  return SB_OK;
}

// Walks of one launch: the same heads and T, Dk on the same side of 64.
int tc_walks(const Walk* walks, int n, float* scratch, cudaStream_t s) {
  TcArgs a;
  memset(&a, 0, sizeof(a));
  int64_t ctas = 0;
  a.nsub = 0;
  for (int i = 0; i < n; ++i) {
    a.w[i] = walks[i];
    for (int e0 = 0; e0 < walks[i].Dv; e0 += 64) {
      a.sub_walk[a.nsub] = i;
      a.sub_e0[a.nsub++] = e0;
    }
  }
  a.heads = walks[0].heads;
  ctas = a.heads * a.nsub;
  const int64_t chunks = (walks[0].T + kL - 1) / kL;
  a.nseg = plan_segments(ctas, chunks);
  a.seg_chunks = (int)((chunks + a.nseg - 1) / a.nseg);
  if (a.nseg > 1) {
    float* p = scratch;
    for (int i = 0; i < n; ++i) {
      a.seg[i] = p;
      p += (int64_t)(a.nseg - 1) * a.heads * walks[i].Dk * walks[i].Dv;
    }
  }
  uintptr_t bits = 0;
  for (int i = 0; i < n; ++i) bits |= (uintptr_t)walks[i].q | (uintptr_t)walks[i].k | (uintptr_t)walks[i].v;
  a.boxes = (bits & 15u) == 0 && walks[0].T % 4 == 0;
  for (int i = 0; i < n && a.boxes; ++i) {
    const Walk& w = walks[i];
    const float* base[3] = {w.q, w.k, w.v};
    for (int x = 0; x < 3; ++x) {
      const uint64_t D = (uint64_t)(x == 2 ? w.Dv : w.Dk), row = (uint64_t)w.T * 4, all = row * D * (uint64_t)w.heads;
      const uint64_t dims[5] = {(uint64_t)w.T, D, (uint64_t)w.heads, 1, 1}, strides[4] = {row, row * D, all, all};
      const uint32_t box[5] = {kL, 64, 1, 1, 1};
      SB_TRY(make_map_5d(&a.map[i][x], base[x], dims, strides, box, 0));
    }
  }
  a.status = status_ptr();
  if (!a.status) return SB_ERR_CUDA;
  const bool wide = walks[0].Dk > 64;
  if (wide) SB_TRY(go<2>(a, s));
  else SB_TRY(go<1>(a, s));
  if (a.nseg > 2) {
    int64_t most = 0;
    for (int i = 0; i < n; ++i) {
      const int64_t total = a.heads * walks[i].Dk * walks[i].Dv;
      most = total > most ? total : most;
    }
    const int64_t blocks = (most + 255) / 256;
    join_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(a, n);
    SB_CUDA(cudaGetLastError());
  }
  const unsigned grid = (unsigned)(ctas * a.nseg);
  if (wide) attention_tc_kernel<2, true><<<grid, kThreads, Shape<2>::smem, s>>>(a);
  else attention_tc_kernel<1, true><<<grid, kThreads, Shape<1>::smem, s>>>(a);
  SB_CUDA(cudaGetLastError());
  return SB_OK;
}

}  // namespace la
}  // namespace sb
