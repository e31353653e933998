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
// does not read it.  All exponents are whole numbers until they meet: the steps of a chunk and the powers of r
// between them may lie further apart than a float's range.  A vector's largest element has 2^13 or more and an fp16 pair steps of 2^-24.
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
// single threads issue the MMAs and the TMA loads and a warp works the items out.  Tensors that TMA cannot
// describe (T % 4 != 0, unaligned) are loaded by the converting threads themselves.
//
// What bounds it is the chain of roles, each a single warpgroup that hands a single buffer on: no unit of the SM
// is near its limit.  A chunk of 128 steps and 64 channels a side (131 KB, 3.0 us of an SM's share of copy
// bandwidth; 0.65 us of MMA time at the bf16 rate) takes 5.2 us on 148 SMs (17 for 128 channels a side, both
// halves of v).  Of that time the loader of k works 54 %, of v 72 %, of q 51 %, the scores' warps 65 %, the
// state's 71 % and the thread that issues MMAs 64 %; the rest they wait for one another.  While they work they
// wait as well, for shared and tensor memory (5.7 of the 14 cycles between a warp's instructions) and for
// instructions to be fetched (3.2): four warps have little to hide either behind.  Issue slots are 33 % used, the
// tensor pipe 20 %, DRAM 25 %.  Steps on the way (us a chunk, each as measured then): one loading
// warpgroup with two operands in registers 15.3, a warpgroup per operand 8.9, the same code for the three 7.7,
// TMA with raw tiles 7.7, waits that hold the warp in hardware instead of polling 6.4, what describes a head in
// shared memory instead of registers 5.5, a register split with 96 for the state's warps too 5.3 (128 channels
// 18.2 before, 15.7 so; 17 since exponents meet as whole numbers and powers of r keep theirs).
//
// The grid is one CTA per SM, which takes its items (a head, one of the walks, 64 columns of v, a segment of the
// axis) one after the other; the loaders are a chunk ahead across them, so short sequences do not fill and
// drain for each head (1024 heads of 128 steps: 91 us with a CTA for each item, 66 so).  With fewer items than SMs
// the axis is cut into segments: a first launch takes each segment's growth from zero, a small one joins them,
// and the walk starts every segment from its own state.
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
// the vectors live.  The sum may not pass 6 * 80.  148 heads of 2048 steps, us: 99 (64 channels) and 277 (128);
// with 88 for a loader, 104 for the state and 40 for the MMAs 25 and 14 more; with 88, 112 and 40 28 and 16; with 88
// for the state and 72 for the scores 1 and 5.
struct Regs {
  static constexpr int load = 96, p = 64, s = 96, mma = 32;
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
  int64_t items;        // (segment, head, sub) triples of this launch, sub fastest; a CTA takes every gridDim-th
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

// Barrier of `threads` threads that tells all of them whether one brought `x`.
__device__ __forceinline__ bool bar_any(int id, int threads, bool x) {
  int any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(any) : "r"((int)x), "r"(id), "r"(threads) : "memory");
  return any != 0;
}

__device__ __forceinline__ bool not_finite(float top) { return __float_as_uint(top) >= 0x7f800000u; }
__device__ __forceinline__ float p2(int n) { return __int_as_float((n + 127) << 23); }   // -126 <= n <= 127
struct Factors {
  float a, b;
};
// 2^n as two factors, so that n may leave the range of a float's exponent
__device__ __forceinline__ Factors p2_wide(int n) {
  n = max(-252, min(n, 254));
  return Factors{p2(n >> 1), p2(n - (n >> 1))};
}
// the same for n from -149 on, and zero below
__device__ __forceinline__ float p2_low(int n) {
  return n >= -126 ? p2(n) : __int_as_float(n >= -149 ? 1 << (n + 149) : 0);
}
// Powers of r leave a float's range within a chunk (r = 0.1 after 38 steps), while the states they apply to have
// 2^254 to lose.  So r = c 2^-kappa with c next to 1, and r^n = c^n 2^(-kappa n): c^n stays within 2^-64 .. 2^64
// and kappa n joins the other exponents.  A power as mantissa and exponent:
struct Power {
  float m;      // 1 to 2, signed
  int e;
};
constexpr int kNoPower = -100000;   // exponent of zero
__device__ __forceinline__ Power power(float c, int down) {
  const uint32_t b = __float_as_uint(c);
  if ((b & 0x7fffffffu) == 0) return Power{0.f, kNoPower};
  if (not_finite(fabsf(c))) return Power{c, -down};
  return Power{__uint_as_float((b & 0x807fffffu) | 0x3f800000u), (int)((b >> 23) & 0xff) - 127 - down};
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
template <int R>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

// What a CTA walks in one go: a segment of a head for one walk and 64 columns of its v.  One thread works the
// items out; the others read what they need from shared memory, where it costs them no registers.
struct Item {
  const float* src[3];       // k, v (from the first column), q
  float* o;
  const float* s_from;       // state before the first step, after the last; nullable
  float* s_to;
  int64_t from_row, from_col, to_row, to_col;
  int nc, t0;                // chunks (0: no more items), first step
  int head, e0, ne, Dk;
  int wi, reverse, after;
  int any_poison;
  int poison[64];            // first spoilt step of each column
  int kappa;
  float pw[32 + kL + 1];     // c^n = r^n 2^(kappa n) at 32 + n; zeros before it are the causal mask
};
constexpr int kItems = 4;    // in the works

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
  __shared__ __align__(16) int col_s[kL];                           // of a column of P
  __shared__ int m_s[4][kL], qe_s[4][kL], mw_s[4];
  __shared__ float scan_s[4];
  __shared__ int kmax_s[2][4];
  __shared__ Item items_s[kItems];
  __shared__ __align__(16) float scale_s[2][64];
  __shared__ float top_s[kL];
  __shared__ int dead_s;
  __shared__ uint32_t tmem_s;
  __shared__ __align__(8) uint64_t bars[42];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, role = tid >> 7, th = tid & 127, tw = warp & 3;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t sbase = base + S_::s_at;
  volatile int* dead = &dead_s;
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  // by stage or chunk parity: two each
  const uint32_t bar_k = bar(0), bar_v = bar(2), bar_free = bar(4), bar_kx = bar(6), bar_kraw = bar(8), bar_vraw = bar(10),
                 bar_q = bar(12), bar_qfree = bar(14);
  const uint32_t bar_sp = bar(16), bar_p = bar(17), bar_ds = bar(18), bar_s = bar(19), bar_o = bar(20), bar_ofree = bar(21),
                 bar_qraw = bar(22), bar_qread = bar(23), bar_end = bar(24), bar_dsfree = bar(25);
  const uint32_t bar_kfree = bar(26), bar_vw = bar(28);
  const uint32_t bar_item = bar(30), bar_itemfree = bar(34), bar_powers = bar(38);   // kItems each

  // Every role goes through the CTA's items, and through the chunks of each; barriers and slots follow the
  // chunk count over all of them (g), so the next item is loaded and converted under the end of the last.
  const int T = (int)args.w[0].T;
  const bool boxes = args.boxes != 0;
  // the n-th item, once it is there; null when there are no more
  auto item_at = [&](int n) -> Item* {
    Item* item = &items_s[n % kItems];
    if (!wait_phase(bar_item + 8 * (n % kItems), (uint32_t)(n / kItems) & 1u, dead) || *dead) return nullptr;
    return *(volatile int*)&item->nc ? item : nullptr;
  };
  // the same for a warpgroup, with or without the powers: all of it goes on, or none
  auto group_item = [&](int n, bool powers) -> Item* {
    Item* item = item_at(n);
    if (item && powers) wait_phase(bar_powers + 8 * (n % kItems), (uint32_t)(n / kItems) & 1u, dead);
    return bar_any(7 + role, 128, item == nullptr) ? nullptr : item;
  };

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
    for (int i = 0; i < kItems; ++i) {
      mbar_init(bar_item + 8 * i, 1);
      mbar_init(bar_powers + 8 * i, 32);
      mbar_init(bar_itemfree + 8 * i, 128);
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
  }
  if (tid < 32 * kItems) items_s[tid >> 5].pw[tid & 31] = 0.f;
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
    regs_inc<Regs::load>();
    const int j = th;
    const bool is_k = role == 0, is_v = role == 1, is_q = role == 2;
    // Passes over an operand.  Dk > 64 needs the largest magnitude of both halves before either is converted:
    // k's raw tiles are looked through first; otherwise the first half is loaded, the second, which is
    // converted while it is there, and the first again.  v: weighted, and as it is.
    const bool ahead = KT == 2 && is_k && boxes;
    const int passes = is_v ? (FULL ? 2 : 1) : (KT == 1 ? 1 : (ahead ? 2 : 3));
    const int mid = is_v || ahead ? 0 : KT - 1;  // the pass after whose load the exponent is known
    int g = 0;
#pragma unroll 1
    for (int n = 0; FULL || !is_q; ++n) {
    Item* const item = group_item(n, is_v);
    if (!item) break;
    int t0 = item->t0;
#pragma unroll 1
    for (int left = item->nc; left > 0; --left, t0 += kL, ++g) {
      const uint32_t slot = base + (is_k ? (uint32_t)(g % NS) * S_::k_bytes
                                         : (is_v ? S_::v_at + (uint32_t)(g % NS) * S_::v_bytes : S_::q_at));
      const int t = t0 + j;
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
            const uint32_t raw_at = slot + (uint32_t)(item->reverse ? kL - 1 - j : j) * 4;
            if (is_q) {
              wait_phase(bar_qraw, (uint32_t)(KT == 1 ? g : 3 * g + pass) & 1u, dead);
            } else if (pass == 0) {
              wait_phase((is_k ? bar_kraw : bar_vraw) + 8 * (g % NS), (uint32_t)(g / NS) & 1u, dead);
              if (ahead) top = top64_shared(raw_at + 2 * kTileB, top);
            }
            load64_shared(x, raw_at + (is_k ? (uint32_t)half * 2 * kTileB : 0u));
            if (is_q) mbar_arrive(bar_qread);
            else bar_sync(3 + role, 128);
          } else {
            const float* at = item->src[role] + (item->reverse ? T - 1 - t : t) + (int64_t)half * 64 * T;
            const int rows = (is_v ? item->ne : item->Dk) - half * 64;
            load64(x, at, T, rows, t < T, t0 + kL <= T);
          }
        }
        if (pass <= mid) top = top64(x, top);
        if (pass == mid) {
          const bool bad = not_finite(top);
          if (is_k) {
            if (bad) {                           // every column of the output is spoilt from this step on
              for (int e = 0; e < 64; ++e) atomicMin(&item->poison[e], t);
              item->any_poison = 1;
              zero = true;
            }
            const int f = fit_exponent(bad ? 0.f : top);
            scale = p2(-f);
            if (!boxes && g >= NS) wait_phase(bar_kfree + 8 * (g % NS), (uint32_t)(g / NS - 1) & 1u, dead);
            f_s[g & 1][j] = bad ? kNoTerm - 1 : (top > 0.f ? f : kNoTerm);
            mbar_arrive(bar_kx + 8 * (g & 1));
          } else if (is_q) {
            zero = bad;
            const int qe = bad ? 0 : fit_exponent(top);
            scale = p2(-qe);
            if (g >= S_::nq)
              wait_phase(bar_qfree + 8 * ((g - S_::nq) & 1), (uint32_t)((g - S_::nq) >> 1) & 1u, dead);
            tc_fence_after();
            qe_s[g & 3][j] = bad ? 0x7fffffff : qe;
          } else {
            // v, and what P and the growth need to know of the steps
            wait_phase(bar_kx + 8 * (g & 1), (uint32_t)(g >> 1) & 1u, dead);
            const int f = f_s[g & 1][j];
            zero = f == kNoTerm - 1;
            if (bad && !zero) {                  // single columns are spoilt; the rest of the vector counts
              const float* at = item->src[1] + (item->reverse ? T - 1 - t : t);
              for (int e = 0; e < item->ne; ++e)
                if (not_finite(fabsf(at[(int64_t)e * T]))) atomicMin(&item->poison[e], t);
              item->any_poison = 1;
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
            const int vg = fit_exponent(top);
            const int fg = (top > 0.f && f > kNoTerm) ? f + vg : kNoTerm;
            // weight of the step in the state, and the largest exponent of the weighted steps
            const int lag = min(kL, T - t0) - item->after - j;
            const Power wt = power(t < T ? item->pw[32 + lag] : 0.f, item->kappa * lag);
            const int key = wt.e != kNoPower && fg != kNoTerm ? fg + wt.e : kNoTerm;
            const int kmax = __reduce_max_sync(0xffffffffu, key);
            if (lane == 0) kmax_s[g & 1][tw] = kmax;
            bar_sync(1, 128);
            const int mw = max(max(kmax_s[g & 1][0], kmax_s[g & 1][1]), max(kmax_s[g & 1][2], kmax_s[g & 1][3]));
            if (!boxes && g >= NS) wait_phase(bar_free + 8 * (g % NS), (uint32_t)(g / NS - 1) & 1u, dead);
            if (FULL) fg_s[g & 1][j] = fg;
            if (j == 0) mw_s[g & 3] = mw;
            scale = p2(-vg);
            // 2^-g r^(..) 2^(fg - mw): the powers of two together.  What this takes below a float's range is
            // nothing in fp16 either.
            scale_w = key != kNoTerm ? wt.m * p2(max(key - mw, -100)) * scale : 0.f;
          }
        }
        if (pass < mid) continue;
        if (__any_sync(0xffffffffu, zero)) {
          if (zero) {
#pragma unroll
            for (int d = 0; d < 32; ++d) x[d] = 0;
          }
        }
        // the weighted rows first, the growth waits for them (when it was changed, 148 heads of 2048 steps: 101 to
        // 99 us, with 128 channels 318 to 298)
        const bool weighted = is_v && pass == 0;
        const float by = weighted ? scale_w : scale;
        const uint64_t sc = pair(by, by);
        if (is_q) {
          // 16 channels of q (one step of an MMA) are 8 columns of hi and 8 of lo, side by side: one store
#pragma unroll
          for (int b = 0; b < 32; b += 8) {
            uint32_t r[16];
#pragma unroll
            for (int e = 0; e < 8; ++e) split2(mul2(x[b + e], sc), &r[e], &r[8 + e]);
            tmem_st16(trow + S_::q + (uint32_t)(g % S_::nq) * 64 + half * 64 + 2 * b, r);
          }
          if constexpr (KT == 1) break;          // (x is not carried on)
          continue;
        }
        // one row of a hi and a lo tile (128-byte swizzle)
        if (weighted && g >= 1) wait_phase(bar_ds, (uint32_t)(g - 1) & 1u, dead);    // read by the growth before
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
          mbar_arrive((is_k ? bar_k : (weighted ? bar_vw : bar_v)) + 8 * (g % NS));
        }
      }
      if (is_q) {
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar_q + 8 * (g & 1));
      }
    }
    }
  } else if (role == 3) {
    // ---------------- scores -> P: thread = row i ----------------
    regs_dec<Regs::p>();
    if constexpr (FULL) {
      const int l = th;
      int g = 0;
#pragma unroll 1
      for (int n = 0;; ++n) {
      const Item* const item = group_item(n, true);
      if (!item) break;
      const int kappa = item->kappa;
      // log2 r, for exponents only; a head that forgets everything at once gets a slope that is steeper than any
      // two steps lie apart
      const float slope = fminf(fmaxf(log2f(fabsf(item->pw[33])) - (float)kappa, -1000.f), 250.f);
#pragma unroll 1
      for (int left = item->nc; left > 0; --left, ++g) {
        const uint32_t sp = trow + S_::sp;
        wait_phase(bar_vw + 8 * (g % NS), (uint32_t)(g / NS) & 1u, dead);     // the steps' exponents
        // running maximum of fg_j + (i - j) log2 r: the scan runs on that less i log2 r
        const int fg = fg_s[g & 1][l];
        float mk = fg == kNoTerm ? -1e30f : (float)fg - (float)l * slope;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float up = __shfl_up_sync(0xffffffffu, mk, o);
          if (lane >= o) mk = fmaxf(mk, up);
        }
        if (lane == 31) scan_s[tw] = mk;
        bar_sync(6, 128);
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (i < tw) mk = fmaxf(mk, scan_s[i]);
        const int m = max(kNoTerm, (int)floorf(fmaxf(mk + (float)l * slope, (float)kNoTerm)) + 1);
        m_s[g & 3][l] = m;
        col_s[l] = fg + kappa * l;
        bar_sync(6, 128);
        wait_phase(bar_sp, (uint32_t)g & 1u, dead);
        tc_fence_after();
        // |q_i . k_j| <= 2^score of the scaled vectors: P is held as its multiple of 2^(m + score - 15).  The
        // exponents of a column and a row meet as whole numbers: as two factors, each relative to a third number,
        // both would have to be floats, and steps of a chunk lie further apart than a float's range.  By the choice
        // of m and with c^n above 2^-64 their difference is below 64; what lies 127 below one is nothing in fp16.
        const int above = 127 - (m + (S_::score - 15) + kappa * l);
        const float* pw = &item->pw[32 + l];      // c^(i - j), zero for j > i: the mask
        const int* col = col_s;
        auto scaled = [above](uint64_t x, int f0, int f1) {
          return mul2(x, pair(__int_as_float(__viaddmin_s32_relu(f0, above, 254) << 23),
                              __int_as_float(__viaddmin_s32_relu(f1, above, 254) << 23)));
        };
#pragma unroll 1
        for (int b = 0; b < 128; b += 32, pw -= 32, col += 32) {
          uint32_t s[32];                        // 16 columns of hi and 16 of lo, in the place of 32 scores
          if (b <= tw * 32) {
            uint32_t r[32];
            tmem_ld32(sp + b, r);
            tmem_ld_wait();
#pragma unroll
            for (int jj = 0; jj < 32; jj += 4) {
              const int4 cf = *reinterpret_cast<const int4*>(col + jj);
              // the power first: its zeros take whatever the steps after i hold
              const uint64_t x = mul2(pair(__uint_as_float(r[jj]), __uint_as_float(r[jj + 1])), pair(pw[-jj], pw[-jj - 1]));
              const uint64_t y = mul2(pair(__uint_as_float(r[jj + 2]), __uint_as_float(r[jj + 3])), pair(pw[-jj - 2], pw[-jj - 3]));
              split2(scaled(x, cf.x, cf.y), &s[jj / 2], &s[16 + jj / 2]);
              split2(scaled(y, cf.z, cf.w), &s[jj / 2 + 1], &s[17 + jj / 2]);
            }
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) s[x] = 0u;
          }
          tmem_st32(sp + b, s);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar_p);
      }
      }
    }
  } else if (role == 4) {
    // ---------------- state (thread = column e, half of Dk) and output (thread = step i) ----------------
    regs_inc<Regs::s>();
    const int l = th, e = l & 63, half = l >> 6;
    constexpr int NSt = 32 * KT;                 // state elements per thread: d = half * NSt ...
    float St[NSt];
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
    // The output of a chunk is written one chunk later, whichever item that belongs to: what it needs is kept.
    int out_g = -1, out_n = 0, out_t0 = 0;
    auto write_output = [&](bool last) {
        const Item& item = items_s[out_n % kItems];
        const int out_t = out_t0 + l;
        wait_phase(bar_o, (uint32_t)out_g & 1u, dead);
        tc_fence_after();
        const int qe = qe_s[out_g & 3][l], m = m_s[out_g & 3][l] + S_::score - 15;
        const bool bad = qe == 0x7fffffff;
        const Factors fi = p2_wide((bad ? 0 : qe) + m);
        // the state's part: times the row's exponent and power before the column's exponent where that takes it
        // down and after it where that takes it up, so that nothing leaves a float's range that comes back into it
        const int lag = l + item.after;
        const Power rp = power(item.pw[32 + lag], item.kappa * lag);
        const int rx_e = (bad ? 0 : qe) + rp.e, first = max(min(rx_e, 0), -126);
        const float nan = __int_as_float(0x7fffffff), rowa = rp.m * p2(first), rowb = p2_low(min(rx_e - first, 127));
        const uint64_t ia = pair(bad ? nan : fi.a, bad ? nan : fi.a), ib = pair(fi.b, fi.b), xa = pair(rowa, rowa),
                       xb = pair(rowb, rowb);
        const int ne = item.ne;
        const bool plain = out_t0 + kL <= T && ne == 64;
        const int live = out_t < T ? ne : 0;
        float* out = item.o + (item.reverse ? T - 1 - out_t : out_t);
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
          const float* sc = &scale_s[out_g & 1][b];
          float y[16];
#pragma unroll
          for (int x = 0; x < 16; x += 2) {
            const uint64_t inter = mul2(mul2(mul2(pair(__uint_as_float(rx[x]), __uint_as_float(rx[x + 1])), xa),
                                             pair(sc[x], sc[x + 1])), xb);
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
              if (b + x < live) *out = y[x];
              out += T;
            }
          }
        }
        if (*(const volatile int*)&item.any_poison != 0 && live > 0) {          // spoilt columns
          out -= (int64_t)64 * T;
          for (int x = 0; x < ne; ++x)
            if (item.poison[x] <= out_t) out[(int64_t)x * T] = nan;
        }
        if (last) mbar_arrive(bar_itemfree + 8 * (out_n % kItems));
    };
    int g = 0;
#pragma unroll 1
    for (int n = 0;; ++n) {
      const Item* const item = group_item(n, true);
      if (!item) break;
      {
      const float* src = item->s_from;
      const int64_t rs = item->from_row, cs = item->from_col;
#pragma unroll
      for (int i = 0; i < NSt; ++i) {
        const int d = half * NSt + i;
        St[i] = (src && d < item->Dk && e < item->ne) ? src[d * rs + (int64_t)e * cs] : 0.f;
      }
      }
      if (FULL) {
        // the published state is replaced once the MMAs of the chunk have read it
        if (g >= 1) wait_phase(bar_qfree + 8 * ((g - 1) & 1), (uint32_t)((g - 1) >> 1) & 1u, dead);
        publish(g & 1);
        mbar_arrive(bar_s);
      }
      int t0 = item->t0;
#pragma unroll 1
      for (int left = item->nc; left > 0; --left, t0 += kL, ++g) {
        if (FULL && out_g >= 0) write_output(out_n != n);
        // the state after the chunk
        const int steps = min(kL, T - t0);
        const Power carry = power(item->pw[32 + steps], item->kappa * steps);
        const float carried = carry.m * p2(max(-126, min(carry.e, 126)));
        if (carry.e < -126) {                    // what of the power is below a float
          const float rest = p2_low(carry.e + 126);
#pragma unroll
          for (int i = 0; i < NSt; ++i) St[i] *= rest;
        }
        wait_phase(bar_ds, (uint32_t)g & 1u, dead);
        tc_fence_after();
        const Factors mw = p2_wide(mw_s[g & 3]);
        const uint64_t ma = pair(mw.a, mw.a), mb = pair(mw.b, mw.b), cy = pair(carried, carried);
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
        if (FULL) {
          out_g = g;
          out_n = n;
          out_t0 = t0;
          if (left > 1) {
            wait_phase(bar_qfree + 8 * (g & 1), (uint32_t)(g >> 1) & 1u, dead);
            publish((g + 1) & 1);
            mbar_arrive(bar_s);
          }
        }
      }
      // the state after the last chunk
      float* dst = item->s_to;
      if (dst && e < item->ne) {
        const int64_t rs = item->to_row, cs = item->to_col;
        const bool bad = item->poison[e] != 0x7fffffff;
#pragma unroll
        for (int i = 0; i < NSt; ++i) {
          const int d = half * NSt + i;
          if (d < item->Dk) dst[d * rs + (int64_t)e * cs] = bad ? __int_as_float(0x7fffffff) : St[i];
        }
      }
      if (!FULL) mbar_arrive(bar_itemfree + 8 * (n % kItems));
    }
    if (FULL && out_g >= 0) write_output(false);
  } else {
    regs_dec<Regs::mma>();
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
      const Item* item = item_at(0);
      if (FULL && item) scores(0);
      // Growth first, it waits for nothing but the state's warps; then the state's part of the output, for
      // which the output before has to be taken away, the read-out, and the next chunk's scores.
      int c = 0;
#pragma unroll 1
      for (int n = 0; item && ok; ++n) {
      const int end = c + *(const volatile int*)&item->nc;
#pragma unroll 1
      for (; c < end && ok; ++c) {
        if (c + 1 == end) item = item_at(n + 1);
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
        if (item) scores(c + 1);
      }
      }
      umma_commit(bar_end);          // everything issued has landed before tensor memory is given back
      if (!mbar_wait(bar_end, 0)) *dead = 1;
    } else if (th == 32 && boxes) {
      // ---------------- raw k and v, a TMA box for 64 channels ----------------
      int k_issued = 0, v_issued = 0;
#pragma unroll 1
      for (int n = 0; !*dead; ++n) {
        const Item* const item = item_at(n);
        if (!item) break;
        const CUtensorMap* maps = args.map[item->wi];
        const int head = item->head, e0 = item->e0;
        int t = item->t0;
#pragma unroll 1
        for (int left = item->nc; left > 0; --left, t += kL) {
          const int g = v_issued;
          const int from = item->reverse ? T - t - kL : t;       // walking back, the last box may start before 0
          const uint32_t bk = bar_kraw + 8 * (g % NS), bv = bar_vraw + 8 * (g % NS), again = (uint32_t)(g / NS - 1) & 1u;
          if (g >= NS) wait_phase(bar_kfree + 8 * (g % NS), again, dead);
          if (*dead) break;
          mbar_expect_tx(bk, S_::k_bytes);
          for (int h = 0; h < KT; ++h)
            tma_load_box(base + (uint32_t)(g % NS) * S_::k_bytes + h * 2 * kTileB, &maps[1], from, 64 * h, head, bk);
          k_issued = g + 1;
          if (g >= NS) wait_phase(bar_free + 8 * (g % NS), again, dead);
          if (*dead) break;
          mbar_expect_tx(bv, S_::v_bytes);
          tma_load_box(base + S_::v_at + (uint32_t)(g % NS) * S_::v_bytes, &maps[2], from, e0, head, bv);
          v_issued = g + 1;
        }
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
      for (int i = 0; !*dead; ++i) {
        const Item* const item = item_at(i);
        if (!item) break;
        const CUtensorMap* map = &args.map[item->wi][0];
        const int head = item->head, reverse = item->reverse, steps = per * item->nc, t0 = item->t0;
#pragma unroll 1
        for (int x = 0; x < steps; ++x) {
          const int t = t0 + x / per * kL;
          if (n >= 1) wait_phase(bar_qread, (uint32_t)(n - 1) & 1u, dead);
          if (*dead) break;
          mbar_expect_tx(bar_qraw, 2 * kTileB);
          tma_load_box(base + S_::q_at, map, reverse ? T - t - kL : t, x % per == 1 ? 64 : 0, head, bar_qraw);
          ++n;
        }
      }
      if (*dead && n > 0) mbar_wait(bar_qraw, (uint32_t)(n - 1) & 1u);
    } else if (tw == 3) {
      // ---------------- items, ahead of the others ----------------
      uint32_t it = blockIdx.x;
#pragma unroll 1
      for (int n = 0;; ++n, it += gridDim.x) {
        Item* const item = &items_s[n % kItems];
        const uint32_t full = bar_item + 8 * (n % kItems);
        if (n >= kItems) wait_phase(bar_itemfree + 8 * (n % kItems), (uint32_t)(n / kItems - 1) & 1u, dead);
        if (__any_sync(0xffffffffu, *dead != 0)) break;          // the others may still be in the items that are there
        if (it >= (uint32_t)args.items) {
          if (lane == 0) {
            *(volatile int*)&item->nc = 0;
            mbar_arrive(full);
          }
          break;
        }
        const int sub = (int)(it % (uint32_t)args.nsub), wi = args.sub_walk[sub], e0 = args.sub_e0[sub];
        const Walk& w = args.w[wi];
        const uint32_t rest = it / (uint32_t)args.nsub;
        const int64_t head = rest % (uint32_t)args.heads, state = head * (int64_t)w.Dk * w.Dv;
        const int seg = (int)(rest / (uint32_t)args.heads);
        item->poison[lane] = item->poison[32 + lane] = 0x7fffffff;
        __syncwarp();
        if (lane == 0) {
          item->src[0] = w.k + head * (int64_t)w.Dk * T;
          item->src[1] = w.v + (head * (int64_t)w.Dv + e0) * T;
          item->src[2] = w.q + head * (int64_t)w.Dk * T;
          if (FULL) item->o = w.o + (head * (int64_t)w.Dv + e0) * T;
          const int64_t between = args.heads * (int64_t)w.Dk * w.Dv;       // of args.seg, rows of Dv
          item->s_from = item->s_to = nullptr;
          item->from_row = item->to_row = w.s_row;
          item->from_col = item->to_col = w.s_col;
          if (seg == 0) {
            if (w.s_in) item->s_from = w.s_in + state + e0 * w.s_col;
          } else if (FULL) {
            item->s_from = args.seg[wi] + (seg - 1) * between + state + e0;
            item->from_row = w.Dv;
            item->from_col = 1;
          }
          if (!FULL) {
            item->s_to = args.seg[wi] + seg * between + state + e0;
            item->to_row = w.Dv;
            item->to_col = 1;
          } else if (seg == args.nseg - 1 && w.s_out) {
            item->s_to = w.s_out + state + e0 * w.s_col;
          }
          item->nc = min(args.seg_chunks, (T + kL - 1) / kL - seg * args.seg_chunks);
          item->t0 = seg * args.seg_chunks * kL;
          item->head = (int)head;
          item->e0 = e0;
          item->ne = min(64, w.Dv - e0);
          item->Dk = w.Dk;
          item->wi = wi;
          item->reverse = w.reverse;
          item->after = w.after;
          item->any_poison = 0;
          mbar_arrive(full);
        }
        // c^n by squaring in 64 bits: r itself does not fit 32 (a slow head multiplies it a thousandfold)
        const double r = 1.0 - (double)w.decay[w.n_decay > 1 ? (w.head0 + head) % w.n_decay : 0] / 4096.0;
        const int kappa = r != 0.0 ? max(-128, min(__float2int_rn(-log2f(fabsf((float)r))), 128)) : 0;
        double b = r * __hiloint2double((1023 + kappa) << 20, 0), p = 1.0;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1, b *= b)
          if (lane & m) p *= b;
        if (lane == 0) item->kappa = kappa;
#pragma unroll
        for (int i = 32; i <= 32 + kL; i += 32, p *= b)          // b: c^32
          if (i + lane <= 32 + kL) item->pw[i + lane] = (float)p;
        mbar_arrive(bar_powers + 8 * (n % kItems));
      }
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
      double b = 1.0 - (double)w.decay[w.n_decay > 1 ? (w.head0 + head) % w.n_decay : 0] / 4096.0, p = 1.0;
      for (int64_t n = (int64_t)args.seg_chunks * kL; n; n >>= 1) {
        if (n & 1) p *= b;
        b *= b;
      }
      float* s = args.seg[wi] + i;
      float x = *s;
      for (int g = 1; g < args.nseg - 1; ++g) {
        s += total;
        x = (float)fma(p, (double)x, (double)*s);     // the power may be less than any float
        *s = x;
      }
    }
  }
}

}  // namespace

// Segments the axis is cut into, each of them `ctas` items of one CTA.  In chunks: a CTA takes its share of
// the items one after the other, each 0.8 longer than its chunks, and 1.6 to fill and drain; a cut axis is
// walked by a first launch too, at half the cost of a chunk, and the join and the launches take 2, and a
// twentieth for each segment.  Measured, us,
// whole against cut in four: 16 heads of 128 channels and 8 chunks 65 and 47, 4 chunks 36 and 35 (the rule leaves
// them whole); 35 heads of 64 and 8 chunks 43 and 35, 70 heads 43 and 55.
struct Cut {
  int nseg;
  double cost;
};
static Cut plan_segments(int64_t ctas, int64_t chunks) {
  const int64_t sms = sm_count();
  Cut best{1, 0};
  for (int64_t n = 1; n <= chunks && n <= 256; ++n) {
    const int64_t per = (chunks + n - 1) / n;
    if ((chunks + per - 1) / per != n) continue;       // the same cut as a smaller n
    double cost = (double)((ctas * n + sms - 1) / sms) * ((double)per + 0.8) + 1.6;
    if (n > 1) cost += (double)((ctas * (n - 1) + sms - 1) / sms) * (0.5 * (double)per + 0.8) + 3.6 + 0.05 * (double)n;
    if (n == 1 || cost < best.cost) best = Cut{(int)n, cost};
    if (ctas * n > 16 * sms) break;
  }
  return best;
}

// Heads that are walked whole by a launch of their own before the others, whose axis is cut, by the same costs:
// as many as fill the SMs evenly.  Measured, us, together against apart (and the ratio of the costs): 180 heads of
// 64 channels and 4096 steps 343 and 268 (0.79), 100 heads of 128 channels and 4096 steps 553 and 495 (0.97), the
// training step of 32 heads of 128 channels and 4096 steps 774 and 692 (0.86), of 256 heads of 64 channels and 2000
// steps 712 and 699 (0.96).
static int64_t whole_heads(int64_t heads, int64_t nsub, int64_t chunks) {
  const int64_t rounds = heads * nsub / sm_count(), first = rounds * sm_count() / nsub;
  if (rounds == 0 || first == heads) return 0;
  const double apart = (double)rounds * ((double)chunks + 0.8) + 1.6 + plan_segments((heads - first) * nsub, chunks).cost;
  return apart < 0.98 * plan_segments(heads * nsub, chunks).cost ? first : 0;
}

int64_t tc_scratch_floats(const Walk* walks, int n) {
  int64_t nsub = 0, floats = 0;
  for (int i = 0; i < n; ++i) nsub += (walks[i].Dv + 63) / 64;
  const int64_t chunks = (walks[0].T + kL - 1) / kL, heads = walks[0].heads - whole_heads(walks[0].heads, nsub, chunks);
  const int nseg = plan_segments(heads * nsub, chunks).nseg;
  if (nseg > 1)
    for (int i = 0; i < n; ++i) floats += (int64_t)(nseg - 1) * heads * walks[i].Dk * walks[i].Dv;
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
    TcArgs b = a;
    b.items = ctas * (a.nseg - 1);
    attention_tc_kernel<KT, false><<<(unsigned)(b.items < sm_count() ? b.items : sm_count()), kThreads, smem, s>>>(b);
    SB_CUDA(cudaGetLastError());
  }
  return SB_OK;
}

// heads [from, from + heads) of the walks, their axis in nseg segments
static int part(const Walk* walks, int n, int64_t from, int64_t heads, int nseg, float* scratch, cudaStream_t s) {
  TcArgs a;
  memset(&a, 0, sizeof(a));
  a.nsub = 0;
  for (int i = 0; i < n; ++i) {
    Walk& w = a.w[i];
    w = walks[i];
    const int64_t k = from * w.Dk * w.T, v = from * w.Dv * w.T, state = from * w.Dk * w.Dv;
    w.heads = heads;
    w.head0 += from;
    w.q += k;
    w.k += k;
    w.v += v;
    w.o += v;
    if (w.s_in) w.s_in += state;
    if (w.s_out) w.s_out += state;
    for (int e0 = 0; e0 < w.Dv; e0 += 64) {
      a.sub_walk[a.nsub] = i;
      a.sub_e0[a.nsub++] = e0;
    }
  }
  a.heads = heads;
  const int64_t ctas = a.heads * a.nsub, chunks = (walks[0].T + kL - 1) / kL;
  a.nseg = nseg;
  a.seg_chunks = (int)((chunks + a.nseg - 1) / a.nseg);
  if (a.nseg > 1) {
    float* p = scratch;
    for (int i = 0; i < n; ++i) {
      a.seg[i] = p;
      p += (int64_t)(a.nseg - 1) * a.heads * walks[i].Dk * walks[i].Dv;
    }
  }
  uintptr_t bits = 0;
  for (int i = 0; i < n; ++i) bits |= (uintptr_t)a.w[i].q | (uintptr_t)a.w[i].k | (uintptr_t)a.w[i].v;
  a.boxes = (bits & 15u) == 0 && walks[0].T % 4 == 0;
  for (int i = 0; i < n && a.boxes; ++i) {
    const Walk& w = a.w[i];
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
  a.items = ctas * a.nseg;
  const unsigned grid = (unsigned)(a.items < sm_count() ? a.items : sm_count());
  if (wide) attention_tc_kernel<2, true><<<grid, kThreads, Shape<2>::smem, s>>>(a);
  else attention_tc_kernel<1, true><<<grid, kThreads, Shape<1>::smem, s>>>(a);
  SB_CUDA(cudaGetLastError());
  return SB_OK;
}

// Walks of one launch: the same heads and T, Dk on the same side of 64.
int tc_walks(const Walk* walks, int n, float* scratch, cudaStream_t s) {
  int64_t nsub = 0;
  for (int i = 0; i < n; ++i) nsub += (walks[i].Dv + 63) / 64;
  const int64_t chunks = (walks[0].T + kL - 1) / kL, heads = walks[0].heads, first = whole_heads(heads, nsub, chunks);
  if (first) SB_TRY(part(walks, n, 0, first, 1, nullptr, s));
  return part(walks, n, first, heads - first, plan_segments((heads - first) * nsub, chunks).nseg, scratch, s);
}

}  // namespace la
}  // namespace sb
