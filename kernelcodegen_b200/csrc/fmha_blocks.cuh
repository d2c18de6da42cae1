// The steps that the tensor-core attention kernels share (fmha_tcgen05.cu, fmha_cached.cu), for use inside an anonymous
// namespace that uses kcg::sm100: packed fp32 arithmetic, the online softmax of one block of 128 keys, and the MMA groups
// of the issuing thread.
#pragma once

// Pairs of exponentials whose index has all bits of this mask set are computed on the FMA pipe
// (exp2_pair_fma) instead of the special-function unit: 0 none, 7 one in eight, 3 one in four.
// Measured on B8 H32 D128 (two-tile kernel): one in four gains 2.5 % at S = 1024 and on causal
// S = 2048 and 0.4 % at S = 4096, one in eight about half of that; accuracy is unchanged (2.3e-3).
#ifndef KCG_FMHA_EMU_MASK
#define KCG_FMHA_EMU_MASK 3
#endif

constexpr int BN = 128;          // keys per block
constexpr float kRescaleThreshold = 8.0f;  // in log2 units: rescale O only when the max grew by > 2^8

__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}


// ---- packed fp32x2 arithmetic (two lanes of fp32 in one 64-bit register) --------------------
// sm_100 executes fma / add on fp32 pairs in one instruction, which halves the FMA-pipe
// instruction count of the softmax.
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x for a pair of values on the FMA and integer pipes instead of the special-function unit:
// n = round(x) by the magic-number addition, f = x - n in [-0.5, 0.5], 2^f by a cubic (relative
// error 1.1e-4, far below the rounding of a 16-bit P), and n added into the exponent field.
// Arguments below -126 (masked scores are -inf) give exactly 0, like the flushing ex2.approx.ftz.
__device__ __forceinline__ void exp2_pair_fma(uint64_t x2, float& p0, float& p1) {
  float x0, x1;
  f2_unpack(x2, x0, x1);
  const uint64_t xc = x2;
  const uint64_t magic = f2_pack(12582912.f, 12582912.f), nmagic = f2_pack(-12582912.f, -12582912.f);
  const uint64_t t = f2_add(xc, magic);                 // low mantissa bits = n
  const uint64_t n = f2_add(t, nmagic);                 // n as a float
  const uint64_t fr = f2_fma(n, f2_pack(-1.f, -1.f), xc);
  uint64_t p = f2_fma(fr, f2_pack(0.0555054f, 0.0555054f), f2_pack(0.2402265f, 0.2402265f));
  p = f2_fma(p, fr, f2_pack(0.6931472f, 0.6931472f));
  p = f2_fma(p, fr, f2_pack(1.0f, 1.0f));
  float t0, t1, q0, q1;
  f2_unpack(t, t0, t1);
  f2_unpack(p, q0, q1);
  p0 = x0 < -126.f ? 0.f : __uint_as_float(__float_as_uint(q0) + (__float_as_uint(t0) << 23));
  p1 = x1 < -126.f ? 0.f : __uint_as_float(__float_as_uint(q1) + (__float_as_uint(t1) << 23));
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

// One key block of the online softmax for the calling thread's query row.  The 128 scores of the
// row sit in tensor memory at s_addr (this thread's lane); columns >= limit are masked.  On return
// P (16-bit, 64 columns) has replaced the first half of the scores, handed to the MMA thread in
// two halves through arrive(half) (called by lane 0 after the warp's stores are complete), the
// output accumulator at o_addr has been rescaled if the running maximum m moved by more than the
// threshold, and m and the running row sum l are up to date.  All 32 lanes of the warp call it.
struct NoHook {
  __device__ __forceinline__ bool operator()() const { return true; }
};

// Two optional hooks serve the kernel whose warpgroups take alternate key blocks of one tile:
// decided() is called (by all lanes) as soon as this block's value of m is final — before the
// exponentials on the ordinary path — and wait_o() before the accumulator is touched for a rescale
// (it returns false if its wait timed out; the rescale is then skipped and the caller gives up).
// kEmuMask: which pairs of exponentials take the FMA pipe (0 where a NaN score must stay one); kThreshold: the growth of
// the maximum, in log2 units, that O is not rescaled for.  kWide: the maximum may be so large that m + kThreshold is rounded up.
template <typename T, int D, int kEmuMask = KCG_FMHA_EMU_MASK, int kThreshold = static_cast<int>(kRescaleThreshold), bool kWide = false,
          typename Arrive, typename Decided = NoHook, typename WaitO = NoHook>
__device__ __forceinline__ bool softmax_block(uint32_t s_addr, uint32_t o_addr, int j, int limit, float c, float& m,
                                              float& l, int lane, Arrive arrive, Decided decided = Decided(),
                                              WaitO wait_o = WaitO()) {
  bool hooks_ok = true;
  auto outgrown = [](float top, float old) {
    return kWide ? top - old > static_cast<float>(kThreshold) : top > old + static_cast<float>(kThreshold);
  };
  uint32_t sreg[BN];
  tmem_ld64(s_addr, reinterpret_cast<uint32_t(&)[64]>(sreg[0]));
  tmem_ld64(s_addr + 64, reinterpret_cast<uint32_t(&)[64]>(sreg[64]));
  tmem_wait_ld();
  if (limit < BN) {
#pragma unroll
    for (int k = 0; k < BN; ++k)
      if (k >= limit) sreg[k] = 0xff800000u;  // -inf
  }
  // eight independent chains of 3-input max (8 dependent steps instead of 16)
  float mx[8];
#pragma unroll
  for (int a = 0; a < 8; ++a) mx[a] = fmaxf(__uint_as_float(sreg[2 * a]), __uint_as_float(sreg[2 * a + 1]));
#pragma unroll
  for (int k = 16; k < BN; k += 16) {
#pragma unroll
    for (int a = 0; a < 8; ++a) mx[a] = max3(mx[a], __uint_as_float(sreg[k + 2 * a]), __uint_as_float(sreg[k + 2 * a + 1]));
  }
  const float mt = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * c;
  uint64_t lsum_a = 0ull, lsum_b = 0ull;  // two (+0.f, +0.f) accumulators
  const uint64_t c2 = f2_pack(c, c);
  // exponentials of one half of the row (64 scores -> 32 packed words, written in place over
  // the words already consumed), then the hand-over of that half of P to the MMA thread
  auto exp_half = [&](int half, uint64_t nm2) {
#pragma unroll
    for (int k = half * 64; k < half * 64 + 64; k += 2) {
      const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(sreg[k]), __uint_as_float(sreg[k + 1])), c2, nm2);
      float p0, p1;
      if (kEmuMask != 0 && ((k >> 1) & kEmuMask) == kEmuMask) {
        exp2_pair_fma(x2, p0, p1);
      } else {
        float x0, x1;
        f2_unpack(x2, x0, x1);
        p0 = fast_exp2(x0);
        p1 = fast_exp2(x1);
      }
      if ((k >> 1) & 1) lsum_b = f2_add(lsum_b, f2_pack(p0, p1));
      else lsum_a = f2_add(lsum_a, f2_pack(p0, p1));
      sreg[k >> 1] = pack2<T>(p0, p1);  // in place: word k/2 is never read again
    }
  };
  auto hand_over = [&](int half) {
    tmem_st32(s_addr + half * 32, reinterpret_cast<uint32_t(&)[32]>(sreg[half * 32]));
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) arrive(half);
  };
  float alpha = 1.f;
  bool half0_done = false;
  // Speculative path (every block after the first that needs no mask): the exponentials of the
  // first half start at once with the running maximum m, so that the maximum of this block is
  // computed in the shadow of the special-function unit instead of in front of it.  That is
  // exact whenever the block's maximum stays within the rescale threshold of m, which is the
  // condition under which m would have been kept anyway; otherwise (rare once a few blocks have
  // been seen) the first half is read again from tensor memory and redone on the ordinary path.
  const bool speculate = __all_sync(0xffffffffu, j > 0 && limit >= BN && m != -INFINITY);
  if (speculate) {
    const float neg_m0 = -m;
    exp_half(0, f2_pack(neg_m0, neg_m0));
    if (!__any_sync(0xffffffffu, outgrown(mt, m))) {
      decided();
      hand_over(0);
      half0_done = true;
    } else {
      tmem_ld64(s_addr, reinterpret_cast<uint32_t(&)[64]>(sreg[0]));   // the first 32 words were overwritten
      tmem_wait_ld();
      lsum_a = 0ull;
      lsum_b = 0ull;
    }
  }
  if (!half0_done) {
    bool rescale = false;
    if ((outgrown(mt, m) || m == -INFINITY) && mt > m) {
      alpha = (m == -INFINITY) ? 0.f : fast_exp2(m - mt);
      rescale = (j > 0);
      m = mt;
    }
    // In the two-tile kernels S_i(j) being complete means PV_i(j-1) is complete, so O_i may be
    // rescaled at once; a kernel where that does not hold passes wait_o.
    if (__any_sync(0xffffffffu, rescale)) {
      hooks_ok = wait_o();
      if (hooks_ok) {
        tc_fence_after();
        const float a = rescale ? alpha : 1.f;
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t oreg[32];
          tmem_ld32(o_addr + cc * 32, oreg);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; ++k) oreg[k] = __float_as_uint(__uint_as_float(oreg[k]) * a);
          tmem_st32(o_addr + cc * 32, oreg);
        }
      }
    }
    decided();
    const float neg_m = (m == -INFINITY) ? 0.f : -m;
    exp_half(0, f2_pack(neg_m, neg_m));
    hand_over(0);
  }
  {
    const float neg_m = (m == -INFINITY) ? 0.f : -m;
    exp_half(1, f2_pack(neg_m, neg_m));
    hand_over(1);
  }
  float l0, l1;
  f2_unpack(f2_add(lsum_a, lsum_b), l0, l1);
  l = l * alpha + (l0 + l1);
  return hooks_ok;
}

// ---- MMA groups of the two-tile kernel's issuing thread ------------------------------------
// The issuing thread is one of the kernel's two bottlenecks: an MMA of 128x128x16 takes the thread
// about as long to issue (65-75 clocks) as the tensor pipe needs to run it (68), and a barrier
// test needs ~140 clocks to answer.  Tested on its own in front of a batch of MMAs, every barrier
// would idle the pipe for that long, five times per key block.  So each batch is one asm block
// that first issues a non-blocking test of the barrier(s) needed *after* it, then the MMAs (and
// the commit), and reads the answers last; only a barrier that was not complete yet is waited
// for in the ordinary way.
//
// Four PV k-steps: O (+)= P[:, 16 kk .. 16 kk + 16) V[16 kk .., :], kk = kk0 .. kk0 + 3.  a_p / vd address
// k-step kk0 (P advances 8 tensor-memory columns, the V descriptor 2048 bytes per k-step).
__device__ __forceinline__ bool pv4_peek(uint32_t d_o, uint32_t a_p, uint64_t vd, uint32_t idesc, uint32_t acc_first,
                                         uint32_t peek_bar, uint32_t peek_par) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P, Q, T;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 v1, v2, v3;\n\t"
      "setp.ne.b32 P, %5, 0;\n\t"
      "setp.eq.b32 T, %5, %5;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 Q, [%6], %7;\n\t"
      "add.u32 a1, %2, 8;\n\tadd.u32 a2, %2, 16;\n\tadd.u32 a3, %2, 24;\n\t"
      "add.s64 v1, %3, 128;\n\tadd.s64 v2, %3, 256;\n\tadd.s64 v3, %3, 384;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], %3, %4, P;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], [a1], v1, %4, T;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], [a2], v2, %4, T;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], [a3], v3, %4, T;\n\t"
      "selp.u32 %0, 1, 0, Q;\n\t}"
      : "=r"(ok)
      : "r"(d_o), "r"(a_p), "l"(vd), "r"(idesc), "r"(acc_first), "r"(peek_bar), "r"(peek_par)
      : "memory");
  return ok != 0;
}
// Four PV k-steps (always accumulating), then — if kWithS — the next score tile S = Q K^T (D / 16
// k-steps, the first one overwriting), then the commit on `commit_bar`; two barriers are tested.
// qd / kd: descriptors of k-step 0 (k-steps advance 32 bytes, the second 64-element half of the
// head dimension lies one 16 KB block further).
#define KCG_SS_STEP(OFF, PRED)                                                            \
  "add.s64 qx, %7, " #OFF ";\n\tadd.s64 kx, %8, " #OFF ";\n\t"                             \
  "tcgen05.mma.cta_group::1.kind::f16 [%6], qx, kx, %9, " #PRED ";\n\t"
template <int D, bool kWithS>
__device__ __forceinline__ void pv4_s_commit_peek2(uint32_t d_o, uint32_t a_p, uint64_t vd, uint32_t idesc_pv, uint32_t d_s,
                                                   uint64_t qd, uint64_t kd, uint32_t idesc_qk, uint32_t commit_bar,
                                                   uint32_t peek1, uint32_t par1, uint32_t peek2, uint32_t par2,
                                                   bool& ok1, bool& ok2) {
  uint32_t r1, r2;
#define KCG_PV4                                                                                    \
  "{\n\t.reg .pred F, Q1, Q2, T;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 v1, v2, v3, qx, kx;\n\t"     \
  "setp.eq.b32 T, %2, %2;\n\t"                                                                     \
  "setp.ne.b32 F, %2, %2;\n\t"                                                                     \
  "mbarrier.test_wait.parity.shared::cta.b64 Q1, [%11], %12;\n\t"                                  \
  "mbarrier.test_wait.parity.shared::cta.b64 Q2, [%13], %14;\n\t"                                  \
  "add.u32 a1, %3, 8;\n\tadd.u32 a2, %3, 16;\n\tadd.u32 a3, %3, 24;\n\t"                           \
  "add.s64 v1, %4, 128;\n\tadd.s64 v2, %4, 256;\n\tadd.s64 v3, %4, 384;\n\t"                       \
  "tcgen05.mma.cta_group::1.kind::f16 [%2], [%3], %4, %5, T;\n\t"                                  \
  "tcgen05.mma.cta_group::1.kind::f16 [%2], [a1], v1, %5, T;\n\t"                                  \
  "tcgen05.mma.cta_group::1.kind::f16 [%2], [a2], v2, %5, T;\n\t"                                  \
  "tcgen05.mma.cta_group::1.kind::f16 [%2], [a3], v3, %5, T;\n\t"
#define KCG_TAIL                                                                                   \
  "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%10];\n\t"               \
  "selp.u32 %0, 1, 0, Q1;\n\tselp.u32 %1, 1, 0, Q2;\n\t}"
#define KCG_OPERANDS                                                                               \
  : "=r"(r1), "=r"(r2)                                                                             \
  : "r"(d_o), "r"(a_p), "l"(vd), "r"(idesc_pv), "r"(d_s), "l"(qd), "l"(kd), "r"(idesc_qk),         \
    "r"(commit_bar), "r"(peek1), "r"(par1), "r"(peek2), "r"(par2)                                  \
  : "memory"
  if constexpr (!kWithS) {
    asm volatile(KCG_PV4 KCG_TAIL KCG_OPERANDS);
  } else if constexpr (D == 128) {
    asm volatile(KCG_PV4 KCG_SS_STEP(0, F) KCG_SS_STEP(2, T) KCG_SS_STEP(4, T) KCG_SS_STEP(6, T) KCG_SS_STEP(1024, T)
                     KCG_SS_STEP(1026, T) KCG_SS_STEP(1028, T) KCG_SS_STEP(1030, T) KCG_TAIL KCG_OPERANDS);
  } else {
    asm volatile(KCG_PV4 KCG_SS_STEP(0, F) KCG_SS_STEP(2, T) KCG_SS_STEP(4, T) KCG_SS_STEP(6, T) KCG_TAIL KCG_OPERANDS);
  }
#undef KCG_PV4
#undef KCG_TAIL
#undef KCG_OPERANDS
  ok1 = r1 != 0;
  ok2 = r2 != 0;
}
#undef KCG_SS_STEP
