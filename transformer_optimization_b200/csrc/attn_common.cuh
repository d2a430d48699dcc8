// Device helpers shared by the attention kernels: tile sizes and the register
// split of the tcgen05 kernels, exponentials, three-input maxima, operand
// packing and TMEM stores.
#pragma once

#include "common.cuh"

namespace tfb {

constexpr int kAttnBM = 128;  // query rows per tile
constexpr int kAttnBN = 128;  // keys per block
constexpr int kAttnTiles = 2;
constexpr int kAttnThreads = 384;
constexpr float kRescaleThreshold = 8.0f;
// Register split: the kernel is built at 168 registers/thread (384 threads,
// 64512 per CTA); warpgroup 0 (producers, MMA) drops to 40 and the two
// softmax warpgroups rise to 232: 128*40 + 256*232 = 64512, the launch pool.
constexpr int kRegsLaunch = 168;
constexpr int kRegsLow = 40;
constexpr int kRegsHigh = 232;
static_assert(128 * kRegsLow + 256 * kRegsHigh <= kAttnThreads * kRegsLaunch, "register split exceeds the pool");

// volatile: the exp-unit sweep must stay between the turn wait and arrive
__device__ __forceinline__ float ex2_f32(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float fmax3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ uint32_t pack_f16x2_rn(float a, float b) {
  uint32_t h;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(b), "f"(a));
  return h;
}

__device__ __forceinline__ uint32_t pack_bf16x2_rn(float a, float b) {
  uint32_t h;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(b), "f"(a));
  return h;
}

// a probability pair in the PV operand type (a in the low half)
template <int DT>
__device__ __forceinline__ uint32_t pack_p(float a, float b) {
  if constexpr (DT == kDtBF16) {
    return pack_bf16x2_rn(a, b);
  } else {
    return pack_f16x2_rn(a, b);
  }
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MMA issue by a whole warp of which one thread is elected: control flow stays
// uniform, so descriptors are formed in uniform registers, where the
// instruction wants them. Issued under `if (lane == 0)` instead, each MMA cost
// the warp 57 (A from shared memory) and 44 cycles (A from TMEM) alone on an SM.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes;
}

__device__ __forceinline__ void umma_f16_ss_if(uint32_t elected, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                               uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}

__device__ __forceinline__ void umma_f16_ts_if(uint32_t elected, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                               uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}

__device__ __forceinline__ void umma_commit_if(uint32_t elected, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(elected)
      : "memory");
}

// Scale columns [0, NO) of this thread's O row in TMEM by alpha.
template <int NO>
__device__ __forceinline__ void rescale_o(uint32_t taddr, float alpha) {
#pragma unroll
  for (int c = 0; c < NO / 32; ++c) {
    uint32_t v[32];
    tmem_ld32(taddr + c * 32, v);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
    tmem_st32(taddr + c * 32, v);
  }
  if constexpr (NO % 32 == 16) {
    uint32_t v[16];
    tmem_ld16(taddr + (NO / 32) * 32, v);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
    tmem_st16(taddr + (NO / 32) * 32, v);
  }
  tmem_wait_st();
}

}  // namespace tfb
