// Attention of a few new tokens per sequence over a paged cache (decode).
//
//   out_r = sum_j softmax_j(scale * q_r . k_j) v_j
//
// for the rows r = (token, query head) that share a key head, at most 16 of
// them per sequence; causal: a token sees the cache up to its own position.
//
// Bound by HBM: every key and value is read once for all of the group's
// query heads, 4 * rows flop per element, far below the tensor rate. So the
// kernel is a streaming kernel: each warp keeps a ring of 16-key tiles of its
// own in shared memory (cp.async, no block barrier in the loop), and the
// products run on mma.sync m16n8k16, whose 16 rows fit the group and whose
// result layout feeds the probabilities straight back as the next operand
// (the tcgen05 form needs 128 rows and a TMEM round trip per tile).
//
// Work is split over keys, not over sequences: all (sequence, key head) items
// are cut into units of 64 keys, numbered through, and each block takes an
// equal run of units, so one 100 000-key sequence and 64 ragged ones both
// fill the card. A run that covers an item writes its result; the one or two
// items that it covers in part leave fp32 partial results, which
// paged_combine_kernel joins in unit order (no atomics: the result does not
// depend on timing). Nothing in the workspace outlives the call.
//
// Scores, maxima and sums are fp32; the probabilities are rounded to the
// 16-bit operand type for the second product (the sum takes them unrounded),
// as in flash_fwd_tcgen05. Keys past a sequence's end are never read: their
// tile rows are zero-filled, so what an unused part of a page holds cannot
// reach a result.
#include "attn_common.cuh"
#include "common.cuh"
#include "launch.h"

namespace tfb {
namespace {

constexpr int kDecWarps = 4;
constexpr int kDecTile = 16;                        // keys per warp and step
constexpr int kDecUnit = kDecWarps * kDecTile;      // keys per unit
constexpr int kDecRows = 16;                        // query rows per item
constexpr int kDecCtasPerSm = 2;

struct DecodeK {
  SeqArgs a;
  int group;       // query heads per key head
  int page_shift;
  float scale_log2;
  float* o_part;   // [2 * gridDim.x][16][HD]
  float* l_part;   // [2 * gridDim.x][16] log2-sum-exp
  int* status;
};

template <int HD>
struct DecCfg {
  static constexpr int kStages = HD == 64 ? 6 : 3;
  static constexpr int kTileBytes = kDecTile * HD * 2;             // K or V tile
  static constexpr int kRing = kDecWarps * kStages * 2 * kTileBytes;  // 96 KB
  static constexpr int kMerge = 2 * kDecRows * HD * 4;              // two warps' O
  static constexpr int kBytes = kRing + kMerge;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;  // 0: zero-filled, the source is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == kDtBF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Query and key lengths of sequence b as the kernels use them, bounded by
// what the call's arrays can hold. A bound that bites is an error of the
// caller's; it is recorded and nothing outside the arrays is touched.
struct SeqLens {
  int q0, q, k;
  bool bad;
};
__device__ __forceinline__ SeqLens decode_lens(const SeqArgs& a, int group, int page_shift, int b) {
  SeqLens s;
  const int c0 = a.cu_q[b], c1 = a.cu_q[b + 1], kv = a.kv_lens[b];
  const long long cap = static_cast<long long>(a.max_pages) << page_shift;
  s.q0 = min(max(c0, 0), static_cast<int>(a.tokens));
  s.q = min(max(c1, s.q0), static_cast<int>(a.tokens)) - s.q0;
  s.q = min(s.q, kDecRows / group);
  s.k = kv < 0 ? 0 : (kv > cap ? static_cast<int>(cap) : kv);
  s.bad = c0 < 0 || c1 < c0 || c1 > a.tokens || s.q != c1 - c0 || s.k != kv;
  return s;
}
__device__ __forceinline__ int units_of(const SeqLens& s) { return s.q > 0 ? (s.k + kDecUnit - 1) / kDecUnit : 0; }

// Sum over all sequences of units, and (optionally) the sequence that holds
// unit number `at` when every sequence's units count kv_heads times: `seq`
// and the number of units before it. One warp.
__device__ __forceinline__ long long find_unit(const DecodeK& p, long long at, int& seq, long long& before) {
  const int lane = lane_id();
  long long run = 0;
  seq = -1;
  before = 0;
  for (int base = 0; base < p.a.batch; base += 32) {
    const int b = base + lane;
    long long n = 0;
    if (b < p.a.batch) n = static_cast<long long>(units_of(decode_lens(p.a, p.group, p.page_shift, b))) * p.a.kv_heads;
    long long inc = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, run + inc > at);
    if (seq < 0 && hit != 0) {
      const int l = __ffs(hit) - 1;
      seq = base + l;
      before = run + __shfl_sync(0xffffffffu, inc - n, l);
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  return run;
}

__device__ __forceinline__ long long run_start(long long total, int block, int blocks) {
  return total * block / blocks;
}

template <int HD, int DT>
__global__ void __launch_bounds__(kDecWarps * 32, kDecCtasPerSm) paged_decode_kernel(const DecodeK p) {
  using C = DecCfg<HD>;
  constexpr int KT = HD / 16;       // k-steps of Q K^T
  constexpr int CH = HD / 8;        // 16-byte chunks per tile row
  constexpr int RPI = 32 / CH;      // tile rows one warp-wide copy covers
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ float s_m[kDecWarps][kDecRows], s_l[kDecWarps][kDecRows];
  const int lane = lane_id();
  const int warp = warp_id();
  const SeqArgs& a = p.a;
  const uint32_t ring = smem_u32(smem) + warp * (C::kStages * 2 * C::kTileBytes);
  float* s_o = reinterpret_cast<float*>(smem + C::kRing);
  pdl_wait();
  pdl_trigger();

  int seq;
  long long before;
  long long total = find_unit(p, -1, seq, before);
  const long long u_end = run_start(total, blockIdx.x + 1, gridDim.x);
  long long u = run_start(total, blockIdx.x, gridDim.x);
  if (u >= u_end) return;
  find_unit(p, u, seq, before);

  bool first_segment = true;
  while (u < u_end) {
    // ---- the item (sequence, key head) and this run's part of it
    SeqLens s = decode_lens(a, p.group, p.page_shift, seq);
    int nu = units_of(s);
    while (nu == 0 || u - before >= static_cast<long long>(nu) * a.kv_heads) {
      before += static_cast<long long>(nu) * a.kv_heads;
      s = decode_lens(a, p.group, p.page_shift, ++seq);
      nu = units_of(s);
    }
    const int kvh = static_cast<int>((u - before) / nu);
    const int c_begin = static_cast<int>(u - before - static_cast<long long>(kvh) * nu);  // first unit of the segment
    const int c_end = static_cast<int>(u_end - u < nu - c_begin ? c_begin + (u_end - u) : nu);
    const bool whole = c_begin == 0 && c_end == nu;
    const int rows = s.q * p.group;

    // ---- queries as mma operands: rows lane/4 and lane/4 + 8
    uint32_t qf[KT][4];
    {
      const int r0 = lane >> 2, r1 = r0 + 8;
      const uint16_t* q = static_cast<const uint16_t*>(a.q);
      const int i0 = r0 / p.group, i1 = r1 / p.group;
      const uint16_t* p0 = q + static_cast<long long>(s.q0 + i0) * a.q_ts +
                           static_cast<long long>(kvh * p.group + (r0 - i0 * p.group)) * a.q_hs + (lane & 3) * 2;
      const uint16_t* p1 = q + static_cast<long long>(s.q0 + i1) * a.q_ts +
                           static_cast<long long>(kvh * p.group + (r1 - i1 * p.group)) * a.q_hs + (lane & 3) * 2;
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        qf[k][0] = r0 < rows ? *reinterpret_cast<const uint32_t*>(p0 + k * 16) : 0u;
        qf[k][1] = r1 < rows ? *reinterpret_cast<const uint32_t*>(p1 + k * 16) : 0u;
        qf[k][2] = r0 < rows ? *reinterpret_cast<const uint32_t*>(p0 + k * 16 + 8) : 0u;
        qf[k][3] = r1 < rows ? *reinterpret_cast<const uint32_t*>(p1 + k * 16 + 8) : 0u;
      }
    }
    // keys row r admits: up to its token's own position (causal)
    const int lim0 = a.causal ? s.k - s.q + (lane >> 2) / p.group + 1 : s.k;
    const int lim1 = a.causal ? s.k - s.q + ((lane >> 2) + 8) / p.group + 1 : s.k;

    const int* table = a.page_table + static_cast<long long>(seq) * a.table_ld;
    const uint16_t* kbase = static_cast<const uint16_t*>(a.k) + static_cast<long long>(kvh) * a.k_hs;
    const uint16_t* vbase = static_cast<const uint16_t*>(a.v) + static_cast<long long>(kvh) * a.v_hs;
    auto page_of = [&](int c) {  // page of this warp's tile of unit c (a tile lies within a page)
      const int key0 = c * kDecUnit + warp * kDecTile;
      return c < c_end && key0 < s.k ? __ldg(table + (key0 >> p.page_shift)) : 0;
    };
    auto issue = [&](int c, int page) {
      if (c < c_end) {
        const int key0 = c * kDecUnit + warp * kDecTile;
        const int stage = (c - c_begin) % C::kStages;
        const uint32_t dst = ring + stage * (2 * C::kTileBytes);
        const bool ok = page >= 0 && page < a.num_pages;
        if (!ok && key0 < s.k && lane == 0) record_error(p.status, kDevBadIndex);
        const int row = key0 & ((1 << p.page_shift) - 1);
        const uint16_t* kp = kbase + static_cast<long long>(ok ? page : 0) * a.k_ps + row * a.k_ts;
        const uint16_t* vp = vbase + static_cast<long long>(ok ? page : 0) * a.v_ps + row * a.v_ts;
        const int ch = lane % CH;
#pragma unroll
        for (int i = 0; i < kDecTile / RPI; ++i) {
          const int r = i * RPI + lane / CH;
          const bool on = ok && key0 + r < s.k;
          const uint32_t d = dst + r * (HD * 2) + ((ch ^ (r & 7)) << 4);
          cp_async16(d, on ? kp + r * a.k_ts + ch * 8 : kbase, on);
          cp_async16(d + C::kTileBytes, on ? vp + r * a.v_ts + ch * 8 : vbase, on);
        }
      }
      cp_commit();
    };

    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

    int ahead[C::kStages];
#pragma unroll
    for (int i = 0; i < C::kStages; ++i) ahead[i] = page_of(c_begin + i);
#pragma unroll
    for (int i = 0; i < C::kStages - 1; ++i) issue(c_begin + i, ahead[i]);
    int page = ahead[C::kStages - 1];
    for (int c = c_begin; c < c_end; ++c) {
      cp_wait<C::kStages - 2>();
      __syncwarp();
      const int key0 = c * kDecUnit + warp * kDecTile;
      // the stage of the tile before this one is free: refill it first, with
      // the page read one step ago
      issue(c + C::kStages - 1, page);
      page = page_of(c + C::kStages);
      if (key0 < s.k) {
        const uint32_t kt = ring + ((c - c_begin) % C::kStages) * (2 * C::kTileBytes);
        const uint32_t vt = kt + C::kTileBytes;
        // S = Q K^T: two 8-key column tiles; matrices (keys 0-7 | 8-15) x (k 0-7 | 8-15)
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
        {
          const int r = (lane & 7) + ((lane >> 4) << 3);
          const int hi = (lane >> 3) & 1;
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            uint32_t b[4];
            ldsm4(kt + r * (HD * 2) + (((2 * k + hi) ^ (r & 7)) << 4), b);
            mma16816<DT>(s0, qf[k], b[0], b[1]);
            mma16816<DT>(s1, qf[k], b[2], b[3]);
          }
        }
        const int kc = key0 + (lane & 3) * 2;
        s0[0] = kc < lim0 ? s0[0] : -INFINITY;
        s0[1] = kc + 1 < lim0 ? s0[1] : -INFINITY;
        s1[0] = kc + 8 < lim0 ? s1[0] : -INFINITY;
        s1[1] = kc + 9 < lim0 ? s1[1] : -INFINITY;
        s0[2] = kc < lim1 ? s0[2] : -INFINITY;
        s0[3] = kc + 1 < lim1 ? s0[3] : -INFINITY;
        s1[2] = kc + 8 < lim1 ? s1[2] : -INFINITY;
        s1[3] = kc + 9 < lim1 ? s1[3] : -INFINITY;
        float t0 = fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s1[0], s1[1]));
        float t1 = fmaxf(fmaxf(s0[2], s0[3]), fmaxf(s1[2], s1[3]));
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2)) * p.scale_log2;
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2)) * p.scale_log2;
        // lazy rescale: a row's reference maximum moves only when the new one
        // is above it by more than 2^8, so the probabilities stay below 2^8
        const bool up = t0 > m0 + 8.f || t1 > m1 + 8.f;
        if (__any_sync(0xffffffffu, up)) {
          const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
          const float a0 = m0 == -INFINITY ? 0.f : ex2_f32(m0 - n0);
          const float a1 = m1 == -INFINITY ? 0.f : ex2_f32(m1 - n1);
          l0 *= a0;
          l1 *= a1;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            o[i][0] *= a0;
            o[i][1] *= a0;
            o[i][2] *= a1;
            o[i][3] *= a1;
          }
          m0 = n0;
          m1 = n1;
        }
        const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
        float e[8];
        e[0] = ex2_f32(fmaf(s0[0], p.scale_log2, -u0));
        e[1] = ex2_f32(fmaf(s0[1], p.scale_log2, -u0));
        e[2] = ex2_f32(fmaf(s0[2], p.scale_log2, -u1));
        e[3] = ex2_f32(fmaf(s0[3], p.scale_log2, -u1));
        e[4] = ex2_f32(fmaf(s1[0], p.scale_log2, -u0));
        e[5] = ex2_f32(fmaf(s1[1], p.scale_log2, -u0));
        e[6] = ex2_f32(fmaf(s1[2], p.scale_log2, -u1));
        e[7] = ex2_f32(fmaf(s1[3], p.scale_log2, -u1));
        l0 += (e[0] + e[1]) + (e[4] + e[5]);
        l1 += (e[2] + e[3]) + (e[6] + e[7]);
        const uint32_t pf[4] = {pack2<DT>(e[0], e[1]), pack2<DT>(e[2], e[3]), pack2<DT>(e[4], e[5]),
                                pack2<DT>(e[6], e[7])};
        // O += P V: V rows are keys; transposed matrices (keys 0-7 | 8-15) x 8 columns
        {
          const int r = (lane & 7) + (((lane >> 3) & 1) << 3);
          const int hi = lane >> 4;
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            uint32_t b[4];
            ldsm4t(vt + r * (HD * 2) + (((2 * n + hi) ^ (r & 7)) << 4), b);
            mma16816<DT>(o[2 * n], pf, b[0], b[1]);
            mma16816<DT>(o[2 * n + 1], pf, b[2], b[3]);
          }
        }
      }
    }
    cp_wait<0>();
    __syncwarp();

    // ---- join the four warps: common maximum, then O summed in warp order
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const int r0 = lane >> 2, r1 = r0 + 8;
    if ((lane & 3) == 0) {
      s_m[warp][r0] = m0;
      s_m[warp][r1] = m1;
      s_l[warp][r0] = l0;
      s_l[warp][r1] = l1;
    }
    __syncthreads();
    float M0 = -INFINITY, M1 = -INFINITY, L0 = 0.f, L1 = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      M0 = fmaxf(M0, s_m[w][r0]);
      M1 = fmaxf(M1, s_m[w][r1]);
    }
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      L0 += s_m[w][r0] == -INFINITY ? 0.f : s_l[w][r0] * ex2_f32(s_m[w][r0] - M0);
      L1 += s_m[w][r1] == -INFINITY ? 0.f : s_l[w][r1] * ex2_f32(s_m[w][r1] - M1);
    }
    const float f0 = m0 == -INFINITY ? 0.f : ex2_f32(m0 - M0);
    const float f1 = m1 == -INFINITY ? 0.f : ex2_f32(m1 - M1);
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      o[i][0] *= f0;
      o[i][1] *= f0;
      o[i][2] *= f1;
      o[i][3] *= f1;
    }
    // warps 2, 3 -> 0, 1, then 1 -> 0
    const int slot = warp & 1;
    float* so = s_o + slot * (kDecRows * HD);
    auto put = [&](float* dst) {
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        *reinterpret_cast<float2*>(dst + (i * 32 + lane) * 4) = make_float2(o[i][0], o[i][1]);
        *reinterpret_cast<float2*>(dst + (i * 32 + lane) * 4 + 2) = make_float2(o[i][2], o[i][3]);
      }
    };
    auto add = [&](const float* src) {
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(src + (i * 32 + lane) * 4);
        o[i][0] += x.x;
        o[i][1] += x.y;
        o[i][2] += x.z;
        o[i][3] += x.w;
      }
    };
    if (warp >= 2) put(so);
    __syncthreads();
    if (warp < 2) add(so);
    if (warp == 1) put(so);
    __syncthreads();
    if (warp == 0) {
      add(s_o + kDecRows * HD);
      const float i0 = L0 > 0.f ? 1.f / L0 : 0.f, i1 = L1 > 0.f ? 1.f / L1 : 0.f;
      const float g0 = L0 > 0.f ? M0 + __log2f(L0) : -INFINITY, g1 = L1 > 0.f ? M1 + __log2f(L1) : -INFINITY;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = half ? r1 : r0;
        if (r >= rows) continue;
        const float inv = half ? i1 : i0, lg = half ? g1 : g0;
        const int tok = s.q0 + r / p.group, head = kvh * p.group + r % p.group;
        if (whole) {
          const long long base = static_cast<long long>(tok) * a.o_ts + static_cast<long long>(head) * a.o_hs + (lane & 3) * 2;
          if (a.out_f32) {
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
              *reinterpret_cast<float2*>(static_cast<float*>(a.out) + base + i * 8) =
                  make_float2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
          } else {
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
              *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + base + i * 8) =
                  pack2<DT>(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
          }
          if (a.lse != nullptr && (lane & 3) == 0)
            a.lse[static_cast<long long>(head) * a.tokens + tok] = lg * 0.69314718055994531f;
        } else {
          const long long part = 2ll * blockIdx.x + (first_segment ? 0 : 1);
          float* dst = p.o_part + (part * kDecRows + r) * HD + (lane & 3) * 2;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i)
            *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
          if ((lane & 3) == 0) p.l_part[part * kDecRows + r] = lg;
        }
      }
    }
    u += c_end - c_begin;
    first_segment = false;
  }
}

// Joins the partial results of every item that more than one block worked on,
// and writes the rows of sequences without keys (out 0, log-sum-exp -inf).
// One block per (sequence, key head).
template <int HD, int DT>
__global__ void __launch_bounds__(128) paged_combine_kernel(const DecodeK p, int blocks) {
  const SeqArgs& a = p.a;
  pdl_wait();
  pdl_trigger();
  const int seq = blockIdx.x, kvh = blockIdx.y;
  const int lane = lane_id(), warp = warp_id();
  const SeqLens s = decode_lens(a, p.group, p.page_shift, seq);
  const int rows = s.q * p.group;
  if (s.bad && kvh == 0 && threadIdx.x == 0) record_error(p.status, kDevBadIndex);
  if (rows == 0) return;
  const int nu = units_of(s);
  long long run = 0, before = 0;  // units of all sequences, and of those before this one
  for (int base = 0; base < a.batch; base += 32) {
    const int b = base + lane;
    long long n = 0;
    if (b < a.batch) n = static_cast<long long>(units_of(decode_lens(a, p.group, p.page_shift, b))) * a.kv_heads;
    long long mine = b < seq ? n : 0;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      n += __shfl_xor_sync(0xffffffffu, n, d);
      mine += __shfl_xor_sync(0xffffffffu, mine, d);
    }
    run += n;
    before += mine;
  }
  const long long ua = before + static_cast<long long>(kvh) * nu, ub = ua + nu;
  // blocks whose runs meet [ua, ub): run_start(c) <= ua < run_start(c + 1)
  int c0 = 0, c1 = -1;
  if (nu > 0) {
    c0 = static_cast<int>(ua * blocks / run);
    while (c0 + 1 < blocks && run_start(run, c0 + 1, blocks) <= ua) ++c0;
    while (run_start(run, c0, blocks) > ua) --c0;
    c1 = static_cast<int>((ub - 1) * blocks / run);
    while (c1 + 1 < blocks && run_start(run, c1 + 1, blocks) <= ub - 1) ++c1;
    while (run_start(run, c1, blocks) > ub - 1) --c1;
    if (c0 == c1) return;  // one block saw all of it and wrote the result
  }
  for (int r = warp; r < rows; r += 4) {
    float m = -INFINITY;
    for (int c = c0; c <= c1; ++c) {
      if (run_start(run, c, blocks) == run_start(run, c + 1, blocks)) continue;  // an empty run wrote nothing
      const long long part = 2ll * c + (run_start(run, c, blocks) >= ua ? 0 : 1);
      m = fmaxf(m, p.l_part[part * kDecRows + r]);
    }
    float l = 0.f, acc[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) acc[i] = 0.f;
    for (int c = c0; c <= c1; ++c) {
      if (run_start(run, c, blocks) == run_start(run, c + 1, blocks)) continue;
      const long long part = 2ll * c + (run_start(run, c, blocks) >= ua ? 0 : 1);
      const float lg = p.l_part[part * kDecRows + r];
      if (lg == -INFINITY) continue;
      const float w = ex2_f32(lg - m);
      l += w;
      const float* src = p.o_part + (part * kDecRows + r) * HD + lane * (HD / 32);
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) acc[i] = fmaf(w, src[i], acc[i]);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int tok = s.q0 + r / p.group, head = kvh * p.group + r % p.group;
    const long long base =
        static_cast<long long>(tok) * a.o_ts + static_cast<long long>(head) * a.o_hs + lane * (HD / 32);
#pragma unroll
    for (int i = 0; i < HD / 32; i += 2) {
      if (a.out_f32) {
        *reinterpret_cast<float2*>(static_cast<float*>(a.out) + base + i) = make_float2(acc[i] * inv, acc[i + 1] * inv);
      } else {
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + base + i) =
            pack2<DT>(acc[i] * inv, acc[i + 1] * inv);
      }
    }
    if (a.lse != nullptr && lane == 0)
      a.lse[static_cast<long long>(head) * a.tokens + tok] =
          l > 0.f ? (m + __log2f(l)) * 0.69314718055994531f : -INFINITY;
  }
}

// Blocks of a call: every SM's share, but no more than there can be units.
int decode_blocks(const SeqArgs& a) {
  const long long units = (a.max_k + kDecUnit - 1) / kDecUnit * a.batch * a.kv_heads;
  const long long most = static_cast<long long>(kDecCtasPerSm) * device_sm_count();
  return static_cast<int>(units < 1 ? 1 : units < most ? units : most);
}

template <int HD, int DT>
int launch_decode(const DecodeK& k, int blocks, cudaStream_t stream) {
  using C = DecCfg<HD>;
  auto kern = paged_decode_kernel<HD, DT>;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_done[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
    if (e != cudaSuccess) return set_error(TF_ERR_LAUNCH, "cudaFuncSetAttribute(paged decode): %s", cudaGetErrorString(e));
    attr_done[dev & 63] = true;
  }
  cudaError_t e = launch_k(kern, dim3(blocks), dim3(kDecWarps * 32), C::kBytes, stream, k);
  if (e == cudaSuccess)
    e = launch_k(paged_combine_kernel<HD, DT>, dim3(k.a.batch, k.a.kv_heads), dim3(128), 0, stream, k, blocks);
  if (e != cudaSuccess) return set_error(TF_ERR_LAUNCH, "paged decode launch: %s", cudaGetErrorString(e));
  return TF_OK;
}

}  // namespace

bool paged_is_decode(const SeqArgs& a) { return a.max_q * (a.heads / a.kv_heads) <= kDecRows; }

long long paged_decode_workspace(const SeqArgs& a) {
  return static_cast<long long>(decode_blocks(a)) * 2 * kDecRows * (a.head_dim + 1) * 4;
}

int paged_decode(const SeqArgs& a, cudaStream_t stream) {
  DecodeK k = {};
  k.a = a;
  k.group = a.heads / a.kv_heads;
  while ((1ll << k.page_shift) < a.page_size) ++k.page_shift;
  k.scale_log2 = a.scale * 1.4426950408889634f;
  const int blocks = decode_blocks(a);
  k.o_part = static_cast<float*>(a.workspace);
  k.l_part = k.o_part + static_cast<long long>(blocks) * 2 * kDecRows * a.head_dim;
  k.status = device_status_ptr();
  if (k.status == nullptr) return last_error_code();
  if (a.bf16)
    return a.head_dim == 64 ? launch_decode<64, kDtBF16>(k, blocks, stream) : launch_decode<128, kDtBF16>(k, blocks, stream);
  return a.head_dim == 64 ? launch_decode<64, kDtF16>(k, blocks, stream) : launch_decode<128, kDtF16>(k, blocks, stream);
}

}  // namespace tfb
