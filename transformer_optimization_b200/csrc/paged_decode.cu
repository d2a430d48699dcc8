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
constexpr int kSeqCache = 32;  // sequences of a block's run whose lengths are kept in shared memory

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
  static constexpr int kStat = 2 * kDecWarps * kDecRows * 4;         // the warps' row maxima and sums
  static constexpr int kBytes = kRing + kMerge + kStat + kSeqCache * 12;
  static_assert(kDecCtasPerSm * (kBytes + 1024) <= 228 * 1024, "two blocks per SM");
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
  s.q = min(s.q, min(kDecRows / group, static_cast<int>(a.max_q)));
  s.k = kv < 0 ? 0 : (kv > cap ? static_cast<int>(cap) : kv);
  s.bad = c0 < 0 || c1 < c0 || c1 > a.tokens || s.q != c1 - c0 || s.k != kv;
  return s;
}
__device__ __forceinline__ int units_of(const SeqLens& s) { return s.q > 0 ? (s.k + kDecUnit - 1) / kDecUnit : 0; }

// Units of all sequences (every key head counted), one warp; four sequences
// per lane are requested at a time.
__device__ __forceinline__ long long total_units(const DecodeK& p) {
  long long n = 0;
#pragma unroll 4
  for (int b = lane_id(); b < p.a.batch; b += 32)
    n += units_of(decode_lens(p.a, p.group, p.page_shift, b));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
  return n * p.a.kv_heads;
}

// The sequence that holds unit `at`, and the number of units before it.
__device__ __forceinline__ int find_unit(const DecodeK& p, long long at, long long& before) {
  const int lane = lane_id();
  long long run = 0;
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
    if (hit != 0) {
      const int l = __ffs(hit) - 1;
      before = run + __shfl_sync(0xffffffffu, inc - n, l);
      return base + l;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  before = run;
  return -1;
}

// Block c's run of units: total / blocks each, one more for the first
// total % blocks.
struct Runs {
  long long per, extra;
  __device__ __forceinline__ Runs(long long total, int blocks) : per(total / blocks), extra(total % blocks) {}
  __device__ __forceinline__ long long start(long long c) const { return c * per + (c < extra ? c : extra); }
  __device__ __forceinline__ int block_of(long long u) const {
    const long long head = extra * (per + 1);
    return static_cast<int>(u < head ? u / (per + 1) : extra + (u - head) / per);
  }
};

template <int HD, int DT>
__global__ void __launch_bounds__(kDecWarps * 32, kDecCtasPerSm) paged_decode_kernel(const DecodeK p) {
  using C = DecCfg<HD>;
  constexpr int KT = HD / 16;       // k-steps of Q K^T
  constexpr int CH = HD / 8;        // 16-byte chunks per tile row
  constexpr int RPI = 32 / CH;      // tile rows one warp-wide copy covers
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = lane_id();
  const int warp = warp_id();
  const SeqArgs& a = p.a;
  const uint32_t ring = smem_u32(smem) + warp * (C::kStages * 2 * C::kTileBytes);
  float* s_o = reinterpret_cast<float*>(smem + C::kRing);
  auto s_m = reinterpret_cast<float(*)[kDecRows]>(smem + C::kRing + C::kMerge);
  auto s_l = s_m + kDecWarps;
  auto s_seq = reinterpret_cast<int(*)[3]>(smem + C::kRing + C::kMerge + C::kStat);
  pdl_wait();
  pdl_trigger();

  const Runs runs(total_units(p), gridDim.x);
  const long long u_begin = runs.start(blockIdx.x);
  const int steps = static_cast<int>(runs.start(blockIdx.x + 1) - u_begin);
  if (steps == 0) return;
  long long before;
  const int seq0 = find_unit(p, u_begin, before);
  for (int i = threadIdx.x; i < kSeqCache; i += kDecWarps * 32) {
    SeqLens s = {};
    if (seq0 + i < a.batch) s = decode_lens(a, p.group, p.page_shift, seq0 + i);
    s_seq[i][0] = s.q0;
    s_seq[i][1] = s.q;
    s_seq[i][2] = s.k;
  }
  __syncthreads();

  // A position in the run: unit c of the nu units of (seq, kvh). Loads run
  // kStages - 1 units ahead of the products with a position of their own, so
  // the ring stays full across items.
  struct At {
    int seq, kvh, c, nu;
    SeqLens s;
  };
  auto enter = [&](At& x, int seq) {  // the first sequence from `seq` on that has units
    while (true) {
      if (seq - seq0 < kSeqCache) {
        const int* e = s_seq[seq - seq0];
        x.s.q0 = e[0];
        x.s.q = e[1];
        x.s.k = e[2];
      } else {
        x.s = decode_lens(a, p.group, p.page_shift, seq);
      }
      x.nu = units_of(x.s);
      if (x.nu > 0) break;
      ++seq;
    }
    x.seq = seq;
  };
  auto advance = [&](At& x, bool more) {  // to the next unit of the run
    if (++x.c < x.nu || !more) return;
    x.c = 0;
    if (++x.kvh == a.kv_heads) {
      x.kvh = 0;
      enter(x, x.seq + 1);
    }
  };
  At now, ahead;
  enter(now, seq0);
  now.kvh = static_cast<int>((u_begin - before) / now.nu);
  now.c = static_cast<int>(u_begin - before - static_cast<long long>(now.kvh) * now.nu);
  ahead = now;

  // this warp's tile of a unit lies within one page: its table entry, and its copy
  auto page_of = [&](const At& x) {
    const int key0 = x.c * kDecUnit + warp * kDecTile;
    return key0 < x.s.k ? a.page_table[x.seq * a.table_ld + (key0 >> p.page_shift)] : 0;
  };
  auto issue = [&](const At& x, int page, int stage) {
    const int key0 = x.c * kDecUnit + warp * kDecTile;
    const uint32_t dst = ring + stage * (2 * C::kTileBytes);
    const bool ok = page >= 0 && page < a.num_pages;
    if (!ok && lane == 0) record_error(p.status, kDevBadIndex);
    const int row = key0 & ((1 << p.page_shift) - 1);
    const int ch = lane % CH;
    const long long pg = ok ? page : 0;
    const uint16_t* kp = static_cast<const uint16_t*>(a.k) + pg * a.k_ps + x.kvh * a.k_hs + row * a.k_ts + ch * 8;
    const uint16_t* vp = static_cast<const uint16_t*>(a.v) + pg * a.v_ps + x.kvh * a.v_hs + row * a.v_ts + ch * 8;
#pragma unroll
    for (int i = 0; i < kDecTile / RPI; ++i) {
      const int r = i * RPI + lane / CH;
      const bool on = ok && key0 + r < x.s.k;
      const uint32_t d = dst + r * (HD * 2) + ((ch ^ (r & 7)) << 4);
      cp_async16(d, on ? kp + r * a.k_ts : static_cast<const uint16_t*>(a.k), on);
      cp_async16(d + C::kTileBytes, on ? vp + r * a.v_ts : static_cast<const uint16_t*>(a.v), on);
    }
  };
  int loaded = 0;  // units issued
  int page = page_of(ahead);
  auto load_next = [&](int stage) {
    if (loaded < steps) {
      if (ahead.c * kDecUnit + warp * kDecTile < ahead.s.k) issue(ahead, page, stage);
      ++loaded;
      advance(ahead, loaded < steps);
      if (loaded < steps) page = page_of(ahead);
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) load_next(i);

  int stage = 0, free_stage = C::kStages - 1;
  bool first_segment = true;
  for (int step = 0; step < steps;) {
    // ---- a segment: this run's part of one item
    const SeqLens s = now.s;
    const int kvh = now.kvh;
    const int c_end = min(now.nu, now.c + steps - step);
    const bool whole = now.c == 0 && c_end == now.nu;
    const int rows = s.q * p.group;

    // queries as mma operands: rows lane/4 and lane/4 + 8
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

    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

    for (int c = now.c; c < c_end; ++c, ++step) {
      cp_wait<C::kStages - 2>();
      __syncwarp();
      load_next(free_stage);  // the stage of the unit before this one
      const int key0 = c * kDecUnit + warp * kDecTile;
      if (key0 < s.k) {
        const uint32_t kt = ring + stage * (2 * C::kTileBytes);
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
      free_stage = stage;
      stage = stage + 1 == C::kStages ? 0 : stage + 1;
    }

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
    // on to the next item (or to the end)
    first_segment = false;
    now.c = c_end - 1;
    advance(now, step < steps);
  }
  cp_wait<0>();
}

// Joins the partial results of every item that more than one block worked on,
// and writes the rows of sequences without keys (out 0, log-sum-exp -inf).
// One block per (sequence, key head) and row; its warps take every fourth
// partial result, so that long joins are not a chain of memory latencies, and
// add up in warp order.
template <int HD, int DT>
__global__ void __launch_bounds__(kDecWarps * 32) paged_combine_kernel(const DecodeK p, int blocks) {
  constexpr int E = HD / 32;
  __shared__ float s_o[kDecWarps][HD];
  __shared__ float s_l[kDecWarps];
  const SeqArgs& a = p.a;
  pdl_wait();
  pdl_trigger();
  const int seq = blockIdx.x / a.kv_heads, kvh = blockIdx.x - seq * a.kv_heads;
  const int r = blockIdx.y;
  const int lane = lane_id(), warp = warp_id();
  const SeqLens s = decode_lens(a, p.group, p.page_shift, seq);
  if (s.bad && kvh == 0 && r == 0 && threadIdx.x == 0) record_error(p.status, kDevBadIndex);
  if (r >= s.q * p.group) return;
  const int nu = units_of(s);
  int c0 = 0, c1 = -1;
  long long ua = 0;
  Runs runs(0, 1);
  if (nu > 0) {
    long long all = 0, mine = 0;  // units of all sequences, and of those before this one
#pragma unroll 4
    for (int b = lane; b < a.batch; b += 32) {
      const int n = units_of(decode_lens(a, p.group, p.page_shift, b));
      all += n;
      mine += b < seq ? n : 0;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, d);
      mine += __shfl_xor_sync(0xffffffffu, mine, d);
    }
    runs = Runs(all * a.kv_heads, blocks);
    ua = mine * a.kv_heads + static_cast<long long>(kvh) * nu;
    c0 = runs.block_of(ua);
    c1 = runs.block_of(ua + nu - 1);
    if (c0 == c1) return;  // one block saw all of it and wrote the result
  }
  // partial result of block c: its first segment's place, unless the block
  // began with an earlier item (only c0 can have)
  const bool late = runs.start(c0) < ua;
  auto part = [&](int c) { return 2ll * c + (late && c == c0 ? 1 : 0); };
  float m = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, p.l_part[part(c) * kDecRows + r]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float l = 0.f, acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int c = c0 + warp; c <= c1; c += kDecWarps) {
    const float lg = p.l_part[part(c) * kDecRows + r];
    const float w = lg == -INFINITY ? 0.f : ex2_f32(lg - m);
    const float* src = p.o_part + (part(c) * kDecRows + r) * HD + lane * E;
    l += w;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = fmaf(w, src[i], acc[i]);
  }
#pragma unroll
  for (int i = 0; i < E; ++i) s_o[warp][lane * E + i] = acc[i];
  if (lane == 0) s_l[warp] = l;
  __syncthreads();
  l = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int tok = s.q0 + r / p.group, head = kvh * p.group + r % p.group;
  const long long base = static_cast<long long>(tok) * a.o_ts + static_cast<long long>(head) * a.o_hs;
  for (int i = threadIdx.x; i < HD; i += kDecWarps * 32) {
    const float x = ((s_o[0][i] + s_o[1][i]) + (s_o[2][i] + s_o[3][i])) * inv;
    if (a.out_f32) {
      static_cast<float*>(a.out)[base + i] = x;
    } else {
      static_cast<uint16_t*>(a.out)[base + i] = static_cast<uint16_t>(pack2<DT>(x, 0.f) & 0xffffu);
    }
  }
  if (a.lse != nullptr && threadIdx.x == 0)
    a.lse[static_cast<long long>(head) * a.tokens + tok] =
        l > 0.f ? (m + __log2f(l)) * 0.69314718055994531f : -INFINITY;
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
    e = launch_k(paged_combine_kernel<HD, DT>,
                 dim3(static_cast<unsigned>(k.a.batch * k.a.kv_heads), static_cast<unsigned>(k.a.max_q * k.group)),
                 dim3(kDecWarps * 32), 0, stream, k, blocks);
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
