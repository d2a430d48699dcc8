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
// own in shared memory, filled by TMA from the page that holds them (no block
// barrier in the loop, no per-lane addresses), and the products run on
// mma.sync m16n8k16, whose 16 rows fit the group and whose result layout feeds
// the probabilities straight back as the next operand (the tcgen05 form needs
// 128 rows and a TMEM round trip per tile). 32 sequences of 8192 keys, 32 heads
// over 8, hd 128: 0.178 ms with the join, 6.03 TB/s; 64 of 100 to 8192: 70.3 us;
// one of 100 000, 16 over 4, hd 64: 23.6 us; one of 1000: 7.5 us, all latency.
//
// Work is split over keys, not over sequences: all (sequence, key head) items
// are cut into units of 64 keys, numbered through with kSegment more places
// per item for its start and end, and each block takes an equal run of places,
// so one 100 000-key sequence and 64 ragged ones both fill the card. A run
// that covers an item writes its result; the one or two items that it covers
// in part leave fp32 partial results, which paged_combine_kernel joins in unit
// order (no atomics: the result does not depend on timing). Nothing in the
// workspace outlives the call.
//
// Scores, maxima and sums are fp32; the probabilities are rounded to the
// 16-bit operand type for the second product (the sum takes them unrounded),
// as in flash_fwd_tcgen05. The value rows of a tile past the sequence's end
// are zeroed before the product, so what an unused part of a page holds cannot
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
constexpr int kSegment = 2;                         // an item's start and end cost about two units (place numbering)
constexpr int kDecCtasPerSm = 2;
constexpr int kSeqCache = 32;  // sequences of a block's run whose lengths are kept in shared memory

struct DecodeK {
  SeqArgs a;
  int group;       // query heads per key head
  int page_shift;
  float scale_log2;
  float* o_part;   // [2 * gridDim.x][16][HD]
  float* l_part;   // [2 * gridDim.x][16] log2-sum-exp
  int2* spans;     // [batch][kv_heads] place of the item's first partial result, blocks that have part in it
  int* status;
};

template <int HD>
struct DecCfg {
  static constexpr int kStages = HD == 64 ? 6 : 3;
  static constexpr int kTileBytes = kDecTile * HD * 2;             // K or V tile
  static constexpr int kRing = kDecWarps * kStages * 2 * kTileBytes;  // 96 KB
  static constexpr int kMerge = kDecWarps * 8 * HD * 4;              // the warps' O, 8 rows
  static constexpr int kStat = 2 * kDecWarps * kDecRows * 4;         // their row maxima and sums
  static constexpr int kBytes = kRing + kMerge + kStat + kSeqCache * 12 + kDecWarps * kStages * 8;
  static_assert(kDecCtasPerSm * (kBytes + 1024) <= 228 * 1024, "two blocks per SM");
};

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
// places of one key head: none without units
__device__ __forceinline__ int places_of(const SeqLens& s) {
  const int n = units_of(s);
  return n > 0 ? n + kSegment : 0;
}

// Places of all sequences (every key head counted), one warp; `mine` is
// sequence lane's. The host bounds the total below 2^31.
__device__ __forceinline__ int total_places(const DecodeK& p, int mine) {
  int n = mine;
#pragma unroll 4
  for (int b = lane_id() + 32; b < p.a.batch; b += 32) n += places_of(decode_lens(p.a, p.group, p.page_shift, b));
  return __reduce_add_sync(0xffffffffu, n) * p.a.kv_heads;
}

// The sequence that holds place `at`, and the number of places before it.
__device__ __forceinline__ int find_place(const DecodeK& p, int mine, int at, int& before) {
  const int lane = lane_id();
  int run = 0;
  for (int base = 0; base < p.a.batch; base += 32) {
    const int b = base + lane;
    int n = mine;
    if (base > 0) n = b < p.a.batch ? places_of(decode_lens(p.a, p.group, p.page_shift, b)) : 0;
    n *= p.a.kv_heads;
    int inc = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, d);
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

// Block c's run of places: total / blocks each, one more for the first
// total % blocks.
struct Runs {
  int per, extra;
  __device__ __forceinline__ Runs(int total, int blocks) : per(total / blocks), extra(total - per * blocks) {}
  __device__ __forceinline__ int start(int c) const { return c * per + min(c, extra); }
  __device__ __forceinline__ int block_of(int u) const {
    const int head = extra * (per + 1);
    return u < head ? u / (per + 1) : extra + (u - head) / per;
  }
};

template <int HD, int DT>
__global__ void __launch_bounds__(kDecWarps * 32, kDecCtasPerSm)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const __grid_constant__ DecodeK p) {
  using C = DecCfg<HD>;
  constexpr int KT = HD / 16;  // k-steps of Q K^T
  constexpr int kStageBytes = 2 * C::kTileBytes;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = lane_id();
  const int warp = warp_id();
  const SeqArgs& a = p.a;
  uint8_t* ring = smem + warp * (C::kStages * kStageBytes);
  float* s_o = reinterpret_cast<float*>(smem + C::kRing);
  auto s_m = reinterpret_cast<float(*)[kDecRows]>(smem + C::kRing + C::kMerge);
  auto s_l = s_m + kDecWarps;
  auto s_seq = reinterpret_cast<int(*)[3]>(smem + C::kRing + C::kMerge + C::kStat);
  uint64_t* full =
      reinterpret_cast<uint64_t*>(smem + C::kRing + C::kMerge + C::kStat + kSeqCache * 12) + warp * C::kStages;
  if (lane == 0) {
    for (int i = 0; i < C::kStages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  pdl_wait();
  pdl_trigger();

  const int mine = lane < a.batch ? places_of(decode_lens(a, p.group, p.page_shift, lane)) : 0;
  const Runs runs(total_places(p, mine), gridDim.x);
  const int u_begin = runs.start(blockIdx.x), u_end = runs.start(blockIdx.x + 1);
  if (u_begin == u_end) return;
  int before;
  const int seq0 = find_place(p, mine, u_begin, before);
  for (int i = threadIdx.x; i < kSeqCache; i += kDecWarps * 32) {
    SeqLens s = {};
    if (seq0 + i < a.batch) s = decode_lens(a, p.group, p.page_shift, seq0 + i);
    s_seq[i][0] = s.q0;
    s_seq[i][1] = s.q;
    s_seq[i][2] = s.k;
  }
  __syncthreads();

  // A position in the run: unit c of the nu units of (seq, kvh), with `left`
  // places of the run from it on. Loads run kStages - 1 units ahead of the
  // products with a position of their own, so the ring stays full across items.
  struct At {
    int seq, kvh, c, nu, left;
    SeqLens s;
  };
  auto enter = [&](At& x, int seq) {  // the first sequence from `seq` on that has units, or none
    x.nu = 0;
    for (; seq < a.batch && x.nu == 0; ++seq) {
      if (seq - seq0 < kSeqCache) {
        const int* e = s_seq[seq - seq0];
        x.s.q0 = e[0];
        x.s.q = e[1];
        x.s.k = e[2];
      } else {
        x.s = decode_lens(a, p.group, p.page_shift, seq);
      }
      x.nu = units_of(x.s);
      x.seq = seq;
    }
    if (x.nu == 0) x.left = 0;
  };
  auto next_item = [&](At& x) {
    x.c = 0;
    if (++x.kvh == a.kv_heads) {
      x.kvh = 0;
      enter(x, x.seq + 1);
    }
  };
  auto step = [&](At& x) {  // past one unit, over the item's end places if it was the last
    --x.left;
    if (++x.c == x.nu) {
      x.left -= kSegment;
      if (x.left > 0) next_item(x);
    }
  };
  At now;
  now.left = u_end - u_begin;
  enter(now, seq0);
  {
    const int places = now.nu + kSegment;
    now.kvh = (u_begin - before) / places;
    now.c = u_begin - before - now.kvh * places;
    if (now.c >= now.nu) {  // the run begins in an item's end places
      now.left -= places - now.c;
      if (now.left > 0) next_item(now);
    }
  }
  At ahead = now;

  // this warp's tile of a unit lies within one page: its table entry
  auto page_of = [&](const At& x) {
    const int key0 = x.c * kDecUnit + warp * kDecTile;
    return x.left > 0 && key0 < x.s.k ? a.page_table[x.seq * a.table_ld + (key0 >> p.page_shift)] : 0;
  };
  int page = page_of(ahead);
  bool ok = true;       // false: a wait of this warp ran out; it loads and takes no more tiles, its results are NaN
  uint32_t loaded = 0;  // bit i: stage i has a tile on its way or not yet taken
  auto load_next = [&](int stage) {
    if (ahead.left <= 0 || !ok) return;
    const int key0 = ahead.c * kDecUnit + warp * kDecTile;
    if (key0 < ahead.s.k) loaded |= 1u << stage;
    if (key0 < ahead.s.k && lane == 0) {
      const bool held = page >= 0 && page < a.num_pages;
      if (!held) record_bad_index(p.status);
      const int z = held ? page : (1 << 30);  // past every cache: zeros
      const int row = key0 & ((1 << p.page_shift) - 1);
      uint8_t* dst = ring + stage * kStageBytes;
      mbar_arrive_expect_tx(&full[stage], kStageBytes);
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        tma_load_4d(dst + c * 2048, &tmK, &full[stage], c * 64, ahead.kvh, row, z);
        tma_load_4d(dst + C::kTileBytes + c * 2048, &tmV, &full[stage], c * 64, ahead.kvh, row, z);
      }
    }
    step(ahead);
    page = page_of(ahead);
  };
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) load_next(i);

  // queries as mma operands: rows lane/4 and lane/4 + 8
  uint32_t qf[KT][4];
  auto load_q = [&](const At& x) {
    const int rows = x.s.q * p.group;
    const int r0 = lane >> 2, r1 = r0 + 8;
    const uint16_t* q = static_cast<const uint16_t*>(a.q);
    const int i0 = r0 / p.group, i1 = r1 / p.group;
    const uint16_t* p0 = q + static_cast<long long>(x.s.q0 + i0) * a.q_ts +
                         static_cast<long long>(x.kvh * p.group + (r0 - i0 * p.group)) * a.q_hs + (lane & 3) * 2;
    const uint16_t* p1 = q + static_cast<long long>(x.s.q0 + i1) * a.q_ts +
                         static_cast<long long>(x.kvh * p.group + (r1 - i1 * p.group)) * a.q_hs + (lane & 3) * 2;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      qf[k][0] = r0 < rows ? *reinterpret_cast<const uint32_t*>(p0 + k * 16) : 0u;
      qf[k][1] = r1 < rows ? *reinterpret_cast<const uint32_t*>(p1 + k * 16) : 0u;
      qf[k][2] = r0 < rows ? *reinterpret_cast<const uint32_t*>(p0 + k * 16 + 8) : 0u;
      qf[k][3] = r1 < rows ? *reinterpret_cast<const uint32_t*>(p1 + k * 16 + 8) : 0u;
    }
  };
  if (now.left > 0) load_q(now);

  int stage = 0, free_stage = C::kStages - 1;
  uint32_t parity = 0;  // bit i: the phase of stage i that its next tile completes
  while (now.left > 0) {
    // ---- a segment: this run's part of one item
    const SeqLens s = now.s;
    const int kvh = now.kvh;
    const int c_begin = now.c;
    const int c_end = min(now.nu, now.c + now.left);
    const bool whole = c_begin == 0 && c_end == now.nu;
    // the item began before this run: its partial result takes the second place
    const bool earlier = now.left != u_end - u_begin && c_begin == 0;
    if (c_begin == 0 && threadIdx.x == 0) {
      const int last = runs.block_of(u_end - now.left + now.nu - 1);
      p.spans[now.seq * a.kv_heads + kvh] =
          make_int2(2 * static_cast<int>(blockIdx.x) + (earlier ? 1 : 0), last - static_cast<int>(blockIdx.x) + 1);
    }
    const int rows = s.q * p.group;
    // keys row r admits: up to its token's own position (causal)
    const int lim0 = a.causal ? s.k - s.q + (lane >> 2) / p.group + 1 : s.k;
    const int lim1 = a.causal ? s.k - s.q + ((lane >> 2) + 8) / p.group + 1 : s.k;
    const int lim_min = a.causal ? s.k - s.q + 1 : s.k;

    float m0 = -INFINITY, m1 = -INFINITY, l0 = ok ? 0.f : NAN, l1 = l0;
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

    for (int c = c_begin; c < c_end; ++c) {
      __syncwarp();           // every lane is done with the tile before this one:
      load_next(free_stage);  // its stage is refilled
      const int key0 = c * kDecUnit + warp * kDecTile;
      if (key0 < s.k && ok &&
          !__all_sync(0xffffffffu, mbar_wait(&full[stage], (parity >> stage) & 1, p.status, kDevTimeoutProducer))) {
        ok = false;
        l0 = l1 = NAN;
      }
      if (key0 < s.k && ok) {
        parity ^= 1u << stage;
        loaded &= ~(1u << stage);
        uint8_t* tile = ring + stage * kStageBytes;
        const uint32_t kt = smem_u32(tile);
        const uint32_t vt = kt + C::kTileBytes;
        if (key0 + kDecTile > s.k) {
          // the sequence ends inside the tile: zero the value rows behind it
          const int valid = s.k - key0;
#pragma unroll
          for (int h = 0; h < HD / 64; ++h)
            for (int i = valid * 8 + lane; i < kDecTile * 8; i += 32)
              *reinterpret_cast<uint4*>(tile + C::kTileBytes + h * 2048 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();  // before the stage's next copy
          __syncwarp();
        }
        // S = Q K^T: two 8-key column tiles; matrices (keys 0-7 | 8-15) x (k 0-7 | 8-15)
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
        {
          const int r = (lane & 7) + ((lane >> 4) << 3);
          const int hi = (lane >> 3) & 1;
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            uint32_t b[4];
            ldsm4(kt + (k >> 2) * 2048 + r * 128 + (((2 * (k & 3) + hi) ^ (r & 7)) << 4), b);
            mma16816<DT>(s0, qf[k], b[0], b[1]);
            mma16816<DT>(s1, qf[k], b[2], b[3]);
          }
        }
        if (key0 + kDecTile > lim_min) {
          const int kc = key0 + (lane & 3) * 2;
          s0[0] = kc < lim0 ? s0[0] : -INFINITY;
          s0[1] = kc + 1 < lim0 ? s0[1] : -INFINITY;
          s1[0] = kc + 8 < lim0 ? s1[0] : -INFINITY;
          s1[1] = kc + 9 < lim0 ? s1[1] : -INFINITY;
          s0[2] = kc < lim1 ? s0[2] : -INFINITY;
          s0[3] = kc + 1 < lim1 ? s0[3] : -INFINITY;
          s1[2] = kc + 8 < lim1 ? s1[2] : -INFINITY;
          s1[3] = kc + 9 < lim1 ? s1[3] : -INFINITY;
        }
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
            ldsm4t(vt + (n >> 2) * 2048 + r * 128 + (((2 * (n & 3) + hi) ^ (r & 7)) << 4), b);
            mma16816<DT>(o[2 * n], pf, b[0], b[1]);
            mma16816<DT>(o[2 * n + 1], pf, b[2], b[3]);
          }
        }
      }
      free_stage = stage;
      stage = stage + 1 == C::kStages ? 0 : stage + 1;
      step(now);
    }
    // the next item's queries, on their way during the join
    if (now.left > 0) load_q(now);

    // ---- join the four warps, 8 rows at a time: each leaves its maximum, sum
    // and O; 16 threads per row add them up in warp order
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const int r0 = lane >> 2;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half * 8 >= rows) break;
      __syncthreads();  // the buffer's last readers are done
      // column groups of 8 are permuted by row, which spreads the banks
      float* so = s_o + (warp * 8 + r0) * HD;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
        *reinterpret_cast<float2*>(so + ((i ^ (r0 & 3)) * 8) + (lane & 3) * 2) =
            make_float2(o[i][2 * half], o[i][2 * half + 1]);
      if ((lane & 3) == 0) {
        s_m[warp][r0] = half ? m1 : m0;
        s_l[warp][r0] = half ? l1 : l0;
      }
      __syncthreads();
      const int row = threadIdx.x >> 4;  // 0..7
      const int r = half * 8 + row;
      if (r < rows) {
        float M = -INFINITY, L = 0.f, f[kDecWarps];
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, s_m[w][row]);
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
          f[w] = s_m[w][row] == -INFINITY ? 0.f : ex2_f32(s_m[w][row] - M);
          L += s_l[w][row] * f[w];
        }
        // 0: no keys for this row (or every score -inf); NaN goes on into the
        // result, the log-sum-exp and the join
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const float lg = L == 0.f ? -INFINITY : M + __log2f(L);
        const int tok = s.q0 + r / p.group, head = kvh * p.group + r % p.group;
        const int col = threadIdx.x & 15;
        const long long place = 2ll * blockIdx.x + (earlier ? 1 : 0);
#pragma unroll
        for (int g = 0; g < HD / 64; ++g) {  // 4 columns each
          const int cc = (g * 16 + col) * 4;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(s_o + (w * 8 + row) * HD + (cc ^ ((row & 3) * 8)));
            x.x = fmaf(y.x, f[w], x.x);
            x.y = fmaf(y.y, f[w], x.y);
            x.z = fmaf(y.z, f[w], x.z);
            x.w = fmaf(y.w, f[w], x.w);
          }
          x = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
          if (!whole) {
            *reinterpret_cast<float4*>(p.o_part + (place * kDecRows + r) * HD + cc) = x;
          } else if (a.out_f32) {
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + static_cast<long long>(tok) * a.o_ts +
                                       static_cast<long long>(head) * a.o_hs + cc) = x;
          } else {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + static_cast<long long>(tok) * a.o_ts +
                                      static_cast<long long>(head) * a.o_hs + cc) =
                make_uint2(pack2<DT>(x.x, x.y), pack2<DT>(x.z, x.w));
          }
        }
        if (col == 0) {
          if (!whole) {
            p.l_part[place * kDecRows + r] = lg;
          } else if (a.lse != nullptr) {
            a.lse[static_cast<long long>(head) * a.tokens + tok] = lg * 0.69314718055994531f;
          }
        }
      }
    }
  }
  // after a wait that ran out: the copies still on their way land before the
  // block's memory is given up (bounded, whatever the status says)
  if (!ok)
    for (int i = 0; i < C::kStages; ++i)
      if (loaded >> i & 1) mbar_wait(&full[i], (parity >> i) & 1, nullptr, kDevTimeoutDrain);
}

// Joins the partial results of every item that more than one block worked on,
// and writes the rows of sequences without keys (out 0, log-sum-exp -inf).
// One block per (sequence, key head) and ROWS rows, 8 / ROWS warps to each:
// the maximum first, then each warp adds up its share of the results, eight of
// them requested at a time, and the warps' sums are added in warp order. What
// bounds it is the chain of latencies (lengths, maximum, results), so a long
// join is spread over the warps; a call with more rows than blocks fit on the
// card takes several to a block. Where an item's partial results are is what
// the block that began it left in `spans`. (Found from the lengths of all
// sequences, a row to a block: 200 sequences of 100 keys, 64 heads over 8, hd 64,
// 83 us against 25, 256 of 600, 32 over 8, hd 128, 150 against 113.)
constexpr int kJoinWarps = 8;
constexpr int kJoinCtasPerSm = 8;  // that are resident

template <int HD, int DT, int ROWS>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_combine_kernel(const __grid_constant__ DecodeK p, int blocks) {
  constexpr int E = HD / 32;
  extern __shared__ float s_w[];  // [warps][blocks] log-sum-exps of a row's partial results
  __shared__ float s_o[kJoinWarps][HD];
  __shared__ float s_l[kJoinWarps], s_max[kJoinWarps];
  const SeqArgs& a = p.a;
  pdl_wait();
  pdl_trigger();
  const int seq = blockIdx.x / a.kv_heads, kvh = blockIdx.x - seq * a.kv_heads;
  const int lane = lane_id(), warp = warp_id();
  constexpr int kStep = kJoinWarps / ROWS;  // warps of a row
  const int r0 = blockIdx.y * ROWS, r = r0 + warp % ROWS;
  const SeqLens s = decode_lens(a, p.group, p.page_shift, seq);
  if (s.bad && kvh == 0 && r0 == 0 && threadIdx.x == 0) record_bad_index(p.status);
  const int end = s.q * p.group;
  if (r0 >= end) return;
  // An item's first partial result is in the first place of its block, or in
  // the second if that block's run began before the item; the others are in
  // the first places of the blocks after it. Items without keys have none.
  int2 span = make_int2(0, 0);
  if (units_of(s) > 0) {
    span = p.spans[blockIdx.x];
    if (span.y == 1) return;  // one block saw all of it and wrote the result
  }
  int n = span.y;
  auto part = [&](int i) -> long long { return i == 0 ? span.x : (span.x & ~1) + 2 * i; };
  if (r >= end) n = 0;
  float m = -INFINITY;
  float* lg = s_w + warp * blocks;
#pragma unroll 4
  for (int i = lane; i < n; i += 32) {
    const float x = p.l_part[part(i) * kDecRows + r];
    lg[i] = x;
    m = fmaxf(m, x);
  }
  __syncwarp();
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float l = 0.f, acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.f;
#pragma unroll 8
  for (int i = warp / ROWS; i < n; i += kStep) {
    const float w = lg[i] == -INFINITY ? 0.f : ex2_f32(lg[i] - m);
    const float* src = p.o_part + (part(i) * kDecRows + r) * HD + lane * E;
    l += w;
    if constexpr (E == 4) {
      const float4 x = *reinterpret_cast<const float4*>(src);
      acc[0] = fmaf(w, x.x, acc[0]);
      acc[1] = fmaf(w, x.y, acc[1]);
      acc[2] = fmaf(w, x.z, acc[2]);
      acc[3] = fmaf(w, x.w, acc[3]);
    } else {
      const float2 x = *reinterpret_cast<const float2*>(src);
      acc[0] = fmaf(w, x.x, acc[0]);
      acc[1] = fmaf(w, x.y, acc[1]);
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) s_o[warp][lane * E + i] = acc[i];
  if (lane == 0) {
    s_l[warp] = l;
    s_max[warp] = m;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * HD; i += kJoinWarps * 32) {
    const int row = i / HD, col = i - row * HD;
    if (r0 + row >= end) return;
    float x = 0.f;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kStep; ++w) {
      l += s_l[row + w * ROWS];
      x += s_o[row + w * ROWS][col];
    }
    x = l == 0.f ? 0.f : x / l;
    const int tok = s.q0 + (r0 + row) / p.group, head = kvh * p.group + (r0 + row) % p.group;
    const long long at = static_cast<long long>(tok) * a.o_ts + static_cast<long long>(head) * a.o_hs + col;
    if (a.out_f32) {
      static_cast<float*>(a.out)[at] = x;
    } else {
      static_cast<uint16_t*>(a.out)[at] = static_cast<uint16_t>(pack2<DT>(x, 0.f) & 0xffffu);
    }
    if (a.lse != nullptr && col == 0)
      a.lse[static_cast<long long>(head) * a.tokens + tok] =
          l == 0.f ? -INFINITY : (s_max[row] + __log2f(l)) * 0.69314718055994531f;
  }
}

// Blocks of a call: every SM's share, but no more than there can be units.
int decode_blocks(const SeqArgs& a) {
  const long long units = ((a.max_k + kDecUnit - 1) / kDecUnit) * a.batch * a.kv_heads;
  const long long most = static_cast<long long>(kDecCtasPerSm) * device_sm_count();
  return static_cast<int>(units < 1 ? 1 : units < most ? units : most);
}

template <int HD, int DT>
int launch_decode(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeK& k, int blocks, cudaStream_t stream) {
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
  cudaError_t e = launch_k(kern, dim3(blocks), dim3(kDecWarps * 32), C::kBytes, stream, tk, tv, k);
  if (e == cudaSuccess) {
    const long long items = k.a.batch * k.a.kv_heads;
    const int most = static_cast<int>(k.a.max_q * k.group);
    int rows = 1;  // per join block
    while (rows < kJoinWarps && rows < most && items * ((most + rows - 1) / rows) > kJoinCtasPerSm * device_sm_count())
      rows *= 2;
    auto join = rows == 1   ? paged_combine_kernel<HD, DT, 1>
                : rows == 2 ? paged_combine_kernel<HD, DT, 2>
                : rows == 4 ? paged_combine_kernel<HD, DT, 4>
                            : paged_combine_kernel<HD, DT, 8>;
    e = launch_k(join, dim3(static_cast<unsigned>(items), (most + rows - 1) / rows), dim3(kJoinWarps * 32),
                 kJoinWarps * blocks * sizeof(float), stream, k, blocks);
  }
  if (e != cudaSuccess) return set_error(TF_ERR_LAUNCH, "paged decode launch: %s", cudaGetErrorString(e));
  return TF_OK;
}

}  // namespace

bool paged_is_decode(const SeqArgs& a) { return a.max_q * (a.heads / a.kv_heads) <= kDecRows; }

long long paged_decode_workspace(const SeqArgs& a) {
  return static_cast<long long>(decode_blocks(a)) * 2 * kDecRows * (a.head_dim + 1) * 4 + a.batch * a.kv_heads * 8;
}

int paged_decode(const SeqArgs& a, cudaStream_t stream) {
  if ((a.max_pages * a.page_size / kDecUnit + 1 + kSegment) * a.batch * a.kv_heads >= (1ll << 31))
    return set_error(TF_ERR_SHAPE, "paged attention: a table of %lld x %lld pages is out of range", a.batch, a.max_pages);
  DecodeK k = {};
  k.a = a;
  k.group = a.heads / a.kv_heads;
  while ((1ll << k.page_shift) < a.page_size) ++k.page_shift;
  k.scale_log2 = a.scale * 1.4426950408889634f;
  const int blocks = decode_blocks(a);
  k.o_part = static_cast<float*>(a.workspace);
  k.l_part = k.o_part + static_cast<long long>(blocks) * 2 * kDecRows * a.head_dim;
  k.spans = reinterpret_cast<int2*>(k.l_part + static_cast<long long>(blocks) * 2 * kDecRows);
  k.status = device_status_ptr();
  if (k.status == nullptr) return last_error_code();
  CUtensorMap tk, tv;
  int rc = make_tmap_4d_f16(&tk, a.k, {a.head_dim, a.kv_heads, a.page_size, a.num_pages}, {a.k_hs, a.k_ts, a.k_ps},
                            {64, 1, kDecTile, 1});
  if (rc) return rc;
  rc = make_tmap_4d_f16(&tv, a.v, {a.head_dim, a.kv_heads, a.page_size, a.num_pages}, {a.v_hs, a.v_ts, a.v_ps},
                        {64, 1, kDecTile, 1});
  if (rc) return rc;
  if (a.bf16)
    return a.head_dim == 64 ? launch_decode<64, kDtBF16>(tk, tv, k, blocks, stream)
                            : launch_decode<128, kDtBF16>(tk, tv, k, blocks, stream);
  return a.head_dim == 64 ? launch_decode<64, kDtF16>(tk, tv, k, blocks, stream)
                          : launch_decode<128, kDtF16>(tk, tv, k, blocks, stream);
}

}  // namespace tfb
