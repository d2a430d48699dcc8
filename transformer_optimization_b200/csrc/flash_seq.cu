// Attention of sequences of different lengths with grouped heads, on the
// 5th-generation tensor cores: queries packed end to end; keys and values
// packed the same way, or in a paged cache.
//
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j      over the keys of i's own sequence,
//   causal: j <= i + (keys - queries), the last query stands at the last key
//
// The pipeline is that of flash_fwd_tcgen05 (flash_attn.cu): two query tiles
// per CTA, S = Q K^T into a ring of TMEM slots, softmax with lazy rescaling in
// registers, P back over its S slot, O += P V from TMEM. Bound by the exp unit at
// hd 64 (busy in 72% of the cycles; 8 sequences of 2048, 16 heads: 0.189 ms, 726
// TFLOP/s) and by the chain of S, softmax and P V at hd 128 (exp unit and tensor
// pipe both busy in 61%; 4 sequences of 4096, 16 heads over 2, causal: 0.267 ms,
// 1028 TFLOP/s). What differs:
//
// * A tile's 128 rows are (token, query head of the group) pairs, so all query
//   heads that share a key head read each K and V tile once: a 4-D tensor map
//   over [token][key head][group head][64 columns] fills 128 / G tokens times
//   G heads per tile in one copy. G heads of one token see the same keys, so
//   the causal limit is per token and a tile spans fewer positions.
// * More items (two tiles of a sequence, a key head) than SMs: seq_plan_kernel
//   lists the tiles by falling number of key blocks and CTAs draw items from
//   the list by a counter, so a long item never starts last. Where the longest
//   is longer than an SM's share of all and half of that again, long tiles are
//   cut into key ranges of half a share (32 sequences of 5 tokens, 64 heads
//   over 8, hd 128, one of 100 000 keys and the others of 1000: 158 us, uncut
//   840). Fewer items: CTA c takes item c, found by a warp scan over the
//   lengths, and where keys are long every tile is cut into as many ranges as
//   fill the SMs. Either way the call needs no host copy of the lengths and
//   keeps nothing, and cuts depend on lengths alone: results repeat bit for
//   bit. (Cutting all work into one equal run per SM instead, at key blocks
//   inside items, was slower: 16 ragged prompts 57 us against 46. SMs that are
//   at different places in the code stall each other's instruction fetch,
//   items in order of size keep them together.)
// * The warps' rings and barriers run on from item to item, so the next item's
//   Q, K and V arrive and its first scores are formed while the last one's
//   softmax and stores still run (a CTA per item spent 5.5 us, hd 64, to
//   7.5 us, hd 128, on start and end, as long as four key blocks take).
// * A key range leaves its normalised fp32 result and log-sum-exp in the
//   workspace; seq_combine_kernel joins a tile's ranges in order.
// * Key blocks start at the sequence's first key, and a copy may run into the
//   next sequence or past a page's end. Such scores are masked as usual; such
//   V rows are zeroed in shared memory before the product (0 * NaN would
//   otherwise reach the result), by the V producer, in the last block of a
//   sequence only.
// * Paged: a key block is 128 (64) / page_size copies, one per page (one copy of a
//   part of a larger page), issued by as many lanes; page indices are read one
//   block ahead. An index outside the cache reads zeros and is reported.
#include "attn_common.cuh"
#include "common.cuh"
#include "launch.h"

namespace tfb {
namespace {

// Where results go.
struct SeqOut {
  void* out;
  long long o_ts, o_hs;
  float* lse;
  float* o_part;    // [slot][HD / 4][256 rows][4]: results of key ranges
  float* lse_part;  // [slot][256 rows], natural log
  int tokens, out_f32;
};

struct SeqWork {
  int seq, tile;  // seq < 0: no more work
  int q0, q_len;  // first query token, queries
  int k0, k_len;  // packed: first key token; keys
  int jb, je;     // key blocks
  int slot;       // where a key range's result goes; -1: the range is all
  int kvh;        // key head
  int n0, n1;     // of the key blocks, those that each tile has
  int ranges;     // of the tile
};

struct SeqK {
  SeqOut o;
  const int* cu_q;
  const int* cu_k;
  const int* kv_lens;
  const int* page_table;
  long long table_ld;
  int num_pages, page_shift, page_box;  // page_box: rows of a page one copy takes
  long long page_cap;                   // keys a page table row can hold
  int batch, heads, group, tokens, k_tokens, max_q;
  int tok_tile;  // tokens per 128-row tile
  int bn_shift;  // log2 of the keys per block
  float scale_log2;
  int causal;
  int kv_heads, max_tiles;
  int splits;       // without a list: key ranges per tile
  int max_slots;    // with a list: key ranges (of all key heads together) that tiles may be cut into
  int* plan;        // null, or: entries in the list, next item, cut tiles, 0, the cut tiles' first entries
  SeqWork* list;    // with a plan: [max_tiles + max_slots]; with splits: [max_tiles], for the join
  int* status;
};

// Register split (see attn_common.cuh): the item loop needs 56 registers in
// the producer and MMA warps, and the softmax fits 224.
constexpr int kSeqRegsLow = 56;
constexpr int kSeqRegsHigh = 224;
static_assert(128 * kSeqRegsLow + 256 * kSeqRegsHigh <= kAttnThreads * kRegsLaunch, "register split exceeds the pool");

// Keys per block, a power of two. hd 64: 128. hd 128: O takes 256 of the 512
// TMEM columns, and what is left holds two slots of 128 or four of 64. With two,
// a tile's next S waits for its last P V, and the softmax stood for 2050 of 4450
// cycles a block; with four of 64 the next S is formed meanwhile (one prompt of
// 16 384 tokens, 16 heads over 2: 1035 us, with two slots 1140).
// Blocks of 64 for hd 64 too, six slots: 8 sequences of 1025 to 2047 tokens 110
// us against 101, there is more to do per block and nothing more to hide.
constexpr int seq_block(int hd) { return hd == 64 ? 128 : 64; }

template <int HD>
struct SeqCfg {
  static constexpr int kBN = seq_block(HD);
  static constexpr int kNS = HD == 64 ? 3 : 4;
  static constexpr int kNQ = HD == 64 ? 2 : 1;      // items whose queries fit
  static constexpr int kStages = 4;                 // of K and of V
  static constexpr int kQBytes = kAttnBM * HD * 2;  // a query tile; 64 columns of it: 16384
  static constexpr int kKvHalf = kBN * 128;         // 64 columns of a key block
  static constexpr int kKvBytes = kBN * HD * 2;
  static constexpr int kQOff = 0;
  static constexpr int kKOff = kQOff + kNQ * kAttnTiles * kQBytes;
  static constexpr int kVOff = kKOff + kStages * kKvBytes;
  static constexpr int kStageOff = kVOff + kStages * kKvBytes;  // 4 KB per softmax warp for the stores
  static constexpr int kBarOff = kStageOff + 8 * 4096;
  // item_full/empty[2], s_done[2], q_full/empty[NQ], v_tail, k_full/empty, v_full/empty,
  // s_full[NS], p_full[NS], drain[2], pv_done[NS], o_done[2]
  static constexpr int kNumBars = 6 + 2 * kNQ + 1 + 4 * kStages + 3 * kNS + 4;
  static constexpr int kBytes = kBarOff + kNumBars * 8 + 16;
  static constexpr int kAlloc = kBytes + 1024;
  static constexpr uint32_t kTmS = 0;
  static constexpr uint32_t kTmO = kNS * kBN;
  static_assert(kNS * kBN + kAttnTiles * HD <= 512, "TMEM budget");
};

// Queries and keys of sequence b, bounded by what the call's arrays hold. A
// bound that bites is an error of the caller's: it is reported, and nothing
// outside the arrays is read or written.
template <bool PAGED>
__device__ __forceinline__ SeqWork seq_lens(const SeqK& p, int b, bool& bad) {
  SeqWork w = {};
  w.seq = b;
  const int c0 = p.cu_q[b], c1 = p.cu_q[b + 1];
  w.q0 = min(max(c0, 0), p.tokens);
  w.q_len = min(min(max(c1, w.q0), p.tokens) - w.q0, p.max_q);
  bad = c0 < 0 || w.q_len != c1 - c0;
  if constexpr (PAGED) {
    const int kv = p.kv_lens[b];
    w.k0 = 0;
    w.k_len = kv < 0 ? 0 : (kv > p.page_cap ? static_cast<int>(p.page_cap) : kv);
    bad = bad || w.k_len != kv;
  } else {
    const int d0 = p.cu_k[b], d1 = p.cu_k[b + 1];
    w.k0 = min(max(d0, 0), p.k_tokens);
    w.k_len = min(max(d1, w.k0), p.k_tokens) - w.k0;
    bad = bad || d0 < 0 || w.k_len != d1 - d0;
  }
  return w;
}

__device__ __forceinline__ int tile_blocks(const SeqK& p, const SeqWork& w, int t0) {
  int k_end = t0 < w.q_len ? w.k_len : 0;
  if (p.causal && k_end > 0) k_end = min(k_end, min(t0 + p.tok_tile, w.q_len) + w.k_len - w.q_len);
  return k_end <= 0 ? 0 : (k_end + (1 << p.bn_shift) - 1) >> p.bn_shift;
}
// The `at`-th CTA tile (2 * tok_tile tokens) of all sequences, one warp.
template <bool PAGED>
__device__ __forceinline__ SeqWork find_tile(const SeqK& p, int at) {
  const int lane = lane_id();
  const int span = 2 * p.tok_tile;
  int run = 0;
  for (int base = 0; base < p.batch; base += 32) {
    const int b = base + lane;
    SeqWork w = {};
    bool bad = false;
    int n = 0;
    if (b < p.batch) {
      w = seq_lens<PAGED>(p, b, bad);
      n = (w.q_len + span - 1) / span;
      if (bad) record_bad_index(p.status);
    }
    int inc = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, run + inc > at);
    if (hit != 0) {
      const int l = __ffs(hit) - 1;
      SeqWork r = {};
      r.seq = base + l;
      r.tile = at - run - __shfl_sync(0xffffffffu, inc - n, l);
      r.q0 = __shfl_sync(0xffffffffu, w.q0, l);
      r.q_len = __shfl_sync(0xffffffffu, w.q_len, l);
      r.k0 = __shfl_sync(0xffffffffu, w.k0, l);
      r.k_len = __shfl_sync(0xffffffffu, w.k_len, l);
      return r;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  SeqWork none = {};
  none.seq = -1;
  return none;
}

// The item's blocks of each tile.
__device__ __forceinline__ void set_blocks(const SeqK& p, SeqWork& w) {
  const int t0 = w.tile * 2 * p.tok_tile;
  w.n0 = max(min(tile_blocks(p, w, t0), w.je) - w.jb, 0);
  w.n1 = max(min(tile_blocks(p, w, t0 + p.tok_tile), w.je) - w.jb, 0);
}

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------

constexpr int kPlanThreads = 1024;
constexpr int kClasses = 64;

// Inclusive sum over the block's threads; `total` is the block's.
__device__ __forceinline__ int block_scan(int x, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += up;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int w = s_warp[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, w, d);
    if (lane >= d) w += up;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  __syncthreads();
  return x + (warp > 0 ? before : 0);
}

// Lists the call's tiles by falling number of key blocks (counting sort over
// kClasses classes), and sets the item counter to the CTAs' first items. One
// block. If tiles may be cut and the longest has half as many blocks again as an
// SM's share of all, tiles longer than half that share become ranges of at most
// that: fewer than 2 * total / range <= 4 per SM, which is what the workspace
// holds (a tile of n > range blocks becomes fewer than 2 n / range). The order within a class depends on timing, results do not.
constexpr int kMinRange = 768;  // keys; a shorter range costs more than it evens out
// Keys a sequence may have from which on the call makes room for cuts, and so
// launches their join, needed or not. Room for them always costs calls that cut
// nothing 1.3 to 1.6 us (16 ragged prompts of up to 2048 tokens 70.2 -> 71.6, 60
// of 100 tokens 25.8 -> 27.1) and 39 or 78 MB of workspace; below the bound a
// long sequence among short ones stays whole (32 sequences of 5 tokens, 64
// heads over 8, hd 128, 1000 keys and one of 4000: 60 us, cut 41; of 8000: 96, cut
// 58; of 2000: 41, cut 43). At 8192 the prompts of ordinary batches pay nothing.
constexpr int kCutKeys = 8192;

template <bool PAGED>
__global__ void __launch_bounds__(kPlanThreads) seq_plan_kernel(const __grid_constant__ SeqK p, int ctas) {
  __shared__ int s_q0[kPlanThreads], s_q[kPlanThreads], s_k0[kPlanThreads], s_k[kPlanThreads];
  __shared__ int s_end[kPlanThreads];  // tiles of the round's sequences up to each
  __shared__ int s_place[kClasses];    // entries of a class, then the place of its next
  __shared__ int s_warp[32];
  __shared__ int s_most, s_slots, s_joins;
  __shared__ unsigned long long s_sum;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int span = 2 * p.tok_tile;
  if (tid < kClasses) s_place[tid] = 0;
  if (tid == 0) {
    s_most = 1;
    s_slots = s_joins = 0;
    s_sum = 0;
  }
  pdl_wait();
  pdl_trigger();
  __syncthreads();
  int most = 1;
  unsigned long long sum = 0;  // blocks, every tile taken as long as its sequence's last (no less than there are)
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    bool bad;
    const SeqWork w = seq_lens<PAGED>(p, b, bad);
    if (bad) record_bad_index(p.status);
    if (w.q_len > 0) {
      const int last = tile_blocks(p, w, (w.q_len - 1) / p.tok_tile * p.tok_tile);
      most = max(most, last);
      sum += static_cast<unsigned long long>((w.q_len + span - 1) / span) * last;
    }
    if (b < kPlanThreads) {
      s_q0[tid] = w.q0;
      s_q[tid] = w.q_len;
      s_k0[tid] = w.k0;
      s_k[tid] = w.k_len;
    }
  }
  most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) {
    atomicMax(&s_most, most);
    atomicAdd(&s_sum, sum);
  }
  __syncthreads();
  most = s_most;
  int range = 0x7fffffff;
  if (p.max_slots > 0) {
    const unsigned long long share = s_sum * p.kv_heads / ctas + 1;
    if (2 * most > 3 * share) range = max(static_cast<int>((share + 1) / 2), kMinRange >> p.bn_shift);
  }
  const float per_class = (kClasses - 1) / static_cast<float>(min(most, range));

  // tile i of the sequences in shared memory
  auto tile_of = [&](int base, int i) {
    int lo = 0, hi = kPlanThreads - 1;  // the first sequence whose end is past i
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_end[mid] > i) {
        hi = mid;
      } else {
        lo = mid + 1;
      }
    }
    SeqWork x = {};
    x.seq = base + lo;
    x.tile = i - (lo > 0 ? s_end[lo - 1] : 0);
    x.q0 = s_q0[lo];
    x.q_len = s_q[lo];
    x.k0 = s_k0[lo];
    x.k_len = s_k[lo];
    x.je = 0x7fffffff;
    set_blocks(p, x);
    x.je = max(x.n0, x.n1);
    x.slot = -1;
    x.ranges = x.je > range ? (x.je + range - 1) / range : 1;
    return x;
  };
  int entries = 0;
  SeqWork kept = {};  // this thread's tile of the only round, from pass to pass
  // pass 0 counts the classes, pass 1 places the entries
  for (int pass = 0; pass < 2; ++pass) {
    for (int base = 0; base < p.batch; base += kPlanThreads) {
      if (p.batch > kPlanThreads) {
        SeqWork w = {};
        bool bad;
        if (base + tid < p.batch) w = seq_lens<PAGED>(p, base + tid, bad);
        s_q0[tid] = w.q0;
        s_q[tid] = w.q_len;
        s_k0[tid] = w.k0;
        s_k[tid] = w.k_len;
      }
      if (pass == 0 || p.batch > kPlanThreads) {
        const int n = base + tid < p.batch ? (s_q[tid] + span - 1) / span : 0;
        int round;
        s_end[tid] = block_scan(n, s_warp, round);
        __syncthreads();
      }
      const int round = s_end[kPlanThreads - 1];
      for (int i = tid; i < round; i += kPlanThreads) {
        const bool keep = p.batch <= kPlanThreads && i == tid;
        SeqWork x = pass == 1 && keep ? kept : tile_of(base, i);
        if (keep) kept = x;
        const int len = (x.je + x.ranges - 1) / x.ranges;
        const int cls = min(max(kClasses - 1 - static_cast<int>(len * per_class), 0), kClasses - 1);
        int at = atomicAdd(&s_place[cls], x.ranges);
        if (pass == 0) continue;
        if (x.ranges == 1) {
          if (at < p.max_tiles + p.max_slots) p.list[at] = x;
          continue;
        }
        const int slot = atomicAdd(&s_slots, x.ranges);
        const int join = atomicAdd(&s_joins, 1);
        if (slot + x.ranges > p.max_slots || at + x.ranges > p.max_tiles + p.max_slots) {
          // more tiles than tokens allow: sequences that lie over one another
          // (reported above). The list ends here, no entry is left unwritten.
          x.seq = -1;
          for (int k = 0; k < x.ranges && at + k < p.max_tiles + p.max_slots; ++k) p.list[at + k] = x;
          if (join < p.max_slots / 2) p.plan[4 + join] = -1;
          continue;
        }
        p.plan[4 + join] = at;
        const int all = x.je;
        x.je = 0;
        for (int k = 0; k < x.ranges; ++k, ++at) {
          x.jb = x.je;
          x.je = min(x.jb + len, all);
          x.slot = slot + k;
          set_blocks(p, x);
          p.list[at] = x;
        }
      }
      __syncthreads();
    }
    if (pass == 0) {
      if (warp == 0) {  // counts -> first places
        int run = 0;
        for (int i = 0; i < kClasses; i += 32) {
          const int c = s_place[i + lane];
          int inc = c;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += up;
          }
          s_place[i + lane] = run + inc - c;
          run += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) s_warp[0] = run;
      }
      __syncthreads();
      entries = s_warp[0];
      __syncthreads();
    }
  }
  if (tid == 0) {
    p.plan[0] = min(entries, p.max_tiles + p.max_slots);
    p.plan[1] = ctas;
    p.plan[2] = min(s_joins, p.max_slots / 2);
  }
}

// mbar_wait with little code: these kernels are sensitive to their size (two
// softmax groups and four other warps, each in another part of it), and every
// wait is inlined. Bounded by the SM's clock, 2 s at 2 GHz.
__device__ __forceinline__ bool seq_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long end = clock64() + 4000000000ll;
  while (!mbar_try_wait(bar, parity)) {
    if (clock64() > end) {
      record_error(status, code);
      return false;
    }
  }
  return true;
}

// two floats in a register pair, and operations on both
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void split_pair(uint64_t d, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(d));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <int HD, int DT, bool PAGED>
__global__ void __launch_bounds__(kAttnThreads, 1)
    flash_seq_tcgen05(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ SeqK p) {
  using C = SeqCfg<HD>;
  constexpr int KS = C::kStages;
  constexpr int NS = C::kNS;
  constexpr int NQ = C::kNQ;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* item_full = bars;
  uint64_t* item_empty = item_full + 2;
  uint64_t* s_done = item_empty + 2;  // every S of the item has been formed
  uint64_t* q_full = s_done + 2;
  uint64_t* q_empty = q_full + NQ;
  uint64_t* v_tail = q_empty + NQ;  // the copy of a sequence's last, partial V block
  uint64_t* k_full = v_tail + 1;
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;
  uint64_t* v_empty = v_full + KS;
  uint64_t* s_full = v_empty + KS;
  uint64_t* p_full = s_full + NS;
  uint64_t* drain = p_full + NS;
  uint64_t* pv_done = drain + 2;
  uint64_t* o_done = pv_done + NS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2);
  __shared__ SeqWork s_item[2];
  __shared__ SeqOut s_out;  // read where it is used: kept out of the softmax loop's registers

  const int warp = warp_id();
  const int lane = lane_id();

  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&tmQ);
    tma_prefetch_map(&tmK);
    tma_prefetch_map(&tmV);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 11);  // warps 1 to 3 and 4 to 11
      mbar_init(&s_done[i], 1);
      mbar_init(&drain[i], 1);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < NQ; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    mbar_init(v_tail, 1);
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
    }
    fence_mbar_init();
    s_out = p.o;
  }
  // item i of the list
  auto listed_item = [&](int i, int items) {
    SeqWork x = {};
    x.seq = -1;
    if (i < items) {
      const int tile = i / p.kv_heads;
      x = p.list[tile];
      x.kvh = i - tile * p.kv_heads;
      if (x.slot >= 0) x.slot = x.slot * p.kv_heads + x.kvh;
    }
    return x;
  };
  // (up to here, and warps other than 3 up to the barrier, only this CTA's
  // shared memory and TMEM are touched)
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  } else if (warp == 3) {
    pdl_wait();
    SeqWork w;
    if (p.plan != nullptr) {
      w = listed_item(blockIdx.x, p.plan[0] * p.kv_heads);
    } else {
      const int per = p.kv_heads * p.splits;
      const int tile = blockIdx.x / per, rest = blockIdx.x - tile * per;
      w = find_tile<PAGED>(p, tile);
      const int range = rest / p.kv_heads;
      w.kvh = rest - range * p.kv_heads;
      w.jb = 0;
      w.je = 0x7fffffff;
      w.slot = -1;
      set_blocks(p, w);
      if (p.splits > 1) {
        const int len = (max(w.n0, w.n1) + p.splits - 1) / p.splits;
        w.jb = range * len;
        w.je = w.jb + len;
        w.slot = (tile * p.splits + range) * p.kv_heads + w.kvh;
        w.ranges = p.splits;
        set_blocks(p, w);
        if (lane == 0 && range == 0 && w.kvh == 0) p.list[tile] = w;
      }
    }
    if (lane == 0) s_item[0] = w;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  // one K or V block: this lane's copy (a page or a part of one, or the
  // whole block of packed keys) and the bytes of all copies
  auto boxes_of = [&](const SeqWork& w, int key) {
    return PAGED ? (min(C::kBN, w.k_len - key) + p.page_box - 1) / p.page_box : 1;
  };
  auto page_of = [&](const SeqWork& w, int key) {
    if constexpr (PAGED) {
      if (key >= w.k_len || lane >= boxes_of(w, key)) return 0;
      return p.page_table[w.seq * p.table_ld + ((key + lane * p.page_box) >> p.page_shift)];
    } else {
      return 0;
    }
  };
  auto load_block = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, const SeqWork& w, int key, int page) {
    const int n = boxes_of(w, key);
    const int rows = PAGED ? p.page_box : C::kBN;
    if (lane == 0) mbar_arrive_expect_tx(bar, n * rows * HD * 2);
    __syncwarp();
    if (lane < n) {
      int y, z;
      if constexpr (PAGED) {
        const bool ok = page >= 0 && page < p.num_pages;
        if (!ok) record_bad_index(p.status);
        y = (key + lane * rows) & ((1 << p.page_shift) - 1);
        z = ok ? page : (1 << 30);  // past every cache: zeros
      } else {
        y = w.k0 + key;
        z = 0;
      }
#pragma unroll
      for (int c = 0; c < HD / 64; ++c)
        tma_load_4d(dst + c * C::kKvHalf + lane * rows * 128, map, bar, c * 64, w.kvh, y, z);
    }
  };
  // item number `it` of this CTA, for the warps that do not draw items:
  // false when a wait ran out
  auto take_item = [&](int it, SeqWork& w, int code) {
    if (!seq_wait(&item_full[it & 1], (it >> 1) & 1, p.status, code)) return false;
    w = s_item[it & 1];
    return true;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSeqRegsLow));
    if (warp == 0) {
      // ---------------- items, Q and K ----------------
      SeqWork w = s_item[0];
      int kc = 0, qn = 0;  // K blocks and Q loads so far
      for (int it = 0;; ++it) {
        if (it >= 2 && !seq_wait(&item_empty[it & 1], ((it >> 1) - 1) & 1, p.status, kDevTimeoutProducer)) break;
        if (lane == 0) {
          if (it > 0) s_item[it & 1] = w;
          mbar_arrive(&item_full[it & 1]);
        }
        if (w.seq < 0) break;
        // the next item's number, on its way while this one is fetched
        int next = 0x7fffffff, items = 0;
        if (p.plan != nullptr) {
          items = p.plan[0] * p.kv_heads;
          if (lane == 0) next = atomicAdd(p.plan + 1, 1);
        }
        const int n = max(w.n0, w.n1);
        bool ok = true;
        int key = w.jb * C::kBN;
        int page = n > 0 ? page_of(w, key) : 0;
        for (int j = 0; j < n; ++j, ++kc, key += C::kBN) {
          const int s = kc % KS;
          const int ahead = j + 1 < n ? page_of(w, key + C::kBN) : 0;
          if (!(ok = seq_wait(&k_empty[s], ((kc / KS) & 1) ^ 1, p.status, kDevTimeoutProducer))) break;
          load_block(smem + C::kKOff + s * C::kKvBytes, &tmK, &k_full[s], w, key, page);
          page = ahead;
          if (j == 0) {
            const int qs = qn % NQ;
            if (!(ok = seq_wait(&q_empty[qs], ((qn / NQ) & 1) ^ 1, p.status, kDevTimeoutProducer))) break;
            if (lane == 0) {
              const int first = w.n0 > 0 ? 0 : 1, last = w.n1 > 0 ? 1 : 0;  // tiles with keys
              mbar_arrive_expect_tx(&q_full[qs], (last - first + 1) * p.tok_tile * p.group * HD * 2);
              for (int t = first; t <= last; ++t)
#pragma unroll
                for (int c = 0; c < HD / 64; ++c)
                  tma_load_4d(smem + C::kQOff + (qs * kAttnTiles + t) * C::kQBytes + c * 16384, &tmQ, &q_full[qs],
                              c * 64, 0, w.kvh, w.q0 + (2 * w.tile + t) * p.tok_tile);
            }
            ++qn;
          }
        }
        if (!ok) break;
        w = listed_item(__shfl_sync(0xffffffffu, next, 0), items);
      }
      for (int i = max(qn - NQ, 0); i < qn; ++i) seq_wait(&q_full[i % NQ], (i / NQ) & 1, p.status, kDevTimeoutDrain);
      for (int i = max(kc - KS, 0); i < kc; ++i) seq_wait(&k_full[i % KS], (i / KS) & 1, p.status, kDevTimeoutDrain);
    } else if (warp == 2) {
      // ---------------- V ----------------
      SeqWork w;
      int vc = 0, tails = 0;
      for (int it = 0; take_item(it, w, kDevTimeoutProducer); ++it) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[it & 1]);
        if (w.seq < 0) break;
        const int n = max(w.n0, w.n1);
        bool ok = true;
        int key = w.jb * C::kBN;
        int page = n > 0 ? page_of(w, key) : 0;
        for (int j = 0; j < n; ++j, ++vc, key += C::kBN) {
          const int s = vc % KS;
          const int ahead = j + 1 < n ? page_of(w, key + C::kBN) : 0;
          if (!(ok = seq_wait(&v_empty[s], ((vc / KS) & 1) ^ 1, p.status, kDevTimeoutProducer))) break;
          uint8_t* dst = smem + C::kVOff + s * C::kKvBytes;
          const int valid = w.k_len - key;
          if (valid >= C::kBN) {
            load_block(dst, &tmV, &v_full[s], w, key, page);
          } else {
            // the sequence ends inside this block: rows from `valid` on hold
            // another sequence's values, an unused part of a page or what the
            // stage held before
            load_block(dst, &tmV, v_tail, w, key, page);
            if (!(ok = seq_wait(v_tail, tails & 1, p.status, kDevTimeoutProducer))) break;
            ++tails;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
              for (int i = valid * 8 + lane; i < C::kBN * 8; i += 32)
                *reinterpret_cast<uint4*>(dst + c * C::kKvHalf + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[s]);
          }
          page = ahead;
        }
        if (!ok) break;
      }
      for (int i = max(vc - KS, 0); i < vc; ++i) seq_wait(&v_full[i % KS], (i / KS) & 1, p.status, kDevTimeoutDrain);
    } else {
      // ---------------- MMA issuers: warp 1 S = Q K^T, warp 3 O += P V ----------------
      // Pairs (tile, block) in the order (0, j), (1, j), (0, j + 1), ... go
      // round the NS slots; slots, stages and their phases are counted on, not
      // computed: what these warps do between two products idles the tensor
      // core. Control flow is the whole warp's, one thread is elected to issue
      // (see attn_common.cuh). Two warps and not one for both products: one has
      // no barrier to wait for between P V and the S that follows it, but does
      // the work of both in turn (8 sequences of 1025 to 2047 tokens, hd 64: 121
      // us against 104).
      const uint32_t sbase = smem_u32(smem);
      const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0);
      const uint32_t el = elect_one();
      auto uniform_wait = [&](uint64_t* bar, uint32_t parity, int* status, int code) {
        return __all_sync(0xffffffffu, seq_wait(bar, parity, status, code)) != 0;
      };
      SeqWork w;
      int slot = 0, ks = 0;
      uint32_t slot_ph = 0, ks_ph = 0;
      if (warp == 1) {
        constexpr uint32_t idesc_s = idesc_16_f32(DT, kAttnBM, C::kBN);
        int qs = 0;
        uint32_t q_ph = 0;
        bool ok = true;
        for (int it = 0; ok && __all_sync(0xffffffffu, take_item(it, w, kDevTimeoutMma)); ++it) {
          const int n0 = __shfl_sync(0xffffffffu, w.n0, 0), n1 = __shfl_sync(0xffffffffu, w.n1, 0);
          const bool end = __shfl_sync(0xffffffffu, w.seq, 0) < 0;
          if (lane == 0) mbar_arrive(&item_empty[it & 1]);
          if (end) break;
          const int n = max(n0, n1);
          if (n == 0) {
            if (lane == 0) mbar_arrive(&s_done[it & 1]);
            continue;
          }
          ok = uniform_wait(&q_full[qs], q_ph, p.status, kDevTimeoutMma);
          const uint32_t qa0 = sbase + C::kQOff + qs * (kAttnTiles * C::kQBytes);
          for (int j = 0; j < n && ok; ++j) {
            if (!(ok = uniform_wait(&k_full[ks], ks_ph, p.status, kDevTimeoutMma))) break;
            const uint32_t ka = sbase + C::kKOff + ks * C::kKvBytes;
#pragma unroll 1
            for (int t = 0; t < kAttnTiles; ++t) {
              if (j >= (t == 0 ? n0 : n1)) continue;
              // the PV that read this slot's last P
              if (!(ok = uniform_wait(&pv_done[slot], slot_ph ^ 1u, p.status, kDevTimeoutMma))) break;
              tc_fence_after();
              const uint32_t qa = qa0 + t * C::kQBytes;
#pragma unroll
              for (int k = 0; k < HD / 16; ++k) {
                const uint32_t in = (k & 3) * 32;
                umma_f16_ss_if(el, tmem_u + C::kTmS + slot * C::kBN,
                               smem_desc_sw128(qa + (k >> 2) * 16384 + in, 16, 1024),
                               smem_desc_sw128(ka + (k >> 2) * C::kKvHalf + in, 16, 1024), idesc_s, k > 0 ? 1u : 0u);
              }
              umma_commit_if(el, &s_full[slot]);
              if (++slot == NS) {
                slot = 0;
                slot_ph ^= 1u;
              }
            }
            umma_commit_if(el, &k_empty[ks]);
            if (++ks == KS) {
              ks = 0;
              ks_ph ^= 1u;
            }
          }
          umma_commit_if(el, &q_empty[qs]);
          umma_commit_if(el, &s_done[it & 1]);
          if (++qs == NQ) {
            qs = 0;
            q_ph ^= 1u;
          }
        }
      } else {
        constexpr uint32_t idesc_o = idesc_16_f32(DT, kAttnBM, HD, false, true);
        bool ok = true;
        for (int it = 0; ok && __all_sync(0xffffffffu, take_item(it, w, kDevTimeoutMma)); ++it) {
          const int n0 = __shfl_sync(0xffffffffu, w.n0, 0), n1 = __shfl_sync(0xffffffffu, w.n1, 0);
          const bool end = __shfl_sync(0xffffffffu, w.seq, 0) < 0;
          if (lane == 0) mbar_arrive(&item_empty[it & 1]);
          if (end) break;
          const int n = max(n0, n1);
          for (int j = 0; j < n && ok; ++j) {
            if (!(ok = uniform_wait(&v_full[ks], ks_ph, p.status, kDevTimeoutMma))) break;
            const uint32_t va = sbase + C::kVOff + ks * C::kKvBytes;
#pragma unroll 1
            for (int t = 0; t < kAttnTiles; ++t) {
              if (j >= (t == 0 ? n0 : n1)) continue;
              // (O of the tile's last item has been read: this P comes from the threads that read it)
              if (!(ok = uniform_wait(&p_full[slot], slot_ph, p.status, kDevTimeoutMma))) break;
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < C::kBN / 16; ++k)
                umma_f16_ts_if(el, tmem_u + C::kTmO + t * HD, tmem_u + C::kTmS + slot * C::kBN + k * 8,
                               smem_desc_sw128(va + k * 2048, C::kKvHalf, 1024), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
              umma_commit_if(el, &pv_done[slot]);
              if (j + 1 == (t == 0 ? n0 : n1)) umma_commit_if(el, &o_done[t]);
              if (++slot == NS) {
                slot = 0;
                slot_ph ^= 1u;
              }
            }
            umma_commit_if(el, &v_empty[ks]);
            if (++ks == KS) {
              ks = 0;
              ks_ph ^= 1u;
            }
          }
        }
      }
      // drain: every MMA this thread issued completes before TMEM is released
      uint64_t* d = &drain[warp == 1 ? 0 : 1];
      umma_commit_if(el, d);
      uniform_wait(d, 0, p.status, kDevTimeoutDrain);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSeqRegsHigh));
    // ---------------- softmax (warps 4..11) ----------------
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int tl = r / p.group;  // token within the tile
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tm_s = tmem_base + lane_off + C::kTmS;
    const uint32_t tm_o = tmem_base + lane_off + C::kTmO + t * HD;
    const float c = p.scale_log2;
    int qc = 0;  // pairs so far
    uint32_t o_ph = 0;

    for (int it = 0;; ++it) {
      if (!seq_wait(&item_full[it & 1], (it >> 1) & 1, p.status, kDevTimeoutSoftmax)) break;
      const SeqWork* item = &s_item[it & 1];
      if (item->seq < 0) break;
      const int n0 = item->n0, n1 = item->n1;
      const int nb = t == 0 ? n0 : n1;
      const int nmin = min(n0, n1);
      bool live;
      int admit;  // keys this row admits, from its first block on
      {
        const int tok = (2 * item->tile + t) * p.tok_tile + tl;
        const int q_len = item->q_len, k_len = item->k_len;
        live = tl < p.tok_tile && tok < q_len;
        admit = (p.causal ? min(k_len, tok + k_len - q_len + 1) : k_len) - item->jb * C::kBN;
      }
      // slot and phase of the tile's next pair in issue order, and of its last
      // one: when that pair's PV has completed, every PV of the tile so far has
      // landed in O. Within the item the slot's barrier is exact: S of this
      // thread's newest pair waited for the PV NS pairs back, so no phase before
      // the awaited one is open, and the slot's next PV comes after this
      // thread's next P. (A single barrier for all of a tile's PVs would not do:
      // with one tile alone they run up to NS behind.) At the item's end the
      // other tile's PVs may come round to the slot, so that wait is on o_done,
      // which completes once per item in which the tile has keys.
      const int q0 = qc + (nmin > 0 ? t : 0);
      int slot = q0 % NS, pv_slot = 0;
      uint32_t slot_ph = (q0 / NS) & 1, pv_ph = 0;
      auto wait_pv = [&] { return seq_wait(&pv_done[pv_slot], pv_ph, p.status, kDevTimeoutSoftmax); };

      float m_ref = -INFINITY;
      float l = 0.f;
      bool ok = true;

      for (int j = 0; j < nb; ++j) {
        if (!(ok = seq_wait(&s_full[slot], slot_ph, p.status, kDevTimeoutSoftmax))) break;
        tc_fence_after();
        // Probabilities are formed against a reference that trails the row's
        // maximum by at most kRescaleThreshold; if a row grows past that, O and l
        // are brought to a new one. The maximum is found beside the
        // exponentials, in the exp unit's shadow, and a pass that turns out to
        // need a new reference is made again, from the scores that still stand in
        // TMEM; only an item's first block has its maximum found first. (Always
        // first: one prompt of 16 384 tokens, hd 128, 1042 us against 960, two
        // chunks of 2000 tokens over 14 000 keys, hd 64, 304 against 285, two
        // prompts of 100 tokens 5.7 against 6.2.) 64 scores at a time: all 128 of
        // an hd 64 block in registers leave no room for the probabilities.
        const int lim = admit - j * C::kBN;
        const bool masked = __any_sync(0xffffffffu, lim < C::kBN);
        auto load = [&](uint32_t (&v)[64], int at) {
          tmem_ld64(tm_s + slot * C::kBN + at, v);
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] = at + i < lim ? v[i] : 0xff800000u;  // -inf
          }
        };
        if (j == 0) {
          float m = -INFINITY;
#pragma unroll 1
          for (int at = 0; at < C::kBN; at += 64) {
            uint32_t v[64];
            load(v, at);
            auto s = [&](int i) { return __uint_as_float(v[i]); };
            float mx[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) mx[k] = fmaxf(s(k), s(8 + k));
#pragma unroll
            for (int b = 16; b < 64; b += 16)
#pragma unroll
              for (int k = 0; k < 8; ++k) mx[k] = fmax3f(mx[k], s(b + k), s(b + 8 + k));
            mx[0] = fmax3f(mx[0], mx[1], mx[2]);
            mx[3] = fmax3f(mx[3], mx[4], mx[5]);
            mx[0] = fmax3f(mx[0], mx[3], fmaxf(mx[6], mx[7]));
            m = fmaxf(m, mx[0]);
          }
          m_ref = m * c;
        }

        uint32_t pk[C::kBN / 2];
        while (true) {
          // Scaling of the next scores, sums and packing of the last are issued
          // between the exponentials, which the exp unit takes one of in 8
          // cycles; scaling and sums two at a time (f32x2).
          constexpr int kAhead = 2;  // pairs; with 4 and 8 the block of 128 spills
          const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
          const uint64_t c2 = pair_of(c, c), m2 = pair_of(-m_use, -m_use);
          uint64_t ls[4] = {0ull, 0ull, 0ull, 0ull};
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int at = 0; at < C::kBN; at += 64) {
            uint32_t v[64];
            load(v, at);
            auto s = [&](int i) { return __uint_as_float(v[i]); };
            uint64_t x[32];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) x[i] = fma_f32x2(pair_of(s(2 * i), s(2 * i + 1)), c2, m2);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float e[4];
              split_pair(x[i], e[0], e[1]);
              split_pair(x[i + 1], e[2], e[3]);
#pragma unroll
              for (int k = 0; k < 4; ++k) e[k] = ex2_f32(e[k]);
              if (i + kAhead < 32) {
                const int a = i + kAhead;
                x[a] = fma_f32x2(pair_of(s(2 * a), s(2 * a + 1)), c2, m2);
                x[a + 1] = fma_f32x2(pair_of(s(2 * a + 2), s(2 * a + 3)), c2, m2);
              }
              mx[i & 3] = fmax3f(mx[i & 3], s(2 * i), s(2 * i + 1));
              mx[(i & 3) + 1] = fmax3f(mx[(i & 3) + 1], s(2 * i + 2), s(2 * i + 3));
              pk[at / 2 + i] = pack_p<DT>(e[0], e[1]);
              pk[at / 2 + i + 1] = pack_p<DT>(e[2], e[3]);
              uint64_t& sum = ls[(i >> 1) & 3];
              sum = add_f32x2(sum, add_f32x2(pair_of(e[0], e[2]), pair_of(e[1], e[3])));
            }
          }
          const float m_row = fmaxf(fmax3f(mx[0], mx[1], mx[2]), mx[3]) * c;

          // rows that are not stored have no vote: results must not depend on them
          const bool need = live && m_row > m_ref + kRescaleThreshold;
          if (!__any_sync(0xffffffffu, need)) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) split_pair(ls[k], y[2 * k], y[2 * k + 1]);
            l += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
            break;
          }
          const float m_new = fmaxf(m_ref, m_row);
          const float alpha = m_ref == -INFINITY ? 0.f : ex2_f32(m_ref - m_new);
          if (!(ok = wait_pv())) break;
          tc_fence_after();
          rescale_o<HD>(tm_o, alpha);
          l *= alpha;
          m_ref = m_new;  // no row is past it now: once more, and no further
        }
        if (!ok) break;

        if constexpr (C::kBN == 128) {
          tmem_st64(tm_s + slot * C::kBN, pk);
        } else {
          tmem_st32(tm_s + slot * C::kBN, pk);
        }
        tmem_wait_st_all();
        tc_fence_before();
        mbar_arrive(&p_full[slot]);
        pv_slot = slot;
        pv_ph = slot_ph;
        slot += j + 1 < nmin ? 2 : j < nmin ? 2 - t : 1;
        if (slot >= NS) {
          slot -= NS;
          slot_ph ^= 1u;
        }
      }
      if (!ok) break;

      // ---------------- epilogue ----------------
      uint32_t ov[HD];
      if (nb > 0) {
        if (!seq_wait(&o_done[t], o_ph, p.status, kDevTimeoutSoftmax)) break;
        o_ph ^= 1u;
        tc_fence_after();
        if constexpr (HD == 128) {
          tmem_ld128(tm_o, ov);
        } else {
          tmem_ld64(tm_o, ov);
        }
        tmem_wait_ld();
        tc_fence_before();
      } else {
#pragma unroll
        for (int i = 0; i < HD; ++i) ov[i] = 0u;
      }
      qc += n0 + n1;
      // a sum of 0 is that of a row without keys (or whose every score is -inf);
      // one of NaN (a score of NaN or +inf) goes on into the result, the
      // log-sum-exp and the join
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float lse = l == 0.f ? -INFINITY : (m_ref + __log2f(l)) * 0.69314718055994531f;
      const SeqOut& o = s_out;
      const int slot_out = item->slot;
      if (slot_out >= 0) {
        // [slot][HD / 4][256 rows][4]: a warp's rows lie side by side
        if (live) {
          const long long row = t * kAttnBM + r;
          o.lse_part[slot_out * static_cast<long long>(kAttnTiles * kAttnBM) + row] = lse;
          if (nb > 0) {
            float4* dst = reinterpret_cast<float4*>(o.o_part) +
                          slot_out * static_cast<long long>(HD / 4 * kAttnTiles * kAttnBM) + row;
#pragma unroll
            for (int i = 0; i < HD / 4; ++i)
              dst[i * (kAttnTiles * kAttnBM)] =
                  make_float4(__uint_as_float(ov[4 * i]) * inv, __uint_as_float(ov[4 * i + 1]) * inv,
                              __uint_as_float(ov[4 * i + 2]) * inv, __uint_as_float(ov[4 * i + 3]) * inv);
          }
        }
      } else {
        const long long token = item->q0 + (2 * item->tile + t) * p.tok_tile + tl;
        const int head = item->kvh * p.group + (r - tl * p.group);
        if (live && o.lse != nullptr) o.lse[static_cast<long long>(head) * o.tokens + token] = lse;
        const long long obase = token * o.o_ts + head * o.o_hs;
        if (o.out_f32) {
          if (live) {
            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(o.out) + obase);
#pragma unroll
            for (int i = 0; i < HD / 4; ++i)
              dst[i] = make_float4(__uint_as_float(ov[4 * i]) * inv, __uint_as_float(ov[4 * i + 1]) * inv,
                                   __uint_as_float(ov[4 * i + 2]) * inv, __uint_as_float(ov[4 * i + 3]) * inv);
          }
        } else {
          // Through shared memory, 64 columns of the warp's 32 rows at a time:
          // stored row by row as they are held, each store would touch 32
          // lines and the stores, not the products, bound short items
          // (hd 128, 4 key blocks: 16.5 us an item, 14.4 without them).
          uint4* stage = reinterpret_cast<uint4*>(smem + C::kStageOff + (warp - 4) * 4096);
          const unsigned rows = __ballot_sync(0xffffffffu, live);
#pragma unroll
          for (int h = 0; h < HD / 64; ++h) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int k = h * 64 + 8 * i;
              stage[lane * 8 + (i ^ (lane & 7))] =
                  make_uint4(pack2<DT>(__uint_as_float(ov[k]) * inv, __uint_as_float(ov[k + 1]) * inv),
                             pack2<DT>(__uint_as_float(ov[k + 2]) * inv, __uint_as_float(ov[k + 3]) * inv),
                             pack2<DT>(__uint_as_float(ov[k + 4]) * inv, __uint_as_float(ov[k + 5]) * inv),
                             pack2<DT>(__uint_as_float(ov[k + 6]) * inv, __uint_as_float(ov[k + 7]) * inv));
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int row = i * 4 + (lane >> 3);
              const long long at = __shfl_sync(0xffffffffu, obase, row);
              if (rows >> row & 1)
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(o.out) + at + h * 64 + (lane & 7) * 8) =
                    stage[row * 8 + ((lane & 7) ^ (row & 7))];
            }
            __syncwarp();
          }
        }
      }
      // A tile without blocks in this item must not run ahead to the next
      // item's slots: waiting there, it would take the phase before the last
      // for the one to come. (Exact here: this item is released only below,
      // so the barrier's next phase cannot have begun.)
      if (!seq_wait(&s_done[it & 1], (it >> 1) & 1, p.status, kDevTimeoutSoftmax)) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[it & 1]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins a tile's key ranges, in order: blocks take (tile, key head, 64 rows), a
// thread per row and quarter of the columns. Four ranges' results are
// requested at a time. How many tiles were cut is on the device, often none:
// the grid is kCombineCtas per SM and runs over what there is.
constexpr int kCombineCtas = 4;

template <int HD, int DT>
__global__ void __launch_bounds__(256) seq_combine_kernel(const __grid_constant__ SeqK p) {
  constexpr int CH = HD / 16;  // float4 columns per thread
  constexpr int kRows = kAttnTiles * kAttnBM;
  pdl_wait();
  pdl_trigger();
  const int items = (p.plan != nullptr ? p.plan[2] : p.max_tiles) * p.kv_heads * (kRows / 64);
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int head_item = item / (kRows / 64), tile = head_item / p.kv_heads, kvh = head_item - tile * p.kv_heads;
    const int at = p.plan != nullptr ? p.plan[4 + tile] : tile;
    if (at < 0) continue;
    const SeqWork w = p.list[at];
    if (w.seq < 0) continue;
    // ranges are kv_heads slots apart; the first is head 0's (list: counted in tiles)
    const long long slot = p.plan != nullptr ? static_cast<long long>(w.slot) * p.kv_heads + kvh : w.slot + kvh;
    const long long apart = static_cast<long long>(p.kv_heads) * kRows;
    const int r = item % (kRows / 64) * 64 + (threadIdx.x & 63);
    const int quarter = threadIdx.x >> 6;
    const int t = r / kAttnBM, rr = r % kAttnBM;
    const int tl = rr / p.group;
    const int tok = (2 * w.tile + t) * p.tok_tile + tl;
    if (tl >= p.tok_tile || tok >= w.q_len) continue;
    const float* lg = p.o.lse_part + slot * kRows + r;
    const float4* part =
        reinterpret_cast<const float4*>(p.o.o_part) + (slot * (HD / 4) + quarter * CH) * kRows + r;
    float m = -INFINITY;
#pragma unroll 8
    for (int k = 0; k < w.ranges; ++k) m = fmaxf(m, lg[k * apart]);
    float l = 0.f;
    float4 acc[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < w.ranges; ++k) {
      const float x = lg[k * apart];
      if (x == -INFINITY) continue;  // without keys for this row: no result was written
      const float f = __expf(x - m);
      l += f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const float4 y = part[k * apart * (HD / 4) + i * kRows];
        acc[i].x = fmaf(f, y.x, acc[i].x);
        acc[i].y = fmaf(f, y.y, acc[i].y);
        acc[i].z = fmaf(f, y.z, acc[i].z);
        acc[i].w = fmaf(f, y.w, acc[i].w);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const long long token = w.q0 + tok;
    const int head = kvh * p.group + (rr - tl * p.group);
    const long long base = token * p.o.o_ts + head * p.o.o_hs + quarter * (HD / 4);
    if (p.o.out_f32) {
#pragma unroll
      for (int i = 0; i < CH; ++i)
        reinterpret_cast<float4*>(static_cast<float*>(p.o.out) + base)[i] =
            make_float4(acc[i].x * inv, acc[i].y * inv, acc[i].z * inv, acc[i].w * inv);
    } else {
#pragma unroll
      for (int i = 0; i < CH; i += 2)
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o.out) + base)[i / 2] =
            make_uint4(pack2<DT>(acc[i].x * inv, acc[i].y * inv), pack2<DT>(acc[i].z * inv, acc[i].w * inv),
                       pack2<DT>(acc[i + 1].x * inv, acc[i + 1].y * inv), pack2<DT>(acc[i + 1].z * inv, acc[i + 1].w * inv));
    }
    if (p.o.lse != nullptr && quarter == 0)
      p.o.lse[static_cast<long long>(head) * p.o.tokens + token] = l == 0.f ? -INFINITY : m + __logf(l);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

struct SeqPlan {
  int tok_tile, tiles, splits, ctas, slots;
  bool listed;  // the tiles are listed by seq_plan_kernel
  long long list_bytes, bytes;
};

// Grid bound and key ranges of a call: every tile pair of every sequence fits
// the smaller of tokens / span + batch and batch * (tile pairs of the longest).
SeqPlan plan_of(const SeqArgs& a) {
  SeqPlan s = {};
  s.tok_tile = kAttnBM / (a.heads / a.kv_heads);
  const long long span = 2 * s.tok_tile;
  const long long by_tokens = a.tokens / span + a.batch;
  const long long by_longest = (a.max_q + span - 1) / span * a.batch;
  s.tiles = static_cast<int>(by_tokens < by_longest ? by_tokens : by_longest);
  const int sms = device_sm_count();
  const long long items = static_cast<long long>(s.tiles) * a.kv_heads;
  s.listed = items > sms;
  s.splits = 1;
  if (!s.listed && items > 0) {
    // as many ranges per tile as fill the SMs, of at least 512 keys (a
    // shorter range costs more in start-up and joining than the SMs it fills)
    long long n = sms / items;
    const long long most = (a.max_k + 127) / 512;
    if (n > most) n = most;
    s.splits = n < 1 ? 1 : n > 64 ? 64 : static_cast<int>(n);
  }
  s.ctas = static_cast<int>(s.listed ? sms : items * s.splits);
  if (s.listed) {
    s.slots = a.max_k >= kCutKeys ? 4 * sms / a.kv_heads : 0;
    s.list_bytes = 16 + (s.slots / 2 * 4 + 15) / 16 * 16 +
                   (s.tiles + static_cast<long long>(s.slots)) * static_cast<long long>(sizeof(SeqWork));
  } else if (s.splits > 1) {
    s.slots = s.tiles * s.splits;
    s.list_bytes = s.tiles * static_cast<long long>(sizeof(SeqWork));
  }
  s.list_bytes = (s.list_bytes + 15) / 16 * 16;
  s.bytes = s.list_bytes + static_cast<long long>(s.slots) * a.kv_heads * (kAttnTiles * kAttnBM) * (a.head_dim + 1) * 4;
  return s;
}

template <int HD, int DT, bool PAGED>
int launch_seq(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const SeqK& k, int ctas,
               cudaStream_t stream) {
  using C = SeqCfg<HD>;
  auto kern = flash_seq_tcgen05<HD, DT, PAGED>;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_done[dev & 63]) {
    // the register split assumes the launch pool of exactly kRegsLaunch
    // registers per thread (see flash_attn.cu)
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return set_error(TF_ERR_LAUNCH, "cudaFuncGetAttributes(flash_seq): %s", cudaGetErrorString(e));
    if (fa.numRegs != kRegsLaunch)
      return set_error(TF_ERR_LAUNCH, "flash_seq built with %d registers/thread, expected %d", fa.numRegs, kRegsLaunch);
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kAlloc);
    if (e != cudaSuccess) return set_error(TF_ERR_LAUNCH, "cudaFuncSetAttribute(flash_seq): %s", cudaGetErrorString(e));
    attr_done[dev & 63] = true;
  }
  cudaError_t e = cudaSuccess;
  if (k.plan != nullptr) e = launch_k(seq_plan_kernel<PAGED>, dim3(1), dim3(kPlanThreads), 0, stream, k, ctas);
  if (e == cudaSuccess) e = launch_k(kern, dim3(ctas), dim3(kAttnThreads), C::kAlloc, stream, tq, tk, tv, k);
  const int joins = k.plan != nullptr ? k.max_slots / 2 : k.splits > 1 ? k.max_tiles : 0;  // at most
  if (e == cudaSuccess && joins > 0) {
    const int blocks = joins * k.kv_heads * (kAttnTiles * kAttnBM / 64);
    e = launch_k(seq_combine_kernel<HD, DT>, dim3(std::min(blocks, kCombineCtas * device_sm_count())), dim3(256), 0,
                 stream, k);
  }
  if (e != cudaSuccess) return set_error(TF_ERR_LAUNCH, "flash_seq launch: %s", cudaGetErrorString(e));
  return TF_OK;
}

}  // namespace

// whether the call's arrays hold any key (without, they may be null)
static bool has_keys(const SeqArgs& a) { return a.page_size > 0 ? a.num_pages > 0 && a.max_pages > 0 : a.k_tokens > 0; }

int seq_check(const SeqArgs& a, const char* fn) {
  const bool paged = a.page_size > 0;
  if (a.head_dim != 64 && a.head_dim != 128)
    return set_error(TF_ERR_SHAPE, "%s: head_dim=%d (64 or 128 supported)", fn, a.head_dim);
  if (a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.heads / a.kv_heads > 128 || a.kv_heads > 65535)
    return set_error(TF_ERR_SHAPE, "%s: %d query heads over %d key heads (a whole number of at most 128 each)", fn,
                     a.heads, a.kv_heads);
  const long long most = 1ll << 30;
  if (a.batch < 0 || a.batch > most || a.tokens < 0 || a.tokens > most || a.k_tokens < 0 || a.k_tokens > most ||
      a.max_q < 0 || a.max_k < 0 || a.batch * a.kv_heads > most)
    return set_error(TF_ERR_SHAPE, "%s: sizes out of range", fn);
  if (!(a.scale > 0.f) || !(a.scale - a.scale == 0.f))
    return set_error(TF_ERR_SHAPE, "%s: scale must be positive and finite", fn);
  if (paged) {
    if (a.page_size < 16 || a.page_size > (1 << 20) || (a.page_size & (a.page_size - 1)))
      return set_error(TF_ERR_SHAPE, "%s: page_size=%lld (a power of two from 16)", fn, a.page_size);
    if (a.num_pages < 0 || a.num_pages > most || a.max_pages < 0 || a.max_pages * a.page_size > most * 2 - 1 ||
        a.max_pages > most)
      return set_error(TF_ERR_SHAPE, "%s: sizes out of range", fn);
  }
  if (a.batch == 0 || a.tokens == 0 || a.max_q == 0) return TF_OK;
  if (a.q == nullptr || a.out == nullptr || a.cu_q == nullptr || (paged ? a.kv_lens : a.cu_k) == nullptr ||
      (has_keys(a) && (a.k == nullptr || a.v == nullptr || (paged && a.page_table == nullptr))))
    return set_error(TF_ERR_SHAPE, "%s: null operand", fn);
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out) || !aligned16(a.workspace))
    return set_error(TF_ERR_ALIGN, "%s: q, keys, values, out and workspace must be 16-byte aligned", fn);
  for (long long s : {a.q_ts, a.q_hs, a.k_ts, a.k_hs, a.v_ts, a.v_hs, a.o_ts, a.o_hs, a.k_ps, a.v_ps})
    if (s < 0 || s % 8) return set_error(TF_ERR_ALIGN, "%s: strides must be multiples of 8 elements", fn);
  if (!rows_apart(a.head_dim, {{a.o_ts, a.tokens}, {a.o_hs, a.heads}}))
    return set_error(TF_ERR_SHAPE, "%s: rows of out overlap", fn);
  return TF_OK;
}

long long seq_workspace(const SeqArgs& a) {
  if (a.batch <= 0 || a.tokens <= 0 || a.max_q <= 0) return 0;
  if (a.page_size > 0 && paged_is_decode(a)) return paged_decode_workspace(a);
  return plan_of(a).bytes;
}

int seq_attention(const SeqArgs& args, cudaStream_t stream) {
  SeqArgs a = args;
  if (a.batch == 0 || a.tokens == 0 || a.max_q == 0) return TF_OK;
  if (!has_keys(a)) {
    // nothing to attend to: every length is cut to 0, so the keys and the
    // table are never read; q's address stands in for the tensor maps
    a.num_pages = a.max_pages = a.k_tokens = 0;
    if (a.k == nullptr) a.k = a.q;
    if (a.v == nullptr) a.v = a.q;
  }
  const long long need = seq_workspace(a);
  if (a.workspace_bytes < need || (need > 0 && a.workspace == nullptr))
    return set_error(TF_ERR_SHAPE, "workspace of %lld bytes needed, %lld given", need, a.workspace_bytes);
  const bool paged = a.page_size > 0;
  if (paged && paged_is_decode(a)) return paged_decode(a, stream);

  const SeqPlan plan = plan_of(a);
  const int group = a.heads / a.kv_heads;
  SeqK k = {};
  k.o.out = a.out;
  k.o.o_ts = a.o_ts;
  k.o.o_hs = a.o_hs;
  k.o.lse = a.lse;
  k.cu_q = a.cu_q;
  k.cu_k = a.cu_k;
  k.kv_lens = a.kv_lens;
  k.page_table = a.page_table;
  k.table_ld = a.table_ld;
  k.batch = static_cast<int>(a.batch);
  k.heads = a.heads;
  k.group = group;
  k.tokens = static_cast<int>(a.tokens);
  k.k_tokens = static_cast<int>(a.k_tokens);
  k.max_q = static_cast<int>(a.max_q < a.tokens ? a.max_q : a.tokens);
  k.tok_tile = plan.tok_tile;
  k.kv_heads = a.kv_heads;
  k.max_tiles = plan.tiles;
  k.splits = plan.splits;
  k.o.tokens = k.tokens;
  char* ws = static_cast<char*>(a.workspace);
  if (plan.listed) {
    k.max_slots = plan.slots;
    k.plan = reinterpret_cast<int*>(ws);
    k.list = reinterpret_cast<SeqWork*>(ws + 16 + (plan.slots / 2 * 4 + 15) / 16 * 16);
  } else if (plan.splits > 1) {
    k.list = reinterpret_cast<SeqWork*>(ws);
  }
  k.o.o_part = reinterpret_cast<float*>(ws + plan.list_bytes);
  k.o.lse_part =
      k.o.o_part + static_cast<long long>(plan.slots) * a.kv_heads * (kAttnTiles * kAttnBM) * a.head_dim;
  k.scale_log2 = a.scale * 1.4426950408889634f;
  k.causal = a.causal;
  k.o.out_f32 = a.out_f32;
  k.status = device_status_ptr();
  if (k.status == nullptr) return last_error_code();

  CUtensorMap tq, tk, tv;
  int rc = make_tmap_4d_f16(&tq, a.q, {a.head_dim, group, a.kv_heads, a.tokens}, {a.q_hs, a.q_hs * group, a.q_ts},
                            {64, group, 1, plan.tok_tile});
  if (rc) return rc;
  const long long rows = paged ? a.page_size : a.k_tokens;
  const int block = seq_block(a.head_dim);
  while ((1 << k.bn_shift) < block) ++k.bn_shift;
  const int box = paged && a.page_size < block ? static_cast<int>(a.page_size) : block;
  const long long pages = paged ? a.num_pages : 1;
  rc = make_tmap_4d_f16(&tk, a.k, {a.head_dim, a.kv_heads, rows, pages}, {a.k_hs, a.k_ts, a.k_ps}, {64, 1, box, 1});
  if (rc) return rc;
  rc = make_tmap_4d_f16(&tv, a.v, {a.head_dim, a.kv_heads, rows, pages}, {a.v_hs, a.v_ts, a.v_ps}, {64, 1, box, 1});
  if (rc) return rc;
  if (paged) {
    while ((1ll << k.page_shift) < a.page_size) ++k.page_shift;
    k.page_box = box;
    k.num_pages = static_cast<int>(a.num_pages);
    k.page_cap = a.max_pages * a.page_size;
  }
#define TFB_SEQ(DT)                                                                                    \
  if (paged)                                                                                           \
    return a.head_dim == 64 ? launch_seq<64, DT, true>(tq, tk, tv, k, plan.ctas, stream)                    \
                            : launch_seq<128, DT, true>(tq, tk, tv, k, plan.ctas, stream);                  \
  return a.head_dim == 64 ? launch_seq<64, DT, false>(tq, tk, tv, k, plan.ctas, stream)                     \
                          : launch_seq<128, DT, false>(tq, tk, tv, k, plan.ctas, stream);
  if (a.bf16) {
    TFB_SEQ(kDtBF16)
  }
  TFB_SEQ(kDtF16)
#undef TFB_SEQ
}

}  // namespace tfb
