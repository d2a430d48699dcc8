// Attention of sequences of different lengths with grouped heads, on the
// 5th-generation tensor cores: queries packed end to end; keys and values
// packed the same way, or in a paged cache.
//
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j      over the keys of i's own sequence,
//   causal: j <= i + (keys - queries), the last query stands at the last key
//
// The pipeline is that of flash_fwd_tcgen05 (flash_attn.cu): two query tiles
// per CTA, S = Q K^T into a ring of TMEM slots, softmax with lazy rescaling in
// registers, P back over its S slot, O += P V from TMEM. What differs:
//
// * A tile's 128 rows are (token, query head of the group) pairs, so all query
//   heads that share a key head read each K and V tile once: a 4-D tensor map
//   over [token][key head][group head][64 columns] fills 128 / G tokens times
//   G heads per tile in one copy. G heads of one token see the same keys, so
//   the causal limit is per token and a tile spans fewer positions.
// * Tiles are cut per sequence. A CTA finds its (sequence, tile) by a warp
//   scan over the offsets (32 sequences per step), so the call needs no plan,
//   no host copy of the lengths and nothing kept from call to call; the grid
//   is the bound tokens / tile + batch, and CTAs past the last tile leave.
// * Key blocks start at the sequence's first key, and a copy may run into the
//   next sequence or past a page's end. Such scores are masked as usual; such
//   V rows are zeroed in shared memory before the product (0 * NaN would
//   otherwise reach the result), by the V producer, in the last block of a
//   sequence only.
// * Paged: a key block is 128 / page_size copies, one per page (one copy of a
//   part of a larger page), issued by as many lanes; page indices are read one
//   block ahead. An index outside the cache reads zeros and is reported.
// * Few tiles and long keys: the key blocks of each tile are cut into
//   `splits` ranges, whose normalised fp32 results and log-sum-exps
//   seq_combine_kernel joins in range order.
#include "attn_common.cuh"
#include "common.cuh"
#include "launch.h"

namespace tfb {
namespace {

struct SeqK {
  void* out;
  long long o_ts, o_hs;
  float* lse;
  const int* cu_q;
  const int* cu_k;
  const int* kv_lens;
  const int* page_table;
  long long table_ld;
  int num_pages, page_shift, page_box;  // page_box: rows of a page one copy takes
  long long page_cap;                   // keys a page table row can hold
  int batch, heads, group, tokens, k_tokens, max_q;
  int tok_tile;  // tokens per 128-row tile
  int splits;
  float* o_part;    // [splits][tokens][heads][HD]
  float* lse_part;  // [splits][tokens][heads], natural log
  float scale_log2;
  int causal, out_f32;
  int* status;
};

template <int HD>
struct SeqCfg {
  static constexpr int kNS = HD == 64 ? 3 : 2;
  static constexpr int kStages = HD == 64 ? 4 : 2;  // of K and of V
  static constexpr int kTileBytes = 128 * HD * 2;
  static constexpr int kQOff = 0;
  static constexpr int kKOff = kQOff + kAttnTiles * kTileBytes;
  static constexpr int kVOff = kKOff + kStages * kTileBytes;
  static constexpr int kBarOff = kVOff + kStages * kTileBytes;
  // q_full, v_tail, k_full/empty, v_full/empty, s_full[NS], p_full[2 x 2],
  // turn[2], drain[2], pv_done[NS]
  static constexpr int kNumBars = 2 + 4 * kStages + kNS + 4 + 2 + 2 + kNS;
  static constexpr int kBytes = kBarOff + kNumBars * 8 + 16;
  static constexpr int kAlloc = kBytes + 1024;
  static constexpr uint32_t kTmS = 0;
  static constexpr uint32_t kTmO = kNS * 128;
  static_assert(kNS * 128 + kAttnTiles * HD <= 512, "TMEM budget");
};

struct SeqWork {
  int seq, tile;    // seq < 0: no work
  int q0, q_len;    // first query token, queries
  int k0, k_len;    // packed: first key token; keys
};

// Queries and keys of sequence b, bounded by what the call's arrays hold. A
// bound that bites is an error of the caller's: it is reported, and nothing
// outside the arrays is read or written.
template <bool PAGED>
__device__ __forceinline__ SeqWork seq_lens(const SeqK& p, int b, bool& bad) {
  SeqWork w;
  w.seq = b;
  w.tile = 0;
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
      if (bad) record_error(p.status, kDevBadIndex);
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
      SeqWork r;
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

template <int HD, int DT, bool PAGED>
__global__ void __launch_bounds__(kAttnThreads, 1)
    flash_seq_tcgen05(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ SeqK p) {
  using C = SeqCfg<HD>;
  constexpr int KS = C::kStages;
  constexpr int NS = C::kNS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* q_full = bars;
  uint64_t* v_tail = q_full + 1;  // the copy of a sequence's last, partial V block
  uint64_t* k_full = v_tail + 1;
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;
  uint64_t* v_empty = v_full + KS;
  uint64_t* s_full = v_empty + KS;
  uint64_t* p_full = s_full + NS;
  uint64_t* turn = p_full + 4;
  uint64_t* drain = turn + 2;
  uint64_t* pv_done = drain + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + NS);
  __shared__ SeqWork s_work;

  const int warp = warp_id();
  const int lane = lane_id();
  const int kvh = blockIdx.y;
  const int split = blockIdx.z;

  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&tmQ);
    tma_prefetch_map(&tmK);
    tma_prefetch_map(&tmV);
    mbar_init(q_full, 1);
    mbar_init(v_tail, 1);
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&p_full[i], 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&turn[i], 128);
      mbar_init(&drain[i], 1);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // everything above touched only this CTA's shared memory and TMEM
  pdl_wait();
  pdl_trigger();
  if (warp == 3) {
    // later tiles of a causal sequence see more keys: hand them out first
    const SeqWork w = find_tile<PAGED>(p, static_cast<int>(gridDim.x - 1 - blockIdx.x));
    if (lane == 0) s_work = w;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const SeqWork w = s_work;
  const int tok0 = w.tile * 2 * p.tok_tile;  // first token of the CTA, within its sequence
  const int shift = w.k_len - w.q_len;       // query i stands at key i + shift

  // key blocks [jb, jb + nblk[t]) of each tile: this split's part
  int nblk[kAttnTiles];
  int nall = 0;
#pragma unroll
  for (int t = 0; t < kAttnTiles; ++t) {
    const int t0 = tok0 + t * p.tok_tile;
    int k_end = w.seq >= 0 && t0 < w.q_len ? w.k_len : 0;
    if (p.causal && k_end > 0) k_end = min(k_end, min(t0 + p.tok_tile, w.q_len) + shift);
    nblk[t] = k_end <= 0 ? 0 : (k_end + kAttnBN - 1) / kAttnBN;
    nall = max(nall, nblk[t]);
  }
  const int per = (nall + p.splits - 1) / p.splits;
  const int jb = split * per;
#pragma unroll
  for (int t = 0; t < kAttnTiles; ++t) nblk[t] = min(max(nblk[t] - jb, 0), per);
  const int nmax = nblk[0] > nblk[1] ? nblk[0] : nblk[1];
  const int nmin = nblk[0] < nblk[1] ? nblk[0] : nblk[1];
  const int t_long = nblk[0] > nblk[1] ? 0 : 1;
  const int n_pairs = nblk[0] + nblk[1];

  // one K or V block: this lane's copy (a page or a part of one, or the
  // whole block of packed keys) and the bytes of all copies
  auto boxes_of = [&](int j) {
    if constexpr (PAGED) {
      const int left = min(kAttnBN, w.k_len - (jb + j) * kAttnBN);
      return (left + p.page_box - 1) / p.page_box;
    } else {
      return 1;
    }
  };
  auto page_of = [&](int j) {
    if constexpr (PAGED) {
      if (j >= nmax || lane >= boxes_of(j)) return 0;
      const int key = (jb + j) * kAttnBN + lane * p.page_box;
      return p.page_table[w.seq * p.table_ld + (key >> p.page_shift)];
    } else {
      return 0;
    }
  };
  auto load_block = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int j, int page) {
    const int key = (jb + j) * kAttnBN;
    const int n = boxes_of(j);
    const int rows = PAGED ? p.page_box : kAttnBN;
    if (lane == 0) mbar_arrive_expect_tx(bar, n * rows * HD * 2);
    __syncwarp();
    if (lane < n) {
      int y, z;
      if constexpr (PAGED) {
        const bool ok = page >= 0 && page < p.num_pages;
        if (!ok) record_error(p.status, kDevBadIndex);
        y = (key + lane * rows) & ((1 << p.page_shift) - 1);
        z = ok ? page : (1 << 30);  // past every cache: zeros
      } else {
        y = w.k0 + key;
        z = 0;
      }
#pragma unroll
      for (int c = 0; c < HD / 64; ++c)
        tma_load_4d(dst + c * 16384 + lane * rows * 128, map, bar, c * 64, kvh, y, z);
    }
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
    if (warp == 0) {
      if (nmax > 0) {
        // ---------------- Q + K producer ----------------
        if (lane == 0) {
          const int tiles = nblk[1] > 0 ? 2 : 1;  // tile 1 has no keys when it has no tokens
          const int first = nblk[0] > 0 ? 0 : 1;
          mbar_arrive_expect_tx(q_full, (tiles - first) * p.tok_tile * p.group * HD * 2);
          for (int t = first; t < tiles; ++t)
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
              tma_load_4d(smem + C::kQOff + t * C::kTileBytes + c * 16384, &tmQ, q_full, c * 64, 0, kvh,
                          w.q0 + tok0 + t * p.tok_tile);
        }
        int page = page_of(0);
        int j = 0;
        for (; j < nmax; ++j) {
          const int s = j % KS;
          const int next = page_of(j + 1);
          if (!mbar_wait(&k_empty[s], ((j / KS) & 1) ^ 1, p.status, kDevTimeoutProducer)) break;
          load_block(smem + C::kKOff + s * C::kTileBytes, &tmK, &k_full[s], j, page);
          page = next;
        }
        mbar_wait(q_full, 0, p.status, kDevTimeoutDrain);
        for (int i = (j > KS ? j - KS : 0); i < j; ++i)
          mbar_wait(&k_full[i % KS], (i / KS) & 1, p.status, kDevTimeoutDrain);
      }
    } else if (warp == 2) {
      if (nmax > 0) {
        // ---------------- V producer ----------------
        int page = page_of(0);
        int j = 0;
        for (; j < nmax; ++j) {
          const int s = j % KS;
          const int next = page_of(j + 1);
          if (!mbar_wait(&v_empty[s], ((j / KS) & 1) ^ 1, p.status, kDevTimeoutProducer)) break;
          uint8_t* dst = smem + C::kVOff + s * C::kTileBytes;
          const int valid = w.k_len - (jb + j) * kAttnBN;
          if (valid >= kAttnBN) {
            load_block(dst, &tmV, &v_full[s], j, page);
          } else {
            // the sequence ends inside this block: rows from `valid` on hold
            // another sequence's values, an unused part of a page or what the
            // stage held before
            load_block(dst, &tmV, v_tail, j, page);
            if (!mbar_wait(v_tail, 0, p.status, kDevTimeoutProducer)) break;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
              for (int i = valid * 8 + lane; i < kAttnBN * 8; i += 32)
                *reinterpret_cast<uint4*>(dst + c * 16384 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[s]);
          }
          page = next;
        }
        for (int i = (j > KS ? j - KS : 0); i < j; ++i)
          mbar_wait(&v_full[i % KS], (i / KS) & 1, p.status, kDevTimeoutDrain);
      }
    } else if (warp == 1 || warp == 3) {
      if (lane == 0 && nmax > 0) {
        // ---------------- MMA issuers: warp 1 S = Q K^T, warp 3 O += P V ----------------
        constexpr uint32_t idesc_s = idesc_16_f32(DT, kAttnBM, kAttnBN);
        constexpr uint32_t idesc_o = idesc_16_f32(DT, kAttnBM, HD, false, true);
        const uint32_t sbase = smem_u32(smem);
        auto pair_of = [&](int q, int& t, int& j) {
          if (q < 2 * nmin) {
            j = q >> 1;
            t = q & 1;
          } else {
            j = nmin + (q - 2 * nmin);
            t = t_long;
          }
        };
        auto last_user = [&](int t, int j) { return t == 1 || j >= nblk[1]; };
        bool ok = true;
        if (warp == 1) {
          ok = mbar_wait(q_full, 0, p.status, kDevTimeoutMma);
          for (int q = 0; q < n_pairs && ok; ++q) {
            int t, j;
            pair_of(q, t, j);
            const int slot = q % NS;
            if (q >= NS && !(ok = mbar_wait(&pv_done[slot], ((q - NS) / NS) & 1, p.status, kDevTimeoutMma))) break;
            if (!(ok = mbar_wait(&k_full[j % KS], (j / KS) & 1, p.status, kDevTimeoutMma))) break;
            tc_fence_after();
            const uint32_t qa = sbase + C::kQOff + t * C::kTileBytes;
            const uint32_t ka = sbase + C::kKOff + (j % KS) * C::kTileBytes;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
              const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
              umma_f16_ss(tmem_base + C::kTmS + slot * 128, smem_desc_sw128(qa + off, 16, 1024),
                          smem_desc_sw128(ka + off, 16, 1024), idesc_s, k > 0 ? 1u : 0u);
            }
            umma_commit(&s_full[slot]);
            if (last_user(t, j)) umma_commit(&k_empty[j % KS]);
          }
        } else {
          for (int q = 0; q < n_pairs && ok; ++q) {
            int t, j;
            pair_of(q, t, j);
            const int slot = q % NS;
            if (!(ok = mbar_wait(&v_full[j % KS], (j / KS) & 1, p.status, kDevTimeoutMma))) break;
            if (!(ok = mbar_wait(&p_full[t * 2 + (j & 1)], (j >> 1) & 1, p.status, kDevTimeoutMma))) break;
            tc_fence_after();
            const uint32_t va = sbase + C::kVOff + (j % KS) * C::kTileBytes;
#pragma unroll
            for (int k = 0; k < kAttnBN / 16; ++k)
              umma_f16_ts(tmem_base + C::kTmO + t * HD, tmem_base + C::kTmS + slot * 128 + k * 8,
                          smem_desc_sw128(va + k * 2048, 16384, 1024), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
            umma_commit(&pv_done[slot]);
            if (last_user(t, j)) umma_commit(&v_empty[j % KS]);
          }
        }
        uint64_t* d = &drain[warp == 1 ? 0 : 1];
        umma_commit(d);
        mbar_wait(d, 0, p.status, kDevTimeoutDrain);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsHigh));
    // ---------------- softmax (warps 4..11) ----------------
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int tl = r / p.group;  // token within the tile
    const int tok = tok0 + t * p.tok_tile + tl;
    const bool live = w.seq >= 0 && tl < p.tok_tile && tok < w.q_len;
    // keys this row admits, from its first block on
    const int admit = (p.causal ? min(w.k_len, tok + shift + 1) : w.k_len) - jb * kAttnBN;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tm_s = tmem_base + lane_off + C::kTmS;
    const uint32_t tm_o = tmem_base + lane_off + C::kTmO + t * HD;
    const int nb = nblk[t];
    const float c = p.scale_log2;

    // issue order of (t, j)
    auto pair_at = [&](int j) { return j < nmin ? 2 * j + t : 2 * nmin + (j - nmin); };
    // every PV up to the tile's block j has landed in O. The slot's barrier is
    // exact: S of this thread's newest pair waited for the PV NS pairs back,
    // so no phase before the awaited one of that slot is open. (One barrier
    // per tile would not do: with one tile alone its PVs run up to NS behind.)
    auto wait_pv = [&](int j) {
      const int q = pair_at(j);
      return mbar_wait(&pv_done[q % NS], (q / NS) & 1, p.status, kDevTimeoutSoftmax);
    };

    float m_ref = -INFINITY;
    float l = 0.f;
    bool ok = true;

    for (int j = 0; j < nb; ++j) {
      const int q = pair_at(j);
      const int slot = q % NS;
      if (!(ok = mbar_wait(&s_full[slot], (q / NS) & 1, p.status, kDevTimeoutSoftmax))) break;
      tc_fence_after();
      float s[128];
      {
        uint32_t v[128];
        tmem_ld128(tm_s + slot * 128, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i] = __uint_as_float(v[i]);
      }
      const int lim = admit - j * kAttnBN;
      if (__any_sync(0xffffffffu, lim < kAttnBN)) {
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i] = i < lim ? s[i] : -INFINITY;
      }

      float mx[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) mx[k] = fmax3f(s[k], s[8 + k], s[16 + k]);
#pragma unroll
      for (int base = 24; base < 120; base += 16)
#pragma unroll
        for (int k = 0; k < 8; ++k) mx[k] = fmax3f(mx[k], s[base + k], s[base + 8 + k]);
#pragma unroll
      for (int k = 0; k < 8; ++k) mx[k] = fmaxf(mx[k], s[120 + k]);
      mx[0] = fmax3f(mx[0], mx[1], mx[2]);
      mx[3] = fmax3f(mx[3], mx[4], mx[5]);
      mx[0] = fmax3f(mx[0], mx[3], fmaxf(mx[6], mx[7]));
      const float m_row = mx[0] * c;

      // rows that are not stored have no vote: results must not depend on them
      const bool need = live && m_row > m_ref + kRescaleThreshold;
      if (j == 0) {
        m_ref = m_row;
      } else if (__any_sync(0xffffffffu, need)) {
        const float m_new = fmaxf(m_ref, m_row);
        const float alpha = m_ref == -INFINITY ? 0.f : ex2_f32(m_ref - m_new);
        if (!(ok = wait_pv(j - 1))) break;
        tc_fence_after();
        rescale_o<HD>(tm_o, alpha);
        l *= alpha;
        m_ref = m_new;
      }
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref;

      uint32_t pk[64];
      float ls[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 128; ++i) s[i] = fmaf(s[i], c, -m_use);
      if (j < nmin && (t == 1 || j > 0)) {
        const uint32_t par = t == 0 ? ((j - 1) & 1) : (j & 1);
        if (!(ok = mbar_wait(&turn[t], par, p.status, kDevTimeoutSoftmax))) break;
      }
#pragma unroll
      for (int i = 0; i < 128; ++i) s[i] = ex2_f32(s[i]);
      if (j < nmin) mbar_arrive(&turn[1 - t]);
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        pk[i] = pack_p<DT>(s[2 * i], s[2 * i + 1]);
        ls[i & 7] += s[2 * i] + s[2 * i + 1];
      }
      l += ((ls[0] + ls[1]) + (ls[2] + ls[3])) + ((ls[4] + ls[5]) + (ls[6] + ls[7]));

      tmem_st64(tm_s + slot * 128, pk);
      tmem_wait_st_all();
      tc_fence_before();
      mbar_arrive(&p_full[t * 2 + (j & 1)]);
    }

    // ---------------- epilogue ----------------
    if (ok) {
      uint32_t ov[HD];
      if (nb > 0) {
        ok = wait_pv(nb - 1);
        if (ok) {
          tc_fence_after();
          if constexpr (HD == 128) {
            tmem_ld128(tm_o, ov);
          } else {
            tmem_ld64(tm_o, ov);
          }
          tmem_wait_ld();
        }
      } else {
#pragma unroll
        for (int i = 0; i < HD; ++i) ov[i] = 0u;
      }
      if (ok && live) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const float lse = l > 0.f ? (m_ref + __log2f(l)) * 0.69314718055994531f : -INFINITY;
        const long long token = w.q0 + tok;
        const int head = kvh * p.group + (r - tl * p.group);
        if (p.splits > 1) {
          const long long at = (split * static_cast<long long>(p.tokens) + token) * p.heads + head;
          p.lse_part[at] = lse;
          if (nb > 0) {
            float4* dst = reinterpret_cast<float4*>(p.o_part + at * HD);
#pragma unroll
            for (int i = 0; i < HD / 4; ++i)
              dst[i] = make_float4(__uint_as_float(ov[4 * i]) * inv, __uint_as_float(ov[4 * i + 1]) * inv,
                                   __uint_as_float(ov[4 * i + 2]) * inv, __uint_as_float(ov[4 * i + 3]) * inv);
          }
        } else {
          if (p.lse != nullptr) p.lse[static_cast<long long>(head) * p.tokens + token] = lse;
          const long long obase = token * p.o_ts + head * p.o_hs;
          if (p.out_f32) {
            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + obase);
#pragma unroll
            for (int i = 0; i < HD / 4; ++i)
              dst[i] = make_float4(__uint_as_float(ov[4 * i]) * inv, __uint_as_float(ov[4 * i + 1]) * inv,
                                   __uint_as_float(ov[4 * i + 2]) * inv, __uint_as_float(ov[4 * i + 3]) * inv);
          } else {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + obase);
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
              dst[i] = make_uint4(
                  pack2<DT>(__uint_as_float(ov[8 * i]) * inv, __uint_as_float(ov[8 * i + 1]) * inv),
                  pack2<DT>(__uint_as_float(ov[8 * i + 2]) * inv, __uint_as_float(ov[8 * i + 3]) * inv),
                  pack2<DT>(__uint_as_float(ov[8 * i + 4]) * inv, __uint_as_float(ov[8 * i + 5]) * inv),
                  pack2<DT>(__uint_as_float(ov[8 * i + 6]) * inv, __uint_as_float(ov[8 * i + 7]) * inv));
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins the ranges of each (token, head): one warp per row, in range order.
// Tokens outside the sequences are left alone.
template <int HD, int DT>
__global__ void __launch_bounds__(256) seq_combine_kernel(const __grid_constant__ SeqK p) {
  pdl_wait();
  pdl_trigger();
  constexpr int E = HD / 32;
  const long long row = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5;
  const int lane = lane_id();
  if (row >= static_cast<long long>(p.tokens) * p.heads) return;
  const long long token = row / p.heads;
  const int head = static_cast<int>(row - token * p.heads);
  if (token < p.cu_q[0] || token >= p.cu_q[p.batch]) return;
  const long long stride = static_cast<long long>(p.tokens) * p.heads;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.lse_part[s * stride + row]);
  float l = 0.f, acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float g = p.lse_part[s * stride + row];
    if (g == -INFINITY) continue;  // a range without keys wrote no result
    const float f = __expf(g - m);
    l += f;
    const float* src = p.o_part + (s * stride + row) * HD + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = fmaf(f, src[i], acc[i]);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const long long base = token * p.o_ts + head * p.o_hs + lane * E;
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    if (p.out_f32) {
      *reinterpret_cast<float2*>(static_cast<float*>(p.out) + base + i) = make_float2(acc[i] * inv, acc[i + 1] * inv);
    } else {
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + base + i) = pack2<DT>(acc[i] * inv, acc[i + 1] * inv);
    }
  }
  if (p.lse != nullptr && lane == 0)
    p.lse[static_cast<long long>(head) * p.tokens + token] = l > 0.f ? m + __logf(l) : -INFINITY;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

struct SeqPlan {
  int tok_tile, tiles, splits;
};

// Grid bound and key split of a call: every CTA tile of every sequence fits
// the smaller of tokens / tile + batch and batch * (tiles of the longest).
// Keys are split when that leaves SMs without a CTA, into ranges of at least
// 4 key blocks (a shorter range costs more in start-up and joining than the
// idle SMs it fills).
SeqPlan plan_of(const SeqArgs& a) {
  SeqPlan s;
  s.tok_tile = kAttnBM / (a.heads / a.kv_heads);
  const long long span = 2 * s.tok_tile;
  const long long by_tokens = a.tokens / span + a.batch;
  const long long by_longest = (a.max_q + span - 1) / span * a.batch;
  s.tiles = static_cast<int>(by_tokens < by_longest ? by_tokens : by_longest);
  const long long ctas = static_cast<long long>(s.tiles) * a.kv_heads;
  const long long blocks = (a.max_k + kAttnBN - 1) / kAttnBN;
  long long n = ctas > 0 ? device_sm_count() / ctas : 1;
  if (n > blocks / 4) n = blocks / 4;
  s.splits = n < 1 ? 1 : n > 64 ? 64 : static_cast<int>(n);
  return s;
}

template <int HD, int DT, bool PAGED>
int launch_seq(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const SeqK& k, dim3 grid,
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
  cudaError_t e = launch_k(kern, grid, dim3(kAttnThreads), C::kAlloc, stream, tq, tk, tv, k);
  if (e == cudaSuccess && k.splits > 1) {
    const long long rows = static_cast<long long>(k.tokens) * k.heads;
    e = launch_k(seq_combine_kernel<HD, DT>, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, stream, k);
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
  return TF_OK;
}

long long seq_workspace(const SeqArgs& a) {
  if (a.batch <= 0 || a.tokens <= 0 || a.max_q <= 0) return 0;
  if (a.page_size > 0 && paged_is_decode(a)) return paged_decode_workspace(a);
  const SeqPlan s = plan_of(a);
  return s.splits > 1 ? a.tokens * a.heads * (a.head_dim + 1) * 4 * s.splits : 0;
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
  k.out = a.out;
  k.o_ts = a.o_ts;
  k.o_hs = a.o_hs;
  k.lse = a.lse;
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
  k.splits = plan.splits;
  k.o_part = static_cast<float*>(a.workspace);
  k.lse_part = k.o_part + a.tokens * a.heads * a.head_dim * plan.splits;
  k.scale_log2 = a.scale * 1.4426950408889634f;
  k.causal = a.causal;
  k.out_f32 = a.out_f32;
  k.status = device_status_ptr();
  if (k.status == nullptr) return last_error_code();

  CUtensorMap tq, tk, tv;
  int rc = make_tmap_4d_f16(&tq, a.q, {a.head_dim, group, a.kv_heads, a.tokens}, {a.q_hs, a.q_hs * group, a.q_ts},
                            {64, group, 1, plan.tok_tile});
  if (rc) return rc;
  const long long rows = paged ? a.page_size : a.k_tokens;
  const int box = paged && a.page_size < kAttnBN ? static_cast<int>(a.page_size) : kAttnBN;
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
  const dim3 grid(plan.tiles, a.kv_heads, plan.splits);
#define TFB_SEQ(DT)                                                                                    \
  if (paged)                                                                                           \
    return a.head_dim == 64 ? launch_seq<64, DT, true>(tq, tk, tv, k, grid, stream)                    \
                            : launch_seq<128, DT, true>(tq, tk, tv, k, grid, stream);                  \
  return a.head_dim == 64 ? launch_seq<64, DT, false>(tq, tk, tv, k, grid, stream)                     \
                          : launch_seq<128, DT, false>(tq, tk, tv, k, grid, stream);
  if (a.bf16) {
    TFB_SEQ(kDtBF16)
  }
  TFB_SEQ(kDtF16)
#undef TFB_SEQ
}

}  // namespace tfb
