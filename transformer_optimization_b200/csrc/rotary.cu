// Rotary positions of queries and keys, optionally written into a paged cache.
//
//   (x_a, x_b) -> m * (x_a cos t - x_b sin t, x_a sin t + x_b cos t),   t = position * freq[i]
//
// for the rot / 2 element pairs of every head, (a, b) = (i, i + rot/2) in the
// half layout and (2i, 2i + 1) in the interleaved one; elements from rot on
// are copied. The angle is formed in 64 bits and in turns, p * f / 2 pi minus
// its nearest whole number, so a position of 10^6 keeps the same absolute
// error (about 1e-7 of a turn, that of the fp32 sincospif after it) as a
// position of 1: in fp32 the product alone would be off by 0.03 rad there.
// The rotation is fp32, rounded once to the 16-bit type.
//
// Bound by HBM: every element is read once and written once, 3 flop each. A
// block takes a few tokens; its threads first request their rows' vectors
// (kRotRows heads per thread, 16 bytes at each end of the pair), then form the
// block's rot/2 angles per token once in shared memory (the fp64 products and
// sincospif are shared by all heads), then rotate and store. So the angles
// cost nothing while the loads are in flight: 50 000 tokens, 32 + 2 x 8 heads of
// 128, into a cache, 0.195 ms, 6.30 TB/s; 24 tokens 4.4 us, all latency. Widths, strides or bases that
// rule out 16-byte vectors take the same kernel with shorter ones.
//
// With a cache, rotated keys and the values go to the cache row of the
// token's slot (page = slot / page_size) instead of a dense output: the three
// passes of a separate rotation and scatter become one.
#include "common.cuh"
#include "launch.h"

namespace tfb {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotRows = 4;  // heads per thread, all requested before the angles are formed

struct RotaryK {
  RotaryArgs a;
  int units;       // work units per head (vector pairs or single vectors)
  int rot_units;   // of these, units that are rotated; the rest are copied
  int groups;      // threads per unit and token: head groups per block
  int tok_block;   // tokens per block
  int rows;        // q heads + k heads + v heads (cache form)
  int* status;
};

template <int VEC>
struct VecOf;
template <>
struct VecOf<8> {
  using T = uint4;
};
template <>
struct VecOf<4> {
  using T = uint2;
};
template <>
struct VecOf<2> {
  using T = uint32_t;
};
template <>
struct VecOf<1> {
  using T = uint16_t;
};

template <int DT>
__device__ __forceinline__ float widen(uint16_t h) {
  if constexpr (DT == kDtBF16) {
    return __uint_as_float(static_cast<uint32_t>(h) << 16);
  } else {
    return __half2float(__ushort_as_half(h));
  }
}

template <int DT>
__device__ __forceinline__ uint16_t narrow(float x) {
  if constexpr (DT == kDtBF16) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  } else {
    return __half_as_ushort(__float2half_rn(x));
  }
}

// One unit: PAIR true: vectors at a and b whose elements pair up; false: one
// vector of adjacent pairs (interleaved layout, VEC >= 2).
template <int VEC, bool PAIR, int DT>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryK p) {
  using V = typename VecOf<VEC>::T;
  constexpr int NA = PAIR ? VEC : VEC / 2;  // angles per unit
  extern __shared__ float s_cs[];           // [tok_block][rot/2] cosines, then the sines
  __shared__ long long s_slot[kRotThreads];  // cache offset of each token, -1: not written
  const RotaryArgs& a = p.a;
  pdl_wait();
  pdl_trigger();

  const int half = a.rot >> 1;
  const int per_tok = p.units * p.groups;
  const int tid = threadIdx.x;
  const int tl = tid / per_tok;
  const int rem = tid - tl * per_tok;
  const int grp = rem / p.units;
  const int u = rem - grp * p.units;
  const long long t0 = static_cast<long long>(blockIdx.x) * p.tok_block;
  const long long t = t0 + tl;
  const bool live = tl < p.tok_block && t < a.tokens;
  const bool turn = u < p.rot_units;

  // element offsets of the unit within its head
  int ea, eb;
  if constexpr (PAIR) {
    if (turn) {
      ea = a.interleaved ? 2 * u : u * VEC;  // interleaved: VEC == 1
      eb = a.interleaved ? 2 * u + 1 : half + u * VEC;
    } else {
      ea = eb = a.rot + (u - p.rot_units) * VEC;
    }
  } else {
    ea = eb = u * VEC;
  }

  const int row0 = (blockIdx.y * p.groups + grp) * kRotRows;
  V va[kRotRows], vb[kRotRows];
#pragma unroll
  for (int i = 0; i < kRotRows; ++i) {
    const int row = row0 + i;
    if (live && row < p.rows) {
      const uint16_t* src;
      if (row < a.heads) {
        src = static_cast<const uint16_t*>(a.q) + t * a.q_ts + row * a.q_hs;
      } else if (row < a.heads + a.kv_heads) {
        src = static_cast<const uint16_t*>(a.k) + t * a.k_ts + (row - a.heads) * a.k_hs;
      } else {
        src = static_cast<const uint16_t*>(a.v) + t * a.v_ts + (row - a.heads - a.kv_heads) * a.v_hs;
      }
      va[i] = *reinterpret_cast<const V*>(src + ea);
      if (PAIR && turn) vb[i] = *reinterpret_cast<const V*>(src + eb);
    }
  }

  // angles of the block's tokens, shared by all heads
  float* s_cos = s_cs;
  float* s_sin = s_cs + p.tok_block * half;
  for (int i = tid; i < p.tok_block * half; i += blockDim.x) {
    const long long tok = t0 + i / half;
    if (tok < a.tokens) {
      const double turns = static_cast<double>(a.positions[tok]) * (a.freqs[i % half] * 0.15915494309189533577);
      float sn, cs;
      sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn, &cs);
      s_cos[i] = cs * a.mscale;
      s_sin[i] = sn * a.mscale;
    }
  }
  if (a.k_cache != nullptr) {
    for (int i = tid; i < p.tok_block; i += blockDim.x) {
      long long off = -1;
      if (t0 + i < a.tokens) {
        const long long slot = a.slots[t0 + i];
        if (slot >= 0) {
          const long long page = slot / a.page_size;
          if (page < a.num_pages) {
            off = page * a.c_ps + (slot - page * a.page_size) * a.c_ts;
          } else if (blockIdx.y == 0) {
            record_bad_index(p.status);
          }
        }
      }
      s_slot[i] = off;
    }
  }
  __syncthreads();
  if (!live) return;

  float cs[NA], sn[NA];
  if (turn) {
    const int base = tl * half + (PAIR ? u * VEC : u * (VEC / 2));
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      cs[i] = s_cos[base + i];
      sn[i] = s_sin[base + i];
    }
  }
#pragma unroll
  for (int i = 0; i < kRotRows; ++i) {
    const int row = row0 + i;
    if (row >= p.rows) break;
    uint16_t* dst;
    if (row < a.heads) {
      dst = static_cast<uint16_t*>(a.q_out) + t * a.qo_ts + row * a.qo_hs;
    } else if (a.k_cache == nullptr) {
      dst = static_cast<uint16_t*>(a.k_out) + t * a.ko_ts + (row - a.heads) * a.ko_hs;
    } else {
      const long long off = s_slot[tl];
      if (off < 0) continue;
      const bool is_k = row < a.heads + a.kv_heads;
      const int h = row - a.heads - (is_k ? 0 : a.kv_heads);
      dst = static_cast<uint16_t*>(is_k ? a.k_cache : a.v_cache) + off + h * a.c_hs;
    }
    if (turn && row < a.heads + a.kv_heads) {
      uint16_t* xa = reinterpret_cast<uint16_t*>(&va[i]);
      if constexpr (PAIR) {
        uint16_t* xb = reinterpret_cast<uint16_t*>(&vb[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float x = widen<DT>(xa[j]), y = widen<DT>(xb[j]);
          xa[j] = narrow<DT>(x * cs[j] - y * sn[j]);
          xb[j] = narrow<DT>(x * sn[j] + y * cs[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          const float x = widen<DT>(xa[2 * j]), y = widen<DT>(xa[2 * j + 1]);
          xa[2 * j] = narrow<DT>(x * cs[j] - y * sn[j]);
          xa[2 * j + 1] = narrow<DT>(x * sn[j] + y * cs[j]);
        }
      }
    }
    *reinterpret_cast<V*>(dst + ea) = va[i];
    if (PAIR && turn) *reinterpret_cast<V*>(dst + eb) = vb[i];
  }
}

// Largest vector width every access of the call allows.
int vector_width(const RotaryArgs& a) {
  const int half = a.rot / 2;
  uint64_t bits = static_cast<uint64_t>(a.rot) | static_cast<uint64_t>(a.head_dim);
  if (!a.interleaved) bits |= static_cast<uint64_t>(half);
  auto add = [&](const void* base, long long ts, long long hs) {
    if (base != nullptr)
      bits |= (reinterpret_cast<uintptr_t>(base) / 2) | static_cast<uint64_t>(ts) | static_cast<uint64_t>(hs);
  };
  add(a.q, a.q_ts, a.q_hs);
  add(a.q_out, a.qo_ts, a.qo_hs);
  add(a.k, a.k_ts, a.k_hs);
  add(a.k_out, a.ko_ts, a.ko_hs);
  add(a.v, a.v_ts, a.v_hs);
  add(a.k_cache, a.c_ts, a.c_hs);
  add(a.v_cache, a.c_ps, a.c_ps);
  return bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
}

template <int VEC, bool PAIR>
cudaError_t launch_vec(RotaryK& k, cudaStream_t stream) {
  const RotaryArgs& a = k.a;
  k.rot_units = PAIR ? a.rot / 2 / VEC : a.rot / VEC;
  k.units = k.rot_units + (a.head_dim - a.rot) / VEC;
  const int want = (k.rows + kRotRows - 1) / kRotRows;  // head groups that cover the rows
  k.groups = want * k.units <= kRotThreads ? want : kRotThreads / k.units;
  k.tok_block = kRotThreads / (k.units * k.groups);
  if (k.tok_block > a.tokens) k.tok_block = static_cast<int>(a.tokens);
  const unsigned gy = static_cast<unsigned>((want + k.groups - 1) / k.groups);
  const unsigned gx = static_cast<unsigned>((a.tokens + k.tok_block - 1) / k.tok_block);
  const int threads = (k.tok_block * k.units * k.groups + 31) / 32 * 32;
  const size_t smem = static_cast<size_t>(k.tok_block) * a.rot * sizeof(float);
  if (a.bf16) return launch_k(rotary_kernel<VEC, PAIR, kDtBF16>, dim3(gx, gy), dim3(threads), smem, stream, k);
  return launch_k(rotary_kernel<VEC, PAIR, kDtF16>, dim3(gx, gy), dim3(threads), smem, stream, k);
}

}  // namespace

int rotary_check(const RotaryArgs& a, const char* fn) {
  if (a.tokens < 0 || a.tokens > (1ll << 31) - 1) return set_error(TF_ERR_SHAPE, "%s: tokens=%lld", fn, a.tokens);
  if (a.heads < 0 || a.kv_heads < 0 || a.heads > 4096 || a.kv_heads > 4096 || a.heads + a.kv_heads == 0)
    return set_error(TF_ERR_SHAPE, "%s: heads=%d kv_heads=%d", fn, a.heads, a.kv_heads);
  if (a.head_dim < 2 || a.head_dim > 256) return set_error(TF_ERR_SHAPE, "%s: head_dim=%d (2 to 256)", fn, a.head_dim);
  if (a.rot < 2 || a.rot % 2 || a.rot > a.head_dim)
    return set_error(TF_ERR_SHAPE, "%s: rotated width %d (even, 2 to head_dim)", fn, a.rot);
  if (!(a.mscale - a.mscale == 0.0f)) return set_error(TF_ERR_SHAPE, "%s: mscale must be finite", fn);
  if (a.tokens == 0) return TF_OK;
  if ((a.heads && (a.q == nullptr || a.q_out == nullptr)) || a.positions == nullptr || a.freqs == nullptr)
    return set_error(TF_ERR_SHAPE, "%s: null operand", fn);
  const bool cache = a.k_cache != nullptr || a.v_cache != nullptr;
  if (a.kv_heads && (a.k == nullptr || (!cache && a.k_out == nullptr)))
    return set_error(TF_ERR_SHAPE, "%s: null operand", fn);
  if (cache) {
    if (a.k_cache == nullptr || a.v_cache == nullptr || a.v == nullptr || a.slots == nullptr || a.kv_heads == 0)
      return set_error(TF_ERR_SHAPE, "%s: null operand", fn);
    if (a.page_size < 1 || a.num_pages < 0) return set_error(TF_ERR_SHAPE, "%s: page_size=%lld", fn, a.page_size);
  }
  for (const void* ptr : {a.q, static_cast<const void*>(a.q_out), a.k, static_cast<const void*>(a.k_out), a.v,
                          static_cast<const void*>(a.k_cache), static_cast<const void*>(a.v_cache)})
    if (reinterpret_cast<uintptr_t>(ptr) % 2) return set_error(TF_ERR_ALIGN, "%s: operands must be 2-byte aligned", fn);
  for (const void* ptr : {static_cast<const void*>(a.positions), static_cast<const void*>(a.freqs),
                          static_cast<const void*>(a.slots)})
    if (reinterpret_cast<uintptr_t>(ptr) % 8)
      return set_error(TF_ERR_ALIGN, "%s: positions, freqs and slots must be 8-byte aligned", fn);
  if ((a.heads && !rows_apart(a.head_dim, {{a.qo_ts, a.tokens}, {a.qo_hs, a.heads}})) ||
      (a.kv_heads && !cache && !rows_apart(a.head_dim, {{a.ko_ts, a.tokens}, {a.ko_hs, a.kv_heads}})) ||
      (cache && !rows_apart(a.head_dim, {{a.c_ps, a.num_pages}, {a.c_ts, a.page_size}, {a.c_hs, a.kv_heads}})))
    return set_error(TF_ERR_SHAPE, "%s: rows of an output overlap", fn);
  return TF_OK;
}

int rotary(const RotaryArgs& a, cudaStream_t stream) {
  if (a.tokens == 0) return TF_OK;
  RotaryK k = {};
  k.a = a;
  k.rows = a.heads + a.kv_heads * (a.k_cache != nullptr ? 2 : 1);
  k.status = device_status_ptr();
  if (k.status == nullptr) return last_error_code();
  const int vec = vector_width(a);
  cudaError_t e;
  if (a.interleaved) {
    e = vec == 8   ? launch_vec<8, false>(k, stream)
        : vec == 4 ? launch_vec<4, false>(k, stream)
        : vec == 2 ? launch_vec<2, false>(k, stream)
                   : launch_vec<1, true>(k, stream);
  } else {
    e = vec == 8   ? launch_vec<8, true>(k, stream)
        : vec == 4 ? launch_vec<4, true>(k, stream)
        : vec == 2 ? launch_vec<2, true>(k, stream)
                   : launch_vec<1, true>(k, stream);
  }
  if (e != cudaSuccess) return set_error(TF_ERR_LAUNCH, "rotary launch: %s", cudaGetErrorString(e));
  return TF_OK;
}

}  // namespace tfb
