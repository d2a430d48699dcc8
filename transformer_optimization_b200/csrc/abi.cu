// The C ABI (include/tfb200.h) and the host helpers shared by the launchers:
// error messages, per-device properties, the device status word and TMA
// tensor-map encoding through the driver entry point (no libcuda link).
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>

#include <cudaTypedefs.h>

#include <cstdlib>

#include "common.cuh"
#include "launch.h"

namespace tfb {

// Status words written by kernels whose bounded waits ran out, or that met a
// bad index (common.cuh). One set per device (every device that loads this
// library holds its own copy).
__device__ int g_tfb_status[kStatusWords] = {};

namespace {
thread_local char g_msg[512] = "";
thread_local int g_code = TF_OK;

constexpr int kMaxDevices = 64;
struct DeviceInfo {
  bool ready = false;
  int sms = 0;
  int* status = nullptr;
};
DeviceInfo g_dev[kMaxDevices];
std::mutex g_dev_mu;

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

// Resolves per-device properties on first use: the device must be sm_100
// (the library holds sm_100a code only) and the status word's device address
// is looked up with the device current.
DeviceInfo* device_info() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) {
    set_error(TF_ERR_DEVICE, "cudaGetDevice: %s", cudaGetErrorString(e));
    return nullptr;
  }
  if (dev < 0 || dev >= kMaxDevices) {
    set_error(TF_ERR_DEVICE, "device index %d out of range", dev);
    return nullptr;
  }
  DeviceInfo& di = g_dev[dev];
  if (di.ready) return &di;
  std::lock_guard<std::mutex> lk(g_dev_mu);
  if (di.ready) return &di;
  cudaDeviceProp prop;
  e = cudaGetDeviceProperties(&prop, dev);
  if (e != cudaSuccess) {
    set_error(TF_ERR_DEVICE, "cudaGetDeviceProperties: %s", cudaGetErrorString(e));
    return nullptr;
  }
  if (prop.major != 10 || prop.minor != 0) {
    set_error(TF_ERR_UNSUPPORTED, "device %d is sm_%d%d; this library is built for sm_100a only", dev,
              prop.major, prop.minor);
    return nullptr;
  }
  void* addr = nullptr;
  e = cudaGetSymbolAddress(&addr, g_tfb_status);
  if (e != cudaSuccess) {
    set_error(TF_ERR_DEVICE, "cudaGetSymbolAddress(status): %s", cudaGetErrorString(e));
    return nullptr;
  }
  di.sms = prop.multiProcessorCount;
  di.status = static_cast<int*>(addr);
  di.ready = true;
  return &di;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  return g_encode;
}
}  // namespace

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_msg, sizeof(g_msg), fmt, ap);
  va_end(ap);
  g_code = code;
  return code;
}

int last_error_code() { return g_code == TF_OK ? TF_ERR_DEVICE : g_code; }

bool pdl_enabled() {
  static const bool on = [] {
    const char* e = getenv("TFB_PDL");
    return !(e != nullptr && e[0] == '0');
  }();
  return on;
}

int device_sm_count() {
  DeviceInfo* di = device_info();
  return di ? di->sms : 148;
}

int* device_status_ptr() {
  DeviceInfo* di = device_info();
  return di ? di->status : nullptr;
}

static int encode(CUtensorMap* map, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
                  const cuuint32_t* box) {
  auto fn = encode_fn();
  if (fn == nullptr) return set_error(TF_ERR_DRIVER, "cuTensorMapEncodeTiled entry point unavailable");
  cuuint32_t elem[4] = {1, 1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(TF_ERR_DRIVER, "cuTensorMapEncodeTiled failed (CUresult %d)", int(r));
  return TF_OK;
}

int make_tmap_2d_f16(CUtensorMap* map, const void* base, long long inner, long long outer, long long ld,
                     int box_inner, int box_outer) {
  if (!aligned16(base) || (ld * 2) % 16 != 0) return set_error(TF_ERR_ALIGN, "tensor map: base/pitch alignment");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * 2)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_outer)};
  return encode(map, 2, base, dims, strides, box);
}

int make_tmap_3d_f16(CUtensorMap* map, const void* base, long long inner, long long rows, long long batches,
                     long long ld, long long bstride, int box_inner, int box_rows) {
  if (!aligned16(base) || (ld * 2) % 16 != 0 || (bstride * 2) % 16 != 0)
    return set_error(TF_ERR_ALIGN, "tensor map: base/pitch alignment");
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows),
                        static_cast<cuuint64_t>(batches)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld * 2), static_cast<cuuint64_t>(bstride * 2)};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_rows), 1};
  return encode(map, 3, base, dims, strides, box);
}

int make_tmap_4d_f16(CUtensorMap* map, const void* base, const long long (&dims)[4], const long long (&pitch)[3],
                     const int (&box)[4]) {
  if (!aligned16(base)) return set_error(TF_ERR_ALIGN, "tensor map: base alignment");
  cuuint64_t d[4], st[3];
  cuuint32_t bx[4];
  for (int i = 0; i < 4; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i] > 0 ? dims[i] : 1);
    bx[i] = static_cast<cuuint32_t>(box[i]);
  }
  for (int i = 0; i < 3; ++i) {
    // the pitch of an axis of one entry is never used; any valid value stands in
    const long long bytes = dims[i + 1] > 1 ? pitch[i] * 2 : 16;
    if (bytes <= 0 || bytes % 16 != 0 || bytes >= (1ll << 40))
      return set_error(TF_ERR_ALIGN, "tensor map: pitch of %lld elements", pitch[i]);
    st[i] = static_cast<cuuint64_t>(bytes);
  }
  return encode(map, 4, base, d, st, bx);
}

}  // namespace tfb

// ---------------------------------------------------------------------------
// extern "C" entry points
// ---------------------------------------------------------------------------

using tfb::set_error;

static inline cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

static inline int begin_call() {
  tfb::g_msg[0] = '\0';
  tfb::g_code = TF_OK;
  return tfb::device_status_ptr() == nullptr ? tfb::last_error_code() : TF_OK;
}

extern "C" {

int tf_abi_version(void) { return 11; }

const char* tf_last_error(void) { return tfb::g_msg; }

int tf_device_status(int* code, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  if (code == nullptr) return set_error(TF_ERR_SHAPE, "tf_device_status: code is NULL");
  cudaError_t e = cudaStreamSynchronize(as_stream(stream));
  if (e != cudaSuccess) return set_error(TF_ERR_DEVICE, "stream synchronize: %s", cudaGetErrorString(e));
  int words[tfb::kStatusWords] = {};
  e = cudaMemcpyFromSymbol(words, tfb::g_tfb_status, sizeof(words));
  if (e != cudaSuccess) return set_error(TF_ERR_DEVICE, "read status: %s", cudaGetErrorString(e));
  const int zero[tfb::kStatusWords] = {};
  e = cudaMemcpyToSymbol(tfb::g_tfb_status, zero, sizeof(zero));
  if (e != cudaSuccess) return set_error(TF_ERR_DEVICE, "clear status: %s", cudaGetErrorString(e));
  const int host = words[0] != 0 ? words[0] : words[1];
  *code = host;
  if (host == tfb::kDevBadIndex)
    return set_error(TF_ERR_TIMEOUT, "a slot, page, length or offset index outside its array (device code %d)", host);
  return host == 0 ? TF_OK : set_error(TF_ERR_TIMEOUT, "a kernel wait ran out (device code %d)", host);
}

int tf_test_wait_timeout(const void* src, int64_t limit_ns, int* out, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  return tfb::wait_timeout_probe(src, limit_ns, out, as_stream(stream));
}

int tf_ln_residual(const void* x, const void* delta, const float* w, const float* b, float eps,
                   const uint8_t* valid, int64_t M, int64_t D, int flags, void* x_out, void* normed,
                   void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  if (D > (1 << 20)) return set_error(TF_ERR_SHAPE, "ln_residual: D too large");
  return tfb::ln_residual(x, delta, w, b, eps, valid, M, static_cast<int>(D), flags, x_out, normed,
                          as_stream(stream));
}

// Internal epilogue code and operand type of a tf_gemm* epilogue argument
// (TF_EPI_BIAS, TF_EPI_BIAS_GELU or TF_EPI_BIAS_GELU_ROUNDED, optionally
// with TF_EPI_BF16); -1 if it names none of them.
static int gemm_epilogue(int epilogue, int& dtype) {
  dtype = (epilogue & TF_EPI_BF16) ? tfb::kDtBF16 : tfb::kDtF16;
  switch (epilogue & 0xF) {
    case TF_EPI_BIAS: return 0;
    case TF_EPI_BIAS_GELU: return 1;
    case TF_EPI_BIAS_GELU_ROUNDED: return 5;
    default: return -1;
  }
}

// Internal residual epilogue, mask mode and operand type of a
// tf_gemm_residual* mask_mode argument; false if it is malformed.
static bool residual_mode(int mask_mode, int& epi, int& mask, int& dtype) {
  if (mask_mode & ~(3 | TF_RES_X16 | TF_RES_BF16)) return false;
  mask = mask_mode & 3;
  if (mask > 2) return false;
  epi = (mask_mode & TF_RES_X16) ? 4 : 2;
  dtype = (mask_mode & TF_RES_BF16) ? tfb::kDtBF16 : tfb::kDtF16;
  return true;
}

static int gemm_common(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias, void* C,
                       int64_t ldc, int64_t M, int64_t N, int64_t K, int epilogue, int tile_n, int pair,
                       void* stream) {
  if (epilogue & ~(0xF | TF_EPI_W_SPLIT | TF_EPI_BF16)) return set_error(TF_ERR_SHAPE, "tf_gemm: unknown epilogue bits");
  int dtype = 0;
  const int epi = gemm_epilogue(epilogue, dtype);
  if (epi < 0) return set_error(TF_ERR_SHAPE, "tf_gemm: epilogue %d", epilogue & 0xF);
  if ((epilogue & TF_EPI_W_SPLIT) && dtype != tfb::kDtF16)
    return set_error(TF_ERR_SHAPE, "tf_gemm: split weights are fp16 only");
  tfb::GemmCall g = {};
  g.A = A;
  g.lda = lda;
  g.W = W;
  g.ldw = ldw;
  g.bias = bias;
  g.C = C;
  g.ldc = ldc;
  g.M = M;
  g.N = N;
  g.K = K;
  g.epilogue = epi;
  g.dtype = dtype;
  g.a_repeat = (epilogue & TF_EPI_W_SPLIT) ? 2 : 1;
  g.tile_n = tile_n;
  g.pair = pair;
  return tfb::gemm_f16(g, as_stream(stream));
}

int tf_gemm(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias, void* C, int64_t ldc,
            int64_t M, int64_t N, int64_t K, int epilogue, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  return gemm_common(A, lda, W, ldw, bias, C, ldc, M, N, K, epilogue, 0, 0, stream);
}

int tf_gemm_tiled(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias, void* C,
                  int64_t ldc, int64_t M, int64_t N, int64_t K, int epilogue, int tile_n, int pair, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  if (tile_n != 0 && tile_n != 64 && tile_n != 128 && tile_n != 256)
    return set_error(TF_ERR_SHAPE, "tf_gemm_tiled: tile_n=%d (0, 64, 128 or 256)", tile_n);
  if (tile_n != 0 && N % tile_n != 0) return set_error(TF_ERR_SHAPE, "tf_gemm_tiled: N %% tile_n != 0");
  if (pair < 0 || pair > 2) return set_error(TF_ERR_SHAPE, "tf_gemm_tiled: pair=%d (0, 1 or 2)", pair);
  if (pair == 2 && tile_n == 64) return set_error(TF_ERR_SHAPE, "tf_gemm_tiled: 2-SM tiles are 128 or 256 wide");
  return gemm_common(A, lda, W, ldw, bias, C, ldc, M, N, K, epilogue, tile_n, pair, stream);
}

static int gemm_residual_common(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias,
                                const void* x_in, void* x_out, int64_t ldx, const uint8_t* valid, int mask_mode,
                                int64_t M, int64_t N, int64_t K, int w_split, int tile_n, int pair, int* ready,
                                void* stream) {
  int epi = 0, mask = 0, dtype = 0;
  if (!residual_mode(mask_mode, epi, mask, dtype))
    return set_error(TF_ERR_SHAPE, "tf_gemm_residual: mask_mode=%d", mask_mode);
  if (w_split && dtype != tfb::kDtF16) return set_error(TF_ERR_SHAPE, "tf_gemm_residual: split weights are fp16 only");
  if (tile_n != 0 && tile_n != 64 && tile_n != 128 && tile_n != 256)
    return set_error(TF_ERR_SHAPE, "tf_gemm_residual: tile_n=%d (0, 64, 128 or 256)", tile_n);
  if (pair < 0 || pair > 2 || (pair == 2 && tile_n == 64))
    return set_error(TF_ERR_SHAPE, "tf_gemm_residual: pair=%d with tile_n=%d", pair, tile_n);
  tfb::GemmCall g = {};
  g.A = A;
  g.lda = lda;
  g.W = W;
  g.ldw = ldw;
  g.bias = bias;
  g.x_in = x_in;
  g.x_out = x_out;
  g.ldx = ldx;
  g.valid = valid;
  g.mask_mode = mask;
  g.M = M;
  g.N = N;
  g.K = K;
  g.epilogue = epi;
  g.dtype = dtype;
  g.a_repeat = w_split ? 2 : 1;
  g.tile_n = tile_n;
  g.pair = pair;
  g.ready = ready;
  return tfb::gemm_f16(g, as_stream(stream));
}

int tf_gemm_residual(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias,
                     const void* x_in, void* x_out, int64_t ldx, const uint8_t* valid, int mask_mode,
                     int64_t M, int64_t N, int64_t K, int w_split, int tile_n, int pair, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  return gemm_residual_common(A, lda, W, ldw, bias, x_in, x_out, ldx, valid, mask_mode, M, N, K, w_split, tile_n,
                              pair, nullptr, stream);
}

int tf_gemm_residual_ready(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias,
                           const void* x_in, void* x_out, int64_t ldx, const uint8_t* valid, int mask_mode,
                           int64_t M, int64_t N, int64_t K, int w_split, int* ready, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  if (ready == nullptr || reinterpret_cast<uintptr_t>(ready) % 4 != 0)
    return set_error(TF_ERR_ALIGN, "tf_gemm_residual_ready: ready must be a non-null int32 array");
  if (ldx != N) return set_error(TF_ERR_SHAPE, "tf_gemm_residual_ready: x_out must be contiguous (ldx == N)");
  return gemm_residual_common(A, lda, W, ldw, bias, x_in, x_out, ldx, valid, mask_mode, M, N, K, w_split, 0, 0,
                              ready, stream);
}

int tf_ln_ready(const void* x, const float* w, const float* b, float eps, const uint8_t* valid, int64_t M,
                int64_t D, int flags, void* normed, int* ready, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  if (D > (1 << 20)) return set_error(TF_ERR_SHAPE, "ln_ready: D too large");
  return tfb::ln_ready(x, w, b, eps, valid, M, static_cast<int>(D), flags, normed, ready, as_stream(stream));
}

int64_t tf_gemm_splitk_workspace(int64_t M, int64_t N, int64_t K, int splits) {
  if (begin_call()) return -1;
  return tfb::gemm_splitk_workspace_bytes(M, N, K, splits);
}

int tf_gemm_splitk(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias, void* C, int64_t ldc,
                   int64_t M, int64_t N, int64_t K, int epilogue, int splits, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  int dtype = 0;
  const int epi = (epilogue & ~(0xF | TF_EPI_BF16)) ? -1 : gemm_epilogue(epilogue, dtype);
  if (epi < 0) return set_error(TF_ERR_SHAPE, "tf_gemm_splitk: epilogue=%d", epilogue);
  tfb::GemmCall g = {};
  g.A = A;
  g.lda = lda;
  g.W = W;
  g.ldw = ldw;
  g.bias = bias;
  g.C = C;
  g.ldc = ldc;
  g.M = M;
  g.N = N;
  g.K = K;
  g.epilogue = epi;
  g.dtype = dtype;
  g.a_repeat = 1;
  return tfb::gemm_splitk_f16(g, splits, static_cast<float*>(workspace), workspace_bytes, as_stream(stream));
}

int tf_gemm_splitk_static(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias, void* C,
                          int64_t ldc, int64_t M, int64_t N, int64_t K, int epilogue, int splits, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  int dtype = 0;
  const int epi = (epilogue & ~(0xF | TF_EPI_BF16)) ? -1 : gemm_epilogue(epilogue, dtype);
  if (epi < 0) return set_error(TF_ERR_SHAPE, "tf_gemm_splitk_static: epilogue=%d", epilogue);
  tfb::GemmCall g = {};
  g.A = A;
  g.lda = lda;
  g.W = W;
  g.ldw = ldw;
  g.bias = bias;
  g.C = C;
  g.ldc = ldc;
  g.M = M;
  g.N = N;
  g.K = K;
  g.epilogue = epi;
  g.dtype = dtype;
  g.a_repeat = 1;
  return tfb::gemm_splitk_static_f16(g, splits, as_stream(stream));
}

int tf_gemm_residual_splitk(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias,
                            const void* x_in, void* x_out, int64_t ldx, const uint8_t* valid, int mask_mode,
                            int64_t M, int64_t N, int64_t K, int splits, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  int epi = 0, mask = 0, dtype = 0;
  if (!residual_mode(mask_mode, epi, mask, dtype))
    return set_error(TF_ERR_SHAPE, "tf_gemm_residual_splitk: mask_mode=%d", mask_mode);
  tfb::GemmCall g = {};
  g.A = A;
  g.lda = lda;
  g.W = W;
  g.ldw = ldw;
  g.bias = bias;
  g.x_in = x_in;
  g.x_out = x_out;
  g.ldx = ldx;
  g.valid = valid;
  g.mask_mode = mask;
  g.M = M;
  g.N = N;
  g.K = K;
  g.epilogue = epi;
  g.dtype = dtype;
  g.a_repeat = 1;
  return tfb::gemm_splitk_f16(g, splits, static_cast<float*>(workspace), workspace_bytes, as_stream(stream));
}

int tf_gemm_residual_ln_splitk(const void* A, int64_t lda, const void* W, int64_t ldw, const float* bias,
                               const void* x_in, void* x_out, int64_t ldx, const uint8_t* valid, int mask_mode,
                               int64_t M, int64_t N, int64_t K, int splits, void* workspace,
                               int64_t workspace_bytes, const float* ln_w, const float* ln_b, float eps,
                               void* normed, int ln_flags, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  int epi = 0, mask = 0, dtype = 0;
  if (!residual_mode(mask_mode, epi, mask, dtype))
    return set_error(TF_ERR_SHAPE, "tf_gemm_residual_ln_splitk: mask_mode=%d", mask_mode);
  tfb::GemmCall g = {};
  g.A = A;
  g.lda = lda;
  g.W = W;
  g.ldw = ldw;
  g.bias = bias;
  g.x_in = x_in;
  g.x_out = x_out;
  g.ldx = ldx;
  g.valid = valid;
  g.mask_mode = mask;
  g.M = M;
  g.N = N;
  g.K = K;
  g.epilogue = epi;
  g.dtype = dtype;
  g.a_repeat = 1;
  tfb::LnFuse ln = {ln_w, ln_b, eps, normed, ln_flags};
  return tfb::gemm_splitk_f16(g, splits, static_cast<float*>(workspace), workspace_bytes, as_stream(stream), &ln);
}

int tf_flash_fwd(const void* q, const void* k, const void* v, int64_t ld_q, int64_t ld_kv, int64_t bs_q,
                 int64_t bs_kv, void* out, int64_t ld_o, int64_t bs_o, float* lse, const uint8_t* key_valid,
                 int64_t batch, int64_t heads, int64_t seq_q, int64_t seq_k, int64_t head_dim, float scale,
                 int64_t q_pos0, int64_t k_pos0, int flags, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  tfb::AttnArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.ld_q = ld_q;
  a.ld_kv = ld_kv;
  a.bs_q = bs_q;
  a.bs_kv = bs_kv;
  a.out = out;
  a.ld_o = ld_o;
  a.bs_o = bs_o;
  a.lse = lse;
  a.key_valid = key_valid;
  a.batch = batch;
  a.heads = heads;
  a.seq_q = seq_q;
  a.seq_k = seq_k;
  a.head_dim = head_dim;
  a.scale = scale;
  a.q_pos0 = q_pos0;
  a.k_pos0 = k_pos0;
  a.flags = flags;
  return tfb::flash_fwd(a, as_stream(stream));
}

int tf_attn_merge(float* o_acc, float* lse_acc, const float* o_part, const float* lse_part, int64_t ld,
                  int64_t bs, void* out16, int64_t ld16, int64_t bs16, int64_t batch, int64_t heads,
                  int64_t seq_q, int64_t head_dim, void* stream) {
  int rc = begin_call();
  if (rc) return rc;
  tfb::MergeArgs a;
  a.o_acc = o_acc;
  a.lse_acc = lse_acc;
  a.o_part = o_part;
  a.lse_part = lse_part;
  a.ld = ld;
  a.bs = bs;
  a.out16 = out16;
  a.ld16 = ld16;
  a.bs16 = bs16;
  a.batch = batch;
  a.heads = heads;
  a.seq_q = seq_q;
  a.head_dim = head_dim;
  return tfb::attn_merge(a, as_stream(stream));
}

// The serving entry points check their arguments before they look for a
// device, so a malformed call gets the same status on any host.
static inline void clear_message() {
  tfb::g_msg[0] = '\0';
  tfb::g_code = TF_OK;
}

static int narrow_dims(const char* fn, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rot) {
  for (int64_t v : {heads, kv_heads, head_dim, rot})
    if (v < 0 || v > (1 << 20)) return set_error(TF_ERR_SHAPE, "%s: sizes out of range", fn);
  return TF_OK;
}

static int rotary_common(const char* fn, tfb::RotaryArgs& a, int64_t heads, int64_t kv_heads, int64_t head_dim,
                         int64_t rot, int flags, void* stream) {
  clear_message();
  if (flags & ~(TF_ROTARY_INTERLEAVED | TF_ROTARY_BF16)) return set_error(TF_ERR_SHAPE, "%s: unknown flags", fn);
  int rc = narrow_dims(fn, heads, kv_heads, head_dim, rot);
  if (rc) return rc;
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.rot = static_cast<int>(rot);
  a.interleaved = (flags & TF_ROTARY_INTERLEAVED) != 0;
  a.bf16 = (flags & TF_ROTARY_BF16) != 0;
  rc = tfb::rotary_check(a, fn);
  if (rc) return rc;
  rc = begin_call();
  if (rc) return rc;
  return tfb::rotary(a, as_stream(stream));
}

int tf_rotary(const void* q, int64_t q_ts, int64_t q_hs, void* q_out, int64_t qo_ts, int64_t qo_hs, const void* k,
              int64_t k_ts, int64_t k_hs, void* k_out, int64_t ko_ts, int64_t ko_hs, const int64_t* positions,
              const double* freqs, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rot,
              float mscale, int flags, void* stream) {
  tfb::RotaryArgs a = {};
  a.q = q;
  a.q_ts = q_ts;
  a.q_hs = q_hs;
  a.q_out = q_out;
  a.qo_ts = qo_ts;
  a.qo_hs = qo_hs;
  a.k = k;
  a.k_ts = k_ts;
  a.k_hs = k_hs;
  a.k_out = k_out;
  a.ko_ts = ko_ts;
  a.ko_hs = ko_hs;
  a.positions = positions;
  a.freqs = freqs;
  a.tokens = tokens;
  a.mscale = mscale;
  return rotary_common("tf_rotary", a, heads, kv_heads, head_dim, rot, flags, stream);
}

int tf_rotary_append(const void* q, int64_t q_ts, int64_t q_hs, void* q_out, int64_t qo_ts, int64_t qo_hs,
                     const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs,
                     const int64_t* positions, const double* freqs, void* k_cache, void* v_cache, int64_t c_ps,
                     int64_t c_ts, int64_t c_hs, int64_t num_pages, int64_t page_size, const int64_t* slots,
                     int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rot, float mscale,
                     int flags, void* stream) {
  clear_message();
  if (tokens > 0 && (k_cache == nullptr || v_cache == nullptr))
    return set_error(TF_ERR_SHAPE, "tf_rotary_append: null cache");
  tfb::RotaryArgs a = {};
  a.q = q;
  a.q_ts = q_ts;
  a.q_hs = q_hs;
  a.q_out = q_out;
  a.qo_ts = qo_ts;
  a.qo_hs = qo_hs;
  a.k = k;
  a.k_ts = k_ts;
  a.k_hs = k_hs;
  a.v = v;
  a.v_ts = v_ts;
  a.v_hs = v_hs;
  a.positions = positions;
  a.freqs = freqs;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.c_ps = c_ps;
  a.c_ts = c_ts;
  a.c_hs = c_hs;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.slots = slots;
  a.tokens = tokens;
  a.mscale = mscale;
  return rotary_common("tf_rotary_append", a, heads, kv_heads, head_dim, rot, flags, stream);
}

// A caller's "no bound" may be any number: bounds past what the arrays can hold
// (tokens and keys are at most 2^30 and 2^31 - 1, see seq_check) are brought
// down to that before sizes are computed from them, in the call and in its
// workspace query alike.
static void cap_bounds(tfb::SeqArgs& a) {
  a.max_q = std::min(a.max_q, 1ll << 30);
  a.max_k = std::min(a.max_k, (1ll << 31) - 1);
}

static int seq_common(const char* fn, tfb::SeqArgs& a, int64_t heads, int64_t kv_heads, int64_t head_dim, int flags,
                      void* stream) {
  clear_message();
  if (flags & ~(TF_ATTN_CAUSAL | TF_ATTN_OUT_F32 | TF_ATTN_BF16)) return set_error(TF_ERR_SHAPE, "%s: unknown flags", fn);
  int rc = narrow_dims(fn, heads, kv_heads, head_dim, 0);
  if (rc) return rc;
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.causal = (flags & TF_ATTN_CAUSAL) != 0;
  a.out_f32 = (flags & TF_ATTN_OUT_F32) != 0;
  a.bf16 = (flags & TF_ATTN_BF16) != 0;
  cap_bounds(a);
  rc = tfb::seq_check(a, fn);
  if (rc) return rc;
  rc = begin_call();
  if (rc) return rc;
  return tfb::seq_attention(a, as_stream(stream));
}

static int64_t seq_workspace_common(const char* fn, int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads,
                                    int64_t head_dim, int64_t max_q, int64_t max_k, int64_t page_size) {
  clear_message();
  if (narrow_dims(fn, heads, kv_heads, head_dim, 0)) return -1;
  tfb::SeqArgs a = {};
  a.tokens = tokens;
  a.batch = batch;
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.max_q = max_q;
  a.max_k = max_k;
  a.page_size = page_size;
  a.scale = 1.f;
  a.q = a.k = a.v = &a;  // sizes only: the pointer and stride checks see a dense, aligned stand-in
  a.out = &a;
  a.o_hs = head_dim;
  a.o_ts = head_dim * heads;
  a.cu_q = a.cu_k = a.kv_lens = reinterpret_cast<const int*>(&a);
  cap_bounds(a);
  if (tfb::seq_check(a, fn)) return -1;
  if (begin_call()) return -1;
  return tfb::seq_workspace(a);
}

int64_t tf_flash_packed_workspace(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                  int64_t max_q, int64_t max_k) {
  return seq_workspace_common("tf_flash_packed_workspace", tokens, batch, heads, kv_heads, head_dim, max_q, max_k, 0);
}

int64_t tf_flash_paged_workspace(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                 int64_t max_q, int64_t max_k) {
  return seq_workspace_common("tf_flash_paged_workspace", tokens, batch, heads, kv_heads, head_dim, max_q, max_k, 16);
}

int tf_flash_packed(const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs,
                    const void* v, int64_t v_ts, int64_t v_hs, const int32_t* cu_q, const int32_t* cu_k, void* out,
                    int64_t o_ts, int64_t o_hs, float* lse, int64_t tokens, int64_t k_tokens, int64_t batch,
                    int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_q, int64_t max_k, float scale,
                    int flags, void* workspace, int64_t workspace_bytes, void* stream) {
  tfb::SeqArgs a = {};
  a.q = q;
  a.q_ts = q_ts;
  a.q_hs = q_hs;
  a.k = k;
  a.k_ts = k_ts;
  a.k_hs = k_hs;
  a.v = v;
  a.v_ts = v_ts;
  a.v_hs = v_hs;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.out = out;
  a.o_ts = o_ts;
  a.o_hs = o_hs;
  a.lse = lse;
  a.tokens = tokens;
  a.k_tokens = k_tokens;
  a.batch = batch;
  a.max_q = max_q;
  a.max_k = max_k;
  a.scale = scale;
  a.workspace = workspace;
  a.workspace_bytes = workspace_bytes;
  return seq_common("tf_flash_packed", a, heads, kv_heads, head_dim, flags, stream);
}

int tf_flash_paged(const void* q, int64_t q_ts, int64_t q_hs, const void* k_cache, const void* v_cache, int64_t c_ps,
                   int64_t c_ts, int64_t c_hs, int64_t num_pages, int64_t page_size, const int32_t* page_table,
                   int64_t table_ld, int64_t max_pages, const int32_t* cu_q, const int32_t* kv_lens, void* out,
                   int64_t o_ts, int64_t o_hs, float* lse, int64_t tokens, int64_t batch, int64_t heads,
                   int64_t kv_heads, int64_t head_dim, int64_t max_q, int64_t max_k, float scale, int flags,
                   void* workspace, int64_t workspace_bytes, void* stream) {
  clear_message();
  if (page_size <= 0) return set_error(TF_ERR_SHAPE, "tf_flash_paged: page_size=%lld", static_cast<long long>(page_size));
  tfb::SeqArgs a = {};
  a.q = q;
  a.q_ts = q_ts;
  a.q_hs = q_hs;
  a.k = k_cache;
  a.v = v_cache;
  a.k_ps = a.v_ps = c_ps;
  a.k_ts = a.v_ts = c_ts;
  a.k_hs = a.v_hs = c_hs;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.page_table = page_table;
  a.table_ld = table_ld;
  a.max_pages = max_pages;
  a.cu_q = cu_q;
  a.kv_lens = kv_lens;
  a.out = out;
  a.o_ts = o_ts;
  a.o_hs = o_hs;
  a.lse = lse;
  a.tokens = tokens;
  a.batch = batch;
  a.max_q = max_q;
  a.max_k = max_k;
  a.scale = scale;
  a.workspace = workspace;
  a.workspace_bytes = workspace_bytes;
  return seq_common("tf_flash_paged", a, heads, kv_heads, head_dim, flags, stream);
}

}  // extern "C"
