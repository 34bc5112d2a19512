// C-ABI layer of libsma.so: argument validation, dispatch to the kernel
// launchers, the thread-local error message, and the device error word the
// kernels raise when a bounded wait gives up.
//
// Mirrors the reference pybind layer (csrc/binding.cpp:9-71), whose checks
// (CUDA tensors, 4-D shapes, fp16/bf16 dtype) become SMA_* status codes here;
// the Python shim turns them into RuntimeError like TORCH_CHECK does.
#include <atomic>
#include <cfloat>
#include <cstdio>
#include <string>

#include <nvtx3/nvToolsExt.h>

#include "sma_capi.h"
#include "sma_internal.h"

namespace {

thread_local std::string g_last_error;
std::atomic<uint64_t> g_timeout_ns{2000000000ull};

// NVTX range over one entry point (host side: argument checks and launches).
// nvtx3 is header-only and costs a branch when no profiler is attached.
struct NvtxRange {
  explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
  NvtxRange(const NvtxRange&) = delete;
  NvtxRange& operator=(const NvtxRange&) = delete;
};

// Device word the kernels OR error bits into (one instance per device).
__device__ uint32_t g_device_error_word;

using sma::kMaxDevices;
// Per-device address caches.  Several host threads may fill an entry on their
// first call; they all store the same value, and the atomics make that
// well-defined.
std::atomic<uint32_t*> g_err_ptr[kMaxDevices] = {};

int fail(int code, const char* msg) {
  g_last_error = msg ? msg : "unknown error";
  return code;
}

int fail_cuda(cudaError_t e, const char* where) {
  g_last_error = std::string(where) + ": " + cudaGetErrorString(e);
  return sma::kErrCuda;
}

// Device address of the error word on the current device.  Every entry point
// that launches calls this first; it also makes the device's primary context
// current on the calling thread, which the runtime otherwise binds only at the
// thread's first runtime call that needs it, while the tensor-map encoding
// (a driver call) needs it bound already.  A host thread whose first CUDA
// work is a call into this library (an autograd worker, say) would otherwise
// fail there.
int error_word(uint32_t** out) {
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fail_cuda(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(sma::kErrCuda, "device index out of range");
  e = cudaSetDevice(dev);
  if (e != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  uint32_t* ptr = g_err_ptr[dev].load(std::memory_order_relaxed);
  if (ptr == nullptr) {
    void* p = nullptr;
    e = cudaGetSymbolAddress(&p, g_device_error_word);
    if (e != cudaSuccess) return fail_cuda(e, "cudaGetSymbolAddress");
    ptr = static_cast<uint32_t*>(p);
    g_err_ptr[dev].store(ptr, std::memory_order_relaxed);
  }
  *out = ptr;
  return sma::kOk;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Fixed device scratch of sma_attn_bwd_noalloc: the FP32 dQ accumulator
// (B*H*N*D floats) followed by Delta (B*H*N floats).  One copy per device,
// part of the module image (so it is reserved on every device where the
// library's module is loaded, whether or not the entry point is called),
// so that entry point allocates nothing.
constexpr int64_t kNoAllocScratchFloats = int64_t{8} << 20;  // 32 MiB
static __device__ __align__(256) float g_bwd_noalloc_scratch[kNoAllocScratchFloats];
std::atomic<float*> g_noalloc_ptr[kMaxDevices] = {};

// Device address of the fixed scratch on the current device (looked up once per device).
int noalloc_scratch(float** out) {
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fail_cuda(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(sma::kErrCuda, "device index out of range");
  float* ptr = g_noalloc_ptr[dev].load(std::memory_order_relaxed);
  if (ptr == nullptr) {
    void* p = nullptr;
    e = cudaGetSymbolAddress(&p, g_bwd_noalloc_scratch);
    if (e != cudaSuccess) return fail_cuda(e, "cudaGetSymbolAddress");
    ptr = static_cast<float*>(p);
    g_noalloc_ptr[dev].store(ptr, std::memory_order_relaxed);
  }
  *out = ptr;
  return sma::kOk;
}


// Checks of the arguments that every entry point on sma_attn_args shares;
// fills `p`.  Sets `*empty` when there is nothing to write.
int cross_params(const sma_attn_args* a, void* stream, sma::CrossParams* p, bool* empty) {
  *empty = false;
  if (a == nullptr) return fail(sma::kErrArg, "attention: null arguments");
  if (a->dtype != SMA_DTYPE_FP16 && a->dtype != SMA_DTYPE_BF16)
    return fail(sma::kErrDtype, "attention: unsupported dtype, need fp16 or bf16");
  constexpr int64_t kMax = int64_t{1} << 30;
  if (a->B < 0 || a->H < 0 || a->Hkv < 0 || a->Nq < 0 || a->Nk < 0 || a->P < 0 || a->D <= 0)
    return fail(sma::kErrArg, "attention: bad dimension");
  if (a->D != 64 && a->D != 128) return fail(sma::kErrUnsupportedD, "attention: head dim must be 64 or 128");
  if (a->Nq > kMax || a->Nk > kMax || a->P > kMax)
    return fail(sma::kErrUnsupportedN, "attention: sequence length above 2^30");
  if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return fail(sma::kErrArg, "attention: scale must be finite and > 0");
  if (a->B == 0 || a->H == 0 || a->Nq == 0) {
    *empty = true;
    return sma::kOk;
  }
  if (a->B > kMax || a->H > kMax || a->Hkv == 0 || a->H % a->Hkv != 0)
    return fail(sma::kErrArg, "attention: the key heads must divide the query heads");
  if (!a->q || !a->out || (a->Nk > 0 && (!a->k || !a->v)) || (a->P > 0 && (!a->k_prefix || !a->v_prefix)))
    return fail(sma::kErrArg, "attention: null pointer");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_prefix) || !aligned16(a->v_prefix) ||
      !aligned16(a->out))
    return fail(sma::kErrArg, "attention: q/k/v/out must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(a->lse) & 3u) return fail(sma::kErrArg, "attention: lse must be 4-byte aligned");
  // Strides of axes that are stepped along: positive multiples of 16 bytes (8 elements).
  auto strides_ok = [](const int64_t* s, const int64_t* n, int axes) {
    for (int i = 0; i < axes; ++i)
      if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 != 0 || s[i] >= (int64_t{1} << 38))) return false;
    return true;
  };
  const int64_t nq[3] = {a->B, a->H, a->Nq}, nk[3] = {a->B, a->Hkv, a->Nk}, npre[2] = {a->Hkv, a->P};
  if (!strides_ok(a->q_stride, nq, 3) || (a->Nk > 0 && (!strides_ok(a->k_stride, nk, 3) || !strides_ok(a->v_stride, nk, 3))) ||
      (a->P > 0 && (!strides_ok(a->kp_stride, npre, 2) || !strides_ok(a->vp_stride, npre, 2))))
    return fail(sma::kErrArg, "attention: strides must be positive multiples of 8 elements");
  if (a->mask && a->lengths) return fail(sma::kErrArg, "attention: give a mask or lengths, not both");
  if (reinterpret_cast<uintptr_t>(a->lengths) & 3u) return fail(sma::kErrArg, "attention: lengths must be 4-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (a->mask && a->mask_stride[i] < 0) return fail(sma::kErrArg, "attention: negative mask stride");
  if (a->bias_table) {
    if (a->P > 0) return fail(sma::kErrArg, "attention: no bias together with a prefix");
    if (a->bias_side < 1 || a->bias_side > SMA_MAX_BIAS_SIDE || !a->bias_starts)
      return fail(sma::kErrArg, "attention: a bias needs 1 to 128 bucket starts for a side");
    if (a->bias_offset <= -kMax || a->bias_offset >= kMax) return fail(sma::kErrArg, "attention: bias offset out of range");
    if ((reinterpret_cast<uintptr_t>(a->bias_table) & 1u) || (reinterpret_cast<uintptr_t>(a->bias_offsets) & 3u))
      return fail(sma::kErrArg, "attention: misaligned bias table or offsets");
    for (int i = 0; i < a->bias_side; ++i)
      if (a->bias_starts[i] < 0 || (i == 0 ? a->bias_starts[0] != 0 : a->bias_starts[i] < a->bias_starts[i - 1]))
        return fail(sma::kErrArg, "attention: bucket starts must ascend from 0");
    if (a->bias_two_sided && a->bias_starts[a->bias_side - 1] == 0)
      return fail(sma::kErrArg, "attention: a two-sided bias needs a bucket start above 0");
  }
  p->dtype = a->dtype;
  p->q = a->q;
  p->k = a->k;
  p->v = a->v;
  p->k_prefix = a->k_prefix;
  p->v_prefix = a->v_prefix;
  for (int i = 0; i < 3; ++i) {
    p->q_stride[i] = a->q_stride[i];
    p->k_stride[i] = a->k_stride[i];
    p->v_stride[i] = a->v_stride[i];
    p->mask_stride[i] = a->mask_stride[i];
  }
  for (int i = 0; i < 2; ++i) {
    p->kp_stride[i] = a->kp_stride[i];
    p->vp_stride[i] = a->vp_stride[i];
  }
  p->mask = static_cast<const uint8_t*>(a->mask);
  p->lengths = a->lengths;
  p->bias.table = a->bias_table;
  p->bias.offsets = a->bias_offsets;
  p->bias.offset = static_cast<int>(a->bias_offset);
  p->bias.H = static_cast<int>(a->H);
  p->bias.side = a->bias_side;
  p->bias.two_sided = a->bias_two_sided != 0;
  if (a->bias_table)
    for (int i = 0; i < a->bias_side; ++i) p->bias.starts[i] = a->bias_starts[i];
  p->out = a->out;
  p->lse = a->lse;
  p->B = a->B;
  p->H = a->H;
  p->Hkv = a->Hkv;
  p->Nq = a->Nq;
  p->Nk = a->Nk;
  p->D = a->D;
  p->P = a->P;
  p->scale = a->scale;
  p->timeout_ns = g_timeout_ns.load(std::memory_order_relaxed);
  p->stream = static_cast<cudaStream_t>(stream);
  return sma::kOk;
}

// What needs the device, once all arguments have been checked.
int device_params(sma::CrossParams* p) { return error_word(&p->err_word); }

}  // namespace

extern "C" {

int sma_pack_mask(const void* mask, void* packed, int64_t B, int64_t H, int64_t N, void* stream) {
  NvtxRange range("sma_pack_mask");
  if (B < 0 || H < 0 || N < 0) return fail(sma::kErrArg, "pack_mask: negative dimension");
  if (B == 0 || H == 0 || N == 0) return sma::kOk;
  if (mask == nullptr || packed == nullptr) return fail(sma::kErrArg, "pack_mask: null pointer");
  const char* msg = nullptr;
  int rc = sma::launch_pack_mask(static_cast<const uint8_t*>(mask), static_cast<uint32_t*>(packed), B * H * N,
                                 N, static_cast<cudaStream_t>(stream), &msg);
  return rc == sma::kOk ? rc : fail(rc, msg);
}

}  // extern "C"

namespace {

// bool_mask != nullptr: the forward reads the bool mask itself and writes the
// packed words to mask_packed (sma_attn_fwd_mask).
int attn_fwd_impl(int dtype, const void* q, const void* k, const void* v, const void* mask_packed,
                  const uint32_t* occupancy, const void* bool_mask, void* out, float* lse, int64_t B, int64_t H,
                  int64_t N, int64_t D, float scale, void* stream) {
  NvtxRange range(bool_mask != nullptr ? "sma_attn_fwd_mask" : "sma_attn_fwd");
  if (dtype != SMA_DTYPE_FP16 && dtype != SMA_DTYPE_BF16)
    return fail(sma::kErrDtype, "attention: unsupported dtype, need fp16 or bf16");
  if (B < 0 || H < 0 || N < 0 || D <= 0) return fail(sma::kErrArg, "attention: bad dimension");
  if (D != 64 && D != 128) return fail(sma::kErrUnsupportedD, "attention: head dim must be 64 or 128");
  if (N > SMA_MAX_SEQ_LEN)
    return fail(sma::kErrUnsupportedN, "attention: sequence length above the supported maximum (65536)");
  if (occupancy != nullptr && N > SMA_MAX_SEQ_LEN_OCCUPANCY)
    return fail(sma::kErrUnsupportedN, "attention: occupancy map given for a sequence length above 8192");
  if (!(scale > 0.f) || !(scale < INFINITY)) return fail(sma::kErrArg, "attention: scale must be finite and > 0");
  if (B == 0 || H == 0 || N == 0) return sma::kOk;
  if (!q || !k || !v || !mask_packed || !out) return fail(sma::kErrArg, "attention: null pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(sma::kErrArg, "attention: q/k/v/out must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(mask_packed) & 3u) != 0 || (lse && (reinterpret_cast<uintptr_t>(lse) & 3u)))
    return fail(sma::kErrArg, "attention: mask_packed/lse must be 4-byte aligned");
  if (bool_mask != nullptr && (N % 32 != 0 || !aligned16(bool_mask) || !aligned16(mask_packed)))
    return fail(sma::kErrArg, "attention: the bool-mask forward needs N % 32 == 0 and 16-byte aligned mask / mask_packed");
  uint32_t* err = nullptr;
  int rc = error_word(&err);
  if (rc != sma::kOk) return rc;
  sma::AttnParams p{};
  p.dtype = dtype;
  p.q = q;
  p.k = k;
  p.v = v;
  p.mask = static_cast<const uint32_t*>(mask_packed);
  p.occ = occupancy;
  p.bmask = static_cast<const uint8_t*>(bool_mask);
  p.packed_out = bool_mask != nullptr ? static_cast<uint32_t*>(const_cast<void*>(mask_packed)) : nullptr;
  p.out = out;
  p.lse = lse;
  p.B = B;
  p.H = H;
  p.N = N;
  p.D = D;
  p.scale = scale;
  p.err_word = err;
  p.timeout_ns = g_timeout_ns.load(std::memory_order_relaxed);
  p.stream = static_cast<cudaStream_t>(stream);
  const char* msg = nullptr;
  rc = sma::launch_attn_fwd(p, &msg);
  return rc == sma::kOk ? rc : fail(rc, msg);
}

}  // namespace

extern "C" {

int sma_attn_fwd(int dtype, const void* q, const void* k, const void* v, const void* mask_packed, void* out,
                 float* lse, int64_t B, int64_t H, int64_t N, int64_t D, float scale, void* stream) {
  return attn_fwd_impl(dtype, q, k, v, mask_packed, nullptr, nullptr, out, lse, B, H, N, D, scale, stream);
}

int sma_attn_fwd_mask(int dtype, const void* q, const void* k, const void* v, const void* mask, void* mask_packed,
                      void* out, float* lse, int64_t B, int64_t H, int64_t N, int64_t D, float scale, void* stream) {
  if (mask == nullptr && B > 0 && H > 0 && N > 0) return fail(sma::kErrArg, "attention: null mask");
  return attn_fwd_impl(dtype, q, k, v, mask_packed, nullptr, mask, out, lse, B, H, N, D, scale, stream);
}

int sma_pack_mask_occupancy(const void* mask, void* packed, void* occupancy, int64_t B, int64_t H, int64_t N,
                            void* stream) {
  NvtxRange range("sma_pack_mask_occupancy");
  if (B < 0 || H < 0 || N < 0) return fail(sma::kErrArg, "pack_mask_occupancy: negative dimension");
  if (N > SMA_MAX_SEQ_LEN_OCCUPANCY)
    return fail(sma::kErrUnsupportedN, "pack_mask_occupancy: sequence length above the occupancy map's maximum (8192)");
  if (B == 0 || H == 0 || N == 0) return sma::kOk;
  const char* msg = nullptr;
  int rc = sma::launch_pack_mask_occ(static_cast<const uint8_t*>(mask), static_cast<uint32_t*>(packed),
                                     static_cast<uint32_t*>(occupancy), B * H, N,
                                     static_cast<cudaStream_t>(stream), &msg);
  return rc == sma::kOk ? rc : fail(rc, msg);
}

int sma_attn_fwd_occupancy(int dtype, const void* q, const void* k, const void* v, const void* mask_packed,
                           const void* occupancy, void* out, float* lse, int64_t B, int64_t H, int64_t N,
                           int64_t D, float scale, void* stream) {
  if (occupancy == nullptr) return fail(sma::kErrArg, "attention: null occupancy map");
  if ((reinterpret_cast<uintptr_t>(occupancy) & 3u) != 0)
    return fail(sma::kErrArg, "attention: occupancy map must be 4-byte aligned");
  return attn_fwd_impl(dtype, q, k, v, mask_packed, static_cast<const uint32_t*>(occupancy), nullptr, out, lse, B, H,
                       N, D, scale, stream);
}

int sma_attn_bwd(int dtype, const void* q, const void* k, const void* v, const void* out, const void* dout,
                 const float* lse, const void* mask_packed, void* dq, void* dk, void* dv, float* dq_accum, float* delta,
                 int64_t B, int64_t H, int64_t N, int64_t D, float scale, void* stream) {
  NvtxRange range("sma_attn_bwd");
  if (dtype != SMA_DTYPE_FP16 && dtype != SMA_DTYPE_BF16)
    return fail(sma::kErrDtype, "backward: unsupported dtype, need fp16 or bf16");
  if (B < 0 || H < 0 || N < 0 || D <= 0) return fail(sma::kErrArg, "backward: bad dimension");
  if (D != 64 && D != 128) return fail(sma::kErrUnsupportedD, "backward: head dim must be 64 or 128");
  if (N > SMA_MAX_SEQ_LEN) return fail(sma::kErrUnsupportedN, "backward: sequence length above the supported maximum (65536)");
  if (!(scale > 0.f) || !(scale < INFINITY)) return fail(sma::kErrArg, "backward: scale must be finite and > 0");
  if (B == 0 || H == 0 || N == 0) return sma::kOk;
  if (!q || !k || !v || !out || !dout || !lse || !mask_packed || !dq || !dk || !dv || !dq_accum || !delta)
    return fail(sma::kErrArg, "backward: null pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(dout) || !aligned16(dq) ||
      !aligned16(dk) || !aligned16(dv) || !aligned16(dq_accum))
    return fail(sma::kErrArg, "backward: q/k/v/out/dout/dq/dk/dv/dq_accum must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(lse) & 3u) || (reinterpret_cast<uintptr_t>(delta) & 3u) ||
      (reinterpret_cast<uintptr_t>(mask_packed) & 3u))
    return fail(sma::kErrArg, "backward: lse/delta/mask_packed must be 4-byte aligned");
  uint32_t* err = nullptr;
  int rc = error_word(&err);
  if (rc != sma::kOk) return rc;
  sma::BwdParams p{};
  p.dtype = dtype;
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.dout = dout;
  p.lse = lse;
  p.mask = static_cast<const uint32_t*>(mask_packed);
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.dq_accum = dq_accum;
  p.delta = delta;
  p.B = B;
  p.H = H;
  p.N = N;
  p.D = D;
  p.scale = scale;
  p.err_word = err;
  p.timeout_ns = g_timeout_ns.load(std::memory_order_relaxed);
  p.stream = static_cast<cudaStream_t>(stream);
  const char* msg = nullptr;
  rc = sma::launch_attn_bwd(p, &msg);
  return rc == sma::kOk ? rc : fail(rc, msg);
}

int sma_attn_bwd_noalloc(int dtype, const void* q, const void* k, const void* v, const void* out, const void* dout,
                         const float* lse, const void* mask_packed, void* dq, void* dk, void* dv, int64_t B,
                         int64_t H, int64_t N, int64_t D, float scale, void* stream) {
  // The checks of sma_attn_bwd, with its codes, come first; then the size
  // of the fixed scratch.
  if (dtype != SMA_DTYPE_FP16 && dtype != SMA_DTYPE_BF16)
    return fail(sma::kErrDtype, "backward: unsupported dtype, need fp16 or bf16");
  if (B < 0 || H < 0 || N < 0 || D <= 0) return fail(sma::kErrArg, "backward: bad dimension");
  if (D != 64 && D != 128) return fail(sma::kErrUnsupportedD, "backward: head dim must be 64 or 128");
  if (N > SMA_MAX_SEQ_LEN) return fail(sma::kErrUnsupportedN, "backward: sequence length above the supported maximum (65536)");
  if (B == 0 || H == 0 || N == 0) return sma::kOk;
  // dQ accumulator + Delta must fit the fixed scratch (checked without overflow).
  const int64_t per_bh = N * (D + 1);
  if (B > kNoAllocScratchFloats || H > kNoAllocScratchFloats || B * H > kNoAllocScratchFloats / per_bh)
    return fail(sma::kErrArg, "backward (no-alloc): B*H*N*(D+1) floats exceed the fixed 32 MiB scratch");
  float* scratch = nullptr;
  int rc = noalloc_scratch(&scratch);
  if (rc != sma::kOk) return rc;
  return sma_attn_bwd(dtype, q, k, v, out, dout, lse, mask_packed, dq, dk, dv, scratch, scratch + B * H * N * D, B,
                      H, N, D, scale, stream);
}

}  // extern "C"

namespace {

// Checks of the 128-row tile kernels on top of cross_params; fills the fields
// that only they use.
int tile_params(const sma_attn_args* a, sma::CrossParams* p) {
  if (a->Nk > SMA_MAX_SEQ_LEN)
    return fail(sma::kErrUnsupportedN, "attention: more keys than the supported maximum (65536)");
  if (a->words) {
    if (a->lengths) return fail(sma::kErrArg, "attention: give a mask or lengths, not both");
    if (!aligned16(a->words)) return fail(sma::kErrArg, "attention: words must be 16-byte aligned");
  } else if (a->mask) {
    return fail(sma::kErrArg, "attention: a mask needs room for its words");
  }
  if (!aligned16(a->out_lo)) return fail(sma::kErrArg, "attention: out_lo must be 16-byte aligned");
  if (a->bias_table) {
    if (!a->bias_distance || !aligned16(a->bias_distance))
      return fail(sma::kErrArg, "attention: a bias needs a 16-byte aligned bias_distance");
    if (a->bias_starts[a->bias_side - 1] > SMA_MAX_BIAS_DISTANCE)
      return fail(sma::kErrUnsupportedN, "attention: bias distance above the supported maximum (65536)");
  }
  p->words = static_cast<uint32_t*>(a->words);
  const int64_t W = (a->Nk + 127) / 128 * 4, n[3] = {a->B, a->H, a->Nq};
  int64_t step = W;
  for (int i = 2; i >= 0; --i) {
    p->word_stride[i] = a->mask_stride[i] != 0 ? step : 0;
    if (a->mask_stride[i] != 0) step *= n[i];
  }
  p->bias_distance = a->bias_distance;
  p->out_lo = a->out_lo;
  return sma::kOk;
}

// No keys at all: out = 0, lse = -FLT_MAX.
int write_nothing(const sma::CrossParams& p) {
  const int64_t rows = p.B * p.H * p.Nq;
  cudaError_t e = cudaMemsetAsync(p.out, 0, static_cast<size_t>(rows * p.D * 2), p.stream);
  if (e == cudaSuccess && p.out_lo != nullptr)
    e = cudaMemsetAsync(p.out_lo, 0, static_cast<size_t>(rows * p.D * 2), p.stream);
  // -FLT_MAX is the bit pattern 0xFF7FFFFF, which no byte fill makes.
  if (e == cudaSuccess && p.lse != nullptr) {
    const int rc = sma::launch_fill(p.lse, rows, -FLT_MAX, p.stream);
    if (rc != sma::kOk) return fail(rc, "attention: fill launch failed");
  }
  return e == cudaSuccess ? sma::kOk : fail_cuda(e, "cudaMemsetAsync");
}

int cross_attn_bwd(const sma_attn_args* args, const void* dout, void* dq, void* dk, void* dv, void* dtable,
                   bool dtable_f32, float* scratch, void* stream) {
  NvtxRange range("sma_cross_attn_bwd");
  sma::CrossParams p{};
  bool empty = false;
  int rc = cross_params(args, stream, &p, &empty);
  if (rc != sma::kOk) return rc;
  if (empty || p.Nk == 0) return fail(sma::kErrArg, "backward: no queries or no keys");
  if (p.P > 0 || p.lengths) return fail(sma::kErrArg, "backward: no prefix and no lengths");
  rc = tile_params(args, &p);
  if (rc != sma::kOk) return rc;
  if (!p.lse || !p.out_lo || !dout || !dq || !dk || !dv || !scratch || (p.bias.table && !dtable))
    return fail(sma::kErrArg, "backward: null pointer");
  if (!aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) || !aligned16(scratch))
    return fail(sma::kErrArg, "backward: dout/dq/dk/dv/scratch must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(dtable) & (dtable_f32 ? 3u : 1u)) return fail(sma::kErrArg, "backward: misaligned dtable");
  rc = device_params(&p);
  if (rc != sma::kOk) return rc;
  const sma::CrossGrads g{dout, dq, dk, dv, dtable, dtable_f32, scratch};
  const char* msg = nullptr;
  rc = sma::launch_attn_cross_bwd(p, g, &msg);
  return rc == sma::kOk ? rc : fail(rc, msg);
}

}  // namespace

extern "C" {

int sma_cross_attn_fwd(const sma_attn_args* args, void* stream) {
  NvtxRange range("sma_cross_attn_fwd");
  sma::CrossParams p{};
  bool empty = false;
  int rc = cross_params(args, stream, &p, &empty);
  if (rc != sma::kOk || empty) return rc;
  if (p.P > 0) return fail(sma::kErrArg, "attention: no prefix here");
  // (A mask over no keys has no bytes and may have no address.)
  if (args->words && !args->mask && p.Nk > 0)
    return fail(sma::kErrArg, "attention: words are packed from a mask, and there is none");
  rc = tile_params(args, &p);
  if (rc == sma::kOk) rc = device_params(&p);
  if (rc != sma::kOk) return rc;
  if (p.Nk == 0) return write_nothing(p);
  const char* msg = nullptr;
  rc = sma::launch_attn_cross(p, &msg);
  return rc == sma::kOk ? rc : fail(rc, msg);
}

int sma_cross_attn_bwd(const sma_attn_args* args, const void* dout, void* dq, void* dk, void* dv, void* dtable,
                       float* scratch, void* stream) {
  return cross_attn_bwd(args, dout, dq, dk, dv, dtable, false, scratch, stream);
}

int sma_cross_attn_bwd_f32_table(const sma_attn_args* args, const void* dout, void* dq, void* dk, void* dv,
                                 float* dtable, float* scratch, void* stream) {
  return cross_attn_bwd(args, dout, dq, dk, dv, dtable, true, scratch, stream);
}

int64_t sma_cross_attn_bwd_scratch(const sma_attn_args* args) {
  sma::CrossParams p{};
  bool empty = false;
  if (cross_params(args, nullptr, &p, &empty) != sma::kOk || empty || p.Nk == 0 || tile_params(args, &p) != sma::kOk)
    return -1;
  return sma::cross_bwd_scratch_floats(p);
}

int sma_prefix_attn_fwd(const sma_attn_args* args, void* stream) {
  NvtxRange range("sma_prefix_attn_fwd");
  sma::CrossParams p{};
  bool empty = false;
  int rc = cross_params(args, stream, &p, &empty);
  if (rc != sma::kOk || empty) return rc;
  rc = tile_params(args, &p);
  if (rc != sma::kOk) return rc;
  if (p.P == 0 || args->mask || args->words || args->bias_table || args->lse || args->out_lo)
    return fail(sma::kErrArg, "attention: a shared prefix takes P > 0 and no mask, bias, lse or out_lo");
  rc = device_params(&p);
  if (rc != sma::kOk) return rc;
  const char* msg = nullptr;
  rc = sma::launch_shared_prefix(p, &msg);
  return rc == sma::kOk ? rc : fail(rc, msg);
}

int sma_rows_attn_fwd(const sma_attn_args* args, void* stream) {
  NvtxRange range("sma_rows_attn_fwd");
  sma::CrossParams p{};
  bool empty = false;
  int rc = cross_params(args, stream, &p, &empty);
  if (rc != sma::kOk || empty) return rc;
  rc = device_params(&p);
  if (rc != sma::kOk) return rc;
  if (p.Nk == 0 && p.P == 0) return write_nothing(p);
  const char* msg = nullptr;
  rc = sma::launch_attn_rows(p, &msg);
  return rc == sma::kOk ? rc : fail(rc, msg);
}

int sma_device_status(void* stream, int clear) {
  uint32_t* err = nullptr;
  int rc = error_word(&err);
  if (rc != sma::kOk) return rc;
  cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "cudaStreamSynchronize");
  uint32_t v = 0;
  e = cudaMemcpyAsync(&v, err, sizeof(v), cudaMemcpyDeviceToHost, static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "read device error word");
  if (clear) {
    // Ordered on the caller's stream, so other streams of the device keep running.
    e = cudaMemsetAsync(err, 0, sizeof(uint32_t), static_cast<cudaStream_t>(stream));
    if (e == cudaSuccess) e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return fail_cuda(e, "clear device error word");
  }
  if (v & sma::kDevErrTimeout) return fail(sma::kErrTimeout, "a device-side wait timed out");
  if (v & sma::kDevErrLayout) return fail(sma::kErrCuda, "attention kernel: shared memory not 1024-byte aligned");
  return sma::kOk;
}

int sma_set_wait_timeout_ns(uint64_t ns) {
  if (ns == 0) return fail(sma::kErrArg, "timeout must be positive");
  g_timeout_ns.store(ns, std::memory_order_relaxed);
  return sma::kOk;
}

int sma_debug_wait_probe(uint64_t timeout_ns, void* stream) {
  uint32_t* err = nullptr;
  int rc = error_word(&err);
  if (rc != sma::kOk) return rc;
  rc = sma::launch_wait_probe(err, timeout_ns, static_cast<cudaStream_t>(stream));
  return rc == sma::kOk ? rc : fail(rc, "wait probe launch failed");
}

const char* sma_last_error(void) { return g_last_error.c_str(); }

int sma_abi_version(void) { return SMA_ABI_VERSION; }

}  // extern "C"
