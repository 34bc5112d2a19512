// Internal launcher interface shared by the kernel translation units and the
// C-ABI layer (sma_capi.cu).  Nothing here is exported from the library.
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace sma {

// Status codes (mirrored by the public SMA_* values in include/sma_capi.h).
enum : int {
  kOk = 0,
  kErrArg = 1,
  kErrDtype = 2,
  kErrUnsupportedD = 3,
  kErrLaunch = 4,
  kErrTimeout = 5,
  kErrUnsupportedN = 6,
  kErrCuda = 7,
};

struct AttnParams {
  int dtype;                  // 0 = fp16, 1 = bf16
  const void* q;              // [B, H, N, D] contiguous
  const void* k;
  const void* v;
  const uint32_t* mask;       // [B, H, N, ceil(N/32)] packed bits, LSB = lowest column
  void* out;                  // [B, H, N, D] contiguous
  float* lse;                 // [B, H, N] or nullptr
  int64_t B, H, N, D;
  float scale;
  const uint32_t* occ;        // [B*H, ceil(N/128), 2] live key-tile bits per query tile, or nullptr
  // Bool-mask input instead of `mask`: [B, H, N, N] bytes (non-zero = attend),
  // N % 32 == 0, 16-byte aligned; the kernel writes the packed words to
  // packed_out ([B, H, N, N/32], 16-byte aligned) and reads them back.
  const uint8_t* bmask;
  uint32_t* packed_out;
  uint32_t* err_word;         // device word the kernel ORs error bits into
  uint64_t timeout_ns;        // bound on every device-side wait
  cudaStream_t stream;
};

// Largest sequence length: the attention kernel keeps one live bit per key
// tile in 32 words per item (1024 tiles of 64 keys); the occupancy map holds
// two 32-bit words (64 key tiles of 128) per query tile.
constexpr int64_t kMaxSeqLen = 65536;
constexpr int64_t kMaxSeqLenOcc = 8192;

int launch_pack_mask(const uint8_t* mask, uint32_t* packed, int64_t rows, int64_t n,
                     cudaStream_t stream, const char** msg);

// Packs like launch_pack_mask and writes the occupancy map `occ`
// ([bh, ceil(n/128), 2] uint32: bit t = key tile t has a set bit in the
// 128-row query tile).  Needs n % 32 == 0, n <= kMaxSeqLenOcc, aligned pointers.
int launch_pack_mask_occ(const uint8_t* mask, uint32_t* packed, uint32_t* occ, int64_t bh, int64_t n,
                         cudaStream_t stream, const char** msg);

int launch_attn_fwd(const AttnParams& p, const char** msg);

struct BwdParams {
  int dtype;                  // 0 = fp16, 1 = bf16
  const void* q;              // [B, H, N, D] contiguous, as for the forward
  const void* k;
  const void* v;
  const void* out;            // the forward's O
  const void* dout;           // upstream gradient of O
  const float* lse;           // [B, H, N] the forward's LSE (natural log, -FLT_MAX for empty rows)
  const uint32_t* mask;       // packed mask
  void* dq;                   // [B, H, N, D] outputs
  void* dk;
  void* dv;
  float* dq_accum;            // [B, H, N, D] FP32 scratch
  float* delta;               // [B, H, N] FP32 scratch
  int64_t B, H, N, D;
  float scale;
  uint32_t* err_word;
  uint64_t timeout_ns;
  cudaStream_t stream;
};

// Backward (attn_bwd.cu): head dims 64 and 128.
int launch_attn_bwd(const BwdParams& p, const char** msg);

// Learned bias by bucketed relative position (rel_bias.cuh has the device side).
constexpr int kMaxBiasSide = 128;
// Relative positions are kept within +-2^30 (sequence lengths and offsets are
// bounded below that), so int arithmetic on them cannot overflow.
constexpr int kMaxBiasOffset = 1 << 30;

struct BiasSpec {
  const void* table;       // [buckets, H] of the inputs' type, or nullptr: no bias
  const int32_t* offsets;  // [B] query offsets, or nullptr: `offset` for all
  int offset;
  int H;
  int side;                // buckets of one side
  int two_sided;
  int starts[kMaxBiasSide];  // smallest distance of each of them, ascending from 0
};

// Attention of queries and keys of different lengths: q [B, H, Nq, D], k and v
// [B, Hkv, Nk, D] (strides in elements, last axis contiguous), Hkv dividing H.
struct CrossParams {
  int dtype;  // 0 = fp16, 1 = bf16
  const void* q;
  const void* k;
  const void* v;
  int64_t q_stride[3], k_stride[3], v_stride[3];  // batch, head, row
  const void* k_prefix;       // [Hkv, P, D] keys in front, shared by the batch
  const void* v_prefix;
  int64_t kp_stride[2], vp_stride[2];  // head, row
  const uint8_t* mask;        // bool bytes, or nullptr
  int64_t mask_stride[3];     // batch, head, query (0: broadcast)
  const int32_t* lengths;     // [B] or nullptr: query i keeps key j < lengths[b] - Nq + 1 + i
  BiasSpec bias;
  void* out;                  // [B, H, Nq, D] contiguous
  float* lse;                 // [B, H, Nq] or nullptr
  // attn_fwd_cross.cu and attn_bwd_cross.cu: the packed mask ([.., W] words with
  // strides {batch, head, query}, 0: broadcast, and behind them the kept keys
  // and the live-tile bits of every tile; nullptr keeps every key), the
  // bias by relative position, [H][bias_stride(length)], and
  // O minus its rounded value, in the inputs' type (nullptr: not wanted).
  uint32_t* words;
  int64_t word_stride[3];
  float* bias_distance;
  void* out_lo;
  // attn_rows.cu: where given, every row is left as a piece for a later merge
  // (max, sum, sum of rounded P, - / FP32 O, not normalised; indexed by
  // (b * H + h) * Nq + i) instead of written to `out`.
  float* part_ml;
  float* part_o;
  int64_t B, H, Hkv, Nq, Nk, D, P;
  float scale;
  uint32_t* err_word;
  uint64_t timeout_ns;
  cudaStream_t stream;
};

// The relative positions d between which buckets change: d <= lo is one
// bucket, d >= hi is one bucket.
inline void bias_range(const BiasSpec& s, int* lo, int* hi) {
  *lo = -s.starts[s.side - 1];
  *hi = s.two_sided ? s.starts[s.side - 1] : 0;
}
// Length of the bias by relative position: lo .. hi and kBiasPad more on
// either side, so that a tile which overlaps (lo, hi) never leaves it.
constexpr int kBiasPad = 256;
// It is kept four times, shifted by 0 .. 3 places, the copies interleaved by
// 16 bytes: floats 16 j + 4 k .. + 3 are values 4 j - k .. + 3.  Any run of
// values can so be read 16 bytes at a time, whatever its start.
inline int64_t bias_stride(int len) { return 16 * ((static_cast<int64_t>(len) + 3) / 4 + 1); }  // floats per head

// Many query rows (attn_fwd_cross.cu), Nk <= kMaxSeqLen.
int launch_attn_cross(const CrossParams& p, const char** msg);
// A shared prefix attended once for the batch, P > 0 (attn_fwd_cross.cu).
int launch_shared_prefix(const CrossParams& p, const char** msg);

// Gradients (attn_bwd_cross.cu), all contiguous; p.out and p.lse are the
// forward's, p.bias_distance as it left it.
struct CrossGrads {
  const void* dout;  // [B, H, Nq, D]
  void* dq;          // [B, H, Nq, D]
  void* dk;          // [B, Hkv, Nk, D]
  void* dv;
  void* dtable;      // [buckets, H], with a bias
  bool dtable_f32;   // dtable is FP32, else of the inputs' type
  float* scratch;    // cross_bwd_scratch_floats elements
};
int64_t cross_bwd_scratch_floats(const CrossParams& p);
int launch_attn_cross_bwd(const CrossParams& p, const CrossGrads& g, const char** msg);

constexpr int kRowsTile = 16;  // rows of a tile of attn_rows.cu

// x[0 .. n) = v (attn_fwd_cross.cu).
int launch_fill(float* x, int64_t n, float v, cudaStream_t stream);

// Few query rows per key head (attn_rows.cu): head dims 64 and 128.
int launch_attn_rows(const CrossParams& p, const char** msg);

// TMA map of the [BH, N, D] view of a contiguous [B, H, N, D] fp16/bf16
// tensor: boxes of 64 head dims (one 128-byte swizzle span) by `rows` rows,
// 128-byte swizzle (tma_map.cu).  Returns the driver's status
// (CUDA_ERROR_NOT_FOUND when the entry point is missing).
CUresult make_tensor_map_3d(CUtensorMap* m, const void* ptr, int dtype, int64_t D, int64_t BH, int64_t N, int rows);
// TMA map of a [B, H, N, D] fp16/bf16 view with element strides {batch, head,
// row}: boxes of 64 head dims by `rows` rows of `heads` heads of `batches`
// batches, 128-byte swizzle; coordinates (d, row, head, batch).
CUresult make_tensor_map_4d(CUtensorMap* m, const void* ptr, int dtype, int64_t D, int64_t N, int64_t H, int64_t B,
                            const int64_t* stride, int rows, int heads = 1, int batches = 1);
// The same view of a contiguous FP32 [BH, N, D] tensor: boxes of 32 elements
// (128 bytes) by `rows` rows, 128-byte swizzle (tma_map.cu).
CUresult make_tensor_map_3d_f32(CUtensorMap* m, const void* ptr, int64_t D, int64_t BH, int64_t N, int rows);
// Message for a failed tensor-map encode: `what` and the driver status.
const char* tensor_map_error(const char* what, CUresult rc);

// Stream-ordered scratch from a per-device memory pool that keeps its memory
// between calls (no release back to the driver), so a steady stream of
// launches allocates only once.  Freed with cudaFreeAsync on the same stream.
cudaError_t scratch_alloc_async(void** p, size_t bytes, cudaStream_t stream);
// A value distinct for every call in the process: 56 bits, never 0.
unsigned long long next_launch_epoch();

// Devices the per-device caches of the launchers cover.
constexpr int kMaxDevices = 64;

// Properties of the current device, queried once per device (thread-safe).
struct DeviceProps {
  int device = -1;
  int sms = 0;
  int l2_bytes = 0;
};
bool device_props(DeviceProps* out, const char** msg);

// Raises `kern`'s dynamic shared-memory limit to `bytes` on the current
// device the first time it is launched there.  `done` is the kernel's own
// per-device flag array; concurrent first calls both set the same attribute.
template <typename Kern>
cudaError_t ensure_smem_limit(Kern kern, size_t bytes, int dev, std::atomic<bool> (&done)[kMaxDevices]) {
  if (done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess) done[dev].store(true, std::memory_order_relaxed);
  return e;
}

// Launches `kern` with programmatic stream serialisation: its CTAs may start
// (and run their set-up) while the previous kernel in the stream finishes;
// the kernel itself calls griddepcontrol.wait before reading global memory.
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kern)(Params...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream,
                       Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...);
}

// Persistent two-chain kernel (attn_fwd_chain.cu): head dims 64 and 128, N up
// to kMaxSeqLen.  launch_attn_fwd dispatches to it when chain_supported().
bool chain_supported(const AttnParams& p);
int launch_attn_fwd_chain(const AttnParams& p, const char** msg);

// Launches one CTA that waits on an mbarrier nothing ever arrives on, using
// the same bounded-wait helper as the attention kernel; it must give up after
// `timeout_ns` and set bit 1 of *err_word.
int launch_wait_probe(uint32_t* err_word, uint64_t timeout_ns, cudaStream_t stream);

// Device error bits.
constexpr uint32_t kDevErrTimeout = 1u;
constexpr uint32_t kDevErrLayout = 2u;  // shared-memory window not 1024-byte aligned

}  // namespace sma
