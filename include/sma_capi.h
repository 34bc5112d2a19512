/*
 * sma_capi.h - C ABI of the B200 sparse-mask attention library (libsma.so).
 *
 * Plain pointers and sizes only: every tensor argument is a device pointer to
 * a contiguous row-major buffer, every stream argument is a cudaStream_t passed
 * as void* (NULL = legacy default stream).  Work is enqueued asynchronously on
 * that stream; nothing synchronises except sma_device_status().
 *
 * Every function returns an SMA_* status.  On a non-zero status,
 * sma_last_error() returns a message describing the failure (thread-local,
 * valid until the next call on the same thread).
 *
 * Each entry point names the reference interface it replaces
 * (yulangz/sparse-mask-attention-auto-research, paths relative to its root).
 */
#ifndef SMA_CAPI_H_
#define SMA_CAPI_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. */
#define SMA_OK 0
#define SMA_ERR_ARG 1             /* bad pointer / size / layout argument          */
#define SMA_ERR_DTYPE 2           /* dtype is neither fp16 nor bf16                 */
#define SMA_ERR_UNSUPPORTED_D 3   /* head dim other than 64 or 128                  */
#define SMA_ERR_LAUNCH 4          /* kernel launch failed                           */
#define SMA_ERR_TIMEOUT 5         /* a device-side wait gave up (see sma_device_status) */
#define SMA_ERR_UNSUPPORTED_N 6   /* sequence length above the path's maximum       */
#define SMA_ERR_CUDA 7            /* CUDA runtime / driver error                    */

/* Element types of q, k, v and out. */
#define SMA_DTYPE_FP16 0
#define SMA_DTYPE_BF16 1

/* Longest supported sequence (both head dims); the occupancy map
 * (sma_pack_mask_occupancy) covers N <= 8192. */
#define SMA_MAX_SEQ_LEN 65536
#define SMA_MAX_SEQ_LEN_OCCUPANCY 8192

#if defined(__GNUC__)
#define SMA_API __attribute__((visibility("default")))
#else
#define SMA_API
#endif
#define SMA_ABI_VERSION 1

/*
 * Pack a bool mask [B, H, N, N] (one byte per element, non-zero = attend)
 * into 32-bit words [B, H, N, ceil(N/32)]: bit b of word w of a row is the
 * mask at column 32*w + b; bits at columns >= N are zero.  The output has the
 * bit pattern of the reference's int32 packed tensor.
 *
 * Replaces: pack_mask()            csrc/binding.cpp:49-66
 *           pack_mask_bits()       csrc/sparse_attention.cu:44-54
 *           (CPU fallback          python/sparse_attention.py:189-206)
 * Unlike the reference binding, the caller allocates `packed`.
 */
SMA_API int sma_pack_mask(const void* mask, void* packed, int64_t B, int64_t H, int64_t N, void* stream);

/*
 * Masked-softmax attention forward:
 *   out[b,h,i,:] = sum_j softmax_j(scale * q_i . k_j  over j with bit(i,j) set) * v[b,h,j,:]
 * q, k, v, out: [B, H, N, D] of `dtype`; mask_packed: [B, H, N, ceil(N/32)]
 * words as produced by sma_pack_mask; lse: [B, H, N] float32 log-sum-exp of
 * the scaled scores, or NULL to skip it (the reference's is_training=false).
 * Rows with no set bit get out = 0 and lse = -FLT_MAX (the reference CUDA
 * convention, csrc/sparse_attention.cu:133,141).
 * Supported: D in {64, 128}, 1 <= N <= SMA_MAX_SEQ_LEN, 16-byte aligned
 * q/k/v/out, scale finite and > 0 (the kernels fold the scale into the
 * exponent after the masked row max; the reference always passes 1/sqrt(D)).
 * When the (batch*head, 128-row query tile) items are fewer than twice the
 * SM count and at least 64 key tiles long, each item is split along keys
 * over several SMs and merged; that path takes scratch (about
 * items * pieces * 128 * (D + 4) floats) from a per-device stream-ordered
 * pool the library keeps, released on `stream` after the launch.
 *
 * Replaces: forward()                          csrc/binding.cpp:9-47
 *           sparse_attention_fwd_fp16/_bf16()  csrc/sparse_attention.cu:149-185
 *           SparseAttentionParams              csrc/sparse_attention.h:12-38
 */
SMA_API int sma_attn_fwd(int dtype, const void* q, const void* k, const void* v, const void* mask_packed,
                 void* out, float* lse, int64_t B, int64_t H, int64_t N, int64_t D, float scale,
                 void* stream);

/*
 * The pack + forward pair in one launch: the attention kernel reads the bool
 * mask [B, H, N, N] (one byte per element, non-zero = attend) itself, packs
 * each query tile's rows as it scans them for live key tiles, and writes the
 * packed words to mask_packed ([B, H, N, N/32], bit for bit what
 * sma_pack_mask writes, kept for the backward).  out and lse are those of
 * sma_attn_fwd on the packed mask, bit for bit.
 * Needs N % 32 == 0 and 16-byte aligned mask and mask_packed (SMA_ERR_ARG
 * otherwise: callers then use sma_pack_mask + sma_attn_fwd); the rest as for
 * sma_attn_fwd.  On B200 the pair of launches is faster (the packer streams
 * the mask at HBM speed, while here each query tile's rows are read and
 * packed by the softmax warps between tiles, on the kernel's critical path),
 * so sparse_attention() uses the pair; this entry saves a launch only.
 *
 * Replaces: the pack_mask() + SparseAttentionFunction forward pair that
 *           sparse_attention() runs   python/sparse_attention.py:122-156
 *           (pack_mask_bits()         csrc/sparse_attention.cu:44-54,
 *            forward()                csrc/binding.cpp:9-47)
 */
SMA_API int sma_attn_fwd_mask(int dtype, const void* q, const void* k, const void* v, const void* mask,
                              void* mask_packed, void* out, float* lse, int64_t B, int64_t H, int64_t N, int64_t D,
                              float scale, void* stream);

/*
 * Fused bool -> bit packing plus occupancy map.  Writes `packed` exactly as
 * sma_pack_mask does and `occupancy`: uint32 [B*H, ceil(N/128), 2], where bit t
 * of the pair for (batch*head, query tile qt) is set iff key tile t (keys
 * 128t .. 128t+127) has a set mask bit in query rows 128qt .. 128qt+127.
 * Needs N % 32 == 0, N <= SMA_MAX_SEQ_LEN_OCCUPANCY, a 16-byte aligned mask and 4-byte
 * aligned outputs (SMA_ERR_ARG / SMA_ERR_UNSUPPORTED_N otherwise; callers
 * then use sma_pack_mask).  The packer reads every mask byte anyway, so the
 * map costs no extra HBM pass.
 * No reference counterpart: the reference's attention re-tests every mask bit.
 */
SMA_API int sma_pack_mask_occupancy(const void* mask, void* packed, void* occupancy, int64_t B, int64_t H,
                                    int64_t N, void* stream);

/*
 * sma_attn_fwd with the occupancy map written by sma_pack_mask_occupancy for
 * the same mask: the head-dim-64 kernel takes its live key tiles from the
 * map instead of scanning the packed rows; results are identical to
 * sma_attn_fwd.  (The map describes 128-key tiles; head dim 128 works on
 * 64-key tiles, scans the packed rows and ignores it.)
 * No reference counterpart.
 */
SMA_API int sma_attn_fwd_occupancy(int dtype, const void* q, const void* k, const void* v, const void* mask_packed,
                                   const void* occupancy, void* out, float* lse, int64_t B, int64_t H, int64_t N,
                                   int64_t D, float scale, void* stream);

/*
 * Masked-softmax attention backward (head dims 64 and 128): given the forward's
 * inputs, its out and lse (as written by sma_attn_fwd with a non-NULL lse)
 * and the upstream gradient dout, writes dq, dk, dv ([B, H, N, D] of `dtype`):
 *   P = exp(scale * q k^T - lse) where the mask bit is set, else 0
 *   dv = P^T dout;  dS = P * (dout v^T - rowsum(dout * out));
 *   dq = scale * dS k;  dk = scale * dS^T q
 * dq_accum (FP32 [B, H, N, D]) and delta (FP32 [B, H, N]) are caller-provided
 * scratch.  Rows with no set bit get dq = 0; keys no row attends get dk = dv = 0.
 * Needs D in {64, 128}, 16-byte aligned q/k/v/out/dout/dq/dk/dv/dq_accum.
 *
 * Replaces: sparse_attn_cuda.backward(dout, q, k, v, out, lse, mask_packed,
 *           dq, dk, dv, scale), called by python/sparse_attention.py:93-96 but
 *           never bound by csrc/binding.cpp; the result follows the
 *           reference's CPU formulas (python/sparse_attention.py:97-111).
 */
SMA_API int sma_attn_bwd(int dtype, const void* q, const void* k, const void* v, const void* out, const void* dout,
                         const float* lse, const void* mask_packed, void* dq, void* dk, void* dv, float* dq_accum,
                         float* delta, int64_t B, int64_t H, int64_t N, int64_t D, float scale, void* stream);

/*
 * sma_attn_bwd with the FP32 scratch taken from a fixed 32 MiB device array
 * inside the library (one per device, found once per device with
 * cudaGetSymbolAddress): no memory is allocated and no allocating routine is
 * called.  Inputs whose B*H*N*(D+1) floats exceed the array return
 * SMA_ERR_ARG (dtype, head dim and sequence length are checked first, with
 * the codes of sma_attn_bwd).  Calls sharing a device share the array: order
 * them on one stream.  The 32 MiB are part of the library's module image, so
 * they are reserved on every device where the module is loaded, whether or
 * not this entry point is ever called.  No reference counterpart.
 */
SMA_API int sma_attn_bwd_noalloc(int dtype, const void* q, const void* k, const void* v, const void* out,
                                 const void* dout, const float* lse, const void* mask_packed, void* dq, void* dk,
                                 void* dv, int64_t B, int64_t H, int64_t N, int64_t D, float scale, void* stream);

/*
 * Arguments of the entry points for queries and keys of different lengths
 * (sma_rows_attn_fwd and its companions below).  Zero-initialise it; fields
 * that an operator does not use stay 0.
 *
 *   q [B, H, Nq, D], k and v [B, Hkv, Nk, D], H % Hkv == 0: query head h
 *   reads key head h / (H / Hkv).  Strides are in elements, for the batch,
 *   head and row axes; the last axis is contiguous.  Base addresses and the
 *   strides of axes longer than 1 are multiples of 16 bytes (strides > 0).
 *
 *   mask: bool bytes (non-zero = attend) at mask + b*mask_stride[0] +
 *   h*mask_stride[1] + i*mask_stride[2] + j, a stride of 0 for an axis the
 *   mask does not depend on; NULL keeps every key.
 *
 *   lengths (device int32 [B], or NULL): instead of a mask, the queries are
 *   the last Nq of the first lengths[b] keys and see keys up to themselves:
 *   query i keeps key j iff j < lengths[b] - Nq + 1 + i.  Lengths are
 *   clamped to [0, Nk].
 *
 *   k_prefix, v_prefix [Hkv, P, D] (strides for head and row): P more keys in
 *   front of the others, the same for the whole batch, kept by every query.
 *
 *   bias: adds bias_table[bucket, h] (of `dtype`, [bias_buckets, H],
 *   contiguous) to the scaled score of query i and key j, bucket being that
 *   of the relative position d = j - i - offset.  One-sided: the last of the
 *   bias_side entries of bias_starts (host array, ascending from 0) that is
 *   <= max(-d, 0).  Two-sided: that of |d|, plus bias_side where d > 0.
 *   offset is bias_offset, or bias_offsets[b] (device int32 [B]) if given.
 */
#define SMA_MAX_BIAS_SIDE 128
#define SMA_MAX_BIAS_DISTANCE 65536 /* largest last start, where bias_distance is used */
/* Floats per head of bias_distance, `last` being the last bucket's start. */
#define SMA_BIAS_DISTANCE_LEN(last, two_sided) (16 * ((((two_sided) ? 2 : 1) * (int64_t)(last) + 516) / 4 + 1))
typedef struct sma_attn_args {
  int32_t dtype;
  float scale;
  int64_t B, H, Hkv, Nq, Nk, D, P;
  const void *q, *k, *v;
  int64_t q_stride[3], k_stride[3], v_stride[3];
  const void *k_prefix, *v_prefix;
  int64_t kp_stride[2], vp_stride[2];
  const void* mask;
  int64_t mask_stride[3];
  const int32_t* lengths;
  const void* bias_table;
  const int32_t* bias_starts;
  const int32_t* bias_offsets;
  int64_t bias_offset;
  int32_t bias_side;
  int32_t bias_two_sided;
  void* out;   /* [B, H, Nq, D] contiguous */
  float* lse;  /* [B, H, Nq] natural-log sum of exponentials, or NULL */
  /* Of the 128-row tile entries: room for the packed mask, int32 words
   * [B, H, Nq, 4 * ceil(Nk / 128)] with length 1 for an axis whose mask_stride
   * is 0 (bit b of word w: column 32 w + b, 0 past Nk), and behind it, for
   * every 128-row tile, the keys that some row keeps and the live key tiles:
   * [B, H, ceil(Nq / 128), 4 * ceil(Nk / 128) + ceil(Nk / 2048)] more. */
  void* words;
  float* bias_distance; /* room for H * SMA_BIAS_DISTANCE_LEN floats */
  void* out_lo;         /* O minus its rounded value, like out, or NULL */
} sma_attn_args;

/*
 * Attention forward for few query rows per key head (a generated token, a
 * few drafted ones): each (batch, key head)'s rows are taken 16 at a time
 * against keys streamed once, split along keys over the SMs when there are
 * few rows.  Any Nq works; the keys are read again for every 16 rows.
 * Takes a bool mask (not packed), lengths, a shared prefix and a bias.  Rows
 * that keep no key get out = 0 and lse = -FLT_MAX.  Keys that none of the 16
 * rows keeps may hold any values.  D in {64, 128}, scale finite and > 0,
 * P and Nk up to 2^30, |bias_offset| < 2^30.  Scratch for the split comes
 * from the library's stream-ordered pool.
 * No reference counterpart.
 */
SMA_API int sma_rows_attn_fwd(const sma_attn_args* args, void* stream);

/*
 * Attention forward for many query rows, on 128-row tiles.  A mask is packed
 * into `words` first, and a bias laid out in bias_distance (the backward reads
 * both, with the lse and out_lo, which training needs).  Queries of the heads
 * that share a key head fill a tile together when Nq <= 64.
 * Nk <= SMA_MAX_SEQ_LEN, no prefix; otherwise as sma_rows_attn_fwd: a key
 * that none of a tile's rows keeps may hold any values, one that some keep
 * must be finite.  Rows that keep no key get out = 0 and lse = -FLT_MAX.
 */
SMA_API int sma_cross_attn_fwd(const sma_attn_args* args, void* stream);

/*
 * Attention behind a prefix shared by the batch.  Where it pays, the prefix is
 * read once for all sequences (its tiles hold the rows of several).  P > 0,
 * Nk <= SMA_MAX_SEQ_LEN, `lengths` or nothing for the sequences' own keys, no
 * mask, no bias, no lse.  Own keys behind a sequence's length may hold anything.
 */
SMA_API int sma_prefix_attn_fwd(const sma_attn_args* args, void* stream);

/*
 * Backward of sma_cross_attn_fwd: `args` are the forward's, with the out, lse,
 * out_lo, words and bias_distance it wrote (`mask` itself is not read).  From dout [B, H, Nq, D]
 * writes dq [B, H, Nq, D], dk and dv [B, Hkv, Nk, D] (summed over the query
 * heads of a key head) and, with a bias, dtable [bias_buckets, H], all
 * contiguous and of `dtype`; formulas as for sma_attn_bwd, and
 *   dtable[bucket, h] = sum of dS over the pairs in the bucket.
 * scratch: sma_cross_attn_bwd_scratch(args) floats.
 * At most 2048 steps of 64 query rows per key head (SMA_ERR_UNSUPPORTED_N).
 * Q, dO and every key must be finite, except that the keys a mask leaves to no
 * query (B and Nk its only axes: padding) may hold anything.  dq is accumulated by atomic
 * adds in FP32, so its last bits can differ from run to run; dk, dv and
 * dtable do not.
 */
SMA_API int sma_cross_attn_bwd(const sma_attn_args* args, const void* dout, void* dq, void* dk, void* dv, void* dtable,
                               float* scratch, void* stream);

/*
 * The same with dtable in FP32, for tables that are kept in FP32 (bias_table
 * is of `dtype` here too): the sum over all queries is not rounded.
 */
SMA_API int sma_cross_attn_bwd_f32_table(const sma_attn_args* args, const void* dout, void* dq, void* dk, void* dv,
                                         float* dtable, float* scratch, void* stream);

/* Floats of scratch either of them needs; -1 for arguments that it refuses. */
SMA_API int64_t sma_cross_attn_bwd_scratch(const sma_attn_args* args);

/*
 * Synchronise `stream`, then report whether any kernel of this library on the
 * current device gave up a bounded device-side wait since the last clear
 * (SMA_ERR_TIMEOUT), or whether the stream holds a CUDA error (SMA_ERR_CUDA).
 * clear != 0 resets the device error word.
 * No reference counterpart (the reference never checks its launches).
 */
SMA_API int sma_device_status(void* stream, int clear);

/*
 * Upper bound, in nanoseconds, of every device-side wait in later launches
 * (default 2e9).  What a CTA that gave up has itself started (copies, matrix
 * products) is waited for at least 2^31 ns, so that it lands before the CTA
 * leaves.  No reference counterpart.
 */
SMA_API int sma_set_wait_timeout_ns(uint64_t ns);

/*
 * Launch a one-CTA kernel that waits, through the library's bounded-wait
 * helper, on a barrier nothing ever signals; it gives up after timeout_ns and
 * raises the device error word.  Used to test failure reporting without
 * faulting or hanging a GPU.  No reference counterpart.
 */
SMA_API int sma_debug_wait_probe(uint64_t timeout_ns, void* stream);

/* Thread-local message for the last non-zero status. */
SMA_API const char* sma_last_error(void);

/* SMA_ABI_VERSION of the loaded library. */
SMA_API int sma_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* SMA_CAPI_H_ */
