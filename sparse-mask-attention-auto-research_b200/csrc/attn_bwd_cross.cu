// Attention backward of queries and keys of different lengths (sm_100a), head
// dims 64 and 128, with key heads shared by query heads and a relative
// position bias and its gradient.
//
//   P  = exp(scale * q k^T + bias - lse) where the mask keeps the pair, else 0
//   dV = P^T dO,  dS = P * (dO V^T - Delta),  Delta_i = sum_d dO_id O_id
//   dQ = scale * dS K,  dK = scale * dS^T Q,  dtable[bucket, h] = sum of dS over the bucket's pairs
//
// Kernels, in stream order: cross_prepare_kernel (Delta, zeros in the FP32 dQ
// accumulator, and the packed mask by key, where query rows have masks of
// their own), cross_bwd_kernel, cross_dq_kernel (accumulator -> dq) and, with a
// bias, bias_reduce_kernel.
//
// cross_bwd_kernel is persistent, one CTA per SM, over items (batch, key head,
// 128-key tile), handed out as CTAs come free (masks leave items of very
// different length).  The last ones, which would not fill a round of the SMs,
// are cut along their query steps into parts that do; the parts leave dK and dV
// in FP32, which cross_dq_kernel adds in order, so that dK and dV do not depend
// on which CTA did what.  K and V of the item stay in shared memory, dK and dV
// accumulate in TMEM over all query heads that share the key head, and the CTA
// walks the item's live steps of 64 query rows (those whose mask block keeps
// a pair).  Two steps are in flight, each with its own S^T / dP^T columns and
// its own four element-wise warps, so that while one step's exponentials run,
// the tensor core works on the other's products:
//
//   MMA warp, step s: S^T = K Q_s^T, dP^T = V dO_s^T             (M = 128 keys, N = 64 queries)
//             step s-1: dV += P^T dO (P from TMEM), dK += dS^T Q (dS from shared memory), dQ product
//   warps 4g..4g+3, steps s = g mod 2: P, dS in registers (thread = key); P
//             rounded over the S^T columns, dS to shared memory
//
// What bounds it: per 64 queries, 16 (D = 64: four S^T, four dP^T, four dV,
// four dK) tensor instructions at 31 to 47 cycles, the dQ product, and 8192
// exponentials with some ten instructions each; with the two in turn (one
// step in flight) each waited for the other.  Measured: B8 H12 Nq512 Nk1024 D64
// with a random mask 68 us (470 TFLOP/s), B4 H32 Hkv8 Nq1024 Nk2048 D128 with a
// mask of random 64 x 64 blocks, 30 % kept, 221 us (470 TFLOP/s of the kept
// blocks, which lie in half of the steps of 128 keys).
//
// The dQ product: D = 64 takes the dS of two steps as one 128-row operand,
// dQ = dS K, in TMEM columns of its own (two buffers).  D = 128 has no columns
// left and computes dQ^T = K^T dS^T of one step over the dP^T columns, which
// the element-wise warps have read by then.  Four epilogue warps add it into
// the FP32 accumulator by TMA bulk reduce-adds.
//
// Warps: 0-7 element-wise (each thread reads the 64 mask bits of its key for a
// step as one 8-byte word, a step ahead), 8 loader (Q, dO, K, V by TMA, LSE and
// Delta by cp.async, kRing steps ahead with nothing held in registers: a
// loader that carried them through registers ran at one step per load
// latency), 9 MMA issuer and TMEM owner, 10-13 epilogue, 14 scanner
// (each item's live steps, kSlots items ahead).  Every wait is bounded and
// reports through the device error word.
//
// P and dS are rounded to the inputs' type, the operand type of the products;
// Delta uses O with the residual of its rounding that the forward kept, since
// an error there shifts a whole row of dS.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "attn_math.cuh"
#include "rel_bias.cuh"
#include "sma_internal.h"
#include "sma_ptx.cuh"

namespace sma {
namespace {

constexpr int kKeys = 128;  // keys of an item
constexpr int kQ = 64;      // query rows of a step
constexpr int kTmemCols = 512;
constexpr int kEwWarps = 8, kLoaderWarp = 8, kMmaWarp = 9, kEpiWarp = 10, kScanWarp = 14;
constexpr int kThreads = 16 * 32;  // warp 15 only fills its warpgroup
// Register split after start-up: the launch gives every thread 128; the two
// warpgroups of loader, MMA, epilogue and scanner drop to 112 and the
// element-wise ones rise to 144: 256 x (112 + 144) = 512 x 128.
constexpr int kRegsOther = 112;
constexpr int kRegsEw = 144;
static_assert(256 * (kRegsOther + kRegsEw) <= kThreads * 128, "register split");
// Items whose live lists the scanner claims and publishes ahead (no more than
// the one being worked on and the next, since a claimed item waits for its
// CTA), and words of a list: one bit per step, up to 2048 steps of the heads
// that share a key head.
constexpr int kSlots = 2;
constexpr int kListWords = 64;
constexpr int kMaxSteps = 32 * kListWords;
constexpr int kMaxParts = 8;  // of an item

// TMEM columns: S^T of stage g, dP^T of stage g, dV, dK, and for D = 64 two dQ buffers.
__host__ __device__ constexpr uint32_t col_s(int g) { return 64u * g; }
__host__ __device__ constexpr uint32_t col_dp(int g) { return 128u + 64u * g; }
constexpr uint32_t kColDV = 256;

template <int D>
struct Cfg {
  static constexpr int kDChunks = D / 64;
  static constexpr uint32_t kColDK = kColDV + D;
  static constexpr bool kPairDQ = D == 64;
  __host__ __device__ static constexpr uint32_t col_dq(int b) { return 384u + 64u * b; }  // D = 64
  static constexpr int kKVBytes = kKeys * D * 2;
  static constexpr int kKVBufs = D == 64 ? 2 : 1;
  static constexpr int kQBytes = kQ * D * 2;
  static constexpr int kRing = D == 64 ? 4 : 3;      // staged steps
  static constexpr int kDSBytes = kKeys * kQ * 2;
  static constexpr int kDSSlots = kPairDQ ? 4 : 2;
  static constexpr int kOffK = 0;
  static constexpr int kOffV = kKVBufs * kKVBytes;
  static constexpr int kOffQ = 2 * kKVBufs * kKVBytes;
  static constexpr int kOffDO = kOffQ + kRing * kQBytes;
  static constexpr int kOffDS = kOffDO + kRing * kQBytes;
  static constexpr int kOffDQ = kOffDS + kDSSlots * kDSBytes;  // 4 KiB box per epilogue warp
  static constexpr int kOffLse = kOffDQ + 4 * 4096;
  static constexpr int kOffDelta = kOffLse + kRing * kQ * 4;
  static constexpr int kOffBias = kOffDelta + kRing * kQ * 4;  // [8 element-wise warps][96]
  static constexpr int kOffCtl = kOffBias + kEwWarps * 96 * 4;
};

struct Ctl {
  uint64_t kv_full[2], kv_free[2];
  uint64_t acc_free;               // dV and dK of a live item read out of TMEM
  uint64_t ld_full[4], tile_free[4];
  uint64_t st_full[2];             // S^T and dP^T of a stage complete
  uint64_t p_full[2];              // its P in TMEM and dS in shared memory
  uint64_t pt_free[2];             // D = 64: its dV and dK products complete
  uint64_t dq_full[2], dq_free[2];  // D = 64: per dQ buffer (pair of steps); D = 128: per stage
  uint64_t item_full[kSlots], item_free[kSlots];
  uint64_t drain;
  uint32_t live_bits[kSlots][kListWords];
  uint32_t n_live[kSlots];
  int unit[kSlots];                // which item or part, -1: no more
  uint32_t tmem_base;
  uint32_t abort_flag;
};

template <int D>
constexpr size_t smem_bytes() {
  return Cfg<D>::kOffCtl + sizeof(Ctl);
}
static_assert(smem_bytes<64>() <= 227 * 1024 && smem_bytes<128>() <= 227 * 1024, "shared memory budget");
static_assert(smem_bytes<64>() > 114 * 1024 && smem_bytes<128>() > 114 * 1024, "one CTA per SM: it takes all of TMEM");
static_assert(Cfg<64>::kOffDQ % 1024 == 0 && Cfg<128>::kOffDQ % 1024 == 0, "swizzle atoms");

// Geometry.  Step ht * QT1 + qt of an item holds tn queries from 64 qt of the
// hb heads from ht * hb of the key head's group (hb > 1 only when the queries
// of several heads fit one step); rows past tn * hb are kept zero in shared
// memory, since the products run over them.
struct BwdGeo {
  int B, H, Hkv, Nq, Nk;
  int tn, hb, gh, rows;    // rows = tn * hb; gh = G / hb
  int QT1;                 // 64-row steps of Nq
  uint32_t qt_magic;       // v / QT1 = umulhi(v, qt_magic) for v < 2^16, or 0: QT1 = 1
  const uint32_t* words;   // packed mask rows (16-byte aligned), or nullptr: every key is kept
  int64_t word_stride[3];  // batch, head, query, in words (0: broadcast)
  int one_row;             // all query rows of an item have the same mask row
  // Otherwise the mask by key, [..][key of KT * 128] 64-bit words of a step's
  // rows, strides in such words for batch, head block (ht) and 64-query step.
  const uint2* words_t;
  int64_t t_stride[3];
  // And which 32-key words of a step keep a pair: 4 bytes (0 / 1) per key tile,
  // strides t_stride / 128 per tile.
  const uint32_t* live_t;
  // Bias in units of log2 by relative position, bias_len values a head
  // (bias_stride in sma_internal.h).
  const float* bias;
  const int32_t* bias_offsets;
  int bias_offset, bias_lo, bias_hi, bias_len;
  int64_t bias_stride;
  // Its gradient by relative position: dS summed along the diagonals of every
  // 32 x 32 block that overlaps (bias_lo, bias_hi), [B*H][KB][slots][64]
  // (entry d - 32 (kb - qb) + off, mod 64), and the sums of the blocks beyond
  // on either side, [B*H][KB][kMaxParts * 2 (stage)][2 (low, high)].
  float* near_part;
  float* far_part;
  int KB, QB, slots, slot_by_query;
  // Units of work: `whole` items, then `cut` items in `parts` parts each, whose
  // dV and dK [cut * parts][128 keys][2 D] FP32 go to part_acc.  CTA c starts
  // with unit c; the others go to whoever asks next (`next`, cleared before).
  int grid, whole, cut, parts;
  int tile_major;          // items by key tile, then (batch, key head), instead of the other way round
  float* part_acc;
  int* next;
};

// (batch, key head) and key tile of item w.
__device__ __forceinline__ void item_place(const BwdGeo& x, int KT, int w, int& bh, int& kt) {
  const int fast = x.tile_major ? x.B * x.Hkv : KT;
  const int slow = w / fast;
  kt = x.tile_major ? slow : w - slow * fast;
  bh = x.tile_major ? w - slow * fast : slow;
}

// Block difference j = kb - qb of the 32 x 32 blocks that overlap (lo, hi):
// their relative positions are 32 j - off + [-31, 31].  The largest such j.
__host__ __device__ inline int bias_block_max(int hi, int off) {
  const int x = hi + off + 30;  // 32 j <= x
  return x >= 0 ? x / 32 : -((-x + 31) / 32);
}

__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xFFFFFFFFu : (n <= 0 ? 0u : (1u << n) - 1u); }

// Next set bit of a live list from cursor (w, x): the step index, or -1.
__device__ __forceinline__ int next_live(const uint32_t* bits, int& w, uint32_t& x) {
  while (x == 0u) {
    if (++w >= kListWords) return -1;
    x = bits[w];
  }
  const int b = __ffs(x) - 1;
  x &= x - 1u;
  return w * 32 + b;
}

// 32 x 32 bit transpose over a warp: bit k of lane r goes to bit r of lane k.
// Five exchanges of halves of ever smaller blocks.
__device__ __forceinline__ uint32_t transpose_bits(uint32_t x, int lane) {
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    const uint32_t low = w == 16 ? 0x0000FFFFu : w == 8 ? 0x00FF00FFu : w == 4 ? 0x0F0F0F0Fu : w == 2 ? 0x33333333u : 0x55555555u;
    const uint32_t y = __shfl_xor_sync(0xffffffffu, x, w);
    x = (lane & w) ? (((y >> w) & low) | (x & ~low)) : ((x & low) | ((y & low) << w));
  }
  return x;
}

// words (rows of queries) -> words_t (BwdGeo): one warp per (batch, head block,
// step, 32 keys), its 64 rows' words transposed, and whether they keep any
// pair (live_t, so that the scanner reads 4 bytes per step).
struct Transpose {
  uint2* out;
  uint8_t* live;
  int Hm, key_words;
  int64_t total;  // warps; 0: nothing to do
};
__device__ __forceinline__ void transpose_words(const BwdGeo& x, const Transpose& tr, int64_t w, int lane) {
  if (w >= tr.total) return;
  // [Bm][Hm head blocks][QT1][key_words]
  const int kw = static_cast<int>(w % tr.key_words);
  int64_t rest = w / tr.key_words;
  const int qt = static_cast<int>(rest % x.QT1);
  rest /= x.QT1;
  const int hm = static_cast<int>(rest % tr.Hm);
  const int64_t b = rest / tr.Hm;
  uint32_t v[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u, hr = i / x.tn, t = qt * kQ + i - hr * x.tn;
    const int64_t h = static_cast<int64_t>(hm) * x.hb + hr;
    v[u] = i < x.rows && t < x.Nq
               ? __ldg(x.words + b * x.word_stride[0] + h * x.word_stride[1] + t * x.word_stride[2] + kw)
               : 0u;
    v[u] = transpose_bits(v[u], lane);
  }
  tr.out[w * 32 + lane] = make_uint2(v[0], v[1]);
  const bool any = __any_sync(0xffffffffu, (v[0] | v[1]) != 0u);
  if (lane == 0) tr.live[w] = any ? 1 : 0;
}

constexpr int kZeroRounds = 4;

// What the backward needs before it starts, in one launch.  Blocks below
// `delta_blocks`, D/8 threads per row: -Delta, Delta = sum_d dO[row, d] *
// (O[row, d] + its rounding residual) in FP32, and -lse * log2(e) (negated, so
// that the element-wise pass adds them in packed pairs), and zeros in the FP32
// dQ accumulator.  The next `zero_blocks`: zeros in the bias gradient's partial
// sums (blocks that no live step visits count as 0).  The others: the mask by
// key, a warp each.  Bound by HBM:
// three 16-bit reads and a 32-bit write per element, and the packed mask once
// in and out (B4 H32 Nq1024 D128, 168 MB: 26 us, 6.5 TB/s).
template <int D, bool BF16>
__global__ void __launch_bounds__(256)
    cross_prepare_kernel(const uint4* __restrict__ dout, const uint4* __restrict__ out, const uint4* __restrict__ out_lo,
                         const float* __restrict__ lse, float* __restrict__ neg_delta, float* __restrict__ neg_lse2,
                         float4* __restrict__ dq_acc, int64_t rows, unsigned delta_blocks, float4* __restrict__ zero,
                         int64_t zeros, unsigned zero_blocks, const __grid_constant__ Transpose tr, const __grid_constant__ BwdGeo x) {
  constexpr int kPerRow = D / 8;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  if (blockIdx.x >= delta_blocks + zero_blocks) {
    transpose_words(x, tr, static_cast<int64_t>(blockIdx.x - delta_blocks - zero_blocks) * 8 + (threadIdx.x >> 5),
                    threadIdx.x & 31);
    return;
  }
  if (blockIdx.x >= delta_blocks) {
#pragma unroll
    for (int u = 0; u < kZeroRounds; ++u) {
      const int64_t i = (static_cast<int64_t>(blockIdx.x - delta_blocks) * kZeroRounds + u) * 256 + threadIdx.x;
      if (i < zeros) zero[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (gid == 0) *x.next = 0;
  const int64_t row = gid / kPerRow;
  float acc = 0.f;
  if (row < rows) {
    const uint4 a = __ldg(dout + gid), b = __ldg(out + gid), c = __ldg(out_lo + gid);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    dq_acc[2 * gid] = zero;
    dq_acc[2 * gid + 1] = zero;
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w}, cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x2 = unpack2<BF16>(aw[e]), y = unpack2<BF16>(bw[e]), z = unpack2<BF16>(cw[e]);
      acc = fmaf(x2.x, y.x + z.x, acc);
      acc = fmaf(x2.y, y.y + z.y, acc);
    }
  }
#pragma unroll
  for (int o = 1; o < kPerRow; o <<= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (row < rows && (threadIdx.x % kPerRow) == 0) {
    neg_delta[row] = -acc;
    // -FLT_MAX, a row that keeps nothing: -inf, so that P = 2^-inf = 0 also where
    // no mask says so (scores of -inf, from a table's entries).
    const float row_lse = lse[row];
    neg_lse2[row] = row_lse == -FLT_MAX ? -INFINITY : -(row_lse * kLog2e);
  }
}

// Blocks below `dq_blocks`: dq[i] = acc[i] in the input dtype, 8 elements per
// thread.  The others: dV and dK of the items cut in parts, the parts added in
// order, 8 elements per thread.  Bound by HBM (B8 H16 N777 D128, 60 MB: 13 us).
template <int D, bool BF16>
__global__ void __launch_bounds__(256)
    cross_dq_kernel(const float4* __restrict__ acc, uint4* __restrict__ dq, int64_t n8, unsigned dq_blocks,
                    uint16_t* __restrict__ dk, uint16_t* __restrict__ dv, int KT, const __grid_constant__ BwdGeo x) {
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  if (blockIdx.x < dq_blocks) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n8) return;
    const float4 a = __ldcs(acc + 2 * i), b = __ldcs(acc + 2 * i + 1);
    dq[i] = make_uint4(pack2<BF16>(a.x, a.y), pack2<BF16>(a.z, a.w), pack2<BF16>(b.x, b.y), pack2<BF16>(b.z, b.w));
    return;
  }
  constexpr int kPerRow = 2 * D / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x - dq_blocks) * 256 + threadIdx.x;
  const int64_t row = i / kPerRow;
  const int c = static_cast<int>(i - row * kPerRow);
  const int item = static_cast<int>(row / kKeys), t = static_cast<int>(row - static_cast<int64_t>(item) * kKeys);
  if (item >= x.cut) return;
  int bh, kt;
  item_place(x, KT, x.whole + item, bh, kt);
  const int key = kt * kKeys + t;
  if (key >= x.Nk) return;
  float sum[8] = {};
  for (int part = 0; part < x.parts; ++part) {
    const float4* src = reinterpret_cast<const float4*>(
        x.part_acc + ((static_cast<int64_t>(item) * x.parts + part) * kKeys + t) * (2 * D) + c * 8);
    const float4 a = __ldcs(src), b = __ldcs(src + 1);
    sum[0] += a.x, sum[1] += a.y, sum[2] += a.z, sum[3] += a.w;
    sum[4] += b.x, sum[5] += b.y, sum[6] += b.z, sum[7] += b.w;
  }
  uint16_t* dst = (c < D / 8 ? dv : dk) + (static_cast<int64_t>(bh) * x.Nk + key) * D + (c < D / 8 ? c : c - D / 8) * 8;
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<BF16>(sum[0], sum[1]), pack2<BF16>(sum[2], sum[3]),
                                              pack2<BF16>(sum[4], sum[5]), pack2<BF16>(sum[6], sum[7]));
}

// Sums of a 32 x 32 block along its diagonals.  ds[e] is lane t's element of
// column e; diagonal k = t - e.  On return lane k holds diagonal k >= 0 in
// `pos` and lane 32 + k diagonal k < 0 in `neg`.  Neighbouring column blocks
// of width w are added with the right one shifted by w lanes; what the shift
// carries round the end belongs to the negative diagonals.
__device__ __forceinline__ void diagonal_sums(const float (&ds)[32], int lane, float& pos, float& neg) {
  float m[16], n[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float r = __shfl_sync(0xffffffffu, ds[2 * i + 1], (lane + 1) & 31);
    m[i] = ds[2 * i] + (lane < 31 ? r : 0.f);
    n[i] = lane < 31 ? 0.f : r;
  }
#pragma unroll
  for (int w = 2; w < 32; w *= 2) {
#pragma unroll
    for (int i = 0; i < 16 / w; ++i) {
      const float r = __shfl_sync(0xffffffffu, m[2 * i + 1], (lane + w) & 31);
      const float r2 = __shfl_sync(0xffffffffu, n[2 * i + 1], (lane + w) & 31);
      m[i] = m[2 * i] + (lane < 32 - w ? r : 0.f);
      n[i] = n[2 * i] + (lane < 32 - w ? r2 : r);
    }
  }
  pos = m[0];
  neg = n[0];
}

template <int D, bool BF16, bool kBias>
__global__ void __launch_bounds__(kThreads, 1)
    cross_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                     const __grid_constant__ CUtensorMap tm_dq, const float* __restrict__ neg_lse2,
                     const float* __restrict__ neg_delta, uint16_t* __restrict__ dk, uint16_t* __restrict__ dv, int KT,
                     float scale, const __grid_constant__ BwdGeo x, uint32_t* err_word,
                     uint64_t timeout_ns) {
  using C = Cfg<D>;
  constexpr int kRing = C::kRing;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  if ((base & 1023u) != 0u) {
    if (threadIdx.x == 0) atomicOr(err_word, kDevErrLayout);
    return;
  }
  Ctl& ctl = *reinterpret_cast<Ctl*>(smem + C::kOffCtl);
  // Per ring slot b, row i: -LSE * log2(e) and -Delta at s_lse / s_delta
  // [b * kQ + i], 0 for rows past the problem's.  Their Q and dO are 0 too, so
  // that without a bias their P is at most 2^0 and reaches nothing; with one it
  // would be e^bias, which no LSE holds down, and the element-wise warps clear
  // their mask bits.
  float* s_lse = reinterpret_cast<float*>(smem + C::kOffLse);
  float* s_delta = reinterpret_cast<float*>(smem + C::kOffDelta);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Counters over all units of the CTA, the same in every role: j units (list
  // slot j % kSlots), li units with a live step (K/V buffer li % kKVBufs), lt
  // live steps (ring slot lt % kRing), the uses of each stage (step t of a unit
  // uses stage t & 1) and lp pairs of steps of one unit (D = 64: dQ buffer
  // lp & 1).
  const int units = x.whole + x.cut * x.parts;
  const int VT = x.gh * x.QT1;
  volatile uint32_t* abort_flag = &ctl.abort_flag;

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&ctl.kv_full[b]), 1);
      mbar_init(smem_u32(&ctl.kv_free[b]), 1);
      mbar_init(smem_u32(&ctl.st_full[b]), 1);
      mbar_init(smem_u32(&ctl.p_full[b]), 4);
      mbar_init(smem_u32(&ctl.pt_free[b]), 1);
      mbar_init(smem_u32(&ctl.dq_full[b]), 1);
      mbar_init(smem_u32(&ctl.dq_free[b]), 4);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(smem_u32(&ctl.ld_full[b]), 1 + 32);  // TMA bytes, and every lane's cp.async
      mbar_init(smem_u32(&ctl.tile_free[b]), 5);  // a stage's element-wise warps and the MMA issuer
    }
    for (int sl = 0; sl < kSlots; ++sl) {
      mbar_init(smem_u32(&ctl.item_full[sl]), 1);
      mbar_init(smem_u32(&ctl.item_free[sl]), kEwWarps + 6);  // element-wise, loader, MMA, 4 epilogue warps
    }
    mbar_init(smem_u32(&ctl.acc_free), 4);
    mbar_init(smem_u32(&ctl.drain), 1);
    ctl.abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (x.rows < kQ) {  // rows the copies never write
    for (int i = threadIdx.x; i < (C::kOffDS - C::kOffQ) / 16; i += kThreads)
      *reinterpret_cast<uint4*>(smem + C::kOffQ + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&ctl.tmem_base), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem_base;
  pdl_launch_dependents();
  pdl_wait_prior_grid();

  auto fail = [&]() {
    ctl.abort_flag = 1;
    atomicOr(err_word, kDevErrTimeout);
  };
  // Batch, key head and key tile of a unit, and the first head of the group.
  struct Item {
    int b, hkv, kt, h0;
    int part;  // -1: a whole item
  };
  auto item_of = [&](int unit) -> Item {
    Item it;
    int w = unit;
    it.part = -1;
    if (unit >= x.whole) {
      const int i = (unit - x.whole) / x.parts;
      it.part = unit - x.whole - i * x.parts;
      w = x.whole + i;
    }
    int bh;
    item_place(x, KT, w, bh, it.kt);
    it.b = bh / x.Hkv;
    it.hkv = bh - it.b * x.Hkv;
    it.h0 = it.hkv * (x.gh * x.hb);
    return it;
  };
  auto step_block = [&](int v) { return x.qt_magic != 0u ? static_cast<int>(__umulhi(v, x.qt_magic)) : v; };
  auto step_head = [&](int v) { return step_block(v) * x.hb; };  // relative to h0
  auto step_q0 = [&](int v) { return (v - step_block(v) * x.QT1) * kQ; };
  // The 128 words (by key) of step v of an item, where the mask is by key.
  auto step_words = [&](const Item& it, int v) {
    const int ht = step_block(v);
    return x.words_t + it.b * x.t_stride[0] + (it.hkv * x.gh + ht) * x.t_stride[1] + (v - ht * x.QT1) * x.t_stride[2] +
           it.kt * kKeys;
  };
  // Whole-warp wait.
  auto wait_all = [&](uint64_t& bar, uint32_t parity) -> bool {
    const bool all = __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&bar), parity, abort_flag, timeout_ns));
    tc_fence_after();
    return all;
  };
  auto arrive_warp = [&](uint64_t& bar) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bar));
  };

  if (warp == kLoaderWarp) {
    // ================================================================ loader
    regs_dec<kRegsOther>();
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      tma_prefetch_desc(&tm_do);
      tma_prefetch_desc(&tm_dq);
    }
    bool ok = true;
    int lt = 0, li = 0;
    // Query and head of this lane's rows (lane, lane + 32) within a step.
    int rt[2], rh[2];
    bool rin[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = lane + 32 * u;
      rin[u] = i < x.rows;
      rh[u] = rin[u] ? i / x.tn : 0;
      rt[u] = rin[u] ? i - rh[u] * x.tn : 0;
    }
    auto issue_kv = [&](const Item& it) -> bool {
      const int b = li % C::kKVBufs;
      if (li >= C::kKVBufs &&
          !__all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&ctl.kv_free[b]), ((li - C::kKVBufs) / C::kKVBufs) & 1,
                                                     abort_flag, timeout_ns)))
        return false;
      if (lane == 0) {
        const uint32_t bar = smem_u32(&ctl.kv_full[b]);
        mbar_arrive_expect_tx(bar, 2 * C::kKVBytes);
#pragma unroll
        for (int dc = 0; dc < C::kDChunks; ++dc) {
          tma_load_4d(base + C::kOffK + b * C::kKVBytes + dc * kKeys * 128, &tm_k, bar, dc * 64, it.kt * kKeys, it.hkv,
                      it.b);
          tma_load_4d(base + C::kOffV + b * C::kKVBytes + dc * kKeys * 128, &tm_v, bar, dc * 64, it.kt * kKeys, it.hkv,
                      it.b);
        }
      }
      ++li;
      return true;
    };
    // Step v of an item into ring slot lt % kRing, once the element-wise warps
    // and the products are done with the step before in it.
    auto stage = [&](const Item& it, int v) -> bool {
      const int b = lt % kRing;
      if (lt >= kRing &&
          !__all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&ctl.tile_free[b]), ((lt - kRing) / kRing) & 1,
                                                     abort_flag, timeout_ns)))
        return false;
      const uint32_t bar = smem_u32(&ctl.ld_full[b]);
      const int q0 = step_q0(v), h0 = it.h0 + step_head(v);
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, 2 * x.rows * D * 2);
#pragma unroll
        for (int dc = 0; dc < C::kDChunks; ++dc) {
          tma_load_4d(base + C::kOffQ + b * C::kQBytes + dc * kQ * 128, &tm_q, bar, dc * 64, q0, h0, it.b);
          tma_load_4d(base + C::kOffDO + b * C::kQBytes + dc * kQ * 128, &tm_do, bar, dc * 64, q0, h0, it.b);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = q0 + rt[u];
        const bool in = rin[u] && t < x.Nq;
        const int64_t row = in ? (static_cast<int64_t>(it.b) * x.H + h0 + rh[u]) * x.Nq + t : 0;
        cp_async4_zfill(smem_u32(s_lse + b * kQ + lane + 32 * u), neg_lse2 + row, in);
        cp_async4_zfill(smem_u32(s_delta + b * kQ + lane + 32 * u), neg_delta + row, in);
      }
      cp_async_arrive(bar);
      ++lt;
      return true;
    };
    for (int j = 0; ok; ++j) {
      const int sl = j % kSlots;
      if (!wait_all(ctl.item_full[sl], (j / kSlots) & 1)) {
        ok = false;
        break;
      }
      if (ctl.unit[sl] < 0) break;
      const int n = static_cast<int>(ctl.n_live[sl]);
      if (n > 0) {
        const Item it = item_of(ctl.unit[sl]);
        ok = issue_kv(it);
        int cw = 0;
        uint32_t cx = ctl.live_bits[sl][0];
        for (int t = 0; ok && t < n; ++t) ok = stage(it, next_live(ctl.live_bits[sl], cw, cx));
        if (!ok) break;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.item_free[sl]));
    }
    cp_async_wait_all();
    if (!ok && lane == 0) {
      fail();
      // Let the copies this warp started land before the CTA exits.
      for (int jj = li - C::kKVBufs; jj < li; ++jj)
        if (jj >= 0) mbar_drain(smem_u32(&ctl.kv_full[jj % C::kKVBufs]), (jj / C::kKVBufs) & 1, timeout_ns);
      for (int g = lt - kRing; g < lt; ++g)
        if (g >= 0) mbar_drain(smem_u32(&ctl.ld_full[g % kRing]), (g / kRing) & 1, timeout_ns);
    }
  } else if (warp == kMmaWarp) {
    // ================================================================ MMA issuer
    // The whole warp walks along, converged; one elected lane issues.
    regs_dec<kRegsOther>();
    bool ok = true;
    {
      constexpr int kBf = BF16 ? 1 : 0;
      constexpr uint32_t idesc_s = make_idesc_f16(kKeys, kQ, kBf, 0);                // S^T, dP^T
      constexpr uint32_t idesc_kv = make_idesc_f16(kKeys, D, kBf, 1);                // dV, dK (B M/N-major)
      constexpr uint32_t idesc_q = make_idesc_f16(128, 64, kBf, 1, 1);               // dQ, dQ^T (A and B M/N-major)
      uint32_t lt = 0, lp = 0, use0 = 0, use1 = 0;  // uses of the stages (no array: g is not known at compile time)
      int li = 0;
      // The step whose products are still to be issued.
      struct {
        bool on = false;
        int g, slot, li, kv;
        bool first, pair_end;
        int kv_free;
        uint32_t use;
      } pend;
      // The descriptor `bytes` further on (addresses fit its field, in units of 16 bytes).
      auto step = [](uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); };
      auto flush = [&]() -> bool {
        if (!pend.on) return true;
        pend.on = false;
        const int g = pend.g;
        // P and dS of the step; before the first products of a live item, the
        // epilogue warps must have read the previous one's dV / dK.
        if (!wait_all(ctl.p_full[g], pend.use & 1)) return false;
        if (pend.first && pend.li > 0 && !wait_all(ctl.acc_free, (pend.li - 1) & 1)) return false;
        const uint32_t sQ = base + C::kOffQ + pend.slot * C::kQBytes, sDO = base + C::kOffDO + pend.slot * C::kQBytes;
        const uint32_t sK = base + C::kOffK + pend.kv * C::kKVBytes;
        const int ds_slot = C::kPairDQ ? static_cast<int>(lp & 1) * 2 + g : g;
        const uint32_t sDS = base + C::kOffDS + ds_slot * C::kDSBytes;
        const uint64_t dDO = smem_desc_sw128(sDO, kQ * 128, 1024), dQ = smem_desc_sw128(sQ, kQ * 128, 1024);
        const uint64_t dDS = smem_desc_sw128(sDS, 16, 1024), dK = smem_desc_sw128(sK, kKeys * 128, 1024);
        // 16 query rows per instruction: 8 packed TMEM columns of P^T, 32
        // bytes of dS's rows, 2048 bytes (16 rows of 128) of dO and Q, whose
        // 64-dim chunks are kQ * 128 bytes apart.
#pragma unroll
        for (int kk = 0; kk < kQ / 16; ++kk)
          mma_ts_warp(tmem + kColDV, tmem + col_s(g) + kk * 8, step(dDO, kk * 2048), idesc_kv,
                 (!pend.first || kk > 0) ? 1u : 0u);
#pragma unroll
        for (int kk = 0; kk < kQ / 16; ++kk)
          mma_ss_warp(tmem + C::kColDK, step(dDS, kk * 32), step(dQ, kk * 2048), idesc_kv,
                      (!pend.first || kk > 0) ? 1u : 0u);
        mma_commit_warp(smem_u32(&ctl.tile_free[pend.slot]));
        if constexpr (C::kPairDQ) {
          mma_commit_warp(smem_u32(&ctl.pt_free[g]));
          if (pend.pair_end) {
            // dQ = dS K of the pair (one step's rows are not used when the
            // item's last pair has only one): 16 keys per instruction, 2048
            // bytes into dS's two 64-query tiles and K.
            const int b = lp & 1;
            if (lp >= 2 && !wait_all(ctl.dq_free[b], ((lp >> 1) - 1) & 1)) return false;
            const uint64_t dPair = smem_desc_sw128(base + C::kOffDS + b * 2 * C::kDSBytes, C::kDSBytes, 1024);
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk)
              mma_ss_warp(tmem + C::col_dq(b), step(dPair, kk * 2048), step(dK, kk * 2048), idesc_q, kk > 0 ? 1u : 0u);
            mma_commit_warp(smem_u32(&ctl.dq_full[b]));
            ++lp;
          }
        } else {
          // dQ^T = K^T dS^T of the step, over its dP^T columns.
          const uint64_t dDSn = smem_desc_sw128(sDS, kKeys * 128, 1024);
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            mma_ss_warp(tmem + col_dp(g), step(dK, kk * 2048), step(dDSn, kk * 2048), idesc_q, kk > 0 ? 1u : 0u);
          mma_commit_warp(smem_u32(&ctl.dq_full[g]));
        }
        if (pend.kv_free >= 0) mma_commit_warp(smem_u32(&ctl.kv_free[pend.kv_free]));
        return true;
      };
      for (int j = 0; ok; ++j) {
        const int sl = j % kSlots;
        if (!wait_all(ctl.item_full[sl], (j / kSlots) & 1)) {
          ok = false;
          break;
        }
        if (ctl.unit[sl] < 0) break;
        const int n = static_cast<int>(ctl.n_live[sl]);
        if (n > 0) {
          const int kv = li % C::kKVBufs;
          const uint32_t sK = base + C::kOffK + kv * C::kKVBytes, sV = base + C::kOffV + kv * C::kKVBytes;
          if (!wait_all(ctl.kv_full[kv], (li / C::kKVBufs) & 1)) {
            ok = false;
            break;
          }
          for (int t = 0; t < n; ++t, ++lt) {
            const int g = t & 1, slot = lt % kRing;
            // The pending step uses this stage (an item that ended on it).
            if (pend.on && pend.g == g && !flush()) {
              ok = false;
              break;
            }
            const uint32_t use = g ? use1 : use0;
            uint64_t& cols_free = C::kPairDQ ? ctl.pt_free[g] : ctl.dq_free[g];
            // The step staged; the stage's columns free: its last P read by
            // the dV product (D = 64), and its dQ^T read out (D = 128).
            if (!wait_all(ctl.ld_full[slot], (lt / kRing) & 1) || (use > 0 && !wait_all(cols_free, (use - 1) & 1))) {
              ok = false;
              break;
            }
            const uint32_t sQ = base + C::kOffQ + slot * C::kQBytes, sDO = base + C::kOffDO + slot * C::kQBytes;
            const uint64_t dK = smem_desc_sw128(sK, 16, 1024), dV = smem_desc_sw128(sV, 16, 1024);
            const uint64_t dQ = smem_desc_sw128(sQ, 16, 1024), dDO = smem_desc_sw128(sDO, 16, 1024);
            // 16 head dims per instruction: swizzle chunk kk / 4 of the rows, 32 bytes into it.
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t ko = (kk >> 2) * (kKeys * 128) + (kk & 3) * 32, qo = (kk >> 2) * (kQ * 128) + (kk & 3) * 32;
              mma_ss_warp(tmem + col_s(g), step(dK, ko), step(dQ, qo), idesc_s, kk > 0 ? 1u : 0u);
            }
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t ko = (kk >> 2) * (kKeys * 128) + (kk & 3) * 32, qo = (kk >> 2) * (kQ * 128) + (kk & 3) * 32;
              mma_ss_warp(tmem + col_dp(g), step(dV, ko), step(dDO, qo), idesc_s, kk > 0 ? 1u : 0u);
            }
            // st_full covers every earlier product, so the ones that last read
            // this step's dS slot have done so before it is rewritten.
            mma_commit_warp(smem_u32(&ctl.st_full[g]));
            if (!flush()) {
              ok = false;
              break;
            }
            pend.on = true;
            pend.g = g;
            pend.slot = slot;
            pend.li = li;
            pend.kv = kv;
            pend.first = t == 0;
            pend.pair_end = g == 1 || t + 1 == n;
            pend.kv_free = t + 1 == n ? kv : -1;
            pend.use = use;
            if (g) ++use1;
            else ++use0;
          }
          if (!ok) break;
          ++li;
          // With two K/V buffers the last step's products may wait for the
          // next item's first S^T, if that item has a live step; its list
          // needs nothing of this item.
          bool keep = false;
          if (C::kKVBufs == 2) {
            const int sl1 = (j + 1) % kSlots;
            if (!wait_all(ctl.item_full[sl1], ((j + 1) / kSlots) & 1)) {
              ok = false;
              break;
            }
            keep = ctl.unit[sl1] >= 0 && ctl.n_live[sl1] > 0u;
          }
          if (!keep && !flush()) {
            ok = false;
            break;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.item_free[sl]));
      }
      if (ok && !flush()) ok = false;
      if (!ok && lane == 0) fail();
      // Every MMA this thread issued must complete before TMEM is released.
      mma_commit_warp(smem_u32(&ctl.drain));
      mbar_drain(smem_u32(&ctl.drain), 0, timeout_ns);
    }
  } else if (warp == kScanWarp) {
    // ================================================================ scanner
    regs_dec<kRegsOther>();
    // Item j's live list: bit v set when some query row of step v keeps a key
    // of the item's tile; a lane looks at one step of 32.
    bool ok = true;
    for (int j = 0;; ++j) {
      const int sl = j % kSlots;
      if (j >= kSlots && !wait_all(ctl.item_free[sl], ((j / kSlots) - 1) & 1)) {
        ok = false;
        break;
      }
      int unit = static_cast<int>(blockIdx.x);
      if (j > 0) {
        if (lane == 0) unit = x.grid + atomicAdd(x.next, 1);
        unit = __shfl_sync(0xffffffffu, unit, 0);
      }
      if (unit >= units) {
        if (lane == 0) {
          ctl.unit[sl] = -1;
          mbar_arrive(smem_u32(&ctl.item_full[sl]));
        }
        break;
      }
      const Item it = item_of(unit);
      uint32_t mine[2] = {0u, 0u};  // words lane and lane + 32 of the list
      if (x.words_t == nullptr) {
        // No mask, or one mask row for the whole item: all steps or none.
        bool any = true;
        if (x.words != nullptr) {
          const uint4 m = __ldg(reinterpret_cast<const uint4*>(x.words + it.b * x.word_stride[0] +
                                                               it.h0 * x.word_stride[1] + it.kt * 4));
          any = (m.x | m.y | m.z | m.w) != 0u;
        }
        if (any) {
          mine[0] = low_bits(VT - 32 * lane);
          mine[1] = low_bits(VT - 32 * (lane + 32));
        }
      } else {
        for (int v0 = 0; v0 < VT; v0 += 128) {
          uint32_t f[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int v = v0 + 32 * u + lane;
            const int64_t tile = (step_words(it, min(v, VT - 1)) - x.words_t) / kKeys;
            f[u] = v < VT ? __ldg(x.live_t + tile) : 0u;
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t bits = __ballot_sync(0xffffffffu, f[u] != 0u);
            const int w = (v0 >> 5) + u;
            if (lane == (w & 31)) {
              if (w < 32) mine[0] = bits;
              else mine[1] = bits;
            }
          }
        }
      }
      if (it.part >= 0) {
        // The part's share of the n live steps, by rank: [part n / parts, (part + 1) n / parts).
        int before[2], all = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int incl = __popc(mine[h]);
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
          }
          before[h] = all + incl - __popc(mine[h]);
          all += __shfl_sync(0xffffffffu, incl, 31);
        }
        const int lo = all * it.part / x.parts, hi = all * (it.part + 1) / x.parts;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int from = max(lo - before[h], 0), to = min(hi - before[h], __popc(mine[h]));
          uint32_t left = mine[h], keep = 0u;
          for (int i = 0; i < to; ++i) {
            const uint32_t low = left & (0u - left);
            if (i >= from) keep |= low;
            left ^= low;
          }
          mine[h] = keep;
        }
      }
      ctl.live_bits[sl][lane] = mine[0];
      ctl.live_bits[sl][lane + 32] = mine[1];
      const int n = __reduce_add_sync(0xffffffffu, __popc(mine[0]) + __popc(mine[1]));
      if (lane == 0) {
        ctl.n_live[sl] = static_cast<uint32_t>(n);
        ctl.unit[sl] = unit;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.item_full[sl]));
    }
    if (!ok && lane == 0) fail();
  } else if (warp < kEwWarps) {
    // ================================================================ element-wise
    regs_inc<kRegsEw>();
    // Thread t = key t of the tile (TMEM lane); stage g = warp / 4.
    const int g = warp >> 2;
    const int t = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float c2 = scale * kLog2e;
    const uint64_t c2x2 = f2(c2, c2);
    float* s_win = reinterpret_cast<float*>(smem + C::kOffBias) + warp * 96;  // kBias: bias by relative position
    bool ok = true;
    uint32_t lt0 = 0, lp0 = 0, use = 0;
    int li = 0;
    // Mask bits of this key for the 64 queries of the next step of this stage.
    uint2 next_words = make_uint2(0u, 0u);
    bool have_words = false;
    auto item_bit = [&](const Item& it) -> uint2 {  // one mask row for the item
      const int key = it.kt * kKeys + t;
      uint32_t bit = key < x.Nk ? 1u : 0u;
      if (x.words != nullptr)
        bit &= __ldg(x.words + it.b * x.word_stride[0] + it.h0 * x.word_stride[1] + (key >> 5)) >> (key & 31);
      return bit ? make_uint2(0xFFFFFFFFu, 0xFFFFFFFFu) : make_uint2(0u, 0u);
    };
    auto fetch_words = [&](const Item& it, int v) {
      return x.words_t != nullptr ? __ldg(step_words(it, v) + t) : item_bit(it);
    };
    for (int j = 0; ok; ++j) {
      const int sl = j % kSlots;
      ok = wait_all(ctl.item_full[sl], (j / kSlots) & 1);
      if (!ok || ctl.unit[sl] < 0) break;
      const int n = static_cast<int>(ctl.n_live[sl]);
      const Item it = item_of(ctl.unit[sl]);
      int cw = 0;
      uint32_t cx = ctl.live_bits[sl][0];
      if (g == 1) next_live(ctl.live_bits[sl], cw, cx);
      int v_next = n > g ? next_live(ctl.live_bits[sl], cw, cx) : -1;
      if (n > g && !have_words) next_words = fetch_words(it, v_next);
      have_words = false;
      // kBias: this warp's 32-key block, and the bias gradient of blocks
      // beyond the last bucket's start, per head.
      int key0 = 0, off = 0, far_head = -1;
      float far_lo = 0.f, far_hi = 0.f, add_lo = 0.f, add_hi = 0.f;
      const float* head_row = nullptr;
      if constexpr (kBias) {
        key0 = it.kt * kKeys + (warp & 3) * 32;
        off = x.bias_offsets == nullptr
                  ? x.bias_offset
                  : max(-kMaxBiasOffset, min(kMaxBiasOffset, __ldg(x.bias_offsets + it.b)));
      }
      // Where the item has one mask row, the K rows of keys it leaves out (they
      // may hold anything) are cleared before the first dQ product, which runs
      // over all keys.
      if (g == 0 && n > 0 && x.words != nullptr && x.one_row) {
        ok = wait_all(ctl.kv_full[li % C::kKVBufs], (li / C::kKVBufs) & 1);
        if (!ok) break;
        if (next_words.x == 0u) {
          uint8_t* krow = smem + C::kOffK + (li % C::kKVBufs) * C::kKVBytes + t * 128;
#pragma unroll
          for (int e = 0; e < D / 8; ++e)
            *reinterpret_cast<uint4*>(krow + (e >> 3) * (kKeys * 128) + (e & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();  // ahead of this thread's arrival on p_full
      }
      if (n > 0) ++li;
      auto flush_far = [&]() {
        if constexpr (kBias) {
          if (far_head < 0) return;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            far_lo += __shfl_xor_sync(0xffffffffu, far_lo, o);
            far_hi += __shfl_xor_sync(0xffffffffu, far_hi, o);
          }
          if (lane == 0) {
            float* dst = x.far_part + (((static_cast<int64_t>(it.b) * x.H + far_head) * x.KB + key0 / 32) * (2 * kMaxParts) +
                                       2 * max(it.part, 0) + g) * 2;
            dst[0] = far_lo;
            dst[1] = far_hi;
          }
          far_lo = far_hi = 0.f;
        }
      };
      for (int tt = g; tt < n; tt += 2, ++use) {
        const uint32_t lt = lt0 + tt;
        const int b = lt % kRing;
        const int v = v_next;
        uint2 words = next_words;
        int head = 0, q0 = 0;
        if constexpr (kBias) {
          head = it.h0 + step_head(v);  // hb = 1
          q0 = step_q0(v);
          if (x.words_t == nullptr) {  // the bits by key end at the last query already
            words.x &= low_bits(x.Nq - q0);
            words.y &= low_bits(x.Nq - q0 - 32);
          }
          if (head != far_head) {
            flush_far();
            far_head = head;
            head_row = x.bias + static_cast<int64_t>(head) * x.bias_stride;
            add_lo = __ldg(head_row);
            add_hi = __ldg(head_row + bias_at(x.bias_len - 1));
          }
        }
        // kBias: relative positions of the step's block c are d0 - 32 c + lane
        // - e.  When it comes near the diagonal band, the 95 values of the
        // step go to this warp's window: value of d at d - d0 + 64.
        const int d0 = key0 - q0 - off;
        bool step_near = false;
        float win[3];
        if constexpr (kBias) {
          step_near = d0 + 31 > x.bias_lo && d0 - 63 < x.bias_hi;
          if (step_near) {
            const float* src = head_row + bias_at(d0 - x.bias_lo + kBiasPad + lane);
#pragma unroll
            for (int u = 0; u < 3; ++u) win[u] = __ldg(src + (u - 2) * (32 * 4));
          }
        }
        // The next step's words, a step ahead; at the last one those of the
        // next item's first (its list needs nothing of this item).
        if (tt + 2 < n) {
          next_live(ctl.live_bits[sl], cw, cx);  // the other stage's
          v_next = next_live(ctl.live_bits[sl], cw, cx);
          if (x.words_t != nullptr) next_words = fetch_words(it, v_next);
        } else {
          const int sl1 = (j + 1) % kSlots;
          ok = wait_all(ctl.item_full[sl1], ((j + 1) / kSlots) & 1);
          if (!ok) break;
          if (ctl.unit[sl1] >= 0 && static_cast<int>(ctl.n_live[sl1]) > g) {
            int w1 = 0;
            uint32_t x1 = ctl.live_bits[sl1][0];
            if (g == 1) next_live(ctl.live_bits[sl1], w1, x1);
            const int v1 = next_live(ctl.live_bits[sl1], w1, x1);
            next_words = fetch_words(item_of(ctl.unit[sl1]), v1);
            have_words = true;
          }
        }
        const float* t_lse = s_lse + b * kQ;
        const float* t_delta = s_delta + b * kQ;
        uint8_t* ds_row = smem + C::kOffDS +
                          (C::kPairDQ ? static_cast<int>((lp0 + (tt >> 1)) & 1) * 2 + g : g) * C::kDSBytes + t * 128;
        ok = wait_all(ctl.ld_full[b], (lt / kRing) & 1) && wait_all(ctl.st_full[g], use & 1);
        if (!ok) break;
        if constexpr (kBias) {
          if (step_near) {
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 3; ++u) s_win[32 * u + lane] = win[u];
            __syncwarp();
          }
        }
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          const uint32_t word = c == 0 ? words.x : words.y;
          float s[32], dp[32];
          tmem_ld32f(t_lane + col_s(g) + c * 32, s);
          tmem_ld32f(t_lane + col_dp(g) + c * 32, dp);
          // kBias: the bias of a block beyond (bias_lo, bias_hi) is one value.
          const int dc = d0 - 32 * c;
          const bool near = kBias && dc + 31 > x.bias_lo && dc - 31 < x.bias_hi;
          tmem_wait_ld();
          uint32_t pw[16], dw[16];
          // P and dS of the block; kB: 0 no bias, 1 one value, 2 the window's.
          // (Told apart outside the loop, which schedules as one block then.)
          auto block = [&](auto kind) {
            constexpr int kB = decltype(kind)::value;
            const uint64_t badd = f2(dc < x.bias_hi ? add_lo : add_hi, dc < x.bias_hi ? add_lo : add_hi);
            const float* brow = s_win + 64 - 32 * c + lane;
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 l4 = *reinterpret_cast<const float4*>(t_lse + c * 32 + e);
              const float4 d4 = *reinterpret_cast<const float4*>(t_delta + c * 32 + e);
              // y = s * scale * log2(e) + bias - lse2 and ds = p * (dp - Delta), two queries per instruction.
              uint64_t l01 = f2(l4.x, l4.y), l23 = f2(l4.z, l4.w);
              if constexpr (kB == 1) {
                l01 = add2(l01, badd);
                l23 = add2(l23, badd);
              } else if constexpr (kB == 2) {
                l01 = add2(l01, f2(brow[-e], brow[-e - 1]));
                l23 = add2(l23, f2(brow[-e - 2], brow[-e - 3]));
              }
              float y[4], p[4], ds[4];
              f2_split(fma2(f2(s[e], s[e + 1]), c2x2, l01), y[0], y[1]);
              f2_split(fma2(f2(s[e + 2], s[e + 3]), c2x2, l23), y[2], y[3]);
#pragma unroll
              for (int u = 0; u < 4; ++u) p[u] = (word & (1u << (e + u))) ? ex2f(y[u]) : 0.f;
              f2_split(mul2(f2(p[0], p[1]), add2(f2(dp[e], dp[e + 1]), f2(d4.x, d4.y))), ds[0], ds[1]);
              f2_split(mul2(f2(p[2], p[3]), add2(f2(dp[e + 2], dp[e + 3]), f2(d4.z, d4.w))), ds[2], ds[3]);
              pw[e / 2] = pack2<BF16>(p[0], p[1]);
              pw[e / 2 + 1] = pack2<BF16>(p[2], p[3]);
              dw[e / 2] = pack2<BF16>(ds[0], ds[1]);
              dw[e / 2 + 1] = pack2<BF16>(ds[2], ds[3]);
              if constexpr (kB != 0) {
#pragma unroll
                for (int u = 0; u < 4; ++u) s[e + u] = ds[u];  // the scores are used up
              }
            }
          };
          if constexpr (kBias) {
            if (near) block(std::integral_constant<int, 2>{});
            else block(std::integral_constant<int, 1>{});
          } else {
            block(std::integral_constant<int, 0>{});
          }
          // A key that keeps no query of the block has dS = 0 whatever its V holds.
          if (word == 0u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) dw[e] = 0u;
            if constexpr (kBias) {
#pragma unroll
              for (int e = 0; e < 32; ++e) s[e] = 0.f;
            }
          }
          // P over S^T columns this warp has read (chunk c writes 16 c ..,
          // which chunks <= c have read).
          tmem_st16(t_lane + col_s(g) + c * 16, pw);
          // dS: row t of the step's tile, queries 32 c .. +31 = 16-byte chunks
          // 4 c .. +3 of its 128 bytes, 128-byte swizzle.
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(ds_row + (((c * 4 + q) ^ (t & 7)) * 16)) =
                make_uint4(dw[4 * q], dw[4 * q + 1], dw[4 * q + 2], dw[4 * q + 3]);
          if constexpr (kBias) {
            if (near) {
              float pos, neg;
              diagonal_sums(s, lane, pos, neg);
              const int kb = key0 / 32, qb = q0 / 32 + c;
              const int slot = x.slot_by_query ? qb : bias_block_max(x.bias_hi, off) - (kb - qb);
              if (qb < x.QB) {
                float* dst =
                    x.near_part + (((static_cast<int64_t>(it.b) * x.H + head) * x.KB + kb) * x.slots + slot) * 64;
                dst[lane] = pos;
                dst[32 + lane] = neg;
              }
            } else {
              uint64_t sum[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) sum[e] = f2(s[2 * e], s[2 * e + 1]);
#pragma unroll
              for (int e = 4; e < 16; ++e) sum[e & 3] = add2(sum[e & 3], f2(s[2 * e], s[2 * e + 1]));
              float a, b2;
              f2_split(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), a, b2);
              if (dc < x.bias_hi) far_lo += a + b2;
              else far_hi += a + b2;
            }
          }
        }
        tmem_wait_st();
        fence_proxy_async_smem();  // dS written by this thread, read by the tensor core
        arrive_warp(ctl.p_full[g]);
        arrive_warp(ctl.tile_free[b]);
      }
      lt0 += n;
      lp0 += (n + 1) / 2;
      if (!ok) break;
      flush_far();
      arrive_warp(ctl.item_free[sl]);
    }
    if (!ok && lane == 0) fail();
  } else if (warp < kScanWarp) {
    // ================================================================ epilogue
    regs_dec<kRegsOther>();
    const int w = (warp - kEpiWarp + 2) & 3;  // a warp reads the TMEM lanes of its index mod 4
    const int t = w * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(w * 32) << 16);
    uint8_t* s_dq = smem + C::kOffDQ + w * 4096;
    const int n_rows = x.hb * x.Nq;  // rows of the accumulator's block that holds a step
    bool ok = true;
    uint32_t lp = 0, use0 = 0, use1 = 0;
    // The staged box (32 rows of 32 columns) is added at (col, row0, block);
    // rows past the block are clipped by the TMA unit.
    auto add_box = [&](int col, int row0, int block) {
      fence_proxy_async_smem();  // staged by every lane, read by the TMA unit
      __syncwarp();
      if (lane == 0 && row0 < n_rows) {
        tma_reduce_add_3d(&tm_dq, smem_u32(s_dq), col, row0, block);
        bulk_commit_group();
      }
    };
    auto box_free = [&]() {
      if (lane == 0) bulk_wait_group_read0();
      __syncwarp();
    };
    for (int j = 0; ok; ++j) {
      const int sl = j % kSlots;
      ok = wait_all(ctl.item_full[sl], (j / kSlots) & 1);
      if (!ok || ctl.unit[sl] < 0) break;
      const int unit = ctl.unit[sl];
      const Item it = item_of(unit);
      const int block0 = (it.b * x.Hkv + it.hkv) * x.gh;
      const int n = static_cast<int>(ctl.n_live[sl]);
      // dV and dK of this key tile (lane t = key), once the item's last products
      // are complete, which the dq_full wait of its last step covers: ahead of
      // that step's dQ, since the next item's first products wait for it.  Zero
      // when no step was live.
      auto write_acc = [&]() {
        // D = 64 reads both out before it stores, so that the next item's first
        // products wait no longer than that; D = 128 has no registers for it.
        const int key = it.kt * kKeys + t;
        const int64_t at = ((static_cast<int64_t>(it.b) * x.Hkv + it.hkv) * x.Nk + key) * D;
        auto read_acc = [&](uint32_t col, float mul, uint32_t (&w)[16]) {
          float u[32];
          tmem_ld32f(t_lane + col, u);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack2<BF16>(u[2 * e] * mul, u[2 * e + 1] * mul);
        };
        auto store_row = [&](uint16_t* dst, const uint32_t (&w)[16]) {
          if (key >= x.Nk) return;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            reinterpret_cast<uint4*>(dst)[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
        };
        if (it.part >= 0) {
          float* dst = x.part_acc + (static_cast<int64_t>(unit - x.whole) * kKeys + t) * (2 * D);
#pragma unroll 1
          for (int h = 0; h < 2 * D / 32; ++h) {  // dV, then dK
            const float mul = h < D / 32 ? 1.f : scale;
            float u[32] = {};
            if (n > 0) {
              tmem_ld32f(t_lane + kColDV + h * 32, u);
              tmem_wait_ld();
            }
#pragma unroll
            for (int q = 0; q < 8; ++q)
              reinterpret_cast<float4*>(dst + h * 32)[q] =
                  make_float4(u[4 * q] * mul, u[4 * q + 1] * mul, u[4 * q + 2] * mul, u[4 * q + 3] * mul);
          }
          if (n > 0) arrive_warp(ctl.acc_free);
        } else if constexpr (D == 64) {
          uint32_t w[4][16] = {};
          if (n > 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              read_acc(kColDV + h * 32, 1.f, w[h]);
              read_acc(C::kColDK + h * 32, scale, w[2 + h]);
            }
            arrive_warp(ctl.acc_free);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            store_row(dv + at + h * 32, w[h]);
            store_row(dk + at + h * 32, w[2 + h]);
          }
        } else {
#pragma unroll 1
          for (int h = 0; h < D / 32; ++h) {
            uint32_t vw[16] = {}, kw[16] = {};
            if (n > 0) {
              read_acc(kColDV + h * 32, 1.f, vw);
              read_acc(C::kColDK + h * 32, scale, kw);
            }
            store_row(dv + at + h * 32, vw);
            store_row(dk + at + h * 32, kw);
          }
          if (n > 0) arrive_warp(ctl.acc_free);
        }
      };
      if (n == 0) write_acc();
      int cw = 0;
      uint32_t cx = ctl.live_bits[sl][0];
      if constexpr (C::kPairDQ) {
        // Thread t = row t of a pair: the first step's 64 rows, then the second's.
        for (int tt = 0; tt < n; tt += 2, ++lp) {
          const int va = next_live(ctl.live_bits[sl], cw, cx);
          const int vb = tt + 1 < n ? next_live(ctl.live_bits[sl], cw, cx) : -1;
          const int b = lp & 1;
          ok = wait_all(ctl.dq_full[b], (lp >> 1) & 1);
          if (!ok) break;
          if (tt + 2 >= n) write_acc();
          float u[64];
          tmem_ld32f(t_lane + C::col_dq(b), u);
          tmem_ld32f(t_lane + C::col_dq(b) + 32, u + 32);
          tmem_wait_ld();
          arrive_warp(ctl.dq_free[b]);
          const int v = w < 2 ? va : vb;
          if (v < 0) continue;
          const int row0 = step_q0(v) + (w & 1) * 32;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            box_free();
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const float* y = u + 32 * h + 4 * c;
              *reinterpret_cast<float4*>(s_dq + lane * 128 + ((c ^ (lane & 7)) * 16)) =
                  make_float4(y[0] * scale, y[1] * scale, y[2] * scale, y[3] * scale);
            }
            add_box(32 * h, row0, block0 + step_block(v));
          }
        }
      } else {
        // Thread t = head dim t; columns are the step's 64 queries.
        for (int tt = 0; tt < n; ++tt) {
          const int v = next_live(ctl.live_bits[sl], cw, cx);
          const int g = tt & 1;
          ok = wait_all(ctl.dq_full[g], (g ? use1 : use0) & 1);
          if (!ok) break;
          if (g) ++use1;
          else ++use0;
          if (tt + 1 == n) write_acc();
          float u[64];
          tmem_ld32f(t_lane + col_dp(g), u);
          tmem_ld32f(t_lane + col_dp(g) + 32, u + 32);
          tmem_wait_ld();
          arrive_warp(ctl.dq_free[g]);
          const int row0 = step_q0(v);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            box_free();
#pragma unroll
            for (int q = 0; q < 32; ++q)
              *reinterpret_cast<float*>(s_dq + q * 128 + (((lane >> 2) ^ (q & 7)) * 16) + (lane & 3) * 4) =
                  u[32 * h + q] * scale;
            add_box(32 * w, row0 + 32 * h, block0 + step_block(v));
          }
        }
      }
      if (!ok) break;
      arrive_warp(ctl.item_free[sl]);
    }
    // The reduce-adds must finish (and stop reading shared memory) before the CTA exits.
    if (lane == 0) bulk_wait_group0();
    if (!ok && lane == 0) fail();
  } else {
    regs_dec<kRegsOther>();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// dtable[bucket][h] = sum of dS over the pairs whose relative position is in
// the bucket: one block per (head, bucket) adds the diagonal sums of the
// blocks near the diagonal, [b][kb] by [d in the bucket's interval], and for
// the last bucket of a side the sums of the blocks beyond.  Every thread adds
// in a fixed order and the threads are added in a fixed tree, so the result
// does not depend on timing; FP32 throughout, rounded once to the table's type
// T (FP32 tables: not at all; a sum over all queries of the batch passes the
// range of fp16 where its terms do not).
// Bound by the latency of its gathers (12 us at B4 H16 N1024, 3.7 MB of sums).
constexpr int kReduceThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kReduceThreads)
    bias_reduce_kernel(const __grid_constant__ BwdGeo x, const __grid_constant__ BiasSpec s, T* __restrict__ dtable) {
  __shared__ float part[kReduceThreads / 32];
  const int h = blockIdx.x, bucket = blockIdx.y;
  const bool high = bucket >= s.side;  // two-sided: keys after the query
  const int i = high ? bucket - s.side : bucket;
  // The bucket's relative positions, as far as they are in near blocks.
  constexpr int kFar = 1 << 28;
  const int first = s.starts[i], next = i + 1 < s.side ? s.starts[i + 1] : kFar;
  int d_lo, d_hi;
  if (high) {
    d_lo = max(1, first);
    d_hi = next - 1;
  } else {
    d_lo = 1 - next;
    d_hi = first == 0 && !s.two_sided ? kFar : -first;
  }
  float acc = 0.f;
  // A warp per batch and stretch of key blocks, so that their loads overlap.
  constexpr int kWarps = kReduceThreads / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = x.B < kWarps ? (kWarps + x.B - 1) / x.B : 1;
  for (int unit = warp; unit < x.B * parts; unit += kWarps) {
    const int b = unit / parts, part = unit - b * parts;
    const int kb0 = x.KB * part / parts, kb1 = x.KB * (part + 1) / parts;
    const int off = x.bias_offsets == nullptr
                        ? x.bias_offset
                        : max(-kMaxBiasOffset, min(kMaxBiasOffset, __ldg(x.bias_offsets + b)));
    const int j_max = bias_block_max(x.bias_hi, off);
    const int j_min = -bias_block_max(-x.bias_lo, -off);
    const int lo = max(d_lo, 32 * j_min - off - 31), hi = min(d_hi, 32 * j_max - off + 31);
    const int64_t n = hi >= lo ? static_cast<int64_t>(hi - lo + 1) * (kb1 - kb0) : 0;
    const float* near_bh = x.near_part + (static_cast<int64_t>(b) * x.H + h) * x.KB * x.slots * 64;
#pragma unroll 4
    for (int64_t w = lane; w < n; w += 32) {
      const int di = static_cast<int>(w / (kb1 - kb0));
      const int kb = kb0 + static_cast<int>(w - static_cast<int64_t>(di) * (kb1 - kb0));
      // d = 32 j - off + k: k in [0, 31] of block j, or k - 32 of block j + 1.
      const int y = lo + di + off;
      const int j = y >= 0 ? y / 32 : -((-y + 31) / 32);
      const int k = y - 32 * j;
      float v[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int jj = j + u, qb = kb - jj;
        const int slot = x.slot_by_query ? qb : j_max - jj;
        if (jj >= j_min && jj <= j_max && qb >= 0 && qb < x.QB && (u == 0 || k != 0))
          v[u] = __ldg(near_bh + (static_cast<int64_t>(kb) * x.slots + slot) * 64 + (u == 0 ? k : k + 32));
      }
      acc += v[0] + v[1];
    }
    const bool low_end = !high && i == s.side - 1;
    const bool high_end = s.two_sided ? high && i == s.side - 1 : i == 0;
    if (low_end || high_end) {
      const float* far_bh = x.far_part + (static_cast<int64_t>(b) * x.H + h) * x.KB * (4 * kMaxParts);
      for (int w = 2 * kMaxParts * kb0 + lane; w < 2 * kMaxParts * kb1; w += 32) {
        if (low_end) acc += __ldg(far_bh + 2 * w);
        if (high_end) acc += __ldg(far_bh + 2 * w + 1);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kReduceThreads / 32; ++w) acc += part[w];
    T& to = dtable[static_cast<int64_t>(bucket) * s.H + h];
    if constexpr (std::is_same_v<T, float>) to = acc;
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) to = __float2bfloat16_rn(acc);
    else to = __float2half_rn(acc);
  }
}

// Fills the geometry; false when the steps of a key head exceed the list.
bool geometry(const CrossParams& p, const DeviceProps& dp, BwdGeo* x) {
  const int sms = dp.sms;
  const int G = static_cast<int>(p.H / p.Hkv);
  x->B = static_cast<int>(p.B);
  x->H = static_cast<int>(p.H);
  x->Hkv = static_cast<int>(p.Hkv);
  x->Nq = static_cast<int>(p.Nq);
  x->Nk = static_cast<int>(p.Nk);
  x->tn = std::min<int>(x->Nq, kQ);
  x->hb = 1;
  const bool bias = p.bias.table != nullptr;
  // With a bias a step holds one head (its blocks belong to one bias row).
  for (int h = 1; !bias && h <= G; ++h)
    if (G % h == 0 && h * x->tn <= kQ) x->hb = h;
  x->gh = G / x->hb;
  x->rows = x->tn * x->hb;
  x->QT1 = (x->Nq + kQ - 1) / kQ;
  // ceil(2^32 / QT1): exact for v < 2^16, as v * (the rounding of it, below
  // QT1 / 2^32 relative) stays below 1 / QT1 for QT1 <= 2^16.
  x->qt_magic = x->QT1 > 1 ? static_cast<uint32_t>((uint64_t{0xFFFFFFFF} + x->QT1) / x->QT1) : 0u;
  x->words = p.words;
  for (int i = 0; i < 3; ++i) x->word_stride[i] = p.word_stride[i];
  x->one_row = p.words != nullptr && (x->Nq == 1 || p.word_stride[2] == 0) && (G == 1 || p.word_stride[1] == 0);
  if (p.words != nullptr && !x->one_row) {
    x->t_stride[2] = (p.Nk + kKeys - 1) / kKeys * kKeys;
    x->t_stride[1] = p.word_stride[1] != 0 ? x->t_stride[2] * x->QT1 : 0;
    x->t_stride[0] = p.word_stride[0] != 0 ? x->t_stride[2] * x->QT1 * (p.word_stride[1] != 0 ? p.H / x->hb : 1) : 0;
  }
  if (bias) {
    x->bias = p.bias_distance;
    x->bias_offsets = p.bias.offsets;
    x->bias_offset = p.bias.offset;
    bias_range(p.bias, &x->bias_lo, &x->bias_hi);
    x->bias_len = x->bias_hi - x->bias_lo + 1 + 2 * kBiasPad;
    x->bias_stride = bias_stride(x->bias_len);
    x->KB = static_cast<int>((p.Nk + kKeys - 1) / kKeys * 4);
    x->QB = (x->Nq + 31) / 32;
    // Block differences that overlap (lo, hi): multiples of 32 in an open
    // interval of length hi - lo + 62.
    const int slots = (x->bias_hi - x->bias_lo + 62 + 31) / 32;
    x->slot_by_query = slots > x->QB ? 1 : 0;
    x->slots = std::min(slots, x->QB);
  }
  // Whole rounds of items, and the rest in parts that make up most of a round,
  // of 4 steps or more: a part costs some steps in itself (start, read-out and
  // the final sum).
  const int64_t items = p.B * p.Hkv * ((p.Nk + kKeys - 1) / kKeys), steps = static_cast<int64_t>(x->gh) * x->QT1;
  x->cut = static_cast<int>(items % sms);
  x->parts = x->cut > 0 ? static_cast<int>(std::max<int64_t>(
                              1, std::min<int64_t>({sms / x->cut, int64_t{kMaxParts}, steps / 4})))
                        : 1;
  if (x->parts == 1) x->cut = 0;
  // By key tile where Q, dO and the dQ accumulator of all heads stay in L2
  // meanwhile: under a causal mask the items with the most steps come first
  // and the shortest last (B4 H16 N1024 D64 with a bias: 81 us, by head 93).
  // Else by head, whose
  // Q and dO the CTAs then share at one time.
  x->tile_major = 8 * p.B * p.H * p.Nq * p.D <= dp.l2_bytes / 2 ? 1 : 0;
  x->whole = static_cast<int>(items - x->cut);
  x->grid = static_cast<int>(std::min<int64_t>(sms, x->whole + int64_t{x->cut} * x->parts));
  return steps <= kMaxSteps;
}

// Offsets, in floats, within the scratch of a backward: the FP32 accumulator of
// dq at 0, -Delta and -lse2, the mask by key and its live bytes, partial sums of
// the bias gradient, dV and dK of parts of items, the next unit.
struct Scratch {
  int64_t delta, words, live, bias, parts, next, end;
};
Scratch scratch_layout(const CrossParams& p, const BwdGeo& x) {
  auto up = [](int64_t n) { return (n + 3) / 4 * 4; };
  const int64_t rows = p.B * p.H * p.Nq;
  Scratch s{};
  s.delta = rows * p.D;
  s.words = s.delta + up(2 * rows);
  const int64_t Bm = p.word_stride[0] != 0 ? p.B : 1, Hm = p.word_stride[1] != 0 ? p.H / x.hb : 1;
  const int64_t masked = Bm * Hm * x.QT1 * x.t_stride[2];  // 0 where the mask is not by key
  s.live = s.words + 2 * masked;
  s.bias = s.live + up(masked / kKeys);
  s.parts = s.bias + (p.bias.table != nullptr ? p.B * p.H * x.KB * (int64_t{64} * x.slots + 4 * kMaxParts) : 0);
  s.next = s.parts + int64_t{x.cut} * x.parts * kKeys * 2 * p.D;
  s.end = s.next + 4;
  return s;
}

template <int D, bool BF16, bool kBias>
int launch(const CrossParams& p, const CrossGrads& g, BwdGeo x, int device, const char** msg) {
  using C = Cfg<D>;
  constexpr size_t kSmemBytes = smem_bytes<D>();
  const int64_t KT = (p.Nk + kKeys - 1) / kKeys;
  const int64_t items = p.B * p.Hkv * KT;
  const int64_t rows = p.B * p.H * p.Nq;
  const int64_t row_blocks = (rows * (D / 8) + 255) / 256;
  if (items > 0x7FFFFFFFll || row_blocks > 0x7FFFFFFFll) {
    *msg = "backward: batch*heads too large";
    return kErrArg;
  }
  CUtensorMap mq, mk, mv, mdo, mdq;
  const int64_t so[3] = {p.H * p.Nq * D, p.Nq * D, D};
  CUresult rc = make_tensor_map_4d(&mq, p.q, p.dtype, D, p.Nq, p.H, p.B, p.q_stride, x.tn, x.hb);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mk, p.k, p.dtype, D, p.Nk, p.Hkv, p.B, p.k_stride, kKeys);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mv, p.v, p.dtype, D, p.Nk, p.Hkv, p.B, p.v_stride, kKeys);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mdo, g.dout, p.dtype, D, p.Nq, p.H, p.B, so, x.tn, x.hb);
  // The accumulator in blocks of hb * Nq rows: a step's rows are consecutive in it.
  if (rc == CUDA_SUCCESS)
    rc = make_tensor_map_3d_f32(&mdq, g.scratch, D, p.B * p.Hkv * x.gh, static_cast<int64_t>(x.hb) * p.Nq, 32);
  if (rc != CUDA_SUCCESS) {
    *msg = tensor_map_error("backward", rc);
    return kErrCuda;
  }
  static std::atomic<bool> smem_set[kMaxDevices] = {};
  auto kern = cross_bwd_kernel<D, BF16, kBias>;
  cudaError_t e = ensure_smem_limit(kern, kSmemBytes, device, smem_set);
  const Scratch at = scratch_layout(p, x);
  float* neg_delta = g.scratch + at.delta;
  float4* dq_accum = reinterpret_cast<float4*>(g.scratch);
  if (kBias) {
    x.near_part = g.scratch + at.bias;
    x.far_part = x.near_part + p.B * p.H * x.KB * x.slots * 64;
  }
  x.part_acc = g.scratch + at.parts;
  x.next = reinterpret_cast<int*>(g.scratch + at.next);
  const int64_t zeros = (at.parts - at.bias) / 4;
  const int64_t zero_blocks = (zeros + 256 * kZeroRounds - 1) / (256 * kZeroRounds);
  Transpose tr{};
  if (x.t_stride[2] != 0) {
    tr.out = reinterpret_cast<uint2*>(g.scratch + at.words);
    tr.live = reinterpret_cast<uint8_t*>(g.scratch + at.live);
    tr.Hm = p.word_stride[1] != 0 ? x.H / x.hb : 1;
    tr.key_words = static_cast<int>(KT * 4);
    tr.total = int64_t{p.word_stride[0] != 0 ? p.B : 1} * tr.Hm * x.QT1 * tr.key_words;
    x.words_t = tr.out;
    x.live_t = reinterpret_cast<const uint32_t*>(tr.live);
  }
  if (row_blocks + zero_blocks + (tr.total + 7) / 8 > 0x7FFFFFFFll) {
    *msg = "backward: batch*heads too large";
    return kErrArg;
  }
  if (e == cudaSuccess)
    e = launch_pdl(cross_prepare_kernel<D, BF16>, static_cast<unsigned>(row_blocks + zero_blocks + (tr.total + 7) / 8), 256, 0,
                   p.stream, static_cast<const uint4*>(g.dout), static_cast<const uint4*>(p.out),
                   static_cast<const uint4*>(p.out_lo), p.lse, neg_delta, neg_delta + rows, dq_accum, rows,
                   static_cast<unsigned>(row_blocks), reinterpret_cast<float4*>(g.scratch + at.bias), zeros,
                   static_cast<unsigned>(zero_blocks), tr, x);
  if (e == cudaSuccess)
    e = launch_pdl(kern, static_cast<unsigned>(x.grid), kThreads, kSmemBytes, p.stream, mq, mk,
                   mv, mdo, mdq, neg_delta + rows, neg_delta, static_cast<uint16_t*>(g.dk), static_cast<uint16_t*>(g.dv),
                   static_cast<int>(KT), p.scale, x, p.err_word, p.timeout_ns);
  const int64_t part_blocks = (int64_t{x.cut} * kKeys * (2 * D / 8) + 255) / 256;
  if (e == cudaSuccess)
    e = launch_pdl(cross_dq_kernel<D, BF16>, static_cast<unsigned>(row_blocks + part_blocks), 256, 0, p.stream, dq_accum,
                   static_cast<uint4*>(g.dq), rows * D / 8, static_cast<unsigned>(row_blocks),
                   static_cast<uint16_t*>(g.dk), static_cast<uint16_t*>(g.dv), static_cast<int>(KT), x);
  if (e == cudaSuccess && kBias) {
    const dim3 grid(static_cast<unsigned>(p.H), static_cast<unsigned>(p.bias.side * (p.bias.two_sided ? 2 : 1)));
    // Not launched early like the others: its few blocks would gather on the
    // SMs that cross_dq_kernel leaves first (B4 H16 N1024 D64 causal, a whole
    // training pass: 158 us, launched early 169).
    using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
    if (g.dtable_f32)
      bias_reduce_kernel<float><<<grid, kReduceThreads, 0, p.stream>>>(x, p.bias, static_cast<float*>(g.dtable));
    else
      bias_reduce_kernel<T><<<grid, kReduceThreads, 0, p.stream>>>(x, p.bias, static_cast<T*>(g.dtable));
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    *msg = cudaGetErrorString(e);
    return kErrLaunch;
  }
  return kOk;
}

template <int D, bool BF16>
int launch_b(const CrossParams& p, const CrossGrads& g, const BwdGeo& x, int device, const char** msg) {
  return p.bias.table != nullptr ? launch<D, BF16, true>(p, g, x, device, msg)
                                 : launch<D, BF16, false>(p, g, x, device, msg);
}

}  // namespace

int64_t cross_bwd_scratch_floats(const CrossParams& p) {
  BwdGeo x{};
  DeviceProps dp;
  const char* msg = nullptr;
  if (!device_props(&dp, &msg)) return -1;
  geometry(p, dp, &x);
  return scratch_layout(p, x).end;
}

int launch_attn_cross_bwd(const CrossParams& p, const CrossGrads& g, const char** msg) {
  BwdGeo x{};
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
  if (!geometry(p, dp, &x)) {
    *msg = "backward: more than 2048 steps of 64 query rows share a key head";
    return kErrUnsupportedN;
  }
  const int dev = dp.device;
  if (p.D == 128) return p.dtype == 1 ? launch_b<128, true>(p, g, x, dev, msg) : launch_b<128, false>(p, g, x, dev, msg);
  return p.dtype == 1 ? launch_b<64, true>(p, g, x, dev, msg) : launch_b<64, false>(p, g, x, dev, msg);
}

}  // namespace sma
