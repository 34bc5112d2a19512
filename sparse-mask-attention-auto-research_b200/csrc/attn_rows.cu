// Attention forward for few query rows per key head (sm_100a): a generated
// token, a few drafted ones, a short question.
//
//   s_ij = scale * q_i . k_j + bias(j - i - offset, h),   O_i = sum_j softmax_j(s_i)_j v_j
//
// over the keys a row keeps (bool mask, length limit, or all), with an
// optional prefix of keys that the whole batch shares in front.  Rows that
// keep no key give O = 0 and lse = -FLT_MAX.
//
// What bounds it: K and V are read once per 16 rows and every key costs a few
// FLOPs per byte, so the kernel is a stream over K and V and the figure of
// merit is HBM bandwidth.  The H / Hkv query heads that share a key head and
// the Nq queries are folded into the rows of one tile (row = g * Nq + i), so
// shared heads share the stream.  Rows fill an m16n8k16 warp MMA: 16 rows are
// what one fragment holds, and a 128-row tcgen05 tile would spend its
// exponentials on padding rows (16384 per 128 keys against the 2048 here).
//
// A work unit is (batch, key head, 16-row tile, piece of the keys).  Its four
// warps work alone: each takes every fourth chunk (8 KiB of keys) of the unit, loads
// it by TMA into its own ring of kStages stages (128-byte swizzle, one
// mbarrier per stage), and keeps its own running maximum, sum and O in
// registers; nothing in the loop waits for another warp.  At the end the
// warps are merged through shared memory in warp order, and the pieces of an
// item through a workspace in piece order by whichever unit finishes last, so
// the result does not depend on timing.
//
// With a bool mask a warp first packs the masks of its next kBatch chunks
// into words (one coalesced byte per lane, a ballot per row and chunk) and
// drops the chunks that no row keeps, before any K or V is requested.
//
// V rows of keys that none of the tile's rows keeps are cleared in shared
// memory before the P V product (0 * Inf or NaN would spoil the sum), so
// unused cache slots and padding may hold anything.
//
// Every wait is bounded and reports through the device error word.
//
// Measured: B16 H32 Hkv8 Nq1 Nk8192 D128, padded to 75 % (403 MB) 78 us, 5.2
// TB/s (lengths of different size leave pieces of different length); B32 H16
// Nq1 Nk2049 D64 with a bias (269 MB) 49 us, 5.5 TB/s.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attn_math.cuh"
#include "rel_bias.cuh"
#include "sma_internal.h"
#include "sma_ptx.cuh"

namespace sma {
namespace {

constexpr int kRows = kRowsTile;  // one m16n8k16 fragment
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;   // chunks in flight per warp
constexpr int kBatch = 32;   // chunks whose masks a warp packs ahead
constexpr int kMaxPieces = 255;

struct RowsParams {
  const uint16_t* q;
  int64_t q_stride[3];
  const uint8_t* mask;
  int64_t mask_stride[3];
  const int32_t* lengths;
  uint16_t* out;
  float* lse;
  float* part_ml;          // every row as a piece for a later merge instead of out / lse (CrossParams)
  float* part_o;
  float* ws;               // [units][16][4] (max, sum, sum of rounded P, -), then [units][16][D]
  unsigned long long* cnt;  // [items]: launch epoch << 8 | pieces finished
  unsigned long long epoch;
  uint32_t* err_word;
  uint64_t timeout_ns;
  int B, H, Hkv, G, Nq, Nk, P;
  int R, RT;               // rows per key head (G * Nq) and 16-row tiles of them
  int pieces;
  int mask_rows;           // 1: all rows of a key head share one mask row, else 0
  float scale_log2;
};

template <int D>
struct RowsCfg {
  // Keys a warp takes at a time: 8 KiB of K and V either way, so that two
  // blocks (eight warps, 192 KiB of loads in flight) fit an SM.
  static constexpr int kChunk = D == 64 ? 32 : 16;
  static constexpr int kTile = kChunk * D * 2;       // K or V of a chunk
  static constexpr int kStageBytes = 2 * kTile;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr size_t kSmem = static_cast<size_t>(kWarps) * kWarpBytes;
  static_assert(kRows * D * 4 <= kWarpBytes, "the merge reuses a warp's ring");
};

struct RowsCtl {
  uint64_t full[kWarps][kStages];
  uint32_t words[kWarps][kBatch][kRows];  // packed masks of the chunks ahead
  int starts[kMaxBiasSide];
  float ml[kWarps][kRows][3];
  uint32_t abort_flag;
  uint32_t last;
};
static_assert(2 * (RowsCfg<128>::kSmem + sizeof(RowsCtl) + 1024) <= 228 * 1024, "two blocks per SM");

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// The n lowest bits, n clamped to [0, 32].
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xFFFFFFFFu : (n <= 0 ? 0u : (1u << n) - 1u); }

template <int D, bool BF16, bool kBias>
__global__ void __launch_bounds__(kThreads, 2)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_kp, const __grid_constant__ CUtensorMap tm_vp,
                     const __grid_constant__ RowsParams p, const __grid_constant__ BiasSpec bias) {
  using C = RowsCfg<D>;
  constexpr int kChunk = C::kChunk, NT = kChunk / 8;  // keys of a chunk, 8-key tiles of it
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  if ((base & 1023u) != 0u) {
    if (threadIdx.x == 0) atomicOr(p.err_word, kDevErrLayout);
    return;
  }
  RowsCtl& ctl = *reinterpret_cast<RowsCtl*>(smem + C::kSmem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = blockIdx.x;
  const int item = unit / p.pieces, piece = unit - item * p.pieces;
  const int bh = item / p.RT, rt = item - bh * p.RT;
  const int b = bh / p.Hkv, hkv = bh - b * p.Hkv;

  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&ctl.full[w][s]), 1);
    ctl.abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if constexpr (kBias) {
    for (int i = threadIdx.x; i < bias.side; i += kThreads) ctl.starts[i] = bias.starts[i];
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait_prior_grid();

  // Rows r0 and r0 + 8 of the tile are this thread's; row = g * Nq + i.
  int row[2], qi[2], head[2];
  bool live_row[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    row[u] = rt * kRows + (lane >> 2) + 8 * u;
    live_row[u] = row[u] < p.R;
    const int rr = live_row[u] ? row[u] : 0;
    const int g = rr / p.Nq;
    qi[u] = rr - g * p.Nq;
    head[u] = hkv * p.G + g;
  }
  // Chunks: the prefix's, then the sequence's own up to its length.
  int len = p.Nk;
  if (p.lengths != nullptr) len = max(0, min(p.Nk, __ldg(p.lengths + b)));
  const int np = (p.P + kChunk - 1) / kChunk;
  const int nc = np + (len + kChunk - 1) / kChunk;
  const int c_lo = static_cast<int>(static_cast<int64_t>(nc) * piece / p.pieces);
  const int c_hi = static_cast<int>(static_cast<int64_t>(nc) * (piece + 1) / p.pieces);
  const int n_mine = c_hi - c_lo > warp ? (c_hi - c_lo - warp + kWarps - 1) / kWarps : 0;
  int limit[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) limit[u] = p.lengths != nullptr ? len - p.Nq + 1 + qi[u] : len;
  // kBias: range of the tile's queries, of the relative positions between
  // which buckets change, and each row's bias beyond them.
  int off = 0, t_lo = 0, t_hi = 0, bias_lo = 0, bias_hi = 0;
  float far_lo[2] = {0.f, 0.f}, far_hi[2] = {0.f, 0.f};
  if constexpr (kBias) {
    off = bias_offset_of(bias, b);
    t_hi = p.Nq - 1;
    bias_lo = -ctl.starts[bias.side - 1];
    bias_hi = bias.two_sided ? -bias_lo : 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!live_row[u]) continue;
      far_lo[u] = bias_value<BF16>(bias, bias.side - 1, head[u]) * kLog2e;
      far_hi[u] = bias_value<BF16>(bias, bias.two_sided ? 2 * bias.side - 1 : 0, head[u]) * kLog2e;
    }
  }

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, lr[2] = {0.f, 0.f};
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

  uint32_t qa[D / 16][4];
  bool have_q = false;
  const uint32_t ring = base + warp * C::kWarpBytes;
  uint32_t n_issued = 0, n_used = 0;
  bool ok = true;
  // The whole warp calls this; lane 0 requests chunk i (of this warp's) into
  // the next stage, which the warp has finished reading.
  auto issue = [&](int i) {
    if (lane == 0) {
      const int c = c_lo + warp + kWarps * i;
      const int s = n_issued % kStages;
      const uint32_t bar = smem_u32(&ctl.full[warp][s]);
      const uint32_t dst = ring + s * C::kStageBytes;
      const bool pre = c < np;
      const int k0 = (pre ? c : c - np) * kChunk;
      const CUtensorMap* mk = pre ? &tm_kp : &tm_k;
      const CUtensorMap* mv = pre ? &tm_vp : &tm_v;
      mbar_arrive_expect_tx(bar, C::kStageBytes);
#pragma unroll
      for (int dc = 0; dc < D / 64; ++dc) {
        tma_load_4d(dst + dc * (kChunk * 128), mk, bar, dc * 64, k0, hkv, pre ? 0 : b);
        tma_load_4d(dst + C::kTile + dc * (kChunk * 128), mv, bar, dc * 64, k0, hkv, pre ? 0 : b);
      }
    }
    ++n_issued;
  };

  const int mask_rows = p.mask_rows ? 1 : min(kRows, p.R - rt * kRows);
  for (int i0 = 0; ok && i0 < n_mine; i0 += kBatch) {
    const int nb = min(kBatch, n_mine - i0);
    uint32_t live = low_bits(nb);
    if (p.mask != nullptr) {
      // Pack the masks of the batch's chunks; a lane reads one key of a row.
      __syncwarp();
      for (int r = 0; r < mask_rows; ++r) {
        const int rr = rt * kRows + r;
        const int g = rr / p.Nq;
        const uint8_t* mrow = p.mask + b * p.mask_stride[0] + (hkv * p.G + g) * p.mask_stride[1] +
                              (rr - g * p.Nq) * p.mask_stride[2];
        constexpr int kPer = 32 / kChunk;  // chunks per ballot
        for (int i = 0; i < nb; i += 8 * kPer) {
          uint8_t x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int ii = i + u * kPer + lane / kChunk;
            const int key = (c_lo + warp + kWarps * (i0 + ii) - np) * kChunk + lane % kChunk;
            x[u] = (ii < nb && key >= 0 && key < len) ? __ldg(mrow + key) : 0;
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const uint32_t w = __ballot_sync(0xffffffffu, x[u] != 0);
            const int ii = i + u * kPer + lane;
            if (lane < kPer && ii < nb) ctl.words[warp][ii][r] = (w >> (lane * kChunk)) & low_bits(kChunk);
          }
        }
      }
      __syncwarp();
      uint32_t any = 0u;
      if (lane < nb)
        for (int r = 0; r < mask_rows; ++r) any |= ctl.words[warp][lane][r];
      const bool keep = lane < nb && (any != 0u || c_lo + warp + kWarps * (i0 + lane) < np);
      live = __ballot_sync(0xffffffffu, keep);
    }
    uint32_t ahead = live;
    for (int s = 0; s < kStages && ahead != 0u; ++s) {
      issue(i0 + __ffs(ahead) - 1);
      ahead &= ahead - 1u;
    }
    if (!have_q) {  // behind the first requests for keys
      have_q = true;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint16_t* src = p.q + b * p.q_stride[0] + head[u] * p.q_stride[1] + qi[u] * p.q_stride[2] + 2 * (lane & 3);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qa[kk][u] = live_row[u] ? *reinterpret_cast<const uint32_t*>(src + kk * 16) : 0u;
          qa[kk][2 + u] = live_row[u] ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8) : 0u;
        }
      }
    }
    while (live != 0u) {
      const int i = __ffs(live) - 1;
      live &= live - 1u;
      const int c = c_lo + warp + kWarps * (i0 + i);
      const bool pre = c < np;
      const int k0 = (pre ? c : c - np) * kChunk;
      const int s = n_used % kStages;
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&ctl.full[warp][s]), (n_used / kStages) & 1,
                                                      &ctl.abort_flag, p.timeout_ns))) {
        ok = false;
        break;
      }
      ++n_used;
      // Which of the chunk's keys each of this thread's rows keeps.
      uint32_t word[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t w;
        if (pre) w = low_bits(p.P - k0);
        else if (p.mask != nullptr) w = ctl.words[warp][i][p.mask_rows ? 0 : (lane >> 2) + 8 * u];
        else w = low_bits(limit[u] - k0);
        word[u] = live_row[u] ? w & low_bits(kChunk) : 0u;
      }
      const uint32_t sK = ring + s * C::kStageBytes, sV = sK + C::kTile;
      // V of keys no row keeps: cleared (see the head comment).
      const uint32_t kept = __reduce_or_sync(0xffffffffu, word[0] | word[1]);
      if (kept != low_bits(kChunk)) {
        if (lane < kChunk && ((kept >> lane) & 1u) == 0u) {
          uint8_t* v = smem + warp * C::kWarpBytes + s * C::kStageBytes + C::kTile + lane * 128;
#pragma unroll
          for (int x = 0; x < D / 8; ++x)
            *reinterpret_cast<uint4*>(v + (x >> 3) * (kChunk * 128) + (x & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();  // before the stage is loaded again
        __syncwarp();
      }

      float sc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
      const int mat = lane >> 3, mrow = lane & 7;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          const int key = (n + (mat >> 1)) * 8 + mrow;
          const int ch = kk * 2 + (mat & 1);
          uint32_t kb[4];
          ldsm4(sK + (ch >> 3) * (kChunk * 128) + key * 128 + (((ch & 7) ^ (key & 7)) << 4), kb);
          mma16816<BF16>(sc[n], qa[kk], kb[0], kb[1]);
          mma16816<BF16>(sc[n + 1], qa[kk], kb[2], kb[3]);
        }
      }
      // Scores in units of log2, masked; then the running maximum.
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] *= p.scale_log2;
      if constexpr (kBias) {
        // A chunk beyond the last bucket's start for all rows has one bias per
        // row, kept in registers.  Otherwise lane x finds the bias of the
        // chunk's key x, row by row, and the rows' threads fetch it from there.
        const int d_first = k0 - t_hi - off, d_last = k0 + kChunk - 1 - t_lo - off;
        if (d_last <= bias_lo || d_first >= bias_hi) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float add = d_last <= bias_lo ? far_lo[u] : far_hi[u];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              sc[n][2 * u] += add;
              sc[n][2 * u + 1] += add;
            }
          }
        } else {
          const int rows = min(kRows, p.R - rt * kRows);
#pragma unroll 2
          for (int r = 0; r < rows; ++r) {
            const int rr = rt * kRows + r, g = rr / p.Nq;
            const int bucket = bias_bucket(bias, ctl.starts, k0 + lane - (rr - g * p.Nq) - off);
            const float x = bias_value<BF16>(bias, bucket, hkv * p.G + g) * kLog2e;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float y = __shfl_sync(0xffffffffu, x, n * 8 + 2 * (lane & 3) + e);
                if (r == (lane >> 2)) sc[n][e] += y;
                if (r == (lane >> 2) + 8) sc[n][2 + e] += y;
              }
          }
        }
      }
      float alpha[2], mu[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t bit = 1u << (n * 8 + 2 * (lane & 3) + e);
            float& x = sc[n][2 * u + e];
            x = (word[u] & bit) ? x : -INFINITY;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m[u], mx);
        mu[u] = m_new == -INFINITY ? 0.f : m_new;
        alpha[u] = ex2f(m[u] - mu[u]);  // 0 while nothing has been kept
        m[u] = m_new;
        l[u] *= alpha[u];
        lr[u] *= alpha[u];
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][0] *= alpha[0];
          o[n][1] *= alpha[0];
          o[n][2] *= alpha[1];
          o[n][3] *= alpha[1];
        }
      }
      // P, rounded to the inputs' type for the product with V (the type the
      // matrix instruction takes); O is divided by the sum of the rounded
      // values, the LSE uses the unrounded ones.
      uint32_t pa[kChunk / 16][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float p0 = ex2f(sc[n][2 * u] - mu[u]), p1 = ex2f(sc[n][2 * u + 1] - mu[u]);
          l[u] += p0 + p1;
          const uint32_t w = pack2<BF16>(p0, p1);
          const float2 rounded = unpack2<BF16>(w);
          lr[u] += rounded.x + rounded.y;
          pa[n >> 1][(n & 1) * 2 + u] = w;
        }
#pragma unroll
      for (int ks = 0; ks < kChunk / 16; ++ks) {
#pragma unroll
        for (int n = 0; n < D / 8; n += 2) {
          const int key = ks * 16 + (mat & 1) * 8 + mrow;
          const int ch = n + (mat >> 1);
          uint32_t vb[4];
          ldsm4_t(sV + (ch >> 3) * (kChunk * 128) + key * 128 + (((ch & 7) ^ (key & 7)) << 4), vb);
          mma16816<BF16>(o[n], pa[ks], vb[0], vb[1]);
          mma16816<BF16>(o[n + 1], pa[ks], vb[2], vb[3]);
        }
      }
      __syncwarp();  // every lane has read the stage
      if (ahead != 0u) {
        issue(i0 + __ffs(ahead) - 1);
        ahead &= ahead - 1u;
      }
    }
  }
  if (!ok && lane == 0) {
    ctl.abort_flag = 1;
    atomicOr(p.err_word, kDevErrTimeout);
    // The copies in flight land before the block leaves.
    for (; n_used < n_issued; ++n_used)
      mbar_drain(smem_u32(&ctl.full[warp][n_used % kStages]), (n_used / kStages) & 1, p.timeout_ns);
  }
  __syncwarp();

  // The four warps' rows, merged in warp order.
  float* po = reinterpret_cast<float*>(smem + warp * C::kWarpBytes);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
    lr[u] += __shfl_xor_sync(0xffffffffu, lr[u], 1);
    lr[u] += __shfl_xor_sync(0xffffffffu, lr[u], 2);
    const int r = (lane >> 2) + 8 * u;
    if ((lane & 3) == 0) {
      ctl.ml[warp][r][0] = m[u];
      ctl.ml[warp][r][1] = l[u];
      ctl.ml[warp][r][2] = lr[u];
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<float2*>(po + r * D + n * 8 + 2 * (lane & 3)) = make_float2(o[n][2 * u], o[n][2 * u + 1]);
  }
  __syncthreads();
  if (ctl.abort_flag != 0u) {
    // Counted all the same: a replay of the launch uses the counter again.
    if (threadIdx.x == 0 && p.pieces > 1 && claim_last_piece(p.cnt + item, p.epoch, p.pieces))
      atomicExch(p.cnt + item, 0ull);
    return;
  }
  const int rows = min(kRows, p.R - rt * kRows);
  constexpr int kVec = D / 4;  // float4 per row
  // Writes row r's column group x: normalised, in the inputs' type, or as a
  // piece for a later merge (FP32, not normalised).
  auto write_out = [&](int r, int x, const float4& a, float inv) {
    const int rr = rt * kRows + r;
    const int g = rr / p.Nq;
    if (p.part_o != nullptr) {
      float* dst = p.part_o + ((static_cast<int64_t>(b) * p.H + hkv * p.G + g) * p.Nq + (rr - g * p.Nq)) * D + 4 * x;
      *reinterpret_cast<float4*>(dst) = a;
      return;
    }
    uint16_t* dst = p.out + ((static_cast<int64_t>(b) * p.H + hkv * p.G + g) * p.Nq + (rr - g * p.Nq)) * D + 4 * x;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF16>(a.x * inv, a.y * inv), pack2<BF16>(a.z * inv, a.w * inv));
  };
  auto write_sums = [&](int r, float M, float sum, float sumr) {
    const int rr = rt * kRows + r;
    const int g = rr / p.Nq;
    const int64_t at = (static_cast<int64_t>(b) * p.H + hkv * p.G + g) * p.Nq + (rr - g * p.Nq);
    if (p.part_ml != nullptr) *reinterpret_cast<float4*>(p.part_ml + at * 4) = make_float4(M, sum, sumr, 0.f);
    if (p.lse != nullptr) p.lse[at] = sum != 0.f ? (M + log2f(sum)) * kLn2 : -FLT_MAX;
  };
  const int64_t n_units = gridDim.x;
  float* ws_ml = p.ws;
  float* ws_o = p.ws + n_units * kRows * 4;
  for (int idx = threadIdx.x; idx < rows * kVec; idx += kThreads) {
    const int r = idx / kVec, x = idx - r * kVec;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ctl.ml[w][r][0]);
    float sum = 0.f, sumr = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = ctl.ml[w][r][0];
      const float f = mw == -INFINITY ? 0.f : ex2f(mw - M);
      const float4 v = *reinterpret_cast<const float4*>(smem + w * C::kWarpBytes + (r * D + 4 * x) * 4);
      sum += f * ctl.ml[w][r][1];
      sumr += f * ctl.ml[w][r][2];
      a.x += f * v.x;
      a.y += f * v.y;
      a.z += f * v.z;
      a.w += f * v.w;
    }
    if (p.pieces == 1) {
      write_out(r, x, a, sumr > 0.f ? 1.f / sumr : 0.f);
      if (x == 0) write_sums(r, M, sum, sumr);
    } else {
      const int64_t at = static_cast<int64_t>(unit) * kRows + r;
      *reinterpret_cast<float4*>(ws_o + at * D + 4 * x) = a;
      if (x == 0) *reinterpret_cast<float4*>(ws_ml + at * 4) = make_float4(M, sum, sumr, 0.f);
    }
  }
  if (p.pieces == 1) return;

  // The unit that completes its item's count merges the pieces in order.
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = claim_last_piece(p.cnt + item, p.epoch, p.pieces);
    // Back to zero, so a replay of the same launch (a CUDA graph: the same
    // workspace and epoch) counts afresh.
    if (last) atomicExch(p.cnt + item, 0ull);
    ctl.last = last ? 1u : 0u;
  }
  __syncthreads();
  if (ctl.last == 0u) return;
  __threadfence();
  float* weight = reinterpret_cast<float*>(smem);  // [pieces][16]
  float* total = weight + kMaxPieces * kRows;      // [16] 1 / sum of rounded P
  float4* part = reinterpret_cast<float4*>(total + kRows);  // [kThreads]
  static_assert(kRows * 8 == kThreads && kMaxPieces * kRows % 4 == 0, "eight threads per row; part is aligned");
  const int64_t u0 = static_cast<int64_t>(item) * p.pieces;
  {
    // Eight threads per row, each every eighth piece, added in a fixed tree.
    const int r = threadIdx.x >> 3, j = threadIdx.x & 7;
    const float* src = ws_ml + (u0 * kRows + r) * 4;
    const int n = r < rows ? p.pieces : 0;
    float M = -INFINITY, sum = 0.f, sumr = 0.f;
#pragma unroll 4
    for (int pc = j; pc < n; pc += 8) M = fmaxf(M, __ldcg(src + pc * (kRows * 4)));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
#pragma unroll 4
    for (int pc = j; pc < n; pc += 8) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(src + pc * (kRows * 4)));
      const float f = v.x == -INFINITY ? 0.f : ex2f(v.x - M);
      weight[pc * kRows + r] = f;
      sum += f * v.y;
      sumr += f * v.z;
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      sumr += __shfl_xor_sync(0xffffffffu, sumr, o);
    }
    if (j == 0 && r < rows) {
      total[r] = sumr > 0.f ? 1.f / sumr : 0.f;
      write_sums(r, M, sum, sumr);
    }
  }
  __syncthreads();
  // Four columns of a row per thread; few rows share the pieces among `groups`
  // threads, whose sums are added in order.
  const int vecs = rows * kVec, groups = max(1, kThreads / vecs);
  for (int i0 = 0; i0 < vecs; i0 += kThreads) {
    const int idx = groups > 1 ? threadIdx.x % vecs : i0 + threadIdx.x, grp = groups > 1 ? threadIdx.x / vecs : 0;
    const int r = idx / kVec, x = idx - r * kVec;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (idx < vecs && grp < groups) {
      const float* src = ws_o + (u0 * kRows + r) * D + 4 * x;
#pragma unroll 8
      for (int pc = grp; pc < p.pieces; pc += groups) {
        const float f = weight[pc * kRows + r];
        const float4 v = __ldcg(reinterpret_cast<const float4*>(src + static_cast<int64_t>(pc) * kRows * D));
        a.x += f * v.x;
        a.y += f * v.y;
        a.z += f * v.z;
        a.w += f * v.w;
      }
    }
    if (groups > 1) {
      part[threadIdx.x] = a;
      __syncthreads();
      if (grp == 0) {
        for (int k = 1; k < groups; ++k) {
          const float4 v = part[k * vecs + idx];
          a.x += v.x;
          a.y += v.y;
          a.z += v.z;
          a.w += v.w;
        }
      }
    }
    if (idx < vecs && grp == 0) write_out(r, x, a, total[r]);
  }
}

// Pieces of the keys per item.  Units run in rounds of `slots`; in steps of a
// chunk per warp (0.75 to 0.8 us) a unit costs its chunks and 4 more, a split 5
// (workspace, merge) and a little per piece.  Measured, one row per key head:
// B1 Hkv1 Nk131072 D64 18 us in 148 pieces, 100 in 8; B1 Hkv8 Nk2048 D128 11.1 in 8, 28.4
// whole; B16 Hkv8 Nk1024 D64 10.6 whole, 11.6 in 2; Nk2048 17.9 whole, 15.2 in 2.
int choose_pieces(int64_t items, int64_t chunks, int64_t slots) {
  const int64_t most = std::min<int64_t>(kMaxPieces, chunks / (2 * kWarps));
  int best = 1;
  double best_cost = 0.0;
  for (int64_t pc = 1; pc <= std::max<int64_t>(most, 1); ++pc) {
    const double rounds = static_cast<double>((items * pc + slots - 1) / slots);
    const double steps = static_cast<double>((chunks + kWarps * pc - 1) / (kWarps * pc));
    const double cost = rounds * (steps + 4.0) + (pc > 1 ? 5.0 + 0.04 * static_cast<double>(pc) : 0.0);
    if (pc == 1 || cost < best_cost * 0.999) {
      best = static_cast<int>(pc);
      best_cost = cost;
    }
  }
  return best;
}

template <int D, bool BF16, bool kBias>
int launch(const CrossParams& a, const char** msg) {
  using C = RowsCfg<D>;
  constexpr size_t kSmem = C::kSmem + sizeof(RowsCtl);
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
  RowsParams p{};
  p.q = static_cast<const uint16_t*>(a.q);
  p.mask = a.mask;
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = a.q_stride[i];
    p.mask_stride[i] = a.mask_stride[i];
  }
  p.lengths = a.lengths;
  p.out = static_cast<uint16_t*>(a.out);
  p.lse = a.lse;
  p.part_ml = a.part_ml;
  p.part_o = a.part_o;
  p.err_word = a.err_word;
  p.timeout_ns = a.timeout_ns;
  p.B = static_cast<int>(a.B);
  p.H = static_cast<int>(a.H);
  p.Hkv = static_cast<int>(a.Hkv);
  p.G = static_cast<int>(a.H / a.Hkv);
  p.Nq = static_cast<int>(a.Nq);
  p.Nk = static_cast<int>(a.Nk);
  p.P = static_cast<int>(a.P);
  p.R = p.G * p.Nq;
  p.RT = (p.R + kRows - 1) / kRows;
  p.mask_rows = a.mask != nullptr && (a.Nq == 1 || a.mask_stride[2] == 0) && (p.G == 1 || a.mask_stride[1] == 0) ? 1 : 0;
  p.scale_log2 = a.scale * kLog2e;
  if (a.H / a.Hkv * a.Nq > 0x7FFFFFFFll - kRows) {
    *msg = "attention: too many query rows";
    return kErrArg;
  }
  const int64_t items = a.B * a.Hkv * p.RT;
  constexpr int kChunk = C::kChunk;
  const int64_t chunks = (a.P + kChunk - 1) / kChunk + (a.Nk + kChunk - 1) / kChunk;
  p.pieces = choose_pieces(items, chunks, 2 * static_cast<int64_t>(dp.sms));
  const int64_t units = items * p.pieces;
  if (units > 0x7FFFFFFFll) {
    *msg = "attention: too many query rows";
    return kErrArg;
  }
  CUtensorMap mk, mv, mkp, mvp;
  CUresult rc = CUDA_SUCCESS;
  if (a.Nk > 0) {
    rc = make_tensor_map_4d(&mk, a.k, a.dtype, D, a.Nk, a.Hkv, a.B, a.k_stride, kChunk);
    if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mv, a.v, a.dtype, D, a.Nk, a.Hkv, a.B, a.v_stride, kChunk);
  }
  if (rc == CUDA_SUCCESS && a.P > 0) {
    const int64_t ks[3] = {0, a.kp_stride[0], a.kp_stride[1]}, vs[3] = {0, a.vp_stride[0], a.vp_stride[1]};
    rc = make_tensor_map_4d(&mkp, a.k_prefix, a.dtype, D, a.P, a.Hkv, 1, ks, kChunk);
    if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mvp, a.v_prefix, a.dtype, D, a.P, a.Hkv, 1, vs, kChunk);
  }
  if (rc != CUDA_SUCCESS) {
    *msg = tensor_map_error("attention", rc);
    return kErrCuda;
  }
  // A map that no chunk uses is a copy of one that is there.
  if (a.Nk == 0) mk = mkp, mv = mvp;
  if (a.P == 0) mkp = mk, mvp = mv;
  static std::atomic<bool> smem_set[kMaxDevices] = {};
  auto kern = attn_rows_kernel<D, BF16, kBias>;
  cudaError_t e = ensure_smem_limit(kern, kSmem, dp.device, smem_set);
  void* ws = nullptr;
  if (e == cudaSuccess && p.pieces > 1) {
    const size_t cnt_bytes = (static_cast<size_t>(items) * 8 + 255) / 256 * 256;
    e = scratch_alloc_async(&ws, cnt_bytes + static_cast<size_t>(units) * kRows * (4 + D) * sizeof(float), a.stream);
    p.cnt = static_cast<unsigned long long*>(ws);
    p.ws = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + cnt_bytes);
    p.epoch = next_launch_epoch();
  }
  if (e == cudaSuccess)
    e = launch_pdl(kern, static_cast<unsigned>(units), kThreads, kSmem, a.stream, mk, mv, mkp, mvp, p, a.bias);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (ws != nullptr) {
    const cudaError_t ef = cudaFreeAsync(ws, a.stream);
    if (e == cudaSuccess) e = ef;
  }
  if (e != cudaSuccess) {
    *msg = cudaGetErrorString(e);
    return kErrLaunch;
  }
  return kOk;
}

template <int D, bool BF16>
int launch_b(const CrossParams& a, const char** msg) {
  return a.bias.table != nullptr ? launch<D, BF16, true>(a, msg) : launch<D, BF16, false>(a, msg);
}

}  // namespace

int launch_attn_rows(const CrossParams& a, const char** msg) {
  if (a.D == 128) return a.dtype == 1 ? launch_b<128, true>(a, msg) : launch_b<128, false>(a, msg);
  return a.dtype == 1 ? launch_b<64, true>(a, msg) : launch_b<64, false>(a, msg);
}

}  // namespace sma
