// Attention forward of queries and keys of different lengths on the two-chain
// kernel (attn_fwd_chain.cuh, kX): its mask packer, the bias laid out by
// relative position, and the host side.
#include "attn_fwd_chain.cuh"

namespace sma {
namespace {

// ---------------------------------------------------------------- bias by relative position
// Value i of head h is log2(e) * table[bucket(lo - kBiasPad + i)][h], laid out
// as bias_stride (sma_internal.h) says: a row of the attention kernel reads the
// bias of consecutive keys in vectors, at any start (B16 H12 N512 D64 with a
// random mask, 32 buckets: 57 us, with a scalar load for every key 59).
struct ExpandParams {
  BiasSpec bias;
  int bf16, lo, len;
  int64_t stride;
  float* out;
  int blocks, head_blocks;  // 0 blocks: no bias
};

__device__ __forceinline__ void expand_bias(const ExpandParams& e, int block, int* starts) {
  __shared__ int bucket[260];  // of values 4 j0 - 3 .. 4 j0 + 256
  __shared__ float value[260];
  for (int i = threadIdx.x; i < e.bias.side; i += 256) starts[i] = e.bias.starts[i];
  __syncthreads();
  pdl_wait_prior_grid();
  const int j0 = block / e.head_blocks * 64;
  for (int i = threadIdx.x; i < 260; i += 256)
    bucket[i] = bias_bucket(e.bias, starts, e.lo - kBiasPad + max(0, min(e.len - 1, 4 * j0 - 3 + i)));
  const int j = threadIdx.x >> 2, k = threadIdx.x & 3;
  for (int h = block % e.head_blocks; h < e.bias.H; h += e.head_blocks) {
    __syncthreads();
    for (int i = threadIdx.x; i < 260; i += 256)
      value[i] = kLog2e * (e.bf16 ? bias_value<true>(e.bias, bucket[i], h) : bias_value<false>(e.bias, bucket[i], h));
    __syncthreads();
    const float* v = value + 4 * j + 3 - k;
    if (16ll * (j0 + j) < e.stride)
      reinterpret_cast<float4*>(e.out + h * e.stride)[4 * (j0 + j) + k] = make_float4(v[0], v[1], v[2], v[3]);
  }
}

// ---------------------------------------------------------------- mask packer
// bool bytes with any batch / head / query strides -> words [Bm, Hm, Qm, W],
// W = 4 ceil(Nk / 128) (whole 128-key tiles; bits at columns >= Nk are 0), and
// for every 128-row tile of the attention kernel (Geo's rows) the bits of its
// live key tiles, which then needs no scan of the words, and the keys that some
// row of the tile keeps (the others' V is cleared there).  One CTA per tile and
// stretch of 8 key tiles or more; a thread packs the words of one column in
// every kPackThreads / columns-th row and notes whether it saw one live.
//
// A word's 32 bytes start at any address: the aligned 16-byte vectors that
// cover them are packed to bits first, and the bits are shifted into place.
// Bound by HBM: every mask byte is read once (a vector shared by two words the
// second time from L1).  Vectors that would reach outside the mask's own span
// [lo, hi) are read byte by byte.
// kAligned: every row starts on 16 bytes, so no word needs a third vector.  B16
// H12 Nq512 Nk512, 50 MB of mask: 13.9 us, 3.6 TB/s (the general form: 19; two
// words a thread in flight instead of four 2 us more, eight 4 us more).
constexpr int kPackThreads = 256;
constexpr int kPackWords = 256;   // words of a row per CTA, at most
constexpr int kPackRounds = 4;    // words per thread with their loads in flight

struct PackParams {
  const uint8_t* mask;
  const uint8_t* hi;          // end of the mask's span
  int64_t sb, sh, sq;
  uint32_t* words;
  uint8_t* occ;               // [Bm][Hb][QT][occ_words * 4], 8 key tiles per byte
  uint32_t* kept;             // [Bm][Hb][QT][W]
  int Hm, Qm, Nk, W;
  int hb, tn, rows;           // heads and queries of a tile, as far as the mask has them
  int Hb, QT;                 // head blocks, query tiles
  int chunks, chunk_log2;     // stretches of a row, 2^chunk_log2 words each
  int occ_words, tile_log2;   // words of live bits per tile; packed words per key tile
};

// With a bias, the first blocks of the launch lay that out.
template <bool kAligned>
__global__ void __launch_bounds__(kPackThreads)
    pack_tiles_kernel(const __grid_constant__ PackParams p, const __grid_constant__ ExpandParams e) {
  pdl_launch_dependents();
  constexpr int kVecs = kAligned ? 2 : 3;
  __shared__ uint32_t live[kPackWords / 2 / 32];  // a key tile is 2 or 4 words
  __shared__ uint32_t kept[kPackWords];
  if (static_cast<int>(blockIdx.x) < e.blocks) {
    static_assert(kPackWords >= kMaxBiasSide && kPackThreads == 256, "bucket starts; threads of expand_bias");
    expand_bias(e, static_cast<int>(blockIdx.x), reinterpret_cast<int*>(kept));
    return;
  }
  const int block = static_cast<int>(blockIdx.x) - e.blocks;
  const int chunk = block % p.chunks;
  int rest = block / p.chunks;
  const int qt = rest % p.QT;
  rest /= p.QT;
  const int hblk = rest % p.Hb;
  const int64_t b = rest / p.Hb;
  if (threadIdx.x < kPackWords / 2 / 32) live[threadIdx.x] = 0u;
  kept[threadIdx.x] = 0u;
  static_assert(kPackThreads == kPackWords, "one thread per column");
  pdl_wait_prior_grid();
  const int c = threadIdx.x & ((1 << p.chunk_log2) - 1), w = (chunk << p.chunk_log2) + c;
  const int valid = p.Nk - 32 * w;
  const int step = kPackThreads >> p.chunk_log2;
  uint32_t any = 0u;
  for (int r0 = threadIdx.x >> p.chunk_log2; w < p.W && r0 < p.rows; r0 += step * kPackRounds) {
    // All loads first: the two or three aligned vectors of each word.
    uint4 x[kPackRounds][kVecs];
    const uint8_t* src[kPackRounds];
    int64_t at[kPackRounds];
    bool whole[kPackRounds];
#pragma unroll
    for (int u = 0; u < kPackRounds; ++u) {
      const int r = r0 + u * step;
      const int hr = p.hb > 1 ? r / p.tn : 0, t = qt * kBM + r - hr * p.tn;
      const int64_t h = static_cast<int64_t>(hblk) * p.hb + hr;
      const bool in = r < p.rows && t < p.Qm;
      at[u] = in ? ((b * p.Hm + h) * p.Qm + t) * p.W + w : -1;
      src[u] = p.mask + b * p.sb + h * p.sh + t * p.sq + 32 * w;
      const int sh = kAligned ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(src[u]) & 15u);
      const uint8_t* v = src[u] - sh;
      whole[u] = in && valid > 0 && v >= p.mask && v + (sh != 0 ? 48 : 32) <= p.hi;
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
      x[u][0] = whole[u] ? __ldcs(reinterpret_cast<const uint4*>(v)) : zero;
      x[u][1] = whole[u] ? __ldcs(reinterpret_cast<const uint4*>(v) + 1) : zero;
      if constexpr (!kAligned)
        x[u][2] = whole[u] && sh != 0 ? __ldcs(reinterpret_cast<const uint4*>(v) + 2) : zero;
    }
#pragma unroll
    for (int u = 0; u < kPackRounds; ++u) {
      uint32_t word = bytes_are_01(x[u][0], x[u][1]) ? pack32_01(x[u][0], x[u][1]) : pack32_any(x[u][0], x[u][1]);
      if constexpr (!kAligned) {
        const int sh = static_cast<int>(reinterpret_cast<uintptr_t>(src[u]) & 15u);
        word = __funnelshift_r(word, pack16_any(x[u][2]), sh);
      }
      word &= (valid >= 32 ? 0xFFFFFFFFu : (1u << max(valid, 0)) - 1u);
      if (at[u] >= 0 && !whole[u])
        for (int i = 0; i < min(valid, 32); ++i) word |= (src[u][i] != 0 ? 1u : 0u) << i;
      if (at[u] >= 0) p.words[at[u]] = word;
      any |= word;
    }
  }
  __syncthreads();
  if (any != 0u) {
    atomicOr(&live[(c >> p.tile_log2) >> 5], 1u << ((c >> p.tile_log2) & 31));
    atomicOr(&kept[c], any);
  }
  __syncthreads();
  if (threadIdx.x < (1 << p.chunk_log2) && w < p.W)
    p.kept[((b * p.Hb + hblk) * p.QT + qt) * p.W + w] = kept[c];
  // Bytes of live bits of a chunk (a row in one chunk may have fewer than 8 tiles, and writes all of its words).
  const int bytes = p.chunks == 1 ? p.occ_words * 4 : 1 << (p.chunk_log2 - p.tile_log2 - 3);
  const int k = chunk * bytes + threadIdx.x;
  if (threadIdx.x < bytes && k < p.occ_words * 4)
    p.occ[((b * p.Hb + hblk) * p.QT + qt) * (p.occ_words * 4) + k] = reinterpret_cast<const uint8_t*>(live)[threadIdx.x];
}

// ---------------------------------------------------------------- merge of a split launch
// Row (b, h, i) of every piece of its item, and `in` (its other keys, attended
// by an earlier launch), merged in that order: weights 2^(m_p - M) against
// the overall maximum M, O = sum w_p O_p / sum w_p l_out_p.  Writes O and the
// LSE, or (`out_ml`) the merged row as a piece for a later merge.  One warp
// per row, so every read is a whole row of D floats; bound by reading the
// pieces, mostly from L2 (they have just been written): 256 pieces of 128 rows,
// D128 (17 MB), 10 us.  Eight pieces in flight (18 pieces a row, whole call:
// 65.1 us, with four 66.1; with two pieces a row no difference).
struct MergeParams {
  const float* ws;   // [units][128][4] (max, sum, sum of rounded P, -) then [units][128][D]
  int64_t units;
  int pieces, groups, QT, head_major;
  const float* in_ml;
  const float* in_o;
  float* out_ml;
  float* out_o;
  uint16_t* out;
  float* lse;
  int64_t rows;      // B * H * Nq
};

constexpr int kMergeWarps = 4;

template <int D, bool BF16>
__global__ void __launch_bounds__(kMergeWarps * 32)
    merge_rows_kernel(const __grid_constant__ MergeParams m, const __grid_constant__ Geo x) {
  constexpr int kPer = D / 32;  // floats per lane
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kMergeWarps + (threadIdx.x >> 5);
  if (row >= m.rows) return;
  const int64_t bh = row / x.Nq;
  const int i = static_cast<int>(row - bh * x.Nq);
  const int b = static_cast<int>(bh / x.H), h = static_cast<int>(bh - static_cast<int64_t>(b) * x.H);
  const int qt = i / kBM, per_kv = x.gh * x.hb;
  const int hkv = h / per_kv, hg = h - hkv * per_kv, bt = b / x.nb;
  const int r = ((b - bt * x.nb) * x.hb + hg % x.hb) * x.tn + (i - qt * kBM);
  const int group = (bt * x.Hkv + hkv) * x.gh + hg / x.hb;
  const int64_t slow = m.QT - 1 - qt;
  const int64_t item = m.head_major ? static_cast<int64_t>(group) * m.QT + slow : slow * m.groups + group;
  const float* ml = m.ws + (item * m.pieces * kBM + r) * 4;
  const float* po = m.ws + m.units * kBM * 4 + (item * m.pieces * kBM + r) * D + lane * kPer;

  float4 in = make_float4(-INFINITY, 0.f, 0.f, 0.f);
  if (m.in_ml != nullptr) in = __ldcg(reinterpret_cast<const float4*>(m.in_ml + row * 4));
  float M = in.x;
  for (int p = lane; p < m.pieces; p += 32) M = fmaxf(M, __ldcg(ml + static_cast<int64_t>(p) * kBM * 4));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float w_in = in.x == -INFINITY ? 0.f : ex2f(in.x - M);
  float l = w_in * in.y, lo = w_in * in.z, acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  if (m.in_o != nullptr) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = w_in * __ldcg(m.in_o + row * D + lane * kPer + e);
  }
#pragma unroll 8
  for (int p = 0; p < m.pieces; ++p) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(ml + static_cast<int64_t>(p) * kBM * 4));
    const float* src = po + static_cast<int64_t>(p) * kBM * D;
    float o[kPer];
    if constexpr (kPer == 4) {
      const float4 f = __ldcg(reinterpret_cast<const float4*>(src));
      o[0] = f.x, o[1] = f.y, o[2] = f.z, o[3] = f.w;
    } else {
      const float2 f = __ldcg(reinterpret_cast<const float2*>(src));
      o[0] = f.x, o[1] = f.y;
    }
    const float w = v.x == -INFINITY ? 0.f : ex2f(v.x - M);
    l += w * v.y;
    lo += w * v.z;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] += w * o[e];
  }
  if (m.out_ml != nullptr) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) m.out_o[row * D + lane * kPer + e] = acc[e];
    if (lane == 0) *reinterpret_cast<float4*>(m.out_ml + row * 4) = make_float4(M, l, lo, 0.f);
    return;
  }
  const float inv = lo > 0.f ? 1.f / lo : 0.f;
  uint32_t* dst = reinterpret_cast<uint32_t*>(m.out + row * D + lane * kPer);
#pragma unroll
  for (int e = 0; e < kPer / 2; ++e) {
    const uint32_t w = pack2<BF16>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    dst[e] = w;
    if (x.out_lo != nullptr) {
      const float2 hi = unpack2<BF16>(w);
      reinterpret_cast<uint32_t*>(x.out_lo + row * D + lane * kPer)[e] =
          pack2<BF16>(fmaf(acc[2 * e], inv, -hi.x), fmaf(acc[2 * e + 1], inv, -hi.y));
    }
  }
  if (m.lse != nullptr && lane == 0) m.lse[row] = l != 0.f ? (M + log2f(l)) * kLn2 : -FLT_MAX;
}

__global__ void __launch_bounds__(256) fill_kernel(float* x, int64_t n, float v) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) x[i] = v;
}

// ---------------------------------------------------------------- host side
// Pieces of the keys per item: units run in rounds of `chains`; a unit costs
// its key tiles and a start, epilogue and merge worth about kUnitTiles.
constexpr int kUnitTiles = 5;
int choose_pieces(int64_t items, int64_t tiles, int64_t chains, bool merge_anyway) {
  int best = 1;
  double best_cost = 0.0;
  const int64_t most = std::min<int64_t>(255, tiles / 2);
  for (int64_t pc = 1; pc <= std::max<int64_t>(most, 1); ++pc) {
    const double rounds = static_cast<double>((items * pc + chains - 1) / chains);
    const double unit = static_cast<double>((tiles + pc - 1) / pc) + kUnitTiles + (pc > 1 && !merge_anyway ? 2 : 0);
    if (pc == 1 || rounds * unit < best_cost * 0.98) {
      best = static_cast<int>(pc);
      best_cost = rounds * unit;
    }
  }
  return best;
}

// The keys of one launch: k and v with their strides {batch, head, row}.
struct Keys {
  const void* k;
  const void* v;
  const int64_t* k_stride;
  const int64_t* v_stride;
  int64_t n;
  bool shared;  // one batch's keys, read by all
};

struct Partial {
  float* ml = nullptr;
  float* o = nullptr;
};

template <int D, bool BF16, bool kSplitK, bool kBias>
int launch(const CrossParams& p, const Keys& keys, Geo x, int pieces, Partial in, Partial out, const char** msg) {
  using C = ChainCfg<D>;
  constexpr size_t kSmemBytes = smem_bytes<D>();
  const int64_t W = (keys.n + 127) / 128 * 4;
  const int64_t KT = x.KTp + (keys.n + C::kBN - 1) / C::kBN;
  const int64_t QT = (p.Nq + kBM - 1) / kBM;
  const int64_t groups = (p.B + x.nb - 1) / x.nb * p.Hkv * x.gh;
  const int64_t total = QT * groups * pieces;
  const int64_t rows = p.B * p.H * p.Nq;
  if (total > 0x3FFFFFFFll || rows > (int64_t{0x7FFFFFFF} * kMergeWarps)) {
    *msg = "attention: too many query rows";
    return kErrArg;
  }
  CUtensorMap mq, mk, mv, mo;
  const int64_t so[3] = {p.H * p.Nq * D, p.Nq * D, D};
  const int64_t kb = keys.shared ? 1 : p.B;
  CUresult rc = make_tensor_map_4d(&mq, p.q, p.dtype, D, p.Nq, p.H, p.B, p.q_stride, x.tn, x.hb, x.nb);
  if (rc == CUDA_SUCCESS && keys.n > 0) {
    rc = make_tensor_map_4d(&mk, keys.k, p.dtype, D, keys.n, p.Hkv, kb, keys.k_stride, C::kBN);
    if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mv, keys.v, p.dtype, D, keys.n, p.Hkv, kb, keys.v_stride, C::kBN);
  }
  if (rc == CUDA_SUCCESS && x.KTp > 0) {
    const int64_t ks[3] = {0, p.kp_stride[0], p.kp_stride[1]}, vs[3] = {0, p.vp_stride[0], p.vp_stride[1]};
    rc = make_tensor_map_4d(&x.tm_kp, p.k_prefix, p.dtype, D, p.P, p.Hkv, 1, ks, C::kBN);
    if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&x.tm_vp, p.v_prefix, p.dtype, D, p.P, p.Hkv, 1, vs, C::kBN);
    if (keys.n == 0) mk = x.tm_kp, mv = x.tm_vp;  // not used: no tile of its own
  }
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mo, p.out, p.dtype, D, p.Nq, p.H, p.B, so, x.tn, x.hb, x.nb);
  if (rc != CUDA_SUCCESS) {
    *msg = tensor_map_error("attention", rc);
    return kErrCuda;
  }
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
  static std::atomic<bool> smem_set[kMaxDevices] = {};
  auto kern = attn_fwd_chain_kernel<D, BF16, false, kSplitK, true, kBias>;
  cudaError_t e = ensure_smem_limit(kern, kSmemBytes, dp.device, smem_set);
  const int o_wide = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0 ? 1 : 0;
  // As for the square kernel: head-major once K and V exceed half of L2.
  const int head_major = 2 * kb * p.Hkv * keys.n * D * 2 > dp.l2_bytes / 2 ? 1 : 0;
  const int grid = static_cast<int>(total < dp.sms ? total : dp.sms);
  SplitParams sp{};
  void* ws = nullptr;
  if constexpr (kSplitK) {
    if (e == cudaSuccess)
      e = scratch_alloc_async(&ws, static_cast<size_t>(total) * kBM * (4 + D) * sizeof(float), p.stream);
    sp.pieces = pieces;
    sp.ws = static_cast<float*>(ws);
  }
  if (e == cudaSuccess)
    e = launch_pdl(kern, static_cast<unsigned>(grid), kThreads, kSmemBytes, p.stream, mq, mk, mv, mo,
                   static_cast<uint16_t*>(p.out), nullptr, nullptr, nullptr, nullptr, p.lse,
                   static_cast<int>(keys.n), static_cast<int>(groups), static_cast<int>(W), static_cast<int>(KT),
                   static_cast<int>(total), 1, o_wide, head_major, 0, p.scale * kLog2e, sp, x, p.err_word,
                   p.timeout_ns);
  if (kSplitK && e == cudaSuccess) {
    MergeParams m{};
    m.ws = sp.ws;
    m.units = total;
    m.pieces = pieces;
    m.groups = static_cast<int>(groups);
    m.QT = static_cast<int>(QT);
    m.head_major = head_major;
    m.in_ml = in.ml;
    m.in_o = in.o;
    m.out_ml = out.ml;
    m.out_o = out.o;
    m.out = static_cast<uint16_t*>(p.out);
    m.lse = p.lse;
    m.rows = rows;
    e = launch_pdl(merge_rows_kernel<D, BF16>, static_cast<unsigned>((rows + kMergeWarps - 1) / kMergeWarps),
                   kMergeWarps * 32, 0, p.stream, m, x);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  if (ws != nullptr) {
    const cudaError_t ef = cudaFreeAsync(ws, p.stream);
    if (e == cudaSuccess) e = ef;
  }
  if (e != cudaSuccess) {
    *msg = cudaGetErrorString(e);
    return kErrLaunch;
  }
  return kOk;
}

// The rows of a tile.
Geo tile_geometry(const CrossParams& p, bool shared_keys) {
  Geo x{};
  x.B = static_cast<int>(p.B);
  x.H = static_cast<int>(p.H);
  x.Hkv = static_cast<int>(p.Hkv);
  x.Nq = static_cast<int>(p.Nq);
  const int G = static_cast<int>(p.H / p.Hkv);
  x.tn = std::min<int>(x.Nq, kBM);
  for (int h = 1; h <= G; ++h)
    if (G % h == 0 && h * x.tn <= kBM) x.hb = h;
  x.gh = G / x.hb;
  x.nb = shared_keys ? std::max(1, std::min<int>(x.B, kBM / (x.tn * x.hb))) : 1;
  x.rows = x.tn * x.hb * x.nb;
  return x;
}

// The packed mask of p: its words, the kept keys of every tile, and the
// live-tile bits, one behind the other.
struct PackLayout {
  int64_t words, kept;   // numbers of words
  int64_t Bm, Hm, Qm;    // lengths of the axes the mask has, 1 for the others
  int64_t Hb, QT;        // head blocks and query tiles it has
  int64_t occ_words;
};
PackLayout pack_layout(const CrossParams& p, const Geo& x) {
  PackLayout l{};
  l.Bm = p.word_stride[0] != 0 ? p.B : 1;
  l.Hm = p.word_stride[1] != 0 ? p.H : 1;
  l.Qm = p.word_stride[2] != 0 ? p.Nq : 1;
  l.words = l.Bm * l.Hm * l.Qm * ((p.Nk + 127) / 128 * 4);
  l.Hb = p.word_stride[1] != 0 ? p.H / x.hb : 1;
  l.QT = p.word_stride[2] != 0 ? (p.Nq + kBM - 1) / kBM : 1;
  l.kept = l.Bm * l.Hb * l.QT * ((p.Nk + 127) / 128 * 4);
  const int64_t bn = p.D == 64 ? 128 : 64;
  l.occ_words = ((p.Nk + bn - 1) / bn + 31) / 32;
  return l;
}

// Packs p's mask and lays its bias out, as far as it has them.
int launch_layout(const CrossParams& p, const char** msg) {
  ExpandParams ex{};
  if (p.bias.table != nullptr) {
    int hi = 0;
    ex.bias = p.bias;
    ex.bf16 = p.dtype;
    bias_range(p.bias, &ex.lo, &hi);
    ex.len = hi - ex.lo + 1 + 2 * kBiasPad;
    ex.stride = bias_stride(ex.len);
    ex.out = p.bias_distance;
    ex.head_blocks = static_cast<int>(std::min<int64_t>(p.H, 1024));
    ex.blocks = static_cast<int>((ex.stride / 16 + 63) / 64) * ex.head_blocks;
  }
  if (p.mask == nullptr && ex.blocks == 0) return kOk;
  const Geo x = tile_geometry(p, false);
  PackParams k{};
  int64_t blocks = 0;
  bool aligned = true;
  if (p.mask != nullptr) {
    const PackLayout l = pack_layout(p, x);
    k.mask = p.mask;
    k.sb = p.mask_stride[0];
    k.sh = p.mask_stride[1];
    k.sq = p.mask_stride[2];
    k.hi = p.mask + (l.Bm - 1) * k.sb + (l.Hm - 1) * k.sh + (l.Qm - 1) * k.sq + p.Nk;
    k.words = p.words;
    k.kept = p.words + l.words;
    k.occ = reinterpret_cast<uint8_t*>(p.words + l.words + l.kept);
    k.Hm = static_cast<int>(l.Hm);
    k.Qm = static_cast<int>(l.Qm);
    k.Nk = static_cast<int>(p.Nk);
    k.W = static_cast<int>((p.Nk + 127) / 128 * 4);
    k.hb = p.word_stride[1] != 0 ? x.hb : 1;
    k.tn = p.word_stride[2] != 0 ? x.tn : 1;
    k.rows = k.hb * k.tn;
    k.Hb = static_cast<int>(l.Hb);
    k.QT = static_cast<int>(l.QT);
    k.occ_words = static_cast<int>(l.occ_words);
    k.tile_log2 = p.D == 64 ? 2 : 1;
    // The longest stretch (fewest CTAs) that still gives every SM a few CTAs; 8
    // key tiles at least.
    DeviceProps dp;
    if (!device_props(&dp, msg)) return kErrCuda;
    const int64_t tiles = l.Bm * l.Hb * l.QT;
    k.chunk_log2 = 8;
    while (k.chunk_log2 > k.tile_log2 + 3 && tiles * (((k.W - 1) >> k.chunk_log2) + 1) < 6 * dp.sms) --k.chunk_log2;
    while ((1 << (k.chunk_log2 - 1)) >= k.W) --k.chunk_log2;
    k.chunks = ((k.W - 1) >> k.chunk_log2) + 1;
    blocks = tiles * k.chunks;
    if (blocks > 0x7FFFFFFFll - ex.blocks) {
      *msg = "attention: mask too large";
      return kErrArg;
    }
    aligned = ((reinterpret_cast<uintptr_t>(p.mask) | k.sb | k.sh | k.sq) & 15) == 0;
  }
  const cudaError_t e = launch_pdl(aligned ? pack_tiles_kernel<true> : pack_tiles_kernel<false>,
                                   static_cast<unsigned>(ex.blocks + blocks), kPackThreads, 0, p.stream, k, ex);
  if (e != cudaSuccess) {
    *msg = cudaGetErrorString(e);
    return kErrLaunch;
  }
  return kOk;
}

// One launch over `keys`.  `partial`: takes in / leaves a piece of every row
// (always the split kernel, whose merge does that).  `with_prefix`: p's prefix
// stands in front of the keys.
int launch_tiles(const CrossParams& p, const Keys& keys, bool with_prefix, bool partial, Partial in, Partial out,
                 const char** msg) {
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
  Geo x = tile_geometry(p, keys.shared);
  x.kv_shared = keys.shared ? 1 : 0;
  x.out_lo = static_cast<uint16_t*>(p.out_lo);
  if (!keys.shared) {
    x.words = p.words;
    for (int i = 0; i < 3; ++i) x.word_stride[i] = p.word_stride[i];
    if (p.words != nullptr) {
      const int64_t W = (p.Nk + 127) / 128 * 4;
      const PackLayout l = pack_layout(p, x);
      x.kept = p.words + l.words;
      x.occ = p.words + l.words + l.kept;
      const int64_t tiles[3] = {l.QT * l.Hb, l.QT, 1};
      for (int i = 0; i < 3; ++i) {
        x.occ_stride[i] = p.word_stride[i] != 0 ? tiles[i] * l.occ_words : 0;
        x.kept_stride[i] = p.word_stride[i] != 0 ? tiles[i] * W : 0;
      }
    }
    x.lengths = p.lengths;
  }
  const int bn = p.D == 64 ? 128 : 64;
  if (with_prefix) {
    x.P = static_cast<int>(p.P);
    x.KTp = (x.P + bn - 1) / bn;
  }
  const bool bias = p.bias.table != nullptr;
  if (bias) {
    x.bias = p.bias_distance;
    x.bias_offsets = p.bias.offsets;
    x.bias_offset = p.bias.offset;
    bias_range(p.bias, &x.bias_lo, &x.bias_hi);
    x.bias_len = x.bias_hi - x.bias_lo + 1 + 2 * kBiasPad;
    x.bias_stride = bias_stride(x.bias_len);
  }
  const int64_t items = (p.B + x.nb - 1) / x.nb * p.Hkv * x.gh * ((p.Nq + kBM - 1) / kBM);
  const int pieces = choose_pieces(items, x.KTp + (keys.n + bn - 1) / bn, 2 * static_cast<int64_t>(dp.sms), partial);
  const bool split = partial || pieces > 1;
#define SMA_LAUNCH(D_, BF_)                                                            \
  (split ? (bias ? launch<D_, BF_, true, true>(p, keys, x, pieces, in, out, msg)       \
                 : launch<D_, BF_, true, false>(p, keys, x, pieces, in, out, msg))     \
         : (bias ? launch<D_, BF_, false, true>(p, keys, x, 1, in, out, msg)           \
                 : launch<D_, BF_, false, false>(p, keys, x, 1, in, out, msg)))
  if (p.D == 128) return p.dtype == 1 ? SMA_LAUNCH(128, true) : SMA_LAUNCH(128, false);
  return p.dtype == 1 ? SMA_LAUNCH(64, true) : SMA_LAUNCH(64, false);
#undef SMA_LAUNCH
}

}  // namespace

int launch_fill(float* x, int64_t n, float v, cudaStream_t stream) {
  if (n <= 0) return kOk;
  fill_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(x, n, v);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

int launch_attn_cross(const CrossParams& p, const char** msg) {
  const int rc = launch_layout(p, msg);
  if (rc != kOk) return rc;
  const Keys keys{p.k, p.v, p.k_stride, p.v_stride, p.Nk, false};
  return launch_tiles(p, keys, false, false, {}, {}, msg);
}

// Three ways, by their cost in us (measured on a B200, see below):
//   rows    the streaming kernel, prefix and own keys per 16 rows: little
//           work, or little to share;
//   tiles   128-row tiles, prefix and own keys in one pass per sequence: the
//           rows of one sequence fill most of a tile;
//   shared  the prefix once for the batch: the sequences' own keys leave a
//           piece of every row (FP32), then the prefix is attended with the
//           rows of several sequences in one tile, and its merge takes those
//           pieces in.
// rows: 8 + 1 per 8.5 MB of keys streamed (from L2 where the prefix is read
// again): B16 Hkv8 P1024 D128 17.1 (shared: 21.1), P4096 39.7 (31.0).  The two
// others: 23 + 7.3 ns (D = 64) or 12.5 ns per 128 x 128 tile, and for `shared`
// the own keys streamed at 6 MB per us (one tile of 16 rows) or 8 us for one
// more launch of tiles: B64 Hkv8 G4 P256 D128 23.1 (rows: 17.4), P1024
// with S256 30.7 (43.5).
int launch_shared_prefix(const CrossParams& p, const char** msg) {
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
  const int64_t rows = p.B * p.H * p.Nq;
  const int64_t group_rows = p.H / p.Hkv * p.Nq;
  const Keys own_keys{p.k, p.v, p.k_stride, p.v_stride, p.Nk, false};
  const int64_t bn = p.D == 64 ? 128 : 64;
  const int64_t own_tiles = (p.Nk + bn - 1) / bn, prefix_tiles = (p.P + bn - 1) / bn;
  {
    const Geo once = tile_geometry(p, true), own = tile_geometry(p, false);
    const double heads = static_cast<double>(p.B * p.Hkv), ns = p.D == 64 ? 7.3e-3 : 12.5e-3;
    const double q_tiles = static_cast<double>((p.Nq + kBM - 1) / kBM);
    const double per_key = 4.0 * static_cast<double>(p.D) * 1e-6;  // MB of K and V
    const double rows_us = 8.0 + heads * static_cast<double>((group_rows + kRowsTile - 1) / kRowsTile) *
                                     static_cast<double>(p.P + p.Nk) * per_key / 8.5;
    const double tile_us = ns * q_tiles * static_cast<double>(bn) / 128.0;  // per group and key tile
    const double own_us = heads * own.gh * tile_us * static_cast<double>(own_tiles);
    const double tiles_us = 23.0 + own_us + heads * own.gh * tile_us * static_cast<double>(prefix_tiles);
    const double shared_us = 23.0 + static_cast<double>((p.B + once.nb - 1) / once.nb * p.Hkv) * once.gh * tile_us *
                                        static_cast<double>(prefix_tiles) +
                             (group_rows <= kRowsTile ? heads * static_cast<double>(p.Nk) * per_key / 6.0 : 8.0 + own_us);
    if (rows_us <= tiles_us && rows_us <= shared_us) return launch_attn_rows(p, msg);
    if (tiles_us <= shared_us && own_tiles + prefix_tiles <= kMaxSeqLen / bn)
      return launch_tiles(p, own_keys, true, false, {}, {}, msg);
  }
  void* ws = nullptr;
  Partial part;
  int rc = kOk;
  if (p.Nk > 0 || p.P > kMaxSeqLen) {
    const cudaError_t e = scratch_alloc_async(&ws, static_cast<size_t>(rows) * (4 + p.D) * sizeof(float), p.stream);
    if (e != cudaSuccess) {
      *msg = cudaGetErrorString(e);
      return kErrCuda;
    }
    part.ml = static_cast<float*>(ws);
    part.o = part.ml + rows * 4;
  }
  if (p.Nk > 0) {
    CrossParams own = p;
    own.P = 0;
    if (group_rows <= kRowsTile) {
      own.part_ml = part.ml;
      own.part_o = part.o;
      rc = launch_attn_rows(own, msg);
    } else {
      rc = launch_tiles(own, own_keys, false, true, {}, part, msg);
    }
  }
  // A prefix longer than a launch's live-tile lists cover goes in stretches.
  for (int64_t at = 0; rc == kOk && at < p.P; at += kMaxSeqLen) {
    const int64_t n = std::min<int64_t>(p.P - at, kMaxSeqLen);
    const int64_t ks[3] = {0, p.kp_stride[0], p.kp_stride[1]}, vs[3] = {0, p.vp_stride[0], p.vp_stride[1]};
    const Keys keys{static_cast<const uint16_t*>(p.k_prefix) + at * ks[2],
                    static_cast<const uint16_t*>(p.v_prefix) + at * vs[2], ks, vs, n, true};
    const bool last = at + n == p.P;
    rc = launch_tiles(p, keys, false, true, at > 0 || p.Nk > 0 ? part : Partial{}, last ? Partial{} : part, msg);
  }
  if (ws != nullptr) {
    const cudaError_t ef = cudaFreeAsync(ws, p.stream);
    if (rc == kOk && ef != cudaSuccess) {
      *msg = cudaGetErrorString(ef);
      rc = kErrCuda;
    }
  }
  return rc;
}

}  // namespace sma
