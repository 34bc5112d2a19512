// Attention forward of queries and keys of different lengths on the two-chain
// kernel (attn_fwd_chain.cuh, kX): its mask packer, the bias laid out by
// relative position, and the host side.
#include "attn_fwd_chain.cuh"

namespace sma {
namespace {

// ---------------------------------------------------------------- mask packer
// bool bytes with any batch / head / query strides -> words [Bm, Hm, Qm, W],
// W = 4 ceil(Nk / 128) (whole 128-key tiles; bits at columns >= Nk are 0).
// One thread per word.  A word's 32 bytes start at any address: the aligned
// 16-byte vectors that cover them are packed to bits first, and the bits are
// shifted into place.  Bound by HBM: every mask byte is read once (a vector
// shared by two words the second time from L1).  Vectors that would reach
// outside the mask's own span [lo, hi) are read byte by byte.
constexpr int kPackThreads = 256;
constexpr int kPackRounds = 4;

__device__ __forceinline__ uint32_t pack_word(const uint8_t* a, const uint8_t* lo, const uint8_t* hi, int valid) {
  const uint32_t keep = valid >= 32 ? 0xFFFFFFFFu : (1u << valid) - 1u;
  const int sh = static_cast<int>(reinterpret_cast<uintptr_t>(a) & 15u);
  const uint8_t* v = a - sh;
  const int bytes = sh == 0 ? 32 : 48;
  if (v >= lo && v + bytes <= hi) {
    const uint4* p = reinterpret_cast<const uint4*>(v);
    unsigned long long bits = pack16_any(__ldg(p)) | (pack16_any(__ldg(p + 1)) << 16);
    if (sh != 0) bits |= static_cast<unsigned long long>(pack16_any(__ldg(p + 2))) << 32;
    return static_cast<uint32_t>(bits >> sh) & keep;
  }
  uint32_t w = 0u;
  for (int i = 0; i < min(valid, 32); ++i) w |= (a[i] != 0 ? 1u : 0u) << i;
  return w;
}

__global__ void __launch_bounds__(kPackThreads)
    pack_rows_kernel(const uint8_t* __restrict__ mask, const uint8_t* hi, uint32_t* __restrict__ words, int64_t sb,
                     int64_t sh, int64_t sq, int Hm, int Qm, int Nk, int W, int64_t total) {
  pdl_launch_dependents();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kPackThreads * kPackRounds) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kPackRounds; ++u) {
    const int64_t idx = first + u * kPackThreads;
    if (idx >= total) return;
    const int64_t row = idx / W;
    const int w = static_cast<int>(idx - row * W);
    const int64_t bh = row / Qm;
    const int q = static_cast<int>(row - bh * Qm);
    const int64_t b = bh / Hm;
    const int64_t h = bh - b * Hm;
    const int valid = Nk - 32 * w;
    words[idx] = valid > 0 ? pack_word(mask + b * sb + h * sh + q * sq + 32 * w, mask, hi, valid) : 0u;
  }
}

// ---------------------------------------------------------------- bias by relative position
// out[h][i] = log2(e) * table[bucket(lo - kBiasPad + i)][h]: the attention
// kernels read the bias of 128 consecutive keys from 128 consecutive floats.
__global__ void __launch_bounds__(256)
    bias_expand_kernel(const __grid_constant__ BiasSpec bias, int bf16, int lo, int len, float* __restrict__ out) {
  __shared__ int starts[kMaxBiasSide];
  for (int i = threadIdx.x; i < bias.side; i += 256) starts[i] = bias.starts[i];
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= len) return;
  const int bucket = bias_bucket(bias, starts, lo - kBiasPad + i);
  for (int h = blockIdx.y; h < bias.H; h += gridDim.y)
    out[static_cast<int64_t>(h) * len + i] =
        kLog2e * (bf16 ? bias_value<true>(bias, bucket, h) : bias_value<false>(bias, bucket, h));
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
int launch(const CrossParams& p, const Keys& keys, const Geo& x, int pieces, Partial in, Partial out, const char** msg) {
  using C = ChainCfg<D>;
  constexpr size_t kSmemBytes = smem_bytes<D>();
  const int64_t W = (keys.n + 127) / 128 * 4;
  const int64_t KT = (keys.n + C::kBN - 1) / C::kBN;
  const int64_t QT = (p.Nq + kBM - 1) / kBM;
  const int64_t groups = (p.B + x.nb - 1) / x.nb * p.Hkv * x.gh;
  const int64_t total = QT * groups * pieces;
  if (total > 0x3FFFFFFFll) {
    *msg = "attention: too many query rows";
    return kErrArg;
  }
  CUtensorMap mq, mk, mv, mo;
  const int64_t so[3] = {p.H * p.Nq * D, p.Nq * D, D};
  const int64_t kb = keys.shared ? 1 : p.B;
  CUresult rc = make_tensor_map_4d(&mq, p.q, p.dtype, D, p.Nq, p.H, p.B, p.q_stride, x.tn, x.hb, x.nb);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mk, keys.k, p.dtype, D, keys.n, p.Hkv, kb, keys.k_stride, C::kBN);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mv, keys.v, p.dtype, D, keys.n, p.Hkv, kb, keys.v_stride, C::kBN);
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
  SplitParamsX sp{};
  void* ws = nullptr;
  if constexpr (kSplitK) {
    const size_t cnt_bytes = (static_cast<size_t>(total / pieces) * 8 + 255) / 256 * 256;
    const size_t rows = static_cast<size_t>(total) * kBM;
    if (e == cudaSuccess) e = scratch_alloc_async(&ws, cnt_bytes + rows * (4 + D) * sizeof(float), p.stream);
    sp.pieces = pieces;
    sp.cnt = static_cast<unsigned long long*>(ws);
    sp.ws = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + cnt_bytes);
    sp.epoch = next_launch_epoch();
    sp.in_ml = in.ml;
    sp.in_o = in.o;
    sp.out_ml = out.ml;
    sp.out_o = out.o;
  }
  if (e == cudaSuccess)
    e = launch_pdl(kern, static_cast<unsigned>(grid), kThreads, kSmemBytes, p.stream, mq, mk, mv, mo,
                   static_cast<uint16_t*>(p.out), nullptr, nullptr, nullptr, nullptr, p.lse,
                   static_cast<int>(keys.n), static_cast<int>(groups), static_cast<int>(W), static_cast<int>(KT),
                   static_cast<int>(total), 1, o_wide, head_major, 0, p.scale * kLog2e, sp, x, p.err_word,
                   p.timeout_ns);
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

// One launch over `keys`.  `partial`: takes in / leaves a piece of every row
// (always the split kernel, which merges).
int launch_tiles(const CrossParams& p, const Keys& keys, bool partial, Partial in, Partial out, const char** msg) {
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
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
  x.nb = keys.shared ? std::max(1, std::min<int>(x.B, kBM / (x.tn * x.hb))) : 1;
  x.rows = x.tn * x.hb * x.nb;
  x.kv_shared = keys.shared ? 1 : 0;
  if (!keys.shared) {
    x.words = p.words;
    for (int i = 0; i < 3; ++i) x.word_stride[i] = p.word_stride[i];
    x.row_shared = p.words != nullptr && (x.Nq == 1 || p.word_stride[2] == 0) && (x.hb == 1 || p.word_stride[1] == 0);
    x.lengths = p.lengths;
  }
  const bool bias = p.bias.table != nullptr;
  if (bias) {
    x.bias = p.bias_distance;
    x.bias_offsets = p.bias.offsets;
    x.bias_offset = p.bias.offset;
    bias_range(p.bias, &x.bias_lo, &x.bias_hi);
    x.bias_len = x.bias_hi - x.bias_lo + 1 + 2 * kBiasPad;
  }
  const int bn = p.D == 64 ? 128 : 64;
  const int64_t items = (p.B + x.nb - 1) / x.nb * p.Hkv * x.gh * ((p.Nq + kBM - 1) / kBM);
  const int pieces = choose_pieces(items, (keys.n + bn - 1) / bn, 2 * static_cast<int64_t>(dp.sms), partial);
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

int launch_pack_rows(const uint8_t* mask, const int64_t* stride, uint32_t* words, int64_t Bm, int64_t Hm, int64_t Qm,
                     int64_t Nk, cudaStream_t stream, const char** msg) {
  const int64_t W = (Nk + 127) / 128 * 4;
  const int64_t total = Bm * Hm * Qm * W;
  if (total == 0) return kOk;
  const int64_t blocks = (total + kPackThreads * kPackRounds - 1) / (kPackThreads * kPackRounds);
  if (blocks > 0x7FFFFFFFll) {
    *msg = "pack_mask: input too large";
    return kErrArg;
  }
  const uint8_t* hi = mask + (Bm - 1) * stride[0] + (Hm - 1) * stride[1] + (Qm - 1) * stride[2] + Nk;
  pack_rows_kernel<<<static_cast<unsigned>(blocks), kPackThreads, 0, stream>>>(
      mask, hi, words, stride[0], stride[1], stride[2], static_cast<int>(Hm), static_cast<int>(Qm),
      static_cast<int>(Nk), static_cast<int>(W), total);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    *msg = cudaGetErrorString(e);
    return kErrLaunch;
  }
  return kOk;
}

int launch_fill(float* x, int64_t n, float v, cudaStream_t stream) {
  if (n <= 0) return kOk;
  fill_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(x, n, v);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

int launch_bias_expand(const CrossParams& p, const char** msg) {
  int lo = 0, hi = 0;
  bias_range(p.bias, &lo, &hi);
  const int len = hi - lo + 1 + 2 * kBiasPad;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((len + 255) / 256), static_cast<unsigned>(std::min<int64_t>(p.H, 1024)));
  cfg.blockDim = dim3(256);
  cfg.stream = p.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, bias_expand_kernel, p.bias, p.dtype, lo, len, p.bias_distance);
  if (e != cudaSuccess) {
    *msg = cudaGetErrorString(e);
    return kErrLaunch;
  }
  return kOk;
}

int launch_attn_cross(const CrossParams& p, const char** msg) {
  if (p.bias.table != nullptr) {
    const int rc = launch_bias_expand(p, msg);
    if (rc != kOk) return rc;
  }
  const Keys keys{p.k, p.v, p.k_stride, p.v_stride, p.Nk, false};
  return launch_tiles(p, keys, false, {}, {}, msg);
}

// Two launches: the sequences' own keys leave a piece of every row (FP32),
// then the prefix is attended once for the whole batch, the rows of several
// sequences in one tile, and its merge takes those pieces in.
int launch_shared_prefix(const CrossParams& p, const char** msg) {
  const int64_t rows = p.B * p.H * p.Nq;
  void* ws = nullptr;
  Partial part;
  int rc = kOk;
  if (p.Nk > 0) {
    const cudaError_t e = scratch_alloc_async(&ws, static_cast<size_t>(rows) * (4 + p.D) * sizeof(float), p.stream);
    if (e != cudaSuccess) {
      *msg = cudaGetErrorString(e);
      return kErrCuda;
    }
    part.ml = static_cast<float*>(ws);
    part.o = part.ml + rows * 4;
    CrossParams own = p;
    own.P = 0;
    own.lse = nullptr;
    if (p.H / p.Hkv * p.Nq <= kRowsTile) {
      own.part_ml = part.ml;
      own.part_o = part.o;
      rc = launch_attn_rows(own, msg);
    } else {
      const Keys keys{p.k, p.v, p.k_stride, p.v_stride, p.Nk, false};
      rc = launch_tiles(own, keys, true, {}, part, msg);
    }
  }
  // A prefix longer than a launch's live-tile lists cover goes in stretches.
  for (int64_t at = 0; rc == kOk && at < p.P; at += kMaxSeqLen) {
    const int64_t n = std::min<int64_t>(p.P - at, kMaxSeqLen);
    const int64_t ks[3] = {0, p.kp_stride[0], p.kp_stride[1]}, vs[3] = {0, p.vp_stride[0], p.vp_stride[1]};
    const Keys keys{static_cast<const uint16_t*>(p.k_prefix) + at * ks[2],
                    static_cast<const uint16_t*>(p.v_prefix) + at * vs[2], ks, vs, n, true};
    const bool last = at + n == p.P;
    if (!last && ws == nullptr) {
      *msg = "attention: prefix too long";
      rc = kErrUnsupportedN;
      break;
    }
    rc = launch_tiles(p, keys, true, part, last ? Partial{} : part, msg);
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
