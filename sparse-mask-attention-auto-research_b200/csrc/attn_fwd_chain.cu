// Host side of the square attention forward (q, k, v and out [B, H, N, D]): the
// kernel is in attn_fwd_chain.cuh.
#include "attn_fwd_chain.cuh"

namespace sma {
namespace {

// ---------------------------------------------------------------- host side

template <int D, bool BF16, bool kBoolIn, bool kSplitK>
int launch(const AttnParams& p, int pieces, const char** msg) {
  using C = ChainCfg<D>;
  constexpr size_t kSmemBytes = smem_bytes<D>();
  const int64_t BH = p.B * p.H;
  const int64_t N = p.N;
  const int64_t W = (N + 31) / 32;
  const int64_t KT = (N + C::kBN - 1) / C::kBN;
  const int64_t QT = (N + kBM - 1) / kBM;
  const int64_t items = QT * BH;
  const int64_t total = kSplitK ? items * pieces : items;  // work units
  if (total > 0x3FFFFFFFll) {
    *msg = "attention: batch*heads too large";
    return kErrArg;
  }
  CUtensorMap mq, mk, mv, mo;
  CUresult rc = make_tensor_map_3d(&mq, p.q, p.dtype, D, BH, N, kBM);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_3d(&mk, p.k, p.dtype, D, BH, N, C::kBN);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_3d(&mv, p.v, p.dtype, D, BH, N, C::kBN);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_3d(&mo, p.out, p.dtype, D, BH, N, kBM);
  if (rc != CUDA_SUCCESS) {
    *msg = tensor_map_error("attention", rc);
    return kErrCuda;
  }
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
  static std::atomic<bool> smem_set[kMaxDevices] = {};
  auto kern = attn_fwd_chain_kernel<D, BF16, kBoolIn, kSplitK, false, false>;
  {
    cudaError_t e = ensure_smem_limit(kern, kSmemBytes, dp.device, smem_set);
    if (e != cudaSuccess) {
      *msg = cudaGetErrorString(e);
      return kErrLaunch;
    }
  }
  // Bool input: the kernel packs into p.packed_out and reads its words back.
  const uint32_t* words = kBoolIn ? p.packed_out : p.mask;
  const int vec = (W % 4 == 0 && (reinterpret_cast<uintptr_t>(words) & 15u) == 0) ? 1 : 0;
  const int o_wide = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0 ? 1 : 0;  // 32-byte O stores (D = 128)
  // Head-major item order once K and V of all heads exceed half of L2.
  const int head_major = 2 * BH * N * D * 2 > dp.l2_bytes / 2 ? 1 : 0;
  const int grid = static_cast<int>(total < dp.sms ? total : dp.sms);
  // The occupancy map describes 128-key tiles: only the D = 64 kernel uses it.
  const uint32_t* occ = (D == 64 && !kBoolIn) ? p.occ : nullptr;
  // Bool input: item i+2's bool rows are prefetched into L2 when item i
  // starts if two rounds of items' rows (2 chains per CTA) take at most 48
  // MB of L2, else at item i's last tile.
  const int pf_early = 2 * static_cast<int64_t>(grid) * 2 * kBM * N <= (int64_t{48} << 20) ? 1 : 0;
  SplitParams sp{};
  void* ws = nullptr;
  if constexpr (kSplitK) {
    // Counters (one per item), then (max, sums) and the FP32 O of every unit.
    const size_t cnt_bytes = (static_cast<size_t>(items) * 8 + 255) / 256 * 256;
    const size_t rows = static_cast<size_t>(total) * kBM;
    cudaError_t ea = scratch_alloc_async(&ws, cnt_bytes + rows * (4 + D) * sizeof(float), p.stream);
    if (ea != cudaSuccess) {
      *msg = cudaGetErrorString(ea);
      return kErrCuda;
    }
    sp.pieces = pieces;
    sp.cnt = static_cast<unsigned long long*>(ws);
    sp.ws = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + cnt_bytes);
    sp.epoch = next_launch_epoch();
  }
  cudaError_t e = launch_pdl(kern, static_cast<unsigned>(grid), kThreads, kSmemBytes, p.stream, mq, mk, mv, mo,
                             static_cast<uint16_t*>(p.out), kBoolIn ? nullptr : p.mask, kBoolIn ? p.bmask : nullptr,
                             kBoolIn ? p.packed_out : nullptr, occ, p.lse, static_cast<int>(N), static_cast<int>(BH),
                             static_cast<int>(W), static_cast<int>(KT), static_cast<int>(total), vec, o_wide,
                             head_major, pf_early, p.scale * kLog2e, sp, NoGeo{}, p.err_word, p.timeout_ns);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (ws != nullptr) {
    cudaError_t ef = cudaFreeAsync(ws, p.stream);
    if (e == cudaSuccess) e = ef;
  }
  if (e != cudaSuccess) {
    static thread_local char buf[256];
    cudaFuncAttributes fa{};
    cudaFuncGetAttributes(&fa, kern);
    snprintf(buf, sizeof(buf), "%s (chain kernel: %d threads, %d regs/thread, max %d threads/block, %zu B dynamic smem)",
             cudaGetErrorString(e), kThreads, fa.numRegs, fa.maxThreadsPerBlock, kSmemBytes);
    *msg = buf;
    return kErrLaunch;
  }
  return kOk;
}

}  // namespace

bool chain_supported(const AttnParams& p) {
  return (p.D == 64 && p.N <= ChainCfg<64>::kMaxN) || (p.D == 128 && p.N <= ChainCfg<128>::kMaxN);
}

template <bool kBoolIn>
int launch_any(const AttnParams& p, int pieces, const char** msg) {
  if (pieces >= 2) {
    if (p.D == 128)
      return p.dtype == 1 ? launch<128, true, kBoolIn, true>(p, pieces, msg) : launch<128, false, kBoolIn, true>(p, pieces, msg);
    return p.dtype == 1 ? launch<64, true, kBoolIn, true>(p, pieces, msg) : launch<64, false, kBoolIn, true>(p, pieces, msg);
  }
  if (p.D == 128)
    return p.dtype == 1 ? launch<128, true, kBoolIn, false>(p, 1, msg) : launch<128, false, kBoolIn, false>(p, 1, msg);
  return p.dtype == 1 ? launch<64, true, kBoolIn, false>(p, 1, msg) : launch<64, false, kBoolIn, false>(p, 1, msg);
}

int launch_attn_fwd_chain(const AttnParams& p, const char** msg) {
  // Split along keys when the items (batch*head x 128-row query tiles) leave
  // chains idle and are long: as many pieces per item as fill the chains,
  // each of at least kSplitMinTiles key tiles (shorter pieces lose to the
  // merge and the per-unit fixed costs).
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
  const int64_t items = (p.N + kBM - 1) / kBM * p.B * p.H;
  const int64_t kt = p.D == 64 ? (p.N + 127) / 128 : (p.N + 63) / 64;
  const int64_t chains = 2 * static_cast<int64_t>(dp.sms);
  int pieces = 1;
  if (items > 0 && items < chains)
    pieces = static_cast<int>(std::min<int64_t>({kt / kSplitMinTiles, chains / items, 255}));
  return p.bmask != nullptr ? launch_any<true>(p, pieces, msg) : launch_any<false>(p, pieces, msg);
}

}  // namespace sma
