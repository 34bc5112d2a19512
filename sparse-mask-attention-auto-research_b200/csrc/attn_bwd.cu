// Host side of the square attention backward: the kernels are in attn_bwd.cuh.
#include "attn_bwd.cuh"

namespace sma {
namespace {

template <int D, bool BF16>
int launch(const BwdParams& p, const char** msg) {
  using C = BwdCfg<D>;
  const int64_t BH = p.B * p.H;
  const int64_t N = p.N;
  const int64_t W = (N + 31) / 32;
  const int64_t KT = (N + kT - 1) / kT;
  const int64_t QT = (N + kT - 1) / kT;
  if (BH * KT > 0x7FFFFFFFll) {
    *msg = "backward: batch*heads too large";
    return kErrArg;
  }
  CUtensorMap mq, mk, mv, mdo, mdq;
  CUresult rc = make_tensor_map_3d(&mq, p.q, p.dtype, D, BH, N, kT);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_3d(&mk, p.k, p.dtype, D, BH, N, kT);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_3d(&mv, p.v, p.dtype, D, BH, N, kT);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_3d(&mdo, p.dout, p.dtype, D, BH, N, kT);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_3d_f32(&mdq, p.dq_accum, D, BH, N, 32);
  if (rc != CUDA_SUCCESS) {
    *msg = tensor_map_error("backward", rc);
    return kErrCuda;
  }
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
  static std::atomic<bool> smem_set[kMaxDevices] = {};
  auto kern = attn_bwd_kernel<D, BF16, false, false>;
  {
    cudaError_t e = ensure_smem_limit(kern, C::kSmemBytes, dp.device, smem_set);
    if (e != cudaSuccess) {
      *msg = cudaGetErrorString(e);
      return kErrLaunch;
    }
  }
  const int64_t rows = BH * N;
  bwd_delta_kernel<D, BF16><<<static_cast<unsigned>((rows * (D / 8) + 255) / 256), 256, 0, p.stream>>>(
      static_cast<const uint4*>(p.dout), static_cast<const uint4*>(p.out), p.delta,
      reinterpret_cast<float4*>(p.dq_accum), rows);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) {
    const int vec = (W % 4 == 0 && (reinterpret_cast<uintptr_t>(p.mask) & 15u) == 0) ? 1 : 0;
    // One CTA per SM (over half of its shared memory and all 512 TMEM columns each).
    const int64_t items = BH * KT;
    const int64_t grid = items < dp.sms ? items : dp.sms;
    kern<<<static_cast<unsigned>(grid), C::kThreads, C::kSmemBytes, p.stream>>>(
        mq, mk, mv, mdo, mdq, p.mask, p.lse, p.delta, static_cast<uint16_t*>(p.dk),
        static_cast<uint16_t*>(p.dv), static_cast<int>(N), static_cast<int>(W), static_cast<int>(KT),
        static_cast<int>(QT), static_cast<int>(items), vec, p.scale, NoGeo{}, p.err_word, p.timeout_ns);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) {
    const int64_t n8 = rows * D / 8;
    bwd_dq_convert_kernel<BF16><<<static_cast<unsigned>((n8 + 255) / 256), 256, 0, p.stream>>>(
        reinterpret_cast<const float4*>(p.dq_accum), static_cast<uint4*>(p.dq), n8);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) {
    *msg = cudaGetErrorString(e);
    return kErrLaunch;
  }
  return kOk;
}

}  // namespace

int launch_attn_bwd(const BwdParams& p, const char** msg) {
  if (p.D != 64 && p.D != 128) {
    *msg = "backward: head dim must be 64 or 128";
    return kErrUnsupportedD;
  }
  if (p.N > kMaxSeqLen) {
    *msg = "backward: sequence length above the supported maximum (65536)";
    return kErrUnsupportedN;
  }
  if (p.D == 128) return p.dtype == 1 ? launch<128, true>(p, msg) : launch<128, false>(p, msg);
  return p.dtype == 1 ? launch<64, true>(p, msg) : launch<64, false>(p, msg);
}

}  // namespace sma
