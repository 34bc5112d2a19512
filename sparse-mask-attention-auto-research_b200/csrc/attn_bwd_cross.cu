// Attention backward of queries and keys of different lengths, with shared key
// heads and a relative position bias: attn_bwd.cuh (kX) and the sum of the
// bias gradient over its buckets.
#include "attn_bwd.cuh"

#include <algorithm>

namespace sma {
namespace {

// dtable[bucket][h] = sum of dS over the pairs whose relative position is in
// the bucket: one block per (head, bucket) adds the diagonal sums of the
// blocks near the diagonal, [b][kb] by [d in the bucket's interval], and for
// the last bucket of a side the sums of the blocks beyond.  Every thread adds
// in a fixed order and the threads are added in a fixed tree, so the result
// does not depend on timing; FP32 throughout, rounded once to the table's type.
constexpr int kReduceThreads = 256;

template <bool BF16>
__global__ void __launch_bounds__(kReduceThreads)
    bias_reduce_kernel(const __grid_constant__ BwdGeo x, const __grid_constant__ BiasSpec s, void* dtable) {
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
  for (int b = 0; b < x.B; ++b) {
    const int off = x.bias_offsets == nullptr
                        ? x.bias_offset
                        : max(-kMaxBiasOffset, min(kMaxBiasOffset, __ldg(x.bias_offsets + b)));
    const int j_max = bias_block_max(x.bias_hi, off);
    const int j_min = -bias_block_max(-x.bias_lo, -off);
    const int lo = max(d_lo, 32 * j_min - off - 31), hi = min(d_hi, 32 * j_max - off + 31);
    const int64_t n = hi >= lo ? static_cast<int64_t>(hi - lo + 1) * x.KB : 0;
    const float* near_bh = x.near_part + (static_cast<int64_t>(b) * x.H + h) * x.KB * x.slots * 64;
    for (int64_t w = threadIdx.x; w < n; w += kReduceThreads) {
      const int kb = static_cast<int>(w / (hi - lo + 1));
      const int d = lo + static_cast<int>(w - static_cast<int64_t>(kb) * (hi - lo + 1));
      // d = 32 j - off + k: k in [0, 31] of block j, or k - 32 of block j + 1.
      const int y = d + off;
      const int j = y >= 0 ? y / 32 : -((-y + 31) / 32);
      const int k = y - 32 * j;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int jj = j + u, qb = kb - jj;
        if (jj < j_min || jj > j_max || qb < 0 || qb >= x.QB || (u == 1 && k == 0)) continue;
        const int slot = x.slot_by_query ? qb : j_max - jj;
        acc += __ldg(near_bh + (static_cast<int64_t>(kb) * x.slots + slot) * 64 + (u == 0 ? k : k + 32));
      }
    }
    const bool low_end = !high && i == s.side - 1;
    const bool high_end = s.two_sided ? high && i == s.side - 1 : i == 0;
    if (low_end || high_end) {
      const float* far_bh = x.far_part + (static_cast<int64_t>(b) * x.H + h) * x.KB * 4;
      for (int w = threadIdx.x; w < 2 * x.KB; w += kReduceThreads) {
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
    const int64_t at = static_cast<int64_t>(bucket) * s.H + h;
    if constexpr (BF16) static_cast<__nv_bfloat16*>(dtable)[at] = __float2bfloat16_rn(acc);
    else static_cast<__half*>(dtable)[at] = __float2half_rn(acc);
  }
}

// Fills the geometry; false when the query tiles of a key head exceed the list.
bool geometry(const CrossParams& p, BwdGeo* x) {
  const int G = static_cast<int>(p.H / p.Hkv);
  x->B = static_cast<int>(p.B);
  x->H = static_cast<int>(p.H);
  x->Hkv = static_cast<int>(p.Hkv);
  x->Nq = static_cast<int>(p.Nq);
  x->tn = std::min<int>(x->Nq, kT);
  x->hb = 1;
  const bool bias = p.bias.table != nullptr;
  // With a bias a tile holds one head (its blocks belong to one bias row).
  for (int h = 1; !bias && h <= G; ++h)
    if (G % h == 0 && h * x->tn <= kT) x->hb = h;
  x->gh = G / x->hb;
  x->rows = x->tn * x->hb;
  x->QT1 = (x->Nq + kT - 1) / kT;
  x->words = p.words;
  for (int i = 0; i < 3; ++i) x->word_stride[i] = p.word_stride[i];
  x->one_row = p.words != nullptr && (x->Nq == 1 || p.word_stride[2] == 0) && (G == 1 || p.word_stride[1] == 0);
  if (bias) {
    x->bias = p.bias_distance;
    x->bias_offsets = p.bias.offsets;
    x->bias_offset = p.bias.offset;
    bias_range(p.bias, &x->bias_lo, &x->bias_hi);
    x->bias_len = x->bias_hi - x->bias_lo + 1 + 2 * kBiasPad;
    x->KB = static_cast<int>((p.Nk + kT - 1) / kT * 4);
    x->QB = (x->Nq + 31) / 32;
    // Block differences that overlap (lo, hi): multiples of 32 in an open
    // interval of length hi - lo + 62.
    const int slots = (x->bias_hi - x->bias_lo + 62 + 31) / 32;
    x->slot_by_query = slots > x->QB ? 1 : 0;
    x->slots = std::min(slots, x->QB);
  }
  return static_cast<int64_t>(x->gh) * x->QT1 <= 32 * kListWords<true>;
}

template <int D, bool BF16, bool kBias>
int launch(const CrossParams& p, const CrossGrads& g, BwdGeo x, const char** msg) {
  using C = BwdCfg<D>;
  const int64_t KT = (p.Nk + kT - 1) / kT;
  const int64_t items = p.B * p.Hkv * KT;
  const int64_t rows = p.B * p.H * p.Nq;
  if (items > 0x7FFFFFFFll || (rows * (D / 8) + 255) / 256 > 0x7FFFFFFFll) {
    *msg = "backward: batch*heads too large";
    return kErrArg;
  }
  CUtensorMap mq, mk, mv, mdo, mdq;
  const int64_t so[3] = {p.H * p.Nq * D, p.Nq * D, D};
  CUresult rc = make_tensor_map_4d(&mq, p.q, p.dtype, D, p.Nq, p.H, p.B, p.q_stride, x.tn, x.hb);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mk, p.k, p.dtype, D, p.Nk, p.Hkv, p.B, p.k_stride, kT);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mv, p.v, p.dtype, D, p.Nk, p.Hkv, p.B, p.v_stride, kT);
  if (rc == CUDA_SUCCESS) rc = make_tensor_map_4d(&mdo, g.dout, p.dtype, D, p.Nq, p.H, p.B, so, x.tn, x.hb);
  // The accumulator in blocks of hb * Nq rows: a tile's rows are consecutive in it.
  if (rc == CUDA_SUCCESS)
    rc = make_tensor_map_3d_f32(&mdq, g.dq_accum, D, p.B * p.Hkv * x.gh, static_cast<int64_t>(x.hb) * p.Nq, 32);
  if (rc != CUDA_SUCCESS) {
    *msg = tensor_map_error("backward", rc);
    return kErrCuda;
  }
  DeviceProps dp;
  if (!device_props(&dp, msg)) return kErrCuda;
  static std::atomic<bool> smem_set[kMaxDevices] = {};
  auto kern = attn_bwd_kernel<D, BF16, true, kBias>;
  cudaError_t e = ensure_smem_limit(kern, C::kSmemBytes, dp.device, smem_set);
  if (e == cudaSuccess && kBias) {
    // Blocks that no live tile visits count as 0.
    const int64_t bh_kb = p.B * p.H * x.KB;
    x.near_part = g.bias_part;
    x.far_part = g.bias_part + bh_kb * x.slots * 64;
    e = cudaMemsetAsync(g.bias_part, 0, static_cast<size_t>(bh_kb) * (x.slots * 64 + 4) * sizeof(float), p.stream);
  }
  if (e == cudaSuccess) {
    bwd_delta_kernel<D, BF16><<<static_cast<unsigned>((rows * (D / 8) + 255) / 256), 256, 0, p.stream>>>(
        static_cast<const uint4*>(g.dout), static_cast<const uint4*>(p.out), g.delta,
        reinterpret_cast<float4*>(g.dq_accum), rows);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) {
    const int64_t grid = items < dp.sms ? items : dp.sms;
    kern<<<static_cast<unsigned>(grid), C::kThreads, C::kSmemBytes, p.stream>>>(
        mq, mk, mv, mdo, mdq, nullptr, p.lse, g.delta, static_cast<uint16_t*>(g.dk), static_cast<uint16_t*>(g.dv),
        static_cast<int>(p.Nk), static_cast<int>(KT * 4), static_cast<int>(KT), x.gh * x.QT1, static_cast<int>(items),
        1, p.scale, x, p.err_word, p.timeout_ns);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) {
    const int64_t n8 = rows * D / 8;
    bwd_dq_convert_kernel<BF16><<<static_cast<unsigned>((n8 + 255) / 256), 256, 0, p.stream>>>(
        reinterpret_cast<const float4*>(g.dq_accum), static_cast<uint4*>(g.dq), n8);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess && kBias) {
    const dim3 grid(static_cast<unsigned>(p.H), static_cast<unsigned>(p.bias.side * (p.bias.two_sided ? 2 : 1)));
    bias_reduce_kernel<BF16><<<grid, kReduceThreads, 0, p.stream>>>(x, p.bias, g.dtable);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) {
    *msg = cudaGetErrorString(e);
    return kErrLaunch;
  }
  return kOk;
}

template <int D, bool BF16>
int launch_b(const CrossParams& p, const CrossGrads& g, const BwdGeo& x, const char** msg) {
  return p.bias.table != nullptr ? launch<D, BF16, true>(p, g, x, msg) : launch<D, BF16, false>(p, g, x, msg);
}

}  // namespace

int64_t cross_bwd_bias_floats(const CrossParams& p) {
  BwdGeo x{};
  geometry(p, &x);
  return p.bias.table != nullptr ? p.B * p.H * x.KB * (int64_t{64} * x.slots + 4) : 0;
}

int launch_attn_cross_bwd(const CrossParams& p, const CrossGrads& g, const char** msg) {
  BwdGeo x{};
  if (!geometry(p, &x)) {
    *msg = "backward: more than 1024 query tiles (128 rows) share a key head";
    return kErrUnsupportedN;
  }
  if (p.D == 128) return p.dtype == 1 ? launch_b<128, true>(p, g, x, msg) : launch_b<128, false>(p, g, x, msg);
  return p.dtype == 1 ? launch_b<64, true>(p, g, x, msg) : launch_b<64, false>(p, g, x, msg);
}

}  // namespace sma
