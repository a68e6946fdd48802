// Attention of new tokens over the paged K/V cache (moe_kv_attend):
//
//   s_j = scale * q . k_j  for the tokens j up to the row's own position
//   o   = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j
//
// in one pass over the keys with the running maximum and sum in fp32.
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kv_internal.h"

namespace moe {

template <bool BF16>
MOE_DEV float2 pair_to_float(uint32_t u) {
  if constexpr (BF16) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
}
template <bool BF16>
MOE_DEV uint32_t float_to_pair(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// A warp per (row, head), each lane HD / 32 dims, one key a step.
template <int HD, bool BF16>
__global__ void __launch_bounds__(128) kv_attend_kernel(const KvView c, const KvBatch b,
                                                        const KvAttend a) {
  pdl_enter();
  constexpr int V = HD / 64;  // pairs a lane
  const int lane = threadIdx.x & 31;
  const int64_t total = static_cast<int64_t>(min(b.q_start[b.n], b.rows)) * a.heads;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * 4;
  for (int64_t it = blockIdx.x * 4 + (threadIdx.x >> 5); it < total; it += warps) {
    const int r = static_cast<int>(it / a.heads), h = static_cast<int>(it - static_cast<int64_t>(r) * a.heads);
    const int e = entry_of_row(b.q_start, b.n, r);
    if (e < 0) continue;
    const int s = b.seqs[e];
    const bool known = s >= 0 && s < c.nseq;
    if (!known && lane == 0) record_error(c.err, DEV_BAD_SEQ);
    const int len = known ? c.len[s] : 0;
    const int64_t pos = static_cast<int64_t>(len) - (b.q_start[e + 1] - r);
    float q[2 * V], o[2 * V];
    const uint32_t* qp = reinterpret_cast<const uint32_t*>(static_cast<const __half*>(a.q) + r * a.qs[0] +
                                                           h * a.qs[1]) + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 f = pair_to_float<BF16>(qp[i]);
      q[2 * i] = f.x * a.scale;
      q[2 * i + 1] = f.y * a.scale;
      o[2 * i] = o[2 * i + 1] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int kvh = h / (a.heads / c.heads);
    for (int64_t j = 0; j <= pos; ++j) {
      const int64_t blk = j >> c.page_shift;
      const int pg = blk < c.max_blocks ? c.table[static_cast<int64_t>(s) * c.max_blocks + blk] : -1;
      if (pg < 0 || pg >= c.pages) {
        if (lane == 0) record_error(c.err, DEV_BAD_PAGE);
        break;
      }
      const int64_t slot = j & (c.page - 1);
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(c.k + a.layer * c.ks[0] + pg * c.ks[1] +
                                                             kvh * c.ks[2] + slot * c.ks[3]) + lane * V;
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(c.v + a.layer * c.vs[0] + pg * c.vs[1] +
                                                             kvh * c.vs[2] + slot * c.vs[3]) + lane * V;
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 f = pair_to_float<BF16>(kp[i]);
        x = fmaf(q[2 * i], f.x, x);
        x = fmaf(q[2 * i + 1], f.y, x);
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      const float mn = fmaxf(m, x);
      const float keep = m == -INFINITY ? 0.f : __expf(m - mn), p = __expf(x - mn);
      m = mn;
      l = l * keep + p;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 f = pair_to_float<BF16>(vp[i]);
        o[2 * i] = fmaf(p, f.x, o[2 * i] * keep);
        o[2 * i + 1] = fmaf(p, f.y, o[2 * i + 1] * keep);
      }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint32_t* op = reinterpret_cast<uint32_t*>(static_cast<__half*>(a.out) + r * a.os[0] + h * a.os[1]) + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) op[i] = float_to_pair<BF16>(o[2 * i] * inv, o[2 * i + 1] * inv);
    if (a.lse && lane == 0) a.lse[r * a.ls[0] + h * a.ls[1]] = l > 0.f ? m + logf(l) : -INFINITY;
  }
}

size_t kv_attend_workspace(const KvView&, int, int, int, int) { return 256; }

cudaError_t kv_launch_attend(const KvView& c, const CUtensorMap&, const CUtensorMap&, bool bf16,
                             const KvBatch& b, const KvAttend& a, void*, int num_sms, cudaStream_t s) {
  const int64_t items = static_cast<int64_t>(b.rows) * a.heads;
  const dim3 grid(static_cast<int>(std::min<int64_t>((items + 3) / 4, num_sms * 16)));
  if (c.hd == 128)
    return bf16 ? pdl_launch(kv_attend_kernel<128, true>, grid, dim3(128), 0, s, c, b, a)
                : pdl_launch(kv_attend_kernel<128, false>, grid, dim3(128), 0, s, c, b, a);
  return bf16 ? pdl_launch(kv_attend_kernel<64, true>, grid, dim3(128), 0, s, c, b, a)
              : pdl_launch(kv_attend_kernel<64, false>, grid, dim3(128), 0, s, c, b, a);
}

}  // namespace moe
