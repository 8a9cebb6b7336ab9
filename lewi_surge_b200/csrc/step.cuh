// Single-token steps of the mixers beside the MoE layer: what a decode loop calls once per token where a prompt goes through the
// chunked kernels.  A row of the batch names the place of its sequence in a pool of states (`slots`; none: row b has state b), which
// is read, moved one token on and written back.  A negative slot is an idle row: zeros, no state touched.  A slot past the pool, or
// one that an earlier row of the batch has, is refused on the device: zeros, no state touched, LEWI_STATUS_BAD_INDEX.
#pragma once

#include "common.cuh"

namespace lewi {
namespace step {

constexpr int kThreads = 128;

// The row's state, or -1 for a row that has none.  All threads of the CTA call it; `pre` runs between the look at the row's own slot and
// the look through those of the rows before it, which is where the state can be requested.
template <class F>
__device__ __forceinline__ int claim_slot(const int32_t* __restrict__ slots, int b, int n_states, F pre) {
  const int mine = slots != nullptr ? slots[b] : b;
  const bool in = mine >= 0 && mine < n_states;
  if (in) pre(mine);
  int taken = 0;
  if (slots != nullptr && in)
    for (int i = threadIdx.x; i < b; i += kThreads) taken |= slots[i] == mine;
  taken = __syncthreads_or(taken);
  if ((taken || mine >= n_states) && threadIdx.x == 0) raise_status(LEWI_STATUS_BAD_INDEX);
  return in && !taken ? mine : -1;
}

// ---------------------------------------------------------------- gated delta rule
// Per (row, head), with a = exp(g) and the state S [K,V] float32:
//   d = beta (v - a k^T S),   o = K^-1/2 (a q^T S + (q.k) d),   S <- a S + k d^T
// which is the recurrence S <- a S, S <- S + beta k (v - k^T S), o = K^-1/2 q^T S with both products taken of the state as it was read, so
// that one pass over it is enough.  A CTA takes 64 columns of V and holds them in registers (16 lanes of 4 columns, 8 rows at a
// time); sums over K are float32, joined over the lanes and the warps in a fixed order.
// Bound by the state's way in and out: 8 bytes per element, 7 flops.  256 rows x 32 heads, K = V = 128 (1.07 GB): 165 us, 6.5 TB/s (32
// columns, no streaming hint: 208; 32 with it 177; 64 without 169; 128 columns 183).
constexpr int kCols = 64, kLanes = kCols / 4, kRowGroups = kThreads / kLanes, kMaxK = 128, kRowsPerThread = kMaxK / kRowGroups;

struct GdnArgs {
  const __nv_bfloat16 *q, *k, *v;            // [B,Hk,K], [B,Hk,K], [B,H,V]; rows of the batch qs, ks, vs elements apart
  long long qs, ks, vs;
  const void *g, *beta;                      // [B,H], float32 or bf16
  int g_f32, beta_f32;
  float* state;                              // [N,H,K,V]
  const int32_t* slots;
  __nv_bfloat16* o;                          // [B,H,V]
  int N, Hk, H, K, V;
  float scale;
};

__device__ __forceinline__ float ld_scalar(const void* p, long long i, int f32) {
  return f32 ? reinterpret_cast<const float*>(p)[i] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

__global__ void __launch_bounds__(kThreads) gdn_step_kernel(const GdnArgs a) {
  __shared__ float s_q[kMaxK], s_k[kMaxK];
  __shared__ float s_sum[kThreads / 32][kLanes][9];
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int l = tid % kLanes, rg = tid / kLanes, col = blockIdx.x * kCols + l * 4;
  const bool live = col < a.V;
  float4 s[kRowsPerThread];
  const int slot = claim_slot(a.slots, b, a.N, [&](int n) {
    const float* base = a.state + ((long long)n * a.H + h) * a.K * a.V + col;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
      const int r = rg + i * kRowGroups;
      s[i] = live && r < a.K ? __ldcs(reinterpret_cast<const float4*>(base + (long long)r * a.V)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int hk = h / (a.H / a.Hk);
    s_q[tid] = tid < a.K ? __bfloat162float(a.q[b * a.qs + hk * a.K + tid]) : 0.f;
    s_k[tid] = tid < a.K ? __bfloat162float(a.k[b * a.ks + hk * a.K + tid]) : 0.f;
  });
  __nv_bfloat16* o = a.o + ((long long)b * a.H + h) * a.V + col;
  if (slot < 0) {
    if (rg == 0 && live) *reinterpret_cast<uint2*>(o) = make_uint2(0u, 0u);
    return;
  }
  const float decay = expf(ld_scalar(a.g, (long long)b * a.H + h, a.g_f32));
  const float beta = ld_scalar(a.beta, (long long)b * a.H + h, a.beta_f32);
  float v[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = live ? __bfloat162float(a.v[b * a.vs + (long long)h * a.V + col + c]) : 0.f;
  float sum[9] = {};   // k^T S and q^T S of the four columns, q.k
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i) {
    const float kk = s_k[rg + i * kRowGroups], qq = s_q[rg + i * kRowGroups];
    sum[0] = fmaf(kk, s[i].x, sum[0]); sum[1] = fmaf(kk, s[i].y, sum[1]); sum[2] = fmaf(kk, s[i].z, sum[2]); sum[3] = fmaf(kk, s[i].w, sum[3]);
    sum[4] = fmaf(qq, s[i].x, sum[4]); sum[5] = fmaf(qq, s[i].y, sum[5]); sum[6] = fmaf(qq, s[i].z, sum[6]); sum[7] = fmaf(qq, s[i].w, sum[7]);
    sum[8] = fmaf(qq, kk, sum[8]);
  }
#pragma unroll
  for (int j = 0; j < 9; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 16);
  if (lane < kLanes) {
#pragma unroll
    for (int j = 0; j < 9; ++j) s_sum[warp][lane][j] = sum[j];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 9; ++j) sum[j] = (s_sum[0][l][j] + s_sum[1][l][j]) + (s_sum[2][l][j] + s_sum[3][l][j]);
  float d[4], out[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    d[c] = beta * (v[c] - decay * sum[c]);
    out[c] = a.scale * fmaf(sum[8], d[c], decay * sum[4 + c]);
  }
  if (!live) return;
  if (rg == 0) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16(out[0], out[1]), pack_bf16(out[2], out[3]));
  float* base = a.state + ((long long)slot * a.H + h) * a.K * a.V + col;
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i) {
    const int r = rg + i * kRowGroups;
    if (r >= a.K) break;
    const float kk = s_k[r];
    __stcs(reinterpret_cast<float4*>(base + (long long)r * a.V),
        make_float4(fmaf(kk, d[0], decay * s[i].x), fmaf(kk, d[1], decay * s[i].y), fmaf(kk, d[2], decay * s[i].z), fmaf(kk, d[3], decay * s[i].w)));
  }
}

// ---------------------------------------------------------------- causal convolution
// y[b,c] = sum_{j<K} w[j,c] z[j,c] with z = the K-1 inputs before this one (the state, oldest first) and x[b,c]; the state becomes
// z[1..].  A thread owns 8 channels; products and sums float32 in the order of the whole-sequence kernel, one rounding at the end.
// 256 rows x 8192 channels, 4 taps (34 MB): 5.7 us, 5.9 TB/s.
struct ConvArgs {
  const __nv_bfloat16* x;   // [B,C], rows xs elements apart
  long long xs;
  const __nv_bfloat16* w;   // [K,C]
  __nv_bfloat16* state;     // [N,K-1,C]
  const int32_t* slots;
  __nv_bfloat16* y;         // [B,C]
  int N, C;
};

template <int KT>
__global__ void __launch_bounds__(kThreads) conv_step_kernel(const ConvArgs a) {
  const int b = blockIdx.y, c0 = (blockIdx.x * kThreads + threadIdx.x) * 8;
  const bool live = c0 < a.C;
  uint4 z[KT], w[KT];
  const int slot = claim_slot(a.slots, b, a.N, [&](int n) {
    if (!live) return;
#pragma unroll
    for (int j = 0; j < KT - 1; ++j) z[j] = *reinterpret_cast<const uint4*>(a.state + ((long long)n * (KT - 1) + j) * a.C + c0);
    z[KT - 1] = ld_nc_v4(a.x + b * a.xs + c0);
#pragma unroll
    for (int j = 0; j < KT; ++j) w[j] = ld_nc_v4(a.w + (long long)j * a.C + c0);
  });
  if (!live) return;
  __nv_bfloat16* y = a.y + (long long)b * a.C + c0;
  if (slot < 0) {
    st_v4(y, make_uint4(0u, 0u, 0u, 0u));
    return;
  }
  float acc[8] = {};
#pragma unroll
  for (int j = 0; j < KT; ++j) {
    const uint32_t zz[4] = {z[j].x, z[j].y, z[j].z, z[j].w}, ww[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      acc[2 * q] = fmaf(bf16_lo(ww[q]), bf16_lo(zz[q]), acc[2 * q]);
      acc[2 * q + 1] = fmaf(bf16_hi(ww[q]), bf16_hi(zz[q]), acc[2 * q + 1]);
    }
  }
  st_v4(y, make_uint4(pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3]), pack_bf16(acc[4], acc[5]), pack_bf16(acc[6], acc[7])));
#pragma unroll
  for (int j = 0; j < KT - 1; ++j) st_v4(a.state + ((long long)slot * (KT - 1) + j) * a.C + c0, z[j + 1]);
}

}  // namespace step
}  // namespace lewi
