// C ABI of what mixes along the sequence, apart from the whole-sequence kernels of lewi_moe.cu: single-token steps of the convolution
// and the gated delta rule, the paged cache, attention (declarations and contracts: include/lewi_moe.h).
#include "attention.cuh"
#include "common.cuh"
#include "paged.cuh"
#include "step.cuh"

using namespace lewi;

namespace lewi {
int take_mixer_status() { return take_status_word(); }
}

namespace {

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline bool aligned(const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(to - 1)) == 0; }
inline bool is_dtype(int d) { return d == LEWI_BF16 || d == LEWI_F32; }
typedef __nv_bfloat16 bf16;

// Elements of a row, and channels that a grid covers, are counted in 32 bits; past its end a grid may reach by as much as this.
constexpr int64_t kMaxRow = 0x7fffffff - 2048;

// Checks of a paged cache; 0 or an error code.
int check_cache(const void* k, const void* v, const int32_t* tables, const int32_t* lengths, int B, int Hkv, int D, int64_t pages, int page,
                int max_pages, int64_t page_stride) {
  if (!k || !v || !tables || !lengths || B <= 0 || Hkv <= 0 || D <= 0 || pages <= 0 || page <= 0 || max_pages <= 0) return LEWI_ERR_ARG;
  if (D > 256 || pages > 0x7fffffff || (int64_t)max_pages * page > 0x7fffffff - 128 || (int64_t)Hkv * D > kMaxRow) return LEWI_ERR_LIMIT;
  if (D % 8 != 0 || !aligned(k, 16) || !aligned(v, 16) || page_stride % 8 != 0 || page_stride < (int64_t)page * Hkv * D) return LEWI_ERR_SHAPE;
  return LEWI_OK;
}

template <int D, bool LONG>
int launch_paged(cudaStream_t st, const paged::Args& a) {
  static bool done[64] = {false};
  using S = paged::Shape<D>;
  if (!allow_smem(paged::attend_kernel<D, LONG>, S::kSmem, done)) return LEWI_ERR_CUDA;
  if (launch_kernel(paged::attend_kernel<D, LONG>, a.ctas, S::kThreads, S::kSmem, st, false, a) != cudaSuccess) {
    (void)cudaGetLastError();
    return LEWI_ERR_CUDA;
  }
  ++launch_counter();
  cudaLaunchConfig_t cfg = {};
  const bool few = (long long)a.c.B * a.Hq <= 2ll * num_sms();   // heads: a CTA each, or a warp each
  cfg.gridDim = dim3((unsigned)(few ? a.Hq : (a.Hq + paged::kJoinWarps - 1) / paged::kJoinWarps), (unsigned)a.c.B);
  cfg.blockDim = dim3(paged::kJoinWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if ((few ? cudaLaunchKernelEx(&cfg, paged::join_kernel<S::kTile, paged::kJoinWarps>, a) : cudaLaunchKernelEx(&cfg, paged::join_kernel<S::kTile, 1>, a)) != cudaSuccess) {
    (void)cudaGetLastError();
    return LEWI_ERR_CUDA;
  }
  ++launch_counter();
  return LEWI_OK;
}

template <int D>
int launch_paged(cudaStream_t st, const paged::Args& a) {
  using S = paged::Shape<D>;
  return (int64_t)a.c.max_pages * a.c.page > (int64_t)S::kTile * S::kChain ? launch_paged<D, true>(st, a) : launch_paged<D, false>(st, a);
}

// Checks of what forward and backward of causal attention share.
int check_attention(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride, const int32_t* cu, int n_seqs,
                    const void* o, int T, int Hq, int Hkv, int D, float scale) {
  if (!q || !k || !v || !o || T <= 0 || n_seqs <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || !(scale > 0.f && scale < 2e38f)) return LEWI_ERR_ARG;
  if (!cu && T % n_seqs != 0) return LEWI_ERR_ARG;
  if (D > attn::kMaxD || T > 0x7fffffff - attn::kTile || (int64_t)Hq * D > kMaxRow || (int64_t)Hkv * D > kMaxRow) return LEWI_ERR_LIMIT;
  if ((attn::most_tiles(T, n_seqs) + n_seqs) * Hq > 0x7fffffff) return LEWI_ERR_LIMIT;
  if ((int64_t)T * (Hq / Hkv) > attn::kMaxGroupRows) return LEWI_ERR_LIMIT;
  if (D % 8 != 0 || Hq % Hkv != 0 || !aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(o, 16)) return LEWI_ERR_SHAPE;
  if (q_stride % 8 != 0 || k_stride % 8 != 0 || v_stride % 8 != 0) return LEWI_ERR_SHAPE;
  if (q_stride < (int64_t)Hq * D || k_stride < (int64_t)Hkv * D || v_stride < (int64_t)Hkv * D) return LEWI_ERR_SHAPE;
  return LEWI_OK;
}

template <int DP, bool TRAIN, bool ONE>
int attention_fwd(cudaStream_t st, const attn::Args& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv) {
  static bool done[64] = {false};
  if (!allow_smem(attn::fwd_kernel<DP, TRAIN, ONE>, attn::FwdShape<DP>::kSmem, done)) return LEWI_ERR_CUDA;
  const long long items = attn::most_tiles(a.seqs.T, a.seqs.n) * (a.shape == attn::kTwoHeads ? a.Hq / 2 : a.Hq);
  attn::fwd_kernel<DP, TRAIN, ONE><<<attn::ctas(items), attn::kFwdThreads, attn::FwdShape<DP>::kSmem, st>>>(tq, tk, tv, a);
  LEWI_CHECK_LAUNCH();
  return LEWI_OK;
}

template <int DP>
int attention_fwd(cudaStream_t st, const attn::Args& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv) {
  const bool one = a.shape == attn::kOneTile;
  if (a.lse != nullptr) return one ? attention_fwd<DP, true, true>(st, a, tq, tk, tv) : attention_fwd<DP, true, false>(st, a, tq, tk, tv);
  return one ? attention_fwd<DP, false, true>(st, a, tq, tk, tv) : attention_fwd<DP, false, false>(st, a, tq, tk, tv);
}

template <int DP>
int attention_bwd(cudaStream_t st, const attn::Args& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& td,
                  const bf16* d_o) {
  const long long rows = (long long)a.seqs.T * a.Hq, per = attn::kDeltaThreads / (DP / 8);
  attn::delta_kernel<DP><<<(unsigned)((rows + per - 1) / per), attn::kDeltaThreads, 0, st>>>(a.o, a.o_rest, d_o, a.delta, a.seqs.T, a.Hq, a.D);
  LEWI_CHECK_LAUNCH();
  const long long tiles = attn::most_tiles(a.seqs.T, a.seqs.n);
  if (a.dk != nullptr) {
    static bool done[64] = {false};
    if (!allow_smem(attn::dkv_kernel<DP>, attn::DkvShape<DP>::kSmem, done)) return LEWI_ERR_CUDA;
    (void)launch_kernel(attn::dkv_kernel<DP>, (int)attn::ctas(tiles * a.Hkv * a.parts), attn::kBwdThreads, attn::DkvShape<DP>::kSmem, st, false, tq, tk,
                        tv, td, a);   // (not early: dQ's kernel, which is, reads delta too)
    LEWI_CHECK_LAUNCH();
  }
  if (a.dq != nullptr) {
    static bool done[64] = {false};
    if (!allow_smem(attn::dq_kernel<DP>, attn::DqShape<DP>::kSmem, done)) return LEWI_ERR_CUDA;
    (void)launch_kernel(attn::dq_kernel<DP>, (int)attn::ctas(tiles * a.Hq), attn::kBwdThreads, attn::DqShape<DP>::kSmem, st, true, tq, tk, tv, td, a);
    LEWI_CHECK_LAUNCH();
  }
  if (a.dk != nullptr) {
    if (a.parts > 1) {
      const long long vecs = (long long)a.seqs.T * a.Hkv * a.D / 4;
      attn::dkv_sum_kernel<<<(unsigned)((vecs + attn::kSumThreads - 1) / attn::kSumThreads), attn::kSumThreads, 0, st>>>(a);
      LEWI_CHECK_LAUNCH();
    }
  }
  return LEWI_OK;
}

inline int64_t delta_bytes(int T, int Hq) { return ((int64_t)T * Hq * 4 + 255) / 256 * 256; }
inline int64_t sums_bytes(int T, int Hkv, int D, int parts) { return parts > 1 ? (int64_t)parts * 2 * T * Hkv * D * 4 : 0; }

inline int paged_ctas(int D) { return num_sms() * (D > 128 ? paged::Shape<256>::kCtas : paged::Shape<128>::kCtas); }
inline int64_t paged_parts_bytes(int D) { return ((int64_t)2 * paged_ctas(D) * paged::kRows * (D + 2) * 4 + 15) / 16 * 16; }
inline int64_t paged_kept_bytes(int D) {
  const int columns = D > 128 ? 256 : D > 64 ? 128 : 64, warps = D > 128 ? paged::Shape<256>::kWarps : paged::Shape<128>::kWarps;
  return (int64_t)paged_ctas(D) * warps * 32 * (columns / 8 * 16 + 8);
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------------------------------------ single-token steps

int lewi_causal_conv1d_step(void* stream, const void* x, int64_t x_stride, const void* w, void* state, const int32_t* slots, void* y, int B,
                            int N, int C, int K) {
  if (!x || !w || !y || B <= 0 || N <= 0 || C <= 0 || K <= 0 || (K > 1 && !state) || (!slots && N < B)) return LEWI_ERR_ARG;
  if (K > 8 || B > 65535 || C > kMaxRow) return LEWI_ERR_LIMIT;
  if (C % 8 != 0 || x_stride % 8 != 0 || x_stride < C || !aligned(x, 16) || !aligned(w, 16) || !aligned(state, 16) || !aligned(y, 16))
    return LEWI_ERR_SHAPE;
  const step::ConvArgs a{reinterpret_cast<const bf16*>(x), x_stride, reinterpret_cast<const bf16*>(w), reinterpret_cast<bf16*>(state), slots,
                         reinterpret_cast<bf16*>(y), N, C};
  const dim3 grid((unsigned)((C / 8 + step::kThreads - 1) / step::kThreads), (unsigned)B);
  cudaStream_t st = as_stream(stream);
  switch (K) {
    case 1: step::conv_step_kernel<1><<<grid, step::kThreads, 0, st>>>(a); break;
    case 2: step::conv_step_kernel<2><<<grid, step::kThreads, 0, st>>>(a); break;
    case 3: step::conv_step_kernel<3><<<grid, step::kThreads, 0, st>>>(a); break;
    case 4: step::conv_step_kernel<4><<<grid, step::kThreads, 0, st>>>(a); break;
    case 5: step::conv_step_kernel<5><<<grid, step::kThreads, 0, st>>>(a); break;
    case 6: step::conv_step_kernel<6><<<grid, step::kThreads, 0, st>>>(a); break;
    case 7: step::conv_step_kernel<7><<<grid, step::kThreads, 0, st>>>(a); break;
    default: step::conv_step_kernel<8><<<grid, step::kThreads, 0, st>>>(a); break;
  }
  LEWI_CHECK_LAUNCH();
  return LEWI_OK;
}

int lewi_gdn_step(void* stream, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                  const void* g, int g_dtype, const void* beta, int beta_dtype, float* state, const int32_t* slots, void* o, int B, int N,
                  int Hk, int H, int K, int V) {
  if (!q || !k || !v || !g || !beta || !state || !o || B <= 0 || N <= 0 || Hk <= 0 || H <= 0 || K <= 0 || V <= 0) return LEWI_ERR_ARG;
  if (!is_dtype(g_dtype) || !is_dtype(beta_dtype) || (!slots && N < B)) return LEWI_ERR_ARG;
  if (K > step::kMaxK || H > 65535 || B > 65535 || V > kMaxRow) return LEWI_ERR_LIMIT;
  if (K % 8 != 0 || V % 8 != 0 || H % Hk != 0 || !aligned(state, 16) || !aligned(o, 8)) return LEWI_ERR_SHAPE;
  if (q_stride < (int64_t)Hk * K || k_stride < (int64_t)Hk * K || v_stride < (int64_t)H * V) return LEWI_ERR_SHAPE;
  const step::GdnArgs a{reinterpret_cast<const bf16*>(q), reinterpret_cast<const bf16*>(k), reinterpret_cast<const bf16*>(v), q_stride, k_stride,
                        v_stride, g, beta, g_dtype == LEWI_F32, beta_dtype == LEWI_F32, state, slots, reinterpret_cast<bf16*>(o), N, Hk, H, K, V,
                        1.f / sqrtf((float)K)};
  const dim3 grid((unsigned)((V + step::kCols - 1) / step::kCols), (unsigned)H, (unsigned)B);
  step::gdn_step_kernel<<<grid, step::kThreads, 0, as_stream(stream)>>>(a);
  LEWI_CHECK_LAUNCH();
  return LEWI_OK;
}

// ------------------------------------------------------------------------------------------------ paged cache

int lewi_paged_cache_write(void* stream, const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* k_cache, void* v_cache,
                           int64_t page_stride, const int32_t* tables, const int32_t* lengths, const int32_t* cu_seqlens, int T, int B,
                           int Hkv, int D, int64_t pages, int page, int max_pages) {
  if (!k || !v || T <= 0) return LEWI_ERR_ARG;
  if (const int rc = check_cache(k_cache, v_cache, tables, lengths, B, Hkv, D, pages, page, max_pages, page_stride)) return rc;
  if (!cu_seqlens && T != B) return LEWI_ERR_ARG;
  const int64_t row = (int64_t)Hkv * D;
  if (!aligned(k, 16) || !aligned(v, 16) || k_stride % 8 != 0 || v_stride % 8 != 0 || k_stride < row || v_stride < row) return LEWI_ERR_SHAPE;
  const paged::WriteArgs a{{tables, lengths, reinterpret_cast<bf16*>(k_cache), reinterpret_cast<bf16*>(v_cache), page_stride, B, Hkv, D,
                            (int)pages, page, max_pages},
                           reinterpret_cast<const bf16*>(k), reinterpret_cast<const bf16*>(v), k_stride, v_stride, cu_seqlens, T};
  constexpr int per = paged::kWriteThreads / 32;
  paged::write_kernel<<<(unsigned)(((int64_t)T + per - 1) / per), paged::kWriteThreads, 0, as_stream(stream)>>>(a);
  LEWI_CHECK_LAUNCH();
  return LEWI_OK;
}

int64_t lewi_paged_attention_workspace_bytes(int D) {
  if (D <= 0) return LEWI_ERR_ARG;
  if (D > 256) return LEWI_ERR_LIMIT;
  return paged_parts_bytes(D) + paged_kept_bytes(D);
}

int lewi_paged_attention(void* stream, const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, int64_t page_stride,
                         const int32_t* tables, const int32_t* lengths, void* o, void* workspace, int64_t workspace_bytes, int B, int Hq,
                         int Hkv, int D, int64_t pages, int page, int max_pages, float scale) {
  if (!q || !o || Hq <= 0 || !(scale > -2e38f && scale < 2e38f)) return LEWI_ERR_ARG;
  if (const int rc = check_cache(k_cache, v_cache, tables, lengths, B, Hkv, D, pages, page, max_pages, page_stride)) return rc;
  if (B > 65535 || (int64_t)Hq * D > kMaxRow) return LEWI_ERR_LIMIT;
  if (Hq % Hkv != 0 || !aligned(q, 4) || q_stride % 2 != 0 || q_stride < (int64_t)Hq * D || !aligned(o, 8)) return LEWI_ERR_SHAPE;
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < lewi_paged_attention_workspace_bytes(D)) return LEWI_ERR_WORKSPACE;
  const int G = Hq / Hkv, MT = (G + paged::kRows - 1) / paged::kRows;
  const paged::Args a{{tables, lengths, const_cast<bf16*>(reinterpret_cast<const bf16*>(k_cache)),
                       const_cast<bf16*>(reinterpret_cast<const bf16*>(v_cache)), page_stride, B, Hkv, D, (int)pages, page, max_pages},
                      reinterpret_cast<const bf16*>(q), q_stride, reinterpret_cast<bf16*>(o), reinterpret_cast<float*>(workspace),
                      reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(workspace) + paged_parts_bytes(D)), Hq, G, MT,
                      paged_ctas(D), scale * 1.4426950408889634f};
  cudaStream_t st = as_stream(stream);
  if (D <= 64) return launch_paged<64>(st, a);
  if (D <= 128) return launch_paged<128>(st, a);
  return launch_paged<256>(st, a);
}

// ------------------------------------------------------------------------------------------------ causal attention

int lewi_causal_attention_fwd(void* stream, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                              const int32_t* cu_seqlens, int n_seqs, void* o, void* o_rest, float* lse, int T, int Hq, int Hkv, int D,
                              float scale) {
  if (const int rc = check_attention(q, q_stride, k, k_stride, v, v_stride, cu_seqlens, n_seqs, o, T, Hq, Hkv, D, scale)) return rc;
  if (lse && !o_rest) return LEWI_ERR_ARG;
  if (!o_rest && T > attn::kChain * attn::kTile) return LEWI_ERR_WORKSPACE;
  if (!aligned(o_rest, 16)) return LEWI_ERR_SHAPE;
  CUtensorMap tq, tk, tv;
  if (!attn::make_rows_map(&tq, q, T, Hq, D, q_stride) || !attn::make_rows_map(&tk, k, T, Hkv, D, k_stride) ||
      !attn::make_rows_map(&tv, v, T, Hkv, D, v_stride))
    return LEWI_ERR_CUDA;
  const attn::Args a{{cu_seqlens, n_seqs, T}, Hq, Hkv, Hq / Hkv, D, scale, scale * 1.4426950408889634f, reinterpret_cast<bf16*>(o),
                     reinterpret_cast<bf16*>(o_rest), lse, nullptr, nullptr, nullptr, nullptr, 1, nullptr, nullptr, nullptr, attn::fwd_item(T, n_seqs, Hq, Hq / Hkv)};
  cudaStream_t st = as_stream(stream);
  return D <= 64 ? attention_fwd<64>(st, a, tq, tk, tv) : attention_fwd<128>(st, a, tq, tk, tv);
}

int64_t lewi_causal_attention_bwd_workspace_bytes(int T, int n_seqs, int Hq, int Hkv, int D) {
  if (T <= 0 || n_seqs <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || Hq % Hkv != 0) return LEWI_ERR_ARG;
  if (D > attn::kMaxD || (int64_t)T * (Hq / Hkv) > attn::kMaxGroupRows) return LEWI_ERR_LIMIT;
  const int parts = attn::dkv_parts(T, n_seqs, Hq, Hkv, D);
  return delta_bytes(T, Hq) + sums_bytes(T, Hkv, D, parts) + attn::chain_kv_bytes(T, Hq / Hkv, parts, D) + attn::chain_q_bytes(T, D);
}

int lewi_causal_attention_bwd(void* stream, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                              const void* o, const void* o_rest, const float* lse, const void* d_o, const int32_t* cu_seqlens, int n_seqs,
                              void* dq, void* dk, void* dv, void* workspace, int64_t workspace_bytes, int T, int Hq, int Hkv, int D, float scale) {
  if (const int rc = check_attention(q, q_stride, k, k_stride, v, v_stride, cu_seqlens, n_seqs, o, T, Hq, Hkv, D, scale)) return rc;
  if (!d_o || !o_rest || !lse || (!dq && !dk) || !dk != !dv) return LEWI_ERR_ARG;
  if (!aligned(d_o, 16) || !aligned(o_rest, 16) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16)) return LEWI_ERR_SHAPE;
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < lewi_causal_attention_bwd_workspace_bytes(T, n_seqs, Hq, Hkv, D))
    return LEWI_ERR_WORKSPACE;
  CUtensorMap tq, tk, tv, td;
  if (!attn::make_rows_map(&tq, q, T, Hq, D, q_stride) || !attn::make_rows_map(&tk, k, T, Hkv, D, k_stride) ||
      !attn::make_rows_map(&tv, v, T, Hkv, D, v_stride) || !attn::make_rows_map(&td, d_o, T, Hq, D, (int64_t)Hq * D))
    return LEWI_ERR_CUDA;
  const int parts = attn::dkv_parts(T, n_seqs, Hq, Hkv, D);
  uint8_t* at = reinterpret_cast<uint8_t*>(workspace) + delta_bytes(T, Hq);
  const int64_t sums = sums_bytes(T, Hkv, D, parts), kept = attn::chain_kv_bytes(T, Hq / Hkv, parts, D);
  const attn::Args a{{cu_seqlens, n_seqs, T}, Hq, Hkv, Hq / Hkv, D, scale, scale * 1.4426950408889634f,
                     const_cast<bf16*>(reinterpret_cast<const bf16*>(o)), const_cast<bf16*>(reinterpret_cast<const bf16*>(o_rest)),
                     const_cast<float*>(lse), reinterpret_cast<float*>(workspace),
                     reinterpret_cast<bf16*>(dq), reinterpret_cast<bf16*>(dk), reinterpret_cast<bf16*>(dv),
                     parts, reinterpret_cast<float*>(at), reinterpret_cast<float4*>(at + sums), reinterpret_cast<float4*>(at + sums + kept)};
  const bf16* g = reinterpret_cast<const bf16*>(d_o);
  return D <= 64 ? attention_bwd<64>(as_stream(stream), a, tq, tk, tv, td, g) : attention_bwd<128>(as_stream(stream), a, tq, tk, tv, td, g);
}

}  // extern "C"
