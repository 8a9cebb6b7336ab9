// A paged key-value cache: new tokens written to their cells, attention of one new token per sequence over what is there.
//
// k_cache, v_cache [pages][page][Hkv][D] bf16 (pages `page_stride` elements apart); a sequence's tokens lie in the pages of its row of
// `tables` [B][max_pages], `lengths[b]` of them.  A length past the table is cut to it and a page that does not exist is left out
// (LEWI_STATUS_BAD_INDEX either way); entries past a sequence's length are not read.
#pragma once

#include "common.cuh"
#include "gdn_mma.cuh"
#include "tcgen05.cuh"

namespace lewi {
namespace paged {

struct Cache {
  const int32_t *tables, *lengths;
  __nv_bfloat16 *k, *v;
  long long page_stride;
  int B, Hkv, D, pages, page, max_pages;
};

// tokens of sequence b that the cache can hold
__device__ __forceinline__ int length_of(const Cache& c, int b) {
  return max(0, (int)min((long long)c.lengths[b], (long long)c.max_pages * c.page));
}
// Element at which cell `pos` of sequence b starts (head 0), -1 where its page does not exist.
__device__ __forceinline__ long long cell_of(const Cache& c, int b, int pos) {
  const unsigned p = (unsigned)pos / (unsigned)c.page;
  const int id = c.tables[(long long)b * c.max_pages + p];
  if (id < 0 || id >= c.pages) return -1;
  return id * c.page_stride + (long long)(pos - (int)p * c.page) * c.Hkv * c.D;
}

// ---------------------------------------------------------------- write
// Token i of sequence b (tokens cu[b] .. cu[b+1]; without cu one token per sequence) goes to cell lengths[b] - n_b + i.  A warp per
// token: 16-byte pieces, every one requested before the first is stored.  Tokens of no sequence are left out; a token before
// the cache's start or past its table raises LEWI_STATUS_BAD_INDEX and is left out.  8191 tokens x 4 heads x 128 (34 MB): 5.7 us, 5.9 TB/s.
constexpr int kWriteThreads = 128;
struct WriteArgs {
  Cache c;
  const __nv_bfloat16 *k, *v;   // [T][Hkv][D], tokens ks, vs elements apart
  long long ks, vs;
  const int32_t* cu;
  int T;
};

__device__ __forceinline__ void write_row(const __nv_bfloat16* __restrict__ src, __nv_bfloat16* __restrict__ dst,
                                          const __nv_bfloat16* __restrict__ src2, __nv_bfloat16* __restrict__ dst2, int vecs, int lane) {
  constexpr int kAhead = 4;
  for (int i0 = lane; i0 < vecs; i0 += 32 * kAhead) {
    uint4 a[kAhead], b[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + 32 * j < vecs) {
        a[j] = ld_nc_v4(src + (i0 + 32 * j) * 8);
        b[j] = ld_nc_v4(src2 + (i0 + 32 * j) * 8);
      }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + 32 * j < vecs) {
        st_v4(dst + (i0 + 32 * j) * 8, a[j]);
        st_v4(dst2 + (i0 + 32 * j) * 8, b[j]);
      }
  }
}

__global__ void __launch_bounds__(kWriteThreads) write_kernel(const WriteArgs a) {
  const long long at = (long long)blockIdx.x * (kWriteThreads / 32) + (threadIdx.x >> 5);   // (threads of 2^27 tokens pass 32 bits)
  if (at >= a.T) return;
  const int t = (int)at, lane = threadIdx.x & 31;
  int b = t, back = 1;   // the token's sequence, and how far from its end it is
  if (a.cu != nullptr) {
    // the last b with cu[b] <= t, 32 bounds at a time; [lo, hi) holds it
    int lo = 0, hi = a.c.B + 1;
    while (hi - lo > 1) {
      const int stride = (hi - lo + 31) / 32, at = lo + lane * stride;
      const unsigned le = __ballot_sync(0xffffffffu, at < hi && a.cu[at] <= t);
      if (le == 0u) break;   // before the first sequence (or bounds that fall)
      const int last = 31 - __clz(le);
      lo += last * stride;
      hi = min(hi, lo + stride);
    }
    if (lo >= a.c.B) return;
    const int first = a.cu[lo], end = a.cu[lo + 1];
    if (first > t || end <= t) return;
    b = lo;
    back = end - t;
  }
  const int len = length_of(a.c, b);
  const long long pos = (long long)a.c.lengths[b] - back;
  const long long cell = pos >= 0 && pos < len ? cell_of(a.c, b, (int)pos) : -1;
  if (cell < 0) {
    if (lane == 0 && (a.cu != nullptr || a.c.lengths[b] > 0)) raise_status(LEWI_STATUS_BAD_INDEX);   // (length 0: an idle row)
    return;
  }
  write_row(a.k + t * a.ks, a.c.k + cell, a.v + t * a.vs, a.c.v + cell, a.c.Hkv * a.c.D / 8, lane);
}

// ---------------------------------------------------------------- attention of one token
// o[b,h] = sum_j p_j v_j, p = softmax(scale q.k_j) over the sequence's cells; one pass with a running maximum and sum (float32).
//
// Bound by the cache's way from HBM: 4 Hkv D bytes per cell (64 sequences of up to 8192, 4 key heads, D = 128: 101 us, 5.3 TB/s, of which 15 us are
// the first loads, which depend on one another, and the join).  The cells of all sequences and key heads are one long list of tiles of
// 64 cells (128 where D <= 64, 96 where D > 128), of which every CTA takes an equal run, whatever the lengths (they are read on the device, so a
// captured launch follows them).  The query heads that share a key head are the 16 rows of an `mma.sync` (m16n8k16), a warp's 16 cells (32 where D <= 64) its columns; a
// warp has its own ring of tiles in shared memory (cp.async) and its own softmax, and nothing is synchronised before a head's
// tiles end.  There the four (six) warps' results are joined; a head that one CTA has whole is written out, of the others every CTA leaves
// its part (at most two per CTA) and `join_kernel` adds them up in the order of the cells.
// p is rounded to bf16 for its product with v (relative 2^-8 at most, as the output's own rounding); its sum is taken before.  A second product with what
// that left would bring errors of 2.1e-3 of the output's norm down to its own rounding's 1.7e-3, and takes 104.5 instead of 101 us (D = 96: 89, 82).
constexpr int kRows = 16, kJoinCols = 32;

// What bounds a warp is the latency of its chain from scores to sums, so as many warps as there is room for share an SM: three CTAs of four with
// two stages (64 sequences of up to 8192, 4 key heads: 101 us, two CTAs with three stages 105; 32 of up to 4000, 16 key heads, D = 64: 60 and
// 64; D = 96, 16 of 16,384: 84 and 102), at D = 256 one of six.
template <int D>
struct Shape {
  static constexpr int kWarps = D == 256 ? 6 : 4, kThreads = kWarps * 32, kCtas = D == 256 ? 1 : 3;   // CTAs per SM
  static constexpr int kChunk = D == 64 ? 32 : 16, kTile = kWarps * kChunk;   // cells that a warp, and all of them, take at a time
  static constexpr int kStage = 2 * kChunk * D * 2, kStages = 2;              // a warp's K and V of them
  // Tiles that a warp sums up in one chain of products, which the tensor core truncates one by one: a sum of one sign over n of its cells comes out short by
  // about n 2^-28 of itself (of 10^6 cells, shared by four warps: 7e-4).  Then its sums are added, rounded to nearest, to those it keeps in memory.
  static constexpr int kChain = 32768 / kChunk;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kSmem = kRing + kWarps * kRows * kJoinCols * 4 + 2 * kWarps * kRows * 4 + kWarps * kStages * 4 + 128;
};

struct Args {
  Cache c;
  const __nv_bfloat16* q;   // [B][Hq][D], rows of the batch qs elements apart
  long long qs;
  __nv_bfloat16* o;         // [B][Hq][D]
  float* part;              // [2 per CTA][16][D] sums, then [2 per CTA][16] maxima, then as many sums of p
  float4* kept;             // per warp [D / 8][32 lanes] sums of a head's chains so far, then per warp [32] maxima of two rows
  int Hq, G, MT, ctas;      // query heads per key head, groups of 16 of them, CTAs of the list
  float scale_log2;
};

// Where the list stands: tile t of `nt` of row group r of sequence b.
struct Cursor {
  int b, r, t, nt;
};

template <int TILE>
__device__ __forceinline__ int tiles_of(const Cache& c, int b) {
  return (length_of(c, b) + TILE - 1) / TILE;
}

template <int TILE>
__device__ __forceinline__ void next_tile(Cursor& u, const Cache& c, int R) {
  if (++u.t < u.nt) return;
  u.t = 0;
  if (++u.r < R) return;
  u.r = 0;
  do {
    if (++u.b >= c.B) return;
    u.nt = tiles_of<TILE>(c, u.b);
  } while (u.nt == 0);
}

// Tiles of all sequences and of those before `upto` (both times R: places in the list); all threads of the CTA call it.
template <int TILE, int WARPS>
__device__ __forceinline__ longlong2 count_tiles(const Cache& c, int upto, long long (&s)[2][WARPS]) {
  long long all = 0, before = 0;
  for (int b = threadIdx.x; b < c.B; b += WARPS * 32) {
    const int n = tiles_of<TILE>(c, b);
    all += n;
    if (b < upto) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    s[0][threadIdx.x >> 5] = all;
    s[1][threadIdx.x >> 5] = before;
  }
  __syncthreads();
  all = before = 0;
#pragma unroll
  for (int x = 0; x < WARPS; ++x) {
    all += s[0][x];
    before += s[1][x];
  }
  return make_longlong2(all, before);
}

// LONG: a head may have more than kChain tiles (apart: the registers that this takes cost 64 sequences of up to 8192, 4 key heads, 104.7 us instead of 101).
template <int D, bool LONG>
__global__ void __launch_bounds__(Shape<D>::kThreads, Shape<D>::kCtas) attend_kernel(const Args a) {
  using S = Shape<D>;
  constexpr int kWarps = S::kWarps;
  constexpr int ST = S::kStages, KS = D / 16, VR = D / 8, CH = S::kChunk;   // 16-wide steps over D, 16-byte vectors of a row
  constexpr int kRowBytes = CH * 128;                                       // a box of 64 columns
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long s_count[2][kWarps];
  __shared__ Cursor s_start;
  grid_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = a.c.Hkv * a.MT;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~(uintptr_t)127);
  float* s_o = reinterpret_cast<float*>(smem + S::kRing);                       // [warp][16][32]
  float* s_m = s_o + kWarps * kRows * kJoinCols;                                // [warp][16]
  float* s_l = s_m + kWarps * kRows;
  uint32_t* s_mask = reinterpret_cast<uint32_t*>(s_l + kWarps * kRows) + warp * ST;   // cells of a stage that count
  const uint32_t ring = ptx::smem_u32(smem) + warp * ST * S::kStage;
  const gdn::LaneOff L = gdn::lane_off(lane);

  // this CTA's run of the list, and where it starts
  const long long total = count_tiles<S::kTile, kWarps>(a.c, 0, s_count).x * R;
  const long long n_ctas = min(total, (long long)a.ctas);   // (so that no run is empty)
  if (blockIdx.x >= n_ctas) return;
  const long long w0 = blockIdx.x * total / n_ctas, w1 = (blockIdx.x + 1) * total / n_ctas;
  if (warp == 0) {   // 32 sequences at a time
    long long at = 0;
    for (int b0 = 0; b0 < a.c.B; b0 += 32) {
      const int n = b0 + lane < a.c.B ? tiles_of<S::kTile>(a.c, b0 + lane) : 0;
      long long upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, (at + upto) * R > w0);
      if (past != 0u) {
        if (lane == __ffs(past) - 1) {
          const long long in = w0 - (at + upto - n) * R;   // place in the sequence's own tiles
          s_start = Cursor{b0 + lane, (int)(in / n), (int)(in % n), n};
        }
        break;
      }
      at += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  __syncthreads();
  Cursor use = s_start, get = use;

  // The cells of the tile that is requested next, looked up one request ahead: where pages hold whole chunks all of them follow the first,
  // otherwise a lane has one.
  const bool in_row = a.c.page % CH == 0;
  const int step = a.c.Hkv * a.c.D, row0 = lane / VR, vec0 = (lane % VR) * 8;   // of this lane's first piece
  long long cell = -1;
  int there = 0;   // cells of the chunk
  bool bad = false;
  auto look = [&] {
    const int pos0 = get.t * S::kTile + warp * CH, pos = in_row ? pos0 : pos0 + lane;
    there = min(max(length_of(a.c, get.b) - pos0, 0), CH);
    cell = -1;
    if (in_row ? there > 0 : lane < there) {
      cell = cell_of(a.c, get.b, pos);
      bad |= cell < 0;
    }
  };
  long long got = w0;
  look();
  auto request = [&](int stage) {
    if (got < w1) {
      const uint32_t at = ring + stage * S::kStage + (vec0 >> 6) * kRowBytes;
      const int head = get.r / a.MT * a.c.D + vec0;
      const bool col = vec0 < a.c.D;
      uint32_t mask;
      if (in_row) {
        const int rows = cell < 0 ? 0 : there;
        mask = rows >= 32 ? 0xffffffffu : (1u << rows) - 1u;
        const __nv_bfloat16 *k = a.c.k + cell + head + (long long)row0 * step, *v = a.c.v + cell + head + (long long)row0 * step;
#pragma unroll
        for (int i = 0; i < CH * VR / 32; ++i) {
          const int row = row0 + i * (32 / VR);
          const bool in = row < rows && col;
          const uint32_t dst = gdn::swz(at, row, vec0 >> 3 & 7);
          ptx::cp_async16(dst, in ? k : a.c.k, in ? 16u : 0u);
          ptx::cp_async16(dst + CH * D * 2, in ? v : a.c.v, in ? 16u : 0u);
          k += (32 / VR) * step;
          v += (32 / VR) * step;
        }
      } else {
        mask = __ballot_sync(0xffffffffu, cell >= 0);
#pragma unroll 1
        for (int i = 0; i < CH * VR / 32; ++i) {
          const int row = row0 + i * (32 / VR);
          const long long from = __shfl_sync(0xffffffffu, cell, row);
          const bool in = from >= 0 && col;
          const long long e = in ? from + head : 0;
          const uint32_t dst = gdn::swz(at, row, vec0 >> 3 & 7);
          ptx::cp_async16(dst, a.c.k + e, in ? 16u : 0u);
          ptx::cp_async16(dst + CH * D * 2, a.c.v + e, in ? 16u : 0u);
        }
      }
      if (lane == 0) s_mask[stage] = mask;
      ++got;
      if (got < w1) {
        next_tile<S::kTile>(get, a.c, R);
        look();
      }
    }
    ptx::cp_async_commit();   // (always a group, so that the groups count the tiles)
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) request(s);

  uint32_t qf[KS][4];
  float o[D / 8][4], m[2], l[2];
  // o and what earlier chains of the head left, relative to the present maximum; `keep`: goes there, and o starts from zero
  auto join_chains = [&](bool earlier, bool keep) {
    float4* at = a.kept + ((long long)blockIdx.x * kWarps + warp) * (D / 8) * 32 + lane;
    float2* max_at = reinterpret_cast<float2*>(a.kept + (long long)a.ctas * kWarps * (D / 8) * 32) + (blockIdx.x * kWarps + warp) * 32 + lane;
    float f[2] = {0.f, 0.f};
    if (earlier) {
      const float2 before = *max_at;
      f[0] = before.x == m[0] ? 1.f : exp2f(before.x - m[0]);
      f[1] = before.y == m[1] ? 1.f : exp2f(before.y - m[1]);
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      if (earlier) {
        const float4 x = at[i * 32];
        o[i][0] = fmaf(x.x, f[0], o[i][0]); o[i][1] = fmaf(x.y, f[0], o[i][1]); o[i][2] = fmaf(x.z, f[1], o[i][2]); o[i][3] = fmaf(x.w, f[1], o[i][3]);
      }
      if (keep) {
        at[i * 32] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
        gdn::zero4(o[i]);
      }
    }
    if (keep) *max_at = make_float2(m[0], m[1]);
  };
  int stage = 0, part = 2 * blockIdx.x;   // where a part is left: the first head's, then the last one's
  for (long long w = w0; w < w1; ++w) {
    if (w == w0 || use.t == 0) {   // a head starts: its queries, nothing seen yet
      const __nv_bfloat16* q = a.q + use.b * a.qs + ((long long)(use.r / a.MT) * a.G + use.r % a.MT * kRows) * a.c.D;
      const int rows = min(kRows, a.G - use.r % a.MT * kRows), r = lane >> 2, c = (lane & 3) * 2;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = r + (e & 1) * 8, col = ks * 16 + c + (e >> 1) * 8;
          qf[ks][e] = row < rows && col < a.c.D ? *reinterpret_cast<const uint32_t*>(q + (long long)row * a.c.D + col) : 0u;
        }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) gdn::zero4(o[i]);
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    }
    request(stage == 0 ? ST - 1 : stage - 1);   // into the stage that was worked through last
    ptx::cp_async_wait<ST - 1>();
    __syncwarp();
    const uint32_t kt = ring + stage * S::kStage, vt = kt + CH * D * 2, mask = s_mask[stage];
    constexpr int NT = CH / 8;   // score tiles of 8 cells
    float s[NT][4] = {};
#pragma unroll
    for (int c = 0; c < NT / 2; ++c) {
      if constexpr (D <= 128) {   // two chains of products, half as long (at 256 there are no registers for it)
        float odd[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < KS; ks += 2) {
          gdn::mma2(s[2 * c], s[2 * c + 1], qf[ks], gdn::ld_b(kt, c * 16, ks, L, kRowBytes));
          gdn::mma2(odd[0], odd[1], qf[ks + 1], gdn::ld_b(kt, c * 16, ks + 1, L, kRowBytes));
        }
        gdn::add4(s[2 * c], odd[0]);
        gdn::add4(s[2 * c + 1], odd[1]);
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) gdn::mma2(s[2 * c], s[2 * c + 1], qf[ks], gdn::ld_b(kt, c * 16, ks, L, kRowBytes));
      }
    }
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool seen = mask >> (j * 8 + (lane & 3) * 2 + (e & 1)) & 1u;
        s[j][e] = seen ? s[j][e] * a.scale_log2 : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[j][e]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
    }
    if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {   // the sums so far, to the new maximum
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float f = m[r] == top[r] ? 1.f : exp2f(m[r] - top[r]);   // (a first maximum: 0; both -inf: 1, of nothing)
        l[r] *= f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][2 * r] *= f;
          o[i][2 * r + 1] *= f;
        }
        m[r] = top[r];
      }
    }
    uint32_t p[NT / 2][4];
    {
      const float z0 = m[0] == -INFINITY ? 0.f : m[0], z1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float p0 = exp2f(s[j][0] - z0), p1 = exp2f(s[j][1] - z0), p2 = exp2f(s[j][2] - z1), p3 = exp2f(s[j][3] - z1);
        l[0] += p0 + p1;
        l[1] += p2 + p3;
        p[j / 2][j % 2 * 2] = pack_bf16(p0, p1);
        p[j / 2][j % 2 * 2 + 1] = pack_bf16(p2, p3);
      }
    }
#pragma unroll
    for (int c = 0; c < NT / 2; ++c)
#pragma unroll
      for (int np = 0; np < D / 16; ++np) gdn::mma2(o[2 * np], o[2 * np + 1], p[c], gdn::ld_b_t(vt, c * 16, np, L, kRowBytes));
    __syncwarp();   // (the stage may be written again)
    stage = stage + 1 == ST ? 0 : stage + 1;

    const bool ends = use.t + 1 == use.nt || w + 1 == w1;   // the head, or this CTA's share of it
    if (LONG && __builtin_expect((use.t + 1) % S::kChain == 0 || (ends && use.t >= S::kChain), 0)) {
      const int first = max(0, use.t - (int)min(w - w0, (long long)use.t));   // the share's first tile
      const bool earlier = first / S::kChain != use.t / S::kChain;
      if (earlier || !ends) join_chains(earlier, !ends);
    }
    if (ends) {
      const int rows = min(kRows, a.G - use.r % a.MT * kRows), r0 = lane >> 2;
      const bool from_start = w - w0 >= use.t, whole = from_start && use.t + 1 == use.nt;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if ((lane & 3) == 0) {
          s_m[warp * kRows + r0 + r * 8] = m[r];
          s_l[warp * kRows + r0 + r * 8] = l[r];
        }
      }
      __syncthreads();
      float f[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mm = -INFINITY;
#pragma unroll
        for (int x = 0; x < kWarps; ++x) mm = fmaxf(mm, s_m[x * kRows + r0 + r * 8]);
        f[r] = m[r] == -INFINITY ? 0.f : m[r] == mm ? 1.f : exp2f(m[r] - mm);
      }
      const int row = threadIdx.x >> 3, c4 = (threadIdx.x & 7) * 4;   // what this thread joins: 4 columns of a row
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) mm = fmaxf(mm, s_m[x * kRows + row % kRows]);
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float mx = s_m[x * kRows + row % kRows], lx = s_l[x * kRows + row % kRows];
        ll += mx == -INFINITY ? lx * 0.f : lx * (mx == mm ? 1.f : exp2f(mx - mm));
      }
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += kJoinCols) {
#pragma unroll
        for (int i = 0; i < kJoinCols / 8; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            *reinterpret_cast<float2*>(s_o + (warp * kRows + r0 + r * 8) * kJoinCols + i * 8 + (lane & 3) * 2) =
                make_float2(o[c0 / 8 + i][2 * r] * f[r], o[c0 / 8 + i][2 * r + 1] * f[r]);
        __syncthreads();
        if (row < rows && c0 + c4 < a.c.D) {   // (16 rows, the first 128 threads)
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < kWarps; ++x) {
            const float4 v = *reinterpret_cast<const float4*>(s_o + (x * kRows + row) * kJoinCols + c4);
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
          }
          if (whole) {
            const long long at = ((long long)use.b * a.Hq + (use.r / a.MT) * a.G + use.r % a.MT * kRows + row) * a.c.D + c0 + c4;
            *reinterpret_cast<uint2*>(a.o + at) = make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv));
          } else {
            *reinterpret_cast<float4*>(a.part + ((long long)part * kRows + row) * a.c.D + c0 + c4) = sum;
          }
        }
        __syncthreads();
      }
      if (!whole && row < kRows && (threadIdx.x & 7) == 0) {
        float* stats = a.part + (long long)2 * a.ctas * kRows * a.c.D + part * kRows + row;
        stats[0] = mm;
        stats[2 * a.ctas * kRows] = ll;
      }
      __syncthreads();   // (s_m and s_l may be written again)
      part = 2 * blockIdx.x + 1;
    }
    if (w + 1 < w1) next_tile<S::kTile>(use, a.c, R);
  }
  ptx::cp_async_wait_all();
  if (bad) raise_status(LEWI_STATUS_BAD_INDEX);
}

// Adds up the parts of the heads that several CTAs worked on, in a fixed order, and writes zeros for sequences without cells.  `PER` warps
// work on a query head and take every PER-th part each: 8 for few heads (one sequence of 100,001, 32 heads, the whole call: 73 us, with one
// 83), one for many (64 sequences x 32 heads: 111, with eight 113).
constexpr int kJoinWarps = 8;
template <int TILE, int PER>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const Args a) {
  __shared__ long long s_count[2][kJoinWarps];
  __shared__ float s_m[kJoinWarps], s_l[kJoinWarps];
  __shared__ float4 s_sum[PER > 1 ? kJoinWarps : 1][64];
  const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = a.c.Hkv * a.MT;
  const int head = blockIdx.x * (kJoinWarps / PER) + warp / PER, mine = warp % PER;
  const longlong2 count = count_tiles<TILE, kJoinWarps>(a.c, b, s_count);
  const int nt = tiles_of<TILE>(a.c, b);
  grid_wait();   // (every CTA, so that what follows this kernel follows the one before it, too)
  if (threadIdx.x == 0 && blockIdx.x == 0 && a.c.lengths[b] > (long long)a.c.max_pages * a.c.page) raise_status(LEWI_STATUS_BAD_INDEX);
  if (head >= a.Hq) return;   // (whole warps, and only where each has a head of its own)
  __nv_bfloat16* o = a.o + ((long long)b * a.Hq + head) * a.c.D;
  if (nt == 0) {
    for (int c = (mine * 32 + lane) * 4; c < a.c.D; c += PER * 128) *reinterpret_cast<uint2*>(o + c) = make_uint2(0u, 0u);
    return;
  }
  const int g = head % a.G, row = g % kRows;
  const long long total = count.x * R, w0 = count.y * R + (long long)((head / a.G) * a.MT + g / kRows) * nt, w1 = w0 + nt;
  const long long n_ctas = min(total, (long long)a.ctas);
  auto cta_of = [&](long long w) { return (int)(((w + 1) * n_ctas - 1) / total); };
  const int c0 = cta_of(w0), c1 = cta_of(w1 - 1);
  if (c0 == c1) return;   // written already
  const int slot0 = 2 * c0 + (w0 == c0 * total / n_ctas ? 0 : 1);   // (every other CTA's run starts inside the head)
  const float* stats = a.part + (long long)2 * a.ctas * kRows * a.c.D + row;
  auto slot_of = [&](int c) { return c == c0 ? slot0 : 2 * c; };
  float mm = -INFINITY;
  for (int c = c0 + mine * 32 + lane; c <= c1; c += PER * 32) mm = fmaxf(mm, stats[slot_of(c) * kRows]);
  mm = warp_max(mm);
  if constexpr (PER > 1) {
    if (lane == 0) s_m[warp] = mm;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kJoinWarps; ++x) mm = fmaxf(mm, s_m[x]);
  }
  float ll = 0.f;
  float4 sum[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};   // columns 4 lane, 128 + 4 lane
#pragma unroll 8
  for (int c = c0 + mine; c <= c1; c += PER) {
    const float mx = stats[slot_of(c) * kRows], lx = stats[(2 * a.ctas + slot_of(c)) * kRows];
    const float f = mx == -INFINITY ? 0.f : mx == mm ? 1.f : exp2f(mx - mm);
    const float* part = a.part + ((long long)slot_of(c) * kRows + row) * a.c.D;
    ll = fmaf(f, lx, mx == -INFINITY ? lx * 0.f + ll : ll);   // (an lx that is not finite is not lost)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (h * 128 + lane * 4 < a.c.D) {
        const float4 v = *reinterpret_cast<const float4*>(part + h * 128 + lane * 4);
        sum[h].x = fmaf(f, v.x, sum[h].x); sum[h].y = fmaf(f, v.y, sum[h].y); sum[h].z = fmaf(f, v.z, sum[h].z); sum[h].w = fmaf(f, v.w, sum[h].w);
      }
  }
  if constexpr (PER > 1) {
    if (lane == 0) s_l[warp] = ll;
#pragma unroll
    for (int h = 0; h < 2; ++h) s_sum[warp][h * 32 + lane] = sum[h];
    __syncthreads();
    if (warp > 0) return;
    ll = 0.f;
    sum[0] = sum[1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < kJoinWarps; ++x) {
      ll += s_l[x];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 y = s_sum[x][h * 32 + lane];
        sum[h].x += y.x; sum[h].y += y.y; sum[h].z += y.z; sum[h].w += y.w;
      }
    }
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (h * 128 + lane * 4 < a.c.D)
      *reinterpret_cast<uint2*>(o + h * 128 + lane * 4) = make_uint2(pack_bf16(sum[h].x * inv, sum[h].y * inv), pack_bf16(sum[h].z * inv, sum[h].w * inv));
}

}  // namespace paged
}  // namespace lewi
