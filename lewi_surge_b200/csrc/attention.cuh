// Causal attention over packed sequences, forward and backward, on the tensor cores (tcgen05).
//
// q, o [T][Hq][D], k, v [T][Hkv][D] bf16; sequence s has the rows cu[s] .. cu[s+1], query head h the keys of head h / G, G = Hq / Hkv.
//   S = scale Q K^T (keys up to the query's own),  P = exp(S - lse),  O = P V
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),  delta = rowsum(dO O),  dQ = scale dS K,  dK = scale dS^T Q
// Everything works on tiles of 128 rows that start at a multiple of 128 within their sequence, so that only the tile pair on the diagonal
// is masked and a sequence's end can only lie in it.  A row of S or dS belongs to one thread (tensor memory lane = row): a maximum or
// a sum over a row needs no other thread.  P and dS go back to tensor memory as bf16, where they are the A operand of the next
// product; scores, softmax, sums and accumulators are float32.  Rows behind a sequence's end that a tile reaches into belong to
// somebody else (or to nobody): of operands that are summed over them they are set to zero after their copy has landed.  Within its own
// sequence a value of v that is not finite reaches back to the start of its tile (0 times it is not 0), as q, k, v and dO do in the
// gradients.
#pragma once

#include "common.cuh"
#include "f32x2.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace lewi {
namespace attn {

constexpr int kTile = 128;
constexpr int kMaxD = 128;

// ---------------------------------------------------------------- which tiles there are
struct Seqs {
  const int32_t* cu;   // null: n sequences of T / n rows
  int n, T;
};
struct Rows {
  int start, len;
};
__device__ __forceinline__ Rows rows_of(const Seqs& q, int s) {
  if (q.cu == nullptr) return {q.T / q.n * s, q.T / q.n};
  const int lo = min(max(q.cu[s], 0), q.T), hi = min(max(q.cu[s + 1], lo), q.T);
  if (lo != q.cu[s] || hi != q.cu[s + 1]) raise_status(LEWI_STATUS_BAD_INDEX);
  return {lo, hi - lo};
}

struct Work {
  int start, len, level;   // the sequence's rows; level < its number of units
  bool any;
};

// The x-th unit of work in the order of falling levels, where sequence s has the levels 0 .. units(tiles of s) - 1 and a level's work
// grows with it: long runs first, whatever the lengths, without a table.  F(i) = sum_s max(0, units - i) counts the units of level i and
// above; the level is the largest i with F(i) > x, and the sequence the (x - F(i + 1))-th of those that have it.  All threads call it.
template <int THREADS, class U>
__device__ __forceinline__ Work find_work(const Seqs& q, int x, U units) {
  constexpr int WARPS = THREADS / 32;
  __shared__ int s_part[2][WARPS];
  __shared__ int s_hit;
  if (q.cu == nullptr) {
    const int len = q.T / q.n, u = units((len + kTile - 1) / kTile), level = u - 1 - x / q.n;
    return {len * (x % q.n), len, level, level >= 0};
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto units_of = [&](int s) { return units((rows_of(q, s).len + kTile - 1) / kTile); };
  if (q.n == 1) {
    const Rows r = rows_of(q, 0);
    const int level = units((r.len + kTile - 1) / kTile) - 1 - x;
    return {r.start, r.len, level, level >= 0};
  }
  if (q.n <= 32) {   // a sequence per lane, every warp for itself
    const int u = lane < q.n ? units_of(lane) : 0;
    auto count = [&](int i) { return __reduce_add_sync(0xffffffffu, max(0, u - i)); };
    if (count(0) <= x) return {0, 0, 0, false};
    int lo = 0, hi = __reduce_max_sync(0xffffffffu, u);   // F(lo) > x, F(hi) = 0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (count(mid) > x) lo = mid;
      else hi = mid;
    }
    unsigned have = __ballot_sync(0xffffffffu, u > lo);
    for (int r = x - count(lo + 1); r > 0; --r) have &= have - 1;
    const Rows r = rows_of(q, __ffs(have) - 1);
    return {r.start, r.len, lo, true};
  }
  // runs of sequences per thread
  const int per = (q.n + THREADS - 1) / THREADS, s0 = min(q.n, (int)threadIdx.x * per), s1 = min(q.n, s0 + per);
  int flip = 0;
  auto block_sum = [&](int v) {
    const int w = __reduce_add_sync(0xffffffffu, v);
    if (lane == 0) s_part[flip][warp] = w;
    __syncthreads();
    int sum = 0;
    for (int i = 0; i < WARPS; ++i) sum += s_part[flip][i];
    flip ^= 1;
    return sum;
  };
  auto mine = [&](int i) {
    int v = 0;
    for (int s = s0; s < s1; ++s) v += max(0, units_of(s) - i);
    return v;
  };
  if (block_sum(mine(0)) <= x) return {0, 0, 0, false};
  int lo = 0, hi = units((q.T + kTile - 1) / kTile) + 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (block_sum(mine(mid)) > x) lo = mid;
    else hi = mid;
  }
  int rank = x - block_sum(mine(lo + 1)), have = 0;
  for (int s = s0; s < s1; ++s) have += units_of(s) > lo;
  int upto = have;   // of this warp's threads up to this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) s_part[flip][warp] = upto;
  if (threadIdx.x == 0) s_hit = 0;
  __syncthreads();
  for (int i = 0; i < warp; ++i) upto += s_part[flip][i];
  if (rank >= upto - have && rank < upto) {
    rank -= upto - have;
    for (int s = s0; s < s1; ++s)
      if (units_of(s) > lo && rank-- == 0) s_hit = s;
  }
  __syncthreads();
  const Rows r = rows_of(q, s_hit);
  return {r.start, r.len, lo, true};
}

// Rows of no sequence become zero: a share of them for every CTA, `vecs` 16-byte pieces each.
__device__ __forceinline__ void zero_gaps(const Seqs& q, __nv_bfloat16* out, int vecs, int threads) {
  if (q.cu == nullptr || threadIdx.x >= threads) return;
  const int first = min(max(q.cu[0], 0), q.T), end = min(max(q.cu[q.n], 0), q.T);
  for (int r = blockIdx.x; r < q.T; r += gridDim.x) {
    if (r >= first && r < end) r += (end - r + gridDim.x - 1) / gridDim.x * gridDim.x;
    if (r >= q.T) break;
    for (int i = threadIdx.x; i < vecs; i += threads) st_v4(out + ((long long)r * vecs + i) * 8, make_uint4(0u, 0u, 0u, 0u));
  }
}

// ---------------------------------------------------------------- pieces
// 2^(x scale + shift) of two scores.  The special function unit gives 16 a cycle and SM, so 128 x 128 of them take as long as two products
// of 128 x 128 x 128; every OF-th pair is made by multiply-adds instead (0: none).
template <int OF>
__device__ __forceinline__ F2 ex2_pair(uint32_t x0, uint32_t x1, F2 scale, F2 shift, int pair) {
  const F2 x = fma2(f2(__uint_as_float(x0), __uint_as_float(x1)), scale, shift);
  if (OF > 0 && pair % (OF > 0 ? OF : 1) == OF - 1) return ex2_poly(x);
  float lo, hi;
  f2_split(x, lo, hi);
  return f2(ex2(lo), ex2(hi));
}
// The backward pass does so where D <= 64, whose products are half as long (T = 8192, 32 heads over 8: dQ 488 -> 465, dK and dV 695 ->
// 670 us); at D = 128 it costs (dQ 648 -> 661, dK and dV 845 -> 875 us).
template <int DP> constexpr int kBwdPoly = DP == 64 ? 4 : 0;

__device__ __forceinline__ F2 hide(F2 v, bool lo_hidden, bool hi_hidden) {
  float lo, hi;
  f2_split(v, lo, hi);
  return f2(lo_hidden ? 0.f : lo, hi_hidden ? 0.f : hi);
}
// Operand tiles in shared memory: boxes of [128 rows][64 columns], 128-byte swizzled, 16 KB apart.
constexpr int kBox = kTile * 128;
template <int DP> constexpr int kTileBytes = kTile * DP * 2;
// K-major (rows are M or N, columns K) and MN-major (rows are K, columns N)
__device__ __forceinline__ uint64_t desc_k(uint32_t tile, int step) {
  return ptx::smem_desc(ptx::smem_desc_hi_sw128(16, 1024), tile + (step >> 2) * kBox + (step & 3) * 32);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, int step) {
  return ptx::smem_desc(ptx::smem_desc_hi_sw128(kBox, 1024), tile + step * 2048);
}
// D (+)= A B over the DP columns of two tiles
template <int DP>
__device__ __forceinline__ void mma_kk(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) ptx::mma_bf16(d, desc_k(a, i), desc_k(b, i), idesc, i > 0);
}
// D (+)= A B over steps [I0, I1) of the 128 rows of a tile; A in tensor memory, its second 64 columns `gap` columns after the first
template <int I0, int I1>
__device__ __forceinline__ void mma_tm(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate, int gap) {
#pragma unroll
  for (int i = I0; i < I1; ++i) ptx::mma_bf16_ta(d, a + (i >> 2) * gap + (i & 3) * 8, desc_mn(b, i), idesc, accumulate || i > I0);
}

template <int DP>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int head, int row) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) ptx::tma_load_3d(dst + c * kBox, tm, bar, c * 64, head, row);
}

// A wait of a whole warp: all lanes get the same answer.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, abort_flag));
}

// What a warp that brings tiles does for one of them.  `valid` rows belong to the sequence; the others are zeroed once the copy has
// landed (on a barrier of the warp's own), and the tile is handed on after that.
template <int DP>
__device__ __forceinline__ bool bring_tile(uint32_t dst, const CUtensorMap* tm, uint32_t full, uint32_t raw, uint32_t& raw_phase, int head, int row,
                                           int valid, volatile int* abort_flag) {
  const bool whole = valid >= kTile;
  if (ptx::elect_one()) {
    ptx::mbar_expect_tx(whole ? full : raw, kTileBytes<DP>);
    load_tile<DP>(dst, tm, whole ? full : raw, head, row);
  }
  __syncwarp();
  if (whole) return true;
  if (!warp_wait(raw, raw_phase, abort_flag)) return false;
  raw_phase ^= 1u;
  for (int i = (threadIdx.x & 31); i < (kTile - valid) * (DP / 8); i += 32) {
    const uint32_t at = dst + (i & 7) * 16 + ((i >> 3) / (kTile - valid)) * kBox + (valid + (i >> 3) % (kTile - valid)) * 128;
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory");
  }
  ptx::fence_proxy_async();
  __syncwarp();
  if (ptx::elect_one()) ptx::mbar_arrive(full);
  __syncwarp();
  return true;
}

// Gives what is still in flight a bounded time to land before shared memory is left (after a wait that ran out).
__device__ __forceinline__ void settle() {
  const unsigned long long t0 = ptx::globaltimer_ns();
  while (ptx::globaltimer_ns() - t0 < 4000000ull) {}
}

struct Args {
  Seqs seqs;
  int Hq, Hkv, G, D;
  float scale, scale_log2;
  __nv_bfloat16* o;        // [T][Hq][D]
  float *lse, *delta;      // [Hq][T], lse in units of log 2
  __nv_bfloat16 *dq, *dk, *dv;
  int parts;               // of a group's heads, one CTA each for dK and dV
  float* sums;             // [part][dV, dK][T][Hkv][D] where there are several
};

__device__ __forceinline__ void store_row32(__nv_bfloat16* dst, const uint32_t (&v)[32], float f, int cols) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i * 8 < cols)
      st_v4(dst + i * 8, make_uint4(pack_bf16(__uint_as_float(v[8 * i]) * f, __uint_as_float(v[8 * i + 1]) * f),
                                    pack_bf16(__uint_as_float(v[8 * i + 2]) * f, __uint_as_float(v[8 * i + 3]) * f),
                                    pack_bf16(__uint_as_float(v[8 * i + 4]) * f, __uint_as_float(v[8 * i + 5]) * f),
                                    pack_bf16(__uint_as_float(v[8 * i + 6]) * f, __uint_as_float(v[8 * i + 7]) * f)));
}

__device__ __forceinline__ void store_part32(float* dst, const uint32_t (&v)[32], float f, int cols) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 4 < cols)
      *reinterpret_cast<float4*>(dst + i * 4) = make_float4(__uint_as_float(v[4 * i]) * f, __uint_as_float(v[4 * i + 1]) * f,
                                                            __uint_as_float(v[4 * i + 2]) * f, __uint_as_float(v[4 * i + 3]) * f);
}

// ---------------------------------------------------------------- forward
// A CTA works on two tiles of queries that share their keys (two heads, or two tiles of one head): while one tile's softmax is made by its
// four warps, the tensor cores multiply for the other, and every key and value tile that is brought serves both.  Warps 0-3 and 4-7: a
// row of S per thread; warp 8: TMA; warp 9: MMA.  Products are issued in the order S0(j+1) after P0 V(j), S1(j+1) after P1 V(j): a
// softmax that finds its scores knows that the product before them is done, so it may scale O then.  It does so only where the
// maximum has grown by more than 8 (in powers of 2; p stays below 2^8, which bf16 and float32 hold as well as 1).
constexpr int kFwdThreads = 384;   // (warps 10 and 11 have nothing to do: registers move between warpgroups of four warps)
template <int DP>
struct FwdShape {
  static constexpr int kStages = DP == 64 ? 6 : 5;
  static constexpr int kSmem = 2 * kTileBytes<DP> + kStages * kTileBytes<DP> + 256;
};

template <int DP>
__global__ void __launch_bounds__(kFwdThreads, 1) fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                                             const __grid_constant__ CUtensorMap tm_v, const Args a) {
  constexpr int ST = FwdShape<DP>::kStages, TB = kTileBytes<DP>;
  extern __shared__ __align__(1024) uint8_t attn_smem[];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t base = ptx::smem_u32(attn_smem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) raise_status(LEWI_STATUS_SMEM_LAYOUT);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int hk = blockIdx.x % a.Hkv;
  zero_gaps(a.seqs, a.o, a.Hq * a.D / 8, kFwdThreads);
  const Work w = find_work<kFwdThreads>(a.seqs, blockIdx.x / a.Hkv, [&](int tiles) { return (tiles * a.G + 1) / 2; });
  if (!w.any) return;
  // the two tiles: units 2 level and 2 level + 1 of the sequence's tiles x heads
  const int tiles = (w.len + kTile - 1) / kTile;
  int tile[2], head[2], blocks[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int u = 2 * w.level + t;
    tile[t] = u / a.G;
    head[t] = hk * a.G + u % a.G;
    blocks[t] = tile[t] < tiles ? tile[t] + 1 : 0;
  }
  const int nb = max(blocks[0], blocks[1]);

  const uint32_t kv = base + 2 * TB, bars = kv + ST * TB;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (ST + s); };
  auto q_full = [&](int t) { return bars + 8u * (2 * ST + t); };
  auto s_full = [&](int t) { return bars + 8u * (2 * ST + 2 + t); };
  auto p_full = [&](int t, int half) { return bars + 8u * (2 * ST + 4 + 2 * t + half); };
  auto o_full = [&](int t) { return bars + 8u * (2 * ST + 8 + t); };
  const uint32_t raw = bars + 8u * (2 * ST + 10);
  volatile int* abort_flag = &s_abort;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      ptx::mbar_init(full(s), 1);
      ptx::mbar_init(empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(q_full(t), 1);
      ptx::mbar_init(s_full(t), 1);
      ptx::mbar_init(p_full(t, 0), 4);
      ptx::mbar_init(p_full(t, 1), 4);
      ptx::mbar_init(o_full(t), 1);
    }
    ptx::mbar_init(raw, 1);
    s_abort = 0;
    ptx::mbar_fence_init();
    ptx::fence_proxy_async();
    ptx::prefetch_tensormap(&tm_q);
    ptx::prefetch_tensormap(&tm_k);
    ptx::prefetch_tensormap(&tm_v);
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem;
  auto s_at = [&](int t) { return tmem + t * 128; };
  auto o_at = [&](int t) { return tmem + 256 + t * 128; };

  // registers: 8 x 216 + 4 x 72 = 12 x 168 a thread, what the launch has
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 8) {
    // ---------------------------------------------------------------- queries, then K0, V0, K1, V1, ..
    bool ok = true;
    if (ptx::elect_one()) {
      for (int t = 0; t < 2; ++t)
        if (blocks[t] > 0) {
          ptx::mbar_expect_tx(q_full(t), TB);
          load_tile<DP>(base + t * TB, &tm_q, q_full(t), head[t], w.start + tile[t] * kTile);
        }
    }
    __syncwarp();
    uint32_t raw_phase = 0;
    for (int n = 0; ok && n < 2 * nb; ++n) {
      const int s = n % ST, j = n >> 1;
      ok = warp_wait(empty(s), (n / ST & 1) ^ 1u, abort_flag);
      if (!ok) break;
      const int valid = (n & 1) != 0 ? w.len - j * kTile : kTile;   // (of K a foreign row only reaches scores that are masked)
      ok = bring_tile<DP>(kv + s * TB, (n & 1) != 0 ? &tm_v : &tm_k, full(s), raw, raw_phase, hk, w.start + j * kTile, valid, abort_flag);
    }
    if (!ok) settle();
  } else if (warp == 9) {
    // ---------------------------------------------------------------- products
    const uint32_t id_s = ptx::instr_desc_bf16(128, 128, 0, 0), id_o = ptx::instr_desc_bf16(128, DP, 0, 1);
    if (ptx::elect_one()) {
      bool ok = ptx::mbar_wait(full(0), 0, abort_flag);
      auto scores = [&](int t, int s) {
        ptx::tc_fence_after();
        mma_kk<DP>(s_at(t), base + t * TB, kv + s * TB, id_s);
        ptx::mma_commit(s_full(t));
      };
      for (int t = 0; ok && t < 2; ++t)
        if (blocks[t] > 0) {
          ok = ptx::mbar_wait(q_full(t), 0, abort_flag);
          if (ok) scores(t, 0);
        }
      if (ok) ptx::mma_commit(empty(0));
      for (int j = 0; ok && j < nb; ++j) {
        const int nv = 2 * j + 1, nk = nv + 1, sv = nv % ST, sk = nk % ST;
        ok = ptx::mbar_wait(full(sv), nv / ST & 1, abort_flag);
        for (int t = 0; ok && t < 2; ++t) {
          if (j >= blocks[t]) continue;
          ok = ptx::mbar_wait(p_full(t, 0), j & 1, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after();
          mma_tm<0, 4>(o_at(t), s_at(t), kv + sv * TB, id_o, j > 0, 32);
          ok = ptx::mbar_wait(p_full(t, 1), j & 1, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after();
          mma_tm<4, 8>(o_at(t), s_at(t), kv + sv * TB, id_o, true, 32);
          if (j + 1 < blocks[t]) {
            ok = ptx::mbar_wait(full(sk), nk / ST & 1, abort_flag);
            if (ok) scores(t, sk);
          } else {
            ptx::mma_commit(o_full(t));
          }
        }
        if (!ok) break;
        ptx::mma_commit(empty(sv));
        if (j + 1 < nb) ptx::mma_commit(empty(sk));
      }
      if (!ok) settle();
    }
    __syncwarp();
  }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2, row = (warp & 3) * 32 + lane, n_blocks = blocks[t];
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // this warp's lanes of tensor memory
    const uint32_t sp = s_at(t) + lanes, op = o_at(t) + lanes;
    float m = 0.f, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_blocks; ++j) {
      ok = warp_wait(s_full(t), j & 1, abort_flag);
      if (!ok) break;
      ptx::tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(sp + c * 32, s[c]);
      ptx::tmem_ld_wait();
      if (j == tile[t]) {   // the diagonal: keys behind the query
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i > row) s[c][i] = 0xff800000u;
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
        for (int i = 1; i < 32; ++i) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][i]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      if (j == 0) {
        m = top;
      } else if (__any_sync(0xffffffffu, (top - m) * a.scale_log2 > 8.f)) {
        const float grown = fmaxf(m, top), f = grown == m ? 1.f : ex2((m - grown) * a.scale_log2);
        m = grown;
        l *= f;
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          uint32_t v[32];
          ptx::tmem_ld_32x32(op + c, v);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
          ptx::tmem_st_32x32(op + c, v);
        }
        ptx::tmem_st_wait();
      }
      const F2 scale = f2(a.scale_log2, a.scale_log2), shift = f2(-m * a.scale_log2, -m * a.scale_log2);
      F2 sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t p[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const F2 x = ex2_pair<4>(s[2 * half + i / 16][i % 16 * 2], s[2 * half + i / 16][i % 16 * 2 + 1], scale, shift, i);
          sum[i & 1] = add2(sum[i & 1], x);
          p[i] = f2_bf16(x);
        }
        ptx::tmem_st_32x32(sp + half * 32, p);
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_full(t, half));
      }
      float lo, hi;
      f2_split(add2(sum[0], sum[1]), lo, hi);
      l += lo + hi;
    }
    if (ok && n_blocks > 0) ok = warp_wait(o_full(t), 0, abort_flag);
    if (ok && n_blocks > 0) {
      ptx::tc_fence_after();
      const int in_seq = tile[t] * kTile + row;
      const long long r = w.start + in_seq;
      const float inv = 1.f / l;
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        uint32_t v[32];
        ptx::tmem_ld_32x32(op + c, v);
        ptx::tmem_ld_wait();
        if (in_seq < w.len) store_row32(a.o + (r * a.Hq + head[t]) * a.D + c, v, inv, a.D - c);
      }
      if (in_seq < w.len) a.lse[(long long)head[t] * a.seqs.T + r] = m * a.scale_log2 + log2f(l);
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- backward: delta
// delta[h][t] = sum_d dO O, DP / 8 lanes per row.
constexpr int kDeltaThreads = 256;
template <int DP>
__global__ void __launch_bounds__(kDeltaThreads) delta_kernel(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ d_o,
                                                              float* __restrict__ delta, int T, int Hq, int D) {
  constexpr int L = DP / 8;
  const long long row = ((long long)blockIdx.x * kDeltaThreads + threadIdx.x) / L;
  const int c = threadIdx.x % L * 8;
  const bool live = row < (long long)T * Hq;
  float sum = 0.f;
  if (live && c < D) {
    const uint4 x = ld_nc_v4(o + row * D + c), y = ld_nc_v4(d_o + row * D + c);
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fmaf(bf16_lo(xs[i]), bf16_lo(ys[i]), fmaf(bf16_hi(xs[i]), bf16_hi(ys[i]), sum));
  }
#pragma unroll
  for (int s = L / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  if (live && c == 0) delta[row % Hq * T + row / Hq] = sum;
}

// ---------------------------------------------------------------- backward: dK and dV
// A CTA has one tile of keys and works through the queries that see it, head by head of the group (or of a part of it: dkv_parts), so that
// dK and dV stay in tensor memory and no sum needs an atomic.  Scores transposed (a row is a key): P^T and dS^T are the A operands of dV = P^T dO and dK = dS^T Q.
// Warps 0-7: elementwise, a thread has 64 of the 128 queries of a row; warp 8: TMA; warp 9: MMA; warp 10: lse and delta.
// Order of products: S(0) dP(0) | dV(i) S(i+1) after P(i), dK(i) dP(i+1) after dS(i): exponentials are made while dK and dP run,
// dS while dV and S do.
constexpr int kBwdThreads = 352;
template <int DP>
struct DkvShape {
  static constexpr int kStages = 2;
  static constexpr int kSmem = (2 + 2 * kStages) * kTileBytes<DP> + kStages * 2 * kTile * 4 + 256;
};

template <int DP>
__global__ void __launch_bounds__(kBwdThreads, 1) dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                                             const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                                                             const Args a) {
  constexpr int ST = DkvShape<DP>::kStages, TB = kTileBytes<DP>;
  extern __shared__ __align__(1024) uint8_t attn_smem[];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t base = ptx::smem_u32(attn_smem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) raise_status(LEWI_STATUS_SMEM_LAYOUT);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int hk = blockIdx.x % a.Hkv, part = blockIdx.x / a.Hkv % a.parts;
  zero_gaps(a.seqs, a.dk, a.Hkv * a.D / 8, kBwdThreads);
  zero_gaps(a.seqs, a.dv, a.Hkv * a.D / 8, kBwdThreads);
  const Work w = find_work<kBwdThreads>(a.seqs, blockIdx.x / (a.Hkv * a.parts), [](int tiles) { return tiles; });
  if (!w.any) return;
  const int head0 = part * a.G / a.parts, heads = (part + 1) * a.G / a.parts - head0;   // of the group
  const int tiles = (w.len + kTile - 1) / kTile, key_tile = tiles - 1 - w.level, per_head = w.level + 1, n_it = per_head * heads;
  auto head_of = [&](int it) { return hk * a.G + head0 + it / per_head; };
  auto tile_of = [&](int it) { return key_tile + it % per_head; };

  const uint32_t k_at = base, v_at = base + TB, ring = base + 2 * TB;   // [stage][Q, dO]
  float* stats = reinterpret_cast<float*>(attn_smem + (2 + 2 * ST) * TB);   // [stage][lse, delta][128]
  const uint32_t bars = base + (2 + 2 * ST) * TB + ST * 2 * kTile * 4;
  const uint32_t k_full = bars, v_full = bars + 8, s_full = bars + 16, dp_full = bars + 24, p_ready = bars + 32, ds_ready = bars + 40, done = bars + 48,
                 raw = bars + 56;
  auto q_full = [&](int s) { return bars + 64u + 8u * s; };
  auto q_empty = [&](int s) { return bars + 64u + 8u * (ST + s); };
  auto do_full = [&](int s) { return bars + 64u + 8u * (2 * ST + s); };
  auto do_empty = [&](int s) { return bars + 64u + 8u * (3 * ST + s); };
  auto st_full = [&](int s) { return bars + 64u + 8u * (4 * ST + s); };
  auto st_empty = [&](int s) { return bars + 64u + 8u * (5 * ST + s); };
  volatile int* abort_flag = &s_abort;
  if (threadIdx.x == 0) {
    for (uint32_t b : {k_full, v_full, s_full, dp_full, done, raw}) ptx::mbar_init(b, 1);
    ptx::mbar_init(p_ready, 8);
    ptx::mbar_init(ds_ready, 8);
    for (int s = 0; s < ST; ++s) {
      ptx::mbar_init(q_full(s), 1);
      ptx::mbar_init(q_empty(s), 1);
      ptx::mbar_init(do_full(s), 1);
      ptx::mbar_init(do_empty(s), 1);
      ptx::mbar_init(st_full(s), 1);
      ptx::mbar_init(st_empty(s), 8);
    }
    s_abort = 0;
    ptx::mbar_fence_init();
    ptx::fence_proxy_async();
    ptx::prefetch_tensormap(&tm_q);
    ptx::prefetch_tensormap(&tm_k);
    ptx::prefetch_tensormap(&tm_v);
    ptx::prefetch_tensormap(&tm_do);
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem, t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 384;

  if (warp == 8) {
    bool ok = true;
    if (ptx::elect_one()) {
      ptx::mbar_expect_tx(k_full, TB);
      load_tile<DP>(k_at, &tm_k, k_full, hk, w.start + key_tile * kTile);
      ptx::mbar_expect_tx(v_full, TB);
      load_tile<DP>(v_at, &tm_v, v_full, hk, w.start + key_tile * kTile);
    }
    __syncwarp();
    uint32_t raw_phase = 0;
    for (int it = 0; ok && it < n_it; ++it) {
      const int s = it % ST, row = tile_of(it) * kTile;
      const uint32_t ph = (it / ST & 1) ^ 1u;
      ok = warp_wait(q_empty(s), ph, abort_flag) &&
           bring_tile<DP>(ring + 2 * s * TB, &tm_q, q_full(s), raw, raw_phase, head_of(it), w.start + row, w.len - row, abort_flag) &&
           warp_wait(do_empty(s), ph, abort_flag) &&
           bring_tile<DP>(ring + (2 * s + 1) * TB, &tm_do, do_full(s), raw, raw_phase, head_of(it), w.start + row, w.len - row, abort_flag);
    }
    if (!ok) settle();
  } else if (warp == 9) {
    const uint32_t id_s = ptx::instr_desc_bf16(128, 128, 0, 0), id_d = ptx::instr_desc_bf16(128, DP, 0, 1);
    if (ptx::elect_one()) {
      auto scores = [&](int it) {   // S^T = K Q^T
        const int s = it % ST;
        if (!ptx::mbar_wait(q_full(s), it / ST & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        mma_kk<DP>(t_s, k_at, ring + 2 * s * TB, id_s);
        ptx::mma_commit(s_full);
        return true;
      };
      auto dps = [&](int it) {   // dP^T = V dO^T
        const int s = it % ST;
        if (!ptx::mbar_wait(do_full(s), it / ST & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        mma_kk<DP>(t_dp, v_at, ring + (2 * s + 1) * TB, id_s);
        ptx::mma_commit(dp_full);
        return true;
      };
      bool ok = ptx::mbar_wait(k_full, 0, abort_flag) && scores(0) && ptx::mbar_wait(v_full, 0, abort_flag) && dps(0);
      for (int it = 0; ok && it < n_it; ++it) {
        const int s = it % ST;
        ok = ptx::mbar_wait(p_ready, it & 1, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after();
        mma_tm<0, 8>(t_dv, t_s, ring + (2 * s + 1) * TB, id_d, it > 0, 64);
        ptx::mma_commit(do_empty(s));
        if (it + 1 < n_it) ok = scores(it + 1);
        ok = ok && ptx::mbar_wait(ds_ready, it & 1, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after();
        mma_tm<0, 8>(t_dk, t_dp, ring + 2 * s * TB, id_d, it > 0, 64);
        ptx::mma_commit(it + 1 < n_it ? q_empty(s) : done);
        if (it + 1 < n_it) ok = dps(it + 1);
      }
      if (!ok) settle();
    }
    __syncwarp();
  } else if (warp == 10) {
    bool ok = true;
    for (int it = 0; ok && it < n_it; ++it) {
      const int s = it % ST;
      const long long at = (long long)head_of(it) * a.seqs.T + w.start;
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = tile_of(it) * kTile + lane + 32 * i;
        x[i] = r < w.len ? -a.lse[at + r] : -INFINITY;   // (behind the end: p = 0)
        y[i] = r < w.len ? -a.delta[at + r] : 0.f;
      }
      ok = warp_wait(st_empty(s), (it / ST & 1) ^ 1u, abort_flag);
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        stats[s * 2 * kTile + lane + 32 * i] = x[i];
        stats[(s * 2 + 1) * kTile + lane + 32 * i] = y[i];
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(st_full(s));
    }
  } else {
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const F2 scale = f2(a.scale_log2, a.scale_log2);
    bool ok = true;
    for (int it = 0; it < n_it; ++it) {
      const int s = it % ST;
      const bool diagonal = tile_of(it) == key_tile;
      const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(stats + s * 2 * kTile + half * 64);   // (both negative, in pairs)
      const ulonglong2* delta = reinterpret_cast<const ulonglong2*>(stats + (s * 2 + 1) * kTile + half * 64);
      ok = warp_wait(st_full(s), it / ST & 1, abort_flag) && warp_wait(s_full, it & 1, abort_flag);
      if (!ok) break;
      ptx::tc_fence_after();
      F2 p[32];
      uint32_t x[2][32], out[32];
      ptx::tmem_ld_32x32(t_s + lanes + half * 64, x[0]);
      ptx::tmem_ld_32x32(t_s + lanes + half * 64 + 32, x[1]);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const ulonglong2 e = lse[i / 2];
        p[i] = ex2_pair<kBwdPoly<DP>>(x[i / 16][i % 16 * 2], x[i / 16][i % 16 * 2 + 1], scale, F2{e.x}, i);
        p[i + 1] = ex2_pair<kBwdPoly<DP>>(x[i / 16][i % 16 * 2 + 2], x[i / 16][i % 16 * 2 + 3], scale, F2{e.y}, i + 1);
      }
      if (diagonal) {
#pragma unroll
        for (int i = 0; i < 32; ++i) p[i] = hide(p[i], half * 64 + 2 * i < row, half * 64 + 2 * i + 1 < row);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) out[i] = f2_bf16(p[i]);
      ptx::tmem_st_32x32(t_s + lanes + half * 64, out);
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(p_ready);
      ok = warp_wait(dp_full, it & 1, abort_flag);
      if (!ok) break;
      ptx::tc_fence_after();
      ptx::tmem_ld_32x32(t_dp + lanes + half * 64, x[0]);
      ptx::tmem_ld_32x32(t_dp + lanes + half * 64 + 32, x[1]);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const ulonglong2 e = delta[i / 2];
        p[i] = mul2(p[i], add2(f2(__uint_as_float(x[i / 16][i % 16 * 2]), __uint_as_float(x[i / 16][i % 16 * 2 + 1])), F2{e.x}));
        p[i + 1] = mul2(p[i + 1], add2(f2(__uint_as_float(x[i / 16][i % 16 * 2 + 2]), __uint_as_float(x[i / 16][i % 16 * 2 + 3])), F2{e.y}));
      }
      if (diagonal) {   // (a pair that is masked adds nothing, whatever dP holds there)
#pragma unroll
        for (int i = 0; i < 32; ++i) p[i] = hide(p[i], half * 64 + 2 * i < row, half * 64 + 2 * i + 1 < row);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) out[i] = f2_bf16(p[i]);
      ptx::tmem_st_32x32(t_dp + lanes + half * 64, out);
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(ds_ready);
        ptx::mbar_arrive(st_empty(s));
      }
    }
    if (ok) ok = warp_wait(done, 0, abort_flag);
    if (ok) {
      ptx::tc_fence_after();
      const int in_seq = key_tile * kTile + row;
      const long long at = ((long long)(w.start + in_seq) * a.Hkv + hk) * a.D, plane = (long long)a.seqs.T * a.Hkv * a.D;
#pragma unroll 1
      for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
        uint32_t x[32];
        ptx::tmem_ld_32x32(t_dv + lanes + c, x);
        ptx::tmem_ld_wait();
        if (in_seq < w.len) {
          if (a.parts == 1) store_row32(a.dv + at + c, x, 1.f, a.D - c);
          else store_part32(a.sums + 2 * part * plane + at + c, x, 1.f, a.D - c);
        }
        ptx::tmem_ld_32x32(t_dk + lanes + c, x);
        ptx::tmem_ld_wait();
        if (in_seq < w.len) {
          if (a.parts == 1) store_row32(a.dk + at + c, x, a.scale, a.D - c);
          else store_part32(a.sums + (2 * part + 1) * plane + at + c, x, a.scale, a.D - c);
        }
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// Adds up the parts, in their order; rows of no sequence have been zeroed and have no parts.
constexpr int kSumThreads = 256;
__global__ void __launch_bounds__(kSumThreads) dkv_sum_kernel(const Args a) {
  const long long plane = (long long)a.seqs.T * a.Hkv * a.D, i = ((long long)blockIdx.x * kSumThreads + threadIdx.x) * 4;
  if (i >= plane) return;
  if (a.seqs.cu != nullptr) {
    const int t = (int)(i / ((long long)a.Hkv * a.D));
    if (t < a.seqs.cu[0] || t >= a.seqs.cu[a.seqs.n]) return;
  }
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f), k = v;
#pragma unroll 4
  for (int p = 0; p < a.parts; ++p) {
    const float4 x = *reinterpret_cast<const float4*>(a.sums + 2 * p * plane + i), y = *reinterpret_cast<const float4*>(a.sums + (2 * p + 1) * plane + i);
    v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    k.x += y.x; k.y += y.y; k.z += y.z; k.w += y.w;
  }
  *reinterpret_cast<uint2*>(a.dv + i) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
  *reinterpret_cast<uint2*>(a.dk + i) = make_uint2(pack_bf16(k.x, k.y), pack_bf16(k.z, k.w));
}

// ---------------------------------------------------------------- backward: dQ
// A CTA has one tile of queries of one head and works through the keys that it sees, with S and dP as in the forward pass.  Scores have two
// places in tensor memory, so that S(j+1) is there when dS(j) has been made; dS(j) takes the place of S(j).
// Order of products: S(0) dP(0) S(1) | dP(j+1) dQ(j) S(j+2) after dS(j).
template <int DP>
struct DqShape {
  static constexpr int kStages = DP == 64 ? 6 : 5;
  static constexpr int kSmem = (2 + kStages) * kTileBytes<DP> + 256;
};
constexpr int kDqThreads = 320;

template <int DP>
__global__ void __launch_bounds__(kDqThreads, 1) dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                                           const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                                                           const Args a) {
  constexpr int ST = DqShape<DP>::kStages, TB = kTileBytes<DP>;
  extern __shared__ __align__(1024) uint8_t attn_smem[];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t base = ptx::smem_u32(attn_smem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) raise_status(LEWI_STATUS_SMEM_LAYOUT);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int head = blockIdx.x % a.Hq, hk = head / a.G;
  zero_gaps(a.seqs, a.dq, a.Hq * a.D / 8, kDqThreads);
  const Work w = find_work<kDqThreads>(a.seqs, blockIdx.x / a.Hq, [](int tiles) { return tiles; });
  if (!w.any) return;
  const int q_row = w.level * kTile, nb = w.level + 1;

  const uint32_t q_at = base, do_at = base + TB, kv = base + 2 * TB, bars = kv + ST * TB;
  const uint32_t q_full = bars, do_full = bars + 8, dp_full = bars + 16, ds_ready = bars + 24, done = bars + 32, raw = bars + 40;
  auto s_full = [&](int b) { return bars + 48u + 8u * b; };
  auto full = [&](int s) { return bars + 64u + 8u * s; };
  auto empty = [&](int s) { return bars + 64u + 8u * (ST + s); };
  volatile int* abort_flag = &s_abort;
  if (threadIdx.x == 0) {
    for (uint32_t b : {q_full, do_full, dp_full, done, raw, s_full(0), s_full(1)}) ptx::mbar_init(b, 1);
    ptx::mbar_init(ds_ready, 8);
    for (int s = 0; s < ST; ++s) {
      ptx::mbar_init(full(s), 1);
      ptx::mbar_init(empty(s), 1);
    }
    s_abort = 0;
    ptx::mbar_fence_init();
    ptx::fence_proxy_async();
    ptx::prefetch_tensormap(&tm_q);
    ptx::prefetch_tensormap(&tm_k);
    ptx::prefetch_tensormap(&tm_v);
    ptx::prefetch_tensormap(&tm_do);
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem, t_dp = tmem + 256, t_dq = tmem + 384;
  auto t_s = [&](int j) { return tmem + (j & 1) * 128; };

  if (warp == 8) {   // Q, K0, dO, V0, K1, V1, ..
    bool ok = true;
    uint32_t raw_phase = 0;
    if (ptx::elect_one()) {
      ptx::mbar_expect_tx(q_full, TB);
      load_tile<DP>(q_at, &tm_q, q_full, head, w.start + q_row);
      ptx::mbar_expect_tx(do_full, TB);
      load_tile<DP>(do_at, &tm_do, do_full, head, w.start + q_row);
    }
    __syncwarp();
    for (int n = 0; ok && n < 2 * nb; ++n) {
      const int s = n % ST, j = n >> 1;
      ok = warp_wait(empty(s), (n / ST & 1) ^ 1u, abort_flag);
      if (!ok) break;
      const int valid = (n & 1) == 0 ? w.len - j * kTile : kTile;   // (of V a foreign row only reaches pairs that are masked)
      ok = bring_tile<DP>(kv + s * TB, (n & 1) != 0 ? &tm_v : &tm_k, full(s), raw, raw_phase, hk, w.start + j * kTile, valid, abort_flag);
    }
    if (!ok) settle();
  } else if (warp == 9) {
    const uint32_t id_s = ptx::instr_desc_bf16(128, 128, 0, 0), id_d = ptx::instr_desc_bf16(128, DP, 0, 1);
    if (ptx::elect_one()) {
      auto scores = [&](int j) {
        const int n = 2 * j, s = n % ST;
        if (!ptx::mbar_wait(full(s), n / ST & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        mma_kk<DP>(t_s(j), q_at, kv + s * TB, id_s);
        ptx::mma_commit(s_full(j & 1));
        return true;
      };
      auto dps = [&](int j) {
        const int n = 2 * j + 1, s = n % ST;
        if (!ptx::mbar_wait(full(s), n / ST & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        mma_kk<DP>(t_dp, do_at, kv + s * TB, id_s);
        ptx::mma_commit(dp_full);
        ptx::mma_commit(empty(s));
        return true;
      };
      bool ok = ptx::mbar_wait(q_full, 0, abort_flag) && scores(0) && ptx::mbar_wait(do_full, 0, abort_flag) && dps(0) && (nb < 2 || scores(1));
      for (int j = 0; ok && j < nb; ++j) {
        ok = ptx::mbar_wait(ds_ready, j & 1, abort_flag) && (j + 1 >= nb || dps(j + 1));
        if (!ok) break;
        ptx::tc_fence_after();
        mma_tm<0, 8>(t_dq, t_s(j), kv + 2 * j % ST * TB, id_d, j > 0, 64);
        ptx::mma_commit(j + 1 < nb ? empty(2 * j % ST) : done);
        if (j + 2 < nb) ok = scores(j + 2);
      }
      if (!ok) settle();
    }
    __syncwarp();
  } else {
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const bool live = q_row + row < w.len;
    const long long at = (long long)head * a.seqs.T + w.start + q_row + row;
    const float lse = live ? a.lse[at] : INFINITY, delta = live ? a.delta[at] : 0.f;
    const F2 scale = f2(a.scale_log2, a.scale_log2), shift = f2(-lse, -lse), minus_delta = f2(-delta, -delta);
    bool ok = true;
    for (int j = 0; j < nb; ++j) {
      const bool diagonal = j == nb - 1;
      ok = warp_wait(s_full(j & 1), j >> 1 & 1, abort_flag);
      if (!ok) break;
      ptx::tc_fence_after();
      F2 p[32];
      uint32_t x[2][32], ds[32];
      ptx::tmem_ld_32x32(t_s(j) + lanes + half * 64, x[0]);
      ptx::tmem_ld_32x32(t_s(j) + lanes + half * 64 + 32, x[1]);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; ++i) p[i] = ex2_pair<kBwdPoly<DP>>(x[i / 16][i % 16 * 2], x[i / 16][i % 16 * 2 + 1], scale, shift, i);
      ok = warp_wait(dp_full, j & 1, abort_flag);
      if (!ok) break;
      ptx::tc_fence_after();
      ptx::tmem_ld_32x32(t_dp + lanes + half * 64, x[0]);
      ptx::tmem_ld_32x32(t_dp + lanes + half * 64 + 32, x[1]);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; ++i)
        p[i] = mul2(p[i], add2(f2(__uint_as_float(x[i / 16][i % 16 * 2]), __uint_as_float(x[i / 16][i % 16 * 2 + 1])), minus_delta));
      if (diagonal) {
#pragma unroll
        for (int i = 0; i < 32; ++i) p[i] = hide(p[i], half * 64 + 2 * i > row, half * 64 + 2 * i + 1 > row);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) ds[i] = f2_bf16(p[i]);
      ptx::tmem_st_32x32(t_s(j) + lanes + half * 64, ds);
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ds_ready);
    }
    if (ok) ok = warp_wait(done, 0, abort_flag);
    if (ok) {
      ptx::tc_fence_after();
      const long long out = ((long long)(w.start + q_row + row) * a.Hq + head) * a.D;
#pragma unroll 1
      for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
        uint32_t x[32];
        ptx::tmem_ld_32x32(t_dq + lanes + c, x);
        ptx::tmem_ld_wait();
        if (live) store_row32(a.dq + out + c, x, a.scale, a.D - c);
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- host side
// [T][heads][D] rows `row` elements and heads D elements apart, boxes of 128 rows x 64 columns of one head
inline bool make_rows_map(CUtensorMap* m, const void* p, int T, int heads, int D, long long row) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)row * 2};
  const cuuint32_t box[3] = {64, 1, kTile};
  return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p, dims, strides, box);
}

// How many CTAs share the heads of a group for a tile of dK and dV.  A tile of the first keys of a long sequence has all its queries, times G
// heads, so few key heads leave a few long runs: as many parts as make 2 CTAs per SM, at least one head each.
inline int dkv_parts(long long tiles, int Hkv, int G) {
  const long long want = 2ll * num_sms(), have = tiles * Hkv;
  return (int)(have >= want ? 1 : (want + have - 1) / have < G ? (want + have - 1) / have : G);
}

// Units that `n` sequences of together T rows can have at most, `per` per tile and one to round up per sequence.
inline long long most_tiles(int T, int n) { return (long long)T / kTile + n; }

}  // namespace attn
}  // namespace lewi
