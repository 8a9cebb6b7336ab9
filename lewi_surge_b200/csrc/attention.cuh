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

#include <cfloat>
#include <type_traits>

#include "common.cuh"
#include "f32x2.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace lewi {
namespace attn {

constexpr int kTile = 128;
constexpr int kMaxD = 128;
// Tiles whose products go into one accumulator.  The tensor core truncates every sum that it makes: a sum of one sign over n rows comes out short by about
// n 2^-27 of itself (o of 2^20 rows, v and the weights alike, by 2^-7).  After so many tiles an accumulator is therefore added to float32 sums kept in
// memory, which rounds to nearest, and starts from zero: 2^-12 at most.
constexpr int kChain = 256;
constexpr int64_t kMaxGroupRows = 1 << 25;   // rows times heads per key head: an item of dK and dV (0.4 s) stays below what a wait may last

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

// What a CTA works on: unit `level` of the sequence at rows start .. start + len, `sub` of the unit's shares.  level < 0: nothing is left.
struct Item {
  int start, len, level, sub;
};

// The kernels run one CTA per SM, which takes items until none is left; a warp of its own looks the next one up while the others work.
// Sequence s has the units 0 .. units(s) - 1 of `rows` rows, a unit's work grows with its number, and every unit has `subs` equal shares.
// Items are numbered by falling unit, all shares of a unit together, and CTA c has the items c, 2 n - 1 - c, 2 n + c, 4 n - 1 - c, .. of n
// CTAs: long runs first, and about as much work for everybody, whatever the lengths.  No table is needed: F(i) = sum_s max(0, units(s) - i)
// counts the units from number i on, so the x-th unit's number is the largest i with F(i) > x, and its sequence is the
// (x - F(i + 1))-th of those that have it.  A search is for a new number only; the sequences that have the same one are walked through.
constexpr int kPlanned = 448;   // sequences whose units are kept in shared memory (further ones are looked up again)
struct Plan {
  int4 item[2];
  int units[kPlanned];
};

// The whole warp calls it; `give` hands an item on and tells whether to go on.
template <class Give>
__device__ __forceinline__ void plan_items(const Seqs& q, int rows, int subs, Plan& plan, Give give) {
  const int lane = threadIdx.x & 31, n = gridDim.x, c = blockIdx.x;
  auto unit_count = [&](int s) { return (rows_of(q, s).len + rows - 1) / rows; };
  const bool alike = q.cu == nullptr, kept = q.n <= kPlanned;
  int most = 0;   // a sequence's units
  if (alike) {
    most = unit_count(0);
  } else {
    bool falls = false;
    for (int s = lane; s < q.n; s += 32) {
      const int u = unit_count(s);
      if (kept) plan.units[s] = u;
      most = max(most, u);
      falls |= q.cu[s + 1] < q.cu[s];
    }
    most = __reduce_max_sync(0xffffffffu, most);
    // Sequences whose bounds ascend share no row, so that there are at most T / rows + n units.  Where bounds fall they could name all rows again
    // and again (more work than any grid should have, more units than 32 bits count): such a call has no sequence at all.
    if (__any_sync(0xffffffffu, falls)) most = 0;
    __syncwarp();
  }
  auto units = [&](int s) { return kept ? plan.units[s] : unit_count(s); };
  auto count = [&](int i) {
    int v = 0;
    for (int s = lane; s < q.n; s += 32) v += max(0, units(s) - i);
    return __reduce_add_sync(0xffffffffu, v);
  };
  const int all = most == 0 ? 0 : alike ? most * q.n : count(0);
  int lo = most, first = 0, end = 0;   // the unit number of the last item, F(lo + 1) and F(lo): units of this number are the x in between
  int s0 = 0, passed = 0;              // the sequences before s0 have `passed` of them
  for (int r = 0;; ++r) {
    const long long id = (long long)r * n + ((r & 1) != 0 ? n - 1 - c : c);
    const int x = (int)min(id / subs, 0x7fffffffll);
    Item item{0, 0, -1, 0};
    if (x < all) {
      int s;
      if (alike) {
        lo = most - 1 - x / q.n;
        s = x % q.n;
      } else {
        if (x >= end) {
          int hi = lo;   // F(hi) <= x
          for (lo = 0; hi - lo > 1;) {
            const int mid = (lo + hi) >> 1;
            if (count(mid) > x) lo = mid;
            else hi = mid;
          }
          first = count(lo + 1);
          end = count(lo);
          s0 = passed = 0;
        }
        unsigned have;   // of 32 sequences those that have the unit
        for (;; s0 += 32) {
          have = __ballot_sync(0xffffffffu, s0 + lane < q.n && units(min(s0 + lane, q.n - 1)) > lo);
          if (x - first < passed + __popc(have) || s0 + 32 >= q.n) break;
          passed += __popc(have);
        }
        for (int rank = x - first - passed; rank > 0; --rank) have &= have - 1;
        s = min(s0 + max(__ffs(have) - 1, 0), q.n - 1);
      }
      const Rows of = rows_of(q, s);
      item = {of.start, of.len, lo, (int)(id % subs)};
    }
    if (!give(r, item) || item.level < 0) return;
  }
}

// Rows of no sequence become zero: a share of them for every CTA, by one warp; `vecs` 16-byte pieces each.
__device__ __forceinline__ void zero_gaps(const Seqs& q, __nv_bfloat16* out, int vecs) {
  if (q.cu == nullptr) return;
  const int lane = threadIdx.x & 31, first = min(max(q.cu[0], 0), q.T), end = min(max(q.cu[q.n], 0), q.T);
  for (int r = blockIdx.x; r < q.T; r += gridDim.x) {
    if (r >= first && r < end) r += (end - r + gridDim.x - 1) / gridDim.x * gridDim.x;
    if (r >= q.T) break;
    for (int i = lane; i < vecs; i += 32) st_v4(out + ((long long)r * vecs + i) * 8, make_uint4(0u, 0u, 0u, 0u));
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
// What rounding `p` to `rounded` left, rounded as well
__device__ __forceinline__ uint32_t rest_bf16(F2 p, uint32_t rounded) {
  float lo, hi;
  f2_split(p, lo, hi);
  return pack_bf16(lo - bf16_lo(rounded), hi - bf16_hi(rounded));
}
// Operand tiles in shared memory: boxes of [128 rows][64 columns], 128-byte swizzled, 16 KB apart.
constexpr int kBox = kTile * 128;
template <int DP> constexpr int kTileBytes = kTile * DP * 2;
// K-major (rows are M or N, columns K) and MN-major (rows are K, columns N)
// (a step is a constant added to a tile's descriptor, whose address field holds all of shared memory: nothing is masked or shifted again)
__device__ __forceinline__ uint64_t desc_k(uint32_t tile, int step) {
  return ptx::smem_desc_hi_sw128(16, 1024) + ((tile >> 4) + (((step >> 2) * kBox + (step & 3) * 32) >> 4));
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, int step) {
  return ptx::smem_desc_hi_sw128(kBox, 1024) + ((tile >> 4) + (step * 2048 >> 4));
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

// A tile reaches into rows that are not its sequence's where `valid` < 128.  Such a tile lands on a barrier of its own (`raw`), and another warp
// zeroes the foreign rows and hands the tile on (`mend_tile`), so that the warp that brings tiles waits for none of them (doing both
// itself it took 1.4 us per such tile, and of short sequences every other tile is one).
template <int DP>
__device__ __forceinline__ void bring_tile(uint32_t dst, const CUtensorMap* tm, uint32_t full, uint32_t raw, int head, int row, int valid) {
  if (ptx::elect_one()) {
    const uint32_t bar = valid >= kTile ? full : raw;
    ptx::mbar_expect_tx(bar, kTileBytes<DP>);
    load_tile<DP>(dst, tm, bar, head, row);
  }
  __syncwarp();
}
template <int DP>
__device__ __forceinline__ bool mend_tile(uint32_t dst, uint32_t full, uint32_t raw, uint32_t phase, int valid, volatile int* abort_flag) {
  if (!warp_wait(raw, phase & 1u, abort_flag)) return false;
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

// A place in a ring of ST and the parity of its phase, moved on instead of divided out of a count.
template <int ST>
struct At {
  uint32_t s, phase;
  __device__ __forceinline__ void on(uint32_t by) {
    s += by;
    if (s >= ST) {
      s -= ST;
      phase ^= 1u;
    }
  }
};

enum FwdItem { kTwoHeads, kTwoTiles, kOneTile };

struct Args {
  Seqs seqs;
  int Hq, Hkv, G, D;
  float scale, scale_log2;
  __nv_bfloat16 *o, *o_rest;   // [T][Hq][D]; what rounding o left of it, for the backward pass and for sums of chains
  float *lse, *delta;      // [Hq][T], lse in units of log 2 (null in a forward pass that none back follows)
  __nv_bfloat16 *dq, *dk, *dv;
  int parts;               // of a group's heads, one CTA each for dK and dV
  float* sums;             // [part][dV, dK][T][Hkv][D] where there are several
  float4 *chain_kv, *chain_q;   // per CTA [dV, dK or dQ][DP / 4][128]: sums of an item's chains so far (null where none is longer than kChain)
  FwdItem shape;           // of the forward pass
};

// A warp's 32 rows x 64 bytes go through shared memory (2 KB of its own), so that a store writes 8 rows x 64 bytes and not a piece of each of
// 32 rows (which took 3700 cycles for a tile of 128 x 128 bf16).  `v`: this lane's row; rows dst + r * stride for r < valid, `bytes` of the 64.
constexpr int kStaging = 8 * 2048, kBarriers = 512;
__device__ __forceinline__ void store_rows(uint8_t* stage, const uint32_t (&v)[16], uint8_t* dst, long long stride, int valid, int bytes) {
  const int lane = threadIdx.x & 31;
  uint4* mine = reinterpret_cast<uint4*>(stage) + lane * 4;
  __syncwarp();   // (what was there has been read)
#pragma unroll
  for (int i = 0; i < 4; ++i) mine[i ^ (lane >> 1 & 3)] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 8 + (lane >> 2), piece = lane & 3;
    const uint4 x = reinterpret_cast<const uint4*>(stage)[row * 4 + (piece ^ (row >> 1 & 3))];
    if (row < valid && piece * 16 < bytes) st_v4(dst + row * stride + piece * 16, x);
  }
}
// 32 accumulator columns as bf16 / 16 of them as float32
__device__ __forceinline__ void pack_row(uint32_t (&out)[16], const uint32_t (&v)[32], float f) {
#pragma unroll
  for (int i = 0; i < 16; ++i) out[i] = pack_bf16(__uint_as_float(v[2 * i]) * f, __uint_as_float(v[2 * i + 1]) * f);
}
__device__ __forceinline__ void half_row(uint32_t (&out)[16], const uint32_t (&v)[32], int half, float f) {
#pragma unroll
  for (int i = 0; i < 16; ++i) out[i] = __float_as_uint(__uint_as_float(v[16 * half + i]) * f);
}

// 32 columns of a row to or from the sums of chains: `at` is the place of the row and the first column, four columns are 128 rows apart.
__device__ __forceinline__ void add_chain(uint32_t (&v)[32], const float4* at) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 x = __ldcg(at + i * kTile);
    v[4 * i] = __float_as_uint(__uint_as_float(v[4 * i]) + x.x);
    v[4 * i + 1] = __float_as_uint(__uint_as_float(v[4 * i + 1]) + x.y);
    v[4 * i + 2] = __float_as_uint(__uint_as_float(v[4 * i + 2]) + x.z);
    v[4 * i + 3] = __float_as_uint(__uint_as_float(v[4 * i + 3]) + x.w);
  }
}
__device__ __forceinline__ void put_chain(const uint32_t (&v)[32], float4* at) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    __stcg(at + i * kTile, make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3])));
}

// What the roles of a kernel share: barriers of the items, the planning warp's loop, and how a warp or a thread takes an item.
struct ItemQueue {
  Plan* plan;
  uint32_t bars;   // full[2], empty[2]
  volatile int* abort_flag;
  __device__ __forceinline__ void init(int readers) const {
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(bars + 8u * s, 1);
      ptx::mbar_init(bars + 16u + 8u * s, readers);
    }
  }
  __device__ __forceinline__ void run(const Seqs& seqs, int rows, int subs) const {
    plan_items(seqs, rows, subs, *plan, [&](int r, const Item& item) {
      if (!warp_wait(bars + 16u + 8u * (r & 1), (r >> 1 & 1) ^ 1u, abort_flag)) return false;
      if ((threadIdx.x & 31) == 0) {
        plan->item[r & 1] = make_int4(item.start, item.len, item.level, item.sub);
        ptx::mbar_arrive(bars + 8u * (r & 1));
      }
      __syncwarp();
      return true;
    });
  }
  __device__ __forceinline__ Item read(int r) const {
    const volatile int4& v = plan->item[r & 1];
    return {v.x, v.y, v.z, v.w};
  }
  // by a whole warp; level < 0 also where a wait ran out
  __device__ __forceinline__ Item take(int r) const {
    if (!warp_wait(bars + 8u * (r & 1), r >> 1 & 1, abort_flag)) return {0, 0, -1, 0};
    const Item item = read(r);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(bars + 16u + 8u * (r & 1));
    return item;
  }
  // by one thread
  __device__ __forceinline__ Item take_alone(int r) const {
    if (!ptx::mbar_wait(bars + 8u * (r & 1), r >> 1 & 1, abort_flag)) return {0, 0, -1, 0};
    const Item item = read(r);
    ptx::mbar_arrive(bars + 16u + 8u * (r & 1));
    return item;
  }
};

// ---------------------------------------------------------------- forward
// A CTA works on two tiles of queries that share their keys: two heads of a group, or, where a group is odd, the tiles 2 u and 2 u + 1 of one
// head.  While one tile's softmax is made by its four warps, the tensor cores multiply for the other, and every key and value tile
// that is brought serves both.  Warps 0-3 and 4-7: a row of S per thread; warp 8: TMA; warp 9: MMA; warp 10: items; warp 11: rows of no
// sequence, and those of other sequences in a tile.  Products are issued in the order S0(j+1) after P0 V(j), S1(j+1) after P1 V(j): a
// softmax that finds its scores knows that the product before them is done, so it may scale O then.  It does so only where the maximum has
// grown by more than 8 (in powers of 2; p stays below 2^8, which bf16 and float32 hold as well as 1).  The next item's queries, first keys
// and scores are on their way while O of this one is written out.  p is rounded to bf16 for its product, its sum l is taken before; in training
// (TRAIN) the first tile of a sequence, whose rows have few keys and errors that no sum averages, is multiplied by what that left as well.
//
// Where such items are too few for the SMs an item is one tile (ONE, by fwd_item).  Its scores have both places, so that those of the next block are there
// when a softmax ends, which then scales O after the product before (pv_done).  Each row's steps are the same, and so are its bits.
//
// What bounds it: a tile's chain S -> softmax -> P -> S, 2900 cycles for both tiles of a block where their products take 2048 (D = 128) or
// 1024 (D = 64) and their exponentials 2048 of the special function unit.  One sequence of 16,384, 16 heads over 2, D = 128: 0.80 ms,
// 1370 TFLOP/s; 8192, 32 over 8, D = 64: 0.34 ms, 800 TFLOP/s.
constexpr int kFwdThreads = 384;
template <int DP>
struct FwdShape {
  static constexpr int kStages = DP == 64 ? 6 : 4;
  static constexpr int kSmem = (2 + kStages) * kTileBytes<DP> + kStaging + kBarriers;
};

template <int DP, bool TRAIN, bool ONE>
__global__ void __launch_bounds__(kFwdThreads, 1) fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                                             const __grid_constant__ CUtensorMap tm_v, const Args a) {
  constexpr int ST = FwdShape<DP>::kStages, TB = kTileBytes<DP>;
  extern __shared__ __align__(1024) uint8_t attn_smem[];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ Plan s_plan;
  __shared__ float s_kept[2 * kTile];   // the maximum that a row's kept sums are relative to
  const uint32_t base = ptx::smem_u32(attn_smem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) raise_status(LEWI_STATUS_SMEM_LAYOUT);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t kv = base + 2 * TB, bars = kv + ST * TB + kStaging;
  auto full = [&](int n) { return bars + 8u * (n % ST); };
  auto empty = [&](int n) { return bars + 8u * (ST + n % ST); };
  auto q_full = [&](int t) { return bars + 8u * (2 * ST + t); };
  auto q_empty = [&](int t) { return bars + 8u * (2 * ST + 2 + t); };
  auto s_full = [&](int t) { return bars + 8u * (2 * ST + 4 + t); };
  auto p_full = [&](int t, int half) { return bars + 8u * (2 * ST + 6 + 2 * t + half); };
  auto o_full = [&](int t) { return bars + 8u * (2 * ST + 10 + t); };
  auto o_empty = [&](int t) { return bars + 8u * (2 * ST + 12 + t); };
  auto raw = [&](int n) { return bars + 8u * (2 * ST + 14 + n % ST); };
  volatile int* abort_flag = &s_abort;
  const ItemQueue items{&s_plan, bars + 8u * (3 * ST + 14), abort_flag};
  const uint32_t pv_done = bars + 8u * (3 * ST + 18);
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      for (uint32_t b : {full(s), empty(s), raw(s)}) ptx::mbar_init(b, 1);
    }
    for (int t = 0; t < 2; ++t) {
      for (uint32_t b : {q_full(t), q_empty(t), s_full(t), o_full(t)}) ptx::mbar_init(b, 1);
      for (uint32_t b : {p_full(t, 0), p_full(t, 1), o_empty(t)}) ptx::mbar_init(b, 4);
    }
    ptx::mbar_init(pv_done, 1);
    items.init(11);
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
  auto tile_of = [&](const Item& w, int t) { return a.shape == kTwoTiles ? 2 * w.level + t : w.level; };
  auto head_of = [&](const Item& w, int t) { return a.shape == kTwoHeads ? 2 * w.sub + t : w.sub; };
  auto blocks_of = [&](const Item& w, int t) { return tile_of(w, t) * kTile < w.len && (t == 0 || !ONE) ? tile_of(w, t) + 1 : 0; };

  // registers: 8 x 216 + 4 x 72 = 12 x 168 a thread, what the launch has
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
      // ---------------------------------------------------------------- queries, then K0, V0, K1, V1, ..
      bool ok = true;
      int n = 0, used[2] = {0, 0};
      for (int r = 0; ok; ++r) {
        const Item w = items.take(r);
        if (w.level < 0) break;
        const int hk = head_of(w, 0) / a.G, nb = max(blocks_of(w, 0), blocks_of(w, 1));
        for (int t = 0; ok && t < 2; ++t) {
          if (blocks_of(w, t) == 0) continue;
          ok = warp_wait(q_empty(t), (used[t] & 1) ^ 1u, abort_flag);
          ++used[t];
          if (ok && ptx::elect_one()) {
            ptx::mbar_expect_tx(q_full(t), TB);
            load_tile<DP>(base + t * TB, &tm_q, q_full(t), head_of(w, t), w.start + tile_of(w, t) * kTile);
          }
          __syncwarp();
        }
        for (int i = 0; ok && i < 2 * nb; ++i, ++n) {
          const int j = i >> 1, valid = (i & 1) != 0 ? w.len - j * kTile : kTile;   // (of K a foreign row only reaches scores that are masked)
          ok = warp_wait(empty(n), (n / ST & 1) ^ 1u, abort_flag);
          if (!ok) break;
          bring_tile<DP>(kv + n % ST * TB, (i & 1) != 0 ? &tm_v : &tm_k, full(n), raw(n), hk, w.start + j * kTile, valid);
        }
      }
      if (s_abort) settle();
    } else if (warp == 9) {
      // ---------------------------------------------------------------- products
      const uint32_t id_s = ptx::instr_desc_bf16(128, 128, 0, 0), id_o = ptx::instr_desc_bf16(128, DP, 0, 1);
      if (ptx::elect_one()) {
        bool ok = true;
        int n = 0, used[2] = {0, 0}, done[2] = {0, 0};   // ring position, items and blocks of each tile so far
        for (int r = 0; ok; ++r) {
          const Item w = items.take_alone(r);
          if (w.level < 0) break;
          const int blocks[2] = {blocks_of(w, 0), blocks_of(w, 1)}, nb = max(blocks[0], blocks[1]);
          if constexpr (ONE) {   // S(0) S(1) | P(j) V(j), S(j + 2) after P(j)
            auto scores = [&](int j) {
              const int x = n + 2 * j;
              if (!ptx::mbar_wait(full(x), x / ST & 1, abort_flag)) return false;
              ptx::tc_fence_after();
              mma_kk<DP>(s_at(done[0] + j & 1), base, kv + x % ST * TB, id_s);
              ptx::mma_commit(s_full(done[0] + j & 1));
              ptx::mma_commit(empty(x));
              if (j + 1 == nb) ptx::mma_commit(q_empty(0));
              return true;
            };
            ok = ptx::mbar_wait(q_full(0), used[0] & 1, abort_flag) && scores(0) && (nb == 1 || scores(1)) &&
                 ptx::mbar_wait(o_empty(0), (used[0] & 1) ^ 1u, abort_flag);
            for (int j = 0; ok && j < nb; ++j) {
              const int x = n + 2 * j + 1, b = done[0] + j;
              ok = ptx::mbar_wait(full(x), x / ST & 1, abort_flag) && ptx::mbar_wait(p_full(b & 1, 0), b >> 1 & 1, abort_flag);
              if (!ok) break;
              ptx::tc_fence_after();
              mma_tm<0, 4>(o_at(0), s_at(b & 1), kv + x % ST * TB, id_o, j % kChain != 0, 32);
              ok = ptx::mbar_wait(p_full(b & 1, 1), b >> 1 & 1, abort_flag);
              if (!ok) break;
              ptx::tc_fence_after();
              mma_tm<4, 8>(o_at(0), s_at(b & 1), kv + x % ST * TB, id_o, true, 32);
              if (TRAIN && nb == 1) mma_tm<0, 8>(o_at(0), s_at(b & 1) + 64, kv + x % ST * TB, id_o, true, 32);
              ptx::mma_commit(pv_done);
              ptx::mma_commit(empty(x));
              if (j + 1 == nb) ptx::mma_commit(o_full(0));
              if (j + 2 < nb) ok = scores(j + 2);
            }
            n += 2 * nb;
            done[0] += nb;
            ++used[0];
          } else {
            auto scores = [&](int t, int j) {
              ptx::tc_fence_after();
              mma_kk<DP>(s_at(t), base + t * TB, kv + (n + 2 * j) % ST * TB, id_s);
              ptx::mma_commit(s_full(t));
              if (j + 1 == blocks[t]) ptx::mma_commit(q_empty(t));
            };
            ok = ptx::mbar_wait(full(n), n / ST & 1, abort_flag);
            for (int t = 0; ok && t < 2; ++t)
              if (blocks[t] > 0) {
                ok = ptx::mbar_wait(q_full(t), used[t] & 1, abort_flag);
                if (ok) scores(t, 0);
              }
            if (!ok) break;
            ptx::mma_commit(empty(n));
            for (int j = 0; ok && j < nb; ++j) {
              const int nv = n + 2 * j + 1, nk = nv + 1;
              ok = ptx::mbar_wait(full(nv), nv / ST & 1, abort_flag);
              for (int t = 0; ok && t < 2; ++t) {
                if (j >= blocks[t]) continue;
                ok = (j > 0 || ptx::mbar_wait(o_empty(t), (used[t] & 1) ^ 1u, abort_flag)) && ptx::mbar_wait(p_full(t, 0), done[t] & 1, abort_flag);
                if (!ok) break;
                ptx::tc_fence_after();
                mma_tm<0, 4>(o_at(t), s_at(t), kv + nv % ST * TB, id_o, j % kChain != 0, 32);
                ok = ptx::mbar_wait(p_full(t, 1), done[t] & 1, abort_flag);
                if (!ok) break;
                ptx::tc_fence_after();
                mma_tm<4, 8>(o_at(t), s_at(t), kv + nv % ST * TB, id_o, true, 32);
                if (TRAIN && blocks[t] == 1) mma_tm<0, 8>(o_at(t), s_at(t) + 64, kv + nv % ST * TB, id_o, true, 32);
                ++done[t];
                if (j + 1 < blocks[t]) {
                  ok = ptx::mbar_wait(full(nk), nk / ST & 1, abort_flag);
                  if (ok) scores(t, j + 1);
                } else {
                  ptx::mma_commit(o_full(t));
                }
              }
              if (!ok) break;
              ptx::mma_commit(empty(nv));
              if (j + 1 < nb) ptx::mma_commit(empty(nk));
            }
            n += 2 * nb;
            for (int t = 0; t < 2; ++t) used[t] += blocks[t] > 0;
          }
        }
        if (s_abort) settle();
      }
      __syncwarp();
    } else if (warp == 10) {
      items.run(a.seqs, a.shape == kTwoTiles ? 2 * kTile : kTile, a.shape == kTwoHeads ? a.Hq / 2 : a.Hq);
    } else {
      zero_gaps(a.seqs, a.o, a.Hq * a.D / 8);
      bool ok = true;
      int n = 0;
      uint32_t phases = 0;   // of the raw barriers, a bit each
      for (int r = 0; ok; ++r) {
        const Item w = items.take(r);
        if (w.level < 0) break;
        const int nb = max(blocks_of(w, 0), blocks_of(w, 1)), valid = w.len - (nb - 1) * kTile;   // of the last values
        n += 2 * nb;
        if (valid >= kTile) continue;
        const int s = (n - 1) % ST;
        ok = mend_tile<DP>(kv + s * TB, full(s), raw(s), phases >> s, valid, abort_flag);
        phases ^= 1u << s;
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // this warp's lanes of tensor memory
    const uint32_t op = o_at(t) + lanes;
    const F2 scale = f2(a.scale_log2, a.scale_log2);
    const float lowest = -0.5f * FLT_MAX / fmaxf(1.f, a.scale_log2);   // (times the scale it is finite)
    int used = 0, done = 0;
    bool ok = true;
    for (int r = 0; ok; ++r) {
      const Item w = items.take(r);
      if (w.level < 0) break;
      const int tile = tile_of(w, t), head = head_of(w, t), n_blocks = blocks_of(w, t);
      if (n_blocks == 0) continue;
      const bool mine = tile * kTile + row < w.len;   // (what other sequences' rows hold decides nothing)
      float m = 0.f, l = 0.f;
      const int row0 = tile * kTile + (warp & 3) * 32, valid = w.len - row0;   // of this warp's rows
      const long long at = ((long long)(w.start + row0) * a.Hq + head) * a.D, stride = (long long)a.Hq * a.D * 2;
      uint8_t* stage = attn_smem + (2 + ST) * TB + warp * 2048;
      auto store = [&](__nv_bfloat16* to, const uint32_t (&x)[16], int c) {
        store_rows(stage, x, reinterpret_cast<uint8_t*>(to + at + c * 32), stride, valid, (a.D - c * 32) * 2);
      };
      auto column = [&](int c, uint32_t (&v)[32]) {
        ptx::tmem_ld_32x32(op + c * 32, v);
        ptx::tmem_ld_wait();
      };
      // adds what earlier chains left in o and o_rest, which is relative to an earlier maximum
      auto add_kept = [&](int c, uint32_t (&v)[32]) {
        const float before = s_kept[threadIdx.x], f = before == m ? 1.f : ex2((before - m) * a.scale_log2);
        const long long from = at + (long long)lane * a.Hq * a.D + c * 32;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (lane >= valid || c * 32 + i * 8 >= a.D) continue;
          const uint4 x = __ldcg(reinterpret_cast<const uint4*>(a.o + from + i * 8)), y = __ldcg(reinterpret_cast<const uint4*>(a.o_rest + from + i * 8));
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t &lo = v[i * 8 + 2 * e], &hi = v[i * 8 + 2 * e + 1];
            lo = __float_as_uint(fmaf(bf16_lo(xs[e]) + bf16_lo(ys[e]), f, __uint_as_float(lo)));
            hi = __float_as_uint(fmaf(bf16_hi(xs[e]) + bf16_hi(ys[e]), f, __uint_as_float(hi)));
          }
        }
      };
      // columns times `inv` to o and, what their rounding leaves, to o_rest
      auto store_twice = [&](int c, const uint32_t (&v)[32], float inv) {
        uint32_t out[16], rest[16];
        pack_row(out, v, inv);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          rest[i] = pack_bf16(__uint_as_float(v[2 * i]) * inv - bf16_lo(out[i]), __uint_as_float(v[2 * i + 1]) * inv - bf16_hi(out[i]));
        store(a.o, out, c);
        store(a.o_rest, rest, c);
      };
      auto block = [&](int j, auto first) {   // (first: in training and of a sequence's first tile; apart, so that the others do not pay for it)
        const int place = ONE ? done & 1 : t;
        const uint32_t sp = s_at(place) + lanes;
        if (!warp_wait(s_full(place), (ONE ? done >> 1 : done) & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(sp + c * 32, s[c]);
        ptx::tmem_ld_wait();
        if (j == tile) {   // the diagonal: keys behind the query
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
          m = fmaxf(top, lowest);   // (scores of -inf only: their p are zero, and what follows is larger)
        } else if (__any_sync(0xffffffffu, mine && (top - m) * a.scale_log2 > 8.f)) {
          if (ONE && !warp_wait(pv_done, (done & 1) ^ 1u, abort_flag)) return false;   // of the block before
          ptx::tc_fence_after();
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
        const F2 shift = f2(-m * a.scale_log2, -m * a.scale_log2);
        F2 sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t p[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            uint32_t &s0 = s[2 * half + i / 16][i % 16 * 2], &s1 = s[2 * half + i / 16][i % 16 * 2 + 1];
            const F2 x = ex2_pair<4>(s0, s1, scale, shift, i);
            sum[i & 1] = add2(sum[i & 1], x);
            p[i] = f2_bf16(x);
            if constexpr (first.value) {
              float lo, hi;
              f2_split(x, lo, hi);
              s0 = __float_as_uint(lo);
              s1 = __float_as_uint(hi);
            }
          }
          ptx::tmem_st_32x32(sp + half * 32, p);
          if constexpr (first.value) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              p[i] = rest_bf16(f2(__uint_as_float(s[2 * half + i / 16][i % 16 * 2]), __uint_as_float(s[2 * half + i / 16][i % 16 * 2 + 1])), p[i]);
            ptx::tmem_st_32x32(sp + 64 + half * 32, p);
          }
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(p_full(place, half));
        }
        float lo, hi;
        f2_split(add2(sum[0], sum[1]), lo, hi);
        l += lo + hi;
        ++done;
        return true;
      };
      if (__builtin_expect(!TRAIN || n_blocks > 1, 1)) {
        int j = 0;
        for (;;) {
          for (const int end = min(j + kChain, n_blocks); ok && j < end; ++j) ok = block(j, std::false_type());
          if (!ok || j == n_blocks) break;
          // a chain ends: O so far is kept in o and o_rest, and starts from zero.  (Its last product is done when the next scores are, as in `block`.)
          ok = ONE ? warp_wait(pv_done, (done & 1) ^ 1u, abort_flag) : warp_wait(s_full(t), done & 1, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t v[32];
            column(c, v);
            if (j > kChain) add_kept(c, v);
            store_twice(c, v, 1.f);
          }
          __syncwarp();   // (rows are read again by other lanes than have stored them)
          s_kept[threadIdx.x] = m;
        }
      } else {
        ok = block(0, std::bool_constant<TRAIN>());
      }
      ok = ok && warp_wait(o_full(t), used & 1, abort_flag);
      if (!ok) break;
      ++used;
      ptx::tc_fence_after();
      if (__builtin_expect(n_blocks > kChain, 0)) {   // (the last chain and the others, for what follows)
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t v[32];
          column(c, v);
          add_kept(c, v);
          ptx::tmem_st_32x32(op + c * 32, v);
        }
        ptx::tmem_st_wait();
      }
      const float inv = 1.f / l;
      auto free_o = [&] {
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(o_empty(t));
      };
      if constexpr (TRAIN) {
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t v[32];
          column(c, v);
          store_twice(c, v, inv);
        }
        free_o();
      } else {
        uint32_t out[DP / 32][16];
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t v[32];
          column(c, v);
          pack_row(out[c], v, inv);
        }
        free_o();   // (the next item's products may go on)
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) store(a.o, out[c], c);
      }
      if (a.lse != nullptr && lane < valid) a.lse[(long long)head * a.seqs.T + w.start + row0 + lane] = m * a.scale_log2 + log2f(l);
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
// delta[h][t] = sum_d dO O, DP / 8 lanes per row.  Where a softmax is nearly all on one key, dP - delta is a small difference of large numbers:
// O is therefore taken with what its rounding left.  dQ of 3000 rows is off by 2.1e-3 of its norm for scores of N(0,1), 3.0e-3 for N(0,100) (with
// the rounded O alone 2.4e-3 and 5.5e-3, for single rows 5e-2); its own rounding is 1.7e-3.
constexpr int kDeltaThreads = 256;
template <int DP>
__global__ void __launch_bounds__(kDeltaThreads) delta_kernel(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ o_rest,
                                                              const __nv_bfloat16* __restrict__ d_o, float* __restrict__ delta, int T, int Hq, int D) {
  constexpr int L = DP / 8;
  grid_launch();
  const long long row = ((long long)blockIdx.x * kDeltaThreads + threadIdx.x) / L;
  const int c = threadIdx.x % L * 8;
  const bool live = row < (long long)T * Hq;
  float sum = 0.f;
  if (live && c < D) {
    const uint4 x = ld_nc_v4(o + row * D + c), z = ld_nc_v4(o_rest + row * D + c), y = ld_nc_v4(d_o + row * D + c);
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, zs[4] = {z.x, z.y, z.z, z.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sum = fmaf(bf16_lo(xs[i]) + bf16_lo(zs[i]), bf16_lo(ys[i]), fmaf(bf16_hi(xs[i]) + bf16_hi(zs[i]), bf16_hi(ys[i]), sum));
  }
#pragma unroll
  for (int s = L / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  if (live && c == 0) delta[row % Hq * T + row / Hq] = sum;
}

// ---------------------------------------------------------------- backward: dK and dV
// An item is a tile of keys: its CTA works through the queries that see it, head by head of the group (or of a part of it: dkv_parts), so that
// dK and dV stay in tensor memory and no sum needs an atomic.  Scores transposed (a row is a key): P^T and dS^T are the A operands of
// dV = P^T dO and dK = dS^T Q.  Warps 0-7: elementwise, a thread has 64 of the 128 queries of a row; warp 8: TMA; warp 9: MMA; warp 10: items;
// warp 11: lse and delta, and the rows of other sequences in a tile.  Scores have kScores places, P(i) takes that of S(i).  Order of products:
// S(0) dP(0) .. S(kScores - 1) | dV(i) S(i + kScores) after P(i), dK(i) dP(i+1) after dS(i): exponentials are made while dK and dP
// run, dS while dV and S do, and with two places, which dV and dK leave at D <= 64, the next scores are there when dS has been made (8192
// rows, 32 heads over 8: 567 us, with one place 715).  dS is rounded to bf16 for its products, as p is: of the error of dQ and dK (2.5e-3 of their
// norm) that is as much as their own rounding; where both tiles are a sequence's first (the norm is largest there) what that left of dS and p is
// multiplied too (8191 rows in 13 sequences, 16 heads over 4, D = 64: 97 us and an error of 2.0e-3, without 90 and 2.4e-3).
// One sequence of 16,384, 16 heads over 2, D = 128: 1.75 ms, 2650 cycles for a pair of tiles whose four products take 2048.
constexpr int kBwdThreads = 384;
template <int DP>
struct DkvShape {
  static constexpr int kScores = DP == 64 ? 2 : 1, kStages = DP == 64 ? 4 : 2;
  static constexpr int kSmem = (2 + 2 * kStages) * kTileBytes<DP> + kStaging + kStages * 2 * kTile * 4 + kBarriers;
};

template <int DP>
__global__ void __launch_bounds__(kBwdThreads, 1) dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                                             const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                                                             const Args a) {
  constexpr int ST = DkvShape<DP>::kStages, NS = DkvShape<DP>::kScores, TB = kTileBytes<DP>;
  extern __shared__ __align__(1024) uint8_t attn_smem[];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ Plan s_plan;
  const uint32_t base = ptx::smem_u32(attn_smem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) raise_status(LEWI_STATUS_SMEM_LAYOUT);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t k_at = base, v_at = base + TB, ring = base + 2 * TB;   // [stage][Q, dO]
  float* stats = reinterpret_cast<float*>(attn_smem + (2 + 2 * ST) * TB + kStaging);   // [stage][-lse, -delta][128]
  const uint32_t bars = base + (2 + 2 * ST) * TB + kStaging + ST * 2 * kTile * 4;
  const uint32_t k_full = bars, v_full = bars + 8, dp_full = bars + 24, ds_ready = bars + 40, acc_full = bars + 48,
                 k_empty = bars + 64, v_empty = bars + 72, acc_empty = bars + 80;
  auto q_full = [&](int n) { return bars + 88u + 8u * (n % ST); };
  auto q_empty = [&](int n) { return bars + 88u + 8u * (ST + n % ST); };
  auto do_full = [&](int n) { return bars + 88u + 8u * (2 * ST + n % ST); };
  auto do_empty = [&](int n) { return bars + 88u + 8u * (3 * ST + n % ST); };
  auto st_full = [&](int n) { return bars + 88u + 8u * (4 * ST + n % ST); };
  auto st_empty = [&](int n) { return bars + 88u + 8u * (5 * ST + n % ST); };
  auto q_raw = [&](int n) { return bars + 88u + 8u * (6 * ST + n % ST); };
  auto do_raw = [&](int n) { return bars + 88u + 8u * (7 * ST + n % ST); };
  auto s_full = [&](int n) { return bars + 88u + 8u * (8 * ST + n % NS); };
  auto p_ready = [&](int n) { return bars + 32u + 24u * (n % NS); };   // (with two places the next P can be there before this one is waited for)
  volatile int* abort_flag = &s_abort;
  const ItemQueue items{&s_plan, bars + 88u + 8u * (8 * ST + NS), abort_flag};
  if (threadIdx.x == 0) {
    for (uint32_t b : {k_full, v_full, k_empty, v_empty, dp_full, acc_full}) ptx::mbar_init(b, 1);
    for (int n = 0; n < NS; ++n) {
      ptx::mbar_init(s_full(n), 1);
      ptx::mbar_init(p_ready(n), 8);
    }
    for (uint32_t b : {ds_ready, acc_empty}) ptx::mbar_init(b, 8);
    for (int s = 0; s < ST; ++s) {
      for (uint32_t b : {q_full(s), q_empty(s), do_full(s), do_empty(s), st_full(s), q_raw(s), do_raw(s)}) ptx::mbar_init(b, 1);
      ptx::mbar_init(st_empty(s), 8);
    }
    items.init(11);
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
  const uint32_t tmem = s_tmem, t_dp = tmem + NS * 128, t_dv = t_dp + 128, t_dk = t_dv + DP;
  auto t_s = [&](int n) { return tmem + n % NS * 128; };

  // An item's products: tile `key` of the keys with the tiles key .. key + per_head - 1 of the queries, head by head.
  struct Span {
    int hk, part, key, per_head, head0, n_it;
  };
  auto span_of = [&](const Item& w) {
    Span s;
    s.hk = w.sub % a.Hkv;
    s.part = w.sub / a.Hkv;
    s.key = (w.len + kTile - 1) / kTile - 1 - w.level;   // the first keys have the most queries
    s.per_head = w.level + 1;
    const int first = s.part * a.G / a.parts;
    s.head0 = s.hk * a.G + first;
    s.n_it = s.per_head * ((s.part + 1) * a.G / a.parts - first);
    return s;
  };

  if (warp == 8) {
    bool ok = true;
    int n = 0;
    for (int r = 0; ok; ++r) {
      const Item w = items.take(r);
      if (w.level < 0) break;
      const Span sp = span_of(w);
      ok = warp_wait(k_empty, (r & 1) ^ 1u, abort_flag);
      if (!ok) break;
      if (ptx::elect_one()) {
        ptx::mbar_expect_tx(k_full, TB);
        load_tile<DP>(k_at, &tm_k, k_full, sp.hk, w.start + sp.key * kTile);
      }
      __syncwarp();
      for (int it = 0; it < sp.n_it; ++it, ++n) {
        const int row = (sp.key + it % sp.per_head) * kTile, head = sp.head0 + it / sp.per_head;
        const uint32_t ph = (n / ST & 1) ^ 1u, at = ring + n % ST * 2 * TB;
        ok = warp_wait(q_empty(n), ph, abort_flag);
        if (!ok) break;
        bring_tile<DP>(at, &tm_q, q_full(n), q_raw(n), head, w.start + row, w.len - row);
        if (it == 0) {   // (V is wanted after the first scores only)
          ok = warp_wait(v_empty, (r & 1) ^ 1u, abort_flag);
          if (!ok) break;
          if (ptx::elect_one()) {
            ptx::mbar_expect_tx(v_full, TB);
            load_tile<DP>(v_at, &tm_v, v_full, sp.hk, w.start + sp.key * kTile);
          }
          __syncwarp();
        }
        ok = warp_wait(do_empty(n), ph, abort_flag);
        if (!ok) break;
        bring_tile<DP>(at + TB, &tm_do, do_full(n), do_raw(n), head, w.start + row, w.len - row);
      }
    }
    if (s_abort) settle();
  } else if (warp == 9) {
    const uint32_t id_s = ptx::instr_desc_bf16(128, 128, 0, 0), id_d = ptx::instr_desc_bf16(128, DP, 0, 1);
    if (ptx::elect_one()) {
      bool ok = true;
      int n = 0, chain = 0;   // chains so far
      for (int r = 0; ok; ++r) {
        const Item w = items.take_alone(r);
        if (w.level < 0) break;
        const Span sp = span_of(w);
        const int n_it = sp.n_it, to_first = sp.per_head;   // pairs of tiles from a first one of both to the next
        int at_first = sp.key == 0 ? 0 : to_first + 1;       // (there is none)
        auto scores = [&](int it) {   // S^T = K Q^T
          const int x = n + it;
          if (!ptx::mbar_wait(q_full(x), x / ST & 1, abort_flag)) return false;
          ptx::tc_fence_after();
          mma_kk<DP>(t_s(x), k_at, ring + x % ST * 2 * TB, id_s);
          ptx::mma_commit(s_full(x));
          if (it + 1 == n_it) ptx::mma_commit(k_empty);
          return true;
        };
        auto dps = [&](int it) {   // dP^T = V dO^T
          const int x = n + it;
          if (!ptx::mbar_wait(do_full(x), x / ST & 1, abort_flag)) return false;
          ptx::tc_fence_after();
          mma_kk<DP>(t_dp, v_at, ring + x % ST * 2 * TB + TB, id_s);
          ptx::mma_commit(dp_full);
          if (it + 1 == n_it) ptx::mma_commit(v_empty);
          return true;
        };
        ok = ptx::mbar_wait(k_full, r & 1, abort_flag) && scores(0) && ptx::mbar_wait(v_full, r & 1, abort_flag) && dps(0) &&
             (NS == 1 || n_it == 1 || scores(1));
        for (int it = 0; ok && it < n_it; ++chain) {
          const int len = min(kChain, n_it - it);
          for (int k = 0; ok && k < len; ++k, ++it) {
            const int x = n + it, at = ring + x % ST * 2 * TB;
            ok = ptx::mbar_wait(p_ready(x), x / NS & 1, abort_flag) && (k > 0 || ptx::mbar_wait(acc_empty, (chain & 1) ^ 1u, abort_flag));
            if (!ok) break;
            ptx::tc_fence_after();
            mma_tm<0, 8>(t_dv, t_s(x), at + TB, id_d, k > 0, 64);
            const bool first = at_first == 0;
            if (++at_first == to_first) at_first = 0;
            if (first) mma_tm<0, 8>(t_dv, t_s(x) + 32, at + TB, id_d, true, 64);
            ptx::mma_commit(do_empty(x));
            if (it + NS < n_it) ok = scores(it + NS);
            ok = ok && ptx::mbar_wait(ds_ready, x & 1, abort_flag);
            if (!ok) break;
            ptx::tc_fence_after();
            mma_tm<0, 8>(t_dk, t_dp, at, id_d, k > 0, 64);
            if (first) mma_tm<0, 8>(t_dk, t_dp + 32, at, id_d, true, 64);
            ptx::mma_commit(q_empty(x));
            if (k + 1 == len) ptx::mma_commit(acc_full);
            if (it + 1 < n_it) ok = dps(it + 1);
          }
        }
        n += n_it;
      }
      if (s_abort) settle();
    }
    __syncwarp();
  } else if (warp == 10) {
    items.run(a.seqs, kTile, a.Hkv * a.parts);
  } else if (warp == 11) {
    grid_launch();   // (delta's kernel was complete when this one began, so it is also for dQ's)
    zero_gaps(a.seqs, a.dk, a.Hkv * a.D / 8);
    zero_gaps(a.seqs, a.dv, a.Hkv * a.D / 8);
    bool ok = true;
    int n = 0;
    uint32_t phases = 0;   // of the raw barriers, a bit per stage
    for (int r = 0; ok; ++r) {
      const Item w = items.take(r);
      if (w.level < 0) break;
      const Span sp = span_of(w);
      for (int it = 0; it < sp.n_it; ++it, ++n) {
        const long long at = (long long)(sp.head0 + it / sp.per_head) * a.seqs.T + w.start;
        float x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (sp.key + it % sp.per_head) * kTile + lane + 32 * i;
          x[i] = row < w.len ? -a.lse[at + row] : -INFINITY;   // (behind the end: p = 0)
          y[i] = row < w.len ? -a.delta[at + row] : 0.f;
        }
        ok = warp_wait(st_empty(n), (n / ST & 1) ^ 1u, abort_flag);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          stats[n % ST * 2 * kTile + lane + 32 * i] = x[i];
          stats[(n % ST * 2 + 1) * kTile + lane + 32 * i] = y[i];
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(st_full(n));
        const int valid = w.len - (sp.key + it % sp.per_head) * kTile;
        if (valid < kTile) {
          const uint32_t at_q = ring + n % ST * 2 * TB, phase = phases >> n % ST;
          ok = mend_tile<DP>(at_q, q_full(n), q_raw(n), phase, valid, abort_flag) && mend_tile<DP>(at_q + TB, do_full(n), do_raw(n), phase, valid, abort_flag);
          phases ^= 1u << n % ST;
          if (!ok) break;
        }
      }
    }
  } else {
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const F2 scale = f2(a.scale_log2, a.scale_log2);
    bool ok = true;
    int n = 0, chain = 0;
    // this warp's pieces of 32 columns: of dV, then of dK
    auto column = [&](int i) { return half * (DP / 2) + i % (DP / 64) * 32; };
    auto kept_at = [&](int i) { return a.chain_kv + ((long long)blockIdx.x * (DP / 2) + (i < DP / 64 ? 0 : DP / 4) + column(i) / 4) * kTile + row; };
    auto piece = [&](int i, uint32_t (&v)[32]) {
      ptx::tmem_ld_32x32((i < DP / 64 ? t_dv : t_dk) + lanes + column(i), v);
      ptx::tmem_ld_wait();
    };
    auto free_sums = [&] {
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(acc_empty);
      ++chain;
    };
    for (int r = 0; ok; ++r) {
      const Item w = items.take(r);
      if (w.level < 0) break;
      const Span sp = span_of(w);
      auto block = [&](bool diagonal, auto first) {   // (first: both tiles are a sequence's first; apart, so that the others do not pay for it)
        const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(stats + n % ST * 2 * kTile + half * 64);   // (both negative, in pairs)
        const ulonglong2* delta = reinterpret_cast<const ulonglong2*>(stats + (n % ST * 2 + 1) * kTile + half * 64);
        if (!warp_wait(st_full(n), n / ST & 1, abort_flag) || !warp_wait(s_full(n), n / NS & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        F2 p[32];
        uint32_t x[2][32], out[32];
        ptx::tmem_ld_32x32(t_s(n) + lanes + half * 64, x[0]);
        ptx::tmem_ld_32x32(t_s(n) + lanes + half * 64 + 32, x[1]);
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
        ptx::tmem_st_32x32(t_s(n) + lanes + half * 64, out);
        if constexpr (first.value) {
#pragma unroll
          for (int i = 0; i < 32; ++i) out[i] = rest_bf16(p[i], out[i]);
          ptx::tmem_st_32x32(t_s(n) + lanes + half * 64 + 32, out);
        }
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_ready(n));
        if (!warp_wait(dp_full, n & 1, abort_flag)) return false;
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
        if constexpr (first.value) {
#pragma unroll
          for (int i = 0; i < 32; ++i) out[i] = rest_bf16(p[i], out[i]);
          ptx::tmem_st_32x32(t_dp + lanes + half * 64 + 32, out);
        }
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(ds_ready);
          ptx::mbar_arrive(st_empty(n));
        }
        ++n;
        return true;
      };
      for (int it = 0, i = 0;;) {
        for (const int end = min(it + kChain, sp.n_it); ok && it < end; ++it) {
          if (__builtin_expect(i > 0 || sp.key > 0, 1)) ok = block(i == 0, std::false_type());
          else ok = block(true, std::true_type());
          if (++i == sp.per_head) i = 0;
        }
        if (!ok || it == sp.n_it) break;
        ok = warp_wait(acc_full, chain & 1, abort_flag);   // a chain ends: the sums so far are kept, and start from zero
        if (!ok) break;
        ptx::tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t v[32];
          piece(c, v);
          if (it > kChain) add_chain(v, kept_at(c));
          put_chain(v, kept_at(c));
        }
        free_sums();
      }
      ok = ok && warp_wait(acc_full, chain & 1, abort_flag);
      if (!ok) break;
      ptx::tc_fence_after();
      if (__builtin_expect(sp.n_it > kChain, 0)) {   // (the last chain and the others, for what follows)
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t v[32];
          piece(c, v);
          add_chain(v, kept_at(c));
          ptx::tmem_st_32x32((c < DP / 64 ? t_dv : t_dk) + lanes + column(c), v);
        }
        ptx::tmem_st_wait();
      }
      const int row0 = sp.key * kTile + (warp & 3) * 32, valid = w.len - row0;
      const long long at = ((long long)(w.start + row0) * a.Hkv + sp.hk) * a.D, plane = (long long)a.seqs.T * a.Hkv * a.D;
      uint8_t* stage = attn_smem + (2 + 2 * ST) * TB + warp * 2048;
      if (a.parts == 1) {
        uint32_t out[DP / 32][16];
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          uint32_t v[32];
          piece(i, v);
          pack_row(out[i], v, i < DP / 64 ? 1.f : a.scale);
        }
        free_sums();   // (the next item's products may go on)
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
          store_rows(stage, out[i], reinterpret_cast<uint8_t*>((i < DP / 64 ? a.dv : a.dk) + at + column(i)), (long long)a.Hkv * a.D * 2, valid,
                     (a.D - column(i)) * 2);
      } else {
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          uint32_t v[32], out[16];
          piece(i, v);
          float* dst = a.sums + (2 * sp.part + (i < DP / 64 ? 0 : 1)) * plane + at + column(i);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            half_row(out, v, h, i < DP / 64 ? 1.f : a.scale);
            store_rows(stage, out, reinterpret_cast<uint8_t*>(dst + h * 16), (long long)a.Hkv * a.D * 4, valid, (a.D - column(i) - h * 16) * 4);
          }
        }
        free_sums();
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
// An item is a tile of queries of one head: its CTA works through the keys that it sees, with S and dP as in the forward pass.  Scores have two
// places in tensor memory, so that S(j+1) is there when dS(j) has been made; dS(j) takes the place of S(j).  Warps as above; warp 11: rows of
// no sequence and of other ones.  Its CTAs begin where those for dK and dV have finished;
// the kernel for dK and dV itself begins only when delta's is complete, so that this one may rely on delta as on every operand (8191 rows in 13
// sequences, 16 heads over 4, D = 64, forward and backward: 200 us, and 209 where that kernel began early as well; 1000 rows, 16 over 2: 64 and 60).
// Order of products: S(0) dP(0) S(1) | dP(j+1) dQ(j) S(j+2) after dS(j).
// Two kernels make seven products of a pair of tiles where one would make five, but that one would have to add to dQ from every tile
// of keys, in an order that changes, or wait for its turn.  One sequence of 16,384, 16 heads over 2, D = 128: 1.2 ms.
// S(j+2) waits for K(j+2), whose place is that of K(j) where there are four: five places take what the staging would (8192 x 32 heads, D = 128:
// 650 us with five, 780 with four), so at D = 128 dQ is stored row by row.
// At D = 64 three products take 770 cycles of 1640 for a pair of tiles, and what the warp that issues them does between them counts: it loops as a whole over
// values that all its lanes share, with one elected for the instructions (8192 x 32 heads: 442 us as a loop of one thread, 405 so), and K and V come
// as pairs on one barrier (398; 408 since there are chains).  The forward pass and the kernel for dK and dV, which wait for their exponentials, lose 2 % by the former.
template <int DP>
struct DqShape {
  static constexpr bool kPairs = DP == 64, kStaged = DP == 64;   // (a place is K's and V's)
  static constexpr int kStages = kPairs ? 4 : 5;
  static constexpr int kSmem = (2 + (kPairs ? 2 : 1) * kStages) * kTileBytes<DP> + (kStaged ? kStaging : 0) + kBarriers;
};

template <int DP>
__global__ void __launch_bounds__(kBwdThreads, 1) dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                                            const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                                                            const Args a) {
  constexpr bool PAIRS = DqShape<DP>::kPairs;
  constexpr int ST = DqShape<DP>::kStages, TB = kTileBytes<DP>, PLACE = PAIRS ? 2 * TB : TB;
  extern __shared__ __align__(1024) uint8_t attn_smem[];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ Plan s_plan;
  const uint32_t base = ptx::smem_u32(attn_smem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) raise_status(LEWI_STATUS_SMEM_LAYOUT);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t q_at = base, do_at = base + TB, kv = base + 2 * TB, bars = kv + ST * PLACE + (DqShape<DP>::kStaged ? kStaging : 0);
  const uint32_t q_full = bars, do_full = bars + 8, q_empty = bars + 16, do_empty = bars + 24, dp_full = bars + 32, ds_ready = bars + 40, acc_full = bars + 48,
                 acc_empty = bars + 56;
  auto s_full = [&](int b) { return bars + 72u + 8u * (b & 1); };
  auto full = [&](int n) { return bars + 88u + 8u * (n % ST); };
  auto empty = [&](int n) { return bars + 88u + 8u * (ST + n % ST); };
  auto raw = [&](int n) { return bars + 88u + 8u * (2 * ST + n % ST); };
  volatile int* abort_flag = &s_abort;
  const ItemQueue items{&s_plan, bars + 88u + 24u * ST, abort_flag};
  if (threadIdx.x == 0) {
    for (uint32_t b : {q_full, do_full, q_empty, do_empty, dp_full, acc_full, s_full(0), s_full(1)}) ptx::mbar_init(b, 1);
    for (uint32_t b : {ds_ready, acc_empty}) ptx::mbar_init(b, 8);
    for (int s = 0; s < ST; ++s) {
      ptx::mbar_init(full(s), PAIRS ? 2 : 1);
      for (uint32_t b : {empty(s), raw(s)}) ptx::mbar_init(b, 1);
    }
    items.init(11);
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
  auto t_s = [&](int b) { return tmem + (b & 1) * 128; };   // (b: blocks so far)

  if (warp == 8) {   // Q, dO, K0, V0, K1, V1, ..
    bool ok = true;
    int n = 0;
    for (int r = 0; ok; ++r) {
      const Item w = items.take(r);
      if (w.level < 0) break;
      const int q_row = w.start + w.level * kTile, nb = w.level + 1, hk = w.sub / a.G;
      ok = warp_wait(q_empty, (r & 1) ^ 1u, abort_flag) && warp_wait(do_empty, (r & 1) ^ 1u, abort_flag);
      if (!ok) break;
      if (ptx::elect_one()) {
        ptx::mbar_expect_tx(q_full, TB);
        load_tile<DP>(q_at, &tm_q, q_full, w.sub, q_row);
        ptx::mbar_expect_tx(do_full, TB);
        load_tile<DP>(do_at, &tm_do, do_full, w.sub, q_row);
      }
      __syncwarp();
      for (int j = 0; ok && j < nb; ++j, ++n) {
        ok = warp_wait(empty(n), (n / ST & 1) ^ 1u, abort_flag);
        if (!ok) break;
        bring_tile<DP>(kv + n % ST * PLACE, &tm_k, full(n), raw(n), hk, w.start + j * kTile, w.len - j * kTile);
        if (!PAIRS) {
          ++n;
          ok = warp_wait(empty(n), (n / ST & 1) ^ 1u, abort_flag);
          if (!ok) break;
        }   // (of V a foreign row only reaches pairs that are masked)
        bring_tile<DP>(kv + n % ST * PLACE + (PAIRS ? TB : 0), &tm_v, full(n), raw(n), hk, w.start + j * kTile, kTile);
      }
    }
    if (s_abort) settle();
  } else if (warp == 9) {
    const uint32_t id_s = ptx::instr_desc_bf16(128, 128, 0, 0), id_d = ptx::instr_desc_bf16(128, DP, 0, 1);
    bool ok = true;
    constexpr int STEP = PAIRS ? 1 : 2;
    At<ST> ks{0, 0}, vs{PAIRS ? 0 : 1, 0}, ds{0, 0};   // K of the next S, V of the next dP, K of the next dQ
    uint32_t bs = 0, b = 0, chain = 0;     // blocks of S and of dQ and chains so far
    for (uint32_t r = 0; ok; ++r) {
      const Item w = items.take(r);
      const int nb = __shfl_sync(0xffffffffu, w.level, 0) + 1;
      if (nb <= 0) break;
      auto scores = [&](int j) {
        if (!warp_wait(full(ks.s), ks.phase, abort_flag)) return false;
        if (ptx::elect_one()) {
          ptx::tc_fence_after();
          mma_kk<DP>(t_s(bs), q_at, kv + ks.s * PLACE, id_s);
          ptx::mma_commit(s_full(bs));
          if (j + 1 == nb) ptx::mma_commit(q_empty);
        }
        __syncwarp();
        ++bs;
        ks.on(STEP);
        return true;
      };
      auto dps = [&](int j) {
        if (!PAIRS && !warp_wait(full(vs.s), vs.phase, abort_flag)) return false;
        if (ptx::elect_one()) {
          ptx::tc_fence_after();
          mma_kk<DP>(t_dp, do_at, kv + vs.s * PLACE + (PAIRS ? TB : 0), id_s);
          ptx::mma_commit(dp_full);
          if (!PAIRS) ptx::mma_commit(empty(vs.s));
          if (j + 1 == nb) ptx::mma_commit(do_empty);
        }
        __syncwarp();
        vs.on(STEP);
        return true;
      };
      ok = warp_wait(q_full, r & 1, abort_flag) && scores(0) && warp_wait(do_full, r & 1, abort_flag) && dps(0) && (nb < 2 || scores(1));
      for (int j = 0; ok && j < nb; ++chain) {
        const int len = min(kChain, nb - j);
        for (int k = 0; ok && k < len; ++k, ++j) {
          ok = warp_wait(ds_ready, b & 1, abort_flag) && (j + 1 >= nb || dps(j + 1)) && (k > 0 || warp_wait(acc_empty, (chain & 1) ^ 1u, abort_flag));
          if (!ok) break;
          if (ptx::elect_one()) {
            ptx::tc_fence_after();
            mma_tm<0, 8>(t_dq, t_s(b), kv + ds.s * PLACE, id_d, k > 0, 64);
            if (nb == 1) mma_tm<0, 8>(t_dq, t_s(b) + 32, kv + ds.s * PLACE, id_d, true, 64);
            ptx::mma_commit(empty(ds.s));
            if (k + 1 == len) ptx::mma_commit(acc_full);
          }
          __syncwarp();
          ++b;
          ds.on(STEP);
          if (j + 2 < nb) ok = scores(j + 2);
        }
      }
    }
    if (s_abort) settle();
    __syncwarp();
  } else if (warp == 10) {
    items.run(a.seqs, kTile, a.Hq);
  } else if (warp == 11) {
    zero_gaps(a.seqs, a.dq, a.Hq * a.D / 8);
    bool ok = true;
    int n = 0;
    uint32_t phases = 0;   // of the raw barriers, a bit each
    for (int r = 0; ok; ++r) {
      const Item w = items.take(r);
      if (w.level < 0) break;
      const int valid = w.len - w.level * kTile, s = (n + (PAIRS ? 1 : 2) * w.level) % ST;   // of the last keys
      n += (PAIRS ? 1 : 2) * (w.level + 1);
      if (valid >= kTile) continue;
      ok = mend_tile<DP>(kv + s * PLACE, full(s), raw(s), phases >> s, valid, abort_flag);
      phases ^= 1u << s;
    }
  } else {
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const F2 scale = f2(a.scale_log2, a.scale_log2);
    bool ok = true;
    int b = 0, chain = 0;
    auto kept_at = [&](int i) { return a.chain_q + ((long long)blockIdx.x * (DP / 4) + (half * (DP / 2) + i * 32) / 4) * kTile + row; };
    auto piece = [&](int i, uint32_t (&v)[32]) {
      ptx::tmem_ld_32x32(t_dq + lanes + half * (DP / 2) + i * 32, v);
      ptx::tmem_ld_wait();
    };
    auto free_sums = [&] {
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(acc_empty);
      ++chain;
    };
    // delta: from the kernel before this one, or from one that was complete, with its writes visible, before that one (dK and dV) began
    if (a.dk == nullptr) grid_wait();
    for (int r = 0; ok; ++r) {
      const Item w = items.take(r);
      if (w.level < 0) break;
      const int nb = w.level + 1, in_seq = w.level * kTile + row;
      const long long at = (long long)w.sub * a.seqs.T + w.start + in_seq;
      const float lse = in_seq < w.len ? a.lse[at] : INFINITY, delta = in_seq < w.len ? a.delta[at] : 0.f;
      const F2 shift = f2(-lse, -lse), minus_delta = f2(-delta, -delta);
      auto block = [&](int j, auto first) {   // (first: the rows and the keys are a sequence's first; apart, so that the others do not pay for it)
        if (!warp_wait(s_full(b), b >> 1 & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        F2 p[32];
        uint32_t x[2][32], ds[32];
        ptx::tmem_ld_32x32(t_s(b) + lanes + half * 64, x[0]);
        ptx::tmem_ld_32x32(t_s(b) + lanes + half * 64 + 32, x[1]);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) p[i] = ex2_pair<kBwdPoly<DP>>(x[i / 16][i % 16 * 2], x[i / 16][i % 16 * 2 + 1], scale, shift, i);
        if (!warp_wait(dp_full, b & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        ptx::tmem_ld_32x32(t_dp + lanes + half * 64, x[0]);
        ptx::tmem_ld_32x32(t_dp + lanes + half * 64 + 32, x[1]);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          p[i] = mul2(p[i], add2(f2(__uint_as_float(x[i / 16][i % 16 * 2]), __uint_as_float(x[i / 16][i % 16 * 2 + 1])), minus_delta));
        if (j + 1 == nb) {   // the diagonal
#pragma unroll
          for (int i = 0; i < 32; ++i) p[i] = hide(p[i], half * 64 + 2 * i > row, half * 64 + 2 * i + 1 > row);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) ds[i] = f2_bf16(p[i]);
        ptx::tmem_st_32x32(t_s(b) + lanes + half * 64, ds);
        if constexpr (first.value) {
#pragma unroll
          for (int i = 0; i < 32; ++i) ds[i] = rest_bf16(p[i], ds[i]);
          ptx::tmem_st_32x32(t_s(b) + lanes + half * 64 + 32, ds);
        }
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ds_ready);
        ++b;
        return true;
      };
      if (__builtin_expect(nb > 1, 1)) {
        for (int j = 0;;) {
          for (const int end = min(j + kChain, nb); ok && j < end; ++j) ok = block(j, std::false_type());
          if (!ok || j == nb) break;
          ok = warp_wait(acc_full, chain & 1, abort_flag);   // a chain ends: dQ so far is kept, and starts from zero
          if (!ok) break;
          ptx::tc_fence_after();
#pragma unroll 1
          for (int i = 0; i < DP / 64; ++i) {
            uint32_t v[32];
            piece(i, v);
            if (j > kChain) add_chain(v, kept_at(i));
            put_chain(v, kept_at(i));
          }
          free_sums();
        }
      } else {
        ok = block(0, std::true_type());
      }
      ok = ok && warp_wait(acc_full, chain & 1, abort_flag);
      if (!ok) break;
      ptx::tc_fence_after();
      if (__builtin_expect(nb > kChain, 0)) {   // (the last chain and the others, for what follows)
#pragma unroll 1
        for (int i = 0; i < DP / 64; ++i) {
          uint32_t v[32];
          piece(i, v);
          add_chain(v, kept_at(i));
          ptx::tmem_st_32x32(t_dq + lanes + half * (DP / 2) + i * 32, v);
        }
        ptx::tmem_st_wait();
      }
      uint32_t out[DP / 64][16];
#pragma unroll
      for (int i = 0; i < DP / 64; ++i) {
        uint32_t v[32];
        piece(i, v);
        pack_row(out[i], v, a.scale);
      }
      free_sums();
      const int row0 = w.level * kTile + (warp & 3) * 32;
#pragma unroll
      for (int i = 0; i < DP / 64; ++i) {
        const int c = half * (DP / 2) + i * 32;
        uint8_t* dst = reinterpret_cast<uint8_t*>(a.dq + ((long long)(w.start + row0) * a.Hq + w.sub) * a.D + c);
        const long long stride = (long long)a.Hq * a.D * 2;
        if constexpr (DqShape<DP>::kStaged) {
          store_rows(attn_smem + 2 * TB + ST * PLACE + warp * 2048, out[i], dst, stride, w.len - row0, (a.D - c) * 2);
        } else if (lane < w.len - row0) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (u * 8 < a.D - c) st_v4(dst + lane * stride + u * 16, make_uint4(out[i][4 * u], out[i][4 * u + 1], out[i][4 * u + 2], out[i][4 * u + 3]));
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
  grid_wait();   // this kernel may have begun while the one for dK and dV was finishing; what follows it follows both
}

// ---------------------------------------------------------------- host side
// [T][heads][D] rows `row` elements and heads D elements apart, boxes of 128 rows x 64 columns of one head
inline bool make_rows_map(CUtensorMap* m, const void* p, int T, int heads, int D, long long row) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)row * 2};
  const cuuint32_t box[3] = {64, 1, kTile};
  return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p, dims, strides, box);
}

// Pairs of tiles of the longest row of tiles, and an SM's share of all of them.  What lengths several sequences have only the device knows: the longest
// is taken to be three times the mean, which is far off where one is long and many are short (4096 + 400 x 10 rows, 32 heads over 1: two parts for dK
// and dV, where by the costs below six would be best).
struct Blocks {
  double longest, share;
};
inline Blocks blocks_of(int T, int n_seqs, int Hq) {
  const double tiles = (double)T / kTile + 0.5 * n_seqs, mean = tiles / n_seqs, longest = n_seqs == 1 ? mean : 3 * mean < tiles ? 3 * mean : tiles;
  return {longest, tiles * (mean + 1) / 2 * Hq / num_sms()};
}

// An item of the forward pass is two heads or two tiles, or one tile where that is over sooner: a block of the former takes 1.6 us for its two
// tiles, of the latter 1.15 us for one (at D = 128; D = 64 goes by the same), and an SM is done with its share or with the longest item.  One sequence, 16 heads over 2, D = 128, two
// heads and one tile: of 256 rows 9.9 and 8.1 us, 1000 19 and 14, 2048 32 and 23, 4096 57 and 65.
inline FwdItem fwd_item(int T, int n_seqs, int Hq, int G) {
  const Blocks b = blocks_of(T, n_seqs, Hq);
  const double two = b.longest > b.share / 2 ? 1.6 * b.longest : 0.8 * b.share, one = 1.15 * (b.longest > b.share ? b.longest : b.share);
  return one < two ? kOneTile : G % 2 == 0 ? kTwoHeads : kTwoTiles;
}

// In how many parts, each a CTA's item, a group's heads are worked through for a tile of dK and dV.  The tile of a long sequence's first keys
// has all its queries, times G heads, so few key heads leave a few long items, while parts cost their way through memory (float32, written and
// read).  Taken is what comes out shortest of the longest item or an even share of everything, at 1.6 us per pair of tiles, and the parts'
// bytes at 5 TB/s.  One sequence of 1000, 16 heads over 2:
// 128 us in one part, 30 in eight; of 16,384: 1975 and 1800 in two.
inline int dkv_parts(int T, int n_seqs, int Hq, int Hkv, int D) {
  const auto [longest, share] = blocks_of(T, n_seqs, Hq);
  int best = 1;
  double least = 0;
  for (int p = 1; p <= Hq / Hkv; ++p) {
    const double item = longest * ((Hq / Hkv + p - 1) / p), us = 1.6 * (item > share ? item : share) + (p > 1 ? 16.0 * T * Hkv * D * p / 5e6 : 0.0);
    if (p == 1 || us < least) {
      best = p;
      least = us;
    }
    if (item <= share) break;   // (more parts only cost their bytes; after some hundreds at most, however many heads share keys)
  }
  return best;
}

inline unsigned ctas(long long items) { return (unsigned)(items < num_sms() ? items : num_sms()); }

// Bytes of the sums of chains, for dV and dK and for dQ: none where no item can have more than kChain pairs of tiles.
inline long long chain_kv_bytes(int T, int G, int parts, int D) {
  return ((long long)T + kTile - 1) / kTile * ((G + parts - 1) / parts) > kChain ? (long long)num_sms() * (D <= 64 ? 64 : 128) * kTile * 8 : 0;
}
inline long long chain_q_bytes(int T, int D) { return T > kChain * kTile ? (long long)num_sms() * (D <= 64 ? 64 : 128) * kTile * 4 : 0; }

// Tiles that `n` sequences of together T rows can have at most.
inline long long most_tiles(int T, int n) { return (long long)T / kTile + n; }

}  // namespace attn
}  // namespace lewi
