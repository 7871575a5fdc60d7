// Attention in which every query sees a span of keys: query i of sequence b
// sees first[b, i] <= j < last[b, i] (two ints a position) in place of the
// causal rule of attn.cu -- rows that pack several documents, prompts seen in
// both directions, sliding windows, padding -- forward and backward, and the
// spans of packed documents.  The reference has no such mode (its node takes a
// causal mode or a mask tensor: engine/src/interp.rs:405-432).
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j - lse_i) for j in the span
//   dP = dO V^T,  delta_i = sum_d dO_id O_id,  dS = P * (dP - delta)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
// Layouts as in attn.cu: q, o [batch, seq, heads, dim], k, v [batch, seq,
// kv_heads, dim] bf16, lse [batch, heads, seq] f32 (natural logarithm).  A query
// that sees nothing gets o = 0, lse = -inf and no gradient.  P, dS and the
// results are rounded to bf16, every sum is f32.
//
// What short documents ask for, and how the kernels differ from attn.cu's:
// * A query tile's rows are the `pack` heads that share a key/value head at a
//   few positions (row = position * pack + head, the order in which a box {64
//   dims, pack heads, positions} lands), not one head's at 128: its rows see
//   nearly the same keys, so little of a key tile is masked at a document's
//   borders, and the heads share the key tile.  Key tiles that no row sees are
//   neither loaded nor multiplied; 32-column chunks that no row of a warp sees
//   are not read, those that all see take the unmasked code.
// * A query tile of a short document has two to six key tiles.  With one CTA
//   a tile, its start (barriers, tensor memory, the first copies: some 6000
//   cycles) and end (4000) were half of its life.  The CTAs stay (one an SM)
//   and take the work of CTAs that have not started (cluster launch control:
//   how long a tile lasts depends on the spans, and a fixed share each left
//   SMs idle for a quarter to a third of the time), a little before their own
//   ends: a scheduler warp reads the next tile's spans, its copies and first
//   product run while the last one's results are stored.
// * Two threads issue a CTA's matrix products, each the chains that depend on
//   themselves only.  A wait costs a thread about 100 cycles even where nothing
//   is to be waited for, a commit up to 60, and the tensor cores' queue is too
//   short to hide them: alone, the products of a forward step take 1290 cycles,
//   with one thread's waits 1800, with two threads' 1340.  (An M = 128, K = 16
//   product takes 64 cycles at N = 128 and 45 to 50 at N = 64.)
#include <cuda_bf16.h>

#include <climits>
#include <cmath>

#include "attn.cuh"

namespace tq {
namespace {

constexpr int kFwdThreads = 384;  // four warps of roles, eight of softmax
constexpr int kBwdWarps = 8;      // that compute, beside the four of roles
constexpr int kBwdThreads = 128 + 32 * kBwdWarps;
constexpr int kParts = kBwdWarps / 4;     // of a streamed 64-wide tile's columns
constexpr int kPartCols = kHalf / kParts;
constexpr int kStageBytes = 4096;  // a storing warp's (store_rows)
// Who reads a tile's description: TMA, two of MMA and every computing warp.
constexpr int kFwdReaders = 3 + 8;
constexpr int kBwdReaders = 3 + kBwdWarps;
// A row's exponentials are taken against the maximum of the first tile that it
// sees until their sum over a tile passes kMost; then against that tile's
// maximum.  P, l and O keep their relative precision at any exponent, so only
// their range counts: O is up to kMost, times the key tiles, above the values it
// sums, which at 2^20 tiles is within f32 for values up to 2^47.
constexpr float kMost = 1.152921504606846976e18f;  // 2^60
constexpr float kGrowLog2 = 50.0f;  // below 60 by more than the log of a tile's keys

struct SpanShape {
  int batch, seq, heads, kv_heads, group;
  float scale_log2;  // softmax scale * log2(e)
  // Query heads a tile holds, the positions in a 128- and a 64-row tile,
  // floor(rows / pack) (rows behind pack * positions hold zeros), and the
  // number of such tiles and of 128-key tiles in a sequence.
  int pack, pos128, pos64, tiles128, tiles64, key_tiles;
};

// A place in a ring of stages and the parity of its phase.
struct Ring {
  int stage, phase;
  __device__ void next(int stages) {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// A query's keys [lo, hi) within [0, seq); 0, 0 when it sees none.
struct Span {
  int lo, hi;
};

__device__ __forceinline__ Span load_span(const int* first, const int* last, int b, int i,
                                          int seq) {
  if (i >= seq) return {0, 0};
  const size_t at = static_cast<size_t>(b) * seq + i;
  // Plain loads: the spans may be the last kernel's, which still ran when this
  // one was started.
  const int lo = max(first[at], 0), hi = min(last[at], seq);
  return lo < hi ? Span{lo, hi} : Span{0, 0};
}

// The keys that any of the positions [i0, i0 + n) sees, [lo, hi) (0, 0 for
// none), for every lane of the calling warp.
__device__ __forceinline__ Span span_of_positions(const int* first, const int* last, int b, int i0,
                                                  int n, int seq) {
  int lo = INT_MAX, hi = 0;
  for (int i = threadIdx.x & 31; i < n; i += 32) {
    const Span s = load_span(first, last, b, i0 + i, seq);
    if (s.lo < s.hi) {
      lo = min(lo, s.lo);
      hi = max(hi, s.hi);
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  return hi > 0 ? Span{lo, hi} : Span{0, 0};
}

// Zeroes rows [from, tile_rows) of `slabs` consecutive slabs (128 bytes a row),
// which no copy fills when a packed tile has fewer rows; made visible to the
// tensor cores by each thread's fence and the barrier after it.
__device__ __forceinline__ void zero_rows(uint8_t* slab, int slabs, int tile_rows, int from) {
  const int per = (tile_rows - from) * 8;  // 16-byte words a slab
  for (int i = threadIdx.x; i < slabs * per; i += blockDim.x)
    *reinterpret_cast<uint4*>(slab + (i / per * tile_rows + from) * 128 + i % per * 16) =
        make_uint4(0, 0, 0, 0);
  if (per > 0) fence_proxy_async_smem();
}

__device__ __forceinline__ F2 exp2_mufu(F2 x) {
  const float2 v = split(x);
  return f2(ex2_approx(v.x), ex2_approx(v.y));
}

__device__ __forceinline__ F2 pair_of(uint32_t a, uint32_t b) {
  return f2(__uint_as_float(a), __uint_as_float(b));
}

__device__ __forceinline__ uint32_t pack_bf16(F2 x) {
  const float2 v = split(x);
  return pack_bf16x2_f32(v.x, v.y);
}

// Bits [a, z) of a word, 0 <= a, z <= 32.
__device__ __forceinline__ uint32_t bit_range(int a, int z) {
  if (a >= z) return 0;
  return (z == 32 ? 0xFFFFFFFFu : (1u << z) - 1u) & ~((1u << a) - 1u);
}

// 2^(r c - m) of 32 scores as bf16 pairs to pk[0, 16); their sum, in two parts.
__device__ __forceinline__ F2 exp_chunk(const uint32_t (&r)[32], F2 c, float m, uint32_t* pk) {
  const F2 shift = f2(-m, -m);
  F2 sum[2];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const F2 q = exp2_mufu(fma2(pair_of(r[2 * e], r[2 * e + 1]), c, shift));
    sum[e & 1] = e < 2 ? q : sum[e & 1] + q;
    pk[e] = pack_bf16(q);
  }
  return sum[0] + sum[1];
}

// The index of a CTA of this grid that has not started and now never will (its
// work is the caller's), or -1 if all have.  One warp; slot: 16 bytes of
// shared memory, bar: an mbarrier of one arrival, both for this alone; n: how
// many calls came before.  Not called again after a -1.
__device__ __forceinline__ int take_cta(uint32_t slot, uint32_t bar, int n, int* status) {
  if ((threadIdx.x & 31) == 0) {
    fence_proxy_async_smem();  // the last answer has been read
    mbar_arrive_expect_tx(bar, 16);
    asm volatile(
        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 "
        "[%0], [%1];" ::"r"(slot),
        "r"(bar)
        : "memory");
  }
  __syncwarp();
  if (!mbar_wait(bar, n & 1, status)) return -1;
  uint32_t x, ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b128 r;\n"
      "ld.shared.b128 r, [%2];\n"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n"
      "selp.u32 %1, 1, 0, p;\n"
      "mov.u32 %0, 0;\n"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n"
      "}\n"
      : "=r"(x), "=r"(ok)
      : "r"(slot)
      : "memory");
  __syncwarp();
  return ok ? static_cast<int>(x) : -1;
}

// Stores 2 N values (bf16 pairs) of a row a lane, through 128 N bytes of the
// warp's in shared memory: an instruction then writes whole stretches of 4 N
// bytes (from a row a lane it would write 32 bytes in each of 32 lines, and the
// warps of a forward tile stood 2000 to 4000 cycles behind their stores).
template <int N>
__device__ __forceinline__ void store_rows(uint8_t* stage, const uint32_t (&w)[N], uint16_t* row,
                                           bool valid) {
  static_assert(N == 16 || N == 32, "64 or 128 bytes a row");
  constexpr int C = N / 4;  // 16-byte chunks a row, in an order that spreads the banks
  auto at = [&](int r, int c) {
    return reinterpret_cast<uint4*>(stage + r * 4 * N + ((c ^ (N == 32 ? r & 7 : r >> 1 & 3)) << 4));
  };
  const int lane = threadIdx.x & 31;
  const uint32_t rows = __ballot_sync(0xffffffffu, valid);
  __syncwarp();  // what was here has been read
#pragma unroll
  for (int c = 0; c < C; ++c)
    *at(lane, c) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
  __syncwarp();
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int r = k * (32 / C) + lane / C, c = lane % C;
    const uint4 x = *at(r, c);
    const uint64_t to = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(row), r);
    if (rows >> r & 1) reinterpret_cast<uint4*>(to)[c] = x;
  }
}

__device__ __forceinline__ bool wide_rows(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 31u) == 0;
}

// ------------------------------------------------------------------ forward --
//
// A tile of work is a pair of adjacent packed query tiles of one sequence and
// key/value head; both share every key/value tile the pair needs.
//   warp 0       TMA: the query tiles, key and value tiles through a ring
//   warps 1, 2   one thread each issues the tcgen05 MMAs of query tile 0, 1;
//                warp 2 also allocates and frees the 512 TMEM columns
//   warp 3       scheduler: the next pairs' descriptions, two in shared memory
//   warps 4-7    softmax of query tile 0 (thread i owns row i, TMEM lane i)
//   warps 8-11   softmax of query tile 1
// TMEM: S_w,b (64 f32 columns each: key tiles of 64, two of each query tile) |
// O_0 | O_1 (dim columns each); P_w,b (bf16 pairs) over S_w,b.  Thread w issues
// S_w(0), S_w(1) and then, per key tile t,
//   O_w += P_w(t) V_t,  S_w(t+2) = Q_w K_{t+2}^T
// S_w(t+2) overwrites P_w(t), so it is issued when that product is done (the
// order of two products is given only where shape and accumulator are the same),
// and a softmax warp has its next scores while it works on these.  (With key
// tiles of 128 and one S a query tile it waited 1300 of 4000 cycles for them.)
// A softmax thread needs no maximum before the exponentials: it keeps a
// reference (kMost) and looks at its sum.  Barriers count through all pairs, and
// no waiter is two phases behind: s_full, p_ready and o_done come in two, by the
// tile's parity, and S_w(t) complete says that O_w's product t-2 is, too.
//
// Four packed rows of 2048 (32 heads over 8 of 128, some six documents a row):
// 70 us, one row of 8191 with documents of up to 2000: 122 us, 0.62 and 1.0
// PFLOP/s of what its tiles multiply.  A step of two 64-key products and two of
// 128 columns takes some 1600 to 1900 cycles of which the tensor cores need 1290
// and the exponentials 1024; the rest is a tile's end (some 4000 cycles: the last
// product, O out of tensor memory, the stores), a fifth of the short documents'
// time.

struct FwdItem {
  int b, h, t0;              // b < 0: no more; first of `pack` heads, first query tile
  int lo0, hi0, lo1, hi1;    // 64-key tiles of the two query tiles
  int pad;
};

template <int D>
struct FwdCfg {
  static_assert(D == 64 || D == 128, "head dim");
  static constexpr int SLABS = D / 64;        // 128-byte swizzle atoms along dim
  static constexpr int QSLAB = kTile * 128;   // 128 rows x 64 bf16
  static constexpr int QTILE = SLABS * QSLAB;
  static constexpr int KSLAB = kHalf * 128;   // 64 rows x 64 bf16
  static constexpr int KTILE = SLABS * KSLAB;
  // A stage holds K_{t+2} and V_t, which are wanted together.
  static constexpr int ST = D == 128 ? 4 : 8;
  static constexpr int Q_OFF = 0;  // two query tiles
  static constexpr int KV_OFF = 2 * QTILE;
  static constexpr int OUT_OFF = KV_OFF + 2 * ST * KTILE;
  static constexpr int ITEM_OFF = OUT_OFF + 8 * kStageBytes;
  static constexpr int TAKE_OFF = ITEM_OFF + 2 * static_cast<int>(sizeof(FwdItem));
  static constexpr int BAR_OFF = TAKE_OFF + 16;
  // q_full, q_empty, kv_full[ST], kv_empty[ST], s_full[2][2], p_ready[2][2],
  // o_done[2][2], o_free[2], item_full[2], item_empty[2], taken; TMEM slot
  static constexpr int NBAR = 2 + 2 * ST + 19;
  static constexpr int SMEM = 1024 + BAR_OFF + 8 * (NBAR + 1);
  static constexpr int S_COL = 0;    // S_w,b (and P_w,b) at 128 w + 64 b
  static constexpr int O_COL = 256;  // O_w at 256 + D w
  static constexpr int TMEM_COLS = 512;
  static_assert(O_COL + 2 * D <= TMEM_COLS, "tensor memory map");
  static_assert(SMEM <= 232448, "shared memory per CTA");
  static_assert(SMEM > 118784, "one CTA per SM");
};

struct FwdParams {
  SpanShape sh;
  const int* first;  // [batch, seq]
  const int* last;
  int n_pairs;
  uint16_t* out;
  float* lse;
  int* status;
};

template <int D>
__global__ void __launch_bounds__(kFwdThreads, 1)
    span_fwd_kernel(const __grid_constant__ CUtensorMap tm_q,
                    const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const FwdParams p) {
  using C = FwdCfg<D>;
  constexpr int ST = C::ST;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const gbase = smem_raw + (base - raw);
  auto q_s = [&](int w) { return base + C::Q_OFF + w * C::QTILE; };
  auto k_s = [&](int s) { return base + C::KV_OFF + 2 * s * C::KTILE; };
  auto v_s = [&](int s) { return base + C::KV_OFF + (2 * s + 1) * C::KTILE; };
  const uint32_t bars = base + C::BAR_OFF;
  const uint32_t q_full = bars, q_empty = bars + 8u;
  auto kv_full = [&](int s) { return bars + 8u * (2 + s); };
  auto kv_empty = [&](int s) { return bars + 8u * (2 + ST + s); };
  constexpr int X = 2 + 2 * ST;
  // n: which of tile w's key tiles it is, counted through all items.
  auto s_full = [&](int w, int n) { return bars + 8u * (X + 2 * w + (n & 1)); };
  auto p_ready = [&](int w, int n) { return bars + 8u * (X + 4 + 2 * w + (n & 1)); };
  auto o_done = [&](int w, int n) { return bars + 8u * (X + 8 + 2 * w + (n & 1)); };
  auto o_free = [&](int w) { return bars + 8u * (X + 12 + w); };
  auto item_full = [&](int i) { return bars + 8u * (X + 14 + i); };
  auto item_empty = [&](int i) { return bars + 8u * (X + 16 + i); };
  const uint32_t taken = bars + 8u * (X + 18);
  const uint32_t tmem_slot = bars + 8u * C::NBAR;
  volatile uint32_t* tmem_slot_ptr =
      reinterpret_cast<volatile uint32_t*>(gbase + (tmem_slot - base));
  FwdItem* const items = reinterpret_cast<FwdItem*>(gbase + C::ITEM_OFF);

  const SpanShape& sh = p.sh;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rows = sh.pack * sh.pos128;  // filled rows of a query tile

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int s = 0; s < ST; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 2);
    }
    for (int w = 0; w < 2; ++w) {
      for (int n = 0; n < 2; ++n) {
        mbar_init(s_full(w, n), 1);
        mbar_init(p_ready(w, n), 4);
        mbar_init(o_done(w, n), 1);
      }
      mbar_init(o_free(w), 4);
      mbar_init(item_full(w), 1);
      mbar_init(item_empty(w), kFwdReaders);
    }
    mbar_init(taken, 1);
    fence_mbar_init();
  }
  zero_rows(gbase + C::Q_OFF, 2 * C::SLABS, kTile, rows);
  if (warp == 2) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot_ptr;
  // Signalled only once this CTA holds its tensor memory: a dependent
  // kernel's CTA placed on this SM may then wait for it, never hold it.
  griddep_launch_dependents();
  griddep_wait();

  // The i-th item's description; one arrival a reader.
  auto wait_item = [&](int i, bool& ok) {
    FwdItem it{-1, 0, 0, 0, 0, 0, 0, 0};
    ok = mbar_wait(item_full(i & 1), (i >> 1) & 1, p.status);
    if (ok) it = items[i & 1];
    return it;
  };

  if (warp < 4) {
    if (warp == 0 && elect_one_sync()) {
      // ----------------------------------------------------------- TMA
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      int ns = 0, nq = 0;  // stages filled, query tiles issued, of all items
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const FwdItem it = wait_item(i, ok);
        if (it.b < 0) break;
        mbar_arrive(item_empty(i & 1));
        const int hk = it.h / sh.group;
        const int j0 = it.hi0 == 0 ? it.lo1 : it.hi1 == 0 ? it.lo0 : min(it.lo0, it.lo1);
        const int n_kv = max(it.hi0, it.hi1) - j0;
        if (n_kv <= 0) continue;
        for (int t = 0; t < n_kv + 2 && ok; ++t, ++ns) {  // K_t and V_{t-2}
          const int s = ns % ST;
          const bool k = t < n_kv, v = t >= 2;
          ok = mbar_wait(kv_empty(s), ((ns / ST) & 1) ^ 1, p.status);
          if (!ok) break;
          if (k || v)
            mbar_arrive_expect_tx(kv_full(s), (static_cast<int>(k) + static_cast<int>(v)) * C::KTILE);
          else
            mbar_arrive(kv_full(s));
          for (int sl = 0; sl < C::SLABS && k; ++sl)
            tma_load_4d(k_s(s) + sl * C::KSLAB, &tm_k, kv_full(s), sl * 64, hk, (j0 + t) * kHalf,
                        it.b);
          for (int sl = 0; sl < C::SLABS && v; ++sl)
            tma_load_4d(v_s(s) + sl * C::KSLAB, &tm_v, kv_full(s), sl * 64, hk,
                        (j0 + t - 2) * kHalf, it.b);
          if (t > 0) continue;
          // The first key tile needs no room of the last item's query tiles.
          ok = mbar_wait(q_empty, (nq & 1) ^ 1, p.status);
          if (!ok) break;
          const int tiles = it.t0 + 1 < sh.tiles128 ? 2 : 1;
          mbar_arrive_expect_tx(q_full, tiles * C::SLABS * rows * 128);
          for (int w = 0; w < tiles; ++w)
            for (int sl = 0; sl < C::SLABS; ++sl)
              tma_load_4d(q_s(w) + sl * C::QSLAB, &tm_q, q_full, sl * 64, it.h,
                          (it.t0 + w) * sh.pos128, it.b);
          ++nq;
        }
      }
      // Never leave a copy in flight.
      if (nq > 0) mbar_wait(q_full, (nq - 1) & 1, p.status);
      for (int j = ns - ST < 0 ? 0 : ns - ST; j < ns; ++j)
        mbar_wait(kv_full(j % ST), (j / ST) & 1, p.status);
    } else if (warp >= 1 && warp <= 2 && elect_one_sync()) {
      // ------------------------------------- MMA of query tile w, a thread each
      constexpr uint32_t idesc_s = make_idesc_bf16(kTile, kHalf, false, false);
      constexpr uint32_t idesc_o = make_idesc_bf16(kTile, D, false, true);
      const int w = warp - 1;
      Ring kv{0, 0};            // the next stage
      int qc = 0;               // query tiles used
      int scores = 0;           // products Q K^T issued
      int steps = 0;            // products P V issued
      int outs = 0;             // O_w begun
      bool ok = true;
      auto issue_s = [&] {  // S_w = Q_w K^T
        const uint32_t d = tmem + C::S_COL + w * kTile + (scores & 1) * kHalf;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_bf16(d, make_sdesc(q_s(w) + (kk >> 2) * C::QSLAB + (kk & 3) * 32, 16, 1024, kSw128),
                    make_sdesc(k_s(kv.stage) + (kk >> 2) * C::KSLAB + (kk & 3) * 32, 16, 1024,
                               kSw128),
                    idesc_s, kk > 0);
        umma_commit(s_full(w, scores));
        ++scores;
      };
      auto issue_pv = [&](bool begin) {  // O_w += P_w V
        const uint32_t a = tmem + C::S_COL + w * kTile + (steps & 1) * kHalf;
#pragma unroll
        for (int kk = 0; kk < kHalf / 16; ++kk)
          umma_bf16_ts(tmem + C::O_COL + w * D, a + kk * 8,
                       make_sdesc(v_s(kv.stage) + kk * 2048, C::KSLAB, 1024, kSw128), idesc_o,
                       (!begin || kk > 0) ? 1u : 0u);
        umma_commit(o_done(w, steps));
        ++steps;
      };
      for (int i = 0; ok; ++i) {
        const FwdItem it = wait_item(i, ok);
        if (it.b < 0) break;
        const int j0 = it.hi0 == 0 ? it.lo1 : it.hi1 == 0 ? it.lo0 : min(it.lo0, it.lo1);
        const int n_kv = max(it.hi0, it.hi1) - j0;
        if (n_kv <= 0) {
          mbar_arrive(item_empty(i & 1));
          continue;
        }
        // Key tile t is j0 + t; query tile w takes part in t of [from, to).  A
        // tile is given back by both threads, by the one that leaves it out too
        // (once it is there: an arrival never runs ahead of its phase).
        const int from = (w == 0 ? it.lo0 : it.lo1) - j0, to = (w == 0 ? it.hi0 : it.hi1) - j0;
        ok = mbar_wait(q_full, qc & 1, p.status);
        if (!ok) break;
        ++qc;
        if (to <= from) mbar_arrive(q_empty);
        for (int t = 0; t < n_kv + 2; ++t) {  // S_w(t) and O_w's product t - 2
          // Four key tiles before the end it is time to look for the next item.
          if (t == max(n_kv - 2, 2)) mbar_arrive(item_empty(i & 1));
          ok = mbar_wait(kv_full(kv.stage), kv.phase, p.status);
          if (!ok) break;
          if (t - 2 >= from && t - 2 < to) {
            ok = mbar_wait(p_ready(w, steps), (steps >> 1) & 1, p.status);
            // O_w's last item has been read before it is begun again.
            if (ok && t - 2 == from && outs > 0)
              ok = mbar_wait(o_free(w), (outs - 1) & 1, p.status);
            if (!ok) break;
            tc_fence_after();
            issue_pv(t - 2 == from);
            outs += t - 2 == from;
          }
          if (t >= from && t < to) {
            // S_w goes over P_w of two tiles ago: its product is done.
            if (scores >= 2)
              ok = mbar_wait(o_done(w, scores), ((scores - 2) >> 1) & 1, p.status);
            if (!ok) break;
            tc_fence_after();
            issue_s();
            if (t + 1 == to) umma_commit(q_empty);
          }
          umma_commit(kv_empty(kv.stage));
          kv.next(ST);
        }
      }
      // Nothing may outlive the CTA's TMEM: wait for the tile's last product.
      if (steps > 0) mbar_wait(o_done(w, steps - 1), ((steps - 1) >> 1) & 1, p.status);
    } else if (warp == 3) {
      // ------------------------------------------------------ scheduler
      const int groups = sh.heads / sh.pack;
      const int bh_count = sh.batch * groups;
      for (int i = 0;; ++i) {
        // Not before the item before it nears its end.
        if (i > 0 && !mbar_wait(item_empty((i - 1) & 1), ((i - 1) >> 1) & 1, p.status)) break;
        const int n = i == 0 ? static_cast<int>(blockIdx.x)
                             : take_cta(base + C::TAKE_OFF, taken, i - 1, p.status);
        FwdItem it{-1, 0, 0, 0, 0, 0, 0, 0};
        if (n >= 0) {
          // Late positions (the heaviest, causally) first.
          const int bh = n % bh_count;
          it.b = bh / groups;
          it.h = bh % groups * sh.pack;
          it.t0 = 2 * (p.n_pairs - 1 - n / bh_count);
          const int i0 = it.t0 * sh.pos128;
          const Span a = span_of_positions(p.first, p.last, it.b, i0, sh.pos128, sh.seq);
          const Span c =
              span_of_positions(p.first, p.last, it.b, i0 + sh.pos128, sh.pos128, sh.seq);
          it.lo0 = a.lo / kHalf;
          it.hi0 = (a.hi + kHalf - 1) / kHalf;
          it.lo1 = c.lo / kHalf;
          it.hi1 = (c.hi + kHalf - 1) / kHalf;
        }
        if (lane == 0) {
          items[i & 1] = it;
          mbar_arrive(item_full(i & 1));
        }
        __syncwarp();
        if (it.b < 0) break;
      }
    }
  } else {
    // --------------------------------------------------------- softmax
    const int w = (warp - 4) >> 2;  // query tile of this warpgroup
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const bool filled = row < rows;
    const int at = row / sh.pack, head = row % sh.pack;  // position and head within the tile
    const uint32_t lrow = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t ocol = lrow + C::O_COL + w * D;
    const float c = sh.scale_log2;
    const F2 cc2 = f2(c, c);
    uint8_t* const out_s = gbase + C::OUT_OFF + (warp - 4) * kStageBytes;
    bool ok = true;
    int steps = 0;  // key tiles of query tile w, of all items
    FwdItem it = wait_item(0, ok);
    __syncwarp();
    if (lane == 0) mbar_arrive(item_empty(0));
    auto span_of_row = [&](const FwdItem& item) {
      return filled && item.b >= 0
                 ? load_span(p.first, p.last, item.b, (item.t0 + w) * sh.pos128 + at, sh.seq)
                 : Span{0, 0};
    };
    Span sp = span_of_row(it);
    for (int i = 0; ok && it.b >= 0; ++i) {
      const int jw = w == 0 ? it.lo0 : it.lo1;
      const int nk = (w == 0 ? it.hi0 : it.hi1) - jw;
      const int qpos = (it.t0 + w) * sh.pos128 + at;
      // What any row of the warp sees, and what every filled row sees.
      const int any_lo = __reduce_min_sync(0xffffffffu, sp.lo < sp.hi ? sp.lo : INT_MAX);
      const int any_hi = __reduce_max_sync(0xffffffffu, sp.hi);
      const int all_lo = __reduce_max_sync(0xffffffffu, filled ? sp.lo : 0);
      const int all_hi = __reduce_min_sync(0xffffffffu, filled ? sp.hi : INT_MAX);
      float m = sp.lo < sp.hi ? -INFINITY : 0.0f;  // -inf: has seen nothing yet
      float l = 0.0f;
      bool begun = __all_sync(0xffffffffu, m != -INFINITY);
      for (int j = 0; j < nk; ++j, ++steps) {
        ok = mbar_wait(s_full(w, steps), (steps >> 1) & 1, p.status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t scol = lrow + C::S_COL + w * kTile + (steps & 1) * kHalf;
        const int kv0 = (jw + j) * kHalf;
        auto none = [&](int c2) {
          return kv0 + 32 * c2 + 32 <= any_lo || kv0 + 32 * c2 >= any_hi;
        };
        auto full = [&](int c2) {
          return kv0 + 32 * c2 >= all_lo && kv0 + 32 * c2 + 32 <= all_hi;
        };
        // Scores that the row does not see become -inf.
        auto mask = [&](int c2, uint32_t(&r)[32]) {
          const int k0 = kv0 + 32 * c2;
          const uint32_t seen =
              bit_range(min(max(sp.lo - k0, 0), 32), min(max(sp.hi - k0, 0), 32));
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(seen >> e & 1)) r[e] = 0xFF800000u;
        };
        // The largest score of the tile that the row sees.
        auto tile_max = [&] {
          float top = -INFINITY;
#pragma unroll 1
          for (int c2 = 0; c2 < 2; ++c2) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(scol + c2 * 32, r);
            tmem_ld_wait(r);
            if (!full(c2)) mask(c2, r);
            float t[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; ++e) t[e & 3] = fmaxf(t[e & 3], __uint_as_float(r[e]));
            top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
          }
          return top * c;
        };
        if (!begun) {
          const float top = tile_max();
          if (m == -INFINITY) m = top;
          begun = __all_sync(0xffffffffu, m != -INFINITY);
        }
        const float mref = m == -INFINITY ? 0.0f : m;
        uint32_t pk[32];
        F2 sum2 = f2(0.0f, 0.0f);
        uint32_t rb[2][32];
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2)
          if (!none(c2)) tmem_ld_32x32b_x32(scol + c2 * 32, rb[c2]);
        tmem_ld_wait(rb[0], rb[1]);
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          if (none(c2)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[c2 * 16 + e] = 0;
          } else {
            if (!full(c2)) mask(c2, rb[c2]);
            sum2 = sum2 + exp_chunk(rb[c2], cc2, mref, pk + c2 * 16);
          }
        }
        float2 sum = split(sum2);
        if (!__any_sync(0xffffffffu, !(sum.x + sum.y <= kMost))) {
          tmem_st_32x32b_x32(scol, pk);
        } else {
          // Some row has outgrown its reference (or holds a NaN, and keeps it).
          // The scores are still there: those rows take the tile's maximum for a
          // new one, the others go through with a factor of 1.  It is applied as
          // the square of its root: itself it may be below 2^-126, which is 0
          // here, where l and O are as much as 2^60 above their first terms.
          const float top = tile_max();
          const bool grow = top > m + kGrowLog2;
          const float f = grow ? ex2_approx(0.5f * (m - top)) : 1.0f;
          if (grow) m = top;
          l = l * f * f;
          if (j > 0) {  // O_w, once its last product is done
            ok = mbar_wait(o_done(w, steps - 1), ((steps - 1) >> 1) & 1, p.status);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int cc = 0; cc < D / 16; ++cc) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(ocol + cc * 16, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f * f);
              tmem_st_32x32b_x16(ocol + cc * 16, o);
            }
          }
          sum2 = f2(0.0f, 0.0f);
#pragma unroll 1
          for (int c2 = 0; c2 < 2; ++c2) {
            uint32_t r[32], pc[16];
            tmem_ld_32x32b_x32(scol + c2 * 32, r);
            tmem_ld_wait(r);
            mask(c2, r);
            sum2 = sum2 + exp_chunk(r, cc2, m == -INFINITY ? 0.0f : m, pc);
            tmem_st_32x32b_x16(scol + c2 * 16, pc);
          }
          sum = split(sum2);
        }
        l += sum.x + sum.y;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(w, steps));
      }
      if (!ok) break;
      // The next item's description and span, read while this one ends.
      const FwdItem nx = wait_item(i + 1, ok);
      __syncwarp();
      if (lane == 0) mbar_arrive(item_empty((i + 1) & 1));
      const Span nsp = span_of_row(nx);
      const bool valid = filled && qpos < sh.seq;
      uint16_t* orow =
          p.out + ((static_cast<size_t>(it.b) * sh.seq + qpos) * sh.heads + it.h + head) * D;
      float* const lse =
          p.lse + (static_cast<size_t>(it.b) * sh.heads + it.h + head) * sh.seq + qpos;
      if (nk > 0) {
        ok = ok && mbar_wait(o_done(w, steps - 1), ((steps - 1) >> 1) & 1, p.status);
        if (!ok) break;
        tc_fence_after();
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // 0: sees nothing
        const F2 inv2 = f2(inv, inv);
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 64) {
          uint32_t o[2][32], wd[32];
          tmem_ld_32x32b_x32(ocol + c0, o[0]);
          tmem_ld_32x32b_x32(ocol + c0 + 32, o[1]);
          tmem_ld_wait(o[0], o[1]);
          if (c0 + 64 == D) {  // O_w may be begun again
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free(w));
          }
#pragma unroll
          for (int e = 0; e < 32; ++e)
            wd[e] = pack_bf16(pair_of(o[e / 16][2 * e % 32], o[e / 16][2 * e % 32 + 1]) * inv2);
          store_rows(out_s, wd, orow + c0, valid);
        }
        if (valid) *lse = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
      } else {  // no row of the tile sees anything
        const uint32_t zero[32] = {};
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 64) store_rows(out_s, zero, orow + c0, valid);
        if (valid) *lse = -INFINITY;
      }
      it = nx;
      sp = nsp;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// ----------------------------------------------------------------- backward --
//
// Three launches, no atomics on results (the gradients are deterministic):
//   prep   per packed query row -lse log2(e) and -delta (f32), in 64-row packed
//          tiles (rows that hold nothing: -inf and 0, so their probabilities
//          are 0), each row's span in the same order, and each tile's spans;
//   dq     a tile of work is a packed 128-row query tile, key tiles of 64:
//            S = Q K_j^T, dP = dO V_j^T (tensor memory, double-buffered),
//            dS = P * (dP - delta), P = exp2(S c - lse2)  (compute warps),
//            dQ += dS K_j  (dS written over S, A from tensor memory).
//          Q and dO lie in tensor memory too (read from shared memory for every
//          key tile: 94 us where it then took 85);
//   dkv    a tile of work is a 128-key tile of one key/value head, with the
//          packed 64-row query tiles that see it:
//            S^T = K Q_i^T, dP^T = V dO_i^T, P^T and dS^T (compute warps, back
//            into tensor memory), dV += P^T dO_i, dK += dS^T Q_i.
//          Its products take 1310 cycles a tile and shared memory, which feeds
//          them 128 KB and takes in 32 KB of copies, 1280 of its 128 bytes a
//          cycle; with P^T and dS^T as operands there too it was 127 us where
//          it then took 103.
// Scores go over operands of two tiles ago once their product is done (without
// that wait dq took 81 us and dk/dv 103).  At four packed rows of 2048 (as
// above): 24, 84 and 108 us.  Which CTA does a tile changes no result.

// The workspace: statistics [batch, heads / pack, tiles64, 64], spans (first
// key, how many) [batch, tiles64, 64], tiles: what any row of a 64-row packed
// query tile sees [batch, tiles64].
struct BwdWork {
  float* nlse2;
  float* ndelta;
  int2* rows;
  Span* tiles;
  size_t bytes;
};

struct PrepParams {
  SpanShape sh;
  const uint16_t* out;
  const uint16_t* dout;
  const float* lse;
  const int* first;
  const int* last;
  BwdWork work;
  unsigned row_blocks;  // blocks from here on do the spans, a warp a tile
};

__device__ __forceinline__ void load_16(const uint16_t* p, bool wide, uint32_t (&w)[8]) {
  if (wide) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                   "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
  }
}

// A CTA a 64-row tile: two rows a thread, 16 elements of each.  Bound by
// reading out and dout (packed rows of 2048: 134 MB in 24 us).  delta is summed
// in f32 of the stored output, which is rounded to bf16 (delta is off by 2^-8 of
// sum |dO O| at most, the order of dS's own rounding): an f32 copy of O would cost
// the forward twice the bytes of its result and this kernel as many again.
template <int D>
__global__ void __launch_bounds__(2 * D) span_prep_kernel(const PrepParams p) {
  constexpr int LANES = D / 16;
  griddep_wait();
  griddep_launch_dependents();
  const SpanShape& sh = p.sh;
  const int filled_rows = sh.pack * sh.pos64;
  if (blockIdx.x >= p.row_blocks) {
    const int t = (blockIdx.x - p.row_blocks) * (2 * D / 32) + (threadIdx.x >> 5);
    if (t >= sh.batch * sh.tiles64) return;
    const int b = t / sh.tiles64;
    const int i0 = t % sh.tiles64 * sh.pos64;
    Span s{sh.seq, 0};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = e * 32 + (threadIdx.x & 31);
      const bool filled = r < filled_rows;
      const Span sp =
          filled ? load_span(p.first, p.last, b, i0 + r / sh.pack, sh.seq) : Span{0, 0};
      // A row that holds nothing (P = 0 by its statistics) must not make the
      // tile a masked one.
      p.work.rows[static_cast<size_t>(t) * kHalf + r] =
          filled ? make_int2(sp.lo, sp.hi - sp.lo) : make_int2(0, sh.seq);
      if (!filled) continue;
      if (sp.lo < sp.hi) s.lo = min(s.lo, sp.lo);
      s.hi = max(s.hi, sp.hi);
    }
    s.lo = __reduce_min_sync(0xffffffffu, s.lo);
    s.hi = __reduce_max_sync(0xffffffffu, s.hi);
    if ((threadIdx.x & 31) == 0) p.work.tiles[t] = s;
    return;
  }
  const int t = blockIdx.x;
  const int groups = sh.heads / sh.pack;
  const int bg = t / sh.tiles64;
  const int b = bg / groups, h0 = bg % groups * sh.pack;
  const int i0 = t % sh.tiles64 * sh.pos64;
  const int sub = threadIdx.x % LANES;
  const bool wide = wide_rows(p.out) && wide_rows(p.dout);
  uint32_t o[2][8], d[2][8];
  float l[2];
  bool real[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = e * 32 + threadIdx.x / LANES;
    const int i = i0 + r / sh.pack, h = h0 + r % sh.pack;
    real[e] = r < filled_rows && i < sh.seq;
    if (!real[e]) continue;
    const size_t off = ((static_cast<size_t>(b) * sh.seq + i) * sh.heads + h) * D + sub * 16;
    load_16(p.out + off, wide, o[e]);
    load_16(p.dout + off, wide, d[e]);
    if (sub == 0) l[e] = p.lse[(static_cast<size_t>(b) * sh.heads + h) * sh.seq + i];
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float acc = 0.0f;
    if (real[e]) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        acc = fmaf(__uint_as_float(o[e][k] << 16), __uint_as_float(d[e][k] << 16), acc);
        acc = fmaf(__uint_as_float(o[e][k] & 0xFFFF0000u),
                   __uint_as_float(d[e][k] & 0xFFFF0000u), acc);
      }
    }
#pragma unroll
    for (int off = 1; off < LANES; off <<= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    if (sub == 0) {
      const size_t row = static_cast<size_t>(t) * kHalf + e * 32 + threadIdx.x / LANES;
      p.work.nlse2[row] = real[e] && l[e] != -INFINITY ? -l[e] * kLog2e : -INFINITY;
      p.work.ndelta[row] = real[e] ? -acc : 0.0f;
    }
  }
}

struct BwdParams {
  SpanShape sh;
  const int* first;  // [batch, seq]
  const int* last;
  BwdWork work;
  float scale;
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  int* status;
};

struct DqItem {
  int b, h, q0;       // b < 0: no more; first of `pack` heads, first position
  int kv0, n_kv;      // 64-key tiles
  int pad[3];
};

template <int D>
struct DqCfg {
  static constexpr int SLABS = D / 64;
  static constexpr int QSLAB = kTile * 128;  // 128 rows x 64 bf16
  static constexpr int QTILE = SLABS * QSLAB;
  static constexpr int KSLAB = kHalf * 128;  // 64 rows x 64 bf16
  static constexpr int KTILE = SLABS * KSLAB;
  static constexpr int KST = D == 128 ? 4 : 8;
  static constexpr int VST = KST;  // (one stage index for both)
  static constexpr int Q_OFF = 0;
  static constexpr int DO_OFF = QTILE;
  static constexpr int K_OFF = 2 * QTILE;
  static constexpr int V_OFF = K_OFF + KST * KTILE;
  static constexpr int OUT_OFF = V_OFF + VST * KTILE;
  static constexpr int ITEM_OFF = OUT_OFF + kBwdWarps * kStageBytes;
  static constexpr int TAKE_OFF = ITEM_OFF + 2 * static_cast<int>(sizeof(DqItem));
  static constexpr int BAR_OFF = TAKE_OFF + 16;
  // q_full, q_empty, k_full[KST], k_empty[KST], v_full[VST], v_empty[VST], s_full[2],
  // ds_ready[2], a_ready, dq_full, dq_free, item_full[2], item_empty[2], taken; TMEM slot
  static constexpr int NBAR = 2 + 2 * KST + 2 * VST + 12;
  static constexpr int SMEM_USED = 1024 + BAR_OFF + 8 * (NBAR + 1);
  // At least ~116 KB, so that one CTA (and its 512 TMEM columns) fits an SM.
  static constexpr int SMEM = SMEM_USED > 118784 ? SMEM_USED : 118784;
  // S_b at 64 b, dS_b (bf16 pairs) over it, each half of the keys in the first
  // 16 of its 32 columns, so that a warp writes only over what it has read.
  static constexpr int S_COL = 0;
  static constexpr int DP_COL = 128;  // dP_b at 128 + 64 b
  static constexpr int DQ_COL = 256;
  static constexpr int Q_COL = 256 + D;  // Q, then dO (bf16 pairs)
  static constexpr int DO_COL = Q_COL + D / 2;
  static constexpr int TMEM_COLS = 512;
  static_assert(DO_COL + D / 2 <= TMEM_COLS, "tensor memory map");
  static_assert(SMEM <= 232448, "shared memory per CTA");
};

template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
    span_dq_kernel(const __grid_constant__ CUtensorMap tm_q,
                   const __grid_constant__ CUtensorMap tm_do,
                   const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const BwdParams p) {
  using C = DqCfg<D>;
  constexpr int KST = C::KST;
  constexpr int VST = C::VST;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const gbase = smem_raw + (base - raw);
  const uint32_t q_s = base + C::Q_OFF;
  const uint32_t do_s = base + C::DO_OFF;
  auto k_s = [&](int s) { return base + C::K_OFF + s * C::KTILE; };
  auto v_s = [&](int s) { return base + C::V_OFF + s * C::KTILE; };
  const uint32_t bars = base + C::BAR_OFF;
  const uint32_t q_full = bars, q_empty = bars + 8u;
  auto k_full = [&](int s) { return bars + 8u * (2 + s); };
  auto k_empty = [&](int s) { return bars + 8u * (2 + KST + s); };
  auto v_full = [&](int s) { return bars + 8u * (2 + 2 * KST + s); };
  auto v_empty = [&](int s) { return bars + 8u * (2 + 2 * KST + VST + s); };
  constexpr int X = 2 + 2 * KST + 2 * VST;
  auto s_full = [&](int b) { return bars + 8u * (X + b); };
  auto ds_ready = [&](int b) { return bars + 8u * (X + 2 + b); };
  const uint32_t a_ready = bars + 8u * (X + 4);
  const uint32_t dq_full = bars + 8u * (X + 5), dq_free = bars + 8u * (X + 6);
  auto item_full = [&](int i) { return bars + 8u * (X + 7 + i); };
  auto item_empty = [&](int i) { return bars + 8u * (X + 9 + i); };
  const uint32_t taken = bars + 8u * (X + 11);
  const uint32_t tmem_slot = bars + 8u * C::NBAR;
  volatile uint32_t* tmem_slot_ptr =
      reinterpret_cast<volatile uint32_t*>(gbase + (tmem_slot - base));
  DqItem* const items = reinterpret_cast<DqItem*>(gbase + C::ITEM_OFF);

  const SpanShape& sh = p.sh;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rows = sh.pack * sh.pos128;  // filled rows of the query tile
  const int groups = sh.heads / sh.pack;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, kBwdWarps);
    for (int s = 0; s < KST; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full(i), 2);
      mbar_init(ds_ready(i), kBwdWarps);
      mbar_init(item_full(i), 1);
      mbar_init(item_empty(i), kBwdReaders);
    }
    mbar_init(a_ready, kBwdWarps);
    mbar_init(dq_full, 1);
    mbar_init(dq_free, kBwdWarps);
    mbar_init(taken, 1);
    fence_mbar_init();
  }
  zero_rows(gbase + C::Q_OFF, 2 * C::SLABS, kTile, rows);  // Q and dO
  if (warp == 2) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot_ptr;
  griddep_launch_dependents();  // this CTA holds its tensor memory
  griddep_wait();

  auto wait_item = [&](int i, bool& ok) {
    DqItem it{-1, 0, 0, 0, 0, {0, 0, 0}};
    ok = mbar_wait(item_full(i & 1), (i >> 1) & 1, p.status);
    if (ok) it = items[i & 1];
    return it;
  };

  if (warp == 0) {
    // ------------------------------------------------------------- TMA
    if (elect_one_sync()) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_do);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      int nk = 0, nv = 0, nq = 0;  // tiles issued, of all items
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const DqItem it = wait_item(i, ok);
        if (it.b < 0) break;
        mbar_arrive(item_empty(i & 1));
        const int hk = it.h / sh.group;
        for (int j = 0; j < it.n_kv && ok; ++j) {
          const int ks = nk % KST, vs = nv % VST;
          ok = mbar_wait(k_empty(ks), ((nk / KST) & 1) ^ 1, p.status);
          if (!ok) break;
          mbar_arrive_expect_tx(k_full(ks), C::KTILE);
          for (int sl = 0; sl < C::SLABS; ++sl)
            tma_load_4d(k_s(ks) + sl * C::KSLAB, &tm_k, k_full(ks), sl * 64, hk,
                        (it.kv0 + j) * kHalf, it.b);
          ++nk;
          if (j == 0) {
            ok = mbar_wait(q_empty, (nq & 1) ^ 1, p.status);
            if (!ok) break;
            mbar_arrive_expect_tx(q_full, 2 * C::SLABS * rows * 128);
            for (int sl = 0; sl < C::SLABS; ++sl) {
              tma_load_4d(q_s + sl * C::QSLAB, &tm_q, q_full, sl * 64, it.h, it.q0, it.b);
              tma_load_4d(do_s + sl * C::QSLAB, &tm_do, q_full, sl * 64, it.h, it.q0, it.b);
            }
            ++nq;
          }
          ok = mbar_wait(v_empty(vs), ((nv / VST) & 1) ^ 1, p.status);
          if (!ok) break;
          mbar_arrive_expect_tx(v_full(vs), C::KTILE);
          for (int sl = 0; sl < C::SLABS; ++sl)
            tma_load_4d(v_s(vs) + sl * C::KSLAB, &tm_v, v_full(vs), sl * 64, hk,
                        (it.kv0 + j) * kHalf, it.b);
          ++nv;
        }
      }
      // Never leave a copy in flight.
      if (nq > 0) mbar_wait(q_full, (nq - 1) & 1, p.status);
      for (int j = nk - KST < 0 ? 0 : nk - KST; j < nk; ++j)
        mbar_wait(k_full(j % KST), (j / KST) & 1, p.status);
      for (int j = nv - VST < 0 ? 0 : nv - VST; j < nv; ++j)
        mbar_wait(v_full(j % VST), (j / VST) & 1, p.status);
    }
  } else if (warp <= 2) {
    // ------------------------------------- MMA: S and dQ (warp 1), dP (warp 2)
    if (elect_one_sync()) {
      constexpr uint32_t idesc_s = make_idesc_bf16(kTile, kHalf, false, false);
      constexpr uint32_t idesc_dq = make_idesc_bf16(kTile, D, false, true);
      const bool first = warp == 1;
      int g = 0;   // key tiles, of all items: buffer g & 1, stage g % KST
      int n = 0;   // items with any
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const DqItem it = wait_item(i, ok);
        if (it.b < 0) break;
        if (it.n_kv == 0) {
          mbar_arrive(item_empty(i & 1));
          continue;
        }
        // dQ += dS K: A = dS from tensor memory, B = K MN-major (N = dim).
        auto issue_dq = [&](int t, bool begin) -> bool {
          if (!mbar_wait(ds_ready(t & 1), (t >> 1) & 1, p.status)) return false;
          // The last item's dQ has been read before it is begun again.
          if (begin && n > 0 && !mbar_wait(dq_free, (n - 1) & 1, p.status)) return false;
          tc_fence_after();
          const int ks = t % KST;
#pragma unroll
          for (int kk = 0; kk < kHalf / 16; ++kk)
            umma_bf16_ts(tmem + C::DQ_COL,
                         tmem + C::S_COL + (t & 1) * kHalf + (kk >> 1) * 32 + (kk & 1) * 8,
                         make_sdesc(k_s(ks) + kk * 2048, C::KSLAB, 1024, kSw128), idesc_dq,
                         (!begin || kk > 0) ? 1u : 0u);
          umma_commit(k_empty(ks));
          return true;
        };
        ok = mbar_wait(a_ready, n & 1, p.status);
        for (int j = 0; j < it.n_kv && ok; ++j, ++g) {
          const int s = g % KST;
          // Four key tiles before the end it is time to look for the next item.
          if (j == max(it.n_kv - 4, 0)) mbar_arrive(item_empty(i & 1));
          // S_g goes over dS of two tiles ago, whose product is done when it
          // gives its keys back; dP_g over that tile's dP, read before its dS
          // was ready.
          ok = first ? mbar_wait(k_full(s), (g / KST) & 1, p.status) &&
                           (g < 2 || mbar_wait(k_empty((g - 2) % KST), ((g - 2) / KST) & 1, p.status))
                     : mbar_wait(v_full(s), (g / VST) & 1, p.status) &&
                           (g < 2 || mbar_wait(ds_ready(g & 1), ((g - 2) >> 1) & 1, p.status));
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + (first ? C::S_COL : C::DP_COL) + (g & 1) * kHalf;
          const uint32_t a = tmem + (first ? C::Q_COL : C::DO_COL);
          const uint32_t b = first ? k_s(s) : v_s(s);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16_ts(d, a + kk * 8,
                         make_sdesc(b + (kk >> 2) * C::KSLAB + (kk & 3) * 32, 16, 1024, kSw128),
                         idesc_s, kk > 0);
          umma_commit(s_full(g & 1));
          if (!first) umma_commit(v_empty(s));
          if (first && j >= 1) ok = issue_dq(g - 1, j == 1);
        }
        if (!ok) break;
        if (first) {
          ok = issue_dq(g - 1, it.n_kv == 1);
          umma_commit(dq_full);
        }
        ++n;
      }
      // Nothing may outlive the CTA's TMEM: the last commit covers every MMA.
      if (n > 0 && first) mbar_wait(dq_full, (n - 1) & 1, p.status);
      if (n > 0 && !first) mbar_wait(s_full((g - 1) & 1), ((g - 1) >> 1) & 1, p.status);
    }
  } else if (warp == 3) {
    // -------------------------------------------------------- scheduler
    const int bh_count = sh.batch * groups;
    for (int i = 0;; ++i) {
      // Not before the item before it nears its end.
      if (i > 0 && !mbar_wait(item_empty((i - 1) & 1), ((i - 1) >> 1) & 1, p.status)) break;
      const int n = i == 0 ? static_cast<int>(blockIdx.x)
                           : take_cta(base + C::TAKE_OFF, taken, i - 1, p.status);
      DqItem it{-1, 0, 0, 0, 0, {0, 0, 0}};
      if (n >= 0) {
        const int bh = n % bh_count;
        it.b = bh / groups;
        it.h = bh % groups * sh.pack;
        it.q0 = (sh.tiles128 - 1 - n / bh_count) * sh.pos128;
        const Span s = span_of_positions(p.first, p.last, it.b, it.q0, sh.pos128, sh.seq);
        it.kv0 = s.lo / kHalf;
        it.n_kv = (s.hi + kHalf - 1) / kHalf - it.kv0;
      }
      if (lane == 0) {
        items[i & 1] = it;
        mbar_arrive(item_full(i & 1));
      }
      __syncwarp();
      if (it.b < 0) break;
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------ compute warps
    // The warpgroups share the 128 rows and split each tile's 64 key columns
    // (the gradient is elementwise given the row's lse and delta), and dQ's
    // columns at the end.  Two of them: four (96 registers a thread) were no
    // faster.
    const int part = (warp - 4) >> 2;
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const bool filled = row < rows;
    const int at = row / sh.pack, head = row % sh.pack;  // position and head within the tile
    const uint32_t lrow = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c = sh.scale_log2;
    const F2 c2 = f2(c, c), scale2 = f2(p.scale, p.scale);
    uint8_t* const out_s = gbase + C::OUT_OFF + (warp - 4) * kStageBytes;
    bool ok = true;
    int g = 0, n = 0, nq = 0;
    struct RowState {
      float nlse2, ndelta;
      Span sp;
    };
    auto row_state = [&](const DqItem& it) {
      RowState s{-INFINITY, 0.0f, {0, 0}};
      const int qpos = it.q0 + at;
      if (it.b >= 0 && filled && qpos < sh.seq) {
        const size_t srow =
            (static_cast<size_t>(it.b * groups + it.h / sh.pack) * sh.tiles64 + qpos / sh.pos64) *
                kHalf +
            qpos % sh.pos64 * sh.pack + head;
        s.nlse2 = p.work.nlse2[srow];
        s.ndelta = p.work.ndelta[srow];
        s.sp = load_span(p.first, p.last, it.b, qpos, sh.seq);
      }
      return s;
    };
    // The item's Q (warpgroup 0) and dO (1) from shared to tensor memory, a row a
    // thread, once the products of the item before have read theirs there (the
    // last tile's scores are complete).
    auto stage = [&](const DqItem& item) {
      if (item.b < 0 || item.n_kv == 0) return;
      ok = ok && mbar_wait(q_full, nq & 1, p.status);
      if (!ok) return;
      ++nq;
      const uint8_t* src = gbase + (part == 0 ? C::Q_OFF : C::DO_OFF) + row * 128;
      const uint32_t dst = lrow + (part == 0 ? C::Q_COL : C::DO_COL);
#pragma unroll
      for (int sl = 0; sl < C::SLABS; ++sl) {
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint4 x =
              *reinterpret_cast<const uint4*>(src + sl * C::QSLAB + ((e ^ (row & 7)) << 4));
          w[4 * e] = x.x;
          w[4 * e + 1] = x.y;
          w[4 * e + 2] = x.z;
          w[4 * e + 3] = x.w;
        }
        tmem_st_32x32b_x32(dst + sl * 32, w);
      }
      tmem_st_wait();
      tc_fence_before();
      fence_proxy_async_smem();  // the reads above come before the next copies
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(q_empty);
        mbar_arrive(a_ready);
      }
    };
    DqItem it = wait_item(0, ok);
    __syncwarp();
    if (lane == 0) mbar_arrive(item_empty(0));
    stage(it);
    RowState st = row_state(it);
    for (int i = 0; ok && it.b >= 0; ++i) {
      const Span sp = st.sp;
      const unsigned len = sp.hi - sp.lo;
      const int any_lo = __reduce_min_sync(0xffffffffu, sp.lo < sp.hi ? sp.lo : INT_MAX);
      const int any_hi = __reduce_max_sync(0xffffffffu, sp.hi);
      const int all_lo = __reduce_max_sync(0xffffffffu, filled ? sp.lo : 0);
      const int all_hi = __reduce_min_sync(0xffffffffu, filled ? sp.hi : INT_MAX);
      const F2 shift = f2(st.nlse2, st.nlse2), nd = f2(st.ndelta, st.ndelta);
      for (int j = 0; j < it.n_kv; ++j, ++g) {
        ok = mbar_wait(s_full(g & 1), (g >> 1) & 1, p.status);
        if (!ok) break;
        tc_fence_after();
        const int k0 = (it.kv0 + j) * kHalf + part * kPartCols;
        const bool none = k0 + kPartCols <= any_lo || k0 >= any_hi;
        uint32_t sv[kPartCols], dv[kPartCols];
        if (!none) {
          tmem_ld_32x32b_x32(lrow + C::S_COL + (g & 1) * kHalf + part * kPartCols, sv);
          tmem_ld_32x32b_x32(lrow + C::DP_COL + (g & 1) * kHalf + part * kPartCols, dv);
          tmem_ld_wait(sv, dv);
        }
        uint32_t pk[kPartCols / 2];
        if (none) {
#pragma unroll
          for (int e = 0; e < kPartCols / 2; ++e) pk[e] = 0;
        } else {
          if (k0 < all_lo || k0 + kPartCols > all_hi) {
            const int col0 = k0 - sp.lo;
#pragma unroll
            for (int e = 0; e < kPartCols; ++e)
              if (static_cast<unsigned>(col0 + e) >= len) sv[e] = 0xFF800000u;  // P = 0
          }
#pragma unroll
          for (int e = 0; e < kPartCols / 2; ++e) {
            const F2 q = exp2_mufu(fma2(pair_of(sv[2 * e], sv[2 * e + 1]), c2, shift));
            pk[e] = pack_bf16(q * (pair_of(dv[2 * e], dv[2 * e + 1]) + nd));
          }
        }
        tmem_st_32x32b_x16(lrow + C::S_COL + (g & 1) * kHalf + part * kPartCols, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready(g & 1));
      }
      if (!ok) break;
      const DqItem nx = wait_item(i + 1, ok);
      __syncwarp();
      if (lane == 0) mbar_arrive(item_empty((i + 1) & 1));
      stage(nx);
      const RowState nst = row_state(nx);
      const int qpos = it.q0 + at;
      const bool valid = filled && qpos < sh.seq;
      uint16_t* orow =
          p.dq + ((static_cast<size_t>(it.b) * sh.seq + qpos) * sh.heads + it.h + head) * D;
      if (it.n_kv > 0) {
        ok = ok && mbar_wait(dq_full, n & 1, p.status);
        if (!ok) break;
        tc_fence_after();
        ++n;
      }
      constexpr int COLS = D / kParts;  // 64 or 32
      uint32_t wd[COLS / 2] = {};
      if (it.n_kv > 0) {
        uint32_t o[COLS / 32][32];
#pragma unroll
        for (int e = 0; e < COLS / 32; ++e)
          tmem_ld_32x32b_x32(lrow + C::DQ_COL + part * COLS + e * 32, o[e]);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < COLS / 32; ++e) keep_behind(o[e]);
        tc_fence_before();  // dQ may be begun again
        __syncwarp();
        if (lane == 0) mbar_arrive(dq_free);
#pragma unroll
        for (int e = 0; e < COLS / 2; ++e)
          wd[e] = pack_bf16(pair_of(o[e / 16][2 * e % 32], o[e / 16][2 * e % 32 + 1]) * scale2);
      }
      store_rows(out_s, wd, orow + part * COLS, valid);
      it = nx;
      st = nst;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

struct DkvItem {
  int b, hk, kv0;  // b < 0: no more; key/value head, first key
  int i0, nq;      // 64-row query tiles that see it
  int pad[3];
};

template <int D>
struct DkvCfg {
  static constexpr int SLABS = D / 64;
  static constexpr int KSLAB = kTile * 128;  // K_j, V_j: 128 rows x 64 bf16
  static constexpr int KTILE = SLABS * KSLAB;
  static constexpr int QSLAB = kHalf * 128;  // Q_i, dO_i: 64 rows x 64 bf16
  static constexpr int QTILE = SLABS * QSLAB;
  static constexpr int QST = D == 128 ? 4 : 8;
  static constexpr int STAT_BYTES = 2 * kHalf * 4;  // the statistics of one query tile
  static constexpr int K_OFF = 0;
  static constexpr int V_OFF = KTILE;
  static constexpr int Q_OFF = 2 * KTILE;
  static constexpr int DO_OFF = Q_OFF + QST * QTILE;
  static constexpr int STAT_OFF = DO_OFF + QST * QTILE;
  static constexpr int OUT_OFF = STAT_OFF + QST * STAT_BYTES;
  static constexpr int OUT_BYTES = kStageBytes / 2;  // 32 columns at a time: no room for more
  static constexpr int ITEM_OFF = OUT_OFF + kBwdWarps * OUT_BYTES;
  static constexpr int TAKE_OFF = ITEM_OFF + 2 * static_cast<int>(sizeof(DkvItem));
  static constexpr int BAR_OFF = TAKE_OFF + 16;
  // kv_full, kv_empty, q_full[QST], q_empty[QST], s_full[2], pds_ready[2], acc_full,
  // acc_free, item_full[2], item_empty[2], taken; then the TMEM slot
  static constexpr int NBAR = 2 + 2 * QST + 11;
  static constexpr int SMEM = 1024 + BAR_OFF + 8 * (NBAR + 1);
  // S^T_b at 64 b and dP^T_b at 128 + 64 b; P^T_b and dS^T_b (bf16 pairs) over
  // them, each 16 queries in the first 8 of those queries' 16 columns, so that
  // a warp writes only over what it has read.
  static constexpr int S_COL = 0;
  static constexpr int DP_COL = 128;
  static constexpr int DV_COL = 256;
  static constexpr int DK_COL = 256 + D;
  static constexpr int TMEM_COLS = 512;
  static_assert(DK_COL + D <= TMEM_COLS, "tensor memory map");
  static_assert(SMEM <= 232448, "shared memory per CTA");
  static_assert(SMEM > 118784, "one CTA per SM");
};

// Lane i holds row i of a 32 x 32 bit matrix (column j in bit j); returns its
// column i (row j in bit j): halves of halves change places, by the lane.
__device__ __forceinline__ uint32_t transpose_bits(uint32_t x) {
  const int lane = threadIdx.x & 31;
  uint32_t m = 0x0000FFFFu;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const uint32_t y = __shfl_xor_sync(0xffffffffu, x, j);
    x = lane & j ? (x & ~m) | ((y & ~m) >> j) : (x & m) | ((y & m) << j);
    m ^= m << (j >> 1);
  }
  return x;
}

template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
    span_dkv_kernel(const __grid_constant__ CUtensorMap tm_q,
                    const __grid_constant__ CUtensorMap tm_do,
                    const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const BwdParams p) {
  using C = DkvCfg<D>;
  constexpr int QST = C::QST;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const gbase = smem_raw + (base - raw);
  const uint32_t k_s = base + C::K_OFF;
  const uint32_t v_s = base + C::V_OFF;
  auto q_s = [&](int s) { return base + C::Q_OFF + s * C::QTILE; };
  auto do_s = [&](int s) { return base + C::DO_OFF + s * C::QTILE; };
  auto stat_s = [&](int s) { return base + C::STAT_OFF + s * C::STAT_BYTES; };
  const uint32_t bars = base + C::BAR_OFF;
  const uint32_t kv_full = bars, kv_empty = bars + 8u;
  auto q_full = [&](int s) { return bars + 8u * (2 + s); };
  auto q_empty = [&](int s) { return bars + 8u * (2 + QST + s); };
  constexpr int X = 2 + 2 * QST;
  auto s_full = [&](int b) { return bars + 8u * (X + b); };
  auto pds_ready = [&](int b) { return bars + 8u * (X + 2 + b); };
  const uint32_t acc_full = bars + 8u * (X + 4), acc_free = bars + 8u * (X + 5);
  auto item_full = [&](int i) { return bars + 8u * (X + 6 + i); };
  auto item_empty = [&](int i) { return bars + 8u * (X + 8 + i); };
  const uint32_t taken = bars + 8u * (X + 10);
  const uint32_t tmem_slot = bars + 8u * C::NBAR;
  volatile uint32_t* tmem_slot_ptr =
      reinterpret_cast<volatile uint32_t*>(gbase + (tmem_slot - base));
  DkvItem* const items = reinterpret_cast<DkvItem*>(gbase + C::ITEM_OFF);

  const SpanShape& sh = p.sh;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rows = sh.pack * sh.pos64;       // filled rows of a query tile
  const int subs = sh.group / sh.pack;       // packs that share the key/value head

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(kv_empty, 2);
    for (int s = 0; s < QST; ++s) {
      mbar_init(q_full(s), 1);
      mbar_init(q_empty(s), 2 + kBwdWarps);  // the MMAs' commits, the warps' stat reads
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full(i), 2);
      mbar_init(pds_ready(i), kBwdWarps);
      mbar_init(item_full(i), 1);
      mbar_init(item_empty(i), kBwdReaders);
    }
    mbar_init(acc_full, 2);
    mbar_init(acc_free, kBwdWarps);
    mbar_init(taken, 1);
    fence_mbar_init();
  }
  zero_rows(gbase + C::Q_OFF, 2 * QST * C::SLABS, kHalf, rows);  // the Q and dO stages
  if (warp == 2) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot_ptr;
  griddep_launch_dependents();  // this CTA holds its tensor memory
  griddep_wait();

  auto wait_item = [&](int i, bool& ok) {
    DkvItem it{-1, 0, 0, 0, 0, {0, 0, 0}};
    ok = mbar_wait(item_full(i & 1), (i >> 1) & 1, p.status);
    if (ok) it = items[i & 1];
    return it;
  };

  if (warp == 0) {
    // ------------------------------------------------------------- TMA
    if (elect_one_sync()) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_do);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      int issued = 0, n = 0;  // query tiles, key tiles
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const DkvItem it = wait_item(i, ok);
        if (it.b < 0) break;
        mbar_arrive(item_empty(i & 1));
        if (it.nq == 0) continue;
        ok = mbar_wait(kv_empty, (n & 1) ^ 1, p.status);
        if (!ok) break;
        mbar_arrive_expect_tx(kv_full, 2 * C::KTILE);
        for (int sl = 0; sl < C::SLABS; ++sl) {
          tma_load_4d(k_s + sl * C::KSLAB, &tm_k, kv_full, sl * 64, it.hk, it.kv0, it.b);
          tma_load_4d(v_s + sl * C::KSLAB, &tm_v, kv_full, sl * 64, it.hk, it.kv0, it.b);
        }
        ++n;
        for (int t = 0; t < subs * it.nq && ok; ++t) {
          const int s = issued % QST;
          ok = mbar_wait(q_empty(s), ((issued / QST) & 1) ^ 1, p.status);
          if (!ok) break;
          const int h = it.hk * sh.group + t / it.nq * sh.pack;
          const int tile = it.i0 + t % it.nq;
          const size_t srow =
              (static_cast<size_t>((it.b * sh.heads + h) / sh.pack) * sh.tiles64 + tile) * kHalf;
          mbar_arrive_expect_tx(q_full(s), 2 * C::SLABS * rows * 128 + C::STAT_BYTES);
          for (int sl = 0; sl < C::SLABS; ++sl) {
            tma_load_4d(q_s(s) + sl * C::QSLAB, &tm_q, q_full(s), sl * 64, h, tile * sh.pos64,
                        it.b);
            tma_load_4d(do_s(s) + sl * C::QSLAB, &tm_do, q_full(s), sl * 64, h, tile * sh.pos64,
                        it.b);
          }
          bulk_load(stat_s(s), p.work.nlse2 + srow, kHalf * 4, q_full(s));
          bulk_load(stat_s(s) + kHalf * 4, p.work.ndelta + srow, kHalf * 4, q_full(s));
          ++issued;
        }
      }
      // Never leave a copy in flight.
      if (n > 0) mbar_wait(kv_full, (n - 1) & 1, p.status);
      for (int t = issued - QST < 0 ? 0 : issued - QST; t < issued; ++t)
        mbar_wait(q_full(t % QST), (t / QST) & 1, p.status);
    }
  } else if (warp <= 2) {
    // --------------------- MMA: S^T and dV (warp 1), dP^T and dK (warp 2)
    if (elect_one_sync()) {
      constexpr uint32_t idesc_s = make_idesc_bf16(kTile, kHalf, false, false);
      constexpr uint32_t idesc_acc = make_idesc_bf16(kTile, D, false, true);
      int g = 0;  // query tiles, of all items: buffer g & 1, stage g % QST
      int n = 0;  // items with any
      const bool first = warp == 1;
      const uint32_t s_col = tmem + (first ? C::S_COL : C::DP_COL);
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const DkvItem it = wait_item(i, ok);
        if (it.b < 0) break;
        const int T = subs * it.nq;
        if (T == 0) {
          mbar_arrive(item_empty(i & 1));
          continue;
        }
        // dV += P^T_t dO_t and dK += dS^T_t Q_t: A from tensor memory, B
        // MN-major (N = dim, K = the tile's 64 queries).
        auto issue_acc = [&](int t, bool begin) -> bool {
          if (!mbar_wait(pds_ready(t & 1), (t >> 1) & 1, p.status)) return false;
          // The last item's dV and dK have been read before they begin again.
          if (begin && n > 0 && !mbar_wait(acc_free, (n - 1) & 1, p.status)) return false;
          tc_fence_after();
          const int s = t % QST;
          const uint32_t b = first ? do_s(s) : q_s(s);
#pragma unroll
          for (int kk = 0; kk < kHalf / 16; ++kk)
            umma_bf16_ts(tmem + (first ? C::DV_COL : C::DK_COL), s_col + (t & 1) * kHalf + kk * 16,
                         make_sdesc(b + kk * 2048, C::QSLAB, 1024, kSw128), idesc_acc,
                         (!begin || kk > 0) ? 1u : 0u);
          umma_commit(q_empty(s));
          return true;
        };
        ok = mbar_wait(kv_full, n & 1, p.status);
        for (int t = 0; t < T && ok; ++t, ++g) {
          const int s = g % QST;
          // Four query tiles before the end it is time to look for the next item.
          if (t == max(T - 4, 0)) mbar_arrive(item_empty(i & 1));
          // S^T_g (dP^T_g) goes over P^T (dS^T) of two tiles ago, whose product
          // is done when its stage is given back.
          ok = mbar_wait(q_full(s), (g / QST) & 1, p.status) &&
               (g < 2 || mbar_wait(q_empty((g - 2) % QST), ((g - 2) / QST) & 1, p.status));
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = first ? k_s : v_s, b = first ? q_s(s) : do_s(s);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16(s_col + (g & 1) * kHalf,
                      make_sdesc(a + (kk >> 2) * C::KSLAB + (kk & 3) * 32, 16, 1024, kSw128),
                      make_sdesc(b + (kk >> 2) * C::QSLAB + (kk & 3) * 32, 16, 1024, kSw128),
                      idesc_s, kk > 0);
          umma_commit(s_full(g & 1));
          if (t + 1 == T) umma_commit(kv_empty);
          if (t >= 1) ok = issue_acc(g - 1, t == 1);
        }
        if (!ok) break;
        ok = issue_acc(g - 1, T == 1);
        umma_commit(acc_full);
        ++n;
      }
      // Nothing may outlive the CTA's TMEM: the last commit covers every MMA.
      if (n > 0) mbar_wait(acc_full, (n - 1) & 1, p.status);
    }
  } else if (warp == 3) {
    // -------------------------------------------------------- scheduler
    const int bk_count = sh.batch * sh.kv_heads;
    for (int i = 0;; ++i) {
      // Not before the item before it nears its end.
      if (i > 0 && !mbar_wait(item_empty((i - 1) & 1), ((i - 1) >> 1) & 1, p.status)) break;
      const int n = i == 0 ? static_cast<int>(blockIdx.x)
                           : take_cta(base + C::TAKE_OFF, taken, i - 1, p.status);
      DkvItem it{-1, 0, 0, 0, 0, {0, 0, 0}};
      if (n >= 0) {
        const int bk = n % bk_count;
        it.b = bk / sh.kv_heads;
        it.hk = bk % sh.kv_heads;
        it.kv0 = n / bk_count * kTile;
        const Span* tiles = p.work.tiles + static_cast<size_t>(it.b) * sh.tiles64;
        int a = INT_MAX, z = -1;  // the first and last query tile that see it
        for (int q = lane; q < sh.tiles64; q += 32)
          if (tiles[q].lo < it.kv0 + kTile && tiles[q].hi > it.kv0) {
            a = min(a, q);
            z = q;
          }
        a = __reduce_min_sync(0xffffffffu, a);
        z = __reduce_max_sync(0xffffffffu, z);
        it.i0 = z >= 0 ? a : 0;
        it.nq = z >= 0 ? z + 1 - a : 0;
      }
      if (lane == 0) {
        items[i & 1] = it;
        mbar_arrive(item_full(i & 1));
      }
      __syncwarp();
      if (it.b < 0) break;
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------ compute warps
    // The warpgroups share the 128 key rows and split each tile's 64 query
    // columns, and dV's and dK's columns at the end.
    const int part = (warp - 4) >> 2;
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t lrow = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c = sh.scale_log2;
    const F2 c2 = f2(c, c);
    uint8_t* const out_s = gbase + C::OUT_OFF + (warp - 4) * C::OUT_BYTES;
    bool ok = true;
    int g = 0, n = 0;
    for (int i = 0; ok; ++i) {
      const DkvItem it = wait_item(i, ok);
      __syncwarp();
      if (lane == 0) mbar_arrive(item_empty(i & 1));
      if (it.b < 0) break;
      const int T = subs * it.nq;
      const size_t tile0 = static_cast<size_t>(it.b) * sh.tiles64 + it.i0;
      const int key0 = it.kv0 + quad * 32;  // the warp's 32 keys
      // The part's spans, a lane each, loaded a tile ahead (tile t % nq).
      const int2* const spans =
          p.work.rows + tile0 * kHalf + part * kPartCols + (lane & (kPartCols - 1));
      int ahead = 0;
      int2 nsp = T > 0 ? spans[0] : make_int2(0, 0);
      for (int t = 0; t < T; ++t, ++g) {
        const int s = g % QST;
        // Which of the tile's queries see which of the warp's keys: all, none,
        // or a bit each (lane i turns its query's span into bits of the keys,
        // the transpose gives each key's queries).
        const int2 sp = nsp;
        if (++ahead == it.nq) ahead = 0;
        nsp = spans[static_cast<size_t>(ahead) * kHalf];
        const int from = min(max(sp.x - key0, 0), 32);
        const int to = min(max(sp.x + sp.y - key0, 0), 32);
        const bool none = !__any_sync(0xffffffffu, from < to);
        const bool some = !__all_sync(0xffffffffu, from == 0 && to == 32);
        const uint32_t seen = !none && some ? transpose_bits(bit_range(from, to)) : 0;
        ok = mbar_wait(s_full(g & 1), (g >> 1) & 1, p.status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t scol = lrow + C::S_COL + (g & 1) * kHalf + part * kPartCols;
        const uint32_t dcol = lrow + C::DP_COL + (g & 1) * kHalf + part * kPartCols;
        uint32_t sv[kPartCols], dv[kPartCols];
        if (!none) {
          tmem_ld_32x32b_x32(scol, sv);
          tmem_ld_32x32b_x32(dcol, dv);
          tmem_ld_wait(sv, dv);
        }
        uint32_t pk[kPartCols / 16][8], dk[kPartCols / 16][8];  // by 16 queries
        if (none) {
#pragma unroll
          for (int e = 0; e < kPartCols / 2; ++e) pk[e / 8][e % 8] = dk[e / 8][e % 8] = 0;
        } else {
          if (some) {
#pragma unroll
            for (int e = 0; e < kPartCols; ++e)
              if (!(seen >> e & 1)) sv[e] = 0xFF800000u;  // P = 0
          }
          // The query tile's statistics (landed with its Q and dO).
          ok = mbar_wait(q_full(s), (g / QST) & 1, p.status);
          if (!ok) break;
          const float* st = reinterpret_cast<const float*>(gbase + (stat_s(s) - base)) + part * kPartCols;
#pragma unroll
          for (int e = 0; e < kPartCols; e += 4) {
            const float4 l4 = *reinterpret_cast<const float4*>(st + e);
            const float4 d4 = *reinterpret_cast<const float4*>(st + kHalf + e);
            const F2 pa = exp2_mufu(fma2(pair_of(sv[e], sv[e + 1]), c2, f2(l4.x, l4.y)));
            const F2 pb = exp2_mufu(fma2(pair_of(sv[e + 2], sv[e + 3]), c2, f2(l4.z, l4.w)));
            uint32_t(&pq)[8] = pk[e / 16];
            uint32_t(&dq)[8] = dk[e / 16];
            pq[e % 16 / 2] = pack_bf16(pa);
            pq[e % 16 / 2 + 1] = pack_bf16(pb);
            dq[e % 16 / 2] = pack_bf16(pa * (pair_of(dv[e], dv[e + 1]) + f2(d4.x, d4.y)));
            dq[e % 16 / 2 + 1] = pack_bf16(pb * (pair_of(dv[e + 2], dv[e + 3]) + f2(d4.z, d4.w)));
          }
          // The stat reads above are ordered before the copies that refill
          // the stage (generic-proxy reads, async-proxy writes).
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(q_empty(s));
#pragma unroll
        for (int e = 0; e < kPartCols / 16; ++e) {
          tmem_st_32x32b_x8(scol + 16 * e, pk[e]);
          tmem_st_32x32b_x8(dcol + 16 * e, dk[e]);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pds_ready(g & 1));
      }
      if (!ok) break;
      if (T > 0) {
        ok = mbar_wait(acc_full, n & 1, p.status);
        if (!ok) break;
        tc_fence_after();
        ++n;
      }
      const int key = it.kv0 + row;
      const bool valid = key < sh.seq;
      const size_t roff = ((static_cast<size_t>(it.b) * sh.seq + key) * sh.kv_heads + it.hk) * D;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const uint32_t col = which == 0 ? C::DV_COL : C::DK_COL;
        const float f = which == 0 ? 1.0f : p.scale;
        const F2 ff = f2(f, f);
        uint16_t* orow = (which == 0 ? p.dv : p.dk) + roff;
        constexpr int COLS = D / kParts;  // 64 or 32
        uint32_t wd[COLS / 32][16] = {};
        if (T > 0) {
          uint32_t o[COLS / 32][32];
#pragma unroll
          for (int e = 0; e < COLS / 32; ++e)
            tmem_ld_32x32b_x32(lrow + col + part * COLS + e * 32, o[e]);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < COLS / 32; ++e) keep_behind(o[e]);
          if (which == 1) {  // dV and dK may begin again
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_free);
          }
#pragma unroll
          for (int e = 0; e < COLS / 2; ++e)
            wd[e / 16][e % 16] =
                pack_bf16(pair_of(o[e / 16][2 * e % 32], o[e / 16][2 * e % 32 + 1]) * ff);
        }
#pragma unroll
        for (int e = 0; e < COLS / 32; ++e)
          store_rows(out_s, wd[e], orow + part * COLS + e * 32, valid);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// --------------------------------------------------------- document spans --
//
// One CTA per row of ids.  A document is a run of equal ids: a position's run
// starts at the last start at or before it and ends before the first one
// behind it.  A warp holds 256 positions in eight coalesced words a lane; a
// vote a word gives where runs start, bit operations the nearest start of a
// lane, and one value a warp in shared memory joins the warps.  A row longer
// than a stretch of 8192 goes stretch by stretch, from the front for the
// starts and from the back for the ends.  Latency is all there is to it: 4 us
// for one row of 8191, 6 with prefixes.

constexpr int kDocWarps = 32;
constexpr int kDocWords = 8;
constexpr int kStretch = kDocWarps * kDocWords * 32;

struct DocParams {
  const void* documents;
  const int* prefix;  // may be null
  int ids64, seq, causal;
  int* first;
  int* last;
};

// A warp's positions [i0, i0 + 256) of a row: bit l of starts[e] says whether a
// run starts at i0 + 32 e + l, bit l of pads[e] whether padding is there.
struct DocWords {
  uint32_t starts[kDocWords], pads[kDocWords];
};

template <typename I>
__device__ __forceinline__ DocWords read_words(const I* ids, int i0, int seq) {
  const int lane = threadIdx.x & 31;
  I v[kDocWords];
#pragma unroll
  for (int e = 0; e < kDocWords; ++e) v[e] = i0 + 32 * e + lane < seq ? ids[i0 + 32 * e + lane] : 0;
  I before = i0 > 0 && i0 <= seq ? ids[i0 - 1] : 0;  // the position ahead of the warp's
  DocWords w;
#pragma unroll
  for (int e = 0; e < kDocWords; ++e) {
    const int i = i0 + 32 * e + lane;
    I prev = __shfl_up_sync(0xffffffffu, v[e], 1);
    if (lane == 0) prev = before;
    before = __shfl_sync(0xffffffffu, v[e], 31);
    w.starts[e] = __ballot_sync(0xffffffffu, i < seq && (i == 0 || v[e] != prev));
    w.pads[e] = __ballot_sync(0xffffffffu, v[e] < 0);
  }
  return w;
}

template <typename I>
__device__ void document_spans(const DocParams& p) {
  __shared__ int sh[kDocWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * p.seq;
  const I* const ids = static_cast<const I*>(p.documents) + base;
  const uint32_t upto = 0xFFFFFFFFu >> (31 - lane);  // this lane and those below
  const int stretches = (p.seq + kStretch - 1) / kStretch;
  const bool ends = !p.causal || p.prefix;
  int from = 0;  // the start of the run that reaches into the stretch
  for (int s = 0; s < stretches; ++s) {
    const int i0 = s * kStretch + warp * (kDocWords * 32);
    const DocWords w = read_words(ids, i0, p.seq);
    int latest = -1;
#pragma unroll
    for (int e = 0; e < kDocWords; ++e)
      if (w.starts[e]) latest = i0 + 32 * e + 31 - __clz(w.starts[e]);
    __syncthreads();  // the last stretch's reads
    if (lane == 0) sh[warp] = latest;
    __syncthreads();
    int in = max(__reduce_max_sync(0xffffffffu, lane < warp ? sh[lane] : -1), from);
    from = max(__reduce_max_sync(0xffffffffu, sh[lane]), from);
#pragma unroll
    for (int e = 0; e < kDocWords; ++e) {
      const int i = i0 + 32 * e + lane;
      const uint32_t mine = w.starts[e] & upto;
      const int start = mine ? i0 + 32 * e + 31 - __clz(mine) : in;
      if (w.starts[e]) in = i0 + 32 * e + 31 - __clz(w.starts[e]);
      if (i >= p.seq) continue;
      const bool pad = w.pads[e] >> lane & 1;
      p.first[base + i] = start;
      if (!ends || pad) p.last[base + i] = pad ? start : i + 1;
    }
  }
  if (!ends) return;
  int next = p.seq;  // the start of the run after the stretch's last
  for (int s = stretches - 1; s >= 0; --s) {
    const int i0 = s * kStretch + warp * (kDocWords * 32);
    const DocWords w = read_words(ids, i0, p.seq);
    int prefix[kDocWords], first[kDocWords];
#pragma unroll
    for (int e = 0; e < kDocWords; ++e) {
      const int i = i0 + 32 * e + lane;
      first[e] = i < p.seq ? p.first[base + i] : 0;  // this thread wrote it
      prefix[e] = p.prefix && i < p.seq ? max(p.prefix[base + i], 0) : 0;
    }
    int earliest = INT_MAX;
#pragma unroll
    for (int e = kDocWords - 1; e >= 0; --e)
      if (w.starts[e]) earliest = i0 + 32 * e + __ffs(w.starts[e]) - 1;
    __syncthreads();
    if (lane == 0) sh[warp] = earliest;
    __syncthreads();
    int in = min(__reduce_min_sync(0xffffffffu, lane > warp ? sh[lane] : INT_MAX), next);
    next = min(__reduce_min_sync(0xffffffffu, sh[lane]), next);
#pragma unroll
    for (int e = kDocWords - 1; e >= 0; --e) {
      const int i = i0 + 32 * e + lane;
      const uint32_t behind = w.starts[e] & ~upto;
      const int stop = behind ? i0 + 32 * e + __ffs(behind) - 1 : in;
      if (w.starts[e]) in = i0 + 32 * e + __ffs(w.starts[e]) - 1;
      if (i >= p.seq || (w.pads[e] >> lane & 1)) continue;
      // Causally up to itself, and its prompt (which ends with the document).
      const int seen = prefix[e] < stop - first[e] ? first[e] + prefix[e] : stop;
      p.last[base + i] = p.causal ? max(i + 1, seen) : stop;
    }
  }
}

__global__ void __launch_bounds__(kDocWarps * 32) document_spans_kernel(const DocParams p) {
  griddep_wait();
  griddep_launch_dependents();
  if (p.ids64)
    document_spans<int64_t>(p);
  else
    document_spans<int>(p);
}

// -------------------------------------------------------------------- host --

// How many of the query heads that share a key/value head a packed tile holds:
// the most, up to 16, that divide them and fill at least 60 of 64 rows (4, 7
// and 8 of groups of those sizes; 7 of a group of 14; 1 of a group of 11).
int pack_of(int group) {
  for (int n = group < 16 ? group : 16; n > 1; --n)
    if (group % n == 0 && kHalf / n * n >= 60) return n;
  return 1;
}

SpanShape make_shape(int64_t batch, int64_t seq, int64_t heads, int64_t kv_heads, float scale) {
  SpanShape s{};
  s.batch = static_cast<int>(batch);
  s.seq = static_cast<int>(seq);
  s.heads = static_cast<int>(heads);
  s.kv_heads = static_cast<int>(kv_heads);
  s.group = static_cast<int>(heads / kv_heads);
  s.scale_log2 = scale * kLog2e;
  s.pack = pack_of(s.group);
  s.pos128 = kTile / s.pack;
  s.pos64 = kHalf / s.pack;
  s.tiles128 = (s.seq + s.pos128 - 1) / s.pos128;
  s.tiles64 = (s.seq + s.pos64 - 1) / s.pos64;
  s.key_tiles = (s.seq + kTile - 1) / kTile;
  return s;
}

BwdWork bwd_work(void* base, const SpanShape& sh) {
  const size_t tiles = static_cast<size_t>(sh.batch) * sh.tiles64;
  const size_t rows = tiles * kHalf * (sh.heads / sh.pack);
  uint8_t* at = static_cast<uint8_t*>(base);
  BwdWork w{};
  w.nlse2 = reinterpret_cast<float*>(at);
  w.ndelta = w.nlse2 + rows;
  w.bytes = 2 * rows * sizeof(float);
  w.rows = reinterpret_cast<int2*>(at + w.bytes);
  w.bytes += tiles * kHalf * sizeof(int2);
  w.tiles = reinterpret_cast<Span*>(at + w.bytes);
  w.bytes += tiles * sizeof(Span);
  return w;
}

int check_span_shape(int64_t batch, int64_t seq, int64_t heads, int64_t kv_heads, int64_t dim,
                     float scale) {
  const int rc = check_shape(batch, seq, heads, kv_heads, dim);
  if (rc) return rc;
  // Packed tiles number at most 64 / 60 of the plain ones and one more.
  if (batch * heads * (seq / kHalf + 2) > (1ll << 30))
    return fail(TQ_ERR_INVALID, "attention: shape too large");
  if (!(scale > 0.0f) || !std::isfinite(scale))
    return fail(TQ_ERR_INVALID, "attention: scale must be positive and finite");
  return TQ_OK;
}

template <int D>
int launch_fwd(const void* q, const void* k, const void* v, FwdParams p, cudaStream_t stream) {
  using C = FwdCfg<D>;
  const SpanShape& sh = p.sh;
  int rc = set_max_smem_once(reinterpret_cast<const void*>(span_fwd_kernel<D>), C::SMEM,
                             "cudaFuncSetAttribute(span_fwd)");
  if (rc) return rc;
  CUtensorMap tq_, tk, tv;
  if ((rc = map_bshd(&tq_, q, sh.batch, sh.seq, sh.heads, D, sh.pos128, sh.pack))) return rc;
  if ((rc = map_bshd(&tk, k, sh.batch, sh.seq, sh.kv_heads, D, kHalf))) return rc;
  if ((rc = map_bshd(&tv, v, sh.batch, sh.seq, sh.kv_heads, D, kHalf))) return rc;
  p.n_pairs = (sh.tiles128 + 1) / 2;
  const unsigned grid = static_cast<unsigned>(sh.batch) * (sh.heads / sh.pack) * p.n_pairs;
  return launch_kernel(span_fwd_kernel<D>, dim3(grid), dim3(kFwdThreads), C::SMEM,
                       stream, 1, "span attention forward launch", tq_, tk, tv, p);
}

template <int D>
int launch_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout,
               const float* lse, BwdParams p, cudaStream_t stream) {
  using Q = DqCfg<D>;
  using KV = DkvCfg<D>;
  const SpanShape& sh = p.sh;
  int rc = set_max_smem_once(reinterpret_cast<const void*>(span_dq_kernel<D>), Q::SMEM,
                             "cudaFuncSetAttribute(span_dq)");
  if (rc) return rc;
  rc = set_max_smem_once(reinterpret_cast<const void*>(span_dkv_kernel<D>), KV::SMEM,
                         "cudaFuncSetAttribute(span_dkv)");
  if (rc) return rc;
  // Query-side maps (128-row tiles for dq, 64-row tiles for dkv) and the
  // key/value maps the other way round.
  const uint32_t pack = sh.pack;
  CUtensorMap q128, do128, k64, v64, q64, do64, k128, v128;
  if ((rc = map_bshd(&q128, q, sh.batch, sh.seq, sh.heads, D, sh.pos128, pack))) return rc;
  if ((rc = map_bshd(&do128, dout, sh.batch, sh.seq, sh.heads, D, sh.pos128, pack))) return rc;
  if ((rc = map_bshd(&k64, k, sh.batch, sh.seq, sh.kv_heads, D, kHalf))) return rc;
  if ((rc = map_bshd(&v64, v, sh.batch, sh.seq, sh.kv_heads, D, kHalf))) return rc;
  if ((rc = map_bshd(&q64, q, sh.batch, sh.seq, sh.heads, D, sh.pos64, pack))) return rc;
  if ((rc = map_bshd(&do64, dout, sh.batch, sh.seq, sh.heads, D, sh.pos64, pack))) return rc;
  if ((rc = map_bshd(&k128, k, sh.batch, sh.seq, sh.kv_heads, D, kTile))) return rc;
  if ((rc = map_bshd(&v128, v, sh.batch, sh.seq, sh.kv_heads, D, kTile))) return rc;
  PrepParams pp{};
  pp.sh = sh;
  pp.out = static_cast<const uint16_t*>(out);
  pp.dout = static_cast<const uint16_t*>(dout);
  pp.lse = lse;
  pp.first = p.first;
  pp.last = p.last;
  pp.work = p.work;
  const int64_t tiles = static_cast<int64_t>(sh.batch) * sh.tiles64;
  constexpr int THREADS = 2 * D, WARPS = THREADS / 32;
  pp.row_blocks = static_cast<unsigned>(tiles * (sh.heads / sh.pack));
  const unsigned span_blocks = static_cast<unsigned>((tiles + WARPS - 1) / WARPS);
  rc = launch_kernel(span_prep_kernel<D>, dim3(pp.row_blocks + span_blocks), dim3(THREADS), 0,
                     stream, 1, "span attention backward prep launch", pp);
  if (rc) return rc;
  const unsigned grid_q = static_cast<unsigned>(sh.batch) * (sh.heads / sh.pack) * sh.tiles128;
  rc = launch_kernel(span_dq_kernel<D>, dim3(grid_q), dim3(kBwdThreads), Q::SMEM,
                     stream, 1, "span attention backward dq launch", q128, do128, k64, v64, p);
  if (rc) return rc;
  const unsigned grid_kv = static_cast<unsigned>(sh.batch) * sh.kv_heads * sh.key_tiles;
  return launch_kernel(span_dkv_kernel<D>, dim3(grid_kv), dim3(kBwdThreads), KV::SMEM,
                       stream, 1, "span attention backward dkv launch", q64, do64, k128, v128, p);
}

}  // namespace
}  // namespace tq

extern "C" int tq_span_attention_fwd(const void* q, const void* k, const void* v,
                                     const int32_t* first, const int32_t* last, int64_t batch,
                                     int64_t seq, int64_t heads, int64_t kv_heads,
                                     int64_t head_dim, float scale, void* out, float* lse,
                                     void* stream) {
  using namespace tq;
  int rc = check_span_shape(batch, seq, heads, kv_heads, head_dim, scale);
  if (rc) return rc;
  if (batch == 0 || seq == 0) return TQ_OK;
  if (!q || !k || !v || !first || !last || !out || !lse)
    return fail(TQ_ERR_INVALID, "attention: null pointer");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) ||
      !aligned(lse, 4))
    return fail(TQ_ERR_MISALIGNED, "attention: q, k, v and out must be 16-byte aligned");
  if (!aligned(first, 4) || !aligned(last, 4))
    return fail(TQ_ERR_MISALIGNED, "attention: first and last must be 4-byte aligned");
  FwdParams p{};
  p.status = device_status_ptr(&rc);
  if (!p.status) return rc;
  p.sh = make_shape(batch, seq, heads, kv_heads, scale);
  p.first = first;
  p.last = last;
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  return head_dim == 64 ? launch_fwd<64>(q, k, v, p, as_stream(stream))
                        : launch_fwd<128>(q, k, v, p, as_stream(stream));
}

extern "C" int tq_span_attention_bwd_workspace_bytes(int64_t batch, int64_t seq, int64_t heads,
                                                     int64_t kv_heads, size_t* bytes) {
  using namespace tq;
  if (!bytes) return fail(TQ_ERR_INVALID, "attention: null bytes pointer");
  const int rc = check_span_shape(batch, seq, heads, kv_heads, 128, 1.0f);
  if (rc) return rc;
  *bytes = bwd_work(nullptr, make_shape(batch, seq, heads, kv_heads, 1.0f)).bytes;
  return TQ_OK;
}

extern "C" int tq_span_attention_bwd(const void* q, const void* k, const void* v,
                                     const int32_t* first, const int32_t* last, const void* out,
                                     const void* dout, const float* lse, int64_t batch,
                                     int64_t seq, int64_t heads, int64_t kv_heads,
                                     int64_t head_dim, float scale, void* dq, void* dk, void* dv,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tq;
  int rc = check_span_shape(batch, seq, heads, kv_heads, head_dim, scale);
  if (rc) return rc;
  if (batch == 0 || seq == 0) return TQ_OK;
  BwdParams p{};
  p.sh = make_shape(batch, seq, heads, kv_heads, scale);
  p.work = bwd_work(workspace, p.sh);
  if (workspace_bytes < p.work.bytes)
    return fail(TQ_ERR_INVALID, "attention: workspace of %zu bytes, %zu needed", workspace_bytes,
                p.work.bytes);
  if (!q || !k || !v || !first || !last || !out || !dout || !lse || !dq || !dk || !dv ||
      !workspace)
    return fail(TQ_ERR_INVALID, "attention: null pointer");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) ||
      !aligned(dout, 16) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16) ||
      !aligned(workspace, 256) || !aligned(lse, 4))
    return fail(TQ_ERR_MISALIGNED,
                "attention: tensors must be 16-byte aligned and the workspace 256-byte aligned");
  if (!aligned(first, 4) || !aligned(last, 4))
    return fail(TQ_ERR_MISALIGNED, "attention: first and last must be 4-byte aligned");
  p.status = device_status_ptr(&rc);
  if (!p.status) return rc;
  p.first = first;
  p.last = last;
  p.scale = scale;
  p.dq = static_cast<uint16_t*>(dq);
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  return head_dim == 64 ? launch_bwd<64>(q, k, v, out, dout, lse, p, as_stream(stream))
                        : launch_bwd<128>(q, k, v, out, dout, lse, p, as_stream(stream));
}

extern "C" int tq_document_spans(const void* documents, int ids_bits, const int32_t* prefix,
                                 int64_t batch, int64_t seq, int causal, int32_t* first,
                                 int32_t* last, void* stream) {
  using namespace tq;
  if (ids_bits != 32 && ids_bits != 64)
    return fail(TQ_ERR_UNSUPPORTED, "document_spans: document ids must be 32- or 64-bit integers");
  if (batch < 0 || seq < 0 || batch > (1ll << 31) - 1 || seq > (1ll << 30))
    return fail(TQ_ERR_INVALID, "document_spans: batch and seq must be >= 0, seq at most 2^30");
  if (batch == 0 || seq == 0) return TQ_OK;
  if (!documents || !first || !last) return fail(TQ_ERR_INVALID, "document_spans: null pointer");
  if (!aligned(documents, ids_bits / 8) || !aligned(prefix, 4) || !aligned(first, 4) ||
      !aligned(last, 4))
    return fail(TQ_ERR_MISALIGNED, "document_spans: a pointer is not aligned to its type");
  DocParams p{};
  p.documents = documents;
  p.prefix = causal ? prefix : nullptr;
  p.ids64 = ids_bits == 64;
  p.seq = static_cast<int>(seq);
  p.causal = causal ? 1 : 0;
  p.first = first;
  p.last = last;
  return launch_kernel(document_spans_kernel, dim3(static_cast<unsigned>(batch)),
                       dim3(kDocWarps * 32), 0, as_stream(stream), 1, "document_spans launch", p);
}
