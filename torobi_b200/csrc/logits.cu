// What a trainer and a scorer read off the logits, beside the cross-entropy:
//
//   token_logprobs  ln q_t of given tokens t, the entropy of q and the most
//                   likely alternatives, q = softmax(z / T) over the row
//   distillation    the divergence KL(p || q) from a teacher's few given
//                   alternatives p, and the hard targets' cross-entropy
//
// and their gradients.  The reference has neither (its loss node is the
// cross-entropy of engine/src/interp.rs:434-444).
//
// Forward.  One pass over the row with the largest logit so far, m, and
// against it s = sum 2^x and a = sum x 2^x, x = (z - m) log2(e)/T: then
// ln q_j = (x_j - log2 s) ln 2 and H = (log2 s - a / s) ln 2, whose terms all
// have one sign.  Sums are f32; the difference comes before the product, so
// that logits of the type's lowest value neither overflow nor lose a row that
// holds nothing else (its distribution is uniform).  A -inf logit has
// probability 0 and adds nothing (x is held at -200, where 2^x is 0, so that
// x 2^x is 0); a row of nothing else has no distribution: ln q = -inf, H = 0
// and a gradient of 0.  NaN and +inf make the row NaN.
//
// Backward.  One pass that reads z and writes dz (which may be z itself).
//   dz_j = [ g ([j = t] - q_j) - h q_j (ln q_j + H) ] / T           (logprobs)
//   dz_j = u/T (q_j - sum_{i: id_i = j} p_i) + v (softmax(z)_j - [j = target])
//
// Rows are read in 32-byte chunks of the address space: a row that starts or
// ends inside one has that chunk read element by element, so any pitch and
// 2- or 4-byte alignment takes the same path.
#include <cuda_bf16.h>

#include <cmath>
#include <cstddef>
#include <type_traits>

#include "tq_ptx.cuh"
#include "tq_runtime.h"

namespace tq {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
// Forward: 32-byte chunks a thread has in flight, and CTAs an SM.  Four and
// four (64 registers) read 2046 x 128256 logits with the entropy in 88 us;
// two and six 92, two and eight 91, four and five 92, one and eight 93, and
// with the registers left to the compiler (two chunks: 92 registers) 115.
constexpr int kInFlight = 4;
constexpr int kPerSm = 4;
constexpr int kMaxTop = 128;     // alternatives a call may ask for or give
constexpr int kMaxSplit = 8;     // CTAs (one cluster) that may share a row
constexpr int kSpare = 32;       // chunks above the threshold taken beyond top
constexpr int kPool = 1024;      // candidates one CTA holds at a time
constexpr int kMaxChunks = 16384;  // chunk maxima one CTA keeps (top > 0)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ uint32_t max_nan_bf2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// Order-preserving image of a float: greater float, greater key; -0 is +0 and
// every NaN is above +inf.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(f + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// ------------------------------------------------------------------- rows --

template <typename T>
struct Elem;
template <>
struct Elem<uint16_t> {  // bf16
  static constexpr int CH = 16;
  static constexpr uint32_t NEG_INF2 = 0xFF80FF80u;
  __device__ static float load(const uint16_t* p) {
    return __uint_as_float(static_cast<uint32_t>(*p) << 16);
  }
  __device__ static void store(uint16_t* p, float f) {
    *p = __bfloat16_as_ushort(__float2bfloat16_rn(f));
  }
  __device__ static void unpack(const uint32_t (&w)[8], float (&f)[16]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ static void pack(const float (&f)[16], uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2_f32(f[2 * i], f[2 * i + 1]);
  }
  // The largest of a chunk, or of several: in a pair's two halves until value().
  using Max = uint32_t;
  using Bits = uint16_t;
  __device__ static Max chunk_max(const uint32_t (&w)[8]) {
    const uint32_t a = max_nan_bf2(max_nan_bf2(w[0], w[1]), max_nan_bf2(w[2], w[3]));
    const uint32_t b = max_nan_bf2(max_nan_bf2(w[4], w[5]), max_nan_bf2(w[6], w[7]));
    return max_nan_bf2(a, b);
  }
  __device__ static Max join(Max a, Max b) { return max_nan_bf2(a, b); }
  __device__ static Bits bits(Max m) {
    return static_cast<Bits>(max_nan_bf2(m, prmt(m, m, 0x1032)));
  }
  __device__ static float value(Max m) {
    return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
  }
  // order_key's upper half of the two values of a word: -0 becomes +0, then
  // negative ones are turned over and the others get the top bit.
  __device__ static uint32_t order_word(uint32_t w) {
    w = bf2_fma(w, 0x3F803F80u, 0);
    return w ^ (((w >> 15) & 0x00010001u) * 0x7FFFu | 0x80008000u);
  }
  __device__ static uint32_t max_words(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  __device__ static bool reaches(uint32_t w, uint32_t t) {
    return (w >> 16) >= t || (w & 0xFFFFu) >= t;
  }
};
template <>
struct Elem<float> {
  static constexpr int CH = 8;
  static constexpr uint32_t NEG_INF2 = 0xFF800000u;
  __device__ static float load(const float* p) { return *p; }
  __device__ static void store(float* p, float f) { *p = f; }
  __device__ static void unpack(const uint32_t (&w)[8], float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  }
  __device__ static void pack(const float (&f)[8], uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[i]);
  }
  using Max = float;
  using Bits = uint32_t;
  __device__ static Max chunk_max(const uint32_t (&w)[8]) {
    float f[8];
    unpack(w, f);
    return max_nan(max_nan(max_nan(f[0], f[1]), max_nan(f[2], f[3])),
                   max_nan(max_nan(f[4], f[5]), max_nan(f[6], f[7])));
  }
  __device__ static Max join(Max a, Max b) { return max_nan(a, b); }
  __device__ static Bits bits(Max m) { return __float_as_uint(m); }
  __device__ static float value(Max m) { return m; }
  __device__ static uint32_t order_word(uint32_t w) { return order_key(__uint_as_float(w)); }
  __device__ static uint32_t max_words(uint32_t a, uint32_t b) { return max(a, b); }
  __device__ static bool reaches(uint32_t w, uint32_t t) { return w >= t; }
};

// A row as the 32-byte chunks of memory that it touches.  Chunks in [lo, hi)
// lie wholly inside the row; chunk 0 and chunk n - 1 may not.
template <typename T>
struct Row {
  static constexpr int CH = Elem<T>::CH;
  const T* base;  // start of chunk 0, 32-byte aligned, at or before the row
  int off;        // elements of chunk 0 before the row
  int vocab;
  int n, lo, hi;
  __device__ Row(const T* row, int v) : vocab(v) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(row);
    off = static_cast<int>((a & 31u) / sizeof(T));
    base = row - off;
    const int64_t end = static_cast<int64_t>(off) + v;
    n = static_cast<int>((end + CH - 1) / CH);
    lo = off ? 1 : 0;
    hi = static_cast<int>(end / CH);
  }
  __device__ const T* chunk(int c) const { return base + static_cast<int64_t>(c) * CH; }
  // Index in the row of a chunk's first element (negative inside chunk 0).
  __device__ int64_t first(int c) const { return static_cast<int64_t>(c) * CH - off; }
  // A chunk that reaches out of the row, -inf where it does.
  __device__ void load_edge(int c, uint32_t (&w)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = Elem<T>::NEG_INF2;
    const int64_t j0 = first(c);
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      if (j0 + e < 0 || j0 + e >= vocab) continue;
      const T v = chunk(c)[e];
      if constexpr (sizeof(T) == 2) {
        const uint32_t sh = (e & 1) * 16;
        w[e / 2] = (w[e / 2] & ~(0xFFFFu << sh)) | (static_cast<uint32_t>(v) << sh);
      } else {
        w[e] = __float_as_uint(v);
      }
    }
  }
};

// A chunk that is read once.  (Not the read-only path: the kernel that writes
// the row may still run when this one is started.)
__device__ __forceinline__ void ld_chunk_once(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                 "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}

__device__ __forceinline__ void ld_chunk(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                 "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}

// The chunks c + u * kThreads, all in flight at once.  PART: those below `end`,
// -inf for the others (a thread's last round: one by one they would cost as
// many latencies).
template <bool PART, typename T, int U>
__device__ __forceinline__ void ld_chunks(const Row<T>& row, int c, int end, uint32_t (&w)[U][8]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!PART || c + u * kThreads < end) {
      ld_chunk_once(row.chunk(c + u * kThreads), w[u]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[u][i] = Elem<T>::NEG_INF2;
    }
  }
}

__device__ __forceinline__ void st_chunk(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
               "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// ------------------------------------------------------------ running sums --

// What a row's sums are of, beside s = sum 2^x: nothing, a = sum x 2^x (the
// entropy's), or a = sum 2^y, y = (z - m) log2(e) (a second temperature, 1);
// at temperature 2, 2^y is the square of 2^x, which spares the MUFU unit the
// second exponential (2046 x 128256: 85 us forward, 118 at temperature 3).
enum Mode { kPlain, kEntropy, kTwo, kSquare };

struct Sums {
  float m = -INFINITY, s = 0.0f, a = 0.0f;
};

// Moves the sums to the reference m (>= their own); c = log2(e)/T.  The bounds
// keep the products finite when the two are a whole range of f32 apart.
template <Mode M>
__device__ __forceinline__ void move_to(Sums& v, float m, float c) {
  const bool none = v.m == -INFINITY;
  const float up = none ? 300.0f : min_nan(m - v.m, 1e30f);
  const float d = min_nan(up * c, 300.0f);  // 2^-300 is 0 already
  const float f = ex2_approx(-d);
  if (M == kEntropy) v.a = f * fmaf(-d, v.s, v.a);
  if (M == kTwo) v.a *= ex2_approx(-up * kLog2e);
  if (M == kSquare) v.a *= f * f;
  v.s *= f;
  v.m = m;
}

template <Mode M>
__device__ __forceinline__ void merge(Sums& v, Sums o, float c) {
  const float m = max_nan(v.m, o.m);
  if (m == -INFINITY) return;
  move_to<M>(v, m, c);
  move_to<M>(o, m, c);
  v.s += o.s;
  v.a += o.a;
}

// 2^x of two x <= 0 on the FMA pipe: x = n + f with n the nearest integer (x +
// 1.5 2^23 has it in its low bits), 2^f by a polynomial fitted to the least
// relative error over [-1/2, 1/2] (2.1e-7 in f32, the MUFU unit's 2^-22), n
// added to the exponent.  Below -125 it stays 2^-125, nothing beside sums >= 1;
// of a NaN any value.
__device__ __forceinline__ F2 exp2_fma(F2 x) {
  const float2 v = split(x);
  x = f2(fmaxf(v.x, -125.0f), fmaxf(v.y, -125.0f));
  const F2 magic = f2(12582912.0f, 12582912.0f), unmagic = f2(-12582912.0f, -12582912.0f);
  const F2 one = f2(1.0f, 1.0f), minus = f2(-1.0f, -1.0f);
  const F2 t = x + magic;
  const F2 f = fma2(t + unmagic, minus, x);
  F2 p = fma2(f2(0.00132764719f, 0.00132764719f), f, f2(0.00967554133f, 0.00967554133f));
  p = fma2(p, f, f2(0.0555071327f, 0.0555071327f));
  p = fma2(p, f, f2(0.240221197f, 0.240221197f));
  p = fma2(p, f, f2(0.693146967f, 0.693146967f));
  p = fma2(p, f, one);
  const float2 a = split(p), n = split(t);
  return f2(__uint_as_float(__float_as_uint(a.x) + (__float_as_uint(n.x) << 23)),
            __uint_as_float(__float_as_uint(a.y) + (__float_as_uint(n.y) << 23)));
}

// Adds U chunks whose largest logit is mx.
template <typename T, Mode M, int U>
__device__ __forceinline__ void add_chunks(Sums& v, const uint32_t (&w)[U][8], float mx, float c) {
  constexpr int CH = Elem<T>::CH;
  const float m = max_nan(v.m, mx);
  if (m == -INFINITY) return;
  move_to<M>(v, m, c);
  F2 s = f2(0.0f, 0.0f), a = s;
  const F2 minus_m = f2(-m, -m), cc = f2(c, c), c1 = f2(kLog2e, kLog2e);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[CH];
    Elem<T>::unpack(w[u], f);
#pragma unroll
    for (int e = 0; e < CH; e += 2) {
      const F2 d = f2(f[e], f[e + 1]) + minus_m;
      float2 x = split(d * cc);
      if (M == kEntropy) x = make_float2(max_nan(x.x, -200.0f), max_nan(x.y, -200.0f));
      const F2 p = f2(ex2_approx(x.x), ex2_approx(x.y));
      s = s + p;
      if (M == kEntropy) a = fma2(p, f2(x.x, x.y), a);
      if (M == kTwo) {
        // Every other pair's on the FMA pipe: two a logit on the MUFU unit
        // took 139 us for 2046 x 128256, where reading them takes 82.
        if (e & 2) {
          a = a + exp2_fma(d * c1);
        } else {
          const float2 y = split(d * c1);
          a = a + f2(ex2_approx(y.x), ex2_approx(y.y));
        }
      }
      if (M == kSquare) a = fma2(p, p, a);
    }
  }
  const float2 ss = split(s), aa = split(a);
  v.s += ss.x + ss.y;
  if (M != kPlain) v.a += aa.x + aa.y;
}

// The block's sums, in sh[0] for every thread after the call.
template <Mode M>
__device__ __forceinline__ void block_sums(Sums v, Sums* sh, float c) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float m = warp_max(v.m);
  if (m != -INFINITY) move_to<M>(v, m, c);
  v.s = warp_add(v.s);
  v.a = warp_add(v.a);
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  if (warp == 0) {
    Sums t;
    if (lane < kWarps) t = sh[lane];
    const float top = warp_max(t.m);
    if (top != -INFINITY) move_to<M>(t, top, c);
    t.s = warp_add(t.s);
    t.a = warp_add(t.a);
    __syncwarp();
    if (lane == 0) sh[0] = t;
  }
  __syncthreads();
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ uint64_t ld_cluster_u64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// The sums of the cluster's CTAs (each one's in its sh[0]), merged in rank
// order; by one thread of the leader, between two cluster barriers.
template <Mode M>
__device__ __forceinline__ Sums cluster_sums(Sums* sh, int split, float c) {
  Sums t = sh[0];
  for (int i = 1; i < split; ++i) {
    const uint32_t at = mapa_shared(smem_u32(sh), i);
    Sums o;
    o.m = ld_cluster_f32(at);
    o.s = ld_cluster_f32(at + 4);
    o.a = ld_cluster_f32(at + 8);
    merge<M>(t, o, c);
  }
  return t;
}

// ------------------------------------------------------------ alternatives --

__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// A logit and its index as one number: greater logit first, then lower index.
__device__ __forceinline__ uint64_t candidate(uint32_t key, uint32_t index) {
  return (static_cast<uint64_t>(key) << 32) | (0xFFFFFFFFu - index);
}

// Sorts n (a power of two) numbers, greatest first.
__device__ void sort_descending(uint64_t* v, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int a = 2 * i - (i & (step - 1)), b = a + step;
        const uint64_t x = v[a], y = v[b];
        if ((x < y) == ((a & size) == 0)) {
          v[a] = y;
          v[b] = x;
        }
      }
    }
  __syncthreads();
}

// The k greatest of n <= kPool distinct numbers in `in` (room for kPool), in
// order, to out[0, k), which may be in itself; places past n get 0.  in may be
// reordered; rank: kThreads ints.
__device__ void greatest(uint64_t* in, int n, int k, uint64_t* out, int* rank) {
  if (n <= kThreads) {
    // Each number's rank is how many are greater: `parts` threads count for
    // one number.
    rank[threadIdx.x] = 0;
    __syncthreads();
    int p = 16;
    while (p < n) p <<= 1;
    const int i = threadIdx.x & (p - 1), parts = kThreads / p;
    const uint64_t x = i < n ? in[i] : 0;
    int greater = 0;
    if (i < n)
      for (int j = threadIdx.x / p; j < n; j += parts) greater += in[j] > x;
    if (greater) atomicAdd(rank + i, greater);
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < n && rank[i] < k) out[rank[i]] = x;
    for (int j = n + threadIdx.x; j < k; j += kThreads) out[j] = 0;
  } else {
    int p = 2 * kThreads;
    while (p < n) p <<= 1;
    for (int i = n + threadIdx.x; i < p; i += kThreads) in[i] = 0;
    sort_descending(in, p);
    for (int i = threadIdx.x; i < k; i += kThreads) out[i] = in[i];
  }
  __syncthreads();
}

template <typename T>
using ChunkKey = typename Elem<T>::Bits;

template <typename T>
__device__ __forceinline__ ChunkKey<T> chunk_key(float m) {
  return static_cast<ChunkKey<T>>(order_key(m) >> (sizeof(T) == 2 ? 16 : 0));
}

struct alignas(16) TopShared {  // mine is read in 16-byte words
  uint64_t best[kMaxTop];
  union {
    uint32_t mine[kThreads];  // the threads' maxima
    int rank[kThreads];
  };
  int chunks[2 * kMaxTop + kSpare];
  int scan[kWarps];
  int above, equal, listed, found;
  uint32_t threshold;
};
static_assert(offsetof(TopShared, mine) % 16 == 0, "16-byte words");

// The largest t that at least `top` of the 256 keys in sh.mine reach; one warp
// searches bit by bit below the highest bit in which the greatest and the
// least key differ.
__device__ __forceinline__ uint32_t threshold(const TopShared& sh, int top) {
  const uint4* k = reinterpret_cast<const uint4*>(sh.mine) + 2 * (threadIdx.x & 31);
  const uint4 a = k[0], b = k[1];
  const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t lo = v[0], hi = v[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min(lo, v[i]);
    hi = max(hi, v[i]);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lo == hi) return hi;
  uint32_t bit = 0x80000000u >> __clz(lo ^ hi);
  uint32_t t = hi & ~(2 * bit - 1);
#pragma unroll 1
  for (; bit; bit >>= 1) {
    const uint32_t probe = t | bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) n += v[i] >= probe;
    if (__reduce_add_sync(0xffffffffu, n) >= top) t = probe;
  }
  return t;
}

// Every element of the chunks listed in [l0, l1) that reaches the threshold,
// behind the sh.found that are in the pool already; a thread a chunk.  Counts
// what does not fit, too.
template <typename T>
__device__ __forceinline__ void gather(const Row<T>& row, int l0, int l1, uint32_t floor_key,
                                       uint64_t* pool, TopShared& sh) {
  constexpr int CH = Elem<T>::CH;
  const float least = key_value(floor_key);
  const bool nan = floor_key > order_key(INFINITY);
  for (int i = l0 + threadIdx.x; i < l1; i += kThreads) {
    const int c = sh.chunks[i];
    uint32_t w[8];
    if (c >= row.lo && c < row.hi)
      ld_chunk_once(row.chunk(c), w);
    else
      row.load_edge(c, w);
    float f[CH];
    Elem<T>::unpack(w, f);
    const int64_t j0 = row.first(c);
    // A bit an element, then one place in the pool a thread.  (A NaN is not
    // below any number; where the threshold is NaN itself, only NaN reaches it.)
    uint32_t hits = 0;
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      const bool in = c >= row.lo && c < row.hi ? true : j0 + e >= 0 && j0 + e < row.vocab;
      if (in && (nan ? f[e] != f[e] : !(f[e] < least))) hits |= 1u << e;
    }
    int at = hits ? atomicAdd(&sh.found, __popc(hits)) : 0;
#pragma unroll
    for (int e = 0; e < CH; ++e)
      if (hits >> e & 1) {
        if (at < kPool) pool[at] = candidate(order_key(f[e]), static_cast<uint32_t>(j0 + e));
        ++at;
      }
  }
  __syncthreads();
}

// The slice's `top` greatest logits, in order, to sh.best (0 past its end).
//   keys[0, n)  the largest logit of each chunk c0 + i, its bits
//   mine        the largest of this thread's chunks (the chunks are disjoint)
// The threshold t is the top-th greatest of the threads' maxima: at least
// `top` chunks reach it, and few more do.  Those are read again, and every
// element that reaches t is a candidate.  A row built against this (equal
// logits, large ones side by side) may have more chunks at or above t than
// the list holds: t then becomes the top-th greatest of all chunk maxima,
// fewer than `top` chunks are above it, and of those that equal it the first
// `top` are enough (ties go to the lowest index, and each holds one).  More
// candidates than the pool holds are gone through in parts.  It is latency
// behind the pass over the row -- one barrier to share the maxima, one scan of
// the keys, one reading of the chunks, one ranking -- and the SM's other three
// CTAs cover only part of it: 4092 x 151936 takes 184 us without alternatives,
// 213 with one, 238 with 64, 267 with 128.
template <typename T>
__device__ void slice_top(const Row<T>& row, int c0, int n, int top, ChunkKey<T>* keys, float mine,
                          bool any, uint64_t* pool, TopShared& sh) {
  constexpr int BITS = 8 * sizeof(ChunkKey<T>);
  constexpr int PER = 16 / sizeof(ChunkKey<T>);  // keys in 16 bytes
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int room = 2 * top + kSpare;
  sh.mine[threadIdx.x] = any ? chunk_key<T>(mine) : 0;
  if (threadIdx.x == 0) sh.listed = sh.found = 0;
  __syncthreads();
  if (warp == 0) {
    const uint32_t found = threshold(sh, top);
    if (lane == 0) sh.threshold = found;
  }
  __syncthreads();
  uint32_t t = sh.threshold;
  for (int i = PER * threadIdx.x; i < n; i += PER * kThreads) {
    // In order from here.  The keys' room is whole 16-byte words; what is
    // behind the last key is not looked at.
    uint4* const at4 = reinterpret_cast<uint4*>(keys + i);
    uint4 q = *at4;
    q.x = Elem<T>::order_word(q.x);
    q.y = Elem<T>::order_word(q.y);
    q.z = Elem<T>::order_word(q.z);
    q.w = Elem<T>::order_word(q.w);
    *at4 = q;
    const uint32_t m =
        Elem<T>::max_words(Elem<T>::max_words(q.x, q.y), Elem<T>::max_words(q.z, q.w));
    if (!Elem<T>::reaches(m, t)) continue;
    const uint32_t words[4] = {q.x, q.y, q.z, q.w};
    uint32_t hits = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const uint32_t k = PER == 4 ? words[e % 4] : words[e / 2] >> (e & 1) * 16 & 0xFFFFu;
      if (k >= t && i + e < n) hits |= 1u << e;
    }
    if (!hits) continue;
    int at = atomicAdd(&sh.listed, __popc(hits));
    for (; hits; hits &= hits - 1, ++at)
      if (at < room) sh.chunks[at] = c0 + i + __ffs(hits) - 1;
  }
  __syncthreads();
  if (sh.listed > room) {
    auto count = [&](uint32_t at, int& above, int& equal) {
      if (threadIdx.x == 0) sh.above = sh.equal = 0;
      __syncthreads();
      int a = 0, q = 0;
      for (int i = threadIdx.x; i < n; i += kThreads) {
        a += keys[i] > at;
        q += keys[i] == at;
      }
      a = __reduce_add_sync(0xffffffffu, a);
      q = __reduce_add_sync(0xffffffffu, q);
      if (lane == 0) {
        atomicAdd(&sh.above, a);
        atomicAdd(&sh.equal, q);
      }
      __syncthreads();
      above = sh.above;
      equal = sh.equal;
      __syncthreads();
    };
    int above, equal;
    t = 0;
#pragma unroll 1
    for (int b = BITS - 1; b >= 0; --b) {
      const uint32_t probe = t | (1u << b);
      count(probe, above, equal);
      if (above + equal >= top) t = probe;
    }
    if (threadIdx.x == 0) sh.listed = 0;
    // The first `top` of the equal ones in index order: each thread counts
    // its own stretch, a prefix sum gives its places.
    const int per = (n + kThreads - 1) / kThreads;
    const int i0 = min(n, static_cast<int>(threadIdx.x) * per), i1 = min(n, i0 + per);
    int q = 0;
    for (int i = i0; i < i1; ++i) q += keys[i] == t;
    int before = q;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, before, off);
      if (lane >= off) before += o;
    }
    if (lane == 31) sh.scan[warp] = before;
    __syncthreads();
    for (int i = 0; i < warp; ++i) before += sh.scan[i];
    before -= q;
    for (int i = i0; i < i1; ++i) {
      const bool eq = keys[i] == t;
      if (keys[i] > t || (eq && before < top)) sh.chunks[atomicAdd(&sh.listed, 1)] = c0 + i;
      before += eq;
    }
    __syncthreads();
  }
  // The keys' room is the candidates' from here.
  const int listed = sh.listed;
  const uint32_t floor_key = t << (32 - BITS);
  gather<T>(row, 0, listed, floor_key, pool, sh);
  if (sh.found <= kPool) {
    greatest(pool, sh.found, top, sh.best, sh.rank);
    return;
  }
  // As many chunks at a time as surely fit beside the best so far.
  constexpr int STEP = (kPool - kMaxTop) / Elem<T>::CH;
  for (int l0 = 0; l0 < listed; l0 += STEP) {
    __syncthreads();
    if (threadIdx.x == 0) sh.found = l0 ? top : 0;
    if (l0)
      for (int i = threadIdx.x; i < top; i += kThreads) {
        const uint64_t x = sh.best[i];
        // Places not yet taken: distinct, below every logit.
        pool[i] = x ? x : static_cast<uint64_t>(i) + 1;
      }
    __syncthreads();
    gather<T>(row, l0, min(listed, l0 + STEP), floor_key, pool, sh);
    greatest(pool, sh.found, top, sh.best, sh.rank);
  }
}

// ----------------------------------------------------------- token_logprobs --

struct LogprobParams {
  const void* z;
  const int64_t* tokens;
  int64_t ld;
  int vocab, split, top;
  float c, inv_t;  // log2(e) / temperature, 1 / temperature
  float* logprobs;
  float* entropy;
  float4* stats;
  float* top_logprobs;
  int64_t* top_ids;
};

// One CTA per row, or a cluster of `split` CTAs when rows are few, each a
// contiguous slice of the row's chunks; rank 0 joins them in rank order.  Bound
// by reading the logits: 2046 x 128256 in 84 us, 6.2 TB/s, one call behind the
// other (behind a backward pass, whose last writes leave L2 meanwhile, 97 to 105);
// 777 x 32003 f32, rows of 16 chunks a thread, 22 us, 4.6 TB/s.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, kPerSm) logprobs_fwd_kernel(const LogprobParams p) {
  constexpr int U = kInFlight;
  extern __shared__ __align__(16) uint64_t pool[];
  __shared__ Sums sums[kWarps];
  __shared__ float2 total;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t r = blockIdx.x / p.split;
  const int rank = static_cast<int>(blockIdx.x % p.split);
  const Row<T> row(static_cast<const T*>(p.z) + r * p.ld, p.vocab);
  const int per = (row.n + p.split - 1) / p.split;
  const int c0 = min(row.n, rank * per), c1 = min(row.n, c0 + per);
  ChunkKey<T>* keys = reinterpret_cast<ChunkKey<T>*>(pool);
  const float c = p.c;
  // The given token's logit, ahead of the row (two loads one behind the other
  // at the row's end would cost as much as the selection).
  bool given = false;
  float picked = 0.0f;
  if (threadIdx.x == 0 && rank == 0) {
    const int64_t tok = p.tokens[r];
    given = tok >= 0 && tok < p.vocab;
    if (given) picked = Elem<T>::load(static_cast<const T*>(p.z) + r * p.ld + tok);
  }
  Sums v;
  float mine = -INFINITY;
  bool any = false;
  auto one = [&](int ch, const uint32_t (&w)[1][8]) {
    const typename Elem<T>::Max cm = Elem<T>::chunk_max(w[0]);
    const float mx = Elem<T>::value(cm);
    if constexpr (TOP) {
      keys[ch - c0] = Elem<T>::bits(cm);
      mine = max_nan(mine, mx);
      any = true;
    }
    add_chunks<T, kEntropy, 1>(v, w, mx, c);
  };
  const int lo = max(c0, row.lo), hi = min(c1, row.hi);
  if (threadIdx.x == 0 && c0 == 0 && c1 > 0 && row.lo == 1) {
    uint32_t w[1][8];
    row.load_edge(0, w[0]);
    one(0, w);
  }
  if (threadIdx.x == kThreads - 1 && c1 == row.n && c0 < c1 && row.hi < row.n &&
      row.n - 1 >= row.lo) {
    uint32_t w[1][8];
    row.load_edge(row.n - 1, w[0]);
    one(row.n - 1, w);
  }
  auto many = [&](int ch, auto part) {
    constexpr bool PART = decltype(part)::value;
    uint32_t w[U][8];
    ld_chunks<PART>(row, ch, hi, w);
    typename Elem<T>::Max all;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const typename Elem<T>::Max cm = Elem<T>::chunk_max(w[u]);
      if constexpr (TOP)
        if (!PART || ch + u * kThreads < hi) keys[ch + u * kThreads - c0] = Elem<T>::bits(cm);
      all = u ? Elem<T>::join(all, cm) : cm;
    }
    const float mx = Elem<T>::value(all);
    if constexpr (TOP) {
      mine = max_nan(mine, mx);
      any = true;
    }
    add_chunks<T, kEntropy, U>(v, w, mx, c);
  };
  int ch = lo + threadIdx.x;
  for (; ch + (U - 1) * kThreads < hi; ch += U * kThreads) many(ch, std::false_type());
  if constexpr (!TOP)  // (with the selection it would spill registers)
    if (ch + kThreads < hi) {
      many(ch, std::true_type());
      ch = hi;
    }
  for (; ch < hi; ch += kThreads) {
    uint32_t w[1][8];
    ld_chunk_once(row.chunk(ch), w[0]);
    one(ch, w);
  }
  block_sums<kEntropy>(v, sums, c);
  uint64_t* best = nullptr;
  int* rank_of = nullptr;
  if constexpr (TOP) {
    __shared__ TopShared sh;
    slice_top<T>(row, c0, c1 - c0, p.top, keys, mine, any, pool, sh);
    best = sh.best;
    rank_of = sh.rank;
  }
  if (p.split > 1) {
    cluster_sync();
    if (rank == 0) {
      if constexpr (TOP)
        for (int i = threadIdx.x; i < p.split * p.top; i += kThreads) {
          const uint64_t x = ld_cluster_u64(mapa_shared(smem_u32(best + i % p.top), i / p.top));
          // Places past a short slice's end: distinct, below every logit.
          pool[i] = x ? x : static_cast<uint64_t>(i) + 1;
        }
      if (threadIdx.x == 0) v = cluster_sums<kEntropy>(sums, p.split, c);
    }
    cluster_sync();  // the leader has read every CTA's shared memory
    if (rank != 0) return;
    if constexpr (TOP) greatest(pool, p.split * p.top, p.top, best, rank_of);
  } else if (threadIdx.x == 0) {
    v = sums[0];
  }
  if (threadIdx.x == 0) {
    const bool none = v.m == -INFINITY;
    const float m = none ? 0.0f : v.m;
    const float l2 = log2f(v.s);  // -inf for a row of nothing but -inf
    const float h = none ? 0.0f : (l2 - v.a / v.s) * kLn2;
    float lp = 0.0f;
    if (given) lp = none ? -INFINITY : fmaf(picked - m, p.inv_t, -l2 * kLn2);
    p.logprobs[r] = lp;
    p.entropy[r] = h;
    if (p.stats) p.stats[r] = make_float4(m, l2, h, 0.0f);
    total = make_float2(m, l2);
  }
  if constexpr (TOP) {
    __syncthreads();
    for (int i = threadIdx.x; i < p.top; i += kThreads) {
      const float z = key_value(static_cast<uint32_t>(best[i] >> 32));
      p.top_logprobs[r * p.top + i] =
          total.y == -INFINITY ? -INFINITY : fmaf(z - total.x, p.inv_t, -total.y * kLn2);
      p.top_ids[r * p.top + i] = 0xFFFFFFFFu - static_cast<uint32_t>(best[i]);
    }
  }
}

// --------------------------------------------------------------- gradients --

// Hands grad(j0, f) the logits f[0, N) of this CTA's share of a row, j0 the
// index of the first, and stores what it leaves in f.  ready() is called once
// by every thread before grad, with the first loads under way.  SAME: z's and
// dz's rows start at the same offset in their 32-byte chunks, so a chunk is
// loaded and stored whole; otherwise elements go one by one.
template <typename T, bool SAME, typename Ready, typename Grad>
__device__ __forceinline__ void row_gradient(const T* z, T* dz, int vocab, int part, int parts,
                                             Ready&& ready, Grad&& grad) {
  constexpr int CH = Elem<T>::CH;
  const Row<T> row(z, vocab);
  const int per = (row.n + parts - 1) / parts;
  const int c0 = min(row.n, part * per), c1 = min(row.n, c0 + per);
  if constexpr (SAME) {
    const int lo = max(c0, row.lo), hi = min(c1, row.hi);
    T* const out = dz - row.off;
    auto finish = [&](int c, uint32_t(&w)[8]) {
      float f[CH];
      Elem<T>::unpack(w, f);
      grad(row.first(c), f);
      Elem<T>::pack(f, w);
      st_chunk(out + static_cast<int64_t>(c) * CH, w);
    };
    // Two chunks' loads in flight a thread before either is finished.
    uint32_t w0[8], w1[8];
    int c = lo + threadIdx.x;
    auto load = [&] {
      if (c < hi) ld_chunk(row.chunk(c), w0);
      if (c + kThreads < hi) ld_chunk(row.chunk(c + kThreads), w1);
    };
    load();
    ready();
    while (c < hi) {
      finish(c, w0);
      if (c + kThreads < hi) finish(c + kThreads, w1);
      c += 2 * kThreads;
      load();
    }
    // The first and last chunk, where they reach out of the row.
    const int64_t head = c0 == 0 && row.lo == 1 ? min(CH - row.off, vocab) : 0;
    const int64_t tail0 =
        c1 == row.n && row.hi < row.n && row.n - 1 >= row.lo ? row.first(row.n - 1) : vocab;
    const int tail = static_cast<int>(vocab - tail0);
    if (c0 < c1 && static_cast<int>(threadIdx.x) < head + tail) {
      const int64_t j =
          static_cast<int>(threadIdx.x) < head ? threadIdx.x : tail0 + (threadIdx.x - head);
      float f[1] = {Elem<T>::load(z + j)};
      grad(j, f);
      Elem<T>::store(dz + j, f[0]);
    }
  } else {
    ready();
    const int64_t j0 = max(row.first(c0), static_cast<int64_t>(0));
    const int64_t j1 = min(row.first(c1), static_cast<int64_t>(vocab));
    for (int64_t j = j0 + threadIdx.x; j < j1; j += kThreads) {
      float f[1] = {Elem<T>::load(z + j)};
      grad(j, f);
      Elem<T>::store(dz + j, f[0]);
    }
  }
}

struct LogprobGradParams {
  const void* z;
  const int64_t* tokens;
  const float4* stats;
  const float* dlogprobs;
  const float* dentropy;
  void* dz;
  int64_t ld, ld_out;
  int vocab, parts;
  float c, inv_t;  // log2(e) / temperature, 1 / temperature
};

// Bound by reading and writing: 2046 x 128256 in 160 us, 6.6 TB/s (in place and
// behind the forward 150, with rows left in L2).
template <typename T, bool SAME>
__global__ void __launch_bounds__(kThreads) logprobs_bwd_kernel(const LogprobGradParams p) {
  griddep_wait();
  griddep_launch_dependents();
  // Last row first: the forward's last rows may still be in L2.
  const int64_t r = gridDim.x / p.parts - 1 - blockIdx.x / p.parts;
  const int part = static_cast<int>(blockIdx.x % p.parts);
  const float c = p.c;
  int64_t tok;
  float m, ca, cb, hot;
  bool zero;
  row_gradient<T, SAME>(
      static_cast<const T*>(p.z) + r * p.ld, static_cast<T*>(p.dz) + r * p.ld_out, p.vocab, part,
      p.parts,
      [&] {
        const float4 st = p.stats[r];  // m, log2 s, entropy
        tok = p.tokens[r];
        const bool picked = tok >= 0 && tok < p.vocab;
        float g = p.dlogprobs ? p.dlogprobs[r] : 0.0f;
        const float h = p.dentropy ? p.dentropy[r] : 0.0f;
        if (!picked) g = 0.0f;
        m = st.x;
        // q_j (g + h (ln q_j + H)) / T = 2^x (ca + cb x); a row that no gradient
        // reaches, or without a distribution, gets zeros whatever it holds.
        zero = (g == 0.0f && h == 0.0f) || st.y == -INFINITY;
        const float inv_s = exp2f(-st.y) * p.inv_t;
        ca = inv_s * (g + h * (st.z - st.y * kLn2));
        cb = inv_s * h * kLn2;
        hot = zero ? 0.0f : g * p.inv_t;
      },
      [&](int64_t j0, auto& f) {
        constexpr int N = sizeof(f) / sizeof(float);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float x = max_nan((f[e] - m) * c, -200.0f);
          f[e] = zero ? 0.0f : -ex2_approx(x) * fmaf(cb, x, ca);
        }
        if (tok >= j0 && tok < j0 + N) {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (tok == j0 + e) f[e] += hot;
        }
      });
}

// ------------------------------------------------------------ distillation --

struct Teacher {
  const void* ids;
  const void* logits;
  int ids64, logits_bf16, k;
  __device__ int64_t id(int64_t i) const {
    return ids64 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
  }
  __device__ float logit(int64_t i) const {
    return logits_bf16 ? Elem<uint16_t>::load(static_cast<const uint16_t*>(logits) + i)
                       : static_cast<const float*>(logits)[i];
  }
};

constexpr int kPerLane = kMaxTop / 32;

// A warp's view of one row's alternatives: ids (-1 where there is none), their
// log2 p and p, with p = 0 for a teacher logit of -inf.
struct Alternatives {
  int id[kPerLane];
  float lp[kPerLane], p[kPerLane];
};

// id(e) and logit(e) answer for entry e < k.
template <typename Id, typename Logit>
__device__ __forceinline__ Alternatives weigh(int k, int vocab, float c, Id&& id_of,
                                              Logit&& logit_of) {
  const int lane = threadIdx.x & 31;
  Alternatives a;
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int e = lane + 32 * i;
    a.id[i] = -1;
    a.lp[i] = -INFINITY;
    if (e < k) {
      const int64_t id = id_of(e);
      if (id >= 0 && id < vocab) {
        a.id[i] = static_cast<int>(id);
        a.lp[i] = logit_of(e);
      }
    }
    mx = max_nan(mx, a.lp[i]);
  }
  mx = warp_max(mx);
  const bool none = mx == -INFINITY;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    a.lp[i] = none ? -INFINITY : (a.lp[i] - mx) * c;
    a.p[i] = exp2f(a.lp[i]);
    s += a.p[i];
  }
  s = warp_add(s);
  const float l = none ? 0.0f : log2f(s);
  const float inv = none ? 0.0f : 1.0f / s;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    a.lp[i] -= l;
    a.p[i] *= inv;
    if (none) a.id[i] = -1;  // nothing has any weight
  }
  return a;
}

struct DistillParams {
  const void* z;
  Teacher teacher;
  const int64_t* targets;  // may be null
  int64_t ld;
  int vocab, split;
  float c, inv_t;  // log2(e) / temperature, 1 / temperature
  float* kl;
  float* ce;
  float4* stats;  // m, log2 s at the temperature, log2 s at 1
};

// kTwo, kSquare: the targets' cross-entropy needs the row's sum at temperature
// 1 too.  Bound by reading the logits: 2046 x 128256 in 84 us with one sum, 85
// with squares, 118 with both exponentials, one call behind the other (behind a
// backward pass 100 to 114 with squares); 511 x 151936 in 37 us, 4.1 TB/s (511
// CTAs leave a seventh of 592 places empty; in halves they cost as much more).
template <typename T, Mode M>
__global__ void __launch_bounds__(kThreads, kPerSm) distill_fwd_kernel(const DistillParams p) {
  constexpr bool TWO = M != kPlain;
  constexpr int U = kInFlight;
  __shared__ Sums sums[kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t r = blockIdx.x / p.split;
  const int rank = static_cast<int>(blockIdx.x % p.split);
  const T* const z = static_cast<const T*>(p.z) + r * p.ld;
  const Row<T> row(z, p.vocab);
  const int per = (row.n + p.split - 1) / p.split;
  const int c0 = min(row.n, rank * per), c1 = min(row.n, c0 + per);
  const float c = p.c;
  // What is given, and the student's logits there, ahead of the row: loads one
  // behind the other at its end would hold up the CTA's last warp.
  __shared__ int ids[kMaxTop + 1];
  __shared__ float given[kMaxTop], picked[kMaxTop + 1];
  if (rank == 0 && threadIdx.x <= kMaxTop) {
    const int e = threadIdx.x, k = p.teacher.k;
    int64_t id = -1;
    if (e < k) id = p.teacher.id(r * k + e);
    if (e == kMaxTop && p.targets) id = p.targets[r];
    if (id < 0 || id >= p.vocab) id = -1;
    ids[e] = static_cast<int>(id);
    picked[e] = id >= 0 ? Elem<T>::load(z + id) : 0.0f;
    if (e < k) given[e] = p.teacher.logit(r * k + e);
  }
  Sums v;
  auto one = [&](const uint32_t (&w)[1][8]) {
    add_chunks<T, M, 1>(v, w, Elem<T>::value(Elem<T>::chunk_max(w[0])), c);
  };
  const int lo = max(c0, row.lo), hi = min(c1, row.hi);
  if (threadIdx.x == 0 && c0 == 0 && c1 > 0 && row.lo == 1) {
    uint32_t w[1][8];
    row.load_edge(0, w[0]);
    one(w);
  }
  if (threadIdx.x == kThreads - 1 && c1 == row.n && c0 < c1 && row.hi < row.n &&
      row.n - 1 >= row.lo) {
    uint32_t w[1][8];
    row.load_edge(row.n - 1, w[0]);
    one(w);
  }
  auto many = [&](int ch, auto part) {
    uint32_t w[U][8];
    ld_chunks<decltype(part)::value>(row, ch, hi, w);
    typename Elem<T>::Max all = Elem<T>::chunk_max(w[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) all = Elem<T>::join(all, Elem<T>::chunk_max(w[u]));
    add_chunks<T, M, U>(v, w, Elem<T>::value(all), c);
  };
  int ch = lo + threadIdx.x;
  for (; ch + (U - 1) * kThreads < hi; ch += U * kThreads) many(ch, std::false_type());
  if (ch + kThreads < hi) {
    many(ch, std::true_type());
  } else if (ch < hi) {
    uint32_t w[1][8];
    ld_chunk_once(row.chunk(ch), w[0]);
    one(w);
  }
  block_sums<M>(v, sums, c);
  if (p.split > 1) {
    cluster_sync();
    if (rank == 0 && threadIdx.x == 0) v = cluster_sums<M>(sums, p.split, c);
    cluster_sync();  // the leader has read every CTA's shared memory
    if (rank != 0) return;
    if (threadIdx.x == 0) sums[0] = v;
  }
  if (threadIdx.x >= 32) return;
  __syncwarp();
  v = sums[0];
  const bool none = v.m == -INFINITY;
  const float m = none ? 0.0f : v.m, l2 = log2f(v.s);
  // (A NaN in the row is in s; in a it may not be.)
  const float l21 = TWO && l2 == l2 ? log2f(v.a) : l2;
  const Alternatives a = weigh(
      p.teacher.k, p.vocab, c, [&](int e) { return ids[e]; }, [&](int e) { return given[e]; });
  float kl = 0.0f;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    if (a.id[i] < 0 || a.p[i] == 0.0f) continue;
    const float lq =
        none ? -INFINITY
             : fmaf(picked[(threadIdx.x & 31) + 32 * i] - m, p.inv_t, -l2 * kLn2);
    kl = fmaf(a.p[i], fmaf(a.lp[i], kLn2, -lq), kl);
  }
  kl = warp_add(kl);
  if (threadIdx.x != 0) return;
  p.kl[r] = kl;
  if (p.ce) {
    float ce = 0.0f;
    if (ids[kMaxTop] >= 0) ce = none ? INFINITY : fmaf(l21, kLn2, m - picked[kMaxTop]);
    p.ce[r] = ce;
  }
  if (p.stats) p.stats[r] = make_float4(m, l2, l21, 0.0f);
}

struct DistillGradParams {
  const void* z;
  Teacher teacher;
  const int64_t* targets;  // may be null
  const float4* stats;
  const float* dkl;
  const float* dce;
  void* dz;
  int64_t ld, ld_out;
  int vocab, parts;
  float c, inv_t;
};

// Every element first as if nothing were given (the two softmaxes alone); the
// few given ones are then written again by the CTA that wrote them, with what
// all their entries in the row take off (the same id may be given twice).
// 2046 x 128256 with 64 alternatives: 170 us, 6.2 TB/s.
template <typename T, bool SAME, Mode M>
__global__ void __launch_bounds__(kThreads) distill_bwd_kernel(const DistillGradParams p) {
  __shared__ int ids[kMaxTop + 1];
  __shared__ float off[kMaxTop + 1];
  griddep_wait();
  griddep_launch_dependents();
  // Last row first: the forward's last rows may still be in L2.
  const int64_t r = gridDim.x / p.parts - 1 - blockIdx.x / p.parts;
  const int part = static_cast<int>(blockIdx.x % p.parts);
  const T* const z = static_cast<const T*>(p.z) + r * p.ld;
  T* const dz = static_cast<T*>(p.dz) + r * p.ld_out;
  const int k = p.teacher.k;
  float m, ca, cb;
  bool zero;
  auto soft = [&](float f) {
    if (zero) return 0.0f;
    const float d = f - m;
    const float e = ex2_approx(d * p.c);
    if (M == kSquare) return e * fmaf(cb, e, ca);
    if (M == kTwo) return fmaf(cb, ex2_approx(d * kLog2e), ca * e);
    return ca * e;
  };
  int mine;
  float zi;
  auto ready = [&] {
    const float4 st = p.stats[r];
    const int64_t target = p.targets ? p.targets[r] : -1;
    const bool picked = target >= 0 && target < p.vocab;
    const float u = p.dkl ? p.dkl[r] * p.inv_t : 0.0f;
    const float v = picked && p.dce ? p.dce[r] : 0.0f;
    bool any = false;
    if (threadIdx.x < 32) {
      const Alternatives a =
          weigh(k, p.vocab, p.c, [&](int e) { return p.teacher.id(r * k + e); },
                [&](int e) { return p.teacher.logit(r * k + e); });
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int e = threadIdx.x + 32 * i;
        if (e < k) {
          ids[e] = a.id[i];
          off[e] = a.id[i] < 0 ? 0.0f : u * a.p[i];
          any |= a.id[i] >= 0;
        }
      }
      if (threadIdx.x == 0) {
        ids[k] = picked ? static_cast<int>(target) : -1;
        off[k] = v;
      }
    }
    // Whether anything of the teacher's is given; also orders ids and off.
    const float us = __syncthreads_or(any) ? u : 0.0f;
    // A row that no gradient reaches gets zeros whatever it holds, and so does
    // one without a distribution, at its given ids and its target too.
    m = st.x;
    zero = (us == 0.0f && v == 0.0f) || st.y == -INFINITY;
    ca = us * exp2f(-st.y);
    cb = v * exp2f(-st.z);
    if (M == kPlain) ca += cb;
    // The given elements' logits, before anything is written over them.
    mine = static_cast<int>(threadIdx.x) <= k ? ids[threadIdx.x] : -1;
    zi = mine >= 0 ? Elem<T>::load(z + mine) : 0.0f;
    __syncthreads();
  };
  row_gradient<T, SAME>(z, dz, p.vocab, part, p.parts, ready, [&](int64_t, auto& f) {
    constexpr int N = sizeof(f) / sizeof(float);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = soft(f[e]);
  });
  __syncthreads();
  if (mine < 0 || zero) return;
  const Row<T> row(z, p.vocab);
  const int per = (row.n + p.parts - 1) / p.parts;
  const int c = (mine + row.off) / Elem<T>::CH;
  if (c / per != part) return;
  float take = 0.0f;
  for (int e = 0; e <= k; ++e)
    if (ids[e] == mine) take += off[e];
  Elem<T>::store(dz + mine, soft(zi) - take);
}

// -------------------------------------------------------------------- host --

int elem_bytes(int dtype) { return dtype == TQ_DTYPE_F32 ? 4 : 2; }

int check_rows(const char* who, const void* z, int dtype, int64_t rows, int64_t vocab, int64_t ld,
               float temperature) {
  if (dtype != TQ_DTYPE_F32 && dtype != TQ_DTYPE_BF16)
    return fail(TQ_ERR_UNSUPPORTED, "%s: logits must be f32 or bf16 (dtype %d)", who, dtype);
  if (rows < 0 || vocab <= 0 || ld < vocab)
    return fail(TQ_ERR_INVALID,
                "%s: need rows >= 0, vocab > 0 and ld >= vocab (got %lld, %lld, %lld)", who,
                (long long)rows, (long long)vocab, (long long)ld);
  if (vocab > (1ll << 31) - 64 || rows > (1ll << 27))
    return fail(TQ_ERR_INVALID, "%s: at most 2^31 - 64 logits a row and 2^27 rows", who);
  if (!(temperature > 0.0f) || !std::isfinite(temperature) ||
      !std::isfinite(kLog2e / temperature))
    return fail(TQ_ERR_INVALID, "%s: temperature must be positive and finite", who);
  if (rows > 0 && !z) return fail(TQ_ERR_INVALID, "%s: null pointer", who);
  if (!aligned(z, elem_bytes(dtype)))
    return fail(TQ_ERR_MISALIGNED, "%s: logits must be aligned to their type", who);
  return TQ_OK;
}

// Forward: how many CTAs (a cluster of a power of two) share a row: enough that
// the grid has one for each of 1.5 SMs, none with less than 512 chunks.  What a
// CTA costs beside its chunks (the joins, the selection) is not split: 148 x
// 151936 takes 20.5 us with one CTA a row, 16.5 with two, 22.5 with four; 257 x
// 96259 f32 22.6, 24.4 and 26.6; 511 x 151936 with 20 alternatives 43, 51 and
// 70; 67 x 128256 with 5 22.6, 20.5 and 18.5.
int split_for(int64_t rows, int64_t vocab, int ch) {
  const int64_t want = 3ll * sm_count() / 2;
  int s = 1;
  while (s < kMaxSplit && rows * s < want && vocab / (2 * s) >= 512ll * ch) s *= 2;
  return s;
}

// Backward: how many CTAs write a row.  As many as leave each `least` chunks
// (short CTAs close together in memory, and a short last wave: 2046 x 128256 by
// one CTA a row 177 us, two 168, four 164, eight 160), and down to 512 where
// the grid would not offer every SM several.
int parts_for(int64_t rows, int64_t vocab, int ch, int least) {
  const int64_t chunks = vocab / ch, want = 4ll * sm_count();
  int s = 1;
  while (s < 16 && chunks >= 2ll * s * (rows * s < want ? 512 : least)) s *= 2;
  return s;
}

// What a CTA of a backward kernel reads before its chunks can be finished is
// hidden behind about so many of them: a few numbers, or the alternatives and
// their softmax (four CTAs a row of 2046 x 128256 170 us, one 188, eight 189).
// What the two give elsewhere, with one, two, four and eight CTAs a row and by
// the rule, us: log probabilities 47, 47, 45, 57 and 45 at 2046 x 32000, 92, 88,
// 86, 83 and 86 at 2046 x 65536, 207, 203, 196, 191 and 191 at 2046 x 151936, 90,
// 88, 86, 84 and 86 at 2046 x 32003 f32; distillation 55, 57, 72, 107 and 55, 100,
// 96, 102, 127 and 96, 219, 209, 201, 219 and 201, and 98, 92, 96, 119 and 92.
constexpr int kLeastLogprobs = 900;
constexpr int kLeastDistill = 1800;

// Whether z's and dz's rows all start at the same offset in a 32-byte chunk.
bool same_offset(const void* z, const void* dz, int64_t rows, int64_t ld, int64_t ld_out,
                 int bytes) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(z), b = reinterpret_cast<uintptr_t>(dz);
  return ((a ^ b) & 31u) == 0 && (rows == 1 || ((ld - ld_out) * bytes) % 32 == 0);
}

}  // namespace
}  // namespace tq

extern "C" int tq_token_logprobs_fwd(const void* logits, int dtype, const int64_t* tokens,
                                     int64_t rows, int64_t vocab, int64_t ld, float temperature,
                                     int64_t top, float* logprobs, float* entropy, float* stats,
                                     float* top_logprobs, int64_t* top_ids, void* stream) {
  using namespace tq;
  const char* who = "token_logprobs";
  int rc = check_rows(who, logits, dtype, rows, vocab, ld, temperature);
  if (rc) return rc;
  const int ch = 32 / elem_bytes(dtype);
  if (top < 0 || top > kMaxTop || top > vocab)
    return fail(TQ_ERR_INVALID, "%s: top (%lld) must be 0 to %d and at most vocab", who,
                (long long)top, kMaxTop);
  if (top > 0 && vocab / ch + 2 > static_cast<int64_t>(kMaxSplit) * kMaxChunks)
    return fail(TQ_ERR_INVALID, "%s: top alternatives need a vocab of at most %lld", who,
                (long long)(static_cast<int64_t>(kMaxSplit) * kMaxChunks - 2) * ch);
  if (rows == 0) return TQ_OK;
  if (!tokens || !logprobs || !entropy || (top > 0 && (!top_logprobs || !top_ids)))
    return fail(TQ_ERR_INVALID, "%s: null pointer", who);
  if (!aligned(tokens, 8) || !aligned(logprobs, 4) || !aligned(entropy, 4) ||
      !aligned(stats, 16) || !aligned(top_logprobs, 4) || !aligned(top_ids, 8))
    return fail(TQ_ERR_MISALIGNED, "%s: a pointer is not aligned to its type (stats: 16 bytes)",
                who);
  LogprobParams p{};
  p.z = logits;
  p.tokens = tokens;
  p.ld = ld;
  p.vocab = static_cast<int>(vocab);
  p.split = split_for(rows, vocab, ch);
  p.top = static_cast<int>(top);
  p.c = kLog2e / temperature;
  p.inv_t = 1.0f / temperature;
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.stats = reinterpret_cast<float4*>(stats);
  p.top_logprobs = top_logprobs;
  p.top_ids = top_ids;
  size_t smem = 0;
  if (top > 0) {
    while ((vocab / ch + 2 + p.split - 1) / p.split > kMaxChunks) p.split *= 2;
    const size_t key = dtype == TQ_DTYPE_F32 ? 4 : 2;
    const size_t keys = static_cast<size_t>((vocab / ch + 2 + p.split - 1) / p.split) * key;
    const size_t room = static_cast<size_t>(kPool) * 8;
    smem = ((keys > room ? keys : room) + 15) / 16 * 16;
  }
  auto kernel = dtype == TQ_DTYPE_F32
                    ? (top > 0 ? logprobs_fwd_kernel<float, true> : logprobs_fwd_kernel<float, false>)
                    : (top > 0 ? logprobs_fwd_kernel<uint16_t, true>
                               : logprobs_fwd_kernel<uint16_t, false>);
  if (top > 0) {
    // The most any call asks for, so that one attribute call serves all.
    rc = set_max_smem_once(reinterpret_cast<const void*>(kernel), kMaxChunks * 4 + 1024,
                           "cudaFuncSetAttribute(token_logprobs)");
    if (rc) return rc;
  }
  return launch_kernel(kernel, dim3(static_cast<unsigned>(rows * p.split)), dim3(kThreads), smem,
                       as_stream(stream), dim3(p.split), "token_logprobs forward launch", p);
}

extern "C" int tq_token_logprobs_bwd(const void* logits, int dtype, const int64_t* tokens,
                                     const float* stats, int64_t rows, int64_t vocab, int64_t ld,
                                     float temperature, const float* dlogprobs,
                                     const float* dentropy, void* dlogits, int64_t ld_out,
                                     void* stream) {
  using namespace tq;
  const char* who = "token_logprobs backward";
  int rc = check_rows(who, logits, dtype, rows, vocab, ld, temperature);
  if (rc) return rc;
  if (ld_out < vocab) return fail(TQ_ERR_INVALID, "%s: ld_out must be at least vocab", who);
  if (rows == 0) return TQ_OK;
  if (!tokens || !stats || !dlogits) return fail(TQ_ERR_INVALID, "%s: null pointer", who);
  if (dlogits == logits && ld_out != ld)
    return fail(TQ_ERR_INVALID, "%s: in place, ld_out must be ld", who);
  if (!aligned(tokens, 8) || !aligned(stats, 16) || !aligned(dlogprobs, 4) ||
      !aligned(dentropy, 4) || !aligned(dlogits, elem_bytes(dtype)))
    return fail(TQ_ERR_MISALIGNED, "%s: a pointer is not aligned to its type (stats: 16 bytes)",
                who);
  LogprobGradParams p{};
  p.z = logits;
  p.tokens = tokens;
  p.stats = reinterpret_cast<const float4*>(stats);
  p.dlogprobs = dlogprobs;
  p.dentropy = dentropy;
  p.dz = dlogits;
  p.ld = ld;
  p.ld_out = ld_out;
  p.vocab = static_cast<int>(vocab);
  p.parts = parts_for(rows, vocab, 32 / elem_bytes(dtype), kLeastLogprobs);
  p.c = kLog2e / temperature;
  p.inv_t = 1.0f / temperature;
  const bool same = same_offset(logits, dlogits, rows, ld, ld_out, elem_bytes(dtype));
  auto kernel = dtype == TQ_DTYPE_F32
                    ? (same ? logprobs_bwd_kernel<float, true> : logprobs_bwd_kernel<float, false>)
                    : (same ? logprobs_bwd_kernel<uint16_t, true>
                            : logprobs_bwd_kernel<uint16_t, false>);
  return launch_kernel(kernel, dim3(static_cast<unsigned>(rows * p.parts)), dim3(kThreads), 0,
                       as_stream(stream), 1, "token_logprobs backward launch", p);
}

namespace tq {
namespace {

// Which sums a call needs: the temperature's alone (0), those at temperature 1
// beside them (1), or as their squares (2).
int which_sums(bool targets, float temperature) {
  return !targets || temperature == 1.0f ? 0 : temperature == 2.0f ? 2 : 1;
}

int check_teacher(const char* who, const void* ids, int ids_bits, const void* logits,
                  int logits_dtype, int64_t k, int64_t rows, Teacher* t) {
  if (k < 1 || k > kMaxTop)
    return fail(TQ_ERR_INVALID, "%s: 1 to %d teacher alternatives a row, got %lld", who, kMaxTop,
                (long long)k);
  if (ids_bits != 32 && ids_bits != 64)
    return fail(TQ_ERR_UNSUPPORTED, "%s: teacher ids must be 32- or 64-bit integers", who);
  if (logits_dtype != TQ_DTYPE_F32 && logits_dtype != TQ_DTYPE_BF16)
    return fail(TQ_ERR_UNSUPPORTED, "%s: teacher logits must be f32 or bf16 (dtype %d)", who,
                logits_dtype);
  if (rows > 0 && (!ids || !logits)) return fail(TQ_ERR_INVALID, "%s: null pointer", who);
  if (!aligned(ids, ids_bits / 8) || !aligned(logits, elem_bytes(logits_dtype)))
    return fail(TQ_ERR_MISALIGNED, "%s: a teacher pointer is not aligned to its type", who);
  t->ids = ids;
  t->logits = logits;
  t->ids64 = ids_bits == 64;
  t->logits_bf16 = logits_dtype == TQ_DTYPE_BF16;
  t->k = static_cast<int>(k);
  return TQ_OK;
}

}  // namespace
}  // namespace tq

extern "C" int tq_distill_fwd(const void* logits, int dtype, const void* teacher_ids, int ids_bits,
                              const void* teacher_logits, int teacher_dtype, int64_t k,
                              const int64_t* targets, int64_t rows, int64_t vocab, int64_t ld,
                              float temperature, float* kl, float* ce, float* stats,
                              void* stream) {
  using namespace tq;
  const char* who = "distillation";
  int rc = check_rows(who, logits, dtype, rows, vocab, ld, temperature);
  if (rc) return rc;
  DistillParams p{};
  rc = check_teacher(who, teacher_ids, ids_bits, teacher_logits, teacher_dtype, k, rows,
                     &p.teacher);
  if (rc) return rc;
  if (rows == 0) return TQ_OK;
  if (!kl || (targets != nullptr) != (ce != nullptr))
    return fail(TQ_ERR_INVALID, "%s: null kl, or targets without ce (they go together)", who);
  if (!aligned(targets, 8) || !aligned(kl, 4) || !aligned(ce, 4) || !aligned(stats, 16))
    return fail(TQ_ERR_MISALIGNED, "%s: a pointer is not aligned to its type (stats: 16 bytes)",
                who);
  p.z = logits;
  p.targets = targets;
  p.ld = ld;
  p.vocab = static_cast<int>(vocab);
  p.split = split_for(rows, vocab, 32 / elem_bytes(dtype));
  p.c = kLog2e / temperature;
  p.inv_t = 1.0f / temperature;
  p.kl = kl;
  p.ce = ce;
  p.stats = reinterpret_cast<float4*>(stats);
  using Kernel = void (*)(const DistillParams);
  const Kernel f32[3] = {distill_fwd_kernel<float, kPlain>, distill_fwd_kernel<float, kTwo>,
                         distill_fwd_kernel<float, kSquare>};
  const Kernel bf16[3] = {distill_fwd_kernel<uint16_t, kPlain>,
                          distill_fwd_kernel<uint16_t, kTwo>,
                          distill_fwd_kernel<uint16_t, kSquare>};
  const Kernel kernel =
      (dtype == TQ_DTYPE_F32 ? f32 : bf16)[which_sums(targets != nullptr, temperature)];
  return launch_kernel(kernel, dim3(static_cast<unsigned>(rows * p.split)), dim3(kThreads), 0,
                       as_stream(stream), dim3(p.split), "distillation forward launch", p);
}

extern "C" int tq_distill_bwd(const void* logits, int dtype, const void* teacher_ids, int ids_bits,
                              const void* teacher_logits, int teacher_dtype, int64_t k,
                              const int64_t* targets, const float* stats, int64_t rows,
                              int64_t vocab, int64_t ld, float temperature, const float* dkl,
                              const float* dce, void* dlogits, int64_t ld_out, void* stream) {
  using namespace tq;
  const char* who = "distillation backward";
  int rc = check_rows(who, logits, dtype, rows, vocab, ld, temperature);
  if (rc) return rc;
  DistillGradParams p{};
  rc = check_teacher(who, teacher_ids, ids_bits, teacher_logits, teacher_dtype, k, rows,
                     &p.teacher);
  if (rc) return rc;
  if (ld_out < vocab) return fail(TQ_ERR_INVALID, "%s: ld_out must be at least vocab", who);
  if (rows == 0) return TQ_OK;
  if (!stats || !dlogits || (dce && !targets))
    return fail(TQ_ERR_INVALID, "%s: null pointer, or dce without targets", who);
  if (dlogits == logits && ld_out != ld)
    return fail(TQ_ERR_INVALID, "%s: in place, ld_out must be ld", who);
  if (!aligned(targets, 8) || !aligned(stats, 16) || !aligned(dkl, 4) || !aligned(dce, 4) ||
      !aligned(dlogits, elem_bytes(dtype)))
    return fail(TQ_ERR_MISALIGNED, "%s: a pointer is not aligned to its type (stats: 16 bytes)",
                who);
  p.z = logits;
  p.targets = targets;
  p.stats = reinterpret_cast<const float4*>(stats);
  p.dkl = dkl;
  p.dce = dce;
  p.dz = dlogits;
  p.ld = ld;
  p.ld_out = ld_out;
  p.vocab = static_cast<int>(vocab);
  p.parts = parts_for(rows, vocab, 32 / elem_bytes(dtype), kLeastDistill);
  p.c = kLog2e / temperature;
  p.inv_t = 1.0f / temperature;
  const bool same = same_offset(logits, dlogits, rows, ld, ld_out, elem_bytes(dtype));
  using Kernel = void (*)(const DistillGradParams);
  const Kernel f32[2][3] = {
      {distill_bwd_kernel<float, false, kPlain>, distill_bwd_kernel<float, false, kTwo>,
       distill_bwd_kernel<float, false, kSquare>},
      {distill_bwd_kernel<float, true, kPlain>, distill_bwd_kernel<float, true, kTwo>,
       distill_bwd_kernel<float, true, kSquare>}};
  const Kernel bf16[2][3] = {
      {distill_bwd_kernel<uint16_t, false, kPlain>, distill_bwd_kernel<uint16_t, false, kTwo>,
       distill_bwd_kernel<uint16_t, false, kSquare>},
      {distill_bwd_kernel<uint16_t, true, kPlain>, distill_bwd_kernel<uint16_t, true, kTwo>,
       distill_bwd_kernel<uint16_t, true, kSquare>}};
  const Kernel kernel =
      (dtype == TQ_DTYPE_F32 ? f32 : bf16)[same][which_sums(dce != nullptr, temperature)];
  return launch_kernel(kernel, dim3(static_cast<unsigned>(rows * p.parts)), dim3(kThreads), 0,
                       as_stream(stream), 1, "distillation backward launch", p);
}
