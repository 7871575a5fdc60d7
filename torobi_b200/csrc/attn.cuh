// What the two attention files share: tile sizes, the shape check and the tensor
// map of [batch, seq, heads, dim].
#pragma once

#include "tq_ptx.cuh"
#include "tq_runtime.h"

namespace tq {

constexpr int kTile = 128;  // query rows and key rows per tile
constexpr int kHalf = 64;   // the streamed tile of the backward kernels
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// [batch, seq, heads, dim] bf16 as a 4D tensor map, one 64-wide dim slab x
// `rows` positions of `pack` heads per box (128-byte swizzle).
inline int map_bshd(CUtensorMap* map, const void* ptr, int64_t batch, int64_t seq, int64_t heads,
                    int64_t dim, uint32_t rows = kTile, uint32_t pack = 1) {
  const uint64_t dims[4] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(heads),
                            static_cast<uint64_t>(seq), static_cast<uint64_t>(batch)};
  const uint64_t strides[3] = {static_cast<uint64_t>(dim) * 2,
                               static_cast<uint64_t>(heads * dim) * 2,
                               static_cast<uint64_t>(seq * heads * dim) * 2};
  const uint32_t box[4] = {64, pack, rows, 1};
  return encode_tmap(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, ptr, dims, strides, box,
                     CU_TENSOR_MAP_SWIZZLE_128B);
}

inline int check_shape(int64_t batch, int64_t seq, int64_t heads, int64_t kv_heads, int64_t dim) {
  if (batch < 0 || seq < 0 || heads <= 0 || kv_heads <= 0)
    return fail(TQ_ERR_INVALID, "attention: batch and seq must be >= 0, heads and kv_heads > 0");
  if (heads % kv_heads != 0)
    return fail(TQ_ERR_INVALID, "attention: heads (%lld) must be a multiple of kv_heads (%lld)",
                (long long)heads, (long long)kv_heads);
  if (dim != 64 && dim != 128)
    return fail(TQ_ERR_UNSUPPORTED, "attention: head dim must be 64 or 128, got %lld",
                (long long)dim);
  const int64_t tiles = (seq + kTile - 1) / kTile;
  if (seq > (1ll << 30) || batch * heads * tiles > (1ll << 31) - 1 ||
      batch * seq * heads * dim > (1ll << 40))
    return fail(TQ_ERR_INVALID, "attention: shape too large");
  return TQ_OK;
}

}  // namespace tq
