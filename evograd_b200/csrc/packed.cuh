// Work plan of a packed batch (documents of different lengths in one token axis)
// and what the packed attention kernels share.
//
// The plan lives in device memory and is built on the device from the sequence
// offsets, so no length ever has to reach the host: a batch can change under a
// captured graph. Layout (32-bit words):
//   header [kPlanHeader]  status, valid tokens, items in use, tokens, item slots
//   items  [slots][4]     {first token of the sequence, its length, weight w, first
//                          padded tile of the sequence}
//   scratch               histogram and prefix sums of the builder
// A sequence of n = ceil(length / 128) tiles has the items w = n .. 1; items are
// sorted by falling w over the whole batch, so a kernel that walks them in order
// starts its heaviest blocks first: the forward's item w is query tile w - 1 (w key
// tiles to visit), the backward's is key tile n - w (w query tiles to visit).
// Tokens behind the last sequence form items with w = 0 (length = rows to clear);
// unused slots have w = -1. Per-row statistics of the backward are padded to whole
// tiles per sequence: row r of tile t of a sequence is padded row
// (first padded tile + t) * 128 + r.
#pragma once

#include "attention_common.cuh"

namespace evg {
namespace packed {

constexpr int kPlanHeader = 16;  // 32-bit words; keeps the items 16-byte aligned
enum PlanWord { kStatus = 0, kValidTokens = 1, kItemsUsed = 2, kTokens = 3, kSlots = 4 };

// Items a batch can need: every non-empty sequence and the tokens behind the last
// one round up to whole tiles.
inline int64_t plan_slots(int64_t tokens, int64_t sequences) {
  const int64_t parts = (sequences < tokens ? sequences : tokens) + 1;
  return (tokens + (attn::kTile - 1) * parts) / attn::kTile;
}
// Most tiles one sequence can have.
inline int64_t plan_max_weight(int64_t tokens) { return (tokens + attn::kTile - 1) / attn::kTile; }

inline int64_t plan_words(int64_t tokens, int64_t sequences) {
  return kPlanHeader + 4 * plan_slots(tokens, sequences) + 2 * (plan_max_weight(tokens) + 2) + sequences;
}

// One tensor [tokens, heads, D] with its strides in elements; the last dimension is
// contiguous.
struct View {
  void* p = nullptr;
  int64_t st = 0, sh = 0;
};

// TMA map of a 16-bit View with coordinates (column, token, head) and [128 x 64]
// tiles, 128-byte swizzle. Columns behind D read as zero, so any head size that is a
// multiple of eight runs in the kernels for 64 or 128.
bool encode_view_map(CUtensorMap* map, const View& v, int fmt, int64_t D, int64_t tokens,
                     int64_t heads);

#ifdef __CUDACC__
__device__ __forceinline__ int4 plan_item(const int* plan, int i) {
  return reinterpret_cast<const int4*>(plan + kPlanHeader)[i];
}

// Zeroes rows [first, 128) of a tile in shared memory (one warp). The rows behind a
// sequence's end belong to the next sequence or to nobody: a product takes them with
// weight zero, which is not enough when they hold an infinity or a NaN.
template <int HD>
__device__ __forceinline__ void clear_tile_rows(uint8_t* tile, int first, int lane) {
#pragma unroll
  for (int a = 0; a < HD / 64; ++a) {
    uint4* base = reinterpret_cast<uint4*>(tile + a * (attn::kTile * 128) + first * 128);
    const int n = (attn::kTile - first) * 8;
    for (int i = lane; i < n; i += 32) base[i] = make_uint4(0, 0, 0, 0);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}
#endif

}  // namespace packed
}  // namespace evg
