// Builder of the packed batch's work plan (packed.cuh): one block, a counting sort
// of the sequences by their number of 128-token tiles, then one warp per sequence
// writes its items. Latency-bound: a handful of dependent passes over the offsets
// (16 sequences, 16384 tokens: a few microseconds, once per batch).
#include <mutex>

#include "packed.cuh"

namespace evg {
namespace packed {

bool encode_view_map(CUtensorMap* map, const View& v, int fmt, int64_t D, int64_t tokens,
                     int64_t heads) {
  using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeFn encode = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres) ==
            cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      encode = (EncodeFn)fn;
  });
  if (!encode) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)tokens, (cuuint64_t)heads};
  // the stride of an axis of length one is never used; give it a legal value
  const cuuint64_t row = (cuuint64_t)((D + 7) / 8 * 16);
  const cuuint64_t strides[2] = {tokens > 1 ? (cuuint64_t)v.st * 2 : row,
                                 heads > 1 ? (cuuint64_t)v.sh * 2 : row};
  const cuuint32_t box[3] = {64, attn::kTile, 1};
  const cuuint32_t elem_strides[3] = {1, 1, 1};
  return encode(map, fmt == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                3, v.p, dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kSharedWeights = 4096;  // tables in shared memory up to half a million tokens

// Exclusive prefix sum over the block; `total` is the sum (same in all threads).
__device__ int block_exclusive_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, s, off);
    if (lane >= off) s += t;
  }
  __syncthreads();  // the previous call's readers are done
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += t;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  total = warp_sums[31];
  return s - v + (warp ? warp_sums[warp - 1] : 0);
}

__global__ void __launch_bounds__(kPlanThreads)
packed_plan_kernel(const int* __restrict__ cu, int n_seq, int tokens, int slots, int max_w,
                   int* __restrict__ plan) {
  __shared__ int warp_sums[32];
  __shared__ int s_valid;
  __shared__ int tables[2 * kSharedWeights];
  int4* items = reinterpret_cast<int4*>(plan + kPlanHeader);
  int* scratch = plan + kPlanHeader + 4 * slots;
  const bool small = max_w + 2 <= kSharedWeights;
  int* at_least = small ? tables : scratch;  // [max_w + 2] sequences with >= w tiles
  int* item0 = at_least + max_w + 2;         // [max_w + 2] first item of weight w
  int* rank = scratch + 2 * (max_w + 2);     // [n_seq] place among the sequences of equally many tiles
  const int tid = threadIdx.x;

  // Offsets must start at 0, never fall and end inside the token axis; anything else
  // makes the whole batch "behind the last sequence" and is reported in the status.
  bool bad = false;
  for (int i = tid; i <= n_seq; i += kPlanThreads) {
    const int c = cu[i];
    bad = bad || c < 0 || c > tokens || (i == 0 && c != 0) || (i < n_seq && cu[i + 1] < c);
  }
  for (int i = tid; i < max_w + 2; i += kPlanThreads) at_least[i] = 0;
  const bool ok = !__syncthreads_or(bad);
  if (tid == 0) s_valid = ok ? cu[n_seq] : 0;
  const int n = ok ? n_seq : 0;
  // histogram of tile counts; a sequence's place inside its bin
  for (int i = tid; i < n; i += kPlanThreads) {
    const int tiles = (cu[i + 1] - cu[i] + attn::kTile - 1) / attn::kTile;
    rank[i] = atomicAdd(at_least + tiles, 1);
  }
  __syncthreads();
  const int valid = s_valid;
  // Suffix sums over w = max_w .. 1 in chunks: at_least[w] = sequences with >= w tiles,
  // item0[w] = items of larger weight.
  int carry_seq = 0, carry_item = 0;
  for (int base = 0; base < max_w; base += kPlanThreads) {
    const int w = max_w - base - tid;
    int total;
    const int h = w >= 1 ? at_least[w] : 0;
    const int c = carry_seq + block_exclusive_scan(h, warp_sums, total) + h;
    carry_seq += total;
    const int mine = w >= 1 ? c : 0;
    const int before = carry_item + block_exclusive_scan(mine, warp_sums, total);
    carry_item += total;
    if (w >= 1) {
      at_least[w] = c;
      item0[w] = before;
    }
  }
  if (tid == 0) at_least[max_w + 1] = 0;
  __syncthreads();
  const int used = carry_item;
  // items: one warp per sequence; padded tiles are numbered in sequence order
  int carry_tile = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + tid;
    const int start = i < n ? cu[i] : 0;
    const int len = i < n ? cu[i + 1] - start : 0;
    const int tiles = (len + attn::kTile - 1) / attn::kTile;
    int total;
    const int tile0 = carry_tile + block_exclusive_scan(tiles, warp_sums, total);
    carry_tile += total;
    const int place = tiles > 0 ? at_least[tiles + 1] + rank[i] : 0;
    // every lane's sequence in turn, 32 items at a time
    unsigned todo = __ballot_sync(0xffffffffu, tiles > 0);
    while (todo) {
      const int src = __ffs(todo) - 1;
      todo &= todo - 1;
      const int s_start = __shfl_sync(0xffffffffu, start, src);
      const int s_len = __shfl_sync(0xffffffffu, len, src);
      const int s_tiles = __shfl_sync(0xffffffffu, tiles, src);
      const int s_tile0 = __shfl_sync(0xffffffffu, tile0, src);
      const int s_place = __shfl_sync(0xffffffffu, place, src);
      for (int w = 1 + (tid & 31); w <= s_tiles; w += 32)
        items[item0[w] + s_place] = make_int4(s_start, s_len, w, s_tile0);
    }
  }
  // rows behind the last sequence, then the unused slots
  const int tail_tiles = (tokens - valid + attn::kTile - 1) / attn::kTile;
  for (int i = tid; i < slots - used; i += kPlanThreads) {
    const int row = valid + i * attn::kTile;
    const bool tail = i < tail_tiles;
    items[used + i] = tail ? make_int4(row, min(attn::kTile, tokens - row), 0, 0)
                           : make_int4(0, 0, -1, 0);
  }
  if (tid == 0) {
    plan[kStatus] = ok ? EVG_OK : EVG_EBADSHAPE;
    plan[kValidTokens] = valid;
    plan[kItemsUsed] = used;
    plan[kTokens] = tokens;
    plan[kSlots] = slots;
  }
}

}  // namespace
}  // namespace packed
}  // namespace evg

using namespace evg;

extern "C" int64_t evg_packed_plan_bytes(int64_t tokens, int64_t sequences) {
  if (tokens < 0 || sequences < 0 || tokens > EVG_PACKED_MAX_TOKENS || sequences > EVG_PACKED_MAX_TOKENS)
    return 0;
  return packed::plan_words(tokens, sequences) * 4;
}

extern "C" int evg_packed_plan(const int32_t* cu_seqlens, int64_t sequences, int64_t tokens,
                               void* plan, int64_t plan_bytes, void* stream) {
  if (!cu_seqlens || !plan) return fail(EVG_ENULL, "packed_plan: null pointer argument");
  if (tokens < 0 || sequences < 0 || tokens > EVG_PACKED_MAX_TOKENS || sequences > EVG_PACKED_MAX_TOKENS)
    return fail(EVG_EBADSHAPE, "packed_plan: tokens=%lld sequences=%lld (0 .. %d each)",
                (long long)tokens, (long long)sequences, EVG_PACKED_MAX_TOKENS);
  if (!aligned16(plan)) return fail(EVG_EALIGN, "packed_plan: the plan must be 16-byte aligned");
  const int64_t need = evg_packed_plan_bytes(tokens, sequences);
  if (plan_bytes < need)
    return fail(EVG_EWORKSPACE, "packed_plan: plan of %lld bytes, need %lld", (long long)plan_bytes,
                (long long)need);
  packed::packed_plan_kernel<<<1, packed::kPlanThreads, 0, (cudaStream_t)stream>>>(
      cu_seqlens, (int)sequences, (int)tokens, (int)packed::plan_slots(tokens, sequences),
      (int)packed::plan_max_weight(tokens), (int*)plan);
  return check_launch("packed_plan");
}
