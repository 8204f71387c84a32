// Causal grouped-query attention over a packed batch, backward (sm_100a).
//
//   P = exp(scale q k^T - lse), delta_i = do_i . o_i, dS = P * (do v^T - delta),
//   dv = P^T do, dk = scale dS^T q, dq = scale dS k
//
// One pass over the visible tiles, five products per (key tile, query tile). A block
// owns one key tile of one k/v head and walks the query tiles behind it, for every
// query head of the group. A tile's two halves of 64 queries are two streams:
//   S^T   = K Q^T,  dP^T = V dO^T   [128 keys x 64 queries], A from tensor memory
//   P^T, dS^T in registers, then 16 bits back into tensor memory over dP^T (the products'
//   operand type: with delta from the rounded o it takes the relative error of bf16 dq and dk
//   from 0.0017, their own last rounding, to 0.0025; a second operand with the remainder
//   would double the dK and dQ products)
//   dV   += P^T dO,  dK += dS^T Q   (A from tensor memory)
//   dQ^T  = K^T dS^T                [128 head columns x 64 queries], A the K tile in shared
// Each stream has eight compute warps of its own, so one stream's exponentials and dS run
// under the other stream's products. dK and dV stay in tensor memory until the end (fixed
// order, no atomics). dQ^T also belongs to other blocks' rows: four warps of their own send
// it to a float32 copy of dQ by asynchronous bulk reductions, so dq can differ in the last
// bit from run to run; a last kernel scales and rounds the copy. Only one block contributes
// to a sequence's first query tile: it rounds and writes those rows at once (32/8 heads of
// 128, 16384 tokens: sequences of 128 tokens 367 -> 208 us, of 512 473 -> 433, of 1024
// 584 -> 564).
//
// K and V are kept in tensor memory as well (HD / 2 columns each): a product of two
// shared-memory operands with 64 columns needs 192 bytes a clock of the shared memory's
// 128 (50 cycles measured, 35 with A in tensor memory), and with both scores and dP^T formed
// that way the operand reads, not the tensor pipe, set the time (416 KB per tile pair
// against 320 KB now, head size 128).
//
// Head size 128: a stream's S^T, dP^T, P^T / dS^T and dQ^T follow one another in the same 64
// columns of tensor memory. Order of the products for tile c (in brackets the stream):
//   S(c)[0]  dV,dK(c-1)[1]  dP(c)[0]  dQ(c-1)[1]  S(c)[1]  dV,dK(c)[0]  dP(c)[1]  dQ(c)[0]
// The tensor pipe runs in order; the streams are half a tile apart, so what one of them
// waits for runs behind the other's products.
// Tensor memory: streams [0,64) and [64,128), K [128,192), V [192,256), dV [256,384),
// dK [384,512). Shared memory: K, two dO and two Q stages, two 16 KB dS^T halves, row
// statistics, 32 KB of dQ on its way out (226 KB). What the rest costs: without the bulk
// reductions 16384 tokens in sequences of 4096 take 14 % less time, with a quarter of the
// dV and dK products 8 % less, with an eighth of the dQ products 10 % less.
//
// Head size 64 leaves room for more: scores, dP^T and the streams' common dQ^T have columns
// of their own, three stages of Q and dO, and a stream's next S^T and dP^T are formed behind
// its dV and dK of this tile; per half tile
//   S(c+1)[b]  dV,dK(c)[b]  dP(c+1)[b]  dQ(c)[b]
// (16/16 heads, 16384 tokens in sequences of 4096: 600 -> 542 us with one 16 KB piece of dQ
// per half; what is left is spread over the dQ warps' turns, 12 %, and waits: no single part
// taken out brings more than 4 %). Leaving out stream 1 where a last query tile has at most 64
// rows cost more registers than it saved work (64-token sequences 177 -> 165 us, 512-token
// ones 433 -> 449).
// Tensor memory: S^T [0,128), dP^T [128,256), K [256,288), V [288,320), dV [320,384),
// dK [384,448), dQ^T [448,512). The dQ^T product keeps its 128 rows: the A operand's second
// 64 columns are whatever follows K in shared memory, and the rows they give are not read
// (a 64-row product has another layout in tensor memory).
//
// float16 has five bits of exponent, so its P and dS go into the products scaled by powers of
// two, which come out of the results again: P by 64 (a shift of the log-sum-exp), dS by 64 G with
//   64 G 2 max|do_i| max|v_j| <= 2^15,  G max|v| <= 2^15   (over a sequence and k/v head)
// so that neither |dS_ij| <= P_ij (|do_i . v_j| + |delta_i|) nor V G overflows. The norms are bounded
// by the largest sum of squares of eight neighbouring elements. G is applied to V on its way into
// tensor memory and to delta in the subtraction, so the walk over the tiles has no instruction more
// for it. (V G is rounded again only below 2^-14, by 2^-25: at worst 2^-13 of the largest |V| G
// where |do| reaches 4096, 2^-9 where it reaches 65504.) Gradients of any size keep the bits that
// gradients of size one have: unscaled, do of 2^-14 over 16000 tokens gave later rows of dq and dk
// errors of 21 % (their own rounding to float16: 1.8 %), and dS above 65504 infinities. P's factor
// is for long rows that rest on one key: 4100 others of weight 2^-21, dv off by 1.2 % without it,
// by 0.06 % with it (a larger one would leave V G less).
// The sums of squares cost a read of V and a memset before: 4 x 4096 tokens, 32/8 heads of 128,
// under 2 %; 128 x 128 tokens 242 us against bfloat16's 218; 16/16 heads of 64, 4096 tokens in
// four sequences, forward and backward, 121 -> 125 us.
//
// Tiles start at the sequence's first token; rows of K, V, Q and dO behind its end are
// other tokens and are zeroed in shared memory, and their statistics make P zero.
#include "attention_bwd_parts.cuh"
#include "packed.cuh"

namespace evg {

__device__ int g_attn_packed_bwd_status = 0;

namespace {

using namespace umma;
using namespace attn;
using namespace attn_bwd;
using namespace packed;

constexpr int kComputeWarps = 16;  // two streams of eight
constexpr int kStreamWarps = 8;
constexpr int kCG = 4;             // column groups of compute warps in the final stores
// TMA warp, MMA warp, compute warps, 4 warps that take dQ^T out of tensor memory
constexpr int kBwdThreads = 32 * (2 + kComputeWarps + 4);
constexpr uint32_t kChunkBytes = 64 * 128 * 2;  // 64 queries x 128 keys of 16-bit dS^T
constexpr uint32_t kDqBytes = 32768;          // float32 dQ on its way out
// Stages of Q and dO, with their rows' statistics.
template <int HD> __host__ __device__ constexpr int bwd_stages() { return HD == 64 ? 3 : 2; }

template <int HD> __host__ __device__ constexpr uint32_t bwd_tile_region() {
  return (1 + 2 * bwd_stages<HD>()) * tile_bytes<HD>() + kDqBytes + 2 * kChunkBytes + 1024 * bwd_stages<HD>() + 128;
}

struct BwdParams {
  const int* plan;
  float* lse2;    // [Hq][slots * 128] log-sum-exp in log2 units, +inf behind a sequence
  float* delta;   // [Hq][slots * 128]
  float* dq_acc;  // [Hq][tokens / 128 tiles][128 x HD], tiles as acc_tile numbers them
  uint32_t* range;  // float16: [do, v][Hkv][seq_tiles], DsRange's words at a sequence's first
                    // padded tile
  int seq_tiles;
  View k, v, dq, dk, dv;
  int tokens, slots, units, head_group, group, D;
  float scale;
  long long wait_limit;
  uint32_t smem_bytes;
};

// Place of query tile t >= 1 of a sequence in the float32 copy. The n - 1 tiles behind the
// first of a sequence at rows [s, s + len) lie before row s + len when counted from s / 128, so
// no two sequences share one and tokens / 128 are enough however many sequences there are.
__device__ __forceinline__ int64_t acc_tile(const BwdParams& p, int head, int seq0, int t) {
  return (int64_t)head * (p.tokens / kTile) + seq0 / kTile + t - 1;
}
// float16: exponent of P's scale, and that of G for a sequence (by its first padded tile) and a
// k/v head.
constexpr int kPExponent = 6;
struct DsRange {
  float most_do, most_v;  // largest sum of squares of eight neighbouring elements
  __device__ __forceinline__ void load(const BwdParams& p, int tile0, int head_kv) {
    const uint32_t* at = p.range + (int64_t)head_kv * p.seq_tiles + tile0;
    most_do = __uint_as_float(at[0]);
    most_v = __uint_as_float(at[(int64_t)p.units * p.seq_tiles]);
  }
  // sqrt(x) < 2^half(x)
  static __device__ __forceinline__ int half(float x) { return ((int)(__float_as_uint(x) >> 23) - 127 + 2) >> 1; }
  // |do_i . v_j| <= HD / 8 sqrt(most_do most_v), and no element of v is above sqrt(most_v).
  template <int HD> __device__ __forceinline__ int exponent() const {
    const int for_ds = 15 - (kPExponent + 1) - (HD == 128 ? 4 : 3) - half(most_do * most_v);
    return min(min(for_ds, 15 - half(most_v)), 29);  // -31 .. 29
  }
};
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ void fence_proxy_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// float32 sums of a contiguous piece of shared memory into global memory, asynchronous
// (both addresses 16-byte aligned, a multiple of 16 bytes), in the thread's bulk group.
__device__ __forceinline__ void bulk_add_f32(float* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.reduce.async.bulk.global.shared::cta.bulk_group.add.f32 [%0], [%1], %2;" ::"l"(dst),
               "r"(smem_u32(src)), "r"(bytes)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// All but the newest N groups of this thread have read their source / are complete.
template <int N> __device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ uint8_t* view_row(const View& v, int64_t token, int head) {
  return reinterpret_cast<uint8_t*>(v.p) + (token * v.st + (int64_t)head * v.sh) * 2;
}

// A [128 x HD] float32 accumulator in tensor memory -> 16-bit rows of a tile in shared
// memory, 16-byte pieces XORed with the row (the compute warps; column groups of HD / kCG).
template <int HD, int FMT>
__device__ __forceinline__ void accumulator_to_tile(uint32_t t_acc, uint8_t* tile, float scale, const Roles& r) {
  constexpr int CW = HD / kCG;  // 32 or 16 columns per warp
  const int col = r.half * CW;
  uint32_t acc[CW];
  __syncwarp();
  tmem_ld(t_acc + ((uint32_t)(r.quarter * 32) << 16) + col, acc);
  tmem_wait_ld();
#pragma unroll
  for (int v = 0; v < CW / 8; ++v) {
    uint4 pk;
    pk.x = pack2<FMT>(__uint_as_float(acc[8 * v + 0]) * scale, __uint_as_float(acc[8 * v + 1]) * scale);
    pk.y = pack2<FMT>(__uint_as_float(acc[8 * v + 2]) * scale, __uint_as_float(acc[8 * v + 3]) * scale);
    pk.z = pack2<FMT>(__uint_as_float(acc[8 * v + 4]) * scale, __uint_as_float(acc[8 * v + 5]) * scale);
    pk.w = pack2<FMT>(__uint_as_float(acc[8 * v + 6]) * scale, __uint_as_float(acc[8 * v + 7]) * scale);
    reinterpret_cast<uint4*>(tile)[r.row * (HD / 8) + ((col / 8 + v) ^ (r.row & 7))] = pk;
  }
}
// That tile's rows inside the sequence -> a View, whole rows at a time (`t`: 0 .. 511).
template <int HD>
__device__ __forceinline__ void tile_to_view(const uint8_t* tile, const View& out, int head, int seq0,
                                             int row0, int L, int D, int t) {
  constexpr int TPR = HD / 8;
#pragma unroll
  for (int i = t; i < kTile * TPR; i += 32 * kComputeWarps) {
    const int row = i / TPR, piece = i % TPR;
    if (row0 + row < L && piece * 8 < D)
      reinterpret_cast<uint4*>(view_row(out, seq0 + row0 + row, head))[piece] =
          reinterpret_cast<const uint4*>(tile)[row * TPR + (piece ^ (row & 7))];
  }
}

template <int HD, int FMT>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_packed_bwd_kernel(const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ CUtensorMap map_do, const BwdParams p) {
  // Key tile n - w of a sequence of n tiles: w query tiles to visit, heaviest first.
  int slot, bh;
  map_block(blockIdx.x, p.slots, p.units, p.head_group, slot, bh);
  const int4 item = plan_item(p.plan, slot);
  if (item.z < 0) return;  // unused slot
  const int seq0 = item.x, L = item.y;
  if (item.z == 0) {  // rows behind the last sequence have zero gradients
    const int vec = p.D / 8;
    for (int i = threadIdx.x; i < L * vec; i += kBwdThreads) {
      const int64_t token = seq0 + i / vec;
      reinterpret_cast<uint4*>(view_row(p.dk, token, bh))[i % vec] = make_uint4(0, 0, 0, 0);
      reinterpret_cast<uint4*>(view_row(p.dv, token, bh))[i % vec] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int n_it = item.z;
  const int last_tile = (L - 1) / kTile;
  const int kvt = last_tile + 1 - n_it;
  const int tail_rows = L - last_tile * kTile;  // valid rows of the last tile
  const int kv0 = kvt * kTile;
  const int n_git = p.group * n_it;  // iteration c = head in group * n_it + it
  const int64_t P = (int64_t)p.slots * kTile;
  const int64_t prow0 = (int64_t)(item.w + kvt) * kTile;  // padded row of query tile it = 0

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr uint32_t TB = tile_bytes<HD>();
  constexpr uint32_t kRegion = bwd_tile_region<HD>();
  constexpr int NST = bwd_stages<HD>();
  constexpr bool kSplit = HD == 64;
  BlockSetup bs = carve(smem_raw, kRegion);
  if ((uint32_t)(bs.smem - smem_raw) + kRegion + (uint32_t)kControlBytes > p.smem_bytes) {
    if (threadIdx.x == 0) atomicCAS(&g_attn_packed_bwd_status, 0, 899);
    return;
  }
  uint8_t* sK = bs.smem;
  uint8_t* sDO0 = sK + TB;         // [NST]
  uint8_t* sQ0 = sDO0 + NST * TB;  // [NST]
  uint8_t* sDS = sQ0 + NST * TB;   // dS^T of the streams
  uint8_t* sDQ = sDS + 2 * kChunkBytes;  // float32 dQ on its way out
  float* s_stat = reinterpret_cast<float*>(sDQ + kDqBytes);  // [NST][lse2 | delta][128]
  uint64_t* kv_full = bs.bars + 0;   // K and V in tensor memory
  uint64_t* done = bs.bars + 1;      // K and V in shared memory; then: all products finished
  uint64_t* s_full = bs.bars + 2;    // [2] by stream, as those below
  uint64_t* x_free = bs.bars + 4;    // [2] the scores have been read
  uint64_t* dp_full = bs.bars + 6;   // [2]
  uint64_t* pds_full = bs.bars + 8;  // [2] P^T / dS^T are in tensor memory
  uint64_t* ds_full = bs.bars + 10;  // [2] dS^T is in shared memory
  uint64_t* dq_full = bs.bars + 12;  // [2]
  uint64_t* d_free = bs.bars + 14;   // [2] dQ^T has been read
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_stat + NST * 256);  // [NST] by stage, as those below
  uint64_t* q_empty = q_full + NST;
  uint64_t* do_full = q_empty + NST;
  uint64_t* do_empty = do_full + NST;
  const Roles r = roles();
  const float scale_log2 = p.scale * kLog2e;
  // A lone token's probability is one whatever its score: its dS is zero, and only rounding
  // noise of dP - delta stands in the accumulators.
  float ds_scale = L > 1 ? p.scale : 0.f;
  DsRange range = {0, 0};
  if constexpr (FMT == 0) range.load(p, item.w, bh);

  if (threadIdx.x == 0) {
    *bs.abort_flag = 0;
    mbar_init(kv_full, kComputeWarps); mbar_init(done, 1);
    for (int i = 0; i < NST; ++i) {
      mbar_init(q_full + i, 1); mbar_init(q_empty + i, 1);
      mbar_init(do_full + i, 1); mbar_init(do_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1); mbar_init(x_free + i, kStreamWarps);
      mbar_init(dp_full + i, 1); mbar_init(pds_full + i, kStreamWarps);
      mbar_init(ds_full + i, kStreamWarps); mbar_init(dq_full + i, 1); mbar_init(d_free + i, 4);
    }
    fence_mbar_init();
    prefetch_tensormap(&map_q); prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v); prefetch_tensormap(&map_do);
  }
  __syncthreads();
  if (threadIdx.x == 0) {  // the first copies do not wait for the tensor memory
    mbar_expect_tx(done, 2 * TB);
    load_tile<HD>(sK, &map_k, seq0 + kv0, bh, done);
    load_tile<HD>(sDS, &map_v, seq0 + kv0, bh, done);  // V only passes through
    mbar_expect_tx(q_full, TB);
    load_tile<HD>(sQ0, &map_q, seq0 + kv0, bh * p.group, q_full);
  }
  if (r.warp == 1) { tmem_alloc(bs.tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *bs.tmem_slot;
  const WaitCtx ctx{bs.abort_flag, &g_attn_packed_bwd_status, p.wait_limit};
  constexpr uint32_t idesc_p = instr_desc_f16(FMT, 128, 64, 0, 0);
  constexpr uint32_t idesc_d = instr_desc_f16(FMT, 128, HD, 0, 1);
  constexpr uint32_t idesc_q = instr_desc_f16(FMT, 128, 64, 1, 1);
  // stream b: scores at tS0 + 64 b, all that follows them at tY0 + 64 b
  const uint32_t tS0 = tmem, tY0 = kSplit ? tmem + 128 : tmem;
  const uint32_t tK = kSplit ? tmem + 256 : tmem + 128, tV = tK + HD / 2;
  const uint32_t tDV = tV + HD / 2, tDK = tDV + HD;
  const uint32_t tDQ0 = kSplit ? tDK + HD : tY0;  // + kDQ b
  constexpr uint32_t kDQ = kSplit ? 0 : 64;

  if (r.is_tma && r.lane == 0) {
    int it = 0, head = bh * p.group, git = 0;
    for (; git < n_git; ++git) {
      const int st = git % NST;
      const uint32_t reuse = (uint32_t)((git / NST - 1) & 1);
      const int q0 = seq0 + (kvt + it) * kTile;
      if (git >= NST) mbar_wait(q_empty + st, reuse, ctx, 821);
      if (*ctx.abort_flag) break;  // no new copies after a timeout
      if (git > 0) {
        mbar_expect_tx(q_full + st, TB);
        load_tile<HD>(sQ0 + st * TB, &map_q, q0, head, q_full + st);
      }
      if (git >= NST) mbar_wait(do_empty + st, reuse, ctx, 831);
      if (!*ctx.abort_flag) {
        const int64_t prow = head * P + prow0 + (int64_t)it * kTile;
        mbar_expect_tx(do_full + st, TB + 1024);
        load_tile<HD>(sDO0 + st * TB, &map_do, q0, head, do_full + st);
        bulk_load_1d(s_stat + st * 256, p.lse2 + prow, 512, do_full + st);
        bulk_load_1d(s_stat + st * 256 + 128, p.delta + prow, 512, do_full + st);
      }
      if (++it == n_it) { it = 0; ++head; }
    }
    if (*ctx.abort_flag) {
      // Let the copies still in flight land before the block returns: each of
      // these waits gives up after the same cycle budget.
      mbar_drain(done, 0, p.wait_limit);
      for (int g = git > NST ? git - NST : 0; g < git; ++g) {
        mbar_drain(q_full + g % NST, (uint32_t)((g / NST) & 1), p.wait_limit);
        mbar_drain(do_full + g % NST, (uint32_t)((g / NST) & 1), p.wait_limit);
      }
    }
  } else if (r.is_mma) {
    const bool lead = elect_one();
    const DescBase kt_base = desc_base_mnmajor(smem_u32(sK), kTile);
    // [128 keys x 64 queries] of stream b into its columns: A = K or V in tensor memory,
    // B = rows [64 b, 64 b + 64) of a Q or dO tile.
    auto issue_rows = [&](int b, uint32_t dst, uint32_t a_tmem, uint32_t tile_saddr, uint64_t* bar) {
      const DescBase rows = desc_base_kmajor(tile_saddr + b * 64 * 128);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        if (lead)
          mma_ts(dst + 64 * b, a_tmem + 8 * ks, desc_at(rows, kstep_kmajor(kTile, ks)), idesc_p,
                 ks > 0 ? 1u : 0u);
      if (lead) mma_commit(bar + b);
    };
    // Query k-step kk of the stream (16 queries): P^T in its columns [16 kk, 16 kk + 8),
    // dS^T in the 8 columns behind it (the layout the compute warps write).
    auto issue_dv = [&](int b, uint32_t do_saddr, bool first) {
      const DescBase dob = desc_base_mnmajor(do_saddr + b * 64 * 128, kTile);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        if (lead)
          mma_ts(tDV, tY0 + 64 * b + kk * 16, desc_at(dob, kstep_mnmajor(kk)), idesc_d,
                 (first && kk == 0) ? 0u : 1u);
    };
    auto issue_dk = [&](int b, uint32_t q_saddr, bool first) {
      const DescBase qb = desc_base_mnmajor(q_saddr + b * 64 * 128, kTile);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        if (lead)
          mma_ts(tDK, tY0 + 64 * b + kk * 16 + 8, desc_at(qb, kstep_mnmajor(kk)), idesc_d,
                 (first && kk == 0) ? 0u : 1u);
    };
    // dQ^T of stream b over its P^T / dS^T: A = K^T (the K tile read MN-major), B = dS^T.
    auto issue_dq = [&](int b) {
      const DescBase dsb = desc_base_mnmajor(smem_u32(sDS) + b * kChunkBytes, kTile);
#pragma unroll
      for (int ks = 0; ks < kTile / 16; ++ks)
        if (lead)
          mma_ss(tDQ0 + kDQ * b, desc_at(kt_base, kstep_mnmajor(ks)), desc_at(dsb, kstep_mnmajor(ks)),
                 idesc_q, ks > 0 ? 1u : 0u);
      if (lead) mma_commit(dq_full + b);
    };
    // Query iteration `it` reads the sequence's last tile: its rows behind the end are zeroed.
    auto clear_tail = [&](uint8_t* tile, int it) {
      if (it == n_it - 1 && tail_rows < kTile) clear_tile_rows<HD>(tile, tail_rows, r.lane);
    };
    mbar_wait(kv_full, 0, ctx, 822);
    if (kvt == last_tile && tail_rows < kTile) clear_tile_rows<HD>(sK, tail_rows, r.lane);
    if constexpr (kSplit) {
      // Stage and parity of tile c's operands.
      auto stage = [&](int c) { return c % NST; };
      auto turn = [&](int c) { return (uint32_t)((c / NST) & 1); };
      auto q_at = [&](int c) { return sQ0 + stage(c) * TB; };
      auto do_at = [&](int c) { return sDO0 + stage(c) * TB; };
      mbar_wait(q_full, 0, ctx, 823);
      clear_tail(sQ0, 0);
      tc_fence_after_sync();
      issue_rows(0, tS0, tK, smem_u32(sQ0), s_full);
      issue_rows(1, tS0, tK, smem_u32(sQ0), s_full);
      mbar_wait(do_full, 0, ctx, 832);
      clear_tail(sDO0, 0);
      tc_fence_after_sync();
      issue_rows(0, tY0, tV, smem_u32(sDO0), dp_full);
      issue_rows(1, tY0, tV, smem_u32(sDO0), dp_full);
      int it = 0;
      for (int c = 0; c < n_git; ++c) {
        const uint32_t par = (uint32_t)(c & 1);
        const bool more = c + 1 < n_git;
        const int it_next = it + 1 == n_it ? 0 : it + 1;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (more) {
            if (b == 0) {
              mbar_wait(q_full + stage(c + 1), turn(c + 1), ctx, 823);
              clear_tail(q_at(c + 1), it_next);
            }
            mbar_wait(x_free + b, par, ctx, 828);
            tc_fence_after_sync();
            issue_rows(b, tS0, tK, smem_u32(q_at(c + 1)), s_full);
          }
          mbar_wait(pds_full + b, par, ctx, 824);
          tc_fence_after_sync();
          issue_dv(b, smem_u32(do_at(c)), b == 0 && c == 0);
          if (b && lead) mma_commit(do_empty + stage(c));
          issue_dk(b, smem_u32(q_at(c)), b == 0 && c == 0);
          if (b && lead) mma_commit(q_empty + stage(c));
          if (more) {
            if (b == 0) {
              mbar_wait(do_full + stage(c + 1), turn(c + 1), ctx, 832);
              clear_tail(do_at(c + 1), it_next);
              tc_fence_after_sync();
            }
            issue_rows(b, tY0, tV, smem_u32(do_at(c + 1)), dp_full);
          }
          mbar_wait(ds_full + b, par, ctx, 825);
          if (b) mbar_wait(d_free + 0, par, ctx, 835);
          else if (c > 0) mbar_wait(d_free + 1, par ^ 1u, ctx, 826);
          tc_fence_after_sync();
          issue_dq(b);
        }
        it = it_next;
        __syncwarp();
      }
    } else {
      int it = 0;  // query tile of iteration c
      for (int c = 0; c <= n_git; ++c) {
        const int st = c & 1;
        const uint32_t par = (uint32_t)(c & 1), full = (uint32_t)((c >> 1) & 1);
        const bool now = c < n_git, behind = c > 0;  // tile c; stream 1's second half of tile c - 1
        uint8_t *q_tile = sQ0 + st * TB, *do_tile = sDO0 + st * TB;
        const uint32_t q_saddr = smem_u32(q_tile), do_saddr = smem_u32(do_tile);
        if (now) {
          mbar_wait(q_full + st, full, ctx, 823);
          clear_tail(q_tile, it);
          if (behind) mbar_wait(d_free + 0, par ^ 1u, ctx, 835);
          tc_fence_after_sync();
          issue_rows(0, tS0, tK, q_saddr, s_full);
        }
        if (behind) {
          mbar_wait(pds_full + 1, par ^ 1u, ctx, 829);
          tc_fence_after_sync();
          issue_dv(1, smem_u32(sDO0 + (st ^ 1) * TB), false);
          if (lead) mma_commit(do_empty + (st ^ 1));
          issue_dk(1, smem_u32(sQ0 + (st ^ 1) * TB), false);
          if (lead) mma_commit(q_empty + (st ^ 1));
        }
        if (now) {
          mbar_wait(do_full + st, full, ctx, 832);
          clear_tail(do_tile, it);
          mbar_wait(x_free + 0, par, ctx, 828);
          tc_fence_after_sync();
          issue_rows(0, tY0, tV, do_saddr, dp_full);
        }
        if (behind) {
          mbar_wait(ds_full + 1, par ^ 1u, ctx, 834);
          tc_fence_after_sync();
          issue_dq(1);
        }
        if (now) {
          if (behind) {
            mbar_wait(d_free + 1, par ^ 1u, ctx, 826);
            tc_fence_after_sync();
          }
          issue_rows(1, tS0, tK, q_saddr, s_full);
          mbar_wait(pds_full + 0, par, ctx, 824);
          tc_fence_after_sync();
          issue_dv(0, do_saddr, c == 0);
          issue_dk(0, q_saddr, c == 0);
          mbar_wait(x_free + 1, par, ctx, 833);
          tc_fence_after_sync();
          issue_rows(1, tY0, tV, do_saddr, dp_full);
          mbar_wait(ds_full + 0, par, ctx, 825);
          tc_fence_after_sync();
          issue_dq(0);
        }
        if (++it == n_it) it = 0;
        __syncwarp();
      }
    }
    if (lead) mma_commit(done);
  } else if (r.warp >= 2 + kComputeWarps) {
    // dQ^T of every half tile to the float32 copy: out of tensor memory (a thread has one
    // head column), into shared memory in the copy's layout, and on by an asynchronous bulk
    // reduction, 16 KB at a time, one piece being written while the other is read.
    // (Reductions issued by these threads, 64 lines each, held up every access of the SM to
    // shared memory and mbarriers for about 1100 cycles per half tile.)
    const uint32_t lane_base = (uint32_t)(r.quarter * 32) << 16;
    constexpr uint32_t kPiece = kDqBytes / 2;
    constexpr int kRows = kPiece / (HD * 4);  // queries: half of a half tile, or all of it
    // (row of the copy, as acc_tile numbers it: the address once per tile, 64-bit, and the loop
    // below not unrolled, or the accumulator's 64 registers spill: 226 us against 216 for the
    // step over 16 sequences of 1 to 900 tokens)
    const int64_t head_rows = (int64_t)(p.tokens / kTile) * kTile, row0 = (int64_t)(seq0 / kTile + kvt - 1) * kTile;
    const bool issuer = r.warp == 2 + kComputeWarps && r.lane == 0;
    if constexpr (FMT == 0) ds_scale *= power_of_two(-kPExponent - range.exponent<HD>());
    int it = 0, head = bh * p.group;
    for (int c = 0; c < n_git; ++c) {
      const uint32_t par = (uint32_t)(c & 1);
      float* tile_dst = p.dq_acc + (head * head_rows + row0 + (int64_t)it * kTile) * HD;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        mbar_wait(dq_full + b, par, ctx, 841);
        __syncwarp();
        tc_fence_after_sync();
        uint32_t acc[2][32];
        tmem_ld(tDQ0 + kDQ * b + lane_base, acc[0]);
        tmem_ld(tDQ0 + kDQ * b + lane_base + 32, acc[1]);
        tmem_wait_ld();
        warp_arrive(d_free + b, r.lane);
        if (kvt == 0 && it == 0) {
          // A sequence's first query tile gets its whole dQ here: rounded, through the same
          // shared memory, and written as whole rows.
          constexpr int TPR = HD / 8;
          if (issuer) bulk_wait_read<0>();  // earlier reductions have read it
          named_barrier_sync(1, 128);
          if (r.row < HD) {
#pragma unroll
            for (int j = 0; j < 64; ++j)
              reinterpret_cast<uint16_t*>(sDQ)[j * HD + r.row] =
                  (uint16_t)pack2<FMT>(__uint_as_float(acc[j >> 5][j & 31]) * ds_scale, 0.f);
          }
          named_barrier_sync(1, 128);
#pragma unroll 1
          for (int k = 0; k < 64 * TPR / 128; ++k) {
            const int i = r.row + 128 * k, row = b * 64 + i / TPR, col = i % TPR;
            if (row < L && col * 8 < p.D)
              reinterpret_cast<uint4*>(view_row(p.dq, seq0 + row, head))[col] =
                  reinterpret_cast<const uint4*>(sDQ)[i];
          }
        } else {
#pragma unroll
          for (int h = 0; h < 64 / kRows; ++h) {
            uint8_t* piece = sDQ + (HD == 64 ? b : h) * kPiece;
            if (issuer) bulk_wait_read<1>();  // this piece's last reduction has read it
            named_barrier_sync(1, 128);
            if (r.row < HD) {
              uint4* dst = reinterpret_cast<uint4*>(piece) + r.row;
#pragma unroll
              for (int j = 0; j < kRows / 4; ++j) {
                const int q = h * kRows + 4 * j;
                dst[j * HD] = make_uint4(acc[q >> 5][q & 31], acc[q >> 5][(q & 31) + 1], acc[q >> 5][(q & 31) + 2],
                                         acc[q >> 5][(q & 31) + 3]);
              }
            }
            fence_proxy_async_smem();
            named_barrier_sync(1, 128);
            if (issuer && !*ctx.abort_flag) bulk_add_f32(tile_dst + (b * 64 + h * kRows) * HD, piece, kPiece);
          }
        }
      }
      if (++it == n_it) { it = 0; ++head; }
    }
    if (issuer) bulk_wait_all();
  } else if (r.is_compute) {
    const uint32_t lane_base = (uint32_t)(r.quarter * 32) << 16;
    const int kv_pos = kv0 + r.row;
    const int b = (r.warp - 2) / kStreamWarps;               // stream
    const int col0 = ((r.warp - 2) % kStreamWarps / 4) * 32;  // first query column inside its half tile
    const uint32_t tY = tY0 + 64 * b + lane_base + col0;
    const f32x2 neg_scale2 = f2_splat(-scale_log2);
    // Stream 0's warps put K, stream 1's V into tensor memory: a thread its key's row (half
    // of it), two 16-bit elements per column, zero behind the sequence's end. (Read from
    // global memory row by row this took 8500 cycles per block.)
    {
      mbar_wait(done, 0, ctx, 849);
      const uint8_t* src = (b ? sDS : sK) + r.row * 128;
      const bool ok = kv_pos < L;
      constexpr int PW = HD / 16;  // 16-byte pieces per warp, all in one 64-column atom
      const int piece0 = (col0 / 32) * PW;
      uint32_t w[4 * PW];
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        const int piece = piece0 + i;
        const uint4 x = ok ? *reinterpret_cast<const uint4*>(src + (piece >> 3) * (kTile * 128) +
                                                             (((piece & 7) ^ (r.row & 7)) << 4))
                           : make_uint4(0, 0, 0, 0);
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      }
      if (FMT == 0 && b) {
        const int gain = range.exponent<HD>();
        const __half2 g1 = __float2half2_rn(power_of_two(gain >> 1)), g2 = __float2half2_rn(power_of_two(gain - (gain >> 1)));
#pragma unroll
        for (int i = 0; i < 4 * PW; ++i) {
          const __half2 x = __hmul2(__hmul2(*reinterpret_cast<const __half2*>(&w[i]), g1), g2);
          w[i] = *reinterpret_cast<const uint32_t*>(&x);
        }
      }
      const uint32_t dst = (b ? tV : tK) + lane_base + piece0 * 4;
#pragma unroll
      for (int i = 0; i < PW / 4; ++i) tmem_st(dst + 16 * i, *reinterpret_cast<uint32_t(*)[16]>(&w[16 * i]));
      tmem_wait_st();
      warp_arrive(kv_full, r.lane);
    }
    const float minus_gain = FMT == 0 ? -power_of_two(range.exponent<HD>()) : -1.f;
    const f32x2 minus_gain2 = f2_splat(minus_gain);
    int it = 0;
    for (int c = 0; c < n_git; ++c) {
      const int st = c % NST;
      const uint32_t par = (uint32_t)(c & 1);
      const float* stat = s_stat + st * 256 + b * 64 + col0;
      // P^T: t = lse2 - s c, p = 2^-t, two columns per packed instruction. On the first
      // query tile, queries before the key are masked. S^T is handed back as soon as its
      // columns are in registers.
      f32x2 p2[16];
      mbar_wait(do_full + st, (uint32_t)((c / NST) & 1), ctx, 842);
      mbar_wait(s_full + b, par, ctx, 843);
      __syncwarp();
      tc_fence_after_sync();
      {
        uint32_t sr[32];
        tmem_ld(tS0 + 64 * b + lane_base + col0, sr);
        tmem_wait_ld();
        warp_arrive(x_free + b, r.lane);
        const float4* lse4 = reinterpret_cast<const float4*>(stat);
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const float4 l4 = lse4[g];
          const f32x2 t01 = f2_fma(f2_make(__uint_as_float(sr[4 * g]), __uint_as_float(sr[4 * g + 1])),
                                   neg_scale2, f2_make(l4.x, l4.y));
          const f32x2 t23 = f2_fma(f2_make(__uint_as_float(sr[4 * g + 2]), __uint_as_float(sr[4 * g + 3])),
                                   neg_scale2, f2_make(l4.z, l4.w));
          float t[4];
          f2_split(t01, t[0], t[1]);
          f2_split(t23, t[2], t[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) t[e] = fast_exp2(-t[e]);
          p2[2 * g] = f2_make(t[0], t[1]);
          p2[2 * g + 1] = f2_make(t[2], t[3]);
        }
      }
      if (it == 0) {
        const int q_first = kv0 + b * 64 + col0;
#pragma unroll
        for (int g = 0; g < 16; ++g) {
          float lo, hi;
          f2_split(p2[g], lo, hi);
          if (q_first + 2 * g < kv_pos) lo = 0.f;
          if (q_first + 2 * g + 1 < kv_pos) hi = 0.f;
          p2[g] = f2_make(lo, hi);
        }
      }
      // dS^T = P^T (dP^T - delta), 16 queries at a time; P^T and dS^T go back over dP^T
      // first: the products that wait for them are the critical path.
      mbar_wait(dp_full + b, par, ctx, 844);
      __syncwarp();
      tc_fence_after_sync();
      uint32_t dd[2][8];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t dr[16], pp[8];
        tmem_ld(tY + 16 * k, dr);
        tmem_wait_ld();
        const float4* del4 = reinterpret_cast<const float4*>(stat + 128 + 16 * k);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 d4 = del4[g];
          const f32x2 a01 = f2_fma(f2_make(d4.x, d4.y), minus_gain2,
                                   f2_make(__uint_as_float(dr[4 * g]), __uint_as_float(dr[4 * g + 1])));
          const f32x2 a23 = f2_fma(f2_make(d4.z, d4.w), minus_gain2,
                                   f2_make(__uint_as_float(dr[4 * g + 2]), __uint_as_float(dr[4 * g + 3])));
          float d[4], pe[4];
          f2_split(f2_mul(p2[8 * k + 2 * g], a01), d[0], d[1]);
          f2_split(f2_mul(p2[8 * k + 2 * g + 1], a23), d[2], d[3]);
          f2_split(p2[8 * k + 2 * g], pe[0], pe[1]);
          f2_split(p2[8 * k + 2 * g + 1], pe[2], pe[3]);
          pp[2 * g] = pack2<FMT>(pe[0], pe[1]);
          pp[2 * g + 1] = pack2<FMT>(pe[2], pe[3]);
          dd[k][2 * g] = pack2<FMT>(d[0], d[1]);
          dd[k][2 * g + 1] = pack2<FMT>(d[2], d[3]);
        }
        tmem_st(tY + 16 * k, pp);
        tmem_st(tY + 16 * k + 8, dd[k]);
      }
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (r.lane == 0) mbar_arrive(pds_full + b);
      // dS^T for the dQ^T product: row r.row (a key) of the half's [128 keys x 64 queries]
      // tile, four 16-byte pieces of its 128 bytes at their swizzled places. The buffer's
      // last reader, the last dQ^T, has to be finished (at head size 128 this dP^T waited
      // for it).
      {
        if (kSplit && c > 0) mbar_wait(dq_full + b, par ^ 1u, ctx, 846);
        uint8_t* row_ptr = sDS + b * kChunkBytes + r.row * 128;
        const int sw = r.row & 7, piece = col0 / 8;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          *reinterpret_cast<uint4*>(row_ptr + (((piece + 2 * k) ^ sw) << 4)) =
              make_uint4(dd[k][0], dd[k][1], dd[k][2], dd[k][3]);
          *reinterpret_cast<uint4*>(row_ptr + (((piece + 2 * k + 1) ^ sw) << 4)) =
              make_uint4(dd[k][4], dd[k][5], dd[k][6], dd[k][7]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (r.lane == 0) mbar_arrive(ds_full + b);
      if (++it == n_it) it = 0;
    }
    // dV and dK through the dO stages, which no product reads any more
    mbar_wait(done, 1, ctx, 847);
    __syncwarp();
    tc_fence_after_sync();
    accumulator_to_tile<HD, FMT>(tDV, sDO0, FMT == 0 ? power_of_two(-kPExponent) : 1.0f, r);
    accumulator_to_tile<HD, FMT>(tDK, sDO0 + TB, FMT == 0 ? ds_scale * power_of_two(-kPExponent) / -minus_gain : ds_scale, r);
    named_barrier_sync(2, 32 * kComputeWarps);
    const int t = (r.warp - 2) * 32 + r.lane;
    tile_to_view<HD>(sDO0, p.dv, bh, seq0, kv0, L, p.D, t);
    tile_to_view<HD>(sDO0 + TB, p.dk, bh, seq0, kv0, L, p.D, t);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (r.warp == 1) tmem_dealloc(tmem, 512);
}

// Row statistics of every item's query tile: delta = do . o and the log-sum-exp in log2
// units, padded rows +inf / 0, and the tile's rows of the float32 dQ copy cleared
// (where the copy is used).
// In rows that see only a few keys dS = P (dP - delta) is often a small difference, to which the
// rounding of o to 16 bits contributes much: relative error of a row's dq over 4000 random draws
// (bf16, head size 128), mean and largest, row 1: 2.6 % and 1500 %, row 2: 0.5 and 25, row 4: 0.3
// and 5, rows 8 to 19: 0.27 and 2 to 3; with delta from its definition 0.23 and 0.4 in all of
// them. So the first kExactRows rows of every sequence sum sum_j P_ij do_i . v_j. (Later rows
// whose softmax rests on one or two keys have the same small difference and take o.)
// A block takes 256 / (HD / 8) rows of one head at a time; bound by the latency of its loads, so six
// blocks share an SM (134 MB of do and o each: 57 us, 120 with two blocks).
constexpr int kExactRows = 8;
template <int FMT> __device__ __forceinline__ float dot8(const uint4& a, const uint4& b) {
  float af[8], bf[8], s = 0.f;
  if constexpr (FMT == 1) { unpack<__nv_bfloat16>(a, af); unpack<__nv_bfloat16>(b, bf); }
  else { unpack<__half>(a, af); unpack<__half>(b, bf); }
#pragma unroll
  for (int i = 0; i < 8; ++i) s += af[i] * bf[i];
  return s;
}

// The larger of m and x >= 0 as float bits; infinities and NaN (their rows' gradients are not
// finite whatever the scale) do not count.
__device__ __forceinline__ uint32_t finite_max(uint32_t m, float x) {
  const uint32_t b = __float_as_uint(x);
  return b < 0x7f800000u && b > m ? b : m;
}
// *at = max(*at, every lane's m).
__device__ __forceinline__ void raise(uint32_t* at, uint32_t m) {
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0 && m) atomicMax(at, m);
}

// c += A B^T over 16 columns of A's rows 0 .. 7 (rows 8 .. 15 are zero) and B's rows 0 .. 7.
template <int FMT>
__device__ __forceinline__ void mma_8x8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
  if constexpr (FMT == 1)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%6,%5,%6}, {%7,%8}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(0), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%6,%5,%6}, {%7,%8}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(0), "r"(b0), "r"(b1));
}
// delta of a sequence's first kExactRows rows by one warp: two 8 x 8 products (queries and keys,
// do and values) in a few matrix instructions each. Lane l holds row l / 4 of either side, 16
// bytes of every 32 columns; which column of a product's 16 they stand for is the same on both
// sides and does not matter. Latency-bound (three dependent loads), so eight sequences share a
// block of their own. Backward of 128 sequences of 128 tokens, 32/8 heads of 128, bfloat16: 218
// us, 212 with delta from o, 266 with these rows summed one by one beside the others; of 32
// sequences of 512: 443 and 441.
template <int HD, int FMT>
__device__ __forceinline__ void exact_delta(const View& dout, const View& q, const float* lse, const BwdParams& p,
                                            const int4& item, int head, float* delta) {
  const int lane = threadIdx.x & 31, r = lane >> 2, part = lane & 3;
  const bool ok = r < item.y;
  const int64_t token = item.x + (ok ? r : 0);
  auto product = [&](const uint8_t* a_row, const uint8_t* b_row, float (&c)[4]) {
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int col = 32 * i + 8 * part;
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      if (ok && col < p.D) {
        a = ld_vec(a_row + 2 * col);
        b = ld_vec(b_row + 2 * col);
      }
      mma_8x8<FMT>(c, a.x, a.y, b.x, b.y);
      mma_8x8<FMT>(c, a.z, a.w, b.z, b.w);
    }
  };
  float s[4] = {0.f, 0.f, 0.f, 0.f}, dp[4] = {0.f, 0.f, 0.f, 0.f};
  product(view_row(q, token, head), view_row(p.k, token, head / p.group), s);
  product(view_row(dout, token, head), view_row(p.v, token, head / p.group), dp);
  const float lse_row = ok ? lse[(int64_t)head * p.tokens + token] : 0.f;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (ok && 2 * part + i <= r) sum += expf(p.scale * s[i] - lse_row) * dp[i];
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
  if (part == 0) delta[r] = sum;
}

template <int HD, int FMT>
__global__ void __launch_bounds__(256, 6)
packed_prepare_kernel(const View dout, const View q, const View o, const float* __restrict__ lse,
                      const BwdParams p) {
  constexpr int TPR = HD / 8;
  constexpr int ROWS = 256 / TPR;
  const int head = blockIdx.y;
  if (blockIdx.x >= p.slots) {  // the first rows of eight items
    const int slot = (blockIdx.x - p.slots) * 8 + threadIdx.x / 32;
    if (slot >= p.slots || blockIdx.z > 0) return;
    const int4 item = plan_item(p.plan, slot);
    if (item.z == 1) exact_delta<HD, FMT>(dout, q, lse, p, item, head, p.delta + ((int64_t)head * p.slots + item.w) * kTile);
    return;
  }
  const int4 item = plan_item(p.plan, blockIdx.x);
  if (item.z <= 0) return;
  const int part = threadIdx.x % TPR;
  const int tile0 = (item.z - 1) * kTile;
  const int64_t prow0 = (int64_t)head * p.slots * kTile + (int64_t)item.w * kTile + tile0;
  const bool takes_v = FMT == 0 && head % p.group == 0;
  uint32_t most_do = 0, most_v = 0;  // float bits: ordered as the numbers
#pragma unroll 1
  for (int r = threadIdx.x / TPR + blockIdx.z * ROWS; r < kTile; r += ROWS * gridDim.z) {
    const bool ok = tile0 + r < item.y, mine = ok && part * 8 < p.D;
    const int64_t token = item.x + tile0 + r;
    uint4 g, ov, vv;
    g = ov = vv = make_uint4(0, 0, 0, 0);
    if (mine) {
      g = ld_vec(view_row(dout, token, head) + part * 16);
      ov = ld_vec(view_row(o, token, head) + part * 16);
      if (takes_v) vv = ld_vec(view_row(p.v, token, head / p.group) + part * 16);
    }
    const float lse_row = ok ? lse[(int64_t)head * p.tokens + token] : 0.f;
    float s = dot8<FMT>(g, ov);
#pragma unroll
    for (int off = TPR / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if constexpr (FMT == 0) {
      most_do = finite_max(most_do, dot8<FMT>(g, g));
      if (takes_v) most_v = finite_max(most_v, dot8<FMT>(vv, vv));
    }
    if (item.z > 1) {
      uint4* acc = reinterpret_cast<uint4*>(p.dq_acc + (acc_tile(p, head, item.x, item.z - 1) * kTile + r) * HD + part * 8);
      acc[0] = acc[1] = make_uint4(0, 0, 0, 0);
    }
    if (part == 0) {
      if (item.z > 1 || r >= kExactRows) p.delta[prow0 + r] = ok ? s : 0.f;
      p.lse2[prow0 + r] = ok ? lse_row * kLog2e - (FMT == 0 ? kPExponent : 0) : INFINITY;
    }
  }
  if constexpr (FMT == 0) {
    uint32_t* at = p.range + (int64_t)(head / p.group) * p.seq_tiles + item.w;
    raise(at, most_do);
    if (takes_v) raise(at + (int64_t)p.units * p.seq_tiles, most_v);
  }
}

// dq = round(scale * float32 copy), zero behind the last sequence. The copy of a tile is
// laid out [query / 4][head column][query % 4]: a thread takes 4 queries x 8 columns.
template <int HD, int FMT>
__global__ void __launch_bounds__(256)
packed_finish_kernel(const BwdParams p) {
  constexpr int TPR = HD / 8;
  constexpr int QUADS = 256 / TPR;  // groups of 4 queries per round
  const int4 item = plan_item(p.plan, blockIdx.x);
  if (item.z < 0 || item.z == 1) return;  // first tiles: written by the products' kernel
  const int head = blockIdx.y;
  const int part = threadIdx.x % TPR;
  if (part * 8 >= p.D) return;
  const int tile0 = item.z > 0 ? (item.z - 1) * kTile : 0;
  const int rows = min(kTile, item.y - tile0);
  float scale = p.scale;
  if constexpr (FMT == 0) {
    if (item.z > 0) {
      DsRange range;
      range.load(p, item.w, head / p.group);
      scale *= power_of_two(-kPExponent - range.exponent<HD>());
    }
  }
  for (int qd = threadIdx.x / TPR + blockIdx.z * QUADS; qd * 4 < rows; qd += QUADS * gridDim.z) {
    float v[4][8];
    if (item.z > 0) {
      const float4* src = reinterpret_cast<const float4*>(p.dq_acc + (acc_tile(p, head, item.x, item.z - 1) * kTile + qd * 4) * HD) + part * 8;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float4 f = __ldcs(src + c);
        v[0][c] = f.x; v[1][c] = f.y; v[2][c] = f.z; v[3][c] = f.w;
      }
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) v[0][c] = v[1][c] = v[2][c] = v[3][c] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (qd * 4 + i < rows) {
        uint4 pk;
        pk.x = pack2<FMT>(v[i][0] * scale, v[i][1] * scale);
        pk.y = pack2<FMT>(v[i][2] * scale, v[i][3] * scale);
        pk.z = pack2<FMT>(v[i][4] * scale, v[i][5] * scale);
        pk.w = pack2<FMT>(v[i][6] * scale, v[i][7] * scale);
        *reinterpret_cast<uint4*>(view_row(p.dq, item.x + tile0 + qd * 4 + i, head) + part * 16) = pk;
      }
  }
}

int read_packed_bwd_status(int reset) {
  int code = 0;
  if (cudaMemcpyFromSymbol(&code, g_attn_packed_bwd_status, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (reset && code != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_attn_packed_bwd_status, &zero, sizeof(int));
  }
  return code;
}
const bool g_packed_bwd_registered = (register_device_status(read_packed_bwd_status), true);

template <int HD, int FMT>
int launch(const View& dout, const View& q, const View& o, const float* lse, BwdParams& p, int64_t Hq, int64_t Hkv, cudaStream_t stream) {
  CUtensorMap mq, mk, mv, mdo;
  if (!encode_view_map(&mq, q, FMT, p.D, p.tokens, Hq) ||
      !encode_view_map(&mk, p.k, FMT, p.D, p.tokens, Hkv) ||
      !encode_view_map(&mv, p.v, FMT, p.D, p.tokens, Hkv) ||
      !encode_view_map(&mdo, dout, FMT, p.D, p.tokens, Hq))
    return fail(EVG_ELAUNCH, "packed_attention_bwd: cuTensorMapEncodeTiled failed");
  size_t smem = bwd_tile_region<HD>() + kControlBytes + 1024;
  const size_t most = (size_t)device_info().max_smem_optin;
  if (smem > most) smem = most;
  p.smem_bytes = (uint32_t)smem;
  auto kern = attn_packed_bwd_kernel<HD, FMT>;
  if (int rc = reserve_smem(kern, smem)) return rc;
  // rows of one tile are cut into `parts` blocks while there are few tiles
  const int64_t tiles = (int64_t)p.slots * Hq;
  constexpr int kMostParts = kTile / (256 / (HD / 8));
  const int64_t want = (4 * (int64_t)device_info().sm_count + tiles - 1) / tiles;
  const int parts = (int)(want < 1 ? 1 : want > kMostParts ? kMostParts : want);
  const dim3 rows_grid((unsigned)p.slots, (unsigned)Hq, (unsigned)parts);
  if (FMT == 0 && cudaMemsetAsync(p.range, 0, (size_t)2 * p.units * p.seq_tiles * 4, stream) != cudaSuccess)
    return check_launch("packed_attention_bwd range");
  const dim3 prepare_grid((unsigned)(p.slots + (p.slots + 7) / 8), rows_grid.y, rows_grid.z);
  packed_prepare_kernel<HD, FMT><<<prepare_grid, 256, 0, stream>>>(dout, q, o, lse, p);
  if (int rc = check_launch("packed_attention_bwd statistics")) return rc;
  kern<<<(unsigned)((int64_t)p.slots * p.units), kBwdThreads, smem, stream>>>(mq, mk, mv, mdo, p);
  if (int rc = check_launch("packed_attention_bwd")) return rc;
  packed_finish_kernel<HD, FMT><<<rows_grid, 256, 0, stream>>>(p);
  return check_launch("packed_attention_bwd dq");
}

}  // namespace

namespace packed {

// Most padded tiles of all sequences together.
int64_t sequence_tiles(int64_t tokens, int64_t sequences) {
  return (tokens + (kTile - 1) * (sequences < tokens ? sequences : tokens)) / kTile;
}
int64_t bwd_workspace_bytes(int64_t tokens, int64_t sequences, int64_t Hq, int64_t D) {
  const int64_t rows = plan_slots(tokens, sequences) * kTile * Hq;
  return rows * 2 * 4 + tokens / kTile * kTile * Hq * (D > 64 ? 128 : 64) * 4 + sequence_tiles(tokens, sequences) * Hq * 8;
}

int launch_bwd(const View& dout, const View& q, const View& k, const View& v, const View& o,
               const float* lse, const View& dq, const View& dk, const View& dv, void* workspace,
               const void* plan, int64_t tokens, int64_t sequences, int64_t Hq, int64_t Hkv,
               int64_t D, float scale, int fmt, cudaStream_t stream) {
  BwdParams p{};
  p.plan = (const int*)plan;
  p.tokens = (int)tokens;
  p.slots = (int)plan_slots(tokens, sequences);
  const int64_t rows = (int64_t)p.slots * kTile * Hq;
  p.lse2 = (float*)workspace;
  p.delta = p.lse2 + rows;
  p.dq_acc = p.delta + rows;
  p.range = (uint32_t*)(p.dq_acc + tokens / kTile * kTile * Hq * (D > 64 ? 128 : 64));
  p.seq_tiles = (int)sequence_tiles(tokens, sequences);
  p.k = k;
  p.v = v;
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.group = (int)(Hq / Hkv);
  p.units = (int)Hkv;
  p.D = (int)D;
  p.head_group = head_group_for((int64_t)p.slots * Hkv, Hkv);
  p.scale = scale;
  p.wait_limit = wait_limit_cycles2();
  if (D > 64)
    return fmt == 1 ? launch<128, 1>(dout, q, o, lse, p, Hq, Hkv, stream)
                    : launch<128, 0>(dout, q, o, lse, p, Hq, Hkv, stream);
  return fmt == 1 ? launch<64, 1>(dout, q, o, lse, p, Hq, Hkv, stream)
                  : launch<64, 0>(dout, q, o, lse, p, Hq, Hkv, stream);
}

}  // namespace packed
}  // namespace evg
