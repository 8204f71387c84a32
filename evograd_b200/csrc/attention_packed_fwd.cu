// Causal grouped-query attention over a packed batch, forward (sm_100a).
//
//   s_ij = scale q_i . k_j (j <= i, same sequence),  o_i = sum_j softmax_j(s_ij) v_j,
//   lse_i = log sum_j exp(s_ij)
//
// 320 threads per block: a TMA producer warp, a tcgen05 issuer warp and two groups
// of four softmax warps, each group with a 128-row query tile of its own (TMEM:
// S_A [0,128), S_B [128,256), O_A [256,256+HD), O_B [384,384+HD)), so one tile's
// softmax runs while the other tile's products do. Per key tile j:
//   O_A += P_A(j) V_j;  S_A(j+1) = Q_A K_{j+1}^T;  O_B += P_B(j) V_j;  S_B(j+1) = ...
//
// The two query tiles of a block share their key tiles. Where the query heads of a
// k/v head can be paired (an even group), they are the SAME positions of two heads:
// both tiles are equally long and a sequence of one tile still fills both groups.
// Otherwise they are two neighbouring tiles of one head.
//
// Tiles start at the sequence's first token (a TMA coordinate along the token axis
// has no alignment rule). The last tile's rows behind the sequence's end are other
// tokens: as keys the causal mask drops them, as values they are zeroed in shared
// memory (0 x infinity), as queries they are computed and not stored.
//
// Bound: the special-function unit and the tensor pipe together (one exponential per
// visible pair and head; 4 HD flop).
#include "packed.cuh"

namespace evg {

__device__ int g_attn_packed_fwd_status = 0;

namespace {

using namespace umma;
using namespace attn;
using namespace packed;

constexpr int kFwdThreads = 320;

struct FwdParams {
  const int* plan;
  void* o;
  int64_t o_st, o_sh;
  float* lse;
  int tokens, slots, units, head_group, group, D;
  int pair_heads;  // the block's two tiles are two heads (else two neighbouring tiles)
  float scale_log2;
  long long wait_limit;
};

// 16-bit rows of one head set to zero, lse to -inf: tokens behind the last sequence.
__device__ __forceinline__ void clear_rows(const FwdParams& p, int row0, int rows, int head) {
  const int vec = p.D / 8;
  uint8_t* o = reinterpret_cast<uint8_t*>(p.o);
  for (int i = threadIdx.x; i < rows * vec; i += kFwdThreads) {
    const int r = i / vec, c = i % vec;
    *reinterpret_cast<uint4*>(o + ((int64_t)(row0 + r) * p.o_st + (int64_t)head * p.o_sh + c * 8) * 2) =
        make_uint4(0, 0, 0, 0);
  }
  for (int r = threadIdx.x; r < rows; r += kFwdThreads)
    p.lse[(int64_t)head * p.tokens + row0 + r] = -INFINITY;
}

template <int HD, int FMT>
__global__ void __launch_bounds__(kFwdThreads, 1)
attn_packed_fwd_kernel(const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const FwdParams p) {
  int slot, unit;
  map_block(blockIdx.x, p.slots, p.units, p.head_group, slot, unit);
  const int4 item = plan_item(p.plan, slot);
  if (item.z < 0) return;  // unused slot
  const int head[2] = {p.pair_heads ? 2 * unit : unit, p.pair_heads ? 2 * unit + 1 : unit};
  const int seq0 = item.x, L = item.y;
  if (item.z == 0) {
    clear_rows(p, seq0, L, head[0]);
    if (p.pair_heads) clear_rows(p, seq0, L, head[1]);
    return;
  }
  const int last_tile = (L - 1) / kTile;
  int qt[2], n_kv[2];
  if (p.pair_heads) {
    qt[0] = qt[1] = item.z - 1;
    n_kv[0] = n_kv[1] = item.z;
  } else {
    // an item of odd weight whose successor exists is that item's tile A
    const int t = item.z - 1;
    if (!(t & 1) && t < last_tile) return;
    qt[0] = t & ~1;
    qt[1] = t | 1;
    n_kv[0] = qt[0] + 1;
    n_kv[1] = (t & 1) ? qt[1] + 1 : 0;
  }
  const bool b_active = n_kv[1] > 0;
  const int n_max = b_active ? n_kv[1] : n_kv[0];
  const int head_kv = head[0] / p.group;

  extern __shared__ uint8_t smem_raw[];
  constexpr uint32_t TB = tile_bytes<HD>();
  BlockSetup bs = carve(smem_raw, 6 * TB);
  uint8_t* sQ[2] = {bs.smem, bs.smem + TB};
  uint8_t* sK[2] = {bs.smem + 2 * TB, bs.smem + 3 * TB};
  uint8_t* sV[2] = {bs.smem + 4 * TB, bs.smem + 5 * TB};
  uint64_t* q_full = bs.bars + 0;
  uint64_t* k_full = bs.bars + 1;   // [2]
  uint64_t* k_empty = bs.bars + 3;  // [2]
  uint64_t* v_full = bs.bars + 5;   // [2]
  uint64_t* v_empty = bs.bars + 7;  // [2]
  uint64_t* s_full = bs.bars + 9;   // [2] tile A, tile B
  uint64_t* p_full = bs.bars + 11;  // [2]
  uint64_t* o_done = bs.bars + 13;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    *bs.abort_flag = 0;
    mbar_init(q_full, 1); mbar_init(o_done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 1); mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 1); mbar_init(v_empty + i, 1);
      mbar_init(s_full + i, 1); mbar_init(p_full + i, 4);
    }
    fence_mbar_init();
    prefetch_tensormap(&map_q); prefetch_tensormap(&map_k); prefetch_tensormap(&map_v);
  }
  __syncthreads();
  if (warp == 1) { tmem_alloc(bs.tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *bs.tmem_slot;
  const WaitCtx ctx{bs.abort_flag, &g_attn_packed_fwd_status, p.wait_limit};
  constexpr uint32_t idesc_s = instr_desc_f16(FMT, 128, 128, 0, 0);
  constexpr uint32_t idesc_o = instr_desc_f16(FMT, 128, HD, 0, 1);
  const uint32_t tS[2] = {tmem, tmem + 128};
  const uint32_t tO[2] = {tmem + 256, tmem + 384};

  if (warp == 0) {
    if (lane == 0) {
      mbar_expect_tx(q_full, (b_active ? 2 : 1) * TB);
      load_tile<HD>(sQ[0], &map_q, seq0 + qt[0] * kTile, head[0], q_full);
      if (b_active) load_tile<HD>(sQ[1], &map_q, seq0 + qt[1] * kTile, head[1], q_full);
      int j = 0;
      for (; j < n_max; ++j) {
        const int st = j & 1;
        if (j >= 2) mbar_wait(k_empty + st, ((j >> 1) - 1) & 1, ctx, 801);
        if (*ctx.abort_flag) break;  // no new copies after a timeout
        mbar_expect_tx(k_full + st, TB);
        load_tile<HD>(sK[st], &map_k, seq0 + j * kTile, head_kv, k_full + st);
        if (j >= 2) mbar_wait(v_empty + st, ((j >> 1) - 1) & 1, ctx, 802);
        if (!*ctx.abort_flag) {
          mbar_expect_tx(v_full + st, TB);
          load_tile<HD>(sV[st], &map_v, seq0 + j * kTile, head_kv, v_full + st);
        }
      }
      if (*ctx.abort_flag) {
        // let the copies still in flight land before the block returns
        mbar_drain(q_full, 0, p.wait_limit);
        for (int g = j > 2 ? j - 2 : 0; g < j; ++g) {
          mbar_drain(k_full + (g & 1), (uint32_t)((g >> 1) & 1), p.wait_limit);
          mbar_drain(v_full + (g & 1), (uint32_t)((g >> 1) & 1), p.wait_limit);
        }
      }
    }
  } else if (warp == 1) {
    const bool lead = elect_one();
    const int tail_rows = L - last_tile * kTile;  // valid rows of the sequence's last tile
    mbar_wait(q_full, 0, ctx, 803);
    mbar_wait(k_full + 0, 0, ctx, 804);
    tc_fence_after_sync();
    issue_scores<HD>(lead, tS[0], smem_u32(sQ[0]), smem_u32(sK[0]), idesc_s);
    if (lead) mma_commit(s_full + 0);
    if (b_active) {
      issue_scores<HD>(lead, tS[1], smem_u32(sQ[1]), smem_u32(sK[0]), idesc_s);
      if (lead) mma_commit(s_full + 1);
    }
    if (lead) mma_commit(k_empty + 0);
    for (int j = 0; j < n_max; ++j) {
      const int st = j & 1, st1 = (j + 1) & 1;
      const uint32_t ph = j & 1;
      mbar_wait(v_full + st, (j >> 1) & 1, ctx, 805);
      if (j == last_tile && tail_rows < kTile) clear_tile_rows<HD>(sV[st], tail_rows, lane);
      if (j < n_kv[0]) {
        mbar_wait(p_full + 0, ph, ctx, 806);
        tc_fence_after_sync();
        issue_accumulate(lead, tO[0], tS[0], smem_u32(sV[st]), idesc_o, j > 0);
      }
      if (j + 1 < n_max) {
        mbar_wait(k_full + st1, ((j + 1) >> 1) & 1, ctx, 807);
        tc_fence_after_sync();
      }
      if (j + 1 < n_kv[0]) {
        issue_scores<HD>(lead, tS[0], smem_u32(sQ[0]), smem_u32(sK[st1]), idesc_s);
        if (lead) mma_commit(s_full + 0);
      }
      if (b_active) {
        mbar_wait(p_full + 1, ph, ctx, 808);
        tc_fence_after_sync();
        issue_accumulate(lead, tO[1], tS[1], smem_u32(sV[st]), idesc_o, j > 0);
      }
      if (lead) mma_commit(v_empty + st);
      if (b_active && j + 1 < n_kv[1]) {
        issue_scores<HD>(lead, tS[1], smem_u32(sQ[1]), smem_u32(sK[st1]), idesc_s);
        if (lead) mma_commit(s_full + 1);
      }
      if (lead && j + 1 < n_max) mma_commit(k_empty + st1);
      __syncwarp();
    }
    if (lead) mma_commit(o_done);
  } else {
    // ---- softmax warps: one query row per thread
    const int wg = (warp - 2) >> 2;  // 0: tile A, 1: tile B
    const int quarter = warp & 3;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int row = quarter * 32 + lane;
    const int my_tile = wg ? qt[1] : qt[0], my_head = wg ? head[1] : head[0];
    const int q_pos = my_tile * kTile + row;  // position inside the sequence
    const int n_mine = wg ? n_kv[1] : n_kv[0];
    const uint32_t tSw = tmem + wg * 128, tOw = tmem + 256 + wg * 128;
    const float scale_log2 = p.scale_log2;
    float m_run = -INFINITY, l_run = 0.f;
    for (int j = 0; j < n_mine; ++j) {
      mbar_wait(s_full + wg, j & 1, ctx, 809);
      __syncwarp();
      tc_fence_after_sync();
      // Pass 1: row maximum. Columns [0, 64) stay in registers for pass 2, [64, 96)
      // arrive in the same round trip to tensor memory and [96, 128) while the first
      // maxima are formed; four partial maxima keep the dependent chains short.
      const int kv0 = j * kTile;
      const bool diag = (j == my_tile);
      uint32_t keep[64], tmp[32];
      tmem_ld32(tSw + lane_base, *reinterpret_cast<uint32_t(*)[32]>(&keep[0]));
      tmem_ld32(tSw + lane_base + 32, *reinterpret_cast<uint32_t(*)[32]>(&keep[32]));
      tmem_ld32(tSw + lane_base + 64, tmp);
      tmem_wait_ld();
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      auto fold = [&](const uint32_t* v, int col0, int n) {
        if (diag) {
#pragma unroll
          for (int i = 0; i < n; ++i) {
            float t = __uint_as_float(v[i]);
            if (kv0 + col0 + i > q_pos) t = -INFINITY;
            mx4[i & 3] = fmaxf(mx4[i & 3], t);
          }
        } else {
#pragma unroll
          for (int i = 0; i < n; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], __uint_as_float(v[i]));
        }
      };
      fold(tmp, 64, 32);
      tmem_ld32(tSw + lane_base + 96, tmp);
      fold(keep, 0, 64);
      tmem_wait_ld();
      fold(tmp, 96, 32);
      // scale_log2 > 0, so scaling commutes with the maximum
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;
      const bool grow = mx > m_run + kRescaleThreshold;  // always true on the first tile
      const float m_new = grow ? mx : m_run;
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
        // Rescale this warp's rows of O (rows that did not grow use alpha = 1). The
        // previous O += P V has completed: the scores just read were issued after it.
        const float alpha = grow ? fast_exp2(m_run - m_new) : 1.0f;
        l_run *= alpha;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t orow[32];
          tmem_ld32(tOw + lane_base + c * 32, orow);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) orow[i] = __float_as_uint(__uint_as_float(orow[i]) * alpha);
          tmem_st32(tOw + lane_base + c * 32, orow);
        }
      }
      m_run = m_new;
      // Pass 2: probabilities. The packed P of chunk c (16 columns) lands in columns
      // [16c, 16c+16), which belong to score chunks already consumed. P is rounded to
      // 16 bits as the tensor cores' operand; its sum is taken before rounding.
      const float neg_m = -m_run;
      float ls4[4] = {0.f, 0.f, 0.f, 0.f};
      auto probs = [&](const uint32_t* v, int c) {
        uint32_t pr[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float p0 = fast_exp2(fmaf(__uint_as_float(v[2 * i]), scale_log2, neg_m));
          float p1 = fast_exp2(fmaf(__uint_as_float(v[2 * i + 1]), scale_log2, neg_m));
          if (diag) {
            if (kv0 + c * 32 + 2 * i > q_pos) p0 = 0.f;
            if (kv0 + c * 32 + 2 * i + 1 > q_pos) p1 = 0.f;
          }
          ls4[i & 3] += p0 + p1;
          pr[i] = pack2<FMT>(p0, p1);
        }
        tmem_st16(tSw + lane_base + c * 16, pr);
      };
      // columns [64, 128) come back from tensor memory under the exponentials of [0, 64)
      uint32_t late[32];
      tmem_ld32(tSw + lane_base + 64, late);
      probs(&keep[0], 0);
      tmem_ld32(tSw + lane_base + 96, tmp);
      probs(&keep[32], 1);
      tmem_wait_ld();
      probs(late, 2);
      probs(tmp, 3);
      l_run += (ls4[0] + ls4[1]) + (ls4[2] + ls4[3]);
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + wg);
    }
    if (n_mine > 0) {
      mbar_wait(o_done, 0, ctx, 810);
      __syncwarp();
      tc_fence_after_sync();
      const float inv_l = 1.0f / l_run;
      const bool row_ok = q_pos < L;
      const int64_t token = seq0 + (row_ok ? q_pos : 0);
      uint8_t* orow_g = reinterpret_cast<uint8_t*>(p.o) + (token * p.o_st + (int64_t)my_head * p.o_sh) * 2;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t orow[32];
        tmem_ld32(tOw + lane_base + c * 32, orow);
        tmem_wait_ld();
        if (row_ok) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            if (c * 32 + v * 8 < p.D) {
              uint4 pk;
              pk.x = pack2<FMT>(__uint_as_float(orow[8 * v + 0]) * inv_l, __uint_as_float(orow[8 * v + 1]) * inv_l);
              pk.y = pack2<FMT>(__uint_as_float(orow[8 * v + 2]) * inv_l, __uint_as_float(orow[8 * v + 3]) * inv_l);
              pk.z = pack2<FMT>(__uint_as_float(orow[8 * v + 4]) * inv_l, __uint_as_float(orow[8 * v + 5]) * inv_l);
              pk.w = pack2<FMT>(__uint_as_float(orow[8 * v + 6]) * inv_l, __uint_as_float(orow[8 * v + 7]) * inv_l);
              *reinterpret_cast<uint4*>(orow_g + (c * 32 + v * 8) * 2) = pk;
            }
          }
        }
      }
      if (row_ok) p.lse[(int64_t)my_head * p.tokens + token] = (m_run + log2f(l_run)) * kLn2;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

int read_packed_fwd_status(int reset) {
  int code = 0;
  if (cudaMemcpyFromSymbol(&code, g_attn_packed_fwd_status, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (reset && code != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_attn_packed_fwd_status, &zero, sizeof(int));
  }
  return code;
}
const bool g_packed_fwd_registered = (register_device_status(read_packed_fwd_status), true);

template <int HD, int FMT>
int launch(const View& q, const View& k, const View& v, const FwdParams& p, int64_t Hq, int64_t Hkv,
           cudaStream_t stream) {
  CUtensorMap mq, mk, mv;
  if (!encode_view_map(&mq, q, FMT, p.D, p.tokens, Hq) ||
      !encode_view_map(&mk, k, FMT, p.D, p.tokens, Hkv) ||
      !encode_view_map(&mv, v, FMT, p.D, p.tokens, Hkv))
    return fail(EVG_ELAUNCH, "packed_attention_fwd: cuTensorMapEncodeTiled failed");
  const size_t smem = 6 * tile_bytes<HD>() + kControlBytes + 1024;
  auto kern = attn_packed_fwd_kernel<HD, FMT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
      cudaSuccess) {
    cudaGetLastError();
    return fail(EVG_ELAUNCH, "packed_attention_fwd: cannot reserve %zu bytes of shared memory", smem);
  }
  kern<<<(unsigned)((int64_t)p.slots * p.units), kFwdThreads, smem, stream>>>(mq, mk, mv, p);
  return check_launch("packed_attention_fwd");
}

}  // namespace

namespace packed {

int launch_fwd(const View& q, const View& k, const View& v, const View& o, float* lse,
               const void* plan, int64_t tokens, int64_t sequences, int64_t Hq, int64_t Hkv,
               int64_t D, float scale, int fmt, cudaStream_t stream) {
  FwdParams p{};
  p.plan = (const int*)plan;
  p.o = o.p;
  p.o_st = o.st;
  p.o_sh = o.sh;
  p.lse = lse;
  p.tokens = (int)tokens;
  p.slots = (int)plan_slots(tokens, sequences);
  p.group = (int)(Hq / Hkv);
  p.D = (int)D;
  p.pair_heads = p.group % 2 == 0;
  p.units = (int)(p.pair_heads ? Hq / 2 : Hq);
  p.head_group = head_group_for((int64_t)p.slots * p.units, p.units);
  p.scale_log2 = scale * kLog2e;
  const int t = tune("attention.wait_limit");
  p.wait_limit = t > 0 ? (long long)t * 1000000ll : 2000000000ll;
  if (D > 64)
    return fmt == 1 ? launch<128, 1>(q, k, v, p, Hq, Hkv, stream) : launch<128, 0>(q, k, v, p, Hq, Hkv, stream);
  return fmt == 1 ? launch<64, 1>(q, k, v, p, Hq, Hkv, stream) : launch<64, 0>(q, k, v, p, Hq, Hkv, stream);
}

}  // namespace packed
}  // namespace evg
