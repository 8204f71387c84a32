// Causal grouped-query attention over a packed batch, forward (sm_100a).
//
//   s_ij = scale q_i . k_j (j <= i, same sequence),  o_i = sum_j softmax_j(s_ij) v_j,
//   lse_i = log sum_j exp(s_ij)
//
// A TMA producer warp, a tcgen05 issuer warp and one or two groups of four softmax warps,
// each group with a 128-row query tile of its own, so one tile's softmax runs while the
// other's products do: two groups share a block's key tiles, or two blocks of one group
// share the SM (the rule is at launch_fwd). Keys come in tiles of 128 and are worked
// through in halves of 64: each group has two score buffers, and while it turns one half's
// scores into probabilities the other half's are being formed, so its warps never wait for
// a product that waits for them (with one 128-key buffer per group the chain
// scores -> softmax -> PV -> next scores took 3980 cycles per key tile). Per half g:
//   O_A += P_A(g) V_g;  S_A(g+2) = Q_A K_{g+2}^T;  O_B += P_B(g) V_g;  S_B(g+2) = ...
// TMEM of G groups: score buffers [128 w, 128 w + 128) of group w (P packed over the scores
// it came from), O [128 G + 128 w, 128 G + 128 w + HD).
//
// Where the query heads of a k/v head can be paired (an even group), a block's two tiles
// are the SAME positions of two heads: both are equally long and a sequence of one tile
// still fills both groups. Otherwise they are two neighbouring tiles of one head.
//
// O leaves through shared memory as whole rows: with a thread writing its own row, 128
// sequences of 128 tokens (32/8 heads of 128) took 143 us, 134 this way
// (132 with the first copies ahead of the tensor memory's allocation).
//
// Tiles start at the sequence's first token (a TMA coordinate along the token axis
// has no alignment rule). The last tile's rows behind the sequence's end are other
// tokens: as keys the causal mask drops them, as values they are zeroed in shared
// memory (0 x infinity), as queries they are computed and not stored.
//
// Bound: the softmax warps' chain per half (TMEM load, maximum, 64 exponentials and their
// packing, TMEM store: 1700-1900 cycles for the two warps of a scheduler, the special-
// function unit busy for 1024 of them) and, in long runs, the power limit. Forming a
// quarter or a third of the exponentials by a polynomial on the FMA pipe was 5-7 %
// slower. 12001 + 2500 + 1000 + 883 tokens, 32/8 heads of 128: 1121 us after a pause (1111
// TFLOP/s), 1155 to 1193 in a long run.
#include "packed.cuh"

namespace evg {

__device__ int g_attn_packed_fwd_status = 0;

namespace {

using namespace umma;
using namespace attn;
using namespace packed;

// TILES query tiles per block: 2, or 1 with two blocks on an SM.
constexpr int fwd_threads(int tiles) { return 64 + 128 * tiles; }
// Stages of the K and V rings. One tile per block at head size 128 has room for one: the
// other block's work covers the wait.
template <int HD, int TILES> __host__ __device__ constexpr int fwd_stages() { return TILES == 1 && HD == 128 ? 1 : 2; }
template <int HD, int TILES> __host__ __device__ constexpr int fwd_smem_tiles() { return TILES + 2 * fwd_stages<HD, TILES>(); }

struct FwdParams {
  const int* plan;
  void* o;
  int64_t o_st, o_sh;
  float* lse;
  int tokens, slots, units, head_group, group, D;
  int pair_heads;  // two tiles: of two heads (else two neighbouring tiles of one)
  float scale_log2;
  long long wait_limit;
};

// Maximum of three (one instruction).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 16-bit rows of one head set to zero, lse to -inf: tokens behind the last sequence.
__device__ __forceinline__ void clear_rows(const FwdParams& p, int row0, int rows, int head) {
  const int vec = p.D / 8;
  uint8_t* o = reinterpret_cast<uint8_t*>(p.o);
  for (int i = threadIdx.x; i < rows * vec; i += blockDim.x) {
    const int r = i / vec, c = i % vec;
    *reinterpret_cast<uint4*>(o + ((int64_t)(row0 + r) * p.o_st + (int64_t)head * p.o_sh + c * 8) * 2) =
        make_uint4(0, 0, 0, 0);
  }
  for (int r = threadIdx.x; r < rows; r += blockDim.x)
    p.lse[(int64_t)head * p.tokens + row0 + r] = -INFINITY;
}

// P and its sum carry a factor 2^p_exponent, which the division by the sum takes out again. float16
// reaches down to 2^-14 with all its bits: where one key has nearly all of a row's weight (a first
// token, say), the others' probabilities can lie below that although they are the result (4100
// keys of 2^-21 each beside one whose value is zero: o off by 1.2 %, 0.035 % with the factor). P is
// at most 2^kRescaleThreshold times it.
template <int FMT> __host__ __device__ constexpr float p_exponent() { return FMT == 0 ? 7.f : 0.f; }
static_assert(kRescaleThreshold + 7.f <= 15.f, "P stays below 65504");

template <int HD, int FMT, int TILES>
__global__ void __launch_bounds__(fwd_threads(TILES), 3 - TILES)
attn_packed_fwd_kernel(const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const FwdParams p) {
  int slot, unit;
  map_block(blockIdx.x, p.slots, p.units, p.head_group, slot, unit);
  const int4 item = plan_item(p.plan, slot);
  if (item.z < 0) return;  // unused slot
  constexpr bool kTwo = TILES == 2;
  constexpr int KST = fwd_stages<HD, TILES>();
  const bool pair_heads = kTwo && p.pair_heads;
  const int head[2] = {pair_heads ? 2 * unit : unit, pair_heads ? 2 * unit + 1 : unit};
  const int seq0 = item.x, L = item.y;
  if (item.z == 0) {
    clear_rows(p, seq0, L, head[0]);
    if (pair_heads) clear_rows(p, seq0, L, head[1]);
    return;
  }
  const int last_tile = (L - 1) / kTile;
  int qt[2], n_kv[2];
  if (pair_heads || !kTwo) {
    qt[0] = qt[1] = item.z - 1;
    n_kv[0] = item.z;
    n_kv[1] = kTwo ? item.z : 0;
  } else {
    // an item of odd weight whose successor exists is that item's tile A
    const int t = item.z - 1;
    if (!(t & 1) && t < last_tile) return;
    qt[0] = t & ~1;
    qt[1] = t | 1;
    n_kv[0] = qt[0] + 1;
    n_kv[1] = (t & 1) ? qt[1] + 1 : 0;
  }
  const bool b_active = kTwo && n_kv[1] > 0;
  const int n_max = b_active ? n_kv[1] : n_kv[0];
  const int head_kv = head[0] / p.group;
  // halves of 64 keys; a last tile of at most 64 tokens has one
  const int tail_rows = L - last_tile * kTile;  // valid rows of the sequence's last tile
  const int n_half[2] = {2 * n_kv[0] - (qt[0] == last_tile && tail_rows <= 64),
                         b_active ? 2 * n_kv[1] - (qt[1] == last_tile && tail_rows <= 64) : 0};

  extern __shared__ uint8_t smem_raw[];
  constexpr uint32_t TB = tile_bytes<HD>();
  BlockSetup bs = carve(smem_raw, fwd_smem_tiles<HD, TILES>() * TB);
  uint8_t* sQ[2] = {bs.smem, bs.smem + (TILES - 1) * TB};
  uint8_t* sK = bs.smem + TILES * TB;  // [KST]
  uint8_t* sV = sK + KST * TB;         // [KST]
  uint64_t* q_full = bs.bars + 0;
  uint64_t* k_full = bs.bars + 1;   // [2]
  uint64_t* k_empty = bs.bars + 3;  // [2]
  uint64_t* v_full = bs.bars + 5;   // [2]
  uint64_t* v_empty = bs.bars + 7;  // [2]
  uint64_t* s_full = bs.bars + 9;    // [tile A, tile B][half]
  uint64_t* p_full = bs.bars + 13;   // [tile A, tile B][half]
  uint64_t* pv_done = bs.bars + 17;  // [tile A, tile B]
  uint64_t* o_done = bs.bars + 19;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    *bs.abort_flag = 0;
    mbar_init(q_full, 1); mbar_init(o_done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 1); mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 1); mbar_init(v_empty + i, 1);
      mbar_init(pv_done + i, 1);
    }
    for (int i = 0; i < 4; ++i) { mbar_init(s_full + i, 1); mbar_init(p_full + i, 4); }
    fence_mbar_init();
    prefetch_tensormap(&map_q); prefetch_tensormap(&map_k); prefetch_tensormap(&map_v);
  }
  __syncthreads();
  if (threadIdx.x == 0) {  // the first copies do not wait for the tensor memory
    mbar_expect_tx(q_full, (b_active ? 2 : 1) * TB);
    load_tile<HD>(sQ[0], &map_q, seq0 + qt[0] * kTile, head[0], q_full);
    if (b_active) load_tile<HD>(sQ[1], &map_q, seq0 + qt[1] * kTile, head[1], q_full);
    mbar_expect_tx(k_full, TB);
    load_tile<HD>(sK, &map_k, seq0, head_kv, k_full);
    mbar_expect_tx(v_full, TB);
    load_tile<HD>(sV, &map_v, seq0, head_kv, v_full);
  }
  if (warp == 1) { tmem_alloc(bs.tmem_slot, 256 * TILES); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *bs.tmem_slot;
  const WaitCtx ctx{bs.abort_flag, &g_attn_packed_fwd_status, p.wait_limit};
  constexpr uint32_t idesc_s = instr_desc_f16(FMT, 128, 64, 0, 0);
  constexpr uint32_t idesc_o = instr_desc_f16(FMT, 128, HD, 0, 1);

  if (warp == 0) {
    if (lane == 0) {
      int j = 1;
      for (; j < n_max; ++j) {
        const int st = j % KST;
        const uint32_t reuse = (uint32_t)((j / KST - 1) & 1);
        if (j >= KST) mbar_wait(k_empty + st, reuse, ctx, 801);
        if (*ctx.abort_flag) break;  // no new copies after a timeout
        mbar_expect_tx(k_full + st, TB);
        load_tile<HD>(sK + st * TB, &map_k, seq0 + j * kTile, head_kv, k_full + st);
        if (j >= KST) mbar_wait(v_empty + st, reuse, ctx, 802);
        if (!*ctx.abort_flag) {
          mbar_expect_tx(v_full + st, TB);
          load_tile<HD>(sV + st * TB, &map_v, seq0 + j * kTile, head_kv, v_full + st);
        }
      }
      if (*ctx.abort_flag) {
        // let the copies still in flight land before the block returns
        mbar_drain(q_full, 0, p.wait_limit);
        for (int g = j > KST ? j - KST : 0; g < j; ++g) {
          mbar_drain(k_full + g % KST, (uint32_t)((g / KST) & 1), p.wait_limit);
          mbar_drain(v_full + g % KST, (uint32_t)((g / KST) & 1), p.wait_limit);
        }
      }
    }
  } else if (warp == 1) {
    const bool lead = elect_one();
    // Scores of half g of tile w (0: A, 1: B): keys [64 hf, 64 hf + 64) of a K tile.
    auto issue_s = [&](int w, int hf, const uint8_t* q_tile, const uint8_t* k_tile) {
      const DescBase qb = desc_base_kmajor(smem_u32(q_tile));
      const DescBase kb = desc_base_kmajor(smem_u32(k_tile) + hf * 64 * 128);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        if (lead)
          mma_ss(tmem + w * 128 + hf * 64, desc_at(qb, kstep_kmajor(kTile, ks)),
                 desc_at(kb, kstep_kmajor(kTile, ks)), idesc_s, ks > 0 ? 1u : 0u);
      if (lead) mma_commit(s_full + 2 * w + hf);
    };
    auto issue_pv = [&](int w, int hf, const uint8_t* v_tile, bool first) {
      const DescBase vb = desc_base_mnmajor(smem_u32(v_tile) + hf * 64 * 128, kTile);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        if (lead)
          mma_ts(tmem + TILES * 128 + w * 128, tmem + w * 128 + hf * 64 + ks * 8, desc_at(vb, kstep_mnmajor(ks)),
                 idesc_o, (first && ks == 0) ? 0u : 1u);
      if (lead) mma_commit(pv_done + w);
    };
    mbar_wait(q_full, 0, ctx, 803);
    mbar_wait(k_full + 0, 0, ctx, 804);
    tc_fence_after_sync();
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      if (hf < n_half[0]) issue_s(0, hf, sQ[0], sK);
      if (kTwo && hf < n_half[1]) issue_s(1, hf, sQ[1], sK);
    }
    if (lead) mma_commit(k_empty + 0);
    for (int j = 0; j < n_max; ++j) {
      const int st = j % KST, st1 = (j + 1) % KST;
      const uint32_t par = j & 1;
      uint8_t* v_tile = sV + st * TB;
      const uint8_t* k_next = sK + st1 * TB;
      mbar_wait(v_full + st, (uint32_t)((j / KST) & 1), ctx, 805);
      if (j == last_tile && tail_rows < kTile) clear_tile_rows<HD>(v_tile, tail_rows, lane);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int g = 2 * j + hf;
        if (g < n_half[0]) {
          mbar_wait(p_full + hf, par, ctx, 806);
          tc_fence_after_sync();
          issue_pv(0, hf, v_tile, g == 0);
        }
        if (hf == 0 && j + 1 < n_max) {
          mbar_wait(k_full + st1, (uint32_t)(((j + 1) / KST) & 1), ctx, 807);
          tc_fence_after_sync();
        }
        if (g + 2 < n_half[0]) issue_s(0, hf, sQ[0], k_next);
        if (kTwo && g < n_half[1]) {
          mbar_wait(p_full + 2 + hf, par, ctx, 808);
          tc_fence_after_sync();
          issue_pv(1, hf, v_tile, g == 0);
          if (g + 2 < n_half[1]) issue_s(1, hf, sQ[1], k_next);
        }
      }
      if (lead) mma_commit(v_empty + st);
      if (lead && j + 1 < n_max) mma_commit(k_empty + st1);
      __syncwarp();
    }
    if (lead) mma_commit(o_done);
  } else {
    // ---- softmax warps: one query row per thread
    const int wg = kTwo ? (warp - 2) >> 2 : 0;  // 0: tile A, 1: tile B
    const int quarter = warp & 3;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int row = quarter * 32 + lane;
    const int my_tile = wg ? qt[1] : qt[0], my_head = wg ? head[1] : head[0];
    const int q_pos = my_tile * kTile + row;  // position inside the sequence
    const int n_mine = wg ? n_half[1] : n_half[0];
    const uint32_t tOw = tmem + TILES * 128 + wg * 128;
    const float scale_log2 = p.scale_log2;
    constexpr float kPExponent = p_exponent<FMT>();
    float m_run = -INFINITY, l_run = 0.f;
    for (int g = 0; g < n_mine; ++g) {
      const int hf = g & 1;
      const uint32_t tSw = tmem + wg * 128 + hf * 64 + lane_base;
      mbar_wait(s_full + 2 * wg + hf, (g >> 1) & 1, ctx, 809);
      __syncwarp();
      tc_fence_after_sync();
      const int kv0 = g * 64;
      const bool diag = (g >> 1) == my_tile;
      uint32_t sr[64];
      tmem_ld32(tSw, *reinterpret_cast<uint32_t(*)[32]>(&sr[0]));
      tmem_ld32(tSw + 32, *reinterpret_cast<uint32_t(*)[32]>(&sr[32]));
      tmem_wait_ld();
      // Four partial maxima keep the comparisons from forming one long dependent chain.
      float mx4[4];
      if (diag) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (kv0 + i > q_pos) sr[i] = __float_as_uint(-INFINITY);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) mx4[i] = fmaxf(__uint_as_float(sr[i]), __uint_as_float(sr[i + 4]));
#pragma unroll
      for (int i = 8; i < 64; i += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mx4[k] = max3(mx4[k], __uint_as_float(sr[i + k]), __uint_as_float(sr[i + k + 4]));
      // scale_log2 > 0, so scaling commutes with the maximum
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;
      const bool grow = mx > m_run + kRescaleThreshold;  // always true on the first half
      const float m_new = grow ? mx : m_run;
      if (g > 0 && __any_sync(0xffffffffu, grow)) {
        // Rescale this warp's rows of O (rows that did not grow use alpha = 1) once the
        // half before this one has been added.
        mbar_wait(pv_done + wg, (g - 1) & 1, ctx, 811);
        __syncwarp();
        tc_fence_after_sync();
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
      // Probabilities: 64 score columns -> 32 packed columns over them. P is rounded to 16
      // bits as the tensor cores' operand; its sum is taken before rounding. A masked score
      // of -infinity gives zero, also while a row has seen nothing else (m_run is -infinity).
      const f32x2 neg_m2 = f2_splat(kPExponent - (m_run == -INFINITY ? 0.f : m_run)), scale2 = f2_splat(scale_log2);
      f32x2 ls2[2] = {0ull, 0ull};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t pr[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f32x2 x = f2_fma(f2_make(__uint_as_float(sr[32 * c + 2 * i]), __uint_as_float(sr[32 * c + 2 * i + 1])),
                                 scale2, neg_m2);
          float lo, hi;
          f2_split(x, lo, hi);
          lo = fast_exp2(lo);
          hi = fast_exp2(hi);
          ls2[i & 1] = f2_add(ls2[i & 1], f2_make(lo, hi));
          pr[i] = pack2<FMT>(lo, hi);
        }
        tmem_st16(tSw + c * 16, pr);
      }
      {
        float a0, a1;
        f2_split(f2_add(ls2[0], ls2[1]), a0, a1);
        l_run += a0 + a1;
      }
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + 2 * wg + hf);
    }
    if (n_mine > 0) {
      mbar_wait(o_done, 0, ctx, 810);
      __syncwarp();
      tc_fence_after_sync();
      // O through the group's Q tile in shared memory (no product reads it any more), so that
      // whole rows leave: 16-byte pieces XORed with the row on the way in.
      const float inv_l = 1.0f / l_run;
      constexpr int TPR = HD / 8;
      uint4* tile = reinterpret_cast<uint4*>(wg ? sQ[1] : sQ[0]);
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t orow[32];
        tmem_ld32(tOw + lane_base + c * 32, orow);
        tmem_wait_ld();
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          uint4 pk;
          pk.x = pack2<FMT>(__uint_as_float(orow[8 * v + 0]) * inv_l, __uint_as_float(orow[8 * v + 1]) * inv_l);
          pk.y = pack2<FMT>(__uint_as_float(orow[8 * v + 2]) * inv_l, __uint_as_float(orow[8 * v + 3]) * inv_l);
          pk.z = pack2<FMT>(__uint_as_float(orow[8 * v + 4]) * inv_l, __uint_as_float(orow[8 * v + 5]) * inv_l);
          pk.w = pack2<FMT>(__uint_as_float(orow[8 * v + 6]) * inv_l, __uint_as_float(orow[8 * v + 7]) * inv_l);
          tile[row * TPR + ((c * 4 + v) ^ (row & 7))] = pk;
        }
      }
      const bool row_ok = q_pos < L;
      const int64_t token = seq0 + (row_ok ? q_pos : 0);
      if (row_ok) p.lse[(int64_t)my_head * p.tokens + token] = (m_run + (log2f(l_run) - kPExponent)) * kLn2;
      named_barrier_sync(1 + wg, 128);
      uint8_t* out = reinterpret_cast<uint8_t*>(p.o) +
                     ((int64_t)(seq0 + my_tile * kTile) * p.o_st + (int64_t)my_head * p.o_sh) * 2;
      const int rows = min(kTile, L - my_tile * kTile);
#pragma unroll
      for (int i = (int)((threadIdx.x - 64) & 127); i < kTile * TPR; i += 128) {
        const int orow = i / TPR, piece = i % TPR;
        if (orow < rows && piece * 8 < p.D)
          *reinterpret_cast<uint4*>(out + (int64_t)orow * p.o_st * 2 + piece * 16) =
              tile[orow * TPR + (piece ^ (orow & 7))];
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 256 * TILES);
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

template <int HD, int FMT, int TILES>
int launch(const View& q, const View& k, const View& v, const FwdParams& p, int64_t Hq, int64_t Hkv,
           cudaStream_t stream) {
  CUtensorMap mq, mk, mv;
  if (!encode_view_map(&mq, q, FMT, p.D, p.tokens, Hq) ||
      !encode_view_map(&mk, k, FMT, p.D, p.tokens, Hkv) ||
      !encode_view_map(&mv, v, FMT, p.D, p.tokens, Hkv))
    return fail(EVG_ELAUNCH, "packed_attention_fwd: cuTensorMapEncodeTiled failed");
  const size_t smem = fwd_smem_tiles<HD, TILES>() * tile_bytes<HD>() + kControlBytes + 1024;
  auto kern = attn_packed_fwd_kernel<HD, FMT, TILES>;
  if (!allow_shared_memory((const void*)kern, smem))
    return fail(EVG_ELAUNCH, "packed_attention_fwd: cannot reserve %zu bytes of shared memory", smem);
  kern<<<(unsigned)((int64_t)p.slots * p.units), fwd_threads(TILES), smem, stream>>>(mq, mk, mv, p);
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
  // Two query tiles per block share their key tiles; with one, two blocks run on an SM and
  // nothing is idle that has no second tile. Measured, one | two, 16384 tokens:
  //   head size 64: one at every length (16/16 heads: 128 tokens a sequence 64 | 98 us, 1024
  //   88 | 102, 16384 729 | 822; 8/2 heads: 128 26 | 26, 1024 41 | 47, 16384 365 | 414)
  //   128, even group (32/8): 1 token 981 | 1208, 64 97 | 102, 512 156 | 154,
  //   2048 307 | 300, 16384 1912 | 1720
  //   128, odd group (9/3), where the second tile is the sequence's next: 64 28 | 46,
  //   512 50 | 58, 2048 107 | 109, 4096 190 | 187, 16384 706 | 651
  // The lengths stay on the device, so the rule goes by the mean over the offsets' entries: empty
  // entries, unused rows and short neighbours count, and one long document among many short ones
  // gets what is best for those (by this table up to 11 % slower for it).
  const int64_t two_from = p.pair_heads ? 256 : 4096;  // tokens per sequence
  const int tiles = D <= 64 || tokens < two_from * sequences ? 1 : 2;
  p.units = (int)(tiles == 2 && p.pair_heads ? Hq / 2 : Hq);
  p.head_group = head_group_for((int64_t)p.slots * p.units, p.units);
  p.scale_log2 = scale * kLog2e;
  const int t = tune("attention.wait_limit");
  p.wait_limit = t > 0 ? (long long)t * 1000000ll : 2000000000ll;
  if (D <= 64)
    return fmt == 1 ? launch<64, 1, 1>(q, k, v, p, Hq, Hkv, stream) : launch<64, 0, 1>(q, k, v, p, Hq, Hkv, stream);
  if (tiles == 1)
    return fmt == 1 ? launch<128, 1, 1>(q, k, v, p, Hq, Hkv, stream) : launch<128, 0, 1>(q, k, v, p, Hq, Hkv, stream);
  return fmt == 1 ? launch<128, 1, 2>(q, k, v, p, Hq, Hkv, stream) : launch<128, 0, 2>(q, k, v, p, Hq, Hkv, stream);
}

}  // namespace packed
}  // namespace evg
