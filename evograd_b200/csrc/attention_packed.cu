// Packed causal attention: the C entry points, and CUDA-core kernels for what the
// tensor-core kernels do not take (float32, head sizes that are no multiple of eight
// or above 128, views that are not 16-byte aligned). One warp owns one row: a query
// row in the forward and in dQ, a key row in dK/dV; every sum has a fixed order.
// They are for small shapes: bound by the chain product -> softmax -> sum of 32 rows at a
// time, about 4.6 us per 32 keys forward, far from any unit's rate.
#include <cmath>

#include "packed.cuh"

namespace evg {
namespace packed {

int launch_fwd(const View& q, const View& k, const View& v, const View& o, float* lse,
               const void* plan, int64_t tokens, int64_t sequences, int64_t Hq, int64_t Hkv,
               int64_t D, float scale, int fmt, cudaStream_t stream);
int launch_bwd(const View& dout, const View& q, const View& k, const View& v, const View& o,
               const float* lse, const View& dq, const View& dk, const View& dv, void* workspace,
               const void* plan, int64_t tokens, int64_t sequences, int64_t Hq, int64_t Hkv,
               int64_t D, float scale, int fmt, cudaStream_t stream);
int64_t bwd_workspace_bytes(int64_t tokens, int64_t sequences, int64_t Hq, int64_t D);

namespace {

constexpr int kWarps = 8;

struct GenericParams {
  const int* plan;
  View q, k, v, o, dout, dq, dk, dv;
  float* lse_out;
  const float* lse;
  float* delta;  // [Hq][tokens]
  int tokens, group, D;
  float scale;
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename T>
__device__ __forceinline__ T* row_ptr(const View& v, int64_t token, int head) {
  return reinterpret_cast<T*>(v.p) + token * v.st + (int64_t)head * v.sh;
}
// 32 rows of a head as float32 in shared memory, `ld` floats apart, by the whole block; rows
// from `n` on and columns from D on are zeros.
template <typename T>
__device__ __forceinline__ void stage_rows(float* dst, int ld, const View& v, int64_t token, int n, int head, int D) {
  const int lane = threadIdx.x & 31, D4 = ld - 4;
#pragma unroll
  for (int k = 0; k < 32 / kWarps; ++k) {
    const int r = (threadIdx.x >> 5) + k * kWarps;
    const T* row = row_ptr<T>(v, token + (r < n ? r : 0), head);
    for (int d = lane; d < D4; d += 32) dst[r * ld + d] = r < n && d < D ? to_f32<T>(row[d]) : 0.f;
  }
}
// One row of a head as float32, by a warp; zeros from D on, or everywhere.
template <typename T>
__device__ __forceinline__ void stage_row(float* dst, const View& v, int64_t token, int head, int D, int D4, bool on) {
  for (int d = threadIdx.x & 31; d < D4; d += 32) dst[d] = on && d < D ? to_f32<T>(row_ptr<T>(v, token, head)[d]) : 0.f;
}
__device__ __forceinline__ float dot_rows(const float* a, const float* b, int D4) {
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int d = 0; d < D4; d += 4) {
    const float4 x = *reinterpret_cast<const float4*>(a + d), y = *reinterpret_cast<const float4*>(b + d);
    s[0] = fmaf(x.x, y.x, s[0]);
    s[1] = fmaf(x.y, y.y, s[1]);
    s[2] = fmaf(x.z, y.z, s[2]);
    s[3] = fmaf(x.w, y.w, s[3]);
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// What the kernels for any head size and type share: a warp owns a row of its item's tile
// (a query's, or in the last kernel a key's) and meets the other side's rows 32 at a time,
// one per lane for the products along the head, all of them for the sums along the rows.
// The block's rows share the 32 through shared memory; what a row does not see is skipped,
// not multiplied by zero. A sequence of 256 float32 tokens, 4/2 heads of 64: forward 37 us,
// backward 152 (153 and 615 with each warp reading the rows for itself).
struct Rows {
  float *a, *b;   // [32][ld]: staged rows of two tensors
  float *x, *y;   // the warp's own rows
  int ld, D4;
  int first, i;   // the block's first row inside the sequence, the warp's
  bool clear, active;
};
__device__ __forceinline__ bool block_rows(Rows& r, const int4& item, float* smem, int D) {
  const int warp = threadIdx.x >> 5;
  if (item.z < 0) return false;  // unused slot
  r.D4 = (D + 3) & ~3;
  r.ld = r.D4 + 4;
  r.a = smem;
  r.b = r.a + 32 * r.ld;
  r.x = r.b + 32 * r.ld + warp * r.D4;
  r.y = r.x + kWarps * r.D4;
  r.clear = item.z == 0;  // rows behind the last sequence
  r.first = (r.clear ? 0 : (item.z - 1) * attn::kTile) + blockIdx.z * kWarps;
  r.i = r.first + warp;
  r.active = r.i < item.y;
  return r.first < item.y;
}
size_t generic_smem(int64_t D, int rows_per_warp) {
  const int64_t D4 = (D + 3) / 4 * 4;
  return (size_t)(2 * 32 * (D4 + 4) + rows_per_warp * kWarps * D4) * sizeof(float);
}

template <typename T, int DT>
__global__ void __launch_bounds__(kWarps * 32)
packed_generic_fwd_kernel(const GenericParams p) {
  extern __shared__ __align__(16) float smem[];
  const int lane = threadIdx.x & 31, D = p.D, h = blockIdx.y, g = h / p.group;
  const int4 item = plan_item(p.plan, blockIdx.x);
  Rows r;
  if (!block_rows(r, item, smem, D)) return;
  const int64_t seq0 = item.x;
  const int i = r.i;
  T* orow = row_ptr<T>(p.o, seq0 + i, h);
  if (r.clear) {
    if (!r.active) return;
    for (int d = lane; d < D; d += 32) orow[d] = from_f32<T>(0.f);
    if (lane == 0) p.lse_out[(int64_t)h * p.tokens + seq0 + i] = -INFINITY;
    return;
  }
  stage_row<T>(r.x, p.q, seq0 + i, h, D, r.D4, r.active);
  float m = -INFINITY, l = 0.f;
  float acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = 0.f;
  const int last = min(r.first + kWarps, item.y) - 1;
  for (int j0 = 0; j0 <= last; j0 += 32) {
    __syncthreads();
    stage_rows<T>(r.a, r.ld, p.k, seq0 + j0, min(32, item.y - j0), g, D);
    stage_rows<T>(r.b, r.ld, p.v, seq0 + j0, min(32, item.y - j0), g, D);
    __syncthreads();
    if (!r.active || j0 > i) continue;
    const int j = j0 + lane;
    const float s = j <= i ? p.scale * dot_rows(r.x, r.a + lane * r.ld, r.D4) : -INFINITY;
    const float m_new = fmaxf(m, warp_max(s));
    const float corr = m_new == m ? 1.f : expf(m - m_new);  // 0 on the first chunk
    // (scores of -infinity are zero weights, also while a row has seen nothing else)
    const float pr = j <= i ? expf(s - (m_new == -INFINITY ? 0.f : m_new)) : 0.f;
    l = l * corr + warp_sum(pr);
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] *= corr;
    const int n = min(32, i - j0 + 1);
#pragma unroll 8
    for (int jj = 0; jj < n; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, pr, jj);
#pragma unroll
      for (int t = 0; t < DT; ++t)
        if (lane + 32 * t < D) acc[t] = fmaf(pj, r.b[jj * r.ld + lane + 32 * t], acc[t]);
    }
    m = m_new;
  }
  if (!r.active) return;
  const float inv = 1.0f / l;
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    const int d = lane + 32 * t;
    if (d < D) orow[d] = from_f32<T>(acc[t] * inv);
  }
  if (lane == 0) p.lse_out[(int64_t)h * p.tokens + seq0 + i] = m + logf(l);
}

// delta_i = sum_{j<=i} p_ij do_i.v_j (from its definition: o is rounded), and dq of the row:
// dq_i = scale * sum_{j<=i} p_ij (do_i.v_j - delta_i) k_j
template <typename T, int DT>
__global__ void __launch_bounds__(kWarps * 32)
packed_generic_dq_kernel(const GenericParams p) {
  extern __shared__ __align__(16) float smem[];
  const int lane = threadIdx.x & 31, D = p.D, h = blockIdx.y, g = h / p.group;
  const int4 item = plan_item(p.plan, blockIdx.x);
  Rows r;
  if (!block_rows(r, item, smem, D)) return;
  const int64_t seq0 = item.x;
  const int i = r.i;
  const float ds_scale = item.y > 1 ? p.scale : 0.f;  // a lone token's dS is zero
  T* out = row_ptr<T>(p.dq, seq0 + i, h);
  if (r.clear) {
    if (r.active)
      for (int d = lane; d < D; d += 32) out[d] = from_f32<T>(0.f);
    return;
  }
  stage_row<T>(r.x, p.q, seq0 + i, h, D, r.D4, r.active);
  stage_row<T>(r.y, p.dout, seq0 + i, h, D, r.D4, r.active);
  const int64_t stat = (int64_t)h * p.tokens + seq0 + i;
  const float lse_i = r.active ? p.lse[stat] : 0.f;
  float delta_i = 0.f;
  float acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = 0.f;
  const int last = min(r.first + kWarps, item.y) - 1;
  for (int pass = 0; pass < 2; ++pass) {
    float sum = 0.f;
    for (int j0 = 0; j0 <= last; j0 += 32) {
      if (pass == 0 || last >= 32) {  // (32 rows are still there)
        __syncthreads();
        stage_rows<T>(r.a, r.ld, p.k, seq0 + j0, min(32, item.y - j0), g, D);
        stage_rows<T>(r.b, r.ld, p.v, seq0 + j0, min(32, item.y - j0), g, D);
        __syncthreads();
      }
      if (!r.active || j0 > i) continue;
      float pr = 0.f, dp = 0.f;
      if (j0 + lane <= i) {
        pr = expf(p.scale * dot_rows(r.x, r.a + lane * r.ld, r.D4) - lse_i);
        dp = dot_rows(r.y, r.b + lane * r.ld, r.D4);
      }
      if (pass == 0) {
        sum += pr * dp;
        continue;
      }
      const float ds = j0 + lane <= i ? pr * (dp - delta_i) : 0.f;
      const int n = min(32, i - j0 + 1);
#pragma unroll 8
      for (int jj = 0; jj < n; ++jj) {
        const float dj = __shfl_sync(0xffffffffu, ds, jj);
#pragma unroll
        for (int t = 0; t < DT; ++t)
          if (lane + 32 * t < D) acc[t] = fmaf(dj, r.a[jj * r.ld + lane + 32 * t], acc[t]);
      }
    }
    if (pass == 0) delta_i = warp_sum(sum);
  }
  if (!r.active) return;
  if (lane == 0) p.delta[stat] = delta_i;
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    const int d = lane + 32 * t;
    if (d < D) out[d] = from_f32<T>(acc[t] * ds_scale);
  }
}

// One key row: dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i over i >= j of the
// sequence and the query heads of the group, in that order.
template <typename T, int DT>
__global__ void __launch_bounds__(kWarps * 32)
packed_generic_dkdv_kernel(const GenericParams p) {
  extern __shared__ __align__(16) float smem[];
  const int lane = threadIdx.x & 31, D = p.D, g = blockIdx.y;
  const int4 item = plan_item(p.plan, blockIdx.x);
  Rows r;
  if (!block_rows(r, item, smem, D)) return;
  const int64_t seq0 = item.x;
  const int j = r.i, L = item.y;
  T* dk = row_ptr<T>(p.dk, seq0 + j, g);
  T* dv = row_ptr<T>(p.dv, seq0 + j, g);
  if (r.clear) {
    if (r.active)
      for (int d = lane; d < D; d += 32) dk[d] = dv[d] = from_f32<T>(0.f);
    return;
  }
  stage_row<T>(r.x, p.k, seq0 + j, g, D, r.D4, r.active);
  stage_row<T>(r.y, p.v, seq0 + j, g, D, r.D4, r.active);
  float ak[DT], av[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) ak[t] = av[t] = 0.f;
  const float ds_scale = L > 1 ? p.scale : 0.f;  // a lone token's dS is zero
  for (int h = g * p.group; h < (g + 1) * p.group; ++h) {
    for (int i0 = r.first; i0 < L; i0 += 32) {
      __syncthreads();
      stage_rows<T>(r.a, r.ld, p.q, seq0 + i0, min(32, L - i0), h, D);
      stage_rows<T>(r.b, r.ld, p.dout, seq0 + i0, min(32, L - i0), h, D);
      __syncthreads();
      if (!r.active) continue;
      const int i = i0 + lane;
      float pr = 0.f, ds = 0.f;
      if (i >= j && i < L) {
        const int64_t stat = (int64_t)h * p.tokens + seq0 + i;
        pr = expf(p.scale * dot_rows(r.x, r.a + lane * r.ld, r.D4) - p.lse[stat]);
        ds = pr * (dot_rows(r.y, r.b + lane * r.ld, r.D4) - p.delta[stat]);
      }
      const int n = min(32, L - i0);
#pragma unroll 8
      for (int ii = max(j - i0, 0); ii < n; ++ii) {
        const float pi = __shfl_sync(0xffffffffu, pr, ii), di = __shfl_sync(0xffffffffu, ds, ii);
#pragma unroll
        for (int t = 0; t < DT; ++t)
          if (lane + 32 * t < D) {
            ak[t] = fmaf(di, r.a[ii * r.ld + lane + 32 * t], ak[t]);
            av[t] = fmaf(pi, r.b[ii * r.ld + lane + 32 * t], av[t]);
          }
      }
    }
  }
  if (!r.active) return;
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    const int d = lane + 32 * t;
    if (d < D) {
      dk[d] = from_f32<T>(ak[t] * ds_scale);
      dv[d] = from_f32<T>(av[t]);
    }
  }
}

View view_of(const evg_packed_view* v) {
  View r;
  r.p = v->data;
  r.st = v->stride_t;
  r.sh = v->stride_h;
  return r;
}

// What the TMA maps and the 16-byte stores need of a view.
bool tile_view(const View& v) { return aligned16(v.p) && v.st % 8 == 0 && v.sh % 8 == 0; }

bool tensor_core_shape(int64_t D, int dtype) {
  return dtype != EVG_F32 && D % 8 == 0 && D <= 128;
}

int check_args(const char* what, const void* plan, int64_t tokens, int64_t sequences, int64_t Hq,
               int64_t Hkv, int64_t D, float scale, int dtype) {
  if (!plan) return fail(EVG_ENULL, "%s: null plan", what);
  if (!aligned16(plan)) return fail(EVG_EALIGN, "%s: the plan must be 16-byte aligned", what);
  if (!(scale > 0.f) || !std::isfinite(scale))
    return fail(EVG_EUNSUPPORTED, "%s: scale %g (must be positive and finite)", what, (double)scale);
  if (tokens < 0 || sequences < 0 || tokens > EVG_PACKED_MAX_TOKENS || sequences > EVG_PACKED_MAX_TOKENS)
    return fail(EVG_EBADSHAPE, "%s: tokens=%lld sequences=%lld (0 .. %d each)", what,
                (long long)tokens, (long long)sequences, EVG_PACKED_MAX_TOKENS);
  if (Hq <= 0 || Hkv <= 0 || D <= 0)
    return fail(EVG_EBADSHAPE, "%s: Hq=%lld Hkv=%lld D=%lld must be positive", what, (long long)Hq,
                (long long)Hkv, (long long)D);
  if (Hq % Hkv != 0)
    return fail(EVG_EBADSHAPE, "%s: %lld query heads are not a multiple of %lld k/v heads", what,
                (long long)Hq, (long long)Hkv);
  if (dtype != EVG_BF16 && dtype != EVG_F16 && dtype != EVG_F32)
    return fail(EVG_EDTYPE, "%s: dtype %d", what, dtype);
  if (D > 256) return fail(EVG_EUNSUPPORTED, "%s: head size %lld > 256", what, (long long)D);
  // one grid dimension of the row kernels is the head; another is tiles x heads
  if (Hq > 65535 || plan_slots(tokens, sequences) * Hq > 0x7fffffff)
    return fail(EVG_EUNSUPPORTED, "%s: %lld heads x %lld tokens is beyond one launch", what,
                (long long)Hq, (long long)tokens);
  return EVG_OK;
}

// Blocks read the inputs while others write: an output may not be an input or another output.
int check_outputs(const char* what, const evg_packed_view* const* views, int inputs, int count) {
  for (int i = inputs; i < count; ++i)
    for (int j = 0; j < i; ++j)
      if (views[i]->data == views[j]->data)
        return fail(EVG_EBADSHAPE, "%s: an output starts where another tensor does", what);
  return EVG_OK;
}

template <typename Kernel>
int launch_generic(const char* what, Kernel kernel, const GenericParams& p, int64_t slots,
                   int64_t heads, int rows_per_warp, cudaStream_t stream) {
  const dim3 grid((unsigned)slots, (unsigned)heads, (unsigned)(attn::kTile / kWarps));
  const size_t smem = generic_smem(p.D, rows_per_warp);
  if (smem > 48 * 1024 && !allow_shared_memory((const void*)kernel, smem))
    return fail(EVG_ELAUNCH, "%s: cannot reserve %zu bytes of shared memory", what, smem);
  kernel<<<grid, kWarps * 32, smem, stream>>>(p);
  return check_launch(what);
}
// Columns of 32 a head needs: `f` gets it as a constant, rounded up to 2, 4 or 8.
template <typename F> int with_columns(int64_t D, F f) {
  if (D <= 64) return f(std::integral_constant<int, 2>{});
  if (D <= 128) return f(std::integral_constant<int, 4>{});
  return f(std::integral_constant<int, 8>{});
}

}  // namespace
}  // namespace packed
}  // namespace evg

using namespace evg;
using namespace evg::packed;

extern "C" int evg_packed_attention_fwd(const evg_packed_view* q, const evg_packed_view* k,
                                        const evg_packed_view* v, const evg_packed_view* o,
                                        float* lse, const void* plan, int64_t tokens,
                                        int64_t sequences, int64_t Hq, int64_t Hkv, int64_t D,
                                        float scale, int dtype, void* stream) {
  const char* what = "packed_attention_fwd";
  if (!q || !k || !v || !o) return fail(EVG_ENULL, "%s: null view", what);
  if (int rc = check_args(what, plan, tokens, sequences, Hq, Hkv, D, scale, dtype)) return rc;
  if (tokens == 0) return EVG_OK;
  if (!q->data || !k->data || !v->data || !o->data || !lse)
    return fail(EVG_ENULL, "%s: null pointer argument", what);
  const evg_packed_view* views[4] = {q, k, v, o};
  if (int rc = check_outputs(what, views, 3, 4)) return rc;
  const View vq = view_of(q), vk = view_of(k), vv = view_of(v), vo = view_of(o);
  cudaStream_t st = (cudaStream_t)stream;
  if (tensor_core_shape(D, dtype) && tile_view(vq) && tile_view(vk) && tile_view(vv) && tile_view(vo))
    return launch_fwd(vq, vk, vv, vo, lse, plan, tokens, sequences, Hq, Hkv, D, scale,
                      dtype == EVG_BF16 ? 1 : 0, st);
  GenericParams p{};
  p.plan = (const int*)plan;
  p.q = vq; p.k = vk; p.v = vv; p.o = vo;
  p.lse_out = lse;
  p.tokens = (int)tokens;
  p.group = (int)(Hq / Hkv);
  p.D = (int)D;
  p.scale = scale;
  const int64_t slots = plan_slots(tokens, sequences);
  return EVG_DISPATCH_DTYPE(dtype, [&] {
    return with_columns(D, [&](auto dt) {
      return launch_generic(what, packed_generic_fwd_kernel<T, decltype(dt)::value>, p, slots, Hq, 1, st);
    });
  });
}

extern "C" int64_t evg_packed_attention_bwd_workspace_bytes(int64_t tokens, int64_t sequences,
                                                            int64_t Hq, int64_t D) {
  if (tokens <= 0 || sequences < 0 || Hq <= 0 || D <= 0 || tokens > EVG_PACKED_MAX_TOKENS ||
      sequences > EVG_PACKED_MAX_TOKENS)
    return 0;
  return bwd_workspace_bytes(tokens, sequences, Hq, D);  // also covers the CUDA-core path
}

extern "C" int evg_packed_attention_bwd(const evg_packed_view* dout, const evg_packed_view* q,
                                        const evg_packed_view* k, const evg_packed_view* v,
                                        const evg_packed_view* o, const float* lse,
                                        const evg_packed_view* dq, const evg_packed_view* dk,
                                        const evg_packed_view* dv, void* workspace,
                                        int64_t workspace_bytes, const void* plan, int64_t tokens,
                                        int64_t sequences, int64_t Hq, int64_t Hkv, int64_t D,
                                        float scale, int dtype, void* stream) {
  const char* what = "packed_attention_bwd";
  const evg_packed_view* views[8] = {dout, q, k, v, o, dq, dk, dv};
  for (const evg_packed_view* x : views)
    if (!x) return fail(EVG_ENULL, "%s: null view", what);
  if (int rc = check_args(what, plan, tokens, sequences, Hq, Hkv, D, scale, dtype)) return rc;
  if (tokens == 0) return EVG_OK;
  bool tiles = tensor_core_shape(D, dtype);
  for (const evg_packed_view* x : views) {
    if (!x->data) return fail(EVG_ENULL, "%s: null pointer argument", what);
    tiles = tiles && tile_view(view_of(x));
  }
  if (!lse) return fail(EVG_ENULL, "%s: null pointer argument", what);
  const int64_t need = evg_packed_attention_bwd_workspace_bytes(tokens, sequences, Hq, D);
  if (!workspace || workspace_bytes < need)
    return fail(EVG_EWORKSPACE, "%s: workspace %lld bytes, need %lld", what,
                (long long)workspace_bytes, (long long)need);
  if (!aligned16(workspace)) return fail(EVG_EALIGN, "%s: the workspace must be 16-byte aligned", what);
  if (int rc = check_outputs(what, views, 5, 8)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (tiles)
    return launch_bwd(view_of(dout), view_of(q), view_of(k), view_of(v), view_of(o), lse,
                      view_of(dq), view_of(dk), view_of(dv), workspace, plan, tokens, sequences, Hq,
                      Hkv, D, scale, dtype == EVG_BF16 ? 1 : 0, st);
  GenericParams p{};
  p.plan = (const int*)plan;
  p.dout = view_of(dout); p.q = view_of(q); p.k = view_of(k); p.v = view_of(v); p.o = view_of(o);
  p.dq = view_of(dq); p.dk = view_of(dk); p.dv = view_of(dv);
  p.lse = lse;
  p.delta = (float*)workspace;
  p.tokens = (int)tokens;
  p.group = (int)(Hq / Hkv);
  p.D = (int)D;
  p.scale = scale;
  const int64_t slots = plan_slots(tokens, sequences);
  return EVG_DISPATCH_DTYPE(dtype, [&] {
    return with_columns(D, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      if (int rc = launch_generic(what, packed_generic_dq_kernel<T, DT>, p, slots, Hq, 2, st)) return rc;
      return launch_generic(what, packed_generic_dkdv_kernel<T, DT>, p, slots, Hkv, 2, st);
    });
  });
}
