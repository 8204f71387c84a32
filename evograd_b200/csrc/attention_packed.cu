// Packed causal attention: the C entry points, and CUDA-core kernels for what the
// tensor-core kernels do not take (float32, head sizes that are no multiple of eight
// or above 128, views that are not 16-byte aligned). One warp owns one row: a query
// row in the forward and in dQ, a key row in dK/dV; every sum has a fixed order.
// These are the small correctness shapes; nothing here is tuned for speed.
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

constexpr int kWarps = 4;
constexpr int kMaxDT = 8;  // head size <= 256

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
template <typename T>
__device__ __forceinline__ float dot_row(const float* a_smem, const T* b_row, int D) {
  float s = 0.f;
  for (int d = 0; d < D; ++d) s = fmaf(a_smem[d], to_f32<T>(b_row[d]), s);
  return s;
}
// The row of (item, row block) this warp owns: false when there is none. i: position in
// the sequence (or token behind the last one, seq0 = that token, for items of weight 0).
__device__ __forceinline__ bool my_row(const int4& item, int& i) {
  if (item.z < 0) return false;
  i = (item.z > 0 ? (item.z - 1) * attn::kTile : 0) + blockIdx.z * kWarps + (threadIdx.x >> 5);
  return i < item.y && (int)(blockIdx.z * kWarps + (threadIdx.x >> 5)) < attn::kTile;
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
packed_generic_fwd_kernel(const GenericParams p) {
  extern __shared__ float smem[];
  const int lane = threadIdx.x & 31, D = p.D, h = blockIdx.y, g = h / p.group;
  float* qs = smem + (threadIdx.x >> 5) * D;
  const int4 item = plan_item(p.plan, blockIdx.x);
  int i;
  if (!my_row(item, i)) return;
  const int64_t seq0 = item.x;
  T* orow = row_ptr<T>(p.o, seq0 + i, h);
  if (item.z == 0) {
    for (int d = lane; d < D; d += 32) orow[d] = from_f32<T>(0.f);
    if (lane == 0) p.lse_out[(int64_t)h * p.tokens + seq0 + i] = -INFINITY;
    return;
  }
  const T* qr = row_ptr<T>(p.q, seq0 + i, h);
  for (int d = lane; d < D; d += 32) qs[d] = to_f32<T>(qr[d]);
  __syncwarp();
  float m = -INFINITY, l = 0.f;
  float acc[kMaxDT];
#pragma unroll
  for (int t = 0; t < kMaxDT; ++t) acc[t] = 0.f;
  for (int j0 = 0; j0 <= i; j0 += 32) {
    const int j = j0 + lane;
    const float s = j <= i ? p.scale * dot_row<T>(qs, row_ptr<T>(p.k, seq0 + j, g), D) : -INFINITY;
    const float m_new = fmaxf(m, warp_max(s));
    const float corr = m_new == m ? 1.f : expf(m - m_new);  // 0 on the first chunk
    const float pr = j <= i ? expf(s - m_new) : 0.f;
    l = l * corr + warp_sum(pr);
#pragma unroll
    for (int t = 0; t < kMaxDT; ++t) acc[t] *= corr;
    const int n = min(32, i - j0 + 1);
    for (int jj = 0; jj < n; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, pr, jj);
      const T* vr = row_ptr<T>(p.v, seq0 + j0 + jj, g);
#pragma unroll
      for (int t = 0; t < kMaxDT; ++t) {
        const int d = lane + 32 * t;
        if (d < D) acc[t] = fmaf(pj, to_f32<T>(vr[d]), acc[t]);
      }
    }
    m = m_new;
  }
  const float inv = 1.0f / l;
#pragma unroll
  for (int t = 0; t < kMaxDT; ++t) {
    const int d = lane + 32 * t;
    if (d < D) orow[d] = from_f32<T>(acc[t] * inv);
  }
  if (lane == 0) p.lse_out[(int64_t)h * p.tokens + seq0 + i] = m + logf(l);
}

// delta_i = sum_{j<=i} p_ij do_i.v_j (from its definition: o is rounded), and dq of the row:
// dq_i = scale * sum_{j<=i} p_ij (do_i.v_j - delta_i) k_j
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
packed_generic_dq_kernel(const GenericParams p) {
  extern __shared__ float smem[];
  const int lane = threadIdx.x & 31, D = p.D, h = blockIdx.y, g = h / p.group;
  float* qs = smem + (threadIdx.x >> 5) * 2 * D;
  float* gs = qs + D;
  const int4 item = plan_item(p.plan, blockIdx.x);
  int i;
  if (!my_row(item, i)) return;
  const int64_t seq0 = item.x;
  const float ds_scale = item.y > 1 ? p.scale : 0.f;  // a lone token's dS is zero
  T* out = row_ptr<T>(p.dq, seq0 + i, h);
  if (item.z == 0) {
    for (int d = lane; d < D; d += 32) out[d] = from_f32<T>(0.f);
    return;
  }
  const T* qr = row_ptr<T>(p.q, seq0 + i, h);
  const T* gr = row_ptr<T>(p.dout, seq0 + i, h);
  for (int d = lane; d < D; d += 32) {
    qs[d] = to_f32<T>(qr[d]);
    gs[d] = to_f32<T>(gr[d]);
  }
  __syncwarp();
  const int64_t stat = (int64_t)h * p.tokens + seq0 + i;
  const float lse_i = p.lse[stat];
  float sum = 0.f;
  for (int j = lane; j <= i; j += 32)
    sum += expf(p.scale * dot_row<T>(qs, row_ptr<T>(p.k, seq0 + j, g), D) - lse_i) *
           dot_row<T>(gs, row_ptr<T>(p.v, seq0 + j, g), D);
  const float delta_i = warp_sum(sum);
  if (lane == 0) p.delta[stat] = delta_i;
  float acc[kMaxDT];
#pragma unroll
  for (int t = 0; t < kMaxDT; ++t) acc[t] = 0.f;
  for (int j0 = 0; j0 <= i; j0 += 32) {
    const int j = j0 + lane;
    float ds = 0.f;
    if (j <= i) {
      const float pr = expf(p.scale * dot_row<T>(qs, row_ptr<T>(p.k, seq0 + j, g), D) - lse_i);
      ds = pr * (dot_row<T>(gs, row_ptr<T>(p.v, seq0 + j, g), D) - delta_i);
    }
    const int n = min(32, i - j0 + 1);
    for (int jj = 0; jj < n; ++jj) {
      const float dj = __shfl_sync(0xffffffffu, ds, jj);
      const T* kr = row_ptr<T>(p.k, seq0 + j0 + jj, g);
#pragma unroll
      for (int t = 0; t < kMaxDT; ++t) {
        const int d = lane + 32 * t;
        if (d < D) acc[t] = fmaf(dj, to_f32<T>(kr[d]), acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kMaxDT; ++t) {
    const int d = lane + 32 * t;
    if (d < D) out[d] = from_f32<T>(acc[t] * ds_scale);
  }
}

// One key row: dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i over i >= j of the
// sequence and the query heads of the group, in that order.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
packed_generic_dkdv_kernel(const GenericParams p) {
  extern __shared__ float smem[];
  const int lane = threadIdx.x & 31, D = p.D, g = blockIdx.y;
  float* ks = smem + (threadIdx.x >> 5) * 2 * D;
  float* vs = ks + D;
  const int4 item = plan_item(p.plan, blockIdx.x);
  int j;
  if (!my_row(item, j)) return;
  const int64_t seq0 = item.x;
  T* dk = row_ptr<T>(p.dk, seq0 + j, g);
  T* dv = row_ptr<T>(p.dv, seq0 + j, g);
  if (item.z == 0) {
    for (int d = lane; d < D; d += 32) dk[d] = dv[d] = from_f32<T>(0.f);
    return;
  }
  const T* kr = row_ptr<T>(p.k, seq0 + j, g);
  const T* vr = row_ptr<T>(p.v, seq0 + j, g);
  for (int d = lane; d < D; d += 32) {
    ks[d] = to_f32<T>(kr[d]);
    vs[d] = to_f32<T>(vr[d]);
  }
  __syncwarp();
  float ak[kMaxDT], av[kMaxDT];
#pragma unroll
  for (int t = 0; t < kMaxDT; ++t) ak[t] = av[t] = 0.f;
  const int L = item.y;
  const float ds_scale = L > 1 ? p.scale : 0.f;  // a lone token's dS is zero
  for (int h = g * p.group; h < (g + 1) * p.group; ++h) {
    for (int i0 = j; i0 < L; i0 += 32) {
      const int i = i0 + lane;
      float pr = 0.f, ds = 0.f;
      if (i < L) {
        const int64_t stat = (int64_t)h * p.tokens + seq0 + i;
        pr = expf(p.scale * dot_row<T>(ks, row_ptr<T>(p.q, seq0 + i, h), D) - p.lse[stat]);
        ds = pr * (dot_row<T>(vs, row_ptr<T>(p.dout, seq0 + i, h), D) - p.delta[stat]);
      }
      const int n = min(32, L - i0);
      for (int ii = 0; ii < n; ++ii) {
        const float pi = __shfl_sync(0xffffffffu, pr, ii), di = __shfl_sync(0xffffffffu, ds, ii);
        const T* qr = row_ptr<T>(p.q, seq0 + i0 + ii, h);
        const T* gr = row_ptr<T>(p.dout, seq0 + i0 + ii, h);
#pragma unroll
        for (int t = 0; t < kMaxDT; ++t) {
          const int d = lane + 32 * t;
          if (d < D) {
            ak[t] = fmaf(di, to_f32<T>(qr[d]), ak[t]);
            av[t] = fmaf(pi, to_f32<T>(gr[d]), av[t]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kMaxDT; ++t) {
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

template <typename Kernel>
int launch_generic(const char* what, Kernel kernel, const GenericParams& p, int64_t slots,
                   int64_t heads, int smem_rows, cudaStream_t stream) {
  const dim3 grid((unsigned)slots, (unsigned)heads, (unsigned)(attn::kTile / kWarps));
  kernel<<<grid, kWarps * 32, (size_t)smem_rows * kWarps * p.D * sizeof(float), stream>>>(p);
  return check_launch(what);
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
    return launch_generic(what, packed_generic_fwd_kernel<T>, p, slots, Hq, 1, st);
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
    if (int rc = launch_generic(what, packed_generic_dq_kernel<T>, p, slots, Hq, 2, st)) return rc;
    return launch_generic(what, packed_generic_dkdv_kernel<T>, p, slots, Hkv, 2, st);
  });
}
