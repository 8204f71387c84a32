// The two RMS norms around a block boundary, with the block's gate and residual scale,
// in one pass (sm_100a). x is the block's output, h the residual stream, both [rows, C]:
//   n  = x rstd1 w_post          rstd1 = (mean x^2 + eps)^-1/2
//   h' = h + alpha gate n        written, the new residual stream
//   y  = h' rstd2 w_pre          rstd2 = (mean h'^2 + eps)^-1/2, the next block's input
// y uses h' before it is rounded to the tensors' type. Backward, with the gradients dy
// of y and dh' of h' (all sums float32, one rounding per output):
//   G  = dh' + rstd2 (t - h'hat mean(t h'hat)),  t = dy w_pre,  h'hat = h' rstd2
//   dh = G,  dn = alpha gate G
//   dx = rstd1 (u - xhat mean(u xhat)),          u = dn w_post, xhat = x rstd1
//   dw_post = sum_rows dn xhat,  dw_pre = sum_rows dy h'hat,  dgate = alpha G n summed
// over what the gate was broadcast over. The gate is absent, [C], [rows] (one number per
// row) or [rows, C].
//
// HBM-bound: four passes over [rows, C] forward (x, h -> h', y), six backward (dy, dh',
// x, h' -> dx, dh), one more each way for a full gate, where the separate operators
// need eight and fourteen.
//
// A row belongs to one warp (up to 64 16-byte vectors) or to one block whose threads
// hold V vectors each; blocks are persistent, a thread keeps its columns for all its
// rows, so the weights and the column sums stay in registers. Column sums leave as one
// float32 partial row per block and are added by a second kernel in a fixed order.
#include "evg_common.cuh"

namespace evg {
namespace {

enum Gate { kNone = 0, kChannel = 1, kToken = 2, kFull = 3 };

struct NormArgs {
  const void *x, *h, *w_post, *w_pre, *gate;  // backward: h is the new stream h'
  void *h_out, *y;                            // forward
  const void *dy, *dh_in;                     // backward
  void *dx, *dh_out, *dgate;                  // dgate: token / full gates only
  float *rstd_post, *rstd_pre;
  float* partial;                             // [2][blocks][C]: dw_pre, dw_post sums
  int64_t rows, C;
  float alpha, eps, inv_c;
};

__device__ __forceinline__ uint4 ld_stream(const void* base, int64_t row, int64_t C, int vec, int elem_bytes) {
  return ld_vec(reinterpret_cast<const uint8_t*>(base) + row * C * elem_bytes + (int64_t)vec * 16);
}
__device__ __forceinline__ void st_stream(void* base, int64_t row, int64_t C, int vec, int elem_bytes, const uint4& v) {
  st_vec(reinterpret_cast<uint8_t*>(base) + row * C * elem_bytes + (int64_t)vec * 16, v);
}

// Sum of NV values over the row's threads: a warp, or the whole block (partials through
// shared memory, [2][NV][32] floats, one barrier: the halves alternate).
template <int NV, bool WARP>
__device__ __forceinline__ void row_sum(float (&v)[NV], float* scratch, int& phase) {
  if constexpr (WARP) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
  } else {
    block_allreduce<NV, SumOp>(v, scratch, phase);
  }
}

// ------------------------------------------------------------------ forward
template <typename T, int V, int GATE, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
post_pre_fwd_kernel(const NormArgs a) {
  constexpr int N = Vec<T>::N, E = sizeof(T);
  __shared__ float scratch[2 * 32];
  int phase = 0;
  const int lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int width = WARP ? 32 : blockDim.x;
  const int nvec = (int)(a.C / N);
  const int64_t stride = WARP ? (int64_t)gridDim.x * (blockDim.x / 32) : gridDim.x;
  int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
  int vec[V];
  bool on[V];
  uint4 wpost[V], wpre[V], gch[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    vec[j] = lane + j * width;
    on[j] = vec[j] < nvec;
    wpost[j] = wpre[j] = gch[j] = make_uint4(0, 0, 0, 0);
    if (on[j]) {
      wpost[j] = ld_vec((const uint8_t*)a.w_post + vec[j] * 16);
      wpre[j] = ld_vec((const uint8_t*)a.w_pre + vec[j] * 16);
      if (GATE == kChannel) gch[j] = ld_vec((const uint8_t*)a.gate + vec[j] * 16);
    }
  }
  uint4 xv[V], hv[V], gv[V];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (on[j]) {
        xv[j] = ld_stream(a.x, r, a.C, vec[j], E);
        hv[j] = ld_stream(a.h, r, a.C, vec[j], E);
        if (GATE == kFull) gv[j] = ld_stream(a.gate, r, a.C, vec[j], E);
      } else {
        xv[j] = hv[j] = gv[j] = make_uint4(0, 0, 0, 0);
      }
  };
  if (row < a.rows) fetch(row);
  for (; row < a.rows; row += stride) {
    float hn[V][N], x[V][N];
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      unpack<T>(xv[j], x[j]);
      unpack<T>(hv[j], hn[j]);
#pragma unroll
      for (int i = 0; i < N; ++i) s[0] = fmaf(x[j][i], x[j][i], s[0]);
    }
    const float gt = GATE == kToken ? to_f32<T>(((const T*)a.gate)[row]) : 1.f;
    uint4 gnow[V];
#pragma unroll
    for (int j = 0; j < V; ++j) gnow[j] = GATE == kFull ? gv[j] : gch[j];
    if (row + stride < a.rows) fetch(row + stride);  // the next row is on its way during the sums
    row_sum<1, WARP>(s, scratch, phase);
    const float r1 = rsqrtf(fmaf(s[0], a.inv_c, a.eps));
    const float scale = r1 * a.alpha * gt;
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float w[N], g[N];
      unpack<T>(wpost[j], w);
      if (GATE == kChannel || GATE == kFull) unpack<T>(gnow[j], g);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float n = x[j][i] * scale * w[i];
        if (GATE == kChannel || GATE == kFull) n *= g[i];
        hn[j][i] += n;
        s[0] = fmaf(hn[j][i], hn[j][i], s[0]);
      }
      if (on[j]) st_stream(a.h_out, row, a.C, vec[j], E, pack<T>(hn[j]));
    }
    row_sum<1, WARP>(s, scratch, phase);
    const float r2 = rsqrtf(fmaf(s[0], a.inv_c, a.eps));
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float w[N], y[N];
      unpack<T>(wpre[j], w);
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = hn[j][i] * r2 * w[i];
      if (on[j]) st_stream(a.y, row, a.C, vec[j], E, pack<T>(y));
    }
    if (lane == 0) {
      a.rstd_post[row] = r1;
      a.rstd_pre[row] = r2;
    }
  }
}

// ----------------------------------------------------------------- backward
template <typename T, int V, int GATE, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : (V == 1 ? 1024 : 512))
post_pre_bwd_kernel(const NormArgs a) {
  constexpr int N = Vec<T>::N, E = sizeof(T);
  extern __shared__ float fold[];  // WARP: one partial row, [2][C]
  __shared__ float scratch[2 * 2 * 32];
  int phase = 0;
  const int lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int width = WARP ? 32 : blockDim.x;
  const int nvec = (int)(a.C / N);
  const int64_t stride = WARP ? (int64_t)gridDim.x * (blockDim.x / 32) : gridDim.x;
  int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
  int vec[V];
  bool on[V];
  uint4 wpost[V], wpre[V], gch[V];
  float spost[V][N], spre[V][N];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    vec[j] = lane + j * width;
    on[j] = vec[j] < nvec;
    wpost[j] = wpre[j] = gch[j] = make_uint4(0, 0, 0, 0);
    if (on[j]) {
      wpost[j] = ld_vec((const uint8_t*)a.w_post + vec[j] * 16);
      wpre[j] = ld_vec((const uint8_t*)a.w_pre + vec[j] * 16);
      if (GATE == kChannel) gch[j] = ld_vec((const uint8_t*)a.gate + vec[j] * 16);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) spost[j][i] = spre[j][i] = 0.f;
  }
  for (; row < a.rows; row += stride) {
    uint4 yv[V], dv[V], xv[V], hv[V], gv[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      yv[j] = dv[j] = xv[j] = hv[j] = gv[j] = make_uint4(0, 0, 0, 0);
      if (on[j]) {
        yv[j] = ld_stream(a.dy, row, a.C, vec[j], E);
        hv[j] = ld_stream(a.h, row, a.C, vec[j], E);
        dv[j] = ld_stream(a.dh_in, row, a.C, vec[j], E);
        xv[j] = ld_stream(a.x, row, a.C, vec[j], E);
        if (GATE == kFull) gv[j] = ld_stream(a.gate, row, a.C, vec[j], E);
      }
    }
    const float r1 = a.rstd_post[row], r2 = a.rstd_pre[row];
    const float gt = GATE == kToken ? to_f32<T>(((const T*)a.gate)[row]) : 1.f;
    float s1[1] = {0.f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float dy[N], h[N], w[N];
      unpack<T>(yv[j], dy);
      unpack<T>(hv[j], h);
      unpack<T>(wpre[j], w);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float p = dy[i] * (h[i] * r2);
        spre[j][i] += p;
        s1[0] = fmaf(p, w[i], s1[0]);
      }
    }
    row_sum<1, WARP>(s1, scratch, phase);
    const float c1 = s1[0] * a.inv_c;
    float G[V][N];
    float s2[2] = {0.f, 0.f};  // sum u xhat; sum G n / alpha (token gate)
    const float ag = a.alpha * gt;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float dy[N], h[N], w[N], d[N], x[N], wp[N], g[N];
      unpack<T>(yv[j], dy);
      unpack<T>(hv[j], h);
      unpack<T>(wpre[j], w);
      unpack<T>(dv[j], d);
      unpack<T>(xv[j], x);
      unpack<T>(wpost[j], wp);
      if (GATE == kChannel) unpack<T>(gch[j], g);
      if (GATE == kFull) unpack<T>(gv[j], g);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        G[j][i] = fmaf(r2, fmaf(dy[i], w[i], -(h[i] * r2 * c1)), d[i]);
        const float q = G[j][i] * (x[i] * r1);  // G xhat
        const float qw = q * wp[i];
        const float gg = GATE == kChannel || GATE == kFull ? ag * g[i] : ag;
        // the column sum leaves out what does not depend on the row (a channel's gate)
        spost[j][i] = fmaf(q, GATE == kFull ? gg : ag, spost[j][i]);
        s2[0] = fmaf(qw, gg, s2[0]);
        if (GATE == kToken) s2[1] += qw;
        if (GATE == kFull) d[i] = a.alpha * qw;
      }
      if (on[j]) {
        st_stream(a.dh_out, row, a.C, vec[j], E, pack<T>(G[j]));
        if (GATE == kFull) st_stream(a.dgate, row, a.C, vec[j], E, pack<T>(d));
      }
    }
    row_sum<2, WARP>(s2, scratch, phase);
    const float c2 = s2[0] * a.inv_c;
    if (GATE == kToken && lane == 0) ((T*)a.dgate)[row] = from_f32<T>(a.alpha * s2[1]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float x[N], wp[N], g[N], o[N];
      unpack<T>(xv[j], x);
      unpack<T>(wpost[j], wp);
      if (GATE == kChannel) unpack<T>(gch[j], g);
      if (GATE == kFull) unpack<T>(gv[j], g);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float gg = GATE == kChannel || GATE == kFull ? ag * g[i] : ag;
        o[i] = r1 * fmaf(gg * G[j][i], wp[i], -(x[i] * r1 * c2));
      }
      if (on[j]) st_stream(a.dx, row, a.C, vec[j], E, pack<T>(o));
    }
  }
  // one float32 partial row per block
  float* pre = a.partial + (int64_t)blockIdx.x * a.C;
  float* post = a.partial + ((int64_t)gridDim.x + blockIdx.x) * a.C;
  if constexpr (!WARP) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (on[j])
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          *reinterpret_cast<float4*>(pre + vec[j] * N + i) = make_float4(spre[j][i], spre[j][i + 1], spre[j][i + 2], spre[j][i + 3]);
          *reinterpret_cast<float4*>(post + vec[j] * N + i) = make_float4(spost[j][i], spost[j][i + 1], spost[j][i + 2], spost[j][i + 3]);
        }
  } else {
    const int C = (int)a.C;  // at most 64 vectors
    for (int w = 0; w < (int)blockDim.x / 32; ++w) {  // the warps' rows in warp order
      if ((int)threadIdx.x / 32 == w) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (on[j])
#pragma unroll
            for (int i = 0; i < N; ++i) {
              float* f = fold + vec[j] * N + i;
              f[0] = w ? f[0] + spre[j][i] : spre[j][i];
              f[C] = w ? f[C] + spost[j][i] : spost[j][i];
            }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
      pre[c] = fold[c];
      post[c] = fold[C + c];
    }
  }
}

// ------------------------------------------------- any width, any alignment
// One block per row, three passes over the row (the later ones from L2); the column sums
// of the backward live in the block's own partial row.
constexpr int kAnyThreads = 256;

template <typename T>
__device__ __forceinline__ float gate_at(const NormArgs& a, int gate, int64_t row, int64_t c) {
  const T* g = (const T*)a.gate;
  return gate == kNone ? 1.f : to_f32<T>(g[gate == kChannel ? c : gate == kToken ? row : row * a.C + c]);
}

template <typename T>
__global__ void __launch_bounds__(kAnyThreads)
post_pre_fwd_any_kernel(const NormArgs a, int gate) {
  __shared__ float scratch[2 * 32];
  int phase = 0;
  const T *wp = (const T*)a.w_post, *wn = (const T*)a.w_pre;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = (const T*)a.x + row * a.C, *h = (const T*)a.h + row * a.C;
    float s[1] = {0.f};
    for (int64_t c = threadIdx.x; c < a.C; c += kAnyThreads) {
      const float v = to_f32<T>(x[c]);
      s[0] = fmaf(v, v, s[0]);
    }
    block_allreduce<1, SumOp>(s, scratch, phase);
    const float r1 = rsqrtf(fmaf(s[0], a.inv_c, a.eps));
    auto stream = [&](int64_t c) {
      return to_f32<T>(h[c]) + to_f32<T>(x[c]) * (r1 * a.alpha) * to_f32<T>(wp[c]) * gate_at<T>(a, gate, row, c);
    };
    s[0] = 0.f;
    for (int64_t c = threadIdx.x; c < a.C; c += kAnyThreads) {
      const float v = stream(c);
      s[0] = fmaf(v, v, s[0]);
    }
    block_allreduce<1, SumOp>(s, scratch, phase);
    const float r2 = rsqrtf(fmaf(s[0], a.inv_c, a.eps));
    for (int64_t c = threadIdx.x; c < a.C; c += kAnyThreads) {
      const float v = stream(c);
      ((T*)a.y)[row * a.C + c] = from_f32<T>(v * r2 * to_f32<T>(wn[c]));
      ((T*)a.h_out)[row * a.C + c] = from_f32<T>(v);
    }
    if (threadIdx.x == 0) {
      a.rstd_post[row] = r1;
      a.rstd_pre[row] = r2;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kAnyThreads)
post_pre_bwd_any_kernel(const NormArgs a, int gate) {
  __shared__ float scratch[2 * 2 * 32];
  int phase = 0;
  const T *wp = (const T*)a.w_post, *wn = (const T*)a.w_pre;
  float* pre = a.partial + (int64_t)blockIdx.x * a.C;
  float* post = a.partial + ((int64_t)gridDim.x + blockIdx.x) * a.C;
  for (int64_t c = threadIdx.x; c < a.C; c += kAnyThreads) pre[c] = post[c] = 0.f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = (const T*)a.x + row * a.C, *h = (const T*)a.h + row * a.C;
    const T *dy = (const T*)a.dy + row * a.C, *dh = (const T*)a.dh_in + row * a.C;
    const float r1 = a.rstd_post[row], r2 = a.rstd_pre[row];
    float s1[1] = {0.f};
    for (int64_t c = threadIdx.x; c < a.C; c += kAnyThreads) {
      const float p = to_f32<T>(dy[c]) * (to_f32<T>(h[c]) * r2);
      pre[c] += p;
      s1[0] = fmaf(p, to_f32<T>(wn[c]), s1[0]);
    }
    block_allreduce<1, SumOp>(s1, scratch, phase);
    const float c1 = s1[0] * a.inv_c;
    auto grad = [&](int64_t c) {
      return fmaf(r2, fmaf(to_f32<T>(dy[c]), to_f32<T>(wn[c]), -(to_f32<T>(h[c]) * r2 * c1)), to_f32<T>(dh[c]));
    };
    float s2[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x; c < a.C; c += kAnyThreads) {
      const float G = grad(c), q = G * (to_f32<T>(x[c]) * r1), qw = q * to_f32<T>(wp[c]);
      const float g = gate_at<T>(a, gate, row, c);
      post[c] = fmaf(q, gate == kChannel ? a.alpha : a.alpha * g, post[c]);
      s2[0] = fmaf(qw, a.alpha * g, s2[0]);
      s2[1] += qw;
      if (gate == kFull) ((T*)a.dgate)[row * a.C + c] = from_f32<T>(a.alpha * qw);
    }
    block_allreduce<2, SumOp>(s2, scratch, phase);
    const float c2 = s2[0] * a.inv_c;
    if (gate == kToken && threadIdx.x == 0) ((T*)a.dgate)[row] = from_f32<T>(a.alpha * s2[1]);
    for (int64_t c = threadIdx.x; c < a.C; c += kAnyThreads) {
      const float G = grad(c), gg = a.alpha * gate_at<T>(a, gate, row, c);
      ((T*)a.dx)[row * a.C + c] = from_f32<T>(r1 * fmaf(gg * G, to_f32<T>(wp[c]), -(to_f32<T>(x[c]) * r1 * c2)));
      ((T*)a.dh_out)[row * a.C + c] = from_f32<T>(G);
    }
  }
}

// Column sums: 32 columns x 8 slices of partial rows per block, added in a fixed order;
// dw_pre = S_pre, dw_post = S_post (times the channel's gate), dgate = w_post S_post.
template <typename T>
__global__ void __launch_bounds__(256)
post_pre_columns_kernel(const float* __restrict__ partial, int blocks, int64_t C,
                        const T* __restrict__ w_post, const T* __restrict__ gate_channel, T* dw_pre,
                        T* dw_post, T* dgate_channel) {
  __shared__ float part[8][33];
  const int which = blockIdx.y;
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  const float* src = partial + (int64_t)which * blocks * C;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < C) {
    int p = threadIdx.y;
    for (; p + 24 < blocks; p += 32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += src[(int64_t)(p + 8 * i) * C + c];
    }
    for (; p < blocks; p += 8) s[0] += src[(int64_t)p * C + c];
  }
  part[threadIdx.y][threadIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (threadIdx.y || c >= C) return;
  float sum = part[0][threadIdx.x];
#pragma unroll
  for (int i = 1; i < 8; ++i) sum += part[i][threadIdx.x];
  if (which == 0) {
    dw_pre[c] = from_f32<T>(sum);
  } else {
    dw_post[c] = from_f32<T>(gate_channel ? sum * to_f32<T>(gate_channel[c]) : sum);
    if (dgate_channel) dgate_channel[c] = from_f32<T>(sum * to_f32<T>(w_post[c]));
  }
}

// ---------------------------------------------------------------- host side
struct Shape {
  bool any;   // the kernels without vectors
  bool warp;  // a warp per row
  int V, threads;
};
// Vectors per thread: two from 257 vectors on (half the threads share each row's two
// reductions), four above 2048; a warp per row up to 64 vectors.
Shape pick_shape(int64_t C, size_t elem, bool aligned) {
  Shape s{};
  if (!aligned || (C * elem) % 16 != 0 || C * elem / 16 > 2048) {
    s.any = true;
    s.threads = kAnyThreads;
    return s;
  }
  const int nvec = (int)(C * elem / 16);
  if (nvec <= 64) {
    s.warp = true;
    s.V = nvec <= 32 ? 1 : 2;
    s.threads = 256;
    return s;
  }
  s.V = nvec <= 256 ? 1 : nvec <= 1024 ? 2 : 1;
  s.threads = (nvec + s.V - 1) / s.V;
  s.threads = (s.threads + 31) / 32 * 32;
  if (s.threads > 1024) { s.any = true; s.threads = kAnyThreads; }
  return s;
}
// Most blocks a backward launches, and with that partial rows.
int most_blocks() { return device_info().sm_count * 8; }

template <typename Kernel>
int blocks_for(Kernel kernel, const Shape& s, int64_t rows, size_t smem) {
  int occ = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kernel, s.threads, smem) != cudaSuccess) {
    cudaGetLastError();
    occ = 1;
  }
  if (occ < 1) occ = 1;
  int64_t n = (int64_t)device_info().sm_count * occ;
  const int64_t per = s.warp ? s.threads / 32 : 1;
  const int64_t need = (rows + per - 1) / per;
  if (n > need) n = need;
  if (n > most_blocks()) n = most_blocks();
  return (int)(n < 1 ? 1 : n);
}

template <typename T, int V, int GATE, bool WARP>
int launch_fwd(const NormArgs& a, const Shape& s, cudaStream_t st) {
  auto k = post_pre_fwd_kernel<T, V, GATE, WARP>;
  k<<<blocks_for(k, s, a.rows, 0), s.threads, 0, st>>>(a);
  return check_launch("post_pre_norm_fwd");
}
template <typename T, int V, int GATE, bool WARP>
int launch_bwd(const NormArgs& a, const Shape& s, cudaStream_t st, int& blocks) {
  auto k = post_pre_bwd_kernel<T, V, GATE, WARP>;
  const size_t smem = WARP ? 2 * a.C * sizeof(float) : 0;
  blocks = blocks_for(k, s, a.rows, smem);
  k<<<blocks, s.threads, smem, st>>>(a);
  return check_launch("post_pre_norm_bwd");
}

#define EVG_PP_GATES(call)                          \
  switch (gate) {                                   \
    case kNone: return call(kNone);                 \
    case kChannel: return call(kChannel);           \
    case kToken: return call(kToken);               \
    default: return call(kFull);                    \
  }

template <typename T>
int run_fwd(const NormArgs& a, int gate, const Shape& s, cudaStream_t st) {
  if (s.any) {
    post_pre_fwd_any_kernel<T><<<blocks_for(post_pre_fwd_any_kernel<T>, s, a.rows, 0), s.threads, 0, st>>>(a, gate);
    return check_launch("post_pre_norm_fwd");
  }
  if (s.warp && s.V == 1) {
#define EVG_PP(g) launch_fwd<T, 1, g, true>(a, s, st)
    EVG_PP_GATES(EVG_PP)
#undef EVG_PP
  }
  if (s.warp) {
#define EVG_PP(g) launch_fwd<T, 2, g, true>(a, s, st)
    EVG_PP_GATES(EVG_PP)
#undef EVG_PP
  }
  if (s.V == 1) {
#define EVG_PP(g) launch_fwd<T, 1, g, false>(a, s, st)
    EVG_PP_GATES(EVG_PP)
#undef EVG_PP
  }
#define EVG_PP(g) launch_fwd<T, 2, g, false>(a, s, st)
  EVG_PP_GATES(EVG_PP)
#undef EVG_PP
}

template <typename T>
int run_bwd_rows(const NormArgs& a, int gate, const Shape& s, cudaStream_t st, int& blocks) {
  if (s.any) {
    blocks = blocks_for(post_pre_bwd_any_kernel<T>, s, a.rows, 0);
    post_pre_bwd_any_kernel<T><<<blocks, s.threads, 0, st>>>(a, gate);
    return check_launch("post_pre_norm_bwd");
  }
  if (s.warp && s.V == 1) {
#define EVG_PP(g) launch_bwd<T, 1, g, true>(a, s, st, blocks)
    EVG_PP_GATES(EVG_PP)
#undef EVG_PP
  }
  if (s.warp) {
#define EVG_PP(g) launch_bwd<T, 2, g, true>(a, s, st, blocks)
    EVG_PP_GATES(EVG_PP)
#undef EVG_PP
  }
  if (s.V == 1) {
#define EVG_PP(g) launch_bwd<T, 1, g, false>(a, s, st, blocks)
    EVG_PP_GATES(EVG_PP)
#undef EVG_PP
  }
#define EVG_PP(g) launch_bwd<T, 2, g, false>(a, s, st, blocks)
  EVG_PP_GATES(EVG_PP)
#undef EVG_PP
}

int check_norm_args(const char* what, int64_t rows, int64_t C, int gate, float alpha, int dtype) {
  if (rows < 0 || C <= 0 || rows > 0x7fffffff || C > (1 << 26))
    return fail(EVG_EBADSHAPE, "%s: rows=%lld hidden=%lld", what, (long long)rows, (long long)C);
  if (gate < kNone || gate > kFull) return fail(EVG_EBADSHAPE, "%s: gate kind %d", what, gate);
  if (dtype != EVG_F32 && dtype != EVG_F16 && dtype != EVG_BF16) return fail(EVG_EDTYPE, "%s: dtype %d", what, dtype);
  (void)alpha;
  return EVG_OK;
}

}  // namespace
}  // namespace evg

using namespace evg;

extern "C" int evg_post_pre_norm_fwd(const void* x, const void* h, const void* w_post,
                                     const void* w_pre, const void* gate, int gate_kind, void* h_out,
                                     void* y, float* rstd_post, float* rstd_pre, int64_t rows,
                                     int64_t hidden, float alpha, float eps, int dtype, void* stream) {
  const char* what = "post_pre_norm_fwd";
  if (int rc = check_norm_args(what, rows, hidden, gate_kind, alpha, dtype)) return rc;
  if (rows == 0) return EVG_OK;
  if (!x || !h || !w_post || !w_pre || !h_out || !y || !rstd_post || !rstd_pre ||
      (gate_kind != kNone && !gate))
    return fail(EVG_ENULL, "%s: null pointer argument", what);
  NormArgs a{};
  a.x = x; a.h = h; a.w_post = w_post; a.w_pre = w_pre; a.gate = gate;
  a.h_out = h_out; a.y = y; a.rstd_post = rstd_post; a.rstd_pre = rstd_pre;
  a.rows = rows; a.C = hidden; a.alpha = alpha; a.eps = eps; a.inv_c = 1.0f / (float)hidden;
  bool aligned = true;
  for (const void* p : {x, h, w_post, w_pre, (const void*)h_out, (const void*)y}) aligned = aligned && aligned16(p);
  if (gate_kind == kChannel || gate_kind == kFull) aligned = aligned && aligned16(gate);
  const Shape s = pick_shape(hidden, dtype_size(dtype), aligned);
  return EVG_DISPATCH_DTYPE(dtype, [&] { return run_fwd<T>(a, gate_kind, s, (cudaStream_t)stream); });
}

extern "C" int64_t evg_post_pre_norm_bwd_workspace_bytes(int64_t rows, int64_t hidden) {
  if (rows <= 0 || hidden <= 0) return 0;
  int64_t blocks = most_blocks();
  if (blocks > rows) blocks = rows;
  return 2 * blocks * hidden * (int64_t)sizeof(float);
}

extern "C" int evg_post_pre_norm_bwd(const void* dy, const void* dh, const void* x, const void* h_out,
                                     const void* w_post, const void* w_pre, const void* gate,
                                     int gate_kind, const float* rstd_post, const float* rstd_pre,
                                     void* dx, void* dres, void* dw_post, void* dw_pre, void* dgate,
                                     void* workspace, int64_t workspace_bytes, int64_t rows,
                                     int64_t hidden, float alpha, int dtype, void* stream) {
  const char* what = "post_pre_norm_bwd";
  if (int rc = check_norm_args(what, rows, hidden, gate_kind, alpha, dtype)) return rc;
  if (rows == 0) return fail(EVG_EBADSHAPE, "%s: rows=0", what);
  if (!dy || !dh || !x || !h_out || !w_post || !w_pre || !rstd_post || !rstd_pre || !dx || !dres ||
      !dw_post || !dw_pre || (gate_kind != kNone && (!gate || !dgate)))
    return fail(EVG_ENULL, "%s: null pointer argument", what);
  const int64_t need = evg_post_pre_norm_bwd_workspace_bytes(rows, hidden);
  if (!workspace || workspace_bytes < need)
    return fail(EVG_EWORKSPACE, "%s: workspace %lld bytes, need %lld", what, (long long)workspace_bytes, (long long)need);
  if (!aligned16(workspace)) return fail(EVG_EALIGN, "%s: the workspace must be 16-byte aligned", what);
  NormArgs a{};
  a.x = x; a.h = h_out; a.w_post = w_post; a.w_pre = w_pre; a.gate = gate;
  a.dy = dy; a.dh_in = dh; a.dx = dx; a.dh_out = dres; a.dgate = dgate;
  a.rstd_post = const_cast<float*>(rstd_post); a.rstd_pre = const_cast<float*>(rstd_pre);
  a.partial = (float*)workspace;
  a.rows = rows; a.C = hidden; a.alpha = alpha; a.inv_c = 1.0f / (float)hidden;
  bool aligned = true;
  for (const void* p : {dy, dh, x, h_out, w_post, w_pre, (const void*)dx, (const void*)dres}) aligned = aligned && aligned16(p);
  if (gate_kind == kChannel) aligned = aligned && aligned16(gate);
  if (gate_kind == kFull) aligned = aligned && aligned16(gate) && aligned16(dgate);
  const Shape s = pick_shape(hidden, dtype_size(dtype), aligned);
  cudaStream_t st = (cudaStream_t)stream;
  return EVG_DISPATCH_DTYPE(dtype, [&] {
    int blocks = 0;
    if (int rc = run_bwd_rows<T>(a, gate_kind, s, st, blocks)) return rc;
    const bool channel = gate_kind == kChannel;
    post_pre_columns_kernel<T><<<dim3((unsigned)((hidden + 31) / 32), 2), dim3(32, 8), 0, st>>>(
        a.partial, blocks, hidden, (const T*)w_post, channel ? (const T*)gate : nullptr, (T*)dw_pre,
        (T*)dw_post, channel ? (T*)dgate : nullptr);
    return check_launch("post_pre_norm_bwd columns");
  });
}
