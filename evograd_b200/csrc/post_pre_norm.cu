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
// x, h' -> dx, dh), one more forward and two backward for a full gate, where the separate
// operators need eight and fourteen. [16384, 4096] bf16 with a channel gate: forward 87 us
// (6.2 TB/s), backward 136 us (5.9 TB/s with its column sums).
//
// A row belongs to one warp (up to 64 16-byte vectors) or to one block whose threads
// hold V vectors each and whose next rows come through a shared-memory ring; blocks are
// persistent, a thread keeps its columns for all its rows, so the weights and the column
// sums stay in registers. Column sums leave as one float32 partial row per block and are
// added by a second kernel in a fixed order.
#include "evg_common.cuh"
#include "shared_memory.cuh"
#include "sm100_umma.cuh"

namespace evg {

__device__ int g_post_pre_device_status = 0;

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
  int stages;                                 // of the ring
};

// How a row reaches its threads.
//   kWarp    a warp per row, global loads (rows of up to 64 16-byte vectors)
//   kDirect  a block per row, global loads (rows of more than 1024 vectors: four per thread)
//   kRing    a block per row; the block's next rows are on their way into a ring of
//            shared-memory stages (untiled bulk copies, one issuing thread, bounded waits)
enum Mode { kWarp = 0, kDirect = 1, kRing = 2 };
constexpr int kMaxStages = 2;
constexpr long long kWaitCycles = 2000000000ll;

struct Ring {
  uint64_t full[kMaxStages];
  int abort_flag;
};

template <int N_ARRAYS, int MODE>
struct Rows {
  const uint8_t* base[N_ARRAYS];
  uint8_t* stages;
  Ring* ring;
  int64_t rows, stride;
  uint32_t row_bytes;
  int n_stages, stage;
  uint32_t parity;
  const uint8_t* at[N_ARRAYS];  // the current row's arrays

  // Ring mode, one thread: row -> stage.
  __device__ __forceinline__ void issue(int s, int64_t row) {
    using namespace umma;
    uint8_t* dst = stages + (size_t)s * N_ARRAYS * row_bytes;
    mbar_expect_tx(ring->full + s, N_ARRAYS * row_bytes);
#pragma unroll
    for (int i = 0; i < N_ARRAYS; ++i)
      bulk_load_1d(dst + i * row_bytes, base[i] + row * row_bytes, row_bytes, ring->full + s);
  }
  __device__ __forceinline__ void start(int64_t first) {
    using namespace umma;
    stage = 0;
    parity = 0;
    if constexpr (MODE == kRing) {
      if (threadIdx.x == 0) {
        ring->abort_flag = 0;
        for (int s = 0; s < n_stages; ++s) mbar_init(ring->full + s, 1);
        fence_mbar_init();
      }
      __syncthreads();
      if (threadIdx.x == 0)
        for (int s = 0; s < n_stages; ++s)
          if (first + s * stride < rows) issue(s, first + s * stride);
    }
  }
  __device__ __forceinline__ void open(int64_t row) {
    if constexpr (MODE == kRing) {
      const umma::WaitCtx ctx{&ring->abort_flag, &g_post_pre_device_status, kWaitCycles};
      umma::mbar_wait(ring->full + stage, parity, ctx, 411);
    }
#pragma unroll
    for (int i = 0; i < N_ARRAYS; ++i)
      at[i] = MODE == kRing ? stages + ((size_t)stage * N_ARRAYS + i) * row_bytes : base[i] + row * row_bytes;
  }
  __device__ __forceinline__ uint4 get(int array, int vec) const {
    if constexpr (MODE == kRing) return *reinterpret_cast<const uint4*>(at[array] + vec * 16);
    else return ld_vec(at[array] + vec * 16);
  }
  // Behind a block barrier that follows the row's last get(): the stage takes the row
  // n_stages further on.
  __device__ __forceinline__ void close(int64_t row) {
    if constexpr (MODE == kRing) {
      const int64_t next = row + n_stages * stride;
      if (threadIdx.x == 0 && next < rows && !*(volatile int*)&ring->abort_flag) issue(stage, next);
      if (++stage == n_stages) { stage = 0; parity ^= 1; }
    }
  }
  __device__ __forceinline__ void finish() {
    if constexpr (MODE == kRing)
      if (threadIdx.x == 0 && *(volatile int*)&ring->abort_flag) umma::settle_after_abort();
  }
};

// Pairs of neighbouring elements as packed float32 (one instruction for both).
template <typename T> __device__ __forceinline__ void unpack2(const uint4& v, f32x2 (&f)[Vec<T>::N / 2]) {
  float e[Vec<T>::N];
  unpack<T>(v, e);
#pragma unroll
  for (int i = 0; i < Vec<T>::N / 2; ++i) f[i] = f2_make(e[2 * i], e[2 * i + 1]);
}
template <typename T> __device__ __forceinline__ uint4 pack2f(const f32x2 (&f)[Vec<T>::N / 2]) {
  float e[Vec<T>::N];
#pragma unroll
  for (int i = 0; i < Vec<T>::N / 2; ++i) f2_split(f[i], e[2 * i], e[2 * i + 1]);
  return pack<T>(e);
}
__device__ __forceinline__ float f2_sum(f32x2 v) {
  float lo, hi;
  f2_split(v, lo, hi);
  return lo + hi;
}

__device__ __forceinline__ void st_row(void* base, int64_t row, uint32_t row_bytes, int vec, const uint4& v) {
  st_vec(reinterpret_cast<uint8_t*>(base) + row * row_bytes + vec * 16, v);
}

// Sum over the row's threads: a warp, or the whole block (one partial per warp through
// shared memory, [2][32] floats that are zero behind the last warp; one barrier, the
// halves alternate).
template <int MODE>
__device__ __forceinline__ float row_sum(float v, float* scratch, int& phase) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if constexpr (MODE != kWarp) {
    float* buf = scratch + phase * 32;
    phase ^= 1;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < (int)blockDim.x; w += 128) {
      const float4 p = *reinterpret_cast<const float4*>(buf + w / 32);
      v += (p.x + p.y) + (p.z + p.w);
    }
  }
  return v;
}

// Three sums at once, in a fixed order. In the first two steps a lane passes on the values
// that its partner will finish, so that six shuffles do the work of fifteen: afterwards
// lane l holds value l % 4 (the fourth is zero) over the warp. Blocks add their warps'
// values the same way behind one barrier ([2][16 warps][4] floats; the halves alternate).
template <int MODE>
__device__ __forceinline__ void row_sum3(float (&v)[3], float* scratch, int& phase) {
  const int lane = threadIdx.x & 31;
  const bool odd = lane & 1, high = lane & 2;
  // even lanes go on with values 0 and 2, odd lanes with 1 and 3
  float p = odd ? v[1] : v[0], q = odd ? 0.f : v[2];
  p += __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[1], 1);
  q += __shfl_xor_sync(0xffffffffu, odd ? v[2] : 0.f, 1);
  float s = high ? q : p;
  s += __shfl_xor_sync(0xffffffffu, high ? p : q, 2);
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if constexpr (MODE != kWarp) {
    float* buf = scratch + phase * 64;
    phase ^= 1;
    if (lane < 4) buf[(threadIdx.x >> 5) * 4 + lane] = s;
    __syncthreads();
    s = buf[lane] + buf[32 + lane];
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) v[i] = __shfl_sync(0xffffffffu, s, i);
}


// The weights of a thread's columns, as packed pairs; `post` is the post weight times a
// channel's gate. A thread keeps their 16-byte vectors in registers for all its rows;
// kDirect reads them for every row.
template <typename T, int V, int GATE, int MODE>
struct Weights {
  static constexpr int P = Vec<T>::N / 2;
  static constexpr int R = MODE != kDirect ? V : 1;
  const NormArgs* a;
  uint4 pre_r[R], post_r[R], gate_r[R];
  __device__ __forceinline__ void load(const NormArgs& args, int lane, int width, int nvec) {
    a = &args;
    if constexpr (MODE != kDirect) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int vec = lane + j * width;
        pre_r[j] = post_r[j] = gate_r[j] = make_uint4(0, 0, 0, 0);
        if (vec < nvec) {
          pre_r[j] = ld_vec((const uint8_t*)args.w_pre + vec * 16);
          post_r[j] = ld_vec((const uint8_t*)args.w_post + vec * 16);
          if (GATE == kChannel) gate_r[j] = ld_vec((const uint8_t*)args.gate + vec * 16);
        }
      }
    }
  }
  __device__ __forceinline__ void pre(int j, int vec, f32x2 (&w)[P]) const {
    if constexpr (MODE != kDirect) unpack2<T>(pre_r[j], w);
    else unpack2<T>(__ldg(reinterpret_cast<const uint4*>(a->w_pre) + vec), w);
  }
  __device__ __forceinline__ void post(int j, int vec, f32x2 (&w)[P]) const {
    f32x2 g[P];
    if constexpr (MODE != kDirect) {
      unpack2<T>(post_r[j], w);
      if (GATE == kChannel) unpack2<T>(gate_r[j], g);
    } else {
      unpack2<T>(__ldg(reinterpret_cast<const uint4*>(a->w_post) + vec), w);
      if (GATE == kChannel) unpack2<T>(__ldg(reinterpret_cast<const uint4*>(a->gate) + vec), g);
    }
    if constexpr (GATE == kChannel) {
#pragma unroll
      for (int i = 0; i < P; ++i) w[i] = f2_mul(w[i], g[i]);
    }
  }
};

// ------------------------------------------------------------------ forward
template <typename T, int V, int GATE, int MODE>
__global__ void __launch_bounds__(MODE == kWarp ? 256 : 512, MODE == kRing && V == 1 ? 2 : 1)
post_pre_fwd_kernel(const NormArgs a) {
  constexpr int N = Vec<T>::N, P = N / 2;
  constexpr int NA = GATE == kFull ? 3 : 2;  // x, h, gate
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ __align__(16) float scratch[2 * 32];
  __shared__ Ring ring;
  int phase = 0;
  const int lane = MODE == kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int width = MODE == kWarp ? 32 : blockDim.x;
  const int nvec = (int)(a.C / N);
  const int64_t stride = MODE == kWarp ? (int64_t)gridDim.x * (blockDim.x / 32) : gridDim.x;
  int64_t row = MODE == kWarp ? (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
  if (threadIdx.x < 64) scratch[threadIdx.x] = 0.f;
  if constexpr (MODE == kDirect) __syncthreads();  // the ring's start has one
  Rows<NA, MODE> in;
  in.base[0] = (const uint8_t*)a.x;
  in.base[1] = (const uint8_t*)a.h;
  if constexpr (GATE == kFull) in.base[2] = (const uint8_t*)a.gate;
  in.stages = dyn;
  in.ring = &ring;
  in.rows = a.rows;
  in.stride = stride;
  in.row_bytes = nvec * 16;
  in.n_stages = a.stages;
  in.start(row);
  Weights<T, V, GATE, MODE> w;
  w.load(a, lane, width, nvec);
  float gt_next = GATE == kToken && row < a.rows ? to_f32<T>(((const T*)a.gate)[row]) : 1.f;
  for (; row < a.rows; row += stride) {
    in.open(row);
    const float gt = gt_next;
    if (GATE == kToken && row + stride < a.rows) gt_next = to_f32<T>(((const T*)a.gate)[row + stride]);
    f32x2 x[V][P], hn[V][P], acc = 0ull;
    uint4 hv[V], gv[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = lane + j * width;
      const bool on = vec < nvec;
      unpack2<T>(on ? in.get(0, vec) : make_uint4(0, 0, 0, 0), x[j]);
      hv[j] = on ? in.get(1, vec) : make_uint4(0, 0, 0, 0);
      if constexpr (GATE == kFull) gv[j] = on ? in.get(2, vec) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) acc = f2_fma(x[j][i], x[j][i], acc);
    const float r1 = rsqrtf(fmaf(row_sum<MODE>(f2_sum(acc), scratch, phase), a.inv_c, a.eps));
    in.close(row);
    const f32x2 scale = f2_splat(r1 * a.alpha * gt);
    acc = 0ull;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = lane + j * width;
      unpack2<T>(hv[j], hn[j]);
      if (vec < nvec) {
        f32x2 wp[P], g[P];
        w.post(j, vec, wp);
        if constexpr (GATE == kFull) unpack2<T>(gv[j], g);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          f32x2 n = f2_mul(x[j][i], wp[i]);
          if constexpr (GATE == kFull) n = f2_mul(n, g[i]);
          hn[j][i] = f2_fma(n, scale, hn[j][i]);
          acc = f2_fma(hn[j][i], hn[j][i], acc);
        }
        st_row(a.h_out, row, in.row_bytes, vec, pack2f<T>(hn[j]));
      }
    }
    const float r2 = rsqrtf(fmaf(row_sum<MODE>(f2_sum(acc), scratch, phase), a.inv_c, a.eps));
    const f32x2 rr = f2_splat(r2);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = lane + j * width;
      if (vec < nvec) {
        f32x2 wn[P];
        w.pre(j, vec, wn);
#pragma unroll
        for (int i = 0; i < P; ++i) wn[i] = f2_mul(f2_mul(hn[j][i], rr), wn[i]);
        st_row(a.y, row, in.row_bytes, vec, pack2f<T>(wn));
      }
    }
    if (lane == 0) {
      a.rstd_post[row] = r1;
      a.rstd_pre[row] = r2;
    }
  }
  in.finish();
}

// ----------------------------------------------------------------- backward
// With U = G w_post gate (the gate of a full or channel kind; a row's number stays outside):
//   sum u xhat = alpha gate_row rstd1 sum U x,  dx = rstd1 alpha gate_row U - x rstd1^2 c2,
// and as G = dh' + rstd2 t - rstd2 c1 h'hat, sum U x is linear in c1 as well:
//   sum U x = sum (dh' + rstd2 t) w x - rstd2 c1 sum h'hat w x,   w = w_post gate,
// so all a row needs comes out of ONE reduction of three sums, and everything else of the
// row happens behind it.
template <typename T, int V, int GATE, int MODE>
__global__ void __launch_bounds__(MODE == kWarp || V == 1 ? 256 : 512, V == 1 ? 2 : 1)
post_pre_bwd_kernel(const NormArgs a) {
  constexpr int N = Vec<T>::N, P = N / 2;
  constexpr int NA = GATE == kFull ? 5 : 4;  // dy, h', dh', x, gate
  extern __shared__ __align__(128) uint8_t dyn[];  // ring stages; kWarp: one partial row, [2][C] floats
  __shared__ __align__(16) float scratch[2 * 64];
  __shared__ Ring ring;
  int phase = 0;
  const int lane = MODE == kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int width = MODE == kWarp ? 32 : blockDim.x;
  const int nvec = (int)(a.C / N);
  const int64_t stride = MODE == kWarp ? (int64_t)gridDim.x * (blockDim.x / 32) : gridDim.x;
  int64_t row = MODE == kWarp ? (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
  for (int i = threadIdx.x; i < 128; i += blockDim.x) scratch[i] = 0.f;
  if constexpr (MODE == kDirect) __syncthreads();
  Rows<NA, MODE> in;
  in.base[0] = (const uint8_t*)a.dy;
  in.base[1] = (const uint8_t*)a.h;
  in.base[2] = (const uint8_t*)a.dh_in;
  in.base[3] = (const uint8_t*)a.x;
  if constexpr (GATE == kFull) in.base[4] = (const uint8_t*)a.gate;
  in.stages = dyn;
  in.ring = &ring;
  in.rows = a.rows;
  in.stride = stride;
  in.row_bytes = nvec * 16;
  in.n_stages = a.stages;
  in.start(row);
  Weights<T, V, GATE, MODE> w;
  w.load(a, lane, width, nvec);
  f32x2 spost[V][P], spre[V][P];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < P; ++i) spost[j][i] = spre[j][i] = 0ull;
  // the row's numbers come one row ahead: nothing else hides their latency
  float r1_next = 0.f, r2_next = 0.f, gt_next = 1.f;
  auto ahead = [&](int64_t r) {
    if (r < a.rows) {
      r1_next = a.rstd_post[r];
      r2_next = a.rstd_pre[r];
      if (GATE == kToken) gt_next = to_f32<T>(((const T*)a.gate)[r]);
    }
  };
  ahead(row);
  for (; row < a.rows; row += stride) {
    const float r1 = r1_next, r2 = r2_next, gt = gt_next;
    ahead(row + stride);
    in.open(row);
    f32x2 t[V][P], h[V][P];
    uint4 dv[V], xv[V], gv[V];
    f32x2 acc[3] = {0ull, 0ull, 0ull};  // t h'hat; (dh' + rstd2 t) w x; h'hat w x
    const f32x2 rr2 = f2_splat(r2);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = lane + j * width;
      if (vec < nvec) {
        f32x2 e[P], wv[P], x[P];
        unpack2<T>(in.get(0, vec), e);
        unpack2<T>(in.get(1, vec), h[j]);
        dv[j] = in.get(2, vec);
        xv[j] = in.get(3, vec);
        if constexpr (GATE == kFull) gv[j] = in.get(4, vec);
        w.pre(j, vec, wv);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          h[j][i] = f2_mul(h[j][i], rr2);  // h'hat
          t[j][i] = f2_mul(e[i], wv[i]);
          spre[j][i] = f2_fma(e[i], h[j][i], spre[j][i]);
          acc[0] = f2_fma(t[j][i], h[j][i], acc[0]);
        }
        unpack2<T>(dv[j], e);
        unpack2<T>(xv[j], x);
        w.post(j, vec, wv);
        if constexpr (GATE == kFull) {
          f32x2 g[P];
          unpack2<T>(gv[j], g);
#pragma unroll
          for (int i = 0; i < P; ++i) wv[i] = f2_mul(wv[i], g[i]);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const f32x2 wx = f2_mul(wv[i], x[i]);
          acc[1] = f2_fma(f2_fma(t[j][i], rr2, e[i]), wx, acc[1]);
          acc[2] = f2_fma(h[j][i], wx, acc[2]);
        }
      }
    }
    float s[3] = {f2_sum(acc[0]), f2_sum(acc[1]), f2_sum(acc[2])};
    row_sum3<MODE>(s, scratch, phase);
    in.close(row);
    const float k1 = -r2 * s[0] * a.inv_c;                    // -rstd2 c1
    const float sum = fmaf(k1, s[2], s[1]) * r1;              // sum U xhat
    const float ag = a.alpha * gt;
    if (GATE == kToken && lane == 0) ((T*)a.dgate)[row] = from_f32<T>(a.alpha * sum);
    const f32x2 kk1 = f2_splat(k1), ku = f2_splat(r1 * ag), kx = f2_splat(-r1 * r1 * ag * sum * a.inv_c);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = lane + j * width;
      if (vec < nvec) {
        f32x2 d[P], x[P], wp[P], g[P];
        unpack2<T>(dv[j], d);
        unpack2<T>(xv[j], x);
        if constexpr (GATE == kFull) unpack2<T>(gv[j], g);
        w.post(j, vec, wp);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const f32x2 G = f2_fma(t[j][i], rr2, f2_fma(h[j][i], kk1, d[i]));
          f32x2 q = f2_mul(G, x[i]);
          f32x2 U = f2_mul(G, wp[i]);
          d[i] = G;
          if constexpr (GATE == kFull) {
            wp[i] = f2_mul(f2_mul(q, wp[i]), ku);             // dgate (ku = rstd1 alpha)
            U = f2_mul(U, g[i]);
            q = f2_mul(q, g[i]);
          }
          spost[j][i] = f2_fma(q, ku, spost[j][i]);
          x[i] = f2_fma(U, ku, f2_mul(x[i], kx));
        }
        st_row(a.dh_out, row, in.row_bytes, vec, pack2f<T>(d));
        if constexpr (GATE == kFull) st_row(a.dgate, row, in.row_bytes, vec, pack2f<T>(wp));
        st_row(a.dx, row, in.row_bytes, vec, pack2f<T>(x));
      }
    }
  }
  in.finish();
  // one float32 partial row per block
  f32x2* pre = reinterpret_cast<f32x2*>(a.partial + (int64_t)blockIdx.x * a.C);
  f32x2* post = reinterpret_cast<f32x2*>(a.partial + ((int64_t)gridDim.x + blockIdx.x) * a.C);
  if constexpr (MODE != kWarp) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = lane + j * width;
      if (vec < nvec)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          pre[vec * P + i] = spre[j][i];
          post[vec * P + i] = spost[j][i];
        }
    }
  } else {
    const int pairs = (int)a.C / 2;  // at most 64 vectors
    f32x2* fold = reinterpret_cast<f32x2*>(dyn);
    for (int wi = 0; wi < (int)blockDim.x / 32; ++wi) {  // the warps' rows in warp order
      if ((int)threadIdx.x / 32 == wi) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int vec = lane + j * width;
          if (vec < nvec)
#pragma unroll
            for (int i = 0; i < P; ++i) {
              f32x2* f = fold + vec * P + i;
              f[0] = wi ? f2_add(f[0], spre[j][i]) : spre[j][i];
              f[pairs] = wi ? f2_add(f[pairs], spost[j][i]) : spost[j][i];
            }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < pairs; c += blockDim.x) {
      pre[c] = fold[c];
      post[c] = fold[pairs + c];
    }
  }
}

// ------------------------------------------- rows off the 16-byte boundaries
// Element by element, but each element once: a row's elements stay in its threads' registers
// as in the kernels above (columns lane, lane + W, ..., K of them), so a warp still reads
// and writes contiguous memory. Elements and weights behind the row's end are zeros, which
// add nothing to any sum.
template <typename T>
__device__ __forceinline__ float gate_at(const NormArgs& a, int gate, int64_t row, int64_t c) {
  const T* g = (const T*)a.gate;
  return gate == kNone ? 1.f : to_f32<T>(g[gate == kChannel ? c : gate == kToken ? row : row * a.C + c]);
}
// *p, or zero (a predicated load: as a branch per element, the loads of a row would wait for
// one another).
template <typename T> __device__ __forceinline__ float ld_if(const T* p, bool on) {
  if constexpr (sizeof(T) == 2) {
    unsigned short r;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b16 %0, 0;\n\t@p ld.global.b16 %0, [%1];\n\t}"
                 : "=h"(r) : "l"(p), "r"((int)on));
    return to_f32<T>(*reinterpret_cast<T*>(&r));
  } else {
    float r;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}"
                 : "=f"(r) : "l"(p), "r"((int)on));
    return r;
  }
}
__host__ __device__ constexpr int ragged_threads(int W) { return W == 32 ? 256 : W; }

template <typename T, int K, int W>
__global__ void __launch_bounds__(ragged_threads(W), K <= 12 ? 1024 / ragged_threads(W) : 1)
post_pre_fwd_ragged_kernel(const NormArgs a, int gate) {
  constexpr int MODE = W == 32 ? kWarp : kDirect;
  __shared__ __align__(16) float scratch[2 * 32];
  int phase = 0;
  const int lane = threadIdx.x % W;
  const int left = (int)a.C - lane;  // column lane + k W exists while k W < left
  const int64_t stride = (int64_t)gridDim.x * (ragged_threads(W) / W);
  int64_t row = (int64_t)blockIdx.x * (ragged_threads(W) / W) + threadIdx.x / W;
  if (threadIdx.x < 64) scratch[threadIdx.x] = 0.f;
  if constexpr (MODE == kDirect) __syncthreads();
  float wp[K], wn[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    wp[k] = ld_if((const T*)a.w_post + lane + k * W, k * W < left);
    wn[k] = ld_if((const T*)a.w_pre + lane + k * W, k * W < left);
    if (gate == kChannel) wp[k] *= ld_if((const T*)a.gate + lane + k * W, k * W < left);
  }
  for (; row < a.rows; row += stride) {
    const int64_t at = row * a.C + lane;
    const T *x = (const T*)a.x + at, *res = (const T*)a.h + at;
    float v[K], h[K], acc = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = ld_if(x + k * W, k * W < left);
      h[k] = ld_if(res + k * W, k * W < left);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) acc = fmaf(v[k], v[k], acc);
    const float r1 = rsqrtf(fmaf(row_sum<MODE>(acc, scratch, phase), a.inv_c, a.eps));
    const float scale = r1 * a.alpha * (gate == kToken ? gate_at<T>(a, gate, row, 0) : 1.f);
    if (gate == kFull) {
      const T* g = (const T*)a.gate + at;
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] *= ld_if(g + k * W, k * W < left);
    }
    acc = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      h[k] = fmaf(v[k] * wp[k], scale, h[k]);
      acc = fmaf(h[k], h[k], acc);
    }
    T *ho = (T*)a.h_out + at, *y = (T*)a.y + at;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k * W < left) ho[k * W] = from_f32<T>(h[k]);
    const float r2 = rsqrtf(fmaf(row_sum<MODE>(acc, scratch, phase), a.inv_c, a.eps));
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k * W < left) y[k * W] = from_f32<T>(h[k] * r2 * wn[k]);
    if (lane == 0) {
      a.rstd_post[row] = r1;
      a.rstd_pre[row] = r2;
    }
  }
}

template <typename T, int K, int W>
__global__ void __launch_bounds__(ragged_threads(W), K == 8 ? 512 / ragged_threads(W) : 1)
post_pre_bwd_ragged_kernel(const NormArgs a, int gate) {
  constexpr int MODE = W == 32 ? kWarp : kDirect;
  extern __shared__ float fold[];  // kWarp: one partial row, [2][C]
  __shared__ __align__(16) float scratch[2 * 64];
  int phase = 0;
  const int C = (int)a.C, lane = threadIdx.x % W;
  const int left = C - lane;  // column lane + k W exists while k W < left
  const int64_t stride = (int64_t)gridDim.x * (ragged_threads(W) / W);
  int64_t row = (int64_t)blockIdx.x * (ragged_threads(W) / W) + threadIdx.x / W;
  for (int i = threadIdx.x; i < 128; i += blockDim.x) scratch[i] = 0.f;
  __syncthreads();
  float wp[K], wn[K], spost[K], spre[K];  // wp: times a channel's gate
#pragma unroll
  for (int k = 0; k < K; ++k) {
    wp[k] = ld_if((const T*)a.w_post + lane + k * W, k * W < left);
    wn[k] = ld_if((const T*)a.w_pre + lane + k * W, k * W < left);
    if (gate == kChannel) wp[k] *= ld_if((const T*)a.gate + lane + k * W, k * W < left);
    spost[k] = spre[k] = 0.f;
  }
  for (; row < a.rows; row += stride) {
    const int64_t at = row * C + lane;
    const T *x = (const T*)a.x + at, *hs = (const T*)a.h + at, *g = (const T*)a.gate + at;
    const T *dy = (const T*)a.dy + at, *dh = (const T*)a.dh_in + at;
    const float r1 = a.rstd_post[row], r2 = a.rstd_pre[row];
    const float gt = gate == kToken ? gate_at<T>(a, gate, row, 0) : 1.f;
    float t[K], h[K], d[K], v[K], s[3] = {0.f, 0.f, 0.f};  // t h'hat; (dh' + rstd2 t) w x; h'hat w x
#pragma unroll
    for (int k = 0; k < K; ++k) {
      t[k] = ld_if(dy + k * W, k * W < left);
      h[k] = ld_if(hs + k * W, k * W < left);
      d[k] = ld_if(dh + k * W, k * W < left);
      v[k] = ld_if(x + k * W, k * W < left);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      h[k] *= r2;
      spre[k] = fmaf(t[k], h[k], spre[k]);
      t[k] *= wn[k];
      float wx = wp[k] * v[k];
      if (gate == kFull) wx *= ld_if(g + k * W, k * W < left);
      s[0] = fmaf(t[k], h[k], s[0]);
      s[1] = fmaf(fmaf(t[k], r2, d[k]), wx, s[1]);
      s[2] = fmaf(h[k], wx, s[2]);
    }
    row_sum3<MODE>(s, scratch, phase);
    const float k1 = -r2 * s[0] * a.inv_c;        // -rstd2 c1
    const float sum = fmaf(k1, s[2], s[1]) * r1;  // sum U xhat
    const float ku = r1 * a.alpha * gt, kx = -r1 * ku * sum * a.inv_c;
    if (gate == kToken && lane == 0) ((T*)a.dgate)[row] = from_f32<T>(a.alpha * sum);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float G = fmaf(t[k], r2, fmaf(h[k], k1, d[k]));
      float q = G * v[k], U = G * wp[k];
      if (gate == kFull) {
        const float gk = ld_if(g + k * W, k * W < left);
        t[k] = q * wp[k] * ku;  // dgate
        q *= gk;
        U *= gk;
      }
      spost[k] = fmaf(q, ku, spost[k]);
      d[k] = G;
      v[k] = fmaf(U, ku, v[k] * kx);
    }
    T *dho = (T*)a.dh_out + at, *dx = (T*)a.dx + at, *dg = (T*)a.dgate + at;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k * W < left) {
        dho[k * W] = from_f32<T>(d[k]);
        dx[k * W] = from_f32<T>(v[k]);
        if (gate == kFull) dg[k * W] = from_f32<T>(t[k]);
      }
  }
  float* pre = a.partial + (int64_t)blockIdx.x * C;
  float* post = a.partial + ((int64_t)gridDim.x + blockIdx.x) * C;
  if constexpr (MODE != kWarp) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k * W < left) {
        pre[lane + k * W] = spre[k];
        post[lane + k * W] = spost[k];
      }
  } else {
    for (int wi = 0; wi < ragged_threads(W) / 32; ++wi) {  // the warps' rows in warp order
      if ((int)threadIdx.x / 32 == wi) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (k * W < left) {
            const int c = lane + k * W;
            fold[c] = wi ? fold[c] + spre[k] : spre[k];
            fold[C + c] = wi ? fold[C + c] + spost[k] : spost[k];
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

// ------------------------------------------------------------- any width
// Rows of more than 8192 elements that are off a 16-byte boundary, and whole vectors beyond 2048
// of them. One block per row, three passes over the row (the later ones from L2); the column sums
// of the backward live in the block's own partial row. [8192, 20000] bf16: forward 943 us, backward
// 2366, where four and six passes of HBM take 200 and 300.
constexpr int kAnyThreads = 256;

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

// Column sums: 32 columns x 32 slices of partial rows per block, a slice's rows four at a
// time, added in a fixed order; dw_pre = S_pre, dw_post = S_post (times the channel's
// gate), dgate = w_post S_post.
template <typename T>
__global__ void __launch_bounds__(1024)
post_pre_columns_kernel(const float* __restrict__ partial, int blocks, int64_t C,
                        const T* __restrict__ w_post, const T* __restrict__ gate_channel, T* dw_pre,
                        T* dw_post, T* dgate_channel) {
  __shared__ float part[32][33];
  const int which = blockIdx.y;
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  const float* src = partial + (int64_t)which * blocks * C;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < C) {
    int p = threadIdx.y;
    for (; p + 96 < blocks; p += 128) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += src[(int64_t)(p + 32 * i) * C + c];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + 32 * i < blocks) s[i] += src[(int64_t)(p + 32 * i) * C + c];
  }
  part[threadIdx.y][threadIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (threadIdx.y || c >= C) return;
  float sum = part[0][threadIdx.x];
#pragma unroll
  for (int i = 1; i < 32; ++i) sum += part[i][threadIdx.x];
  if (which == 0) {
    dw_pre[c] = from_f32<T>(sum);
  } else {
    dw_post[c] = from_f32<T>(gate_channel ? sum * to_f32<T>(gate_channel[c]) : sum);
    if (dgate_channel) dgate_channel[c] = from_f32<T>(sum * to_f32<T>(w_post[c]));
  }
}

// ---------------------------------------------------------------- host side
int read_post_pre_status(int reset) {
  int code = 0;
  if (cudaMemcpyFromSymbol(&code, g_post_pre_device_status, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (reset && code != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_post_pre_device_status, &zero, sizeof(int));
  }
  return code;
}
const bool g_post_pre_registered = (register_device_status(read_post_pre_status), true);

struct Shape {
  enum { kVectors, kRagged, kAny } kind;
  int mode, V, threads, stages;  // V: vectors per thread, elements for kRagged
};
// One vector per thread up to 512 (forward) or 256 vectors (backward), two up to 1024, four
// above: the forward (few registers) runs best with the most threads, the backward with half
// of them and twice the work between its barriers ([16384, 4096] bf16: 87 against 96 us with
// two vectors forward, 136 against 158 us with one vector backward); a warp per row up to 64
// vectors. Rows off a 16-byte boundary take the ragged kernels up to 8192 elements, a warp
// per row up to 256, 8, 12 or 16 elements per thread (16384 rows of bf16 forward + backward,
// against the kernels that read the row three times: 201 columns 138 -> 34 us, 1001
// 284 -> 105, 4098 961 -> 526, 6001 1668 -> 648, 8001 2418 -> 1204; with one shape of 16
// elements from 4097 on, 4098 took 894); all wider rows the kernels for any width, aligned ones
// beyond 2048 vectors too.
Shape pick_shape(int64_t C, size_t elem, bool aligned, bool backward) {
  const int one_vector_most = backward ? 256 : 512;
  Shape s{};
  if (!aligned || (C * elem) % 16 != 0 || C * elem / 16 > 2048) {
    const int W = C <= 256 ? 32 : C <= 1024 ? 128 : C <= 2048 ? 256 : 512;
    s.mode = W == 32 ? kWarp : kDirect;
    s.V = C <= 8 * W ? 8 : C <= 12 * W ? 12 : 16;
    s.threads = ragged_threads(W);
    s.kind = Shape::kRagged;
    if (C > 8192) {
      s.kind = Shape::kAny;
      s.threads = kAnyThreads;
    }
    return s;
  }
  const int nvec = (int)(C * elem / 16);
  if (nvec <= 64) {
    s.mode = kWarp;
    s.V = nvec <= 32 ? 1 : 2;
    s.threads = 256;
    return s;
  }
  s.V = nvec <= one_vector_most ? 1 : nvec <= 1024 ? 2 : 4;
  s.threads = ((nvec + s.V - 1) / s.V + 31) / 32 * 32;
  // Ring of two stages for rows of up to 1024 vectors (five arrays of 16 KB twice: 160 KB); a third
  // or fourth stage, or wider vectors for fewer blocks, measured 1-4 % slower (a block waits for
  // its own reductions, not for its rows, so more blocks beat deeper rings).
  s.mode = s.V <= 2 ? kRing : kDirect;
  s.stages = kMaxStages;
  return s;
}
// Most blocks a backward launches, and with that partial rows.
int most_blocks() { return device_info().sm_count * 8; }

// Blocks of a kernel that fit an SM. Asking takes the host about as long as a launch, so
// a thread remembers its last answers (a fixed property of kernel, block and device).
int occupancy(const void* kernel, int threads, size_t smem) {
  struct Known {
    const void* kernel;
    int device, threads, blocks;
    size_t smem;
  };
  static thread_local Known known[8] = {};
  static thread_local unsigned next = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  for (const Known& k : known)
    if (k.kernel == kernel && k.device == dev && k.threads == threads && k.smem == smem) return k.blocks;
  int occ = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kernel, threads, smem) != cudaSuccess) {
    cudaGetLastError();
    return 1;  // of this call only
  }
  if (occ < 1) occ = 1;
  known[next++ % 8] = Known{kernel, dev, threads, occ, smem};
  return occ;
}

template <typename Kernel>
int blocks_for(Kernel kernel, const Shape& s, int64_t rows, size_t smem) {
  const int occ = occupancy((const void*)kernel, s.threads, smem);
  int64_t n = (int64_t)device_info().sm_count * occ;
  const int64_t per = s.kind != Shape::kAny && s.mode == kWarp ? s.threads / 32 : 1;
  const int64_t need = (rows + per - 1) / per;
  if (n > need) n = need;
  if (n > most_blocks()) n = most_blocks();
  return (int)(n < 1 ? 1 : n);
}

template <typename Kernel>
int launch_rows(const char* what, Kernel kernel, const NormArgs& a, const Shape& s, size_t smem,
                cudaStream_t st, int& blocks) {
  // (the limit without the attribute, 48 KB, includes the static part)
  if (smem > 32 * 1024 && !allow_shared_memory((const void*)kernel, smem))
    return fail(EVG_ELAUNCH, "%s: cannot reserve %zu bytes of shared memory", what, smem);
  blocks = blocks_for(kernel, s, a.rows, smem);
  kernel<<<blocks, s.threads, smem, st>>>(a);
  return check_launch(what);
}

template <typename T, int V, int MODE>
int launch_fwd(const NormArgs& a, int gate, const Shape& s, cudaStream_t st) {
  const size_t smem = MODE == kRing ? (size_t)s.stages * (gate == kFull ? 3 : 2) * a.C * sizeof(T) : 0;
  const char* what = "post_pre_norm_fwd";
  int blocks;
  switch (gate) {
    case kNone: return launch_rows(what, post_pre_fwd_kernel<T, V, kNone, MODE>, a, s, smem, st, blocks);
    case kChannel: return launch_rows(what, post_pre_fwd_kernel<T, V, kChannel, MODE>, a, s, smem, st, blocks);
    case kToken: return launch_rows(what, post_pre_fwd_kernel<T, V, kToken, MODE>, a, s, smem, st, blocks);
    default: return launch_rows(what, post_pre_fwd_kernel<T, V, kFull, MODE>, a, s, smem, st, blocks);
  }
}
template <typename T, int V, int MODE>
int launch_bwd(const NormArgs& a, int gate, const Shape& s, cudaStream_t st, int& blocks) {
  const size_t smem = MODE == kDirect ? 0
                      : MODE == kWarp ? 2 * a.C * sizeof(float)
                                      : (size_t)s.stages * (gate == kFull ? 5 : 4) * a.C * sizeof(T);
  const char* what = "post_pre_norm_bwd";
  switch (gate) {
    case kNone: return launch_rows(what, post_pre_bwd_kernel<T, V, kNone, MODE>, a, s, smem, st, blocks);
    case kChannel: return launch_rows(what, post_pre_bwd_kernel<T, V, kChannel, MODE>, a, s, smem, st, blocks);
    case kToken: return launch_rows(what, post_pre_bwd_kernel<T, V, kToken, MODE>, a, s, smem, st, blocks);
    default: return launch_rows(what, post_pre_bwd_kernel<T, V, kFull, MODE>, a, s, smem, st, blocks);
  }
}

template <typename T>
int run_fwd(const NormArgs& a, int gate, const Shape& s, cudaStream_t st) {
  if (s.kind == Shape::kRagged) {
    auto run = [&](auto kernel) {
      kernel<<<blocks_for(kernel, s, a.rows, 0), s.threads, 0, st>>>(a, gate);
      return check_launch("post_pre_norm_fwd");
    };
    return s.mode == kWarp    ? run(post_pre_fwd_ragged_kernel<T, 8, 32>)
           : s.threads == 128 ? run(post_pre_fwd_ragged_kernel<T, 8, 128>)
           : s.threads == 256 ? run(post_pre_fwd_ragged_kernel<T, 8, 256>)
           : s.V == 8         ? run(post_pre_fwd_ragged_kernel<T, 8, 512>)
           : s.V == 12        ? run(post_pre_fwd_ragged_kernel<T, 12, 512>)
                              : run(post_pre_fwd_ragged_kernel<T, 16, 512>);
  }
  if (s.kind == Shape::kAny) {
    post_pre_fwd_any_kernel<T><<<blocks_for(post_pre_fwd_any_kernel<T>, s, a.rows, 0), s.threads, 0, st>>>(a, gate);
    return check_launch("post_pre_norm_fwd");
  }
  if (s.mode == kWarp) return s.V == 1 ? launch_fwd<T, 1, kWarp>(a, gate, s, st) : launch_fwd<T, 2, kWarp>(a, gate, s, st);
  if (s.mode == kRing) return s.V == 1 ? launch_fwd<T, 1, kRing>(a, gate, s, st) : launch_fwd<T, 2, kRing>(a, gate, s, st);
  return launch_fwd<T, 4, kDirect>(a, gate, s, st);
}

template <typename T>
int run_bwd_rows(const NormArgs& a, int gate, const Shape& s, cudaStream_t st, int& blocks) {
  if (s.kind == Shape::kRagged) {
    auto run = [&](auto kernel) {
      const size_t smem = s.mode == kWarp ? 2 * a.C * sizeof(float) : 0;
      blocks = blocks_for(kernel, s, a.rows, smem);
      kernel<<<blocks, s.threads, smem, st>>>(a, gate);
      return check_launch("post_pre_norm_bwd");
    };
    return s.mode == kWarp    ? run(post_pre_bwd_ragged_kernel<T, 8, 32>)
           : s.threads == 128 ? run(post_pre_bwd_ragged_kernel<T, 8, 128>)
           : s.threads == 256 ? run(post_pre_bwd_ragged_kernel<T, 8, 256>)
           : s.V == 8         ? run(post_pre_bwd_ragged_kernel<T, 8, 512>)
           : s.V == 12        ? run(post_pre_bwd_ragged_kernel<T, 12, 512>)
                              : run(post_pre_bwd_ragged_kernel<T, 16, 512>);
  }
  if (s.kind == Shape::kAny) {
    blocks = blocks_for(post_pre_bwd_any_kernel<T>, s, a.rows, 0);
    post_pre_bwd_any_kernel<T><<<blocks, s.threads, 0, st>>>(a, gate);
    return check_launch("post_pre_norm_bwd");
  }
  if (s.mode == kWarp)
    return s.V == 1 ? launch_bwd<T, 1, kWarp>(a, gate, s, st, blocks) : launch_bwd<T, 2, kWarp>(a, gate, s, st, blocks);
  if (s.mode == kRing)
    return s.V == 1 ? launch_bwd<T, 1, kRing>(a, gate, s, st, blocks) : launch_bwd<T, 2, kRing>(a, gate, s, st, blocks);
  return launch_bwd<T, 4, kDirect>(a, gate, s, st, blocks);
}

int check_norm_args(const char* what, int64_t rows, int64_t C, int gate, int dtype) {
  if (rows < 0 || C <= 0 || rows > 0x7fffffff || C > (1 << 26))
    return fail(EVG_EBADSHAPE, "%s: rows=%lld hidden=%lld", what, (long long)rows, (long long)C);
  if (gate < kNone || gate > kFull) return fail(EVG_EBADSHAPE, "%s: gate kind %d", what, gate);
  if (dtype != EVG_F32 && dtype != EVG_F16 && dtype != EVG_BF16) return fail(EVG_EDTYPE, "%s: dtype %d", what, dtype);
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
  if (int rc = check_norm_args(what, rows, hidden, gate_kind, dtype)) return rc;
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
  const Shape s = pick_shape(hidden, dtype_size(dtype), aligned, false);
  a.stages = s.stages;
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
  if (int rc = check_norm_args(what, rows, hidden, gate_kind, dtype)) return rc;
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
  const Shape s = pick_shape(hidden, dtype_size(dtype), aligned, true);
  a.stages = s.stages;
  cudaStream_t st = (cudaStream_t)stream;
  return EVG_DISPATCH_DTYPE(dtype, [&] {
    int blocks = 0;
    if (int rc = run_bwd_rows<T>(a, gate_kind, s, st, blocks)) return rc;
    const bool channel = gate_kind == kChannel;
    post_pre_columns_kernel<T><<<dim3((unsigned)((hidden + 31) / 32), 2), dim3(32, 32), 0, st>>>(
        a.partial, blocks, hidden, (const T*)w_post, channel ? (const T*)gate : nullptr, (T*)dw_pre,
        (T*)dw_post, channel ? (T*)dgate : nullptr);
    return check_launch("post_pre_norm_bwd columns");
  });
}
