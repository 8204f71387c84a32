// Rotary embedding from position numbers (sm_100a), forward and backward in one
// kernel family: of rotary pair i at position p
//   theta = p f_i,  y1 = m (x1 cos theta - x2 sin theta),  y2 = m (x2 cos theta + x1 sin theta)
// and the backward is the transpose (sine negated, the same factor m). Pairs are the
// two halves of the first `rd` columns, or neighbouring columns (interleaved); columns
// behind rd pass through.
//
// theta / 2 pi is formed and reduced to half a turn in float64 (positions reach far
// beyond what float32 resolves), then one float32 sincospi. A block computes the
// angles of its few tokens once, into shared memory, and uses them for all heads of
// both tensors: with 40 heads of 128 the 64 angles of a token cost a sixth of the
// instructions of its 320 vectors. No table of positions exists in device memory.
//
// HBM-bound: one read and one write per element. q, k [16384, 32 + 8, 128] bf16, forward
// and backward: 108 us, 6.2 TB/s. A thread holds ONE item (two 16-byte vectors) and 40
// registers keep six blocks on an SM: more blocks in different phases (angles, loads,
// stores) hide the latencies better than more loads per thread (two items per thread,
// four blocks: 125 us; four items, 71 registers: 171 us). Blocks of about 768 items
// (three rounds) against 512 and 2048: 108, 110, 115 us.
#include "evg_common.cuh"

namespace evg {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTensors = 2;
constexpr int kTableFloats = 8192;   // shared memory for angles: 32 KB

// n / d for 0 <= n, n * d < 2^32.
struct Divisor {
  uint32_t m;
  __host__ void set(uint32_t v) {
    m = v == 1 ? 0 : (uint32_t)((0xffffffffull + v) / v);  // ceil(2^32 / v)
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return m ? __umulhi(n, m) : n; }
};

struct PosTensor {
  const void* x;
  void* y;
  int heads;
  int64_t xst, xsh, yst, ysh;
};
struct PosArgs {
  PosTensor t[kMaxTensors];
  const void* positions;
  const void* inv_freq;
  int64_t tokens;
  int tokens_per_block, heads_per_block, total_heads;
  int rd, pairs;       // rotated columns, rd / 2
  int rot_vecs, rot_items;    // vectors of V columns that rotate (one half of them in the half layout)
  int copy_vecs, copy_items;  // and that are copied; an item is up to two vectors
  int items;                  // per row
  Divisor by_items, by_heads;
  int pos64, freq64;
  float mscale;
  int inverse;
};

template <typename T, int V> struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// (cos, sin) of the block's tokens into shared memory, [token][pair e of a vector][vector]
// with PV pairs per vector, so the threads of a warp read neighbouring words.
template <int PV>
__device__ __forceinline__ void fill_table(const PosArgs& a, int64_t t0, int nt, int vecs, float2* table) {
  for (int j = threadIdx.x; j < nt * a.pairs; j += kThreads) {
    const int tok = j / a.pairs, i = j % a.pairs;
    const double pos = a.pos64 ? (double)((const int64_t*)a.positions)[t0 + tok]
                               : (double)((const int32_t*)a.positions)[t0 + tok];
    const double f = a.freq64 ? ((const double*)a.inv_freq)[i] : (double)((const float*)a.inv_freq)[i];
    const double turns = pos * (f * 0.15915494309189533576888);  // 1 / (2 pi)
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    table[(tok * PV + i % PV) * vecs + i / PV] = make_float2(c * a.mscale, (a.inverse ? -s : s) * a.mscale);
  }
}

// V elements per vector, an item is two of them. Half layout: V pairs, the vectors rd / 2
// apart. Interleaved, and the columns that are only copied: two vectors of V / 2 pairs
// (or V copied columns) each, half of the row's vectors apart; the second is missing in the
// last item of an odd number.
// COPY: there are columns that are only copied.
template <typename T, int V, bool INTER, bool COPY>
__global__ void __launch_bounds__(kThreads, 6)
rope_positions_kernel(const __grid_constant__ PosArgs a) {
  constexpr int PV = INTER ? V / 2 : V;  // pairs per vector
  extern __shared__ float2 table[];
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens_per_block;
  const int nt = (int)(a.tokens - t0 < a.tokens_per_block ? a.tokens - t0 : a.tokens_per_block);
  const int h0 = blockIdx.y * a.heads_per_block;
  const int nh = a.total_heads - h0 < a.heads_per_block ? a.total_heads - h0 : a.heads_per_block;
  fill_table<PV>(a, t0, nt, a.rot_vecs, table);
  __syncthreads();

  const int n = nt * nh * a.items;
  for (int idx = threadIdx.x; idx < n; idx += kThreads) {
    const uint32_t row = a.by_items.div(idx);
    int item = idx - row * a.items;
    const int tok = a.by_heads.div(row);
    const int h = h0 + row - tok * nh;
    const int which = h >= a.t[0].heads;
    const PosTensor& tz = a.t[which];
    const int head = h - (which ? a.t[0].heads : 0);
    const int64_t t = t0 + tok;
    const bool rot = !COPY || item < a.rot_items;
    item -= rot ? 0 : a.rot_items;
    const int apart = rot ? a.rot_items : a.copy_items;  // vectors between the item's two
    const int col = (rot ? 0 : a.rd) + item * V;
    const bool two = (rot && !INTER) || item + apart < (rot ? a.rot_vecs : a.copy_vecs);
    const T* src = (const T*)tz.x + t * tz.xst + head * tz.xsh + col;
    T* dst = (T*)tz.y + t * tz.yst + head * tz.ysh + col;
    Pack<T, V> lo = *reinterpret_cast<const Pack<T, V>*>(src), hi = lo;
    if (two) hi = *reinterpret_cast<const Pack<T, V>*>(src + apart * V);
    if (rot) {
      const float2* cs = table + tok * PV * a.rot_vecs + item;
#pragma unroll
      for (int e = 0; e < PV; ++e) {
        if constexpr (INTER) {
          const float2 w = cs[e * a.rot_vecs];
          const float2 z = two ? cs[e * a.rot_vecs + apart] : w;
          const float a1 = to_f32<T>(lo.v[2 * e]), a2 = to_f32<T>(lo.v[2 * e + 1]);
          const float b1 = to_f32<T>(hi.v[2 * e]), b2 = to_f32<T>(hi.v[2 * e + 1]);
          lo.v[2 * e] = from_f32<T>(fmaf(a1, w.x, -(a2 * w.y)));
          lo.v[2 * e + 1] = from_f32<T>(fmaf(a2, w.x, a1 * w.y));
          hi.v[2 * e] = from_f32<T>(fmaf(b1, z.x, -(b2 * z.y)));
          hi.v[2 * e + 1] = from_f32<T>(fmaf(b2, z.x, b1 * z.y));
        } else {
          const float2 w = cs[e * a.rot_vecs];
          const float x1 = to_f32<T>(lo.v[e]), x2 = to_f32<T>(hi.v[e]);
          lo.v[e] = from_f32<T>(fmaf(x1, w.x, -(x2 * w.y)));
          hi.v[e] = from_f32<T>(fmaf(x2, w.x, x1 * w.y));
        }
      }
    }
    *reinterpret_cast<Pack<T, V>*>(dst) = lo;
    if (two) *reinterpret_cast<Pack<T, V>*>(dst + apart * V) = hi;
  }
}

// Interleaved pairs whose elements are not aligned to a pair: element by element.
template <typename T>
__global__ void __launch_bounds__(kThreads)
rope_positions_scalar_kernel(const __grid_constant__ PosArgs a) {
  extern __shared__ float2 table[];  // [token][pair]
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens_per_block;
  const int nt = (int)(a.tokens - t0 < a.tokens_per_block ? a.tokens - t0 : a.tokens_per_block);
  const int h0 = blockIdx.y * a.heads_per_block;
  const int nh = a.total_heads - h0 < a.heads_per_block ? a.total_heads - h0 : a.heads_per_block;
  fill_table<1>(a, t0, nt, a.pairs, table);
  __syncthreads();
  const int n = nt * nh * a.items;
  for (int idx = threadIdx.x; idx < n; idx += kThreads) {
    const uint32_t row = a.by_items.div(idx);
    const int item = idx - row * a.items;
    const int tok = a.by_heads.div(row);
    const int h = h0 + row - tok * nh;
    const int which = h >= a.t[0].heads;
    const PosTensor& tz = a.t[which];
    const int head = h - (which ? a.t[0].heads : 0);
    const T* src = (const T*)tz.x + (t0 + tok) * tz.xst + head * tz.xsh;
    T* dst = (T*)tz.y + (t0 + tok) * tz.yst + head * tz.ysh;
    if (item < a.pairs) {
      const float2 w = table[tok * a.pairs + item];
      const float x1 = to_f32<T>(src[2 * item]), x2 = to_f32<T>(src[2 * item + 1]);
      dst[2 * item] = from_f32<T>(fmaf(x1, w.x, -(x2 * w.y)));
      dst[2 * item + 1] = from_f32<T>(fmaf(x2, w.x, x1 * w.y));
    } else {
      const int col = a.rd + item - a.pairs;
      dst[col] = src[col];
    }
  }
}

template <typename T>
int launch_positions(PosArgs& a, int count, int64_t D, bool interleaved, cudaStream_t stream) {
  // Widest vector every address is a multiple of.
  int V = 16 / (int)sizeof(T);
  auto fits = [&](int v) {
    if ((interleaved ? a.rd : a.pairs) % v || (D - a.rd) % v) return false;
    for (int i = 0; i < count; ++i) {
      const PosTensor& t = a.t[i];
      const uintptr_t bytes = v * sizeof(T);
      if ((uintptr_t)t.x % bytes || (uintptr_t)t.y % bytes || t.xst % v || t.xsh % v || t.yst % v ||
          t.ysh % v)
        return false;
    }
    return true;
  };
  while (V > 1 && !fits(V)) V /= 2;
  const bool scalar = interleaved && V == 1;
  a.rot_vecs = scalar ? a.pairs : (interleaved ? a.rd : a.pairs) / V;
  a.rot_items = interleaved && !scalar ? (a.rot_vecs + 1) / 2 : a.rot_vecs;
  a.copy_vecs = (int)((D - a.rd) / V);
  a.copy_items = scalar ? a.copy_vecs : (a.copy_vecs + 1) / 2;
  a.items = a.rot_items + a.copy_items;
  // A block takes whole tokens with all their heads, about three rounds of items, fewer
  // when that would leave SMs without a block; heads are cut when one token is too much
  // for a block or there are few tokens.
  const int64_t per_token = (int64_t)a.total_heads * a.items;
  const int sms = device_info().sm_count;
  int64_t tb = (kThreads * 3 + per_token - 1) / per_token;
  if (tb > (a.tokens + 2 * sms - 1) / (2 * sms)) tb = (a.tokens + 2 * sms - 1) / (2 * sms);
  if (tb > kTableFloats / 2 / a.pairs) tb = kTableFloats / 2 / a.pairs;
  if (tb < 1) tb = 1;
  int64_t hb = a.total_heads;
  const int64_t blocks_t = (a.tokens + tb - 1) / tb;
  if (blocks_t < sms || per_token > kThreads * 64) {
    // one round of items per block while tokens alone do not fill the machine
    const int64_t rounds = blocks_t < sms ? 1 : 64;
    hb = (kThreads * rounds + a.items - 1) / a.items;
    if (hb > a.total_heads) hb = a.total_heads;
    if ((a.total_heads + hb - 1) / hb > 65535) hb = (a.total_heads + 65534) / 65535;
  }
  a.tokens_per_block = (int)tb;
  a.heads_per_block = (int)hb;
  a.by_items.set(a.items);
  // The last block along the heads has fewer: it divides by its own count below, so cut evenly
  // where possible and otherwise keep one token per block (the quotient is then zero).
  if (a.total_heads % hb && tb > 1) {
    a.tokens_per_block = 1;
    tb = 1;
  }
  a.by_heads.set((uint32_t)hb);
  const dim3 grid((unsigned)((a.tokens + tb - 1) / tb), (unsigned)((a.total_heads + hb - 1) / hb));
  const size_t smem = (size_t)tb * a.pairs * sizeof(float2);
  if (scalar) {
    rope_positions_scalar_kernel<T><<<grid, kThreads, smem, stream>>>(a);
    return check_launch("rope_positions");
  }
#define EVG_ROPE_V(v)                                                                           \
  if (V == v) {                                                                                 \
    constexpr int w = v < 2 ? 2 : v; /* interleaved pairs are whole vectors */                  \
    if (interleaved && a.copy_vecs) rope_positions_kernel<T, w, true, true><<<grid, kThreads, smem, stream>>>(a); \
    else if (interleaved) rope_positions_kernel<T, w, true, false><<<grid, kThreads, smem, stream>>>(a);          \
    else if (a.copy_vecs) rope_positions_kernel<T, v, false, true><<<grid, kThreads, smem, stream>>>(a);          \
    else rope_positions_kernel<T, v, false, false><<<grid, kThreads, smem, stream>>>(a);        \
  }
  if constexpr (sizeof(T) == 2) EVG_ROPE_V(8)
  EVG_ROPE_V(4) EVG_ROPE_V(2) EVG_ROPE_V(1)
#undef EVG_ROPE_V
  return check_launch("rope_positions");
}

}  // namespace
}  // namespace evg

using namespace evg;

extern "C" int evg_rope_positions(const evg_rope_positions_tensor* tensors, int count,
                                  const void* positions, int position_bytes, const void* inv_freq,
                                  int freq_bytes, int64_t tokens, int64_t head_dim,
                                  int64_t rotary_dim, int interleaved, float mscale, int dtype,
                                  int inverse, void* stream) {
  const char* what = "rope_positions";
  if (!tensors) return fail(EVG_ENULL, "%s: null pointer argument", what);
  if (count < 1 || count > kMaxTensors)
    return fail(EVG_EBADSHAPE, "%s: count=%d (1 or 2 tensors per launch)", what, count);
  if (tokens < 0 || tokens > 0x7fffffff || head_dim <= 0 || head_dim > 4096 || rotary_dim < 2 ||
      rotary_dim % 2 || rotary_dim > head_dim)
    return fail(EVG_EBADSHAPE,
                "%s: tokens=%lld head_dim=%lld (at most 4096) rotary_dim=%lld (even, 2 .. head_dim)",
                what, (long long)tokens, (long long)head_dim, (long long)rotary_dim);
  if ((position_bytes != 4 && position_bytes != 8) || (freq_bytes != 4 && freq_bytes != 8))
    return fail(EVG_EDTYPE, "%s: positions of %d bytes, frequencies of %d bytes (4 or 8 each)", what,
                position_bytes, freq_bytes);
  PosArgs a{};
  int64_t total = 0;
  for (int i = 0; i < count; ++i) {
    const evg_rope_positions_tensor& t = tensors[i];
    if (t.heads < 0 || t.heads > 65535)
      return fail(EVG_EBADSHAPE, "%s: tensor %d has %lld heads (0 .. 65535)", what, i, (long long)t.heads);
    if (tokens > 0 && t.heads > 0 && (!t.x || !t.y))
      return fail(EVG_ENULL, "%s: tensor %d has a null pointer", what, i);
    a.t[i] = PosTensor{t.x, t.y, (int)t.heads, t.x_stride_t, t.x_stride_h, t.y_stride_t, t.y_stride_h};
    total += t.heads;
  }
  if (tokens == 0 || total == 0) return EVG_OK;
  // Rows are turned at the same time: in place is one row over itself, anything else a race.
  for (int i = 0; i < count; ++i)
    for (int j = 0; j < count; ++j) {
      const evg_rope_positions_tensor &y = tensors[i], &x = tensors[j];
      if (y.heads == 0 || x.heads == 0) continue;
      const bool moved = (tokens > 1 && y.y_stride_t != x.x_stride_t) || (x.heads > 1 && y.y_stride_h != x.x_stride_h);
      if ((y.y == x.x && (i != j || moved)) || (i < j && y.y == x.y))
        return fail(EVG_EBADSHAPE, "%s: output %d lies over another tensor, or over its own in another order", what, i);
    }
  if (!positions || !inv_freq) return fail(EVG_ENULL, "%s: null pointer argument", what);
  if ((uintptr_t)positions % position_bytes || (uintptr_t)inv_freq % freq_bytes)
    return fail(EVG_EALIGN, "%s: positions / frequencies are not aligned to their element", what);
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.tokens = tokens;
  a.total_heads = (int)total;
  a.rd = (int)rotary_dim;
  a.pairs = (int)(rotary_dim / 2);
  a.pos64 = position_bytes == 8;
  a.freq64 = freq_bytes == 8;
  a.mscale = mscale;
  a.inverse = inverse != 0;
  return EVG_DISPATCH_DTYPE(dtype, [&] {
    return launch_positions<T>(a, count, head_dim, interleaved != 0, (cudaStream_t)stream);
  });
}
