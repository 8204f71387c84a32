// Global gradient norm over many tensors and clipping (sm_100a):
//   N = sqrt(sum over all tensors of g^2),  g <- g c,  c = min(1, max_norm / (N + 1e-6))
//
// Two kernels over a list of tensors that travels in the kernel's parameters (no copy
// to the device, capturable): every block squares its 16384-element chunks in float32 (a
// thread's at most 64 squares per chunk; in float64 where float32 has too little range) and
// adds the chunks up in float64, one partial per block; the second kernel's blocks each add all partials in the same fixed order
// and scale their chunks. Fixed order throughout, so the result is reproducible. The
// second kernel walks the chunks backwards: what the first one read last is still in L2.
//
// HBM-bound: two reads and one write per element (the scaling needs the finished norm);
// in place and with nothing to clip, one read. 218 M bf16 elements, two reads and a write:
// 218 us, 6.0 TB/s. Four resident blocks per SM with four loads in flight per thread
// against six and eight blocks (spills: 237 us) or eight loads (224 us).
#include <algorithm>
#include <memory>
#include <new>

#include "evg_common.cuh"

namespace evg {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 16384;  // elements
constexpr int kBlocksPerSm = 4;  // all resident: the chunks are walked in order
constexpr int kUnroll = 4;       // 16-byte loads in flight per thread
constexpr int kMaxBlocks = 148 * 8;

struct Entry {
  const void* in;
  void* out;
  int64_t n;
  int first_chunk;
  int dtype;  // | 8: addresses are 16-byte aligned
};
template <int CAP> struct Table {
  Entry e[CAP];
  int count, chunks;
};

template <int CAP>
__device__ __forceinline__ int find_entry(const Table<CAP>& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first_chunk <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// A thread's part of a chunk's squares; `bits`: all elements' bits but the signs, or-ed.
template <typename T>
__device__ __forceinline__ float chunk_squares(const T* p, int n, bool vec, uint32_t& bits) {
  constexpr int N = Vec<T>::N;
  constexpr uint32_t kNoSigns = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
  bits = 0;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  int done = 0;
  if (vec) {
    const int nv = n / N;
    done = nv * N;
    for (int base = threadIdx.x; base < nv; base += kThreads * kUnroll) {
      uint4 v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (base + u * kThreads < nv) v[u] = ld_vec(p + (int64_t)(base + u * kThreads) * N);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (base + u * kThreads < nv) {
          float f[N];
          unpack<T>(v[u], f);
          bits |= (v[u].x | v[u].y | v[u].z | v[u].w) & kNoSigns;
#pragma unroll
          for (int i = 0; i < N; ++i) s[u & 3] = fmaf(f[i], f[i], s[u & 3]);
        }
    }
  }
  for (int i = done + threadIdx.x; i < n; i += kThreads) {
    const float f = to_f32<T>(p[i]);
    bits |= __float_as_uint(f) & 0x7fffffffu;
    s[0] = fmaf(f, f, s[0]);
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}
// A thread whose squares leave float32 adds the same elements again in float64: an infinite sum
// (elements from 1.8e19 on), or one below 2^-110 with an element that is not zero (elements
// below 2.8e-17; a square below 2^-126 is off by up to 2^-150, 64 of them from there on by less
// than 2^-33 of the sum). Chunks of zeros, common in the gradients of embeddings, are read once.
template <typename T>
__device__ __forceinline__ double chunk_sum(const T* p, int n, bool vec) {
  uint32_t bits;
  const float s = chunk_squares(p, n, vec, bits);
  if (s <= 3.402823466e38f && (s >= 0x1p-110f || bits == 0)) return (double)s;
  double d = 0.0;
  auto add = [&](int i) {
    const double f = (double)to_f32<T>(p[i]);
    d = fma(f, f, d);
  };
  constexpr int N = Vec<T>::N;
  const int nv = vec ? n / N : 0;
  for (int v = threadIdx.x; v < nv; v += kThreads)
    for (int i = 0; i < N; ++i) add(v * N + i);
  for (int i = nv * N + threadIdx.x; i < n; i += kThreads) add(i);
  return d;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* in, T* out, int n, bool vec, float c) {
  constexpr int N = Vec<T>::N;
  int done = 0;
  if (vec) {
    const int nv = n / N;
    done = nv * N;
    for (int base = threadIdx.x; base < nv; base += kThreads * kUnroll) {
      uint4 v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (base + u * kThreads < nv) v[u] = *reinterpret_cast<const uint4*>(in + (int64_t)(base + u * kThreads) * N);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (base + u * kThreads < nv) {
          float f[N];
          unpack<T>(v[u], f);
#pragma unroll
          for (int i = 0; i < N; ++i) f[i] *= c;
          st_vec(out + (int64_t)(base + u * kThreads) * N, pack<T>(f));
        }
    }
  }
  for (int i = done + threadIdx.x; i < n; i += kThreads) out[i] = from_f32<T>(to_f32<T>(in[i]) * c);
}

__device__ __forceinline__ double block_sum(double v, double* scratch) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) s += scratch[w];
  return s;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
grad_squares_kernel(const __grid_constant__ Table<CAP> t, double* __restrict__ partial) {
  __shared__ double scratch[kThreads / 32];
  double mine = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const Entry& e = t.e[find_entry(t, c)];
    const int64_t at = (int64_t)(c - e.first_chunk) * kChunk;
    const int n = (int)(e.n - at < kChunk ? e.n - at : kChunk);
    const bool vec = e.dtype & 8;
    switch (e.dtype & 7) {
      case EVG_F32: mine += chunk_sum((const float*)e.in + at, n, vec); break;
      case EVG_F16: mine += chunk_sum((const __half*)e.in + at, n, vec); break;
      default: mine += chunk_sum((const __nv_bfloat16*)e.in + at, n, vec); break;
    }
  }
  const double s = block_sum(mine, scratch);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
grad_scale_kernel(const __grid_constant__ Table<CAP> t, const double* __restrict__ partial,
                  int partials, float max_norm, int clip, float* __restrict__ norm_out) {
  __shared__ double scratch[kThreads / 32];
  double s = 0.0;
  for (int i = threadIdx.x; i < partials; i += kThreads) s += partial[i];
  const double norm = sqrt(block_sum(s, scratch));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  if (!clip) return;
  const double ratio = (double)max_norm / (norm + 1e-6);
  const float coef = ratio > 1.0 ? 1.0f : (float)ratio;  // a NaN norm stays NaN
  for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const Entry& e = t.e[find_entry(t, c)];
    if (coef == 1.0f && e.in == e.out) continue;  // in place with nothing to clip
    const int64_t at = (int64_t)(c - e.first_chunk) * kChunk;
    const int n = (int)(e.n - at < kChunk ? e.n - at : kChunk);
    const bool vec = e.dtype & 8;
    switch (e.dtype & 7) {
      case EVG_F32: chunk_scale((const float*)e.in + at, (float*)e.out + at, n, vec, coef); break;
      case EVG_F16: chunk_scale((const __half*)e.in + at, (__half*)e.out + at, n, vec, coef); break;
      default: chunk_scale((const __nv_bfloat16*)e.in + at, (__nv_bfloat16*)e.out + at, n, vec, coef); break;
    }
  }
}

int64_t launches_for(int64_t count, int cap) { return count > 0 ? (count + cap - 1) / cap : 1; }

template <int CAP>
int run(const void* const* in, void* const* out, const int64_t* numel, const int* dtypes,
        int64_t count, float max_norm, int clip, float* norm, double* partial, cudaStream_t st) {
  const int resident = device_info().sm_count * kBlocksPerSm;
  const int most = resident < kMaxBlocks ? resident : kMaxBlocks;
  const int64_t launches = launches_for(count, CAP);
  int used = 0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t l = 0; l < launches; ++l) {
      // the second pass takes the lists in reverse as well
      const int64_t first = (pass ? launches - 1 - l : l) * CAP;
      Table<CAP> t;
      t.count = 0;
      t.chunks = 0;
      for (int64_t i = first; i < count && i < first + CAP; ++i) {
        if (numel[i] == 0) continue;
        Entry& e = t.e[t.count++];
        e.in = in[i];
        e.out = out ? out[i] : const_cast<void*>(in[i]);
        e.n = numel[i];
        e.first_chunk = t.chunks;
        e.dtype = dtypes[i] | (aligned16(e.in) && aligned16(e.out) ? 8 : 0);
        t.chunks += (int)((numel[i] + kChunk - 1) / kChunk);
      }
      int blocks = t.chunks < most ? t.chunks : most;
      if (blocks < 1) blocks = 1;
      if (pass == 0) {
        grad_squares_kernel<CAP><<<blocks, kThreads, 0, st>>>(t, partial + used);
        used += blocks;
      } else {
        grad_scale_kernel<CAP><<<clip ? blocks : 1, kThreads, 0, st>>>(t, partial, used, max_norm, clip,
                                                                       l == 0 ? norm : nullptr);
      }
      if (int rc = check_launch("clip_grads")) return rc;
      if (pass == 1 && !clip) break;
    }
  }
  return EVG_OK;
}

constexpr int kSmallCap = 48, kLargeCap = 480;

// Memory of one tensor. Blocks scale the tensors at the same time, so what one of them writes
// may not overlap anything that another reads or writes.
struct Span {
  uintptr_t begin, end;
  bool written;
};
int check_overlaps(const char* what, const void* const* in, void* const* out, const int64_t* numel,
                   const int* dtypes, int64_t count) {
  constexpr int kFew = 96;
  Span few[kFew];
  std::unique_ptr<Span[]> many;
  Span* spans = few;
  if (2 * count > kFew) {
    many.reset(new (std::nothrow) Span[2 * count]);
    if (!many) return fail(EVG_ELAUNCH, "%s: no host memory for %lld tensors", what, (long long)count);
    spans = many.get();
  }
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (numel[i] == 0) continue;
    const uintptr_t bytes = (uintptr_t)numel[i] * dtype_size(dtypes[i]), a = (uintptr_t)in[i];
    const bool in_place = !out || out[i] == in[i];
    spans[n++] = Span{a, a + bytes, in_place};
    if (!in_place) spans[n++] = Span{(uintptr_t)out[i], (uintptr_t)out[i] + bytes, true};
  }
  const auto before = [](const Span& x, const Span& y) { return x.begin < y.begin; };
  if (!std::is_sorted(spans, spans + n, before)) std::sort(spans, spans + n, before);
  uintptr_t reach = 0, written = 0;  // ends of the spans so far
  for (int64_t i = 0; i < n; ++i) {
    const Span& s = spans[i];
    if (s.begin < (s.written ? reach : written))
      return fail(EVG_EBADSHAPE, "%s: a tensor that is written overlaps another one", what);
    reach = std::max(reach, s.end);
    if (s.written) written = std::max(written, s.end);
  }
  return EVG_OK;
}

}  // namespace
}  // namespace evg

using namespace evg;

extern "C" int64_t evg_clip_grads_workspace_bytes(int64_t count) {
  if (count < 0) return 0;
  return launches_for(count, kLargeCap) * kMaxBlocks * (int64_t)sizeof(double);
}

extern "C" int evg_clip_grads(const void* const* grads, void* const* outs, const int64_t* numel,
                              const int* dtypes, int64_t count, float max_norm, int clip,
                              float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "clip_grads";
  if (count < 0) return fail(EVG_EBADSHAPE, "%s: count=%lld", what, (long long)count);
  if (!norm || (count > 0 && (!grads || !numel || !dtypes)))
    return fail(EVG_ENULL, "%s: null pointer argument", what);
  if (clip && !(max_norm >= 0.f))
    return fail(EVG_EBADSHAPE, "%s: max_norm %g (must not be negative)", what, (double)max_norm);
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (numel[i] < 0) return fail(EVG_EBADSHAPE, "%s: tensor %lld has %lld elements", what, (long long)i, (long long)numel[i]);
    if (dtypes[i] != EVG_F32 && dtypes[i] != EVG_F16 && dtypes[i] != EVG_BF16)
      return fail(EVG_EDTYPE, "%s: tensor %lld has dtype %d", what, (long long)i, dtypes[i]);
    if (numel[i] > 0 && (!grads[i] || (outs && !outs[i])))
      return fail(EVG_ENULL, "%s: tensor %lld has a null pointer", what, (long long)i);
    chunks += (numel[i] + kChunk - 1) / kChunk;
  }
  if (chunks > 0x7fffffff) return fail(EVG_EUNSUPPORTED, "%s: too many elements", what);
  const int64_t need = evg_clip_grads_workspace_bytes(count);
  if (!workspace || workspace_bytes < need)
    return fail(EVG_EWORKSPACE, "%s: workspace %lld bytes, need %lld", what, (long long)workspace_bytes, (long long)need);
  if (!aligned16(workspace)) return fail(EVG_EALIGN, "%s: the workspace must be 16-byte aligned", what);
  if (clip)
    if (int rc = check_overlaps(what, grads, outs, numel, dtypes, count)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  // a short list travels in 2 KB of kernel parameters instead of 16
  return count <= kSmallCap
             ? run<kSmallCap>(grads, outs, numel, dtypes, count, max_norm, clip, norm, (double*)workspace, st)
             : run<kLargeCap>(grads, outs, numel, dtypes, count, max_norm, clip, norm, (double*)workspace, st);
}
