// Group norm with an activation, channels last, forward and backward.
//
//   sample n, group g (m = length * channels / groups values): mean, var = mean of (x - mean)^2, r = 1 / sqrt(var + eps)
//   xh = (x - mean) r      z = xh w[c] + b[c]      y = act(z)
//   backward, dz = dy act'(z):   db[c] = sum_{n,l} dz     dw[c] = sum_{n,l} dz xh
//     A = 1/m sum_group w dz     B = 1/m sum_group w dz xh     dx = r (w dz - A - xh B)
//
// Memory-bound.  In a channels-last array the channels of a group lie side by side and its positions far apart, so a
// workgroup takes whole rows (all channels, or a slab of whole groups where a row is too wide) of a stretch of positions:
// its accesses are contiguous whatever the groups are.  A thread keeps to V neighbouring channels and walks over positions.
//
// Statistics: float32.  Each thread sums its values and squares about the first of them - a member of the set it
// describes, so at most a factor (number of values) of the sum of squares cancels, whatever the mean is - and the parts
// are joined by counts, means and sums of squared deviations, which cancels nothing.  The backward pass needs only
// sums per (sample, channel); the groups' A and B and the parameters' gradients are sums of those.
#include <hip/hip_runtime.h>
#include <algorithm>

#include "nsa_elem.h"

#define GN_THREADS 256

// ---------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------

__device__ __forceinline__ float gn_sigmoid(float z) { return 1.0f / (1.0f + expf(-z)); }

template <int ACT>
__device__ __forceinline__ float gn_act(float z) {
  if constexpr (ACT == NSA_FN_RELU) return z < 0.0f ? 0.0f : z;  // (NaN stays)
  else if constexpr (ACT == NSA_FN_TANH) return tanhf(z);
  else if constexpr (ACT == NSA_FN_SILU) return z * gn_sigmoid(z);
  else return z;
}

template <int ACT>
__device__ __forceinline__ float gn_slope(float z) {
  if constexpr (ACT == NSA_FN_RELU) return z > 0.0f ? 1.0f : 0.0f;
  else if constexpr (ACT == NSA_FN_TANH) {
    const float t = tanhf(z);
    return 1.0f - t * t;
  } else if constexpr (ACT == NSA_FN_SILU) {
    const float s = gn_sigmoid(z);
    return s * (1.0f + z * (1.0f - s));
  } else return 1.0f;
}

// ---------------------------------------------------------------------------
// how the work is cut
// ---------------------------------------------------------------------------

// A slab is `gps` whole groups, `width` channels.  A workgroup works on (sample, slab, chunk of positions); thread t on
// channels [V j, V j + V) of the slab, j = t % vecs, and on positions t / vecs, + rows, ...  A group wider than a
// workgroup (one group per slab then) is walked in `tiles` steps of vecs * V channels.
struct GnShape {
  long long samples, length;
  int channels, groups, cpg;   // cpg: channels per group
  int gps, width, slabs;       // slab
  int vecs, rows, tiles;       // threads of a workgroup: vecs * rows <= GN_THREADS
  int chunks;                  // of a sample's positions
  long long chunk;             // positions per chunk
};

struct GnParams {  // weight and bias in float32 or in x's type, or none
  const void *w, *b;
  int f32;
};

template <typename T>
__device__ __forceinline__ float gn_param(const void* p, int f32, int c, float none) {
  if (p == nullptr) return none;
  return f32 ? ((const float*)p)[c] : (float)((const T*)p)[c];
}

struct GnPlace {  // what this workgroup works on
  long long n, l0, l1;
  int slab, chunk, j, r;
  bool active;
};

__device__ __forceinline__ GnPlace gn_place(const GnShape& s) {
  GnPlace p;
  long long b = blockIdx.x;
  p.chunk = (int)(b % s.chunks);
  b /= s.chunks;
  p.slab = (int)(b % s.slabs);
  p.n = b / s.slabs;
  p.l0 = p.chunk * s.chunk;
  p.l1 = p.l0 + s.chunk < s.length ? p.l0 + s.chunk : s.length;
  p.j = threadIdx.x % s.vecs;
  p.r = threadIdx.x / s.vecs;
  p.active = p.r < s.rows;
  return p;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

// (mean, sum of squared deviations) of each group over this workgroup's positions -> part[(n * chunks + chunk) * groups + g]
template <typename T, int V>
__global__ void __launch_bounds__(GN_THREADS) gn_stats(GnShape s, const T* __restrict__ x, float2* __restrict__ part) {
  __shared__ float means[GN_THREADS * V], devs[GN_THREADS * V];
  __shared__ int counts[GN_THREADS];
  const GnPlace p = gn_place(s);
  float shift[V], sum[V], sq[V];
#pragma unroll
  for (int i = 0; i < V; ++i) shift[i] = sum[i] = sq[i] = 0.0f;
  int count = 0;
  if (p.active) {
    for (int t = 0; t < s.tiles; ++t) {
      const int c = (t * s.vecs + p.j) * V;
      if (c >= s.width) break;
      const T* px = x + (p.n * s.length + p.l0 + p.r) * s.channels + p.slab * s.width + c;
      for (long long l = p.l0 + p.r; l < p.l1; l += s.rows, px += (long long)s.rows * s.channels) {
        float v[V];
        nsa_load<T, V>(px, v);
        if (count == 0) {
#pragma unroll
          for (int i = 0; i < V; ++i) shift[i] = v[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = v[i] - shift[i];
          sum[i] += d;
          sq[i] = fmaf(d, d, sq[i]);
        }
        ++count;
      }
    }
  }
  const float inv = count > 0 ? 1.0f / (float)count : 0.0f;
  counts[threadIdx.x] = count;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float d = sum[i] * inv;
    means[threadIdx.x * V + i] = shift[i] + d;
    devs[threadIdx.x * V + i] = fmaxf(sq[i] - sum[i] * d, 0.0f);
  }
  __syncthreads();
  // a wave per group joins the parts: rows x (channels of the group in a tile), in a fixed order
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int span = s.vecs * V;                              // channels in the parts of a row
  const int in_group = s.cpg < span ? s.cpg : span;         // of them, in one group
  const long long rows_here = p.l1 - p.l0;
  const float total = (float)rows_here * (float)s.cpg;
  for (int g = wave; g < s.gps; g += GN_THREADS / 64) {
    const int first = g * s.cpg, parts = in_group * s.rows;
    float a = 0.0f;
    for (int e = lane; e < parts; e += 64) {
      const int c = first + e % in_group, r = e / in_group, t = r * s.vecs + c / V;
      a += (float)counts[t] * means[r * span + c];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o);
    const float mean = a / total;
    float m2 = 0.0f;
    for (int e = lane; e < parts; e += 64) {
      const int c = first + e % in_group, r = e / in_group, t = r * s.vecs + c / V;
      const float d = means[r * span + c] - mean;
      m2 += devs[r * span + c] + (counts[t] > 0 ? (float)counts[t] * d * d : 0.0f);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m2 += __shfl_xor(m2, o);
    if (lane == 0) part[(p.n * s.chunks + p.chunk) * s.groups + p.slab * s.gps + g] = make_float2(mean, m2);
  }
}

// the chunks of a (sample, group) joined; a thread each
__global__ void __launch_bounds__(GN_THREADS) gn_stats_join(GnShape s, const float2* __restrict__ part, float eps,
                                                            float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  const long long i = (long long)blockIdx.x * GN_THREADS + threadIdx.x;
  if (i >= s.samples * s.groups) return;
  const long long n = i / s.groups, g = i % s.groups;
  double mean = 0.0, m2 = 0.0, count = 0.0;
  for (int k = 0; k < s.chunks; ++k) {
    const float2 q = part[(n * s.chunks + k) * s.groups + g];
    const long long l0 = k * s.chunk, rows = (l0 + s.chunk < s.length ? l0 + s.chunk : s.length) - l0;
    const double c = (double)rows * s.cpg, d = (double)q.x - mean, all = count + c;
    mean += d * (c / all);
    m2 += (double)q.y + d * d * (count * c / all);
    count = all;
  }
  mean_out[i] = (float)mean;
  rstd_out[i] = (float)(1.0 / sqrt(m2 / count + (double)eps));
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_apply(GnShape s, const T* __restrict__ x, GnParams q,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd,
                                                       T* __restrict__ y) {
  const GnPlace p = gn_place(s);
  if (!p.active) return;
  for (int t = 0; t < s.tiles; ++t) {
    const int c = (t * s.vecs + p.j) * V;
    if (c >= s.width) break;
    float mu[V], rs[V], w[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int ch = p.slab * s.width + c + i;
      mu[i] = mean[p.n * s.groups + ch / s.cpg];
      rs[i] = rstd[p.n * s.groups + ch / s.cpg];
      w[i] = gn_param<T>(q.w, q.f32, ch, 1.0f);
      b[i] = gn_param<T>(q.b, q.f32, ch, 0.0f);
    }
    long long at = (p.n * s.length + p.l0 + p.r) * s.channels + p.slab * s.width + c;
    for (long long l = p.l0 + p.r; l < p.l1; l += s.rows, at += (long long)s.rows * s.channels) {
      float v[V];
      nsa_load<T, V>(x + at, v);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = gn_act<ACT>(fmaf((v[i] - mu[i]) * rs[i], w[i], b[i]));
      nsa_store<T, V>(y + at, v);
    }
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// sums over this workgroup's positions, per channel: part[(n * chunks + chunk) * channels + c] = {sum dz, sum dz xh}
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_sums(GnShape s, const T* __restrict__ x, const T* __restrict__ dy,
                                                      GnParams q, const float* __restrict__ mean,
                                                      const float* __restrict__ rstd, float2* __restrict__ part) {
  __shared__ float2 red[GN_THREADS * V];
  const GnPlace p = gn_place(s);
  for (int t = 0; t < s.tiles; ++t) {
    const int c = (t * s.vecs + p.j) * V;
    float s1[V], s2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0f;
    if (p.active && c < s.width) {
      float mu[V], rs[V], w[V], b[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int ch = p.slab * s.width + c + i;
        mu[i] = mean[p.n * s.groups + ch / s.cpg];
        rs[i] = rstd[p.n * s.groups + ch / s.cpg];
        w[i] = gn_param<T>(q.w, q.f32, ch, 1.0f);
        b[i] = gn_param<T>(q.b, q.f32, ch, 0.0f);
      }
      long long at = (p.n * s.length + p.l0 + p.r) * s.channels + p.slab * s.width + c;
      for (long long l = p.l0 + p.r; l < p.l1; l += s.rows, at += (long long)s.rows * s.channels) {
        float v[V], g[V];
        nsa_load<T, V>(x + at, v);
        nsa_load<T, V>(dy + at, g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float xh = (v[i] - mu[i]) * rs[i];
          const float dz = g[i] * gn_slope<ACT>(fmaf(xh, w[i], b[i]));
          s1[i] += dz;
          s2[i] = fmaf(dz, xh, s2[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = make_float2(s1[i], s2[i]);
    __syncthreads();
    const int span = s.vecs * V;
    for (int e = threadIdx.x; e < span; e += GN_THREADS) {
      const int ch = t * span + e;
      if (ch < s.width) {
        float2 a = make_float2(0.0f, 0.0f);
        for (int r = 0; r < s.rows; ++r) {
          a.x += red[r * span + e].x;
          a.y += red[r * span + e].y;
        }
        part[(p.n * s.chunks + p.chunk) * s.channels + p.slab * s.width + ch] = a;
      }
    }
    __syncthreads();
  }
}

// A wave per (sample, group): the chunks' sums joined into chunk 0's place, and the group's A and B
template <typename T>
__global__ void __launch_bounds__(GN_THREADS) gn_sums_join(GnShape s, float2* __restrict__ part, GnParams q,
                                                           float2* __restrict__ ab) {
  const long long i = (long long)blockIdx.x * (GN_THREADS / 64) + (threadIdx.x >> 6);
  if (i >= s.samples * s.groups) return;
  const long long n = i / s.groups;
  const int g = (int)(i % s.groups), lane = threadIdx.x & 63;
  float a = 0.0f, b = 0.0f;
  for (int c = g * s.cpg + lane; c < (g + 1) * s.cpg; c += 64) {
    float2* first = part + n * s.chunks * s.channels + c;
    float2 t = first[0];
    for (int k = 1; k < s.chunks; ++k) {
      const float2 o = first[(long long)k * s.channels];
      t.x += o.x;
      t.y += o.y;
    }
    first[0] = t;
    const float w = gn_param<T>(q.w, q.f32, c, 1.0f);
    a = fmaf(w, t.x, a);
    b = fmaf(w, t.y, b);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    a += __shfl_xor(a, o);
    b += __shfl_xor(b, o);
  }
  const float m = (float)s.length * (float)s.cpg;
  if (lane == 0) ab[i] = make_float2(a / m, b / m);
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_dx(GnShape s, const T* __restrict__ x, const T* __restrict__ dy, GnParams q,
                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                    const float2* __restrict__ ab, T* __restrict__ dx) {
  const GnPlace p = gn_place(s);
  if (!p.active) return;
  for (int t = 0; t < s.tiles; ++t) {
    const int c = (t * s.vecs + p.j) * V;
    if (c >= s.width) break;
    float mu[V], rs[V], w[V], b[V], ga[V], gb[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int ch = p.slab * s.width + c + i;
      const long long k = p.n * s.groups + ch / s.cpg;
      mu[i] = mean[k];
      rs[i] = rstd[k];
      ga[i] = ab[k].x;
      gb[i] = ab[k].y;
      w[i] = gn_param<T>(q.w, q.f32, ch, 1.0f);
      b[i] = gn_param<T>(q.b, q.f32, ch, 0.0f);
    }
    long long at = (p.n * s.length + p.l0 + p.r) * s.channels + p.slab * s.width + c;
    for (long long l = p.l0 + p.r; l < p.l1; l += s.rows, at += (long long)s.rows * s.channels) {
      float v[V], g[V];
      nsa_load<T, V>(x + at, v);
      nsa_load<T, V>(dy + at, g);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (v[i] - mu[i]) * rs[i];
        const float dz = g[i] * gn_slope<ACT>(fmaf(xh, w[i], b[i]));
        v[i] = rs[i] * (w[i] * dz - ga[i] - xh * gb[i]);
      }
      nsa_store<T, V>(dx + at, v);
    }
  }
}

// The parameters' gradients: `count` records of [channels] sums, `stride` apart, added in a fixed order.  A workgroup per 64
// channels, four waves that take every fourth record each.
template <typename T>
__global__ void __launch_bounds__(GN_THREADS) gn_param_grads(int channels, long long count, long long stride,
                                                             const float2* __restrict__ part, int f32,
                                                             void* __restrict__ dw, void* __restrict__ db) {
  __shared__ float2 red[GN_THREADS];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
  float2 t = make_float2(0.0f, 0.0f);
  if (c < channels)
    for (long long k = wave; k < count; k += GN_THREADS / 64) {
      const float2 o = part[k * stride + c];
      t.x += o.x;
      t.y += o.y;
    }
  red[threadIdx.x] = t;
  __syncthreads();
  if (wave != 0 || c >= channels) return;
  for (int w = 1; w < GN_THREADS / 64; ++w) {
    t.x += red[w * 64 + threadIdx.x].x;
    t.y += red[w * 64 + threadIdx.x].y;
  }
  if (f32) {
    if (dw != nullptr) ((float*)dw)[c] = t.y;
    if (db != nullptr) ((float*)db)[c] = t.x;
  } else {
    if (dw != nullptr) ((T*)dw)[c] = (T)t.y;
    if (db != nullptr) ((T*)db)[c] = (T)t.x;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

// workgroups wanted of a launch: a few for each of the 256 compute units, so that no unit waits for a long one
const long long GN_GROUPS_WANTED = 2048;
// positions of a chunk at least, per row of threads: below it a workgroup's start costs more than its work
const long long GN_CHUNK_ROWS = 8;

GnShape gn_shape(long long samples, long long length, int channels, int groups, int bytes, uintptr_t addresses, int& v) {
  GnShape s;
  s.samples = samples;
  s.length = length;
  s.channels = channels;
  s.groups = groups;
  s.cpg = channels / groups;
  v = 16 / bytes;
  while (v > 1 && (channels % v != 0 || addresses % (uintptr_t)(v * bytes) != 0)) v >>= 1;
  for (;; v >>= 1) {  // the widest access with which slabs of whole groups begin at a multiple of it
    const int most = GN_THREADS * v;
    s.gps = groups;
    if (channels > most) {
      s.gps = std::max(1, most / s.cpg);
      while (s.gps > 1 && (groups % s.gps != 0 || (s.gps * s.cpg) % v != 0)) --s.gps;
    }
    s.width = s.gps * s.cpg;
    s.slabs = groups / s.gps;
    if (v == 1 || s.slabs == 1 || s.width % v == 0) break;
  }
  const int vectors = s.width / v;  // (channels, or a slab of it, is a multiple of v)
  s.vecs = std::min(vectors, GN_THREADS);
  s.tiles = (vectors + s.vecs - 1) / s.vecs;
  s.rows = s.tiles > 1 ? 1 : GN_THREADS / s.vecs;
  const long long per = samples * s.slabs;
  long long chunks = std::max(1LL, (GN_GROUPS_WANTED + per - 1) / per);
  chunks = std::min(chunks, std::max(1LL, length / (s.rows * GN_CHUNK_ROWS)));
  s.chunk = (length + chunks - 1) / chunks;
  s.chunks = (int)((length + s.chunk - 1) / s.chunk);
  return s;
}

// An upper bound that does not ask for the addresses: chunks do not grow with a narrower access by more than the rows do
size_t gn_workspace(long long samples, long long length, int channels, int groups, int bytes, bool backward) {
  size_t most = 0;
  for (int align = bytes; align <= 16; align *= 2) {
    int v;
    const GnShape s = gn_shape(samples, length, channels, groups, bytes, (uintptr_t)align, v);
    const size_t parts = (size_t)s.samples * s.chunks * (backward ? s.channels : s.groups) * sizeof(float2);
    most = std::max(most, parts);
  }
  return most + (backward ? (size_t)samples * groups * sizeof(float2) : 0) + 256;
}

int gn_check(const char* what, long long samples, long long length, int channels, int groups, int dtype, int weight_dtype,
             int activation) {
  if (samples < 0 || length < 0 || channels < 1 || groups < 1 || channels % groups != 0)
    return nsa_fail(NSA_E_ARG, "%s: bad shape (channels must be a multiple of groups)", what);
  if (!nsa_elem_known(dtype)) return nsa_fail(NSA_E_ARG, "%s: unknown type %d", what, dtype);
  if (weight_dtype != NSA_DT_F32 && weight_dtype != dtype)
    return nsa_fail(NSA_E_ARG, "%s: weight and bias are float32 or of x's type", what);
  if (activation < NSA_FN_NONE || activation > NSA_FN_SILU) return nsa_fail(NSA_E_ARG, "%s: unknown activation %d", what, activation);
  if (samples > 0 && length > 0 && samples > (1LL << 46) / length / channels) return nsa_fail(NSA_E_ARG, "%s: too large", what);
  return NSA_OK;
}

int gn_done(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? NSA_OK : nsa_fail(NSA_E_HIP, "%s: %s", what, hipGetErrorString(e));
}

#define GN_ACTS(act, KERNEL, T, V, ...)                                                             \
  switch (act) {                                                                                    \
    case NSA_FN_RELU: hipLaunchKernelGGL((KERNEL<T, V, NSA_FN_RELU>), __VA_ARGS__); break;          \
    case NSA_FN_TANH: hipLaunchKernelGGL((KERNEL<T, V, NSA_FN_TANH>), __VA_ARGS__); break;          \
    case NSA_FN_SILU: hipLaunchKernelGGL((KERNEL<T, V, NSA_FN_SILU>), __VA_ARGS__); break;          \
    default: hipLaunchKernelGGL((KERNEL<T, V, NSA_FN_NONE>), __VA_ARGS__); break;                   \
  }

template <typename T, int V>
void gn_forward(const GnShape& s, const void* x, GnParams q, float eps, int act, void* y, float* mean, float* rstd,
                float2* part, hipStream_t st) {
  const dim3 grid((unsigned)(s.samples * s.slabs * s.chunks)), block(GN_THREADS);
  hipLaunchKernelGGL((gn_stats<T, V>), grid, block, 0, st, s, (const T*)x, part);
  const long long pairs = s.samples * s.groups;
  hipLaunchKernelGGL(gn_stats_join, dim3((unsigned)((pairs + GN_THREADS - 1) / GN_THREADS)), block, 0, st, s, part, eps, mean,
                     rstd);
  GN_ACTS(act, gn_apply, T, V, grid, block, 0, st, s, (const T*)x, q, mean, rstd, (T*)y)
}

template <typename T, int V>
void gn_backward(const GnShape& s, const void* x, const void* dy, GnParams q, int act, const float* mean, const float* rstd,
                 void* dx, void* dw, void* db, float2* part, float2* ab, hipStream_t st) {
  const dim3 grid((unsigned)(s.samples * s.slabs * s.chunks)), block(GN_THREADS);
  GN_ACTS(act, gn_sums, T, V, grid, block, 0, st, s, (const T*)x, (const T*)dy, q, mean, rstd, part)
  const long long pairs = s.samples * s.groups;
  hipLaunchKernelGGL((gn_sums_join<T>), dim3((unsigned)((pairs + GN_THREADS / 64 - 1) / (GN_THREADS / 64))), block, 0, st, s,
                     part, q, ab);
  if (dx != nullptr) {
    GN_ACTS(act, gn_dx, T, V, grid, block, 0, st, s, (const T*)x, (const T*)dy, q, mean, rstd, ab, (T*)dx)
  }
  if (dw != nullptr || db != nullptr)
    hipLaunchKernelGGL((gn_param_grads<T>), dim3((unsigned)((s.channels + 63) / 64)), block, 0, st, s.channels, s.samples,
                       (long long)s.chunks * s.channels, part, q.f32, dw, db);
}

// one call per element type and access width
#define GN_WIDTHS(T, F, ...)                            \
  if (v == 1) F<T, 1>(__VA_ARGS__);                     \
  else if (v == 2) F<T, 2>(__VA_ARGS__);                \
  else if (v == 4) F<T, 4>(__VA_ARGS__);                \
  else if constexpr (sizeof(T) == 2) F<T, 8>(__VA_ARGS__);

}  // namespace

extern "C" NSA_API size_t nsa_group_norm_workspace(long long samples, long long length, int channels, int groups, int dtype,
                                                   int backward) {
  if (samples <= 0 || length <= 0 || channels < 1 || groups < 1 || channels % groups != 0 || !nsa_elem_known(dtype)) return 0;
  return gn_workspace(samples, length, channels, groups, nsa_elem_bytes(dtype), backward != 0);
}

extern "C" NSA_API int nsa_group_norm_forward(long long samples, long long length, int channels, int groups, int dtype,
                                              const void* x_dev, int weight_dtype, const void* weight_dev,
                                              const void* bias_dev, float eps, int activation, void* y_dev, float* mean_dev,
                                              float* rstd_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
  const char* what = "nsa_group_norm_forward";
  if (const int rc = gn_check(what, samples, length, channels, groups, dtype, weight_dtype, activation)) return rc;
  if (samples == 0 || length == 0) return NSA_OK;
  if (!x_dev || !y_dev || !mean_dev || !rstd_dev || !workspace_dev) return nsa_fail(NSA_E_ARG, "%s: NULL argument", what);
  if (workspace_bytes < nsa_group_norm_workspace(samples, length, channels, groups, dtype, 0))
    return nsa_fail(NSA_E_ARG, "%s: workspace too small", what);
  int v;
  const GnShape s = gn_shape(samples, length, channels, groups, nsa_elem_bytes(dtype), (uintptr_t)x_dev | (uintptr_t)y_dev, v);
  if (s.samples * s.slabs * s.chunks >= (1LL << 31)) return nsa_fail(NSA_E_ARG, "%s: too many samples", what);
  const GnParams q = {weight_dev, bias_dev, weight_dtype == NSA_DT_F32};
  hipStream_t st = (hipStream_t)stream;
  float2* part = (float2*)workspace_dev;
  if (dtype == NSA_DT_F32) { GN_WIDTHS(float, gn_forward, s, x_dev, q, eps, activation, y_dev, mean_dev, rstd_dev, part, st) }
  else if (dtype == NSA_DT_BF16) { GN_WIDTHS(nsa_bf16, gn_forward, s, x_dev, q, eps, activation, y_dev, mean_dev, rstd_dev, part, st) }
  else { GN_WIDTHS(nsa_f16, gn_forward, s, x_dev, q, eps, activation, y_dev, mean_dev, rstd_dev, part, st) }
  return gn_done(what);
}

extern "C" NSA_API int nsa_group_norm_backward(long long samples, long long length, int channels, int groups, int dtype,
                                               const void* x_dev, const void* dy_dev, int weight_dtype,
                                               const void* weight_dev, const void* bias_dev, int activation,
                                               const float* mean_dev, const float* rstd_dev, void* dx_dev, void* dweight_dev,
                                               void* dbias_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
  const char* what = "nsa_group_norm_backward";
  if (const int rc = gn_check(what, samples, length, channels, groups, dtype, weight_dtype, activation)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const int f32 = weight_dtype == NSA_DT_F32;
  if (samples == 0 || length == 0) {  // no rows: the parameters' gradients are zero
    if (dweight_dev == nullptr && dbias_dev == nullptr) return NSA_OK;
    hipLaunchKernelGGL((gn_param_grads<nsa_f16>), dim3((unsigned)((channels + 63) / 64)), dim3(GN_THREADS), 0, st, channels,
                       0LL, 0LL, (const float2*)nullptr, f32, dweight_dev, dbias_dev);  // (zero has the same bits in both 16-bit types)
    return gn_done(what);
  }
  if (!x_dev || !dy_dev || !mean_dev || !rstd_dev || !workspace_dev) return nsa_fail(NSA_E_ARG, "%s: NULL argument", what);
  if (workspace_bytes < nsa_group_norm_workspace(samples, length, channels, groups, dtype, 1))
    return nsa_fail(NSA_E_ARG, "%s: workspace too small", what);
  int v;
  const GnShape s = gn_shape(samples, length, channels, groups, nsa_elem_bytes(dtype),
                             (uintptr_t)x_dev | (uintptr_t)dy_dev | (uintptr_t)dx_dev, v);
  if (s.samples * s.slabs * s.chunks >= (1LL << 31)) return nsa_fail(NSA_E_ARG, "%s: too many samples", what);
  const GnParams q = {weight_dev, bias_dev, f32};
  float2* ab = (float2*)workspace_dev;
  float2* part = ab + samples * groups;
  if (dtype == NSA_DT_F32) { GN_WIDTHS(float, gn_backward, s, x_dev, dy_dev, q, activation, mean_dev, rstd_dev, dx_dev, dweight_dev, dbias_dev, part, ab, st) }
  else if (dtype == NSA_DT_BF16) { GN_WIDTHS(nsa_bf16, gn_backward, s, x_dev, dy_dev, q, activation, mean_dev, rstd_dev, dx_dev, dweight_dev, dbias_dev, part, ab, st) }
  else { GN_WIDTHS(nsa_f16, gn_backward, s, x_dev, dy_dev, q, activation, mean_dev, rstd_dev, dx_dev, dweight_dev, dbias_dev, part, ab, st) }
  return gn_done(what);
}
