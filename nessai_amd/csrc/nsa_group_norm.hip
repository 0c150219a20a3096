// Group norm with an activation, channels last, forward and backward.
//
//   sample n, group g (m = length * channels / groups values): mean, var = mean of (x - mean)^2, r = 1 / sqrt(var + eps)
//   xh = (x - mean) r      z = xh w[c] + b[c]      y = act(z)
//   backward, dz = dy act'(z):   db[c] = sum_{n,l} dz     dw[c] = sum_{n,l} dz xh
//     A = 1/m sum_group w dz     B = 1/m sum_group w dz xh     dx = r (w dz - A - xh B)
//
// Three ways, by the size of a sample (gn_rows, gn_tile_threads):
//   rows of a power of two of channels     one pass, shuffles:    200003 x 128 float32, 32 groups: forward 40 us (205 MB at
//                                          5.1 TB/s), with the backward pass 106 us (512 MB at 4.8 TB/s); as tiles 60 and 197
//   up to 8192 values (backward 4096)      one pass through LDS:  1000 x 64 x 128 float32: forward 20 us
//   longer samples                         statistics, their join, then the values once more: 16 x 4096 x 256 bfloat16
//                                          (34 MB): 11 + 4 + 19 us, the second reading out of the last-level cache
// A large copy on this card runs at 5.07 TB/s.
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

// 1 / (1 + e^-z) by the hardware's 2^x and reciprocal (1 ulp each; the product z log2(e) adds |z| ulp, where e^-z decides)
__device__ __forceinline__ float gn_sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
}

// 2 / (1 + e^-2z) - 1; near zero, where that is a difference of equal numbers, the series z - z^3/3 + 2 z^5/15 - 17 z^7/315
// (the next term is 62 z^9 / 2835: below 2^-27 of z at the border)
__device__ __forceinline__ float gn_tanh(float z) {
  const float s = z * z;
  const float near = z * fmaf(s, fmaf(s, fmaf(s, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
  return fabsf(z) < 0.15f ? near : fmaf(2.0f, gn_sigmoid(2.0f * z), -1.0f);
}

template <int ACT>
__device__ __forceinline__ float gn_act(float z) {
  if constexpr (ACT == NSA_FN_RELU) return z < 0.0f ? 0.0f : z;  // (NaN stays)
  else if constexpr (ACT == NSA_FN_TANH) return gn_tanh(z);
  else if constexpr (ACT == NSA_FN_SILU) return z * gn_sigmoid(z);
  else return z;
}

template <int ACT>
__device__ __forceinline__ float gn_slope(float z) {
  if constexpr (ACT == NSA_FN_RELU) return z > 0.0f ? 1.0f : 0.0f;
  else if constexpr (ACT == NSA_FN_TANH) {  // 1 - tanh^2 = 4 s (1 - s) with s = sigmoid(2 z)
    const float s = gn_sigmoid(2.0f * z);
    return 4.0f * s * (1.0f - s);
  } else if constexpr (ACT == NSA_FN_SILU) {
    const float s = gn_sigmoid(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
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

// Which workgroup of a launch this is.  A launch holds fewer than 2^32 threads in a dimension - 2^24 workgroups of 256, which
// many samples of many groups pass - so more than GN_GRID_X workgroups lie in rows of as many (gn_grid); those behind the
// last one have nothing to do, each as a whole.  (Not by gridDim: reading it costs a load before anything else can begin.)
#define GN_GRID_X (1 << 20)
__device__ __forceinline__ long long gn_block() { return (long long)blockIdx.y * GN_GRID_X + blockIdx.x; }

// i = q d + r, in 32 bits where i fits (a division of 64 bits is a hundred instructions)
__device__ __forceinline__ long long gn_split(long long i, int d, int& r) {
  long long q;
  if ((unsigned long long)i >> 32 == 0) q = (uint32_t)i / (uint32_t)d;
  else q = i / d;
  r = (int)(i - q * d);
  return q;
}

struct GnPlace {  // what this workgroup works on
  long long n, l0, l1;  // n >= samples: nothing
  int slab, chunk, j, r;
  bool active;
};

__device__ __forceinline__ GnPlace gn_place(const GnShape& s) {
  GnPlace p;
  p.n = gn_split(gn_split(gn_block(), s.chunks, p.chunk), s.slabs, p.slab);
  p.l0 = p.chunk * s.chunk;
  p.l1 = p.l0 + s.chunk < s.length ? p.l0 + s.chunk : s.length;
  p.j = threadIdx.x % s.vecs;
  p.r = threadIdx.x / s.vecs;
  p.active = p.r < s.rows;
  return p;
}

// f(i, channel, index of its (sample, group)) for the V channels from c of the slab on: one division, not V
template <int V, typename F>
__device__ __forceinline__ void gn_group_of(const GnShape& s, const GnPlace& p, int c, F f) {
  const int first = p.slab * s.width + c;
  int g = first / s.cpg, in = first - g * s.cpg;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    f(i, first + i, p.n * s.groups + g);
    if (++in == s.cpg) {
      in = 0;
      ++g;
    }
  }
}

// This thread's positions of the chunk, GN_AHEAD at a time: ask(slot, offset) for all of them, then use(slot, offset).  The
// offset is that of the thread's channels c at a position.
#define GN_AHEAD 4
template <typename ASK, typename USE>
__device__ __forceinline__ void gn_positions(const GnShape& s, const GnPlace& p, int c, ASK ask, USE use) {
  const long long row = (long long)s.rows * s.channels;
  long long at = (p.n * s.length + p.l0 + p.r) * s.channels + p.slab * s.width + c;
  long long l = p.l0 + p.r;
  for (; l + (GN_AHEAD - 1) * s.rows < p.l1; l += GN_AHEAD * s.rows, at += GN_AHEAD * row) {
#pragma unroll
    for (int k = 0; k < GN_AHEAD; ++k) ask(k, at + k * row);
#pragma unroll
    for (int k = 0; k < GN_AHEAD; ++k) use(k, at + k * row);
  }
  for (; l < p.l1; l += s.rows, at += row) {
    ask(0, at);
    use(0, at);
  }
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
  if (p.n >= s.samples) return;
  float shift[V], sum[V], sq[V];
#pragma unroll
  for (int i = 0; i < V; ++i) shift[i] = sum[i] = sq[i] = 0.0f;
  int count = 0;
  if (p.active) {
    for (int t = 0; t < s.tiles; ++t) {
      const int c = (t * s.vecs + p.j) * V;
      if (c >= s.width) break;
      NsaPack<T, V> px[GN_AHEAD];
      gn_positions(s, p, c, [&](int k, long long at) { px[k] = *reinterpret_cast<const NsaPack<T, V>*>(x + at); },
                   [&](int k, long long) {
                     if (count == 0) {
#pragma unroll
                       for (int i = 0; i < V; ++i) shift[i] = (float)px[k].v[i];
                     }
#pragma unroll
                     for (int i = 0; i < V; ++i) {
                       const float d = (float)px[k].v[i] - shift[i];
                       sum[i] += d;
                       sq[i] = fmaf(d, d, sq[i]);
                     }
                     ++count;
                   });
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
  // A team of lanes per group joins the parts - rows x (channels of the group in a tile) - in a fixed order; as many lanes
  // as give every group of the slab a team.
  const int span = s.vecs * V;                              // channels in the parts of a row
  const int in_group = s.cpg < span ? s.cpg : span;         // of them, in one group
  const int parts = in_group * s.rows;
  int team = 1;
  while (team < 64 && team * 2 * s.gps <= GN_THREADS && team * 2 <= parts) team *= 2;
  const int lane = threadIdx.x & (team - 1);
  const float total = (float)(p.l1 - p.l0) * (float)s.cpg;
  for (int g = threadIdx.x / team; g < s.gps; g += GN_THREADS / team) {
    const int first = g * s.cpg;
    float a = 0.0f;
    for (int e = lane; e < parts; e += team) {
      const int r = e / in_group, c = first + e - r * in_group;
      a += (float)counts[r * s.vecs + c / V] * means[r * span + c];
    }
    for (int o = team >> 1; o > 0; o >>= 1) a += __shfl_xor(a, o);
    const float mean = a / total;
    float m2 = 0.0f;
    for (int e = lane; e < parts; e += team) {
      const int r = e / in_group, c = first + e - r * in_group, count_here = counts[r * s.vecs + c / V];
      const float d = means[r * span + c] - mean;
      m2 += devs[r * span + c] + (count_here > 0 ? (float)count_here * d * d : 0.0f);
    }
    for (int o = team >> 1; o > 0; o >>= 1) m2 += __shfl_xor(m2, o);
    if (lane == 0) part[(p.n * s.chunks + p.chunk) * s.groups + p.slab * s.gps + g] = make_float2(mean, m2);
  }
}

// the chunks of a (sample, group) joined in 64 bits: a wave each, lane by lane, then lane with lane
__global__ void __launch_bounds__(GN_THREADS) gn_stats_join(GnShape s, const float2* __restrict__ part, float eps,
                                                            float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  const long long i = gn_block() * (GN_THREADS / 64) + (threadIdx.x >> 6);
  if (i >= s.samples * s.groups) return;
  int g;
  const long long n = gn_split(i, s.groups, g);
  const int lane = threadIdx.x & 63;
  double mean = 0.0, m2 = 0.0, count = 0.0;
  auto join = [&](double mean_b, double m2_b, double count_b) {
    const double all = count + count_b, d = mean_b - mean;
    if (all > 0.0) {
      mean += d * (count_b / all);
      m2 += m2_b + d * d * (count * count_b / all);
      count = all;
    }
  };
  for (int k = lane; k < s.chunks; k += 64) {
    const float2 q = part[(n * s.chunks + k) * s.groups + g];
    const long long l0 = k * s.chunk, rows = (l0 + s.chunk < s.length ? l0 + s.chunk : s.length) - l0;
    join((double)q.x, (double)q.y, (double)rows * s.cpg);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double mean_b = __shfl_down(mean, o), m2_b = __shfl_down(m2, o), count_b = __shfl_down(count, o);
    if (lane + o < 64) join(mean_b, m2_b, count_b);  // (lane 0 ends with all of them, in order)
  }
  if (lane == 0) {
    mean_out[i] = (float)mean;
    rstd_out[i] = (float)(1.0 / sqrt(m2 / count + (double)eps));
  }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_apply(GnShape s, const T* __restrict__ x, GnParams q,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd,
                                                       T* __restrict__ y) {
  const GnPlace p = gn_place(s);
  if (!p.active || p.n >= s.samples) return;
  for (int t = 0; t < s.tiles; ++t) {
    const int c = (t * s.vecs + p.j) * V;
    if (c >= s.width) break;
    float mu[V], rs[V], w[V], b[V];
    gn_group_of<V>(s, p, c, [&](int i, int ch, long long k) {
      mu[i] = mean[k];
      rs[i] = rstd[k];
      w[i] = gn_param<T>(q.w, q.f32, ch, 1.0f);
      b[i] = gn_param<T>(q.b, q.f32, ch, 0.0f);
    });
    NsaPack<T, V> px[GN_AHEAD];
    gn_positions(s, p, c, [&](int k, long long at) { px[k] = *reinterpret_cast<const NsaPack<T, V>*>(x + at); },
                 [&](int k, long long at) {
                   float v[V];
#pragma unroll
                   for (int i = 0; i < V; ++i) v[i] = gn_act<ACT>(fmaf(((float)px[k].v[i] - mu[i]) * rs[i], w[i], b[i]));
                   nsa_store<T, V>(y + at, v);
                 });
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
  if (p.n >= s.samples) return;
  for (int t = 0; t < s.tiles; ++t) {
    const int c = (t * s.vecs + p.j) * V;
    float s1[V], s2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0f;
    if (p.active && c < s.width) {
      float mu[V], rs[V], w[V], b[V];
      gn_group_of<V>(s, p, c, [&](int i, int ch, long long k) {
        mu[i] = mean[k];
        rs[i] = rstd[k];
        w[i] = gn_param<T>(q.w, q.f32, ch, 1.0f);
        b[i] = gn_param<T>(q.b, q.f32, ch, 0.0f);
      });
      NsaPack<T, V> px[GN_AHEAD], pd[GN_AHEAD];
      gn_positions(s, p, c,
                   [&](int k, long long at) {
                     px[k] = *reinterpret_cast<const NsaPack<T, V>*>(x + at);
                     pd[k] = *reinterpret_cast<const NsaPack<T, V>*>(dy + at);
                   },
                   [&](int k, long long) {
#pragma unroll
                     for (int i = 0; i < V; ++i) {
                       const float xh = ((float)px[k].v[i] - mu[i]) * rs[i];
                       const float dz = (float)pd[k].v[i] * gn_slope<ACT>(fmaf(xh, w[i], b[i]));
                       s1[i] += dz;
                       s2[i] = fmaf(dz, xh, s2[i]);
                     }
                   });
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

// The chunks' sums of 64 channels of a sample joined into chunk 0's place; sixteen waves share the chunks out.  For groups wider
// than that, which gn_sums_join would leave to one workgroup each: 27287 x 935 float32 in one group, 0.3 ms.
#define GN_JOIN_THREADS 1024
__global__ void __launch_bounds__(GN_JOIN_THREADS) gn_sums_columns(GnShape s, float2* __restrict__ part) {
  __shared__ float2 red[GN_JOIN_THREADS];
  const int slabs = (s.channels + 63) / 64, share = threadIdx.x >> 6;
  int slab;
  const long long n = gn_split(gn_block(), slabs, slab);
  if (n >= s.samples) return;
  const int c = slab * 64 + (threadIdx.x & 63);
  float2* p = part + n * s.chunks * s.channels + c;
  float2 a = make_float2(0.0f, 0.0f);
  if (c < s.channels) {
#pragma unroll 4
    for (int k = share; k < s.chunks; k += GN_JOIN_THREADS / 64) {
      const float2 o = p[(long long)k * s.channels];
      a.x += o.x;
      a.y += o.y;
    }
  }
  red[threadIdx.x] = a;
  __syncthreads();
  if (share != 0 || c >= s.channels) return;
  for (int k = 1; k < GN_JOIN_THREADS / 64; ++k) {
    a.x += red[k * 64 + threadIdx.x].x;
    a.y += red[k * 64 + threadIdx.x].y;
  }
  p[0] = a;
}

// A workgroup per (sample, group): the first `chunks` chunks' sums joined into chunk 0's place, and the group's A and B.  `across` threads
// (a power of two) lie along the channels, the others share the chunks out.
template <typename T>
__global__ void __launch_bounds__(GN_THREADS) gn_sums_join(GnShape s, int chunks, int across, float2* __restrict__ part,
                                                           GnParams q,
                                                           float2* __restrict__ ab) {
  __shared__ float2 red[GN_THREADS];
  int g;
  const long long pair = gn_block(), n = gn_split(pair, s.groups, g);
  if (n >= s.samples) return;
  const int lane = threadIdx.x % across, share = threadIdx.x / across;
  const int shares = GN_THREADS / across;
  float2 t = make_float2(0.0f, 0.0f);  // this thread's part of A and B
  for (int base = 0; base < s.cpg; base += across) {
    const int c = g * s.cpg + base + lane;
    float2 a = make_float2(0.0f, 0.0f);
    if (base + lane < s.cpg) {
      const float2* p = part + n * s.chunks * s.channels + c;
#pragma unroll 4
      for (int k = share; k < chunks; k += shares) {
        const float2 o = p[(long long)k * s.channels];
        a.x += o.x;
        a.y += o.y;
      }
    }
    red[threadIdx.x] = a;
    __syncthreads();
    if (share == 0 && base + lane < s.cpg) {
      for (int k = 1; k < shares; ++k) {
        a.x += red[k * across + lane].x;
        a.y += red[k * across + lane].y;
      }
      part[n * s.chunks * s.channels + c] = a;
      const float w = gn_param<T>(q.w, q.f32, c, 1.0f);
      t.x = fmaf(w, a.x, t.x);
      t.y = fmaf(w, a.y, t.y);
    }
    __syncthreads();
  }
  red[threadIdx.x] = t;
  __syncthreads();
  for (int half = across >> 1; half > 0; half >>= 1) {
    if (threadIdx.x < half) {
      red[threadIdx.x].x += red[threadIdx.x + half].x;
      red[threadIdx.x].y += red[threadIdx.x + half].y;
    }
    __syncthreads();
  }
  const float m = (float)s.length * (float)s.cpg;
  if (threadIdx.x == 0) ab[pair] = make_float2(red[0].x / m, red[0].y / m);
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_dx(GnShape s, const T* __restrict__ x, const T* __restrict__ dy, GnParams q,
                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                    const float2* __restrict__ ab, T* __restrict__ dx) {
  const GnPlace p = gn_place(s);
  if (!p.active || p.n >= s.samples) return;
  for (int t = 0; t < s.tiles; ++t) {
    const int c = (t * s.vecs + p.j) * V;
    if (c >= s.width) break;
    float mu[V], rs[V], w[V], b[V], ga[V], gb[V];
    gn_group_of<V>(s, p, c, [&](int i, int ch, long long k) {
      mu[i] = mean[k];
      rs[i] = rstd[k];
      ga[i] = ab[k].x;
      gb[i] = ab[k].y;
      w[i] = gn_param<T>(q.w, q.f32, ch, 1.0f);
      b[i] = gn_param<T>(q.b, q.f32, ch, 0.0f);
    });
    NsaPack<T, V> px[GN_AHEAD], pd[GN_AHEAD];
    gn_positions(s, p, c,
                 [&](int k, long long at) {
                   px[k] = *reinterpret_cast<const NsaPack<T, V>*>(x + at);
                   pd[k] = *reinterpret_cast<const NsaPack<T, V>*>(dy + at);
                 },
                 [&](int k, long long at) {
                   float v[V];
#pragma unroll
                   for (int i = 0; i < V; ++i) {
                     const float xh = ((float)px[k].v[i] - mu[i]) * rs[i];
                     const float dz = (float)pd[k].v[i] * gn_slope<ACT>(fmaf(xh, w[i], b[i]));
                     v[i] = rs[i] * (w[i] * dz - ga[i] - xh * gb[i]);
                   }
                   nsa_store<T, V>(dx + at, v);
                 });
  }
}

// The parameters' gradients: `count` records of [channels] sums, `stride` apart, added in 64 bits (there may be as many
// records as samples) and a fixed order.  A workgroup per GN_PARAM_CH channels; its threads share the records out.
#define GN_PARAM_THREADS 1024
#define GN_PARAM_CH 16
template <typename T>
__global__ void __launch_bounds__(GN_PARAM_THREADS) gn_param_grads(int channels, long long count, long long stride,
                                                                   const float2* __restrict__ part, int f32,
                                                                   void* __restrict__ dw, void* __restrict__ db) {
  constexpr int LANES = GN_PARAM_THREADS / GN_PARAM_CH;
  __shared__ double2 red[GN_PARAM_THREADS];
  const long long c = gn_block() * GN_PARAM_CH + threadIdx.x % GN_PARAM_CH;
  const int lane = threadIdx.x / GN_PARAM_CH;
  double2 t = make_double2(0.0, 0.0);
  if (c < channels) {
    const float2* p = part + c;
#pragma unroll 4
    for (long long k = lane; k < count; k += LANES) {
      const float2 o = p[k * stride];
      t.x += (double)o.x;
      t.y += (double)o.y;
    }
  }
  red[threadIdx.x] = t;
  __syncthreads();
#pragma unroll
  for (int half = LANES / 2; half > 0; half >>= 1) {
    if (lane < half) {
      red[threadIdx.x].x += red[threadIdx.x + half * GN_PARAM_CH].x;
      red[threadIdx.x].y += red[threadIdx.x + half * GN_PARAM_CH].y;
    }
    __syncthreads();
  }
  if (lane != 0 || c >= channels) return;
  t = red[threadIdx.x];
  if (f32) {
    if (dw != nullptr) ((float*)dw)[c] = (float)t.y;
    if (db != nullptr) ((float*)db)[c] = (float)t.x;
  } else {
    if (dw != nullptr) ((T*)dw)[c] = (T)(float)t.y;
    if (db != nullptr) ((T*)db)[c] = (T)(float)t.x;
  }
}

// ---------------------------------------------------------------------------
// small samples: whole samples in one workgroup, each value read once
// ---------------------------------------------------------------------------

// A tile of `per` whole samples, at most THREADS * GN_EACH values, contiguous in memory.  Its values go through LDS in
// float32: a team of `team` lanes takes a (sample, group), whose channels may lie anywhere in a thread's accesses.
#define GN_EACH 16
struct GnTile {
  long long samples;
  int length, channels, groups, cpg;
  int values;                 // of a sample: length * channels
  int per;                    // samples of a tile
  int team, step_l, step_c;   // lanes per (sample, group); `team` values on = step_l positions and step_c channels on
  uint32_t by_values, by_channels, by_cpg;  // 2^32 / d + 1 (0: d = 1): quotients of numbers up to 2^14 by d up to 2^14
  int fixed;                  // a thread's accesses all lie in the same channels
};

__device__ __forceinline__ int gn_div(int n, uint32_t by) { return by != 0 ? (int)__umulhi((uint32_t)n, by) : n; }

// f(value index in the tile) over the values of group g of sample s, lane by lane of its team
template <typename F>
__device__ __forceinline__ void gn_walk(const GnTile& q, int s, int g, int lane, F f) {
  int l = gn_div(lane, q.by_cpg), c = lane - l * q.cpg;
  int at = s * q.values + l * q.channels + g * q.cpg + c;
  const int step = q.step_l * q.channels + q.step_c, wrap = q.channels - q.cpg;
  while (l < q.length) {
    f(at, g * q.cpg + c);
    l += q.step_l;
    c += q.step_c;
    at += step;
    if (c >= q.cpg) {
      c -= q.cpg;
      ++l;
      at += wrap;
    }
  }
}

__device__ __forceinline__ float gn_team_sum(float a, int team) {
  for (int o = team >> 1; o > 0; o >>= 1) a += __shfl_xor(a, o);
  return a;
}

// group, weight and bias of the V channels at value e of a tile; wb: {weight, bias} of every channel, in LDS (from memory they
// cost a load per value where a thread's channels change from access to access)
template <int V>
__device__ __forceinline__ void gn_channels(const GnTile& q, const float2* wb, int e, int (&g)[V], float (&w)[V],
                                            float (&b)[V]) {
  const int c = e - gn_div(e, q.by_channels) * q.channels;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 t = wb[c + i];
    g[i] = gn_div(c + i, q.by_cpg);
    w[i] = t.x;
    b[i] = t.y;
  }
}

template <typename T, int V, int ACT, int THREADS>
__global__ void __launch_bounds__(THREADS) gn_tile_forward(GnTile q, const T* __restrict__ x, GnParams par, float eps,
                                                           float* __restrict__ mean, float* __restrict__ rstd,
                                                           T* __restrict__ y) {
  constexpr int STEPS = GN_EACH / V;
  extern __shared__ float lds[];
  float* buf = lds;                                    // [THREADS * GN_EACH]
  float2* stat = (float2*)(lds + THREADS * GN_EACH);   // [per * groups]
  float2* wb = stat + q.per * q.groups;                // [channels]
  const long long first = gn_block() * q.per;
  if (first >= q.samples) return;
  for (int c = threadIdx.x; c < q.channels; c += THREADS)
    wb[c] = make_float2(gn_param<T>(par.w, par.f32, c, 1.0f), gn_param<T>(par.b, par.f32, c, 0.0f));
  const int here = q.samples - first < q.per ? (int)(q.samples - first) : q.per;
  const int values = here * q.values;
  const long long base = first * q.values;
  float v[STEPS][V];
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int e = (k * THREADS + threadIdx.x) * V;
    if (e < values) nsa_load<T, V>(x + base + e, v[k]);
  }
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int e = (k * THREADS + threadIdx.x) * V;
    if (e < values) nsa_store<float, V>(buf + e, v[k]);
  }
  __syncthreads();
  const int pairs = here * q.groups, lane = threadIdx.x & (q.team - 1);
  const float m = (float)q.length * (float)q.cpg;
  for (int p = threadIdx.x / q.team; p < pairs; p += THREADS / q.team) {
    const int s = p / q.groups, g = p - s * q.groups;
    const float shift = buf[s * q.values + g * q.cpg];
    float a = 0.0f;
    gn_walk(q, s, g, lane, [&](int at, int) { a += buf[at] - shift; });
    const float mu = shift + gn_team_sum(a, q.team) / m;
    float b = 0.0f;
    gn_walk(q, s, g, lane, [&](int at, int) {
      const float d = buf[at] - mu;
      b = fmaf(d, d, b);
    });
    const float rs = 1.0f / sqrtf(gn_team_sum(b, q.team) / m + eps);
    if (lane == 0) {
      stat[p] = make_float2(mu, rs);
      mean[first * q.groups + p] = mu;
      rstd[first * q.groups + p] = rs;
    }
  }
  __syncthreads();
  float w[V], b[V];
  int g[V];
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int e = (k * THREADS + threadIdx.x) * V;
    if (e >= values) continue;
    const int s = gn_div(e, q.by_values);
    if (k == 0 || !q.fixed) gn_channels<V>(q, wb, e, g, w, b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 t = stat[s * q.groups + g[i]];
      v[k][i] = gn_act<ACT>(fmaf((v[k][i] - t.x) * t.y, w[i], b[i]));
    }
    nsa_store<T, V>(y + base + e, v[k]);
  }
}

// The same tiles backward: dz and dz xh through LDS, from which the teams take A and B and the threads the columns' sums
// for the parameters.  A workgroup walks over tiles, keeps the columns' sums in LDS and writes one record of them at the end:
// part[block][channels].
template <typename T, int V, int ACT, int THREADS>
__global__ void __launch_bounds__(THREADS) gn_tile_backward(GnTile q, const T* __restrict__ x, const T* __restrict__ dy,
                                                            GnParams par, const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, T* __restrict__ dx,
                                                            float2* __restrict__ part) {
  constexpr int STEPS = GN_EACH / V;
  extern __shared__ float lds[];
  float* bz = lds;                                            // [THREADS * GN_EACH]  dz
  float* bzx = lds + THREADS * GN_EACH;                       //                      dz xh
  float2* ab = (float2*)(lds + 2 * THREADS * GN_EACH);        // [per * groups]
  float2* stat = ab + q.per * q.groups;                       // [per * groups]
  float2* wb = stat + q.per * q.groups;                       // [channels] weight, bias
  float2* cols = wb + q.channels;                             // [subs][channels]
  const int subs = q.channels < THREADS ? THREADS / q.channels : 1;
  for (int c = threadIdx.x; c < q.channels; c += THREADS)
    wb[c] = make_float2(gn_param<T>(par.w, par.f32, c, 1.0f), gn_param<T>(par.b, par.f32, c, 0.0f));
  for (int i = threadIdx.x; i < subs * q.channels; i += THREADS) cols[i] = make_float2(0.0f, 0.0f);
  const float m = (float)q.length * (float)q.cpg;
  const long long tiles = (q.samples + q.per - 1) / q.per;
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long first = tile * q.per, base = first * q.values;
    const int here = q.samples - first < q.per ? (int)(q.samples - first) : q.per;
    const int values = here * q.values;
    float v[STEPS][V], z[STEPS][V], w[V], b[V];
    int g[V];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const int e = (k * THREADS + threadIdx.x) * V;
      if (e < values) {
        nsa_load<T, V>(x + base + e, v[k]);
        nsa_load<T, V>(dy + base + e, z[k]);
      }
    }
    for (int p = threadIdx.x; p < here * q.groups; p += THREADS)
      stat[p] = make_float2(mean[first * q.groups + p], rstd[first * q.groups + p]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const int e = (k * THREADS + threadIdx.x) * V;
      if (e >= values) continue;
      const int p = gn_div(e, q.by_values) * q.groups;
      if (k == 0 || !q.fixed) gn_channels<V>(q, wb, e, g, w, b);
      float zx[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 t = stat[p + g[i]];
        v[k][i] = (v[k][i] - t.x) * t.y;
        z[k][i] *= gn_slope<ACT>(fmaf(v[k][i], w[i], b[i]));
        zx[i] = z[k][i] * v[k][i];
      }
      nsa_store<float, V>(bz + e, z[k]);
      nsa_store<float, V>(bzx + e, zx);
    }
    __syncthreads();
    const int pairs = here * q.groups, lane = threadIdx.x & (q.team - 1);
    if (dx != nullptr)
      for (int p = threadIdx.x / q.team; p < pairs; p += THREADS / q.team) {
        const int s = p / q.groups, g = p - s * q.groups;
        float a = 0.0f, b = 0.0f;
        gn_walk(q, s, g, lane, [&](int at, int c) {
          a = fmaf(wb[c].x, bz[at], a);
          b = fmaf(wb[c].x, bzx[at], b);
        });
        a = gn_team_sum(a, q.team);
        b = gn_team_sum(b, q.team);
        if (lane == 0) ab[p] = make_float2(a / m, b / m);
      }
    if (part != nullptr) {
      const int rows = here * q.length;
      for (int i = threadIdx.x; i < subs * q.channels; i += THREADS) {
        const int sub = i / q.channels, c = i - sub * q.channels;
        float2 t = make_float2(0.0f, 0.0f);
        for (int r = sub; r < rows; r += subs) {
          t.x += bz[r * q.channels + c];
          t.y += bzx[r * q.channels + c];
        }
        cols[i].x += t.x;
        cols[i].y += t.y;
      }
    }
    __syncthreads();
    if (dx != nullptr) {
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {
        const int e = (k * THREADS + threadIdx.x) * V;
        if (e >= values) continue;
        const int s = gn_div(e, q.by_values);
        if (!q.fixed) gn_channels<V>(q, wb, e, g, w, b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 t = ab[s * q.groups + g[i]];
          z[k][i] = stat[s * q.groups + g[i]].y * (w[i] * z[k][i] - t.x - v[k][i] * t.y);
        }
        nsa_store<T, V>(dx + base + e, z[k]);
      }
    }
    __syncthreads();  // (the next tile's statistics take the place of these)
  }
  if (part != nullptr)
    for (int c = threadIdx.x; c < q.channels; c += THREADS) {
      float2 t = cols[c];
      for (int s = 1; s < subs; ++s) {
        t.x += cols[s * q.channels + c].x;
        t.y += cols[s * q.channels + c].y;
      }
      part[(long long)blockIdx.x * q.channels + c] = t;
    }
}

// ---------------------------------------------------------------------------
// rows of a power of two of channels: no LDS, no division
// ---------------------------------------------------------------------------

// length 1, channels and channels per group powers of two: a group is a power of two of neighbouring lanes, which add by
// shuffles; a thread's accesses all lie in the same V channels, whose parameters and column sums it keeps in registers.
struct GnRows {
  long long vectors;  // samples * channels / V
  int vecs;           // accesses of a row (a power of two, at most GN_THREADS)
  int span;           // lanes of a group (a power of two, at most 64)
  int channels, groups;
};
#define GN_ROW_STEPS 4  // accesses of a thread in flight

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_rows_forward(GnRows q, const T* __restrict__ x, GnParams par, float eps,
                                                              float* __restrict__ mean, float* __restrict__ rstd,
                                                              T* __restrict__ y) {
  const int c = (threadIdx.x & (q.vecs - 1)) * V;
  float w[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = gn_param<T>(par.w, par.f32, c + i, 1.0f);
    b[i] = gn_param<T>(par.b, par.f32, c + i, 0.0f);
  }
  const float inv = 1.0f / (float)(q.span * V);
  const long long base = gn_block() * GN_THREADS * GN_ROW_STEPS + threadIdx.x;
  float v[GN_ROW_STEPS][V];
#pragma unroll
  for (int k = 0; k < GN_ROW_STEPS; ++k)
    if (base + k * GN_THREADS < q.vectors) nsa_load<T, V>(x + (base + k * GN_THREADS) * V, v[k]);
#pragma unroll
  for (int k = 0; k < GN_ROW_STEPS; ++k) {
    const long long e = base + k * GN_THREADS;
    if (e >= q.vectors) break;  // (whole rows: the lanes of a group leave together)
    const float shift = __shfl(v[k][0], (threadIdx.x & 63) & ~(q.span - 1));
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) s += v[k][i] - shift;
    for (int o = q.span >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o);
    const float mu = fmaf(s, inv, shift);
    float d2 = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) d2 = fmaf(v[k][i] - mu, v[k][i] - mu, d2);
    for (int o = q.span >> 1; o > 0; o >>= 1) d2 += __shfl_xor(d2, o);
    const float rs = 1.0f / sqrtf(fmaf(d2, inv, eps));
    if ((threadIdx.x & (q.span - 1)) == 0) {
      mean[e / q.span] = mu;
      rstd[e / q.span] = rs;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[k][i] = gn_act<ACT>(fmaf((v[k][i] - mu) * rs, w[i], b[i]));
    nsa_store<T, V>(y + e * V, v[k]);
  }
}

// part[block][channels]: the column sums of this workgroup's rows
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_rows_backward(GnRows q, const T* __restrict__ x, const T* __restrict__ dy,
                                                               GnParams par, const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, T* __restrict__ dx,
                                                               float2* __restrict__ part) {
  const int c = (threadIdx.x & (q.vecs - 1)) * V;
  float w[V], b[V], s1[V], s2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = gn_param<T>(par.w, par.f32, c + i, 1.0f);
    b[i] = gn_param<T>(par.b, par.f32, c + i, 0.0f);
    s1[i] = s2[i] = 0.0f;
  }
  const float inv = 1.0f / (float)(q.span * V);
  const long long step = (long long)gridDim.x * GN_THREADS * GN_ROW_STEPS;
  for (long long base = (long long)blockIdx.x * GN_THREADS * GN_ROW_STEPS + threadIdx.x; base < q.vectors; base += step) {
    NsaPack<T, V> px[GN_ROW_STEPS], pd[GN_ROW_STEPS];
    float mu[GN_ROW_STEPS], rs[GN_ROW_STEPS];
#pragma unroll
    for (int k = 0; k < GN_ROW_STEPS; ++k) {
      const long long e = base + k * GN_THREADS;
      if (e < q.vectors) {
        px[k] = *reinterpret_cast<const NsaPack<T, V>*>(x + e * V);
        pd[k] = *reinterpret_cast<const NsaPack<T, V>*>(dy + e * V);
        mu[k] = mean[e / q.span];
        rs[k] = rstd[e / q.span];
      }
    }
#pragma unroll
    for (int k = 0; k < GN_ROW_STEPS; ++k) {
      const long long e = base + k * GN_THREADS;
      if (e >= q.vectors) break;
      float xh[V], dz[V], a = 0.0f, ax = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xh[i] = ((float)px[k].v[i] - mu[k]) * rs[k];
        dz[i] = (float)pd[k].v[i] * gn_slope<ACT>(fmaf(xh[i], w[i], b[i]));
        s1[i] += dz[i];
        s2[i] = fmaf(dz[i], xh[i], s2[i]);
        dz[i] *= w[i];
        a += dz[i];
        ax = fmaf(dz[i], xh[i], ax);
      }
      for (int o = q.span >> 1; o > 0; o >>= 1) {
        a += __shfl_xor(a, o);
        ax += __shfl_xor(ax, o);
      }
      a *= inv;
      ax *= inv;
#pragma unroll
      for (int i = 0; i < V; ++i) dz[i] = rs[k] * (dz[i] - a - xh[i] * ax);
      if (dx != nullptr) nsa_store<T, V>(dx + e * V, dz);
    }
  }
  if (part == nullptr) return;
  __shared__ float2 red[GN_THREADS * V];
#pragma unroll
  for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = make_float2(s1[i], s2[i]);
  __syncthreads();
  for (int ch = threadIdx.x; ch < q.channels; ch += GN_THREADS) {
    float2 t = red[ch];
    for (int r = q.channels; r < GN_THREADS * V; r += q.channels) {
      t.x += red[r + ch].x;
      t.y += red[r + ch].y;
    }
    part[(long long)blockIdx.x * q.channels + ch] = t;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

// workgroups wanted of a launch: a few for each of the 256 compute units, so that no unit waits for a long one
const long long GN_GROUPS_WANTED = 1024;
// positions of a chunk at least, per row of threads: below it a workgroup's start costs more than its work
const long long GN_CHUNK_ROWS = 8;

// ... and at most: the float32 sums of a thread stay this short, whatever the lengths
const long long GN_CHUNK_MOST = 128;

GnShape gn_shape(long long samples, long long length, int channels, int groups, int bytes, uintptr_t addresses, int& v) {
  GnShape s;
  s.samples = samples;
  s.length = length;
  s.channels = channels;
  s.groups = groups;
  s.cpg = channels / groups;
  v = 16 / bytes;
  while (v > 1 && (channels % v != 0 || addresses % (uintptr_t)(v * bytes) != 0)) v >>= 1;
  if (length == 1 && (channels & (channels - 1)) == 0 && s.cpg >= 2)  // (gn_rows: no access over two groups)
    while (v > s.cpg) v >>= 1;
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
  chunks = std::max(chunks, (length * s.tiles + s.rows * GN_CHUNK_MOST - 1) / (s.rows * GN_CHUNK_MOST));
  s.chunk = (length + chunks - 1) / chunks;
  s.chunks = (int)((length + s.chunk - 1) / s.chunk);
  return s;
}

// `blocks` workgroups as gn_block counts them
dim3 gn_grid(long long blocks) {
  if (blocks <= GN_GRID_X) return dim3((unsigned)blocks);
  return dim3(GN_GRID_X, (unsigned)((blocks + GN_GRID_X - 1) / GN_GRID_X));
}
const long long GN_BLOCKS_MOST = 65535LL * GN_GRID_X;  // (a grid's second dimension has 16 bits)

const size_t GN_LDS = 152 * 1024;  // of a workgroup's 160 KB
const int GN_TILE_BLOCKS = 1024;  // workgroups of the one-pass backward kernels: one record of column sums each

// the largest of the launches for these samples: slabs and chunks, groups, or columns of 64 channels
long long gn_blocks(const GnShape& s) {
  return s.samples * std::max((long long)s.slabs * s.chunks, std::max((long long)s.groups, (s.channels + 63LL) / 64));
}

bool gn_tile(long long samples, long long length, int channels, int groups, int v, int most, GnTile& q) {
  if (length * channels > most) return false;
  q.samples = samples;
  q.length = (int)length;
  q.channels = channels;
  q.groups = groups;
  q.cpg = channels / groups;
  q.values = q.length * channels;
  q.per = most / q.values;
  // (accesses of v values must not run over a tile's end, and samples begin at multiples of v: channels is one)
  const int threads = most / GN_EACH, group = q.length * q.cpg;
  q.team = 1;
  while (q.team < 64 && q.team * 2 <= group && q.per * groups * q.team < threads) q.team *= 2;
  q.step_l = q.team / q.cpg;
  q.step_c = q.team % q.cpg;
  q.fixed = threads * v % channels == 0;
  auto by = [](int d) { return d == 1 ? 0u : (uint32_t)((1ULL << 32) / d + 1); };
  q.by_values = by(q.values);
  q.by_channels = by(channels);
  q.by_cpg = by(q.cpg);
  return true;
}

bool gn_rows(const GnShape& s, int v, GnRows& q) {
  if (s.length != 1 || (s.channels & (s.channels - 1)) != 0 || s.cpg < v) return false;  // (groups divides a power of two)
  q.vecs = s.channels / v;
  q.span = s.cpg / v;
  if (q.vecs > GN_THREADS || q.span > 64) return false;
  q.vectors = s.samples * q.vecs;
  q.channels = s.channels;
  q.groups = s.groups;
  return true;
}

size_t gn_tile_lds(const GnTile& q, int threads, bool backward) {
  const size_t stat = (size_t)q.per * q.groups * sizeof(float2), wb = (size_t)q.channels * sizeof(float2);
  if (!backward) return (size_t)threads * GN_EACH * 4 + stat + wb;
  return (size_t)threads * GN_EACH * 8 + 2 * stat + wb + (size_t)std::max(threads, q.channels) * sizeof(float2);
}

// Whether the one-pass tiles take these samples, with 256 threads (4096 values) or, forward, 512 (8192); 0: they do not.
// 1000 samples of 8192 float32 values: 20 us in a tile, 30 in the three passes below; of 16384 bfloat16 values the passes are
// faster (2000 samples: 58 us against 86 in tiles of that size, of which two fit a compute unit).  Backward, where a tile
// needs twice the LDS, larger ones do not pay.
int gn_tile_threads(long long samples, long long length, int channels, int groups, int v, bool backward, GnTile& q) {
  for (int threads = 256; threads <= (backward ? 256 : 512); threads *= 2)
    if (gn_tile(samples, length, channels, groups, v, threads * GN_EACH, q) && gn_tile_lds(q, threads, backward) <= GN_LDS)
      return threads;
  return 0;
}

// An upper bound that does not ask for the addresses: where the one-pass kernels take the samples (whatever the access width),
// the records of the backward pass; otherwise the chunks' sums at the widest access that any address allows.
size_t gn_workspace(long long samples, long long length, int channels, int groups, int bytes, bool backward) {
  GnTile q;
  if (gn_tile_threads(samples, length, channels, groups, 1, backward, q) != 0)
    return 256 + (backward ? (size_t)std::min(samples, (long long)GN_TILE_BLOCKS) * channels * sizeof(float2) : 0);
  size_t most = 0;
  for (int align = bytes; align <= 16; align *= 2) {
    int v;
    const GnShape s = gn_shape(samples, length, channels, groups, bytes, (uintptr_t)align, v);
    most = std::max(most, (size_t)s.samples * s.chunks * (backward ? s.channels : s.groups) * sizeof(float2));
  }
  return most + (backward ? (size_t)samples * groups * sizeof(float2) : 0) + 256;
}

int gn_check(const char* what, long long samples, long long length, int channels, int groups, int dtype, int weight_dtype,
             int activation) {
  if (samples < 0 || length < 0 || channels < 1 || groups < 1 || channels % groups != 0)
    return nsa_fail(NSA_E_ARG, "%s: bad shape (channels must be a multiple of groups)", what);
  // (channels are counted in 32 bits, in steps of a workgroup that run past the last one)
  if (channels > (1 << 30)) return nsa_fail(NSA_E_ARG, "%s: at most 2^30 channels", what);
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

// a launch with more dynamic LDS than the 64 KB that need no asking
#define GN_TILE_LAUNCH(KERNEL, lds, ...)                                                                                  \
  {                                                                                                                       \
    if ((lds) > 64 * 1024)                                                                                                \
      (void)hipFuncSetAttribute((const void*)(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, (int)(lds));           \
    hipLaunchKernelGGL((KERNEL), __VA_ARGS__);                                                                            \
  }
#define GN_TILE_ACTS(act, KERNEL, T, V, THREADS, lds, ...)                                                                \
  switch (act) {                                                                                                          \
    case NSA_FN_RELU: GN_TILE_LAUNCH((KERNEL<T, V, NSA_FN_RELU, THREADS>), lds, __VA_ARGS__) break;                       \
    case NSA_FN_TANH: GN_TILE_LAUNCH((KERNEL<T, V, NSA_FN_TANH, THREADS>), lds, __VA_ARGS__) break;                       \
    case NSA_FN_SILU: GN_TILE_LAUNCH((KERNEL<T, V, NSA_FN_SILU, THREADS>), lds, __VA_ARGS__) break;                       \
    default: GN_TILE_LAUNCH((KERNEL<T, V, NSA_FN_NONE, THREADS>), lds, __VA_ARGS__) break;                                \
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
  GnRows rows;
  if (gn_rows(s, V, rows)) {
    const long long per = GN_THREADS * GN_ROW_STEPS;
    GN_ACTS(act, gn_rows_forward, T, V, gn_grid((rows.vectors + per - 1) / per), dim3(GN_THREADS), 0, st, rows,
            (const T*)x, q, eps, mean, rstd, (T*)y)
    return;
  }
  GnTile tile;
  if (const int threads = gn_tile_threads(s.samples, s.length, s.channels, s.groups, V, false, tile)) {
    const size_t lds = gn_tile_lds(tile, threads, false);
    const dim3 tiles = gn_grid((s.samples + tile.per - 1) / tile.per);
    if (threads == 256) {
      GN_TILE_ACTS(act, gn_tile_forward, T, V, 256, lds, tiles, dim3(256), lds, st, tile, (const T*)x, q, eps, mean, rstd, (T*)y)
    } else {
      GN_TILE_ACTS(act, gn_tile_forward, T, V, 512, lds, tiles, dim3(512), lds, st, tile, (const T*)x, q, eps, mean, rstd, (T*)y)
    }
    return;
  }
  const dim3 grid = gn_grid(s.samples * s.slabs * s.chunks), block(GN_THREADS);
  hipLaunchKernelGGL((gn_stats<T, V>), grid, block, 0, st, s, (const T*)x, part);
  const long long pairs = s.samples * s.groups;
  hipLaunchKernelGGL(gn_stats_join, gn_grid((pairs + GN_THREADS / 64 - 1) / (GN_THREADS / 64)), block, 0, st, s, part, eps, mean,
                     rstd);
  GN_ACTS(act, gn_apply, T, V, grid, block, 0, st, s, (const T*)x, q, mean, rstd, (T*)y)
}

template <typename T, int V>
void gn_backward(const GnShape& s, const void* x, const void* dy, GnParams q, int act, const float* mean, const float* rstd,
                 void* dx, void* dw, void* db, float2* part, float2* ab, hipStream_t st) {
  const bool sums = dw != nullptr || db != nullptr;
  auto params = [&](long long count, long long stride) {
    if (sums)
      hipLaunchKernelGGL((gn_param_grads<T>), gn_grid((s.channels + GN_PARAM_CH - 1LL) / GN_PARAM_CH),
                         dim3(GN_PARAM_THREADS), 0, st, s.channels, count, stride, part, q.f32, dw, db);
  };
  GnRows rows;
  if (gn_rows(s, V, rows)) {
    const long long per = GN_THREADS * GN_ROW_STEPS;
    const long long blocks = std::min((rows.vectors + per - 1) / per, (long long)GN_TILE_BLOCKS);
    GN_ACTS(act, gn_rows_backward, T, V, dim3((unsigned)blocks), dim3(GN_THREADS), 0, st, rows, (const T*)x, (const T*)dy, q,
            mean, rstd, (T*)dx, sums ? part : nullptr)
    return params(blocks, s.channels);
  }
  GnTile tile;
  if (gn_tile_threads(s.samples, s.length, s.channels, s.groups, V, true, tile) != 0) {
    const size_t lds = gn_tile_lds(tile, 256, true);
    const int blocks = (int)std::min((s.samples + tile.per - 1) / tile.per, (long long)GN_TILE_BLOCKS);
    GN_TILE_ACTS(act, gn_tile_backward, T, V, 256, lds, dim3(blocks), dim3(256), lds, st, tile, (const T*)x, (const T*)dy, q,
                 mean, rstd, (T*)dx, sums ? part : nullptr)
    return params(blocks, s.channels);
  }
  const dim3 grid = gn_grid(s.samples * s.slabs * s.chunks), block(GN_THREADS);
  GN_ACTS(act, gn_sums, T, V, grid, block, 0, st, s, (const T*)x, (const T*)dy, q, mean, rstd, part)
  const long long pairs = s.samples * s.groups;
  int across = 1;
  while (across < GN_THREADS && across < s.cpg) across *= 2;
  const bool wide = s.cpg > 64 && s.chunks > 1;
  if (wide)
    hipLaunchKernelGGL(gn_sums_columns, gn_grid(s.samples * ((s.channels + 63) / 64)), dim3(GN_JOIN_THREADS), 0, st, s,
                       part);
  hipLaunchKernelGGL((gn_sums_join<T>), gn_grid(pairs), block, 0, st, s, wide ? 1 : s.chunks, across, part, q, ab);
  if (dx != nullptr) {
    GN_ACTS(act, gn_dx, T, V, grid, block, 0, st, s, (const T*)x, (const T*)dy, q, mean, rstd, ab, (T*)dx)
  }
  params(s.samples, (long long)s.chunks * s.channels);
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
  if (gn_blocks(s) > GN_BLOCKS_MOST) return nsa_fail(NSA_E_ARG, "%s: too many samples", what);
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
    hipLaunchKernelGGL((gn_param_grads<nsa_f16>), gn_grid((channels + GN_PARAM_CH - 1LL) / GN_PARAM_CH),
                       dim3(GN_PARAM_THREADS), 0, st, channels, 0LL, 0LL, (const float2*)nullptr, f32, dweight_dev, dbias_dev);  // (zero has the same bits in both 16-bit types)
    return gn_done(what);
  }
  if (!x_dev || !dy_dev || !mean_dev || !rstd_dev || !workspace_dev) return nsa_fail(NSA_E_ARG, "%s: NULL argument", what);
  if (workspace_bytes < nsa_group_norm_workspace(samples, length, channels, groups, dtype, 1))
    return nsa_fail(NSA_E_ARG, "%s: workspace too small", what);
  int v;
  const GnShape s = gn_shape(samples, length, channels, groups, nsa_elem_bytes(dtype),
                             (uintptr_t)x_dev | (uintptr_t)dy_dev | (uintptr_t)dx_dev, v);
  if (gn_blocks(s) > GN_BLOCKS_MOST) return nsa_fail(NSA_E_ARG, "%s: too many samples", what);
  const GnParams q = {weight_dev, bias_dev, f32};
  GnTile tile;
  const bool chunked = gn_tile_threads(samples, length, channels, groups, v, true, tile) == 0;
  float2* ab = (float2*)workspace_dev;
  float2* part = ab + (chunked ? samples * groups : 0);
  if (dtype == NSA_DT_F32) { GN_WIDTHS(float, gn_backward, s, x_dev, dy_dev, q, activation, mean_dev, rstd_dev, dx_dev, dweight_dev, dbias_dev, part, ab, st) }
  else if (dtype == NSA_DT_BF16) { GN_WIDTHS(nsa_bf16, gn_backward, s, x_dev, dy_dev, q, activation, mean_dev, rstd_dev, dx_dev, dweight_dev, dbias_dev, part, ab, st) }
  else { GN_WIDTHS(nsa_f16, gn_backward, s, x_dev, dy_dev, q, activation, mean_dev, rstd_dev, dx_dev, dweight_dev, dbias_dev, part, ab, st) }
  return gn_done(what);
}
