// The norm over many gradient tensors and the clip that follows it:
//   T = (sum |g|^p)^(1/p), p = 1, 2 or infinity, over every element of every tensor
//   g <- g * min(1, max_norm / (T + 1e-6))      (rounded once to the gradient's type)
// as torch.nn.utils.clip_grad_norm_ does in the reference's loop (src/nessai/flowmodel/base.py:437-441).
//
// Both are bound by memory: the norm reads every gradient once, the clip reads and writes it once more because the
// factor is known only after the last element.  What many small tensors cost is launches, so the tensors are merged
// into runs (neighbours in memory become one), the runs travel as kernel arguments, NG_RUNS of them per launch, and
// every workgroup takes an equal, contiguous share of the launch's elements whatever the tensors' sizes are.  The
// shares are read in a fixed order and their partial sums added in a fixed order: equal inputs at equal places give equal
// bits.  1.2 GB of float32 in 400 tensors: norm in 219 us (5.5 TB/s; a large copy on this card: 5.07 TB/s, read and written).
// 80 MB of bfloat16 in 301 tensors: norm 18 us (4.4 TB/s), clip 30 us (5.3 TB/s).  Squares and sums are held in 64 bits: a square of a float32 over- or underflows in 32.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <new>
#include <vector>

#include "nsa_elem.h"

#define NG_RUNS 320          // runs per launch: 8 + 4 bytes each, inside the 4 KB of a kernel's arguments
#define NG_MOST (1LL << 31)  // elements per launch: their numbers fit 32 bits (a longer run is cut)
#define NG_THREADS 256
#define NG_BLOCKS 2048       // workgroups of a launch at most: 8 per compute unit ...
#define NG_BLOCKS_MIN 128    // ... and fewer where there are many launches: every partial sum is read by all of them
#define NG_SHARE 4096        // elements of a workgroup's share: a multiple of this

struct NgRuns {
  void* ptr[NG_RUNS];
  uint32_t first[NG_RUNS + 1];  // elements in front of run k
  int count;
};

// |a| and |b| -> the larger one, NaN if either is one (fmaxf drops it)
__device__ __forceinline__ float ng_max(float a, float b) { return (a > b || a != a) ? a : b; }

// Four running sums: neighbouring elements go to different ones, so that no 64-bit addition waits for the one before it.
template <int KIND>
struct NgAcc {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  __device__ __forceinline__ void add(float v, int i) {
    double& a = s[i & 3];
    if constexpr (KIND == NSA_NORM_L2) a = fma((double)v, (double)v, a);
    else if constexpr (KIND == NSA_NORM_L1) a += (double)fabsf(v);
    else a = (double)ng_max((float)a, fabsf(v));
  }
  static __device__ __forceinline__ double two(double a, double b) {
    if constexpr (KIND == NSA_NORM_INF) return (a > b || a != a) ? a : b;
    else return a + b;
  }
  __device__ __forceinline__ double all() const { return two(two(s[0], s[1]), two(s[2], s[3])); }
};

template <int KIND, int THREADS>
__device__ __forceinline__ double ng_block_join(double s) {  // the sum on every thread, in a fixed order
  __shared__ double part[THREADS / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s = NgAcc<KIND>::two(s, __shfl_xor(s, o));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  s = part[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) s = NgAcc<KIND>::two(s, part[w]);
  __syncthreads();
  return s;
}

// the elements [lo, hi) of the launch, run by run: f(pointer, length), each a contiguous piece
template <typename F>
__device__ __forceinline__ void ng_pieces(const NgRuns& r, uint32_t lo, uint32_t hi, F f) {
  int a = 0, b = r.count;  // first[a] <= lo < first[b]
  while (b - a > 1) {
    const int m = (a + b) >> 1;
    if (r.first[m] <= lo) a = m;
    else b = m;
  }
  while (lo < hi) {
    const uint32_t end = r.first[a + 1] < hi ? r.first[a + 1] : hi;
    f(r.ptr[a], lo - r.first[a], end - lo);
    lo = end;
    ++a;
  }
}

// One contiguous piece, cut into single elements up to the first 16-byte border, accesses of 16 bytes - NG_AHEAD of them
// asked for before the first is used - and single elements behind the last border.
//   one(pointer): a single element;  wide(pointer, count): `count` accesses, NG_THREADS of them apart
#define NG_AHEAD 4
template <typename T, typename ONE, typename WIDE>
__device__ __forceinline__ void ng_piece(T* p, long long len, ONE one, WIDE wide) {
  constexpr int V = 16 / sizeof(T);
  long long head = (16 - ((uintptr_t)p & 15)) & 15;
  head = head / (long long)sizeof(T) < len ? head / (long long)sizeof(T) : len;
  const long long body = (len - head) / V * V;
  if (threadIdx.x < head) one(p + threadIdx.x);
  T* q = p + head;
  long long i = (long long)threadIdx.x * V;
  for (; i + (NG_AHEAD - 1) * NG_THREADS * V < body; i += NG_AHEAD * NG_THREADS * V) wide(q + i, NG_AHEAD);
  for (; i < body; i += NG_THREADS * V) wide(q + i, 1);
  const long long rest = len - head - body;  // fewer than V
  if (threadIdx.x < rest) one(q + body + threadIdx.x);
}

// A launch of many short runs (fewer than NG_FLAT elements each on average): element by element, each thread finds the run of
// its own ones.  Piece by piece, 570 tensors of a dozen elements took 0.5 ms: every piece costs a workgroup its latency.
#define NG_FLAT 1024
template <typename T, typename F>
__device__ __forceinline__ void ng_flat(const NgRuns& r, uint32_t lo, uint32_t hi, F f) {
  __shared__ uint32_t first[NG_RUNS + 1];
  for (int k = threadIdx.x; k <= r.count; k += NG_THREADS) first[k] = r.first[k];
  __syncthreads();
#pragma unroll 4
  for (uint32_t e = lo + threadIdx.x; e < hi; e += NG_THREADS) {
    int a = 0, b = r.count;
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (first[m] <= e) a = m;
      else b = m;
    }
    f((T*)r.ptr[a] + (e - first[a]));
  }
}
__device__ __forceinline__ bool ng_is_flat(const NgRuns& r) { return r.first[r.count] / NG_FLAT < (uint32_t)r.count; }

template <typename T, int KIND>
__global__ void __launch_bounds__(NG_THREADS) ng_partial(NgRuns r, uint32_t share, double* __restrict__ partial) {
  constexpr int V = 16 / sizeof(T);
  NgAcc<KIND> acc;
  const uint32_t lo = blockIdx.x * share, total = r.first[r.count], hi = total - lo < share ? total : lo + share;
  if (ng_is_flat(r)) {
    ng_flat<const T>(r, lo, hi, [&](const T* p) { acc.add((float)*p, 0); });
  } else {
  ng_pieces(r, lo, hi, [&](const void* base, uint32_t at, uint32_t len) {
    ng_piece((const T*)base + at, len, [&](const T* p) { acc.add((float)*p, 0); },
             [&](const T* p, int count) {
               float v[NG_AHEAD][V];
#pragma unroll
               for (int k = 0; k < NG_AHEAD; ++k)
                 if (k < count) nsa_load<T, V>(p + k * NG_THREADS * V, v[k]);
#pragma unroll
               for (int k = 0; k < NG_AHEAD; ++k)
                 if (k < count) {
#pragma unroll
                   for (int i = 0; i < V; ++i) acc.add(v[k][i], i);
                 }
             });
  });
  }
  const double s = ng_block_join<KIND, NG_THREADS>(acc.all());
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

template <int KIND>
__device__ __forceinline__ float ng_total(const double* __restrict__ partial, int n_partial) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n_partial; i += NG_THREADS) s = NgAcc<KIND>::two(s, partial[i]);
  s = ng_block_join<KIND, NG_THREADS>(s);
  return (float)(KIND == NSA_NORM_L2 ? sqrt(s) : s);
}

template <int KIND>
__global__ void __launch_bounds__(NG_THREADS) ng_finish(const double* __restrict__ partial, int n_partial,
                                                        float* __restrict__ norm_out) {
  const float norm = ng_total<KIND>(partial, n_partial);
  if (threadIdx.x == 0) norm_out[0] = norm;
}

// min(1, max_norm / (norm + 1e-6)) in float32, NaN kept
__device__ __forceinline__ float ng_factor(float norm, float max_norm) {
  const float f = max_norm / (norm + 1e-6f);
  return f > 1.0f ? 1.0f : f;
}

// Every workgroup adds up the partial sums by itself (at most a few thousand values out of the L2 cache, in the same
// order everywhere) instead of waiting for one that does: one launch less between the norm and the product.
template <typename T, int KIND>
__global__ void __launch_bounds__(NG_THREADS) ng_scale(NgRuns r, uint32_t share, const double* __restrict__ partial,
                                                       int n_partial, float max_norm, float* __restrict__ norm_out) {
  constexpr int V = 16 / sizeof(T);
  const float norm = ng_total<KIND>(partial, n_partial);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out != nullptr) norm_out[0] = norm;
  const float f = ng_factor(norm, max_norm);
  if (f == 1.0f) return;  // (a product by one changes nothing)
  // the shares from the last to the first: what the norm read last is the likeliest to be in a cache still
  const uint32_t lo = (gridDim.x - 1 - blockIdx.x) * share, total = r.first[r.count];
  const uint32_t hi = total - lo < share ? total : lo + share;
  if (ng_is_flat(r)) return ng_flat<T>(r, lo, hi, [&](T* p) { *p = (T)((float)*p * f); });
  ng_pieces(r, lo, hi, [&](void* base, uint32_t at, uint32_t len) {
    ng_piece((T*)base + at, len, [&](T* p) { *p = (T)((float)*p * f); },
             [&](T* p, int count) {
               float v[NG_AHEAD][V];
#pragma unroll
               for (int k = 0; k < NG_AHEAD; ++k)
                 if (k < count) nsa_load<T, V>(p + k * NG_THREADS * V, v[k]);
#pragma unroll
               for (int k = 0; k < NG_AHEAD; ++k)
                 if (k < count) {
#pragma unroll
                   for (int i = 0; i < V; ++i) v[k][i] *= f;
                   nsa_store<T, V>(p + k * NG_THREADS * V, v[k]);
                 }
             });
  });
}

// A few thousand elements: norm and clip in one workgroup and one launch, each element kept in a register between
// them: 9600 float32 in 4.0 us, in two launches 4.4; 16384, the most a workgroup's registers take, in 4.5 and 5.0.
#define NG_SMALL_THREADS 1024
#define NG_SMALL_EACH 16
#define NG_SMALL (NG_SMALL_THREADS * NG_SMALL_EACH)
template <typename T, int KIND>
__global__ void __launch_bounds__(NG_SMALL_THREADS) ng_small(NgRuns r, int clip, float max_norm,
                                                             float* __restrict__ norm_out) {
  __shared__ int first[NG_RUNS + 1];
  __shared__ T* ptr[NG_RUNS];
  for (int k = threadIdx.x; k <= r.count; k += NG_SMALL_THREADS) {
    first[k] = (int)r.first[k];
    if (k < r.count) ptr[k] = (T*)r.ptr[k];
  }
  __syncthreads();
  const int total = first[r.count];
  T* at[NG_SMALL_EACH];
  float v[NG_SMALL_EACH];
#pragma unroll
  for (int k = 0; k < NG_SMALL_EACH; ++k) {
    const int e = k * NG_SMALL_THREADS + threadIdx.x;
    v[k] = 0.0f;
    if (e < total) {
      int a = 0, b = r.count;
      while (b - a > 1) {
        const int m = (a + b) >> 1;
        if (first[m] <= e) a = m;
        else b = m;
      }
      at[k] = ptr[a] + (e - first[a]);
      v[k] = (float)*at[k];
    }
  }
  NgAcc<KIND> acc;
#pragma unroll
  for (int k = 0; k < NG_SMALL_EACH; ++k) acc.add(v[k], k);
  const double s = ng_block_join<KIND, NG_SMALL_THREADS>(acc.all());
  const float norm = (float)(KIND == NSA_NORM_L2 ? sqrt(s) : s);
  if (threadIdx.x == 0) norm_out[0] = norm;
  const float f = clip ? ng_factor(norm, max_norm) : 1.0f;
  if (f == 1.0f) return;
#pragma unroll
  for (int k = 0; k < NG_SMALL_EACH; ++k)
    if (k * NG_SMALL_THREADS + (int)threadIdx.x < total) *at[k] = (T)(v[k] * f);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

struct Run {
  char* ptr;
  long long n;
  int dtype;
};

// The tensors as runs, in the order of their places, tensors side by side merged.  false: two of them overlap.
bool ng_runs(int count, void* const* tensors, const long long* sizes, const int* dtypes, std::vector<Run>& runs) {
  runs.clear();
  runs.reserve(count);
  for (int i = 0; i < count; ++i)
    if (sizes[i] > 0) runs.push_back({(char*)tensors[i], sizes[i], dtypes[i]});
  std::sort(runs.begin(), runs.end(), [](const Run& a, const Run& b) { return a.ptr < b.ptr; });
  bool apart = true;
  size_t kept = 0;
  for (size_t i = 0; i < runs.size(); ++i) {
    if (kept > 0) {
      Run& last = runs[kept - 1];
      char* end = last.ptr + last.n * nsa_elem_bytes(last.dtype);
      if (runs[i].ptr < end) apart = false;
      if (runs[i].ptr == end && runs[i].dtype == last.dtype) {
        last.n += runs[i].n;
        continue;
      }
    }
    runs[kept++] = runs[i];
  }
  runs.resize(kept);
  std::stable_sort(runs.begin(), runs.end(), [](const Run& a, const Run& b) { return a.dtype < b.dtype; });
  return apart;
}

struct Launch {
  NgRuns r;
  int dtype, blocks;
  uint32_t share;
};

void ng_launches(const std::vector<Run>& runs, std::vector<Launch>& out) {
  out.clear();
  size_t i = 0;
  long long done = 0;  // of run i
  while (i < runs.size()) {
    Launch l;
    l.dtype = runs[i].dtype;
    l.r.count = 0;
    l.r.first[0] = 0;
    while (i < runs.size() && l.r.count < NG_RUNS && runs[i].dtype == l.dtype) {
      const long long room = NG_MOST - l.r.first[l.r.count], n = std::min(runs[i].n - done, room);
      if (n == 0) break;
      l.r.ptr[l.r.count] = runs[i].ptr + done * nsa_elem_bytes(l.dtype);
      l.r.first[l.r.count + 1] = (uint32_t)(l.r.first[l.r.count] + n);
      ++l.r.count;
      done += n;
      if (done == runs[i].n) {
        ++i;
        done = 0;
      }
    }
    out.push_back(l);
  }
  const int blocks = std::max(NG_BLOCKS_MIN, 2 * NG_BLOCKS / (int)(out.size() + 1));
  for (Launch& l : out) {
    const long long total = l.r.first[l.r.count], shares = (total + NG_SHARE - 1) / NG_SHARE;
    l.share = (uint32_t)((shares + blocks - 1) / blocks * NG_SHARE);
    if (total / NG_FLAT < l.r.count) l.share = NG_THREADS * 4;  // (ng_flat: four elements a thread, all asked for at once)
    l.blocks = (int)((total + l.share - 1) / l.share);
  }
}

#define NG_KINDS(T, KERNEL, ...)                                                    \
  switch (kind) {                                                                   \
    case NSA_NORM_L1: hipLaunchKernelGGL((KERNEL<T, NSA_NORM_L1>), __VA_ARGS__); break;   \
    case NSA_NORM_L2: hipLaunchKernelGGL((KERNEL<T, NSA_NORM_L2>), __VA_ARGS__); break;   \
    default: hipLaunchKernelGGL((KERNEL<T, NSA_NORM_INF>), __VA_ARGS__); break;           \
  }
#define NG_DISPATCH(dtype, KERNEL, ...)                              \
  switch (dtype) {                                                   \
    case NSA_DT_F32: NG_KINDS(float, KERNEL, __VA_ARGS__) break;     \
    case NSA_DT_BF16: NG_KINDS(nsa_bf16, KERNEL, __VA_ARGS__) break; \
    default: NG_KINDS(nsa_f16, KERNEL, __VA_ARGS__) break;           \
  }

int ng_run(const char* what, int count, void* const* tensors, const long long* sizes, const int* dtypes, int kind,
           bool clip, float max_norm, double* workspace, size_t workspace_bytes, float* norm_out, hipStream_t s) {
  if (count < 0 || (count > 0 && (!tensors || !sizes || !dtypes)) || !norm_out || !workspace)
    return nsa_fail(NSA_E_ARG, "%s: NULL argument", what);
  if (kind != NSA_NORM_L1 && kind != NSA_NORM_L2 && kind != NSA_NORM_INF)
    return nsa_fail(NSA_E_ARG, "%s: unknown norm %d", what, kind);
  if (clip && !(max_norm >= 0.0f)) return nsa_fail(NSA_E_ARG, "%s: max_norm must not be negative or NaN", what);
  for (int i = 0; i < count; ++i) {
    if (!nsa_elem_known(dtypes[i])) return nsa_fail(NSA_E_ARG, "%s: unknown type %d of tensor %d", what, dtypes[i], i);
    if (sizes[i] < 0 || (sizes[i] > 0 && !tensors[i])) return nsa_fail(NSA_E_ARG, "%s: bad tensor %d", what, i);
    if ((uintptr_t)tensors[i] % nsa_elem_bytes(dtypes[i]) != 0)
      return nsa_fail(NSA_E_ARG, "%s: tensor %d is not aligned to its elements", what, i);
  }
  try {
    std::vector<Run> runs;
    std::vector<Launch> launches;
    const bool apart = ng_runs(count, tensors, sizes, dtypes, runs);
    if (clip && !apart) return nsa_fail(NSA_E_ARG, "%s: two gradients overlap in memory", what);
    ng_launches(runs, launches);
    size_t partials = 0;
    for (const Launch& l : launches) partials += l.blocks;
    if (workspace_bytes < partials * sizeof(double)) return nsa_fail(NSA_E_ARG, "%s: workspace too small", what);
    if (launches.size() == 1 && launches[0].r.first[launches[0].r.count] <= NG_SMALL) {
      const Launch& l = launches[0];
      NG_DISPATCH(l.dtype, ng_small, dim3(1), dim3(NG_SMALL_THREADS), 0, s, l.r, clip ? 1 : 0, max_norm, norm_out)
      const hipError_t e = hipGetLastError();
      return e == hipSuccess ? NSA_OK : nsa_fail(NSA_E_HIP, "%s: %s", what, hipGetErrorString(e));
    }
    int n_partial = 0;
    for (const Launch& l : launches) {
      NG_DISPATCH(l.dtype, ng_partial, dim3(l.blocks), dim3(NG_THREADS), 0, s, l.r, l.share, workspace + n_partial)
      n_partial += l.blocks;
    }
    if (!clip || launches.empty()) {
      if (kind == NSA_NORM_L1)
        hipLaunchKernelGGL(ng_finish<NSA_NORM_L1>, dim3(1), dim3(NG_THREADS), 0, s, workspace, n_partial, norm_out);
      else if (kind == NSA_NORM_L2)
        hipLaunchKernelGGL(ng_finish<NSA_NORM_L2>, dim3(1), dim3(NG_THREADS), 0, s, workspace, n_partial, norm_out);
      else
        hipLaunchKernelGGL(ng_finish<NSA_NORM_INF>, dim3(1), dim3(NG_THREADS), 0, s, workspace, n_partial, norm_out);
    } else {
      float* out = norm_out;
      for (const Launch& l : launches) {
        NG_DISPATCH(l.dtype, ng_scale, dim3(l.blocks), dim3(NG_THREADS), 0, s, l.r, l.share, workspace, n_partial,
                    max_norm, out)
        out = nullptr;
      }
    }
  } catch (const std::bad_alloc&) {
    return nsa_fail(NSA_E_ARG, "%s: out of host memory", what);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? NSA_OK : nsa_fail(NSA_E_HIP, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace

// One partial sum per workgroup.  `count` tensors make at most count / NG_RUNS + 3 launches (one not full for each type) and
// one more for every NG_MOST elements; with L launches a launch has at most max(NG_BLOCKS_MIN, 2 NG_BLOCKS / (L + 1)) groups.
extern "C" NSA_API size_t nsa_grad_norm_workspace(int count, long long elements) {
  const size_t launches = (size_t)std::max(count, 0) / NG_RUNS + 3 + (size_t)(std::max(elements, 0LL) / NG_MOST);
  return (launches * std::max(NG_BLOCKS_MIN, NG_RUNS * NG_FLAT / (NG_THREADS * 4)) + 2 * NG_BLOCKS) * sizeof(double);
}

extern "C" NSA_API int nsa_grad_norm(int count, void* const* tensors, const long long* sizes, const int* dtypes, int kind,
                                     void* workspace_dev, size_t workspace_bytes, float* norm_out_dev, void* stream) {
  return ng_run("nsa_grad_norm", count, tensors, sizes, dtypes, kind, false, 0.0f, (double*)workspace_dev, workspace_bytes,
                norm_out_dev, (hipStream_t)stream);
}

extern "C" NSA_API int nsa_grad_clip(int count, void* const* tensors, const long long* sizes, const int* dtypes, int kind,
                                     float max_norm, void* workspace_dev, size_t workspace_bytes, float* norm_out_dev,
                                     void* stream) {
  return ng_run("nsa_grad_clip", count, tensors, sizes, dtypes, kind, true, max_norm, (double*)workspace_dev,
                workspace_bytes, norm_out_dev, (hipStream_t)stream);
}
