// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = W[id_i] * scale                      dW[v] = scale * sum_{i : id_i = v} dy[i]
//
// The lookup moves rows: a team of lanes takes a row, 16 bytes to a lane where rows and addresses allow it.  200003 rows of
// 512 bfloat16 out of a table of 410 MB: 74 us, 5.5 TB/s (a large copy on this card: 5.07 TB/s).
//
// The gradient must add the rows of equal ids.  Float atomics would add them in an order that changes from run to run, so
// the tokens are sorted by id first - a stable radix sort of (id, position), 8 bits to a pass, as many passes as the
// table's size has digits - and the sums then run over neighbours, in the order of the positions: equal inputs give equal
// bits.  The sorted list is cut into chunks of equal length, whatever the frequencies of the ids: an id inside one chunk
// is finished there; one that runs over a chunk's border leaves float32 partial sums, which a second kernel joins.
// 131072 rows of 320 bfloat16 into 32768 (84 MB in, 21 MB out): 61 us; sorting and clearing 15 + 12, adding 21, joining 13.
// The sums are bound by gathering rows (4.0 TB/s), the sort of so few tokens by the latency of its short kernels.  Sorting
// 10^6 tokens into 5000 takes 43 us (counts 14, scans 10, scatters 19) for 48 MB read and written.
#include <hip/hip_runtime.h>
#include <algorithm>

#include "nsa_elem.h"

#define EMB_THREADS 256
#define EMB_MANY 1500000                      // tokens from which a sorting tile has 16 keys per thread instead of 4
#define EMB_AHEAD 8                           // rows in flight per team
#define EMB_FEW_AHEAD 16                      // the same where a row is four bytes a lane
#define EMB_FEW 64                            // (rows + 1) x columns per lane of a gradient summed in LDS (64 KB)

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------

template <typename T, typename ID, int V>
__global__ void __launch_bounds__(EMB_THREADS) emb_lookup(long long tokens, long long vocab, int width,
                                                          const ID* __restrict__ ids, const T* __restrict__ weight,
                                                          float scale, int lanes, T* __restrict__ out) {
  const int teams = EMB_THREADS / lanes, lane = threadIdx.x % lanes;
  for (long long row = (long long)blockIdx.x * teams + threadIdx.x / lanes; row < tokens; row += (long long)gridDim.x * teams) {
    const long long id = (long long)ids[row];
    const bool known = id >= 0 && id < vocab;
    for (int c = lane * V; c < width; c += lanes * V) {
      float v[V];
      if (known) {
        nsa_load<T, V>(weight + id * width + c, v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= scale;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = __builtin_nanf("");
      }
      nsa_store<T, V>(out + row * width + c, v);
    }
  }
}

// ---------------------------------------------------------------------------
// clearing the gradient's rows
// ---------------------------------------------------------------------------

// `halves` 16-bit words of the table set to zero by `threads` threads of which this is the i-th
__device__ __forceinline__ void emb_clear(uint16_t* __restrict__ table, long long halves, long long i, long long threads) {
  if ((uintptr_t)table % 16 == 0 && halves % 8 == 0) {
    const NsaPack<uint32_t, 4> zero = {{0u, 0u, 0u, 0u}};
    for (; i < halves / 8; i += threads) reinterpret_cast<NsaPack<uint32_t, 4>*>(table)[i] = zero;
  } else {
    for (; i < halves; i += threads) table[i] = 0;
  }
}

// the table alone: no tokens
__global__ void __launch_bounds__(EMB_THREADS) emb_zero(uint16_t* __restrict__ table, long long halves) {
  emb_clear(table, halves, (long long)blockIdx.x * EMB_THREADS + threadIdx.x, (long long)gridDim.x * EMB_THREADS);
}

// ---------------------------------------------------------------------------
// stable radix sort of (id, position)
// ---------------------------------------------------------------------------

// the key of a token: its id, or `vocab` (behind every row) for a token without a gradient
template <typename ID>
__device__ __forceinline__ uint32_t emb_key(const ID* ids, long long i, long long vocab, long long padding) {
  const long long id = (long long)ids[i];
  return id >= 0 && id < vocab && id != padding ? (uint32_t)id : (uint32_t)vocab;
}

// the lanes of the wave that are `here` and have this lane's digit
__device__ __forceinline__ unsigned long long emb_same(uint32_t digit, bool here) {
  unsigned long long same = __ballot(here);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const unsigned long long set = __ballot((digit >> b) & 1u);
    same &= (digit >> b) & 1u ? set : ~set;
  }
  return same;
}

// digit counts of every tile: counts[digit][tile]; the first pass reads the ids themselves (keys == nullptr), and workgroups
// of it behind the tiles clear the table and the list of runs
template <typename ID, int ITEMS>
__global__ void __launch_bounds__(EMB_THREADS) emb_count(int n, const ID* __restrict__ ids, long long vocab,
                                                         long long padding, const uint32_t* __restrict__ keys, int shift,
                                                         int tiles, uint32_t* __restrict__ counts,
                                                         uint16_t* __restrict__ table, long long halves,
                                                         uint32_t* __restrict__ runs) {
  __shared__ uint32_t bins[256];
  if ((int)blockIdx.x >= tiles) {
    if ((int)blockIdx.x == tiles && threadIdx.x == 0) runs[0] = 0;
    emb_clear(table, halves, (long long)(blockIdx.x - tiles) * EMB_THREADS + threadIdx.x,
              (long long)(gridDim.x - tiles) * EMB_THREADS);
    return;
  }
  bins[threadIdx.x] = 0;
  __syncthreads();
  const long long base = (long long)blockIdx.x * (EMB_THREADS * ITEMS);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const long long i = base + k * EMB_THREADS + threadIdx.x;
    if (i < n) {
      const uint32_t key = keys != nullptr ? keys[i] : emb_key(ids, i, vocab, padding);
      atomicAdd(&bins[(key >> shift) & 255u], 1u);
    }
  }
  __syncthreads();
  counts[(long long)threadIdx.x * tiles + blockIdx.x] = bins[threadIdx.x];
}

// one workgroup per digit: its tiles' counts become the counts in front of them, totals[digit] their sum
__global__ void __launch_bounds__(EMB_THREADS) emb_scan(int tiles, uint32_t* __restrict__ counts,
                                                        uint32_t* __restrict__ totals) {
  __shared__ uint32_t wave_sum[EMB_THREADS / 64];
  uint32_t* row = counts + (long long)blockIdx.x * tiles;
  uint32_t carry = 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int base = 0; base < tiles; base += EMB_THREADS) {
    const int i = base + threadIdx.x;
    const uint32_t v = i < tiles ? row[i] : 0u;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t t = __shfl_up(s, o);
      if (lane >= o) s += t;
    }
    if (lane == 63) wave_sum[wave] = s;
    __syncthreads();
    uint32_t before = carry, all = 0;
    for (int w = 0; w < EMB_THREADS / 64; ++w) {
      if (w < wave) before += wave_sum[w];
      all += wave_sum[w];
    }
    if (i < tiles) row[i] = before + s - v;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// The tile's keys to their places.  Each wave owns a contiguous quarter of the tile and counts its digits first; the place
// of a key is then (keys of smaller digits) + (the digit's keys in earlier tiles, in earlier waves, in earlier rounds of
// this wave, in lower lanes): equal digits keep their order.
template <typename ID, int ITEMS>
__global__ void __launch_bounds__(EMB_THREADS) emb_scatter(int n, const ID* __restrict__ ids, long long vocab,
                                                           long long padding, const uint32_t* __restrict__ keys,
                                                           const uint32_t* __restrict__ pos, int shift,
                                                           const uint32_t* __restrict__ counts,
                                                           const uint32_t* __restrict__ totals,
                                                           uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out) {
  constexpr int WAVES = EMB_THREADS / 64;
  __shared__ uint32_t place[WAVES][256];
  __shared__ uint32_t wave_sum[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int w = 0; w < WAVES; ++w) place[w][threadIdx.x] = 0;
  // keys of smaller digits: an exclusive scan of the 256 totals, one digit per thread
  const uint32_t total = totals[threadIdx.x];
  uint32_t s = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = __shfl_up(s, o);
    if (lane >= o) s += t;
  }
  if (lane == 63) wave_sum[wave] = s;
  __syncthreads();
  uint32_t first = s - total;
  for (int w = 0; w < wave; ++w) first += wave_sum[w];

  const long long base = (long long)blockIdx.x * (EMB_THREADS * ITEMS) + wave * (64 * ITEMS) + lane;
  uint32_t key[ITEMS], from[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const long long i = base + k * 64;
    key[k] = from[k] = 0;
    if (i < n) {
      key[k] = keys != nullptr ? keys[i] : emb_key(ids, i, vocab, padding);
      from[k] = pos != nullptr ? pos[i] : (uint32_t)i;
      atomicAdd(&place[wave][(key[k] >> shift) & 255u], 1u);
    }
  }
  __syncthreads();
  uint32_t at = first + counts[(long long)threadIdx.x * gridDim.x + blockIdx.x];
  for (int w = 0; w < WAVES; ++w) {
    const uint32_t c = place[w][threadIdx.x];
    place[w][threadIdx.x] = at;
    at += c;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const bool here = base + k * 64 < n;
    const uint32_t digit = (key[k] >> shift) & 255u;
    const unsigned long long same = emb_same(digit, here);
    const uint32_t rank = __popcll(same & ((1ULL << lane) - 1ULL));
    if (here) {
      const uint32_t to = __hip_atomic_load(&place[wave][digit], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) + rank;
      keys_out[to] = key[k];
      pos_out[to] = from[k];
    }
    __builtin_amdgcn_wave_barrier();  // every lane has read its place before the round's count is added
    if (here && rank == 0) atomicAdd(&place[wave][digit], (uint32_t)__popcll(same));
    __builtin_amdgcn_wave_barrier();
  }
}

// A few thousand tokens: every pass of the sort in one workgroup, the pairs in LDS between them, as many passes as the table
// has digits.  The other workgroups of the launch clear the table meanwhile.  The whole gradient of 4096 tokens into 60000 x 32
// float32 takes 21 us so, 34 with a launch for each step; 1000 into 1000 x 32 take 20 and 27.
#define EMB_SHORT_THREADS 1024
#define EMB_SHORT_ITEMS 4
#define EMB_SHORT (EMB_SHORT_THREADS * EMB_SHORT_ITEMS)
template <typename ID>
__global__ void __launch_bounds__(EMB_SHORT_THREADS) emb_sort_short(int n, const ID* __restrict__ ids, long long vocab,
                                                                    long long padding, int passes,
                                                                    uint32_t* __restrict__ keys_out,
                                                                    uint32_t* __restrict__ pos_out,
                                                                    uint16_t* __restrict__ table, long long halves,
                                                                    uint32_t* __restrict__ runs) {
  constexpr int WAVES = EMB_SHORT_THREADS / 64;
  if (blockIdx.x > 0) {
    emb_clear(table, halves, (blockIdx.x - 1LL) * EMB_SHORT_THREADS + threadIdx.x, (gridDim.x - 1LL) * EMB_SHORT_THREADS);
    return;
  }
  __shared__ uint32_t place[WAVES][256];
  __shared__ uint32_t wave_sum[4];
  __shared__ uint32_t key_at[EMB_SHORT], pos_at[EMB_SHORT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, base = wave * (64 * EMB_SHORT_ITEMS) + lane;
  if (threadIdx.x == 0) runs[0] = 0;
  uint32_t key[EMB_SHORT_ITEMS], from[EMB_SHORT_ITEMS];
#pragma unroll
  for (int k = 0; k < EMB_SHORT_ITEMS; ++k) {
    const int i = base + k * 64;
    key[k] = i < n ? emb_key(ids, i, vocab, padding) : 0u;
    from[k] = (uint32_t)i;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = 8 * p;
    for (int i = threadIdx.x; i < WAVES * 256; i += EMB_SHORT_THREADS) place[i >> 8][i & 255] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EMB_SHORT_ITEMS; ++k)
      if (base + k * 64 < n) atomicAdd(&place[wave][(key[k] >> shift) & 255u], 1u);
    __syncthreads();
    // a digit per thread of the first four waves: its total, the totals in front of it, and the waves' places
    uint32_t total = 0, s = 0;
    if (threadIdx.x < 256) {
      for (int w = 0; w < WAVES; ++w) total += place[w][threadIdx.x];
      s = total;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t t = __shfl_up(s, o);
        if (lane >= o) s += t;
      }
      if (lane == 63) wave_sum[wave] = s;
    }
    __syncthreads();
    if (threadIdx.x < 256) {
      uint32_t at = s - total;
      for (int w = 0; w < wave; ++w) at += wave_sum[w];
      for (int w = 0; w < WAVES; ++w) {
        const uint32_t c = place[w][threadIdx.x];
        place[w][threadIdx.x] = at;
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EMB_SHORT_ITEMS; ++k) {
      const bool here = base + k * 64 < n;
      const uint32_t digit = (key[k] >> shift) & 255u;
      const unsigned long long same = emb_same(digit, here);
      const uint32_t rank = __popcll(same & ((1ULL << lane) - 1ULL));
      if (here) {
        const uint32_t to = __hip_atomic_load(&place[wave][digit], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) + rank;
        key_at[to] = key[k];
        pos_at[to] = from[k];
      }
      __builtin_amdgcn_wave_barrier();
      if (here && rank == 0) atomicAdd(&place[wave][digit], (uint32_t)__popcll(same));
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EMB_SHORT_ITEMS; ++k)
      if (base + k * 64 < n) {
        key[k] = key_at[base + k * 64];
        from[k] = pos_at[base + k * 64];
      }
  }
#pragma unroll
  for (int k = 0; k < EMB_SHORT_ITEMS; ++k)
    if (base + k * 64 < n) {
      keys_out[base + k * 64] = key[k];
      pos_out[base + k * 64] = from[k];
    }
}

// ---------------------------------------------------------------------------
// sums over equal ids
// ---------------------------------------------------------------------------

// A team of `lanes` lanes takes a chunk of sorted positions, V columns to a lane; EMB_AHEAD rows are asked for before the first
// is added.  slots[chunk][0]: the partial sum of an id that began in an earlier chunk; [1]: of one that began here and
// goes on in the next: such a chunk is entered into the list `runs` (its length in runs[0]), in any order - the runs are
// joined one by one.
template <typename T, int V>
__global__ void __launch_bounds__(EMB_THREADS) emb_reduce(int n, uint32_t vocab, int width, int lanes, int chunk_len,
                                                          const uint32_t* __restrict__ keys,
                                                          const uint32_t* __restrict__ pos, const T* __restrict__ dy,
                                                          float scale, T* __restrict__ dweight,
                                                          float* __restrict__ slots, uint32_t* __restrict__ runs) {
  const int teams = EMB_THREADS / lanes;
  const long long chunk = (long long)blockIdx.x * teams + threadIdx.x / lanes;
  const long long begin = chunk * chunk_len;
  const int c = (blockIdx.y * lanes + threadIdx.x % lanes) * V;
  if (begin >= n || c >= width) return;
  const int len = begin + chunk_len < n ? chunk_len : (int)(n - begin);
  const bool goes_on = begin + len < n && keys[begin + len] == keys[begin + len - 1];
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  uint32_t key = keys[begin];
  bool earlier = begin > 0 && keys[begin - 1] == key;
  auto leave = [&](bool later) {  // the sum of `key` to where it belongs
    if (key != vocab) {
      if (earlier || later) {
        nsa_store<float, V>(slots + (2 * chunk + (earlier ? 0 : 1)) * width + c, acc);
      } else {
        float out[V];
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = acc[v] * scale;
        nsa_store<T, V>(dweight + (long long)key * width + c, out);
      }
    }
  };
  for (int i = 0; i < len; i += EMB_AHEAD) {
    uint32_t k[EMB_AHEAD];
    NsaPack<T, V> row[EMB_AHEAD];
#pragma unroll
    for (int j = 0; j < EMB_AHEAD; ++j) {
      const long long at = begin + (i + j < len ? i + j : len - 1);
      k[j] = keys[at];
      row[j] = *reinterpret_cast<const NsaPack<T, V>*>(dy + (long long)pos[at] * width + c);
    }
#pragma unroll
    for (int j = 0; j < EMB_AHEAD; ++j) {
      if (i + j >= len) break;
      if (k[j] != key) {
        leave(false);
        key = k[j];
        earlier = false;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += (float)row[j].v[v];
    }
  }
  leave(goes_on);
  if (c == 0 && goes_on && !earlier && key != vocab) runs[1 + atomicAdd(runs, 1u)] = (uint32_t)chunk;
}

// The runs over chunk borders, one by one: a workgroup takes EMB_JOIN_COLS columns of a run at a time; its four waves share
// the run's chunks out and their sums are added in order.
#define EMB_JOIN_COLS 64
template <typename T>
__global__ void __launch_bounds__(EMB_THREADS) emb_join(int n, int width, int chunk_len, const uint32_t* __restrict__ keys,
                                                        float scale, const float* __restrict__ slots,
                                                        const uint32_t* __restrict__ runs, T* __restrict__ dweight) {
  __shared__ float sums[EMB_THREADS];
  const long long chunks = (n - 1LL) / chunk_len + 1;
  const int slabs = (width + EMB_JOIN_COLS - 1) / EMB_JOIN_COLS;
  const long long items = (long long)runs[0] * slabs;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const long long chunk = runs[1 + item / slabs];
    const uint32_t key = keys[(chunk + 1) * chunk_len];
    // the last chunk that begins inside the run: in steps that double, then by halves
    long long last = chunk + 1, step = 1;
    while (last + step < chunks && keys[(last + step) * chunk_len] == key) {
      last += step;
      step *= 2;
    }
    for (; step > 0; step >>= 1)
      if (last + step < chunks && keys[(last + step) * chunk_len] == key) last += step;
    const int c = (int)(item % slabs) * EMB_JOIN_COLS + (threadIdx.x & 63), part = threadIdx.x >> 6;
    float acc = 0.0f;
    if (c < width) {
#pragma unroll 8
      for (long long k = chunk + 1 + part; k <= last; k += EMB_THREADS / 64) acc += slots[2 * k * width + c];
    }
    sums[threadIdx.x] = acc;
    __syncthreads();
    if (part == 0 && c < width) {
      acc += slots[(2 * chunk + 1) * width + c];
      for (int p = 1; p < EMB_THREADS / 64; ++p) acc += sums[p * 64 + threadIdx.x];
      dweight[(long long)key * width + c] = (T)(acc * scale);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// tables of a few rows: no sorting
// ---------------------------------------------------------------------------

// A table of fewer than EMB_FEW rows (half of that in 16 bits) fits in LDS many times over: every lane keeps a copy of its own
// columns for all rows and adds its tokens there, in their order - no two lanes ever add to the same place.  A row takes
// `lanes` lanes, W columns (4 bytes) each; a wave works on 64 / lanes tokens at a time.  The copies of a workgroup are added in
// order and left as part[block][row][column].
// Its bound is the work per token - loads of four bytes a lane, then a read, an add and a write in LDS that the next token waits
// for.  Offsets are 32 bits from the workgroup's first row, and where a token has a wave to itself (WAVE) its id, the test of it
// and its address are scalar: 10^6 rows of 64 float32 into 40 in 86 us (3.0 TB/s; 107 without either).  Sorted, the
// same gradient takes 134 us, 1000 rows of 16 into 6 take 18 instead of 6 us, 100000 of 64 into 62 29 instead of 23.
template <typename T, typename ID, int W, bool WAVE>
__global__ void __launch_bounds__(EMB_THREADS) emb_few(long long tokens, int vocab, int width, int lanes, int share,
                                                       const ID* __restrict__ ids, long long padding,
                                                       const T* __restrict__ dy, float* __restrict__ part) {
  extern __shared__ float acc[];  // [vocab + 1][EMB_THREADS][W]
  const int cells = vocab * EMB_THREADS * W;
  for (int i = threadIdx.x; i < cells; i += EMB_THREADS) acc[i] = 0.0f;
  __syncthreads();
  const int c = (blockIdx.y * lanes + threadIdx.x % lanes) * W;
  const int teams = EMB_THREADS / lanes;
  const int team = WAVE ? __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) : (int)threadIdx.x / lanes;
  const long long lo = (long long)blockIdx.x * share;
  const int len = tokens - lo < share ? (int)(tokens - lo) : share;
  const ID* id_of = ids + lo;
  const char* row_of = (const char*)(dy + lo * width);
  const uint32_t stride = (uint32_t)width * sizeof(T), lane_at = (uint32_t)c * sizeof(T);
  float* mine = acc + threadIdx.x * W;
  if (c < width) {
    for (int i = team; i < len; i += teams * EMB_FEW_AHEAD) {
      ID id[EMB_FEW_AHEAD];
      NsaPack<T, W> row[EMB_FEW_AHEAD];
#pragma unroll
      for (int j = 0; j < EMB_FEW_AHEAD; ++j) {  // (behind the end: the last token again, which is passed over below)
        const int at = i + j * teams < len ? i + j * teams : len - 1;
        id[j] = id_of[at];
        row[j] = *reinterpret_cast<const NsaPack<T, W>*>(row_of + ((uint32_t)at * stride + lane_at));
      }
      __builtin_amdgcn_sched_barrier(0);  // (all of them asked for before anything is waited for)
#pragma unroll
      for (int j = 0; j < EMB_FEW_AHEAD; ++j) {
        const bool counts = (i + j * teams < len) & ((unsigned long long)(long long)id[j] < (unsigned long long)vocab) &
                            ((long long)id[j] != padding);
        float* p = mine + (counts ? (int)id[j] : vocab) * (EMB_THREADS * W);  // (the others into a row that nobody reads)
#pragma unroll
        for (int w = 0; w < W; ++w) p[w] += (float)row[j].v[w];  // (LDS float atomics take three times as long)
      }
    }
  }
  __syncthreads();
  const int span = lanes * W;
  for (int i = threadIdx.x; i < vocab * span; i += EMB_THREADS) {
    const int row = i / span, e = i - row * span, col = blockIdx.y * span + e;
    if (col >= width) continue;
    float s = 0.0f;
    for (int t = 0; t < teams; ++t) s += acc[(row * EMB_THREADS + t * lanes) * W + e];
    part[((long long)blockIdx.x * vocab + row) * width + col] = s;
  }
}

// dweight = scale * sum over the workgroups' records, in 64 bits
#define EMB_SUM_THREADS 1024
#define EMB_SUM_CELLS 32
template <typename T>
__global__ void __launch_bounds__(EMB_SUM_THREADS) emb_few_join(int cells, int count, const float* __restrict__ part,
                                                                float scale, T* __restrict__ dweight) {
  constexpr int LANES = EMB_SUM_THREADS / EMB_SUM_CELLS;
  __shared__ double red[EMB_SUM_THREADS];
  const int i = blockIdx.x * EMB_SUM_CELLS + threadIdx.x % EMB_SUM_CELLS, lane = threadIdx.x / EMB_SUM_CELLS;
  double s = 0.0;
  if (i < cells) {
#pragma unroll 4
    for (int k = lane; k < count; k += LANES) s += (double)part[(long long)k * cells + i];
  }
  red[threadIdx.x] = s;
  __syncthreads();
#pragma unroll
  for (int half = LANES / 2; half > 0; half >>= 1) {
    if (lane < half) red[threadIdx.x] += red[threadIdx.x + half * EMB_SUM_CELLS];
    __syncthreads();
  }
  if (lane == 0 && i < cells) dweight[i] = (T)(float)(red[threadIdx.x] * (double)scale);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

// the widest access, in elements, that rows of `width` elements at these addresses allow
int emb_vector(int width, int bytes, uintptr_t addresses) {
  int v = 16 / bytes;
  while (v > 1 && (width % v != 0 || addresses % (uintptr_t)(v * bytes) != 0)) v >>= 1;
  return v;
}

// Lanes of a team, a power of two, for rows of `vectors` accesses of `bytes` each.  A short row: one access of each lane.  A
// longer one: as many lanes as make 128 bytes side by side (a wave at most), or more where that leaves at most an eighth of
// them idle in their last round; 40 accesses of 16 bytes, for one, are five rounds of 8.
int emb_lanes(int vectors, int bytes) {
  const int least = std::min(64, 128 / bytes);
  int best = 1;
  while (best < least && best < vectors) best *= 2;
  for (int l = 2 * best; l <= 64 && vectors > best; l *= 2)
    if ((vectors + l - 1) / l * l * 8 <= vectors * 9) best = l;
  return best;
}

int emb_passes(long long vocab) {  // 8 bits each; the largest key is `vocab` itself
  int bits = 1;
  while (bits < 32 && (vocab >> bits) != 0) ++bits;
  return (bits + 7) / 8;
}

// Sorting tiles of 1024 or 4096 keys: the larger ones need fewer counts, the smaller ones leave no compute unit idle.  The whole
// gradient into 5000 x 8 float32 with 4 and with 16 keys per thread: 100000 tokens 43 and 58 us, 600000 82 and 90, 10^6 97 and
// 100, 4 x 10^6 280 and 255.
long long emb_tiles(long long n) {
  const int tile = EMB_THREADS * (n < EMB_MANY ? 4 : 16);
  return (n + tile - 1) / tile;
}

// sorted positions per team of the reduction: short chunks for few tokens (all compute units at work; 20000 x 64 float32: 34 us in
// chunks of 32, 41 of 64), longer ones for many (fewer partial sums to join)
int emb_chunk(long long n) {
  int len = 32;
  while (len < 256 && n / len > 16384) len *= 2;
  return len;
}

// the few-rows form: lanes per row (4-byte accesses; a power of two), and the tokens of a workgroup
struct EmbFew {
  bool use;
  int words, lanes, slabs, blocks;  // words: columns per lane
  int share;
};

EmbFew emb_few_plan(long long n, long long vocab, int width, int bytes) {
  EmbFew f;
  f.words = bytes == 2 && width % 2 == 0 ? 2 : 1;
  f.use = (vocab + 1) * f.words <= EMB_FEW && n > 0;
  if (!f.use) return f;
  const int vectors = width / f.words;
  f.lanes = 1;
  while (f.lanes < 64 && f.lanes < vectors) f.lanes *= 2;
  f.slabs = (vectors + f.lanes - 1) / f.lanes;
  const long long step = (long long)(EMB_THREADS / f.lanes) * EMB_FEW_AHEAD;  // tokens of a workgroup in flight
  // as many workgroups as the 256 compute units hold at once, 160 KB of LDS each: one more would run alone behind them
  const long long fit = 256 * std::min(8LL, 160 * 1024 / ((vocab + 1) * EMB_THREADS * f.words * 4));
  const long long blocks = std::max(1LL, std::min(fit / f.slabs, n / step));
  const long long share = (n + blocks - 1) / blocks;
  f.share = (int)share;
  f.blocks = (int)((n + share - 1) / share);
  if (share * width * bytes >= (1LL << 31) || share >= (1LL << 30)) f.use = false;  // (offsets inside a workgroup's share are 32 bits)
  return f;
}

struct EmbSpace {
  uint32_t *keys[2], *pos[2], *counts, *totals, *runs;
  float* slots;
  size_t bytes;
};

EmbSpace emb_space(char* p, long long n, int width) {
  EmbSpace w;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* q = p + at;
    at += (bytes + 255) & ~(size_t)255;
    return q;
  };
  const long long tiles = emb_tiles(n), chunks = (n + emb_chunk(n) - 1) / emb_chunk(n);
  for (int i = 0; i < 2; ++i) {
    w.keys[i] = (uint32_t*)take(n * 4);
    w.pos[i] = (uint32_t*)take(n * 4);
  }
  w.counts = (uint32_t*)take(tiles * 256 * 4);
  w.totals = (uint32_t*)take(256 * 4);
  w.runs = (uint32_t*)take((1 + chunks) * 4);
  w.slots = (float*)take((size_t)chunks * 2 * width * 4);
  w.bytes = at;
  return w;
}

int emb_check(const char* what, long long tokens, long long vocab, int width, int dtype, int ids_bytes) {
  if (tokens < 0 || vocab < 1 || width < 1) return nsa_fail(NSA_E_ARG, "%s: bad size", what);
  if (tokens >= (1LL << 31) || vocab >= (1LL << 31))
    return nsa_fail(NSA_E_ARG, "%s: at most 2^31 - 1 tokens and rows", what);
  if (width > (1 << 20)) return nsa_fail(NSA_E_ARG, "%s: at most 2^20 columns", what);
  if (!nsa_elem_known(dtype)) return nsa_fail(NSA_E_ARG, "%s: unknown type %d", what, dtype);
  if (ids_bytes != 4 && ids_bytes != 8) return nsa_fail(NSA_E_ARG, "%s: ids are int32 or int64", what);
  return NSA_OK;
}

int emb_done(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? NSA_OK : nsa_fail(NSA_E_HIP, "%s: %s", what, hipGetErrorString(e));
}

template <typename T, typename ID, int V>
void emb_lookup_launch(long long tokens, long long vocab, int width, const void* ids, const void* weight, float scale,
                       void* out, hipStream_t s) {
  const int lanes = emb_lanes((width + V - 1) / V, V * (int)sizeof(T)), teams = EMB_THREADS / lanes;
  const long long groups = (tokens + teams - 1) / teams;
  hipLaunchKernelGGL((emb_lookup<T, ID, V>), dim3((unsigned)std::min(groups, 65536LL)), dim3(EMB_THREADS), 0, s, tokens,
                     vocab, width, (const ID*)ids, (const T*)weight, scale, lanes, (T*)out);
}

template <typename T, typename ID>
void emb_lookup_typed(long long tokens, long long vocab, int width, const void* ids, const void* weight, float scale,
                      void* out, hipStream_t s) {
  const int v = emb_vector(width, sizeof(T), (uintptr_t)weight | (uintptr_t)out);
  if constexpr (sizeof(T) == 2) {
    if (v == 8) return emb_lookup_launch<T, ID, 8>(tokens, vocab, width, ids, weight, scale, out, s);
  }
  if (v == 4) return emb_lookup_launch<T, ID, 4>(tokens, vocab, width, ids, weight, scale, out, s);
  if (v == 2) return emb_lookup_launch<T, ID, 2>(tokens, vocab, width, ids, weight, scale, out, s);
  emb_lookup_launch<T, ID, 1>(tokens, vocab, width, ids, weight, scale, out, s);
}

template <typename T, int V>
void emb_reduce_launch(int n, long long vocab, int width, const EmbSpace& w, int side, const void* dy, float scale,
                       void* dweight, hipStream_t s) {
  const int lanes = emb_lanes((width + V - 1) / V, V * (int)sizeof(T)), teams = EMB_THREADS / lanes, len = emb_chunk(n);
  const long long chunks = ((long long)n + len - 1) / len;
  const int slabs = (width + lanes * V - 1) / (lanes * V);
  hipLaunchKernelGGL((emb_reduce<T, V>), dim3((unsigned)((chunks + teams - 1) / teams), slabs), dim3(EMB_THREADS), 0, s, n,
                     (uint32_t)vocab, width, lanes, len, w.keys[side], w.pos[side], (const T*)dy, scale, (T*)dweight,
                     w.slots, w.runs);
  const long long borders = ((long long)n - 1) / len, items = borders * ((width + EMB_JOIN_COLS - 1) / EMB_JOIN_COLS);
  if (borders > 0)
    hipLaunchKernelGGL((emb_join<T>), dim3((unsigned)std::min(items, 2048LL)), dim3(EMB_THREADS), 0, s, n, width, len,
                       w.keys[side], scale, w.slots, w.runs, (T*)dweight);
}

template <typename T, typename ID, int W>
void emb_few_launch(const EmbFew& f, long long n, int vocab, int width, const void* ids, long long padding, const void* dy,
                    float scale, void* dweight, float* part, hipStream_t s) {
  const size_t lds = (size_t)(vocab + 1) * EMB_THREADS * W * 4;
  if (f.lanes == 64)
    hipLaunchKernelGGL((emb_few<T, ID, W, true>), dim3(f.blocks, f.slabs), dim3(EMB_THREADS), lds, s, n, vocab, width,
                       f.lanes, f.share, (const ID*)ids, padding, (const T*)dy, part);
  else
    hipLaunchKernelGGL((emb_few<T, ID, W, false>), dim3(f.blocks, f.slabs), dim3(EMB_THREADS), lds, s, n, vocab, width,
                       f.lanes, f.share, (const ID*)ids, padding, (const T*)dy, part);
  const int cells = vocab * width;
  hipLaunchKernelGGL((emb_few_join<T>), dim3((cells + EMB_SUM_CELLS - 1) / EMB_SUM_CELLS), dim3(EMB_SUM_THREADS), 0, s, cells,
                     f.blocks, part, scale, (T*)dweight);
}

struct EmbTable {  // the gradient's rows, to be cleared
  uint16_t* at;
  long long halves;
};

template <typename ID, int ITEMS>
int emb_sort(int n, long long vocab, const ID* ids, long long padding, const EmbSpace& w, const EmbTable& t, hipStream_t s) {
  const unsigned tiles = (unsigned)emb_tiles(n);
  const unsigned clear = (unsigned)std::max(1LL, std::min(t.halves / (8 * EMB_THREADS), 4096LL));
  const int passes = emb_passes(vocab);
  for (int p = 0; p < passes; ++p) {
    const uint32_t* keys = p == 0 ? nullptr : w.keys[p & 1];
    const uint32_t* pos = p == 0 ? nullptr : w.pos[p & 1];
    hipLaunchKernelGGL((emb_count<ID, ITEMS>), dim3(p == 0 ? tiles + clear : tiles), dim3(EMB_THREADS), 0, s, n, ids, vocab,
                       padding, keys, 8 * p, (int)tiles, w.counts, t.at, t.halves, w.runs);
    hipLaunchKernelGGL(emb_scan, dim3(256), dim3(EMB_THREADS), 0, s, (int)tiles, w.counts, w.totals);
    hipLaunchKernelGGL((emb_scatter<ID, ITEMS>), dim3(tiles), dim3(EMB_THREADS), 0, s, n, ids, vocab, padding, keys, pos,
                       8 * p, w.counts, w.totals, w.keys[(p + 1) & 1], w.pos[(p + 1) & 1]);
  }
  return passes & 1;
}

template <typename ID>
int emb_sort(int n, long long vocab, const void* ids, long long padding, const EmbSpace& w, const EmbTable& t,
             hipStream_t s) {
  if (n <= EMB_SHORT) {
    const long long clear = std::max(1LL, std::min(t.halves / (8 * EMB_SHORT_THREADS), 2048LL));
    hipLaunchKernelGGL((emb_sort_short<ID>), dim3((unsigned)(1 + clear)), dim3(EMB_SHORT_THREADS), 0, s, n, (const ID*)ids,
                       vocab, padding, emb_passes(vocab), w.keys[0], w.pos[0], t.at, t.halves, w.runs);
    return 0;
  }
  return n < EMB_MANY ? emb_sort<ID, 4>(n, vocab, (const ID*)ids, padding, w, t, s)
                      : emb_sort<ID, 16>(n, vocab, (const ID*)ids, padding, w, t, s);
}

template <typename T>
void emb_backward_typed(int n, long long vocab, int width, const void* ids, int ids_bytes, const void* dy, float scale,
                        long long padding, void* dweight, const EmbSpace& w, hipStream_t s) {
  const EmbFew f = emb_few_plan(n, vocab, width, sizeof(T));
  if (f.use && (uintptr_t)dy % (f.words * sizeof(T)) == 0) {
    float* part = (float*)w.keys[0];
    if (ids_bytes == 4) {
      if constexpr (sizeof(T) == 2)
        if (f.words == 2) return emb_few_launch<T, int, 2>(f, n, (int)vocab, width, ids, padding, dy, scale, dweight, part, s);
      return emb_few_launch<T, int, 1>(f, n, (int)vocab, width, ids, padding, dy, scale, dweight, part, s);
    }
    if constexpr (sizeof(T) == 2)
      if (f.words == 2) return emb_few_launch<T, long long, 2>(f, n, (int)vocab, width, ids, padding, dy, scale, dweight, part, s);
    return emb_few_launch<T, long long, 1>(f, n, (int)vocab, width, ids, padding, dy, scale, dweight, part, s);
  }
  const EmbTable t = {(uint16_t*)dweight, vocab * width * (long long)(sizeof(T) / 2)};
  if (n == 0) {  // (all rows are zero)
    hipLaunchKernelGGL(emb_zero, dim3((unsigned)std::max(1LL, std::min(t.halves / (8 * EMB_THREADS), 4096LL))),
                       dim3(EMB_THREADS), 0, s, t.at, t.halves);
    return;
  }
  const int side = ids_bytes == 4 ? emb_sort<int>(n, vocab, ids, padding, w, t, s)
                                  : emb_sort<long long>(n, vocab, ids, padding, w, t, s);
  const int v = emb_vector(width, sizeof(T), (uintptr_t)dy | (uintptr_t)dweight);
  if constexpr (sizeof(T) == 2) {
    if (v == 8) return emb_reduce_launch<T, 8>(n, vocab, width, w, side, dy, scale, dweight, s);
  }
  if (v == 4) return emb_reduce_launch<T, 4>(n, vocab, width, w, side, dy, scale, dweight, s);
  if (v == 2) return emb_reduce_launch<T, 2>(n, vocab, width, w, side, dy, scale, dweight, s);
  emb_reduce_launch<T, 1>(n, vocab, width, w, side, dy, scale, dweight, s);
}

}  // namespace

extern "C" NSA_API int nsa_embedding_forward(long long tokens, long long vocab, int width, int dtype, const void* ids_dev,
                                             int ids_bytes, const void* weight_dev, float scale, void* out_dev,
                                             void* stream) {
  if (const int rc = emb_check("nsa_embedding_forward", tokens, vocab, width, dtype, ids_bytes)) return rc;
  if (tokens == 0) return NSA_OK;
  if (!ids_dev || !weight_dev || !out_dev) return nsa_fail(NSA_E_ARG, "nsa_embedding_forward: NULL argument");
  hipStream_t s = (hipStream_t)stream;
#define EMB_LOOKUP(T)                                                                                              \
  (ids_bytes == 4 ? emb_lookup_typed<T, int>(tokens, vocab, width, ids_dev, weight_dev, scale, out_dev, s)           \
                  : emb_lookup_typed<T, long long>(tokens, vocab, width, ids_dev, weight_dev, scale, out_dev, s))
  if (dtype == NSA_DT_F32) EMB_LOOKUP(float);
  else if (dtype == NSA_DT_BF16) EMB_LOOKUP(nsa_bf16);
  else EMB_LOOKUP(nsa_f16);
#undef EMB_LOOKUP
  return emb_done("nsa_embedding_forward");
}

extern "C" NSA_API size_t nsa_embedding_workspace(long long tokens, long long vocab, int width, int dtype) {
  if (tokens <= 0 || vocab <= 0 || width <= 0 || !nsa_elem_known(dtype)) return 0;
  const EmbFew f = emb_few_plan(tokens, vocab, width, nsa_elem_bytes(dtype));
  const size_t few = f.use ? (size_t)f.blocks * vocab * width * sizeof(float) : 0;
  return std::max(few, emb_space(nullptr, tokens, width).bytes);
}

extern "C" NSA_API int nsa_embedding_backward(long long tokens, long long vocab, int width, int dtype, const void* ids_dev,
                                              int ids_bytes, const void* dy_dev, float scale, long long padding,
                                              void* dweight_dev, void* workspace_dev, size_t workspace_bytes,
                                              void* stream) {
  if (const int rc = emb_check("nsa_embedding_backward", tokens, vocab, width, dtype, ids_bytes)) return rc;
  if (!dweight_dev) return nsa_fail(NSA_E_ARG, "nsa_embedding_backward: NULL argument");
  if (tokens > 0 && (!ids_dev || !dy_dev || !workspace_dev))
    return nsa_fail(NSA_E_ARG, "nsa_embedding_backward: NULL argument");
  if (workspace_bytes < nsa_embedding_workspace(tokens, vocab, width, dtype))
    return nsa_fail(NSA_E_ARG, "nsa_embedding_backward: workspace too small");
  const EmbSpace w = emb_space((char*)workspace_dev, tokens, width);
  hipStream_t s = (hipStream_t)stream;
  const int n = (int)tokens;
  if (dtype == NSA_DT_F32) emb_backward_typed<float>(n, vocab, width, ids_dev, ids_bytes, dy_dev, scale, padding, dweight_dev, w, s);
  else if (dtype == NSA_DT_BF16) emb_backward_typed<nsa_bf16>(n, vocab, width, ids_dev, ids_bytes, dy_dev, scale, padding, dweight_dev, w, s);
  else emb_backward_typed<nsa_f16>(n, vocab, width, ids_dev, ids_bytes, dy_dev, scale, padding, dweight_dev, w, s);
  return emb_done("nsa_embedding_backward");
}
