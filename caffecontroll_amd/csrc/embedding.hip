// Embedding lookup and its gradient.
//
//   forward    out[t] = scale * table[ids[t]]
//   backward   dtable[v] = scale * sum over { t : ids[t] == v } of dout[t]
//
// The lookup moves 2 * tokens * width elements and multiplies once per element: bound by HBM, and by launch latency
// for a decoding step's few rows.  The gradient sorts the tokens by id (stable, so a row's tokens keep their order and
// the sum does not depend on timing), then every row of the table is summed by the lanes that own its columns: dout is
// read once, dtable written once, no atomics.
#include "narrow.h"

namespace cct {

constexpr int EMB_THREADS = 256;

struct EmbShape {
  int tokens, width, vocab, padding;
  float scale;
  size_t table_stride, out_stride;
  int stream;      // the result goes past the caches
  int clear_rows;  // the table is cleared row by row
};
// Results above this do not stay in the caches anyway (L2: 32 MB); written past them they leave them to the rows that are read
// (65536 tokens of 2048 bf16: 77 instead of 92 us; the gradient of 131072 rows of 4096: 3 % less).
constexpr size_t EMB_STREAM_BYTES = (size_t)32 << 20;

// ---- forward -----------------------------------------------------------------------------------------------------
// A workgroup's lanes are laid over (row, 16-byte vector of the row); the vectors of a row belong to one group of lanes (a
// power of two of at most 256), a wider row takes several trips, or several workgroups where there are few rows.  65536
// tokens of 2048 bf16: 77 us, 7.0 TB/s (ids that come again are read from a cache); 8 tokens of 4096: 4 us, a launch.
template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_forward_kernel(T *__restrict__ out, const T *__restrict__ table,
                                                                        const int *__restrict__ ids, EmbShape s,
                                                                        int log_lanes) {
  constexpr int V = Num<T>::V;
  const int lanes = 1 << log_lanes;
  const int t = blockIdx.x * (EMB_THREADS >> log_lanes) + (threadIdx.x >> log_lanes);
  if (t >= s.tokens) return;
  const int id = ids[t];
  const bool pad = id == s.padding, ok = !pad && (unsigned)id < (unsigned)s.vocab;
  const T *row = table + (size_t)(ok ? id : 0) * s.table_stride;
  T *dst = out + (size_t)t * s.out_stride;
  const float fill = pad ? 0.0f : __builtin_nanf("");
  for (int col = ((threadIdx.x & (lanes - 1)) + blockIdx.y * lanes) * V; col < s.width; col += lanes * V * gridDim.y) {
    float f[V];
    if (ok) {
      load_vec<T>(f, row, col, s.width);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= s.scale;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = fill;
    }
    if (s.stream)
      store_vec_stream<T>(dst, f, col, s.width);
    else
      store_vec<T>(dst, f, col, s.width);
  }
}

// ---- sorting the tokens by id --------------------------------------------------------------------------------------
// Keys: the id, or `vocab` (behind every valid one) for tokens that give no gradient.
__device__ __forceinline__ uint32_t sort_key(int id, int padding, int vocab) {
  return id == padding || (unsigned)id >= (unsigned)vocab ? (uint32_t)vocab : (uint32_t)id;
}

// The table cleared by workgroups of 4 KB each, in address order (6.8 TB/s; with 32 KB a workgroup 5.1 TB/s for 1 GB), whose
// stores are aligned whatever the width is; or by rows, where they have gaps between them or the table is too long for that.
constexpr size_t EMB_CLEAR_BLOCKS = (size_t)1 << 23;  // a launch has fewer than 2^32 lanes
static unsigned clear_blocks_of(EmbShape &s, int vec) {
  const size_t dense = ((size_t)s.vocab * s.width + EMB_THREADS * vec - 1) / (EMB_THREADS * vec);
  s.clear_rows = s.table_stride != (size_t)s.width || dense > EMB_CLEAR_BLOCKS;
  return (unsigned)(s.clear_rows ? min((size_t)s.vocab, EMB_CLEAR_BLOCKS) : dense);
}
template <class T>
__device__ __forceinline__ void clear_block(T *__restrict__ dtable, const EmbShape &s, uint32_t block, uint32_t blocks) {
  constexpr int V = Num<T>::V;
  float zero[V];
#pragma unroll
  for (int i = 0; i < V; ++i) zero[i] = 0.0f;
  const auto clear = [&](T *at, int left) {
    if (s.stream)
      store_vec_stream<T>(at, zero, 0, left);
    else
      store_vec<T>(at, zero, 0, left);
  };
  if (!s.clear_rows) {
    const size_t at = ((size_t)block * EMB_THREADS + threadIdx.x) * V, end = (size_t)s.vocab * s.width;
    if (at < end) clear(dtable + at, (int)min(end - at, (size_t)V));
    return;
  }
  for (uint32_t v = block; v < (uint32_t)s.vocab; v += blocks)
    for (int col = threadIdx.x * V; col < s.width; col += EMB_THREADS * V)
      clear(dtable + (size_t)v * s.table_stride + col, s.width - col);
}

// Few tokens: a token's place is the number of tokens that come before it, counted directly.  All keys lie in LDS; 16 lanes
// share a token and take four keys at a time.  Of a workgroup's 16 tokens, those before the first of them come earlier
// with an equal key too, those behind the last one do not, so but for one stretch of 16 every key costs one comparison.
// tokens^2 comparisons over the whole chip in one launch: 5 us at 4096 tokens.
constexpr int EMB_RANK_MAX = 8192;
constexpr int EMB_RANK_LANES = 16;
constexpr int EMB_RANK_TOKENS = EMB_THREADS / EMB_RANK_LANES;
// Workgroups behind those that rank clear the table: the two have nothing to do with one another.
template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_rank_kernel(uint32_t *__restrict__ keys, int *__restrict__ order,
                                                                     const int *__restrict__ ids, T *__restrict__ dtable,
                                                                     EmbShape s, int rank_blocks) {
  extern __shared__ __align__(16) uint32_t all[];
  if ((int)blockIdx.x >= rank_blocks) return clear_block<T>(dtable, s, blockIdx.x - rank_blocks, gridDim.x - rank_blocks);
  const int tokens = s.tokens, padding = s.padding, vocab = s.vocab;
  const int lane = threadIdx.x % EMB_RANK_LANES, t0 = blockIdx.x * EMB_RANK_TOKENS;
  const int t = t0 + threadIdx.x / EMB_RANK_LANES;
  const int pad = (tokens + 63) & ~63;
  typedef int i4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
#pragma unroll 4
  for (int i = threadIdx.x * 4; i < pad; i += EMB_THREADS * 4) {
    i4 v = {0, 0, 0, 0};
    if (i + 4 <= tokens) {
      v = *reinterpret_cast<const i4 *>(ids + i);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < tokens) v[k] = ids[i + k];
    }
    u4 u;
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = i + k < tokens ? sort_key(v[k], padding, vocab) : 0xFFFFFFFFu;  // behind every key
    *reinterpret_cast<u4 *>(all + i) = u;
  }
  __syncthreads();
  const uint32_t key = t < tokens ? all[t] : 0u;
  int before = 0;
  auto count = [&](int from, int to, uint32_t below) {
#pragma unroll 4
    for (int i = from + lane * 4; i < to; i += EMB_RANK_LANES * 4) {
      const u4 k = *reinterpret_cast<const u4 *>(all + i);
      before += (k[0] < below) + (k[1] < below) + (k[2] < below) + (k[3] < below);
    }
  };
  count(0, t0, key + 1);                          // (t0 is a multiple of 16, vocab + 1 does not overflow)
  if (t0 + lane < tokens) {
    const uint32_t k = all[t0 + lane];
    before += k < key || (k == key && t0 + lane < t);
  }
  count(t0 + EMB_RANK_TOKENS, pad, key);
#pragma unroll
  for (int m = EMB_RANK_LANES / 2; m > 0; m >>= 1) before += __shfl_xor(before, m, 64);
  if (lane == 0 && t < tokens) {
    keys[before] = key;
    order[before] = t;
  }
}

// Many tokens: least-significant-digit radix sort, 9 bits a pass.  One workgroup per tile of 1024 tokens counts its
// digits; the second launch of a pass turns the tiles' counts into places (digits ascending, tiles ascending within a
// digit) and moves the tile in order, so every pass is stable.  Above EMB_TILES_MAX tiles a launch between them adds up the
// tiles' counts once, instead of every workgroup for itself.
constexpr int EMB_BITS = 9, EMB_BINS = 1 << EMB_BITS;
constexpr int EMB_ITEMS = 4, EMB_TILE = EMB_THREADS * EMB_ITEMS;
constexpr uint32_t EMB_TILES_MAX = 128;
constexpr int EMB_WAVES = EMB_THREADS / 64;

// The token (and its key) at a place of a pass's input: the first pass reads the ids themselves.
__device__ __forceinline__ uint32_t pass_key(const uint32_t *__restrict__ keys, const int *__restrict__ ids, int i,
                                             int padding, int vocab) {
  return keys ? keys[i] : sort_key(ids[i], padding, vocab);
}

// Workgroups behind the tiles' clear the table.
template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_count_kernel(uint32_t *__restrict__ counts,
                                                                      const uint32_t *__restrict__ keys,
                                                                      const int *__restrict__ ids, T *__restrict__ dtable,
                                                                      EmbShape s, int shift, int tiles) {
  __shared__ uint32_t bins[EMB_BINS];
  if ((int)blockIdx.x >= tiles) return clear_block<T>(dtable, s, blockIdx.x - tiles, gridDim.x - tiles);
  const int tokens = s.tokens, padding = s.padding, vocab = s.vocab;
  for (int i = threadIdx.x; i < EMB_BINS; i += EMB_THREADS) bins[i] = 0;
  __syncthreads();
  for (int i = 0; i < EMB_ITEMS; ++i) {
    const int at = blockIdx.x * EMB_TILE + i * EMB_THREADS + threadIdx.x;
    if (at < tokens) atomicAdd(&bins[(pass_key(keys, ids, at, padding, vocab) >> shift) & (EMB_BINS - 1)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < EMB_BINS; i += EMB_THREADS) counts[(size_t)blockIdx.x * EMB_BINS + i] = bins[i];
}

// counts[tile] becomes the sum over the tiles before it, and a row behind the last tile holds all of them.
__global__ __launch_bounds__(EMB_BINS) void embedding_scan_kernel(uint32_t *__restrict__ counts, uint32_t tiles) {
  uint32_t sum = 0, tile = 0;
  for (; tile + 8 <= tiles; tile += 8) {
    uint32_t c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) c[k] = counts[(size_t)(tile + k) * EMB_BINS + threadIdx.x];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      counts[(size_t)(tile + k) * EMB_BINS + threadIdx.x] = sum;
      sum += c[k];
    }
  }
  for (; tile < tiles; ++tile) {
    const uint32_t c = counts[(size_t)tile * EMB_BINS + threadIdx.x];
    counts[(size_t)tile * EMB_BINS + threadIdx.x] = sum;
    sum += c;
  }
  counts[(size_t)tiles * EMB_BINS + threadIdx.x] = sum;
}

__global__ __launch_bounds__(EMB_THREADS) void embedding_move_kernel(uint32_t *__restrict__ keys_out,
                                                                     int *__restrict__ order_out,
                                                                     const uint32_t *__restrict__ keys,
                                                                     const int *__restrict__ order,
                                                                     const int *__restrict__ ids,
                                                                     const uint32_t *__restrict__ counts, int tokens,
                                                                     int padding, int vocab, int shift) {
  __shared__ uint32_t place[EMB_BINS];               // where this tile's first token of a digit goes
  __shared__ uint32_t seen[EMB_WAVES][EMB_BINS];     // tokens of a digit in a wavefront's part so far
  __shared__ uint32_t scan[EMB_THREADS];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  // per digit: tokens in all tiles, and in the tiles before this one
  constexpr int PER = EMB_BINS / EMB_THREADS;
  uint32_t all[PER], before[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) all[j] = before[j] = 0;
  if (gridDim.x > EMB_TILES_MAX) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      before[j] = counts[(size_t)blockIdx.x * EMB_BINS + tid * PER + j];
      all[j] = counts[(size_t)gridDim.x * EMB_BINS + tid * PER + j];
    }
  } else {
#pragma unroll 16
    for (uint32_t tile = 0; tile < gridDim.x; ++tile) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const uint32_t c = counts[(size_t)tile * EMB_BINS + tid * PER + j];
        all[j] += c;
        before[j] += tile < blockIdx.x ? c : 0u;
      }
    }
  }
  uint32_t mine = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) mine += all[j];
  scan[tid] = mine;
  __syncthreads();
  for (int d = 1; d < EMB_THREADS; d <<= 1) {
    const uint32_t v = tid >= d ? scan[tid - d] : 0u;
    __syncthreads();
    scan[tid] += v;
    __syncthreads();
  }
  uint32_t at = scan[tid] - mine;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    place[tid * PER + j] = at + before[j];
    at += all[j];
  }
  for (int i = tid; i < EMB_WAVES * EMB_BINS; i += EMB_THREADS) (&seen[0][0])[i] = 0;
  __syncthreads();
  // wavefront w takes the tile's tokens [w * 256, ...) 64 at a time, in order: a token's rank within its wavefront's
  // part is the count of its digit so far plus the lanes of the same digit below it
  uint32_t key[EMB_ITEMS], rank[EMB_ITEMS];
  const int first = blockIdx.x * EMB_TILE + wave * (EMB_ITEMS * 64) + lane;
#pragma unroll
  for (int i = 0; i < EMB_ITEMS; ++i) {
    const int p = first + i * 64;
    const bool have = p < tokens;
    key[i] = have ? pass_key(keys, ids, p, padding, vocab) : 0u;
    const uint32_t digit = (key[i] >> shift) & (EMB_BINS - 1);
    uint64_t same = __ballot(have);
#pragma unroll
    for (int b = 0; b < EMB_BITS; ++b) {
      const bool bit = (digit >> b) & 1u;
      const uint64_t ones = __ballot(bit);
      same &= bit ? ones : ~ones;
    }
    const uint32_t below = __popcll(same & ((1ull << lane) - 1ull));
    const uint32_t so_far = seen[wave][digit];
    rank[i] = so_far + below;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // every lane has read before the first of its digit adds
    if (have && below == 0) seen[wave][digit] = so_far + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  for (int d = tid; d < EMB_BINS; d += EMB_THREADS) {
    uint32_t base = place[d];
#pragma unroll
    for (int w = 0; w < EMB_WAVES; ++w) {
      const uint32_t c = seen[w][d];
      seen[w][d] = base;
      base += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EMB_ITEMS; ++i) {
    const int p = first + i * 64;
    if (p < tokens) {
      const uint32_t to = seen[wave][(key[i] >> shift) & (EMB_BINS - 1)] + rank[i];
      keys_out[to] = key[i];
      order_out[to] = order ? order[p] : p;
    }
  }
}

// ---- summing the rows ----------------------------------------------------------------------------------------------
// First place in the sorted keys whose key is not below `key`.
__device__ __forceinline__ int lower_bound(const uint32_t *__restrict__ keys, int n, uint32_t key) {
  int lo = 0, len = n;
  while (len > 0) {
    const int half = len >> 1;
    const bool below = keys[lo + half] < key;
    lo = below ? lo + half + 1 : lo;
    len = below ? len - half - 1 : half;
  }
  return lo;
}

// The same by a whole wavefront, 64 places at a time.
__device__ __forceinline__ int wave_lower_bound(const uint32_t *__restrict__ keys, int n, uint32_t key, int lane) {
  int lo = 0, len = n;
  while (len > 0) {
    const int step = (len + 63) >> 6;
    const int at = lane * step;
    const int below = __popcll(__ballot(at < len && keys[lo + min(at, len - 1)] < key));
    if (below == 0) return lo;
    const int skip = (below - 1) * step + 1;
    len = min(step - 1, len - skip);
    lo += skip;
  }
  return lo;
}

// Sums of dout[order[p]] over the places [p0, p1): TRIPS vectors of a row at columns col, col + stride, ...
template <class T, int TRIPS>
__device__ __forceinline__ void sum_rows(float (&acc)[TRIPS][Num<T>::V], const T *__restrict__ dout,
                                         const int *__restrict__ order, int p0, int p1, int col, int stride,
                                         const EmbShape &s) {
  constexpr int V = Num<T>::V;
#pragma unroll
  for (int k = 0; k < TRIPS; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[k][i] = 0.0f;
  int p = p0;
  for (; p + 4 <= p1; p += 4) {  // four rows in flight, added in order
    float f[4][TRIPS][V];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const T *row = dout + (size_t)order[p + j] * s.out_stride;
#pragma unroll
      for (int k = 0; k < TRIPS; ++k) load_vec<T>(f[j][k], row, col + k * stride, s.width);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < TRIPS; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[k][i] += f[j][k][i];
  }
  for (; p < p1; ++p) {
    const T *row = dout + (size_t)order[p] * s.out_stride;
    float f[TRIPS][V];
#pragma unroll
    for (int k = 0; k < TRIPS; ++k) load_vec<T>(f[k], row, col + k * stride, s.width);
#pragma unroll
    for (int k = 0; k < TRIPS; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[k][i] += f[k][i];
  }
}

template <class T>
__device__ __forceinline__ void store_row(T *__restrict__ row, float (&acc)[Num<T>::V], int col, const EmbShape &s,
                                          int accumulate) {
  constexpr int V = Num<T>::V;
  float old[V];
  if (accumulate) load_vec<T>(old, row, col, s.width);
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = accumulate ? old[i] + acc[i] * s.scale : acc[i] * s.scale;
  if (s.stream)
    store_vec_stream<T>(row, acc, col, s.width);
  else
    store_vec<T>(row, acc, col, s.width);
}

// An id with more than EMB_RUN tokens is summed in pieces of EMB_RUN sorted places.  Piece j covers places
// [j * EMB_RUN, (j + 1) * EMB_RUN) and can hold parts of two such ids: slot 0 the one that holds its first place, slot 1
// one that begins inside.  Ids with fewer tokens are summed whole by the workgroup that owns their row.
constexpr int EMB_RUN = 16;
constexpr int EMB_ROWS = 8;  // rows of the table per workgroup, at least
constexpr int EMB_PLACES = EMB_ROWS * EMB_RUN;  // tokens of a workgroup's rows that it holds in LDS
// what the joining launch needs to know of the long id that begins in a piece; first == last: there is none
struct EmbRun {
  int first, last;  // its places
  int id;
};

// Piece `piece` of the ids that are summed in pieces, by a workgroup; bounds: four words of LDS.
template <class T>
__device__ __forceinline__ void sum_piece(float *__restrict__ parts, EmbRun *__restrict__ runs, const T *__restrict__ dout,
                                          const uint32_t *__restrict__ keys, const int *__restrict__ order, int piece,
                                          int *bounds, const EmbShape &s) {
  constexpr int V = Num<T>::V;
  const int tid = threadIdx.x, a = piece * EMB_RUN, b = min(a + EMB_RUN, s.tokens);
  // wavefronts 0 and 1: the id at the piece's first place; 2 and 3: the one at its last
  const uint32_t key = keys[tid < 128 ? a : b - 1];
  const int at = wave_lower_bound(keys, s.tokens, key + ((tid >> 6) & 1), tid & 63);
  if ((tid & 63) == 0) bounds[tid >> 6] = at;
  __syncthreads();
  if (tid == 128) {
    const bool begins = key < (uint32_t)s.vocab && bounds[3] - bounds[2] > EMB_RUN && bounds[2] >= a;
    runs[piece] = begins ? EmbRun{bounds[2], bounds[3], (int)key} : EmbRun{0, 0, 0};
  }
  for (int slot = 0; slot < 2; ++slot) {
    const int r0 = bounds[2 * slot], r1 = bounds[2 * slot + 1];
    if (r1 - r0 <= EMB_RUN || keys[r0] >= (uint32_t)s.vocab || (slot == 1 && r0 <= a)) continue;
    const int p0 = max(r0, a), p1 = min(r1, b);
    float *dst = parts + ((size_t)piece * 2 + slot) * s.width;
    for (int col = tid * V; col < s.width; col += EMB_THREADS * V) {
      float acc[1][V];
      sum_rows<T, 1>(acc, dout, order, p0, p1, col, 0, s);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (col + i < s.width) dst[col + i] = acc[0][i];
    }
  }
}

template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_sum_kernel(T *__restrict__ dtable, float *__restrict__ parts,
                                                                    EmbRun *__restrict__ runs,
                                                                    const T *__restrict__ dout,
                                                                    const uint32_t *__restrict__ keys,
                                                                    const int *__restrict__ order, EmbShape s,
                                                                    int accumulate, int log_lanes, int pieces) {
  constexpr int V = Num<T>::V;
  __shared__ int bounds[EMB_THREADS + 1];
  __shared__ int window[2];
  __shared__ int places[EMB_PLACES];
  const int tid = threadIdx.x, lanes = 1 << log_lanes, lane = tid & (lanes - 1), group = tid >> log_lanes;
  const int groups = EMB_THREADS >> log_lanes;
  if ((int)blockIdx.x >= pieces) {
    const int rows = max(EMB_ROWS, groups);
    const int v0 = ((int)blockIdx.x - pieces) * rows, n = min(rows, s.vocab - v0);
    if (tid < 128) {
      const int at = wave_lower_bound(keys, s.tokens, (uint32_t)(v0 + (tid < 64 ? 0 : n)), tid & 63);
      if ((tid & 63) == 0) window[tid >> 6] = at;
    }
    __syncthreads();
    const int lo = window[0], len = window[1] - lo;
    for (int i = tid; i < min(len, EMB_PLACES); i += EMB_THREADS) places[i] = order[lo + i];
    for (int i = tid; i <= n; i += EMB_THREADS) bounds[i] = lo + lower_bound(keys + lo, len, (uint32_t)(v0 + i));
    __syncthreads();
    for (int r = group; r < n; r += groups) {
      const int p0 = bounds[r], p1 = bounds[r + 1];
      if (p1 - p0 > EMB_RUN || (accumulate && p1 == p0)) continue;
      T *row = dtable + (size_t)(v0 + r) * s.table_stride;
      // (a workgroup with a long id among its rows may have places beyond those in LDS)
      const bool held = p1 - lo <= EMB_PLACES;
      const int stride = lanes * V;
      for (int col = lane * V; col < s.width; col += 2 * stride) {
        float acc[2][V];
        if (held)
          sum_rows<T, 2>(acc, dout, places, p0 - lo, p1 - lo, col, stride, s);
        else
          sum_rows<T, 2>(acc, dout, order, p0, p1, col, stride, s);
        store_row<T>(row, acc[0], col, s, accumulate);
        store_row<T>(row, acc[1], col + stride, s, accumulate);
      }
    }
    return;
  }
  sum_piece<T>(parts, runs, dout, keys, order, blockIdx.x, bounds, s);
}

// The same from the tokens' side, for a table whose other rows have been cleared beside the sort: a group of lanes takes
// EMB_RUN_PLACES sorted places and sums the ids that begin there.  No row is looked up, and rows without tokens cost this
// launch nothing (4099 tokens, 10007 rows of 1001 fp32: 34 us with the kernel above in its place).
constexpr int EMB_RUN_PLACES = 2;
template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_runs_kernel(T *__restrict__ dtable, float *__restrict__ parts,
                                                                     EmbRun *__restrict__ runs,
                                                                     const T *__restrict__ dout,
                                                                     const uint32_t *__restrict__ keys,
                                                                     const int *__restrict__ order, EmbShape s,
                                                                     int accumulate, int log_lanes, int pieces) {
  constexpr int V = Num<T>::V;
  constexpr int MOST = EMB_THREADS * EMB_RUN_PLACES + EMB_RUN + 1;
  __shared__ uint32_t key_sh[MOST + 1];  // [0]: the place before the first
  __shared__ int place_sh[MOST];
  if ((int)blockIdx.x < pieces) return sum_piece<T>(parts, runs, dout, keys, order, blockIdx.x, place_sh, s);
  const int tid = threadIdx.x, lanes = 1 << log_lanes, lane = tid & (lanes - 1), group = tid >> log_lanes;
  const int places = (EMB_THREADS >> log_lanes) * EMB_RUN_PLACES, first = ((int)blockIdx.x - pieces) * places;
  for (int i = tid; i <= places + EMB_RUN; i += EMB_THREADS) {
    const int p = first + i;
    key_sh[i + 1] = p < s.tokens ? keys[p] : 0xFFFFFFFFu;
    place_sh[i] = p < s.tokens ? order[p] : 0;
  }
  if (tid == 0) key_sh[0] = first > 0 ? keys[first - 1] : 0xFFFFFFFFu;
  __syncthreads();
  for (int q = 0; q < EMB_RUN_PLACES; ++q) {
    const int at = group * EMB_RUN_PLACES + q;
    const uint32_t key = key_sh[at + 1];
    if (key >= (uint32_t)s.vocab || key_sh[at] == key) continue;  // (what lies past the tokens is above every id)
    int length = 1;
    while (length <= EMB_RUN && key_sh[at + 1 + length] == key) ++length;
    if (length > EMB_RUN) continue;  // in pieces
    for (int col = lane * V; col < s.width; col += lanes * V) {
      float acc[1][V];
      sum_rows<T, 1>(acc, dout, place_sh, at, at + length, col, 0, s);
      store_row<T>(dtable + (size_t)key * s.table_stride, acc[0], col, s, accumulate);
    }
  }
}

// The pieces of a long id, added in order: workgroups of the EMB_JOIN pieces among which it begins, 256 columns each, their
// four wavefronts taking every fourth piece.  (One workgroup per piece and 256 columns are mostly workgroups that find
// nothing: 36 us for 65536 tokens of width 4096.)
constexpr int EMB_JOIN = 16;
constexpr int EMB_JOIN_WAVES = 4;
template <class T>
__global__ __launch_bounds__(EMB_JOIN_WAVES * 64) void embedding_join_kernel(T *__restrict__ dtable,
                                                                     const float *__restrict__ parts,
                                                                     const EmbRun *__restrict__ runs, EmbShape s,
                                                                     int accumulate, int pieces) {
  __shared__ f32x4 sums[EMB_JOIN_WAVES][64];
  const int tid = threadIdx.x, lane = tid & 63, group = tid >> 6;
  const int first = blockIdx.x * EMB_JOIN, slot = first + (lane & (EMB_JOIN - 1));
  const EmbRun mine = slot < pieces ? runs[slot] : EmbRun{0, 0, 0};  // all of them with one load
  uint64_t found = __ballot(lane < EMB_JOIN && mine.first != mine.last);
  while (found) {
    const int which = __builtin_ctzll(found), piece = first + which;
    found &= found - 1;
    const EmbRun run{__shfl(mine.first, which, 64), __shfl(mine.last, which, 64), __shfl(mine.id, which, 64)};
    const int end = (run.last - 1) / EMB_RUN;
    for (int c0 = blockIdx.y * 256; c0 < s.width; c0 += gridDim.y * 256) {
      const int col = c0 + lane * 4;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      auto add = [&](int j) {
        float f[4];
        load_vec<float>(f, parts + (size_t)(j * 2 + (j == piece && run.first != piece * EMB_RUN)) * s.width, col, s.width);
        acc += f32x4{f[0], f[1], f[2], f[3]};
      };
      int j = piece + group;
      if (j <= end) add(j);
      j += EMB_JOIN_WAVES;
      if (col + 4 <= s.width)
        for (; j + 7 * EMB_JOIN_WAVES <= end; j += 8 * EMB_JOIN_WAVES) {  // eight loads in flight, added in order
          Num<float>::vec v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            v[k] = *reinterpret_cast<const Num<float>::vec *>(parts + (size_t)(j + EMB_JOIN_WAVES * k) * 2 * s.width + col);
#pragma unroll
          for (int k = 0; k < 8; ++k) acc += f32x4{v[k][0], v[k][1], v[k][2], v[k][3]};
        }
      for (; j <= end; j += EMB_JOIN_WAVES) add(j);
      __syncthreads();
      if (group > 0) sums[group][lane] = acc;
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int w = 1; w < EMB_JOIN_WAVES; ++w) acc += sums[w][lane];
        T *dst = dtable + (size_t)run.id * s.table_stride + col;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < s.width) dst[i] = (T)(accumulate ? (float)dst[i] + acc[i] * s.scale : acc[i] * s.scale);
      }
    }
  }
}

// Few tokens: one launch without a sort (16 tokens, 10007 rows of 1024 fp32: 8 us, 7 us of them clearing 41 MB; 12 us with
// the ranking).  Every workgroup reads all ids, keeps those of its rows with their tokens in order,
// and adds each row's up.  (A row that has all of them is a chain of tokens / 4 loads: 32 at most.)
constexpr int EMB_FEW = 128;
template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_few_kernel(T *__restrict__ dtable, const T *__restrict__ dout,
                                                                    const int *__restrict__ ids, EmbShape s,
                                                                    int accumulate, int log_lanes, int rows) {
  constexpr int V = Num<T>::V;
  __shared__ int token[EMB_FEW], row_of[EMB_FEW], held;
  const int tid = threadIdx.x, lanes = 1 << log_lanes, lane = tid & (lanes - 1), group = tid >> log_lanes;
  const int groups = EMB_THREADS >> log_lanes;
  const int v0 = blockIdx.x * rows, n = min(rows, s.vocab - v0);
  if (tid < 64) {
    int count = 0;
    for (int base = 0; base < s.tokens; base += 64) {
      const int t = base + tid;
      const uint32_t key = t < s.tokens ? sort_key(ids[t], s.padding, s.vocab) : (uint32_t)s.vocab;
      const bool here = key >= (uint32_t)v0 && key < (uint32_t)(v0 + n);
      const uint64_t all = __ballot(here);
      if (here) {
        const int at = count + __popcll(all & ((1ull << tid) - 1ull));
        token[at] = t;
        row_of[at] = (int)key - v0;
      }
      count += __popcll(all);
    }
    if (tid == 0) held = count;
  }
  __syncthreads();
  const int count = held;
  for (int r = group; r < n; r += groups) {
    int mine = 0;
    for (int i = 0; i < count; ++i) mine += row_of[i] == r;
    if (accumulate && mine == 0) continue;
    T *row = dtable + (size_t)(v0 + r) * s.table_stride;
    for (int col = lane * V; col < s.width; col += lanes * V) {
      float acc[V];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.0f;
      int next = 0;
      for (int left = mine; left > 0; left -= 4) {  // four rows in flight, added in order
        float f[4][V];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= left) break;
          while (row_of[next] != r) ++next;
          load_vec<T>(f[j], dout + (size_t)token[next++] * s.out_stride, col, s.width);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] += j < left ? f[j][i] : 0.0f;
      }
      store_row<T>(row, acc, col, s, accumulate);
    }
  }
}

// Lanes that share a row: as many as it has 16-byte vectors, up to 2^most.
template <class T>
static int row_lanes_log2(int width, int most) {
  const int vecs = (width + Num<T>::V - 1) / Num<T>::V;
  int l = 0;
  while ((1 << l) < vecs && l < most) ++l;
  return l;
}

static int check_embedding(const cct_embedding_args *a, const char *who) {
  CCT_REQUIRE(a != nullptr, "%s: null argument block", who);
  CCT_REQUIRE(a->dtype == CCT_F32 || a->dtype == CCT_BF16, "%s: dtype %d is neither CCT_F32 nor CCT_BF16", who, a->dtype);
  CCT_REQUIRE(a->tokens >= 0 && a->width > 0 && a->vocab > 0, "%s: tokens %d, width %d, vocab %d", who, a->tokens,
              a->width, a->vocab);
  // a launch has fewer than 2^32 lanes and 2^16 workgroups along y
  CCT_REQUIRE(a->width <= (1 << 20) && a->tokens <= (1 << 23) && a->vocab <= (1 << 26),
              "%s: tokens %d, width %d, vocab %d: at most 2^23, 2^20, 2^26", who, a->tokens, a->width, a->vocab);
  CCT_REQUIRE((a->table_stride == 0 || a->table_stride >= (size_t)a->width) &&
                  (a->out_stride == 0 || a->out_stride >= (size_t)a->width),
              "%s: a row stride is smaller than the width %d", who, a->width);
  return 0;
}

static EmbShape shape_of(const cct_embedding_args *a, int result_rows) {
  const bool stream = (size_t)result_rows * a->width * dtype_bytes(a->dtype) > EMB_STREAM_BYTES;
  return EmbShape{a->tokens, a->width, a->vocab, a->padding_id, a->scale,
                  a->table_stride ? a->table_stride : (size_t)a->width, a->out_stride ? a->out_stride : (size_t)a->width,
                  stream ? 1 : 0, 0};
}

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// keys and order (twice: the radix passes alternate), the tiles' digit counts, the pieces' sums
struct EmbWorkspace {
  size_t keys[2], order[2], counts, parts, runs, total;
};
static EmbWorkspace embedding_layout(const cct_embedding_args *a) {
  EmbWorkspace w;
  // (none of it is used for EMB_FEW tokens or fewer)
  const size_t n = a->tokens > EMB_FEW ? a->tokens : 0, tiles = (n + EMB_TILE - 1) / EMB_TILE;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  const bool radix = a->tokens > EMB_RANK_MAX;
  for (int i = 0; i < 2; ++i) {
    w.keys[i] = take(i == 0 || radix ? n * 4 : 0);
    w.order[i] = take(i == 0 || radix ? n * 4 : 0);
  }
  w.counts = take(radix ? (tiles + 1) * EMB_BINS * 4 : 0);
  w.parts = take((n + EMB_RUN - 1) / EMB_RUN * 2 * a->width * sizeof(float));
  w.runs = take((n + EMB_RUN - 1) / EMB_RUN * sizeof(EmbRun));
  w.total = at;
  return w;
}

template <class T>
static int embedding_forward(void *out, const void *table, const int *ids, const EmbShape &s) {
  const int l = row_lanes_log2<T>(s.width, 8);
  const int per = EMB_THREADS >> l;
  const unsigned blocks = (s.tokens + per - 1) / per;
  // one trip over a row per workgroup where few rows would leave the chip empty
  const unsigned trips = (s.width + Num<T>::V * (1 << l) - 1) / (Num<T>::V * (1 << l));
  const unsigned cols = blocks >= 2048u ? 1u : min(trips, 64u);
  embedding_forward_kernel<T><<<dim3(blocks, cols), EMB_THREADS, 0, ctx().stream>>>((T *)out, (const T *)table, ids, s, l);
  CCT_LAUNCH_CHECK();
  note_kernel("embedding_forward_kernel<%s> rows per workgroup=%d", Num<T>::NAME, per);
  return 0;
}

template <class T>
static int sort_tokens(char *ws, const EmbWorkspace &w, const int *ids, const EmbShape &s, T *dtable, unsigned clear_blocks,
                       uint32_t **keys, int **order) {
  hipStream_t st = ctx().stream;
  uint32_t *k[2] = {(uint32_t *)(ws + w.keys[0]), (uint32_t *)(ws + w.keys[1])};
  int *o[2] = {(int *)(ws + w.order[0]), (int *)(ws + w.order[1])};
  const unsigned tiles = (s.tokens + EMB_TILE - 1) / EMB_TILE;
  uint32_t *counts = (uint32_t *)(ws + w.counts);
  int from = -1;  // the first pass reads the ids
  for (int shift = 0; shift < 32 && ((uint32_t)s.vocab >> shift) != 0; shift += EMB_BITS) {
    const int to = from == 0 ? 1 : 0;
    const uint32_t *kin = from < 0 ? nullptr : k[from];
    const int *oin = from < 0 ? nullptr : o[from];
    // the table is cleared beside the first pass's count
    embedding_count_kernel<T><<<tiles + (from < 0 ? clear_blocks : 0u), EMB_THREADS, 0, st>>>(
        counts, kin, ids, dtable, s, shift, (int)tiles);
    CCT_LAUNCH_CHECK();
    if (tiles > EMB_TILES_MAX) {
      embedding_scan_kernel<<<1, EMB_BINS, 0, st>>>(counts, tiles);
      CCT_LAUNCH_CHECK();
    }
    embedding_move_kernel<<<tiles, EMB_THREADS, 0, st>>>(k[to], o[to], kin, oin, ids, counts, s.tokens, s.padding, s.vocab,
                                                         shift);
    CCT_LAUNCH_CHECK();
    from = to;
  }
  *keys = k[from];
  *order = o[from];
  return 0;
}

template <class T>
static int embedding_backward(void *dtable, const void *dout, const int *ids, EmbShape s, int accumulate, char *ws,
                              const EmbWorkspace &w) {
  hipStream_t st = ctx().stream;
  const int l = row_lanes_log2<T>(s.width, 8), rows = max(EMB_ROWS, EMB_THREADS >> l);
  const int row_blocks = (s.vocab + rows - 1) / rows;
  if (s.tokens <= EMB_FEW) {
    embedding_few_kernel<T><<<row_blocks, EMB_THREADS, 0, st>>>((T *)dtable, (const T *)dout, ids, s, accumulate, l, rows);
    CCT_LAUNCH_CHECK();
    note_kernel("embedding_few_kernel<%s> rows per workgroup=%d", Num<T>::NAME, rows);
    return 0;
  }
  const int pieces = (s.tokens + EMB_RUN - 1) / EMB_RUN;
  float *parts = (float *)(ws + w.parts);
  EmbRun *runs = (EmbRun *)(ws + w.runs);
  const bool ranked = s.tokens <= EMB_RANK_MAX;
  // Visiting only the rows with tokens writes those twice; looking every row's tokens up costs a search a row.  Rows of less
  // than 4 KB: the search is the larger (131072 rows of 1024 bf16, 16384 to 524288 tokens as text has them: 81 to 525 us visited,
  // 121 to 687 looked up; all different or uniform 74 to 452, 114 to 565; rows of 512 bytes to 2 KB alike, by up to 1.8; one of 34
  // sizes 4 % the other way).  Longer rows: by how many have tokens, which only the ids say.  131072 rows of 4096 bf16,
  // tokens as text has them: 225, 273, 373 (0.15 of the rows), 546 us (0.25) visited for 16384, 32768, 65536, 131072 tokens, 250,
  // 311, 420, 589 looked up; all different: 225, 268, 402, 604 and 237, 228, 368, 493.  fp32, 16384 rows of 4096, as many
  // tokens: 128 and 138, all different 145 and 113.  From more tokens than half the rows they are looked up.
  const bool visit = ranked || s.width * sizeof(T) < 4096 || s.tokens <= s.vocab / 2;
  const unsigned clear_blocks = accumulate || !visit ? 0u : clear_blocks_of(s, Num<T>::V);
  uint32_t *keys = (uint32_t *)(ws + w.keys[0]);
  int *order = (int *)(ws + w.order[0]);
  if (ranked) {
    const int rank_blocks = (s.tokens + EMB_RANK_TOKENS - 1) / EMB_RANK_TOKENS;
    const size_t lds = ((size_t)s.tokens + 63) / 64 * 64 * sizeof(uint32_t);
    embedding_rank_kernel<T><<<rank_blocks + clear_blocks, EMB_THREADS, lds, st>>>(keys, order, ids, (T *)dtable, s,
                                                                                  rank_blocks);
    CCT_LAUNCH_CHECK();
  } else if (int rc = sort_tokens<T>(ws, w, ids, s, (T *)dtable, clear_blocks, &keys, &order)) {
    return rc;
  }
  if (visit) {
    const int places = (EMB_THREADS >> l) * EMB_RUN_PLACES, blocks = (s.tokens + places - 1) / places;
    embedding_runs_kernel<T><<<pieces + blocks, EMB_THREADS, 0, st>>>((T *)dtable, parts, runs, (const T *)dout, keys, order,
                                                                     s, accumulate, l, pieces);
    CCT_LAUNCH_CHECK();
    note_kernel("embedding_runs_kernel<%s> pieces=%d", Num<T>::NAME, pieces);
  } else {
    // the pieces first: they take the longest
    embedding_sum_kernel<T><<<pieces + row_blocks, EMB_THREADS, 0, st>>>((T *)dtable, parts, runs, (const T *)dout, keys, order,
                                                                        s, accumulate, l, pieces);
    CCT_LAUNCH_CHECK();
    note_kernel("embedding_sum_kernel<%s> rows per workgroup=%d pieces=%d", Num<T>::NAME, rows, pieces);
  }
  {
    const int cols = min((s.width + 255) / 256, 64);
    const dim3 grid((pieces + EMB_JOIN - 1) / EMB_JOIN, cols);
    embedding_join_kernel<T><<<grid, EMB_JOIN_WAVES * 64, 0, st>>>((T *)dtable, parts, runs, s, accumulate, pieces);
    CCT_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace cct

using namespace cct;

extern "C" int cct_hip_embedding_forward(void *out, const void *table, const int *ids, const cct_embedding_args *args) {
  if (int rc = check_embedding(args, "embedding_forward")) return rc;
  if (args->tokens == 0) return 0;
  CCT_REQUIRE(out && table && ids, "embedding_forward: null array");
  CCT_ENSURE_INIT();
  const EmbShape s = shape_of(args, args->tokens);
  return args->dtype == CCT_BF16 ? embedding_forward<bf16>(out, table, ids, s) : embedding_forward<float>(out, table, ids, s);
}

extern "C" size_t cct_hip_embedding_workspace_bytes(const cct_embedding_args *args) {
  return check_embedding(args, "embedding_workspace_bytes") ? 0 : embedding_layout(args).total;
}

extern "C" int cct_hip_embedding_backward(void *dtable, const void *dout, const int *ids, const cct_embedding_args *args,
                                          int accumulate, void *workspace, size_t workspace_bytes) {
  if (int rc = check_embedding(args, "embedding_backward")) return rc;
  if (args->tokens == 0 && accumulate) return 0;
  CCT_REQUIRE(dtable && (args->tokens == 0 || (dout && ids)), "embedding_backward: null array");
  const EmbWorkspace w = embedding_layout(args);
  CCT_REQUIRE(workspace_bytes >= w.total && (workspace || w.total == 0) && ((uintptr_t)workspace & 15) == 0,
              "embedding_backward: the workspace holds %zu bytes and starts at %p; it needs %zu, aligned to 16",
              workspace_bytes, workspace, w.total);
  CCT_ENSURE_INIT();
  const EmbShape s = shape_of(args, args->vocab);
  char *ws = (char *)workspace;
  return args->dtype == CCT_BF16 ? embedding_backward<bf16>(dtable, dout, ids, s, accumulate, ws, w)
                                 : embedding_backward<float>(dtable, dout, ids, s, accumulate, ws, w);
}
