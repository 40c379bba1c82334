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
};

// ---- forward -----------------------------------------------------------------------------------------------------
// A workgroup's lanes are laid over (row, 16-byte vector of the row); `cols` vectors of a row belong to one group of
// lanes (a power of two of at most 256), a wider row takes several trips.
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
    store_vec<T>(dst, f, col, s.width);
  }
}

// ---- sorting the tokens by id --------------------------------------------------------------------------------------
// Keys: the id, or `vocab` (behind every valid one) for tokens that give no gradient.
__device__ __forceinline__ uint32_t sort_key(int id, int padding, int vocab) {
  return id == padding || (unsigned)id >= (unsigned)vocab ? (uint32_t)vocab : (uint32_t)id;
}

// Few tokens: a token's place is the number of tokens that come before it, counted directly.  EMB_RANK_LANES lanes share
// a token, the ids pass through LDS in blocks.  tokens^2 comparisons over the whole chip in one launch.
constexpr int EMB_RANK_MAX = 8192;
constexpr int EMB_RANK_LANES = 16;
constexpr int EMB_RANK_BLOCK = 2048;
__global__ __launch_bounds__(EMB_THREADS) void embedding_rank_kernel(uint32_t *__restrict__ keys, int *__restrict__ order,
                                                                     const int *__restrict__ ids, int tokens,
                                                                     int padding, int vocab) {
  __shared__ uint32_t block[EMB_RANK_BLOCK];
  const int lane = threadIdx.x % EMB_RANK_LANES;
  const int t = blockIdx.x * (EMB_THREADS / EMB_RANK_LANES) + threadIdx.x / EMB_RANK_LANES;
  const uint32_t key = t < tokens ? sort_key(ids[t], padding, vocab) : 0u;
  int before = 0;
  for (int base = 0; base < tokens; base += EMB_RANK_BLOCK) {
    const int n = min(EMB_RANK_BLOCK, tokens - base);
    __syncthreads();
    for (int i = threadIdx.x; i < EMB_RANK_BLOCK; i += EMB_THREADS)
      block[i] = i < n ? sort_key(ids[base + i], padding, vocab) : 0xFFFFFFFFu;
    __syncthreads();
    for (int i = lane; i < n; i += EMB_RANK_LANES) {
      const uint32_t other = block[i];
      before += (other < key || (other == key && base + i < t)) ? 1 : 0;
    }
  }
#pragma unroll
  for (int m = EMB_RANK_LANES / 2; m > 0; m >>= 1) before += __shfl_xor(before, m, 64);
  if (lane == 0 && t < tokens) {
    keys[before] = key;
    order[before] = t;
  }
}

// Many tokens: least-significant-digit radix sort, 9 bits a pass.  One workgroup per tile of 4096 tokens counts its
// digits; the second launch of a pass turns the tiles' counts into places (digits ascending, tiles ascending within a
// digit) and moves the tile in order, so every pass is stable.
constexpr int EMB_BITS = 9, EMB_BINS = 1 << EMB_BITS;
constexpr int EMB_ITEMS = 16, EMB_TILE = EMB_THREADS * EMB_ITEMS;
constexpr int EMB_WAVES = EMB_THREADS / 64;

// The token (and its key) at a place of a pass's input: the first pass reads the ids themselves.
__device__ __forceinline__ uint32_t pass_key(const uint32_t *__restrict__ keys, const int *__restrict__ ids, int i,
                                             int padding, int vocab) {
  return keys ? keys[i] : sort_key(ids[i], padding, vocab);
}

__global__ __launch_bounds__(EMB_THREADS) void embedding_count_kernel(uint32_t *__restrict__ counts,
                                                                      const uint32_t *__restrict__ keys,
                                                                      const int *__restrict__ ids, int tokens,
                                                                      int padding, int vocab, int shift) {
  __shared__ uint32_t bins[EMB_BINS];
  for (int i = threadIdx.x; i < EMB_BINS; i += EMB_THREADS) bins[i] = 0;
  __syncthreads();
  for (int i = 0; i < EMB_ITEMS; ++i) {
    const int at = blockIdx.x * EMB_TILE + i * EMB_THREADS + threadIdx.x;
    if (at < tokens) atomicAdd(&bins[(pass_key(keys, ids, at, padding, vocab) >> shift) & (EMB_BINS - 1)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < EMB_BINS; i += EMB_THREADS) counts[(size_t)blockIdx.x * EMB_BINS + i] = bins[i];
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
  for (uint32_t tile = 0; tile < gridDim.x; ++tile) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t c = counts[(size_t)tile * EMB_BINS + tid * PER + j];
      all[j] += c;
      before[j] += tile < blockIdx.x ? c : 0u;
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
  // wavefront w takes the tile's tokens [w * 1024, ...) 64 at a time, in order: a token's rank within its wavefront's
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

// sum of dout[order[p]] over the places [p0, p1), columns [col, col + V)
template <class T>
__device__ __forceinline__ void sum_rows(float (&acc)[Num<T>::V], const T *__restrict__ dout,
                                         const int *__restrict__ order, int p0, int p1, int col, const EmbShape &s) {
  constexpr int V = Num<T>::V;
  int p = p0;
  for (; p + 4 <= p1; p += 4) {  // four rows in flight, added in order
    float f[4][V];
#pragma unroll
    for (int j = 0; j < 4; ++j) load_vec<T>(f[j], dout + (size_t)order[p + j] * s.out_stride, col, s.width);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += f[j][i];
  }
  for (; p < p1; ++p) {
    float f[V];
    load_vec<T>(f, dout + (size_t)order[p] * s.out_stride, col, s.width);
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += f[i];
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
  store_vec<T>(row, acc, col, s.width);
}

// An id with more than EMB_RUN tokens is summed in pieces of EMB_RUN sorted places.  Piece j covers places
// [j * EMB_RUN, (j + 1) * EMB_RUN) and can hold parts of two such ids: slot 0 the one that holds its first place, slot 1
// one that begins inside.  Ids with fewer tokens are summed whole by the workgroup that owns their row.
constexpr int EMB_RUN = 64;
constexpr int EMB_ROWS = 8;  // rows of the table per workgroup and trip, at least

template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_sum_kernel(T *__restrict__ dtable, float *__restrict__ parts,
                                                                    const T *__restrict__ dout,
                                                                    const uint32_t *__restrict__ keys,
                                                                    const int *__restrict__ order, EmbShape s,
                                                                    int accumulate, int log_lanes, int row_blocks) {
  constexpr int V = Num<T>::V;
  __shared__ int bounds[EMB_THREADS + 1];
  const int tid = threadIdx.x, lanes = 1 << log_lanes, lane = tid & (lanes - 1), group = tid >> log_lanes;
  const int groups = EMB_THREADS >> log_lanes;
  if ((int)blockIdx.x < row_blocks) {
    const int rows = max(EMB_ROWS, groups);
    const int v0 = blockIdx.x * rows, n = min(rows, s.vocab - v0);
    for (int i = tid; i <= n; i += EMB_THREADS) bounds[i] = lower_bound(keys, s.tokens, (uint32_t)(v0 + i));
    __syncthreads();
    for (int r = group; r < n; r += groups) {
      const int p0 = bounds[r], p1 = bounds[r + 1];
      if (p1 - p0 > EMB_RUN || (accumulate && p1 == p0)) continue;
      T *row = dtable + (size_t)(v0 + r) * s.table_stride;
      for (int col = lane * V; col < s.width; col += lanes * V) {
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
        sum_rows<T>(acc, dout, order, p0, p1, col, s);
        store_row<T>(row, acc, col, s, accumulate);
      }
    }
    return;
  }
  const int piece = blockIdx.x - row_blocks;
  if (tid < 2) {
    const int a = piece * EMB_RUN, b = min(a + EMB_RUN, s.tokens);
    const uint32_t key = keys[tid == 0 ? a : b - 1];
    int p0 = lower_bound(keys, s.tokens, key), p1 = lower_bound(keys, s.tokens, key + 1);
    const bool take = key < (uint32_t)s.vocab && p1 - p0 > EMB_RUN && (tid == 0 || p0 > a);
    bounds[2 * tid] = take ? max(p0, a) : 0;
    bounds[2 * tid + 1] = take ? min(p1, b) : 0;
  }
  __syncthreads();
  for (int slot = 0; slot < 2; ++slot) {
    const int p0 = bounds[2 * slot], p1 = bounds[2 * slot + 1];
    if (p0 == p1) continue;
    float *dst = parts + ((size_t)piece * 2 + slot) * s.width;
    for (int col = tid * V; col < s.width; col += EMB_THREADS * V) {
      float acc[V];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.0f;
      sum_rows<T>(acc, dout, order, p0, p1, col, s);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (col + i < s.width) dst[col + i] = acc[i];
    }
  }
}

// The pieces of a long id, added in order: the workgroup of the piece in which it begins, four columns groups of lanes
// taking every fourth piece each.
template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_join_kernel(T *__restrict__ dtable,
                                                                     const float *__restrict__ parts,
                                                                     const uint32_t *__restrict__ keys, EmbShape s,
                                                                     int accumulate) {
  __shared__ int bounds[3];
  __shared__ float sums[4][64];
  const int tid = threadIdx.x, piece = blockIdx.x;
  if (tid == 0) {
    // an id that begins in this piece and has more than EMB_RUN tokens holds the piece's last place
    const int last = piece * EMB_RUN + EMB_RUN - 1;
    int p0 = 0, p1 = 0, key = 0;
    if (last < s.tokens) {
      key = (int)keys[last];
      p0 = lower_bound(keys, s.tokens, (uint32_t)key);
      p1 = lower_bound(keys, s.tokens, (uint32_t)key + 1);
      if (key >= s.vocab || p1 - p0 <= EMB_RUN || p0 < piece * EMB_RUN) p0 = p1 = 0;
    }
    bounds[0] = p0;
    bounds[1] = p1;
    bounds[2] = key;
  }
  __syncthreads();
  const int p0 = bounds[0], p1 = bounds[1];
  if (p0 == p1) return;
  const int end = (p1 - 1) / EMB_RUN;
  const int lane = tid & 63, group = tid >> 6, col = blockIdx.y * 64 + lane;
  const bool have = col < s.width;
  float acc = 0.0f;
  for (int j = piece + group; j <= end && have; j += 4) {
    const int slot = j == piece && p0 != piece * EMB_RUN ? 1 : 0;
    acc += parts[((size_t)j * 2 + slot) * s.width + col];
  }
  sums[group][lane] = acc;
  __syncthreads();
  if (group == 0 && have) {
    acc = ((sums[0][lane] + sums[1][lane]) + sums[2][lane]) + sums[3][lane];
    T *dst = dtable + (size_t)bounds[2] * s.table_stride + col;
    *dst = (T)(accumulate ? (float)*dst + acc * s.scale : acc * s.scale);
  }
}

// Lanes that share a row: as many as it has 16-byte vectors, up to a workgroup.
template <class T>
static int row_lanes_log2(int width) {
  const int vecs = (width + Num<T>::V - 1) / Num<T>::V;
  int l = 0;
  while ((1 << l) < vecs && l < 8) ++l;
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

static EmbShape shape_of(const cct_embedding_args *a) {
  return EmbShape{a->tokens, a->width, a->vocab, a->padding_id, a->scale,
                  a->table_stride ? a->table_stride : (size_t)a->width, a->out_stride ? a->out_stride : (size_t)a->width};
}

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// keys and order (twice: the radix passes alternate), the tiles' digit counts, the pieces' sums
struct EmbWorkspace {
  size_t keys[2], order[2], counts, parts, total;
};
static EmbWorkspace embedding_layout(const cct_embedding_args *a) {
  EmbWorkspace w;
  const size_t n = a->tokens, tiles = (n + EMB_TILE - 1) / EMB_TILE;
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
  w.counts = take(radix ? tiles * EMB_BINS * 4 : 0);
  w.parts = take(a->tokens > EMB_RUN ? (n + EMB_RUN - 1) / EMB_RUN * 2 * a->width * sizeof(float) : 0);
  w.total = at;
  return w;
}

template <class T>
static int embedding_forward(void *out, const void *table, const int *ids, const EmbShape &s) {
  const int l = row_lanes_log2<T>(s.width);
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

static int sort_tokens(char *ws, const EmbWorkspace &w, const int *ids, const EmbShape &s, uint32_t **keys, int **order) {
  hipStream_t st = ctx().stream;
  uint32_t *k[2] = {(uint32_t *)(ws + w.keys[0]), (uint32_t *)(ws + w.keys[1])};
  int *o[2] = {(int *)(ws + w.order[0]), (int *)(ws + w.order[1])};
  if (s.tokens <= EMB_RANK_MAX) {
    const int per = EMB_THREADS / EMB_RANK_LANES;
    embedding_rank_kernel<<<(s.tokens + per - 1) / per, EMB_THREADS, 0, st>>>(k[0], o[0], ids, s.tokens, s.padding, s.vocab);
    CCT_LAUNCH_CHECK();
    *keys = k[0];
    *order = o[0];
    return 0;
  }
  const unsigned tiles = (s.tokens + EMB_TILE - 1) / EMB_TILE;
  uint32_t *counts = (uint32_t *)(ws + w.counts);
  int from = -1;  // the first pass reads the ids
  for (int shift = 0; shift < 32 && ((uint32_t)s.vocab >> shift) != 0; shift += EMB_BITS) {
    const int to = from == 0 ? 1 : 0;
    const uint32_t *kin = from < 0 ? nullptr : k[from];
    const int *oin = from < 0 ? nullptr : o[from];
    embedding_count_kernel<<<tiles, EMB_THREADS, 0, st>>>(counts, kin, ids, s.tokens, s.padding, s.vocab, shift);
    CCT_LAUNCH_CHECK();
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
static int embedding_backward(void *dtable, const void *dout, const int *ids, const EmbShape &s, int accumulate, char *ws,
                              const EmbWorkspace &w) {
  hipStream_t st = ctx().stream;
  uint32_t *keys = nullptr;
  int *order = nullptr;
  if (s.tokens > 0)
    if (int rc = sort_tokens(ws, w, ids, s, &keys, &order)) return rc;
  const int l = row_lanes_log2<T>(s.width), rows = max(EMB_ROWS, EMB_THREADS >> l);
  const int row_blocks = (s.vocab + rows - 1) / rows;
  const int pieces = s.tokens > EMB_RUN ? (s.tokens + EMB_RUN - 1) / EMB_RUN : 0;
  float *parts = (float *)(ws + w.parts);
  embedding_sum_kernel<T><<<row_blocks + pieces, EMB_THREADS, 0, st>>>((T *)dtable, parts, (const T *)dout, keys, order, s,
                                                                      accumulate, l, row_blocks);
  CCT_LAUNCH_CHECK();
  note_kernel("embedding_sum_kernel<%s> rows per workgroup=%d pieces=%d", Num<T>::NAME, rows, pieces);
  if (pieces) {
    embedding_join_kernel<T><<<dim3(pieces, (s.width + 63) / 64), EMB_THREADS, 0, st>>>((T *)dtable, parts, keys, s,
                                                                                       accumulate);
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
  const EmbShape s = shape_of(args);
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
  const EmbShape s = shape_of(args);
  char *ws = (char *)workspace;
  return args->dtype == CCT_BF16 ? embedding_backward<bf16>(dtable, dout, ids, s, accumulate, ws, w)
                                 : embedding_backward<float>(dtable, dout, ids, s, accumulate, ws, w);
}
