// Vocabulary loss: the softmax loss of an inner-product layer with a large vocabulary of outputs, without its scores.
//
//   l[t][v] = x[t] . w[v] + bias[v]      lse[t] = log sum_v exp l[t][v]      loss[t] = lse[t] - l[t][label[t]]
//   G[t][v] = exp(l[t][v] - lse[t]) - [v == label[t]]
//   dx[t] = g[t] * sum_v G[t][v] w[v]    dw[v] = sum_t g[t] G[t][v] x[t]     db[v] = sum_t g[t] G[t][v]
//
// Every product is one kernel, C[m][n] = sum_k A[m][k] B[n][k] with both operands contiguous along k, and four ways to
// use a finished tile:
//   STATS  m = vocabulary, n = token: maximum and sum of the tile's scores per token (a few bytes instead of the tile), the
//          label's score, and the scores themselves where the caller keeps them for the gradient;
//   GRAD   the same product again with lse known: G of a piece of the vocabulary, written as G[t][v] (the operand of dx)
//          and as g[t] G[t][v] transposed (the operand of dw), and the column sums for db;
//   SLAB   m = width, n = token, k = the piece's vocabulary: dx in fp32, added up over the pieces;
//   OUT    m = width, n = vocabulary, k = token: dw of the piece, stored once in its own type.
// The k-contiguous forms of w and x that the last two need (w piece and x transposed) are made by a copy kernel.
//
// Bound: matrix-core rate.  2 tokens*width*vocab operations for the loss, 4 more for the gradients and 2 for the scores
// again where they were not kept.
#include <type_traits>

#include "mfma_common.h"
#include "narrow.h"

namespace cct {

// ---- the product kernel ----------------------------------------------------------------------------------------
// A workgroup owns a BM x BN tile of C and walks k in steps of 128 bytes (64 bf16 or 32 fp32 elements) through two LDS
// stages.  Rows of a stage are 128 bytes, 16-byte chunk c of row r lies in slot c ^ ((r >> 1) & 7): the 16 lanes of a
// fragment read (16 rows, one chunk) then touch all 64 banks once.  global -> LDS copies cannot permute what a lane
// receives, so the lane that fills slot s of row r fetches chunk s ^ ((r >> 1) & 7).
// Fragments of v_mfma_f32_16x16x32_bf16 and v_mfma_f32_16x16x4_f32: lane l holds 16 bytes of row l % 16, chunk l / 16
// of a 64-byte group; C element r of lane l is row 4 * (l / 16) + r, column l % 16.  For fp32 the four elements of a
// chunk feed four MFMAs (the sum over k may run in any order as long as both operands use the same one).
enum Use { USE_STATS = 0, USE_GRAD = 1, USE_SLAB = 2, USE_OUT = 3 };

template <int BM_, int BN_, int WM_, int WN_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;  // 16 x 16 blocks of a wavefront
  static constexpr int JA = BM / 8 / WAVES, JB = BN / 8 / WAVES;  // 1 KB copies per wavefront and step
  static constexpr int STAGE = (BM + BN) * 128;
  static_assert(BM % (WM * 16) == 0 && BN % (WN * 16) == 0, "wavefront tiles are whole blocks");
  static_assert(JA * 8 * WAVES == BM && JB * 8 * WAVES == BN, "whole copies");
  // copy i of an operand fills rows 8 i + lane / 8; with an even number of wavefronts the swizzle of a lane is the same
  // for all of its copies
  static_assert(WAVES % 2 == 0, "even number of wavefronts");
};

struct ProductArgs {
  const char *A, *B;
  size_t lda, ldb;  // bytes between rows
  int M, N;
  uint32_t kbytes;  // bytes of a row of A and B that take part; multiple of 16
  int tiles_m, tiles_n, splits, steps_per_split;
  uint32_t blocks;
  // STATS, GRAD (m = rows v0 + m of the vocabulary, n = token)
  const void *bias;          // of the piece's first row, or null
  const int *labels;
  int v0, vocab, ignore;
  SoftStat *part;            // STATS: [tile of the whole vocabulary][token]
  int part_row;              // first tile of the piece
  float *label_score;        // STATS: [token]
  float *scores;             // STATS: [token][ldg] raw scores, or null
  const float *lse, *gscale; // GRAD; gscale: loss_grad or null
  void *g, *gt;              // GRAD: [token][ldg], [vocabulary row][ldgt]
  size_t ldg, ldgt;          // elements
  int mpad, npad;            // GRAD: columns of g and of gt, whole 16-byte chunks (past M and N they are zero)
  float *db_part;            // GRAD: [tile_n][row of the piece] or null
  int db_ld;
  // SLAB: C [split][N][M] fp32.  OUT: C [n][ldc] elements
  void *C;
  size_t ldc;
  int accumulate;
};

template <class T>
__device__ __forceinline__ void mfma_chunk(f32x4 &c, const f32x4 &a, const f32x4 &b);
template <>
__device__ __forceinline__ void mfma_chunk<bf16>(f32x4 &c, const f32x4 &a, const f32x4 &b) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ void mfma_chunk<float>(f32x4 &c, const f32x4 &a, const f32x4 &b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
}

// G of one score: the label's own entry is p - 1
__device__ __forceinline__ float grad_entry(float score, float lse, bool is_label) {
  const float p = exp2_fast((score - lse) * kLog2e);
  return is_label ? p - 1.0f : p;
}

// A token's part in the gradient: its label's row (or -1), its lse and its weight; ignored tokens have weight 0 and
// their G is 0 whatever their scores are.
struct TokenGrad {
  int label;
  float lse, weight;
  bool live;
};
__device__ __forceinline__ TokenGrad token_grad(int t, int tokens, const int *__restrict__ labels, int ignore,
                                                const float *__restrict__ lse, const float *__restrict__ gscale) {
  TokenGrad g{-1, 0.0f, 0.0f, false};
  if (t < tokens) {
    g.label = labels[t];
    g.live = g.label != ignore;
    g.lse = lse[t];
    g.weight = g.live ? (gscale ? gscale[t] : 1.0f) : 0.0f;
  }
  return g;
}

template <class T>
__device__ __forceinline__ void store4(T *p, const float (&f)[4]) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  vec4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (T)f[i];
  *reinterpret_cast<vec4 *>(p) = v;
}

template <class T, class S, int USE>
__global__ __launch_bounds__(S::THREADS) void vocab_product_kernel(ProductArgs p) {
  extern __shared__ __align__(16) char lds[];
  constexpr int MI = S::MI, NI = S::NI;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / S::WN, wn = wave % S::WN;
  const uint32_t id = xcd_remap(blockIdx.x, p.blocks);
  const uint32_t split = id / (uint32_t)(p.tiles_m * p.tiles_n);
  const uint32_t tile = id - split * (uint32_t)(p.tiles_m * p.tiles_n);
  // tiles in bands of eight along m: neighbours in time share rows of both operands in an XCD's L2
  const uint32_t band = tile / (8u * p.tiles_n), in_band = tile - band * 8u * p.tiles_n;
  const uint32_t band_m = min(8u, (uint32_t)p.tiles_m - band * 8u);
  const int tm = (int)(band * 8u + in_band % band_m), tn = (int)(in_band / band_m);
  const int m0 = tm * S::BM, n0 = tn * S::BN;

  // global -> LDS copies: lane offsets within the tile's rows (rows past the end repeat the last one: their results
  // are never used)
  const rsrc_t ra = make_rsrc(p.A + (size_t)m0 * p.lda), rb = make_rsrc(p.B + (size_t)n0 * p.ldb);
  const int crow = wave * 8 + (lane >> 3);
  const uint32_t chunk = ((uint32_t)(lane & 7) ^ ((uint32_t)(crow >> 1) & 7u)) * 16u;
  uint32_t va[S::JA], vb[S::JB];
#pragma unroll
  for (int j = 0; j < S::JA; ++j) va[j] = (uint32_t)min(crow + j * S::WAVES * 8, p.M - 1 - m0) * (uint32_t)p.lda + chunk;
#pragma unroll
  for (int j = 0; j < S::JB; ++j) vb[j] = (uint32_t)min(crow + j * S::WAVES * 8, p.N - 1 - n0) * (uint32_t)p.ldb + chunk;
  auto stage = [&](int buf, int step) {
    const uint32_t k = (uint32_t)step * 128u;
    const bool in = k + chunk < p.kbytes;  // chunks past the end of k are filled with zeros
    char *base = lds + buf * S::STAGE + wave * 1024;
#pragma unroll
    for (int j = 0; j < S::JA; ++j)
      lds_dma16(ra, in ? va[j] : kOutOfRange, k, (float *)(base + j * S::WAVES * 1024));
#pragma unroll
    for (int j = 0; j < S::JB; ++j)
      lds_dma16(rb, in ? vb[j] : kOutOfRange, k, (float *)(base + S::BM * 128 + j * S::WAVES * 1024));
  };

  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int frow = lane & 15, fgroup = lane >> 4, fswz = (frow >> 1) & 7;
  const int fa = (wm * MI * 16 + frow) * 128, fb = S::BM * 128 + (wn * NI * 16 + frow) * 128;
  const int steps = (int)((p.kbytes + 127u) / 128u);
  const int s0 = (int)split * p.steps_per_split, s1 = min(steps, s0 + p.steps_per_split);
  if (s0 < s1) stage(0, s0);
  for (int s = s0; s < s1; ++s) {
    lds_dma_wait();
    __syncthreads();
    const int buf = (s - s0) & 1;
    if (s + 1 < s1) stage(buf ^ 1, s + 1);
    const char *base = lds + buf * S::STAGE;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const int slot = ((sub * 4 + fgroup) ^ fswz) * 16;
      f32x4 a[MI], b[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) a[i] = *reinterpret_cast<const f32x4 *>(base + fa + i * 2048 + slot);
#pragma unroll
      for (int j = 0; j < NI; ++j) b[j] = *reinterpret_cast<const f32x4 *>(base + fb + j * 2048 + slot);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) mfma_chunk<T>(acc[i][j], a[i], b[j]);
    }
  }

  // this lane's elements: rows mrow + 16 i + r, columns ncol + 16 j
  const int mrow = m0 + wm * MI * 16 + fgroup * 4, ncol = n0 + wn * NI * 16 + frow;

  if constexpr (USE == USE_STATS || USE == USE_GRAD) {
    if (p.bias) {
      const T *bias = (const T *)p.bias;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float b = mrow + i * 16 + r < p.M ? (float)bias[mrow + i * 16 + r] : 0.0f;
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j][r] += b;
        }
    }
  }

  if constexpr (USE == USE_STATS) {
    __syncthreads();  // the stages are done with
    SoftStat *sh = (SoftStat *)lds;  // [WM][BN]
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int t = ncol + j * 16;
      const int label = t < p.N ? p.labels[t] : -1;
      SoftStat st{neg_inf(), 0.0f};
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int m = mrow + i * 16 + r;
          if (p.v0 + m == label && m < p.M) p.label_score[t] = acc[i][j][r];
          if (p.scores && t < p.N && m < p.M) p.scores[(size_t)t * p.ldg + m] = acc[i][j][r];
          acc[i][j][r] = m < p.M ? acc[i][j][r] : neg_inf();
          st.m = fmaxf(st.m, acc[i][j][r]);
        }
      const float base = st.m == neg_inf() ? 0.0f : st.m;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.s += exp2_fast((acc[i][j][r] - base) * kLog2e);
      st = shfl_xor_join(st, 16, kLog2e);
      st = shfl_xor_join(st, 32, kLog2e);
      if (fgroup == 0) sh[wm * S::BN + (wn * NI + j) * 16 + frow] = st;
    }
    __syncthreads();
    for (int n = tid; n < S::BN; n += S::THREADS) {
      if (n0 + n >= p.N) break;
      SoftStat st = sh[n];
#pragma unroll
      for (int w = 1; w < S::WM; ++w) st = join(st, sh[w * S::BN + n], kLog2e);
      p.part[(size_t)(p.part_row + tm) * p.N + n0 + n] = st;
    }
  }

  if constexpr (USE == USE_GRAD) {
    __syncthreads();
    float *sums = (float *)lds;  // [WN][BM] column sums for db
    float rows[MI][4];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) rows[i][r] = 0.0f;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int t = ncol + j * 16;
      const TokenGrad tg = token_grad(t, p.N, p.labels, p.ignore, p.lse, p.gscale);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int m = mrow + i * 16;
        float g[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool live = tg.live && m + r < p.M;
          g[r] = live ? grad_entry(acc[i][j][r], tg.lse, p.v0 + m + r == tg.label) : 0.0f;
        }
        if (t < p.N && m < p.mpad) store4<T>((T *)p.g + (size_t)t * p.ldg + m, g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float gw = g[r] * tg.weight;
          rows[i][r] += gw;
          if (m + r < p.M && t < p.npad) ((T *)p.gt)[(size_t)(m + r) * p.ldgt + t] = (T)gw;
        }
      }
    }
    if (p.db_part) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int d = 1; d < 16; d <<= 1) rows[i][r] += __shfl_xor(rows[i][r], d, 64);
          if (frow == 0) sums[wn * S::BM + (wm * MI + i) * 16 + fgroup * 4 + r] = rows[i][r];
        }
      __syncthreads();
      for (int m = tid; m < S::BM; m += S::THREADS) {
        if (m0 + m >= p.M) break;
        float s = sums[m];
#pragma unroll
        for (int w = 1; w < S::WN; ++w) s += sums[w * S::BM + m];
        p.db_part[(size_t)tn * p.db_ld + m0 + m] = s;
      }
    }
  }

  if constexpr (USE == USE_SLAB || USE == USE_OUT) {
    typedef typename std::conditional<USE == USE_SLAB, float, T>::type Out;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int n = ncol + j * 16;
      if (n >= p.N) continue;
      Out *row = (Out *)p.C + (USE == USE_SLAB ? ((size_t)split * p.N + n) * p.M : (size_t)n * p.ldc);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int m = mrow + i * 16;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m + r < p.M) {
            float v = acc[i][j][r];
            if (USE == USE_SLAB && p.accumulate) v += (float)row[m + r];
            row[m + r] = (Out)v;
          }
      }
    }
  }
}

// ---- copies ------------------------------------------------------------------------------------------------------
// dst[c][r] = src[r][c] for c < cols, with columns [rows, rpad) of dst zero; tokens that the loss ignores count as rows of
// zeros (labels given), so that whatever their x holds stays out of the products.
template <class T>
__global__ __launch_bounds__(256) void vocab_transpose_kernel(T *__restrict__ dst, const T *__restrict__ src, size_t ld_src,
                                                              size_t ld_dst, int rows, int cols, int rpad,
                                                              const int *__restrict__ labels, int ignore) {
  __shared__ T tile[64][64 + 4 / sizeof(T)];
  const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = r0 + y + i * 4, c = c0 + x;
    const bool in = r < rows && c < cols && !(labels && labels[r] == ignore);
    tile[y + i * 4][x] = in ? src[(size_t)r * ld_src + c] : (T)0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = c0 + y + i * 4, r = r0 + x;
    if (c < cols && r < rpad) dst[(size_t)c * ld_dst + r] = tile[x][y + i * 4];
  }
}

// dst[r][c] = src[r][c], rows of dst filled up to cpad with zeros: operands whose rows do not start at 16-byte
// boundaries or are no whole number of 16-byte chunks
template <class T>
__global__ __launch_bounds__(256) void vocab_pack_kernel(T *__restrict__ dst, const T *__restrict__ src, size_t ld_src,
                                                         int cols, int cpad) {
  const size_t r = blockIdx.x;
  constexpr int V = Num<T>::V;
  for (int c = threadIdx.x * V; c < cpad; c += 256 * V) {
    float f[V];
    load_vec<T>(f, src + r * ld_src, c, cols);
    store_vec<T>(dst + r * cpad, f, c, cpad);
  }
}

// ---- joining -----------------------------------------------------------------------------------------------------
// The tiles' statistics of each token, in order: 16 tokens per workgroup, 16 lanes each taking every 16th tile.
__global__ __launch_bounds__(256) void vocab_loss_kernel(float *__restrict__ loss, float *__restrict__ lse,
                                                         const SoftStat *__restrict__ part,
                                                         const float *__restrict__ label_score,
                                                         const int *__restrict__ labels, int tokens, int tiles, int vocab,
                                                         int ignore) {
  __shared__ SoftStat sh[16][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, t = blockIdx.x * 16 + x;
  SoftStat st{neg_inf(), 0.0f};
  if (t < tokens)
    for (int i = y; i < tiles; i += 16) st = join(st, part[(size_t)i * tokens + t], kLog2e);
  sh[y][x] = st;
  __syncthreads();
  if (y == 0 && t < tokens) {
#pragma unroll
    for (int i = 1; i < 16; ++i) st = join(st, sh[i][x], kLog2e);
    const float l = log_sum(st, 1.0f);
    const int label = labels[t];
    lse[t] = l;
    loss[t] = label == ignore ? 0.0f
              : (unsigned)label < (unsigned)vocab ? l - label_score[t]
                                                  : __builtin_nanf("");
  }
}

// G and its transpose from kept scores, 64 x 64 entries a workgroup, and the column sums of the tile.
template <class T>
__global__ __launch_bounds__(256) void vocab_grad_kernel(T *__restrict__ g, T *__restrict__ gt,
                                                         const float *__restrict__ scores, float *__restrict__ db_part,
                                                         const int *__restrict__ labels, const float *__restrict__ lse,
                                                         const float *__restrict__ gscale, int tokens, int vocab, int v0,
                                                         int rows, int ignore, size_t ld_scores, size_t ldg, size_t ldgt,
                                                         int mpad, int npad, int db_ld) {
  __shared__ float tile[64][65];
  __shared__ float sums[4][64];
  const int m0 = blockIdx.x * 64, t0 = blockIdx.y * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const int m = m0 + x;
  float sum = 0.0f;
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int t = t0 + y + i * 4;
    const TokenGrad tg = token_grad(t, tokens, labels, ignore, lse, gscale);
    float v = 0.0f;
    if (tg.live && m < rows) v = grad_entry(scores[(size_t)t * ld_scores + m], tg.lse, v0 + m == tg.label);
    if (t < tokens && m < mpad) g[(size_t)t * ldg + m] = (T)v;
    v *= tg.weight;
    sum += v;
    tile[y + i * 4][x] = v;
  }
  sums[y][x] = sum;
  __syncthreads();
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int mm = m0 + y + i * 4, t = t0 + x;
    if (mm < rows && t < npad) gt[(size_t)mm * ldgt + t] = (T)tile[x][y + i * 4];
  }
  if (db_part && y == 0 && m < rows)
    db_part[(size_t)blockIdx.y * db_ld + m] = ((sums[0][x] + sums[1][x]) + sums[2][x]) + sums[3][x];
}

// dx[t] = weight * sum of the slabs, in order
template <class T>
__global__ __launch_bounds__(256) void vocab_dx_kernel(T *__restrict__ dx, const float *__restrict__ slabs,
                                                       const int *__restrict__ labels, const float *__restrict__ gscale,
                                                       int ignore, int tokens, int width, size_t ldx, int splits) {
  const int t = blockIdx.x;
  const bool live = labels[t] != ignore;
  const float weight = gscale ? gscale[t] : 1.0f;
  for (int c = threadIdx.x; c < width; c += 256) {
    float s = 0.0f;
    for (int i = 0; i < splits; ++i) s += slabs[((size_t)i * tokens + t) * width + c];
    dx[(size_t)t * ldx + c] = (T)(live ? s * weight : 0.0f);
  }
}

template <class T>
__global__ __launch_bounds__(256) void vocab_db_kernel(T *__restrict__ db, const float *__restrict__ part, int rows, int ld,
                                                       int tiles) {
  const int m = blockIdx.x * 256 + threadIdx.x;
  if (m >= rows) return;
  float s = 0.0f;
  for (int i = 0; i < tiles; ++i) s += part[(size_t)i * ld + m];
  db[m] = (T)s;
}

template <class T>
__global__ __launch_bounds__(256) void vocab_zero_kernel(T *__restrict__ p, size_t ld, int cols) {
  for (int c = threadIdx.x; c < cols; c += 256) p[(size_t)blockIdx.x * ld + c] = (T)0.0f;
}

// ---- host --------------------------------------------------------------------------------------------------------
typedef Shape<256, 256, 2, 4> ShapeL;
typedef Shape<128, 128, 2, 2> ShapeM;
typedef Shape<64, 32, 4, 1> ShapeS;

static int idiv(int a, int b) { return (a + b - 1) / b; }
static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Which tile: the largest that still gives most of the 256 CUs a workgroup (`splits_ok`: the launch may also be cut
// along k); few columns take the narrow tile.
enum ShapeId { SHAPE_L, SHAPE_M, SHAPE_S };
static ShapeId choose_shape(int M, int N) {
  if (N <= 32) return SHAPE_S;
  if ((long)idiv(M, 256) * idiv(N, 256) >= 192) return SHAPE_L;
  return SHAPE_M;
}
static int shape_bm(ShapeId s) { return s == SHAPE_L ? ShapeL::BM : s == SHAPE_M ? ShapeM::BM : ShapeS::BM; }
static int shape_bn(ShapeId s) { return s == SHAPE_L ? ShapeL::BN : s == SHAPE_M ? ShapeM::BN : ShapeS::BN; }

constexpr size_t kKeepBytes = (size_t)512 << 20;   // fp32 scores kept between forward and backward of one call
constexpr size_t kPieceBytes = (size_t)384 << 20;  // automatic piece: G, its transpose and w's transpose

// a tile's rows are addressed with 32-bit byte offsets: 256 rows of a piece's columns in fp32 are 2^30 bytes
constexpr int kPieceMax = 1 << 20;

struct VocabPlan {
  int tokens, width, vocab, dtype;
  size_t el, ldx, ldw;
  int unit;            // elements of a 128-byte step
  int piece, pieces;   // rows of w at a time
  bool keep;           // forward_backward keeps the scores (one piece)
  int np, hp, vp;      // row lengths of transposed and packed operands: tokens, width, piece rounded up to whole steps
  int nk;              // tokens rounded up to whole 16-byte chunks: what the transposed operands hold of k
  ShapeId fs, dxs, dws;
  int stats_tiles;
  int dx_splits;
  size_t part, label_score, xpack, wpack, g, gt, wt, xt, slabs, db, scores, total_forward, total;
};

static VocabPlan vocab_plan(const cct_vocab_loss_args *a) {
  VocabPlan p;
  p.tokens = a->tokens;
  p.width = a->width;
  p.vocab = a->vocab;
  p.dtype = a->dtype;
  p.el = dtype_bytes(a->dtype);
  p.ldx = a->x_stride ? a->x_stride : (size_t)a->width;
  p.ldw = a->w_stride ? a->w_stride : (size_t)a->width;
  p.unit = 128 / (int)p.el;
  p.np = idiv(p.tokens, p.unit) * p.unit;
  p.hp = idiv(p.width, p.unit) * p.unit;
  p.nk = idiv(p.tokens, p.unit / 8) * (p.unit / 8);
  const int vmax = idiv(p.vocab, 256) * 256;
  if (a->piece > 0) {
    p.piece = (int)min((((size_t)a->piece + 255) / 256) * 256, (size_t)kPieceMax);
  } else {
    // a power of two, so that the tiles of a piece fill whole rounds of the chip
    const size_t row = (2 * (size_t)p.np + p.hp) * p.el;
    size_t want = kPieceBytes / (row ? row : 1), rows = 1024;
    while (rows * 2 <= want && rows < (size_t)vmax) rows *= 2;
    p.piece = rows > (size_t)vmax ? vmax : (int)rows;
  }
  if (p.piece > vmax) p.piece = vmax;
  if (p.piece > kPieceMax) p.piece = kPieceMax;
  p.keep = a->piece <= 0 && vmax <= kPieceMax && (size_t)p.tokens * p.vocab * 4 <= kKeepBytes;
  if (p.keep) p.piece = vmax;
  p.pieces = idiv(p.vocab, p.piece);
  p.vp = p.piece;
  p.fs = choose_shape(p.piece, p.tokens);
  p.stats_tiles = 0;
  for (int v = 0; v < p.vocab; v += p.piece)
    p.stats_tiles += idiv(p.vocab - v < p.piece ? p.vocab - v : p.piece, shape_bm(p.fs));
  p.dxs = choose_shape(p.width, p.tokens);
  p.dws = choose_shape(p.width, p.piece);
  const long dx_tiles = (long)idiv(p.width, shape_bm(p.dxs)) * idiv(p.tokens > 0 ? p.tokens : 1, shape_bn(p.dxs));
  const int steps = p.vp / p.unit;
  // short of workgroups: cut along the vocabulary, no part shorter than eight steps
  long splits = 512 / dx_tiles;
  if (splits > steps / 8) splits = steps / 8;
  if (splits > 64) splits = 64;
  p.dx_splits = splits < 1 ? 1 : (int)splits;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  const size_t n = p.tokens;
  p.part = take((size_t)p.stats_tiles * n * sizeof(SoftStat));
  p.label_score = take(n * 4);
  p.xpack = take(n * p.hp * p.el);
  p.wpack = take((size_t)p.piece * p.hp * p.el);
  p.total_forward = at;
  p.g = take(n * p.vp * p.el);
  p.gt = take((size_t)p.vp * p.np * p.el);
  p.wt = take((size_t)p.width * p.vp * p.el);
  p.xt = take((size_t)p.width * p.np * p.el);
  p.slabs = take((size_t)p.dx_splits * n * p.width * 4);
  p.db = take((size_t)idiv(p.tokens, 32) * p.vp * 4);
  p.scores = take(p.keep ? n * p.vp * 4 : 0);
  p.total = at;
  return p;
}

template <class T, class S, int USE>
static int launch_product(ProductArgs &p) {
  auto kern = vocab_product_kernel<T, S, USE>;
  static LdsGrant grant;
  const size_t bytes = 2 * S::STAGE;
  if (int rc = grant_dynamic_lds((const void *)kern, bytes, grant)) return rc;
  p.tiles_m = idiv(p.M, S::BM);
  p.tiles_n = idiv(p.N, S::BN);
  const int steps = (int)((p.kbytes + 127u) / 128u);
  p.steps_per_split = idiv(steps, p.splits);
  const unsigned long blocks = (unsigned long)p.tiles_m * p.tiles_n * p.splits;
  CCT_REQUIRE(blocks * S::THREADS < (1ul << 32), "vocab_loss: %lu workgroups are too many for one launch", blocks);
  p.blocks = (uint32_t)blocks;
  kern<<<p.blocks, S::THREADS, bytes, ctx().stream>>>(p);
  CCT_LAUNCH_CHECK();
  note_kernel("vocab_product_kernel<%s, Shape<%d, %d, %d, %d>, %d> splits=%d", Num<T>::NAME, S::BM, S::BN, S::WM, S::WN, USE,
              p.splits);
  return 0;
}

template <class T, int USE>
static int product(ShapeId s, ProductArgs &p) {
  switch (s) {
    case SHAPE_L: return launch_product<T, ShapeL, USE>(p);
    case SHAPE_M: return launch_product<T, ShapeM, USE>(p);
    default: return launch_product<T, ShapeS, USE>(p);
  }
}

struct VocabCall {
  float *loss;
  float *lse;
  const float *lse_in;  // backward alone
  void *dx, *dw, *db;
  const void *x, *w, *bias;
  const int *labels;
  const float *gscale;
  int ignore;
  char *ws;
  bool forward, backward;
};

// operand rows as the product kernel needs them: 16-byte aligned, whole 16-byte chunks
static bool direct_rows(const void *p, size_t ld, int width, size_t el) {
  return ((uintptr_t)p & 15) == 0 && (ld * el & 15) == 0 && ((size_t)width * el & 15) == 0;
}

template <class T>
static int vocab_run(const VocabPlan &p, const VocabCall &c) {
  hipStream_t st = ctx().stream;
  const int n = p.tokens;
  const bool keep = p.keep && c.forward && c.backward;
  SoftStat *part = (SoftStat *)(c.ws + p.part);
  float *label_score = (float *)(c.ws + p.label_score);
  T *g = (T *)(c.ws + p.g), *gt = (T *)(c.ws + p.gt), *wt = (T *)(c.ws + p.wt), *xt = (T *)(c.ws + p.xt);
  float *slabs = (float *)(c.ws + p.slabs), *db_part = (float *)(c.ws + p.db);
  const char *x = (const char *)c.x;
  size_t ldx = p.ldx * p.el;
  uint32_t kbytes = (uint32_t)(p.width * p.el);
  if (!direct_rows(c.x, p.ldx, p.width, p.el) || !direct_rows(c.w, p.ldw, p.width, p.el)) {
    // both operands are packed when one has to be: they walk k alike
    T *xp = (T *)(c.ws + p.xpack);
    vocab_pack_kernel<T><<<n, 256, 0, st>>>(xp, (const T *)c.x, p.ldx, p.width, p.hp);
    CCT_LAUNCH_CHECK();
    x = (const char *)xp;
    ldx = p.hp * p.el;
    kbytes = (uint32_t)(p.hp * p.el);
  }
  const bool pack = x != (const char *)c.x;
  auto scores_of = [&](int v0, int rows, ProductArgs &a) -> int {
    a = ProductArgs{};
    a.A = (const char *)c.w + (size_t)v0 * p.ldw * p.el;
    a.lda = p.ldw * p.el;
    if (pack) {
      T *wp = (T *)(c.ws + p.wpack);
      vocab_pack_kernel<T><<<rows, 256, 0, st>>>(wp, (const T *)a.A, p.ldw, p.width, p.hp);
      CCT_LAUNCH_CHECK();
      a.A = (const char *)wp;
      a.lda = p.hp * p.el;
    }
    a.B = x;
    a.ldb = ldx;
    a.M = rows;
    a.N = n;
    a.kbytes = kbytes;
    a.splits = 1;
    a.bias = c.bias ? (const char *)c.bias + (size_t)v0 * p.el : nullptr;
    a.labels = c.labels;
    a.v0 = v0;
    a.vocab = p.vocab;
    a.ignore = c.ignore;
    a.ldg = p.vp;
    return 0;
  };
  if (c.forward) {
    int tiles = 0;
    for (int v0 = 0; v0 < p.vocab; v0 += p.piece) {
      const int rows = min(p.piece, p.vocab - v0);
      ProductArgs a;
      if (int rc = scores_of(v0, rows, a)) return rc;
      a.part = part;
      a.part_row = tiles;
      a.label_score = label_score;
      a.scores = keep ? (float *)(c.ws + p.scores) : nullptr;
      if (int rc = product<T, USE_STATS>(p.fs, a)) return rc;
      tiles += a.tiles_m;
    }
    vocab_loss_kernel<<<idiv(n, 16), 256, 0, st>>>(c.loss, c.lse, part, label_score, c.labels, n, tiles, p.vocab, c.ignore);
    CCT_LAUNCH_CHECK();
  }
  if (!c.backward) return 0;
  const float *lse = c.forward ? c.lse : c.lse_in;
  if (c.dw) {
    vocab_transpose_kernel<T><<<dim3(idiv(p.np, 64), idiv(p.width, 64)), 256, 0, st>>>(
        xt, (const T *)c.x, p.ldx, p.np, n, p.width, p.nk, c.labels, c.ignore);
    CCT_LAUNCH_CHECK();
  }
  for (int v0 = 0; v0 < p.vocab; v0 += p.piece) {
    const int rows = min(p.piece, p.vocab - v0);
    const int mpad = idiv(rows, p.unit / 8) * (p.unit / 8);
    int db_tiles;
    if (keep) {
      vocab_grad_kernel<T><<<dim3(idiv(mpad, 64), idiv(p.np, 64)), 256, 0, st>>>(
          g, gt, (const float *)(c.ws + p.scores), c.db ? db_part : nullptr, c.labels, lse, c.gscale, n, p.vocab, v0, rows,
          c.ignore, p.vp, p.vp, p.np, mpad, p.nk, p.vp);
      CCT_LAUNCH_CHECK();
      db_tiles = idiv(p.np, 64);
    } else {
      ProductArgs a;
      if (int rc = scores_of(v0, rows, a)) return rc;
      a.lse = lse;
      a.gscale = c.gscale;
      a.g = g;
      a.gt = gt;
      a.ldgt = p.np;
      a.mpad = mpad;
      a.npad = p.nk;
      a.db_part = c.db ? db_part : nullptr;
      a.db_ld = p.vp;
      if (int rc = product<T, USE_GRAD>(p.fs, a)) return rc;
      db_tiles = a.tiles_n;
    }
    if (c.db) {
      vocab_db_kernel<T><<<idiv(rows, 256), 256, 0, st>>>((T *)c.db + v0, db_part, rows, p.vp, db_tiles);
      CCT_LAUNCH_CHECK();
    }
    if (c.dx) {
      vocab_transpose_kernel<T><<<dim3(idiv(mpad, 64), idiv(p.width, 64)), 256, 0, st>>>(
          wt, (const T *)c.w + (size_t)v0 * p.ldw, p.ldw, p.vp, rows, p.width, mpad, nullptr, 0);
      CCT_LAUNCH_CHECK();
      ProductArgs a{};
      a.A = (const char *)wt;
      a.lda = p.vp * p.el;
      a.B = (const char *)g;
      a.ldb = p.vp * p.el;
      a.M = p.width;
      a.N = n;
      a.kbytes = (uint32_t)(mpad * p.el);
      a.splits = p.dx_splits;
      a.C = slabs;
      a.accumulate = v0 > 0;
      if (int rc = product<T, USE_SLAB>(p.dxs, a)) return rc;
    }
    if (c.dw) {
      ProductArgs a{};
      a.A = (const char *)xt;
      a.lda = p.np * p.el;
      a.B = (const char *)gt;
      a.ldb = p.np * p.el;
      a.M = p.width;
      a.N = rows;
      a.kbytes = (uint32_t)(p.nk * p.el);
      a.splits = 1;
      a.C = (T *)c.dw + (size_t)v0 * p.ldw;
      a.ldc = p.ldw;
      if (int rc = product<T, USE_OUT>(p.dws, a)) return rc;
    }
  }
  if (c.dx) {
    vocab_dx_kernel<T><<<n, 256, 0, st>>>((T *)c.dx, slabs, c.labels, c.gscale, c.ignore, n, p.width, p.ldx, p.dx_splits);
    CCT_LAUNCH_CHECK();
  }
  return 0;
}

static int check_vocab(const cct_vocab_loss_args *a, const char *who) {
  CCT_REQUIRE(a != nullptr, "%s: null argument block", who);
  CCT_REQUIRE(a->dtype == CCT_F32 || a->dtype == CCT_BF16, "%s: dtype %d is neither CCT_F32 nor CCT_BF16", who, a->dtype);
  CCT_REQUIRE(a->tokens >= 0 && a->width > 0 && a->vocab > 0 && a->piece >= 0, "%s: tokens %d, width %d, vocab %d, piece %d",
              who, a->tokens, a->width, a->vocab, a->piece);
  CCT_REQUIRE(a->tokens <= (1 << 20) && a->width <= (1 << 16) && a->vocab < (1 << 24),
              "%s: tokens %d, width %d, vocab %d: at most 2^20, 2^16, 2^24 - 1", who, a->tokens, a->width, a->vocab);
  CCT_REQUIRE((a->x_stride == 0 || a->x_stride >= (size_t)a->width) && (a->w_stride == 0 || a->w_stride >= (size_t)a->width),
              "%s: a row stride is smaller than the width %d", who, a->width);
  CCT_REQUIRE(a->x_stride <= (1u << 20) && a->w_stride <= (1u << 20), "%s: row strides of at most 2^20 elements", who);
  return 0;
}

static int check_vocab_workspace(const VocabPlan &p, const void *ws, size_t bytes, bool training, const char *who) {
  const size_t need = training ? p.total : p.total_forward;
  CCT_REQUIRE(bytes >= need && (ws || need == 0) && ((uintptr_t)ws & 15) == 0,
              "%s: the workspace holds %zu bytes and starts at %p; it needs %zu, aligned to 16", who, bytes, ws, need);
  return 0;
}

static int vocab_dispatch(const VocabPlan &p, const VocabCall &c) {
  CCT_ENSURE_INIT();
  return p.dtype == CCT_BF16 ? vocab_run<bf16>(p, c) : vocab_run<float>(p, c);
}

// No tokens: the sums over the tokens are zero.
static int vocab_zero_gradients(const VocabPlan &p, void *dw, void *db) {
  CCT_ENSURE_INIT();
  hipStream_t st = ctx().stream;
  if (p.dtype == CCT_BF16) {
    if (dw) vocab_zero_kernel<bf16><<<p.vocab, 256, 0, st>>>((bf16 *)dw, p.ldw, p.width);
    if (db) vocab_zero_kernel<bf16><<<1, 256, 0, st>>>((bf16 *)db, 0, p.vocab);
  } else {
    if (dw) vocab_zero_kernel<float><<<p.vocab, 256, 0, st>>>((float *)dw, p.ldw, p.width);
    if (db) vocab_zero_kernel<float><<<1, 256, 0, st>>>((float *)db, 0, p.vocab);
  }
  CCT_LAUNCH_CHECK();
  return 0;
}

}  // namespace cct

using namespace cct;

extern "C" size_t cct_hip_vocab_loss_workspace_bytes(const cct_vocab_loss_args *args, int training) {
  if (check_vocab(args, "vocab_loss_workspace_bytes")) return 0;
  const VocabPlan p = vocab_plan(args);
  return training ? p.total : p.total_forward;
}

extern "C" int cct_hip_vocab_loss_forward(float *loss, float *lse, const void *x, const void *w, const void *bias,
                                          const int *labels, const cct_vocab_loss_args *args, void *workspace,
                                          size_t workspace_bytes) {
  const char *who = "vocab_loss_forward";
  if (int rc = check_vocab(args, who)) return rc;
  if (args->tokens == 0) return 0;
  CCT_REQUIRE(loss && lse && x && w && labels, "%s: null array", who);
  const VocabPlan p = vocab_plan(args);
  if (int rc = check_vocab_workspace(p, workspace, workspace_bytes, false, who)) return rc;
  VocabCall c{};
  c.loss = loss;
  c.lse = lse;
  c.x = x;
  c.w = w;
  c.bias = bias;
  c.labels = labels;
  c.ignore = args->ignore_label;
  c.ws = (char *)workspace;
  c.forward = true;
  return vocab_dispatch(p, c);
}

extern "C" int cct_hip_vocab_loss_backward(void *dx, void *dw, void *db, const void *x, const void *w, const void *bias,
                                           const int *labels, const float *lse, const float *loss_grad,
                                           const cct_vocab_loss_args *args, void *workspace, size_t workspace_bytes) {
  const char *who = "vocab_loss_backward";
  if (int rc = check_vocab(args, who)) return rc;
  CCT_REQUIRE(dx || dw || db, "%s: no gradient is asked for", who);
  const VocabPlan p = vocab_plan(args);
  if (args->tokens == 0) return vocab_zero_gradients(p, dw, db);
  CCT_REQUIRE(x && w && labels && lse, "%s: null array", who);
  if (int rc = check_vocab_workspace(p, workspace, workspace_bytes, true, who)) return rc;
  VocabCall c{};
  c.lse_in = lse;
  c.dx = dx;
  c.dw = dw;
  c.db = db;
  c.x = x;
  c.w = w;
  c.bias = bias;
  c.labels = labels;
  c.gscale = loss_grad;
  c.ignore = args->ignore_label;
  c.ws = (char *)workspace;
  c.backward = true;
  return vocab_dispatch(p, c);
}

extern "C" int cct_hip_vocab_loss_forward_backward(float *loss, float *lse, void *dx, void *dw, void *db, const void *x,
                                                   const void *w, const void *bias, const int *labels,
                                                   const float *loss_grad, const cct_vocab_loss_args *args,
                                                   void *workspace, size_t workspace_bytes) {
  const char *who = "vocab_loss_forward_backward";
  if (int rc = check_vocab(args, who)) return rc;
  CCT_REQUIRE(dx || dw || db, "%s: no gradient is asked for", who);
  const VocabPlan p = vocab_plan(args);
  if (args->tokens == 0) return vocab_zero_gradients(p, dw, db);
  CCT_REQUIRE(loss && lse && x && w && labels, "%s: null array", who);
  if (int rc = check_vocab_workspace(p, workspace, workspace_bytes, true, who)) return rc;
  VocabCall c{};
  c.loss = loss;
  c.lse = lse;
  c.dx = dx;
  c.dw = dw;
  c.db = db;
  c.x = x;
  c.w = w;
  c.bias = bias;
  c.labels = labels;
  c.gscale = loss_grad;
  c.ignore = args->ignore_label;
  c.ws = (char *)workspace;
  c.forward = c.backward = true;
  return vocab_dispatch(p, c);
}
