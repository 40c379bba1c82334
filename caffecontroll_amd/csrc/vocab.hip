// Vocabulary loss: the softmax loss of an inner-product layer with a large vocabulary of outputs, without its scores.
//
//   l[t][v] = x[t] . w[v] + bias[v]      lse[t] = log sum_v exp l[t][v]      loss[t] = lse[t] - l[t][label[t]]
//   G[t][v] = r[t] * (exp(l[t][v] - lse[t]) - [v == label[t]]),  r[t] = loss_grad[t] / c,  c = max finite |loss_grad|
//   dx[t] = c * sum_v G[t][v] w[v]       dw[v] = c * sum_t G[t][v] x[t]      db[v] = c * sum_t G[t][v]
//
// G is what bf16 products take as an operand, so it is rounded once.  The weights enter it relative to the largest of
// them: equal weights (a mean over tokens) are then exactly 1 and add no rounding of their own, which would be the
// same for every token and not average out.
//
// Every product is one kernel, C[m][n] = sum_k A[m][k] B[n][k], with operands that are contiguous along k or along
// their rows, and four ways to use a finished tile:
//   STATS  m = vocabulary, n = token: maximum and sum of the tile's scores per token (a few bytes instead of the tile) and
//          the label's score;
//   GRAD   the same product again with lse known: G of a piece of the vocabulary and the column sums for db;
//   SLAB   fp32 parts of a result, cut along k and added up by a later kernel: dx over the pieces (m = width, n = token,
//          k = vocabulary), and scores that are kept;
//   OUT    m = width, n = vocabulary, k = token: dw of the piece, stored once in its own type.
//
// The loss of few tokens over rows of odd lengths has a kernel of its own, a walk over w.
//
// Bound: matrix-core rate.  2 tokens*width*vocab operations for the loss, 4 more for the gradients and 2 for the scores
// again where they were not kept.
#include <type_traits>

#include "mfma_common.h"
#include "narrow.h"

namespace cct {

// ---- the product kernel ----------------------------------------------------------------------------------------
// A workgroup owns a BM x BN tile of C and walks k in steps of 64 bf16 or 32 fp32 elements through two LDS stages (four for
// the narrow tile, whose workgroups are often alone on a CU and wait for memory) that global -> LDS copies fill, 1 KB a
// wavefront at a time.
// Fragments of v_mfma_f32_16x16x32_bf16 and v_mfma_f32_16x16x4_f32: lane l holds 16 bytes of row l % 16, elements
// along k of chunk l / 16; C element r of lane l is row 4 * (l / 16) + r, column l % 16.  For fp32 the four elements of a
// chunk feed four MFMAs (the sum over k may run in any order as long as both operands use the same one).
// Bound by the matrix cores and, in bf16, by the clock that their power leaves (1.96 GHz at 60 % MFMA use): 8192 tokens,
// width 4096, pieces of 16384 rows of bf16 run at 1300 (STATS), 1240 (GRAD), 1250 (SLAB) and 1300 TFLOP/s (OUT), where the
// library's 8192^3 product reaches 1284; 2048 tokens, width 2048, 32768 rows of fp32 at 143 TFLOP/s (library 153).
enum Use { USE_STATS = 0, USE_GRAD = 1, USE_SLAB = 2, USE_OUT = 3 };

template <int BM_, int BN_, int WM_, int WN_, int STAGES_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;  // 16 x 16 blocks of a wavefront
  static constexpr int STAGE = (BM + BN) * 128;               // bytes
  static_assert(BM % (WM * 16) == 0 && BN % (WN * 16) == 0, "wavefront tiles are whole blocks");
  static_assert(WAVES % 2 == 0, "the swizzle of a lane's copies relies on an even number of wavefronts");
};

typedef __attribute__((address_space(3))) char lds_char;

// 16 bytes a lane from global memory into LDS: lane l's land at dst + 16 l; an offset past the descriptor's 2^31 bytes fetches
// nothing and writes zeros.  The instruction itself instead of its builtin: the compiler would wait for all copies
// in flight before every ds_read_b64_tr_b16, whose address it cannot tell from theirs (a product with such an operand: 1.43
// instead of 0.83 ms).  It has no result register; copy_wait() and a barrier stand before the reads that need it.  M0 holds
// the LDS address; the compiler's warning that it keeps M0 for itself is why the asm says that it writes it.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy16(const char *base, uint32_t lane_offset, uint32_t offset, lds_char *dst) {
  const uint64_t at = (uint64_t)base;
  const u32x4 rsrc = {(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, kOutOfRange, 0x00020000u};
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"((uint32_t)(uintptr_t)dst),
      "v"(lane_offset), "s"(rsrc), "s"(offset)
      : "memory", "m0");
}
#pragma clang diagnostic pop
// all but the last N copies of this wavefront have landed
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// One operand's tile of R rows: its copies into LDS and its fragments.
//
// Contiguous along k (KC): an LDS row is 128 bytes of one operand row; 16-byte chunk c of row r lies in slot
// c ^ ((r >> 1) & 7), so that the 16 lanes of a fragment read (16 rows, one chunk) touch all 64 banks once.
//
// Contiguous along the rows: an LDS row holds the R elements of one k.  bf16 fragments come from ds_read_b64_tr_b16, which
// gives lane l four elements along k of column l % 16 out of the 4 x 16 elements that its group of 16 lanes points
// at; fp32 fragments from single words.  32-byte pairs (bf16; 64-byte granules for fp32) of an LDS row are permuted by
// k so that the eight k a half wavefront reads at once (four for fp32) lie in different banks.
//
// A copy cannot permute what a lane receives, so the lane that fills a slot fetches the chunk that belongs there.
template <class T, int R, int WAVES, bool KC>
struct Operand {
  static constexpr int J = R / 8 / WAVES;          // copies of a wavefront per step
  static constexpr int KS = 128 / (int)sizeof(T);  // k of a step
  static constexpr int ROWB = R * (int)sizeof(T);  // bytes of an LDS row when contiguous along the rows
  static_assert(J * 8 * WAVES == R, "whole copies");
  static_assert(KC || R >= 64, "an LDS row holds the banks' permutation");

  const char *base;
  size_t step_bytes;
  uint32_t offset[J];
  uint32_t chunk;  // KC: byte of this lane's chunk within a step
  int krow;        // else: k of this lane's first copy within a step

  static __device__ __forceinline__ int swizzle(int k) {
    if (sizeof(T) == 4) return ((k >> 2) & 3) << 2;
    return R >= 128 ? ((k & 3) | ((k >> 3) & 1) << 2) << 1 : (((k >> 1) & 1) | ((k >> 3) & 1) << 1) << 1;
  }

  // rows [r0, ...) of an operand of `rows` rows, `ld` bytes apart along its slow direction; `row_bytes`: what may be read
  // of that many bytes along the fast one when contiguous along the rows
  __device__ __forceinline__ void init(const char *p, size_t ld, int r0, int rows, uint32_t row_bytes, int wave, int lane) {
    if constexpr (KC) {
      base = p + (size_t)r0 * ld;
      step_bytes = 128;
      const int row = wave * 8 + (lane >> 3);
      chunk = ((uint32_t)(lane & 7) ^ ((uint32_t)(row >> 1) & 7u)) * 16u;
      // rows past the end repeat the last one: their results are never used
#pragma unroll
      for (int j = 0; j < J; ++j) offset[j] = (uint32_t)min(row + j * WAVES * 8, rows - 1 - r0) * (uint32_t)ld + chunk;
    } else {
      base = p + (size_t)r0 * sizeof(T);
      step_bytes = (size_t)KS * ld;
      const int at = wave * 1024 + lane * 16;
      krow = at / ROWB;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int k = krow + j * (WAVES * 1024 / ROWB);
        const uint32_t c = (uint32_t)(((at % ROWB) >> 4) ^ swizzle(k)) * 16u;
        offset[j] = (uint32_t)r0 * (uint32_t)sizeof(T) + c < row_bytes ? (uint32_t)k * (uint32_t)ld + c : kOutOfRange;
      }
    }
  }

  // copy j of step `step` into LDS at `dst`; what lies past the end of k becomes zero
  __device__ __forceinline__ void copy(lds_char *dst, int j, int step, int K, uint32_t kbytes, int wave) const {
    lds_char *to = dst + wave * 1024 + j * WAVES * 1024;
    if constexpr (KC) {
      const uint32_t k = (uint32_t)step * 128u;
      copy16(base, k + chunk < kbytes ? offset[j] : kOutOfRange, k, to);
    } else {
      const int left = K - step * KS;
      copy16(base + (size_t)step * step_bytes, krow + j * (WAVES * 1024 / ROWB) < left ? offset[j] : kOutOfRange, 0, to);
    }
  }

  // byte offsets of this lane's part of block b (16 rows), without the step's k
  static __device__ __forceinline__ int frag_offset(int b, int lane) {
    const int row = lane & 15, g = lane >> 4;
    if (KC) return (b * 16 + row) * 128 + ((g ^ ((row >> 1) & 7)) * 16);
    if (sizeof(T) == 4) return g * 4 * ROWB + ((b ^ g) << 6) + row * 4;
    const int k = g * 8 + (row >> 2);
    return k * ROWB + (((b << 1) ^ swizzle(k)) << 4) + (row & 3) * 8;
  }
  // the 16 bytes of half step `sub`; at = stage + frag_offset
  static __device__ __forceinline__ f32x4 fragment(lds_char *tile, int at, int sub) {
    typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    typedef __attribute__((address_space(3))) float lds_float;
    if constexpr (KC) {
      return *(lds_f32x4 *)(tile + (at ^ (sub * 64)));
    } else if constexpr (sizeof(T) == 4) {
      f32x4 f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = *(lds_float *)(tile + at + (sub * 16 + e) * ROWB);
      return f;
    } else {
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + at + sub * 32 * ROWB));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + at + (sub * 32 + 4) * ROWB));
      return __builtin_bit_cast(f32x4, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

struct ProductArgs {
  const char *A, *B;
  size_t lda, ldb;  // bytes between rows (between k for operands contiguous along the rows)
  int M, N, K;
  uint32_t kbytes;          // operands contiguous along k: bytes of a row that take part, a multiple of 16
  uint32_t abytes, bbytes;  // operands contiguous along the rows: bytes of one k that may be read, multiples of 16
  int tiles_m, tiles_n, splits, steps_per_split;
  uint32_t blocks;
  // STATS, GRAD (m = rows v0 + m of the vocabulary, n = token)
  const void *bias;          // of the piece's first row, or null
  const int *labels;
  int v0, ignore;
  SoftStat *part;            // STATS: [tile of the whole vocabulary][token]
  int part_row;              // first tile of the piece
  float *label_score;        // STATS: [token]
  const float *lse, *weight, *wmax;  // GRAD; weight: loss_grad or null, wmax: its largest finite magnitude
  void *g;                   // GRAD: [token][ldg]
  size_t ldg;                // elements
  int mpad;                  // GRAD: columns of g, whole 16-byte chunks (those past M are zero)
  float *db_part;            // GRAD: [tile_n][row of the piece] or null
  int db_ld;
  // SLAB: C [split][N][ldc] fp32.  OUT: C [n][ldc] elements, times *wmax
  void *C;
  size_t ldc;
  int accumulate;
  // OUT: rows are whole cache lines, written past the caches (512 tokens, 32000 rows of 2048 bf16: 80 -> 74 us; rows of 776,
  // whose lines are written in parts: 37 -> 44)
  int stream;
};

__device__ __forceinline__ f32x4 mfma_bf16(const f32x4 &a, const f32x4 &b, const f32x4 &c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A token's part in the gradient.  Ignored tokens have no part: their G is 0 whatever their scores are.
struct TokenGrad {
  int label;
  float lse, weight;
  bool live;
};
__device__ __forceinline__ TokenGrad token_grad(int t, int tokens, const int *__restrict__ labels, int ignore,
                                                const float *__restrict__ lse, const float *__restrict__ weight,
                                                const float *__restrict__ wmax) {
  TokenGrad g{-1, 0.0f, 0.0f, false};
  if (t < tokens) {
    g.label = labels[t];
    g.live = g.label != ignore;
    g.lse = lse[t];
    g.weight = weight ? weight[t] / *wmax : 1.0f;
  }
  return g;
}
// A large score that was computed in another order than the lse's may lie above it by its own rounding: p is cut at one (NaN
// stays).
__device__ __forceinline__ float probability_cut(float score, float lse) {
  const float e = (score - lse) * kLog2e;
  return exp2_fast(e > 0.0f ? 0.0f : e);
}
__device__ __forceinline__ float grad_entry(float score, const TokenGrad &tg, bool is_label) {
  const float p = probability_cut(score, tg.lse);
  return tg.live ? tg.weight * (p - (is_label ? 1.0f : 0.0f)) : 0.0f;
}

// Sum over the 16 lanes of a row of lanes, in all of them (rotations by 8, 4, 2, 1 within the row).
template <int ROT>
__device__ __forceinline__ float row_rotate(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + ROT, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_sum16(float v) {
  v += row_rotate<8>(v);
  v += row_rotate<4>(v);
  v += row_rotate<2>(v);
  return v + row_rotate<1>(v);
}

// Four consecutive elements, of which those below `left` exist.
template <class T>
__device__ __forceinline__ void store4(T *p, const float (&f)[4], int left) {
  typedef T vec4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (left >= 4) {
    vec4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (T)f[i];
    *reinterpret_cast<vec4 *>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = (T)f[i];
  }
}

template <class T, class S, int USE, bool KA, bool KB>
__global__ __launch_bounds__(S::THREADS) void vocab_product_kernel(ProductArgs p) {
  extern __shared__ __align__(16) char lds[];
  typedef Operand<T, S::BM, S::WAVES, KA> OpA;
  typedef Operand<T, S::BN, S::WAVES, KB> OpB;
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

  OpA opa;
  OpB opb;
  opa.init(p.A, p.lda, m0, p.M, p.abytes, wave, lane);
  opb.init(p.B, p.ldb, n0, p.N, p.bbytes, wave, lane);

  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  int fa[MI], fb[NI];
#pragma unroll
  for (int i = 0; i < MI; ++i) fa[i] = OpA::frag_offset(wm * MI + i, lane);
#pragma unroll
  for (int j = 0; j < NI; ++j) fb[j] = OpB::frag_offset(wn * NI + j, lane);

  const int steps = (p.K + OpA::KS - 1) / OpA::KS;
  const int s0 = (int)split * p.steps_per_split, s1 = min(steps, s0 + p.steps_per_split);
  // what lies past this workgroup's part of k counts as past the end: such copies fetch nothing and only keep the count
  const int K = min(p.K, s1 * OpA::KS);
  const uint32_t kbytes = min(p.kbytes, (uint32_t)s1 * 128u);
  constexpr int COPIES = OpA::J + OpB::J;
  auto copy = [&](int c, int buf, int step) {
    lds_char *t = (lds_char *)lds + buf * S::STAGE;
    if (c < OpA::J)
      opa.copy(t, c, step, K, kbytes, wave);
    else
      opb.copy(t + S::BM * 128, c - OpA::J, step, K, kbytes, wave);
  };
  auto stage = [&](int buf, int step) {
#pragma unroll
    for (int c = 0; c < COPIES; ++c) copy(c, buf, step);
  };
  if constexpr (std::is_same<T, float>::value) {
    // fp32: a step's MFMAs take eight times as long as its reads; one barrier per step and the compiler's own order (with
    // the phases below: 4 to 6 % slower).  The four MFMAs of a chunk go round the blocks: neighbours in time do not wait for
    // one another's accumulator (1 % against four in a row).
    if (s0 < s1) {
#pragma unroll
      for (int i = 0; i + 1 < S::STAGES; ++i) stage(i, s0 + i);
    }
    int buf = 0, fill = S::STAGES - 1;
    for (int s = s0; s < s1; ++s) {
      copy_wait<(S::STAGES - 2) * COPIES>();
      __syncthreads();
      stage(fill, s + S::STAGES - 1);
      lds_char *ta = (lds_char *)lds + buf * S::STAGE, *tb = ta + S::BM * 128;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        f32x4 a[MI], b[NI];
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = OpA::fragment(ta, fa[i], sub);
#pragma unroll
        for (int j = 0; j < NI; ++j) b[j] = OpB::fragment(tb, fb[j], sub);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][e], b[j][e], acc[i][j], 0, 0, 0);
      }
      fill = buf;
      buf = buf + 1 == S::STAGES ? 0 : buf + 1;
    }
  } else {
    // A step is cut into phases of MH x NI blocks; while one phase's MFMAs run, the next one's fragments are read.  The last
    // phase of a step reads the next stage, so the barrier stands before it: every wavefront then has all it needs of
    // this stage in registers, and copies may overwrite it.  Reads and copies stand between the MFMAs in the order of the
    // source, so that neither unit gets a burst that holds the other up.
    constexpr int MH = MI % 2 == 0 ? MI / 2 : MI, H = MI / MH, PHASES = 2 * H, MFMAS = MH * NI;
    f32x4 a[2][MH], b[2][NI];
    auto read = [&](int item, int to, int buf, int sub, int h) {  // items 0..MH-1: A, then B
      lds_char *t = (lds_char *)lds + buf * S::STAGE;
      if (item < MH)
        a[to][item] = OpA::fragment(t, fa[h * MH + item], sub);
      else
        b[sub][item - MH] = OpB::fragment(t + S::BM * 128, fb[item - MH], sub);
    };
    if (s0 < s1) {
#pragma unroll
      for (int i = 0; i < S::STAGES; ++i) stage(i, s0 + i);
      copy_wait<(S::STAGES - 1) * COPIES>();
      __syncthreads();
#pragma unroll
      for (int i = 0; i < MH + NI; ++i) read(i, 0, 0, 0, 0);
    }
    int buf = 0;
    for (int s = s0; s < s1; ++s) {
      const int next = buf + 1 == S::STAGES ? 0 : buf + 1;
#pragma unroll
      for (int q = 0; q < PHASES; ++q) {
        const bool last = q + 1 == PHASES;
        const int sub = q / H, h = q % H, nsub = last ? 0 : (q + 1) / H, nh = last ? 0 : (q + 1) % H;
        if (last) {
          copy_wait<(S::STAGES - 2) * COPIES>();
          __syncthreads();
        }
        const int reads = MH + (nh == 0 ? NI : 0), copies = last ? COPIES : 0, items = reads + copies;
#pragma unroll
        for (int m = 0; m < MFMAS; ++m) {
#pragma unroll
          for (int it = 0; it < items; ++it) {
            if (it * MFMAS / items != m) continue;
            // the last phase alternates between copies and reads (what is read behind the last step is not used)
            const bool paired = it < 2 * min(copies, reads);
            const int c = !last ? -1 : paired ? ((it & 1) ? -1 : it / 2) : copies > reads ? it - reads : -1;
            const int r = !last ? it : paired ? it / 2 : it - copies;
            if (c >= 0)
              copy(c, buf, s + S::STAGES);
            else
              read(r, (q + 1) & 1, last ? next : buf, nsub, nh);
          }
          const int i = m / NI, j = m % NI;
          acc[h * MH + i][j] = mfma_bf16(a[q & 1][i], b[sub][j], acc[h * MH + i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      buf = next;
    }
  }
  copy_wait<0>();  // no copy may land after this workgroup's use of its LDS

  // this lane's elements: rows mrow + 16 i + r, columns ncol + 16 j
  const int fgroup = lane >> 4, frow = lane & 15;
  const int mrow = m0 + wm * MI * 16 + fgroup * 4, ncol = n0 + wn * NI * 16 + frow;

  // The epilogues' exponents are score * log2 e - base * log2 e in one instruction, whose second product is rounded once for
  // all rows.  That rounding moves every exponent by up to 2^-24 of the product, 0.09 at this bound; scores past it are
  // subtracted first.  (Without a bound the largest score's own power leaves the type's range from 2e9 on.)
  constexpr float kScaledMax = 1 << 20;
  // bf16 rows leave through LDS, so that a store has up to 256 bytes of one, 16 a lane, instead of 32 with 8 straight from
  // the accumulators (dw of 64 tokens of 2048, 32000 rows: 51 -> 38 us; G of the largest step: 26.8 -> 26.65 ms in all).  A
  // wavefront takes its own part of the stages, as many rows at a time as it holds; the 16-byte chunks lie swizzled by the
  // row.  (fp32 stores have 16 bytes a lane as it is: no gain.)
  const auto store_rows = [&](bf16 *C, size_t ld, int cols) {
    typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
    typedef Num<bf16>::vec chunk_any;
    constexpr int ROW = MI * 16, CR = ROW / 8, ROWBYTES = ROW * 2;
    constexpr int AREA = S::STAGES * S::STAGE / S::WAVES, FIT = AREA / (16 * ROWBYTES), JP = FIT < NI ? FIT : NI;
    static_assert(JP >= 1 && NI % JP == 0 && 64 % CR == 0, "a wavefront's rows have to fit its part of the stages");
    const auto swizzle = [](int row) { return CR >= 16 ? row & 15 : (row & 15) / (16 / CR); };
    lds_char *area = (lds_char *)lds + wave * AREA;
    const int c = lane % CR, m = m0 + wm * ROW + c * 8, left = cols - m;
#pragma unroll
    for (int j0 = 0; j0 < NI; j0 += JP) {
#pragma unroll
      for (int j = j0; j < j0 + JP; ++j)
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const int chunk = (2 * i + fgroup / 2) ^ swizzle(frow);
          bf16x4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = (bf16)acc[i][j][r];
          const int at = ((j - j0) * 16 + frow) * ROWBYTES + chunk * 16 + fgroup % 2 * 8;
          *(__attribute__((address_space(3))) bf16x4 *)(area + at) = v;
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
      for (int r = lane / CR; r < JP * 16; r += 64 / CR) {
        const int n = n0 + (wn * NI + j0) * 16 + r;
        const bf16x8 v = *(__attribute__((address_space(3))) bf16x8 *)(area + r * ROWBYTES + (c ^ swizzle(r)) * 16);
        if (n >= p.N || left <= 0) continue;
        bf16 *to = C + (size_t)n * ld + m;
        if (left >= 8) {
          if (USE == USE_OUT && p.stream)
            __builtin_nontemporal_store((chunk_any)v, (chunk_any *)to);
          else
            *(chunk_any *)to = v;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < left) to[e] = v[e];
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  };

  if constexpr (USE == USE_STATS || USE == USE_GRAD) {
    __syncthreads();  // the stages are done with
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
    if (m0 + S::BM > p.M) {  // rows past the piece have no part in any sum
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (mrow + i * 16 + r >= p.M)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j][r] = neg_inf();
    }
  }

  if constexpr (USE == USE_STATS) {
    SoftStat *sh = (SoftStat *)lds;  // [WM][BN]
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int t = ncol + j * 16;
      const int label = t < p.N ? p.labels[t] : -1;
      // the label among this lane's rows: 16 i + r, or out of their range
      const int at = label >= p.v0 && label < p.v0 + p.M ? label - p.v0 - mrow : -1;
      const bool here = at >= 0 && at < MI * 16 && (at & 15) < 4;
      SoftStat st{neg_inf(), 0.0f};
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.m = fmaxf(st.m, acc[i][j][r]);
      if (__any(here)) {  // few of a wavefront's tokens have their label among its rows
        float score = 0.0f;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) score = at == i * 16 + r ? acc[i][j][r] : score;
        if (here) p.label_score[t] = score;
      }
      const float base = st.m == neg_inf() ? 0.0f : st.m;
      if (MI == 1 || __any(fabsf(base) > kScaledMax)) {  // (four scores: the correction below costs more than it saves)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) st.s += exp2_fast((acc[i][j][r] - base) * kLog2e);
      } else {
        const float scaled = base * kLog2e;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) st.s += exp2_fast(__builtin_fmaf(acc[i][j][r], kLog2e, -scaled));
        st.s *= exp2_fast(-__builtin_fmaf(base, kLog2e, -scaled));  // the rounding of `scaled`, the same in every term
      }
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
    float *sums = (float *)lds;  // [WN][BM] column sums for db
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int t = ncol + j * 16;
      const TokenGrad tg = token_grad(t, p.N, p.labels, p.ignore, p.lse, p.weight, p.wmax);
      const int at = tg.label >= p.v0 && tg.label < p.v0 + p.M ? tg.label - p.v0 - mrow : -1;
      if (__any(fabsf(tg.lse) > kScaledMax)) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] = probability_cut(acc[i][j][r], tg.lse);
      } else {
        const float scaled = tg.lse * kLog2e;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] = exp2_fast(__builtin_fmaf(acc[i][j][r], kLog2e, -scaled));
      }
      if (__any(at >= 0 && at < MI * 16 && (at & 15) < 4)) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] -= at == i * 16 + r ? 1.0f : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int m = mrow + i * 16;
        float g[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          g[r] = tg.live ? tg.weight * acc[i][j][r] : 0.0f;
          acc[i][j][r] = g[r];
        }
        if (sizeof(T) == 4 && t < p.N && m < p.mpad) store4<T>((T *)p.g + (size_t)t * p.ldg + m, g, 4);
      }
    }
    if constexpr (sizeof(T) == 2) {
      store_rows((T *)p.g, p.ldg, p.mpad);
      __syncthreads();
    }
    if (p.db_part) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float row = acc[i][0][r];
#pragma unroll
          for (int j = 1; j < NI; ++j) row += acc[i][j][r];
          row = row_sum16(row);
          if (frow == 0) sums[wn * S::BM + (wm * MI + i) * 16 + fgroup * 4 + r] = row;
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
    const float scale = USE == USE_OUT && p.wmax ? *p.wmax : 1.0f;
    if constexpr (USE == USE_OUT) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] *= scale;
    }
    if constexpr (sizeof(Out) == 2) {
      __syncthreads();  // the stages are done with
      store_rows((Out *)p.C, p.ldc, p.M);
    } else {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int n = ncol + j * 16;
        if (n >= p.N) continue;
        Out *row = (Out *)p.C + (USE == USE_SLAB ? ((size_t)split * p.N + n) * p.ldc : (size_t)n * p.ldc);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const int m = mrow + i * 16, left = p.M - m;
          if (left <= 0) continue;
          float f[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f[r] = acc[i][j][r];
            if (USE == USE_SLAB && p.accumulate && r < left) f[r] += (float)row[m + r];
          }
          store4<Out>(row + m, f, left);
        }
      }
    }
  }
}

// ---- copies and statistics before the products ---------------------------------------------------------------------
// dst[r][c] = src[r][c], rows of dst filled up to cpad with zeros: operands whose rows do not start at 16-byte
// boundaries or are no whole number of 16-byte chunks.  Rows [0, rows) of one matrix, then those of another; the lanes of
// a workgroup are laid over (row, vector).  HBM: 16 us for 118050 rows of 119 bf16 (58 MB; 80 us with a workgroup a row).
template <class T>
__global__ __launch_bounds__(256) void vocab_pack_kernel(T *__restrict__ dst, const T *__restrict__ src, size_t ld_src,
                                                         int rows, T *__restrict__ dst2, const T *__restrict__ src2,
                                                         size_t ld_src2, int rows2, int cols, int cpad, int log_lanes) {
  constexpr int V = Num<T>::V;
  const int lanes = 1 << log_lanes;
  int r = blockIdx.x * (256 >> log_lanes) + (threadIdx.x >> log_lanes);
  if (r >= rows + rows2) return;
  const bool second = r >= rows;
  if (second) r -= rows;
  const T *from = second ? src2 + (size_t)r * ld_src2 : src + (size_t)r * ld_src;
  T *to = (second ? dst2 : dst) + (size_t)r * cpad;
  for (int c = (threadIdx.x & (lanes - 1)) * V; c < cpad; c += lanes * V) {
    float f[V];
    load_vec<T>(f, from, c, cols);
    store_vec<T>(to, f, c, cpad);
  }
}

// The largest magnitude among the finite weights of the tokens that are not ignored, by one workgroup; 1 where none is above
// zero.  It divides every token's weight and multiplies every result, so a weight that is NaN or infinite has no say in it:
// such a weight stays what it is, in its own token's G.
__device__ __forceinline__ void largest_weight(float *__restrict__ wmax, float *sh, const float *__restrict__ weight,
                                               const int *__restrict__ labels, int tokens, int ignore) {
  float m = 0.0f;
  for (int t = threadIdx.x; t < tokens; t += 256) {
    const float w = fabsf(weight[t]);
    if (labels[t] != ignore && w < __builtin_inff()) m = fmaxf(m, w);
  }
  sh[threadIdx.x] = m;
  __syncthreads();
  for (int d = 128; d > 0; d >>= 1) {
    if ((int)threadIdx.x < d) sh[threadIdx.x] = fmaxf(sh[threadIdx.x], sh[threadIdx.x + d]);
    __syncthreads();
  }
  if (threadIdx.x == 0) *wmax = sh[0] > 0.0f ? sh[0] : 1.0f;
}

// x as dw's operand, zero for ignored tokens, so that whatever their x holds stays out of the product.  bf16: transposed,
// xt[c][t] = x[t][c] for t < tpad (zero past the end), since a transposed read of both operands from LDS is slower than
// of one.  fp32: xl[t][c] for c < cpad.  With weights, one workgroup more takes the largest of them.  HBM, and a few
// microseconds beside the products: 42 us for 8192 x 4096 bf16 transposed, 9 us for 2048 x 1024 fp32.
template <class T>
__global__ __launch_bounds__(256) void vocab_live_kernel(T *__restrict__ xl, const T *__restrict__ x, size_t ldx, int tokens,
                                                         int width, int cpad, const int *__restrict__ labels, int ignore,
                                                         const float *__restrict__ weight, float *__restrict__ wmax) {
  constexpr int V = Num<T>::V;
  __shared__ float sh[256];
  const int t = blockIdx.x;
  if (t == tokens) return largest_weight(wmax, sh, weight, labels, tokens, ignore);
  const bool live = labels[t] != ignore;
  for (int c = threadIdx.x * V; c < cpad; c += 256 * V) {
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = 0.0f;
    if (live) load_vec<T>(f, x + (size_t)t * ldx, c, width);
    store_vec<T>(xl + (size_t)t * cpad, f, c, cpad);
  }
}
template <class T>
__global__ __launch_bounds__(256) void vocab_xt_kernel(T *__restrict__ xt, const T *__restrict__ x, size_t ldx, size_t ldt,
                                                       int tokens, int width, int tpad, int tiles_t,
                                                       const int *__restrict__ labels, int ignore,
                                                       const float *__restrict__ weight, float *__restrict__ wmax,
                                                       int tiles) {
  __shared__ T tile[64][64 + 4 / sizeof(T)];
  if ((int)blockIdx.x == tiles) {
    largest_weight(wmax, (float *)tile, weight, labels, tokens, ignore);
    return;
  }
  const int t0 = (int)(blockIdx.x % tiles_t) * 64, c0 = (int)(blockIdx.x / tiles_t) * 64;
  const int lane = threadIdx.x & 63, y = threadIdx.x >> 6;
  int label[16];
  T v[16];
  const int c = min(c0 + lane, width - 1);
#pragma unroll
  for (int i = 0; i < 16; ++i) label[i] = labels[min(t0 + y + i * 4, tokens - 1)];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = x[(size_t)min(t0 + y + i * 4, tokens - 1) * ldx + c];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    tile[y + i * 4][lane] = t0 + y + i * 4 < tokens && c0 + lane < width && label[i] != ignore ? v[i] : (T)0.0f;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = c0 + y + i * 4, t = t0 + lane;
    if (c < width && t < tpad) xt[(size_t)c * ldt + t] = tile[lane][y + i * 4];
  }
}

// ---- joining -----------------------------------------------------------------------------------------------------
// lse is one float, off by 2^-24 of the largest score; the loss is formed from the statistics, so that the loss of a confident
// token, or of one whose every score is near the type's lowest value, is not lost in that.
__device__ __forceinline__ float store_loss(float *__restrict__ loss, float *__restrict__ lse, int t, SoftStat st, int label,
                                            float score, int vocab, int ignore) {
  const float l = log_sum(st, 1.0f);
  lse[t] = l;
  loss[t] = label == ignore ? 0.0f : (unsigned)label < (unsigned)vocab ? label_loss(st, score, 1.0f) : __builtin_nanf("");
  return l;
}

// The tiles' statistics of each token: 16 tokens per workgroup, 16 lanes each taking every 16th tile (many tokens), or one
// token per workgroup (few tokens, so that the launch is not one workgroup's walk over the tiles: 4 instead of 11 us for 16
// tokens and 500 tiles).  8192 tokens, 512 tiles: 8 us, 4.2 TB/s.
template <int TOK>
__global__ __launch_bounds__(256) void vocab_loss_kernel(float *__restrict__ loss, float *__restrict__ lse,
                                                         const SoftStat *__restrict__ part,
                                                         const float *__restrict__ label_score,
                                                         const int *__restrict__ labels, int tokens, int tiles, int vocab,
                                                         int ignore) {
  constexpr int LANES = 256 / TOK;
  __shared__ SoftStat sh[LANES][TOK + 1];
  const int x = threadIdx.x % TOK, y = threadIdx.x / TOK, t = blockIdx.x * TOK + x;
  SoftStat st{neg_inf(), 0.0f};
  if (t < tokens) {
    int i = y;
    for (; i + 7 * LANES < tiles; i += 8 * LANES) {  // eight loads in flight
      SoftStat v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[(size_t)(i + k * LANES) * tokens + t];
#pragma unroll
      for (int k = 0; k < 8; ++k) st = join(st, v[k], kLog2e);
    }
    for (; i < tiles; i += LANES) st = join(st, part[(size_t)i * tokens + t], kLog2e);
  }
  sh[y][x] = st;
  __syncthreads();
  for (int d = LANES / 2; d > 0; d >>= 1) {
    if (y < d) sh[y][x] = join(sh[y][x], sh[y + d][x], kLog2e);
    __syncthreads();
  }
  if (y == 0 && t < tokens)
    store_loss(loss, lse, t, sh[0][x], labels[t], label_score[t], vocab, ignore);
}

// The loss of at most 64 tokens where w's rows would have to be packed first: one walk over w, its rows as they lie, bound by
// reading them.  A wave takes 16 rows: lane l reads 16 bytes of row l & 15 and has with them its operand of a matrix
// instruction, against the tokens' x, which lie in LDS in the order of that operand: all of them, or panel by panel of the
// width with up to four times 16 rows a wave for each.  With few rows `split` waves share them, each a range of the width, and
// the first one adds the sums up in order.  A lane keeps the running statistics of its token.  The chunk that holds a row's
// end is the row's last 16 bytes, where those that the chunk before has too count as zero: no load has a branch
// around it.  bf16, 2 tokens: 118050 rows of 119 in 13.6 us (30.7 with packing and the tiles above), 131071 rows of 4095 in 222
// us, 4.8 TB/s (585); 64 tokens: 298 us (665).  fp32, 131071 rows of 4095: 2 tokens 367 us (1218), 64 tokens 722 us (1390).
constexpr int kFewTokens = 64, kFewWaves = 8;
// 16 bytes of a row of any alignment.  bf16 rows of odd lengths start between dwords, and 16 rows' 16-byte loads at such
// addresses take twice the time of dword-aligned ones: those five dwords are read that hold the elements, and shifted.
struct RowBytes {
  uint32_t d[5], odd;
};
template <class T>
__device__ __forceinline__ RowBytes row_load(const T *p) {
  typedef u32x4 __attribute__((aligned(4))) u32x4_dword;
  RowBytes b;
  b.odd = sizeof(T) == 2 ? (uint32_t)(uintptr_t)p & 2 : 0;
  const uint32_t *q = (const uint32_t *)((const char *)p - b.odd);
  const u32x4 v = *(const u32x4_dword *)q;
#pragma unroll
  for (int i = 0; i < 4; ++i) b.d[i] = v[i];
  b.d[4] = sizeof(T) == 2 ? q[b.odd ? 4 : 3] : 0;  // none past the elements' own dwords
  return b;
}
template <class T>
__device__ __forceinline__ auto row_value(const RowBytes &b) {
  typedef T vecT __attribute__((ext_vector_type(Num<T>::V)));
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = sizeof(T) == 2 ? __builtin_amdgcn_alignbit(b.d[i + 1], b.d[i], b.odd * 8) : b.d[i];
  return __builtin_bit_cast(vecT, v);
}
constexpr int kFewLds = 144 << 10, kFewPanel = 64 << 10;  // x in LDS: all of it, or by panels
constexpr int kFewRows = 4;                               // tiles of a wave for each staging of a panel
struct FewShape {
  int split;        // waves that share rows
  int panel, rows;  // steps of the width in LDS, tiles of a wave where that is less than all of them
};
template <class T, int NT, bool PANELS>
__global__ __launch_bounds__(kFewWaves * 64) void vocab_few_kernel(SoftStat *__restrict__ part,
                                                                   float *__restrict__ label_score,
                                                                   const T *__restrict__ x, const T *__restrict__ w,
                                                                   const T *__restrict__ bias,
                                                                   const int *__restrict__ labels, size_t ldx, size_t ldw,
                                                                   int tokens, int width, int vocab, FewShape shape) {
  constexpr int V = Num<T>::V, K = 4 * V, R = PANELS ? kFewRows : 1;
  typedef T vecT __attribute__((ext_vector_type(V)));
  extern __shared__ __align__(16) char lds[];
  const int steps = (width + K - 1) / K, split = PANELS ? 1 : shape.split;
  vecT *xs = (vecT *)lds;                                         // [step of the panel][16 tokens][lane]
  f32x4 *sums = (f32x4 *)(xs + (size_t)shape.panel * NT * 64);    // [wave][16 tokens][lane], where waves share rows
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const auto stage = [&](int first, int count) {
    for (int i = tid; i < count * NT * 64; i += kFewWaves * 64) {
      const int l = i & 63, t = (i >> 6) % NT * 16 + (l & 15), col = (first + (i >> 6) / NT) * K + (l >> 4) * V;
      const int from = min(col, width - V);
      const vecT raw = row_value<T>(row_load(x + (size_t)min(t, tokens - 1) * ldx + from));
      vecT v;
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = t < tokens && from + e >= col ? raw[e] : (T)0.0f;
      xs[i] = v;
    }
  };
  if (!PANELS) {
    stage(0, steps);
    __syncthreads();
  }
  const int group = wave / split, share = wave % split;
  const int rows = PANELS ? shape.rows : 1, stride = kFewWaves / split * rows;  // tiles of a wave, of a workgroup
  const int per = (steps + split - 1) / split;
  const int tiles = (vocab + 15) / 16;
  SoftStat st[NT];
  int label[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    st[n] = SoftStat{neg_inf(), 0.0f};
    label[n] = n * 16 + (lane & 15) < tokens ? labels[n * 16 + (lane & 15)] : -1;
  }
  for (int first = (int)blockIdx.x * stride; first < tiles; first += (int)gridDim.x * stride) {
    const int tile0 = first + group * rows;
    f32x4 sum[R][NT];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) sum[i][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = 0; p0 < steps; p0 += shape.panel) {
      if (PANELS) {
        __syncthreads();  // the panel before has been used
        stage(p0, min(shape.panel, steps - p0));
        __syncthreads();
      }
      const int k0 = PANELS ? p0 : share * per, k1 = min(steps, PANELS ? p0 + shape.panel : k0 + per);
      const int whole = min(k1, steps - 1);  // steps before the one that holds the rows' end
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (i >= rows) break;
        const T *row = w + (size_t)min((tile0 + i) * 16 + (lane & 15), vocab - 1) * ldw;
        const auto multiply = [&](vecT a, int k) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const vecT b = xs[((k - (PANELS ? p0 : 0)) * NT + n) * 64 + lane];
            if constexpr (sizeof(T) == 2) {
              sum[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, sum[i][n], 0, 0, 0);
            } else {
#pragma unroll
              for (int e = 0; e < V; ++e)
                sum[i][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], sum[i][n], 0, 0, 0);
            }
          }
        };
        const T *at = row + (lane >> 4) * V;
        constexpr int AHEAD = 8;
        int k = k0;
        for (; k + AHEAD <= whole; k += AHEAD) {
          RowBytes a[AHEAD];
#pragma unroll
          for (int j = 0; j < AHEAD; ++j) a[j] = row_load(at + (k + j) * K);
          __builtin_amdgcn_sched_barrier(0);  // all of them are in flight before the first is used
#pragma unroll
          for (int j = 0; j < AHEAD; ++j) multiply(row_value<T>(a[j]), k + j);
        }
        for (; k < whole; ++k) multiply(row_value<T>(row_load(at + k * K)), k);
        if (k0 < k1 && k1 == steps) {
          const int col = (steps - 1) * K + (lane >> 4) * V, from = min(col, width - V);
          const vecT raw = row_value<T>(row_load(row + from));
          vecT a;
#pragma unroll
          for (int e = 0; e < V; ++e) a[e] = from + e >= col ? raw[e] : (T)0.0f;
          multiply(a, steps - 1);
        }
      }
    }
    if (split > 1) {
      __syncthreads();  // the sums of the rows before have been read
      if (share != 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n) sums[(wave * NT + n) * 64 + lane] = sum[0][n];
      }
      __syncthreads();
      if (share != 0) continue;
      for (int o = 1; o < split; ++o) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const f32x4 other = sums[((wave + o) * NT + n) * 64 + lane];
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[0][n][r] += other[r];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i >= rows) break;
      const int v = (tile0 + i) * 16 + (lane >> 4) * 4;
      float add[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) add[r] = bias && v + r < vocab ? (float)bias[v + r] : 0.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float score[4], m = st[n].m;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          score[r] = v + r < vocab ? sum[i][n][r] + add[r] : neg_inf();
          m = fmaxf(m, score[r]);
        }
        const unsigned of = (unsigned)label[n] - (unsigned)v;
        if (of < 4u && label[n] < vocab) {
          float s = score[0];
#pragma unroll
          for (int r = 1; r < 4; ++r) s = of == (unsigned)r ? score[r] : s;
          label_score[n * 16 + (lane & 15)] = s;
        }
        const float base = m == neg_inf() ? 0.0f : m;
        float s = st[n].s * (st[n].m == m ? 1.0f : exp2_fast((st[n].m - base) * kLog2e));
#pragma unroll
        for (int r = 0; r < 4; ++r) s += exp2_fast((score[r] - base) * kLog2e);
        st[n] = SoftStat{m, s};
      }
    }
  }
  __shared__ SoftStat sh[kFewWaves][NT * 16];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    st[n] = shfl_xor_join(st[n], 16, kLog2e);
    st[n] = shfl_xor_join(st[n], 32, kLog2e);
    if (lane < 16) sh[wave][n * 16 + lane] = st[n];
  }
  __syncthreads();
  if (tid < tokens) {
    SoftStat all = sh[0][tid];
    for (int i = split; i < kFewWaves; i += split) all = join(all, sh[i][tid], kLog2e);
    part[(size_t)blockIdx.x * tokens + tid] = all;
  }
}

// Kept scores of a token: the parts that the product was cut into are added up in order, then lse and loss (forward),
// then G (backward) in T; fp32 G takes the place of the scores, and so does bf16's unrounded G where db needs its column
// sums.  ld is a multiple of four and rows start at 16-byte boundaries.
constexpr int kRowThreads = 512;
struct RowArgs {
  float *scores;
  const void *bias;
  const int *labels;
  const float *weight, *wmax;
  int tokens, vocab, splits, ignore, mpad, keep_g;
  size_t ld;
};
template <class T>
__device__ __forceinline__ void add_bias(f32x4 &v, const RowArgs &p, int c) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < p.vocab) v[i] += (float)((const T *)p.bias)[c + i];
}
// The sums over [begin, end) of a row, and if asked for their statistics, by a workgroup: its first lane has them.
template <class T>
__device__ __forceinline__ SoftStat row_stats(float *__restrict__ row, const RowArgs &p, int begin, int end, bool stats) {
  __shared__ SoftStat sh[kRowThreads / 64];
  const int tid = threadIdx.x;
  const size_t part = (size_t)p.tokens * p.ld;
  SoftStat st{neg_inf(), 0.0f};
  for (int c = begin + tid * 4; c < end; c += kRowThreads * 4) {
    f32x4 v = *reinterpret_cast<const f32x4 *>(row + c);
    if (p.splits > 1) {
      for (int i = 1; i < p.splits; ++i) v += *reinterpret_cast<const f32x4 *>(row + i * part + c);
      *reinterpret_cast<f32x4 *>(row + c) = v;
    }
    if (!stats) continue;
    if (p.bias) add_bias<T>(v, p, c);
    float m = st.m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = c + i < p.vocab ? v[i] : neg_inf();
      m = fmaxf(m, v[i]);
    }
    const float base = m == neg_inf() ? 0.0f : m;
    float s = st.s * (st.m == m ? 1.0f : exp2_fast((st.m - base) * kLog2e));
#pragma unroll
    for (int i = 0; i < 4; ++i) s += exp2_fast((v[i] - base) * kLog2e);
    st = SoftStat{m, s};
  }
  if (stats) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) st = shfl_xor_join(st, m, kLog2e);
    if ((tid & 63) == 0) sh[tid >> 6] = st;
    __syncthreads();  // (also: these sums are written)
    if (tid == 0) {
#pragma unroll
      for (int i = 1; i < kRowThreads / 64; ++i) st = join(st, sh[i], kLog2e);
    }
  }
  return st;
}
template <class T>
__device__ __forceinline__ float row_score(const float *__restrict__ row, const RowArgs &p, int label) {
  return row[label] + (p.bias ? (float)((const T *)p.bias)[label] : 0.0f);
}
// G over [begin, end) of a row
template <class T>
__device__ __forceinline__ void row_grad(T *__restrict__ g, float *__restrict__ row, const RowArgs &p, int t, float lse,
                                         int begin, int end) {
  const TokenGrad tg = token_grad(0, 1, p.labels + t, p.ignore, &lse, p.weight ? p.weight + t : nullptr, p.wmax);
  for (int c = begin + threadIdx.x * 4; c < end; c += kRowThreads * 4) {
    float f[4];
    f32x4 v = *reinterpret_cast<const f32x4 *>(row + c);
    if (p.bias) add_bias<T>(v, p, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = c + i < p.vocab ? grad_entry(v[i], tg, c + i == tg.label) : 0.0f;
    if (p.keep_g || std::is_same<T, float>::value) *reinterpret_cast<f32x4 *>(row + c) = f32x4{f[0], f[1], f[2], f[3]};
    if (!std::is_same<T, float>::value) store4<T>(g + (size_t)t * p.ld + c, f, 4);
  }
}

// A workgroup per token; the second walk over the row finds it in a cache.  HBM: 120 us for 2048 tokens and 32768 rows of
// fp32 (537 MB, 4.5 TB/s).
template <class T>
__global__ __launch_bounds__(kRowThreads) void vocab_row_kernel(float *__restrict__ loss, float *__restrict__ lse_out,
                                                                const float *__restrict__ lse_in, T *__restrict__ g,
                                                                RowArgs p) {
  __shared__ float lse_sh;
  const int t = blockIdx.x;
  float *row = p.scores + (size_t)t * p.ld;
  if (loss || p.splits > 1) {
    const SoftStat st = row_stats<T>(row, p, 0, p.vocab, loss != nullptr);
    if (loss && threadIdx.x == 0) {
      const int label = p.labels[t];
      lse_sh = store_loss(loss, lse_out, t, st, label,
                          (unsigned)label < (unsigned)p.vocab ? row_score<T>(row, p, label) : 0.0f, p.vocab, p.ignore);
    }
  }
  if (!loss && threadIdx.x == 0) lse_sh = lse_in[t];
  if (!g) return;
  __syncthreads();
  row_grad<T>(g, row, p, t, lse_sh, 0, p.mpad);
}

// The same for few tokens with long rows, each cut into ranges of `len`: statistics of the ranges, then G, whose workgroups
// join the ranges for themselves (8 tokens, 50000 rows of bf16: 10 us, with a workgroup a token 38).
template <class T>
__global__ __launch_bounds__(kRowThreads) void vocab_range_stats_kernel(SoftStat *__restrict__ part,
                                                                        float *__restrict__ label_score, RowArgs p, int len) {
  const int t = blockIdx.y, begin = (int)blockIdx.x * len, end = min(p.vocab, begin + len);
  float *row = p.scores + (size_t)t * p.ld;
  const SoftStat st = row_stats<T>(row, p, begin, end, part != nullptr);
  if (!part || threadIdx.x != 0) return;
  part[(size_t)blockIdx.x * p.tokens + t] = st;
  const int label = p.labels[t];
  if (label >= begin && label < end) label_score[t] = row_score<T>(row, p, label);
}
template <class T>
__global__ __launch_bounds__(kRowThreads) void vocab_range_grad_kernel(float *__restrict__ loss, float *__restrict__ lse_out,
                                                                       const float *__restrict__ lse_in,
                                                                       const SoftStat *__restrict__ part,
                                                                       const float *__restrict__ label_score,
                                                                       T *__restrict__ g, RowArgs p, int len) {
  __shared__ float lse_sh;
  const int t = blockIdx.y, begin = (int)blockIdx.x * len;
  const int end = blockIdx.x + 1 == gridDim.x ? p.mpad : begin + len;
  if (loss) {
    if (threadIdx.x < 64) {
      SoftStat st = threadIdx.x < gridDim.x ? part[(size_t)threadIdx.x * p.tokens + t] : SoftStat{neg_inf(), 0.0f};
#pragma unroll
      for (int m = 32; m > 0; m >>= 1) st = shfl_xor_join(st, m, kLog2e);
      if (threadIdx.x == 0) {
        lse_sh = log_sum(st, 1.0f);
        if (blockIdx.x == 0) store_loss(loss, lse_out, t, st, p.labels[t], label_score[t], p.vocab, p.ignore);
      }
    }
  } else if (threadIdx.x == 0) {
    lse_sh = lse_in[t];
  }
  __syncthreads();
  row_grad<T>(g, p.scores + (size_t)t * p.ld, p, t, lse_sh, begin, end);
}

// What is left behind the products, in one launch.  db = *wmax times the column sums of kept G: 64 columns a workgroup, its 16
// wavefronts taking every 16th token each.  dx[t] = *wmax times the sum of the slabs, in order, four columns a lane.  HBM
// (8192 x 4096 from one slab: 37 us, 5.4 TB/s) and the launch, which is why the two share it (256 tokens of 4096, 1000 rows of
// fp32: 82 us a step with two launches, 80 with one).
constexpr int kFinishThreads = 1024;
struct FinishArgs {
  const float *slabs, *g, *wmax;
  int tokens, width, splits, db_blocks, rows, dx_lanes;
  size_t ldx, ld, ldg;
};
template <class T>
__global__ __launch_bounds__(kFinishThreads) void vocab_finish_kernel(T *__restrict__ dx, T *__restrict__ db, FinishArgs p) {
  __shared__ float sh[16][64];
  const float weight = p.wmax ? *p.wmax : 1.0f;
  if ((int)blockIdx.x < p.db_blocks) {
    const int lane = threadIdx.x & 63, y = threadIdx.x >> 6, m = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (m < p.rows) {
#pragma unroll 8
      for (int t = y; t < p.tokens; t += 16) s += p.g[(size_t)t * p.ldg + m];
    }
    sh[y][lane] = s;
    __syncthreads();
    if (y == 0 && m < p.rows) {
#pragma unroll
      for (int i = 1; i < 16; ++i) s += sh[i][lane];
      db[m] = (T)(s * weight);
    }
    return;
  }
  if ((int)threadIdx.x >= p.dx_lanes) return;
  const unsigned vecs = (unsigned)(p.width + 3) / 4;
  const size_t all = (size_t)p.tokens * vecs, stride = (size_t)(gridDim.x - p.db_blocks) * p.dx_lanes;
  for (size_t i = (size_t)(blockIdx.x - p.db_blocks) * p.dx_lanes + threadIdx.x; i < all; i += stride) {
    const size_t t = all >> 32 ? i / vecs : (unsigned)i / vecs;
    const int c = (int)(i - t * vecs) * 4;
    f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < p.splits; ++k) s += *reinterpret_cast<const f32x4 *>(p.slabs + ((size_t)k * p.tokens + t) * p.ld + c);
    const float f[4] = {s[0] * weight, s[1] * weight, s[2] * weight, s[3] * weight};
    store4<T>(dx + t * p.ldx + c, f, p.width - c);
  }
}

template <class T>
__global__ __launch_bounds__(256) void vocab_db_kernel(T *__restrict__ db, const float *__restrict__ part,
                                                       const float *__restrict__ wmax, int rows, int ld, int tiles) {
  const int m = blockIdx.x * 256 + threadIdx.x;
  if (m >= rows) return;
  float s = 0.0f;
#pragma unroll 4
  for (int i = 0; i < tiles; ++i) s += part[(size_t)i * ld + m];
  db[m] = (T)(wmax ? s * *wmax : s);
}

template <class T>
__global__ __launch_bounds__(256) void vocab_zero_kernel(T *__restrict__ p, size_t ld, int cols) {
  for (int c = threadIdx.x; c < cols; c += 256) p[(size_t)blockIdx.x * ld + c] = (T)0.0f;
}

// ---- host --------------------------------------------------------------------------------------------------------
typedef Shape<256, 256, 2, 4, 2> ShapeL;
typedef Shape<256, 256, 4, 2, 2> ShapeLA;  // the same tile with fewer fragments of A per wavefront: A contiguous along its rows
typedef Shape<128, 128, 2, 2, 2> ShapeM;
typedef Shape<64, 64, 2, 2, 2> ShapeN;
typedef Shape<64, 32, 4, 1, 2> ShapeS;
typedef Shape<64, 32, 4, 1, 4> ShapeD;  // few workgroups: deeper prefetch instead of more of them on a CU

static int idiv(int a, int b) { return (a + b - 1) / b; }
static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Which tile a product takes and into how many parts it is cut along k: the cheapest by a small model of the chip.  A
// workgroup's step costs `alone` microseconds when it has a CU to itself and `full` when `occ` of them share it; `finish`
// is what a round of tiles pays before and after its steps.  Measured with each tile pinned: tokens 256, width 4096, 1000
// rows (alone) and tokens 2048, width 2048, 32768 rows (full).
struct TileCost {
  int bm, bn, occ;
  double alone[2], full[2], finish;  // fp32, bf16
};
enum ShapeId { SHAPE_L, SHAPE_M, SHAPE_N, SHAPE_S, SHAPE_D, SHAPES };
static const TileCost kTiles[SHAPES] = {
    {ShapeL::BM, ShapeL::BN, 1, {7.35, 1.28}, {7.50, 1.62}, 10.0},
    {ShapeM::BM, ShapeM::BN, 2, {2.06, 0.70}, {3.88, 1.05}, 6.0},
    {ShapeN::BM, ShapeN::BN, 4, {0.60, 0.44}, {1.97, 0.67}, 3.0},
    {ShapeS::BM, ShapeS::BN, 6, {0.42, 0.42}, {1.50, 0.71}, 2.0},
    {ShapeD::BM, ShapeD::BN, 3, {0.36, 0.20}, {0.85, 0.41}, 2.0},
};
constexpr double kLaunchUs = 3.0, kBytesPerUs = 5.0e6;  // what a launch costs, and a pass over memory

struct Choice {
  ShapeId shape;
  int splits;
  double us;
};
// scores that stay inside; kept scores, fp32 parts along k; dx, the same with w read across its rows; dx written at once; rows
// of dw
enum ProductKind { REDUCED, PARTS, TURNED, TURNED_ROWS, ROWS };
static double shape_us(int shape, int splits, int M, int N, int K, int dtype, ProductKind kind) {
  const int d = dtype == CCT_BF16 ? 1 : 0, steps = idiv(K, d ? 64 : 32);
  const TileCost &c = kTiles[shape];
  const double w = (double)idiv(M, c.bm) * idiv(N > 0 ? N : 1, c.bn) * splits, round = 256.0 * c.occ;
  const double rounds = (double)(long)(w / round), per_cu = (double)(long)((w - rounds * round + 255.0) / 256.0);
  const double last = per_cu * c.full[d] / c.occ;
  const double step = rounds * c.full[d] + (per_cu > 0 ? (last > c.alone[d] ? last : c.alone[d]) : 0.0);
  const double el = d ? 2 : 4, out = (double)M * N;
  // across rows narrow tiles take pieces of 128 bytes, and tiles along n fetch them again, mostly from a cache (dx of 131072
  // rows of 4096 bf16: 64 tokens 332 us with 64 x 32 and 264 with 128 x 128, 128 tokens 400 us with 64 x 64)
  const double again = 1.0 + 0.2 * (idiv(N > 0 ? N : 1, c.bn) - 1), rate = c.bm >= 128 ? 4.1e6 : 3.5e6;
  const bool turned = kind == TURNED || kind == TURNED_ROWS;
  const double in_us = turned ? ((double)M * again + N) * K * el / rate : ((double)M + N) * K * el / kBytesPerUs;
  const double work = step * idiv(steps, splits), ends = c.finish * (rounds + (per_cu > 0 ? 1 : 0));
  const double us = kLaunchUs + (work > in_us ? work : in_us) + ends;
  // parts are written by the product and read by what joins them
  if (kind == PARTS || kind == TURNED) return us + 2.0 * splits * out * 4.0 / kBytesPerUs;
  // rows are written while others are computed, or bound the launch
  const double rows_us = kLaunchUs + in_us + out * el / kBytesPerUs;
  return (kind == ROWS || kind == TURNED_ROWS) && rows_us > us ? rows_us : us;
}
static Choice choose(int tile, int M, int N, int K, int dtype, ProductKind kind) {
  const bool narrow = kind != ROWS;  // an operand that is contiguous along its rows needs 64 of them
  const int steps = idiv(K, dtype == CCT_BF16 ? 64 : 32);
  const int pinned = tile >= 1 && tile <= SHAPES ? tile : 0;  // the tuning override
  Choice best{SHAPE_M, 1, 1e30};
  for (int s = 0; s < SHAPES; ++s) {
    if (s >= SHAPE_S && !narrow) continue;
    if (pinned && s != (pinned > SHAPE_S && !narrow ? (int)SHAPE_N : pinned - 1)) continue;
    for (int splits = 1; splits <= 64; splits *= 2) {
      if (splits > 1 && ((kind != PARTS && kind != TURNED) || steps < 4 * splits)) break;
      const double us = shape_us(s, splits, M, N, K, dtype, kind);
      if (us < best.us) best = Choice{(ShapeId)s, splits, us};
    }
  }
  return best;
}

// The rows of the vocabulary that a product's tiles cover in whole rounds of the chip, and the tile for the rest in a launch of
// its own, where that is cheaper than one more round with few tiles (1023 tokens of 1000 bf16, 50021 rows: the loss 132 -> 116
// us, dw with the scores 301 -> 271; less inside a step that the clock holds back).  `rows` are M, or N where across is set.
struct Cut {
  int main;  // rows of the first launch: all of them, where there is no second one
  Choice rest;
};
static Cut cut_rows(int tile, const Choice &c, int rows, int other, int K, int dtype, bool across) {
  const Cut whole{rows, c};
  if (other == 0 || tile) return whole;
  const TileCost &t = kTiles[c.shape];
  const long per = idiv(other, across ? t.bm : t.bn), block = across ? t.bn : t.bm, round = 256l * t.occ;
  const long blocks = (rows + block - 1) / block, rounds = blocks * per / round, main = rounds * round / per * block;
  if (main == 0 || main >= rows) return whole;
  const auto us = [&](int n) {
    return across ? shape_us(c.shape, 1, other, n, K, dtype, ROWS) : shape_us(c.shape, 1, n, other, K, dtype, REDUCED);
  };
  const int left = rows - (int)main;
  const Choice rest = across ? choose(tile, other, left, K, dtype, ROWS) : choose(tile, left, other, K, dtype, REDUCED);
  // (2538 tokens of 824, 44875 rows, 6.9 rounds of tiles: no gain by this estimate, a step of 944 us instead of 890.  40 bf16 steps
  // of 16 to 4096 tokens, widths 64 to 4096, 1000 to 65536 rows, all cut where they can be or none: 3 % faster to 20 % slower; by
  // this rule within 0.3 % of the better one, but for steps below 60 us: 3 %)
  return us((int)main) + rest.us < 0.92 * us(rows) ? Cut{(int)main, rest} : whole;
}

constexpr size_t kKeepBytes = (size_t)512 << 20;   // fp32 scores that may be kept
constexpr size_t kPieceBytes = (size_t)384 << 20;  // automatic piece: G and w's packed copy
// a tile's rows are addressed with 32-bit byte offsets: 256 rows of a piece's columns in fp32 are 2^30 bytes
constexpr int kPieceMax = 1 << 20;

// rows that the product kernel can take as they are, if they start at a multiple of 16 bytes
static bool whole_chunks(size_t ld, int width, size_t el) { return (ld * el & 15) == 0 && ((size_t)width * el & 15) == 0; }

struct VocabPlan {
  int tokens, width, vocab, dtype;
  size_t el, ldx, ldw;
  int unit;            // elements of a 128-byte step
  bool packed;         // rows of x or w are no whole 16-byte chunks: those operands are copied
  int piece, loss_piece;  // rows of w at a time; for the loss alone, which keeps nothing of them
  int hp, np, vp;      // row lengths of packed operands, x's transpose and G: width, tokens, piece, in whole steps
  Choice stats, grad, kept, dx, dw;
  Cut stats_cut[2], grad_cut[2], dw_cut[2];  // [1]: of the last piece, whose rows may be fewer
  bool dx_at_once;
  // whether a call keeps the scores (which takes a single piece) or reduces them tile by tile
  bool keep_forward, keep_backward[2], keep_both[2];  // [1]: db is asked for
  int stats_tiles;
  int ranges, range;   // a token's kept scores are cut into so many ranges of so many
  int few_blocks;      // workgroups of a few tokens' forward pass (0: it takes the tiles)
  FewShape few;
  size_t few_lds;
  size_t part, label_score, xpack, wpack, scores, xl, wmax, g, slabs, db, total_forward, total;
};

// All that a call's launches and its workspace have to agree on: the tuning overrides are read here, once, whatever another
// thread sets in the meantime.
static VocabPlan vocab_plan(const cct_vocab_loss_args *a) {
  VocabPlan p;
  const int tile = tuning().vocab_tile, keep = tuning().vocab_keep;
  p.tokens = a->tokens;
  p.width = a->width;
  p.vocab = a->vocab;
  p.dtype = a->dtype;
  p.el = dtype_bytes(a->dtype);
  p.ldx = a->x_stride ? a->x_stride : (size_t)a->width;
  p.ldw = a->w_stride ? a->w_stride : (size_t)a->width;
  p.unit = 128 / (int)p.el;
  p.hp = idiv(p.width, p.unit) * p.unit;
  p.np = (idiv(p.tokens, p.unit) + 1) * p.unit;
  const size_t n = p.tokens;
  const int vmax = idiv(p.vocab, 256) * 256;
  p.packed = !whole_chunks(p.ldx, p.width, p.el) || !whole_chunks(p.ldw, p.width, p.el);
  // a piece's tiles, with the smallest tile, are fewer than 2^32 lanes in a launch
  size_t most = ((size_t)1 << 34) / (n > (size_t)p.hp ? n : (size_t)p.hp) & ~(size_t)255;
  if (most < 256) most = 256;
  if (most > (size_t)kPieceMax) most = kPieceMax;
  if (a->piece > 0) {
    p.piece = (int)min((((size_t)a->piece + 255) / 256) * 256, most);
  } else {
    // all of the vocabulary, or a power of two, so that the tiles of a piece fill whole rounds of the chip
    const size_t row = (n + p.hp) * p.el, want = kPieceBytes / row;
    size_t rows = 1024;
    while (rows * 2 <= want && rows < (size_t)vmax) rows *= 2;
    if ((size_t)vmax <= want) rows = vmax;
    p.piece = (int)min(rows, most);
  }
  if (p.piece > vmax) p.piece = vmax;
  // kept scores: all of the vocabulary at once, and so its packed copy
  const bool may_keep = (size_t)vmax <= most && (a->piece <= 0 || p.piece == vmax) &&
                        (!p.packed || (size_t)vmax * p.hp * p.el <= kPieceBytes);
  p.loss_piece = a->piece > 0 || p.packed ? p.piece : (int)min((size_t)vmax, most);
  p.stats = choose(tile, min(p.loss_piece, p.vocab), p.tokens, p.width, p.dtype, REDUCED);
  p.grad = choose(tile, min(p.piece, p.vocab), p.tokens, p.width, p.dtype, REDUCED);
  p.kept = choose(tile, p.vocab, p.tokens, p.width, p.dtype, PARTS);
  const double score_bytes = (double)n * vmax * 4;
  const double stats_us = p.stats.us * idiv(p.vocab, p.loss_piece) + kLaunchUs;
  const double grad_scores_us = p.grad.us * idiv(p.vocab, p.piece) + kLaunchUs;
  // (the choice's own cost has the scores written and read once; G is written on top, in place of the scores in fp32)
  const double join_us = kLaunchUs, grad_us = (double)n * vmax * p.el / kBytesPerUs;
  const bool fits = may_keep && score_bytes * p.kept.splits <= (double)kKeepBytes;
  p.keep_forward = fits && p.kept.us + join_us < stats_us;
  bool keep_any = p.keep_forward;
  for (int db = 0; db < 2; ++db) {
    // the column sums read the kept G (in bf16 it is written in fp32 for them), those of a GRAD product come with it
    const double db_us = db ? kLaunchUs + score_bytes * (p.el == 4 ? 1 : 2) / kBytesPerUs : 0.0;
    p.keep_backward[db] = fits && p.kept.us + join_us + grad_us + db_us < grad_scores_us;
    p.keep_both[db] = fits && p.kept.us + join_us + grad_us + db_us < stats_us + grad_scores_us;
    if (keep) p.keep_forward = p.keep_backward[db] = p.keep_both[db] = fits && keep == 1;
    keep_any = keep_any || p.keep_forward || p.keep_backward[db] || p.keep_both[db];
  }
  if (keep_any) p.piece = p.loss_piece = vmax;
  p.vp = p.piece + p.unit;
  p.stats = choose(tile, min(p.loss_piece, p.vocab), p.tokens, p.width, p.dtype, REDUCED);
  p.grad = choose(tile, min(p.piece, p.vocab), p.tokens, p.width, p.dtype, REDUCED);
  p.dx = choose(tile, p.width, p.tokens, p.piece, p.dtype, TURNED);
  // one piece and one part: dx at once, without a launch that joins (bf16, 8 tokens of 64, 500 rows: 19.6 us a step, 24.6 with
  // it; 4000 tokens of 4096, 20011 rows: 1682 and 1731).  In fp32 the estimate for few workgroups is too good by a sixth (576
  // tokens of 1408, 6400 rows: 318 us a step at once, 286 in parts).  Drawn sizes, always at once against never: 40 in fp32 0.8 %
  // faster to 3.6 times slower, 30 in bf16 8 % faster to 2.7 times slower; the rule is within 1.5 % of the better one (a bf16 step
  // of 31 us: 9 %).
  const Choice at_once = choose(tile, p.width, p.tokens, p.piece, p.dtype, TURNED_ROWS);
  p.dx_at_once = p.piece >= p.vocab && at_once.us < (p.el == 4 ? 0.85 : 1.0) * (p.dx.us + kLaunchUs);
  if (p.dx_at_once) p.dx = at_once;
  p.dw = choose(tile, p.width, p.piece, p.tokens, p.dtype, ROWS);
  p.stats_tiles = 0;
  for (int last = 0; last < 2; ++last) {
    const auto rows_of = [&](int piece) { return last ? p.vocab - (idiv(p.vocab, piece) - 1) * piece : min(piece, p.vocab); };
    const int loss_rows = rows_of(p.loss_piece), rows = rows_of(p.piece);
    p.stats_cut[last] = cut_rows(tile, p.stats, loss_rows, p.tokens, p.width, p.dtype, false);
    p.grad_cut[last] = cut_rows(tile, p.grad, rows, p.tokens, p.width, p.dtype, false);
    p.dw_cut[last] = cut_rows(tile, p.dw, rows, p.width, p.tokens, p.dtype, true);
    const Cut &cut = p.stats_cut[last];
    const int tiles = idiv(cut.main, kTiles[p.stats.shape].bm) + idiv(loss_rows - cut.main, kTiles[cut.rest.shape].bm);
    p.stats_tiles += last ? tiles : (idiv(p.vocab, p.loss_piece) - 1) * tiles;
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  // a few tokens' forward pass: 16 rows a wave or shared by up to eight, so that about 2048 waves have work; as many
  // workgroups as the chip holds at once.  x by panels from 16384 rows on: fewer leave compute units without a workgroup (64
  // tokens of 1001 fp32: 45 us up to there, the tiles 23 us with 4001 rows and 47 us with 16001)
  const int few_n = n <= 16 ? 1 : n <= 32 ? 2 : 4, few_steps = idiv(p.width, 64 / (int)p.el), few_tiles = idiv(p.vocab, 16);
  FewShape &f = p.few;
  f = FewShape{1, few_steps, 1};
  while (f.split < kFewWaves && few_tiles * f.split < 2048 && few_steps >= 8 * f.split) f.split *= 2;
  p.few_lds = (size_t)few_steps * few_n * 1024 + (f.split > 1 ? kFewWaves * few_n * 1024 : 0);
  if (p.few_lds > (size_t)kFewLds) {
    f = FewShape{1, kFewPanel / (few_n * 1024), max(1, min(kFewRows, few_tiles / (kFewWaves * 512)))};
    p.few_lds = kFewPanel;
  }
  p.few_blocks = 0;
  if (!whole_chunks(p.ldw, p.width, p.el) && p.tokens <= kFewTokens && p.width * p.el >= 16 && !tile && keep != 1 &&
      (f.panel == few_steps || few_tiles >= 1024))
    p.few_blocks = min(idiv(few_tiles, kFewWaves / f.split * f.rows),
                       p.few_lds <= 36 << 10 ? 1024 : p.few_lds <= 72 << 10 ? 512 : 256);
  // ranges of a token's kept scores: about 1024 workgroups, of 4096 scores or more, where a token would have four or more
  p.ranges = min(min(1024 / max(p.tokens, 1), p.vocab / 4096), 64);
  if (p.ranges < 4) p.ranges = 1;
  p.range = idiv(idiv(p.vocab, p.ranges), 64) * 64;
  p.ranges = idiv(p.vocab, p.range);
  p.part = take((size_t)max(max(p.stats_tiles, p.few_blocks), p.ranges) * n * sizeof(SoftStat));
  p.label_score = take(n * 4);
  const size_t few_forward = at;
  p.xpack = take(p.packed ? n * p.hp * p.el : 0);
  p.wpack = take(p.packed ? (size_t)p.piece * p.hp * p.el : 0);
  const size_t score_space = (size_t)p.kept.splits * n * p.vp * 4;
  p.scores = take(p.keep_forward ? score_space : 0);
  p.total_forward = p.few_blocks ? few_forward : at;
  if (!p.keep_forward) p.scores = take(keep_any ? score_space : 0);
  p.xl = take((p.el == 2 ? (size_t)p.width * p.np : n * p.hp) * p.el);
  p.wmax = take(4);
  const bool g_in_scores = p.el == 4 && p.keep_backward[0] && p.keep_backward[1] && p.keep_both[0] && p.keep_both[1];
  p.g = take(g_in_scores ? 0 : n * p.vp * p.el);
  p.slabs = take(p.dx_at_once ? 0 : (size_t)p.dx.splits * n * p.hp * 4);
  p.db = take((size_t)idiv(p.tokens, 32) * p.vp * 4);
  p.total = at;
  return p;
}

template <class T, class S, int USE, bool KA, bool KB>
static int launch_product(ProductArgs &p) {
  auto kern = vocab_product_kernel<T, S, USE, KA, KB>;
  static LdsGrant grant;
  const size_t bytes = S::STAGES * S::STAGE;
  if (int rc = grant_dynamic_lds((const void *)kern, bytes, grant)) return rc;
  p.tiles_m = idiv(p.M, S::BM);
  p.tiles_n = idiv(p.N, S::BN);
  const int steps = idiv(p.K, 128 / (int)sizeof(T));
  p.steps_per_split = idiv(steps, p.splits);
  const unsigned long blocks = (unsigned long)p.tiles_m * p.tiles_n * p.splits;
  CCT_REQUIRE(blocks * S::THREADS < (1ul << 32), "vocab_loss: %lu workgroups are too many for one launch", blocks);
  p.blocks = (uint32_t)blocks;
  kern<<<p.blocks, S::THREADS, bytes, ctx().stream>>>(p);
  CCT_LAUNCH_CHECK();
  note_kernel("vocab_product_kernel<%s, Shape<%d, %d, %d, %d, %d>, %d, %s, %s> splits=%d m=%d n=%d", Num<T>::NAME, S::BM, S::BN,
              S::WM, S::WN, S::STAGES, USE, KA ? "true" : "false", KB ? "true" : "false", p.splits, p.M, p.N);
  return 0;
}

template <class T, int USE, bool KA, bool KB>
static int product(const Choice &c, ProductArgs &p) {
  p.splits = c.splits;
  switch (c.shape) {
    case SHAPE_L: return launch_product<T, typename std::conditional<KA, ShapeL, ShapeLA>::type, USE, KA, KB>(p);
    case SHAPE_M: return launch_product<T, ShapeM, USE, KA, KB>(p);
    case SHAPE_N: return launch_product<T, ShapeN, USE, KA, KB>(p);
    default:
      // an operand that is contiguous along its rows needs 64 of them
      if constexpr (KB) {
        if (c.shape == SHAPE_S) return launch_product<T, ShapeS, USE, KA, KB>(p);
        return launch_product<T, ShapeD, USE, KA, KB>(p);
      }
      return launch_product<T, ShapeN, USE, KA, KB>(p);
  }
}

struct VocabCall {
  float *loss;
  float *lse;
  const float *lse_in;  // backward alone
  void *dx, *dw, *db;
  const void *x, *w, *bias;
  const int *labels;
  const float *weight;
  int ignore;
  char *ws;
  bool forward, backward;
};

template <class T, int NT>
static int vocab_few(const VocabPlan &p, const VocabCall &c) {
  SoftStat *part = (SoftStat *)(c.ws + p.part);
  float *label_score = (float *)(c.ws + p.label_score);
  const bool panels = p.few.panel < idiv(p.width, 4 * Num<T>::V);
  auto kern = panels ? vocab_few_kernel<T, NT, true> : vocab_few_kernel<T, NT, false>;
  static LdsGrant grants[2];
  if (int rc = grant_dynamic_lds((const void *)kern, kFewLds, grants[panels])) return rc;
  kern<<<p.few_blocks, kFewWaves * 64, p.few_lds, ctx().stream>>>(part, label_score, (const T *)c.x, (const T *)c.w,
                                                                 (const T *)c.bias, c.labels, p.ldx, p.ldw, p.tokens,
                                                                 p.width, p.vocab, p.few);
  CCT_LAUNCH_CHECK();
  note_kernel("vocab_few_kernel<%s, %d, %s> split=%d rows=%d", Num<T>::NAME, NT, panels ? "true" : "false", p.few.split,
              p.few.rows);
  vocab_loss_kernel<1><<<p.tokens, 256, 0, ctx().stream>>>(c.loss, c.lse, part, label_score, c.labels, p.tokens,
                                                          p.few_blocks, p.vocab, c.ignore);
  CCT_LAUNCH_CHECK();
  return 0;
}

template <class T>
static int vocab_run(const VocabPlan &p, const VocabCall &c) {
  hipStream_t st = ctx().stream;
  const int n = p.tokens;
  if (!c.backward && p.few_blocks)
    return n <= 16 ? vocab_few<T, 1>(p, c) : n <= 32 ? vocab_few<T, 2>(p, c) : vocab_few<T, 4>(p, c);
  const int db = c.db ? 1 : 0;
  const bool keep = c.forward && c.backward ? p.keep_both[db] : c.forward ? p.keep_forward : p.keep_backward[db];
  SoftStat *part = (SoftStat *)(c.ws + p.part);
  float *label_score = (float *)(c.ws + p.label_score), *scores = (float *)(c.ws + p.scores);
  float *slabs = (float *)(c.ws + p.slabs), *db_part = (float *)(c.ws + p.db);
  T *g = (T *)(c.ws + p.g), *xl = (T *)(c.ws + p.xl);
  constexpr bool kXt = !std::is_same<T, float>::value;  // x transposed for dw
  if (keep && p.el == 4) g = (T *)scores;  // fp32 G takes the scores' place
  const size_t packed = p.hp * p.el;
  const int chunk = p.unit / 8;  // elements of 16 bytes
  const bool direct_x = whole_chunks(p.ldx, p.width, p.el), direct_w = whole_chunks(p.ldw, p.width, p.el);
  const char *x = (const char *)(direct_x ? c.x : c.ws + p.xpack);
  const size_t ldx = direct_x ? p.ldx * p.el : packed;
  bool x_packed = direct_x;
  const float *wmax = nullptr;
  if (c.backward) {
    if (c.weight) wmax = (const float *)(c.ws + p.wmax);
    float *wm = (float *)(c.ws + p.wmax);
    if constexpr (kXt) {
      const int tiles_t = idiv(n, 64), tiles = tiles_t * idiv(p.width, 64);
      vocab_xt_kernel<T><<<tiles + (c.weight ? 1 : 0), 256, 0, st>>>(xl, (const T *)c.x, p.ldx, p.np, n, p.width,
                                                                    idiv(n, chunk) * chunk, tiles_t, c.labels, c.ignore,
                                                                    c.weight, wm, tiles);
    } else {
      vocab_live_kernel<T><<<n + (c.weight ? 1 : 0), 256, 0, st>>>(xl, (const T *)c.x, p.ldx, n, p.width, p.hp, c.labels,
                                                                  c.ignore, c.weight, wm);
    }
    CCT_LAUNCH_CHECK();
  }
  // the piece's rows of w as an operand; the first call sees to x too
  const size_t ldw = direct_w ? p.ldw * p.el : packed;
  auto rows_of_w = [&](int v0, int rows, const char **out) -> int {
    const T *src = (const T *)c.w + (size_t)v0 * p.ldw;
    T *wp = (T *)(c.ws + p.wpack);
    *out = (const char *)(direct_w ? src : wp);
    const int xrows = x_packed ? 0 : n, wrows = direct_w ? 0 : rows;
    x_packed = true;
    if (xrows + wrows == 0) return 0;
    int l = 0;
    while (l < 8 && (1 << l) * Num<T>::V < p.hp) ++l;
    vocab_pack_kernel<T><<<idiv(xrows + wrows, 256 >> l), 256, 0, st>>>((T *)(c.ws + p.xpack), (const T *)c.x, p.ldx, xrows, wp,
                                                                       src, p.ldw, wrows, p.width, p.hp, l);
    CCT_LAUNCH_CHECK();
    return 0;
  };
  auto score_args = [&](const char *w, int v0, int rows) {
    ProductArgs a{};
    a.A = w;
    a.lda = ldw;
    a.B = x;
    a.ldb = ldx;
    a.M = rows;
    a.N = n;
    a.K = p.width;
    a.kbytes = (uint32_t)((p.width * p.el + 15) & ~(size_t)15);
    a.bias = c.bias ? (const char *)c.bias + (size_t)v0 * p.el : nullptr;
    a.labels = c.labels;
    a.v0 = v0;
    a.ignore = c.ignore;
    return a;
  };
  const char *w = nullptr;
  if (keep) {
    if (int rc = rows_of_w(0, p.vocab, &w)) return rc;
    ProductArgs a = score_args(w, 0, p.vocab);
    a.C = scores;
    a.ldc = p.vp;
    if (int rc = product<T, USE_SLAB, true, true>(p.kept, a)) return rc;
    RowArgs r{scores, c.bias, c.labels, c.weight, wmax, n, p.vocab, p.kept.splits, c.ignore, idiv(p.vocab, chunk) * chunk,
              c.db ? 1 : 0, (size_t)p.vp};
    if (p.ranges > 1) {
      const dim3 grid(p.ranges, n);
      if (c.forward || r.splits > 1) {
        vocab_range_stats_kernel<T><<<grid, kRowThreads, 0, st>>>(c.forward ? part : nullptr, label_score, r, p.range);
        CCT_LAUNCH_CHECK();
      }
      if (c.backward)
        vocab_range_grad_kernel<T><<<grid, kRowThreads, 0, st>>>(c.forward ? c.loss : nullptr, c.lse, c.lse_in, part,
                                                                label_score, g, r, p.range);
      else
        vocab_loss_kernel<1><<<n, 256, 0, st>>>(c.loss, c.lse, part, label_score, c.labels, n, p.ranges, p.vocab, c.ignore);
    } else {
      vocab_row_kernel<T><<<n, kRowThreads, 0, st>>>(c.forward ? c.loss : nullptr, c.lse, c.lse_in, c.backward ? g : nullptr,
                                                    r);
    }
    CCT_LAUNCH_CHECK();
  } else if (c.forward) {
    int tiles = 0;
    for (int v0 = 0; v0 < p.vocab; v0 += p.loss_piece) {
      const int rows = min(p.loss_piece, p.vocab - v0);
      if (int rc = rows_of_w(v0, rows, &w)) return rc;
      const Cut &cut = p.stats_cut[v0 + rows == p.vocab];
      for (int r0 = 0; r0 < rows; r0 = r0 == 0 ? cut.main : rows) {
        ProductArgs a = score_args(w + r0 * ldw, v0 + r0, r0 == 0 ? cut.main : rows - r0);
        a.part = part;
        a.part_row = tiles;
        a.label_score = label_score;
        if (int rc = product<T, USE_STATS, true, true>(r0 == 0 ? p.stats : cut.rest, a)) return rc;
        tiles += a.tiles_m;
      }
    }
    if (n >= 2048)
      vocab_loss_kernel<16><<<idiv(n, 16), 256, 0, st>>>(c.loss, c.lse, part, label_score, c.labels, n, tiles, p.vocab,
                                                        c.ignore);
    else
      vocab_loss_kernel<1><<<n, 256, 0, st>>>(c.loss, c.lse, part, label_score, c.labels, n, tiles, p.vocab, c.ignore);
    CCT_LAUNCH_CHECK();
  }
  if (!c.backward) return 0;
  const float *lse = c.forward ? c.lse : c.lse_in;
  for (int v0 = 0; v0 < p.vocab; v0 += p.piece) {
    const int rows = min(p.piece, p.vocab - v0), mpad = idiv(rows, chunk) * chunk;
    if (!keep) {
      if (int rc = rows_of_w(v0, rows, &w)) return rc;
      const Cut &cut = p.grad_cut[v0 + rows == p.vocab];
      for (int r0 = 0; r0 < rows; r0 = r0 == 0 ? cut.main : rows) {
        const int some = r0 == 0 ? cut.main : rows - r0;
        ProductArgs a = score_args(w + r0 * ldw, v0 + r0, some);
        a.lse = lse;
        a.weight = c.weight;
        a.wmax = wmax;
        a.g = g + r0;
        a.ldg = p.vp;
        a.mpad = r0 + some == rows ? mpad - r0 : some;
        a.db_part = c.db ? db_part : nullptr;
        a.db_ld = p.vp;
        if (int rc = product<T, USE_GRAD, true, true>(r0 == 0 ? p.grad : cut.rest, a)) return rc;
        if (c.db) {
          vocab_db_kernel<T><<<idiv(some, 256), 256, 0, st>>>((T *)c.db + v0 + r0, db_part, wmax, some, p.vp, a.tiles_n);
          CCT_LAUNCH_CHECK();
        }
      }
    }
    if (c.dx) {
      ProductArgs a{};
      a.A = w;
      a.lda = ldw;
      a.abytes = (uint32_t)(direct_w ? p.width * p.el : packed);
      a.B = (const char *)g;
      a.ldb = p.vp * p.el;
      a.M = p.width;
      a.N = n;
      a.K = rows;
      a.kbytes = (uint32_t)(mpad * p.el);
      if (p.dx_at_once) {
        a.wmax = wmax;
        a.C = c.dx;
        a.ldc = p.ldx;
        if (int rc = product<T, USE_OUT, false, true>(p.dx, a)) return rc;
      } else {
        a.C = slabs;
        a.ldc = p.hp;
        a.accumulate = v0 > 0;
        if (int rc = product<T, USE_SLAB, false, true>(p.dx, a)) return rc;
      }
    }
    if (c.dw) {
      const Cut &cut = p.dw_cut[v0 + rows == p.vocab];
      for (int r0 = 0; r0 < rows; r0 = r0 == 0 ? cut.main : rows) {
        const int some = r0 == 0 ? cut.main : rows - r0;
        ProductArgs a{};
        a.A = (const char *)xl;
        a.lda = kXt ? p.np * p.el : packed;
        a.abytes = (uint32_t)packed;
        a.kbytes = (uint32_t)(idiv(n, chunk) * chunk * p.el);
        a.B = (const char *)(g + r0);
        a.ldb = p.vp * p.el;
        a.bbytes = (uint32_t)((r0 + some == rows ? mpad - r0 : some) * p.el);
        a.M = p.width;
        a.N = some;
        a.K = n;
        a.wmax = wmax;
        a.C = (T *)c.dw + (size_t)(v0 + r0) * p.ldw;
        a.ldc = p.ldw;
        a.stream = ((p.ldw * p.el | (uintptr_t)a.C) & 127) == 0;
        if (int rc = product<T, USE_OUT, kXt, false>(r0 == 0 ? p.dw : cut.rest, a)) return rc;
      }
    }
  }
  const int db_blocks = keep && c.db ? idiv(p.vocab, 64) : 0;
  // fewer lanes of a workgroup take part where that puts more of them to work (320 tokens of 200: 32 instead of 34 us with dx)
  const size_t dx_vecs = c.dx && !p.dx_at_once ? (size_t)n * idiv(p.width, 4) : 0;
  int dx_lanes = kFinishThreads;
  while (dx_lanes > 64 && dx_vecs / dx_lanes < 512) dx_lanes /= 2;
  const unsigned dx_blocks = (unsigned)min((dx_vecs + dx_lanes - 1) / dx_lanes, (size_t)1 << 21);
  if (db_blocks + dx_blocks > 0) {
    const FinishArgs f{slabs, scores, wmax, n, p.width, p.dx.splits, db_blocks, p.vocab, dx_lanes, p.ldx, (size_t)p.hp,
                       (size_t)p.vp};
    vocab_finish_kernel<T><<<db_blocks + dx_blocks, kFinishThreads, 0, st>>>((T *)c.dx, (T *)c.db, f);
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

static int check_vocab_rows(const VocabPlan &p, const void *x, const void *w, const char *who) {
  CCT_REQUIRE(!(whole_chunks(p.ldx, p.width, p.el) && ((uintptr_t)x & 15)) &&
                  !(whole_chunks(p.ldw, p.width, p.el) && ((uintptr_t)w & 15)),
              "%s: x at %p, w at %p: rows of whole 16-byte chunks have to start at a multiple of 16 bytes", who, x, w);
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
  if (int rc = check_vocab_rows(p, x, w, who)) return rc;
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
  if (int rc = check_vocab_rows(p, x, w, who)) return rc;
  VocabCall c{};
  c.lse_in = lse;
  c.dx = dx;
  c.dw = dw;
  c.db = db;
  c.x = x;
  c.w = w;
  c.bias = bias;
  c.labels = labels;
  c.weight = loss_grad;
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
  if (int rc = check_vocab_rows(p, x, w, who)) return rc;
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
  c.weight = loss_grad;
  c.ignore = args->ignore_label;
  c.ws = (char *)workspace;
  c.forward = c.backward = true;
  return vocab_dispatch(p, c);
}
