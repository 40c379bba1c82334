// Distillation loss from a teacher's top logits, on stored scores.
//
//   q = softmax(top_logits / T) over a token's list,  p = softmax(logits / T) over the vocabulary
//   lse = log sum exp(logits / T),  loss = T^2 sum_k q_k (log q_k - logits[id_k] / T + lse), from the statistics behind lse
//   dlogits_v = loss_grad * T * (p_v - sum of q_k over id_k == v)
//
// Exponentials are v_exp_f32 of (difference * log2 e / T).  Bound by HBM: the scores are read once for the loss (2051 tokens,
// 112896 bf16 scores: 89 us, 5.2 TB/s), and once for loss and gradient where a row fits a workgroup's registers; the list
// costs a few hundred bytes a token.
#include "narrow.h"

namespace cct {

constexpr int DST_THREADS = 256;
constexpr int DST_WAVES = DST_THREADS / 64;
constexpr int DST_TOP_MAX = 1024;

struct DistillShape {
  int tokens, vocab, top;
  float temperature, inv_t, scale2;  // T, 1 / T, log2(e) / T
  size_t logits_stride, top_stride;
  int splits, chunk;  // a row is cut into `splits` ranges of `chunk` elements
};

__device__ __forceinline__ SoftStat wave_join(SoftStat a, float scale2) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) a = shfl_xor_join(a, m, scale2);
  return a;
}

// A vector of values on top of a running maximum and sum.
template <int V>
__device__ __forceinline__ void add_values(SoftStat &st, const float (&z)[V], float scale2) {
  float m = st.m;
#pragma unroll
  for (int i = 0; i < V; ++i) m = fmaxf(m, z[i]);
  const float base = m == neg_inf() ? 0.0f : m;  // nothing but -inf so far: 2^(-inf) = 0 without -inf - -inf
  float s = st.s * (st.m == m ? 1.0f : exp2_fast((st.m - base) * scale2));
#pragma unroll
  for (int i = 0; i < V; ++i) s += exp2_fast((z[i] - base) * scale2);
  st.m = m;
  st.s = s;
}

// Maximum and sum of the scores [begin, end) of a row, by a workgroup; its first wavefront has the result.
template <class T>
__device__ __forceinline__ SoftStat range_stats(const T *__restrict__ row, int begin, int end, const DistillShape &s) {
  constexpr int V = Num<T>::V;
  __shared__ SoftStat sh[DST_WAVES];
  SoftStat st{neg_inf(), 0.0f};
  for (int col = begin + threadIdx.x * V; col < end; col += DST_THREADS * V) {
    float z[V];
    load_vec<T>(z, row, col, s.vocab);
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = col + i < end ? z[i] : neg_inf();
    add_values<V>(st, z, s.scale2);
  }
  st = wave_join(st, s.scale2);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = st;
  __syncthreads();
  st = sh[0];
#pragma unroll
  for (int w = 1; w < DST_WAVES; ++w) st = join(st, sh[w], s.scale2);
  return st;
}

// One range of one token.
template <class T>
__global__ __launch_bounds__(DST_THREADS) void distill_stats_kernel(SoftStat *__restrict__ part,
                                                                    const T *__restrict__ logits, DistillShape s) {
  const int t = blockIdx.x / s.splits, cut = blockIdx.x % s.splits;
  const SoftStat st = range_stats<T>(logits + (size_t)t * s.logits_stride, cut * s.chunk, min(s.vocab, (cut + 1) * s.chunk), s);
  if (threadIdx.x == 0) part[blockIdx.x] = st;
}

// softmax(logits / T) of one score: 2^((score - m) log2 e / T - log2 of the sum).  The difference comes first, so that scores of
// any size keep theirs, and none is above m.  A backward pass that has nothing but the lse takes T lse as m and a
// sum of one: off by the rounding of both, 2^-23 |lse| in the exponent, and cut at one, which that may pass.
struct Student {
  float m, log2_sum;
};
__device__ __forceinline__ Student student(SoftStat st) { return Student{st.m, __builtin_log2f(st.s)}; }
__device__ __forceinline__ float probability(float score, const Student &p, const DistillShape &s) {
  return exp2_fast(__builtin_fmaf(score - p.m, s.scale2, -p.log2_sum));
}
__device__ __forceinline__ float probability_cut(float score, const Student &p, const DistillShape &s) {
  const float e = __builtin_fmaf(score - p.m, s.scale2, -p.log2_sum);
  return exp2_fast(e > 0.0f ? 0.0f : e);  // (NaN stays)
}

// The teacher's distribution of one token, by one wavefront: lane l holds entries l, l + 64, ...
struct Teacher {
  float m, s;   // maximum and sum over the valid entries
  bool bad;     // an entry names a row outside the vocabulary
  // whether any entry has weight (one that is NaN has: the token's results are NaN then)
  __device__ __forceinline__ bool some() const { return m != neg_inf() || s != 0.0f; }
};
__device__ __forceinline__ Teacher teacher_stats(const int *__restrict__ ids, const float *__restrict__ top, int n,
                                                 int vocab, float scale2, int lane) {
  SoftStat st{neg_inf(), 0.0f};
  bool bad = false;
  for (int k = lane; k < n; k += 64) {
    const int id = ids[k];
    bad |= id >= vocab;
    float z[1] = {id >= 0 ? top[k] : neg_inf()};
    add_values<1>(st, z, scale2);
  }
  st = wave_join(st, scale2);
  return Teacher{st.m, st.s, __any(bad) != 0};
}

// q of one entry; 0 where it has no weight
__device__ __forceinline__ float teacher_weight(const Teacher &te, int id, float top, float scale2) {
  if (id < 0 || !te.some()) return 0.0f;
  return exp2_fast((top - te.m) * scale2) / te.s;
}

// Joins a token's ranges and computes its loss: one wavefront per token.
template <class T>
__device__ __forceinline__ void distill_loss_wave(float *__restrict__ loss, float *__restrict__ lse, SoftStat st,
                                                  const T *__restrict__ row, const int *__restrict__ ids,
                                                  const float *__restrict__ top, const DistillShape &s, int t, int lane) {
  const float l = log_sum(st, s.inv_t);
  const Teacher te = teacher_stats(ids, top, s.top, s.vocab, s.scale2, lane);
  const float logs = __builtin_log2f(te.s) * kLn2;
  float sum = 0.0f;
  for (int k = lane; k < s.top; k += 64) {
    const int id = ids[k];
    const float q = teacher_weight(te, id, top[k], s.scale2);
    if (q != 0.0f && id < s.vocab) sum += q * (((top[k] - te.m) * s.inv_t - logs) + label_loss(st, (float)row[id], s.inv_t));
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m, 64);
  if (lane == 0) {
    lse[t] = l;
    loss[t] = te.bad ? __builtin_nanf("") : s.temperature * s.temperature * sum;
  }
}

// Rows of a single range: statistics and loss in one launch, a workgroup per token.
template <class T>
__global__ __launch_bounds__(DST_THREADS) void distill_token_kernel(float *__restrict__ loss, float *__restrict__ lse,
                                                                    const T *__restrict__ logits,
                                                                    const int *__restrict__ ids,
                                                                    const float *__restrict__ top, DistillShape s) {
  const int t = blockIdx.x;
  const T *row = logits + (size_t)t * s.logits_stride;
  const SoftStat st = range_stats<T>(row, 0, s.vocab, s);
  if (threadIdx.x < 64)
    distill_loss_wave<T>(loss, lse, st, row, ids + (size_t)t * s.top_stride, top + (size_t)t * s.top_stride, s, t,
                         threadIdx.x);
}

template <class T>
__global__ __launch_bounds__(DST_THREADS) void distill_loss_kernel(float *__restrict__ loss, float *__restrict__ lse,
                                                                   const SoftStat *__restrict__ part,
                                                                   const T *__restrict__ logits,
                                                                   const int *__restrict__ ids,
                                                                   const float *__restrict__ top, DistillShape s) {
  const int t = blockIdx.x * DST_WAVES + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= s.tokens) return;
  SoftStat st{neg_inf(), 0.0f};
  for (int i = lane; i < s.splits; i += 64) st = join(st, part[(size_t)t * s.splits + i], s.scale2);
  st = wave_join(st, s.scale2);
  distill_loss_wave<T>(loss, lse, st, logits + (size_t)t * s.logits_stride, ids + (size_t)t * s.top_stride,
                       top + (size_t)t * s.top_stride, s, t, lane);
}

// A token's list in LDS, as the gradient needs it: for the first entry of every id in [begin, end), the id, its score and the
// weight of all entries with that id; -1 as the id of every other entry.  Returns whether the token has any weight at
// all.  All lanes of the workgroup call it.
struct EntryLists {
  int *id, *seen;  // `seen`: the ids before equal ones are merged
  float *q, *sum, *z;
};
__device__ __forceinline__ EntryLists entry_lists(float *lds, int top) {
  return EntryLists{(int *)lds, (int *)lds + top, lds + 2 * top, lds + 3 * top, lds + 4 * top};
}
template <class T>
__device__ __forceinline__ bool gather_entries(const EntryLists &e, const T *row, const int *__restrict__ ids,
                                               const float *__restrict__ top, int begin, int end, const DistillShape &s) {
  const int threads = blockDim.x, tid = threadIdx.x;
  // every wavefront computes the statistics by itself: the list is short, and no exchange is needed
  const Teacher te = teacher_stats(ids, top, s.top, s.vocab, s.scale2, tid & 63);
  for (int k = tid; k < s.top; k += threads) {
    const int id = ids[k];
    const float w = teacher_weight(te, id, top[k], s.scale2);
    const bool here = id >= begin && id < end && w != 0.0f;
    e.seen[k] = here ? id : -1;
    e.q[k] = w;
    e.z[k] = here ? (float)row[id] : 0.0f;
  }
  __syncthreads();
  for (int k = tid; k < s.top; k += threads) {
    const int id = e.seen[k];
    float sum = 0.0f;
    bool first = id >= 0;
    for (int j = 0; first && j < s.top; ++j)
      if (e.seen[j] == id) {
        first = j >= k;
        sum += e.q[j];
      }
    e.id[k] = first ? id : -1;
    e.sum[k] = sum;
  }
  __syncthreads();
  return te.some();
}

// The entries of a list on top of what the row's lanes wrote.
template <class T>
__device__ __forceinline__ void store_entries(T *dst, const EntryLists &e, float g, const Student &p, const DistillShape &s) {
  for (int k = threadIdx.x; k < s.top; k += blockDim.x)
    if (e.id[k] >= 0) dst[e.id[k]] = (T)(g * (probability_cut(e.z[k], p, s) - e.sum[k]));
}

// The gradient of one range of one token's scores; part: its ranges' statistics (at most 64, joined by every wavefront for
// itself), or null where there is only the lse.
template <class T>
__global__ __launch_bounds__(DST_THREADS) void distill_grad_kernel(T *dlogits, const T *logits,
                                                                   const int *__restrict__ ids,
                                                                   const float *__restrict__ top,
                                                                   const float *__restrict__ lse,
                                                                   const SoftStat *__restrict__ part,
                                                                   const float *__restrict__ loss_grad, DistillShape s) {
  constexpr int V = Num<T>::V;
  extern __shared__ float lists[];
  const EntryLists e = entry_lists(lists, s.top);
  const int t = blockIdx.x / s.splits, cut = blockIdx.x % s.splits;
  const int begin = cut * s.chunk, end = min(s.vocab, begin + s.chunk);
  const T *row = logits + (size_t)t * s.logits_stride;
  T *dst = dlogits + (size_t)t * s.logits_stride;
  const bool weight =
      gather_entries<T>(e, row, ids + (size_t)t * s.top_stride, top + (size_t)t * s.top_stride, begin, end, s);
  const float g = s.temperature * (loss_grad ? loss_grad[t] : 1.0f);
  Student p{0.0f, 0.0f};
  if (part) {
    const int lane = threadIdx.x & 63;
    p = student(wave_join(lane < s.splits ? part[(size_t)t * s.splits + lane] : SoftStat{neg_inf(), 0.0f}, s.scale2));
  } else {
    p.m = lse[t] * s.temperature;
  }
  for (int col = begin + threadIdx.x * V; col < end; col += DST_THREADS * V) {
    float f[V];
    load_vec<T>(f, row, col, end);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = weight ? g * probability_cut(f[i], p, s) : 0.0f;
    store_vec<T>(dst, f, col, end);
  }
  if (!weight) return;
  __syncthreads();
  store_entries<T>(dst, e, g, p, s);
}

// Loss and gradient of whole rows, each read once: a workgroup keeps its row in registers from the statistics to the
// gradient, and fetches its next row into the registers that the gradient has left.  ITEMS vectors a lane; one entry of the
// list a lane (top <= THREADS).  The statistics are taken vector by vector as they arrive, with a running maximum: the
// exponentials (two per score, 16 us of a 128 K row's 26 us of traffic) then run beside the loads and stores, where a pass for
// the maximum first had them wait for the whole row (4096 rows of 131072 bf16 scores: 490 us, 4.4 TB/s, against 585).
template <class T, int THREADS, int ITEMS>
__global__ __launch_bounds__(THREADS) void distill_row_kernel(float *__restrict__ loss, float *__restrict__ lse, T *dlogits,
                                                              const T *logits, const int *__restrict__ ids,
                                                              const float *__restrict__ top,
                                                              const float *__restrict__ loss_grad, DistillShape s) {
  constexpr int V = Num<T>::V, WAVES = THREADS / 64;
  typedef typename Num<T>::vec vec;
  __shared__ SoftStat sh_row[WAVES], sh_top[WAVES];
  __shared__ float sh_loss[WAVES];
  __shared__ int sh_id[THREADS];
  __shared__ float sh_q[THREADS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int whole = s.vocab / V * V;  // the vectors; what is left of the row is one element a lane
  const int tail = whole + tid < s.vocab ? whole + tid : -1;
  const bool entry = tid < s.top;
  vec v[ITEMS];
  T rest = (T)0.0f;
  int id = -1;
  float weight = 0.0f, z = 0.0f;
  auto fetch = [&](int i, const T *row) {
    const int col = (i * THREADS + tid) * V;
    if (col < whole) v[i] = *reinterpret_cast<const vec *>(row + col);
  };
  {
    const int t = blockIdx.x;
    const T *row = logits + (size_t)t * s.logits_stride;
    if (entry) {
      id = ids[(size_t)t * s.top_stride + tid];
      weight = top[(size_t)t * s.top_stride + tid];
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) fetch(i, row);
    if (tail >= 0) rest = row[tail];
    if (id >= 0 && id < s.vocab) z = (float)row[id];
  }
  for (int t = blockIdx.x; t < s.tokens; t += gridDim.x) {
    const bool inside = id >= 0 && id < s.vocab;
    // this lane's part of the row, and the teacher's weights
    SoftStat st{neg_inf(), 0.0f};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if ((i * THREADS + tid) * V < whole) {
        float f[V];
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = (float)v[i][k];
        add_values<V>(st, f, s.scale2);
      }
    if (tail >= 0) {
      const float f[1] = {(float)rest};
      add_values<1>(st, f, s.scale2);
    }
    st = wave_join(st, s.scale2);
    SoftStat te{id >= 0 ? weight : neg_inf(), 0.0f};
    te.s = te.m == neg_inf() ? 0.0f : 1.0f + (weight - weight);  // NaN for a weight that is one, or infinite
    te = wave_join(te, s.scale2);
    if (lane == 0) {
      sh_row[wave] = st;
      sh_top[wave] = te;
    }
    const bool bad = __syncthreads_or(entry && id >= s.vocab);
    st = lane < WAVES ? sh_row[lane] : SoftStat{neg_inf(), 0.0f};
    te = lane < WAVES ? sh_top[lane] : SoftStat{neg_inf(), 0.0f};
#pragma unroll
    for (int d = WAVES / 2; d > 0; d >>= 1) {
      st = shfl_xor_join(st, d, s.scale2);
      te = shfl_xor_join(te, d, s.scale2);
    }
    st.m = __shfl(st.m, 0, 64);
    st.s = __shfl(st.s, 0, 64);
    te.m = __shfl(te.m, 0, 64);
    te.s = __shfl(te.s, 0, 64);
    const float l = log_sum(st, s.inv_t);
    const Student p = student(st);
    const Teacher teacher{te.m, te.s, false};
    const bool some = teacher.some();
    // this lane's entry
    const float q = teacher_weight(teacher, id, weight, s.scale2);
    float term = 0.0f;
    if (inside && q != 0.0f)
      term = q * (((weight - te.m) * s.inv_t - __builtin_log2f(te.s) * kLn2) + label_loss(st, z, s.inv_t));
    const bool mine = inside && q != 0.0f;
    sh_id[tid] = mine ? id : -1;
    sh_q[tid] = q;
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) term += __shfl_xor(term, m, 64);
    if (lane == 0) sh_loss[wave] = term;
    __syncthreads();
    // equal ids are one entry of the gradient: the first of them, with the weight of all
    bool first = mine;
    float sum = 0.0f;
    for (int j = 0; first && j < s.top; ++j)
      if (sh_id[j] == id) {
        first = j >= tid;
        sum += sh_q[j];
      }
    const float g = s.temperature * (loss_grad ? loss_grad[t] : 1.0f);
    T *dst = dlogits + (size_t)t * s.logits_stride;
    const float entry_grad = g * (probability(z, p, s) - sum);
    const int entry_id = id;
    const int next = t + (int)gridDim.x;
    const bool more = next < s.tokens;
    const T *next_row = logits + (size_t)(more ? next : t) * s.logits_stride;
    if (entry && more) {
      id = ids[(size_t)next * s.top_stride + tid];
      weight = top[(size_t)next * s.top_stride + tid];
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int col = (i * THREADS + tid) * V;
      if (col < whole) {
        vec out;
#pragma unroll
        for (int k = 0; k < V; ++k) out[k] = (T)(some ? g * probability((float)v[i][k], p, s) : 0.0f);
        __builtin_nontemporal_store(out, reinterpret_cast<vec *>(dst + col));
      }
      if (more) fetch(i, next_row);
    }
    if (tail >= 0) {
      dst[tail] = (T)(some ? g * probability((float)rest, p, s) : 0.0f);
      if (more) rest = next_row[tail];
    }
    if (more && id >= 0 && id < s.vocab) z = (float)next_row[id];
    __syncthreads();  // the entry goes on top of what the row's lanes wrote
    if (first && some) dst[entry_id] = (T)entry_grad;
    if (tid == 0) {
      float sum_loss = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) sum_loss += sh_loss[w];
      lse[t] = l;
      loss[t] = bad ? __builtin_nanf("") : s.temperature * s.temperature * sum_loss;
    }
  }
}

static int check_distill(const cct_distill_loss_args *a, const char *who) {
  CCT_REQUIRE(a != nullptr, "%s: null argument block", who);
  CCT_REQUIRE(a->dtype == CCT_F32 || a->dtype == CCT_BF16, "%s: dtype %d is neither CCT_F32 nor CCT_BF16", who, a->dtype);
  CCT_REQUIRE(a->tokens >= 0 && a->vocab > 0 && a->top > 0, "%s: tokens %d, vocab %d, top %d", who, a->tokens, a->vocab,
              a->top);
  CCT_REQUIRE(a->top <= DST_TOP_MAX, "%s: top %d is above %d", who, a->top, DST_TOP_MAX);
  CCT_REQUIRE(a->tokens <= (1 << 20) && a->vocab <= (1 << 26), "%s: tokens %d, vocab %d: at most 2^20, 2^26", who,
              a->tokens, a->vocab);
  CCT_REQUIRE(a->temperature > 0.0f && a->temperature < __builtin_inff(), "%s: temperature %g is not a positive number", who,
              (double)a->temperature);
  // T^2, 1 / T and log2 e / T are normal numbers
  CCT_REQUIRE(a->temperature >= 0x1p-60f && a->temperature <= 0x1p60f, "%s: temperature %g is not within 2^-60 to 2^60", who,
              (double)a->temperature);
  CCT_REQUIRE((a->logits_stride == 0 || a->logits_stride >= (size_t)a->vocab) &&
                  (a->top_stride == 0 || a->top_stride >= (size_t)a->top),
              "%s: a row stride is smaller than its row", who);
  return 0;
}

static DistillShape distill_shape(const cct_distill_loss_args *a) {
  DistillShape s;
  s.tokens = a->tokens;
  s.vocab = a->vocab;
  s.top = a->top;
  s.temperature = a->temperature;
  s.inv_t = (float)(1.0 / (double)a->temperature);
  s.scale2 = (float)(1.4426950408889634 / (double)a->temperature);
  s.logits_stride = a->logits_stride ? a->logits_stride : (size_t)a->vocab;
  s.top_stride = a->top_stride ? a->top_stride : (size_t)a->top;
  // enough ranges to give each of 256 CUs several workgroups, none shorter than 4096 elements
  const int per = 8192 / (a->tokens > 0 ? a->tokens : 1) + 1;
  int splits = (a->vocab + 4095) / 4096;
  if (splits > per) splits = per;
  if (splits > 64) splits = 64;
  if (splits < 1) splits = 1;
  const int chunk = (a->vocab + splits - 1) / splits;
  s.chunk = (chunk + 7) & ~7;
  s.splits = (a->vocab + s.chunk - 1) / s.chunk;
  return s;
}

static size_t distill_bytes(const cct_distill_loss_args *a) {
  const DistillShape s = distill_shape(a);
  return (size_t)s.tokens * s.splits * sizeof(SoftStat);
}

template <class T>
static int distill_forward(float *loss, float *lse, const void *logits, const int *ids, const float *top,
                           const DistillShape &s, void *ws, bool keep_stats) {
  hipStream_t st = ctx().stream;
  if (s.splits == 1 && !keep_stats) {
    distill_token_kernel<T><<<s.tokens, DST_THREADS, 0, st>>>(loss, lse, (const T *)logits, ids, top, s);
    CCT_LAUNCH_CHECK();
    note_kernel("distill_token_kernel<%s>", Num<T>::NAME);
    return 0;
  }
  SoftStat *part = (SoftStat *)ws;
  distill_stats_kernel<T><<<(unsigned)s.tokens * s.splits, DST_THREADS, 0, st>>>(part, (const T *)logits, s);
  CCT_LAUNCH_CHECK();
  distill_loss_kernel<T><<<(s.tokens + DST_WAVES - 1) / DST_WAVES, DST_THREADS, 0, st>>>(loss, lse, part,
                                                                                       (const T *)logits, ids, top, s);
  CCT_LAUNCH_CHECK();
  note_kernel("distill_stats_kernel<%s> splits=%d", Num<T>::NAME, s.splits);
  return 0;
}

template <class T>
static int distill_backward(void *dlogits, const void *logits, const int *ids, const float *top, const float *lse,
                            const SoftStat *part, const float *loss_grad, const DistillShape &s) {
  distill_grad_kernel<T><<<(unsigned)s.tokens * s.splits, DST_THREADS, 5 * s.top * sizeof(float), ctx().stream>>>(
      (T *)dlogits, (const T *)logits, ids, top, lse, part, loss_grad, s);
  CCT_LAUNCH_CHECK();
  note_kernel("distill_grad_kernel<%s> splits=%d", Num<T>::NAME, s.splits);
  return 0;
}

// Rows that one workgroup holds in its registers (16 vectors a lane at most); longer rows are read twice.  One launch beats the
// three of the split form for a single row too (a CU alone moves a row of 128 K bf16 scores in 6 us).
template <class T>
static int distill_both(float *loss, float *lse, void *dlogits, const void *logits, const int *ids, const float *top,
                        const float *loss_grad, const DistillShape &s, void *ws) {
  const int vecs = s.vocab / Num<T>::V;
#define CCT_DISTILL_ROW(THREADS, ITEMS, GROUPS)                                                                            \
  if (vecs <= THREADS * ITEMS && s.top <= THREADS) {                                                                      \
    const int grid = min(s.tokens, 256 * GROUPS);                                                                        \
    distill_row_kernel<T, THREADS, ITEMS><<<grid, THREADS, 0, ctx().stream>>>(                     \
        loss, lse, (T *)dlogits, (const T *)logits, ids, top, loss_grad, s);                                              \
    CCT_LAUNCH_CHECK();                                                                                                   \
    note_kernel("distill_row_kernel<%s, %d, %d> grid=%d", Num<T>::NAME, THREADS, ITEMS, grid);                             \
    return 0;                                                                                                             \
  }
  CCT_DISTILL_ROW(256, 4, 8)
  CCT_DISTILL_ROW(512, 8, 2)
  CCT_DISTILL_ROW(1024, 8, 1)
  CCT_DISTILL_ROW(1024, 16, 1)
#undef CCT_DISTILL_ROW
  if (int rc = distill_forward<T>(loss, lse, logits, ids, top, s, ws, true)) return rc;
  return distill_backward<T>(dlogits, logits, ids, top, lse, (const SoftStat *)ws, loss_grad, s);
}

static int check_distill_workspace(const cct_distill_loss_args *a, const void *ws, size_t bytes, const char *who) {
  const size_t need = distill_bytes(a);
  CCT_REQUIRE(bytes >= need && (ws || need == 0) && ((uintptr_t)ws & 15) == 0,
              "%s: the workspace holds %zu bytes and starts at %p; it needs %zu, aligned to 16", who, bytes, ws, need);
  return 0;
}

}  // namespace cct

using namespace cct;

extern "C" size_t cct_hip_distill_loss_workspace_bytes(const cct_distill_loss_args *args) {
  return check_distill(args, "distill_loss_workspace_bytes") ? 0 : distill_bytes(args);
}

extern "C" int cct_hip_distill_loss_forward(float *loss, float *lse, const void *logits, const int *top_ids,
                                            const float *top_logits, const cct_distill_loss_args *args, void *workspace,
                                            size_t workspace_bytes) {
  if (int rc = check_distill(args, "distill_loss_forward")) return rc;
  if (args->tokens == 0) return 0;
  CCT_REQUIRE(loss && lse && logits && top_ids && top_logits, "distill_loss_forward: null array");
  if (int rc = check_distill_workspace(args, workspace, workspace_bytes, "distill_loss_forward")) return rc;
  CCT_ENSURE_INIT();
  const DistillShape s = distill_shape(args);
  return args->dtype == CCT_BF16 ? distill_forward<bf16>(loss, lse, logits, top_ids, top_logits, s, workspace, false)
                                 : distill_forward<float>(loss, lse, logits, top_ids, top_logits, s, workspace, false);
}

extern "C" int cct_hip_distill_loss_backward(void *dlogits, const void *logits, const int *top_ids, const float *top_logits,
                                             const float *lse, const float *loss_grad, const cct_distill_loss_args *args,
                                             void *workspace, size_t workspace_bytes) {
  if (int rc = check_distill(args, "distill_loss_backward")) return rc;
  if (args->tokens == 0) return 0;
  CCT_REQUIRE(dlogits && lse && logits && top_ids && top_logits, "distill_loss_backward: null array");
  if (int rc = check_distill_workspace(args, workspace, workspace_bytes, "distill_loss_backward")) return rc;
  CCT_ENSURE_INIT();
  const DistillShape s = distill_shape(args);
  return args->dtype == CCT_BF16 ? distill_backward<bf16>(dlogits, logits, top_ids, top_logits, lse, nullptr, loss_grad, s)
                                 : distill_backward<float>(dlogits, logits, top_ids, top_logits, lse, nullptr, loss_grad, s);
}

extern "C" int cct_hip_distill_loss_forward_backward(float *loss, float *lse, void *dlogits, const void *logits,
                                                     const int *top_ids, const float *top_logits, const float *loss_grad,
                                                     const cct_distill_loss_args *args, void *workspace,
                                                     size_t workspace_bytes) {
  const char *who = "distill_loss_forward_backward";
  if (int rc = check_distill(args, who)) return rc;
  if (args->tokens == 0) return 0;
  CCT_REQUIRE(loss && lse && dlogits && logits && top_ids && top_logits, "%s: null array", who);
  if (int rc = check_distill_workspace(args, workspace, workspace_bytes, who)) return rc;
  CCT_ENSURE_INIT();
  const DistillShape s = distill_shape(args);
  return args->dtype == CCT_BF16
             ? distill_both<bf16>(loss, lse, dlogits, logits, top_ids, top_logits, loss_grad, s, workspace)
             : distill_both<float>(loss, lse, dlogits, logits, top_ids, top_logits, loss_grad, s, workspace);
}
