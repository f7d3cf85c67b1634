// What stands behind a vocabulary head (gfx950): log probabilities of given
// tokens with entropy and top alternatives, and the distillation loss from a
// teacher's top logits, both forward and backward.
//
// A row x of V logits at temperature T, all in fp32 whatever the logits' type:
//   M = max x_i,  L = log sum exp((x_i - M) / T),  lp_i = (x_i - M) / T - L
//   logprob = lp_t,   H = L - sum exp((x_i - M) / T) ((x_i - M) / T) / exp(L)
//   dx_i = (g ([i = t] - p_i) - gH p_i (lp_i + H)) / T
//   top-k: by (value, lower index); NaN above every number, as torch sorts it
//   loss = sum_j q_j (log q_j - lp_{id_j}),  q = softmax(teacher / T) over the used slots
//   dx_i = g (p_i - sum_{j: id_j = i} q_j) / T
// M and L are kept apart: their sum would lose L where |M| is large (a row of
// the type's lowest value).  Subtracting M before the division by T keeps
// every finite row finite.
//
// Defined edges: a row whose target is `ignore` is neither read nor gives a
// gradient (0, ids -1); a row of only -inf has logprob -inf, entropy 0 and no
// gradient; NaN or +inf in a row, or a target out of range, makes its results
// NaN; a teacher row without a used slot (id -1) or with only -inf gives
// loss 0 and no gradient.
#include "common.h"

namespace {

constexpr int NT = 256;
constexpr int TOP_MAX = 128;      // alternatives a row: at most one a thread

// order of a value as an unsigned number: -inf lowest, NaN highest, -0 as +0;
// 0 itself is no value's
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// unique a row: larger value first, then the lower index
__device__ __forceinline__ uint64_t full_key(float v, uint32_t i) {
  return ((uint64_t)order_key(v) << 32) | (uint32_t)~i;
}

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();                       // red may still be read from the last call
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
  for (int i = 1; i < NT / 64; ++i) r += red[i];
  return r;
}
__device__ __forceinline__ float block_max(float v, float* red) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
  for (int i = 1; i < NT / 64; ++i) r = fmaxf(r, red[i]);
  return r;
}
__device__ __forceinline__ uint64_t block_max_key(uint64_t v, uint64_t* red) {
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor((unsigned long long)v, o, 64);
    v = u > v ? u : v;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t r = red[0];
  for (int i = 1; i < NT / 64; ++i) r = red[i] > r ? red[i] : r;
  return r;
}

// lp_i; -inf in a row of only -inf
__device__ __forceinline__ float log_prob(float x, float M, float L, float inv_t) {
  return M == -INFINITY ? -INFINITY : (x - M) * inv_t - L;
}

struct Row {
  const void* x;
  long long ld, rows, V;
  float inv_t;
};

// M, L and sum exp(d) d / sum exp(d) of a row, d = (x - M) / T
template <int DT>
__device__ __forceinline__ void row_stats(const typename DTypeTraits<DT>::raw_t* x, long long V,
                                          float inv_t, float* red, float& M, float& L, float& t) {
  float m = -INFINITY;
  for (long long i = threadIdx.x; i < V; i += NT) m = fmaxf(m, DTypeTraits<DT>::to_f32(x[i]));
  M = block_max(m, red);
  const float base = M == -INFINITY ? 0.f : M;
  float s = 0.f, a = 0.f;
  for (long long i = threadIdx.x; i < V; i += NT) {
    const float d = (DTypeTraits<DT>::to_f32(x[i]) - base) * inv_t;
    const float e = __expf(d);
    s += e;
    a = fmaf(e, fmaxf(d, -1e30f), a);    // exp(-inf) = 0 times a finite number
  }
  s = block_sum(s, red);
  a = block_sum(a, red);
  L = logf(s);
  t = a / s;
}

struct LogprobArgs {
  Row r;
  const long long* targets;
  long long ignore;
  float *logprob, *entropy, *top_lp, *stats;
  long long* top_ids;
  int k;
};

template <int DT>
__global__ __launch_bounds__(NT) void logprob_fwd_kernel(const LogprobArgs a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  __shared__ float red[NT / 64];
  __shared__ uint64_t redk[NT / 64];
  const long long row = blockIdx.x;
  const raw_t* x = (const raw_t*)a.r.x + row * a.r.ld;
  const long long tgt = a.targets ? a.targets[row] : 0;
  if (a.targets && tgt == a.ignore) {
    if (threadIdx.x < a.k) {
      a.top_lp[row * a.k + threadIdx.x] = -INFINITY;
      a.top_ids[row * a.k + threadIdx.x] = -1;
    }
    if (threadIdx.x == 0) {
      if (a.logprob) a.logprob[row] = 0.f;
      if (a.entropy) a.entropy[row] = 0.f;
      a.stats[2 * row] = -INFINITY;
      a.stats[2 * row + 1] = 0.f;
    }
    return;
  }
  float M, L, t;
  row_stats<DT>(x, a.r.V, a.r.inv_t, red, M, L, t);
  if (threadIdx.x == 0) {
    const bool bad = tgt < 0 || tgt >= a.r.V;
    if (a.logprob)
      a.logprob[row] = bad ? NAN : log_prob(DTypeTraits<DT>::to_f32(x[tgt]), M, L, a.r.inv_t);
    if (a.entropy) a.entropy[row] = M == -INFINITY ? 0.f : L - t;
    a.stats[2 * row] = M;
    a.stats[2 * row + 1] = L;
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < a.k; ++j) {
    uint64_t best = 0;
    for (long long i = threadIdx.x; i < a.r.V; i += NT) {
      const uint64_t key = full_key(DTypeTraits<DT>::to_f32(x[i]), (uint32_t)i);
      if (key < last && key > best) best = key;
    }
    last = block_max_key(best, redk);
    if (threadIdx.x == 0) {
      const long long id = (uint32_t)~(uint32_t)last;
      a.top_ids[row * a.k + j] = id;
      a.top_lp[row * a.k + j] = log_prob(DTypeTraits<DT>::to_f32(x[id]), M, L, a.r.inv_t);
    }
  }
}

struct LogprobBwd {
  Row r;
  const long long* targets;
  long long ignore;
  const float *stats, *entropy, *g, *gh;
  long long gs, ghs;
  void* dx;
};

template <int DT>
__global__ __launch_bounds__(NT) void logprob_bwd_kernel(const LogprobBwd a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  const long long row = blockIdx.x, V = a.r.V;
  const raw_t* x = (const raw_t*)a.r.x + row * a.r.ld;
  raw_t* dx = (raw_t*)a.dx + row * V;
  const long long tgt = a.targets ? a.targets[row] : 0;
  const float M = a.stats[2 * row], L = a.stats[2 * row + 1];
  const bool zero = (a.targets && tgt == a.ignore) || M == -INFINITY;
  float g = a.g ? a.g[row * a.gs] : 0.f;
  if (a.g && (tgt < 0 || tgt >= V)) g = NAN;
  const float gh = a.gh ? a.gh[row * a.ghs] : 0.f, H = a.gh ? a.entropy[row] : 0.f;
  for (long long i = threadIdx.x; i < V; i += NT) {
    float v = 0.f;
    if (!zero) {
      const float lp = (DTypeTraits<DT>::to_f32(x[i]) - M) * a.r.inv_t - L;
      v = -__expf(lp) * (g + gh * (fmaxf(lp, -1e30f) + H));
      if (a.g && i == tgt) v += g;
      v *= a.r.inv_t;
    }
    dx[i] = DTypeTraits<DT>::from_f32(v);
  }
}

// The teacher's side of a row: slot j in thread j.  Returns false for a row
// without a used slot (or with only -inf); q, log q of the thread's slot
// (0, -inf for an unused one).  bad: an id out of range, or NaN.
__device__ __forceinline__ float teacher_value(const void* t, long long i, int dt) {
  if (dt == KDT_F32) return ((const float*)t)[i];
  const uint16_t v = ((const uint16_t*)t)[i];
  return dt == KDT_BF16 ? bf16_bits_to_f32(v) : f16_bits_to_f32(v);
}

struct Teacher {
  const long long* ids;
  const void* t;
  int dt, K;
};

__device__ __forceinline__ bool teacher_row(const Teacher& h, long long row, long long V,
                                            float inv_t, float* red, long long& id, float& q,
                                            float& logq) {
  const int j = threadIdx.x;
  id = j < h.K ? h.ids[row * h.K + j] : -1;
  float t = id == -1 ? -INFINITY : teacher_value(h.t, row * h.K + j, h.dt);
  if (id < -1 || id >= V) { t = NAN; id = -1; }
  const float top = block_max(t, red);
  const float nan = block_sum(t != t ? 1.f : 0.f, red);
  if (top == -INFINITY && nan == 0.f) return false;
  const float d = (t - top) * inv_t;
  const float Z = block_sum(__expf(d), red);
  q = __expf(d) / Z;
  logq = d - logf(Z);
  return true;
}

struct DistillArgs {
  Row r;
  Teacher h;
  float *loss, *stats;
};

template <int DT>
__global__ __launch_bounds__(NT) void distill_fwd_kernel(const DistillArgs a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  __shared__ float red[NT / 64];
  const long long row = blockIdx.x;
  const raw_t* x = (const raw_t*)a.r.x + row * a.r.ld;
  long long id;
  float q, logq, M, L, t;
  if (!teacher_row(a.h, row, a.r.V, a.r.inv_t, red, id, q, logq)) {
    if (threadIdx.x == 0) {
      a.loss[row] = 0.f;
      a.stats[2 * row] = -INFINITY;
      a.stats[2 * row + 1] = 0.f;
    }
    return;
  }
  row_stats<DT>(x, a.r.V, a.r.inv_t, red, M, L, t);
  float term = 0.f;
  if (q != 0.f)
    term = q * (logq - (id < 0 ? NAN : log_prob(DTypeTraits<DT>::to_f32(x[id]), M, L, a.r.inv_t)));
  term = block_sum(term, red);
  if (threadIdx.x == 0) {
    a.loss[row] = term;
    a.stats[2 * row] = M;
    a.stats[2 * row + 1] = L;
  }
}

struct DistillBwd {
  Row r;
  Teacher h;
  const float *stats, *g;
  long long gs;
  void* dx;
};

template <int DT>
__global__ __launch_bounds__(NT) void distill_bwd_kernel(const DistillBwd a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  __shared__ float red[NT / 64];
  __shared__ long long ids[TOP_MAX];
  __shared__ float qs[TOP_MAX];
  const long long row = blockIdx.x, V = a.r.V;
  const raw_t* x = (const raw_t*)a.r.x + row * a.r.ld;
  raw_t* dx = (raw_t*)a.dx + row * V;
  long long id;
  float q = 0.f, logq;
  const bool some = teacher_row(a.h, row, V, a.r.inv_t, red, id, q, logq);
  const float M = a.stats[2 * row], L = a.stats[2 * row + 1];
  const bool zero = !some || M == -INFINITY;
  const float g = a.g[row * a.gs] * a.r.inv_t;
  // an id out of range or NaN in the teacher's row made every q NaN
  const float all = some && block_sum(q, red) != block_sum(q, red) ? NAN : 1.f;
  for (long long i = threadIdx.x; i < V; i += NT) {
    float v = 0.f;
    if (!zero) v = g * all * __expf((DTypeTraits<DT>::to_f32(x[i]) - M) * a.r.inv_t - L);
    dx[i] = DTypeTraits<DT>::from_f32(v);
  }
  if (zero) return;
  if (threadIdx.x < a.h.K) {
    ids[threadIdx.x] = id;
    qs[threadIdx.x] = q;
  }
  __syncthreads();                       // dx of the row is written, too
  if (threadIdx.x < a.h.K && id >= 0) {
    // the same id twice: its masses are added in slot order, by its first slot
    float sum = 0.f;
    bool first = true;
    for (int j = 0; j < a.h.K; ++j)
      if (ids[j] == id) {
        if (j < (int)threadIdx.x) first = false;
        sum += qs[j];
      }
    if (first) {
      const float p = __expf((DTypeTraits<DT>::to_f32(x[id]) - M) * a.r.inv_t - L);
      dx[id] = DTypeTraits<DT>::from_f32(g * (p - sum));
    }
  }
}

bool row_ok(const Row& r, int dt) {
  return r.x && r.rows > 0 && r.rows <= 0x7fffffffLL && r.V > 0 && r.V <= 0x7fffffffLL &&
         r.inv_t > 0.f && (dt == KDT_F32 || dt == KDT_BF16 || dt == KDT_F16);
}
bool teacher_ok(const Teacher& h) {
  return h.ids && h.t && h.K > 0 && h.K <= TOP_MAX &&
         (h.dt == KDT_F32 || h.dt == KDT_BF16 || h.dt == KDT_F16);
}

}  // namespace

#define VOCAB_LAUNCH(kernel, dt, grid, stream, args)                                          \
  do {                                                                                        \
    if (dt == KDT_F32)                                                                        \
      hipLaunchKernelGGL(kernel<KDT_F32>, grid, dim3(NT), 0, stream, args);                   \
    else if (dt == KDT_BF16)                                                                  \
      hipLaunchKernelGGL(kernel<KDT_BF16>, grid, dim3(NT), 0, stream, args);                  \
    else                                                                                      \
      hipLaunchKernelGGL(kernel<KDT_F16>, grid, dim3(NT), 0, stream, args);                   \
  } while (0)

KFAC_API int kfac_vocab_top_max() { return TOP_MAX; }

// targets null: no logprob; entropy null: none; k 0: no alternatives.
// stats: (M, L) a row, for the backward pass.
KFAC_API int kfac_logprob_forward(const void* x, long long ld, int dt, long long rows,
                                  long long V, float inv_t, const long long* targets,
                                  long long ignore, int k, float* logprob, float* entropy,
                                  float* top_lp, long long* top_ids, float* stats,
                                  hipStream_t stream) {
  LogprobArgs a = {{x, ld, rows, V, inv_t}, targets, ignore, logprob, entropy, top_lp, stats,
                   top_ids, k};
  if (!row_ok(a.r, dt) || !stats || k < 0 || k > TOP_MAX || k > V || (logprob && !targets) ||
      (k && (!top_lp || !top_ids)))
    return -2;
  VOCAB_LAUNCH(logprob_fwd_kernel, dt, dim3((unsigned)rows), stream, a);
  return (int)hipGetLastError();
}

// g, gh: gradients of logprob and entropy, one a row at a distance of gs, ghs
// elements (0: the same for every row); either may be null
KFAC_API int kfac_logprob_backward(const void* x, long long ld, int dt, long long rows,
                                   long long V, float inv_t, const long long* targets,
                                   long long ignore, const float* stats, const float* entropy,
                                   const float* g, long long gs, const float* gh, long long ghs,
                                   void* dx, hipStream_t stream) {
  LogprobBwd a = {{x, ld, rows, V, inv_t}, targets, ignore, stats, entropy, g, gh, gs, ghs, dx};
  if (!row_ok(a.r, dt) || !stats || !dx || (g && !targets) || (gh && !entropy)) return -2;
  VOCAB_LAUNCH(logprob_bwd_kernel, dt, dim3((unsigned)rows), stream, a);
  return (int)hipGetLastError();
}

KFAC_API int kfac_distill_forward(const void* x, long long ld, int dt, long long rows,
                                  long long V, float inv_t, const long long* ids,
                                  const void* teacher, int tdt, int K, float* loss, float* stats,
                                  hipStream_t stream) {
  DistillArgs a = {{x, ld, rows, V, inv_t}, {ids, teacher, tdt, K}, loss, stats};
  if (!row_ok(a.r, dt) || !teacher_ok(a.h) || !loss || !stats) return -2;
  VOCAB_LAUNCH(distill_fwd_kernel, dt, dim3((unsigned)rows), stream, a);
  return (int)hipGetLastError();
}

KFAC_API int kfac_distill_backward(const void* x, long long ld, int dt, long long rows,
                                   long long V, float inv_t, const long long* ids,
                                   const void* teacher, int tdt, int K, const float* stats,
                                   const float* g, long long gs, void* dx, hipStream_t stream) {
  DistillBwd a = {{x, ld, rows, V, inv_t}, {ids, teacher, tdt, K}, stats, g, gs, dx};
  if (!row_ok(a.r, dt) || !teacher_ok(a.h) || !stats || !g || !dx) return -2;
  VOCAB_LAUNCH(distill_bwd_kernel, dt, dim3((unsigned)rows), stream, a);
  return (int)hipGetLastError();
}
