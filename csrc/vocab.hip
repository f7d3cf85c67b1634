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
// Forward: ONE pass over the row.  A thread keeps the running maximum m of its
// elements, s = sum exp((x - m) / T) and a = sum exp((x - m) / T) (x - m) / T, each
// brought to a new maximum once per tile of 16 elements; the threads'
// (m, s, a) are joined at the end.  The alternatives need no second pass: the
// k-th largest of the threads' maxima is a bound that at least k elements
// reach, and of the threads that reach it only the runs of tiles whose maximum
// does are looked at again: about k of 2048.  A row is cut over several
// workgroups where there are few rows, and joined by a second kernel.
// Backward: one read and one write of the row from the saved (M, L).
//
// Both are bound by HBM: 4 to 8 instructions and one exponential an element are
// about 60 % of the time that a 16-bit element takes to arrive.
//
// Times below are medians of a kernel's launches on one MI355X, three sets of inputs
// in turn; of two sides, both with the code as it stands but for the choice.
//
// Defined edges: a row whose target is `ignore` is neither read nor gives a
// gradient (0, ids -1); a row of only -inf has logprob -inf, entropy 0 and no
// gradient; NaN or +inf in a row makes its results and its gradient NaN (a row of
// only NaN, or of NaN and -inf, too), a target out of range its logprob and the
// logprob's gradient; a teacher row without a used slot (id -1) or with only -inf
// gives loss 0 and no gradient.
#include "records.h"
#include "rows.h"

namespace {

typedef KfacVocabFwd Fwd;
typedef KfacVocabBwd Bwd;

constexpr int TOP_MAX = 128;      // alternatives, and slots of a teacher's row
constexpr int MAX_V = 1 << 30;    // elements of a row: 32-bit offsets within it
constexpr int MAX_SPLITS = 64;    // workgroups a row
// workgroups a launch, which has fewer than 2^32 threads: more rows take several launches
constexpr long long MAX_GROUPS = 1 << 22;
// Logits that the 256 MB of last-level cache cannot hold beside their gradient
// are read past it (non-temporal): the backward pass would not find them there.
// us forward + backward, streamed | not: 4096 x 131072 bf16 169 + 366 | 216 + 347,
// 8192 x 50001 bf16 146 + 285 | 177 + 276, 2048 x 32064 fp32 52 + 92 | 75 + 81, 16384 x
// 16000 bf16 101 + 214 | 130 + 199; 700 x 10000 fp32, which it holds, 9 + 11 unstreamed.
constexpr long long STREAM_FROM = 128LL << 20;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// An exponent far below what exp2 gives 0 for, whose product with that 0 is 0.
constexpr float LOWEST = -1e9f;

enum Mode { LOGPROB = 0, DISTILL = 1 };

// order of a value as an unsigned number: -inf lowest, NaN highest, -0 as +0;
// 0 itself is no value's
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// unique a row: larger value first, then the lower index
__device__ __forceinline__ uint64_t full_key(float v, uint32_t i) {
  return ((uint64_t)order_key(v) << 32) | (uint32_t)~i;
}

// One workgroup of NT threads: reductions to every thread, in a fixed order.
template <int NT> struct Group {
  static __device__ __forceinline__ float sum(float v, float* red) {
    v = wave_sum(v);
    if (NT <= 64) return v;
    __syncthreads();                     // red may still be read from the last call
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) r += red[i];
    return r;
  }
  static __device__ __forceinline__ float max(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    if (NT <= 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) r = fmaxf(r, red[i]);
    return r;
  }
};

// lp_i; -inf in a row of only -inf
__device__ __forceinline__ float log_prob(float x, float M, float L, float inv_t) {
  return M == -INFINITY ? -INFINITY : (x - M) * inv_t - L;
}

// A part of a row: what one of the `splits` workgroups of a row hands on.
struct Part { float m, s, a, pad; };

// Elements i .. i + V - 1 of a row of n, -inf from `end` on.
template <int DT>
__device__ __forceinline__ void fetch(const AS1 typename DTypeTraits<DT>::raw_t* x, int i, int end,
                                      int n, float* f) {
  constexpr int V = row_vec<DT>();
  if (n < V) {                           // no 16 bytes in the whole row
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = i + e < end ? DTypeTraits<DT>::to_f32(x[i + e]) : -INFINITY;
    return;
  }
  vec_to_f32<DT>(clip_vec<DT, true>(load_vec<DT, true>(x, i, n), i, n), f);
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (i + e >= end) f[e] = -INFINITY;
}

// The running (m, s, a) of one thread over N more elements: s = sum e^(..),
// a = sum e^(..) u with u = (x - m) / T in units of log 2.  c1 = log2 e / T.
// Both return the elements' maximum.
template <int N, bool ENT>
__device__ __forceinline__ float raise(const float* f, float c1, float& m, float& s, float& a) {
  float tile = f[0];
#pragma unroll
  for (int e = 1; e < N; ++e) tile = fmaxf(tile, f[e]);
  const float top = fmaxf(m, tile);
  const float back = fmaxf((m - (top == -INFINITY ? 0.f : top)) * c1, LOWEST);
  const float scale = __builtin_amdgcn_exp2f(back);
  if (ENT) a = scale * fmaf(back, s, a);
  s *= scale;
  m = top;
  return tile;
}
template <int N, bool ENT>
__device__ __forceinline__ void add_any(const float* f, float c1, float m, float& s, float& a) {
  const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float u = (f[e] - base) * c1, x = __builtin_amdgcn_exp2f(u);
    s += x;
    if (ENT) a = fmaf(x, fmaxf(u, LOWEST), a);        // exp(-inf) = 0 times a finite number
  }
}
template <int N, bool ENT>
__device__ __forceinline__ float fold_any(const float* f, float c1, float& m, float& s, float& a) {
  const float tile = raise<N, ENT>(f, c1, m, s, a);
  add_any<N, ENT>(f, c1, m, s, a);
  return tile;
}
// The same with one instruction less an element, u' = x c1 - R with R = m c1
// rounded: every u' of the tile is off by the same d = m c1 - R, which is known
// exactly and taken out of the sums.  Not where R is so large that d is no
// small number (or no number), and not where an entropy's product meets a -inf.
template <int N, bool ENT>
__device__ __forceinline__ float fold(const float* f, float c1, float& m, float& s, float& a) {
  const float tile = raise<N, ENT>(f, c1, m, s, a);
  const float R = m * c1;
  if (!__any(!(fabsf(R) < 0x1p20f))) {
    float st = 0.f, at = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float u = fmaf(f[e], c1, -R), x = __builtin_amdgcn_exp2f(u);
      st += x;
      if (ENT) at = fmaf(x, u, at);
    }
    if (!ENT || !__any(at != at)) {
      const float d = fmaf(m, c1, -R), fix = __builtin_amdgcn_exp2f(-d);
      s = fmaf(st, fix, s);
      if (ENT) a = fmaf(fmaf(-d, st, at), fix, a);
      return tile;
    }
  }
  add_any<N, ENT>(f, c1, m, s, a);
  return tile;
}

// How a workgroup walks a chunk of a row: whole 16-byte lines from the first
// one on, element head + (j NT + thread) V in access j; the fewer than V
// elements before that line are the last thread's, so that 8192 x 50001 bf16 takes as
// long as x 50000, 143 and 145 us.  (With accesses at odd multiples of two bytes, 1.4 times.)
template <int DT> struct Walk {
  int begin, end, n, head;        // chunk, row's length, first line's element
  template <class P> __device__ __forceinline__ Walk(P x, int b, int e, int len) {
    constexpr int V = row_vec<DT>(), ES = 16 / V;
    const int past = (int)(((uintptr_t)(x + b) & 15) / ES);
    begin = b;
    end = e;
    n = len;
    head = past ? b + V - past : b;
    if (head > e) head = e;
  }
};

// A tile is 16 elements a thread (us with 32 | 16: 8192 x 50001 bf16 139 | 132, with
// entropy 138 | 138, with 32 alternatives too 332 | 164; 32768 x 2000 33 | 30, 4096 x
// 131072 159 | 160).  Of the largest values of a thread's elements SLOTS are kept, each
// of a run of tiles.
constexpr int SLOTS = 8;

template <int DT, int NT, bool ENT, bool TOP>
__device__ __forceinline__ void scan(const AS1 typename DTypeTraits<DT>::raw_t* x,
                                     const Walk<DT> w, bool stream, float c1, int shift,
                                     float (*slot)[NT], float& m, float& s, float& a) {
  constexpr int V = row_vec<DT>(), U = 16 / V, STEP = NT * V;
  m = -INFINITY;
  s = a = 0.f;
  float run = -INFINITY;
  int tile = 0, at = w.head;
  // two loops: one with a choice of loads in it ends with plain ones in both
  auto tiles = [&](auto load) {
    u32x4n nxt[U];                 // the next tile's loads are in flight over this one's work
    const AS1 u32x4u* p = (const AS1 u32x4u*)(x + at + threadIdx.x * V);
    if (at + U * STEP <= w.end) {
#pragma unroll
      for (int u = 0; u < U; ++u) nxt[u] = load(p + u * NT);
    }
    for (; at + U * STEP <= w.end; at += U * STEP, ++tile) {
      u32x4n raw[U];
      float f[U * V];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = nxt[u];
      p += U * NT;
      if (at + 2 * U * STEP <= w.end) {
#pragma unroll
        for (int u = 0; u < U; ++u) nxt[u] = load(p + u * NT);
      }
      // left to itself the scheduler moves loads to where they are used in some of the
      // variants (8192 x 50001 bf16 with one alternative 143 us without this, 140 with)
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < U; ++u) vec_to_f32<DT>(raw[u], f + u * V);
      const float top = fold<U * V, ENT>(f, c1, m, s, a);
      if (TOP) {
        run = fmaxf(run, top);
        if (((tile + 1) & ((1 << shift) - 1)) == 0) {
          slot[tile >> shift][threadIdx.x] = run;
          run = -INFINITY;
        }
      }
    }
  };
  if (stream) tiles([](const AS1 u32x4u* p) -> u32x4n { return __builtin_nontemporal_load(p); });
  else tiles([](const AS1 u32x4u* p) -> u32x4n { return *p; });
  // what is left, fewer than U accesses a thread, and what lies before the first line
  const bool first = threadIdx.x == NT - 1 && w.head > w.begin;
  float before[V];
  if (first) fetch<DT>(x, w.begin, w.head, w.n, before);
  if (at < w.end) {
    float f[U * V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      fetch<DT>(x, at + threadIdx.x * V + u * STEP, w.end, w.n, f + u * V);
    run = fmaxf(run, fold_any<U * V, ENT>(f, c1, m, s, a));
  }
  if (TOP) slot[tile >> shift][threadIdx.x] = run;
  if (first) fold_any<V, ENT>(before, c1, m, s, a);
}

// (m, s, a) joined over the workgroup.  Maxima pass over NaN, so that a row of only
// NaN and -inf has the maximum of a masked one: its sum is NaN, and makes the row's
// M, and by it all that follows, NaN.
template <int NT, bool ENT>
__device__ __forceinline__ void join(float c1, float* red, float& m, float& s, float& a) {
  const float M = Group<NT>::max(m, red);
  const float back = fmaxf((m - (M == -INFINITY ? 0.f : M)) * c1, LOWEST);
  const float scale = __builtin_amdgcn_exp2f(back);
  if (ENT) a = Group<NT>::sum(scale * fmaf(back, s, a), red);
  s = Group<NT>::sum(s * scale, red);
  m = s == s ? M : NAN;
}

// How many of count keys are larger than v, eight reads of LDS in flight (us one by one,
// each waited for | so: 32768 x 8000 bf16 with 128 alternatives 408 | 328, 65536 x 512
// 588 | 472).  The list goes on with zeros up to a multiple of eight.
constexpr int RANK_STEP = 8;
__device__ __forceinline__ int larger_than(const uint64_t* list, int count, uint64_t v) {
  int n = 0;
  for (int j = 0; j < count; j += RANK_STEP) {
    uint64_t o[RANK_STEP];
#pragma unroll
    for (int e = 0; e < RANK_STEP; ++e) o[e] = list[j + e];
#pragma unroll
    for (int e = 0; e < RANK_STEP; ++e) n += o[e] > v;
  }
  return n;
}
// those zeros; N, the list's size, is a multiple of eight
template <int N>
__device__ __forceinline__ void pad_list(uint64_t (&list)[N], int count) {
  static_assert(N % RANK_STEP == 0, "");
  if ((int)threadIdx.x < (-count & (RANK_STEP - 1))) list[count + threadIdx.x] = 0;
}

template <int NT> struct TopShared {
  static constexpr int CAND = 4 * NT < RANK_STEP ? RANK_STEP : 4 * NT;
  alignas(16) uint64_t cand[CAND];
  static constexpr int LIST = 2 * NT;   // slots to be read again
  union {
    float slot[SLOTS][NT];
    alignas(16) uint64_t kept[CAND];
  };
  uint32_t key[NT];
  union {
    unsigned short list[LIST];
    int ties[NT];
  };
  int hist[256];
  int n, entries, bound;
  int kept_n;                    // of `kept`: apart from n, which waves may still be reading
};

// The largest bound that at least k of a wave's N keys a lane reach, bit by bit
// from the top; 0 where there are fewer.  Keys equal above bit LOW are equal.
template <int N, int LOW>
__device__ __forceinline__ uint32_t kth_of_wave(const uint32_t* own, int k) {
  uint32_t bound = 0;
  for (int bit = 31; bit >= LOW; --bit) {
    const uint32_t next = bound | 1u << bit;
    int count = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) count += __popcll(__ballot(own[j] >= next));
    if (count >= k) bound = next;
  }
  return bound;
}

// The k largest (value, lower index) of a chunk of a row as full keys, largest
// first, handed to out(rank, key); fewer than k elements give fewer.  m, s: the
// calling thread's running maximum and sum; sh.slot: its tiles' maxima, 2^shift
// tiles a slot.
//
// The k-th largest of the threads' maxima bounds the k-th largest element from
// below, and whatever reaches it lies in a slot whose maximum does: about k
// slots of all the 8 NT are read again.  (Every element is a candidate where
// fewer than k threads have any: at most k V of them.)
template <int DT, int NT, class Out>
__device__ __forceinline__ void top_of_chunk(const AS1 typename DTypeTraits<DT>::raw_t* x,
                                             const Walk<DT> w, float m, float s, int k, int shift,
                                             TopShared<NT>& sh, Out out) {
  constexpr int V = row_vec<DT>(), STEP = NT * V;
  // low bits of a key that say nothing: bf16 fills 16 bits of an fp32, fp16 19
  constexpr int LOW = DT == KDT_F32 ? 0 : DT == KDT_BF16 ? 16 : 8;
  const int tid = threadIdx.x, mine = w.head + tid * V;
  const int per = (w.end - w.head + STEP - 1) / STEP;        // accesses a thread at most
  const bool first = tid == NT - 1 && w.head > w.begin;      // has the elements before the lines
  // visit(f, i, e1): elements i .. e1 - 1 of this thread, access by access
  auto each = [&](int j0, int j1, auto visit) {
    for (int j = j0; j < j1 && mine + j * STEP < w.end; ++j) {
      float f[V];
      const int i = mine + j * STEP;
      fetch<DT>(x, i, w.end, w.n, f);
      visit(f, i, w.end);
    }
  };
  auto before = [&](auto visit) {
    if (first) {
      float f[V];
      fetch<DT>(x, w.begin, w.head, w.n, f);
      visit(f, w.begin, w.head);
    }
  };
  // this thread's largest key; a NaN or +inf made s NaN, the maximum passes over NaN
  uint32_t key = mine < w.end || first ? order_key(m) : 0u;
  if (s != s) {
    key = 0;
    auto most = [&](const float* f, int i, int e1) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t o = i + e < e1 ? order_key(f[e]) : 0u;
        key = o > key ? o : key;
      }
    };
    each(0, per, most);
    before(most);
  }
  sh.key[tid] = key;
  if (tid == 0) sh.n = sh.entries = sh.kept_n = 0;
  __syncthreads();
  if (tid < 64) {
    uint32_t own[NT / 64];
#pragma unroll
    for (int j = 0; j < NT / 64; ++j) own[j] = sh.key[tid + 64 * j];
    const uint32_t bound = kth_of_wave<NT / 64, LOW>(own, k);
    if (tid == 0) sh.bound = (int)bound;
  }
  __syncthreads();
  const uint32_t bound = (uint32_t)sh.bound ? (uint32_t)sh.bound : 1u;
  auto take = [&](const float* f, int i, int e1) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (i + e < e1 && order_key(f[e]) >= bound) {
        const int c = atomicAdd(&sh.n, 1);
        if (c < TopShared<NT>::CAND) sh.cand[c] = full_key(f[e], (uint32_t)(i + e));
      }
  };
  const int lines = (V == 4 ? 2 : 1) + shift;      // log2 of a slot's accesses
  if (key >= bound) {
    for (int q = 0; q < SLOTS && q << lines < per; ++q)
      if (s != s || order_key(sh.slot[q][tid]) >= bound) {
        const int c = atomicAdd(&sh.entries, 1);
        if (c < TopShared<NT>::LIST) sh.list[c] = (unsigned short)(q * NT + tid);
      }
    before(take);
  }
  __syncthreads();
  // the slots' accesses shared out over the workgroup: one round trip, as a rule
  const int entries = sh.entries;
  if (entries <= TopShared<NT>::LIST) {
    for (int it = tid; it < entries << lines; it += NT) {
      const int at = sh.list[it >> lines], q = at / NT;
      const int i = w.head + (at % NT) * V + ((q << lines) + (it & ((1 << lines) - 1))) * STEP;
      if (i < w.end) {
        float f[V];
        fetch<DT>(x, i, w.end, w.n, f);
        take(f, i, w.end);
      }
    }
  }
  __syncthreads();
  if (sh.n > TopShared<NT>::CAND || entries > TopShared<NT>::LIST) {
    // Too many equal or crowded values: the k-th largest key exactly, by counting
    // its digits from the top; then the larger ones and, in the order of their
    // indices, as many equal ones as are wanted -- k in all.
    int need = k;
    uint32_t prefix = 0;
    for (int shift_d = 24; shift_d >= LOW; shift_d -= 8) {
      for (int j = tid; j < 256; j += NT) sh.hist[j] = 0;
      __syncthreads();
      auto count = [&](const float* f, int i, int e1) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint32_t o = order_key(f[e]);
          if (i + e < e1 && (uint64_t)o >> (shift_d + 8) == prefix)
            atomicAdd(&sh.hist[(o >> shift_d) & 255], 1);
        }
      };
      each(0, per, count);
      before(count);
      __syncthreads();
      int digit = 255, left = need;
      while (digit > 0 && sh.hist[digit] < left) left -= sh.hist[digit--];
      need = left;
      prefix = prefix << 8 | (uint32_t)digit;
      __syncthreads();
    }
    const uint32_t low = LOW ? (1u << LOW) - 1u : 0u, kth = prefix << LOW;   // of the digits counted
    if (tid == 0) sh.n = 0;
    __syncthreads();
    auto larger = [&](const float* f, int i, int e1) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i + e < e1 && order_key(f[e]) > (kth | low))
          sh.cand[atomicAdd(&sh.n, 1)] = full_key(f[e], (uint32_t)(i + e));
    };
    each(0, per, larger);
    before(larger);
    __syncthreads();
    // equal ones in the order of their indices: V a thread from the chunk's begin on
    int have = sh.n;                       // k - need
    for (int at = w.begin; at < w.end && have < k; at += STEP) {
      float f[V];
      const int i = at + tid * V;
      int mine_n = 0;
      if (i < w.end) {
        fetch<DT>(x, i, w.end, w.n, f);
#pragma unroll
        for (int e = 0; e < V; ++e)
          mine_n += i + e < w.end && (order_key(f[e]) | low) == (kth | low);
      }
      __syncthreads();
      sh.ties[tid] = mine_n;
      __syncthreads();
      int rank = have, all = have;
      for (int j = 0; j < NT; ++j) {
        rank += j < tid ? sh.ties[j] : 0;
        all += sh.ties[j];
      }
      if (mine_n) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (i + e < w.end && (order_key(f[e]) | low) == (kth | low)) {
            if (rank < k) sh.cand[rank] = full_key(f[e], (uint32_t)(i + e));
            ++rank;
          }
      }
      have = all;
    }
    __syncthreads();
    if (tid == 0) sh.n = k;
    __syncthreads();
  }
  // Their order by counting, for each, the larger ones: quadratic, so that of many
  // those below the k-th are dropped first.  us never | beyond 400 | always, bf16 with
  // 128: 65536 x 512 1320 | 476 | 477, 32768 x 1000 2064 | 246 | 243, x 2000 258 | 223 | 255,
  // x 8000 352 | 285 | 319, 8192 x 32064 159 | 149 | 155, 16384 x 1000 fp32 126 | 113 | 159,
  // 700 x 10000 fp32 17 | 17 | 23; with 64: 32768 x 1000 175 | 147 | 195, x 2000 181 | 151 |
  // 157.  (Of 21 sizes one, 65536 x 512 with 64, would want fewer than 400: 577 | 551 | 395.)
  int count = sh.n;
  const uint64_t* cand = sh.cand;
  if (count > 400) {
    if (tid < 64) {
      uint32_t own[TopShared<NT>::CAND / 64];
#pragma unroll
      for (int j = 0; j < TopShared<NT>::CAND / 64; ++j)
        own[j] = tid + 64 * j < count ? (uint32_t)(sh.cand[tid + 64 * j] >> 32) : 0u;
      const uint32_t kth = kth_of_wave<TopShared<NT>::CAND / 64, LOW>(own, k);
      if (tid == 0) sh.bound = (int)kth;
    }
    __syncthreads();
    const uint32_t kth = (uint32_t)sh.bound;
    for (int c = tid; c < count; c += NT)
      if ((uint32_t)(sh.cand[c] >> 32) >= kth) sh.kept[atomicAdd(&sh.kept_n, 1)] = sh.cand[c];
    __syncthreads();
    count = sh.kept_n;
    cand = sh.kept;
    pad_list(sh.kept, count);
  } else {
    pad_list(sh.cand, count);
  }
  __syncthreads();
  for (int c = tid; c < count; c += NT) {
    const uint64_t v = cand[c];
    const int rank = larger_than(cand, count, v);
    if (rank < k) out(rank, v);
  }
}

__device__ __forceinline__ float any_value(const void* t, long long i, int dt) {
  if (dt == KDT_F32) return ((const float*)t)[i];
  const uint16_t v = ((const uint16_t*)t)[i];
  return dt == KDT_BF16 ? bf16_bits_to_f32(v) : f16_bits_to_f32(v);
}

struct SlotShared {
  alignas(16) int id[TOP_MAX];
  alignas(16) float q[TOP_MAX];
};

// The teacher's side of a row, and the loss, from the student's (M, L).
template <int DT, int NT>
__device__ __forceinline__ void distill_row(const Fwd& a, long long row, float M, float L,
                                            SlotShared& sh, float* red) {
  const AS1 typename DTypeTraits<DT>::raw_t* x =
      gptr((const typename DTypeTraits<DT>::raw_t*)a.x) + row * a.ld;
  constexpr int P = (TOP_MAX + NT - 1) / NT;       // slots a thread
  int id[P];
  float t[P], top = -INFINITY;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int j = threadIdx.x + p * NT;
    const long long v = j < a.K ? a.ids[row * a.K + j] : -1;
    t[p] = v == -1 ? -INFINITY : any_value(a.teacher, row * a.K + j, a.tdt);
    if (v < -1 || v >= a.V) t[p] = NAN;            // makes the row's sum NaN
    id[p] = v < 0 || v >= a.V ? -1 : (int)v;
    top = fmaxf(top, t[p]);
  }
  top = Group<NT>::max(top, red);
  if (top == -INFINITY) top = 0.f;                 // only -inf and NaN
  float z = 0.f;
#pragma unroll
  for (int p = 0; p < P; ++p) z += __builtin_amdgcn_exp2f((t[p] - top) * a.inv_t * LOG2E);
  z = Group<NT>::sum(z, red);
  const float logz = logf(z);
  float term = 0.f, q[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const float d = (t[p] - top) * a.inv_t;
    q[p] = __builtin_amdgcn_exp2f(d * LOG2E) / z;
    const int j = threadIdx.x + p * NT;
    if (j < a.K && q[p] != 0.f) {
      // q (log q - lp) with q taken into lp's product first: of a token masked by the
      // type's lowest value (x - M) / T is past fp32's range, and q may be nothing
      const float c = id[p] < 0 ? NAN : M == -INFINITY ? -INFINITY
                                      : DTypeTraits<DT>::to_f32(x[id[p]]) - M;
      term += q[p] * (d - logz + (M == -INFINITY ? 0.f : L)) - q[p] * c * a.inv_t;
    }
    if (j < TOP_MAX) {
      sh.id[j] = id[p];
      sh.q[j] = q[p];
    }
  }
  term = Group<NT>::sum(term, red);
  if (threadIdx.x == 0) {
    a.loss[row] = term;
    if (a.stats) {
      a.stats[2 * row] = M;
      a.stats[2 * row + 1] = z == z ? L : NAN;     // NaN all along the gradient's row
    }
  }
  if (!a.keep_ids) return;
  __syncthreads();
  // the same id twice: its masses are added in slot order, into its first slot
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int j = threadIdx.x + p * NT;
    if (j >= a.K) break;
    float mass = 0.f;
    bool first = true;
    for (int o = 0; o < a.K; o += RANK_STEP) {     // behind the K slots stand unused ones
      int at[RANK_STEP];
      float m[RANK_STEP];
#pragma unroll
      for (int e = 0; e < RANK_STEP; ++e) {
        at[e] = sh.id[o + e];
        m[e] = sh.q[o + e];
      }
#pragma unroll
      for (int e = 0; e < RANK_STEP; ++e) {
        if (at[e] == id[p] && o + e < j) first = false;
        mass += at[e] == id[p] ? m[e] : 0.f;
      }
    }
    a.keep_ids[row * a.K + j] = first ? id[p] : -1;
    a.keep_q[row * a.K + j] = mass;
  }
}

// whether a row of slots has any mass
template <int NT>
__device__ __forceinline__ bool has_teacher(const Fwd& a, long long row, float* red) {
  float any = 0.f;
  for (int j = threadIdx.x; j < a.K; j += NT)
    if (a.ids[row * a.K + j] != -1) {
      const long long v = a.ids[row * a.K + j];
      const float t = any_value(a.teacher, row * a.K + j, a.tdt);
      if (t != -INFINITY || v < -1 || v >= a.V) any = 1.f;
    }
  return Group<NT>::max(any, red) > 0.f;
}

template <int DT, int NT>
__device__ __forceinline__ void logprob_row(const Fwd& a, long long row, float M, float s,
                                            float sum, float& L) {
  L = logf(s);
  if (threadIdx.x != 0) return;
  const AS1 typename DTypeTraits<DT>::raw_t* x =
      gptr((const typename DTypeTraits<DT>::raw_t*)a.x) + row * a.ld;
  if (a.logprob) {
    const long long t = a.targets[row];
    a.logprob[row] =
        t < 0 || t >= a.V ? NAN : log_prob(DTypeTraits<DT>::to_f32(x[t]), M, L, a.inv_t);
  }
  if (a.entropy) a.entropy[row] = M == -INFINITY ? 0.f : L - sum / s * LN2;
  if (a.stats) {
    a.stats[2 * row] = M;
    a.stats[2 * row + 1] = L;
  }
}

// One workgroup a chunk of a row.  4096 x 131072 bf16 169 us (6.4 TB/s), 1792 of 2048 x
// 32064 fp32 with entropy, in a training step, 48 us (4.7 TB/s), 8192 x 50001 bf16 with
// entropy and 32 alternatives 186 us (4.4 TB/s; 143 us without either), 700 x 10000 fp32
// with 5 of them 12.7 us; one row of 131072 7.4 us, where the round trips to memory count.
// (Six waves a SIMD also where both entropy and alternatives want registers: us without
// | with this, 8192 x 50001 bf16 with 32 of them 176 | 171, 4096 x 131072 with 20 203 | 202.
// Elsewhere it gains nothing: 8192 x 50001 130 | 136, with entropy 137 | 140.)
template <int DT, int NT, int MODE, bool ENT, bool TOP>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(NT == 256 && ENT && TOP ? 6 : 1)))
void vocab_fwd_kernel(const Fwd a, int splits, int chunk) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  __shared__ float red[NT / 64];
  __shared__ TopShared<TOP ? NT : 1> tops;        // without TOP a few bytes that nobody reads
  const long long row = blockIdx.x / splits;
  const int part = blockIdx.x % splits, n = (int)a.V;
  const int begin = part * chunk, end = n - begin < chunk ? n : begin + chunk;
  const AS1 raw_t* x = gptr((const raw_t*)a.x) + row * a.ld;
  const bool skip = MODE == DISTILL ? !has_teacher<NT>(a, row, red)
                                    : a.targets && a.targets[row] == a.ignore;
  if (skip) {
    if (part != 0) return;
    if (TOP)
      for (int j = threadIdx.x; j < a.k; j += NT) {
        a.top_lp[row * a.k + j] = -INFINITY;
        a.top_ids[row * a.k + j] = -1;
      }
    if (threadIdx.x == 0) {
      if (a.loss) a.loss[row] = 0.f;
      if (a.logprob) a.logprob[row] = 0.f;
      if (a.entropy) a.entropy[row] = 0.f;
      if (a.stats) {
        a.stats[2 * row] = -INFINITY;
        a.stats[2 * row + 1] = 0.f;
      }
    }
    return;
  }
  const float c1 = a.inv_t * LOG2E;
  const Walk<DT> w(x, begin, end, n);
  // tiles a slot: the least power of two that leaves no more than SLOTS of them
  const int tiles = (end - w.head) / (NT * 16) + 1;
  const int shift = tiles <= SLOTS ? 0 : 32 - __clz((tiles - 1) / SLOTS);
  float m, s, sum;
  scan<DT, NT, ENT, TOP>(x, w, a.stream, c1, shift, (float(*)[NT])tops.slot, m, s, sum);
  float M = m, S = s;
  join<NT, ENT>(c1, red, M, S, sum);
  if (splits > 1) {
    Part* p = (Part*)a.ws + row * splits + part;
    if (threadIdx.x == 0) *p = Part{M, S, sum, 0.f};
    if constexpr (TOP) {
      uint64_t* keys = (uint64_t*)((Part*)a.ws + a.rows * splits) + (row * splits + part) * a.k;
      for (int j = threadIdx.x; j < a.k; j += NT)
        if (j >= end - begin) keys[j] = 0;         // fewer elements than k
      top_of_chunk<DT, NT>(x, w, m, s, a.k, shift, tops,
                           [&](int rank, uint64_t key) { keys[rank] = key; });
    }
    return;
  }
  if constexpr (MODE == DISTILL) {
    __shared__ SlotShared slots;
    distill_row<DT, NT>(a, row, M, logf(S), slots, red);
  } else {
    float L;
    logprob_row<DT, NT>(a, row, M, S, sum, L);
    if constexpr (TOP) {
      top_of_chunk<DT, NT>(x, w, m, s, a.k, shift, tops, [&](int rank, uint64_t key) {
        a.top_ids[row * a.k + rank] = (uint32_t)~(uint32_t)key;
        a.top_lp[row * a.k + rank] = log_prob(key_value((uint32_t)(key >> 32)), M, L, a.inv_t);
      });
    }
  }
}

// Joins the parts of a row (one of 131072 in 32 parts, 20 alternatives: 5.0 us, the
// launch and four dependent loads).  The alternatives: every part has its own k largest
// in order; with j of a part's keys at least as large as the r-th largest of
// all parts' j-th keys, r j >= k, that key is a bound which at least k keys
// reach and no more than r k + splits j.
constexpr int JOIN_NT = 256;
constexpr int JOIN_CAND = 2560;

__host__ __device__ constexpr int join_depth(int k, int splits) {
  const int j = (4 * k + splits - 1) / splits;
  return j < k ? j : k;
}

template <int DT, int MODE, bool ENT, bool TOP>
__global__ __launch_bounds__(JOIN_NT) void vocab_join_kernel(const Fwd a, int splits) {
  constexpr int NT = JOIN_NT;
  __shared__ float red[NT / 64];
  const long long row = blockIdx.x;
  const bool skip = MODE == DISTILL ? !has_teacher<NT>(a, row, red)
                                    : a.targets && a.targets[row] == a.ignore;
  if (skip) return;                                // the first kernel wrote the row
  const Part* p = (const Part*)a.ws + row * splits;
  float m = -INFINITY, s = 0.f, sum = 0.f;
  if (threadIdx.x < splits) {
    const Part v = p[threadIdx.x];
    m = v.m;
    s = v.s;
    sum = v.a;
  }
  join<NT, true>(a.inv_t * LOG2E, red, m, s, sum);
  if constexpr (MODE == DISTILL) {
    __shared__ SlotShared slots;
    distill_row<DT, NT>(a, row, m, logf(s), slots, red);
  } else {
    float L;
    logprob_row<DT, NT>(a, row, m, s, sum, L);
    if constexpr (TOP) {
      __shared__ alignas(16) uint64_t cand[JOIN_CAND], head[MAX_SPLITS];
      __shared__ uint64_t bound_s;
      __shared__ int count;
      const uint64_t* keys =
          (const uint64_t*)((const Part*)a.ws + a.rows * splits) + row * splits * a.k;
      const int depth = join_depth(a.k, splits), r = (a.k + depth - 1) / depth;
      const uint64_t mine = threadIdx.x < splits ? keys[threadIdx.x * a.k + depth - 1] : 0;
      if (threadIdx.x < MAX_SPLITS) head[threadIdx.x] = mine;
      if (threadIdx.x == 0) {
        count = 0;
        bound_s = 1;
      }
      __syncthreads();
      if (threadIdx.x < splits && mine) {
        if (larger_than(head, splits, mine) == r - 1) bound_s = mine;        // keys are unique: one thread
      }
      __syncthreads();
      const uint64_t bound = bound_s;
      // loads in flight (us with one | eight: 16 x 200000 bf16 with 128 alternatives 26 | 20,
      // one row of 131072 with 20 5.7 | 5.1)
      constexpr int U = 8;
      for (int i = threadIdx.x; i < splits * a.k; i += U * NT) {
        uint64_t key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) key[u] = i + u * NT < splits * a.k ? keys[i + u * NT] : 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (key[u] >= bound) {
            const int c = atomicAdd(&count, 1);
            if (c < JOIN_CAND) cand[c] = key[u];
          }
      }
      __syncthreads();
      const int n = count < JOIN_CAND ? count : JOIN_CAND;
      pad_list(cand, n);
      __syncthreads();
      for (int c = threadIdx.x; c < n; c += NT) {
        const uint64_t v = cand[c];
        const int rank = larger_than(cand, n, v);
        if (rank < a.k) {
          a.top_ids[row * a.k + rank] = (uint32_t)~(uint32_t)v;
          a.top_lp[row * a.k + rank] = log_prob(key_value((uint32_t)(v >> 32)), m, L, a.inv_t);
        }
      }
    }
  }
}

// One workgroup writes one tile of four 16-byte accesses a thread, then corrects
// the few elements that carry the target's or the teacher's mass.  A read and a
// write of every element: 4096 x 131072 bf16 375 us (5.7 TB/s; one access a thread
// in a bare copy reaches 6.2), 2048 x 32064 fp32, 1792 of them read, 88 us (5.6 TB/s).
constexpr int BWD_NT = 256;

template <int DT> constexpr int bwd_chunk() { return BWD_NT * row_vec<DT>() * 4; }

template <int DT, int MODE, bool ENT>
__global__ __launch_bounds__(BWD_NT) void vocab_bwd_kernel(const Bwd a, int splits) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  constexpr int V = row_vec<DT>(), U = 4, STEP = BWD_NT * V, CHUNK = bwd_chunk<DT>();
  const long long row = blockIdx.x / splits;
  const int n = (int)a.V, part = blockIdx.x % splits;
  const AS1 raw_t* x = gptr((const raw_t*)a.x) + row * a.ld;
  AS1 raw_t* dx = gptr((raw_t*)a.dx) + row * a.V;
  // whole 16-byte lines of dx; the first workgroup has what lies before them, too
  const int past = (int)(((uintptr_t)dx & 15) / (16 / V));
  const int head = past && V - past < n ? V - past : past ? n : 0;
  const int from = head + part * CHUNK, begin = part ? from : 0;
  const int end = n - from < CHUNK ? n : from + CHUNK;
  const float M = a.stats[2 * row], L = a.stats[2 * row + 1];
  const long long tgt = MODE == LOGPROB && a.targets ? a.targets[row] : 0;
  const bool zero = M == -INFINITY || (MODE == LOGPROB && a.targets && tgt == a.ignore);
  float g = a.g ? a.g[row * a.gs] : 0.f;
  if (MODE == LOGPROB && a.g && (tgt < 0 || tgt >= n)) g = NAN;
  const float gh = ENT ? a.gh[row * a.ghs] : 0.f, H = ENT ? a.entropy[row] : 0.f;
  const float sign = MODE == LOGPROB ? -a.inv_t : a.inv_t;
  const float gs = g * sign, ghs = gh * sign;
  // p_i (g + gh (lp_i + H)), the correction's mass apart
  auto value = [&](float xi) {
    const float lp = (xi - M) * a.inv_t - L, p = __builtin_amdgcn_exp2f(lp * LOG2E);
    return ENT ? p * fmaf(ghs, fmaxf(lp, LOWEST) + H, gs) : p * gs;
  };
  if (part == 0 && threadIdx.x < head)
    dx[threadIdx.x] = DTypeTraits<DT>::from_f32(
        zero ? 0.f : value(DTypeTraits<DT>::to_f32(x[threadIdx.x])));
  for (int at = from; at < end; at += U * STEP) {
    const int i = at + threadIdx.x * V;
    float f[U * V];
    if (zero) {
#pragma unroll
      for (int e = 0; e < U * V; ++e) f[e] = 0.f;
    } else if (at + U * STEP <= end) {
      u32x4n raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = *(const AS1 u32x4u*)(x + i + u * STEP);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < U; ++u) vec_to_f32<DT>(raw[u], f + u * V);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) fetch<DT>(x, i + u * STEP, end, n, f + u * V);
    }
    if (!zero) {
#pragma unroll
      for (int e = 0; e < U * V; ++e) f[e] = value(f[e]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) store_vec<DT, true>(dx, i + u * STEP, end, f + u * V);
  }
  if (zero || (MODE == LOGPROB && !a.g)) return;
  __syncthreads();                       // the workgroup's stores come first
  if (MODE == LOGPROB) {
    if (threadIdx.x == 0 && tgt >= begin && tgt < end)
      dx[tgt] = DTypeTraits<DT>::from_f32(value(DTypeTraits<DT>::to_f32(x[tgt])) - gs);
  } else {
    for (int j = threadIdx.x; j < a.K; j += BWD_NT) {
      const int id = a.keep_ids[row * a.K + j];
      if (id >= begin && id < end)
        dx[id] = DTypeTraits<DT>::from_f32(
            gs * (__builtin_amdgcn_exp2f(((DTypeTraits<DT>::to_f32(x[id]) - M) * a.inv_t - L) * LOG2E) -
                  a.keep_q[row * a.K + j]));
    }
  }
}

// Threads a workgroup.  A row of at most 8 accesses a lane is a wave's; with
// enough rows to fill the chip by waves, one of 32 is, too, and saves the
// workgroup's barriers (us with 64 | 256: 65536 x 512 bf16 33 | 116, 32768 x 2000 30 | 66,
// 32768 x 8000 84 | 102, with entropy 88 | 125, with 32 alternatives 150 | 194; 16384 x
// 16000 with entropy 88 | 94; but 700 x 16000 8.8 | 7.9).  Half of a wave's lanes have
// to be more than the alternatives.
int fwd_threads(int dt, long long rows, long long V, int k) {
  const int vec = dt == KDT_F32 ? 4 : 8;
  return k <= 32 && V <= 64 * vec * (rows >= 4096 ? 32 : 8) ? 64 : 256;
}

// Workgroups a row: enough to have four for every CU, but none with less than
// two 16-byte accesses a thread.
int fwd_splits(int dt, long long rows, long long V, int k) {
  if (fwd_threads(dt, rows, V, k) == 64) return 1;
  const long long least = 256LL * (dt == KDT_F32 ? 4 : 8) * 2, most = (V + least - 1) / least;
  long long n = (1024 + rows - 1) / rows;
  if (n > most) n = most;
  if (n > MAX_SPLITS) n = MAX_SPLITS;
  return n < 1 || rows >= 512 ? 1 : (int)n;
}

bool dtype_ok(int dt) { return dt == KDT_F32 || dt == KDT_BF16 || dt == KDT_F16; }

template <class T> T* at(T* p, long long n) { return p ? p + n : p; }
const void* at(const void* p, long long n, int dt) {
  return at((const char*)p, n * (dt == KDT_F32 ? 4 : 2));
}

// rows r0 .. r0 + rows - 1 of a
Fwd some_rows(Fwd a, long long r0, long long rows) {
  a.x = at(a.x, r0 * a.ld, a.dt);
  a.targets = at(a.targets, r0);
  a.logprob = at(a.logprob, r0);
  a.entropy = at(a.entropy, r0);
  a.top_lp = at(a.top_lp, r0 * a.k);
  a.top_ids = at(a.top_ids, r0 * a.k);
  a.stats = at(a.stats, 2 * r0);
  a.ids = at(a.ids, r0 * a.K);
  a.teacher = at(a.teacher, r0 * a.K, a.tdt);
  a.loss = at(a.loss, r0);
  a.keep_ids = at(a.keep_ids, r0 * a.K);
  a.keep_q = at(a.keep_q, r0 * a.K);
  a.rows = rows;
  return a;
}
Bwd some_rows(Bwd a, long long r0, long long rows) {
  a.x = at(a.x, r0 * a.ld, a.dt);
  a.stats = at(a.stats, 2 * r0);
  a.entropy = at(a.entropy, r0);
  a.targets = at(a.targets, r0);
  a.g = at(a.g, r0 * a.gs);
  a.gh = at(a.gh, r0 * a.ghs);
  a.keep_ids = at(a.keep_ids, r0 * a.K);
  a.keep_q = at(a.keep_q, r0 * a.K);
  a.dx = (void*)at(a.dx, r0 * a.V, a.dt);
  a.rows = rows;
  return a;
}

// one launch for each range of rows that has at most MAX_GROUPS workgroups
template <class Args, class Launch> void each_range(const Args& a, int splits, Launch launch) {
  const long long most = MAX_GROUPS / splits;
  for (long long r0 = 0; r0 < a.rows; r0 += most)
    launch(some_rows(a, r0, a.rows - r0 < most ? a.rows - r0 : most));
}

template <int DT, int MODE, bool ENT, bool TOP>
void launch_fwd(const Fwd& a, hipStream_t st) {
  const int splits = fwd_splits(a.dt, a.rows, a.V, a.k);
  if (splits == 1 && fwd_threads(a.dt, a.rows, a.V, a.k) == 64) {
    each_range(a, 1, [&](const Fwd& r) {
      hipLaunchKernelGGL((vocab_fwd_kernel<DT, 64, MODE, ENT, TOP>), dim3((unsigned)r.rows),
                         dim3(64), 0, st, r, 1, (int)r.V);
    });
    return;
  }
  const int vec = row_vec<DT>();
  const int chunk = (int)((a.V + splits - 1) / splits + vec - 1) / vec * vec;
  each_range(a, splits, [&](const Fwd& r) {
    hipLaunchKernelGGL((vocab_fwd_kernel<DT, 256, MODE, ENT, TOP>),
                       dim3((unsigned)(r.rows * splits)), dim3(256), 0, st, r, splits, chunk);
  });
  if (splits > 1)                          // few rows: one range
    hipLaunchKernelGGL((vocab_join_kernel<DT, MODE, ENT, TOP>), dim3((unsigned)a.rows),
                       dim3(JOIN_NT), 0, st, a, splits);
}

template <int DT> void launch_fwd_any(const Fwd& a, hipStream_t st) {
  if (a.loss) launch_fwd<DT, DISTILL, false, false>(a, st);
  else if (a.k && a.entropy) launch_fwd<DT, LOGPROB, true, true>(a, st);
  else if (a.k) launch_fwd<DT, LOGPROB, false, true>(a, st);
  else if (a.entropy) launch_fwd<DT, LOGPROB, true, false>(a, st);
  else launch_fwd<DT, LOGPROB, false, false>(a, st);
}

template <int DT> void launch_bwd(const Bwd& a, hipStream_t st) {
  const int splits = (int)((a.V + bwd_chunk<DT>() - 1) / bwd_chunk<DT>());
  each_range(a, splits, [&](const Bwd& r) {
    const dim3 grid((unsigned)(r.rows * splits)), block(BWD_NT);
    if (r.keep_ids)
      hipLaunchKernelGGL((vocab_bwd_kernel<DT, DISTILL, false>), grid, block, 0, st, r, splits);
    else if (r.gh)
      hipLaunchKernelGGL((vocab_bwd_kernel<DT, LOGPROB, true>), grid, block, 0, st, r, splits);
    else
      hipLaunchKernelGGL((vocab_bwd_kernel<DT, LOGPROB, false>), grid, block, 0, st, r, splits);
  });
}

}  // namespace

KFAC_API int kfac_vocab_top_max() { return TOP_MAX; }

// bytes of the workspace of one forward call (0: none)
KFAC_API long long kfac_vocab_ws_bytes(int dt, long long rows, long long V, int k) {
  const int splits = fwd_splits(dt, rows, V, k);
  return splits == 1 ? 0 : rows * splits * (long long)(sizeof(Part) + 8LL * k);
}

KFAC_API int kfac_vocab_forward(const KfacVocabFwd* args, hipStream_t stream) {
  Fwd a = *args;
  if (!a.x || a.rows <= 0 || a.V <= 0 || a.V > MAX_V || a.rows > 0x7fffffffLL / MAX_SPLITS ||
      !(a.inv_t > 0.f) || !dtype_ok(a.dt))
    return -2;
  if (a.loss ? !a.ids || !a.teacher || !a.keep_ids != !a.keep_q || !a.keep_ids != !a.stats ||
                   !dtype_ok(a.tdt) || a.K < 1 || a.K > TOP_MAX || a.k
             : a.k < 0 || a.k > TOP_MAX || a.k > a.V || (a.logprob && !a.targets) ||
                   (a.k && (!a.top_lp || !a.top_ids)))
    return -2;
  if (!a.ws && kfac_vocab_ws_bytes(a.dt, a.rows, a.V, a.k)) return -2;
  a.stream = a.rows * a.V * (a.dt == KDT_F32 ? 4 : 2) > STREAM_FROM;
  if (a.dt == KDT_F32) launch_fwd_any<KDT_F32>(a, stream);
  else if (a.dt == KDT_BF16) launch_fwd_any<KDT_BF16>(a, stream);
  else launch_fwd_any<KDT_F16>(a, stream);
  return (int)hipGetLastError();
}

KFAC_API int kfac_vocab_backward(const KfacVocabBwd* args, hipStream_t stream) {
  const Bwd a = *args;
  if (!a.x || !a.dx || !a.stats || a.rows <= 0 || a.V <= 0 || a.V > MAX_V ||
      a.rows > 0x7fffffffLL / ((a.V + 4095) / 4096) || !(a.inv_t > 0.f) || !dtype_ok(a.dt))
    return -2;
  if (a.keep_ids ? !a.keep_q || !a.g || a.K < 1 || a.K > TOP_MAX
                 : (!a.g && !a.gh) || (a.g && !a.targets) || (a.gh && !a.entropy))
    return -2;
  if (a.dt == KDT_F32) launch_bwd<KDT_F32>(a, stream);
  else if (a.dt == KDT_BF16) launch_bwd<KDT_BF16>(a, stream);
  else launch_bwd<KDT_F16>(a, stream);
  return (int)hipGetLastError();
}
