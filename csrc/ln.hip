// Layer norm over the last dimension, forward and backward, with the residual
// add in front of it (gfx950): the normalisation layers of the Transformer LM.
//
//   forward    s = x + z (rounded to the stream's type S; s = x without z)
//              mu = mean(s), r = 1 / sqrt(mean((s - mu)^2) + eps)
//              h = (s - mu) r,  y = h w + b
//   backward   g = dy w
//              dx = dz = ds + r (g - mean(g) - h mean(g h))
//              dw = sum_rows dy h,  db = sum_rows dy
//
// Rows are strided (ld), their elements contiguous; statistics, h and every
// sum are held in fp32, the variance about the mean (two passes over the row).
// The sums over rows (dw, db) run over fixed row chunks and then over the
// chunks in order: no atomics, bitwise reproducible.
//
// Times below are medians of a kernel's launches on one MI355X, three sets of inputs
// in turn; of two sides, both with the code as it stands but for the choice.
#include "records.h"
#include "rows.h"

namespace {

typedef KfacLnFwd Fwd;
typedef KfacLnBwd Bwd;

constexpr int NT = 256, LT = 1024;     // threads: columns' sums, long rows
// A launch has fewer than 2^32 threads: workgroups of 1024 stride over what is more
// than this many of them.
constexpr long long MAX_GROUPS = 1 << 16;

__device__ __forceinline__ float ld_any(const void* p, long long i, int dt) {
  if (dt == KDT_F32) return ((const float*)p)[i];
  const uint16_t v = ((const uint16_t*)p)[i];
  return dt == KDT_BF16 ? bf16_bits_to_f32(v) : f16_bits_to_f32(v);
}
__device__ __forceinline__ void st_any(void* p, long long i, int dt, float v) {
  if (dt == KDT_F32) ((float*)p)[i] = v;
  else ((uint16_t*)p)[i] = dt == KDT_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
}

// sum over the workgroup, the same in every thread (waves added in order)
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();                       // red may still be read from the last call
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
  for (int i = 1; i < LT / 64; ++i) r += red[i];
  return r;
}

// A power of two below 1 / D: elements times it have a sum within fp32 wherever they
// are (a row masked by its type's lowest value); what else it changes is the lowest
// bits of terms below 2^-126, far below a variance's square root in fp32.
__device__ __forceinline__ float sum_scale(long long D) {
  return ldexpf(1.f, __clzll(D) - 64);
}

// Rows that no workgroup's registers hold: the workgroup walks the row, once for
// each statistic and once for the result; from the second time on it comes from a
// cache.  1024 x 65536 fp16: 97 us forward (2.8 TB/s of what has to move), 226 us
// backward, 92 of them for the weights' gradients.

// V elements at i, zeros from n on
template <int DT>
__device__ __forceinline__ void walk_load(const AS1 typename DTypeTraits<DT>::raw_t* row,
                                          long long i, long long n, float* f) {
  constexpr int V = row_vec<DT>();
  if (i + V <= n) {
    vec_to_f32<DT>(*(const AS1 u32x4u*)(row + i), f);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = i + e < n ? DTypeTraits<DT>::to_f32(row[i + e]) : 0.f;
  }
}
// V elements at i of a row of any type (uniform over the launch)
template <int V>
__device__ __forceinline__ void walk_any(const void* p, long long off, int dt, long long i,
                                         long long n, float* f) {
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = i + e < n ? ld_any(p, off + i + e, dt) : 0.f;
}
template <int DT>
__device__ __forceinline__ void walk_other(const void* p, long long off, int dt, long long i,
                                           long long n, float* f) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  if (dt == DT) walk_load<DT>(gptr((const raw_t*)p) + off, i, n, f);
  else walk_any<row_vec<DT>()>(p, off, dt, i, n, f);
}
template <int DT>
__device__ __forceinline__ void walk_store(void* p, long long off, int dt, long long i,
                                           long long n, const float* f) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  constexpr int V = row_vec<DT>();
  if (dt == DT && i + V <= n) {
    *(AS1 u32x4u*)(gptr((raw_t*)p) + off + i) = f32_to_vec<DT>(f);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (i + e < n) st_any(p, off + i + e, dt, f[e]);
  }
}

template <int DT>
__global__ __launch_bounds__(LT) void ln_fwd_long_kernel(const Fwd a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  constexpr int V = row_vec<DT>(), STEP = LT * V;
  __shared__ float red[LT / 64];
  const long long D = a.D, t0 = threadIdx.x * V;
  const float scale = sum_scale(D);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const long long yo = row * D;
    const AS1 raw_t* x = gptr((const raw_t*)a.x) + row * a.ldx;
    float acc = 0.f;
    for (long long i = t0; i < D; i += STEP) {
      float f[V];
      walk_load<DT>(x, i, D, f);
      if (a.z) {
        float g[V];
        walk_other<DT>(a.z, row * a.ldz, a.zdt, i, D, g);
#pragma unroll
        for (int e = 0; e < V; ++e)      // the sum as it is stored is what is normed
          f[e] = DTypeTraits<DT>::to_f32(DTypeTraits<DT>::from_f32(f[e] + g[e]));
        walk_store<DT>(a.s, yo, DT, i, D, f);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) acc = fmaf(f[e], scale, acc);
    }
    const AS1 raw_t* s = a.z ? gptr((const raw_t*)a.s) + yo : x;     // each thread's own stores
    const float mu = block_sum(acc, red) / ((float)D * scale);
    acc = 0.f;
    for (long long i = t0; i < D; i += STEP) {
      float f[V];
      walk_load<DT>(s, i, D, f);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = f[e] - mu;
        acc = fmaf(d, i + e < D ? d : 0.f, acc);
      }
    }
    const float rstd = 1.f / sqrtf(block_sum(acc, red) / (float)D + a.eps);
    for (long long i = t0; i < D; i += STEP) {
      float f[V], w[V], b[V];
      walk_load<DT>(s, i, D, f);
      if (a.w) walk_other<DT>(a.w, 0, a.wdt, i, D, w);
      if (a.b) walk_other<DT>(a.b, 0, a.bdt, i, D, b);
#pragma unroll
      for (int e = 0; e < V; ++e)
        f[e] = fmaf((f[e] - mu) * rstd, a.w ? w[e] : 1.f, a.b ? b[e] : 0.f);
      walk_store<DT>(a.y, yo, a.ydt, i, D, f);
    }
    if (threadIdx.x == 0 && a.mean) {
      a.mean[row] = mu;
      a.rstd[row] = rstd;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(LT) void ln_bwd_long_kernel(const Bwd a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  constexpr int V = row_vec<DT>(), STEP = LT * V;
  __shared__ float red[LT / 64];
  const long long D = a.D, t0 = threadIdx.x * V;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const AS1 raw_t* s = gptr((const raw_t*)a.s) + row * a.lds;
    const float mu = a.mean[row], rstd = a.rstd[row];
    float c1 = 0.f, c2 = 0.f;
    for (long long i = t0; i < D; i += STEP) {
      float g[V], h[V], w[V];
      walk_other<DT>(a.dy, row * a.lddy, a.ydt, i, D, g);
      walk_load<DT>(s, i, D, h);
      if (a.w) walk_other<DT>(a.w, 0, a.wdt, i, D, w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float v = a.w ? g[e] * w[e] : g[e];
        c1 += v;
        c2 = fmaf(v, (h[e] - (i + e < D ? mu : 0.f)) * rstd, c2);
      }
    }
    c1 = block_sum(c1, red) / (float)D;
    c2 = block_sum(c2, red) / (float)D;
    for (long long i = t0; i < D; i += STEP) {
      float g[V], h[V], w[V], d[V];
      walk_other<DT>(a.dy, row * a.lddy, a.ydt, i, D, g);
      walk_load<DT>(s, i, D, h);
      if (a.w) walk_other<DT>(a.w, 0, a.wdt, i, D, w);
      if (a.ds) walk_load<DT>(gptr((const raw_t*)a.ds) + row * a.ldds, i, D, d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float v = a.w ? g[e] * w[e] : g[e];
        g[e] = rstd * (v - c1 - (h[e] - mu) * rstd * c2) + (a.ds ? d[e] : 0.f);
      }
      walk_store<DT>(a.dx, row * D, DT, i, D, g);
      if (a.dz) walk_store<DT>(a.dz, row * D, a.zdt, i, D, g);
    }
  }
}

// V columns a thread over one chunk of rows: part[chunk][0 dw, 1 db][D]
template <int DT>
__global__ __launch_bounds__(NT) void ln_param_part_kernel(const Bwd a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  constexpr int V = row_vec<DT>();
  const long long c = ((long long)blockIdx.x * NT + threadIdx.x) * V;
  if (c >= a.D) return;
  const long long per = (a.rows + a.chunks - 1) / a.chunks;
  const long long r0 = blockIdx.y * per, r1 = r0 + per < a.rows ? r0 + per : a.rows;
  float dw[V], db[V];
#pragma unroll
  for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.f;
  for (long long r = r0; r < r1; ++r) {
    float g[V], h[V];
    walk_other<DT>(a.dy, r * a.lddy, a.ydt, c, a.D, g);
    walk_load<DT>(gptr((const raw_t*)a.s) + r * a.lds, c, a.D, h);
    const float mu = a.mean[r], rstd = a.rstd[r];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      dw[e] = fmaf(g[e], (h[e] - mu) * rstd, dw[e]);
      db[e] += g[e];
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (c + e < a.D) {
      a.part[2LL * blockIdx.y * a.D + c + e] = dw[e];
      a.part[(2LL * blockIdx.y + 1) * a.D + c + e] = db[e];
    }
}

// ---------------------------------------------------------------------------
// Rows of up to 16384 elements: a row is held in the registers of TR threads, E
// elements each in 16-byte accesses, so that x, z (forward) and dy, s, ds
// (backward) are read once and the statistics are taken from registers.
// Workgroups of 256 threads hold 256 / TR rows at a time (TR >= 256: one) and
// stride over the rows.

template <int TR> struct RowSum {      // sums over the TR threads of a row
  static constexpr int W = TR / 64;    // waves a row
  static constexpr int BT = TR < 256 ? 256 : TR;
  // red: one float a wave of the workgroup, not read or written between this
  // call's barrier and the next call's (two buffers in turn)
  static __device__ __forceinline__ float sum(float v, float* red) {
    v += dpp_f<0xB1>(v);               // quad_perm [1,0,3,2]
    v += dpp_f<0x4E>(v);               // quad_perm [2,3,0,1]
    v += dpp_f<0x141>(v);              // row_half_mirror
    v += dpp_f<0x140>(v);              // row_mirror: 16 lanes
    if (TR >= 32) v = swap_sum16(v);
    if (TR >= 64) v = swap_sum32(v);
    if (TR <= 64) return v;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    kfac_lds_barrier();
    const int w0 = wave / (W ? W : 1) * W;
    float r = red[w0];
#pragma unroll
    for (int i = 1; i < W; ++i) r += red[w0 + i];
    return r;
  }
};

// A thread's R accesses, issued back to back.  One that lies behind the row's
// end for the whole wave is left out: a size class may be half empty.
// TINY: the row may be shorter than one access.
template <int DT, bool TAIL, bool STREAM, bool TINY, int R>
__device__ __forceinline__ void load_all(const AS1 typename DTypeTraits<DT>::raw_t* row, int t0,
                                         int step, int n, u32x4n* raw) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    raw[r] = (u32x4n)0u;
    if constexpr (TINY) {
      constexpr int V = row_vec<DT>();
      if (n < V) {                       // the row's elements last, as clip_vec expects them
        float f[V];
#pragma unroll
        for (int e = 0; e < V; ++e)
          f[e] = t0 == 0 && r == 0 && e >= V - n ? DTypeTraits<DT>::to_f32(row[e - (V - n)]) : 0.f;
        raw[r] = f32_to_vec<DT>(f);
        continue;
      }
    }
    if (r == 0 || __builtin_amdgcn_readfirstlane(t0 + r * step) < n)
      raw[r] = load_vec<DT, TAIL, STREAM>(row, t0 + r * step, n);
  }
}

// E elements in one of the three types (uniform over the launch): the weights,
// and z, dy, dz or y where their type is not the stream's.  V elements in
// accesses of at most 16 bytes; the access past the row's end one by one.
template <int DT, int V, int R>
__device__ __forceinline__ void load_as(const void* p, long long off, int t0, int step, int n,
                                        float* f) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  typedef raw_t vec_t __attribute__((ext_vector_type(V)));
  typedef vec_t vec_u __attribute__((aligned(sizeof(raw_t))));
  const AS1 raw_t* q = gptr((const raw_t*)p) + off;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = t0 + r * step;
    if (i + V <= n) {
      const vec_t v = *(const AS1 vec_u*)(q + i);
#pragma unroll
      for (int e = 0; e < V; ++e) f[r * V + e] = DTypeTraits<DT>::to_f32(v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        f[r * V + e] = i + e < n ? DTypeTraits<DT>::to_f32(q[i + e]) : 0.f;
    }
  }
}
template <int DT, int V, int R>
__device__ __forceinline__ void store_as(void* p, long long off, int t0, int step, int n,
                                         const float* f) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  typedef raw_t vec_t __attribute__((ext_vector_type(V)));
  typedef vec_t vec_u __attribute__((aligned(sizeof(raw_t))));
  AS1 raw_t* q = gptr((raw_t*)p) + off;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = t0 + r * step;
    vec_t v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = DTypeTraits<DT>::from_f32(f[r * V + e]);
    if (i + V <= n) {
      *(AS1 vec_u*)(q + i) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i + e < n) q[i + e] = v[e];
    }
  }
}
template <int V, int R>
__device__ __forceinline__ void load_other(const void* p, long long off, int dt, int t0, int step,
                                           int n, float* f) {
  if (dt == KDT_F32) load_as<KDT_F32, V, R>(p, off, t0, step, n, f);
  else if (dt == KDT_BF16) load_as<KDT_BF16, V, R>(p, off, t0, step, n, f);
  else load_as<KDT_F16, V, R>(p, off, t0, step, n, f);
}
template <int V, int R>
__device__ __forceinline__ void store_other(void* p, long long off, int dt, int t0, int step,
                                            int n, const float* f) {
  if (dt == KDT_F32) store_as<KDT_F32, V, R>(p, off, t0, step, n, f);
  else if (dt == KDT_BF16) store_as<KDT_BF16, V, R>(p, off, t0, step, n, f);
  else store_as<KDT_F16, V, R>(p, off, t0, step, n, f);
}

// Bound by HBM: x and z in, s and y out.  32768 x 8192 bf16 418 us (5.1 TB/s), 8192
// x 4096 fp32 83 us (6.4 TB/s), without z 43 us (6.2 TB/s); a row that fills its
// registers by two thirds or starts at an odd element is slower (16384 x 4104 fp16 74
// us in a training step, x 4097 86 us, x 4096 66 us).  x fp32 and z bf16, as under
// autocast: 32768 x 8192 702 us (5.4 TB/s).  One row of 512: 2 us; 700 x 650 fp32: 5.8 us.
template <int DT, int TR, int E, bool TAIL>
__global__ __launch_bounds__(RowSum<TR>::BT) void ln_fwd_kernel(const Fwd a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  constexpr int V = row_vec<DT>(), R = E / V, BT = RowSum<TR>::BT, RPW = BT / TR;
  __shared__ float red[2][BT / 64];
  const int t = threadIdx.x % TR, sub = threadIdx.x / TR;
  const int D = (int)a.D, t0 = t * V, step = TR * V;
  const float inv_d = 1.f / (float)D, scale = sum_scale(D);
  float w[E], b[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { w[e] = 1.f; b[e] = 0.f; }
  if (a.w) load_other<V, R>(a.w, 0, a.wdt, t0, step, D, w);
  if (a.b) load_other<V, R>(a.b, 0, a.bdt, t0, step, D, b);
  for (long long base = (long long)blockIdx.x * RPW; base < a.rows;
       base += (long long)gridDim.x * RPW) {
    const bool live = base + sub < a.rows;
    const long long row = live ? base + sub : a.rows - 1;
    const AS1 raw_t* x = gptr((const raw_t*)a.x) + row * a.ldx;
    float f[E];
    u32x4n raw[R];
    if (a.z) {
      float g[E];
      // x and z are read for the last time: s is what the backward pass reads
      // (16384 x 4096 fp16 in a training step: 106 us as plain loads, 104 so; 32768 x
      // 8192 bf16 409 and 405)
      load_all<DT, TAIL, true, E == 8 && TR == 16 && TAIL, R>(x, t0, step, D, raw);
      if (a.zdt == DT) {
        const AS1 raw_t* z = gptr((const raw_t*)a.z) + row * a.ldz;
        u32x4n zraw[R];
        load_all<DT, TAIL, true, E == 8 && TR == 16 && TAIL, R>(z, t0, step, D, zraw);
#pragma unroll
        for (int r = 0; r < R; ++r)
          vec_to_f32<DT>(clip_vec<DT, TAIL>(zraw[r], t0 + r * step, D), g + r * V);
      } else {
        load_other<V, R>(a.z, row * a.ldz, a.zdt, t0, step, D, g);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = t0 + r * step;
        vec_to_f32<DT>(clip_vec<DT, TAIL>(raw[r], i, D), f + r * V);
#pragma unroll
        for (int e = 0; e < V; ++e)       // the sum as it is stored is what is normed
          f[r * V + e] = DTypeTraits<DT>::to_f32(
              DTypeTraits<DT>::from_f32(f[r * V + e] + g[r * V + e]));
        if (live) store_vec<DT, TAIL>(gptr((raw_t*)a.s) + row * D, i, D, f + r * V);
      }
    } else {
      load_all<DT, TAIL, false, E == 8 && TR == 16 && TAIL, R>(x, t0, step, D, raw);
#pragma unroll
      for (int r = 0; r < R; ++r)
        vec_to_f32<DT>(clip_vec<DT, TAIL>(raw[r], t0 + r * step, D), f + r * V);
    }
    float acc = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc = fmaf(f[e], scale, acc);
    // exact for a constant row
    const float mu = RowSum<TR>::sum(acc, red[0]) / ((float)D * scale);
    acc = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = f[r * V + e] - mu;
        f[r * V + e] = d;
        acc = fmaf(d, t0 + r * step + e < D ? d : 0.f, acc);
      }
    const float rstd = 1.f / sqrtf(RowSum<TR>::sum(acc, red[1]) * inv_d + a.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = fmaf(f[e] * rstd, w[e], b[e]);
    if (live) {
      if (a.ydt == DT) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          store_vec<DT, TAIL>(gptr((raw_t*)a.y) + row * D, t0 + r * step, D, f + r * V);
      } else {
        store_other<V, R>(a.y, row * D, a.ydt, t0, step, D, f);
      }
      if (t == 0 && a.mean) {
        a.mean[row] = mu;
        a.rstd[row] = rstd;
      }
    }
  }
}

// dx (and dz), and the workgroup's rows' part of dw and db in registers: two
// floats an element, added over the workgroup's row groups at the end.  Bound by
// HBM: dy, ds and s in, dx out.  32768 x 8192 bf16 390 us (5.5 TB/s), 65536 x 650
// fp32 127 us (5.4 TB/s), 700 x 650 fp32 6.7 us.  16384 x 4104 fp16 113 us (4.8 TB/s),
// 8192 x 16384 fp16 200 us (5.4 TB/s; in fp32, where some registers spill, 5.3).  An fp32
// stream with dz in bf16: 32768 x 8192 875 us (5.5 TB/s).
template <int DT, int TR, int E, bool TAIL>
__global__ __launch_bounds__(RowSum<TR>::BT) void ln_bwd_kernel(const Bwd a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  constexpr int V = row_vec<DT>(), R = E / V, BT = RowSum<TR>::BT, RPW = BT / TR;
  __shared__ float red[2][BT / 64];
  __shared__ float fold[RPW > 1 ? RPW * TR * E : 1];
  const int t = threadIdx.x % TR, sub = threadIdx.x / TR;
  const int D = (int)a.D, t0 = t * V, step = TR * V;
  const float inv_d = 1.f / (float)D;
  float w[E], dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { w[e] = 1.f; dw[e] = 0.f; db[e] = 0.f; }
  if (a.w) load_other<V, R>(a.w, 0, a.wdt, t0, step, D, w);
  for (long long base = (long long)blockIdx.x * RPW; base < a.rows;
       base += (long long)gridDim.x * RPW) {
    const bool live = base + sub < a.rows;
    const long long row = live ? base + sub : a.rows - 1;
    const AS1 raw_t* s = gptr((const raw_t*)a.s) + row * a.lds;
    const AS1 raw_t* ds = gptr((const raw_t*)a.ds) + row * a.ldds;
    float h[E], g[E];
    u32x4n sraw[R], eraw[R];
    load_all<DT, TAIL, true, E == 8 && TR == 16 && TAIL, R>(s, t0, step, D, sraw);
    if (a.ds) load_all<DT, TAIL, true, E == 8 && TR == 16 && TAIL, R>(ds, t0, step, D, eraw);
    if (a.ydt == DT) {
      const AS1 raw_t* dy = gptr((const raw_t*)a.dy) + row * a.lddy;
      u32x4n graw[R];
      load_all<DT, TAIL, true, E == 8 && TR == 16 && TAIL, R>(dy, t0, step, D, graw);
#pragma unroll
      for (int r = 0; r < R; ++r)
        vec_to_f32<DT>(clip_vec<DT, TAIL>(graw[r], t0 + r * step, D), g + r * V);
    } else {
      load_other<V, R>(a.dy, row * a.lddy, a.ydt, t0, step, D, g);
    }
    const float mu = a.mean[row], rstd = a.rstd[row];
#pragma unroll
    for (int r = 0; r < R; ++r)
      vec_to_f32<DT>(clip_vec<DT, TAIL>(sraw[r], t0 + r * step, D), h + r * V);
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = (h[e] - mu) * rstd;
    // past the row's end g is 0 and h is (0 - mu) rstd, to be 0 too where that is no
    // number (a select in every row: 16384 x 4097 fp16 106 -> 118 us)
    if (__any(!(fabsf(mu * rstd) < INFINITY))) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (t0 + e / V * step + e % V >= D) h[e] = 0.f;
    }
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!live) g[e] = 0.f;
      dw[e] = fmaf(g[e], h[e], dw[e]);
      db[e] += g[e];
      g[e] *= w[e];
      c1 += g[e];
      c2 = fmaf(g[e], h[e], c2);
    }
    if (a.dx) {
      c1 = RowSum<TR>::sum(c1, red[0]) * inv_d;
      c2 = RowSum<TR>::sum(c2, red[1]) * inv_d;
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] = rstd * (g[e] - c1 - h[e] * c2);
      if (a.ds) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          vec_to_f32<DT>(clip_vec<DT, TAIL>(eraw[r], t0 + r * step, D), h + r * V);
#pragma unroll
          for (int e = 0; e < V; ++e) g[r * V + e] += h[r * V + e];
        }
      }
      if (live) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          store_vec<DT, TAIL>(gptr((raw_t*)a.dx) + row * D, t0 + r * step, D, g + r * V);
        if (a.dz) store_other<V, R>(a.dz, row * D, a.zdt, t0, step, D, g);
      }
    }
  }
  if (!a.part) return;
  float* out = a.part + 2LL * blockIdx.x * D;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float* v = k ? db : dw;
    if (RPW > 1) {                        // row groups added in order
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) fold[(sub * E + e) * TR + t] = v[e];
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          for (int j = 1; j < RPW; ++j) v[e] += fold[(j * E + e) * TR + t];
      }
    }
    if (sub == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        store_vec<KDT_F32, true>(gptr(out + (long long)k * D), t0 + r * step, D, v + r * V);
      if (V == 8) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          store_vec<KDT_F32, true>(gptr(out + (long long)k * D), t0 + r * step + 4, D,
                                   v + r * V + 4);
      }
    }
  }
}

// dw, db from the parts, 32 columns a workgroup: each of 32 threads a column
// adds every 32nd part in order, then the 32 sums are added in order (256 parts
// of 8192 columns: 5 us)
__global__ __launch_bounds__(1024) void ln_param_sum_kernel(const Bwd a) {
  __shared__ float sh[2][32][33];
  const int cx = threadIdx.x & 31, k0 = threadIdx.x >> 5;
  for (long long c0 = blockIdx.x * 32LL; c0 < a.D; c0 += gridDim.x * 32LL) {
    const long long c = c0 + cx;
    float dw = 0.f, db = 0.f;
    if (c < a.D) {
#pragma unroll 4
      for (int k = k0; k < a.chunks; k += 32) {
        dw += a.part[2LL * k * a.D + c];
        db += a.part[(2LL * k + 1) * a.D + c];
      }
    }
    sh[0][k0][cx] = dw;
    sh[1][k0][cx] = db;
    __syncthreads();
    if (k0 < 2 && c < a.D) {
      float v = 0.f;
      for (int k = 0; k < 32; ++k) v += sh[k0][k][cx];
      if (k0 == 0 && a.dw) st_any(a.dw, c, a.wdt, v);
      if (k0 == 1 && a.db) st_any(a.db, c, a.bdt, v);
    }
    __syncthreads();                       // sh is written again
  }
}

bool dtype_ok(int dt) { return dt == KDT_F32 || dt == KDT_BF16 || dt == KDT_F16; }

constexpr long long LONG_ROW = 16384;     // longer rows: the kernels that loop over the row

// Threads and elements a row (TR, E): the first that holds D.  24 elements a thread
// stand where a class of 16 with twice the threads would be half empty and is slower
// (us with 16 | with 24; fp16, a training step without a residual):
//   forward    131072 x 300 57 | 44, 65536 x 650 53 | 42, 32768 x 1280 48 | 33, 16384 x
//              4104 84 | 72 (32768 x 2560 85 | 86); but 8192 x 10240 95 | 108
//   backward   65536 x 650 78 | 58, 32768 x 1280 71 | 52, 32768 x 2560 134 | 99, 16384 x
//              4104 127 | 90, 8192 x 10240 195 | 108; but 131072 x 300 72 | 106
// In fp32 they gain little (16384 x 5120 forward 143 | 147, backward 188 | 175; 65536 x 650
// 84 | 87 and 95 | 89) and cost time where there are few rows (700 x 650: 5.7 | 7.2 and
// 7.0 | 8.9), so there they are taken only for wide rows' gradients.
// (The backward pass of more than 12288 elements, 16 of 1024 threads | 32 of 512: 8192 x
// 14336 fp16 248 | 142, 4096 x 16384 fp32 267 | 144.)
#define LN_FWD_SIZES(F) \
  F(16, 8) F(32, 8) F(16, 24) F(64, 8) F(32, 24) F(64, 16) F(64, 24) F(128, 16) F(128, 24) \
  F(256, 16) F(256, 24) F(512, 16) F(1024, 16)
#define LN_BWD_SIZES(F) \
  F(16, 8) F(32, 8) F(64, 8) F(32, 24) F(64, 16) F(64, 24) F(128, 16) F(128, 24) F(256, 16) F(256, 24) \
  F(512, 16) F(512, 24) F(512, 32)

constexpr bool size_of_type(int dt, int tr, int e) {
  return dt != KDT_F32 || e != 24 || tr == 512;
}

bool looped(long long D) { return D > LONG_ROW; }

unsigned groups(long long n) { return (unsigned)(n < MAX_GROUPS ? n : MAX_GROUPS); }

// workgroups that stride over the rows: at most `cap` of 256 threads (fewer, wider ones alike)
long long row_blocks(long long rows, int tr, long long cap) {
  const long long per = tr < 256 ? 256 / tr : 1, most = tr > 256 ? cap * 256 / tr : cap;
  const long long n = (rows + per - 1) / per;
  return n < most ? n : most;
}

// A workgroup loads the weights once for all its rows.  With 24 elements of 16 bits a
// thread no more workgroups than run at once, three a CU (us with 4096 | 768: 5001 x
// 4097 fp16 38 | 26, 16384 x 4104 80 | 74, 32768 x 1280 41 | 33, 65536 x 650 52 | 43).
// Of 512 threads and more half as many.  Over 512 .. 32768 rows of 6200 .. 16384 elements
// in 16 and 32 bits, without z: 0.78 .. 1.03 of the time (2048 x 8191 fp16 27 | 21, 8192 x
// 8191 80 | 65, 8192 x 16384 bf16 111 | 107, 32768 x 8192 fp32 385 | 389).  With z, where s
// moves as well, 0.82 .. 1.04 up to 4096 rows (2048 x 8191 45 | 36, 4096 x 8191 71 | 64),
// nothing from 8192 to 16384 (0.97 .. 1.06, the last 8192 x 16384 fp32), and up to 3 %
// lost beyond (32768 x 8192 bf16 402 | 412, 24576 x 8191 376 | 383).
long long fwd_blocks(const Fwd& a, int tr, int e) {
  const bool half = tr >= 512 && (!a.z || a.rows < 16384);
  return row_blocks(a.rows, tr, e == 24 ? 768 : half ? 2048 : 4096);
}
// A workgroup leaves 8 D bytes of sums: fewer of them for longer rows (us with
// 512 | 1024, the sums' kernel among them: 16384 x 4096 fp16 91 | 97, 65536 x 650 fp32
// 99 | 110, 8192 x 12000 fp16 134 | 142; 131072 x 512 fp16 103 | 81, 131072 x 300 108 | 79,
// 1048576 x 64 170 | 121).
long long bwd_blocks(long long rows, long long D, int tr) {
  return row_blocks(rows, tr, D > 512 ? 512 : 1024);
}

int param_chunks(long long rows, long long D, int dt) {
  if (!looped(D)) {
#define F(TR, E) if (D <= TR * E && size_of_type(dt, TR, E)) return (int)bwd_blocks(rows, D, TR);
    LN_BWD_SIZES(F)
#undef F
  }
  const long long c = (rows + 63) / 64;
  return (int)(c < 512 ? c : 512);
}

template <int DT, int TR, int E>
void launch_fwd(const Fwd& a, hipStream_t st) {
  const dim3 grid((unsigned)fwd_blocks(a, TR, E)), block(RowSum<TR>::BT);
  if (a.D % row_vec<DT>())
    hipLaunchKernelGGL((ln_fwd_kernel<DT, TR, E, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((ln_fwd_kernel<DT, TR, E, false>), grid, block, 0, st, a);
}
template <int DT, int TR, int E>
void launch_bwd(const Bwd& a, hipStream_t st) {
  const dim3 grid((unsigned)bwd_blocks(a.rows, a.D, TR)), block(RowSum<TR>::BT);
  if (a.D % row_vec<DT>())
    hipLaunchKernelGGL((ln_bwd_kernel<DT, TR, E, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((ln_bwd_kernel<DT, TR, E, false>), grid, block, 0, st, a);
}
template <int DT> void launch_fwd_any(const Fwd& a, hipStream_t st) {
  if (looped(a.D)) {
    hipLaunchKernelGGL(ln_fwd_long_kernel<DT>, dim3(groups(a.rows)), dim3(LT), 0, st, a);
    return;
  }
#define F(TR, E) \
  if constexpr (size_of_type(DT, TR, E)) if (a.D <= TR * E) return launch_fwd<DT, TR, E>(a, st);
  LN_FWD_SIZES(F)
#undef F
}
template <int DT> void launch_bwd_any(const Bwd& a, hipStream_t st) {
  if (looped(a.D)) {
    if (a.dx)
      hipLaunchKernelGGL(ln_bwd_long_kernel<DT>, dim3(groups(a.rows)), dim3(LT), 0, st, a);
    const long long cols = NT * row_vec<DT>();
    if (a.part)
      hipLaunchKernelGGL(ln_param_part_kernel<DT>,
                         dim3((unsigned)((a.D + cols - 1) / cols), a.chunks), dim3(NT), 0, st, a);
    return;
  }
#define F(TR, E) \
  if constexpr (size_of_type(DT, TR, E)) if (a.D <= TR * E) return launch_bwd<DT, TR, E>(a, st);
  LN_BWD_SIZES(F)
#undef F
}

}  // namespace

// floats of the workspace of one backward call that asks for dw or db
KFAC_API long long kfac_ln_ws_floats(long long rows, long long D, int sdt) {
  return 2LL * param_chunks(rows, D, sdt) * D;
}

KFAC_API int kfac_ln_forward(const KfacLnFwd* args, hipStream_t stream) {
  const Fwd a = *args;
  if (!a.x || !a.y || a.rows <= 0 || a.rows > 0x7fffffffLL || a.D <= 0 || !dtype_ok(a.sdt) ||
      !dtype_ok(a.ydt) || (a.z && (!a.s || !dtype_ok(a.zdt))) || (a.w && !dtype_ok(a.wdt)) ||
      (a.b && !dtype_ok(a.bdt)) || !a.mean != !a.rstd)
    return -2;
  if (a.sdt == KDT_F32) launch_fwd_any<KDT_F32>(a, stream);
  else if (a.sdt == KDT_BF16) launch_fwd_any<KDT_BF16>(a, stream);
  else launch_fwd_any<KDT_F16>(a, stream);
  return (int)hipGetLastError();
}

KFAC_API int kfac_ln_backward(const KfacLnBwd* args, hipStream_t stream) {
  Bwd a = *args;
  if (!a.dy || !a.s || !a.mean || !a.rstd || a.rows <= 0 || a.rows > 0x7fffffffLL || a.D <= 0 ||
      !dtype_ok(a.sdt) || !dtype_ok(a.ydt) || (a.dz && (!a.dx || !dtype_ok(a.zdt))) ||
      ((a.w || a.dw) && !dtype_ok(a.wdt)) || (a.db && !dtype_ok(a.bdt)) ||
      ((a.dw || a.db) && !a.part))
    return -2;
  if (!a.dw && !a.db) a.part = nullptr;
  a.chunks = param_chunks(a.rows, a.D, a.sdt);
  if (a.sdt == KDT_F32) launch_bwd_any<KDT_F32>(a, stream);
  else if (a.sdt == KDT_BF16) launch_bwd_any<KDT_BF16>(a, stream);
  else launch_bwd_any<KDT_F16>(a, stream);
  if (a.part)
    hipLaunchKernelGGL(ln_param_sum_kernel, dim3(groups((a.D + 31) / 32)), dim3(1024), 0, stream,
                       a);
  return (int)hipGetLastError();
}
