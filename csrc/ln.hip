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
#include "rows.h"

// argument records (ops/ln.py packs the same fields); chunks is set here
struct KfacLnFwd {
  const void *x, *z, *w, *b;
  void *y, *s;
  float *mean, *rstd;
  long long ldx, ldz, rows, D;
  int sdt, zdt, wdt, bdt, ydt;
  float eps;
};

struct KfacLnBwd {
  const void *dy, *ds, *s, *w;
  const float *mean, *rstd;
  void *dx, *dz, *dw, *db;
  float* part;
  long long lddy, ldds, lds, rows, D;
  int sdt, zdt, wdt, bdt, ydt, chunks;
};

namespace {

typedef KfacLnFwd Fwd;
typedef KfacLnBwd Bwd;

constexpr int NT = 256;

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
  for (int i = 1; i < NT / 64; ++i) r += red[i];
  return r;
}

__global__ __launch_bounds__(NT) void ln_fwd_long_kernel(const Fwd a) {
  __shared__ float red[NT / 64];
  const long long row = blockIdx.x, D = a.D;
  const long long xo = row * a.ldx, zo = row * a.ldz, yo = row * D;
  float acc = 0.f;
  for (long long i = threadIdx.x; i < D; i += NT) {
    float v = ld_any(a.x, xo + i, a.sdt);
    if (a.z) {
      v += ld_any(a.z, zo + i, a.zdt);
      st_any(a.s, yo + i, a.sdt, v);
      v = ld_any(a.s, yo + i, a.sdt);    // this thread's own store: the rounded sum is normed
    }
    acc += v;
  }
  const void* sp = a.z ? a.s : a.x;
  const long long so = a.z ? yo : xo;
  const float mu = block_sum(acc, red) / (float)D;
  acc = 0.f;
  for (long long i = threadIdx.x; i < D; i += NT) {
    const float d = ld_any(sp, so + i, a.sdt) - mu;
    acc = fmaf(d, d, acc);
  }
  const float rstd = 1.f / sqrtf(block_sum(acc, red) / (float)D + a.eps);
  for (long long i = threadIdx.x; i < D; i += NT) {
    float v = (ld_any(sp, so + i, a.sdt) - mu) * rstd;
    if (a.w) v *= ld_any(a.w, i, a.wdt);
    if (a.b) v += ld_any(a.b, i, a.bdt);
    st_any(a.y, yo + i, a.ydt, v);
  }
  if (threadIdx.x == 0 && a.mean) {
    a.mean[row] = mu;
    a.rstd[row] = rstd;
  }
}

__global__ __launch_bounds__(NT) void ln_bwd_long_kernel(const Bwd a) {
  __shared__ float red[NT / 64];
  const long long row = blockIdx.x, D = a.D;
  const long long go = row * a.lddy, eo = row * a.ldds, so = row * a.lds, xo = row * D;
  const float mu = a.mean[row], rstd = a.rstd[row];
  float c1 = 0.f, c2 = 0.f;
  for (long long i = threadIdx.x; i < D; i += NT) {
    float g = ld_any(a.dy, go + i, a.ydt);
    if (a.w) g *= ld_any(a.w, i, a.wdt);
    c1 += g;
    c2 = fmaf(g, (ld_any(a.s, so + i, a.sdt) - mu) * rstd, c2);
  }
  c1 = block_sum(c1, red) / (float)D;
  c2 = block_sum(c2, red) / (float)D;
  for (long long i = threadIdx.x; i < D; i += NT) {
    float g = ld_any(a.dy, go + i, a.ydt);
    if (a.w) g *= ld_any(a.w, i, a.wdt);
    const float h = (ld_any(a.s, so + i, a.sdt) - mu) * rstd;
    float d = rstd * (g - c1 - h * c2);
    if (a.ds) d += ld_any(a.ds, eo + i, a.sdt);
    st_any(a.dx, xo + i, a.sdt, d);
    if (a.dz) st_any(a.dz, xo + i, a.zdt, d);
  }
}

// one column a thread over one chunk of rows: part[chunk][0 dw, 1 db][D]
__global__ __launch_bounds__(NT) void ln_param_part_kernel(const Bwd a) {
  const long long c = (long long)blockIdx.x * NT + threadIdx.x;
  if (c >= a.D) return;
  const long long per = (a.rows + a.chunks - 1) / a.chunks;
  const long long r0 = blockIdx.y * per, r1 = r0 + per < a.rows ? r0 + per : a.rows;
  float dw = 0.f, db = 0.f;
  for (long long r = r0; r < r1; ++r) {
    const float g = ld_any(a.dy, r * a.lddy + c, a.ydt);
    dw = fmaf(g, (ld_any(a.s, r * a.lds + c, a.sdt) - a.mean[r]) * a.rstd[r], dw);
    db += g;
  }
  a.part[(2LL * blockIdx.y) * a.D + c] = dw;
  a.part[(2LL * blockIdx.y + 1) * a.D + c] = db;
}

// ---------------------------------------------------------------------------
// Rows of V .. 16384 elements: a row is held in the registers of TR threads, E
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

template <int DT, int TR, int E, bool TAIL>
__global__ __launch_bounds__(RowSum<TR>::BT) void ln_fwd_kernel(const Fwd a) {
  typedef typename DTypeTraits<DT>::raw_t raw_t;
  constexpr int V = row_vec<DT>(), R = E / V, BT = RowSum<TR>::BT, RPW = BT / TR;
  __shared__ float red[2][BT / 64];
  const int t = threadIdx.x % TR, sub = threadIdx.x / TR;
  const int D = (int)a.D, t0 = t * V, step = TR * V;
  const float inv_d = 1.f / (float)D;
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
#pragma unroll
    for (int r = 0; r < R; ++r) raw[r] = load_vec<DT, TAIL>(x, t0 + r * step, D);
    if (a.z) {
      float g[E];
      if (a.zdt == DT) {
        const AS1 raw_t* z = gptr((const raw_t*)a.z) + row * a.ldz;
        u32x4n zraw[R];
#pragma unroll
        for (int r = 0; r < R; ++r) zraw[r] = load_vec<DT, TAIL>(z, t0 + r * step, D);
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
#pragma unroll
      for (int r = 0; r < R; ++r)
        vec_to_f32<DT>(clip_vec<DT, TAIL>(raw[r], t0 + r * step, D), f + r * V);
    }
    float acc = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc += f[e];
    const float mu = RowSum<TR>::sum(acc, red[0]) * inv_d;
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
// floats an element, added over the workgroup's row groups at the end
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
#pragma unroll
    for (int r = 0; r < R; ++r) sraw[r] = load_vec<DT, TAIL>(s, t0 + r * step, D);
    if (a.ds) {
#pragma unroll
      for (int r = 0; r < R; ++r) eraw[r] = load_vec<DT, TAIL>(ds, t0 + r * step, D);
    }
    if (a.ydt == DT) {
      const AS1 raw_t* dy = gptr((const raw_t*)a.dy) + row * a.lddy;
      u32x4n graw[R];
#pragma unroll
      for (int r = 0; r < R; ++r) graw[r] = load_vec<DT, TAIL>(dy, t0 + r * step, D);
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
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[e] = (h[e] - mu) * rstd;
      if (!live) g[e] = 0.f;
      dw[e] = fmaf(g[e], h[e], dw[e]);           // past the row's end g is 0
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
// adds every 32nd part in order, then the 32 sums are added in order
__global__ __launch_bounds__(1024) void ln_param_sum_kernel(const Bwd a) {
  __shared__ float sh[2][32][33];
  const int cx = threadIdx.x & 31, k0 = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + cx;
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
}

bool dtype_ok(int dt) { return dt == KDT_F32 || dt == KDT_BF16 || dt == KDT_F16; }

// Threads and elements a row (TR, E): the narrowest that hold D.
constexpr long long LONG_ROW = 16384;     // longer rows: the kernels that loop over the row

#define LN_SIZES(F) F(16, 8) F(32, 8) F(64, 8) F(64, 16) F(128, 16) F(256, 16) F(512, 16) F(1024, 16)

bool looped(int dt, long long D) { return D > LONG_ROW || D < (dt == KDT_F32 ? 4 : 8); }

// threads a row
int row_threads(long long D) {
  int n = 0;
#define F(TR, E) if (!n && D <= TR * E) n = TR;
  LN_SIZES(F)
#undef F
  return n;
}

// workgroups that stride over the rows: at most `cap` of 256 threads (fewer, wider ones alike)
long long row_blocks(long long rows, long long D, long long cap) {
  const int tr = row_threads(D);
  const long long per = tr < 256 ? 256 / tr : 1, most = tr > 256 ? cap * 256 / tr : cap;
  const long long n = (rows + per - 1) / per;
  return n < most ? n : most;
}

constexpr long long FWD_BLOCKS = 4096, BWD_BLOCKS = 1024;

int param_chunks(int dt, long long rows, long long D) {
  if (!looped(dt, D)) return (int)row_blocks(rows, D, BWD_BLOCKS);
  const long long c = (rows + 63) / 64;
  return (int)(c < 512 ? c : 512);
}

template <int DT, int TR, int E>
void launch_fwd(const Fwd& a, hipStream_t st) {
  const dim3 grid((unsigned)row_blocks(a.rows, a.D, FWD_BLOCKS)), block(RowSum<TR>::BT);
  if (a.D % row_vec<DT>())
    hipLaunchKernelGGL((ln_fwd_kernel<DT, TR, E, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((ln_fwd_kernel<DT, TR, E, false>), grid, block, 0, st, a);
}
template <int DT, int TR, int E>
void launch_bwd(const Bwd& a, hipStream_t st) {
  const dim3 grid((unsigned)row_blocks(a.rows, a.D, BWD_BLOCKS)), block(RowSum<TR>::BT);
  if (a.D % row_vec<DT>())
    hipLaunchKernelGGL((ln_bwd_kernel<DT, TR, E, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((ln_bwd_kernel<DT, TR, E, false>), grid, block, 0, st, a);
}
template <int DT> void launch_fwd_any(const Fwd& a, hipStream_t st) {
  const int n = row_threads(a.D);
  bool done = false;
#define F(TR, E) if (!done && n == TR && a.D <= TR * E) { launch_fwd<DT, TR, E>(a, st); done = true; }
  LN_SIZES(F)
#undef F
}
template <int DT> void launch_bwd_any(const Bwd& a, hipStream_t st) {
  const int n = row_threads(a.D);
  bool done = false;
#define F(TR, E) if (!done && n == TR && a.D <= TR * E) { launch_bwd<DT, TR, E>(a, st); done = true; }
  LN_SIZES(F)
#undef F
}

}  // namespace

// floats of the workspace of one backward call that asks for dw or db
KFAC_API long long kfac_ln_ws_floats(int sdt, long long rows, long long D) {
  return 2LL * param_chunks(sdt, rows, D) * D;
}

// The argument record of ops/ln.py (`bytes`: its size there).  z and s null:
// the norm of x.  w, b may be null; mean, rstd (fp32, one a row) may be null
// where no backward pass follows.
KFAC_API int kfac_ln_forward(const KfacLnFwd* args, int bytes, hipStream_t stream) {
  if (bytes != (int)sizeof(KfacLnFwd)) return -2;
  const Fwd a = *args;
  if (!a.x || !a.y || a.rows <= 0 || a.rows > 0x7fffffffLL || a.D <= 0 || !dtype_ok(a.sdt) ||
      !dtype_ok(a.ydt) || (a.z && (!a.s || !dtype_ok(a.zdt))) || (a.w && !dtype_ok(a.wdt)) ||
      (a.b && !dtype_ok(a.bdt)) || !a.mean != !a.rstd)
    return -2;
  if (looped(a.sdt, a.D))
    hipLaunchKernelGGL(ln_fwd_long_kernel, dim3((unsigned)a.rows), dim3(NT), 0, stream, a);
  else if (a.sdt == KDT_F32)
    launch_fwd_any<KDT_F32>(a, stream);
  else if (a.sdt == KDT_BF16)
    launch_fwd_any<KDT_BF16>(a, stream);
  else
    launch_fwd_any<KDT_F16>(a, stream);
  return (int)hipGetLastError();
}

// ds (the gradient that reaches s itself), dx, dz, dw, db may be null; part
// (kfac_ln_ws_floats) is needed where dw or db is asked for
KFAC_API int kfac_ln_backward(const KfacLnBwd* args, int bytes, hipStream_t stream) {
  if (bytes != (int)sizeof(KfacLnBwd)) return -2;
  Bwd a = *args;
  if (!a.dy || !a.s || !a.mean || !a.rstd || a.rows <= 0 || a.rows > 0x7fffffffLL || a.D <= 0 ||
      !dtype_ok(a.sdt) || !dtype_ok(a.ydt) || (a.dz && (!a.dx || !dtype_ok(a.zdt))) ||
      ((a.w || a.dw) && !dtype_ok(a.wdt)) || (a.db && !dtype_ok(a.bdt)) ||
      ((a.dw || a.db) && !a.part))
    return -2;
  if (!a.dw && !a.db) a.part = nullptr;
  a.chunks = param_chunks(a.sdt, a.rows, a.D);
  if (looped(a.sdt, a.D)) {
    if (a.dx) hipLaunchKernelGGL(ln_bwd_long_kernel, dim3((unsigned)a.rows), dim3(NT), 0, stream, a);
    if (a.part)
      hipLaunchKernelGGL(ln_param_part_kernel, dim3((unsigned)((a.D + NT - 1) / NT), a.chunks),
                         dim3(NT), 0, stream, a);
  } else if (a.sdt == KDT_F32) {
    launch_bwd_any<KDT_F32>(a, stream);
  } else if (a.sdt == KDT_BF16) {
    launch_bwd_any<KDT_BF16>(a, stream);
  } else {
    launch_bwd_any<KDT_F16>(a, stream);
  }
  if (a.part)
    hipLaunchKernelGGL(ln_param_sum_kernel, dim3((unsigned)((a.D + 31) / 32)), dim3(1024), 0,
                       stream, a);
  return (int)hipGetLastError();
}
