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
#include "common.h"

namespace {

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

struct Fwd {
  const void *x, *z, *w, *b;
  void *y, *s;
  float *mean, *rstd;
  long long ldx, ldz, rows, D;
  int sdt, zdt, wdt, bdt, ydt;
  float eps;
};

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
  if (threadIdx.x == 0) {
    a.mean[row] = mu;
    a.rstd[row] = rstd;
  }
}

struct Bwd {
  const void *dy, *ds, *s, *w;
  const float *mean, *rstd;
  void *dx, *dz, *dw, *db;
  float* part;
  long long lddy, ldds, lds, rows, D;
  int sdt, zdt, wdt, bdt, ydt, chunks;
};

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

__global__ __launch_bounds__(NT) void ln_param_sum_kernel(const Bwd a) {
  const long long c = (long long)blockIdx.x * NT + threadIdx.x;
  if (c >= a.D) return;
  float dw = 0.f, db = 0.f;
  for (int k = 0; k < a.chunks; ++k) {
    dw += a.part[2LL * k * a.D + c];
    db += a.part[(2LL * k + 1) * a.D + c];
  }
  if (a.dw) st_any(a.dw, c, a.wdt, dw);
  if (a.db) st_any(a.db, c, a.bdt, db);
}

int param_chunks(long long rows) {
  const long long c = (rows + 63) / 64;
  return (int)(c < 512 ? c : 512);
}

bool dtype_ok(int dt) { return dt == KDT_F32 || dt == KDT_BF16 || dt == KDT_F16; }

}  // namespace

// floats of the workspace of one backward call that asks for dw or db
KFAC_API long long kfac_ln_ws_floats(long long rows, long long D) {
  return 2LL * param_chunks(rows) * D;
}

// z and s null: the norm of x.  w, b may be null.  mean, rstd: fp32, one a row.
KFAC_API int kfac_ln_forward(const void* x, long long ldx, int sdt, const void* z, long long ldz,
                             int zdt, const void* w, int wdt, const void* b, int bdt, void* y,
                             int ydt, void* s, float* mean, float* rstd, long long rows,
                             long long D, float eps, hipStream_t stream) {
  if (rows <= 0 || rows > 0x7fffffffLL || D <= 0 || !dtype_ok(sdt) || !dtype_ok(ydt) ||
      (z && (!s || !dtype_ok(zdt))) || (w && !dtype_ok(wdt)) || (b && !dtype_ok(bdt)))
    return -2;
  Fwd a = {x, z, w, b, y, s, mean, rstd, ldx, ldz, rows, D, sdt, zdt, wdt, bdt, ydt, eps};
  hipLaunchKernelGGL(ln_fwd_long_kernel, dim3((unsigned)rows), dim3(NT), 0, stream, a);
  return (int)hipGetLastError();
}

// ds (the gradient that reaches s itself), dx, dz, dw, db may be null; part
// is read only where dw or db is asked for
KFAC_API int kfac_ln_backward(const void* dy, long long lddy, int ydt, const void* ds,
                              long long ldds, const void* s, long long lds, int sdt,
                              const void* w, int wdt, int bdt, const float* mean,
                              const float* rstd, void* dx, void* dz, int zdt, void* dw, void* db,
                              float* part, long long rows, long long D, hipStream_t stream) {
  if (rows <= 0 || rows > 0x7fffffffLL || D <= 0 || !dtype_ok(sdt) || !dtype_ok(ydt) ||
      (dz && (!dx || !dtype_ok(zdt))) || ((w || dw) && !dtype_ok(wdt)) ||
      (db && !dtype_ok(bdt)) || ((dw || db) && !part))
    return -2;
  Bwd a = {dy, ds, s, w, mean, rstd, dx, dz, dw, db, part, lddy, ldds, lds, rows, D,
           sdt, zdt, wdt, bdt, ydt, param_chunks(rows)};
  if (dx) hipLaunchKernelGGL(ln_bwd_long_kernel, dim3((unsigned)rows), dim3(NT), 0, stream, a);
  if (dw || db) {
    const unsigned cols = (unsigned)((D + NT - 1) / NT);
    hipLaunchKernelGGL(ln_param_part_kernel, dim3(cols, a.chunks), dim3(NT), 0, stream, a);
    hipLaunchKernelGGL(ln_param_sum_kernel, dim3(cols), dim3(NT), 0, stream, a);
  }
  return (int)hipGetLastError();
}
