// Argument records and entry points of the operators that csrc/torch_ops.cpp
// binds: plain C, read by hipcc and by the host compiler.
#pragma once

struct ihipStream_t;

// layer norm (csrc/ln.hip).  Element types are KfacDType codes (csrc/common.h).
// z and s null: the norm of x.  w, b may be null; mean, rstd (fp32, one a row)
// may be null where no backward pass follows.
struct KfacLnFwd {
  const void *x, *z, *w, *b;
  void *y, *s;
  float *mean, *rstd;
  long long ldx, ldz, rows, D;
  int sdt, zdt, wdt, bdt, ydt;
  float eps;
};

// ds (the gradient that reaches s itself), dx, dz, dw, db may be null; part
// (kfac_ln_ws_floats) is needed where dw or db is asked for.  chunks is set inside.
struct KfacLnBwd {
  const void *dy, *ds, *s, *w;
  const float *mean, *rstd;
  void *dx, *dz, *dw, *db;
  float* part;
  long long lddy, ldds, lds, rows, D;
  int sdt, zdt, wdt, bdt, ydt, chunks;
};

// rows of logits (csrc/vocab.hip).  Log probabilities: targets null: no
// logprob; entropy null: none; k 0: no alternatives.  Distillation: loss set,
// with ids and teacher.  stats, and keep_ids and keep_q of a distillation, null
// where no backward pass follows.  ws: kfac_vocab_ws_bytes.  stream is set inside.
struct KfacVocabFwd {
  const void* x;
  const long long* targets;
  float *logprob, *entropy, *top_lp;
  long long* top_ids;
  float* stats;                   // (M, L) a row
  const long long* ids;
  const void* teacher;
  float* loss;
  int* keep_ids;                  // each id once, and its mass
  float* keep_q;
  void* ws;
  long long ld, rows, V, ignore;
  int dt, k, K, tdt, stream;
  float inv_t;
};

// g, gh: gradients of logprob (or of the loss) and of the entropy, one a row at
// a distance of gs, ghs elements (0: the same for every row); gh, and g of log
// probabilities, may be null
struct KfacVocabBwd {
  const void* x;
  const float *stats, *entropy;
  const long long* targets;
  const float *g, *gh;
  const int* keep_ids;
  const float* keep_q;
  void* dx;
  long long ld, rows, V, ignore, gs, ghs;
  int dt, K;
  float inv_t;
};

extern "C" {
int kfac_ln_forward(const KfacLnFwd* args, ihipStream_t* stream);
int kfac_ln_backward(const KfacLnBwd* args, ihipStream_t* stream);
long long kfac_ln_ws_floats(long long rows, long long D, int sdt);
int kfac_vocab_forward(const KfacVocabFwd* args, ihipStream_t* stream);
int kfac_vocab_backward(const KfacVocabBwd* args, ihipStream_t* stream);
long long kfac_vocab_ws_bytes(int dt, long long rows, long long V, int k);
}
