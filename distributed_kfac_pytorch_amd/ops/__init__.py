"""gfx950 HIP kernels (csrc/) bound through ctypes, plus their CPU twins.

_lib       library loader (fails loudly on GPU tensors when not built)
factors    implicit-im2col MFMA SYRK + fused EMA (K1-K5)
eigen      batched Jacobi eigensolver (K6) / Cholesky inverse (K9)
precond    eigenbasis preconditioning, grouped KL-dot + apply (K7, K8, K10, K11)
comm_pack  triu pack/unpack for the factor all-reduce arena (K12)
bn         fused BatchNorm (+ add) (+ ReLU) of the image models
ln         layer norm (+ residual add) of the Transformer LM
vocab      log probabilities, entropy, top alternatives and top-logit distillation
           behind the language models' vocabulary head
"""
from . import _lib, factors, eigen, precond, comm_pack, bn, ln, vocab

__all__ = ['_lib', 'factors', 'eigen', 'precond', 'comm_pack', 'bn', 'ln', 'vocab',
           'native_available']


def native_available():
    return _lib.available()
