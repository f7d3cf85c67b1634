"""K-FAC-friendly modules (reference: kfac/modules/__init__.py) and the
Transformer LM's layer norm."""
from .lstm import LSTMCellBase, LSTMCellKFAC, LSTMCell, LSTMLayer, LSTM
from .layer_norm import LayerNorm

__all__ = ['LSTMCellBase', 'LSTMCellKFAC', 'LSTMCell', 'LSTMLayer', 'LSTM', 'LayerNorm']
