"""Dense attention backends (h3b tcgen05 kernel; FA4 selectable) and block-sparse attention."""

from .dense_fa4 import DenseFA4MiniMaxH3Processor, install_dense_fa4
from .sparse import install_sparse_attention, remove_sparse_attention

__all__ = ["DenseFA4MiniMaxH3Processor", "install_dense_fa4", "install_sparse_attention", "remove_sparse_attention"]
