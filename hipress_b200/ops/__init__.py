"""Compression operators: algorithm table and tensor-level encode/decode."""
from .algorithms import AlgSpec, algorithm_names, get_algorithm  # noqa: F401
from .compressor import Compressor, PayloadError, sparse_pairs  # noqa: F401
from .custom import CustomCompressor, register_algorithm, unregister_algorithm  # noqa: F401
from .layers import attention, layer_norm, linear, self_attention  # noqa: F401
from .losses import TokenLogProbs, cross_entropy, token_log_probs  # noqa: F401
from .random_drop import dropout  # noqa: F401
