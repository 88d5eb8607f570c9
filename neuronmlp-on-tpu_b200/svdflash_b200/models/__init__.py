"""Model hooks: the SVD / dense LLaMA MLP modules, the MLP-only block stack, the
decoder layers with attention over a paged cache, and the safetensors
checkpoint loader (hf_svd)."""
from . import hf_svd  # noqa: F401
from .decoder import DecoderLayer, PagedDecoder  # noqa: F401
from .svd_mlp import DenseLlamaMLP, MlpBlockStack, SvdLlamaMLP, SvdMlpBlock  # noqa: F401
