"""B200-native (sm_100a) activation-sparse FFN hot path with the reference's API.

Reference: Maccy-Z/autoresearch2 (old/lib_sparse/sparse.py, old/sparse_pack.py,
old/sparse_unpack.py, old/full_matmul/sparse_pack.py).  All compute runs in
libsparseffn.so (hand-written CUDA for sm_100a behind a C ABI,
include/sparseffn.h); there is no CPU or fallback path.  The operations are also
registered as torch.library ops (sparseffn::*, library.py) for torch.compile.
Beside the FFN: token_logprobs and distill_topk (logits.py) on the output
distribution, residual_norm (norms.py) around the blocks, gated_ffn (glu.py),
and activations and products in 8 bits (fp8.py).
"""
from .bitsparse import (BitsparseTensor, TensorBuffer, bitsparse_pack, bitsparse_pack_async, bitsparse_unpack,
                        check_status, compress_dense, dense_to_tilesparse, get_globals, grad_relu2_,
                        init_sparse_buffer, mask_with_bitmask_, reconstruct_bitmask, reset_sparse_globals,
                        spAx, tile_unpack)
from .ffn import (FFNSparse, FFNSpRelu2, backward_mode, compact_k, set_backward, set_compact_k,
                  set_sparse_mma, sparse_mma)
from .fp8 import Fp8Tensor, ckpt_linear, fp8_matmul, fp8_pack, fp8_unpack
from .glu import gated_ffn
from .logits import TokenLogprobs, distill_topk, token_logprobs
from .norms import residual_norm
from . import (bitshift, deep, ffn, fp8, glu, gpt, library, logits, norms, parallel, sp24,  # library registers the
               tiled)  # sparseffn:: ops

__all__ = [
    "BitsparseTensor", "TensorBuffer", "bitsparse_pack", "bitsparse_pack_async", "bitsparse_unpack", "check_status",
    "compress_dense", "reconstruct_bitmask",
    "dense_to_tilesparse", "get_globals", "grad_relu2_", "init_sparse_buffer",
    "mask_with_bitmask_", "reset_sparse_globals", "spAx", "tile_unpack", "FFNSparse",
    "FFNSpRelu2", "set_sparse_mma", "sparse_mma", "set_compact_k", "compact_k", "set_backward", "backward_mode",
    "TokenLogprobs", "token_logprobs", "distill_topk", "residual_norm",
    "Fp8Tensor", "fp8_pack", "fp8_unpack", "fp8_matmul", "ckpt_linear", "gated_ffn",
    "bitshift", "deep", "fp8", "glu", "gpt", "library", "logits", "norms", "parallel", "sp24", "tiled",
]
