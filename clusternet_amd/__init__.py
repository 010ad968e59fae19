"""clusternet_amd: MI355X (gfx950) implementation of clusterNet's matrix-multiply and 8-bit codec
path.  The product is the C-ABI library libcnhip.so (see include/cnhip.h) and the C++
ClusterNet / Matrix facade over it; this package is the thin Python host binding used by the
tests and the benchmark.  PyTorch appears only as the owner of device memory and streams.
"""
from ._lib import (CnError, absmax, absmax_compression_8bit, compression_8bit, compression_8bit_axpy, decompression_8bit, decompression_8bit_axpy, dequantize_4bit, dot, dotT,
                   embedding, embedding_grad, Tdot, gemm, gemm_w4, gemm_w8, init, lib, lib_path,
                   muon_update, num_compute_units, orthogonalize, quantize_4bit, rmsprop_update, table, W4)

__all__ = ["CnError", "absmax", "absmax_compression_8bit", "compression_8bit", "compression_8bit_axpy", "decompression_8bit", "decompression_8bit_axpy", "dequantize_4bit", "dot",
           "dotT", "embedding", "embedding_grad", "Tdot", "gemm", "gemm_w4", "gemm_w8", "init", "lib", "lib_path", "muon_update", "num_compute_units",
           "orthogonalize", "quantize_4bit", "rmsprop_update",
           "table", "W4"]
