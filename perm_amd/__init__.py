"""perm_amd -- MI355X-native encoder hot path of coldpress (asystemoffields/PERM).

Drop-in GPU backend for the reference's encode stage: the same Python API as
``coldpress.kquant`` (QUANTIZE / DEQUANTIZE / roundtrip), ``coldpress.ef``
(cholesky_inv_upper, ef_encode) and the Hessian hook of ``coldpress.hessians``,
executed by hand-written gfx950 HIP kernels in ``libcoldpress_hip.so`` through a
C ABI (include/coldpress_hip.h). PyTorch provides device memory and streams.

``mxfp4`` and ``kvcache`` (no counterpart in the reference) are operators for answering
with a model in low bits: MXFP4 weights and activations and their product, and attention
over a paged 8-bit key / value cache. ``kvpages`` hands that cache's pages out, several answers
to a prompt sharing them, and ``sampling`` draws the next tokens.

There is no CPU fallback: every entry point raises if the HIP library is not
built or no GPU is visible.
"""
__version__ = "0.1.0"
