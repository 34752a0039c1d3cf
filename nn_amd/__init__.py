"""nn_amd — MI355X (gfx950) quantized-linear hot path for alabsystems/nn.

Hand-written HIP kernels behind a C ABI (``include/nnq.h``, ``libnnq.so``) for
the dequant-fused matmul over GGUF Q8_0 / Q4_K / Q6_K blocks and the GPT-OSS
MXFP4 mixture-of-experts layer (GPT-OSS and nn-core OCP MXFP4 layouts); ``nn_amd.quantized`` mirrors the reference's
operator surface in Python.  Beside it: 4-bit group-scaled and MXFP4 linears, token log probabilities, beam search.
"""
from .quantized import (  # noqa: F401
    BeamSelection, BiasMismatch, DataLengthMismatch, InvalidShape, Layout, Mxfp4Rows, NonFiniteData, NotQuantized, QuantizedMatmulError,
    QuantizedMLP, QuantizedMoE, QuantizedWeight, QuantType, RankMismatch, ShapeMismatch, TensorError, TokenLogprobs,
    Unsupported, WeightRank,
    WrongQuantType, argmax, beam_reorder, beam_select, dequantize_mxfp4_ocp, device_count, init, linear_argmax, linear_logprobs, linear_sample,
    mxfp4_linear, quantize_mxfp4_rows, sample_token, token_logprobs,
    quantize_mxfp4, quantize_mxfp4_ocp, quantize_q4_k, quantize_q6_k, quantize_q8_0, quantized_linear, quantized_matmul_q4_k, quantized_matmul_q6_k, quantized_matmul_q8_0,
    synth_normal)
