"""kquant_amd: MI355X-native block-scaled quantization hot path of kquant.

Drop-in modules mirroring kquant's API:
  kquant_amd.io.mxfp4         <- kquant/io/mxfp4.py
  kquant_amd.mxfp8            <- kquant/mxfp8.py
  kquant_amd.mxfp4            MXFP4 quantizer (absent from kquant)
  kquant_amd.constants        <- kquant/constants.py (format block)
  kquant_amd.grouped          products grouped by expert, with gradients (absent from kquant)
  kquant_amd.loss             cross entropy of a vocabulary head, with gradients (absent from kquant)
  kquant_amd.int8             rows in 8-bit integers for linear and grouped (absent from kquant)
  kquant_amd.sampling         the next token from a head's logits (absent from kquant)

Every compute call runs a HIP kernel of libkquant_amd.so (C ABI in
include/kquant_amd.h) on the GPU.
"""

from . import constants  # noqa: F401

__all__ = ["constants"]
