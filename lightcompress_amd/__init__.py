"""lightcompress_amd — MI355X (gfx950) kernels behind the LightCompress (`llmc`)
layer-wise quantization API: quantizer primitives, RTN partials, int4 packing, GPTQ and AWQ, and
what runs and judges the w8a8 result: ``w8a8`` (products, norms), ``logprobs``; microscaled 4-bit
numbers and their products: ``mxfp4``, and layers of experts kept in them: ``moe``.

The package is a thin Python mirror of the reference's class API over a C-ABI
shared library (``liblcq.so``, declared in ``include/lcq.h``) of hand-written
HIP kernels.  Build it with ``python -m lightcompress_amd.build``.
"""
from .quant import FloatQuantizer, IntegerQuantizer, Weight48IntegerQuantizer  # noqa: F401
