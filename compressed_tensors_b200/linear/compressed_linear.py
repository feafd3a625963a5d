"""A Linear that holds its weight compressed and decompresses it on the GPU at its first forward
(linear/compressed_linear.py:33-109 of the reference: same construction through `from_linear`, same parameter
names, same status transitions COMPRESSED -> FROZEN)."""
import warnings
from typing import Dict, Optional, Tuple

import torch
from torch import Tensor
from torch.nn import Parameter
from torch.nn.functional import linear
from torch.nn.modules import Linear

from .. import torch_ops as ops
from ..compressors.base import BaseCompressor
from ..quantization.lifecycle.initialize import initialize_module_for_quantization
from ..quantization.quant_config import QuantizationStatus
from ..quantization.quant_scheme import QuantizationScheme

__all__ = ["CompressedLinear"]


class CompressedLinear(Linear):
    keep_packed = False
    # Above this a decompression and one library product take less than the packed product, which reads the weight again for every 32
    # tokens (14336 x 4096: 19 us for 16 tokens, 36 for 32, twice that for 33, against 43 to 44 for dequantize and product).
    packed_tokens = 32

    def __init__(self, *args, **kwargs) -> None:
        super().__init__(*args, **kwargs)
        warnings.warn("CompressedLinear should not be initialized directly. Use the from_linear method instead.", UserWarning)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, module: Linear, quantization_scheme: QuantizationScheme, quantization_format: str, keep_packed: bool = False):
        """Turn `module` into a CompressedLinear in place: register the scheme's scales / zero points and the
        format's compressed parameters (empty, to be filled by a checkpoint load) and drop the dense weight.
        With `keep_packed` the weight stays compressed: few tokens are multiplied by the packed 4-bit codes themselves, more of them
        by a dense weight that lives for the one call."""
        module.__class__ = CompressedLinear
        module.keep_packed = bool(keep_packed)
        module.compressor = BaseCompressor.load_from_registry(quantization_format)
        device = module.weight.device
        initialize_module_for_quantization(module, quantization_scheme, force_zero_point=False)
        info: Dict[str, Tuple] = module.compressor.compression_param_info(module.weight.shape, quantization_scheme.weights)
        delattr(module, "weight")
        for name, (shape, dtype) in info.items():
            module.register_parameter(name, Parameter(torch.empty(shape, device=device, dtype=dtype), requires_grad=False))
        module.quantization_status = QuantizationStatus.COMPRESSED
        return module

    def packed_product(self, input: Tensor) -> Optional[Tensor]:
        """input @ weight.T + bias on the packed codes, or None where the product does not take the call: more than
        `packed_tokens` tokens, a wanted gradient, anything but float16 / bfloat16 on a GPU and 4-bit codes in groups or channels."""
        args = self.quantization_scheme.weights
        if (input.dtype not in (torch.bfloat16, torch.float16) or not input.is_cuda or input.numel() == 0
                or input.numel() > self.packed_tokens * input.shape[-1] or args.num_bits != 4 or getattr(self, "weight_g_idx", None) is not None
                or (self.bias is not None and self.bias.dtype is not input.dtype)
                or (torch.is_grad_enabled() and (input.requires_grad or (self.bias is not None and self.bias.requires_grad)))):
            return None
        scale, packed = self.weight_scale, getattr(self, "weight_packed", None)
        fp4 = packed is not None and packed.dtype is torch.uint8
        if packed is None or (fp4 and (scale.dtype is not torch.float8_e4m3fn or getattr(self, "weight_global_scale", None) is None)):
            return None
        rows, groups = self.out_features, scale.numel() // self.out_features
        if groups < 1 or groups * rows != scale.numel() or self.in_features % groups:
            return None
        zero_point, global_scale, codec, qtype = getattr(self, "weight_zero_point", None), None, "pack32", ops.QINT
        if fp4:
            zero_point, global_scale, codec, qtype = None, self.weight_global_scale, "fp4x2", ops.QFLOAT
        elif zero_point is not None and zero_point.dtype is torch.int32:
            zero_point = ops.unpack_int32(zero_point, 4, (rows, groups), packed_dim=0).contiguous()
        return ops.dequantize_linear(input, packed, scale, zero_point, qtype=qtype, col_group=self.in_features // groups, scale_row_stride=groups,
                                     codec=codec, global_scale=global_scale, bias=self.bias)

    def forward(self, input: Tensor) -> Tensor:
        """Decompress once (unpack + dequantize kernels), keep the dense weight, then the ordinary linear; or, with
        `keep_packed`, the product with the packed codes."""
        if self.keep_packed and self.quantization_status == QuantizationStatus.COMPRESSED:
            out = self.packed_product(input)
            return out if out is not None else linear(input, self.compressor.decompress_module(self), self.bias)
        if self.quantization_status == QuantizationStatus.COMPRESSED:
            self.register_parameter("weight", Parameter(self.compressor.decompress_module(self), requires_grad=False))
            self.quantization_status = QuantizationStatus.FROZEN
        return linear(input, self.weight, self.bias)
