"""``PackedFP4Linear``: a linear whose weight exists in packed form only, for a few rows of activations.

What becomes of a ``UE5M3Linear`` whose weight scale the post-load lifecycle has frozen when a model
answers token by token.  The weight's values are those of the frozen layer; its activations, unlike
that layer's, are not quantized.
"""

from __future__ import annotations

import torch
from torch import Tensor

from ue5m3_fp4.nn.convert import ConversionRecord
from ue5m3_fp4.nn.linear import UE5M3Linear
from ue5m3_fp4.packed import PackedFP4Tensor


class PackedFP4Linear(torch.nn.Module):
    """``x @ W.T + bias`` with a packed weight; no gradients.  Reads 0.5 byte per weight element and
    one byte per block, once for every 64 rows of bf16 ``x`` and every 32 of fp32: made for the tokens of a decoding
    step.  Whole prompts are right too, but read and decode the weight that often; where they
    dominate, the frozen ``UE5M3Linear`` (whose GEMM quantizes its activations) is the faster form."""

    def __init__(self, weight: PackedFP4Tensor, bias: Tensor | None = None) -> None:
        super().__init__()
        if not isinstance(weight, PackedFP4Tensor):
            raise TypeError("weight must be a PackedFP4Tensor")
        if bias is not None and tuple(bias.shape) != (weight.rows,):
            raise ValueError("bias must have one element per weight row")
        self.in_features, self.out_features = weight.cols, weight.rows
        self.block_size, self.blocking = weight.block_size, weight.blocking
        self.tensor_amax, self.scale_target, self.module_name = weight.tensor_amax, weight.scale_target, weight.name
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.detach())

    @classmethod
    def from_frozen(cls, module: UE5M3Linear) -> PackedFP4Linear:
        """The packed form of a linear whose weight amax is frozen (``UE5M3Linear.packed_weight``): of the weight
        that ``load_packed_weight`` has installed, if it has."""

        if not isinstance(module, UE5M3Linear):
            raise TypeError("from_frozen expects a UE5M3Linear")
        return cls(module.packed_weight(), module.bias)

    def get_extra_state(self) -> Tensor:
        """The tensor scale: codes and block scales mean nothing without it."""

        return torch.tensor([self.tensor_amax, self.scale_target], dtype=torch.float64)

    def set_extra_state(self, state: Tensor) -> None:
        if not isinstance(state, Tensor) or tuple(state.shape) != (2,):
            raise ValueError("the state of a packed linear holds its tensor amax and its scale target")
        self.tensor_amax, self.scale_target = (float(value) for value in state.tolist())

    def forward(self, inputs: Tensor) -> Tensor:
        from ue5m3_fp4.serving import packed_matvec

        if inputs.shape[-1] != self.in_features:
            raise ValueError(f"Expected input width {self.in_features}, got {inputs.shape[-1]}")
        return packed_matvec(inputs, self.codes, self.scales, rows=self.out_features, cols=self.in_features,
                             block_size=self.block_size, two_dimensional=self.blocking == "2d",
                             tensor_amax=self.tensor_amax, scale_target=self.scale_target, bias=self.bias)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"block_size={self.block_size}, blocking={self.blocking}")


def pack_frozen_linears(model: torch.nn.Module) -> tuple[ConversionRecord, ...]:
    """Replace every child ``UE5M3Linear`` of a model whose weights the post-load lifecycle has frozen by
    its :class:`PackedFP4Linear`, in place; the full-precision weights are then no longer part of the
    model.  Raises before any change when a weight is not frozen."""

    if not isinstance(model, torch.nn.Module):
        raise TypeError("model must be a torch.nn.Module")
    if isinstance(model, UE5M3Linear):
        raise ValueError("pack_frozen_linears cannot replace the model root")
    found = [(name, module) for name, module in model.named_modules(remove_duplicate=False)
             if isinstance(module, UE5M3Linear)]
    packed = {id(module): PackedFP4Linear.from_frozen(module) for _, module in found}
    records = []
    for name, module in found:
        parent_name, _, child = name.rpartition(".")
        setattr(model.get_submodule(parent_name) if parent_name else model, child, packed[id(module)])
        records.append(ConversionRecord(name, module.in_features, module.out_features, module.bias is not None))
    return tuple(records)


__all__ = ["PackedFP4Linear", "pack_frozen_linears"]
