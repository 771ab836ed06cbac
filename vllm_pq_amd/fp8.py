"""Block-scaled 8-bit floating point linears beside the product-quantised ones.

A PQ checkpoint may hold some of its modules (those that product quantisation hurts most) as e4m3 values with one fp32 scale per
128 x 128 block instead; PQConfig's `fp8_modules` names them and get_quant_method hands out this method for them:

    weight            [N, K]                            float8_e4m3fn
    weight_scale_inv  [ceil(N / 128), ceil(K / 128)]    fp32, the factor a stored value is multiplied by

Activations are quantised per token and group of 128 features when the layer runs (ops.fp8_block_linear), or arrive in that form from
the step in front of the layer (apply_after_norm, apply_after_silu_and_mul).
"""
import re
from typing import Dict, List, Optional, Set, Tuple

import torch
from torch.nn.parameter import Parameter

from . import ops
from .compat import LinearMethodBase, set_weight_attrs

# the checkpoint's names of what a fused layer stacks (the model loaders' stacked-parameter mapping)
_FUSED = {"qkv_proj": ("q_proj", "k_proj", "v_proj"), "gate_up_proj": ("gate_proj", "up_proj")}


def is_fp8_module(prefix: str, patterns: List[str]) -> bool:
    """Whether the module `prefix` is named by one of the regular expressions: searched in the checkpoint's names of what it
    stacks (all of them or none), else in its own name."""
    head, _, last = prefix.rpartition(".")
    names = [f"{head}.{n}" if head else n for n in _FUSED.get(last, ())]
    found = [n for n in names if any(re.search(p, n) for p in patterns)]
    if found and found != names:
        raise ValueError(f"fp8_modules names only a part of what {prefix} stacks: {', '.join(found)}")
    return bool(found) or any(re.search(p, prefix) for p in patterns)


def checkpoint_fp8_modules(modules: Dict[str, int], patterns: List[str]) -> Set[str]:
    """Those of a checkpoint's modules (name: out_features) that become e4m3 layers under `patterns`: a module goes by the layer
    that stacks it where the checkpoint holds all that this layer stacks, else by its own name, and either by is_fp8_module, as a
    model that loads the checkpoint has it.  Refused: an expression that names none of them, and a stacked matrix whose rows do
    not fill its scale blocks, which create_weights would not take."""
    found, used = set(), set()
    for m, rows in modules.items():
        head, _, last = m.rpartition(".")
        layer = m
        for fused, parts in _FUSED.items():
            if last in parts and all((f"{head}.{n}" if head else n) in modules for n in parts):
                layer = f"{head}.{fused}" if head else fused
        if is_fp8_module(layer, patterns):
            if layer != m and rows % ops.FP8_GROUP:
                raise ValueError(f"{m}: {rows} output features are not a multiple of the scale block ({ops.FP8_GROUP}), which a part "
                                 f"of {layer} has to be in e4m3")
            found.add(m)
            used.update(p for p in patterns if re.search(p, m) or re.search(p, layer))
    for p in patterns:
        if p not in used:
            raise ValueError(f"fp8_modules: {p!r} names none of the modules that are quantised")
    return found


def fp8_quantize_weight(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Dense [N, K] -> (weight, weight_scale_inv): every 128 x 128 block divided by its largest magnitude / 448."""
    if weight.dim() != 2:
        raise ValueError(f"weight must be [out_features, in_features], got {tuple(weight.shape)}")
    G = ops.FP8_GROUP
    N, K = weight.shape
    w = torch.nn.functional.pad(weight.detach().to(torch.float32), (0, -K % G, 0, -N % G))
    b = w.view(w.shape[0] // G, G, w.shape[1] // G, G)
    scale = b.abs().amax((1, 3)).clamp_min(2.0 ** -96) / 448.0
    q = (b / scale[:, None, :, None]).to(ops.FP8_DTYPE).view(w.shape)
    return q.view(torch.uint8)[:N, :K].contiguous().view(ops.FP8_DTYPE), scale


def fp8_reconstruct(weight: torch.Tensor, weight_scale_inv: torch.Tensor) -> torch.Tensor:
    """fp32 dense weight (plain torch; for error reports and tests)."""
    G = ops.FP8_GROUP
    N, K = weight.shape
    s = weight_scale_inv.repeat_interleave(G, 0)[:N].repeat_interleave(G, 1)[:, :K]
    return weight.to(torch.float32) * s


class BlockFP8LinearMethod(LinearMethodBase):
    """Linear method of the modules held in e4m3."""

    def __init__(self, quant_config):
        self.quant_config = quant_config

    def create_weights(self, layer: torch.nn.Module, input_size_per_partition: int,
                       output_partition_sizes: List[int], input_size: int, output_size: int,
                       params_dtype: torch.dtype, **extra_weight_attrs):
        G = ops.FP8_GROUP
        if params_dtype not in (torch.half, torch.bfloat16):
            raise ValueError("Only half and bfloat16 are currently supported by pq")
        # a scale block must not straddle two ranks or two matrices of a fused layer
        if input_size_per_partition != input_size and input_size_per_partition % G:
            raise ValueError(f"The input size per rank, {input_size_per_partition}, is not a multiple of the scale block ({G}). "
                             "This can be caused by too large tensor parallel size.")
        n_out = sum(output_partition_sizes)
        if (len(output_partition_sizes) > 1 or n_out != output_size) and any(s % G for s in output_partition_sizes):
            raise ValueError(f"The output sizes {output_partition_sizes} are not multiples of the scale block ({G}). "
                             "This can be caused by too large tensor parallel size.")
        weight = Parameter(torch.empty(n_out, input_size_per_partition, dtype=ops.FP8_DTYPE), requires_grad=False)
        set_weight_attrs(weight, {"input_dim": 1, "output_dim": 0})
        scale = Parameter(torch.empty((n_out + G - 1) // G, (input_size_per_partition + G - 1) // G, dtype=torch.float32),
                          requires_grad=False)
        set_weight_attrs(scale, {"input_dim": 1, "output_dim": 0, "packed_dim": 0, "pack_factor": G})
        for name, p in (("weight", weight), ("weight_scale_inv", scale)):
            layer.register_parameter(name, p)
            set_weight_attrs(p, extra_weight_attrs)

    def process_weights_after_loading(self, layer: torch.nn.Module) -> None:
        for p in (layer.weight, layer.weight_scale_inv):
            if not p.data.is_contiguous():
                p.data = p.data.contiguous()

    def apply(self, layer: torch.nn.Module, x: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        return ops.fp8_block_linear(x, layer.weight, layer.weight_scale_inv, bias)

    def apply_after_norm(self, layer: torch.nn.Module, x: torch.Tensor, residual: Optional[torch.Tensor],
                         norm_weight: torch.Tensor, eps: float, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """`self.apply(layer, RMSNorm(x, residual))` with the norm writing the layer's 8-bit input: `residual` (where there
        is one) becomes x + residual in place, x keeps its values."""
        if residual is None:
            q, s = ops.rms_norm_fp8(x, norm_weight, eps)
        else:
            q, s = ops.fused_add_rms_norm_fp8(x, residual, norm_weight, eps)
        return ops.fp8_block_gemm(q, s, layer.weight, layer.weight_scale_inv, bias, x.dtype)

    def apply_after_silu_and_mul(self, layer: torch.nn.Module, gate_up: torch.Tensor,
                                 bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """`self.apply(layer, SiluAndMul()(gate_up))` with the activation writing the layer's 8-bit input."""
        q, s = ops.silu_and_mul_fp8(gate_up)
        return ops.fp8_block_gemm(q, s, layer.weight, layer.weight_scale_inv, bias, gate_up.dtype)

    def apply_silu_and_mul(self, layer: torch.nn.Module, x: torch.Tensor,
                           bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """`SiluAndMul()(self.apply(layer, x, bias))` for a gate/up layer, as PQLinearMethod has it."""
        y = self.apply(layer, x, bias)
        out = torch.empty(y.shape[:-1] + (y.shape[-1] // 2,), dtype=y.dtype, device=y.device)
        ops.silu_and_mul(out, y)
        return out
