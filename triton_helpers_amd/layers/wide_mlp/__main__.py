"""``python -m triton_helpers.layers.wide_mlp benchmark|profile ...``, in the manner of the other layers' command lines.

Dimensions: ``x (L, D)`` and its residual through a block with ``H`` hidden channels.  Providers: torch's own operators (``baseline``), the
block that trains with 8-bit checkpoints (``checkpointed``), and the block in 8 bits (``int8``, which has no backward: name the other two for
the modes ``bwd`` and ``fwd-bwd``).
"""
import torch
import torch.nn.functional as F

from ...benchmark import Workload, run_cli
from .module import WideMLP


def _inputs(L, D, H, device="cuda", dtype=torch.float16, requires_grad=False):
    block = WideMLP(D, H).to(device=device, dtype=dtype).requires_grad_(requires_grad)

    def rows():
        return torch.randn(L, D, device=device).to(dtype).requires_grad_(requires_grad)

    return {"block": block, "x": rows(), "residual": rows()}


def _int8_inputs(L, D, H, device="cuda", dtype=torch.float16, requires_grad=False):
    if requires_grad:
        raise ValueError("the int8 block has no backward: use -p baseline checkpointed")
    inputs = _inputs(L, D, H, device, dtype)
    return {**inputs, "block": inputs["block"].to_int8(dtype)}


def _baseline(block, x, residual):
    stream = x + residual
    y = F.rms_norm(stream, stream.shape[-1:], block.norm.weight, block.norm.eps)
    return F.linear(F.gelu(F.linear(y, block.up.weight, block.up.bias)), block.down.weight, block.down.bias) + stream


def _block(block, x, residual):
    out, stream = block(x, residual)
    return out + stream


def main(argv=None):
    return run_cli(
        "Wide-MLP",
        [Workload("baseline", _inputs, _baseline), Workload("checkpointed", _inputs, _block), Workload("int8", _int8_inputs, _block)],
        dims={"L": ((512, 2048, 8192), "values"), "D": (1024, "values"), "H": (4096, "values")},
        argv=argv,
    )


if __name__ == "__main__":
    main()
