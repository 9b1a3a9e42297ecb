"""Newton-Schulz orthogonalisation front door.

Same public surface as the reference's ``muon_fused/ns_step.py``:
``fused_newton_schulz(G, steps=5, workspace=None)`` (ns_step.py:85-123) and
``workspace_size(m, n)`` (ns_step.py:61-79).  Differences by design:

* CUDA only.  The reference silently falls back to a PyTorch loop on CPU
  tensors, on a missing extension and on *any* runtime error
  (ns_step.py:111-123); here a CPU tensor or a failing kernel raises.
* ``workspace_size`` returns bytes (the reference's C++ value,
  torch_binding.cu:16-18).  Callers that allocate that many bf16 elements, as
  the reference's optimizer does (optimizer.py:90-92), simply over-allocate.
"""

from __future__ import annotations

import torch

from muon_fused import _fused_muon_C as _C

# Newton-Schulz quintic coefficients (reference ns_step.py:39).
NS_COEFFS = (3.4445, -4.7750, 2.0315)


def workspace_size(m: int, n: int) -> int:
    """Bytes of device workspace needed for an (m, n) gradient matrix."""
    return _C.workspace_size(m, n)


def fused_newton_schulz(
    G: torch.Tensor,
    steps: int = 5,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Approximate orthogonal factor of ``G`` by ``steps`` quintic
    Newton-Schulz iterations; returns bf16 with ``G``'s shape.

    Args:
        G: 2-D CUDA tensor of any floating dtype (cast to bf16 internally).
        steps: number of iterations (default 5).
        workspace: optional pre-allocated CUDA buffer of at least
            ``workspace_size(*G.shape)`` bytes; reused across calls.
    """
    assert G.ndim == 2, f"Expected 2-D tensor, got {G.ndim}-D"
    if not G.is_cuda:
        raise RuntimeError(
            "fused_newton_schulz needs a CUDA tensor; this build has no CPU fallback")
    return _C.fused_newton_schulz(G, steps, workspace)


def _check_heads(shape, heads: int, dim: int) -> int:
    """Width of a head; raises where the projection does not divide into heads."""
    if dim not in (0, 1):
        raise RuntimeError(f"dim must be 0 (heads are rows) or 1 (columns), got {dim}")
    side = int(shape[-2 + dim])
    if heads < 1 or side % heads:
        raise RuntimeError(f"{side} {'columns' if dim else 'rows'} do not divide into {heads} heads")
    return side // heads


def _heads_form(d: int, n: int, steps: int) -> str:
    """How heads of width d and long side n run: "gram" on d x d matrices, "across" on
    n x n ones where n is the shorter side, "batch" through the batched bf16 path.

    The Gram forms hold matrices of at most 128 on chip.  Rounding that leaks into what
    a head does not span grows by 3.4445^2 a step in A: after five steps a head of rank 1
    is off by 0.7 %, after eight by anything.  A head has full rank on its shorter side."""
    if d > 128 or steps > 5:
        return "batch"
    return "across" if n < d else "gram"


def workspace_size_heads(shape, heads: int, *, dim: int = 0, steps: int = 5) -> int:
    """Bytes of device workspace ``fused_newton_schulz_heads`` needs for a
    (rows, cols) or (batch, rows, cols) projection."""
    d = _check_heads(shape, heads, dim)
    batch = int(shape[0]) if len(shape) == 3 else 1
    rows, cols = int(shape[-2]), int(shape[-1])
    n = cols if dim == 0 else rows
    form = _heads_form(d, n, steps)
    if form == "gram":
        return _C.workspace_size_heads(batch, rows, cols, heads, dim)
    if form == "across":
        block = (d, n) if dim == 0 else (n, d)
        return _C.workspace_size_heads(batch * heads, *block, 1, 1 - dim)
    return _C.workspace_size_batched(batch * heads, d, n)


def fused_newton_schulz_heads(
    G: torch.Tensor,
    heads: int,
    steps: int = 5,
    workspace: torch.Tensor | None = None,
    *,
    dim: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Newton-Schulz of every attention head of a projection by itself.

    A head is a block of ``rows / heads`` rows (``dim=0``: query, key and value
    projections, one matrix or fused) or of ``cols / heads`` columns (``dim=1``:
    output projection); each is normalised by its own Frobenius norm and
    orthogonalised as ``fused_newton_schulz`` does a matrix.  Returns bf16 with
    ``G``'s shape.

    Heads up to 128 wide iterate, for up to 5 steps, on head x head matrices
    (long side x long side where that is shorter) in split fp16: the result is
    the exact one up to its bf16 rounding, on ill-conditioned heads too; the
    error of heads whose long side has rank 1 to 4 only is 0.7 to 0.25 % after
    five steps.  Wider heads, and more steps, run as a batch of matrices on the
    bf16 path of ``fused_newton_schulz``, with its error.  Both that route and the
    one for heads wider than long copy G (unless the heads lie in it as a batch) and
    the result with torch, beside the workspace.

    Args:
        G: CUDA tensor (rows, cols), or (batch, rows, cols) for same-shape
            projections, of any floating dtype.  fp32 and fp64 are rounded to
            bf16 first, as in ``fused_newton_schulz``; bf16 and, off the
            batched path, fp16 are taken as they are.
        heads: heads per projection.
        steps: number of iterations (default 5).
        workspace: optional pre-allocated CUDA buffer of at least
            ``workspace_size_heads(G.shape, heads, dim=dim, steps=steps)`` bytes.
        dim: 0 where heads are blocks of rows, 1 where of columns.
        out: optional contiguous bf16 tensor of ``G``'s shape for the result;
            must not share memory with ``G``.
    """
    assert G.ndim in (2, 3), f"Expected a 2-D or 3-D tensor, got {G.ndim}-D"
    if not G.is_cuda:
        raise RuntimeError(
            "fused_newton_schulz_heads needs a CUDA tensor; this build has no CPU fallback")
    d = _check_heads(G.shape, heads, dim)
    form = _heads_form(d, G.shape[-1 - dim], steps)
    if form == "gram":
        return _C.newton_schulz_heads(G, heads, steps, dim, workspace, out)
    if out is not None and (out.shape != G.shape or out.dtype != torch.bfloat16
                            or not out.is_contiguous() or out.is_neg()
                            or out.device != G.device):
        raise RuntimeError("out must be a contiguous bf16 tensor shaped like G on its device")
    if G.numel() == 0:
        return torch.empty(G.shape, dtype=torch.bfloat16, device=G.device) if out is None else out
    blocks = G.unflatten(G.ndim - 2 + dim, (heads, d))
    if dim == 1:
        blocks = blocks.movedim(-2, -3)  # heads before rows
    each = blocks.reshape(-1, *blocks.shape[-2:])
    if form == "across":
        res = _C.newton_schulz_heads(each, 1, steps, 1 - dim, workspace)
    else:
        res = _C.fused_newton_schulz_batched(each, steps, workspace)
    res = res.view(blocks.shape)
    if dim == 1:
        res = res.movedim(-3, -2)
    res = res.reshape(G.shape)
    return res if out is None else out.copy_(res)
