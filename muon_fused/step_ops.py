"""Operators of the optimizer step around Newton-Schulz.

``fused_adamw``          AdamW over a list of tensors in one launch;
``fused_normed_update``  weight decay + neuron-wise normalised update of
                         same-shape matrices.

Both update their tensors in place on torch's current CUDA stream, never
synchronise the host and raise ``RuntimeError`` on bad input.  They work on the
tensors' values outside autograd (as an optimizer step under ``no_grad``) and
bump the version counters of what they write, so a backward pass through values
saved before the call fails instead of using the new ones.
"""

from __future__ import annotations

import ctypes
import functools
import math
import operator
import warnings
from collections.abc import Iterable, Sequence

import torch
from torch.autograd.graph import increment_version

from muon_fused import _lib
from muon_fused._fused_muon_C import _check_cuda, _on_device, _stream, workspace_for

STEP_DTYPES = {torch.float32: _lib.FM_DT_F32, torch.bfloat16: _lib.FM_DT_BF16,
               torch.float16: _lib.FM_DT_F16}


class UnfitTensors(_lib.FusedMuonError):
    """Tensors that torch's ops take and the kernel does not: they share memory or are
    negative views.  Nothing was written."""


_DTYPE = operator.attrgetter("dtype")


def _check_list(tensors, name: str, count: int | None = None) -> list[torch.Tensor]:
    if isinstance(tensors, torch.Tensor) or not isinstance(tensors, Iterable):
        raise RuntimeError(f"{name} must be a list of tensors")
    tensors = list(tensors)
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{name} must be a list of tensors, got {type(t).__name__} in it")
    if count is not None and len(tensors) != count:
        raise RuntimeError(f"{name} must have one tensor per parameter, got {len(tensors)} "
                           f"for {count}")
    return tensors


def _bump(tensors) -> None:
    """Tell autograd of the writes; inference tensors keep no version."""
    increment_version([t for t in tensors if not t.is_inference()])


def _overlap(written, read) -> bool:
    """Whether one of the contiguous tensors ``written`` shares memory with another tensor of
    either list (as the C entries check within a call)."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.nbytes, w) for ts, w in ((written, 1), (read, 0))
                   for t in ts if t.numel())
    end = written_end = 0  # furthest end so far, of all and of the written ones
    for lo, hi, w in spans:
        if lo < written_end or (w and lo < end):
            return True
        end = max(end, hi)
        if w:
            written_end = max(written_end, hi)
    return False


def _check_adamw(params, grads, moments1, moments2) -> list[tuple]:
    """Raise unless the kernel may work on the tensors; their types otherwise."""
    _check_cuda(params[0], "params")
    lists = (params, grads, moments1, moments2)
    if len(set().union(*(map(torch.Tensor.get_device, ts) for ts in lists))) != 1:
        raise RuntimeError("fused_adamw needs all tensors on one device")
    if not all(all(map(torch.Tensor.is_contiguous, ts)) for ts in lists):
        raise RuntimeError("fused_adamw needs contiguous tensors")
    if any(any(map(torch.Tensor.is_neg, ts)) for ts in lists):
        raise UnfitTensors("fused_adamw needs tensors that are not negative views")
    if not all(all(map(torch.Tensor.is_same_size, params, ts)) for ts in lists[1:]):
        raise RuntimeError("params, grads and moments must have the same shapes")
    types = list(zip(*(map(_DTYPE, ts) for ts in lists)))
    for pt, gt, mt, vt in set(types):
        if pt not in STEP_DTYPES or gt != pt:
            raise RuntimeError(f"params and grads must be fp32, bf16 or fp16 of one type, got "
                               f"{pt} and {gt}")
        if mt != vt or mt not in (pt, torch.float32):
            raise RuntimeError(f"moments must have the parameter's type or fp32, got {mt} and {vt}")
    return types


@functools.cache
def adamw_ready(device: int) -> bool:
    """Whether the kernels run here: an sm_100 device, and the library built.  FusedMuon's
    AdamW groups, which need nothing else of the library, use torch's ops otherwise."""
    if torch.cuda.get_device_capability(device) != (10, 0):
        return False
    try:
        _lib.step_ext()
    except (ImportError, OSError) as e:
        warnings.warn(f"AdamW groups run as torch ops: {e}", RuntimeWarning, stacklevel=2)
        return False
    return True


def adamw_launch(params, grads, moments1, moments2, alphas, lr: float, wd: float, betas,
                 eps: float) -> None:
    """One call: lists of one parameter type and one moment type; ``alphas``
    holds each tensor's -lr/scale.  Version counters stay as they are."""
    rc = _lib.step_ext().adamw(params, grads, moments1, moments2, alphas, float(1 - lr * wd),
                               1 - betas[0], 1 - betas[1], float(eps), False)
    if rc is not None:
        _check_adamw_status(rc)
        return
    _check_adamw(params, grads, moments1, moments2)
    ptr = torch.Tensor.data_ptr
    table = b"".join(map(_lib.ADAMW_TENSOR.pack, map(ptr, params), map(ptr, grads),
                         map(ptr, moments1), map(ptr, moments2),
                         map(torch.Tensor.numel, params), alphas))
    p0 = params[0]
    with _on_device(p0):
        _check_adamw_status(_lib.load().fm_adamw(
            table, len(params), STEP_DTYPES[p0.dtype], STEP_DTYPES[moments1[0].dtype],
            float(1 - lr * wd), 1 - betas[0], 1 - betas[1], float(eps), _stream(p0)))


def _check_adamw_status(rc: int) -> None:
    if rc == _lib.FM_E_INVALID and b"overlap" in _lib.load().fm_last_error():
        raise UnfitTensors("fused_adamw: tensors overlap in memory")
    _lib.check(rc, "fm_adamw")


def adamw_alpha(lr: float, betas, step: int) -> float:
    """-lr/scale, scale = (1 - b1^t)/sqrt(1 - b2^t) (reference optimizer.py:191-200)."""
    return -lr / ((1 - betas[0] ** step) / (1 - betas[1] ** step) ** 0.5)


def fused_adamw(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    moments1: Sequence[torch.Tensor],
    moments2: Sequence[torch.Tensor],
    steps: int | Sequence[int],
    *,
    lr: float,
    wd: float = 0.1,
    betas: tuple[float, float] = (0.9, 0.95),
    eps: float = 1e-8,
) -> None:
    """AdamW step of every tensor of a list, in place::

        m = lerp(m, g, 1 - b1);  v = lerp(v, g², 1 - b2)
        p = p·(1 - lr·wd) - lr·sqrt(1 - b2^t)/(1 - b1^t) · m/(eps + sqrt(v))

    Args:
        params, grads: contiguous CUDA tensors (fp32, bf16 or fp16) on one
            device; a gradient has its parameter's shape and type.
        moments1, moments2: the running moments, of the parameter's type (every
            op then rounds to it, as the optimizer's torch ops did) or fp32.
        steps: the step count t >= 1 of each tensor (after this step), or one
            for all.
        lr, wd, betas, eps: as in :class:`FusedMuon`.

    A list may mix types and sizes; tensors of zero elements are skipped.  What
    a call writes must not share memory with another of its tensors.
    """
    if not all(0.0 <= b < 1.0 for b in betas):
        raise RuntimeError(f"betas must be in [0, 1), got {betas}")
    if type(steps) is not int and isinstance(steps, Sequence):
        if any(t < 1 for t in steps):
            raise RuntimeError("steps must be >= 1")
        alphas = [adamw_alpha(lr, betas, int(t)) for t in steps]
    else:
        if steps < 1:
            raise RuntimeError("steps must be >= 1")
        alphas = adamw_alpha(lr, betas, int(steps))
    # the plain case in one call; anything else is checked here and taken apart
    rc = _lib.step_ext().adamw(params, grads, moments1, moments2, alphas, float(1 - lr * wd),
                               1 - betas[0], 1 - betas[1], float(eps), True)
    if rc is not None:
        _lib.check(rc, "fm_adamw")
        return
    params = _check_list(params, "params")
    n = len(params)
    grads = _check_list(grads, "grads", n)
    moments1 = _check_list(moments1, "moments1", n)
    moments2 = _check_list(moments2, "moments2", n)
    if not isinstance(alphas, list):
        alphas = [alphas] * n
    elif len(alphas) != n:
        raise RuntimeError(f"steps must be an int or one per parameter, got {len(alphas)} for {n}")
    if n == 0:
        return
    lists = (params, grads, moments1, moments2)
    types = _check_adamw(*lists)
    kinds = dict.fromkeys(types)
    # a launch sees the tensors of its own kind only
    if len(kinds) > 1 and _overlap(params + moments1 + moments2, grads):
        raise RuntimeError("fused_adamw: tensors overlap in memory")
    for kind in kinds:
        idx = [i for i in range(n) if types[i] == kind]
        some = [[ts[i] for i in idx] for ts in lists]
        adamw_launch(*some, [alphas[i] for i in idx], lr, wd, betas, eps)
        _bump(some[0] + some[2] + some[3])


def normed_workspace_size(count: int, rows: int) -> int:
    """Bytes of device workspace ``fused_normed_update`` needs for ``count`` matrices."""
    out = ctypes.c_uint64(0)
    _lib.check(_lib.load().fm_normed_workspace_size(int(count), int(rows), ctypes.byref(out)),
               "fm_normed_workspace_size")
    return int(out.value)


def _refuse_normed(p0, p, u, v, rows) -> None:
    """Name what is wrong with one matrix of a fused_normed_update call."""
    if not (p.device == u.device == v.device == p0.device):
        raise RuntimeError("fused_normed_update needs all tensors on one device")
    if p.dtype != p0.dtype or p.shape != p0.shape:
        raise RuntimeError("the params of one call must have one shape and type")
    if u.dtype != torch.bfloat16 or u.numel() != p.numel() or not u.dim() or u.size(0) != rows:
        raise RuntimeError("updates must be bf16 and shaped like the parameters")
    if v.dtype != torch.float32 or v.shape != (rows,):
        raise RuntimeError("row_moments must be fp32 vectors of one element per row")
    if p.is_neg() or u.is_neg() or v.is_neg():
        raise RuntimeError("fused_normed_update needs tensors that are not negative views")
    raise RuntimeError("fused_normed_update needs contiguous tensors")


def fused_normed_update(
    params: Sequence[torch.Tensor],
    updates: torch.Tensor | Sequence[torch.Tensor],
    row_moments: Sequence[torch.Tensor],
    *,
    lr: float,
    wd: float = 0.1,
    beta2: float = 0.95,
    eps: float = 1e-8,
    workspace: torch.Tensor | None = None,
) -> None:
    """Decay + neuron-wise normalised update of same-shape matrices, in place.

    For each matrix (rows = output neurons) with its orthogonalised update u::

        s_i = mean_j u_ij²;  v_i = beta2·v_i + (1 - beta2)·s_i
        r_i = 1/(sqrt(v_i) + eps);  F = ‖diag(r)·u‖_F
        p_ij = p_ij·(1 - lr·wd) - lr·0.2·sqrt(rows·cols)/(F + 1e-7) · r_i·u_ij

    so that every neuron moves at a rate of its own while the update's root
    mean square stays 0.2·lr, the size Muon's learning-rate scale aims at.

    Args:
        params: contiguous CUDA parameters (fp32, bf16 or fp16) of one shape
            and type; more than two dimensions are seen as (size(0), -1).
        updates: a contiguous bf16 (count, rows, cols) tensor, or one bf16
            tensor per parameter.
        row_moments: an fp32 tensor of ``rows`` elements per parameter (v).
        workspace: optional CUDA buffer of at least
            ``normed_workspace_size(count, rows)`` bytes.
    """
    if not 0.0 <= beta2 < 1.0:
        raise RuntimeError(f"beta2 must be in [0, 1), got {beta2}")
    # the plain case in one call; anything else is checked here
    rc = _lib.step_ext().normed(params, updates, row_moments, float(1 - lr * wd), float(lr * 0.2),
                                float(beta2), float(eps), workspace)
    if rc is not None:
        _lib.check(rc, "fm_muon_apply_normed")
        return
    params = _check_list(params, "params")
    n = len(params)
    updates = _check_list(updates.unbind(0) if isinstance(updates, torch.Tensor) else updates,
                          "updates", n)
    row_moments = _check_list(row_moments, "row_moments", n)
    if n == 0:
        return
    p0 = params[0]
    _check_cuda(p0, "params")
    if p0.dim() < 2:
        raise RuntimeError("fused_normed_update needs matrices")
    dtype, numel, rows = p0.dtype, p0.numel(), p0.size(0)
    if dtype not in STEP_DTYPES:
        raise RuntimeError(f"params must be fp32, bf16 or fp16, got {dtype}")
    device, cols = p0.get_device(), numel // rows if rows else 0
    for p, u, v in zip(params, updates, row_moments):
        if not (p.dtype is dtype and p.is_same_size(p0) and u.dtype is torch.bfloat16
                and u.numel() == numel and (u.size(0) if u.dim() else -1) == rows
                and v.dtype is torch.float32 and v.dim() == 1 and v.numel() == rows
                and p.get_device() == u.get_device() == v.get_device() == device
                and p.is_contiguous() and u.is_contiguous() and v.is_contiguous()
                and not (p.is_neg() or u.is_neg() or v.is_neg())):
            _refuse_normed(p0, p, u, v, rows)
    if numel == 0:
        return
    workspace = workspace_for(p0, normed_workspace_size(n, rows), workspace)
    ptr = torch.Tensor.data_ptr
    table = b"".join(map(_lib.NORMED_MATRIX.pack, map(ptr, params), map(ptr, updates),
                         map(ptr, row_moments)))
    with _on_device(p0):
        _lib.check(_lib.load().fm_muon_apply_normed(
            table, n, rows, cols, STEP_DTYPES[p0.dtype], float(1 - lr * wd),
            float(lr * 0.2 * math.sqrt(rows * cols)), float(beta2), float(eps), workspace.data_ptr(), workspace.nbytes,
            _stream(p0)), "fm_muon_apply_normed")
    _bump(params + row_moments)
