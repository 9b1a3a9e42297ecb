"""FusedMuon — Muon with the B200 Newton-Schulz engine.

Same constructor, defaults, state keys and group semantics as the reference
(muon_fused/optimizer.py:51-202):

* groups with ``use_muon=True`` run SGD-momentum (nesterov by default), the
  Newton-Schulz orthogonalisation, decoupled weight decay and the
  ``0.2·sqrt(max(A, B))`` learning-rate scale (optimizer.py:120-163);
* every other group runs the reference's AdamW variant
  (optimizer.py:165-200) — including the quirk that a plain parameter list
  has no ``use_muon`` key and therefore takes the AdamW branch.  On CUDA the
  whole group is one launch (``fused_adamw``) with the reference's results.

Beyond the reference, a Muon group may name

* ``heads`` and ``heads_dim``: its matrices are attention projections whose
  heads are blocks of rows (``heads_dim=0``) or columns (``1``); each head is
  orthogonalised by itself (``fused_newton_schulz_heads``) and the learning-rate
  scale takes the head's shape;
* ``normed_beta2``: the update is normalised per output neuron by a running
  second moment (``fused_normed_update``; state key ``row_moment``).

B200-specific behaviour:

* Parameters of a Muon group are processed through ``muon_fused.sharding``:
  under ``torch.distributed`` with world size > 1 each rank orthogonalises
  only the matrices it owns (FLOP-balanced assignment) and the bf16 updates
  are all-gathered over NCCL; with one process everything is local.
* Momentum state is kept only by the owning rank, so ``state_dict`` is
  rank-local when sharded until ``consolidate_state_dict()`` broadcasts every
  buffer from its owner; keys are the reference's ``momentum_buffer``.
"""

from __future__ import annotations

import math
import operator
from typing import Any

import torch
from torch.optim import Optimizer

from muon_fused import _fused_muon_C as _C
from muon_fused import _lib
from muon_fused.ns_step import fused_newton_schulz_heads, workspace_size, workspace_size_heads
from muon_fused.step_ops import (STEP_DTYPES, UnfitTensors, adamw_alpha, adamw_launch,
                                 adamw_ready, fused_normed_update, normed_workspace_size)

# Parameter / gradient dtypes the fused elementwise kernels handle.
_EW_DTYPES = {torch.float32: _lib.FM_DT_F32, torch.bfloat16: _lib.FM_DT_BF16,
              torch.float16: _lib.FM_DT_F16}


# Tensor types whose memory is what data_ptr() says (a DTensor's is not).
_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _overlapping(tensors, contiguous=()) -> bool:
    """Whether two of the tensors reach into the same memory (strided ones: from their first
    to their last element).  ``contiguous`` ones, known as such, are read in bulk: 85 of them
    take 44 µs so and 88 one by one."""
    los = list(map(torch.Tensor.data_ptr, contiguous))
    spans = list(zip(los, map(operator.add, los, map(_NBYTES, contiguous))))
    for t in tensors:
        if type(t) in _PLAIN and t.layout is torch.strided and t.numel():
            last = sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
            spans.append((t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()))
    spans.sort()
    end = 0
    for lo, hi in spans:
        if lo < end and lo < hi:
            return True
        if hi > end:
            end = hi
    return False


_NBYTES = operator.attrgetter("nbytes")


def _ns_batched(G: torch.Tensor, steps: int, workspace: torch.Tensor, out: torch.Tensor):
    """Batched Newton-Schulz used by the optimizer (module level so a test can
    substitute a CPU implementation in a gloo child process)."""
    return _C.fused_newton_schulz_batched(G, steps, workspace, out=out)


def _ns_heads_batched(G: torch.Tensor, heads: int, dim: int, steps: int, workspace: torch.Tensor,
                      out: torch.Tensor):
    """Per-head Newton-Schulz used by the optimizer (substituted like ``_ns_batched``)."""
    return fused_newton_schulz_heads(G, heads, steps, workspace, dim=dim, out=out)


class FusedMuon(Optimizer):
    """Muon optimizer with fused Newton-Schulz orthogonalisation.

    Args:
        param_groups: iterable of parameters or of group dicts; groups with
            ``"use_muon": True`` take the Muon path, all others AdamW.  A Muon
            group may also set ``"heads"`` (with ``"heads_dim"``, 0 or 1,
            default 0) and ``"normed_beta2"``, see above; its matrices then
            have 2-D shapes that divide into the heads.
        lr: base learning rate (default ``1e-3``).
        wd: decoupled weight decay (default ``0.1``).
        momentum: SGD momentum of Muon groups (default ``0.95``).
        nesterov: Nesterov momentum (default ``True``).
        ns_steps: Newton-Schulz iterations (default ``5``).
        adamw_betas: AdamW betas (default ``(0.9, 0.95)``).
        adamw_eps: AdamW epsilon (default ``1e-8``).
        process_group: process group to shard Muon work over; defaults to
            the world group when ``torch.distributed`` is initialised.
        bucket_bytes: size of each all-gather bucket of packed updates when
            sharded (default 256 MiB).
        batch_bytes: device memory one batched Newton-Schulz call may use for
            its inputs, outputs and workspace (default 4 GiB); same-shape
            matrices are batched up to this budget.
        collective: how a sharded step shares the updates: ``"nccl"`` (bucketed
            all-gather of the bf16 updates, then every rank applies every
            update) or ``"param_gather"`` (each owner applies its own updates,
            then the bucket's parameters are all-gathered in place; the
            parameters' ``.data`` are moved into per-bucket flat buffers for
            this, see ``sharding.ParamStore``).  Both give bit-identical
            parameters.
        adamw_state_dtype: type of the AdamW moments: ``None`` (default) is the
            gradient's, as the reference; ``torch.float32`` keeps them in fp32
            beside 16-bit parameters (and changes nothing for wider ones).
    """

    def __init__(
        self,
        param_groups,
        lr: float = 1e-3,
        wd: float = 0.1,
        momentum: float = 0.95,
        nesterov: bool = True,
        ns_steps: int = 5,
        adamw_betas: tuple[float, float] = (0.9, 0.95),
        adamw_eps: float = 1e-8,
        process_group=None,
        bucket_bytes: int = 256 << 20,
        batch_bytes: int = 4 << 30,
        collective: str = "nccl",
        adamw_state_dtype: torch.dtype | None = None,
    ):
        if adamw_state_dtype not in (None, torch.float32):
            raise ValueError(f"adamw_state_dtype must be None or torch.float32, got "
                             f"{adamw_state_dtype}")
        self._adamw_state_dtype = adamw_state_dtype
        defaults: dict[str, Any] = dict(
            lr=lr, wd=wd, momentum=momentum, nesterov=nesterov, ns_steps=ns_steps,
            adamw_betas=adamw_betas, adamw_eps=adamw_eps,
        )
        super().__init__(param_groups, defaults)
        self._process_group = process_group
        self._bucket_bytes = int(bucket_bytes)
        self._batch_bytes = int(batch_bytes)
        if collective not in ("nccl", "param_gather"):
            raise ValueError(f"collective must be 'nccl' or 'param_gather', got {collective!r}")
        self._collective = collective
        self._init_caches()

    def _init_caches(self) -> None:
        """What the steps keep beside the state; a copy starts without it."""
        self._workspaces: dict[tuple, torch.Tensor] = {}
        self._plans: dict[tuple, Any] = {}
        self._arena: dict[torch.device, torch.Tensor] = {}
        self._stores: dict[tuple, Any] = {}
        # id(group) -> (params, owner rank per param, momentum dtype per param)
        # of the group's last sharded step (consolidate_state_dict)
        self._owners: dict[int, tuple] = {}
        # parameter -> the one rank that holds its row_moment (after owner-applied steps)
        self._row_owner: dict[torch.Tensor, int] = {}

    # Constructor options that a copy keeps (a process group cannot be copied: the copy
    # uses the world group), with their defaults for optimizers pickled without them.
    _COPIED = {"_adamw_state_dtype": None, "_bucket_bytes": 256 << 20, "_batch_bytes": 4 << 30,
               "_collective": "nccl"}

    def __getstate__(self):
        return {**super().__getstate__(), **{name: getattr(self, name) for name in self._COPIED}}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)  # load_state_dict comes here too, with a live optimizer
        for name, value in self._COPIED.items():
            self.__dict__.setdefault(name, value)
        if "_owners" not in self.__dict__:
            self._process_group = None
            self._init_caches()

    def add_param_group(self, param_group) -> None:
        """As ``Optimizer.add_param_group``, checking a Muon group's options first."""
        if not isinstance(param_group, dict):
            super().add_param_group(param_group)  # raises as the base class does
            return
        heads, dim = param_group.get("heads"), param_group.get("heads_dim", 0)
        beta2 = param_group.get("normed_beta2")
        if (heads is not None or beta2 is not None) and not param_group.get("use_muon", False):
            raise ValueError("heads and normed_beta2 are options of use_muon groups")
        if beta2 is not None and not 0.0 <= beta2 < 1.0:
            raise ValueError(f"normed_beta2 must be in [0, 1), got {beta2}")
        if heads is not None:
            if int(heads) < 1 or dim not in (0, 1):
                raise ValueError(f"heads must be >= 1 and heads_dim 0 or 1, got {heads}, {dim}")
            params = param_group["params"]
            param_group["params"] = params = ([params] if isinstance(params, torch.Tensor)
                                              else list(params))
            for p in params:
                p = p[1] if isinstance(p, tuple) else p  # a named parameter
                if p.ndim != 2 or p.shape[dim] % heads:
                    raise ValueError(f"a {tuple(p.shape)} parameter does not divide into {heads} "
                                     f"heads along dimension {dim}")
        super().add_param_group(param_group)

    # ------------------------------------------------------------------ helpers
    @staticmethod
    def adjust_lr_for_muon(lr: float, param_shape: torch.Size) -> float:
        """``lr · 0.2 · sqrt(max(A, B))`` over the first two dims (optimizer.py:79-84)."""
        A, B = param_shape[:2]
        return lr * 0.2 * math.sqrt(max(A, B))

    def _get_workspace(self, m: int, n: int, device: torch.device) -> torch.Tensor:
        """Cached workspace per (device, orientation-free shape) (optimizer.py:86-94)."""
        key = (device, min(m, n), max(m, n))
        ws = self._workspaces.get(key)
        if ws is None:
            ws = torch.empty(workspace_size(m, n), dtype=torch.uint8, device=device)
            self._workspaces[key] = ws
        return ws

    def _world(self):
        import torch.distributed as dist

        if not (dist.is_available() and dist.is_initialized()):
            return None, 0, 1
        pg = self._process_group
        return pg, dist.get_rank(pg), dist.get_world_size(pg)

    # ------------------------------------------------------------------ Muon
    def _momentum_into(self, p: torch.Tensor, g: torch.Tensor, dst: torch.Tensor, momentum: float,
                       nesterov: bool) -> None:
        """buf ← μ·buf + g; dst ← bf16(g + μ·buf) (nesterov) or bf16(buf)
        (optimizer.py:139-149).

        On CUDA this is one fused kernel (fm_muon_momentum) writing the bf16
        Newton-Schulz input straight into ``dst``; the buffer is bit-identical
        to the reference's torch ops.  CPU tensors (no Newton-Schulz path
        exists for them) keep the reference's torch ops."""
        state = self.state[p]
        if "momentum_buffer" not in state:
            state["momentum_buffer"] = torch.zeros_like(g)
        buf = state["momentum_buffer"]
        dt = _EW_DTYPES.get(g.dtype)
        if g.is_cuda and dt is not None and buf.is_contiguous() and dst.is_contiguous():
            gc = g.contiguous().resolve_neg()
            with torch.cuda.device(g.device):
                _lib.check(_lib.load().fm_muon_momentum(
                    buf.data_ptr(), gc.data_ptr(), dst.data_ptr(), g.numel(), dt,
                    float(momentum), 1 if nesterov else 0,
                    torch.cuda.current_stream(g.device).cuda_stream), "fm_muon_momentum")
            return
        buf.mul_(momentum).add_(g)
        dst.copy_(g.add(buf, alpha=momentum) if nesterov else buf)

    def _scratch(self, device: torch.device, nbytes: int) -> torch.Tensor:
        """One reusable device buffer per device for batch inputs, outputs and
        the Newton-Schulz workspace.  Reuse is safe because every user is
        ordered on the same stream."""
        buf = self._arena.get(device)
        if buf is None or buf.numel() < nbytes:
            buf = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
            self._arena[device] = buf
        return buf

    @staticmethod
    def _ns_workspace(group, batch: int, rows: int, cols: int) -> int:
        """Workspace bytes of a group's Newton-Schulz call on ``batch`` matrices."""
        if group.get("heads") is None:
            return _C.workspace_size_batched(batch, rows, cols)
        return workspace_size_heads((batch, rows, cols), group["heads"],
                                    dim=group.get("heads_dim", 0), steps=group["ns_steps"])

    def _batch_limit(self, rows: int, cols: int, group=None) -> int:
        """Matrices per batched call so inputs, outputs and workspace of one
        batch stay within ``batch_bytes``."""
        group = group or {}
        per = self._ns_workspace(group, 1, rows, cols) + 4 * rows * cols
        # at most 65535 heads in one per-head call
        most = min(64, 65535 // (group.get("heads") or 1))
        return max(1, min(most, self._batch_bytes // per))

    def _orthogonalise_batch(self, params, group, out=None) -> torch.Tensor:
        """Momentum + Newton-Schulz for same-shape parameters in one batched
        call; returns (B, rows, cols) bf16 updates (written into ``out`` when
        given, e.g. a slice of the all-gather send buffer)."""
        g0 = params[0].grad
        rows = g0.size(0)
        cols = g0.numel() // rows
        B = len(params)
        dev = g0.device
        n_el = B * rows * cols
        dir_bytes = (2 * n_el + 255) // 256 * 256
        ws_bytes = self._ns_workspace(group, B, rows, cols)
        out_bytes = 0 if out is not None else (2 * n_el + 255) // 256 * 256
        arena = self._scratch(dev, dir_bytes + out_bytes + ws_bytes)
        dirs = arena[:2 * n_el].view(torch.bfloat16).view(B, rows, cols)
        if out is None:
            out = arena[dir_bytes:dir_bytes + 2 * n_el].view(torch.bfloat16).view(B, rows, cols)
        ws = arena[dir_bytes + out_bytes:dir_bytes + out_bytes + ws_bytes]
        for b, p in enumerate(params):
            g = p.grad
            if g.ndim > 2:
                g = g.view(g.size(0), -1)
            self._momentum_into(p, g, dirs[b], group["momentum"], group["nesterov"])
        if group.get("heads") is None:
            _ns_batched(dirs, group["ns_steps"], ws, out)
        else:
            _ns_heads_batched(dirs, group["heads"], group.get("heads_dim", 0), group["ns_steps"],
                              ws, out)
        return out

    def _apply_updates(self, group, params, updates) -> None:
        """Apply a batch's updates (``updates[b]`` to ``params[b]``, one shape)."""
        beta2 = group.get("normed_beta2")
        lr, wd = group["lr"], group["wd"]
        if beta2 is None:
            for p, u in zip(params, updates):
                self._apply_update(p, u, lr, wd, self._update_shape(group, p))
            return
        by_type: dict[torch.dtype, list] = {}
        for p, u in zip(params, updates):
            state = self.state[p]
            if "row_moment" not in state:
                state["row_moment"] = torch.zeros(p.shape[0], dtype=torch.float32, device=p.device)
            data, v = p.data, state["row_moment"]
            if (data.is_cuda and data.dtype in STEP_DTYPES and data.is_contiguous()
                    and not data.is_neg() and type(p) in _PLAIN):
                rows = data.shape[0]
                by_type.setdefault(data.dtype, []).append((data.view(rows, -1), u.view(rows, -1), v))
            else:
                self._normed_update_torch(data, u, v, lr, wd, beta2)
        for items in by_type.values():
            data, us, vs = zip(*items)
            ws = self._normed_scratch(data[0].device, len(data), data[0].shape[0])
            fused_normed_update(data, us, vs, lr=lr, wd=wd, beta2=beta2, workspace=ws)

    @staticmethod
    def _normed_update_torch(data, u, v, lr: float, wd: float, beta2: float,
                             eps: float = 1e-8) -> None:
        """``fused_normed_update`` of one matrix in torch ops (CPU tensors, fp64
        and non-contiguous parameters)."""
        o = u.reshape(u.shape[0], -1).to(torch.promote_types(data.dtype, torch.float32))
        v.copy_(beta2 * v + (1 - beta2) * o.square().mean(1))
        o = o / (v.to(o.dtype).sqrt() + eps)[:, None]
        step = lr * 0.2 * math.sqrt(o.numel()) / (o.norm() + 1e-7)
        data.copy_(data.to(o.dtype) * (1 - lr * wd) - (step * o).view(data.shape))

    def _normed_scratch(self, device: torch.device, count: int, rows: int) -> torch.Tensor:
        """Workspace of the normalised update, apart from the batch's arena (the
        updates that it reads live there).  One per size, kept: a captured step
        goes on using the ones that it was captured with."""
        key = (device, "normed", count, rows)
        buf = self._workspaces.get(key)
        if buf is None:
            buf = torch.empty(normed_workspace_size(count, rows), dtype=torch.uint8, device=device)
            self._workspaces[key] = buf
        return buf

    @staticmethod
    def _update_shape(group, p: torch.Tensor):
        """Shape that the learning-rate scale goes by: the parameter's, or a head's."""
        heads = group.get("heads")
        if heads is None:
            return p.shape
        shape = list(p.shape)
        shape[group.get("heads_dim", 0)] //= heads
        return torch.Size(shape)

    @staticmethod
    def _apply_update(p: torch.Tensor, u: torch.Tensor, lr: float, wd: float, shape=None) -> None:
        """p ← p·(1 − lr·wd) − lr'·u (optimizer.py:157-163), one fused pass
        (fm_muon_apply) on CUDA, bit-identical to the two torch ops."""
        if u.shape != p.shape:
            u = u.view_as(p)
        alpha = -FusedMuon.adjust_lr_for_muon(lr, p.shape if shape is None else shape)
        dt = _EW_DTYPES.get(p.dtype)
        data = p.data
        if (data.is_cuda and dt is not None and data.is_contiguous() and u.is_contiguous()
                and u.dtype == torch.bfloat16):
            with torch.cuda.device(data.device):
                _lib.check(_lib.load().fm_muon_apply(
                    data.data_ptr(), dt, u.data_ptr(), data.numel(), float(1 - lr * wd),
                    float(alpha), torch.cuda.current_stream(data.device).cuda_stream),
                    "fm_muon_apply")
            return
        data.mul_(1 - lr * wd)
        data.add_(u, alpha=alpha)

    def _muon_group_local(self, group) -> None:
        """All matrices on this process: same-shape parameters are batched
        into one Newton-Schulz call (the reference loops one matrix at a time,
        optimizer.py:128-163)."""
        by_shape: dict[tuple, list] = {}
        for p in group["params"]:
            if p.grad is None:
                continue
            key = (p.grad.device, p.shape[0], p.grad.numel() // p.shape[0])
            by_shape.setdefault(key, []).append(p)
        for (_, rows, cols), plist in by_shape.items():
            lim = self._batch_limit(rows, cols, group)
            for k in range(0, len(plist), lim):
                chunk = plist[k:k + lim]
                out = self._orthogonalise_batch(chunk, group)
                self._apply_updates(group, chunk, out.unbind(0))

    def _muon_group_sharded(self, group, pg, rank: int, world: int) -> None:
        from muon_fused import sharding

        params = [p for p in group["params"] if p.grad is not None]
        if not params:
            return
        key = (id(group), tuple(id(p) for p in params), world)
        plan = self._plans.get(key)
        if plan is None:
            plan = sharding.ShardPlan.build([tuple(p.shape) for p in params], world,
                                            self._bucket_bytes)
            self._plans[key] = plan

        self._owners[id(group)] = (params, list(plan.owner), [p.grad.dtype for p in params])
        for p, r in zip(params, plan.owner):
            if r != rank and p in self.state:  # e.g. after loading a consolidated checkpoint
                self.state[p].pop("momentum_buffer", None)
        store = self._stores.get(key)
        # supports() is checked before the store exists: afterwards the parameters
        # deliberately share the store's flat buffers
        gather = self._collective == "param_gather" and (store is not None
                                                         or sharding.ParamStore.supports(params))
        if group.get("normed_beta2") is not None:
            self._place_row_moments(params, plan.owner if gather else None, pg, rank)

        def compute(indices, out) -> None:
            rows, cols = out.shape[1], out.shape[2]
            lim = self._batch_limit(rows, cols, group)
            for k in range(0, len(indices), lim):
                self._orthogonalise_batch([params[i] for i in indices[k:k + lim]], group,
                                          out[k:k + lim])

        def apply(i: int, u: torch.Tensor) -> None:
            self._apply_updates(group, [params[i]], [u])

        dev = params[0].device
        if gather:
            if store is None:
                store = sharding.ParamStore(plan, params, dev)
                self._stores[key] = store
            store.bind(params)
            sharding.run_sharded_param_gather(store, rank, pg, compute, apply)
            return
        sharding.run_sharded(plan, rank, pg, dev, compute, apply)

    def _place_row_moments(self, params, owner, pg, rank: int) -> None:
        """Row moments to where a sharded step applies updates: to each parameter's owner, or
        to every rank (``owner`` None).  Every rank takes the same broadcasts."""
        for i, p in enumerate(params):
            had = self._row_owner.get(p)
            if had is not None and (owner is None or owner[i] != had):
                self._broadcast_row_moment(p, had, pg)
                del self._row_owner[p]
            if owner is not None:
                self._row_owner[p] = owner[i]
                if owner[i] != rank and p in self.state:
                    self.state[p].pop("row_moment", None)

    def _broadcast_row_moment(self, p, r: int, pg) -> None:
        import torch.distributed as dist

        st = self.state[p]
        if "row_moment" not in st:
            st["row_moment"] = torch.zeros(p.shape[0], dtype=torch.float32, device=p.device)
        dist.broadcast(st["row_moment"], src=dist.get_global_rank(pg, r) if pg is not None else r,
                       group=pg)

    # ------------------------------------------------------------------ AdamW
    def _moment_dtype(self, t: torch.Tensor) -> torch.dtype:
        """Type of the moments of a gradient (or parameter) like ``t``: fp32 state is for
        16-bit ones, and nothing wider is cut down to it."""
        if self._adamw_state_dtype is None:
            return t.dtype
        return torch.promote_types(t.dtype, self._adamw_state_dtype)

    @staticmethod
    def _adamw_kind(p, g, buf1, buf2):
        """What the fused kernel groups these tensors by; None where it does not take them."""
        dtype = p.dtype
        if (p.is_cuda and dtype in STEP_DTYPES and g.dtype == dtype
                and type(p) in _PLAIN and type(g) in _PLAIN and not g.is_sparse
                and buf1.dtype == buf2.dtype and buf1.dtype in (dtype, torch.float32)
                and g.device == buf1.device == buf2.device == p.device
                and g.shape == buf1.shape == buf2.shape == p.shape
                and p.is_contiguous() and g.is_contiguous() and buf1.is_contiguous()
                and buf2.is_contiguous() and adamw_ready(p.get_device())):
            return p.device, dtype, buf1.dtype
        return None

    def _adamw_group(self, group) -> None:
        """Reference AdamW branch (optimizer.py:165-200): the tensors that the
        fused kernel takes in one launch, the others in the reference's torch
        ops.  Both give the same values."""
        kinds: dict[Any, list] = {}  # tensors of a kind, in the group's order
        items = []
        for p in group["params"]:
            g = p.grad
            if g is None:
                continue
            state = self.state[p]
            if "step" not in state:
                state["step"] = 0
                dtype = self._moment_dtype(g)
                state["moment1"] = torch.zeros_like(g, dtype=dtype)
                state["moment2"] = torch.zeros_like(g, dtype=dtype)
            state["step"] += 1
            item = p, g, state["moment1"], state["moment2"], state["step"]
            items.append(item)
            kinds.setdefault(self._adamw_kind(*item[:4]), []).append(item)
        if len(kinds) > 1 and _overlapping(
                [item[0] for item in kinds.get(None, ())],
                [item[0] for kind, some in kinds.items() if kind is not None for item in some]):
            # tied storage, perhaps of two kinds: one after the other, as listed
            for item in items:
                self._adamw_items(self._adamw_kind(*item[:4]), [item], group)
            return
        for kind, some in kinds.items():
            self._adamw_items(kind, some, group)

    def _adamw_items(self, kind, items, group) -> None:
        """Step of tensors of one kind, as if one after the other."""
        lr, wd, betas, eps = group["lr"], group["wd"], group["adamw_betas"], group["adamw_eps"]
        if kind is not None:
            alphas: dict[int, float] = {}  # -lr/scale by step
            for *_, step in items:
                if step not in alphas:
                    alphas[step] = adamw_alpha(lr, betas, step)
            *lists, steps = map(list, zip(*items))
            try:
                adamw_launch(*lists, [alphas[t] for t in steps], lr, wd, betas, eps)
                return
            except UnfitTensors:  # some share memory or have torch's negative bit
                if len(items) > 1:
                    for item in items:
                        self._adamw_items(kind, [item], group)
                    return
        for item in items:
            self._adamw_torch(*item, lr, wd, betas, eps)

    @staticmethod
    def _adamw_torch(p, g, buf1, buf2, step: int, lr: float, wd: float, betas, eps: float) -> None:
        """The branch's torch ops on one tensor."""
        beta1, beta2 = betas
        data = p.data
        if buf1.dtype != g.dtype and buf1.dtype == torch.float32:  # beside 16-bit parameters
            g = g.to(buf1.dtype)
            data = data.to(buf1.dtype)
        buf1.lerp_(g, 1 - beta1)
        buf2.lerp_(g.square(), 1 - beta2)
        g = buf1 / (eps + buf2.sqrt())
        bias_correction1 = 1 - beta1 ** step
        bias_correction2 = 1 - beta2 ** step
        scale = bias_correction1 / bias_correction2 ** 0.5
        data.mul_(1 - lr * wd)
        data.add_(g, alpha=-lr / scale)
        if data.dtype != p.dtype:
            p.data.copy_(data)

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def consolidate_state_dict(self) -> None:
        """Make every rank's optimizer state complete after sharded steps.

        Under sharding a matrix's momentum buffer lives only on the rank that
        owns it.  This broadcasts every buffer from its owner, so that
        ``state_dict()`` on any rank then holds the same keys and values as a
        single-process run (and as the reference optimizer,
        optimizer.py:140-141): ready to save, and to load into a run with any
        number of ranks (a sharded step keeps only the buffers its rank owns).
        A collective: every rank of the process group calls it.  Without
        sharding it does nothing.
        """
        pg, rank, world = self._world()
        if world <= 1:
            return
        import torch.distributed as dist

        for group in self.param_groups:
            rec = self._owners.get(id(group))
            if rec is None:
                continue
            params, owner, dtypes = rec
            for p, r, dt in zip(params, owner, dtypes):
                st = self.state[p]
                buf = st.get("momentum_buffer") if r == rank else None
                if buf is None:
                    # the buffer has the gradient's 2-D view shape (see _orthogonalise_batch)
                    shape = (p.shape[0], p.numel() // p.shape[0]) if p.ndim > 2 else p.shape
                    buf = torch.empty(shape, dtype=dt, device=p.device)
                    st["momentum_buffer"] = buf
                src = dist.get_global_rank(pg, r) if pg is not None else r
                dist.broadcast(buf, src=src, group=pg)
                if group.get("normed_beta2") is not None:
                    self._broadcast_row_moment(p, self._row_owner.get(p, r), pg)
            last = set(params)
            for p in group["params"]:  # without a gradient in the last step
                if p not in last and p in self._row_owner:
                    self._broadcast_row_moment(p, self._row_owner[p], pg)

    def load_state_dict(self, state_dict) -> None:
        """As ``Optimizer.load_state_dict``, which casts state to the parameter's
        type, but the fp32 statistics stay fp32: ``row_moment``, and the AdamW
        moments where ``adamw_state_dtype`` asks for it."""
        seen = [state_dict]
        # after the user's pre-hooks, which may replace the dict, and before the post-hooks
        hooks = [self.register_load_state_dict_pre_hook(lambda _, sd: seen.append(sd)),
                 self.register_load_state_dict_post_hook(lambda opt: opt._restore_fp32(seen[-1]),
                                                         prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _restore_fp32(self, state_dict) -> None:
        keys = ["row_moment"]
        if self._adamw_state_dtype is not None:
            keys += ["moment1", "moment2"]
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i, {})
            for key in keys:
                dtype = torch.float32 if key == "row_moment" else self._moment_dtype(p)
                if key in saved and self.state[p][key].dtype != dtype:
                    self.state[p][key] = saved[key].to(device=p.device, dtype=dtype, copy=True)

    def step(self, closure=None):
        """One optimisation step (optimizer.py:99-202)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        pg, rank, world = self._world()
        for group in self.param_groups:
            if group.get("use_muon", False):
                if world > 1:
                    self._muon_group_sharded(group, pg, rank, world)
                else:
                    self._muon_group_local(group)
            else:
                self._adamw_group(group)
        return loss
