"""FusedMuon's per-head and normalised Muon groups and its fp32 AdamW state, on
the CPU: option checks, formulas, checkpoints, and the sharded step on gloo."""

import copy
import math
import os
import pickle
import tempfile

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import muon_fused.optimizer as opt_mod
from muon_fused import FusedMuon
from tests.test_sharding import _free_port, _patch_ns

A, B, C = 3.4445, -4.7750, 2.0315


def _ns64(x, steps):
    x = x.double()
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        a = x @ x.T
        x = A * x + (B * a + C * a @ a) @ x
    return x


def heads_on_cpu(G, heads, dim, steps, workspace, out):
    for b in range(G.shape[0]):
        out[b].copy_(torch.cat([_ns64(h, steps) for h in G[b].chunk(heads, dim)], dim))


def _patch():
    _patch_ns()
    opt_mod._ns_heads_batched = heads_on_cpu
    opt_mod.workspace_size_heads = lambda *a, **k: 256


SHAPES = [(32, 48), (32, 48), (64, 16), (48, 24)]
GROUPS = [{"heads": 4, "heads_dim": 0, "normed_beta2": 0.9}, {"heads": 2, "heads_dim": 1},
          {"normed_beta2": 0.95}]


def _params():
    g = torch.Generator().manual_seed(0)
    return [[torch.nn.Parameter(torch.randn(s, generator=g) * 0.02) for s in SHAPES]
            for _ in GROUPS]


def _groups(params):
    return [{"params": ps, "use_muon": True, **opts} for ps, opts in zip(params, GROUPS)]


def _set_grads(params, step):
    g = torch.Generator().manual_seed(100 + step)
    for ps in params:
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g) * 1e-3


def _run(steps, **kw):
    params = _params()
    opt = FusedMuon(_groups(params), lr=0.02, **kw)
    for s in range(steps):
        _set_grads(params, s)
        opt.step()
    return params, opt


@pytest.fixture
def patched(monkeypatch):
    for name in ("_ns_batched", "_ns_heads_batched", "workspace_size_heads"):
        monkeypatch.setattr(opt_mod, name, getattr(opt_mod, name))
    from muon_fused import _fused_muon_C as _C

    monkeypatch.setattr(_C, "workspace_size_batched", _C.workspace_size_batched)
    _patch()


def test_options_are_checked():
    w = torch.nn.Parameter(torch.zeros(32, 48))
    for bad in ({"heads": 5}, {"heads": 0}, {"heads": 4, "heads_dim": 2}, {"heads": 5, "heads_dim": 1},
                {"normed_beta2": 1.0}):
        with pytest.raises(ValueError):
            FusedMuon([{"params": [w], "use_muon": True, **bad}])
    with pytest.raises(ValueError, match="use_muon"):
        FusedMuon([{"params": [w], "heads": 4}])
    with pytest.raises(ValueError, match="divide"):
        FusedMuon([{"params": torch.nn.Parameter(torch.zeros(8, 4, 4)), "use_muon": True, "heads": 4}])
    with pytest.raises(ValueError, match="adamw_state_dtype"):
        FusedMuon([w], adamw_state_dtype=torch.bfloat16)
    opt = FusedMuon([{"params": (p for p in [w]), "use_muon": True, "heads": 4, "heads_dim": 0}])
    assert opt.param_groups[0]["params"] == [w]


def test_step_follows_the_formulas(patched):
    """Two steps of each kind of group against the update written out: momentum,
    per-head (or whole) Newton-Schulz rounded to bf16, row normalisation, decay."""
    params, _ = _run(2)
    want = _params()
    for ps, opts in zip(want, GROUPS):
        for k, p in enumerate(ps):
            w, buf, v = p.detach().clone(), torch.zeros_like(p), torch.zeros(p.shape[0])
            for s in range(2):
                _set_grads(want, s)
                buf = 0.95 * buf + p.grad
                d = (p.grad + 0.95 * buf).bfloat16()
                heads, dim = opts.get("heads", 1), opts.get("heads_dim", 0)
                if opts.get("heads"):
                    u = torch.cat([_ns64(h, 5) for h in d.chunk(heads, dim)], dim).bfloat16()
                else:
                    u = torch.empty(1, *p.shape, dtype=torch.bfloat16)
                    opt_mod._ns_batched(d[None], 5, None, u)
                    u = u[0]
                shape = list(p.shape)
                shape[dim] //= heads
                beta2 = opts.get("normed_beta2")
                if beta2 is None:
                    w = w * (1 - 0.02 * 0.1) - 0.02 * 0.2 * math.sqrt(max(shape)) * u.float()
                else:
                    o = u.float()
                    v = beta2 * v + (1 - beta2) * o.square().mean(1)
                    o = o / (v.sqrt() + 1e-8)[:, None]
                    w = w * (1 - 0.02 * 0.1) - 0.02 * 0.2 * math.sqrt(o.numel()) / o.norm() * o
            torch.testing.assert_close(params[GROUPS.index(opts)][k].detach(), w, rtol=2e-5, atol=1e-7)


def test_state_keeps_fp32_statistics_across_a_checkpoint(patched):
    w = torch.nn.Parameter((torch.randn(32, 48) * 0.02).bfloat16())
    e = torch.nn.Parameter((torch.randn(7, 5) * 0.02).bfloat16())

    def make():
        return FusedMuon([{"params": [w], "use_muon": True, "normed_beta2": 0.9}, {"params": [e]}],
                         adamw_state_dtype=torch.float32)

    opt = make()
    w.grad, e.grad = torch.randn_like(w) * 1e-3, torch.randn_like(e) * 1e-3
    opt.step()
    assert opt.state[w]["row_moment"].dtype == torch.float32
    assert opt.state[e]["moment1"].dtype == opt.state[e]["moment2"].dtype == torch.float32
    saved = copy.deepcopy(opt.state_dict())
    new = make()
    new.load_state_dict(saved)
    for p, keys in ((w, ["row_moment"]), (e, ["moment1", "moment2"])):
        for k in keys:
            assert new.state[p][k].dtype == torch.float32
            assert torch.equal(new.state[p][k], opt.state[p][k])
    assert new.param_groups[0]["normed_beta2"] == 0.9
    new.step()


def test_adamw_fp32_state_on_cpu():
    """16-bit parameters with fp32 moments: computed in fp32, rounded once."""
    p = torch.nn.Parameter((torch.randn(50) * 0.02).bfloat16())
    g = (torch.randn(50) * 1e-3).bfloat16()
    p0 = p.detach().double()
    opt = FusedMuon([p], lr=0.01, adamw_state_dtype=torch.float32)
    p.grad = g
    opt.step()
    m, v = 0.1 * g.double(), 0.05 * g.double() ** 2
    want = p0 * (1 - 0.01 * 0.1) - 0.01 * (0.05 ** 0.5 / 0.1) * m / (1e-8 + v.sqrt())
    err = (p.detach().double() - want).abs()
    assert bool((err <= want.abs() * 2.0 ** -8 + 1e-6).all())


def _worker(rank, world, port, outdir, collective):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    import datetime

    dist.init_process_group("gloo", rank=rank, world_size=world,
                            timeout=datetime.timedelta(seconds=60))
    _patch()
    try:
        params, opt = _run(2, bucket_bytes=8192, collective=collective)
        rows = sum("row_moment" in opt.state[p] for ps in params for p in ps)
        opt.consolidate_state_dict()
        torch.save({"params": [p.detach() for ps in params for p in ps], "rows": rows,
                    "state": opt.state_dict()["state"]}, os.path.join(outdir, f"rank{rank}.pt"))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("collective", ["nccl", "param_gather"])
def test_sharded_options_equal_single_process(patched, collective):
    params, opt = _run(2)
    ref = [p.detach() for ps in params for p in ps]
    state = opt.state_dict()["state"]
    outdir = tempfile.mkdtemp()
    mp.spawn(_worker, args=(2, _free_port(), outdir, collective), nprocs=2, join=True)
    rows = 0
    for r in range(2):
        res = torch.load(os.path.join(outdir, f"rank{r}.pt"))
        for a, b in zip(res["params"], ref):
            assert torch.equal(a, b)
        for k, v in state.items():  # consolidated: every rank has every statistic
            assert torch.equal(res["state"][k]["momentum_buffer"], v["momentum_buffer"])
            if "row_moment" in v:
                assert torch.equal(res["state"][k]["row_moment"], v["row_moment"])
        rows += res["rows"]
    # the all-gather applies every update on every rank, the owner's apply only its own
    normed = 2 * len(SHAPES)
    assert rows == (2 * normed if collective == "nccl" else normed)


def test_adamw_groups_need_neither_the_library_nor_an_sm100_device(monkeypatch):
    from muon_fused import _lib, step_ops

    def missing():
        raise ImportError("libfused_muon.so is missing")

    capability = [(10, 0)]
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda d=None: capability[0])
    monkeypatch.setattr(_lib, "step_ext", lambda: None)
    assert step_ops.adamw_ready.__wrapped__(0)
    monkeypatch.setattr(_lib, "step_ext", missing)
    with pytest.warns(RuntimeWarning, match="torch ops"):
        assert not step_ops.adamw_ready.__wrapped__(0)
    capability[0] = (9, 0)
    assert not step_ops.adamw_ready.__wrapped__(0)


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex64, torch.float32])
def test_fp32_state_option_changes_nothing_for_wider_parameters(dtype):
    """fp64 and complex parameters keep moments of their own type, through a checkpoint too."""
    g = torch.Generator().manual_seed(0)
    p0 = torch.randn(20, generator=g, dtype=dtype)
    grads = [torch.randn(20, generator=g, dtype=dtype) for _ in range(3)]
    runs = []
    for state_dtype in (None, torch.float32):
        p = torch.nn.Parameter(p0.clone())
        opt = FusedMuon([p], lr=0.01, adamw_state_dtype=state_dtype)
        for step, grad in enumerate(grads):
            p.grad = grad.clone()
            opt.step()
            if step == 1:
                saved = copy.deepcopy(opt.state_dict())
                opt = FusedMuon([p], lr=0.01, adamw_state_dtype=state_dtype)
                opt.load_state_dict(saved)
        runs.append((p.detach(), opt.state[p]["moment1"], opt.state[p]["moment2"]))
    for a, b in zip(*runs):
        assert a.dtype == b.dtype == dtype and torch.equal(a, b)


def test_loading_hooks_see_and_replace_the_state(patched):
    """What a pre-hook puts in the place of the dict is loaded, in fp32 where that is kept,
    and a post-hook has the last word."""
    w = torch.nn.Parameter((torch.randn(32, 48) * 0.02).bfloat16())
    e = torch.nn.Parameter((torch.randn(7, 5) * 0.02).bfloat16())
    opt = FusedMuon([{"params": [w], "use_muon": True, "normed_beta2": 0.9}, {"params": [e]}],
                    adamw_state_dtype=torch.float32)
    w.grad, e.grad = torch.randn_like(w) * 1e-3, torch.randn_like(e) * 1e-3
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    doubled = copy.deepcopy(saved)
    for st in doubled["state"].values():
        for key in ("row_moment", "moment1"):
            if key in st:
                st[key] = st[key] * 2 + 1e-4
    seen = []
    opt.register_load_state_dict_pre_hook(lambda o, sd: doubled)
    opt.register_load_state_dict_post_hook(
        lambda o: seen.append((o.state[w]["row_moment"].dtype, o.state[e]["moment1"].dtype))
        or o.state[e]["moment2"].zero_())
    for _ in range(2):
        opt.load_state_dict(saved)
        assert torch.equal(opt.state[w]["row_moment"], doubled["state"][0]["row_moment"])
        assert torch.equal(opt.state[e]["moment1"], doubled["state"][1]["moment1"])
        assert not opt.state[e]["moment2"].any()
    assert seen == [(torch.float32, torch.float32)] * 2
    assert len(opt._optimizer_load_state_dict_pre_hooks) == 1
    assert len(opt._optimizer_load_state_dict_post_hooks) == 1


@pytest.mark.parametrize("how", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_copies_of_the_optimizer(patched, how):
    """A copy keeps the options, steps as the original does and loads its checkpoints."""
    def make():
        g = torch.Generator().manual_seed(3)
        w = torch.nn.Parameter(torch.randn(32, 48, generator=g) * 0.02)
        e = torch.nn.Parameter((torch.randn(7, generator=g) * 0.02).bfloat16())
        return FusedMuon([{"params": [w], "use_muon": True, "heads": 4, "normed_beta2": 0.9},
                          {"params": [e]}], lr=0.02, adamw_state_dtype=torch.float32)

    def step(opt, seed):
        g = torch.Generator().manual_seed(seed)
        for group in opt.param_groups:
            for p in group["params"]:
                p.grad = (torch.randn(p.shape, generator=g) * 1e-3).to(p.dtype)
        opt.step()
        return [p.detach() for group in opt.param_groups for p in group["params"]]

    def values(opt):
        return [t for st in opt.state_dict()["state"].values() for t in st.values()
                if isinstance(t, torch.Tensor)]

    opt = make()
    fresh = how(opt)  # before the first step: it makes its own state
    for seed in (1, 2):
        want = step(opt, seed)
        for a, b in zip(want + values(opt), step(fresh, seed) + values(fresh)):
            assert a.dtype == b.dtype and torch.equal(a, b)
    later = how(opt)
    other = make()
    other.load_state_dict(copy.deepcopy(later.state_dict()))
    later.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert all(t.dtype == torch.float32 for t in values(other)[1:])
    for a, b in zip(step(opt, 3) + values(opt), step(later, 3) + values(later)):
        assert a.dtype == b.dtype and torch.equal(a, b)


def _run_uneven(case, **kw):
    """Three steps of a normalised group that param_gather cannot serve in all of them: two
    matrices that are slices of one tensor, or a step in which the lightest has no gradient
    (afterwards the parameters live in the gather's flat buffers)."""
    params = _params()[0]
    if case == "shared":
        base = torch.cat([params[0].detach(), params[1].detach()])
        params[:2] = [torch.nn.Parameter(base[:32]), torch.nn.Parameter(base[32:])]
    opt = FusedMuon([{"params": params, "use_muon": True, "normed_beta2": 0.9}], lr=0.02, **kw)
    for s in range(4):
        _set_grads([params], s)
        if case == "missing" and s in (1, 3):
            params[2].grad = None
        opt.step()
    return params, opt


def _uneven_worker(rank, world, port, outdir, case):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    import datetime

    dist.init_process_group("gloo", rank=rank, world_size=world,
                            timeout=datetime.timedelta(seconds=60))
    _patch()
    try:
        params, opt = _run_uneven(case, bucket_bytes=8192, collective="param_gather")
        opt.consolidate_state_dict()
        torch.save({"params": [p.detach() for p in params], "state": opt.state_dict()["state"]},
                   os.path.join(outdir, f"rank{rank}.pt"))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("case", ["shared", "missing"])
def test_row_moments_where_param_gather_falls_back(patched, case):
    """A step that falls back to the update all-gather applies every update on every rank, so
    every rank needs every row moment."""
    params, opt = _run_uneven(case)
    state = opt.state_dict()["state"]
    outdir = tempfile.mkdtemp()
    mp.spawn(_uneven_worker, args=(2, _free_port(), outdir, case), nprocs=2, join=True)
    for r in range(2):
        res = torch.load(os.path.join(outdir, f"rank{r}.pt"))
        for i, (a, p) in enumerate(zip(res["params"], params)):
            assert torch.equal(a, p.detach()), (r, i)
        for k, v in state.items():
            assert torch.equal(res["state"][k]["row_moment"], v["row_moment"]), (r, k)


def test_which_parameters_reach_into_the_same_memory():
    x = torch.zeros(64)
    for yes in ([x[:32], x[31:]], [x.view(8, 8).T, x[63:]], [x[:48], x[2:3], x[40:]]):
        assert opt_mod._overlapping(yes) and opt_mod._overlapping(yes[:1], yes[1:])
    assert opt_mod._overlapping([], [x[:32], x[31:]])
    for no in ([x[:32], x[32:]], [x[5:5], x], [x, x[5:5]], [x[:1].expand(9), x[1:]],
               [x[:32].view(4, 8).T, x[32:]], [torch.zeros(3, 0).T, x]):
        assert not opt_mod._overlapping(no) and not opt_mod._overlapping(no[:1], no[1:])
