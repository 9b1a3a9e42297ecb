"""The operators together as FusedMuon runs them on the GPU: attention
projections by heads, feed-forward matrices with normalised updates, embeddings
and norms with AdamW."""

import copy
import math

import pytest
import torch

from tests.test_heads_gpu import ref64

pytestmark = pytest.mark.gpu

DEV = "cuda"
LR, WD, MU = 0.02, 0.1, 0.95
D, H, FF, V = 256, 4, 512, 1001


def _rand(shape, seed, scale, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _groups(dtype):
    shapes = [[(3 * D, D), (3 * D, D)], [(D, D), (D, D)], [(FF, D), (D, FF), (FF, D)],
              [(V, D), (D,), (D,), (7,)]]
    opts = [{"use_muon": True, "heads": 3 * H}, {"use_muon": True, "heads": H, "heads_dim": 1},
            {"use_muon": True, "normed_beta2": 0.9}, {}]
    k = 0
    groups = []
    for ss, o in zip(shapes, opts):
        ps = []
        for s in ss:
            ps.append(torch.nn.Parameter(_rand(s, k, 0.02, dtype)))
            k += 1
        groups.append({"params": ps, **o})
    return groups


def _set_grads(groups, step):
    k = 1000 * (step + 1)
    for g in groups:
        for p in g["params"]:
            p.grad = _rand(p.shape, k, 1e-3, p.dtype)
            k += 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_whole_step_against_64_bits(cuda_lib, dtype):
    """Three steps; the reference takes the optimizer's own momentum direction
    (bit-checked elsewhere) and computes everything after it in 64 bits.  A
    step's update differs by the head form's rounding (2^-8 + 1e-3 in the norm;
    1e-2 for the whole-matrix form of the normalised group) and the weights'
    own rounding, half a step of their type per op and step."""
    from muon_fused import FusedMuon

    groups = _groups(dtype)
    opt = FusedMuon(groups, lr=LR, wd=WD, momentum=MU, adamw_state_dtype=torch.float32)
    half = torch.finfo(dtype).eps / 2
    stats = {}
    for step in range(3):
        _set_grads(groups, step)
        before = {p: p.detach().double().clone() for g in groups for p in g["params"]}
        opt.step()
        for g in opt.param_groups:
            for p in g["params"]:
                p0, gr, got = before[p], p.grad, p.detach().double()
                if not g.get("use_muon"):
                    m, v = stats.get(p, (0.0, 0.0))
                    m, v = 0.9 * m + 0.1 * gr.double(), 0.95 * v + 0.05 * gr.double() ** 2
                    stats[p] = (m, v)
                    t = step + 1
                    d = LR * (1 - 0.95 ** t) ** 0.5 / (1 - 0.9 ** t) * m / (1e-8 + v.sqrt())
                    want = p0 * (1 - LR * WD) - d
                    # two op-by-op roundings at most, and 2^-20 of the fp32 chain
                    tol = 2 * half * want.abs() + 2.0 ** -20 * (d.abs() + p0.abs()) + 1e-9
                    assert bool(((got - want).abs() <= tol).all())
                    continue
                buf = opt.state[p]["momentum_buffer"]
                dirn = (gr.float() + MU * buf.float()).to(dtype).bfloat16()
                if g.get("heads"):
                    dim = g.get("heads_dim", 0)
                    u = ref64(dirn, g["heads"], 5, dim)
                    shape = list(p.shape)
                    shape[dim] //= g["heads"]
                    d, gate = LR * 0.2 * math.sqrt(max(shape)) * u, 2.0 ** -8 + 1e-3
                else:
                    u = ref64(dirn, 1, 5, 0)
                    v = stats.get(p, torch.zeros(p.shape[0], device=DEV, dtype=torch.float64))
                    v = 0.9 * v + 0.1 * u.square().mean(1)
                    stats[p] = v
                    o = u / v.sqrt()[:, None]
                    d, gate = LR * 0.2 * math.sqrt(u.numel()) * o / o.norm(), 2e-2
                want = p0 * (1 - LR * WD) - d
                rounding = 2 * half * float(want.norm())
                assert float((got - want).norm()) <= gate * float(d.norm()) + rounding
    from muon_fused import _lib

    assert _lib.device_error() == 0


def test_captured_step_equals_eager(cuda_lib):
    """Muon groups of all kinds, captured and replayed (AdamW's step count is a
    host number, so it stays out of a captured step)."""
    from muon_fused import FusedMuon

    results = []
    for captured in (False, True):
        groups = _groups(torch.float32)[:3]
        opt = FusedMuon(groups, lr=LR)
        _set_grads(groups, 0)
        static = [p.grad for g in groups for p in g["params"]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            opt.step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        if captured:
            with torch.cuda.graph(graph):
                opt.step()
        for step in (1, 2):
            k = 1000 * (step + 1)
            for i, s in enumerate(static):
                s.copy_(_rand(s.shape, k + i, 1e-3))
            graph.replay() if captured else opt.step()
        torch.cuda.synchronize()
        results.append([p.detach() for g in groups for p in g["params"]]
                       + [opt.state[p]["row_moment"] for p in groups[2]["params"]])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def _chain(params, state, step, lr, wd):
    """The AdamW branch's torch ops, tensor by tensor."""
    for p in params:
        if p.grad is None:
            continue
        m, v = state.setdefault(p, (torch.zeros_like(p.grad), torch.zeros_like(p.grad)))
        m.lerp_(p.grad, 1 - 0.9)
        v.lerp_(p.grad.square(), 1 - 0.95)
        u = m / (1e-8 + v.sqrt())
        scale = (1 - 0.9 ** step) / (1 - 0.95 ** step) ** 0.5
        p.data.mul_(1 - lr * wd)
        p.data.add_(u, alpha=-lr / scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_adamw_group_keeps_its_results(cuda_lib, dtype):
    """Lists with a transposed parameter, a channels-last one, a missing gradient
    and tied storage: the values of the torch ops, bit for bit."""
    from muon_fused import FusedMuon

    def make():
        base = _rand((40, 30), 1, 0.02, dtype)
        shared = _rand((64,), 2, 0.02, dtype)
        ts = [_rand((33, 17), 0, 0.02, dtype), base.T, shared, shared.view(8, 8), shared[32:],
              _rand((4, 6, 5, 5), 3, 0.02, dtype).to(memory_format=torch.channels_last),
              _rand((9,), 4, 0.02, dtype), _rand((0, 3), 5, 1.0, dtype)]
        return [torch.nn.Parameter(t) for t in ts]

    a, b = make(), make()
    assert a[2].data_ptr() == a[3].data_ptr()
    opt = FusedMuon([{"params": a}], lr=0.01)
    state = {}
    for step in range(1, 4):
        for i, (p, r) in enumerate(zip(a, b)):
            if i == 6 and step == 2:
                p.grad = r.grad = None
                continue
            g = _rand(p.shape, 100 * step + i, 1e-3, dtype).contiguous(
                memory_format=torch.channels_last if p.ndim == 4 else torch.contiguous_format)
            p.grad, r.grad = g.clone(), g.clone()
        opt.step()
        for p in b:
            if p.grad is not None:
                n = state.setdefault(("n", p), 0) + 1
                state[("n", p)] = n
                _chain([p], state, n, 0.01, 0.1)
    for i, (p, r) in enumerate(zip(a, b)):
        assert torch.equal(p.detach(), r.detach()), i


def test_adamw_group_leaves_version_counters(cuda_lib):
    """The branch writes through .data: a graph kept across a step can still run backward."""
    from muon_fused import FusedMuon

    p = torch.nn.Parameter(torch.ones(64, device=DEV))
    loss = (p * p).sum()
    loss.backward(retain_graph=True)
    FusedMuon([p], lr=0.01).step()
    loss.backward()


def test_checkpoint_resumes_bit_for_bit(cuda_lib):
    from muon_fused import FusedMuon

    groups = _groups(torch.bfloat16)
    opt = FusedMuon(groups, lr=LR, adamw_state_dtype=torch.float32)
    _set_grads(groups, 0)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    other = [{**g, "params": [torch.nn.Parameter(p.detach().clone()) for p in g["params"]]}
             for g in groups]
    opt2 = FusedMuon(other, lr=LR, adamw_state_dtype=torch.float32)
    opt2.load_state_dict(saved)
    for gs, o in ((groups, opt), (other, opt2)):
        _set_grads(gs, 1)
        o.step()
    for g, h in zip(groups, other):
        for p, q in zip(g["params"], h["params"]):
            assert torch.equal(p.detach(), q.detach())


def test_mixed_types_of_one_shape_in_a_normed_group(cuda_lib):
    from muon_fused import FusedMuon

    ps = [torch.nn.Parameter(_rand((64, 48), i, 0.02, dt)) for i, dt in
          enumerate([torch.float32, torch.bfloat16, torch.float32])]
    ps.append(torch.nn.Parameter(_rand((64, 12, 2, 2), 3, 0.02)))
    ps.append(torch.nn.Parameter(_rand((48, 64), 4, 0.02).T))  # not contiguous: torch ops
    opt = FusedMuon([{"params": ps, "use_muon": True, "normed_beta2": 0.9}], lr=LR)
    for i, p in enumerate(ps):
        p.grad = _rand(p.shape, 10 + i, 1e-3, p.dtype)
    before = [p.detach().double().clone() for p in ps]
    opt.step()
    for p, p0 in zip(ps, before):
        d = p.detach().double() - p0 * (1 - LR * WD)
        # a normalised update has root mean square 0.2·lr; bf16 weights round by 2^-8 of theirs
        rms = float(d.square().mean().sqrt())
        assert abs(rms - 0.2 * LR) <= 0.02 * 0.2 * LR
        assert opt.state[p]["row_moment"].shape == (p.shape[0],)


@pytest.mark.parametrize("what", ["device", "shape"])
def test_adamw_state_that_no_longer_fits_is_refused(cuda_lib, what):
    """A moment left on the CPU, or of the size that the parameter had before."""
    from muon_fused import FusedMuon

    p = torch.nn.Parameter(_rand((64, 16), 1, 0.02))
    q = torch.nn.Parameter(_rand((33,), 2, 0.02))
    opt = FusedMuon([{"params": [p, q]}])
    for x in (p, q):
        x.grad = _rand(x.shape, 3, 1e-3)
    opt.step()
    state = opt.state[p]
    if what == "device":
        state["moment2"] = state["moment2"].cpu()
    else:
        state["moment1"] = state["moment1"][:32].clone()
    with pytest.raises(RuntimeError):
        opt.step()


def test_adamw_launch_checks_what_it_cannot_take(cuda_lib):
    from muon_fused.step_ops import adamw_launch

    p, g, m, v = (_rand((64,), i, 1.0) for i in range(4))
    for bad in ([p], [g], [m], [v.cpu()]), ([p], [g], [m], [v[:32]]), ([p], [g[::2]], [m], [v]):
        with pytest.raises(RuntimeError):
            adamw_launch(*bad, [-0.1], 0.1, 0.0, (0.9, 0.95), 1e-8)
    assert torch.equal(p, _rand((64,), 0, 1.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_with_the_negative_bit(cuda_lib, dtype):
    """A contiguous gradient that torch negates in the view gives what its values give, in
    every kind of group."""
    from muon_fused import FusedMuon

    results = []
    for negate in (torch.neg, torch._neg_view):
        groups = _groups(dtype)
        opt = FusedMuon(groups, lr=LR)
        for step in range(2):
            _set_grads(groups, step)
            for g in groups:
                for p in g["params"]:
                    p.grad = negate(p.grad)
                    assert p.grad.is_neg() == (negate is torch._neg_view) and p.grad.is_contiguous()
            opt.step()
        results.append([p.detach() for g in groups for p in g["params"]])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_adamw_tensors_that_share_memory(cuda_lib):
    """Tied storage of which the kernel takes one view only, gradients that are a parameter's
    or a moment's own memory, a moment used twice: the values of the torch ops in the group's
    order, bit for bit."""
    from muon_fused import FusedMuon

    def make():
        w = _rand((24, 40), 1, 0.02)
        flat = _rand((64,), 2, 0.02)
        ts = [w, w.T, _rand((30,), 3, 0.02), w[:, ::2], flat[:32], _rand((5,), 4, 0.02, torch.bfloat16),
              flat[16:48], _rand((7, 3), 5, 0.02)]
        return [torch.nn.Parameter(t) for t in ts]

    def set_grads(ps, step):
        for i, p in enumerate(ps):
            p.grad = _rand(p.shape, 100 * step + i, 1e-3, p.dtype)
        ps[2].grad = ps[2].detach()  # the parameter itself
        ps[4].grad = ps[6].detach()  # the values of another one that is written

    a, b = make(), make()
    opt = FusedMuon([{"params": a}], lr=0.5, wd=0.3)
    state = {}
    for step in (1, 2, 3):
        set_grads(a, step)
        set_grads(b, step)
        opt.step()
        for p in b:
            _chain([p], state, step, 0.5, 0.3)
        if step == 1:  # two parameters of one size that share a moment from here on
            opt.state[a[2]]["moment2"] = opt.state[a[7]]["moment2"].view(-1)[:1].expand(30).clone()
            state[b[2]] = (state[b[2]][0], state[b[7]][1].view(-1)[:1].expand(30).clone())
            opt.state[a[6]]["moment1"] = opt.state[a[4]]["moment1"]
            state[b[6]] = (state[b[4]][0], state[b[6]][1])
    for i, (p, r) in enumerate(zip(a, b)):
        assert torch.equal(p.detach(), r.detach()), i


@pytest.mark.parametrize("dtype,state", [(torch.float32, None), (torch.bfloat16, None),
                                         (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
def test_adamw_group_without_the_extension(cuda_lib, monkeypatch, dtype, state):
    """The torch ops where the kernels cannot run, the same values."""
    from muon_fused import FusedMuon, _lib, step_ops

    def missing():
        raise ImportError("not built")

    a = [torch.nn.Parameter(_rand(s, i, 0.02, dtype)) for i, s in enumerate([(33, 17), (9,), (4, 5, 6)])]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    opts = [FusedMuon([{"params": ps}], lr=0.01, adamw_state_dtype=state) for ps in (a, b)]
    for step in range(2):
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad = _rand(p.shape, 10 * step + i, 1e-3, dtype)
            q.grad = p.grad.clone()
        opts[0].step()
        with monkeypatch.context() as m:
            m.setattr(_lib, "step_ext", missing)
            step_ops.adamw_ready.cache_clear()
            with pytest.warns(RuntimeWarning, match="not built"):
                opts[1].step()
        step_ops.adamw_ready.cache_clear()
    for p, q in zip(a, b):
        assert torch.equal(p.detach(), q.detach())
