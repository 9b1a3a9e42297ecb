"""fused_adamw and fused_normed_update on the GPU: against the torch chain they
replace (bit for bit) and against their formulas in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
LR, WD = 0.01, 0.1
U32 = 2.0 ** -24  # half a step of fp32, relative


def _rand(shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _adam_state(shapes, dtype, mdtype, seed=0):
    st = [], [], [], []
    for i, s in enumerate(shapes):
        st[0].append(_rand(s, seed + 4 * i, 0.02, dtype))
        st[1].append(_rand(s, seed + 4 * i + 1, 1e-3, dtype))
        st[2].append(_rand(s, seed + 4 * i + 2, 3e-4, mdtype))
        st[3].append((_rand(s, seed + 4 * i + 3, 1e-3).square() + 1e-8).to(mdtype))
    return st


def _torch_chain(p, g, m, v, step, lr, wd, betas, eps):
    """The optimizer's torch ops (reference muon_fused/optimizer.py:185-200)."""
    m.lerp_(g, 1 - betas[0])
    v.lerp_(g.square(), 1 - betas[1])
    u = m / (eps + v.sqrt())
    scale = (1 - betas[0] ** step) / (1 - betas[1] ** step) ** 0.5
    p.mul_(1 - lr * wd)
    p.add_(u, alpha=-lr / scale)


def _same(x, y):
    """Equal values; a NaN equals a NaN (in fp16 the chain's eps of 1e-8 rounds
    to zero, so 0/0 arises where a gradient's square underflows)."""
    return torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(0.0), y.nan_to_num(0.0))


SHAPES = [(1,), (7,), (4096,), (2049, 3), (2, 3, 5), (0,), (65537,), (64, 2048)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("betas,eps", [((0.9, 0.95), 1e-8), ((0.4, 0.3), 1e-6), ((0.0, 0.5), 1e-4)])
def test_adamw_equals_torch_chain(cuda_lib, dtype, betas, eps):
    """Moments of the parameter's type: every value of two steps is the torch
    chain's, on both branches of lerp (weight below and from 0.5)."""
    from muon_fused import fused_adamw

    a = _adam_state(SHAPES, dtype, dtype)
    b = [[t.clone() for t in ts] for ts in a]
    for step in (1, 2):
        fused_adamw(*a, step, lr=LR, wd=WD, betas=betas, eps=eps)
        for p, g, m, v in zip(*b):
            _torch_chain(p, g, m, v, step, LR, WD, betas, eps)
    for xs, ys in zip(a, b):
        for x, y in zip(xs, ys):
            assert _same(x, y), (int((x != y).sum()), int(x.isnan().sum()))


def _adam64(p, g, m, v, step, lr, wd, betas, eps):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    m = m + (1 - betas[0]) * (g - m)
    v = v + (1 - betas[1]) * (g * g - v)
    u = lr * (1 - betas[1] ** step) ** 0.5 / (1 - betas[0] ** step) * m / (eps + v.sqrt())
    return p * (1 - lr * wd) - u, m, v, u


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step", [1, 1000])
def test_adamw_fp32_moments_against_64_bits(cuda_lib, dtype, step):
    """m and v: g - m, the product and the sum, each operand at most |g| + |m|
    (or g² + v): 4 roundings of it, and the weight's own.  p: 10 roundings (m,
    v's root, eps, quotient, decay, alpha and their constants) of the update, 3
    of p, then half a step of p's type; fp16 results may be subnormal, whose
    step is 2^-24."""
    from muon_fused import fused_adamw

    st = _adam_state(SHAPES, dtype, torch.float32, seed=50)
    refs = [_adam64(*x, step, LR, WD, (0.9, 0.95), 1e-8) for x in zip(*st)]
    old = [[t.clone() for t in ts] for ts in st]
    fused_adamw(*st, [step] * len(SHAPES), lr=LR, wd=WD)
    half = torch.finfo(dtype).eps / 2
    for i, (rp, rm, rv, ru) in enumerate(refs):
        p0, g0, m0, v0 = (t[i].double() for t in old)
        assert ((st[2][i].double() - rm).abs() <= 6 * U32 * (g0.abs() + m0.abs())).all()
        assert ((st[3][i].double() - rv).abs() <= 6 * U32 * (g0 * g0 + v0)).all()
        # m's absolute error reaches u through m/(eps + sqrt v)
        um = ru.abs() * (g0.abs() + m0.abs()) / rm.abs().clamp_min(1e-300)
        fp32 = U32 * (10 * ru.abs() + 6 * um + 6 * ru.abs() * (g0 * g0 + v0) / rv + 3 * p0.abs())
        tol = fp32 + (half * (rp.abs() + fp32) if dtype != torch.float32 else 0.0)
        tol = tol + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert ((st[0][i].double() - rp).abs() <= tol).all(), i


def test_adamw_mixed_types_views_and_long_lists(cuda_lib):
    """700 tensors of three types in one call (past one launch's table), some
    of them views whose data starts off a 16-byte boundary: equal to one call
    per tensor, each on aligned copies."""
    from muon_fused import fused_adamw

    st = [], [], [], []
    for i in range(700):
        dt = (torch.float32, torch.bfloat16, torch.float16)[i % 3]
        off = i % 4
        n = 1 + (i * 37) % 3000
        for k, ts in enumerate(_adam_state([(n + off,)], dt, torch.float32 if i % 2 else dt, seed=4 * i)):
            st[k].append(ts[0][off:])
    alone = [[t.clone() for t in ts] for ts in st]
    fused_adamw(*st, [1 + i % 5 for i in range(700)], lr=LR, wd=WD)
    for i in range(700):
        fused_adamw(*[[ts[i]] for ts in alone], 1 + i % 5, lr=LR, wd=WD)
    for xs, ys in zip(st, alone):
        for x, y in zip(xs, ys):
            assert _same(x, y)


def test_adamw_accepts_what_it_documents(cuda_lib):
    """Tuples, parameters, subclasses of tensors and a count per tensor, in the
    plain case (one C++ call) and beside it, give the same values."""
    from muon_fused import fused_adamw

    class Sub(torch.Tensor):
        pass

    st = _adam_state([(33,), (5, 7)], torch.float32, torch.float32)
    want = [[t.clone() for t in ts] for ts in st]
    fused_adamw(*want, [3, 4], lr=LR, wd=WD)
    for wrap in (lambda t: torch.nn.Parameter(t, requires_grad=False), lambda t: t.as_subclass(Sub)):
        got = [[t.clone() for t in ts] for ts in st]
        got[0] = [wrap(t) for t in got[0]]
        fused_adamw(*map(tuple, got), (3, 4), lr=LR, wd=WD)
        for xs, ys in zip(got, want):
            for x, y in zip(xs, ys):
                assert torch.equal(x.detach().as_subclass(torch.Tensor), y)
    with pytest.raises(RuntimeError, match="one per parameter"):
        fused_adamw(*st, [1, 2, 3], lr=LR)
    with pytest.raises(RuntimeError, match="one tensor per parameter"):
        fused_adamw(st[0], st[1][:1], st[2], st[3], 1, lr=LR)


def test_adamw_nonfinite_values_stay_in_place(cuda_lib):
    """inf and NaN gradients give what torch gives, in their elements only."""
    from muon_fused import fused_adamw

    a = _adam_state([(5000,)], torch.float32, torch.float32)
    a[1][0][17], a[1][0][4111], a[1][0][4999] = math.inf, math.nan, -math.inf
    b = [[t.clone() for t in ts] for ts in a]
    fused_adamw(*a, 3, lr=LR, wd=WD)
    _torch_chain(*[ts[0] for ts in b], 3, LR, WD, (0.9, 0.95), 1e-8)
    for xs, ys in zip(a, b):
        assert _same(xs[0], ys[0])


def test_adamw_past_32_bit_offsets(cuda_lib):
    """A tensor of 2^31 + 4099 elements: its end equals the same values alone."""
    from muon_fused import fused_adamw

    n, k = (1 << 31) + 4099, 5000
    dt = torch.bfloat16
    big = [torch.full((n,), x, dtype=dt, device=DEV) for x in (0.5, 1e-3, 1e-4, 1e-6)]
    small = [ts[0] for ts in _adam_state([(k,)], dt, dt, seed=9)]
    for b, s in zip(big, small):
        b[-k:].copy_(s)
    one = [torch.full((8,), x, dtype=dt, device=DEV) for x in (0.5, 1e-3, 1e-4, 1e-6)]
    for xs in (big, small, one):
        fused_adamw(*[[x] for x in xs], 2, lr=LR, wd=WD)
    for b, s, o in zip(big, small, one):
        assert torch.equal(b[-k:], s)
        assert bool((b[:-k] == o[0]).all())


def _normed64(p, u, v, lr, wd, beta2, eps):
    rows = p.shape[0]
    p64, u64 = p.double().reshape(rows, -1), u.double().reshape(rows, -1)
    v64 = beta2 * v.double() + (1 - beta2) * u64.square().mean(1)
    o = u64 / (v64.sqrt() + eps)[:, None]
    step = lr * 0.2 * math.sqrt(u64.numel())
    d = step / (o.norm() + 1e-7) * o
    return (p64 * (1 - lr * wd) - d).reshape(p.shape), v64, d.reshape(p.shape)


NORMED_SHAPES = [(1, 1), (1, 40), (40, 1), (3, 5), (64, 64), (100, 77), (33, 4097), (17, 9001),
                 (64, 32, 3, 3), (2500, 130)]


@pytest.mark.parametrize("shape", NORMED_SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_normed_against_64_bits(cuda_lib, shape, dtype):
    """v: a row's sum of c squares is added in chains of at most c/128 + 60 terms
    (c/1024 past 4096 columns; a lane's chains, then 2 + 5 + 8): that many
    roundings, and 6 for the mean and the mix.  The update: v's error halves in
    the root, F's is no larger, and 12 roundings of their own; p adds 2 and its
    type's half step (fp16 subnormals: 2^-25)."""
    from muon_fused import fused_normed_update

    rows, cols = shape[0], math.prod(shape[1:])
    n = 3
    ps = [_rand(shape, i, 0.02, dtype) for i in range(n)]
    us = _rand((n, rows, cols), 10, 1 / math.sqrt(max(rows, cols)), torch.bfloat16)
    us[1, rows // 2] = 0  # a neuron without an update
    vs = [_rand((rows,), 20 + i, 1.0).square() / max(rows, cols) for i in range(n)]
    refs = [_normed64(p, u, v, LR, WD, 0.95, 1e-8) for p, u, v in zip(ps, us, vs)]
    p0 = [p.double() for p in ps]
    fused_normed_update(ps, us, vs, lr=LR, wd=WD)
    depth = cols / 32 / 4 + 60 if cols <= 4096 else cols / 256 / 4 + 60
    rv_tol = (depth + 6) * U32
    half = torch.finfo(dtype).eps / 2
    for i, (rp, rv, rd) in enumerate(refs):
        assert ((vs[i].double() - rv).abs() <= rv_tol * rv).all()
        fp32 = (2 * rv_tol + 12 * U32 + (rows / 592 + 60) * U32) * rd.abs() + 2 * U32 * p0[i].abs()
        tol = fp32 + half * (rp.abs() + fp32) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert ((ps[i].double() - rp).abs() <= tol).all(), i


def test_normed_zero_update_only_decays(cuda_lib):
    from muon_fused import fused_normed_update

    p = [_rand((32, 48), 0)]
    want = p[0] * (1 - LR * WD)
    v = [torch.zeros(32, device=DEV)]
    fused_normed_update(p, torch.zeros(1, 32, 48, dtype=torch.bfloat16, device=DEV), v, lr=LR, wd=WD)
    assert torch.equal(p[0], want) and not v[0].any()


def test_normed_shared_update_and_refusals(cuda_lib):
    """Two parameters may read one update; nothing written may be given twice."""
    from muon_fused import fused_adamw, fused_normed_update

    u = _rand((8, 16), 3, 0.1, torch.bfloat16)
    a, b = _rand((8, 16), 4), _rand((8, 16), 4)
    va, vb = torch.zeros(8, device=DEV), torch.zeros(8, device=DEV)
    fused_normed_update([a, b], [u, u], [va, vb], lr=LR)
    assert torch.equal(a, b) and torch.equal(va, vb)
    bad = [([a, a], [u, u], [va, vb]), ([a, b], [u, u], [va, va]),
           ([a], [a.view(-1)[:64].view(torch.bfloat16).view(8, 16)], [va])]
    for args in bad:
        with pytest.raises(RuntimeError, match="overlap"):
            fused_normed_update(*args, lr=LR)
    with pytest.raises(RuntimeError, match="one shape and type"):
        fused_normed_update([a, b[:4]], [u, u], [va, vb], lr=LR)
    with pytest.raises(RuntimeError, match="contiguous"):
        fused_normed_update([a.T], [u.view(16, 8)], [torch.zeros(16, device=DEV)], lr=LR)
    with pytest.raises(RuntimeError, match="bf16"):
        fused_normed_update([a], [u.float()], [va], lr=LR)
    with pytest.raises(RuntimeError, match="row_moments"):
        fused_normed_update([a], [u], [va.bfloat16()], lr=LR)
    with pytest.raises(RuntimeError, match="one device"):
        fused_normed_update([a], [u.cpu()], [va], lr=LR)
    z = [torch.zeros(4, device=DEV) for _ in range(4)]
    with pytest.raises(RuntimeError, match="overlap"):
        fused_adamw([z[0], z[0]], z[:2], z[1:3], z[2:], 1, lr=LR)
    with pytest.raises(RuntimeError, match="shapes"):
        fused_adamw([z[0]], [z[1].view(2, 2)], [z[2]], [z[3]], 1, lr=LR)
    with pytest.raises(RuntimeError, match="one type"):
        fused_adamw([z[0]], [z[1].double()], [z[2]], [z[3]], 1, lr=LR)
    with pytest.raises(RuntimeError, match="moments"):
        fused_adamw([z[0]], [z[1]], [z[2].half()], [z[3].half()], 1, lr=LR)
    with pytest.raises(RuntimeError, match="contiguous"):
        w = [torch.zeros(4, 2, device=DEV).T for _ in range(4)]
        fused_adamw(*[[x] for x in w], 1, lr=LR)


def test_normed_long_list_views_and_repeatability(cuda_lib):
    """70 matrices (past one launch's table and the L2 grouping) at unaligned
    addresses equal one call per matrix on aligned copies, and a second run."""
    from muon_fused import fused_normed_update

    r, c = 41, 67

    def views(seed):
        ps = [_rand((r * c + 3,), seed + i, 0.02, torch.bfloat16)[i % 4:i % 4 + r * c].view(r, c)
              for i in range(70)]
        us = [_rand((r * c + 7,), seed + 100 + i, 0.1, torch.bfloat16)[i % 8:i % 8 + r * c].view(r, c)
              for i in range(70)]
        return ps, us, [torch.full((r,), 1e-3, device=DEV) for _ in range(70)]

    ps, us, vs = views(0)
    fused_normed_update(ps, us, vs, lr=LR, wd=WD)
    again = views(0)
    fused_normed_update(*again, lr=LR, wd=WD)
    for i, (p, u, v) in enumerate(zip(*views(0))):
        p, u = p.clone(), u.clone()
        fused_normed_update([p], [u], [v], lr=LR, wd=WD)
        assert torch.equal(ps[i], again[0][i]) and torch.equal(vs[i], again[2][i])
        # row sums start at another 16-byte boundary, so they may round differently
        torch.testing.assert_close(vs[i], v, rtol=1e-5, atol=0)
        torch.testing.assert_close(ps[i].float(), p.float(), rtol=2 * 2.0 ** -8, atol=1e-9)


def test_normed_past_32_bit_offsets(cuda_lib):
    """A (33, 2^26) matrix (2^31 + 2^26 elements): its last rows against 64 bits."""
    from muon_fused import fused_normed_update

    rows, cols = 33, 1 << 26
    p = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    u = torch.full((rows, cols), 2.0 ** -13, dtype=torch.bfloat16, device=DEV)
    u[-1] = 2.0 ** -12
    v = torch.zeros(rows, device=DEV)
    fused_normed_update([p], [u], [v], lr=1.0, wd=0.0, beta2=0.75)
    # v_i = u²/4, r_i u = 2 (up to eps) for every row: the whole update is 0.2
    want = torch.tensor(-0.2).bfloat16().item()
    step = 2.0 ** -10
    assert float((p[0].float() - want).abs().max()) <= step
    assert float((p[-1].float() - want).abs().max()) <= step
    torch.testing.assert_close(v[-1].item(), 2.0 ** -26, rtol=1e-5, atol=0)


def test_step_ops_on_a_side_stream_and_in_a_graph(cuda_lib):
    from muon_fused import fused_adamw, fused_normed_update

    a = _adam_state([(3000,), (17, 9)], torch.float32, torch.float32)
    b = [[t.clone() for t in ts] for ts in a]
    p, u, v = _rand((64, 96), 1, 0.02), _rand((1, 64, 96), 2, 0.1, torch.bfloat16), torch.zeros(64, device=DEV)
    p2, v2 = p.clone(), v.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        fused_adamw(*a, 1, lr=LR, wd=WD)
        fused_normed_update([p], u, [v], lr=LR, wd=WD)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        fused_adamw(*a, 1, lr=LR, wd=WD)
        fused_normed_update([p], u, [v], lr=LR, wd=WD)
    for _ in range(2):
        graph.replay()
    for _ in range(3):
        fused_adamw(*b, 1, lr=LR, wd=WD)
        fused_normed_update([p2], u, [v2], lr=LR, wd=WD)
    torch.cuda.synchronize()
    for xs, ys in zip(a, b):
        for x, y in zip(xs, ys):
            assert torch.equal(x, y)
    assert torch.equal(p, p2) and torch.equal(v, v2)


def test_inference_tensors(cuda_lib):
    from muon_fused import fused_adamw, fused_normed_update

    with torch.inference_mode():
        st = _adam_state([(9,)], torch.float32, torch.float32)
        p, u, v = _rand((4, 8), 0), _rand((1, 4, 8), 1, 0.1, torch.bfloat16), torch.zeros(4, device=DEV)
        want = [[t.clone() for t in ts] for ts in st]
        fused_adamw(*st, 1, lr=LR)
        fused_normed_update([p], u, [v], lr=LR)
    _torch_chain(*[ts[0].clone() for ts in want], 1, LR, 0.1, (0.9, 0.95), 1e-8)
    assert bool(v.all()) and not torch.equal(st[0][0], want[0][0])


def test_writes_are_seen_by_autograd(cuda_lib):
    """A backward through a value saved before the step fails instead of using the new one."""
    from muon_fused import fused_adamw

    p = torch.nn.Parameter(torch.ones(8, device=DEV))
    loss = (p * p).sum()
    z = torch.zeros(8, device=DEV)
    with torch.no_grad():
        fused_adamw([p], [torch.ones(8, device=DEV)], [z.clone()], [z.clone()], 1, lr=LR)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("beta2", [0.9, 0.999, 0.9999])
def test_normed_row_moment_of_slow_decays(cuda_lib, beta2):
    """v takes (1 - beta2) of a row's mean square, with the weight rounded once: from v = 0
    the result is the mean square (cols/128 + 60 sums at most, and 6 roundings for the mean,
    the weight and the mix) and no more, and so after 30 steps of it."""
    from muon_fused import fused_normed_update

    rows, cols = 40, 96
    u = _rand((1, rows, cols), 3, 0.1, torch.bfloat16)
    p, v = _rand((rows, cols), 4, 0.02), torch.zeros(rows, device=DEV)
    v64 = torch.zeros(rows, device=DEV, dtype=torch.float64)
    for step in range(1, 31):
        fused_normed_update([p], u, [v], lr=LR, wd=WD, beta2=beta2)
        v64 = beta2 * v64 + (1 - beta2) * u[0].double().square().mean(1)
        # a step's own roundings, and beta2's and the sum's for each step before
        tol = (cols / 128 + 60 + 6 + 2 * step) * U32
        assert ((v.double() - v64).abs() <= tol * v64).all(), step


def test_normed_refuses_negative_views(cuda_lib):
    """Torch's negative bit is in the view, not in memory, which is what the kernels use."""
    from muon_fused import fused_normed_update

    neg = torch._neg_view
    p, u, v = _rand((8, 16), 1), _rand((1, 8, 16), 2, 0.1, torch.bfloat16), torch.ones(8, device=DEV)
    for args in ([neg(p)], u, [v]), ([p], neg(u), [v]), ([p], [neg(u[0])], [v]), ([p], u, [neg(v)]):
        with pytest.raises(RuntimeError, match="negative"):
            fused_normed_update(*args, lr=LR)
    assert torch.equal(p, _rand((8, 16), 1)) and bool((v == 1).all())


def test_adamw_mixed_types_are_checked_together(cuda_lib):
    """Tensors of different kinds that share memory are refused before anything is written;
    where a call is good, autograd sees the writes of every kind."""
    from muon_fused import fused_adamw

    st = [a + b + c for a, b, c in zip(*(_adam_state([(64,)], dt, torch.float32, seed=k) for k, dt in
                                         enumerate((torch.float32, torch.bfloat16, torch.float16))))]
    before = [[t.clone() for t in ts] for ts in st]
    versions = [[t._version for t in ts] for ts in st]
    bad = [list(ts) for ts in st]
    bad[0][1] = st[2][0].view(torch.bfloat16)[:64]  # a bf16 parameter in an fp32 moment
    read = [list(ts) for ts in st]
    read[1][2] = st[0][0].view(torch.float16)[64:]  # an fp16 gradient in an fp32 parameter
    same = [list(ts) for ts in st]
    same[2][2] = same[3][2]  # wrong within the last kind only
    for args in (bad, read, same):
        with pytest.raises(RuntimeError, match="overlap"):
            fused_adamw(*args, 1, lr=LR)
    for xs, ys, vs in zip(st, before, versions):
        for x, y, v in zip(xs, ys, vs):
            assert torch.equal(x, y) and x._version == v
    fused_adamw(*st, 1, lr=LR)
    for k, (xs, vs) in enumerate(zip(st, versions)):
        for x, v in zip(xs, vs):
            assert (x._version > v) == (k != 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mdtype", ["own", torch.float32])
def test_values_of_inference_tensors(cuda_lib, dtype, mdtype):
    """Inference tensors leave the one-call route for the checked one: every value is that of
    ordinary tensors, which the other tests hold against the chain and the formulas."""
    from muon_fused import fused_adamw, fused_normed_update

    mt = dtype if mdtype == "own" else mdtype
    plain = _adam_state(SHAPES, dtype, mt, seed=30)
    chain = [[t.clone() for t in ts] for ts in plain]
    rows, cols, n = 37, 129, 3
    ps = [_rand((rows, cols), i, 0.02, dtype) for i in range(n)]
    us = _rand((n, rows, cols), 10, 0.1, torch.bfloat16)
    vs = [_rand((rows,), 20 + i, 0.1).square() for i in range(n)]
    with torch.inference_mode():
        inf = [[t.clone() for t in ts] for ts in plain]
        ps2, us2, vs2 = [p.clone() for p in ps], us.clone(), [v.clone() for v in vs]
        assert all(t.is_inference() for ts in (*inf, ps2, [us2], vs2) for t in ts)
        for step in (1, 2):
            fused_adamw(*inf, step, lr=LR, wd=WD)
            fused_normed_update(ps2, us2, vs2, lr=LR, wd=WD)
    for step in (1, 2):
        fused_adamw(*plain, step, lr=LR, wd=WD)
        fused_normed_update(ps, us, vs, lr=LR, wd=WD)
        if mt == dtype:
            for p, g, m, v in zip(*chain):
                _torch_chain(p, g, m, v, step, LR, WD, (0.9, 0.95), 1e-8)
    for xs, ys, zs in zip(inf, plain, chain if mt == dtype else plain):
        for x, y, z in zip(xs, ys, zs):
            assert _same(x, y) and _same(x, z)
    for x, y in zip(ps2 + vs2, ps + vs):
        assert torch.equal(x, y)
