"""fused_newton_schulz_heads on the GPU against its definition in 64 bits.

Tolerances.  The output's own rounding is half a bf16 step, 2^-8 of each value,
so at most 2^-8 in the Frobenius norm.  Before it: A and Q carry 22 bits, and an
error of A relative to a small eigenvalue grows by 3.4445² a step, 2^-22·11.9^4 =
5e-3 at worst in directions that start at 1e-4 of the largest, which hold a
small part of the norm; Q enters the last product with 17 bits, 2^-17·3.4445^5 =
4e-3 of such a direction again.  Together under 1e-3 of the whole norm: gate
2^-8 + 1e-3.  Single elements: their rounding, and 4e-3 of the largest value.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
A, B, C = 3.4445, -4.7750, 2.0315
FRO = 2.0 ** -8 + 1e-3


def ref64(G, heads, steps, dim):
    g = (G if G.dim() == 3 else G[None]).double()
    x = torch.stack(g.chunk(heads, 1 + dim), 1)
    x = x / (x.flatten(2).norm(dim=2)[..., None, None] + 1e-7)
    for _ in range(steps):
        a = x @ x.mT if dim == 0 else x.mT @ x
        p = B * a + C * (a @ a)
        x = A * x + (p @ x if dim == 0 else x @ p)
    return torch.cat(x.unbind(1), 1 + dim).reshape(G.shape)


def check(out, G, heads, steps, dim, fro=FRO, elem=4e-3):
    assert out.dtype == torch.bfloat16 and out.shape == G.shape
    ref = ref64(G, heads, steps, dim)
    diff = out.double() - ref
    blocks = torch.stack((diff if diff.dim() == 3 else diff[None]).chunk(heads, 1 + dim), 1)
    rblocks = torch.stack((ref if ref.dim() == 3 else ref[None]).chunk(heads, 1 + dim), 1)
    rel = blocks.flatten(2).norm(dim=2) / rblocks.flatten(2).norm(dim=2).clamp_min(1e-30)
    assert float(rel.max()) <= fro, (float(rel.max()), int(rel.argmax()))
    big = float(ref.abs().max())
    assert bool((diff.abs() <= 2.0 ** -8 * ref.abs() + elem * big).all()), float(diff.abs().max()) / big


def rand(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.mark.parametrize("d,n", [(128, 512), (64, 512), (128, 4096), (64, 64), (96, 200), (16, 72),
                                 (8, 1024), (128, 8), (72, 1000), (32, 2304), (112, 65)])
@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_aligned(cuda_lib, d, n, dim, dtype):
    from muon_fused import fused_newton_schulz_heads

    heads = 5
    shape = (heads * d, n) if dim == 0 else (n, heads * d)
    G = rand(shape, d + n, dtype)
    check(fused_newton_schulz_heads(G, heads, dim=dim), G, heads, 5, dim)


@pytest.mark.parametrize("d,n", [(1, 1), (1, 130), (3, 1), (37, 129), (65, 333), (127, 1001), (100, 7)])
@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_odd_sizes(cuda_lib, d, n, dim, dtype):
    """Rows, heads and outputs off 16-byte boundaries (copied input, plain stores)."""
    from muon_fused import fused_newton_schulz_heads

    heads = 3
    shape = (2, heads * d, n) if dim == 0 else (2, n, heads * d)
    G = rand(shape, d * n, dtype)
    check(fused_newton_schulz_heads(G, heads, dim=dim), G, heads, 5, dim)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("dim", [0, 1])
def test_wide_types_are_rounded_to_bf16_first(cuda_lib, dtype, dim):
    from muon_fused import fused_newton_schulz_heads

    G = rand((256, 192), 3, dtype)
    out = fused_newton_schulz_heads(G, 2, dim=dim)
    assert torch.equal(out, fused_newton_schulz_heads(G.bfloat16(), 2, dim=dim))


@pytest.mark.parametrize("steps", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("d", [48, 128])
def test_steps(cuda_lib, steps, d):
    from muon_fused import fused_newton_schulz_heads

    for dim in (0, 1):
        G = rand((4 * d, 1024) if dim == 0 else (1024, 4 * d), steps)
        check(fused_newton_schulz_heads(G, 4, steps, dim=dim), G, 4, steps, dim)


@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("kind", ["cond1e2", "cond1e5", "rank8", "momentum"])
def test_ill_conditioned_heads(cuda_lib, kind, dim):
    """Where the bf16 iteration is off by 5 to 50 %."""
    from muon_fused import fused_newton_schulz_heads

    heads, d, n = 4, 128, 1024
    gen = torch.Generator().manual_seed(1)
    blocks = []
    for _ in range(heads):
        if kind.startswith("cond"):
            u = torch.linalg.qr(torch.randn(d, d, generator=gen))[0]
            v = torch.linalg.qr(torch.randn(n, d, generator=gen))[0]
            x = (u * torch.logspace(0, -math.log10(float(kind[4:])), d)) @ v.T
        elif kind == "rank8":
            x = torch.randn(d, 8, generator=gen) @ torch.randn(8, n, generator=gen)
        else:
            s = 4.0 / torch.arange(1, 17)
            x = 1e-3 * (torch.randn(d, n, generator=gen)
                        + (torch.randn(d, 16, generator=gen) * s) @ torch.randn(16, n, generator=gen))
        blocks.append(x)
    G = torch.cat(blocks).bfloat16().to(DEV)
    G = G if dim == 0 else G.T.contiguous()
    check(fused_newton_schulz_heads(G, heads, dim=dim), G, heads, 5, dim)


@pytest.mark.parametrize("dim", [0, 1])
def test_scales_of_the_input(cuda_lib, dim):
    """Gradients from 1e-10 to 1e4, a head of zeros among them."""
    from muon_fused import fused_newton_schulz_heads

    scale = torch.tensor([1e-10, 1e-5, 0.0, 1.0, 1e4], device=DEV).repeat_interleave(64)
    G = rand((320, 512), 2, torch.float32) * scale[:, None]
    G = (G if dim == 0 else G.T.contiguous()).bfloat16()
    out = fused_newton_schulz_heads(G, 5, dim=dim)
    check(out, G, 5, 5, dim)
    assert not out.narrow(dim, 128, 64).any()


@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nonfinite_stays_in_its_head(cuda_lib, dim, bad):
    from muon_fused import fused_newton_schulz_heads

    G = rand((3 * 80, 256), 5) if dim == 0 else rand((256, 3 * 80), 5)
    clean = fused_newton_schulz_heads(G, 3, dim=dim)
    G2 = G.clone()
    G2.narrow(dim, 80, 80)[3, 5] = bad
    out = fused_newton_schulz_heads(G2, 3, dim=dim)
    for h in range(3):
        got = out.narrow(dim, 80 * h, 80)
        if h == 1:
            assert bool(got.isnan().all())
        else:
            assert torch.equal(got, clean.narrow(dim, 80 * h, 80))


@pytest.mark.parametrize("dim", [0, 1])
def test_strides_batches_and_views(cuda_lib, dim):
    """Row strides beyond the columns, batch strides, transposed inputs and
    unaligned bases give what a contiguous copy gives."""
    from muon_fused import fused_newton_schulz_heads

    base = rand((3, 300, 400), 7)
    views = [base[:, :256, :384], base[:, 4:260, 8:392], base[::2, :256, 3:387],
             base.transpose(1, 2)[:, :384, :256].transpose(1, 2)[:, :256, :384], base[1, :256, :384]]
    for v in views:
        want = fused_newton_schulz_heads(v.contiguous(), 4, dim=dim)
        assert torch.equal(fused_newton_schulz_heads(v, 4, dim=dim), want)
        check(want, v, 4, 5, dim)


def test_batch_equals_single_calls_bit_for_bit_without_splits(cuda_lib):
    """200 heads fill the GPU without splitting the long side, as does one head
    of 256 columns: same order of sums, same bits; and runs repeat."""
    from muon_fused import fused_newton_schulz_heads

    G = rand((50, 4 * 64, 256), 8)
    out = fused_newton_schulz_heads(G, 4)
    assert torch.equal(out, fused_newton_schulz_heads(G, 4))
    for b in (0, 17, 49):
        assert torch.equal(out[b], fused_newton_schulz_heads(G[b], 4))


def test_many_heads_across_waves(cuda_lib):
    from muon_fused import fused_newton_schulz_heads

    for dim in (0, 1):
        G = rand((6, 64 * 32, 192) if dim == 0 else (6, 192, 64 * 32), 9)
        check(fused_newton_schulz_heads(G, 64, dim=dim), G, 64, 5, dim)


@pytest.mark.parametrize("heads", [1, 18, 20, 24, 29, 37, 49, 74, 75])
def test_every_split_of_the_long_side(cuda_lib, heads):
    """148 // heads splits, 8 at most, at least 256 elements each: cluster sizes 8 to 1."""
    from muon_fused import fused_newton_schulz_heads

    for n in (2048, 1900):
        G = rand((heads * 24, n), heads)
        check(fused_newton_schulz_heads(G, heads), G, heads, 5, 0)


@pytest.mark.parametrize("d,n", [(128, 65536), (64, 200001)])
def test_long_sides(cuda_lib, d, n):
    from muon_fused import fused_newton_schulz_heads

    G = rand((2 * d, n), 1)
    check(fused_newton_schulz_heads(G, 2), G, 2, 5, 0)
    T = G.T.contiguous()
    check(fused_newton_schulz_heads(T, 2, dim=1), T, 2, 5, 1)


def test_two_calls_at_once(cuda_lib):
    """Calls that overlap on two streams, with their own workspaces."""
    from muon_fused import fused_newton_schulz_heads

    Gs = [rand((16 * 128, 1024), s) for s in (1, 2)]
    want = [fused_newton_schulz_heads(G, 16) for G in Gs]
    streams = [torch.cuda.Stream() for _ in Gs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(fused_newton_schulz_heads(Gs[k], 16))
    torch.cuda.synchronize()
    for k in range(2):
        for o in got[k]:
            assert torch.equal(o, want[k])


@pytest.mark.parametrize("dim", [0, 1])
def test_wide_heads_run_as_a_batch(cuda_lib, dim):
    """Heads of 256: the bf16 path's accuracy (1e-2, as its own tests)."""
    from muon_fused import fused_newton_schulz_heads

    G = rand((512, 1024) if dim == 0 else (1024, 512), 10)
    out = fused_newton_schulz_heads(G, 2, dim=dim)
    ref = ref64(G, 2, 5, dim)
    assert float((out.double() - ref).norm() / ref.norm()) <= 1e-2
    buf = torch.empty_like(G)
    assert fused_newton_schulz_heads(G, 2, dim=dim, out=buf) is buf and torch.equal(buf, out)


def test_past_32_bit_offsets(cuda_lib):
    """Five projections of 128 x 2^22 (2.7e9 elements): the last one's values."""
    from muon_fused import fused_newton_schulz_heads

    n = 1 << 22
    G = torch.zeros(5, 128, n, dtype=torch.bfloat16, device=DEV)
    G[4, :, -128:] = rand((128, 128), 11)
    out = fused_newton_schulz_heads(G, 1)
    assert not out[:4].any() and not out[4, :, :-128].any()
    check(out[4, :, -128:].contiguous(), G[4, :, -128:].contiguous(), 1, 5, 0)


def test_workspace_out_stream_and_refusals(cuda_lib):
    from muon_fused import fused_newton_schulz_heads, workspace_size_heads

    G = rand((256, 512), 12)
    want = fused_newton_schulz_heads(G, 4)
    ws = torch.empty(workspace_size_heads(G.shape, 4), dtype=torch.uint8, device=DEV)
    out = torch.full((256, 512), 7.0, dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fused_newton_schulz_heads(G, 4, workspace=ws, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert got is out and torch.equal(out, want)
    small = torch.empty(16, dtype=torch.uint8, device=DEV)
    assert torch.equal(fused_newton_schulz_heads(G, 4, workspace=small), want)
    with pytest.raises(RuntimeError, match="share memory"):
        fused_newton_schulz_heads(G, 4, out=G)
    with pytest.raises(RuntimeError, match="out must be"):
        fused_newton_schulz_heads(G, 4, out=out.float())
    with pytest.raises(RuntimeError, match="divide"):
        fused_newton_schulz_heads(G, 3)
    with pytest.raises(RuntimeError, match="dim must be"):
        fused_newton_schulz_heads(G, 4, dim=2)
    with pytest.raises(RuntimeError, match="steps"):
        fused_newton_schulz_heads(G, 4, -1)
    with pytest.raises(RuntimeError, match="dtype"):
        fused_newton_schulz_heads(G.int(), 4)
    assert fused_newton_schulz_heads(G[:, :0], 4).shape == (256, 0)


def test_no_device_error(cuda_lib):
    from muon_fused import _lib

    assert _lib.device_error() == 0


@pytest.mark.parametrize("dim", [0, 1])
def test_graph_replay(cuda_lib, dim):
    from muon_fused import fused_newton_schulz_heads

    G = rand((256, 320), 13)
    fused_newton_schulz_heads(G, 4, dim=dim)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused_newton_schulz_heads(G, 4, dim=dim)
    for seed in (14, 15):
        G.copy_(rand((256, 320), seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fused_newton_schulz_heads(G.clone(), 4, dim=dim))


def test_out_bumps_its_version(cuda_lib):
    """A backward pass through values that the call overwrote fails."""
    from muon_fused import fused_newton_schulz_heads

    G = torch.randn(128, 64, device="cuda", dtype=torch.bfloat16)
    for A in (G, G.t().contiguous().t()):  # taken as it is, copied first
        out = torch.empty(128, 64, device="cuda", dtype=torch.bfloat16)
        before = out._version
        fused_newton_schulz_heads(A, 2, out=out)
        assert out._version > before


@pytest.mark.parametrize("shape", [(0, 512, 64), (512, 0), (2, 512, 0)])
def test_empty_wide_heads(cuda_lib, shape):
    from muon_fused import fused_newton_schulz_heads

    G = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
    assert fused_newton_schulz_heads(G, 2).shape == G.shape


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("heads,d,n", [(149, 128, 200), (300, 65, 131)])
def test_more_heads_than_sms(cuda_lib, heads, d, n, steps):
    """Two and three rounds of heads on the GPU; runs repeat."""
    from muon_fused import fused_newton_schulz_heads

    for dim, dtype in ((0, torch.bfloat16), (1, torch.float16)):
        G = rand((heads * d, n) if dim == 0 else (n, heads * d), steps, dtype)
        out = fused_newton_schulz_heads(G, heads, steps, dim=dim)
        check(out, G, heads, steps, dim)
        assert torch.equal(out, fused_newton_schulz_heads(G, heads, steps, dim=dim))


@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("steps", [2, 5])
def test_ill_conditioned_heads_among_many(cuda_lib, dim, steps):
    """Condition 1 to 1e5, rank 8 and a zero head among 160; NaN stays in its head."""
    from muon_fused import fused_newton_schulz_heads

    heads, d, n = 160, 128, 256
    gen = torch.Generator().manual_seed(11)
    u = torch.linalg.qr(torch.randn(heads, d, d, generator=gen))[0]
    v = torch.linalg.qr(torch.randn(heads, n, d, generator=gen))[0]
    s = torch.stack([torch.logspace(0, -5.0 * h / heads, d) for h in range(heads)])
    s[7, 8:] = 0
    s[9] = 0
    blocks = (u * s[:, None]) @ v.mT
    G = blocks.reshape(heads * d, n).bfloat16().to(DEV)
    G = G if dim == 0 else G.T.contiguous()
    out = fused_newton_schulz_heads(G, heads, steps, dim=dim)
    check(out, G, heads, steps, dim)
    assert not bool(out.narrow(dim, 9 * d, d).any())
    G2 = G.clone()
    G2.narrow(dim, 150 * d, d)[3, 5] = math.nan
    out2 = fused_newton_schulz_heads(G2, heads, steps, dim=dim)
    assert bool(out2.narrow(dim, 150 * d, d).isnan().all())
    assert torch.equal(out2.narrow(dim, 0, 150 * d), out.narrow(dim, 0, 150 * d))
    assert torch.equal(out2.narrow(dim, 151 * d, 9 * d), out.narrow(dim, 151 * d, 9 * d))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("dim", [0, 1])
def test_views_of_wide_types(cuda_lib, dtype, dim):
    """Rows on and off 16-byte boundaries, whole and broken chunks of eight."""
    from muon_fused import fused_newton_schulz_heads

    base = rand((3, 300, 404), 12, torch.float32).to(dtype)
    for v in (base[:, :256, :384], base[:, 1:257, 4:388], base[:, :256, 1:385], base[::2, :252, :324],
              base[1, :256, :384], base[0, :1, :400]):
        heads = 4 if dim == 1 or v.shape[-2] > 1 else 1
        out = fused_newton_schulz_heads(v, heads, dim=dim)
        assert torch.equal(out, fused_newton_schulz_heads(v.bfloat16().contiguous(), heads, dim=dim))
        check(out, v.bfloat16(), heads, 5, dim)


@pytest.mark.parametrize("steps", [6, 8])
@pytest.mark.parametrize("dim", [0, 1])
def test_more_steps_run_as_a_batch(cuda_lib, steps, dim):
    """The Gram form would blow up what a head does not span."""
    from muon_fused import fused_newton_schulz, fused_newton_schulz_heads

    G = rand((256, 320) if dim == 0 else (320, 256), 16)
    out = fused_newton_schulz_heads(G, 4, steps, dim=dim)
    for b, o in zip(G.chunk(4, dim), out.chunk(4, dim)):
        ref = ref64(b, 1, steps, dim)
        # two bf16 iterations that differ in nothing but their batch: 2e-2 between them
        assert float((o.double() - ref).norm() / ref.norm()) <= 2e-2
        assert float((o.double() - fused_newton_schulz(b.contiguous(), steps).double()).norm()
                     / ref.norm()) <= 2e-2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("d,n", [(128, 1), (128, 2), (100, 9), (64, 63), (128, 127), (17, 16)])
def test_heads_wider_than_long(cuda_lib, d, n, dim, dtype):
    """The long side is the shorter one: full rank there, so exact up to the rounding."""
    from muon_fused import fused_newton_schulz_heads, workspace_size_heads

    for batch in (None, 3):
        shape = (5 * d, n) if dim == 0 else (n, 5 * d)
        G = rand(shape if batch is None else (batch, *shape), d + n, dtype)
        out = fused_newton_schulz_heads(G, 5, dim=dim)
        check(out, G, 5, 5, dim)
        buf = torch.empty_like(out)
        ws = torch.empty(workspace_size_heads(G.shape, 5, dim=dim), dtype=torch.uint8, device=DEV)
        assert fused_newton_schulz_heads(G, 5, workspace=ws, dim=dim, out=buf) is buf
        assert torch.equal(buf, out)
        with pytest.raises(RuntimeError, match="out must be"):
            fused_newton_schulz_heads(G, 5, dim=dim, out=buf.float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("rank", [1, 2, 4, 8])
def test_low_rank_heads(cuda_lib, rank, dim, dtype):
    """What a head does not span carries rounding of 2^-22 a product from A into Q, there
    times 3.4445 for every step that follows: at most five steps' worth of 3.4445^5 · 2^-22
    · sqrt(d) against singular values that end at 0.7 or above, beside the output's 2^-8
    (and as much of the largest value in an element, whose row of Q has d such roundings)."""
    from muon_fused import fused_newton_schulz_heads

    heads, d, n = 4, 128, 512
    gen = torch.Generator().manual_seed(rank)
    u = torch.randint(-3, 4, (heads * d, rank), generator=gen).double()  # exact in 16 bits
    v = torch.randint(-3, 4, (rank, n), generator=gen).double()
    G = (u @ v).to(dtype).to(DEV)
    assert torch.equal(G.double().cpu(), u @ v)
    G = G if dim == 0 else G.T.contiguous()
    leak = 5 * A ** 5 * 2.0 ** -22 * d ** 0.5 / 0.7
    check(fused_newton_schulz_heads(G, heads, dim=dim), G, heads, 5, dim, 2.0 ** -8 + leak, leak)


@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("heads,d,n", [(300, 128, 192), (160, 128, 2880), (310, 64, 1048), (600, 64, 176)])
def test_blocks_past_the_end_among_many_heads(cuda_lib, heads, d, n, dim):
    """The last 128 elements of the long side are half or a quarter there, so that some
    warps skip their block of that unit, and every CTA of the output product goes on to the
    next head: the staged blocks of the skipping warps must not be overwritten while a store
    still reads them.  Runs repeat bit for bit."""
    from muon_fused import fused_newton_schulz_heads

    G = rand((heads * d, n) if dim == 0 else (n, heads * d), n)
    out = fused_newton_schulz_heads(G, heads, dim=dim)
    check(out, G, heads, 5, dim)
    for _ in range(20):
        assert torch.equal(out, fused_newton_schulz_heads(G, heads, dim=dim))


@pytest.mark.parametrize("shape,heads,steps", [((128, 256), 2, 5), ((128, 16), 2, 5), ((512, 64), 2, 5),
                                               ((128, 256), 2, 7)])
@pytest.mark.parametrize("dim", [0, 1])
def test_negative_views(cuda_lib, shape, heads, steps, dim):
    """Torch's negative bit is in the view, not in memory: every route takes the values."""
    from muon_fused import fused_newton_schulz, fused_newton_schulz_heads

    G = rand(shape if dim == 0 else shape[::-1], 21)
    neg = torch._neg_view(G)
    assert neg.is_neg() and neg.is_contiguous()
    want = fused_newton_schulz_heads(-G, heads, steps, dim=dim)
    assert torch.equal(fused_newton_schulz_heads(neg, heads, steps, dim=dim), want)
    assert torch.equal(fused_newton_schulz(neg), fused_newton_schulz(-G))
    with pytest.raises(RuntimeError, match="out must be"):
        fused_newton_schulz_heads(G, heads, steps, dim=dim, out=torch._neg_view(want))


@pytest.mark.parametrize("steps", [0, 5, 6])
@pytest.mark.parametrize("d", [40, 200])
def test_one_row_and_repeated_rows(cuda_lib, d, steps):
    """Heads of a single row (or column) on the long side, and inputs whose rows or columns
    are one expanded in memory, on every route: what contiguous copies give."""
    from muon_fused import fused_newton_schulz, fused_newton_schulz_heads

    x = rand((1, 4 * d), d)
    cases = [(x, 4, 1), (x.T, 4, 0), (x.T.contiguous().T, 4, 1), (rand((3, 1, 4 * d), 1), 4, 1),
             (rand((300, 1), 2).expand(300, 4 * d), 4, 1), (rand((1, 300), 3).expand(4 * d, 300), 4, 0),
             (rand((1, 2 * d, 64), 4).expand(3, 2 * d, 64), 2, 0)]
    for G, heads, dim in cases:
        plain = torch.empty(G.shape, dtype=G.dtype, device=DEV).copy_(G)
        out = fused_newton_schulz_heads(G, heads, steps, dim=dim)
        assert torch.equal(out, fused_newton_schulz_heads(plain, heads, steps, dim=dim))
        if G.shape[-1 - dim] == 1:  # a head is a vector v, and its iterates are s_k·v/|v|
            for h, o in zip(plain.double().chunk(heads, -2 + dim), out.double().chunk(heads, -2 + dim)):
                s = 1.0
                for _ in range(steps):
                    s = A * s + B * s ** 3 + C * s ** 5
                want = s * h / h.flatten(-2).norm(dim=-1)[..., None, None]
                # the bf16 path rounds every iterate, A and the factor: 1e-2 as in its own tests
                assert float((o - want).norm()) <= 1e-2 * float(want.norm())
        if G.dim() == 2:
            assert torch.equal(fused_newton_schulz(G, steps), fused_newton_schulz(plain, steps))
