"""Workspaces that a kernel must not write through: on the host, or without the bytes that
``nbytes`` promises behind the first one."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
HEADS = [((256, 512), 4, 0, 5), ((512, 256), 4, 1, 5),  # on head x head matrices
         ((256, 16), 2, 0, 5), ((512, 256), 2, 0, 5), ((256, 512), 4, 0, 6)]  # across, batched


def _rand(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)


def _calls():
    """(bytes, call with a workspace) of every entry point that takes one."""
    from muon_fused import (_fused_muon_C as C, fused_newton_schulz, fused_newton_schulz_heads,
                            fused_normed_update, workspace_size, workspace_size_heads)
    from muon_fused.step_ops import normed_workspace_size

    for shape, heads, dim, steps in HEADS:
        G = _rand(shape, 1)
        yield (workspace_size_heads(shape, heads, dim=dim, steps=steps),
               lambda ws, G=G, h=heads, d=dim, s=steps: fused_newton_schulz_heads(G, h, s, ws, dim=d))
    G = _rand((256, 320), 2)
    yield workspace_size(256, 320), lambda ws: fused_newton_schulz(G, workspace=ws)
    B = _rand((3, 128, 192), 3)
    yield C.workspace_size_batched(3, 128, 192), lambda ws: C.fused_newton_schulz_batched(B, 5, ws)
    u = _rand((2, 64, 96), 4)

    def normed(ws):
        ps = [_rand((64, 96), k).float() for k in (5, 6)]
        vs = [torch.ones(64, device=DEV) for _ in ps]
        fused_normed_update(ps, u, vs, lr=0.1, workspace=ws)
        return torch.stack(ps)

    yield normed_workspace_size(2, 64), normed


def test_host_workspaces_are_refused(cuda_lib):
    for need, call in _calls():
        with pytest.raises(RuntimeError, match="workspace must be a CUDA tensor"):
            call(torch.empty(need, dtype=torch.uint8))


def test_workspaces_without_their_bytes_are_replaced(cuda_lib):
    """One byte expanded to many, and every other one of a buffer whose rest is in use."""
    for need, call in _calls():
        want = call(None)
        byte = torch.full((1,), 7, dtype=torch.uint8, device=DEV)
        assert torch.equal(call(byte.expand(need + 256)), want)
        whole = torch.full((2 * need + 512,), 7, dtype=torch.uint8, device=DEV)
        assert torch.equal(call(whole[::2]), want)
        assert bool((whole == 7).all()) and bool((byte == 7).all())
        good = torch.empty(need, dtype=torch.uint8, device=DEV)
        assert torch.equal(call(good), want)
