"""Argument checks of the per-head Newton-Schulz that need no GPU."""

import pytest
import torch

from muon_fused import _lib, fused_newton_schulz_heads, workspace_size_heads


def test_front_door_refusals():
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_newton_schulz_heads(torch.zeros(8, 8), 2)
    with pytest.raises(AssertionError):
        fused_newton_schulz_heads(torch.zeros(8), 2)
    with pytest.raises(RuntimeError, match="divide"):
        workspace_size_heads((10, 8), 3)
    with pytest.raises(RuntimeError, match="dim must be"):
        workspace_size_heads((10, 8), 2, dim=2)
    with pytest.raises(RuntimeError, match="divide"):
        workspace_size_heads((10, 8), 0)


@pytest.mark.parametrize("shape,heads,dim", [((64, 100), 4, 0), ((100, 64), 4, 1), ((3, 254, 9), 2, 0)])
def test_workspace_holds_the_copy_and_the_matrices(shape, heads, dim):
    batch = shape[0] if len(shape) == 3 else 1
    rows, cols = shape[-2:]
    need = workspace_size_heads(shape, heads, dim=dim)
    side = min((rows, cols)[dim] // heads, (rows, cols)[1 - dim])  # the matrices' side
    dp = 64 if side <= 64 else 128
    assert need >= batch * heads * dp * dp * (4 + 4) + 2 * batch * rows * cols
    assert need % 256 == 0


def test_wide_heads_use_the_batched_workspace():
    assert workspace_size_heads((512, 64), 2) == _lib.workspace_bytes_batched(2, 256, 64)
    assert workspace_size_heads((256, 64), 2, steps=9) == _lib.workspace_bytes_batched(2, 128, 64)


def test_c_entry_refuses_before_device_work():
    lib = _lib.load()

    def call(G=0x1000, dtype=0, batch=1, rows=8, cols=8, ld=8, bs=0, heads=2, dim=0, out=0x100000,
             steps=5, ws=0x200000, wsb=1 << 30):
        return lib.fm_newton_schulz_heads(G, dtype, batch, rows, cols, ld, bs, heads, dim, out, steps,
                                          ws, wsb, None)

    for kw, text in (({"G": 0}, b"null"), ({"dtype": 7}, b"dtype"), ({"steps": 9}, b"steps"),
                     ({"steps": -1}, b"steps"), ({"heads": 3}, b"divide"), ({"dim": 2}, b"dim"),
                     ({"rows": 258}, b"wider"), ({"ld": 7}, b"ldg"),
                     ({"batch": 2, "bs": 63}, b"overlap"), ({"ws": 0x200080}, b"aligned"),
                     ({"out": 0x1040}, b"share memory"), ({"ws": 0x100000}, b"share memory"),
                     ({"rows": 140000, "heads": 70000}, b"65535"), ({"rows": 0}, b"positive")):
        assert call(**kw) == _lib.FM_E_INVALID, kw
        assert text in lib.fm_last_error(), kw
    assert call(wsb=64) == _lib.FM_E_WORKSPACE
