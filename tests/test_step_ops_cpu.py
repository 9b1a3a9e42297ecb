"""Argument checks of the step operators that need no GPU."""

import pytest
import torch

from muon_fused import _lib, fused_adamw, fused_normed_update


def _four(**kw):
    return [[torch.zeros(4, **kw)] for _ in range(4)]


def test_public_names():
    import muon_fused

    assert {"fused_adamw", "fused_normed_update"} <= set(muon_fused.__all__)


def test_adamw_refusals():
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_adamw(*_four(), 1, lr=0.1)
    with pytest.raises(RuntimeError, match="list of tensors"):
        fused_adamw(torch.zeros(4), *_four()[1:], 1, lr=0.1)
    with pytest.raises(RuntimeError, match="one tensor per parameter"):
        fused_adamw(_four()[0], [], *_four()[2:], 1, lr=0.1)
    with pytest.raises(RuntimeError, match="steps"):
        fused_adamw(*_four(), 0, lr=0.1)
    with pytest.raises(RuntimeError, match="steps"):
        fused_adamw(*_four(), [1, 2], lr=0.1)
    with pytest.raises(RuntimeError, match="betas"):
        fused_adamw(*_four(), 1, lr=0.1, betas=(1.0, 0.9))
    fused_adamw([], [], [], [], 1, lr=0.1)  # an empty list is nothing to do


def test_normed_refusals():
    p, u, v = torch.zeros(4, 6), torch.zeros(1, 4, 6, dtype=torch.bfloat16), torch.zeros(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_normed_update([p], u, [v], lr=0.1)
    with pytest.raises(RuntimeError, match="list of tensors"):
        fused_normed_update(p, u, [v], lr=0.1)
    with pytest.raises(RuntimeError, match="beta2"):
        fused_normed_update([p], u, [v], lr=0.1, beta2=1.0)
    with pytest.raises(RuntimeError, match="one tensor per parameter"):
        fused_normed_update([p, p], u, [v, v], lr=0.1)
    fused_normed_update([], [], [], lr=0.1)


def test_c_entries_refuse_before_device_work():
    lib = _lib.load()
    t = _lib.ADAMW_TENSOR.pack(256, 256, 256, 0, 8, -0.1)
    assert lib.fm_adamw(t, 1, _lib.FM_DT_F32, _lib.FM_DT_F32, 1, 0.1, 0.1, 1e-8, None) == _lib.FM_E_INVALID
    assert b"null" in lib.fm_last_error()
    t = _lib.ADAMW_TENSOR.pack(256, 256, 256, 256, -8, -0.1)
    assert lib.fm_adamw(t, 1, _lib.FM_DT_F32, _lib.FM_DT_F32, 1, 0.1, 0.1, 1e-8, None) == _lib.FM_E_INVALID
    assert lib.fm_adamw(t, 1, _lib.FM_DT_F64, _lib.FM_DT_F64, 1, 0.1, 0.1, 1e-8, None) == _lib.FM_E_INVALID
    assert b"dtype" in lib.fm_last_error()
    assert lib.fm_adamw(t, 1, _lib.FM_DT_F32, _lib.FM_DT_BF16, 1, 0.1, 0.1, 1e-8, None) == _lib.FM_E_INVALID
    assert lib.fm_adamw(None, 1, _lib.FM_DT_F32, _lib.FM_DT_F32, 1, 0.1, 0.1, 1e-8, None) == _lib.FM_E_INVALID
    assert lib.fm_adamw(None, 0, _lib.FM_DT_F32, _lib.FM_DT_F32, 1, 0.1, 0.1, 1e-8, None) == _lib.FM_OK
    m = _lib.NORMED_MATRIX.pack(256, 256, 256)
    args = (1, 4, 8, _lib.FM_DT_F32, 1, 0.1, 0.95, 1e-8)
    assert lib.fm_muon_apply_normed(m, *args, 256, 16, None) == _lib.FM_E_WORKSPACE
    assert lib.fm_muon_apply_normed(m, *args, 128, 1 << 20, None) == _lib.FM_E_INVALID
    assert lib.fm_muon_apply_normed(m, 1, 4, 8, _lib.FM_DT_F64, 1, 0.1, 0.95, 1e-8, 256, 1 << 20,
                                    None) == _lib.FM_E_INVALID
    assert lib.fm_muon_apply_normed(_lib.NORMED_MATRIX.pack(256, 0, 256), *args, 256, 1 << 20,
                                    None) == _lib.FM_E_INVALID


def test_c_entries_refuse_overlapping_memory():
    lib = _lib.load()

    def adam(*rows):
        return lib.fm_adamw(b"".join(_lib.ADAMW_TENSOR.pack(*r) for r in rows), len(rows),
                            _lib.FM_DT_F32, _lib.FM_DT_F32, 1, 0.1, 0.1, 1e-8, None)

    ok = (0x1000, 0x2000, 0x3000, 0x4000, 8, -0.1)
    for bad in [(0x1000, 0x2000, 0x3000, 0x4000, 8, -0.1),  # the same tensor twice
                (0x5000, 0x6000, 0x401C, 0x7000, 8, -0.1),  # starts in the last element
                (0x5000, 0x3010, 0x6000, 0x7000, 8, -0.1),  # a gradient inside a moment
                (0x5000, 0x6000, 0x6004, 0x7000, 8, -0.1)]:
        assert adam(ok, bad) == _lib.FM_E_INVALID and b"overlap" in lib.fm_last_error()
    # inside a longer span that neither neighbour in the order touches
    assert adam((0x1000, 0x9000, 0xA000, 0xB000, 1000, 0.0), (0x1100, 0x9FFC, 0xAFFC, 0xBFFC, 1, 0.0),
                ) == _lib.FM_E_INVALID
    m = [_lib.NORMED_MATRIX.pack(0x1000, 0x2000, 0x3000), _lib.NORMED_MATRIX.pack(0x4000, 0x2000, 0x3008)]
    args = (4, 8, _lib.FM_DT_F32, 1, 0.1, 0.95, 1e-8, 0x100000, 1 << 20, None)
    assert lib.fm_muon_apply_normed(b"".join(m), 2, *args) == _lib.FM_E_INVALID
    assert b"overlap" in lib.fm_last_error()


@pytest.mark.parametrize("count,rows", [(1, 1), (3, 4096), (70, 41)])
def test_normed_workspace_size(count, rows):
    from muon_fused.step_ops import normed_workspace_size

    assert normed_workspace_size(count, rows) >= 4 * count * rows


def test_struct_sizes_match_the_header():
    # 4 pointers, int64, float and its padding; 3 pointers
    assert _lib.ADAMW_TENSOR.size == 48 and _lib.NORMED_MATRIX.size == 24


def test_overlap_of_written_and_read_tensors():
    from muon_fused.step_ops import _overlap

    x = torch.zeros(64)
    assert not _overlap([x[:16], x[16:32]], [x[32:], x[40:48]])  # reads may overlap
    assert not _overlap([x[8:8]], [x])
    assert _overlap([x[:16], x[15:32].view(torch.bfloat16)], [])
    assert _overlap([x[:16]], [x[15:]])
    assert _overlap([x[40:41]], [x[:64], x[2:3]])  # inside a longer span before its neighbour


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("bad", [None, [None], [1.0], 3])
def test_lists_of_something_else_are_refused(which, bad):
    """A gradient that is None, a number, no list at all: a RuntimeError that names the list."""
    name = ("params", "grads", "moments1", "moments2")[which]
    args = _four()
    args[which] = bad
    with pytest.raises(RuntimeError, match=name + " must be a list of tensors"):
        fused_adamw(*args, 1, lr=0.1)
    if which < 3:
        name = ("params", "updates", "row_moments")[which]
        args = [[torch.zeros(4, 6)], [torch.zeros(4, 6, dtype=torch.bfloat16)], [torch.zeros(4)]]
        args[which] = bad
        with pytest.raises(RuntimeError, match=name + " must be a list of tensors"):
            fused_normed_update(*args, lr=0.1)
