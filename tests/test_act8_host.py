"""Refusals of the 8-bit activation checkpoints, on the host."""
import ctypes

import pytest
import torch

from neurofluid_amd import act8


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def fake(rows, K):
    return act8.Act8(t(rows * ((K + 31) // 32 * 32), dtype=torch.uint8), t(64, dtype=torch.uint8), (rows, K), torch.float32)


@pytest.mark.parametrize("x, err", [(t(4, 5, dtype=torch.float64), TypeError), (t(4, 5, dtype=torch.int32), TypeError), (torch.tensor(1.0), ValueError),
                                    (t(4, 5), RuntimeError), (t(1, 1).expand((1 << 30) + 1, 1), ValueError)])
def test_pack_refuses(x, err):
    with pytest.raises(err):
        act8.pack(x)


@pytest.mark.parametrize("dy, ck, err", [
    (t(4, 5, dtype=torch.float64), fake(4, 6), TypeError), (t(4, 5), t(4, 6), TypeError), (t(3, 5), fake(4, 6), ValueError),
    (t(4, 0), fake(4, 6), ValueError), (t(4, 5), fake(4, 0), ValueError), (t(4, 5), fake(4, 6), RuntimeError)])
def test_wgrad_refuses(dy, ck, err):
    with pytest.raises(err):
        act8.wgrad(dy, ck)


def test_wgrad_refuses_numbers_that_the_c_entry_would_cut():
    for job in ((0, 2 ** 32 + 5, 0, 6, True), (2 ** 32, 5, 0, 6, True), (0, 5, 0, 2 ** 33 + 6, False)):
        with pytest.raises(ValueError, match="pass"):
            act8.wgrad_jobs(t(4, 5), fake(4, 6), [job])


def test_a_checkpoint_that_is_not_whole_is_refused():
    whole = fake(70, 40)
    for codes, scales in ((whole.codes[:-1], whole.scales), (whole.codes, t(255, dtype=torch.uint8)), (whole.codes, t(256)),
                          (t(2 * whole.codes.numel(), dtype=torch.uint8)[::2], t(256, dtype=torch.uint8))):
        with pytest.raises(ValueError, match="must be"):
            act8.Act8(codes, scales, (70, 40), torch.float32).unpack()
    act8.Act8(whole.codes, t(256, dtype=torch.uint8), (70, 40), torch.float32)._whole("here")


@pytest.mark.parametrize("rows", [0, 1, 63, 64, 65, 1000])
@pytest.mark.parametrize("K", [0, 1, 31, 32, 33, 2432])
def test_sizes_are_the_c_entries(rows, K):
    from neurofluid_amd import _lib, build
    build.build()
    lib = _lib.load()
    want = (lib.nf_act8_code_bytes(rows, K), lib.nf_act8_scale_bytes(rows, K))
    assert act8._sizes(rows, K) == want


def test_unpack_refuses():
    with pytest.raises(TypeError):
        fake(2, 3).unpack(torch.float64)


@pytest.mark.parametrize("x, w, b, err", [
    (t(4, 5, dtype=torch.bfloat16), t(3, 5), None, TypeError), (t(4, 5), t(3, 5, dtype=torch.float16), None, TypeError),
    (t(4, 5), t(3, 6), None, ValueError), (t(4, 5), t(5), None, ValueError), (t(4, 5), t(3, 5), t(4), ValueError), (t(4, 5), t(3, 5), t(3, 1), ValueError),
    (t(4, 5), t(0, 5), None, ValueError), (t(4, 5), t(3, 5), t(3), RuntimeError)])
def test_linear_refuses(x, w, b, err):
    with pytest.raises(err):
        act8.linear(x, w, b)


def test_nerf_refuses():
    from neurofluid_amd.nerf import NeRF
    with pytest.raises(ValueError):
        NeRF(in_channels_xyz=198, in_channels_dir=54, act_checkpoint="int4")
    with pytest.raises(NotImplementedError):
        NeRF(in_channels_xyz=63, in_channels_dir=27, act_checkpoint="e4m3")
    a, b = NeRF(in_channels_xyz=198, in_channels_dir=54, act_checkpoint="e4m3"), NeRF(in_channels_xyz=198, in_channels_dir=54)
    assert list(a.state_dict()) == list(b.state_dict())


def test_c_entries_refuse():
    from neurofluid_amd import _lib, build
    build.build()
    lib = _lib.load()
    assert lib.nf_act8_code_bytes(3, 33) == 3 * 64 and lib.nf_act8_scale_bytes(65, 33) == 128 * 2 and lib.nf_act8_code_bytes(0, 4) == 0
    assert lib.nf_act8_pack(5, None, 0, 1, 1, None, None, None) < 0 and b"dtype" in lib.nf_last_error()
    assert lib.nf_act8_pack(0, None, 4, 4, 4, None, None, None) < 0 and b"null" in lib.nf_last_error()
    assert lib.nf_act8_pack(0, None, 4, -1, 4, None, None, None) < 0
    assert lib.nf_act8_unpack(0, None, None, 4, 4, None, 4, None) < 0
    job = lambda *a: (_lib.Act8Job * 1)(_lib.Act8Job(*a))
    for bad in (job(0, 5, 0, 4, 1), job(1, 4, 0, 4, 1), job(0, 4, 16, 4, 1), job(0, 4, 0, 65, 1), job(-1, 2, 0, 4, 1), job(0, 0, 0, 4, 1), job(2 ** 31 - 1, 2, 0, 4, 1)):
        assert lib.nf_act8_wgrad(0, None, 4, 4, None, None, 64, 8, 1, bad, None, None, None, None) < 0
        assert lib.nf_act8_wgrad_workspace_floats(8, 4, 64, 1, bad) == 0
    for dy_cols, x_cols in ((2 ** 31 - 1, 64), (4, 2 ** 31 - 1)):
        assert lib.nf_act8_wgrad(0, None, 4, dy_cols, None, None, x_cols, 8, 1, job(0, 4, 0, 4, 1), None, None, None, None) < 0 and b"bad sizes" in lib.nf_last_error()
    many = (_lib.Act8Job * 2)(_lib.Act8Job(0, 2 ** 30, 0, 1, 1), _lib.Act8Job(0, 2 ** 30, 0, 1, 1))
    assert lib.nf_act8_wgrad(0, None, 4, 2 ** 30, None, None, 64, 8, 2, many, None, None, None, None) < 0 and b"outputs" in lib.nf_last_error()
    ok = job(0, 4, 32, 4, 1)
    assert lib.nf_act8_wgrad(0, None, 4, 4, None, None, 64, 8, 0, ok, None, None, None, None) < 0
    assert lib.nf_act8_wgrad(0, None, 4, 4, None, None, 64, 8, 1, ok, None, None, None, None) < 0 and b"null" in lib.nf_last_error()
    assert lib.nf_act8_wgrad_workspace_floats(100000, 4, 64, 1, ok) > 0


def test_codes_in_host_memory_are_refused():
    """A whole checkpoint that was moved to the host: its pointers are not the GPU's to read."""
    ck = act8.Act8(t(70 * 64, dtype=torch.uint8), t(256, dtype=torch.uint8), (70, 40), torch.float32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ck.unpack()
    with pytest.raises(RuntimeError, match="on the GPU"):
        act8.wgrad(t(70, 4), ck)


def test_forward_mode_is_refused(monkeypatch):
    from torch.autograd import forward_ad as fw
    monkeypatch.setattr(act8.ops, "_require_cuda", lambda *a: None)
    ck = act8.Act8(t(4 * 32, dtype=torch.uint8), t(64, dtype=torch.uint8), (4, 6), torch.float32)
    with fw.dual_level():
        dual = lambda *shape: fw.make_dual(t(*shape), torch.ones(*shape))
        for call in (lambda: act8.pack(dual(4, 6)), lambda: act8.wgrad(dual(4, 5), ck), lambda: act8.linear(dual(4, 6), t(5, 6)),
                     lambda: act8.linear(t(4, 6), dual(5, 6)), lambda: act8.linear(t(4, 6), t(5, 6), dual(5)),
                     lambda: act8._LinearFn.backward(None, dual(4, 5))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_sizes_that_the_c_entries_would_cut_are_refused(monkeypatch):
    """(Storage that is never touched: no memory behind it.)"""
    monkeypatch.setattr(act8.ops, "_require_cuda", lambda *a: None)
    rows = 2 ** 32 + 5
    big = act8.Act8(torch.empty(32 * rows, dtype=torch.uint8, device="meta"), torch.empty(rows + 64, dtype=torch.uint8, device="meta"), (rows, 1), torch.float32)
    with pytest.raises(ValueError, match="more than"):
        big.unpack()
    with pytest.raises(ValueError, match="more than"):
        act8.wgrad(torch.empty(1, 1, device="meta").expand(rows, 4), big)
    with pytest.raises(ValueError, match="more than"):
        act8.wgrad_jobs(t(1, 1).expand(4, rows), fake(4, 6), [(0, 5, 0, 6, True)])
    for x, w in ((t(1, 1).expand(rows, 1), t(3, 1)), (t(1, 1), t(1, 1).expand(rows, 1)), (t(1, 1).expand(1, rows), t(1, 1).expand(2, rows))):
        with pytest.raises(ValueError, match="more than"):
            act8.linear(x, w)


def test_a_nerf_without_the_choice_has_none():
    """A module that was pickled whole before act_checkpoint existed."""
    from neurofluid_amd.nerf import NeRF
    net = NeRF(in_channels_xyz=198, in_channels_dir=54)
    old = NeRF.__new__(NeRF)
    old.__setstate__({k: v for k, v in net.__dict__.items() if k != "act_checkpoint"})
    assert old.act_checkpoint is None and "act_checkpoint" not in old.__dict__


def test_more_tiles_than_an_int_counts():
    """2^46 tiles, whose count in 32 bits is 0 (and was divided by): in a process of its own."""
    import os
    import subprocess
    import sys
    from neurofluid_amd import build
    build.build()
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = "\n".join(["from neurofluid_amd import _lib", "lib = _lib.load()",
                      "for m, k in ((30, 30), (24, 30), (30, 23)):",
                      "    j = (_lib.Act8Job * 1)(_lib.Act8Job(0, 1 << m, 0, 1 << k, 1))",
                      "    assert lib.nf_act8_wgrad_workspace_floats(1, 1 << m, 1 << k, 1, j) == 0",
                      "    assert lib.nf_act8_wgrad(1, None, 1 << m, 1 << m, None, None, 1 << k, 1, 1, j, None, None, None, None) < 0 and b'tiles' in lib.nf_last_error()"])
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100, cwd=root)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
