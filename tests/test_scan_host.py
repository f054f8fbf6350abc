"""The gated recurrence's refusals: everything that is refused is refused on the host, before anything touches a GPU."""
import ctypes

import pytest
import torch

from neurofluid_amd import scan


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("gate, x, kw, err", [
    (t(2, 5, 3, dtype=torch.float64), t(2, 5, 3, dtype=torch.float64), {}, TypeError),
    (t(2, 5, 3, dtype=torch.bfloat16), t(2, 5, 3), {}, TypeError),                       # a 16-bit gate beside 32-bit x
    (t(2, 5, 3, dtype=torch.float16), t(2, 5, 3, dtype=torch.bfloat16), {}, TypeError),
    (t(2, 5, 2), t(2, 5, 3), {}, ValueError),
    (t(1, 5, 3), t(2, 5, 3), {}, ValueError),                                             # (expand() it)
    (t(5, 3), t(2, 5, 3), {}, ValueError),
    (t(2, 5, 0), t(2, 5, 0), {}, ValueError),
    (t(5, 3), t(5, 3), {}, ValueError),                                                   # 2-d without row_splits
    (t(2, 5, 3), t(2, 5, 3), dict(row_splits=torch.zeros(2, dtype=torch.int64)), ValueError),
    (t(5, 3), t(5, 3), dict(row_splits=torch.zeros(2, dtype=torch.int32)), ValueError),
    (t(5, 3), t(5, 3), dict(row_splits=torch.zeros(0, dtype=torch.int64)), ValueError),
    (t(5, 3), t(5, 3), dict(row_splits=torch.zeros(3, dtype=torch.int64), h0=t(3, 3)), ValueError),
    (t(2, 5, 3), t(2, 5, 3), dict(h0=t(2, 4)), ValueError),
    (t(2, 5, 3), t(2, 5, 3), dict(h0=t(2, 3, dtype=torch.bfloat16)), ValueError),
    (t(2, 5, 3), t(2, 5, 3), {}, RuntimeError),                                           # on the CPU: no fallback
])
def test_gated_scan_refuses(gate, x, kw, err):
    with pytest.raises(err):
        scan.gated_scan(gate, x, **kw)


@pytest.mark.parametrize("gate, x, state, kw, err", [
    (t(2, 5, 3), t(2, 5, 3), t(2, 5, 3), {}, ValueError),
    (t(4, 3), t(4, 3), t(4, 2), {}, ValueError),
    (t(4, 3), t(4, 3), t(4, 3, dtype=torch.float16), {}, ValueError),
    (t(4, 3), t(4, 3), t(3, 4).t(), {}, ValueError),                                      # channels apart
    (t(4, 3), t(4, 3), t(1, 3).expand(4, 3), {}, ValueError),                             # one state for all rows
    (t(4, 3), t(4, 3), t(4, 3), dict(out=t(4, 1).expand(4, 3)), ValueError),
    (t(4, 3).requires_grad_(), t(4, 3), t(4, 3), {}, RuntimeError),
    (t(4, 3), t(4, 3), t(4, 3), {}, RuntimeError),
])
def test_gated_scan_step_refuses(gate, x, state, kw, err):
    with pytest.raises(err):
        scan.gated_scan_step(gate, x, state, **kw)


def test_no_axis_of_steps_is_refused():
    one = torch.ones(5)
    for x in (one, one[0]):
        with pytest.raises(ValueError, match="axis"):
            scan.gated_scan(x, x)
        with pytest.raises(ValueError, match="axis"):
            scan.gated_scan_step(x, x, x)


def test_gated_scan_step_refuses_an_out_that_overlaps_the_state():
    buf = t(6, 3)
    with pytest.raises(ValueError, match="overlaps"):
        scan.gated_scan_step(t(4, 3), t(4, 3), buf[:4], out=buf[1:5])


def test_c_entries_refuse():
    from neurofluid_amd import _lib, build
    build.build()
    lib = _lib.load()
    s = _lib.Scan(dtype=7, B=1, T=4, D=4)
    assert lib.nf_scan_plan(ctypes.byref(s), None) < 0 and b"dtype" in lib.nf_last_error()
    s = _lib.Scan(dtype=0, B=1, T=4, D=0)
    assert lib.nf_scan_plan(ctypes.byref(s), None) < 0 and b"sizes" in lib.nf_last_error()
    s = _lib.Scan(dtype=0, B=1, T=4, D=4)
    assert lib.nf_scan_fwd(ctypes.byref(s), None) < 0 and b"plan" in lib.nf_last_error()
    n = ctypes.c_size_t()
    assert lib.nf_scan_plan(ctypes.byref(s), ctypes.byref(n)) == 0 and s.vec in (1, 2, 4) and n.value >= 4
    assert lib.nf_scan_fwd(ctypes.byref(s), None) < 0 and b"null" in lib.nf_last_error()
    assert lib.nf_scan_step(0, 0, 0, 0, -1, 4, None, 0, None, 0, None, 0, None, 0, None, None) < 0
    assert lib.nf_scan_step(0, 0, 0, 0, 1, 4, None, 0, None, 0, None, 0, None, 0, None, None) < 0
    # a long, narrow sequence is cut: the plan asks for room for the chunks
    s = _lib.Scan(dtype=1, B=1, T=100000, D=64)
    assert lib.nf_scan_plan(ctypes.byref(s), None) == 0 and lib.nf_scan_workspace_bytes(ctypes.byref(s), 0) > 0


def test_the_packed_descriptor_is_the_struct():
    """scan._PACK writes nf_scan_t as ctypes lays it out (every field with a value of its own)."""
    from neurofluid_amd import _lib
    assert scan._PACK.size == ctypes.sizeof(_lib.Scan)
    names = [n for n, _ in _lib.Scan._fields_]
    buf = bytearray(scan._PACK.size)
    scan._PACK.pack_into(buf, 0, *range(1, len(names) + 1))
    s = _lib.Scan.from_buffer(buf)
    assert [getattr(s, n) for n in names] == list(range(1, len(names) + 1))


@pytest.fixture
def no_gpu(monkeypatch):
    """The host side on CPU tensors: the C entries note what they are given and do nothing."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            def entry(*args):
                calls.append((name, args))
                return 0
            return entry
    lib = Lib()
    monkeypatch.setattr(scan._lib, "load", lambda: lib)
    monkeypatch.setattr(scan._lib, "raw_stream", lambda q: 0)
    monkeypatch.setattr(scan.ops, "_require_cuda", lambda *a: None)
    return calls


@pytest.mark.parametrize("own_out", [False, True])
def test_step_counts_as_a_change_in_place(no_gpu, own_out):
    """A recorded operation that keeps the state refuses its backward once a step has written there, as after any in-place operation."""
    w, s = torch.ones(4, 3, requires_grad=True), t(4, 3)
    y, before = (w * s).sum(), s._version
    with torch.no_grad():
        scan.gated_scan_step(t(4, 3), t(4, 3), t(4, 3) if own_out else s, **(dict(out=s) if own_out else {}))
    assert no_gpu and s._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    # ... seen through a view too; a state that is only read stays as it was
    rows, read = t(8, 5), t(4, 3)
    before = rows._version, read._version
    scan.gated_scan_step(t(4, 3), t(4, 3), read, out=rows[::2, 1:4])
    assert (rows._version, read._version) == (before[0] + 1, before[1])
    with torch.inference_mode():
        scan.gated_scan_step(t(4, 3), t(4, 3), t(4, 3))


def test_step_refuses_an_out_with_gradients():
    with pytest.raises(RuntimeError, match="no gradients"):
        scan.gated_scan_step(t(4, 3), t(4, 3), t(4, 3), out=t(4, 3).requires_grad_())


@pytest.mark.parametrize("rows, D", [(2 ** 32, 1), (2 ** 32 + 5, 1), (2 ** 31, 1), (1, 2 ** 31)])
def test_step_refuses_sizes_that_the_c_entry_would_cut(no_gpu, rows, D):
    """(Views and storage that is never touched: no memory behind it.)"""
    x = t(1, 1, dtype=torch.bfloat16).expand(rows, D)
    state = torch.empty(rows, D, device="meta")

    class OnTheCpu(torch.Tensor):
        device = torch.device("cpu")
    with pytest.raises(ValueError, match="more than"):
        scan.gated_scan_step(x, x, state.as_subclass(OnTheCpu))
    assert not no_gpu


def test_step_takes_an_out_beside_the_state_in_the_same_rows(no_gpu):
    """The check of overlaps against a comparison of every address, over all pairs of windows of one buffer."""
    x = t(3, 2)
    buf = t(60)
    taken = refused = 0
    for stride_a in (2, 3, 5):
        for stride_b in (2, 3, 5):
            for at_a in range(0, 30, 7):
                for at_b in range(0, 40):
                    state, out = buf.as_strided((3, 2), (stride_a, 1), at_a), buf.as_strided((3, 2), (stride_b, 1), at_b)
                    where = lambda base, st: {base + r * st + c for r in range(3) for c in range(2)}
                    same, apart = (at_a, stride_a) == (at_b, stride_b), not where(at_a, stride_a) & where(at_b, stride_b)
                    if same or (apart and stride_a == stride_b):
                        scan.gated_scan_step(x, x, state, out=out)
                        taken += 1
                    elif not apart:
                        with pytest.raises(ValueError, match="overlaps"):
                            scan.gated_scan_step(x, x, state, out=out)
                        refused += 1
    assert taken > 100 and refused > 100
    one = buf.as_strided((1, 2), (0, 1), 1)               # (one row: any stride)
    with pytest.raises(ValueError, match="overlaps"):
        scan.gated_scan_step(t(1, 2), t(1, 2), buf[None, :2], out=one)
    with pytest.raises(ValueError, match="overlaps"):
        scan.gated_scan_step(t(1, 2), t(1, 2), buf.as_strided((1, 2), (0, 1), 0), out=one)


def test_forward_mode_is_refused(no_gpu):
    """A dual tensor has no requires_grad and its primal's pointer: without a refusal its tangent is dropped."""
    from torch.autograd import forward_ad as fw
    with fw.dual_level():
        dual = lambda *shape: fw.make_dual(t(*shape), torch.ones(*shape))
        for args in ((dual(2, 5, 3), t(2, 5, 3)), (t(2, 5, 1), dual(2, 5, 3)), (t(2, 5, 3), t(2, 5, 3), dual(2, 3))):
            for mode in (torch.no_grad, torch.enable_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                    scan.gated_scan(*args)
        for args in ((dual(4, 3), t(4, 3), t(4, 3)), (t(4, 1), dual(4, 3), t(4, 3)), (t(4, 3), t(4, 3), dual(4, 3)), (t(4, 3), t(4, 3), t(4, 3), dual(4, 3))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                scan.gated_scan_step(*args[:3], **(dict(out=args[3]) if len(args) > 3 else {}))

        class Ctx:
            pass
        with pytest.raises(NotImplementedError, match="forward-mode"):
            scan._ScanFn.backward(Ctx(), dual(2, 5, 3), None)
        assert not no_gpu
        scan.gated_scan_step(t(4, 3), t(4, 3), t(4, 3))          # (tensors without a tangent are served inside a level too)
        assert no_gpu
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda x: scan.gated_scan(t(2, 5, 3), x)[0], (t(2, 5, 3),), (t(2, 5, 3),))
