"""The extension module that looks at tensors and calls launchers with them, on CPU tensors as far as that goes."""
import ctypes
import subprocess

import numpy as np
import pytest
import torch

from railgun_b200 import native, ops
from test_fastcall import SOURCE


@pytest.fixture(scope="module")
def tensors():
    try:
        return native.load_module("fasttensor")
    except native.NativeToolMissing as e:
        pytest.skip(str(e))


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    where = tmp_path_factory.mktemp("probe")
    src, lib = where / "probe.cpp", where / "probe.so"
    src.write_text(SOURCE + 'extern "C" unsigned long long low(void* p, void* q, int n) { return (unsigned)((*(int*)p) + 10 * ((char*)q)[n]); }')
    subprocess.run([native._find("g++", ["/usr/bin/g++"]), "-O2", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    return ctypes.CDLL(str(lib))


def address(f):
    return ctypes.cast(f, ctypes.c_void_p).value


def test_arguments_in_their_places(tensors, probe):
    args = (0x123456789abc, -7, 1.5, None, 1 << 40, -2.25, 3, 4, np.int32(5), 6, 0.1, 8, True, 0x7fffffffffff)
    assert tensors.call(address(probe.probe), "pifpifiiiifiip", *args) == 2 ** 14 - 1
    assert tensors.call(address(probe.low), "ppi", torch.tensor([7], dtype=torch.int32), b"\1\2\3", 2) == 37


def test_what_it_refuses(tensors, probe):
    f = address(probe.probe)
    for bad in (("address", "i", 1), (f, 5, 1), (f, "ii", 1), (f, "i", 1, 2), (f, "i", 2.0), (f, "i", None), (f, "f", "text"), (f, "p", 2.0), (f, "p", "text"),
                (f, "x", 1), (f, "i" * 49, *range(49)), (f, "f" * 9, *[0.5] * 9), ()):
        with pytest.raises(TypeError):
            tensors.call(*bad)
    with pytest.raises(ValueError):
        tensors.call(0, "i", 1)


def test_what_does_not_fit(tensors):
    """A tensor on the CPU never fits, nor does what is no tensor."""
    x = torch.zeros(3, 4, dtype=torch.int32)
    for t in (x, None, 5, "text", np.zeros(3)):
        assert tensors.fits(t, torch.int32, 0, 3, 4) is False and tensors.rows(t, torch.int32, 0, 1) is None
        assert tensors.fits_all(0, t, torch.int32, 3, 4) is False
        assert tensors.addresses([t], 0) is None and tensors.addresses(t, 0) is None
    assert tensors.addresses([], 0) is None
    assert tensors.fits_all(0) is True and tensors.fits_all(0, x) is False and tensors.fits_all(0, 5, torch.int32) is False
    with pytest.raises(TypeError):
        tensors.fits(x)
    with pytest.raises(TypeError):
        tensors.fits_all()
    with pytest.raises(TypeError):
        tensors.empty("int32", 0, 3)


def test_matrices_that_share_memory(tensors, monkeypatch):
    """The module and the way through Python against marks in memory."""
    flat = torch.zeros(400, dtype=torch.int16)
    for rows in (0, 1, 2, 5):
        for xs, ys in ((10, 10), (10, 7), (30, 30), (4, 4)):
            for columns in (1, 3, 4):
                for xo, yo in ((0, 0), (0, 3), (3, 0), (0, 4), (4, 0), (0, 26), (0, 10), (0, 33), (12, 60), (60, 12), (20, 30), (0, 200), (200, 0), (7, 40)):
                    x, y = (flat.as_strided((rows, 4), (step, 1), o) for step, o in ((xs, xo), (ys, yo)))
                    flat.zero_()
                    x[:, :columns] = 1
                    want = not y[:, :columns].any().item()
                    got = []
                    for module in (tensors, False):
                        monkeypatch.setattr(ops, "_tensors", module)
                        got.append(ops._rows_apart(x, y, columns))
                    assert got[0] is got[1] and (want or not got[0])        # never apart where they are not
                    assert got[0] == want or (xs != ys)                      # rows at different distances may be refused
    for bad in ((flat, flat, 3), (x, y.float(), 3), (x, y[1:], 3), (x, y), (x, y, 1.0), (x, None, 3)):
        with pytest.raises(TypeError):
            tensors.apart(*bad)


@pytest.mark.gpu
def test_what_fits(tensors):
    x = torch.zeros(3, 4, 5, dtype=torch.int32, device="cuda:0")
    assert tensors.fits(x, torch.int32, 0, 3, 4, 5) and tensors.fits(x, None, 0, None, 4, None) and tensors.fits(x[:, :, 0].contiguous(), torch.int32, 0, 3, 4)
    for dtype, device, sizes in ((torch.float32, 0, (3, 4, 5)), (torch.int32, 1, (3, 4, 5)), (torch.int32, 0, (3, 4)), (torch.int32, 0, (3, 4, 6))):
        assert not tensors.fits(x, dtype, device, *sizes)
    assert not tensors.fits(x.transpose(0, 1), torch.int32, 0, 4, 3, 5)
    m = torch.zeros(6, 10, device="cuda:0")
    assert tensors.rows(m[:, 2:9], torch.float32, 0, 7) == (6, 10) and tensors.rows(m[:, 2:9], torch.float32, 0, 8) is None
    assert tensors.rows(m.t(), torch.float32, 0, 1) is None and tensors.rows(m[0].expand(3, 10), torch.float32, 0, 1) is None
    a, b = torch.zeros(2, 3, device="cuda:0"), torch.zeros(2, 3, device="cuda:0")
    assert np.frombuffer(tensors.addresses([a, b], 0), np.uint64).tolist() == [a.data_ptr(), b.data_ptr()]
    assert tensors.addresses((a, b), 0) is not None
    for other in (b[:1], b.double(), b.t(), b.cpu(), None):
        assert tensors.addresses([a, other], 0) is None
    new = tensors.empty(torch.bfloat16, 0, 2, 0, 7)
    assert new.shape == (2, 0, 7) and new.dtype == torch.bfloat16 and new.device == a.device


@pytest.mark.gpu
def test_addresses_of_tensors_that_share_memory(tensors):
    x = torch.zeros(10, 3, device="cuda:0")
    for bad in ([x, x], [x[:9], x[1:]], [x[1:], x[:9]], [x[:5], x[5:], x[4:9]]):
        assert tensors.addresses(bad, 0) is None
        with pytest.raises(ops.KernelError, match="share memory"):
            ops.copy_pages(bad, [(0, 1, -1)])
    assert np.frombuffer(tensors.addresses([x[5:], x[:5]], 0), np.uint64).tolist() == [x[5:].data_ptr(), x.data_ptr()]


@pytest.mark.gpu
def test_without_the_module_calls_are_the_same(monkeypatch):
    """The way through Python alone, which machines without torch's headers take."""
    def run():
        p, cu, starts = (torch.tensor(v, dtype=torch.int32, device="cuda:0") for v in ([-1, 0, 0, 1, -1, 0], [0, 4, 6], [5, 9]))
        masks, positions = ops.draft_tree(p, cu, starts, max_rows=4)
        g = torch.Generator(device="cuda:0").manual_seed(1)
        cache = torch.randn(4, 2, 1, 8, 16, device="cuda:0", generator=g)
        q, table = torch.randn(6, 32, device="cuda:0", generator=g), torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda:0")
        out = torch.empty(6, 32, device="cuda:0")
        ops.tree_attention(q, out, cache, table, cu, starts, masks, 2, 1, 16, 0.25, max_rows=4, max_context=16)
        kept = ops.keep_drafts(cache, table, cu, starts, p, cu.new_tensor([0, 1, 2, 3, 0, 1]), cu.new_tensor([2, 9, 9, 9, 9, 9]), max_rows=4)
        ops.copy_pages([cache], [(0, 3, 5)])
        return [masks, positions, out, *kept, cache]
    with_it = run()
    monkeypatch.setattr(ops, "_tensors", False)
    for a, b in zip(with_it, run()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_several_at_once(tensors):
    x, y = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.zeros(5, device="cuda")
    f32, i32 = torch.float32, torch.int32
    assert tensors.fits_all(0, x, i32, 3, 4, y, f32, None, x, i32, np.int64(3), None)
    for bad in ((x, i32, 3, 4, y, f32, 4), (x, i32, 3, y, f32, 5), (x, i32, 3, 4, y, i32, 5), (x, i32, 3, 4, y[::2], f32, None), (x, i32, 3, 4, y.cpu(), f32, 5),
                (x, i32, 3, 4, None, f32, 5), (x, i32, 3, 4, y)):
        assert tensors.fits_all(0, *bad) is False
    assert tensors.fits_all(1, x, i32, 3, 4) is False
