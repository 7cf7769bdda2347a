"""CPU: the refusals of the row lookup, at the Python surface and at the C ABI."""
import ctypes as C

import pytest
import torch

from vegs_amd import _capi, embedding


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        embedding.lookup(torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU"):
        embedding.lookup([[1.0]], torch.zeros(2, dtype=torch.int64))


def _lookup(**over):
    some = 1 << 20                                        # (a made-up address: nothing is launched for a refused call)
    args = dict(table=some, ids=some, row_scale=None, n=5, rows=7, width=3, table_stride=3, table_dtype=0, out_dtype=0, ids_64=0,
                scale=1.0)
    args.update(over)
    return _capi.VrLookup(*[args[f] for f, _ in _capi.VrLookup._fields_])


BAD = [dict(n=-1), dict(n=1 << 30), dict(rows=-1), dict(rows=0x7fffffff), dict(width=0), dict(width=(1 << 24) + 1),
       dict(table_stride=2), dict(table_dtype=3), dict(table_dtype=-1), dict(out_dtype=1), dict(table_dtype=1, out_dtype=2),
       dict(table=None), dict(ids=None), dict(table=(1 << 20) + 2), dict(ids=(1 << 20) + 4, ids_64=1), dict(ids=(1 << 20) + 2),
       dict(row_scale=(1 << 20) + 1)]


@pytest.mark.parametrize("over", BAD, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_c_entries_refuse_bad_lookups(over):
    lib = _capi.load()
    some = 1 << 20
    bad = _lookup(**over)
    assert lib.vr_lookup_forward(C.byref(bad), some, None) == -1
    assert b"lookup" in lib.vr_last_error()
    assert lib.vr_lookup_backward(C.byref(bad), some, 3, some, None, some, 1 << 30, None) == -1


def test_c_entries_refuse_bad_outputs_and_scratch():
    lib = _capi.load()
    some, good = 1 << 20, _lookup()
    assert lib.vr_lookup_forward(None, some, None) == -1
    assert lib.vr_lookup_forward(C.byref(good), None, None) == -1
    assert lib.vr_lookup_forward(C.byref(good), some + 2, None) == -1
    assert lib.vr_lookup_scratch_bytes(5, 7, 3) == 0      # few entries are sorted on the chip
    good = _lookup(n=5000)
    need = lib.vr_lookup_scratch_bytes(5000, 7, 3)
    assert need > 0
    for grad, stride, d_table, d_scale, scratch, nbytes in ((None, 3, some, None, some, need), (some, 2, some, None, some, need),
                                                            (some + 2, 3, some, None, some, need), (some, 3, some + 2, None, some, need),
                                                            (some, 3, some, some + 2, some, need), (some, 3, some, None, None, need),
                                                            (some, 3, some, None, some + 16, need), (some, 3, some, None, some, need - 1)):
        assert lib.vr_lookup_backward(C.byref(good), grad, stride, d_table, d_scale, scratch, nbytes, None) == -1
    for sizes in ((-1, 7, 3), (1 << 30, 7, 3), (5, -1, 3), (5, 0x7fffffff, 3), (5, 7, 0), (5, 7, (1 << 24) + 1)):
        assert lib.vr_lookup_scratch_bytes(*sizes) == 0


def test_nothing_to_do_launches_nothing():
    """No entries forward, neither gradient wanted backward: fine without a GPU."""
    lib = _capi.load()
    assert lib.vr_lookup_forward(C.byref(_lookup(n=0, ids=None)), None, None) == 0
    assert lib.vr_lookup_backward(C.byref(_lookup()), 1 << 20, 3, None, None, None, 0, None) == 0


def test_rows_that_lie_apart_are_taken_as_they_are():
    t = torch.zeros(6, 5, 4)
    assert embedding._row_layout(t, 1, 20)[1] == 20
    part = t[:, 1:3]                                       # rows of 8 values, 20 apart
    same, stride = embedding._row_layout(part, 1, 8)
    assert same is part and stride == 20
    for other in (t[:, :, 1:], t.transpose(0, 1), t[:1].expand(6, 5, 4), t[:, ::2]):
        copy, stride = embedding._row_layout(other, 1, other[0].numel())
        assert copy.is_contiguous() and stride == other[0].numel()
    copy, stride = embedding._row_layout(part, 2, 4)       # two leading dimensions: not one stride
    assert copy.is_contiguous() and stride == 4


_EMPTY = r"""
import sys
sys.path.insert(0, %r)
import ctypes as C
from vegs_amd import _capi
lib, some = _capi.load(), 1 << 20
for dtype, width in ((0, 3), (0, 256), (0, 257), (0, 1000), (1, 513), (2, 1 << 22)):
    empty = _capi.VrLookup(some, None, None, 0, 7, width, width, dtype, dtype, 0, 1.0)
    for d_table, d_scale in ((some, some), (some, None), (None, some), (None, None)):
        lib.vr_lookup_backward(C.byref(empty), None, width, d_table, d_scale, None, 0, None)
    print(dtype, width, lib.vr_lookup_backward(C.byref(empty), None, width, None, some, None, 0, None), flush=True)
"""


def test_gradients_of_no_entries_do_not_end_the_process():
    """In a process of its own that sees no GPU (the addresses are made up: there the launch that clears the gradient fails)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _EMPTY % root], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1"))
    assert r.returncode == 0, (r.returncode, r.stdout[-500:], r.stderr[-2000:])
    assert [line.split()[2] for line in r.stdout.split("\n") if line] == ["0"] * 6       # the scales' gradient of no entries: nothing to do


def test_the_widest_row():
    """2^22 values; with strides that would take more, so that it is the width that is refused."""
    lib = _capi.load()
    some, most = 1 << 20, 1 << 22
    for width, ok in ((most, True), (most + 1, False)):
        assert (lib.vr_lookup_scratch_bytes(5000, 7, width) > 0) == ok
        wide = _lookup(width=width, table_stride=width + 1, n=0, ids=None)
        assert lib.vr_lookup_forward(C.byref(wide), None, None) == (0 if ok else -1)
        assert lib.vr_lookup_backward(C.byref(wide), None, width + 1, None, some, None, 0, None) == (0 if ok else -1)
        assert ok or b"width" in lib.vr_last_error()
        wide = _lookup(width=width, table_stride=width + 1)
        if not ok:
            assert lib.vr_lookup_forward(C.byref(wide), some, None) == -1
            assert lib.vr_lookup_backward(C.byref(wide), some, width + 1, some, None, some, 1 << 40, None) == -1


def test_few_entries_take_no_scratch():
    """The count up to which the caller does not ask."""
    lib = _capi.load()
    for rows, width in ((1, 1), (7, 3), (1 << 20, 4096), (5, 1 << 22)):
        assert lib.vr_lookup_scratch_bytes(embedding._ALONE, rows, width) == 0
        assert lib.vr_lookup_scratch_bytes(embedding._ALONE + 1, rows, width) > 0
