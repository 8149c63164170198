"""CPU-only checks of include/trips_loss.h: symbols, sizes of the ctypes mirrors, what the entry points refuse before they touch a
device; the oracle's generator against its published vectors."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from tests import loss_reference as ref
from trips_amd import _lib, abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ERR = (abi.TRIPS_ERR_INVALID_ARG, abi.TRIPS_ERR_UNSUPPORTED, abi.TRIPS_ERR_WORKSPACE_SMALL)
CTX = C.create_string_buffer(4096)
AT = 1 << 20
NAN = float("nan")


def test_library_exports_what_the_header_declares():
    lib = _lib.load()
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "trips_loss.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(trips_[a-z0-9_]+)\s*\(", src)))
    assert names == sorted(_lib.LOSS_SYMBOLS)
    for n in names:
        assert hasattr(lib, n)


def test_ctypes_mirrors_have_c_sizes(tmp_path):
    prog = tmp_path / "sizes.c"
    prog.write_text('#include <stdio.h>\n#include "trips_loss.h"\nint main(){printf("%zu %zu %zu %zu %zu %d %d %d\\n",'
                    "sizeof(TripsTableLossDesc),offsetof(TripsTableLossDesc,scale),offsetof(TripsTableLossDesc,d_table_stride),sizeof(TripsDropoutDesc),"
                    "offsetof(TripsDropoutDesc,step),TRIPS_REDUCE_NONE,TRIPS_REDUCE_SUM,TRIPS_REDUCE_MEAN);return 0;}\n")
    exe = tmp_path / "sizes"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(prog), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert got == [C.sizeof(abi.TripsTableLossDesc), abi.TripsTableLossDesc.scale.offset, abi.TripsTableLossDesc.d_table_stride.offset, C.sizeof(abi.TripsDropoutDesc),
                   abi.TripsDropoutDesc.step.offset, abi.TRIPS_REDUCE_NONE, abi.TRIPS_REDUCE_SUM, abi.TRIPS_REDUCE_MEAN]


def _loss(**kw):
    d = abi.TripsTableLossDesc(abi.TRIPS_ABI_VERSION, 0, 1, 0, 50, 100, 16, 1.0, 16, 16, 16, 16)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _bytes(backward=None):
    n = C.c_size_t(0)
    if backward is None:
        assert _lib.load().trips_table_loss_kept_size(C.byref(_loss()), C.byref(n)) == 0
        return n.value
    assert _lib.load().trips_table_loss_workspace_size(C.byref(_loss()), backward, C.byref(n)) == 0
    return n.value


BAD_DESC = [dict(abi_version=1), dict(dtype=1), dict(dtype=9), dict(index_dtype=2), dict(reduction=3), dict(reduction=-1), dict(num_rows=-1), dict(num_rows=1 << 28),
            dict(num_entries=-1), dict(num_entries=1 << 31), dict(num_channels=0), dict(num_channels=1 << 17), dict(scale=NAN), dict(scale=float("inf")), dict(rows_stride=-1),
            dict(table_stride=-1), dict(table_stride=1 << 41),
            dict(dtype=2, num_rows=20_000_000, num_entries=2_000_000_000)]
BAD_CALL = [dict(ctx=None), dict(table=None), dict(table=AT + 1), dict(kept=None), dict(kept=AT + 128), dict(kept_size=_bytes() - 1), dict(workspace=None), dict(workspace=AT + 128)]


@pytest.mark.parametrize("desc,call", [(d, {}) for d in BAD_DESC] + [({}, c) for c in BAD_CALL] + [
    ({}, dict(rows=None)), ({}, dict(rows=AT + 2)), ({}, dict(target=None)), ({}, dict(target=AT + 2)), ({}, dict(loss=None)), ({}, dict(loss=AT + 2)), ({}, dict(size=_bytes(0) - 1)), (dict(index_dtype=0), dict(target=AT + 4)), (dict(dtype=2), dict(rows=AT + 1)),
    (dict(num_rows=0, reduction=1), dict(loss=None))])
def test_loss_refuses(desc, call):
    lib = _lib.load()
    rc = lib.trips_table_loss_forward(call.get("ctx", C.addressof(CTX)), C.byref(_loss(**desc)), call.get("rows", AT), call.get("table", AT), call.get("target", AT),
                                      call.get("loss", AT), call.get("kept", AT), call.get("kept_size", 1 << 40), call.get("workspace", AT), call.get("size", 1 << 40), None)
    assert rc in ERR and lib.trips_last_error_string()


@pytest.mark.parametrize("desc,call", [(d, {}) for d in BAD_DESC] + [({}, c) for c in BAD_CALL] + [
    ({}, dict(d_loss=None)), ({}, dict(d_loss=AT + 2)), ({}, dict(size=_bytes(1) - 1)), ({}, dict(d_rows=AT + 2)), ({}, dict(d_table=AT + 1)),
    (dict(d_rows_stride=15), {}), (dict(d_table_stride=0), {}), (dict(d_table_stride=-1), {})])
def test_loss_backward_refuses(desc, call):
    lib = _lib.load()
    rc = lib.trips_table_loss_backward(call.get("ctx", C.addressof(CTX)), C.byref(_loss(**desc)), call.get("table", AT), call.get("kept", AT), call.get("kept_size", 1 << 40),
                                       call.get("d_loss", AT), call.get("d_rows", AT), call.get("d_table", AT), call.get("workspace", AT),
                                       call.get("size", 1 << 40), None)
    assert rc in ERR and lib.trips_last_error_string()


def test_workspaces_are_those_of_a_piece():
    """Not of the logits: 16,384 rows of a table of 262,143 entries would be 17 GB of them."""
    n = C.c_size_t(0)
    for dtype in (0, 2, 3):
        d = _loss(dtype=dtype, num_rows=16_384, num_entries=262_143, num_channels=1024, rows_stride=1024, table_stride=1024)
        for backward in (0, 1):
            assert _lib.load().trips_table_loss_workspace_size(C.byref(d), backward, C.byref(n)) == 0
            assert n.value < 3 << 30, (dtype, backward, n.value)


@pytest.mark.parametrize("desc,call", [(dict(abi_version=1), {}), (dict(dtype=1), {}), (dict(n=-1), {}), (dict(n=1 << 40), {}), (dict(p=-0.1), {}), (dict(p=1.1), {}), (dict(p=NAN), {}),
                                       ({}, dict(ctx=None)), ({}, dict(x=None)), ({}, dict(x=AT + 2)), ({}, dict(out=None)), ({}, dict(out=AT + 1)), ({}, dict(residual=AT + 2)),
                                       ({}, dict(step_at=AT + 2)), ({}, dict(step_used=AT + 1)), (dict(dtype=2), dict(x=AT + 1))])
def test_dropout_refuses(desc, call):
    lib = _lib.load()
    d = abi.TripsDropoutDesc(abi.TRIPS_ABI_VERSION, 0, 100, 0.5, 1, 2, 3)
    for k, v in desc.items():
        setattr(d, k, v)
    rc = lib.trips_dropout(call.get("ctx", C.addressof(CTX)), C.byref(d), call.get("x", AT), call.get("residual"), call.get("step_at"), call.get("step_used"),
                           call.get("out", AT), None)
    assert rc in ERR and lib.trips_last_error_string()


def test_python_refusals_without_a_gpu():
    from trips_amd.dropout import dropout
    from trips_amd.table_loss import table_cross_entropy
    x, w, target = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int32)
    for grad in (False, True):
        with pytest.raises(RuntimeError, match="GPU"):
            table_cross_entropy(x.requires_grad_(grad), w, target)
        with pytest.raises(RuntimeError, match="GPU"):
            dropout(x, 0.5, 1)
    with pytest.raises(ValueError, match="int32 or int64"):
        table_cross_entropy(x, w, target.float())
    with pytest.raises(ValueError, match="reduction"):
        table_cross_entropy(x, w, target, reduction="max")
    with pytest.raises(ValueError, match="32 bits"):
        dropout(x, 0.5, 1, call=-1)
    with pytest.raises(ValueError, match="p:"):
        dropout(x, 2.0, 1)
    with pytest.raises(ValueError, match="x:"):
        dropout(x.detach().long(), 0.5, 1)


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))])
def test_the_oracles_generator(counter, key, want):
    """The known answers that the generator was published with."""
    got = ref.philox(np.array([counter], dtype=np.uint64), key)
    assert tuple(int(v) for v in got[0]) == want


def test_the_oracles_gradients():
    """Loss's formulas against torch's in double precision, and its bound against float32's own error."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(30, 12, generator=g).requires_grad_(), torch.randn(70, 12, generator=g).requires_grad_()
    target = torch.randint(0, 70, (30,), generator=g)
    target[::4] = -1
    inside = target >= 0
    weights = torch.rand(30, generator=g) * inside
    want = ref.Loss(x, w, target, -0.7, weights.numpy())
    for dtype, bounds in ((torch.float64, None), (torch.float32, want)):
        a, b = x.detach().to(dtype).requires_grad_(), w.detach().to(dtype).requires_grad_()
        scale = float(np.float32(-0.7))
        losses = torch.nn.functional.cross_entropy(scale * a @ b.t(), target.clamp(min=0), reduction="none") * inside
        grads = torch.autograd.grad((losses * weights.to(dtype)).sum(), (a, b))
        for got, w_, bound in zip((losses, *grads), (want.losses, want.d_rows, want.d_table), (want.loss_bound, want.d_rows_bound, want.d_table_bound)):
            ref.within(got, w_, bound if bounds else np.full(w_.shape, 1e-12), "oracle")
