"""CPU-only checks of include/trips_optim.h and include/trips_lookup.h: symbols, sizes of the ctypes mirrors, and what the
entry points refuse before they touch a device."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

from tests import optim_reference as ref
from trips_amd import _lib, abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ERR = (abi.TRIPS_ERR_INVALID_ARG, abi.TRIPS_ERR_UNSUPPORTED, abi.TRIPS_ERR_WORKSPACE_SMALL)


@pytest.mark.parametrize("header,symbols", [("trips_optim.h", _lib.OPTIM_SYMBOLS), ("trips_lookup.h", _lib.LOOKUP_SYMBOLS)])
def test_library_exports_what_the_header_declares(header, symbols):
    lib = _lib.load()
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", header)).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(trips_[a-z0-9_]+)\s*\(", src)))
    assert names == sorted(symbols)
    for n in names:
        assert hasattr(lib, n)


def test_ctypes_mirrors_have_c_sizes(tmp_path):
    prog = tmp_path / "sizes.c"
    prog.write_text('#include <stdio.h>\n#include "trips_lookup.h"\nint main(){printf("%zu %zu %zu %zu %zu %zu %zu %d %d\\n",'
                    "sizeof(TripsAdamWTensor),offsetof(TripsAdamWTensor,lr),sizeof(TripsAdamWOptions),offsetof(TripsAdamWOptions,grad_norm),"
                    "sizeof(TripsGradTensor),sizeof(TripsLookupDesc),offsetof(TripsLookupDesc,scale),"
                    "TRIPS_GRAD_NORM_WORKSPACE_BYTES,TRIPS_MOMENT_BLOCK);return 0;}\n")
    exe = tmp_path / "sizes"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(prog), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert got == [C.sizeof(abi.TripsAdamWTensor), abi.TripsAdamWTensor.lr.offset, C.sizeof(abi.TripsAdamWOptions),
                   abi.TripsAdamWOptions.grad_norm.offset, C.sizeof(abi.TripsGradTensor), C.sizeof(abi.TripsLookupDesc),
                   abi.TripsLookupDesc.scale.offset, abi.TRIPS_GRAD_NORM_WORKSPACE_BYTES, abi.TRIPS_MOMENT_BLOCK]


# A context stands behind a pointer that is not looked into before all arguments are checked; addresses are never used here.
CTX = C.create_string_buffer(4096)
AT = 1 << 20


def _step_bytes(n):
    b = C.c_size_t(0)
    assert _lib.load().trips_adamw_workspace_size(n, C.byref(b)) == 0
    return b.value


STEP_BYTES = _step_bytes(2)


def _tensor(**kw):
    t = abi.TripsAdamWTensor(AT, AT, AT, AT, AT, AT, None, AT, 1000, 0, 0, 0, 32, 1e-3, 0.9, 0.999, 1e-8, 0.01)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def _options(**kw):
    o = abi.TripsAdamWOptions(abi.TRIPS_ABI_VERSION, 0, None, 0, 0.0, 1.0)
    for k, v in kw.items():
        setattr(o, k, v)
    return o


NAN = float("nan")


@pytest.mark.parametrize("tensor,options,call", [
    (dict(n=-1), {}, {}), (dict(n=1 << 39), {}, {}), (dict(weights=None), {}, {}), (dict(grads=None), {}, {}),
    (dict(first_moment=None), {}, {}), (dict(second_moment=None), {}, {}), (dict(step=None), {}, {}), (dict(step=AT + 2), {}, {}),
    (dict(state_bits=8, first_scale=None), {}, {}), (dict(state_bits=8, second_scale=AT + 1), {}, {}), (dict(state_bits=4), {}, {}),
    (dict(weight_dtype=abi.TRIPS_DTYPE_F64), {}, {}), (dict(grad_dtype=7), {}, {}), (dict(copy=AT, copy_dtype=1), {}, {}),
    (dict(weights=AT + 2), {}, {}), (dict(weights=AT + 1, weight_dtype=2), {}, {}), (dict(first_moment=AT + 1), {}, {}),
    (dict(copy=AT + 1, copy_dtype=2), {}, {}), (dict(beta1=1.0), {}, {}), (dict(beta2=-0.1), {}, {}), (dict(beta1=NAN), {}, {}),
    (dict(lr=NAN), {}, {}), (dict(lr=-1.0), {}, {}), (dict(eps=float("inf")), {}, {}), (dict(weight_decay=-1.0), {}, {}),
    ({}, dict(abi_version=1), {}), ({}, dict(compute_norm=1), {}), ({}, dict(max_norm=1.0), {}), ({}, dict(max_norm=NAN), {}),
    ({}, dict(loss_scale=0.0), {}), ({}, dict(loss_scale=NAN), {}), ({}, dict(loss_scale=float("inf")), {}),
    ({}, dict(grad_norm=AT + 1), {}),
    ({}, {}, dict(workspace=None)), ({}, {}, dict(workspace=AT + 128)), ({}, {}, dict(size=STEP_BYTES - 1)),
    ({}, {}, dict(ctx=None)), ({}, {}, dict(count=-1)),
])
def test_adamw_refuses(tensor, options, call):
    lib = _lib.load()
    tensors = (abi.TripsAdamWTensor * 2)(_tensor(), _tensor(**tensor))
    rc = lib.trips_adamw_step(call.get("ctx", C.addressof(CTX)), tensors, call.get("count", 2), C.byref(_options(**options)),
                              call.get("workspace", AT), call.get("size", STEP_BYTES), None)
    assert rc in ERR and lib.trips_last_error_string()


@pytest.mark.parametrize("tensor,call", [
    (dict(n=-1), {}), (dict(grads=None), {}), (dict(grads=AT + 2), {}), (dict(dtype=1), {}), ({}, dict(out=None)), ({}, dict(out=AT + 2)),
    ({}, dict(max_norm=NAN)), ({}, dict(loss_scale=-1.0)), ({}, dict(workspace=None)), ({}, dict(size=100)), ({}, dict(count=-1)),
])
def test_norm_refuses(tensor, call):
    lib = _lib.load()
    t = abi.TripsGradTensor(AT, 1000, 0)
    for k, v in tensor.items():
        setattr(t, k, v)
    tensors = (abi.TripsGradTensor * 1)(t)
    rc = lib.trips_grad_norm(C.addressof(CTX), tensors, call.get("count", 1), call.get("max_norm", 1.0), call.get("loss_scale", 1.0),
                             call.get("out", AT), call.get("workspace", AT), call.get("size", abi.TRIPS_GRAD_NORM_WORKSPACE_BYTES), None)
    assert rc in ERR and lib.trips_last_error_string()


def _lookup(**kw):
    d = abi.TripsLookupDesc(abi.TRIPS_ABI_VERSION, 0, 0, 1, 100, 50, 4, 0, 100, 50, 1.0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD_DESC = [dict(abi_version=1), dict(layout=2), dict(dtype=1), dict(dtype=9), dict(index_dtype=2), dict(num_texels=-1),
            dict(num_texels=0x7fffffff), dict(num_points=-1), dict(num_points=1 << 31), dict(num_channels=0), dict(num_channels=1 << 20),
            dict(table_stride=-1), dict(values_stride=-1)]


@pytest.mark.parametrize("desc,call", [(d, {}) for d in BAD_DESC] + [
    (dict(values_stride=49), {}), (dict(layout=1, values_stride=3), {}), ({}, dict(table=None)), ({}, dict(table=AT + 2)),
    ({}, dict(index=None)), ({}, dict(index=AT + 2)), (dict(index_dtype=0), dict(index=AT + 4)), ({}, dict(values=None)),
    (dict(dtype=2), dict(values=AT + 1)), ({}, dict(ctx=None)), ({}, dict(workspace=None)),
    ({}, dict(workspace=AT + 16)), ({}, dict(size=100))])
def test_lookup_refuses(desc, call):
    lib = _lib.load()
    rc = lib.trips_lookup_forward(call.get("ctx", C.addressof(CTX)), C.byref(_lookup(**desc)), call.get("table", AT), call.get("index", AT),
                                  call.get("values", AT), call.get("workspace", AT), call.get("size", 1 << 30), None)
    assert rc in ERR and lib.trips_last_error_string()


@pytest.mark.parametrize("desc,call", [(d, {}) for d in BAD_DESC] + [
    (dict(table_stride=99), {}), (dict(layout=1, table_stride=3), {}), ({}, dict(d_values=None)), ({}, dict(order=None)), ({}, dict(order=AT + 1)),
    ({}, dict(starts=None)), ({}, dict(d_table=None)), (dict(dtype=3), dict(d_table=AT + 1)), ({}, dict(workspace=None)),
    ({}, dict(size=255)), (dict(num_points=1000), dict(size=700)), (dict(layout=1, table_stride=4, values_stride=4, num_points=1_000_000), dict(size=700))])
def test_lookup_backward_refuses(desc, call):
    lib = _lib.load()
    rc = lib.trips_lookup_backward(C.addressof(CTX), C.byref(_lookup(**desc)), call.get("d_values", AT), call.get("order", AT),
                                   call.get("starts", AT), call.get("d_table", AT), call.get("workspace", AT), call.get("size", 1 << 30), None)
    assert rc in ERR and lib.trips_last_error_string()


@pytest.mark.parametrize("call", [dict(texels=-1), dict(texels=0x7fffffff), dict(points=-1), dict(points=1 << 31), dict(index_dtype=2),
                                  dict(index=None), dict(index=AT + 2), dict(order=None), dict(starts=None), dict(starts=AT + 2),
                                  dict(workspace=None), dict(workspace=AT + 8), dict(size=10)])
def test_plan_refuses(call):
    lib = _lib.load()
    n = C.c_size_t(0)
    if "texels" in call or "points" in call:
        assert lib.trips_lookup_plan_workspace_size(call.get("texels", 100), call.get("points", 50_000), C.byref(n)) in ERR
    rc = lib.trips_lookup_plan(C.addressof(CTX), call.get("texels", 100), call.get("points", 50_000), call.get("index", AT),
                               call.get("index_dtype", 1), call.get("order", AT), call.get("starts", AT), call.get("workspace", AT),
                               call.get("size", 1 << 30), None)
    assert rc in ERR and lib.trips_last_error_string()


def test_python_refusals_without_a_gpu():
    import torch
    from trips_amd import lookup
    from trips_amd.adamw import AdamW, grad_norm
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="GPU"):
        AdamW([p]).step()
    with pytest.raises(RuntimeError, match="GPU"):
        grad_norm([p.grad])
    with pytest.raises(RuntimeError, match="GPU"):
        lookup.lookup(torch.zeros(4, 4), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="int32 or int64"):
        lookup.lookup(torch.zeros(4, 4), torch.zeros(3))
    with pytest.raises(ValueError, match="layout"):
        lookup.lookup(torch.zeros(4, 4), torch.zeros(3, dtype=torch.int32), layout=5)


def test_the_oracles_8_bit_floats_are_torchs():
    """What the oracle decodes, against the types that the codes are kept in; and its rounding leaves representable numbers alone."""
    import torch
    codes = np.arange(256)
    for dtype, mantissa, bias, largest in ((torch.float8_e4m3fn, 3, 7, 448.0), (torch.float8_e5m2, 2, 15, 57344.0)):
        want = torch.arange(256, dtype=torch.uint8).view(dtype).double().numpy()
        finite = np.isfinite(want)
        np.testing.assert_array_equal(ref.fp8_values(mantissa, bias, codes)[finite], want[finite])
        assert np.nanmax(want[finite]) == largest
        x = want[finite & (want >= 0)]
        got, scale, _ = ref.encode(x, np.full(x.size, 65535.0 * 0.3).astype(int).astype(float), mantissa, bias, largest, False)
        np.testing.assert_array_equal(ref.decode(got, scale, mantissa, bias), x)


def test_mixed_bits_are_even_and_independent():
    """The two halves that round a moment each: means, and correlations between halves, neighbours, steps and seeds, within 5
    deviations of those of independent uniform numbers (2^20 of them)."""
    n = 1 << 20
    place = np.arange(n, dtype=np.uint64)
    draws = []
    for seed, t in ((0, 1), (0, 2), (1, 1)):
        bits = ref.mix(place ^ ref.mix(seed + t * 0x9E3779B9))
        for half in (bits & np.uint64(0xFFFF), bits >> np.uint64(16)):
            u = (half.astype(np.float64) + 0.5) / 65536 - 0.5
            assert abs(u.mean()) < 5 * np.sqrt(1 / 12 / n)
            assert abs((u[1:] * u[:-1]).mean() * 12) < 5 / np.sqrt(n)
            draws.append(u)
    for i in range(len(draws)):
        for j in range(i):
            assert abs((draws[i] * draws[j]).mean() * 12) < 5 / np.sqrt(n), (i, j)
