"""What the cross entropy takes and refuses at the ends of its ranges, and what it asks for in memory there. On the CPU: sizes and refusals touch no device."""
import ctypes as C

import pytest
import torch

from trips_amd import _lib, abi

F32, BF16, F16 = 0, 2, 3


def _desc(n, t, c, dtype=F32, scale=1.0):
    return abi.TripsTableLossDesc(abi.TRIPS_ABI_VERSION, dtype, abi.TRIPS_INDEX_I64, abi.TRIPS_REDUCE_MEAN, n, t, c, scale, c, c, c, c)


def _workspace(backward, *args, **kw):
    bytes_ = C.c_size_t(0)
    rc = _lib.load().trips_table_loss_workspace_size(C.byref(_desc(*args, **kw)), backward, C.byref(bytes_))
    return rc, bytes_.value


@pytest.mark.parametrize("scale,taken", [(2.35e38, True), (-2.35e38, True), (2.4e38, False), (-3.4e38, False), (1e-45, True), (0.0, True)])
def test_scales(scale, taken):
    """What the kernels multiply by is scale log2 e: infinite from 2.36e38 on."""
    rc, _ = _workspace(0, 10, 10, 8, scale=scale)
    assert rc == (abi.TRIPS_OK if taken else abi.TRIPS_ERR_INVALID_ARG)
    assert taken or b"scale" in _lib.load().trips_last_error_string()


def test_refusals_name_what_they_refuse():
    """The targets and the cross entropy, not an index and lookups."""
    from trips_amd.table_loss import table_cross_entropy
    x, w, target = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int32)
    for grad in (False, True):
        x.requires_grad_(grad)
        with pytest.raises(ValueError, match="^target: int32 or int64"):
            table_cross_entropy(x, w, target.float())
        with pytest.raises(RuntimeError, match="^the cross entropy needs tensors on a GPU"):
            table_cross_entropy(x, w, target)
    from trips_amd.lookup import lookup
    with pytest.raises(ValueError, match="^index: int32 or int64"):
        lookup(w, target.float())
    with pytest.raises(RuntimeError, match="^lookups need tensors on a GPU"):
        lookup(w, target)


@pytest.mark.parametrize("n,taken", [((1 << 28) - 16, True), ((1 << 28) - 15, False), ((1 << 28) - 1, False)])
def test_rows(n, taken):
    """A launch of 16 threads a row has fewer than 2^32."""
    assert _workspace(0, n, 2, 1)[0] == (abi.TRIPS_OK if taken else abi.TRIPS_ERR_INVALID_ARG)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,t", [(131_072, 262_144), (262_144, 262_144), (8191, 2_000_000_000), (300_000, 20_000_000), (1 << 26, 66_000), (1 << 26, 33_000), (5, 2_000_000_000), (1, 1), (0, 0), (0, 5), (5, 0)])
@pytest.mark.parametrize("c", [1, 8, 1000])
def test_the_losss_workspace_does_not_grow_with_rows_times_entries(n, t, c, dtype):
    """Maxima and sums of a GiB of tiles at once, or of 256 entries (four tiles at most, of 8 bytes a row each); 64 MiB of entries that are copied, or 256 of
    them; 8 bytes a row besides."""
    rc, got = _workspace(0, n, t, c, dtype)
    assert rc == abi.TRIPS_OK
    assert got <= max(1 << 30, n * 4 * 8) + max(64 << 20, 256 * 4 * (c + 8)) + 8 * n + (1 << 20), got / 2 ** 30


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,t,c", [(6_000_000, 150, 16), (6_000_000, 2, 16), (1_000_000, 2, 16), (1_100_000, 40, 6), (1 << 21, 256, 1000), (100_000_000, 33, 3), (1 << 27, 100_000, 16),
                                   (16_384, 262_143, 1024), (500_000, 70_000, 64), (3, 200_000, 2000), (5, 1, 1)])
def test_the_gradients_workspace_is_bounded(n, t, c, dtype):
    """A GiB of d_ij, a quarter of that of a gradient's parts or one part of it in 32 bits (of a million rows at most, of the table where there are more rows than that, else of a
    piece of it), copied entries, and small things: whatever the rows times the entries are."""
    rc, got = _workspace(1, n, t, c, dtype)
    assert rc == abi.TRIPS_OK
    padded = 4 * (c + 8)
    rows, table = (min(n, 1 << 20) + 256) * padded, (t + 65536) * padded
    assert got <= (1 << 30) + max(256 << 20, rows) + max(256 << 20, table) + max(64 << 20, 256 * padded) + (1 << 20), got / 2 ** 30


def test_few_entries_take_no_more_than_whole_tiles():
    """1000 rows and two entries: d_ij in 64 columns (the least step of the gradients), not in 256."""
    assert _workspace(1, 1000, 2, 16)[1] < _workspace(1, 1000, 200, 16)[1] - 1024 * 64 * 4
