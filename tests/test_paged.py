"""Refusals of the operators over a paged cache and of their C entry points, the frequencies of a rotation, and the division that finds
a position's page. No GPU."""
import ctypes
import random

import pytest
import torch

import hexmi
from hexmi import _lib, ops


def test_frequencies():
    f = hexmi.rope_frequencies(8, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    for bad in (0, 3, -2):
        with pytest.raises(ValueError):
            hexmi.rope_frequencies(bad, device="cpu")
    with pytest.raises(ValueError):
        hexmi.rope_frequencies(8, 0.0, device="cpu")


def rows(**kw):
    q, k = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, 2, 64, dtype=torch.float16)
    w, f, p = torch.ones(64, dtype=torch.float16), torch.ones(32, dtype=torch.float64), torch.arange(3)
    return {**dict(q=q, k=k, q_weight=w, k_weight=w, inv_freq=f, positions=p), **kw}


@pytest.mark.parametrize("change, error", [
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float64)), TypeError), (dict(q=torch.zeros(3, 256, dtype=torch.float16)), ValueError),
    (dict(k=torch.zeros(3, 2, 64)), TypeError), (dict(k=torch.zeros(3, 2, 32, dtype=torch.float16)), ValueError),
    (dict(k=torch.zeros(2, 2, 64, dtype=torch.float16)), ValueError), (dict(q_weight=torch.ones(32, dtype=torch.float16)), ValueError),
    (dict(k_weight=torch.ones(64)), ValueError), (dict(k=None), ValueError), (dict(inv_freq=torch.ones(32)), TypeError),
    (dict(inv_freq=torch.ones(33, dtype=torch.float64)), ValueError), (dict(positions=None), ValueError),
    (dict(positions=torch.zeros(3)), ValueError), (dict(positions=torch.arange(4)), ValueError), (dict(pairs="both"), ValueError),
    (dict(k=None, k_weight=None, k_out=torch.zeros(3, 2, 64, dtype=torch.float16)), ValueError),
])
def test_rows_refusals(change, error):
    with pytest.raises(error, match="hexmi.qk_norm_rope"):
        hexmi.qk_norm_rope(**rows(**change))


def batch(**kw):
    """A call's arguments, the pages on the host: what comes before the pages' place is refused first."""
    t = torch.float16
    base = dict(k=torch.zeros(2, 2, 64, dtype=t), v=torch.zeros(2, 2, 64, dtype=t), k_pages=torch.zeros(3, 2, 16, 64, dtype=t),
                v_pages=torch.zeros(3, 2, 16, 64, dtype=t), page_table=torch.zeros(2, 2, dtype=torch.int32),
                lengths=torch.ones(2, dtype=torch.int32))
    return {**base, **kw}


@pytest.mark.parametrize("change, error", [
    (dict(k=torch.zeros(2, 2, 64)), TypeError), (dict(v=torch.zeros(2, 1, 64, dtype=torch.float16)), ValueError),
    (dict(k_pages=torch.zeros(3, 4, 16, 64, dtype=torch.float16)), ValueError), (dict(k_weight=torch.ones(2, dtype=torch.float16)), ValueError),
    (dict(inv_freq=torch.ones(8)), TypeError), (dict(q=torch.zeros(3, 4, 64, dtype=torch.float16)), ValueError),
    (dict(q_weight=torch.ones(64, dtype=torch.float16)), ValueError), (dict(pairs=1), ValueError),
    (dict(), ValueError),                                             # pages on the host
])
def test_append_refusals(change, error):
    with pytest.raises(error, match="hexmi.paged_append"):
        hexmi.paged_append(**batch(**change))


@pytest.mark.parametrize("change, error", [
    (dict(q=torch.zeros(2, 4, 64)), TypeError), (dict(q=torch.zeros(2, 3, 64, dtype=torch.float16)), ValueError),
    (dict(q=torch.zeros(2, 4, 32, dtype=torch.float16)), ValueError), (dict(sm_scale=0.0), ValueError), (dict(sm_scale=-1.0), ValueError),
    (dict(sm_scale=float("nan")), ValueError), (dict(shared_pages=torch.zeros(1)), ValueError),
    (dict(shared_pages=torch.zeros(3, dtype=torch.int32)), ValueError), (dict(), ValueError),
    (dict(q=torch.zeros(2, 4, 20, dtype=torch.float16), k_pages=torch.zeros(3, 2, 16, 20, dtype=torch.float16)), ValueError),
    (dict(q=torch.zeros(2, 4, 264, dtype=torch.float16), k_pages=torch.zeros(3, 2, 16, 264, dtype=torch.float16)), ValueError),
])
def test_attention_refusals(change, error):
    a = batch(q=torch.zeros(2, 4, 64, dtype=torch.float16))
    del a["k"], a["v"]
    with pytest.raises(error, match="hexmi.paged_attention"):
        hexmi.paged_attention(**{**a, **change})


class OnDevice(torch.Tensor):
    """A host tensor that says that it is on the GPU: the checks of ops.py behind the pages' place, without one."""
    device = property(lambda self: torch.device("cuda", 0))


@pytest.mark.parametrize("change", [
    dict(page_table=torch.zeros(2, 2, dtype=torch.int64)), dict(page_table=torch.zeros(3, 2, dtype=torch.int32)),
    dict(lengths=torch.ones(2)), dict(lengths=torch.ones(3, dtype=torch.int32)), dict(starts=torch.zeros(2, dtype=torch.int32)),
    dict(starts=torch.zeros(1, 3, dtype=torch.int32)), dict(v_pages=torch.zeros(3, 2, 16, 32, dtype=torch.float16)),
])
def test_batch_refusals(change):
    a = batch(starts=None)
    a = {**a, **change}
    pages = [a[n].as_subclass(OnDevice) for n in ("k_pages", "v_pages")]
    with pytest.raises(ValueError, match="hexmi.paged_append"):
        ops._paged_operands("paged_append", 2, *pages, a["page_table"], a["lengths"], a["starts"])
    strided = [torch.zeros(3, 2, 16, 128, dtype=torch.float16)[..., ::2].as_subclass(OnDevice)] * 2
    with pytest.raises(ValueError, match="adjacent"):
        ops._paged_operands("paged_append", 2, *strided, batch()["page_table"], batch()["lengths"], None)


def test_slices_of_one_projection_are_apart():
    wide = torch.zeros(5, 12 * 8)
    q, k, v = (t.unflatten(1, (-1, 8)) for t in wide.split((64, 16, 16), 1))
    assert ops._apart(q, k) and ops._apart(k, q) and ops._apart(v, q) and ops._apart(k, v)
    assert not ops._apart(q, q) and not ops._apart(q, wide.view(5, 12, 8)) and not ops._apart(q[:, 1:], q[:, :2])
    assert not ops._apart(q, wide.view(10, 6, 8)) and ops._apart(q[:2], q[2:])
    crossed = torch.zeros(5, 8, 2, 8)
    assert not ops._apart(crossed[:, :, 0], crossed[:, :, 1])          # interleaved heads: taken as shared



def c_batch(**kw):
    b = dict(k_pages=4096, v_pages=4096, k_page=2048, k_head=1024, k_slot=64, v_page=2048, v_head=1024, v_slot=64, num_pages=3, page_size=16,
             kv_heads=2, dim=64, page_table=4096, table_row=2, table_cols=2, lengths=4096, starts=None, sequences=2, tokens=2)
    return _lib.PagedBatch(**{**b, **kw})


def c_rows(heads=2, **kw):
    return _lib.HeadRows(**{**dict(x=4096, out=4096, weight=None, heads=heads, token=64 * heads, head=64, out_token=64 * heads, out_head=64), **kw})


TURN = dict(inv_freq=4096, columns=64, pairs=0, eps=1e-5)


@pytest.mark.parametrize("change, turn, status", [
    (dict(num_pages=0), {}, _lib.EINVAL), (dict(page_size=0), {}, _lib.EINVAL), (dict(sequences=3), {}, _lib.EINVAL),
    (dict(table_row=1), {}, _lib.EINVAL), (dict(tokens=-1), {}, _lib.EINVAL), (dict(lengths=None), {}, _lib.EINVAL),
    (dict(page_table=None), {}, _lib.EINVAL), (dict(k_pages=None), {}, _lib.EINVAL), (dict(kv_heads=3), {}, _lib.EINVAL),
    (dict(page_size=1 << 30, table_cols=2), {}, _lib.ENOTSUP), (dict(num_pages=1 << 32), {}, _lib.ENOTSUP),
    (dict(sequences=1 << 31, tokens=1 << 31), {}, _lib.ENOTSUP),
    ({}, dict(columns=63), _lib.EINVAL), ({}, dict(columns=66), _lib.EINVAL), ({}, dict(pairs=2), _lib.EINVAL), ({}, dict(inv_freq=None), _lib.EINVAL),
    (dict(tokens=0, sequences=0), {}, _lib.OK),
])
def test_append_entry_refuses_before_it_launches(change, turn, status):
    f = _lib.lib().hexmi_paged_append
    assert f(c_rows(), c_rows(), None, _lib.Rotation(**{**TURN, **turn}), c_batch(**change), _lib.F16, None) == status


def test_entries_refuse_missing_operands_and_types():
    lib, turn = _lib.lib(), _lib.Rotation(**TURN)
    assert lib.hexmi_paged_append(None, c_rows(), None, turn, c_batch(), _lib.F16, None) == _lib.EINVAL
    assert lib.hexmi_paged_append(c_rows(), c_rows(), None, None, c_batch(), _lib.F16, None) == _lib.EINVAL
    assert lib.hexmi_paged_append(c_rows(), c_rows(), None, turn, None, _lib.F16, None) == _lib.EINVAL
    assert lib.hexmi_paged_append(c_rows(), c_rows(), None, turn, c_batch(), _lib.F32, None) == _lib.ENOTSUP
    assert lib.hexmi_paged_append(c_rows(), c_rows(x=None), None, turn, c_batch(), _lib.F16, None) == _lib.EINVAL
    assert lib.hexmi_paged_append(c_rows(), c_rows(), c_rows(out=None), turn, c_batch(), _lib.F16, None) == _lib.EINVAL
    f = lib.hexmi_qk_norm_rope
    assert f(None, None, turn, 4096, 0, 3, 64, _lib.F16, None) == _lib.EINVAL
    assert f(c_rows(), None, turn, None, 0, 3, 64, _lib.F16, None) == _lib.EINVAL
    assert f(c_rows(), c_rows(out=None), turn, 4096, 0, 3, 64, _lib.F16, None) == _lib.EINVAL
    assert f(c_rows(), None, turn, 4096, 0, -1, 64, _lib.F16, None) == _lib.EINVAL
    assert f(c_rows(), None, turn, 4096, 0, 0, 64, _lib.F16, None) == _lib.OK
    assert f(c_rows(), None, turn, 4096, 0, 3, 600, _lib.F16, None) == _lib.ENOTSUP
    assert f(c_rows(), None, turn, 4096, 0, 3, 64, _lib.I8, None) == _lib.ENOTSUP


@pytest.mark.parametrize("change, q, shared, scale, dtype, status", [
    ({}, dict(heads=3), 0, 1.0, _lib.F16, _lib.EINVAL), ({}, dict(heads=4), 0, 0.0, _lib.F16, _lib.EINVAL),
    ({}, dict(heads=4), 0, float("inf"), _lib.F16, _lib.EINVAL), ({}, dict(heads=4), 3, 1.0, _lib.F16, _lib.EINVAL),
    ({}, dict(heads=4), -1, 1.0, _lib.F16, _lib.EINVAL), ({}, dict(heads=4), 0, 1.0, _lib.F32, _lib.ENOTSUP),
    (dict(dim=60), dict(heads=4), 0, 1.0, _lib.F16, _lib.ENOTSUP), (dict(dim=264), dict(heads=4), 0, 1.0, _lib.F16, _lib.ENOTSUP),
    (dict(k_slot=60), dict(heads=4), 0, 1.0, _lib.F16, _lib.ENOTSUP), (dict(v_pages=4098), dict(heads=4), 0, 1.0, _lib.F16, _lib.ENOTSUP),
    ({}, dict(heads=4, x=4104), 0, 1.0, _lib.F16, _lib.ENOTSUP), ({}, dict(heads=4, out=None), 0, 1.0, _lib.F16, _lib.EINVAL),
    (dict(lengths=None), dict(heads=4), 0, 1.0, _lib.F16, _lib.EINVAL), (dict(tokens=0, sequences=0), dict(heads=4), 0, 1.0, _lib.F16, _lib.OK),
])
def test_attention_entry_refuses_before_it_launches(change, q, shared, scale, dtype, status):
    f = _lib.lib().hexmi_paged_attention
    assert f(c_rows(**q), c_batch(**change), 4096, shared, scale, dtype, None, 0, None) == status


def test_division_by_a_product():
    """paged.h's divider: floor(n / d) of every n below 2^31 (the ends of the multiples of d, and others)."""
    rng = random.Random(1)
    for d in list(range(1, 300)) + [rng.randrange(1, 1 << 31) for _ in range(300)] + [1 << i for i in range(31)] + [(1 << 31) - 1]:
        shift = (d - 1).bit_length()
        m = ((1 << (31 + shift)) + d - 1) // d
        assert m < 1 << 32
        for n in [0, d - 1, d, (1 << 31) - 1] + [k * d + e for k in (1, 2, 7, ((1 << 31) - 1) // d) for e in (-1, 0, 1)] + [rng.randrange(1 << 31) for _ in range(20)]:
            if 0 <= n < 1 << 31:
                assert n * m >> 31 + shift == n // d, (n, d)


def test_more_rows_than_a_join_takes_are_refused():
    f = _lib.lib().hexmi_paged_attention
    big = dict(tokens=1 << 22, starts=4096)
    assert f(c_rows(heads=32), c_batch(**big), 4096, 1, 1.0, _lib.F16, 4096, 1 << 60, None) == _lib.ENOTSUP       # behind a prefix
    assert _lib.lib().hexmi_paged_attention_workspace(c_batch(**big), 32, 1) == 0
    assert f(c_rows(heads=32), c_batch(**big), 4096, 1, 1.0, _lib.F16, None, 0, None) == _lib.ENOTSUP


@pytest.mark.parametrize("slot", [-64, (1 << 26) + 8])
@pytest.mark.parametrize("which", ["k_slot", "v_slot"])
def test_slots_that_32_bit_offsets_do_not_reach_are_refused(which, slot):
    f = _lib.lib().hexmi_paged_attention
    assert f(c_rows(heads=4), c_batch(**{which: slot}), None, 0, 1.0, _lib.F16, 4096, 1 << 40, None) == _lib.ENOTSUP


@pytest.mark.parametrize("dim", range(8, 257, 8))
def test_tiles_copy_no_columns_past_a_head(dim):
    """What a tile copies of a key's row stands within the row, whatever the LDS row is wide: behind the last row of the pages there is
    nothing."""
    column = _lib.lib().hexmi_paged_tile_column
    chunks = [column(dim, c) for c in range(40)]
    row = chunks.index(-1)
    assert set(chunks[row:]) == {-1} and row * 8 >= dim
    assert chunks[:dim // 8] == list(range(0, dim, 8))                # the head's own chunks hold its own columns
    assert all(0 <= c and c + 8 <= dim for c in chunks[:row])
    assert all(column(d, 0) == -1 for d in (0, -8, dim + 1, 264)) and column(dim, -1) == -1


@pytest.mark.parametrize("sequences", [0, 1, 2, 70])
@pytest.mark.parametrize("shared", [0, 1])
@pytest.mark.parametrize("starts", [None, 4096])
def test_a_batch_without_new_tokens_is_nothing(sequences, shared, starts):
    """A step in which no sequence has a new token: no workspace, and nothing is launched."""
    lib = _lib.lib()
    b = c_batch(tokens=0, sequences=sequences if starts else 0, starts=starts)
    assert lib.hexmi_paged_attention_workspace(b, 4, shared) == 0
    assert lib.hexmi_paged_attention(c_rows(heads=4), b, 4096, shared, 1.0, _lib.F16, None, 0, None) == _lib.OK
    assert lib.hexmi_paged_append(c_rows(), c_rows(), c_rows(heads=4), _lib.Rotation(**TURN), b, _lib.F16, None) == _lib.OK
    assert lib.hexmi_paged_attention(c_rows(heads=3), b, 4096, shared, 1.0, _lib.F16, None, 0, None) == _lib.EINVAL      # refused as any other
