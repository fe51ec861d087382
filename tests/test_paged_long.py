"""Refusals of a paged cache in 8 bits, of windows, forks and compaction, and of their C entry points. No GPU."""
import os
import shutil
import subprocess

import pytest
import torch

import hexmi
from hexmi import _lib, ops

E4M3 = torch.float8_e4m3fn


class OnDevice(torch.Tensor):
    """A host tensor that says that it is on the GPU: the checks behind the pages' place, without one."""
    device = property(lambda self: torch.device("cuda", 0))


def batch(**kw):
    t = torch.float16
    base = dict(k_pages=torch.zeros(3, 2, 16, 64, dtype=E4M3), v_pages=torch.zeros(3, 2, 16, 64, dtype=E4M3),
                page_table=torch.zeros(2, 2, dtype=torch.int32), lengths=torch.ones(2, dtype=torch.int32),
                k_scales=torch.zeros(3, 2, 1, dtype=torch.uint8), v_scales=torch.zeros(3, 2, 1, dtype=torch.uint8))
    return {**base, **kw}


SCALES = [
    (dict(k_scales=None), TypeError), (dict(v_scales=None), TypeError), (dict(k_scales=None, v_scales=None), TypeError),
    (dict(k_scales=torch.zeros(3, 2, 1)), TypeError), (dict(k_pages=torch.zeros(3, 2, 16, 64, dtype=torch.float16)), TypeError),
    (dict(k_scales=torch.zeros(3, 2, dtype=torch.uint8)), ValueError), (dict(v_scales=torch.zeros(3, 2, 2, dtype=torch.uint8)), ValueError),
    ({n: torch.zeros(3, 2, 3, dtype=torch.uint8) for n in ("k_scales", "v_scales")}, ValueError),
    ({n: torch.zeros(3, 2, 0, dtype=torch.uint8) for n in ("k_scales", "v_scales")}, ValueError),
    ({n: torch.zeros(2, 2, 1, dtype=torch.uint8) for n in ("k_scales", "v_scales")}, ValueError),
    ({**{n: torch.zeros(3, 2, 128, 64, dtype=E4M3) for n in ("k_pages", "v_pages")}}, ValueError),       # blocks of 128
    (dict(), ValueError),                                             # pages on the host
]


@pytest.mark.parametrize("change, error", SCALES)
def test_scales_refusals(change, error):
    a = batch(**change)
    rows = torch.zeros(2, 2, 64, dtype=torch.float16)
    with pytest.raises(error, match="hexmi.paged_append"):
        hexmi.paged_append(rows, rows.clone(), **a)
    with pytest.raises(error, match="hexmi.paged_attention"):
        hexmi.paged_attention(rows, **a)
    index = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(error, match="hexmi.paged_fork"):
        hexmi.paged_fork(parents=index, pages=index, **a)
    with pytest.raises(error, match="hexmi.paged_compact"):
        hexmi.paged_compact(**a)


@pytest.mark.parametrize("change, error", [
    (dict(k=torch.zeros(2, 2, 64)), TypeError), (dict(k=torch.zeros(2, 2, 60, dtype=torch.float16)), ValueError),
])
def test_append_refusals(change, error):
    a = batch(k=torch.zeros(2, 2, 64, dtype=torch.float16), v=torch.zeros(2, 2, 64, dtype=torch.float16))
    with pytest.raises(error, match="hexmi.paged_append"):
        hexmi.paged_append(**{**a, **change})


def test_append_in_8_bits_refuses_other_dims():
    for dim in (20, 264):
        a = batch(**{n: torch.zeros(3, 2, 16, dim, dtype=E4M3) for n in ("k_pages", "v_pages")})
        with pytest.raises(ValueError, match="multiple of 8"):
            hexmi.paged_append(*(torch.zeros(2, 2, dim, dtype=torch.float16) for _ in range(2)), **a)


def test_append_refuses_scales_that_are_one_tensor():
    scales = torch.zeros(3, 2, 1, dtype=torch.uint8)
    rows = torch.zeros(2, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="scales of their own"):
        hexmi.paged_append(rows, rows.clone(), **batch(k_scales=scales, v_scales=scales))
    s = c_scales(v_scales=4096)
    assert _lib.lib().hexmi_paged_append_ex(c_rows(), c_rows(), None, TURN, c_batch(), s, _lib.F16, None) == _lib.EINVAL


@pytest.mark.parametrize("window, sinks", [(0, 0), (-1, 0), (2.0, 0), (True, 0), (5, -1), (5, 1.0), (None, 4), (torch.tensor(4), 0)])
def test_window_refusals(window, sinks):
    with pytest.raises(ValueError, match="window"):
        hexmi.paged_attention(torch.zeros(2, 2, 64, dtype=torch.float16), **batch(), window=window, sinks=sinks)
    with pytest.raises(ValueError, match="window"):
        hexmi.paged_compact(**batch(), window=window, sinks=sinks)


def test_no_shared_pages_within_a_window():
    with pytest.raises(ValueError, match="shared pages"):
        hexmi.paged_attention(torch.zeros(2, 2, 64, dtype=torch.float16), **batch(), window=5, shared_pages=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("change", [
    dict(parents=torch.zeros(2)), dict(pages=torch.zeros(3, dtype=torch.int32)), dict(parents=torch.zeros(1, 2, dtype=torch.int32)),
])
def test_fork_refusals(change):
    index = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="hexmi.paged_fork"):
        hexmi.paged_fork(**{**batch(), "parents": index, "pages": index, **change})


def test_pages_that_are_copied_are_of_16_bits_or_8():
    pages = [torch.zeros(3, 2, 16, 64) for _ in range(2)]
    with pytest.raises(TypeError, match="hexmi.paged_compact"):
        hexmi.paged_compact(*pages, torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    one = torch.zeros(3, 2, 16, 64, dtype=torch.float16).as_subclass(OnDevice)
    with pytest.raises(ValueError, match="pages of their own"):
        hexmi.paged_compact(one, one, torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32))


def test_index_results_are_checked():
    dev = torch.device("cpu")
    for bad in (torch.zeros(2, 3), torch.zeros(3, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="table_out"):
            ops._index_out("paged_fork", "table_out", bad, (2, 3), (), dev)
    good = torch.zeros(2, 3, dtype=torch.int32)
    assert ops._index_out("paged_fork", "table_out", good, (2, 3), (None,), dev) is good
    assert ops._index_out("paged_fork", "table_out", good, (2, 3), (good[1:],), dev) is not good


def test_batches_of_16_bits_are_as_large_as_before_there_were_8():
    """What a unit counts for beside its own blocks of 128 keys belongs to a cache in 8 bits: in 16, 2090000 sequences of 1026 blocks and one more
    each stay below 2^31."""
    lib, q = _lib.lib(), c_rows(heads=1)
    of = lambda blocks: c_batch(kv_heads=1, table_cols=blocks * 8, table_row=blocks * 8, sequences=2090000, tokens=65536, starts=4096)
    need = lambda blocks, s=None: lib.hexmi_paged_attention_ex_workspace(of(blocks), 1, 0, s, 0, 0)
    assert need(1026) > 0 and need(1027) == 0 and need(1025, c_scales()) > 0 and need(1026, c_scales()) == 0
    assert lib.hexmi_paged_attention_workspace(of(1026), 1, 0) == need(1026)
    # past that check (to a workspace that is too small), and not
    assert lib.hexmi_paged_attention(q, of(1026), None, 0, 1.0, _lib.F16, 4096, 1, None) == _lib.EINVAL
    assert lib.hexmi_paged_attention(q, of(1027), None, 0, 1.0, _lib.F16, 4096, 1, None) == _lib.ENOTSUP
    for blocks, status in ((1025, _lib.EINVAL), (1026, _lib.ENOTSUP)):
        assert lib.hexmi_paged_attention_ex(q, of(blocks), c_scales(), None, 0, 0, 0, 1.0, _lib.F16, 4096, 1, None) == status


def c_batch(**kw):
    b = dict(k_pages=4096, v_pages=4096, k_page=2048, k_head=1024, k_slot=64, v_page=2048, v_head=1024, v_slot=64, num_pages=3, page_size=16,
             kv_heads=2, dim=64, page_table=4096, table_row=2, table_cols=2, lengths=4096, starts=None, sequences=2, tokens=2)
    return _lib.PagedBatch(**{**b, **kw})


def c_rows(heads=2, **kw):
    return _lib.HeadRows(**{**dict(x=4096, out=4096, weight=None, heads=heads, token=64 * heads, head=64, out_token=64 * heads, out_head=64), **kw})


def c_scales(**kw):
    return _lib.PagedScales(**{**dict(k_scales=4096, v_scales=8192, k_page=2, k_head=1, k_block=1, v_page=2, v_head=1, v_block=1, block=16), **kw})


TURN = _lib.Rotation(inv_freq=4096, columns=64, pairs=0, eps=1e-5)
BAD_SCALES = [(dict(block=0), _lib.EINVAL), (dict(block=3), _lib.EINVAL), (dict(k_scales=None), _lib.EINVAL), (dict(v_scales=None), _lib.EINVAL)]


@pytest.mark.parametrize("change, status", BAD_SCALES)
def test_entries_refuse_bad_scales(change, status):
    lib, s = _lib.lib(), c_scales(**change)
    assert lib.hexmi_paged_append_ex(c_rows(), c_rows(), None, TURN, c_batch(), s, _lib.F16, None) == status
    assert lib.hexmi_paged_attention_ex(c_rows(heads=4), c_batch(), s, None, 0, 0, 0, 1.0, _lib.F16, 4096, 1 << 40, None) == status
    assert lib.hexmi_paged_fork(c_batch(), s, 4096, 4096, 2, 4096, 2, 4096, _lib.F16, None) == status
    assert lib.hexmi_paged_compact(c_batch(), s, 0, 0, 4096, 2, 4096, _lib.F16, 4096, 1 << 40, None) == status


def test_blocks_of_more_than_64_slots_are_refused():
    lib, s, b = _lib.lib(), c_scales(block=128), c_batch(page_size=128)
    assert lib.hexmi_paged_append_ex(c_rows(), c_rows(), None, TURN, b, s, _lib.F16, None) == _lib.ENOTSUP
    assert lib.hexmi_paged_attention_ex(c_rows(heads=4), b, s, None, 0, 0, 0, 1.0, _lib.F16, 4096, 1 << 40, None) == _lib.ENOTSUP


@pytest.mark.parametrize("change, rows, status", [
    (dict(k_slot=60), {}, _lib.ENOTSUP), (dict(v_pages=4100), {}, _lib.ENOTSUP), ({}, dict(x=4104), _lib.ENOTSUP), ({}, dict(token=4), _lib.ENOTSUP),
    (dict(dim=60), {}, _lib.EINVAL), (dict(dim=264), {}, _lib.ENOTSUP), (dict(kv_heads=3), {}, _lib.EINVAL), (dict(lengths=None), {}, _lib.EINVAL),
    (dict(k_pages=None), {}, _lib.EINVAL), (dict(tokens=0, sequences=0), {}, _lib.OK),
])
def test_append_entry_refuses_before_it_launches(change, rows, status):
    f = _lib.lib().hexmi_paged_append_ex
    assert f(c_rows(**rows), c_rows(), None, TURN, c_batch(**change), c_scales(), _lib.F16, None) == status
    assert f(None, c_rows(), None, TURN, c_batch(), c_scales(), _lib.F16, None) == _lib.EINVAL
    assert f(c_rows(), c_rows(), None, TURN, c_batch(), c_scales(), _lib.F32, None) == _lib.ENOTSUP
    assert f(c_rows(), c_rows(), c_rows(out=4104), TURN, c_batch(), c_scales(), _lib.F16, None) == _lib.ENOTSUP


@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("change, q, shared, window, sinks, scale, dtype, status", [
    ({}, dict(heads=3), 0, 5, 0, 1.0, _lib.F16, _lib.EINVAL), ({}, {}, 0, -1, 0, 1.0, _lib.F16, _lib.EINVAL), ({}, {}, 0, 5, -1, 1.0, _lib.F16, _lib.EINVAL),
    ({}, {}, 1, 5, 0, 1.0, _lib.F16, _lib.ENOTSUP), ({}, {}, 0, 5, 0, 0.0, _lib.F16, _lib.EINVAL), ({}, {}, 0, 5, 0, 1.0, _lib.F32, _lib.ENOTSUP),
    (dict(dim=60), {}, 0, 5, 0, 1.0, _lib.F16, _lib.ENOTSUP), (dict(k_slot=60), {}, 0, 5, 0, 1.0, _lib.F16, _lib.ENOTSUP),
    (dict(k_slot=-64), {}, 0, 5, 0, 1.0, _lib.F16, _lib.ENOTSUP), (dict(v_slot=(1 << 26) + 64), {}, 0, 5, 0, 1.0, _lib.F16, _lib.ENOTSUP),
    (dict(v_pages=4100), {}, 0, 5, 0, 1.0, _lib.F16, _lib.ENOTSUP), ({}, dict(x=4104), 0, 5, 0, 1.0, _lib.F16, _lib.ENOTSUP),
    ({}, dict(out=None), 0, 5, 0, 1.0, _lib.F16, _lib.EINVAL), (dict(lengths=None), {}, 0, 5, 0, 1.0, _lib.F16, _lib.EINVAL),
    (dict(tokens=0, sequences=0), {}, 0, 5, 0, 1.0, _lib.F16, _lib.OK), ({}, {}, 3, 0, 0, 1.0, _lib.F16, _lib.EINVAL),
])
def test_attention_entry_refuses_before_it_launches(scaled, change, q, shared, window, sinks, scale, dtype, status):
    f = _lib.lib().hexmi_paged_attention_ex
    s = c_scales() if scaled else None
    assert f(c_rows(**{"heads": 4, **q}), c_batch(**change), s, 4096, shared, window, sinks, scale, dtype, 4096, 1 << 40, None) == status


def test_pages_in_8_bits_off_their_boundaries_are_refused():
    f = _lib.lib().hexmi_paged_attention_ex
    for change in (dict(k_pages=4104), dict(v_slot=72, v_head=1152, v_page=2304)):
        assert f(c_rows(heads=4), c_batch(**change), c_scales(), None, 0, 0, 0, 1.0, _lib.F16, 4096, 1 << 40, None) == _lib.ENOTSUP


def test_fork_and_compact_entries_refuse_before_they_launch():
    lib = _lib.lib()
    fork = lambda b=c_batch(), s=c_scales(), parents=4096, pages=4096, rows=2, table=4096, pitch=2, lengths=4096, dtype=_lib.F16: \
        lib.hexmi_paged_fork(b, s, parents, pages, rows, table, pitch, lengths, dtype, None)
    assert fork(b=None) == _lib.EINVAL and fork(parents=None) == _lib.EINVAL and fork(pages=None) == _lib.EINVAL
    assert fork(table=None) == _lib.EINVAL and fork(lengths=None) == _lib.EINVAL and fork(pitch=1) == _lib.EINVAL and fork(rows=-1) == _lib.EINVAL
    assert fork(dtype=_lib.F32) == _lib.ENOTSUP and fork(rows=0) == _lib.OK and fork(b=c_batch(k_pages=None)) == _lib.EINVAL
    assert fork(b=c_batch(lengths=None)) == _lib.EINVAL and fork(b=c_batch(num_pages=0)) == _lib.EINVAL and fork(rows=1 << 40) == _lib.ENOTSUP
    compact = lambda b=c_batch(), s=c_scales(), window=0, sinks=0, table=4096, pitch=2, count=4096, dtype=_lib.F16, ws=4096, room=1 << 40: \
        lib.hexmi_paged_compact(b, s, window, sinks, table, pitch, count, dtype, ws, room, None)
    assert compact(b=None) == _lib.EINVAL and compact(window=-1) == _lib.EINVAL and compact(sinks=-1) == _lib.EINVAL
    assert compact(table=None) == _lib.EINVAL and compact(count=None) == _lib.EINVAL and compact(pitch=1) == _lib.EINVAL
    assert compact(ws=None) == _lib.EINVAL and compact(ws=4100) == _lib.EINVAL and compact(dtype=_lib.F32) == _lib.ENOTSUP
    need = lib.hexmi_paged_compact_workspace(c_batch())
    assert need > 0 and compact(room=need - 1) == _lib.EINVAL
    assert lib.hexmi_paged_compact_workspace(c_batch(num_pages=0)) == 0 and lib.hexmi_paged_compact_workspace(None) == 0


@pytest.mark.parametrize("ahead", [-1, 1.0, True, None])
def test_compact_refuses_what_is_no_number_of_positions(ahead):
    with pytest.raises(ValueError, match="ahead"):
        hexmi.paged_compact(**batch(), ahead=ahead)
    if ahead == -1:
        assert _lib.lib().hexmi_paged_compact_ex(c_batch(), c_scales(), None, 0, 0, 0, ahead, 4096, 2, None, 4096, _lib.F16, 4096, 1 << 40, None) == _lib.EINVAL


def test_compact_refuses_bad_shared_pages():
    for bad in (torch.zeros(1), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="hexmi.paged_compact: shared_pages"):
            hexmi.paged_compact(**batch(), shared_pages=bad)
    with pytest.raises(ValueError, match="no shared pages within a window"):
        hexmi.paged_compact(**batch(), shared_pages=torch.zeros(1, dtype=torch.int32), window=5)
    f = _lib.lib().hexmi_paged_compact_ex
    call = lambda pages, n, out, window=0: f(c_batch(), c_scales(), pages, n, window, 0, 0, 4096, 2, out, 4096, _lib.F16, 4096, 1 << 40, None)
    assert call(None, 1, 4096) == call(4096, 1, None) == call(4096, 3, 4096) == call(4096, -1, 4096) == _lib.EINVAL
    assert call(4096, 1, 4096, window=5) == _lib.ENOTSUP


@pytest.mark.parametrize("change", [dict(k_page=1 << 32), dict(v_page=-2048)])
def test_strides_past_32_bits_are_refused_within_a_window(change):
    f = _lib.lib().hexmi_paged_attention_ex
    for scales, window in ((None, 5), (c_scales(), 0)):
        assert f(c_rows(heads=4), c_batch(**change), scales, None, 0, window, 0, 1.0, _lib.F16, 4096, 1 << 40, None) == _lib.ENOTSUP
    for change in (dict(k_page=1 << 32), dict(v_block=-1)):
        assert f(c_rows(heads=4), c_batch(), c_scales(**change), None, 0, 0, 0, 1.0, _lib.F16, 4096, 1 << 40, None) == _lib.ENOTSUP


SEEN = r"""
#include <cstdio>
#include "paged_seen.h"
int main() {
  const int at[] = {0, 1, 2, 31, 32, 33, 63, 64, 500, 4096, 0x3fffffff, 0x7ffffbe0, 0x7fffffff}, sinks[] = {-0x7fffffff, -1, 0, 1, 31, 32, 33, 0x7fffffff};
  for (int keys : at)
    for (int first : at)
      for (int window : at)
        for (int s : sinks) {
          if (window == 0) continue;
          unsigned want = 0;
          for (long long i = 0; i < 32; ++i) {
            const long long key = (long long)first + i;
            if (key < keys && (key >= (long long)keys - window || i < s)) want |= 1u << i;
          }
          if (hexmi::seen_of_32(keys, first, window, s) != want) return printf("%d %d %d %d\n", keys, first, window, s), 1;
        }
  return 0;
}
"""


def test_which_keys_a_row_sees_is_worked_out_without_overflow(tmp_path):
    """The bits of 32 keys against their definition in 64 bits, with the checks of undefined behaviour on: rows of few keys beside blocks of far
    ones, windows as wide as any cache."""
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no C++ compiler for host code")
    source, program = tmp_path / "seen.cpp", tmp_path / "seen"
    source.write_text(SEEN)
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hexagon-mlir_amd", "csrc")
    subprocess.run([compiler, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", csrc, str(source), "-o", str(program)], check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout + run.stderr
