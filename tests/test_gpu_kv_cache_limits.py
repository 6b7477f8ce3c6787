"""Bounds of the 8-bit key/value cache: lengths, page ids, sizes and layouts that do not fit, on both attention paths (codes
read in place, and expanded for the packed kernel)."""
import math

import pytest
import torch

import transformerengine_b200 as te
from test_gpu_kv_cache import _cum, _filled, _i32
from transformerengine_b200.attention import kv_cache as kc

pytestmark = pytest.mark.gpu

both_paths = pytest.mark.parametrize("expand", [False, True], ids=["in_place", "expanded"])


def _path(monkeypatch, expand):
    monkeypatch.setattr(kc, "_expands", lambda *a: expand)


def _reported():
    """Whether a kernel reported lengths or pages that do not fit; clears the report."""
    try:
        te.check_status()
    except RuntimeError as e:
        assert "31" in str(e)
        return True
    return False


def _queries(rows, heads=8, d=128, seed=0, dtype=torch.bfloat16):
    return torch.randn(rows, heads, d, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _litter(like):
    """Leaves NaN in the memory that the next tensor of this size gets."""
    x = torch.full_like(like, math.nan)
    torch.cuda.synchronize()
    del x


# ------------------------------------------------------------------------------------------- lengths that do not fit
@both_paths
@pytest.mark.parametrize("cu,fits", [([0, 100], [0, 70]), ([0, 40, 100], [0, 40, 70]), ([0, 40, 200, 300], [0, 40, 70, 70])])
def test_queries_beyond_the_packed_rows_are_cut_and_reported(cu, fits, expand, monkeypatch):
    _path(monkeypatch, expand)
    lens = [300, 200, 250][:len(cu) - 1]
    cache, table = _filled(lens, 2, 64, 128, torch.Generator().manual_seed(1))
    q = _queries(70)
    kw = dict(max_q=160, max_kv=300)
    want = kc.attend(q, cache, table, _i32(fits), _i32(lens), **kw)
    assert not _reported()
    got = kc.attend(q, cache, table, _i32(cu), _i32(lens), **kw)
    assert _reported() and torch.equal(got, want)


@both_paths
@pytest.mark.parametrize("cu", [[-5, 20], [0, 50, 20], [90, 95], [0, -3, 30]])
def test_offsets_out_of_order_stay_within_the_output(cu, expand, monkeypatch):
    _path(monkeypatch, expand)
    lens = [300, 200][:len(cu) - 1]
    cache, table = _filled(lens, 2, 64, 128, torch.Generator().manual_seed(2))
    o = kc.attend(_queries(70), cache, table, _i32(cu), _i32(lens), max_q=70, max_kv=300)
    assert _reported() and o.shape == (70, 8, 128)


@both_paths
def test_sequences_longer_than_max_kv_are_cut_and_reported(expand, monkeypatch):
    _path(monkeypatch, expand)
    lens = [300, 90, 260]
    cache, table = _filled(lens, 2, 64, 128, torch.Generator().manual_seed(3))
    q, cu = _queries(130), _i32([0, 80, 90, 130])
    want = kc.attend(q, cache, table, cu, _i32([200, 90, 200]), max_q=80, max_kv=200)
    assert not _reported()
    got = kc.attend(q, cache, table, cu, _i32(lens), max_q=80, max_kv=200)
    assert _reported() and torch.equal(got, want)
    got = kc.attend(q, cache, table, cu, _i32([200, -90, 200]), max_q=80, max_kv=200)
    assert _reported() and (got[80:90] == 0).all() and torch.equal(got[:80], want[:80])


@both_paths
def test_queries_beyond_max_q_are_zero_and_reported(expand, monkeypatch):
    _path(monkeypatch, expand)
    lens = [300, 90, 260]
    cache, table = _filled(lens, 2, 64, 128, torch.Generator().manual_seed(4))
    q, cu = _queries(141), _cum([100, 10, 30])
    keep = list(range(64)) + list(range(100, 140))
    want = kc.attend(q[keep], cache, table, _i32(_cum([64, 10, 30])), _i32(lens), max_q=64, max_kv=300)
    assert not _reported()
    _litter(q)
    got = kc.attend(q, cache, table, _i32(cu), _i32(lens), max_q=64, max_kv=300)
    assert _reported() and torch.equal(got[keep], want)
    assert (got[64:100] == 0).all() and (got[140:] == 0).all()
