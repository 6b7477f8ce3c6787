"""Bounds of the 8-bit key/value cache: lengths, page ids, sizes and layouts that do not fit, on both attention paths (codes
read in place, and expanded for the packed kernel)."""
import math

import pytest
import torch

import transformerengine_b200 as te
from test_gpu_kv_cache import _check_attend, _cum, _filled, _i32, _oracle
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


# ------------------------------------------------------------------------------------------------- pages not held
@both_paths
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_pages_that_are_not_held_read_as_zeros_and_are_reported(bad, d, expand, monkeypatch):
    if expand and d != 128:
        pytest.skip("the expansion serves head dim 128")
    _path(monkeypatch, expand)
    lens, qs = [300, 200, 130], [70, 1, 5]
    cache, table = _filled(lens, 2, 64, d, torch.Generator().manual_seed(5))
    cache = kc.FP8KVCache(*(torch.cat([t.view(torch.uint8), torch.zeros_like(t.view(torch.uint8)[:1])]).view(t.dtype) for t in cache))
    cache.k_scale[-1], cache.v_scale[-1] = 1.0, 1.0
    zeros = table.clone()
    table[0, 1], table[1, 3], zeros[0, 1], zeros[1, 3] = bad, bad, len(cache.k) - 1, len(cache.k) - 1
    q, kw = _queries(sum(qs), d=d), dict(max_q=70, max_kv=300)
    want = kc.attend(q, cache, zeros, _i32(_cum(qs)), _i32(lens), **kw)
    assert not _reported()
    got = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), **kw)
    assert _reported() and torch.equal(got, want)
    # and on the CPU (fp32; the kernels round the probabilities to the type or to fp16, the result to the type)
    ref = kc.attend(q.cpu(), kc.FP8KVCache(*(t.cpu() for t in cache)), table.clamp(max=len(cache.k)).masked_fill(table == bad, -1).cpu(),
                    _i32(_cum(qs)).cpu(), _i32(lens).cpu(), **kw)
    assert ((got.cpu().float() - ref.float()).abs() <= 2 * 2.0 ** -8 * ref.abs().float() + 2 * 2.0 ** -8 * 6.0).all()
    # a table that ends before the sequence does
    got = kc.attend(q, cache, zeros[:, :3].contiguous(), _i32(_cum(qs)), _i32(lens), **kw)
    zeros[0, 3:] = len(cache.k) - 1
    assert _reported() and torch.equal(got[:70], kc.attend(q, cache, zeros, _i32(_cum(qs)), _i32(lens), **kw)[:70])


@both_paths
def test_pages_out_of_sight_are_not_reported(expand, monkeypatch):
    _path(monkeypatch, expand)
    lens, qs = [300, 200, 500], [20, 0, 33]
    cache, table = _filled(lens, 2, 32, 128, torch.Generator().manual_seed(6))
    q, kw = _queries(53), dict(max_q=33, max_kv=500, window=(40, 0), sink_tokens=20)
    want = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), **kw)
    table[1] = -1                                       # nobody asks
    table[0, 1:(300 - 20 - 40) // 32] = -1              # between the sinks and the first query's window
    table[2, 1:(500 - 33 - 40) // 32] = -1
    got = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), **kw)
    assert not _reported() and torch.equal(got, want)
    table[2, (500 - 33 - 40) // 32] = -1                # its last tokens are within the window
    kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), **kw)
    assert _reported()


# ----------------------------------------------------------------------------------------------- layouts and sizes
def test_a_cache_at_an_odd_address_is_refused():
    pool = torch.zeros(2 * 2 * 16 * 64 + 8, dtype=torch.uint8, device="cuda")
    odd = pool[8:].view(2, 2, 16, 64).view(torch.float8_e4m3fn)
    cache = kc.FP8KVCache.allocate(2, 2, 16, 64, device="cuda")
    x = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    one = (_i32([[0]]), _i32([0, 1]), _i32([1]))
    for bad in (cache._replace(k=odd), cache._replace(v=odd)):
        with pytest.raises(RuntimeError, match="16 bytes"):
            kc.append(bad, x, x, *one)
        with pytest.raises(RuntimeError, match="16 bytes"):
            kc.attend(x, bad, *one, max_q=1, max_kv=1)
        with pytest.raises(RuntimeError, match="16 bytes"):
            kc.gather(bad, one[0], one[2], _i32([0]), 1, torch.bfloat16)
        kc.copy_pages([bad], [0], [1])                 # copies take any address
    te.check_status()


@both_paths
@pytest.mark.parametrize("qs", [[1, 1, 1], [3, 0, 40]])
def test_max_q_may_be_any_bound(qs, expand, monkeypatch):
    _path(monkeypatch, expand)
    lens = [300, 0, 5000]
    cache, table = _filled(lens, 2, 64, 128, torch.Generator().manual_seed(7))
    q = _queries(sum(qs))
    want = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=sum(qs), max_kv=5000)
    for loose in (10 ** 6, 2 ** 31 - 1, 2 ** 40):
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        assert torch.equal(want, kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=loose, max_kv=5000))
        assert torch.cuda.max_memory_allocated() - held < 2 ** 27
    te.check_status()


def test_no_query_rows_with_a_large_max_q():
    cache, table = _filled([300] * 4, 8, 64, 128, torch.Generator().manual_seed(8))
    q = torch.zeros(0, 64, 128, device="cuda", dtype=torch.bfloat16)
    o = kc.attend(q, cache, table, _i32([0] * 5), _i32([300] * 4), max_q=500, max_kv=300)
    assert o.shape == (0, 64, 128)
    te.check_status()


# --------------------------------------------------------------------------------------- which path, and its memory
def _peak(call):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    out = call()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - held


def test_a_chunk_beside_decoding_sequences():
    """One prompt chunk among single tokens: read in place, as 63 of the sequences would be."""
    lens, qs = [900 + 13 * i for i in range(64)], [1] * 64
    qs[17] = 300
    cache, table = _filled(lens, 8, 64, 128, torch.Generator().manual_seed(9))
    q = _queries(sum(qs), heads=32)
    o, used = _peak(lambda: kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=300, max_kv=max(lens)))
    assert used < 2 ** 26                               # the expansion would take 0.5 GB
    each = [kc.attend(q[a:b], cache, table[i:i + 1], _i32([0, b - a]), _i32(lens[i:i + 1]), max_q=b - a, max_kv=lens[i])
            for i, (a, b) in enumerate(zip(_cum(qs), _cum(qs)[1:]))]
    # both round the probabilities (2^-11, or 2^-8 where the chunk alone is expanded) and the result once; |v| < 6
    err = (o.float() - torch.cat(each).float()).abs()
    assert (err <= 2.0 ** -7 * o.abs().float() + 2 * 2.0 ** -8 * 6.0).all()
    te.check_status()


@pytest.mark.parametrize("window", [-1, 500])
def test_a_loose_max_kv_takes_bounded_memory(window):
    lens, qs = [700, 300, 80], [300, 200, 80]
    cache, table = _filled(lens, 8, 64, 128, torch.Generator().manual_seed(10))
    q, kw = _queries(sum(qs), heads=32), dict(max_q=300, window=(window, 0), sink_tokens=4)
    want = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_kv=700, **kw)
    for loose in (10 ** 6, 4 * 10 ** 6, 2 ** 31 - 1):
        o, used = _peak(lambda: kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_kv=loose, **kw))
        assert used <= kc._EXPAND_BYTES + 2 ** 26
        # one path against the other: rounding of the probabilities to 8 and 11 bits, and of the result, |v| < 6
        assert ((o.float() - want.float()).abs() <= 2.0 ** -7 * want.abs().float() + 2 * 2.0 ** -8 * 6.0).all()
    te.check_status()


def test_sequences_expanded_in_groups_give_the_same(monkeypatch):
    _path(monkeypatch, True)
    lens, qs = [700, 300, 80, 1000, 64], [100, 0, 80, 130, 3]
    cache, table = _filled(lens, 2, 64, 128, torch.Generator().manual_seed(11))
    q = _queries(sum(qs) + 7)
    run = lambda: kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=130, max_kv=1000)  # noqa: E731
    want = run()
    for groups in (2, 3, 5):
        monkeypatch.setattr(kc, "_EXPAND_BYTES", kc._expansion_bytes(8, 2, 128, 130, 1000) * -(-5 // groups))
        _litter(q)
        assert torch.equal(run(), want)
    te.check_status()


@both_paths
@pytest.mark.parametrize("how", ["address", "stride"])
def test_queries_at_odd_addresses_and_strides(how, expand, monkeypatch):
    _path(monkeypatch, expand)
    lens, qs = [300, 200], [70, 5]
    cache, table = _filled(lens, 2, 64, 128, torch.Generator().manual_seed(12))
    q = _queries(sum(qs))
    if how == "address":
        odd = torch.zeros(q.numel() + 3, dtype=q.dtype, device="cuda")[3:].view(q.shape)
    else:
        odd = torch.zeros(sum(qs), 8, 132, dtype=q.dtype, device="cuda")[..., :128]
    odd.copy_(q)
    run = lambda x: kc.attend(x, cache, table, _i32(_cum(qs)), _i32(lens), max_q=70, max_kv=300)  # noqa: E731
    assert torch.equal(run(odd), run(q))
    te.check_status()


@pytest.mark.parametrize("packed", [False, True])
def test_training_attention_takes_tensors_at_odd_addresses(packed):
    """Forward and backward, as from tensors where the kernels can read them in place."""
    odd = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731
    lens = [200, 57]
    q, k, v, do = (_queries(sum(lens), h, seed=h + i) for i, h in enumerate((4, 2, 2, 4)))

    def run(change):
        x = [change(t).requires_grad_() for t in (q, k, v)]
        if packed:
            attn = te.DotProductAttention(4, 128, num_gqa_groups=2, qkv_format="thd", attn_mask_type="padding_causal", window_size=(60, 0),
                                          sink_tokens=5).cuda()
            o = attn(*x, cu_seqlens_q=_i32(_cum(lens)), cu_seqlens_kv=_i32(_cum(lens)))
            return (o, *torch.autograd.grad(o, x, change(do).view_as(o)))
        o = te.functional.attention(*(t.transpose(0, 1)[None] for t in x), causal=True, window=(60, 0), sink_tokens=5)
        return (o, *torch.autograd.grad(o, x, change(do).transpose(0, 1)[None]))

    for a, b in zip(run(odd), run(torch.clone)):
        assert torch.equal(a, b)
    te.check_status()


# ------------------------------------------------------------------------------------------------------- accuracy
@pytest.mark.parametrize("d,hq,n,qn", [(128, 8, 8000, 1), (64, 8, 3000, 4), (256, 4, 5000, 1), (128, 8, 600, 3)])
@pytest.mark.parametrize("share", [0.999, 0.9999])
def test_a_dominating_first_token_leaves_the_others_their_part(d, hq, n, qn, share):
    """Token 0 takes almost all of the probability and has no value: what the others add up to is the result."""
    g = torch.Generator().manual_seed(13)
    table = _i32([list(range(-(-n // 64)))])
    cache = kc.FP8KVCache.allocate(table.shape[1], 2, 64, d, device="cuda")
    x = torch.randn(2, n, 2, d, generator=g)
    x[0, :, :, 0], x[0, 0], x[1, 0] = 0.0, 0.0, 0.0
    x[0, 0, :, 0] = 16.0
    x = x.cuda()
    kc.append(cache, x[0], x[1], table, _i32([0, n]), _i32([n]))
    q = torch.randn(qn, hq, d, generator=g) * 0.5
    q[..., 0] = math.log(share / (1 - share) * n) * math.sqrt(d) / 16.0
    q = q.to(torch.bfloat16).cuda()
    o = kc.attend(q, cache, table, _i32([0, qn]), _i32([n]), max_q=qn, max_kv=n).double()
    dec = [c.float().double() * s.double().repeat_interleave(16, dim=2)[..., None] for c, s in
           ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    k, v = (t[table[0].long()].transpose(0, 1).reshape(2, -1, d)[:, :n] for t in dec)
    for a in range(hq):
        s = q[:, a].double() @ k[a // (hq // 2)].T / math.sqrt(d)
        pos = n - qn + torch.arange(qn, device="cuda")[:, None]
        p = torch.softmax(s.masked_fill(torch.arange(n, device="cuda")[None] > pos, -math.inf), -1)
        assert (p[:, 0] > share - 0.05).all()
        want, mass = p @ v[a // (hq // 2)], p @ v[a // (hq // 2)].abs()
        # the result and the probabilities (fp16) are rounded once; as much again as the latter for fp32 scores and sums;
        # probabilities below 2^-29 of the largest lose up to 2^-40 of it
        tol = 2.0 ** -8 * want.abs() + 2 * 2.0 ** -11 * mass + n * 2.0 ** -40 * 6.0
        err = (o[:, a] - want).abs()
        assert (err <= tol).all(), (err / tol).max()
    te.check_status()


@pytest.mark.parametrize("max_kv", [None, 1, 2 ** 40])
def test_gather_of_many_sequences_with_any_bound(max_kv):
    """One long sequence among short ones: fewer CTAs than blocks, whatever bound sizes the launch."""
    lens = [20000] + [17 + i % 50 for i in range(300)]
    cache, table = _filled(lens, 8, 64, 64, torch.Generator().manual_seed(14))
    rows = sum(lens)
    k, v = kc.gather(cache, table, _i32(lens), _i32(_cum(lens)[:-1]), rows, torch.float32, max_kv=max_kv)
    for i in (0, 1, 150, 300):
        at = _cum(lens)[i]
        pages = table[i][:-(-lens[i] // 64)].long()
        for got, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
            x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()
            x = (x * scales[pages].repeat_interleave(16, dim=2)[..., None]).transpose(1, 2).reshape(-1, 8, 64)[:lens[i]]
            assert torch.equal(got[at:at + lens[i]], x)                  # codes times powers of two: exact
    te.check_status()


# -------------------------------------------------------------------------------------------------- prompt chunks
@pytest.mark.parametrize("d,hq,hk", [(64, 8, 2), (256, 4, 1), (128, 8, 2)])
@pytest.mark.parametrize("qs,lens,window,sinks", [([700, 1, 129, 0, 1], [1500, 3000, 129, 64, 20], -1, 0),
                                                  ([513, 2, 1, 300], [600, 2500, 7, 1000], 200, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_chunks_beside_single_tokens_match_64_bits(d, hq, hk, qs, lens, window, sinks, dtype):
    cache, table = _filled(lens, hk, 64, d, torch.Generator().manual_seed(d + len(qs)))
    q = _queries(sum(qs) + 3, hq, d, dtype=dtype)
    o = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=max(qs), max_kv=max(lens), window=(window, 0), sink_tokens=sinks)
    te.check_status()
    want, mass = _oracle(q, cache, table, qs, lens, window, sinks)
    expanded = kc._expands(len(qs), hq, hk, d, max(qs), len(q), max(lens)) and d == 128
    _check_attend(o, want, mass, lens, 6.0, torch.finfo(dtype).eps / 2 if expanded else 2.0 ** -11)
    assert (o[sum(qs):] == 0).all()
