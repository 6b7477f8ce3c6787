"""The 8-bit paged key/value cache and attention with visible first tokens on the GPU, against plain forms in 64 bits."""
import math

import pytest
import torch

import transformerengine_b200 as te
from transformerengine_b200.attention import kv_cache as kc

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cum(x):
    out = [0]
    for n in x:
        out.append(out[-1] + n)
    return out


def _to_cpu(cache):
    return kc.FP8KVCache(*(t.cpu() for t in cache))


def _same(a, b):
    return all(torch.equal(x.cpu().view(torch.uint8), y.cpu().view(torch.uint8)) for x, y in zip(a, b))


def _table(lens, ps, g, spare=2):
    """Pages dealt out in random order; unused entries -1."""
    need = [-(-n // ps) for n in lens]
    ids = torch.randperm(sum(need) + spare, generator=g).tolist()
    t = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        t[i, :n] = torch.tensor(ids[:n], dtype=torch.int32)
        ids = ids[n:]
    return t.cuda(), sum(need) + spare


def _filled(lens, h, ps, d, g, dtype=torch.bfloat16, strong=1.0):
    """A cache filled by append; slots that hold nothing are NaN codes."""
    table, pages = _table(lens, ps, g)
    cache = kc.FP8KVCache.allocate(pages, h, ps, d, device="cuda")
    cache.k.view(torch.uint8).fill_(0x7f)
    cache.v.view(torch.uint8).fill_(0x7f)
    t = sum(lens)
    x = torch.randn(2, t, h, d, generator=g)
    x[0, :, :, ::5] *= strong
    x = x.to(dtype).cuda()
    kc.append(cache, x[0], x[1], table, _i32(_cum(lens)), _i32(lens))
    return cache, table


def _decode(cache, row, n):
    """Keys and values [h, n, d] of one sequence in 64 bits."""
    pages = [p for p in row.tolist() if p >= 0]
    out = []
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = c.float().double() * s.double().repeat_interleave(16, dim=2)[..., None]
        out.append(torch.cat([x[p] for p in pages], dim=1)[:, :n] if pages else x[0][:, :0])
    return out


def _oracle(q, cache, table, qs, lens, window, sinks, causal=True):
    """(output, sum of probability * |value|) in 64 bits."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(out)
    cu = _cum(qs)
    for i, (m, n) in enumerate(zip(qs, lens)):
        if m == 0 or n == 0:
            continue
        k, v = _decode(cache, table[i], n)
        g = q.shape[1] // k.shape[0]
        p = n - m + torch.arange(m, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        seen = (j <= p) if causal else torch.ones(m, n, dtype=torch.bool, device="cuda")
        if window >= 0:
            seen = seen & ((p - j <= window) | (j < sinks))
        for a in range(q.shape[1]):
            s = q[cu[i]:cu[i + 1], a].double() @ k[a // g].T / math.sqrt(q.shape[2])
            w = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -math.inf), -1))
            out[cu[i]:cu[i + 1], a] = w @ v[a // g]
            mass[cu[i]:cu[i + 1], a] = w @ v[a // g].abs()
    return out, mass


def _check_attend(o, want, mass, lens, vmax, half_step_of_p):
    # rounding of the output (half a step of its type), of the probabilities (half a step of the type they are multiplied
    # in, on every term; fp16 codes below 2^-14 of the largest: 2^-25 each), and as much again as the latter for the fp32
    # scores (|score| below 2^5: 2^-19 relative in p, sums of up to 2^12 terms)
    tol = torch.finfo(o.dtype).eps / 2 * want.abs() + 2 * half_step_of_p * mass + max(lens) * 2.0 ** -25 * vmax + 1e-30
    err = (o.double() - want).abs()
    assert torch.isfinite(o).all()
    assert (err <= tol).all(), (err / tol).max()


# ------------------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,h,ps", [(128, 8, 64), (64, 3, 16), (256, 1, 48), (128, 2, 32)])
def test_append_matches_the_reference_bit_for_bit(dtype, d, h, ps):
    g = torch.Generator().manual_seed(d + h)
    total = [70, 1, 16, 33, 200]
    table, pages = _table(total, ps, g)
    gpu = kc.FP8KVCache.allocate(pages, h, ps, d, device="cuda")
    gpu.k.view(torch.uint8).fill_(0x55)
    cpu = _to_cpu(gpu)
    lens = [0] * 5
    for step in ([3, 1, 16, 0, 17], [1, 0, 0, 15, 1], [30, 0, 0, 17, 100], [36, 0, 0, 1, 82]):
        lens = [a + b for a, b in zip(lens, step)]
        t = sum(step)
        wide = (torch.randn(t, 2 * h + 1, d, generator=g) * 10.0 ** torch.randn(t, 1, 1, generator=g)).to(dtype)
        wide[0, 0, 3], wide[0, 1, 5], wide[0, -1, 7] = math.nan, math.inf, -math.inf
        k, v = wide[:, :h], wide[:, h:2 * h]                               # strided views of one projection
        kc.append(cpu, k, v, table.cpu(), _i32(_cum(step)).cpu(), _i32(lens).cpu())
        wg = wide.cuda()
        kc.append(gpu, wg[:, :h], wg[:, h:2 * h], table, _i32(_cum(step)), _i32(lens), max_new=min(step))   # a low hint only sizes the grid
        assert _same(gpu, cpu)
    te.check_status()


def test_append_takes_rows_at_odd_addresses():
    g = torch.Generator().manual_seed(0)
    table = _i32([[0, 1]])
    flat = torch.randn(20 * 2 * 64 + 3, generator=g).to(torch.bfloat16).cuda()
    odd = flat[3:].view(20, 2, 64)                                      # 6 bytes off
    a, b = (kc.FP8KVCache.allocate(2, 2, 16, 64, device="cuda") for _ in range(2))
    kc.append(a, odd, odd, table, _i32([0, 20]), _i32([20]))
    kc.append(b, odd.clone(), odd.clone(), table, _i32([0, 20]), _i32([20]))
    assert _same(a, b)
    te.check_status()


# ------------------------------------------------------------------------------------------------------------ attend
CASES = [
    # d, hq, hk, page, q lengths, kv lengths, window, sinks, dtype
    (128, 32, 8, 64, [1] * 6, [200, 1, 16, 17, 0, 33], -1, 0, torch.bfloat16),
    (128, 4, 4, 16, [1] * 3, [5000, 31, 2049], -1, 0, torch.float16),                 # one head per group, several CTAs per sequence
    (128, 16, 1, 32, [1, 1], [700, 3], -1, 0, torch.bfloat16),                        # sixteen rows
    (128, 40, 2, 64, [1, 1], [129, 1000], 100, 4, torch.bfloat16),                    # twenty rows: two tiles
    (128, 8, 2, 48, [3, 0, 5, 4], [600, 10, 4, 1111], -1, 0, torch.bfloat16),         # drafted tokens; more queries than tokens
    (128, 8, 8, 64, [1, 2, 1], [4096, 4097, 40], 1023, 4, torch.bfloat16),            # window and sinks
    (128, 8, 8, 64, [1, 2, 1], [4096, 4097, 40], 0, 0, torch.float16),                # window of the token itself
    (128, 8, 4, 64, [2, 2], [300, 900], 200, 150, torch.bfloat16),                    # sinks reach the window
    (128, 8, 4, 64, [2, 2], [300, 900], 50, 100000, torch.bfloat16),                  # everything is a sink
    (64, 16, 4, 32, [4, 1, 2], [3000, 64, 65], 2047, 4, torch.float16),
    (64, 8, 8, 16, [1, 1], [15, 4097], -1, 0, torch.bfloat16),
    (256, 8, 1, 64, [1, 1, 1], [100, 3000, 1], -1, 0, torch.bfloat16),
    (256, 8, 4, 16, [2, 5], [513, 777], 77, 3, torch.float16),
    (256, 8, 2, 64, [20, 9], [2000, 300], -1, 0, torch.bfloat16),                     # sixteen rows of a wide head at a time
    (256, 4, 1, 16, [50, 1, 33], [50, 700, 900], 60, 2, torch.float16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:4]) + f"-w{c[6]}-s{c[7]}")
def test_attend_matches_64_bits(case):
    d, hq, hk, ps, qs, lens, window, sinks, dtype = case
    g = torch.Generator().manual_seed(sum(lens))
    cache, table = _filled(lens, hk, ps, d, g, strong=3.0)
    wide = torch.randn(sum(qs) + 3, hq + 2, d, generator=g).to(dtype).cuda()
    q = wide[:, :hq]                                                     # strided rows, three of them behind the last sequence
    o = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=max(qs), max_kv=max(lens), window=(window, 0), sink_tokens=sinks)
    te.check_status()
    want, mass = _oracle(q, cache, table, qs, lens, window, sinks)
    assert o.shape == q.shape and o.is_contiguous()
    _check_attend(o, want, mass, lens, 6.0, 2.0 ** -11)
    assert (o[sum(qs):] == 0).all()
    for i, (m, n) in enumerate(zip(qs, lens)):                            # rows that see nothing
        lost = max(0, m - n)
        assert (o[_cum(qs)[i]:_cum(qs)[i] + lost] == 0).all()


@pytest.mark.parametrize("qs,lens,window,sinks", [([100, 300, 1], [700, 300, 129], -1, 0), ([257, 40], [2000, 41], 128, 5),
                                                  ([65, 0, 70], [65, 9, 69], 10, 2), ([130, 20], [1000, 900], 700, 300)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("expand", [True, False])
def test_attend_of_prompt_chunks(qs, lens, window, sinks, dtype, expand, monkeypatch):
    monkeypatch.setattr(kc, "_expands", lambda *a: expand)
    g = torch.Generator().manual_seed(7)
    cache, table = _filled(lens, 2, 64, 128, g)
    q = torch.randn(sum(qs) + 1, 8, 128, generator=g).to(dtype).cuda()
    o = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=max(qs), max_kv=max(lens), window=(window, 0), sink_tokens=sinks)
    te.check_status()
    want, mass = _oracle(q, cache, table, qs, lens, window, sinks)
    # the packed kernels round the probabilities to the inputs' type
    _check_attend(o, want, mass, lens, 6.0, torch.finfo(dtype).eps / 2 if expand else 2.0 ** -11)
    assert (o[sum(qs):] == 0).all()


def test_attend_takes_any_window_and_scale(monkeypatch):
    """Windows and sinks beyond every length, more queries than tokens, a negative scale."""
    g = torch.Generator().manual_seed(18)
    qs, lens = [7, 3], [4, 300]
    cache, table = _filled(lens, 2, 64, 128, g)
    q = torch.randn(10, 4, 128, generator=g).to(torch.bfloat16).cuda()
    kw = dict(max_q=7, max_kv=300)
    o = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), window=(2 ** 31 - 1, 0), sink_tokens=2 ** 31 - 1, **kw)
    assert torch.equal(o, kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), **kw))
    q = torch.randn(100, 4, 128, generator=g).to(torch.bfloat16).cuda()
    monkeypatch.setattr(kc, "_expands", lambda *a: True)                     # not taken: they need a positive scale
    o = kc.attend(q, cache, table, _i32([0, 0, 100]), _i32(lens), max_q=100, max_kv=300, scale=-128 ** -0.5)
    want, mass = _oracle(-q, cache, table, [0, 100], lens, -1, 0)
    _check_attend(o, want, mass, lens, 6.0, 2.0 ** -11)
    te.check_status()


def test_attend_without_causal_mask():
    g = torch.Generator().manual_seed(8)
    qs, lens = [3, 2], [70, 500]
    cache, table = _filled(lens, 2, 64, 128, g)
    q = torch.randn(5, 8, 128, generator=g).to(torch.bfloat16).cuda()
    o = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=3, max_kv=500, causal=False)
    want, mass = _oracle(q, cache, table, qs, lens, -1, 0, causal=False)
    _check_attend(o, want, mass, lens, 6.0, 2.0 ** -11)


@pytest.mark.parametrize("spread", [1.0, 40.0])
def test_attend_with_scales_far_apart(spread):
    """Blocks whose values differ by many powers of two, a block of zeros, and large queries."""
    g = torch.Generator().manual_seed(9)
    lens = [400]
    table, pages = _table(lens, 64, g)
    cache = kc.FP8KVCache.allocate(pages, 2, 64, 128, device="cuda")
    x = torch.randn(2, 400, 2, 128, generator=g)
    size = torch.exp2(torch.round(spread * torch.rand(25, generator=g))).repeat_interleave(16)
    x[1] *= size[:, None, None]
    x[1, 32:64] = 0
    x = x.cuda()
    kc.append(cache, x[0], x[1], table, _i32([0, 400]), _i32(lens))
    q = (torch.randn(1, 8, 128, generator=g) * 2.0 ** 20).to(torch.bfloat16).cuda()
    for scale in (2.0 ** -20 / 11, 2.0 ** -16 / 11):
        o = kc.attend(q, cache, table, _i32([0, 1]), _i32(lens), max_q=1, max_kv=400, scale=scale)
        k, v = _decode(cache, table[0], 400)
        for a in range(8):
            s = q[0, a].double() @ k[a // 4].T * scale
            p = torch.softmax(s, -1)
            want, mass = p @ v[a // 4], p @ v[a // 4].abs()
            # as above; probability * scale is largest for one block and the codes below 2^-14 of it lose up to 2^-25
            floor = 400 * 2.0 ** -25 * (p * v[a // 4].abs().amax(-1)).max() * 2 ** 5
            err = (o[0, a].double() - want).abs()
            assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -9 * mass + floor).all()
    te.check_status()


def test_nan_reaches_only_who_sees_it():
    g = torch.Generator().manual_seed(10)
    lens, qs = [300, 300], [1, 1]
    cache, table = _filled(lens, 2, 64, 128, g)
    cache.v.view(torch.uint8)[int(table[0, 1]), 0, 3] = 0x7f               # token 67 of sequence 0, head 0
    q = torch.randn(2, 8, 128, generator=g).to(torch.bfloat16).cuda()
    run = lambda w: kc.attend(q, cache, table, _i32([0, 1, 2]), _i32(lens), max_q=1, max_kv=300, window=(w, 0), sink_tokens=2)  # noqa: E731
    o = run(-1)
    assert torch.isnan(o[0, :4]).all() and torch.isfinite(o[0, 4:]).all() and torch.isfinite(o[1]).all()
    assert torch.isfinite(run(230)).all()                                   # keys 69 .. 299 and the two sinks
    assert torch.isnan(run(232)[0, :4]).all()
    te.check_status()


def test_attend_replays_in_a_graph_and_on_another_stream():
    g = torch.Generator().manual_seed(11)
    lens = [100, 3000, 64]
    cache, table = _filled([n + 4 for n in lens], 8, 64, 128, g)
    q = torch.randn(3, 32, 128, generator=g).to(torch.bfloat16).cuda()
    new = torch.randn(2, 3, 8, 128, generator=g).to(torch.bfloat16).cuda()
    kv_lens, cu = _i32(lens), _i32([0, 1, 2, 3])

    def step():
        kc.append(cache, new[0], new[1], table, cu, kv_lens, max_new=1)
        return kc.attend(q, cache, table, cu, kv_lens, max_q=1, max_kv=3100)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        kv_lens += 1
        graph.replay()
        got, held = out.clone(), [t.clone() for t in cache]
        want = step()
        assert torch.equal(got, want) and _same(held, cache)
    te.check_status()


@pytest.mark.parametrize("n,qn,hq,hk,longest", [(200, 1, 4, 1, 4000), (300, 3, 16, 2, 2500), (3, 40, 8, 1, 9000), (2, 1, 8, 8, 20000)])
def test_attend_shares_ragged_sequences_over_the_ctas(n, qn, hq, hk, longest):
    """More sequences than threads, several tiles of rows, sequences cut at any place, among them empty and tiny ones."""
    g = torch.Generator().manual_seed(n)
    lens = [int(longest ** x) for x in torch.rand(n, generator=g).tolist()]
    lens[0], lens[-1], lens[n // 2] = longest, 0, 1
    qs = [int(x) for x in torch.randint(0, qn + 1, (n,), generator=g)]
    qs[0] = qn
    cache, table = _filled(lens, hk, 16, 64, g)
    q = torch.randn(sum(qs) + 5, hq, 64, generator=g).to(torch.float16).cuda()
    o = kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=qn, max_kv=longest)
    te.check_status()
    want, mass = _oracle(q, cache, table, qs, lens, -1, 0)
    _check_attend(o, want, mass, lens, 6.0, 2.0 ** -11)
    assert torch.equal(o, kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=qn, max_kv=longest))   # no order changes it
    assert (o[sum(qs):] == 0).all()


def test_calls_on_two_streams_do_not_meet():
    g = torch.Generator().manual_seed(19)
    a, ta = _filled([9000, 500], 4, 64, 128, g)
    b, tb = _filled([7000, 8000], 4, 64, 128, g)
    q = torch.randn(2, 16, 128, generator=g).to(torch.bfloat16).cuda()
    run = lambda c, t, lens: kc.attend(q, c, t, _i32([0, 1, 2]), _i32(lens), max_q=1, max_kv=9000)  # noqa: E731
    want = run(a, ta, [9000, 500]), run(b, tb, [7000, 8000])
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(one):
            x = run(a, ta, [9000, 500])
        with torch.cuda.stream(two):
            y = run(b, tb, [7000, 8000])
        got.append((x, y))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[0]) and torch.equal(y, want[1]) for x, y in got)
    te.check_status()


def test_offsets_beyond_32_bits():
    """The last pages of a cache of 5 GB of codes: append, attend, gather and copies reach them."""
    g = torch.Generator().manual_seed(20)
    big = kc.FP8KVCache.allocate(40000, 8, 128, 128, device="cuda")
    small = kc.FP8KVCache.allocate(8, 8, 128, 128, device="cuda")
    x = torch.randn(2, 300, 8, 128, generator=g).to(torch.bfloat16).cuda()
    q = torch.randn(70, 32, 128, generator=g).to(torch.bfloat16).cuda()
    outs = []
    for cache, first in ((big, 39996), (small, 4)):
        table = _i32([[first + 3, first + 1, first + 2]])
        kc.append(cache, x[0], x[1], table, _i32([0, 300]), _i32([300]))
        kc.copy_pages([cache], [first + 1], [first])
        table[0, 1] = first
        for rows in (1, 70):
            outs.append(kc.attend(q[:rows], cache, table, _i32([0, rows]), _i32([300]), max_q=rows, max_kv=300))
        outs += kc.gather(cache, table, _i32([300]), _i32([0]), 300, torch.float32)
    half = len(outs) // 2
    assert all(torch.equal(a, b) for a, b in zip(outs[:half], outs[half:]))
    assert big.k_scale[:39996].abs().sum() == 0
    te.check_status()


def test_bad_pages_and_lengths_are_reported():
    g = torch.Generator().manual_seed(12)
    cache, table = _filled([100], 2, 64, 128, g)
    q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16).cuda()
    before = [t.clone() for t in cache]
    x = torch.zeros(1, 2, 128, device="cuda")
    for bad in (_i32([[0, 99]]), _i32([[0, -1]])):
        kc.attend(q, cache, bad, _i32([0, 1]), _i32([100]), max_q=1, max_kv=100)
        with pytest.raises(RuntimeError, match="31"):
            te.check_status()
        kc.append(cache, x, x, bad, _i32([0, 1]), _i32([100]))
        with pytest.raises(RuntimeError, match="31"):
            te.check_status()
    kc.attend(q, cache, table, _i32([0, 1]), _i32([1000]), max_q=1, max_kv=2000)        # beyond the table
    with pytest.raises(RuntimeError, match="31"):
        te.check_status()
    kc.append(cache, x, x, table, _i32([0, 1]), _i32([0]))                              # fewer tokens than new ones
    with pytest.raises(RuntimeError, match="31"):
        te.check_status()
    kc.attend(q, cache, _i32([[-1, int(table[0, 1])]]), _i32([0, 1]), _i32([100]), max_q=1, max_kv=100, window=(30, 0))   # not needed
    te.check_status()
    assert _same(cache, before)


def test_refusals_on_the_gpu():
    cache = kc.FP8KVCache.allocate(2, 2, 16, 64, device="cuda")
    one = (_i32([[0]]), _i32([0, 1]), _i32([1]))
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    kw = dict(max_q=1, max_kv=1)
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        kc.attend(q.float(), cache, *one, **kw)
    with pytest.raises(RuntimeError, match="multiple of the cache"):
        kc.attend(q[:, :3], cache, *one, **kw)
    with pytest.raises(RuntimeError, match="kv_lens"):
        kc.attend(q, cache, one[0], one[1], one[2].long(), **kw)
    with pytest.raises(RuntimeError, match="page_table"):
        kc.attend(q, cache, one[0].cpu(), *one[1:], **kw)
    with pytest.raises(RuntimeError, match="one type"):
        kc.append(cache, q[:, :2], q[:, :2].float(), *one)
    with pytest.raises(RuntimeError, match="must be"):
        kc.append(cache, q, q, *one)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        kc.append(cache._replace(k=cache.k.view(torch.uint8)), q[:, :2], q[:, :2], *one)
    t = torch.zeros(3, 5, device="cuda")
    for src, dst in (([0, 1], [2, 2]), ([0], [3]), ([-1], [0]), ([0, 1], [1, 2])):
        with pytest.raises(ValueError, match="copy_pages"):
            kc.copy_pages([t], src, dst)
    with pytest.raises(RuntimeError, match="contiguous"):
        kc.copy_pages([t.t()], [0], [1])
    assert kc.attend(q[:0], cache, _i32([[0]]), _i32([0, 0]), _i32([1]), max_q=0, max_kv=1).shape == (0, 4, 64)


# ------------------------------------------------------------------------------------------------------ gather, copies
@pytest.mark.parametrize("d,dtype", [(64, torch.float32), (128, torch.bfloat16), (256, torch.float16)])
def test_gather_matches_the_reference(d, dtype):
    g = torch.Generator().manual_seed(13)
    lens = [130, 1, 0, 77]
    cache, table = _filled(lens, 3, 32, d, g, dtype=torch.float32, strong=1e4)
    k, v = kc.gather(cache, table, _i32(lens), _i32([0, 130, 140, 140]), 217, dtype)
    kr, vr = kc.gather(_to_cpu(cache), table.cpu(), _i32(lens).cpu(), _i32([0, 130, 140, 140]).cpu(), 217, dtype)
    for a, b in ((k, kr), (v, vr)):
        for s, n in ((0, 131), (140, 77)):
            assert torch.equal(a[s:s + n].cpu(), b[s:s + n])
    te.check_status()


@pytest.mark.parametrize("pairs", [1, 70, 1500])
def test_copy_pages_moves_every_tensor(pairs):
    g = torch.Generator().manual_seed(14)
    pages = 2 * pairs + 5
    perm = torch.randperm(pages, generator=g).tolist()
    src, dst = perm[:pairs], perm[pairs:2 * pairs]
    odd = torch.randint(0, 255, (pages * 7 + 1,), generator=g, dtype=torch.uint8).cuda()
    tensors = [torch.randn(pages, 2, 33, generator=g).cuda(), odd[1:].view(pages, 7), torch.randn(pages, 64, generator=g).to(torch.bfloat16).cuda(),
               torch.randn(pages, 3, generator=g).cuda()] * 1
    tensors += [torch.randn(pages, 1, generator=g).cuda() for _ in range(130)]       # more than one launch's table
    cache = kc.FP8KVCache.allocate(pages, 2, 16, 64, device="cuda")
    cache.k.view(torch.uint8).random_(0, 255)
    cache.v_scale.normal_()
    want = [t.clone() for t in tensors + list(cache)]
    for w in want:
        w.view(torch.uint8)[torch.tensor(dst)] = w.view(torch.uint8)[torch.tensor(src)].clone()
    kc.copy_pages(tensors + [cache], src, dst)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(tensors + list(cache), want))


# --------------------------------------------------------------------------------- window with visible first tokens
def _formula(q, k, v, do, window, sinks, causal, off):
    """Output and gradients in 64 bits, and for each the sum of the magnitudes of the terms it adds up."""
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    b, hq, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    g = hq // hk
    i, j = torch.arange(sq, device=q.device)[:, None] + off, torch.arange(sk, device=q.device)[None]
    seen = (j >= i - window[0]) | (j < sinks)
    right = 0 if causal else window[1]
    if right >= 0:
        seen = seen & (j <= i + right)
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = (q @ kk.transpose(-1, -2)) * d ** -0.5
    p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -math.inf), -1))
    o = p @ vv
    dp = do @ vv.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * d ** -0.5
    big = p * (dp.abs() + delta.abs() + (do.abs() * o.abs()).sum(-1, keepdim=True)) * d ** -0.5
    fold = lambda t: t.reshape(b, hk, g, sk, d).sum(2)  # noqa: E731
    t = lambda x: x.transpose(-1, -2)  # noqa: E731
    return ((o, p @ vv.abs()), (ds @ kk, big @ kk.abs()), (fold(t(ds) @ q), fold(t(big) @ q.abs())),
            (fold(t(p) @ do), fold(t(p) @ do.abs())))


SINKS = [
    # b, hq, hk, sq, sk, window, sinks, causal, bottom_right
    (1, 4, 2, 333, 333, (64, 0), 4, True, True),
    (2, 2, 2, 1, 700, (100, 0), 3, True, True),
    (1, 2, 1, 700, 700, (0, 0), 1, True, True),
    (1, 4, 4, 1000, 1000, (129, 0), 130, True, True),         # sinks over two key blocks
    (1, 2, 2, 600, 600, (300, 0), 250, True, True),           # sinks reach the first windows
    (1, 2, 2, 300, 300, (20, 0), 1000, True, True),           # all keys are sinks
    (1, 2, 1, 700, 300, (50, 0), 6, True, False),             # late queries see the sinks alone
    (1, 2, 2, 300, 900, (40, 0), 5, True, True),
    (1, 2, 2, 500, 500, (30, 40), 7, False, True),
    (1, 2, 2, 300, 100, (30, 0), 7, True, True),              # early queries see nothing
]


@pytest.mark.parametrize("case", SINKS, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_window_with_sinks_forward_and_backward(case, dtype):
    b, hq, hk, sq, sk, window, sinks, causal, br = case
    g = torch.Generator().manual_seed(sq + sk)
    mk = lambda h, s: torch.randn(b, s, h, 128, generator=g).to(dtype).cuda().permute(0, 2, 1, 3)  # noqa: E731
    q, k, v, do = mk(hq, sq).requires_grad_(), mk(hk, sk).requires_grad_(), mk(hk, sk).requires_grad_(), mk(hq, sq)
    o = te.functional.attention(q, k, v, causal=causal, window=window, bottom_right=br, sink_tokens=sinks, out_format="bshd")
    grads = torch.autograd.grad(o, (q, k, v), do)
    te.check_status()
    half = torch.finfo(dtype).eps / 2
    want = _formula(q, k, v, do, window, sinks, causal, sk - sq if br else 0)
    # the result, the probabilities (or dS) and, inside dS, the output that delta is made of are each rounded once to the
    # type; group sums of key gradients once more
    for a, (x, mass) in zip((o, *grads), want):
        assert torch.isfinite(a).all()
        err = (a.double() - x).abs()
        tol = 2 * half * x.abs() + 3 * half * mass + 1e-6
        assert (err <= tol).all(), (err / tol).max()


def test_packed_sequences_with_sinks():
    g = torch.Generator().manual_seed(15)
    lens = [200, 1, 517]
    q, k, v = (torch.randn(sum(lens), h, 128, generator=g).to(torch.bfloat16).cuda().requires_grad_() for h in (4, 2, 2))
    do = torch.randn(sum(lens), 4 * 128, generator=g).to(torch.bfloat16).cuda()
    attn = te.DotProductAttention(4, 128, num_gqa_groups=2, qkv_format="thd", attn_mask_type="padding_causal", window_size=(60, 0),
                                  sink_tokens=5).cuda()
    o = attn(q, k, v, cu_seqlens_q=_i32(_cum(lens)), cu_seqlens_kv=_i32(_cum(lens)))
    grads = torch.autograd.grad(o, (q, k, v), do)
    at = 0
    for n in lens:
        cut = lambda t: t[at:at + n].view(n, -1, 128).transpose(0, 1)[None]  # noqa: E731
        want = _formula(cut(q), cut(k), cut(v), cut(do), (60, 0), 5, True, 0)
        for a, (x, mass) in zip((o, *grads), want):
            err = (cut(a.detach()).double() - x).abs()
            assert (err <= 2.0 ** -7 * x.abs() + 3 * 2.0 ** -8 * mass + 1e-6).all()
        at += n
    te.check_status()


def test_zero_sinks_are_the_plain_window():
    g = torch.Generator().manual_seed(16)
    q, k, v = (torch.randn(1, 2, 400, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(3))
    a = te.functional.attention(q, k, v, causal=True, window=(70, 0))
    assert torch.equal(a, te.functional.attention(q, k, v, causal=True, window=(70, 0), sink_tokens=0))
    b = te.functional.attention(q, k, v, causal=True)
    assert torch.equal(b, te.functional.attention(q, k, v, causal=True, sink_tokens=9))      # no window: nothing to see past


# ------------------------------------------------------------------------------------------------ as a model uses them
from collections import OrderedDict  # noqa: E402


@pytest.mark.parametrize("head_dim", [64, 128])
def test_model_on_the_8_bit_cache_with_forks_drafts_and_compaction(head_dim):
    """Prompt, forks, single tokens, drafts cut back, compaction, pages out of the window reused: the logits stay by the
    full pass's, and by those of the CPU path on the same codes' rounding."""
    from transformerengine_b200.models.mistral import MistralConfig, MistralModel
    torch.manual_seed(3)
    cfg = MistralConfig.tiny(hidden_size=512, num_heads=512 // head_dim, num_kv_heads=2, head_dim=head_dim, sliding_window=100, sink_tokens=5)
    model = MistralModel(cfg).cuda().eval()
    tokens = torch.randint(0, cfg.vocab_size, (2, 320), device="cuda")
    with torch.no_grad():
        full = model(tokens).transpose(0, 1).float()
        params = model.make_inference_params(4, 400, is_paged=True, page_size=32, total_num_pages=64, cache_dtype=torch.float8_e4m3fn)
        m = params.cache_manager
        at = 300
        params.pre_step(OrderedDict([(0, at), (1, at)]))
        got = [model(tokens[:, :at], inference_params=params).transpose(0, 1).float()]
        rows = []
        for n, junk in ((1, 0), (1, 0), (2, 3), (1, 0), (5, 2)):
            params.fork_sequence(1, 9 + at)                                # a fork that is gone with the next step
            params.pre_step(OrderedDict([(0, n + junk), (1, n + junk), (9 + at, 1)]))
            pad = torch.zeros(1, n + junk, dtype=torch.long, device="cuda")
            step = torch.cat([tokens[:, at:at + n], torch.randint(0, cfg.vocab_size, (2, junk), device="cuda")], 1)
            y = model(torch.cat([step, pad]), inference_params=params).transpose(0, 1).float()
            rows.append(y[:2, :n])
            at += n
            for i in (0, 1):
                params.truncate_sequence(i, at)
            if n == 2:
                params.compact()
        got = torch.cat(got + rows, 1)
    te.check_status()
    assert m.page_table[0][0] >= 0 and m.page_table[0][2] == -1
    for i in (0, 1):
        # keys and values off by up to 2^-4 each, in two layers
        assert (got[i] - full[i, :at]).norm() / full[i, :at].norm() < 2.0 ** -3
    out = model.generate(tokens[:, :50], 30, is_paged=True, page_size=32, total_num_pages=16, cache_dtype=torch.float8_e4m3fn)
    assert out.shape == (2, 80)
    te.check_status()


def test_16_bit_pages_fork_and_copy_on_the_gpu():
    m = te.PagedKVCacheManager(8, 16, 2, 64, torch.bfloat16, 4, 128, device="cuda")
    x = torch.randn(22, 2, 64, device="cuda", dtype=torch.bfloat16)
    m.pre_step(OrderedDict([(0, 20)]))
    m.step(1, x[:20], x[:20] + 1, [0, 20])
    m.post_step()
    m.fork_sequence(0, 1)
    m.pre_step(OrderedDict([(0, 1), (1, 1)]))
    k, v, _ = m.step(1, x[20:], x[20:] + 1, [0, 1, 2])
    assert torch.equal(k, torch.cat([x[:21], x[:20], x[21:]])) and torch.equal(v, k + 1)
    te.check_status()


def test_forward_and_backward_with_sinks_in_a_captured_graph():
    """Replays give the eager results.  The captured leaves are their own (views of the same memory): autograd ties a
    leaf's gradient node to the stream of the eager graph that made it, so PyTorch itself cannot capture a backward pass
    of leaves whose eager graph is still alive."""
    g = torch.Generator().manual_seed(17)
    q, k, v = (torch.randn(1, h, 300, 128, generator=g).to(torch.bfloat16).cuda().requires_grad_() for h in (4, 2, 2))
    do = torch.randn(1, 4, 300, 128, generator=g).to(torch.bfloat16).cuda()

    def both():
        own = [t.detach().requires_grad_() for t in (q, k, v)]
        o = te.functional.attention(*own, causal=True, window=(50, 0), sink_tokens=4)
        return (o.detach(), *torch.autograd.grad(o, own, do))

    kept = te.functional.attention(q, k, v, causal=True, window=(50, 0), sink_tokens=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for t in got:
        t.zero_()
    graph.replay()
    want = (kept.detach(), *torch.autograd.grad(kept, (q, k, v), do))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    te.check_status()
