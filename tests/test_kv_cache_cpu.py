"""The 8-bit paged key/value cache on CPU: rounding, scales, masks, page operations, refusals."""
import math

import pytest
import torch

import transformerengine_b200 as te
from transformerengine_b200.attention import kv_cache as kc


def _pool(pages, h, ps, d):
    return kc.FP8KVCache.allocate(pages, h, ps, d, device="cpu")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _decode(cache):
    out = []
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        out.append(c.float().double() * s.double().repeat_interleave(16, dim=2)[..., None])
    return out


def _round_e4m3_64(y):
    """Nearest e4m3 value, ties to even, saturating, in 64 bits."""
    mag = y.abs()
    step = 2.0 ** ((torch.frexp(mag)[1] - 1).clamp(-6, 60) - 3).double()
    return torch.sign(y) * (torch.round(mag / step) * step).clamp(max=448.0)


@pytest.mark.parametrize("top,exp", [(448.0, 0), (448.0 * 2 ** -8, -8), (449.0, 1), (1.0, -8), (0.0, -60), (1e30, 60), (2.0 ** -80, -60),
                                     (1.75, -8), (1.7500001, -7)])
def test_block_scale_is_the_smallest_power_of_two(top, exp):
    assert kc.block_scale(torch.tensor([top])).item() == 2.0 ** exp


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_append_rounds_once_and_rounds_held_codes_again_when_the_scale_rises(dtype):
    h, ps, d = 2, 32, 24
    cache = _pool(4, h, ps, d)
    table = _i32([[3, 1]])
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, h, d, generator=g).to(dtype)
    x[5] *= 100.0                                     # raises the first block's scale after five tokens
    want = [torch.zeros(h, 48, d, dtype=torch.float64), torch.zeros(h, 3, dtype=torch.float64)]
    done = 0
    for n in (5, 1, 7, 20, 7):
        done += n
        kc.append(cache, x[done - n:done], -x[done - n:done], table, _i32([0, n]), _i32([done]))
        for t in range(done - n, done):               # one token at a time: the same codes by another road
            b = t // 16
            s = kc.block_scale(x[t].float().abs().amax(-1)).double()
            if t % 16:
                s = torch.maximum(s, want[1][:, b])
                held = slice(b * 16, t)
                want[0][:, held] = _round_e4m3_64(want[0][:, held] / s[:, None, None]) * s[:, None, None]
            want[1][:, b] = s
            want[0][:, t] = _round_e4m3_64(x[t].double() / s[:, None]) * s[:, None]
    kv = [torch.cat([c[3], c[1]], dim=1)[:, :40] for c in _decode(cache)]
    # a run of tokens sets the block's scale at once, so codes may be rounded once less than token by token: the second
    # rounding only reaches subnormal codes, half a step of 2^-9 scale each
    tol = want[1].repeat_interleave(16, dim=1)[:, :40, None] * 2.0 ** -10
    assert ((kv[0] - want[0][:, :40]).abs() <= tol).all() and ((kv[1] + want[0][:, :40]).abs() <= tol).all()
    # against the values themselves: half a step of e4m3 relative (2^-4), or of its subnormals, twice
    x64 = x.double().transpose(0, 1)
    assert ((kv[0] - x64).abs() <= x64.abs() * 2.0 ** -4 + 2 * tol).all()
    assert (cache.k_scale[0] == 0).all() and (cache.k_scale[2] == 0).all()      # other pages untouched


def test_append_handles_what_is_not_finite():
    cache = _pool(1, 1, 16, 8)
    x = torch.ones(3, 1, 8)
    x[0, 0, 0], x[1, 0, 1], x[2, 0, 2] = math.nan, math.inf, -math.inf
    kc.append(cache, x, x, _i32([[0]]), _i32([0, 3]), _i32([3]))
    k = _decode(cache)[0][0, 0]
    assert cache.k_scale[0, 0, 0] == 2.0 ** -8
    assert math.isnan(k[0, 0]) and k[1, 1] == 448 / 256 and k[2, 2] == -448 / 256 and k[0, 1] == 1.0


@pytest.mark.parametrize("window,sinks,causal", [(-1, 0, True), (0, 0, True), (5, 0, True), (5, 3, True), (30, 3, True), (-1, 0, False)])
def test_attend_matches_the_definition(window, sinks, causal):
    h, hq, ps, d = 2, 6, 16, 8
    lens, qs = [37, 0, 1, 16, 3], [4, 2, 1, 0, 5]     # the last sequence has more queries than tokens
    cache = _pool(8, h, ps, d)
    table = _i32([[5, 0, 7], [-1, -1, -1], [2, -1, -1], [1, -1, -1], [4, -1, -1]])
    g = torch.Generator().manual_seed(1)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x = torch.randn(2, cu[-1], h, d, generator=g)
    kc.append(cache, x[0], x[1], table, _i32(cu), _i32(lens))
    cq = [0]
    for n in qs:
        cq.append(cq[-1] + n)
    q = torch.randn(cq[-1] + 2, hq, d, generator=g)
    o = kc.attend(q, cache, table, _i32(cq), _i32(lens), max_q=5, max_kv=37, causal=causal, window=(window, 0 if causal else -1),
                  sink_tokens=sinks)
    kv = _decode(cache)
    want = torch.zeros(q.shape, dtype=torch.float64)
    for i, (n, m) in enumerate(zip(lens, qs)):
        pages = [p for p in table[i].tolist() if p >= 0]
        if not pages:
            continue
        k, v = (torch.cat([c[p] for p in pages], dim=1)[:, :n] for c in kv)
        for r in range(m):
            p = n - m + r
            j = torch.arange(n)
            seen = (j <= p) if causal else torch.ones(n, dtype=torch.bool)
            if window >= 0:
                seen = seen & ((p - j <= window) | (j < sinks))
            if not seen.any():
                continue
            for a in range(hq):
                s = (k[a // 3] @ q[cq[i] + r, a].double()) / math.sqrt(d)
                want[cq[i] + r, a] = torch.softmax(s.masked_fill(~seen, -math.inf), 0) @ v[a // 3]
    # fp32 scores and sums of some tens of terms
    torch.testing.assert_close(o.double(), want, rtol=1e-5, atol=1e-5)
    assert (o[cq[-1]:] == 0).all()


def test_gather_and_copy_pages():
    cache = _pool(6, 2, 16, 8)
    x = torch.randn(40, 2, 8)
    table = _i32([[4, 2, 0], [1, -1, -1]])
    kc.append(cache, x, x + 1, table, _i32([0, 30, 40]), _i32([30, 10]))
    k, v = kc.gather(cache, table, _i32([30, 10]), _i32([0, 30]), 40, torch.float32)
    assert (k - x).abs().max() < 0.2 and (v - x - 1).abs().max() < 0.3      # half a step of values below 5
    plain = torch.arange(6.0)[:, None].repeat(1, 3)
    kc.copy_pages([cache, plain], [4, 2, 4], torch.tensor([3, 5, 0]))
    k2, _ = kc.gather(cache, _i32([[3, 5], [0, -1]]), _i32([30, 10]), _i32([0, 30]), 40, torch.float32)
    assert torch.equal(k2[:30], k[:30]) and torch.equal(k2[30:], k[:10])
    assert plain[:, 0].tolist() == [4.0, 1.0, 2.0, 4.0, 4.0, 2.0]
    kc.copy_pages([], [0], [1])
    kc.copy_pages([plain], [], [])


def test_refusals():
    cache = _pool(3, 1, 16, 8)
    plain = torch.zeros(3, 2)
    for src, dst, what in (([0, 1], [2, 2], "twice"), ([0], [3], "range"), ([-1], [0], "range"), ([0, 1], [1, 2], "read and written"),
                           ([0], [1, 2], "as many")):
        with pytest.raises(ValueError, match=what):
            kc.copy_pages([plain], src, dst)
    with pytest.raises(ValueError, match="multiple of 16"):
        kc.FP8KVCache.allocate(2, 1, 24, 64)
    with pytest.raises(ValueError, match="head dims"):
        kc.FP8KVCache.allocate(2, 1, 16, 80, device="cuda")
    q = torch.zeros(1, 1, 8, requires_grad=True)
    meta = dict(max_q=1, max_kv=1)
    with pytest.raises(RuntimeError, match="no backward"):
        kc.attend(q, cache, _i32([[0]]), _i32([0, 1]), _i32([1]), **meta)
    q = q.detach()
    with pytest.raises(ValueError, match="left side only"):
        kc.attend(q, cache, _i32([[0]]), _i32([0, 1]), _i32([1]), window=(3, 2), **meta)
    with pytest.raises(ValueError, match="causal mask"):
        kc.attend(q, cache, _i32([[0]]), _i32([0, 1]), _i32([1]), window=(3, -1), causal=False, **meta)
    with pytest.raises(ValueError, match="negative"):
        kc.attend(q, cache, _i32([[0]]), _i32([0, 1]), _i32([1]), sink_tokens=-1, **meta)
    with pytest.raises(ValueError, match="holds no page"):
        kc.append(cache, torch.zeros(1, 1, 8), torch.zeros(1, 1, 8), _i32([[-1]]), _i32([0, 1]), _i32([1]))


# ------------------------------------------------------------------------------------- window with visible first tokens
def _formula(q, k, v, do, window, sinks, causal, off):
    """Output and gradients of windowed attention in 64 bits from the formulas."""
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    b, hq, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    g = hq // hk
    i, j = torch.arange(sq, device=q.device)[:, None] + off, torch.arange(sk, device=q.device)[None]
    seen = (j >= i - window[0]) | (j < sinks) if window[0] >= 0 else torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    right = 0 if causal else window[1]
    if right >= 0:
        seen = seen & (j <= i + right)
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = (q @ kk.transpose(-1, -2)) * d ** -0.5
    p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -math.inf), -1))
    o = p @ vv
    ds = p * (do @ vv.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * d ** -0.5
    fold = lambda t: t.reshape(b, hk, g, sk, d).sum(2)  # noqa: E731
    return o, ds @ kk, fold(ds.transpose(-1, -2) @ q), fold(p.transpose(-1, -2) @ do)


@pytest.mark.parametrize("sq,sk,window,sinks,causal,bottom_right", [
    (20, 20, (4, 0), 2, True, True), (20, 33, (4, 0), 3, True, True), (33, 20, (4, 0), 3, True, False), (16, 16, (0, 0), 16, True, True),
    (12, 12, (3, 2), 2, False, True), (12, 12, (-1, 0), 2, True, True)])
def test_window_with_sinks_and_its_gradients(sq, sk, window, sinks, causal, bottom_right):
    g = torch.Generator().manual_seed(2)
    mk = lambda h, s: torch.randn(2, h, s, 8, generator=g).requires_grad_()  # noqa: E731
    q, k, v, do = mk(4, sq), mk(2, sk), mk(2, sk), torch.randn(2, 4, sq, 8, generator=g)
    o = te.functional.attention(q, k, v, causal=causal, window=window, bottom_right=bottom_right, sink_tokens=sinks)
    grads = torch.autograd.grad(o, (q, k, v), do)
    want = _formula(q, k, v, do, window, sinks, causal, sk - sq if bottom_right else 0)
    for a, b in zip((o, *grads), want):
        torch.testing.assert_close(a.double(), b, rtol=1e-4, atol=1e-5)
    # the formulas against a central difference along a random direction, in 64 bits
    step, at = 1e-5, [t.detach().double() for t in (q, k, v)]
    for n in range(3):
        way = torch.randn(at[n].shape, generator=g, dtype=torch.float64)
        f = [(_formula(*[t + e * way if m == n else t for m, t in enumerate(at)], do, window, sinks, causal,
                       sk - sq if bottom_right else 0)[0] * do.double()).sum() for e in (step, -step)]
        torch.testing.assert_close((f[0] - f[1]) / (2 * step), (want[n + 1] * way).sum(), rtol=1e-6, atol=1e-7)


def test_sink_tokens_refuses_a_negative_count():
    q = torch.zeros(1, 1, 2, 8)
    with pytest.raises(ValueError, match="negative"):
        te.functional.attention(q, q, q, causal=True, window=(1, 0), sink_tokens=-1)


# ----------------------------------------------------------------------------------------- managers, modules, generation
from collections import OrderedDict  # noqa: E402


def _paged(fp8, **kw):
    d = dict(total_num_pages=8, page_size=16, num_heads_kv=1, head_dim_k=8, dtype=torch.float32, max_batch_size=4,
             max_sequence_length=128, device="cpu")
    d.update(kw)
    return (te.FP8PagedKVCacheManager if fp8 else te.PagedKVCacheManager)(**d)


def _tokens(m, x):
    """One step of every sequence in m.step_dict: keys x, values -x."""
    cu = [0]
    for n in m.step_dict.values():
        cu.append(cu[-1] + n)
    k, v, lens = m.step(1, x, -x, cu)
    m.post_step()
    return k, lens


@pytest.mark.parametrize("fp8", [False, True])
def test_forked_sequences_share_pages_until_one_writes(fp8):
    m = _paged(fp8)
    g = torch.Generator().manual_seed(3)
    # powers of two are exact in 8 bits
    x = torch.exp2(torch.randint(-3, 4, (40, 1, 8), generator=g).float())
    m.pre_step(OrderedDict([(0, 20)]))
    _tokens(m, x[:20])
    m.fork_sequence(0, 1)
    m.fork_sequence(0, 2)
    assert m.page_table[1] == m.page_table[0] and len(m.free_pages) == 6
    m.pre_step(OrderedDict([(0, 1), (1, 1), (2, 0)]))
    assert m.page_table[0][0] == m.page_table[1][0] == m.page_table[2][0]
    assert len({m.page_table[i][1] for i in range(3)}) == 3 and len(m.free_pages) == 4
    k, lens = _tokens(m, x[20:22])
    assert lens == [21, 21, 20]
    assert torch.equal(k[:20], x[:20]) and torch.equal(k[20], x[20]) and torch.equal(k[21:41], x[:20]) and torch.equal(k[41], x[21])
    assert torch.equal(k[42:], x[:20])
    m.truncate_sequence(1, 16)                        # its copy of the second page goes back
    assert len(m.free_pages) == 5 and m.lengths[1] == 16
    m.deallocate_sequence(0)
    assert len(m.free_pages) == 6                     # the first page has two owners left
    moved = m.compact()
    used = {p for t in m.page_table.values() for p in t}
    assert used == set(range(len(used))) and sorted(m.free_pages + list(used)) == list(range(8)) and moved <= 2
    m.pre_step(OrderedDict([(1, 2), (2, 1)]))
    k, _ = _tokens(m, x[22:25])
    assert torch.equal(k[:16], x[:16]) and torch.equal(k[16:18], x[22:24]) and torch.equal(k[18:38], x[:20]) and torch.equal(k[38], x[24])
    m.pre_step(OrderedDict())
    assert len(m.free_pages) == 8 and not m.page_refs


def test_manager_refusals():
    m = _paged(True)
    m.pre_step(OrderedDict([(0, 20)]))
    m.post_step()
    for call, what in ((lambda: m.fork_sequence(5, 6), "unknown"), (lambda: m.fork_sequence(0, 0), "exists"),
                       (lambda: m.truncate_sequence(0, 21), "cannot cut"), (lambda: m.truncate_sequence(9, 0), "unknown")):
        with pytest.raises(ValueError, match=what):
            call()
    m.fork_sequence(0, 1), m.fork_sequence(0, 2), m.fork_sequence(0, 3)
    with pytest.raises(ValueError, match="max_batch_size"):
        m.fork_sequence(0, 4)
    with pytest.raises(AssertionError, match="out of pages"):
        m.pre_step(OrderedDict([(0, 1), (1, 1), (2, 90), (3, 0)]))
    with pytest.raises(ValueError, match="multiple of 16"):
        _paged(True, page_size=8)
    kw = dict(num_heads_kv=1, head_dim_k=8, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError, match="is paged"):
        te.InferenceParams(2, 32, cache_dtype=torch.float8_e4m3fn, **kw)
    with pytest.raises(ValueError, match="cache_dtype"):
        te.InferenceParams(2, 32, cache_dtype=torch.int8, **kw)
    with pytest.raises(ValueError, match="8-bit cache"):
        te.InferenceParams(2, 32, window_size=4, **kw)
    with pytest.raises(ValueError, match="need a paged cache"):
        te.InferenceParams(2, 32, **kw).fork_sequence(0, 1)


def test_pages_out_of_the_window_return_to_the_pool():
    m = _paged(True, window_size=20, sink_tokens=3, total_num_pages=5)
    g = torch.Generator().manual_seed(4)
    x = torch.exp2(torch.randint(-3, 4, (100, 1, 8), generator=g).float())
    q = torch.randn(100, 2, 8, generator=g)
    full = kc.FP8KVCache.allocate(7, 1, 16, 8, device="cpu")
    kc.append(full, x, -x, _i32([list(range(7))]), _i32([0, 100]), _i32([100]))
    done = 0
    for n in [30] + [10] * 7:
        m.pre_step(OrderedDict([(0, n)]))
        o = m.attend(1, q[done:done + n], x[done:done + n], -x[done:done + n], scale=1.0, causal=True, window=(20, 0), sink_tokens=3)
        m.post_step()
        done += n
        want = kc.attend(q[done - n:done], full, _i32([list(range(7))]), _i32([0, n]), _i32([done]), max_q=n, max_kv=done, scale=1.0,
                         window=(20, 0), sink_tokens=3)
        torch.testing.assert_close(o, want, rtol=0, atol=0)
    assert m.page_table[0][0] >= 0 and m.page_table[0][1] == -1 and len(m.page_table[0]) == 7
    with pytest.raises(ValueError, match="given back"):
        m.truncate_sequence(0, 40)
    m.truncate_sequence(0, 97)
    with pytest.raises(ValueError, match="keeps a window"):
        m.attend(1, q[:1], x[:1], x[:1], scale=1.0, causal=True, window=(21, 0), sink_tokens=3)
    with pytest.raises(ValueError, match="keeps a window"):
        m.attend(1, q[:1], x[:1], x[:1], scale=1.0, causal=True, window=None, sink_tokens=3)


@pytest.mark.parametrize("fmt", ["bshd", "sbhd"])
@pytest.mark.parametrize("window,sinks", [(None, 0), ((4, 0), 2)])
def test_incremental_attention_on_the_8_bit_cache(fmt, window, sinks):
    """Step by step equals one pass, up to the rounding of keys and values (half a step of e4m3 and a requantization)."""
    torch.manual_seed(0)
    b, h, hk, d, total = 2, 4, 2, 16, 20
    mha = te.MultiheadAttention(h * d, h, num_gqa_groups=hk, attention_dropout=0.0, attn_mask_type="causal", qkv_format=fmt, bias=False,
                                params_dtype=torch.float32, device="cpu", window_size=window, sink_tokens=sinks).eval()
    rope = te.RotaryPositionEmbedding(d)(64)          # the cache's length: padding has positions too
    x = torch.randn(b, total, h * d)
    cut = lambda t: t if fmt == "bshd" else t.transpose(0, 1)  # noqa: E731
    with torch.no_grad():
        full = cut(mha(cut(x), rotary_pos_emb=rope))
        params = te.InferenceParams(4, 64, num_heads_kv=hk, head_dim_k=d, dtype=torch.float32, is_paged=True, page_size=16,
                                    total_num_pages=16, qkv_format=fmt, device="cpu", cache_dtype=torch.float8_e4m3fn)
        outs, pos = [], 0
        for n in (7, 3, 1, 1, 8):
            params.pre_step(OrderedDict((i, n) for i in range(b)))
            outs.append(cut(mha(cut(x[:, pos:pos + n]), rotary_pos_emb=rope, inference_params=params)))
            pos += n
        # a ragged step: the second sequence is padded
        params.truncate_sequence(0, 18)
        params.truncate_sequence(1, 19)
        params.pre_step(OrderedDict([(0, 2), (1, 1)]))
        ragged = torch.stack([x[0, 18:20], torch.cat([x[1, 19:20], torch.full((1, h * d), 9.0)])])
        again = cut(mha(cut(ragged), rotary_pos_emb=rope, inference_params=params))
    inc = torch.cat(outs, dim=1)
    assert (inc - full).norm() / full.norm() < 2.0 ** -3      # keys and values off by up to 2^-4 each
    assert (again[0] - full[0, 18:20]).norm() / full[0, 18:20].norm() < 2.0 ** -3
    assert (again[1, :1] - full[1, 19:20]).norm() / full[1, 19:20].norm() < 2.0 ** -3
    with pytest.raises(RuntimeError, match="no backward"):
        mha(cut(x[:, :1].repeat(1, 2, 1)), rotary_pos_emb=rope, inference_params=params)
    params.pre_step(OrderedDict([(0, 1), (1, 1)]))
    k, v = params.convert_paged_to_nonpaged(None)
    assert k.shape == (2, 32, hk, d) and torch.isfinite(k).all()


def test_variants_without_a_cache_kernel_read_expanded_keys():
    torch.manual_seed(1)
    attn = te.DotProductAttention(4, 16, num_gqa_groups=2, qkv_format="bshd", attn_mask_type="causal", softmax_type="off-by-one",
                                  layer_number=1).eval()
    params = te.InferenceParams(1, 64, num_heads_kv=2, head_dim_k=16, dtype=torch.float32, is_paged=True, page_size=16, total_num_pages=4,
                                device="cpu", cache_dtype=torch.float8_e4m3fn)
    q, k, v = torch.randn(1, 9, 4, 16), torch.exp2(torch.randint(-3, 3, (1, 9, 2, 16)).float()), torch.ones(1, 9, 2, 16)
    with torch.no_grad():
        params.pre_step(OrderedDict([(0, 9)]))
        o = attn(q, k, v, inference_params=params)
        torch.testing.assert_close(o, attn(q, k, v), rtol=1e-5, atol=1e-6)     # these keys and values are exact in 8 bits
        params = te.InferenceParams(1, 64, num_heads_kv=2, head_dim_k=16, dtype=torch.float32, is_paged=True, page_size=16, total_num_pages=4,
                                    device="cpu", cache_dtype=torch.float8_e4m3fn, window_size=3)
        params.pre_step(OrderedDict([(0, 9)]))
        with pytest.raises(ValueError, match="keeps a window"):               # this layer looks at everything
            attn(q, k, v, inference_params=params)


def test_generation_with_forks_and_an_8_bit_cache():
    """The whole run: a windowed model with sinks decodes, forks a sequence, drops drafts, and the pool is compacted."""
    from transformerengine_b200.models.mistral import MistralConfig, MistralModel
    torch.manual_seed(2)
    cfg = MistralConfig.tiny(params_dtype=torch.float32, sliding_window=24, sink_tokens=4)
    model = MistralModel(cfg, device="cpu").eval()
    prompt = torch.randint(0, cfg.vocab_size, (2, 40))
    kw = dict(is_paged=True, page_size=16, total_num_pages=16)
    out = model.generate(prompt, 20, cache_dtype=torch.float8_e4m3fn, **kw)
    assert out.shape == (2, 60)
    # logits against the full pass on the generated tokens: what the cache rounds moves them by a few percent
    with torch.no_grad():
        full = model(out).transpose(0, 1)
        params = model.make_inference_params(4, 96, cache_dtype=torch.float8_e4m3fn, **kw)
        assert params.cache_manager.window_size == 23 and params.cache_manager.sink_tokens == 4
        params.pre_step(OrderedDict([(0, 50), (1, 50)]))
        model(out[:, :50], inference_params=params)
        params.fork_sequence(1, 7)
        params.pre_step(OrderedDict([(0, 3), (1, 3), (7, 3)]))
        model(torch.cat([out[:, 50:53], out[:1, 30:33]]), inference_params=params)
        params.truncate_sequence(7, 50)
        params.compact()
        params.pre_step(OrderedDict([(1, 3), (7, 6)]))
        step = torch.cat([torch.cat([out[1:, 53:56], out[1:, :3]], 1), out[1:, 50:56]])
        logits = model(step, inference_params=params).transpose(0, 1)
    for got, at in ((logits[0, :3], slice(53, 56)), (logits[1], slice(50, 56))):
        assert (got - full[1, at]).norm() / full[1, at].norm() < 2.0 ** -3


@pytest.mark.parametrize("family", ["mistral", "gpt", "gemma"])
def test_generation_example_on_the_8_bit_cache(family):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "generation.py")
    spec = importlib.util.spec_from_file_location("generation_example", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    out = mod.main(["--family", family, "--cache-8bit", "1", "--batch", "3", "--prompt", "6", "--new-tokens", "4"])
    assert out.shape == (3, 10)
