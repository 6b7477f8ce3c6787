"""Windows of attention beyond every length and beyond 32 bits."""
import pytest
import torch

import transformerengine_b200 as te
from test_gpu_kv_cache import _cum, _filled, _i32
from transformerengine_b200.attention import kv_cache as kc

pytestmark = pytest.mark.gpu

HUGE = [2 ** 31 - 1, 2 ** 32, 2 ** 40]


def _grads(o, leaves, do):
    return (o.detach(), *torch.autograd.grad(o, leaves, do))


@pytest.mark.parametrize("left", HUGE)
@pytest.mark.parametrize("sinks", [0, 5])
@pytest.mark.parametrize("sq,sk,br", [(300, 300, True), (200, 500, True), (500, 200, False), (400, 150, True)])
def test_a_window_beyond_every_length_hides_nothing(left, sinks, sq, sk, br):
    g = torch.Generator().manual_seed(sq)
    mk = lambda h, s: torch.randn(1, h, s, 128, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    q, k, v, do = mk(4, sq).requires_grad_(), mk(2, sk).requires_grad_(), mk(2, sk).requires_grad_(), mk(4, sq)
    run = lambda w: _grads(te.functional.attention(q, k, v, causal=True, window=(w, 0), bottom_right=br, sink_tokens=sinks), (q, k, v), do)  # noqa: E731
    for a, b in zip(run(left), run(sq + sk)):
        assert torch.equal(a, b)
    # without a window: other kernels, the same masks; results and gradients are sums of up to 500 terms around 1
    for a, b in zip(run(left), _grads(te.functional.attention(q, k, v, causal=True, bottom_right=br), (q, k, v), do)):
        assert (a - b).float().norm() <= 2.0 ** -7 * b.float().norm()
    te.check_status()


@pytest.mark.parametrize("window", [(2 ** 32, 2 ** 32), (2 ** 31 - 1, 3), (3, 2 ** 31 - 1), (2 ** 40, 2 ** 40 + 5)])
def test_huge_sides_without_a_causal_mask(window):
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(1, 2, 300, 128, generator=g).to(torch.bfloat16).cuda().requires_grad_() for _ in range(4))
    run = lambda w: _grads(te.functional.attention(q, k, v, window=w), (q, k, v), do)  # noqa: E731
    for a, b in zip(run(window), run(tuple(min(x, 600) for x in window))):
        assert torch.equal(a, b)
    te.check_status()


@pytest.mark.parametrize("left", HUGE)
@pytest.mark.parametrize("sinks", [0, 5])
def test_huge_windows_over_packed_sequences(left, sinks):
    g = torch.Generator().manual_seed(2)
    lens = [200, 1, 317]
    q, k, v = (torch.randn(sum(lens), h, 128, generator=g).to(torch.bfloat16).cuda().requires_grad_() for h in (4, 2, 2))
    do = torch.randn(sum(lens), 4 * 128, generator=g).to(torch.bfloat16).cuda()

    def run(w):
        attn = te.DotProductAttention(4, 128, num_gqa_groups=2, qkv_format="thd", attn_mask_type="padding_causal", window_size=(w, 0),
                                      sink_tokens=sinks).cuda()
        return _grads(attn(q, k, v, cu_seqlens_q=_i32(_cum(lens)), cu_seqlens_kv=_i32(_cum(lens))), (q, k, v), do)

    for a, b in zip(run(left), run(317)):
        assert torch.equal(a, b)
    te.check_status()


@pytest.mark.parametrize("left", HUGE)
@pytest.mark.parametrize("expand", [False, True])
def test_huge_windows_over_the_8_bit_cache(left, expand, monkeypatch):
    monkeypatch.setattr(kc, "_expands", lambda *a: expand)
    lens, qs = [700, 40, 64], [300, 70, 64]            # one with more queries than tokens
    cache, table = _filled(lens, 2, 64, 128, torch.Generator().manual_seed(3))
    q = torch.randn(sum(qs), 8, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    run = lambda w, s: kc.attend(q, cache, table, _i32(_cum(qs)), _i32(lens), max_q=300, max_kv=700, window=(w, 0), sink_tokens=s)  # noqa: E731
    for sinks in (0, 6, 2 ** 40):
        assert torch.equal(run(left, sinks), run(1000, sinks))
    assert (run(left, 0)[300:330] == 0).all()
    te.check_status()
