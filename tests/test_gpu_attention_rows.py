"""Packed attention where sequences times heads times the longest sequence pass 32 bits."""
import pytest
import torch

import transformerengine_b200 as te

pytestmark = pytest.mark.gpu


def test_backward_with_more_than_2_to_32_score_rows():
    g = torch.Generator().manual_seed(0)
    n, hq, longest = 33, 128, 2 ** 20                # a bound far above the lengths, as a captured step has it
    lens = [3 + i for i in range(n)]
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    q, k, v = (torch.randn(sum(lens), h, 128, generator=g).to(torch.bfloat16).cuda().requires_grad_() for h in (hq, 1, 1))
    do = torch.randn(sum(lens), hq * 128, generator=g).to(torch.bfloat16).cuda()
    attn = te.DotProductAttention(hq, 128, num_gqa_groups=1, qkv_format="thd", attn_mask_type="padding_causal").cuda()

    def run(bound):
        o = attn(q, k, v, cu_seqlens_q=cu, cu_seqlens_kv=cu, max_seqlen_q=bound, max_seqlen_kv=max(lens))
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))

    assert n * hq * longest > 2 ** 32
    want = run(max(lens))
    got = run(longest)
    te.check_status()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    torch.cuda.empty_cache()                         # 35 GB of row sums
