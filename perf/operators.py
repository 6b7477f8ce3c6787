"""Workloads of the streaming-attention operators: attention through a sliding window with visible first tokens
(training), and the 8-bit paged key/value cache that serves the same models (append, attend, page copies).

``run`` computes an operator either in its plain form (elementary torch operations in 32 bits, rounded once at the
end; ``own = False``) or through this package's entry points (``own = True``).  ``exact`` restates the definition in
64 bits.  Definitions, with ``g = hq / hk`` query heads per key head and all masks aligned bottom-right:

* visible(i, j): ``j <= p_i`` and (``p_i - j <= window`` or ``j < sinks``), ``p_i`` = position of query i; a window of
  -1 is unbounded.  ``o_i = sum_j softmax_j(scale q_i k_j | visible) v_j``; a row that sees nothing is 0.
* the cache holds e4m3 codes ``[pages, heads, page, d]`` and one power-of-two scale for every 16 tokens of a head,
  the smallest one (2^-60 .. 2^60) with ``max|x| <= 448 scale``; appending to a partly filled block may raise its
  scale, and its older codes are then rounded again.
"""
import math

import torch

own = False

BLOCK = 16                      # tokens that share a scale
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


# --------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one optimizer step's attention of a Mistral-like layer: the smallest (a debugging run, odd length) ...
        dict(name="train_small_odd", kind="train", b=1, hq=4, hk=2, s=333, window=64, sinks=4, dtype="fp16", layout="bshd"),
        # ... an ordinary micro-batch of the 8B geometry, and a long document with Mistral's window
        dict(name="train_4k", kind="train", b=2, hq=32, hk=8, s=4096, window=1023, sinks=4, dtype="bf16", layout="sbhd"),
        dict(name="train_16k", kind="train", b=1, hq=16, hk=4, s=16384, window=4095, sinks=16, dtype="bf16", layout="bshd"),
        # one decoding step's new tokens of a full serving batch, and the tokens of a few ragged prompts
        dict(name="append_decode", kind="append", n=256, hk=8, d=128, page=64, lo=1, hi=1, ctx=1500, dtype="bf16"),
        dict(name="append_prompts", kind="append", n=7, hk=8, d=128, page=64, lo=300, hi=8000, ctx=100, dtype="bf16"),
        # a single short conversation (latency), the full serving batch, few very long documents
        dict(name="attend_one_short", kind="attend", n=1, hq=32, hk=8, d=128, page=64, kv_lo=200, kv_hi=200, qn=1, window=-1,
             sinks=0, dtype="bf16"),
        dict(name="attend_batch64", kind="attend", n=64, hq=32, hk=8, d=128, page=64, kv_lo=500, kv_hi=8000, qn=1, window=-1,
             sinks=0, dtype="bf16"),
        dict(name="attend_long", kind="attend", n=4, hq=64, hk=8, d=128, page=128, kv_lo=60000, kv_hi=130000, qn=1, window=-1,
             sinks=0, dtype="bf16"),
        # streaming: window and sinks over endless conversations; four drafted tokens verified at a time, head dim 64
        dict(name="attend_stream_d64", kind="attend", n=96, hq=16, hk=4, d=64, page=32, kv_lo=3000, kv_hi=20000, qn=4,
             window=2047, sinks=4, dtype="fp16"),
        # the next chunk of two long prompts
        dict(name="attend_chunk", kind="attend", n=2, hq=32, hk=8, d=128, page=64, kv_lo=4000, kv_hi=9000, qn=1024, window=-1,
             sinks=0, dtype="bf16"),
        # the last pages of eight forked conversations, and a compaction of the pool, over all layers of a model
        dict(name="pages_fork", kind="pages", layers=32, pages=256, moved=8, hk=8, d=128, page=64),
        dict(name="pages_compact", kind="pages", layers=32, pages=1024, moved=400, hk=8, d=128, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["train", "append", "attend", "attend", "pages"])
    hk = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 4, 8])
    dt = rng.choice(["bf16", "fp16"])
    if kind == "train":
        s = _log(rng, 2, 8192)
        return dict(kind=kind, b=rng.choice([1, 2]), hq=hk * min(g, 32 // hk), hk=hk, s=s, window=rng.randint(0, 2 * s) // 2,
                    sinks=rng.choice([0, 1, 4, 64, 130]), dtype=dt, layout=rng.choice(["bshd", "sbhd"]))
    if kind == "append":
        lo = _log(rng, 1, 2000)
        return dict(kind=kind, n=_log(rng, 1, 64), hk=hk, d=rng.choice([64, 128, 256]), page=rng.choice([16, 32, 64, 128]),
                    lo=rng.choice([1, lo]), hi=lo, ctx=_log(rng, 1, 2000), dtype=dt)
    if kind == "attend":
        qn = rng.choice([1, 1, 1, 2, 5, _log(rng, 8, 700)])
        hi = max(qn, _log(rng, 1, 30000))
        n = max(1, min(_log(rng, 1, 128), 400000 // (hi * (1 + qn // 8))))
        d = rng.choice([64, 128, 128, 256])
        return dict(kind=kind, n=n, hq=hk * g, hk=hk, d=d, page=rng.choice([16, 32, 64, 128]), kv_lo=max(qn, hi // rng.choice([1, 3, 10])),
                    kv_hi=hi, qn=qn, window=rng.choice([-1, -1, rng.randint(0, hi)]), sinks=rng.choice([0, 1, 4, 100]), dtype=dt)
    pages = _log(rng, 8, 600)
    return dict(kind=kind, layers=rng.randint(1, 32), pages=pages, moved=rng.randint(1, pages // 2), hk=hk, d=rng.choice([64, 128, 256]),
                page=rng.choice([16, 32, 64]))


# --------------------------------------------------------------------------------------------------- what a user has
def _lens(gen, n, lo, hi):
    lens = torch.randint(lo, hi + 1, (n,), generator=gen)
    lens[0] = hi
    return lens


def _cumulative(lens):
    return torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32)


def _codes(x, scale):
    """e4m3 codes of x / scale (the scale is a power of two), rounded to nearest, ties to even."""
    return (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _scale_for(top):
    """The smallest power of two with top <= 448 * scale."""
    m, e = torch.frexp(top.float())
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-60, 60)
    e = torch.where(top > 0, e, torch.full_like(e, -60)).to(torch.int32)
    return ((e + 127) << 23).view(torch.float32)      # 2^e by its bits


def _cache(g, pages, hk, page, d):
    """A filled cache: keys with a few strong channels, as after a rotation, and plain values."""
    out = []
    for strong in (True, False):
        x = torch.randn(pages, hk, page, d, generator=g, device="cuda")
        if strong:
            x[..., ::17] *= 4.0
        x *= torch.exp(0.5 * torch.randn(pages, hk, page // BLOCK, 1, 1, generator=g, device="cuda")).expand(
            -1, -1, -1, BLOCK, 1).reshape(pages, hk, page, 1)
        s = _scale_for(x.reshape(pages, hk, page // BLOCK, BLOCK * d).abs().amax(-1))
        out += [_codes(x, s.repeat_interleave(BLOCK, dim=-1)[..., None]), s]
    return out


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    st = {"case": c}
    if c["kind"] == "train":
        shape = {"bshd": lambda n: (c["b"], c["s"], n, 128), "sbhd": lambda n: (c["s"], c["b"], n, 128)}[c["layout"]]
        view = {"bshd": (0, 2, 1, 3), "sbhd": (1, 2, 0, 3)}[c["layout"]]
        rnd = lambda n: torch.randn(shape(n), generator=g, device="cuda").to(DT[c["dtype"]]).permute(view)  # noqa: E731
        st.update(q=rnd(c["hq"]).requires_grad_(), k=rnd(c["hk"]).requires_grad_(), v=rnd(c["hk"]).requires_grad_(), do=rnd(c["hq"]))
        return st
    if c["kind"] == "pages":
        k, ks, v, vs = _cache(g, c["pages"] * c["layers"], c["hk"], c["page"], c["d"])
        stack = lambda t: t.reshape(c["layers"], c["pages"], *t.shape[1:])  # noqa: E731
        perm = torch.randperm(c["pages"], generator=h).to(torch.int32)
        st.update(k=stack(k), ks=stack(ks), v=stack(v), vs=stack(vs), src=perm[:c["moved"]].clone(),
                  dst=perm[c["pages"] - c["moved"]:].clone())
        return st
    if c["kind"] == "append":
        new = _lens(h, c["n"], c["lo"], c["hi"])
        old = torch.randint(0, c["ctx"] + 1, (c["n"],), generator=h)
        st["max_new"], lens = int(new.max()), new + old
        st["cu_new"] = _cumulative(new).cuda()
        t = int(new.sum())
        mixed = torch.randn(t, 2 * c["hk"], c["d"], generator=g, device="cuda").to(DT[c["dtype"]])
        st["new_k"], st["new_v"] = mixed[:, :c["hk"]], mixed[:, c["hk"]:]      # views of one projection's output
    else:
        lens = _lens(h, c["n"], c["kv_lo"], c["kv_hi"])
        st["max_kv"] = int(lens.max())
        qn = torch.full((c["n"],), c["qn"])
        st["cu_q"] = _cumulative(qn).cuda()
        st["q"] = (1.5 * torch.randn(int(qn.sum()), c["hq"], c["d"], generator=g, device="cuda")).to(DT[c["dtype"]])
    width = -(-int(lens.max()) // c["page"])
    need = -(-lens // c["page"])
    # a pool of a size of its own, whatever lengths the seed gives
    total = c["n"] * -(-(c["hi"] + c["ctx"]) // c["page"]) if c["kind"] == "append" else int(need.sum()) + 3
    ids = torch.randperm(total, generator=h).to(torch.int32)
    table = torch.full((c["n"], width), -1, dtype=torch.int32)
    at = 0
    for i, w in enumerate(need.tolist()):
        table[i, :w] = ids[at:at + w]
        at += w
    st["table"], st["lens"] = table.cuda(), lens.to(torch.int32).cuda()
    st["k"], st["ks"], st["v"], st["vs"] = _cache(g, total, c["hk"], c["page"], c["d"])
    return st


# ------------------------------------------------------------------------------------------------------ the plain form
def _plain_train(q, k, v, do, window, sinks):
    b, hq, s, d = q.shape
    hk = k.shape[1]
    qf, dof = (x.detach().float().reshape(b, hk, hq // hk, s, d) for x in (q, do))
    kf, vf = (x.detach().float()[:, :, None] for x in (k, v))
    i = torch.arange(s, device=q.device)
    off = i[:, None] - i[None, :]
    hidden = (off < 0) | ((off > window) & (i[None, :] >= sinks))
    p = ((qf @ kf.transpose(-1, -2)) * d ** -0.5).masked_fill_(hidden, -torch.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = p @ vf
    dv = (p.transpose(-1, -2) @ dof).sum(2)
    ds = dof @ vf.transpose(-1, -2)
    ds = ds.sub_((dof * o).sum(-1, keepdim=True)).mul_(p).mul_(d ** -0.5)
    dq = (ds @ kf).reshape(b, hq, s, d)
    dk = (ds.transpose(-1, -2) @ qf).sum(2)
    return [x.to(q.dtype) for x in (o.reshape(b, hq, s, d), dq, dk, dv)]


def _plain_append(codes, scales, new, table, cu, lens, max_new, page):
    n, hk, d = lens.numel(), new.shape[1], new.shape[2]
    old = lens - (cu[1:] - cu[:-1])
    nb = (max_new + BLOCK - 2) // BLOCK + 1
    blk = torch.div(old, BLOCK, rounding_mode="floor")[:, None] + torch.arange(nb, device=new.device)     # [n, nb]
    pos = blk[..., None] * BLOCK + torch.arange(BLOCK, device=new.device)                                # [n, nb, 16]
    live = blk * BLOCK < lens[:, None]
    per = page // BLOCK
    pg = table.long().gather(1, torch.div(blk, per, rounding_mode="floor").clamp(max=table.shape[1] - 1).long())
    pg, sub = pg[live], (blk % per)[live].long()
    pos, old_b, cu_b, len_b = pos[live], old[:, None].expand(n, nb)[live], cu[:-1, None].expand(n, nb)[live], lens[:, None].expand(n, nb)[live]
    fresh = (pos >= old_b[:, None]) & (pos < len_b[:, None])                                              # [m, 16]
    kept = pos < old_b[:, None]
    x = new.float()[(cu_b[:, None] + pos - old_b[:, None]).clamp(0, new.shape[0] - 1)].transpose(1, 2)        # [m, h, 16, d]
    held = codes.view(torch.uint8).view(-1, hk, per, BLOCK, d)[pg, :, sub].view(torch.float8_e4m3fn)         # [m, h, 16, d]
    was = scales[pg, :, sub]                                                                              # [m, h]
    top = torch.where(fresh[:, None, :, None], x.abs(), torch.zeros_like(x)).amax((-1, -2))
    now = _scale_for(top)
    now = torch.where(kept.any(-1)[:, None], torch.maximum(now, was), now)
    again = _codes(held.float() * was[..., None, None], now[..., None, None])
    put = torch.where(fresh[:, None, :, None], _codes(x, now[..., None, None]).view(torch.uint8),
                      torch.where(kept[:, None, :, None], again.view(torch.uint8), held.view(torch.uint8)))
    codes.view(torch.uint8).view(-1, hk, per, BLOCK, d)[pg, :, sub] = put
    scales[pg, :, sub] = now


def _plain_attend(st):
    c, q, lens, cu = st["case"], st["q"], st["lens"].long(), st["cu_q"].long()
    n, hk, d = c["n"], c["hk"], c["d"]
    gq = c["hq"] // hk
    table = st["table"].long().clamp(min=0)

    def values(codes, scales):
        x = codes.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()             # [n, w, h, page, d]
        x = x.view(n, -1, hk, c["page"] // BLOCK, BLOCK, d) * scales[table][..., None, None]
        return x.view(n, -1, hk, c["page"], d).transpose(1, 2).reshape(n, hk, 1, -1, d)

    qn = cu[1:] - cu[:-1]
    iq = torch.arange(c["qn"], device=q.device)
    real = iq[None] < qn[:, None]                                                            # [n, qmax]
    at = (cu[:-1, None] + iq).clamp(max=q.shape[0] - 1)
    qf = q.float()[at].view(n, c["qn"], hk, gq, d).permute(0, 2, 3, 1, 4)                    # [n, h, g, qmax, d]
    s = (qf @ values(st["k"], st["ks"]).transpose(-1, -2)) * d ** -0.5
    pos = (lens - qn)[:, None] + iq
    j = torch.arange(s.shape[-1], device=q.device)
    off = pos[..., None] - j
    hidden = (off < 0) | (j >= lens[:, None, None])
    if c["window"] >= 0:
        hidden = hidden | ((off > c["window"]) & (j >= c["sinks"]))
    s = s.masked_fill_(hidden[:, None, None], -torch.inf)
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(top > -torch.inf, top, torch.zeros_like(top))).exp_()
    total = s.sum(-1, keepdim=True)
    o = (s @ values(st["v"], st["vs"])) / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4).reshape(n, c["qn"], c["hq"], d)[real].to(q.dtype)


def run(state):
    c = state["case"]
    if c["kind"] == "train":
        q, k, v, do = state["q"], state["k"], state["v"], state["do"]
        if not own:
            return _plain_train(q, k, v, do, c["window"], c["sinks"])
        import transformerengine_b200 as te
        o = te.functional.attention(q, k, v, causal=True, window=(c["window"], 0), sink_tokens=c["sinks"], out_format=c["layout"])
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]
    if c["kind"] == "pages":
        if own:
            import transformerengine_b200 as te
            if "layers" not in state:       # a program holds its layers' caches one by one
                state["layers"] = [te.kv_cache.FP8KVCache(*t) for t in zip(*(state[kind].unbind(0) for kind in ("k", "v", "ks", "vs")))]
            te.kv_cache.copy_pages(state["layers"], state["src"], state["dst"])
        else:
            src, dst = state["src"].cuda().long(), state["dst"].cuda().long()
            k, v = state["k"].view(torch.uint8), state["v"].view(torch.uint8)
            k[:, dst], v[:, dst] = k[:, src], v[:, src]
            state["ks"][:, dst], state["vs"][:, dst] = state["ks"][:, src], state["vs"][:, src]
        return [state[kind] for kind in ("k", "ks", "v", "vs")]
    if c["kind"] == "append":
        if own:
            import transformerengine_b200 as te
            te.kv_cache.append(te.kv_cache.FP8KVCache(state["k"], state["v"], state["ks"], state["vs"]), state["new_k"], state["new_v"],
                               state["table"], state["cu_new"], state["lens"], max_new=state["max_new"])
        else:
            _plain_append(state["k"], state["ks"], state["new_k"], state["table"], state["cu_new"], state["lens"],
                              state["max_new"], c["page"])
            _plain_append(state["v"], state["vs"], state["new_v"], state["table"], state["cu_new"], state["lens"],
                              state["max_new"], c["page"])
        return [state[kind] for kind in ("k", "ks", "v", "vs")]
    if own:
        import transformerengine_b200 as te
        return te.kv_cache.attend(state["q"], te.kv_cache.FP8KVCache(state["k"], state["v"], state["ks"], state["vs"]), state["table"],
                                  state["cu_q"], state["lens"], max_q=c["qn"], max_kv=state["max_kv"],
                                  window=(c["window"], 0), sink_tokens=c["sinks"])
    return _plain_attend(state)


# --------------------------------------------------------------------------------------------------------- what it costs
def _seen(p, window, sinks):
    """Keys that the query at position p sees."""
    return p + 1 if window < 0 else min(p + 1, window + 1) + max(0, min(sinks, p - window))


def work(case):
    c = case
    if c["kind"] == "train":
        pairs = sum(_seen(p, c["window"], c["sinks"]) for p in range(c["s"])) * c["b"] * c["hq"]
        # forward q k^T and p v; backward q k^T again, dO v^T, p^T dO, dS k, dS^T q
        size = c["b"] * c["s"] * 128 * 2
        return {"bytes": size * (4 * c["hq"] + 4 * c["hk"]), "flops": 14.0 * 128 * pairs}
    if c["kind"] == "pages":
        page = c["hk"] * (c["page"] * c["d"] + c["page"] // BLOCK * 4) * 2
        return {"bytes": 2.0 * c["layers"] * c["moved"] * page, "flops": 0.0}
    if c["kind"] == "append":
        t = c["n"] * (c["lo"] + c["hi"]) / 2
        return {"bytes": t * c["hk"] * c["d"] * 2 * (2 + 1), "flops": 0.0}
    mean = (c["kv_lo"] + c["kv_hi"]) / 2
    first = max(0, int(mean) - c["qn"])
    pairs = sum(_seen(p, c["window"], c["sinks"]) for p in range(first, int(mean)))
    read = min(mean, _seen(first, c["window"], c["sinks"]) + c["qn"] - 1)
    return {"bytes": c["n"] * (2.0 * read * c["hk"] * (c["d"] + 4 / BLOCK) + 2 * c["qn"] * c["hq"] * c["d"] * 2),
            "flops": 4.0 * c["n"] * c["hq"] * c["d"] * pairs}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def _exact_power(e):
    return torch.tensor([2.0 ** n for n in range(-100, 101)], dtype=torch.float64, device=e.device)[e.long() + 100]


def _exact_round(y):
    """To the nearest e4m3 value, ties to even, saturating: y in 64 bits."""
    mag = y.abs()
    step = _exact_power((torch.frexp(mag)[1] - 1).clamp(-6, 60) - 3)      # frexp: mag = m * 2^e with m in [0.5, 1)
    return torch.sign(y) * (torch.round(mag / step) * step).clamp(max=448.0)


def _exact_scale(top):
    """The least power of two that is at least top / 448."""
    m, e = torch.frexp(top / 448.0)
    return _exact_power(torch.where(m == 0.5, e - 1, e).clamp(-60, 60).masked_fill(top == 0, -60))


def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    if c["kind"] == "train":
        q, k, v, do = (st[x].detach().double() for x in ("q", "k", "v", "do"))
        gq, s = c["hq"] // c["hk"], c["s"]
        o, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
        pos = torch.arange(s, device="cuda")
        rows = max(1, (1 << 26) // s)
        for b in range(c["b"]):
            for h in range(c["hq"]):
                for r in range(0, s, rows):
                    i = pos[r:r + rows, None]
                    seen = (pos <= i) & ((i - pos <= c["window"]) | (pos < c["sinks"]))
                    a = torch.where(seen, q[b, h, r:r + rows] @ k[b, h // gq].T / math.sqrt(128.0), -math.inf)
                    a = torch.softmax(a, dim=-1)
                    o[b, h, r:r + rows] = a @ v[b, h // gq]
                    dv[b, h // gq] += a.T @ do[b, h, r:r + rows]
                    da = do[b, h, r:r + rows] @ v[b, h // gq].T
                    da = a * (da - (a * da).sum(-1, keepdim=True)) / math.sqrt(128.0)
                    dq[b, h, r:r + rows] = da @ k[b, h // gq]
                    dk[b, h // gq] += da.T @ q[b, h, r:r + rows]
        return [o, dq, dk, dv]
    if c["kind"] == "pages":
        out = []
        for x in (st["k"].float(), st["ks"], st["v"].float(), st["vs"]):
            y = x.clone()
            y[:, st["dst"].long().cuda()] = x[:, st["src"].long().cuda()]
            out.append(y)
        return out
    if c["kind"] == "append":
        out = []
        cu, lens, table = st["cu_new"].tolist(), st["lens"].tolist(), st["table"].tolist()
        for codes, scales, new in ((st["k"], st["ks"], st["new_k"]), (st["v"], st["vs"], st["new_v"])):
            val, sc = codes.double(), scales.double()
            for i in range(c["n"]):
                x = new[cu[i]:cu[i + 1]].double().transpose(0, 1)                       # [h, t, d]
                first, done = lens[i] - x.shape[1], 0
                while done < x.shape[1]:
                    at = first + done
                    take = min(BLOCK - at % BLOCK, x.shape[1] - done)
                    pg, row, blk = table[i][at // c["page"]], at % c["page"], at % c["page"] // BLOCK
                    part = x[:, done:done + take]
                    want = _exact_scale(part.abs().amax((1, 2)))
                    if at % BLOCK:
                        head = slice(row - at % BLOCK, row)
                        up = torch.maximum(want, sc[pg, :, blk])
                        val[pg, :, head] = _exact_round(val[pg, :, head] * (sc[pg, :, blk] / up)[:, None, None])
                        want = up
                    sc[pg, :, blk] = want
                    val[pg, :, row:row + take] = _exact_round(part / want[:, None, None])
                    done += take
            out += [val, sc]
        return out
    cu, lens = st["cu_q"].tolist(), st["lens"].tolist()
    gq, out = c["hq"] // c["hk"], torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(c["n"]):
        pages = st["table"][i, :-(-lens[i] // c["page"])].long()
        kv = []
        for codes, scales in ((st["k"], st["ks"]), (st["v"], st["vs"])):
            x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
            x = x * scales[pages].double().repeat_interleave(BLOCK, dim=2)[..., None]
            kv.append(x.transpose(0, 1).reshape(c["hk"], -1, c["d"])[:, :lens[i]])
        pos = torch.arange(lens[i], device="cuda")
        for h in range(c["hq"]):
            a = st["q"][cu[i]:cu[i + 1], h].double()
            p = lens[i] - a.shape[0] + torch.arange(a.shape[0], device="cuda")[:, None]
            seen = pos <= p
            if c["window"] >= 0:
                seen = seen & ((p - pos <= c["window"]) | (pos < c["sinks"]))
            a = torch.where(seen, a @ kv[0][h // gq].T / math.sqrt(c["d"]), -math.inf)
            out[cu[i]:cu[i + 1], h] = torch.softmax(a, dim=-1) @ kv[1][h // gq]
    return out
