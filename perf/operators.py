"""The operators around the paged block KV cache, as data: which sizes, which inputs, one pass of
each in plain torch operations and through the framework's entry points, the work a pass cannot
do without, and the results in 64 bits.

A case is a dict of plain values; ``kind`` names the operator:

  pages   ``ops.assign_pages`` and ``ops.release_pages``: the page table, slots and positions of
          a step's new tokens from the requests' lengths, and the step taken back again (a
          draft that was rejected), which leaves the pool as it was
  rope    ``ops.norm_rope_kv_write``: RMSNorm of every query and key head, the position
          rotation, and the K / V rows' write into the page pool
  score   ``ops.token_logprobs``: log probabilities of given tokens, the entropy and the most
          probable alternatives of every logits row
"""
from __future__ import annotations

import math

import torch

own = False

HEADS = ((28, 4), (12, 2))  # query / KV heads of the repository's two layouts
VOCAB = 152064
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _pages(name=None, **kw):
    return _named(dict(dict(kind="pages", requests=16, width=8, rows=0, min_len=1056, max_len=4096, prompts=0,
                            longest=0, page=32, room=1.5), **kw), name)


def _rope(name=None, **kw):
    return _named(dict(dict(kind="rope", batch=16, seq=8, q_heads=28, kv_heads=4, head_dim=128, rotary=128,
                            interleaved=False, norm=True, scaling=1.0, far=4096, page=32, head_major=False,
                            ragged=False, dtype="bf16"), **kw), name)


def _score(name=None, **kw):
    return _named(dict(dict(kind="score", batch=16, rows=8, vocab=VOCAB, given=1, top=5, banned=0.0, dtype="bf16"),
                       **kw), name)


def _named(case, name):
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # a sub-block step of 16 requests with contexts of a generation: the host waits for it
        _pages("pages_step_16x8"),
        # continuous batching: 300 requests, 40 of them new prompts, all tokens in one packed list;
        # the pool is short, so that the last prompts have to wait
        _pages("pages_mixed_300", requests=300, width=0, rows=16384, min_len=1, max_len=3000, prompts=40, longest=517,
               room=0.9),
        # the largest batch: whole 32-token blocks of 2048 requests on small pages
        _pages("pages_block_2048x32", requests=2048, width=32, min_len=0, max_len=9000, page=16),
        # one user, one new token: the smallest call
        _rope("rope_token_1x1", batch=1, seq=1, far=900),
        # a sub-block step of 16 sequences on head-major pages, some with fewer than 8 tokens left
        _rope("rope_step_16x8", head_major=True, ragged=True),
        # callers in fp32: two short prompts of odd length, no norms
        _rope("rope_fp32_2x157", batch=2, seq=157, q_heads=12, kv_heads=2, norm=False, dtype="fp32"),
        # a packed list of tokens: neighbours rotated, half of a head of 96, fp16
        _rope("rope_packed_1x1501", batch=1, seq=1501, q_heads=12, kv_heads=2, head_dim=96, rotary=48,
              interleaved=True, far=30000, page=16, dtype="fp16"),
        # a batch of long prompts at far positions with stretched frequencies: the largest call
        _rope("rope_prompt_4x4096", batch=4, seq=4096, scaling=8.0, far=120000),
        # the alternatives that a user of one request is shown, fp32 logits
        _score("score_token_1", batch=1, rows=1, top=20, dtype="fp32"),
        # a sub-block step's tokens, with their confidence in words of probability and entropy
        _score("score_step_16x8"),
        # multiple choice: five candidates per question, a small vocabulary of odd size, words banned
        _score("score_choices_333", batch=333, rows=1, vocab=32001, given=5, top=8, banned=0.05, dtype="fp16"),
        # likelihood of four texts: every token's log probability, the three best beside it
        _score("score_text_4x512", batch=4, rows=512, top=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "rope", "score"])
    if kind == "pages":
        requests = _log(rng, 1, 2048)
        lo = rng.choice([0, 1, _log(rng, 1, 3000)])
        common = dict(requests=requests, min_len=lo, max_len=lo + _log(rng, 1, 6000), page=rng.choice([16, 32, 64]),
                      room=rng.uniform(0.5, 2.0))
        if rng.random() < 0.5:
            return _pages(width=rng.choice([1, 4, 8, 32]), **common)
        prompts = rng.randint(0, min(requests, 60))
        return _pages(width=0, rows=requests + prompts * 300, prompts=prompts, longest=_log(rng, 2, 500), **common)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "rope":
        hq, hkv = rng.choice(HEADS + ((8, 8), (5, 1)))
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        most = 4 * 4096 * 28 * 128 // (hq * dim) // (2 if dtype == "fp32" else 1)
        tokens = _log(rng, 1, min(most, 16384))
        batch = min(tokens, _log(rng, 1, 64))
        return _rope(batch=batch, seq=max(1, tokens // batch), q_heads=hq, kv_heads=hkv, head_dim=dim,
                     rotary=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.choice([False, True]),
                     norm=rng.choice([False, True, True]), scaling=rng.choice([1.0, 4.0]), far=_log(rng, 1, 200000),
                     page=rng.choice([16, 32]), head_major=rng.choice([False, True]), ragged=rng.choice([False, True]),
                     dtype=dtype)
    vocab = rng.choice([VOCAB, VOCAB, 32001, _log(rng, 50, 260000)])
    rows = min(_log(rng, 1, 2048), 2048 * VOCAB // vocab // (2 if dtype == "fp32" else 1))
    per = rng.choice([1, 1, 8])
    return _score(batch=max(1, rows // per), rows=per, vocab=vocab, given=rng.choice([1, 1, 3]),
                  top=rng.choice([0, 1, 5, 20]), banned=rng.choice([0.0, 0.0, 0.1]), dtype=dtype)


# ---------------------------------------------------------------------------------------
# inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(g, lo, hi, *shape):
    """Whole numbers lo..hi."""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _prepare_pages(case, g):
    n, page = case["requests"], case["page"]
    lens = _ints(g, case["min_len"], case["max_len"], n)
    if case["width"]:  # most requests use the whole width, some end inside it
        new = torch.minimum(_ints(g, 1, 2 * case["width"], n), torch.tensor(case["width"], device="cuda"))
    else:
        new = torch.ones(n, dtype=torch.int32, device="cuda")
        if case["prompts"]:
            at = torch.randperm(n, generator=g, device="cuda")[:case["prompts"]]
            new[at] = _ints(g, 1, case["longest"], case["prompts"])
            lens[at] = 0
    new = new.to(torch.int32)
    have = (lens + page - 1) // page
    need, used = int(((lens + new + page - 1) // page - have).sum()), int(have.sum())
    most = (case["max_len"] + max(case["width"], case["longest"]) + page - 1) // page + 1
    pool = n * most
    count = min(int(need * case["room"]) + 1, pool - used)
    ids = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    first = (torch.cumsum(have, 0) - have)[:, None]
    j = torch.arange(most, device="cuda")[None]
    table = torch.where(j < have[:, None], ids[(first + j).clamp(max=pool - 1)], 0).to(torch.int32)
    free_all = torch.zeros(pool + 1, dtype=torch.int32, device="cuda")  # the last one takes what goes nowhere
    free_all[:count] = ids[used:used + count]
    return {"new": new, "lens": lens, "table": table, "free_all": free_all, "free": free_all[:pool],
            "count": torch.full((1,), count, dtype=torch.int32, device="cuda")}


def _frequencies(rotary, base, scaling):
    """f_i = base^(-2 i / R), the slow ones divided by `scaling` (a ramp between)."""
    f = 1.0 / base ** (torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    if scaling != 1.0:
        turns = 4096 * f / (2 * math.pi)  # over the length that the model was trained on
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / scaling * (1.0 - keep)
    return f.float().cuda()


def _prepare_rope(case, g):
    b, s, hkv, d, page = case["batch"], case["seq"], case["kv_heads"], case["head_dim"], case["page"]
    dt = DTYPES[case["dtype"]]
    hq = case["q_heads"]
    # the projections' output, one row of q, k and v heads per token
    x = torch.randn(b, s, hq + 2 * hkv, d, generator=g, device="cuda")
    x = (x * torch.rand(1, 1, hq + 2 * hkv, 1, generator=g, device="cuda").add(0.2).mul(3.0)).to(dt)
    start = _ints(g, 0, case["far"], b, 1).long()
    t = torch.arange(s, device="cuda")[None]
    pages = (b * s + page - 1) // page + 3
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:b * s].view(b, s)
    if case["ragged"]:  # rows behind a sequence's last token have no slot
        slots = torch.where(t < _ints(g, (s + 1) // 2, s, b, 1), slots, -1)
    st = {"q": x[:, :, :hq], "k": x[:, :, hq:hq + hkv], "v": x[:, :, hq + hkv:], "slots": slots,
          "positions": (start + t).to(torch.int32), "qw": None, "kw": None}
    if case["norm"]:
        st["qw"] = torch.rand(d, generator=g, device="cuda").add(0.5).to(dt)
        st["kw"] = torch.rand(d, generator=g, device="cuda").add(0.5).to(dt)
    st["freq"] = _frequencies(case["rotary"], 1e6, case["scaling"])
    st["scale"] = 1.0 if case["scaling"] == 1.0 else 0.1 * math.log(case["scaling"]) + 1.0
    for name in ("k", "v"):
        # one page more than the pool has: rows without a slot go there in the plain form
        if case["head_major"]:
            all_ = torch.randn(pages + 1, hkv, page, d, generator=g, device="cuda").to(dt).transpose(1, 2)
        else:
            all_ = torch.randn(pages + 1, page, hkv, d, generator=g, device="cuda").to(dt)
        st[name + "_all"], st[name + "_pool"] = all_, all_[:pages]
    return st


def _prepare_score(case, g):
    shape = (case["batch"], case["rows"], case["vocab"])
    x = torch.randn(*shape, generator=g, device="cuda").mul_(2.0)
    # half of the rows have a word that stands out
    word = torch.randint(0, shape[2], (*shape[:2], 1), generator=g, device="cuda")
    lift = torch.rand(*shape[:2], 1, generator=g, device="cuda").mul_(24.0).sub_(12.0).clamp_(min=0.0)
    x.scatter_add_(2, word, lift)
    if case["banned"]:
        x.masked_fill_(torch.rand(shape[2], generator=g, device="cuda") < case["banned"], -math.inf)
    given = torch.randint(0, shape[2], (*shape[:2], case["given"]), generator=g, device="cuda")
    given[..., :1] = torch.where(lift > 0, word, given[..., :1])
    return {"logits": x.to(DTYPES[case["dtype"]]), "given": given}


def prepare(case, seed):
    g = _gen(seed)
    st = {"pages": _prepare_pages, "rope": _prepare_rope, "score": _prepare_score}[case["kind"]](case, g)
    st["case"] = case
    return st


# ---------------------------------------------------------------------------------------
# plain forms

def _plain_pages(st):
    case, page = st["case"], st["case"]["page"]
    table, lens, free, count = st["table"], st["lens"], st["free"], st["count"]
    most = table.shape[1]
    new = st["new"].long().clamp(min=0)
    old = lens.long()
    have, total = (old + page - 1) // page, (old + new + page - 1) // page
    if case["width"]:
        fits = new <= case["width"]
        b = torch.arange(len(new), device=new.device)[:, None].expand(-1, case["width"])
        t = torch.arange(case["width"], device=new.device)[None].expand(len(new), -1)
        live = t < new[:, None]
    else:
        end = torch.cumsum(new, 0)
        fits = end <= case["rows"]
        r = torch.arange(case["rows"], device=new.device)
        b = torch.searchsorted(end, r, right=True)
        live = b < len(new)
        b = b.clamp(max=len(new) - 1)
        t = r - (end - new)[b]
    asks = (new > 0) & (total <= most) & fits
    need = torch.where(asks, total - have, 0)
    upto = torch.cumsum(need, 0)
    ok = asks & ((need == 0) | (upto <= count))
    # the pages that are handed out, from the free list's end
    j = torch.arange(most, device=new.device)[None]
    nth = (upto - need)[:, None] + j - have[:, None]
    fresh = ok[:, None] & (j >= have[:, None]) & (j < total[:, None])
    table.copy_(torch.where(fresh, free[(count - 1 - nth).clamp(0, len(free) - 1)], table))
    taken = torch.where(ok, need, 0).sum()
    granted = torch.where(ok, new, 0)
    seqlens = (old + granted).to(torch.int32)
    # rows
    pos = old[b] + t
    at = pos // page
    slots = table[b, at.clamp(max=most - 1)].long() * page + pos % page
    slots = torch.where(live & ok[b], slots, -1)
    positions = torch.where(live, pos, 0).to(torch.int32)
    out = {"slots": slots, "positions": positions, "starts": lens.clone(), "seqlens": seqlens,
           "granted": granted.to(torch.int32)}
    if not case["width"]:
        out["sequences"] = torch.where(live, b, -1).to(torch.int32)
        out["row_starts"] = torch.cat([end.new_zeros(1), end]).to(torch.int32)
    count.sub_(taken)
    lens.copy_(seqlens)
    # and back: pages behind the kept lengths, last ones first
    keep = torch.minimum(out["starts"].clamp(min=0), lens).long()
    have, kept = (lens.long() + page - 1) // page, (keep + page - 1) // page
    back = have - kept
    every = torch.cumsum(back, 0)
    nth = (every - back)[:, None] + j - kept[:, None]
    gone = (j >= kept[:, None]) & (j < have[:, None])
    to = torch.where(gone, count + every[-1] - 1 - nth, len(free))
    st["free_all"].scatter_(0, to.view(-1), table.view(-1))
    count.add_(every[-1])
    lens.copy_(keep)
    return out


def _rotate(x, cos, sin, rotary, interleaved):
    part = x[..., :rotary]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., :rotary // 2], part[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _plain_rope(st):
    case = st["case"]
    angle = st["positions"].double()[..., None] * st["freq"].double()
    cos, sin = ((f(angle) * st["scale"]).float()[:, :, None] for f in (torch.cos, torch.sin))

    def turned(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
        return _rotate(y, cos, sin, case["rotary"], case["interleaved"]).to(x.dtype)

    q, k = turned(st["q"], st["qw"]), turned(st["k"], st["kw"])
    pages = st["k_pool"].shape[0]
    slots = torch.where(st["slots"] < 0, pages * case["page"], st["slots"])
    page, at = slots // case["page"], slots % case["page"]
    st["k_all"][page, at] = k
    st["v_all"][page, at] = st["v"]
    return q


def _plain_score(st):
    x, top = st["logits"].float(), st["case"]["top"]
    m = x.max(-1, keepdim=True).values
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = torch.log(total)
    # a banned word's -inf times its probability of 0 counts as 0
    inner = torch.where(e > 0, e * (x - m), 0.0).sum(-1)
    out = {"logprobs": x.gather(-1, st["given"]) - m - lse, "entropy": lse[..., 0] - inner / total[..., 0]}
    if top:
        # one key per word, larger for larger logits and, of equal ones, for lower indices
        bits = (x + 0.0).view(torch.int32).long()
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        keys = bits * 2 ** 20 + (2 ** 20 - 1 - torch.arange(x.shape[-1], device=x.device))
        keys = torch.topk(keys, top, -1).values
        out["top_tokens"] = 2 ** 20 - 1 - keys % 2 ** 20
        out["top_logprobs"] = x.gather(-1, out["top_tokens"]) - m - lse
    return out


def run(state):
    case = state["case"]
    if own:
        from fast_v2_amd import ops
    if case["kind"] == "pages":
        if own:
            pool = (state["lens"], state["table"], state["free"], state["count"], case["page"])
            rows = ops.assign_pages(state["new"], *pool, width=case["width"], rows=case["rows"])
            ops.release_pages(rows.starts, *pool)
            out = {"slots": rows.slots, "positions": rows.positions, "starts": rows.starts, "seqlens": rows.seqlens,
                   "granted": rows.granted}
            if not case["width"]:
                out["sequences"], out["row_starts"] = rows.sequences, rows.row_starts
        else:
            out = _plain_pages(state)
        out.update(table=state["table"], free=state["free"], count=state["count"], lens=state["lens"])
        return out
    if case["kind"] == "rope":
        if own:
            q = ops.norm_rope_kv_write(state["q"], state["k"], state["v"], state["positions"], state["freq"],
                                       q_weight=state["qw"], k_weight=state["kw"], eps=1e-6,
                                       k_cache=state["k_pool"], v_cache=state["v_pool"], slots=state["slots"],
                                       interleaved=case["interleaved"], rope_scale=state["scale"])
        else:
            q = _plain_rope(state)
        return {"q": q, "k_pool": state["k_pool"], "v_pool": state["v_pool"]}
    if own:
        s = ops.token_logprobs(state["logits"], state["given"], top_k=case["top"])
        out = {"logprobs": s.logprobs, "entropy": s.entropy}
        if case["top"]:
            out["top_tokens"], out["top_logprobs"] = s.top_tokens, s.top_logprobs
        return out
    return _plain_score(state)


# ---------------------------------------------------------------------------------------
# work and results in 64 bits

def work(case):
    """Bytes with every input read and every output written once; operations as multiplications,
    additions, comparisons and exponentials."""
    elt = 4 if case.get("dtype") == "fp32" else 2
    if case["kind"] == "pages":
        n, page = case["requests"], case["page"]
        rows = case["rows"] or n * case["width"]
        pages = n + rows // page  # table entries looked up, of which the new ones are handed out and taken back
        per_row = 12 if case["width"] else 16
        return {"bytes": n * 4 * 9 + rows * per_row + pages * 4 * 3, "flops": rows * 4 + n * 16}
    if case["kind"] == "rope":
        tokens, hq, hkv, d = case["batch"] * case["seq"], case["q_heads"], case["kv_heads"], case["head_dim"]
        moved = tokens * (hq + 2 * hkv) * d * 2 * elt
        return {"bytes": moved + tokens * 12, "flops": tokens * (hq + hkv) * (4 * d * case["norm"] + 3 * case["rotary"])}
    n = case["batch"] * case["rows"]
    return {"bytes": n * (case["vocab"] * elt + case["given"] * 12 + 4 + case["top"] * 12),
            "flops": n * case["vocab"] * 6}


def exact(case, seed):
    if case["kind"] == "pages":
        return None  # whole numbers throughout
    st = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, st)
    return _exact_score(case, st)


def _exact_rope(case, st):
    """Each pair of dimensions as a complex number, turned by exp(i position f)."""
    half = case["rotary"] // 2
    turn = torch.polar(torch.full_like(st["positions"], st["scale"], dtype=torch.float64)[..., None],
                       st["positions"].double()[..., None] * st["freq"].double())[:, :, None]
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    out = []
    for x, w in ((st["q"], st["qw"]), (st["k"], st["kw"])):
        y = x.double()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / case["head_dim"] + 1e-6).sqrt() * w.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    pools = []
    live = st["slots"] >= 0
    at = st["slots"][live]
    for pool, rows in ((st["k_pool"], out[1]), (st["v_pool"], st["v"].double())):
        p = pool.double().contiguous()
        p.view(-1, *p.shape[2:])[at] = rows[live]
        pools.append(p)
    return {"q": out[0], "k_pool": pools[0], "v_pool": pools[1]}


def _exact_score(case, st):
    parts = []
    x, given = st["logits"].flatten(0, 1), st["given"].flatten(0, 1)
    for r in range(0, x.shape[0], 128):
        y = x[r:r + 128].double()
        p = (y - y.amax(-1, keepdim=True)).exp()
        lse = p.sum(-1, keepdim=True).log() + y.amax(-1, keepdim=True)
        logp = y - lse
        entropy = -(logp.exp() * logp.clamp(min=-1e4)).sum(-1)
        order = torch.sort(y, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        parts.append((logp.gather(-1, given[r:r + 128]), entropy, order, logp.gather(-1, order)))
    lead = (case["batch"], case["rows"])
    logprobs, entropy, tokens, best = (torch.cat(p).view(*lead, *p[0].shape[1:]) for p in zip(*parts))
    out = {"logprobs": logprobs, "entropy": entropy}
    if case["top"]:
        out["top_tokens"], out["top_logprobs"] = tokens, best
    return out
