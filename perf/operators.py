"""The operators that let a GPT-2 answer from a paged key-value cache, as measured cases.

Five operators (``commefficient_amd/ops/decode.py``), each with its plain form in elementary
torch operations, its definition in 64 bits and its cases:

* ``kv_extend``: block tables and slot maps from request lengths;
* ``kv_write``: the keys and values of new tokens into their slots;
* ``paged_attention``: one new token a sequence against its pages;
* ``beam_select``: the best continuations over beams and vocabulary;
* ``beam_reorder``: tables and part-filled pages after the beams changed places.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one reply of a small GPT-2: 12 heads of 64 over a short dialogue, the new token's row
        # appended by the same call; bound by latency
        dict(name="attend_reply", op="attend", type="bf16", seqs=1, empty=0, kv_heads=12, group=1,
             head=64, page=16, longest=300, append=True, token_major=False),
        # a batch of 16 dialogues with 4 beams each, ragged up to GPT-2's 1,024 positions
        dict(name="attend_beams", op="attend", type="bf16", seqs=64, empty=0, kv_heads=12, group=1,
             head=64, page=16, longest=1024, append=True, token_major=False),
        # few long contexts with shared key heads: the cache's length is split and joined
        dict(name="attend_long", op="attend", type="bf16", seqs=8, empty=0, kv_heads=8, group=4,
             head=128, page=64, longest=65536, append=False, token_major=False),
        # a model kept in fp32, an odd batch with empty rows, one token a page
        dict(name="attend_fp32", op="attend", type="fp32", seqs=33, empty=3, kv_heads=12, group=1,
             head=64, page=1, longest=777, append=True, token_major=False),
        # one dialogue's beams over GPT-2's vocabulary and its five special tokens
        dict(name="select_reply", op="select", type="bf16", requests=1, beams=4, vocab=50262, keep=4,
             finished=False),
        # a batch of dialogues, twice as many candidates as beams, some beams at their end
        dict(name="select_batch", op="select", type="bf16", requests=64, beams=8, vocab=50262,
             keep=16, finished=True),
        # the states of one dialogue's beams over 12 layers
        dict(name="reorder_reply", op="reorder", type="bf16", requests=1, beams=4, layers=12,
             kv_heads=12, head=64, page=16, longest=300),
        # a batch of dialogues' beams over 12 layers
        dict(name="reorder_batch", op="reorder", type="bf16", requests=64, beams=8, layers=12,
             kv_heads=12, head=64, page=16, longest=500),
        # sixteen prompts enter an empty cache
        dict(name="extend_prompts", op="extend", seqs=16, page=16, longest=500, step=False),
        # one more token for every sequence of a large batch
        dict(name="extend_tokens", op="extend", seqs=4096, page=16, longest=1024, step=True),
        # a prompt's rows out of the packed query-key-value product
        dict(name="write_prompt", op="write", type="bf16", rows=300, kv_heads=12, head=64, page=16),
        # a large batch of prompts
        dict(name="write_batch", op="write", type="bf16", rows=65536, kv_heads=8, head=128, page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "attend", "select", "select", "reorder", "extend", "write"))
    ty = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    page = rng.choice((1, 8, 16, 16, 24, 32, 64, 128))
    head = rng.choice((32, 64, 64, 128, 256))
    if op == "attend":
        c = dict(op=op, type=ty, seqs=_log(rng, 1, 256), empty=0, kv_heads=rng.choice((1, 2, 3, 8, 12, 16)),
                 group=rng.choice((1, 1, 2, 4, 7, 8, 16, 20)), head=head, page=page, longest=_log(rng, 1, 65536),
                 append=rng.random() < 0.6, token_major=rng.random() < 0.25)
        c["empty"] = rng.randrange(0, 1 + c["seqs"] // 8)
        # no more than the largest listed case reads, and than its plain form widens
        most = 8 * 65536 * 8 * 128
        while c["seqs"] * c["longest"] * c["kv_heads"] * c["head"] * SIZE[ty] > 2 * most or \
                c["seqs"] * c["longest"] * c["kv_heads"] * c["group"] > 8 * 65536 * 32:
            c["longest"] = max(1, c["longest"] * 2 // 3)
        return c
    if op == "select":
        beams = rng.choice((1, 2, 3, 4, 5, 8, 16))
        c = dict(op=op, type=ty, requests=_log(rng, 1, 64), beams=beams, vocab=_log(rng, 100, 262144),
                 keep=beams * rng.choice((1, 2)), finished=rng.random() < 0.5)
        while c["requests"] * beams * c["vocab"] > 64 * 8 * 50262:
            c["requests"] = max(1, c["requests"] * 2 // 3)
        return c
    if op == "reorder":
        c = dict(op=op, type=ty, requests=_log(rng, 1, 64), beams=rng.choice((2, 3, 4, 5, 8, 16)),
                 layers=rng.choice((2, 6, 12, 24)), kv_heads=rng.choice((1, 2, 8, 12)), head=head, page=page,
                 longest=_log(rng, 1, 1024))
        while _reorder_pages(c) * page * c["kv_heads"] * head * c["layers"] * 2 * SIZE[ty] > 2.0e9:
            if c["requests"] > 1:
                c["requests"] = c["requests"] * 2 // 3
            else:
                c["longest"], c["layers"] = max(1, c["longest"] * 2 // 3), max(2, c["layers"] * 2 // 3)
        return c
    if op == "extend":
        c = dict(op=op, seqs=_log(rng, 1, 4096), page=page, longest=_log(rng, 1, 4096), step=rng.random() < 0.5)
        while not c["step"] and c["seqs"] * c["longest"] > 1 << 20:
            c["longest"] = max(1, c["longest"] * 2 // 3)
        while c["seqs"] * c["longest"] > 1 << 23:
            c["longest"] = max(1, c["longest"] * 2 // 3)
        return c
    c = dict(op=op, type=ty, rows=_log(rng, 1, 65536), kv_heads=rng.choice((1, 2, 3, 8, 12)), head=head, page=page)
    while c["rows"] * c["kv_heads"] * head * SIZE[ty] > 65536 * 8 * 128 * 2:
        c["rows"] = c["rows"] * 2 // 3
    return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(n, longest, empty=0):
    """n lengths spread evenly from longest / n up to the longest, the first ``empty`` of them 0."""
    v = [max(1, longest * (i + 1) // n) for i in range(n)]
    v[:empty] = [0] * min(empty, n)
    return v


def _shuffled(values, g, dtype=torch.int32):
    t = torch.tensor(values, dtype=dtype, device=DEV)
    return t[torch.randperm(len(values), generator=g, device=DEV)]


def _randn(shape, g, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _reorder_pages(c):
    return c["requests"] * (-(-c["longest"] // c["page"]) + c["beams"])


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    return {"attend": _prepare_attend, "select": _prepare_select, "reorder": _prepare_reorder,
            "extend": _prepare_extend, "write": _prepare_write}[c["op"]](c, g)


def _prepare_attend(c, g):
    ty, n, ps, kh, hd = TYPES[c["type"]], c["seqs"], c["page"], c["kv_heads"], c["head"]
    lens = _shuffled(_lengths(n, c["longest"], c["empty"]), g)
    width = -(-c["longest"] // ps)
    # every sequence's pages lie scattered over the pool, as after hours of serving
    need = (lens.long() + ps - 1) // ps
    pages = sum(-(-x // ps) for x in _lengths(n, c["longest"], c["empty"])) + 3
    ids = torch.randperm(pages - 1, generator=g, device=DEV).int()
    first = need.cumsum(0) - need
    col = torch.arange(width, device=DEV)
    at = (first[:, None] + col).clamp_max(pages - 2)
    table = torch.where(col < need[:, None], ids[at], torch.full_like(at, -1, dtype=torch.int32))
    shape = (pages, ps, kh, hd) if c["token_major"] else (pages, kh, ps, hd)
    kc, vc = _randn(shape, g, ty), _randn(shape, g, ty)
    if c["token_major"]:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    qh = kh * c["group"]
    # rows of the model's packed query-key-value product
    qkv = _randn((n, (qh + 2 * kh) * hd), g, ty)
    q = qkv[:, :qh * hd].view(n, qh, hd)
    k = qkv[:, qh * hd:(qh + kh) * hd].view(n, kh, hd)
    v = qkv[:, (qh + kh) * hd:].view(n, kh, hd)
    return dict(case=c, q=q, k=k if c["append"] else None, v=v if c["append"] else None, kc=kc, vc=vc,
                table=table, lens=lens, longest=c["longest"])


def _prepare_select(c, g):
    b, j, v = c["requests"], c["beams"], c["vocab"]
    # a language model's logits, in rows padded to a multiple of 8 as the tied head writes them
    buf = torch.empty((b, j, -(-v // 8) * 8), dtype=TYPES[c["type"]], device=DEV)
    buf.copy_(3.0 * torch.randn(buf.shape, generator=g, device=DEV))
    logits = buf[..., :v]
    # one token in sixteen is forbidden
    logits.masked_fill_(torch.rand(v, generator=g, device=DEV) < 1 / 16, -math.inf)
    scores = -10.0 - 2.0 * torch.rand((b, j), generator=g, device=DEV)
    finished = None
    if c["finished"]:
        finished = torch.rand((b, j), generator=g, device=DEV) < 0.25
    return dict(case=c, logits=logits, scores=scores, finished=finished, eos=v // 2, keep=c["keep"])


def _prepare_reorder(c, g):
    ty, b, j, ps = TYPES[c["type"]], c["requests"], c["beams"], c["page"]
    per = _shuffled(_lengths(b, c["longest"]), g)
    width = -(-c["longest"] // ps) + 1
    pages = _reorder_pages(c)
    ids = torch.randperm(pages, generator=g, device=DEV).int()
    # full pages are the request's, any of its beams' tables may name them in any order; the
    # part-filled page is the beam's own
    shared = ids[:pages - b * j].view(b, -1)
    tail = ids[pages - b * j:].view(b, j)
    mix = torch.randint(0, shared.shape[1], (b, j, width), generator=g, device=DEV)
    table = torch.gather(shared[:, None].expand(b, j, -1), 2, mix)
    full = (per // ps).long()[:, None, None].expand(b, j, 1)
    table.scatter_(2, full, tail[..., None])
    kv = torch.empty((c["layers"], 2, pages, c["kv_heads"], ps, c["head"]), dtype=ty, device=DEV)
    kv.normal_(generator=g)
    parent = torch.randint(0, j, (b, j), generator=g, device=DEV)
    return dict(case=c, parent=parent, table=table.view(b * j, width).contiguous(),
                lens=per.repeat_interleave(j).contiguous(), kv=kv)


def _prepare_extend(c, g):
    n, ps, longest = c["seqs"], c["page"], c["longest"]
    spread = _lengths(n, longest)
    if c["step"]:
        lens, new = _shuffled(spread, g), torch.ones(n, dtype=torch.int32, device=DEV)
        rows = n
    else:
        lens, new = torch.zeros(n, dtype=torch.int32, device=DEV), _shuffled(spread, g)
        rows = sum(spread)
    width = longest // ps + 1
    pages = sum(-(-(x + 1) // ps) for x in spread) + 7
    ids = torch.randperm(pages, generator=g, device=DEV).int()
    have = (lens.long() + ps - 1) // ps
    first = have.cumsum(0) - have
    col = torch.arange(width, device=DEV)
    table = torch.where(col < have[:, None], ids[(first[:, None] + col).clamp_max(pages - 1)], -1).int()
    return dict(case=c, table=table, lens=lens, new=new, pool=ids, used=have.sum().int().reshape(1), page=ps,
                rows=rows)


def _prepare_write(c, g):
    ty, t, kh, hd, ps = TYPES[c["type"]], c["rows"], c["kv_heads"], c["head"], c["page"]
    pages = -(-t // ps) + 5
    kv = torch.zeros((2, pages, kh, ps, hd), dtype=ty, device=DEV)
    qkv = _randn((t, 3 * kh * hd), g, ty)
    k = qkv[:, kh * hd:2 * kh * hd].view(t, kh, hd)
    v = qkv[:, 2 * kh * hd:].view(t, kh, hd)
    ids = torch.randperm(pages - 1, generator=g, device=DEV)
    row = torch.arange(t, device=DEV)
    slots = ids[row // ps] * ps + row % ps
    slots[torch.rand(t, generator=g, device=DEV) < 1 / 64] = -1  # padding rows
    return dict(case=c, k=k, v=v, kc=kv[0], vc=kv[1], slots=slots)


# -------------------------------------------------------------------- runs
def run(state):
    return _RUNS[state["case"]["op"]](state)


def _run_attend(s):
    if own:
        from commefficient_amd.ops import decode
        out = decode.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], k=s["k"], v=s["v"],
                                     max_len=s["longest"])
        return (out, s["kc"], s["vc"]) if s["k"] is not None else out
    q, kc, vc, lens = s["q"], s["kc"], s["vc"], s["lens"].long()
    n, qh, hd = q.shape
    kh, ps = kc.shape[1], kc.shape[2]
    if s["k"] is not None:
        # the rows of sequences without tokens write the cache's last slot with what it holds
        last = (lens - 1).clamp_min(0)
        page = s["table"].gather(1, (last // ps)[:, None]).long()[:, 0]
        page, off = torch.where(lens > 0, page, kc.shape[0] - 1), torch.where(lens > 0, last % ps, ps - 1)
        some = (lens > 0)[:, None, None]
        kc[page, :, off] = torch.where(some, s["k"], kc[page, :, off])
        vc[page, :, off] = torch.where(some, s["v"], vc[page, :, off])
    pos = torch.arange(s["longest"], device=q.device)
    page = s["table"][:, pos // ps].long().clamp_min(0)
    keys = kc[page, :, pos % ps].permute(0, 2, 1, 3).float()       # [n, kh, longest, hd]
    x = q.float().view(n, kh, qh // kh, hd) @ keys.transpose(2, 3) * (hd ** -0.5)
    del keys
    inside = (pos < lens[:, None])[:, None, None]
    x = x.masked_fill(~inside, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(x - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    values = vc[page, :, pos % ps].permute(0, 2, 1, 3).float()
    out = (p @ values).reshape(n, qh, hd).to(q.dtype)
    return (out, kc, vc) if s["k"] is not None else out


def _run_select(s):
    if own:
        from commefficient_amd.ops import decode
        return decode.beam_select(s["logits"], s["scores"], s["keep"], finished=s["finished"], eos=s["eos"])
    # 64 bits: candidates of different beams may lie closer than fp32 tells apart
    x = s["logits"].double()
    b, j, v = x.shape
    top = x.amax(-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    if s["finished"] is not None:
        ended = torch.full((v,), -math.inf, dtype=x.dtype, device=x.device)
        ended[s["eos"]] = 0.0
        x = torch.where(s["finished"][..., None], ended, x)
    x = (x + s["scores"].double()[..., None]).view(b, j * v)
    x, at = torch.sort(x, dim=1, descending=True, stable=True)
    x, at = x[:, :s["keep"]], at[:, :s["keep"]]
    at = torch.where(x > -math.inf, at, torch.zeros_like(at))
    return x.float(), at // v, at % v


def _run_reorder(s):
    if own:
        from commefficient_amd.ops import decode
        decode.beam_reorder(s["parent"], s["table"], s["lens"], s["kv"])
        return s["table"], s["kv"]
    parent, table, lens, kv = s["parent"], s["table"], s["lens"], s["kv"]
    b, j = parent.shape
    ps = kv.shape[4]
    src = (torch.arange(b, device=parent.device)[:, None] * j + parent).view(-1)
    full, rest = (lens // ps).long(), lens % ps
    there, here = table[src], table.clone()
    col = torch.arange(table.shape[1], device=table.device)
    table.copy_(torch.where(col < full[:, None], there, here))
    at = full.clamp_max(table.shape[1] - 1)[:, None]
    take, put = there.gather(1, at)[:, 0].long(), here.gather(1, at)[:, 0].long()
    some = torch.arange(ps, device=table.device) < rest[:, None]
    kv[:, :, put] = torch.where(some[:, None, :, None], kv[:, :, take], kv[:, :, put])
    return table, kv


def _run_extend(s):
    if own:
        from commefficient_amd.ops import decode
        r = decode.kv_extend(s["table"], s["lens"], s["new"], s["pool"], s["used"], s["page"], s["rows"])
        return (s["table"],) + tuple(r)
    table, lens, new, ps, rows = s["table"], s["lens"].long(), s["new"].long(), s["page"], s["rows"]
    pool, used = s["pool"], s["used"].long()
    n, width = table.shape
    dev = table.device
    end = new.clamp_min(0).cumsum(0)
    start = end - new.clamp_min(0)
    have = (lens + ps - 1) // ps
    fits = (new >= 0) & (lens >= 0) & (lens + new <= width * ps) & (end <= rows)
    need = torch.where(fits, (lens + new + ps - 1) // ps - have, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= pool.numel() - used))
    got = torch.where(served, need, 0)
    first = upto - need + used
    col = torch.arange(width, device=dev)
    fresh = (col >= have[:, None]) & (col < (have + got)[:, None])
    taken = pool[(first[:, None] + col - have[:, None]).clamp(0, pool.numel() - 1)]
    table.copy_(torch.where(fresh, taken, table))
    row = torch.arange(rows, device=dev)
    seq = torch.searchsorted(end, row, right=True)
    real = seq < n
    seq = seq.clamp_max(n - 1)
    pos = lens[seq] + row - start[seq]
    ok = real & served[seq]
    pos = torch.where(ok, pos, 0)
    slots = table[seq, pos // ps].long() * ps + pos % ps
    slots = torch.where(ok, slots, -1)
    seq = torch.where(real, seq, -1)
    starts = torch.cat([start, end[-1:]]).clamp_max(rows)
    lens = torch.where(served, lens + new, lens)
    return (table, slots, pos.int(), seq.int(), starts.int(), lens.int(), (used + got.sum()).int(),
            (~served).sum().int().reshape(1))


def _run_write(s):
    if own:
        from commefficient_amd.ops import decode
        decode.kv_write(s["k"], s["v"], s["kc"], s["vc"], s["slots"])
        return s["kc"], s["vc"]
    kc, vc, slots = s["kc"], s["vc"], s["slots"]
    ps = kc.shape[2]
    # padding rows write the cache's last slot, which no row names, with what it holds
    some = (slots >= 0) & (slots < kc.shape[0] * ps)
    at = torch.where(some, slots, kc.shape[0] * ps - 1)
    page, off, keep = at // ps, at % ps, some[:, None, None]
    kc[page, :, off] = torch.where(keep, s["k"], kc[page, :, off])
    vc[page, :, off] = torch.where(keep, s["v"], vc[page, :, off])
    return kc, vc


_RUNS = {"attend": _run_attend, "select": _run_select, "reorder": _run_reorder, "extend": _run_extend,
         "write": _run_write}


# -------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "attend":
        held = _lengths(c["seqs"], c["longest"], c["empty"])
        row = c["kv_heads"] * c["head"] * SIZE[c["type"]]
        rows = c["seqs"] * c["group"] * 2 + 2 * sum(held)          # q, out, and the cache's keys and values
        rows += 2 * (c["seqs"] - c["empty"]) if c["append"] else 0  # the new rows' stores
        tables = 4 * (sum(-(-x // c["page"]) for x in held) + c["seqs"])
        return {"bytes": rows * row + tables, "flops": 4 * sum(held) * c["kv_heads"] * c["group"] * c["head"]}
    if c["op"] == "select":
        n = c["requests"] * c["beams"]
        return {"bytes": n * c["vocab"] * SIZE[c["type"]] + 4 * n + 20 * c["requests"] * c["keep"],
                "flops": 4 * n * c["vocab"]}
    if c["op"] == "reorder":
        # a beam stays where it is with probability 1 / beams
        moved = [x for x in _lengths(c["requests"], c["longest"]) for _ in range(c["beams"])]
        page_row = c["layers"] * 2 * c["kv_heads"] * c["head"] * SIZE[c["type"]]
        stay = 1 - 1 / c["beams"]
        return {"bytes": stay * sum(2 * (x % c["page"]) * page_row + 8 * (x // c["page"]) for x in moved)
                + 12 * len(moved), "flops": 0}
    if c["op"] == "extend":
        spread = _lengths(c["seqs"], c["longest"])
        rows = c["seqs"] if c["step"] else sum(spread)
        if c["step"]:
            taken = sum(x % c["page"] == 0 for x in spread)
        else:
            taken = sum(-(-x // c["page"]) for x in spread)
        return {"bytes": 16 * c["seqs"] + 16 * rows + 8 * taken + (4 * rows if c["step"] else 0), "flops": 0}
    row = c["kv_heads"] * c["head"] * SIZE[c["type"]]
    return {"bytes": c["rows"] * (4 * row + 8), "flops": 0}


# ------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "select": _exact_select}.get(case["op"], _exact_moves)(s)


def _exact_moves(s):
    return None  # whole numbers and copies: the plain form's values are the only ones


def _exact_attend(s):
    q, lens, table = s["q"].double(), s["lens"].tolist(), s["table"]
    n, qh, hd = q.shape
    kh, ps = s["kc"].shape[1], s["kc"].shape[2]
    out = torch.zeros_like(q)
    for i, length in enumerate(lens):
        if length == 0:
            continue
        pages = table[i, :(length + ps - 1) // ps].long()
        k, v = (c[pages].transpose(1, 2).reshape(-1, kh, hd)[:length].double() for c in (s["kc"], s["vc"]))
        if s["k"] is not None:
            k[length - 1], v[length - 1] = s["k"][i].double(), s["v"][i].double()
        for h in range(kh):
            rows = q[i, h * (qh // kh):(h + 1) * (qh // kh)]
            w = torch.softmax(torch.mm(rows, k[:, h].t()) / math.sqrt(hd), dim=1)
            out[i, h * (qh // kh):(h + 1) * (qh // kh)] = torch.mm(w, v[:, h])
    return (out, None, None) if s["k"] is not None else out


def _exact_select(s):
    x, scores, ended = s["logits"], s["scores"].double(), s["finished"]
    b, j, v = x.shape
    best, frm, tok = [], [], []
    for i in range(b):
        lp = torch.log_softmax(x[i].double(), dim=1) + scores[i][:, None]
        if ended is not None:
            lp[ended[i]] = -math.inf
            lp[:, s["eos"]] = torch.where(ended[i], scores[i], lp[:, s["eos"]])
        flat = lp.reshape(-1)
        least = torch.topk(flat, min(s["keep"], flat.numel())).values[-1]
        at = torch.nonzero((flat >= least) & (flat > -math.inf))[:, 0]
        order = sorted(zip((-flat[at]).tolist(), at.tolist()))[:s["keep"]]
        order += [(math.inf, 0)] * (s["keep"] - len(order))
        best.append([-a for a, _ in order])
        frm.append([k // v for _, k in order])
        tok.append([k % v for _, k in order])
    return (torch.tensor(best, dtype=torch.float64, device=x.device), torch.tensor(frm, device=x.device),
            torch.tensor(tok, device=x.device))
