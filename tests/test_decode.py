"""Generation from a paged key-value cache (ops/decode.py, csrc/kvcache.hip,
paged_attention.hip, beam.hip, models/gpt2.py generate).

Every operator on CPU (plain C++ loops) and GPU (HIP kernels) against a plain
64-bit PyTorch form, at the sizes, strides and masks where it can go wrong;
their refusals; the operators together as captured steps and as GPT-2 replies.
"""
import itertools
import math

import pytest
import torch

from commefficient_amd.models.gpt2 import build_double_heads, generate
from commefficient_amd.ops import decode

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24  # half a step of fp32
INF, NAN = math.inf, math.nan


def _g(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------- extend
def _extend_oracle(table, lens, new, pool, used, page, rows):
    """kv_extend sequence by sequence."""
    table, lens = table.clone(), lens.tolist()
    slots, pos, seq, start = [-1] * rows, [0] * rows, [-1] * rows, []
    row = upto = got = missed = 0
    avail = max(0, pool.numel() - used) if used >= 0 else 0
    out = []
    for i, (n, e) in enumerate(zip(lens, new.tolist())):
        add = max(e, 0)
        start.append(min(row, rows))
        need = 0
        fits = e >= 0 and n >= 0 and row + add <= rows and n + e <= table.shape[1] * page
        if fits:
            need = -(-(n + e) // page) - -(-n // page)
        upto += need
        ok = fits and (need == 0 or upto <= avail)
        if ok:
            for c in range(need):
                table[i, -(-n // page) + c] = pool[used + upto - need + c]
            got += need
        missed += not ok
        for r in range(row, min(row + add, rows)):
            seq[r] = i
            if ok:
                pos[r] = n + r - row
                slots[r] = int(table[i, pos[r] // page]) * page + pos[r] % page
        out.append(n + e if ok else n)
        row += add
    start.append(min(row, rows))
    return table, slots, pos, seq, start, out, used + got, missed


def _extend_case(name):
    g = _g(hash_of(name))
    if name == "none":
        return torch.full((0, 4), -1), [], [], 8, 0, 4, 0
    if name == "prompt":
        return torch.full((1, 3), -1), [0], [33], 8, 1, 16, 33
    if name == "mixed":  # inside a page, onto a page's end, past it, nothing, empty
        return torch.full((6, 4), 5), [3, 4, 7, 8, 0, 1], [1, 4, 2, 0, 9, 15], 64, 7, 4, 40
    if name == "refused":  # negative counts and lengths, a short table row, too few rows
        return torch.full((6, 2), 9), [1, -1, 7, 2, 3, 0], [-2, 1, 2, 1, 0, 4], 64, 0, 4, 5
    if name == "exhausted":  # the pool ends inside the third sequence; no page is needed for the last
        return torch.full((5, 4), 3), [0, 4, 4, 4, 1], [8, 1, 9, 1, 2], 6, 2, 4, 21
    if name == "spent":  # more pages taken than the pool has
        return torch.full((2, 4), 3), [1, 4], [2, 1], 3, 7, 4, 3
    if name == "many":
        n = 2500
        lens = torch.randint(0, 40, (n,), generator=g).tolist()
        new = torch.randint(0, 9, (n,), generator=g).tolist()
        return torch.randint(0, 5000, (n, 7), generator=g), lens, new, 4000, 11, 7, sum(new) + 5
    if name == "step":
        n = 1027
        lens = torch.randint(0, 60, (n,), generator=g).tolist()
        return torch.randint(0, 5000, (n, 4), generator=g), lens, [1] * n, 600, 0, 16, n
    if name == "crowd":  # more sequences than one launch plans, the pool's end among them
        n = 9001
        lens = torch.randint(0, 60, (n,), generator=g).tolist()
        return torch.randint(0, 5000, (n, 4), generator=g), lens, torch.randint(-1, 3, (n,), generator=g).tolist(), \
            900, 3, 16, 3 * n
    if name == "row":  # one sequence takes them all
        return torch.full((5000, 3), 4), [0] * 5000, [0] * 4444 + [33] + [0] * 555, 50, 0, 16, 40
    if name == "long":
        return torch.full((3, 3000), -1), [0, 0, 0], [2900, 17, 2999], 9000, 0, 1, 6000
    raise KeyError(name)


def hash_of(name):
    return sum(ord(c) * 131 ** i for i, c in enumerate(name)) % (1 << 30)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", ["none", "prompt", "mixed", "refused", "exhausted", "spent", "many", "step",
                                  "long", "crowd", "row"])
@pytest.mark.parametrize("device", DEVICES)
def test_extend(device, name, in_place):
    table, lens, new, pages, used, page, rows = _extend_case(name)
    lens, new = torch.tensor(lens, dtype=torch.int32), torch.tensor(new, dtype=torch.int32)
    table = table.int()
    pool = torch.randperm(pages, generator=_g(3)).int()
    want = _extend_oracle(table, lens, new, pool, used, page, rows)
    wide = torch.full((table.shape[0], table.shape[1] + 3), 77, dtype=torch.int32, device=device)
    t = wide[:, :table.shape[1]]  # rows further apart than they are wide
    t.copy_(table)
    ln, us = lens.to(device), torch.tensor([used], dtype=torch.int32, device=device)
    r = decode.kv_extend(t, ln, new.to(device), pool.to(device), us, page, rows, in_place=in_place)
    got = (t, r.slots, r.pos, r.seq, r.start, r.lens, r.used, r.missed)
    want = want[:6] + ([want[6]], [want[7]])
    for what, x, y in zip(("table",) + decode.KVExtend._fields, got, want):
        assert x.cpu().tolist() == (y.tolist() if isinstance(y, torch.Tensor) else y), what
    assert bool((wide[:, table.shape[1]:] == 77).all())
    assert r.slots.dtype == torch.int64 and r.pos.dtype == r.start.dtype == torch.int32
    if in_place:
        assert r.lens is ln and r.used is us
    else:
        assert ln.cpu().tolist() == lens.tolist() and int(us) == used


def test_extend_refusals():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    ok = dict(table=i(2, 4), lens=i(2), new=i(2), pool=i(8), used=i(1), page_size=16, rows=4)
    decode.kv_extend(**ok)
    for bad in (dict(table=i(2, 4).long()), dict(table=i(4, 2).t()), dict(table=i(1, 4).expand(2, 4)),
                dict(lens=i(3)), dict(lens=i(4)[::2]), dict(new=i(2).long()), dict(pool=i(2, 4)), dict(used=i(2)),
                dict(page_size=0), dict(page_size=1 << 21), dict(rows=-1), dict(rows=(1 << 30) + 1)):
        with pytest.raises(RuntimeError, match="kv_extend"):
            decode.kv_extend(**{**ok, **bad})


# -------------------------------------------------------------------- write
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,rows,heads,dim,page,layout", [
    (BF, 0, 2, 64, 16, "plain"), (BF, 1, 1, 8, 1, "plain"), (BF, 37, 12, 64, 16, "packed"),
    (HF, 130, 3, 40, 24, "packed"), (FP, 65, 2, 32, 7, "token_major"), (BF, 33, 2, 5, 3, "packed"),
    (FP, 19, 3, 3, 4, "plain"), (BF, 50, 4, 64, 16, "shifted"), (HF, 21, 2, 64, 8, "columns"),
    (BF, 3000, 8, 128, 64, "packed")])
def test_write(device, dtype, rows, heads, dim, page, layout):
    g = _g(rows + dim)
    pages = -(-rows // page) + 3
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    if layout == "packed":
        qkv = rnd(rows, 3 * heads * dim)
        k, v = (qkv[:, j * heads * dim:(j + 1) * heads * dim].view(rows, heads, dim) for j in (1, 2))
    elif layout == "shifted":  # rows that start 2 bytes past a multiple of 16
        qkv = rnd(rows, 2 * heads * dim + 8)
        k = qkv[:, 1:1 + heads * dim].view(rows, heads, dim)
        v = qkv[:, 1 + heads * dim:1 + 2 * heads * dim].view(rows, heads, dim)
    elif layout == "columns":  # no unit stride over the head
        k, v = (rnd(rows, dim, heads).transpose(1, 2) for _ in range(2))
    else:
        k, v = rnd(rows, heads, dim), rnd(rows, heads, dim)
    if layout == "token_major":
        kc, vc = (rnd(pages, page, heads, dim).transpose(1, 2) for _ in range(2))
    else:
        kc, vc = rnd(2, pages, heads, page, dim)
    slots = torch.randperm(pages * page, generator=g)[:rows]
    for at, bad in zip(range(0, rows, 5), itertools.cycle((-1, pages * page, -(1 << 40), 1 << 40))):
        slots[at] = bad
    wk, wv = kc.clone(), vc.clone()
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            wk[s // page, :, s % page] = k[r]
            wv[s // page, :, s % page] = v[r]
    decode.kv_write(k, v, kc, vc, slots.to(device))
    assert torch.equal(kc, wk) and torch.equal(vc, wv)


def test_write_refusals():
    z = torch.zeros
    ok = dict(k=z(3, 2, 4), v=z(3, 2, 4), k_cache=z(5, 2, 8, 4), v_cache=z(5, 2, 8, 4),
              slots=torch.arange(3))
    decode.kv_write(**ok)
    for bad in (dict(k=z(3, 2, 5)), dict(v=z(2, 2, 4)), dict(k=z(3, 2, 4).to(BF)), dict(v_cache=z(5, 2, 8, 5)), dict(v_cache="k_cache"),
                dict(k_cache=z(5, 2, 4, 8).transpose(2, 3)), dict(k_cache=z(1, 2, 8, 4).expand(5, 2, 8, 4)),
                dict(slots=torch.arange(2)), dict(slots=torch.arange(3).int()),
                dict(k=z(3, 2, 4, requires_grad=True)),
                dict(k=z(3, 2, 4).double(), v=z(3, 2, 4).double(), k_cache=z(5, 2, 8, 4).double(),
                     v_cache=z(5, 2, 8, 4).double())):
        if bad.get("v_cache") == "k_cache":
            bad = dict(v_cache=ok["k_cache"])
        with pytest.raises(RuntimeError, match="kv_write"):
            decode.kv_write(**{**ok, **bad})


# ---------------------------------------------------------------- attention
def _pages_for(lens, page, g, spare=2, width=None):
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(sum(need) + spare, generator=g).int()
    table = torch.full((len(lens), width or max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, sum(need) + spare


def _attention_oracle(q, kc, vc, table, lens, scale, k=None, v=None):
    """(out, bound) in 64 bits; k, v stand for the last token.

    bound: a score is a dot product of ``dim`` exact products summed in fp32,
    off by at most dim U sum|q k| scale (and U for the scale): dx.  Its weight
    is then off by 2 dx and a few U for exp, the sums of L weights by L U, and
    the two-piece 16-bit weights by 2^-16 (bf16) or 2^-22 (fp16) of a weight;
    an fp16 weight below 2^-24 keeps 2^-35.  The result is rounded once."""
    n, heads, dim = q.shape
    kh, page = kc.shape[1], kc.shape[2]
    out, bound = torch.zeros(n, heads, dim, dtype=torch.float64), torch.zeros(n, heads, dim, dtype=torch.float64)
    pieces = {BF: 2.0 ** -16, HF: 2.0 ** -22, FP: 0.0}[q.dtype]
    for i, L in enumerate(lens):
        if L <= 0:
            continue
        ids = table[i, :-(-L // page)].long()
        keys, vals = (c[ids].transpose(1, 2).reshape(-1, kh, dim)[:L].double().clone() for c in (kc, vc))
        if k is not None:
            keys[L - 1], vals[L - 1] = k[i].double(), v[i].double()
        for h in range(heads):
            c = h // (heads // kh)
            qh = q[i, h].double()
            x = keys[:, c] @ qh * scale
            p = torch.softmax(x, 0)
            out[i, h] = p @ vals[:, c]
            dx = float(((keys[:, c].abs() @ qh.abs()).max() * scale).abs()) * (dim + 2) * U
            rel = 2 * dx + (L + 32) * U + pieces
            bound[i, h] = rel * (p @ vals[:, c].abs())
            if q.dtype == HF:
                bound[i, h] += 2.0 ** -35 * vals[:, c].abs().sum(0)
    return out, bound + out.abs() * (torch.finfo(q.dtype).eps / 2) + 1e-30


def _attention_case(dtype, lens, kv_heads, group, dim, page, layout="plain", seed=0):
    g = _g(seed + dim)
    n, heads = len(lens), kv_heads * group
    table, pages = _pages_for(lens, page, g)
    shape = (pages, page, kv_heads, dim) if layout == "token_major" else (pages, kv_heads, page, dim)
    kc, vc = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    if layout == "token_major":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    if layout == "packed":
        qkv = torch.randn(n, (heads + 2 * kv_heads) * dim, generator=g).to(dtype)
        q = qkv[:, :heads * dim].view(n, heads, dim)
        k, v = (qkv[:, (heads + j * kv_heads) * dim:(heads + (j + 1) * kv_heads) * dim].view(n, kv_heads, dim)
                for j in (0, 1))
    elif layout == "shifted":
        q, k, v = (torch.randn(n, h * dim + 9, generator=g).to(dtype)[:, 1:1 + h * dim].view(n, h, dim)
                   for h in (heads, kv_heads, kv_heads))
    else:
        q, k, v = (torch.randn(n, h, dim, generator=g).to(dtype) for h in (heads, kv_heads, kv_heads))
    return q, k, v, kc, vc, table


def _on(device, x):
    """x on the device with the strides that it has."""
    if device == "cpu" or x is None:
        return x
    if x.numel() == 0:
        return x.to(device)
    need = 1 + sum((s - 1) * st for s, st in zip(x.shape, x.stride())) + x.storage_offset()
    return x.as_strided((need,), (1,), 0).to(device).as_strided(x.shape, x.stride(), x.storage_offset())


RAGGED = [1, 0, 2, 31, 32, 33, 16, 15, 17, 63, 64, 65, 100, 127, 128, 129]


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("dtype,lens,kv_heads,group,dim,page,layout", [
    (BF, RAGGED, 3, 1, 64, 16, "packed"), (HF, RAGGED, 2, 4, 64, 16, "plain"), (FP, RAGGED, 2, 1, 64, 1, "packed"),
    (BF, RAGGED, 1, 7, 128, 24, "token_major"), (FP, RAGGED, 2, 3, 32, 8, "token_major"),
    (BF, [200, 1, 77], 2, 20, 32, 5, "plain"), (HF, [333, 40], 1, 33, 256, 64, "packed"),
    (BF, [9, 300], 2, 16, 256, 3, "shifted"), (FP, [500, 1], 1, 17, 256, 128, "plain"),
    (FP, [130, 3], 2, 5, 128, 32, "shifted"), (HF, [1000], 1, 1, 32, 2, "plain"), (BF, [777], 12, 1, 64, 16, "packed"),
    (BF, [0], 1, 1, 64, 16, "plain"), (HF, [1], 1, 2, 128, 16, "plain")])
@pytest.mark.parametrize("device", DEVICES)
def test_attention(device, dtype, lens, kv_heads, group, dim, page, layout, append):
    q, k, v, kc, vc, table = _attention_case(dtype, lens, kv_heads, group, dim, page, layout)
    scale = dim ** -0.5
    want, bound = _attention_oracle(q, kc, vc, table, lens, scale, *((k, v) if append else ()))
    # what no sequence holds is NaN and infinite
    held = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for i, n in enumerate(lens):
        for t in range(n - (1 if append else 0)):
            held[table[i, t // page].long(), t % page] = True
    junk = torch.where(torch.arange(dim) % 2 == 0, NAN, INF).to(dtype)
    kc, vc = (torch.where(held[:, None, :, None], c, junk) for c in (kc, vc))
    if layout == "token_major":
        kc, vc = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc))
    wk, wv = kc.clone(), vc.clone()
    if append:
        for i, n in enumerate(lens):
            if n:
                wk[table[i, (n - 1) // page], :, (n - 1) % page] = k[i]
                wv[table[i, (n - 1) // page], :, (n - 1) % page] = v[i]
    dk, dv = _on(device, kc), _on(device, vc)
    wide = torch.full((len(lens), table.shape[1] + 3), 1 << 30, dtype=torch.int32)  # rows further apart
    wide[:, :table.shape[1]] = table
    for hint, t in ((None, table.to(device)), (1, wide.to(device)[:, :table.shape[1]])):
        out = decode.paged_attention(_on(device, q), dk, dv, t,
                                     torch.tensor(lens, dtype=torch.int32, device=device),
                                     k=_on(device, k) if append else None, v=_on(device, v) if append else None,
                                     max_len=hint)
        assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
        err = (out.cpu().double() - want).abs()
        assert bool((err <= bound).all()), (float((err / bound).max()), int((err > bound).sum()))
        assert torch.equal(dk.cpu().nan_to_num(3.0), wk.nan_to_num(3.0))
        assert torch.equal(dv.cpu().nan_to_num(3.0), wv.nan_to_num(3.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,longest,kv_heads,group,dim,page", [
    (BF, 1, 20000, 2, 1, 64, 16), (BF, 3, 9000, 1, 4, 128, 64), (HF, 2, 6001, 1, 8, 64, 1),
    (FP, 2, 5000, 2, 1, 64, 16), (BF, 70, 700, 4, 2, 64, 16), (BF, 300, 260, 2, 1, 32, 8)])
def test_attention_split_gpu(dtype, n, longest, kv_heads, group, dim, page):
    """Long caches and large batches: split and joined, the same with any hint of the
    length, and bit for bit the same from call to call."""
    lens = [max(0, longest * (i + 1) // n - 3 * (i % 4)) for i in range(n)]
    q, k, v, kc, vc, table = _attention_case(dtype, lens, kv_heads, group, dim, page, seed=5)
    want, bound = _attention_oracle(q, kc, vc, table, lens, 0.3, k, v)
    a = [_on("cuda", x) for x in (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))]
    kw = dict(k=k.cuda(), v=v.cuda(), scale=0.3)
    outs = [decode.paged_attention(*a, max_len=h, **kw) for h in (None, longest, 1, 1 << 29)]
    for out in outs:
        err = (out.cpu().double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())
    assert torch.equal(outs[1], decode.paged_attention(*a, max_len=longest, **kw))


@pytest.mark.parametrize("device", DEVICES)
def test_attention_bad_pages(device):
    """A page outside the cache, or a table too short, makes that sequence's rows NaN and
    no other's; the new row is stored where its own page is sound."""
    q, k, v, kc, vc, table = _attention_case(BF, [40, 40, 40, 70, 5], 2, 2, 64, 16)
    table[1, 1] = -1
    table[2, 2] = kc.shape[0]
    lens = torch.tensor([40, 40, 40, 81, -3], dtype=torch.int32)
    table = table[:, :5].contiguous()
    assert table.shape[1] == 5
    want, bound = _attention_oracle(q, kc, vc, table, [40, 0, 0, 0, 0], 0.125, k, v)
    wk = kc.clone()
    for i in (0, 1):
        wk[table[i, 2], :, 7] = k[i]
    dk, dv = kc.to(device), vc.to(device)
    out = decode.paged_attention(q.to(device), dk, dv, table.to(device), lens.to(device), k=k.to(device),
                                 v=v.to(device)).cpu().double()
    assert bool(((out[0] - want[0]).abs() <= bound[0]).all())
    assert bool(out[1:4].isnan().all()) and bool((out[4] == 0).all())
    assert torch.equal(dk.cpu(), wk)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_extremes(device):
    """Scores far apart, infinite ones, and values that are infinite or NaN where the
    sequence does hold them."""
    q, k, v, kc, vc, table = _attention_case(FP, [70, 70, 70, 70], 1, 1, 64, 16)
    q[0] *= 1000.0
    vc[table[1, 2], 0, 3, 5] = INF
    vc[table[2, 0], 0, 1, 7] = NAN
    q[3, 0] = 0.0
    q[3, 0, 0] = 1.0
    kc[table[3], 0, :, 0] = -INF
    kc[table[3, 1], 0, 2, 0] = 2.0  # the one key with a finite score
    lens = torch.full((4,), 70, dtype=torch.int32)
    out = decode.paged_attention(q.to(device), kc.to(device), vc.to(device), table.to(device),
                                 lens.to(device)).cpu().double()
    x = kc[table[0, :5].long(), 0].reshape(-1, 64)[:70].double() @ q[0, 0].double() * 0.125
    top = int(x.argmax())
    assert float(x.max() - x.sort().values[-2]) > 20  # the other 69 weigh under 69 exp(-20) = 1.5e-7
    torch.testing.assert_close(out[0, 0], vc[table[0, top // 16], 0, top % 16].double(), rtol=1e-5, atol=1e-5)
    assert out[1, 0, 5] == INF and out[1].isinf().sum() == 1
    assert bool(out[2, 0, 7].isnan()) and out[2].isnan().sum() == 1
    assert torch.equal(out[3, 0], vc[table[3, 1], 0, 2].double())
    kc[table[3, 1], 0, 2, 0] = -INF  # no score above -inf
    out = decode.paged_attention(q.to(device), kc.to(device), vc.to(device), table.to(device), lens.to(device))
    assert bool((out[3] == 0).all())


def test_attention_refusals():
    z = torch.zeros
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    c = z(5, 2, 8, 64)
    ok = dict(q=z(3, 4, 64), k_cache=c, v_cache=c.clone(), table=i(3, 2), lens=i(3))
    decode.paged_attention(**ok)
    c48 = z(5, 2, 8, 48)
    for bad in (dict(q=z(3, 3, 64)), dict(q=z(2, 4, 64)), dict(q=z(3, 4, 32)), dict(q=z(3, 4, 64).to(BF)),
                dict(q=z(3, 4, 48), k_cache=c48, v_cache=c48.clone()), dict(table=i(3, 2).long()),
                dict(table=i(2, 3).t()), dict(lens=i(2)), dict(lens=i(3).long()), dict(k=z(3, 2, 64)),
                dict(k=z(3, 4, 64), v=z(3, 4, 64)), dict(v_cache=z(5, 2, 4, 64)), dict(q=z(3, 4, 64, requires_grad=True)),
                dict(k_cache=z(5, 2, 64, 8).transpose(2, 3))):
        with pytest.raises(RuntimeError, match="paged_attention"):
            decode.paged_attention(**{**ok, **bad})


# ------------------------------------------------------------------- select
def _select_oracle(logits, scores, keep, finished, eos):
    x, B = logits.double(), logits.shape[0]
    J, V = logits.shape[1:]
    best, parent, token = (torch.zeros(B, keep, dtype=t) for t in (torch.float64, torch.int64, torch.int64))
    best.fill_(-INF)
    gaps = []
    for b in range(B):
        c = []
        for j in range(J):
            s = float(scores[b, j])
            if not math.isfinite(s):
                continue
            if finished is not None and bool(finished[b, j]):
                c.append((-s, j * V + eos))
                continue
            row = x[b, j]
            if bool(row.isnan().any()) or row.max() in (INF, -INF):
                continue
            y = s + (row - torch.logsumexp(row, 0))
            n = min(V, 4 * keep + 64)
            cut = float(y.topk(n).values[-1])
            c += [(-float(y[i]), j * V + int(i)) for i in torch.nonzero((y >= cut) & (y > -INF))[:, 0]]
        c.sort()
        gaps += [b2[0] - a[0] for a, b2 in zip(c[:keep], c[1:keep + 1]) if a[1] // V != b2[1] // V]
        for n, (s, i) in enumerate(c[:keep]):
            best[b, n], parent[b, n], token[b, n] = -s, i // V, i % V
    return best, parent, token, min(gaps, default=1.0)


def _select_case(name):
    """(logits, scores, keep, finished, eos)"""
    g = _g(hash_of(name))
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if name == "one":
        return rnd(1, 1, 1), rnd(1, 1), 1, None, -1
    if name == "few":  # fewer continuations than places
        return rnd(2, 2, 3).to(BF), rnd(2, 2), 16, torch.tensor([[True, False], [True, True]]), 2
    if name == "odd":
        return rnd(3, 4, 1001).to(BF), rnd(3, 4), 4, None, -1
    if name == "wide":
        return rnd(2, 3, 50262).to(HF), rnd(2, 3), 6, None, -1
    if name == "padded":  # rows apart, as the tied head's
        return rnd(2, 4, 50264).to(BF)[..., :50262], rnd(2, 4), 8, None, -1
    if name == "unaligned":
        return rnd(2, 4, 8200).to(BF)[..., 3:8196], rnd(2, 4), 8, None, -1
    if name == "columns":
        return rnd(2, 700, 3).transpose(1, 2), rnd(2, 3), 5, None, -1
    if name == "first":  # a search's first step: one beam's row for all
        s = torch.full((2, 4), -INF)
        s[:, 0] = 0.0
        return rnd(2, 1, 4099).expand(2, 4, 4099), s, 4, None, -1
    if name == "equal":  # nothing but ties: the lowest tokens of the lowest beam
        return torch.zeros(2, 3, 9001), torch.zeros(2, 3), 33, None, -1
    if name == "steps":  # many exact ties among a few values, signed zeros among them
        x = torch.randint(-2, 3, (2, 4, 20011), generator=g).float()
        x[x == 0] = torch.where(torch.rand(int((x == 0).sum()), generator=g) < 0.5, 0.0, -0.0)
        return x.to(BF), torch.zeros(2, 4), 64, None, -1
    if name == "masked":  # rows of the lowest value, of -inf, with NaN, with +inf, and one token left
        x = rnd(6, 2, 5000)
        x[0] = torch.finfo(FP).min
        x[1, 0] = -INF
        x[2, 0, 4999] = NAN
        x[3, 1, 17] = INF
        x[4] = -INF
        x[5] = -INF
        x[5, 1, 4321] = -3.0e38
        return x, rnd(6, 2), 8, None, -1
    if name == "dead":  # scores that are not finite
        s = rnd(3, 3)
        s[0, 1], s[1, 0], s[2] = -INF, NAN, INF
        return rnd(3, 3, 777).to(BF), s, 3, None, -1
    if name == "finished":
        x = rnd(4, 8, 3001).to(BF)
        x[0, 0] = NAN  # a finished beam's logits do not matter
        f = torch.rand(4, 8, generator=g) < 0.5
        f[0, 0] = True
        return x, rnd(4, 8), 16, f, 3000
    if name == "spread":  # logits so far apart that few weights count
        return 40 * rnd(3, 5, 2049), 9 * rnd(3, 5), 10, None, -1
    if name == "sorted":  # the best all in one stretch of the row
        return (torch.arange(30000.) / 1000).expand(2, 2, 30000).contiguous(), rnd(2, 2), 64, None, -1
    if name == "batch":  # enough rows for the bound that the waves share, in steps and in ties
        x = rnd(40, 4, 33001)
        x[::3] = (x[::3] * 2).round() / 2
        x[5, 1] = -INF
        x[5, 1, 77] = 0.0
        x[6, :, 100:] = -INF
        return x.to(BF), rnd(40, 4).mul(8).round() / 8 + torch.arange(4) / 3, 16, None, -1
    if name == "short":  # fewer 16-byte pieces than places
        return rnd(5, 16, 401).to(BF), rnd(5, 16), 64, None, -1
    if name == "huge":
        return rnd(1, 2, 250007), rnd(1, 2), 4, None, -1
    raise KeyError(name)


@pytest.mark.parametrize("name", ["one", "few", "odd", "wide", "padded", "unaligned", "columns", "first", "equal",
                                  "steps", "masked", "dead", "finished", "spread", "sorted", "batch", "short", "huge"])
@pytest.mark.parametrize("device", DEVICES)
def test_select(device, name):
    """Scores are off by fp32's rounding of the result and, on the GPU, by a log of a sum
    whose terms are each off by at most 32 U (exp of an argument of at most 20) and whose
    fp32 partial sums add 32 U: 64 U = 2^-18.  Candidates of different beams are further
    apart than that (or tie exactly), so the choice is the oracle's."""
    logits, scores, keep, finished, eos = _select_case(name)
    best, parent, token, gap = _select_oracle(logits, scores, keep, finished, eos)
    assert gap == 0.0 or gap > 2.0 ** -17, gap
    x = logits.to(device) if name == "columns" else _on(device, logits)
    got = decode.beam_select(x, scores.to(device), keep, finished=None if finished is None else finished.to(device),
                             eos=eos)
    assert got[0].dtype == FP and got[1].dtype == got[2].dtype == torch.int64
    assert got[1].cpu().tolist() == parent.tolist()
    assert got[2].cpu().tolist() == token.tolist()
    s = got[0].cpu().double()
    assert torch.equal(s.isinf(), best.isinf())
    far = torch.where(best.isinf(), 0.0, (s - best).abs())
    assert bool((far <= U * best.abs().nan_to_num(0, 0, 0) + 2.0 ** -18).all()), float(far.max())


def test_select_default_keep_and_refusals():
    x, s = torch.randn(2, 3, 11, generator=_g(1)), torch.zeros(2, 3)
    assert decode.beam_select(x, s)[0].shape == (2, 3)
    assert decode.beam_select(x[:0], s[:0])[1].shape == (0, 3)
    f = torch.zeros(2, 3, dtype=torch.bool)
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(scores=s[:1]), dict(scores=s.double()),
                dict(keep=0), dict(keep=65), dict(finished=f), dict(finished=f, eos=11),
                dict(finished=f.int(), eos=1), dict(finished=f[:, :2], eos=1),
                dict(logits=x.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="beam_select"):
            decode.beam_select(**{**dict(logits=x, scores=s), **bad})


# ------------------------------------------------------------------ reorder
@pytest.mark.parametrize("dtype,requests,beams,layers,heads,page,dim,lens", [
    (BF, 1, 1, 2, 1, 16, 64, [5]), (BF, 3, 4, 2, 2, 16, 64, [5, 16, 47]), (FP, 2, 3, 1, 3, 1, 32, [9, 1]),
    (HF, 4, 8, 3, 2, 8, 40, [0, 7, 8, 23]), (BF, 2, 32, 1, 1, 24, 5, [25, 71]), (BF, 2, 17, 2, 1, 4, 8, [3, 13]),
    (FP, 1, 2, 1, 1, 5, 3, [14])])
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("device", DEVICES)
def test_reorder(device, strided, dtype, requests, beams, layers, heads, page, dim, lens):
    g = _g(beams + page)
    n = requests * beams
    width = max(lens) // page + 2
    pages = n * width
    table = torch.randperm(pages, generator=g).int().view(n, width)
    parent = torch.randint(0, beams, (requests, beams), generator=g)
    if requests > 2:  # all change places in a circle
        parent[2] = torch.arange(beams).roll(1)
    full = torch.tensor(lens, dtype=torch.int32).repeat_interleave(beams)
    kv = torch.randn(layers, 2, pages, heads, page, dim, generator=g).to(dtype)
    want_t, want = table.clone(), kv.clone()
    for i in range(n):
        src, L = i // beams * beams + int(parent.view(-1)[i]), int(full[i])
        want_t[i, :L // page] = table[src, :L // page]
        at, r = L // page, L % page
        want[:, :, table[i, at], :, :r] = kv[:, :, table[src, at], :, :r]
    if strided:
        kv = kv.permute(2, 0, 1, 4, 3, 5).contiguous().permute(1, 2, 0, 4, 3, 5)
    t, c = table.to(device), _on(device, kv)
    if strided:
        t = torch.cat([t, torch.full_like(t, -5)], 1)[:, :width]
    decode.beam_reorder(parent.to(device), t, full.to(device), c)
    assert torch.equal(t.cpu(), want_t)
    assert torch.equal(c.cpu(), want)


@pytest.mark.parametrize("device", DEVICES)
def test_reorder_leaves_what_it_cannot_move(device):
    """Parents that are none of the request's beams, unequal lengths, pages outside the
    cache, and tables that are too short leave the beam as it is."""
    kv = torch.randn(1, 2, 40, 1, 4, 8, generator=_g(1))
    table = torch.arange(24).int().view(8, 3)
    lens = torch.tensor([6, 6, 6, 5, 6, 6, 13, 13], dtype=torch.int32)
    parent = torch.tensor([[-1, 4, 0, 0], [1, 0, 3, 2]])
    table[4, 1] = 40  # request 1: beam 0's part-filled page is outside the cache
    want_t, want = table.clone(), kv.clone()
    want_t[2, :1] = table[0, :1]
    want[:, :, table[2, 1], :, :2] = kv[:, :, table[0, 1], :, :2]
    t, c = table.to(device), kv.to(device)
    decode.beam_reorder(parent.to(device), t, lens.to(device), c)
    assert torch.equal(t.cpu(), want_t)
    assert torch.equal(c.cpu(), want)


def test_reorder_refusals():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    ok = dict(parent=torch.zeros(2, 3, dtype=torch.int64), table=i(6, 4), lens=i(6), kv=torch.zeros(2, 2, 5, 1, 4, 8))
    decode.beam_reorder(**ok)
    for bad in (dict(parent=torch.zeros(2, 2, dtype=torch.int64)), dict(parent=i(2, 3)), dict(table=i(6, 4).long()),
                dict(lens=i(5)), dict(kv=torch.zeros(2, 5, 1, 4, 8)), dict(kv=torch.zeros(2, 3, 5, 1, 4, 8)),
                dict(kv=torch.zeros(2, 2, 5, 1, 4, 8).double()),
                dict(kv=torch.zeros(2, 2, 1, 1, 4, 8).expand(2, 2, 5, 1, 4, 8)),
                dict(parent=torch.zeros(1, 33, dtype=torch.int64), table=i(33, 4), lens=i(33))):
        with pytest.raises(RuntimeError, match="beam_reorder"):
            decode.beam_reorder(**{**ok, **bad})


# ----------------------------------------------------------------- together
class _Steps:
    """A batch's answering steps on one layer whose query, key and value rows are looked
    up by token."""

    def __init__(self, device, requests=3, beams=4, page=4, vocab=97, heads=2, dim=32, longest=64):
        g = _g(11)
        self.J, self.B, self.V = beams, requests, vocab
        self.rows = torch.randn(vocab, 3 * heads * dim, generator=g).to(device)
        self.head = torch.randn(heads * dim, vocab, generator=g).to(device)
        n = requests * beams
        self.cache = decode.PagedKV(1, heads, dim, n, n * (longest // page + 2), page, longest, FP, device)
        self.one = torch.ones(n, dtype=torch.int32, device=device)
        self.dims = (n, heads, dim)
        self.scores = torch.randn(requests, beams, generator=g).to(device)
        self.token = torch.randint(0, vocab, (n,), generator=g).to(device)
        self.parent = torch.randint(0, beams, (requests, beams), generator=g).to(device)
        self.history = self.token.cpu().view(requests, beams, 1).clone()

    def step(self):
        n, heads, dim = self.dims
        self.cache.extend(self.one, n)
        q, k, v = (t.view(n, heads, dim) for t in self.rows[self.token].split(heads * dim, dim=1))
        y = self.cache.attend(0, q, k, v).view(n, -1)
        s, p, t = decode.beam_select((y @ self.head).view(self.B, self.J, self.V), self.scores)
        self.cache.reorder(p)
        self.scores.copy_(s)
        self.parent.copy_(p)
        self.token.copy_(t.view(-1))
        self.y = y

    def expect(self):
        """The step's scores from every beam's whole history, in 64 bits."""
        n, heads, dim = self.dims
        out = []
        for b, j in itertools.product(range(self.B), range(self.J)):
            x = self.rows.cpu().double()[self.history[b, j]].view(-1, 3, heads, dim)
            q, k, v = x[-1, 0], x[:, 1], x[:, 2]
            p = torch.softmax(torch.stack([k[:, h] @ q[h] for h in range(heads)]) * dim ** -0.5, 1)
            out.append(torch.cat([p[h] @ v[:, h] for h in range(heads)]))
        return torch.stack(out)


def _run_steps(s, step, steps):
    # 64 terms a sum at most, values of about 1: 2^-24 x 64 x a few of them
    for _ in range(steps):
        before = s.scores.cpu().double().clone()
        y = s.expect()
        step()
        torch.testing.assert_close(s.y.cpu().double(), y, rtol=1e-4, atol=1e-4)
        x = torch.log_softmax((y @ s.head.cpu().double()).view(s.B, s.J, s.V), 2) + before[..., None]
        best = x.view(s.B, -1).topk(s.J)
        torch.testing.assert_close(s.scores.cpu().double(), best.values, rtol=1e-4, atol=1e-3)
        p, t = s.parent.cpu(), s.token.cpu().view(s.B, s.J)
        s.history = torch.cat([s.history.gather(1, p[..., None].expand(-1, -1, s.history.shape[2])), t[..., None]], 2)
    assert int(s.cache.missed) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_inference_mode_and_grad_mode(device):
    """The operators run under inference_mode, and on tensors of it afterwards."""
    with torch.inference_mode():
        s = _Steps(device)
        s.step()
        s.step()
        assert int(s.cache.missed) == 0 and s.cache.lens.cpu().tolist() == [2] * 12
    r = decode.kv_extend(s.cache.table.clone(), s.cache.lens, s.one, s.cache.pool, s.cache.used, 4, 12)
    assert r.lens.cpu().tolist() == [3] * 12 and s.cache.lens.cpu().tolist() == [2] * 12


@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("device", DEVICES)
def test_steps_together(device, page):
    s = _Steps(device, page=page)
    _run_steps(s, s.step, 19)


@pytest.mark.gpu
def test_steps_captured_gpu():
    """A captured step replayed, with eager work and waits between the replays; two graphs of
    different batches live at once."""
    a, b = _Steps("cuda", page=4), _Steps("cuda", requests=2, beams=3, page=8, vocab=301)
    graphs = []
    for s in (a, b):
        keep = {k: v.clone() for k, v in vars(s).items() if isinstance(v, torch.Tensor)}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.step()
        graphs.append(graph)
        s.cache.reset()
        for name in ("scores", "token", "parent"):
            getattr(s, name).copy_(keep[name])
    for _ in range(6):
        for s, graph in zip((a, b), graphs):
            _run_steps(s, graph.replay, 2)
            torch.randn(1 << 16, device="cuda").sum().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,group,dim", [(BF, 16, 256), (FP, 16, 256), (FP, 1, 256), (BF, 1, 64)])
def test_attention_captured_gpu(dtype, group, dim):
    """Replays follow the lengths, tables and rows that they find (the first call of a variant
    may be the captured one)."""
    lens = [70, 33, 5]
    q, k, v, kc, vc, table = _attention_case(dtype, lens, 1, group, dim, 16)
    dev = [_on("cuda", x) for x in (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))]
    kw = dict(k=k.cuda(), v=v.cuda())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = decode.paged_attention(*dev, **kw)
    for now in ([70, 33, 5], [1, 32, 0], [64, 2, 4], [70, 33, 5]):
        dev[0].copy_(torch.randn(q.shape, generator=_g(sum(now))).to(dtype))
        dev[4].copy_(torch.tensor(now, dtype=torch.int32))
        kc, vc = dev[1].cpu(), dev[2].cpu()
        graph.replay()
        torch.randn(1 << 14, device="cuda").sum().item()
        want, bound = _attention_oracle(dev[0].cpu(), kc, vc, table, now, dim ** -0.5, k, v)
        assert bool(((out.cpu().double() - want).abs() <= bound).all())


@pytest.mark.gpu
def test_other_stream_gpu():
    """The operators run on the caller's current stream."""
    lens = [300, 17, 1024]
    q, k, v, kc, vc, table = _attention_case(BF, lens, 4, 1, 64, 16)
    a = [_on("cuda", x) for x in (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))]
    want = decode.paged_attention(*a)
    x, sc = torch.randn(4, 4, 30011, generator=_g(2)).cuda(), torch.zeros(4, 4, device="cuda")
    sel = decode.beam_select(x, sc)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-4
        q2, x2 = a[0] + big[0, 0].to(BF) * 0, x + big[0, 0] * 0  # (produced late, on this stream)
        got = decode.paged_attention(q2, *a[1:])
        sel2 = decode.beam_select(x2, sc)
    side.synchronize()
    if bool(torch.isfinite(big[0, 0])):
        assert torch.equal(got, want)
        assert all(torch.equal(p, r) for p, r in zip(sel, sel2))


# ------------------------------------------------------------------ replies
def _tiny(n_embd, n_head, dtype, device, n_positions=96):
    torch.manual_seed(0)
    m = build_double_heads("gpt2", n_special=5, n_layer=2, n_embd=n_embd, n_head=n_head, n_positions=n_positions)
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(3.0)
    return m.to(dtype).to(device).eval()


def _search(m, prompt, types, reply_type, beams, steps, eos, alpha):
    """Beam search by whole forward passes of the HF module in fp32."""
    live = [(0.0, [], False)]
    dev = m.transformer.wte.weight.device
    for _ in range(steps):
        c = []
        for s, out, end in live:
            if end:
                c.append((s, out, True))
                continue
            ids = torch.tensor([prompt + out], device=dev)
            tt = None if types is None else torch.tensor([types + [reply_type] * len(out)], device=dev)
            x = m.lm_head(m.transformer(input_ids=ids, token_type_ids=tt)[0][0, -1])
            lp = torch.log_softmax(x.double(), 0)
            v, i = lp.topk(beams)
            c += [(s + a, out + [t], t == eos) for a, t in zip(v.tolist(), i.tolist())]
        live = sorted(c, key=lambda r: -r[0])[:beams]
    s, out, end = max(live, key=lambda r: r[0] / len(r[1]) ** alpha)
    return (out[:-1] if end else out), s / len(out) ** alpha


@pytest.mark.parametrize("types,beams,page", [(False, 3, 4), (True, 1, 16), (True, 4, 1)])
@pytest.mark.parametrize("device", DEVICES)
def test_generate_matches_whole_passes(device, types, beams, page):
    m = _tiny(64, 2, FP, device)
    g = _g(5)
    prompts = [torch.randint(0, 50262, (n,), generator=g).tolist() for n in (16, 1, 37, 4)]
    tt = [[50259] * len(p) for p in prompts] if types else None
    with torch.no_grad():
        free = [_search(m, p, tt and tt[i], 50260, beams, 9, None, 1.0) for i, p in enumerate(prompts)]
    kw = dict(max_new_tokens=9, num_beams=beams, token_types=tt, reply_type=50260 if types else None, page_size=page)
    got = generate(m, prompts, **kw)
    for (a, s), (b, r) in zip(got, free):
        assert a == b and abs(s - r) < 1e-3 * abs(r)
    # the same with an end that one of the replies meets
    eos = free[2][0][4]
    with torch.no_grad():
        want = [_search(m, p, tt and tt[i], 50260, beams, 9, eos, 0.7) for i, p in enumerate(prompts)]
    got = generate(m, prompts, eos=eos, length_penalty=0.7, **kw)
    for (a, s), (b, r) in zip(got, want):
        assert a == b and abs(s - r) < 1e-3 * abs(r)


@pytest.mark.gpu
def test_generate_native_bf16_gpu():
    """On the native kernels a reply's score is that of the HF forward of the same tokens:
    bf16 rounds the hidden states to 2^-8 of their size, logits of up to ~30 to 2^-4."""
    m = _tiny(256, 4, BF, "cuda")
    g = _g(6)
    prompts = [torch.randint(0, 50262, (n,), generator=g).tolist() for n in (16, 3, 50)]
    out = generate(m, prompts, max_new_tokens=12, num_beams=4)
    out += generate(m, prompts[1:2], max_new_tokens=12, num_beams=1)
    ref = m.float()
    for p, (tokens, score) in zip(prompts + prompts[1:2], out):
        assert len(tokens) == 12
        with torch.no_grad():
            x = ref.lm_head(ref.transformer(torch.tensor([p + tokens], device="cuda"))[0][0])
        lp = torch.log_softmax(x.double(), 1)[len(p) - 1:-1]
        s = float(lp.gather(1, torch.tensor(tokens, device="cuda")[:, None]).mean())
        assert abs(s - score) < 0.25, (s, score)


def test_generate_refusals():
    m = _tiny(64, 2, FP, "cpu", n_positions=32)
    assert generate(m, []) == []
    for kw in (dict(prompts=[[1], []]), dict(prompts=[[1]], max_new_tokens=0), dict(prompts=[[1]], num_beams=0), dict(prompts=[[1]], num_beams=33),
               dict(prompts=[[1] * 20], max_new_tokens=13), dict(prompts=[[1]], token_types=[[1]]),
               dict(prompts=[[1, 2]], token_types=[[1]], reply_type=1), dict(prompts=[[1]], eos=50262)):
        with pytest.raises(ValueError):
            generate(m, **kw)
    o = build_double_heads("openai-gpt", n_special=0, n_layer=1, n_embd=32, n_head=2)
    for other in (o, torch.nn.Linear(2, 2)):
        with pytest.raises(ValueError, match="GPT-2"):
            generate(other, [[1]])


@pytest.mark.parametrize("dtype,device", [(BF, "cpu"), pytest.param(HF, "cuda", marks=pytest.mark.gpu),
                                          pytest.param(BF, "cuda", marks=pytest.mark.gpu)])
def test_generate_other_types(dtype, device):
    """Models that the native junctions do not cover (fp16, 64 columns) answer too: as many
    tokens as asked for, of the vocabulary, with the score of the HF forward of the same
    tokens (16-bit hidden states: logits of up to ~30 rounded to 2^-4)."""
    m = _tiny(64, 2, dtype, device)
    prompts = [[11, 7000, 42], [50000]]
    for p, (tokens, score) in zip(prompts, generate(m, prompts, max_new_tokens=5, num_beams=2, page_size=2)):
        assert len(tokens) == 5 and all(0 <= t < 50262 for t in tokens)
        with torch.no_grad():
            ref = m.float()
            x = ref.lm_head(ref.transformer(torch.tensor([p + tokens], device=device))[0][0])
            m.to(dtype)
        lp = torch.log_softmax(x.double(), 1)[len(p) - 1:-1]
        s = float(lp.gather(1, torch.tensor(tokens, device=device)[:, None]).mean())
        assert abs(s - score) < 0.25, (s, score)


# ------------------------------------------------------------------- driver
def _driver_args(tmp_path, monkeypatch, extra):
    from commefficient_amd.utils.args import parse_args
    monkeypatch.chdir(tmp_path)
    return parse_args(default_lr=4e-2, argv=[
        "--dataset_name", "PERSONA", "--synthetic", "--num_clients", "6", "--num_workers", "2",
        "--local_batch_size", "2", "--mode", "uncompressed", "--local_momentum", "0", "--num_epochs", "1",
        "--max_rounds", "1", "--valid_batch_size", "2", "--num_candidates", "2", "--replies", "3",
        "--max_reply", "6", "--num_beams", "3"] + extra, probe_port=False)


def _check_replies(printed, n_tokens):
    rows = [eval(x, {"__builtins__": {}}, {"nan": NAN}) for x in printed.splitlines() if x.startswith("{'dialogue'")]
    assert len(rows) == 3
    for r in rows:
        assert len(r["dialogue"]) > 10 and len(r["gold"]) >= 8 and len(r["reply"]) <= 6
        assert all(0 <= t < n_tokens for t in r["reply"]) and r["score"] < 0


def test_driver_prints_replies(tmp_path, monkeypatch, capsys):
    from commefficient_amd.train import gpt2 as driver
    driver.main(_driver_args(tmp_path, monkeypatch, ["--gpt2_size", "tiny", "--device", "cpu"]))
    _check_replies(capsys.readouterr().out, 50262)


def test_driver_refuses_replies_of_openai_gpt(tmp_path, monkeypatch):
    from commefficient_amd.train import gpt2 as driver
    with pytest.raises(ValueError, match="--replies"):
        driver.main(_driver_args(tmp_path, monkeypatch, ["--gpt2_size", "tiny", "--device", "cpu",
                                                         "--model_checkpoint", "openai-gpt"]))


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [[], ["--finetune"]])
def test_driver_prints_replies_native_gpu(extra, tmp_path, monkeypatch, capsys):
    from commefficient_amd.train import gpt2 as driver
    driver.main(_driver_args(tmp_path, monkeypatch, ["--gpt2_size", "mini", "--device", "cuda"] + extra))
    _check_replies(capsys.readouterr().out, 50262)
