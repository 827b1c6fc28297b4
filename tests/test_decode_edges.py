"""Generation from a paged key-value cache where it meets its edges: infinite values,
beams that tie, models that are not configured as GPT-2 is, overlapping caches, sizes at
the launches' limits, and the kernel variants that groups of fp32 heads take."""
import itertools
import math

import pytest
import torch

from commefficient_amd.ops import decode

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24  # half a step of fp32
INF, NAN = math.inf, math.nan


def _g(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------- attention
def _cache(dtype, lens, kv_heads, group, dim, page, seed):
    """Random q, k and v caches and tables; pages in a random order."""
    g = _g(seed)
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(sum(need) + 1, generator=g).int()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        table[i, :n] = ids[sum(need[:i]):sum(need[:i + 1])]
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    return rnd(len(lens), kv_heads * group, dim), rnd(len(ids), kv_heads, page, dim), \
        rnd(len(ids), kv_heads, page, dim), table


def _attention(q, kc, vc, table, lens, scale):
    """(out, bound) in 64 bits, every product on its own so that infinities act as IEEE says.

    bound: a score is a sum of ``dim`` exact products in fp32 and a scale, off by at most
    dx = (dim + 2) U scale max sum|q k|; its weight by 2 dx and 32 U for exp2 and the powers' argument,
    the sums of L weights by L U, two 16-bit pieces of a weight by 2^-16 (bf16) and 2^-22 (fp16,
    and 2^-35 where a weight is below 2^-24); one rounding of the result at the end."""
    heads, dim = q.shape[1:]
    kh, page = kc.shape[1:3]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    pieces = {BF: 2.0 ** -16, HF: 2.0 ** -22, FP: 0.0}[q.dtype]
    for i, n in enumerate(lens):
        if n == 0:
            continue
        ids = table[i, :-(-n // page)].long()
        k, v = (c[ids].transpose(1, 2).reshape(-1, kh, dim)[:n].double() for c in (kc, vc))
        for h in range(heads):
            c = h // (heads // kh)
            x = (k[:, c] * q[i, h].double()).sum(1) * scale
            p = torch.softmax(x, 0)
            out[i, h] = (p[:, None] * v[:, c]).sum(0)
            dx = float((k[:, c] * q[i, h].double()).abs().sum(1).max()) * scale * (dim + 2) * U
            size = v[:, c].abs().nan_to_num(0.0, 0.0, 0.0)
            bound[i, h] = (2 * dx + (n + 32) * U + pieces) * (p @ size)
            if q.dtype == HF:
                bound[i, h] += 2.0 ** -35 * size.sum(0)
    return out, bound + out.abs().nan_to_num(0.0, 0.0, 0.0) * (torch.finfo(q.dtype).eps / 2) + 1e-30


def _close(got, want, bound):
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    odd = ~want.isfinite()
    assert torch.equal(got[odd].nan_to_num(0.5), want[odd].nan_to_num(0.5))
    err = torch.where(odd, 0.0, (got - want).abs())
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype,kv_heads,group,dim,page", [
    (BF, 2, 1, 64, 16), (HF, 2, 1, 64, 16), (BF, 1, 4, 128, 8), (HF, 1, 20, 32, 3), (BF, 1, 2, 256, 16),
    (HF, 1, 3, 256, 1), (FP, 1, 1, 64, 16), (FP, 1, 3, 64, 4)])
@pytest.mark.parametrize("device", DEVICES)
def test_attention_infinite_values(device, dtype, kv_heads, group, dim, page):
    """A value that is infinite makes its column infinite whatever its weight, two of opposite
    signs or a NaN make it NaN, and no other column, head or sequence changes."""
    lens = [70, 1, 33, 64, 300]
    q, kc, vc, table = _cache(dtype, lens, kv_heads, group, dim, page, seed=dim + page)
    at = lambda i, t: (table[i, t // page].long(), slice(None), t % page)  # noqa: E731
    for i, t, col, x in ((0, 3, 0, INF), (0, 69, 1, -INF), (0, 5, 2, INF), (0, 6, 2, -INF), (0, 40, dim - 1, NAN),
                         (0, 41, dim - 2, INF), (0, 42, dim - 2, INF), (1, 0, 7, INF), (1, 0, 8, -INF),
                         (3, 63, 5, -INF), (4, 0, 1, INF), (4, 299, 1, INF), (4, 128, dim // 2, NAN),
                         (4, 200, dim // 2 + 1, -INF)):
        page_at, _, off = at(i, t)
        vc[page_at, :, off, col] = x
    q[1] = 0.0
    want, bound = _attention(q, kc, vc, table, lens, dim ** -0.5)
    assert want[1, :, 7].eq(INF).all() and want[0, :, 2].isnan().all()
    out = decode.paged_attention(q.to(device), kc.to(device), vc.to(device), table.to(device),
                                 torch.tensor(lens, dtype=torch.int32, device=device))
    _close(out, want, bound)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("device", DEVICES)
def test_attention_infinite_values_beside_weights_of_all_kinds(device, dtype):
    """Weights that 16 bits hold exactly, that they round up or down, equal ones, and the new
    token's row; a weight of exactly 0 beside an infinite value is NaN, as 0 x inf is."""
    dim, lens = 64, [1, 2, 8, 32, 77, 6]
    q, kc, vc, table = _cache(dtype, lens, 1, 1, dim, 16, seed=9)
    q.zero_()
    q[3:5, 0, 0] = 1.0
    q[5, 0, 1] = 1.0
    for i, n in enumerate(lens):
        for t in range(n):
            vc[table[i, t // 16], 0, t % 16, t % dim] = INF if t % 3 else -INF
    kc[table[5, 0], 0, 2, 1] = -INF  # (no weight, beside column 2's infinity)
    want, bound = _attention(q, kc, vc, table, lens, 0.25)
    assert want[5, 0, 2].isnan() and want[:5, 0, 0].eq(-INF).sum() == 4
    k, v = (torch.stack([c[table[i, (n - 1) // 16], :, (n - 1) % 16] for i, n in enumerate(lens)]) for c in (kc, vc))
    a = [x.to(device) for x in (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))]
    _close(decode.paged_attention(*a, scale=0.25), want, bound)
    _close(decode.paged_attention(*a, scale=0.25, k=k.to(device), v=v.to(device)), want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_attention_infinite_values_of_a_split_sequence_gpu(dtype):
    lens = [9000, 5000]
    q, kc, vc, table = _cache(dtype, lens, 2, 1, 64, 16, seed=3)
    for i, t, col, x in ((0, 8999, 4, INF), (0, 17, 9, -INF), (1, 4000, 4, NAN), (1, 100, 63, INF), (1, 4999, 63, -INF)):
        vc[table[i, t // 16], 1, t % 16, col] = x
    want, bound = _attention(q, kc, vc, table, lens, 0.125)
    out = decode.paged_attention(*(x.cuda() for x in (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))))
    _close(out, want, bound)


# ------------------------------------------------------------------- select
def _select(logits, scores, keep, finished=None, eos=-1):
    """(scores, parents, tokens, least gap between different beams that do not tie) in 64 bits,
    the sums of exponentials exactly rounded."""
    B, J, V = logits.shape
    out, gap = [], INF
    for b in range(B):
        c = []
        for j in range(J):
            s = float(scores[b, j])
            if finished is not None and bool(finished[b, j]):
                c.append((-s, j, eos))
                continue
            x = logits[b, j].double()
            m = float(x.max())
            lse = m + math.log(math.fsum((x - m).exp().tolist()))
            y = s + (x - lse)
            some = torch.nonzero(y >= y.topk(min(V, keep)).values[-1])[:, 0]
            c += [(-float(y[v]), j, int(v)) for v in some]
        c.sort()
        gap = min([gap] + [y[0] - x[0] for x, y in zip(c[:keep], c[1:keep + 1]) if x[1] != y[1] and x[0] != y[0]])
        out.append(c[:keep])
    return [torch.tensor([[f(r) for r in row] for row in out]) for f in (lambda r: -r[0], lambda r: r[1], lambda r: r[2])] \
        + [gap]


def _selects(device, logits, scores, keep, finished=None, eos=-1):
    best, parent, token, gap = _select(logits, scores, keep, finished, eos)
    # two sums of V terms in 64 bits, one after the other at the worst, and the scores' own roundings
    assert gap > (2 * (logits.shape[2] + 64) + 8 * float(scores.abs().max())) * 2.0 ** -53, gap
    got = decode.beam_select(logits.to(device), scores.to(device), keep, eos=eos,
                             finished=None if finished is None else finished.to(device))
    assert got[1].cpu().tolist() == parent.tolist()
    assert got[2].cpu().tolist() == token.tolist()
    # fp32's rounding, and the sums' 2^-24 (5 + 2.25 log V) where no candidates were close
    err = U * best.abs() + U * (5 + 2.25 * math.log(logits.shape[2]))
    assert bool(((got[0].cpu().double() - best).abs() <= err).all())


@pytest.mark.parametrize("dtype,requests,beams,vocab,keep", [
    (FP, 2, 8, 50257, 16), (BF, 3, 4, 50262, 8), (HF, 2, 5, 4099, 5), (FP, 4, 3, 1001, 64), (BF, 1, 16, 33, 32),
    (BF, 33, 8, 16411, 8), (FP, 1, 33, 9001, 40)])
@pytest.mark.parametrize("device", DEVICES)
def test_select_equal_rows_go_by_the_lower_beam(device, dtype, requests, beams, vocab, keep):
    """The same logits at every alignment, with equal scores: each token of the lowest beams first."""
    x = (3 * torch.randn(requests, 1, vocab, generator=_g(vocab))).to(dtype).expand(-1, beams, -1).contiguous()
    s = torch.randn(requests, 1, generator=_g(1)).expand(-1, beams).contiguous()
    _selects(device, x, s, keep)


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("device", DEVICES)
def test_select_beams_closer_than_fp32(device, dtype):
    """Rows whose log-sum-exps differ by 1e-9 to 1e-6, far below what fp32 holds of them, in
    an order that is not the beams'; every seventh row twice."""
    requests, beams, vocab = 4, 8, 20011
    x = (2 * torch.randn(requests, 1, vocab, generator=_g(4))).to(dtype).expand(-1, beams, -1).contiguous()
    order = torch.stack([torch.randperm(beams, generator=_g(i)) for i in range(requests)])
    for b, j in itertools.product(range(requests), range(beams)):
        # e^-9 of a sum of about e^12: some 1e-9 more a token that comes up from e^-25
        x[b, j, 100:10100:7] = -25.0
        x[b, j, 100:100 + 7 * int(order[b, j] // 2) * 3:7] = -9.0 if b < 2 else -5.0
    s = torch.tensor([0.0, -1.5, 0.25, -30.0])[:, None].expand(-1, beams).contiguous()
    _selects(device, x, s, 16)
    _selects(device, x, s, 1)
    _selects(device, x, s, 64)


@pytest.mark.parametrize("scale", [1e-6, 1e5, 1e12, 1e37])
@pytest.mark.parametrize("device", DEVICES)
def test_select_equal_rows_of_any_size(device, scale):
    """Tiny and huge logits, whose sums are those of one term or of all alike."""
    x = (scale * torch.rand(2, 1, 3001, generator=_g(12))).expand(-1, 6, -1).contiguous()
    x[1, 2:4] = x[1, 4:6].flip(1)  # (other rows with the same sum, but for its order)
    x[1, 2:4, 77] = x[1, :1].amax() + 2 * scale
    _selects(device, x, torch.zeros(2, 6), 12)


@pytest.mark.parametrize("device", DEVICES)
def test_select_close_beams_among_thousands_of_ties(device):
    """More candidates at the bound than the lists hold, of beams that all but tie."""
    x = torch.randint(-2, 3, (2, 4, 20011), generator=_g(6)).float()
    x[:, 1] = x[:, 0]
    x[:, 1, 7] = -2.0 - 2.0 ** -10  # the upper beam's sum is the smaller one
    x[:, 0, 7] = -2.0
    x[1, 3] = x[1, 2]
    _selects(device, x, torch.zeros(2, 4), 64)
    _selects(device, x.to(BF), torch.zeros(2, 4), 33)


@pytest.mark.parametrize("device", DEVICES)
def test_select_finished_beams_beside_close_ones(device):
    """Scores of beams at their end lie exactly on, and an fp32 step beside, those of others."""
    x = torch.full((3, 4, 4097), -INF)
    x[:, :, 11] = 0.0  # the one token: log-softmax 0
    x[:, 3, 12] = -20.0
    s = torch.tensor([[-1.0, -1.0, -1.0, -1.0], [-1.0, -1.0 - 2.0 ** -23, -1.0, -1.0 + 2.0 ** -24],
                      [-2.0 ** 20, -2.0 ** 20, -2.0 ** 20 - 0.125, -2.0 ** 20]])
    f = torch.tensor([[False, True, True, False], [True, False, False, False], [False, False, True, False]])
    _selects(device, x, s, 4, f, 11)
    _selects(device, x, s, 2, f, 5)


@pytest.mark.gpu
def test_select_close_beams_captured_gpu():
    """The second look is the replay's, whatever the first call met."""
    x = torch.randn(3, 4, 5003, generator=_g(8))
    s = torch.zeros(3, 4)
    dx, ds = x.cuda(), s.cuda()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = decode.beam_select(dx, ds, 8)
    same = x[:, :1].expand(-1, 4, -1).contiguous()
    for now in (x, same, x, same.flip(0), same):
        dx.copy_(now)
        torch.randn(1 << 14, device="cuda").sum().item()
        graph.replay()
        best, parent, token, _ = _select(now, s, 8)
        assert out[1].cpu().tolist() == parent.tolist() and out[2].cpu().tolist() == token.tolist()
        assert bool(((out[0].cpu().double() - best).abs() <= U * best.abs() + 32 * U).all())


# ------------------------------------------------------------------ replies
def _gpt2(dtype, device, n_embd=64, n_head=2, gain=4.0, **cfg):
    """A random GPT-2 double-heads model with a configuration of its own."""
    from transformers import GPT2Config, GPT2DoubleHeadsModel
    torch.manual_seed(3)
    m = GPT2DoubleHeadsModel(GPT2Config(vocab_size=997, n_positions=64, n_embd=n_embd, n_head=n_head, n_layer=3,
                                        **cfg))
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(gain)
    return m.to(dtype).to(device).eval()


_CONFIGS = [dict(activation_function="relu"), dict(activation_function="gelu"), dict(activation_function="silu"),
            dict(scale_attn_by_inverse_layer_idx=True), dict(scale_attn_weights=False),
            dict(scale_attn_weights=False, scale_attn_by_inverse_layer_idx=True, activation_function="gelu_new"),
            dict(n_inner=96), dict(reorder_and_upcast_attn=True), dict(layer_norm_epsilon=0.5),
            dict(add_cross_attention=True), dict(tie_word_embeddings=False), dict(activation_function="gelu_pytorch_tanh")]


@pytest.mark.parametrize("cfg", _CONFIGS, ids=lambda c: ",".join(c))
@pytest.mark.parametrize("device", DEVICES)
def test_generate_follows_the_configuration(device, cfg):
    """A GPT-2 with another activation, attention scaling, width or norm than the default
    answers as its own whole forward passes do."""
    from commefficient_amd.models.gpt2 import generate
    from test_decode import _search
    m = _gpt2(FP, device, **cfg)
    prompts = [torch.randint(0, 997, (n,), generator=_g(n)).tolist() for n in (7, 1, 18)]
    got = generate(m, prompts, max_new_tokens=5, num_beams=3, page_size=4)
    with torch.no_grad():
        want = [_search(m, p, None, None, 3, 5, None, 1.0) for p in prompts]
    for (a, s), (b, r) in zip(got, want):
        assert a == b and abs(s - r) < 1e-3 * abs(r)


@pytest.mark.gpu
@pytest.mark.parametrize("cfg", [dict(scale_attn_weights=False), dict(scale_attn_by_inverse_layer_idx=True),
                                 dict(activation_function="relu"), {}], ids=lambda c: ",".join(c) or "default")
def test_generate_follows_the_configuration_bf16_gpu(cfg):
    """bf16 models of 64 columns a head, whose prompts the whole-sequence kernel takes where
    it may: scores are those of the fp32 passes of the same tokens, hidden states rounded
    to 2^-8 and logits of up to ~30 to 2^-4."""
    from commefficient_amd.models.gpt2 import generate
    m = _gpt2(BF, "cuda", n_embd=256, n_head=4, gain=2.0, **cfg)
    prompts = [torch.randint(0, 997, (n,), generator=_g(n)).tolist() for n in (7, 1, 18)]
    out = generate(m, prompts, max_new_tokens=6, num_beams=2)
    ref = m.float()
    for p, (tokens, score) in zip(prompts, out):
        with torch.no_grad():
            x = ref.lm_head(ref.transformer(torch.tensor([p + tokens], device="cuda"))[0][0])
        lp = torch.log_softmax(x.double(), 1)[len(p) - 1:-1]
        assert abs(float(lp.gather(1, torch.tensor(tokens, device="cuda")[:, None]).mean()) - score) < 0.25


def test_generate_refuses_before_it_runs(monkeypatch):
    """Tokens outside the vocabulary, heads that single-token attention does not have and other
    types are refused on the host, with nothing run."""
    from commefficient_amd.models import gpt2
    m = _gpt2(FP, "cpu")
    monkeypatch.setattr(gpt2, "PagedKV", None)  # (what a run begins with)
    ok = dict(prompts=[[1, 2], [3]], token_types=[[4, 5], [6]], reply_type=7)
    for bad in (dict(prompts=[[1, 997], [3]]), dict(prompts=[[1, 2], [-1]]), dict(token_types=[[4, 5], [997]]),
                dict(token_types=[[4, -2], [5]]), dict(reply_type=997), dict(reply_type=-1), dict(page_size=0),
                dict(page_size=-4), dict(eos=-1)):
        with pytest.raises(ValueError):
            gpt2.generate(m, **{**ok, **bad})
    for other in (_gpt2(FP, "cpu", n_embd=96, n_head=2), _gpt2(FP, "cpu", n_head=4), m.double()):
        with pytest.raises(ValueError, match="columns"):
            gpt2.generate(other, **ok)


# ------------------------------------------------------------------- driver
def _driver_args(tmp_path, monkeypatch, *extra):
    from commefficient_amd.utils.args import parse_args
    monkeypatch.chdir(tmp_path)
    return parse_args(default_lr=4e-2, argv=[
        "--dataset_name", "PERSONA", "--model", "GPT2DoubleHeads", "--synthetic", "--num_clients", "6", "--num_workers",
        "2", "--local_batch_size", "2", "--mode", "uncompressed", "--local_momentum", "0", "--num_epochs", "1",
        "--max_rounds", "1", "--valid_batch_size", "2", "--num_candidates", "2", "--gpt2_size", "tiny", "--device",
        "cpu", "--replies", "2", *extra], probe_port=False)


def test_replies_come_after_the_checkpoint(tmp_path, monkeypatch):
    """A reply that fails costs neither the checkpoint nor the server's state."""
    from commefficient_amd.train import gpt2 as driver
    args = _driver_args(tmp_path, monkeypatch, "--checkpoint", "--checkpoint_path", str(tmp_path / "ck"))

    def fails(*a):
        raise RuntimeError("no reply")
    monkeypatch.setattr(driver, "sample_replies", fails)
    with pytest.raises(RuntimeError, match="no reply"):
        driver.main(args)
    saved = sorted(p.name for p in tmp_path.glob("ck*"))
    assert saved == ["ckGPT2DoubleHeads.fedstate.pt", "ckGPT2DoubleHeads.pt"]


@pytest.mark.parametrize("extra", [["--num_beams", "33"], ["--num_beams", "0"], ["--max_reply", "0"], ["--replies", "-1"]],
                         ids=" ".join)
def test_reply_arguments_are_checked_when_parsed(extra, tmp_path, monkeypatch):
    with pytest.raises(ValueError, match="--replies"):
        _driver_args(tmp_path, monkeypatch, *extra)


def test_replies_longer_than_the_model_are_refused_before_training(tmp_path, monkeypatch):
    from commefficient_amd.train import gpt2 as driver
    monkeypatch.setattr(driver, "FedModel", None)  # (what training begins with)
    with pytest.raises(ValueError, match="--replies"):
        driver.main(_driver_args(tmp_path, monkeypatch, "--max_reply", "1024"))


# ----------------------------------------------------------------- refusals
def test_caches_that_overlap_themselves_are_not_written():
    """Slots that share memory would be racing stores: refused where a call writes, whatever the
    strides' order; caches with gaps, in any order of their dimensions, are not."""
    z, i = torch.zeros, lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    rows = dict(k=z(3, 2, 32), v=z(3, 2, 32))
    one = dict(q=z(3, 2, 32), table=i(3, 1), lens=i(3))
    buf = torch.zeros(1 << 16)
    bad = [(1, 1, 1, 1), (512, 256, 16, 1), (256, 512, 32, 1), (2048, 31, 64, 1), (32, 1024, 96, 1)]
    good = [(512, 256, 32, 1), (512, 32, 64, 1), (40, 160, 320, 1), (2048, 1024, 96, 1), (32, 4096, 512, 1)]
    for strides in bad + good:
        kc, vc = (buf.as_strided((4, 2, 8, 32), strides, at) for at in (0, 1 << 15))
        calls = [lambda: decode.kv_write(**rows, k_cache=kc, v_cache=vc, slots=torch.arange(3)),
                 lambda: decode.paged_attention(k_cache=kc, v_cache=vc, **one, **rows)]
        for call in calls:
            if strides in bad:
                with pytest.raises(RuntimeError, match="overlaps itself"):
                    call()
            else:
                call()
        decode.paged_attention(k_cache=kc, v_cache=vc, **one)  # (reads only)
    six = dict(parent=torch.zeros(1, 2, dtype=torch.int64), table=i(2, 2), lens=i(2))
    decode.beam_reorder(**six, kv=buf.as_strided((2, 2, 4, 1, 8, 32), (4096, 2048, 512, 7, 40, 1)))
    for strides in ((2048, 1024, 250, 1, 32, 1), (100, 1024, 256, 1, 32, 1), (2048, 1024, 256, 1, 31, 1)):
        with pytest.raises(RuntimeError, match="beam_reorder.*overlaps itself"):
            decode.beam_reorder(**six, kv=buf.as_strided((2, 2, 4, 1, 8, 32), strides))


def test_caches_of_one_head_or_page_take_any_stride_there():
    """A dimension of one element has no step to be wrong."""
    kc, vc = (torch.randn(1 << 12, generator=_g(j)).as_strided((6, 1, 8, 32), (300, 0, 32, 1)) for j in (1, 2))
    k = torch.randn(3, 1, 32)
    decode.kv_write(k, k, kc, vc, torch.tensor([0, 47, 9]))
    assert torch.equal(kc[5, :, 7], k[1]) and torch.equal(vc[1, :, 1], k[2])


def test_select_refuses_rows_whose_places_would_pass_32_bits():
    """The kernels count a row's elements in 32 bits, with room for a workgroup behind its end."""
    most = 2 ** 31 - 2 ** 16
    for beams, vocab in ((1, most + 1), (1, 2 ** 31 - 1), (2, 2 ** 30)):
        with pytest.raises(RuntimeError, match="beams x vocabulary"):
            decode.beam_select(torch.zeros(1, 1, 1)[:0].expand(0, beams, vocab), torch.zeros(0, beams))
    assert decode.beam_select(torch.zeros(1, 1, 1)[:0].expand(0, 1, most), torch.zeros(0, 1))[0].shape == (0, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_of_millions_of_rows_gpu(dtype):
    """2^23 sequences whose tables allow 320 tokens: 8 waves each would pass a launch's 2^32 threads."""
    n, page = 1 << 23, 320
    g = _g(2)
    kc, vc = (torch.randn(5, 1, page, 32, generator=g).to(dtype).cuda() for _ in range(2))
    q = torch.randn(1, 1, 32, generator=g).to(dtype)
    table = torch.arange(5).int().repeat(-(-n // 5))[:n].view(n, 1)
    lens = torch.zeros(n, dtype=torch.int32)
    some = [0, 1, 12345, n // 2, n - 1]
    lens[some] = torch.tensor([320, 1, 77, 129, 300], dtype=torch.int32)
    out = decode.paged_attention(q.cuda().expand(n, 1, 32), kc, vc, table.cuda(), lens.cuda())
    assert int((out != 0).any(2).sum()) == len(some)
    want, bound = _attention(q.expand(len(some), 1, 32), kc.cpu(), vc.cpu(), table[some], lens[some].tolist(), 32 ** -0.5)
    _close(out[some], want, bound)


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("lens", [[1, 33, 64, 17, 0], [65, 1, 256, 200, 97], [257, 600, 12, 333, 480], [5000, 3077]],
                         ids=["1wave", "4waves", "8waves", "split"])
@pytest.mark.parametrize("kv_heads,group,dim,page", [(2, 2, 32, 16), (1, 2, 64, 1), (2, 2, 128, 24), (2, 1, 128, 16),
                                                     (1, 1, 32, 5), (1, 1, 256, 8), (1, 4, 256, 16)])
@pytest.mark.parametrize("device", DEVICES)
def test_attention_fp32_variants(device, kv_heads, group, dim, page, lens, append):
    """Every form that fp32 caches take: groups of one and two heads on the vector units, others on
    the matrix units, each with 1, 4 and 8 waves and split."""
    q, kc, vc, table = _cache(FP, lens, kv_heads, group, dim, page, seed=dim + group)
    want, bound = _attention(q, kc, vc, table, lens, dim ** -0.5)
    kw = {}
    if append:  # the last rows come with the call, the slots hold junk
        last = [(table[i, (n - 1) // page].long(), (n - 1) % page) for i, n in enumerate(lens) if n]
        k, v = (torch.zeros(len(lens), kv_heads, dim) for _ in range(2))
        wk, wv = kc.clone(), vc.clone()
        for i, (p, o) in zip([i for i, n in enumerate(lens) if n], last):
            k[i], v[i] = kc[p, :, o], vc[p, :, o]
            kc[p, :, o], vc[p, :, o] = NAN, INF
        kw = dict(k=k.to(device), v=v.to(device))
    dk, dv = kc.to(device), vc.to(device)
    out = decode.paged_attention(q.to(device), dk, dv, table.to(device),
                                 torch.tensor(lens, dtype=torch.int32, device=device), **kw)
    _close(out, want, bound)
    if append:
        assert torch.equal(dk.cpu(), wk) and torch.equal(dv.cpu(), wv)


@pytest.mark.parametrize("dtype,requests,beams,vocab,keep", [(BF, 2, 16, 20011, 64), (FP, 1, 40, 301, 64),
                                                             (HF, 3, 9, 33333, 48), (BF, 1, 1, 50262, 64)])
@pytest.mark.parametrize("device", DEVICES)
def test_select_many_places(device, dtype, requests, beams, vocab, keep):
    """More candidates than the second kernel holds, most of which the waves' bound lets pass."""
    x = (3 * torch.randn(requests, beams, vocab, generator=_g(keep + vocab))).to(dtype)
    _selects(device, x, torch.randn(requests, beams, generator=_g(2)), keep)
