"""GPT-2 / OpenAI-GPT double-heads models for PersonaChat-style federated training.

The reference loads ``pytorch_transformers.GPT2DoubleHeadsModel`` (LM head tied
to ``wte`` + multiple-choice head) and adds 5 special tokens
(/root/reference/CommEfficient/gpt2_train.py:4-6,26-32,101-112,262-273), giving
124,444,417 trainable parameters.  Here the same HF ``transformers``
architecture is built from its config with random init (no network, no
pretrained checkpoints in this environment), with SDPA attention so the
attention runs on the ROCm fused kernels.  The training loss matches
gpt2_train.py:88-99 (``lm_coef * lm + mc_coef * mc``).
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import transformer as _tx
from ..ops.decode import PagedKV, beam_select

SPECIAL_TOKENS = ["<bos>", "<eos>", "<speaker1>", "<speaker2>", "<pad>"]
ATTR_TO_SPECIAL_TOKEN = {"bos_token": "<bos>", "eos_token": "<eos>", "pad_token": "<pad>",
                         "additional_special_tokens": ["<speaker1>", "<speaker2>"]}


def build_double_heads(model_checkpoint: str = "gpt2", n_special: int = 5, n_layer=None,
                       n_embd=None, n_head=None, n_positions=None):
    import os
    from transformers import (GPT2Config, GPT2DoubleHeadsModel, OpenAIGPTConfig,
                              OpenAIGPTDoubleHeadsModel)
    is_gpt2 = "gpt2" in model_checkpoint
    if os.path.isdir(model_checkpoint):  # a local HF directory (e.g. --finetune)
        cls = GPT2DoubleHeadsModel if is_gpt2 else OpenAIGPTDoubleHeadsModel
        return cls.from_pretrained(model_checkpoint)
    cfg = GPT2Config() if is_gpt2 else OpenAIGPTConfig()
    for k, v in (("n_layer", n_layer), ("n_embd", n_embd), ("n_head", n_head),
                 ("n_positions", n_positions)):
        if v is not None:
            setattr(cfg, k, v)
    if is_gpt2:  # (HF's OpenAI-GPT has no SDPA attention: it keeps the eager one)
        try:
            cfg._attn_implementation = "sdpa"
        except Exception:
            pass
    if is_gpt2 and cfg.activation_function == "gelu_new":
        # the same tanh-approximation GELU as one fused kernel each way
        # (torch's gelu(approximate="tanh")) instead of HF's ~8 elementwise ops
        cfg.activation_function = "gelu_pytorch_tanh"
    model = (GPT2DoubleHeadsModel if is_gpt2 else OpenAIGPTDoubleHeadsModel)(cfg)
    if n_special:
        model.resize_token_embeddings(cfg.vocab_size + n_special, mean_resizing=False)
    return model


class GPT2DoubleHeads(nn.Module):
    """Registry wrapper so ``--model GPT2DoubleHeads`` works like the CV models."""

    def __init__(self, model_checkpoint="gpt2", **kw):
        super().__init__()
        self.model = build_double_heads(model_checkpoint, **{k: v for k, v in kw.items()
                                                             if k in ("n_layer", "n_embd",
                                                                      "n_head", "n_positions",
                                                                      "n_special")})

    def forward(self, *a, **kw):
        return self.model(*a, **kw)

    def save_pretrained(self, d):
        self.model.save_pretrained(d)

    def generate(self, prompts, **kw):
        return generate(self, prompts, **kw)


def double_heads_loss(model, batch, lm_coef=1.0, mc_coef=1.0):
    """(loss, lm_loss, mc_loss, mc_correct_frac) for one PersonaChat batch
    ``(input_ids[B,C,L], mc_token_ids[B,C], lm_labels[B,C,L], mc_labels[B], token_type_ids[B,C,L])``."""
    input_ids, mc_token_ids, lm_labels, mc_labels, token_type_ids = batch
    m = model.model if isinstance(model, GPT2DoubleHeads) else model
    out = m(input_ids=input_ids, token_type_ids=token_type_ids, mc_token_ids=mc_token_ids)
    lm_logits, mc_logits = out.logits, out.mc_logits
    # shift for next-token prediction; -100 labels are ignored (pad / persona)
    shift_logits = lm_logits[..., :-1, :].contiguous()
    shift_labels = lm_labels[..., 1:].contiguous()
    lm_loss = F.cross_entropy(shift_logits.view(-1, shift_logits.size(-1)).float(),
                              shift_labels.view(-1), ignore_index=-100)
    mc_loss = F.cross_entropy(mc_logits.float(), mc_labels)
    acc = (mc_logits.argmax(dim=-1) == mc_labels).float().mean()
    return lm_coef * lm_loss + mc_coef * mc_loss, lm_loss, mc_loss, acc


# ------------------------------------------------------------- generation
def _blocks(tr, x, attend):
    """ln_f output [rows, H] of GPT-2's blocks on the token rows ``x``, without
    dropout; ``attend(layer, qkv [rows, 3H])`` -> [rows, H].  The junction kernels
    where they cover the model (ops/transformer.py), else torch's and the model's own
    activation."""
    eps = float(tr.config.layer_norm_epsilon)
    if _tx.native_ok(tr, x):
        ln = tr.h[0].ln_1
        h, y = _tx._Impl.resid_ln_fwd(x, None, None, ln.weight, ln.bias, 0.0, 0, eps, True)[:2]
        for i, blk in enumerate(tr.h):
            o = attend(i, _tx._mm(y, blk.attn.c_attn.weight, blk.attn.c_attn.bias))
            p = _tx._mm(o, blk.attn.c_proj.weight)
            h, y = _tx._Impl.resid_ln_fwd(h, p, blk.attn.c_proj.bias, blk.ln_2.weight, blk.ln_2.bias,
                                          0.0, 0, eps, True)[:2]
            f = _tx._Impl.bias_gelu_fwd(_tx._mm(y, blk.mlp.c_fc.weight), blk.mlp.c_fc.bias)
            p = _tx._mm(f, blk.mlp.c_proj.weight)
            ln = tr.h[i + 1].ln_1 if i + 1 < len(tr.h) else tr.ln_f
            h, y = _tx._Impl.resid_ln_fwd(h, p, blk.mlp.c_proj.bias, ln.weight, ln.bias, 0.0, 0, eps, True)[:2]
        return y
    tanh_gelu = tr.config.activation_function in ("gelu_new", "gelu_pytorch_tanh")
    for i, blk in enumerate(tr.h):
        y = F.layer_norm(x, x.shape[-1:], blk.ln_1.weight, blk.ln_1.bias, eps)
        o = attend(i, torch.addmm(blk.attn.c_attn.bias, y, blk.attn.c_attn.weight))
        x = x + torch.addmm(blk.attn.c_proj.bias, o, blk.attn.c_proj.weight)
        y = F.layer_norm(x, x.shape[-1:], blk.ln_2.weight, blk.ln_2.bias, eps)
        f = torch.addmm(blk.mlp.c_fc.bias, y, blk.mlp.c_fc.weight)
        f = F.gelu(f, approximate="tanh") if tanh_gelu else blk.mlp.act(f)
        x = x + torch.addmm(blk.mlp.c_proj.bias, f, blk.mlp.c_proj.weight)
    return F.layer_norm(x, x.shape[-1:], tr.ln_f.weight, tr.ln_f.bias, eps)


def can_generate(cfg):
    """Whether ``generate`` covers models of this configuration: GPT-2 with heads of a
    width that single-token attention has (ops/decode.py)."""
    return (getattr(cfg, "model_type", "") == "gpt2" and cfg.n_embd % cfg.n_head == 0
            and cfg.n_embd // cfg.n_head in (32, 64, 128, 256))


def _attention_scale(cfg, layer):
    """What GPT-2's configuration multiplies the scores of a layer (from 0) by."""
    scale = (cfg.n_embd // cfg.n_head) ** -0.5 if cfg.scale_attn_weights else 1.0
    return scale / (layer + 1) if cfg.scale_attn_by_inverse_layer_idx else scale


def _prompt_attention(qkv, start, lens, longest, nh, scale):
    """Causal attention of packed prompts (host lengths ``lens``), qkv [rows, 3H]."""
    H = qkv.shape[1] // 3
    if (qkv.is_cuda and qkv.dtype == torch.bfloat16 and H // nh == 64 and longest <= _tx.ATTN_MAX_LEN
            and scale == 0.125):
        n = torch.tensor(lens, dtype=torch.int32, device=qkv.device)
        return _tx._Attention.apply(qkv, start[:-1].contiguous(), n, nh, 0.0, 0, longest)
    out, at = [], 0
    for n in lens:
        q, k, v = (t.view(1, n, nh, H // nh).transpose(1, 2) for t in qkv[at:at + n].split(H, dim=1))
        o = F.scaled_dot_product_attention(q, k, v, is_causal=True, scale=scale)
        out.append(o.transpose(1, 2).reshape(n, H))
        at += n
    return torch.cat(out)


@torch.no_grad()
def generate(model, prompts, *, max_new_tokens=20, num_beams=4, eos=None, token_types=None,
             reply_type=None, length_penalty=1.0, page_size=16):
    """Beam-search continuations of ``prompts`` (lists of token ids) by a GPT-2
    double-heads or LM-head model: [(token ids, score)], one a prompt, without
    the prompt and without ``eos``.

    A reply ends at ``eos`` (None: never) or after ``max_new_tokens``; the score is
    the sum of its tokens' log-probabilities (``eos`` among them) over its length
    ** ``length_penalty``.  ``token_types`` (a list beside each prompt) and
    ``reply_type`` (the type of every new token) add their embeddings as in
    training.  The keys and values live in pages (ops/decode.py): a request's
    beams share the prompt's, and no step waits for the GPU (the search ends
    early only where all replies of the batch ended, looked up every 8 tokens).
    What it does not cover -- other models, heads of other than 32, 64, 128 or 256
    columns, tokens outside the vocabulary -- is a ValueError before anything runs.

    The reference evaluates perplexity and candidate ranking only
    (gpt2_train.py:149-253); replies follow its model and input format."""
    m = model.model if isinstance(model, GPT2DoubleHeads) else model
    tr = getattr(m, "transformer", None)
    cfg = getattr(tr, "config", None)
    if getattr(cfg, "model_type", "") != "gpt2":
        raise ValueError("generate() covers GPT-2 models, not %r" % getattr(cfg, "model_type", type(m).__name__))
    lens = [len(p) for p in prompts]
    if not lens:
        return []
    if min(lens) < 1 or max_new_tokens < 1 or not 1 <= num_beams <= 32:
        raise ValueError("generate() needs a token in every prompt, a new token and 1 to 32 beams")
    if max(lens) + max_new_tokens > cfg.n_positions:
        raise ValueError("a prompt of %d tokens and %d new ones are more than the model's %d positions"
                         % (max(lens), max_new_tokens, cfg.n_positions))
    if (token_types is None) != (reply_type is None):
        raise ValueError("token_types and reply_type come together")
    if token_types is not None and [len(t) for t in token_types] != lens:
        raise ValueError("token_types need a type for every token of every prompt")
    wte, wpe = tr.wte.weight, tr.wpe.weight
    if eos is not None and not 0 <= eos < wte.shape[0]:
        raise ValueError("eos %r is not in the vocabulary" % (eos,))
    for what, lists in (("prompts", prompts), ("token_types", token_types or []),
                        ("reply_type", [] if reply_type is None else [[reply_type]])):
        for row in lists:  # (on a GPU the lookup itself would end the process)
            if not (0 <= min(row) and max(row) < wte.shape[0]):
                raise ValueError("%s name tokens that are not among the vocabulary's %d" % (what, wte.shape[0]))
    dev, B, J, nh = wte.device, len(prompts), num_beams, cfg.n_head
    H = cfg.n_embd
    hd = H // nh
    if not can_generate(cfg) or wte.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("generate() covers heads of 32, 64, 128 or 256 columns in bfloat16, float16 or float32, "
                         "not %d heads over %d columns in %s" % (nh, H, wte.dtype))
    if page_size < 1:
        raise ValueError("a page holds at least a token, not %r" % (page_size,))
    scales = [_attention_scale(cfg, i) for i in range(len(tr.h))]
    longest = max(lens) + max_new_tokens
    pages = sum(-(-n // page_size) for n in lens) + B * J * (1 + -(-max_new_tokens // page_size))
    cache = PagedKV(len(tr.h), nh, hd, B * J, pages, page_size, longest, wte.dtype, dev)

    def embed(ids, pos, types):
        x = F.embedding(ids, wte) + F.embedding(pos, wpe)
        return x if types is None else x + F.embedding(types, wte)

    def flat(lists):
        return torch.tensor([t for row in lists for t in row], dtype=torch.int64).to(dev)

    # the prompts, once a request, in its first beam's sequence
    new = torch.zeros(B, J, dtype=torch.int32)
    new[:, 0] = torch.tensor(lens, dtype=torch.int32)
    rows = sum(lens)
    r = cache.extend(new.view(-1).to(dev), rows)
    start = r.start[::J].contiguous()

    def attend_prompt(layer, qkv):
        k, v = (qkv[:, i * H:(i + 1) * H].view(rows, nh, hd) for i in (1, 2))
        cache.write(layer, k, v, r.slots)
        return _prompt_attention(qkv, start, lens, max(lens), nh, scales[layer])

    types = flat(token_types) if token_types is not None else None
    y = _blocks(tr, embed(flat(prompts), r.pos, types), attend_prompt)
    logits = _tx.lm_head(m, y[start[1:].long() - 1])
    cache.share(J)
    logits = logits.view(B, 1, -1).expand(B, J, -1)
    scores = torch.full((B, J), -math.inf, device=dev)
    scores[:, 0] = 0.0

    one = torch.ones(B * J, dtype=torch.int32, device=dev)
    types = torch.full((B * J,), reply_type, dtype=torch.int64, device=dev) if reply_type is not None else None
    finished = torch.zeros(B, J, dtype=torch.bool, device=dev) if eos is not None else None
    length = torch.zeros(B, J, device=dev)
    steps = []

    def attend_token(layer, qkv):
        q, k, v = (qkv[:, i * H:(i + 1) * H].view(B * J, nh, hd) for i in range(3))
        return cache.attend(layer, q, k, v, scale=scales[layer], max_len=longest).view(B * J, H)

    for t in range(max_new_tokens):
        if t:
            cache.reorder(parent)
            r = cache.extend(one, B * J)
            y = _blocks(tr, embed(token.view(-1), r.pos, types), attend_token)
            logits = _tx.lm_head(m, y).view(B, J, -1)
        scores, parent, token = beam_select(logits, scores, finished=finished, eos=-1 if eos is None else eos)
        steps.append((parent, token))
        if eos is None:
            length += 1
            continue
        ended = finished.gather(1, parent)
        length = length.gather(1, parent) + (~ended).float()
        finished = ended | (token == eos)
        if t % 8 == 7 and bool(finished.all()):
            break
    rank = scores / length.clamp_min(1.0) ** length_penalty
    best, at = rank.max(1)
    parents, tokens = (torch.stack(s).cpu().tolist() for s in zip(*steps))
    replies = []
    for b, (j, score) in enumerate(zip(at.tolist(), best.tolist())):
        out = []
        for par, tok in zip(reversed(parents), reversed(tokens)):
            out.append(tok[b][j])
            j = par[b][j]
        out.reverse()
        replies.append((out[:out.index(eos)] if eos in out else out, score))
    return replies
