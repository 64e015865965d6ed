"""Measured cases of the paged key/value cache and of the per-head norm with rotation: the attention of new tokens over a
paged cache, the append that puts them there, and the norm and rotation of queries and keys in training.

Each case is what a program does around one attention layer.  Where ``own`` is false ``run`` computes the operator from its
formula with elementary torch operations in 32 bits; where it is true it makes the calls a user of this package makes.
"""
import math

import torch

own = False

EPS = 1e-5

# --------------------------------------------------------------------------------------------------------------- cases


def attend(name, seqs, chunks, new, cached, ragged, heads, kv, hs, page, act, cache, pad=0):
    """Attention of the new tokens of ``seqs`` sequences, each over its own pages.  The first ``chunks`` sequences bring up to
    ``new`` tokens, the others one; up to ``cached`` keys lie before them.  ragged: the share by which lengths are spread."""
    return dict(name=name, kind="attend", seqs=seqs, chunks=chunks, new=new, cached=cached, ragged=ragged, heads=heads, kv=kv, hs=hs,
                page=page, act=act, cache=cache, pad=pad)


def append(name, seqs, chunks, new, cached, ragged, heads, kv, hs, page, act, cache, norm, halves, pad=0):
    """Norm and rotation of the new tokens' queries and keys, and the keys and values into their pages."""
    return dict(attend(name, seqs, chunks, new, cached, ragged, heads, kv, hs, page, act, cache, pad), kind="append", norm=norm,
                halves=halves)


def train(name, B, T, heads, kv, hs, act, halves):
    """Norm and rotation of a layer's queries and keys, forward and backward: from the packed projection to (B,H,T,D) tensors,
    and their gradients back into the packed one."""
    return dict(name=name, kind="train", B=B, T=T, heads=heads, kv=kv, hs=hs, act=act, halves=halves)


def listed():
    return [
        # the smallest call: a token of a llama2.c 110M model for one user, fp32 as its checkpoint is
        attend("attend_one_token_f32", 1, 0, 1, 700, 0.0, 12, 12, 64, 16, "f32", "f32"),
        # serving: one token of each of 64 sequences of ragged length
        attend("attend_64_sequences", 64, 0, 1, 4095, 0.7, 32, 8, 128, 64, "bf16", "bf16"),
        # two users deep into long documents
        attend("attend_long_cache", 2, 0, 1, 70001, 0.2, 32, 8, 128, 32, "bf16", "bf16"),
        # a chunk of a long prompt over what is in the cache already
        attend("attend_chunk_16k", 1, 1, 2048, 16384, 0.0, 32, 8, 128, 128, "bf16", "bf16"),
        # fresh prompts of odd lengths, 64-wide heads without sharing
        attend("attend_prompts_64", 8, 8, 1000, 0, 0.6, 16, 16, 64, 32, "bf16", "bf16"),
        # a serving step that takes two prompts' chunks along with the other sequences' single tokens
        attend("attend_mixed_step", 24, 2, 500, 3000, 0.5, 32, 8, 128, 16, "bf16", "bf16"),
        # prompts of a llama2.c model through fp32 activations and an fp32 cache
        attend("attend_chunk_f32", 4, 4, 200, 512, 0.5, 6, 6, 48, 16, "f32", "f32"),
        # fp32 activations over a bf16 cache, as the decode step of this package has them
        attend("attend_tokens_f32_bf16", 16, 0, 1, 2048, 0.5, 32, 32, 128, 64, "f32", "bf16"),
        # the append of one serving step
        append("append_64_tokens", 64, 0, 1, 1023, 0.7, 32, 8, 128, 64, "bf16", "bf16", True, True),
        # the append of a prompt
        append("append_prompt", 1, 1, 4095, 0, 0.0, 32, 8, 128, 64, "bf16", "bf16", True, False),
        # training: one GPT-2-small layer in fp32
        train("train_f32", 8, 1024, 12, 12, 64, "f32", False),
        # training: long sequences of wide bf16 heads that share keys
        train("train_bf16", 2, 4095, 32, 8, 128, "bf16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above."""
    kind = rng.choice(["one", "one", "one", "chunk", "chunk", "mixed", "append", "append", "train", "train"])
    heads = rng.choice([4, 6, 8, 12, 16, 32])
    kv = rng.choice([h for h in (heads, heads // 2, heads // 4) if h > 0 and heads % h == 0])
    hs = rng.choice([32, 48, 64, 64, 96, 128, 128])
    act, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")])
    page = rng.choice([16, 32, 64, 128, 256])
    ragged = round(rng.uniform(0.0, 0.9), 2)
    pad = rng.choice([0, 0, 7])
    if kind == "one":
        seqs = _log(rng, 1, 64)
        most = 500_000_000 // (seqs * kv * hs * 2 * (2 if cache == "bf16" else 4))   # keys that half a gigabyte of pages holds
        c = attend("", seqs, 0, 1, _log(rng, 1, min(65536, most)), ragged, heads, kv, hs, page, act, cache, pad)
    elif kind == "chunk":
        seqs = rng.randint(1, 8)
        new = _log(rng, 2, 2048 // seqs)
        c = attend("", seqs, seqs, new, rng.choice([0, _log(rng, 16, 8192)]), ragged, heads, kv, hs, page, act, cache, pad)
    elif kind == "mixed":
        seqs = rng.randint(4, 24)
        c = attend("", seqs, rng.randint(1, 3), _log(rng, 16, 400), _log(rng, 64, 2500), ragged, heads, kv, hs, page, act, cache, pad)
    elif kind == "append":
        seqs = _log(rng, 1, 64)
        c = append("", seqs, rng.choice([0, min(seqs, 4)]), _log(rng, 1, 1024), _log(rng, 1, 1024), ragged, heads, kv, hs, page, act, cache,
                   rng.random() < 0.7, rng.random() < 0.5, pad)
    else:
        c = train("", _log(rng, 1, 8), _log(rng, 16, 2047), heads, kv, hs, act, rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------- preparing a state


def _spread(b, most, ragged):
    """A length of at most ``most`` for sequence ``b``: spread by the golden ratio, the first one the longest."""
    return most - int(most * ragged * ((b * 0.6180339887498949) % 1.0))


def _lengths(c):
    """New tokens of each sequence and keys it holds with them."""
    new = [max(1, _spread(b, c["new"], c["ragged"])) if b < c["chunks"] else 1 for b in range(c["seqs"])]
    return new, [n + _spread(b, c["cached"], c["ragged"]) for b, n in enumerate(new)]


def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _rotation(c, length, gen):
    """Tables of the rotation and the norms' weights, as a model holds them."""
    half = c["hs"] // 2
    freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * freq
    weight = 1.0 + 0.2 * torch.randn(2, c["hs"], device="cuda", generator=gen)
    return dict(cos=angle.cos().float(), sin=angle.sin().float(), wq=weight[0].contiguous(), wk=weight[1].contiguous())


def _normal(shape, dtype, gen, scale=1.0):
    return torch.randn(shape, device="cuda", generator=gen).mul_(scale).to(dtype)


def prepare(case, seed):
    c = case
    gen = torch.Generator("cuda").manual_seed(int(seed))
    act = _type(c["act"])
    if c["kind"] == "train":
        B, T, H, KV, D = c["B"], c["T"], c["heads"], c["kv"], c["hs"]
        s = dict(c=c, **_rotation(c, T, gen))
        # the packed projection, with a scale per channel as a trained layer's has
        s["qkv"] = (torch.randn(B, T, (H + 2 * KV) * D, device="cuda", generator=gen)
                    * (0.5 + torch.rand((H + 2 * KV) * D, device="cuda", generator=gen))).to(act)
        s["dq_out"], s["dk_out"] = _normal((B, H, T, D), act, gen, 0.1), _normal((B, KV, T, D), act, gen, 0.1)
        s["q_out"], s["k_out"] = torch.empty_like(s["dq_out"]), torch.empty_like(s["dk_out"])
        s["dqkv"] = torch.zeros_like(s["qkv"])
        return s
    H, KV, D, page = c["heads"], c["kv"], c["hs"], c["page"]
    new, length = _lengths(c)
    pages = [-(-n // page) for n in length]
    n_pages, stride = sum(pages) + 3, max(pages) + 1
    order = torch.randperm(n_pages, device="cuda", generator=gen, dtype=torch.int32)
    count = torch.tensor(pages, device="cuda")
    column = torch.arange(stride, device="cuda")
    first = torch.cumsum(count, 0) - count
    table = torch.where(column[None, :] < count[:, None], order[(first[:, None] + column[None, :]).clamp(max=n_pages - 1)], -1)
    s = dict(c=c, used=sum(new), n_tokens=sum(new) + c["pad"], max_new=max(new), max_len=max(length), table=table.to(torch.int32))
    s["lengths"] = torch.tensor(length, device="cuda", dtype=torch.int32)
    s["starts"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    s["k_pages"] = _normal((n_pages, page, KV, D), _type(c["cache"]), gen)
    s["v_pages"] = _normal((n_pages, page, KV, D), _type(c["cache"]), gen)
    if c["kind"] == "attend":
        s["q"] = _normal((s["n_tokens"], H, D), act, gen)
        s["out"] = torch.zeros_like(s["q"])
    else:
        s.update(_rotation(c, s["max_len"], gen))
        s["qkv"] = _normal((s["n_tokens"], H + 2 * KV, D), act, gen)   # the packed projection of the new tokens
        s["q_out"] = torch.zeros(s["n_tokens"], H, D, device="cuda", dtype=act)
    return s


# ------------------------------------------------------------------------------------------------------ the plain forms


def _rotate(x, cos, sin, halves):
    """(..., D) with cos, sin (..., D/2): pair p is (x[p], x[p + D/2]) with ``halves``, else (x[2p], x[2p + 1])."""
    if halves:
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _norm_rotate(x, w, cos, sin, norm, halves):
    x = x.float()
    if norm:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    return _rotate(x, cos, sin, halves)


def _tokens(s):
    """Sequence and index within the chunk of each token, and its position."""
    t = torch.arange(s["used"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    index = t - s["starts"][seq]
    count = s["starts"][1:] - s["starts"][:-1]
    return seq, index, s["lengths"][seq].long() - count[seq] + index


def _plain_attend(s):
    c = s["c"]
    B, N, L, KV, D, page = c["seqs"], s["max_new"], s["max_len"], c["kv"], c["hs"], c["page"]
    G = c["heads"] // KV
    key = torch.arange(L, device="cuda")
    row = s["table"].long()[:, key // page].clamp(min=0) * page + key % page                    # (B, L)
    k = s["k_pages"].view(-1, KV, D)[row].float().permute(0, 2, 3, 1)                            # (B, KV, D, L)
    v = s["v_pages"].view(-1, KV, D)[row].float().permute(0, 2, 1, 3)                            # (B, KV, L, D)
    count = (s["starts"][1:] - s["starts"][:-1]).long()
    at = (s["starts"][:-1, None] + torch.arange(N, device="cuda")).clamp(max=s["n_tokens"] - 1)  # (B, N)
    q = s["q"][at].float().view(B, N, KV, G, D).permute(0, 2, 3, 1, 4).reshape(B, KV, G * N, D)
    score = torch.matmul(q, k).mul_(1.0 / math.sqrt(D)).view(B, KV, G, N, L)
    last = (s["lengths"].long() - count)[:, None] + torch.arange(N, device="cuda")               # (B, N): the last key a token sees
    score.masked_fill_((key > last[:, :, None])[:, None, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    score.div_(score.sum(-1, keepdim=True))
    out = torch.matmul(score.view(B, KV, G * N, L), v).view(B, KV, G, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, KV * G, D)
    seq, index, _ = _tokens(s)
    s["out"][: s["used"]] = out[seq, index].to(s["out"].dtype)
    return {"out": s["out"]}


def _plain_append(s):
    c = s["c"]
    H, KV, D, page, used = c["heads"], c["kv"], c["hs"], c["page"], s["used"]
    seq, _, pos = _tokens(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    qkv = s["qkv"][:used]
    row = s["table"][seq, pos // page].long() * page + pos % page
    s["q_out"][:used] = _norm_rotate(qkv[:, :H], s["wq"], cos, sin, c["norm"], c["halves"]).to(s["q_out"].dtype)
    s["k_pages"].view(-1, KV, D)[row] = _norm_rotate(qkv[:, H:H + KV], s["wk"], cos, sin, c["norm"], c["halves"]).to(s["k_pages"].dtype)
    s["v_pages"].view(-1, KV, D)[row] = qkv[:, H + KV:].to(s["v_pages"].dtype)
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_train_part(s, x, w, g):
    """x (B,T,h,D) from the projection, g (B,h,T,D): output, gradients of x and w."""
    x, g = x.float(), g.float().transpose(1, 2)
    cos, sin = s["cos"][:, None], s["sin"][:, None]
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    unit = x * inv
    y = _rotate(unit * w, cos, sin, s["c"]["halves"])
    g = _rotate(g, cos, -sin, s["c"]["halves"])
    dw = (g * unit).sum((0, 1, 2))
    g = g * w
    return y.transpose(1, 2), inv * (g - unit * (g * unit).mean(-1, keepdim=True)), dw


def _plain_train(s):
    c = s["c"]
    B, T, H, KV, D = c["B"], c["T"], c["heads"], c["kv"], c["hs"]
    x = s["qkv"].view(B, T, H + 2 * KV, D)
    q, dq, dwq = _plain_train_part(s, x[:, :, :H], s["wq"], s["dq_out"])
    k, dk, dwk = _plain_train_part(s, x[:, :, H:H + KV], s["wk"], s["dk_out"])
    d = s["dqkv"].view(B, T, H + 2 * KV, D)
    d[:, :, :H], d[:, :, H:H + KV] = dq.to(d.dtype), dk.to(d.dtype)
    return {"q": q.to(d.dtype), "k": k.to(d.dtype), "dqkv": s["dqkv"], "dwq": dwq, "dwk": dwk}


# -------------------------------------------------------------------------------------------- the calls of this package


def _own_cache(s):
    from mycaffe_b200 import paged
    if "cache" not in s:
        s["cache"] = paged.PagedCache(s["k_pages"], s["v_pages"], s["c"]["heads"])
        if "cos" in s:
            s["rotation"] = paged.QkNormRope(s["cos"], s["sin"], s["wq"], s["wk"], eps=EPS, norm=s["c"]["norm"], halves=s["c"]["halves"])
    cache = s["cache"]
    return cache, cache.batch(s["starts"], s["lengths"], s["table"], s["n_tokens"], s["max_new"], s["max_len"])


def _own_attend(s):
    cache, batch = _own_cache(s)
    cache.attend(batch, s["q"], s["out"])
    return {"out": s["out"]}


def _own_append(s):
    c = s["c"]
    cache, batch = _own_cache(s)
    H, KV = c["heads"], c["kv"]
    cache.append(batch, s["rotation"], s["qkv"][:, :H], s["qkv"][:, H:H + KV], s["qkv"][:, H + KV:], s["q_out"])
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_train(s):
    from mycaffe_b200 import paged
    c = s["c"]
    B, T, H, KV, D = c["B"], c["T"], c["heads"], c["kv"], c["hs"]
    if "rotation" not in s:
        s["rotation"] = paged.QkNormRope(s["cos"], s["sin"], s["wq"], s["wk"], eps=EPS, norm=True, halves=c["halves"])
    rotation = s["rotation"]
    x, d = s["qkv"].view(B, T, H + 2 * KV, D), s["dqkv"].view(B, T, H + 2 * KV, D)
    rotation.forward(x[:, :, :H], x[:, :, H:H + KV], s["q_out"].transpose(1, 2), s["k_out"].transpose(1, 2))
    dwq, dwk = rotation.backward(x[:, :, :H], x[:, :, H:H + KV], s["dq_out"].transpose(1, 2), s["dk_out"].transpose(1, 2),
                                 d[:, :, :H], d[:, :, H:H + KV])
    return {"q": s["q_out"], "k": s["k_out"], "dqkv": s["dqkv"], "dwq": dwq, "dwk": dwk}


def run(state):
    kind = state["c"]["kind"]
    if own:
        return _own_attend(state) if kind == "attend" else _own_append(state) if kind == "append" else _own_train(state)
    return _plain_attend(state) if kind == "attend" else _plain_append(state) if kind == "append" else _plain_train(state)


# ----------------------------------------------------------------------------------------------- work and exact results


def work(case):
    c = case
    size = 2 if c["act"] == "bf16" else 4
    if c["kind"] == "train":
        # forward: q and k read and written; backward: q, k and the gradients read, dq and dk written
        n = c["B"] * c["T"] * (c["heads"] + c["kv"]) * c["hs"]
        return {"bytes": 5 * n * size + c["T"] * c["hs"] * 4, "flops": 26 * n}
    new, length = _lengths(c)
    tokens = sum(new)
    csize = 2 if c["cache"] == "bf16" else 4
    if c["kind"] == "append":
        q, kv = tokens * c["heads"] * c["hs"], tokens * c["kv"] * c["hs"]
        return {"bytes": (2 * q + 2 * kv) * size + 2 * kv * csize + tokens * c["hs"] * 4, "flops": 8 * (q + kv)}
    seen = sum(n * (le - n) + n * (n + 1) // 2 for n, le in zip(new, length))   # (token, key) pairs
    return {"bytes": 2 * tokens * c["heads"] * c["hs"] * size + 2 * sum(length) * c["kv"] * c["hs"] * csize,
            "flops": 4 * seen * c["heads"] * c["hs"]}


def _exact_attend(s):
    c = s["c"]
    G, D, page = c["heads"] // c["kv"], c["hs"], c["page"]
    out = s["out"].double()
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for b, n_keys in enumerate(lengths):
        ids = s["table"][b, : -(-n_keys // page)].long()
        k, v = (p[ids].reshape(-1, c["kv"], D)[:n_keys].double() for p in (s["k_pages"], s["v_pages"]))
        rows = torch.arange(starts[b], starts[b + 1], device="cuda")
        hidden = torch.arange(n_keys, device="cuda") > (n_keys - starts[b + 1] + rows)[:, None]
        for h in range(c["heads"]):
            logits = s["q"][rows, h].double() @ k[:, h // G].T / math.sqrt(D)
            out[rows, h] = torch.softmax(logits.masked_fill(hidden, -math.inf), -1) @ v[:, h // G]
    return {"out": out}


def _exact_rotation(x, w, cos, sin, norm, halves):
    """The norm and rotation by complex numbers; differentiable."""
    if norm:
        x = w * x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS)
    half = x.shape[-1] // 2
    pair = x.unflatten(-1, (2, half)).movedim(-2, -1) if halves else x.unflatten(-1, (half, 2))
    turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.complex(cos, sin))
    return (turned.movedim(-1, -2) if halves else turned).flatten(-2)


def _exact_append(s):
    c = s["c"]
    H, KV, page = c["heads"], c["kv"], c["page"]
    q, k_pages, v_pages = s["q_out"].double(), s["k_pages"].double(), s["v_pages"].double()
    cos, sin, wq, wk = (s[n].double() for n in ("cos", "sin", "wq", "wk"))
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for b, n_keys in enumerate(lengths):
        x = s["qkv"][starts[b]:starts[b + 1]].double()
        at = torch.arange(n_keys - x.shape[0], n_keys, device="cuda")
        turn = (cos[at, None], sin[at, None], c["norm"], c["halves"])
        ids, slot = s["table"][b, at // page].long(), at % page
        q[starts[b]:starts[b + 1]] = _exact_rotation(x[:, :H], wq, *turn)
        k_pages[ids, slot] = _exact_rotation(x[:, H:H + KV], wk, *turn)
        v_pages[ids, slot] = x[:, H + KV:]
    return {"q": q, "k_pages": k_pages, "v_pages": v_pages}


def _exact_train(s):
    c = s["c"]
    B, T, H, KV, D = c["B"], c["T"], c["heads"], c["kv"], c["hs"]
    x = s["qkv"].double().view(B, T, H + 2 * KV, D).requires_grad_()
    wq, wk = s["wq"].double().requires_grad_(), s["wk"].double().requires_grad_()
    turn = (s["cos"].double()[:, None], s["sin"].double()[:, None], True, c["halves"])
    q = _exact_rotation(x[:, :, :H], wq, *turn).transpose(1, 2)
    k = _exact_rotation(x[:, :, H:H + KV], wk, *turn).transpose(1, 2)
    dx, dwq, dwk = torch.autograd.grad([q, k], [x, wq, wk], [s["dq_out"].double(), s["dk_out"].double()])
    return {"q": q.detach(), "k": k.detach(), "dqkv": dx.view(B, T, -1), "dwq": dwq, "dwk": dwk}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "train": _exact_train}[case["kind"]](s)
