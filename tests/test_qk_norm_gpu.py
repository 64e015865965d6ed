"""The per-head norm with rotation, forward and backward, and the append to a paged cache, against their formulas in 64 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}   # half a step, relative
EPS = 1e-5


def tables(n, D, gen):
    angle = torch.rand(n, D // 2, device="cuda", generator=gen, dtype=torch.float64) * 6.28
    return angle.cos().float(), angle.sin().float()


def turn(x, cos, sin, halves):
    if halves:
        a, b = x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def formula(x, w, cos, sin, norm, halves):
    """In 64 bits; differentiable."""
    if norm:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        x = x if w is None else x * w
    return x if cos is None else turn(x, cos, sin, halves)


def pair_size(y, halves):
    """Each element's magnitude together with its pair's: what a rotation's rounding is relative to."""
    if halves:
        a, b = y.chunk(2, -1)
        return torch.cat([torch.hypot(a, b)] * 2, -1)
    return torch.hypot(y[..., 0::2], y[..., 1::2]).repeat_interleave(2, -1)


def close(got, ref, dtype, size, steps):
    """One rounding to the output's type, and ``steps`` fp32 roundings (2^-24 each) relative to ``size``."""
    tol = ref.abs() * HALF[dtype] + size * (steps * 2.0 ** -24) * (1 + HALF[dtype]) + 1e-37
    over = ((got.double() - ref).abs() / tol).amax().item()
    assert over <= 1.0, over


CASES = [  # B, T, heads, kv heads, D
    (1, 1, 1, 1, 64), (2, 7, 3, 1, 64), (3, 33, 4, 2, 48), (2, 65, 5, 5, 96), (1, 130, 8, 2, 128), (1, 9, 2, 1, 16), (1, 5, 2, 1, 256),
    (2, 3, 4, 0, 32), (1, 4, 1, 1, 112), (1, 700, 6, 2, 80)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("norm,weights,rotate", [(True, True, True), (True, False, True), (False, False, True), (True, True, False)])
def test_forward_and_backward(dtype, halves, norm, weights, rotate):
    from mycaffe_b200 import paged
    dt = DT[dtype]
    for B, T, H, KV, D in CASES:
        gen = torch.Generator("cuda").manual_seed(B * T + D)
        cos, sin = tables(T + 3, D, gen) if rotate else (None, None)
        wq, wk = (1 + 0.3 * torch.randn(D, device="cuda", generator=gen) for _ in range(2)) if weights else (None, None)
        rot = paged.QkNormRope(cos, sin, wq, wk, eps=EPS, norm=norm, halves=halves)
        # parts of a packed projection, and (B, heads, T, D) outputs
        qkv = torch.randn(B, T, H + 2 * KV, D, device="cuda", generator=gen).to(dt)
        q, k = qkv[:, :, :H], qkv[:, :, H:H + KV] if KV else None
        new = lambda h: torch.full((B, h, T, D), 7.0, device="cuda", dtype=dt).transpose(1, 2)
        q_out, k_out = new(H), new(KV) if KV else None
        rot.forward(q, k, q_out, k_out)
        gq, gk = (torch.randn(B, h, T, D, device="cuda", generator=gen).to(dt).transpose(1, 2) for h in (H, KV))
        dqkv = torch.full_like(qkv, 7.0)
        dw = rot.backward(q, k, gq, gk if KV else None, dqkv[:, :, :H], dqkv[:, :, H:H + KV] if KV else None)
        assert (dqkv[:, :, H + KV:] == 7.0).all()
        c64, s64 = (None, None) if cos is None else (cos[:T].double()[:, None], sin[:T].double()[:, None])
        for x, y, g, dx, w, dwi in ((q, q_out, gq, dqkv[:, :, :H], wq, dw[0]), (k, k_out, gk, dqkv[:, :, H:H + KV], wk, dw[1])):
            if x is None:
                assert dwi is None
                continue
            x64 = x.double().requires_grad_()
            w64 = None if w is None else w.double().requires_grad_()
            ref = formula(x64, w64, c64, s64, norm, halves)
            grads = torch.autograd.grad(ref, [x64] + ([w64] if w64 is not None else []), g.double())
            # forward: the sum of D squares (D roundings, halved by the root), root, reciprocal, two products, a rotation of three
            close(y, ref.detach(), dt, pair_size(ref.detach(), halves), (D / 2 + 8 if norm else 0) + 4)
            # backward: g and g w a few roundings; inv (D/2 + 4), twice with xhat; the mean of D products (D)
            inv = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + EPS).detach() if norm else torch.ones_like(x64[..., :1])
            size = pair_size(g.double(), halves)
            big = size * (1 if w64 is None else w64.detach().abs())
            unit = (x64 * inv).detach()
            if norm:
                big = inv * (big + unit.abs() * (big * unit.abs()).mean(-1, keepdim=True))
            close(dx, grads[0], dt, big, (2 * D + 16 if norm else 0) + 4)
            if norm and w64 is not None:
                n = B * T * x.shape[2]
                total = (size * unit.abs()).sum((0, 1, 2))
                over = ((dwi.double() - grads[1]).abs() / (total * (D / 2 + 16 + min(n, 4000)) * 2.0 ** -24)).amax().item()
                assert over <= 1.0, over
            else:
                assert dwi is None


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_against_differences(dtype):
    """The forward's own change along a direction, taken in the inputs that the types hold, against the backward."""
    from mycaffe_b200 import paged
    gen = torch.Generator("cuda").manual_seed(5)
    B, T, H, D = 1, 12, 2, 64
    cos, sin = tables(T, D, gen)
    w = 1 + 0.3 * torch.randn(D, device="cuda", generator=gen)
    rot = paged.QkNormRope(cos, sin, w, None, eps=EPS)
    x = torch.randn(B, T, H, D, device="cuda", generator=gen).to(DT[dtype])
    g = torch.randn(B, T, H, D, device="cuda", generator=gen).to(DT[dtype])
    dx = torch.empty_like(x)
    dw, _ = rot.backward(x, None, g, None, dx, None)
    way = torch.randn(B, T, H, D, device="cuda", generator=gen, dtype=torch.float64)
    h = 1e-4
    f = lambda a, b: (formula(a, b, cos.double()[:, None], sin.double()[:, None], True, False) * g.double()).sum()
    slope = (f(x.double() + h * way, w.double()) - f(x.double() - h * way, w.double())) / (2 * h)
    # differences: h^2 times a third derivative of order one per element; dx: its type's half step of each product
    tol = (dx.double() * way).abs().sum() * HALF[DT[dtype]] + x.numel() * h * h * 100
    assert abs(slope - (dx.double() * way).sum()) <= tol
    one = torch.randn(D, device="cuda", generator=gen, dtype=torch.float64)
    slope = (f(x.double(), w.double() + h * one) - f(x.double(), w.double() - h * one)) / (2 * h)
    assert abs(slope - (dw.double() * one).sum()) <= (dw.double() * one).abs().sum() * 1e-4


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_positions_in_place_and_outside_the_tables(dtype):
    from mycaffe_b200 import paged
    gen = torch.Generator("cuda").manual_seed(6)
    B, T, H, KV, D = 2, 5, 3, 1, 64
    cos, sin = tables(40, D, gen)
    rot = paged.QkNormRope(cos, sin, halves=True)
    pos = torch.tensor([[39, 0, 7, 7, 3], [1, 40, 2, -1, 5]], dtype=torch.int32, device="cuda")
    q, k = (torch.randn(B, T, h, D, device="cuda", generator=gen).to(DT[dtype]) for h in (H, KV))
    q[1, 1], q[1, 3] = math.nan, math.inf                    # of rows that are refused nothing comes out
    x, y = q.clone(), k.clone()
    rot.forward(x, y, x, y, positions=pos)                   # in place
    safe = pos.clamp(0, 39).long()
    good = ((pos >= 0) & (pos < 40))[:, :, None, None]
    for got, src in ((x, q), (y, k)):
        clean = torch.where(good, src, 1.0)
        ref = torch.where(good, formula(clean.double(), None, cos.double()[safe][:, :, None], sin.double()[safe][:, :, None], True, True), 0.0)
        close(got, ref, DT[dtype], pair_size(ref, True), D / 2 + 12)
        assert not got[1, 1].any() and not got[1, 3].any()
    cache = paged.PagedCache(torch.zeros(1, 16, 1, 64, device="cuda"), torch.zeros(1, 16, 1, 64, device="cuda"), 1)
    st = cache.status()
    assert st[0] == 3 and st[1] in (6, 8) and st[2] in (40, -1) and st[3] == 2
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    rot.backward(q, k, torch.ones_like(q), torch.ones_like(k), dq, dk, positions=pos)
    assert not dq[1, 1].any() and not dq[1, 3].any() and torch.isfinite(dq.float()).all() and dq[0].any()
    cache.status()


def test_backward_in_a_graph_follows_its_inputs():
    from mycaffe_b200 import paged
    gen = torch.Generator("cuda").manual_seed(8)
    cos, sin = tables(64, 64, gen)
    w = torch.ones(64, device="cuda")
    rot = paged.QkNormRope(cos, sin, w, w)
    q, k, gq, gk = (torch.randn(2, 64, h, 64, device="cuda", generator=gen) for h in (4, 2, 4, 2))
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        rot.backward(q, k, gq, gk, dq, dk)
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        dw = rot.backward(q, k, gq, gk, dq, dk)
        graph.capture_end()
        for t in (q, k, gq, gk):
            t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
        graph.replay()
    torch.cuda.synchronize()
    a, b = torch.empty_like(q), torch.empty_like(k)
    ref = rot.backward(q, k, gq, gk, a, b)
    assert torch.equal(a, dq) and torch.equal(b, dk) and all(torch.equal(x, y) for x, y in zip(ref, dw))   # a fixed order: the same bits
    del graph


# ------------------------------------------------------------------------------------------------------------- append


TYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hs,halves,norm", [(32, False, True), (48, True, True), (64, False, False), (96, True, False), (128, False, True), (128, True, True)])
def test_append(act, cache, hs, halves, norm):
    from paged_util import Setup
    from mycaffe_b200 import paged
    seqs = [(1, 1), (20, 37), (0, 9), (1, 64), (17, 17), (3, 131)]
    s = Setup(seqs, 6, 2, hs, 16, act, cache, seed=hs, pad=5)
    gen = torch.Generator("cuda").manual_seed(1)
    cos, sin = tables(131, hs, gen)
    wq, wk = (1 + 0.3 * torch.randn(hs, device="cuda", generator=gen) for _ in range(2))
    rot = paged.QkNormRope(cos, sin, wq, wk, eps=EPS, norm=norm, halves=halves)
    qkv = torch.randn(s.n_tokens, 10, hs, device="cuda", generator=gen).to(s.act)
    qkv[0, 8, 3] = math.inf                                  # a value is only copied
    qkv[s.used:] = math.nan
    before = s.k_pages.clone(), s.v_pages.clone()
    out = torch.full((s.n_tokens, 6, hs), 7.0, device="cuda", dtype=s.act)
    s.cache.append(s.batch, rot, qkv[:, :6], qkv[:, 6:8], qkv[:, 8:], out)
    assert s.cache.status() == (0, 0, 0, 0)
    assert (out[s.used:] == 7.0).all()
    written = torch.zeros(s.k_pages.shape[:2], dtype=torch.bool, device="cuda")
    t = 0
    for b, (new, n) in enumerate(seqs):
        for pos in range(n - new, n):
            c, si = cos[pos].double(), sin[pos].double()
            page, slot = int(s.table[b, pos // 16]), pos % 16
            for got, x, w, dt in ((out[t], qkv[t, :6], wq, s.act), (s.k_pages[page, slot], qkv[t, 6:8], wk, s.cache_t)):
                ref = formula(x.double(), w.double(), c, si, norm, halves)
                close(got, ref, dt, pair_size(ref, halves), (hs / 2 + 8 if norm else 0) + 4)
            assert torch.equal(s.v_pages[page, slot], qkv[t, 8:].to(s.cache_t))
            written[page, slot] = True
            t += 1
    for now, was in zip((s.k_pages, s.v_pages), before):     # nothing else was touched
        assert torch.equal(now[~written].nan_to_num(9.0), was[~written].nan_to_num(9.0))


@pytest.mark.parametrize("act,cache", TYPES)
def test_append_refusals_on_the_device(act, cache):
    from paged_util import Setup
    from mycaffe_b200 import paged
    s = Setup([(2, 30), (3, 40), (1, 20)], 2, 1, 64, 16, act, cache, seed=3)
    gen = torch.Generator("cuda").manual_seed(2)
    cos, sin = tables(39, 64, gen)                           # position 39 has no row
    rot = paged.QkNormRope(cos, sin)
    q, k, v = (torch.randn(s.n_tokens, h, 64, device="cuda", generator=gen).to(s.act) for h in (2, 1, 1))
    before = s.k_pages.clone()
    out = torch.full_like(q, 7.0)
    s.cache.append(s.batch, rot, q, k, v, out)
    assert s.cache.status() == (3, 4, 39, 1)
    assert not out[4].any() and out[:4].any(-1).all() and out[5].any()
    page = int(s.table[1, 2])
    assert torch.equal(s.k_pages[page, 7].nan_to_num(9.0), before[page, 7].nan_to_num(9.0))
    s.table[2, 1] = -1                                       # the new token's page is not held
    s.cache.append(s.batch, rot, q, k, v, out)
    st = s.cache.status()
    assert st[3] == 2 and st[0] in (2, 3)
    bad = torch.tensor([30, 2, 20], device="cuda", dtype=torch.int32)
    out.fill_(7.0)
    s.cache.append(s.cache.batch(s.starts, bad, s.table, s.n_tokens, 3, 40), rot, q, k, v, out)
    assert s.cache.status()[:1] != (0,) and not out[2:5].any() and out[:2].any()


@pytest.mark.parametrize("act,cache", TYPES)
def test_prompt_in_chunks_and_token_by_token(act, cache):
    """A run as a server has it: one prompt appended and attended to in chunks of odd lengths, then token by token, equals the whole prompt
    at once; other sequences step along."""
    from paged_util import Setup
    from mycaffe_b200 import paged
    gen = torch.Generator("cuda").manual_seed(4)
    n, H, KV, D, page = 150, 4, 2, 64, 16
    cos, sin = tables(n, D, gen)
    w = 1 + 0.2 * torch.randn(D, device="cuda", generator=gen)
    rot = paged.QkNormRope(cos, sin, w, w, halves=True)
    s = Setup([(n, n), (n, n)], H, KV, D, page, act, cache)
    qkv = torch.randn(2, n, H + 2 * KV, D, device="cuda", generator=gen).to(s.act)

    def steps(sizes):
        s.k_pages.fill_(math.nan), s.v_pages.fill_(math.nan)
        outs, at = [[], []], 0
        for m in sizes:
            x = qkv[:, at:at + m].reshape(2 * m, H + 2 * KV, D)
            at += m
            starts = torch.tensor([0, m, 2 * m], dtype=torch.int32, device="cuda")
            lengths = torch.tensor([at, at], dtype=torch.int32, device="cuda")
            b = s.cache.batch(starts, lengths, s.table, 2 * m, m, at)
            q = torch.empty(2 * m, H, D, device="cuda", dtype=s.act)
            out = torch.empty_like(q)
            s.cache.append(b, rot, x[:, :H], x[:, H:H + KV], x[:, H + KV:], q)
            s.cache.attend(b, q, out)
            outs[0].append(out[:m])
            outs[1].append(out[m:])
        return torch.stack([torch.cat(o) for o in outs]).double(), s.k_pages.clone()

    whole, pages = steps([n])
    parts, pages2 = steps([1, 63, 2, 64] + [1] * 20)
    assert torch.equal(pages.nan_to_num(9.0), pages2.nan_to_num(9.0))
    # the two differ by two evaluations' roundings of outputs that are averages of values of unit size
    tol = {"f32f32": 1e-5, "f32bf16": 2e-4, "bf16bf16": 4 * 2.0 ** -8}[act + cache] * whole.abs().amax()
    assert (whole - parts).abs().amax() <= tol
    assert s.cache.status() == (0, 0, 0, 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("halves", [False, True])
def test_positions_with_norm_and_weights(dtype, halves):
    """Explicit positions, some twice, some outside the tables: the norm, both inputs' gradients and both weights' follow them."""
    from mycaffe_b200 import paged
    gen = torch.Generator("cuda").manual_seed(7)
    B, T, H, KV, D, dt = 3, 37, 5, 2, 96, DT[dtype]
    cos, sin = tables(50, D, gen)
    wq, wk = (1 + 0.3 * torch.randn(D, device="cuda", generator=gen) for _ in range(2))
    rot = paged.QkNormRope(cos, sin, wq, wk, eps=EPS, halves=halves)
    pos = torch.randint(0, 50, (B, T), device="cuda", generator=gen, dtype=torch.int32)
    pos[0, 3], pos[2, 36] = 50, -1
    good = ((pos >= 0) & (pos < 50))[:, :, None, None]
    at = pos.clamp(0, 49).long()
    c64, s64 = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    x = [torch.randn(B, T, h, D, device="cuda", generator=gen).to(dt) for h in (H, KV)]
    g = [torch.randn(B, T, h, D, device="cuda", generator=gen).to(dt) for h in (H, KV)]
    y, dx = [torch.full_like(t, 7.0) for t in x], [torch.full_like(t, 7.0) for t in x]
    rot.forward(*x, *y, positions=pos)
    dw = rot.backward(*x, *g, *dx, positions=pos)
    for i, w in enumerate((wq, wk)):
        x64, w64 = x[i].double().requires_grad_(), w.double().requires_grad_()
        ref = torch.where(good, formula(x64, w64, c64, s64, True, halves), 0.0)
        grads = torch.autograd.grad(ref, [x64, w64], g[i].double())
        # the bounds of test_forward_and_backward
        close(y[i], ref.detach(), dt, pair_size(ref.detach(), halves), D / 2 + 12)
        inv = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + EPS).detach()
        size, unit = pair_size(g[i].double(), halves), (x64 * inv).detach()
        big = size * w64.detach().abs()
        close(dx[i], grads[0], dt, inv * (big + unit.abs() * (big * unit.abs()).mean(-1, keepdim=True)), 2 * D + 20)
        total = (size * unit.abs()).sum((0, 1, 2))
        over = ((dw[i].double() - grads[1]).abs() / (total * (D / 2 + 16 + B * T * x[i].shape[2]) * 2.0 ** -24)).amax().item()
        assert over <= 1.0, over
    paged.PagedCache(torch.zeros(1, 16, 1, 64, device="cuda"), torch.zeros(1, 16, 1, 64, device="cuda"), 1).status()
