"""Attention of new tokens over a paged cache against its formula in 64 bits.  What no sequence owns of the pool is NaN, so that a
read behind a length, or of a page that is not held, shows."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")]


def setup(*a, **k):
    from paged_util import Setup
    return Setup(*a, **k)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hs", [32, 48, 64, 96, 128])
def test_single_tokens(act, cache, hs):
    s = setup([(1, n) for n in (1, 2, 15, 16, 17, 127, 128, 129, 300)], 4, 2, hs, 16, act, cache)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    assert s.cache.status() == (0, 0, 0, 0)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (4, 1), (6, 2), (8, 8), (16, 1)])
def test_chunks(act, cache, heads, kv):
    s = setup([(1, 1), (2, 2), (33, 33), (130, 131), (5, 200), (64, 128), (1, 77)], heads, kv, 64, 32, act, cache, seed=1)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("page", [16, 64, 128, 256, 1024])
def test_pages(act, cache, page):
    s = setup([(40, 300), (1, 1030), (7, 7)], 8, 2, 128, page, act, cache, seed=2)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()


@pytest.mark.parametrize("act,cache", TYPES)
def test_long_single_tokens_are_split(act, cache):
    s = setup([(1, 5003), (1, 129), (1, 2500)], 4, 1, 128, 64, act, cache, seed=3)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()


@pytest.mark.parametrize("act,cache", TYPES)
def test_chunk_over_a_long_cache_is_split(act, cache):
    s = setup([(37, 4001), (1, 9)], 4, 4, 64, 32, act, cache, seed=4)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()


@pytest.mark.parametrize("act,cache", TYPES)
def test_pages_not_held(act, cache):
    """The middle, the first, the last and all pages of a sequence are gone; a token with no key left gives zeros."""
    s = setup([(3, 100), (40, 90), (1, 64), (20, 20), (1, 1500)], 4, 2, 64, 16, act, cache, seed=5,
              drop=[(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (1, 3), (2, 3), (3, 0), (3, 1)] + [(4, i) for i in range(3, 60)])
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    assert not s.out[s.starts[3]:s.starts[4]].any()
    assert s.cache.status() == (0, 0, 0, 0)


@pytest.mark.parametrize("act,cache", TYPES)
def test_padding_and_sequences_without_tokens(act, cache):
    s = setup([(0, 50), (3, 10), (0, 0), (1, 40), (0, 17)], 4, 4, 64, 16, act, cache, seed=6, pad=9, max_new=50, max_len=64)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()                                   # rows behind the last sequence: still 7
    s.lengths[0], s.lengths[2], s.lengths[4] = 1 << 20, -3, 0     # lengths of sequences without tokens are not looked at
    s.out.fill_(7.0)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    assert s.cache.status() == (0, 0, 0, 0)


@pytest.mark.parametrize("act,cache", TYPES)
def test_strides_and_scale(act, cache):
    """q and out as parts of wider rows, pages apart from one another, a scale of the caller's."""
    s = setup([(20, 150), (1, 33)], 4, 2, 64, 16, act, cache, seed=7, stride_pages=64)
    wide = torch.zeros(s.n_tokens, 10, 80, device="cuda", dtype=s.act)
    wide[:, 2:6, :64] = s.q
    out = torch.full_like(wide, 7.0)
    s.cache.attend(s.batch, wide[:, 2:6, :64], out[:, 5:9, :64], scale=0.21)
    s.out = out[:, 5:9, :64].contiguous()
    s.check(scale=0.21)
    out[:, 5:9, :64] = 7.0
    assert (out == 7.0).all()


@pytest.mark.parametrize("act,cache", TYPES)
def test_more_sequences_than_a_warp_looks_at_once(act, cache):
    s = setup([(1 + b % 3, 3 + b) for b in range(70)], 2, 1, 32, 16, act, cache, seed=8)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()


@pytest.mark.parametrize("act,cache", TYPES)
def test_large_logits(act, cache):
    """One key far above the others, and the maximum moving late: the sums are rescaled."""
    s = setup([(5, 400), (1, 700)], 2, 2, 64, 32, act, cache, seed=9)
    s.q *= 6.0
    s.cache.attend(s.batch, s.q, s.out)
    s.check()


@pytest.mark.parametrize("act,cache", TYPES)
def test_captured_and_on_another_stream(act, cache):
    """A captured call follows new lengths and queries; two graphs in flight at once do not share a workspace."""
    a, b = (setup([(1, 2000), (3, 300)], 4, 1, 64, 16, act, cache, seed=10 + i) for i in range(2))
    side = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for s, st in zip((a, b), side):
        with torch.cuda.stream(st):
            s.cache.attend(s.batch, s.q, s.out)
            st.synchronize()
            g = torch.cuda.CUDAGraph()
            g.capture_begin()
            s.cache.attend(s.batch, s.q, s.out)
            g.capture_end()
            graphs.append(g)
    for s in (a, b):
        s.q.copy_(torch.randn_like(s.q.float()).to(s.q.dtype))
        s.lengths.copy_(torch.tensor([1990, 299], device="cuda", dtype=torch.int32))
        s.seqs = [(1, 1990), (3, 299)]
        s.k, s.v = [k[:n] for k, (_, n) in zip(s.k, s.seqs)], [v[:n] for v, (_, n) in zip(s.v, s.seqs)]
        s.held = [h[:n] for h, (_, n) in zip(s.held, s.seqs)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, side):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s in (a, b):
        s.check()
    del graphs


@pytest.mark.parametrize("act,cache", TYPES)
def test_refused_sequences_give_zeros_and_a_status(act, cache):
    s = setup([(2, 40), (3, 50), (4, 60)], 4, 2, 64, 16, act, cache, seed=12)
    ref, tol = s.exact()
    bad = torch.tensor([40, 2, 60], device="cuda", dtype=torch.int32)       # fewer positions than new tokens
    batch = s.cache.batch(s.starts, bad, s.table, s.n_tokens, s.max_new, s.max_len)
    s.cache.attend(batch, s.q, s.out)
    assert s.cache.status() == (1, 1, 2, 1)
    assert not s.out[2:5].any()
    keep = [0, 1, 5, 6, 7, 8]
    assert ((s.out.double() - ref).abs()[keep] <= tol[keep]).all()
    assert s.cache.status() == (0, 0, 0, 0)
    long = torch.tensor([40, 50, 61], device="cuda", dtype=torch.int32)      # longer than the bound
    s.cache.attend(s.cache.batch(s.starts, long, s.table, s.n_tokens, s.max_new, 60), s.q, s.out)
    assert s.cache.status() == (1, 2, 61, 1) and not s.out[5:].any()


@pytest.mark.parametrize("act,cache", TYPES)
def test_page_ids_outside_the_pool_are_left_out(act, cache):
    s = setup([(2, 40), (1, 50)], 4, 2, 64, 16, act, cache, seed=13, drop=[(1, 1)])
    s.table[1, 1] = s.k_pages.shape[0]
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    st = s.cache.status()
    assert st[:3] == (2, 1, s.k_pages.shape[0]) and st[3] >= 1
    s.table[1, 1] = -2
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    assert s.cache.status()[:3] == (2, 1, -2)


def test_runs_alike():
    """The same call gives the same bits."""
    s = setup([(1, 3000), (50, 700)], 8, 2, 128, 64, "bf16", "bf16", seed=14)
    s.cache.attend(s.batch, s.q, s.out)
    first = s.out.clone()
    for _ in range(3):
        s.out.zero_()
        s.cache.attend(s.batch, s.q, s.out)
        assert torch.equal(first, s.out)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hs", [64, 128])
def test_many_key_tiles_for_each_block(act, cache, hs):
    """Work enough that every block of the launch has several items, and items of many key tiles: single tokens."""
    s = setup([(1, 100 + 531 * b % 4000) for b in range(24)], 16, 8, hs, 32, act, cache, seed=15, drop=[(3, 2), (7, 0)])
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    assert s.cache.status() == (0, 0, 0, 0)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hs", [64, 128])
def test_many_key_tiles_for_each_block_of_chunks(act, cache, hs):
    """The same for chunks of many tokens among single ones."""
    s = setup([(300, 2000), (1, 1500), (129, 129), (1, 2900), (400, 420)], 16, 4, hs, 64, act, cache, seed=16)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    assert s.cache.status() == (0, 0, 0, 0)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hs", [48, 128])
@pytest.mark.parametrize("long", [False, True])
def test_values_that_are_not_finite_reach_only_the_tokens_that_see_them(act, cache, hs, long):
    """A later token of the same chunk holds an infinity or NaN: the tokens before it come out as without it."""
    n = 3000 if long else 100
    s = setup([(40, n), (1, 30)], 4, 2, hs, 16, act, cache, seed=17)
    clean = [v.clone() for v in s.v], [k.clone() for k in s.k]
    at = [(n - 25, 0, 5, math.inf), (n - 12, 1, hs - 1, math.nan), (n - 12, 1, 0, -math.inf)]
    for pos, h, col, x in at:
        s.v_pages[int(s.table[0, pos // 16]), pos % 16, h, col] = x
        s.v[0][pos, h, col] = 0.0
    s.k_pages[int(s.table[0, (n - 3) // 16]), (n - 3) % 16] = math.nan      # the last three tokens see a NaN logit
    s.cache.attend(s.batch, s.q, s.out)
    ref, tol = s.exact()
    hit = torch.zeros_like(ref, dtype=torch.bool)
    for pos, h, col, _ in at:
        hit[pos - (n - 40):40, 2 * h:2 * h + 2, col] = True
    hit[37:40] = True
    out = s.out.double()
    assert not torch.isfinite(out[hit]).any()
    assert torch.isfinite(out[~hit]).all()
    assert ((out - ref).abs() <= tol)[~hit].all()
    assert torch.isinf(out[15:28, :2, 5]).all() and (out[15:28, :2, 5] > 0).all()


@pytest.mark.parametrize("hs", [32, 48, 64, 96, 128])
def test_fp32_tiles(hs):
    """Rows that fill fp32 tiles and leave one ragged, over splits and pages that are gone."""
    s = setup([(31, 31), (33, 700), (64, 64), (9, 2100), (100, 130)], 6, 2, hs, 16, "f32", "f32", seed=18, drop=[(1, 0), (1, 5), (3, 100)])
    s.cache.attend(s.batch, s.q, s.out)
    s.check()


@pytest.mark.parametrize("bf16", [False, True])
def test_function_ids(bf16):
    """Append and attention, and the norm with its backward, through handles and function ids as a MyCaffe layer calls them."""
    import numpy as np
    from mycaffe_b200 import CudaDnn, function_ids as ids, paged
    from mycaffe_b200.cudadnn import CudaDnnError
    rng = np.random.default_rng(0)
    cuda = CudaDnn(0)
    new = cuda.AllocMemoryBf16 if bf16 else cuda.AllocMemory
    H, KV, D, page, seqs = 4, 2, 64, 16, [(1, 1), (20, 50), (1, 40)]
    need = [-(-n // page) for _, n in seqs]
    pages, T = sum(need), sum(n for n, _ in seqs)
    table = np.full((3, 4), -1, np.int32)
    order = rng.permutation(pages)
    for b, n in enumerate(need):
        table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
    ints = {}
    for name, a in dict(starts=np.cumsum([0] + [n for n, _ in seqs]), lengths=[n for _, n in seqs], table=table).items():
        a = np.ascontiguousarray(a, np.int32)
        ints[name] = cuda.AllocMemory(a.size)
        cuda.SetMemoryInt32(ints[name], a.reshape(-1))
    w = 1 + 0.2 * rng.standard_normal(D).astype(np.float32)
    hw = cuda.AllocMemory(w)
    kv0 = [rng.standard_normal((pages, page, KV, D)).astype(np.float32) for _ in range(2)]
    hK, hV = new(kv0[0]), new(kv0[1])
    q, k, v = (rng.standard_normal((T, h, D)).astype(np.float32) for h in (H, KV, KV))
    hq, hk, hv, hqo, ho = new(q), new(k), new(v), new(q.size), new(q.size)
    hP = cuda.CreatePaged(pages, page, H, KV, D, bf16, 64, 10000.0, ids.MCA_QK_NORM | ids.MCA_ROPE_HALVES)
    args = (hK, hV, ints["starts"], ints["lengths"], ints["table"], 4, 3, T, 20, 50)
    cuda.PagedAppend(hP, hq, hk, hv, hw, hw, *args, hqo)
    cuda.PagedAttention(hP, hqo, *args, ho)
    # the same through the tensors' own calls
    dt = torch.bfloat16 if bf16 else torch.float32
    t = lambda a: torch.tensor(a, device="cuda").to(dt)
    kt, vt = t(kv0[0]), t(kv0[1])
    inv = 10000.0 ** (-np.arange(0, D, 2) / D)
    ang = torch.tensor(np.arange(64)[:, None] * inv[None], device="cuda")
    rot = paged.QkNormRope(ang.cos().float(), ang.sin().float(), torch.tensor(w, device="cuda"), torch.tensor(w, device="cuda"), halves=True)
    cache = paged.PagedCache(kt, vt, H)
    i = lambda a: torch.tensor(np.ascontiguousarray(a, np.int32), device="cuda")
    b = cache.batch(i(np.cumsum([0] + [n for n, _ in seqs])), i([n for _, n in seqs]), i(table), T, 20, 50)
    qo, out = torch.empty(T, H, D, device="cuda", dtype=dt), torch.empty(T, H, D, device="cuda", dtype=dt)
    cache.append(b, rot, t(q), t(k), t(v), qo)
    cache.attend(b, qo, out)
    # the tables differ in their last bits (powf, cosf in fp32 at the library's host): 1e-5 of unit-sized values, or one step of bf16
    tol = 2.0 ** -7 if bf16 else 1e-4
    for h, ref in ((hqo, qo), (hK, kt), (hV, vt), (ho, out)):
        got = cuda.GetMemory(h, ref.numel()).reshape(ref.shape)
        ref = ref.float().cpu().numpy()
        assert np.abs(got - ref).max() <= tol * np.abs(ref).max()
    # a refused sequence comes back as an error, with its number
    cuda.SetMemoryInt32(ints["lengths"], np.array([1, 5, 40], np.int32))
    with pytest.raises(CudaDnnError) as err:
        cuda.PagedAttention(hP, hqo, *args, ho)
    assert err.value.code == ids.ERROR_PARAM_OUT_OF_RANGE and "1 (5)" in err.value.native_message
    cuda.SetAsync(True)
    cuda.PagedAttention(hP, hqo, *args, ho)
    with pytest.raises(CudaDnnError):
        cuda.SynchronizeDevice()
    cuda.SetAsync(False)
    with pytest.raises(CudaDnnError):
        cuda.PagedAttention(hP + 100, hqo, *args, ho)
    with pytest.raises(CudaDnnError):
        cuda.PagedAttention(hP, cuda.AllocMemory(q.size - 4), *args, ho)
    # training form
    B, S = 2, 16
    x = [rng.standard_normal((B, S, h, D)).astype(np.float32) for h in (H, KV, H, KV)]
    hx = [new(a) for a in x]
    hR = cuda.CreateRope(0, 0, x[0].size, B, S, H, D)
    hy, hd = [new(a.size) for a in x[:2]], [new(a.size) for a in x[:2]]
    hdw = [cuda.AllocMemory(D) for _ in range(2)]
    cuda.QkNormRopeForward(hR, hx[0], hx[1], hw, hw, B, S, H, KV, D, *hy)
    cuda.QkNormRopeBackward(hR, hx[0], hx[1], hw, hw, B, S, H, KV, D, hx[2], hx[3], *hd, *hdw)
    tx = [t(a) for a in x]
    rot = paged.QkNormRope(ang.cos().float(), ang.sin().float(), torch.tensor(w, device="cuda"), torch.tensor(w, device="cuda"))
    y, d = [torch.empty_like(a) for a in tx[:2]], [torch.empty_like(a) for a in tx[:2]]
    rot.forward(tx[0], tx[1], *y)
    dw = rot.backward(*tx, *d)
    for h, ref in zip(hy + hd + hdw, y + d + list(dw)):
        got = cuda.GetMemory(h, ref.numel()).reshape(ref.shape)
        ref = ref.float().cpu().numpy()
        assert np.abs(got - ref).max() <= tol * np.abs(ref).max()
    cuda.FreePaged(hP)
    cuda.Dispose()


@pytest.mark.parametrize("hs,page", [(128, 16), (128, 128), (64, 32)])
def test_long_mixed_step_runs_alike(hs, page):
    """Chunks among single tokens over long caches, in which values arrive late: right, and the same bits each time."""
    s = setup([(300, 3300), (219, 2500)] + [(1, 3000 - 190 * b) for b in range(12)], 32, 8, hs, page, "bf16", "bf16", seed=19)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = None
    for _ in range(12):
        flush.zero_()                                  # the pages come from memory, not from the cache
        s.out.fill_(7.0)
        s.cache.attend(s.batch, s.q, s.out)
        first = s.out.clone() if first is None else first
        assert torch.equal(first, s.out)
    s.check()
    assert s.cache.status() == (0, 0, 0, 0)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_pages_beyond_32_bit_offsets(act, cache, new):
    """The same pages at the end of a pool of more than 2^32 bytes give the same bits, through append and attention."""
    from mycaffe_b200 import paged
    s = setup([(new, 300), (1, 130)], 8, 4, 128, 256, act, cache, seed=20)
    rot = paged.QkNormRope(None, None, norm=False)
    k, v = (torch.randn(s.n_tokens, 4, 128, device="cuda").to(s.act) for _ in range(2))
    n, size = s.k_pages.shape[0], s.k_pages.element_size() * s.k_pages[0].numel()
    many = (1 << 32) // size + 64
    big = [torch.empty((many,) + tuple(s.k_pages.shape[1:]), device="cuda", dtype=s.cache_t) for _ in range(2)]
    for b, p in zip(big, (s.k_pages, s.v_pages)):
        b[many - n:] = p
    far = torch.where(s.table >= 0, s.table + (many - n), s.table).to(torch.int32).contiguous()
    wide = paged.PagedCache(big[0], big[1], 8)
    batch = wide.batch(s.starts, s.lengths, far, s.n_tokens, s.max_new, s.max_len)
    q, out = torch.empty_like(s.q), torch.empty_like(s.out)
    wide.append(batch, rot, s.q, k, v, q)
    wide.attend(batch, q, out)
    s.cache.append(s.batch, rot, s.q, k, v, q)
    s.cache.attend(s.batch, q, s.out)
    assert torch.equal(out, s.out) and torch.isfinite(out.float()).all()
    assert wide.status() == (0, 0, 0, 0)
    for b, p in zip(big, (s.k_pages, s.v_pages)):
        assert torch.equal(b[many - n:].nan_to_num(9.0), p.nan_to_num(9.0))


def far_below(s, level):
    """Queries along one direction and keys against it: every scaled logit lies near `level`, far below zero."""
    u = torch.randn(s.kv, s.hs, device="cuda").sign()
    group = s.heads // s.kv
    near = lambda *n: 1.0 + torch.randn(*n, 1, device="cuda") / 64
    s.q.copy_((u.repeat_interleave(group, 0) * near(s.n_tokens, s.heads)).to(s.act))
    for b, (_, n) in enumerate(s.seqs):
        s.k[b] = (u * near(n, s.kv) * (level / math.sqrt(s.hs))).to(s.cache_t)
        for i, page in enumerate(s.table[b].tolist()):
            rows = s.k[b][i * s.page:(i + 1) * s.page]
            if page >= 0 and len(rows):
                s.k_pages[page, : len(rows)] = rows


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("new,seqs,heads", [(1, 1, 4), (1, 400, 4), (40, 1, 2), (40, 40, 2), (300, 1, 4), (300, 12, 4)])
@pytest.mark.parametrize("gone", [[0, 1, 2, 3, 6, 7, 8], [0, 1, 4, 5, 8, 9]])
def test_logits_far_below_zero_behind_pages_that_are_gone(act, cache, hs, new, seqs, heads, gone):
    """A window whose first key tiles are not held, and one in the middle; and every other tile: the softmax of what is left does not
    depend on where the logits lie.  One sequence is shared out over the blocks of the launch, of many each is one block's."""
    n, page = 700, 64
    if seqs == 400:
        n, gone = 330, [0, 1, 2, 3]
    s = setup([(new, n - b % 7) for b in range(seqs)], heads, 1, hs, page, act, cache, seed=21, drop=[(b, i) for b in range(seqs) for i in gone])
    far_below(s, -150.0)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    assert s.cache.status() == (0, 0, 0, 0)


def with_words(s):
    """The setup's cache with status words of its own, and a batch of it."""
    from mycaffe_b200 import paged
    words = torch.zeros(paged.STATUS_WORDS, dtype=torch.int32, device="cuda")
    c = paged.PagedCache(s.k_pages, s.v_pages, s.heads, status=words)
    return c, lambda lengths=s.lengths: c.batch(s.starts, lengths, s.table, s.n_tokens, s.max_new, s.max_len), words


@pytest.mark.parametrize("act,cache", TYPES)
def test_status_words_of_a_cache(act, cache):
    """What a cache with words of its own refuses is told to those who ask it, and to no one else."""
    from mycaffe_b200 import paged
    a, b = (setup([(2, 40), (3, 50)], 4, 2, 64, 16, act, cache, seed=22 + i) for i in range(2))
    (ca, ba, _), (cb, bb, _) = with_words(a), with_words(b)
    bad = torch.tensor([40, 2], device="cuda", dtype=torch.int32)
    rot = paged.QkNormRope(None, None, norm=False)
    k, v = (torch.randn(a.n_tokens, 2, 64, device="cuda").to(a.act) for _ in range(2))
    ca.attend(ba(bad), a.q, a.out)
    cb.attend(bb(), b.q, b.out)
    assert cb.status() == (0, 0, 0, 0) and a.cache.status() == (0, 0, 0, 0)
    assert ca.status() == (1, 1, 2, 1) and ca.status() == (0, 0, 0, 0)
    b.check()
    cb.append(bb(bad), rot, b.q, k, v, torch.empty_like(b.q))
    a.cache.attend(a.cache.batch(a.starts, bad, a.table, a.n_tokens, a.max_new, a.max_len), a.q, a.out)
    assert ca.status() == (0, 0, 0, 0)
    assert cb.status() == (1, 1, 2, 1) and a.cache.status() == (1, 1, 2, 1)


@pytest.mark.parametrize("own", [False, True])
def test_status_says_what_was_refused_first(own):
    """The attention's refusal before the append's, and the other way round; all are counted."""
    from mycaffe_b200 import paged
    s = setup([(2, 40), (3, 50)], 4, 2, 64, 16, "bf16", "bf16", seed=24, drop=[(0, 1)])
    c, batch, _ = with_words(s)
    if not own:
        c, batch = s.cache, lambda n=s.lengths: s.cache.batch(s.starts, n, s.table, s.n_tokens, s.max_new, s.max_len)
    s.table[0, 1] = -7
    bad = torch.tensor([40, 2], device="cuda", dtype=torch.int32)
    rot = paged.QkNormRope(None, None, norm=False)
    k, v = (torch.randn(s.n_tokens, 2, 64, device="cuda").to(s.act) for _ in range(2))
    attend = lambda: c.attend(batch(), s.q, s.out)
    append = lambda: c.append(batch(bad), rot, s.q, k, v, torch.empty_like(s.q))
    attend()
    torch.cuda.synchronize()
    append()
    st = c.status()
    assert st[:3] == (2, 0, -7) and st[3] >= 2
    append()
    torch.cuda.synchronize()
    attend()
    st = c.status()
    assert st[:3] == (1, 1, 2) and st[3] >= 2
    assert c.status() == (0, 0, 0, 0)


def test_function_ids_tell_each_handle_its_own_refusals():
    """Two kernel indices of one device, and two handles of one: a refusal comes back to the caller that made it."""
    import numpy as np
    from mycaffe_b200 import CudaDnn, function_ids as ids
    from mycaffe_b200.cudadnn import CudaDnnError
    rng = np.random.default_rng(0)

    def caller(cuda):
        H, D, page, n = 2, 64, 16, 40
        hP = cuda.CreatePaged(3, page, H, H, D)
        x = [cuda.AllocMemory(rng.standard_normal(m).astype(np.float32)) for m in (n * H * D, 3 * page * H * D, 3 * page * H * D, n * H * D)]
        ints = []
        for a in ([0, n], [n], [0, 1, 2]):
            ints.append(cuda.AllocMemory(len(a)))
            cuda.SetMemoryInt32(ints[-1], np.array(a, np.int32))
        return hP, ints[1], lambda: cuda.PagedAttention(hP, x[0], x[1], x[2], *ints, 3, 1, n, n, n, x[3])

    one, two = CudaDnn(0), CudaDnn(0)
    (hA, lenA, callA), (hB, _, callB), (hC, lenC, callC) = caller(one), caller(two), caller(one)
    one.SetMemoryInt32(lenA, np.array([5], np.int32))
    one.SetAsync(True)
    callA()
    two.SynchronizeDevice()
    callB()                                       # another kernel index: none of its calls was refused
    callC()                                       # another handle of the same one
    with pytest.raises(CudaDnnError) as err:
        one.SynchronizeDevice()
    assert err.value.code == ids.ERROR_PARAM_OUT_OF_RANGE and "0 (5)" in err.value.native_message
    one.SetAsync(False)
    callB(), callC()
    with pytest.raises(CudaDnnError):
        callA()
    one.SetMemoryInt32(lenA, np.array([40], np.int32))
    callA()
    one.SetMemoryInt32(lenC, np.array([3], np.int32))
    one.SetAsync(True)
    callC()
    one.FreePaged(hC)                             # freed before anyone asked
    callA()
    with pytest.raises(CudaDnnError) as err:
        one.SynchronizeDevice()
    assert "0 (3)" in err.value.native_message
    one.SynchronizeDevice()
    two.FreePaged(hB)
    one.Dispose()
    two.Dispose()


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("seqs", [[(2, 5003), (1, 129), (2, 2500)], [(300, 2000), (5, 700), (2, 40)]])
def test_calls_after_a_wait_that_gave_up(act, seqs):
    """With the wait words set (by the self-check's wait, which nothing arrives for) a call touches neither the output nor anything
    else, whatever its workspace holds; once they are read it is right again, and what was refused meanwhile is told after them."""
    import ctypes as C
    from mycaffe_b200 import paged
    s = setup(seqs, 8, 2, 64, 16, act, "bf16", seed=25, pad=3)
    c, batch, words = with_words(s)
    wide = torch.full((s.n_tokens + 8, 10, 64), 7.0, device="cuda", dtype=s.act)
    out = wide[4:-4, 1:9]
    lib, dt = c._lib, paged._DTYPES[s.act]
    shape = tuple(s.q.shape)
    q, o = (paged._heads(t, "t", shape, s.act, t.device) for t in (s.q, out))

    def attend(b, work):
        stream = torch.cuda.current_stream().cuda_stream
        return lib.mca_paged_attention(c._ref, b.ref, dt, C.byref(q), 0.0, C.byref(o), work.data_ptr(), work.numel(), stream)

    b = batch()
    need = lib.mca_paged_attention_workspace_bytes(c._ref, b.ref, dt)
    assert need > 0
    work = torch.ones(need // 4, dtype=torch.int32, device="cuda").view(torch.uint8)   # block 1's row 1 of one row, wherever it is read as such
    assert lib.mca_wait_probe(words.data_ptr() + 16, 1000, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert words.tolist() == [0, 0, 0, 0, 1, 99, 0, 0]
    assert attend(b, work) == 0
    torch.cuda.synchronize()
    assert (wide == 7.0).all()
    bad = s.lengths.clone()
    bad[1] = seqs[1][1] + s.max_len
    assert attend(batch(bad), work) == 0
    assert c.status() == (4, 99, 0, 1)
    rows = slice(4 + seqs[0][0], 4 + seqs[0][0] + seqs[1][0])
    assert not wide[rows, 1:9].any()                   # a refused sequence's rows are zeros as ever
    wide[rows, 1:9] = 7.0
    assert (wide == 7.0).all()
    assert c.status() == (1, 1, seqs[1][1] + s.max_len, 1) and c.status() == (0, 0, 0, 0)
    assert attend(b, work) == 0
    s.out = out.contiguous()
    s.check()
    wide[4:-4, 1:9] = 7.0
    assert (wide == 7.0).all() and c.status() == (0, 0, 0, 0)


@pytest.mark.parametrize("act,cache,heads,new", [("f32", "f32", 2, 1), ("f32", "f32", 4, 1), ("f32", "f32", 8, 1), ("f32", "f32", 4, 40),
                                                 ("f32", "bf16", 2, 1), ("bf16", "bf16", 4, 1), ("bf16", "bf16", 4, 40)])
@pytest.mark.parametrize("n", [100, 1500])
def test_logits_of_minus_infinity_weigh_nothing(act, cache, heads, new, n):
    """Keys whose logits are minus infinity, met first, in between and alone, through each of the kernels."""
    s = setup([(new, n), (new, n), (new, new)], heads, 2, 64, 16, act, cache, seed=26)
    s.q[..., 3] = s.q[..., 3].abs() + 0.125
    for b, at in enumerate([list(range(21)) + [40, 41, 57, 90], list(range(0, n, 2)), range(new)]):
        for pos in at:
            s.k_pages[int(s.table[b, pos // 16]), pos % 16, :, 3] = -math.inf
            s.held[b][pos] = False
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    assert not s.out[2 * new:].any()


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("heads,kv", [(65, 1), (71, 1), (129, 1), (142, 1), (300, 2)])
@pytest.mark.parametrize("seqs", [[(1, 700), (1, 1), (1, 130)], [(1, 2), (5, 300), (20, 20)]])
def test_more_heads_to_a_key_than_a_tile_has_rows(act, cache, heads, kv, seqs):
    """The query heads that share a key fill more than one tile: parts of the group, whole and ragged."""
    s = setup(seqs, heads, kv, 32, 16, act, cache, seed=27, pad=2, drop=[(0, 0)] if seqs[0][1] > 16 else ())
    s.cache.attend(s.batch, s.q, s.out)
    s.check()
    assert s.cache.status() == (0, 0, 0, 0)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("heads,kv", [(5, 1), (14, 2), (21, 3), (24, 2)])
def test_groups_that_do_not_divide_a_tile(act, cache, heads, kv):
    s = setup([(1, 900), (150, 400), (33, 33), (2, 129)], heads, kv, 128, 32, act, cache, seed=28)
    s.cache.attend(s.batch, s.q, s.out)
    s.check()


def test_a_pool_of_more_elements_than_64_bits_count_is_refused():
    """Its size would wrap, and handles that are far too small would pass for its pages."""
    from mycaffe_b200 import CudaDnn, function_ids as ids
    from mycaffe_b200.cudadnn import CudaDnnError
    cuda = CudaDnn(0)
    with pytest.raises(CudaDnnError) as err:
        cuda.CreatePaged(1 << 26, 1 << 16, 1 << 15, 1 << 15, 128)      # 2^64 elements
    assert err.value.code == ids.ERROR_PARAM_OUT_OF_RANGE
    cuda.FreePaged(cuda.CreatePaged(1 << 24, 1 << 16, 1 << 15, 1 << 15, 128))   # 2^62
    cuda.Dispose()


def test_the_message_belongs_to_the_error_that_is_returned():
    """A wait that gave up and a refused sequence, both in asynchronous mode: the code is the first's, and so is the text."""
    import numpy as np
    from mycaffe_b200 import CudaDnn, function_ids as ids
    from mycaffe_b200.cudadnn import CudaDnnError
    cuda = CudaDnn(0)
    H, D, page, n = 2, 64, 16, 40
    hCudnn = cuda.CreateCuDNN()
    hAttn = cuda.CreateAttn()
    cuda.SetAttn(hCudnn, hAttn, 0, True, 1, 256, 2, 64, 0.0, 0, ids.MCA_DTYPE_BF16, ids.MCA_FLAG_CAUSAL_IMPLICIT)
    hP = cuda.CreatePaged(3, page, H, H, D)
    x = [cuda.AllocMemory(np.ones(m, np.float32)) for m in (n * H * D, 3 * page * H * D, 3 * page * H * D, n * H * D)]
    ints = []
    for a in ([0, n], [5], [0, 1, 2]):
        ints.append(cuda.AllocMemory(len(a)))
        cuda.SetMemoryInt32(ints[-1], np.array(a, np.int32))
    cuda.SetAsync(True)
    cuda._invoke(ids.MCA_FN_WAIT_PROBE, None, [hAttn, 1000])
    cuda.PagedAttention(hP, x[0], x[1], x[2], *ints, 3, 1, n, n, n, x[3])
    with pytest.raises(CudaDnnError) as err:
        cuda.SynchronizeDevice()
    assert err.value.code == ids.ERROR_ATTN_KERNEL_TIMEOUT
    assert "stage 99" in err.value.native_message and "lengths" not in err.value.native_message
    cuda.SynchronizeDevice()
    cuda.Dispose()
