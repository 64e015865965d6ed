"""What the paged-cache and norm entry points refuse, before any device is touched."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from mycaffe_b200 import build, _lib
    build.build()
    return _lib.load()


OUT_OF_RANGE, NULL, SHAPE, SMALL = 90001, 90002, 90901, 90905
A = 0x10000   # an aligned address that nothing reads


def cache(**k):
    from mycaffe_b200.paged import McaPagedCache
    d = dict(k_pages=A, v_pages=A, page_stride=16 * 2 * 64, n_pages=4, page_size=16, n_heads=4, n_kv_heads=2, head_size=64, dtype=2)
    return McaPagedCache(**{**d, **k})


def batch(**k):
    from mycaffe_b200.paged import McaPagedBatch
    d = dict(starts=A, lengths=A, page_table=A, table_stride=4, n_seqs=2, n_tokens=3, max_new=2, max_len=64)
    return McaPagedBatch(**{**d, **k})


def heads(n, **k):
    from mycaffe_b200.paged import McaHeads
    return McaHeads(**{**dict(data=A, stride_b=0, stride_t=n * 64, stride_h=64), **k})


def rotation(**k):
    from mycaffe_b200.paged import McaQkRotation
    return McaQkRotation(**{**dict(q_weight=None, k_weight=None, cos_table=A, sin_table=A, table_len=64, flags=1, eps=1e-5), **k})


def attend(lib, c=None, b=None, dtype=2, q=None, out=None, scale=0.0, work=A, size=1 << 30):
    c, b = cache() if c is None else c, batch() if b is None else b
    q, out = heads(4) if q is None else q, heads(4) if out is None else out
    return lib.mca_paged_attention(C.byref(c), C.byref(b), dtype, C.byref(q), scale, C.byref(out), work, size, None)


CACHE = [(dict(k_pages=None), NULL), (dict(v_pages=None), NULL), (dict(dtype=1), SHAPE), (dict(head_size=80), SHAPE), (dict(n_pages=0), OUT_OF_RANGE),
         (dict(n_heads=3), OUT_OF_RANGE), (dict(n_heads=0), OUT_OF_RANGE), (dict(n_kv_heads=0), OUT_OF_RANGE), (dict(page_size=24), OUT_OF_RANGE),
         (dict(page_size=8), OUT_OF_RANGE), (dict(page_size=1 << 17), OUT_OF_RANGE), (dict(page_stride=16 * 2 * 64 - 8), OUT_OF_RANGE),
         (dict(page_stride=16 * 2 * 64 + 4), OUT_OF_RANGE), (dict(k_pages=A + 8), OUT_OF_RANGE)]
BATCH = [(dict(starts=None), NULL), (dict(lengths=None), NULL), (dict(page_table=None), NULL), (dict(n_seqs=0), OUT_OF_RANGE),
         (dict(n_seqs=70000), OUT_OF_RANGE), (dict(n_tokens=-1), OUT_OF_RANGE), (dict(max_new=0), OUT_OF_RANGE), (dict(max_len=0), OUT_OF_RANGE),
         (dict(max_len=65), OUT_OF_RANGE), (dict(table_stride=0), OUT_OF_RANGE), (dict(lengths=A + 2), OUT_OF_RANGE)]


@pytest.mark.parametrize("change,code", CACHE)
def test_cache_descriptors(lib, change, code):
    c, b, r = cache(**change), batch(), rotation()
    assert attend(lib, c=c) == code
    assert lib.mca_paged_attention_workspace_bytes(C.byref(c), C.byref(b), 2) == -1
    q, k = heads(4), heads(2)
    assert lib.mca_paged_append(C.byref(c), C.byref(b), C.byref(r), 2, C.byref(q), C.byref(k), C.byref(k), C.byref(q), None) == code


@pytest.mark.parametrize("change,code", BATCH)
def test_batch_descriptors(lib, change, code):
    c, b, r = cache(), batch(**change), rotation()
    assert attend(lib, b=b) == code
    assert lib.mca_paged_attention_workspace_bytes(C.byref(c), C.byref(b), 2) == -1
    q, k = heads(4), heads(2)
    assert lib.mca_paged_append(C.byref(c), C.byref(b), C.byref(r), 2, C.byref(q), C.byref(k), C.byref(k), C.byref(q), None) == code


def test_attention_arguments(lib):
    f32 = cache(dtype=0)
    assert attend(lib, c=f32, dtype=2) == SHAPE                     # bf16 activations over fp32 pages
    assert attend(lib, dtype=1) == SHAPE
    assert attend(lib, scale=-1.0) == OUT_OF_RANGE
    assert attend(lib, scale=float("nan")) == OUT_OF_RANGE
    assert attend(lib, scale=float("inf")) == OUT_OF_RANGE
    assert attend(lib, q=heads(4, data=None)) == NULL
    assert attend(lib, out=heads(4, data=A + 8)) == OUT_OF_RANGE
    assert attend(lib, q=heads(4, stride_t=258)) == OUT_OF_RANGE
    assert attend(lib, out=heads(4, stride_h=68)) == OUT_OF_RANGE
    assert lib.mca_paged_attention(None, None, 2, None, 0.0, None, None, 0, None) == NULL
    long = batch(table_stride=4096, max_len=65536)
    c = cache()
    need = lib.mca_paged_attention_workspace_bytes(C.byref(c), C.byref(long), 2)
    assert need > 0
    assert attend(lib, b=long, work=None) == SMALL
    assert attend(lib, b=long, size=need - 1) == SMALL
    assert attend(lib, b=long, work=A + 4) == OUT_OF_RANGE
    assert attend(lib, b=batch(n_tokens=0)) == 0                    # no rows: nothing to do
    assert lib.mca_paged_status(None) == NULL


def test_workspace_is_bounded_by_the_machine(lib):
    """bf16 pages: two parts for each block of the launch, whatever the lengths."""
    c = cache(n_heads=32, n_kv_heads=8, head_size=128, page_stride=16 * 8 * 128)
    sizes = {n: lib.mca_paged_attention_workspace_bytes(C.byref(c), C.byref(batch(n_seqs=64, n_tokens=64, max_new=1, table_stride=1 << 16, max_len=n)), 2)
             for n in (128, 129, 4096, 1 << 20)}
    assert sizes[128] == 0 < sizes[129] <= sizes[4096] == sizes[1 << 20] <= 148 * (2 * 4 * 130 * 4 + 32)


def norm(lib, r=None, dtype=0, B=1, T=8, H=2, KV=1, D=64, q=None, k=None, qo=None, ko=None, pos=None):
    r = rotation() if r is None else r
    v = [heads(2) if q is None else q, heads(1) if k is None else k, heads(2) if qo is None else qo, heads(1) if ko is None else ko]
    return lib.mca_qk_norm_rope_forward(C.byref(r), C.byref(v[0]), C.byref(v[1]), pos, dtype, B, T, H, KV, D, C.byref(v[2]), C.byref(v[3]), None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=1), SHAPE), (dict(D=8), SHAPE), (dict(D=72), SHAPE), (dict(D=272), SHAPE), (dict(B=0), OUT_OF_RANGE), (dict(T=0), OUT_OF_RANGE),
    (dict(T=65), OUT_OF_RANGE), (dict(H=0), OUT_OF_RANGE), (dict(KV=-1), OUT_OF_RANGE), (dict(pos=A + 2), OUT_OF_RANGE),
    (dict(B=1 << 20, T=64, H=64), OUT_OF_RANGE)])
def test_norm_arguments(lib, change, code):
    assert norm(lib, **change) == code


def test_norm_views_and_rotation(lib):
    assert norm(lib, q=heads(2, data=None)) == NULL
    assert norm(lib, ko=heads(1, stride_t=66)) == OUT_OF_RANGE
    assert norm(lib, k=heads(1, stride_b=2)) == OUT_OF_RANGE
    for change, code in [(dict(sin_table=None), NULL), (dict(table_len=0), OUT_OF_RANGE), (dict(flags=4), OUT_OF_RANGE), (dict(eps=-1.0), OUT_OF_RANGE),
                         (dict(eps=float("nan")), OUT_OF_RANGE), (dict(flags=0, q_weight=A), OUT_OF_RANGE), (dict(k_weight=A + 4), OUT_OF_RANGE),
                         (dict(cos_table=A + 8), OUT_OF_RANGE)]:
        assert norm(lib, r=rotation(**change)) == code, change
    assert lib.mca_qk_norm_rope_forward(None, None, None, None, 0, 1, 1, 1, 1, 64, None, None, None) == NULL


def test_norm_backward_arguments(lib):
    r, a, b = rotation(q_weight=A, k_weight=A), heads(2), heads(1)

    def call(dq=A, dk=A, scratch=A, n=1 << 20, r=r, KV=1):
        return lib.mca_qk_norm_rope_backward(C.byref(r), C.byref(a), C.byref(b), None, C.byref(a), C.byref(b), 0, 1, 8, 2, KV, 64, C.byref(a), C.byref(b),
                                             dq, dk, scratch, n, None)
    need = lib.mca_qk_norm_rope_backward_scratch_floats(64)
    assert need > 0 and lib.mca_qk_norm_rope_backward_scratch_floats(40) == -1
    assert call(scratch=None) == NULL
    assert call(n=need - 1) == SMALL
    assert call(r=rotation(flags=0)) == OUT_OF_RANGE                 # a weight's gradient without the norm
    assert call(KV=0) == OUT_OF_RANGE                                # a key weight's gradient without keys
    assert call(dq=A + 2) == OUT_OF_RANGE


def test_python_checks():
    torch = pytest.importorskip("torch")
    from mycaffe_b200 import paged
    k = torch.zeros(4, 16, 2, 64)
    with pytest.raises(ValueError):
        paged.PagedCache(k, torch.zeros(4, 16, 2, 32), 4)
    with pytest.raises(ValueError):
        paged.PagedCache(k, k.transpose(1, 2).contiguous().transpose(1, 2), 4)
    with pytest.raises(TypeError):
        paged.PagedCache(k.half(), k.half(), 4)
    c = paged.PagedCache(k, k.clone(), 4)
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)
    c.batch(i(3), i(2), i(2, 4), 3, 2, 64)
    for bad in [(i(2), i(2), i(2, 4)), (i(3).long(), i(2), i(2, 4)), (i(3), i(2), i(3, 4)), (i(3), i(2), i(2, 8)[:, ::2])]:
        with pytest.raises(ValueError):
            c.batch(*bad, 3, 2, 64)
    with pytest.raises(ValueError):
        paged.QkNormRope(torch.zeros(8, 32), None)
    with pytest.raises(ValueError):
        paged.QkNormRope(torch.zeros(8, 32), torch.zeros(8, 16))
    with pytest.raises(ValueError):
        paged.QkNormRope(torch.zeros(8, 32), torch.zeros(8, 32), torch.ones(32))
    r = paged.QkNormRope(torch.zeros(8, 32), torch.zeros(8, 32))
    with pytest.raises(ValueError):
        r.check(128, k.device)


def test_status_words(lib):
    """A cache's own status words: 16-byte aligned, and asked for by their address."""
    st = (C.c_int * 4)()
    assert lib.mca_paged_status_of(None, st) == NULL and lib.mca_paged_status_of(A, None) == NULL
    assert lib.mca_paged_status_of(A + 4, st) == OUT_OF_RANGE
    c, b = cache(status=A + 4), batch()
    assert attend(lib, c=c) == OUT_OF_RANGE
    assert lib.mca_paged_attention_workspace_bytes(C.byref(c), C.byref(b), 2) == -1
    assert lib.mca_paged_attention_workspace_bytes(C.byref(cache(status=A)), C.byref(b), 2) == lib.mca_paged_attention_workspace_bytes(
        C.byref(cache()), C.byref(b), 2)


def test_status_words_of_a_tensor():
    torch = pytest.importorskip("torch")
    from mycaffe_b200 import paged
    k = torch.zeros(4, 16, 2, 64)
    words = torch.zeros(paged.STATUS_WORDS, dtype=torch.int32)
    assert paged.PagedCache(k, k.clone(), 4, status=words).c.status == words.data_ptr()
    assert paged.PagedCache(k, k.clone(), 4).c.status is None
    for bad in (words[:4], words.long(), torch.zeros(16, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            paged.PagedCache(k, k.clone(), 4, status=bad)


def test_scales(lib):
    """Zero is the C side's default; what is not a positive factor in powers of two is refused, and by the tensors' call zero too."""
    for bad in (-0.125, -1e-45, 1e-45, 1e-38 / 2, 2.5e38, 3.4e38, float("inf"), float("nan")):
        assert attend(lib, scale=bad) == OUT_OF_RANGE, bad
    b = batch(n_tokens=0)
    for good in (0.0, -0.0, 1e-37, 2.3e38):
        assert attend(lib, b=b, scale=good) == 0, good
    torch = pytest.importorskip("torch")
    from mycaffe_b200 import paged
    k = torch.zeros(4, 16, 2, 64)
    c = paged.PagedCache(k, k.clone(), 4)
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)
    b, q = c.batch(i(3), i(2), i(2, 4), 3, 2, 64), torch.zeros(3, 4, 64)
    for bad in (0.0, -0.125, float("nan")):
        with pytest.raises(ValueError):
            c.attend(b, q, q.clone(), scale=bad)


def test_a_batch_of_another_device_is_refused():
    torch = pytest.importorskip("torch")
    from mycaffe_b200 import paged
    k, far = torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64, device="meta")
    c, other = paged.PagedCache(k, k.clone(), 4), paged.PagedCache(far, far.clone(), 4)
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)
    b = c.batch(i(3), i(2), i(2, 4), 3, 2, 64)
    q, kv = torch.zeros(3, 4, 64, device="meta"), torch.zeros(3, 2, 64, device="meta")
    with pytest.raises(ValueError, match="batch"):
        other.attend(b, q, q.clone())
    with pytest.raises(ValueError, match="batch"):
        other.append(b, paged.QkNormRope(None, None), q, kv, kv, q.clone())


def test_norm_rows_beyond_31_bits(lib):
    """B x T x heads is bounded where it does not wrap, too: (2^31 - 1)^2 x 4 is negative in 64 bits."""
    r, q, k = rotation(), heads(4), heads(2)
    call = lambda B, T, H, KV: lib.mca_qk_norm_rope_forward(C.byref(r), C.byref(q), C.byref(k), A, 2, B, T, H, KV, 64, C.byref(q), C.byref(k), None)
    most = (1 << 31) - 1
    for B, T, H, KV in [(most, most, 4, 2), (most, most, 2, 4), (1 << 16, 1 << 15, 1, 1), (1 << 16, 1 << 14, 2, 1), (1 << 16, 1 << 14, 1, 2), (1, most, 3, 0)]:
        assert call(B, T, H, KV) == OUT_OF_RANGE, (B, T, H, KV)


def test_outputs_whose_rows_lie_on_one_another_are_refused():
    """An expanded tensor is an input like any other; as an output its rows would race for the same memory."""
    torch = pytest.importorskip("torch")
    from mycaffe_b200 import paged
    k = torch.zeros(4, 16, 2, 64)
    c = paged.PagedCache(k, k.clone(), 4)
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)
    b, q, kv = c.batch(i(3), i(2), i(2, 4), 3, 2, 64), torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    rot = paged.QkNormRope(None, None)
    refused = lambda what: pytest.raises(ValueError, match=f"{what}: an expanded")
    for out in (torch.zeros(1, 4, 64).expand(3, 4, 64), torch.zeros(3, 1, 64).expand(3, 4, 64)):
        with refused("out"):
            c.attend(b, q, out)
        with refused("q_out"):
            c.append(b, rot, q, kv, kv, out)
        x, y, wide = q[None], kv[None], out[None]
        with refused("q_out"):
            rot.forward(x, y, wide, y.clone())
        with refused("k_out"):
            rot.forward(x, y, x.clone(), torch.zeros(1, 3, 1, 64).expand(1, 3, 2, 64))
        with refused("dq"):
            rot.backward(x, y, out[None], y, wide, y.clone())
        with refused("dk"):
            rot.backward(x, y, wide, y, x.clone(), torch.zeros(1, 1, 2, 64).expand(1, 3, 2, 64))
