"""b200_paged_append against its definition in 64 bits: every value is computed in F32 (two products, one sum) and rounded once."""
import importlib

import numpy as np
import pytest

import b200
import plain_paged as P

pytestmark = pytest.mark.gpu
GUARD = 64   # elements behind every output, which stay as they were


@pytest.fixture(scope="module")
def p():
    b200.load()
    return importlib.import_module("llama_rust_b200.paged")


def device(a):
    return b200.load().device_array(a)


def run(p, ty="F16", xt="F32", page=16, kv=2, heads=4, d=64, n_dims=None, mode=2, pos=(0,), seq=None, n_seq=2, table_pages=6, seed=0, bad=None, pad=0, stride_gap=0, off=0, rope_rows=128, page_gap=0):
    """pad: extra elements between tokens; off: elements that the inputs begin behind an aligned address"""
    m = b200.load()
    rng = np.random.default_rng(seed)
    n, n_dims = len(pos), d if n_dims is None else n_dims
    TY = {"F32": p.F32, "F16": p.F16, "BF16": p.BF16}
    n_pages = n_seq * table_pages + 1
    tables = rng.permutation(n_pages)[: n_seq * table_pages].reshape(n_seq, table_pages).astype(np.int32)
    if bad:
        tables[bad[0], bad[1]] = bad[2]
    seqs = list(range(n)) if seq is None else list(seq)
    pages = [P.rounded(rng.standard_normal((n_pages, page, kv, d)), ty) for _ in range(2)]
    x = {name: P.rounded(rng.standard_normal((n, h, d)) * 2, xt) for name, h in (("q", heads), ("k", kv), ("v", kv))}
    rows = P.rope_rows(rope_rows, d, n_dims)
    want = P.append(pages[0], pages[1], tables.tolist(), x["q"], x["k"], x["v"], list(pos), seqs, rows, n_dims, mode)
    size = 4 if xt == "F32" else 2

    def strided(a):   # tokens h * d + pad elements apart, `off` elements into the buffer
        flat = np.zeros((n, a.shape[1] * d + pad))
        flat[:, : a.shape[1] * d] = a.reshape(n, -1)
        return device(P.bits(np.concatenate([np.zeros(off), flat.reshape(-1)]), xt))

    dx = {k: strided(a) for k, a in x.items()}
    page_elems = page * kv * d + page_gap
    store = []
    for a in pages:
        flat = np.full((n_pages, page_elems), -7.0)
        flat[:, : page * kv * d] = a.reshape(n_pages, -1)
        store.append(device(P.bits(flat, ty)))
    dq = device(P.bits(np.full(n * heads * d + GUARD, -7.0), ty))
    keep = [device(tables), device(np.array(pos, dtype=np.int32)), device(np.array(seqs, dtype=np.int32)), device(rows)]
    cache = p.Cache(TY[ty], page, n_pages, kv, d, store[0].ptr, store[1].ptr, keep[0].ptr, table_pages, n_seq, page_stride=page_elems * 2 if page_gap else 0)
    st = {k: ((h * d + pad) * size, d * size) for k, h in (("q", heads), ("k", kv), ("v", kv))}
    p.Append(cache, n, TY[xt], dx["k"].ptr + off * size, dx["v"].ptr + off * size, keep[1].ptr, seq=None if seq is None else keep[2].ptr, q=dx["q"].ptr + off * size if heads else None,
             q_out=dq.ptr if heads else None, n_head=heads, rope=keep[3].ptr, rope_rows=rope_rows, n_dims=n_dims, mode=mode, k_strides=st["k"], v_strides=st["v"], q_strides=st["q"])(None)
    m.synchronize()
    assert m.kernel_error() == (7 if want[5] else 0)
    # two products and their sum in F32: three roundings of at most 2^-24 of the magnitudes; then half a step of the type
    def near(got, exact, size, touched):
        tol = P.HALF_STEP[ty] * (np.abs(exact) + 2.0 ** -22 * size) + 2.0 ** -22 * size + P.SMALLEST[ty]
        assert (np.abs(got - exact)[touched] <= tol[touched]).all(), np.nanmax((np.abs(got - exact) / tol)[touched])

    got_q = P.values(dq.download(np.uint16, n * heads * d + GUARD), ty)
    assert (got_q[n * heads * d:] == -7.0).all()
    got_q = got_q[: n * heads * d].reshape(n, heads, d)
    untouched = np.isnan(want[0])
    assert (got_q[untouched] == -7.0).all()
    near(got_q, np.where(untouched, 0.0, want[0]), want[3], ~untouched)
    for which, exact, mag in ((0, want[1], want[4]), (1, want[2], np.zeros(want[2].shape))):
        got = P.values(store[which].download(np.uint16, n_pages * page_elems), ty).reshape(n_pages, page_elems)
        assert (got[:, page * kv * d:] == -7.0).all()
        got = got[:, : page * kv * d].reshape(exact.shape)
        moved = exact != pages[which]
        assert np.array_equal(got[~moved], pages[which][~moved])
        near(got, exact, mag, moved)
    return got_q


@pytest.mark.parametrize("ty", ["F16", "BF16"])
@pytest.mark.parametrize("xt", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("mode", [0, 2])
def test_types_and_modes(p, ty, xt, mode):
    run(p, ty, xt, mode=mode, pos=[5, 16, 31, 0, 95], seq=[0, 1, 0, 1, 1], d=128)


@pytest.mark.parametrize("d,n_dims", [(64, 32), (64, 0), (128, 16), (16, 16), (48, 32), (80, 80), (128, 10), (96, 2), (1024, 512), (64, 62)])
@pytest.mark.parametrize("mode", [0, 2])
def test_head_sizes_and_partial_rotation(p, d, n_dims, mode):
    run(p, d=d, n_dims=n_dims, mode=mode, pos=[3, 40, 17], seq=[0, 1, 1])


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kv,heads", [(1, 1), (8, 32), (3, 0), (2, 14), (16, 16)])
def test_pages_and_heads(p, page, kv, heads):
    run(p, "BF16", page=page, kv=kv, heads=heads, pos=[page - 1, page, 0, 1, 2 * page + 3], seq=[0, 0, 1, 1, 0], table_pages=3, rope_rows=3 * page)


@pytest.mark.parametrize("n", [1, 2, 63, 300])
def test_one_token_to_a_prompt(p, n):
    run(p, pos=list(range(n)), seq=[1] * n, n_seq=2, table_pages=20, rope_rows=512)


def test_sequences_may_be_implied(p):
    run(p, pos=[9, 0, 33], n_seq=3)


@pytest.mark.parametrize("pad,off", [(4, 0), (3, 0), (0, 1), (1, 3), (8, 8)])
@pytest.mark.parametrize("xt", ["F32", "BF16"])
def test_strides_and_unaligned_rows(p, xt, pad, off):
    run(p, "BF16", xt, pos=[0, 20, 21], seq=[0, 1, 1], pad=pad, off=off)


def test_pages_with_something_between_them(p):
    run(p, pos=[0, 20, 95], seq=[0, 1, 1], page_gap=64)


def test_padding_tokens_leave_everything(p):
    run(p, pos=[-1, 4, -5, -1], seq=[0, 1, 9, -3])


@pytest.mark.parametrize("kw", [dict(pos=[1, 96], seq=[0, 1]), dict(pos=[1, 2], seq=[0, 2]), dict(pos=[1, 2], seq=[-1, 0]), dict(pos=[20, 40], seq=[0, 1], bad=(1, 2, 13)), dict(pos=[20, 40], seq=[0, 1], bad=(1, 2, -1)),
                                dict(pos=[20, 40], seq=[0, 1], rope_rows=40)])
def test_what_has_no_place_is_left_out_and_reported(p, kw):
    run(p, **kw)


def test_infinities_and_nan_reach_their_own_cells_only(p):
    m = b200.load()
    x = np.ones((2, 1, 64), dtype=np.float32)
    x[0, 0, 3], x[0, 0, 40] = np.inf, np.nan
    pages = device(np.zeros((4, 16, 1, 64), dtype=np.uint16))
    keep = [device(x), device(np.array([3, 5], dtype=np.int32)), device(np.zeros(2, dtype=np.int32)), device(np.arange(4, dtype=np.int32)), device(P.rope_rows(16, 64, 64))]
    cache = p.Cache(p.F16, 16, 4, 1, 64, pages.ptr, pages.ptr, keep[3].ptr, 4, 1)
    p.Append(cache, 2, p.F32, keep[0].ptr, keep[0].ptr, keep[1].ptr, seq=keep[2].ptr, rope=keep[4].ptr, rope_rows=16, n_dims=0)(None)
    got = pages.download(np.uint16, 4 * 16 * 64).view(np.float16).reshape(4, 16, 64)
    assert np.isinf(got[0, 3, 3]) and np.isnan(got[0, 3, 40]) and np.isfinite(got).sum() == got.size - 2 and (got[0, 5] == 1).all()
    assert m.kernel_error() == 0


def test_queries_may_be_turned_in_place(p):
    m = b200.load()
    rng = np.random.default_rng(4)
    q = P.rounded(rng.standard_normal((5, 4, 64)), "BF16")
    rows, pos = P.rope_rows(64, 64, 64), [7, 0, 63, 20, 33]
    dq, dk, pages = device(P.bits(q, "BF16")), device(P.bits(q, "BF16")), device(np.zeros((10, 16, 4, 64), dtype=np.uint16))
    keep = [device(np.array(pos, dtype=np.int32)), device(np.arange(10, dtype=np.int32).reshape(5, 2).repeat(2, 1)), device(rows)]
    cache = p.Cache(p.BF16, 16, 10, 4, 64, pages.ptr, pages.ptr, keep[1].ptr, 4, 5)
    p.Append(cache, 5, p.BF16, dk.ptr, dk.ptr, keep[0].ptr, q=dq.ptr, q_out=dq.ptr, n_head=4, rope=keep[2].ptr, rope_rows=64, n_dims=64)(None)
    got = P.values(dq.download(np.uint16, q.size), "BF16").reshape(q.shape)
    for t in range(5):
        want, size = P.rotated(q[t], rows[pos[t]], 64, 2)
        assert (np.abs(got[t] - want) <= P.HALF_STEP["BF16"] * (np.abs(want) + 2.0 ** -22 * size) + 2.0 ** -22 * size).all()
    assert m.kernel_error() == 0
