"""What the operators over a paged cache refuse before anything touches a device, and the sizes of their workspaces: host arithmetic only."""
import ctypes as C
import importlib

import pytest

import b200


@pytest.fixture(scope="module")
def p():
    b200.load()
    return importlib.import_module("llama_rust_b200.paged")


A = 1 << 20   # an address that nobody reads here


def cache_of(p, **kw):
    a = dict(ty=p.F16, page_size=16, n_pages=8, n_head_kv=2, d=64, k=A, v=A, tables=A, table_ld=4, n_seq=4)
    a.update(kw)
    return p.Cache(**a)


def append_of(p, cache=None, **kw):
    a = dict(n_tok=3, x_type=p.F32, k=A, v=A, pos=A, seq=A, q=A, q_out=A, n_head=4, rope=A, rope_rows=64, n_dims=64, mode=p.NEOX)
    a.update(kw)
    return p.Append(cache or cache_of(p), **a)


def attn_of(p, cache=None, **kw):
    a = dict(n_seq=4, n_head=4, q=A, dst=A, lens=A, scale=0.125, shared=A, group_first=A, n_group=1, max_len=64, max_shared=32, max_group=4, workspace=(A, 1 << 30))
    a.update(kw)
    return p.PrefixAttn(cache or cache_of(p), **a)


def select_of(p, **kw):
    a = dict(logits_type=p.F32, n_request=2, n_beam=4, n_vocab=1000, k=8, logits=A, scores=A, out_scores=A, out_tokens=A, out_parents=A, workspace=(A, 1 << 30))
    a.update(kw)
    return p.BeamSelect(**a)


def reorder_of(p, **kw):
    a = dict(n_request=2, n_beam=4, parents=A, tables_in=2 * A, tables_out=3 * A, table_ld=4, lens_in=4 * A, lens_out=5 * A, row_of=6 * A, page_size=16, n_pages=8, page_bytes=4096, pools=[8 * A])
    a.update(kw)
    return p.BeamReorder(**a)


def refused(call, words):
    with pytest.raises(Exception) as e:
        call(None)
    assert words in str(e.value) and "status 3" in str(e.value), str(e.value)


@pytest.mark.parametrize("kw,words", [
    (dict(ty=0), "neither F16 nor BF16"), (dict(page_size=8), "pages of 8"), (dict(page_size=48), "pages of 48"), (dict(page_size=512), "pages of 512"), (dict(n_head_kv=0), "key heads"), (dict(d=72), "72 channels"),
    (dict(d=2048), "2048 channels"), (dict(d=0), "0 channels"), (dict(k=None), "null cache"), (dict(v=A + 8), "16-byte aligned"), (dict(tables=None), "null cache"), (dict(n_pages=0), "empty"),
    (dict(table_ld=0), "empty"), (dict(table_ld=1 << 31), "too large"), (dict(page_stride=1 << 40), "page stride"), (dict(n_seq=0), "empty"), (dict(page_stride=2048), "page stride"), (dict(page_stride=16 * 256 + 8), "page stride")])
def test_cache_arguments(p, kw, words):
    refused(append_of(p, cache_of(p, **kw)), words)
    refused(attn_of(p, cache_of(p, **kw)), words)


@pytest.mark.parametrize("kw,words", [
    (dict(x_type=8), "input type"), (dict(n_tok=-1), "tokens"), (dict(n_head=-1), "query heads"), (dict(n_dims=33), "rotating channels"), (dict(n_dims=128), "rotating channels"), (dict(mode=1), "mode 1"),
    (dict(pos=None), "null operand"), (dict(k=None), "null operand"), (dict(q_out=None), "null operand"), (dict(rope=None), "needs its table"), (dict(rope_rows=0), "needs its table"), (dict(rope_ld=32), "needs its table"),
    (dict(k=A + 2), "aligned to their elements"), (dict(q_out=A + 1), "aligned to their elements"), (dict(v_strides=(514, 256)), "aligned to their elements")])
def test_append_arguments(p, kw, words):
    refused(append_of(p, **kw), words)


@pytest.mark.parametrize("kw,words", [
    (dict(n_seq=5), "tables for 4"), (dict(n_seq=-1), "rows"), (dict(n_head=5), "over 2 key heads"), (dict(n_head=0), "heads"), (dict(n_group=5), "5 groups"), (dict(n_group=-1), "groups"), (dict(max_len=-1), "negative"),
    (dict(scale=float("nan")), "not finite"), (dict(scale=float("inf")), "not finite"), (dict(q=None), "null operand"), (dict(lens=None), "null operand"), (dict(shared=None), "null operand"), (dict(q=A + 8), "16 bytes"),
    (dict(dst_strides=(520, 128)), "16 bytes"), (dict(workspace=(A, 100)), "workspace"), (dict(workspace=(A + 16, 1 << 30)), "workspace"), (dict(workspace=(None, 1 << 30)), "workspace")])
def test_attention_arguments(p, kw, words):
    refused(attn_of(p, **kw), words)


def test_attention_head_sizes(p):
    for d in (16, 80, 96, 256):
        refused(attn_of(p, cache_of(p, d=d)), "64 and 128 are served")


@pytest.mark.parametrize("kw,words", [
    (dict(logits_type=8), "logits of type"), (dict(n_beam=0), "beams"), (dict(n_beam=65), "beams"), (dict(n_request=-1), "requests"), (dict(k=0), "candidates"), (dict(k=129), "candidates"), (dict(n_vocab=0), "vocabulary"),
    (dict(n_vocab=(1 << 24) + 1), "vocabulary"), (dict(logits_ld=999), "vocabulary"), (dict(logits=None), "null operand"), (dict(out_parents=None), "null operand"), (dict(done=A, end_token=1000), "end token"),
    (dict(done=A, end_token=-1), "end token"), (dict(logits=A + 2), "aligned to their type"), (dict(workspace=(A, 64)), "workspace"), (dict(n_request=65535, n_beam=64), "too many")])
def test_select_arguments(p, kw, words):
    refused(select_of(p, **kw), words)


@pytest.mark.parametrize("kw,words", [
    (dict(n_beam=0), "beams"), (dict(n_beam=65), "beams"), (dict(n_request=-1), "requests"), (dict(table_ld=0), "rows of 0 pages"), (dict(page_size=0), "of 0 positions"), (dict(page_bytes=4100), "multiples of 16"),
    (dict(page_bytes=0), "pages of 0 bytes"), (dict(page_stride=2048), "apart"), (dict(n_pages=0), "0 pages"), (dict(parents=None), "null operand"), (dict(tables_out=2 * A), "overlaps"), (dict(tables_out=2 * A + 64), "overlaps"),
    (dict(lens_out=4 * A), "overlaps"), (dict(row_of=A), "overlaps"), (dict(row_of=5 * A + 4), "overlaps"), (dict(pools=[8 * A + 8]), "16-byte aligned"), (dict(pools=[None]), "null")])
def test_reorder_arguments(p, kw, words):
    refused(reorder_of(p, **kw), words)


def test_null_argument_structs(p):
    for name in ("paged_append", "prefix_attn", "beam_select", "beam_reorder"):
        assert getattr(p.lib, "b200_" + name)(None, None) == 3 and b"null arguments" in p.lib.b200_last_error()
    assert p.lib.b200_prefix_attn_workspace_nbytes(None) == 0 and p.lib.b200_beam_select_workspace_nbytes(None) == 0


def test_empty_calls_are_done_at_once(p):
    append_of(p, n_tok=0)(None)
    attn_of(p, n_seq=0, n_group=0)(None)
    select_of(p, n_request=0)(None)
    reorder_of(p, n_request=0)(None)


def test_workspaces_hold_every_part(p):
    n = p.lib.b200_prefix_attn_workspace_nbytes
    small, large = attn_of(p), attn_of(p, cache_of(p, n_seq=64, table_ld=4096), n_seq=64, max_len=32768, max_shared=32000, max_group=64)
    assert n(C.byref(small.args)) >= 4 * 4 * (8 + 64 * 4) and n(C.byref(large.args)) > n(C.byref(small.args))
    assert n(C.byref(attn_of(p, n_head=5).args)) == 0
    s = p.lib.b200_beam_select_workspace_nbytes
    assert s(C.byref(select_of(p, n_vocab=128256).args)) > s(C.byref(select_of(p).args)) >= 8 * 8 * 8
    assert s(C.byref(select_of(p, k=0).args)) == 0


def test_sizes_that_shape_the_launch_may_be_anything(p):
    most = 2 ** 31 - 1
    import ctypes
    for kw in (dict(max_group=most, max_shared=most, max_len=most), dict(max_group=most), dict(max_shared=most), dict(max_len=most), dict(max_group=0, max_shared=0, max_len=0)):
        call = attn_of(p, **kw)
        assert p.lib.b200_prefix_attn_workspace_nbytes(ctypes.byref(call.args)) > 0, kw
