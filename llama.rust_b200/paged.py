"""ctypes wrappers of include/paged_b200.h: decoding several continuations of one prompt over a paged cache.  An object holds the addresses, sizes and
workspace of one call (of a layer, say) and is called with a stream, once a step: what changes from step to step (positions, lengths, tables,
parents) lies on the device.  Addresses are integers, as DeviceBuffer.ptr or a tensor's data_ptr() give them; the memory behind them is the
caller's and must outlive the object's use."""
import ctypes as C

from . import BF16, F16, F32, DeviceBuffer, check, lib  # noqa: F401

vp, i64, i32, f32, sz = C.c_void_p, C.c_int64, C.c_int32, C.c_float, C.c_size_t
SIZE = {F32: 4, F16: 2, BF16: 2}
NORMAL, NEOX = 0, 2


class CacheArgs(C.Structure):
    """struct b200_paged_cache"""
    _fields_ = [("type", i32), ("page_size", i32), ("n_pages", i64), ("n_head_kv", i64), ("d", i64), ("k", vp), ("v", vp), ("page_stride", i64), ("tables", vp),
                ("table_ld", i64), ("n_seq", i64)]


class AppendArgs(C.Structure):
    """struct b200_paged_append_args"""
    _fields_ = [("cache", CacheArgs), ("n_tok", i64), ("pos", vp), ("seq", vp), ("x_type", i32), ("n_head", i32), ("k", vp), ("k_nb1", i64), ("k_nb2", i64),
                ("v", vp), ("v_nb1", i64), ("v_nb2", i64), ("q", vp), ("q_nb1", i64), ("q_nb2", i64), ("q_out", vp), ("q_out_nb1", i64), ("q_out_nb2", i64),
                ("rope", vp), ("rope_rows", i64), ("rope_ld", i64), ("n_dims", i32), ("mode", i32)]


class PrefixAttnArgs(C.Structure):
    """struct b200_prefix_attn_args"""
    _fields_ = [("cache", CacheArgs), ("n_seq", i64), ("n_head", i32), ("n_group", i32), ("q", vp), ("q_nb1", i64), ("q_nb2", i64), ("dst", vp), ("dst_nb1", i64),
                ("dst_nb2", i64), ("lens", vp), ("shared", vp), ("group_first", vp), ("sinks", vp), ("scale", f32), ("max_len", i32), ("max_shared", i32),
                ("max_group", i32), ("workspace", vp), ("workspace_nbytes", sz)]


class BeamSelectArgs(C.Structure):
    """struct b200_beam_select_args"""
    _fields_ = [("logits_type", i32), ("n_request", i32), ("n_beam", i32), ("k", i32), ("n_vocab", i64), ("logits_ld", i64), ("logits", vp), ("scores", vp), ("done", vp),
                ("end_token", i32), ("out_scores", vp), ("out_tokens", vp), ("out_parents", vp), ("workspace", vp), ("workspace_nbytes", sz)]


class BeamReorderArgs(C.Structure):
    """struct b200_beam_reorder_args"""
    _fields_ = [("n_request", i32), ("n_beam", i32), ("parents", vp), ("tables_in", vp), ("tables_out", vp), ("table_ld", i64), ("lens_in", vp), ("lens_out", vp), ("row_of", vp),
                ("page_size", i32), ("n_pools", i32), ("n_pages", i64), ("page_bytes", i64), ("page_stride", i64), ("pools", C.POINTER(vp))]


lib.b200_paged_append.argtypes = [C.POINTER(AppendArgs), vp]
lib.b200_prefix_attn_workspace_nbytes.argtypes = [C.POINTER(PrefixAttnArgs)]
lib.b200_prefix_attn_workspace_nbytes.restype = sz
lib.b200_prefix_attn.argtypes = [C.POINTER(PrefixAttnArgs), vp]
lib.b200_beam_select_workspace_nbytes.argtypes = [C.POINTER(BeamSelectArgs)]
lib.b200_beam_select_workspace_nbytes.restype = sz
lib.b200_beam_select.argtypes = [C.POINTER(BeamSelectArgs), vp]
lib.b200_beam_reorder.argtypes = [C.POINTER(BeamReorderArgs), vp]


class Cache:
    """A layer's pages [n_pages][page_size][n_head_kv][d] of keys and of values, and the tables [n_seq][table_ld] of page ids"""

    def __init__(self, ty, page_size, n_pages, n_head_kv, d, k, v, tables, table_ld, n_seq, page_stride=0):
        self.args = CacheArgs(ty, page_size, n_pages, n_head_kv, d, k, v, page_stride, tables, table_ld, n_seq)


class Call:
    """args, the entry point and its name; a workspace of the object's own unless it is given one (address, bytes)"""

    def __init__(self, name, args, workspace=None):
        self.name, self.args, self.ref = name, args, C.byref(args)
        self.run = getattr(lib, "b200_" + name)
        size = getattr(lib, "b200_%s_workspace_nbytes" % name, None) if hasattr(args, "workspace") else None
        if workspace is not None:
            args.workspace, args.workspace_nbytes = workspace
        elif size is not None:
            n = size(self.ref)   # 0: the call will say what it refuses
            self.own = DeviceBuffer(n) if n else None
            args.workspace, args.workspace_nbytes = (self.own.ptr, n) if n else (None, 0)

    def __call__(self, stream=None):
        rc = self.run(self.ref, stream)
        if rc:
            check(rc, self.name)


class Append(Call):
    """b200_paged_append: k, v [n_tok][n_head_kv][d] (and q [n_tok][n_head][d]) of x_type, to positions pos of sequences seq; rows back to back
    unless strides are given: (bytes per token, bytes per head)"""

    def __init__(self, cache, n_tok, x_type, k, v, pos, seq=None, q=None, q_out=None, n_head=0, rope=None, rope_rows=0, rope_ld=None, n_dims=0, mode=NEOX,
                 k_strides=None, v_strides=None, q_strides=None, q_out_strides=None):
        c, size = cache.args, SIZE.get(x_type, 1)
        kv = (c.n_head_kv * c.d * size, c.d * size)
        super().__init__("paged_append", AppendArgs(c, n_tok, pos, seq, x_type, n_head, k, *(k_strides or kv), v, *(v_strides or kv),
                                                    q, *(q_strides or (n_head * c.d * size, c.d * size)), q_out, *(q_out_strides or (n_head * c.d * 2, c.d * 2)),
                                                    rope, rope_rows, c.d if rope_ld is None else rope_ld, n_dims, mode))


class PrefixAttn(Call):
    """b200_prefix_attn: q, dst [n_seq][n_head][d] of the cache's type; lens, shared [n_seq], group_first [n_group + 1] on the device"""

    def __init__(self, cache, n_seq, n_head, q, dst, lens, scale, shared=None, group_first=None, n_group=0, sinks=None, max_len=0, max_shared=0, max_group=0,
                 q_strides=None, dst_strides=None, workspace=None):
        d = cache.args.d
        dense = (n_head * d * 2, d * 2)
        super().__init__("prefix_attn", PrefixAttnArgs(cache.args, n_seq, n_head, n_group, q, *(q_strides or dense), dst, *(dst_strides or dense), lens, shared, group_first,
                                                       sinks, scale, max_len, max_shared, max_group, None, 0), workspace)


class BeamSelect(Call):
    """b200_beam_select: logits [n_request n_beam][n_vocab] and scores in, the k best (score, token, parent) of every request out"""

    def __init__(self, logits_type, n_request, n_beam, n_vocab, k, logits, scores, out_scores, out_tokens, out_parents, done=None, end_token=0, logits_ld=None, workspace=None):
        super().__init__("beam_select", BeamSelectArgs(logits_type, n_request, n_beam, k, n_vocab, n_vocab if logits_ld is None else logits_ld, logits, scores, done, end_token,
                                                       out_scores, out_tokens, out_parents, None, 0), workspace)


class BeamReorder(Call):
    """b200_beam_reorder: tables, lengths and the pages of `pools` (addresses) after parents [n_request][n_beam]"""

    def __init__(self, n_request, n_beam, parents, tables_in, tables_out, table_ld, lens_in, lens_out, row_of, page_size, n_pages, page_bytes, pools, page_stride=0):
        self.pools = (vp * max(len(pools), 1))(*pools)
        super().__init__("beam_reorder", BeamReorderArgs(n_request, n_beam, parents, tables_in, tables_out, table_ld, lens_in, lens_out, row_of, page_size, len(pools), n_pages,
                                                         page_bytes, page_stride, self.pools))
