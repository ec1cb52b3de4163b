"""The operators over a paged cache as a program uses them: a beam search with append, attention, choice and reorder in turn against the same search in 64 bits
that keeps every beam's whole history; captured steps that are replayed while lengths and parents change; two streams side by side."""
import importlib

import numpy as np
import pytest

import b200
import plain_paged as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def p():
    b200.load()
    return importlib.import_module("llama_rust_b200.paged")


class Toy:
    """A one-layer model over a vocabulary: rows of four matrices by token for q, k and v, logits = head @ (attention output + embedding)"""
    V, H, KV, D, PAGE = 300, 4, 2, 64, 16

    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        self.q, self.k, self.v = (rng.standard_normal((self.V, h, self.D)).astype(np.float32) for h in (self.H, self.KV, self.KV))
        self.embed = rng.standard_normal((self.V, self.H * self.D)).astype(np.float32)
        self.head = (rng.standard_normal((self.V, self.H * self.D)) * 0.2).astype(np.float32)
        self.rope = P.rope_rows(512, self.D, self.D)

    def logits(self, out, tokens):
        return (out.reshape(len(tokens), -1) + self.embed[tokens]).astype(np.float64) @ self.head.astype(np.float64).T

    def history(self, tokens):
        """keys and values of a whole history as the cache holds them (F16), the last token's query"""
        k = np.stack([P.rounded(P.rotated(self.k[t], self.rope[i], self.D, 2)[0], "F16") for i, t in enumerate(tokens)])
        v = np.stack([P.rounded(self.v[t], "F16") for t in tokens])
        return k, v, P.rounded(P.rotated(self.q[tokens[-1]], self.rope[len(tokens) - 1], self.D, 2)[0], "F16")


@pytest.mark.parametrize("seed,prompts,beams", [(0, (37, 5), 4), (1, (64,), 8), (2, (16, 33, 1), 3)])
def test_beam_search(p, seed, prompts, beams):
    m, toy, steps = b200.load(), Toy(seed), 24
    rng = np.random.default_rng(100 + seed)
    R, B = len(prompts), beams
    prompts = [rng.integers(0, toy.V, n).tolist() for n in prompts]
    # tables: the prompt's whole pages are shared, the others are every beam's own
    per = -(-(max(map(len, prompts)) + steps) // toy.PAGE)
    tables, n_pages = np.zeros((R * B, per), dtype=np.int32), 0
    for r in range(R):
        whole = len(prompts[r]) // toy.PAGE
        for b in range(B):
            for i in range(per):
                tables[r * B + b, i] = tables[r * B, i] if b and i < whole else n_pages
                n_pages += not (b and i < whole)
    n = R * B
    new = lambda x, ty=np.float32: m.device_array(np.asarray(x, dtype=ty))  # noqa: E731
    k_pages, v_pages = (new(np.zeros((n_pages, toy.PAGE, toy.KV, toy.D)), np.uint16) for _ in range(2))
    table, table2 = new(tables, np.int32), new(np.zeros_like(tables), np.int32)
    lens, lens2, row_of = new([len(prompts[i // B]) for i in range(n)], np.int32), new(np.zeros(n), np.int32), new(np.zeros(n), np.int32)
    shared = new([len(prompts[i // B]) // toy.PAGE * toy.PAGE for i in range(n)], np.int32)
    groups, rope = new(range(0, n + 1, B), np.int32), new(toy.rope)
    scores, tokens, parents = (new(np.zeros(n), t) for t in (np.float32, np.int32, np.int32))
    cache = lambda: p.Cache(p.F16, toy.PAGE, n_pages, toy.KV, toy.D, k_pages.ptr, v_pages.ptr, table.ptr, per, n)  # noqa: E731

    def append(toks, pos, seq, q_out):
        x = [new(a[toks]) for a in (toy.k, toy.v, toy.q)]
        where = [new(pos, np.int32), new(seq, np.int32)]
        p.Append(cache(), len(toks), p.F32, x[0].ptr, x[1].ptr, where[0].ptr, seq=where[1].ptr, q=x[2].ptr, q_out=q_out.ptr, n_head=toy.H, rope=rope.ptr, rope_rows=512, n_dims=toy.D)(None)
        m.synchronize()

    # the prompts but their last token; a beam's own copy of the part behind the shared pages
    for r, toks in enumerate(prompts):
        for b in range(B):
            at = [i for i in range(len(toks) - 1) if b == 0 or i >= len(toks) // toy.PAGE * toy.PAGE]
            if at:
                append([toks[i] for i in at], at, [r * B + b] * len(at), new(np.zeros(len(at) * toy.H * toy.D), np.uint16))
    last = [prompts[i // B][-1] for i in range(n)]
    score = np.full((R, B), -np.inf, dtype=np.float32)
    score[:, 0] = 0.0   # one beam to begin with
    history = [[list(q) for _ in range(B)] for q in prompts]
    for step in range(steps):
        pos = [len(prompts[i // B]) - 1 + step for i in range(n)]
        q_out, out = (new(np.zeros(n * toy.H * toy.D), np.uint16) for _ in range(2))
        append(last, pos, list(range(n)), q_out)
        lens.upload(np.array([x + 1 for x in pos], dtype=np.int32))
        p.PrefixAttn(cache(), n, toy.H, q_out.ptr, out.ptr, lens.ptr, toy.D ** -0.5, shared=shared.ptr, group_first=groups.ptr, n_group=R, max_len=max(pos) + 1, max_shared=64, max_group=B)(None)
        got = P.values(out.download(np.uint16, n * toy.H * toy.D), "F16").reshape(n, toy.H, toy.D)
        # every beam against attention over its whole history
        for r in range(R):
            for b in range(B):
                k, v, q = toy.history(history[r][b])
                w = np.exp(np.einsum("phd,hd->hp", k.repeat(2, 1), q) * toy.D ** -0.5)
                want = np.einsum("hp,phd->hd", w / w.sum(1, keepdims=True), v.repeat(2, 1))
                # a cached key or query that F32 rounds to the neighbouring half differs by one step: well within 2^-8 of a score of about 10
                assert np.abs(got[r * B + b] - want).max() < 0.03, (step, r, b)
        logits = toy.logits(got, np.array(last)).astype(np.float32).reshape(R, B, toy.V)
        x = new(logits)
        scores.upload(score)
        p.BeamSelect(p.F32, R, B, toy.V, B, x.ptr, scores.ptr, scores.ptr, tokens.ptr, parents.ptr)(None)   # the new scores in the place of the old
        want = P.select(logits, score.astype(np.float64), B)
        tok, par = tokens.download(np.int32, n), parents.download(np.int32, n)
        assert np.array_equal(tok.reshape(R, B), want[1]) and np.array_equal(par.reshape(R, B), want[2])
        score = scores.download(np.float32, n).reshape(R, B)
        assert np.abs(score - want[0]).max() < 1e-4
        p.BeamReorder(R, B, parents.ptr, table.ptr, table2.ptr, per, lens.ptr, lens2.ptr, row_of.ptr, toy.PAGE, n_pages, toy.PAGE * toy.KV * toy.D * 2, [k_pages.ptr, v_pages.ptr])(None)
        table, table2, lens, lens2 = table2, table, lens2, lens
        history = [[history[r][par[r * B + b]] + [int(tok[r * B + b])] for b in range(B)] for r in range(R)]
        last = tok.tolist()
        assert lens.download(np.int32, n).tolist() == [x + 1 for x in pos]
    assert m.kernel_error() == 0
    assert len({tuple(h) for h in history[0]}) == B


def problem(torch, seed, n=6, shared=200, own=60):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {}
    s["k"], s["v"] = (torch.randn((n * 20, 16, 2, 128), generator=g, device="cuda").bfloat16() for _ in range(2))
    s["tables"] = torch.randperm(n * 20, generator=g, device="cuda").int().view(n, 20).contiguous()
    s["x"] = torch.randn((3, n, 8, 128), generator=g, device="cuda")
    s["pos"] = torch.full((n,), shared + own - 1, device="cuda", dtype=torch.int32)
    s["lens"], s["shared"] = s["pos"] + 1, torch.full_like(s["pos"], shared)
    s["first"] = torch.tensor([0, n], device="cuda", dtype=torch.int32)
    s["rope"] = torch.from_numpy(P.rope_rows(512, 128, 128)).cuda()
    s["q"], s["out"] = (torch.zeros((n, 8, 128), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    s["logits"] = torch.randn((n, 5000), generator=g, device="cuda") * 3
    s["scores"] = -torch.rand((n,), generator=g, device="cuda")
    s["best"], s["tok"], s["par"] = torch.zeros((n,), device="cuda"), *(torch.zeros((n,), device="cuda", dtype=torch.int32) for _ in range(2))
    s["tables2"], s["lens2"], s["row"] = torch.zeros_like(s["tables"]), torch.zeros_like(s["lens"]), torch.zeros_like(s["lens"])
    return s


def step_of(p, s, n=6):
    at = {k: v.data_ptr() for k, v in s.items()}
    c = p.Cache(p.BF16, 16, n * 20, 2, 128, at["k"], at["v"], at["tables"], 20, n)
    token = 8 * 128 * 4
    kv = (token, 128 * 4)
    calls = [p.Append(c, n, p.F32, at["x"], at["x"] + n * token, at["pos"], q=at["x"] + 2 * n * token, q_out=at["q"], n_head=8, rope=at["rope"], rope_rows=512, n_dims=128, k_strides=kv, v_strides=kv),
             p.PrefixAttn(c, n, 8, at["q"], at["out"], at["lens"], 128 ** -0.5, shared=at["shared"], group_first=at["first"], n_group=1, max_len=260, max_shared=200, max_group=n),
             p.BeamSelect(p.F32, 1, n, 5000, n, at["logits"], at["scores"], at["best"], at["tok"], at["par"]),
             p.BeamReorder(1, n, at["par"], at["tables"], at["tables2"], 20, at["lens"], at["lens2"], at["row"], 16, n * 20, 16 * 2 * 128 * 2, [at["k"], at["v"]])]

    def run(stream):
        for c in calls:
            c(stream)
    return run


RESULTS = ("q", "k", "v", "out", "best", "tok", "par", "tables2", "lens2", "row")


def test_captured_steps_follow_what_changes_on_the_device(p):
    import torch
    s, eager = problem(torch, 1), problem(torch, 1)
    run, run_eager = step_of(p, s), step_of(p, eager)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(torch.cuda.current_stream().cuda_stream)
    for turn in range(4):
        for x in (s, eager):
            x["pos"].fill_(200 + 13 * turn)
            x["lens"].copy_(x["pos"] + 1)
            x["lens"][turn] = 0
            x["pos"][turn] = -1
            x["shared"].fill_(200 - 50 * turn)
            x["logits"].copy_(torch.roll(x["logits"], 7, 0))
        torch.cuda.synchronize()
        graph.replay()
        run_eager(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for name in RESULTS:
            assert torch.equal(s[name], eager[name]), (turn, name)
    assert b200.load().kernel_error() == 0


def test_two_streams_side_by_side(p):
    import torch
    a, b, c = problem(torch, 1), problem(torch, 2), problem(torch, 1)
    d = problem(torch, 2)
    runs = [step_of(p, x) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, run in zip(streams, runs):
            run(st.cuda_stream)
    torch.cuda.synchronize()
    for x in (c, d):
        r = step_of(p, x)
        for _ in range(10):
            r(None)
    torch.cuda.synchronize()
    for x, y in ((a, c), (b, d)):
        for name in RESULTS:
            assert torch.equal(x[name], y[name]), name
    assert b200.load().kernel_error() == 0


def test_host_memory_is_refused(p):
    import torch
    s = problem(torch, 1)
    host = np.zeros(1 << 20, dtype=np.uint8)
    base = (host.ctypes.data + 255) // 256 * 256
    c = p.Cache(p.BF16, 16, 120, 2, 128, base, base, s["tables"].data_ptr(), 20, 6)
    for call in (p.Append(c, 6, p.F32, s["x"].data_ptr(), s["x"].data_ptr(), s["pos"].data_ptr(), n_dims=0),
                 p.PrefixAttn(c, 6, 8, s["q"].data_ptr(), s["out"].data_ptr(), s["lens"].data_ptr(), 0.1, max_len=100),
                 p.BeamSelect(p.F32, 1, 6, 5000, 6, base, s["scores"].data_ptr(), s["best"].data_ptr(), s["tok"].data_ptr(), s["par"].data_ptr()),
                 p.BeamReorder(1, 6, s["par"].data_ptr(), s["tables"].data_ptr(), s["tables2"].data_ptr(), 20, s["lens"].data_ptr(), s["lens2"].data_ptr(), None, 16, 120, 64, [base])):
        with pytest.raises(Exception, match="host memory|kernel can touch"):
            call(None)
    torch.cuda.synchronize()


def test_every_operand_in_host_memory_is_refused(p):
    import torch
    host = np.zeros(1 << 20, dtype=np.uint8)
    base = (host.ctypes.data + 255) // 256 * 256
    room = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    at = [room.data_ptr() + (i << 16) for i in range(16)]
    c = p.Cache(p.BF16, 16, 4, 2, 64, at[0], at[1], at[2], 4, 2)
    calls = (p.Append(c, 2, p.F32, at[3], at[4], at[5], seq=at[6], q=at[7], q_out=at[8], n_head=4, rope=at[9], rope_rows=8, rope_ld=64, n_dims=64),
             p.PrefixAttn(c, 2, 4, at[3], at[4], at[5], 0.1, shared=at[6], group_first=at[7], n_group=1, sinks=at[8], max_len=40, max_shared=32, max_group=2),
             p.BeamSelect(p.F32, 1, 2, 1000, 2, at[3], at[4], at[5], at[6], at[7], done=at[8]),
             p.BeamReorder(1, 2, at[3], at[4], at[5], 4, at[6], at[7], at[8], 16, 4, 64, [at[9], at[10]]))
    refused = 0
    for call in calls:
        call(None)   # as it stands it runs
        for args in (call.args, getattr(call.args, "cache", None)):
            for name, ty in (args._fields_ if args is not None else ()):
                if ty is not p.vp:
                    continue
                kept = getattr(args, name)
                setattr(args, name, base)
                with pytest.raises(Exception, match="host memory|kernel can touch"):
                    call(None)
                setattr(args, name, kept)
                refused += 1
    calls[3].pools[1] = base
    with pytest.raises(Exception, match="host memory|kernel can touch"):
        calls[3](None)
    torch.cuda.synchronize()
    # groups of zeros: [0, 0) holds none of the two sequences, which attention reports
    assert refused == 7 + 3 + 7 + 3 + 7 + 6 and b200.load().kernel_error() == 7
