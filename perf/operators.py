"""The operators of decoding several continuations of one prompt over a paged cache, as they are measured: a step's keys and values appended with their
rotation (`append`), attention of single rows whose sequences share their first positions (`attention`), the choice of a request's best continuations
(`select`), and the tables, lengths and pages that follow the chosen beams (`reorder`).

`listed()` names the cases, `draw()` gives further ones of the same ranges, `prepare()` makes what a program holds before the call, `run()` is one pass:
with `own` the library's calls, without it the same in elementary torch operations.  `work()` says what a pass cannot do without, `exact()` the result in
64 bits.  Lengths follow from the case, values from the seed."""
import importlib
import importlib.util
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}


def _paged():
    """the package's module of these operators (its folder's name has a dot, so it is loaded by path)"""
    if "llama_rust_b200" not in sys.modules:
        spec = importlib.util.spec_from_file_location("llama_rust_b200", os.path.join(ROOT, "llama.rust_b200", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["llama_rust_b200"] = mod
        spec.loader.exec_module(mod)
    return importlib.import_module("llama_rust_b200.paged")


def listed():
    return [
        # one token of each of four beams: a layer's smallest step, all latency
        {"name": "append_4_beams", "op": "append", "seqs": 4, "tokens": 1, "past": 700, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "mode": 2, "x": "F32", "cache": "F16", "page": 16},
        # a long prompt read in one portion, adjacent channels rotating
        {"name": "append_prompt_8192", "op": "append", "seqs": 1, "tokens": 8192, "past": 0, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "mode": 0, "x": "F32", "cache": "BF16", "page": 64},
        # portions of five prompts in one step, half of a small head rotating, activations in 16 bits, portions that begin and end inside pages
        {"name": "append_5_portions_d64", "op": "append", "seqs": 5, "tokens": 67, "past": 1003, "heads": 14, "kv_heads": 2, "dim": 64, "rot": 32, "mode": 2, "x": "BF16", "cache": "BF16", "page": 32},
        # eight beams of a short prompt: latency counts
        {"name": "attention_8_beams_1000", "op": "attention", "groups": 1, "per": 8, "shared": 1000, "own": 24, "heads": 32, "kv_heads": 8, "dim": 128, "cache": "F16", "page": 16, "sinks": False},
        # four requests of sixteen beams each
        {"name": "attention_4x16_beams_4096", "op": "attention", "groups": 4, "per": 16, "shared": 4096, "own": 128, "heads": 32, "kv_heads": 8, "dim": 128, "cache": "BF16", "page": 32, "sinks": False},
        # sixty-four conversations behind one long system prompt: as much to multiply as to read
        {"name": "attention_64_rows_32768", "op": "attention", "groups": 1, "per": 64, "shared": 32768, "own": 512, "heads": 32, "kv_heads": 8, "dim": 128, "cache": "BF16", "page": 64, "sinks": False},
        # small heads with keys of their own and sinks, odd lengths, a shared part that ends inside a page
        {"name": "attention_3x7_d64_2047", "op": "attention", "groups": 3, "per": 7, "shared": 2047, "own": 333, "heads": 16, "kv_heads": 16, "dim": 64, "cache": "F16", "page": 16, "sinks": True},
        # four beams of one request: the smallest choice there is
        {"name": "select_4_beams_32000", "op": "select", "requests": 1, "beams": 4, "vocab": 32000, "k": 4, "logits": "F32", "done": 0},
        # eight requests of eight beams, the vocabulary of the benchmark's model, twice as many candidates as beams
        {"name": "select_8x8_128256", "op": "select", "requests": 8, "beams": 8, "vocab": 128256, "k": 16, "logits": "F32", "done": 0},
        # logits in 16 bits (many ties), an odd vocabulary, beams that have ended
        {"name": "select_32x5_50001_bf16", "op": "select", "requests": 32, "beams": 5, "vocab": 50001, "k": 5, "logits": "BF16", "done": 1},
        # four recurrent states (16 heads of 128 x 256) in each of 24 layers
        {"name": "reorder_4_states", "op": "reorder", "requests": 1, "beams": 4, "pools": 24, "page": 1, "shared": 0, "own": 1, "row": 16 * 128 * 256, "type": "F32"},
        # eight requests of eight beams 300 tokens behind a shared prompt, keys and values of 16 layers
        {"name": "reorder_8x8_pages", "op": "reorder", "requests": 8, "beams": 8, "pools": 32, "page": 16, "shared": 1024, "own": 300, "row": 8 * 128, "type": "BF16"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "attention", "attention", "select", "reorder"])
    if op == "append":
        dim, kv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        seqs = log(1, 64)
        return {"op": op, "seqs": seqs, "tokens": log(1, max(2, 8192 // seqs)), "past": log(1, 4096) - 1, "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2]), "mode": rng.choice([0, 2]), "x": rng.choice(["F32", "F32", "F16", "BF16"]), "cache": rng.choice(["F16", "BF16"]), "page": rng.choice([16, 32, 64, 128])}
    if op == "attention":
        dim, kv = rng.choice([64, 128, 128]), rng.choice([2, 4, 8])
        groups = log(1, 8)
        per = log(1, 64 // groups)
        heads = kv * rng.choice([1, 2, 4])
        return {"op": op, "groups": groups, "per": per, "shared": log(1, 32768 // groups), "own": log(1, 512), "heads": heads, "kv_heads": kv, "dim": dim,
                "cache": rng.choice(["F16", "BF16"]), "page": rng.choice([16, 32, 64, 128]), "sinks": rng.random() < 0.3}
    if op == "select":
        requests, beams = log(1, 32), log(1, 16)
        while requests * beams > 64:
            requests = (requests + 1) // 2
        return {"op": op, "requests": requests, "beams": beams, "vocab": log(1000, 128256), "k": beams * rng.choice([1, 2]), "logits": rng.choice(["F32", "F32", "F16", "BF16"]), "done": rng.choice([0, 1])}
    requests, beams = log(1, 8), log(2, 8)
    if rng.random() < 0.4:
        return {"op": op, "requests": requests, "beams": beams, "pools": log(1, 24), "page": 1, "shared": 0, "own": 1, "row": 4 * log(16, 65536), "type": "F32"}
    return {"op": op, "requests": requests, "beams": beams, "pools": 2 * log(1, 16), "page": rng.choice([16, 32, 64]), "shared": log(1, 1024), "own": log(1, 300),
            "row": rng.choice([1, 2, 4, 8]) * rng.choice([64, 128]), "type": rng.choice(["F16", "BF16"])}


# ---- lengths, which follow from the case ---------------------------------------------------------------------------------------------

def _lens(c):
    """positions of every sequence of an attention case: ragged behind the shared ones, and of eight or more the last is padding"""
    n = c["groups"] * c["per"]
    lens = [c["shared"] + c["own"] - (37 * i) % (c["own"] // 4 + 1) for i in range(n)]
    if n >= 8:
        lens[-1] = 0
    return lens


def _distinct(beams):
    """of a request's beams, those that are continued"""
    return (beams + 1) // 2


def work(c):
    size = {"F32": 4, "F16": 2, "BF16": 2}
    if c["op"] == "append":
        n = c["seqs"] * c["tokens"]
        elems = n * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": elems * (size[c["x"]] + 2) + min(n, c["past"] + c["tokens"]) * c["rot"] * 4 + 12 * n, "flops": 3 * n * (c["heads"] + c["kv_heads"]) * c["rot"]}
    if c["op"] == "attention":
        lens = _lens(c)
        shared = sum(max([min(n, c["shared"]) for n in lens[g * c["per"]:(g + 1) * c["per"]]]) for g in range(c["groups"]))
        cells = shared + sum(max(0, n - c["shared"]) for n in lens)
        return {"bytes": cells * c["kv_heads"] * c["dim"] * 4 + len(lens) * c["heads"] * c["dim"] * 4 + 4 * (cells // c["page"] + 2 * len(lens)),
                "flops": 4 * c["heads"] * c["dim"] * sum(lens)}
    if c["op"] == "select":
        rows = c["requests"] * c["beams"]
        return {"bytes": rows * c["vocab"] * size[c["logits"]] + 5 * rows + 12 * c["requests"] * c["k"], "flops": 4 * rows * c["vocab"]}
    n = c["requests"] * c["beams"]
    pages = _pages(c["shared"] + c["own"], c["page"]) - c["shared"] // c["page"]
    moved = c["requests"] * (c["beams"] - _distinct(c["beams"])) * pages * c["pools"] * c["page"] * c["row"] * size[c["type"]]
    return {"bytes": 2 * moved + 8 * n * (_pages(c["shared"] + c["own"], c["page"]) + 2), "flops": 0}


def _pages(n, page):
    return -(-n // page)


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------

def prepare(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    rng = random.Random(int(seed))
    s = {"case": c}
    {"append": _prepare_append, "attention": _prepare_attention, "select": _prepare_select, "reorder": _prepare_reorder}[c["op"]](s, c, gen, rng)
    if own:
        s["call"] = _call(s, c)   # made once, as a decoding program makes it for a layer; it holds addresses, sizes and a workspace
    return s


def _randn(gen, shape, dtype=torch.float32, dev=1.0):
    return (torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32) * dev).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tables(seqs, per_group, shared_pages, pages, rng):
    """page ids in no order: of `seqs` sequences in groups of per_group, the first shared_pages are the group's, the others each sequence's own"""
    groups = seqs // per_group
    ids = list(range(groups * shared_pages + seqs * (pages - shared_pages)))
    rng.shuffle(ids)
    ids = torch.tensor(ids, dtype=torch.int32)
    common = ids[: groups * shared_pages].view(groups, 1, shared_pages).expand(groups, per_group, shared_pages).reshape(seqs, shared_pages)
    return torch.cat([common, ids[groups * shared_pages:].view(seqs, pages - shared_pages)], 1).contiguous().cuda(), len(ids)


def _prepare_append(s, c, gen, rng):
    n, kv, d = c["seqs"] * c["tokens"], c["kv_heads"], c["dim"]
    last = c["past"] + c["tokens"]
    s["tables"], n_pages = _tables(c["seqs"], 1, 0, _pages(last, c["page"]), rng)
    s["k_pages"], s["v_pages"] = (_randn(gen, (n_pages, c["page"], kv, d), TYPES[c["cache"]]) for _ in range(2))
    s["q"], s["k"], s["v"] = (_randn(gen, (n, h, d), TYPES[c["x"]]) for h in (c["heads"], kv, kv))
    s["q_out"] = torch.zeros((n, c["heads"], d), dtype=TYPES[c["cache"]], device="cuda")
    at = torch.arange(c["seqs"], device="cuda", dtype=torch.int32)
    s["pos"] = (c["past"] + torch.arange(c["tokens"], device="cuda", dtype=torch.int32)).repeat(c["seqs"]).contiguous()
    s["seq"] = at.repeat_interleave(c["tokens"]).contiguous()
    # (cos, sin) by position, as a program keeps it for its whole context
    angle = torch.arange(last, device="cuda", dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
    s["rope"] = torch.zeros((last, d), device="cuda")
    s["rope"][:, 0:c["rot"]:2], s["rope"][:, 1:c["rot"]:2] = angle.cos(), angle.sin()


def _prepare_attention(s, c, gen, rng):
    n, kv, d = c["groups"] * c["per"], c["kv_heads"], c["dim"]
    s["tables"], n_pages = _tables(n, c["per"], c["shared"] // c["page"], _pages(c["shared"] + c["own"], c["page"]), rng)
    s["k_pages"], s["v_pages"] = (_randn(gen, (n_pages, c["page"], kv, d), TYPES[c["cache"]]) for _ in range(2))
    s["q"] = _randn(gen, (n, c["heads"], d), TYPES[c["cache"]], 1.5)
    s["out"] = torch.zeros((n, c["heads"], d), dtype=TYPES[c["cache"]], device="cuda")
    s["lens"] = _i32(_lens(c))
    s["shared"] = _i32([c["shared"]] * n)
    s["group_first"] = _i32(list(range(0, n + 1, c["per"])))
    s["sinks"] = _randn(gen, (c["heads"],)) if c["sinks"] else None


def _prepare_select(s, c, gen, rng):
    rows = c["requests"] * c["beams"]
    # a head's logits: most words far below a few likely ones
    x = _randn(gen, (rows, c["vocab"]), dev=2.0)
    x[:, ::61] *= 2.5
    s["logits"] = x.to(TYPES[c["logits"]])
    s["scores"] = -torch.rand((c["requests"], c["beams"]), device="cuda", generator=gen) * 4.0 - 10.0
    # every second request has a beam that has ended
    ended = [rng.randrange(c["beams"]) if c["done"] and c["beams"] > 1 and r & 1 else -1 for r in range(c["requests"])]
    s["done"] = torch.tensor([[int(b == e) for b in range(c["beams"])] for e in ended], dtype=torch.uint8, device="cuda")
    s["end"] = c["vocab"] // 3
    shape = (c["requests"], c["k"])
    s["out_scores"] = torch.zeros(shape, device="cuda")
    s["out_tokens"], s["out_parents"] = (torch.zeros(shape, dtype=torch.int32, device="cuda") for _ in range(2))


def _prepare_reorder(s, c, gen, rng):
    n, last = c["requests"] * c["beams"], c["shared"] + c["own"]
    s["tables"], n_pages = _tables(n, c["beams"], c["shared"] // c["page"], _pages(last, c["page"]), rng)
    s["pools"] = [_randn(gen, (n_pages, c["page"] * c["row"]), TYPES[c["type"]]) for _ in range(c["pools"])]
    parents = []
    for _ in range(c["requests"]):
        alive = rng.sample(range(c["beams"]), _distinct(c["beams"]))
        mine = alive + [rng.choice(alive) for _ in range(c["beams"] - len(alive))]
        rng.shuffle(mine)
        parents.append(mine)
    s["parents"] = _i32(parents)
    s["lens"] = _i32([last] * n)
    s["new_tables"], s["new_lens"], s["row_of"] = torch.zeros_like(s["tables"]), torch.zeros_like(s["lens"]), torch.zeros_like(s["lens"])


# ---- one pass ------------------------------------------------------------------------------------------------------------------------------

def _call(s, c):
    """the call object that a decoding program makes once and keeps"""
    p, at = _paged(), (lambda name: s[name].data_ptr())
    ty = {"F32": p.F32, "F16": p.F16, "BF16": p.BF16}
    if c["op"] in ("append", "attention"):
        cache = p.Cache(ty[c["cache"]], c["page"], s["k_pages"].shape[0], c["kv_heads"], c["dim"], at("k_pages"), at("v_pages"), at("tables"), s["tables"].shape[1], s["tables"].shape[0])
    if c["op"] == "append":
        return p.Append(cache, s["pos"].numel(), ty[c["x"]], at("k"), at("v"), at("pos"), seq=at("seq"), q=at("q"), q_out=at("q_out"), n_head=c["heads"],
                        rope=at("rope"), rope_rows=s["rope"].shape[0], n_dims=c["rot"], mode=c["mode"])
    if c["op"] == "attention":
        return p.PrefixAttn(cache, s["q"].shape[0], c["heads"], at("q"), at("out"), at("lens"), c["dim"] ** -0.5, shared=at("shared"), group_first=at("group_first"), n_group=c["groups"],
                            sinks=at("sinks") if c["sinks"] else None, max_len=c["shared"] + c["own"], max_shared=c["shared"], max_group=c["per"])
    if c["op"] == "select":
        return p.BeamSelect(ty[c["logits"]], c["requests"], c["beams"], c["vocab"], c["k"], at("logits"), at("scores"), at("out_scores"), at("out_tokens"), at("out_parents"),
                            done=at("done"), end_token=s["end"])
    size = s["pools"][0].element_size()
    return p.BeamReorder(c["requests"], c["beams"], at("parents"), at("tables"), at("new_tables"), s["tables"].shape[1], at("lens"), at("new_lens"), at("row_of"), c["page"],
                         s["pools"][0].shape[0], c["page"] * c["row"] * size, [x.data_ptr() for x in s["pools"]])


def run(s):
    op = s["case"]["op"]
    if own:
        s["call"](torch.cuda.current_stream().cuda_stream)
        return _outputs(s, op)
    return {"append": _append, "attention": _attention, "select": _select, "reorder": _reorder}[op](s, s["case"])


def _outputs(s, op):
    if op == "append":
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if op == "attention":
        return s["out"]
    if op == "select":
        return {"scores": s["out_scores"], "tokens": s["out_tokens"], "parents": s["out_parents"]}
    return {"pools": s["pools"], "tables": s["new_tables"], "lens": s["new_lens"], "row_of": s["row_of"]}


def _rotated(x, c, rope):
    """x [tokens, heads, dim] in 32 bits, its first `rot` channels turned; rope [tokens, dim]"""
    r = c["rot"]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["mode"] == 0 else (x[..., : r // 2], x[..., r // 2: r])
    cos, sin = rope[:, None, 0:r:2], rope[:, None, 1:r:2]
    y = x.clone()
    if c["mode"] == 0:
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    else:
        y[..., : r // 2], y[..., r // 2: r] = a * cos - b * sin, a * sin + b * cos
    return y


def _append(s, c):
    pos, seq = s["pos"].long(), s["seq"].long()
    page, inside = s["tables"][seq, pos // c["page"]].long(), pos % c["page"]
    rope = s["rope"][pos]
    s["q_out"].copy_(_rotated(s["q"].float(), c, rope))
    s["k_pages"][page, inside] = _rotated(s["k"].float(), c, rope).to(s["k_pages"].dtype)
    s["v_pages"][page, inside] = s["v"].to(s["v_pages"].dtype)
    return _outputs(s, "append")


def _attention(s, c):
    G, B, kv, d, P, ps = c["groups"], c["per"], c["kv_heads"], c["dim"], c["shared"], c["page"]
    n, each = G * B, c["heads"] // kv
    lens, shared, tables = s["lens"].long(), s["shared"].long(), s["tables"].long()
    q = s["q"].float().view(n, kv, each, d) * d ** -0.5

    def rows(pages, seq, pos):
        return pages[tables[seq, pos // ps], pos % ps].float()

    # the shared positions once for a group, all its rows together
    first, at = torch.arange(0, n, B, device="cuda")[:, None], torch.arange(P, device="cuda")[None]
    pk, pv = rows(s["k_pages"], first, at), rows(s["v_pages"], first, at)                      # [G, P, kv, d]
    qg = q.view(G, B, kv, each, d).permute(0, 2, 1, 3, 4).reshape(G, kv, B * each, d)
    sp = torch.matmul(qg, pk.permute(0, 2, 3, 1)).view(G, kv, B, each, P).permute(0, 2, 1, 3, 4).reshape(n, kv, each, P)
    sp = sp.masked_fill((at >= torch.minimum(lens, shared)[:, None])[:, None, None], -math.inf)
    # the others of each sequence
    seq = torch.arange(n, device="cuda")[:, None]
    ot = shared[:, None] + torch.arange(c["own"], device="cuda")[None]
    ok, ov = rows(s["k_pages"], seq, ot), rows(s["v_pages"], seq, ot)                          # [n, own, kv, d]
    so = torch.matmul(q, ok.permute(0, 2, 3, 1)).masked_fill((ot >= lens[:, None])[:, None, None], -math.inf)
    top = torch.maximum(sp.amax(-1), so.amax(-1))
    sink = s["sinks"].view(1, kv, each) if s["sinks"] is not None else None
    if sink is not None:
        top = torch.maximum(top, sink)
    top = top.clamp_min(-3.0e38)[..., None]
    wp, wo = torch.exp(sp - top), torch.exp(so - top)
    total = wp.sum(-1, keepdim=True) + wo.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink[..., None] - top)
    wg = wp.view(G, B, kv, each, P).permute(0, 2, 1, 3, 4).reshape(G, kv, B * each, P)
    yp = torch.matmul(wg, pv.permute(0, 2, 1, 3)).view(G, kv, B, each, d).permute(0, 2, 1, 3, 4).reshape(n, kv, each, d)
    y = yp + torch.matmul(wo, ov.permute(0, 2, 1, 3))
    y = torch.where(total > 0, y / total, torch.zeros_like(y))
    s["out"].copy_(y.view(n, c["heads"], d))
    return s["out"]


def _select(s, c):
    # in 64 bits: whole numbers come of which of two near values is larger
    R, B, V, k = c["requests"], c["beams"], c["vocab"], c["k"]
    x = s["logits"].double()
    x = x.masked_fill(torch.isnan(x), -math.inf)
    top = x.amax(1, keepdim=True)
    off = torch.where(x == top, torch.zeros_like(x), x - top)
    gain = (off - torch.log(torch.exp(off).sum(1, keepdim=True))).masked_fill(torch.isneginf(x), -math.inf)
    score = s["scores"].double().view(R * B, 1) + gain
    done = s["done"].view(R * B, 1) != 0
    ends = torch.arange(V, device="cuda")[None] == s["end"]
    score = torch.where(done, torch.where(ends, s["scores"].double().view(R * B, 1), torch.full_like(score, -math.inf)), score)
    best, at = torch.sort(score.view(R, B * V), dim=1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    none = torch.isneginf(best)
    s["out_scores"].copy_(best)
    s["out_tokens"].copy_(torch.where(none, torch.full_like(at, -1), at % V))
    s["out_parents"].copy_(torch.where(none, torch.full_like(at, -1), at // V))
    return _outputs(s, "select")


def _reorder(s, c):
    R, B, ps = c["requests"], c["beams"], c["page"]
    par = s["parents"].long()
    beam = torch.arange(B, device="cuda")
    used = par >= 0
    same = (par[:, :, None] == par[:, None, :]) & (beam[None, :] < beam[:, None])[None]          # [r, j, an earlier child of the same parent]
    first = used & ~same.any(2)
    alive = (par[:, :, None] == beam[None, None]).any(1)
    # a parent's first child takes its row; its other children, then the beams not in use, the rows of beams without a child
    extra, idle = used & ~first, ~used
    rank = torch.where(extra, extra.cumsum(1) - 1, extra.sum(1, keepdim=True) + idle.cumsum(1) - 1).clamp(0, B - 1)
    free = torch.sort(alive.to(torch.int8), dim=1, stable=True)[1]
    row = torch.where(first, par, torch.gather(free, 1, rank))
    base = (torch.arange(R, device="cuda") * B)[:, None]
    row_of, source = (base + row).view(-1), (base + torch.where(used, par, row)).view(-1)
    s["row_of"].copy_(row.reshape(-1))
    s["new_tables"].copy_(s["tables"][row_of])
    s["new_lens"].copy_(torch.where(used.view(-1), s["lens"][source], torch.zeros_like(s["lens"])))
    to, frm = s["tables"][row_of].long(), s["tables"][source].long()
    moves = extra.view(-1, 1) & (torch.arange(to.shape[1], device="cuda")[None] * ps < s["lens"][source][:, None]) & (to != frm)
    frm = torch.where(moves, frm, to).view(-1)
    to = to.view(-1)
    for pool in s["pools"]:
        pool[to] = pool[frm]
    return _outputs(s, "reorder")


# ---- the same in 64 bits, from the definitions ------------------------------------------------------------------------------------------------

def exact(c, seed):
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    return {"append": _exact_append, "attention": _exact_attention, "select": _exact_select, "reorder": _exact_reorder}[c["op"]](s, c)


def _exact_append(s, c):
    r, out = c["rot"], []
    # a pair of channels as one complex number, times e^(i angle)
    turn = torch.complex(s["rope"][:, 0:r:2].double(), s["rope"][:, 1:r:2].double())[s["pos"].long()][:, None]
    for x in (s["q"], s["k"]):
        x = x.double()
        if c["mode"] == 0:
            z = torch.view_as_real(torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2)) * turn).reshape(*x.shape[:-1], r)
        else:
            z = torch.complex(x[..., : r // 2], x[..., r // 2: r]) * turn
            z = torch.cat([z.real, z.imag], -1)
        out.append(torch.cat([z, x[..., r:]], -1))
    flat = s["tables"].long().gather(1, (s["pos"].long() // c["page"]).view(c["seqs"], -1)).view(-1) * c["page"] + s["pos"].long() % c["page"]
    pages = []
    for old, new in ((s["k_pages"], out[1]), (s["v_pages"], s["v"].double())):
        pages.append(old.double().view(-1, c["kv_heads"], c["dim"]).index_copy(0, flat, new).view(old.shape))
    return {"q": out[0], "k_pages": pages[0], "v_pages": pages[1]}


def _exact_attention(s, c):
    each, lens = c["heads"] // c["kv_heads"], _lens(c)
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if n == 0:
            continue
        g = i // c["per"] * c["per"]
        p = torch.arange(n, device="cuda")
        line = torch.where(p < c["shared"], s["tables"][g, p // c["page"]], s["tables"][i, p // c["page"]]).long()
        k, v = (x[line, p % c["page"]].double().repeat_interleave(each, 1) for x in (s["k_pages"], s["v_pages"]))
        a = torch.einsum("hd,phd->hp", s["q"][i].double(), k) / math.sqrt(c["dim"])
        if s["sinks"] is not None:
            a = torch.cat([a, s["sinks"].double()[:, None]], 1)
        y[i] = torch.einsum("hp,phd->hd", torch.softmax(a, 1)[:, :n], v)
    return y


def _exact_select(s, c):
    x = s["logits"].double()
    total = s["scores"].double().view(-1, 1) + (x - torch.logsumexp(x, 1, keepdim=True))
    held = s["done"].view(-1) != 0
    total[held] = -math.inf
    total[held, s["end"]] = s["scores"].double().view(-1)[held]
    return {"scores": torch.topk(total.view(c["requests"], -1), c["k"], dim=1).values, "tokens": None, "parents": None}


def _exact_reorder(s, c):
    B, pages = c["beams"], _pages(c["shared"] + c["own"], c["page"])
    tables, frm, to = s["tables"].tolist(), [], []
    for r, par in enumerate(s["parents"].tolist()):
        free = [b for b in range(B) if b not in par]
        for j, p in enumerate(par):
            if p in par[:j]:
                a, b = tables[r * B + p][:pages], tables[r * B + free.pop(0)][:pages]
                frm += [x for x, y in zip(a, b) if x != y]
                to += [y for x, y in zip(a, b) if x != y]
    pools = [x.double().index_copy(0, torch.tensor(to, device="cuda"), x[torch.tensor(frm, device="cuda")].double()) for x in s["pools"]] if to else [x.double() for x in s["pools"]]
    return {"pools": pools, "tables": None, "lens": None, "row_of": None}
