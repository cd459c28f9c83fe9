"""The operators of yue2_rs_b200.ops as timed cases: packed prompt attention, drafted-tree
attention over paged K/V, the QK norm + rotation + append pass, and the page moves (copy, gather).

Each case has a plain form (elementary torch operations in 32 bits) and, with `own` set, the
framework's call. A pool is [pages, layers, K|V, kv heads, 64 positions, dim], the layout of the
engine's own caches."""
import math
import random

import numpy as np
import torch

own = False

PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _ints(text):
    return [int(x) for x in str(text).split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


# ------------------------------------------------------------------ cases
def listed():
    big = {"heads": 24, "kv": 8, "dim": 128, "dtype": "bf16"}     # the 3B-shaped model's layout
    mid = {"heads": 8, "kv": 2, "dim": 128, "dtype": "bf16"}      # the reduced model's layout
    small = {"heads": 4, "kv": 2, "dim": 64, "dtype": "f16"}      # a small layout in the other type
    return [
        # the cond and uncond prompts of one song, prefilled together
        {"name": "packed-cfg-pair", "op": "packed", "lens": "1024,1024", "causal": True, **big},
        # short prompts of many small requests, one-token ones among them: latency
        {"name": "packed-short", "op": "packed", "lens": "1,17,40,1,129,64,5,77,200,3,31,96", "causal": True, **small},
        # a long prompt in one batch with ordinary, short and empty ones
        {"name": "packed-long", "op": "packed", "lens": "777,16384,1,4099,0,2050,130", "causal": True, **big},
        # the acoustic frames of two songs: every row sees every row of its own song
        {"name": "packed-frames", "op": "packed", "lens": "4098,1501", "causal": False, **big},
        # one token of each CFG row at the headline context: the single-token form
        {"name": "tree-one-token", "op": "tree", "nodes": "1,1", "context": "1030,1029", "chain": True, "layers": 2, "layer": 1, **big},
        # drafted trees of a batch of songs at mixed contexts
        {"name": "tree-batch", "op": "tree", "nodes": "16,12,16,7,16,16,1,16", "context": "4096,3001,1024,5120,63,2047,8191,4500",
         "chain": False, "layers": 1, "layer": 0, **big},
        # full trees over two whole contexts
        {"name": "tree-long", "op": "tree", "nodes": "64,48", "context": "24512,20001", "chain": False, "layers": 1, "layer": 0, **big},
        # one decode step of the CFG pair
        {"name": "append-pair", "op": "append", "rows": 2, "spread": 1030, "k_out": False, "layers": 2, "layer": 1, **mid},
        # the prompts of a batch in one pass, K kept packed for the prompt attention
        {"name": "append-prompts", "op": "append", "rows": 8192, "spread": 4096, "k_out": True, "layers": 1, "layer": 0, **big},
        # forking a prompt for several takes: the tail pages of all layers
        {"name": "copy-tails", "op": "copy", "pages": 8, "count": 0, "layers": 28, **big},
        # accepting a path of each drafted tree, in place
        {"name": "gather-accept", "op": "gather", "seqs": 16, "begin": 160, "keep": 8, "span": 64, "in_place": True, "layers": 28, **big},
        # dropping half the positions of a long cache into fresh pages
        {"name": "gather-evict", "op": "gather", "seqs": 1, "begin": 0, "keep": 4001, "span": 8192, "in_place": False, "layers": 28, **big},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    if case["op"] == "packed":
        return sum(n * n for n in _ints(case["lens"])) * case["heads"] * case["dim"] * (1 if case["causal"] else 2)
    if case["op"] == "tree":
        return sum((c + t) * (64 + t) for c, t in zip(_ints(case["context"]), _ints(case["nodes"]))) * case["heads"] * case["dim"]
    return 0


def draw(rng):
    heads, kv, dim = rng.choice([(24, 8, 128), (24, 8, 128), (16, 8, 128), (8, 2, 128), (4, 2, 64), (8, 8, 64), (8, 1, 128), (16, 4, 64)])
    shape = {"heads": heads, "kv": kv, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "bf16", "f16"])}
    op = rng.choice(["packed", "packed", "tree", "tree", "append", "copy", "gather"])
    top = {c["name"]: _cost(c) for c in listed()}
    if op == "packed":
        while True:
            case = {"op": op, "lens": _text(_log_int(rng, 1, 16384) - (rng.random() < 0.05) for _ in range(_log_int(rng, 1, 32))),
                    "causal": rng.random() < 0.75, **shape}
            lens = _ints(case["lens"])
            if 0 < sum(lens) <= 24576 and _cost(case) <= top["packed-long"]:
                return case
    if op == "tree":
        while True:
            n = _log_int(rng, 1, 32)
            case = {"op": op, "nodes": _text(_log_int(rng, 1, 64) for _ in range(n)),
                    "context": _text(_log_int(rng, 1, 24512) - 1 for _ in range(n)), "chain": rng.random() < 0.4, "layers": rng.choice([1, 2]), "layer": 0, **shape}
            case["layer"] = case["layers"] - 1
            if _cost(case) <= top["tree-long"] and sum(_ints(case["context"])) <= 60000:
                return case
    if op == "append":
        layers = rng.choice([1, 2])
        return {"op": op, "rows": _log_int(rng, 1, 8192), "spread": _log_int(rng, 64, 8192), "k_out": rng.random() < 0.5,
                "layers": layers, "layer": layers - 1, **shape}
    layers = rng.choice([2, 16, 28])
    if op == "copy":
        return {"op": op, "pages": _log_int(rng, 1, 48), "count": rng.choice([0, 64, 64, rng.randint(1, 63)]), "layers": layers, **shape}
    if rng.random() < 0.5:
        keep = _log_int(rng, 1, 24)
        return {"op": op, "seqs": _log_int(rng, 1, 24), "begin": rng.randint(0, 200), "keep": keep, "span": 64, "in_place": True, "layers": layers, **shape}
    span = _log_int(rng, 2, 8192)
    return {"op": op, "seqs": 1, "begin": 0, "keep": rng.randint(1, max(1, span // 2)), "span": span, "in_place": False, "layers": layers, **shape}


# ------------------------------------------------------------------ inputs
def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if math.prod(shape) < 1 << 24 else dtype).to(dtype)


def _pool(gen, pages, case):
    return _randn(gen, (pages, case["layers"], 2, case["kv"], PAGE, case["dim"]), DTYPES[case["dtype"]])


def _dev(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _tables(rng, pages_of):
    """Page tables [seqs, longest] over a shuffled pool that holds exactly these pages."""
    total = sum(pages_of)
    order = list(range(total))
    rng.shuffle(order)
    table = np.zeros((len(pages_of), max(1, max(pages_of))), dtype=np.int32)
    at = 0
    for s, n in enumerate(pages_of):
        table[s, :n] = order[at:at + n]
        at += n
    return max(1, total), table


def _masks(rng, nodes):
    """Ancestors-and-self bits of random trees, 64 bits a node."""
    out = []
    for n in nodes:
        bits = []
        for j in range(n):
            parent = rng.randint(max(-1, j - 8), j - 1)
            bits.append((bits[parent] if parent >= 0 else 0) | (1 << j))
        out += bits
    return np.array(out, dtype=np.uint64).view(np.int64)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dtype, heads, kv, dim = DTYPES[case["dtype"]], case["heads"], case["kv"], case["dim"]
    st = {"case": case}
    if case["op"] == "packed":
        lens = _ints(case["lens"])
        # q, k and v as a layer's projection leaves them: parts of one row
        qkv = _randn(gen, (sum(lens), heads + 2 * kv, dim), dtype)
        st.update(q=qkv[:, :heads], k=qkv[:, heads:heads + kv], v=qkv[:, heads + kv:], lens=lens,
                  cu=_dev(np.concatenate([[0], np.cumsum(lens)])))
    elif case["op"] == "tree":
        nodes, ctx = _ints(case["nodes"]), _ints(case["context"])
        pages, table = _tables(rng, [-(-(c + t) // PAGE) for c, t in zip(ctx, nodes)])
        mask = None if case["chain"] else _masks(rng, nodes)
        st.update(pool=_pool(gen, pages, case), table=_dev(table), context=_dev(ctx), cu=_dev(np.concatenate([[0], np.cumsum(nodes)])),
                  mask=None if mask is None else _dev(mask, torch.int64), q=_randn(gen, (sum(nodes), heads, dim), dtype), nodes=nodes, ctx=ctx)
    elif case["op"] == "append":
        rows, spread = case["rows"], case["spread"]
        pages = -(-rows // PAGE) + 2
        half = dim // 2
        freq = 10000.0 ** (-np.arange(half) / half)
        angle = np.arange(spread)[:, None] * freq[None]
        st.update(qkv=_randn(gen, (rows, heads + 2 * kv, dim), dtype), pool=_pool(gen, pages, case),
                  q_norm=1 + 0.1 * _randn(gen, (dim,), torch.float32), k_norm=1 + 0.1 * _randn(gen, (dim,), torch.float32),
                  cos=torch.tensor(np.cos(angle), dtype=torch.float32).cuda(), sin=torch.tensor(np.sin(angle), dtype=torch.float32).cuda(),
                  positions=_dev([rng.randrange(spread) for _ in range(rows)] if rows < spread else [i % spread for i in range(rows)]),
                  slots=_dev(np.random.RandomState(seed % (1 << 31)).permutation(pages * PAGE)[:rows], torch.int64) if rows < 1024
                  else torch.arange(rows, dtype=torch.int64, device="cuda") + 37)
    elif case["op"] == "copy":
        n = case["pages"]
        order = rng.sample(range(2 * n), 2 * n)
        counts = [case["count"] or rng.randint(1, PAGE) for _ in range(n)]
        st.update(pool=_pool(gen, 2 * n, case), src=_dev(order[:n]), dst=_dev(order[n:]), count=_dev(counts), src_h=order[:n], dst_h=order[n:], counts=counts)
    else:
        seqs, begin, keep, span = case["seqs"], case["begin"], case["keep"], case["span"]
        if case["in_place"]:  # nodes past the places that the path moves to
            kept = [sorted(rng.sample(range(begin + keep, begin + span), min(keep, span - keep))) for _ in range(seqs)]
            pages, table = _tables(rng, [-(-(begin + span) // PAGE)] * seqs)
            src, dst = table, table
        else:
            kept = [sorted(rng.sample(range(span), keep)) for _ in range(seqs)]
            pages, both = _tables(rng, [-(-span // PAGE)] * seqs + [-(-(begin + keep) // PAGE)] * seqs)
            src, dst = both[:seqs], both[seqs:]
        cu = np.concatenate([[0], np.cumsum([len(x) for x in kept])])
        st.update(pool=_pool(gen, pages, case), src=_dev(src), dst=None if case["in_place"] else _dev(dst), begin=_dev([begin] * seqs),
                  cu=_dev(cu), keep=_dev([p for x in kept for p in x]), kept=kept, src_h=src, dst_h=dst)
    if own:
        from yue2_rs_b200 import ops
        st["ops"] = ops
        if "pool" in st:
            st["handle"] = ops.KvPool(st["pool"])
    return st


# ------------------------------------------------------------------ the plain forms
def _softmax_rows(s, visible):
    s = torch.where(visible, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _plain_packed(st):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    group, scale = heads // kv, 1 / math.sqrt(dim)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    at = 0
    for n in st["lens"]:
        col = torch.arange(n, device=q.device)
        for g in range(kv if n else 0):
            kk, vv = k[at:at + n, g].float(), v[at:at + n, g].float()
            for r0 in range(0, n, 4096):
                r1 = min(n, r0 + 4096)
                qq = q[at + r0:at + r1, g * group:(g + 1) * group].float().transpose(0, 1)
                see = col[None] <= col[r0:r1, None] if case["causal"] else torch.ones((r1 - r0, n), dtype=torch.bool, device=q.device)
                o = _softmax_rows(qq @ kk.T * scale, see) @ vv
                out[at + r0:at + r1, g * group:(g + 1) * group] = o.transpose(0, 1).to(q.dtype)
        at += n
    return out


def _plain_tree(st):
    case, q = st["case"], st["q"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    group, scale = heads // kv, 1 / math.sqrt(dim)
    out = torch.empty_like(q)
    at = 0
    for s, (t, c) in enumerate(zip(st["nodes"], st["ctx"])):
        n = c + t
        pages = st["table"][s, :-(-n // PAGE)].long()
        both = st["pool"][pages, case["layer"]].float()  # [pages, 2, kv, 64, dim]
        both = both.permute(1, 2, 0, 3, 4).reshape(2, kv, -1, dim)[:, :, :n]
        j = torch.arange(t, device=q.device)
        if st["mask"] is None:
            tail = j[None] <= j[:, None]
        else:
            tail = (st["mask"][at:at + t, None] >> j[None]) & 1 == 1
        see = torch.cat([torch.ones((t, c), dtype=torch.bool, device=q.device), tail], 1)
        qq = q[at:at + t].float().reshape(t, kv, group, dim).permute(1, 2, 0, 3)  # [kv, group, t, dim]
        p = _softmax_rows(qq @ both[0][:, None].transpose(-1, -2) * scale, see)
        o = p @ both[1][:, None]
        out[at:at + t] = o.permute(2, 0, 1, 3).reshape(t, heads, dim).to(q.dtype)
        at += t
    return out


def _plain_append(st):
    case, qkv, pool = st["case"], st["qkv"], st["pool"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    half = dim // 2
    pos = st["positions"].long()
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]

    def turn(x, gain):
        x = x.float()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(qkv.dtype)

    q, k, v = turn(qkv[:, :heads], st["q_norm"]), turn(qkv[:, heads:heads + kv], st["k_norm"]), qkv[:, heads + kv:]
    page, place = st["slots"] // PAGE, st["slots"] % PAGE
    pool[page, case["layer"], 0, :, place] = k
    pool[page, case["layer"], 1, :, place] = v
    return {"q": q, "k": k, "pool": pool} if case["k_out"] else {"q": q, "pool": pool}


def _plain_copy(st):
    pool = st["pool"]
    for a, b, n in zip(st["src_h"], st["dst_h"], st["counts"]):
        pool[b, :, :, :, :n] = pool[a, :, :, :, :n]
    return pool


def _plain_gather(st):
    pool, at = st["pool"], 0
    for s, kept in enumerate(st["kept"]):
        if not kept:
            continue
        src = st["keep"][at:at + len(kept)].long()
        to = st["begin"][s].long() + torch.arange(len(kept), device=src.device)
        table = st["src"][s].long()
        into = table if st["dst"] is None else st["dst"][s].long()
        pool[into[to // PAGE], :, :, :, to % PAGE] = pool[table[src // PAGE], :, :, :, src % PAGE]
        at += len(kept)
    return pool


# ------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        return {"packed": _plain_packed, "tree": _plain_tree, "append": _plain_append, "copy": _plain_copy, "gather": _plain_gather}[op](st)
    ops = st["ops"]
    if op == "packed":
        return ops.attention_packed(st["q"], st["k"], st["v"], st["cu"], causal=case["causal"])
    if op == "tree":
        return ops.attention_tree(st["q"], st["handle"], case["layer"], st["table"], st["context"], st["cu"], mask=st["mask"])
    if op == "append":
        k_out = torch.empty((case["rows"], case["kv"], case["dim"]), dtype=st["qkv"].dtype, device="cuda") if case["k_out"] else None
        q = ops.qk_rope_append(st["qkv"], st["q_norm"], st["k_norm"], 1e-6, st["cos"], st["sin"], st["positions"], st["handle"], case["layer"],
                               st["slots"], k_out=k_out)
        return {"q": q, "k": k_out, "pool": st["pool"]} if case["k_out"] else {"q": q, "pool": st["pool"]}
    if op == "copy":
        ops.kv_copy(st["handle"], st["src"], st["dst"], st["count"])
    else:
        ops.kv_gather(st["handle"], st["src"], st["dst"], st["begin"], st["cu"], st["keep"])
    return st["pool"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if case["op"] == "packed":
        lens = _ints(case["lens"])
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": sum(lens) * 2 * (heads + kv) * dim * 2, "flops": 4 * pairs * heads * dim}
    if case["op"] == "tree":
        nodes, ctx = _ints(case["nodes"]), _ints(case["context"])
        pairs = sum(t * c + (t * (t + 1) // 2 if case["chain"] else t) for c, t in zip(ctx, nodes))
        return {"bytes": sum(c + t for c, t in zip(ctx, nodes)) * 2 * kv * dim * 2 + sum(nodes) * 2 * heads * dim * 2, "flops": 4 * pairs * heads * dim}
    if case["op"] == "append":
        row = (heads + 2 * kv) * dim * 2 * 2 + (kv * dim * 2 if case["k_out"] else 0)
        return {"bytes": case["rows"] * row + min(case["rows"], case["spread"]) * dim * 4, "flops": case["rows"] * (heads + kv) * dim * 7}
    place = case["layers"] * 2 * kv * dim * 2
    if case["op"] == "copy":
        return {"bytes": case["pages"] * (case["count"] or 32) * place * 2, "flops": 0}
    keep = min(case["keep"], case["span"] - case["keep"]) if case["in_place"] else case["keep"]
    return {"bytes": case["seqs"] * keep * place * 2, "flops": 0}


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if case["op"] in ("copy", "gather"):
        # where each position's values come from, then one indexed read of the whole pool
        pool = st["pool"]
        origin = np.arange(pool.shape[0] * PAGE)
        before = origin.copy()
        if case["op"] == "copy":
            for a, b, n in zip(st["src_h"], st["dst_h"], st["counts"]):
                origin[b * PAGE:b * PAGE + n] = before[a * PAGE:a * PAGE + n]
        else:
            for s, kept in enumerate(st["kept"]):
                for i, p in enumerate(kept):
                    t = case["begin"] + i
                    origin[st["dst_h"][s, t // PAGE] * PAGE + t % PAGE] = before[st["src_h"][s, p // PAGE] * PAGE + p % PAGE]
        by_place = pool.permute(0, 4, 1, 2, 3, 5).reshape(-1, case["layers"], 2, kv, dim)[torch.from_numpy(origin).cuda()]
        return by_place.reshape(-1, PAGE, case["layers"], 2, kv, dim).permute(0, 2, 3, 4, 1, 5).to(torch.float64)
    if case["op"] == "append":
        # the rotation as a product of complex numbers
        x = st["qkv"].to(torch.float64)
        turn = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"].long()].unsqueeze(1)

        def rotated(y, gain):
            y = y * (y.pow(2).sum(-1, keepdim=True) / dim + 1e-6).rsqrt() * gain.double()
            z = torch.complex(y[..., :dim // 2].contiguous(), y[..., dim // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        q, k = rotated(x[:, :heads], st["q_norm"]), rotated(x[:, heads:heads + kv], st["k_norm"])
        flat = st["pool"].double()
        rows = flat[:, case["layer"]].permute(0, 3, 1, 2, 4).reshape(-1, 2, kv, dim).clone()  # by slot
        rows[st["slots"]] = torch.stack([k, x[:, heads + kv:]], 1)
        flat[:, case["layer"]] = rows.reshape(-1, PAGE, 2, kv, dim).permute(0, 2, 3, 1, 4)
        return {"q": q, "k": k, "pool": flat} if case["k_out"] else {"q": q, "pool": flat}
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    counts, contexts = (st["lens"], [0] * len(st["lens"])) if case["op"] == "packed" else (st["nodes"], st["ctx"])
    first = 0
    for s, (rows, ctx) in enumerate(zip(counts, contexts)):
        last = first + rows
        where = torch.arange(ctx + rows, device="cuda")
        for h in range(heads if rows else 0):
            if case["op"] == "packed":
                keys, values = st["k"][first:last, h * kv // heads].double(), st["v"][first:last, h * kv // heads].double()
            else:
                at = st["table"][s].long()[where // PAGE]
                keys, values = (st["pool"][at, case["layer"], w, h * kv // heads, where % PAGE].double() for w in (0, 1))
            for a in range(0, rows, 2048):
                b = min(rows, a + 2048)
                logit = torch.einsum("id,jd->ij", st["q"][first + a:first + b, h].double(), keys).div_(dim ** 0.5)
                if case["op"] == "tree" and not case["chain"]:
                    unseen = (torch.bitwise_right_shift(st["mask"][first + a:first + b, None], (where - ctx).clamp(min=0)[None]) & 1) == 0
                    unseen[:, :ctx] = False
                    logit.masked_fill_(unseen, float("-inf"))
                elif case["op"] == "tree" or case["causal"]:
                    logit.masked_fill_(where[None] > ctx + torch.arange(a, b, device="cuda")[:, None], float("-inf"))
                weight = torch.exp(logit - torch.logsumexp(logit, 1, keepdim=True))
                out[first + a:first + b, h] = torch.einsum("ij,jd->id", weight, values)
        first = last
    return out
