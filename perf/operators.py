"""Operators on a paged cache whose sequences share blocks, sized for timing: copying, forking and
moving blocks, and attention of new tokens over blocks that several rows share.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare` makes what
a program holds before the call, `run` is one pass (in plain torch operations, or with `own` set
through the framework's entry points), `work` says what a pass cannot do without and `exact` gives
the attention in 64 bits.

The shapes are the engine's: Qwen2.5-1.5B's cache (28 layers, 2 kv heads of 128, blocks of 16 tokens)
under 12 query heads, and other head counts, layer counts and block sizes of the same kernels.
"""
import math
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    engine = {"layers": 28, "kv_heads": 2, "block": 16, "dtype": "bf16"}
    return [
        # a short chat's seven blocks brought over into another cache
        {"name": "copy_7", "kind": "copy", "pairs": 7, "spare": 9, **engine},
        # a cache of many chats rebuilt in a larger one
        {"name": "copy_1500", "kind": "copy", "pairs": 1500, "spare": 100, **engine},
        # a chat answered twice: one more sequence over its history
        {"name": "fork_1_of_203", "kind": "fork", "children": 1, "tokens": 203, **engine},
        # many replies drawn for one long history
        {"name": "fork_64_of_12345", "kind": "fork", "children": 64, "tokens": 12345, **engine},
        # a few holes closed after a chat was dropped
        {"name": "move_20", "kind": "move", "pairs": 20, "rows": 6, "spare": 10, **engine},
        # half of a large pool moved together, in fp16 with larger blocks
        {"name": "move_400_fp16", "kind": "move", "pairs": 400, "rows": 61, "spare": 50,
         "layers": 28, "kv_heads": 2, "block": 64, "dtype": "fp16"},
        # two replies to a short prompt decoding side by side, the smallest call there is
        {"name": "decode_2_of_100", **_attend(2, 1, (100, 100), (1, 20), (1, 1), 0)},
        # sixteen replies over one history of ordinary length
        {"name": "decode_16_of_2048", **_attend(16, 1, (2048, 2048), (1, 512), (1, 1), 1)},
        # a batch of chats, each with a few replies at once, of uneven counts and lengths, in fp16
        {"name": "decode_40_in_9",
         **_attend(40, 9, (300, 6000), (1, 700), (1, 1), 2, dtype="fp16")},
        # drafts of several tokens checked at once, ragged, behind a shared history
        {"name": "chunk_12_of_3001", **_attend(12, 1, (3001, 3001), (20, 300), (1, 17), 3)},
        # next messages of chats that share one long system prompt
        {"name": "chunk_8x150_of_5000", **_attend(8, 1, (5000, 5000), (150, 900), (90, 150), 4)},
        # a wide search over a context as long as the model takes
        {"name": "decode_64_of_31000", **_attend(64, 1, (31000, 31000), (1, 1024), (1, 1), 5)},
    ]


def _attend(rows, groups, prefix, tail, new, mix, heads=12, kv_heads=2, block=16, dtype="bf16"):
    """An attention case: `rows` rows in `groups` groups, each group sharing a prefix of between
    prefix[0] and prefix[1] keys (whole blocks of them); a row has between tail[0] and tail[1] keys of
    its own, between new[0] and new[1] of them this step's queries.  `mix` fixes the lengths."""
    return {"kind": "attend", "rows": rows, "groups": groups, "prefix_lo": prefix[0],
            "prefix_hi": prefix[1], "tail_lo": tail[0], "tail_hi": tail[1], "new_lo": new[0],
            "new_hi": new[1], "mix": mix, "heads": heads, "kv_heads": kv_heads, "block": block,
            "dtype": dtype}


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


_LARGEST = {c["kind"]: c for c in listed()[1::2] + listed()[-1:]}


def draw(rng):
    kind = rng.choice(["copy", "fork", "move", "attend", "attend", "attend"])
    while True:
        case = _drawn(rng, kind)
        most, need = work(_LARGEST[kind]), work(case)
        if need["bytes"] <= most["bytes"] and need["flops"] <= most["flops"]:
            return case


def _drawn(rng, kind):
    dtype = rng.choice(["bf16", "fp16"])
    if kind != "attend":
        shape = {"kind": kind, "layers": rng.randint(1, 28), "kv_heads": rng.choice([1, 2, 2, 4, 8]),
                 "block": rng.choice([16, 16, 32, 64, 128]), "dtype": dtype}
        if kind == "copy":
            return {**shape, "pairs": _log(rng, 1, 1500), "spare": rng.randint(0, 200)}
        if kind == "fork":
            return {**shape, "children": _log(rng, 1, 64), "tokens": _log(rng, 1, 12345)}
        return {**shape, "pairs": _log(rng, 1, 1500), "rows": _log(rng, 1, 100),
                "spare": rng.randint(0, 200)}
    heads, kv_heads = rng.choice([(12, 2), (12, 2), (16, 4), (8, 8), (32, 8), (14, 2), (5, 1)])
    rows = _log(rng, 2, 64)
    p0, p1 = sorted((_log(rng, 16, 31000), _log(rng, 16, 31000)))
    new = rng.choice([1, 1, _log(rng, 1, 150)])
    return _attend(rows, _log(rng, 1, rows), (p0, p1), (new, new + _log(rng, 1, 1024)),
                   (max(1, new // 3), new), rng.randint(10, 10 ** 6), heads, kv_heads,
                   rng.choice([16, 16, 32, 64]), dtype)


# -- inputs ---------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _pool(g, dtype, layers, blocks, case):
    """A cache's buffer [layers, 2, slots, kv_heads, 128], filled layer by layer."""
    buf = torch.empty(layers, 2, blocks * case["block"], case["kv_heads"], 128, dtype=dtype,
                      device=DEV)
    for layer in buf:
        layer.copy_(_randn(g, dtype, *layer.shape))
    return buf


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _split(r, total, parts):
    """`total` as `parts` whole numbers of at least one, at random."""
    cuts = sorted(r.sample(range(1, total), parts - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _batch(case):
    """Rows of an attention case: their groups' sizes, the groups' shared keys (whole blocks), each
    row's keys behind the shared ones and its new tokens."""
    r, bs = random.Random(case["mix"]), case["block"]
    sizes = _split(r, case["rows"], case["groups"])
    prefix = [max(bs, r.randint(case["prefix_lo"], case["prefix_hi"]) // bs * bs)
              for _ in sizes]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["rows"])]
    tail = [max(n, r.randint(case["tail_lo"], case["tail_hi"])) for n in new]
    return sizes, prefix, new, tail


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    dtype, bs, r = DTYPES[case["dtype"]], case["block"], random.Random(seed)
    s = {"kind": kind, "block": bs}
    if kind == "copy":
        n = case["pairs"]
        total = n + case["spare"]
        s["src"] = _pool(g, dtype, case["layers"], total, case)
        s["dst"] = torch.zeros_like(s["src"])
        s["pairs"] = _i32(list(zip(r.sample(range(total), n), r.sample(range(total), n))))
        return s
    if kind == "fork":
        # the parent's blocks scattered over the pool, one more block for every child's last tokens
        n, length = case["children"], case["tokens"]
        whole, rest = divmod(length, bs)
        held = whole + (rest > 0)
        ids = list(range(held + n + 3))
        r.shuffle(ids)
        slots = r.sample(range(n + 4), n + 1)
        s["pool"] = _pool(g, dtype, case["layers"], held + n + 3, case)
        s["tables"] = torch.zeros(n + 4, held + 8, dtype=torch.int32, device=DEV)
        s["lens"] = torch.zeros(n + 4, dtype=torch.int32, device=DEV)
        s["tables"][slots[0], :held] = _i32(ids[:held])
        s["lens"][slots[0]] = length
        s["children"] = _i32([[slots[0], c, length, ids[held + i] if rest else -1]
                              for i, c in enumerate(slots[1:])])
        return s
    if kind == "move":
        # as many holes at the front as there are used blocks behind the used ones' number
        n, rows = case["pairs"], case["rows"]
        used = max(n, rows) + case["spare"]
        src = sorted(r.sample(range(used, used + n + 9), n))
        dst = sorted(r.sample(range(used), n))
        live = sorted(set(range(used)) - set(dst)) + src
        new_ids = list(range(used + n + 9))
        for a, b in zip(src, dst):
            new_ids[a] = b
        r.shuffle(live)
        counts = _split(random.Random(31 * n + rows), len(live), rows)
        slots = r.sample(range(rows + 5), rows)
        s["pool"] = _pool(g, dtype, case["layers"], used + n + 9, case)
        s["tables"] = torch.zeros(rows + 5, max(counts) + 4, dtype=torch.int32, device=DEV)
        for slot, count in zip(slots, counts):
            s["tables"][slot, :count] = _i32([live.pop() for _ in range(count)])
        s["rows"] = _i32(list(zip(slots, counts)))
        s["pairs"], s["new_ids"] = _i32(list(zip(src, dst))), _i32(new_ids)
        return s
    sizes, prefix, new, tail = _batch(case)
    tables, free = [], 0
    for size, p in zip(sizes, prefix):
        shared = list(range(free, free + p // bs))
        free += len(shared)
        for _ in range(size):
            mine = -(-tail[len(tables)] // bs)
            tables.append(shared + list(range(free, free + mine)))
            free += mine
    blocks = free + 8
    ids = list(range(blocks))
    r.shuffle(ids)
    width = max(len(t) for t in tables)
    shared_of = [p for size, p in zip(sizes, prefix) for _ in range(size)]
    lens = [p + t for p, t in zip(shared_of, tail)]
    cu_q, cu_rows = [0], [0]
    for n in new:
        cu_q.append(cu_q[-1] + n)
    for n in sizes:
        cu_rows.append(cu_rows[-1] + n)
    buf = _pool(g, dtype, 1, blocks, case)
    s.update(k=buf[0, 0], v=buf[0, 1], q=_randn(g, dtype, cu_q[-1], case["heads"], 128),
             table=_i32([[ids[x] for x in t] + [0] * (width - len(t)) for t in tables]),
             lens=_i32(lens), cu_q=_i32(cu_q), cu_rows=_i32(cu_rows), prefix=_i32(prefix),
             longest=max(lens), most_new=max(new))
    return s


# -- one pass -------------------------------------------------------------------------------------
def run(state):
    s, kind = state, state["kind"]
    if own:
        if "my-inference-engine_amd" not in sys.path:
            sys.path.insert(0, "my-inference-engine_amd")
        from kernels import blocks, shared
        if kind == "copy":
            return blocks.copy_blocks(s["src"], s["dst"], s["pairs"], s["block"])
        if kind == "fork":
            blocks.fork_rows(s["pool"], s["tables"], s["lens"], s["children"], s["block"])
            return s["pool"], s["tables"], s["lens"]
        if kind == "move":
            blocks.move_blocks(s["pool"], s["tables"], s["rows"], s["pairs"], s["new_ids"],
                               s["block"])
            return s["pool"], s["tables"]
        return shared.fa2_paged_shared(s["q"], s["k"], s["v"], s["cu_q"], s["table"], s["lens"],
                                       s["most_new"], s["cu_rows"], s["prefix"],
                                       block_size=s["block"], max_kv_len=s["longest"])
    if kind == "copy":
        src, dst = _blocks(s["src"], s), _blocks(s["dst"], s)
        pairs = s["pairs"].long()
        dst[:, pairs[:, 1]] = src[:, pairs[:, 0]]
        return s["dst"]
    if kind == "fork":
        return _plain_fork(s)
    if kind == "move":
        pool, pairs = _blocks(s["pool"], s), s["pairs"].long()
        pool[:, pairs[:, 1]] = pool[:, pairs[:, 0]]
        rows = s["rows"].long()
        held = s["tables"][rows[:, 0]]
        at = torch.arange(held.shape[1], device=DEV)[None, :]
        s["tables"][rows[:, 0]] = torch.where(at < rows[:, 1:], s["new_ids"][held.long()], held)
        return s["pool"], s["tables"]
    return _plain_attention(s)


def _blocks(buf, s):
    """A cache's buffer as [planes, blocks, one block's values]."""
    return buf.view(buf.shape[0] * 2, buf.shape[2] // s["block"], -1)


def _plain_fork(s):
    pool, tables, lens, bs = _blocks(s["pool"], s), s["tables"], s["lens"], s["block"]
    children = s["children"].long()
    parent, child, length, new = children.unbind(1)
    whole = (length // bs)[:, None]
    at = torch.arange(tables.shape[1], device=DEV)[None, :]
    theirs = tables[parent]
    last = theirs.gather(1, whole).long()[:, 0]
    mine = torch.where(at < whole, theirs, tables[child])
    mine = torch.where((at == whole) & (new[:, None] >= 0), new[:, None].int(), mine)
    tables[child] = mine
    lens[child] = length.int()
    # the tokens of a started block; a child without one rewrites a parent's block with itself
    token = pool.shape[2] // bs
    to = torch.where(new >= 0, new, last)
    old, cur = pool[:, last], pool[:, to]
    part = torch.arange(pool.shape[2], device=DEV)[None, :] // token < (length % bs)[:, None]
    pool[:, to] = torch.where(part[None], old, cur)
    return s["pool"], tables, lens


def _plain_attention(s):
    """Every row's keys gathered out of the pool and attended to in 32 bits, all rows padded to the
    longest."""
    q, table, lens, bs = s["q"], s["table"].long(), s["lens"], s["block"]
    B, Tm, S = table.shape[0], s["most_new"], s["longest"]
    Hq, Hkv, d = q.shape[1], s["k"].shape[1], q.shape[2]
    starts, counts = s["cu_q"][:-1], s["cu_q"][1:] - s["cu_q"][:-1]
    at = torch.arange(S, device=DEV)
    slots = table[:, at // bs] * bs + at % bs
    token = torch.arange(Tm, device=DEV)
    real = token[None, :] < counts[:, None]
    index = (starts[:, None] + token[None, :])[real]
    qd = torch.zeros(B, Tm, Hq, d, device=DEV)
    qd[real] = q.float()[index]
    qd = qd.view(B, Tm, Hkv, Hq // Hkv, d).transpose(1, 2).reshape(B, Hkv, -1, d)
    k = s["k"][slots].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"][slots].float().transpose(1, 2).contiguous()
    scores = torch.matmul(qd, k).view(B, Hkv, Tm, -1, S) * (1.0 / math.sqrt(d))
    seen = at[None, None, :] < (lens - counts + 1)[:, None, None] + token[None, :, None]
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, -1, S), v).view(B, Hkv, Tm, -1, d)
    out = torch.empty(q.shape, device=DEV)
    out[index] = o.transpose(1, 2).reshape(B, Tm, Hq, d)[real]
    return out.to(q.dtype)


# -- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    bs = case["block"]
    if case["kind"] == "attend":
        sizes, prefix, new, tail = _batch(case)
        shared_of = [p for size, p in zip(sizes, prefix) for _ in range(size)]
        keys = sum(prefix) + sum(tail)
        # query i of n sees all but the n - 1 - i last keys
        pairs = sum(n * (p + t) - n * (n - 1) // 2 for p, t, n in zip(shared_of, tail, new))
        entries = keys // bs + 4 * case["rows"]
        return {"bytes": keys * case["kv_heads"] * 512 + sum(new) * case["heads"] * 512 + 4 * entries,
                "flops": 512 * case["heads"] * pairs}
    token = case["layers"] * 2 * case["kv_heads"] * 256
    if case["kind"] == "copy":
        return {"bytes": 2 * case["pairs"] * (bs * token + 4), "flops": 0}
    if case["kind"] == "fork":
        rest, held = case["tokens"] % bs, -(-case["tokens"] // bs)
        return {"bytes": (case["children"] + 1) * (rest * token + 4 * held) + 20 * case["children"],
                "flops": 0}
    used = max(case["pairs"], case["rows"]) + case["spare"]
    return {"bytes": 2 * case["pairs"] * bs * token + 12 * used + 8 * (case["pairs"] + case["rows"]),
            "flops": 0}


# -- the same in 64 bits --------------------------------------------------------------------------
def exact(case, seed):
    """The attention row by row; the block operations compute nothing."""
    if case["kind"] != "attend":
        return None
    s = prepare(case, seed)
    bs, group = case["block"], case["heads"] // case["kv_heads"]
    cu, lens = s["cu_q"].tolist(), s["lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        blocks = s["table"][b, :-(-n // bs)].long()
        slots = (blocks[:, None] * bs + torch.arange(bs, device=DEV)).reshape(-1)[:n]
        kk, vv = s["k"][slots].double(), s["v"][slots].double()
        qq = s["q"][cu[b]:cu[b + 1]].double()
        hidden = torch.ones(len(qq), n, dtype=torch.bool, device=DEV).triu(n - len(qq) + 1)
        for h in range(case["heads"]):
            score = qq[:, h] @ kk[:, h // group].t().contiguous() * 128 ** -0.5
            weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            out[cu[b]:cu[b + 1], h] = weight @ vv[:, h // group].contiguous()
    return out
