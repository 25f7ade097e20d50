"""Operators of speculative decoding with a tree of drafted tokens, as cases that can be timed.

A drafter proposes a tree of tokens for every sequence; one pass of the model gives every node its target distribution;
the walk from the root keeps the nodes that are accepted. Three operators of the library make up that step:

* ``tree``    attention of the drafted nodes: node i of a slot sees the slot's prefix, its own ancestors and itself
              (their rows were appended behind the prefix), over an f32, q8_0 or q4_0 cache.
* ``verify``  the walk: a drafted child is kept with probability min(1, target / draft), what its rejection leaves is
              the target less the draft, and the next token is drawn from what is left where the walk ends. The
              random numbers are inputs.
* ``keep``    the cache rows of the kept path move together behind the prefix, in every layer.

``own`` says whether `run` makes the library's calls or computes the operators from elementary torch operations.
Heads, layers and the depths are those of the library's other cases: 24 query heads over 4 KV heads of 256, 16 layers.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

LAYERS = 16
DTYPE_ID = {"f32": 0, "q8": 1, "q4": 2}      # as the chunk entries number the caches
BLOCK_BYTES = {"q8": 34, "q4": 18}           # of 32 values
HEADROOM = 40                                # cache rows kept past the longest slot's


def _tree(name, dtype, nodes, low, high, slots=1, width=4, heads=24, kv=4, dim=256):
    return {"name": name, "op": "tree", "dtype": dtype, "nodes": nodes, "low": low, "high": high, "slots": slots,
            "width": width, "heads": heads, "kv": kv, "dim": dim, "shape_seed": 5}


def _verify(name, slots, nodes, vocab, draft=True, width=4):
    return {"name": name, "op": "verify", "slots": slots, "nodes": nodes, "vocab": vocab, "draft": draft,
            "width": width, "shape_seed": 7}


def _keep(name, dtype, nodes, slots):
    return {"name": name, "op": "keep", "dtype": dtype, "nodes": nodes, "slots": slots, "low": 300, "high": 2000,
            "width": 2, "heads": 24, "kv": 4, "dim": 256, "shape_seed": 9}


def listed():
    return [
        # the first drafted chain of a short conversation: launches and set-up count
        _tree("tree q8 4 at 640", "q8", 4, 640, 640, width=1),
        # an everyday step of one conversation
        _tree("tree q8 16 at 8192", "q8", 16, 8192, 8192),
        # the unquantised cache at the depth up to which it is usually taken
        _tree("tree f32 13 at 2048", "f32", 13, 2048, 2048),
        # the small cache format on a document-sized context
        _tree("tree q4 21 at 32768", "q4", 21, 32768, 32768),
        # a server's conversations of unequal length, each with its own tree
        _tree("tree q8 8 slots of 10", "q8", 10, 512, 8192, slots=8),
        # a wide tree over the longest context
        _tree("tree q8 64 at 100000", "q8", 64, 100000, 100000),
        # a small head size, by which small drafting models run
        _tree("tree q8 12 at 1000, heads of 64", "q8", 12, 1000, 1000, heads=8, kv=2, dim=64),
        # one conversation's drafted chain
        _verify("verify 1 x 8 of 151936", 1, 8, 151936, width=1),
        # a batch of trees; rows of an odd length
        _verify("verify 8 x 16 of 50257", 8, 16, 50257),
        # a large batch whose drafts were looked up, without probabilities of their own
        _verify("verify 32 x 8 of 151936, looked up", 32, 8, 151936, draft=False),
        # the end of one conversation's step
        _keep("keep q8 1 x 16", "q8", 16, 1),
        # the end of a server's step, over the unquantised cache
        _keep("keep f32 8 x 10", "f32", 10, 8),
    ]


def _spread(rng: random.Random, low: int, high: int) -> int:
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng: random.Random):
    op = rng.choice(["tree", "tree", "tree", "verify", "verify", "keep"])
    seed = rng.randrange(1 << 20)
    if op == "tree":
        heads, kv, dim = rng.choice([(24, 4, 256), (24, 4, 256), (24, 4, 256), (6, 1, 256), (8, 2, 64)])
        slots = rng.choice([1, 1, rng.randint(2, 16)])
        most = 100000 if slots == 1 else 8192
        if dim == 64:
            most = 4096
        dtype = rng.choice(["q8", "q8", "q4", "f32"])
        if dtype == "f32":
            most = min(most, 8192)
        high = _spread(rng, 30, most)
        return {"op": op, "dtype": dtype, "nodes": _spread(rng, 1, 64 if slots == 1 else 32), "low": max(1, high // 8) if
                slots > 1 else high, "high": high, "slots": slots, "width": rng.randint(1, 6), "heads": heads, "kv": kv,
                "dim": dim, "shape_seed": seed}
    if op == "verify":
        nodes = _spread(rng, 2, 32)
        vocab = rng.choice([32000, 50257, 128256, 151936, _spread(rng, 1000, 200000)])
        return {"op": op, "slots": _spread(rng, 1, min(32, max(1, 80_000_000 // (nodes * vocab)))), "nodes": nodes,
                "vocab": vocab, "draft": rng.random() < 0.7, "width": rng.randint(1, 6), "shape_seed": seed}
    high = _spread(rng, 40, 2000)
    return {"op": op, "dtype": rng.choice(["q8", "q8", "q4", "f32"]), "nodes": rng.randint(2, 64), "slots":
            _spread(rng, 1, 8), "low": max(1, high // 4), "high": high, "width": rng.randint(1, 6), "heads": 24, "kv": 4,
            "dim": 256, "shape_seed": seed}


# ---- shapes: lengths and trees of a case, on the host ------------------------------------------------------------

def _shapes(case):
    """(prefix length, live nodes, parents) of every slot; node 0 is the root, a node's parent is an earlier one."""
    r = random.Random(case["shape_seed"])
    nodes, slots, width = case["nodes"], case["slots"], case["width"]
    got = []
    for _ in range(slots):
        base = r.randint(case.get("low", 0), case.get("high", 0))
        live = nodes if slots == 1 else r.randint((nodes + 1) // 2, nodes)
        parents = [-1] + [r.randrange(max(0, i - width), i) for i in range(1, nodes)]
        got.append((base, live, parents))
    return got


def _depth(parents, i):
    d = 1
    while parents[i] >= 0:
        i, d = parents[i], d + 1
    return d


def _paths(case):
    """A path from the root of every slot's tree, as the walk would keep it, of the live nodes."""
    r = random.Random(case["shape_seed"] + 1)
    got = []
    for _, live, parents in _shapes(case):
        path = [0]
        while True:
            below = [i for i in range(live) if parents[i] == path[-1]]
            if not below or r.random() < 0.1:
                break
            path.append(r.choice(below))
        got.append(path)
    return got


def _row_values(case):
    return case["kv"] * case["dim"]


def _row_bytes(case):
    """Of one KV head's K (or V) row."""
    return case["dim"] * 4 if case["dtype"] == "f32" else case["dim"] // 32 * BLOCK_BYTES[case["dtype"]]


# ---- inputs ------------------------------------------------------------------------------------------------------

def _encode(x, dtype):
    """Rows of f32 values, in blocks of 32 along the last axis, as q8_0 or q4_0 bytes."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    if dtype == "q8":
        scale = b.abs().amax(-1, keepdim=True) / 127.0
        code = torch.round(b / scale).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        scale = b.abs().amax(-1, keepdim=True) / 7.0
        c = (torch.round(b / scale) + 8.0).clamp(0, 15).to(torch.uint8)
        code = c[..., :16] | c[..., 16:] << 4
    return torch.cat([scale.to(torch.float16).view(torch.uint8), code], -1).reshape(*x.shape[:-1], -1)


def _cache(case, gen, stride, layers):
    """[layers][K, V][slots][rows of every KV head], head after head, or [row][KV heads * dim] for f32."""
    slots, kv, dim = case["slots"], case["kv"], case["dim"]
    if case["dtype"] == "f32":
        return torch.randn(layers, 2, slots, stride, kv * dim, device="cuda", generator=gen)
    kept = torch.empty(layers, 2, slots, kv, stride, _row_bytes(case), dtype=torch.uint8, device="cuda")
    for layer in range(layers):
        for which in range(2):
            for slot in range(slots):
                kept[layer, which, slot] = _encode(torch.randn(kv, stride, dim, device="cuda", generator=gen),
                                                   case["dtype"])
    return kept


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = _shapes(case)
    s = {"case": case}
    s["pos"] = _ints([[base, base + live] for base, live, _ in shapes])
    s["parents"] = _ints([parents for _, _, parents in shapes])
    slots, nodes = case["slots"], case["nodes"]
    if case["op"] in ("tree", "keep"):
        stride = case["high"] + nodes + HEADROOM
        s["stride"] = stride
        s["slot_bytes"] = case["kv"] * stride * _row_bytes(case)
        s["kv"] = _cache(case, gen, stride, LAYERS if case["op"] == "keep" else 1)
    if case["op"] == "tree":
        width = case["heads"] * case["dim"]
        s["q"] = 1.5 * torch.randn(slots, nodes, width, device="cuda", generator=gen)
        s["out"] = torch.zeros(slots, nodes, width, device="cuda")
    elif case["op"] == "keep":
        paths = _paths(case)
        s["path"] = _ints([p + [-1] * (nodes - len(p)) for p in paths])
        s["count"] = _ints([len(p) for p in paths])
        s["keys"], s["values"] = ([s["kv"][layer, which] for layer in range(LAYERS)] for which in range(2))
    else:
        vocab = case["vocab"]
        logits = 3.0 * torch.randn(slots, nodes, vocab, device="cuda", generator=gen)
        s["target"] = torch.softmax(logits, -1)
        # the drafter's view of the same context
        near = torch.softmax(logits + 0.8 * torch.randn(slots, nodes, vocab, device="cuda", generator=gen), -1)
        del logits
        # a node's token was drawn from its parent's draft
        above = s["parents"].clamp(min=0).long()
        draws = torch.rand(slots, nodes, 1, device="cuda", generator=gen)
        tokens = torch.empty(slots, nodes, dtype=torch.int32, device="cuda")
        for slot in range(slots):
            run_sum = near[slot].cumsum(-1)[above[slot]]
            tokens[slot] = torch.searchsorted(run_sum, draws[slot] * run_sum[:, -1:])[:, 0].clamp(max=vocab - 1).int()
        s["tokens"] = tokens
        s["draft"] = near if case["draft"] else None
        s["uniform"] = torch.rand(slots, nodes, device="cuda", generator=gen)
        s["path"] = torch.empty(slots, nodes, dtype=torch.int32, device="cuda")
        s["count"] = torch.empty(slots, dtype=torch.int32, device="cuda")
        s["next"] = torch.empty(slots, dtype=torch.int32, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"tree": _plain_tree, "verify": _plain_verify, "keep": _plain_keep}[s["case"]["op"]](s)


def _run_own(s):
    from hipml_b200 import api

    c = s["case"]
    if c["op"] == "tree":
        if "workspace" not in s:   # scratch that an engine keeps
            s["workspace"] = torch.empty(api.attn_tree_workspace_bytes(c["heads"], c["kv"], c["dim"], c["nodes"],
                                                                       c["slots"]), dtype=torch.uint8, device="cuda")
        api.attn_tree(s["pos"], s["parents"], s["q"], s["kv"][0, 0], s["kv"][0, 1], s["out"], c["heads"], c["kv"],
                      c["dim"], s["stride"], 1.0 / math.sqrt(c["dim"]), c["nodes"], c["slots"], s["slot_bytes"],
                      s["workspace"], kv_dtype=DTYPE_ID[c["dtype"]])
        return s["out"]
    if c["op"] == "verify":
        api.tree_verify(s["pos"], s["parents"], s["tokens"], s["target"], s["draft"], s["uniform"], s["path"],
                        s["count"], s["next"], c["nodes"], c["slots"], c["vocab"])
        return {"path": s["path"], "count": s["count"], "next": s["next"]}
    api.kv_path_keep(s["pos"], s["path"], s["count"], s["keys"], s["values"], c["kv"], c["dim"], s["stride"], c["nodes"],
                     c["slots"], s["slot_bytes"], kv_dtype=DTYPE_ID[c["dtype"]])
    return s["kv"]


def _values(cache, dtype, kv, dim):
    """[slots][KV heads][rows][dim] f32 of a cache."""
    if dtype == "f32":
        return cache.unflatten(-1, (kv, dim)).transpose(1, 2)
    blocks = cache.unflatten(-1, (dim // 32, BLOCK_BYTES[dtype]))
    scale = blocks[..., :2].contiguous().view(torch.float16).float()
    code = blocks[..., 2:]
    if dtype == "q8":
        value = code.contiguous().view(torch.int8).float()
    else:
        value = torch.cat([code & 15, code >> 4], -1).float() - 8.0
    return (scale * value).flatten(-2)


def _plain_tree(s):
    c, stride = s["case"], s["stride"]
    slots, nodes, heads, kv, dim = c["slots"], c["nodes"], c["heads"], c["kv"], c["dim"]
    base, live = s["pos"][:, 0].long(), (s["pos"][:, 1] - s["pos"][:, 0]).long()
    # which nodes a node sees: powers of "is the parent or the node itself"
    at = torch.arange(nodes, device="cuda")
    link = (s["parents"].long()[:, :, None] == at) | torch.eye(nodes, dtype=torch.bool, device="cuda")
    above = torch.linalg.matrix_power(link.double(), nodes) > 0
    row = torch.arange(stride, device="cuda") - base[:, None]
    drafted = above.gather(2, row.clamp(0, nodes - 1)[:, None, :].expand(-1, nodes, -1))
    sees = (row < 0)[:, None, :] | drafted & ((row >= 0) & (row < live[:, None]))[:, None, :]
    k = _values(s["kv"][0, 0], c["dtype"], kv, dim)
    q = s["q"].view(slots, nodes, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = (q @ k.transpose(-1, -2)).unflatten(2, (heads // kv, nodes)) * (1.0 / math.sqrt(dim))
    del k
    score = torch.where(sees[:, None, None], score, -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True)).flatten(2, 3)
    del score
    v = _values(s["kv"][0, 1], c["dtype"], kv, dim)
    out = (weight @ v) / weight.sum(-1, keepdim=True)
    out = out.unflatten(2, (heads // kv, nodes)).permute(0, 3, 1, 2, 4).flatten(2)
    return torch.where((at < live[:, None])[:, :, None], out, s["out"])


def _plain_verify(s):
    c = s["case"]
    slots, nodes = c["slots"], c["nodes"]
    target, draft, live = s["target"], s["draft"], s["pos"][:, 1] - s["pos"][:, 0]
    each = torch.arange(slots, device="cuda")
    token = torch.arange(c["vocab"], device="cuda")
    here = torch.zeros(slots, dtype=torch.long, device="cuda")     # the last node kept
    left = target[:, 0].double()                                   # what the next token would be drawn from
    total = torch.ones(slots, dtype=torch.float64, device="cuda")  # `left` is over this
    kept = torch.zeros(slots, nodes, dtype=torch.bool, device="cuda")
    kept[:, 0] = True
    u = s["uniform"].double()
    # the children of the node that was kept last come in order behind it
    for i in range(1, nodes):
        child = (s["parents"][:, i] == here) & (live > i)
        x = s["tokens"][:, i].long()
        odds = 1.0 if draft is None else draft[each, here, x].double()
        take = child & (u[:, i] * odds * total < left[each, x])
        if draft is None:
            rest = torch.where(token == x[:, None], 0.0, left)
        else:
            rest = (left / total[:, None] - draft[each, here].double()).clamp(min=0.0)
        mass = rest.sum(-1)
        turn = child & ~take & (mass > 0)
        left = torch.where(turn[:, None], rest, left)
        total = torch.where(turn, mass, total)
        here = torch.where(take, i, here)
        left = torch.where(take[:, None], target[:, i].double(), left)
        total = torch.where(take, 1.0, total)
        kept[:, i] = take
    run_sum = left.cumsum(-1)
    past = run_sum > u[:, :1] * run_sum[:, -1:]
    following = torch.where(past, token, c["vocab"]).amin(-1)
    last = torch.where(left > 0, token, -1).amax(-1)
    count = kept.sum(-1)
    at = torch.arange(nodes, device="cuda")
    order = torch.where(kept, at, nodes).sort(-1).values
    return {"path": torch.where(at < count[:, None], order, -1).int(), "count": count.int(),
            "next": torch.minimum(following, last).int()}


def _plain_keep(s):
    c = s["case"]
    slots, nodes = c["slots"], c["nodes"]
    base = s["pos"][:, :1].long()
    at = torch.arange(nodes, device="cuda")
    to = base + at
    # rows behind the path stay: they are written with what they hold
    source = base + torch.where(at < s["count"][:, None], s["path"].long(), at)
    each = torch.arange(slots, device="cuda")[:, None]
    kv = s["kv"]
    if c["dtype"] == "f32":
        kv[:, :, each, to] = kv[:, :, each, source]
    else:
        rows = kv.permute(2, 4, 0, 1, 3, 5)    # [slots][rows] first
        rows[each, to] = rows[each, source]
    return kv


def work(case):
    """Bytes: every visible cache row once, the query and output rows; one target row (and draft row) of each slot, which
    is what the walk cannot end without; the moved rows in and out. Operations: 2 * 2 * dim for every visible (query
    head, row) pair; one subtraction, comparison and sum for every probability."""
    shapes, slots, nodes = _shapes(case), case["slots"], case["nodes"]
    if case["op"] == "tree":
        width = case["heads"] * case["dim"]
        rows = sum(base + live for base, live, _ in shapes)
        pairs = sum(live * base + sum(_depth(parents, i) for i in range(live)) for base, live, parents in shapes)
        return {"bytes": 2 * rows * case["kv"] * _row_bytes(case) + sum(2 * live * width * 4 for _, live, _ in shapes),
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    if case["op"] == "verify":
        read = slots * case["vocab"] * 4 * (2 if case["draft"] else 1)
        return {"bytes": read + slots * nodes * 20, "flops": 3 * slots * case["vocab"]}
    moved = sum(sum(1 for i, node in enumerate(p) if i != node) for p in _paths(case))
    return {"bytes": 2 * LAYERS * 2 * case["kv"] * _row_bytes(case) * moved + slots * (nodes + 3) * 4, "flops": 0}


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "verify": _exact_verify, "keep": _exact_keep}[case["op"]](s)


def _exact_tree(s):
    c = s["case"]
    kv, dim, group = c["kv"], c["dim"], c["heads"] // c["kv"]
    out = s["out"].double()
    for slot, (base, live, parents) in enumerate(_shapes(c)):
        end = base + live
        sees = np.zeros((live, end), dtype=bool)
        sees[:, :base] = True
        for i in range(live):
            j = i
            while j >= 0:
                sees[i, base + j] = True
                j = parents[j]
        hidden = torch.from_numpy(~sees).cuda().repeat_interleave(group, 0)
        for h in range(kv):
            k, v = (_exact_rows(s["kv"][0, which, slot], c, h, end) for which in range(2))
            q = s["q"][slot, :live].double().view(live, c["heads"], dim)[:, h * group:(h + 1) * group].reshape(-1, dim)
            score = (q @ k.T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
            y = torch.softmax(score, -1) @ v
            out[slot, :live, h * group * dim:(h + 1) * group * dim] = y.view(live, group * dim)
    return out


def _exact_rows(cache, c, h, end):
    """The first `end` rows of KV head h as 64-bit values."""
    dim = c["dim"]
    if c["dtype"] == "f32":
        return cache[:end, h * dim:(h + 1) * dim].double()
    raw = cache[h, :end].reshape(-1, BLOCK_BYTES[c["dtype"]])
    scale = raw[:, :2].contiguous().view(torch.float16).double()
    if c["dtype"] == "q8":
        code = raw[:, 2:].contiguous().view(torch.int8).double()
    else:
        low, high = raw[:, 2:] % 16, raw[:, 2:] // 16
        code = torch.cat([low, high], 1).double() - 8
    return (scale * code).view(end, dim)


def _exact_verify(s):
    """One slot after the other, node after node, as the rule is written."""
    c = s["case"]
    nodes = c["nodes"]
    path = torch.full((c["slots"], nodes), -1, dtype=torch.int32)
    count, following = torch.zeros(c["slots"], dtype=torch.int32), torch.zeros(c["slots"], dtype=torch.int32)
    tokens, uniform = s["tokens"].tolist(), s["uniform"].double().tolist()
    for slot, (_, live, parents) in enumerate(_shapes(c)):
        here, kept = 0, [0]
        while True:
            p = s["target"][slot, here].double()
            found = -1
            for child in [i for i in range(here + 1, live) if parents[i] == here]:
                x = tokens[slot][child]
                if c["draft"]:
                    q = s["draft"][slot, here].double()
                else:
                    q = torch.zeros_like(p)
                    q[x] = 1.0
                if uniform[slot][child] * float(q[x]) < float(p[x]):
                    found = child
                    break
                rest = torch.relu(p - q)
                if float(rest.sum()) > 0:
                    p = rest / rest.sum()
            if found < 0:
                break
            here = found
            kept.append(here)
        run_sum = torch.cumsum(p, 0)
        past = torch.nonzero(run_sum > uniform[slot][0] * float(run_sum[-1]))
        following[slot] = int(past[0]) if len(past) else int(torch.nonzero(p > 0)[-1])
        path[slot, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
        count[slot] = len(kept)
    return {"path": path, "count": count, "next": following}


def _exact_keep(s):
    c = s["case"]
    paths = s["path"].tolist()
    for slot, (base, _, _) in enumerate(_shapes(c)):
        for i, node in enumerate(paths[slot][:int(s["count"][slot])]):
            # (a path's nodes ascend: a row is read before it is written)
            if c["dtype"] == "f32":
                s["kv"][:, :, slot, base + i] = s["kv"][:, :, slot, base + node]
            else:
                s["kv"][:, :, slot, :, base + i] = s["kv"][:, :, slot, :, base + node]
    return s["kv"]
