"""The work by which the operators for requests that share their beginning are measured: attention of a decode batch whose rows share long
prefixes (read once for all of them), and the copies of cache pages and of per-request states by which a request is forked and a cache compacted.

``own`` False: the definition in elementary torch operations.  ``own`` True: the calls of ``delta_b200.kernels.ops``.
"""
import math
import random

import torch

own = False
DEVICE = "cuda:0"
F64 = torch.float64
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ the cases
# Attention: ``groups`` "rows x prefix tokens" of each group of requests that share their first tokens, ``loose`` rows that share nothing,
# ``low`` and ``high`` the range of the tokens that a row holds of its own.  ``scattered``: pages in any order, as a long served pool has
# them; else in runs, as a fresh pool hands them out.

def listed():
    return [
        # two samples of a short prompt, a Yi-6B layer: the smallest call, where latency counts
        dict(name="attention_pair", kind="attention", heads=32, kv_heads=4, head_dim=128, page=16, dtype="bf16", groups="2x256", loose=0,
             low=1, high=40, scattered=False),
        # eight samples of one prompt at the benchmark's batch and context
        dict(name="attention_samples_8", kind="attention", heads=32, kv_heads=4, head_dim=128, page=16, dtype="bf16", groups="8x4096", loose=0,
             low=1, high=512, scattered=False),
        # 64 samples of a 2,048-token prompt with up to 512 generated tokens each: the benchmark's largest batch
        dict(name="attention_samples_64", kind="attention", heads=32, kv_heads=4, head_dim=128, page=16, dtype="bf16", groups="64x2048", loose=0,
             low=1, high=512, scattered=False),
        # a Yi-34B layer (seven query heads to a key-value head): three system prompts of odd lengths, rows that share nothing, pages all over the pool
        dict(name="attention_mixed", kind="attention", heads=56, kv_heads=8, head_dim=128, page=16, dtype="bf16", groups="17x1333,9x4001,5x100",
             loose=3, low=1, high=700, scattered=True),
        # many samples of the benchmark's long prompt: the largest call, bound by the tensor cores
        dict(name="attention_long", kind="attention", heads=32, kv_heads=4, head_dim=128, page=16, dtype="bf16", groups="48x30000", loose=0,
             low=200, high=1000, scattered=False),
        # heads of 64 and small pages
        dict(name="attention_heads_64", kind="attention", heads=16, kv_heads=2, head_dim=64, page=8, dtype="bf16", groups="16x3000", loose=1,
             low=1, high=300, scattered=False),
        # the 32-bit path
        dict(name="attention_f32", kind="attention", heads=32, kv_heads=4, head_dim=128, page=16, dtype="f32", groups="8x2048", loose=0,
             low=1, high=256, scattered=False),
        # one request of a Yi-6B model forked once: the seven tokens of its last page that are held, in 32 layers
        dict(name="pages_fork_1", kind="pages", layers=32, outer=8, page=16, width=128, pool=600, copies=1, sources=1, part=7),
        # the same for 63 more samples of it
        dict(name="pages_fork_63", kind="pages", layers=32, outer=8, page=16, width=128, pool=600, copies=63, sources=1, part=13),
        # a cache compacted: whole pages of 16 layers into the holes that finished requests left
        dict(name="pages_compact", kind="pages", layers=16, outer=8, page=16, width=128, pool=2500, copies=1100, sources=1100, part=0),
        # the states of a fork in a design with recurrent layers: matrix memories, their normalisers, short convolutions, a count
        dict(name="slots_fork_1", kind="slots", layers=6, slots=16, shapes="16x128x128,16x128,3x1027,1", copies=1),
        # fifteen forks at once
        dict(name="slots_fork_15", kind="slots", layers=6, slots=16, shapes="16x128x128,16x128,3x1027,1", copies=15),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "pages", "slots"])
    if kind == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 3, 4, 7, 8, 16])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        head_dim = rng.choice([64, 128])
        groups, keys = [], 0
        for _ in range(rng.randint(1, 4)):
            rows, prefix = _spread(rng, 2, 48), _spread(rng, 20, 20000)
            if (keys + rows * prefix) * heads * head_dim <= 2.5e9:
                groups.append(f"{rows}x{prefix}")
                keys += rows * prefix
        low = rng.randint(1, 100)
        return dict(kind="attention", heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=rng.choice([8, 16, 32]), dtype=dtype,
                    groups=",".join(groups) or "3x333", loose=rng.randint(0, 6), low=low, high=low + _spread(rng, 1, 900),
                    scattered=rng.random() < 0.5)
    if kind == "pages":
        page, pool = rng.choice([8, 16, 32]), _spread(rng, 60, 1200)
        outer, width, copies = rng.choice([1, 2, 8, 16]), rng.choice([36, 64, 128, 320]), _spread(rng, 1, pool // 2 - 1)
        layers = max(1, min(rng.randint(1, 32), int(1.1e9 / (pool * outer * page * width * 2))))
        return dict(kind="pages", layers=layers, outer=outer, page=page, width=width, pool=pool, copies=copies, sources=rng.choice([1, copies]),
                    part=rng.choice([0, rng.randint(1, page)]))
    slots = rng.randint(2, 64)
    return dict(kind="slots", layers=rng.randint(1, 8), slots=slots, shapes=f"{rng.randint(1, 16)}x64x{rng.choice([64, 128])},{rng.randint(1, 5)}x{rng.randint(1, 2000)},1",
                copies=rng.randint(1, slots - 1))


def _groups(case):
    return [tuple(int(v) for v in g.split("x")) for g in case["groups"].split(",")]


def _lengths(case):
    """The keys of every row, groups first, and the shared tokens (whole pages) of every group: by the case alone."""
    groups = [(rows, prefix // case["page"] * case["page"]) for rows, prefix in _groups(case)]
    shared = [p for rows, p in groups for _ in range(rows)] + [0] * case["loose"]
    span = case["high"] - case["low"]
    own_keys = [case["low"] + int(span * ((i * 0.6180339887498949 + 0.37) % 1.0)) for i in range(len(shared))]
    return [p + n for p, n in zip(shared, own_keys)], groups


def work(case):
    if case["kind"] == "attention":
        keys, groups = _lengths(case)
        size = 4 if case["dtype"] == "f32" else 2
        read = sum(keys) - sum((rows - 1) * p for rows, p in groups)       # every shared key once
        row = case["heads"] * case["head_dim"]
        return {"bytes": size * (read * 2 * case["kv_heads"] * case["head_dim"] + 2 * len(keys) * row), "flops": 4 * row * sum(keys)}
    if case["kind"] == "pages":
        item = case["layers"] * case["outer"] * (case["part"] or case["page"]) * case["width"] * 2
        return {"bytes": item * (case["copies"] + case["sources"]), "flops": 0}
    item = case["layers"] * sum(4 * math.prod(int(v) for v in s.split("x")) for s in case["shapes"].split(","))
    return {"bytes": item * (case["copies"] + 1), "flops": 0}


# ------------------------------------------------------------------ what a program has in hand

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    order = random.Random(seed)
    if case["kind"] == "attention":
        return _prepare_attention(case, gen, order)
    if case["kind"] == "pages":
        pages = torch.randn((case["layers"], case["pool"], case["outer"], case["page"], case["width"]), dtype=torch.bfloat16, device=DEVICE, generator=gen)
        ids = order.sample(range(case["pool"]), case["sources"] + case["copies"])
        src, dst = ids[:case["sources"]], ids[case["sources"]:]
        src = src * (case["copies"] // case["sources"])
        tokens = [case["part"]] * case["copies"] if case["part"] else None
        return dict(kind="pages", pages=pages, src=src, dst=dst, tokens=tokens)
    states = [torch.randn((case["slots"], *(int(v) for v in s.split("x"))), dtype=torch.float32, device=DEVICE, generator=gen)
              for _ in range(case["layers"]) for s in case["shapes"].split(",")]
    slots = order.sample(range(case["slots"]), case["copies"] + 1)
    return dict(kind="slots", states=states, src=slots[:1] * case["copies"], dst=slots[1:])


def _prepare_attention(case, gen, order):
    ps, kv_heads, hd, dtype = case["page"], case["kv_heads"], case["head_dim"], TYPES[case["dtype"]]
    keys, groups = _lengths(case)
    held = [-(-n // ps) for n in keys]
    shared = [p // ps for rows, p in groups for _ in range(rows)] + [0] * case["loose"]
    total = sum(p // ps for _, p in groups) + sum(n - s for n, s in zip(held, shared))
    ids = list(range(total + 5))
    if case["scattered"]:
        order.shuffle(ids)
    next_id = iter(ids).__next__
    table = torch.full((len(keys), max(held) + 3), -1, dtype=torch.int32)
    row = 0
    for rows, prefix in groups + [(1, 0)] * case["loose"]:
        first = [next_id() for _ in range(prefix // ps)]
        for _ in range(rows):
            mine = first + [next_id() for _ in range(held[row] - len(first))]
            table[row, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            row += 1
    # the rows of a batch stand in the order of their admission, not group by group
    place = list(range(len(keys)))
    order.shuffle(place)
    at = torch.tensor(place)
    sorted_rows = torch.argsort(at).to(torch.int32)         # row of the batch that holds request i
    starts = [0]
    for rows, _ in groups:
        starts.append(starts[-1] + rows)
    ints = dict(dtype=torch.int32, device=DEVICE)
    return dict(
        kind="attention", scale=1.0 / math.sqrt(hd),
        q=1.5 * torch.randn((len(keys), case["heads"], hd), dtype=torch.float32, device=DEVICE, generator=gen).to(dtype),
        kv=torch.randn((len(ids), 2, kv_heads, ps, hd), dtype=dtype, device=DEVICE, generator=gen),
        block_table=table[at].to(DEVICE), kv_len=torch.tensor(keys, dtype=torch.int32)[at].to(DEVICE),
        members=sorted_rows[:starts[-1]].to(DEVICE), group_start=torch.tensor(starts, **ints),
        group_prefix=torch.tensor([p for _, p in groups], **ints))


# ------------------------------------------------------------------ one pass

def run(state):
    if own:
        return _own(state)
    if state["kind"] == "attention":
        return _plain_attention(state)
    if state["kind"] == "pages":
        return _plain_pages(state)
    src, dst = torch.tensor(state["src"], device=DEVICE), torch.tensor(state["dst"], device=DEVICE)
    for s in state["states"]:
        s[dst] = s[src]
    return state["states"]


def _own(state):
    from delta_b200.kernels import ops
    if state["kind"] == "attention":
        out = torch.empty_like(state["q"])
        ops.attention_shared_prefix(state["q"], out, state["kv"], state["block_table"], state["kv_len"], state["members"],
                                    state["group_start"], state["group_prefix"], scale=state["scale"])
        return out
    if state["kind"] == "pages":
        ops.copy_pages(state["pages"], state["src"], state["dst"], tokens=state["tokens"], token_axis=1)
        return state["pages"]
    ops.copy_slots(state["states"], state["src"], state["dst"])
    return state["states"]


def _plain_attention(s):
    q, kv, table, kv_len = s["q"], s["kv"], s["block_table"].long().clamp_min(0), s["kv_len"].long()
    rows, heads, hd = q.shape
    kv_heads, ps = kv.shape[2], kv.shape[3]
    width = table.shape[1] * ps

    def gather(which):      # [rows, kv heads, keys, head size]
        return kv[table, which].permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, width, hd).float()

    scores = torch.matmul(q.view(rows, kv_heads, heads // kv_heads, hd).float(), gather(0).transpose(2, 3)) * s["scale"]
    seen = torch.arange(width, device=q.device)[None, :] < kv_len[:, None]
    scores = torch.where(seen[:, None, None, :], scores, torch.full((), -math.inf, device=q.device))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(p, gather(1)) / p.sum(-1, keepdim=True)
    return out.reshape(rows, heads, hd).to(q.dtype)


def _plain_pages(s):
    pages = s["pages"]
    src, dst = torch.tensor(s["src"], device=DEVICE), torch.tensor(s["dst"], device=DEVICE)
    if s["tokens"] is None:
        pages[:, dst] = pages[:, src]
        return pages
    tokens = torch.tensor(s["tokens"], device=DEVICE)
    taken = torch.arange(pages.shape[3], device=DEVICE)[None, :] < tokens[:, None]
    pages[:, dst] = torch.where(taken[None, :, None, :, None], pages[:, src], pages[:, dst])
    return pages


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "pages":
        before, after = s["pages"], s["pages"].to(F64)
        for a, b in zip(s["src"], s["dst"]):
            after[:, b, :, :case["part"] or case["page"]] = before[:, a, :, :case["part"] or case["page"]].to(F64)
        return after
    if case["kind"] == "slots":
        after = [x.to(F64) for x in s["states"]]
        for x, y in zip(s["states"], after):
            for a, b in zip(s["src"], s["dst"]):
                y[b] = x[a].to(F64)
        return after
    q, kv, out = s["q"], s["kv"], []
    lengths, table = s["kv_len"].tolist(), s["block_table"].tolist()
    heads, hd, ps = q.shape[1], q.shape[2], kv.shape[3]
    per = heads // kv.shape[2]
    for b, n in enumerate(lengths):
        cached = kv[torch.tensor(table[b][:-(-n // ps)], device=q.device)].to(F64)          # [pages, 2, kv heads, page, head size]
        cached = cached.movedim(0, 2).reshape(2, kv.shape[2], -1, hd)[:, :, :n]
        logits = torch.einsum("ghd,gkd->ghk", q[b].to(F64).view(-1, per, hd), cached[0]) * s["scale"]
        out.append(torch.einsum("ghk,gkd->ghd", torch.softmax(logits, -1), cached[1]).reshape(heads, hd))
    return torch.stack(out)
