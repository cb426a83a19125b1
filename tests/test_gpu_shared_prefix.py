"""Attention over shared prefixes against the softmax written out in float64.

Queries, keys and values are small whole numbers and the scale is a power of two, so every score is exact in both types.  A few keys (the
first and last of the prefix and of the row, those at page and tile borders, some at random) score about 8 above the rest and share nearly
the whole weight: one that is missed or wrongly seen moves the output by its share, about 1 / 30 of a value, while values are -1 or 1.

What rounding can do, to a value of at most 1: the exponent is off by 2^-24 of itself (two products, at most 20 in size) and the
exponential by 2 units of 2^-23, together below 2^-18; sums of n weights by n 2^-24, in the numerator and in the denominator; bfloat16 rounds the
weights (2^-8) and the result (2^-8).  A merge rounds a few times more (below 2^-20)."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def tolerance(dtype, keys):
    return 2.0 ** -17 + 2 * keys * 2.0 ** -24 + (2 * 2.0 ** -8 if dtype == "bfloat16" else 0.0)


def make(dtype, H, KV, hd, ps, groups, loose, own, seed=0, scattered=False, wide=2, q_gap=0):
    """groups: [(rows, prefix)], own: keys of each row alone (groups' rows first, then the loose ones)."""
    rnd, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    shared = [p // ps * ps for n, p in groups for _ in range(n)] + [0] * loose
    lens = [a + b for a, b in zip(shared, own)]
    rows = len(lens)
    held = [-(-n // ps) for n in lens]
    n_pages = sum(p // ps for _, p in groups) + sum(h - s // ps for h, s in zip(held, shared)) + 3
    ids = list(range(n_pages))
    if scattered:
        rnd.shuffle(ids)
    take = iter(ids).__next__
    table = torch.full((rows, max(held + [0]) + wide), -1, dtype=torch.int32)
    row = 0
    for n, p in groups + [(1, 0)] * loose:
        first = [take() for _ in range(p // ps)]
        for _ in range(n):
            mine = first + [take() for _ in range(held[row] - len(first))]
            table[row, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            row += 1
    u = torch.randint(0, 2, (KV, hd), generator=gen) * 2 - 1
    q = u.repeat_interleave(H // KV, 0)[None] + torch.randint(0, 12, (rows, H, hd), generator=gen).eq(0).int() * (torch.randint(0, 2, (rows, H, hd), generator=gen) * 2 - 1)
    kv = torch.randint(0, 2, (n_pages, 2, KV, ps, hd), generator=gen) * 2 - 1
    for r in range(rows):
        special = {0, shared[r] - 1, shared[r], lens[r] - 1} | {rnd.randrange(lens[r]) for _ in range(4) if lens[r]}
        special |= {x * rnd.randrange(1 + lens[r] // x) - rnd.randrange(2) for x in (ps, 64, 128) if lens[r]}
        for k in special:
            if 0 <= k < lens[r]:
                kv[table[r, k // ps], 0, :, k % ps] = u
    order = list(range(rows))
    rnd.shuffle(order)                      # where request i stands in the batch: order.index(i)
    at = torch.tensor(order, dtype=torch.long)
    back = torch.argsort(at)
    starts = [0]
    for n, _ in groups:
        starts.append(starts[-1] + n)
    i32 = dict(dtype=torch.int32, device="cuda")
    qd = torch.zeros((rows, H * hd + q_gap), dtype=DT[dtype], device="cuda")
    qd[:, :H * hd] = q[at].reshape(rows, -1).to("cuda", DT[dtype])
    return dict(q=qd[:, :H * hd].unflatten(1, (H, hd)) if q_gap else qd.view(rows, H, hd), kv=kv.to("cuda", DT[dtype]), block_table=table[at].contiguous().cuda(),
                kv_len=torch.tensor(lens, dtype=torch.int32)[at].cuda(), members=back[:starts[-1]].to(torch.int32).cuda(),
                group_start=torch.tensor(starts, **i32), group_prefix=torch.tensor([p for _, p in groups], **i32), scale=8.0 / hd if hd >= 8 else 1.0)


def reference(c):
    out = []
    q, kv, table = c["q"].double().cpu(), c["kv"].double().cpu(), c["block_table"].cpu()
    H, hd, KV, ps = q.shape[1], q.shape[2], kv.shape[2], kv.shape[3]
    for r, n in enumerate(c["kv_len"].tolist()):
        x = kv[table[r, :-(-n // ps)].long()].permute(1, 2, 0, 3, 4).reshape(2, KV, -1, hd)[:, :, :n]
        s = torch.einsum("kgd,ksd->kgs", q[r].view(KV, H // KV, hd), x[0]) * c["scale"]
        out.append(torch.einsum("kgs,ksd->kgd", torch.softmax(s, -1), x[1]).reshape(H, hd) if n else torch.zeros(H, hd, dtype=torch.float64))
    return torch.stack(out)


def call(c, out=None, **more):
    from delta_b200.kernels import ops
    out = torch.full_like(c["q"], 7.0) if out is None else out
    args = {k: v for k, v in c.items() if k not in ("q",)}
    err = ops.new_error_record("cuda")
    ops.attention_shared_prefix(c["q"], out, err=err, **{**args, **more})
    torch.cuda.synchronize()
    ops.raise_if_error(err)
    return out


def check(dtype, c):
    got, want = call(c), reference(c)
    assert torch.isfinite(got.float()).all()
    off = (got.double().cpu() - want).abs().amax().item()
    assert off <= tolerance(dtype, int(c["kv_len"].max())), off


SHAPES = [  # H, KV, hd, ps
    (32, 4, 128, 16), (56, 8, 128, 16), (16, 2, 64, 8), (4, 2, 16, 16), (4, 1, 32, 8), (6, 6, 128, 32), (32, 2, 128, 64), (3, 1, 64, 128)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("scattered", [False, True], ids=["runs", "scattered"])
def test_one_group(dtype, shape, scattered):
    check(dtype, make(dtype, *shape, [(5, 700)], 0, [1, 40, 128, 129, 300], seed=1, scattered=scattered))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(2, 1, 132, 16), (6, 2, 200, 8), (4, 4, 256, 16), (34, 2, 256, 32), (32, 1, 128, 16), (24, 1, 64, 16), (40, 2, 4, 16), (62, 2, 128, 8),
                                   (8, 2, 128, 10), (8, 2, 64, 1), (8, 2, 128, 48), (4, 2, 128, 256), (16, 2, 64, 100)], ids=lambda s: "x".join(map(str, s)))
def test_wide_heads_many_heads_odd_pages(dtype, shape):
    """Heads of 129 to 256, more than 16 query heads to a key-value head, pages whose size is no power of two or larger than a tile."""
    check(dtype, make(dtype, *shape, [(5, 700), (9, 333)], 2, [1, 40, 128, 129, 300, 2, 3, 64, 65, 31, 32, 33, 7, 100, 17, 530], seed=35, scattered=True))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", SHAPES[:5], ids=lambda s: "x".join(map(str, s)))
def test_groups_and_loose_rows(dtype, shape):
    groups = [(3, 1000), (1, 333), (20, 129), (2, 5)]
    own = [random.Random(5).choice([1, 2, 17, 127, 128, 129, 255, 400]) for _ in range(26 + 4)]
    check(dtype, make(dtype, *shape, groups, 4, own, seed=2, scattered=True))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("case", [([(2, 128)], 0, [0, 1]), ([(2, 128)], 0, [0, 0]), ([], 3, [0, 1, 200]), ([(1, 16)], 0, [1]), ([(2, 0)], 1, [1, 0, 0]),
                                  ([(40, 16)], 0, [1] * 40), ([(2, 15)], 0, [3, 4])], ids=str)
def test_small_and_empty(dtype, case):
    """Rows with no key of their own, rows with no key at all (zeros), prefixes below a page, one row in a group."""
    check(dtype, make(dtype, 32, 4, 128, 16, *case, seed=3))


@pytest.mark.parametrize("dtype", list(DT))
def test_long_prefix_and_many_ranges(dtype):
    """A line of tiles that blocks walk in several rounds, and a prefix that is cut over most of them."""
    check(dtype, make(dtype, 8, 8, 64, 16, [(3, 60000)], 2, [5, 700, 1, 9000, 30000], seed=4))


@pytest.mark.parametrize("dtype", list(DT))
def test_rows_that_lie_apart(dtype):
    c = make(dtype, 8, 2, 64, 16, [(4, 300)], 1, [3, 50, 1, 20, 260], seed=5, q_gap=2 * 2 * 64)
    assert not c["q"].is_contiguous()
    wide = torch.full((5, 3, 8, 64), 5.0, dtype=DT[dtype], device="cuda")
    got = call(c, out=wide[:, 1])
    assert (got.double().cpu() - reference(c)).abs().amax() <= tolerance(dtype, 600)
    assert (wide[:, 0] == 5).all() and (wide[:, 2] == 5).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_no_row_reads_does_not_matter(dtype, bad):
    """Entries behind a row's last key, and whole pages of others, hold what an earlier request left."""
    c = make(dtype, 32, 4, 128, 16, [(5, 530)], 1, [1, 40, 128, 129, 300, 77], seed=6)
    want = reference(c)
    table, ps = c["block_table"].cpu(), 16
    used = torch.zeros(c["kv"].shape[0], ps, dtype=torch.bool)
    for r, n in enumerate(c["kv_len"].tolist()):
        for k in range(n):
            used[table[r, k // ps], k % ps] = True
    hole = (~used).cuda()[:, None, None, :, None].expand_as(c["kv"])
    c["kv"][hole] = bad
    assert (call(c).double().cpu() - want).abs().amax() <= tolerance(dtype, 900)


@pytest.mark.parametrize("dtype", list(DT))
def test_same_bits_again_and_captured(dtype):
    """The sums' order is fixed; a captured call reads its tables anew at every replay."""
    a = make(dtype, 32, 4, 128, 16, [(5, 700), (3, 64)], 2, [1, 40, 128, 129, 300, 5, 6, 7, 90, 91], seed=7)
    b = make(dtype, 32, 4, 128, 16, [(6, 640), (2, 128)], 2, [1, 4, 12, 200, 300, 50, 60, 7, 0, 19], seed=8, scattered=True)
    b["block_table"] = torch.nn.functional.pad(b["block_table"], (0, max(0, a["block_table"].shape[1] - b["block_table"].shape[1])), value=-1)
    a["block_table"] = torch.nn.functional.pad(a["block_table"], (0, max(0, b["block_table"].shape[1] - a["block_table"].shape[1])), value=-1)
    n = max(a["kv"].shape[0], b["kv"].shape[0])
    for c in (a, b):
        c["kv"] = torch.cat([c["kv"], c["kv"][:1].expand(n - c["kv"].shape[0], -1, -1, -1, -1)]) if c["kv"].shape[0] < n else c["kv"]
        c["block_table"] = c["block_table"].contiguous()
    first = {id(c): call(c).clone() for c in (a, b)}
    for c in (a, b):
        assert torch.equal(call(c), first[id(c)])
    held = {k: v.clone() for k, v in a.items() if isinstance(v, torch.Tensor)}
    out = torch.empty_like(a["q"])
    from delta_b200.kernels import ops
    run = lambda: ops.attention_shared_prefix(out=out, scale=a["scale"], **held)      # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for c in (b, a, b):
        for k, v in held.items():
            v.copy_(c[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first[id(c)])


@pytest.mark.parametrize("dtype", list(DT))
def test_one_work_buffer_for_many_calls(dtype):
    """Whatever an earlier call (or nobody) left in the working memory, a call takes its own list of pieces: eager ones, two recorded ones in turn."""
    from delta_b200.kernels import ops
    cases = [make(dtype, 32, 4, 128, 16, [(9, 1500), (4, 2000)], 1, [31 * i % 211 + 1 for i in range(14)], seed=30),
             make(dtype, 32, 4, 128, 16, [(2, 4000)], 12, [17 * i % 907 + 1 for i in range(14)], seed=31, scattered=True),
             make(dtype, 32, 4, 128, 16, [], 14, [61 * i % 1501 for i in range(14)], seed=32)]
    want = [call(c).clone() for c in cases]
    need = max(ops.attention_shared_prefix_floats(14, c["group_prefix"].numel(), c["members"].numel(), 32, 4, 128, 16, c["block_table"].shape[1], c["kv"].shape[0], c["kv"].dtype)
               for c in cases)
    work = torch.empty(need, device="cuda")
    outs, graphs = [torch.empty_like(c["q"]) for c in cases], []

    def run(i):
        ops.attention_shared_prefix(out=outs[i], work=work, **cases[i])
    for junk in (0, -1, 0x7F800001):
        work.view(torch.int32).fill_(junk)
        for i in (0, 1, 2, 1, 0, 0):
            run(i)
            assert torch.equal(outs[i], want[i])
    for i in range(3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(i)
        graphs.append(g)
    rnd = random.Random(33)
    for n in range(60):
        i = rnd.randrange(3)
        outs[i].fill_(3.0)
        if n % 4 == 0:
            work.view(torch.int32).random_()
        graphs[i].replay()
        if n % 3 == 0:
            run((i + 1) % 3)
        assert torch.equal(outs[i], want[i])


@pytest.mark.parametrize("dtype", list(DT))
def test_two_streams_at_once(dtype):
    cases = [make(dtype, 32, 4, 128, 16, [(8, 1500)], 1, [3 * i + 1 for i in range(9)], seed=s) for s in (9, 10)]
    want = [call(c).clone() for c in cases]
    from delta_b200.kernels import ops
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [torch.empty_like(c["q"]) for c in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, o, st in zip(cases, outs, streams):
            with torch.cuda.stream(st):
                ops.attention_shared_prefix(out=o, **c)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dtype", list(DT))
def test_wrong_tables_are_recorded(dtype):
    """Every index that comes from the device is checked before it is used: a wrong one is an error on the host, not a fault."""
    from delta_b200.kernels.lib import KernelError

    def broken(key, at, value):
        c = make(dtype, 32, 4, 128, 16, [(4, 320), (2, 64)], 1, [5, 6, 7, 8, 9, 150, 11], seed=11)
        c[key] = c[key].clone()
        c[key][at] = value
        return c
    row = make(dtype, 32, 4, 128, 16, [(4, 320), (2, 64)], 1, [5, 6, 7, 8, 9, 150, 11], seed=11)["members"][0].item()
    for c in (broken("members", 1, row), broken("members", 1, 99), broken("members", 2, -1), broken("group_start", 1, 1 << 20), broken("group_start", 0, -4),
              broken("group_prefix", 0, 1 << 29), broken("group_prefix", 1, -16), broken("kv_len", row, 100), broken("kv_len", row, 1 << 30)):
        with pytest.raises(KernelError, match="share a prefix"):
            call(c)
    for page in (-1, -7, 1 << 20):
        with pytest.raises(KernelError, match="page id out of range"):
            call(broken("block_table", (slice(None), 3), page))
    check(dtype, make(dtype, 32, 4, 128, 16, [(4, 320), (2, 64)], 1, [5, 6, 7, 8, 9, 150, 11], seed=11))


def right_but_for(c, wrong=()):
    """The call records an error and every row but ``wrong`` is what its keys give; twice the same bits."""
    from delta_b200.kernels import ops
    from delta_b200.kernels.lib import KernelError
    with pytest.raises(KernelError, match="share a prefix|page id out of range"):      # (which comes first: a wrong first member's table is too short as well)
        call(c)
    outs = []
    for _ in range(2):
        outs.append(ops.attention_shared_prefix(out=torch.full_like(c["q"], 7.0), **c))
    torch.cuda.synchronize()
    keys = c["block_table"].shape[1] * c["kv"].shape[3]
    ok = torch.tensor([r not in wrong and 0 <= n <= keys for r, n in enumerate(c["kv_len"].tolist())])
    want = reference(dict(c, kv_len=torch.where(ok, c["kv_len"].cpu(), 0)))
    off = (outs[0].double().cpu() - want)[ok].abs().amax().item()
    assert off <= tolerance(str(c["q"].dtype)[6:], int(c["kv_len"].cpu()[ok].max())), off
    assert torch.equal(outs[0][ok.cuda()], outs[1][ok.cuda()])         # (the others may be any bits)
    return outs[0]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(32, 4, 128, 16), (4, 2, 16, 16)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("again", [(0, 9), (5, 9), (8, 0), (11, 10)], ids=str)
def test_a_row_named_twice_spoils_no_other(dtype, shape, again):
    """Place ``again[1]`` of the members names the row of place ``again[0]`` too: another place of its group, or of a group with another prefix."""
    c = make(dtype, *shape, [(4, 1320), (4, 640), (4, 64)], 3, [random.Random(21).choice((1, 7, 40, 200)) for _ in range(15)], seed=21)
    c["members"] = c["members"].clone()
    row = int(c["members"][again[0]])
    c["members"][again[1]] = row
    # (a group reads its pages through its first member's table)
    right_but_for(c, c["members"][:4].tolist() if again[1] == 0 else ())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(32, 4, 128, 16), (4, 2, 16, 16)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("length", [0, 1, 100, 639, -5, 1 << 30])
def test_a_row_that_is_shorter_than_its_prefix_reads_its_keys_alone(dtype, shape, length):
    c = make(dtype, *shape, [(4, 1320), (4, 640)], 2, [1, 7, 40, 200, 3, 90, 1, 300, 5, 66], seed=22, scattered=True)
    row = int(c["members"][5])
    c["kv_len"] = c["kv_len"].clone()
    c["kv_len"][row] = length
    out = right_but_for(c)
    if length <= 0 or length > 5000:
        assert (out[row] == 0).all()


def test_refusals():
    from delta_b200.kernels import ops
    from delta_b200.kernels.lib import KernelError
    c = make("bfloat16", 8, 2, 64, 16, [(2, 64)], 0, [1, 2], seed=12)
    out = torch.empty_like(c["q"])

    def refused(match, out=out, **change):
        with pytest.raises(KernelError, match=match):
            ops.attention_shared_prefix(out=out, **{**c, **change})
    refused("do not fit", kv=c["kv"].float())
    refused("do not fit", kv_len=c["kv_len"][:1])
    refused("do not fit", group_start=c["group_start"][:1])
    refused("expected", out=out.float())
    refused("one behind the other", q=c["q"].transpose(1, 2).contiguous().transpose(1, 2))
    refused("dtype", members=c["members"].long())
    refused("is on 'cpu'", members=c["members"].cpu())
    refused("must be positive", scale=-1.0)
    refused("floats of working memory", work=torch.empty(8, device="cuda"))
    refused("16-byte", kv=torch.empty(c["kv"].numel() + 4, dtype=torch.bfloat16, device="cuda")[4:].view_as(c["kv"]))
    many = 1025
    refused("at most", out=torch.empty(many, 8, 64, dtype=torch.bfloat16, device="cuda"), q=torch.empty(many, 8, 64, dtype=torch.bfloat16, device="cuda"),
            kv_len=torch.zeros(many, dtype=torch.int32, device="cuda"), block_table=torch.zeros(many, 4, dtype=torch.int32, device="cuda"))
    empty = ops.attention_shared_prefix(c["q"][:0], out[:0], c["kv"], c["block_table"][:0], c["kv_len"][:0], c["members"][:0], c["group_start"][:1] * 0,
                                        c["group_prefix"][:0], scale=1.0)
    assert empty.numel() == 0


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("starts", [[0, 6, 0, 6], [6, 0, 6, 0], [2, 4, 3, 6], [0, 0, 7, 6], [0, -1, 3, 6]], ids=str)
def test_starts_out_of_order_leave_no_group(dtype, starts):
    """Groups that overlap would be more pieces than there is room for: none is taken, which is recorded, and every row reads its keys alone."""
    from delta_b200.kernels import ops
    from delta_b200.kernels.lib import KernelError
    c = make(dtype, 32, 4, 128, 16, [(6, 320), (0, 320), (0, 320)], 1, [5, 6, 7, 8, 9, 150, 11], seed=14)
    c["group_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    with pytest.raises(KernelError, match="share a prefix"):
        call(c)
    out = torch.full_like(c["q"], 7.0)
    ops.attention_shared_prefix(out=out, **c)
    off = (out.double().cpu() - reference(c)).abs().amax().item()
    assert off <= tolerance(dtype, int(c["kv_len"].max())), off


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("heads", [(32, 4, 128), (4, 2, 16)], ids=str)
def test_groups_over_the_same_pages(dtype, heads):
    """32 groups of the same pages are more tiles than the pool has pages for: the rows read alone, and nothing is wrong.  Two groups of them are taken."""
    for groups in (32, 2):
        c = make(dtype, *heads, 16, [(64, 4000)], 2, [random.Random(i).choice((1, 9, 16, 30)) for i in range(66)], seed=34)
        per = 64 // groups
        c["group_start"] = torch.arange(0, 65, per, dtype=torch.int32, device="cuda")
        c["group_prefix"] = torch.full((groups,), 4000, dtype=torch.int32, device="cuda")
        check(dtype, c)


@pytest.mark.parametrize("dtype", list(DT))
def test_groups_of_nobody(dtype):
    c = make(dtype, 8, 2, 64, 16, [], 3, [1, 20, 150], seed=15)
    c["group_start"], c["group_prefix"] = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (5, 4))
    check(dtype, c)


@pytest.mark.parametrize("dtype", list(DT))
def test_results_over_the_queries_are_refused(dtype):
    from delta_b200.kernels.lib import KernelError
    c = make(dtype, 8, 2, 64, 16, [(3, 64)], 1, [1, 20, 150, 9], seed=16)
    n = c["q"].shape[0]
    wide = torch.zeros(n + 1, 3 * 512, dtype=DT[dtype], device="cuda")
    side = lambda at, first=0: wide[first:first + n, at:at + 512].unflatten(1, (8, 64))      # noqa: E731
    side(512).copy_(c["q"])
    c["q"] = side(512)
    for out in (side(512), side(512, 1), side(256), side(1024 - 256), wide.view(-1)[512 + 1024:][:n * 1024].view(n, 1024)[:, :512].unflatten(1, (8, 64))):
        with pytest.raises(KernelError, match="overwrite"):
            call(c, out=out)
    want = reference(c)
    for out in (side(0), side(1024), side(1024, 1)):         # columns beside them are nobody's
        got = call(c, out=out)
        assert (got.double().cpu() - want).abs().amax().item() <= tolerance(dtype, int(c["kv_len"].max()))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("case", [(32, 4, 128, [(700, 4096), (300, 1504)], 24), (32, 16, 64, [(1000, 160)], 24), (8, 8, 64, [(2, 32)] * 500, 24)], ids=["ranges", "pieces", "groups"])
def test_most_rows(dtype, case):
    """As many rows as a call takes: blocks walk several ranges of groups and several lists of pieces."""
    H, KV, hd, groups, loose = case
    rnd = random.Random(17)
    rows = sum(n for n, _ in groups) + loose
    assert rows == 1024
    c = make(dtype, H, KV, hd, 16, groups, loose, [rnd.choice((0, 1, 15, 16, 17, 40, 70)) for _ in range(rows)], seed=17)
    got = call(c)
    some = torch.tensor(rnd.sample(range(rows), 40))
    part = dict(c, q=c["q"][some.cuda()], block_table=c["block_table"][some.cuda()], kv_len=c["kv_len"][some.cuda()])
    off = (got[some.cuda()].double().cpu() - reference(part)).abs().amax().item()
    assert off <= tolerance(dtype, int(c["kv_len"].max())), off
    assert torch.isfinite(got.float()).all()
    assert torch.equal(call(c), got)
