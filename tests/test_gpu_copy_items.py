"""Copies of pages and slots against the same copies of a clone: every bit, in place, as if all were read before any is written."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def copies(kind, n, rnd):
    ids = list(range(n))
    rnd.shuffle(ids)
    if kind == "apart":
        return ids[:n // 2], ids[n // 2:n // 2 * 2]
    if kind == "one to many":
        return [ids[0]] * (n - 1), ids[1:]
    if kind == "cycle":
        return ids, ids[1:] + ids[:1]
    if kind == "chain":
        return ids[:-1], ids[1:]
    if kind == "swaps":
        return ids[:n // 2 * 2], [ids[i ^ 1] for i in range(n // 2 * 2)]
    if kind == "nothing moves":
        return ids, ids
    dst = ids[:rnd.randint(1, n)]
    return [rnd.randrange(n) for _ in dst], dst        # anything: trees, cycles, items that stay


KINDS = ["apart", "one to many", "cycle", "chain", "swaps", "nothing moves", "any", "any 2", "any 3"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pages", [2, 9, 60, 400, 2000])
@pytest.mark.parametrize("layout", [(2, 4, 16, 128), (16, 36), (3, 5), (1,)], ids=str)
def test_pages(kind, pages, layout):
    from delta_b200.kernels import ops
    rnd = random.Random(repr((kind, pages)))
    dtype = {128: torch.bfloat16, 36: torch.bfloat16, 5: torch.float32, 1: torch.uint8}[layout[-1]]
    x = torch.randint(0, 200, (3, pages, *layout), device="cuda").to(dtype)
    want = x.clone()
    src, dst = copies(kind, pages, rnd)
    want[:, dst] = x[:, src]
    ops.copy_pages(x, src, dst)
    assert torch.equal(x, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout,axis", [((2, 4, 16, 128), 2), ((16, 36), 0), ((3, 8), 1)], ids=str)
def test_parts_of_pages(kind, layout, axis):
    """Only the first tokens of a page are copied; the others stay what they were."""
    from delta_b200.kernels import ops
    for pages in (7, 130):
        rnd = random.Random(repr((kind, pages, layout)))
        x = torch.randn(2, pages, *layout, device="cuda").to(torch.bfloat16)
        src, dst = copies(kind, pages, rnd)
        tokens = [rnd.randint(0, layout[axis]) for _ in src]
        want = x.clone()
        for a, b, n in zip(src, dst, tokens):
            want.select(1, b).narrow(axis + 1, 0, n).copy_(x.select(1, a).narrow(axis + 1, 0, n))
        ops.copy_pages(x, torch.tensor(src), torch.tensor(dst), tokens=tokens, token_axis=axis)
        assert torch.equal(x, want)


@pytest.mark.parametrize("kind", KINDS)
def test_slots(kind):
    from delta_b200.kernels import ops
    slots = 17
    gen = torch.Generator(device="cuda").manual_seed(0)
    shapes = [(4, 16, 16), (3, 1027), (), (7,), (0,), (2, 3)]
    types = [torch.float32, torch.float32, torch.int32, torch.uint8, torch.float32, torch.bfloat16]
    states = [torch.randint(0, 250, (slots, *s), device="cuda", generator=gen).to(t) for s, t in zip(shapes, types)]
    states += [torch.randn(slots, 33, device="cuda") for _ in range(40)]           # more tensors than one launch takes
    want = [s.clone() for s in states]
    src, dst = copies(kind, slots, random.Random(kind))
    for w, s in zip(want, states):
        w[dst] = s[src]
    ops.copy_slots(dict(enumerate(states)), src, dst)
    assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_far_pages():
    """Offsets beyond 32 bits."""
    from delta_b200.kernels import ops
    x = torch.empty(3, 70000, 2, 16, 1024, dtype=torch.bfloat16, device="cuda")       # 13.8 GB, a layer 4.6 GB
    for i, p in enumerate((1, 69998, 35000)):
        x[:, p] = torch.arange(3, device="cuda", dtype=torch.bfloat16)[:, None, None, None] * 8 + i
    ops.copy_pages(x, [1, 69998, 35000], [69998, 35000, 0])
    for p, i in ((1, 0), (69998, 0), (35000, 1), (0, 2)):
        assert all((x[layer, p] == layer * 8 + i).all() for layer in range(3))


def test_captured():
    from delta_b200.kernels import ops
    from delta_b200.kernels.lib import KernelError
    x = torch.randn(4, 30, 16, 64, device="cuda")
    want = x.clone()
    want[:, [1, 2, 3]] = x[:, [3, 1, 2]]
    graph = torch.cuda.CUDAGraph()
    keep = x.clone()
    ops.copy_pages(keep, [0], [1])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.copy_pages(x, [3, 1, 2], [1, 2, 3])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, want)
    big = torch.zeros(1, 4000, 16, device="cuda")
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(KernelError, match="captured"):
            ops.copy_pages(big, list(range(2000)), list(range(2000, 4000)))
        big.zero_()


def test_refusals():
    from delta_b200.kernels import ops
    from delta_b200.kernels.lib import KernelError
    x = torch.zeros(2, 8, 16, 4, device="cuda")
    for match, args in [("written twice", (x, [0, 1], [3, 3])), ("goes from", (x, [0], [8])), ("goes from", (x, [-1], [2])), ("2 sources, 1 targets", (x, [0, 1], [2])),
                        ("whole numbers", (x, [0.5], [1])), ("not contiguous", (x.transpose(0, 1), [0], [1])), ("which items", (x, torch.tensor([0]).cuda(), [1])),
                        ("expected", (x[0, 0], [0], [1]))]:
        with pytest.raises(KernelError, match=match):
            ops.copy_pages(*args)
    with pytest.raises(KernelError, match="token axis"):
        ops.copy_pages(x, [0], [1], tokens=[2])
    with pytest.raises(KernelError, match="asks for 17 tokens"):
        ops.copy_pages(x, [0], [1], tokens=[17], token_axis=0)
    with pytest.raises(KernelError, match="same number of slots"):
        ops.copy_slots([x, x[:1]], [0], [1])
    ops.copy_pages(x, [], [])
    ops.copy_slots([], [], [])


def test_slots_that_share_memory_are_refused():
    from delta_b200.kernels import ops
    from delta_b200.kernels.lib import KernelError
    x = torch.zeros(8, 4, device="cuda")
    keep = x.clone()
    for states in ([x, x], {0: x, 1: torch.zeros(8, 2, device="cuda"), 2: x.view(8, 2, 2)}, [x, x.view(-1)[4:28].view(8, 3)]):
        with pytest.raises(KernelError, match="share memory"):
            ops.copy_slots(states, [0], [1])
    assert torch.equal(x, keep)


def test_many_slots_of_many_tensors():
    """More copies than travel in a launch's arguments, more tensors than one launch takes."""
    from delta_b200.kernels import ops
    rnd = random.Random(5)
    states = [torch.randn(4000, 1 + i % 5, device="cuda") for i in range(40)]
    want = [s.clone() for s in states]
    dst = rnd.sample(range(4000), 2500)
    src = [rnd.randrange(4000) for _ in dst]
    for w, s in zip(want, states):
        w[dst] = s[src]
    ops.copy_slots(states, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_the_largest_slots():
    """2^31 - 1 bytes that only fit byte by byte: the last block's places pass 2^31."""
    n = (1 << 31) - 1
    a = torch.zeros((2, n), dtype=torch.uint8, device="cuda")
    a[0, ::997] = 7
    a[0, -300:] = torch.arange(300, device="cuda").to(torch.uint8)
    from delta_b200.kernels import ops
    ops.copy_slots([a], [0], [1])
    torch.cuda.synchronize()
    assert torch.equal(a[0], a[1]) and int(a[1, -1]) == 299 - 256
