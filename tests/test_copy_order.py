"""The order in which copies among items are made, and what is refused: on the host."""
import random

import numpy as np
import pytest
import torch

from delta_b200.kernels import lib, ops
from delta_b200.kernels.lib import KernelError

AHEAD = 8


def order(src, dst, items, units_bytes=16, tokens=None, whole=0):
    n = len(src)
    a = [np.asarray(v, dtype=np.int32) for v in (src, dst)]
    t = np.asarray(tokens, dtype=np.int32) if tokens is not None else None
    table = np.array([[4096, units_bytes, units_bytes * items, 1 | units_bytes << 32, 16 | whole << 32 if whole else 0]], dtype=np.int64)
    out = np.full(5 * n + 2, -99, dtype=np.int32)
    lanes = lib.load().dk_copy_items_order(table.ctypes.data, 1, a[0].ctypes.data, a[1].ctypes.data, t.ctypes.data if t is not None else None, n, items,
                                           out.ctypes.data, out.ctypes.data + 16 * n)
    lib.check(min(lanes, 0), "copy_items", 0)
    return out[:4 * n].reshape(n, 4), out[4 * n:4 * n + lanes + 1], lanes


def replay(old, entries, starts, lanes, shuffle):
    """What the kernel's threads do: eight reads ahead of their writes, lanes in any order."""
    new = list(old)
    for lane in shuffle.sample(range(lanes), lanes):
        kept = None
        for i in range(starts[lane], starts[lane + 1], AHEAD):
            batch = []
            for s, d, n, f in entries[i:min(i + AHEAD, starts[lane + 1])]:
                if f & 1:
                    kept = new[d]
                batch.append((d, kept if f & 2 else new[s]))
            for d, v in batch:
                new[d] = v
    return new


@pytest.mark.parametrize("items", [1, 2, 3, 8, 30, 200, 1000])
def test_as_if_all_were_read_first(items):
    rnd = random.Random(items)
    for trial in range(60):
        dst = rnd.sample(range(items), rnd.randint(0, items if trial % 5 else min(items, 3)))      # (few copies of many items are looked up otherwise)
        src = [rnd.randrange(items) for _ in dst] if trial % 3 else rnd.sample(dst, len(dst))       # any copies; permutations
        entries, starts, lanes = order(src, dst, items, units_bytes=16 * rnd.choice([1, 4096, 1 << 16]))
        old = list(range(items))
        want = list(old)
        for s, d in zip(src, dst):
            want[d] = old[s]
        assert replay(old, entries, starts, lanes, rnd) == want
        if lanes:
            assert starts[0] == 0 and (np.diff(starts) > 0).all() and starts[lanes] == sum(s != d for s, d in zip(src, dst))


def test_refused():
    for match, args in [("written twice", ([0, 1], [2, 2], 4)), ("goes from", ([0], [4], 4)), ("goes from", ([4], [0], 4)), ("goes from", ([-1], [0], 4))]:
        with pytest.raises(KernelError, match=match):
            order(*args)
    with pytest.raises(KernelError, match="asks for 17 tokens"):
        order([0], [1], 4, tokens=[17], whole=16)


def test_a_launch_takes_as_many_copies_as_its_caller_says():
    assert lib.load().dk_copy_items_inline() == ops._COPIES_INLINE
    assert lib.load().dk_sizeof_copy_tensor() == 5 * 8


def test_no_cpu_path():
    with pytest.raises(KernelError, match="no CPU path"):
        ops.copy_pages(torch.zeros(1, 4, 8), [0], [1])
    with pytest.raises(KernelError, match="no CPU path"):
        ops.copy_slots([torch.zeros(4, 8)], [0], [1])
    q = torch.zeros(2, 4, 16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(KernelError, match="no CPU path"):
        ops.attention_shared_prefix(q, q, torch.zeros(4, 2, 2, 8, 16), torch.zeros(2, 3, dtype=torch.int32), i, i, i[:2], i[:1], scale=1.0)


@pytest.mark.parametrize("copies", [1, 4])
def test_tensors_that_share_memory_are_refused(copies):
    """Each would overwrite what the other still reads.  (The addresses are never followed here.)"""
    a = np.arange(copies, dtype=np.int32)
    out = np.zeros(5 * copies + 2, dtype=np.int32)

    def call(*pairs):
        table = np.array(pairs, dtype=np.int64)
        to = a + copies
        lanes = lib.load().dk_copy_slots_order(table.ctypes.data, len(pairs), a.ctypes.data, to.ctypes.data, copies, 8, out.ctypes.data, out.ctypes.data + 16 * copies)
        lib.check(min(lanes, 0), "copy_slots", 0)
        return lanes
    assert call((4096, 64), (4160, 64), (8192, 800)) >= 1
    assert call((4096, 64), (0, 0), (0, 0)) >= 1            # empty tensors
    for pairs in [((4096, 64), (4096, 64)), ((4096, 64), (8192, 64), (4152, 64)), ((8192, 64), (4096, 8192))]:
        with pytest.raises(KernelError, match="share memory"):
            call(*pairs)
    with pytest.raises(KernelError, match="no size that is taken"):
        call((4096, 8 << 31))
