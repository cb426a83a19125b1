"""What attention over shared prefixes asks for under an engine's limits: working memory, rows (no GPU: sizes and choices only)."""
import types

import pytest
import torch

from delta_b200.kernels import lib, ops
from delta_b200.kernels.lib import KernelError
from delta_b200.parts import attention_kernels


@pytest.fixture(autouse=True)
def on_device_0(monkeypatch):
    monkeypatch.setattr(ops, "_device_index", lambda: 0)


def context(rows, max_rows, max_pages=64, dtype=torch.bfloat16):
    """As much of a step as the part looks at; ``asked`` gets what working memory is asked for."""
    asked = []
    ctx = types.SimpleNamespace(shared=dict(g=None), plain_kernels=frozenset(), num_rows=rows, max_rows=max_rows, max_pages=max_pages, dtype=dtype,
                                cache=types.SimpleNamespace(max_pages_per_request=max_pages))
    ctx.scratch_if_there = lambda key, shape, dtype, bound=None: asked.append((shape[0], bound[0])) or torch.empty(0)
    return ctx, asked


def cache_view(pages=1000, KV=2, ps=16, hd=64, group="g"):
    return types.SimpleNamespace(group=group, page_size=ps, pages=types.SimpleNamespace(shape=(pages, 2, KV, ps, hd)))


@pytest.mark.parametrize("max_rows", [8, 1024, 1025, 2000, 100000])
def test_an_engine_of_many_slots(max_rows):
    """A call takes 1,024 rows; the engine may have more slots, and a step of few rows still goes there."""
    ctx, calls = context(8, max_rows)
    assert attention_kernels.shared_work(ctx, cache_view(), 2, 2, 64) is not None
    (asked, bound), = calls
    assert asked == ops.attention_shared_prefix_floats(8, 4, 8, 2, 2, 64, 16, 64, 1000, torch.bfloat16)
    most = min(max_rows, 1024)
    assert bound == ops.attention_shared_prefix_floats(most, most // 2, most, 2, 2, 64, 16, 64, 1000, torch.bfloat16) >= asked
    with pytest.raises(KernelError, match="at most 1024 rows"):
        ops.attention_shared_prefix_floats(1025, 4, 8, 2, 2, 64, 16, 64, 1000, torch.bfloat16)
    assert attention_kernels.shared_work(context(1025, 2000)[0], cache_view(), 2, 2, 64) is None
    assert attention_kernels.shared_work(context(8, 8)[0], cache_view(group="another"), 2, 2, 64) is None


def test_a_device_without_room(monkeypatch):
    """The cache may hold nearly all of the device: a step goes on without the kernels whose working memory is not to be had, and so do all later ones."""
    from delta_b200.engine.context import StepContext
    ctx = StepContext.__new__(StepContext)
    ctx._scratch_pool, ctx.device, tries = {}, "cpu", []

    def full(*a, **k):
        tries.append(1)
        raise torch.OutOfMemoryError("full")
    with monkeypatch.context() as m:
        m.setattr(torch, "empty", full)
        with pytest.warns(RuntimeWarning, match="'shared'.*without it"):
            assert ctx.scratch_if_there("shared", (5,), torch.float32, bound=(50,)) is None
        with pytest.raises(torch.OutOfMemoryError):
            ctx.scratch("other", (5,), torch.float32)
    assert ctx.scratch_if_there("shared", (5,), torch.float32) is None and len(tries) == 2
    assert ctx.scratch_if_there("another", (5,), torch.float32, bound=(50,)).shape == (5,)


def megabytes(rows, keys, pool, dtype=torch.bfloat16, KV=8, H=32):
    return ops.attention_shared_prefix_floats(rows, rows // 2, rows, H, KV, 128, 16, keys // 16, pool // 16, dtype) * 4 / 1e6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_working_memory_goes_with_the_cache(dtype):
    """Groups hold no more than the pool does: long tables over a small pool ask for no more than a tenth of one layer's share of it and a piece's results
    (128 queries of 132 floats; 32 in 32 bits) for every segment and block."""
    item = torch.empty((), dtype=dtype).element_size()
    queries, grid = (128, 148) if dtype == torch.bfloat16 else (32, 444)
    for rows, keys, pool in [(64, 131072, 262144), (64, 131072, 1 << 20), (256, 65536, 262144), (1024, 131072, 262144), (8, 8192, 65536)]:
        layer = pool * 2 * 8 * 128 * item / 1e6
        rpt = queries // 4
        pieces = 8 * (rows // rpt + rows // 2) + grid + rows * 8 + 2 * grid
        behind_all = rows // rpt * 8 * keys / (rpt * 4) / 48          # one group of all rows over the longest table, 48 tiles to a piece
        assert megabytes(rows, keys, pool, dtype) < 0.1 * layer + (pieces + behind_all) * queries * 132 * 4 * 1.1 / 1e6
    assert megabytes(64, 131072, 262144, dtype) < 0.4 * megabytes(64, 131072, 1 << 24, dtype)
    # more rows or longer tables never ask for less: an engine's buffer is made for its largest step
    sizes = [megabytes(r, k, 262144, dtype) for r in range(2, 200, 7) for k in (4096, 131072)]
    assert all(a <= b for a, b in zip(sizes[::2], sizes[2::2])) and all(a <= b for a, b in zip(sizes[1::2], sizes[3::2])) and all(a <= b for a, b in zip(sizes[::2], sizes[1::2]))
