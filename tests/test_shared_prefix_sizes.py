"""What attention over shared prefixes asks for under an engine's limits: working memory, rows (no GPU: sizes and choices only)."""
import ctypes
import types

import pytest
import torch

from delta_b200.kernels import lib, ops
from delta_b200.kernels.lib import KernelError
from delta_b200.parts import attention_kernels


@pytest.fixture(autouse=True)
def on_device_0(monkeypatch):
    monkeypatch.setattr(ops, "_device_index", lambda: 0)


def context(rows, max_rows, max_pages=64, pages=1000, scratch=None):
    """As much of a step as the part looks at; ``calls`` gets what would be launched."""
    calls = []
    tables = dict(kv_len=0, members=0, group_start=0, group_prefix=0)
    ctx = types.SimpleNamespace(shared=dict(g=tables), plain_kernels=frozenset(), num_rows=rows, max_rows=max_rows, max_pages=max_pages, err=None,
                                cache=types.SimpleNamespace(max_pages_per_request=max_pages))
    ctx.scratch = scratch or (lambda key, shape, dtype, bound=None: calls.append((shape[0], bound[0])))
    return ctx, calls


def cache_view(pages=1000, KV=2, ps=16, hd=64):
    return types.SimpleNamespace(group="g", page_size=ps, block_table=None, pages=types.SimpleNamespace(shape=(pages, 2, KV, ps, hd)))


@pytest.mark.parametrize("max_rows", [8, 1024, 1025, 2000, 100000])
def test_an_engine_of_many_slots(monkeypatch, max_rows):
    """A call takes 1,024 rows; the engine may have more slots, and a step of few rows still goes there."""
    monkeypatch.setattr(ops, "attention_shared_prefix", lambda *a, **k: None)
    qkv, out = torch.zeros(8, 6 * 64, dtype=torch.bfloat16), torch.zeros(8, 2 * 64, dtype=torch.bfloat16)
    ctx, calls = context(8, max_rows)
    attention_kernels.run_shared(ctx, qkv, out, cache_view(), 2, 2, 64, 0.125)
    (asked, bound), = calls
    assert asked == ops.attention_shared_prefix_floats(8, 4, 8, 2, 2, 64, 16, 64, 1000, torch.bfloat16)
    most = min(max_rows, 1024)
    assert bound == ops.attention_shared_prefix_floats(most, most // 2, most, 2, 2, 64, 16, 64, 1000, torch.bfloat16) >= asked
    with pytest.raises(KernelError, match="at most 1024 rows"):
        ops.attention_shared_prefix_floats(1025, 4, 8, 2, 2, 64, 16, 64, 1000, torch.bfloat16)
