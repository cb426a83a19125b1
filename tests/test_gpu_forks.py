"""Requests forked from one another through the engine: the same tokens as requests that compute everything themselves, with prompts computed
once, in every design (recurrent states, windows, latent caches), under preemption, from recorded steps, and with the cache compacted
in the middle; and attention that reads shared pages once against attention that does not."""
import json
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import burolorn_helpers
import helpers
import mevulix_helpers
import mufalix_helpers
import pibalorn_helpers
import roletar_helpers
import vazunex_helpers

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
DESIGNS = dict(roletar=roletar_helpers, pibalorn=pibalorn_helpers, mufalix=mufalix_helpers, mevulix=mevulix_helpers, vazunex=vazunex_helpers,
               burolorn=burolorn_helpers)


def backend(model, dtype="float32", graph=False, min_bytes=None, **kw):
    from delta_b200.engine import LMBackend
    e = LMBackend(dtype=dtype, device="cuda:0", cuda_graph_decode=graph)
    e.load_model(model)
    e.setup_caches(check_kernel_errors=True, **dict(dict(max_batch_size=8, max_seq_length=256, page_size=16), **kw))
    if min_bytes is not None:
        e.runner.shared_prefix_min_bytes = min_bytes
    return e


def done(e):
    e.runner.cache.check()
    assert all(v == 0 for v in e.runner.cache.pages_in_use().values())


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graphs"])
@pytest.mark.parametrize("min_bytes", [None, 0], ids=["apart", "shared"])
@pytest.mark.parametrize("which", "ABCD")
def test_samples_are_what_separate_requests_are(model_folders, which, min_bytes, graph):
    vocab = helpers.tiny_config(which)["vocab_size"]
    prompts = [helpers.random_tokens(n, vocab, 40 + n) for n in (33, 70)]
    ps = helpers.PAGE_SIZE[which]
    e = backend(model_folders[which], graph=graph, min_bytes=min_bytes, page_size=ps)
    outs = e.generate(prompts, 12, temperature=0.8, seed=5, samples=3)
    assert e.scheduler.stats["forks"] == 4 and e.scheduler.stats["prompt_tokens"] == 33 + 70 + 4
    done(e)
    want = backend(model_folders[which], page_size=ps).generate([p for p in prompts for _ in range(3)], 12, temperature=0.8, seed=5)
    assert outs == want
    if graph:
        shared = any(isinstance(k, tuple) for k in e.runner._graphs)
        assert shared == (min_bytes == 0) and e.runner.graph_replays > 0 and not e.runner.graph_fallbacks


def test_a_common_first_part(model_folders):
    vocab = helpers.tiny_config("B")["vocab_size"]
    common = helpers.random_tokens(50, vocab, 1)
    prompts = [common + helpers.random_tokens(n, vocab, 60 + n) for n in (1, 20, 7, 90)]
    e = backend(model_folders["B"], graph=True, min_bytes=0, page_size=8, max_tokens_per_step=32)
    outs = e.generate(prompts, 10, share_prefix=True)
    assert e.scheduler.stats["forks"] == 3 and e.scheduler.stats["prompt_tokens"] == 50 + 1 + 20 + 7 + 90
    done(e)
    assert outs == backend(model_folders["B"], page_size=8).generate(prompts, 10)
    # samples of prompts with a common first part: the pages are divided where that saves the most
    e = backend(model_folders["B"], graph=True, min_bytes=0, page_size=8)
    outs = e.generate(prompts[1:], 10, samples=2, share_prefix=True, temperature=0.7, seed=9)
    assert e.scheduler.stats["forks"] == 5
    done(e)
    assert outs == backend(model_folders["B"], page_size=8).generate([p for p in prompts[1:] for _ in range(2)], 10, temperature=0.7, seed=9)


@pytest.mark.parametrize("budget", [32, 512])
def test_samples_of_prompts_with_a_common_first_part_compute_each_once(model_folders, budget):
    vocab = helpers.tiny_config("B")["vocab_size"]
    common = helpers.random_tokens(50, vocab, 1)
    prompts = [common + helpers.random_tokens(n, vocab, 60 + n) for n in (20, 7)]
    e = backend(model_folders["B"], min_bytes=0, page_size=8, max_tokens_per_step=budget)
    outs = e.generate(prompts, 6, samples=3, share_prefix=True, temperature=0.7, seed=9)
    assert e.scheduler.stats["forks"] == 5 and e.scheduler.stats["prompt_tokens"] == 50 + 20 + 7 + 2 * 2
    done(e)
    assert outs == backend(model_folders["B"], page_size=8).generate([p for p in prompts for _ in range(3)], 6, temperature=0.7, seed=9)


@pytest.mark.parametrize("design", list(DESIGNS))
@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graphs"])
def test_every_design_can_be_forked(design, graph, tmp_path):
    from roletar_helpers import write_folder
    h = DESIGNS[design]
    cfg, weights = h.build("mix", 3)[:2] if hasattr(h, "build") else (h.config("mix"), h.make_weights(h.config("mix"), 3))
    folder = write_folder(tmp_path, design, cfg, weights)
    prompt = helpers.random_tokens(37, cfg["vocab"], 8)
    e = backend(folder, graph=graph, max_tokens_per_step=64)
    outs = e.generate([prompt], 8, samples=4, temperature=0.6, seed=2)
    assert e.scheduler.stats["forks"] == 3 and e.scheduler.stats["prompt_tokens"] == 37 + 3
    done(e)
    assert outs == backend(folder, max_tokens_per_step=64).generate([prompt] * 4, 8, temperature=0.6, seed=2)


@pytest.mark.parametrize("design", list(DESIGNS))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graphs"])
def test_every_design_reads_shared_pages_once(design, dtype, graph, tmp_path):
    """Whatever else a design has in its layers, those that read every page take the shared ones once; in bfloat16 every sample runs to its end."""
    from roletar_helpers import write_folder
    h = DESIGNS[design]
    cfg, weights = h.build("mix", 3)[:2] if hasattr(h, "build") else (h.config("mix"), h.make_weights(h.config("mix"), 3))
    folder = write_folder(tmp_path, design, cfg, weights)
    prompt = helpers.random_tokens(37, cfg["vocab"], 8)
    e = backend(folder, dtype=dtype, graph=graph, min_bytes=0, max_tokens_per_step=64)
    outs = e.generate([prompt], 8, samples=4, temperature=0.6, seed=2)
    assert e.scheduler.stats["forks"] == 3 and all(len(o) == 8 for o in outs)
    done(e)
    if dtype == "float32":
        assert outs == backend(folder, max_tokens_per_step=64).generate([prompt] * 4, 8, temperature=0.6, seed=2)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graphs"])
@pytest.mark.parametrize("min_bytes", [None, 0], ids=["apart", "shared"])
def test_samples_with_chosen_pages(model_folders, min_bytes, graph):
    """Layers that choose pages for others: their choices are a request's own, full layers read shared pages once."""
    vocab = helpers.tiny_config("A")["vocab_size"]
    prompts = [helpers.random_tokens(n, vocab, 40 + n) for n in (75, 130)]
    sel = dict(enable_selective_cache=True, full_cache_layers=[0], subset_cache_size=4, page_size=8)
    e = backend(model_folders["A"], graph=graph, min_bytes=min_bytes, **sel)
    outs = e.generate(prompts, 20, temperature=0.8, seed=5, samples=3)
    assert e.scheduler.stats["forks"] == 4
    done(e)
    assert outs == backend(model_folders["A"], **sel).generate([p for p in prompts for _ in range(3)], 20, temperature=0.8, seed=5)


def test_forks_under_preemption(model_folders):
    """A pool that cannot hold all samples to their end: some are preempted and forked again or computed anew."""
    vocab = helpers.tiny_config("A")["vocab_size"]
    prompt = helpers.random_tokens(40, vocab, 3)
    want = backend(model_folders["A"]).generate([prompt] * 5, 60, temperature=0.9, seed=4)
    e = backend(model_folders["A"], graph=True, min_bytes=0, num_pages=14)
    assert e.generate([prompt], 60, samples=5, temperature=0.9, seed=4) == want
    assert e.scheduler.stats["preemptions"] > 0 and e.scheduler.stats["forks"] >= 4
    done(e)


@pytest.mark.parametrize("dtype,which", [("float32", "A"), ("bfloat16", "D")])
def test_compaction_in_the_middle(model_folders, dtype, which):
    vocab = helpers.tiny_config(which)["vocab_size"]
    prompts = [helpers.random_tokens(n, vocab, 70 + n) for n in (90, 40)]
    outs = []
    for compact in (False, True):
        e = backend(model_folders[which], dtype=dtype, graph=True, num_pages=200)
        pool = next(iter(e.runner.cache.groups.values())).pool
        taken = pool.alloc(200)
        pool.free(taken[::3])                      # what is left to the requests lies scattered
        e.add_requests(prompts, 200, samples=3, temperature=0.7, seed=1, max_new_tokens=40)
        for _ in range(20):
            e.step()
        if compact:
            # (the pages that stand for other requests are nobody's in the tables: they are given back first)
            pool.free([p for i, p in enumerate(taken) if i % 3])
            moved = e.compact_cache()
            assert sum(moved.values()) > 10
            for g in e.runner.cache.groups.values():
                for s in range(8):
                    held = g.held(s)
                    assert all(b == a + 1 or (a % 8 == 7 and b % 8 == 0) for a, b in zip(held, held[1:])) or not e.runner.cache.is_live(s) or g.pool.holders(held[0]) > 1
            assert sum(e.compact_cache().values()) <= sum(moved.values())
            e.runner.cache.check()
        e.run_scheduler_loop()
        outs.append([r.output for r in e.scheduler.requests])
    assert outs[0] == outs[1] and all(len(o) == 40 for o in outs[0])


@pytest.mark.parametrize("heads", [(6, 2, 64), (8, 1, 128), (24, 2, 128)], ids=str)
def test_shared_pages_read_once_in_bfloat16(heads):
    """The same tokens through a runner that reads shared pages once and one that does not.  Two layers whose attention outputs are rounded at
    most three times differently (2^-8 of a value each): logits within 2 x 3 x 2^-8 of the largest."""
    from delta_b200.config import EngineConfig
    from delta_b200.engine.step import ModelRunner, RowInput
    H, KV, hd = heads
    cfg = dict(architectures=["LlamaForCausalLM"], hidden_size=192, num_hidden_layers=2, num_attention_heads=H, num_key_value_heads=KV, head_dim=hd,
               intermediate_size=208, vocab_size=384, rope_theta=1e6, rms_norm_eps=1e-5, max_position_embeddings=512, tie_word_embeddings=False)
    logits = []
    for min_bytes in (1 << 60, 0):
        r = ModelRunner(config_json=cfg, seed=1, engine_config=EngineConfig(max_batch=8, max_seq_len=512, page_size=16, dtype="bfloat16"))
        r.shared_prefix_min_bytes = min_bytes
        prompt = helpers.random_tokens(301, 384, 5)
        slot = r.cache.acquire_slot()
        r.run_rows([RowInput(slot, prompt, 0)])
        slots = [slot] + r.cache.fork(slot, 301, 2) + r.cache.fork(slot, 200, 2)
        lone = r.cache.acquire_slot()
        r.run_rows([RowInput(lone, helpers.random_tokens(77, 384, 6), 0)])
        slots.insert(2, lone)
        mine = []
        for step in range(6):
            rows = [RowInput(s, helpers.random_tokens(1, 384, 100 * step + i), int(r.cache.seq_len[s]), [0]) for i, s in enumerate(slots)]
            assert bool(r._shared_groups(rows, [1] * 6)) == (min_bytes == 0)
            mine.append(r.run_rows(rows))
        r.check_errors()
        logits.append(torch.stack(mine).double())
    off = (logits[0] - logits[1]).abs().max() / logits[0].abs().max()
    assert off <= 6 * 2.0 ** -8, off
    assert off > 0           # two ways, not one


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graphs"])
def test_an_engine_of_more_slots_than_a_call_takes_rows(model_folders, graph):
    vocab = helpers.tiny_config("A")["vocab_size"]
    prompt = helpers.random_tokens(40, vocab, 3)
    e = backend(model_folders["A"], graph=graph, min_bytes=0, max_batch_size=1100, max_seq_length=64, num_pages=2000)
    outs = e.generate([prompt], 6, samples=5, temperature=0.9, seed=4)
    assert e.scheduler.stats["forks"] == 4
    done(e)
    assert outs == backend(model_folders["A"]).generate([prompt] * 5, 6, temperature=0.9, seed=4)
    from delta_b200.parts.attention_kernels import SHARED_WORK
    assert SHARED_WORK in e.runner._scratch


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graphs"])
def test_an_engine_without_room_for_the_working_memory(model_folders, graph, monkeypatch):
    """Rows that share pages read them each for itself then."""
    from delta_b200.engine.context import StepContext
    from delta_b200.parts.attention_kernels import SHARED_WORK
    have = StepContext.scratch

    def scratch(self, key, *a, **k):
        if key == SHARED_WORK:
            raise torch.OutOfMemoryError("the device is full")
        return have(self, key, *a, **k)
    monkeypatch.setattr(StepContext, "scratch", scratch)
    prompt = helpers.random_tokens(40, helpers.tiny_config("A")["vocab_size"], 3)
    e = backend(model_folders["A"], graph=graph, min_bytes=0)
    with pytest.warns(RuntimeWarning, match="no memory on the device"):
        outs = e.generate([prompt], 8, samples=5, temperature=0.9, seed=4)
    assert e.scheduler.stats["forks"] == 4 and not e.runner.graph_fallbacks
    done(e)
    assert outs == backend(model_folders["A"]).generate([prompt] * 5, 8, temperature=0.9, seed=4)


def test_command_line(model_folders, tmp_path):
    out = tmp_path / "r.json"
    r = subprocess.run([sys.executable, "-m", "delta_b200.cli", "--model", str(model_folders["A"]), "--B", "6", "--max_len", "128", "--dataset", "random", "--num_samples",
                        "2", "--prompt_len", "20", "--samples", "3", "--share_prefix", "--max_new_tokens", "5", "--temperature", "0.8", "--dtype", "float32",
                        "--cuda_graph_decode", "--out", str(out)], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    got = json.loads(out.read_text())
    assert got["summary"]["forks"] == 4 and got["summary"]["prompt_tokens"] == 2 * 20 + 4 and len(got["results"]) == 6
