"""Requests that share pages, moved pages, and the scheduler's families: bookkeeping on the host (no GPU)."""
import random

import pytest
import torch

from delta_b200.cache import CacheManager, OutOfPages, PagePool
from delta_b200.engine.scheduler import FINISHED, RUNNING, WAITING, Scheduler
from delta_b200.parts.base import PAGE, CacheSpec, StateSpec


def manager(num_pages=32, page_size=4, max_slots=6, max_seq_len=64, window=None, states=None, run_tokens=0, **kw):
    specs = {0: CacheSpec((2, 2, PAGE, 8), run_tokens=run_tokens), 1: CacheSpec((2, 2, PAGE, 8), run_tokens=run_tokens)}
    if window:
        specs[2] = CacheSpec((2, 2, PAGE, 8), window)
    return CacheManager(specs, states or {}, max_slots=max_slots, max_seq_len=max_seq_len, page_size=page_size,
                        num_pages=num_pages, dtype=torch.float32, device="cpu", **kw)


def hold(m, n):
    s = m.acquire_slot()
    m.grow(s, n)
    m.advance(s, n)
    return s


def only(m):
    return next(iter(m.groups.values()))


def test_a_page_is_free_when_its_last_holder_gives_it_back():
    p = PagePool(8, run_pages=4)
    a = p.alloc(3)
    p.share(a[:2])
    assert p.holders(a[0]) == 2 and p.holders(a[2]) == 1 and p.holders(7) == 0 and p.holders(99) == 0
    p.free(a)
    assert p.free_pages == 6 and p.held_pages == 2
    p.check()
    with pytest.raises(ValueError, match="twice"):
        p.free([a[2]])
    with pytest.raises(ValueError, match="held by nobody"):
        p.share([a[2]])
    p.free(a[:2])
    assert p.free_pages == 8
    p.check()


def test_moved_pages_keep_their_holders():
    p = PagePool(16, run_pages=4)
    a = p.alloc(6)
    p.share([a[1]])
    p.relocate({a[1]: 9, a[2]: a[1], a[5]: 15})
    p.check()
    assert [p.holders(x) for x in (a[0], a[1], a[2], 9, 15, a[5])] == [1, 1, 0, 2, 1, 0]
    with pytest.raises(ValueError, match="cannot be moved"):
        p.relocate({a[0]: 9})
    with pytest.raises(ValueError, match="held by nobody"):
        p.relocate({a[2]: 12})


@pytest.mark.parametrize("length", [1, 3, 4, 11, 12, 13])
def test_fork_shares_whole_pages_and_copies_the_last(length):
    m = manager()
    g = only(m)
    a = hold(m, 13)
    g.pages.copy_(torch.randn(g.pages.shape))
    before = g.pages.clone()
    free = g.pool.free_pages
    new = m.fork(a, length, 2)
    whole, rest = divmod(length, 4)
    assert free - g.pool.free_pages == (2 if rest else 0)
    m.check()
    for s in new:
        assert m.seq_len[s] == length and g.table[s, :whole].tolist() == g.table[a, :whole].tolist()
        assert (g.table[s, whole + (1 if rest else 0):] == -1).all()
        if rest:
            page = int(g.table[s, whole])
            assert page != g.table[a, whole]
            assert torch.equal(g.pages[:, page, :, :, :rest], before[:, int(g.table[a, whole]), :, :, :rest])
            assert torch.equal(g.pages[:, page, :, :, rest:], before[:, page, :, :, rest:])       # the others are left as they were
    m.grow(new[0], length + 9)
    m.release_slot(a)
    m.check()
    m.release_slot(new[1])
    m.release_slot(new[0])
    m.check()
    assert g.pool.held_pages == 0


def test_fork_is_all_or_nothing():
    m = manager(num_pages=6, max_slots=4)
    a = hold(m, 18)                                     # five pages
    with pytest.raises(OutOfPages):
        m.fork(a, 17, 2)
    with pytest.raises(RuntimeError, match="no free request slot"):
        m.fork(a, 16, 4)
    assert m.free_slots == 3 and only(m).pool.free_pages == 1
    for bad in (0, 19, -1):
        with pytest.raises(ValueError, match="cannot be forked"):
            m.fork(a, bad)
    m.check()
    assert len(m.fork(a, 16, 3)) == 3                   # whole pages only: nothing is taken
    m.check()


def test_fork_behind_a_window_and_with_states():
    m = manager(window=8, states={"s": StateSpec((3,), torch.float32, 0.5)})
    a = hold(m, 22)
    m.states["s"][a] = torch.tensor([1.0, 2.0, 3.0])
    with pytest.raises(ValueError, match="cannot be forked"):
        m.fork(a, 21)                                   # the state is that of 22 tokens
    b = m.fork(a)[0]
    assert m.states["s"][b].tolist() == [1.0, 2.0, 3.0]
    m.check()
    for _ in range(3):
        for s in (a, b):
            n = int(m.seq_len[s]) + 5
            m.grow(s, n)
            m.advance(s, n)
            m.check()
    m.release_slot(a)
    m.release_slot(b)
    assert all(g.pool.held_pages == 0 for g in m.groups.values())
    m = manager(window=8, states={"s": StateSpec((3,), torch.float32, 0.5)}, states_follow_tokens=False)
    a = hold(m, 30)
    m.states["s"][a] = 7
    with pytest.raises(ValueError, match="cannot be forked"):
        m.fork(a, 12)                                   # what the window has passed is gone
    assert m.states["s"][m.fork(a, 29)[0]].tolist() == [0.5] * 3
    m.check()


@pytest.mark.parametrize("follow", [True, False])
def test_a_fork_writes_each_state_tensor_once(follow):
    """However many forks: one copy of the states (or one fill, where they are made anew), not a fill for every tensor and slot."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Writes(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.ops = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func._schema.is_mutable:
                self.ops.append((str(func), args[0].untyped_storage().data_ptr()))
            return func(*args, **(kwargs or {}))
    m = manager(num_pages=64, max_slots=12, states={k: StateSpec((3,), torch.float32, 0.5) for k in "abcde"}, states_follow_tokens=follow)
    a = hold(m, 8)
    for s in m.states.values():
        s.copy_(torch.arange(13.0)[:, None].expand(13, 3))
    with Writes() as w:
        new = m.fork(a, 8 if follow else 4, 9)
    storages = {s.untyped_storage().data_ptr() for s in m.states.values()}
    assert len([x for x in w.ops if x[1] in storages]) == 5, w.ops
    for s in m.states.values():
        assert (s[new] == (float(a) if follow else 0.5)).all()
        assert all((s[x] == float(x)).all() for x in range(13) if x not in new)
    m.check()


def test_shared_prefixes():
    m = manager(num_pages=64, max_slots=8)
    name, g = next(iter(m.groups.items()))
    a = hold(m, 30)                                     # seven whole pages
    b, c = m.fork(a, 28, 2)                             # all seven
    d = m.fork(a, 9)[0]                                 # two of them
    e = hold(m, 12)
    f = m.fork(e, 8)[0]
    assert m.shared_prefixes(name, [a, b]) == [([0, 1], 7)]
    assert m.shared_prefixes(name, [e]) == [] and m.shared_prefixes(name, [a, e]) == []
    assert m.shared_prefixes(name, [d, a]) == [([0, 1], 2)]
    # of four, three share seven pages: 14 saved, where all four would save 6; the rows keep their places
    assert sorted(m.shared_prefixes(name, [e, a, d, c, f, b])) == [([0, 4], 2), ([1, 3, 5], 7)]
    m.release_slot(b)
    m.release_slot(c)
    assert m.shared_prefixes(name, [a, d, e]) == [([0, 1], 2)]
    m.release_slot(a)
    assert m.shared_prefixes(name, [d, e]) == []


def test_compaction_moves_contents_with_the_tables():
    rnd = random.Random(0)
    for trial in range(20):
        m = manager(num_pages=40, max_slots=8, max_seq_len=64, run_tokens=16)       # runs of four pages
        name, g = next(iter(m.groups.items()))
        live = [hold(m, rnd.randint(1, 20)) for _ in range(3)]
        live += m.fork(live[0], rnd.randint(1, int(m.seq_len[live[0]])), 2)
        for _ in range(40):
            s = rnd.choice(live)
            n = int(m.seq_len[s]) + rnd.randint(1, 6)
            if rnd.random() < 0.2 and len(live) > 1:
                m.release_slot(s)
                live.remove(s)
            elif m.can_grow(s, n):
                m.grow(s, n)
                m.advance(s, n)
            if m.free_slots and rnd.random() < 0.3 and g.pool.free_pages > 3:
                live.append(hold(m, rnd.randint(1, 12)))
        g.pages.copy_(torch.arange(g.pages.shape[1], dtype=torch.float32)[None, :, None, None, None, None].expand_as(g.pages))
        want = {s: [g.pages[:, p].clone() for p in g.held(s)] for s in live}
        free = g.pool.free_pages
        moved = m.compact()[name]
        m.check()
        assert g.pool.free_pages == free
        for s in live:
            assert all(torch.equal(g.pages[:, p], x) for p, x in zip(g.held(s), want[s]))
        assert m.compact()[name] <= moved
        for s in live:
            if m.can_grow(s, int(m.seq_len[s]) + 4):
                m.grow(s, int(m.seq_len[s]) + 4)
        m.check()


def test_compaction_makes_runs():
    m = manager(num_pages=32, max_slots=4, run_tokens=16, shuffle_seed=None)
    name, g = next(iter(m.groups.items()))
    a, b = m.acquire_slot(), m.acquire_slot()
    # two requests whose pages lie alternately
    pages = g.pool.alloc(16)
    for i, s in enumerate((a, b)):
        g.table[s, :8] = pages[i::2]
        g.num_logical[s] = 8
        m.seq_len[s] = 32
    m.check()
    assert m.compact()[name] > 0
    for s in (a, b):
        held = g.held(s)
        assert held == list(range(held[0], held[0] + 4)) + list(range(held[4], held[4] + 4)) and held[0] % 4 == held[4] % 4 == 0
    m.check()
    assert m.compact() == {name: 0}
    scattered = manager(num_pages=32, run_tokens=16, shuffle_seed=3)
    hold(scattered, 20)
    assert sum(scattered.compact().values()) == 0


def test_compaction_that_is_refused_moves_nothing():
    """Pages that are held but stand in no table may be a move's target: the pool refuses before any page is copied."""
    m = manager(num_pages=32, max_slots=4, run_tokens=16)
    name, g = next(iter(m.groups.items()))
    foreign = g.pool.alloc(4)
    a, b = m.acquire_slot(), m.acquire_slot()
    pages = g.pool.alloc(16)
    for i, s in enumerate((a, b)):
        g.table[s, :8] = pages[i::2]
        g.num_logical[s] = 8
        m.seq_len[s] = 32
    g.pages.copy_(torch.arange(33.0)[None, :, None, None, None, None].expand_as(g.pages))
    before, table = g.pages.clone(), g.table.copy()
    with pytest.raises(ValueError, match="cannot be moved"):
        m.compact()
    assert torch.equal(g.pages, before) and (g.table == table).all()
    g.pool.check()
    g.pool.free(foreign)
    assert m.compact()[name] > 0
    m.check()


# ---------------------------------------------------------------- the scheduler

def run(s, cache, tokens=lambda r: len(r.output), watch=None, steps=500):
    """Runs to the end with made-up tokens; returns the prompt tokens each request computed."""
    done = {}
    for _ in range(steps):
        if not s.has_work():
            break
        plan = s.schedule()
        cache.check()
        for x in plan:
            assert x.request.computed == x.start and int(cache.seq_len[x.request.slot]) == x.start
            if not x.decode:
                done[x.request.id] = done.get(x.request.id, 0) + x.count
        if watch:
            watch(plan)
        s.complete(plan, [tokens(x.request) for x in plan if x.samples])
        cache.check()
    assert not s.has_work()
    return done


def requests(s, prompts, new=5, **kw):
    return [s.add_request(p, 64, max_new_tokens=new, **kw) for p in prompts]


def test_samples_compute_their_prompt_once():
    c = manager(num_pages=64)
    s = Scheduler(c, max_batch=6, max_tokens_per_step=16)
    other = requests(s, [[9] * 5])
    rs = requests(s, [list(range(21))] * 4)
    s.relate(rs, 20)
    done = run(s, c)
    assert sorted(done[r.id] for r in rs) == [1, 1, 1, 21] and done[other[0].id] == 5
    assert s.stats["forks"] == 3 and all(r.status == FINISHED and len(r.output) == 5 for r in rs)
    assert only(c).pool.held_pages == 0


def test_a_common_first_part_is_computed_once():
    c = manager(num_pages=64)
    s = Scheduler(c, max_batch=6, max_tokens_per_step=8)
    prompts = [list(range(18)) + [100 + i] * (1 + 3 * i) for i in range(4)]
    rs = requests(s, prompts)
    s.relate(rs, 18)
    done = run(s, c)
    assert [done[r.id] for r in rs] == [19, 4, 7, 10] and s.stats["forks"] == 3
    with pytest.raises(ValueError, match="are not the same"):
        s.relate(rs[1:], 19)


def test_states_are_forked_where_they_are():
    """A model with recurrent states stops its portion where the others begin, so that nothing is computed twice there either."""
    c = manager(num_pages=64, states={"s": StateSpec((2,), torch.float32, 0.0)})
    s = Scheduler(c, max_batch=6, max_tokens_per_step=64)
    rs = requests(s, [list(range(21))] * 3)
    s.relate(rs, 20)
    sums = lambda r: float(sum(r.tokens[:r.computed]))       # noqa: E731  (a state that tells what it has seen)

    def watch(plan):
        for x in plan:
            assert c.states["s"][x.request.slot, 0] == sums(x.request)
            c.states["s"][x.request.slot, 0] += sum(x.request.tokens[x.start:x.start + x.count])
    done = run(s, c, watch=watch)
    assert sorted(done[r.id] for r in rs) == [1, 1, 21] and s.stats["forks"] == 2


def test_families_under_a_short_pool():
    """Few pages and slots: some are forked, some are preempted and computed again; everything ends, no page is lost."""
    rnd = random.Random(1)
    for trial in range(30):
        c = manager(num_pages=rnd.randint(17, 24), max_slots=rnd.randint(2, 5), states={"s": StateSpec((1,), torch.float32, 0.0)} if trial % 3 == 0 else None,
                    window=8 if trial % 4 == 1 else None)
        s = Scheduler(c, max_batch=c.max_slots, max_tokens_per_step=rnd.choice([3, 8, 40]), decode_singly=trial % 5 == 0)
        s.decode_while_prefill = trial % 7 != 0
        common = [rnd.randrange(50) for _ in range(rnd.randint(1, 20))]
        rs = []
        for _ in range(3):
            prompt = common + [rnd.randrange(50) for _ in range(rnd.randint(1, 8))]
            mine = requests(s, [prompt] * rnd.randint(1, 3), new=rnd.randint(1, 12))
            s.relate(mine, len(prompt) - 1)
            rs += mine
        s.relate(rs, len(common))
        run(s, c, steps=3000)
        assert all(r.status == FINISHED and r.output for r in rs), [r.finish_reason for r in rs]
        assert all(g.pool.held_pages == 0 for g in c.groups.values())


@pytest.mark.parametrize("budget", [8, 16, 64, 512])
@pytest.mark.parametrize("states", [False, True])
def test_samples_of_prompts_with_a_common_first_part(budget, states):
    """Two families in one another: the common part is computed once, then every prompt's rest once, and its samples wait for it."""
    c = manager(num_pages=300, max_slots=12, states={"s": StateSpec((2,), torch.float32, 0.0)} if states else None)
    s = Scheduler(c, max_batch=12, max_tokens_per_step=budget)
    rs = []
    for i in range(3):
        mine = requests(s, [list(range(20)) + [100 * i + 60 + j for j in range(40)]] * 4, new=3)
        s.relate(mine, 59)
        rs += mine
    s.relate(rs, 20)
    done = run(s, c)
    assert [done[r.id] for r in rs] == [60, 1, 1, 1, 40, 1, 1, 1, 40, 1, 1, 1]
    assert s.stats["forks"] == 11 and all(r.status == FINISHED for r in rs)


def test_forks_pass_an_older_request_only_while_their_family_runs():
    """A fork needs few pages and may start before an older request that waits for many: the families under way end, later ones wait behind it."""
    c = manager(num_pages=20, max_slots=12)
    s = Scheduler(c, max_batch=12, max_tokens_per_step=64)
    first = requests(s, [list(range(21))], new=12)
    big = s.add_request([7] * 62, 64, max_new_tokens=2)
    first += requests(s, [list(range(21))] * 3, new=12)
    s.relate(first, 20)
    later = []

    def watch(plan):
        if len(later) < 40:
            mine = requests(s, [[50 + len(later)] * 9] * 2, new=3)
            s.relate(mine, 8)
            later.extend(mine)
    run(s, c, watch=watch, steps=2000)
    assert all(r.status == FINISHED for r in s.requests)
    assert all(r.admitted_order < big.admitted_order < x.admitted_order for r in first for x in later)


def test_a_follower_computes_for_itself_when_nobody_holds_the_beginning():
    c = manager(num_pages=64, max_slots=1)
    s = Scheduler(c, max_batch=1, max_tokens_per_step=64)
    rs = requests(s, [list(range(10))] * 2)
    s.relate(rs, 9)
    done = run(s, c)
    assert [done[r.id] for r in rs] == [10, 10] and s.stats["forks"] == 0


def test_only_whole_relations():
    c = manager()
    s = Scheduler(c, max_batch=2, max_tokens_per_step=64)
    a, b = requests(s, [[1], [1]])
    s.relate([a, b], 1)              # nothing of a prompt of one token can be shared: its last token is computed
    s.relate([a], 5)
    assert not a.families and not b.families and a.status == WAITING
    run(s, c)
    assert RUNNING not in (a.status, b.status)
