"""The scheduler with trees of drafted tokens: what a step takes for them, and what they give way to (no GPU)."""

import random

from tests.test_scheduler import check_queues, make_scheduler, seq
from tokensprint_b200.engine.scheduler import Scheduler
from tokensprint_b200.engine.speculation import Tree


def chain(nodes):
    return Tree(list(range(1, nodes + 1)), list(range(-1, nodes - 1)))


def decoding(s: Scheduler, lengths, **sampling):
    """Requests whose prompts have run: all tokens but the newest are cached."""
    out = [seq(n, max_tokens=1000, **sampling) for n in lengths]
    for x in out:
        s.add_sequence(x)
    step = s.schedule()
    assert step == out
    s.postprocess(step, [1] * len(step), list(range(len(step))))
    return out


def check_step(s: Scheduler, step, budget):
    check_queues(s)
    assert sum(x.num_new_tokens for x in step) <= budget
    for x in step:
        if x.tree is not None:
            assert x.num_new_tokens == len(x.tree) and x.cache.num_tokens == x.num_cached_tokens + len(x.tree)


def test_a_request_that_took_anothers_place_reserves_for_the_tree_it_has(tmp_path):
    """Neither the tree nor its root finds a page; the last request goes, and the tree has room."""
    s = make_scheduler(tmp_path, num_pages=4, page_size=4)
    a, b = decoding(s, [8, 8])
    a.tree = chain(5)
    step = s.schedule()
    assert step == [a] and s.num_preemptions == 1 and b.cache is None
    assert len(a.tree) == 5
    check_step(s, step, 512)


def test_the_root_alone_where_the_place_taken_is_too_small(tmp_path):
    s = make_scheduler(tmp_path, num_pages=4, page_size=4)
    a, b = decoding(s, [8, 8])
    a.tree = chain(9)
    step = s.schedule()
    assert step == [a] and len(a.tree) == 1 and len(a.cache.tables[0]) == 3
    check_step(s, step, 512)


def test_drafts_give_their_pages_back_before_a_request_loses_its_place(tmp_path):
    """Plain decoding would run both: the first one's drafts hold the page that the second one's next token needs."""
    s = make_scheduler(tmp_path, num_pages=6, page_size=4)
    a, b = decoding(s, [8, 8])
    a.tree = chain(8)
    step = s.schedule()
    assert step == [a, b] and s.num_preemptions == 0
    assert len(a.tree) == 1 and b.num_new_tokens == 1 and s.cache_manager.pools[0].num_free == 0
    check_step(s, step, 512)


def test_only_drafts_that_hold_pages_are_given_up(tmp_path):
    """The nearest request's drafts fit its last page; the one before it holds a page for its own."""
    s = make_scheduler(tmp_path, num_pages=9, page_size=4)
    a, b, c = decoding(s, [8, 9, 8])
    a.tree, b.tree = chain(8), chain(2)
    step = s.schedule()
    assert step == [a, b, c] and s.num_preemptions == 0 and len(a.tree) == 1 and len(b.tree) == 2
    check_step(s, step, 512)


def test_drafts_leave_a_token_of_the_budget_for_every_request_behind(tmp_path):
    s = make_scheduler(tmp_path, num_pages=100, page_size=4, budget=10, chunked=True)
    rows = []
    for n in (2, 2, 2, 2):
        rows += [seq(n, max_tokens=1000)]
        s.add_sequence(rows[-1])
    step = s.schedule()
    s.postprocess(step, [1] * 4, list(range(4)))
    for sizes, want in (((7, 7, 7, 7), [7, 1, 1, 1]), ((8, 8, 8, 8), [1, 1, 1, 1]), ((3, 4, 3, 3), [3, 4, 1, 1]), ((1, 1, 1, 7), [1, 1, 1, 7])):
        for x, n in zip(rows, sizes):
            x.tree = chain(n)
        step = s.schedule()
        assert step == rows and [x.num_new_tokens for x in step] == want
        check_step(s, step, 10)
        s.postprocess_trees(step, [[1]] * 4)


def test_drafts_never_cost_a_request_its_place(tmp_path):
    """Beside a scheduler without drafts: with them nobody is preempted who is not without them, and everybody runs who runs there."""
    rng = random.Random(3)
    for case in range(60):
        pages, lengths = rng.randrange(8, 24), [rng.randrange(1, 17) for _ in range(rng.randrange(1, 6))]
        budget = rng.choice([64, 128])
        with_drafts, plain = (make_scheduler(tmp_path, num_pages=pages, page_size=4, budget=budget, max_model_len=64) for _ in range(2))
        try:
            xs, ys = decoding(with_drafts, lengths, ignore_eos=True), decoding(plain, lengths, ignore_eos=True)
        except AssertionError:  # (not all of them are admitted at once)
            continue
        for x in xs:
            x.tree = chain(rng.randrange(1, 20)) if rng.random() < 0.8 else None
        ran, ran_plain = with_drafts.schedule(), plain.schedule()
        check_step(with_drafts, ran, budget)
        assert with_drafts.num_preemptions == plain.num_preemptions
        assert [xs.index(x) for x in ran] == [ys.index(y) for y in ran_plain]
