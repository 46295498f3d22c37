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
