"""Requests that share their first positions, on the host: pages and their holders, the batch's runs of
neighbours, and the engine over the test-only kernel table."""

import numpy as np
import pytest
import torch

from somi_inference_b200.cache import CacheManager
from somi_inference_b200.cache.pages import OutOfPages, PagePool
from somi_inference_b200.engine import Engine, StepEntry
from somi_inference_b200.engine.batch import BatchBuilder
from somi_inference_b200.parts.base import CacheNeeds, PagedKVNeeds, StateNeeds
from tests.plain import qwen2_plain as plain
from tests.plain.host_ops import HostOps
from tests.tiny import make_model, random_tokens


def manager(needs=None, pages=20, page_size=4):
    needs = needs or [CacheNeeds(paged=PagedKVNeeds(1, 16, None))]
    return CacheManager(needs, [None] * len(needs), num_pages=pages, page_size=page_size, max_requests=6, max_positions=64,
                        dtype=torch.float32, device="cpu")


def grow(m, r, n):
    m.reserve(r, n)
    m.commit(r)


def test_a_shared_page_is_free_with_its_last_holder():
    p = PagePool(4)
    a = p.take(2)
    p.share(a)
    p.share(a[:1])
    assert [p.holders(x) for x in a] == [3, 2] and p.num_held == 2
    p.give_back(a)
    p.give_back(a)
    assert p.num_held == 1 and p.is_held(a[0]) and not p.is_held(a[1])
    with pytest.raises(RuntimeError):
        p.give_back(a[1:])
    with pytest.raises(RuntimeError):
        p.share(a)                                       # a[1] is free: nothing is shared
    assert p.holders(a[0]) == 1
    p.give_back(a[:1])
    assert p.num_free == 4


def test_forks_share_whole_pages_in_any_order_of_release():
    g = np.random.default_rng(0)
    for _ in range(30):
        m = manager()
        m.register("of")
        grow(m, "of", 11)
        for i in range(3):
            m.fork(i, "of", 8)
            assert m.length(i) == 8 and m.held_pages(i, 0) == m.held_pages("of", 0)[:2]
        assert m.free_pages() == [20 - 3]
        for i in range(3):
            grow(m, i, int(g.integers(1, 9)))
            m.reserve(i, 5)
            m.cancel(i)
            m.check_consistency()
        grow(m, "of", 3)
        live = ["of", 0, 1, 2]
        first = {r: m.held_pages(r, 0)[:2] for r in live}
        assert len({tuple(v) for v in first.values()}) == 1
        tails = [p for r in live for p in m.held_pages(r, 0)[2:]]
        assert len(set(tails)) == len(tails) and not set(tails) & set(first["of"])
        for r in g.permutation(np.array(live, dtype=object)):
            m.release(r)
            m.check_consistency()
        assert m.free_pages() == [20] and not m.any_family


def test_families():
    m = manager()
    for r in ("a", "b"):
        m.register(r)
        grow(m, r, 12)
    assert m.family("a") == (0, 0)
    m.fork("a1", "a", 8)
    m.fork("a2", "a", 4)
    m.fork("a11", "a1", 8)
    m.fork("b1", "b", 12)
    assert m.family("a") == m.family("a1") == m.family("a11") == (1, 8) and m.family("a2") == (1, 4)
    assert m.family("b") == m.family("b1") == (2, 12)


def test_what_cannot_be_forked_is_refused_and_changes_nothing():
    m = manager()
    m.register("a")
    grow(m, "a", 9)
    for of, n in (("x", 4), ("a", 0), ("a", 3), ("a", 12), ("a", -4)):
        with pytest.raises(ValueError):
            m.fork("r", of, n)
    with pytest.raises(ValueError):
        m.fork("a", "a", 4)
    for needs in ([CacheNeeds(paged=PagedKVNeeds(1, 16, 8))],
                  [CacheNeeds(paged=PagedKVNeeds(1, 16, None), state=StateNeeds({"s": ((2,), torch.float32)}))]):
        other = manager(needs)
        other.register("a")
        grow(other, "a", 8)
        with pytest.raises(ValueError):
            other.fork("r", "a", 4)
        assert not other.is_registered("r")
    for i in range(5):
        m.fork(i, "a", 4)
    with pytest.raises(OutOfPages):
        m.fork("r", "a", 4)                              # every slot is taken
    assert not m.is_registered("r")
    m.check_consistency()


def test_the_batch_names_neighbours_that_share():
    m = manager(pages=40)
    b = BatchBuilder(m, device="cpu", q_tile_sizes=(16,))
    for r in ("a", "b", "c"):
        m.register(r)
        grow(m, r, 12)

    def build(*entries):
        for r, n in entries:
            m.reserve(r, n)
        batch, _ = b.build([StepEntry(r, [0] * n, [0]) for r, n in entries])
        for r, _ in entries:
            m.cancel(r)
        return batch

    plain_key = build(("a", 1), ("b", 1)).layout_key
    assert build(("a", 1), ("b", 1)).shared is None
    m.fork("a1", "a", 8)
    m.fork("a2", "a", 4)
    m.fork("b1", "b", 12)
    assert build(("a", 1), ("b", 1)).shared is None and build(("a", 1), ("b", 1)).layout_key == plain_key
    s = build(("a", 1), ("a1", 1), ("c", 1), ("b", 1), ("b1", 1), ("a2", 1)).shared
    assert s.group_off.tolist() == [0, 2, 3, 5, 6] and s.prefix_len.tolist() == [8, 0, 12, 0]
    assert s.saved_bits == (8 + 12).bit_length()
    s = build(("a", 1), ("a1", 1), ("a2", 1)).shared
    assert s.group_off.tolist() == [0, 3] and s.prefix_len.tolist() == [4]
    # portions come first, in the order in which they were given
    batch = build(("a2", 1), ("b", 3), ("a", 1), ("b1", 2), ("c", 1))
    assert batch.host.requests == ["b", "b1", "a2", "a", "c"]
    assert batch.shared.group_off.tolist() == [0, 2, 4, 5] and batch.shared.prefix_len.tolist() == [12, 4, 0]
    assert build(("a", 1), ("c", 1), ("a1", 1)).shared is None      # no neighbours


def test_neighbours_that_share_nothing_are_one_run():
    """Only the runs that share count: a step of many requests has no more groups than a block keeps copies of."""
    m = CacheManager([CacheNeeds(paged=PagedKVNeeds(1, 16, None))], [None], num_pages=200, page_size=4, max_requests=60,
                     max_positions=64, dtype=torch.float32, device="cpu")
    b = BatchBuilder(m, device="cpu", q_tile_sizes=(16,))
    alone = [f"alone{i}" for i in range(40)]
    for r in ("a", "b", *alone):
        m.register(r)
        grow(m, r, 8)
    for r, of in (("a1", "a"), ("a2", "a"), ("b1", "b")):
        m.fork(r, of, 8)

    def runs(*order, portion=()):
        for r in order:
            m.reserve(r, 2 if r in portion else 1)
        s = b.build([StepEntry(r, [0, 0] if r in portion else [0], [0]) for r in order])[0].shared
        for r in order:
            m.cancel(r)
        return s.group_off.tolist(), s.prefix_len.tolist(), s.saved_bits

    assert runs(*alone, "a", "a1", "a2") == ([0, 40, 43], [0, 8], (16).bit_length())
    assert runs("a", "a1", *alone, "b", "b1") == ([0, 2, 42, 44], [8, 0, 8], (16).bit_length())
    assert runs("b", "alone0", "a", "b1", "a1", "a2", "alone1") == ([0, 4, 6, 7], [0, 8, 0], (8).bit_length())
    # portions come first
    assert runs(*alone, "a", "a1", "b", "b1", portion=("alone3", "b", "b1")) == ([0, 1, 3, 42, 44], [0, 8, 0, 8], (16).bit_length())


def test_a_batch_says_what_its_portions_share():
    """What decides which kernels a step launches is part of its layout."""
    m = CacheManager([CacheNeeds(paged=PagedKVNeeds(1, 16, None))], [None], num_pages=2000, page_size=4, max_requests=20,
                     max_positions=4000, dtype=torch.float32, device="cpu")
    b = BatchBuilder(m, device="cpu", q_tile_sizes=(16,))
    for r, n in (("a", 300), ("b", 8), ("new", 0), ("deep", 256), ("deeper", 1200)):
        m.register(r)
        if n:
            grow(m, r, n)
    for r, of, n in (("a1", "a", 300), ("a2", "a", 300), ("b1", "b", 8), ("b2", "b", 8)):
        m.fork(r, of, n)

    def build(**entries):
        for r, n in entries.items():
            m.reserve(r, n)
        batch = b.build([StepEntry(r, [0] * n, [0]) for r, n in entries.items()])[0]
        for r in entries:
            m.cancel(r)
        return batch

    def facts(**entries):
        return build(**entries).shared.portions

    assert facts(a=1, a1=1) is None                               # single tokens only
    assert facts(a=1, a1=1, new=3) == (0, False, False)
    assert facts(b=2, b1=1, a=1, a1=1) == ((8).bit_length(), False, False)      # the run of portions goes on among single tokens
    assert facts(b=1, b1=1, a=2, a1=3) == ((300).bit_length(), True, False)
    assert facts(a=1, a1=1, deep=64) == (0, True, False) and facts(a=1, a1=1, deep=65) == (0, False, False)
    assert facts(a=1, a1=1, b=1, b1=1, new=1024) == (0, False, False) and facts(a=1, a1=1, new=1025) == (0, False, True)
    assert facts(a=1, a1=1, deeper=300) == (0, True, False)
    # equal sizes, other facts: other layouts
    one, two = build(a=1, a1=1, deep=64, new=66), build(a=1, a1=1, deep=66, new=64)
    assert one.layout_key != two.layout_key and one.layout_key[:-1] == two.layout_key[:-1]


@pytest.fixture(scope="module")
def root(tmp_path_factory):
    return str(tmp_path_factory.mktemp("fork"))


def test_forked_requests_continue_like_whole_ones(root):
    d = make_model("A", root, torch.float32, std=0.08)
    cfg, w = plain.load_folder(d)
    eng = Engine(d, dtype="float32", page_size=16, num_pages=12, device="cpu", ops=HostOps())
    prompt = random_tokens(37, cfg["vocab_size"], 1)
    eng.step([StepEntry("p", prompt, [36])])
    assert eng.fork("none", "p", 15) == 0 and not eng.has("none")
    for of, n in (("p", 38), ("p", -1), ("unknown", 16)):
        with pytest.raises(ValueError):
            eng.fork("none", of, n)
    ends = {f"r{i}": random_tokens(n, cfg["vocab_size"], 2 + i) for i, n in enumerate((7, 1, 20))}
    assert [eng.fork(r, "p") for r in ends] == [32] * 3
    assert eng.length("r1") == 32 and eng.cache.free_pages() == [12 - 3]
    got = eng.step([StepEntry(r, prompt[32:] + t, [4 + len(t)]) for r, t in ends.items()])
    for row, t in zip(got, ends.values()):
        assert (row - plain.logits(cfg, w, prompt + t)[-1]).abs().max() < 3e-5
    eng.end("p")
    got = eng.step([StepEntry(r, [3], [0]) for r in ends])
    for row, t in zip(got, ends.values()):
        assert (row - plain.logits(cfg, w, prompt + t + [3])[-1]).abs().max() < 3e-5
    for r in ends:
        eng.end(r)
    assert eng.cache.free_pages() == [12]
