"""PagePool's forks, copy-on-write and compaction on the host: who owns what
afterwards, against a model of the contents (CPU only)."""

import random

import pytest

from mini_engine_hip.cache.page_pool import PagePool


class Model:
    """A pool whose pages hold a list of (request, position) marks; moves copy them."""

    def __init__(self, pool):
        self.pool, self.pages, self.text = pool, {}, {}

    def run(self, moves):
        sources, targets = [s for s, _ in moves], [d for _, d in moves]
        assert len(set(targets)) == len(targets) and not set(sources) & set(targets)
        for src, dst in moves:
            self.pages[dst] = list(self.pages.get(src, []))

    def write(self, request, value):
        """Append one token to a request's text and to its page."""
        size, at = self.pool.block_size, len(self.text[request])
        page, moves = self.pool.make_writable(request, at // size)
        self.run(moves)
        assert self.pool.refcount(page) == 1
        row = self.pages.setdefault(page, [])
        row[at % size:] = [value]
        self.text[request].append(value)

    def check(self):
        size, held = self.pool.block_size, [0] * self.pool.num_blocks
        for request, text in self.text.items():
            table = self.pool.table(request)
            for page in table:
                held[page] += 1
            for at, value in enumerate(text):
                assert self.pages[table[at // size]][at % size] == value
        for page in range(self.pool.num_blocks):
            assert self.pool.refcount(page) >= held[page]
        assert self.pool.free_blocks == sum(self.pool.refcount(p) == 0 for p in range(self.pool.num_blocks))


def test_fork_shares_whole_pages_and_copies_the_partial_one():
    pool = PagePool(8, 4)
    table = pool.allocate("a", 12)
    child, moves = pool.fork("a", "b", 10)
    assert child[:2] == table[:2] and child[2] not in table and moves == [(table[2], child[2])]
    assert [pool.refcount(p) for p in table] == [2, 2, 1] and pool.refcount(child[2]) == 1
    child, moves = pool.fork("a", "c", 8)
    assert child == table[:2] and moves == []
    child, moves = pool.fork("a", "d", 0)
    assert child == [] and moves == []
    pool.free("a")
    pool.free("b")
    pool.free("c")
    pool.free("d")
    assert pool.free_blocks == 8


def test_fork_refusals_change_nothing():
    pool = PagePool(3, 4)
    pool.allocate("a", 9)
    for args, error in ((("a", "a", 4), ValueError), (("a", "b", 13), ValueError), (("a", "b", -1), ValueError),
                        (("x", "b", 0), KeyError), (("a", "b", 9), MemoryError)):
        with pytest.raises(error):
            pool.fork(*args)
        assert [pool.refcount(p) for p in pool.table("a")] == [1, 1, 1] and pool.free_blocks == 0
    with pytest.raises(IndexError):
        pool.make_writable("a", 3)
    pool.pin(pool.table("a")[:1])
    with pytest.raises(MemoryError):
        pool.make_writable("a", 0)
    assert pool.refcount(pool.table("a")[0]) == 2


def test_compaction_moves_pages_down_and_leaves_pinned_ones():
    pool = PagePool(10, 4, order=[9, 0, 8, 1, 7, 2, 6, 3, 5, 4])
    pool.allocate("a", 12)          # 9, 0, 8
    pool.allocate("b", 8)           # 1, 7
    pool.fork("a", "c", 8)          # shares 9, 0
    pool.pin([8])
    moves = pool.compact()
    assert moves == [(7, 3), (9, 2)]
    assert pool.table("a") == [2, 0, 8] and pool.table("c") == [2, 0] and pool.table("b") == [1, 3]
    assert pool.refcount(2) == 2 and pool.refcount(9) == 0 and pool.refcount(8) == 2
    assert pool.allocate("d", 4) == [4]
    assert pool.compact() == []


@pytest.mark.parametrize("seed", range(8))
def test_random_life_of_a_pool(seed):
    """Allocations, forks, writes, frees, pins and compactions: every request reads its own text at every step."""
    rng = random.Random(seed)
    pool = PagePool(60, rng.choice([1, 3, 4]), order=rng.sample(range(60), 60))
    model, names, pinned = Model(pool), 0, []
    for _ in range(400):
        step = rng.choice("awwwwffxpuc")
        live = list(model.text)
        try:
            if step == "a":
                names += 1
                pool.allocate(f"r{names}", rng.randint(1, 6 * pool.block_size))
                model.text[f"r{names}"] = []
            elif step == "w" and live:
                request = rng.choice(live)
                if len(model.text[request]) < len(pool.table(request)) * pool.block_size:
                    model.write(request, rng.random())
            elif step == "f" and live:
                names += 1
                parent = rng.choice(live)
                count = rng.randint(0, len(model.text[parent]))
                _, moves = pool.fork(parent, f"r{names}", count)
                model.text[f"r{names}"] = model.text[parent][:count]
                model.run(moves)
            elif step == "x" and live:
                request = rng.choice(live)
                pool.free(request)
                del model.text[request]
            elif step == "p" and live and pool.table(request := rng.choice(live)):
                pinned.append(rng.choice(pool.table(request)))
                pool.pin(pinned[-1:])
            elif step == "u" and pinned:
                pool.unpin([pinned.pop()])
            elif step == "c":
                moves = pool.compact()
                assert [s for s, _ in moves] == sorted(s for s, _ in moves) and all(d < s for s, d in moves)
                model.run(moves)
        except MemoryError:
            pass
        model.check()


def test_extension_appends_private_pages():
    pool = PagePool(8, 4)
    table = pool.allocate("a", 6)
    assert pool.extend("a", 8) == table and pool.extend("a", 0) == table
    child, _ = pool.fork("a", "b", 8)  # whole pages: not one token fits behind them
    assert child == table
    grown = pool.extend("b", 9)
    assert grown[:2] == table and len(grown) == 3 and pool.refcount(grown[2]) == 1 and pool.table("b") == grown
    assert pool.table("a") == table
    assert len(pool.extend("a", 20)) == 5 and pool.free_blocks == 2
    for args, error in ((("b", 24), MemoryError), (("b", -1), ValueError), (("x", 4), KeyError)):
        with pytest.raises(error):
            pool.extend(*args)
        assert pool.table("b") == grown and pool.free_blocks == 2
    pool.free("a")
    pool.free("b")
    assert pool.free_blocks == 8


@pytest.mark.parametrize("seed", range(8))
def test_branches_grow_past_their_fork(seed):
    """Forks at any length, page boundaries among them; every branch then writes on, through compactions too."""
    rng = random.Random(seed)
    size = rng.choice([1, 3, 4])
    pool = PagePool(120, size, order=rng.sample(range(120), 120))
    model = Model(pool)
    pool.allocate("r0", size)
    model.text["r0"] = []
    for step in range(300):
        request = rng.choice(list(model.text))
        text = model.text[request]
        if step % 12 == 11 and len(model.text) < 6:
            count = rng.choice([0, len(text), len(text) // size * size, rng.randint(0, len(text))])
            child = f"r{step}"
            _, moves = pool.fork(request, child, count)
            model.run(moves)
            model.text[child] = text[:count]
        elif step % 31 == 30:
            model.run(pool.compact())
        elif len(text) < 15 * size:
            pool.extend(request, len(text) + 1)
            model.write(request, rng.random())
        model.check()
    assert min(len(text) for text in model.text.values()) > size and len(model.text) == 6
