"""The book of cache pages: sharing, forks, copy on write, freeing, compaction. Host memory only; a numpy array stands for the cache."""
import random

import numpy as np
import pytest

from augur_v100_b200 import kv


class Shadow:
    """A pool with a cache of token values beside it, written and copied as a step would, and the tokens that each sequence should see."""

    def __init__(self, pages, page_tokens):
        self.pool, self.cache, self.tokens, self.count = kv.KvPagePool(pages, page_tokens), np.full((pages, page_tokens), -1), {}, 0

    def copy(self, copies):
        assert len(set(copies.destinations)) == len(copies.destinations) and not set(copies.destinations) & set(copies.sources)
        self.cache[copies.destinations] = self.cache[copies.sources]

    def write(self, sequence, tokens):
        before = self.pool.length(sequence)
        self.copy(self.pool.extend(sequence, tokens))
        pages = self.pool.page_list(sequence)
        for at in range(before, before + tokens):
            self.count += 1
            self.cache[pages[at // self.pool.page_tokens], at % self.pool.page_tokens] = self.count
            self.tokens[sequence].append(self.count)

    def check(self):
        pool = self.pool
        held = np.zeros(pool.pages, dtype=int)
        for sequence, tokens in self.tokens.items():
            pages = pool.page_list(sequence)
            assert pool.length(sequence) == len(tokens) and len(pages) == -(-len(tokens) // pool.page_tokens)
            assert list(self.cache[pages].reshape(-1)[:len(tokens)]) == tokens
            for page in pages:
                held[page] += 1
        assert list(held) == pool._holders and pool.free_pages() == int((held == 0).sum())


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("page_tokens", [1, 4, 16])
def test_sequences_keep_their_tokens(seed, page_tokens):
    rng = random.Random(seed * 31 + page_tokens)
    s = Shadow(40, page_tokens)
    for _ in range(300):
        live = list(s.tokens)
        act = rng.choice(("create", "write", "write", "write", "fork", "truncate", "free", "compact"))
        try:
            if act == "create" or not live:
                sequence = s.pool.create()
                s.tokens[sequence] = []
            elif act == "write":
                s.write(rng.choice(live), rng.choice((0, 1, 1, 5, 23)))
            elif act == "fork":
                sequence = rng.choice(live)
                twin, copies = s.pool.fork(sequence)
                s.copy(copies)
                s.tokens[twin] = list(s.tokens[sequence])
            elif act == "truncate":
                sequence = rng.choice(live)
                keep = rng.randint(0, len(s.tokens[sequence]))
                s.pool.truncate(sequence, keep)
                del s.tokens[sequence][keep:]
            elif act == "free":
                sequence = rng.choice(live)
                s.pool.free(sequence)
                del s.tokens[sequence]
            else:
                s.copy(s.pool.compact())
                used = s.pool.pages - s.pool.free_pages()
                assert all(page < used for sequence in s.tokens for page in s.pool.page_list(sequence))
        except kv.OutOfPages:
            if act in ("write", "fork") and len(live) > 1:        # make room
                s.pool.free(live[0])
                del s.tokens[live[0]]
        s.check()


def test_a_pool_without_room_changes_nothing():
    pool = kv.KvPagePool(2, 16)
    a = pool.create()
    pool.extend(a, 17)
    with pytest.raises(kv.OutOfPages):
        pool.extend(a, 16)
    with pytest.raises(kv.OutOfPages):
        pool.fork(a)
    assert pool.length(a) == 17 and pool.page_list(a) == [0, 1] and pool.sequences() == [a]
    pool.truncate(a, 16)
    twin, copies = pool.fork(a)                       # full pages are shared: nothing to copy
    assert copies == ([], []) and pool.page_list(twin) == [0] and pool.free_pages() == 1
    pool.truncate(twin, 3)
    copies = pool.extend(twin, 1)                     # a shared page is not written: it is copied first
    assert copies == ([0], [1]) and pool.page_list(twin) == [1] and pool.page_list(a) == [0]


def test_tables_and_refusals():
    pool = kv.KvPagePool(8, 16)
    a, b = pool.create(), pool.create()
    pool.extend(a, 40)
    table = pool.table([a, None, b])
    assert table.tolist() == [[0, 1, 2], [-1, -1, -1], [-1, -1, -1]] and table.dtype == kv.torch.int32
    assert pool.table([], 4).shape == (0, 4) and pool.table([b]).shape == (1, 1)
    for bad in (lambda: pool.table([a], 2), lambda: pool.extend(a, -1), lambda: pool.truncate(a, 41), lambda: pool.truncate(a, -1),
                lambda: kv.KvPagePool(0, 16)):
        with pytest.raises(ValueError):
            bad()
    pool.free(a)
    for gone in (lambda: pool.free(a), lambda: pool.length(a), lambda: pool.fork(a)):
        with pytest.raises(KeyError):
            gone()
