"""CPU: what a full paged cache can still do."""
import random

import pytest

from test_paged_kv_cpu import cache  # noqa: F401  (the fixture: a cache on the CPU with plain page copies)


def stamp(c, seq):
    """Writes each token's place and the sequence into its page, where the sequence alone has it."""
    for i, p in enumerate(c.pages_of(seq)):
        if c._users[p] == 1:
            for t in range(min(16, c.length(seq) - 16 * i)):
                c.k_pages[0, p, 0, t, 0] = 16 * i + t
                c.k_pages[0, p, 0, t, 1] = seq


def tokens(c, seq):
    return [c.k_pages[0, p, 0, t, 0].item() for i, p in enumerate(c.pages_of(seq)) for t in range(min(16, c.length(seq) - 16 * i))]


def test_truncate_reuses_a_page_that_it_gives_up(cache):  # noqa: F811
    c = cache(pages=3)
    a = c.new_sequence()
    c.step([a], [32])
    stamp(c, a)
    (b,) = c.fork(a)
    c.step([b], [5])
    assert c.free_pages == 0
    c.truncate(b, 20)  # page 1 is a's too, page 2 b's own
    assert c.pages_of(a) == [0, 1] and c.pages_of(b) == [0, 2] and c.free_pages == 0
    assert c._users == [2, 1, 1] and tokens(c, b) == list(range(20)) and tokens(c, a) == list(range(32))
    c.free(a)
    assert c._users == [1, 0, 1] and c.free_pages == 1


def test_truncate_of_a_full_cache_without_a_page_of_its_own_changes_nothing(cache):  # noqa: F811
    from qik.paged_kv import CacheFull
    c = cache(pages=2)
    a = c.new_sequence()
    c.step([a], [32])
    (b,) = c.fork(a)
    with pytest.raises(CacheFull):
        c.truncate(b, 20)
    assert c.pages_of(b) == [0, 1] and c.length(b) == 32 and c._users == [2, 2]
    c.truncate(b, 16)
    assert c.pages_of(b) == [0] and c._users == [2, 1]


def test_a_failed_copy_within_truncate_changes_nothing(cache, monkeypatch):  # noqa: F811
    import qik.paged_kv as P
    for pages in (3, 4):
        c = cache(pages=pages)
        a = c.new_sequence()
        c.step([a], [32])
        (b,) = c.fork(a)
        c.step([b], [5])
        before = (c._users[:], sorted(c._free), c.pages_of(b), c.length(b))
        with monkeypatch.context() as m:
            m.setattr(P, "copy_pages", lambda *x: (_ for _ in ()).throw(RuntimeError("no")))
            with pytest.raises(RuntimeError):
                c.truncate(b, 20)
        assert before == (c._users[:], sorted(c._free), c.pages_of(b), c.length(b))


def test_random_use_of_a_small_cache(cache):  # noqa: F811
    """Tokens stay, and every page has as many users as sequences hold it."""
    from qik.paged_kv import CacheFull
    r, c, refused = random.Random(5), cache(pages=6), 0
    for _ in range(1500):
        seqs = c.sequences()
        told = {s: c.length(s) for s in seqs}
        try:
            op = r.random()
            if not seqs or op < 0.2:
                s = c.new_sequence()
                c.step([s], [r.randint(1, 40)])
            elif op < 0.45:
                (s,) = c.fork(r.choice(seqs))
            elif op < 0.6:
                s = r.choice(seqs)
                c.step([s], [r.randint(1, 20)])
            elif op < 0.9:
                s = r.choice(seqs)
                n = r.randint(0, c.length(s))
                gives_up = [p for p in c.pages_of(s)[n // 16 + 1:] if c._users[p] == 1]
                could = c.free_pages > 0 or bool(gives_up)
                try:
                    c.truncate(s, n)
                except CacheFull:
                    assert not could
                    raise
            else:
                c.free(r.choice(seqs))
                continue
            stamp(c, s)
        except CacheFull:
            refused += 1
            assert all(c.length(s) == n for s, n in told.items())
            for s in c.sequences()[:2]:
                c.free(s)
        for s in c.sequences():
            assert tokens(c, s) == list(range(c.length(s)))
        assert [sum(p in c.pages_of(s) for s in c.sequences()) for p in range(6)] == c._users
        assert sorted(c._free) == [p for p in range(6) if c._users[p] == 0]
    assert refused > 20
