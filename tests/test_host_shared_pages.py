"""Shared pages, forked and truncated page tables (no GPU)."""
import numpy as np
import pytest

from mlcompiler_b200.host import PagePool, RequestKVState


def filled(pool, tokens, page_size=4, rid=0):
    s = RequestKVState(page_size, rid)
    for _ in range(tokens):
        assert s.extend_one_token(pool) is not None
    return s


def test_share_and_release():
    pool = PagePool(3)
    a = pool.allocate()
    assert pool.owners(a) == 1 and pool.owners(a + 1) == 0 and pool.owners(99) == 0
    assert not pool.share(a + 1) and not pool.share(99)
    assert pool.share(a) and pool.share(a) and pool.owners(a) == 3
    assert pool.pages_in_use() == 1
    assert pool.release(a) and pool.release(a)
    assert pool.owners(a) == 1 and pool.pages_in_use() == 1 and pool.pages_free() == 2
    assert pool.release(a)
    assert pool.owners(a) == 0 and pool.pages_in_use() == 0 and pool.pages_free() == 3
    assert pool.allocate() == a                        # released last, handed out first


@pytest.mark.parametrize("tokens", [1, 3, 4, 5, 8, 11])
def test_fork_shares_everything(tokens):
    pool = PagePool(8)
    parent = filled(pool, tokens)
    child = RequestKVState(64, 1)                      # takes over the parent's page size
    used = pool.pages_in_use()
    assert child.fork(parent, pool)
    assert child.page_table == parent.page_table and child.total_tokens() == tokens
    assert child.tokens_in_last_page == parent.tokens_in_last_page
    assert pool.pages_in_use() == used and all(pool.owners(p) == 2 for p in parent.page_table)
    assert not child.fork(parent, pool) and not parent.fork(parent, pool)
    parent.release_all(pool)
    assert pool.pages_in_use() == used and all(pool.owners(p) == 1 for p in child.page_table)
    child.release_all(pool)
    assert pool.pages_in_use() == 0


def test_extending_into_a_shared_page_copies_it():
    pool = PagePool(6)
    parent = filled(pool, 6)                           # pages 0, 1; two tokens in page 1
    kids = []
    for r in (1, 2):
        c = RequestKVState(4, r)
        assert c.fork(parent, pool)
        kids.append(c)
    assert pool.owners(1) == 3
    assert kids[0].extend_one_token(pool) is None and kids[0].page_table == [0, 1]
    assert kids[0].extend_one_token_owned(pool) == (2, 2, (1, 2))
    assert kids[1].extend_one_token_owned(pool) == (3, 2, (1, 3))
    assert parent.extend_one_token_owned(pool) == (1, 2, None)     # nobody else is left on it
    assert kids[0].page_table == [0, 2] and kids[1].page_table == [0, 3]
    assert [pool.owners(p) for p in range(4)] == [3, 1, 1, 1]
    assert kids[0].extend_one_token_owned(pool) == (2, 3, None)
    assert kids[0].extend_one_token_owned(pool) == (4, 0, None)    # a full page is not written into


def test_extending_fails_without_a_free_page_and_changes_nothing():
    pool = PagePool(2)
    parent = filled(pool, 6)
    child = RequestKVState(4, 1)
    assert child.fork(parent, pool)
    assert child.extend_one_token_owned(pool) is None
    assert child.page_table == [0, 1] and child.total_tokens() == 6 and pool.owners(1) == 2


@pytest.mark.parametrize("keep", range(0, 12))
def test_truncate(keep):
    pool = PagePool(4)
    s = filled(pool, 11)
    assert not s.truncate(pool, 12)
    assert s.truncate(pool, keep)
    assert s.total_tokens() == keep and len(s.page_table) == -(-keep // 4) and pool.pages_in_use() == len(s.page_table)
    assert s.extend_one_token(pool) == (keep // 4, keep % 4) or keep % 4 == 0
    assert s.total_tokens() == keep + 1


def test_truncate_gives_back_only_its_own_share():
    pool = PagePool(4)
    parent = filled(pool, 11)
    child = RequestKVState(4, 1)
    assert child.fork(parent, pool)
    assert child.truncate(pool, 3)
    assert pool.pages_in_use() == 3 and [pool.owners(p) for p in range(3)] == [2, 1, 1]
    assert child.extend_one_token_owned(pool) == (3, 3, (0, 3))
    assert parent.total_tokens() == 11


def test_random_forks_against_a_model():
    """Every page's owners are the states that list it, whatever the order of forks, extensions, truncations and releases."""
    rng = np.random.default_rng(1)
    pool = PagePool(40)
    states = [filled(pool, 9)]
    for _ in range(600):
        op = rng.integers(5)
        s = states[rng.integers(len(states))]
        if op == 0 and len(states) < 6:
            c = RequestKVState(4, 7)
            assert c.fork(s, pool) == bool(s is not c)
            states.append(c)
        elif op == 1 and len(states) > 1:
            s.release_all(pool)
            states.remove(s)
        elif op == 2:
            assert s.truncate(pool, int(rng.integers(s.total_tokens() + 1)))
        else:
            before, total = s.page_table, s.total_tokens()
            got = s.extend_one_token_owned(pool)
            if got is None:
                assert s.page_table == before and s.total_tokens() == total
            else:
                assert s.total_tokens() == total + 1 and s.locate(total) == got[:2] and pool.owners(got[0]) == 1
                if got[2]:
                    assert before[-1] == got[2][0] and s.page_table[-1] == got[2][1] == got[0]
        listed = {}
        for t in states:
            for p in t.page_table:
                listed[p] = listed.get(p, 0) + 1
        assert all(pool.owners(p) == listed.get(p, 0) for p in range(40))
        assert pool.pages_in_use() == len(listed) and pool.pages_in_use() + pool.pages_free() == 40


def test_a_free_page_is_not_released_again():
    pool = PagePool(4)
    a, b = pool.allocate(), pool.allocate()
    assert pool.release(a)
    assert not pool.release(a) and not pool.release(3)  # free, and never handed out
    assert pool.pages_in_use() == 1 and pool.pages_free() == 3 and pool.owners(b) == 1
    got = [pool.allocate() for _ in range(3)]
    assert sorted(got + [b]) == [0, 1, 2, 3] and pool.allocate() is None


def test_a_copy_that_could_not_be_made_is_taken_back():
    pool = PagePool(6)
    parent = filled(pool, 6)                           # pages 0, 1; two tokens in page 1
    child = RequestKVState(4, 1)
    assert child.fork(parent, pool)
    page, slot, copy = child.extend_one_token_owned(pool)
    assert (page, slot, copy) == (2, 2, (1, 2))
    assert not child.undo_copy(pool, 1, 3) and not child.undo_copy(pool, 5, 2)     # not its page; a free page
    assert child.page_table == [0, 2] and pool.owners(2) == 1
    assert child.undo_copy(pool, 1, 2)
    assert child.page_table == [0, 1] and [pool.owners(p) for p in range(3)] == [2, 2, 0]
    assert child.total_tokens() == 7 and child.truncate(pool, 6)
    assert child.extend_one_token_owned(pool) == (2, 2, (1, 2))
