"""plan_shared_prefixes and SequenceState.fork_prefix (host only)."""
import pytest

import kvflux_b200 as kv


def pool(capacity=4000, block=16):
    return kv.PhysicalBlockPool(capacity, block)


def grown(p, rid, tokens):
    s = kv.SequenceState(rid, p)
    if tokens:
        s.append_tokens(tokens)
    return s


def children(source, pages, extra):
    """One sequence per entry of `extra`: the source's first pages and that many tokens of its own."""
    out = []
    for i, n in enumerate(extra):
        c = source.fork_prefix(100 + i, pages)
        if n:
            c.append_tokens(n)
        out.append(c)
    return out


def plan(seqs):
    return [(g.rows, g.prefix_tokens) for g in kv.plan_shared_prefixes(seqs)]


def test_forks_of_one_prompt_share_its_full_pages():
    p = pool()
    src = grown(p, 1, 20 * 16 + 5)
    seqs = [src] + children(src, 20, [1, 40, 0, 7])
    assert plan(seqs) == [(5, 320)]


def test_a_shorter_common_prefix_ends_where_tables_differ():
    p = pool()
    src = grown(p, 1, 50 * 16)
    assert plan([src] + children(src, 30, [100, 100])) == [(3, 480)]


def test_prompts_of_their_own_are_groups_of_their_own():
    p = pool()
    a, b = grown(p, 1, 160), grown(p, 2, 16 * 40)
    seqs = children(a, 10, [1, 2, 3]) + children(b, 40, [9, 9])
    assert plan(seqs) == [(3, 160), (2, 640)]


def test_short_and_lonely_prefixes_share_nothing_and_merge():
    p = pool()
    a, b = grown(p, 1, 16 * 7), grown(p, 2, 16 * 100)
    lone = [grown(p, 10 + i, 300) for i in range(3)]
    assert plan(children(a, 7, [1, 1, 1]) + lone) == [(6, 0)]
    assert plan(lone[:2] + children(b, 100, [5, 5]) + lone[2:]) == [(2, 0), (2, 1600), (1, 0)]


def test_a_run_does_not_give_up_more_than_it_gains():
    """Two rows share 100 pages; a third shares 40 with them: 2 x 40 < 1 x 100. A third with 60 joins."""
    p = pool()
    src = grown(p, 1, 16 * 100)
    two = children(src, 100, [1, 1])
    assert plan(two + children(src, 40, [16 * 70])) == [(2, 1600), (1, 0)]
    assert plan(two + children(src, 60, [16 * 70])) == [(3, 960)]


def test_partial_shared_pages_do_not_count():
    p = pool()
    src = grown(p, 1, 16 * 9 + 3)
    twins = [src.fork_shared(2), src.fork_shared(3)]  # the partial page too
    assert plan(twins) == [(2, 144)]


def test_edges():
    p = pool()
    assert plan([]) == []
    empty = kv.SequenceState(1, p)
    assert plan([empty, grown(p, 2, 500), empty]) == [(3, 0)]
    with pytest.raises(ValueError):
        kv.plan_shared_prefixes([empty, None])
    with pytest.raises(ValueError):
        kv.plan_shared_prefixes([empty, kv.SequenceState(1, pool())])


def test_fork_prefix_shares_and_returns_pages():
    p = pool(capacity=12, block=4)
    src = grown(p, 1, 4 * 5 + 2)
    with pytest.raises(IndexError):
        src.fork_prefix(2, 6)  # the sixth page is not full
    c = src.fork_prefix(2, 5)
    assert c.num_tokens() == 20 and c.request_id() == 2 and p.available() == 6
    assert [c.physical_block_id(i) for i in range(5)] == [src.physical_block_id(i) for i in range(5)]
    assert c.block_table().ref_count(0) == 2 and src.block_table().ref_count(5) == 1
    c.append_tokens(3)  # a page of its own
    assert p.available() == 5 and c.physical_block_id(5) != src.physical_block_id(5)
    c.move_from(src.fork_prefix(3, 0))
    assert c.num_tokens() == 0 and p.available() == 6 and src.block_table().ref_count(0) == 1


@pytest.mark.parametrize("pages", [31, 32, 33, 63, 64, 65, 100])
def test_common_pages_end_at_any_entry(pages):
    p = pool()
    src = grown(p, 1, 120 * 16)
    assert plan([src] + children(src, pages, [900, 900])) == [(3, pages * 16)]
    assert plan(children(src, pages, [900]) + [src]) == [(2, pages * 16)]
