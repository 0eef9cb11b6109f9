"""fork_sequence, compact_sequence, write_paged_kv_rotated and
paged_attention_batch_shared: each one's checks and effects, and a run of them
as a serving loop makes it (prompt, forks, decode steps over the shared
prefix, an eviction, more steps) with every attention output checked in 64
bits over what the cache holds.

Attention tolerance: Q and the weights are pairs of 16-bit values, off by at
most 2^-17 of themselves (bf16: unit 2^-7, low part up to 2^-8, whose unit is
2^-16); with A = the row's largest sum |q_i k_i| / sqrt(hd),
a score is off by at most A (2^-17 + hd 2^-23), which counts twice (weight and
sum); 2^-17 + 2^-21 for weights and exponential, n 2^-23 for n additions; all
against sum p |v|."""
import math

import numpy as np
import pytest
import torch

import kvflux_b200 as kv

pytestmark = pytest.mark.gpu

KVH, QH, HD, BS = 2, 8, 128, 16


def storages(pool, layers=2, dtype=kv.DType.BFloat16):
    return [kv.PagedKVStorage(pool, KVH, HD, dtype, 0) for _ in range(layers)]


def cached(storage, seq):
    """K and V of a sequence as [tokens][heads][hd], as stored."""
    n = seq.num_tokens()
    k, v = (torch.zeros(n, KVH, HD, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kv.read_paged_kv(storage, seq, k, v)
    return k.cpu(), v.cpu()


def fill(layers, seq, first, gen):
    """Random K/V at positions first.. of a sequence, in every layer."""
    n = seq.num_tokens() - first
    slots = kv.build_slot_mapping([(seq, t) for t in range(first, seq.num_tokens())])
    for s in layers:
        k, v = (torch.randn(n, KVH, HD, generator=gen).bfloat16().cuda() for _ in range(2))
        kv.write_paged_kv(s, k, v, slots)


def check_row(q, k, v, got):
    q = q.double().view(KVH, -1, HD)
    k, v = (x.double().permute(1, 0, 2) for x in (k, v))
    p = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(HD), -1)
    a = (q.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) / math.sqrt(HD)
    tol = (p @ v.abs()) * (2 * a * (2.0**-17 + HD * 2.0**-23) + 2.0**-17 + 2.0**-21 + k.shape[1] * 2.0**-23)
    assert torch.all((got.double().view(KVH, -1, HD) - p @ v).abs() <= tol)


def test_forks_share_full_pages_and_own_the_last():
    pool = kv.PhysicalBlockPool(64, BS)
    layers = storages(pool, 3)
    gen = torch.Generator().manual_seed(1)
    src = kv.SequenceState(1, pool)
    src.append_tokens(5 * BS + 3)
    fill(layers, src, 0, gen)
    kids = kv.fork_sequence(layers, src, [2, 3, 4, 5])
    assert [c.request_id() for c in kids] == [2, 3, 4, 5] and pool.available() == 64 - 6 - 4
    for s in layers:
        want = cached(s, src)
        for c in kids:
            got = cached(s, c)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for c in kids:
        assert c.physical_block_id(4) == src.physical_block_id(4) and c.physical_block_id(5) != src.physical_block_id(5)
    # Source and children append without copy-on-write, apart from one another.
    before = cached(layers[0], src)[0]
    for c in [*kids, src]:
        c.append_token()
        fill(layers, c, c.num_tokens() - 1, gen)
    last = [cached(layers[0], c)[0] for c in [*kids, src]]
    for i, x in enumerate(last):
        assert torch.equal(x[:-1], before)
        assert all(not torch.equal(x[-1], y[-1]) for y in last[i + 1:])
    del kids, c
    assert pool.available() == 64 - 6


def test_forks_of_whole_pages_copy_nothing():
    pool = kv.PhysicalBlockPool(8, BS)
    layers = storages(pool, 1)
    src = kv.SequenceState(1, pool)
    src.append_tokens(3 * BS)
    kids = kv.fork_sequence(layers, src, [2, 3])
    assert pool.available() == 5 and [c.num_tokens() for c in kids] == [48, 48]
    assert kv.fork_sequence(layers, src, []) == []
    empty = kv.fork_sequence(layers, kv.SequenceState(9, pool), [4])
    assert empty[0].num_tokens() == 0


def test_fork_that_runs_out_of_pages_changes_nothing():
    pool = kv.PhysicalBlockPool(6, BS)
    layers = storages(pool, 1)
    src = kv.SequenceState(1, pool)
    src.append_tokens(3 * BS + 1)
    with pytest.raises(kv.CapacityError):
        kv.fork_sequence(layers, src, [2, 3, 4])
    assert pool.available() == 2 and src.block_table().ref_count(0) == 1


def test_fork_and_compaction_refuse_foreign_sequences_and_layers():
    pool, other = kv.PhysicalBlockPool(8, BS), kv.PhysicalBlockPool(8, BS)
    layers = storages(pool, 1)
    seq = kv.SequenceState(1, other)
    seq.append_tokens(20)
    odd = [layers[0], kv.PagedKVStorage(pool, KVH, 64, kv.DType.BFloat16, 0)]
    mine = kv.SequenceState(2, pool)
    mine.append_tokens(20)
    for bad_layers, s in ((layers, seq), ([], mine), (odd, mine)):
        with pytest.raises(ValueError):
            kv.fork_sequence(bad_layers, s, [3])
        with pytest.raises(ValueError):
            kv.compact_sequence(bad_layers, s, [0])
    for keep, err in (([1, 1], ValueError), ([3, 2], ValueError), ([0, 20], IndexError)):
        with pytest.raises(err):
            kv.compact_sequence(layers, mine, keep)
    assert mine.num_tokens() == 20


KEEPS = {
    "every other": lambda n: list(range(0, n, 2)),
    "a prefix": lambda n: list(range(40)),
    "all but the first": lambda n: list(range(1, n)),
    "sinks and a window": lambda n: [*range(BS), *range(n - 37, n)],
    "one": lambda n: [n - 1],
    "none": lambda n: [],
    "all": lambda n: list(range(n)),
}


@pytest.mark.parametrize("keep", KEEPS.values(), ids=KEEPS.keys())
def test_compaction_keeps_rows_in_order_and_frees_pages(keep):
    pool = kv.PhysicalBlockPool(64, BS)
    layers = storages(pool)
    gen = torch.Generator().manual_seed(2)
    seq = kv.SequenceState(7, pool)
    seq.append_tokens(9 * BS + 5)
    fill(layers, seq, 0, gen)
    twin = seq.fork_shared(8)  # keeps the old pages alive and must not change
    old = [cached(s, seq) for s in layers]
    rows = keep(seq.num_tokens())
    kv.compact_sequence(layers, seq, rows)
    assert seq.num_tokens() == len(rows) and seq.request_id() == 7 and seq.num_allocated_blocks() == -(-len(rows) // BS)
    for s, (k, v) in zip(layers, old):
        assert torch.equal(cached(s, twin)[0], k)
        if rows:
            gk, gv = cached(s, seq)
            assert torch.equal(gk, k[rows]) and torch.equal(gv, v[rows])
    del twin
    import gc

    gc.collect()
    assert pool.available() == 64 - seq.num_allocated_blocks()


def test_compaction_that_runs_out_of_pages_changes_nothing():
    pool = kv.PhysicalBlockPool(4, BS)
    layers = storages(pool, 1)
    seq = kv.SequenceState(1, pool)
    seq.append_tokens(3 * BS)
    with pytest.raises(kv.CapacityError):
        kv.compact_sequence(layers, seq, list(range(1, 3 * BS - 1)))
    assert seq.num_tokens() == 3 * BS and pool.available() == 1


def test_rotated_write_refuses_bad_arguments():
    pool = kv.PhysicalBlockPool(8, BS)
    s = storages(pool, 1)[0]
    table = kv.RotaryTable(100, HD)
    width = (QH + 2 * KVH) * HD
    qkv = torch.zeros(2, width, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(2, QH, HD, device="cuda")
    q, k, v = (qkv.data_ptr() + 2 * HD * x for x in (0, QH, QH + KVH))

    def call(q=q, k=k, v=v, sq=width, sk=width, sv=width, pos=(0, 1), slots=(3, 4), out=out, table=table, hq=QH, **kw):
        kv.write_paged_kv_rotated(s, table, q, k, v, sq, sk, sv, hq, list(pos), list(slots), out, **kw)

    call()
    call(pos=(), slots=(), k=None)
    for bad, err in ((dict(q=None), ValueError), (dict(k=None), ValueError), (dict(out=None), ValueError), (dict(sq=QH * HD - 1), ValueError),
                     (dict(sk=1), ValueError), (dict(pos=(0,)), ValueError), (dict(pos=(0, 100)), IndexError), (dict(slots=(3, 128)), IndexError),
                     (dict(slots=(3, 3)), ValueError), (dict(out=qkv), ValueError), (dict(out=s.key_base()), ValueError),
                     (dict(k=torch.zeros(2, width)), ValueError), (dict(query_weight=torch.zeros(HD)), ValueError),
                     (dict(table=kv.RotaryTable(10, 2 * HD)), ValueError), (dict(epsilon=-1.0), ValueError)):
        with pytest.raises(err):
            call(**bad)
    for args in ((0, HD), (10, 0), (10, 3)):
        with pytest.raises(ValueError):
            kv.RotaryTable(*args)
    with pytest.raises(ValueError):
        kv.RotaryTable(10, HD, 10000.0, 1.0, False, 99)


def test_shared_batch_checks_and_matches_the_plain_batch():
    pool = kv.PhysicalBlockPool(2048, BS)
    s = storages(pool, 1)[0]
    gen = torch.Generator().manual_seed(3)
    src = kv.SequenceState(1, pool)
    src.append_tokens(60 * BS)
    fill([s], src, 0, gen)
    lone = kv.SequenceState(50, pool)
    lone.append_tokens(33)
    fill([s], lone, 0, gen)
    seqs = [src, lone]
    for i in range(140):  # more groups than one launch takes: pairs of forks of prompts of their own
        if i % 2 == 0:
            prompt = kv.SequenceState(100 + i, pool)
            prompt.append_tokens(8 * BS)
            fill([s], prompt, 0, gen)
        c = prompt.fork_prefix(1000 + i, 8)
        c.append_tokens(1 + i % 5)
        fill([s], c, 8 * BS, gen)
        seqs.append(c)
    for i in range(3):
        c = src.fork_prefix(500 + i, 60)
        c.append_tokens(1 + 7 * i)
        fill([s], c, 60 * BS, gen)
        seqs.append(c)
    assert len(kv.plan_shared_prefixes(seqs)) > 2
    q = torch.randn(len(seqs), QH, HD, generator=gen)
    dq = q.cuda()
    out = torch.zeros(len(seqs), QH, HD, device="cuda")
    for _ in range(2):  # the second call finds its table on the device
        out.zero_()
        kv.paged_attention_batch_shared(s, seqs, dq, out, QH)
        got = out.cpu()
        for r, seq in enumerate(seqs):
            check_row(q[r], *cached(s, seq), got[r])
    kv.paged_attention_batch(s, seqs, dq, out, QH)
    plain = out.cpu()
    assert float((plain - got).abs().max()) < 1e-4
    kv.paged_attention_batch_shared(s, [], dq, out, QH)
    for bad in (lambda: kv.paged_attention_batch_shared(s, [src, None], dq, out, QH),
                lambda: kv.paged_attention_batch_shared(s, [src], dq, out, 3),
                lambda: kv.paged_attention_batch_shared(s, [src], dq, dq, QH),
                lambda: kv.paged_attention_batch_shared(s, [src], None, out, QH),
                lambda: kv.paged_attention_batch_shared(s, [kv.SequenceState(9, pool)], dq, out, QH)):
        with pytest.raises(ValueError):
            bad()


def test_a_serving_loop():
    pool = kv.PhysicalBlockPool(400, BS)
    layers = storages(pool)
    gen = torch.Generator().manual_seed(4)
    table = kv.RotaryTable(2000, HD)
    wq, wk = ((1 + 0.1 * torch.randn(HD, generator=gen)).cuda() for _ in range(2))
    width = (QH + 2 * KVH) * HD

    def step(layer, seqs, first):
        """Projections of positions first[i].. of each sequence through norm, rotation and write; their rotated Q."""
        writes = [(s, t) for s, f in zip(seqs, first) for t in range(f, s.num_tokens())]
        qkv = torch.randn(len(writes), width, generator=gen).bfloat16().cuda()
        out = torch.zeros(len(writes), QH, HD, device="cuda")
        p = qkv.data_ptr()
        kv.write_paged_kv_rotated(layer, table, p, p + 2 * QH * HD, p + 2 * (QH + KVH) * HD, width, width, width, QH,
                                  [t for _, t in writes], kv.build_slot_mapping(writes), out, wq, wk, 1e-5)
        # What was cached: the formula's K, rounded once, and V as given.
        x = qkv.cpu().double().view(len(writes), -1, HD)[:, QH:QH + KVH]
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * wk.cpu().double()
        angle = torch.tensor([t for _, t in writes]).double()[:, None] * 10000.0 ** (-torch.arange(0, HD, 2).double() / HD)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x[..., :HD // 2], x[..., HD // 2:]
        want = torch.cat([a * c - b * s, b * c + a * s], -1)
        size = torch.cat([a.abs() + b.abs()] * 2, -1)
        row = 0
        for sq, f in zip(seqs, first):
            n = sq.num_tokens() - f
            k, v = cached(layer, sq)
            # half a unit of bf16; FP32 roundings of norm, table and rotation as in test_gpu_rotary, one more for the table
            tol = want[row:row + n].abs() * 2.0**-8 + size[row:row + n] * (HD + 10) * 2.0**-23
            assert torch.all((k[f:].double() - want[row:row + n]).abs() <= tol)
            assert torch.equal(v[f:], qkv.cpu().view(len(writes), -1, HD)[row:row + n, QH + KVH:])
            row += n
        return out

    def decode(seqs):
        first = [s.num_tokens() for s in seqs]
        for s in seqs:
            s.append_token()
        for layer in layers:
            q = step(layer, seqs, first)
            o = torch.zeros_like(q)
            kv.paged_attention_batch_shared(layer, seqs, q, o, QH)
            for r, s in enumerate(seqs):
                check_row(q[r].cpu(), *cached(layer, s), o[r].cpu())

    prompt = kv.SequenceState(1, pool)
    prompt.append_tokens(20 * BS + 9)
    for layer in layers:
        step(layer, [prompt], [0])
    seqs = [prompt, *kv.fork_sequence(layers, prompt, list(range(2, 8)))]
    for _ in range(3):
        decode(seqs)
    assert kv.plan_shared_prefixes(seqs)[0].rows == 7
    # One request drops old tokens; the others' shared pages stay.
    kept = [*range(BS), *range(100, seqs[3].num_tokens())]
    before = [cached(layer, seqs[0])[0] for layer in layers]
    kv.compact_sequence(layers, seqs[3], kept)
    assert seqs[3].num_tokens() == len(kept)
    for layer, k in zip(layers, before):
        assert torch.equal(cached(layer, seqs[0])[0], k)
    for _ in range(2):
        decode(seqs)
    assert kv.device_status(0) == 0
