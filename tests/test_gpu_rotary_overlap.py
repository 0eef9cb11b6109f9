"""write_paged_kv_rotated refuses inputs inside the cache it writes, and a Q
output over anything it reads; a refused call leaves the cache as it was."""
import pytest
import torch

import kvflux_b200 as kv

pytestmark = pytest.mark.gpu

KVH, QH, HD, BS, N = 2, 4, 64, 16, 3


@pytest.fixture
def setup(cuda):
    pool = kv.PhysicalBlockPool(8, BS)
    storage = kv.PagedKVStorage(pool, KVH, HD, kv.DType.BFloat16, 0)
    seq = kv.SequenceState(1, pool)
    seq.append_tokens(5 * BS)
    k, v = (torch.randn(5 * BS, KVH, HD, device="cuda").bfloat16() for _ in range(2))
    kv.write_paged_kv(storage, k, v, kv.build_slot_mapping([(seq, t) for t in range(5 * BS)]))
    return storage, seq, k, v


@pytest.mark.parametrize("inside", ["query", "key", "value", "query_weight", "key_weight", "out"])
@pytest.mark.parametrize("where", ["first", "last"])
def test_nothing_lies_in_the_cache(setup, inside, where):
    storage, seq, k, v = setup
    width = (QH + 2 * KVH) * HD
    qkv = torch.randn(N, width, device="cuda").bfloat16()
    q = qkv.data_ptr()
    a = dict(query=q, key=q + 2 * QH * HD, value=q + 2 * (QH + KVH) * HD, query_weight=torch.ones(HD, device="cuda"),
             key_weight=torch.ones(HD, device="cuda"), out=torch.zeros(N, QH, HD, device="cuda"))
    end = storage.key_base() + storage.layout().total_bytes()
    span = {"query_weight": 4 * HD, "key_weight": 4 * HD, "out": 4 * N * QH * HD}.get(inside, 2 * ((N - 1) * width + (QH if inside == "query" else KVH) * HD))
    a[inside] = storage.key_base() if where == "first" else end - span
    table = kv.RotaryTable(10, HD)
    with pytest.raises(ValueError):
        kv.write_paged_kv_rotated(storage, table, a["query"], a["key"], a["value"], width, width, width, QH, [0, 1, 2], [0, 17, 34], a["out"],
                                  query_weight=a["query_weight"], key_weight=a["key_weight"])
    got = [torch.empty_like(x) for x in (k, v)]
    kv.read_paged_kv(storage, seq, *got)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)


@pytest.mark.parametrize("over", ["query_weight", "key_weight", "table"])
def test_the_q_output_lies_over_no_input(setup, over):
    storage = setup[0]
    width = (QH + 2 * KVH) * HD
    qkv = torch.randn(N, width, device="cuda").bfloat16()
    q = qkv.data_ptr()
    table = kv.RotaryTable(100, HD)
    room = torch.ones(2 * HD + N * QH * HD, device="cuda")
    w = {"query_weight": room[:HD], "key_weight": room[HD:2 * HD]}
    out = table.device_table() if over == "table" else w[over]
    with pytest.raises(ValueError):
        kv.write_paged_kv_rotated(storage, table, q, q + 2 * QH * HD, q + 2 * (QH + KVH) * HD, width, width, width, QH, [0, 1, 2], [0, 17, 34], out,
                                  query_weight=w["query_weight"], key_weight=w["key_weight"])
    # Behind them there is room.
    kv.write_paged_kv_rotated(storage, table, q, q + 2 * QH * HD, q + 2 * (QH + KVH) * HD, width, width, width, QH, [0, 1, 2], [0, 17, 34],
                              room[2 * HD:], query_weight=w["query_weight"], key_weight=w["key_weight"])
    assert kv.device_status(0) == 0
