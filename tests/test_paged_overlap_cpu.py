"""Outputs that lie over what the same launch reads are refused before anything runs. Device checks and the launch itself are put out of the way, so that a call gets as far on the CPU."""
import pytest
import torch

from muillm_amd import paged_ops

ROWS, HEADS, KV, DIM = 6, 4, 2, 64


@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(paged_ops, "_places", lambda kv, table, lengths, offsets, n_rows: (table.shape[0], table.shape[1], table.shape[1]))
    monkeypatch.setattr(paged_ops, "_call", lambda index, fn, args: calls.append(args) or 0)
    return calls


def append(q, k, v, out):
    kv = paged_ops.PagedKV.empty(8, KV, 64, DIM, "cpu")
    n = k.shape[0]
    return paged_ops.paged_append(q, k, v, kv, torch.zeros((n, 1), dtype=torch.int32), torch.ones(n, dtype=torch.int64), out=out)


def buffer(rows, heads):
    return torch.zeros((rows, heads, DIM), dtype=torch.float16)


@pytest.mark.parametrize("which", [0, 1])
def test_queries_over_keys_or_values_are_refused(launched, which):
    q = buffer(ROWS, HEADS)
    whole = torch.zeros(4 * ROWS * HEADS * DIM, dtype=torch.float16)
    out = whole[ROWS * HEADS * DIM:2 * ROWS * HEADS * DIM].view(ROWS, HEADS, DIM)
    size = ROWS * KV * DIM
    for at, bad in ((ROWS * HEADS * DIM - size, False), (ROWS * HEADS * DIM - size + 8, True), (ROWS * HEADS * DIM + 64, True), (2 * ROWS * HEADS * DIM - 8, True),
                    (2 * ROWS * HEADS * DIM, False)):
        mine = whole[at:at + size].view(ROWS, KV, DIM)
        kv = [buffer(ROWS, KV), buffer(ROWS, KV)]
        kv[which] = mine
        launched.clear()
        if bad:
            with pytest.raises(RuntimeError, match="lie over"):
                append(q, *kv, out)
            assert not launched
        else:
            assert append(q, *kv, out) is out and len(launched) == 1


def test_queries_in_place_whose_heads_are_keys_are_refused(launched):
    q = buffer(ROWS, HEADS)
    with pytest.raises(RuntimeError, match="lie over"):
        append(q, q[:, :KV], buffer(ROWS, KV), q)
    with pytest.raises(RuntimeError, match="lie over"):
        append(q, buffer(ROWS, KV), q[:, KV:2 * KV], q)
    assert not launched
    assert append(q, q[:, :KV], q[:, KV:2 * KV], None) is not q and len(launched) == 1


def test_one_tokens_projection_turned_in_place_is_not(launched):
    proj = torch.zeros((1, (HEADS + 2 * KV) * DIM), dtype=torch.float16)
    q, k, v = (x.unflatten(1, (-1, DIM)) for x in proj.split([HEADS * DIM, KV * DIM, KV * DIM], 1))
    assert append(q, k, v, q) is q and len(launched) == 1
    k = proj[:, (HEADS - 1) * DIM:(HEADS + 1) * DIM].unflatten(1, (-1, DIM))
    with pytest.raises(RuntimeError, match="lie over"):
        append(q, k, v, q)


def test_strided_keys_end_where_their_last_head_does(launched):
    rest = torch.zeros(ROWS * (KV + 1) * DIM + ROWS * HEADS * DIM, dtype=torch.float16)
    k = rest[:ROWS * (KV + 1) * DIM].view(ROWS, KV + 1, DIM)[:, :KV]
    out = rest[ROWS * (KV + 1) * DIM - DIM:][:ROWS * HEADS * DIM].view(ROWS, HEADS, DIM)
    assert append(buffer(ROWS, HEADS), k, buffer(ROWS, KV), out) is out
    out = rest[ROWS * (KV + 1) * DIM - DIM - 8:][:ROWS * HEADS * DIM].view(ROWS, HEADS, DIM)
    with pytest.raises(RuntimeError, match="lie over"):
        append(buffer(ROWS, HEADS), k, buffer(ROWS, KV), out)


def test_attention_over_its_queries_is_refused_still(launched):
    kv = paged_ops.PagedKV.empty(8, KV, 64, DIM, "cpu")
    q = buffer(2, HEADS)
    with pytest.raises(RuntimeError, match="lie over"):
        paged_ops.paged_attention(q, kv, torch.zeros((2, 1), dtype=torch.int32), torch.ones(2, dtype=torch.int64), out=q)
    assert not launched
