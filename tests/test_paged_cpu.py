"""The paged cache and its operators without a GPU: layouts, and calls that are refused before anything runs."""
import re

import pytest
import torch

from muillm_amd import _lib, muillm_ext, paged_ops

ARG, UNSUPPORTED, ALIGNMENT = -1, -2, -4
P = 4096  # an aligned address that no refused call touches


def append_args(**kw):
    a = dict(stream=None, dtype=0, q=P, qt=512, qh=128, k=P, kt=512, kh=128, v=P, vt=512, vh=128, kp=P, vp=P, ks=P, vs=P, n_pages=4, page=64, table=P, stride=2, pages=2,
             lengths=P, offsets=None, positions=None, inv_freq=P, rot=128, interleaved=0, factor=1.0, q_out=P, rows=2, requests=2, most=1, heads=4, kv_heads=2, dim=128)
    a.update(kw)
    order = "q k v kp vp ks vs table lengths offsets positions inv_freq q_out qt qh kt kh vt vh stride dtype n_pages page pages rows requests most heads kv_heads dim rot interleaved factor"
    return [a["stream"], _lib.PAGED_APPEND_ARGS.pack(*(a[x] or 0 for x in order.split()))]


@pytest.mark.parametrize("change,status", [
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(kp=None), ARG), (dict(vs=None), ARG), (dict(table=None), ARG), (dict(lengths=None), ARG), (dict(q_out=None), ARG),
    (dict(n_pages=0), ARG), (dict(pages=0), ARG), (dict(stride=1), ARG), (dict(rows=0), ARG), (dict(requests=0), ARG), (dict(most=0), ARG), (dict(kv_heads=0), ARG),
    (dict(heads=0), ARG), (dict(rot=-16), ARG), (dict(rot=144), ARG), (dict(inv_freq=None), ARG), (dict(rows=3), ARG), (dict(dtype=2), ARG), (dict(dtype=7), ARG),
    (dict(page=32), UNSUPPORTED), (dict(page=96), UNSUPPORTED), (dict(pages=1 << 25, stride=1 << 25), UNSUPPORTED), (dict(page=512), UNSUPPORTED), (dict(dim=96, rot=64), UNSUPPORTED), (dict(rot=8), UNSUPPORTED),
    (dict(q=P + 2), ALIGNMENT), (dict(k=P + 8), ALIGNMENT), (dict(vp=P + 4), ALIGNMENT), (dict(kt=508), ALIGNMENT), (dict(vh=132), ALIGNMENT), (dict(qt=1), ALIGNMENT),
])
def test_append_refusals(change, status):
    assert _lib.load().mui_paged_append(*append_args(**change)) == status


def attention_args(**kw):
    a = dict(stream=None, dtype=0, q=P, qt=512, qh=128, kp=P, vp=P, ks=P, vs=P, n_pages=4, page=64, table=P, stride=2, pages=2, lengths=P, offsets=None, scale=0.1, window=0,
             keep=0, most=1, longest=128, scratch=None, nbytes=0, out=P, rows=2, requests=2, heads=4, kv_heads=2, dim=128)
    a.update(kw)
    order = "q kp vp ks vs table lengths offsets scratch out nbytes qt qh stride dtype n_pages page pages rows requests most longest window keep heads kv_heads dim scale"
    return [a["stream"], _lib.PAGED_ATTENTION_ARGS.pack(*(a[x] or 0 for x in order.split()))]


@pytest.mark.parametrize("change,status", [
    (dict(q=None), ARG), (dict(kp=None), ARG), (dict(vp=None), ARG), (dict(ks=None), ARG), (dict(table=None), ARG), (dict(lengths=None), ARG), (dict(out=None), ARG),
    (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=float("nan")), ARG), (dict(window=-1), ARG), (dict(keep=-1), ARG), (dict(most=0), ARG),
    (dict(longest=0), ARG), (dict(heads=5), ARG), (dict(heads=0), ARG), (dict(rows=0), ARG), (dict(rows=3), ARG), (dict(stride=1), ARG), (dict(dtype=2), ARG),
    (dict(page=16), UNSUPPORTED), (dict(dim=192), UNSUPPORTED), (dict(pages=1 << 25, stride=1 << 25), UNSUPPORTED), (dict(requests=70000, rows=70000), UNSUPPORTED),
    (dict(q=P + 4), ALIGNMENT), (dict(out=P + 8), ALIGNMENT), (dict(kp=P + 1), ALIGNMENT), (dict(qh=4), ALIGNMENT),
    (dict(pages=2000, stride=2000, longest=100000), ARG),  # needs scratch and has none
])
def test_attention_refusals(change, status):
    assert _lib.load().mui_paged_attention(*attention_args(**change)) == status


def test_scratch_of_bad_sizes_is_nothing():
    lib = _lib.load()
    assert lib.mui_paged_attention_scratch_bytes(0, 1, 1, 100, 0, 0, 4, 2, 128) == 0
    assert lib.mui_paged_attention_scratch_bytes(1, 1, 1, 100, 0, 0, 3, 2, 128) == 0
    assert lib.mui_paged_attention_scratch_bytes(1, 1, 1, 0x7fffffff, 0, 0, 4, 2, 128) > 0


def sampling_args(**kw):
    a = dict(row_stream=None, dtype=0, logits=P, stride=100000, rows=2, vocab=100000, u=P, ts=None, t=1.0, ks=None, k=0, ps=None, p=1.0, ms=None, m=0.0, token=P, probability=None,
             ws=P, nbytes=1 << 40)
    a.update(kw)
    order = "logits u ts ks ps ms token probability ws nbytes stride dtype rows vocab k t p m"
    return [a["row_stream"], _lib.SAMPLE_FILTERED_ARGS.pack(*(a[x] or 0 for x in order.split()))]


@pytest.mark.parametrize("change,status", [
    (dict(logits=None), ARG), (dict(u=None), ARG), (dict(token=None), ARG), (dict(ws=None), ARG), (dict(rows=0), ARG), (dict(vocab=0), ARG), (dict(stride=99999), ARG),
    (dict(dtype=2), ARG), (dict(nbytes=1000), ARG), (dict(rows=70000), UNSUPPORTED), (dict(vocab=0x7fffffff, stride=0x7fffffff), UNSUPPORTED), (dict(ws=P + 8), ALIGNMENT),
])
def test_sampling_refusals(change, status):
    assert _lib.load().mui_sample_filtered(*sampling_args(**change)) == status


def test_workspace_grows_with_rows_and_parts():
    lib = _lib.load()
    assert lib.mui_sample_filtered_workspace_bytes(0, 10) == 0 and lib.mui_sample_filtered_workspace_bytes(1, 0) == 0
    assert lib.mui_sample_filtered_workspace_bytes(256, 1000) == 0  # (one workgroup's counts stay with it)
    one = lib.mui_sample_filtered_workspace_bytes(256, 100000)
    assert one > 0 and lib.mui_sample_filtered_workspace_bytes(512, 100000) == 2 * one
    assert lib.mui_sample_filtered_workspace_bytes(256, 400000) >= 3 * one


def cpu_cache(page=64, dim=128, kv_heads=2, n=3):
    return paged_ops.PagedKV.empty(n, kv_heads, page, dim, "cpu")


def test_empty_pages_and_dense():
    kv = cpu_cache()
    assert (kv.n_pages, kv.kv_heads, kv.page, kv.dim) == (3, 2, 64, 128)
    kv.k.view(torch.uint8)[1, 0, 0, 1, 5, 7] = 0x38      # 1.0: token 5, dimension 71
    kv.v.view(torch.uint8)[1, 1, 0, 9, 2, 3, 1] = 0x40   # 2.0: token 16 * 3 + 4 * 2 + 1, dimension 9
    kv.k_scale[1, 0], kv.v_scale[1, 1] = 0.5, 4.0
    k, v = kv.dense(torch.tensor([2, 1], dtype=torch.int32), 128)
    assert k.shape == v.shape == (2, 128, 128)
    assert float(k[0, 64 + 5, 71]) == 0.5 and float(k.abs().sum()) == 0.5
    assert float(v[1, 64 + 57, 9]) == 8.0 and float(v.abs().sum()) == 8.0


def test_cache_refuses_other_shapes_and_types():
    kv = cpu_cache()
    for bad in (lambda: paged_ops.PagedKV(kv.v, kv.k, kv.k_scale, kv.v_scale), lambda: paged_ops.PagedKV(kv.k[:2], kv.v, kv.k_scale, kv.v_scale),
                lambda: paged_ops.PagedKV(kv.k.view(torch.uint8), kv.v, kv.k_scale, kv.v_scale), lambda: paged_ops.PagedKV(kv.k, kv.v, kv.k_scale[:2], kv.v_scale),
                lambda: paged_ops.PagedKV(kv.k, kv.v, kv.k_scale, kv.v_scale.double()), lambda: paged_ops.PagedKV.empty(2, 2, 32, 128, "cpu"),
                lambda: paged_ops.PagedKV.empty(2, 2, 64, 96, "cpu"), lambda: paged_ops.PagedKV(kv.k[:, ::2], kv.v[:, ::2], kv.k_scale[:, ::2], kv.v_scale[:, ::2])):
        with pytest.raises(RuntimeError):
            bad()


def test_tensors_of_the_cpu_are_refused():
    kv = cpu_cache()
    x = torch.zeros((2, 2, 128), dtype=torch.float16)
    table, lengths = torch.zeros((2, 1), dtype=torch.int32), torch.ones(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_ops.paged_append(None, x, x, kv, table, lengths)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_ops.paged_attention(x, kv, table, lengths)
    with pytest.raises(RuntimeError, match="CUDA"):
        muillm_ext.mui_sample_filtered(torch.zeros((1, 10), dtype=torch.float16), torch.zeros(1))


@pytest.mark.parametrize("dim,heads", [(64, 8), (128, 8), (128, 4), (256, 2)])
def test_a_bound_above_the_rows_asks_for_no_more(dim, heads):
    lib = _lib.load()
    for rows in (1, 7, 40, 200):
        one = lib.mui_paged_attention_scratch_bytes(rows, 4, rows, 5000, 0, 0, heads, 2, dim)
        assert one == lib.mui_paged_attention_scratch_bytes(rows, 4, 0x7fffffff, 5000, 0, 0, heads, 2, dim) < 1 << 30


def test_the_packed_arguments_are_the_headers_structs():
    """Numbers of members of each kind, in the header's order: pointers, sizes, longs, ints, floats."""
    kinds = [("P", r"\*"), ("N", r"^size_t "), ("l", r"^long "), ("i", r"^int "), ("f", r"^float ")]
    for name, packed in (("mui_paged_append_args", _lib.PAGED_APPEND_ARGS), ("mui_paged_attention_args", _lib.PAGED_ATTENTION_ARGS),
                         ("mui_sample_filtered_args", _lib.SAMPLE_FILTERED_ARGS)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, _lib.header_text(), flags=re.S).group(1)
        found = ""
        for member in body.split(";"):
            if member.strip():
                kind = next(k for k, pattern in kinds if re.search(pattern, member.strip()))
                found += kind * (member.count(",") + 1)
        expanded = re.sub(r"(\d*)([A-Za-z])", lambda m: m.group(2) * int(m.group(1) or 1), packed.format)
        assert found == expanded, name
        assert packed.size % 8 == 0


def test_no_arguments_are_refused():
    lib = _lib.load()
    assert lib.mui_paged_append(None, None) == lib.mui_paged_attention(None, None) == lib.mui_sample_filtered(None, None) == ARG
