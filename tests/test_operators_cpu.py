"""The 8-bit cache, drafted trees and scored tokens without a GPU: masks, layouts, and every call that is refused before anything is launched."""
import ctypes as C
import types

import numpy as np
import pytest
import torch

from paligemma_multimodal_system_b200 import _lib, build, seq_ops
from paligemma_multimodal_system_b200.cache import KvSpec, SequenceStore

BAD = -1  # PG_ERR_ARG


@pytest.fixture(scope="module")
def library():
    build.build()
    return _lib.lib()


def test_masks_hold_a_token_and_its_path():
    parents = [-1, 0, 0, 1, 3, -1]
    masks, depth = seq_ops._tree_masks([parents, None], [6, 3])
    assert masks.shape == (9, 1) and depth.tolist() == [0, 1, 1, 2, 3, 0, 0, 1, 2]
    assert masks[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b11011, 0b100000, 0b1, 0b11, 0b111]


def test_masks_of_many_tokens_take_several_words():
    masks, depth = seq_ops._tree_masks([None], [70])
    assert masks.shape == (70, 3) and depth[-1] == 69
    assert masks[69].tolist() == [0xFFFFFFFF, 0xFFFFFFFF, 0x3F] and masks[32].tolist() == [0xFFFFFFFF, 1, 0]


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 2, 0], [-2], [-1, 0]])
def test_parents_come_first(parents):
    with pytest.raises(ValueError, match="parents"):
        seq_ops._tree_masks([parents], [len(parents) if parents != [-1, 0] else 3])


def test_packed_arguments_have_the_structs_sizes():
    assert _lib.ATTN_ROWS.size == 192 and _lib.PREPARE_E4M3.size == 192 and _lib.READ_E4M3.size == 112


def test_a_spec_with_heads_is_the_plain_one():
    assert KvSpec(128, 64, 2) == ("kv", 128, 64) and KvSpec(128, 64, 2)[0] == "kv" and KvSpec(128, 64, 2).heads == 2


def test_store_formats():
    store = SequenceStore([KvSpec(128, 64, 2), ("state", (3,)), None, ("latent", 40)], 200, 2, torch.bfloat16, device="cpu", kv_format="e4m3")
    k, v = store.k_pages[0], store.v_pages[0]
    assert k.codes.shape == (4, 64, 128) and k.powers.shape == (4, 2, 64) and v.codes.shape == (4, 64, 64) and (k.heads, k.size, v.size) == (2, 64, 32)
    assert store.k_pages[3].dtype == torch.bfloat16 and store.state[1].dtype == torch.float32 and store.k_pages[2] is None
    with pytest.raises(ValueError, match="unknown cache format"):
        SequenceStore([KvSpec(128, 64, 2)], 64, 1, torch.bfloat16, device="cpu", kv_format="int4")
    with pytest.raises(ValueError, match="how many heads"):
        SequenceStore([("kv", 128, 64)], 64, 1, torch.bfloat16, device="cpu", kv_format="e4m3")
    for spec in (KvSpec(48, 48, 2), KvSpec(512, 512, 2), KvSpec(64, 20, 1)):
        with pytest.raises(ValueError, match="multiple of 16"):
            SequenceStore([spec], 64, 1, torch.bfloat16, device="cpu", kv_format="e4m3")


def test_pages_that_do_not_belong_together():
    ok = seq_ops.QuantizedPages.empty(3, 64, 2, 32, device="cpu")
    assert (ok.pages, ok.page, ok.heads, ok.size) == (3, 64, 2, 32)
    u8 = torch.uint8
    for codes, powers in ((torch.zeros(3, 64, 64), torch.zeros(3, 2, 64, dtype=u8)), (torch.zeros(3, 64, 64, dtype=u8), torch.zeros(3, 64, 2, dtype=u8)),
                          (torch.zeros(3, 64, 64, dtype=u8), torch.zeros(2, 2, 64, dtype=u8)), (torch.zeros(3, 64, 63, dtype=u8), torch.zeros(3, 2, 64, dtype=u8)),
                          (torch.zeros(3, 64, 128, dtype=u8)[..., ::2], torch.zeros(3, 2, 64, dtype=u8)), (torch.zeros(64, 64, dtype=u8), torch.zeros(2, 64, dtype=u8))):
        with pytest.raises(ValueError):
            seq_ops.QuantizedPages(codes, powers)


def _batch(**more):
    b = types.SimpleNamespace(T=2, E=1, max_n=2, singles=0, max_single_ctx=0, dense_max_len=2, max_pages=1, tree=None, at=None)
    b.__dict__.update(more)
    return b


def test_attention_refuses_what_it_cannot_read():
    q, out = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 64, dtype=torch.bfloat16)
    pages, other = torch.zeros(1, 64, 32, dtype=torch.bfloat16), torch.zeros(1, 64, 32)
    k8 = seq_ops.QuantizedPages.empty(1, 64, 1, 32, device="cpu")
    call = lambda *a, **kw: seq_ops.attn_tree(*a, _batch(), 2, 1, 32, 32, 0.1, 0.0, 64, **kw)  # noqa: E731
    for args in ((q, other, other, None, out), (q, k8, pages, None, out), (q, pages, k8, None, out), (q, pages, pages, None, out.float()), (q.half(), pages.half(), pages.half(), None, out.half()),
                 (q, pages, pages, torch.zeros(2, 64), out), (q[:1], pages, pages, None, out), (q.t().contiguous().t(), pages, pages, None, out)):
        with pytest.raises(ValueError):
            call(*args)
    with pytest.raises(ValueError):
        seq_ops.attn_tree(q, k8, k8, None, out, _batch(), 4, 2, 16, 16, 0.1, 0.0, 64)  # one head in the pages, two asked for
    with pytest.raises(ValueError, match="masks"):
        seq_ops.attn_tree(q, pages, pages, None, out, _batch(tree=torch.zeros(3, 1, dtype=torch.int32)), 2, 1, 32, 32, 0.1, 0.0, 64)
    with pytest.raises(ValueError, match="one key row"):
        seq_ops.attn_ragged(q, pages, pages, None, out, _batch(tree=torch.zeros(2, 1, dtype=torch.int32)), 2, 1, 32, 32, 0.1, 0.0, 64, krow=32, vrow=32)
    with pytest.raises(ValueError, match="own width"):
        seq_ops.attn_ragged(q, k8, k8, None, out, _batch(singles=1), 2, 1, 32, 32, 0.1, 0.0, 64, krow=32, vrow=32)
    big = torch.zeros(1, 64, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="up to 128"):
        seq_ops.attn_tree(torch.zeros(2, 256, dtype=torch.bfloat16), big, big, None, torch.zeros(2, 256, dtype=torch.bfloat16), _batch(), 1, 1, 256, 256, 0.1, 0.0, 64)
    with pytest.raises(ValueError):
        seq_ops.kv_read(pages, pages, _batch(), torch.bfloat16)
    with pytest.raises(ValueError):
        seq_ops.kv_read(k8, k8, _batch(), torch.float16)


def test_scores_refuse_what_they_cannot_read():
    x, t = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="on the device"):
        seq_ops.token_logprobs(x, t)
    with pytest.raises(ValueError):
        seq_ops.token_logprobs(x.to(torch.bfloat16), t)


P = 0x1000  # an address that nothing reads: every call below is refused


def _rows(**kw):
    a = dict(q=P, k=P, v=P, kp=0, vp=0, gate=0, ldg=0, out=P, row0=P, n=P, ctx=P, pt=P, pos=P, tree=0, score=0, max_pages=4, page=64, words=0, entries=1, rows=1, max_n=1, busy=1, longest=10,
             singles=0, H=2, G=1, dim=64, vdim=64, f32=0, e4m3=0, gph=0, scale=1.0, cap=0.0)
    a.update(kw)
    return _lib.ATTN_ROWS.pack(*a.values())


@pytest.mark.parametrize("bad", [dict(entries=0), dict(entries=70000), dict(rows=0), dict(max_n=0), dict(max_n=70000), dict(H=3, G=2), dict(H=0), dict(G=0), dict(dim=0), dict(vdim=0), dict(max_pages=0),
                                 dict(longest=0), dict(page=16), dict(page=48), dict(page=96), dict(dim=136), dict(vdim=136), dict(dim=20), dict(vdim=12), dict(k=P + 8), dict(v=P + 4),
                                 dict(tree=P, words=0), dict(e4m3=1), dict(e4m3=1, kp=P, vp=P + 1), dict(e4m3=1, kp=P, vp=P, dim=24), dict(e4m3=1, kp=P, vp=P, vdim=24), dict(f32=1, dim=6)])
def test_attention_of_rows_is_refused_at_the_entry(library, bad):
    a = _rows(**bad)
    assert library.pg_attn_rows(a, 0, 0, 0) == BAD and library.pg_attn_rows_scratch(a) == BAD


def test_options_without_positions_are_refused(library):
    score = _lib.AttnScore(window=5)
    a = _rows(pos=0, score=C.addressof(score))
    assert library.pg_attn_rows(a, 0, 0, 0) == BAD
    half = _lib.AttnScore(dist_a=P)
    assert library.pg_attn_rows(_rows(score=C.addressof(half)), 0, 0, 0) == BAD
    assert library.pg_attn_rows(None, 0, 0, 0) == BAD


def test_scratch_is_asked_for_and_missed(library):
    """Few entries over long contexts join through scratch; without it, or with too little, the call is refused."""
    a = _rows(longest=100000, busy=1)
    need = library.pg_attn_rows_scratch(a)
    assert need >= 0
    if need:
        assert library.pg_attn_rows(a, 0, 0, 0) == BAD and library.pg_attn_rows(a, P, need - 4, 0) == BAD and library.pg_attn_rows(a, P + 4, need, 0) == BAD


@pytest.mark.parametrize("at,value", [(18, 0), (19, 0), (20, 0), (21, 20), (22, 272), (23, 7), (23, 66), (24, 3), (24, -1), (16, 0), (17, 0), (9, P + 8), (10, P + 8), (12, P + 2), (11, 0)])
def test_the_front_end_is_refused_at_the_entry(library, at, value):
    a = [P, 512, P, 0, P, P, P, 0, 0, P, P, P, P, P, 0, 0, 4, 64, 3, 2, 1, 64, 64, 32, 0, 0, 0, 0, 1e-6, 1.0, 0.0]
    a[at] = value
    if at == 24:
        a[24] = value
    assert library.pg_attn_prepare_e4m3(_lib.PREPARE_E4M3.pack(*a), 0) == BAD


@pytest.mark.parametrize("at,value", [(10, 0), (11, 0), (12, 0), (12, 70000), (13, 0), (14, 0), (15, 24), (16, 8), (0, P + 8), (2, P + 4), (8, P + 2), (9, P + 8)])
def test_the_read_back_is_refused_at_the_entry(library, at, value):
    a = [P, P, P, P, P, P, P, P, P, P, 4, 64, 1, 70, 2, 64, 64, 0]
    a[at] = value
    assert library.pg_kv_read_e4m3(_lib.READ_E4M3.pack(*a), 0) == BAD


@pytest.mark.parametrize("bad", [dict(rows=0), dict(V=0), dict(top=-1), dict(top=33), dict(top=11), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan")),
                                 dict(ld=9), dict(logits=0), dict(tokens=0), dict(out=0), dict(ids=0), dict(logits=P + 2)])
def test_scores_are_refused_at_the_entry(library, bad):
    a = dict(logits=P, ld=10, tokens=P, out=P, ids=P, rows=2, V=10, top=3, temperature=1.0)
    a.update(bad)
    assert library.pg_token_logprobs(a["logits"], a["ld"], a["tokens"], a["out"], P, P, a["ids"], P, a["rows"], a["V"], a["top"], a["temperature"], 0) == BAD
