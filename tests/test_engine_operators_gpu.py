"""The 8-bit cache, drafted trees and scored tokens as the ragged-step engine uses them together.

Sequential runs and trees differ in kernels, not in arithmetic: fp32 models agree to rounding (sums of a few thousand terms through a handful of layers: 2e-4 of the logits'
root mean square, the bound that the model's own tests use), bf16 ones to the rounding of activations (4e-2).  Over the 8-bit cache a key or value that lies within rounding of a
border may take either of two codes, 2^-3 of the element apart at most: some elements in a hundred thousand, 2e-3 of the logits in fp32."""
import os

import pytest
import torch

from oracle import mapedra_oracle as O
from test_mapedra_gpu import attn_layer, build, light_layer, make_cfg, run_cut, toks

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 2e-4, torch.bfloat16: 4e-2}

ATTENTION = make_cfg([attn_layer(heads=4, kv_heads=2, dim=64, vdim=64, rot=32, ff=96), attn_layer(heads=8, kv_heads=1, dim=32, vdim=64, rot=16, ff=0),
                      attn_layer(heads=2, kv_heads=2, dim=128, vdim=128, rot=64, ff=64)], width=96, vocab=80, side=8)
MIXED = make_cfg([attn_layer(heads=4, kv_heads=2, dim=64, vdim=64, rot=32, ff=96), light_layer(), attn_layer(heads=4, kv_heads=1, dim=32, vdim=48, rot=16, ff=64)], width=96, vocab=80)


def rel_err(got, ref):
    got, ref = got.double().cpu(), ref.double().cpu()
    return float((got - ref).pow(2).mean().sqrt() / ref.pow(2).mean().sqrt())


def engine(cfg, dtype, kv_format=None, seed=3, max_tokens=2048, slots=4):
    from paligemma_multimodal_system_b200.engine import SequenceEngine
    return SequenceEngine(build(cfg, O.random_weights(cfg, seed=seed), dtype), max_tokens, slots, kv_format=kv_format)


def paths_of(parents):
    """Every node's path from its root."""
    out = []
    for i, up in enumerate(parents):
        out.append((out[up] if up >= 0 else []) + [i])
    return out


@pytest.mark.parametrize("kv_format", [None, "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("context", [1, 61, 200])
def test_a_drafted_tree_gives_every_paths_logits(dtype, kv_format, context):
    parents = [-1, 0, 0, 1, 2, 2, -1, 6, 5]
    prompt, other, drafts = toks(context, 80, 1), toks(17, 80, 2), toks(len(parents), 80, 3)
    eng = engine(ATTENTION, dtype, kv_format)
    eng.step([("a", prompt, []), ("b", other, [])])
    got = eng.step_drafts([("b", drafts[:4], [-1, 0, 1, 1]), ("a", drafts, parents)])
    assert got.shape == (4 + len(parents), 80) and eng.store.live["a"].length == context
    ref = engine(ATTENTION, dtype, kv_format)
    tol = TOL[dtype] if kv_format is None or dtype == torch.bfloat16 else 2e-3
    for first, pr, ups, ds in ((0, other, [-1, 0, 1, 1], drafts[:4]), (4, prompt, parents, drafts)):
        for i, path in enumerate(paths_of(ups)):
            full = pr + [ds[j] for j in path]
            want = run_cut(ref, ("x", first, i), full, [len(pr), 1])[-1:]
            assert rel_err(got[first + i:first + i + 1], want) < tol, (first, i)


@pytest.mark.parametrize("kv_format", [None, "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("path", [[], [0], [0, 2, 5, 8], [6, 7]])
def test_accepted_paths_go_on_as_if_they_had_been_fed(dtype, kv_format, path):
    parents = [-1, 0, 0, 1, 2, 2, -1, 6, 5]
    prompt, drafts, later = toks(125, 80, 1), toks(len(parents), 80, 3), toks(70, 80, 4)  # (the rows cross the border at 128)
    eng, ref = engine(ATTENTION, dtype, kv_format), engine(ATTENTION, dtype, kv_format)
    eng.step([("a", prompt, [])])
    eng.step_drafts([("a", drafts, parents)])
    eng.accept("a", path)
    assert eng.store.live["a"].length == 125 + len(path)
    got = run_cut(eng, "a", later, [1, 30, 1])
    want = run_cut(ref, "a", prompt + [drafts[i] for i in path] + later, [125] + [1] * (len(path) + 1) + [30, 1])[125 + len(path):]
    assert rel_err(got, want) < (TOL[dtype] if kv_format is None or dtype == torch.bfloat16 else 2e-3)
    assert not eng._drafted


def test_drafts_are_refused_where_they_cannot_be():
    eng = engine(ATTENTION, torch.float32)
    eng.step([("a", [1, 2, 3], [])])
    for bad in ([("zz", [1], [-1])], [("a", [], [])], [("a", [1, 2], [-1])], [("a", [1, 2], [-1, 1])], [("a", [1], [-2])], [("a", [99], [-1])], [("a", [1], [-1]), ("a", [1], [-1])], []):
        with pytest.raises((KeyError, ValueError, IndexError)):
            eng.step_drafts(bad)
    with pytest.raises(KeyError):
        eng.accept("a", [])
    eng.step_drafts([("a", [5, 6, 7], [-1, 0, 0])])
    for bad in ([1], [0, 0], [0, 1, 2], [3], [-1]):
        with pytest.raises(ValueError):
            eng.accept("a", bad)
    eng.step([("a", [4], [])])  # the request went on without them
    with pytest.raises(KeyError):
        eng.accept("a", [0])
    with pytest.raises(ValueError, match="no branches"):
        e = engine(MIXED, torch.float32)
        e.step([("a", [1], [])])
        e.step_drafts([("a", [1], [-1])])


@pytest.mark.parametrize("cfg", [ATTENTION, MIXED])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_8_bit_cache_does_not_depend_on_the_cut(cfg, dtype):
    """Whole prompts, portions and single tokens (prompt attention over rows read back, decode attention over the codes, a replayed graph) see the same cache."""
    tk = toks(150, 80, 6)
    eng = engine(cfg, dtype, "e4m3")
    whole = run_cut(eng, "a", tk, [150])
    for cuts in ([1], [64, 1, 40, 1], [70, 80]):
        assert rel_err(run_cut(eng, "a", tk, cuts), whole) < (2e-3 if dtype == torch.float32 else TOL[dtype]), cuts
    plain = run_cut(engine(cfg, dtype), "a", tk, [150])
    assert 1e-4 < rel_err(whole, plain) < 0.15  # elements are off by 2^-4 at most, sums over keys and sizes by less


def test_the_8_bit_cache_takes_half_the_memory():
    eng, plain = engine(ATTENTION, torch.bfloat16, "e4m3"), engine(ATTENTION, torch.bfloat16)
    held = sum(p.codes.nbytes + p.powers.nbytes for p in eng.store.k_pages + eng.store.v_pages)
    assert held < 0.53 * sum(p.nbytes for p in plain.store.k_pages + plain.store.v_pages)


@pytest.mark.parametrize("kv_format", [None, "e4m3"])
def test_other_models_over_the_8_bit_cache(kv_format):
    """Windows, sinks, distance penalties, borrowed keys, logistic weights: the layers of the other decoders take the same pages."""
    from paligemma_multimodal_system_b200.cache import SequenceStore
    from paligemma_multimodal_system_b200.mixers import WindowedSoftmaxAttention
    from paligemma_multimodal_system_b200.seq_ops import Precision, make_step_batch
    g = torch.Generator().manual_seed(4)
    D, T = 64, 90

    def run(mx, cuts, dtype, fmt, h):
        store = SequenceStore(mx.cache_specs(), 256, 1, dtype, kv_format=fmt)
        rec, out, at, prec = store.admit("a"), [], 0, Precision(dtype)
        for n in cuts:
            store.reserve("a", n)
            b = make_step_batch([dict(tokens=[0] * n, ctx=at, slot=rec.slot, pages=rec.pages)])
            out.append(mx(h[at:at + n].contiguous(), b, store, 0, prec))
            store.commit("a", n)
            at += n
        return torch.cat(out)

    for make in (lambda: WindowedSoftmaxAttention(D, 4, 2, 32, 32, 0.2, 1e-5, window=20, keep_first=3, sink=True, rot_dims=16, qk_norm=True),
                 lambda: WindowedSoftmaxAttention(D, 4, 2, 32, 32, 0.2, 1e-5, distance_penalty=True, temperature=True, head_gate=True),
                 lambda: WindowedSoftmaxAttention(D, 2, 2, 48, 48, 0.2, 1e-5, value_is_key=True, unit_sink=True, rot_dims=48)):
        mx = make()
        tensors = {}

        def take(name, shape):
            return tensors.setdefault(name, torch.rand(shape, generator=g) + 0.1 if name in ("r1", "r2", "temp", "sink") else torch.randn(shape, generator=g) * (shape[-1] ** -0.5 if shape else 1))

        mx.load(take, "")
        mx.pack(Precision(torch.float32))
        h = torch.randn(T, D, generator=g).cuda()
        whole = run(mx, [T], torch.float32, kv_format, h)
        assert rel_err(run(mx, [1] * T, torch.float32, kv_format, h), whole) < 2e-3
        assert rel_err(run(mx, [50, 1, 39], torch.float32, kv_format, h), whole) < 2e-3


def test_generated_tokens_come_with_their_log_probabilities():
    for dtype in (torch.float32, torch.bfloat16):
        eng = engine(MIXED, dtype)
        prompts = [toks(9, 80, 1), toks(30, 80, 2), toks(3, 80, 3)]
        plain = eng.generate(prompts, 6)
        tokens, said = eng.generate(prompts, 6, logprobs=4)
        assert tokens == plain and [len(r) for r in said] == [len(t) for t in tokens]
        for pr, ts, rs in zip(prompts, tokens, said):
            seq = pr + ts
            logits = run_cut(eng, "x", seq[:-1], [len(pr)] + [1] * len(ts))[len(pr) - 1:].double().cpu()
            want = torch.log_softmax(logits, -1)
            for i, (t, r) in enumerate(zip(ts, rs)):
                assert r["rank"] == 0 and r["top"][0][0] == t and len(r["top"]) == 4
                assert abs(r["logprob"] - float(want[i, t])) < 10 * TOL[dtype] and r["top"][0][1] == r["logprob"]
                assert abs(r["entropy"] + float((want[i].exp() * want[i]).sum())) < 10 * TOL[dtype]
                assert all(a[1] >= b[1] for a, b in zip(r["top"], r["top"][1:]))
        sampled, said = eng.generate(prompts, 5, do_sample=True, temperature=0.7, top_p=0.9, seed=5, logprobs=0)
        assert [len(r) for r in said] == [len(t) for t in sampled] and all(not r["top"] and r["logprob"] <= 0 for rs in said for r in rs)


@pytest.mark.parametrize("step_tokens", [1, 7, 512])
def test_scored_prompts(step_tokens):
    eng = engine(MIXED, torch.float32)
    prompts = [toks(25, 80, 1), [5], toks(2, 80, 2), toks(70, 80, 3)]
    got = eng.score(prompts, top=3, step_tokens=step_tokens)
    assert [len(r) for r in got] == [24, 0, 1, 69] and not eng.store.live
    for pr, rs in zip(prompts, got):
        if len(pr) == 1:
            continue
        logs = torch.log_softmax(run_cut(eng, "x", pr[:-1], [len(pr) - 1]).double().cpu(), -1)
        for i, r in enumerate(rs):
            order = torch.sort(logs[i], descending=True, stable=True)
            assert abs(r["logprob"] - float(logs[i, pr[i + 1]])) < 2e-3
            assert [v for _, v in r["top"]] == pytest.approx(order.values[:3].tolist(), abs=2e-3)
    with pytest.raises(IndexError):
        eng.score([[80]])


def test_a_run_of_them_together():
    """Greedy decoding with drafted trees over the 8-bit cache: tokens whose drafts agree with the model's own choice are kept, their scores come from the same logits; the
    tokens are those of decoding one by one."""
    from paligemma_multimodal_system_b200 import seq_ops
    prompt = toks(40, 80, 9)
    one = engine(ATTENTION, torch.float32, "e4m3")
    want = one.generate([prompt], 24)[0]
    eng = engine(ATTENTION, torch.float32, "e4m3")
    last = int(eng.step([("a", prompt, [len(prompt) - 1])]).argmax())
    got, steps, r = [last], 0, torch.Generator().manual_seed(1)
    while len(got) < 24:
        # the first draft is the token that was chosen last; below it guesses, one of them right every other time
        at = len(got)
        right = want[at:at + 2] if steps % 2 == 0 else []
        drafts, parents = [got[-1]], [-1]
        for t in right:
            drafts += [int(torch.randint(0, 80, (1,), generator=r)), t]
            up = len(drafts) - 4 if len(drafts) > 3 else 0
            parents += [max(up, 0) if len(parents) == 1 else len(drafts) - 3, max(up, 0) if len(parents) == 1 else len(drafts) - 3]
        logits = eng.step_drafts([("a", drafts, parents)])
        best = logits.argmax(-1).to(torch.int32)
        lp, _, rank, _, _ = seq_ops.token_logprobs(logits, best, top=1)
        assert (rank == 0).all() and torch.isfinite(lp).all()
        node, path, best = 0, [0], best.tolist()
        while True:
            got.append(best[node])
            below = [i for i, p in enumerate(parents) if p == node and drafts[i] == best[node]]
            if not below or len(got) >= 24:
                break
            node = below[0]
            path.append(node)
        eng.accept("a", path)
        steps += 1
    assert got == want and steps < 23


def test_the_command_prints_them(tmp_path, capsys):
    import json
    from safetensors.torch import save_file
    from paligemma_multimodal_system_b200.inference import generate_token_ids
    w = O.random_weights(MIXED, seed=3)
    os.makedirs(tmp_path, exist_ok=True)
    with open(tmp_path / "config.json", "w") as f:
        json.dump(MIXED, f)
    save_file({k: v.to(torch.bfloat16).contiguous() for k, v in w.items()}, str(tmp_path / "model.safetensors"))
    tokens, said = generate_token_ids(str(tmp_path), "5 17 3; 8 9", 4, 0.8, 0.9, False, dtype="float32", logprobs=2, kv_format="e4m3")
    text = capsys.readouterr().out
    assert [len(t) for t in tokens] == [4, 4] and text.count("logprob") == 8 and len(said[0][0]["top"]) == 2
    assert generate_token_ids(str(tmp_path), "5 17 3; 8 9", 4, 0.8, 0.9, False, dtype="float32", kv_format="e4m3") == tokens


def test_a_step_that_fails_leaves_no_drafts(monkeypatch):
    eng = engine(ATTENTION, torch.float32)
    eng.step([("a", toks(70, 80, 1), [])])
    first = eng.step_drafts([("a", [3, 4], [-1, 0])])
    with monkeypatch.context() as m:
        m.setattr(eng.model, "step", lambda *a: (_ for _ in ()).throw(RuntimeError("no step")))
        with pytest.raises(RuntimeError):
            eng.step_drafts([("a", [5, 6, 7], [-1, 0, 1])])
    with pytest.raises(KeyError):  # (the first drafts' rows may be written over)
        eng.accept("a", [0])
    assert torch.equal(eng.step_drafts([("a", [3, 4], [-1, 0])]), first)


@pytest.mark.parametrize("count", [-1, 33, 81])
def test_counts_of_alternatives_are_refused_before_anything_runs(count):
    eng = engine(ATTENTION, torch.float32)
    with pytest.raises(ValueError):
        eng.generate([[1, 2, 3]], 4, logprobs=count)
    with pytest.raises(ValueError):
        eng.score([[1, 2, 3]], top=count)
    assert not eng.store.live
