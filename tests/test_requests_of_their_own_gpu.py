"""What requests of the ragged-step engine have of their own: forks over shared pages, adapters, drafted tokens that are judged.  Bounds as in test_engine_operators_gpu.py: kernels of other
shapes add in another order, 2e-4 of the logits' root mean square in fp32, 4e-2 in bf16."""
import json
import os

import pytest
import torch

from oracle import kovusun_oracle as KO
from oracle import mapedra_oracle as O
from test_engine_operators_gpu import ATTENTION, MIXED, TOL, engine, rel_err
from test_mapedra_gpu import run_cut, toks

pytestmark = pytest.mark.gpu


def build(cfg, w, dtype):
    """Weights as they are: merged ones are not bf16's."""
    from paligemma_multimodal_system_b200.modeling_kovusun import KovusunConfig, KovusunForCausalLM
    from paligemma_multimodal_system_b200.modeling_mapedra import MapedraConfig, MapedraForCausalLM
    if cfg["architecture"] == "Kovusun":
        return KovusunForCausalLM(KovusunConfig(cfg), dtype).load_weights(w)
    return MapedraForCausalLM(MapedraConfig(cfg), dtype).load_weights(w)


@pytest.mark.parametrize("cfg", [ATTENTION, MIXED])
@pytest.mark.parametrize("dtype,kv_format", [(torch.float32, None), (torch.bfloat16, None), (torch.float32, "e4m3")])
@pytest.mark.parametrize("context", [5, 64, 150])
def test_forks_go_on_as_their_origin_would(cfg, dtype, kv_format, context):
    prompt, later = toks(context, 80, 1), [toks(70, 80, s) for s in (2, 3, 4)]
    eng, ref = engine(cfg, dtype, kv_format), engine(cfg, dtype, kv_format)
    eng.step([("a", prompt, [])])
    free = len(eng.store.pool.free)
    eng.fork("a", ["b", "c"])
    assert free - len(eng.store.pool.free) == (2 if context % 64 else 0)
    got = [run_cut_live(eng, rid, t, [1, 30, 39]) for rid, t in zip("abc", later)]
    tol = TOL[dtype] if kv_format is None else 2e-3
    for g, t in zip(got, later):
        assert rel_err(g, run_cut(ref, "x", prompt + t, [context, 1, 30, 39])[context:]) < tol
    for rid in "acb":
        eng.release(rid)
    assert sorted(eng.store.pool.free) == list(range(eng.store.pool.num_pages)) and not eng.store.pool.shared


def run_cut_live(eng, rid, tokens, cuts):
    """Logits of `tokens` behind what a live request has stored."""
    out, at = [], 0
    for n in cuts:
        part = tokens[at:at + n]
        out.append(eng.step([(rid, part, range(len(part)))]))
        at += n
    return torch.cat(out)


def test_a_prefix_is_shared_by_what_follows_it():
    prefix, tails = toks(130, 80, 7), [toks(20, 80, s) for s in (8, 9)]
    eng, ref = engine(ATTENTION, torch.float32), engine(ATTENTION, torch.float32)
    eng.step([("p", prefix + toks(30, 80, 5), [])])
    eng.fork("p", ["a", "b"], length=130)
    pages = [eng.store.live[r].pages for r in "pab"]
    assert pages[0][:2] == pages[1][:2] == pages[2][:2] and len({p[2] for p in pages}) == 3
    eng.release("p")
    for rid, t in zip("ab", tails):
        assert rel_err(run_cut_live(eng, rid, t, [20]), run_cut(ref, "x", prefix + t, [150])[130:]) < TOL[torch.float32]
    eng.fork("a", ["c"], length=64)  # whole pages: nothing is copied
    assert eng.store.live["c"].pages == eng.store.live["a"].pages[:1]


def test_forks_that_are_refused_leave_everything_as_it_was():
    eng = engine(MIXED, torch.float32, max_tokens=192, slots=3)
    eng.step([("a", toks(70, 80, 1), [])])
    state = (list(eng.store.pool.free), dict(eng.store.pool.shared), list(eng.store.free_slots), list(eng.store.live))
    for call, error in ((("zz", ["b"]), KeyError), (("a", ["a"]), KeyError), (("a", ["b", "b"]), KeyError), (("a", ["b"], 0), ValueError), (("a", ["b"], 71), ValueError),
                        (("a", ["b"], 69), ValueError), (("a", ["b", "c", "d"]), MemoryError), (("a", ["b", "c"]), MemoryError)):
        with pytest.raises(error):
            eng.fork(*call)
        assert state == (sorted(eng.store.pool.free), eng.store.pool.shared, sorted(eng.store.free_slots), list(eng.store.live))


def adapter(model_sites, width_of, g, rank, weights, size=0.4):
    out = {}
    for w in weights:
        depth, cols = width_of[w]
        out[f"{w}.A"] = torch.randn(rank, depth, generator=g) * depth ** -0.5
        out[f"{w}.B"] = torch.randn(cols, rank, generator=g) * rank ** -0.5 * size
    return out


def shapes(sets):
    return {w: (depth, cols) for depth, parts in sets.sites.values() for w, cols in parts}


def merged(weights, tensors, scale):
    w = {k: v.clone() for k, v in weights.items()}
    for k in tensors:
        if k.endswith(".A"):
            w[k[:-2]] = w[k[:-2]] + scale * (tensors[k[:-2] + ".B"].double() @ tensors[k].double()).to(w[k[:-2]].dtype)
    return w


@pytest.mark.parametrize("cfg", [ATTENTION, MIXED])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_request_has_the_model_that_its_adapter_makes(cfg, dtype):
    """Beside the weights is as good as merged into them; requests without one, with one and with the other run in one step: prompts, portions, single tokens, a replayed graph."""
    from paligemma_multimodal_system_b200.adapters import AdapterSet
    from paligemma_multimodal_system_b200.engine import SequenceEngine
    weights, g = O.random_weights(cfg, seed=3), torch.Generator().manual_seed(1)
    model = build(cfg, weights, dtype)
    sets = AdapterSet(model, 3, 12)
    names = sorted(shapes(sets))
    assert any(n.endswith("mix.q") for n in names) and any(n.endswith("mlp.down") for n in names)
    first, second = adapter(sets, shapes(sets), g, 12, names), adapter(sets, shapes(sets), g, 4, names[::2])
    sets.load("unused", adapter(sets, shapes(sets), g, 3, names[:1]))
    sets.load("one", first, scale=0.7), sets.load("two", second)
    eng = SequenceEngine(model, 2048, 4, adapters=sets)
    prompts = {r: toks(n, 80, s) for r, n, s in (("p", 9, 1), ("a", 70, 2), ("b", 33, 3), ("c", 1, 4))}
    use = {"a": "one", "b": "two", "c": "one"}
    steps = [[("p", 9), ("a", 40), ("c", 1)], [("a", 30), ("b", 33)]] + [[(r, 1) for r in "pabc"]] * 4
    follow = {r: toks(4, 80, 10 + s) for s, r in enumerate("pabc")}
    fed, got = {r: 0 for r in prompts}, {r: [] for r in prompts}
    for st in steps:
        entries = []
        for r, n in st:
            full = prompts[r] + follow[r]
            entries.append((r, full[fed[r]:fed[r] + n], [n - 1]))
            fed[r] += n
        logits = eng.step(entries, adapters=use)
        for i, (r, _) in enumerate(st):
            got[r].append(logits[i])
    for r, name in (("p", None), ("a", "one"), ("b", "two"), ("c", "one")):
        tensors, scale = {None: ({}, 0), "one": (first, 0.7), "two": (second, 1.0)}[name]
        ref = SequenceEngine(build(cfg, merged(weights, tensors, scale), dtype), 2048, 4)
        full = prompts[r] + follow[r]
        cuts = [len(prompts[r])] + [1] * 4
        want = run_cut(ref, r, full, cuts)[len(prompts[r]) - 1:]
        # (bf16: merged weights are rounded anew, as far again as the activations)
        assert rel_err(torch.stack(got[r][-5:]), want) < (TOL[dtype] if dtype == torch.float32 else 2 * TOL[dtype]), r
    with pytest.raises(ValueError, match="in use"):
        eng.remove_adapter("one")
    with pytest.raises(ValueError, match="keeps"):
        eng.step([("a", [1], [])], adapters={"a": "two"})
    with pytest.raises(KeyError):
        eng.step([("new", [1], [])], adapters={"new": "nobody"})
    eng.release("a"), eng.release("c")
    eng.remove_adapter("one")
    # its place is taken by another: what it left is gone, a captured step sees the new one
    sets.load("three", second)
    again = eng.step([("d", prompts["b"], [32])], adapters={"d": "three"})
    assert rel_err(again, got["b"][0][None]) < TOL[dtype]


def test_adapters_that_are_refused():
    from paligemma_multimodal_system_b200.adapters import AdapterSet
    sets = AdapterSet(build(ATTENTION, O.random_weights(ATTENTION, seed=3), torch.float32), 1, 4)
    depth, cols = shapes(sets)["l0.mix.q"]
    good = {"l0.mix.q.A": torch.zeros(4, depth), "l0.mix.q.B": torch.zeros(cols, 4)}
    for bad, error in (({}, KeyError), ({"l0.mix.q.A": good["l0.mix.q.A"]}, KeyError), ({**good, "l0.mix.z.A": torch.zeros(1, 1)}, KeyError), ({**good, "odd": torch.zeros(1)}, KeyError),
                       ({**good, "l0.mix.q.A": torch.zeros(5, depth), "l0.mix.q.B": torch.zeros(cols, 5)}, ValueError), ({**good, "l0.mix.q.B": torch.zeros(cols + 1, 4)}, ValueError),
                       ({**good, "l0.mix.q.A": torch.zeros(4, depth - 1)}, ValueError), ({"l0.mlp.gate.A": torch.zeros(4, depth), "l0.mlp.gate.B": torch.zeros(96, 4)}, KeyError)):
        with pytest.raises(error):
            sets.load("x", bad)
        assert not sets.names and not sets.banks
    sets.load("x", good)
    with pytest.raises(KeyError):
        sets.load("x", good)
    with pytest.raises(MemoryError):
        sets.load("y", good)
    for slots, rank in ((0, 4), (1, 0), (1, 129)):
        with pytest.raises(ValueError):
            AdapterSet(build(ATTENTION, O.random_weights(ATTENTION, seed=3), torch.float32), slots, rank)


def periodic(n, V=80, seed=2):
    """Text that repeats itself, so that guesses from it are worth something."""
    base = toks(7, V, seed)
    return (base * (n // 7 + 1))[:n]


@pytest.mark.parametrize("kv_format", [None, "e4m3"])
def test_drafted_generation_says_what_greedy_decoding_says(kv_format):
    from paligemma_multimodal_system_b200.engine import LookupDrafter
    prompts = [toks(40, 80, 9), periodic(60), toks(3, 80, 4), periodic(64, seed=6), toks(130, 80, 5)]
    eng = engine(ATTENTION, torch.float32, kv_format)
    want, said = eng.generate(prompts, 40, logprobs=2)
    calls = []

    def oracle(history):  # a tree: the right continuation behind a wrong child, and some noise
        calls.append(len(history))
        for p, w in zip(prompts, want):
            if history[:len(p)] == p:
                nxt = (w + [0] * 8)[len(history) - len(p):][:4]
                return [(nxt[0] + 1) % 80, nxt[0], 3, nxt[1], nxt[2], 11, nxt[3]], [-1, -1, 0, 1, 3, 1, 4]
        raise AssertionError

    got, told = eng.generate(prompts, 40, draft=oracle, logprobs=2)
    assert got == want and [len(r) for r in told] == [40] * 5
    assert len(calls) < 5 * 40 / 3  # (four or five tokens a step)
    for a, b in zip(said, told):
        assert all(x["rank"] == y["rank"] == 0 and abs(x["logprob"] - y["logprob"]) < 5e-3 for x, y in zip(a, b))
    assert eng.generate(prompts, 40, draft=LookupDrafter(3)) == want
    assert eng.generate(prompts, 40, draft=lambda h: ([], [])) == want
    eos = want[1][17]
    assert eng.generate(prompts, 40, eos_token_id=eos, draft=oracle) == eng.generate(prompts, 40, eos_token_id=eos)
    assert not eng.store.live and not eng._drafted


def test_sampled_drafts_follow_the_models_distribution():
    """The first token behind a prompt, sampled over many runs with a drafted tree: counts are binomial under the model's own distribution."""
    from verify_reference import distribution
    prompt = toks(12, 80, 3)
    eng = engine(ATTENTION, torch.float32, slots=16)
    logits = eng.step([("p", prompt, [len(prompt) - 1])])[0].cpu()
    eng.release("p")
    p = distribution(logits, 1.5, 0.8)
    eng.step([("p", prompt[:-1], [])])
    names = [f"r{i}" for i in range(15)]
    counts, rounds = torch.zeros(80), 60
    guess = [int(i) for i in p.topk(2).indices]
    for r in range(rounds):
        eng.fork("p", names)
        out = eng.step_verify([(n, [prompt[-1]] + guess, [-1, 0, 0]) for n in names], do_sample=True, temperature=1.5, top_p=0.8)
        for path, token in out:
            counts[guess[path[1] - 1] if len(path) > 1 else token] += 1
        for n in names:
            eng.release(n)
    N = rounds * len(names)
    assert (counts[p == 0] == 0).all()
    assert ((counts - N * p).abs() <= 5 * (N * p * (1 - p)).sqrt() + 1e-6).all()


def test_a_drafting_models_distributions_are_taken():
    """With the draft's distributions equal to the model's own every child that it drew stays."""
    prompt = toks(30, 80, 3)
    eng = engine(ATTENTION, torch.float32)
    eng.step([("a", prompt[:-1], [])])
    eng.fork("a", ["b"])
    rows = eng.step_drafts([("b", [prompt[-1], 5, 6], [-1, 0, 1])])
    out = eng.step_verify([("a", [prompt[-1], 5, 6], [-1, 0, 1])], True, 1.0, 1.0, uniforms=torch.full((3, 2), 0.5, device="cuda"), draft_logits=rows)
    assert out[0][0] == [0, 1, 2] and eng.store.live["a"].length == 32
    for bad in (dict(uniforms=torch.zeros(1, 2, device="cuda")), dict(draft_logits=rows)):
        with pytest.raises(ValueError):
            eng.step_verify([("a", [1], [-1])], **bad)
    for toks_, parents in (([1, 2], [-1, -1]), ([1], [0]), ([], [])):
        with pytest.raises(ValueError):
            eng.step_verify([("a", toks_, parents)])


def test_a_run_of_them_together():
    """Two adapters over one prefix: the prefix is run once for each, answers fork from it, drafted trees are judged under each request's own weights, accepted rows stay, and the
    forks' tokens are those of the merged models, one by one."""
    from paligemma_multimodal_system_b200.adapters import AdapterSet
    from paligemma_multimodal_system_b200.engine import SequenceEngine
    weights, g = O.random_weights(ATTENTION, seed=3), torch.Generator().manual_seed(6)
    model = build(ATTENTION, weights, torch.float32)
    sets = AdapterSet(model, 2, 8)
    tensors = {n: adapter(sets, shapes(sets), g, 8, sorted(shapes(sets)), size=0.8) for n in ("one", "two")}
    for n, t in tensors.items():
        sets.load(n, t)
    eng = SequenceEngine(model, 4096, 8, kv_format="e4m3", adapters=sets)
    prefix, asks = toks(75, 80, 1), [toks(5, 80, 2), toks(9, 80, 3)]
    want = {}
    for n in (None, "one", "two"):
        ref = SequenceEngine(build(ATTENTION, merged(weights, tensors.get(n, {}), 1.0), torch.float32), 4096, 8, kv_format="e4m3")
        want[n] = ref.generate([prefix + a for a in asks], 16)
    eng.step([(("p", n), prefix, []) for n in (None, "one", "two")], adapters={("p", n): n for n in ("one", "two")})
    for n in (None, "one", "two"):
        eng.fork(("p", n), [(n, i) for i in range(2)])
        eng.release(("p", n))
    rids = [(n, i) for n in (None, "one", "two") for i in range(2)]
    first = eng.step([(r, asks[r[1]], [len(asks[r[1]]) - 1]) for r in rids]).argmax(-1).tolist()
    got, steps = {r: [t] for r, t in zip(rids, first)}, 0
    while any(len(v) < 16 for v in got.values()):
        entries = []
        for r in rids:
            nxt = (want[r[0]][r[1]] + [0] * 4)[len(got[r]):][:2 + steps % 2]
            toks_, parents = [got[r][-1], 7], [-1, 0]
            for t in nxt:
                toks_.append(t)
                parents.append(0 if len(toks_) == 3 else len(toks_) - 2)
            entries.append((r, toks_, parents))
        for (r, toks_, _), (path, token) in zip(entries, eng.step_verify(entries)):
            got[r] += [toks_[i] for i in path[1:]] + [token]
        steps += 1
    for r in rids:
        assert got[r][:16] == want[r[0]][r[1]], r
    assert steps < 8
    assert eng.generate([prefix + asks[0]] * 3, 16, adapters=[None, "one", "two"], draft=lambda h: (h[-2:], [-1, 0])) == [want[n][0] for n in (None, "one", "two")]


def test_models_of_another_family_take_adapters():
    """Kovusun: norms in front, output projections that add into the residual stream, biases, borrowed keys and values."""
    from paligemma_multimodal_system_b200.adapters import AdapterSet
    from paligemma_multimodal_system_b200.engine import SequenceEngine
    from test_kovusun_gpu import BASE_CFG as cfg
    weights, g = KO.random_weights(cfg, seed=3), torch.Generator().manual_seed(2)
    for dtype in (torch.float32, torch.bfloat16):
        model = build(cfg, weights, dtype)
        sets = AdapterSet(model, 2, 8)
        t = adapter(sets, shapes(sets), g, 8, sorted(shapes(sets)))
        sets.load("one", t)
        V = model.vocab_size
        eng, ref = SequenceEngine(model, 1024, 2, adapters=sets), SequenceEngine(build(cfg, merged(weights, t, 1.0), dtype), 1024, 2)
        full = toks(50, V, 3)
        got = [eng.step([("a", full[:46], range(46))], adapters={"a": "one"})] + [eng.step([("a", [x], [0])]) for x in full[46:]]
        assert rel_err(torch.cat(got), run_cut(ref, "a", full, [46, 1, 1, 1, 1])) < (TOL[dtype] if dtype == torch.float32 else 2 * TOL[dtype])


def test_the_command_guesses(tmp_path, capsys):
    from safetensors.torch import save_file
    from paligemma_multimodal_system_b200.inference import generate_token_ids
    w = O.random_weights(ATTENTION, seed=3)
    os.makedirs(tmp_path, exist_ok=True)
    with open(tmp_path / "config.json", "w") as f:
        json.dump(ATTENTION, f)
    save_file({k: v.to(torch.bfloat16).contiguous() for k, v in w.items()}, str(tmp_path / "model.safetensors"))
    plain = generate_token_ids(str(tmp_path), "5 17 3 5 17 3 5; 8 9", 12, 0.8, 0.9, False, dtype="float32")
    assert generate_token_ids(str(tmp_path), "5 17 3 5 17 3 5; 8 9", 12, 0.8, 0.9, False, dtype="float32", draft=3) == plain


def test_forks_beside_drafts_that_wait_and_of_latent_rows():
    eng, ref = engine(ATTENTION, torch.float32), engine(ATTENTION, torch.float32)
    prompt, drafts, later = toks(70, 80, 1), toks(4, 80, 2), toks(9, 80, 3)
    eng.step([("a", prompt, [])])
    eng.step_drafts([("a", drafts, [-1, 0, 0, 2])])
    eng.fork("a", ["b"])  # what is not accepted is not the fork's
    with pytest.raises(KeyError):
        eng.accept("b", [0])
    eng.accept("a", [0, 2, 3])
    assert (eng.store.live["a"].length, eng.store.live["b"].length) == (73, 70)
    for rid, full in (("a", prompt + [drafts[i] for i in (0, 2, 3)]), ("b", prompt)):
        assert rel_err(run_cut_live(eng, rid, later, [1, 8]), run_cut(ref, "x", full + later, [len(full), 1, 8])[len(full):]) < TOL[torch.float32]
    # one cached row a token, borrowed by another layer
    from test_pukerax_gpu import BASE_CFG, engine_for
    from oracle import pukerax_oracle as PO
    w = PO.random_weights(BASE_CFG, seed=3)
    V = BASE_CFG["vocab"]
    eng, ref = engine_for(BASE_CFG, w, torch.float32), engine_for(BASE_CFG, w, torch.float32)
    prompt, later = toks(90, V, 4), toks(6, V, 5)
    eng.step([("a", prompt, [])])
    eng.fork("a", ["b"], length=77)
    for rid, full in (("a", prompt), ("b", prompt[:77])):
        assert rel_err(run_cut_live(eng, rid, later, [1, 5]), run_cut(ref, "x", full + later, [len(full), 1, 5])[len(full):]) < TOL[torch.float32]


@pytest.mark.parametrize("family,seed", [("fadosun", 2), ("padulorn", 3), ("zigivik", 2), ("pukerax", 3)])
def test_adapters_and_forks_of_every_family(family, seed):
    """Beside the weights is as good as merged into them, whatever a family's sub-layers do with their projections; a fork has copies of what its layers keep."""
    import importlib
    from paligemma_multimodal_system_b200.adapters import AdapterSet
    from paligemma_multimodal_system_b200.engine import SequenceEngine
    t = importlib.import_module(f"test_{family}_gpu")
    cfg, g = t.BASE_CFG, torch.Generator().manual_seed(seed)
    weights = t.steady_weights(cfg, seed=2) if family == "padulorn" else t.O.random_weights(cfg, seed=seed)
    weights = {k: v.to(torch.bfloat16).float() for k, v in weights.items()}  # (as `build` loads them; merged ones are loaded as they are)
    model = t.build(cfg, weights, torch.float32)
    sets = AdapterSet(model, 2, 8)
    own = adapter(sets, shapes(sets), g, 8, sorted(shapes(sets)), size=0.2)
    assert shapes(sets) and all(w in weights for w in shapes(sets)) and (family == "fadosun" or any(w.endswith("mix.o") for w in shapes(sets)))  # (its mixers take none)
    sets.load("one", own)
    V = model.vocab_size
    eng, ref = SequenceEngine(model, 1024, 3, adapters=sets), SequenceEngine(type(model)(model.config, torch.float32).load_weights(merged(weights, own, 1.0)), 1024, 3)
    full, other = toks(52, V, 3), toks(30, V, 4)
    got = eng.step([("a", full[:40], range(40)), ("b", other, [29])], adapters={"a": "one"})
    want = run_cut(ref, "a", full, [40, 8, 1, 1, 1, 1])
    assert rel_err(got[:40], want[:40]) < TOL[torch.float32]
    plain = SequenceEngine(model, 1024, 3)
    assert rel_err(got[40:], run_cut(plain, "b", other, [30])[29:]) < TOL[torch.float32]
    eng.fork("a", ["c"])
    rest = [eng.step([("a", full[40:48], range(8)), ("c", full[40:48], range(8))])] + [eng.step([("c", [x], [0]), ("a", [x], [0])]) for x in full[48:]]
    a = torch.cat([rest[0][:8]] + [r[1:] for r in rest[1:]])
    c = torch.cat([rest[0][8:]] + [r[:1] for r in rest[1:]])
    assert rel_err(a, want[40:]) < TOL[torch.float32] and rel_err(c, want[40:]) < TOL[torch.float32]


def test_guesses_that_are_wrong_leave_no_request_behind():
    eng, prompts = engine(ATTENTION, torch.float32), [toks(20, 80, 1), toks(33, 80, 2)]
    want = eng.generate(prompts, 12)

    def raises(history):
        raise OSError("no guess")

    for draft, error in ((raises, OSError), (lambda h: ([5, 6], [-1]), ValueError), (lambda h: ([5], [3]), ValueError), (lambda h: ([80], [-1]), IndexError), (lambda h: ([-1], [-1]), IndexError)):
        with pytest.raises(error):
            eng.generate(prompts, 12, draft=draft)
        assert not eng.store.live and len(eng.store.free_slots) == eng.store.num_slots and len(eng.store.pool.free) == eng.store.pool.num_pages
    assert eng.generate(prompts, 12, draft=lambda h: ([5, 6, 7], [-1, -1, 0])) == want
    assert eng.generate(prompts, 12, draft=lambda h: ([5] * 40, range(-1, 39))) == want  # more than there is room for
    assert eng.generate(prompts, 12, draft=lambda h: ([], [])) == want
