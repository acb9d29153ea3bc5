"""The 8-bit paged cache: rows quantised as they are written (pg_attn_prepare_e4m3) and read back (pg_kv_read_e4m3), against the format's definition in 64 bits.

Without a norm and a rotation the stored bytes are determined: they are compared as bytes.  With them the kernel's fp32 element y' is off the exact y by a few roundings of the
row's root mean square, the weight, the cosine and the two products: 2^-20 of the pair's length.  Rounding to a code adds half a step: 2^-4 relative, or 2^-10 of the row's power
below 2^-6 of it."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE = 64


def powers_of(x):
    """Bytes for heads x [..., size] (float64): the least e with 448 * 2^e >= largest finite magnitude."""
    a = np.abs(np.where(np.isfinite(x), x, 0.0)).max(-1)
    e = np.full(a.shape, -127)
    for k in range(-127, 121):
        e = np.where(448.0 * 2.0 ** (k - 1) < a, k, e) if k > -127 else e
    return (e + 127).astype(np.uint8)


def codes_of(x, byte):
    y = x / 2.0 ** (byte.astype(np.float64) - 127)[..., None]
    ay = np.abs(np.where(np.isfinite(y), y, 0.0))
    step = 2.0 ** (np.floor(np.log2(np.maximum(ay, 2.0 ** -6))) - 3)
    v = np.round(ay / step) * step  # (numpy rounds halves to even)
    ex = np.floor(np.log2(np.maximum(v, 2.0 ** -6)))
    code = np.where(v < 2.0 ** -6, v / 2.0 ** -9, (ex + 7) * 8 + (v / 2.0 ** ex - 1) * 8).astype(np.int64)
    code = np.where(np.isfinite(x), code, 0x7f)
    return code, np.signbit(x)


def values_of(codes, powers):
    """codes uint8 [rows, heads, size], powers uint8 [rows, heads] -> float64."""
    c = codes.astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((c & 0x7f) == 0x7f, np.nan, v)
    return np.where(c >> 7, -v, v) * (2.0 ** (powers.astype(np.float64) - 127))[..., None]


def batch_of(lens, seed=0, parents=None, spare=3):
    """StepBatch of entries (n, ctx) with pages handed out in any order from a pool with some to spare."""
    from paligemma_multimodal_system_b200 import seq_ops
    need = [(n + c + PAGE - 1) // PAGE for n, c in lens]
    order = np.random.RandomState(seed).permutation(sum(need) + spare).tolist()
    entries = []
    for i, (n, c) in enumerate(lens):
        e = dict(tokens=[1] * n, ctx=c, slot=i, pages=[order.pop() for _ in range(need[i])])
        if parents is not None:
            e["parents"] = parents[i]
        entries.append(e)
    return seq_ops.make_step_batch(entries), entries, sum(need) + spare


def stored(pages, entry, rows, G):
    """(codes [rows, G, size], powers [rows, G]) of one entry's first rows."""
    c, p = pages.codes.cpu().numpy(), pages.powers.cpu().numpy()
    at = [(entry["pages"][j // PAGE], j % PAGE) for j in range(rows)]
    return np.stack([c[a, b].reshape(G, -1) for a, b in at]), np.stack([p[a, :, b] for a, b in at])


def fresh(pool, G, size):
    from paligemma_multimodal_system_b200.seq_ops import QuantizedPages
    q = QuantizedPages.empty(pool, PAGE, G, size)
    q.codes.fill_(0x7f)  # whatever is not written is no number
    q.powers.fill_(200)
    return q


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,dim,vdim", [(4, 2, 64, 64), (3, 3, 16, 48), (8, 1, 128, 64), (2, 1, 256, 256), (5, 5, 96, 32)])
@pytest.mark.parametrize("lens", [[(1, 0)], [(1, 63), (1, 64), (3, 62)], [(70, 5), (1, 200), (129, 0)]])
def test_stored_bytes(dtype, H, G, dim, vdim, lens):
    from paligemma_multimodal_system_b200 import seq_ops
    b, entries, pool = batch_of(lens)
    g = torch.Generator(device="cuda").manual_seed(dim + b.T)
    proj = torch.randn(b.T, (H + G) * dim + G * vdim, generator=g, device="cuda") * torch.exp2(torch.randint(-20, 20, (b.T, 1), generator=g, device="cuda").float())
    proj[0, H * dim:H * dim + dim] = 0  # a head of zeros
    proj[0, H * dim + 1] = -0.0
    proj[-1, -vdim] = math.inf  # what is not finite is kept as NaN, beside its neighbours
    proj[-1, -vdim + 1] = math.nan
    proj[-1, -vdim + 2] = 448.0 * 2.0 ** 30  # (the top of the head: a power that is met exactly)
    if dtype == torch.float32:
        proj[0, (H + G) * dim:(H + G) * dim + vdim] = 1e-40  # below the normal numbers
    proj = proj.to(dtype)
    q = torch.empty(b.T, H * dim, device="cuda", dtype=dtype)
    kq, vq = fresh(pool, G, dim), fresh(pool, G, vdim)
    before = kq.codes.clone()
    freq = torch.zeros(1, device="cuda", dtype=torch.float64)
    seq_ops.attn_prepare(proj, b, freq, None, None, q, kq, vq, H, G, dim, vdim, 0, 1e-6, PAGE, norm_qk=False, norm_v=False)
    assert torch.equal(q, proj[:, :H * dim])
    x = proj.double().cpu().numpy()
    r = 0
    for (n, ctx), e in zip(lens, entries):
        for pages, lo, size in ((kq, H * dim, dim), (vq, (H + G) * dim, vdim)):
            rows = x[r:r + n, lo:lo + G * size].reshape(n, G, size)
            codes, powers = stored(pages, e, ctx + n, G)
            want = powers_of(rows)
            assert np.array_equal(powers[ctx:], want)
            code, sign = codes_of(rows, want)
            assert np.array_equal(codes[ctx:] & 0x7f, code)
            assert np.array_equal((codes[ctx:] >> 7 == 1) | (code == 0x7f), sign | (code == 0x7f))
            assert (codes[:ctx] == 0x7f).all() and (powers[:ctx] == 200).all()  # rows of earlier steps: as they were
        r += n
    written = sum(n for n, _ in lens)
    assert int((kq.codes != before).any(-1).sum()) <= written


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm,rot,weights,from_k", [(True, 64, True, False), (True, 32, False, False), ("projection", 64, True, False), (False, 64, False, True), (True, 6, True, False)])
def test_norms_and_rotation(dtype, norm, rot, weights, from_k):
    from paligemma_multimodal_system_b200 import seq_ops
    H, G, dim, vdim, eps = 4, 2, 64, 64, 1e-6
    lens = [(1, 900), (37, 100000 % 977), (3, 0)]
    b, entries, pool = batch_of(lens, 1)
    g = torch.Generator(device="cuda").manual_seed(5)
    cols = (H + G) * dim + (0 if from_k else G * vdim)
    proj = torch.randn(b.T, cols, generator=g, device="cuda").to(dtype)
    other = None if from_k else torch.randn(b.T, G * vdim, generator=g, device="cuda").to(dtype)
    mode = seq_ops.NORM_PROJECTION if norm == "projection" else norm
    wq = 1 + 0.2 * torch.randn(H * dim if norm == "projection" else dim, generator=g, device="cuda") if weights else None
    wk = 1 + 0.2 * torch.randn(G * dim if norm == "projection" else dim, generator=g, device="cuda") if weights else None
    freq = 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / max(rot, 1))
    q = torch.empty(b.T, H * dim, device="cuda", dtype=dtype)
    kq, vq = fresh(pool, G, dim), fresh(pool, G, vdim)
    seq_ops.attn_prepare(proj, b, freq, wq, wk, q, kq, vq, H, G, dim, vdim, rot, eps, PAGE, norm_qk=mode, norm_v=not from_k, v_from_k=from_k, rot_gain=1.5, v_other=other, v_mix=0.25)
    # the cache of the activations' type takes the same rows: the same queries
    q2, kp, vp = torch.empty_like(q), torch.zeros(pool, PAGE, G * dim, device="cuda", dtype=dtype), torch.zeros(pool, PAGE, G * vdim, device="cuda", dtype=dtype)
    seq_ops.attn_prepare(proj, b, freq, wq, wk, q2, kp, vp, H, G, dim, vdim, rot, eps, PAGE, norm_qk=mode, norm_v=not from_k, v_from_k=from_k, rot_gain=1.5, v_other=other, v_mix=0.25)
    half = torch.finfo(dtype).eps / 2
    assert torch.all((q.double() - q2.double()).abs() <= 2 * half * q2.double().abs() + 2.0 ** -19)
    x = proj.double().cpu().numpy()

    def normed(y, w, whole):
        ms = (y ** 2).mean((-2, -1) if whole else -1, keepdims=True)
        y = y / np.sqrt(ms + eps)
        return y if w is None else y * w.double().cpu().numpy().reshape((-1, dim) if whole else (dim,))

    k = x[:, H * dim:(H + G) * dim].reshape(-1, G, dim)
    v = k if from_k else x[:, (H + G) * dim:].reshape(-1, G, vdim)
    if norm:
        k = normed(k, wk, norm == "projection")
    ang = b.pos.double().cpu().numpy()[:, None] * freq.cpu().numpy()
    c, s = 1.5 * np.cos(ang)[:, None], 1.5 * np.sin(ang)[:, None]
    k = k.copy()
    k[..., :rot:2], k[..., 1:rot:2] = k[..., :rot:2] * c - k[..., 1:rot:2] * s, k[..., 1:rot:2] * c + k[..., :rot:2] * s
    if not from_k:
        v = 0.75 * (v / np.sqrt((v ** 2).mean(-1, keepdims=True) + eps)) + 0.25 * other.double().cpu().numpy().reshape(-1, G, vdim)
    r = 0
    for (n, ctx), e in zip(lens, entries):
        for pages, y in ((kq, k[r:r + n]), (vq, v[r:r + n])):
            codes, powers = (z[ctx:] for z in stored(pages, e, ctx + n, G))
            got, p = values_of(codes, powers), 2.0 ** (powers.astype(np.float64) - 127)[..., None]
            top = np.abs(y).max(-1, keepdims=True)
            assert (top <= 448 * p * (1 + 2.0 ** -18)).all() and (top >= 224 * p * (1 - 2.0 ** -18)).all()
            assert (np.abs(got - y) <= 2.0 ** -4 * np.abs(y) + 2.0 ** -10 * p + 2.0 ** -18 * top).all()
        r += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G,dim,vdim", [(2, 64, 64), (1, 16, 256), (3, 96, 32)])
def test_read_back(dtype, G, dim, vdim):
    from paligemma_multimodal_system_b200 import seq_ops
    lens = [(2, 0), (1, 300), (70, 58), (64, 0), (5, 1000), (65, 63)]
    b, entries, pool = batch_of(lens, 2)
    kq, vq = seq_ops.QuantizedPages.empty(pool, PAGE, G, dim), seq_ops.QuantizedPages.empty(pool, PAGE, G, vdim)
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in (kq, vq):
        p.codes.copy_(torch.randint(0, 256, p.codes.shape, generator=g, device="cuda", dtype=torch.uint8))
        p.powers.copy_(torch.randint(0, 240, p.powers.shape, generator=g, device="cuda", dtype=torch.uint8))
    k, v = seq_ops.kv_read(kq, vq, b, dtype)
    assert k.shape == (b.dense_rows, G * dim) and v.shape == (b.dense_rows, G * vdim)
    row0 = b.dense_row0.cpu().tolist()
    for i, ((n, ctx), e) in enumerate(zip(lens, entries)):
        if n == 1:
            continue
        for pages, out in ((kq, k), (vq, v)):
            codes, powers = stored(pages, e, n + ctx, G)
            want = torch.from_numpy(values_of(codes, powers).reshape(n + ctx, -1)).float().to(dtype)
            got = out[row0[i]:row0[i] + n + ctx].cpu()
            assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float())) and torch.equal(got.isnan(), want.isnan())
            tail = out[row0[i] + n + ctx:row0[i] + (n + ctx + 63) // 64 * 64]
            assert not tail.any()


def test_rows_on_odd_addresses_and_pitches():
    from paligemma_multimodal_system_b200 import seq_ops
    H, G, dim = 2, 1, 32
    b, entries, pool = batch_of([(5, 3), (1, 64)], 3)
    wide = torch.randn(b.T, (H + 2 * G) * dim + 9, device="cuda").to(torch.bfloat16)
    proj = wide[:, 3:3 + (H + 2 * G) * dim]
    freq = torch.zeros(1, device="cuda", dtype=torch.float64)
    outs = []
    for rows in (proj, proj.contiguous()):
        q, kq, vq = torch.empty(b.T, H * dim, device="cuda", dtype=torch.bfloat16), fresh(pool, G, dim), fresh(pool, G, dim)
        seq_ops.attn_prepare(rows, b, freq, None, None, q, kq, vq, H, G, dim, dim, 0, 1e-6, PAGE, norm_qk=True, norm_v=True)
        outs.append((q, kq.codes, kq.powers, vq.codes, vq.powers))
    for x, y in zip(*outs):
        assert torch.equal(x, y)


def test_many_rows_take_four_tokens_a_block():
    """2400 and more rows: four tokens share a block's angles; the same bytes as in small steps."""
    from paligemma_multimodal_system_b200 import seq_ops
    H, G, dim = 2, 2, 64
    b, entries, pool = batch_of([(2500, 11), (1, 7), (30, 0)], 4)
    proj = torch.randn(b.T, (H + 2 * G) * dim, device="cuda").to(torch.bfloat16)
    freq = 1e4 ** (-2.0 * torch.arange(32, dtype=torch.float64, device="cuda") / 64)

    def go(rows, batch):
        q = torch.empty(batch.T, H * dim, device="cuda", dtype=torch.bfloat16)
        seq_ops.attn_prepare(rows, batch, freq, None, None, q, kq, vq, H, G, dim, dim, 64, 1e-6, PAGE, norm_qk=True, norm_v=False)
        return q

    kq, vq = fresh(pool, G, dim), fresh(pool, G, dim)
    q = go(proj, b)
    all_at_once = [q, kq.codes, kq.powers, vq.codes, vq.powers]
    kq, vq = fresh(pool, G, dim), fresh(pool, G, dim)
    parts, r = [], 0
    for e, (n, ctx) in zip(entries, [(2500, 11), (1, 7), (30, 0)]):
        for lo in range(0, n, 700):
            m = min(700, n - lo)
            parts.append(go(proj[r + lo:r + lo + m], seq_ops.make_step_batch([dict(e, tokens=[1] * m, ctx=ctx + lo)])))
        r += n
    for x, y in zip(all_at_once, [torch.cat(parts), kq.codes, kq.powers, vq.codes, vq.powers]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,G,dim,mode", [(1, 1, 16, True), (37, 3, 96, "projection"), (3001, 2, 256, True), (6000, 8, 128, True), (6001, 3, 64, "projection")])
def test_codes_of_computed_elements_are_the_nearest(dtype, rows, G, dim, mode):
    """Without a rotation an fp32 element is within 2^-20 of the exact one: a sum of squares of 8 products a lane and 5 exchanges (13 half steps of 2^-24, halved by the root), the
    mean, the root to 2 steps, two products.  What that could move to another code is made in double (off by 2^-48 or so), so that bytes are determined here too."""
    from paligemma_multimodal_system_b200 import seq_ops
    H, eps = 1, 2.0 ** -20
    b, entries, pool = batch_of([(rows, 5)], rows)
    g = torch.Generator(device="cuda").manual_seed(rows)
    proj = torch.randn(b.T, (H + 2 * G) * dim, generator=g, device="cuda").to(dtype)
    n = dim if mode is True else G * dim
    wk = 1 + 0.2 * torch.randn(n, generator=g, device="cuda")
    wq = torch.ones(dim if mode is True else H * dim, device="cuda")
    kq, vq, q = fresh(pool, G, dim), fresh(pool, G, dim), torch.empty(b.T, H * dim, device="cuda", dtype=dtype)
    seq_ops.attn_prepare(proj, b, torch.zeros(1, device="cuda", dtype=torch.float64), wq, wk, q, kq, vq, H, G, dim, dim, 0, eps, PAGE,
                         norm_qk=True if mode is True else seq_ops.NORM_PROJECTION, norm_v=True)
    x = proj.double().cpu().numpy()
    for pages, lo, w in ((kq, H * dim, wk.double().cpu().numpy()), (vq, (H + G) * dim, None)):
        y = x[:, lo:lo + G * dim].reshape(rows, G, dim)
        whole = w is not None and mode is not True
        y = y / np.sqrt((y ** 2).mean((-2, -1) if whole else -1, keepdims=True) + eps)
        y = y if w is None else y * (w.reshape(1, G, dim) if whole else w)
        codes, powers = stored(pages, entries[0], 5 + rows, G)
        want = powers_of(y)
        assert np.array_equal(powers[5:], want)
        code, sign = codes_of(y, want)
        assert np.array_equal(codes[5:] & 0x7f, code)
        assert np.array_equal(codes[5:] >> 7 == 1, sign)
