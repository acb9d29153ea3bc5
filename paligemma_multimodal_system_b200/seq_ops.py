"""Host wrappers of the ragged-step kernels (csrc/seq_elementwise.cu, csrc/seq_mixers.cu) and the step's batch descriptor.

`Precision` says in which type activations and matrix operands live: bf16 (tcgen05 GEMMs with fp32 accumulation wherever
the shape allows TMA, the plain-FMA kernel otherwise) or fp32 (plain FMAs, or for many tokens three bf16 terms a value on the
tensor cores with an error no larger than theirs; no reduced-precision tensor mode).
Norm statistics, attention scores and probabilities, recurrent states and the residual stream are fp32 in both.
"""
import dataclasses
from typing import List, Optional, Sequence

import numpy as np
import torch

from . import _lib


class Precision:
    def __init__(self, dtype: torch.dtype):
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("activation type must be torch.bfloat16 or torch.float32")
        self.dtype = dtype
        self.f32 = int(dtype == torch.float32)

    def empty(self, *shape):
        return torch.empty(*shape, device="cuda", dtype=self.dtype)


@dataclasses.dataclass
class StepBatch:
    """One ragged step on the device.  Rows are tokens; entry e owns rows [row0[e], row0[e] + n[e])."""
    T: int
    E: int
    max_n: int
    tokens: torch.Tensor      # int32 [T]
    pos: torch.Tensor         # int32 [T] position of the row inside its sequence
    row_entry: torch.Tensor   # int32 [T]
    row0: torch.Tensor        # int32 [E]
    n: torch.Tensor           # int32 [E]
    ctx: torch.Tensor         # int32 [E] tokens of the sequence already stored before this step
    slot: torch.Tensor        # int32 [E] recurrent-state slot
    page_table: torch.Tensor  # int32 [E, max_pages]
    max_pages: int
    singles: int = 0          # entries with one new token (decode rows)
    max_single_ctx: int = 0   # the longest context among them
    single_rows: Optional[tuple] = None  # (first, one past the last) row between which all of them lie; None: unknown
    # dense scratch layout of the entries with several new tokens (mixers that rebuild per-head keys / values from a compact
    # cache): entry e owns rows [dense_row0[e], + ctx + n) of a dense matrix, starting on a page boundary, so that
    # dense_pages[e] = consecutive page numbers is a page table over the scratch and the paged attention kernels read it
    dense_row0: Optional[torch.Tensor] = None   # int32 [E]
    dense_pages: Optional[torch.Tensor] = None  # int32 [E, dense_max_pages]
    dense_max_pages: int = 0
    dense_rows: int = 0       # rows of the scratch matrix (a multiple of the page size)
    dense_max_len: int = 0    # the longest ctx + n among those entries
    # what one layer of the CURRENT step leaves for later ones (rotation tables, a layer's values); a model that uses it starts every step
    # with a fresh one (`step_scope`)
    shared: Optional[dict] = None
    min_n: int = 1            # the fewest new tokens of an entry (1 where that is not known)

    # drafted trees: `pos`, which turns queries and keys, is then ctx + depth; rows are stored one behind another at cache rows `at`, and a row sees the
    # drafted rows of its entry whose bit is set in its mask (bit m % 32 of word m / 32)
    # (taken by name, or behind the others; `dataclasses.replace` keeps them)
    at: dataclasses.InitVar[Optional[torch.Tensor]] = None    # int32 [T]; None: pos
    tree: dataclasses.InitVar[Optional[torch.Tensor]] = None  # int32 [T, words]; None: rows see every row in front of them

    def __post_init__(self, at, tree):
        self.at, self.tree = at, tree


TreeBatch = StepBatch  # (another name for a step that has these two)
StepBatch.parents = StepBatch.adapters = None


@dataclasses.dataclass
class RequestBatch(StepBatch):
    """A step whose requests have something of their own (`dataclasses.replace` keeps both)."""
    parents: dataclasses.InitVar[Optional[torch.Tensor]] = None  # int32 [T], drafted trees: the row of its entry that a row follows, -1 the stored tokens
    adapters: dataclasses.InitVar[Optional[object]] = None  # low-rank adapters of the entries (adapters.StepAdapters)

    def __post_init__(self, at, tree, parents, adapters):
        self.at, self.tree, self.parents, self.adapters = at, tree, parents, adapters


def _single_rows(ns):
    """The rows between which the entries of one new token lie."""
    first, last, r = None, 0, 0
    for k in ns:
        if k == 1:
            first, last = r if first is None else first, r + 1
        r += k
    return None if first is None else (first, last)


def _tree_masks(parents, ns):
    """parents: per entry a list (parents[i] < i is the row that row i follows, -1 the stored tokens) or None for a chain.  Returns (mask words uint32 [T, words],
    depth of every row)."""
    words = (max(ns) + 31) // 32
    masks, depth, r = np.zeros((sum(ns), words), dtype=np.uint32), np.zeros(sum(ns), dtype=np.int32), 0
    for up, n in zip(parents, ns):
        up = range(-1, n - 1) if up is None else [int(x) for x in up]
        if len(up) != n or any(not -1 <= x < i for i, x in enumerate(up)):
            raise ValueError("parents: one for every token, an earlier token of the entry or -1")
        for i, x in enumerate(up):
            if x >= 0:
                masks[r + i], depth[r + i] = masks[r + x], depth[r + x] + 1
            masks[r + i, i // 32] |= np.uint32(1 << (i % 32))
        r += n
    return masks, depth


def make_step_batch(entries: Sequence[dict]) -> StepBatch:
    """entries: dicts with tokens (list[int]), ctx (int), slot (int), pages (list[int]); drafted trees: parents (list[int], see _tree_masks; entries without are
    chains).  One host buffer, one copy."""
    E = len(entries)
    ns = [len(e["tokens"]) for e in entries]
    T = sum(ns)
    if E == 0 or min(ns) <= 0:
        raise ValueError("a step needs at least one entry and every entry at least one token")
    max_pages = max(1, max(len(e["pages"]) for e in entries))
    lens = [e["ctx"] + k if k > 1 else 0 for e, k in zip(entries, ns)]
    dpages = [(l + 63) // 64 for l in lens]
    dmax = max(1, max(dpages))
    masks = depth = None
    if any(e.get("parents") is not None for e in entries):
        masks, depth = _tree_masks([e.get("parents") for e in entries], ns)
    words = 0 if masks is None else masks.shape[1]
    plain = 3 * T + 4 * E + E * max_pages + E + E * dmax
    buf = np.zeros(plain + (0 if masks is None else T * (2 + words)), dtype=np.int32)
    tokens, pos, row_entry = buf[:T], buf[T:2 * T], buf[2 * T:3 * T]
    o = 3 * T
    row0, n, ctx, slot = buf[o:o + E], buf[o + E:o + 2 * E], buf[o + 2 * E:o + 3 * E], buf[o + 3 * E:o + 4 * E]
    pt = buf[o + 4 * E:o + 4 * E + E * max_pages].reshape(E, max_pages)
    o2 = o + 4 * E + E * max_pages
    drow0, dpt = buf[o2:o2 + E], buf[o2 + E:plain].reshape(E, dmax)
    page0 = 0
    for i in range(E):
        drow0[i] = page0 * 64
        dpt[i, :dpages[i]] = np.arange(page0, page0 + dpages[i])
        page0 += dpages[i]
    r = 0
    for i, e in enumerate(entries):
        k = ns[i]
        if (e["ctx"] + k + 63) // 64 > len(e["pages"]):
            raise ValueError("entry does not own enough pages for its new tokens")
        tokens[r:r + k] = e["tokens"]
        pos[r:r + k] = np.arange(e["ctx"], e["ctx"] + k)
        row_entry[r:r + k] = i
        row0[i], n[i], ctx[i], slot[i] = r, k, e["ctx"], e["slot"]
        pt[i, :len(e["pages"])] = e["pages"]
        r += k
    if masks is not None:
        buf[plain:plain + T] = pos
        buf[plain + T:plain + 2 * T] = np.concatenate([np.arange(-1, k - 1) if e.get("parents") is None else np.asarray(e["parents"]) for e, k in zip(entries, ns)])
        buf[plain + 2 * T:] = masks.reshape(-1).view(np.int32)
        pos[:] = ctx[row_entry] + depth
    dev = torch.from_numpy(buf).pin_memory().to("cuda", non_blocking=True)
    o = 3 * T
    drafted = {} if masks is None else dict(at=dev[plain:plain + T], parents=dev[plain + T:plain + 2 * T], tree=dev[plain + 2 * T:].view(T, words))
    return (StepBatch if masks is None else RequestBatch)(T=T, E=E, max_n=max(ns), min_n=min(ns), tokens=dev[:T], pos=dev[T:2 * T], row_entry=dev[2 * T:3 * T], row0=dev[o:o + E],
                     n=dev[o + E:o + 2 * E], ctx=dev[o + 2 * E:o + 3 * E], slot=dev[o + 3 * E:o + 4 * E],
                     page_table=dev[o + 4 * E:o2].view(E, max_pages), max_pages=max_pages, singles=sum(k == 1 for k in ns),
                     max_single_ctx=max([e["ctx"] for e, k in zip(entries, ns) if k == 1], default=0), single_rows=_single_rows(ns),
                     dense_row0=dev[o2:o2 + E], dense_pages=dev[o2 + E:plain].view(E, dmax), dense_max_pages=dmax, dense_rows=page0 * 64,
                     dense_max_len=max(lens), **drafted)


def with_adapters(b: StepBatch, adapters) -> RequestBatch:
    """The same step whose entries have adapters (adapters.StepAdapters)."""
    return RequestBatch(**{f.name: getattr(b, f.name) for f in dataclasses.fields(b)}, at=b.at, tree=b.tree, parents=b.parents, adapters=adapters)


def adapt(b: Optional[StepBatch], site: str, x, y, gain=1.0):
    """Adds what the step's adapters have beside the projection `site` of x to y; nothing in a step without adapters."""
    if b is not None and b.adapters is not None:
        b.adapters.add(site, x, y, gain)


def step_scope(b: StepBatch) -> StepBatch:
    """The same step with an empty `shared`."""
    return dataclasses.replace(b, shared={})


class StaticDecodeBatch:
    """Fixed-address StepBatch for steps of E single-token entries (a decode step), so that the step can be captured once in a
    CUDA graph and replayed: `fill` rewrites the pinned host image and copies it over the device buffer in stream order.
    `pages_cap` is the page-table width the graph was captured with; `ctx_cap` the context bound that fixed its key split."""

    def __init__(self, E: int, pages_cap: int, ctx_cap: int):
        self.E, self.pages_cap, self.ctx_cap = E, pages_cap, ctx_cap
        n = 7 * E + E * pages_cap
        self.host = torch.zeros(n, dtype=torch.int32).pin_memory()
        self.dev = torch.zeros(n, dtype=torch.int32, device="cuda")
        d = self.dev
        self.batch = StepBatch(T=E, E=E, max_n=1, tokens=d[:E], pos=d[E:2 * E], row_entry=d[2 * E:3 * E], row0=d[3 * E:4 * E], n=d[4 * E:5 * E],
                               ctx=d[5 * E:6 * E], slot=d[6 * E:7 * E], page_table=d[7 * E:].view(E, pages_cap), max_pages=pages_cap, singles=E,
                               max_single_ctx=ctx_cap)
        self.rows = torch.arange(E, device="cuda", dtype=torch.int64)
        self._copied = None

    def fill(self, entries: Sequence[dict]):
        E, h = self.E, self.host.numpy()
        assert len(entries) == E
        if self._copied is not None:
            self._copied.synchronize()  # the previous image must have left the pinned buffer before it is rewritten
        h[7 * E:] = 0
        pt = h[7 * E:].reshape(E, self.pages_cap)
        for i, e in enumerate(entries):
            assert len(e["tokens"]) == 1 and len(e["pages"]) <= self.pages_cap and e["ctx"] <= self.ctx_cap
            h[i], h[E + i], h[2 * E + i], h[3 * E + i], h[4 * E + i], h[5 * E + i], h[6 * E + i] = e["tokens"][0], e["ctx"], i, i, 1, e["ctx"], e["slot"]
            pt[i, :len(e["pages"])] = e["pages"]
        self.dev.copy_(self.host, non_blocking=True)
        self._copied = torch.cuda.Event()
        self._copied.record()


def _aligned(t, n=16):
    return t.data_ptr() % n == 0


def _on_current_device(t):
    """Launches go to the current device's current stream: its kernels read and write its own memory."""
    if t.device.index != torch._C._cuda_getDevice():
        raise ValueError(f"the tensors lie on {t.device}, the current device is cuda:{torch._C._cuda_getDevice()}")


# ACT_SILU_GLU: grouped products only (gate / up rows alternate); ACT_GELU is the tanh form, ACT_GELU_ERF the exact one
ACT_NONE, ACT_GELU, ACT_RELU2, ACT_SILU_GLU, ACT_GELU_ERF = 0, 1, 2, 3, 6


def _linear_fp32_split(x, w, out, bias, accumulate, scale):
    """fp32 products of many tokens on the tensor cores (three bf16 terms a value); False where the plain-FMA form is faster or has to take the call: it needs no
    scratch, so a device without room for that (256 MB at most) is served as well."""
    T, K = x.shape
    F = w.shape[0]
    if not (x.is_cuda and w.is_cuda and _aligned(x) and _aligned(w) and _aligned(out)) or (x.stride(0) | w.stride(0) | out.stride(0)) % 4:
        return False
    need = (_lib.lib().pg_gemm_fp32_scratch_add if accumulate else _lib.lib().pg_gemm_fp32_scratch)(T, F, K)
    if not need:
        return False
    try:
        scratch = torch.empty(need, device=x.device, dtype=torch.uint8)
    except torch.OutOfMemoryError:
        return False
    _lib.check(_lib.lib().pg_gemm_fp32_split(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), out.data_ptr(), out.stride(0), _lib.ptr(bias), accumulate, scale,
                                             T, F, K, scratch.data_ptr(), need, _lib.stream()), "pg_gemm_fp32_split")
    return True


def linear(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor, act: int = ACT_NONE, bias: Optional[torch.Tensor] = None, zeros: bool = False):
    """out[t, f] = act(sum_k x[t, k] w[f, k] + bias[f]) (bias fp32 or None).  x, w share a type (bf16 / fp32); out is bf16 or fp32.  bf16 operands go to the
    tcgen05 kernel when TMA can describe them (16-byte pitches and bases), everything else to the plain-FMA kernel.
    act = ACT_RELU2 (relu squared; out in the operands' type): in the tensor-core kernel's bf16 epilogue, else a pass of its own.
    zeros: out holds zeros (a product that shares K out over the GPU need not clear it first)."""
    T, K = x.shape
    F = w.shape[0]
    assert x.dtype == w.dtype and w.shape[1] == K and out.shape[0] == T and out.shape[1] == F
    assert x.stride(1) == 1 and w.stride(1) == 1 and out.stride(1) == 1
    if (x.dtype == torch.bfloat16 and K % 8 == 0 and x.stride(0) % 8 == 0 and w.stride(0) % 8 == 0 and F % 8 == 0
            and out.stride(0) % 8 == 0 and _aligned(x) and _aligned(w) and _aligned(out)):
        assert act == ACT_NONE or out.dtype == torch.bfloat16
        if act != ACT_NONE:
            return _lib.gemm(x, w, out, mode=_lib.EPI_BF16, act_gelu=act, swap=1 if T <= 128 else 0, bias=bias)
        if out.dtype == torch.float32 and bias is None:
            assert x.is_cuda and w.is_cuda and w.dim() == 2
            fn = _lib.lib().pg_linear_f32_zeros if zeros else _lib.lib().pg_linear_f32
            _lib.check(fn(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), out.data_ptr(), out.stride(0), T, F, K, _lib.stream()),
                       "pg_linear_f32")
            return out
        return _lib.gemm(x, w, out, mode=_lib.EPI_F32 if out.dtype == torch.float32 else _lib.EPI_BF16, swap=1 if T <= 128 else 0, bias=bias)
    if x.dtype == torch.float32 and out.dtype != torch.float32:
        raise ValueError("fp32 operands produce fp32 outputs")
    assert bias is None or (bias.dtype == torch.float32 and bias.numel() == F and bias.is_contiguous())
    if x.dtype == torch.float32 and _linear_fp32_split(x, w, out, bias, 0, 1.0):
        pass
    elif bias is not None:
        _lib.check(_lib.lib().pg_gemm_simt_bias(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), out.data_ptr(), out.stride(0), bias.data_ptr(), 0, 1.0,
                                                T, F, K, int(x.dtype == torch.float32), int(out.dtype == torch.float32), _lib.stream()), "pg_gemm_simt_bias")
    else:
        _lib.check(_lib.lib().pg_gemm_simt(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), out.data_ptr(), out.stride(0), T, F, K,
                                           int(x.dtype == torch.float32), int(out.dtype == torch.float32), _lib.stream()), "pg_gemm_simt")
    if act == ACT_RELU2:
        _lib.check(_lib.lib().pg_relu2(out.data_ptr(), out.stride(0), T, F, int(out.dtype == torch.float32), _lib.stream()), "pg_relu2")
    elif act != ACT_NONE:
        raise ValueError("the plain-FMA product has no fused activation but relu squared")
    return out


def linear_add(x: torch.Tensor, w: torch.Tensor, resid: torch.Tensor, bias: Optional[torch.Tensor] = None, scale: float = 1.0):
    """resid[t, f] += (sum_k x[t, k] w[f, k] + bias[f]) * scale: a projection that ends in the fp32 residual stream.  bf16 operands TMA can
    describe: the tcgen05 kernel adds the residual in its epilogue (or red.adds split-K partials into it when there are few
    tiles); everything else: the plain-FMA kernel reads and rewrites the residual element."""
    T, K = x.shape
    F = w.shape[0]
    assert x.dtype == w.dtype and w.shape[1] == K and resid.shape == (T, F) and resid.dtype == torch.float32 and resid.is_contiguous()
    assert x.stride(1) == 1 and w.stride(1) == 1
    if (x.dtype == torch.bfloat16 and K % 8 == 0 and x.stride(0) % 8 == 0 and w.stride(0) % 8 == 0 and F % 8 == 0 and _aligned(x) and _aligned(w)
            and _aligned(resid)):
        return _lib.gemm_residual(x, w, resid, bias=bias, scale=float(scale))
    assert bias is None or (bias.dtype == torch.float32 and bias.numel() == F and bias.is_contiguous())
    if x.dtype == torch.float32 and _linear_fp32_split(x, w, resid, bias, 1, float(scale)):
        return resid
    _lib.check(_lib.lib().pg_gemm_simt_bias(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), resid.data_ptr(), resid.stride(0), _lib.ptr(bias), 1, float(scale),
                                            T, F, K, int(x.dtype == torch.float32), 1, _lib.stream()), "pg_gemm_simt_bias")
    return resid


def layernorm_shift(x, w1, b1, out1, eps, shift=None, state=None, b: "StepBatch" = None, w2=None, b2=None, out2=None):
    """out1 = LN(x; w1, b1) -- blended with the previous token's when `shift` [D] is given (state: fp32 [slots, D], the batch says which
    row continues which sequence) -- and out2 = LN(x; w2, b2) from the same statistics.  x fp32 [rows, D]; outputs bf16 or fp32."""
    rows, D = x.shape
    assert x.dtype == torch.float32 and x.is_contiguous() and out1.is_contiguous() and out1.shape == x.shape
    for t in (w1, b1, shift, w2, b2):
        assert t is None or (t.dtype == torch.float32 and t.is_contiguous() and t.numel() == D)
    assert out2 is None or (out2.is_contiguous() and out2.shape == x.shape and out2.dtype == out1.dtype and w2 is not None and b2 is not None)
    if shift is not None:
        assert state is not None and state.dtype == torch.float32 and state.is_contiguous() and state.shape[-1] == D and b is not None and b.T == rows
    _lib.check(_lib.lib().pg_layernorm_shift(x.data_ptr(), w1.data_ptr(), b1.data_ptr(), _lib.ptr(shift), _lib.ptr(w2), _lib.ptr(b2), out1.data_ptr(),
                                             _lib.ptr(out2), _lib.ptr(state), *((b.pos.data_ptr(), b.row_entry.data_ptr(), b.row0.data_ptr(),
                                                                                 b.n.data_ptr(), b.slot.data_ptr()) if shift is not None else (0, 0, 0, 0, 0)),
                                             rows, D, float(eps), int(out1.dtype == torch.float32), _lib.stream()), "pg_layernorm_shift")


def rmsnorm_conv(x, w, out_h, out_conv, eps, conv_w=None, state=None, b: "StepBatch" = None):
    """h = x / rms(x) * w (w fp32: [D], or one number) -> out_h; out_conv = h + causal convolution of h over time per channel (conv_w fp32
    [taps, D], tap-major, the oldest tap first; the last taps - 1 rows h of every sequence are kept in state fp32 [slots, taps - 1, D]; the batch says which rows continue which
    sequence).  conv_w None: a bare norm.  x fp32 [rows, D]; outputs bf16 or fp32 (either may be None)."""
    rows, D = x.shape
    assert x.dtype == torch.float32 and x.is_contiguous() and w.dtype == torch.float32 and w.numel() in (1, D) and w.is_contiguous()
    outs = [o for o in (out_h, out_conv) if o is not None]
    assert outs and all(o.is_contiguous() and o.shape == x.shape and o.dtype == outs[0].dtype for o in outs)
    taps = 0
    if conv_w is not None:
        assert conv_w.dtype == torch.float32 and conv_w.is_contiguous() and conv_w.shape[1] == D and out_conv is not None
        taps = conv_w.shape[0]
        if taps > 1:
            assert state is not None and state.dtype == torch.float32 and state.is_contiguous() and tuple(state.shape[1:]) == (taps - 1, D)
            assert b is not None and b.T == rows
    ent = (b.row_entry.data_ptr(), b.row0.data_ptr(), b.n.data_ptr(), b.ctx.data_ptr(), b.slot.data_ptr()) if taps > 1 else (0, 0, 0, 0, 0)
    _lib.check(_lib.lib().pg_rmsnorm_conv(x.data_ptr(), w.data_ptr(), int(w.numel() == 1 and D != 1), _lib.ptr(conv_w), taps, _lib.ptr(state) if taps > 1 else 0,
                                          _lib.ptr(out_h), _lib.ptr(out_conv), *ent, rows, b.E if taps > 1 else 0, D, float(eps), int(outs[0].dtype == torch.float32), _lib.stream()),
               "pg_rmsnorm_conv")


def polynorm(z, coef, out, eps):
    """out = a N(z) + b N(z^2) + c N(z^3) + e per row, N(v) = v / sqrt(mean(v^2) + eps), (a, b, c, e) = coef (fp32 [4], device)."""
    rows, F = z.shape
    assert z.dtype == out.dtype and out.shape == z.shape and z.stride(1) == 1 and out.stride(1) == 1 and coef.dtype == torch.float32 and coef.numel() == 4
    _lib.check(_lib.lib().pg_polynorm(z.data_ptr(), z.stride(0), coef.data_ptr(), out.data_ptr(), out.stride(0), rows, F, float(eps),
                                      int(z.dtype == torch.float32), _lib.stream()), "pg_polynorm")
    return out


def sigmoid_gate_mul(y, gate):
    """y[t, c] *= sigmoid(gate[t, c]) in place (one type; any row pitch)."""
    rows, n = y.shape
    assert gate.shape == y.shape and gate.dtype == y.dtype and y.stride(1) == 1 and gate.stride(1) == 1
    _lib.check(_lib.lib().pg_sigmoid_gate_mul(y.data_ptr(), y.stride(0), gate.data_ptr(), gate.stride(0), rows, n, int(y.dtype == torch.float32),
                                              _lib.stream()), "pg_sigmoid_gate_mul")
    return y


GLU_SILU, GLU_CLAMPED, GLU_RELU = 1, 2, 3


def glu(gu, out, kind, limit=0.0, alpha=1.0):
    """out[t, f] from the [gate | up] product gu [rows, 2F]: GLU_SILU silu(g) * u; GLU_RELU relu(g) * u; GLU_CLAMPED min(g, limit) * sigmoid(alpha * .) * (clamp(u) + 1)."""
    rows, F = out.shape
    assert gu.shape[1] == 2 * F and gu.dtype == out.dtype and gu.stride(1) == 1 and out.stride(1) == 1
    _lib.check(_lib.lib().pg_glu(gu.data_ptr(), gu.stride(0), out.data_ptr(), out.stride(0), rows, F, int(kind), float(limit), float(alpha),
                                 int(out.dtype == torch.float32), _lib.stream()), "pg_glu")
    return out


def embed_rows(tokens, table, col0, D, scale, out_act=None):
    """fp32 rows [tokens, D]; out_act (the table's type, [tokens, D]) receives a copy."""
    out = torch.empty(tokens.numel(), D, device="cuda", dtype=torch.float32)
    assert out_act is None or (out_act.dtype == table.dtype and out_act.is_contiguous() and out_act.shape == out.shape)
    _lib.check(_lib.lib().pg_embed_rows(tokens.data_ptr(), table.data_ptr(), table.stride(0), int(col0), out.data_ptr(), _lib.ptr(out_act), tokens.numel(), D,
                                        float(scale), int(table.dtype == torch.float32), _lib.stream()), "pg_embed_rows")
    return out


def group_rmsnorm_add(y, w, x, out_act, groups, eps, clear=False):
    """x += gnorm(y) * w (x fp32, in place; x None: bare norm); out_act (bf16 / fp32, may be None) gets a copy of the result; clear: y becomes zero."""
    rows, D = y.shape
    assert y.dtype == torch.float32 and y.stride(1) == 1 and w.dtype == torch.float32 and w.numel() == D
    assert x is None or (x.dtype == torch.float32 and x.is_contiguous() and x.shape == y.shape)
    assert out_act is None or (out_act.is_contiguous() and out_act.shape == y.shape)
    fn = _lib.lib().pg_group_rmsnorm_add_clear if clear else _lib.lib().pg_group_rmsnorm_add
    _lib.check(fn(y.data_ptr(), y.stride(0), w.data_ptr(), _lib.ptr(x), _lib.ptr(out_act), rows, D, int(groups),
                                               float(eps), int(out_act is not None and out_act.dtype == torch.float32), _lib.stream()),
               "pg_group_rmsnorm_add")


def rmsnorm_gate(o, w, gate, out, eps):
    rows, D = o.shape
    assert o.dtype == torch.float32 and o.is_contiguous() and gate.dtype == out.dtype and out.is_contiguous() and gate.stride(1) == 1
    _lib.check(_lib.lib().pg_rmsnorm_gate(o.data_ptr(), w.data_ptr(), gate.data_ptr(), gate.stride(0), out.data_ptr(), rows, D, float(eps),
                                          int(out.dtype == torch.float32), _lib.stream()), "pg_rmsnorm_gate")


def geglu(gu, out):
    rows, F = out.shape
    assert gu.shape[1] == 2 * F and gu.dtype == out.dtype
    _lib.check(_lib.lib().pg_geglu(gu.data_ptr(), gu.stride(0), out.data_ptr(), out.stride(0), rows, F, int(out.dtype == torch.float32),
                                   _lib.stream()), "pg_geglu")


def side_gate(z, tokens, table, col0, out, n):
    rows, n_pad = out.shape
    assert z.dtype == torch.float32 and out.dtype == table.dtype
    _lib.check(_lib.lib().pg_side_gate(z.data_ptr(), z.stride(0), tokens.data_ptr(), table.data_ptr(), table.stride(0), int(col0), out.data_ptr(),
                                       out.stride(0), rows, int(n), n_pad, int(out.dtype == torch.float32), _lib.stream()), "pg_side_gate")


def token_side_fits(rows, D, n_pad, dtype):
    """The line up to which the side input is one launch: every row reads the weights from L2 for itself, so its four CTAs a row have to be one wave (two CTAs per SM
    in bf16, one in fp32) and a weight row short.  2048 wide, 64 inner values, separate / one launch in us: bf16 1 row 9.3 / 5.9, 48 rows 10.7 / 7.8, 96 rows 12.0 / 14.0;
    fp32 5 rows 9.7 / 7.3, 48 rows 14.2 / 13.8, 96 rows 14.5 / 20.8; 4096 wide fp32, 1 row 9.7 / 10.8."""
    f32 = dtype == torch.float32
    return rows <= (32 if f32 else 64) and D % 256 == 0 and D <= (2048 if f32 else 4096) and n_pad <= 256


def token_side(act, w_gate, tokens, table, col0, n, w_proj, norm_w, x, out_act, eps):
    """x += rms-norm(w_proj (gelu_tanh(w_gate act) * table[token, col0 : col0 + n])) * norm_w in one launch; out_act (bf16 models) receives a copy of x."""
    rows, D = x.shape
    n_pad = w_gate.shape[0]
    assert act.is_contiguous() and act.shape == x.shape and x.is_contiguous() and x.dtype == torch.float32 and x.is_cuda and act.is_cuda
    assert act.dtype == w_gate.dtype == w_proj.dtype == table.dtype and w_gate.is_contiguous() and w_proj.is_contiguous() and w_proj.shape == (D, n_pad)
    assert norm_w.dtype == torch.float32 and norm_w.is_contiguous() and norm_w.numel() == D and table.stride(1) == 1 and tokens.numel() == rows
    assert out_act is None or (out_act.is_contiguous() and out_act.shape == x.shape and out_act.dtype == act.dtype)
    _lib.check(_lib.lib().pg_token_side(act.data_ptr(), w_gate.data_ptr(), tokens.data_ptr(), table.data_ptr(), table.stride(0), int(col0), w_proj.data_ptr(),
                                        norm_w.data_ptr(), x.data_ptr(), _lib.ptr(out_act), rows, D, int(n), n_pad, float(eps), int(act.dtype == torch.float32),
                                        _lib.stream()), "pg_token_side")


NORM_PROJECTION = "projection"  # attn_prepare: one norm over all of q, one over all of k


def attn_prepare(qkv, b: StepBatch, freq, q_norm, k_norm, q_out, k_pages, v_pages, H, G, dim, vdim, rot_dims, eps, page, norm_qk=True, norm_v=True,
                 v_from_k=False, rot_gain=1.0, v_other=None, v_mix=0.0):
    """q_norm / k_norm None: norms without a weight; norm_qk / norm_v False: no q/k norm / no value norm; k_pages and v_pages None: the
    rows hold queries only (the layer attends over another layer's cache); v_from_k: the rows have no value columns, the values are the
    keys as projected (before norm and rotation); norm_qk NORM_PROJECTION: the norms run over all heads at once (weights of that size);
    rot_gain multiplies cosines and sines; v_other [T, G * vdim]: the values become (1 - v_mix) v + v_mix v_other.
    k_pages and v_pages may be QuantizedPages: the rows are quantised as they are written."""
    for w, heads in ((q_norm, H), (k_norm, G)):
        assert w is None or (w.dtype == torch.float32 and w.is_contiguous() and w.numel() == (heads * dim if norm_qk is NORM_PROJECTION else dim))
    assert v_other is None or (v_other.dtype == qkv.dtype and v_other.stride(1) == 1 and v_other.shape == (b.T, G * vdim))
    assert qkv.stride(1) == 1 and freq.dtype == torch.float64 and qkv.dtype == q_out.dtype and (k_pages is None) == (v_pages is None)
    mode = 2 if norm_qk is NORM_PROJECTION else int(bool(norm_qk))
    if isinstance(k_pages, QuantizedPages) or isinstance(v_pages, QuantizedPages):
        _check_quantized(k_pages, v_pages, G, dim, vdim, page)
        _on_current_device(qkv)
        assert q_out.is_contiguous()
        a = _lib.PREPARE_E4M3.pack(qkv.data_ptr(), qkv.stride(0), b.pos.data_ptr(), _lib.ptr(b.at), b.row_entry.data_ptr(), b.page_table.data_ptr(), freq.data_ptr(),
                                   _lib.ptr(q_norm), _lib.ptr(k_norm), q_out.data_ptr(), k_pages.codes.data_ptr(), k_pages.powers.data_ptr(), v_pages.codes.data_ptr(),
                                   v_pages.powers.data_ptr(), _lib.ptr(v_other), 0 if v_other is None else v_other.stride(0), b.max_pages, page, b.T, H, G, dim, vdim, rot_dims,
                                   mode, bool(norm_v), bool(v_from_k), qkv.dtype == torch.float32, eps, rot_gain, v_mix)
        _lib.check(_lib.lib().pg_attn_prepare_e4m3(a, _lib.stream()), "pg_attn_prepare_e4m3")
        return
    assert k_pages is None or k_pages.dtype == qkv.dtype
    _lib.check(_lib.lib().pg_attn_prepare_at(qkv.data_ptr(), qkv.stride(0), b.pos.data_ptr(), _lib.ptr(b.at), b.row_entry.data_ptr(), b.page_table.data_ptr(),
                                             b.max_pages, page, freq.data_ptr(), _lib.ptr(q_norm), _lib.ptr(k_norm), q_out.data_ptr(), _lib.ptr(k_pages), _lib.ptr(v_pages),
                                             b.T, H, G, dim, vdim, rot_dims, float(eps), mode, int(bool(norm_v)), int(bool(v_from_k)), float(rot_gain), _lib.ptr(v_other),
                                             0 if v_other is None else v_other.stride(0), float(v_mix), int(qkv.dtype == torch.float32), _lib.stream()), "pg_attn_prepare_at")


# ---- the 8-bit cache -------------------------------------------------------------------------------------------------
class QuantizedPages:
    """One operand (keys or values) of a layer's paged cache in 8 bits: e4m3 codes uint8 [pages, page, heads * size] and one power of two per row and head,
    2^(byte - 127), uint8 [pages, heads, page] -- the least that takes the head's largest finite element to 448 or below.  An element is code * power; what
    is not finite is kept as NaN.  `attn_prepare` writes them, `attn_ragged` and `attn_tree` read them, `kv_read` gives rows back in an activation type."""

    __slots__ = ("codes", "powers", "pages", "page", "heads", "size")

    def __init__(self, codes: torch.Tensor, powers: torch.Tensor):
        if codes.dtype != torch.uint8 or powers.dtype != torch.uint8 or codes.dim() != 3 or powers.dim() != 3:
            raise ValueError("8-bit pages are uint8 codes [pages, page, heads * size] and uint8 powers [pages, heads, page]")
        pages, page, width = codes.shape
        pages2, heads, page2 = powers.shape
        if pages != pages2 or page != page2 or heads < 1 or width % heads or not (codes.is_contiguous() and powers.is_contiguous()):
            raise ValueError(f"8-bit pages that do not belong together: codes {tuple(codes.shape)}, powers {tuple(powers.shape)}")
        self.codes, self.powers, self.pages, self.page, self.heads, self.size = codes, powers, pages, page, heads, width // heads

    @classmethod
    def empty(cls, pages: int, page: int, heads: int, size: int, device="cuda"):
        return cls(torch.zeros(pages, page, heads * size, device=device, dtype=torch.uint8), torch.zeros(pages, heads, page, device=device, dtype=torch.uint8))


def _check_quantized(k: "QuantizedPages", v: "QuantizedPages", G, dim, vdim, page):
    if not isinstance(k, QuantizedPages) or not isinstance(v, QuantizedPages):
        raise ValueError("keys and values are kept in one form: both in 8 bits or neither")
    if dim % 16 or vdim % 16 or dim > 256 or vdim > 256:
        raise ValueError(f"the 8-bit cache keeps heads of a multiple of 16 elements up to 256: got {dim} and {vdim}")
    if k.heads != G or v.heads != G or k.size != dim or v.size != vdim or k.page != page or v.page != page:
        raise ValueError(f"8-bit pages of {k.heads} / {v.heads} heads of {k.size} / {v.size} and {k.page} / {v.page} rows for {G} heads of {dim} / {vdim} and pages of {page}")


def kv_read(k_pages: "QuantizedPages", v_pages: "QuantizedPages", b: StepBatch, dtype: torch.dtype):
    """Keys and values of every entry with several new tokens, stored and new, in `dtype` (bf16 / fp32): [dense_rows, heads * size] each, in the dense scratch
    layout of the batch (read through b.dense_pages); zeros behind an entry's last row."""
    if not isinstance(k_pages, QuantizedPages) or not isinstance(v_pages, QuantizedPages):
        raise ValueError("kv_read reads 8-bit pages")
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("rows come back as torch.bfloat16 or torch.float32")
    G, page, dim, vdim = k_pages.heads, k_pages.page, k_pages.size, v_pages.size
    _check_quantized(k_pages, v_pages, G, dim, vdim, page)
    _on_current_device(k_pages.codes)
    k = torch.empty(b.dense_rows, G * dim, device=k_pages.codes.device, dtype=dtype)
    v = torch.empty(b.dense_rows, G * vdim, device=k_pages.codes.device, dtype=dtype)
    if b.dense_rows:
        a = _lib.READ_E4M3.pack(k_pages.codes.data_ptr(), k_pages.powers.data_ptr(), v_pages.codes.data_ptr(), v_pages.powers.data_ptr(), b.page_table.data_ptr(),
                                b.dense_row0.data_ptr(), b.n.data_ptr(), b.ctx.data_ptr(), k.data_ptr(), v.data_ptr(), b.max_pages, page, b.E, b.dense_max_len, G, dim, vdim,
                                dtype == torch.float32)
        _lib.check(_lib.lib().pg_kv_read_e4m3(a, _lib.stream()), "pg_kv_read_e4m3")
    return k, v


class ScoreOptions:
    """The optional parts of a softmax attention's score and mask, as the kernels read them (PgAttnScore): a sliding window of
    `window` keys (None: all) that keeps the first `keep_first` keys of the sequence visible, a per-head sink logit in the softmax
    denominator, a penalty dist_a[h] * log(1 + dist_b[h] * distance), a per-head score multiplier.  logistic: no softmax -- a visible
    key weighs sigmoid(score + head_bias[h]), unnormalised.  out_scale multiplies the output, whose rows are out_ld elements apart
    (0: dense).  Tensors: fp32 [H] on the device."""

    def __init__(self, heads, window=None, keep_first=0, sink=None, dist_a=None, dist_b=None, head_scale=None, logistic=False, head_bias=None,
                 out_scale=1.0, out_ld=0):
        for t in (sink, dist_a, dist_b, head_scale, head_bias):
            assert t is None or (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous() and t.numel() == heads)
        assert (dist_a is None) == (dist_b is None)
        self.window = int(window) if window else 0
        self.keep_first = int(keep_first) if self.window else 0
        self._keep = (sink, dist_a, dist_b, head_scale, head_bias)  # the struct holds raw pointers
        assert not logistic or sink is None
        self.logistic, self.out_scale, self.out_ld = bool(logistic), float(out_scale), int(out_ld)
        # nothing but a plain sliding window
        self.window_only = (sink is None and dist_a is None and head_scale is None and not self.keep_first and not logistic and self.out_scale == 1.0
                            and not self.out_ld)
        self.c = _lib.AttnScore(self.window, self.keep_first, _lib.ptr(sink), _lib.ptr(dist_a), _lib.ptr(dist_b), _lib.ptr(head_scale), int(self.logistic),
                                _lib.ptr(head_bias), self.out_scale, self.out_ld)

    def visible_keys(self, context):
        """Upper bound of the keys a query at position `context` reads."""
        return context + 1 if not self.window else min(context + 1, self.window + self.keep_first)


# head sizes (dim, vdim) the tensor-core attention kernel is instantiated for
MMA_HEAD_SIZES = {(32, 32), (64, 64), (128, 128), (64, 128), (128, 64), (96, 64), (192, 128)}


# (row width, value width) of a one-row-per-token cache the tensor-core decode kernel is instantiated for
LATENT_MMA_SIZES = {(96, 64), (160, 128), (192, 128), (288, 256), (544, 512), (576, 512)}


def attn_ragged(q, k_pages, v_pages, gate, out, b: StepBatch, H, G, dim, vdim, scale, softcap, page, decode_kernel=True, tensor_cores=True,
                krow=0, vrow=0, gate_per_head=False, only_singles=False, skip_singles=False, score: Optional["ScoreOptions"] = None):
    """Entries with several new rows go to a tiled kernel -- on the tensor cores for bf16 activations and the usual head
    sizes (fp32 probabilities as three bf16 terms), plain fp32 FMAs otherwise -- and entries with ONE new row (decoded tokens)
    to the key-split kernel (`decode_kernel=False`: everything through the tiled kernel).  Same arithmetic, other summation
    order.  krow / vrow: elements per cache row when it is not G * dim / G * vdim (a latent cache: one row is key and value);
    gate_per_head: the gate holds one scalar per head instead of one per output element; only_singles / skip_singles: rows of
    entries with several new tokens / with one new token are left alone (another form computes them).  score: window, sink, distance
    penalty and per-head multiplier (ScoreOptions; None: plain causal attention).
    Pages in 8 bits (QuantizedPages): decoded tokens read the codes, entries with several new rows go over rows read back (kv_read).  A batch of drafted trees:
    attn_tree."""
    import ctypes as C
    if b.tree is not None:
        if krow or vrow or only_singles or skip_singles:
            raise ValueError("drafted trees go over a cache of one key row and one value row a token, all entries in one call")
        return attn_tree(q, k_pages, v_pages, gate, out, b, H, G, dim, vdim, scale, softcap, page, gate_per_head=gate_per_head, score=score)
    if isinstance(k_pages, QuantizedPages) or isinstance(v_pages, QuantizedPages):
        _check_quantized(k_pages, v_pages, G, dim, vdim, page)
        if krow or vrow:
            raise ValueError("8-bit pages have rows of their own width")
        if b.singles < b.E and not only_singles:
            k, v = kv_read(k_pages, v_pages, b, q.dtype)
            attn_ragged(q, k, v, gate, out, dense_view(b), H, G, dim, vdim, scale, softcap, 64, decode_kernel, tensor_cores, gate_per_head=gate_per_head, skip_singles=True,
                        score=score)  # (the scratch's pages hold 64 rows, whatever the cache's do)
        if b.singles and not skip_singles:
            _attn_rows(q, k_pages, v_pages, gate, out, b, H, G, dim, vdim, scale, softcap, page, gate_per_head, score, singles=True)
        return
    L, f32 = _lib.lib(), int(q.dtype == torch.float32)
    sx = C.addressof(score.c) if score is not None else 0
    reach = score.visible_keys(b.max_single_ctx) if score is not None else b.max_single_ctx + 1  # keys a decoded token reads at most
    ldg = 0 if gate is None else gate.stride(0)
    gph = int(bool(gate_per_head))
    singles = b.singles if (decode_kernel or skip_singles) else 0
    dense_rows = krow in (0, G * dim) and vrow in (0, G * vdim)
    if only_singles:
        pass
    elif (singles < b.E and tensor_cores and not f32 and dense_rows and (dim, vdim) in MMA_HEAD_SIZES
            and (gate is None or gph or (ldg % 2 == 0 and gate.data_ptr() % 4 == 0))):
        _lib.check(L.pg_attn_ragged_mma_sized(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _lib.ptr(gate), ldg, out.data_ptr(), b.row0.data_ptr(),
                                        b.n.data_ptr(), b.ctx.data_ptr(), b.page_table.data_ptr(), b.max_pages, page, b.E, b.max_n, H, G, dim, vdim,
                                        float(scale), float(softcap or 0.0), int(singles > 0), gph, b.E - singles, b.dense_max_len, sx, _lib.stream()),
                   "pg_attn_ragged_mma_sized")
    elif singles < b.E:
        _lib.check(L.pg_attn_ragged(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _lib.ptr(gate), ldg, out.data_ptr(), b.row0.data_ptr(),
                                    b.n.data_ptr(), b.ctx.data_ptr(), b.page_table.data_ptr(), b.max_pages, page, b.E, b.max_n, H, G, dim, vdim,
                                    float(scale), float(softcap or 0.0), int(singles > 0), f32, int(krow), int(vrow), gph, sx, _lib.stream()),
                   "pg_attn_ragged")
    latent = (k_pages.data_ptr() == v_pages.data_ptr() and G == 1 and krow == vrow == dim and k_pages.shape[-1] == dim)
    if (singles and not skip_singles and latent and tensor_cores and not f32 and (dim, vdim) in LATENT_MMA_SIZES and softcap in (0, 0.0, None)
            and (gate is None or gph) and (score is None or score.window_only)):
        # one-row-per-token cache, every head of a token against the same key tile: tensor cores
        window = score.window if score is not None else 0
        tiles = b.max_single_ctx // 64 + 1
        if window:
            tiles = min(tiles, (window + 62) // 64 + 1)  # a window of w keys touches at most this many 64-key tiles
        vs = 2 if vdim > 256 else 1  # value halves are CTAs of their own
        nsplit = max(1, min(tiles, (4 * _lib.num_sms()) // (singles * -(-H // 64) * vs), 32))  # measured: 4 CTAs per SM beat 2 despite the larger merge
        partial = torch.empty(b.E * H * nsplit * (vdim + 2), device="cuda", dtype=torch.float32) if nsplit > 1 else None
        _lib.check(L.pg_attn_latent_decode_mma(q.data_ptr(), k_pages.data_ptr(), _lib.ptr(gate), ldg, out.data_ptr(), _lib.ptr(partial), b.row0.data_ptr(),
                                               b.n.data_ptr(), b.ctx.data_ptr(), b.page_table.data_ptr(), b.max_pages, page, b.E, nsplit, H, dim, vdim,
                                               float(scale), int(window), _lib.stream()), "pg_attn_latent_decode_mma")
        if nsplit > 1:
            _lib.check(L.pg_attn_decode_merge(partial.data_ptr(), _lib.ptr(gate), ldg, out.data_ptr(), b.row0.data_ptr(), b.n.data_ptr(), b.E, nsplit, H,
                                              vdim, gph, 0, 0, _lib.stream()), "pg_attn_decode_merge")
    elif singles and not skip_singles:
        tiles = (reach - 1) // 32 + 1
        # three CTAs of four warps per SM at once: what one wave holds, and at least two 32-key tiles for every warp.  The general kernel has eight warps and two CTAs an SM, and
        # takes the same split: us, this / two waves of CTAs with two tiles a warp, bf16 128 / 256 64 x 2250 318 / 347, 1 x 3000 89 / 134; fp32 latent 288 / 256 5 x 1100
        # 681 / 1099, 1 x 3000 795 / 1307
        nsplit = max(1, min(3 * _lib.num_sms() // (G * singles), tiles // 8, 32))
        partial = torch.empty(b.E * H * nsplit * (vdim + 2), device="cuda", dtype=torch.float32) if nsplit > 1 else None
        _lib.check(L.pg_attn_decode(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _lib.ptr(gate), ldg, out.data_ptr(), _lib.ptr(partial),
                                    b.row0.data_ptr(), b.n.data_ptr(), b.ctx.data_ptr(), b.page_table.data_ptr(), b.max_pages, page, b.E, nsplit,
                                    H, G, dim, vdim, float(scale), float(softcap or 0.0), f32, int(krow), int(vrow), gph, sx, _lib.stream()),
                   "pg_attn_decode")


def _attn_rows(q, k_pages, v_pages, gate, out, b: StepBatch, H, G, dim, vdim, scale, softcap, page, gate_per_head, score, singles):
    if dim > 128 or vdim > 128:
        raise ValueError(f"attention of a few rows takes heads of up to 128 elements: got {dim} and {vdim}")
    if q.dtype not in (torch.bfloat16, torch.float32) or out.dtype != q.dtype or (gate is not None and (gate.dtype != q.dtype or gate.stride(-1) != 1)):
        raise ValueError("queries, gate and output share a type, torch.bfloat16 or torch.float32")
    if q.numel() != b.T * H * dim or not q.is_contiguous() or out.stride(-1) != 1 or H % G:
        raise ValueError("queries are [rows, heads * size], heads a multiple of the key / value heads")
    wide = H * vdim
    pitch = score.out_ld if score is not None and score.out_ld else wide
    if not (out.is_contiguous() and out.numel() == b.T * wide and pitch == wide) and (
            out.dim() != 2 or out.shape[0] != b.T or out.shape[1] < wide or (b.T > 1 and out.stride(0) != pitch)):
        raise ValueError(f"the output's rows are {wide} elements, {pitch} apart: got {tuple(out.shape)} with strides {out.stride()}")
    if gate is not None and (gate.dim() != 2 or gate.shape[0] < b.T or gate.shape[1] < (H if gate_per_head else wide)):
        raise ValueError(f"the gate has one number for every {'head' if gate_per_head else 'output'} of every row: got {tuple(gate.shape)}")
    import ctypes as C
    _on_current_device(q)
    quantized = isinstance(k_pages, QuantizedPages)
    tree = None if singles else b.tree
    kv = ((k_pages.codes.data_ptr(), v_pages.codes.data_ptr(), k_pages.powers.data_ptr(), v_pages.powers.data_ptr()) if quantized else
          (k_pages.data_ptr(), v_pages.data_ptr(), 0, 0))
    a = _lib.ATTN_ROWS.pack(q.data_ptr(), *kv, 0 if gate is None else gate.data_ptr(), 0 if gate is None else gate.stride(0), out.data_ptr(), b.row0.data_ptr(), b.n.data_ptr(),
                            b.ctx.data_ptr(), b.page_table.data_ptr(), b.pos.data_ptr(), 0 if tree is None else tree.data_ptr(), 0 if score is None else C.addressof(score.c),
                            b.max_pages, page, 0 if tree is None else tree.shape[1], b.E, b.T, b.max_n, b.singles if singles else b.E,
                            b.max_single_ctx + 1 if singles else max(b.max_single_ctx + 1, b.dense_max_len), singles, H, G, dim, vdim, q.dtype == torch.float32, quantized,
                            bool(gate_per_head), scale, softcap or 0.0)
    L = _lib.lib()
    need = L.pg_attn_rows_scratch(a)
    scratch = torch.empty(need, device=q.device, dtype=torch.uint8) if need > 0 else None
    _lib.check(L.pg_attn_rows(a, 0 if scratch is None else scratch.data_ptr(), need, _lib.stream()), "pg_attn_rows")


def attn_tree(q, k_pages, v_pages, gate, out, b: StepBatch, H, G, dim, vdim, scale, softcap, page, gate_per_head=False, score: Optional["ScoreOptions"] = None):
    """Attention of drafted trees (b.tree; None: chains): every new row sees all stored keys of its entry and the drafted rows in its mask, softmax, gate and score
    options as attn_ragged; windows and distances go by b.pos.  The drafted rows' keys and values are in the cache already (attn_prepare with b.at).  The cache:
    pages of q's type or QuantizedPages.  Heads of up to 128 elements in whole 16-byte pieces, pages of 32, 64, 128 .. rows.  A row whose mask is empty and
    whose entry has nothing stored gets zeros."""
    if isinstance(k_pages, QuantizedPages) or isinstance(v_pages, QuantizedPages):
        _check_quantized(k_pages, v_pages, G, dim, vdim, page)
    elif k_pages.dtype != q.dtype or v_pages.dtype != q.dtype:
        raise ValueError("a cache that is not in 8 bits has the queries' type")
    elif k_pages.shape[1:] != (page, G * dim) or v_pages.shape[1:] != (page, G * vdim) or not k_pages.is_contiguous() or not v_pages.is_contiguous():
        raise ValueError(f"pages of {tuple(k_pages.shape)} and {tuple(v_pages.shape)} for {G} heads of {dim} / {vdim} and pages of {page} rows")
    if b.tree is not None and (b.tree.dtype != torch.int32 or b.tree.dim() != 2 or b.tree.shape[0] != b.T or not b.tree.is_contiguous()):
        raise ValueError("masks are int32 [rows, words]")
    _attn_rows(q, k_pages, v_pages, gate, out, b, H, G, dim, vdim, scale, softcap, page, gate_per_head, score, singles=False)


# ---- rows of the cache from one place to another -----------------------------------------------------------------------
class CachePages:
    """The paged operands of a cache, all layers together, as `copy_pages` and `keep_rows` take them: tensors [pages, page, width] of any type and QuantizedPages.
    Made once for a cache: a table of where they lie is kept on the device."""

    def __init__(self, operands: Sequence, page: int):
        flat = []
        for o in operands:
            flat += [(o.codes, 0), (o.powers, o.heads)] if isinstance(o, QuantizedPages) else [(o, 0)]
        if not flat:
            raise ValueError("a cache has at least one operand")
        if len(flat) > 65535:
            raise ValueError(f"at most 65535 operands: got {len(flat)}")
        if len({t.data_ptr() for t, _ in flat}) != len(flat):
            raise ValueError("an operand is named twice: its rows would move twice")
        self.operands, self.page, self.pages, self.device = list(operands), int(page), flat[0][0].shape[0], flat[0][0].device
        table, self.most_page_bytes, self.most_columns = b"", 0, 0
        for t, heads in flat:
            if t.dim() != 3 or not t.is_contiguous() or t.shape[0] != self.pages or t.shape[2 if heads else 1] != page or t.numel() == 0:
                raise ValueError(f"operands are dense [pages, {page}, width] of {self.pages} pages: got {tuple(t.shape)}")
            if not t.is_cuda or t.device != self.device:
                raise ValueError("the operands of a cache lie on one device")
            row = t.shape[2] * t.element_size()
            unit = next(u for u in (16, 4, 2, 1) if (row | t.data_ptr()) % u == 0)
            if row * page >= 1 << 31:
                raise ValueError("a page has less than 2 GB")
            self.most_page_bytes = max(self.most_page_bytes, t.stride(0) * t.element_size())
            self.most_columns = max(self.most_columns, heads or row // unit)
            table += _lib.PAGE_OPERAND.pack(t.data_ptr(), t.stride(0) * t.element_size(), row, heads, unit, self.pages)
        self.count = len(flat)
        self.table = torch.frombuffer(bytearray(table), dtype=torch.uint8).to(self.device)

    def __reduce__(self):  # (a copy's table says where the copies lie)
        return type(self), (self.operands, self.page)


def copy_pages(cache: CachePages, moves):
    """moves: whole numbers [n, 3] on the host, (source page, destination page, rows): the first `rows` rows of the source page go to the destination page, in every
    operand.  No destination is another move's source or destination."""
    moves = np.asarray(moves)
    if moves.size == 0:
        return
    if moves.ndim != 2 or moves.shape[1] != 3 or moves.dtype.kind not in "iu":
        raise ValueError("moves are (source page, destination page, rows)")
    n = len(moves)
    if n <= 32:  # (a few numbers are looked over faster one by one)
        rows = moves.tolist()
        inside = all(0 <= a < cache.pages and 0 <= b < cache.pages and 0 <= r <= cache.page for a, b, r in rows)
        to = {b for _, b, _ in rows}
        apart = len(to) == n and not any(a in to for a, _, _ in rows)
    else:
        most = moves.max(0).tolist()
        inside = moves.min() >= 0 and most[0] < cache.pages and most[1] < cache.pages and most[2] <= cache.page
        to = set(moves[:, 1].tolist())
        apart = len(to) == n and to.isdisjoint(moves[:, 0].tolist())
    if not inside:
        raise IndexError(f"moves go between pages 0 .. {cache.pages - 1} and take up to {cache.page} rows")
    if not apart:
        raise ValueError("a page that is copied to is no other move's source or destination")
    _on_current_device(cache.table)
    moves = moves.astype(np.int32)
    _lib.check(_lib.lib().pg_copy_pages(cache.table.data_ptr(), cache.count, cache.page, cache.most_page_bytes, moves.tobytes(), n, _lib.stream()), "pg_copy_pages")


def keep_rows(cache: CachePages, b: StepBatch, path: torch.Tensor, kept: torch.Tensor):
    """The drafted rows path[e, :kept[e]] of every entry (int32 [entries, width] and [entries] on the device, `verify_drafts`' outputs) move together behind the entry's stored
    rows, in every operand: cache row ctx + i takes row ctx + path[e, i].  Paths ascend (a token stands behind the one it follows); numbers outside the entry's rows are
    skipped."""
    if path.dtype != torch.int32 or path.dim() != 2 or path.shape[0] != b.E or not path.is_contiguous() or path.shape[1] < 1:
        raise ValueError("paths are int32 [entries, width]")
    if kept.dtype != torch.int32 or kept.shape != (b.E,) or not kept.is_contiguous():
        raise ValueError("kept is int32 [entries]")
    if path.device != cache.device or kept.device != cache.device or b.page_table.device != cache.device:
        raise ValueError(f"paths, counts and page table lie on the cache's device, {cache.device}")
    _on_current_device(cache.table)
    a = _lib.KEEP_ROWS.pack(cache.table.data_ptr(), b.page_table.data_ptr(), b.n.data_ptr(), b.ctx.data_ptr(), path.data_ptr(), kept.data_ptr(), cache.count, cache.page,
                            cache.most_columns, b.max_pages, path.shape[1], b.E)
    _lib.check(_lib.lib().pg_keep_rows(a, _lib.stream()), "pg_keep_rows")


# ---- low-rank adapters of the step's requests -----------------------------------------------------------------------
ADAPTER_MOST_RANK, ADAPTER_MOST_PARTS = 128, 8


class AdapterBank:
    """The low-rank adapters that stand beside one shared projection [columns, K]: adapter s adds scale[s] * b[s] (a[s] x).  The projection's columns are `parts` runs
    (a joint query, key and value projection has three); each run has `rank` rows of a[s] for itself: a [slots, len(parts) * rank, K], b [slots, sum(parts), rank], both
    bf16 or fp32 on the device, scale fp32 [slots].  They are laid out anew, once; `put` replaces one.  (Parameters are taken as numbers: nothing here has gradients.)"""

    @torch.no_grad()
    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor, parts: Sequence[int]):
        parts = [int(n) for n in parts]
        if not 1 <= len(parts) <= ADAPTER_MOST_PARTS or min(parts) < 1:
            raise ValueError(f"1 .. {ADAPTER_MOST_PARTS} runs of at least one column: got {parts}")
        if a.dim() != 3 or b.dim() != 3 or a.dtype != b.dtype or a.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("a is [slots, parts * rank, K] and b [slots, columns, rank], both torch.bfloat16 or torch.float32")
        slots, rows, K = a.shape
        rank = b.shape[2]
        if slots < 1 or K < 1 or b.shape[0] != slots or b.shape[1] != sum(parts) or rows != len(parts) * rank or not 1 <= rank <= ADAPTER_MOST_RANK:
            raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} for runs of {parts} columns and a rank of 1 .. {ADAPTER_MOST_RANK}")
        if scale.dtype != torch.float32 or scale.shape != (slots,):
            raise ValueError("one fp32 factor for every adapter")
        if not a.is_cuda or b.device != a.device or scale.device != a.device:
            raise ValueError("adapters lie on one device")
        self.columns = (*parts, *(0,) * (ADAPTER_MOST_PARTS - len(parts)))
        self.parts, self.slots, self.rank, self.K, self.F, self.dtype, self.device = tuple(parts), slots, rank, K, sum(parts), a.dtype, a.device
        self.index = a.get_device()
        r8 = -(-rank // 8) * 8  # (ranks and depths in whole 16-byte pieces; zeros behind)
        self.rank8, self.scale = r8, scale.clone()
        if self.dtype == torch.bfloat16:  # blocks of 64 k's, see _pieces
            self.a = a.new_zeros(slots, -(-K // 64), -(-len(parts) * r8 // 16) * 16, 8, 8)
        else:
            self.a = a.new_zeros(slots, len(parts) * r8, -(-K // 8) * 8)
        self.b = b.new_zeros(slots, self.F, r8)
        for p in range(len(parts)):
            self._put_a(slice(None), p, a[:, p * rank:(p + 1) * rank])
        self.b[:, :, :rank] = b

    def _put_a(self, slot, part, a):
        """a [.., r, K] into rows of the run; bf16: [K / 64, rows, 8, 8], in row n the eight pieces of eight k's exchanged by n % 8, the matrix unit's operand layout."""
        r, here = a.shape[-2], slice(part * self.rank8, part * self.rank8 + a.shape[-2])
        if self.dtype != torch.bfloat16:
            self.a[slot, here, :self.K] = a
            return
        blocks = self.a.shape[1]
        wide = a.new_zeros(*a.shape[:-1], 64 * blocks)
        wide[..., :self.K] = a
        pieces = wide.unflatten(-1, (blocks, 8, 8)).movedim(-4, -3)  # [.., blocks, r, 8, 8]
        order = torch.arange(8, device=a.device) ^ (torch.arange(here.start, here.start + r, device=a.device) % 8)[:, None]
        self.a[slot, :, here] = pieces.gather(-2, order[..., None].expand(pieces.shape))

    @classmethod
    def empty(cls, slots: int, rank: int, K: int, parts: Sequence[int], dtype: torch.dtype, device="cuda"):
        return cls(torch.zeros(slots, len(parts) * rank, K, device=device, dtype=dtype), torch.zeros(slots, sum(parts), rank, device=device, dtype=dtype),
                   torch.zeros(slots, device=device), parts)

    @torch.no_grad()
    def put(self, slot: int, part: int, a: torch.Tensor, b: torch.Tensor):
        """One run's matrices of one adapter: a [r, K], b [columns of the run, r], r up to the bank's rank (the rest becomes zero)."""
        r = a.shape[0]
        if not 0 <= slot < self.slots or not 0 <= part < len(self.parts):
            raise IndexError(f"adapter {slot}, run {part} of {self.slots} adapters with {len(self.parts)} runs")
        if a.dim() != 2 or b.dim() != 2 or r > self.rank or a.shape[1] != self.K or tuple(b.shape) != (self.parts[part], r):
            raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} for {self.parts[part]} columns of a depth of {self.K} and a rank up to {self.rank}")
        col = sum(self.parts[:part])
        full = torch.zeros(self.rank8, self.K, device=self.device, dtype=self.dtype)
        full[:r] = a.to(self.device, self.dtype)
        self._put_a(slot, part, full)
        there = self.b[slot, col:col + self.parts[part]]
        there.zero_()
        there[:, :r] = b.to(self.device, self.dtype)

    def clear(self, slot: int):
        self.a[slot].zero_()
        self.b[slot].zero_()
        self.scale[slot] = 0


def _adapter_tile_rows(rows: int, adapters: int, processors: int) -> int:
    """Tiles of 128 rows go over the tensor memory, and their way is long: they pay once tiles of 16 are more than the processors, where adapters fill half of one on average.  A plan serves
    every projection of a step and does not know their ranks, by which the border moves both ways (K 2048, 2560 columns, us with 16 and 128: 7 adapters of 320 rows, rank 3 x 16 16 and 22,
    3 x 64 30 and 25; of 384 rows 24 and 22, 47 and 24; 48 of 64 rows 25 and 32, 60 and 38).  Projections that the tensor memory does not take (more runs or higher ranks than its operands have
    room for) run a tile of 128 as eight of 16, as long as those: four runs of rank 64 over 7 x 384 rows 94."""
    return 128 if rows > max(16 * processors, 64 * adapters - 1) else 16


class AdapterPlan:
    """Which rows of a step go through which adapter: entries of ns[e] rows, one behind the other, with adapters[e] (-1: none).  Rows of one adapter stand together in
    tiles, whichever entries they belong to.  tiles: a fixed number of them (a plan that is `fill`ed again, for a step that is captured).  tile_rows: how many rows a tile
    has at most, 16 or 128 (None: by the rows)."""

    def __init__(self, ns: Sequence[int], adapters: Sequence[int], device="cuda", tiles: Optional[int] = None, tile_rows: Optional[int] = None):
        if tile_rows not in (None, 16, 128):
            raise ValueError(f"tiles of 16 or 128 rows: got {tile_rows}")
        self.T, self.fixed, self._copied, self.host, self.tile_rows = 0, tiles, None, None, tile_rows
        self._make(ns, adapters, device)

    def _order(self, ns, adapters):
        ns, who = np.asarray(ns, dtype=np.int64), np.asarray(adapters, dtype=np.int64)
        if ns.ndim != 1 or ns.shape != who.shape or ns.size == 0 or ns.min() < 1:
            raise ValueError("one adapter (-1: none) for every entry, and entries of at least one row")
        if who.min() < -1:
            raise IndexError("adapters are 0 .. slots - 1, -1 for none")
        rows = np.repeat(who, ns)
        order = np.argsort(rows, kind="stable")
        rows = rows[order]
        first = np.concatenate([[0], np.flatnonzero(rows[1:] != rows[:-1]) + 1])
        return order, rows[first], first, np.diff(first, append=len(rows))

    def _make(self, ns, adapters, device):
        order, ids, first, count = self._order(ns, adapters)
        size = self.tile_rows or (16 if self.fixed is not None else _adapter_tile_rows(len(order), len(ids), _lib.num_sms() if torch.device(device).type == "cuda" else 148))
        tiles = [(a, f + o, min(size, c - o)) for a, f, c in zip(ids.tolist(), first.tolist(), count.tolist()) for o in range(0, c, size)]
        n = len(tiles) if self.fixed is None else self.fixed
        if len(tiles) > n:
            raise ValueError(f"{len(tiles)} tiles, room for {n}")
        T = len(order)
        if self.host is None:
            self.T, self.tile_rows, self.tile_count = T, size, n
            self.host = torch.zeros(T + 3 * n, dtype=torch.int32)
            if torch.device(device).type == "cuda":
                self.host = self.host.pin_memory()
            self.dev = torch.empty_like(self.host, device=device)
            self.rows, self.tiles, self.index = self.dev[:T], self.dev[T:], self.dev.get_device()
        elif T != self.T:
            raise ValueError(f"a plan of {self.T} rows is filled with {T}")
        h = self.host.numpy()
        h[:T] = order
        h[T:] = 0
        h[T:T + 3 * len(tiles)] = np.asarray(tiles).reshape(-1)
        self.most = int(ids[-1])
        self.dev.copy_(self.host, non_blocking=True)
        if self.fixed is not None and self.dev.is_cuda:
            self._copied = torch.cuda.Event()
            self._copied.record()

    def fill(self, ns: Sequence[int], adapters: Sequence[int]):
        """Other adapters for as many rows, at the same addresses."""
        if self.fixed is None:
            raise ValueError("only a plan with a fixed number of tiles is filled again")
        if self._copied is not None:
            self._copied.synchronize()  # the image before must have left the pinned buffer
        self._make(ns, adapters, self.dev.device)


def _rows_overlap(a, a_pitch, a_bytes, b, b_pitch, b_bytes, rows):
    """Whether two row matrices (where they begin, bytes from row to row, bytes of a row) have bytes in common; column slices that stand side by side in one matrix have none."""
    if a + (rows - 1) * a_pitch + a_bytes <= b or b + (rows - 1) * b_pitch + b_bytes <= a:
        return False
    d = (b - a) % a_pitch
    return a_pitch != b_pitch or d < a_bytes or a_pitch - d < b_bytes


def adapter_add(x: torch.Tensor, y: torch.Tensor, bank: AdapterBank, plan: AdapterPlan, out: Optional[torch.Tensor] = None, gain: float = 1.0):
    """out[t] = y[t] + gain * scale[s] * b[s] (a[s] x[t]) for the rows of adapter s, y[t] for those without (out None: y, in place).  x [rows, K] of the bank's type, y and
    out [rows, columns] bf16 or fp32 (fp32 beside fp32 adapters), unit last strides, any row pitch.  The sum over K and over the rank is fp32 (tiles of
    128 rows: the tensor cores' own, K / 16 additions that are cut off); y is added to it and rounded once.  A row of x that is not
    finite makes its own row of out NaN."""
    out = y if out is None else out
    T, K, F, dtype, index = plan.T, bank.K, bank.F, bank.dtype, bank.index
    if x.dtype != dtype or x.shape != (T, K):
        raise ValueError(f"x is [{T}, {K}] of {dtype}: got {tuple(x.shape)} of {x.dtype}")
    wide = y.dtype == torch.float32
    if not (wide or y.dtype == torch.bfloat16) or out.dtype != y.dtype or (dtype == torch.float32 and not wide):
        raise ValueError("y and out share a type, torch.bfloat16 or torch.float32; torch.float32 beside fp32 adapters")
    if y.shape != (T, F) or out.shape != (T, F):
        raise ValueError(f"y and out are [{T}, {F}]: got {tuple(y.shape)} and {tuple(out.shape)}")
    (lx, ux), (ly, uy), (lo, uo) = x.stride(), y.stride(), out.stride()
    if T == 1:
        lx, ly, lo = K, F, F
    if (ux != 1 and K > 1) or ((uy != 1 or uo != 1) and F > 1) or lx < K or ly < F or lo < F:
        raise ValueError("elements of a row stand side by side, rows do not overlap")
    if x.get_device() != index or y.get_device() != index or out.get_device() != index:
        raise ValueError(f"rows and adapters lie on one device: got {x.device}, {y.device}, {out.device} and {bank.device}")
    px, py, po, ex, ey = x.data_ptr(), y.data_ptr(), out.data_ptr(), 4 if dtype == torch.float32 else 2, 4 if wide else 2
    if _rows_overlap(po, lo * ey, F * ey, px, lx * ex, K * ex, T) or (not (lo == ly and po == py) and _rows_overlap(po, lo * ey, F * ey, py, ly * ey, F * ey, T)):
        raise ValueError("out is y or lies apart from it, and apart from x")
    if plan.most >= bank.slots:
        raise IndexError(f"adapter {plan.most} of {bank.slots}")
    if plan.index != index:
        raise ValueError(f"the plan lies on {plan.dev.device}, the adapters on {bank.device}")
    _on_current_device(bank.a)
    L = _lib.lib()

    def packed(shares):
        return _lib.ADAPTER.pack(px, py, bank.a.data_ptr(), bank.b.data_ptr(), po, bank.scale.data_ptr(), plan.rows.data_ptr(), plan.tiles.data_ptr(), shares, lx, ly, lo, *bank.columns,
                                 len(bank.parts), K, F, bank.rank8, bank.slots, plan.tile_count, plan.tile_rows, T, dtype == torch.float32, wide, gain)

    a, scratch = packed(0), None
    if plan.tile_rows > 16:
        need = L.pg_adapter_scratch(a)
        if need:
            scratch = torch.empty(need // 4, device=x.device, dtype=torch.float32)
            a = packed(scratch.data_ptr())
    _lib.check(L.pg_adapter_add(a, _lib.stream()), "pg_adapter_add")
    return out


# ---- verified drafts -------------------------------------------------------------------------------------------------
def _check_rows_of_logits(logits, b: StepBatch, what):
    if (logits.dim() != 2 or logits.dtype != torch.float32 or logits.stride(1) != 1 or not logits.is_cuda or logits.shape[0] != b.T
            or (b.T > 1 and logits.stride(0) < logits.shape[1])):
        raise ValueError(f"{what} are fp32 [rows of the step, vocab] on the device, entries of a row side by side: got {tuple(logits.shape)} of {logits.dtype} for {b.T} rows")


def verify_drafts(logits: torch.Tensor, b: StepBatch, uniforms: Optional[torch.Tensor] = None, draft_logits: Optional[torch.Tensor] = None, temperature: float = 1.0,
                  top_p: float = 1.0, draft_temperature: Optional[float] = None, draft_top_p: Optional[float] = None):
    """Which tokens of every entry's drafted tree (b.tokens, b.parents) stay, and the token behind them: (path int32 [entries, max_n], kept int32 [entries], next int32 [entries]).
    logits fp32 [rows, vocab] (any row pitch): row v of an entry says what follows token v.  The first row of an entry is its pending token, which stays: path[e, 0] = 0; rows below
    -1 are never reached.  path[e, :kept[e]] are the rows of the walk, -1 behind them.

    uniforms None: greedy -- the walk goes on at the first child that carries the row's first largest entry.  Else fp32 [rows, 2] from [0, 1), and a row's distribution is
    softmax(logits / temperature) cut to the tokens above which at most top_p of the mass lies (equal logits stay together).  Without draft_logits a token is drawn from it
    with uniforms[v, 1], the first id whose running sum is above that part of the whole, and the walk goes on at the first child that carries it.  draft_logits (as logits; row v:
    what v's children were drawn from, one after another, with draft_temperature and draft_top_p, the target's where they are None): child i stays with probability
    min(1, r / q) under uniforms[i, 0], r = p at first and the normalised max(r - q, 0) after each rejected one; where none stays the token is drawn from r.  Either way the
    kept tokens and the next one are distributed as the target's own.  Rows without a distribution (a NaN, a +inf, nothing but -inf; the draft's where there are children) end
    the walk with next -1."""
    _check_rows_of_logits(logits, b, "logits")
    V = logits.shape[1]
    if not 0 < V < 1 << 30:
        raise ValueError(f"rows of 1 .. 2^30 - 1 entries: got {V}")
    if b.parents is None or b.parents.dtype != torch.int32 or b.parents.shape != (b.T,) or not b.parents.is_contiguous():
        raise ValueError("the step's parents (RequestBatch) are int32 [rows]")
    if b.tokens.dtype != torch.int32 or b.tokens.shape != (b.T,) or not b.tokens.is_contiguous():
        raise ValueError("the step's tokens are int32 [rows]")
    if uniforms is not None and (uniforms.dtype != torch.float32 or uniforms.shape != (b.T, 2) or not uniforms.is_contiguous()):
        raise ValueError("random numbers are fp32 [rows, 2]")
    if draft_logits is not None:
        if uniforms is None:
            raise ValueError("drafted distributions need random numbers: a greedy walk takes none")
        _check_rows_of_logits(draft_logits, b, "draft_logits")
        if draft_logits.shape != logits.shape:
            raise ValueError(f"draft_logits are as wide as logits: got {tuple(draft_logits.shape)} and {tuple(logits.shape)}")
    draft_temperature, draft_top_p = temperature if draft_temperature is None else draft_temperature, top_p if draft_top_p is None else draft_top_p
    for t, p in ((temperature, top_p), (draft_temperature, draft_top_p)):
        if not 1e-30 < float(t) < float("inf"):
            raise ValueError("a temperature is above 1e-30 and finite")
        if not 0.0 <= float(p) <= 1.0:
            raise ValueError("top_p is 0 .. 1")
    for t in (uniforms, draft_logits, b.parents, b.tokens, b.row0, b.n):
        if t is not None and t.device != logits.device:
            raise ValueError(f"logits, random numbers and the step lie on one device: got {t.device} and {logits.device}")
    _on_current_device(logits)
    i32 = dict(dtype=torch.int32, device=logits.device)
    path, ends, outcome = torch.empty(b.E, b.max_n, **i32), torch.empty(2, b.E, **i32), torch.empty(2 * b.T + 1, **i32)
    pitch = V if b.T == 1 else logits.stride(0)
    dpitch = 0 if draft_logits is None else V if b.T == 1 else draft_logits.stride(0)
    a = _lib.VERIFY.pack(logits.data_ptr(), _lib.ptr(draft_logits), _lib.ptr(uniforms), b.tokens.data_ptr(), b.parents.data_ptr(), b.row0.data_ptr(), b.n.data_ptr(), path.data_ptr(),
                         ends.data_ptr(), ends.data_ptr() + 4 * b.E, outcome.data_ptr(), pitch, dpitch, b.max_n, temperature, top_p, draft_temperature, draft_top_p, b.E, b.T, b.max_n, V)
    _lib.check(_lib.lib().pg_verify_drafts(a, _lib.stream()), "pg_verify_drafts")
    return path, ends[0], ends[1]


# ---- scored tokens ---------------------------------------------------------------------------------------------------
def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, temperature: float = 1.0):
    """logits fp32 [rows, vocab] (any row pitch), tokens int32 [rows]: under softmax(logits / temperature) the log probability of every row's token, the entropy in
    nats, the token's rank (0: the most likely one; ties: the lower id is in front) and the `top` (0 .. 32) most likely ids with their log probabilities:
    (fp32 [rows], fp32 [rows], int32 [rows], int32 [rows, top], fp32 [rows, top]).  A token outside the vocabulary, or whose own logit is a NaN: NaN and rank -1.  Masked entries are -inf; a row
    with a NaN, a +inf or nothing but -inf has NaN for its numbers."""
    if logits.dim() != 2 or logits.dtype != torch.float32 or logits.stride(1) != 1 or not logits.is_cuda:
        raise ValueError("logits are fp32 [rows, vocab] on the device, entries of a row side by side")
    rows, V = logits.shape
    if tokens.dtype != torch.int32 or tokens.shape != (rows,) or not tokens.is_contiguous() or tokens.device != logits.device:
        raise ValueError("one int32 token for every row of the logits, on their device")
    if not 0 <= int(top) <= min(32, V):
        raise ValueError(f"top is 0 .. 32 and at most the vocabulary: got {top}")
    if not 0.0 < float(temperature) < float("inf"):
        raise ValueError("the temperature is positive and finite")
    _on_current_device(logits)
    top = int(top)
    lp, entropy, top_lp, rank, ids = logits.new_empty(rows), logits.new_empty(rows), logits.new_empty((rows, top)), tokens.new_empty(rows), tokens.new_empty((rows, top))
    if rows:
        _lib.check(_lib.lib().pg_token_logprobs(logits.data_ptr(), logits.stride(0) if rows > 1 else V, tokens.data_ptr(), lp.data_ptr(), entropy.data_ptr(), rank.data_ptr(), ids.data_ptr(),
                                                top_lp.data_ptr(), rows, V, top, float(temperature), _lib.stream()), "pg_token_logprobs")
    return lp, entropy, rank, ids, top_lp


# ---- multi-stream residual -------------------------------------------------------------------------------------------
def embed_streams(tokens, table, S, D, scale=1.0):
    xs = torch.empty(tokens.numel(), S, D, device="cuda", dtype=torch.float32)
    _lib.check(_lib.lib().pg_embed_streams(tokens.data_ptr(), table.data_ptr(), table.stride(0), xs.data_ptr(), tokens.numel(), S, D, float(scale),
                                           int(table.dtype == torch.float32), _lib.stream()), "pg_embed_streams")
    return xs


def stream_mix_norm(xs, y=None, mix=None, write=None, read=None, norm_w=None, out_act=None, eps=1e-6):
    """One pass over the stream rows xs [T, S, D] (fp32, in place): the write-back of a finished sub-layer (y fp32 [T, D], mix
    [S, S] from x to, write [S]) and / or the normalised read of the next one (read [S], norm_w [D] -> out_act [T, D])."""
    T, S, D = xs.shape
    assert xs.dtype == torch.float32 and xs.is_contiguous()
    assert y is None or (y.dtype == torch.float32 and y.stride(1) == 1 and y.shape == (T, D))
    for t in (mix, write, read, norm_w):
        assert t is None or (t.dtype == torch.float32 and t.is_contiguous())
    assert out_act is None or (out_act.is_contiguous() and out_act.shape == (T, D))
    _lib.check(_lib.lib().pg_stream_mix_norm(xs.data_ptr(), _lib.ptr(y), 0 if y is None else y.stride(0), _lib.ptr(mix), _lib.ptr(write), _lib.ptr(read),
                                             _lib.ptr(norm_w), _lib.ptr(out_act), T, S, D, float(eps),
                                             int(out_act is not None and out_act.dtype == torch.float32), _lib.stream()), "pg_stream_mix_norm")
    return out_act


# ---- latent attention ------------------------------------------------------------------------------------------------
_BATCH_PLANS = {}


def _batch_plan(T, B):
    """Tile list (batch index, first row, rows) of a batched product over the same T rows for every index, in the layout of
    pg_moe_plan; made once per (T, B) on the host."""
    key = (T, B)
    if key not in _BATCH_PLANS:
        if torch.cuda.is_current_stream_capturing():
            return None
        tile = _lib.lib().pg_moe_tile_rows()
        rows = [(b, r0, min(tile, T - r0)) for b in range(B) for r0 in range(0, T, tile)]
        buf = np.zeros(4 + 3 * len(rows), dtype=np.int32)
        buf[0] = len(rows)
        buf[4:] = np.asarray(rows, dtype=np.int32).reshape(-1)
        _BATCH_PLANS[key] = (torch.from_numpy(buf).to("cuda"), len(rows))
        torch.cuda.current_stream().synchronize()
    return _BATCH_PLANS[key]


def linear_batched(x, w, out):
    """out[:, b, :] = x[:, b, :] @ w[b].T for every b: x [T, B, K] and out [T, B, F] are views with unit last stride, w [B, F, K].
    bf16 operands whose slices start on 16-byte boundaries run on the tensor cores (the grouped kernel of the routed experts with
    one "expert" per batch index); everything else on plain fp32 FMAs."""
    T, B, K = x.shape
    F = w.shape[1]
    assert w.shape == (B, F, K) and out.shape == (T, B, F) and x.dtype == w.dtype and w.is_contiguous()
    assert x.stride(2) == 1 and out.stride(2) == 1
    if (x.dtype == torch.bfloat16 and K % 8 == 0 and x.stride(0) % 8 == 0 and x.stride(1) % 8 == 0 and x.data_ptr() % 16 == 0
            and w.data_ptr() % 16 == 0 and len(_BATCH_PLANS) < 4096):
        plan = _batch_plan(T, B)
        if plan is not None and plan[1] <= 65535:
            _lib.check(_lib.lib().pg_moe_gemm(x.data_ptr(), x.stride(0), plan[0].data_ptr(), 0, w.data_ptr(), F * K, K, out.data_ptr(), out.stride(0),
                                              plan[0].data_ptr(), plan[1], F, K, 0, 0, int(out.dtype == torch.float32), x.stride(1), out.stride(1),
                                              _lib.stream()), "pg_moe_gemm")
            return out
    _lib.check(_lib.lib().pg_gemm_simt_batched(x.data_ptr(), x.stride(0), x.stride(1), w.data_ptr(), K, F * K, out.data_ptr(), out.stride(0),
                                               out.stride(1), T, F, K, B, int(x.dtype == torch.float32), int(out.dtype == torch.float32),
                                               _lib.stream()), "pg_gemm_simt_batched")
    return out


def latent_prepare(proj, b: StepBatch, freq, q_norm, c_norm, cq_out, pages, q_rank, rank, rot, rot_dims, eps, page, rot_gain=1.0):
    """pages None: the layer reads another layer's cached rows; only the normalised query latent is made."""
    assert proj.stride(1) == 1 and freq.dtype == torch.float64 and (pages is None or (pages.dtype == proj.dtype and pages.shape[-1] == rank + rot))
    assert cq_out is None or (cq_out.dtype == proj.dtype and cq_out.is_contiguous())
    _lib.check(_lib.lib().pg_latent_prepare(proj.data_ptr(), proj.stride(0), b.pos.data_ptr(), b.row_entry.data_ptr(), b.page_table.data_ptr(),
                                            b.max_pages, page, freq.data_ptr(), _lib.ptr(q_norm), _lib.ptr(c_norm), _lib.ptr(cq_out), _lib.ptr(pages),
                                            b.T, q_rank, rank, rot, rot_dims, float(eps), float(rot_gain), int(proj.dtype == torch.float32), _lib.stream()),
               "pg_latent_prepare")


def rotate_heads(src, dst, pos, freq, rot_dims, rot_gain=1.0):
    """src, dst: [T, H, n] views (unit last stride, any row / head pitch) of one type; the first rot_dims of every head vector are
    rotated in interleaved pairs by pos[t] * freq[i]; rot_gain multiplies cosines and sines."""
    T, H, n = src.shape
    assert dst.shape == src.shape and src.dtype == dst.dtype and src.stride(2) == 1 and dst.stride(2) == 1
    _lib.check(_lib.lib().pg_rotate_heads(src.data_ptr(), src.stride(0), src.stride(1), dst.data_ptr(), dst.stride(0), dst.stride(1), pos.data_ptr(),
                                          freq.data_ptr(), T, H, n, rot_dims, float(rot_gain), int(src.dtype == torch.float32), _lib.stream()), "pg_rotate_heads")


def latent_expand(pages, b: StepBatch, w_ukv, H, dim, rot, vdim, rank, page, prec):
    """Per-head keys [plain | rotated] and values of every multi-token entry's context + new tokens, rebuilt from the cached
    latent rows into dense scratch: k [dense_rows, H * (dim + rot)], v [dense_rows, H * vdim] (read through b.dense_pages)."""
    L, f32 = _lib.lib(), int(pages.dtype == torch.float32)
    lat = prec.empty(b.dense_rows, rank)
    _lib.check(L.pg_latent_gather(pages.data_ptr(), b.page_table.data_ptr(), b.max_pages, page, b.dense_row0.data_ptr(), b.n.data_ptr(), b.ctx.data_ptr(),
                                  lat.data_ptr(), b.E, b.dense_max_len, rank, rank + rot, f32, _lib.stream()), "pg_latent_gather")
    up = linear(lat, w_ukv, prec.empty(b.dense_rows, H * (dim + vdim)))
    k = prec.empty(b.dense_rows, H * (dim + rot))
    v = prec.empty(b.dense_rows, H * vdim)
    _lib.check(L.pg_latent_pack_kv(up.data_ptr(), up.stride(0), pages.data_ptr(), b.page_table.data_ptr(), b.max_pages, page, b.dense_row0.data_ptr(),
                                   b.n.data_ptr(), b.ctx.data_ptr(), k.data_ptr(), v.data_ptr(), b.E, b.dense_max_len, H, dim, rot, vdim, rank, f32,
                                   _lib.stream()), "pg_latent_pack_kv")
    return k, v


def dense_view(b: StepBatch) -> StepBatch:
    """The same step with the dense scratch layout in place of the cache's page table."""
    return dataclasses.replace(b, page_table=b.dense_pages, max_pages=b.dense_max_pages)


# ---- routed feed-forward ---------------------------------------------------------------------------------------------
ROUTE_LOGISTIC, ROUTE_GROUP_BEST_TWO, ROUTE_PLAIN_WEIGHTS = 1, 2, 4


def moe_route(logits, correction, n_real, top, group_count, group_keep, scale, logit_bias=None, flags=0):
    """logits fp32 [T, n_all] (+ logit_bias fp32 [n_all]) -> ids int32 [T, top], weights fp32 [T, top], counts int32 [n_real] (device).  flags:
    ROUTE_LOGISTIC -- scores are sigmoid(logit) instead of the softmax; ROUTE_GROUP_BEST_TWO -- a group counts the sum of its two best
    choices; ROUTE_PLAIN_WEIGHTS -- the chosen scores are not divided by their sum."""
    T, n_all = logits.shape
    assert logits.dtype == torch.float32 and logits.stride(1) == 1
    ids = torch.empty(T, top, device="cuda", dtype=torch.int32)
    wts = torch.empty(T, top, device="cuda", dtype=torch.float32)
    counts = torch.empty(max(1, n_real), device="cuda", dtype=torch.int32)
    _lib.check(_lib.lib().pg_moe_route(logits.data_ptr(), logits.stride(0), _lib.ptr(correction), ids.data_ptr(), wts.data_ptr(), counts.data_ptr(), T,
                                       n_all, n_real, top, int(group_count), int(group_keep), float(scale), _lib.ptr(logit_bias), int(flags), _lib.stream()), "pg_moe_route")
    return ids, wts, counts


class MoePlan:
    """Device-side order of the (token, choice) pairs by expert and the list of row tiles the grouped products walk.  n_real 0 (identity outputs only): no pair has an
    expert row, there is nothing to walk and no count to read."""

    def __init__(self, ids, counts, n_real):
        L = _lib.lib()
        T, top = ids.shape
        self.pairs, self.top = T * top, top
        if not n_real:
            self.pair_row = torch.full((self.pairs,), -1, device=ids.device, dtype=torch.int32)
            return
        self.max_tiles = -(-self.pairs // L.pg_moe_tile_rows()) + n_real
        i32 = dict(device="cuda", dtype=torch.int32)
        self.offsets = torch.empty(n_real + 1, **i32)
        self.fill = torch.empty(n_real, **i32)
        self.plan = torch.empty(4 + 3 * self.max_tiles, **i32)
        self.sorted_pair = torch.empty(self.pairs, **i32)
        self.pair_row = torch.empty(self.pairs, **i32)
        _lib.check(L.pg_moe_plan(counts.data_ptr(), ids.data_ptr(), self.offsets.data_ptr(), self.fill.data_ptr(), self.plan.data_ptr(),
                                 self.sorted_pair.data_ptr(), self.pair_row.data_ptr(), self.pairs, n_real, self.max_tiles, _lib.stream()), "pg_moe_plan")


def moe_gemm(x, plan: MoePlan, w, out, gather, act=0):
    """out[row] = act(x[src(row)] @ w[expert(row)].T) over the plan's tiles; gather: x rows are tokens (src = pair // top),
    else x rows are already in sorted order.  w [n_real, F, K] contiguous."""
    n_real, F, K = w.shape
    assert w.is_contiguous() and x.dtype == w.dtype and x.stride(1) == 1 and out.stride(1) == 1 and x.shape[1] == K
    assert out.shape[1] == (F // 2 if act == ACT_SILU_GLU else F)
    _lib.check(_lib.lib().pg_moe_gemm(x.data_ptr(), x.stride(0), plan.sorted_pair.data_ptr(), plan.top if gather else 0, w.data_ptr(), F * K, K,
                                      out.data_ptr(), out.stride(0), plan.plan.data_ptr(), plan.max_tiles, F, K, int(act),
                                      int(x.dtype == torch.float32), int(out.dtype == torch.float32), 0, 0, _lib.stream()), "pg_moe_gemm")
    return out


def moe_products(x, plan: MoePlan, w_up, w_down, xg, mid, eo, act):
    """eo[row] = act(x[token of row] @ w_up[expert(row)].T) @ w_down[expert(row)].T over the plan's rows (bf16; eo fp32); xg, mid: scratch."""
    n_real, D, F = w_down.shape
    assert x.is_cuda and w_up.is_cuda and w_down.is_cuda and xg.is_cuda and mid.is_cuda and eo.is_cuda
    assert x.dtype == w_up.dtype == w_down.dtype == xg.dtype == mid.dtype == torch.bfloat16 and eo.dtype == torch.float32 and x.stride(1) == 1
    assert all(t.is_contiguous() for t in (w_up, w_down, xg, mid, eo)) and x.shape[1] == D and w_up.shape == (n_real, 2 * F if act == ACT_SILU_GLU else F, D)
    assert xg.shape == (plan.pairs, D) and mid.shape == (plan.pairs, F) and eo.shape == (plan.pairs, D)
    _lib.check(_lib.lib().pg_moe_products(x.data_ptr(), x.stride(0), plan.sorted_pair.data_ptr(), plan.offsets.data_ptr() + 4 * n_real, plan.top, xg.data_ptr(),
                                          w_up.data_ptr(), w_down.data_ptr(), mid.data_ptr(), eo.data_ptr(), plan.plan.data_ptr(), plan.max_tiles, plan.pairs,
                                          n_real, D, F, int(act), _lib.stream()), "pg_moe_products")
    return eo


def moe_gather_rows(x, plan: MoePlan, out):
    """out[row] = x[token of sorted pair `row`]: every expert's tokens as one contiguous run of rows."""
    assert x.dtype == out.dtype and x.stride(1) == 1 and out.stride(1) == 1 and out.shape[0] >= plan.pairs
    _lib.check(_lib.lib().pg_moe_gather_rows(x.data_ptr(), x.stride(0), plan.sorted_pair.data_ptr(), plan.offsets[-1:].data_ptr(), plan.top, out.data_ptr(),
                                             out.stride(0), plan.pairs, x.shape[1], int(x.dtype == torch.float32), _lib.stream()), "pg_moe_gather_rows")
    return out


def moe_combine(expert_out, plan: MoePlan, ids, weights, h, shared_out, y, shared_gate=None, accumulate=False):
    """y[t] (+)= sum_k weights[t, k] * expert row (or h[t] for an identity expert) + sigmoid(shared_gate[t]) * shared_out[t]; shared_gate:
    fp32 logits, one per token (a strided column view), None: the shared term counts fully; accumulate: add into y."""
    T, D = y.shape
    assert expert_out is not None or not hasattr(plan, "plan")  # (without expert rows no pair may have one)
    assert shared_gate is None or (shared_gate.dtype == torch.float32 and shared_gate.shape[0] == T)
    assert y.dtype == torch.float32 and y.is_contiguous() and h.stride(1) == 1
    assert expert_out is None or (expert_out.dtype == torch.float32 and expert_out.stride(1) == 1)
    _lib.check(_lib.lib().pg_moe_combine(_lib.ptr(expert_out), 0 if expert_out is None else expert_out.stride(0), plan.pair_row.data_ptr(), ids.data_ptr(),
                                         weights.data_ptr(), h.data_ptr(), h.stride(0), _lib.ptr(shared_out), 0 if shared_out is None else shared_out.stride(0),
                                         y.data_ptr(), T, D, plan.top, int(h.dtype == torch.float32), _lib.ptr(shared_gate),
                                         0 if shared_gate is None else shared_gate.stride(0), int(bool(accumulate)), _lib.stream()), "pg_moe_combine")
    return y


def routed_ff(h, form, y, accumulate):
    """A whole routed feed-forward by one call (_lib.RoutedFf names the weights and sizes); y fp32 [T, D]."""
    import ctypes as C
    assert h.is_cuda and h.dtype == torch.bfloat16 and h.stride(1) == 1 and h.shape == (form.tokens, form.D) and y.dtype == torch.float32 and y.is_contiguous() and y.shape == h.shape
    need = _lib.lib().pg_routed_ff_scratch(C.addressof(form))
    scratch = torch.empty(need, device=h.device, dtype=torch.uint8)
    _lib.check(_lib.lib().pg_routed_ff(C.addressof(form), h.data_ptr(), h.stride(0), y.data_ptr(), int(bool(accumulate)), scratch.data_ptr(), need, _lib.stream()),
               "pg_routed_ff")
    return y


COMBINE_NORM_MAX_WIDTH = 12288  # a row of sums stays in shared memory


def moe_combine_norm_add(expert_out, plan: MoePlan, weights, norm_w, x, out_act, eps):
    """y = sum_k weights[t, k] * expert row; x += y / rms(y) * norm_w in place; out_act (may be None) gets the new row."""
    T, D = x.shape
    assert x.dtype == torch.float32 and x.is_contiguous() and expert_out.dtype == torch.float32 and expert_out.stride(1) == 1 and norm_w.numel() == D
    assert norm_w.dtype == torch.float32 and (out_act is None or (out_act.is_contiguous() and out_act.shape == x.shape))
    _lib.check(_lib.lib().pg_moe_combine_norm_add(expert_out.data_ptr(), expert_out.stride(0), plan.pair_row.data_ptr(), weights.data_ptr(), norm_w.data_ptr(),
                                                  x.data_ptr(), _lib.ptr(out_act), T, D, plan.top, float(eps),
                                                  int(out_act is not None and out_act.dtype == torch.float32), _lib.stream()), "pg_moe_combine_norm_add")


# a portion at least this long is advanced in 32-token blocks; shorter ones (decode above all) token by token
LINEAR_ATTN_CHUNK_MIN = 8


def linear_attn(qkv, state, decay, out, b: StepBatch, H, dim, vdim, chunked=None):
    """S <- decay S + k v^T, out = S^T q per head (fp32 [T, H * vdim]) with q, k and v through silu.  Portions of some length go in blocks -- for bf16 head sizes that fit
    an entry's own length decides, and on the tensor cores where there are enough of them -- the others token by token (chunked True / False: one form for every entry)."""
    import ctypes as C
    assert state.dtype == torch.float32 and out.dtype == torch.float32 and out.is_contiguous() and qkv.stride(1) == 1
    f32 = int(qkv.dtype == torch.float32)
    n_min = {None: LINEAR_ATTN_CHUNK_MIN, True: 1, False: FOREVER}[chunked]
    # not for a few heads of a few sequences: there the other block form has more CTAs (its value blocks get narrower), and a chain of blocks is what takes the time (us, FMA / tensor:
    # 32 CTAs of 64 columns, 2000 tokens 330 / 370, 2 x 1000 tokens 171 / 191; 64 CTAs of 2000 tokens 458 / 371, of 100 tokens 35 / 29)
    # Single tokens own no blocks (2000 tokens beside 40 of them, 16 heads, FMA / tensor with the form for few CTAs / with that for many 332 / 375 / 414); beside them the FMA form's narrow
    # blocks pay for fewer heads (24 329 / 373, 28 382 / 373).
    portions = b.E - (b.singles if n_min > 1 else 0)
    fits = not f32 and dim % 8 == 0 and dim <= 128 and vdim % 8 == 0 and qkv.stride(0) % 8 == 0 and _aligned(qkv)
    tensor_cores = portions * H * ((vdim + 63) // 64) >= (64 if portions == b.E else 25)

    def go(fn, lo, hi, *tail):
        ops = _lib.LinearAttnOps(1, 1.0, 0, 0, lo, hi, portions if lo == n_min else 0)
        _lib.check(fn(qkv.data_ptr(), qkv.stride(0), state.data_ptr(), decay.data_ptr(), out.data_ptr(), b.row0.data_ptr(), b.n.data_ptr(), b.ctx.data_ptr(),
                      b.slot.data_ptr(), b.E, H, dim, vdim, C.addressof(ops), *tail, _lib.stream()), "pg_linear_attn")

    L = _lib.lib()
    if b.max_n < n_min:
        go(L.pg_linear_attn_scan, 1, FOREVER, f32)
    elif not fits:
        go(L.pg_linear_attn_chunked, 1, FOREVER, f32)
    else:
        if tensor_cores:
            go(L.pg_linear_attn_blocks, n_min, FOREVER)
        else:
            go(L.pg_linear_attn_chunked, n_min, FOREVER, f32)
        if b.min_n < n_min:
            go(L.pg_linear_attn_scan, 1, n_min - 1, f32)


def rotary_table(b: StepBatch, freq, rot_dims, dim, gain=1.0):
    """fp32 [T, 2, pairs]: cosines and sines of the step's rows for every pair of a head of `dim` elements (1 and 0 past the rotated ones)."""
    pairs = (dim + 7) // 8 * 4
    assert freq.dtype == torch.float64 and rot_dims <= dim
    out = torch.empty(b.T, 2, pairs, device="cuda", dtype=torch.float32)
    _lib.check(_lib.lib().pg_rotary_table(b.pos.data_ptr(), freq.data_ptr(), out.data_ptr(), b.T, int(rot_dims), pairs, float(gain), _lib.stream()), "pg_rotary_table")
    return out


def retention(qkv, state, decay, out, b: StepBatch, H, dim, vdim, kscale=1.0, rotate=None, blocks=None):
    """S <- decay S + k v^T, out = S^T q per head (fp32 [T, H * vdim]) with q and k turned in neighbouring pairs by `rotate` (rotary_table; None:
    not turned) and k times kscale.  Entries with several new tokens go in blocks -- on the tensor cores for bf16 head sizes that fit --
    the others token by token (blocks True / False: one form for every entry); an entry's own length decides."""
    import ctypes as C
    assert state.dtype == torch.float32 and tuple(state.shape[1:]) == (H, dim, vdim) and out.dtype == torch.float32 and out.is_contiguous() and qkv.stride(1) == 1
    assert rotate is None or (rotate.dtype == torch.float32 and rotate.is_contiguous() and rotate.shape[0] == b.T and 2 * rotate.shape[2] >= dim)
    f32 = int(qkv.dtype == torch.float32)
    tensor_cores = not f32 and dim % 8 == 0 and dim <= 128 and vdim % 8 == 0 and qkv.stride(0) % 8 == 0 and _aligned(qkv)
    n_min = {None: RECURRENCE_BLOCK_MIN if tensor_cores else LINEAR_ATTN_CHUNK_MIN, True: 1, False: FOREVER}[blocks]

    def go(fn, lo, hi, *tail):
        ops = _lib.LinearAttnOps(0, float(kscale), _lib.ptr(rotate), 0 if rotate is None else rotate.shape[2], lo, hi, b.E - b.singles if lo == n_min > 1 else 0)
        _lib.check(fn(qkv.data_ptr(), qkv.stride(0), state.data_ptr(), decay.data_ptr(), out.data_ptr(), b.row0.data_ptr(), b.n.data_ptr(), b.ctx.data_ptr(),
                      b.slot.data_ptr(), b.E, H, dim, vdim, C.addressof(ops), *tail, _lib.stream()), "pg_linear_attn")

    L = _lib.lib()
    if b.max_n >= n_min:
        if tensor_cores:
            go(L.pg_linear_attn_blocks, n_min, FOREVER)
        else:
            go(L.pg_linear_attn_chunked, n_min, FOREVER, f32)
    if b.max_n < n_min or (n_min > 1 and b.E > 1):
        go(L.pg_linear_attn_scan, 1, n_min - 1, f32)
    return out


# ---- recurrent mixers --------------------------------------------------------------------------------------------------
def _entry_ptrs(b: StepBatch):
    return dict(entry_row0=b.row0.data_ptr(), entry_n=b.n.data_ptr(), entry_ctx=b.ctx.data_ptr(), entry_slot=b.slot.data_ptr(), entries=b.E)


class ConvSections:
    """Channel sections of a short convolution: dicts with groups, size (channels of a group), total (channels; default groups * size), xcol
    (first input column), ccol (first channel of weights, state and output), unit (inverse norms wanted) and scale (factor of the inverse norm)."""

    def __init__(self, sections):
        assert 1 <= len(sections) <= 3
        self.c = _lib.ConvSections()
        self.c.count = len(sections)
        self.unit_groups = 0
        for i, s in enumerate(sections):
            for k in ("groups", "size", "xcol", "ccol"):
                getattr(self.c, k)[i] = int(s[k])
            self.c.total[i] = int(s.get("total", s["groups"] * s["size"]))
            self.c.unit[i] = int(bool(s.get("unit")))
            self.c.scale[i] = float(s.get("scale", 1.0))
            if s.get("unit"):
                self.unit_groups += int(s["groups"])


def short_conv(x, w, state, out, sections: ConvSections, b: StepBatch, bias=None, inv=None):
    """out = silu(causal convolution over time of x's columns, per channel); w fp32 [taps, C] tap-major; state fp32 [slots, taps - 1, C] (None
    for one tap); inv fp32 [T, unit groups] receives scale / sqrt(sum y^2 + 1e-6) of every group of the unit sections."""
    import ctypes as C
    taps, chans = w.shape
    assert w.dtype == torch.float32 and w.is_contiguous() and x.dtype == out.dtype and x.stride(1) == 1 and out.stride(1) == 1 and out.shape == (b.T, chans)
    assert taps == 1 or (state.dtype == torch.float32 and state.is_contiguous() and tuple(state.shape[1:]) == (taps - 1, chans))
    assert bias is None or (bias.dtype == torch.float32 and bias.numel() == chans)
    assert (inv is None) == (sections.unit_groups == 0) and (inv is None or (inv.dtype == torch.float32 and inv.is_contiguous() and inv.shape == (b.T, sections.unit_groups)))
    _lib.check(_lib.lib().pg_short_conv_sized(x.data_ptr(), x.stride(0), w.data_ptr(), _lib.ptr(bias), _lib.ptr(state), out.data_ptr(), out.stride(0), _lib.ptr(inv),
                                              sections.unit_groups, C.addressof(sections.c), taps, chans, b.row0.data_ptr(), b.n.data_ptr(), b.ctx.data_ptr(),
                                              b.slot.data_ptr(), b.E, b.max_n, b.E - b.singles, int(x.dtype == torch.float32), _lib.stream()), "pg_short_conv")
    return out


def recurrence_block(vdim):
    """Value columns one CTA of the recurrent kernels owns (the normaliser of a matrix memory is kept once per such block)."""
    return 64 if vdim % 4 == 0 else 16


# an entry with at least this many new tokens is advanced in blocks on the tensor cores (bf16, head sizes that are multiples of 8 up to 128),
# anything else token by token; the form an entry takes depends on its own length only
RECURRENCE_BLOCK_MIN = 16
FOREVER = 1 << 30


def _in_blocks(q, k, v, dim, vdim, b: StepBatch, blocks):
    """None: token by token; else the least number of new tokens that goes through the block kernels."""
    fits = (q.dtype == torch.bfloat16 and dim % 8 == 0 and dim <= 128 and vdim % 8 == 0
            and all(t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0 for t in (q, k, v)))
    n_min = RECURRENCE_BLOCK_MIN if blocks is None else (1 if blocks else FOREVER)
    return n_min if fits and b.max_n >= n_min else None


def delta_rule(q, k, v, beta, inv, decay, A_log, dt_bias, state, out, b: StepBatch, H, G, dim, vdim, blocks=None):
    """Delta rule with a decay per head and key channel (pg_delta_blocks / pg_delta_scan; blocks True / False: one form for every entry that fits
    it; `decay` is scratch afterwards): q, k [T, G * dim], v [T, H * vdim], beta [T, H] column views in the
    activation type, inv fp32 [T, 2 G] (inverse norms of q, then k), decay fp32 [T, H * dim] (before bias and softplus) -> out fp32."""
    import ctypes as C
    assert state.dtype == torch.float32 and tuple(state.shape[1:]) == (H, dim, vdim) and out.dtype == torch.float32 and out.is_contiguous()
    assert decay.dtype == torch.float32 and decay.stride(1) == 1 and all(t.stride(1) == 1 and t.dtype == q.dtype for t in (q, k, v, beta))
    a = _lib.DeltaArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), beta=beta.data_ptr(), ldq=q.stride(0), ldk=k.stride(0), ldv=v.stride(0),
                       ldb=beta.stride(0), inv=inv.data_ptr(), ldi=inv.stride(0), decay=decay.data_ptr(), lda=decay.stride(0), A_log=A_log.data_ptr(),
                       dt_bias=dt_bias.data_ptr(), state=state.data_ptr(), out=out.data_ptr(), H=H, G=G, dim=dim, vdim=vdim, **_entry_ptrs(b))
    n_min = _in_blocks(q, k, v, dim, vdim, b, blocks) if decay.stride(0) % 4 == 0 else None
    if n_min is not None:
        scratch = torch.empty((b.T // 16 + b.E + 1) * H * 192, 4, device="cuda", dtype=torch.int32)
        _lib.check(_lib.lib().pg_delta_blocks(C.addressof(a), decay.data_ptr(), scratch.data_ptr(), b.max_n, n_min, _lib.stream()), "pg_delta_blocks")
    if n_min is None or (n_min > 1 and b.E > 1):
        _lib.check(_lib.lib().pg_delta_scan(C.addressof(a), 1, FOREVER if n_min is None else n_min - 1, int(q.dtype == torch.float32), _lib.stream()),
                   "pg_delta_scan")
    return out


STATE_SPACE, MATRIX_MEMORY = 0, 1


def gated_recurrence(kind, q, k, v, gate1, gate2, p1, p2, p3, state, norm_state, out, b: StepBatch, H, G, dim, vdim, qscale=1.0, cap=0.0,
                     blocks=None):
    """Recurrence with one scalar decay per head and token (pg_gated_blocks / pg_gated_scan, `blocks` as in delta_rule; kind STATE_SPACE or
    MATRIX_MEMORY) -> out fp32 [T, H * vdim]."""
    import ctypes as C
    assert state.dtype == torch.float32 and tuple(state.shape[1:]) == (H, dim, vdim) and out.dtype == torch.float32 and out.is_contiguous()
    assert all(t is None or (t.stride(1) == 1 and t.dtype == q.dtype) for t in (q, k, v, gate1, gate2)) and (gate2 is None or gate2.stride(0) == gate1.stride(0))
    if kind == MATRIX_MEMORY:
        vb = recurrence_block(vdim)
        assert norm_state.dtype == torch.float32 and tuple(norm_state.shape[1:]) == (-(-vdim // vb), H, dim + 1)
    a = _lib.GatedArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), ldq=q.stride(0), ldk=k.stride(0), ldv=v.stride(0), qscale=float(qscale),
                       gate1=gate1.data_ptr(), gate2=_lib.ptr(gate2), ldg=gate1.stride(0), p1=p1.data_ptr(), p2=p2.data_ptr(), p3=_lib.ptr(p3), cap=float(cap),
                       state=state.data_ptr(), norm_state=_lib.ptr(norm_state), out=out.data_ptr(), H=H, G=G, dim=dim, vdim=vdim, **_entry_ptrs(b))
    n_min = _in_blocks(q, k, v, dim, vdim, b, blocks)
    if n_min is not None:
        _lib.check(_lib.lib().pg_gated_blocks(C.addressof(a), int(kind), n_min, _lib.stream()), "pg_gated_blocks")
    if n_min is None or (n_min > 1 and b.E > 1):
        _lib.check(_lib.lib().pg_gated_scan(C.addressof(a), int(kind), 1, FOREVER if n_min is None else n_min - 1, int(q.dtype == torch.float32),
                                            _lib.stream()), "pg_gated_scan")
    return out


GATE_NONE, GATE_SIGMOID_AFTER, GATE_SILU_BEFORE, GATE_SILU_AFTER = 0, 1, 2, 3


def group_norm_gate(o, w, gate, out, groups, eps, mode, scale=1.0):
    """out = scale * norm(o) * w * sigmoid(gate) (GATE_SIGMOID_AFTER), * silu(gate) (GATE_SILU_AFTER) or scale * norm(o * silu(gate)) * w
    (GATE_SILU_BEFORE), the norm in `groups` equal parts of the row; w fp32 [D], one group's [D / groups] or None; out may be a column slice."""
    rows, D = o.shape
    assert o.dtype == torch.float32 and o.is_contiguous() and out.shape == o.shape and out.stride(1) == 1
    assert w is None or (w.dtype == torch.float32 and w.is_contiguous())
    assert gate is None or (gate.dtype == out.dtype and gate.stride(1) == 1)
    _lib.check(_lib.lib().pg_group_norm_gate(o.data_ptr(), _lib.ptr(w), 0 if w is None else w.numel(), _lib.ptr(gate), 0 if gate is None else gate.stride(0), int(mode),
                                             out.data_ptr(), out.stride(0), rows, D, int(groups), float(eps), float(scale), int(out.dtype == torch.float32),
                                             _lib.stream()), "pg_group_norm_gate")
    return out


def gated_layernorm_add(y, gate, gate_b, w1, b1, x, eps, w2=None, b2=None, out=None):
    """x += LN(y * sigmoid(gate + gate_b); w1, b1) in place (fp32); out (activation type) = LN(x; w2, b2), the next sub-layer's input, when given.
    gate: bf16, or fp32 beside any output type."""
    rows, D = x.shape
    assert y.dtype == torch.float32 and y.shape == x.shape and y.stride(1) == 1 and x.dtype == torch.float32 and x.is_contiguous()
    assert gate is None or (gate.shape == x.shape and gate.stride(1) == 1 and gate.dtype in (torch.float32, torch.bfloat16))
    assert out is None or (out.is_contiguous() and out.shape == x.shape and w2 is not None and b2 is not None)
    gate_f32 = int(gate is None or gate.dtype == torch.float32)
    act_f32 = int(out.dtype == torch.float32) if out is not None else gate_f32
    assert gate_f32 or not act_f32
    _lib.check(_lib.lib().pg_gated_layernorm_add(y.data_ptr(), y.stride(0), _lib.ptr(gate), 0 if gate is None else gate.stride(0), _lib.ptr(gate_b),
                                                 w1.data_ptr(), b1.data_ptr(), x.data_ptr(), _lib.ptr(w2), _lib.ptr(b2), _lib.ptr(out), rows, D, float(eps),
                                                 gate_f32, act_f32, _lib.stream()), "pg_gated_layernorm_add")
