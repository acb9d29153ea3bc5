"""Rows of an 8-bit cache that were read back lie in runs of 64, whatever the cache's own pages hold (no device: the library is a stub that keeps its calls)."""
import pytest
import torch

from paligemma_multimodal_system_b200 import _lib, seq_ops


class _Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.mark.parametrize("page", [32, 64, 128])
@pytest.mark.parametrize("dtype,name,at", [(torch.bfloat16, "pg_attn_ragged_mma_sized", 11), (torch.float32, "pg_attn_ragged", 11)])
def test_prompt_attention_walks_the_scratch_by_its_own_pages(monkeypatch, page, dtype, name, at):
    library = _Library()
    monkeypatch.setattr(_lib, "lib", lambda: library)
    monkeypatch.setattr(_lib, "stream", lambda: 0)
    monkeypatch.setattr(seq_ops, "_on_current_device", lambda t: None)
    z = torch.zeros(1, dtype=torch.int32)
    b = seq_ops.StepBatch(T=40, E=1, max_n=40, min_n=40, tokens=z, pos=z, row_entry=z, row0=z, n=z, ctx=z, slot=z, page_table=z.view(1, 1), max_pages=1, singles=0, dense_row0=z,
                          dense_pages=torch.zeros(1, 3, dtype=torch.int32), dense_max_pages=3, dense_rows=192, dense_max_len=170)
    pages = seq_ops.QuantizedPages.empty(6, page, 2, 64, device="cpu")
    q, out = torch.zeros(40, 4 * 64, dtype=dtype), torch.zeros(40, 4 * 64, dtype=dtype)
    seq_ops.attn_ragged(q, pages, pages, None, out, b, 4, 2, 64, 64, 0.125, 0.0, page)
    (read, packed), (attend, args) = library.calls
    assert read == "pg_kv_read_e4m3" and _lib.READ_E4M3.unpack(packed[0])[11] == page  # the cache's rows by the cache's pages
    assert attend == name and args[at - 1:at + 1] == (3, 64)                            # the scratch's by the scratch's
