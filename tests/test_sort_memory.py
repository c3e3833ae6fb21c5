"""What a sort keeps alive: its tables, and not the scratch of the call that made them.  Runs on CPU: the library is replaced by one
that looks at the addresses it is given."""
import contextlib

import pytest
import torch

from tilelang_moe_b200 import kernels, ops


class _Library:
    need = 0
    seen = None

    def moe_sort_workspace(self, n, E):
        return self.need

    def moe_sort(self, ids, is64, n, E, counts, offsets, perm, row_of, ws, ws_bytes, stream):
        type(self).seen = dict(counts=(counts, 4 * (E + 1)), offsets=(offsets, 4 * (E + 2)), perm=(perm, 4 * n), row_of=(row_of, 4 * n), ws=(ws, ws_bytes))
        return 0


@pytest.fixture(autouse=True)
def on_host(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops._lib, "load", _Library)


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (8, 2, 8), (2000, 8, 256), (0, 4, 3), (999, 3, 5119)])
@pytest.mark.parametrize("need", [0, 2, 36, 4097, 65536, 65537, 1 << 20])
def test_scratch_does_not_outlive_the_call(monkeypatch, T, k, E, need):
    monkeypatch.setattr(_Library, "need", need)
    sort = kernels.moe_sort(torch.zeros(T, k, dtype=torch.int32), E)
    tables = 4 * (E + 1) + 4 * (E + 2) + 2 * 4 * T * k
    kept = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in (sort.offsets, sort.perm, sort.row_of)}
    assert sum(kept.values()) <= tables + 65536
    at = _Library.seen
    assert at["offsets"][0] == sort.offsets.data_ptr() and at["ws"][1] == need
    assert T == 0 or (at["perm"][0], at["row_of"][0]) == (sort.perm.data_ptr(), sort.row_of.data_ptr())
    # nothing overlaps
    spans = sorted((p, p + n) for p, n in at.values() if n and p)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    assert all(p % 4 == 0 for p, n in at.values() if n)
