"""The Python side of the paged cache and the token log probabilities, without a GPU: host tensors
stand in where no call is made."""
import types

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def batch(monkeypatch):
    """A batch over host tensors (its pointers are used by no call that these tests make)."""
    from cortexsdr_amd import paged

    monkeypatch.setattr(paged, "_torch", lambda: torch)
    monkeypatch.setattr(paged, "_on_device", lambda torch, what, *ts: 0)
    cache = types.SimpleNamespace(k=torch.zeros(4096, dtype=torch.uint8), kv_dtype="f16",
                                  v=torch.zeros(4096, dtype=torch.uint8), page_size=16, n_pages=1,
                                  n_kv_heads=2, head_dim=64)
    return paged.PagedBatch(cache, torch.zeros(2, 1, dtype=torch.int32),
                            torch.ones(2, dtype=torch.int32))


def test_table_and_lens_are_not_replaced(batch):
    """The library holds their addresses: another tensor in their place would be ignored."""
    lens = batch.lens
    for name in ("table", "lens"):
        with pytest.raises(AttributeError):
            setattr(batch, name, torch.zeros(2, dtype=torch.int32))
    batch.lens.fill_(5)
    assert batch.lens is lens and lens.tolist() == [5, 5]
