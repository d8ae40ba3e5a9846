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


@pytest.fixture
def calls(batch, monkeypatch):
    """The batch's launches, recorded in place of being made."""
    from cortexsdr_amd import paged

    monkeypatch.setattr(paged, "_stream_of", lambda torch, dev, stream: 0)
    made = []
    batch._append = lambda *a: made.append(("append", a)) or 0
    batch._attn = lambda *a: made.append(("attn", a)) or 0
    batch._lib = types.SimpleNamespace(
        csdr_paged_read=lambda *a: made.append(("read", a)) or 0,
        csdr_paged_attn_workspace_bytes=lambda *a: made.append(("bytes", a)) or 0)
    return made


def test_no_tokens_is_no_call(batch, calls, monkeypatch):
    """A scheduler's empty step: empty results, nothing launched."""
    from cortexsdr_amd import logprobs

    q, k = torch.zeros(0, 4, 64), torch.zeros(0, 2, 64)
    start = torch.zeros(3, dtype=torch.int32)
    assert batch.append(q, k, k, theta=1e4).shape == (0, 4, 64)
    assert batch.append(q, k, k, q_start=start, max_q=0).shape == (0, 4, 64)
    assert batch.append(None, k, k) is None
    assert batch.attend(q).shape == (0, 4, 64)
    assert batch.attend(q, q_start=start, max_q=0, out=q) is q
    for t in batch.read(0):
        assert t.shape == (0, 2, 64)
    with pytest.raises(ValueError):
        batch.attend(torch.zeros(0, 4, 32))  # still checked
    assert not calls

    monkeypatch.setattr(logprobs, "_torch", lambda: torch)
    monkeypatch.setattr(logprobs, "_on_device", lambda torch, what, *ts: 0)
    r = logprobs.token_logprobs(torch.zeros(0, 100), torch.zeros(0, dtype=torch.int32), top_n=3)
    assert r.logprobs.shape == r.entropy.shape == (0,)
    assert r.top_ids.shape == r.top_logprobs.shape == (0, 3)
    assert logprobs.token_logprobs(torch.zeros(0, 100)).top_ids is None


def test_most_of_the_tokens_as_a_tensor(batch, calls):
    """max_q as what the caller's own arithmetic left it in."""
    q, start = torch.zeros(2, 4, 64), torch.tensor([0, 2, 2], dtype=torch.int32)
    batch.attend(q, q_start=start, max_q=start.diff().max())
    assert type(calls[-1][1][5]) is int and calls[-1][1][5] == 2


FAR = -2 ** 32  # FAR + 5 is 5 to a C int


def test_numbers_below_an_int_stay_negative(batch, calls):
    """Such a window, bound or most of tokens reaches the library as a negative number, which it
    refuses, and not as what is left of its low bits."""
    q, start = torch.zeros(2, 4, 64), torch.zeros(3, dtype=torch.int32)
    batch.attend(q, window=FAR + 5, max_len=FAR + 7, q_start=start, max_q=FAR + 9)
    name, a = calls[-1]
    assert name == "attn" and a[10]._obj.window < 0 and a[8] < 0 and a[5] < 0
    batch.read(2, q_start=start, max_q=FAR + 9)
    assert calls[-1][1][3] < 0
    batch.workspace_bytes(FAR + 2, 4, q_start=start, max_q=FAR + 9, max_len=FAR + 7)
    name, a = calls[-1]
    assert name == "bytes" and a[1] < 0 and a[3] < 0 and a[5] < 0
    batch.workspace_bytes(2, 2 ** 32 + 4)
    assert calls[-1][1][4] == 2 ** 31 - 1


@pytest.mark.parametrize("over", [dict(n_pages=2 ** 32 + 1), dict(page_size=2 ** 32 + 16),
                                  dict(n_kv_heads=2 ** 32 + 2), dict(head_dim=2 ** 32 + 64),
                                  dict(head_dim=64 - 2 ** 32)])
def test_cache_shapes_past_an_int(monkeypatch, over):
    from cortexsdr_amd import paged

    monkeypatch.setattr(paged, "_torch", lambda: torch)
    monkeypatch.setattr(paged, "_on_device", lambda torch, what, *ts: 0)
    a = dict(n_pages=1, page_size=16, n_kv_heads=2, head_dim=64)
    k = torch.zeros(1, 4096, dtype=torch.uint8)
    paged.PagedCache(**a, k=k, v=k)
    with pytest.raises(ValueError):
        paged.PagedCache(**{**a, **over}, k=k, v=k)


@pytest.mark.parametrize("top_n", [2 ** 32 + 3, 2 ** 31, 65, -1, FAR + 3])
def test_more_places_than_the_top_has(monkeypatch, top_n):
    """Refused by the library as it is, without a list of that length first."""
    from cortexsdr_amd import _lib, logprobs, paged

    monkeypatch.setattr(paged, "_torch", lambda: torch)
    monkeypatch.setattr(logprobs, "_torch", lambda: torch)
    monkeypatch.setattr(logprobs, "_on_device", lambda torch, what, *ts: 0)
    monkeypatch.setattr(logprobs, "_stream_of", lambda torch, dev, stream: 0)
    sizes, empty = [], logprobs._empty
    monkeypatch.setattr(logprobs, "_empty", lambda torch, shape, *a: sizes.append(shape) or
                        empty(torch, (2, 8), *a))
    with pytest.raises(_lib.CsdrError, match="top_n"):
        logprobs.token_logprobs(torch.zeros(2, 100), top_n=top_n)
    assert sizes == [(2, 2)]
