"""Host side of the decoding path, without a GPU: sizes of caches, counts of 64 bits."""
import pytest
import torch

from mk_iii_technologies_tsrn_b200 import dropin, ops


class _Asked(Exception):
    pass


@pytest.fixture
def asked(monkeypatch):
    """The slots that generate() asks a cache for."""
    def cache(layers, batch, heads, channels, max_slots, **kw):
        raise _Asked(max_slots)

    monkeypatch.setattr(dropin, "TropicalPagedKVCache", cache)
    model = dropin.TropicalDecoderModel(20, d_model=16, nhead=2, num_layers=1, dim_feedforward=16,
                                        max_seq_len=200).eval()

    def slots(L, new, **kw):
        with pytest.raises(_Asked) as e:
            model.generate(torch.zeros(2, L, dtype=torch.int64), new, **kw)
        return e.value.args[0]

    return slots


def test_a_budget_takes_no_more_room_than_the_tokens(asked):
    assert asked(10, 5) == 14
    assert asked(10, 5, keep=10 ** 9) == 14 and asked(10, 5, keep=14) == 14
    assert asked(10, 1, keep=3, page_size=4) == 10
    assert asked(10, 100, keep=20, page_size=16) == 36            # the budget and a page
    assert asked(60, 100, keep=20, page_size=16) == 60            # the prompt
    assert asked(10, 100, keep=20, page_size=10 ** 6) == 109      # (a page is beyond all tokens)


def test_counts_of_requests_keep_their_meaning():
    k = torch.tensor([2 ** 32 + 1, 2 ** 31, -2 ** 40, 0, 50, 2 ** 63 - 1])
    assert ops._counts_of_rows(k).tolist() == [2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, 0, 50, 2 ** 31 - 1]
    for dtype in (torch.int32, torch.int16, torch.uint8):
        assert ops._counts_of_rows(torch.tensor([3, 0], dtype=dtype)).tolist() == [3, 0]
    for bad in (torch.tensor([0.9, 5.0]), torch.tensor([True, False])):
        with pytest.raises(ValueError, match="top_k"):
            ops.sample_tokens(torch.randn(2, 9), torch.rand(2), top_k=bad)
