"""Host side of the decoding path, without a GPU: sizes of caches, counts of 64 bits, rows
that share memory."""
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


def _layouts(dtype=torch.float32, device="cpu"):
    """(cache [pages, slots, heads, 8], whether its rows lie apart)."""
    flat = torch.zeros(4096, dtype=dtype, device=device)

    def view(shape, *strides):
        return flat.as_strided((*shape, 8), (*strides, 1))

    return [
        (view((4, 4, 2), 64, 16, 8), True),
        (view((4, 4, 2), 64, 8, 32), True),                   # heads before slots
        (view((4, 4, 2), 16, 64, 8), True),                   # slots before pages
        (view((4, 4, 2), 8, 64, 32), True),
        (view((3, 5, 1), 80, 16, 0), True),                   # room behind every row; a single head
        (view((1, 1, 7), 0, 0, 9), True),
        (view((0, 4, 2), 0, 0, 0), True),
        (flat.view(4, 2, 8, 64).transpose(1, 2)[..., :8], True),
        (view((4, 4, 2), 64, 8, 8), False),                   # a slot's second head is the next one's first
        (view((4, 4, 2), 16, 8, 64), False),
        (view((4, 4, 2), 56, 16, 8), False),                  # a page begins in the one before
        (view((4, 4, 2), 64, 12, 8), False),
        (view((4, 4, 2), 64, 16, 4), False),
        (view((4, 4, 2), 0, 16, 8), False),
        (view((2, 2, 2), 8, 8, 8), False),
    ]


def test_caches_whose_rows_overlap_are_refused():
    table = torch.zeros(1, 2, dtype=torch.int32)
    for k, apart in _layouts():
        if apart:
            ops._paged_inputs(k, k, table, 1, "")
        else:
            with pytest.raises(ValueError, match="apart"):
                ops._paged_inputs(k, k, table, 1, "")
    flat = torch.zeros(400)
    ops._mass_inputs(flat.as_strided((3, 2, 10), (10, 30, 1)), 3, 2, "mass")
    ops._mass_inputs(flat.as_strided((1, 2, 10), (0, 12, 1)), 1, 2, "mass")
    for strides in ((10, 20, 1), (20, 9, 1), (10, 10, 1), (15, 10, 1)):
        with pytest.raises(ValueError, match="separate"):
            ops._mass_inputs(flat.as_strided((3, 2, 10), strides), 3, 2, "mass")
