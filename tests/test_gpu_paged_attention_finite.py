"""The numeric tests of paged attention once more, with a check that a NaN does not pass: every output
within its tolerance, every tolerance finite."""
import pytest
import torch

import test_gpu_paged_attention as base

pytestmark = pytest.mark.gpu


def _check(o, want, off, v, dtype):
    top = v.double().abs().max()
    tol = 2 * off[..., None] * top * torch.ones_like(want)
    if dtype == torch.bfloat16:
        tol = tol + want.abs() * 2.0 ** -8 + top * 2.0 ** -16
    assert bool(tol.isfinite().all()) and o.shape == want.shape
    assert bool(((o.double() - want).abs() <= tol).all())


@pytest.fixture(autouse=True)
def positive(monkeypatch):
    monkeypatch.setattr(base, "_check", _check)


def test_the_check_fails_on_nan():
    one = torch.ones(1, 1, 1, dtype=torch.float64)
    for o, v in ((float("nan"), 1.0), (1.0, float("nan")), (1.0, float("inf")), (1.1, 1.0)):
        with pytest.raises(AssertionError):
            _check(one.float() * o, one, one[0] * 1e-6, torch.tensor(v), torch.float32)
    _check(one.float(), one, one[0] * 1e-6, torch.tensor(1.0), torch.float32)


test_matches_the_definition = base.test_matches_the_definition
test_new_token_counts_and_is_stored = base.test_new_token_counts_and_is_stored
test_gate_of_zero_and_one = base.test_gate_of_zero_and_one
test_bad_pages_and_lengths = base.test_bad_pages_and_lengths
test_shared_pages_may_be_read_by_all = base.test_shared_pages_may_be_read_by_all
test_rows_at_any_stride = base.test_rows_at_any_stride
test_offsets_beyond_32_bits = base.test_offsets_beyond_32_bits
test_shapes_of_the_cut = base.test_shapes_of_the_cut
test_lengths_around_the_tiles = base.test_lengths_around_the_tiles
