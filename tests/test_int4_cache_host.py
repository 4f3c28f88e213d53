"""Cropping of the transformers cache view over ragged sequences, on a stand-in for its manager (no GPU)."""
import pytest

from logitfill_amd.packed import LogitFillCache


class _Layer:
    def __init__(self, lengths):
        self.lengths = list(lengths)


class _Manager:
    """What the view sees of an ``Int4KVManager``."""

    def __init__(self, lengths):
        self.layers, self.calls = [_Layer(lengths), _Layer(lengths)], 0

    seq_len = property(lambda self: self.layers[-1].lengths[0])

    def truncate(self, lengths):
        self.calls += 1
        for layer in self.layers:
            assert all(0 <= n <= have for n, have in zip(lengths, layer.lengths))
            layer.lengths = list(lengths)


@pytest.mark.parametrize("lengths,crop,want", [
    ([100, 60], -3, [97, 57]),
    ([60, 100], -3, [57, 97]),
    ([60, 100], 80, [60, 80]),
    ([5, 10], 7, [5, 7]),
    ([10, 5], -6, [4, 0]),
    ([10, 5], 0, [0, 0]),
    ([10, 5], 11, [10, 5]),
    ([0, 4], -1, [0, 3]),
])
def test_crop_is_of_every_sequence(lengths, crop, want):
    mgr = _Manager(lengths)
    cache = LogitFillCache(mgr)
    cache.crop(crop)
    assert [layer.lengths for layer in mgr.layers] == [want] * 2
    assert cache.get_seq_length() == want[0] and mgr.calls == int(want != lengths)
