"""What speculative.Head, and a stream that is given one, refuse before a pass has run.  No GPU is needed: nothing is computed."""
import math

import pytest
import torch


@pytest.fixture(scope="module")
def spec():
    import __graft_entry__ as ge
    ge.build()
    from crucible_strix_halo_b200 import speculative
    return speculative


def _matrix(rows):
    from crucible_strix_halo_b200 import layers
    return layers.Mx4.empty(rows, 64, device="cpu")


@pytest.mark.parametrize("rows,refused", [
    (1003, {}), (1003, dict(vocabulary=1003)),                   # outputs of the head product hold a multiple of 32 columns
    (1024, dict(vocabulary=1025)), (1024, dict(vocabulary=0)),
    (64, dict(bias=torch.zeros(63))), (64, dict(bias=torch.zeros(64).double())), (64, dict(bias=torch.zeros(128)[::2])),
    (64, dict(repetition=0.0)), (64, dict(repetition=math.nan)), (64, dict(frequency=math.inf)), (64, dict(presence=math.nan)),
])
def test_heads_that_are_refused(spec, rows, refused):
    with pytest.raises(ValueError):
        spec.Head(_matrix(rows), **refused)


def test_a_vocabulary_smaller_than_the_matrix(spec):
    head = spec.Head(_matrix(1024), vocabulary=1003, bias=torch.zeros(1003))
    assert head.counts.shape == (1003,) and head.logits.shape == (13, 1024)
    assert spec.Head(_matrix(1024)).counts.shape == (1024,)


def test_a_head_of_fewer_rows_than_a_span(spec):
    with pytest.raises(ValueError, match="rows"):
        spec.SpecStream(None, [], None, None, None, 64, span=9, head=spec.Head(_matrix(64), rows=8))
