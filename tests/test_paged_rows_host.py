"""How Engine takes the paged calls' token rows: views whose rows are whole and aligned as they are, others copied."""

import types

import pytest
import torch

from fast_dllm_relax_b200.engine import Engine

SELF = types.SimpleNamespace(dtype=torch.bfloat16, device=torch.device("cpu"), _esz=2)


def take(t, rows, cols):
    out = Engine._token_rows(SELF, t, rows, cols, "rows")
    assert out.shape == (rows, cols) and torch.equal(out, t.reshape(rows, cols))
    assert out.stride(1) == 1 and out.stride(0) >= cols and out.stride(0) * 2 % 16 == 0 and out.data_ptr() % 16 == 0
    return out


def values(*shape):
    return torch.arange(torch.Size(shape).numel(), dtype=torch.float32).bfloat16().view(shape)


def test_aligned_views_pass_as_they_are():
    wide = values(6, 192)
    for view in (wide[:, :64], wide[:, 64:128], wide[::2, 128:], wide[2:3, 64:128]):
        assert take(view, *view.shape).data_ptr() == view.data_ptr()


def test_other_views_are_copied():
    wide = values(6, 193)
    for view in (wide[:, 1:65], wide[:, :64], values(64, 3).t(), values(6, 1)[:, :1].expand(6, 64), wide[1:2, 1:65]):
        take(view, *view.shape)


@pytest.mark.parametrize("view", [values(64, 1).t(), values(64, 2)[:, :1].t(), values(64)[None],
                                  values(64).as_strided((1, 64), (3, 1)), values(72)[8:].as_strided((1, 64), (0, 1))],
                         ids=["column", "strided-column", "row", "short-stride", "no-stride"])
def test_one_row_of_any_stride(view):
    take(view, 1, 64)


def test_more_dimensions_are_flattened_where_the_rows_stay():
    take(values(3, 4, 16), 3, 64)
    take(values(1, 2, 2, 16), 1, 64)


def test_no_rows():
    assert Engine._token_rows(SELF, values(0, 64), 0, 64, "rows").shape == (0, 64)


@pytest.mark.parametrize("t", [values(3, 64).float(), values(2, 64), values(3, 32), values(192), values(3, 2, 16)], ids=lambda t: str(tuple(t.shape)))
def test_other_shapes_and_types_are_refused(t):
    with pytest.raises(ValueError, match="expected"):
        Engine._token_rows(SELF, t, 3, 64, "rows")
