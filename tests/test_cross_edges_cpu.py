"""Refusals of the backward entry for FP32 tables.  CPU only: no call here
launches work."""

import pytest

import python._lib as L
from test_cross_attention_cpu import BIAS, TRAIN, lib, raw  # noqa: F401


@pytest.mark.parametrize(
    "kw,pointers",
    [
        (dict(lse=16), {}),
        (dict(TRAIN, Nk=0), {}),
        (dict(TRAIN, **BIAS, distance=16), dict(dtable=None)),
        (dict(TRAIN, **BIAS, distance=16), dict(dtable=18)),  # aligned for a 16-bit table only
        (dict(TRAIN, **BIAS, distance=16), dict(dq=8)),
    ],
)
def test_fp32_table_entry_refuses(lib, kw, pointers):  # noqa: F811
    at = dict(dict(dout=16, dq=16, dk=16, dv=16, dtable=16, scratch=16), **pointers)
    assert lib.sma_cross_attn_bwd_f32_table(raw(**kw), *at.values(), None) == L.SMA_ERR_ARG
    assert lib.sma_last_error()
