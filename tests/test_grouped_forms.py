"""Which kernel a 16-bit product takes: the cases of test_gpu_grouped_forms.py are those of the forms that they name,
and no form is without one.  No GPU: the choice is the host's."""
from __future__ import annotations

import pytest

import test_gpu_grouped_forms as F
from hmoe import capi


def test_every_form_has_cases():
    by_kind = {}
    for form, kind, *_ in F.CASES + F.ADAPTERS:
        by_kind.setdefault(kind, set()).add(form)
    streams = {F.S1, F.S2, F.S4}
    assert by_kind[F.MATMUL] == {256, 128, 64, 32} | streams
    assert by_kind[F.SWIGLU] == {256, 128, 64, 32} | streams
    assert by_kind[F.TRANSPOSED] == {256, 128, 64, 32, 0} and by_kind[F.SWIGLU_GRAD] == {128, 64, 32, 0}
    assert by_kind[F.WEIGHT_GRAD] == {256, 64, 32, 0}
    assert by_kind[F.ADAPTER] == {256, 128, 64, 32} | streams | {F.S8}
    assert by_kind[F.ADAPTER_T] == {256, 128, 64, 32, 0}


@pytest.mark.parametrize("case", F.CASES, ids=lambda c: f"{c[0]}-{c[1]}-{c[3]}x{c[4]}")
def test_grouped(case):
    form, kind, counts, inner, cols, rank, aligned = case
    assert F._form(capi, kind, counts, inner, cols, rank, aligned) == form


@pytest.mark.parametrize("case", F.ADAPTERS, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}")
def test_adapters(case):
    form, kind, rows, inner, cols, rank, aligned = case
    assert capi.load().hm_debug_grouped_form(kind, 1, rows, inner, cols, rank, aligned) == form


def test_no_call():
    f = capi.load().hm_debug_grouped_form
    for bad in ((-1, 1, 1, 1, 1, 0, 1), (7, 1, 1, 1, 1, 0, 1), (0, 0, 1, 1, 1, 0, 1), (0, 1, 0, 1, 1, 0, 1),
                (0, 1025, 1, 1, 1, 0, 1), (0, 1, 1, 0, 1, 0, 1), (0, 1, 1, 1, 1 << 27, 0, 1)):
        assert f(*bad) == -1, bad
