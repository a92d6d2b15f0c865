"""Outputs of the serving operators that lie over what is read are refused, before
anything touches a GPU."""

import pytest

from rpgbarengine_amd import serving
from test_cpu_serving import A, ref, refused, rows, seqs
from test_cpu_serving_more import edits, quant


@pytest.mark.parametrize("kind,size", [(0, 4), (1, 2), (30, 2)])
@pytest.mark.parametrize("n,stride,out_stride,off", [
    (3, 300, 300, 1), (3, 300, 300, -1), (3, 300, 300, 299), (3, 300, 300, 300), (3, 300, 300, -600), (3, 300, 300, 899),
    (3, 640, 640, 299), (3, 640, 640, 341), (3, 640, 640, -341 - 640), (3, 640, 640, 640), (1, 300, 300, 299), (1, 300, 300, -299),
    (3, 640, 700, 300), (3, 0, 300, 299), (3, 0, 300, -600), (2, 300, 1000, -700)])
def test_logits_edited_over_themselves(kind, size, n, stride, out_stride, off):
    refused(serving._lib().rpg_hip_edit_logits(kind, A, n, 300, stride, ref(edits(history=None)), A + off * size, out_stride, None),
            "out overlaps logits")


@pytest.mark.parametrize("n,stride,out_stride,off", [
    (3, 300, 300, 900), (3, 300, 300, -900), (3, 640, 640, 300), (3, 640, 640, 340), (3, 640, 640, -300), (3, 640, 640, 640 + 320),
    (1, 300, 300, 300), (1, 300, 300, -300), (3, 0, 300, 300), (3, 0, 300, -900), (3, 300, 300, 0)])
def test_logits_apart_are_no_overlap(n, stride, out_stride, off):
    """What is refused here is the next argument in order."""
    refused(serving._lib().rpg_hip_edit_logits(1, A, n, 300, stride, ref(edits(repetition=A + 1)), A + off * 2, out_stride, None),
            "row parameter")


@pytest.mark.parametrize("kind", [0, 1, 30])
def test_keys_and_values_read_into_the_same_rows(kind):
    refused(serving._lib().rpg_hip_quant_read(ref(quant()), ref(seqs()), kind, ref(rows()), ref(rows()), None), "the same rows")
