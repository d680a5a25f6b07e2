"""CPU: the oracle of the expert-sorted data movement against small cases worked
by hand, and the refusals of its entry points (C ABI and Python) before any launch."""
import ctypes

import pytest
import torch

import fack_b200 as fb
from fack_b200 import _lib, moe
from oracle import moe as orc

OK_PTR = 1 << 20     # a well-aligned address that nothing may follow
BAD_SHAPE, BAD_ALIGN, BAD_STRIDE, WS, BAD_ARG = (_lib.FACK_ERR_BAD_SHAPE, _lib.FACK_ERR_BAD_ALIGN,
                                                 _lib.FACK_ERR_BAD_STRIDE, _lib.FACK_ERR_WS_TOO_SMALL,
                                                 _lib.FACK_ERR_BAD_ARG)


def test_oracle_sort_by_hand():
    ids = torch.tensor([[2, 0], [2, 2], [-1, 0], [9, 1]])
    row_of, src, offsets = orc.sort_ref(ids, 3)
    assert offsets.tolist() == [0, 2, 3, 6]
    assert src.tolist() == [1, 5, 7, 0, 2, 3, -1, -1]
    assert row_of.tolist() == [[3, 0], [4, 5], [-1, 1], [-1, 2]]
    x = torch.arange(4.0)[:, None] + 1
    assert orc.gather_ref(x, src, 2)[:, 0].tolist() == [1, 3, 4, 1, 2, 2, 0, 0]
    out, _ = orc.combine_ref(torch.arange(8.0)[:, None], torch.full((4, 2), 0.5), row_of)
    assert out[:, 0].tolist() == [1.5, 4.5, 0.5, 1.0]


def sort_args(**kw):
    a = dict(ids=OK_PTR, ids_bytes=8, T=4, topk=2, E=8, row_of=OK_PTR, src=OK_PTR, offsets=OK_PTR, ws=None, nb=0)
    a.update(kw)
    return (*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(T=0), BAD_SHAPE), (dict(topk=0), BAD_SHAPE), (dict(topk=65), BAD_SHAPE), (dict(E=0), BAD_SHAPE),
    (dict(E=1025), BAD_SHAPE), (dict(T=1 << 30, topk=2), BAD_SHAPE), (dict(ids_bytes=2), BAD_ARG),
    (dict(ids=None), BAD_ALIGN), (dict(ids=OK_PTR + 4), BAD_ALIGN), (dict(src=OK_PTR + 2), BAD_ALIGN),
    (dict(T=1 << 20), WS), (dict(T=1 << 20, ws=OK_PTR, nb=16), WS)])
def test_sort_refusals(kw, status):
    assert _lib.load().fack_moe_sort(*sort_args(**kw)) == status


def test_sort_workspace_is_small_and_zero_for_few_pairs():
    nb = ctypes.c_size_t(1)
    f = _lib.load().fack_moe_sort_workspace_size
    assert f(1, 8, 256, ctypes.byref(nb)) == 0 and nb.value == 0
    assert f(1 << 20, 8, 256, ctypes.byref(nb)) == 0 and 0 < nb.value <= 256 * 256 * 4
    assert f(1, 8, 256, None) == BAD_ARG


def call(name, **kw):
    base = {
        "fack_moe_gather": dict(x=OK_PTR, dtype=1, ldx=64, T=4, topk=2, D=64, row_of=OK_PTR, offsets=OK_PTR, E=8,
                                y=OK_PTR, ldy=64),
        "fack_moe_gather_quant": dict(x=OK_PTR, dtype=1, ldx=256, T=4, topk=2, D=256, row_of=OK_PTR, offsets=OK_PTR,
                                      E=8, y=OK_PTR, ldy=256, xs=OK_PTR, lds=2),
        "fack_moe_combine": dict(y=OK_PTR, dtype=1, ldy=64, w=OK_PTR, T=4, topk=2, D=64, row_of=OK_PTR, out=OK_PTR,
                                 ldo=64),
        "fack_moe_combine_bwd": dict(dout=OK_PTR, dtype=1, ldd=64, y=OK_PTR, ldy=64, w=OK_PTR, T=4, topk=2, D=64,
                                     row_of=OK_PTR, offsets=OK_PTR, E=8, dy=OK_PTR, lddy=64, dw=OK_PTR)}[name]
    assert set(kw) <= set(base)
    return getattr(_lib.load(), name)(*{**base, **kw}.values(), None)


@pytest.mark.parametrize("name,kw,status", [
    ("fack_moe_gather", dict(dtype=3), BAD_ARG), ("fack_moe_gather", dict(D=0), BAD_SHAPE),
    ("fack_moe_gather", dict(D=(1 << 20) + 1, ldy=1 << 21), BAD_SHAPE), ("fack_moe_gather", dict(ldy=63), BAD_STRIDE),
    ("fack_moe_gather", dict(ldx=-1), BAD_STRIDE), ("fack_moe_gather", dict(x=OK_PTR + 1), BAD_ALIGN),
    ("fack_moe_gather", dict(row_of=None), BAD_ALIGN), ("fack_moe_gather", dict(E=0), BAD_SHAPE),
    ("fack_moe_gather_quant", dict(dtype=2), BAD_ARG), ("fack_moe_gather_quant", dict(D=192, ldx=192), BAD_SHAPE),
    ("fack_moe_gather_quant", dict(ldy=128), BAD_STRIDE), ("fack_moe_gather_quant", dict(lds=1), BAD_STRIDE),
    ("fack_moe_gather_quant", dict(ldx=260), BAD_STRIDE), ("fack_moe_gather_quant", dict(x=OK_PTR + 2), BAD_ALIGN),
    ("fack_moe_combine", dict(dtype=7), BAD_ARG), ("fack_moe_combine", dict(topk=65), BAD_SHAPE),
    ("fack_moe_combine", dict(ldo=1), BAD_STRIDE), ("fack_moe_combine", dict(out=None), BAD_ALIGN),
    ("fack_moe_combine", dict(w=OK_PTR + 2), BAD_ALIGN),
    ("fack_moe_combine_bwd", dict(dy=None, dw=None), BAD_ARG), ("fack_moe_combine_bwd", dict(w=None), BAD_ALIGN),
    ("fack_moe_combine_bwd", dict(y=None), BAD_ALIGN), ("fack_moe_combine_bwd", dict(lddy=3), BAD_STRIDE),
    ("fack_moe_combine_bwd", dict(T=0), BAD_SHAPE)])
def test_row_entry_refusals(name, kw, status):
    assert call(name, **kw) == status


def test_python_entries_refuse_cpu_tensors_and_wrong_forms():
    ids = torch.zeros((4, 2), dtype=torch.int64)
    plan = fb.MoePlan(*orc.sort_ref(ids, 3))
    x = torch.zeros((4, 128))
    for f in (lambda: fb.moe_sort(ids, 3), lambda: fb.moe_sort(None, 3), lambda: fb.moe_gather(x, plan),
              lambda: fb.moe_gather_quant(x, plan), lambda: fb.moe_combine(torch.zeros((8, 128)), torch.ones((4, 2)), plan),
              lambda: fb.moe_combine(torch.zeros((8, 128)), None, plan),
              lambda: fb.moe_combine_backward(x, None, torch.ones((4, 2)), plan), lambda: fb.moe_gather(None, plan),
              lambda: fb.moe_gather(x.clone().requires_grad_(), plan)):
        with pytest.raises(ValueError):
            f()


def test_plan_checks():
    ids = torch.zeros((4, 2), dtype=torch.int64)
    plan = fb.MoePlan(*orc.sort_ref(ids, 3))
    cpu = torch.device("cpu")
    assert moe._check_plan(plan, cpu) == (4, 2, 3)
    for bad in (plan._replace(row_of=plan.row_of.long()), plan._replace(src=plan.src[:7]),
                plan._replace(offsets=plan.offsets[:1]), plan._replace(row_of=plan.row_of.t()),
                plan._replace(row_of=plan.row_of.reshape(-1)), plan._replace(offsets=None), tuple(plan), None):
        with pytest.raises(ValueError):
            moe._check_plan(bad, cpu)


def test_quant_rows_of_every_type_are_16_byte_strides():
    """fp32 strides are multiples of 4 elements, bf16 ones of 8."""
    for dtype, bad in ((0, (257, 258, 262)), (1, (257, 260, 268))):
        for ldx in bad:
            assert call("fack_moe_gather_quant", dtype=dtype, ldx=ldx) == BAD_STRIDE
