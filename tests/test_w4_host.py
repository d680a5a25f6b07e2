"""CPU: the oracle of the 4-bit products on a case worked by hand, and the
refusals of their entry points (C ABI and Python) before any launch."""
import pytest
import torch

import fack_b200 as fb
from fack_b200 import _lib
from oracle import w4 as orc

OK_PTR = 1 << 20     # a well-aligned address that nothing may follow
BAD_SHAPE, BAD_ALIGN, BAD_STRIDE, BAD_ARG = (_lib.FACK_ERR_BAD_SHAPE, _lib.FACK_ERR_BAD_ALIGN,
                                             _lib.FACK_ERR_BAD_STRIDE, _lib.FACK_ERR_BAD_ARG)
F32, BF16, F16 = _lib.FACK_DTYPE_F32, _lib.FACK_DTYPE_BF16, _lib.FACK_DTYPE_F16


def test_oracle_by_hand():
    w = torch.zeros((1, 32), dtype=torch.uint8)
    w[0, 0], w[0, 31] = 0x3A, 0xF0            # codes 10, 3, 0, ..., 0, 15
    scales = torch.tensor([[0.5], [2.0]])
    v = orc.weights_ref(w, scales, None)
    assert v[0, :3].tolist() == [1.0, -2.5, -4.0] and v[0, 31] == -4.0 and v[0, 32] == -16.0 and v[0, 63] == 14.0
    v = orc.weights_ref(w, scales, torch.tensor([[3], [15]], dtype=torch.uint8))
    assert v[0, :2].tolist() == [3.5, 0.0] and v[0, 62:].tolist() == [-30.0, 0.0]


def call(experts=False, **kw):
    a = dict(x=OK_PTR, dtype=BF16, ldx=256, w=OK_PTR, scales=OK_PTR, sdtype=BF16, zeros=None, G=128)
    if experts:
        a.update(src=OK_PTR, offsets=OK_PTR, T=4, topk=2, E=8, y=OK_PTR, ldy=64, N=64, K=256)
    else:
        a.update(y=OK_PTR, ldy=64, M=4, N=64, K=256)
    assert set(kw) <= set(a)
    a.update(kw)
    lib = _lib.load()
    return (lib.fack_gemv_w4_experts if experts else lib.fack_gemv_w4)(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(N=63), BAD_SHAPE), (dict(N=0), BAD_SHAPE), (dict(N=72), BAD_SHAPE), (dict(K=0), BAD_SHAPE),
    (dict(K=(1 << 20) + 128), BAD_SHAPE), (dict(G=16), BAD_ARG), (dict(G=96), BAD_ARG), (dict(G=192), BAD_ARG),
    (dict(K=320), BAD_ARG), (dict(G=0), BAD_ARG), (dict(G=-128), BAD_ARG), (dict(dtype=F32), BAD_ARG),
    (dict(sdtype=F16), BAD_ARG), (dict(dtype=F16), BAD_ARG), (dict(x=OK_PTR + 8), BAD_ALIGN), (dict(w=None), BAD_ALIGN),
    (dict(w=OK_PTR + 1), BAD_ALIGN), (dict(scales=OK_PTR + 2), BAD_ALIGN), (dict(zeros=OK_PTR + 1), BAD_ALIGN),
    (dict(y=OK_PTR + 1), BAD_ALIGN), (dict(ldx=260), BAD_STRIDE), (dict(ldx=-8), BAD_STRIDE), (dict(ldy=63), BAD_STRIDE)])
@pytest.mark.parametrize("experts", [False, True])
def test_refusals(experts, kw, status):
    assert call(experts, **kw) == status


@pytest.mark.parametrize("experts,kw,status", [
    (False, dict(M=0), BAD_SHAPE), (True, dict(T=0), BAD_SHAPE), (True, dict(topk=65), BAD_SHAPE),
    (True, dict(E=0), BAD_SHAPE), (True, dict(E=1025), BAD_SHAPE), (True, dict(T=1 << 30), BAD_SHAPE),
    (True, dict(offsets=None), BAD_ALIGN), (True, dict(src=OK_PTR + 1), BAD_ALIGN)])
def test_refusals_of_one_form(experts, kw, status):
    assert call(experts, **kw) == status


def test_python_entries_refuse_cpu_tensors():
    x, w, s = torch.zeros((2, 256), dtype=torch.bfloat16), torch.zeros((64, 128), dtype=torch.uint8), torch.ones((2, 64))
    plan = fb.MoePlan(torch.zeros((2, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                      torch.zeros(4, dtype=torch.int32))
    for f in (lambda: fb.gemv_w4(x, w, s), lambda: fb.gemv_w4_experts(x, w[None], s[None], plan),
              lambda: fb.gemv_w4(None, w, s)):
        with pytest.raises(ValueError):
            f()


def test_weight_checks():
    """Every mismatch of a 4-bit weight's parts, on the CPU."""
    from fack_b200.w4 import _check_weight
    x, w, s = torch.zeros((2, 256), dtype=torch.bfloat16), torch.zeros((64, 128), dtype=torch.uint8), torch.ones((2, 64))
    z = torch.zeros((2, 64), dtype=torch.uint8)
    assert _check_weight(x, w, s, z, ()) == (64, 256, 128)
    assert _check_weight(x, w, torch.ones((1, 64)), None, ()) == (64, 256, 256)
    assert _check_weight(x, w[None], s[None].bfloat16(), z[None], (1,)) == (64, 256, 128)
    for bad in ((x, w.int(), s, z, ()), (x, w[:, :64], s, z, ()), (x, w, s.half(), z, ()), (x, w, s[:, :48], z, ()),
                (x, w, s, z[:1], ()), (x, w, s.t().contiguous().t(), z, ()), (x, w[:, ::2], s, z, ()),
                (x, w, torch.ones((3, 64)), None, ()), (x, w, torch.ones((16, 64)), None, ()),
                (x, w[:40], s[:, :40].contiguous(), None, ()), (x, w[None], s[None], None, (2,)), (x, w, s, z.int(), ()),
                (x.clone().requires_grad_(), w, s, z, ()), (x, w, s.clone().requires_grad_(), z, ()),
                (x, None, s, z, ()), (x, w, None, z, ())):
        with pytest.raises(ValueError):
            _check_weight(*bad)
    with torch.no_grad():
        assert _check_weight(x.clone().requires_grad_(), w, s, z, ()) == (64, 256, 128)


@pytest.mark.parametrize("args,status", [
    ((0, 0, 0, 64, 256, 128), BAD_SHAPE), ((4, 2, 0, 64, 256, 128), BAD_SHAPE), ((4, 0, 8, 64, 256, 128), BAD_SHAPE),
    ((4, 65, 8, 64, 256, 128), BAD_SHAPE), ((4, 2, 1025, 64, 256, 128), BAD_SHAPE), ((1 << 30, 2, 8, 64, 256, 128), BAD_SHAPE),
    ((4, 0, 0, 72, 256, 128), BAD_SHAPE), ((4, 0, 0, 64, 0, 128), BAD_SHAPE), ((4, 0, 0, 64, 256, 96), BAD_ARG),
    ((4, 0, 0, 64, 320, 128), BAD_ARG)])
def test_plan_refusals(args, status):
    import ctypes
    out = [ctypes.c_int() for _ in range(4)]
    assert _lib.load().fack_gemv_w4_plan(*args, *map(ctypes.byref, out)) == status
    assert _lib.load().fack_gemv_w4_plan(4, 0, 0, 64, 256, 128, None, *map(ctypes.byref, out[1:])) == BAD_ARG
