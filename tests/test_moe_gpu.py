"""GPU: tokens sorted by expert and back against the 64-bit oracle.

Tolerances, from the arithmetic.  A copy and a sort are exact.  A sum of n
products in fp32 is off by at most n * 2^-24 of the sum of their magnitudes
(n fused multiply-adds, each rounded once); a rounding to type t adds
finfo(t).eps / 2 of the value, or half of its smallest subnormal below the
normal range."""
import pytest
import torch

import fack_b200 as fb
from oracle import moe as orc

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rounding(t, ref):
    """How far a value within fp32 reach of ref may be after one rounding to t."""
    info = torch.finfo(t)
    return ref.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def close(got, ref, tol):
    off = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got.float()).all()
    assert bool((off <= tol).all()), f"off by {float(off.max()):.3g}, {float((off - tol).max()):.3g} over"


def make_ids(T, k, E, seed, kind="topk", dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if kind == "topk":
        ids = torch.stack([torch.randperm(max(E, k), generator=g)[:k] for _ in range(T)]) if T else torch.zeros((0, k))
    elif kind == "one":                       # every pair to one expert
        ids = torch.full((T, k), E - 1)
    elif kind == "none":                      # nothing stays here
        ids = torch.where(torch.rand((T, k), generator=g) < 0.5, -1, E)
    else:                                     # any value, repeats within a token, far outside the range
        ids = torch.randint(-3, E + 3, (T, k), generator=g)
        ids[torch.rand((T, k), generator=g) < 0.05] = 2 ** 31 - 1 if dtype == torch.int32 else 2 ** 32 + 1
    return ids.to(dtype)


def gpu_plan(T, k, E, seed, dev, kind="any"):
    return fb.moe_sort(make_ids(T, k, E, seed, kind).to(dev), E)


@pytest.mark.parametrize("kind", ["topk", "one", "none", "any"])
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 256), (7, 3, 5), (64, 8, 64), (255, 2, 1024), (600, 8, 130),
                                   (3000, 8, 256), (9001, 6, 64), (20000, 1, 1000)])
def test_sort(cuda_device, T, k, E, kind):
    for dtype in (torch.int32, torch.int64):
        ids = make_ids(T, k, E, T + k + E, kind, dtype)
        plan = fb.moe_sort(ids.to(cuda_device), E)
        for got, ref in zip(plan, orc.sort_ref(ids, E)):
            assert got.dtype == torch.int32 and torch.equal(got.cpu(), ref)


def test_sort_many_chunks_a_block_against_a_stable_sort(cuda_device):
    T, k, E = 300001, 7, 97                   # over two million pairs: blocks walk several chunks each
    ids = make_ids(T, k, E, 3, "any").to(cuda_device)
    plan = fb.moe_sort(ids, E)
    flat = ids.reshape(-1)
    key, order = torch.sort(torch.where((flat >= 0) & (flat < E), flat, E), stable=True)
    offsets = torch.searchsorted(key, torch.arange(E + 1, device=cuda_device))
    src = torch.where(torch.arange(T * k, device=cuda_device) < offsets[E], order, -1)
    assert torch.equal(plan.offsets.long(), offsets) and torch.equal(plan.src.long(), src)
    n = int(offsets[E])
    row_of = torch.full((T * k,), -1, device=cuda_device)
    row_of[order[:n]] = torch.arange(n, device=cuda_device)
    assert torch.equal(plan.row_of.reshape(-1).long(), row_of)


def test_sort_takes_strided_ids(cuda_device):
    ids = make_ids(33, 4, 9, 5, "any").to(cuda_device)
    wide = torch.full((33, 8), 77, dtype=torch.int64, device=cuda_device)
    wide[:, ::2] = ids
    for view in (wide[:, ::2], ids.t().contiguous().t()):
        for a, b in zip(fb.moe_sort(view, 9), fb.moe_sort(ids, 9)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,E,D", [(1, 1, 1, 1), (1, 8, 16, 7168), (5, 3, 4, 33), (40, 8, 12, 2048), (130, 2, 9, 130),
                                     (400, 5, 3, 264), (17, 64, 30, 72)])
def test_gather_and_its_gradient(cuda_device, dtype, T, k, E, D):
    plan = gpu_plan(T, k, E, D + T, cuda_device)
    g = torch.Generator().manual_seed(T)
    x = torch.randn((T, D), generator=g).to(dtype)
    y = fb.moe_gather(x.to(cuda_device), plan)
    assert torch.equal(y.cpu(), orc.gather_ref(x, plan.src, k))
    xg = x.to(cuda_device).requires_grad_()
    y = fb.moe_gather(xg, plan)
    dy = torch.randn((T * k, D), generator=g).to(dtype)
    y.backward(dy.to(cuda_device))
    ref, mag = orc.combine_ref(dy, None, plan.row_of)
    close(xg.grad, ref, k * U32 * mag + rounding(dtype, ref))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,E,D", [(1, 1, 1, 1), (1, 8, 16, 7168), (5, 3, 4, 33), (40, 8, 12, 2048), (130, 2, 9, 130),
                                     (400, 5, 3, 264), (17, 64, 30, 72), (3, 9, 20, 4097)])
def test_combine_and_its_gradients(cuda_device, dtype, T, k, E, D):
    plan = gpu_plan(T, k, E, D + T + 1, cuda_device)
    g = torch.Generator().manual_seed(T)
    y = torch.randn((T * k, D), generator=g).to(dtype)
    routed = int(plan.offsets[-1])
    y[routed:] = float("nan")                 # nobody's rows are never read
    w = torch.randn((T, k), generator=g)
    dout = torch.randn((T, D), generator=g).to(dtype)
    ref, mag = orc.combine_ref(y, w, plan.row_of)
    out = fb.moe_combine(y.to(cuda_device), w.to(cuda_device), plan)
    close(out, ref, k * U32 * mag + rounding(dtype, ref))
    yg, wg = y.to(cuda_device).requires_grad_(), w.to(cuda_device).requires_grad_()
    out = fb.moe_combine(yg, wg, plan)
    dy, dw = torch.autograd.grad(out, (yg, wg), dout.to(cuda_device))
    rdy, rdw, mag = orc.combine_bwd_ref(dout, y, w, plan.row_of)
    assert dw.dtype == torch.float32
    close(dy, rdy, U32 * rdy.abs() + rounding(dtype, rdy))
    close(dw, rdw, D * U32 * mag)


def test_one_gradient_at_a_time(cuda_device):
    plan = gpu_plan(40, 4, 6, 1, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    y = torch.randn((160, 96), generator=g, device=cuda_device)
    w = torch.rand((40, 4), generator=g, device=cuda_device)
    dout = torch.randn((40, 96), generator=g, device=cuda_device)
    dy, dw = fb.moe_combine_backward(dout, y, w, plan)
    yg, wg = y.clone().requires_grad_(), w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(fb.moe_combine(yg, w, plan), yg, dout)[0], dy)
    assert torch.equal(torch.autograd.grad(fb.moe_combine(y, wg, plan), wg, dout)[0], dw)
    assert fb.moe_combine_backward(dout, None, w, plan, need_dweights=False)[1] is None
    assert torch.equal(fb.moe_combine_backward(dout, y, w, plan, need_dy=False)[1], dw)


def test_gradients_against_differences(cuda_device):
    """Both operators are linear in each argument, so a central difference of
    step 1 is the derivative up to fp32 rounding: of the outputs (k products
    each) and of the sums over T*D = 12000 of them, all in 64 bits after that."""
    T, k, E, D = 60, 3, 7, 200
    plan = gpu_plan(T, k, E, 11, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(4)
    rand = lambda *s: torch.randn(s, generator=g, device=cuda_device)  # noqa: E731
    y, w, x, dout, dy = rand(T * k, D), rand(T, k), rand(T, D), rand(T, D), rand(T * k, D)
    vy, vw, vx = rand(T * k, D), rand(T, k), rand(T, D)
    inner = lambda a, b: float((a.double() * b.double()).sum())  # noqa: E731

    def diff(f, at, v, weight):
        up, down = f(at + v), f(at - v)
        # an output is off by (k + 1) fp32 roundings of its terms' magnitudes, and the perturbed argument is
        # rounded once, which the linear map passes on: k + 2.  The terms' magnitudes, summed over the outputs,
        # are k * E|N(0,2)| * E|N(0,2)| = 3.8 each on average; 60 + the outputs' own stands far above that
        tol = (k + 2) * U32 * float((weight.abs().double() * (up.abs().double() + down.abs().double() + 60.0)).sum())
        return inner(weight, up.double() - down.double()) / 2, tol

    routed = int(plan.offsets[-1])
    vy[routed:] = 0
    fd, tol = diff(lambda a: fb.moe_combine(a, w, plan), y, vy, dout)
    gy, gw = fb.moe_combine_backward(dout, y, w, plan)
    assert abs(fd - inner(gy, vy)) <= tol
    fd, tol = diff(lambda a: fb.moe_combine(y, a, plan), w, vw, dout)
    assert abs(fd - inner(gw, vw)) <= tol + D * U32 * float((vw.abs() * 60 * D).sum())
    fd, tol = diff(lambda a: fb.moe_gather(a, plan), x, vx, dy)
    assert abs(fd - inner(fb.moe_gather_backward(dy, plan), vx)) <= tol


def test_gradients_that_autograd_hands_out_broadcast_or_transposed(cuda_device):
    T, k, E, D = 30, 4, 8, 64
    plan = gpu_plan(T, k, E, 5, cuda_device)
    x = torch.randn((T, D), device=cuda_device)
    w = torch.rand((T, k), device=cuda_device)
    y = torch.randn((T * k, D), device=cuda_device)
    ones_t, ones_r = torch.ones((T, D), device=cuda_device), torch.ones((T * k, D), device=cuda_device)
    xg = x.clone().requires_grad_()
    fb.moe_gather(xg, plan).sum().backward()                       # a gradient of stride (0, 0)
    assert torch.equal(xg.grad, fb.moe_gather_backward(ones_r, plan))
    xg = x.clone().requires_grad_()
    col = torch.randn((D, T * k), device=cuda_device)
    (fb.moe_gather(xg, plan).t() * col).sum().backward()           # a transposed one
    assert torch.equal(xg.grad, fb.moe_gather_backward(col.t().contiguous(), plan))
    yg, wg = y.clone().requires_grad_(), w.clone().requires_grad_()
    fb.moe_combine(yg, wg, plan).sum().backward()
    dy, dw = fb.moe_combine_backward(ones_t, y, w, plan)
    assert torch.equal(yg.grad, dy) and torch.equal(wg.grad, dw)
    # broadcast inputs: one token's row for all, one weight row for all; their gradients sum over the tokens
    row, gate = torch.randn((1, D), device=cuda_device).requires_grad_(), torch.rand((1, k), device=cuda_device)
    out = fb.moe_gather(row.expand(T, D), plan)
    assert torch.equal(out, fb.moe_gather(row.detach().repeat(T, 1), plan))
    out.backward(ones_r)
    assert torch.equal(row.grad[0], torch.full((D,), float(plan.offsets[-1]), device=cuda_device))
    assert torch.equal(fb.moe_combine(y, gate.expand(T, k), plan), fb.moe_combine(y, gate.repeat(T, 1), plan))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off,width", [(0, 80), (1, 77), (2, 72), (8, 88), (4, 76), (0, 66), (0, 68)])
def test_strided_and_unaligned_rows(cuda_device, dtype, off, width):
    T, k, E, D = 20, 3, 5, 64
    plan = gpu_plan(T, k, E, off, cuda_device)
    wide = torch.randn((T * k, width + off), device=cuda_device).to(dtype)
    y = wide[:, off:off + D]
    w = torch.rand((T, k), device=cuda_device)
    x = y[:T]
    assert torch.equal(fb.moe_gather(x, plan), fb.moe_gather(x.contiguous(), plan))
    assert torch.equal(fb.moe_combine(y, w, plan), fb.moe_combine(y.contiguous(), w, plan))
    got, ref = fb.moe_combine_backward(x, y, w, plan), fb.moe_combine_backward(x.contiguous(), y.contiguous(), w, plan)
    assert torch.equal(got[0], ref[0])
    mag = orc.combine_bwd_ref(x, y, w, plan.row_of)[2]              # another access width adds in another order
    close(got[1], ref[1].cpu().double(), 2 * D * U32 * mag)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,k,E,K", [(1, 1, 1, 128), (3, 8, 20, 7168), (50, 2, 6, 640), (300, 4, 9, 1152), (6, 20, 8, 256)])
def test_gather_quant(cuda_device, dtype, T, k, E, K):
    plan = gpu_plan(T, k, E, K + T, cuda_device)
    g = torch.Generator().manual_seed(T)
    x = torch.randn((T, K), generator=g)
    x[0, :128] = 0
    if T > 2:
        x[1] *= 1e-30
        x[2, ::7] = -0.0
    x = torch.where(torch.rand((T, K), generator=g) < 1e-2, x * 50, x).to(dtype)
    xq, xs = fb.moe_gather_quant(x.to(cuda_device), plan)
    rq, rs = orc.gather_quant_ref(x, plan.src, k)
    assert torch.equal(xs.cpu(), rs) and torch.equal(xq.cpu().view(torch.uint8), rq.view(torch.uint8))
    q, s = fb.quantize_activations(x.to(cuda_device), layout="logical")      # the operator it joins with the gather
    rows = fb.moe_gather(torch.arange(T, device=cuda_device, dtype=torch.float32)[:, None], plan).long()[:, 0]
    n = int(plan.offsets[-1])
    assert torch.equal(xs[:n], s[rows[:n]])
    assert torch.equal(xq[:n].view(torch.uint8), q.view(torch.uint8)[rows[:n]])


def test_gather_quant_extremes(cuda_device):
    """NaN makes its own group NaN and no other; an infinity makes its finite
    neighbours 0; a group below what a scale can hold is zero, scale 1."""
    plan = fb.moe_sort(torch.zeros((4, 1), dtype=torch.int32, device=cuda_device), 1)
    x = torch.ones((4, 256))
    x[0, 3] = float("nan")
    x[1, 5] = float("inf")
    x[2, :128] = torch.finfo(torch.float32).max
    x[3, :128] = 0
    x[3, 7] = 1e-43
    xq, xs = fb.moe_gather_quant(x.to(cuda_device), plan)
    xq, xs = xq.float().cpu(), xs.cpu()
    assert xs[0, 0].isnan() and xq[0, :128].isnan().all() and (xq[0, 128:] == 240).all()
    assert xs[1, 0].isinf() and xq[1, 5].isnan() and (xq[1, :5] == 0).all() and (xq[1, 6:128] == 0).all()
    assert (xq[2, :128] == 240).all() and xs[3, 0] == 1 and (xq[3, :128] == 0).all()


def test_infinities_and_nan_stay_with_their_tokens(cuda_device):
    T, k, E, D = 12, 2, 4, 40
    plan = gpu_plan(T, k, E, 9, cuda_device, "topk")
    x = torch.randn((T, D), device=cuda_device)
    x[3] = float("nan")
    x[5] = float("inf")
    y = fb.moe_gather(x, plan)
    out = fb.moe_combine(y, torch.full((T, k), 0.5, device=cuda_device), plan)
    assert out[3].isnan().all() and out[5].isinf().all()
    keep = [t for t in range(T) if t not in (3, 5)]
    assert torch.equal(out[keep], x[keep])                    # 0.5 x + 0.5 x


def test_no_tokens(cuda_device):
    plan = fb.moe_sort(torch.zeros((0, 4), dtype=torch.int64, device=cuda_device), 6)
    assert plan.offsets.tolist() == [0] * 7 and plan.row_of.shape == (0, 4) and plan.src.numel() == 0
    x = torch.zeros((0, 256), device=cuda_device, requires_grad=True)
    w = torch.zeros((0, 4), device=cuda_device, requires_grad=True)
    y = fb.moe_gather(x, plan)
    out = fb.moe_combine(y, w, plan)
    out.sum().backward()
    assert out.shape == (0, 256) and x.grad.shape == (0, 256) and w.grad.shape == (0, 4)
    assert fb.moe_gather_quant(x.detach(), plan)[1].shape == (0, 2)


def test_plan_entries_out_of_range_count_as_unrouted(cuda_device):
    """A plan that moe_sort did not make cannot reach outside the rows."""
    T, k, D = 6, 2, 32
    row_of = torch.tensor([[0, 1], [2 ** 31 - 1, 3], [-5, 12], [-2 ** 31, 5], [99, 7], [8, 9]], dtype=torch.int32)
    src = torch.zeros(T * k, dtype=torch.int32)
    offsets = torch.tensor([0, -7], dtype=torch.int32)        # every row counts as behind the last
    plan = fb.MoePlan(*(t.to(cuda_device) for t in (row_of, src, offsets)))
    y = torch.randn((T * k, D), device=cuda_device)
    w = torch.rand((T, k), device=cuda_device)
    ref, mag = orc.combine_ref(y, w, torch.where((row_of < 0) | (row_of >= T * k), -1, row_of))
    close(fb.moe_combine(y, w, plan), ref, k * U32 * mag + rounding(torch.float32, ref))
    fb.moe_gather(y[:T], plan), fb.moe_combine_backward(y[:T], y, w, plan), fb.moe_gather_quant(
        torch.randn((T, 128), device=cuda_device), plan)
    torch.cuda.synchronize()


def test_refusals(cuda_device):
    plan = gpu_plan(4, 2, 3, 0, cuda_device)
    x = torch.zeros((4, 128), device=cuda_device)
    w = torch.ones((4, 2), device=cuda_device)
    y = torch.zeros((8, 128), device=cuda_device)
    for f in (lambda: fb.moe_sort(torch.zeros((4, 65), dtype=torch.int32, device=cuda_device), 3),
              lambda: fb.moe_sort(plan.row_of, 0), lambda: fb.moe_sort(plan.row_of, 1025),
              lambda: fb.moe_sort(plan.row_of.float(), 3), lambda: fb.moe_sort(plan.src, 3),
              lambda: fb.moe_gather(x[:3], plan), lambda: fb.moe_gather(x.double(), plan),
              lambda: fb.moe_gather(x.t(), plan), lambda: fb.moe_gather(x[:, :0], plan),
              lambda: fb.moe_gather(x, plan._replace(src=plan.src.cpu())),
              lambda: fb.moe_combine(y[:7], w, plan), lambda: fb.moe_combine(y, w.half(), plan),
              lambda: fb.moe_combine(y, w[:, :1], plan), lambda: fb.moe_combine(y, None, plan),
              lambda: fb.moe_combine_backward(x, y.half(), w, plan), lambda: fb.moe_combine_backward(x, None, w, plan),
              lambda: fb.moe_gather_quant(x[:, :100], plan), lambda: fb.moe_gather_quant(x.half(), plan),
              lambda: fb.moe_gather_quant(x.clone().requires_grad_(), plan),
              lambda: fb.moe_gather_quant(torch.zeros((4, 260), device=cuda_device)[:, 1:129], plan)):
        with pytest.raises(ValueError):
            f()


def layer(x, ids, w):
    plan = fb.moe_sort(ids, 16)
    y = fb.moe_gather(x, plan)
    out = fb.moe_combine(y, w, plan)
    dy, dw = fb.moe_combine_backward(out, y, w, plan)
    return plan, y, out, dw, fb.moe_gather_backward(dy, plan)


def test_two_captured_graphs_and_another_stream(cuda_device):
    """Sort to gradients captured twice (several sort blocks, so each has a
    workspace), replayed in turn with new inputs, beside an eager run on another stream."""
    T, k, D = 4000, 4, 72
    g = torch.Generator(device=cuda_device).manual_seed(8)
    sets = [(torch.randn((T, D), generator=g, device=cuda_device),
             torch.randint(-2, 18, (T, k), generator=g, device=cuda_device),
             torch.rand((T, k), generator=g, device=cuda_device)) for _ in range(3)]
    flat = lambda r: [*r[0], *r[1:]]  # noqa: E731
    ref = [[t.clone() for t in flat(layer(*s))] for s in sets]
    torch.cuda.synchronize()
    graphs = []
    for s in sets[:2]:
        static = [t.clone() for t in s]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(*static)
        graphs.append((graph, static, out))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for turn in range(3):
        for i, (graph, static, out) in enumerate(graphs):
            which = (i + turn) % 3
            for a, b in zip(static, sets[which]):
                a.copy_(b)
            graph.replay()
            with torch.cuda.stream(side):
                eager = layer(*sets[2])
            torch.cuda.synchronize()
            for a, b in zip(flat(out), ref[which]):
                assert torch.equal(a, b)
            for a, b in zip(flat(eager), ref[2]):
                assert torch.equal(a, b)


def test_gradients_inside_a_capture(cuda_device):
    """A captured pass may differentiate what it computes; a leaf is refused (before
    anything is recorded), the backward functions are the way for one."""
    T, k, E, D = 50, 3, 8, 96
    plan = gpu_plan(T, k, E, 2, cuda_device)
    x, w, dout = torch.randn((T, D), device=cuda_device), torch.rand((T, k), device=cuda_device), torch.randn((T, D), device=cuda_device)

    def step(a, b):
        y = fb.moe_gather(a * 2, plan)
        out = fb.moe_combine(y, b * 0.5, plan)
        return [out, *torch.autograd.grad(out, (a, b), dout)]

    ref = step(x.clone().requires_grad_(), w.clone().requires_grad_())
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(a, b)
    graph.replay()
    torch.cuda.synchronize()
    for g, r in zip(got, ref):
        assert torch.equal(g, r)
    y = fb.moe_gather(x, plan)
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        for f in (lambda: fb.moe_gather(a, plan), lambda: fb.moe_combine(y, b, plan),
                  lambda: fb.moe_combine(y.detach().requires_grad_(), w, plan)):
            with pytest.raises(ValueError):
                f()
        dx = fb.moe_gather_backward(y, plan)
    other.replay()
    torch.cuda.synchronize()
    assert torch.equal(dx, fb.moe_gather_backward(y, plan))


def test_rows_beyond_32_bit_offsets(cuda_device):
    """Sorted rows past 2^31 elements: the last rows land where they belong."""
    T, k, D = 40000, 8, 7168                       # 2.3e9 elements of y
    x = torch.randint(-99, 99, (T, D), device=cuda_device, dtype=torch.int8).to(torch.bfloat16)
    plan = fb.moe_sort(torch.arange(k, device=cuda_device).expand(T, k), k)     # expert j owns rows j*T ..
    y = fb.moe_gather(x, plan)
    assert torch.equal(y[-T:], x) and torch.equal(y[:T], x)
    out = fb.moe_combine(y, torch.full((T, k), 0.125, device=cuda_device), plan)
    assert torch.equal(out, x)                     # eight exact eighths
    dy, dw = fb.moe_combine_backward(x[:, :].contiguous(), y, torch.ones((T, k), device=cuda_device), plan)
    assert torch.equal(dy, y) and torch.equal(dw[:, 0], dw[:, 7])


def test_sort_quantise_gemm_combine(cuda_device):
    """The operators in the order a routed layer uses them, with the FP8 GEMM as
    the experts' product, against the same chain of the CPU oracles."""
    from fack_b200 import data
    from oracle.blockscale import exact_gemm_f64
    T, k, E, N, K = 37, 2, 5, 256, 512
    g = torch.Generator().manual_seed(1)
    x = torch.randn((T, K), generator=g)
    ids = make_ids(T, k, E, 6, "topk")
    w = torch.rand((T, k), generator=g)
    weights = [data.make_weights(N, K, "normal", seed=e) for e in range(E)]
    plan = fb.moe_sort(ids.to(cuda_device), E)
    xq, xs = fb.moe_gather_quant(x.to(cuda_device), plan)
    y = torch.zeros((T * k, N), dtype=torch.bfloat16, device=cuda_device)
    bounds = plan.offsets.tolist()
    for e, (wq, ws) in enumerate(weights):
        a, b = bounds[e], bounds[e + 1]
        if b > a:
            fb.gemm_blockscale(xq[a:b], wq.to(cuda_device), xs[a:b], ws.to(cuda_device), out=y[a:b])
    out = fb.moe_combine(y, w.to(cuda_device), plan)
    row_of, src, offsets = orc.sort_ref(ids, E)
    rq, rs = orc.gather_quant_ref(x, src, k)
    ry = torch.cat([exact_gemm_f64(rq[a:b], *(weights[e][:1]), rs[a:b], weights[e][1])
                    for e, (a, b) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:]))])
    ref, mag = orc.combine_ref(ry, w, row_of)
    # the GEMM's own tolerance (rtol = atol = 1e-2 before the combine), weights below 1, two rows a token
    close(out, ref, 1e-2 * mag + 1e-2 * k + rounding(torch.bfloat16, ref))


def test_gradients_of_gradients_are_refused(cuda_device):
    """create_graph gives the first gradients as usual; a second derivative through
    them is an error, not a silent zero."""
    ids = torch.tensor([[0, 1], [1, 2]], device=cuda_device)
    plan = fb.moe_sort(ids, 3)
    x = torch.randn((2, 8), device=cuda_device, requires_grad=True)
    y = torch.randn((4, 8), device=cuda_device, requires_grad=True)
    gates = torch.rand((2, 2), device=cuda_device, requires_grad=True)
    for out, leaf in ((fb.moe_gather(x, plan), x), (fb.moe_combine(y, gates, plan), gates)):
        g = torch.randn_like(out, requires_grad=True)
        first, = torch.autograd.grad(out, leaf, g, create_graph=True)
        with pytest.raises(RuntimeError):
            first.sum().backward()


FRESH_SORT = """
import torch
import fack_b200 as fb
from oracle.moe import sort_ref
E, T, k = {E}, {T}, {k}
ids = torch.randint(-1, E + 1, (T, k), generator=torch.Generator().manual_seed(E))
for got, ref in zip(fb.moe_sort(ids.cuda(), E), sort_ref(ids, E)):
    assert torch.equal(got.cpu(), ref)
print("sorted")
"""


@pytest.mark.parametrize("E,T,k", [(844, 432, 8), (845, 1, 1), (846, 432, 8), (720, 2945, 1), (721, 3000, 2), (1024, 512, 8)])
def test_sort_as_the_first_call_of_a_process(cuda_device, E, T, k):
    """Shared memory just below and above what a kernel has without asking for more."""
    import subprocess
    import sys
    from pathlib import Path
    run = subprocess.run([sys.executable, "-c", FRESH_SORT.format(E=E, T=T, k=k)],
                         cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "sorted" in run.stdout, run.stdout + run.stderr


def test_sorts_of_several_expert_counts_from_several_threads(cuda_device):
    import threading
    cases = []
    for E in (725, 1024, 880, 64):
        ids = torch.randint(-1, E + 1, (1500, 3), generator=torch.Generator().manual_seed(E))
        cases.append((ids.to(cuda_device), E, orc.sort_ref(ids, E)))
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(300):
                ids, E, ref = cases[(first + i) % len(cases)]
                try:
                    plan = fb.moe_sort(ids, E)
                    if i % 10 == 0 and not all(torch.equal(a.cpu(), b) for a, b in zip(plan, ref)):
                        wrong.append((first, i))
                except RuntimeError as e:
                    wrong.append((first, i, str(e)))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong, wrong[:3]


def test_forward_mode_is_refused(cuda_device):
    """A dual tensor does not require grad: without a check its tangent would be dropped."""
    import torch.autograd.forward_ad as fwd
    plan = fb.moe_sort(torch.tensor([[0, 1], [1, 2], [0, 2]], device=cuda_device), 3)
    x, y = torch.randn((3, 128), device=cuda_device), torch.randn((6, 128), device=cuda_device)
    w = torch.rand((3, 2), device=cuda_device)
    codes = torch.randint(0, 256, (32, 64), device=cuda_device, dtype=torch.uint8)
    s = torch.ones((1, 32), device=cuda_device)
    xb = x.bfloat16()
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for f in (lambda: fb.moe_gather(dual(x), plan), lambda: fb.moe_combine(dual(y), w, plan),
                  lambda: fb.moe_combine(y, dual(w), plan), lambda: fb.moe_gather_quant(dual(x), plan),
                  lambda: fb.moe_gather_backward(dual(y), plan), lambda: fb.moe_combine_backward(dual(x), y, w, plan),
                  lambda: fb.moe_combine_backward(x, dual(y), w, plan), lambda: fb.moe_combine_backward(x, y, dual(w), plan),
                  lambda: fb.moe_gather(dual(x).requires_grad_(), plan),
                  lambda: fb.gemv_w4(dual(xb), codes, s), lambda: fb.gemv_w4(xb, codes, dual(s)),
                  lambda: fb.gemv_w4(xb, codes, s, out=dual(torch.zeros((3, 32), device=cuda_device).bfloat16()))):
            with pytest.raises(ValueError, match="forward"):
                f()
        assert torch.equal(fb.moe_gather(x, plan), x[plan.src.long() // 2])


def test_quant_fp32_rows_of_any_16_byte_stride(cuda_device):
    """The kernel reads 16 bytes at a time: strides of 4, 8 and 12 elements modulo 16."""
    plan = fb.moe_sort(torch.tensor([[0, 1], [1, 2], [0, 2]], device=cuda_device), 3)
    wide = torch.randn((3, 272), device=cuda_device)
    for off, ld in ((0, 260), (4, 264), (8, 268), (0, 272)):
        x = wide.as_strided((3, 256), (ld, 1), off)
        for a, b in zip(fb.moe_gather_quant(x, plan), fb.moe_gather_quant(x.contiguous(), plan)):
            assert torch.equal(a.float(), b.float())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gather_quant_beside_the_quantiser_on_what_is_not_finite(cuda_device, dtype):
    """Equal where a group is finite with a scale above 0 or all zero; what the two do with the rest."""
    T, K, inf, nan = 10, 384, float("inf"), float("nan")
    plan = fb.moe_sort(torch.zeros((T, 1), dtype=torch.int32, device=cuda_device), 1)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(1))
    for t, k, v in ((0, 3, nan), (1, 130, inf), (2, 131, -inf), (3, 5, inf), (3, 6, nan), (4, 0, inf), (4, 127, -inf),
                    (5, 383, nan)):
        x[t, k] = v
    x[6, 128:256] = 0
    x[7, :128] = 1e-40                                  # both types hold about this; the scale is about 4e-43
    x[8, :128] = 2.0 ** -149 if dtype == torch.float32 else 1.0
    x = x.to(dtype)
    group = x.float().view(T, -1, 128)
    xq, xs = (t.float().cpu() for t in fb.moe_gather_quant(x.to(cuda_device), plan))
    q, s = (t.float().cpu() for t in fb.quantize_activations(x.to(cuda_device), layout="logical"))
    xq, q = xq.view_as(group), q.view_as(group)
    has_nan, has_inf = group.isnan().any(2), group.isinf().any(2)
    tiny = (group.abs().amax(2) > 0) & (group.abs().amax(2) / 240.0 == 0)
    same = ~(has_nan | has_inf | tiny)
    assert torch.equal(xs[same], s[same]) and torch.equal(xq[same], q[same])
    assert xs[has_nan].isnan().all() and xq[has_nan].isnan().all() and not s[has_nan].isnan().any()
    only = has_inf & ~has_nan
    assert xs[only].isinf().all() and s[only].isinf().all()
    assert torch.equal(xq[only].isnan(), group[only].isinf()) and (xq[only].nan_to_num(0.0) == 0).all()
    assert torch.equal(q[only], torch.where(group[only].isinf(), -240.0, 0.0))
    assert (xs[tiny] == 1).all() and (xq[tiny] == 0).all() and (s[tiny] == 0).all() and (q[tiny] == 240).all()
    assert int(tiny.sum()) == (1 if dtype == torch.float32 else 0)


def test_gather_quant_codes_on_midpoints(cuda_device):
    """bf16 values that lie between two codes exactly, with scales that are no powers of two: the
    definition divides by 240 and by the scale, and a product with a rounded reciprocal would
    take some of them the other way."""
    g = torch.Generator().manual_seed(3)
    T, K = 64, 7168
    x = torch.randn((T, K), generator=g)
    x = torch.where(torch.rand((T, K), generator=g) < 1e-3, x * 50, x).bfloat16()
    group = x.float().view(T, -1, 128)
    scale = group.abs().amax(2, keepdim=True) / 240.0
    other = group.abs().amax(2, keepdim=True) * torch.tensor(1.0 / 240.0)
    by = lambda s: (group / s).clamp(-240, 240).to(torch.float8_e4m3fn).float()  # noqa: E731
    assert (by(scale) != by(other)).sum() > 500               # such values are among them
    plan = fb.moe_sort(torch.arange(T, device=cuda_device)[:, None] % 5, 5)
    xq, xs = fb.moe_gather_quant(x.to(cuda_device), plan)
    rows = plan.src.cpu().long()
    assert torch.equal(xs.cpu(), scale[rows, :, 0]) and torch.equal(xq.float().cpu(), by(scale).view(T, K)[rows])


def test_a_graphed_callable(cuda_device):
    """torch.cuda.make_graphed_callables: its static inputs are leaves, taken through a view;
    outputs and gradients equal those of the eager layer, for new inputs too."""
    T, k, E, D = 70, 3, 8, 96
    plan = gpu_plan(T, k, E, 6, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(7)
    rand = lambda *s: torch.randn(s, generator=g, device=cuda_device)  # noqa: E731

    def layer(x, w):
        y = fb.moe_gather(x.view_as(x), plan)
        return fb.moe_combine(y * 3, w.view_as(w), plan)

    x, w = rand(T, D).requires_grad_(), rand(T, k).requires_grad_()
    graphed = torch.cuda.make_graphed_callables(layer, (x, w))
    for _ in range(3):
        a, b, dout = rand(T, D), rand(T, k), rand(T, D)
        got, ref = [], []
        for f, out in ((graphed, got), (layer, ref)):
            xa, wb = a.clone().requires_grad_(), b.clone().requires_grad_()
            y = f(xa, wb)
            out += [y.detach().clone(), *(t.clone() for t in torch.autograd.grad(y, (xa, wb), dout))]
        for p, q in zip(got, ref):
            assert torch.equal(p, q)


# rows wide enough for two places a thread, tokens enough for a block each: the second place whole, partly
# filled and (fp32) with several rounds; one and two, three and four slots, and five, which take one place
TWO_PLACES = [(300, 1, 7, 1024), (300, 2, 9, 1032), (301, 2, 9, 7168), (297, 2, 5, 4104), (301, 3, 6, 2056),
              (333, 4, 8, 4104), (299, 4, 12, 1024), (298, 5, 9, 2056)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,E,D", TWO_PLACES)
def test_two_places_of_a_row_at_once(cuda_device, dtype, T, k, E, D):
    plan = gpu_plan(T, k, E, D + T, cuda_device)
    g = torch.Generator().manual_seed(T + D)
    y, dout = torch.randn((T * k, D), generator=g).to(dtype), torch.randn((T, D), generator=g).to(dtype)
    w = torch.randn((T, k), generator=g)
    y[int(plan.offsets[-1]):] = float("nan")
    yd, dd, wd = y.to(cuda_device), dout.to(cuda_device), w.to(cuda_device)
    ref, mag = orc.combine_ref(y, w, plan.row_of)
    close(fb.moe_combine(yd, wd, plan), ref, k * U32 * mag + rounding(dtype, ref))
    ref, mag = orc.combine_ref(y, None, plan.row_of)
    close(fb.moe_gather_backward(yd, plan), ref, k * U32 * mag + rounding(dtype, ref))
    rdy, rdw, mag = orc.combine_bwd_ref(dout, y, w, plan.row_of)
    dy, dw = fb.moe_combine_backward(dd, yd, wd, plan)
    close(dy, rdy, U32 * rdy.abs() + rounding(dtype, rdy))
    close(dw, rdw, D * U32 * mag)
    assert torch.equal(fb.moe_combine_backward(dd, None, wd, plan, need_dweights=False)[0], dy)
    assert torch.equal(fb.moe_combine_backward(dd, yd, wd, plan, need_dy=False)[1], dw)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_a_plan_with_entries_out_of_range(cuda_device, dtype):
    """No row lies behind the last one, so nothing but the valid entries writes."""
    T, k, D = 6, 2, 128
    row_of = torch.tensor([[0, 1], [2 ** 31 - 1, 3], [-5, 12], [-2 ** 31, 5], [99, 7], [8, 9]], dtype=torch.int32)
    valid = (row_of >= 0) & (row_of < T * k)
    plan = fb.MoePlan(*(t.to(cuda_device) for t in (row_of, torch.zeros(T * k, dtype=torch.int32),
                                                    torch.tensor([0, T * k], dtype=torch.int32))))
    g = torch.Generator().manual_seed(1)
    x, y = torch.randn((T, D), generator=g).to(dtype), torch.randn((T * k, D), generator=g).to(dtype)
    w = torch.rand((T, k), generator=g)
    got = fb.moe_gather(x.to(cuda_device), plan).cpu()
    dy, dw = (t.cpu() for t in fb.moe_combine_backward(*(t.to(cuda_device) for t in (x, y, w)), plan))
    quant = None if dtype == torch.float16 else [t.cpu() for t in fb.moe_gather_quant(x.to(cuda_device), plan)]
    whole = None if dtype == torch.float16 else [t.cpu() for t in fb.quantize_activations(x.to(cuda_device), layout="logical")]
    _, rdw, mag = orc.combine_bwd_ref(x, y, w, torch.where(valid, row_of, -1))
    close(dw, rdw, D * U32 * mag)
    assert (dw[~valid] == 0).all()
    for t, j in valid.nonzero().tolist():
        r = int(row_of[t, j])
        want = w[t, j].double() * x[t].double()
        assert torch.equal(got[r], x[t])
        close(dy[r], want, U32 * want.abs() + rounding(dtype, want))
        if quant:
            assert torch.equal(quant[0][r].view(torch.uint8), whole[0][t].view(torch.uint8)) and torch.equal(quant[1][r], whole[1][t])
