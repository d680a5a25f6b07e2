"""GPU: products with 4-bit weights against the 64-bit oracle.

Tolerances, from the arithmetic.  A product x * (code - zero) is exact.  The
tensor core adds 16 of them and its accumulator at a time, each of the 17 terms
good to 2^-23 of the largest; a group of G' = min(G, 128) takes G'/16 such steps.
The scaled groups are then added in fp32 (K/1024 of them a warp, 8 warps, one
product and one addition each).  So an output is off by at most
(17 G'/16 + K/512 + 18) * 2^-23 of the sum of its terms' magnitudes, and half a
unit of its type.  With one-figure whole numbers and powers of two nothing rounds
at all and the outputs are equal."""
import pytest
import torch

import fack_b200 as fb
from oracle import moe as moe_orc
from oracle import w4 as orc

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def tolerance(ref, mag, K, G, dtype):
    info = torch.finfo(dtype)
    return (17 * min(G, 128) / 16 + K / 512 + 18) * 2.0 ** -23 * mag + ref.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def close(got, ref, tol):
    assert torch.isfinite(got.float()).all()
    off = (got.cpu().double() - ref).abs()
    assert bool((off <= tol).all()), f"off by {float(off.max()):.3g}, {float((off - tol).max()):.3g} over"


def weight(lead, N, K, G, zeros, sdtype, seed, exact=False):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 256, (*lead, N, K // 2), generator=g, dtype=torch.uint8)
    if exact:
        s = torch.exp2(torch.randint(-1, 1, (*lead, K // G, N), generator=g).float())
    else:
        s = (torch.rand((*lead, K // G, N), generator=g) + 0.5) * 0.02
    z = torch.randint(0, 16, (*lead, K // G, N), generator=g, dtype=torch.uint8) if zeros else None
    return w, s.to(sdtype), z


def to(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


def few_ones(M, K, seed, dtype):
    """Rows with four entries of +-1: outputs below 4 * 15, whole or half, exact in every type."""
    g = torch.Generator().manual_seed(seed)
    x = torch.zeros((M, K))
    for m in range(M):
        at = torch.randperm(K, generator=g)[:4]
        x[m, at] = torch.randint(0, 2, (len(at),), generator=g).float() * 2 - 1
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128, 384])
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 13, 16, 17, 33, 70])
def test_exact(cuda_device, dtype, zeros, G, M):
    for N, steps in ((16, 1), (48, 3), (144, 5), (4624, 9), (32, 40)):
        K = G * steps
        sdtype = torch.float32 if steps % 2 else dtype
        w, s, z = weight((), N, K, G, zeros, sdtype, M + N, exact=True)
        x = few_ones(M, K, M + K, dtype)
        y = fb.gemv_w4(*to(cuda_device, x, w, s, z))
        assert y.dtype == dtype and torch.equal(y.cpu().double(), orc.product_ref(x, w, s, z)[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,G,zeros", [(1, 7168, 2048, 128, False), (3, 2048, 7168, 64, True), (16, 1040, 4096, 32, True),
                                           (24, 528, 1056, 32, False), (8, 64, 18432, 18432, True), (1, 16, 32, 32, True)])
def test_random(cuda_device, dtype, M, N, K, G, zeros):
    w, s, z = weight((), N, K, G, zeros, dtype, M + N + K)
    x = torch.randn((M, K), generator=torch.Generator().manual_seed(K)).to(dtype)
    y = fb.gemv_w4(*to(cuda_device, x, w, s, z))
    ref, mag = orc.product_ref(x, w, s, z)
    close(y, ref, tolerance(ref, mag, K, G, dtype))
    assert torch.equal(y, fb.gemv_w4(*to(cuda_device, x, w, s, z)))


def test_strides_out_and_broadcast_rows(cuda_device):
    w, s, z = to(cuda_device, *weight((), 80, 256, 64, True, torch.float32, 1))
    wide = torch.randn((6, 512), device=cuda_device).bfloat16()
    x = wide[:, 64:320]
    ref = fb.gemv_w4(x.contiguous(), w, s, z)
    assert torch.equal(fb.gemv_w4(x, w, s, z), ref)
    out = torch.full((7, 97), 5.0, device=cuda_device, dtype=torch.bfloat16)
    view = out[:6, 3:83]
    assert fb.gemv_w4(x, w, s, z, out=view) is view
    assert torch.equal(view, ref) and (out[6] == 5).all() and (out[:, :3] == 5).all() and (out[:, 83:] == 5).all()
    assert torch.equal(fb.gemv_w4(x[:1].expand(6, 256), w, s, z), ref[:1].expand(6, 80))
    assert fb.gemv_w4(x[:0], w, s, z).shape == (0, 80)


def test_high_bits_of_zero_points_are_not_read(cuda_device):
    w, s, z = to(cuda_device, *weight((), 32, 128, 32, True, torch.float32, 1))
    x = torch.randn((2, 128), device=cuda_device).half()
    assert torch.equal(fb.gemv_w4(x, w, s, z | 0xa0), fb.gemv_w4(x, w, s, z))


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan_stay_with_their_token_and_row(cuda_device, dtype):
    w, s, z = weight((), 48, 256, 64, True, torch.float32, 3)
    x = torch.randn((11, 256)).to(dtype)
    clean = fb.gemv_w4(*to(cuda_device, x, w, s, z))
    x[2, 17], x[9, 255] = float("nan"), float("inf")
    s[1, 5] = float("nan")
    y = fb.gemv_w4(*to(cuda_device, x, w, s, z))
    assert y[2].isnan().all() and not y[9].isfinite().any() and y[:, 5].isnan().all()
    keep = [m for m in range(11) if m not in (2, 9)]
    cols = [n for n in range(48) if n != 5]
    assert torch.equal(y[keep][:, cols], clean[keep][:, cols])


def test_overflow_is_infinite_and_large_values_are_summed(cuda_device):
    """fp16 outputs past the type's range are infinite; partial sums beyond it are not."""
    w = torch.full((16, 64), 0xff, dtype=torch.uint8, device=cuda_device)      # codes 15: value 7
    s = torch.ones((1, 16), device=cuda_device)
    x = torch.full((2, 128), 60000.0, device=cuda_device, dtype=torch.float16)
    x[1, 64:] = -60000.0
    y = fb.gemv_w4(x, w, s)
    assert y[0].isinf().all() and (y[1] == 0).all()


def make_ids(T, k, E, seed, kind):
    g = torch.Generator().manual_seed(seed)
    if kind == "topk":
        return torch.stack([torch.randperm(max(E, k), generator=g)[:k] for _ in range(T)])
    if kind == "one":
        return torch.full((T, k), E - 1)
    if kind == "none":
        return torch.full((T, k), -1)
    return torch.randint(-2, E + 2, (T, k), generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["topk", "one", "none", "any"])
@pytest.mark.parametrize("T,k,E,N,K,G", [(1, 1, 1, 16, 32, 32), (1, 8, 40, 48, 320, 64), (9, 3, 4, 208, 256, 128),
                                         (40, 4, 7, 64, 1152, 384), (100, 2, 300, 16, 96, 32), (77, 5, 6, 32, 128, 128)])
def test_experts(cuda_device, dtype, kind, T, k, E, N, K, G):
    ids = make_ids(T, k, E, T + E, kind)
    plan = fb.moe_sort(ids.to(cuda_device), E)
    row_of, src, offsets = moe_orc.sort_ref(ids, E)
    zeros = T % 2 == 1
    w, s, z = weight((E,), N, K, G, zeros, torch.float32 if k % 2 else dtype, T + K, exact=True)
    x = few_ones(T, K, T, dtype)
    xs = moe_orc.gather_ref(x, src, k)
    ref = orc.experts_ref(xs, w, s, z, offsets, T * k)[0]
    wd, sd, zd = to(cuda_device, w, s, z)
    y = fb.gemv_w4_experts(x.to(cuda_device), wd, sd, plan, zd)
    assert torch.equal(y.cpu().double(), ref)
    xs[int(offsets[-1]):] = float("nan")                      # rows of nobody are not read
    out = torch.full((T * k, N), float("nan"), dtype=dtype, device=cuda_device)
    y = fb.gemv_w4_experts(xs.to(cuda_device), wd, sd, plan, zd, sorted_rows=True, out=out)
    assert y is out and torch.equal(y.cpu().double(), ref)


def test_experts_random(cuda_device):
    T, k, E, N, K, G = 30, 4, 10, 336, 2048, 128
    ids = make_ids(T, k, E, 1, "topk")
    plan = fb.moe_sort(ids.to(cuda_device), E)
    src, offsets = plan.src.cpu(), plan.offsets.cpu()
    for dtype in TYPES:
        w, s, z = weight((E,), N, K, G, True, dtype, 5)
        x = torch.randn((T, K), generator=torch.Generator().manual_seed(2)).to(dtype)
        y = fb.gemv_w4_experts(x.to(cuda_device), *to(cuda_device, w, s), plan, z.to(cuda_device))
        ref, mag = orc.experts_ref(moe_orc.gather_ref(x, src, k), w, s, z, offsets, T * k)
        close(y, ref, tolerance(ref, mag, K, G, dtype))


def test_experts_beyond_32_bit_offsets(cuda_device):
    """A stack of experts past 2^31 codes and bytes: the last expert's weights."""
    E, N, K, G = 24, 16384, 16384, 128                        # 3.2e9 bytes
    w = torch.zeros((E, N, K // 2), dtype=torch.uint8, device=cuda_device)
    s = torch.ones((E, K // G, N), dtype=torch.bfloat16, device=cuda_device)
    last, ls, _ = weight((), N, K, G, False, torch.bfloat16, 4, exact=True)
    w[-1], s[-1] = last.to(cuda_device), ls.to(cuda_device)
    x = few_ones(2, K, 1, torch.bfloat16).to(cuda_device)
    plan = fb.moe_sort(torch.tensor([[E - 1], [3]], device=cuda_device), E)
    y = fb.gemv_w4_experts(x, w, s, plan)
    assert torch.equal(y[1], fb.gemv_w4(x[:1], last.to(cuda_device), ls.to(cuda_device))[0])
    assert torch.equal(y[0].float(), (x[1].float().sum() * -8).expand(N))


def test_plans_that_are_none(cuda_device):
    """Offsets that do not ascend route nothing; a src outside the pairs is a row of zeros."""
    T, k, E, N, K = 3, 2, 3, 32, 64
    w, s, _ = to(cuda_device, *weight((E,), N, K, 64, False, torch.float32, 1))
    x = torch.ones((T, K), device=cuda_device, dtype=torch.bfloat16)
    row_of = torch.zeros((T, k), dtype=torch.int32, device=cuda_device)
    src = torch.tensor([0, -1, 2 ** 31 - 1, -2 ** 31, 6, 5], dtype=torch.int32, device=cuda_device)
    for bad in ([0, 4, 2, 6], [-1, 2, 4, 6], [0, 2, 4, 7], [0, 2 ** 31 - 1, 4, 6]):
        plan = fb.MoePlan(row_of, src, torch.tensor(bad, dtype=torch.int32, device=cuda_device))
        assert (fb.gemv_w4_experts(x, w, s, plan) == 0).all()
    plan = fb.MoePlan(row_of, src, torch.tensor([0, 2, 4, 6], dtype=torch.int32, device=cuda_device))
    y = fb.gemv_w4_experts(x, w, s, plan)
    assert (y[1:5] == 0).all()
    assert torch.equal(y[0], fb.gemv_w4(x[:1], w[0], s[0])[0]) and torch.equal(y[5], fb.gemv_w4(x[:1], w[2], s[2])[0])


def test_refusals(cuda_device):
    w, s, z = to(cuda_device, *weight((), 32, 128, 64, True, torch.float32, 1))
    x = torch.zeros((2, 128), device=cuda_device, dtype=torch.bfloat16)
    plan = fb.moe_sort(torch.zeros((2, 2), dtype=torch.int32, device=cuda_device), 1)
    shifted = torch.zeros((2, 136), device=cuda_device, dtype=torch.bfloat16)[:, 1:129]
    for f in (lambda: fb.gemv_w4(x.float(), w, s), lambda: fb.gemv_w4(x, w.cpu(), s), lambda: fb.gemv_w4(x[:, :64], w, s),
              lambda: fb.gemv_w4(shifted, w, s), lambda: fb.gemv_w4(x.t(), w, s), lambda: fb.gemv_w4(x, w, s.half()),
              lambda: fb.gemv_w4(x, w, s, z.float()), lambda: fb.gemv_w4(x, w, s, out=x),
              lambda: fb.gemv_w4(x, w, s, out=torch.zeros((2, 32), device=cuda_device)),
              lambda: fb.gemv_w4(x.clone().requires_grad_(), w, s),
              lambda: fb.gemv_w4(x, w, s, out=torch.zeros((1, 32), device=cuda_device, dtype=torch.bfloat16).expand(2, 32)),
              lambda: fb.gemv_w4_experts(x, w, s, plan), lambda: fb.gemv_w4_experts(x, w[None], s[None], plan, sorted_rows=True),
              lambda: fb.gemv_w4_experts(x[:1], w[None], s[None], plan),
              lambda: fb.gemv_w4_experts(x, w[None].repeat(2, 1, 1), s[None].repeat(2, 1, 1), plan)):
        with pytest.raises(ValueError):
            f()


def routed_layer(x, ids, gates, w1, s1, w2, s2, z2, E):
    plan = fb.moe_sort(ids, E)
    h = fb.gemv_w4_experts(x, w1, s1, plan)
    a, b = h.float().chunk(2, dim=1)
    act = (a * torch.sigmoid(a) * b).to(x.dtype)
    y = fb.gemv_w4_experts(act, w2, s2, plan, z2, sorted_rows=True)
    return fb.moe_combine(y, gates, plan), act, y


def test_a_routed_layer_and_its_graph(cuda_device):
    """Sort, first product from the tokens, gated activation, second product on
    the sorted rows, combine: each step against its oracle on the step's own
    input, then captured and replayed with other inputs beside eager calls."""
    T, k, E, D, H = 21, 3, 8, 256, 192
    g = torch.Generator().manual_seed(3)
    w1, s1, _ = weight((E,), 2 * H, D, 64, False, torch.bfloat16, 1)
    w2, s2, z2 = weight((E,), D, H, 64, True, torch.float32, 2)
    sets = [[torch.randn((T, D), generator=g).bfloat16(), torch.randint(-1, E + 1, (T, k), generator=g),
             torch.rand((T, k), generator=g)] for _ in range(3)]
    dev = to(cuda_device, w1, s1, w2, s2, z2)
    runs = []
    for x, ids, gates in sets:
        out, act, y = routed_layer(*to(cuda_device, x, ids, gates), *dev, E)
        row_of, src, offsets = moe_orc.sort_ref(ids, E)
        n = int(offsets[-1])
        ref, mag = orc.experts_ref(act.cpu(), w2, s2, z2, offsets, T * k)
        close(y, ref, tolerance(ref, mag, H, 64, torch.bfloat16))
        assert (y[n:] == 0).all()
        ref, mag = moe_orc.combine_ref(y, gates, row_of)
        # k fused multiply-adds in fp32, then half a step of bf16: 8 significant bits put neighbours 2^-7 of
        # 1 apart, so half a step is up to 2^-8 of the value (eps / 2)
        close(out, ref, k * 2.0 ** -24 * mag + ref.abs() * (torch.finfo(torch.bfloat16).eps / 2) + 2.0 ** -133)
        runs.append(out.clone())
    static = to(cuda_device, *(t.clone() for t in sets[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = routed_layer(*static, *dev, E)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in (1, 2, 0):
        for a, b in zip(static, sets[i]):
            a.copy_(b)
        graph.replay()
        with torch.cuda.stream(side):
            eager = routed_layer(*to(cuda_device, *sets[2]), *dev, E)[0]
        torch.cuda.synchronize()
        assert torch.equal(out, runs[i]) and torch.equal(eager, runs[2])


FIRST_CALLS = """
import torch
import fack_b200 as fb
d = torch.device("cuda", 0)
T, k, E = 700, 4, 6                                   # several sort blocks
ids = torch.arange(T * k, device=d).reshape(T, k) % E
x = torch.randn((T, 256), device=d).bfloat16()
w = torch.randint(0, 256, (E, 64, 128), dtype=torch.uint8, device=d)
s = torch.rand((E, 4, 64), device=d)
gates = torch.rand((T, k), device=d)

def step():
    plan = fb.moe_sort(ids, E)
    xq, xs = fb.moe_gather_quant(x, plan)
    y = fb.gemv_w4_experts(x, w, s, plan)
    out = fb.moe_combine(y, gates, plan)
    dy, dw = fb.moe_combine_backward(out, y, gates, plan)
    return [*plan, xq.view(torch.uint8), xs, y, out, dy, dw, fb.moe_gather_backward(fb.moe_gather(x, plan), plan),
            fb.gemv_w4(x[:3], w[0], s[0])]

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):                         # nothing of the library has run before
    got = step()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in got]
assert all(torch.equal(a, b) for a, b in zip(got, step())) and fb.device_status() == 0
print("captured first")
"""


def test_a_process_whose_first_calls_are_captured(cuda_device):
    import subprocess
    import sys
    from pathlib import Path
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=Path(__file__).resolve().parents[1], capture_output=True,
                         text=True, timeout=300)
    assert run.returncode == 0 and "captured first" in run.stdout, run.stdout + run.stderr


def test_calls_from_two_threads(cuda_device):
    """The C entries' own state (kernel attributes, plans) under concurrent first and later calls."""
    import threading
    g = torch.Generator().manual_seed(5)
    cases = []
    for i, (M, N, K, G) in enumerate([(1, 48, 256, 64), (9, 96, 512, 128), (3, 32, 160, 32), (16, 64, 1024, 256)]):
        w, s, z = weight((), N, K, G, i % 2 == 1, torch.float32, i, exact=True)
        x = few_ones(M, K, i, torch.float16)
        cases.append((to(cuda_device, x, w, s, z), orc.product_ref(x, w, s, z)[0]))
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(60):
                args, ref = cases[(first + i) % len(cases)]
                y = fb.gemv_w4(*args)
                if not torch.equal(y.cpu().double(), ref):
                    wrong.append((first, i))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong and fb.device_status() == 0


@pytest.mark.parametrize("M", [1, 13, 40])
@pytest.mark.parametrize("N,K,G", [(16 * 37, 128 * 9, 128), (16 * 293, 128 * 2, 256), (4096 + 16, 96, 32), (16 * 600, 64, 64),
                                   (16 * 1031, 128, 128)])
def test_exact_over_the_plans(cuda_device, M, N, K, G):
    """Row counts that leave items, parts of items and the last box of an item partly filled."""
    w, s, z = weight((), N, K, G, M == 13, torch.bfloat16, N + K, exact=True)
    x = few_ones(M, K, N, torch.bfloat16)
    assert torch.equal(fb.gemv_w4(*to(cuda_device, x, w, s, z)).cpu().double(), orc.product_ref(x, w, s, z)[0])


def test_the_longest_rows(cuda_device):
    """K = 2^20, and one token more than fits a tile."""
    N, K, G = 16, 1 << 20, 4096
    w, s, _ = weight((), N, K, G, False, torch.float32, 3, exact=True)
    x = few_ones(9, K, 4, torch.bfloat16)
    assert torch.equal(fb.gemv_w4(*to(cuda_device, x, w, s)).cpu().double(), orc.product_ref(x, w, s, None)[0])


def test_a_stack_of_most_experts(cuda_device):
    """1024 experts, a few of which have rows: the first, the last and neighbours."""
    E, N, K = 1024, 32, 64
    w, s, _ = weight((E,), N, K, 32, False, torch.float32, 1, exact=True)
    ids = torch.tensor([[0, 1023], [511, 512], [1023, 1023], [7, -1], [1024, 0]])
    plan = fb.moe_sort(ids.to(cuda_device), E)
    x = few_ones(5, K, 2, torch.float16)
    row_of, src, offsets = moe_orc.sort_ref(ids, E)
    ref = orc.experts_ref(moe_orc.gather_ref(x, src, 2), w, s, None, offsets, 10)[0]
    assert torch.equal(fb.gemv_w4_experts(*to(cuda_device, x, w, s), plan).cpu().double(), ref)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,G", [(160, 32), (32, 32), (64, 64), (192, 64)])
def test_the_next_experts_scales_are_not_met(cuda_device, dtype, K, G):
    """K ends inside a block of 128: what lies behind it belongs to the next expert."""
    E, N = 3, 48
    w, s, z = weight((E,), N, K, G, True, torch.float32, K, exact=True)
    x, ids = few_ones(4, K, K, dtype), torch.tensor([[0], [2], [0], [2]])
    s[1] = float("inf")
    plan = moe_orc.sort_ref(ids, E)
    ref, _ = orc.experts_ref(x[plan[1].long()], w, s, z, plan[2], 4)
    y = fb.gemv_w4_experts(*to(cuda_device, x, w, s), fb.MoePlan(*to(cuda_device, *plan)), to(cuda_device, z)[0])
    assert torch.equal(y.cpu().double(), ref)


def test_an_out_that_requires_grad_is_refused(cuda_device):
    w, s, _ = to(cuda_device, *weight((), 32, 64, 64, False, torch.float32, 1))
    x = torch.ones((2, 64), device=cuda_device).bfloat16()
    out = torch.zeros((2, 32), device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="out"):
        fb.gemv_w4(x, w, s, out=out)
    assert (out == 0).all()
    with torch.no_grad():
        assert fb.gemv_w4(x, w, s, out=out) is out
    assert torch.equal(out.detach(), fb.gemv_w4(x, w, s))


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("sdtype,M,N,K,G", [(torch.bfloat16, 2, 26304, 128, 128), (torch.bfloat16, 6, 53200, 256, 128),
                                            (torch.float32, 1, 21568, 128, 128), (torch.float32, 5, 21568, 128, 128),
                                            (torch.float32, 20, 41104, 128, 128), (torch.float32, 19, 43104, 1024, 256)])
def test_parts_without_their_last_group(cuda_device, sdtype, M, N, K, G, zeros):
    """Row parts one group short, one slice of K, and a stage that the boxes of scales fill to its
    end: a load for the missing group past its box would leave the kernel's shared memory."""
    w, s, z = weight((), N, K, G, zeros, sdtype, N + K, exact=True)
    x = few_ones(M, K, N, torch.bfloat16)
    assert torch.equal(fb.gemv_w4(*to(cuda_device, x, w, s, z)).cpu().double(), orc.product_ref(x, w, s, z)[0])


def test_offsets_that_start_above_zero(cuda_device):
    """Such offsets leave rows to no expert: nothing is routed, and every row is written."""
    E, N, K = 3, 32, 64
    w, s, _ = to(cuda_device, *weight((E,), N, K, 64, False, torch.float32, 1))
    x = torch.ones((3, K), device=cuda_device, dtype=torch.bfloat16)
    row_of = torch.arange(6, dtype=torch.int32, device=cuda_device).reshape(3, 2)
    src = torch.arange(6, dtype=torch.int32, device=cuda_device)
    for bad in ([2, 4, 6, 6], [6, 6, 6, 6], [1, 1, 1, 1], [-1, 2, 4, 6]):
        plan = fb.MoePlan(row_of, src, torch.tensor(bad, dtype=torch.int32, device=cuda_device))
        out = torch.full((6, N), float("nan"), device=cuda_device, dtype=torch.bfloat16)
        assert (fb.gemv_w4_experts(x, w, s, plan, out=out) == 0).all()


def plan_of(tokens, N, K, G, topk=0, experts=0):
    """(tokens a tile, groups a warp, slices of K, groups an item) of a call."""
    import ctypes
    from fack_b200 import _lib
    out = [ctypes.c_int() for _ in range(4)]
    assert _lib.load().fack_gemv_w4_plan(tokens, topk, experts, N, K, G, *map(ctypes.byref, out)) == 0
    return tuple(v.value for v in out)


LARGE_K = {32: 416, 64: 448, 128: 384, 256: 512}       # three or four blocks of 128; those of 32 and 64 end inside one
# tokens and rows of layers whose warps take four groups of 16 rows: with 8 and 16 tokens a tile, items of one
# box and of two, full and with parts a group short
LARGE = [(21, 5936), (40, 3152), (40, 28336), (40, 25104), (40, 5504), (40, 3936), (40, 23536), (40, 15120)]
LARGE_EXPERTS = [(33, 4, 4, 896), (33, 2, 2, 1504), (150, 2, 2, 3472), (150, 4, 4, 1840), (150, 4, 4, 352), (150, 2, 2, 512),
                 (150, 2, 2, 2944), (150, 2, 2, 1952)]


@pytest.mark.parametrize("G", [32, 64, 128, 256])
def test_the_large_layers_take_every_form_of_four_groups_a_warp(cuda_device, G):
    def form(p):
        tile, groups, split, item = p
        return groups, tile > 8, item > 16, item < groups * 8 // split

    want = {(4, two, boxes, part) for two in (False, True) for boxes in (False, True) for part in (False, True)}
    assert {form(plan_of(M, N, LARGE_K[G], G)) for M, N in LARGE} == want
    assert {form(plan_of(T, N, LARGE_K[G], G, k, E)) for T, k, E, N in LARGE_EXPERTS} == want


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128, 256])
@pytest.mark.parametrize("M,N", LARGE)
def test_exact_with_four_groups_a_warp(cuda_device, M, N, G, zeros):
    K, dtype = LARGE_K[G], TYPES[(M + N // 16 + zeros) % 2]
    w, s, z = weight((), N, K, G, zeros, torch.float32 if N % 32 else dtype, N + G, exact=True)
    x = few_ones(M, K, N, dtype)
    assert torch.equal(fb.gemv_w4(*to(cuda_device, x, w, s, z)).cpu().double(), orc.product_ref(x, w, s, z)[0])


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128, 256])
@pytest.mark.parametrize("T,k,E,N", LARGE_EXPERTS)
def test_experts_with_four_groups_a_warp(cuda_device, T, k, E, N, G, zeros):
    K, dtype = LARGE_K[G], TYPES[(T + N // 16 + zeros) % 2]
    w, s, z = weight((E,), N, K, G, zeros, dtype if N % 32 else torch.float32, N + G, exact=True)
    ids, x = make_ids(T, k, E, N, "any"), few_ones(T, K, N, dtype)
    row_of, src, offsets = moe_orc.sort_ref(ids, E)
    ref = orc.experts_ref(moe_orc.gather_ref(x, src, k), w, s, z, offsets, T * k)[0]
    plan = fb.moe_sort(ids.to(cuda_device), E)
    xd, wd, sd, zd = to(cuda_device, x, w, s, z)
    assert torch.equal(fb.gemv_w4_experts(xd, wd, sd, plan, zd).cpu().double(), ref)
    rows = fb.moe_gather(xd, plan)
    assert torch.equal(fb.gemv_w4_experts(rows, wd, sd, plan, zd, sorted_rows=True).cpu().double(), ref)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,G", [(1, 37888, 1344, 32), (3, 33344, 1344, 64), (8, 65536, 2048, 128), (2, 57344, 1024, 256),
                                     (13, 65536, 704, 64), (11, 57344, 672, 32)])
def test_exact_in_wide_layers(cuda_device, M, N, K, G, zeros):
    w, s, z = weight((), N, K, G, zeros, torch.bfloat16, N + G, exact=True)
    x = few_ones(M, K, N, torch.bfloat16)
    tile, groups, split, item = plan_of(M, N, K, G)
    assert tile == M and groups == 4
    assert torch.equal(fb.gemv_w4(*to(cuda_device, x, w, s, z)).cpu().double(), orc.product_ref(x, w, s, z)[0])


def test_the_plan_of_nearly_all_experts(cuda_device):
    """63 of 64 experts a token: the chance that an expert has no row is below what a double holds
    from 180 tokens on; the plan is that of one token less or of all experts, not one for no rows."""
    for N, K in ((4096, 2048), (7168, 512)):
        want = plan_of(150, N, K, 128, 63, 64)
        assert want[0] == 16
        for T in (170, 171, 180, 200, 203, 204, 260):
            assert plan_of(T, N, K, 128, 63, 64)[:2] == want[:2] == plan_of(T, N, K, 128, 64, 64)[:2]
