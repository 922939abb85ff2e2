"""GPU numerics of a stack's FFN over ragged rows, output by output, and of the product that
multiplies by gelu's slope as it leaves (dx of the second product, of ragged_ffn alone). Bounds
by element, from the arithmetic: an fp32 sum of n products by at most n * 2^-23 of the sum of
their sizes (the matrix instructions may truncate), a rounding to bf16 by 2^-8 of the value."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from learning_at_home_amd.ops import _C
    from learning_at_home_amd.ops import functional as Fops
    from learning_at_home_amd.parallel import ExpertStack, FusedExpertSGD

DEV = "cuda:0"
BF = 2.0 ** -8


def offsets_of(counts):
    return F.pad(torch.tensor(counts, device=DEV).cumsum(0), (1, 0)).int()


def within(name, got, want, tol):
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    over = (got.double() - want).abs() - 1.02 * tol - 1e-30
    assert not (over > 0).any(), f"{name}: {over.max().item():.3g} over its bound"


# many rows and tiles; few of both; few, and a contraction long enough for parts
@pytest.mark.parametrize("counts,K", [([20000, 1, 129, 0, 128, 257, 15000], 72), ([70, 0, 130, 1], 136),
                                      ([70, 0, 130, 1], 1032)], ids=["large", "small", "parts"])
@pytest.mark.parametrize("N", [8, 136, 520, 2056])
def test_products_times_slope(counts, K, N):
    """out[r] = (W[e]^T d[r]) * slope[r], for ragged columns too; zeros for rows of nobody."""
    E, end, R = len(counts), sum(counts), sum(counts) + 37
    g = torch.Generator(device=DEV).manual_seed(K + N)
    d = torch.randn(R, K, device=DEV, generator=g).bfloat16()
    w = (torch.randn(E, K, N, device=DEV, generator=g) * K ** -0.5).bfloat16()
    slope = (torch.rand(R, N, device=DEV, generator=g) * 1.26 - 0.13).half()
    slope[::5, ::3] = 2.0 ** -20  # below fp16's normal range
    slope[1::7] = 0.0
    d[end:] = float("nan")
    offsets = offsets_of(counts)
    out = _C.ragged_nn(d, w, offsets, slope)
    plain = _C.ragged_nn(d, w, offsets)
    assert not out[end:].any() and not plain[end:].any()
    at = offsets.tolist()
    for e in range(E):
        s = slice(at[e], at[e + 1])
        dd, wd, sd = d[s].double(), w[e].double(), slope[s].double()
        sums, size = dd @ wd, K * 2.0 ** -23 * (dd.abs() @ wd.abs())
        within("plain", plain[s], sums, BF * sums.abs() + size)
        # the product with the slope in fp32: 2^-24 of it
        within("slope", out[s], sums * sd, (BF + 2.0 ** -24) * (sums * sd).abs() + size * sd.abs())
    assert torch.equal(out, _C.ragged_nn(d, w, offsets, slope))


@pytest.mark.parametrize("d,ffn", [(64, 192), (128, 320), (320, 64)])
@pytest.mark.parametrize("counts", [[5, 0, 130, 64], [0, 1, 0, 0], [0, 0, 0, 0], [3000, 0, 9000, 1], [20000, 18000, 0, 300]],
                         ids=str)
def test_ffn_by_element(counts, d, ffn):
    torch.manual_seed(0)
    stack = ExpertStack(4, d, ffn).to(DEV)
    stack.init_gpu_state()
    offsets, end = offsets_of(counts), sum(counts)
    x = torch.randn(end + 9, d, device=DEV).bfloat16()
    dy = torch.randn(end + 9, d, device=DEV).bfloat16()
    x[end:], dy[end:] = float("nan"), float("inf")
    for g in (stack.main_grad_W1, stack.main_grad_W2, stack.main_grad_b1, stack.main_grad_b2):
        g.fill_(1e9)  # a first backward writes
    x.requires_grad_(True)
    y = Fops.ragged_ffn(x, offsets, stack)
    y.backward(dy)
    assert not y[end:].any() and not x.grad[end:].any()
    at, xs = offsets.tolist(), x.detach().double()
    for e, n in enumerate(counts):
        s = slice(at[e], at[e + 1])
        xe, de = xs[s], dy[s].double()
        W1, b1, W2, b2 = (t[e].detach().double() for t in (stack.W1c, stack.b1_f32, stack.W2c, stack.b2_f32))
        u = (xe @ W1.t() + b1).requires_grad_(True)
        h = F.gelu(u, approximate="tanh")
        slope, = torch.autograd.grad(h.sum(), u)
        u, h = u.detach(), h.detach()
        # the sum before gelu; gelu's slope is at most 1.13, its own at most 1; exp2 and reciprocal 2^-20
        off = (d + 2) * 2.0 ** -23 * (xe.abs() @ W1.abs().t() + b1.abs())
        h_off = BF * h.abs() + 1.13 * off + 2.0 ** -20 * u.abs()
        out = h @ W2.t() + b2
        within("y", y[s].detach(), out, BF * out.abs() + h_off @ W2.abs().t()
               + (ffn + 2) * 2.0 ** -23 * (h.abs() @ W2.abs().t() + b2.abs()))
        back = de @ W2
        dh = back * slope
        # the slope in fp16 (2^-11 of it, or 2^-25), the product's sum, then one rounding to bf16
        dh_off = (BF + 2.0 ** -11) * dh.abs() + back.abs() * (off + 2.0 ** -20 + 2.0 ** -25) \
            + d * 2.0 ** -23 * (de.abs() @ W2.abs()) * slope.abs()
        dx = dh @ W1
        within("dx", x.grad[s], dx, BF * dx.abs() + dh_off @ W1.abs() + ffn * 2.0 ** -23 * (dh.abs() @ W1.abs()))
        for name, got, want, tol in (
                ("W1", stack.main_grad_W1, dh.t() @ xe, dh_off.t() @ xe.abs() + n * 2.0 ** -23 * (dh.abs().t() @ xe.abs())),
                ("b1", stack.main_grad_b1, dh.sum(0), dh_off.sum(0) + n * 2.0 ** -23 * dh.abs().sum(0)),
                ("W2", stack.main_grad_W2, de.t() @ h, de.abs().t() @ h_off + n * 2.0 ** -23 * (de.abs().t() @ h.abs())),
                ("b2", stack.main_grad_b2, de.sum(0), n * 2.0 ** -23 * de.abs().sum(0))):
            within(name, got[e], want, tol)


def test_scale_is_held_for_the_side_stream():
    """The step on the side stream still waits to read the scale: its memory may not be given away."""
    torch.manual_seed(0)
    stack = ExpertStack(2, 128, 128).to(DEV)
    stack.init_gpu_state()
    opt, side = FusedExpertSGD(stack, lr=0.5), torch.cuda.Stream()
    opt.set_side_stream(side)
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda._sleep(1000)
    start.record()
    torch.cuda._sleep(1_000_000)
    stop.record()
    stop.synchronize()
    cycles = int(200 / max(start.elapsed_time(stop), 1e-3) * 1_000_000)  # a fifth of a second
    stack.main_grad_W1.fill_(1.0)
    stack.grad_ready = True
    before = stack.W1.detach().clone()
    norm, scale = Fops.grad_clip_scale(opt.gradients(), 1.0)
    want, at = before - 0.5 * scale, scale.data_ptr()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(cycles)
    opt.step(grad_scale=scale)
    free = torch.zeros((), device=DEV)  # what no other stream holds is given away at once
    free_at = free.data_ptr()
    del scale, free
    others = [torch.empty((), device=DEV) for _ in range(5000)]  # a small segment and more
    assert not side.query(), "the step was over before the memory was asked for"
    taken = {t.data_ptr() for t in others}
    assert at not in taken and free_at in taken
    for t in others[:64]:
        t.fill_(1e9)
    torch.cuda.synchronize()
    assert torch.isfinite(norm) and torch.allclose(stack.W1, want, rtol=1e-6, atol=1e-7)
