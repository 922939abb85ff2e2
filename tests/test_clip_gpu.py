"""GPU numerics of the gradient norm, clipping and the clipped step (ops/clip.py)
against plain torch in 64 bits. The norm: squares and up to 64 sums of a thread
in fp32 (off by 2^-24 each: 2^-18 of the sum, all terms being positive), the
rest in fp64, one rounding: within 2^-18 of it. A step: fp32 operations, a
rounding of 2^-24 each."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from learning_at_home_amd.ops import functional as Fops
    from learning_at_home_amd.optim import MasterSGD
    from learning_at_home_amd.parallel import ExpertAdam, ExpertStack, FusedExpertSGD

DEV = "cuda:0"
NORM_TOL = 2.0 ** -18


def tensors(sizes, dtypes, scale=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, device=DEV, generator=g) * scale).to(dtypes[i % len(dtypes)])
            for i, n in enumerate(sizes)]


def norm64(ts):
    return torch.stack([t.double().square().sum() for t in ts]).sum().sqrt()


SIZES = {
    "one": [1],
    "small": [1, 7, 8, 9, 255, 256, 2048, 2049],
    "chunks": [16384, 16383, 16385, 100000, 3],
    "empty-among": [0, 5, 0, 70000, 0],
    "many": [i * 13 % 997 + 1 for i in range(200)],
    "large": [40_000_001],
}


@pytest.mark.parametrize("sizes", list(SIZES), ids=str)
@pytest.mark.parametrize("dtypes", [("float32",), ("bfloat16",), ("float16",), ("float32", "bfloat16", "float16")],
                         ids="-".join)
def test_norm_and_clip(sizes, dtypes):
    ts = tensors(SIZES[sizes], [getattr(torch, d) for d in dtypes])
    want = norm64(ts)
    for max_norm in (float(want) * 0.25, float(want) * 4):
        norm, scale = Fops.grad_clip_scale(ts, max_norm)
        assert norm.dtype == scale.dtype == torch.float32 and norm.dim() == scale.dim() == 0
        assert (norm.double() - want).abs() <= NORM_TOL * want
        s64 = (max_norm / (want + 1e-6)).clamp(max=1.0)
        assert (scale.double() - s64).abs() <= 2 * NORM_TOL * s64
        mine = [t.clone() for t in ts]
        assert torch.equal(Fops.clip_grad_norm_(mine, max_norm), norm)
        for a, t in zip(mine, ts):
            assert torch.equal(a, (t.float() * scale).to(t.dtype))
    again, _ = Fops.grad_clip_scale(ts, 1.0)
    assert torch.equal(again, norm)


def test_unaligned_and_strided():
    base = torch.randn(50_001, device=DEV)
    views = [base[1:40_000], base[3:3 + 16384], torch.randn(300, 200, device=DEV).t(),
             torch.randn(64, 64, device=DEV)[::2, ::2]]
    want = norm64(views)
    norm, scale = Fops.grad_clip_scale(views, 1.0)
    assert (norm.double() - want).abs() <= NORM_TOL * want
    mine = [torch.empty_strided(v.shape, v.stride(), device=DEV).copy_(v) for v in views]
    Fops.clip_grad_norm_(mine, 1.0)
    for a, v in zip(mine, views):
        assert torch.equal(a, v * scale)


def test_types_that_are_not_the_kernels():
    """fp64 gradients, fp32 parameters, one of several not contiguous."""
    ts = [torch.randn(100, device=DEV, dtype=torch.float64), torch.randn(7, device=DEV)]
    want = norm64(ts)
    norm, scale = Fops.grad_clip_scale(ts, 0.5)
    assert (norm.double() - want).abs() <= NORM_TOL * want
    mine = [t.clone() for t in ts]
    Fops.clip_grad_norm_(mine, 0.5)
    for a, t in zip(mine, ts):
        assert torch.equal(a, t * scale)
    m = [torch.randn(4, 6, device=DEV), torch.randn(5, device=DEV), torch.randn(6, 4, device=DEV).t()]
    g = [torch.randn(4, 6, device=DEV), torch.randn(5, device=DEV).bfloat16(), torch.randn(4, 6, device=DEV)]
    p = [m[0].clone(), m[1].bfloat16(), m[2].bfloat16()]
    assert not p[2].is_contiguous()
    want = [a - 0.1 * scale * b.float() for a, b in zip(m, g)]
    Fops.master_sgd_step_(p, m, g, lr=0.1, grad_scale=scale)
    for a, b, c in zip(m, want, p):
        assert torch.allclose(a, b, rtol=2.0 ** -22, atol=1e-9) and torch.equal(c, a.to(c.dtype))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_not_finite(bad):
    ts = tensors([1000, 20000], [torch.float32])
    ts[1][12345] = bad
    norm, scale = Fops.grad_clip_scale(ts, 1.0)
    assert torch.isinf(norm) if bad == float("inf") else torch.isnan(norm)
    assert scale == 0 if bad == float("inf") else torch.isnan(scale)


def test_zero_gradients():
    norm, scale = Fops.grad_clip_scale([torch.zeros(100, device=DEV)], 1.0)
    assert norm == 0 and scale == 1


@pytest.mark.parametrize("momentum,decay", [(0.0, 0.0), (0.9, 0.0), (0.9, 0.01), (0.0, 0.1)])
@pytest.mark.parametrize("gtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("scaled", [True, False])
def test_master_step(momentum, decay, gtype, scaled):
    sizes = [1, 2047, 2048, 2049, 16384, 50003] + [5] * 70
    m = tensors(sizes, [torch.float32], seed=1)
    g = tensors(sizes, [getattr(torch, gtype)], seed=2)
    b = tensors(sizes, [torch.float32], seed=3) if momentum else None
    p = [t.bfloat16() for t in m]
    scale = torch.tensor(0.37, device=DEV) if scaled else None
    want_m, want_b = [], []
    for i in range(len(sizes)):
        u = g[i].double() * (scale.double() if scaled else 1.0) + decay * m[i].double()
        if momentum:
            u = momentum * b[i].double() + u
            want_b.append(u)
        want_m.append(m[i].double() - 0.05 * u)
    size = [0.05 * (t.double().abs() + decay * q.double().abs() + (r.double().abs() if momentum else 0)) + q.double().abs()
            for t, q, r in zip(g, m, b or m)]
    Fops.master_sgd_step_(p, m, g, lr=0.05, momentum=momentum, weight_decay=decay, momentum_bufs=b, grad_scale=scale)
    for i in range(len(sizes)):
        assert ((m[i].double() - want_m[i]).abs() <= 6 * 2.0 ** -24 * size[i]).all()
        assert torch.equal(p[i], m[i].bfloat16())
        if momentum:
            assert ((b[i].double() - want_b[i]).abs() <= 6 * 2.0 ** -24 * 25 * size[i]).all()


def test_captured():
    g = tensors([1000, 30000, 77], [torch.bfloat16])
    m = tensors([1000, 30000, 77], [torch.float32], seed=1)
    p = [t.bfloat16() for t in m]

    def step():
        norm, scale = Fops.grad_clip_scale(g, 1.0)
        Fops.master_sgd_step_(p, m, g, lr=0.1, grad_scale=scale)
        return norm

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step()
    for i in range(3):
        for t in g:
            t.mul_(i + 1)
        keep = [t.clone() for t in m]
        graph.replay()
        torch.cuda.synchronize()
        got, got_norm = [t.clone() for t in m], norm.clone()
        for t, k in zip(m, keep):
            t.copy_(k)
        assert torch.equal(step(), got_norm)
        for a, t in zip(got, m):
            assert torch.equal(a, t)


def test_master_sgd_with_a_bound():
    """MasterSGD(max_grad_norm) against its own step on gradients clipped before."""
    def make():
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(*s, device=DEV).bfloat16()) for s in ((64, 33), (500,), (3, 5, 7))]
        for p in ps:
            p.grad = torch.randn_like(p)
        return ps

    a, b = make(), make()
    bound = MasterSGD(a, lr=0.1, momentum=0.9, weight_decay=0.01, max_grad_norm=0.5)
    plain = MasterSGD(b, lr=0.1, momentum=0.9, weight_decay=0.01)
    for _ in range(3):
        norm, scale = Fops.grad_clip_scale([p.grad for p in b], 0.5)
        bound.step()
        assert torch.equal(bound.last_grad_norm, norm)
        keep = [p.grad for p in b]
        for p in b:
            p.grad = None
        for p, g in zip(b, keep):
            p.grad = g.float().mul(scale).to(g.dtype)  # rounded once more than the fused step
        plain.step()
        for p, g in zip(b, keep):
            p.grad = g
    for x, y, g in zip(bound.masters, plain.masters, keep):
        # three steps of lr 0.1 and at most 2.71 gradients each, rounded to bf16: 2^-8
        assert ((x - y).abs() <= 0.1 * 3 * 2.71 * 2.0 ** -8 * g.float().abs() * float(scale) + 1e-6).all()


@pytest.mark.parametrize("mode", ["master", "momentum", "sr", "adam"])
def test_expert_steps_scaled(mode):
    """A scaled step is the step of scaled gradients: a power of two scales exactly."""
    scale = torch.tensor(0.25, device=DEV)
    out = []
    for scaled in (True, False):
        torch.manual_seed(0)
        stack = ExpertStack(3, 128, 64).to(DEV)
        stack.init_gpu_state(master_weights=mode != "sr")
        for g in (stack.main_grad_W1, stack.main_grad_W2, stack.main_grad_b1, stack.main_grad_b2):
            g.normal_()
            if not scaled:
                g.mul_(0.25)
        stack.grad_ready = True
        opt = (ExpertAdam(stack, lr=0.1) if mode == "adam" else
               FusedExpertSGD(stack, lr=0.1, momentum=0.9 if mode == "momentum" else 0.0, weight_decay=0.01,
                              stochastic_rounding=mode == "sr"))
        assert len(opt.gradients()) == 4
        opt.step(grad_scale=scale) if scaled else opt.step()
        out.append([stack.W1c, stack.W2c, stack.W1t, stack.W2t, stack.b1_f32, stack.b2_f32])
        assert opt.gradients() == []
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_scale_on_a_side_stream():
    torch.manual_seed(0)
    stack = ExpertStack(2, 128, 128).to(DEV)
    stack.init_gpu_state()
    opt = FusedExpertSGD(stack, lr=0.5)
    opt.set_side_stream(torch.cuda.Stream())
    stack.main_grad_W1.fill_(1.0)
    stack.grad_ready = True
    before = stack.W1.detach().clone()
    norm, scale = Fops.grad_clip_scale(opt.gradients(), 1.0)
    opt.step(grad_scale=scale)
    want = before - 0.5 * scale
    del norm, scale
    torch.empty(1, device=DEV).fill_(1e9)  # would take the scale's place if it were free
    torch.cuda.synchronize()
    assert torch.allclose(stack.W1, want, rtol=1e-6, atol=1e-7)


def test_refusals():
    with pytest.raises(ValueError, match="one device"):
        Fops.grad_clip_scale([torch.zeros(3, device=DEV), torch.zeros(3)], 1.0)
    with pytest.raises(ValueError, match="same shapes"):
        Fops.master_sgd_step_([torch.zeros(3, device=DEV).bfloat16()], [torch.zeros(3, device=DEV)],
                              [torch.zeros(4, device=DEV)], lr=0.1)
    torch.manual_seed(0)
    stack = ExpertStack(2, 256, 256).to(DEV)
    stack.init_gpu_state(master_weights=False)
    opt = FusedExpertSGD(stack, stochastic_rounding=True, fused_backward=True)
    with pytest.raises(RuntimeError, match="fused_backward"):
        opt.gradients()
    with pytest.raises(RuntimeError, match="fused_backward"):
        opt.step(grad_scale=torch.ones((), device=DEV))
