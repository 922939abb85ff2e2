"""Calls at the edges of the ragged expert path, on the GPU: arguments that do not go
together, no tokens, weights of little mass, derivatives that the operators do not have."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from learning_at_home_amd.ops import functional as Fops
    from learning_at_home_amd.parallel import ExpertParallelMoE, ExpertStack

DEV = "cuda:0"
BF = 2.0 ** -8  # one rounding to bf16: half a step


class TestRowsRefuse:
    """All refused on the host, before anything is launched."""

    def setup_method(self):
        self.layout = Fops.ragged_layout(torch.tensor([[0, 2], [2, 1], [-1, 1]], dtype=torch.int32, device=DEV), 3)
        self.x = torch.zeros(3, 8, device=DEV).bfloat16()
        self.y = torch.zeros(6, 8, device=DEV).bfloat16()
        self.w = torch.ones(3, 2, device=DEV)

    def test_gather(self):
        for x, match in ((self.x[:2], "x must be"), (self.x.float(), "bf16"), (self.x[:, :4], "multiple of 8"),
                         (self.x.cpu(), "one device")):
            with pytest.raises(ValueError, match=match):
                Fops.ragged_gather(x, self.layout)
        on_host = type(self.layout)(*(t.cpu() for t in self.layout))
        with pytest.raises(ValueError, match="one device"):
            Fops.ragged_gather(self.x, on_host)

    def test_combine(self):
        for change, match in ((dict(y=self.y[:5]), "y must be"), (dict(y=self.y.float()), "bf16"),
                              (dict(y=self.y[:, :4]), "multiple of 8"), (dict(y=self.y.cpu()), "one device"),
                              (dict(weights=self.w[:, :1]), "weights must be"), (dict(weights=self.w[:2]), "weights must be"),
                              (dict(weights=self.w.double()), "fp32"), (dict(weights=self.w.cpu()), "one device"),
                              (dict(layout=type(self.layout)(*(t.cpu() for t in self.layout))), "one device")):
            with pytest.raises(ValueError, match=match):
                Fops.ragged_combine(**{**dict(y=self.y, layout=self.layout, weights=self.w), **change})
        for y, match in ((self.y[:5], "y must be"), (self.y[:, :4], "multiple of 8"), (self.y.cpu(), "one device")):
            with pytest.raises(ValueError, match=match):
                Fops.ragged_ungather(y, self.layout)


def test_rows_from_views():
    """Rows, weights and gradients that are strided or start off 16 bytes give what copies of them give."""
    g = torch.Generator().manual_seed(0)
    layout = Fops.ragged_layout(torch.randint(-1, 5, (40, 2), generator=g).int().to(DEV), 5)
    x = torch.randn(40, 24, generator=g).bfloat16().to(DEV)
    w = torch.rand(40, 2, generator=g).to(DEV)
    dy = torch.randn(40, 24, generator=g).bfloat16().to(DEV)

    def off(t):
        out = torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)[1:].view(t.shape)
        return out.copy_(t)

    def run(x, w, dy):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        rows = Fops.ragged_gather(x, layout)
        out = Fops.ragged_combine(rows, layout, w)
        return (rows.detach(), out.detach(), Fops.ragged_ungather(rows, layout).detach(),
                *torch.autograd.grad(out, (x, w), dy))

    want = run(x, w, dy)
    wide = torch.zeros(40, 31, device=DEV).bfloat16()
    wide[:, 5:29] = x
    pairs = torch.zeros(40, 4, device=DEV)
    pairs[:, ::2] = w
    for got in (run(off(x), off(w), off(dy)), run(wide[:, 5:29], pairs[:, ::2], off(dy))):
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("least", [0.0, 0.2])
@pytest.mark.parametrize("D", [8, 24, 1032])
def test_weights_of_little_mass(D, least):
    """However small the weights are together, they are normalised; min_mass bounds that."""
    g = torch.Generator().manual_seed(D)
    T, k = 60, 4
    ids = torch.randint(0, 9, (T, k), generator=g).int()
    ids[torch.rand(T, k, generator=g) < 0.3] = -1
    ids[7] = -1
    layout = Fops.ragged_layout(ids.to(DEV), 9)
    w = torch.rand(T, k, generator=g) * 10.0 ** -torch.arange(T)[:, None].div(2, rounding_mode="floor")  # down to 1e-29
    w = w.to(DEV).requires_grad_(True)
    y = torch.randn(T * k, D, generator=g).bfloat16().to(DEV).requires_grad_(True)
    dy = torch.randn(T, D, generator=g).bfloat16().to(DEV)
    out = Fops.ragged_combine(y, layout, w, min_mass=least)
    dyy, dw = torch.autograd.grad(out, (y, w), dy)
    yd, wd = y.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    there = (layout.rows >= 0).double()
    mass = (wd * there).sum(1, keepdim=True)
    div = torch.where(mass > 0, mass.clamp(min=least), 1.0)
    share = wd * there / div
    rows = yd[layout.rows.clamp(min=0).long()]
    want = (share[..., None] * rows).sum(1)
    dyy64, dw64 = torch.autograd.grad(want, (yd, wd), dy.double())
    # shares: a sum of 4, an inverse and a product in fp32; then k products and sums; one rounding to bf16
    part = 16 * 2.0 ** -24
    with torch.no_grad():
        size = (share[..., None] * rows.abs()).sum(1)
        assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + part * size + 1e-30).all()
        assert ((dyy.double() - dyy64).abs() <= (2.0 ** -8 + part) * 1.01 * dyy64.abs() + 1e-30).all()
        # <dy, y_j> - <dy, y> with y as it was rounded, over the mass
        a = dy.double().abs()
        dots = (a[:, None] * rows.abs()).sum(-1) + (a * want.abs()).sum(-1, keepdim=True)
        tol = (2.0 ** -8 * 1.01 * (a * want.abs()).sum(-1, keepdim=True) + (D + 16) * 2.0 ** -24 * dots) / div
        assert torch.isfinite(dw).all()
        assert ((dw.double() - dw64).abs() <= (tol + part * dw64.abs()) * there + 1e-30).all()
    assert not out[7].any() and not dw[7].any()


class TestBiasGradient:
    @pytest.mark.parametrize("counts", [[1, 0, 2, 3, 1], [0, 0, 700, 128, 129, 127], [40000, 1, 0, 300], [0, 0], [1] * 600],
                             ids=["few", "tiles", "long", "none", "many"])
    @pytest.mark.parametrize("N", [8, 40, 136, 264, 2056])
    @pytest.mark.parametrize("bias", [torch.float32, torch.bfloat16])
    def test_sums_before_the_rounding(self, counts, N, bias):
        """Behind gelu, db adds what dx and dW take rounded to bf16: here within fp32 and the slope's fp16."""
        K, E, R = 8, len(counts), sum(counts) + 7
        g = torch.Generator(device=DEV).manual_seed(N + R)
        x = torch.randn(R, K, device=DEV, generator=g).bfloat16()
        w = torch.randn(E, N, K, device=DEV, generator=g).bfloat16()
        b = torch.randn(E, N, device=DEV, generator=g).to(bias)
        dy = torch.randn(R, N, device=DEV, generator=g).bfloat16()
        offsets = torch.nn.functional.pad(torch.tensor(counts, device=DEV).cumsum(0), (1, 0)).int()
        x[offsets[-1]:], dy[offsets[-1]:] = float("nan"), float("inf")  # rows of nobody

        def grads(which):
            leaves = [t.detach().clone().requires_grad_(n in which) for n, t in (("x", x), ("w", w), ("b", b))]
            y = Fops.grouped_linear(leaves[0], leaves[1], offsets, leaves[2], "gelu")
            return dict(zip(which, torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)))

        full = grads("xwb")
        at = offsets.tolist()
        for e in range(E) if E < 100 else range(0, E, 97):
            s = slice(at[e], at[e + 1])
            xd, wd, n = x[s].double(), w[e].double(), at[e + 1] - at[e]
            u = (xd @ wd.t() + b[e].double()).requires_grad_(True)
            dp, = torch.autograd.grad(torch.nn.functional.gelu(u, approximate="tanh"), u, dy[s].double())
            off = (K + 2) * 2.0 ** -23 * (xd.abs() @ wd.abs().t() + b[e].double().abs())
            # the slope: fp16 (2^-11 of it, 2^-25 below its normal range), its argument's error (its own slope
            # is at most 1), exp2 and reciprocal; then n products and sums in fp32; the result's own rounding
            tol = (2.0 ** -11 * dp.abs() + dy[s].double().abs() * (off + 2.0 ** -20)).sum(0) * 1.01
            tol = tol + (n + 1) * 2.0 ** -24 * dp.abs().sum(0) + torch.finfo(bias).eps / 2 * dp.sum(0).abs()
            assert ((full["b"][e].double() - dp.sum(0)).abs() <= tol * 1.01 + 1e-30).all()
        for which in ("b", "xb", "wb", "xw"):
            got = grads(which)
            for n in which:
                assert torch.equal(got[n], full[n]), (which, n)


class TestNoTokens:
    def make_stack(self):
        torch.manual_seed(0)
        stack = ExpertStack(4, 128, 256).to(DEV)
        stack.init_gpu_state()
        return stack

    def test_rows(self):
        """Gather, FFN and combine of no rows, forward and backward; nothing is left for a later check."""
        stack = self.make_stack()
        layout = Fops.ragged_layout(torch.empty(0, 2, dtype=torch.int32, device=DEV), 4)
        x = torch.empty(0, 128, device=DEV).bfloat16().requires_grad_(True)
        w = torch.empty(0, 2, device=DEV, requires_grad=True)
        for g in (stack.main_grad_W1, stack.main_grad_W2, stack.main_grad_b1, stack.main_grad_b2):
            g.fill_(1.0)
        rows = Fops.ragged_gather(x, layout)
        out = Fops.ragged_combine(Fops.ragged_ffn(rows, layout.offsets, stack), layout, w)
        assert rows.shape == out.shape == (0, 128) and Fops.ragged_ungather(rows, layout).shape == (0, 128)
        out.sum().backward()
        assert x.grad.shape == (0, 128) and w.grad.shape == (0, 2)
        for g in (stack.main_grad_W1, stack.main_grad_W2, stack.main_grad_b1, stack.main_grad_b2):
            assert not g.any()
        Fops.ragged_layout(torch.zeros(5, 2, dtype=torch.int32, device=DEV), 4)
        torch.cuda.synchronize()

    def test_rank_without_rows(self):
        """What a rank does that receives nothing while its own tokens go elsewhere: its layout has
        experts and no rows, and what it sent comes back."""
        stack = self.make_stack()
        arrived = torch.empty(0, 128, device=DEV).bfloat16().requires_grad_(True)
        layout = Fops.ragged_layout(torch.empty(0, dtype=torch.int32, device=DEV).unsqueeze(1), 4)
        y = Fops.ragged_ffn(Fops.ragged_gather(arrived, layout), layout.offsets, stack)
        y = Fops.ragged_ungather(y, layout)
        y.backward(torch.empty(0, 128, device=DEV).bfloat16())
        assert arrived.grad.shape == (0, 128) and stack.grad_ready and not stack.main_grad_W1.any()
        assert not Fops.ragged_layout(torch.full((3, 1), -1, dtype=torch.int32, device=DEV), 4).offsets.any()

    @pytest.mark.parametrize("dropless", [False, True])
    def test_layer(self, dropless):
        torch.manual_seed(5)
        moe = ExpertParallelMoE(128, 256, 8, k=2, dropless=dropless, z_loss_coef=0.1).to(DEV).bfloat16()
        moe.experts.float()
        moe.experts.init_gpu_state()
        x = torch.randn(0, 128, device=DEV).bfloat16().requires_grad_(True)
        y = moe(x)
        assert y.shape == (0, 128) and moe.aux_loss == 0 and not moe.last_counts.any()
        (y.sum() + moe.aux_loss).backward()
        assert x.grad.shape == (0, 128) and not moe.gate.weight.grad.any()
        moe(torch.randn(3, 128, device=DEV).bfloat16())  # no error was left behind
        torch.cuda.synchronize()


class TestDerivativesThatAreNotThere:
    def test_forward_mode(self):
        """A tangent is refused, not dropped; the CPU's plain torch keeps it."""
        torch.manual_seed(0)
        stack = ExpertStack(2, 128, 256).to(DEV)
        stack.init_gpu_state()
        x, w = torch.randn(4, 128, device=DEV).bfloat16(), torch.randn(2, 16, 128, device=DEV).bfloat16()
        b = torch.randn(2, 16, device=DEV)
        off = torch.tensor([0, 1, 4], dtype=torch.int32, device=DEV)
        layout = Fops.ragged_layout(torch.tensor([[0], [1], [1], [1]], dtype=torch.int32, device=DEV), 2)
        with fwd.dual_level():
            def dual(t):
                return fwd.make_dual(t, torch.ones_like(t))

            for call in (lambda: Fops.grouped_linear(dual(x), w, off), lambda: Fops.grouped_linear(x, dual(w), off),
                         lambda: Fops.grouped_linear(x, w, off, dual(b)), lambda: Fops.ragged_ffn(dual(x), off, stack),
                         lambda: Fops.ragged_gather(dual(x), layout),
                         lambda: Fops.ragged_combine(x, layout, dual(torch.ones(4, 1, device=DEV))),
                         lambda: Fops.grad_clip_scale([dual(b)], 1.0), lambda: Fops.clip_grad_norm_([b, dual(b.clone())], 1.0)):
                with pytest.raises(NotImplementedError, match="forward"):
                    call()
        Fops.grouped_linear(x, w, off, b)

    @pytest.mark.parametrize("what", ["gather", "ungather", "combine", "ffn"])
    def test_second_derivatives(self, what):
        """With create_graph=True the gradients are the same, and refuse to be differentiated."""
        torch.manual_seed(0)
        stack = ExpertStack(2, 128, 256).to(DEV)
        stack.init_gpu_state()
        layout = Fops.ragged_layout(torch.tensor([[0, 1], [1, -1], [1, 0]], dtype=torch.int32, device=DEV), 2)
        T = 3 if what == "gather" else 6
        x = torch.randn(T, 128, device=DEV).bfloat16().requires_grad_(True)
        w = torch.rand(3, 2, device=DEV, requires_grad=True)

        def call(x, w):
            return {"gather": lambda: Fops.ragged_gather(x, layout), "ungather": lambda: Fops.ragged_ungather(x, layout),
                    "combine": lambda: Fops.ragged_combine(x, layout, w),
                    "ffn": lambda: Fops.ragged_ffn(x, layout.offsets, stack)}[what]()

        leaves = (x, w) if what == "combine" else (x,)
        y = call(x, w)
        dy = torch.randn_like(y).requires_grad_(True)
        plain = torch.autograd.grad(call(x, w), leaves, dy)
        grads = torch.autograd.grad(call(x, w), leaves, dy, create_graph=True)
        for a, b in zip(plain, grads):
            assert torch.equal(a, b) and b.requires_grad
            with pytest.raises(RuntimeError, match="once"):
                torch.autograd.grad(b.float().square().sum(), dy, retain_graph=True)
            if what != "gather" and what != "ungather":  # linear: nothing of x in its gradient
                with pytest.raises(RuntimeError, match="once"):
                    torch.autograd.grad(b.float().square().sum(), leaves[-1], retain_graph=True)


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)], ids=str)
def test_norm_of_large_gradients(dtypes):
    """Finite gradients whose squares are beyond fp32 have a finite norm."""
    g = torch.Generator(device=DEV).manual_seed(0)
    ts = [torch.randn(n, device=DEV, generator=g).mul(s).to(dtypes[i % len(dtypes)]) for i, (n, s) in enumerate(
        [(16384, 1e25), (5, 1e30), (100_003, 1.0), (40_000, 1e19)])]
    want = torch.stack([t.double().square().sum() for t in ts]).sum().sqrt()
    norm, scale = Fops.grad_clip_scale(ts, 2.0)
    # squares and up to 64 sums in fp32, all positive: 2^-18 of the sum
    assert torch.isfinite(norm) and (norm.double() - want).abs() <= 2.0 ** -18 * want
    assert (scale.double() * want - 2.0).abs() <= 2 * 2.0 ** -18 * 2.0
    mine = [t.clone() for t in ts]
    Fops.clip_grad_norm_(mine, 2.0)
    after = torch.stack([t.double().square().sum() for t in mine]).sum().sqrt()
    # each element rounded to its type, and what was 1.0 is gone below fp32's range beside the largest
    assert (after - 2.0).abs() <= 2 * max(torch.finfo(t).eps / 2 for t in dtypes) * 2.0 + 2.0 ** -16
    ts[2][7] = float("inf")
    assert torch.isinf(Fops.grad_clip_scale(ts, 2.0)[0]) and Fops.grad_clip_scale(ts, 2.0)[1] == 0


def test_the_same_tensor_twice():
    """Written twice at once it would be scaled or stepped once or twice: refused, and nothing is written."""
    a, b = torch.ones(5, device=DEV), torch.ones(5, device=DEV)
    with pytest.raises(ValueError, match="twice"):
        Fops.clip_grad_norm_([a, b, a], 0.5)
    p, m, v = ([torch.ones(5, device=DEV).to(t) for _ in range(2)] for t in (torch.bfloat16, torch.float32, torch.float32))
    for change in (dict(params=[p[0], p[0]]), dict(masters=[m[0], m[0]]), dict(momentum_bufs=[v[1], v[1]])):
        args = dict(params=p, masters=m, grads=[a, a], lr=0.1, momentum=0.9, momentum_bufs=v)
        with pytest.raises(ValueError, match="twice"):
            Fops.master_sgd_step_(**{**args, **change})
    assert all((t == 1).all() for t in (a, b, *p, *m, *v))
    empty = torch.ones(0, device=DEV)
    Fops.clip_grad_norm_([empty, a, empty], 0.5)
    Fops.master_sgd_step_(p, m, [b, b], lr=0.1)  # read twice is fine
    assert (m[0] == m[1]).all() and (m[0] < 1).all()


def test_scale_is_one_number():
    """A vector as long as a tensor would scale it element by element on the CPU."""
    p, m, g = (torch.ones(3, device=DEV) for _ in range(3))
    for scale in (torch.ones(3, device=DEV), torch.ones(0, device=DEV)):
        with pytest.raises(ValueError, match="one number"):
            Fops.master_sgd_step_([p], [m], [g], lr=0.1, grad_scale=scale)
    with pytest.raises(ValueError, match="one number"):
        Fops.master_sgd_step_([p], [m], [g], lr=0.1, grad_scale=torch.ones(()))
    assert (m == 1).all()
    Fops.master_sgd_step_([p], [m], [g], lr=0.5, grad_scale=torch.full((1,), 0.5, device=DEV))
    assert (m == 0.75).all()


def test_masked_slots_reach_nothing():
    """NaN and infinity in a masked slot's weight, in rows of nobody or in another token's row stay there."""
    g = torch.Generator().manual_seed(0)
    ids = torch.tensor([[2, 0], [-1, 1], [1, -1], [-1, -1], [0, 2]], dtype=torch.int32).to(DEV)
    layout = Fops.ragged_layout(ids, 3)
    y = torch.randn(10, 8, generator=g).to(DEV, torch.bfloat16)
    w, dy = torch.rand(5, 2, generator=g).to(DEV), torch.randn(5, 8, generator=g).to(DEV, torch.bfloat16)

    def run(y, w):
        y, w = y.clone().requires_grad_(True), w.clone().requires_grad_(True)
        out = Fops.ragged_combine(y, layout, w)
        return (out.detach(), *torch.autograd.grad(out, (y, w), dy))

    clean = run(y, w)
    y2, w2 = y.clone(), w.clone()
    y2[6:] = float("nan")  # rows of nobody
    w2[1, 0], w2[2, 1], w2[3, 0] = float("nan"), float("inf"), float("nan")
    for a, b in zip(run(y2, w2), clean):
        assert torch.equal(a, b)
    y2[0] = float("inf")  # row 0 is token 0's or 4's, which alone may see it
    token = int((layout.rows == 0).any(1).nonzero())
    keep = [t for t in range(5) if t != token]
    out, dyy, dw = run(y2, w2)
    assert torch.equal(out[keep], clean[0][keep]) and torch.equal(dw[keep], clean[2][keep])
    own = layout.rows[token].tolist()
    assert all(torch.equal(dyy[r], clean[1][r]) for r in range(10) if r not in own)
