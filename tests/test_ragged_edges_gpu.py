"""Calls at the edges of the ragged expert path, on the GPU: arguments that do not go
together, no tokens, weights of little mass, derivatives that the operators do not have."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from learning_at_home_amd.ops import functional as Fops

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
