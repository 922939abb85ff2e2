"""The ragged expert path and gradient clipping on the CPU: meaning, gradients,
refusals, and the sharded dropless layer over gloo."""
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp
import torch.nn.functional as F

from learning_at_home_amd.ops import functional as Fops
from learning_at_home_amd.ops import ragged
from learning_at_home_amd.optim import MasterSGD
from learning_at_home_amd.parallel import ExpertAdam, ExpertParallelMoE, ExpertStack


def test_layout_by_hand():
    got = Fops.ragged_layout(torch.tensor([[1, 0], [2, -1], [1, 4]], dtype=torch.int32), 4)
    assert got.offsets.tolist() == [0, 1, 3, 4, 4]
    assert got.order.tolist() == [1, 0, 4, 2, -1, -1]
    assert got.rows.tolist() == [[1, 0], [3, -1], [2, -1]]


def test_gather_and_combine_invert():
    x = torch.randn(6, 8, dtype=torch.double)
    layout = Fops.ragged_layout(torch.tensor([[0, 2], [2, 1], [-1, 1], [-1, -1], [0, 1], [2, 0]]), 3)
    rows = Fops.ragged_gather(x, layout)
    for r, s in enumerate(layout.order.tolist()):
        assert torch.equal(rows[r], x[s // 2] if s >= 0 else torch.zeros(8, dtype=torch.double))
    w = torch.tensor([0.3, 0.7], dtype=torch.double).repeat(6, 1)
    out = Fops.ragged_combine(rows, layout, w)
    keep = [0, 1, 2, 4, 5]  # weights are normalised over the slots with a row
    assert torch.allclose(out[keep], x[keep]) and not out[3].any()
    back = Fops.ragged_ungather(rows, layout)
    for s, r in enumerate(layout.rows.flatten().tolist()):
        assert torch.equal(back[s], x[s // 2] if r >= 0 else torch.zeros(8, dtype=torch.double))


@pytest.mark.parametrize("activation", [None, "gelu"])
def test_grouped_linear_gradients(activation):
    offsets = torch.tensor([0, 2, 2, 5], dtype=torch.int32)
    x = torch.randn(6, 4, dtype=torch.double, requires_grad=True)
    w = torch.randn(3, 5, 4, dtype=torch.double, requires_grad=True)
    b = torch.randn(3, 5, dtype=torch.double, requires_grad=True)
    assert torch.autograd.gradcheck(lambda x, w, b: Fops.grouped_linear(x, w, offsets, b, activation), (x, w, b))
    y = Fops.grouped_linear(x, w, offsets, b, activation)
    assert not y[5].any()
    want = x[3] @ w[2].t() + b[2]
    assert torch.allclose(y[3], F.gelu(want, approximate="tanh") if activation else want)


class TestRefusals:
    x, w = torch.zeros(4, 8), torch.zeros(2, 16, 8)
    off = torch.tensor([0, 1, 4], dtype=torch.int32)

    @pytest.mark.parametrize("ids", [torch.zeros(4, dtype=torch.int32), torch.zeros(4, 2),
                                     torch.zeros(4, 2, dtype=torch.int16)])
    def test_layout_ids(self, ids):
        with pytest.raises(ValueError, match="topk_idx"):
            Fops.ragged_layout(ids, 3)

    @pytest.mark.parametrize("E", [0, -1, 4097])
    def test_layout_experts(self, E):
        with pytest.raises(ValueError, match="experts"):
            Fops.ragged_layout(torch.zeros(1, 1, dtype=torch.int32), E)

    @pytest.mark.parametrize("change,match", [
        (dict(x=torch.zeros(4, 7)), "x must be"),
        (dict(x=torch.zeros(4)), "x must be"),
        (dict(weight=torch.zeros(16, 8)), "weight"),
        (dict(offsets=torch.tensor([0, 4], dtype=torch.int32)), "offsets"),
        (dict(offsets=torch.tensor([0, 1, 4])), "offsets"),
        (dict(bias=torch.zeros(16)), "bias"),
        (dict(activation="relu"), "activation"),
        (dict(x=torch.zeros(4, 8, dtype=torch.double)), "one type"),
        (dict(x=torch.zeros(4, 8, device="meta")), "one device"),
    ])
    def test_product(self, change, match):
        args = dict(x=self.x, weight=self.w, offsets=self.off)
        with pytest.raises(ValueError, match=match):
            Fops.grouped_linear(**{**args, **change})

    @pytest.mark.parametrize("x,w,match", [
        (torch.zeros(4, 8), torch.zeros(2, 16, 8), "bf16"),
        (torch.zeros(4, 12).bfloat16(), torch.zeros(2, 16, 12).bfloat16(), "multiples of 8"),
        (torch.zeros(4, 8).bfloat16(), torch.zeros(2, 9, 8).bfloat16(), "multiples of 8"),
        (torch.zeros(4, 8).bfloat16(), torch.zeros(2, 0, 8).bfloat16(), "empty"),
        (torch.zeros(4, 8).bfloat16(), torch.empty(1, 1 << 15, 1 << 15, device="meta", dtype=torch.bfloat16), "2.30"),
    ])
    def test_what_the_kernels_do_not_take(self, x, w, match):
        with pytest.raises(ValueError, match=match):
            ragged._check_gpu_product(x, w)

    def test_ffn(self):
        stack = ExpertStack(2, 8, 16)
        with pytest.raises(ValueError, match="x must be"):
            Fops.ragged_ffn(torch.zeros(4, 9), self.off, stack)
        with pytest.raises(ValueError, match="offsets"):
            Fops.ragged_ffn(torch.zeros(4, 8), self.off[:2], stack)

    def test_clip(self):
        with pytest.raises(ValueError, match="no tensors"):
            Fops.grad_clip_scale([], 1.0)
        with pytest.raises(ValueError, match="positive"):
            Fops.grad_clip_scale([torch.zeros(1)], 0.0)
        with pytest.raises(ValueError, match="one device"):
            Fops.grad_clip_scale([torch.zeros(1), torch.zeros(1, device="meta")], 1.0)
        with pytest.raises(ValueError, match="positive"):
            MasterSGD([torch.nn.Parameter(torch.zeros(1))], max_grad_norm=-1.0)

    @pytest.mark.parametrize("change,match", [
        (dict(grads=[]), "go together"),
        (dict(momentum=0.9), "momentum_bufs"),
        (dict(grads=[torch.zeros(4)]), "shapes"),
        (dict(masters=[torch.zeros(3).bfloat16()]), "fp32"),
        (dict(momentum_bufs=[torch.zeros(2)]), "shapes"),
    ])
    def test_step(self, change, match):
        args = dict(params=[torch.zeros(3)], masters=[torch.zeros(3)], grads=[torch.zeros(3)], lr=0.1)
        with pytest.raises(ValueError, match=match):
            Fops.master_sgd_step_(**{**args, **change})

    def test_moe(self):
        with pytest.raises(ValueError, match="a2a_chunks"):
            ExpertParallelMoE(8, 16, 4, dropless=True, a2a_chunks=2)


def test_norm_and_clip_as_torch():
    ps = [torch.nn.Parameter(torch.randn(s)) for s in ((3, 4), (7,), ())]
    for p in ps:
        p.grad = torch.randn_like(p)
    mine = [p.grad.clone() for p in ps]
    want = torch.nn.utils.clip_grad_norm_(ps, 0.5)
    got = Fops.clip_grad_norm_(mine, 0.5)
    assert torch.allclose(got, want, rtol=2.0 ** -18)
    for a, p in zip(mine, ps):
        assert torch.allclose(a, p.grad, rtol=2.0 ** -18)


@pytest.mark.parametrize("momentum,decay", [(0.0, 0.0), (0.9, 0.01)])
def test_scaled_master_step(momentum, decay):
    """MasterSGD with a scale of 1 against its plain step."""
    out = []
    for scale in (None, torch.ones(())):
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(5, 3).bfloat16()), torch.nn.Parameter(torch.randn(4).bfloat16())]
        opt = MasterSGD(ps, lr=0.1, momentum=momentum, weight_decay=decay)
        ps[0].grad = torch.randn(5, 3).bfloat16()  # the other has none
        for _ in range(3):
            opt.step(grad_scale=scale)
        out.append((opt.masters, ps))
    for a, b in zip(out[0][0] + out[0][1], out[1][0] + out[1][1]):
        assert torch.equal(a, b)


def test_adam_scaled():
    out = []
    for scale in (None, torch.tensor(0.5)):
        torch.manual_seed(0)
        stack = ExpertStack(2, 8, 16)
        opt = ExpertAdam(stack)
        assert opt.gradients() == []
        for p in stack.parameters():
            p.grad = torch.randn_like(p) * (0.5 if scale is None else 1.0)
        assert len(opt.gradients()) == 4
        opt.step(grad_scale=scale)
        out.append([p.detach().clone() for p in stack.parameters()])
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("k", [1, 2])
def test_dropless_as_roomy_capacity(k):
    out = []
    for dropless in (False, True):
        torch.manual_seed(3)
        moe = ExpertParallelMoE(16, 32, 8, k=k, capacity_factor=8.0, dropless=dropless).eval()
        x = torch.randn(30, 16, requires_grad=True)
        y = moe(x)
        (y * torch.arange(16)).sum().backward()
        out.append((y, x.grad, *(p.grad for p in moe.parameters()), moe.aux_loss, moe.last_counts))
    for a, b in zip(*out):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


def test_dropless_departed_experts():
    torch.manual_seed(3)
    moe = ExpertParallelMoE(16, 32, 8, k=2, dropless=True, router_noise_std=0.0)
    moe.update_membership(None, [1], 2)  # slot 0's experts 0..3 are gone; this rank is slot 1
    moe.experts = ExpertStack(4, 16, 32)
    x = torch.randn(10, 16, requires_grad=True)
    y = moe(x)
    y.sum().backward()
    assert moe.last_counts[:4].sum() == 0 and moe.last_counts[4:].sum() == 20
    assert torch.isfinite(x.grad).all() and moe.experts.W1.grad.abs().sum() > 0


def _sharded_worker(rank, world, port, full, x, dy, queue):
    import torch.distributed as dist

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.manual_seed(0)
    moe = ExpertParallelMoE(16, 32, 8, k=2, dropless=True).eval()
    with torch.no_grad():
        moe.gate.weight.copy_(full["gate"])
        for n in ("W1", "W2", "W1_bias", "W2_bias"):
            getattr(moe.experts, n).copy_(full[n][rank * 4 : rank * 4 + 4])
    leaf = x[rank].clone().requires_grad_(True)
    y = moe(leaf)
    (y * dy[rank]).sum().backward()
    queue.put((rank, y.detach().numpy(), leaf.grad.numpy(), moe.experts.W1.grad.numpy()))
    dist.barrier()
    dist.destroy_process_group()


def test_sharded_over_gloo():
    """Two ranks with uneven tokens against one process."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    torch.manual_seed(1)
    moe = ExpertParallelMoE(16, 32, 8, k=2, dropless=True).eval()
    full = {"gate": moe.gate.weight.detach(), **{n: getattr(moe.experts, n).detach()
                                                 for n in ("W1", "W2", "W1_bias", "W2_bias")}}
    x = [torch.randn(13, 16), torch.randn(5, 16)]
    dy = [torch.randn(13, 16), torch.randn(5, 16)]
    want, grads = [], []
    for a, d in zip(x, dy):
        leaf = a.clone().requires_grad_(True)
        y = moe(leaf)
        (y * d).sum().backward()
        want.append(y.detach())
        grads.append(leaf.grad)
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    procs = [ctx.Process(target=_sharded_worker, args=(r, 2, port, full, x, dy, queue)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict((r[0], r[1:]) for r in (queue.get(timeout=120) for _ in procs))
    for p in procs:
        p.join(60)
    for r in range(2):
        y, dx, dW1 = (torch.from_numpy(a) for a in got[r])
        assert torch.allclose(y, want[r], rtol=1e-5, atol=1e-6)
        assert torch.allclose(dx, grads[r], rtol=1e-4, atol=1e-5)
        assert torch.allclose(dW1, moe.experts.W1.grad[r * 4 : r * 4 + 4], rtol=1e-4, atol=1e-5)
