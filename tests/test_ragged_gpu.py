"""GPU numerics of the ragged expert path (ops/ragged.py) against plain torch in
64 bits. Bounds come from the arithmetic: inputs are bf16 and exact in both, a
sum of n products in fp32 is off by at most n * 2^-23 of the sum of their sizes
(half a step for each addition is 2^-24; the matrix instructions may truncate),
one rounding to bf16 by half a step, 2^-8 of the value."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from learning_at_home_amd.models import GraphDecoder, TransformerDMoE, TransformerDMoEConfig
    from learning_at_home_amd.ops import functional as Fops
    from learning_at_home_amd.parallel import ExpertParallelMoE, ExpertStack, FusedExpertSGD

DEV = "cuda:0"
BF = 2.0 ** -8  # one rounding to bf16


def offsets_of(counts):
    return F.pad(torch.tensor(counts, device=DEV).cumsum(0), (1, 0)).int()


def problem(counts, K, N, tail=0, bias=torch.float32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    E, R = len(counts), sum(counts) + tail
    return (rand(R, K).bfloat16(), (rand(E, N, K) * K ** -0.5).bfloat16(),
            None if bias is None else rand(E, N).to(bias), offsets_of(counts), rand(R, N).bfloat16())


def exact(x, w, b, offsets, dy, gelu):
    """Every output in 64 bits, and how far the kernels may be from it."""
    at = offsets.tolist()
    x, w, dy = x.double(), w.double(), dy.double()
    b = torch.zeros(w.shape[:2], device=DEV, dtype=torch.double) if b is None else b.double()
    R, K, N = x.shape[0], x.shape[1], w.shape[1]
    out = {n: torch.zeros(s, device=DEV, dtype=torch.double) for n, s in
           (("y", (R, N)), ("dx", (R, K)), ("dw", w.shape), ("db", b.shape))}
    tol = {n: torch.zeros_like(v) for n, v in out.items()}
    for e in range(w.shape[0]):
        s = slice(at[e], at[e + 1])
        n = at[e + 1] - at[e]
        u = (x[s] @ w[e].t() + b[e]).requires_grad_(True)
        # the sum before gelu, whose slope is at most 1.13; its exp2 and reciprocal: 2^-20 of the value
        off = (K + 2) * 2.0 ** -23 * (x[s].abs() @ w[e].abs().t() + b[e].abs())
        y = F.gelu(u, approximate="tanh") if gelu else u * 1
        out["y"][s] = y.detach()
        tol["y"][s] = BF * y.detach().abs() + (1.13 * off + 2.0 ** -20 * u.detach().abs() if gelu else off)
        dp, = torch.autograd.grad(y, u, dy[s])
        # with gelu: the slope (its second derivative is at most 1) is rounded to fp16 (2^-11 of it, or
        # 2^-25 where it is below fp16's normal range), dP to bf16
        doff = (BF + 2.0 ** -11) * 1.01 * dp.abs() + dy[s].abs() * (off + 2.0 ** -20) * 1.01 if gelu else torch.zeros_like(dp)
        dx = dp @ w[e]
        out["dx"][s] = dx
        tol["dx"][s] = BF * dx.abs() + (doff @ w[e].abs()) * 1.01 + N * 2.0 ** -23 * (dp.abs() @ w[e].abs())
        out["dw"][e] = dp.t() @ x[s]
        tol["dw"][e] = BF * out["dw"][e].abs() + 1.01 * doff.t() @ x[s].abs() + n * 2.0 ** -23 * (dp.abs().t() @ x[s].abs())
        out["db"][e] = dp.sum(0)
        tol["db"][e] = BF * out["db"][e].abs() + 1.01 * doff.sum(0) + n * 2.0 ** -23 * dp.abs().sum(0)
    return out, tol


def close(name, got, want, tol):
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), name
    over = (got.double() - want).abs() - tol * (1 + 2.0 ** -10) - 1e-30
    assert not (over > 0).any(), f"{name}: {over.max().item():.3g} over its bound"


def run_all(x, w, b, offsets, dy, gelu):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    b_leaf = leaves[2] if b is not None else None
    y = Fops.grouped_linear(leaves[0], leaves[1], offsets, b_leaf, "gelu" if gelu else None)
    grads = torch.autograd.grad(y, leaves, dy)
    return dict(zip(("y", "dx", "dw", "db"), (y.detach(), *grads)))


COUNTS = {
    "one-row": [1],
    "few": [3, 0, 1, 0, 0, 17, 2, 1],
    "none": [0, 0, 0],
    "tiles": [128, 129, 127, 0, 256, 1],
    "skewed": [0, 700, 0, 1, 5, 0],
    "many": [i % 7 for i in range(300)],
}


class TestLayout:
    @pytest.mark.parametrize("T,k,E", [(1, 1, 1), (8, 4, 256), (5, 2, 3), (1000, 4, 12), (1024, 4, 256),
                                       (1025, 4, 256), (4097, 1, 1024), (3000, 8, 4096), (20000, 4, 4096),
                                       (65537, 1, 1024), (98304, 4, 256), (9, 1, 257)])
    @pytest.mark.parametrize("wide", [False, True])
    def test_sorted(self, T, k, E, wide):
        g = torch.Generator().manual_seed(T + E)
        ids = torch.randint(-1 - E // 8, E + E // 8 + 1, (T, k), generator=g)
        ids = ids if wide else ids.int()
        got = Fops.ragged_layout(ids.to(DEV), E)
        want = Fops.ragged_layout(ids, E)
        for a, b in zip(got, want):
            assert a.dtype == torch.int32 and torch.equal(a.cpu(), b)

    @pytest.mark.parametrize("fill", [-1, 0, 6, 7])
    def test_one_choice(self, fill):
        ids = torch.full((5000, 2), fill, dtype=torch.int32)
        for a, b in zip(Fops.ragged_layout(ids.to(DEV), 7), Fops.ragged_layout(ids, 7)):
            assert torch.equal(a.cpu(), b)

    def test_no_tokens(self):
        got = Fops.ragged_layout(torch.empty(0, 4, dtype=torch.int32, device=DEV), 5)
        assert got.offsets.tolist() == [0] * 6 and got.order.numel() == 0 and got.rows.shape == (0, 4)

    def test_strided_ids(self):
        ids = torch.randint(0, 9, (50, 6)).int()
        got = Fops.ragged_layout(ids.to(DEV)[:, ::2], 9)
        for a, b in zip(got, Fops.ragged_layout(ids[:, ::2], 9)):
            assert torch.equal(a.cpu(), b)

    def test_captured(self):
        ids = torch.randint(0, 256, (6000, 4), device=DEV, dtype=torch.int32)
        Fops.ragged_layout(ids, 256)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = Fops.ragged_layout(ids, 256)
        for seed in range(3):
            new = torch.randint(-1, 256, (6000, 4), generator=torch.Generator().manual_seed(seed)).int()
            ids.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, Fops.ragged_layout(new, 256)):
                assert torch.equal(a.cpu(), b)


class TestGroupedLinear:
    @pytest.mark.parametrize("counts", list(COUNTS), ids=str)
    @pytest.mark.parametrize("K,N", [(8, 8), (136, 328), (64, 256), (520, 72)])
    @pytest.mark.parametrize("gelu", [False, True])
    def test_forward_and_gradients(self, counts, K, N, gelu):
        p = problem(COUNTS[counts], K, N, tail=5)
        want, tol = exact(*p, gelu)
        got = run_all(*p, gelu)
        for name in got:
            close(name, got[name], want[name], tol[name])
        with torch.no_grad():
            y = Fops.grouped_linear(p[0], p[1], p[3], p[2], "gelu" if gelu else None)
        close("y", y, want["y"], tol["y"])

    @pytest.mark.parametrize("bias", [None, torch.bfloat16])
    def test_bias_types(self, bias):
        p = problem([40, 3, 200], 72, 136, tail=1, bias=bias)
        want, tol = exact(*p, False)
        got = run_all(*p, False)
        for name in got:
            close(name, got[name], want[name], tol[name])

    def test_against_differences(self):
        """The gradient along a direction against the change of a 64-bit loss."""
        x, w, b, offsets, dy = problem([9, 0, 33], 40, 24)
        got = run_all(x, w, b, offsets, dy, True)
        gen = torch.Generator(device=DEV).manual_seed(1)

        def loss(x, w, b):
            return (exact(x, w, b, offsets, dy, True)[0]["y"] * dy.double()).sum()

        for name, at, leaf in (("dx", 0, x), ("dw", 1, w), ("db", 2, b)):
            d = torch.randn(leaf.shape, device=DEV, generator=gen, dtype=torch.double)
            h = 1e-4
            args = [t.double() for t in (x, w, b)]
            up, down = list(args), list(args)
            up[at], down[at] = args[at] + h * d, args[at] - h * d
            slope = (loss(*up) - loss(*down)) / (2 * h)
            mine = (got[name].double() * d).sum()
            tol = (exact(x, w, b, offsets, dy, True)[1][name] * d.abs()).sum() + 1e-5 * slope.abs() + 1e-5
            assert (mine - slope).abs() <= tol

    def test_rows_of_nobody(self):
        """What stands behind the last group, and in other groups, reaches nothing."""
        x, w, b, offsets, dy = problem([50, 70, 0, 9], 72, 136, tail=40)
        clean = run_all(x, w, b, offsets, dy, True)
        assert not clean["y"][129:].any() and not clean["dx"][129:].any()
        assert not clean["dw"][2].any() and not clean["db"][2].any()
        x2, dy2, w2 = x.clone(), dy.clone(), w.clone()
        x2[129:], dy2[129:] = float("nan"), float("inf")
        w2[2] = float("nan")  # an expert without rows
        got = run_all(x2, w2, b, offsets, dy2, True)
        for name in got:
            assert torch.equal(got[name], clean[name]), name
        x3 = x.clone()
        x3[60] = float("inf")  # a row of expert 1
        got = run_all(x3, w, b, offsets, dy, False)
        fine = run_all(x, w, b, offsets, dy, False)
        keep = torch.ones(169, dtype=torch.bool, device=DEV)
        keep[60] = False
        assert torch.equal(got["y"][keep], fine["y"][keep])
        assert torch.equal(got["dw"][[0, 2, 3]], fine["dw"][[0, 2, 3]])

    def test_views(self):
        """Rows of a wider tensor, a start off 16 bytes, a gradient that is expanded."""
        x, w, b, offsets, _ = problem([13, 20], 64, 128)
        wide = torch.zeros(33, 100, device=DEV, dtype=torch.bfloat16)
        wide[:, 3:67] = x
        off = torch.empty(w.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view_as(w).copy_(w)
        assert off.data_ptr() % 16
        base = Fops.grouped_linear(x, w, offsets, b)
        assert torch.equal(Fops.grouped_linear(wide[:, 3:67], off, offsets, b), base)
        leaf = x.clone().requires_grad_(True)
        Fops.grouped_linear(leaf, w, offsets, b).sum().backward()
        want = run_all(x, w, b, offsets, torch.ones_like(base), False)["dx"]
        assert torch.equal(leaf.grad, want)

    def test_only_what_is_asked(self):
        x, w, b, offsets, dy = problem([13, 20], 64, 128)
        full = run_all(x, w, b, offsets, dy, False)
        for i, name in enumerate(("dx", "dw", "db")):
            leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
            y = Fops.grouped_linear(leaves[0], leaves[1], offsets, leaves[2])
            grad, = torch.autograd.grad(y, leaves[i], dy)
            assert torch.equal(grad, full[name])

    @pytest.mark.parametrize("change,match", [
        (dict(x=torch.zeros(4, 7).bfloat16()), "x must be"),
        (dict(x=torch.zeros(4, 8)), "bf16"),
        (dict(weight=torch.zeros(2, 9, 8).bfloat16()), "multiples of 8"),
        (dict(weight=torch.zeros(2, 0, 8).bfloat16()), "empty"),
        (dict(offsets=torch.tensor([0, 1, 4])), "offsets"),
        (dict(offsets=torch.tensor([0, 4]).int()), "offsets"),
        (dict(bias=torch.zeros(2, 8)), "bias"),
        (dict(bias=torch.zeros(2, 16).half()), "bias"),
        (dict(activation="relu"), "activation"),
        (dict(weight=torch.zeros(4097, 16, 8).bfloat16(), offsets=torch.zeros(4098).int()), "4096"),
    ])
    def test_refusals(self, change, match):
        args = dict(x=torch.zeros(4, 8).bfloat16(), weight=torch.zeros(2, 16, 8).bfloat16(),
                    offsets=torch.tensor([0, 1, 4]).int(), bias=None, activation=None)
        args.update(change)
        with pytest.raises(ValueError, match=match):
            Fops.grouped_linear(*(t.to(DEV) if isinstance(t, torch.Tensor) else t for t in args.values()))

    def test_refuses_two_devices_and_second_derivatives(self):
        x, w, b, offsets, dy = problem([3, 2], 8, 16)
        with pytest.raises(ValueError, match="one device"):
            Fops.grouped_linear(x, w.cpu(), offsets)
        x.requires_grad_(True)
        y = Fops.grouped_linear(x, w, offsets)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(y, x, dy, create_graph=True)

    @pytest.mark.parametrize("counts", [[5000, 1, 0, 3000], [0, 0, 70000], [300] * 16])
    @pytest.mark.parametrize("gelu", [False, True])
    def test_rows_in_parts(self, counts, gelu):
        """Fewer tiles than CUs: each expert's rows are summed in parts and joined."""
        p = problem(counts, 136, 72, tail=7, bias=torch.bfloat16)
        want, tol = exact(*p, gelu)
        got = run_all(*p, gelu)
        for name in got:
            close(name, got[name], want[name], tol[name])
        again = run_all(*p, gelu)
        for name in got:
            assert torch.equal(got[name], again[name])

    # tiles of fewer rows than their half, of all, of one more; one expert alone; none at all
    @pytest.mark.parametrize("counts", [[20000, 1, 129, 0, 128, 127, 257, 15000], [0, 0, 36000], [0, 0, 0],
                                        [i * 37 % 500 for i in range(140)]])
    @pytest.mark.parametrize("K,N", [(520, 520), (8, 2056), (64, 2048), (2056, 8), (200, 1992)])
    def test_large_tiles(self, counts, K, N):
        """Many rows an expert and many tiles: forward, or dx, or both by the large tiles."""
        p = problem(counts, K, N, tail=40 if sum(counts) else 40000, bias=torch.bfloat16 if K == 520 else torch.float32)
        gelu = N != 2048
        want, tol = exact(*p, gelu)
        got = run_all(*p, gelu)
        for name in got:
            close(name, got[name], want[name], tol[name])
        again = run_all(*p, gelu)
        for name in got:
            assert torch.equal(got[name], again[name])
        with torch.no_grad():  # without the slope
            y = Fops.grouped_linear(p[0], p[1], p[3], None if K == 8 else p[2], "gelu" if gelu else None)
        if K == 8:
            want, tol = exact(p[0], p[1], None, p[3], p[4], gelu)
        close("y", y, want["y"], tol["y"])

    @pytest.mark.parametrize("counts", [[0, 3000, 1, 700, 700, 0, 20000, 64, 65] * 8, [300] * 65, [0] * 69 + [30000]])
    def test_weight_gradients_by_rows(self, counts):
        """More tiles than blocks, experts of very different rows."""
        p = problem(counts, 264, 776, tail=9)
        want, tol = exact(*p, False)
        got = run_all(*p, False)
        for name in got:
            close(name, got[name], want[name], tol[name])

    @pytest.mark.parametrize("counts", ["tiles", "skewed", "many"])
    @pytest.mark.parametrize("K,N", [(264, 1288), (72, 2048), (8, 4096)])
    @pytest.mark.parametrize("gelu", [False, True])
    def test_wide_outputs(self, counts, K, N, gelu):
        """Too many outputs for the small tiles, too few rows for the large ones."""
        p = problem(COUNTS[counts], K, N, tail=5, bias=torch.bfloat16 if gelu else torch.float32)
        want, tol = exact(*p, gelu)
        got = run_all(*p, gelu)
        for name in got:
            close(name, got[name], want[name], tol[name])
        with torch.no_grad():
            y = Fops.grouped_linear(p[0], p[1], p[3], p[2], "gelu" if gelu else None)
        close("y", y, want["y"], tol["y"])

    @pytest.mark.parametrize("counts", [[70, 0, 130, 1], [3, 0, 1], [600, 700]])
    @pytest.mark.parametrize("K,N", [(1032, 2056), (2000, 1288), (4096, 1288), (1032, 136)])
    @pytest.mark.parametrize("gelu", [False, True])
    def test_contraction_in_parts(self, counts, K, N, gelu):
        """Fewer tiles than CUs and a long contraction: summed in parts and joined."""
        p = problem(counts, K, N, tail=7, bias=torch.bfloat16 if gelu else torch.float32)
        want, tol = exact(*p, gelu)
        got = run_all(*p, gelu)
        for name in got:
            close(name, got[name], want[name], tol[name])
        again = run_all(*p, gelu)
        for name in got:
            assert torch.equal(got[name], again[name])
        with torch.no_grad():
            y = Fops.grouped_linear(p[0], p[1], p[3], p[2], "gelu" if gelu else None)
        close("y", y, want["y"], tol["y"])

    def test_parts_captured(self):
        x, w, b, offsets, dy = problem([70, 0, 130, 1], 1032, 2056, tail=100)
        leaves = [t.requires_grad_(True) for t in (x, w, b)]

        def step():
            y = Fops.grouped_linear(x, w, offsets, b, "gelu")
            return (y, *torch.autograd.grad(y, leaves, dy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for _ in range(2):  # each with sums of its own
            graphs.append((torch.cuda.CUDAGraph(), []))
            with torch.cuda.graph(graphs[-1][0]):
                graphs[-1][1].extend(step())
        for counts in ([70, 0, 130, 1], [0, 301, 0, 0], [10, 20, 30, 40]):
            with torch.no_grad():
                offsets.copy_(offsets_of(counts))
            torch.cuda.synchronize()
            for graph, _ in graphs:
                with torch.cuda.stream(side):
                    graph.replay()
                step()
            torch.cuda.synchronize()
            now = step()
            for _, held in graphs:
                for a, b_ in zip(held, now):
                    assert torch.equal(a, b_)

    def test_no_rows(self):
        p = problem([0, 0, 0], 40, 24)
        assert p[0].shape == (0, 40)
        got = run_all(*p, True)
        assert got["y"].shape == (0, 24) and got["dx"].shape == (0, 40)
        assert not got["dw"].any() and not got["db"].any()
        with torch.no_grad():
            assert Fops.grouped_linear(p[0], p[1], p[3]).shape == (0, 24)

    @pytest.mark.parametrize("each", [1, 3, 100])
    def test_most_experts(self, each):
        p = problem([each] * 4096, 8, 136, tail=1)
        want, tol = exact(*p, False)
        got = run_all(*p, False)
        for name in got:
            close(name, got[name], want[name], tol[name])

    def test_weight_gradients_of_wide_outputs(self):
        """More than 256 tiles an expert: none is worth pieces."""
        p = problem([600, 0, 400], 4352, 4360)
        want, tol = exact(*p, False)
        got = run_all(*p, False)
        for name in got:
            close(name, got[name], want[name], tol[name])

    @pytest.mark.parametrize("gelu", [False, True])
    def test_weight_gradients_in_pieces(self, gelu):
        """Some experts with many more rows than others, more tiles than blocks: pieces for them."""
        counts = [0, 30000, 1, 500, 6400, 0, 64, 12345] + [300] * 42
        p = problem(counts, 776, 264, tail=9, bias=torch.bfloat16 if gelu else torch.float32)
        want, tol = exact(*p, gelu)
        got = run_all(*p, gelu)
        for name in got:
            close(name, got[name], want[name], tol[name])
        again = run_all(*p, gelu)
        for name in got:
            assert torch.equal(got[name], again[name])
        x, dy = p[0], p[4]
        for accumulate in (False, True):  # a stack's own sums
            from learning_at_home_amd.ops import _C

            dw = torch.ones(len(counts), 264, 776, device=DEV)
            db = torch.ones(len(counts), 264, device=DEV)
            _C.ragged_tn(dy, x, p[3], dw, db, accumulate)
            want, tol = exact(x, p[1], None, p[3], dy, False)
            # without the rounding to bf16; the sum with what was there is rounded once more
            for name, g in (("dw", dw), ("db", db)):
                close(name, g, want[name] + accumulate,
                      tol[name] - BF * want[name].abs() + 2.0 ** -23 * (want[name].abs() + 1))

    def test_weights_past_the_cache(self):
        p = problem([3] * 38 + [0, 140], 2056, 2048, tail=3)
        assert p[1].numel() * 2 > 256 << 20
        want, tol = exact(*p, True)
        got = run_all(*p, True)
        for name in got:
            close(name, got[name], want[name], tol[name])

    def test_large_tiles_keep_to_their_rows(self):
        x, w, b, offsets, dy = problem([20000, 300, 0, 16000], 264, 520, tail=300)
        end = 36300
        clean = run_all(x, w, b, offsets, dy, True)
        assert not clean["y"][end:].any() and not clean["dx"][end:].any()
        x2, dy2, w2 = x.clone(), dy.clone(), w.clone()
        x2[end:], dy2[end:] = float("nan"), float("inf")
        w2[2] = float("nan")
        got = run_all(x2, w2, b, offsets, dy2, True)
        for name in got:
            assert torch.equal(got[name], clean[name]), name

    def test_large_tiles_captured_and_beside_others(self):
        """Graphs of different sizes, replayed at once on two streams, with eager work between."""
        cases = []
        for counts, K, N in (([20000, 300, 0, 16000], 264, 520), ([3000, 5000], 128, 72), ([9000, 30000], 520, 600)):
            x, w, b, offsets, dy = problem(counts, K, N, tail=300)
            leaves = [t.requires_grad_(True) for t in (x, w, b)]

            def step(x=x, w=w, b=b, offsets=offsets, dy=dy, leaves=leaves):
                y = Fops.grouped_linear(x, w, offsets, b, "gelu")
                return (y, *torch.autograd.grad(y, leaves, dy))

            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = step()
            cases.append((graph, held, step, side, dy))
        for i in range(3):
            for _, _, _, _, dy in cases:
                dy.add_(i)
            torch.cuda.synchronize()
            for graph, _, _, side, _ in cases:
                with torch.cuda.stream(side):
                    graph.replay()
            now = [step() for _, _, step, _, _ in cases]
            torch.cuda.synchronize()
            for (_, held, _, _, _), eager in zip(cases, now):
                for a, b_ in zip(held, eager):
                    assert torch.equal(a, b_)

    @pytest.mark.parametrize("counts", [[1], [0, 3, 0, 0, 1, 0], [2] * 20, [0] * 300 + [40], [1] * 4096])
    @pytest.mark.parametrize("K,N", [(8, 8), (1000, 40), (256, 264)])
    def test_few_rows(self, counts, K, N):
        p = problem(counts, K, N, tail=2)
        for gelu in (False, True):
            want, tol = exact(*p, gelu)
            with torch.no_grad():
                y = Fops.grouped_linear(p[0], p[1], p[3], p[2], "gelu" if gelu else None)
            close("y", y, want["y"], tol["y"])

    def test_same_bits_again(self):
        p = problem([300, 0, 77, 512], 256, 520, seed=3)
        a, b = run_all(*p, True), run_all(*p, True)
        for name in a:
            assert torch.equal(a[name], b[name])

    def test_other_stream(self):
        p = problem([300, 77], 256, 512)
        want = run_all(*p, True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run_all(*p, True)
        torch.cuda.current_stream().wait_stream(side)
        for name in want:
            assert torch.equal(got[name], want[name])

    def test_captured_forward_and_backward(self):
        x, w, b, offsets, dy = problem([300, 0, 77], 136, 264, tail=20)
        leaves = [t.requires_grad_(True) for t in (x, w, b)]

        def step():
            y = Fops.grouped_linear(x, w, offsets, b, "gelu")
            return (y, *torch.autograd.grad(y, leaves, dy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for i, counts in enumerate(([300, 0, 77], [1, 376, 0], [0, 0, 0], [100, 100, 100])):
            with torch.no_grad():
                offsets.copy_(offsets_of(counts))
                dy.add_(i)
            graph.replay()
            torch.cuda.synchronize()
            for a, b_ in zip(held, step()):
                assert torch.equal(a, b_)

    @pytest.mark.parametrize("wide_out", [True, False])
    def test_past_32_bits(self, wide_out):
        """More than 2^31 elements, and 2^32 bytes in one group, on either side."""
        R, K, N = (270336, 8, 8192) if wide_out else (270336, 8192, 8)
        counts = [3, R - 8, 4]
        x = torch.randn(64, K, device=DEV).bfloat16().repeat(R // 64, 1)
        w = (torch.randn(3, N, K, device=DEV) * K ** -0.5).bfloat16()
        offsets = offsets_of(counts)
        x.requires_grad_(True), w.requires_grad_(True)
        y = Fops.grouped_linear(x, w, offsets)
        e = torch.bucketize(torch.arange(R, device=DEV), offsets[1:].long(), right=True)
        for r in (0, 3, 262143, 262144, R - 10, R - 6, R - 5, R - 2):
            row = x[r].double() @ w[e[r].clamp(max=2)].double().t() * (r < R - 1)
            size = x[r].double().abs() @ w[e[r].clamp(max=2)].double().abs().t()
            close("y", y[r], row, BF * row.abs() + K * 2.0 ** -23 * size)
        assert not y[R - 1:].any()
        dy = torch.randn(64, N, device=DEV).bfloat16().repeat(R // 64, 1)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        # rows repeat with period 64: the large group's sum is that of its rows by period
        times = torch.bincount(torch.arange(3, R - 5, device=DEV) % 64, minlength=64).double()
        base, dbase = x[:64].double(), dy[:64].double()
        want = (dbase * times[:, None]).t() @ base
        size = (dbase.abs() * times[:, None]).t() @ base.abs()
        close("dw", dw[1], want, BF * want.abs() + R * 2.0 ** -23 * size)
        r = R - 6
        want = dy[r].double() @ w[1].double()
        close("dx", dx[r], want, BF * want.abs() + N * 2.0 ** -23 * (dy[r].double().abs() @ w[1].double().abs()))


def make_stack(E, d, ffn, seed=0):
    torch.manual_seed(seed)
    stack = ExpertStack(E, d, ffn).to(DEV)
    stack.init_gpu_state()
    return stack


class TestRaggedFFN:
    @pytest.mark.parametrize("counts", [[5, 0, 130, 64], [0, 1, 0, 0], [300, 300, 1, 2], [3000, 0, 9000, 1],
                                        [20000, 18000, 0, 300]])
    def test_against_double(self, counts):
        stack = make_stack(4, 128, 512 if sum(counts) > 30000 else 256)
        offsets = offsets_of(counts)
        R = sum(counts) + 3
        x = torch.randn(R, 128, device=DEV).bfloat16().requires_grad_(True)
        dy = torch.randn(R, 128, device=DEV).bfloat16()
        y = Fops.ragged_ffn(x, offsets, stack)
        y.backward(dy)
        W = [t.detach().double().requires_grad_(True)
             for t in (stack.W1c, stack.b1_f32, stack.W2c, stack.b2_f32)]
        xd = x.detach().double().requires_grad_(True)
        at = offsets.tolist()
        parts = []
        for e in range(4):
            h = F.gelu(xd[at[e]:at[e + 1]] @ W[0][e].t() + W[1][e], approximate="tanh")
            parts.append(h @ W[2][e].t() + W[3][e])
        want = torch.cat(parts)
        want.backward(dy[: at[-1]].double())
        # the largest value's share: four roundings to bf16 on a path (h, dh twice,
        # the result), each 2^-8, over sums whose terms are no larger in all than
        # sqrt(256) of their sum's usual size
        for name, got, ref in (("y", y[: at[-1]], want), ("dx", x.grad, xd.grad), ("W1", stack.main_grad_W1, W[0].grad),
                               ("b1", stack.main_grad_b1, W[1].grad), ("W2", stack.main_grad_W2, W[2].grad),
                               ("b2", stack.main_grad_b2, W[3].grad)):
            if ref.numel():
                assert (got.double() - ref).abs().max() <= 4 * BF * 16 ** 0.5 * ref.abs().max() + 1e-6, name
        first = stack.main_grad_W1.clone()
        assert stack.grad_ready
        Fops.ragged_ffn(x, offsets, stack).backward(dy)  # further backwards of a step add
        assert torch.allclose(stack.main_grad_W1, 2 * first, rtol=1e-6, atol=1e-7)
        with torch.no_grad():
            assert torch.equal(Fops.ragged_ffn(x, offsets, stack), y)

    def test_refuses_fused_backward(self):
        torch.manual_seed(0)
        stack = ExpertStack(2, 256, 256).to(DEV)
        stack.init_gpu_state(master_weights=False)
        FusedExpertSGD(stack, stochastic_rounding=True, fused_backward=True)
        x = torch.randn(4, 256, device=DEV).bfloat16().requires_grad_(True)
        with pytest.raises(RuntimeError, match="fused_backward"):
            Fops.ragged_ffn(x, offsets_of([2, 2]), stack)


def make_moe(dropless, E=8, k=2, d=128, ffn=256, factor=8.0):
    torch.manual_seed(5)
    moe = ExpertParallelMoE(d, ffn, E, k=k, capacity_factor=factor, dropless=dropless).to(DEV).bfloat16()
    moe.experts.float()
    moe.experts.init_gpu_state()
    return moe


class TestDroplessMoE:
    @pytest.mark.parametrize("T", [1, 7, 300])
    def test_same_as_roomy_capacity(self, T):
        """With room for every slot the two layouts compute the same layer."""
        x = torch.randn(T, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(T)).bfloat16()
        out = []
        for dropless in (False, True):
            moe = make_moe(dropless).eval()
            leaf = x.clone().requires_grad_(True)
            y = moe(leaf)
            (y.float() * torch.arange(128, device=DEV) / 128).sum().backward()
            st = moe.experts
            out.append((y, leaf.grad, moe.gate.weight.grad, st.main_grad_W1, st.main_grad_W2, st.main_grad_b1,
                        st.main_grad_b2, moe.aux_loss, moe.last_counts))
        for i, (a, b) in enumerate(zip(*out)):
            # the same roundings at the same places; sums in another order: a few bf16 steps of the largest
            assert (a.double() - b.double()).abs().max() <= 6 * BF * a.double().abs().max() + 1e-6, i

    def test_every_slot_counts(self):
        """All tokens to one expert: capacity would drop most, here none is."""
        moe = make_moe(True, factor=1.0).eval()
        with torch.no_grad():
            moe.gate.weight.zero_()  # equal logits: ties go to the lowest experts
        x = torch.randn(500, 128, device=DEV).bfloat16()
        with torch.no_grad():
            y = moe(x)
        assert moe.last_counts.sum() == 1000
        w = moe.experts
        want = 0
        chosen = moe.last_counts.nonzero().flatten().tolist()
        assert len(chosen) == 2
        for e in chosen:
            h = F.gelu(x.float() @ w.W1c[e].float().t() + w.b1_f32[e], approximate="tanh")
            want = want + 0.5 * (h @ w.W2c[e].float().t() + w.b2_f32[e])
        assert (y.float() - want).abs().max() <= 6 * BF * want.abs().max()

    def test_training_step_end_to_end(self):
        """Layout, products, combine, norm, clipped steps: as a training step runs them."""
        from learning_at_home_amd.optim import MasterSGD

        cfg = TransformerDMoEConfig(vocab_size=512, d_model=128, n_heads=2, n_layers=2, seq_len=64,
                                    num_experts=8, k_best=2, ffn_dim=256)
        torch.manual_seed(0)
        model = TransformerDMoE(cfg, lambda i, c: ExpertParallelMoE(
            c.d_model, c.ffn_dim, c.num_experts, k=c.k_best, dropless=True)).to(DEV).bfloat16()
        opts = []
        for block in model.blocks:
            block.moe.experts.float()
            block.moe.experts.init_gpu_state()
            opts.append(FusedExpertSGD(block.moe.experts, lr=0.1))
        trunk = MasterSGD([p for n, p in model.named_parameters() if ".moe.experts." not in n], lr=0.1)
        ids = torch.randint(0, 512, (4, 65), device=DEV)
        loss = model.loss(ids[:, :-1], ids[:, 1:], fused_ce=True)
        loss.backward()
        grads = trunk.gradients() + [g for o in opts for g in o.gradients()]
        assert len(grads) == len(trunk.params) + 8
        norm, scale = Fops.grad_clip_scale(grads, 1e-2)
        want = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
        assert (norm.double() - want).abs() <= 2.0 ** -20 * want
        before = opts[0].stack.W1.detach().clone()
        g = opts[0].stack.main_grad_W1.clone()
        master, mg = trunk.masters[0].clone(), trunk.params[0].grad.clone()
        for o in opts:
            o.step(grad_scale=scale)
        trunk.step(grad_scale=scale)
        assert torch.allclose(opts[0].stack.W1, before - 0.1 * g * scale, rtol=2e-7, atol=1e-9)
        assert torch.allclose(trunk.masters[0], master - 0.1 * mg.float() * scale, rtol=2e-7, atol=1e-9)
        assert torch.equal(trunk.params[0], trunk.masters[0].bfloat16())

    def test_graph_decode(self):
        cfg = TransformerDMoEConfig(vocab_size=512, d_model=128, n_heads=2, n_layers=2, seq_len=64,
                                    num_experts=8, k_best=2, ffn_dim=256)
        torch.manual_seed(0)
        model = TransformerDMoE(cfg, lambda i, c: ExpertParallelMoE(
            c.d_model, c.ffn_dim, c.num_experts, k=c.k_best, dropless=True)).to(DEV).bfloat16().eval()
        for block in model.blocks:
            block.moe.experts.float()
            block.moe.experts.init_gpu_state()
        prompt = torch.randint(0, 512, (3, 9), device=DEV)
        eager = GraphDecoder(model, batch_size=3, use_graph=False).generate(prompt, 20)
        graph = GraphDecoder(model, batch_size=3, use_graph=True).generate(prompt, 20)
        assert torch.equal(eager, graph)
