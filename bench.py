#!/usr/bin/env python3
"""Flagship benchmark: training tokens/sec of Transformer-DMoE 256-expert on
1..8 MI355X GPUs (BASELINE.json headline metric, config #2).

One process per GPU over RCCL; expert-parallel MoE FFN layers (RCCL
all-to-all dispatch, CDNA4 HIP kernels) + data-parallel trunk with
asynchronous SGD and periodic Moshpit-style averaging (RcclAverager on a
side stream) — the reference's no-global-barrier training semantics.

Contract (round driver): `python bench.py --gpus N --steps K --warmup W`;
for N>1 launched via torch.distributed.run. Rank 0 prints ONE JSON line.
Synthetic data (no network), random-init weights, bf16 compute.
"""
import argparse
import json
import os
import time

import torch
import torch.distributed as dist

from learning_at_home_amd.models import TransformerDMoE, TransformerDMoEConfig
from learning_at_home_amd.parallel import ExpertParallelMoE, FusedExpertSGD
from learning_at_home_amd.averaging import RcclAverager
from learning_at_home_amd.ops import HAS_HIP
from learning_at_home_amd.ops.functional import clip_grad_norm_, grad_clip_scale
from learning_at_home_amd.optim import MasterSGD


def build_model(cfg: TransformerDMoEConfig, args, device, group=None):
    world = dist.get_world_size() if dist.is_initialized() else 1
    # "auto": overlap the a2a with expert compute at N>1 (4 chunks), no
    # chunking at N=1 where there is no collective to hide
    chunks = (4 if world > 1 else 1) if args.a2a_chunks == 0 else args.a2a_chunks

    def moe_factory(layer_idx, c):
        return ExpertParallelMoE(
            d_model=c.d_model, ffn_dim=c.ffn_dim, num_experts=c.num_experts,
            k=c.k_best, capacity_factor=args.capacity_factor,
            aux_loss_coef=args.aux_coef, group=group,
            a2a_chunks=1 if args.dropless else chunks, dropless=args.dropless,
        )

    model = TransformerDMoE(cfg, moe_factory)
    if device.type == "cuda":
        model = model.to(device=device, dtype=torch.bfloat16)
        for block in model.blocks:
            block.moe.experts.float()
            block.moe.experts.init_gpu_state(master_weights=args.master_weights)
    else:
        model = model.to(device)
    return model


def main():
    # DHT peers are mp.Processes; fork after HIP init is unsafe on ROCm, and
    # set_device precedes DHT creation in the multi-GPU path -> use spawn
    import multiprocessing as _mp

    try:
        _mp.set_start_method("spawn", force=True)
    except RuntimeError:
        pass

    p = argparse.ArgumentParser()
    p.add_argument("--gpus", type=int, default=1)
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--warmup", type=int, default=5)
    p.add_argument("--d-model", type=int, default=1024)
    p.add_argument("--ffn-dim", type=int, default=4096)
    p.add_argument("--layers", type=int, default=6)
    p.add_argument("--heads", type=int, default=16)
    p.add_argument("--experts", type=int, default=256)
    p.add_argument("--k", type=int, default=4)
    p.add_argument("--seq", type=int, default=1024)
    p.add_argument("--batch", type=int, default=96, help="per-GPU batch size")
    p.add_argument("--vocab", type=int, default=32000)
    p.add_argument("--capacity-factor", type=float, default=1.5)
    p.add_argument("--a2a-chunks", type=int, default=0,
                   help="0 = auto (4 at N>1 to overlap the dispatch/return "
                        "all-to-all with expert compute, 1 at N=1)")
    p.add_argument("--aux-coef", type=float, default=0.01)
    p.add_argument("--lr", type=float, default=0.01)
    p.add_argument("--averaging-period", type=int, default=10)
    p.add_argument("--no-averager", action="store_true")
    p.add_argument("--fixed-batch", action="store_true",
                   help="reuse ONE synthetic batch every step (memorization "
                        "sanity check: loss must fall; NOT a valid bench mode)")
    p.add_argument("--master-weights", action="store_true",
                   help="fp32 master weights for experts (default: bf16 + "
                        "stochastic-rounding SGD, the fast path)")
    p.add_argument("--metrics", action="store_true",
                   help="print per-stage timers + expert-load stats to stderr")
    p.add_argument("--fused-ce", dest="fused_ce", action="store_true", default=True,
                   help="chunked fused linear+cross-entropy (default ON since "
                        "round 2: the ce.hip online-lse kernels make it +2%% "
                        "tokens/s AND it never materializes the [T, vocab] "
                        "logits, -46 GB at the flagship config)")
    p.add_argument("--no-fused-ce", dest="fused_ce", action="store_false")
    p.add_argument("--loss-every", type=int, default=0,
                   help="if >0, rank 0 prints the step loss to stderr every N "
                        "timed steps (long-horizon stability monitoring)")
    p.add_argument("--dropless", action="store_true",
                   help="experts without capacity: rows sorted by expert, ragged "
                        "products, nothing dropped (default: capacity buffers)")
    p.add_argument("--clip-norm", type=float, default=0.0,
                   help="if >0, bound the norm of all gradients together (trunk and "
                        "expert shards of this rank) to this; scaled on the GPU")
    p.add_argument("--no-dht", action="store_true",
                   help="skip the per-rank Kademlia DHT peer + expert announce "
                        "(north-star parity: each GPU rank hosts a shard AND a "
                        "DHT peer with liveness-leased expert uids)")
    args = p.parse_args()

    world_size = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local_rank = int(os.environ.get("LOCAL_RANK", "0"))
    use_cuda = torch.cuda.is_available()

    if world_size > 1:
        backend = "nccl" if use_cuda else "gloo"
        if use_cuda:
            torch.cuda.set_device(local_rank)
        dist.init_process_group(backend, rank=rank, world_size=world_size)
    device = torch.device(f"cuda:{local_rank}" if use_cuda else "cpu")

    if use_cuda:
        cfg = TransformerDMoEConfig(
            vocab_size=args.vocab, d_model=args.d_model, n_heads=args.heads,
            n_layers=args.layers, seq_len=args.seq, num_experts=args.experts,
            k_best=args.k, ffn_dim=args.ffn_dim,
        )
        B = args.batch
    else:  # CPU smoke fallback: tiny config so plain `python bench.py` runs anywhere
        cfg = TransformerDMoEConfig(
            vocab_size=1024, d_model=128, n_heads=4, n_layers=2, seq_len=64,
            num_experts=8, k_best=2, ffn_dim=256,
        )
        B = 2

    # per-rank DHT peer: announce this rank's expert shard under liveness
    # leases (discovery/elasticity control plane; fail-soft for the bench)
    dht = None
    if not args.no_dht:
        try:
            from learning_at_home_amd import DHT
            import threading

            if world_size > 1:
                seed_ep = [None]
                if rank == 0:
                    seed = DHT(start=True)
                    seed_ep = [list(seed.endpoint)]
                dist.broadcast_object_list(seed_ep, src=0)
                peers = [tuple(seed_ep[0])] if rank != 0 else []
                dht = seed if rank == 0 else DHT(initial_peers=peers, start=True)
            else:
                dht = DHT(start=True)
            n_local = cfg.num_experts // world_size
            uids = [f"bench_expert.{rank * n_local + i}.{layer}"
                    for i in range(n_local) for layer in range(cfg.n_layers)]
            dht.declare_experts(uids, "127.0.0.1", 40000 + rank, expiration=60.0)

            def announce_loop():
                import random as _r
                import time as _t

                while True:
                    _t.sleep(20.0 + _r.random() * 2.0)  # de-sync rank bursts
                    try:
                        dht.declare_experts(uids, "127.0.0.1", 40000 + rank, expiration=60.0)
                    except Exception:  # noqa: BLE001
                        return

            threading.Thread(target=announce_loop, daemon=True).start()
        except Exception as e:  # noqa: BLE001
            print(f"[bench] DHT control plane disabled: {e!r}")
            dht = None

    torch.manual_seed(1234 + rank)
    model = build_model(cfg, args, device)

    # optimizers: fused async SGD per expert stack; plain SGD for the trunk
    expert_opts = []
    trunk_params = []
    for name, param in model.named_parameters():
        if ".moe.experts." not in name:
            trunk_params.append(param)
    opt_stream = torch.cuda.Stream(device=device) if use_cuda else None
    for block in model.blocks:
        if device.type == "cuda" and HAS_HIP:
            opt = FusedExpertSGD(block.moe.experts, lr=args.lr,
                                 stochastic_rounding=not args.master_weights)
            # overlap the expert update with the NEXT step's forward: layer
            # L's weights aren't read again until layer L's MoE runs
            opt.set_side_stream(opt_stream)
            expert_opts.append(opt)
        else:
            expert_opts.append(torch.optim.SGD(block.moe.experts.parameters(), lr=args.lr))
    # trunk in bf16 needs fp32 masters: plain SGD on bf16 loses sub-ulp updates
    trunk_opt = (MasterSGD(trunk_params, lr=args.lr) if use_cuda
                 else torch.optim.SGD(trunk_params, lr=args.lr))

    averager = None
    if world_size > 1 and not args.no_averager:
        averager = RcclAverager(trunk_params, dtype=torch.float32 if device.type != "cuda" else torch.bfloat16)

    tokens_per_step_per_rank = B * cfg.seq_len

    fixed = None
    if args.fixed_batch:
        fixed = torch.randint(0, cfg.vocab_size, (B, cfg.seq_len + 1), device=device)

    def make_batch():
        ids = fixed if fixed is not None else torch.randint(
            0, cfg.vocab_size, (B, cfg.seq_len + 1), device=device)
        return ids[:, :-1], ids[:, 1:]

    from learning_at_home_amd.utils.monitor import StageTimers, expert_load_stats

    timers = StageTimers() if args.metrics else None
    if timers is not None:  # per-stage MoE observability on the first layer
        model.blocks[0].moe.stage_timers = timers

    def train_step(step_idx):
        from contextlib import nullcontext

        tm = timers if timers is not None else (lambda s: nullcontext())
        inputs, labels = make_batch()
        with tm("forward"):
            loss = model.loss(inputs, labels, fused_ce=args.fused_ce)
        trunk_opt.zero_grad(set_to_none=True)
        with tm("backward"):
            loss.backward()
        scale = None
        if args.clip_norm > 0 and use_cuda:
            grads = trunk_opt.gradients() + [g for opt in expert_opts for g in opt.gradients()]
            scale = grad_clip_scale(grads, args.clip_norm)[1]
        elif args.clip_norm > 0:  # plain optimizers take no scale: the gradients themselves
            clip_grad_norm_([p.grad for p in model.parameters() if p.grad is not None], args.clip_norm)
        scaled = {} if scale is None else {"grad_scale": scale}
        with tm("expert_opt"):
            for opt in expert_opts:
                opt.step(**scaled)  # async per-shard SGD (fused on GPU)
                if isinstance(opt, torch.optim.SGD):
                    opt.zero_grad(set_to_none=True)
        if averager is not None:
            averager.wait()  # previous round must have landed before we step
            if getattr(averager, "_round_pending", False):
                averager._round_pending = False
                if isinstance(trunk_opt, MasterSGD):
                    trunk_opt.sync_masters_from_params()  # averaged values win
        with tm("trunk_opt"):
            trunk_opt.step(**scaled)
        if averager is not None and (step_idx + 1) % args.averaging_period == 0:
            averager.step(async_op=True)  # overlapped on the side stream
            averager._round_pending = True
        return loss

    def barrier_sync():
        if world_size > 1:
            dist.barrier()
        if use_cuda:
            torch.cuda.synchronize()

    for i in range(args.warmup):
        train_step(i)
    barrier_sync()
    t0 = time.perf_counter()
    last_loss = None
    for i in range(args.steps):
        last_loss = train_step(args.warmup + i).detach()
        if args.loss_every and rank == 0 and (i % args.loss_every == 0 or i == args.steps - 1):
            import sys as _sys

            print(f"[loss] step {i}: {float(last_loss):.4f}", file=_sys.stderr)
    barrier_sync()
    elapsed = time.perf_counter() - t0

    # max over ranks = the slowest rank defines the job's wall time
    if world_size > 1:
        t = torch.tensor([elapsed], device=device if use_cuda else "cpu",
                         dtype=torch.float64 if not use_cuda else torch.float32)
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        elapsed = float(t.item())

    ms_per_step = elapsed / args.steps * 1000.0
    total_tokens_per_s = tokens_per_step_per_rank * world_size * args.steps / elapsed

    # truthful labels: only claim dp/averager when one ran
    par = f"ep{world_size}"
    if averager is not None:
        par += f"+dp{world_size} (async SGD, RCCL averager every {args.averaging_period})"
    else:
        par += " (async expert SGD)"

    # capacity-drop observability: fraction of routed
    # (token, expert) assignments dropped by the capacity clamp, last step
    drop_fracs = []
    for block in model.blocks:
        c = block.moe.last_counts
        if c is not None and args.dropless:
            drop_fracs.append(0.0)
        elif c is not None:
            cap = block.moe.capacity(tokens_per_step_per_rank)
            total = float(c.sum().item())
            kept = float(c.clamp(max=cap).sum().item())
            if total > 0:
                drop_fracs.append((total - kept) / total)
    dropped_frac = round(sum(drop_fracs) / len(drop_fracs), 4) if drop_fracs else None

    if rank == 0:
        print(json.dumps({
            "metric": "training tokens/sec, Transformer-DMoE 256-expert",
            "value": round(total_tokens_per_s, 1),
            "unit": "tokens/s",
            "n_gpus": world_size,
            "steps": args.steps,
            "warmup": args.warmup,
            "ms_per_step": round(ms_per_step, 2),
            "higher_is_better": True,
            "scaling": "weak",
            "vs_baseline": None,
            "dtype": "bf16" if use_cuda else "fp32",
            "data": "synthetic (random tokens, random-init weights)",
            "config": {
                "model": f"Transformer-DMoE d{cfg.d_model} L{cfg.n_layers} "
                         f"E{cfg.num_experts} top{cfg.k_best} ffn{cfg.ffn_dim}",
                "global_batch": B * world_size,
                "seq_len": cfg.seq_len,
                "parallelism": par,
                "capacity_factor": None if args.dropless else args.capacity_factor,
                **({"clip_norm": args.clip_norm} if args.clip_norm > 0 else {}),
                "dropped_token_frac": dropped_frac,
                "last_loss": round(float(last_loss), 4) if last_loss is not None else None,
            },
        }))

    if args.metrics and rank == 0:
        import sys

        print("[metrics] stages:", timers.report(), file=sys.stderr)
        from learning_at_home_amd.utils.monitor import amd_smi_snapshot

        if use_cuda:
            snap = amd_smi_snapshot()
            print("[metrics] smi keys:", sorted(snap.keys()), file=sys.stderr)
        counts = model.blocks[0].moe.last_counts
        if counts is not None:
            cap = model.blocks[0].moe.capacity(tokens_per_step_per_rank)
            print("[metrics] expert load (layer 0):",
                  json.dumps(expert_load_stats(counts.cpu(), cap)), file=sys.stderr)

    if dht is not None:
        dht.shutdown()
    if world_size > 1:
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
