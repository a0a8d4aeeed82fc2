"""Teach a fly actor's memory over decisions from recorded stretches, then play it moment by moment.

    python -m flyguy_amd.remember --data GAME.bin [MORE.bin ...] --graph GRAPH.npz [--start CKPT.pt] [--hops 3]
        [--teacher T.pt] [--stretch 256] [--cars 16] [--steps 500] [--lr 1e-3] [--temp 0.5] [--heads 8] [--dim 64]
        [--rule decay|delta] [--norm] [--dropout 0] [--out runs/remember/memory.pt] [--device cuda] [--kernel hip|torch] [--seed 0]

DATA: FLYD files or FLYR recordings of the bot as flyguy_amd.teach reads them, their moments in the order they were played;
the answers are those in the files, or a fly-actor --teacher's.  The actor itself (--start, or a fresh one) stays as it is:
what is taught are the memory's projections, norms and read-out (MemoryActor), by KL(teacher || student) over whole
stretches.  Memory and actor are written out together; flyguy_amd.memory.MemoryActor.load reads them.  At the end a stretch is
played moment by moment from an empty memory, and compared with the stretch read at once.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import numpy as np
import torch

from .fly import FlyActor
from .memory import MemoryActor
from .teach import _actor_weights, kl_to, moments


def _actor(graph: str, checkpoint: Path | None, hops: int, kernel: str) -> FlyActor:
    ck = {} if checkpoint is None else torch.load(checkpoint, map_location="cpu", weights_only=True)
    cfg = (ck.get("config") or {}).get("model", {})
    f = FlyActor(graph, 517, 90, hops=int(cfg.get("fly_hops", hops)), fan=int(cfg.get("fly_fan", 16)))
    if ck:
        f.load_state_dict(_actor_weights(ck), strict=False)
    f.kernel = kernel
    return f.requires_grad_(False)


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--data", nargs="+", type=Path, required=True)
    ap.add_argument("--graph", required=True)
    ap.add_argument("--start", type=Path, default=None)
    ap.add_argument("--teacher", type=Path, default=None)
    ap.add_argument("--hops", type=int, default=3, help="hops of an actor whose checkpoint does not say")
    ap.add_argument("--stretch", type=int, default=256)
    ap.add_argument("--cars", type=int, default=16, help="stretches per step")
    ap.add_argument("--steps", type=int, default=500)
    ap.add_argument("--lr", type=float, default=1e-3)
    ap.add_argument("--temp", type=float, default=0.5)
    ap.add_argument("--heads", type=int, default=8)
    ap.add_argument("--dim", type=int, default=64)
    ap.add_argument("--rule", default="decay", choices=["decay", "delta"], help="a memory that adds, or one that corrects")
    ap.add_argument("--norm", action="store_true", help="a layer norm of the firing before the memory")
    ap.add_argument("--dropout", type=float, default=0.0, help="the share of the memory's read-out dropped while teaching")
    ap.add_argument("--out", type=Path, default=Path("runs") / "remember" / "memory.pt")
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--kernel", default="hip", choices=["hip", "torch"])
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args(argv)
    if min(args.steps, args.cars, args.stretch) < 1:
        raise SystemExit("--steps, --cars and --stretch are at least 1")
    if not 0 <= args.dropout <= 1:
        raise SystemExit("--dropout is a share from 0 to 1")
    dev = torch.device(args.device)
    torch.manual_seed(args.seed)
    rng = np.random.default_rng(args.seed)

    games = [moments(p) for p in args.data]
    if args.teacher is None and any(a is None for _, a in games):
        raise SystemExit("no teacher's answers in a file and no --teacher")
    games = [(o, a) for o, a in games if len(o) >= args.stretch]
    if not games:
        raise SystemExit(f"no file holds {args.stretch} moments")
    teacher = None if args.teacher is None else _actor(args.graph, args.teacher, args.hops, args.kernel).to(dev)
    net = MemoryActor(_actor(args.graph, args.start, args.hops, args.kernel), heads=args.heads, dim=args.dim,
                      positions=max(args.stretch, 65536), rule=args.rule, norm=args.norm, dropout=args.dropout).to(dev)
    learns = [p for p in net.parameters() if p.requires_grad]
    opt = torch.optim.Adam(learns, lr=args.lr)

    def draw():
        """(observations, the teacher's probabilities) of `cars` stretches, their games and places drawn at random."""
        obs, ans = [], []
        for i in rng.integers(0, len(games), args.cars):
            o, a = games[i]
            b = int(rng.integers(0, len(o) - args.stretch + 1))
            obs.append(torch.from_numpy(np.array(o[b:b + args.stretch], np.float32)))
            if teacher is None:
                ans.append(torch.from_numpy(np.array(a[b:b + args.stretch], np.float32)))
        x = torch.stack(obs).to(dev)
        with torch.no_grad():
            t = torch.stack(ans).to(dev) if teacher is None else teacher(x.flatten(0, 1)).unflatten(0, x.shape[:2])
            return x, torch.softmax(t / args.temp, -1)

    began, first = time.time(), None
    for step in range(1, args.steps + 1):
        x, target = draw()
        loss = kl_to(target, net(x)[0]).mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        if step % 50 == 0 or step in (1, args.steps):
            now = float(loss.detach())
            first = now if first is None else first
            print(f"step {step:,} | KL {now:.4f} | {step * x.shape[0] * x.shape[1] / (time.time() - began):,.0f} moments/s",
                  flush=True)
    args.out.parent.mkdir(parents=True, exist_ok=True)
    torch.save({**net.checkpoint(args.graph), "taught_steps": args.steps}, args.out)

    x, _ = draw()
    net.eval()                                # (nothing is dropped in play)
    with torch.no_grad():
        at_once, _ = net(x)
        live = net.state(x.shape[0])
        played = torch.stack([net.step(x[:, t], live) for t in range(x.shape[1])], 1)
    off = float((played - at_once).abs().max() / at_once.abs().max().clamp_min(1e-30))
    same = float((played.argmax(-1) == at_once.argmax(-1)).float().mean())
    print(f"{args.out}: KL {first:.4f} -> {now:.4f}; played moment by moment: logits off by {off:.1e} of the largest, first "
          f"choice the same in {same:.4f} of moments")
    return 0


if __name__ == "__main__":
    sys.exit(main())
