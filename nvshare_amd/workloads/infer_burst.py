"""Bursty inference job (BASELINE.json config #5: Jupyter-style pods).

Alternates short inference bursts with idle think-time, the pattern
nvshare's early-release path is built for: during think-time the client
voluntarily releases the GPU lock so other pods run.

--model session holds a paged key/value cache over its think-time: each
burst is a turn of --batch sessions, a chunk of --prompt new tokens and then
--infers-per-burst single ones, and the cache has to come back from each
pause bit for bit.
"""

from __future__ import annotations

import argparse
import time

from nvshare_amd.workloads.common import Timer, add_common_args, emit, sync


def main(argv: list[str] | None = None) -> None:
    ap = argparse.ArgumentParser()
    add_common_args(ap)
    ap.add_argument("--model", default="resnet50")
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--image", type=int, default=224)
    ap.add_argument("--bursts", type=int, default=5)
    ap.add_argument("--infers-per-burst", type=int, default=20)
    ap.add_argument("--think-s", type=float, default=2.0)
    ap.add_argument("--prompt", type=int, default=256,
                    help="new tokens of a session's turn")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--head-dim", type=int, default=128)
    ap.add_argument("--page", type=int, default=64,
                    help="tokens in a page of the cache")
    ap.add_argument("--cache", default="same", choices=["same", "e4m3"],
                    help="type of the cache: the model's, or 8 bits")
    ap.add_argument("--dtype", default="bfloat16",
                    choices=["bfloat16", "float16"],
                    help="type of the session model")
    args = ap.parse_args(argv)
    if args.model == "session":
        run_sessions(args)
        return

    import torch

    from nvshare_amd.workloads.train_resnet import build

    dev = torch.device(args.device)
    model = build(args.model, 1000).to(dev).eval()
    x = torch.randn(args.batch, 3, args.image, args.image, device=dev)

    infers = 0
    with Timer() as t:
        with torch.no_grad():
            for _ in range(args.bursts):
                for _ in range(args.infers_per_burst):
                    model(x)
                    infers += 1
                sync(args.device)
                time.sleep(args.think_s)
    emit({
        "workload": "infer_burst", "label": args.label,
        "seconds": t.seconds, "bursts": args.bursts, "infers": infers,
        "batch": args.batch, "device": args.device,
        "infers_per_s": infers / t.seconds,
    })


def run_sessions(args: argparse.Namespace) -> None:
    from nvshare_amd.workloads.common import die
    from nvshare_amd.workloads.session import Sessions

    for name, least in (("batch", 1), ("bursts", 1), ("prompt", 1),
                        ("layers", 1), ("page", 1), ("heads", 1),
                        ("kv_heads", 1), ("infers_per_burst", 0),
                        ("think_s", 0)):
        if not getattr(args, name) >= least:
            die(f"session: --{name.replace('_', '-')} "
                f"{getattr(args, name)} is less than {least}")
    if args.heads % args.kv_heads:
        die(f"session: --heads {args.heads} is no multiple of --kv-heads "
            f"{args.kv_heads}")
    if args.head_dim not in (64, 128, 256):
        die(f"session: --head-dim {args.head_dim} is not one of 64, 128 and "
            "256")
    turn = args.prompt + args.infers_per_burst
    model = Sessions(args.batch, args.bursts * turn, args.layers, args.heads,
                     args.kv_heads, args.head_dim, args.page, args.cache,
                     args.dtype, args.device)
    infers = 0
    with Timer() as t:
        for _ in range(args.bursts):
            model.step(args.prompt)
            for _ in range(args.infers_per_burst):
                model.step(1)
            infers += 1 + args.infers_per_burst
            sync(args.device)
            before = model.fingerprint()
            time.sleep(args.think_s)
            if model.fingerprint() != before:
                die("session: the cache changed over a pause")
    off = model.check()
    emit({
        "workload": "infer_burst", "label": args.label,
        "seconds": t.seconds, "bursts": args.bursts, "infers": infers,
        "batch": args.batch, "device": args.device,
        "infers_per_s": infers / t.seconds,
        "tokens": args.batch * model.tokens, "max_diff": off,
    })


if __name__ == "__main__":
    main()
