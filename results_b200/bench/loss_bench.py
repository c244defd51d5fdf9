"""Vocabulary losses bench: a training step (loss and gradient of the logits) of
each loss, and the log-probabilities alone, on the vocabularies of the package's
models.

    python -m results_b200.bench.loss_bench --rows 1,64,1024,4096 --dtype bfloat16 --csv out.csv

Time: CUDA events, median of --iters runs after --warmup; an L2-sized buffer is
written between runs whose logits fit L2. GB/s counts the logits read once and
the gradient written once. Logits are N(0, 2.5) from a fixed seed.
"""
from __future__ import annotations

import argparse

import torch

from ..models.shapes import glm4_9b_specs, qwen35_a3b_specs
from ..ops import losses
from ..utils import csvfmt
from .codec_bench import L2_FLUSH_BYTES, _time

HEADER = ["loss", "rows", "vocab", "dtype", "time_us", "gb_s"]


def vocabularies() -> list[int]:
    return [next(s.shape[0] for s in specs(layers=1) if s.name == "lm_head.weight")
            for specs in (glm4_9b_specs, qwen35_a3b_specs)]


def run(rows_list, vocabs, dtype, iters=10, warmup=3, top=64):
    out = []
    for vocab in vocabs:
        for rows in rows_list:
            rows += rows % 2  # the preference loss takes pairs
            g = torch.Generator(device="cuda").manual_seed(rows)
            x = torch.randn(rows, vocab, device="cuda", generator=g, dtype=dtype).mul_(2.5).requires_grad_(True)
            y = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
            ids = torch.randint(0, vocab, (rows, top), device="cuda", generator=g)
            teacher = torch.randn(rows, top, device="cuda", generator=g)
            with torch.no_grad():
                old = losses.token_logprobs(x, y)
            adv = torch.randn(rows, device="cuda", generator=g)
            steps = {
                "policy": lambda: losses.policy_loss(x, y, old, adv, ref_logp=old, kl_coef=0.05).loss,
                "preference": lambda: losses.preference_loss(x.view(2, rows // 2, vocab), y.view(2, -1)).loss,
                "distill": lambda: losses.distill_loss(x, ids, teacher).loss,
            }
            nbytes = x.numel() * x.element_size()
            flush = torch.empty(L2_FLUSH_BYTES, dtype=torch.uint8, device="cuda") if nbytes < (128 << 20) else None
            ms = {"logprobs": _time(lambda: losses.token_logprobs(x.detach(), y), iters, warmup, flush)}
            for name, f in steps.items():
                ms[name] = _time(lambda: torch.autograd.grad(f(), x), iters, warmup, flush)
            for name, t in ms.items():
                moved = nbytes * (1 if name == "logprobs" else 2)
                out.append({"loss": name, "rows": rows, "vocab": vocab, "dtype": str(dtype).replace("torch.", ""),
                            "time_us": round(t * 1e3, 1), "gb_s": round(moved / t / 1e6, 1)})
    return out


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rows", default="2,64,1024,4096")
    ap.add_argument("--vocab", default="", help="comma separated; default: the models' vocabularies")
    ap.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float16", "float32"])
    ap.add_argument("--top", type=int, default=64, help="teacher's entries a row")
    ap.add_argument("--iters", type=int, default=10)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--csv", default=None)
    a = ap.parse_args(argv)
    vocabs = [int(v) for v in a.vocab.split(",")] if a.vocab else vocabularies()
    rows = run([int(r) for r in a.rows.split(",")], vocabs, getattr(torch, a.dtype), a.iters, a.warmup, a.top)
    for r in rows:
        print(r, flush=True)
    if a.csv:
        csvfmt.write_rows(a.csv, HEADER, rows)
        csvfmt.write_sidecar(a.csv, {"bench": "loss", "dtype": a.dtype, "timing": "CUDA events, median of iters"})
    return rows


if __name__ == "__main__":
    main()
