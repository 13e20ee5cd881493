"""A whole mixture-of-experts layer for a few tokens (``ops.moe_decode``) against the expert loop.

    python benchmarks/moe_decode.py [--tokens 1,8,32,64] [--iters 20]

Shapes: a Mixtral-8x22B-shape layer (8 experts of 6144 x 16384, top-2) and a layer of many small
experts (64 of 2048 x 1024, top-6), random-init bf16. For each token count: device time of the one call
(CUDA-event medians; L2 flushed by reading 256 MB), of ``MixtralLayer.moe_single`` (per-expert gather,
fused GEMMs, scatter-add, with its host synchronisations: wall clock), and the time of the bytes of
the experts that the tokens chose at the measured copy bandwidth (a stream of reads alone can be faster
than a copy: no floor).
"""

from __future__ import annotations

import argparse
import json
import os
import statistics as st
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "benchmarks")]

from decode import hbm_gbs, timed  # noqa: E402

SHAPES = {"mixtral8x22b": (6144, 16384, 8, 2), "small_experts": (2048, 1024, 64, 6)}


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--shapes", default=",".join(SHAPES))
    ap.add_argument("--tokens", default="1,8,32,64")
    ap.add_argument("--iters", type=int, default=20)
    a = ap.parse_args()
    from flextensor_b200 import ops
    from flextensor_b200.models.mixtral import MixtralLayer, tiny_mixtral
    from flextensor_b200.ops import native
    from flextensor_b200.parallel.ep import route_topk

    dev = torch.device("cuda", 0)
    flush = torch.ones(256 << 20, dtype=torch.uint8, device=dev)
    for name in a.shapes.split(","):
        D, F, E, topk = SHAPES[name]
        with torch.device(dev):
            layer = MixtralLayer(tiny_mixtral(dim=D, n_heads=D // 128, n_kv_heads=1, ffn_dim=F, n_experts=E, topk=topk))
        layer = layer.to(torch.bfloat16).requires_grad_(False)
        for p in layer.parameters():
            p.normal_(0.0, 0.02)
        gu, dn = [e.w_gate_up for e in layer.experts], [e.w_down for e in layer.experts]
        for T in (int(t) for t in a.tokens.split(",")):
            torch.manual_seed(T)
            h, x = (torch.randn(T, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
            ids, wts = route_topk(h, layer.router, topk)
            at_copy = ids.unique().numel() * 6 * D * F / (hbm_gbs() * 1e3)
            t = timed(lambda: ops.moe_decode(h, layer.router, gu, dn, topk, residual=x), a.iters, flush)
            loop = []
            for _ in range(3 + a.iters):
                torch.cuda.synchronize()
                t0 = time.perf_counter()
                layer.moe_single(h, *route_topk(h, layer.router, topk), x.clone(), "fused")
                torch.cuda.synchronize()
                loop.append((time.perf_counter() - t0) * 1e6)
            assert native.device_error(reset=True) == 0
            print(json.dumps({"shape": name, "tokens": T, "experts": ids.unique().numel(), "at_copy_rate_us": round(at_copy, 1),
                              "moe_decode_us": round(t, 1), "x_copy_rate": round(t / at_copy, 2),
                              "expert_loop_us": round(st.median(loop[3:]), 1)}))


if __name__ == "__main__":
    main()
