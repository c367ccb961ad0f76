"""One MoE layer with a scored router, served with 4-bit weights:
sigmoid scores with a balance bias, 8 expert groups of which 4 are on offer,
top-8, and a shared expert of another width than the routed ones.

    python examples/w4_scored_layer.py [--tokens 64]
"""

from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from extend_nano_vllm_b200 import ExpertParallelMoE  # noqa: E402


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--tokens", type=int, default=64)
    tokens = parser.parse_args().tokens
    hidden, inter, experts, top_k = 2048, 768, 128, 8
    layer = ExpertParallelMoE(hidden, inter, experts, top_k, norm_topk_prob=True,
                              shared_expert_intermediate_size=1024)
    layer = layer.to(device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0.0, 0.02)
    layer.set_scored_routing("sigmoid", bias=torch.randn(experts) * 0.05, num_groups=8,
                             topk_groups=4, group_score="top2", scale=2.5)
    x = torch.randn(tokens, hidden, device="cuda", dtype=torch.bfloat16)

    def timed() -> tuple[torch.Tensor, float]:
        for _ in range(3):
            out = layer(x)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        for _ in range(20):
            out = layer(x)
        end.record()
        torch.cuda.synchronize()
        return out, start.elapsed_time(end) / 20 * 1e3

    with torch.no_grad():
        full, t_full = timed()
        size = layer.expert_parameter_bytes
        layer.quantize_w4(group=128)
        out, t_w4 = timed()
    off = float((out.float() - full.float()).norm() / full.float().norm())
    print(f"{tokens} tokens: bf16 experts {size / 1e6:.0f} MB, {t_full:.1f} us; "
          f"4-bit {layer.expert_parameter_bytes / 1e6:.0f} MB, {t_w4:.1f} us; "
          f"outputs differ by {off:.3f} (rounding the weights to 4 bits)")


if __name__ == "__main__":
    main()
