"""Scored routing under expert parallelism: two gloo ranks on CPU, every dispatch
backend against the unsharded layer, with biases and expert groups that no softmax
top-k would give.  The kernels are the oracle's; the exchange logic is under test."""

import datetime
import multiprocessing as mp

import numpy as np
import pytest
import torch

from test_ep_gloo import COUNTS, SHAPE, _free_port, _layer, _tokens
from oracle.cpu_ops import CpuOps

ROUTING = dict(score="sigmoid", num_groups=4, topk_groups=2, group_score="max", scale=2.5)


class ScoredCpuOps(CpuOps):
    def route_scored_topk(self, logits, top_k, *, score, bias, num_groups, topk_groups,
                          group_score, renormalize, scale):
        assert score == "sigmoid" and group_score == "max" and renormalize
        s = torch.sigmoid(logits.double())
        by = (s + bias.double()).unflatten(-1, (num_groups, -1))
        first = by.amax(-1).sort(dim=-1, descending=True, stable=True).indices[:, :topk_groups]
        kept = torch.zeros(by.shape[:-1], dtype=torch.bool).scatter_(1, first, True)
        choice = by.masked_fill(~kept[..., None], -torch.inf).flatten(1)
        ids = choice.sort(dim=-1, descending=True, stable=True).indices[:, :top_k].contiguous()
        w = s.gather(1, ids)
        return (w / w.sum(-1, keepdim=True) * scale).bfloat16(), ids


def _scored(rank, world, backend, kw):
    layer = _layer(rank, world, backend, kw)
    # Not a constant: the experts' order of choice is not that of their scores.
    layer.set_scored_routing(bias=torch.linspace(0.3, -0.3, SHAPE["experts"]), **ROUTING)
    layer.to(torch.bfloat16)
    layer._ops = ScoredCpuOps()
    return layer


def _worker(rank, port, backend, kw, queue):
    import torch.distributed as dist
    from extend_nano_vllm_b200 import dist_env
    try:
        dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", world_size=2,
                                rank=rank, timeout=datetime.timedelta(seconds=60))
        own = backend in ("all_to_all_nvlink", "allgather_reduce", "allgather_reducescatter")
        dist_env.set_moe_token_counts(None if backend.startswith("all_to_all") and not own
                                      else COUNTS)
        tokens = (_tokens(rank) if own else _tokens(0) if backend.startswith("all_to_all")
                  else torch.cat([_tokens(0), _tokens(1)]))
        with torch.no_grad():
            out = _scored(rank, 2, backend, kw)(tokens)
        queue.put((rank, out.float().numpy(), ""))
        dist.barrier()
        dist.destroy_process_group()
    except Exception:  # noqa: BLE001 - reported to the parent
        import traceback
        queue.put((rank, None, traceback.format_exc()))


@pytest.mark.timeout(300)
@pytest.mark.parametrize("backend,kw", [
    ("all_to_all_nvlink", {}), ("all_to_all_nvlink", dict(expert_capacity_factor=0.6)),
    ("allgather_reduce", {}), ("allgather_reducescatter", dict(expert_capacity_factor=0.6)),
    ("replicated", {}), ("all_to_all", {}), ("all_to_all_reduce", {})])
def test_backends_match_the_unsharded_layer(backend, kw):
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, port, backend, kw, queue)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        results = {}
        for _ in range(2):
            rank, out, error = queue.get(timeout=120)
            assert not error, error
            results[rank] = out
    finally:
        for p in procs:
            p.join(timeout=30)
            if p.is_alive():
                p.terminate()
    rank0 = backend in ("all_to_all", "all_to_all_reduce")
    tokens = _tokens(0) if rank0 else torch.cat([_tokens(0), _tokens(1)])
    with torch.no_grad():
        expected = _scored(0, 1, "replicated", kw)(tokens).float().numpy()
        softmax = _layer(0, 1, "replicated", kw)(tokens).float().numpy()
    assert not np.allclose(expected, softmax, rtol=2e-2, atol=2e-3)
    if rank0 or backend == "replicated":
        np.testing.assert_array_equal(results[0], results[1])
        got = results[0]
    else:
        got = np.concatenate([results[0], results[1]])
    if rank0 or backend == "all_to_all_nvlink":
        np.testing.assert_array_equal(got, expected)
    else:  # partial outputs are summed in bf16 by the collective
        np.testing.assert_allclose(got, expected, rtol=2e-2, atol=2e-3)
