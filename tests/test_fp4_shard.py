"""The sharded 4-bit top-k: each rank answers an equal range of rows, every rank gets all of them.
On CPU with gloo, the device's part played by numpy; on a GPU with a world of one."""
import os

import numpy as np
import pytest

import _fp4_ref as ref
from test_shard_gloo import free_port


class _Context:
    def __init__(self, values, fmt):
        self.values, self.fmt, self.asked = values, fmt, []

    def lowrank4_topk(self, k, r0, r1):
        self.asked.append((r0, r1))
        idx, val = np.empty((r1 - r0, k), np.int32), np.empty((r1 - r0, k), np.float32)
        for i in range(r0, r1):
            idx[i - r0], val[i - r0] = (t[0] for t in ref.topk(self.values[i:i + 1], self.values, k, i, self.fmt))
        return idx, val


class _Estimator:
    def __init__(self, values, fmt):
        self.ctx, self.fmt, self.n = _Context(values, fmt), fmt, len(values)

    def _context(self):
        return self.ctx

    def _lowrank4(self):
        return self.fmt

    def _lowrank_rows(self):
        return self.n


def _values(n, fmt):
    x = np.random.default_rng(n).normal(size=(n, 24))
    return ref.values(*ref.quantize(x, fmt), fmt)


def _worker(rank, world, port, n, fmt, out):
    import torch.distributed as dist
    from rfx_b200.shard import lowrank_topk_sharded
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    est = _Estimator(_values(n, fmt), fmt)
    out[rank] = (*lowrank_topk_sharded(est, 7, dist), est.ctx.asked)
    dist.destroy_process_group()


@pytest.mark.parametrize("world,n,fmt", [(2, 301, "nvfp4"), (3, 100, "mxfp4"), (3, 2, "nvfp4")])
def test_every_rank_gets_every_row(world, n, fmt):
    import torch.multiprocessing as mp
    out = mp.get_context("spawn").Manager().dict()
    mp.spawn(_worker, args=(world, free_port(), n, fmt, out), nprocs=world, join=True)
    idx, val = ref.topk(_values(n, fmt), _values(n, fmt), 7, 0, fmt)
    asked = [out[r][2][0] for r in range(world)]
    assert asked[0][0] == 0 and asked[-1][1] == n
    assert all(asked[r][1] == asked[r + 1][0] for r in range(world - 1))
    for r in range(world):
        assert np.array_equal(out[r][0], idx) and np.array_equal(out[r][1], val)


def _gpu_worker(rank, port, fmt, out):
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    sys.path[:0] = [here, os.path.join(os.path.dirname(here), "rfx-fuse_b200")]
    import torch
    import torch.distributed as dist
    import rfx_b200
    from rfx_b200.shard import fit_sharded
    from _helpers import synth
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    torch.cuda.set_device(0)
    dist.init_process_group("nccl", rank=0, world_size=1, device_id=torch.device("cuda", 0))
    X, y = synth("multiclass", 900, 8, 33)
    kw = dict(nsample=900, ntree=8, mtry=3, minndsize=1, compute_proximity=True, compute_importance=False,
              use_qlora=True, quant_mode=fmt, rank=16, show_progress=False)
    est = rfx_b200.RandomForestClassifier(**kw)
    fit_sharded(est, X, y, dist, 0)
    sharded = (est.get_lowrank_factors()[0], *est.get_lowrank_topk(10), est.get_lowrank_product(5, 200))
    part = est.get_lowrank_topk(10, 130, 140)
    alone = rfx_b200.RandomForestClassifier(**kw)
    alone.fit(X, y)
    single = (alone.get_lowrank_factors()[0], *alone.get_lowrank_topk(10), alone.get_lowrank_product(5, 200))
    out["sharded"], out["part"], out["single"] = sharded, part, single
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_a_sharded_fit_of_one_rank(fmt):
    """fit_sharded quantises the factors too, and its answers are those of fit."""
    import torch.multiprocessing as mp
    out = mp.get_context("spawn").Manager().dict()
    mp.spawn(_gpu_worker, args=(free_port(), fmt, out), nprocs=1, join=True)
    A, idx, val, P = out["sharded"]
    wi, wv = ref.topk(A, A, 10, 0, fmt)
    assert np.array_equal(idx, wi) and np.array_equal(val, wv)
    assert np.array_equal(out["part"][0], wi[130:140]) and np.array_equal(out["part"][1], wv[130:140])
    for got, want in zip(out["sharded"], out["single"]):
        assert np.array_equal(got, want)
