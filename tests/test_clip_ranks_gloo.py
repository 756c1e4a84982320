"""Clipping by the global norm when the batch is shared out over ranks: two processes on the CPU (gloo).  The
all-reduce, MLP.update and the scale that it hands on are the product's; the update kernel is replaced by its formula."""
import os
import socket
import sys
from types import SimpleNamespace

import numpy as np
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
N, COUNTS, LIMIT, LR = 2, [37, 8, 101], 3.0, 0.5


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def local_gradient(rank):
    return np.random.default_rng(100 + rank).integers(-8, 8, sum(COUNTS)).astype(np.float32)      # sums are exact


def clipped(w, g, gscale, limit):
    """update_multi_(SGD, gscale, gclip_global=limit): the norm of gscale*g, the update with the factor"""
    norm = abs(gscale) * float(np.sqrt((g.astype(np.float64) ** 2).sum()))
    factor = limit / norm if norm > limit else 1.0
    return w - LR * gscale * (factor * g.astype(np.float64)), norm


def _worker(rank, world, port, out):
    sys.path.insert(0, os.path.join(ROOT, "knet.jl_b200"))
    from knet_sm100 import dp, mlp, train
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    offsets = np.concatenate([[0], np.cumsum(COUNTS)])
    for captured in (False, True):
        flat = torch.from_numpy(local_gradient(rank))
        for b in dp.bucket_bounds(offsets):
            dp.allreduce_bucket(flat, b).wait()
        w = np.zeros(sum(COUNTS))
        calls = []

        def update(plan, opt, gscale, gclip_global=0):
            nonlocal w
            w, norm = clipped(w, flat.numpy(), gscale, gclip_global)
            return norm

        def global_norm(plan, gclip, gscale):
            calls.append((gclip, gscale))
            return clipped(w, flat.numpy(), gscale, gclip)[1], torch.ones(1)

        mlp.update_multi_, mlp._global_norm = update, global_norm
        me = SimpleNamespace(offsets=offsets, world=world, sharded=False, state=[], esize=4, gclip_global=LIMIT, probe=None, launches=0,
                             plan=SimpleNamespace(table=torch.zeros(1), ntensors=3, total_chunks=3), L=3, S="32", _capturing=captured,
                             opt=train.Adam() if captured else train.SGD(lr=LR), _dev_step=torch.zeros(1),
                             _kn=lambda label, nbytes, call, name, *a, launches=1: calls.append((name, a[-2])))
        mlp.MLP.update(me)
        if captured:
            assert calls == [(LIMIT, 1 / world), ("knet_adam_multi_gcg_32", 1 / world)]      # norm and update see one scale
        out[rank, captured] = (w.copy(), float(me.gnorm))
    dist.barrier()
    dist.destroy_process_group()


def test_ranks_clip_by_the_norm_of_the_mean_gradient():
    mgr = mp.Manager()
    out = mgr.dict()
    mp.spawn(_worker, args=(N, _free_port(), out), nprocs=N, join=True)
    mean = sum(local_gradient(r) for r in range(N)) / N
    want, norm = clipped(np.zeros(sum(COUNTS)), mean, 1.0, LIMIT)
    assert norm > LIMIT
    for captured in (False, True):
        for r in range(N):
            w, got = out[r, captured]
            assert got == norm
            if not captured:
                np.testing.assert_allclose(w, want, rtol=1e-15)
