"""A clipped step of the data-parallel trainer, two ranks on one GPU (gloo moves host copies): the norm is the union batch's,
equal on both, and both update with gradients clipped by it."""
import os
import time

import pytest
import torch

from test_zz_gpu_two_rank import DEV, _free_port, _trainer_args

pytestmark = pytest.mark.gpu
LIMIT = 1e-3


def _worker(rank, port, out_dir):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.cuda.set_device(0)
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        from cinema_amd.trainer import HotPathTrainer, SubjectStore
        torch.manual_seed(100 + rank)
        store = SubjectStore.synthetic(2, (20, 20, 20), 155.0 / 20, [155, 155, 155], 2, 10, seed=50 + rank, device=DEV)
        store.shuffle(torch.Generator(device=DEV).manual_seed(7 + rank))
        args = _trainer_args()
        args["optimizer"]["max_grad_norm"] = LIMIT
        tr = HotPathTrainer(args, store, DEV, keep_grads=True)
        groups = tr.opt_local.param_groups + tr.opt_mlp.param_groups
        before = [p.detach().cpu().clone() for g in groups for p in g["params"]]
        tr.step(0, 512 - 130 * rank)
        torch.cuda.synchronize()
        out = {"before": before, "after": [p.detach().cpu() for g in groups for p in g["params"]],
               "grads": [p.grad.detach().cpu() for g in groups for p in g["params"]],
               "lr": [g["lr"] for g in groups for _ in g["params"]], "tables": sum(len(g["params"]) for g in tr.opt_local.param_groups),
               "norms": [o.grad_norm.cpu() for o in (tr.opt_local, tr.opt_mlp)]}
        torch.save(out, os.path.join(out_dir, f"rank{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_two_ranks_clip_by_the_union_norm(tmp_path):
    import torch.multiprocessing as mp
    ctx = mp.start_processes(_worker, args=(_free_port(), str(tmp_path)), nprocs=2, join=False, start_method="spawn")
    deadline = time.time() + 90.0
    done = False
    while not done and time.time() < deadline:
        done = ctx.join(timeout=2.0)
    if not done:
        for pr in ctx.processes:
            if pr.is_alive():
                pr.kill()
        for pr in ctx.processes:
            pr.join(10)
        pytest.fail("two ranks sharing one GPU did not finish one clipped step in 90 s")
    ranks = [torch.load(tmp_path / f"rank{r}.pt", weights_only=True) for r in range(2)]
    n = ranks[0]["tables"]
    tables = [g.double().flatten() / 2 for r in ranks for g in r["grads"][:n]]
    shared = [g.double().flatten() for g in ranks[0]["grads"][n:]]
    assert all(torch.equal(a, b) for a, b in zip(ranks[0]["grads"][n:], ranks[1]["grads"][n:]))
    total = float(torch.cat(tables + shared).norm())
    assert total > 2 * LIMIT
    for r in ranks:
        assert all(v.dtype == torch.float32 and abs(float(v) - total) <= total * 2.0 ** -22 for v in r["norms"])
        for b, a, g, lr in zip(r["before"], r["after"], r["grads"], r["lr"]):
            q = torch.nn.Parameter(b.clone())
            q.grad = g * (LIMIT / (total + 1e-6))
            torch.optim.AdamW([q], lr=lr, weight_decay=0.0).step()
            # first step: lr * g / (|g| + 1e-8); where |g| is near that the factor's 2^-22 moves the update by as much
            assert float((a - q.detach()).abs().max()) <= lr * 2e-5 + float(b.abs().max()) * 2.0 ** -22
    assert all(torch.equal(a, b) for a, b in zip(ranks[0]["after"][n:], ranks[1]["after"][n:]))
