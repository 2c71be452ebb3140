"""max_grad_norm with several ranks: the norm is that of the summed gradient on every rank, the replicas stay bit-identical, and the step is the
unclipped one's times the factor - with the row-range all-reduce and with both direct exchanges of the feature trainer, and with the one bucket of
the RGB trainer.  Two ranks share one GPU; what torch.distributed sums goes through host memory (gloo is given CPU tensors only)."""
import math
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_gpu_dist import _free_port

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class _Done:
    def wait(self):
        return True


def _staged_all_reduce(original):
    def all_reduce(tensor, op=dist.ReduceOp.SUM, group=None, async_op=False):
        if not tensor.is_cuda:
            return original(tensor, op=op, group=group, async_op=async_op)
        host = tensor.cpu()
        original(host, op=op, group=group)
        tensor.copy_(host)
        return _Done() if async_op else None
    return all_reduce


def _join(rank, world, port):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    os.environ.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
    torch.cuda.set_device(0)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    dist.all_reduce = _staged_all_reduce(dist.all_reduce)


def _seg_worker(rank, world, port, out, jobs):
    _join(rank, world, port)
    from instascene_amd import scenes, rasterizer as rz
    from instascene_amd.harness import SegTrainer
    rz.set_mode("exact")
    rz.set_tracer(False)
    sc, cams = scenes.synthetic_scene(4000, 16, 5, math.log(0.04)), scenes.ring_cameras(6, 128, 96)
    for name, exchange, bound in jobs:
        if isinstance(bound, str):                          # a part of the norm that another job measured
            bound = 0.3 * torch.load(os.path.join(out, f"{bound}_{rank}.pt"))["norms"][0][0]
        tr = SegTrainer(sc, cams, device="cuda", sample_batchsize=2048, n_labels=12, use_class_feat=True, seed=3, rank=rank, world=world,
                        max_grad_norm=bound)
        tr.exchange = exchange
        tr.warm_view_caches()
        norms, first = [], None
        clip = tr.opt._clip_coef

        def spy(grads, max_norm):
            coef = clip(grads, max_norm)
            norms.append((float(tr.opt.last_grad_norm), float(grads[0].double().norm()), float(coef)))
            return coef

        tr.opt._clip_coef = spy
        for it in range(3):
            tr.step(it)
            if first is None:
                first = tr.opt.exp_avg.cpu()
        torch.cuda.synchronize()
        torch.save({"p": tr.model._seg_feature.detach().cpu(), "m": tr.opt.exp_avg.cpu(), "first": first, "norms": norms, "bound": bound},
                   os.path.join(out, f"{name}_{rank}.pt"))
        dist.barrier()
    dist.destroy_process_group()


@pytest.mark.timeout(300)
def test_feature_trainer_on_two_ranks(tmp_path):
    jobs = [("wide", "rccl", 1e9), ("rccl", "rccl", "wide"), ("peer", "peer", "wide"), ("compact", "peer_compact", "wide")]
    mp.spawn(_seg_worker, args=(2, _free_port(), str(tmp_path), jobs), nprocs=2, join=True)
    run = {name: [torch.load(tmp_path / f"{name}_{r}.pt") for r in range(2)] for name, _, _ in jobs}
    for name, (a, b) in run.items():
        assert len(a["norms"]) == 3 and a["norms"] == b["norms"], name          # every rank: the norm of the whole sum
        assert torch.equal(a["p"], b["p"]) and torch.equal(a["m"], b["m"]), name
        for norm, exact, coef in a["norms"]:
            assert exact > 0 and abs(norm - exact) <= 2 * U * exact             # one root in 64 bits, one rounding
            want = min(1.0, a["bound"] / (norm + 1e-6))
            assert abs(coef - want) <= 4 * U * want
    assert run["wide"][0]["norms"][0][2] == 1.0 and run["rccl"][0]["norms"][0][2] < 0.31
    for name in ("peer", "compact"):                        # (two ranks: every sum is a + b)
        assert torch.equal(run[name][0]["p"], run["rccl"][0]["p"]) and torch.equal(run[name][0]["m"], run["rccl"][0]["m"]), name
    # the first step's moment is 0.1 of the clipped gradient: three products in turn, each side
    want = run["wide"][0]["first"].double() * run["rccl"][0]["norms"][0][2]
    assert bool(((run["rccl"][0]["first"].double() - want).abs() <= 4 * U * want.abs() + 2.0 ** -149).all())


def _rgb_worker(rank, world, port, out):
    _join(rank, world, port)
    from instascene_amd import scenes, rasterizer as rz
    from instascene_amd.harness import RgbTrainer
    rz.set_mode("exact")
    rz.set_tracer(False)
    sc, cams = scenes.synthetic_scene(3000, 4, 7, math.log(0.05)), scenes.ring_cameras(4, 96, 64)
    targets = [torch.rand(3, 64, 96, generator=torch.Generator().manual_seed(k)) for k in range(4)]
    results, bound = {}, 1e9
    for name, fused in (("wide", True), ("fused", True), ("torch", False)):
        tr = RgbTrainer(sc, cams, targets, device="cuda", rank=rank, world=world, max_grad_norm=bound, fused_update=fused)
        tr.step(0)
        norm = float(tr.last_grad_norm)
        params = {k: getattr(tr.model, k).detach().cpu() for k in ("_xyz", "_features_dc", "_features_rest", "_opacity", "_scaling", "_rotation")}
        if fused:
            avg = {k: v.cpu() for k, v in tr.opt.exp_avg.items()}
        else:
            names = dict(xyz="_xyz", f_dc="_features_dc", f_rest="_features_rest", opacity="_opacity", scaling="_scaling", rotation="_rotation")
            avg = {k: tr.opt.state[getattr(tr.model, v)]["exp_avg"].cpu() for k, v in names.items()}
        results[name] = {"norm": norm, "params": params, "avg": avg, "bound": bound}
        bound = 0.3 * results["wide"]["norm"]
    torch.cuda.synchronize()
    torch.save(results, os.path.join(out, f"rgb_{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.timeout(300)
def test_rgb_trainer_on_two_ranks(tmp_path):
    mp.spawn(_rgb_worker, args=(2, _free_port(), str(tmp_path)), nprocs=2, join=True)
    a, b = (torch.load(tmp_path / f"rgb_{r}.pt") for r in range(2))
    for name in a:
        assert a[name]["norm"] == b[name]["norm"] and all(torch.equal(a[name]["params"][k], b[name]["params"][k]) for k in a[name]["params"]), name
    assert a["fused"]["norm"] == a["wide"]["norm"]
    coef = 0.3 * a["wide"]["norm"] / (a["wide"]["norm"] + 1e-6)
    for k, wide in a["wide"]["avg"].items():
        want = wide.double() * coef
        # (the factor is applied to each raw gradient before the moment's own product: four roundings each side, the factor's four)
        assert bool(((a["fused"]["avg"][k].double() - want).abs() <= 12 * U * want.abs() + 2.0 ** -148).all()), k
        # torch's optimiser on gradients that autograd's chain rule made: another order of the same products
        assert float((a["torch"]["avg"][k].double() - want).norm()) <= 1e-3 * float(want.norm()), k
    assert abs(a["torch"]["norm"] - a["wide"]["norm"]) <= 1e-4 * a["wide"]["norm"]
