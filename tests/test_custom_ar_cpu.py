"""The first-contact check of the custom all-reduce, its protocols replaced by the process group's own sums: a rank that finds a
difference, or whose launch raises, stays in step with the others, and all of them switch that protocol off."""
import os
import socket

import pytest
import torch
import torch.distributed as dist


def _rank(rank, world, port, fault, q):
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.set_num_threads(1)
    from datetime import timedelta

    from xgserve.parallel.custom_ar import CustomAllReduce
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=20))
    torch.cuda.synchronize = lambda *a: None
    other = dist.new_group(list(range(world)), timeout=timedelta(seconds=20))   # (the protocols' own links)
    calls = {"pull": 0, "pull_resid": 0}

    def bad(name):
        calls[name] += 1
        return rank == 1 and calls[name] == 4 and fault in ("wrong " + name, "raise " + name)

    class Fake(CustomAllReduce):
        def __init__(self):
            self.rank, self.world, self.device = rank, world, torch.device("cpu")
            self.slot, self.ll_max, self.resid_ll, self.shared_device, self.data, self.sig, self._opened = 8 << 20, 0, False, True, 0, 0, []
            self._gemm_ar = None

        def all_reduce(self, x, out=None):
            b = bad("pull")
            y = x.float()
            dist.all_reduce(y, group=other)
            if b and fault.startswith("raise"):
                raise RuntimeError("planted")
            return (y + (100.0 if b else 0.0)).bfloat16()

        def all_reduce_resid(self, part, r, ss):
            b = bad("pull_resid")
            y = part.sum(0)
            dist.all_reduce(y, group=other)
            if b and fault.startswith("raise"):
                raise RuntimeError("planted")
            r.copy_((r.float() + y + (100.0 if b else 0.0)).bfloat16())
            T, H = r.shape
            ss.copy_((r.float().view(T, H // 1024, 1024) ** 2).sum(-1).t().reshape(-1))

        def set_timeout(self, seconds):
            pass

        def serve_timeout(self, seconds=None):
            return 2.0

        def timeouts(self):
            return 0

        def reset_errors(self):
            pass

        def _two_shot(self, nbytes):
            return False

    try:
        ar = Fake()
        res = ar.self_test(dist.group.WORLD, dist.group.WORLD)
        q.put((rank, res, ar.verified_counts))
        dist.destroy_process_group()
    except Exception as e:  # noqa: BLE001 - reported to the parent
        q.put((rank, repr(e), None))


@pytest.mark.parametrize("fault", ["none", "wrong pull", "wrong pull_resid", "raise pull"])
def test_a_rank_that_differs_stays_in_step(fault):
    from xgserve.parallel.custom_ar import CustomAllReduce
    n = CustomAllReduce.SELF_TEST_ITERS
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = torch.multiprocessing.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, fault, q)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        got = {r[0]: r[1:] for r in (q.get(timeout=100) for _ in procs)}
    finally:
        for p in procs:
            p.join(timeout=20)
            if p.is_alive():
                p.kill()
    for rank in (0, 1):
        res, counts = got[rank]
        assert isinstance(res, dict), res
        for name in ("pull", "pull_resid"):
            planted = fault.endswith(" " + name)
            assert res[name] == (not planted)
            assert counts[name] == (3 if planted and rank == 1 else n)
        assert res["ll"] is None and res["gemm_ar"] is None
