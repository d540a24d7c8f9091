"""A gloo job's collectives never see a GPU tensor: GradSync copies to the host and back around each.  Here on the CPU with the copies switched on by hand
(world 2): the same sums, and no collective is given the buffers themselves."""
import os
import socket
import sys

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SEGS = [(0, 1088), (1088, 5248), (5248, 5571)]
FORMS = [dict(algo="allreduce"), dict(algo="direct"), dict(algo="direct", payload="bf16"), dict(algo="direct", writeback=False),
         dict(algo="direct", payload="bf16", writeback=False, prepacked=True)]


def _worker(rank, world, port, out_dir):
    sys.path.insert(0, ROOT)
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from em_adapt_tensorflow_amd import dist as ours
    given = []
    for name in ("all_reduce", "all_to_all_single", "all_gather_into_tensor"):
        def wrap(*a, _f=getattr(dist, name), **kw):
            given.extend(t.untyped_storage().data_ptr() for t in a if torch.is_tensor(t))
            return _f(*a, **kw)
        setattr(dist, name, wrap)
    got = {}
    for k, form in enumerate(FORMS):
        for forced in (False, True):
            flat = torch.tensor(np.random.default_rng(7 * k + rank).normal(0, 1, SEGS[-1][1]).astype(np.float32))
            sync = ours.GradSync(flat, SEGS, bucket_bytes=2048 * 4, **form)
            assert sync.through_host is False
            sync.through_host = forced
            if sync.prepacked:
                sync.sendfull[:flat.numel()] = flat
            given.clear()
            for _ in range(2):
                for s, e in SEGS:
                    sync.segment_ready(s, e)
                sync.wait()
            own = {t.untyped_storage().data_ptr() for t in (flat, sync.gathered, sync.sendfull) if t is not None}
            if form["algo"] == "direct":
                own |= {t.untyped_storage().data_ptr() for t in (sync._send, sync._recv, sync._shard, sync._shard_p)}
            assert given and (own.isdisjoint(given) if forced else not own.isdisjoint(given))
            got["flat%d%d" % (k, forced)] = flat.numpy()
            if sync.gathered is not None:
                got["gathered%d%d" % (k, forced)] = sync.gathered.float().numpy()
    np.savez(os.path.join(out_dir, "rank%d.npz" % rank), **got)
    dist.barrier()
    dist.destroy_process_group()


def test_host_copies_give_the_same_sums(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    for rank in (0, 1):
        got = dict(np.load(tmp_path / ("rank%d.npz" % rank)))
        assert len(got) == 2 * (len(FORMS) + 4)
        for name in got:
            if name.endswith("0"):
                assert np.array_equal(got[name], got[name[:-1] + "1"]), name


@pytest.mark.parametrize("backend,is_cuda,want", [("gloo", True, True), ("gloo", False, False), ("nccl", True, False)])
def test_when_tensors_travel_through_the_host(monkeypatch, backend, is_cuda, want):
    from em_adapt_tensorflow_amd import dist as ours
    monkeypatch.setattr(dist, "get_backend", lambda group=None: backend)
    assert ours._through_host(is_cuda) is want
