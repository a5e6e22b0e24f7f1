"""Device tensors of a gloo group go through host memory (dp._collective): the same workers as on host tensors, with the staging forced on
host tensors - every result equals the unstaged one bit for bit, and no collective is handed a tensor the caller holds."""
import numpy as np
import pytest
import torch
import torch.distributed as dist

import test_dp_gloo as G


def _staged(rank, world, port, q, worker, *args):
    from libra_amd import dp
    dp._staged = lambda t, group: True
    held, seen = set(), []
    for name in ("all_reduce", "reduce_scatter_tensor", "all_gather_into_tensor"):
        def wrapped(*ts, _fn=getattr(dist, name), **kw):
            seen.extend(t.untyped_storage().data_ptr() for t in ts)
            return _fn(*ts, **kw)
        setattr(dist, name, wrapped)
    init = dp.GradBuckets.__init__

    def hold(self, *a, **kw):
        init(self, *a, **kw)
        held.update(b.flat.untyped_storage().data_ptr() for b in self.buckets)
    dp.GradBuckets.__init__ = hold
    worker(rank, world, port, q, *args)
    assert seen and held and not held & set(seen)


def _run(worker, *args):
    ctx = G.mp.get_context("spawn")
    q, port = ctx.Queue(), G._free_port()
    ps = [ctx.Process(target=_staged, args=(r, 2, port, q, worker, *args)) for r in range(2)]
    [p.start() for p in ps]
    res = sorted((q.get(timeout=180) for _ in range(2)), key=lambda t: t[0])
    [p.join(60) for p in ps]
    assert all(p.exitcode == 0 for p in ps)
    return res


def _same(a, b):
    if isinstance(a, dict):
        assert a.keys() == b.keys()
        for k in a:
            _same(a[k], b[k])
    elif isinstance(a, (list, tuple)):
        assert len(a) == len(b)
        for x, y in zip(a, b):
            _same(x, y)
    elif isinstance(a, np.ndarray):
        assert np.array_equal(a, b)
    else:
        assert a == b


@pytest.mark.parametrize("mode", ["allreduce", "rs_ag"])
def test_staged_exchange(mode):
    _same(_run(G._worker_modes, mode), G._run(G._worker_modes, 2, mode))


@pytest.mark.parametrize("mode", ["allreduce", "zero1"])
def test_staged_sharded_optimizer(mode):
    _same(_run(G._worker_zero1, mode), G._run(G._worker_zero1, 2, mode))


@pytest.mark.parametrize("mode", ["allreduce", "zero1"])
def test_staged_clipping_and_resume(mode):
    _same(_run(G._worker_clip, mode), G._run(G._worker_clip, 2, mode))


def test_wait_copies_once():
    from libra_amd import dp

    class Work:
        n = 0

        def wait(self):
            Work.n += 1
    dst, host = torch.zeros(3), torch.ones(3)
    w = dp._StagedWork(Work(), host, dst)
    w.wait()
    dst.add_(1)
    w.wait()
    assert Work.n == 1 and dst.tolist() == [2, 2, 2]


@pytest.mark.parametrize("config,staged", [("cpu:gloo,cuda:gloo", True), ("cpu:gloo,cuda:nccl", False), ("cuda:nccl", False), ("cuda:nccl,cpu:gloo", False),
                                           ("cpu:mpi,cuda:mpi", False)])
def test_only_gloo_is_staged(config, staged, monkeypatch):
    """What counts is the backend of the tensor's device type: a group initialised without a backend ("cpu:gloo,cuda:nccl") or for devices
    only ("cuda:nccl") carries device tensors over RCCL, directly."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from libra_amd import dp
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "undefined")
    monkeypatch.setattr(dist, "get_backend_config", lambda group=None: config)
    sent = []
    work = object()
    with FakeTensorMode():
        t = torch.empty(8, device="cuda")
        assert dp._staged(t, None) is staged and dp._staged(torch.empty(8), None) is False
        if not staged:
            assert dp._collective(lambda *ts, group, async_op: sent.extend(ts) or work, t) is work and sent == [t]


def test_the_backend_of_a_real_group(monkeypatch):
    """get_backend_config of the groups that can be made here names the backend of every device type."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from libra_amd import dp
    for backend in ("gloo", "cpu:gloo,cuda:gloo", "cpu:gloo"):
        dist.init_process_group(backend, init_method=f"tcp://127.0.0.1:{G._free_port()}", rank=0, world_size=1)
        try:
            with FakeTensorMode():
                assert dp._staged(torch.empty(4, device="cuda"), None) is ("cuda" in backend or backend == "gloo")
                assert dp._staged(torch.empty(4, device="cuda"), dist.group.WORLD) is ("cuda" in backend or backend == "gloo")
        finally:
            dist.destroy_process_group()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gather", [False, True])
def test_device_copies_of_a_staged_collective(dtype, gather, monkeypatch):
    """The copies themselves, one process and no group: what the collective is handed are host tensors with the values of the work queued on
    the current stream until then; wait(), called with another stream current, leaves the result on the device for every stream."""
    from libra_amd import dp
    monkeypatch.setattr(dp, "_staged", lambda t, group: t.is_cuda)
    n, dev = 100003, "cuda"
    seen = []

    class Work:
        def __init__(self, done):
            self.done = done

        def wait(self):
            self.done()

    def collective(out, *inp, group, async_op, scale):
        assert async_op and group is None and not out.is_cuda and not any(t.is_cuda for t in inp)
        src = inp[0] if inp else out
        seen.append(src.clone())

        def done():
            out.copy_(src.repeat(out.numel() // src.numel()) * scale)
        return Work(done)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    a = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(0)).to(dtype)
    big = torch.ones(2048, 2048, device=dev)
    flat = torch.zeros(2 * n if gather else n, dtype=dtype, device=dev)
    mine = flat[:n]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):                                             # (work in front of the values)
            big = big @ big * 2.0 ** -11
        mine.copy_(a.to(dev) * big[0, 0].to(dtype))
        w = dp._collective(collective, flat, mine, scale=2) if gather else dp._collective(collective, flat, scale=2)
    with torch.cuda.stream(other):
        w.wait()
        got = flat.clone()
        flat.add_(1)
        w.wait()                                                        # (a second wait copies nothing)
    torch.cuda.synchronize()
    assert torch.equal(seen[0], a) and torch.equal(got.cpu(), (2 * a).repeat(2 if gather else 1))
    assert torch.equal(flat.cpu(), (2 * a).repeat(2 if gather else 1) + 1)
