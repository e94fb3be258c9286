"""Collectives of the package on device tensors over gloo: gloo itself sees host copies only (its own staging of device tensors has hung
with several ranks on one GPU), the results land in the device tensors."""
import socket

import pytest
import torch
import torch.distributed as dist

from nrhints_amd import parallel
from nrhints_amd.training import FlatGradAllReduce

pytestmark = pytest.mark.gpu


def test_gloo_is_handed_host_tensors(monkeypatch):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1)
    seen = []
    try:
        for name in ("all_reduce", "broadcast", "all_gather_into_tensor"):
            def spy(*a, _f=getattr(dist, name), **k):
                seen.append(all(not t.is_cuda for t in a if torch.is_tensor(t)))
                return _f(*a, **k)
            monkeypatch.setattr(dist, name, spy)
        x = torch.arange(6.0, device="cuda").reshape(2, 3)
        y = torch.empty(2, 3, device="cuda")
        parallel.all_reduce(x)
        parallel.broadcast(x)
        parallel.all_gather_into(y, x)
        assert torch.equal(x.cpu(), torch.arange(6.0).reshape(2, 3)) and torch.equal(x, y)
        p = torch.nn.Parameter(torch.ones(5, device="cuda"))
        p.grad = torch.full((5,), 3.0, device="cuda")
        sync = FlatGradAllReduce([p], always=True)
        sync.broadcast_parameters()
        sync()
        assert p.grad.tolist() == [3.0] * 5 and p.tolist() == [1.0] * 5
        assert len(seen) == 5 and all(seen)
    finally:
        dist.destroy_process_group()
