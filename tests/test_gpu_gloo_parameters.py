"""Collectives of the package on parameters that live on the GPU, over gloo: written in place as on any backend."""
import socket

import pytest
import torch
import torch.distributed as dist

from nrhints_amd import parallel

pytestmark = pytest.mark.gpu


def test_parameters_over_gloo():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1)
    try:
        p = torch.nn.Parameter(torch.arange(4.0, device="cuda"))
        q = torch.nn.Parameter(torch.zeros(4, device="cuda"))
        at = p.data_ptr()
        parallel.all_reduce(p)
        parallel.broadcast(p)
        parallel.all_gather_into(q, p)
        assert p.tolist() == q.tolist() == [0.0, 1.0, 2.0, 3.0] and p.data_ptr() == at and p.is_leaf and p.requires_grad
    finally:
        dist.destroy_process_group()
