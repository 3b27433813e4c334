"""Data-parallel averaging of a model with a table in front of its reported layers (gloo, two ranks, no GPU)."""
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from sparc_amd.parallel import LayerwiseReducer, reduce_gradients, reported_parameters


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.table = torch.nn.Parameter(torch.randn(7, 3))
        self.layers = torch.nn.ModuleList([torch.nn.Linear(3, 4)])

    def mlp_parameters(self):
        return [p for layer in self.layers for p in layer.parameters()]


def _worker(rank, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    torch.manual_seed(0)
    net = Net()
    assert [id(p) for p in reported_parameters(net)] == [id(p) for p in net.layers[0].parameters()]
    reducer = LayerwiseReducer(reported_parameters(net))
    for step in range(2):
        gen = torch.Generator().manual_seed(10 * step + rank)
        local = [torch.randn(p.shape, generator=gen) for p in net.parameters()]
        for p in net.parameters():
            p.grad = None
        reducer(0, local[1], local[2])               # the backward reports its layer ...
        net.table.grad = local[0]                    # ... and autograd leaves the table's gradient
        reduce_gradients(net, reducer)
        both = [torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * step + r)) for r in range(2) for p in [net.table]]
        assert torch.allclose(net.table.grad, (both[0] + both[1]) / 2)
    # a model that reports nothing: everything in one bucket
    for p in net.parameters():
        p.grad = torch.full(p.shape, float(rank))
    reduce_gradients(net, reducer)
    out.put([p.grad.flatten().tolist() for p in net.parameters()])
    dist.barrier()
    dist.destroy_process_group()


def test_table_gradient_is_averaged_with_the_layers():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    ctx = mp.get_context("spawn")
    out = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, port, out)) for r in range(2)]
    for p in procs:
        p.start()
    got = [out.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert all(v == 0.5 for grads in got for g in grads for v in g)
