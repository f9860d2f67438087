"""nn.Dropout's (seed, call) is the layer's own: it moves with the module, is copied with it, is no part of the state_dict, and no
wrapper that keeps buffers alike over ranks touches it."""
import copy
import os

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from repdl_amd import nn


def _rank(rank, path):
    os.environ["GLOO_SOCKET_IFNAME"] = "lo"
    dist.init_process_group("gloo", init_method="file://" + path, rank=rank, world_size=2)
    model = torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.BatchNorm1d(4), nn.Dropout(0.5, seed=100 + rank)).eval()
    model[1].running_mean.fill_(float(rank))
    wrapped = torch.nn.parallel.DistributedDataParallel(model)  # (its default: rank 0's buffers, at the start and before every forward pass)
    assert model[2].rng_state.tolist() == [100 + rank, 0]
    model[2].rng_state[1] = 5 + rank
    wrapped(torch.ones(2, 4))  # (dropout passes through: no GPU is needed)
    assert model[2].rng_state.tolist() == [100 + rank, 5 + rank]
    assert model[1].running_mean.tolist() == [0.0] * 4  # the buffers were indeed broadcast
    dist.destroy_process_group()


def test_every_rank_keeps_its_own_masks(tmp_path):
    mp.spawn(_rank, args=(str(tmp_path / "store"),), nprocs=2)


def test_what_a_module_does_with_it():
    layer = nn.Dropout(0.5, seed=9)
    assert not list(layer.buffers()) and not list(layer.parameters()) and not layer.state_dict()
    layer.rng_state[1] = 4
    for other in (copy.deepcopy(layer), copy.deepcopy(torch.nn.Sequential(layer))[0]):
        assert other.rng_state.tolist() == [9, 4] and other.rng_state is not layer.rng_state
    net = torch.nn.Sequential(layer)
    for move in (net.half, net.double, net.bfloat16, net.cpu, lambda: net.to("cpu", torch.float16)):
        assert move()[0].rng_state.tolist() == [9, 4] and net[0].rng_state.dtype == torch.int64
    assert net.to("meta")[0].rng_state.device.type == "meta"  # it goes where the module goes


def test_the_seed_is_drawn_on_the_cpu():
    """Also where a default device is set, whose generator -- and whose values, if it has any -- would be another's."""
    torch.manual_seed(3)
    want = [nn.Dropout(0.5).rng_state.tolist() for _ in range(2)]
    torch.manual_seed(3)
    with torch.device("meta"):
        assert nn.Dropout(0.5).rng_state.is_meta
    assert nn.Dropout(0.5).rng_state.tolist() == want[1]
