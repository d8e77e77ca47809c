"""liquid_cache_amd.sharding gives gloo host memory only (no GPU: a stand-in for a tensor that lives elsewhere)."""
import pytest
import torch
import torch.distributed as dist

from liquid_cache_amd import sharding as sh


class Elsewhere:
    """What the exchange may do with a tensor of another device: ask for its device, copy it to the host and back."""

    def __init__(self, values):
        self.values = torch.tensor(values, dtype=torch.int64)
        self.device = torch.device("meta")

    def cpu(self):
        return self.values.clone()

    def copy_(self, host):
        assert host.device.type == "cpu"
        self.values.copy_(host)
        return self


@pytest.fixture()
def gloo(tmp_path, monkeypatch):
    """A group of one rank whose collectives record the device of what they are given."""
    dist.init_process_group("gloo", init_method="file://%s" % (tmp_path / "store"), rank=0, world_size=1)
    seen = []

    def recorded(name):
        f = getattr(dist, name)

        def call(*args, **kw):
            for a in args:
                seen.extend((name, t.device.type) for t in (a if isinstance(a, list) else [a]))
            return f(*args, **kw)
        monkeypatch.setattr(dist, name, call)

    recorded("all_reduce")
    recorded("all_gather")
    yield seen
    dist.destroy_process_group()


def test_counts(gloo):
    t = Elsewhere([41])
    assert sh.all_reduce_count(t) is t
    assert t.values.tolist() == [41] and gloo == [("all_reduce", "cpu")]


def test_another_operation(gloo):
    t = Elsewhere([3, 9])
    sh.all_reduce(t, op=dist.ReduceOp.MAX)
    assert t.values.tolist() == [3, 9] and gloo == [("all_reduce", "cpu")]


def test_gathered_tensors(gloo):
    outs = [Elsewhere([0, 0])]
    sh.all_gather(outs, Elsewhere([5, 6]))
    assert outs[0].values.tolist() == [5, 6] and set(gloo) == {("all_gather", "cpu")}


@pytest.mark.parametrize("words", [[], [7], [1, 2, 3]])
def test_mask_segments(gloo, words):
    got = sh.all_gather_mask_segments(Elsewhere(words))
    assert [(g.device.type, g.numel()) for g in got] == [("meta", len(words))]
    assert gloo and {d for _, d in gloo} == {"cpu"}
    assert [g.tolist() for g in sh.all_gather_mask_segments(torch.tensor(words, dtype=torch.int64))] == [words]


def test_pipelined_counts(gloo):
    red = sh.PipelinedCountAllReduce(lambda: Elsewhere([0]), 2)
    for step in range(5):
        red.acquire().values.fill_(100 + step)
        red.submit()
    red.drain()
    assert red.last().values.tolist() == [104] and gloo == [("all_reduce", "cpu")] * 5


def test_host_tensors_are_given_as_they_are(gloo):
    t = torch.tensor([8], dtype=torch.int64)
    assert sh.all_reduce_count(t) is t
    assert gloo == [("all_reduce", "cpu")] and t.tolist() == [8]


@pytest.mark.parametrize("backend", ["gloo", "cpu:gloo,cuda:gloo"])
def test_a_device_tensor_goes_through_the_host_however_the_backend_is_named(tmp_path, backend):
    dist.init_process_group(backend, init_method="file://%s" % (tmp_path / "store"), rank=0, world_size=1)
    try:
        t = Elsewhere([4])
        t.device = torch.device("cuda")
        assert sh._through_host(t, None)
        assert not sh._through_host(torch.tensor([4]), None)
    finally:
        dist.destroy_process_group()


def test_a_device_of_another_backend_takes_its_tensors_itself(monkeypatch):
    monkeypatch.setattr(dist, "get_backend_config", lambda group=None: "cpu:gloo,cuda:nccl")
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "cpu:gloo,cuda:nccl")
    t = Elsewhere([4])
    t.device = torch.device("cuda")
    assert not sh._through_host(t, None)
