"""Gradient buckets of a model on the GPU over a gloo group: every collective is given host memory."""
import pytest
import torch
import torch.distributed as dist

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture
def gloo(tmp_path):
    dist.init_process_group("gloo", init_method="file://%s" % (tmp_path / "store"), rank=0, world_size=1)
    yield
    dist.destroy_process_group()


def test_buckets_and_broadcasts_go_through_host_memory(gloo, monkeypatch):
    from dtt import dist as D
    seen = []
    for name in ("all_reduce", "broadcast"):
        def checked(t, *a, _f=getattr(dist, name), _n=name, **k):
            assert t.device.type == "cpu", "%s of a tensor on %s" % (_n, t.device)
            seen.append(_n)
            return _f(t, *a, **k)
        monkeypatch.setattr(dist, name, checked)
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 3, padding=1), torch.nn.BatchNorm2d(8), torch.nn.Conv2d(8, 5, 1)).to(DEV)
    model[2].weight.data = model[2].weight.data.contiguous(memory_format=torch.channels_last)
    before = [t.clone() for t in list(model.parameters()) + list(model.buffers())]
    runner = D.DataParallelSnippets(model, 1, bucket_bytes=256, force_buckets=True)
    runner._sync_initial_state()                    # (one rank does not call it by itself)
    assert all(torch.equal(a, b) for a, b in zip(before, list(model.parameters()) + list(model.buffers())))
    raw = {}
    for n, p in model.named_parameters():
        p.register_hook(lambda g, n=n: raw.__setitem__(n, g.detach().clone()))
    for step in range(2):
        runner.zero_grad(set_to_none=True)
        runner(torch.randn(2, 3, 9, 7, device=DEV)).square().mean().backward()
        runner.finish_gradients()
        assert all(torch.equal(p.grad, raw[n]) for n, p in model.named_parameters())      # the sum over one rank
    assert runner.time_allreduce_ms(2) > 0
    assert seen.count("broadcast") == 8 and seen.count("all_reduce") >= 6                 # 6 parameters, 2 float buffers
