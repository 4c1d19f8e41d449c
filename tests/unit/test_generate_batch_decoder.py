"""The captured decoding step of Gemma.generate_batch, with CUDA's graph calls replaced by records (CPU)."""

import contextlib

import pytest
import torch

from mint_b200.kvcache.paged import PagedKVCache
from mint_b200.models import gemma
from mint_b200.models.gemma import Gemma, GemmaConfig

CFG = dict(embed_dim=64, hidden_dim=128, seq_length=48, vocab_size=100, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=16)


def _model():
    torch.manual_seed(3)
    return Gemma(GemmaConfig(**CFG)).eval()


@pytest.fixture()
def fake_cuda(monkeypatch):
    """Records of the graph calls; a captured step runs at once, a replay runs it again."""
    log = {"devices": [], "graphs": [], "replays": 0}

    class FakeGraph:
        def replay(self):
            log["replays"] += 1
            assert log["devices"][-1] == torch.device("cuda", 1)

    @contextlib.contextmanager
    def device(dev):
        log["devices"].append(torch.device(dev))
        yield
        log["devices"].pop()

    @contextlib.contextmanager
    def graph(g, **kw):
        log["graphs"].append((g, kw, list(log["devices"])))
        yield

    monkeypatch.setattr(torch.cuda, "CUDAGraph", FakeGraph)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    monkeypatch.setattr(torch.cuda, "Stream", lambda dev: ("stream", torch.device(dev)))
    return log


def _decoder():
    cache = PagedKVCache(2, 8, 8, 2, 16, max_batch=2, max_seq_len=32)
    cache.plan([3, 2])
    decoder = gemma._Decoder(_model(), cache, cuda_graph=True)
    decoder.device, decoder.use_graph = torch.device("cuda", 1), True
    return decoder


def test_capture_and_replay_are_on_the_caches_device(fake_cuda):
    decoder = _decoder()
    with torch.no_grad():
        for _ in range(4):
            decoder.step([0, 1], [5, 6])
    assert len(fake_cuda["graphs"]) == 1 and fake_cuda["replays"] == 3
    _, kw, devices = fake_cuda["graphs"][0]
    assert kw["stream"] == ("stream", torch.device("cuda", 1)) and devices == [torch.device("cuda", 1)]


@pytest.mark.parametrize("dtype,head_dim,kernels,graph", [
    (torch.bfloat16, 128, "on", True), (torch.float16, 64, "on", True), (torch.bfloat16, 256, "on", True),
    (torch.float32, 128, "on", False), (torch.bfloat16, 32, "on", False), (torch.bfloat16, 96, "on", False),
    (torch.bfloat16, 128, "off", False),
])
def test_only_steps_of_kernels_are_captured(dtype, head_dim, kernels, graph, monkeypatch):
    """The PyTorch forms synchronize, which ends a capture with an error."""
    monkeypatch.setenv("MINT_DISABLE_KERNELS", "1" if kernels == "off" else "0")

    class Pages:  # stands for a CUDA tensor
        device, shape = torch.device("cuda", 0), (1, 1, 1, 8, head_dim)

    class Cache:
        device, k_pages, max_batch = torch.device("cuda", 0), Pages, 2

    Cache.dtype = dtype
    monkeypatch.setattr(torch, "zeros", lambda *a, **k: None)
    assert gemma._Decoder(_model_stub(), Cache, cuda_graph=True).use_graph == graph
    assert not gemma._Decoder(_model_stub(), Cache, cuda_graph=False).use_graph


def _model_stub():
    return type("Stub", (), {"_before_forward": None})()


def test_other_threads_calls_do_not_end_the_capture(fake_cuda):
    decoder = _decoder()
    with torch.no_grad():
        for _ in range(2):
            decoder.step([0, 1], [5, 6])
    assert fake_cuda["graphs"][0][1]["capture_error_mode"] == "thread_local"
