"""Who has the position rotation in the append: the cache's choice, or the model's where it has none; one
engine's choice is not another's. Layers and caches on the host, the launches' places taken."""
from __future__ import annotations

import copy
from types import SimpleNamespace

import pytest
import torch

from winnow_amd import packed_backend as pb
from winnow_amd.page_pool import PagePool


class Qwen2Attention(torch.nn.Module):
    def __init__(self, config):
        super().__init__()
        self.config, self.head_dim, self.layer_idx, self.scaling = config, 128, 0, 0.1
        self.q_proj = self.k_proj = self.v_proj = self.o_proj = torch.nn.Identity()

    def forward(self, hidden_states, position_embeddings=None, attention_mask=None, past_key_values=None, **kwargs):
        return "its own"


class _Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.config = SimpleNamespace(architectures=[pb.SUPPORTED_ARCH[0]], _attn_implementation=pb.ATTN_NAME)
        self.layers = torch.nn.ModuleList(Qwen2Attention(self.config) for _ in range(2))
        self.w = torch.nn.Parameter(torch.zeros(1))


@pytest.fixture
def ran(monkeypatch):
    """Runs both layers with a cache: how many of them had the append rotate."""
    fused = []
    monkeypatch.setattr(pb.PagedPackedCache, "update_rotated", lambda self, q, k, v, cos, sin, layer: (fused.append(layer), (q, None))[1])
    monkeypatch.setattr(pb, "winnow_packed_attention", lambda module, q, *a, **kw: (q, None))
    monkeypatch.setattr(pb, "_plain", lambda t: True)
    pool = PagePool(num_layers=1, num_pages=4, num_kv_heads=1, page_size=16, nb_k=64, nb_v=64)

    @torch.no_grad()
    def run(model, **kw):
        fused.clear()
        cache = pb.PagedPackedCache(pool, ["a"], [0], k_quant=None, v_quant=None, head_dim=128, **kw)
        for layer in model.layers:
            layer(torch.zeros(1, 1, 128), position_embeddings=(None, None), past_key_values=cache)
        return len(fused)
    return run


def test_the_cache_decides_and_else_the_model(ran):
    model = _Model()
    assert [ran(model, fuse_rotary=x) for x in (None, False, True)] == [0, 0, 0]       # no class that could
    assert len(pb.rotary_layers(model)) == 2
    assert [ran(model, fuse_rotary=x) for x in (None, False, True)] == [0, 0, 2]
    assert pb.fuse_rotary(model) == 2 == pb.fuse_rotary(model)
    assert [ran(model, fuse_rotary=x) for x in (None, False, True)] == [2, 0, 2]
    other = copy.deepcopy(model)
    assert pb.fuse_rotary(model, False) == 2
    assert [ran(model, fuse_rotary=x) for x in (None, False, True)] == [0, 0, 2]
    assert ran(other) == 2


def test_an_engine_leaves_the_model_to_others(ran):
    from winnow_amd.engine import Engine, EngineConfig
    model = _Model()
    pool = PagePool(num_layers=1, num_pages=4, num_kv_heads=1, page_size=16, nb_k=64, nb_v=64)
    fused, plain, either = (Engine(model, pool, None, None, 128, config=EngineConfig(**cfg)) for cfg in (
        dict(fuse_rotary=True), dict(fuse_rotary=False), dict()))
    assert ran(model) == 0
    assert [ran(model, fuse_rotary=e.cfg.fuse_rotary) for e in (fused, plain, either)] == [2, 0, 0]
    pb.fuse_rotary(model)
    assert [ran(model, fuse_rotary=e.cfg.fuse_rotary) for e in (fused, plain, either)] == [2, 0, 2]
