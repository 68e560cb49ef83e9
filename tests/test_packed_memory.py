"""The memory that a cache held in 4 bits takes beside its pages: the pages of one layer in 16 bits, for portions of prompts."""
import json

import pytest
import torch

import conftest


def model_of(tmp_path, cfg, dtype=torch.bfloat16):
    from ferrum_b200.config import registry
    folder = tmp_path / "m"
    folder.mkdir(exist_ok=True)
    (folder / "config.json").write_text(json.dumps(cfg))
    arch, parsed = registry.read_config(str(folder))
    return arch.build(parsed, dtype, "cpu")


def test_scratch_of_a_position(tmp_path):
    from ferrum_b200.cache import CacheStorage
    model = model_of(tmp_path, conftest.MID_E)
    assert CacheStorage.scratch_bytes_per_token_of(model, torch.bfloat16) == 0
    model.set_cache_bits(4)
    # one layer's keys and values of 2 heads of 128, whatever the number of layers
    assert CacheStorage.scratch_bytes_per_token_of(model, torch.bfloat16) == 2 * 2 * 128 * 2
    model = model_of(tmp_path, dict(conftest.MID_E, num_hidden_layers=5))
    model.set_cache_bits(4)
    assert CacheStorage.scratch_bytes_per_token_of(model, torch.bfloat16) == 2 * 2 * 128 * 2


def test_a_buffer_that_grows_leaves_its_memory_first(monkeypatch):
    """A buffer that no captured step reads is given up before a larger one takes its place, so that both are never held at a time."""
    from ferrum_b200.engine import batch
    s = batch.Scratch("cpu", guard=0)
    old, held = s.get("grows", (10, 4), torch.float32, limit=1000, captured=False).data_ptr(), []
    real = torch.empty
    monkeypatch.setattr(batch.torch, "empty", lambda *a, **k: held.append("grows" in s._bufs or "grows" in s._views) or real(*a, **k))
    assert s.get("grows", (10, 4), torch.float32, limit=1000, captured=False).data_ptr() == old and not held
    new = s.get("grows", (15, 4), torch.float32, limit=1000, captured=False)
    assert held == [False] and new.shape == (15, 4) and s._bufs["grows"].numel() == 80 and s.generation == 0
    s.get("stays", (4,), torch.float32), s.get("stays", (9,), torch.float32)
    assert s.generation == 2


@pytest.mark.gpu
@pytest.mark.parametrize("bits,a_token", [(None, 2 * 1024), (4, 2 * 288 + 1024)])
def test_pages_fit_the_memory_with_what_they_take_beside_them(cuda, model_dirs, monkeypatch, bits, a_token):
    """The number of pages that follows from the free memory: two layers of 2 heads of 128, and one layer's 16-bit pages where the cache holds 4 bits."""
    from ferrum_b200 import Engine
    room = 3 << 20
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (int(((2 << 30) + room) / 0.85) + 1, 180 << 30))
    eng = Engine(model_dirs["E"], dtype="bfloat16", cache_bits=bits, max_model_len=2048)
    pages = eng.cache.pools[0].shape[1]
    assert pages * 16 * a_token <= room < (pages + 1) * 16 * a_token


@pytest.mark.gpu
def test_engines_that_share_a_model_share_its_cache_bits(cuda, model_dirs):
    """A second engine on a model does not change the cache under the first; one that wants other bits is refused as long as the first lives."""
    import gc

    from ferrum_b200 import Engine
    from ferrum_b200.engine.api import load_model
    from ferrum_b200.errors import ConfigError
    model, _ = load_model(model_dirs["E"], "bfloat16", max_positions=256)
    make = lambda bits: Engine(model=model, cache_bits=bits, num_pages=16, max_model_len=256)
    for mine, other in ((16, 4), (4, 16)):
        first = make(mine)
        want = first.generate([[5, 17, 3]], 6)
        with pytest.raises(ConfigError, match="another engine"):
            make(other)
        second = make(mine)
        assert second.generate([[5, 17, 3]], 6) == want and make(None).generate([[5, 17, 3]], 6) == want
        assert first.generate([[5, 17, 3, 9]], 6) == second.generate([[5, 17, 3, 9]], 6)
        del first, second
        gc.collect()
