"""A cache held in 4 bits, as far as it goes without a GPU: layout, plans, refusals."""
import types

import numpy as np
import pytest
import torch

from ferrum_b200.errors import ConfigError, KernelError


def test_block_bytes():
    from ferrum_b200.ops import lib as ops
    assert [ops.packed_block_bytes(d) for d in (64, 128, 32, 96, 256, 0)] == [1152, 2304, 0, 0, 0, 0]


def build(cfg, dtype):
    from ferrum_b200.config import registry
    arch, parsed = registry.read_config(cfg)
    return arch.build(parsed, dtype, "cpu")


def test_layout_of_a_packed_cache(tmp_path):
    import json

    import conftest
    from ferrum_b200.cache import CacheStorage
    folder = tmp_path / "m"
    folder.mkdir()
    (folder / "config.json").write_text(json.dumps(conftest.MID_E))
    model = build(str(folder), torch.bfloat16)
    wide = CacheStorage.bytes_per_token_of(model, torch.bfloat16)
    model.set_cache_bits(4)
    assert CacheStorage.bytes_per_token_of(model, torch.bfloat16) * 32 == wide * 9            # 4.5 bits instead of 16
    cache = CacheStorage(model, torch.bfloat16, "cpu", page_size=32, num_pages=5, max_requests=2, max_model_len=100)
    assert [tuple(p.shape) for p in cache.pools] == [(2, 5, 2, 2, 2304)] and cache.pools[0].dtype == torch.uint8
    view = cache.layer_cache(1)
    assert view.page_stride == 2 * 2 * 2304 and view.plane.data_ptr() == cache.pools[0][1].data_ptr()
    with pytest.raises(ConfigError, match="multiple of 16"):
        CacheStorage(model, torch.bfloat16, "cpu", page_size=24, num_pages=5, max_requests=2, max_model_len=100)
    model.set_cache_bits(16)
    assert CacheStorage.bytes_per_token_of(model, torch.bfloat16) == wide


def test_models_that_cannot_hold_it(tmp_path):
    import json

    import conftest
    import vikupel_configs
    for name, cfg, dtype in (("float32", conftest.MID_E, torch.float32), ("heads of 16", conftest.TINY_A, torch.bfloat16)):
        folder = tmp_path / name.replace(" ", "_")
        folder.mkdir()
        (folder / "config.json").write_text(json.dumps(cfg))
        model = build(str(folder), dtype)
        with pytest.raises(ConfigError, match="4 bits"):
            model.set_cache_bits(4)
        with pytest.raises(ConfigError, match="8 bits"):
            model.set_cache_bits(8)
    folder = tmp_path / "other"
    folder.mkdir()
    (folder / "config.json").write_text(json.dumps(vikupel_configs.VIKUPEL_B))
    with pytest.raises(ConfigError, match="4 bits"):
        build(str(folder), torch.bfloat16).set_cache_bits(4)


def test_pages_of_prompt_portions():
    """unpack_plan names the pages that requests of many rows see, from their window's first key on, and where they go."""
    from ferrum_b200.engine.batch import PlanStore
    from ferrum_b200.parts import attention_plan
    ctx = types.SimpleNamespace(step_cache={}, plan_store=PlanStore("cpu"), n_reqs=4, h_pos0=[100, 70, 0, 33], h_q_len=[1, 20, 40, 9], h2d_bytes=0,
                                block_tables=[torch.zeros(4, 8, dtype=torch.int32)])
    items, table = attention_plan.unpack_plan(ctx, 0, 4, 0, 16, 16)
    assert items.tolist() == [[1, p] for p in range(6)] + [[2, p] for p in range(3)] + [[3, p] for p in range(3)]
    want = np.full((4, 8), -1)
    want[1, :6], want[2, :3], want[3, :3] = range(6), range(6, 9), range(9, 12)
    assert np.array_equal(table.numpy(), want)
    assert attention_plan.unpack_plan(ctx, 0, 4, 0, 16, 16)[0] is items                        # once a step
    items, table = attention_plan.unpack_plan(ctx, 0, 4, 10, 16, 16)
    assert items.tolist() == [[1, 3], [1, 4], [1, 5], [2, 0], [2, 1], [2, 2], [3, 1], [3, 2]]
    assert table[1].tolist() == [-1, -1, -1, 0, 1, 2, -1, -1]


def test_wrappers_refuse_what_the_kernels_are_not_built_for():
    from ferrum_b200.ops import lib as ops
    cpu = torch.zeros(4, 512, dtype=torch.bfloat16)
    i32 = torch.zeros(4, dtype=torch.int32)
    plane = torch.zeros(2, 1, 1, 1152, dtype=torch.uint8)
    with pytest.raises(KernelError, match="CUDA tensor"):
        ops.rope_cache_write_packed(cpu, 4, i32, i32, i32.view(2, 2), None, plane, 1152, 16, 2, 1, 64, 0, 0, i32)
    with pytest.raises(KernelError, match="CUDA tensor"):
        ops.attention_packed(cpu, cpu, 1, i32.view(2, 2), i32, i32, plane, 1152, 16, 2, 1, 64, 1.0, 0, i32, torch.zeros(1), i32)
    lib = ops.lib()
    null = None
    # the library's own checks come before any launch
    assert lib.ferrum_attention_packed(null, 512, null, 512, ops.BF16, null, 1152, 2, 24, null, 4, null, null, 1, 1, null, ops.c_longlong(1 << 40), null, 99, 2, 1, 64,
                                       ops.c_float(1.0), 0, ops.c_void_p(16), null) == 1
    assert b"multiple of 16" in lib.ferrum_last_error()
    assert lib.ferrum_attention_packed(null, 512, null, 512, ops.BF16, null, 1152, 2, 16, null, 4, null, null, 1, 1, null, ops.c_longlong(1 << 40), null, 99, 2, 1, 96,
                                       ops.c_float(1.0), 0, ops.c_void_p(16), null) == 1
    assert b"64 or 128" in lib.ferrum_last_error()
    assert lib.ferrum_unpack_cache(null, 1152, 2, 16, null, 1, 4, null, 1, null, ops.F32, 1, 64, ops.c_void_p(16), null) == 1
    assert b"16-bit" in lib.ferrum_last_error()
    assert lib.ferrum_rope_cache_write_packed(null, ops.BF16, 1, 100, null, 512, null, null, null, 4, null, 0, null, 1152, 2, 16, 2, 1, 64, 0, 0, 1,
                                              ops.c_void_p(16), null) == 1
    assert b"too short" in lib.ferrum_last_error()
