"""What the operators of a cache held in 4 bits refuse before anything is launched."""
import types

import pytest
import torch

from ferrum_b200.errors import KernelError


def test_the_library_wants_an_error_flag():
    from ferrum_b200.ops import lib as ops
    lib, null = ops.lib(), None
    # (no tokens, no items: there would be nothing to launch)
    assert lib.ferrum_rope_cache_write_packed(null, ops.BF16, 0, 512, null, 512, null, null, null, 4, null, 0, 16, 1152, 2, 16, 2, 1, 64, 0, 0, 1, null, null) == 1
    assert b"error flag" in lib.ferrum_last_error()
    assert lib.ferrum_unpack_cache(null, 1152, 2, 16, null, 1, 4, null, 0, null, ops.BF16, 1, 64, null, null) == 1
    assert b"error flag" in lib.ferrum_last_error()


@pytest.fixture
def calls(monkeypatch):
    """The wrappers over a library that only notes its calls, with tensors of this machine in the place of the GPU's."""
    from ferrum_b200.ops import lib as ops
    made = []

    def need(t, dtype, name, ndim=None):
        if not isinstance(t, torch.Tensor) or (dtype is not None and t.dtype != dtype) or (ndim is not None and t.dim() != ndim):
            raise KernelError(f"{name} is not as it must be")

    def dense(t, dtype, name, ndim):
        need(t, dtype, name, ndim)
        return t.data_ptr()
    ops.packed_block_bytes(64), ops.attention_packed_rows()
    entry = lambda name: lambda *a: made.append((name, a)) or 0
    fake = types.SimpleNamespace(**{n: entry(n) for n in ("ferrum_rope_cache_write_packed", "ferrum_unpack_cache", "ferrum_attention_packed")})
    monkeypatch.setattr(ops, "_need", need)
    monkeypatch.setattr(ops, "_dense", dense)
    monkeypatch.setattr(ops, "_stream_at", lambda: 0)
    monkeypatch.setattr(ops, "lib", lambda: fake)
    return made


def operators(ops):
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    plane, x = torch.zeros(2, 1, 1, 1152, dtype=torch.uint8), torch.zeros(1, 256, dtype=torch.bfloat16)
    return {"write": lambda err: ops.rope_cache_write_packed(x, 1, i32(1), i32(1), i32(1, 2), None, plane, 1152, 16, 2, 1, 64, 0, 0, err),
            "unpack": lambda err: ops.unpack_cache(plane, 1152, 16, i32(1, 2), i32(1, 2), torch.zeros(1, 2, 1, 16, 64, dtype=torch.bfloat16), err),
            "attention": lambda err: ops.attention_packed(x, torch.zeros_like(x), 1, i32(1, 2), i32(2), i32(1), plane, 1152, 16, 2, 1, 64, 1.0, 0, err, torch.zeros(1), i32(2))}


@pytest.mark.parametrize("name", ["write", "unpack", "attention"])
def test_the_error_flag_is_looked_at(calls, name):
    from ferrum_b200.ops import lib as ops
    call = operators(ops)[name]
    call(torch.zeros(1, dtype=torch.int32))
    assert len(calls) == 1
    for err in (None, torch.zeros(1), torch.zeros(1, dtype=torch.int64), 16, torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(KernelError, match="err"):
            call(err)
    assert len(calls) == 1


def test_tiles_follow_the_rows_of_the_requests_that_are_read(calls):
    """The kernel is chosen by the rows of the requests that it reads, not by a step's other tokens."""
    from ferrum_b200.ops import lib as ops
    assert [ops.attention_packed_tiles(*f) for f in ((1, 1), (64, 64), (65, 64), (96, 64), (97, 64), (128, 64), (2, 1))] == [1, 1, 1, 1, 2, 2, 2]
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    x, plane = torch.zeros(40, 256, dtype=torch.bfloat16), torch.zeros(2, 1, 1, 1152, dtype=torch.uint8)
    call = lambda tokens, requests, Hq, few=None: ops.attention_packed(x, torch.zeros_like(x), tokens, i32(requests, 2), i32(requests + 1), i32(requests), plane, 1152, 16, Hq, 1, 64,
                                                                       1.0, 0, i32(1), torch.zeros(1), i32(2 * requests), few=few)
    for tokens, requests, Hq, few, tiles in ((4, 4, 2, None, 1), (8, 4, 2, None, 2), (4, 4, 16, None, 2), (3, 4, 2, None, 1), (40, 4, 2, (3, 3), 1), (40, 4, 2, (6, 3), 2)):
        calls.clear()
        call(tokens, requests, Hq, few)
        assert len(calls) == 1 and calls[0][1][14] == tiles
    calls.clear()
    call(0, 4, 2), call(40, 1, 2, (0, 0))
    assert not calls


@pytest.mark.parametrize("G,new,few", [(4, [1] * 64 + [512], (64, 64)), (4, [1] * 63 + [3, 70, 90], (65, 64)), (8, [1, 2, 0, 3], (3, 2)), (4, [1, 2, 2], (3, 3)), (16, [1, 40], (2, 1))])
def test_a_step_with_portions_of_prompts_names_its_decoded_tokens(monkeypatch, G, new, few):
    from ferrum_b200.ops import lib as ops
    from ferrum_b200.parts.attention import PagedAttention
    seen = []

    class Enough(Exception):
        pass

    def attention(*a, few=None):
        seen.append(few)
        raise Enough
    monkeypatch.setattr(ops, "attention_packed", attention)
    mixer = PagedAttention(G * 64, G, 1, 64, None, torch.bfloat16)
    mixer.set_cache_bits(4)
    ctx = types.SimpleNamespace(step_cache={}, h_q_len=new, max_q_len=max(new), n_reqs=len(new), n_tokens=sum(new), q_start=None, pos0=None, err=None, block_tables=[None],
                                buf=lambda *a: None, zeros=lambda *a: None)
    cache = types.SimpleNamespace(group=0, plane=None, page_stride=1152, page_size=16)
    with pytest.raises(Enough):
        mixer.attend(torch.zeros(1, 1, dtype=torch.bfloat16), None, ctx, cache)
    assert seen == [few]
