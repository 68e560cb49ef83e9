"""Attention over a cache held in 4 bits near the ends of its types, against 64 bits."""
import math

import pytest
import torch

import packed_helpers as H

pytestmark = pytest.mark.gpu


def step_over(keys, vals, q, dtype, D=128):
    """A `Step` of one request whose cache holds keys, vals (float32 [Hkv, L, D]) and whose last tokens have the queries q ([n, Hq, D])."""
    Hkv, L = keys.shape[:2]
    n, Hq = q.shape[:2]
    c = H.Cache([L], Hkv, D, 16, dtype, 1)
    m = -(-L // 16)
    codes, step, mid = H.quantise(torch.stack([keys, vals]), dtype)
    both = H.values(codes, step, mid)
    c.keys, c.vals, c.mids = [both[0]], [both[1]], [mid[1].double().repeat_interleave(64, -1)]
    pad = lambda t: torch.cat([t, torch.zeros(*t.shape[:2], 16 * m - L, t.shape[-1], dtype=t.dtype, device="cuda")], 2).unflatten(2, (m, 1, 16)).transpose(1, 2)
    c.plane[c.table[0].long()] = H.block_bytes(*[[pad(t)[i] for t in (codes, step, mid)] for i in (0, 1)], dtype)
    s = H.Step(c, [n], Hq, 2)
    s.qkv[:, :Hq * D] = q.reshape(n, Hq * D).to(dtype)
    return s


# exponents of the queries, of the keys: their product is about one, or (the keys' exponent 0) far above or below
@pytest.mark.parametrize("dtype,up,down", [(torch.bfloat16, u, -u) for u in (100, 114, 116, 120, 124, -100, -116, -122)] +
                         [(torch.float16, 13, -10), (torch.float16, -18, 12), (torch.float16, -22, 12)])
@pytest.mark.parametrize("n,L", [(1, 300), (3, 1000)])
def test_queries_of_every_size(cuda, dtype, up, down, n, L):
    """Rows of queries next to the type's largest and smallest numbers over keys that make their scores ordinary ones."""
    g = torch.Generator(device="cuda").manual_seed(L)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, keys = rand(n, 4, 128).clamp(-3.9, 3.9) * 2.0 ** up, rand(1, L, 128) * 2.0 ** down
    s = step_over(keys, rand(1, L, 128), q, dtype)
    s.check(s.attend(), f"queries of 2^{up}")


@pytest.mark.parametrize("n", [1, 3])
def test_a_row_far_larger_than_the_others(cuda, n):
    """bfloat16 rows 2^60 and 2^110 apart in one tile: each is right for itself."""
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    for up, k in ((60, -55), (110, -105)):
        q = rand(n, 4, 128).clamp(-3.9, 3.9)
        q[:, 1] *= 2.0 ** up
        s = step_over(rand(1, 500, 128) * 2.0 ** k, rand(1, 500, 128), q, torch.bfloat16)
        s.check(s.attend(), f"rows 2^{up} apart")


@pytest.mark.parametrize("up", [112, 116, 119])
def test_scores_next_to_the_largest_number(cuda, up):
    """Ordinary keys under queries that are next to bfloat16's largest: the key with the largest score is all that counts, its value comes out."""
    g = torch.Generator(device="cuda").manual_seed(up)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, keys = rand(2, 4, 128).clamp(-3.9, 3.9) * 2.0 ** up, rand(1, 400, 128)
    s = step_over(keys, rand(1, 400, 128), q, torch.bfloat16)
    scores = torch.einsum("nhd,ld->nhl", s.qkv[:, :512].double().view(2, 4, 128), s.cache.keys[0][0])
    scores[0, :, 399] = -math.inf                   # (the first token does not see the second's key)
    best = scores.topk(2, -1)
    assert bool((best.values[..., 0] - best.values[..., 1] > 1e-4 * best.values[..., 0]).all())
    want = s.cache.vals[0][0][best.indices[..., 0]]
    got = s.attend().view(2, 4, 128).double()
    # a weight of one exactly; the step times it has a float16's 11 bits, the result a bfloat16's 8
    assert bool(((got - want).abs() <= (H.HALF_STEP[torch.bfloat16] + 2.0 ** -11) * (want.abs() + s.cache.mids[0].abs().max()) + 1e-7).all())


@pytest.mark.parametrize("dtype,up", [(torch.bfloat16, u) for u in (12, 20, 40, 90)] + [(torch.float16, 12), (torch.float16, 14)])
@pytest.mark.parametrize("n", [1, 4])
def test_equal_scores_far_from_zero(cuda, dtype, up, n):
    """A few equal keys whose scores, up to 2^97, leave all others behind: whatever float32 makes of such a score, it is the same for each, and the result is the
    mean of their values."""
    g = torch.Generator(device="cuda").manual_seed(up)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q = rand(1, 1, 128).repeat(n, 4, 1)
    keys, vals = 0.1 * rand(1, 1500, 128), rand(1, 1500, 128)
    at = torch.tensor([3, 4, 70, 701, 702, 1333, 1490], device="cuda")
    scale_up = 2.0 ** min(up, 12)
    keys[0, at] = 3 * q[0, 0]
    s = step_over(keys * scale_up, vals, q * 2.0 ** (up - min(up, 12) + (0 if dtype == torch.bfloat16 else 8)), dtype)
    picked = s.cache.vals[0][0, at]
    # seven weights of one: each step times it has a float16's 11 bits, the result the type's own
    part = ((picked - s.cache.mids[0][0, at]).abs() + s.cache.mids[0][0, at].abs()).mean(0)
    out = s.attend().view(n * 4, 128).double()
    assert bool(((out - picked.mean(0)).abs() <= 2.0 ** -11 * part + H.HALF_STEP[dtype] * picked.mean(0).abs() * 1.01 + 1e-6).all())
