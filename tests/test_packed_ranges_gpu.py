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


FACTORS = [(torch.bfloat16, 2.0 ** 20, 2.0 ** -20), (torch.bfloat16, 2.0 ** 60, 2.0 ** -60), (torch.bfloat16, 1.0, 2.0 ** -32), (torch.bfloat16, 2.0 ** 30, 1.0),
           (torch.float16, 2.0 ** 13, 2.0 ** -11)]


@pytest.mark.parametrize("dtype,large,small", FACTORS)
@pytest.mark.parametrize("n", [1, 4])
@pytest.mark.parametrize("kind", ["heads", "halves", "both"])
def test_values_far_apart(cuda, dtype, large, small, n, kind):
    """Query heads of a KV head that look at keys with large and with small values, and heads whose halves are large and small: each row and half keeps
    its own precision.  Compared after a factor that makes the smallest values about one, so that the bound's absolute part is nothing."""
    g = torch.Generator(device="cuda").manual_seed(n)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    L, D = 1100, 128
    side = torch.where(torch.arange(L, device="cuda") % 7 < 3, 1.0, -1.0)
    keys = 0.2 * rand(1, L, D)
    keys[0, :, 0] = 60 * side                                          # (a group of its own range in keys: the other elements of that half are lost in its steps)
    vals = rand(1, L, D)
    if kind != "halves":
        vals *= torch.where(side > 0, large, small)[None, :, None]
    if kind != "heads":
        vals[..., 64:] *= small if kind == "halves" else 2.0 ** -6
    q = 0.5 * rand(n, 4, D)
    q[..., 0] = torch.tensor([30.0, -30.0, 30.0, -30.0], device="cuda")       # scores of +-159: what a head looks away from weighs e^-300
    s = step_over(keys, vals, q, dtype)
    out = s.attend().view(n, 4, D).double()
    assert s.ctx.err.item() == 0
    up = 2.0 ** 6 / small
    want, bound = H.attention(s.qkv[:, :4 * D].view(n, 4, D), s.cache.keys[0], s.cache.vals[0] * up, s.cache.mids[0] * up, L - n, s.mixer.scale, 0, dtype)
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 * up             # (half a step of float16's subnormal numbers)
    over = ((out * up - want).abs() / bound).amax((0, 2)).tolist()
    assert max(over) <= 1, over


@pytest.mark.parametrize("far", [1e9, 1e12, 1e25])
@pytest.mark.parametrize("heads", [1, 4, 7])
def test_a_value_that_no_row_attends_to(cuda, far, heads):
    """However large a value is that no row attends to, in tiles that the rows fill and in tiles that they do not."""
    g = torch.Generator(device="cuda").manual_seed(heads)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    L = 2100
    q = rand(1, 1, 128).repeat(1, heads, 1)
    keys, vals = 0.3 * rand(1, L, 128), rand(1, L, 128)
    keys[0, 37] = -60 * q[0, 0]
    vals[0, 37] *= far
    s = step_over(keys, vals, q, torch.bfloat16)
    s.check(s.attend(), f"{far}")


@pytest.mark.parametrize("large,small", [(1e15, 1e-20), (1e25, 1e-20), (1e10, 1e-25)])
def test_small_values_behind_large_ones(cuda, large, small):
    """Keys with large values, then keys that outweigh them by far with small ones: the sums so far shrink to nothing, the small values keep their bits."""
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    L = 2100
    q = rand(1, 1, 128).repeat(1, 4, 1)
    keys, vals = 0.3 * rand(1, L, 128), rand(1, L, 128)
    keys[0, -500:] += 160 * math.sqrt(128) / q[0, 0].square().sum() * q[0, 0]
    vals[:, :-500] *= large
    vals[:, -500:] *= small
    s = step_over(keys, vals, q, torch.bfloat16)
    out = s.attend().view(1, 4, 128).double()
    want, bound = H.attention(s.qkv[:, :512].view(1, 4, 128), s.cache.keys[0], s.cache.vals[0] / small, s.cache.mids[0] / small, L - 1, s.mixer.scale, 0, torch.bfloat16)
    assert bool(((out / small - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("ahead", [False, True])
def test_many_equal_keys_of_small_weight(cuda, dtype, ahead):
    """60,000 equal keys, each of 2^-15 of one key's weight, whose weights times a step all round the same way; ahead: behind a key of larger values that
    the heavy one then outweighs by 2^10."""
    g = torch.Generator(device="cuda").manual_seed(9)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    L = 60000
    q = rand(1, 1, 128).repeat(1, 4, 1).to(dtype).float()
    keys, vals = torch.zeros(1, L, 128, device="cuda"), rand(1, 1, 128).repeat(1, L, 1)
    one = math.sqrt(128) * math.log(2) / q[0, 0].square().sum() * q[0, 0]            # a score of one power of two
    keys[0, 40] = 15 * one
    vals[0, 40] = rand(128)
    if ahead:
        keys[0, 2], vals[0, 2] = 5 * one, 1000 * rand(128)
    s = step_over(keys, vals, q, dtype)
    s.check(s.attend(), "light keys")


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("n,L", [(1, 1), (1, 200), (3, 70)])
def test_the_largest_values(cuda, dtype, n, L):
    """Groups that reach the type's largest values, whose outermost levels lie beyond it: results are what the values would be, brought back into the type, as
    pages brought back to 16 bits are.  (bfloat16: one key, as float32 sums of more leave float32.)"""
    if dtype == torch.bfloat16 and L > 1:
        L, n = 1, 1
    top = torch.finfo(dtype).max
    vals = torch.zeros(1, L, 128, device="cuda")
    vals[..., :32], vals[..., 32:64] = top, -top
    vals[..., 64:96] = top
    keys = torch.zeros(1, L, 128, device="cuda")
    s = step_over(keys, vals, torch.ones(n, 2, 128, device="cuda"), dtype)
    assert float(s.cache.vals[0].max()) > top
    out = s.attend().view(n, 2, 128).double()
    want = s.cache.vals[0][0, 0].clamp(-top, top)
    assert bool(torch.isfinite(out).all()) and bool(((out - want).abs() <= 2 * H.HALF_STEP[dtype] * top).all())


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("tiles", [1, 2])
@pytest.mark.parametrize("total,new,Hq,Hkv,D,window", [([700], [1], 32, 8, 128, 0), ([300, 5, 2049], [1] * 3, 16, 1, 64, 0), ([90, 200, 31], [2, 1, 2], 14, 2, 128, 0),
                                                       ([500, 20, 77, 600], [4] * 4, 8, 4, 64, 1), ([900, 3, 128], [3, 3, 1], 5, 1, 128, 100),
                                                       ([1 + 13 * i % 200 for i in range(300)], [1 + i % 4 for i in range(300)], 12, 3, 128, 0), ([700, 90, 33], [1, 90, 4], 8, 2, 128, 0)])
def test_either_number_of_tiles(cuda, monkeypatch, dtype, tiles, total, new, Hq, Hkv, D, window):
    """The rule that picks a pass's rows is one of speed: with either number every request's rows are right."""
    from ferrum_b200.ops import lib as ops
    monkeypatch.setattr(ops, "attention_packed_tiles", lambda *few: tiles)
    total = [max(t, n) for t, n in zip(total, new)]
    s = H.Step(H.Cache(total, Hkv, D, 16, dtype, 5), new, Hq, 6, window)
    out = s.attend()
    assert s.ctx.err.item() == 0
    s.check(out, f"{tiles} tiles")


def test_calls_at_the_same_time(cuda):
    """Calls on streams of their own, each with its own workspace and counters, do not disturb each other."""
    from ferrum_b200.ops import lib as ops
    steps, calls = [], []
    for i, (total, new) in enumerate((([30000], [1]), ([700, 90, 2000], [1, 1, 1]), ([4000, 20], [4, 2]), ([300] * 20, [1] * 20))):
        s = H.Step(H.Cache(total, 2, 128, 16, torch.bfloat16, i), new, 8, 10 + i)
        out = torch.empty(s.qkv.shape[0], 8 * 128, dtype=torch.bfloat16, device="cuda")
        part, counters = torch.empty(ops.attention_packed_workspace(128), device="cuda"), torch.zeros(4 * len(new), dtype=torch.int32, device="cuda")
        steps.append((s, out, counters, torch.cuda.Stream()))
        calls.append(lambda s=s, out=out, part=part, counters=counters: ops.attention_packed(
            s.qkv, out, s.qkv.shape[0], s.ctx.block_tables[0], s.ctx.q_start, s.ctx.pos0, s.view.plane, s.view.page_stride, 16, 8, 2, 128, s.mixer.scale, 0, s.ctx.err, part, counters))
    torch.cuda.synchronize()
    for _ in range(20):
        for (_, _, _, stream), call in zip(steps, calls):
            with torch.cuda.stream(stream):
                call()
    torch.cuda.synchronize()
    for i, (s, out, counters, _) in enumerate(steps):
        assert s.ctx.err.item() == 0 and not counters.any()
        s.check(out, f"call {i}")


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("light", [3, 40, 400])
@pytest.mark.parametrize("scale", [0.7, 1.0, 1.9])
def test_middles_of_a_heavy_key(cuda, dtype, light, scale):
    """A key of nearly all the weight whose values are their group's middle, 0, but for two: what the others' small values add up to is left, even elements and odd
    ones.  Two sums, of the codes and of 8, are cut at 2^-17 of 8 steps of the heavy key each, beside the bound of float32 sums."""
    g = torch.Generator(device="cuda").manual_seed(light)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    L = light + 1
    q = rand(1, 1, 128).repeat(1, 4, 1).to(dtype).float()
    keys, vals = 0.02 * rand(1, L, 128), 0.02 * rand(1, L, 128)
    keys[0, 5 % L] += 7 * math.sqrt(128) / q[0, 0].square().sum() * q[0, 0]
    vals[0, 5 % L] = 0
    vals[0, 5 % L, ::64], vals[0, 5 % L, 1::64] = -8 * scale, 7 * scale
    s = step_over(keys, vals, q, dtype)
    out = s.attend().view(1, 4, 128).double()
    want, bound = H.attention(s.qkv[:, :512].view(1, 4, 128), s.cache.keys[0], s.cache.vals[0], s.cache.mids[0], L - 1, s.mixer.scale, 0, dtype)
    assert bool(((out - want).abs() <= bound + 2 * 2.0 ** -17 * 8 * scale).all())
