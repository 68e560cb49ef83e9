"""A cache held in 4 bits: the write, the way back to 16 bits, and attention over it, against plain implementations in 64 bits."""
import math

import pytest
import torch

import packed_helpers as H

pytestmark = pytest.mark.gpu


def err_flag():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def write(x, Hq, Hkv, D, page, positions, request, table, cos_sin, R, pairing, plane, q_out=None, write_kv=True):
    from ferrum_b200.ops import lib as ops
    err = err_flag()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    ops.rope_cache_write_packed(x, x.shape[0], i32(positions), i32(request), table, cos_sin, plane, plane.stride(0), page, Hq, Hkv, D, R, pairing, err,
                                q_out=q_out, write_kv=write_kv)
    return err.item()


def rotary(n, R):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))
    return torch.stack([angle.cos(), angle.sin()], -1).float().cuda()


def turned(x, cos_sin, positions, R, pairing):
    """float32 rows [T, heads, D] after the rotation, an operation at a time."""
    x = x.float().clone()
    if R == 0:
        return x
    cs = cos_sin[torch.tensor(positions, device="cuda")][:, None]
    first = slice(0, R, 2) if pairing == 0 else slice(0, R // 2)
    second = slice(1, R, 2) if pairing == 0 else slice(R // 2, R)
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]
    return x


# one token and many; heads in groups and alone; the rotary table over all, part or none of a head, both pairings; an odd rotated half
@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("T,Hq,Hkv,D,page,R,pairing", [(1, 4, 2, 128, 16, 128, 1), (37, 3, 1, 64, 32, 64, 0), (130, 8, 8, 128, 48, 64, 0),
                                                       (3, 6, 2, 64, 16, 0, 1), (65, 5, 5, 64, 64, 34, 1), (18, 2, 1, 128, 16, 6, 0), (9, 2, 2, 128, 16, 10, 1)])
def test_write_is_the_definition(cuda, dtype, T, Hq, Hkv, D, page, R, pairing):
    """Codes, pairs and turned queries equal the definition bit for bit; all other bytes of the pages stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(T)
    x = (3 * torch.randn(T, (Hq + 2 * Hkv) * D, device="cuda", generator=g)).to(dtype)
    first = 11
    positions = list(range(first, first + T))
    n_pages = -(-(first + T) // page)
    table = torch.arange(n_pages, dtype=torch.int32, device="cuda").flip(0).contiguous()[None]
    plane = torch.randint(0, 256, (n_pages + 1, Hkv, page // 16, 18 * D), dtype=torch.uint8, device="cuda", generator=g)
    before, cos_sin = plane.clone(), rotary(first + T, R) if R else None
    q_out = torch.full((T + 1, Hq * D + 8), 7, dtype=dtype, device="cuda")
    keep = x.clone()
    assert write(x, Hq, Hkv, D, page, positions, [0] * T, table, cos_sin, R, pairing, plane, q_out=q_out) == 0
    assert torch.equal(x, keep)
    rows = x.view(T, -1, D)
    qk = turned(rows[:, :Hq + Hkv], cos_sin, positions, R, pairing)
    assert torch.equal(q_out[:T, :Hq * D], qk[:, :Hq].reshape(T, -1).to(dtype))
    assert bool((q_out[T] == 7).all()) and bool((q_out[:, Hq * D:] == 7).all())
    # the expected plane: the old one with this step's rows put in
    row = D // 2
    for part, src in ((0, qk[:, Hq:]), (1, rows[:, Hq + Hkv:].float())):
        codes, step, mid = H.quantise(src, dtype)
        c = codes.to(torch.uint8)
        c = c[..., ::2] + 16 * c[..., 1::2]
        pair = torch.stack([step, mid], -1).contiguous().view(torch.uint8).flatten(-2)
        for i, pos in enumerate(positions):
            b = before[table[0, pos // page], :, pos % page // 16]
            at, size = pos % 16, pair.shape[-1]
            b[:, part * 16 * row + at * row:part * 16 * row + (at + 1) * row] = c[i]
            o = 16 * D + part * 16 * size + at * size
            b[:, o:o + size] = pair[i]
    assert torch.equal(plane, before)
    # in place, as the mixer calls it, and without a cache write
    assert write(x, Hq, Hkv, D, page, positions, [0] * T, table, cos_sin, R, pairing, plane, write_kv=False) == 0
    assert torch.equal(x[:, :Hq * D], q_out[:T, :Hq * D]) and torch.equal(x[:, (Hq + Hkv) * D:], keep[:, (Hq + Hkv) * D:])
    assert torch.equal(plane, before)


@pytest.mark.parametrize("T,Hq,Hkv,D,R,pairing", [(221, 6, 3, 128, 128, 1), (223, 6, 3, 128, 128, 1), (700, 30, 5, 64, 32, 0)])
def test_write_of_many_tokens_is_the_definition(cuda, T, Hq, Hkv, D, R, pairing):
    """As above on both sides of where a warp starts to take several heads of a token."""
    for dtype in H.DTYPES:
        test_write_is_the_definition(cuda, dtype, T, Hq, Hkv, D, 32, R, pairing)


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("kind", ["halves", "next to halves", "subnormal steps", "all sizes"])
def test_codes_next_to_halves(cuda, dtype, kind):
    """Values half way between two levels go to the even one, values next to that to theirs; steps below the smallest normal number and of all sizes."""
    D, page, T = 128, 16, 800
    g = torch.Generator(device="cuda").manual_seed(5)
    v = torch.randint(0, 31, (T, D), device="cuda", generator=g).float()         # range 30: a step of 2, every odd value half way
    v[:, ::64], v[:, 1::64] = 0.0, 30.0
    if kind == "next to halves":                                                 # (the type's next number up or down)
        v = v.to(dtype)
        v = (v.view(torch.int16) + torch.randint(-1, 2, (T, D), device="cuda", generator=g).to(torch.int16) * (v > 0)).view(dtype).float()
    elif kind == "subnormal steps":
        v = v * (2.0 ** -131 if dtype == torch.bfloat16 else 2.0 ** -19)
    elif kind == "all sizes":
        e = torch.randint(-100 if dtype == torch.bfloat16 else -12, 100 if dtype == torch.bfloat16 else 12, (T, 1), device="cuda", generator=g)
        v = torch.randn(T, D, device="cuda", generator=g) * 2.0 ** e
    x = torch.cat([torch.zeros(T, D, device="cuda"), v, v.flip(0)], 1).to(dtype)
    table, plane = torch.arange(T // page, dtype=torch.int32, device="cuda")[None], torch.zeros(T // page, 1, 1, 18 * D, dtype=torch.uint8, device="cuda")
    assert write(x, 1, 1, D, page, list(range(T)), [0] * T, table, None, 0, 0, plane) == 0
    cut = lambda t: t.unflatten(0, (T // page, 1, 1, 16))
    want = H.block_bytes(*[[cut(t) for t in H.quantise(x[:, part * D:(part + 1) * D].float(), dtype)] for part in (1, 2)], dtype)
    assert torch.equal(plane, want)


@pytest.mark.parametrize("dtype", H.DTYPES)
def test_write_of_special_values(cuda, dtype):
    """Constant groups come back exactly, as does a group of zeros; a NaN or an infinity spoils its own group alone; the type's largest
    values neither overflow nor leave their range; the error of every element is at most half a step, and a step's and a middle's own rounding."""
    from ferrum_b200.ops import lib as ops
    D, page, T = 128, 16, 9
    g = torch.Generator(device="cuda").manual_seed(3)
    v = torch.randn(T, D, device="cuda", generator=g)
    top = torch.finfo(dtype).max
    v[0] = 0.0
    v[1, :64], v[1, 64:] = 1.5, -0.3
    v[2, 5] = math.nan
    v[3, 70] = math.inf
    v[4, 3] = -math.inf
    v[5, :64] = top; v[5, :32] = -top
    v[6] *= 1e-30 if dtype == torch.bfloat16 else 1e-6
    v[7, 0] = 1000.0
    v[8] = 100.0 + 0.25 * v[8]
    x = torch.cat([torch.zeros(T, 2 * D, device="cuda"), v], 1).to(dtype)
    table, plane = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, 1, 18 * D, dtype=torch.uint8, device="cuda")
    assert write(x, 1, 1, D, page, list(range(T)), [0] * T, table, None, 0, 0, plane) == 0
    back, err = torch.empty(1, 2, 1, page, D, dtype=dtype, device="cuda"), err_flag()
    ops.unpack_cache(plane, plane.stride(0), page, table, torch.zeros(1, 2, dtype=torch.int32, device="cuda"), back, err)
    got, want = back[0, 1, 0, :T].double(), x[:, 2 * D:].double()
    assert err.item() == 0 and torch.equal(got[:2], want[:2]) and not back[0, 0, 0].any()
    groups = torch.isfinite(got).view(T, 2, 64)
    spoiled = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    spoiled[2, 0] = spoiled[3, 1] = spoiled[4, 0] = True
    assert torch.equal(groups.all(-1), ~spoiled) and torch.equal(groups.any(-1), ~spoiled)
    fine = ~spoiled
    w, b = want.view(T, 2, 64)[fine], got.view(T, 2, 64)[fine]
    step = (w.amax(-1) - w.amin(-1)) / 15
    h = H.HALF_STEP[dtype]
    tiny = torch.finfo(dtype).smallest_normal * 2 * h          # a subnormal step is off by up to half the type's smallest number
    lim = step * (0.5 + 16 * h) + h * w.abs().amax(-1) * 3 + 16 * tiny
    assert bool(((w - b).abs().amax(-1) <= lim).all())


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("D,Hkv,page", [(64, 3, 16), (128, 1, 48), (128, 2, 64)])
def test_unpack(cuda, dtype, D, Hkv, page):
    """Every element is its value rounded once; a page that is missing or outside the plane arrives as zeros and raises error 5."""
    from ferrum_b200.ops import lib as ops
    c = H.Cache([5 * page], Hkv, D, page, dtype, 1, fill=0)
    for items, wrong in (([[0, 4], [0, 0], [0, 2]], []), ([[0, 1], [0, 6], [0, 3]], [1])):
        table = torch.cat([c.table, torch.tensor([[-1, -1, 1000]], dtype=torch.int32, device="cuda")], 1)
        err, out = err_flag(), torch.full((len(items) + 1, 2, Hkv, page, D), 5, dtype=dtype, device="cuda")
        ops.unpack_cache(c.plane, c.plane.stride(0), page, table, torch.tensor(items, dtype=torch.int32, device="cuda"), out, err)
        assert err.item() == (5 if wrong else 0) and bool((out[-1] == 5).all())
        for i, (_, lp) in enumerate(items):
            want = torch.zeros(2, Hkv, page, D, dtype=torch.float64, device="cuda")
            if i not in wrong:
                want[0], want[1] = (t[0][:, lp * page:(lp + 1) * page] for t in (c.keys, c.vals))
            assert torch.equal(out[i], want.to(dtype))
    err = err_flag()
    ops.unpack_cache(c.plane, c.plane.stride(0), page, table, torch.tensor([[0, 7], [0, 90], [7, 0]], dtype=torch.int32, device="cuda"),
                     torch.empty(3, 2, Hkv, page, D, dtype=dtype, device="cuda"), err)
    assert err.item() == 5


# (lengths in all, new tokens, Hq, Hkv, D, page, window): one key; lengths around a block, a page and a tile; groups of 1 to 16 heads; several
# tokens a request; windows inside a block, across pages and beyond the context
DECODE = [([1], [1], 4, 2, 64, 16, 0), ([16, 17, 15, 1, 2], [1] * 5, 8, 1, 128, 16, 0), ([63, 64, 65, 128, 129, 1000], [1] * 6, 6, 3, 128, 16, 0),
          ([700], [1], 32, 8, 128, 16, 0), ([300, 5, 2049], [1] * 3, 16, 1, 64, 64, 0), ([40, 333], [1, 3], 4, 1, 128, 48, 0),
          ([90, 200, 16], [16, 5, 16], 2, 2, 64, 16, 0), ([90, 200, 31], [2, 1, 2], 14, 2, 128, 32, 0), ([500, 20, 77], [1] * 3, 8, 4, 128, 16, 30),
          ([500, 20, 77, 600], [4] * 4, 8, 4, 64, 16, 1), ([900, 3, 128], [3, 3, 1], 5, 1, 128, 16, 100), ([5000, 40], [1] * 2, 4, 4, 128, 32, 3000),
          ([20000], [1], 8, 2, 128, 64, 0), ([260] * 40, [1] * 40, 8, 8, 64, 16, 0),
          # more requests than a block has threads, with fewer and with more (request, head) pairs than CTAs; a long context among short ones;
          # rows in two tiles of eight
          ([1 + 7 * i % 90 for i in range(200)], [1] * 200, 4, 1, 64, 16, 0), ([1 + 13 * i % 200 for i in range(300)], [1] * 300, 6, 3, 128, 16, 0),
          ([30000] + [50] * 30, [1] * 31, 8, 2, 64, 64, 0), ([9000] + [70] * 100, [1] * 101, 8, 8, 128, 32, 0), ([4000, 3, 50, 900], [2, 0, 0, 1], 8, 1, 64, 16, 0)]


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decoded_tokens(cuda, dtype, case):
    total, new, Hq, Hkv, D, page, window = DECODE[case]
    s = H.Step(H.Cache(total, Hkv, D, page, dtype, case), new, Hq, 100 + case, window)
    out = s.attend()
    assert s.ctx.err.item() == 0
    s.check(out, f"case {case}")
    assert torch.equal(out, s.attend()) and not any(t.any() for t in s.ctx._zeros.values())        # the same twice, the counters left as they were


PROMPT = [([40], [40], 8, 2, 64, 16, 0), ([300], [300], 4, 4, 128, 16, 0), ([700, 90, 33], [200, 90, 17], 8, 8, 128, 32, 0),
          ([700, 513, 60], [150, 1, 60], 12, 4, 64, 16, 100), ([130, 1, 5], [50, 1, 5], 32, 1, 64, 48, 0)]


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("case", range(len(PROMPT)))
def test_prompt_portions(cuda, dtype, case):
    """Portions of prompts, alone and beside decoded tokens in one step."""
    total, new, Hq, Hkv, D, page, window = PROMPT[case]
    s = H.Step(H.Cache(total, Hkv, D, page, dtype, case), new, Hq, 100 + case, window)
    out = s.attend()
    assert s.ctx.err.item() == 0
    s.check(out, f"case {case}")


@pytest.mark.parametrize("dtype", H.DTYPES)
def test_scores_far_apart(cuda, dtype):
    """Scores of hundreds: the largest wins, nothing overflows."""
    c = H.Cache([333, 20], 2, 128, 16, dtype, 5, spread=4.0, offset=3.0)
    s = H.Step(c, [1, 2], 8, 6)
    s.qkv *= 12
    s.check(s.attend(), "large scores")


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("kind", ["zeros", "constant", "growing", "shrinking", "tiny", "far offset"])
@pytest.mark.parametrize("new", [[1, 1], [4, 2]])
def test_values_of_many_sizes(cuda, dtype, kind, new):
    """Groups without a range (steps of 0), steps that grow or shrink by orders of magnitude along a context, very small ones, values far from 0."""
    spread, offset = {"zeros": (0.0, 0.0), "constant": (0.0, 1.0), "tiny": (1e-5, 1e-5), "far offset": (0.1, 30.0)}.get(kind, (1.0, 1.0))
    size = None
    if kind in ("growing", "shrinking"):
        size = lambda m: 10.0 ** torch.linspace(-4, 3, m, device="cuda").flip(0 if kind == "shrinking" else ())
    c = H.Cache([900, 70], 2, 128, 16, dtype, 31, spread=spread, offset=offset, size=size)
    s = H.Step(c, new, 8, 32)
    s.check(s.attend(), kind)


@pytest.mark.parametrize("dtype", H.DTYPES)
@pytest.mark.parametrize("seen", ["never", "first"])
def test_a_value_far_larger_than_the_others(cuda, dtype, seen):
    """A value 10^4 (float16) or 10^7 times as large as the others under a key that no row attends to, or that was the best one seen before a far better
    one came: the others' weights keep their precision."""
    far = 1e4 if dtype == torch.float16 else 1e7
    c = H.Cache([2100], 1, 128, 16, dtype, 41, spread=0.3, offset=0.0)
    s = H.Step(c, [1], 4, 42)
    # the key at 37 is the negative query, so that its score is far below all others; or (first) the query, and the last 500 keys are twice that
    q = s.qkv[0, :128].float()
    s.qkv[:, :512] = s.qkv[:, :128].repeat(1, 4)
    kv = torch.stack([c.keys[0].float(), c.vals[0].float()])                       # [2, 1, 2100, 128]
    kv[0, 0, 37] = -8 * q if seen == "never" else 4 * q
    if seen == "first":
        kv[0, 0, -500:] += 8 * q
    kv[1, 0, 37] *= far
    codes, step, mid = H.quantise(kv, dtype)
    vals = H.values(codes, step, mid)
    c.keys, c.vals, c.mids = [vals[0]], [vals[1]], [mid[1].double().repeat_interleave(64, -1)]
    pad = lambda t: torch.cat([t, torch.zeros(2, 1, 12, t.shape[-1], dtype=t.dtype, device="cuda")], 2).unflatten(2, (132, 1, 16)).transpose(1, 2)
    c.plane[c.table[0].long()] = H.block_bytes(*[[pad(t)[i] for t in (codes, step, mid)] for i in (0, 1)], dtype)
    s.check(s.attend(), seen)


@pytest.mark.parametrize("small", [1e-20, 1e-31, 1e-34])
@pytest.mark.parametrize("kind", ["all", "the best keys'", "the best keys', of large ones"])
def test_values_near_the_smallest(cuda, kind, small):
    """bfloat16 values down to the smallest normal steps: all of them, or those of the last 500 keys, whose scores are ten above the others' (so that the
    others' values make the result all the same).  Compared after a factor that makes the result about one."""
    c = H.Cache([2100], 1, 128, 16, torch.bfloat16, 43, spread=0.3, offset=0.0)
    s = H.Step(c, [1], 4, 44)
    q = s.qkv[0, :128].float()
    s.qkv[:, :512] = s.qkv[:, :128].repeat(1, 4)
    kv = torch.stack([c.keys[0].float(), c.vals[0].float()])
    kv[0, 0, -500:] += 10 / (s.mixer.scale * q.square().sum()) * q
    large = 1e15 if kind.endswith("large ones") else 1.0
    kv[1, 0, :1600] *= small if kind == "all" else large
    kv[1, 0, 1600:] *= small
    codes, step, mid = H.quantise(kv, torch.bfloat16)
    assert bool((step[1].float() >= torch.finfo(torch.bfloat16).smallest_normal).all())
    pad = lambda t: torch.cat([t, torch.zeros(2, 1, 12, t.shape[-1], dtype=t.dtype, device="cuda")], 2).unflatten(2, (132, 1, 16)).transpose(1, 2)
    c.plane[c.table[0].long()] = H.block_bytes(*[[pad(t)[i] for t in (codes, step, mid)] for i in (0, 1)], torch.bfloat16)
    up = 1 / small if kind == "all" else 1e5 / large
    vals = H.values(codes, step, mid)
    want, bound = H.attention(s.qkv[:1, :512].view(1, 4, 128), vals[0], vals[1] * up, mid[1].double().repeat_interleave(64, -1) * up, 2099, s.mixer.scale, 0, torch.bfloat16)
    got = s.attend().view(1, 4, 128).double() * up
    assert bool(((got - want).abs() <= bound).all()), ((got - want).abs() / bound).max().item()


@pytest.mark.parametrize("where", [-1, -1000, 16 * 13 - 1, 10 ** 6, 2 ** 31 - 1])
@pytest.mark.parametrize("n_reqs", [2, 40])
def test_positions_beyond_the_table_raise_the_flag(cuda, where, n_reqs):
    """A request whose keys no page of the table could hold raises error 5; the other requests' rows stay right."""
    c = H.Cache([100, 200] + [30] * (n_reqs - 2), 2, 128, 16, torch.float16, 4)
    assert c.width == 13
    s = H.Step(c, [1, 2] + [1] * (n_reqs - 2), 8, 5)
    s.ctx.pos0[1] = where
    out = s.attend()
    assert s.ctx.err.item() == 5
    keep = [0] + list(range(3, n_reqs + 1))
    s.new[1], s.qkv = 0, s.qkv[keep]
    s.check(out[keep])


def test_out_in_the_place_of_q_is_refused(cuda):
    from ferrum_b200.ops import lib as ops
    c = H.Cache([100], 2, 64, 16, torch.bfloat16, 8)
    s = H.Step(c, [1], 8, 9)
    part, counters = torch.empty(ops.attention_packed_workspace(64), device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ops.KernelError, match="out must not be q"):
        ops.attention_packed(s.qkv, s.qkv, 1, s.ctx.block_tables[0], s.ctx.q_start, s.ctx.pos0, c.plane, c.plane.stride(0), 16, 8, 2, 64, 0.125, 0, s.ctx.err, part, counters)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-4, 3.0])
def test_score_scales(cuda, scale):
    for new in ([1, 1], [3, 2], [40, 1]):
        s = H.Step(H.Cache([300, 77], 2, 64, 16, torch.float16, 33), new, 8, 34)
        s.mixer.scale = scale
        s.check(s.attend(), f"scale {scale}")


@pytest.mark.parametrize("new,window", [([1, 2], 0), ([2, 4], 40)])
def test_nan_in_hidden_places_stays_there(cuda, new, window):
    """Keys and values that a row does not see (behind it in its own request, ahead of its window, on pages of nobody) may be NaN; a NaN that a
    row sees spoils that row alone."""
    c = H.Cache([200, 333], 2, 128, 16, torch.bfloat16, 35, fill=255)
    s = H.Step(c, new, 8, 36, window)
    want = s.attend()
    s.check(want, "hidden")
    pairs = c.plane.view(torch.bfloat16)                        # a block: 16 * D / 2 pairs' worth of codes first
    at = lambda pos: (int(c.table[1, pos // 16].item()), slice(None), pos % 16 // 16, slice(8 * 128 + pos % 16 * 4, 8 * 128 + pos % 16 * 4 + 4))
    if window:
        pairs[at(333 - 4 - window - 1)] = float("nan")          # ahead of every row's window
        assert torch.equal(s.attend(), want)
        pairs[at(333 - 4 - window + 1)] = float("nan")          # the first row sees it, the others do not
        out = s.attend()
        assert torch.isnan(out[2]).all() and torch.equal(out[[0, 1, 3, 4, 5]], want[[0, 1, 3, 4, 5]])
    else:
        pairs[at(332)] = float("nan")                           # the last token's own key: hidden from the one before it
        out = s.attend()
        assert torch.equal(out[:2], want[:2]) and torch.isnan(out[2]).all()


def test_rows_of_other_requests_and_wider_rows(cuda):
    """attention_packed leaves the rows of requests with many rows, and of no request, as they were; rows may lie apart."""
    from ferrum_b200.ops import lib as ops
    c = H.Cache([100, 60, 40], 2, 64, 16, torch.bfloat16, 8)
    s = H.Step(c, [1, 50, 4], 8, 9, extra_columns=24)
    s.qkv[:, -24:] = float("nan")
    out = torch.full((60, 8 * 64 + 8), 3, dtype=torch.bfloat16, device="cuda")
    part, counters = torch.empty(ops.attention_packed_workspace(64), device="cuda"), torch.zeros(12, dtype=torch.int32, device="cuda")
    ops.attention_packed(s.qkv, out, 55, s.ctx.block_tables[0], s.ctx.q_start, s.ctx.pos0, c.plane, c.plane.stride(0), 16, 8, 2, 64, 0.125, 0, s.ctx.err, part, counters)
    assert s.ctx.err.item() == 0 and not counters.any() and bool((out[1:51] == 3).all()) and bool((out[55:] == 3).all()) and bool((out[:, 512:] == 3).all())
    want = s.attend()
    for rows in (slice(0, 1), slice(51, 55)):
        assert torch.equal(out[rows, :512], want[rows])


def test_missing_pages_raise_the_flag(cuda):
    """A key's page that the table does not name, or that lies outside the plane, raises error 5; the other requests' rows stay right."""
    for wrong in (-1, 10 ** 6):
        c = H.Cache([100, 200], 2, 128, 16, torch.float16, 4)
        s = H.Step(c, [1, 1], 8, 5)
        s.ctx.block_tables[0][1, 3] = wrong
        out = s.attend()
        assert s.ctx.err.item() == 5
        s.new, s.past = s.new[:1], s.past[:1]
        s.check(out[:1])


def test_write_refuses_positions_without_a_page(cuda):
    D, page = 64, 16
    x = torch.ones(1, 3 * D, device="cuda").bfloat16()
    for pos, table, R, code in ((40, [0, 1], 0, 3), (5, [-1, 1], 0, 4), (20, [0, 7], 0, 4), (9, [0, 1], 64, 2), (-1, [0, 1], 0, 2)):
        plane = torch.full((2, 1, 1, 18 * D), 9, dtype=torch.uint8, device="cuda")
        assert write(x, 1, 1, D, page, [pos], [0], torch.tensor([table], dtype=torch.int32, device="cuda"), rotary(9, 64) if R else None, R, 0, plane) == code
        assert bool((plane == 9).all())


def test_another_stream_and_a_replayed_graph(cuda):
    """A captured call reads the lengths, tables and pages of the time it is replayed; a call on another stream is ordered by that stream."""
    c = H.Cache([700, 40, 260], 2, 128, 16, torch.bfloat16, 20)
    s = H.Step(c, [1, 1, 1], 8, 21)
    want = s.attend()
    stream, other = torch.cuda.Stream(), torch.empty_like(want)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        s.mixer.attend(s.qkv, other, s.ctx, s.view)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, want)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        s.mixer.attend(s.qkv, out, s.ctx, s.view)
    for past in ([699, 39, 259], [500, 3, 0], [16, 15, 17]):
        s.ctx.pos0.copy_(torch.tensor(past, dtype=torch.int32, device="cuda"))
        graph.replay()
        s.past = past
        for r, p in enumerate(past):
            q = s.qkv[r:r + 1, :8 * 128].view(1, 8, 128)
            ref, bound = H.attention(q, c.keys[r][:, :p + 1], c.vals[r][:, :p + 1], c.mids[r][:, :p + 1], p, s.mixer.scale, 0, torch.bfloat16)
            assert bool(((out[r].view(1, 8, 128).double() - ref).abs() <= bound).all())


def engine(model_dirs, name, bits, **kw):
    from ferrum_b200 import Engine
    return Engine(model_dirs[name], dtype="bfloat16", cache_bits=bits, max_model_len=512, num_pages=kw.pop("num_pages", 128), **kw)


def quantised_write(ops):
    """A cache write for an engine with 16-bit pages whose pages then hold what 4 bits leave: the packed write into a twin of the
    plane, and the rows' pages brought back."""
    twins = {}

    def write(qkv, T, positions, request, table, cos_sin, plane, page_stride, page, Hq, Hkv, D, R, pairing, write_kv, err, partials=None):
        assert partials is None
        twin = twins.setdefault(plane.data_ptr(), torch.zeros(plane.shape[0], Hkv, page // 16, 18 * D, dtype=torch.uint8, device="cuda"))
        ops.rope_cache_write_packed(qkv, T, positions, request, table, cos_sin, twin, twin.stride(0), page, Hq, Hkv, D, R, pairing, err)
        items = (table >= 0).nonzero().int().contiguous()
        back = torch.empty(len(items), *plane.shape[1:], dtype=plane.dtype, device="cuda")
        ops.unpack_cache(twin, twin.stride(0), page, table, items, back, err)
        plane[table[table >= 0].long()] = back
    return write


@pytest.mark.parametrize("name", ["D", "E", "G"])
def test_engine_over_a_packed_cache(cuda, model_dirs, name, monkeypatch):
    """Logits equal those of the kernels for 16-bit pages over the same quantised keys and values (each side is within the suite's bound of
    the exact result, so that they are within twice that of each other), and do not depend on how a prompt is cut into portions.
    G: 32 query heads on a KV head, more rows a token than decoded tokens may have."""
    import helpers
    from ferrum_b200.engine.batch import StepEntry
    from ferrum_b200.ops import lib as ops
    eng, wide = engine(model_dirs, name, 4), engine(model_dirs, name, None)
    wide.runner.use_graphs = wide.runner.ctx.defer_residuals = False
    vocab = eng.model.n_vocab
    tokens = [(7 * i * i + 3 * i) % vocab for i in range(150)]

    def logits(e, cuts):
        slot, rows, at = e.cache.open(), [], 0
        for n in cuts:
            rows.append(e.step_raw([StepEntry(slot, at, tokens[at:at + n], list(range(n)))]).clone())
            at += n
        e.cache.close(slot)
        return torch.cat(rows).cpu()
    whole = logits(eng, [150])
    for cuts in ([64, 1, 1, 30, 54], [1] * 40 + [110], [149, 1]):
        helpers.assert_close_16bit(logits(eng, cuts), whole, f"packed {name} {cuts[:3]}", c=2 * helpers.C_16BIT["bfloat16"])
    plain = logits(wide, [150])
    monkeypatch.setattr(ops, "rope_cache_write", quantised_write(ops))
    helpers.assert_close_16bit(logits(wide, [150]), whole, f"packed {name}", c=2 * helpers.C_16BIT["bfloat16"])
    assert not torch.equal(plain, whole)


def test_engine_graphs_preemption_and_filters(cuda, model_dirs):
    """Decode steps over a packed cache replay graphs; requests that are preempted and recomputed, beside others, draw the same tokens as alone."""
    from ferrum_b200 import SamplingParams
    sp = SamplingParams(0.8, 0.9, 5, 40, 0.01)
    roomy = engine(model_dirs, "E", 4)
    prompts = [[11, 5, 900, 3] * 10, [4] * 33, [77, 8]]
    alone = [roomy.generate([p], 40, sp.temperature, sp.seed, (), sp.top_k, sp.top_p, sp.min_p)[0] for p in prompts]
    assert roomy.runner.graph_replays > 0
    roomy.runner.use_graphs = False
    assert [len(t) for t in alone] == [40] * 3
    assert roomy.generate(prompts[:1], 40, sp.temperature, sp.seed, (), sp.top_k, sp.top_p, sp.min_p)[0] == alone[0]
    assert roomy.stats()["pages_used"] == [0]
    tight = engine(model_dirs, "E", 4, num_pages=9)
    out = tight.generate(prompts, 40, sp.temperature, sp.seed, (), sp.top_k, sp.top_p, sp.min_p)
    assert tight.stats()["preemptions"] > 0 and [len(t) for t in out] == [40] * 3


def test_engine_refuses_models_that_cannot(cuda, model_dirs):
    from ferrum_b200 import Engine
    from ferrum_b200.errors import ConfigError
    with pytest.raises(ConfigError, match="4 bits"):
        Engine(model_dirs["A"], dtype="float32", cache_bits=4, num_pages=16, max_model_len=64)
    with pytest.raises(ConfigError, match="multiple of 16"):
        Engine(model_dirs["D"], dtype="bfloat16", cache_bits=4, num_pages=16, max_model_len=64, page_size=8)


def test_command_line(cuda, model_dirs):
    """`ferrum generate` with a cache in 4 bits and filters: the tokens of the Python entry point; what it refuses."""
    import json
    import subprocess
    import sys

    from conftest import ROOT
    run = lambda *args: subprocess.run([sys.executable, ROOT + "/bin/ferrum", "generate", "--model", *args], capture_output=True, text=True, cwd=ROOT, timeout=600)
    common = ("--prompt-tokens", "5,17,3", "--max-new-tokens", "6", "--num-pages", "16", "--max-model-len", "64")
    p = run(model_dirs["D"], *common, "--cache-bits", "4", "--temperature", "0.7", "--top-k", "30", "--top-p", "0.9", "--min-p", "0.01", "--seed", "5", "--profile")
    assert p.returncode == 0, p.stderr
    eng = engine(model_dirs, "D", 4)
    assert json.loads(p.stdout)["tokens"] == eng.generate([[5, 17, 3]], 6, 0.7, 5, (), 30, 0.9, 0.01)[0]
    assert "attention_packed" in p.stderr and "sample_filtered" in p.stderr
    for args, word in ((("--top-p", "1.5", "--temperature", "1"), "top_p"), (("--cache-bits", "8"), "8 bits"), (("--page-size", "8", "--cache-bits", "4"), "multiple of 16")):
        p = run(model_dirs["D"], *common, *args)
        assert p.returncode == 1 and word in p.stderr, p.stderr
