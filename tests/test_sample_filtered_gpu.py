"""Draws with filters from given random numbers, against the definition in 64 bits.  Ids have to be equal wherever the random number, and the
borders of the filters, are further than 1e-11 of the mass from a change of the id: the kernel's masses are whole multiples of
2^-44 or finer, summed exactly, so that a row of 150,000 is off by less than 150,000 * 2^-45 = 4.3e-9 of the largest weight in the
worst case and by 2e-12 in a random one."""
import math
import types

import numpy as np
import pytest
import torch

import plain_sampling as P

pytestmark = pytest.mark.gpu


def sample(logits, temperature, top_k, top_p, min_p, u, rows=None, n=None, also_to=None):
    from ferrum_b200.ops import lib as ops
    n = len(u) if n is None else n
    dev = lambda v, dt: None if v is None else torch.tensor(np.asarray(v), dtype=dt, device="cuda")
    ids, err = torch.full((logits.shape[0],), -7, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.sample_filtered(logits, n, ids, err, dev(temperature, torch.float32), dev(top_k, torch.int32), dev(top_p, torch.float32),
                        dev(min_p, torch.float32), dev(u, torch.float64), rows=dev(rows, torch.int32), also_to=also_to)
    return ids.tolist(), err.item()


def check(logits, temperature, top_k, top_p, min_p, u):
    got, err = sample(logits, temperature, top_k, top_p, min_p, u)
    assert err == 0
    host = logits.cpu().numpy()
    for r in range(len(u)):
        want, room = P.draw(host[r], temperature[r], top_k[r], top_p[r], min_p[r], u[r])
        assert got[r] == want or room < 1e-11, (r, got[r], want, room, temperature[r], top_k[r], top_p[r], min_p[r], u[r])


def rows_of(kind, n, V, g):
    x = torch.randn(n, V, device="cuda", generator=g)
    if kind == "ties":
        x = torch.round(2 * x) / 2
    elif kind == "equal":
        x = torch.full_like(x, 1.25)
    elif kind == "wide":
        x = 60 * x
    elif kind == "peak":
        x[:, V // 3] += 30
    elif kind == "two levels":
        x = torch.where(x > 0, 0.0, -1.0)
    elif kind == "masked":
        x[:, ::2] = -math.inf
    elif kind == "lowest":
        x[:, 1::3] = torch.finfo(torch.float32).min
    elif kind == "tiny":
        x = x * 1e-42
    else:
        x = 3 * x
    return x


KINDS = ["plain", "ties", "equal", "wide", "peak", "two levels", "masked", "lowest", "tiny"]


# vocabularies around a warp, a block's threads, the cluster's slices and beyond
@pytest.mark.parametrize("V", [1, 2, 31, 257, 1000, 8191, 16384, 32003, 128256])
@pytest.mark.parametrize("kind", KINDS)
def test_draws(cuda, V, kind):
    g = torch.Generator(device="cuda").manual_seed(V)
    rng = np.random.default_rng(V + len(kind))
    n = 12 if V > 20000 else 24
    x = rows_of(kind, n, V, g)
    some = lambda v, off: np.where(rng.random(n) < 0.6, v, off)
    check(x, rng.uniform(0.3, 2.0, n), some(np.exp(rng.uniform(0, np.log(V + 1), n)).astype(int), 0), some(rng.uniform(0.02, 0.999, n), 1.0),
          some(rng.uniform(0, 0.3, n), 0.0), rng.random(n))


@pytest.mark.parametrize("n,V", [(1, 128256), (9, 70000), (10, 70000), (19, 65536), (3, 400001), (2, 760000), (150, 900)])
def test_launch_shapes(cuda, n, V):
    """Clusters of every size, rows that outgrow the shared memory, cuts that outgrow the lists of what lies above them."""
    g = torch.Generator(device="cuda").manual_seed(n)
    rng = np.random.default_rng(n)
    for kind in ("plain", "ties"):
        x = rows_of(kind, n, V, g)
        some = lambda v, off: np.where(rng.random(n) < 0.6, v, off)
        check(x, rng.uniform(0.7, 1.5, n), some(np.exp(rng.uniform(0, np.log(V + 1), n)).astype(int), 0), some(rng.uniform(0.5, 0.999, n), 1.0),
              some(rng.uniform(0, 0.05, n), 0.0), rng.random(n))


@pytest.mark.parametrize("V", [9000, 16384, 40000, 70001])
def test_a_draw_does_not_depend_on_the_rows_beside_it(cuda, V):
    """Rows drawn alone, a few and all at a time (by clusters of other sizes) get the same ids."""
    g = torch.Generator(device="cuda").manual_seed(V)
    rng = np.random.default_rng(V)
    n = 34
    x = rows_of("ties", n, V, g)
    t, u = rng.uniform(0.7, 1.5, n), rng.random(n)
    k, p, m = rng.choice([0, 1, 40, 3000], n), rng.choice([1.0, 0.9, 0.4], n), rng.choice([0.0, 0.02], n)
    want, err = sample(x, t, k, p, m, u)
    assert err == 0
    for size in (1, 3, 7, 16):
        for a in range(0, n, 5 * size):
            part = slice(a, a + size)
            assert sample(x[part].contiguous(), t[part], k[part], p[part], m[part], u[part])[0] == want[part]


@pytest.mark.parametrize("V", [700, 50000])
def test_edges_of_the_filters(cuda, V):
    """k of 1, V and beyond; p next to 0 and 1; min_p of 1; random numbers 0 and next to 1; a temperature next to 0 and a large one."""
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.round(rows_of("plain", 16, V, g) * 8) / 8
    below = 1 - 2.0 ** -53
    t = [1.0] * 13 + [1e-6, 1e30, 0.0]
    k = [1, V, V + 5, 0, 0, 0, 0, 2, 0, 0, -3, 5, 5, 0, 0, 40]
    p = [1.0, 1.0, 1.0, 1e-30, float(np.nextafter(np.float32(1), np.float32(0))), 1.0, 0.5, 0.5, 1.0, 1.0, 0.3, 1.0, 1.0, 1.0, 0.5, 0.1]
    m = [0, 0, 0, 0, 0, 1.0, 0, 0, 0, 0, -1.0, 0, 0, 0, 0, 0.5]
    u = [0.7, 0.3, 0.9, 0.99, 0.5, 0.2, 0.0, below, 0.0, below, 0.1, 0.0, below, 0.5, 0.25, 0.9]
    check(x, t, k, p, m, u)
    got, _ = sample(x, t, k, p, m, u)
    top = x.max(-1).values
    for r in (0, 3, 5, 15):                # k of 1, p next to 0 and T = 0 leave the lowest of the largest, min_p of 1 one of the largest
        assert x[r, got[r]] == top[r]
    assert got[0] == x[0].argmax().item() and got[15] == x[15].argmax().item()


def test_filters_may_be_left_out(cuda):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = rows_of("plain", 8, 5000, g)
    u = np.linspace(0.01, 0.99, 8)
    got, err = sample(x, [0.8] * 8, None, None, None, u)
    assert err == 0 and got == sample(x, [0.8] * 8, [0] * 8, [1.0] * 8, [0.0] * 8, u)[0]


def test_frequencies(cuda):
    """Over evenly spread random numbers every id comes as often as its probability says."""
    x = torch.tensor([[2.0, 0.5, 1.0, -1.0, 2.0, 0.0]], device="cuda").repeat(4096, 1)
    u = (np.arange(4096) + 0.5) / 4096
    got, _ = sample(x, [0.9] * 4096, [5] * 4096, [0.95] * 4096, [0.05] * 4096, u)
    w = P.kept(x[0].cpu().numpy(), 0.9, 5, 0.95, 0.05)
    assert np.abs(np.bincount(got, minlength=6) - 4096 * w / w.sum()).max() <= 1


@pytest.mark.parametrize("V", [33, 20000])
def test_nan_and_infinite_logits(cuda, V):
    """NaN is never drawn and counts for nothing; +infinity takes all; a row of -infinity is a row of equals; a row of NaN raises error 6."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(5, V, device="cuda", generator=g)
    x[0, ::2] = math.nan
    x[1, 7], x[1, 20] = math.inf, math.inf
    x[2] = -math.inf
    x[3] = -math.inf
    x[3, 11] = math.nan
    x[4, 1:] = math.nan
    for k, p, m in ((0, 1.0, 0.0), (9, 0.8, 0.0), (0, 0.5, 0.2)):
        check(x, [1.0] * 5, [k] * 5, [p] * 5, [m] * 5, [0.1, 0.6, 0.99, 0.4, 0.7])
    x[2] = math.nan
    ids, err = sample(x, [1.0] * 5, [0] * 5, [1.0] * 5, [0.0] * 5, [0.5] * 5)
    assert err == 6 and ids[2] == -1 and ids[4] == 0


@pytest.mark.parametrize("t,p,m", [(-1.0, 0.5, 0.0), (math.nan, 0.5, 0.0), (math.inf, 0.5, 0.0), (1.0, 0.0, 0.0), (1.0, -0.1, 0.0), (1.0, math.nan, 0.0),
                                   (1.0, 0.5, 1.5), (1.0, 0.5, math.nan)])
def test_parameters_out_of_range(cuda, t, p, m):
    x = torch.randn(3, 100, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    ids, err = sample(x, [1.0, t, 1.0], [5] * 3, [0.9, p, 0.9], [0.0, m, 0.0], [0.5] * 3)
    good, _ = sample(x, [1.0] * 3, [5] * 3, [0.9] * 3, [0.0] * 3, [0.5] * 3)
    assert err == 7 and ids[1] == -1 and ids[0] == good[0] and ids[2] == good[2]


def test_random_numbers_out_of_range_are_brought_into_it(cuda):
    x = torch.zeros(4, 50, device="cuda")
    assert sample(x, [1.0] * 4, [0] * 4, [1.0] * 4, [0.0] * 4, [-0.5, 1.0, 7.0, math.nan])[0] == [0, 49, 49, 0]


def test_picked_rows_strides_and_a_second_place(cuda):
    """Only the rows named are drawn, from logits whose rows lie apart; `also_to` gets the same ids."""
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.full((6, 1100), math.nan, device="cuda")
    wide[:, :1003] = torch.randn(6, 1003, device="cuda", generator=g)
    x, also = wide[:, :1003], torch.full((9,), -9, dtype=torch.int32, device="cuda")
    ids, err = sample(x, [1.0, 0.5], [0, 7], [0.7, 1.0], [0.0, 0.0], [0.3, 0.8], rows=[4, 1], n=2, also_to=also)
    host = x.cpu().numpy()
    want = {4: P.draw(host[4], 1.0, 0, 0.7, 0.0, 0.3)[0], 1: P.draw(host[1], 0.5, 7, 1.0, 0.0, 0.8)[0]}
    assert err == 0 and ids == [want.get(r, -7) for r in range(6)] and also.tolist() == [want.get(r, -9) for r in range(9)]
    assert sample(x, [1.0], None, None, None, [0.5], n=0)[0] == [-7] * 6
    ids, err = sample(x, [1.0, 1.0, 1.0], None, None, None, [0.3, 0.3, 0.3], rows=[6, 2, -1])       # rows that are not there
    assert err == 7 and ids[2] >= 0 and ids[:2] + ids[3:] == [-7] * 5


def test_replayed_graph_and_another_stream(cuda):
    from ferrum_b200.ops import lib as ops
    g = torch.Generator(device="cuda").manual_seed(5)
    x = 2 * torch.randn(9, 40000, device="cuda", generator=g)
    t, k, p, m = torch.full((9,), 0.9, device="cuda"), torch.full((9,), 60, dtype=torch.int32, device="cuda"), torch.full((9,), 0.9, device="cuda"), torch.zeros(9, device="cuda")
    u = torch.rand(9, device="cuda", generator=g, dtype=torch.float64)
    ids, err = torch.empty(9, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.sample_filtered(x, 9, ids, err, t, k, p, m, u)
    want, graph = ids.clone(), torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ids.fill_(-1)
        ops.sample_filtered(x, 9, ids, err, t, k, p, m, u)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(ids, want)
    with torch.cuda.graph(graph):
        ops.sample_filtered(x, 9, ids, err, t, k, p, m, u)
    for _ in range(3):
        u.copy_(torch.rand(9, device="cuda", generator=g, dtype=torch.float64))
        graph.replay()
        got = ids.tolist()
        ops.sample_filtered(x, 9, ids, err, t, k, p, m, u)
        assert ids.tolist() == got and err.item() == 0


def test_sampler_mixes_rows_with_and_without_filters(cuda):
    """`DeviceSampler`: rows without filters draw as they do without the others; rows with filters draw by the definition."""
    from ferrum_b200.sampling import DeviceSampler, Filters
    from ferrum_b200.sampling.sampler import uniform
    g = torch.Generator(device="cuda").manual_seed(6)
    x = 2 * torch.randn(5, 3001, device="cuda", generator=g)
    row = lambda t, c: types.SimpleNamespace(temperature=t, seed=41, counter=c)
    rows = [row(0.0, 0), row(0.8, 1), row(0.7, 2), row(1.1, 3), row(0.0, 4)]
    sampler = DeviceSampler(8)
    plain, code = sampler.sample(x, rows)
    f = Filters(20, 0.9, 0.01)
    got, code2 = sampler.sample(x, rows, [None, None, f, f, f])
    assert code == code2 == 0 and got[:2] == plain[:2] and got[4] == plain[4]
    host = x.cpu().numpy()
    for i in (2, 3):
        assert got[i] == P.draw(host[i], rows[i].temperature, 20, 0.9, 0.01, uniform(41, rows[i].counter))[0]
    assert sampler.sample(x[2:4], rows[2:4], [f, f])[0] == got[2:4]            # alone: the same draws
    assert sampler.sample(x, rows, [Filters()] * 5)[0] == plain


def test_engine_draws_with_filters(cuda, model_dirs):
    """Requests with filters of their own beside others; the draws do not depend on the batch, and each follows the definition on the
    model's own logits; a filter of one token is greedy."""
    from ferrum_b200 import Engine, SamplingParams
    from ferrum_b200.engine.batch import StepEntry
    eng = Engine(model_dirs["D"], dtype="bfloat16", num_pages=64, max_model_len=256)
    prompts = [[5, 17, 3, 40], [9, 8, 7], [100, 200, 300, 7, 7]]
    sp = SamplingParams(0.9, 0.8, 12, 50, 0.02)

    def run(requests):
        ids = [eng.submit(p, 8, s) for p, s in requests]
        out = {i: [] for i in ids}
        done = 0
        while done < len(ids):
            for ev in eng.step():
                if ev.kind == "token":
                    out[ev.id].append(ev.token)
                else:
                    done += 1
        assert not eng._filters
        return [out[i] for i in ids]
    greedy = run([(p, SamplingParams()) for p in prompts])
    one = run([(p, SamplingParams(1.0, 1.0, 3, 1)) for p in prompts])
    assert one == greedy
    alone = run([(prompts[1], sp)])[0]
    mixed = run([(prompts[0], SamplingParams()), (prompts[1], sp), (prompts[2], SamplingParams(0.5, 1.0, 2))])
    assert mixed[0] == greedy[0]
    for tokens in (alone, mixed[1]):
        slot = eng.cache.open()
        seq = prompts[1] + tokens
        logits = eng.step_raw([StepEntry(slot, 0, seq[:-1], list(range(len(prompts[1]) - 1, len(seq) - 1)))]).cpu().numpy()
        eng.cache.close(slot)
        for i, t in enumerate(tokens):
            # (filters a little wider: these logits come from a prompt's step, whose 16-bit roundings fall otherwise)
            assert P.kept(logits[i], 0.9, 60, 0.85, 0.015)[t] > 0
    rid = eng.submit(prompts[0], 8, sp)
    eng.cancel(rid)
    assert not eng._filters
