"""Requests with filters in an engine, draw by draw: every id follows from its own step's logits, the request's own filters and the random number of (seed, tokens
generated so far), whoever shares the step and whatever was recomputed."""
import pytest

import plain_sampling as P

pytestmark = pytest.mark.gpu


class Record:
    """Notes what an engine's sampler is given and what it returns."""

    def __init__(self, eng):
        self.draws, self.open = [], {}
        launch, collect = eng.sampler.launch, eng.sampler.collect

        def noted_launch(logits, rows, also_to=None, filters=None):
            ticket = launch(logits, rows, also_to=also_to, filters=filters)
            self.open[id(ticket)] = (ticket, logits[:len(rows)].clone(), [(r.id, r.temperature, r.seed, r.counter) for r in rows], list(filters or [None] * len(rows)))
            return ticket

        def noted_collect(ticket):
            ids, code = collect(ticket)
            _, logits, rows, filters = self.open.pop(id(ticket))
            self.draws.append((logits.cpu().numpy(), rows, filters, ids))
            return ids, code
        eng.sampler.launch, eng.sampler.collect = noted_launch, noted_collect


def check(record, requests, out):
    """requests: id -> (temperature, seed, top_k, top_p, min_p); out: id -> its tokens."""
    from ferrum_b200.sampling import Filters
    from ferrum_b200.sampling.sampler import uniform
    seen = {rid: {} for rid in requests}
    shared = 0
    for logits, rows, filters, ids in record.draws:
        shared = max(shared, len(rows))
        for x, (rid, t, seed, counter), f, token in zip(logits, rows, filters, ids):
            temperature, own_seed, k, p, m = requests[rid]
            assert (t, seed) == (pytest.approx(temperature), own_seed)
            if t > 0 and Filters(k, p, m).on:
                assert f == Filters(k, p, m)
                want, room = P.draw(x, t, k, p, m, uniform(own_seed, counter))
                assert token == want or room < 1e-11
            else:
                assert f is None and (t > 0 or token == P.draw(x, 0.0, 0, 1.0, 0.0, 0.0)[0])
            # (a token drawn for a request that had finished meanwhile is dropped; one drawn again after a preemption keeps its number)
            seen[rid].setdefault(counter, []).append(token)
    for rid, tokens in out.items():
        for i, token in enumerate(tokens):
            assert token in seen[rid][i], (rid, i)
    return shared


def run(eng, wanted, tokens):
    """Submits (prompt, SamplingParams) and runs all to their end: id -> tokens."""
    ids = [eng.submit(p, tokens, s) for p, s in wanted]
    out, left = {i: [] for i in ids}, len(ids)
    while left:
        for ev in eng.step():
            if ev.kind == "token":
                out[ev.id].append(ev.token)
            else:
                left -= 1
    assert not eng._filters
    return out


def requests_of(out, wanted):
    return {rid: (s.temperature, s.seed, s.top_k, s.top_p, s.min_p) for rid, (_, s) in zip(out, wanted)}


@pytest.mark.parametrize("bits", [16, 4])
def test_every_draw_follows_its_own_steps_logits(cuda, model_dirs, bits):
    from ferrum_b200 import Engine, SamplingParams
    eng = Engine(model_dirs["D"], dtype="bfloat16", num_pages=64, max_model_len=256, cache_bits=bits)
    wanted = [([5, 17, 3, 40], SamplingParams()), ([9, 8, 7], SamplingParams(0.9, 0.8, 12, 50, 0.02)), ([100, 200, 300, 7, 7], SamplingParams(0.5, 1.0, 2)),
              ([3] * 40, SamplingParams(1.4, 0.95, 3)), ([1, 2], SamplingParams(0.8, 1.0, 12, 0, 0.1))]
    record = Record(eng)
    out = run(eng, wanted, 20)
    assert all(len(t) == 20 for t in out.values())
    assert check(record, requests_of(out, wanted), out) == 5


@pytest.mark.parametrize("bits", [16, 4])
def test_preempted_requests_keep_their_filters_and_numbers(cuda, model_dirs, bits):
    from ferrum_b200 import Engine, SamplingParams
    eng = Engine(model_dirs["E"], dtype="bfloat16", num_pages=9, max_model_len=512, cache_bits=bits)
    wanted = [([11, 5, 900, 3] * 10, SamplingParams(0.8, 0.9, 5, 40, 0.01)), ([4] * 33, SamplingParams(1.1, 0.7, 6)), ([77, 8], SamplingParams(0.8, 1.0, 7, 9, 0.05))]
    record = Record(eng)
    out = run(eng, wanted, 40)
    assert eng.stats()["preemptions"] > 0 and all(len(t) == 40 for t in out.values())
    check(record, requests_of(out, wanted), out)
