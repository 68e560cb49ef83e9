"""Filtered draws: parameters at the ends of their ranges, calls from several threads."""
import math

import numpy as np
import pytest
import torch

from test_sample_filtered_gpu import sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_p", [1.5, math.inf, float(np.nextafter(np.float32(1), np.float32(2))), -math.inf])
@pytest.mark.parametrize("V", [100, 40000])
def test_top_p_out_of_range(cuda, top_p, V):
    """A top_p beyond 1 is refused as one below 0 is, for its row alone."""
    x = torch.randn(3, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    ids, err = sample(x, [1.0] * 3, [5, 0, 5], [0.9, top_p, 1.0], [0.0] * 3, [0.5] * 3)
    good, code = sample(x, [1.0] * 3, [5, 0, 5], [0.9, 1.0, 1.0], [0.0] * 3, [0.5] * 3)
    assert code == 0 and err == 7 and ids == [good[0], -1, good[2]]


def test_calls_from_several_threads(cuda):
    """Rows of different lengths, whose CTAs hold slices of different sizes, drawn by threads at a time, each on a stream of its own."""
    import threading
    g = torch.Generator(device="cuda").manual_seed(3)
    sizes = [900, 15000, 40000, 128256, 200001, 300000]
    logits = [torch.randn(2, V, device="cuda", generator=g) for V in sizes]
    draw = lambda x: sample(x, [0.8, 1.1], [50, 0], [0.9, 0.8], [0.0, 0.01], [0.3, 0.7])
    got, together = [None] * len(sizes), threading.Barrier(len(sizes))
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            together.wait(60)
            try:
                got[i] = [draw(logits[i]) for _ in range(20)]
            except Exception as e:      # noqa: BLE001 (the thread's own failure is the test's)
                got[i] = e
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(300)
    for x, all_of in zip(logits, got):
        want = draw(x)
        assert want[1] == 0 and all_of == [want] * 20


def test_greedy_requests_do_not_look_at_top_p(cuda, model_dirs):
    """Without a temperature top_p stands for nothing, as it did before there were filters, whatever it is; with one it has to be in its range."""
    from ferrum_b200 import Engine, SamplingParams
    from ferrum_b200.errors import InvalidRequest
    eng = Engine(model_dirs["D"], dtype="bfloat16", num_pages=16, max_model_len=64)

    def run(sp):
        out = []
        rid = eng.submit([5, 17, 3], 5, sp)
        while True:
            for ev in eng.step():
                assert ev.id == rid
                if ev.kind != "token":
                    return out
                out.append(ev.token)
    want = run(SamplingParams())
    for top_p in (0.0, -1.0, 2.0, math.nan, 0.5):
        assert run(SamplingParams(0.0, top_p)) == want
    for top_p in (0.0, 2.0, math.nan):
        with pytest.raises(InvalidRequest, match="top_p"):
            eng.submit([5, 17, 3], 5, SamplingParams(0.7, top_p))
    assert not eng._filters
