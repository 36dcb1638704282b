"""The engine's 8-bit copies and weights that change."""

import asyncio

import pytest
import torch

from accerl_agent_b200 import ops
from accerl_agent_b200.models.transformer import build_model
from test_engine_int8 import PROMPTS, generate_without_shutdown, make


@pytest.mark.gpu
def test_copies_on_several_streams_are_all_awaited():
    """Two halves of the weights on two streams, the first behind a kernel that runs for a while, and a third update on
    the current stream: the next step quantises none of them before they are there."""
    cfg, m, engine = make("cuda")
    eng = engine(quantization="int8")
    generate_without_shutdown(eng, PROMPTS[:1], "a")
    other = build_model(cfg, "full", torch.device("cuda"), m.params.dtype, with_grads=False)
    other.init_weights(seed=8, std=0.08)
    n = m.params.numel() // 2
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        torch.cuda._sleep(400_000_000)  # some 0.2 s
    eng.load_flat_weights(other.params[:n], stream=first)
    eng.load_flat_weights(other.params[n:], start=n, stream=second)
    eng.load_flat_weights(other.params[-8:], start=m.params.numel() - 8)
    generate_without_shutdown(eng, PROMPTS[:1], "b")
    torch.cuda.synchronize()
    for name, w in eng._w8.items():
        expect = ops.quantize_rows(other.w(name))
        assert torch.equal(w.q, expect.q) and torch.equal(w.scale, expect.scale), name
    asyncio.run(eng.shutdown())


def test_a_change_during_the_quantising_is_not_lost(monkeypatch):
    """``weights_changed`` from another thread while the 8-bit copies are being made: they are made once more."""
    cfg, m, engine = make("cpu")
    eng = engine(quantization="int8")
    real, calls = ops.quantize_rows, []

    def quantize(x, out=None):
        r = real(x, out=out)
        calls.append(1)
        if len(calls) == 1:  # the copy just made is already old
            m.params.mul_(1.5)
            eng.weights_changed()
        return r

    monkeypatch.setattr(ops, "quantize_rows", quantize)
    eng.weights_changed()
    generate_without_shutdown(eng, PROMPTS[:1], "a")
    for name, w in eng._w8.items():
        assert torch.equal(w.scale, real(m.w(name)).scale), name
    # a refresh that fails is tried again
    eng.weights_changed()

    def fail(x, out=None):
        raise RuntimeError("no")

    monkeypatch.setattr(ops, "quantize_rows", fail)
    with pytest.raises(RuntimeError):
        eng._refresh_int8()
    m.params.mul_(2.0)
    monkeypatch.setattr(ops, "quantize_rows", real)
    eng._refresh_int8()
    for name, w in eng._w8.items():
        assert torch.equal(w.scale, real(m.w(name)).scale), name
    asyncio.run(eng.shutdown())


def test_a_busy_step_loop_does_not_starve_a_pause():
    """Steps that follow each other without a break: a pause, or a weight update, gets in within a few of them."""
    import threading
    import time

    cfg, m, engine = make("cpu")
    eng = engine()
    steps, stop = [0], threading.Event()

    def loop():
        while not stop.is_set():
            with eng._step_lock:
                steps[0] += 1
                sum(range(20000))

    t = threading.Thread(target=loop)
    t.start()
    try:
        waited = []
        for _ in range(20):
            time.sleep(0.005)
            before = steps[0]
            eng.load_flat_weights(m.params)
            waited.append(steps[0] - before)
        assert max(waited) < 100, waited  # thousands with a plain lock
    finally:
        stop.set()
        t.join()
