"""The engine's draws behind a batched prefill, the model's before it has any
logits: where test_engine_sampling does not go."""
import ctypes as C

import numpy as np
import pytest

from shukuchi_b200 import gguf, synth
from test_engine import Config
from test_engine_sampling import engine, uniforms
from test_sample import NONE
from test_sample_borders import permissible

pytestmark = pytest.mark.gpu


def test_engine_draws_behind_a_prefill(tmp_path, monkeypatch):
    """The first token is drawn from the prefill's own logits, the others from the steps': each against the logits that
    the same generation returns."""
    monkeypatch.setenv("SHUKUCHI_HBM_RESIDENT", "1")
    m = synth.make_model("small", seed=33)
    path = str(tmp_path / "small.gguf")
    gguf.write_model(path, m)
    L, n, vocab = engine(), 6, m.shape.n_vocab
    prompt = np.random.default_rng(5).integers(0, vocab, 9).astype(np.uint32)
    h = L.engine_open(path.encode(), C.byref(Config(4, 1, 3, 32, 0, 0)))
    assert h, "engine_open failed"

    def run(prefill, *settings):
        monkeypatch.setenv("SHUKUCHI_PREFILL", str(prefill))
        assert L.engine_set_sampling(h, *settings) == 0
        ids, logits = np.zeros(n, np.uint32), np.zeros((n, vocab), np.float32)
        assert L.engine_generate_ids(h, prompt.ctypes.data, prompt.size, n, ids.ctypes.data, logits.ctypes.data) == n
        return ids, logits

    try:
        _, stepped = run(0, 0.0, 0, 1.0, 0.0, 0)
        greedy, filled = run(4, 0.0, 0, 1.0, 0.0, 0)
        assert np.array_equal(greedy, filled.argmax(1))
        assert not np.array_equal(stepped[0], filled[0])  # f16 products: the prefill ran
        t = float(np.float32(np.std(filled[0]) / 2))
        seen = set()
        for settings in ((t, 0, 1.0, 0.0), (t, 40, 0.95, 0.02)):
            for seed in (1, 2, 3):
                ids, logits = run(4, *settings, seed)
                assert np.array_equal(logits[0], filled[0])
                seen.add(tuple(ids))
                _, k, top_p, min_p = settings
                for token, z, u in zip(ids, logits, uniforms(seed, n)):
                    tokens = permissible(z, u, t, k, float(np.float32(top_p)), float(np.float32(min_p)))[0]
                    assert len(tokens) <= 2 and int(token) in tokens
        assert len(seen) > 1
    finally:
        L.engine_close(h)


def test_model_sample_before_any_logits(ctx):
    from shukuchi_b200.device_model import GpuDecoder
    dec = GpuDecoder(ctx, synth.make_model("tiny", seed=7), max_seq=32)
    try:
        for t in (0.0, 1.0):
            assert dec.m.sample(0.5, temperature=t, top_k=20, top_p=0.9) == (NONE, 0.0)
        nxt = dec.m.token_step(3, 0, want_next=True)
        assert dec.m.sample(0.5, temperature=0.0) == (nxt, 1.0)
    finally:
        dec.close()


def test_engine_sampling_arguments(tmp_path, monkeypatch):
    """What is refused leaves the settings before it in place; every finite temperature, a negative top_p (one token) and
    a negative min_p (off) are taken."""
    monkeypatch.setenv("SHUKUCHI_HBM_RESIDENT", "1")
    m = synth.make_model("small", seed=33)
    path = str(tmp_path / "small.gguf")
    gguf.write_model(path, m)
    L, vocab, nan, inf = engine(), m.shape.n_vocab, float("nan"), float("inf")
    h = L.engine_open(path.encode(), C.byref(Config(4, 1, 3, 32, 0, 0)))
    assert h, "engine_open failed"

    def run():
        prompt, ids = np.array([3, 5], np.uint32), np.zeros(4, np.uint32)
        assert L.engine_generate_ids(h, prompt.ctypes.data, 2, 4, ids.ctypes.data, None) == 4
        return ids.tolist()

    try:
        greedy = run()
        assert L.engine_set_sampling(h, 3.3e38, 0, 1.0, -1.0, 9) == 0
        hot = run()
        assert hot != greedy and max(hot) < vocab
        for bad in ((-1.0, 0, 1.0, 0.0), (nan, 0, 1.0, 0.0), (inf, 0, 1.0, 0.0), (1.0, 0, nan, 0.0), (1.0, 0, 1.0, nan)):
            assert L.engine_set_sampling(h, *bad, 1) == -1
            assert run() == hot
        assert L.engine_set_sampling(h, 3.3e38, 0, -1.0, 0.0, 9) == 0
        assert run() == greedy
    finally:
        L.engine_close(h)
