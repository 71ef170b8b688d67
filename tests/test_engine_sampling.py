"""The engine's and the model's draws: tokens against the operator's definition
on the logits that the same steps return."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from shukuchi_b200 import cuda as sc
from shukuchi_b200 import gguf, synth
from test_engine import ENGINE, Config, lib
from test_sample import kept_weights

gpu = pytest.mark.gpu


def engine():
    L = lib()
    L.engine_set_sampling.argtypes = [C.c_void_p, C.c_float, C.c_int, C.c_float, C.c_float, C.c_uint64]
    return L


def uniforms(seed, n):
    """SplitMix64, the top 24 bits."""
    out, m = [], (1 << 64) - 1
    for _ in range(n):
        seed = (seed + 0x9E3779B97F4A7C15) & m
        z = seed
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & m
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & m
        out.append(((z ^ (z >> 31)) >> 40) * 2.0 ** -24)
    return out


def is_the_draw(logits, token, u, temperature, top_k, top_p, min_p):
    w, close = kept_weights(logits, temperature, top_k, top_p, min_p)
    if close:
        return True  # a border within rounding of the exponential
    ends, slack = np.cumsum(w), 4e-7 * w.sum() + len(w)
    return w[token] > 0 and ends[token] - w[token] - slack <= u * w.sum() < ends[token] + slack


def test_refused_without_a_handle():
    assert engine().engine_set_sampling(None, 1.0, 0, 1.0, 0.0, 0) == -1
    assert sc.lib().shk_cuda_model_sample(None, C.byref(sc.Sampling()), 0.5, None, None, None) == -1


@pytest.fixture(scope="module")
def model_file(tmp_path_factory):
    m = synth.make_model("small", seed=33)
    path = str(tmp_path_factory.mktemp("gguf") / "small.gguf")
    gguf.write_model(path, m)
    return m, path


@gpu
@pytest.mark.parametrize("resident", [1, 0])
def test_engine_draws(model_file, resident, monkeypatch):
    m, path = model_file
    monkeypatch.setenv("SHUKUCHI_HBM_RESIDENT", str(resident))
    L, n, vocab = engine(), 12, m.shape.n_vocab
    prompt = np.random.default_rng(5).integers(0, vocab, 6).astype(np.uint32)
    h = L.engine_open(path.encode(), C.byref(Config(4, 1, 3, 32, 0, 0)))
    assert h, "engine_open failed"

    def run(*settings):
        assert L.engine_set_sampling(h, *settings) == 0
        ids, logits = np.zeros(n, np.uint32), np.zeros((n, vocab), np.float32)
        assert L.engine_generate_ids(h, prompt.ctypes.data, prompt.size, n, ids.ctypes.data, logits.ctypes.data) == n
        return ids, logits

    try:
        greedy, first = run(0.0, 0, 1.0, 0.0, 7)
        assert np.array_equal(greedy, first.argmax(1))
        # the temperature that spreads this model's logits over some tokens
        t = float(np.std(first[0])) / 2
        seen = set()
        for settings in ((t, 0, 1.0, 0.0), (t, 40, 0.95, 0.02), (t / 2, 0, 0.9, 0.0), (t, 1, 1.0, 0.0)):
            for seed in (1, 2 ** 63 + 5):
                ids, logits = run(*settings, seed)
                again, _ = run(*settings, seed)
                assert np.array_equal(ids, again)
                for token, z, u in zip(ids, logits, uniforms(seed, n)):
                    assert is_the_draw(z, int(token), u, *settings)
                if settings[1] == 1:
                    assert np.array_equal(ids, greedy)
                seen.add(tuple(ids))
        assert len(seen) > 4
        assert L.engine_set_sampling(h, -1.0, 0, 1.0, 0.0, 0) == -1
        assert L.engine_set_sampling(h, float("nan"), 0, 1.0, 0.0, 0) == -1
        assert np.array_equal(run(0.0, 0, 1.0, 0.0, 0)[0], greedy)
    finally:
        L.engine_close(h)


@gpu
def test_cli_draws(model_file):
    m, path = model_file
    cli = os.path.join(os.path.dirname(ENGINE), "shukuchi")
    run = lambda *a: subprocess.run([cli, path, "--tokens", "1,5,9", "--max-tokens", "8", *a], capture_output=True, text=True)
    # (the synthetic model's logits are far apart: this temperature makes them equal)
    greedy, hot = run(), run("--temperature", "1e30", "--seed", "3")
    assert greedy.returncode == hot.returncode == 0 and greedy.stdout != hot.stdout
    assert run("--temperature", "1e30", "--seed", "3").stdout == hot.stdout
    assert run("--temperature", "1e30", "--seed", "4").stdout != hot.stdout
    assert run("--temperature", "5", "--top-k", "1").stdout == greedy.stdout
    assert run("--temperature", "-1").returncode == 1


@gpu
def test_model_sample(ctx):
    from shukuchi_b200.device_model import GpuDecoder
    model = synth.make_model("tiny", seed=7)
    dec = GpuDecoder(ctx, model, max_seq=32)
    try:
        vocab = model.shape.n_vocab
        logits = np.zeros(vocab, np.float32)
        nxt = dec.m.token_step(3, 0, want_next=True, logits_host_ptr=logits.ctypes.data)
        assert dec.m.sample(0.3, temperature=0.0) == (nxt, 1.0)
        t = float(np.std(logits))
        for u in (0.0, 0.25, 0.999):
            token, prob = dec.m.sample(u, temperature=t, top_k=20, top_p=0.9)
            w, close = kept_weights(logits, t, 20, 0.9, 0.0)
            assert close or (is_the_draw(logits, token, u, t, 20, 0.9, 0.0) and abs(prob - w[token] / w.sum()) < 1e-6)
        assert dec.m.token_step(nxt, 1, want_next=True) == dec.m.sample(0.5, temperature=0.0)[0]
        for u in (-0.1, 1.0, float("nan")):
            with pytest.raises(sc.ShkError):
                dec.m.sample(u)
    finally:
        dec.close()
