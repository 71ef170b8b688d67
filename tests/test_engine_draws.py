"""The model's draws before it has any logits: where test_engine_sampling does not go."""
import pytest

from shukuchi_b200 import synth
from test_sample import NONE

pytestmark = pytest.mark.gpu


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
