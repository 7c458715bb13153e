"""The cache, the attention and the MoE layer together: a decoder fed a prompt at once, by parts or token by token, over
forked, rolled-back and compacted sequences, gives the same distributions."""
import importlib.util
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
EXAMPLE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "decode.py")
# The ways to feed a token differ in the order of 32-bit sums, and a rounding to bf16 (2^-8) that falls the other way
# is passed on: about ten a layer, two layers, relative to values of the logits' spread (rms 1.4), three deviations of
# that: 20 * 2^-8 * 1.4 * 3 = 0.33.  All experts are chosen, so that no choice can flip.
TOL = 0.33


def load():
    spec = importlib.util.spec_from_file_location("decode_example", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("window", [0, 9])
def test_ways_to_feed_the_same_tokens_agree(cuda_device, window):
    mod = load()
    model = mod.Decoder(experts=2, top_k=2, vocab=64, window=window)
    for w in model.blocks:
        w["o"] /= 4
    model.embed /= 16
    tokens = torch.randint(0, 64, (1, 40), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    whole = model.step(tokens, mod.ints(0))
    parts = torch.cat([model.step(t, mod.ints(1)) for t in tokens.split([7, 1, 20, 12], 1)], 1)
    torch.testing.assert_close(parts, whole, atol=TOL, rtol=0)
    # forked after 16 + 5 tokens, fed a wrong draft that is rolled back, then the rest
    model.step(tokens[:, :21], mod.ints(2))
    model.cache.fork(mod.ints(2), mod.ints(3))
    model.step(tokens[:, :5].expand(2, -1), mod.ints(2, 3))
    model.cache.truncate(mod.ints(3, 2), mod.ints(21, 21))
    model.cache.free(mod.ints(1, 2))
    model.cache.compact()
    rest = model.step(tokens[:, 21:], mod.ints(3))
    torch.testing.assert_close(rest, whole[:, 21:], atol=TOL, rtol=0)
    model.step(tokens[:, :1], mod.ints(0))
    assert model.cache.check_device_status() == 0
    assert int(model.cache.refcounts.sum()) == 3 + 3


def test_example_runs(cuda_device):
    done = subprocess.run([sys.executable, EXAMPLE], capture_output=True, text=True, timeout=240)
    assert done.returncode == 0, done.stderr[-2000:]
    assert "lengths [57, 57, 57]" in done.stdout and done.stdout.rstrip().endswith("status 0")
