"""Edges of the rules on the logits: sizes of shared memory around the limit that needs no opt-in."""

import math
import os
import subprocess
import sys

import pytest
import torch

from cohere_inference_b200.synth import synthetic_model

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
from test_gpu_operators import gen, rules_of, run_rules, tables, under_rules  # noqa: E402
from test_gpu_rules_and_caches import decoder, start  # noqa: E402

pytestmark = pytest.mark.gpu


def in_a_fresh_process(call):
    """No earlier call of this process has set a kernel's attributes there."""
    r = subprocess.run([sys.executable, "-c", f"import test_gpu_operator_edges as t; t.{call}; print('done')"], capture_output=True,
                       text=True, timeout=600, cwd=HERE, env={**os.environ, "PYTHONPATH": os.path.dirname(HERE)})
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr


def around_48_kb(kind):
    """128 rows of 16384 logits and 1024 biases ask for 47112 + 4 * columns bytes of dynamic shared memory, beside 256 static ones."""
    from cohere_inference_b200 import native as nv
    rows, vocab, max_bias = 128, 16384, 1024
    for cols in (446, 447, 466, 510, 511):  # 48 896: just fits without an opt-in; 48 900; ...; 49 152; 49 156
        t = tables(rows, vocab, cols, max_bias, cols)
        active = torch.arange(rows, dtype=torch.int32, device="cuda")
        logits = ((torch.randn(rows, vocab, generator=gen(cols), device="cuda") * 16).round() / 8).clamp(-12, 12).to(kind)
        token, best, status = run_rules(nv, logits, vocab, active, rows, rules_of(nv, t))
        assert status == 0
        for r in (0, 77, 127):
            x = under_rules(logits[r], r, t)
            assert int(token[r]) == int((x == x.max()).nonzero()[0]) and float(best[r]) == float(x.max())


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
def test_logit_rules_around_the_default_shared_memory(kind):
    in_a_fresh_process(f"around_48_kb(t.torch.{kind})")


def most_biases():
    dec = decoder(synthetic_model(0), slots=128, max_new_tokens=448, int8=True, logit_rules=True, max_bias=1024)
    slots, b = start(dec, [dict(repetition=1.5, bias={v: -math.inf for v in range(1024)})] * 5)
    for _ in range(20):
        dec.step(b)
    dec.check_status()


def test_decoder_with_the_most_biases():
    in_a_fresh_process("most_biases()")
