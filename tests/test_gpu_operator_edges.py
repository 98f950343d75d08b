"""Edges of the rules on the logits and of the 8-bit product: sizes of shared memory around the limit that needs no opt-in, slots without
tokens, NaN through the activations, rows whose choice nobody takes, a request's rules on their way through the scheduler."""

import math
import os
import subprocess
import sys
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from cohere_inference_b200.synth import synthetic_model, synthetic_requests

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
from test_gpu_operators import gen, rules_of, run_rules, tables, under_rules  # noqa: E402
from test_gpu_rules_and_caches import decoder, start  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nv():
    from cohere_inference_b200 import native
    native.lib()
    return native


@pytest.fixture(scope="module")
def model16():
    return synthetic_model(0)


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


@pytest.mark.parametrize("last", [-1, -2, -9, -(1 << 31)])
def test_logit_rules_of_a_slot_without_tokens(nv, last):
    """Below -1 is no token, as -1 is: every listed bias counts, every logit is written."""
    rows, vocab, slots, n = 3, 5000, 3, 12
    t = tables(slots, vocab, 40, n, 31)
    t["last"][:], t["bias_n"][:] = -1, n
    t["params"][:, :3] = torch.tensor([2.0, 1.0, 0.5], device="cuda")
    t["mask_on"][:] = torch.tensor([0, 1, 0, 0], device="cuda")
    active = torch.arange(rows, dtype=torch.int32, device="cuda")
    logits = ((torch.randn(rows, vocab, generator=gen(32), device="cuda") * 16).round() / 8).clamp(-12, 12)
    want = [under_rules(logits[r], r, t) for r in range(rows)]
    t["last"][:] = last
    out = torch.full((rows, vocab), 77.0, device="cuda")
    token, best, status = run_rules(nv, logits, vocab, active, slots, rules_of(nv, t), out, vocab)
    for r, x in enumerate(want):
        assert int(token[r]) == int((x == x.max()).nonzero()[0]) and float(best[r]) == float(x.max())
        assert torch.equal(out[r].double(), x)
    assert status == 0


@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("out_type", [torch.float32, torch.float16, torch.bfloat16])
def test_w8a8_bad_rows_stay_bad(act, out_type):
    """A row with an infinity or NaN gives NaN, whatever the activation; the others what they give alone."""
    from cohere_inference_b200.packing import W8A8Linear
    g = gen(2)
    m, k, n = 70, 200, 90
    lin = W8A8Linear.from_weight(torch.randn(n, k, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda"), act)
    x = torch.randn(m, k, generator=g, device="cuda")
    clean = lin(x, dtype=out_type)
    x[4, 9], x[5, 0], x[6, k - 1] = math.nan, math.inf, -math.inf
    y = lin(x, dtype=out_type)
    assert y[4:7].isnan().all()
    rest = torch.arange(m, device="cuda")
    rest = rest[(rest < 4) | (rest > 6)]
    assert torch.equal(y[rest], clean[rest]) and (act != "relu" or (clean >= 0).all())


NOTHING = np.zeros(16384, bool)


@pytest.mark.parametrize("kw", [dict(), dict(chains=2, slots=16, buckets=(16,)), dict(graphs=False, pdl=0)])
def test_only_choices_that_are_taken_are_reported(model16, kw):
    """A mask that allows nothing is no mistake of a row whose prompt is still fed, nor of one that has ended; it is one as soon as
    the row's choice is taken."""
    from cohere_inference_b200.native import NativeError
    dec = decoder(model16, int8=True, logit_rules=True, **kw)
    frames, memory, prompts = [60, 60], torch.randn(120, 1024, device="cuda"), [np.arange(1, 11), np.arange(3, 5)]
    with torch.cuda.stream(dec.stream):
        dec.stream.wait_stream(torch.cuda.default_stream())
        dec.fill_cross(memory, frames, [1, 6])
    dec.admit([1, 6], prompts, frames, max_new=[48, 3], rules=[dict(mask=NOTHING), None])
    b = dec.set_active([1, 6])
    for _ in range(4):  # the second: one step of its prompt, then the three tokens of its budget
        dec.step(b)
    dec.check_status()
    assert int(dec.finished[6]) == 1
    dec.set_mask([6], [NOTHING])
    for _ in range(5):  # the first: positions 5 to 9 of its prompt
        dec.step(b)
    dec.check_status()
    assert int(dec.pos[1]) == 9 and int(dec.tok[1]) == 10
    dec.step(b)
    with pytest.raises(NativeError, match="left no token"):
        dec.check_status()
    assert int(dec.tok[1]) == 0


def test_w8a8_check_status(nv):
    """Nothing to report after calls; a word set on the device (as a wait that runs out sets it) is reported and cleared."""
    from cohere_inference_b200.packing import W8A8Linear
    lin = W8A8Linear(torch.eye(64, dtype=torch.int8, device="cuda"), torch.ones(64, device="cuda"))
    x = torch.randn(5, 64, device="cuda")
    y = lin(x)
    lin.check_status()
    with torch.cuda.stream(torch.cuda.Stream()):
        lin.status.fill_(nv.ST_TIMEOUT)
        with pytest.raises(nv.NativeError, match="ran out"):
            lin.check_status()
    assert torch.equal(lin(x), y)
    lin.check_status()


def test_rules_of_requests_reach_the_decoder(model16):
    """Through DecodeScheduler: a banned token never comes, where it came without the ban, and penalised requests get the tokens that a
    decoder gives which admits the same rules directly (steps of eight rows on both sides: a row's bits are its own)."""
    from cohere_inference_b200.scheduler import DecodeScheduler
    plain = [SimpleNamespace(**{**r.__dict__, "frames": min(r.frames, 60), "target": 20}) for r in synthetic_requests(12, seed=3)]
    memory = lambda r: np.random.default_rng(r.frames).standard_normal((r.frames, 1024)).astype(np.float32)  # noqa: E731
    new = lambda: decoder(model16, int8=True, logit_rules=True, buckets=(8,))  # noqa: E731
    run = lambda rs: [np.asarray(x) for x in DecodeScheduler(new(), memory).run(rs)]  # noqa: E731
    before = run(plain)
    made = [t[len(r.prompt):] for t, r in zip(before, plain)]
    rules = [dict(bias={int(v): -math.inf for v in set(made[i][::2].tolist())}) if i % 2 else dict(repetition=2.0 if i % 4 else 0.25)
             for i in range(12)]
    ruled = [SimpleNamespace(**{**r.__dict__, "rules": x}) for r, x in zip(plain, rules)]
    got = run(ruled)
    for i in range(1, 12, 2):
        assert not set(got[i][len(plain[i].prompt):].tolist()) & set(rules[i]["bias"])
    for i in range(0, 12, 2):
        dec, n = new(), len(plain[i].prompt)
        with torch.cuda.stream(dec.stream):
            dec.fill_cross(torch.from_numpy(memory(plain[i])).cuda(), [plain[i].frames], [0])
        dec.admit([0], [np.asarray(plain[i].prompt)], [plain[i].frames], [20], rules=[rules[i]])
        b = dec.set_active([0])
        for _ in range(n - 1 + 20):
            dec.step(b)
        dec.check_status()
        assert np.array_equal(got[i], dec.out[0, :n + 20].cpu().numpy())
    # some repeat themselves without a penalty, some do not: one of the two penalties shows
    assert sum(not np.array_equal(got[i], before[i]) for i in range(0, 12, 2)) >= 3
