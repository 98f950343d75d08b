"""What the operators' Python side does on the host: no GPU, the device's words are set by hand."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from cohere_inference_b200 import native as nv
from cohere_inference_b200.packing import W8A8Linear
from cohere_inference_b200.scheduler import DecodeScheduler
from cohere_inference_b200.stream_decoder import StreamDecoder


def test_w8a8_status_is_reported_once():
    lin = object.__new__(W8A8Linear)
    lin.status = torch.zeros(1, dtype=torch.int32)
    lin.check_status()
    lin.status |= nv.ST_TIMEOUT
    with pytest.raises(nv.NativeError, match="ran out"):
        lin.check_status()
    assert int(lin.status) == 0
    lin.check_status()


@pytest.mark.parametrize("raw", [None, lambda device: 100 + device])
def test_stream_handle(monkeypatch, raw):
    """With and without torch's undocumented way to the current stream's handle."""
    monkeypatch.setattr(nv, "_raw_stream", raw)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: SimpleNamespace(cuda_stream=101))
    assert nv.stream_ptr() == 101 and nv.stream_ptr(SimpleNamespace(cuda_stream=7)) == 7


def rule_tables(rules):
    d = SimpleNamespace(vocab=20, max_bias=4, _rule_ints=6 + 2 * 4 + 1)
    return StreamDecoder._rule_tables(d, list(range(len(rules))), rules)


class Decoder:
    """As much of a decoder as a run looks at before its first request; a call that starts one fails the test."""
    slots, max_new_tokens, eos = 3, 8, -1
    vocab, max_bias, _rule_ints = 20, 4, 6 + 2 * 4 + 1
    check_rules, _rule_tables, _mask_words = StreamDecoder.check_rules, StreamDecoder._rule_tables, StreamDecoder._mask_words

    def __init__(self, logit_rules):
        self.logit_rules, self.out = logit_rules, np.zeros((4, 12), np.int64)

    def fill_cross(self, *args):
        raise AssertionError("a request was started")

    admit = set_active = step = fill_cross


@pytest.mark.parametrize("logit_rules, rules", [(False, dict(repetition=2.0)), (True, dict(repetition=-2.0)), (True, dict(mask=np.ones(19, bool)))])
def test_a_run_refuses_rules_before_it_starts(logit_rules, rules):
    """The last request's rules are refused before the first is admitted, and the scheduler keeps its slots."""
    request = lambda **kw: SimpleNamespace(prompt=[1, 2], frames=5, target=4, arrival=0.0, **kw)  # noqa: E731
    sched = DecodeScheduler(Decoder(logit_rules), lambda r: np.zeros((r.frames, 4), np.float32))
    with pytest.raises(ValueError):
        sched.run([request(), request(rules=None), request(rules=rules)])
    assert sorted(sched.free) == [0, 1, 2] and sched.stats.admitted == 0


@pytest.mark.parametrize("rule", [
    dict(repetition=1e-50), dict(repetition=1e39), dict(repetition=-1.0), dict(presence=1e39), dict(frequency=-1e39),
    dict(bias={3: 1e39}), dict(bias={3: -3.5e38}), dict(bias={3.7: 1.0}), dict(bias={np.float32(0.5): 1.0}),
])
def test_rules_that_the_tables_cannot_hold_are_refused(rule):
    with pytest.raises(ValueError):
        rule_tables([rule])


def test_rules_that_the_tables_hold():
    rec = rule_tables([dict(repetition=1e-40, presence=3e38, frequency=-3e38, bias={3: np.inf, 4.0: -np.inf, "5": 3.4e38, np.int64(6): 1}),
                       None, dict(repetition=np.float32(1.25), bias={})])
    f = rec.view(np.float32)
    assert rec[:, 0].tolist() == [0, 1, 2] and rec[:, 4].tolist() == [4, 0, 0] and rec[0, 6:10].tolist() == [3, 4, 5, 6]
    assert np.array_equal(f[0, 1:4], np.array([1e-40, 3e38, -3e38], np.float32)) and f[0, 1] > 0
    assert np.array_equal(f[0, 10:14], np.array([np.inf, -np.inf, 3.4e38, 1.0], np.float32))
    assert f[1, 1:4].tolist() == [1.0, 0.0, 0.0] and f[2, 1:4].tolist() == [1.25, 0.0, 0.0]


def test_how_far_the_4_bit_format_is_off():
    """Half a step; 2^-21 more where the step or the lowest value is below fp16's normal numbers. In 64 bits, from the definition."""
    rng = np.random.default_rng(0)
    off, spread = (10.0 ** rng.uniform(-9, 4.5, (2, 4000, 1)))
    x = torch.from_numpy(rng.choice([-1.0, 0.0, 1.0], (4000, 1)) * off + spread * rng.standard_normal((4000, 64)))
    x[0], x[1], x[2, 1:] = 3.7, -2.0 ** -20, x[2, 0]  # constant groups
    x = x.clamp(-32752.0, 32752.0).bfloat16().double()
    lo = x.amin(1, keepdim=True).half().double()
    step = ((x.amax(1, keepdim=True) - lo) / 15).half().double()
    code = torch.where(step > 0, ((x - lo) / torch.where(step > 0, step, 1.0)).round().clamp(0, 15), 0.0)
    far = (lo + code * step - x).abs() - step.abs() / 2
    normal = ((step >= 2.0 ** -14) & (lo.abs() >= 2.0 ** -14)).flatten()
    assert normal.sum() > 500 and (~normal).sum() > 500
    assert far[normal].max() <= 0 and far.max() <= 2.0 ** -21
