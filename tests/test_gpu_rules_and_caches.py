"""The decoder's 4-bit caches, 8-bit prefill and rules on the logits, through StreamDecoder and DecodeScheduler: against the
oracle and against plain arithmetic on what the decoder holds."""

import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from cohere_inference_b200.synth import synthetic_model, synthetic_requests

pytestmark = pytest.mark.gpu




@pytest.fixture(scope="module")
def model16():
    return synthetic_model(0)


def decoder(model, **kw):
    from cohere_inference_b200 import StreamDecoder
    return StreamDecoder(model.cuda(), **{**dict(slots=8, max_new_tokens=48, max_prompt=16, max_audio_s=30.0, eos=-1), **kw})


def inputs(seed=17):
    rng = np.random.default_rng(seed)
    frames = [50, 375, 211, 125, 300]
    memory = [rng.standard_normal((t, 1024)).astype(np.float32) for t in frames]
    prompts = [rng.integers(0, 16384, n).astype(np.int64) for n in (10, 3, 16, 1, 10)]
    return frames, memory, prompts, [5, 0, 7, 2, 3]


def start(dec, rules=None, dtype=torch.float32, seed=17):
    frames, memory, prompts, slots = inputs(seed)
    with torch.cuda.stream(dec.stream):
        dec.fill_cross(torch.from_numpy(np.concatenate(memory)).cuda().to(dtype), frames, slots)
    dec.admit(slots, prompts, frames, **({} if rules is None else dict(rules=rules)))
    return slots, dec.set_active(slots)


def values(codes, pairs):
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double().unflatten(-1, (-1, 64))
    return (q * pairs[..., :1].double() + pairs[..., 1:].double()).flatten(-2)


def stored(x):
    """(..., D) -> the values a 4-bit cache holds of it, and half of each value's step."""
    x = x.bfloat16().double().unflatten(-1, (-1, 64))
    lo = x.amin(-1, keepdim=True).half().double()
    step = ((x.amax(-1, keepdim=True) - lo) / 15).half().double()
    return (lo + ((x - lo) / step).round().clamp(0, 15) * step).flatten(-2), (step / 2 + 0 * x).flatten(-2)


@pytest.mark.parametrize("heads", [16, 8])
def test_prefill_fills_4_bit_caches(model16, heads):
    """fill_cross into 4-bit caches holds what the quantiser makes of the keys and values that it writes into bf16 caches; both
    come from the same product, so codes differ only where the fp32 result rounds to another bf16 (never: same kernel)."""
    model = model16 if heads == 16 else synthetic_model(3, heads=8, head_dim=128, act="relu")
    plain, small = decoder(model, int8=True), decoder(model, int8=True, kv_int4=True)
    frames, _, _, slots = inputs()
    for dec in (plain, small):
        start(dec)
        dec.stream.synchronize()
        dec.check_status()
    for part in ("k", "v"):
        full, codes, pairs = getattr(plain, "cross_" + part), getattr(small, "cross_" + part), getattr(small, f"cross_{part}s")
        for n, s in zip(frames, slots):
            want, _ = stored(full[:, s, :, :n].float())
            assert torch.equal(values(codes[:, s, :, :n], pairs[:, s, :, :n]), want)
        assert int(codes[:, slots[0], :, frames[0]:].sum()) == 0  # behind the clip nothing was written


@pytest.mark.parametrize("mode", [dict(int8=True), dict(), dict(fp16_weights=True), dict(int8=True, ffn_sparse=True)])
@pytest.mark.parametrize("heads", [16, 8])
def test_steps_over_4_bit_caches(model16, heads, mode):
    """Forty steps over 4-bit caches: every self-attention key and value is the quantiser's image of what the step computed (its
    neighbours' steps say how far), and a second decoder, or the same one replayed, gives the same bits."""
    model = model16 if heads == 16 else synthetic_model(3, heads=8, head_dim=128, act="relu")
    dec = decoder(model, kv_int4=True, record=True, **mode)
    runs = []
    for _ in range(2):
        dec.reset()
        slots, b = start(dec)
        for _ in range(40):
            dec.step(b)
        dec.stream.synchronize()
        dec.check_status()
        runs.append((dec.out.clone(), dec.logits[:5].clone(), dec.self_k[:, slots, :, :40].clone()))
    for x, y in zip(*runs):
        assert torch.equal(x, y)
    # the same tokens forced into a bf16-cache decoder: layer 0's keys come from the embedding alone, so its caches hold the
    # same vectors, here in 4 bits
    ref = decoder(model, **mode)
    slots, b = start(ref)
    for t in range(40):
        ref.step(b)
        ref.stream.synchronize()
        ref.tok.copy_(dec.out[:, min(t + 1, dec.out.shape[1] - 1)])
    for part in ("k", "v"):
        full = getattr(ref, "self_" + part)[0, slots, :, :40].float()
        got = values(getattr(dec, "self_" + part)[0, slots, :, :40], getattr(dec, f"self_{part}s")[0, slots, :, :40])
        want, half = stored(full)
        # one bf16 step of the product's rounding order apart at most, and half a step of the format
        assert ((got - full.double()).abs() <= half * 1.01 + 2.0 ** -8 * full.abs().double() + 2.0 ** -11 * want.abs()).all()


@pytest.mark.parametrize("heads", [16, 8])
@pytest.mark.parametrize("rows", [5, 40])
def test_steps_over_4_bit_caches_do_not_depend_on_how_they_are_launched(model16, heads, rows):
    """Graphs of programmatic launches against plain launches, one kernel fully before the next: the same bits for 60 steps, so
    no step reads a key or a pair from before it was written."""
    model = model16 if heads == 16 else synthetic_model(3, heads=8, head_dim=128, act="relu")
    rng = np.random.default_rng(9)
    frames = rng.integers(20, 300, rows).tolist()
    memory = torch.randn(sum(frames), 1024, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    prompts, slots = [rng.integers(0, 16384, 5) for _ in range(rows)], list(range(rows))
    got = []
    for kw in (dict(), dict(pdl=0, graphs=False)):
        dec = decoder(model, slots=48, max_new_tokens=70, int8=True, kv_int4=True, record=True, **kw)
        with torch.cuda.stream(dec.stream):
            dec.fill_cross(memory, frames, slots)
        dec.admit(slots, prompts, frames)
        b = dec.set_active(slots)
        for _ in range(60):
            dec.step(b)
        dec.stream.synchronize()
        dec.check_status()
        got.append((dec.out[:rows].clone(), dec.logits[:rows].clone(), dec.self_k.clone(), dec.self_vs.clone()))
    for x, y in zip(*got):
        assert torch.equal(x[:, :rows] if x.dim() > 2 else x, y[:, :rows] if y.dim() > 2 else y)


def test_4_bit_caches_stay_near_the_oracle(model16):
    """Logits over 4-bit caches against the bf16-cache decoder on the same tokens. A cached value is off by at most half a
    step, a fifteenth of its group's range / 2, that is about 0.1 of its spread, at random: with 50 keys and more an
    attention output moves by a few percent, which eight layers pass on; the logits' spread is about 1."""
    full, small = (decoder(model16, int8=True, record=True, kv_int4=x) for x in (False, True))
    slots, b = start(full)
    start(small)
    far = []
    for t in range(30):
        full.step(b), small.step(b)
        full.stream.synchronize(), small.stream.synchronize()
        far.append(float((full.logits[:5] - small.logits[:5]).abs().max()))
        small.tok.copy_(full.tok)
    spread = float(full.logits[:5].std())
    print(f"4-bit caches: largest logit difference {max(far):.3f}, spread {spread:.3f}")
    assert max(far) <= 0.5 * spread


@pytest.mark.parametrize("kw", [dict(), dict(kv_int8=True), dict(kv_int4=True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [16, 8])
def test_prefill_in_8_bits(model16, heads, dtype, kw):
    """fill_cross with both products in 8-bit integers against the same arithmetic in 64 bits."""
    from cohere_inference_b200.packing import quantize_rows
    model = (model16 if heads == 16 else synthetic_model(3, heads=8, head_dim=128, act="relu", bias_std=0.05)).cuda()
    dec = decoder(model, int8=True, prefill_int8=True, **kw)
    frames, memory, _, slots = inputs()
    x = torch.from_numpy(np.concatenate(memory)).cuda().to(dtype)
    start(dec, dtype=dtype)
    dec.stream.synchronize()
    dec.check_status()
    d = model.model.decoder

    def product(a, w, b):
        s = (a.abs().amax(1, keepdim=True) / 127).float().double()
        q, sw = quantize_rows(w.float())
        return ((a / s).round() @ q.double().T) * s * sw.double() + b.double()
    mid = product(x.double(), d.proj.weight, d.proj.bias).float().double()
    cur = 0
    for li, layer in enumerate(d.layers):
        for part, proj in (("k", layer.encoder_attn.k_proj), ("v", layer.encoder_attn.v_proj)):
            y = product(mid, proj.weight, proj.bias).unflatten(1, (dec.h, dec.d))
            cur = 0
            for n, s in zip(frames, slots):
                want = y[cur:cur + n].transpose(0, 1)
                cur += n
                cache, extra = getattr(dec, "cross_" + part)[li, s, :, :n], getattr(dec, f"cross_{part}s")
                # the rows between are fp32: a code of the second product can fall on the other side of a half, one 127th of its
                # row's largest value times one weight; and the formats' own rounding on top (bf16, then half a step)
                scale = (mid.abs().amax() / 127) * proj.weight.abs().max().double()
                slack = 4 * scale + 2.0 ** -8 * want.abs()
                if dec.kv_int4:
                    got, step = values(cache, extra[li, s, :, :n]), extra[li, s, :, :n, :, 0].double().repeat_interleave(64, -1)
                    slack = slack + 0.51 * step + 2.0 ** -10 * want.abs()
                elif dec.kv_int8:
                    got = cache.double() * extra[li, s, :, :n, None].double()
                    slack = slack + 0.51 * extra[li, s, :, :n, None].double()
                else:
                    got = cache.double()
                assert ((got - want).abs() <= slack).all()


def test_packed_8_bit_prefill_round_trip(model16, tmp_path):
    dec = decoder(model16, int8=True, prefill_int8=True, kv_int4=True, logit_rules=True)
    path = str(tmp_path / "packed.pt")
    digest = dec.save_packed(path)
    from cohere_inference_b200 import StreamDecoder
    again = StreamDecoder.from_packed(path, slots=8, max_new_tokens=48, max_prompt=16, max_audio_s=30.0, eos=-1, kv_int4=True,
                                      logit_rules=True)
    assert again.weights_digest() == digest and again.prefill_int8 and again.kv_int4
    outs = []
    for d in (dec, again):
        slots, b = start(d, [dict(repetition=1.3)] * 5)
        for _ in range(20):
            d.step(b)
        d.stream.synchronize()
        d.check_status()
        outs.append((d.out.clone(), d.cross_k.clone()))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


RULES = [dict(repetition=1.5), dict(presence=0.75, frequency=0.25), None,
         dict(repetition=0.5, bias={7: 2.0, 9: -math.inf, 16383: 1.5, 0: -1.0}), dict(frequency=-0.5, bias={11: 0.25})]


def expected(dec, row, slot, rule, mask):
    """The token the rules choose from the row's logits (fp64), and how close another one comes."""
    x = dec.logits[row].double()
    pos, plen = int(dec.pos[slot]), int(dec.plen[slot])
    hist = dec.out[slot, :pos].cpu().tolist()  # the step has advanced: its own choice is at pos
    r = rule or {}
    rep = r.get("repetition", 1.0)
    for v in set(hist):
        x[v] = x[v] / rep if x[v] > 0 else x[v] * rep
    made = hist[plen:]
    for v in set(made):
        x[v] -= r.get("frequency", 0.0) * made.count(v) + r.get("presence", 0.0)
    for v, b in r.get("bias", {}).items():
        x[v] += b
    if mask is not None:
        x[~torch.as_tensor(mask).cuda()] = -math.inf
    top = torch.topk(x, 2)
    return int(top.indices[0]), float(top.values[0] - top.values[1])


@pytest.mark.parametrize("kw", [dict(int8=True), dict(), dict(int8=True, kv_int4=True, device_sched=True), dict(int8=True, head_umma=False),
                                dict(int8=True, graphs=False), dict(fp16_weights=True, chains=2)])
def test_rules_in_the_step(model16, kw):
    """Every step's choice of every row is the one its rules give for the logits the step computed; a mask set between the steps
    counts from the next one on; a slot admitted again starts without the rules it had."""
    dec = decoder(model16, logit_rules=True, **kw)
    slots, b = start(dec, RULES)
    rng = np.random.default_rng(1)
    masks = [None] * 5
    checked = 0
    for t in range(40):
        if t == 20:
            masks[1], masks[2] = rng.random(16384) < 0.3, rng.random(16384) < 0.01
            dec.set_mask([slots[1], slots[2]], [masks[1], torch.from_numpy(masks[2])])
        if t == 30:
            masks[1] = None
            dec.set_mask([slots[1]], [None])
        dec.step(b)
        dec.stream.synchronize()
        for row, (s, rule) in enumerate(zip(slots, RULES)):
            if int(dec.pos[s]) < int(dec.plen[s]):
                continue  # the prompt is forced
            token, gap = expected(dec, row, s, rule, masks[row])
            if gap > 1e-5:  # fp32 rounds five times, of values below 20
                assert int(dec.tok[s]) == token, (t, row)
                checked += 1
    assert checked > 120
    dec.check_status()
    # the same slots again, without rules: the tokens of a plain decoder on the same kernels (a fused step adds up in another
    # order, which turns a near-tie now and then)
    plain = decoder(model16, **{**kw, "fused_rows": 0})
    dec.reset()
    for d in (dec, plain):
        start(d, seed=23)
        for _ in range(30):
            d.step(b)
        d.stream.synchronize()
    assert torch.equal(dec.out[slots], plain.out[slots])


def test_a_mask_that_allows_nothing_is_reported(model16):
    dec = decoder(model16, int8=True, logit_rules=True)
    slots, b = start(dec, [None, dict(mask=np.zeros(16384, bool)), None, None, None])
    for _ in range(6):
        dec.step(b)
    dec.stream.synchronize()
    assert int(dec.tok[slots[1]]) == 0
    from cohere_inference_b200.native import NativeError
    with pytest.raises(NativeError, match="left no token"):
        dec.check_status()


def test_rules_through_the_scheduler(model16):
    """Requests that ban a token never get it, those that may only say two tokens say them; the others are as without rules."""
    from cohere_inference_b200.scheduler import DecodeScheduler
    reqs = synthetic_requests(12, seed=3)
    only = np.zeros(16384, bool)
    only[[5, 6]] = True
    plain = [SimpleNamespace(**{**r.__dict__, "frames": min(r.frames, 60), "target": 20}) for r in reqs]
    ruled = [SimpleNamespace(**{**r.__dict__, "rules": None if i % 3 == 0 else dict(mask=only) if i % 3 == 1 else dict(repetition=2.0)})
             for i, r in enumerate(plain)]
    memory = lambda r: np.random.default_rng(r.frames).standard_normal((r.frames, 1024)).astype(np.float32)  # noqa: E731
    got = []
    for rs in (plain, ruled):
        dec = decoder(model16, int8=True, kv_int4=True, logit_rules=True)
        got.append(DecodeScheduler(dec, memory).run(rs))
        dec.check_status()
    for i in range(12):
        a, b = (np.asarray(got[k][i]) for k in (0, 1))
        if i % 3 == 0:
            assert np.array_equal(a, b)
        elif i % 3 == 1:
            assert set(b[len(plain[i].prompt):].tolist()) <= {5, 6}


def test_refusals(model16):
    from cohere_inference_b200 import StreamDecoder
    m = model16.cuda()
    with pytest.raises(AssertionError):
        StreamDecoder(m, slots=2, int8=True, kv_int4=True, kv_int8=True)
    with pytest.raises(AssertionError):
        StreamDecoder(m, slots=2, kv_int4=True, attn_ring=True)
    with pytest.raises(ValueError):
        StreamDecoder(m, slots=2, logit_rules=True, max_bias=0)
    dec = decoder(model16, int8=True, logit_rules=True, max_bias=3)
    prompt = [np.array([1, 2])]
    for bad in ([], [None, None], [dict(temperature=1.0)], [dict(repetition=0.0)], [dict(repetition=float("nan"))],
                [dict(presence=float("inf"))], [dict(bias={1: 1.0, 2: 1.0, 3: 1.0, 4: 1.0})], [dict(bias={16384: 1.0})],
                [dict(bias={-1: 1.0})], [dict(bias={1: float("nan")})], [dict(mask=np.ones(16383, bool))], [dict(mask=np.ones(16384))]):
        with pytest.raises(ValueError):
            dec.admit([0], prompt, [5], rules=bad)
    for slots, masks in (([0], []), ([8], [None]), ([-1], [None]), ([0], [np.ones(3, bool)])):
        with pytest.raises(ValueError):
            dec.set_mask(slots, masks)
    plain = decoder(model16, int8=True)
    with pytest.raises(ValueError):
        plain.admit([0], prompt, [5], rules=[None])
    with pytest.raises(ValueError):
        plain.set_mask([0], [None])
