"""Operators around the decoding step, as measured cases: attention over a key/value cache held in 4 bits, the fill of
such a cache, rules on the logits (penalties for repeated tokens, biases, grammar masks) with the greedy choice, and the
matrix product in 8-bit integers with a scale for each row and each channel.

A case is a dict of plain values. `run` computes the operator in elementary torch operations, or, with `own` set, by the
calls a user of this package makes; `exact` computes it from its definition in 64 bits.

The definitions
  4-bit cache   a head vector is rounded to bf16 (clamped to +-32752, NaN as 0) and cut into groups of 64 dims; per group
                lo = fp16(min), step = fp16((max - lo) / 15), code = clamp(rint((x - lo) / step), 0, 15) (0 where step is
                0), and the value it stands for is lo + code * step. Byte i of a vector holds dim 2i in its low half and
                dim 2i + 1 in its high half; the group's (step, lo) lie beside it as two fp16 numbers.
  attention     one new token per row over its slot's cached keys and values. Self: the row's new key and value are
                written at position n and attended as bf16 values beside the n cached ones. Cross: n cached ones; a row
                without any gives zeros.
  rules         a token's logit x: x / r or x * r (x > 0 or not) where the token occurs in the slot's tokens so far,
                less frequency * (times generated), less presence where generated, plus the biases listed for it, and
                -inf where the slot's mask leaves it out; then the first index of the largest.
  product       q = rint(x / s) with s = max(|row|) / 127 per row, y = (q . w) * s * s_w + bias.
"""

import math

import torch

own = False

ATTEND, FILL, RULES, PRODUCT = "attend", "fill", "rules", "product"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = 32752.0  # the 4-bit format's largest magnitude: a group's range then stays inside fp16


def listed():
    return [
        # one speaker's stream: the smallest step there is, 8 x 128 heads, self-attention of a half-spoken sentence
        dict(name="attend-self-one", op=ATTEND, self=True, rows=1, heads=8, dim=128, cap=465, shortest=217, longest=217,
             out="f16"),
        # cross-attention of a full batch of clips of 50 to 375 frames, 16 x 64 heads
        dict(name="attend-cross-64", op=ATTEND, self=False, rows=64, heads=16, dim=64, cap=451, shortest=50, longest=375,
             out="f16"),
        # 128 slots of ragged lengths, some just admitted, the step of the continuous batch
        dict(name="attend-self-128", op=ATTEND, self=True, rows=128, heads=16, dim=64, cap=465, shortest=0, longest=457,
             out="f16"),
        # hours of audio in a row: few rows over a long axis, odd lengths, fp32 out for the split-operand mode
        dict(name="attend-long", op=ATTEND, self=False, rows=24, heads=8, dim=128, cap=33000, shortest=1, longest=32771,
             out="f32"),
        # one admitted clip of 14 s into the caches of 8 layers
        dict(name="fill-one", op=FILL, clips=1, shortest=175, longest=175, layers=8, heads=8, dim=128, frames=451),
        # a full batch admitted at once
        dict(name="fill-64", op=FILL, clips=64, shortest=50, longest=375, layers=8, heads=16, dim=64, frames=451),
        # one stream with a repetition penalty, a few banned tokens and a grammar
        dict(name="rules-one", op=RULES, rows=1, vocab=16384, kind="f32", history=217, biases=24, mask=True, out=False),
        # the same for 128 slots
        dict(name="rules-128", op=RULES, rows=128, vocab=16384, kind="f32", history=457, biases=64, mask=True, out=False),
        # a large vocabulary in 16 bits, an odd one, the processed logits wanted too
        dict(name="rules-wide", op=RULES, rows=96, vocab=151931, kind="bf16", history=2100, biases=300, mask=True, out=True),
        # a step's rows through one feed-forward projection
        dict(name="product-64", op=PRODUCT, m=64, k=1024, n=4096, x="f32", out="f16", bias=True),
        # the encoder rows of a few clips, odd sizes
        dict(name="product-odd", op=PRODUCT, m=1571, k=1300, n=1111, x="bf16", out="f32", bias=True),
        # cross keys and values of all layers for 64 clips
        dict(name="product-cross", op=PRODUCT, m=13600, k=1024, n=16384, x="f32", out="bf16", bias=True),
    ]


def draw(rng):
    def spread(lo, hi):  # evenly over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice((ATTEND, ATTEND, FILL, RULES, RULES, PRODUCT))
    if op == ATTEND:
        dim = rng.choice((64, 128))
        heads = rng.choice((1024 // dim, 1024 // dim, rng.randint(1, 24)))
        rows = spread(1, 200)
        longest = spread(1, max(2, min(120000, 24 * 8 * 32771 * 128 // (rows * heads * dim * 2))))
        return dict(op=op, self=rng.random() < 0.5, rows=rows, heads=heads, dim=dim, cap=longest + rng.randint(1, 90),
                    shortest=rng.randint(0, longest), longest=longest, out=rng.choice(("f16", "f32")))
    if op == FILL:
        dim = rng.choice((64, 128))
        frames = rng.randint(20, 460)
        longest = rng.randint(1, frames)
        return dict(op=op, clips=spread(1, 48), shortest=rng.randint(1, longest), longest=longest,
                    layers=rng.randint(1, 8), heads=1024 // dim, dim=dim, frames=frames)
    if op == RULES:
        return dict(op=op, rows=spread(1, 128), vocab=spread(50, 110000), kind=rng.choice(("f32", "f16", "bf16")),
                    history=spread(1, 2100), biases=rng.choice((0, spread(1, 300))), mask=rng.random() < 0.7,
                    out=rng.random() < 0.5)
    return dict(op=op, m=spread(1, 12000), k=spread(40, 2500), n=spread(30, 7000), x=rng.choice(("f32", "f16", "bf16")),
                out=rng.choice(("f32", "f16", "bf16")), bias=rng.random() < 0.7)


def _lengths(c, count):
    """Evenly from the shortest to the longest."""
    lo, hi = c["shortest"], c["longest"]
    return [hi if count == 1 else lo + (hi - lo) * i // (count - 1) for i in range(count)]


def work(c):
    if c["op"] == ATTEND:
        keys, new = sum(_lengths(c, c["rows"])), c["rows"] if c["self"] else 0
        vec, one = c["dim"] // 2 + 4 * (c["dim"] // 64), c["heads"] * c["dim"]
        return {"bytes": 2 * keys * c["heads"] * vec + c["rows"] * one * (4 + TYPES[c["out"]].itemsize) +
                new * (2 * one * 4 + 2 * c["heads"] * vec + 2 * one * 4),
                "flops": 4 * (keys + new) * one}
    if c["op"] == FILL:
        values = sum(_lengths(c, c["clips"])) * c["layers"] * 2 * c["heads"] * c["dim"]
        return {"bytes": values * 8 + values // 2 + values // 16, "flops": 6 * values}
    if c["op"] == RULES:
        size, cells = TYPES[c["kind"]].itemsize, c["rows"] * c["vocab"]
        return {"bytes": cells * size * (2 if c["out"] else 1) + (cells // 8 if c["mask"] else 0) +
                c["rows"] * (8 * c["history"] + 8 * c["biases"] + 24), "flops": 2 * cells}
    m, k, n = c["m"], c["k"], c["n"]
    return {"bytes": m * k * TYPES[c["x"]].itemsize + n * k + 4 * n * (2 if c["bias"] else 1) +
            m * n * TYPES[c["out"]].itemsize, "flops": 2 * m * n * k}


# ---- the 4-bit format ---------------------------------------------------------------------------------------------------


def _quantise(x):
    """x (..., D) fp32 -> codes uint8 (..., D / 2) and (step, lo) fp16 (..., D / 64, 2)."""
    g = x.bfloat16().float().nan_to_num(0.0, LIMIT, -LIMIT).clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 64))
    lo = g.amin(-1).half()
    step = ((g.amax(-1).double() - lo.double()) / 15).half()
    s = step.float().unsqueeze(-1)
    code = ((g - lo.float().unsqueeze(-1)).double() / s.double()).round().clamp(0, 15)
    code = torch.where(s > 0, code, 0.0).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.stack((step, lo), -1)


def _values(codes, meta):
    """What codes and (step, lo) stand for, in fp32."""
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, 64))
    return (q * meta[..., :1].float() + meta[..., 1:].float()).flatten(-2)


# ---- inputs -------------------------------------------------------------------------------------------------------------


def prepare(c, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    return {ATTEND: _prepare_attend, FILL: _prepare_fill, RULES: _prepare_rules, PRODUCT: _prepare_product}[c["op"]](c, gen, host)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _prepare_attend(c, gen, host):
    rows, heads, dim, cap = c["rows"], c["heads"], c["dim"], c["cap"]
    lens = torch.tensor(_lengths(c, rows), dtype=torch.int32)[torch.randperm(rows, generator=host)]
    slots = rows + 2  # two more than are active, and the dummy slot behind them
    active = torch.randperm(slots, generator=host)[:rows].to(torch.int32)
    n = torch.ones(slots + 1, dtype=torch.int32)
    n[active.long()] = lens
    codes, meta = [], []
    offset = _randn(gen, 2, heads, 1, dim)  # channels have means of their own
    for part in range(2):
        k = torch.zeros(slots + 1, heads, cap, dim // 2, dtype=torch.uint8, device="cuda")
        m = torch.zeros(slots + 1, heads, cap, dim // 64, 2, dtype=torch.float16, device="cuda")
        for s in range(slots + 1):
            k[s], m[s] = _quantise(_randn(gen, heads, cap, dim) + offset[part])
        codes.append(k), meta.append(m)
    q = _randn(gen, rows, (3 if c["self"] else 1) * heads * dim)
    s = dict(c, active=active.cuda(), n=n.cuda(), q=q, k=codes[0], v=codes[1], km=meta[0], vm=meta[1], slots=slots,
             out_t=torch.empty(rows, heads * dim, dtype=TYPES[c["out"]], device="cuda"))
    s["at"] = s["n"][s["active"].long()]  # the position each row appends at
    s["kv"] = torch.empty(rows, 2 * heads * dim, device="cuda")
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if own:
        from cohere_inference_b200 import native as nv
        words = nv.lib().b200dec_attention_q4_scratch_floats(rows, heads, dim, cap)
        s["part"] = torch.empty(words, device="cuda")
        s["count"] = torch.zeros(rows * heads, dtype=torch.int32, device="cuda")
    return s


def _prepare_fill(c, gen, host):
    lens = _lengths(c, c["clips"])
    slots = torch.randperm(c["clips"], generator=host).tolist()
    slot_of = torch.cat([torch.full((n,), s, dtype=torch.int32) for s, n in zip(slots, lens)])
    frame_of = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens])
    L, heads, dim, rows = c["layers"], c["heads"], c["dim"], sum(lens)
    kv = _randn(gen, rows, L * 2 * heads * dim) * 0.7 + _randn(gen, L * 2 * heads * dim)
    cache = (L, c["clips"] + 1, heads, c["frames"])
    return dict(c, rows=rows, kv=kv, slot_of=slot_of.cuda(), frame_of=frame_of.cuda(), back=torch.empty_like(kv),
                k=torch.zeros(*cache, dim // 2, dtype=torch.uint8, device="cuda"),
                v=torch.zeros(*cache, dim // 2, dtype=torch.uint8, device="cuda"),
                km=torch.zeros(*cache, dim // 64, 2, dtype=torch.float16, device="cuda"),
                vm=torch.zeros(*cache, dim // 64, 2, dtype=torch.float16, device="cuda"))


def _prepare_rules(c, gen, host):
    rows, vocab, cols, slots = c["rows"], c["vocab"], c["history"], c["rows"] + 1
    rand = lambda *shape: torch.rand(*shape, generator=host)  # noqa: E731
    active = torch.randperm(slots, generator=host)[:rows].to(torch.int32)
    # text repeats itself: ids fall off quickly from the most frequent one
    history = (vocab * rand(slots + 1, cols) ** 4).long().clamp(max=vocab - 1)
    last = (cols * (1 - 0.6 * rand(slots + 1))).int().clamp(0, cols - 1)
    if rows > 2:
        last[active[1].long()] = -1  # a slot without a token yet
    plen = (1 + 10 * rand(slots + 1)).int()
    params = torch.stack((1 + 0.5 * rand(slots + 1), rand(slots + 1), 0.3 * rand(slots + 1), torch.zeros(slots + 1)), 1)
    params[rand(slots + 1) < 0.2] = torch.tensor([1.0, 0.0, 0.0, 0.0])  # a request that asks for nothing
    width = max(1, c["biases"])
    ids = (vocab * rand(slots + 1, width)).int().clamp(max=vocab - 1)
    values = 4 * torch.randn(slots + 1, width, generator=host)
    values[rand(slots + 1, width) < 0.2] = -math.inf  # banned tokens
    count = (c["biases"] * (0.3 + 0.7 * rand(slots + 1))).ceil().int().clamp(max=c["biases"])
    words = -(-vocab // 32)
    # a grammar leaves a handful of tokens or nearly all of them
    bits = torch.randint(-2**31, 2**31, (4, slots + 1, words), generator=gen, device="cuda")
    few = (torch.rand(slots + 1, 1, generator=gen, device="cuda") < 0.5)
    mask = torch.where(few, bits[0] & bits[1] & bits[2] & bits[3], bits[0] | bits[1] | bits[2] | bits[3]).to(torch.int32)
    if rows >= 8:
        mask[active[2].long()] = 0  # a grammar at its dead end
    logits = (3 * _randn(gen, rows, vocab)).to(TYPES[c["kind"]])
    s = dict(c, slots=slots, words=words, active=active.cuda(), history_t=history.cuda(), last=last.cuda(),
             plen=plen.cuda(), params=params.cuda(), ids=ids.cuda(), values=values.cuda(), count=count.cuda(),
             mask_t=mask, logits=logits, out_t=torch.empty_like(logits) if c["out"] else None,
             best=torch.empty(rows, device="cuda"), token=torch.empty(rows, dtype=torch.int32, device="cuda"),
             status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if own:
        from cohere_inference_b200 import native as nv
        p = nv.ptr
        s["rules"] = nv.Rules(p(s["params"]), p(s["history_t"]), p(s["last"]), p(s["plen"]),
                              *((p(s["ids"]), p(s["values"]), p(s["count"])) if c["biases"] else (None, None, None)),
                              p(s["mask_t"]) if c["mask"] else None, None, cols, c["biases"])
    return s


def _prepare_product(c, gen, host):
    m, k, n = c["m"], c["k"], c["n"]
    x = _randn(gen, m, k) * (1 + 3 * (torch.rand(k, generator=gen, device="cuda") < 0.02))  # a few loud channels
    w = 0.02 * _randn(gen, n, k)
    scale = w.abs().amax(1) / 127
    q = (w / scale[:, None]).round().clamp(-127, 127).to(torch.int8)
    s = dict(c, x_t=x.to(TYPES[c["x"]]), q=q, scale=scale, bias_t=_randn(gen, n) if c["bias"] else None,
             out_t=torch.empty(m, n, dtype=TYPES[c["out"]], device="cuda"),
             status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if own:
        from cohere_inference_b200.packing import W8A8Linear
        s["linear"] = W8A8Linear(q, scale, s["bias_t"])
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return {ATTEND: _own_attend, FILL: _own_fill, RULES: _own_rules, PRODUCT: _own_product}[s["op"]](s)
    return {ATTEND: _attend, FILL: _fill, RULES: _rules, PRODUCT: _product}[s["op"]](s)


def _own_attend(s):
    from cohere_inference_b200 import native as nv
    lib, p, st = nv.lib(), nv.ptr, nv.stream_ptr()
    rows, heads, dim, cap, kind = s["rows"], s["heads"], s["dim"], s["cap"], nv.OUT_F16 if s["out"] == "f16" else nv.OUT_F32
    caches = p(s["k"]), p(s["v"]), p(s["km"]), p(s["vm"])
    nv.check(lib.b200dec_attention_q4(int(s["self"]), p(s["active"]), p(s["q"]), s["q"].shape[1], *caches, p(s["n"]), None,
                                      s["slots"], heads, dim, cap, dim ** -0.5, p(s["out_t"]), kind, rows, p(s["part"]),
                                      p(s["count"]), p(s["status"]), 0, st))
    if not s["self"]:
        return s["out_t"]
    nv.check(lib.b200dec_gather_kv_q4(p(s["kv"]), p(s["active"]), p(s["at"]), *caches, rows, 1, s["slots"] + 1, heads, dim,
                                      cap, st))
    return s["out_t"], s["kv"]


def _attend(s):
    rows, heads, dim = s["rows"], s["heads"], s["dim"]
    slot, at = s["active"].long(), s["at"].long()
    most = s["longest"]
    k = _values(s["k"][slot, :, :most], s["km"][slot, :, :most])  # (rows, heads, most, dim)
    v = _values(s["v"][slot, :, :most], s["vm"][slot, :, :most])
    parts = s["q"].view(rows, -1, heads, dim)
    q = parts[:, 0, :, :, None] * dim ** -0.5
    score = (k @ q).squeeze(-1)
    keep = torch.arange(most, device=slot.device) < at[:, None]
    score = score.masked_fill(~keep[:, None], -math.inf)
    if s["self"]:
        new = parts[:, 1:].bfloat16().float()  # (rows, 2, heads, dim)
        score = torch.cat((score, (new[:, 0, :, None] @ q).squeeze(-1)), -1)
        v = torch.cat((v, new[:, 1, :, None]), 2)
        heads_i = torch.arange(heads, device=slot.device)
        where = slot[:, None], heads_i, at[:, None]
        codes, meta = _quantise(parts[:, 1:])
        for cache, part in ((s["k"], 0), (s["v"], 1)):
            cache[where] = codes[:, part]
        for cache, part in ((s["km"], 0), (s["vm"], 1)):
            cache[where] = meta[:, part]
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    e = (score - top).exp()
    out = (e[:, :, None] @ v).squeeze(2) / e.sum(-1, keepdim=True).clamp(min=1e-38)
    out = out.flatten(1).to(TYPES[s["out"]])
    if not s["self"]:
        return out
    back = torch.stack((_values(s["k"][where], s["km"][where]), _values(s["v"][where], s["vm"][where])), 1)
    return out, back.flatten(1)


def _own_fill(s):
    from cohere_inference_b200 import native as nv
    lib, p, st = nv.lib(), nv.ptr, nv.stream_ptr()
    rest = (p(s["slot_of"]), p(s["frame_of"]), p(s["k"]), p(s["v"]), p(s["km"]), p(s["vm"]), s["rows"], s["layers"],
            s["clips"] + 1, s["heads"], s["dim"], s["frames"], st)
    nv.check(lib.b200dec_scatter_kv_q4(p(s["kv"]), *rest))
    nv.check(lib.b200dec_gather_kv_q4(p(s["back"]), *rest))
    return s["back"]


def _fill(s):
    slot, frame = s["slot_of"].long(), s["frame_of"].long()
    codes, meta = _quantise(s["kv"].view(s["rows"], s["layers"], 2, s["heads"], s["dim"]))
    back = []
    for part, (cache, m) in enumerate(((s["k"], s["km"]), (s["v"], s["vm"]))):
        cache[:, slot, :, frame] = codes[:, :, part]
        m[:, slot, :, frame] = meta[:, :, part]
        back.append(_values(cache[:, slot, :, frame], m[:, slot, :, frame]))
    return torch.stack(back, 2).flatten(1)


def _own_rules(s):
    import ctypes
    from cohere_inference_b200 import native as nv
    p = nv.ptr
    kind = {"f32": nv.T_F32, "f16": nv.T_F16, "bf16": nv.T_BF16}[s["kind"]]
    nv.check(nv.lib().b200dec_logit_rules(p(s["logits"]), kind, s["vocab"], s["rows"], s["vocab"], p(s["active"]),
                                          s["slots"], ctypes.byref(s["rules"]), p(s["out_t"]), s["vocab"], p(s["best"]),
                                          p(s["token"]), p(s["status"]), 0, nv.stream_ptr()))
    return (s["token"], s["best"], s["out_t"]) if s["out"] else (s["token"], s["best"])


def _rules(s):
    rows, vocab, slot = s["rows"], s["vocab"], s["active"].long()
    x = s["logits"].float()
    r, presence, frequency = (s["params"][slot, i, None] for i in range(3))
    tokens = s["history_t"][slot]
    at = torch.arange(tokens.shape[1], device=x.device)
    here = at <= s["last"][slot, None]
    seen = torch.zeros_like(x).scatter_add_(1, tokens, here.float()) > 0
    times = torch.zeros_like(x).scatter_add_(1, tokens, (here & (at >= s["plen"][slot, None])).float())
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - frequency * times - presence * (times > 0)
    if s["biases"]:
        listed_ = torch.arange(s["biases"], device=x.device) < s["count"][slot, None]
        bias = torch.where(listed_, s["values"][slot], 0.0)
        x = x + torch.zeros_like(x).scatter_add_(1, s["ids"][slot].long(), bias)
    if s["mask"]:
        bits = s["mask_t"][slot][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32) & 1
        x = x.masked_fill(bits.flatten(1)[:, :vocab] == 0, -math.inf)
    best = x.amax(1)
    index = torch.arange(vocab, device=x.device, dtype=torch.int32)
    token = torch.where(x == best[:, None], index, vocab).amin(1).to(torch.int32)
    return (token, best, x.to(TYPES[s["kind"]])) if s["out"] else (token, best)


def _own_product(s):
    return s["linear"](s["x_t"], out=s["out_t"])


def _product(s):
    x = s["x_t"].float()
    scale = (x.abs().amax(1, keepdim=True).clamp(min=1e-12).double() / 127).float()
    q = (x.double() / scale.double()).round().clamp(-127, 127)
    y = (q @ s["q"].double().T).float() * (scale * s["scale"])
    if s["bias"]:
        y = y + s["bias_t"]
    return y.to(TYPES[s["out"]])


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------


def exact(c, seed):
    s = prepare(c, seed)
    return {ATTEND: _exact_attend, FILL: _exact_fill, RULES: _exact_rules, PRODUCT: _exact_product}[c["op"]](s)


def _exact_unpack(codes, meta):
    v = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    v[..., 0::2], v[..., 1::2] = codes % 16, codes // 16
    for g in range(meta.shape[-2]):
        v[..., 64 * g:64 * g + 64] *= meta[..., g, :1].double()
        v[..., 64 * g:64 * g + 64] += meta[..., g, 1:].double()
    return v


def _exact_stored(x):
    """The values a 4-bit cache holds of x (..., D) fp32."""
    x = x.to(torch.bfloat16).double().clamp(-LIMIT, LIMIT)
    out = torch.empty_like(x)
    for g in range(0, x.shape[-1], 64):
        part = x[..., g:g + 64]
        low = part.min(-1, keepdim=True).values.half().double()
        step = ((part.max(-1, keepdim=True).values - low) / 15).half().double()
        code = torch.round((part - low) / torch.where(step == 0, 1.0, step)) * (step != 0)
        out[..., g:g + 64] = low + step * code.clamp(0, 15)
    return out


def _exact_attend(s):
    rows, heads, dim = s["rows"], s["heads"], s["dim"]
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda")
    for r in range(rows):
        slot, n = int(s["active"][r]), int(s["at"][r])
        k, v = (_exact_unpack(s[a][slot, :, :n], s[b][slot, :, :n]) for a, b in (("k", "km"), ("v", "vm")))
        q = s["q"][r].view(-1, heads, dim).double()
        if s["self"]:
            k, v = (torch.cat((t, s["q"][r].view(3, heads, 1, dim)[i].bfloat16().double()), 1) for i, t in ((1, k), (2, v)))
        elif n == 0:
            continue
        score = torch.einsum("hd,hnd->hn", q[0], k) / math.sqrt(dim)
        out[r] = torch.einsum("hn,hnd->hd", torch.softmax(score, -1), v)
    if not s["self"]:
        return out.flatten(1)
    return out.flatten(1), _exact_stored(s["q"].view(rows, 3, heads, dim)[:, 1:]).flatten(1)


def _exact_fill(s):
    return _exact_stored(s["kv"].view(s["rows"], -1, s["dim"])).flatten(1)


def _exact_rules(s):
    rows, vocab = s["rows"], s["vocab"]
    outs, tokens, bests = [], [], []
    for r in range(rows):
        slot = int(s["active"][r])
        x = s["logits"][r].double()
        rep, presence, frequency = (float(v) for v in s["params"][slot, :3].double())
        last, plen = int(s["last"][slot]), int(s["plen"][slot])
        so_far = s["history_t"][slot, :last + 1]
        made = torch.bincount(so_far[plen:], minlength=vocab) if plen <= last else torch.zeros(vocab, device="cuda")
        known = torch.unique(so_far)
        x[known] = torch.where(x[known] > 0, x[known] / rep, x[known] * rep)
        x = x - frequency * made.double() - presence * (made > 0).double()
        if s["biases"]:
            k = int(s["count"][slot])
            x = x + torch.zeros_like(x).index_add_(0, s["ids"][slot, :k].long(), s["values"][slot, :k].double())
        if s["mask"]:
            word = torch.arange(vocab, device="cuda") // 32
            bit = 2 ** (torch.arange(vocab, device="cuda") % 32)
            x[(s["mask_t"][slot].long()[word] & bit) == 0] = -math.inf
        outs.append(x), bests.append(x.max())
        tokens.append((x == x.max()).nonzero()[0, 0])
    token, best = torch.stack(tokens).to(torch.int32), torch.stack(bests)
    return (token, best, torch.stack(outs)) if s["out"] else (token, best)


def _exact_product(s):
    x = s["x_t"].double()
    scale = (x.abs().max(1, keepdim=True).values.clamp(min=1e-12) / 127).float().double()
    q = torch.round(x / scale).clamp(-127, 127)
    y = (q @ s["q"].double().T) * scale * s["scale"].double()
    return y + s["bias_t"].double() if s["bias"] else y
