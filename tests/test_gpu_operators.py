"""The 4-bit cache calls, the rules on the logits and the 8-bit product against plain implementations in 64 bits, at the sizes,
lengths and masks where they can go wrong. Tolerances count roundings: half a step is 2^-24 of the value in fp32, 2^-11 in
fp16, 2^-8 in bf16."""

import ctypes as C
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LIMIT = 32752.0


@pytest.fixture(scope="module")
def nv():
    from cohere_inference_b200 import native
    native.lib()
    return native


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


# ---- the 4-bit format in 64 bits --------------------------------------------------------------------------------------


def quantise(x):
    """codes uint8 (..., D / 2), pairs fp16 (..., D / 64, 2), values fp64 (..., D)."""
    x = torch.nan_to_num(x.bfloat16().double(), 0.0, LIMIT, -LIMIT).clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 64))
    lo = x.amin(-1, keepdim=True).half()
    step = ((x.amax(-1, keepdim=True) - lo.double()) / 15).half()
    s = step.double()
    code = torch.where(s > 0, ((x - lo.double()) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15), 0.0)
    q = code.to(torch.uint8).flatten(-2)
    return q[..., 0::2] | q[..., 1::2] << 4, torch.cat((step, lo), -1), (lo.double() + code * s).flatten(-2)


def values(codes, pairs):
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double().unflatten(-1, (-1, 64))
    return (q * pairs[..., :1].double() + pairs[..., 1:].double()).flatten(-2)


def awkward_rows(n, width, seed):
    """Gaussian head vectors of 64, and among them constant, zero, tiny, huge, infinite and NaN ones and ones with a far offset."""
    x = torch.randn(n, width // 64, 64, generator=gen(seed), device="cuda")
    kinds = torch.arange(n * width // 64, device="cuda").view(n, -1) % 12
    x = torch.where((kinds == 1)[..., None], 0.0, x)
    x = torch.where((kinds == 2)[..., None], 3.7, x)
    x = torch.where((kinds == 3)[..., None], x * 1e-6, x)
    x = torch.where((kinds == 4)[..., None], x * 1e4, x)
    x = torch.where((kinds == 5)[..., None], x * 1e30, x)
    x = torch.where((kinds == 6)[..., None], x * 0.01 - 900.0, x)
    x[..., 5] = torch.where(kinds == 7, math.inf, x[..., 5])
    x[..., 6] = torch.where(kinds == 8, -math.inf, x[..., 6])
    x[..., 7] = torch.where(kinds == 9, math.nan, x[..., 7])
    x = torch.where((kinds == 10)[..., None], (x * 4).round() / 4, x)  # a coarse grid: quotients on the halves
    return x.view(n, width).contiguous()


@pytest.mark.parametrize("layers, heads, dim, frames, slots, nrows", [
    (1, 1, 64, 1, 1, 1), (8, 16, 64, 375, 5, 700), (8, 8, 128, 375, 5, 333), (2, 3, 128, 7, 3, 21), (1, 5, 64, 40, 2, 80),
])
def test_scatter_and_gather_q4(nv, layers, heads, dim, frames, slots, nrows):
    width = layers * 2 * heads * dim
    kv = awkward_rows(nrows, width, 1)
    at = torch.randperm(slots * frames, generator=torch.Generator().manual_seed(2))[:nrows].to(torch.int32).cuda()
    slot_of, frame_of = (at // frames).contiguous(), (at % frames).contiguous()
    shape = layers, slots + 1, heads, frames
    new = lambda: (torch.full((*shape, dim // 2), 0xA5, dtype=torch.uint8, device="cuda"),  # noqa: E731
                   torch.full((*shape, dim // 64, 2), 7.0, dtype=torch.float16, device="cuda"))
    (k, km), (v, vm) = new(), new()
    want = [t.clone() for t in (k, km, v, vm)]
    codes, pairs, held = quantise(kv.view(nrows, layers, 2, heads, dim))
    s, f = slot_of.long(), frame_of.long()
    for part, (c, m) in enumerate(((want[0], want[1]), (want[2], want[3]))):
        c[:, s, :, f], m[:, s, :, f] = codes[:, :, part], pairs[:, :, part]
    p = nv.ptr
    sizes = (nrows, layers, slots + 1, heads, dim, frames, nv.stream_ptr())
    nv.check(nv.lib().b200dec_scatter_kv_q4(p(kv), p(slot_of), p(frame_of), p(k), p(v), p(km), p(vm), *sizes))
    for got, ref in zip((k, km, v, vm), want):  # everything outside the rows is as it was
        assert torch.equal(got.view(torch.uint8), ref.view(torch.uint8))
    back = torch.empty_like(kv)
    nv.check(nv.lib().b200dec_gather_kv_q4(p(back), p(slot_of), p(frame_of), p(k), p(v), p(km), p(vm), *sizes))
    assert torch.equal(back, held.flatten(1).float())  # lo + code * step, rounded once


def test_scatter_and_gather_q4_outside(nv):
    """Rows outside the caches are dropped by the one and zeros to the other; no memory next to the caches is touched."""
    layers, heads, dim, frames, slots = 2, 16, 64, 9, 3
    kv = torch.randn(6, layers * 2 * heads * dim, generator=gen(3), device="cuda")
    slot_of = torch.tensor([0, -1, 4, 1, 2, 3], dtype=torch.int32, device="cuda")
    frame_of = torch.tensor([8, 0, 0, 9, -1, 0], dtype=torch.int32, device="cuda")
    shape = layers, slots + 1, heads, frames
    k, v = (torch.zeros(*shape, dim // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    km, vm = (torch.zeros(*shape, 1, 2, dtype=torch.float16, device="cuda") for _ in range(2))
    p, sizes = nv.ptr, (6, layers, slots + 1, heads, dim, frames, nv.stream_ptr())
    nv.check(nv.lib().b200dec_scatter_kv_q4(p(kv), p(slot_of), p(frame_of), p(k), p(v), p(km), p(vm), *sizes))
    touched = (km != 0).flatten(4).any(-1).any(0).any(1)  # (slots + 1, frames)
    assert touched.nonzero().tolist() == [[0, 8], [3, 0]]
    back = torch.full_like(kv, 5.0)
    nv.check(nv.lib().b200dec_gather_kv_q4(p(back), p(slot_of), p(frame_of), p(k), p(v), p(km), p(vm), *sizes))
    assert (back[1:5] == 0).all() and (back[0] != 0).any() and (back[5] != 0).any()


# ---- attention ----------------------------------------------------------------------------------------------------------


def make_caches(slots, heads, cap, dim, seed, scale=1.0):
    out = []
    for i in range(2):
        x = scale * (torch.randn(slots + 1, heads, cap, dim, generator=gen(seed + i), device="cuda") +
                     torch.randn(1, heads, 1, dim, generator=gen(seed + 10 + i), device="cuda"))
        codes, pairs, _ = quantise(x)
        out += [codes, pairs]
    return out[0], out[2], out[1], out[3]  # k, v, km, vm


def attend(nv, self, active, q, caches, n, slots, heads, dim, cap, out, sched=None, work=None, pdl=0, scale=None, ldq=None):
    k, v, km, vm = caches
    rows = active.numel()
    lib, p = nv.lib(), nv.ptr
    if work is None:
        work = (torch.empty(lib.b200dec_attention_q4_scratch_floats(rows, heads, dim, cap), device="cuda"),
                torch.zeros(rows * heads, dtype=torch.int32, device="cuda"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    nv.check(lib.b200dec_attention_q4(int(self), p(active), q.data_ptr(), ldq or q.shape[1], p(k), p(v), p(km), p(vm), p(n), p(sched),
                                      slots, heads, dim, cap, dim ** -0.5 if scale is None else scale, p(out),
                                      nv.OUT_F16 if out.dtype == torch.float16 else nv.OUT_F32, rows, p(work[0]) if work[0] is not None else None,
                                      p(work[1]) if work[1] is not None else None, p(status), pdl, nv.stream_ptr()))
    return int(status.item())


def reference(self, active, q, caches, n, heads, dim, scale=None):
    """(rows, heads * dim) in fp64, and how far fp32 arithmetic may be from it. A score is a sum over dim of products of
    an operand kept to 2^-22 and exact codes, in two groups, plus lo times a sum: no more than 3 dim roundings of 2^-24 of
    the sum of magnitudes T; e^score is then off by T dim 2^-22 in proportion, the weights are kept to 2^-21 (their two
    halves, the exponential's 2^-22), and the sums over n keys and the merges round a few times more per 32 keys."""
    rows = active.numel()
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda")
    far = torch.zeros(rows, heads, 1, dtype=torch.float64, device="cuda")
    scale = dim ** -0.5 if scale is None else scale
    for r in range(rows):
        s, m = int(active[r]), int(n[int(active[r])])
        k, v = values(caches[0][s, :, :m], caches[2][s, :, :m]), values(caches[1][s, :, :m], caches[3][s, :, :m])
        x = q[r].view(-1, heads, dim).double()
        if self:
            k, v = (torch.cat((t, q[r].view(3, heads, 1, dim)[i].bfloat16().double()), 1) for i, t in ((1, k), (2, v)))
        if k.shape[1] == 0:
            continue
        score = torch.einsum("hd,hnd->hn", x[0], k) * scale
        out[r] = torch.einsum("hn,hnd->hd", torch.softmax(score, -1), v)
        size = (x[0].abs()[:, None] * (k.abs() + caches[2][s, :, :1, :, 1].double().abs().amax()
                                       if m else k.abs())).sum(-1).amax(-1) * abs(scale)
        keys = k.shape[1]
        far[r, :, 0] = (2 * size * 2.0 ** -22 * dim + 2.0 ** -20 + (keys / 32 + 40) * 2.0 ** -24) * 3 * v.abs().amax((1, 2))
    return out.flatten(1), far.expand(-1, -1, dim).flatten(1)


def check(out, ref, far):
    allowed = far + (HALF[out.dtype] if out.dtype != torch.float32 else 0.0) * ref.abs() + 2.0 ** -25
    worst = ((out.double() - ref).abs() / allowed).max()
    assert worst <= 1, float(worst)


LENGTHS = (0, 1, 2, 15, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 383)


@pytest.mark.parametrize("out_type", [torch.float16, torch.float32])
@pytest.mark.parametrize("heads, dim", [(16, 64), (8, 128), (3, 64), (5, 128)])
@pytest.mark.parametrize("self", [True, False])
def test_attention_q4_lengths(nv, self, heads, dim, out_type):
    """Every length at the edges of a block, a warp's turn and a chunk, in one call; cross rows without a key give zeros; the new
    key and value are held as the format says, and nothing else of the caches changes."""
    cap, rows = 384, len(LENGTHS)
    slots = rows + 3
    active = torch.randperm(slots, generator=torch.Generator().manual_seed(heads))[:rows].to(torch.int32).cuda()
    n = torch.full((slots + 1,), 5, dtype=torch.int32, device="cuda")
    n[active.long()] = torch.tensor(LENGTHS, dtype=torch.int32, device="cuda")
    caches = make_caches(slots, heads, cap, dim, 7)
    q = torch.randn(rows, (3 if self else 1) * heads * dim, generator=gen(8), device="cuda")
    want = [t.clone() for t in caches]
    ref, far = reference(self, active, q, caches, n, heads, dim)
    if self:
        codes, pairs, _ = quantise(q.view(rows, 3, heads, dim)[:, 1:])
        for r in range(rows):
            s, at = int(active[r]), LENGTHS[r]
            want[0][s, :, at], want[1][s, :, at] = codes[r, 0], codes[r, 1]
            want[2][s, :, at], want[3][s, :, at] = pairs[r, 0], pairs[r, 1]
    out = torch.full((rows, heads * dim), 9.0, dtype=out_type, device="cuda")
    assert attend(nv, self, active, q, caches, n, slots, heads, dim, cap, out) == 0
    check(out, ref, far)
    if not self:
        assert (out[0] == 0).all()
    for got, t in zip(caches, want):
        assert torch.equal(got, t)


@pytest.mark.parametrize("rows, heads, dim, cap, longest", [
    (1, 1, 64, 1, 1), (1, 8, 128, 465, 217), (1, 16, 64, 5000, 4999), (2, 3, 128, 20000, 19876), (128, 16, 64, 451, 375),
    (200, 2, 64, 70, 66), (37, 8, 128, 2049, 2049), (1, 1, 128, 140001, 140001),
])
def test_attention_q4_shapes(nv, rows, heads, dim, cap, longest):
    """One row to many, chunks and none, long rows, with and without the workspace, and rows by a schedule: the same values."""
    slots = rows + 1
    active = torch.randperm(slots, generator=torch.Generator().manual_seed(rows))[:rows].to(torch.int32).cuda()
    lens = torch.linspace(longest, 1 if rows > 1 else longest, rows).round().int()
    n = torch.ones(slots + 1, dtype=torch.int32, device="cuda")
    n[active.long()] = lens.cuda()
    caches = make_caches(slots, heads, cap, dim, 9)
    q = 2 * torch.randn(rows, heads * dim, generator=gen(10), device="cuda")
    ref, far = reference(False, active, q, caches, n, heads, dim)
    out = torch.empty(rows, heads * dim, device="cuda")
    assert attend(nv, False, active, q, caches, n, slots, heads, dim, cap, out) == 0
    check(out, ref, far)
    again = torch.empty_like(out)
    assert attend(nv, False, active, q, caches, n, slots, heads, dim, cap, again, work=(None, None)) == 0
    check(again, ref, far)
    if rows <= 256:
        sched = torch.empty(rows, 4, dtype=torch.int32, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        p = nv.ptr
        nv.check(nv.lib().b200dec_row_schedule(p(active), None, p(n), slots, 1, cap, rows, 0, None, p(sched), p(status), nv.stream_ptr()))
        ranked = torch.empty_like(out)
        assert attend(nv, False, active, q, caches, n, slots, heads, dim, cap, ranked, sched=sched) == 0
        check(ranked, ref, far)


@pytest.mark.parametrize("scale", [1e-12, 1e-3, 30.0, 3e5])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_q4_magnitudes(nv, scale, dim):
    """Queries and cache values far from one: both products work on operands scaled into fp16's range. Scores stay moderate:
    the softmax scale undoes the query's."""
    heads, cap, rows = 4, 300, 3
    active = torch.arange(rows, dtype=torch.int32, device="cuda")
    n = torch.full((rows + 1,), 290, dtype=torch.int32, device="cuda")
    caches = make_caches(rows, heads, cap, dim, 11)
    q = scale * torch.randn(rows, heads * dim, generator=gen(12), device="cuda")
    softmax = dim ** -0.5 / scale
    ref, far = reference(False, active, q, caches, n, heads, dim, softmax)
    out = torch.empty(rows, heads * dim, device="cuda")
    assert attend(nv, False, active, q, caches, n, rows, heads, dim, cap, out, scale=softmax) == 0
    check(out, ref, far)
    # values of unlike sizes from key to key: 2^-14 to 2^12 times, growing and falling
    size = 2.0 ** (torch.arange(cap, device="cuda") % 27 - 14)
    x = torch.randn(rows + 1, heads, cap, dim, generator=gen(13), device="cuda") * size[:, None]
    codes, pairs, _ = quantise(x)
    mixed = caches[0], codes, caches[2], pairs
    ref, far = reference(False, active, q, mixed, n, heads, dim, softmax)
    assert attend(nv, False, active, q, mixed, n, rows, heads, dim, cap, out, scale=softmax) == 0
    check(out, ref, far)


def test_attention_q4_peaked_and_tiny_weights(nv):
    """One key far above the rest, then 30000 keys whose weights are 2^-30 of the largest: their share is kept. A weight times
    its step is held to 2^-32 of a warp's largest step, so a key's 15 steps (1 here) are off by 2^-32 at most, and only for
    the 64 keys of the warp that meets the high one (chunks of 256 keys, four warps): the others' largest weight is their own."""
    heads, dim, cap = 1, 64, 30001
    q = torch.zeros(1, dim, device="cuda")
    q[0, 0] = 8.0
    k = torch.zeros(2, 1, cap, dim, device="cuda")
    k[0, 0, 100, 0] = 30 * math.log(2)  # score 8 * that / 8 = 30 ln 2
    v = torch.zeros(2, 1, cap, dim, device="cuda")
    v[0, 0, :, 1::2] = 1.0
    v[0, 0, 100] = 0.0
    v[0, 0, 100, 0] = 1.0  # keeps its pair from being empty
    (kc, kp, _), (vc, vp, _) = quantise(k), quantise(v)
    active, n = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((2,), cap, dtype=torch.int32, device="cuda")
    out = torch.empty(1, dim, device="cuda")
    caches = kc, vc, kp, vp
    ref, _ = reference(False, active, q, caches, n, heads, dim, 1 / 8)
    assert attend(nv, False, active, q, caches, n, 1, heads, dim, cap, out, scale=1 / 8) == 0
    assert float(ref[0, 1]) > 2e-5  # 30000 * 2^-30: each below fp16's least step, their sum not
    assert torch.allclose(out.double(), ref, rtol=2e-4, atol=64 * 2.0 ** -32)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("self", [True, False])
def test_attention_q4_awkward_vectors(nv, self, dim):
    """Constant, zero, tiny and far-off vectors among the cached ones and as the new key and value: pairs with step 0, groups of a
    key with unlike steps, and nothing but constants in a whole row."""
    heads, cap, rows = 2, 150, 3
    x = awkward_rows(2 * (rows + 1) * cap, heads * dim, 21).view(2, rows + 1, cap, heads, dim).transpose(2, 3)
    x = torch.nan_to_num(x, 0.0, 2.0, -2.0).clamp(-1000, 1000)
    x[:, 1] = x[:, 1, :, :1, :1]  # slot 1: every vector of a head the same constant
    (k, km, _), (v, vm, _) = quantise(x[0]), quantise(x[1])
    active = torch.tensor([2, 1, 0], dtype=torch.int32, device="cuda")
    n = torch.tensor([149, 140, 37, 1], dtype=torch.int32, device="cuda")
    q = 0.01 * torch.randn(rows, (3 if self else 1) * heads * dim, generator=gen(22), device="cuda")
    if self:
        q[0, heads * dim:] = 0.25  # a constant key and value
    caches = k, v, km, vm
    ref, far = reference(self, active, q, caches, n, heads, dim)
    out = torch.empty(rows, heads * dim, device="cuda")
    assert attend(nv, self, active, q, caches, n, rows, heads, dim, cap, out) == 0
    check(out, ref, far)


def test_far_offsets_in_4_bit_caches(nv):
    """A cache whose last slots lie beyond 2^32 bytes: filled, appended to, attended and read back there."""
    slots, heads, cap, dim, n = 41, 16, 220000, 64, 333
    shape = 1, slots + 1, heads, cap
    k, v = (torch.zeros(*shape, dim // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    km, vm = (torch.zeros(*shape, 1, 2, dtype=torch.float16, device="cuda") for _ in range(2))
    assert slots * heads * cap * dim // 2 > 2 ** 32
    kv = torch.randn(n, 2 * heads * dim, generator=gen(30), device="cuda")
    slot_of = torch.full((n,), slots - 1, dtype=torch.int32, device="cuda")
    frame_of = torch.arange(n, dtype=torch.int32, device="cuda")
    p, sizes = nv.ptr, (1, slots + 1, heads, dim, cap, nv.stream_ptr())
    nv.check(nv.lib().b200dec_scatter_kv_q4(p(kv), p(slot_of), p(frame_of), p(k), p(v), p(km), p(vm), n, *sizes))
    active = slot_of[:1].contiguous()
    lens = torch.zeros(slots + 1, dtype=torch.int32, device="cuda")
    lens[slots - 1] = n
    q = torch.randn(1, 3 * heads * dim, generator=gen(31), device="cuda")
    caches = k[0], v[0], km[0], vm[0]
    ref, far = reference(True, active, q, caches, lens, heads, dim)
    out = torch.empty(1, heads * dim, device="cuda")
    assert attend(nv, True, active, q, caches, lens, slots, heads, dim, cap, out) == 0
    check(out, ref, far)
    rows = torch.cat((kv, q[:, heads * dim:]))
    slot_of, frame_of = torch.full((n + 1,), slots - 1, dtype=torch.int32, device="cuda"), torch.arange(n + 1, dtype=torch.int32, device="cuda")
    back = torch.empty_like(rows)
    nv.check(nv.lib().b200dec_gather_kv_q4(p(back), p(slot_of), p(frame_of), p(k), p(v), p(km), p(vm), n + 1, *sizes))
    assert torch.equal(back, quantise(rows.view(n + 1, -1, dim))[2].flatten(1).float())


def test_attention_q4_out_of_range(nv):
    """Lengths and slots outside the tables are clamped and reported; the neighbours are right all the same."""
    heads, dim, cap, slots = 2, 64, 40, 3
    caches = make_caches(slots, heads, cap, dim, 15)
    for self, bad_n, bit in ((True, 40, nv.ST_POS_RANGE), (True, -1, nv.ST_POS_RANGE), (False, 41, nv.ST_FRAMES_RANGE),
                             (False, -3, nv.ST_FRAMES_RANGE)):
        q = torch.randn(3, 3 * heads * dim if self else heads * dim, generator=gen(16), device="cuda")
        active = torch.tensor([1, 0, 2], dtype=torch.int32, device="cuda")
        n = torch.tensor([bad_n, 7, 30, 1], dtype=torch.int32, device="cuda")
        mine = [t.clone() for t in caches]
        ref, far = reference(self, active[[0, 2]], q[[0, 2]], mine, n, heads, dim)
        out = torch.empty(3, heads * dim, device="cuda")
        assert attend(nv, self, active, q, mine, n, slots, heads, dim, cap, out) == bit
        check(out[[0, 2]], ref, far)
    for bad in (-1, 4):
        q = torch.randn(2, heads * dim, generator=gen(17), device="cuda")
        active = torch.tensor([bad, 2], dtype=torch.int32, device="cuda")
        n = torch.tensor([7, 7, 30, 1], dtype=torch.int32, device="cuda")
        out = torch.empty(2, heads * dim, device="cuda")
        assert attend(nv, False, active, q, caches, n, slots, heads, dim, cap, out) == nv.ST_SLOT_RANGE
        ref, far = reference(False, torch.tensor([3, 2], device="cuda"), q, caches, n, heads, dim)  # the dummy stands in
        check(out, ref, far)


def test_attention_q4_rows_apart_replay_and_stream(nv):
    """Query rows with a distance of their own, on a stream of its own, captured and replayed: every replay the same bits, the
    counters zero again, and the workspace's leftovers change nothing."""
    heads, dim, cap, rows = 8, 128, 3000, 2
    active = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    n = torch.tensor([2999, 1200, 1], dtype=torch.int32, device="cuda")
    caches = make_caches(rows, heads, cap, dim, 18)
    wide = torch.randn(rows, heads * dim + 12, generator=gen(19), device="cuda")
    q = wide[:, 4:4 + heads * dim]
    ref, far = reference(False, active, q.contiguous(), caches, n, heads, dim)
    lib = nv.lib()
    work = (torch.full((lib.b200dec_attention_q4_scratch_floats(rows, heads, dim, cap),), math.nan, device="cuda"),
            torch.zeros(rows * heads, dtype=torch.int32, device="cuda"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty(rows, heads * dim, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    p = nv.ptr

    def call():
        nv.check(lib.b200dec_attention_q4(0, p(active), q.data_ptr(), wide.shape[1], *(p(t) for t in caches), p(n), None, rows, heads,
                                          dim, cap, dim ** -0.5, p(out), nv.OUT_F32, rows, p(work[0]), p(work[1]), p(status), 0,
                                          nv.stream_ptr()))
    with torch.cuda.stream(side):
        call()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
        seen = []
        for _ in range(5):
            out.fill_(7.0)
            graph.replay()
            side.synchronize()
            seen.append(out.clone())
    check(seen[0], ref, far)
    assert all(torch.equal(seen[0], t) for t in seen) and int(work[1].abs().sum()) == 0 and int(status) == 0


# ---- rules on the logits --------------------------------------------------------------------------------------------------


def tables(slots, vocab, cols, max_bias, seed, exact=True):
    """Rules whose fp32 arithmetic is exact: penalties of powers of two, biases on a grid."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    t = dict(history=(vocab * rnd(slots + 1, cols) ** 3).long().clamp(max=vocab - 1),
             last=(cols * (1.2 * rnd(slots + 1) - 0.1)).int().clamp(-1, cols - 1), plen=(cols * rnd(slots + 1) * 0.6).int())
    t["params"] = torch.stack((2.0 ** (rnd(slots + 1) * 3 - 1).round(), (rnd(slots + 1) * 8).round() / 4,
                               (rnd(slots + 1) * 8).round() / 8, rnd(slots + 1)), 1)
    t["params"][rnd(slots + 1) < 0.3, :3] = torch.tensor([1.0, 0.0, 0.0])
    width = max(1, max_bias)
    t["bias_ids"] = (vocab * rnd(slots + 1, width)).int().clamp(max=vocab - 1)
    t["bias"] = (torch.randn(slots + 1, width, generator=g) * 16).round() / 4
    t["bias"][rnd(slots + 1, width) < 0.2] = -math.inf
    t["bias_n"] = (rnd(slots + 1) * (max_bias + 0.99)).int()
    if max_bias > 3:
        t["bias_ids"][:, 1] = t["bias_ids"][:, 0]  # one token listed twice, a third time further on
        t["bias_ids"][:, 3] = t["bias_ids"][:, 0]
    words = (vocab + 31) // 32
    t["mask"] = torch.randint(-2**31, 2**31, (slots + 1, words), generator=g).to(torch.int32)
    t["mask_on"] = (rnd(slots + 1) < 0.7).to(torch.uint8)
    return {k: v.cuda().contiguous() for k, v in t.items()}


def rules_of(nv, t, biases=True, mask=True, mask_on=True):
    p = nv.ptr
    lists = (p(t["bias_ids"]), p(t["bias"]), p(t["bias_n"])) if biases else (None, None, None)
    return nv.Rules(p(t["params"]), p(t["history"]), p(t["last"]), p(t["plen"]), *lists, p(t["mask"]) if mask else None,
                    p(t["mask_on"]) if mask_on else None, t["history"].shape[1], t["bias"].shape[1])


def under_rules(logits, slot, t, biases=True, mask=True, mask_on=True):
    """One row in fp64."""
    x, vocab = logits.double().clone(), logits.numel()
    rep, presence, frequency = t["params"][slot, :3].double().tolist()
    have = t["history"][slot, :int(t["last"][slot]) + 1]
    made = have[int(t["plen"][slot]):]
    have, made = (h[(h >= 0) & (h < vocab)] for h in (have, made))
    for v in torch.unique(have).tolist():
        x[v] = x[v] / rep if x[v] > 0 else x[v] * rep
    times = torch.bincount(made, minlength=vocab).double()
    x = x - frequency * times - presence * (times > 0)
    if biases:
        for i in range(int(t["bias_n"][slot])):
            v = int(t["bias_ids"][slot, i])
            if 0 <= v < vocab:
                x[v] += t["bias"][slot, i].double()
    if mask and (not mask_on or t["mask_on"][slot]):
        bits = (t["mask"][slot].long()[:, None] >> torch.arange(32, device="cuda")) & 1
        x[bits.flatten()[:vocab] == 0] = -math.inf
    return x


def run_rules(nv, logits, ldl, active, slots, rules, out=None, ldo=0, best=True, pdl=0, vocab=None):
    rows = active.numel()
    kind = {torch.float32: nv.T_F32, torch.float16: nv.T_F16, torch.bfloat16: nv.T_BF16}[logits.dtype]
    value = torch.full((rows,), 5.0, device="cuda")
    token = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    nv.check(nv.lib().b200dec_logit_rules(logits.data_ptr(), kind, ldl, rows, vocab or logits.shape[1], nv.ptr(active), slots,
                                          C.byref(rules), None if out is None else out.data_ptr(), ldo,
                                          nv.ptr(value) if best else None, nv.ptr(token), nv.ptr(status), pdl, nv.stream_ptr()))
    return token, value, int(status.item())


@pytest.mark.parametrize("biases, mask, mask_on", [(True, True, True), (False, True, False), (True, False, False), (False, False, False)])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows, vocab, cols, max_bias", [
    (1, 1, 1, 1), (3, 31, 5, 4), (5, 33, 40, 9), (2, 2048, 7, 1024), (7, 4097, 300, 60), (2, 16384, 458, 33), (130, 500, 20, 5),
    (3, 140003, 2000, 300),
])
def test_logit_rules(nv, rows, vocab, cols, max_bias, kind, biases, mask, mask_on):
    """Logits on a grid of 1/8, so that nothing rounds and equal logits are common: values bit for bit, the first index of the
    largest."""
    slots = rows + 2
    t = tables(slots, vocab, cols, max_bias, vocab + rows)
    active = torch.randperm(slots, generator=torch.Generator().manual_seed(5))[:rows].to(torch.int32).cuda()
    logits = ((torch.randn(rows, vocab, generator=gen(vocab), device="cuda") * 16).round() / 8).clamp(-12, 12).to(kind)
    kept = logits.clone()
    out = torch.full((rows, vocab), 77.0, dtype=kind, device="cuda")
    token, best, status = run_rules(nv, logits, vocab, active, slots, rules_of(nv, t, biases, mask, mask_on), out, vocab)
    assert torch.equal(logits, kept)
    empty = False
    for r in range(rows):
        x = under_rules(logits[r], int(active[r]), t, biases, mask, mask_on)
        top = x.max()
        first = int((x == top).nonzero()[0])
        empty |= bool(top == -math.inf) and int(active[r]) != slots
        assert int(token[r]) == first and float(best[r]) == float(top), (r, int(token[r]), first)
        assert torch.equal(out[r].double(), x.to(kind).double())
    assert status == (nv.ST_NO_TOKEN if empty else 0)
    plain, _, _ = run_rules(nv, logits, vocab, active, slots, rules_of(nv, t, biases, mask, mask_on), best=False)
    assert torch.equal(plain, token)
    run_rules(nv, logits, vocab, active, slots, rules_of(nv, t, biases, mask, mask_on), logits, vocab)  # in place
    assert torch.equal(logits, out)


@pytest.mark.parametrize("offset, pad", [(0, 0), (1, 0), (0, 3), (3, 5), (4, 8)])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_logit_rules_rows_apart(nv, kind, offset, pad):
    """Rows any distance apart and any alignment, in and out; what is between the rows stays as it was."""
    rows, vocab, slots = 6, 5003, 6
    t = tables(slots, vocab, 50, 8, 3)
    active = torch.tensor([5, 0, 6, 2, 3, 1], dtype=torch.int32, device="cuda")  # the dummy among them
    wide = torch.randn(rows * (vocab + pad) + offset + 16, generator=gen(4), device="cuda").to(kind)
    logits = wide[offset:offset + rows * (vocab + pad)].view(rows, vocab + pad)
    room = torch.full_like(wide, 3.0)
    out = room[offset:offset + rows * (vocab + pad)].view(rows, vocab + pad)
    token, best, _ = run_rules(nv, logits, vocab + pad, active, slots, rules_of(nv, t), out, vocab + pad, vocab=vocab)
    for r in range(rows):
        x = under_rules(logits[r, :vocab], int(active[r]), t)
        # three roundings of the value and of what is added to it, and the one to the type
        size = logits[r, :vocab].double().abs() * 4 + 20
        fine = torch.isfinite(x)
        assert torch.equal(fine, torch.isfinite(out[r, :vocab]))
        assert ((out[r, :vocab].double() - x)[fine].abs() <= (size * 4 * HALF[torch.float32] + x.abs() * HALF[kind])[fine]).all()
        assert float(x[int(token[r])]) >= float(x.max()) - 4 * HALF[torch.float32] * 40
        assert (out[r, vocab:] == 3.0).all()
    assert (room[:offset] == 3.0).all() and (room[offset + rows * (vocab + pad):] == 3.0).all()


def test_logit_rules_corners(nv):
    """Infinities, NaN, ids outside the vocabulary, a long history, counts past the tables, and a graph replayed."""
    rows, vocab, slots, cols = 4, 3000, 4, 9000
    t = tables(slots, vocab, cols, 6, 8)
    t["last"][:] = torch.tensor([cols - 1, cols + 50, -9, 4, 0], device="cuda")
    t["plen"][:] = torch.tensor([0, 10, 3, 9, 1], device="cuda")
    t["history"][0, ::7] = -1
    t["history"][0, 1::7] = vocab
    t["history"][0, 2::7] = 1 << 40
    t["bias_n"][:] = torch.tensor([6, 99, -2, 0, 0], device="cuda")
    t["bias_ids"][0, :] = torch.tensor([-1, vocab, 17, 17, 1 << 30, 5], dtype=torch.int32, device="cuda")
    t["mask_on"][:] = 0
    active = torch.arange(rows, dtype=torch.int32, device="cuda")
    logits = ((torch.randn(rows, vocab, generator=gen(9), device="cuda") * 16).round() / 8)
    logits[2, 40] = math.inf
    logits[2, 41] = math.inf
    logits[3, :] = -math.inf
    logits[3, 50] = math.nan
    rules = rules_of(nv, t)
    t["last"][1], t["bias_n"][1], t["bias_n"][2] = cols + 50, 99, -2
    token, best, status = run_rules(nv, logits, vocab, active, slots, rules)
    t["last"][1], t["bias_n"][1], t["bias_n"][2] = cols - 1, 6, 0
    for r in (0, 1):
        x = under_rules(logits[r], r, t)
        assert int(token[r]) == int((x == x.max()).nonzero()[0]) and float(best[r]) == float(x.max())
    assert int(token[2]) == 40 and float(best[2]) == math.inf
    assert int(token[3]) == 0 and float(best[3]) == -math.inf and status == nv.ST_NO_TOKEN
    bad = torch.tensor([0, 9, -1, 1], dtype=torch.int32, device="cuda")
    token, best, status = run_rules(nv, logits, vocab, bad, slots, rules)
    assert status == nv.ST_SLOT_RANGE | nv.ST_NO_TOKEN  # rows 1 and 2 went by the dummy's rules; row 3 has no number above -inf
    side = torch.cuda.Stream()
    value, pick, st = torch.empty(rows, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    p = nv.ptr
    call = lambda: nv.check(nv.lib().b200dec_logit_rules(p(logits), 0, vocab, rows, vocab, p(active), slots, C.byref(rules), None, 0,  # noqa: E731
                                                         p(value), p(pick), p(st), 0, nv.stream_ptr()))
    with torch.cuda.stream(side):
        call()
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            call()
        logits[0] = -logits[0]  # on this stream: the replay sees it
        graph.replay()
        side.synchronize()
    x = under_rules(logits[0], 0, t)
    assert int(pick[0]) == int((x == x.max()).nonzero()[0])


def test_logit_rules_far_offsets(nv):
    """Rows beyond 2^32 elements, a vocabulary of 2^24 that no CTA marks in one go, and tokens in its last places."""
    rows, vocab, slots = 258, 1 << 24, 258
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    assert (rows - 1) * vocab > 2 ** 32 - 1
    t = tables(slots, vocab, 20, 2, 3)
    t["last"][:], t["plen"][:], t["bias_n"][:] = 19, 0, 0
    t["params"][:] = torch.tensor([1.0, 0.0, 0.5, 0.0], device="cuda")
    last = rows - 1
    t["history"][last] = vocab - 5
    logits[last, vocab - 5] = 9.0   # taken 20 times: 9 - 10
    logits[last, vocab - 3] = 3.0
    logits[last, 7] = 2.0
    logits[0, 1 << 23] = 1.0
    active = torch.arange(rows, dtype=torch.int32, device="cuda")
    token, best, status = run_rules(nv, logits, vocab, active, slots, rules_of(nv, t, mask=False))
    assert int(token[last]) == vocab - 3 and float(best[last]) == 3.0
    assert int(token[0]) == 1 << 23 and float(best[0]) == 1.0 and status == 0


# ---- the 8-bit product ------------------------------------------------------------------------------------------------------


def product(x, q, scale, bias, act):
    """fp64, and the sum of the magnitudes that round."""
    x = x.double()
    s = (x.abs().amax(1, keepdim=True).clamp(min=1e-12) / 127).float().double()
    a = (x / s).round().clamp(-127, 127)
    y = (a @ q.double().T) * (s * scale.double())
    size = y.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    if act == "relu":
        y = y.clamp(min=0)
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    return y, size


@pytest.mark.parametrize("x_type, out_type", [(torch.float32, torch.float32), (torch.float16, torch.bfloat16),
                                              (torch.bfloat16, torch.float16), (torch.float32, torch.float16)])
@pytest.mark.parametrize("m, k, n", [
    (1, 1, 1), (1, 1024, 1024), (3, 16, 63), (64, 1024, 4096), (127, 129, 65), (128, 128, 64), (129, 1000, 130), (300, 333, 257),
    (1000, 512, 2000), (2100, 4096, 1024), (700, 70, 5001), (3000, 130, 2000), (3329, 1000, 1900), (2200, 1500, 2305),
])
def test_w8a8_linear(nv, m, k, n, x_type, out_type):
    from cohere_inference_b200.packing import W8A8Linear
    g = gen(m + k + n)
    x = torch.randn(m, k, generator=g, device="cuda").to(x_type)
    x[m // 2] = 0  # a row of zeros
    q = torch.randint(-127, 128, (n, k), generator=g, device="cuda").to(torch.int8)
    scale = torch.rand(n, generator=g, device="cuda") * 0.01 + 1e-4
    for bias, act in ((None, None), (torch.randn(n, generator=g, device="cuda"), "gelu"), (torch.randn(n, generator=g, device="cuda"), "relu")):
        lin = W8A8Linear(q, scale, bias, act)
        y = lin(x, dtype=out_type)
        ref, size = product(x, q, scale, bias, act)
        # the sum's conversion, the scales' product, their product and the bias: four roundings of the magnitudes; GELU's erf and
        # products a few more of a result no larger than those, whose slope is at most 1.13
        far = (5 if act != "gelu" else 16) * HALF[torch.float32] * size + HALF[out_type] * ref.abs() + (2.0 ** -25 if out_type == torch.float16 else 0)
        worst = ((y.double() - ref).abs() - far).max()
        assert y.dtype == out_type and worst <= 0, float(worst)
        assert int(lin.status) == 0


def test_w8a8_far_offsets(nv):
    """Results beyond 2^32 bytes."""
    from cohere_inference_b200.packing import W8A8Linear
    g = gen(40)
    m, k, n = 70001, 64, 16400
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.float32)
    q = torch.randint(-127, 128, (n, k), generator=g, device="cuda").to(torch.int8)
    scale = torch.rand(n, generator=g, device="cuda") * 0.01
    y = W8A8Linear(q, scale)(x)
    assert (m - 1) * n * 4 > 2 ** 32
    for rows in (slice(0, 3), slice(m // 2, m // 2 + 3), slice(m - 3, m)):
        ref, size = product(x[rows], q, scale, None, None)
        assert ((y[rows].double() - ref).abs() <= 5 * HALF[torch.float32] * size).all()


def test_w8a8_quantises_as_if_exact(nv):
    """Quotients on and beside the halves: the codes are those of the exact quotient, ties to even (a unit matrix shows them)."""
    from cohere_inference_b200.packing import W8A8Linear
    k = 256
    x = torch.empty(200, k, device="cuda")
    top = torch.rand(200, generator=gen(1), device="cuda") * 10 + 0.1
    s = (top.double() / 127).float()
    half = torch.arange(k, device="cuda") % 127 + 0.5
    x[:] = (half * s[:, None].double()).float()  # the nearest fp32 to (i + 1/2) s, and its neighbours
    x[:, 100:] = torch.nextafter(x[:, 100:], torch.tensor(math.inf, device="cuda"))
    x[:, 180:] = -x[:, 180:]
    x = torch.where(x.abs() > top[:, None], top[:, None], x)
    x[:, 0] = top
    x[0] = torch.arange(k, device="cuda") % 128 * 0.5
    x[0, 0] = 127.0  # s = 1: exact ties
    lin = W8A8Linear(torch.eye(k, dtype=torch.int8, device="cuda"), torch.ones(k, device="cuda"))
    s = (x.double().abs().amax(1, keepdim=True) / 127).float()
    assert torch.equal(lin(x), (x.double() / s.double()).round().float() * s)


def test_w8a8_rows_with_infinities_and_rows_apart(nv):
    """An infinity or NaN makes its own row NaN and no other; x and out rows any distance apart; out's surroundings stay."""
    from cohere_inference_b200.packing import W8A8Linear
    g = gen(2)
    m, k, n = 70, 200, 90
    lin = W8A8Linear.from_weight(torch.randn(n, k, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda"))
    wide = torch.randn(m, k + 7, generator=g, device="cuda")
    x = wide[:, 3:3 + k]
    x[4, 9], x[5, 0], x[6, k - 1] = math.nan, math.inf, -math.inf
    room = torch.full((m, n + 9), 3.0, device="cuda")
    out = room[:, 1:1 + n]
    assert lin(x, out=out) is out
    dense = lin(x.contiguous())
    assert torch.equal(out.isnan().any(1).nonzero().flatten().cpu(), torch.tensor([4, 5, 6])) and out[4:7].isnan().all()
    assert torch.equal(out.nan_to_num(-1.0), dense.nan_to_num(-1.0))
    assert (room[:, 0] == 3.0).all() and (room[:, 1 + n:] == 3.0).all()
    assert lin(x[:0]).shape == (0, n)
    assert torch.equal(lin(x[10:11]), dense[10:11])
    assert torch.equal(lin(x.T.contiguous().T).nan_to_num(-1.0), dense.nan_to_num(-1.0))  # columns apart: copied first


def test_w8a8_streams_and_replay(nv):
    """Calls on two streams at once and inside a captured graph give the bits of a call alone."""
    from cohere_inference_b200.packing import W8A8Linear
    g = gen(3)
    lin = W8A8Linear.from_weight(torch.randn(1500, 700, generator=g, device="cuda"), act="relu")
    xs = [torch.randn(900, 700, generator=g, device="cuda") for _ in range(2)]
    alone = [lin(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(lin(xs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, alone[i]) for i in range(2) for y in got[i])
    x = xs[0].clone()
    with torch.cuda.stream(streams[0]):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            y = lin(x)
        for i in (1, 0):
            x.copy_(xs[i])
            graph.replay()
            streams[0].synchronize()
            assert torch.equal(y, alone[i])


def test_w8a8_refusals(nv):
    from cohere_inference_b200.packing import W8A8Linear
    q, s = torch.ones(8, 16, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    lin = W8A8Linear(q, s)
    x = torch.ones(3, 16, device="cuda")
    for bad in (x[:, :15], x.double(), x.cpu(), x[0], x.int()):
        with pytest.raises(ValueError):
            lin(bad)
    for bad in (torch.empty(3, 9, device="cuda"), torch.empty(2, 8, device="cuda"), torch.empty(3, 8, device="cuda", dtype=torch.float64),
                torch.empty(8, 3, device="cuda").T, torch.empty(3, 8)):
        with pytest.raises(ValueError):
            lin(x, out=bad)
    with pytest.raises(ValueError):
        lin(x, out=torch.empty(3, 8, device="cuda"), dtype=torch.float16)
    for args in ((q, s, None, "tanh"), (q.cpu(), s), (q.float(), s), (q[:0], s[:0]), (q, s[:7]), (q, s, torch.ones(7, device="cuda")),
                 (torch.ones(1, 131073, dtype=torch.int8, device="cuda"), s[:1])):
        with pytest.raises(ValueError):
            W8A8Linear(*args)
