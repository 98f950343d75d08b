"""What the 4-bit cache calls, the rules on the logits and the 8-bit product refuse, and their host-side queries: checks that
need no GPU (every refusal comes before the first CUDA call)."""

import ctypes as C

import pytest

A = 1 << 20  # an address that is never followed: aligned to everything the calls ask for


@pytest.fixture(scope="module")
def nv():
    from cohere_inference_b200 import build, native
    build.build()
    native.lib()
    return native


def refused(nv, rc, text):
    assert rc == 1 and text in nv.lib().b200dec_last_error().decode(), (rc, nv.lib().b200dec_last_error())


ATTEND = dict(self=1, active=A, q=A, ldq=3 * 1024, k=A, v=A, km=A, vm=A, n=A, sched=None, slots=4, heads=8, dim=128, cap=465,
              scale=0.1, out=A, kind=0, rows=2, part=A, count=A, status=A, pdl=0, stream=None)


@pytest.mark.parametrize("change, text", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(vm=None), "null"), (dict(out=None), "null"), (dict(active=None), "null"),
    (dict(n=None), "null"), (dict(status=None), "null"), (dict(part=None), "go together"), (dict(count=None), "go together"),
    (dict(dim=96), "head_dim"), (dict(rows=0), "rows"), (dict(rows=65536), "rows"), (dict(heads=0), "heads"), (dict(cap=0), "cap"),
    (dict(cap=(1 << 30) + 1), "cap"), (dict(slots=-1), "slots"), (dict(ldq=3 * 1024 - 4), "ldq"), (dict(ldq=3 * 1024 + 2), "ldq"),
    (dict(self=0, ldq=1020), "ldq"), (dict(q=A + 4), "ldq"), (dict(k=A + 8), "alignment"), (dict(km=A + 2), "alignment"),
    (dict(sched=A + 4), "alignment"), (dict(kind=2), "out_kind"),
    (dict(rows=65535, heads=8192, ldq=3 * 8192 * 128), "rows x"), (dict(dim=128, km=A + 4), "alignment"),
])
def test_attention_q4(nv, change, text):
    refused(nv, nv.lib().b200dec_attention_q4(*{**ATTEND, **change}.values()), text)


def test_attention_q4_workspace(nv):
    f = nv.lib().b200dec_attention_q4_scratch_floats
    assert f(0, 8, 128, 465) == f(1, 0, 128, 465) == f(1, 8, 128, 0) == 0
    assert f(128, 16, 64, 465) >= 128 * 16 * 66 and f(1, 8, 128, 1 << 30) <= 8 * 128 * 130
    for rows, heads, cap in ((1, 8, 1), (1, 8, 131072), (24, 8, 33000), (300, 1, 70)):  # whole chunks of 66 or 130 floats
        assert f(rows, heads, 64, cap) % (rows * heads * 66) == 0 and f(rows, heads, 128, cap) % (rows * heads * 130) == 0


KV = dict(kv=A, slot_of=A, frame_of=A, ck=A, cv=A, ckm=A, cvm=A, nrows=3, layers=8, slots=5, heads=16, dim=64, frames=375, stream=None)


@pytest.mark.parametrize("name", ["b200dec_scatter_kv_q4", "b200dec_gather_kv_q4"])
@pytest.mark.parametrize("change, text", [
    (dict(kv=None), "null"), (dict(slot_of=None), "null"), (dict(frame_of=None), "null"), (dict(cvm=None), "null"),
    (dict(nrows=-1), "nrows"), (dict(dim=32), "head_dim"), (dict(layers=0), "layers"), (dict(frames=0), "frames"),
    (dict(heads=0), "heads"), (dict(slots=0), "slots"), (dict(layers=1 << 20), "layers"), (dict(kv=A + 16), "alignment"),
    (dict(ck=A + 2), "alignment"), (dict(ckm=A + 2), "alignment"),
])
def test_kv_q4(nv, name, change, text):
    refused(nv, getattr(nv.lib(), name)(*{**KV, **change}.values()), text)
    assert getattr(nv.lib(), name)(*{**KV, "nrows": 0}.values()) == 0  # nothing to do is no error


RULES = dict(logits=A, kind=0, ldl=100, rows=2, vocab=100, active=A, slots=4, rules=None, out=None, ldo=0, best=A, token=A, status=A,
             pdl=0, stream=None)
TABLES = dict(params=A, history=A, last=A, plen=A, bias_ids=A, bias=A, bias_n=A, mask=None, mask_on=None, hist_cols=10, max_bias=4)


@pytest.mark.parametrize("change, tables, text", [
    (dict(logits=None), {}, "null"), (dict(token=None), {}, "null"), (dict(status=None), {}, "null"), (dict(active=None), {}, "null"),
    (dict(kind=3), {}, "kind"), (dict(rows=0), {}, "rows"), (dict(vocab=0, ldl=0), {}, "vocab"), (dict(vocab=101), {}, "vocab"),
    (dict(vocab=(1 << 24) + 1, ldl=1 << 25), {}, "vocab"), (dict(out=A, ldo=99), {}, "vocab"), (dict(slots=-1), {}, "slots"),
    (dict(logits=A + 2), {}, "alignment"), ({}, dict(params=None), "penalties"), ({}, dict(params=A + 8), "penalties"),
    ({}, dict(history=None), "penalties"), ({}, dict(last=None), "penalties"), ({}, dict(plen=None), "penalties"),
    ({}, dict(hist_cols=0), "penalties"), ({}, dict(bias=None), "bias list"), ({}, dict(bias_n=None), "bias list"),
    ({}, dict(bias_ids=None), "bias list"), ({}, dict(max_bias=0), "max_bias"), ({}, dict(max_bias=1025), "max_bias"),
])
def test_logit_rules(nv, change, tables, text):
    r = nv.Rules(*{**TABLES, **tables}.values())
    refused(nv, nv.lib().b200dec_logit_rules(*{**RULES, "rules": C.byref(r), **change}.values()), text)


def test_logit_rules_without_tables(nv):
    refused(nv, nv.lib().b200dec_logit_rules(*RULES.values()), "null")


@pytest.mark.parametrize("args, text", [
    ((None, 0, 4, 64, 64, A, A, None), "null"), ((A, 0, 4, 64, 64, None, A, None), "null"), ((A, 0, 4, 64, 64, A, None, None), "null"),
    ((A, 0, 0, 64, 64, A, A, None), "m 0"), ((A, 0, 4, 0, 64, A, A, None), "k 0"), ((A, 0, 4, 64, 63, A, A, None), "ldx"),
    ((A, 0, 4, 131073, 131073, A, A, None), "k 131073"), ((A, 7, 4, 64, 64, A, A, None), "kind"),
    ((A, 0, 4, 64, 64, A + 512, A, None), "alignment"), ((A + 2, 0, 4, 64, 64, A, A, None), "alignment"),
    ((A + 1, 1, 4, 64, 64, A, A, None), "alignment"),
])
def test_w8a8_pack_rows(nv, args, text):
    refused(nv, nv.lib().b200dec_w8a8_pack_rows(*args), text)


LINEAR = dict(rows_image=A, row_scale=A, m=4, k=64, weight=A, w_scale=A, bias=None, n=10, act=0, out=A, kind=0, ldo=10, status=A,
              stream=None)


@pytest.mark.parametrize("change, text", [
    (dict(rows_image=None), "null"), (dict(row_scale=None), "null"), (dict(weight=None), "null"), (dict(w_scale=None), "null"),
    (dict(out=None), "null"), (dict(status=None), "null"), (dict(m=0), "m 0"), (dict(n=0), "n 0"), (dict(k=0), "k 0"),
    (dict(k=131073), "k 131073"), (dict(ldo=9), "ldo"), (dict(m=(1 << 30) + 1), "m "), (dict(n=(1 << 30) + 1, ldo=1 << 31), "n "), (dict(kind=3), "out_kind"), (dict(act=3), "act"),
    (dict(rows_image=A + 512), "alignment"), (dict(weight=A + 16), "alignment"), (dict(w_scale=A + 4), "alignment"),
    (dict(bias=A + 8), "alignment"), (dict(out=A + 2), "alignment"),
])
def test_w8a8_linear(nv, change, text):
    refused(nv, nv.lib().b200dec_w8a8_linear(*{**LINEAR, **change}.values()), text)


PREFILL = dict(rows_image=A, row_scale=A, m=4, k=64, weight=A, w_scale=A, bias=None, n=16384, mode=1, pieces=A, n_pieces=1, ck=A,
               cv=A, cks=A, cvs=A, layers=8, slots=5, heads=16, dim=64, frames=375, status=A, stream=None)


@pytest.mark.parametrize("change, text", [
    (dict(rows_image=None), "null"), (dict(status=None), "null"), (dict(m=0), "m 0"), (dict(mode=0), "mode 0"), (dict(mode=4), "mode 4"),
    (dict(pieces=None), "pieces"), (dict(n_pieces=0), "pieces"), (dict(ck=None), "pieces"), (dict(mode=3, cks=None), "pieces"),
    (dict(mode=2, cvs=None), "pieces"), (dict(ck=A + 8), "alignment"), (dict(weight=A + 512), "alignment"), (dict(dim=32), "head_dim"),
    (dict(n=16128), "n 16128"), (dict(layers=1, heads=1, dim=64, n=128), "256"), (dict(frames=0), "n 16384"),
])
def test_w8a8_prefill(nv, change, text):
    refused(nv, nv.lib().b200dec_w8a8_prefill(*{**PREFILL, **change}.values()), text)


def test_w8a8_sizes(nv):
    lib = nv.lib()
    assert lib.b200dec_w8a8_rows_bytes(1, 1) == 128 * 128 and lib.b200dec_w8a8_rows_bytes(129, 1300) == 256 * 1408
    assert lib.b200dec_w8a8_weight_bytes(1, 129) == 256 * 256 and lib.b200dec_w8a8_rows_bytes(0, 64) == 0
    assert lib.b200dec_w8a8_rows_bytes(1, 0) == lib.b200dec_w8a8_rows_bytes(-1, 64) == lib.b200dec_w8a8_weight_bytes(0, 64) == -1
    assert lib.b200dec_w8a8_rows_bytes(1, 131073) == lib.b200dec_w8a8_weight_bytes(1, 131073) == -1
    refused(nv, lib.b200dec_w8a8_tile_weight(None, 4, 4, A, None), "1 KB")
    refused(nv, lib.b200dec_w8a8_tile_weight(A, 4, 4, A + 512, None), "1 KB")


@pytest.mark.parametrize("change", [dict(out=A + 1), dict(out=A + 2, kind=1), dict(out=A + 3, kind=1)])
def test_attention_q4_results_off_their_alignment(nv, change):
    refused(nv, nv.lib().b200dec_attention_q4(*{**ATTEND, **change}.values()), "alignment of out")


@pytest.mark.parametrize("change", [dict(mode=2, cks=A + 2), dict(mode=2, cvs=A + 1), dict(mode=3, cks=A + 2), dict(mode=3, cvs=A + 3)])
def test_w8a8_prefill_scales_off_their_alignment(nv, change):
    refused(nv, nv.lib().b200dec_w8a8_prefill(*{**PREFILL, **change}.values()), "alignment")
