"""Drafted decoding over an 8-bit cache without a GPU: what the entry points refuse, and the plain forms against each other."""
import ctypes as C

import pytest
import torch

import kv8_util as K
from conftest import pkg

BUF = 0x10000   # an aligned address that nothing reads: every call here is refused before a launch


def _lib():
    return pkg("_abi").lib()


def _append(**kw):
    a = dict(qkv=BUF, ld=48 * 128, pos=BUF, slots=BUF, cos=BUF, q=BUF, ldq=32 * 128, k=BUF, v=BUF, ke=BUF, ve=BUF, n_blocks=9, T=3, hq=32, hkv=8, block=128)
    a.update(kw)
    return _lib().b200_rope_kv_append_fp8(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    ({"qkv": None}, -1), ({"pos": None}, -1), ({"slots": None}, -1), ({"cos": None}, -1), ({"q": None}, -1), ({"k": None}, -1), ({"ve": None}, -1),
    ({"T": -1}, -1), ({"hq": 0}, -1), ({"hkv": 0}, -1), ({"hq": 33}, -1), ({"ld": 47 * 128}, -1), ({"ld": 48 * 128 + 4}, -1), ({"ldq": 31 * 128}, -1),
    ({"ldq": 32 * 128 + 1}, -1), ({"block": 0}, -3), ({"block": 8}, -3), ({"block": 48}, -3), ({"block": 192}, -3), ({"n_blocks": 0}, -1), ({"n_blocks": -4}, -1),
    ({"n_blocks": 2 ** 21}, -1), ({"n_blocks": 2 ** 62}, -1), ({"qkv": BUF + 8}, -1), ({"q": BUF + 2}, -1), ({"k": BUF + 4}, -1), ({"cos": BUF + 8}, -1)])
def test_append_refuses(kw, code):
    assert _append(**kw) == code
    assert b"rope_kv_append_fp8" in _lib().b200_last_error()


def _attend(prefill, **kw):
    lib = _lib()
    a = dict(q=BUF, ldq=32 * 128, k=BUF, v=BUF, ke=BUF, ve=BUF, n_blocks=9, bt=BUF, stride=4, seq=None, ctx=BUF, out=BUF, ldo=32 * 128, T=3, hq=32, hkv=8, block=128)
    a.update({k: v for k, v in kw.items() if k in a})
    tail = dict(most=5, scale=0.1, ws=BUF, size=1 << 40)
    tail.update({k: v for k, v in kw.items() if k in tail})
    if not prefill:
        tail.pop("most")
    return (lib.b200_paged_attn_prefill_fp8 if prefill else lib.b200_paged_attn_decode_fp8)(*a.values(), *tail.values(), None)


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("kw,code", [
    ({"q": None}, -1), ({"k": None}, -1), ({"v": None}, -1), ({"ke": None}, -1), ({"ve": None}, -1), ({"bt": None}, -1), ({"ctx": None}, -1), ({"out": None}, -1),
    ({"T": -2}, -1), ({"hq": 31}, -1), ({"hkv": 0}, -1), ({"hq": 34, "hkv": 2}, -3), ({"stride": 0}, -1), ({"block": 100}, -3), ({"block": 24}, -3),
    ({"n_blocks": 0}, -1), ({"n_blocks": 1 << 40}, -1), ({"ldq": 32 * 128 - 8}, -1), ({"ldo": 32 * 128 + 2}, -1), ({"q": BUF + 2}, -1), ({"out": BUF + 8}, -1),
    ({"ke": BUF + 1}, -1), ({"v": BUF + 8}, -1), ({"scale": float("inf")}, -1), ({"scale": float("nan")}, -1), ({"ws": None}, -1), ({"size": 0}, -1), ({"ws": BUF + 8}, -1)])
def test_attention_refuses(prefill, kw, code):
    if kw == {"size": 0} or kw == {"ws": None}:
        assert _lib().b200_paged_attn_fp8_workspace_bytes(3, 32, 8) > 0
    assert _attend(prefill, **kw) == code
    assert (b"paged_attn_prefill_fp8" if prefill else b"paged_attn_decode_fp8") in _lib().b200_last_error()


def test_attention_of_no_rows_is_nothing():
    assert _attend(False, T=0, ws=None, size=0) == 0 and _attend(True, T=0, ws=None, size=0) == 0
    assert _attend(True, most=-1) == -1
    assert _lib().b200_paged_attn_fp8_workspace_bytes(0, 32, 8) == 0 and _lib().b200_paged_attn_fp8_workspace_bytes(5, 32, 0) == 0


def _verify(**kw):
    a = dict(target=BUF, ldt=1000, draft=BUF, ldd=1000, tokens=BUF, starts=BUF, temp=BUF, uni=BUF, S=2, n=7, V=1000, out=BUF, kept=BUF, ws=BUF, size=1 << 40)
    a.update(kw)
    return _lib().b200_verify_drafts(*a.values(), None)


@pytest.mark.parametrize("kw", [{"target": None}, {"tokens": None}, {"starts": None}, {"out": None}, {"kept": None}, {"uni": None}, {"S": -1}, {"n": -1}, {"V": 0},
                                {"ldt": 999}, {"ldd": 999}, {"ws": None}, {"size": 8}, {"ws": BUF + 4}])
def test_verify_refuses(kw):
    assert _verify(**kw) == -1
    assert b"verify_drafts" in _lib().b200_last_error()


def test_verify_has_limits():
    assert _verify(V=393217, ldt=2 ** 21, ldd=2 ** 21) == -3 and b"393216" in _lib().b200_last_error()
    assert _verify(n=65536) == -3 and b"65535" in _lib().b200_last_error()


def test_verify_of_no_sequences_is_nothing():
    assert _verify(S=0, n=0, ws=None, size=0) == 0
    assert _lib().b200_verify_drafts_workspace_bytes(0, 1000) == 0


def test_plain_quantisation_is_what_the_format_says():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 128, generator=g) * torch.exp2(torch.randn(500, 1, generator=g) * 8)
    x[0] = 0
    x[1] = 448 * 2.0 ** -3
    x[2, 5] = float("nan")
    codes, exps = K.quantise(x)
    back = K.values(codes, exps)
    fine = torch.arange(500) != 2
    top = codes.view(K.E4M3).double().abs().amax(-1)
    assert ((top >= 224) | (exps == 27))[fine].all() and (top <= 448)[fine].all()   # the smallest exponent that holds the row
    assert int(exps[1]) == 127 - 3 and int(exps[0]) == 27 and int(exps[2]) == 255 and bool((codes[2] == 0x7f).all())
    assert ((back - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + torch.exp2(exps.double() - 127)[:, None] * 2.0 ** -10)[fine].all()
    assert torch.equal(back[fine], back[fine].to(torch.bfloat16).double())


def test_plain_check_keeps_what_the_drafter_had_right():
    V, g = 50, torch.Generator().manual_seed(4)
    target = torch.randn(3, V, generator=g).to(torch.bfloat16)
    out, kept, _ = K.verify(target, target, torch.tensor([7, 9, 0]), [0, 3], torch.ones(1), torch.full((3, 2), 0.999))
    assert out.tolist()[:2] == [7, 9] and kept.tolist() == [2]           # p = q: u q < p for every u below 1
    best = target.double().argmax(1)
    out, kept, _ = K.verify(target, None, torch.tensor([int(best[0]), int(best[1]) + 1, 0]), [0, 3], None, None)
    assert out.tolist() == [int(best[0]), int(best[1]), -1] and kept.tolist() == [1]


def test_abi_integers_are_wide_enough():
    sig = pkg("_abi").SIGNATURES
    assert sig["b200_paged_attn_fp8_workspace_bytes"][0] is C.c_int64 and sig["b200_verify_drafts_workspace_bytes"][0] is C.c_int64


def test_attention_counts_its_tiles_in_32_bits():
    """Rows times kv heads times tiles of the block table stay below 2^31."""
    assert _attend(True, T=70000, stride=1 << 20, hkv=32) == -3 and b"70000 rows" in _lib().b200_last_error()
    assert _attend(False, T=1, stride=2 ** 31 - 1, block=1024, n_blocks=5) == -3
    assert _attend(True, most=2 ** 31 - 1, ws=None) == -1   # (a bound above the rows is none)


def test_plain_check_of_equal_probabilities():
    """The plain form's leftovers where target and drafter agree but for a few entries."""
    V, g = 400, torch.Generator().manual_seed(6)
    target = torch.randn(2, V, generator=g).to(torch.bfloat16)
    draft = target.clone()
    draft[0, 7], draft[0, 9] = target[0, 9], target[0, 7]   # two entries trade places: all others are equally probable
    lower, higher = (7, 9) if target[0, 7] < target[0, 9] else (9, 7)
    out, kept, _ = K.verify(target, draft, torch.tensor([lower, 0]), [0, 2], torch.ones(1), torch.tensor([[0.999, 0.5], [0.5, 0.5]]))
    assert int(kept[0]) == 0 and int(out[0]) == higher


@pytest.mark.parametrize("V", [1, 300, 2048, 2049, 16032, 32000, 65537, 128256, 152064, 393216])
def test_workspaces_for_many_rows_do_for_fewer(V):
    """A caller asks once, for its largest step: the size of drafts' checks never falls as rows or entries rise, and a step of that size has what it needs."""
    lib = _lib()
    sizes = [lib.b200_verify_drafts_workspace_bytes(n, V) for n in range(5000)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[1] > 0
    assert all(lib.b200_verify_drafts_workspace_bytes(n, V) <= lib.b200_verify_drafts_workspace_bytes(n, V + 1000) for n in (1, 7, 48, 320, 65535))
    # what a step of n rows writes, restated: 16 bytes a row, slice and kind of row
    for n in list(range(1, 400)) + [999, 1776, 1777, 5000, 65535]:
        want = max(1, 148 * 24 // max(1, 2 * n))
        length = -(-V // want)
        length = -(-length // 8192) * 8192 if length > 4096 else max(2048, -(-length // 8) * 8)
        assert lib.b200_verify_drafts_workspace_bytes(n, V) >= n * 2 * 16 * -(-V // length)


def test_attention_workspaces_for_many_rows_do_for_fewer():
    lib = _lib()
    for hq, hkv in ((1, 1), (32, 8), (40, 8), (64, 4), (128, 128)):
        sizes = [lib.b200_paged_attn_fp8_workspace_bytes(n, hq, hkv) for n in range(3000)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("stride,block", [(2 ** 24, 128), (2 ** 27, 16), (2 ** 24 - 1, 128), (2 ** 21, 1024), (2 ** 31 - 1, 128)])
def test_attention_counts_tokens_in_32_bits(prefill, stride, block):
    """One row and one kv head: few enough tiles, but a table of more tokens than the kernels can count to the end of the last tile."""
    assert _attend(prefill, T=1, hq=1, hkv=1, stride=stride, block=block) == -3
    assert b"tokens" in _lib().b200_last_error()


@pytest.mark.parametrize("S", [2 ** 28, 2 ** 29 + 1, 2 ** 31 - 1])
def test_verify_counts_its_clusters_in_32_bits(S):
    """Eight CTAs a sequence: of more sequences only some would be looked at (2^29 + 1: one)."""
    assert _verify(S=S) == -3 and b"sequences" in _lib().b200_last_error()
