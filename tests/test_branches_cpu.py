"""Several continuations of a sequence without a GPU: what the entry points refuse, and the plain forms against small examples."""
import pytest
import torch

import branches_util as U
from conftest import pkg

BUF = 0x10000   # an aligned address that nothing reads: every call here is refused before a launch


def _lib():
    return pkg("_abi").lib()


def _attend(**kw):
    a = dict(q=BUF, ldq=32 * 128, k=BUF, v=BUF, n_blocks=9, bt=BUF, stride=4, seq=None, ctx=BUF, masks=BUF, words=2, out=BUF, ldo=32 * 128, T=3, hq=32, hkv=8, block=128,
             scale=0.1, ws=BUF, size=1 << 40)
    a.update(kw)
    return _lib().b200_paged_attn_tree(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    ({"q": None}, -1), ({"k": None}, -1), ({"v": None}, -1), ({"bt": None}, -1), ({"ctx": None}, -1), ({"out": None}, -1), ({"masks": None}, -1), ({"words": -1}, -1),
    ({"words": 33}, -3), ({"T": -2}, -1), ({"hq": 31}, -1), ({"hkv": 0}, -1), ({"hq": 34, "hkv": 2, "ldq": 34 * 128, "ldo": 34 * 128}, -3), ({"stride": 0}, -1),
    ({"block": 100}, -3), ({"block": 8}, -3), ({"block": 192}, -3), ({"n_blocks": 0}, -1), ({"n_blocks": 1 << 40}, -1), ({"ldq": 32 * 128 - 8}, -1), ({"ldo": 32 * 128 + 2}, -1),
    ({"q": BUF + 2}, -1), ({"out": BUF + 8}, -1), ({"k": BUF + 8}, -1), ({"v": BUF + 4}, -1), ({"masks": BUF + 2}, -1), ({"scale": float("inf")}, -1), ({"scale": float("nan")}, -1),
    ({"scale": 0.0}, -1), ({"scale": -1.0}, -1), ({"ws": None}, -1), ({"size": 0}, -1), ({"ws": BUF + 8}, -1), ({"stride": 2 ** 24, "block": 128}, -3), ({"T": 4097}, -3)])
def test_attention_refuses(kw, code):
    assert _attend(**kw) == code
    assert b"paged_attn_tree" in _lib().b200_last_error()


def test_attention_refuses_tables_whose_places_are_no_ints():
    """A mask's last bit lies up to 1024 tokens behind a context, tiles are looked up to 2048 tokens ahead."""
    assert _attend(T=1, hq=1, hkv=1, ldq=128, ldo=128, stride=2 ** 24 - 16, block=128) == -3 and b"tokens" in _lib().b200_last_error()
    assert _attend(T=1, hq=1, hkv=1, ldq=128, ldo=128, stride=2 ** 24 - 32, block=128) == -3 and b"tokens" in _lib().b200_last_error()
    assert _attend(T=1, hq=1, hkv=1, ldq=128, ldo=128, stride=2 ** 24 - 33, block=128, size=0) == -1 and b"workspace" in _lib().b200_last_error()
    assert _attend(T=4096, stride=2 ** 17, block=128) == -3 and b"rows" in _lib().b200_last_error()   # rows x heads x tiles


def test_attention_of_no_rows_is_nothing():
    assert _attend(T=0, ws=None, size=0) == 0
    assert _lib().b200_paged_attn_tree_workspace_bytes(0, 32, 8) == 0 and _lib().b200_paged_attn_tree_workspace_bytes(5, 32, 0) == 0
    assert _lib().b200_paged_attn_tree_workspace_bytes(5, 32, 8) > 0


def _select(**kw):
    a = dict(logits=BUF, ld=1000, scores=None, starts=BUF, S=2, n=7, V=1000, take=8, rows=BUF, tokens=BUF, out=BUF, ws=BUF, size=1 << 40)
    a.update(kw)
    return _lib().b200_beam_select(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    ({"logits": None}, -1), ({"starts": None}, -1), ({"rows": None}, -1), ({"tokens": None}, -1), ({"out": None}, -1), ({"S": -1}, -1), ({"n": -1}, -1), ({"V": 0}, -1),
    ({"ld": 999}, -1), ({"take": 0}, -1), ({"take": -3}, -1), ({"take": 129}, -3), ({"V": 393217, "ld": 2 ** 20}, -3), ({"n": 65536}, -3), ({"S": 2 ** 28}, -3), ({"ws": None}, -1),
    ({"size": 8}, -1), ({"ws": BUF + 4}, -1), ({"logits": BUF + 1}, -1)])
def test_select_refuses(kw, code):
    assert _select(**kw) == code
    assert b"beam_select" in _lib().b200_last_error()


def test_select_of_no_sequences_is_nothing_and_one_workspace_does_for_fewer_rows():
    assert _select(S=0) == 0
    size = _lib().b200_beam_select_workspace_bytes
    assert size(0, 5, 5) == 0 and size(5, 0, 5) == 0 and size(5, 5, 0) == 0
    for V in (1, 1000, 2049, 32000, 128256, 393216):
        need = [size(n, V, 16) for n in range(1, 1500)]
        assert all(a <= b for a, b in zip(need, need[1:]))


def _accept(**kw):
    a = dict(target=BUF, drafts=BUF, parents=BUF, starts=BUF, slots=BUF, S=2, n=7, out=BUF, rows=BUF, accepted=BUF, src=BUF, dst=BUF)
    a.update(kw)
    return _lib().b200_accept_tree(*a.values(), None)


@pytest.mark.parametrize("kw", [{"target": None}, {"drafts": None}, {"parents": None}, {"starts": None}, {"out": None}, {"rows": None}, {"accepted": None}, {"S": -1}, {"n": -1},
                                {"slots": None}, {"src": None}, {"dst": None}, {"slots": None, "src": None}])
def test_accept_refuses(kw):
    assert _accept(**kw) == -1
    assert b"accept_tree" in _lib().b200_last_error()
    assert _accept(S=0) == 0


def _move(**kw):
    a = dict(a=BUF, b=BUF, layers=2, stride=1 << 30, blocks=9, heads=8, block=128, row=256, src=BUF, dst=BUF, starts=BUF, groups=3, most=64)
    a.update(kw)
    return _lib().b200_cache_move(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    ({"a": None}, -1), ({"src": None}, -1), ({"dst": None}, -1), ({"starts": None}, -1), ({"layers": 0}, -1), ({"blocks": 0}, -1), ({"heads": 0}, -1), ({"block": 0}, -1),
    ({"row": 0}, -1), ({"groups": -1}, -1), ({"most": -1}, -1), ({"most": 1025}, -3), ({"blocks": 2 ** 25}, -3), ({"stride": 9 * 8 * 128 * 256 - 16}, -1),
    ({"row": 1 << 60}, -1), ({"layers": 1 << 20, "heads": 1 << 12, "blocks": 1, "row": 1, "block": 1}, -3)])
def test_move_refuses(kw, code):
    assert _move(**kw) == code
    assert b"cache_move" in _lib().b200_last_error()


def test_move_of_nothing():
    assert _move(groups=0) == 0 and _move(most=0) == 0


def test_plain_walk_takes_the_first_child_that_agrees():
    #        0 -> 1, 2, 3 (drafts 5, 7, 7); 2 -> 4 (9); 3 -> 5 (9); 4 -> 6 (1)
    parents = torch.tensor([-1, 0, 0, 0, 2, 3, 4])
    drafts = torch.tensor([0, 5, 7, 7, 9, 9, 1])
    target = torch.tensor([7, 0, 9, 9, 2, 1, 3])
    out, path, accepted, src, dst = U.accept(target, drafts, parents, torch.tensor([0, 7]), torch.arange(10, 17))
    assert out.tolist() == [7, 9, 2, -1, -1, -1, -1] and path.tolist() == [0, 2, 4, -1, -1, -1, -1] and accepted.tolist() == [2]
    assert src.tolist() == [-1, 12, 14, -1, -1, -1, -1] and dst.tolist() == [-1, 11, 12, -1, -1, -1, -1]


def test_plain_selection_of_ties_and_dead_beams():
    x = torch.tensor([[0.0, 1.0, 1.0], [0.0, 1.0, 1.0], [float("nan"), 9.0, 9.0], [5.0, float("-inf"), float("-inf")]]).to(torch.bfloat16)
    scores = torch.tensor([-1.0, -1.0, 0.0, float("-inf")])
    rows, tokens, out = U.select(x, scores, torch.tensor([0, 4]), 8)
    assert rows.tolist() == [[0, 0, 1, 1, 0, 1, -1, -1]] and tokens.tolist() == [[1, 2, 1, 2, 0, 0, -1, -1]]
    assert bool(torch.isfinite(out[0, :6]).all()) and bool((out[0, 6:] == float("-inf")).all())


def test_plain_attention_sees_the_way_to_the_root():
    assert U.lines([-1, 0, 0, 1, 3]) == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4]]
    m = U.masks([[0, 31, 33], []], 2)
    assert m.tolist() == [[1 - 2 ** 31, 2], [0, 0]]
