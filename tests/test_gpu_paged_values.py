"""Attention over a paged cache where the numbers themselves are the difficulty: slots that a row does not see but that are far
larger than those it sees, values and steps at the upper end of their types, scores whose fp32 steps are larger than one.
Against tests/checkers_paged.py (64 bits, within the bound that the roundings give)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from bolt_amd import capi, host_paged as hp  # noqa: E402
from checkers_paged import COMBOS, TYPES, Case, assert_attention, rotated  # noqa: E402
from test_gpu_paged import angles, attend, bits, ready, sync  # noqa: E402,F401

PROMPT = pytest.mark.parametrize("prompt", [False, True])


# ---- append -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("bf16", "i8"), ("f16", "f16")])
def test_a_token_without_a_slot_has_a_query_all_the_same(act, cache, turned):
    """Positions behind the page table, like page numbers outside the pool: nothing is stored, and the query is turned as any other.
    Positions in front of the sequence, and behind the angles where there are any, leave qOut as it is."""
    angles_for = 40
    c = Case(act, cache, 4, 2, 64, 8, (30, 20, 3), (26, 20, 5), seed=49, max_pages=2)
    c.table[1, 0] = c.pages + 7
    pc, pb, _ = c.gpu()
    g = torch.Generator().manual_seed(50)
    q, k = (torch.randn(c.rows, h, 64, generator=g).to(TYPES[act]) for h in (4, 2))
    cos, sin = angles(angles_for, 64)
    out = torch.full_like(q, 9.0).cuda()
    for limit in (angles_for, 18) if turned else (angles_for,):
        out.fill_(9.0)
        r = hp.Rotary(cos[:limit].cuda(), sin[:limit].cuda()) if turned else None
        hp.kv_cache_append(pc, pb, k.cuda(), k.cuda(), q.cuda(), r, out)
        sync()
        pos = torch.tensor([t - n + i for t, n in zip(c.lengths, c.new) for i in range(n)])
        left = (pos < 0) | (turned & (pos >= limit))
        at = pos.clamp(0, limit - 1)
        want = (rotated(q.float(), cos[at], sin[at], False) if turned else q.float()).to(TYPES[act])
        want[left] = 9.0
        assert torch.equal(bits(out), bits(want))
    stored = torch.zeros(c.pages, c.page, dtype=torch.bool)
    for b in range(3):
        for p in range(c.lengths[b] - c.new[b], 16):
            if 0 <= p < c.lengths[b] and int(c.table[b, p // 8]) < c.pages:
                stored[int(c.table[b, p // 8]), p % 8] = True
    for now, was in zip(pc.keep, (c.k, c.v, c.ks, c.vs)):
        if was is not None:
            assert torch.equal(bits(now.transpose(1, 2)[~stored.cuda()]), bits(was.transpose(1, 2)[~stored]))


# ---- slots that a row does not see ------------------------------------------------------------------
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [16, 2])
@pytest.mark.parametrize("step", [2.0 ** 8, 1e12, 1e30, 2.0 ** 125])
def test_large_finite_steps_of_later_tokens_change_nothing(act, page, step):
    """the value step of one token in the middle of a prompt, and of every later one, far above the others': the rows before it
    have the bytes of the cache without it, and the rows from it on what the formula gives"""
    new, past, spot = 90, 3, 41
    c = Case(act, "i8", 4, 2, 64, page, (new + past,), (new,), seed=41)
    clean = attend(c, True)
    assert_attention(clean, c)
    for behind in (1, new - spot):
        keep = c.vs.clone()
        for p in range(spot + past, spot + past + behind):
            c.vs[int(c.table[0, p // page]), :, p % page] = 1.0 / step
        out = attend(c, True)
        assert torch.equal(bits(out[:spot]), bits(clean[:spot])), (behind, step)
        if 127 * step < torch.finfo(TYPES[act]).max:                           # (else the rows behind are infinite, or of no sign that the bound leaves)
            assert_attention(out, c)
        c.vs = keep


@PROMPT
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("step", [2.0 ** 8, 1e12, 1e30, 2.0 ** 125])
def test_large_finite_steps_in_front_of_a_window_change_nothing(act, prompt, step):
    """slots that lie in the first tile that a window reaches into, in front of the window"""
    new, window, total = (9 if prompt else 1), 30, 160
    c = Case(act, "i8", 4, 2, 64, 16, (total,), (new,), seed=42, window=window)
    clean = attend(c, prompt)
    assert_attention(clean, c)
    first = total - new + 1 - window                                           # the first key that any row sees
    for p in range(first // 64 * 64, first):
        c.vs[int(c.table[0, p // 16]), :, p % 16] = 1.0 / step
    assert first % 32
    assert torch.equal(bits(attend(c, prompt)), bits(clean))


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_steps_of_all_sizes_along_a_prompt(act):
    """steps that grow from token to token by a factor of four, and that fall: every row sees other ones, and the largest it sees
    is its newest or its oldest"""
    largest = 8.0 if act == "f16" else 56.0                                    # 127 times which is a number of the type
    for grow in (2.0, -2.0):
        c = Case(act, "i8", 4, 2, 64, 16, (57,), (57,), seed=43)
        for p in range(57):
            c.vs[int(c.table[0, p // 16]), :, p % 16] = 2.0 ** (grow * (28 - p) + 56 - largest)
        assert_attention(attend(c, True), c)


# ---- values at the upper end of their types -----------------------------------------------------------
def shares(act, cache, prompt, **kw):
    """a case whose keys one workgroup has, and one whose keys several share"""
    for total in (40, 3000):
        yield Case(act, cache, 4, 2, 64, 16, (total,), (7,) if prompt else (1,), seed=44, **kw)


@PROMPT
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("size,stored", [(100, 64), (110, 4), (116, 1), (126, 0)])
def test_steps_up_to_the_largest(act, prompt, size, stored):
    """one slot in 16 holds values of a step of 2^size, up to 2^116 (fp32 holds the sum of some 2^10 of them)"""
    for c in shares(act, "i8", prompt):
        c.vs[:, :, ::16] = torch.where(c.vs[:, :, ::16].isnan(), c.vs[:, :, ::16], 2.0 ** -size)
        c.v[:, :, ::16] = c.v[:, :, ::16].sign() * stored
        assert_attention(attend(c, prompt), c)


@PROMPT
@pytest.mark.parametrize("size", [1e34, 1e36, 2e37])
def test_large_values_of_a_bf16_cache(prompt, size):
    for c in shares("bf16", "bf16", prompt):
        c.v = (c.v.float().clamp(-1, 1) * size).bfloat16()
        c.q = (c.q.float() * 4).bfloat16()                                     # few keys have most of the weight
        assert_attention(attend(c, prompt), c)


# ---- scores -------------------------------------------------------------------------------------------
@PROMPT
@pytest.mark.parametrize("act,cache", COMBOS)
@pytest.mark.parametrize("size", [3e7, 3e8, 1e9, -1e9, 7e10])
def test_scores_whose_steps_are_larger_than_one(act, cache, prompt, size):
    """|scores| of 10^7 to 10^9: fp32's steps there are 2 to 64. Every key of a sequence is the same, so that the weights are equal
    whatever the score is"""
    c = Case(act, cache, 4, 2, 64, 16, (150, 40), (20, 1) if prompt else (1, 1), seed=45)
    own = c.k[int(c.table[0, 0]), :, :1].clone()                               # [kv, 1, dim] of a slot that has values
    c.k = own.expand(c.pages, *own.shape).expand(-1, -1, c.page, -1).contiguous()
    if c.ks is not None:
        c.ks[:] = 50.0
    c.q = c.q[:1, :1].expand_as(c.q).contiguous()
    score = float((c.q[0, 0].double() @ (own[0, 0].double() / (1 if c.ks is None else 50.0))))
    scale = float(np.float32(size / score))
    out = attend(c, prompt, scale=scale).double().cpu().numpy()
    even = Case(act, cache, 4, 2, 64, 16, (150, 40), c.new, seed=45)
    even.q = torch.zeros_like(c.q)                                             # the same weights: all scores zero
    ref, bound = even.attention()
    mine = np.zeros(c.rows, dtype=bool)
    mine[:int(c.offsets[-1])] = True
    # heads of the second key head have other scores, equal among their keys all the same
    assert (np.abs(out - ref) <= bound)[mine].all()


@pytest.mark.parametrize("act,cache", COMBOS)
def test_keys_of_later_tokens_do_not_change_how_a_row_is_rounded(act, cache):
    """one later token after another gets a key whose scores are some forty times the others': the rows before it, in the same
    tile and the same wave, keep their bytes"""
    new, past = 150, 3
    c = Case(act, cache, 8, 2, 64, 16, (new + past,), (new,), seed=46)
    clean = attend(c, True)
    assert_attention(clean, c)
    for spot in (20, 69, 77, 90, 101, 130, 149):
        page, slot = int(c.table[0, (spot + past) // 16]), (spot + past) % 16
        target = c.ks if cache == "i8" else c.k
        keep = target.clone()
        target[page, :, slot] *= 1 / 40 if cache == "i8" else 40
        assert torch.equal(bits(attend(c, True)[:spot]), bits(clean[:spot])), spot
        target.copy_(keep)


@PROMPT
@pytest.mark.parametrize("size", [-0.9, -2.0, -2.3])
def test_scores_close_to_the_lowest_number(prompt, size):
    """every key's score is the same, size times 10^38: the weights are equal"""
    for total in (40, 3000):
        c = Case("bf16", "bf16", 4, 2, 64, 16, (total,), (7,) if prompt else (1,), seed=47)
        c.k[c.k.isfinite()] = 0.0
        c.k[..., 5] = torch.where(c.k[..., 5].isnan(), c.k[..., 5], 1e19)
        even = Case("bf16", "bf16", 4, 2, 64, 16, (total,), c.new, seed=47)
        even.q = torch.zeros_like(c.q)
        c.q = torch.zeros_like(c.q)
        c.q[..., 5] = size * 1e19
        out = attend(c, prompt, scale=1.0).double().cpu().numpy()
        ref, bound = even.attention()
        assert (np.abs(out - ref) <= bound).all()


@PROMPT
@pytest.mark.parametrize("act,cache", COMBOS)
@pytest.mark.parametrize("total", [40, 700, 3000])
def test_scores_of_minus_infinity(act, cache, prompt, total):
    """Where every key that a row sees has a score of minus infinity the formula is 0 / 0: the row shows it, as one that sees nothing
    (zeros) does not. Where some keys have, the others are all there is. What is not stored counts for neither."""
    new = 3 if prompt else 1
    c = Case(act, cache, 4, 2, 64, 16, (total, 20, 3), (new, new, new), seed=48)
    c.q = torch.ones_like(c.q)
    c.k = c.k.abs() if cache == "i8" else c.k
    c.table[1] = -1                                                            # a sequence without pages

    def lower(pages):
        if cache == "i8":
            c.ks[pages] = -0.0                                                 # stored / scale: minus infinity, or 0 / 0
            c.k[pages] = c.k[pages].clamp(min=1)
        else:
            c.k[pages, :, :, 9] = float("-inf")
    some = c.table[0, :2].long()
    want = Case(act, cache, 4, 2, 64, 16, (total, 20, 3), (new, new, new), seed=48)
    want.k, want.q, want.ks, want.vs, want.v = c.k.clone(), c.q, c.ks, c.vs, c.v
    want.ks = None if c.ks is None else c.ks.clone()
    want.table = c.table.clone()
    want.table[0, :2] = -1
    lower(some)
    out = attend(c, prompt)
    if (act, cache) == ("f32", "f16"):                                         # two parts to a query: infinities may be NaN
        assert out[:new].isnan().all()
        out[:new] = attend(want, prompt)[:new]
    assert_attention(out, want)
    assert not out[new:2 * new].any()
    lower(c.table[0, :-(-total // 16)].long())
    out = attend(c, prompt)
    assert out[:new].isnan().all() and not out[new:2 * new].any() and torch.equal(bits(out[2 * new:]), bits(attend(want, prompt)[2 * new:]))


@PROMPT
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_scores_that_rise_by_one_step_of_four(prompt, act):
    """Scores of 4e7 to 6e7 (to the base 2), where fp32's steps are 4, rising by one step behind the first tile: a weight of 16 times the first
    ones', which is inside the formula's range and has to be inside the kernels'"""
    for a in range(36000, 60000, 1500):
        c = Case(act, "f16", 4, 2, 64, 16, (200,), (20,) if prompt else (1,), seed=51)
        c.q = torch.zeros_like(c.q)
        c.q[..., :2] = 1.0
        c.k[c.k.isfinite()] = 0.0
        own = torch.tensor([int(c.table[0, p // 16]) * 16 + p % 16 for p in range(200)])
        k = torch.zeros(c.pages * 16, 2, 64, dtype=torch.float16)
        k[own, :, 0] = float(a // 32 * 32)                                     # a number of the type
        k[own[64:], :, 1] = 2.0 ** -8
        c.k = k.view(c.pages, 16, 2, 64).transpose(1, 2).contiguous()
        assert_attention(attend(c, prompt, scale=1024 / 1.4426950408889634), c, 1024 / 1.4426950408889634)
