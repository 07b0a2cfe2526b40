"""Paged key / value cache on the GPU against tests/checkers_paged.py: append bit for bit, attention within the bound that
its roundings give (derived there)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from bolt_amd import capi, host_paged as hp  # noqa: E402
from checkers_paged import COMBOS, TYPES, Case, assert_attention, quantised, rotated  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def ready():
    assert torch.cuda.is_available()
    capi.check(capi.lib().bolt_gfx950_init(), "init")


def sync():
    capi.check(capi.lib().bolt_gfx950_synchronize(), "sync")
    torch.cuda.synchronize()


def bits(t):
    t = t.cpu().contiguous()
    return t.view({4: torch.int32, 2: torch.int16, 1: torch.int8}[t.element_size()])


def angles(positions, rot, seed=0, interleaved=False):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(positions, rot // 2, generator=g, dtype=torch.float64) * 6.3
    return a.cos().float(), a.sin().float()


def attend(case, prompt, **kw):
    cache, batch, q = case.gpu(offsets=prompt)
    out = torch.full_like(q, 77.0)
    fn = hp.paged_attention_prompt if prompt else hp.paged_attention_decode
    fn(cache, batch, q, out=out, window=case.window, **kw)
    sync()
    return out


def test_rows_four_billion_elements_apart_are_refused():
    """2^32 + 128 elements between rows: 128 in 32 bits"""
    c = Case("f16", "f16", 2, 2, 64, 16, (9, 5), (1, 1), seed=1)
    cache, batch, q = c.gpu(offsets=False)
    far = torch.empty((1 << 32) + 256, dtype=torch.float16, device="cuda").as_strided((2, 2, 64), ((1 << 32) + 128, 64, 1))
    for call in (lambda: hp.paged_attention_decode(cache, batch, far), lambda: hp.paged_attention_decode(cache, batch, q, out=far),
                 lambda: hp.kv_cache_append(cache, batch, far, q), lambda: hp.kv_cache_append(cache, batch, q, q, q, None, far)):
        with pytest.raises(capi.BoltError, match="2\\^32"):
            call()


# ---- append -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("act,cache", COMBOS)
@pytest.mark.parametrize("dim,page,rot,interleaved,new,past", [
    (64, 16, 64, False, (5, 0, 17, 1), (0, 9, 30, 15)),
    (128, 8, 128, True, (1, 33), (7, 0)),
    (128, 64, 32, False, (70,), (60,)),
    (64, 1, 16, True, (3, 2), (0, 5)),
    (128, 4096, 0, False, (2, 9), (4094, 0)),
    (128, 16, 80, False, (6,), (11,)),
    (64, 8, 48, True, (6,), (11,)),
    (64, 2, 64, False, tuple(i * 7 % 4 for i in range(150)), tuple(i * 5 % 9 for i in range(150))),
])
def test_append(act, cache, dim, page, rot, interleaved, new, past):
    print("append", act, cache, dim, page, rot, interleaved, new, past, flush=True)
    heads, kv = 6, 3
    total = [p + n for p, n in zip(past, new)]
    c = Case(act, cache, heads, kv, dim, page, total, new, seed=dim + page + rot, rows=sum(new) + 3)
    pc, pb, _ = c.gpu()
    g = torch.Generator().manual_seed(9)
    qkv = (torch.randn(c.rows, (heads + 2 * kv) * dim, generator=g) * 3).to(TYPES[act])
    qkv[0, heads * dim:heads * dim + dim] = 0                                  # a key row of zeros
    if act != "f16":
        qkv[0, heads * dim + dim:heads * dim + 2 * dim] = 1e-39                # one of subnormal numbers
    q, k, v = qkv.view(c.rows, heads + 2 * kv, dim).split((heads, kv, kv), 1)
    cos, sin = angles(max(total), max(rot, 16))
    rotary = hp.Rotary(cos.cuda(), sin.cuda(), interleaved) if rot else None
    dq, dk, dv = qkv.cuda().view(c.rows, heads + 2 * kv, dim).split((heads, kv, kv), 1)
    q_out = torch.full((c.rows, heads, dim), 55.0, dtype=TYPES[act], device="cuda")
    hp.kv_cache_append(pc, pb, dk, dv, dq, rotary, q_out)
    sync()
    mine = int(c.offsets[-1])
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    pos = torch.tensor([t - n + i for t, n in zip(total, new) for i in range(n)])
    turn = (lambda x: rotated(x, cos[pos], sin[pos], interleaved)) if rot else (lambda x: x)
    assert torch.equal(bits(q_out[:mine]), bits(turn(q[:mine].float()).to(TYPES[act]))) and (q_out[mine:] == 55).all()
    at, slot = c.table[seq, pos // page].long(), pos % page
    for x, was, scale, now, now_scale in ((turn(k[:mine].float()), c.k, c.ks, pc.keep[0], pc.keep[2]), (v[:mine].float(), c.v, c.vs, pc.keep[1], pc.keep[3])):
        want, want_scale = was.clone(), None if scale is None else scale.clone()
        if cache == "i8":
            want[at, :, slot], want_scale[at, :, slot] = quantised(x)
            assert torch.equal(bits(now_scale), bits(want_scale))
        else:
            want[at, :, slot] = x.to(TYPES[cache])
        assert torch.equal(bits(now), bits(want))                              # every other slot as it was


def test_append_without_queries_in_place_and_one_row_each():
    c = Case("f32", "f16", 4, 2, 64, 16, (5, 0, 33), (1, 1, 1), seed=3)
    pc, pb, _ = c.gpu(offsets=False)
    cos, sin = angles(64, 64)
    r = hp.Rotary(cos.cuda(), sin.cuda())
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(3, h, 64, generator=g) for h in (4, 2, 2))
    dq = q.cuda()
    assert hp.kv_cache_append(pc, pb, k.cuda(), v.cuda(), dq, r, dq) is dq
    sync()
    pos = torch.tensor([4, 0, 32])
    want = rotated(q, cos[pos], sin[pos], False)
    want[1] = q[1]                                                             # length 0: nobody's row
    assert torch.equal(dq.cpu(), want)
    first = pc.keep[0].clone()
    assert hp.kv_cache_append(pc, pb, k.cuda(), v.cuda(), None, r) is None
    sync()
    assert torch.equal(bits(pc.keep[0]), bits(first))


@pytest.mark.parametrize("cache", ["f16", "i8"])
def test_append_leaves_out_what_has_no_place(cache):
    """page numbers outside the pool, positions behind the page table, in front of the sequence and behind the angles"""
    c = Case("f32", cache, 2, 1, 64, 8, (20, 30, 3, 16), (20, 6, 5, 2), seed=5, max_pages=3)
    c.table[0, 1], c.table[0, 2], c.table[3, 0] = -5, c.pages, 0x7fffffff
    pc, pb, _ = c.gpu()
    cos, sin = angles(14, 64)                                                  # sequence 3: position 14, 15 not covered
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(c.rows, h, 64, generator=g) for h in (2, 1, 1))
    q_out = torch.full_like(q, 9.0).cuda()
    hp.kv_cache_append(pc, pb, k.cuda(), v.cuda(), q.cuda(), hp.Rotary(cos.cuda(), sin.cuda()), q_out)
    sync()
    want_k, want_v, want_q = c.k.clone(), c.v.clone(), torch.full_like(q, 9.0)
    ks, vs = (None, None) if c.ks is None else (c.ks.clone(), c.vs.clone())
    for b in range(4):
        for i in range(c.new[b]):
            p, row = c.lengths[b] - c.new[b] + i, int(c.offsets[b]) + i
            if p < 0 or p >= 14:
                continue
            want_q[row] = rotated(q[row:row + 1], cos[p:p + 1], sin[p:p + 1], False)[0]
            page = int(c.table[b, p // 8])
            if 0 <= page < c.pages:
                kk = rotated(k[row:row + 1], cos[p:p + 1], sin[p:p + 1], False)[0, 0]
                if cache == "i8":
                    want_k[page, 0, p % 8], ks[page, 0, p % 8] = quantised(kk)
                    want_v[page, 0, p % 8], vs[page, 0, p % 8] = quantised(v[row, 0])
                else:
                    want_k[page, 0, p % 8], want_v[page, 0, p % 8] = kk.half(), v[row, 0].half()
    assert torch.equal(q_out.cpu(), want_q)
    for now, want in zip(pc.keep, (want_k, want_v, ks, vs)):
        assert want is None or torch.equal(bits(now), bits(want))


def test_append_of_infinities_and_nan_shows_them():
    c = Case("f32", "i8", 1, 1, 64, 8, (3,), (3,), seed=5)
    pc, pb, _ = c.gpu()
    k = torch.ones(3, 1, 64)
    k[0, 0, 5], k[1, 0, 9] = float("nan"), float("-inf")
    hp.kv_cache_append(pc, pb, k.cuda(), k.cuda())
    sync()
    scale = pc.keep[2].cpu()[c.table[0, 0].long(), 0, :3]
    assert torch.isnan(scale[0]) and scale[1] == 0 and scale[2] == 127


def test_append_of_more_rows_than_a_grid_is_wide():
    """2^26 + 2 rows of 64 threads, all but the last three nobody's"""
    rows, g = (1 << 26) + 2, torch.Generator().manual_seed(7)
    c = Case("f16", "f16", 1, 1, 64, 8, (3,), (3,), seed=7)
    pc, _, _ = c.gpu()
    new = torch.empty(rows, 1, 64, dtype=torch.float16, device="cuda")
    new[-3:] = last = torch.randn(3, 1, 64, generator=g).half().cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = hp.PagedBatch(c.table.cuda(), torch.tensor([3], **i32), torch.tensor([rows - 3, rows], **i32), rows)
    torch.cuda.synchronize()
    hp.kv_cache_append(pc, batch, new, new)
    sync()
    for now, was in zip(pc.keep[:2], (c.k, c.v)):
        want = was.clone()
        want[c.table[0, 0].long(), 0, :3] = last[:, 0].cpu()
        assert torch.equal(bits(now), bits(want))


# ---- attention --------------------------------------------------------------------------------------
DECODE = [
    # heads, kv_heads, dim, page, lengths, window
    (12, 12, 64, 16, (1, 2, 0, 16, 17, 130), 0),
    (8, 1, 128, 8, (1, 63, 64, 65, 300), 0),
    (28, 4, 128, 32, (257, 31, 1000), 0),
    (6, 2, 64, 1, (45, 7), 0),
    (40, 2, 128, 128, (700, 129), 100),
    (3, 3, 64, 4096, (1, 4097, 515), 33),
    (16, 8, 128, 64, (2500, 1, 0, 640), 1),
    (8, 2, 128, 16, (5, 128, 0, 77), 0),                                       # a table of one tile
    (71, 1, 64, 16, (40, 90), 0),                                              # five tiles of queries, the last of seven
    (1024, 1024, 64, 16, (5, 140), 0),                                         # more columns than workgroups fit the chip
    (16, 16, 128, 16, tuple(i * 37 % 400 for i in range(67)), 0),              # shares that hold several sequences and parts of others
    (2, 1, 64, 8, tuple(i * 53 % 270 for i in range(300)), 0),                 # sequences left whole,
    (8, 8, 128, 16, tuple(i * 211 % 1009 for i in range(33)), 0),
    (12, 12, 64, 32, tuple(i * 977 % 2100 for i in range(24)), 500),           # those that a window makes short, too,
    (8, 4, 128, 64, tuple(i * 977 % 2100 for i in range(70)), 1024),
    (8, 4, 128, 64, tuple(i * 977 % 2100 for i in range(20)), 1025),           # and as many that are not
]


@pytest.mark.parametrize("act,cache", COMBOS)
@pytest.mark.parametrize("shape", DECODE, ids=lambda s: str(s)[:40])
def test_decode(act, cache, shape):
    heads, kv, dim, page, lengths, window = shape
    print("decode", act, cache, shape, flush=True)
    c = Case(act, cache, heads, kv, dim, page, lengths, [1] * len(lengths), seed=heads + sum(lengths), window=window)
    out = attend(c, False)
    assert assert_attention(out, c).all()
    for b, n in enumerate(lengths):
        assert n or not out[b].any()                                           # no keys: zeros


PROMPT = [
    # heads, kv_heads, dim, page, past, new, window, rows behind the last sequence
    (12, 12, 64, 16, (0, 0, 0), (1, 2, 37), 0, 0),
    (4, 1, 128, 8, (0, 5, 64), (70, 1, 33), 0, 5),
    (14, 2, 128, 32, (31, 0, 100), (1, 0, 130), 0, 1),
    (6, 2, 64, 1, (3,), (29,), 0, 0),
    (8, 2, 128, 128, (300, 0), (65, 129), 40, 2),
    (3, 3, 64, 4096, (4090, 0), (9, 64), 0, 0),
    (10, 2, 64, 64, (0, 17), (200, 3), 1, 0),
    (71, 1, 64, 16, (40, 0), (3, 5), 0, 0),
    (2, 1, 128, 8, tuple(i * 29 % 90 for i in range(130)), tuple(i * 7 % 5 for i in range(130)), 0, 3),
    (8, 1, 64, 16, (700, 20, 0), (7, 40, 1), 0, 0),                            # keys of a tile shared out, of some and not of others
    (16, 2, 128, 32, (900, 3), (20, 20), 500, 0),
]


@pytest.mark.parametrize("act,cache", COMBOS)
@pytest.mark.parametrize("shape", PROMPT, ids=lambda s: str(s)[:40])
def test_prompt(act, cache, shape):
    heads, kv, dim, page, past, new, window, spare = shape
    print("prompt", act, cache, shape, flush=True)
    c = Case(act, cache, heads, kv, dim, page, [p + n for p, n in zip(past, new)], new, seed=heads + sum(new), window=window, rows=sum(new) + spare)
    out = attend(c, True)
    mine = assert_attention(out, c)
    assert mine.sum() == sum(new) and (out[torch.from_numpy(~mine).cuda()] == 77).all()


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("bf16", "bf16"), ("f16", "i8")])
def test_attention_with_lists_that_point_outside(prompt, act, cache):
    """Page numbers outside the pool are keys that nobody sees; lengths behind the page table end with it; more new tokens than
    the sequence is long: the first ones see nothing"""
    new = (3, 2, 4, 1) if prompt else (1, 1, 1, 1)
    c = Case(act, cache, 4, 2, 64, 8, (30, 21, 2, 8), new, seed=8, max_pages=3)
    c.table[0, 1], c.table[1, 0], c.table[1, 1], c.table[1, 2], c.table[3, 0] = -1, c.pages, -(1 << 31), 0x7fffffff, 12345678
    out = attend(c, prompt)
    assert_attention(out, c)
    assert not out[int(c.offsets[1])].any() and not out[int(c.offsets[3])].any()


LOW, HIGH = -(1 << 31), (1 << 31) - 1


@pytest.mark.parametrize("cache_type", ["f16", "i8"])
@pytest.mark.parametrize("offsets,lengths", [
    ((0, 5, 3, 9, 9), (20, 11, 24, 0)), ((-5, 3, 2, HIGH, 7), (HIGH, LOW, 17, -1)), ((HIGH, LOW, HIGH, 0, LOW), (24, 24, 24, 24)),
    ((0, HIGH, 0, HIGH, 0), (HIGH, 24, 5, 1)), ((9, 10, 11, 12, 13), (1, 2, 3, 4)), ((-9, -4, 0, 1, 2), (9, 24, 9, 24)),
] + [(tuple(i * 7919 % 23 - 6 for i in range(81)), tuple(i * 31 % 40 - 4 for i in range(80)))], ids=lambda s: str(s)[:40])
def test_lists_of_anything_stay_inside_the_buffers(cache_type, offsets, lengths):
    """Offsets that do not ascend, behind and in front of the rows; lengths of any size: what the calls answer means nothing, but
    nothing around the rows and the pool's pages changes"""
    print("lists", cache_type, offsets[:5], lengths[:5], flush=True)
    rows, n = 9, len(lengths)
    c = Case("f16", cache_type, 6, 2, 64, 8, (24,) * n, (1,) * n, seed=31)
    outer = [None if t is None else torch.cat([t[:2], t, t[:2]]).cuda() for t in (c.k, c.v, c.ks, c.vs)]
    before = [None if t is None else t.clone() for t in outer]
    cache = hp.PagedKvCache(*(None if t is None else t[2:-2] for t in outer))
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = hp.PagedBatch(c.table.cuda(), torch.tensor(lengths, **i32), torch.tensor(offsets, **i32), rows)
    wide = [torch.full((rows + 4, 6, 64), 5.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    q, k = (torch.ones(rows, h, 64, dtype=torch.float16, device="cuda") for h in (6, 2))
    r = hp.Rotary(*(torch.ones(24, 32, device="cuda") for _ in range(2)))
    hp.kv_cache_append(cache, batch, k, k, q, r, wide[0][2:-2])
    hp.paged_attention_prompt(cache, batch, q, out=wide[1][2:-2])
    sync()
    for t in wide:
        assert (t[:2] == 5).all() and (t[-2:] == 5).all()
    for t, was in zip(outer, before):
        for end in (slice(0, 2), slice(-2, None)):
            assert t is None or torch.equal(bits(t[end]), bits(was[end]))


@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "i8")])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_token_sees_nothing_of_later_ones(act, cache, bad):
    """infinities and NaN in the key and the value of a later token, in the same tile: the rows before it are those of the clean
    cache, the rows from it on show them; and behind a window they are gone again"""
    new, spot = 90, 41
    c = Case(act, cache, 4, 2, 64, 16, (new + 3,), (new,), seed=11)
    clean = attend(c, True)
    page, slot = int(c.table[0, (spot + 3) // 16]), (spot + 3) % 16
    for which in ("k", "v"):
        scales, store = (c.ks, c.ks) if which == "k" else (c.vs, c.vs)
        target = store if cache == "i8" else (c.k if which == "k" else c.v)
        keep = target.clone()
        if cache == "i8":
            target[page, :, slot] = bad
        else:
            target[page, :, slot, 7] = bad
        out = attend(c, True)
        assert torch.equal(bits(out[:spot]), bits(clean[:spot])), which
        if not (cache == "i8" and np.isinf(bad)):                              # a scale of infinity stands for zeros
            assert not torch.isfinite(out[spot:].float()).all(dim=-1).any() if which == "v" else True
        c.window = 20
        windowed = attend(c, True)
        target.copy_(keep)
        again = attend(c, True)
        assert torch.equal(bits(windowed[:spot]), bits(again[:spot])) and torch.equal(bits(windowed[spot + 20:]), bits(again[spot + 20:])), which
        c.window = 0


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("act,cache", COMBOS)
def test_large_and_small_scores(prompt, act, cache):
    """queries whose scores span hundreds: the softmax is nearly one key; and nearly equal ones; fp16's largest and smallest"""
    for size in (60.0, 1e-4, 0.0):
        c = Case(act, cache, 4, 2, 64, 16, (150, 40), (20, 1) if prompt else (1, 1), seed=12)
        c.q = (c.q.float() * size).to(TYPES[act])
        if cache != "i8":
            c.k[c.k.isfinite()] *= 0.01 if size == 60.0 else 1.0
        assert_attention(attend(c, prompt), c)


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("act,cache", COMBOS)
def test_scales_below_zero_and_of_zero(prompt, act, cache):
    c = Case(act, cache, 4, 2, 128, 16, (150, 40, 0), (20, 1, 0) if prompt else (1, 1, 1), seed=25)
    for scale in (-0.3, 0.0, -1e-3):
        assert_attention(attend(c, prompt, scale=scale), c, scale)


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_scales_of_an_int8_cache_of_either_sign_and_any_size(act, prompt):
    """real = stored / scale, whatever the scale is: negative ones, and values 2^40 apart, the largest steps among the last keys"""
    c = Case(act, "i8", 4, 2, 64, 16, (150, 40), (20, 1) if prompt else (1, 1), seed=32)
    g = torch.Generator().manual_seed(33)
    sign = 1 - 2 * torch.randint(0, 2, c.vs.shape, generator=g)
    c.ks, c.vs = c.ks * sign, c.vs * sign.roll(1, 0)
    assert_attention(attend(c, prompt), c)
    c.vs = c.vs * 2.0 ** torch.randint(-20, 21, c.vs.shape, generator=g)
    c.vs[c.table[0, :2].long()] *= 2.0 ** 30                                   # small values first
    assert_attention(attend(c, prompt), c)


@pytest.mark.parametrize("cache_type", ["f16", "i8"])
def test_sequences_that_share_pages(cache_type):
    """a common beginning in the same pages, once in one sequence's own order and once twice in one table"""
    for prompt in (False, True):
        c = Case("f16", cache_type, 6, 3, 64, 16, (50, 60, 48), (3, 9, 2) if prompt else (1, 1, 1), seed=26)
        c.table[1, :2] = c.table[0, :2]
        c.table[2, 0] = c.table[2, 1] = c.table[0, 1]
        assert_attention(attend(c, prompt), c)


@pytest.mark.parametrize("cache_type", ["f16", "i8"])
def test_a_table_of_two_billion_positions_for_many(cache_type):
    """130 rows of 2^31 - 4096 positions each, which are more tiles of 128 keys than 31 bits count; lengths among them are short,
    but for two whose keys fill several tiles of the larger ones"""
    lengths = [1 + i * 97 % 300 for i in range(128)] + [5000, 1300]
    c = Case("f16", cache_type, 2, 1, 64, 4096, lengths, [1] * 130, seed=27)
    want = attend(c, False)
    assert_attention(want, c)
    cache, batch, q = c.gpu(offsets=False)
    table = torch.full((130, (1 << 31) // 4096 - 1), -1, dtype=torch.int32, device="cuda")
    table[:, :c.max_pages] = c.table.cuda()
    torch.cuda.synchronize()
    out = hp.paged_attention_decode(cache, hp.PagedBatch(table, batch.keep[1]), q)
    sync()
    assert_attention(out, c)


def test_queries_beyond_the_range_of_fp16():
    for size in (3e6, 1e-9, 3e30):
        c = Case("f32", "f16", 4, 2, 64, 16, (70,), (9,), seed=13)
        c.q = c.q * size
        for prompt in (True, False):
            c.new, c.offsets, c.rows = ([9], torch.tensor([0, 9], dtype=torch.int32), 9) if prompt else ([1], torch.tensor([0, 1], dtype=torch.int32), 1)
            c.q = c.q[:c.rows]
            assert_attention(attend(c, prompt, scale=0.125 / size), c, 0.125 / size)
    c = Case("bf16", "i8", 4, 2, 64, 16, (70,), (9,), seed=13)
    c.q = (c.q.float() * 1e30).bfloat16()
    assert_attention(attend(c, True, scale=1e-31), c, 1e-31)


@pytest.mark.parametrize("prompt", [False, True])
def test_strided_rows(prompt):
    """q and out as parts of wider rows, around which nothing changes"""
    c = Case("f16", "f16", 6, 2, 128, 16, (50, 33), (7, 3) if prompt else (1, 1), seed=14)
    cache, batch, q = c.gpu(offsets=prompt)
    wide_q = torch.full((c.rows, 10, 128), float("nan"), dtype=torch.float16, device="cuda")
    wide_q[:, 2:8] = q
    wide = torch.full((c.rows, 9, 128), 5.0, dtype=torch.float16, device="cuda")
    fn = hp.paged_attention_prompt if prompt else hp.paged_attention_decode
    fn(cache, batch, wide_q[:, 2:8], out=wide[:, 1:7])
    sync()
    assert_attention(wide[:, 1:7], c)
    assert (wide[:, 0] == 5).all() and (wide[:, 7:] == 5).all()


@pytest.mark.parametrize("prompt", [False, True])
def test_same_bytes_again_and_on_another_stream(prompt):
    c = Case("f16", "f16", 16, 4, 128, 16, (3000, 700, 90), (40, 200, 90) if prompt else (1, 1, 1), seed=15)
    first = attend(c, prompt)
    cache, batch, q = c.gpu(offsets=prompt)
    fn = hp.paged_attention_prompt if prompt else hp.paged_attention_decode
    ws = hp.paged_attention_workspace(cache, batch, 16)
    ws.fill_(255)                                                              # what a workspace holds before does not matter
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    capi.check(capi.lib().bolt_gfx950_set_stream(stream.cuda_stream), "set_stream")
    try:
        outs = [torch.empty_like(q) for _ in range(3)]
        torch.cuda.synchronize()
        for o in outs:
            fn(cache, batch, q, out=o, workspace=ws)
        sync()
    finally:
        capi.check(capi.lib().bolt_gfx950_set_stream(None), "set_stream")
    mine = slice(0, int(c.offsets[-1]))
    for o in outs:
        assert torch.equal(bits(o[mine]), bits(first[mine]))


@pytest.mark.parametrize("prompt", [False, True])
def test_what_a_call_allocates_is_not_handed_out_before_its_work_is_done(prompt):
    """The library's stream is behind; torch's own goes on and asks for memory of the sizes that the call has just let go"""
    c = Case("f32", "f16", 8, 2, 128, 16, (900, 400), (9, 1) if prompt else (1, 1), seed=24)
    want = attend(c, prompt)
    cache, batch, q = c.gpu(offsets=prompt)
    fn = hp.paged_attention_prompt if prompt else hp.paged_attention_decode
    size = hp.paged_attention_workspace(cache, batch, 8).numel()
    side = torch.cuda.Stream()
    capi.check(capi.lib().bolt_gfx950_set_stream(side.cuda_stream), "set_stream")
    try:
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        out = fn(cache, batch, q)
        taken = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]
        torch.cuda.current_stream().synchronize()
        sync()
    finally:
        capi.check(capi.lib().bolt_gfx950_set_stream(None), "set_stream")
    mine = slice(0, int(c.offsets[-1]))
    assert torch.equal(bits(out[mine]), bits(want[mine])) and all((t == 255).all() for t in taken)


@pytest.mark.parametrize("cache_type", ["f16", "i8"])
def test_offsets_beyond_32_bits(cache_type):
    """a pool of more than 2^32 elements, the sequence in its last pages"""
    page, dim = 4096, 128
    pages = (1 << 32) // (page * dim) + 5
    dtype = TYPES[cache_type]
    k, v = (torch.zeros(pages, 1, page, dim, dtype=dtype, device="cuda") for _ in range(2))
    scales = [torch.ones(pages, 1, page, device="cuda") for _ in range(2)] if cache_type == "i8" else [None, None]
    cache = hp.PagedKvCache(k, v, *scales)
    c = Case("f16", cache_type, 4, 1, dim, page, (page + 77,), (page + 77,), seed=16, spare=0)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    c.table = torch.tensor([[1, 0]], dtype=torch.int32)                        # the same two pages of a small pool
    lengths = torch.tensor([page + 77], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(17)
    kn, vn = (torch.randn(page + 77, 1, dim, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    hp.kv_cache_append(cache, hp.PagedBatch(table, lengths, torch.tensor([0, page + 77], dtype=torch.int32, device="cuda"), page + 77), kn, vn)
    q = torch.randn(1, 4, dim, generator=g, device="cuda", dtype=torch.float16)
    out = hp.paged_attention_decode(cache, hp.PagedBatch(table, lengths), q)
    last = hp.paged_attention_prompt(cache, hp.PagedBatch(table, lengths, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1), q)
    sync()
    c.k, c.v = k[-2:].cpu(), v[-2:].cpu()
    if cache_type == "i8":
        c.ks, c.vs = scales[0][-2:].cpu(), scales[1][-2:].cpu()
    c.pages, c.new, c.offsets, c.rows, c.q = 2, [1], torch.tensor([0, 1], dtype=torch.int32), 1, q.cpu()
    assert_attention(out, c)
    assert_attention(last, c)
    assert not k[:-2].any() and not v[:-2].any()


def test_captured_step_replayed_with_other_lengths():
    """append and attention of one step in a graph; lengths, pages and inputs change between the replays, and the library's
    eager calls run in between; a second graph with a workspace of its own is replayed beside it"""
    heads, kv, dim, page, batch = 8, 2, 64, 16, 5
    g = torch.Generator(device="cuda").manual_seed(18)
    pages = 60
    cos, sin = angles(160, dim)
    rotary = hp.Rotary(cos.cuda(), sin.cuda())

    def fresh():
        k, v = (torch.randn(pages, kv, page, dim, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
        return hp.PagedKvCache(k, v)
    lengths = torch.ones(batch, dtype=torch.int32, device="cuda")
    table = torch.randperm(pages, generator=g, device="cuda")[:batch * 10].to(torch.int32).view(batch, 10).contiguous()
    b = hp.PagedBatch(table, lengths)
    qkv = torch.zeros(batch, heads + 2 * kv, dim, device="cuda")
    q, k, v = qkv.split((heads, kv, kv), 1)

    def step(cache, ws, q_out, out):
        hp.kv_cache_append(cache, b, k, v, q, rotary, q_out)
        hp.paged_attention_decode(cache, b, q_out, out=out, workspace=ws)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    capi.check(capi.lib().bolt_gfx950_set_stream(side.cuda_stream), "set_stream")
    try:
        sides = []
        for _ in range(2):
            cache = fresh()
            ws = hp.paged_attention_workspace(cache, b, heads)
            q_out, out = (torch.zeros(batch, heads, dim, device="cuda") for _ in range(2))
            torch.cuda.synchronize()
            step(cache, ws, q_out, out)                                        # nothing left to initialise inside the capture
            sync()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(cache, ws, q_out, out)
            sides.append((cache, ws, q_out, out, graph))
        for n in (1, 0, 7, 150, 16, 33):
            lengths.copy_(torch.tensor([n, max(n - 1, 0), (3 * n) % 160, 1, 0], dtype=torch.int32))
            qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
            eager = []
            for cache, _, q_out, _, _ in sides:                                # rows of empty places are nobody's: both start from the same
                twin, q_twin, out = hp.PagedKvCache(cache.keep[0].clone(), cache.keep[1].clone()), q_out.clone(), torch.zeros(batch, heads, dim, device="cuda")
                ws = hp.paged_attention_workspace(twin, b, heads)
                torch.cuda.synchronize()
                step(twin, ws, q_twin, out)
                sync()
                eager.append((twin, out))
            for one in sides:
                one[4].replay()
            torch.cuda.synchronize()
            for one, (twin, out) in zip(sides, eager):
                assert torch.equal(bits(one[0].keep[0]), bits(twin.keep[0])) and torch.equal(bits(one[0].keep[1]), bits(twin.keep[1])), n
                assert torch.equal(bits(one[3]), bits(out)), n
    finally:
        capi.check(capi.lib().bolt_gfx950_set_stream(None), "set_stream")


@pytest.mark.parametrize("act,cache_type", [("f16", "f16"), ("bf16", "i8")])
def test_captured_prompts_replayed_with_other_lengths(act, cache_type):
    """a chunk of prompts in a graph: offsets, lengths and queries change between the replays, empty places and none at all among
    them; the library's eager calls run in between and give the same bytes"""
    c = Case(act, cache_type, 8, 2, 128, 16, (400, 90, 33), (30, 9, 1), seed=28, rows=48)
    cache, batch, q = c.gpu()
    _, lengths, offsets = batch.keep
    ws = hp.paged_attention_workspace(cache, batch, 8)
    out = torch.full_like(q, 7.0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    capi.check(capi.lib().bolt_gfx950_set_stream(side.cuda_stream), "set_stream")
    try:
        hp.paged_attention_prompt(cache, batch, q, out=out, workspace=ws)
        sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            hp.paged_attention_prompt(cache, batch, q, out=out, workspace=ws)
        g = torch.Generator().manual_seed(29)
        for held, new in (((400, 90, 33), (30, 9, 1)), ((17, 0, 0), (17, 0, 0)), ((0, 0, 0), (0, 0, 0)), ((399, 64, 1), (1, 40, 1)), ((200, 80, 20), (7, 0, 41))):
            c.lengths, c.new = list(held), list(new)
            c.offsets = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)
            c.q = torch.randn(c.q.shape, generator=g).to(TYPES[act])
            for to, values in ((lengths, torch.tensor(held, dtype=torch.int32)), (offsets, c.offsets), (q, c.q), (out, torch.full_like(c.q, 7.0))):
                to.copy_(values)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            mine = assert_attention(out, c)
            assert (out[torch.from_numpy(~mine).cuda()] == 7).all()
            eager = torch.full_like(q, 7.0)
            torch.cuda.synchronize()
            hp.paged_attention_prompt(cache, batch, q, out=eager)
            sync()
            assert torch.equal(bits(eager), bits(out))
    finally:
        capi.check(capi.lib().bolt_gfx950_set_stream(None), "set_stream")


def test_first_call_of_a_kind_inside_a_capture():
    """a process that has called bolt_gfx950_init and nothing else"""
    import subprocess
    import sys
    code = """
import sys; sys.path[:0] = %r
import torch
from bolt_amd import capi, host_paged as hp
from checkers_paged import Case, assert_attention
capi.check(capi.lib().bolt_gfx950_init(), "init")
c = Case("f16", "f16", 4, 2, 64, 16, (50, 7), (20, 1), seed=34)
cache, batch, q = c.gpu()
out, side = torch.zeros_like(q), torch.cuda.Stream()
ws = hp.paged_attention_workspace(cache, batch, 4)
torch.cuda.synchronize()
capi.check(capi.lib().bolt_gfx950_set_stream(side.cuda_stream), "set_stream")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    hp.paged_attention_prompt(cache, batch, q, out=out, workspace=ws)
for _ in range(3):
    out.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert_attention(out, c)
print("captured")
""" % (sys.path,)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_two_threads_at_once():
    """every thread has a stream of its own; workspaces are apart, the cache is shared"""
    import threading
    c = Case("f16", "f16", 16, 4, 128, 16, (1500, 700, 90), (1, 1, 1), seed=30)
    p = Case("f16", "f16", 16, 4, 128, 16, (1500, 700, 90), (40, 200, 90), seed=30)
    want = [attend(c, False), attend(p, True)]
    sides = [(hp.paged_attention_decode, *c.gpu(offsets=False)), (hp.paged_attention_prompt, *p.gpu())]
    torch.cuda.synchronize()
    outs, errors = [[], []], []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            capi.check(capi.lib().bolt_gfx950_set_stream(stream.cuda_stream), "set_stream")
            fn, cache, batch, q = sides[i]
            with torch.cuda.stream(stream):
                for _ in range(20):
                    outs[i].append(fn(cache, batch, q))
            stream.synchronize()
            capi.check(capi.lib().bolt_gfx950_set_stream(None), "set_stream")
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i, case in enumerate((c, p)):
        mine = slice(0, int(case.offsets[-1]))
        assert len(outs[i]) == 20 and all(torch.equal(bits(o[mine]), bits(want[i][mine])) for o in outs[i])


@pytest.mark.parametrize("cache_type", ["f16", "i8"])
def test_generation_over_an_int8_projection(cache_type):
    """What the operators are for: hidden states go through the library's int8 QKV product, prompts are stored and attended, then
    tokens one by one; every row is held against attention over the cache's own contents, in which a token that came in a
    prompt and one that came alone are the same bytes"""
    from bolt_amd import host
    heads, kv, dim, page, hidden = 4, 2, 64, 16, 128
    width = (heads + 2 * kv) * dim
    rng = np.random.default_rng(19)
    weight = torch.from_numpy(rng.integers(-127, 128, size=(width, hidden), dtype=np.int8)).cuda()
    blob, bdesc, rhs = host.mmm_transform_rhs(weight, capi.DF_TRANSPOSE, hidden, width)
    column = torch.full((width,), 200.0, device="cuda")
    lengths, steps = [21, 1, 40], 5
    most = max(lengths) + steps
    x = torch.from_numpy(rng.standard_normal((3, most, hidden)).astype(np.float32)).cuda()
    scale_in = torch.tensor([40.0], device="cuda")                             # static: the products of a row do not depend on its batch

    def project(rows):
        n = rows.shape[0]
        u8 = (rows * 40.0 + 128.0).round().clamp(1, 255).to(torch.uint8)
        out = torch.empty(n, width, device="cuda")
        capi.check(capi.lib().bolt_gfx950_mmm_int8_perchannel(n, width, hidden, u8.data_ptr(), blob.data_ptr(), blob.data_ptr() + rhs,
                                                             out.data_ptr(), scale_in.data_ptr(), column.data_ptr(), None), "project")
        return out.view(n, heads + 2 * kv, dim).split((heads, kv, kv), 1)
    held = -(-most // page)
    dtype = TYPES[cache_type]

    def pool():
        k, v = (torch.zeros(3 * held, kv, page, dim, dtype=dtype, device="cuda") for _ in range(2))
        s = [torch.ones(3 * held, kv, page, device="cuda") for _ in range(2)] if cache_type == "i8" else [None, None]
        return hp.PagedKvCache(k, v, *s)
    table = torch.randperm(3 * held, device="cuda").to(torch.int32).view(3, held).contiguous()
    cos, sin = angles(most, dim)
    rotary = hp.Rotary(cos.cuda(), sin.cuda())

    def check(cache, batch_lengths, new, q, out):
        c = Case("f32", cache_type, heads, kv, dim, page, batch_lengths, new, seed=1)
        c.table, c.pages, c.max_pages = table.cpu(), 3 * held, held
        c.k, c.v, c.ks, c.vs = (None if t is None else t.cpu() for t in cache.keep)
        c.q = q.cpu()
        assert assert_attention(out, c).all()

    def prompt(cache, upto):
        n = torch.tensor(upto, dtype=torch.int32, device="cuda")
        offsets = torch.cat([n.new_zeros(1), n.cumsum(0, dtype=torch.int32)])
        b = hp.PagedBatch(table, n, offsets, sum(upto))
        q, k, v = project(torch.cat([x[i, :u] for i, u in enumerate(upto)]))
        q = hp.kv_cache_append(cache, b, k, v, q, rotary)
        out = hp.paged_attention_prompt(cache, b, q)
        sync()
        return q, out
    cache = pool()
    q, out = prompt(cache, lengths)
    check(cache, lengths, lengths, q, out)
    for step in range(steps):
        now = [n + step + 1 for n in lengths]
        b = hp.PagedBatch(table, torch.tensor(now, dtype=torch.int32, device="cuda"))
        q, k, v = project(torch.stack([x[i, n - 1] for i, n in enumerate(now)]))
        q = hp.kv_cache_append(cache, b, k, v, q, rotary)
        out = hp.paged_attention_decode(cache, b, q)
        sync()
        check(cache, now, [1, 1, 1], q, out)
    whole = pool()
    prompt(whole, [n + steps for n in lengths])
    for one, other in zip(cache.keep, whole.keep):
        assert one is None or torch.equal(bits(one), bits(other))


def test_host_mirror_refuses():
    c = Case("f16", "f16", 4, 2, 64, 16, (9, 5), (1, 1), seed=1)
    cache, batch, q = c.gpu(offsets=False)
    ragged = c.gpu()[1]
    k = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    for call in (lambda: hp.paged_attention_decode(cache, batch, q[:1]), lambda: hp.paged_attention_decode(cache, batch, q.float()[..., :32]),
                 lambda: hp.paged_attention_decode(cache, batch, q.transpose(1, 2)), lambda: hp.paged_attention_decode(cache, batch, q.cpu()),
                 lambda: hp.paged_attention_decode(cache, batch, q.bfloat16()), lambda: hp.paged_attention_decode(cache, ragged, q),
                 lambda: hp.paged_attention_prompt(cache, batch, q), lambda: hp.paged_attention_decode(cache, batch, q, out=q),
                 lambda: hp.paged_attention_decode(cache, batch, q, out=torch.empty_like(q).float()), lambda: hp.paged_attention_decode(cache, batch, q[:, :3]),
                 lambda: hp.paged_attention_decode(cache, batch, q, workspace=torch.empty(0, dtype=torch.uint8, device="cuda")),
                 lambda: hp.paged_attention_decode(cache, batch, q, window=-1), lambda: hp.paged_attention_decode(cache, batch, q, window=1 << 32),
                 lambda: hp.kv_cache_append(cache, batch, k, k, q[0]), lambda: hp.kv_cache_append(cache, batch, k[:1], k), lambda: hp.kv_cache_append(cache, batch, k.bfloat16(), k.bfloat16()),
                 lambda: hp.kv_cache_append(cache, batch, k, k.float()), lambda: hp.kv_cache_append(cache, batch, k, k, q.float()),
                 lambda: hp.kv_cache_append(cache, batch, k, k, q, hp.Rotary(torch.zeros(9, 4, device="cuda"), torch.zeros(9, 4, device="cuda")))):
        with pytest.raises(capi.BoltError):
            call()
