"""Plain restatement, on the CPU, of the paged key / value cache's operators, and the inputs its tests share.

Attention is computed in 64 bits from the stored values, one row at a time, together with how far an implementation may be
off that rounds where the operator says it does. For a row with weights w, values v and scores s over n keys:
  A = sum w |v|                                         (elementwise; |out| <= A)
  ds: a score is a sum of head_dim products in fp32, scaled: (head_dim + 4) 2^-24 sum |q k| scale, and the exponential of an
      fp32 argument x is off by about |x| 2^-24 + 2^-22 relatively
  du: the rounding of the weights to the type the products run in (16-bit types round to nearest: eps / 2; fp32
      activations carry two 16-bit parts, 2^-21)
  dn: the sums over n keys in fp32, (n + 16) 2^-24
  da: fp16 products (an fp16 or int8 cache) hold the weights scaled so that the row's largest is 2^13 at least, where fp16's
      smallest step is 2^-24: each of n weights is off by up to 2^-37 of the largest, whatever it is itself, and the
      sum of the weights is no smaller than the largest: n 2^-37 max |v|. int8 values carry their slot's step in the weight,
      over a power of two up to twice the largest step: n 2^-37 2 127 max step
  |error| <= da + (2 ds + 2 du + 2 dn) A + (eps / 2) |out| + tiny    (weights and their sum each are off by ds + du + dn)
  tiny: below the smallest normal number n the output type's steps are n eps wide and stay that wide towards zero, so that
      rounding to the nearest is off by up to n eps / 2 there, however small the value (fp16: 2^-14 2^-10 / 2 = 2^-25)"""
import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
COMBOS = [("f32", "f16"), ("f32", "i8"), ("f16", "f16"), ("f16", "i8"), ("bf16", "bf16"), ("bf16", "i8")]


class Case:
    """A cache, a batch of sequences with `lengths` keys of which `new` are new, and the rows of its new tokens, on the CPU.
    Slots that no sequence owns hold NaN (scales of an int8 cache do), so that reading one shows."""

    def __init__(self, act, cache, heads, kv_heads, dim, page, lengths, new, seed, window=0, spare=3, rows=None, max_pages=None):
        g = torch.Generator().manual_seed(seed)
        self.act, self.cache, self.heads, self.kv_heads, self.dim, self.page = act, cache, heads, kv_heads, dim, page
        self.lengths, self.new, self.window = list(lengths), list(new), window
        held = [-(-n // page) for n in lengths]
        self.pages = sum(held) + spare
        self.max_pages = max_pages or max(max(held), 1)
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lengths), self.max_pages), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(held):
            n = min(n, self.max_pages)
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv_heads, page, dim)
        if cache == "i8":
            self.k, self.v = (torch.randint(-127, 128, shape, generator=g).to(torch.int8) for _ in range(2))
            self.ks, self.vs = (30 + 40 * torch.rand(shape[:3], generator=g) for _ in range(2))
        else:
            self.k, self.v = (torch.randn(shape, generator=g).to(TYPES[cache]) for _ in range(2))
            self.ks = self.vs = None
        owned = torch.zeros(shape[:3], dtype=torch.bool)
        for b, n in enumerate(lengths):
            for p in range(min(n, self.max_pages * page)):
                owned[self.table[b, p // page], :, p % page] = True
        for t in (self.ks, self.vs) if cache == "i8" else (self.k, self.v):
            t[~owned] = float("nan")
        self.offsets = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)
        self.rows = rows or max(int(self.offsets[-1]), 1)
        self.q = torch.randn((self.rows, heads, dim), generator=g).to(TYPES[act])

    def gpu(self, offsets=True):
        """(PagedKvCache, PagedBatch, q) on the GPU"""
        from bolt_amd import host_paged as hp
        cache = hp.PagedKvCache(*(None if t is None else t.cuda() for t in (self.k, self.v, self.ks, self.vs)))
        batch = hp.PagedBatch(self.table.cuda(), torch.tensor(self.lengths, dtype=torch.int32, device="cuda"),
                              self.offsets.cuda() if offsets else None, self.rows if offsets else None)
        return cache, batch, self.q.cuda()

    def stored(self, b, j):
        """(positions with a page, keys, values, steps of the values) of sequence b, key head j, in 64 bits"""
        pos = [p for p in range(min(self.lengths[b], self.max_pages * self.page)) if 0 <= int(self.table[b, p // self.page]) < self.pages]
        page = self.table[b, torch.tensor([p // self.page for p in pos], dtype=torch.long)].long()
        slot = torch.tensor([p % self.page for p in pos], dtype=torch.long)
        k, v = self.k[page, j, slot].double(), self.v[page, j, slot].double()
        if self.ks is not None:
            k = k / self.ks[page, j, slot].double()[:, None]
            v = v / self.vs[page, j, slot].double()[:, None]
        steps = np.ones(len(pos)) if self.vs is None else 1 / self.vs[page, j, slot].double().numpy()
        return np.array(pos, dtype=np.int64), k.numpy(), v.numpy(), steps

    def attention(self, scale=None):
        """(out, bound) as float64 arrays [rows, heads, dim]; rows that nobody owns are NaN"""
        scale = self.dim ** -0.5 if scale is None else scale
        out = np.full((self.rows, self.heads, self.dim), np.nan)
        bound = np.zeros_like(out)
        wide = self.act == "f32"
        unit = {"f32": 2.0 ** -21, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}["f16" if self.cache == "i8" and not wide else self.act]
        info = torch.finfo(TYPES[self.act])
        half, tiny = info.eps / 2, info.smallest_normal * info.eps / 2
        q = self.q.double().numpy()
        for b, (total, n) in enumerate(zip(self.lengths, self.new)):
            for j in range(self.kv_heads):
                pos, k, v, steps = self.stored(b, j)
                for i in range(n):
                    p = total - n + i
                    sees = (pos <= p) & (pos > p - self.window if self.window else True)
                    for h in range(j * self.heads // self.kv_heads, (j + 1) * self.heads // self.kv_heads):
                        row = int(self.offsets[b]) + i
                        if p < 0 or not sees.any():
                            out[row, h] = 0
                            continue
                        kk, vv = k[sees], v[sees]
                        s = kk @ q[row, h] * scale
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        a = w @ np.abs(vv)
                        ds = (self.dim + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[row, h])).max() * abs(scale) + \
                            (np.abs(s).max() + np.abs(s - s.max()).max()) * 1.45 * 2.0 ** -24 + 2.0 ** -22
                        if wide:  # two 16-bit parts of q
                            ds += 2.0 ** -21 * (np.abs(kk) @ np.abs(q[row, h])).max() * abs(scale)
                        out[row, h] = w @ vv
                        da = 0.0 if self.cache == "bf16" else len(w) * 2.0 ** -37 * (np.abs(vv).max(0) if self.cache == "f16" else 254 * steps[sees].max())
                        bound[row, h] = da + 2 * (ds + unit + (len(w) + 16) * 2.0 ** -24) * a + half * np.abs(out[row, h]) + tiny
        return out, bound


def assert_attention(got, case, scale=None):
    want, bound = case.attention(scale)
    info = torch.finfo(got.dtype)
    # the largest number is (2 - eps) 2^e, a step there is eps 2^e: from half a step above it on, rounding to the nearest gives infinity
    over = info.max * (2 - info.eps / 2) / (2 - info.eps)
    got = got.double().cpu().numpy()
    infinite = np.isinf(got) & (np.sign(got) == np.sign(want)) & (np.abs(want) + bound >= over)
    got = np.where(infinite, want, got)
    mine = ~np.isnan(want[:, 0, 0])
    bad = ~(np.abs(got - want) <= bound) & mine[:, None, None]
    assert not bad.any(), "%d values off, the worst by %g with a bound of %g, first at %s" % (
        bad.sum(), np.nanmax(np.where(bad, np.abs(got - want), 0)), bound[bad].max(), np.argwhere(bad)[0])
    return mine


def rotated(x, cos, sin, interleaved):
    """x: fp32 [rows, heads, dim]; cos, sin: fp32 [rows, rot / 2]; single fp32 operations in the order of the definition"""
    x, rot = x.clone(), 2 * cos.shape[1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, s = cos[:, None], sin[:, None]
    ra, rb = a * c - b * s, b * c + a * s
    if interleaved:
        x[..., 0:rot:2], x[..., 1:rot:2] = ra, rb
    else:
        x[..., :rot // 2], x[..., rot // 2:rot] = ra, rb
    return x


def quantised(x):
    """(int8, scale) of fp32 head rows [..., dim]: the reciprocal first, then one product"""
    top = x.abs().amax(-1)
    scale = torch.where(top == 0, torch.ones_like(top), (1.0 / top * 127.0).clamp(max=torch.finfo(torch.float32).max))
    return (x * scale[..., None]).round().clamp(-127, 127).to(torch.int8), scale
