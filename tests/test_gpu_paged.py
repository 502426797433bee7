"""The paged cache on the device against the definitions in 64 bits (oracle/paged_oracle.py): writing, reading back, and the
attention over it, at the sizes, masks and strides where they can go wrong."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def pkg():
    import toolbox_for_asr_and_tts_amd as p

    p.load()
    return p


@pytest.fixture(scope="module")
def ctx(pkg):
    return pkg.Context()


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def values_of(cache, name):
    """What the cache's buffer stands for, float64 [pages, heads, page, D]."""
    t = getattr(cache, name)
    if cache.dtype != E4M3:
        return t.double().cpu().numpy()
    return po.dequantise(t.view(torch.uint8).cpu().numpy(), getattr(cache, name + "_exp").cpu().numpy())


class Setup:
    """A cache full of values, a table in no order and a batch of (positions, new rows) pairs."""

    def __init__(self, pkg, ctx, lens, dtype=F16, store=None, dim=128, heads=2, page=16, seed=0, scale=1.0, spare=2):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype, self.page, self.heads, self.dim = dtype, page, heads, dim
        kv, q = [n for n, _ in lens], [m for _, m in lens]
        need = [-(-n // page) for n in kv]
        width = max(1, max(need, default=1))
        n_pages = sum(need) + spare
        order = np.random.default_rng(seed).permutation(n_pages)
        table, at = np.full((len(kv), width), -1), 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.free = order[at:]
        self.cache = pkg.PagedKvCache.allocate(ctx, n_pages, page, heads, dim, store or dtype)
        for name in ("k", "v"):
            t = getattr(self.cache, name)
            x = torch.randn(t.shape, generator=self.g, device="cuda") * scale
            if store == E4M3:
                t.view(torch.uint8).copy_((x * 90).clamp(-448, 448).to(E4M3).view(torch.uint8))
                e = getattr(self.cache, name + "_exp")
                e.copy_(torch.randint(119, 122, e.shape, generator=self.g, device="cuda"))
            else:
                t.copy_(x)
        self.kv, self.nq, self.table = np.array(kv), np.array(q), table
        self.cu = np.concatenate([[0], np.cumsum(q)]).astype(np.int64)
        self.n = int(self.cu[-1])

    def plan(self):
        return i32(self.cu), i32(self.kv), i32(self.table)

    def rows(self, n, heads, scale=1.0):
        return (torch.randn(n, heads, self.dim, generator=self.g, device="cuda") * scale).to(self.dtype)


def bound(dtype, dim, n, out, absv, reach, vmax):
    """How far a correct result may be from the exact one.  Scores: a sum of dim products in fp32 in any order, its scaling and
    the running maximum each rounded, so off by at most (dim + 6) 2^-24 times the largest scale * sum |q k|; a weight (and
    the sum of weights below it) is off by that much relatively, plus 2^-22 for the exponential, on both sides.  Weights
    are rounded to the type (half a step, relatively; in fp16 at least 2^-25 absolutely, against a sum of at least
    one).  Products and sums are fp32 over n terms.  The result is rounded once (fp16: at least 2^-25)."""
    half = torch.finfo(dtype).eps / 2
    rel = 2 * ((dim + 6) * 2.0 ** -24 * reach[..., None] + 2.0 ** -22) + half + (n + 8) * 2.0 ** -24
    tiny = (n * vmax + 1) * 2.0 ** -25 if dtype == F16 else 0.0
    return absv * rel * 1.01 + np.abs(out) * half + tiny + 1e-30


def check_attend(s, q, out, untouched=None, **kw):
    k, v = values_of(s.cache, "k"), values_of(s.cache, "v")
    want, absv, reach, owned = po.attend(q.double().cpu().numpy(), k, v, s.cu, s.kv, s.table, s.page, **kw)
    got = out.double().cpu().numpy()
    if untouched is not None and not owned.all():
        assert (got[~owned] == untouched).all(), "rows behind the last sequence were written"
    vmax = float(np.abs(v[np.isfinite(v)]).max())
    tol = bound(s.dtype, s.dim, int(s.kv.max()), want, absv, reach, vmax)
    for bad in (np.isnan, np.isposinf, np.isneginf):
        np.testing.assert_array_equal(bad(got[owned]), bad(want[owned]))
    fine = np.isfinite(want) & owned[:, None, None]
    err = np.abs(got - want)[fine]
    assert (err <= tol[fine]).all(), f"off by {(err / tol[fine]).max():.3g} of the bound, {err.max():.3g}"


ATTEND = {
    # name: (positions, new rows) per sequence, cache heads, query heads per cache head, page, kw
    "one token": ([(1, 1)], 1, 1, 16, {}),
    "two positions": ([(2, 1)], 2, 3, 16, {}),
    "tokens": ([(500, 1), (17, 1), (64, 1), (65, 1), (1, 1)], 4, 1, 64, {}),
    "grouped tokens": ([(333, 1), (128, 1), (31, 1)], 2, 8, 32, {}),
    "wide group": ([(200, 1), (77, 2)], 1, 40, 16, {}),
    "group of seven": ([(130, 5), (64, 5)], 2, 7, 16, {}),
    "long": ([(5003, 1), (2049, 1)], 1, 4, 128, {}),
    "long rows": ([(3001, 40)], 1, 3, 64, {}),
    "frames": ([(60, 10), (10, 10), (45, 10), (7, 7)], 4, 1, 16, dict(causal=False, window=50)),
    "whole chunk": ([(90, 33), (40, 40)], 2, 1, 16, dict(causal=False)),
    "prompt": ([(200, 200), (150, 31)], 2, 2, 32, {}),
    "prompt over cache": ([(700, 130), (400, 257)], 1, 2, 64, {}),
    "window": ([(600, 140), (300, 1), (90, 90)], 2, 2, 16, dict(window=37)),
    "window and sinks": ([(900, 140), (500, 1), (70, 70)], 1, 4, 32, dict(window=64, sinks=4)),
    "window of one": ([(300, 70), (65, 1)], 2, 1, 16, dict(window=1)),
    "many sinks": ([(800, 66), (300, 3)], 1, 2, 16, dict(window=20, sinks=130)),
    "sinks meet the window": ([(150, 150)], 1, 1, 16, dict(window=30, sinks=100)),
    "window past the start": ([(100, 100)], 1, 2, 16, dict(window=2147483647, sinks=2147483647)),
    "empty sequences": ([(0, 0), (50, 0), (40, 3), (0, 0), (33, 33)], 2, 2, 16, {}),
    "more rows than positions": ([(3, 9), (0, 2), (40, 1)], 2, 1, 16, {}),
    "largest pages": ([(700, 20), (256, 1)], 2, 2, 256, {}),
    "scale": ([(300, 20)], 2, 2, 64, dict(scale=0.5)),
    "negative scale": ([(300, 1)], 2, 2, 64, dict(scale=-0.05)),
    "max_kv": ([(300, 5), (100, 1)], 2, 2, 16, dict(max_kv=130, causal=False)),
}


@pytest.mark.parametrize("dtype, store, dim", [(F16, None, 128), (BF16, None, 64), (BF16, E4M3, 128), (F16, E4M3, 64), (F16, None, 64)],
                         ids=["f16-128", "bf16-64", "bf16-e4m3-128", "f16-e4m3-64", "f16-64"])
@pytest.mark.parametrize("name", ATTEND)
def test_attend(pkg, ctx, name, dtype, store, dim):
    lens, heads, group, page, kw = ATTEND[name]
    s = Setup(pkg, ctx, lens, dtype, store, dim, heads, page, seed=len(name))
    # q as a slice of a wider projection, and two rows that belong to nobody
    wide = s.rows(s.n + 2, heads * group + 3, 1.5)
    q = wide[:, 1:1 + heads * group]
    out = torch.full((s.n + 2, heads * group, dim), 7.0, dtype=dtype, device="cuda")
    got = s.cache.attend(q, *s.plan(), out=out, **kw)
    assert got is out
    check_attend(s, q, out, untouched=7.0, **kw)


def repeats(lens, heads, group, e4m3, cus, window=0, sinks=0):
    """How often a batch has to hold `lens` for its rows to be taken in tiles of 128: rows * heads * key tiles from 64 * 3
    (8-bit caches: 6) per compute unit on, a window's key tiles being those of its keys, the tokens of a sequence and 3."""
    tokens = sum(q for _, q in lens)
    tiles = -(-max(n for n, _ in lens) // 64)
    if window:
        tiles = min(tiles, (window + sinks + tokens // len(lens)) // 64 + 3)
    return -(-64 * (6 if e4m3 else 3) * cus // (tokens * group * heads * tiles))


@pytest.mark.parametrize("dtype, store, dim", [(F16, None, 128), (BF16, None, 64), (F16, E4M3, 128), (BF16, E4M3, 64)],
                         ids=["f16-128", "bf16-64", "f16-e4m3-128", "bf16-e4m3-64"])
@pytest.mark.parametrize("name", ["long rows", "whole chunk", "prompt", "prompt over cache", "window", "window and sinks", "many sinks", "sinks meet the window",
                                  "empty sequences"])
def test_attend_in_tiles_of_128_rows(pkg, ctx, name, dtype, store, dim):
    lens, heads, group, page, kw = ATTEND[name]
    heads = 8
    kv = [n for n, _ in lens]
    n = repeats(lens, heads, group, store == E4M3, torch.cuda.get_device_properties(0).multi_processor_count, kw.get("window", 0), kw.get("sinks", 0))
    s = Setup(pkg, ctx, lens * n, dtype, store, dim, heads, page, seed=len(name))
    q = s.rows(s.n, heads * group, 1.5)
    assert max(kv) <= s.table.shape[1] * page < max(kv) + page
    out = s.cache.attend(q, *s.plan(), **kw)
    few = sorted({0, len(lens) - 1, len(lens) * (n - 1), len(lens) * n - 1})  # some of the sequences, each with its rows
    for b in few:
        part = Setup.__new__(Setup)
        part.__dict__.update(s.__dict__)
        part.kv, part.table, part.cu = s.kv[b:b + 1], s.table[b:b + 1], np.array([0, s.nq[b]])
        part.n = int(s.nq[b])
        at = int(s.cu[b])
        if part.n:
            check_attend(part, q[at:at + part.n], out[at:at + part.n], **kw)


def test_attend_strided_output_and_one_large_score(pkg, ctx):
    """An output inside a wider array, and scores far above the rest of their row (the running maximum moves late)."""
    s = Setup(pkg, ctx, [(700, 3), (390, 40)], F16, heads=2, page=32, seed=5)
    q = s.rows(s.n, 4)
    for b, p in ((0, 650), (1, 300), (1, 351)):
        s.cache.k[s.table[b, p // 32], :, p % 32] = 6.0 * q[int(s.cu[b + 1]) - 1, ::2]
    wide = torch.full((s.n, 7, s.dim), 3.0, dtype=F16, device="cuda")
    s.cache.attend(q, *s.plan(), out=wide[:, 2:6])
    check_attend(s, q, wide[:, 2:6])
    assert bool((wide[:, :2] == 3).all()) and bool((wide[:, 6] == 3).all())


@pytest.mark.parametrize("store", [None, E4M3], ids=["16", "e4m3"])
@pytest.mark.parametrize("rows, others", [(1, 0), (3, 0), (70, 0), (150, 0), (70, 60), (150, 60)])  # (60 others: tiles of 128 rows)
def test_attend_hidden_infinities_and_nan(pkg, ctx, store, rows, others):
    """What no row sees (behind the end, on pages of others) is NaN and infinite; what later rows see alone must not reach
    the earlier ones."""
    s = Setup(pkg, ctx, [(203, rows), (180, 1)] + [(130, 130)] * others, F16, store, 128, 2, 16, seed=9)
    c = s.cache
    assert not others or repeats([(203, rows), (180, 1)] + [(130, 130)] * others, 2, 2, bool(store), 256, 20, 3) == 1
    bad_page = int(s.free[0])
    for t in (c.k, c.v):
        raw = t.view(torch.uint8) if store else t
        raw[bad_page] = 0x7f if store else float("nan")
        last = int(s.table[0, 203 // 16])
        raw[last, :, 203 % 16:] = 0x7f if store else float("inf")
        last = int(s.table[1, 180 // 16])
        raw[last, :, 180 % 16:] = 0xff if store else float("nan")
    if rows > 1:  # the last row's own key and value: it alone sees them
        page, at = int(s.table[0, 202 // 16]), 202 % 16
        (c.v.view(torch.uint8) if store else c.v)[page, 0, at, 5] = 0x7f if store else float("nan")
        if not store:
            c.v[page, 1, at, 9], c.v[page, 1, at, 100] = float("inf"), float("-inf")
    q = s.rows(s.n, 4)
    check_attend(s, q, c.attend(q, *s.plan()))
    check_attend(s, q, c.attend(q, *s.plan(), window=20, sinks=3), window=20, sinks=3)


SEEN = {
    # name: (positions, new rows) per sequence, kw: tiles of 16 rows (one wave; four; in parts), of 32, of 128 (whole; in parts)
    "one wave": ([(100, 1)], {}),
    "token": ([(420, 1), (300, 1)], {}),
    "parts": ([(9000, 1)], {}),
    "chunk": ([(420, 20)], {}),
    "chunk in parts": ([(5000, 25)], {}),
    "window": ([(900, 3)], dict(window=400, sinks=40)),
    "prompts": ([(500, 200)] * 60, {}),
    "prompts under a window": ([(700, 300)] * 40, dict(window=300, sinks=70)),
    "prompts in parts": ([(8000, 200)], dict(causal=False)),
}


@pytest.mark.parametrize("dtype, dim", [(F16, 128), (BF16, 128), (F16, 64)], ids=["f16", "bf16", "f16-64"])
@pytest.mark.parametrize("later", [False, True], ids=["below", "left behind"])
@pytest.mark.parametrize("name", SEEN)
def test_values_that_are_infinite_count_however_small_their_weight(pkg, ctx, name, later, dtype, dim):
    """Infinite values at positions inside every mask, with a weight that every format holds (20 nats below the largest: also one
    that 16 bits lose) and with one of e^-110, of which 32 bits hold nothing: by a score of its own (`below`), or because a
    later position's is so much larger (`left behind`).  Rows that do not see them are as if they were not there."""
    lens, kw = SEEN[name]
    s = Setup(pkg, ctx, lens, dtype, None, dim, 2, 32, seed=len(name))
    c, q = s.cache, s.rows(s.n, 4, 0.1)
    q[..., 0] = 16.0  # with channel 0 of the keys: a position's score in nats
    c.k[..., 0] = 0.0
    unit = dim ** 0.5 / 16

    def put(b, p, nats, values):
        page, at = int(s.table[b, p // 32]), p % 32
        c.k[page, :, at, 0] = nats * unit
        for (head, channel), v in values.items():
            c.v[page, head, at, channel] = v

    inf, nan = float("inf"), float("nan")
    some = sorted({0, len(lens) - 1})
    for b in some:
        n, m = lens[b]
        first = max(0, n - m - kw.get("window", n) + 2)  # positions that all rows see lie from here to n - m
        at = [first + (n - m - first) * i // 5 for i in (0, 1, 2, 3)]
        put(b, at[0], 0.0 if later else -110.0, {(0, 3): inf, (1, 40): -inf, (0, 9): inf})
        put(b, at[1], -20.0, {(0, 5): -inf, (0, 9): inf})
        put(b, at[2], 0.0 if later else -110.0, {(1, 7): nan, (0, 9): -inf, (0, 11): inf})
        put(b, at[3], 110.0 if later else 1.0, {})
        if m > 1:
            put(b, n - m // 2, -110.0, {(0, 21): inf, (1, 21): -inf})  # half of the rows see this one (all, without the causal mask)
    if "in parts" in name or name == "parts":
        assert ctx.lib.asrfe_paged_attention_workspace_bytes(ctx.handle, c._ref, s.n, 4, len(lens), s.table.shape[1] * 32) > 0
    out = c.attend(q, *s.plan(), **kw)
    for b in some:
        part = Setup.__new__(Setup)
        part.__dict__.update(s.__dict__)
        part.kv, part.table, part.cu = s.kv[b:b + 1], s.table[b:b + 1], np.array([0, s.nq[b]])
        a = int(s.cu[b])
        check_attend(part, q[a:a + int(s.nq[b])], out[a:a + int(s.nq[b])], **kw)


@pytest.mark.parametrize("name", SEEN)
def test_large_values_left_behind_leave_nothing(pkg, ctx, name):
    """Values of 1e36 under weights that a later score makes e^-110: their sums are brought down by factors that 32 bits do not
    hold.  What is left of them may be 2^-149 each.  (A weight may be 2^8 before that: larger values could overflow.)"""
    lens, kw = SEEN[name]
    s = Setup(pkg, ctx, lens, BF16, None, 128, 2, 32, seed=len(name))
    c, q = s.cache, s.rows(s.n, 4, 0.1)
    q[..., 0] = 16.0
    c.k[..., 0] = 0.0
    n, m = lens[0]
    first = max(0, n - m - kw.get("window", n) + 2)
    at = [first + (n - m - first) * i // 5 for i in (0, 1, 3)]
    for i, p in enumerate(at):
        page = int(s.table[0, p // 32])
        c.k[page, :, p % 32, 0] = 110 * 128 ** 0.5 / 16 if i == 2 else 0.0
        if i < 2:
            c.v[page, :, p % 32, i::7] = (1e36, -1e36)[i]
    out = c.attend(q, *s.plan(), **kw)
    k, v = values_of(c, "k"), values_of(c, "v")
    want, absv, reach, _ = po.attend(q[:m].double().cpu().numpy(), k, v, [0, m], [n], s.table[:1], 32, **kw)
    tol = bound(BF16, 128, n, want, absv, reach, 0.0) + 1e36 * 2.0 ** -149 * 4
    err = np.abs(out[:m].double().cpu().numpy() - want)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("store", [None, E4M3], ids=["16", "e4m3"])
@pytest.mark.parametrize("lens", [[(4003, 1)], [(4003, 25), (900, 3)], [(2100, 100)] * 60], ids=["token", "chunk", "tiles of 128"])
@pytest.mark.parametrize("nats", [9, 13, 16, 18, 21])
def test_small_weights_beside_a_sink(pkg, ctx, nats, lens, store):
    """The first position takes nearly all weight and has a value of zero: the result is what thousands of weights of e^-nats
    leave.  Bound: as elsewhere, but a weight is held to 2^-34 of the largest one absolutely."""
    s = Setup(pkg, ctx, lens, F16, store, 128, 2, 16, seed=nats)
    assert len(lens) < 60 or repeats(lens, 2, 2, bool(store), 256) == 1
    c, q = s.cache, s.rows(s.n, 4, 0.02)
    q[..., 0] = 16.0  # with channel 0 of the keys, zero but for the first position's: its score is `nats`, about
    if store:
        c.k_exp.fill_(123)
        c.v_exp.fill_(127)
    first = i32(s.table[:, 0]).long()

    def put(t, at, value):
        if store:
            t.view(torch.uint8)[at] = torch.tensor(value).to(E4M3).view(torch.uint8).item()
        else:
            t[at] = value

    put(c.k, (..., 0), 0.0)
    put(c.k, (first, slice(None), 0, 0), nats * 128 ** 0.5 / 16 * (16 if store else 1))
    put(c.v, ..., 1.0)
    put(c.v, (..., slice(1, None, 2)), 24.0)
    put(c.v, (first, slice(None), 0), 0.0)
    out = s.cache.attend(q, *s.plan())
    k, v = values_of(c, "k"), values_of(c, "v")
    rows = np.unique(np.linspace(0, s.n - 1, 12).astype(int))  # some of the rows, each as a batch of its own sequence
    for t in rows:
        b = int(np.searchsorted(s.cu, t, side="right") - 1)
        n = int(s.kv[b] - s.cu[b + 1] + t + 1)
        want, absv, reach, _ = po.attend(q[t:t + 1].double().cpu().numpy(), k, v, [0, 1], [n], s.table[b:b + 1], 16)
        tol = bound(F16, 128, n, want, absv, reach, 0.0) + n * 24.0 * 2.0 ** -34
        err = np.abs(out[t:t + 1].double().cpu().numpy() - want)
        assert (err <= tol).all(), (t, n, float((err / tol).max()), float(want.max()))


IN_TILES = {"16": ([(37, 1)] * 150, 2, 1), "32": ([(60, 30), (45, 28)] * 6, 2, 1), "128": ([(330, 200)] * 80, 2, 2)}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", IN_TILES)
def test_every_scale_of_values_in_attention(pkg, ctx, rows, dim, dtype):
    """A window of one position gives the position's value with a weight of one, that is, the stored number in the product's
    type: every scale 0 .. 254 and every code, rounded to nearest and, in fp16, kept inside its range."""
    lens, heads, group = IN_TILES[rows]
    assert rows != "128" or repeats(lens, heads, group, True, 256, 1) == 1
    s = Setup(pkg, ctx, lens, dtype, E4M3, dim, heads, 16, seed=dim)
    c = s.cache
    codes = torch.randint(0, 254, c.v.shape, generator=s.g, device="cuda")
    c.v.view(torch.uint8).copy_(codes + (codes >= 127))  # (all but the NaN)
    c.v_exp.copy_(torch.randint(0, 255, c.v_exp.shape, generator=s.g, device="cuda"))
    out = c.attend(s.rows(s.n, heads * group), *s.plan(), window=1).cpu()
    v = values_of(c, "v")
    for b in {0, 1, len(lens) // 2, len(lens) - 1}:
        n, m = lens[b]
        got = out[int(s.cu[b]):int(s.cu[b + 1])]
        want = torch.from_numpy(np.repeat(po.dense(v, s.table, 16, b, n)[0][n - m:], group, axis=1))
        fine = (want.abs() >= 2.0 ** -126) | (want == 0)  # (what is subnormal in fp32 and bf16 may be flushed)
        fine &= want.abs() < 3e38
        want = (want.clamp(-65504, 65504) if dtype == F16 else want).to(dtype)
        assert torch.equal(got[fine], want[fine])


SCALES = {
    # name: exponents of keys, of values, size of the queries
    "at the border": ((134, 135), (134, 135), 1e-4),
    "large": ((133, 134, 135, 136, 140, 143), (133, 135, 137, 143), 1e-4),
    "large keys": ((134, 135, 138), (119, 120), 1e-4),
    "a few large keys": ((119,) * 40 + (135, 139), (119, 120), 1e-3),
    "large values": ((118, 119), (134, 135, 139), 1.0),
    "a few large values": ((118, 119), (119,) * 40 + (135, 141), 1.0),
    "small": ((100, 104, 108, 111), (100, 103, 106, 110), 60.0),
    "all sizes": ((100, 110, 120, 128, 134, 135, 137), (100, 110, 120, 128, 134, 135, 137), 1e-4),
}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", IN_TILES)
@pytest.mark.parametrize("name", SCALES)
def test_attend_scales_of_all_sizes(pkg, ctx, name, rows, dim, dtype):
    """Keys and values take part as what they are in the product's type: exact in bf16, in fp16 rounded to nearest where they are
    below 2^-14 and kept inside +-65504."""
    lens, heads, group = IN_TILES[rows]
    s = Setup(pkg, ctx, lens, dtype, E4M3, dim, heads, 16, seed=len(name))
    c = s.cache
    for t, exps in ((c.k_exp, SCALES[name][0]), (c.v_exp, SCALES[name][1])):
        t.copy_(torch.tensor(exps, device="cuda")[torch.randint(len(exps), t.shape, generator=s.g, device="cuda")])
    q = s.rows(s.n, heads * group, SCALES[name][2])
    for kw in ({}, dict(window=20, sinks=3)):
        out = c.attend(q, *s.plan(), **kw)
        k, v = (torch.from_numpy(values_of(c, x)) for x in "kv")
        if dtype == F16:
            k, v = (t.clamp(-65504, 65504).to(F16).double() for t in (k, v))
        k, v, vmax = k.numpy(), v.numpy(), float(v.abs().max())
        for b in {0, len(lens) - 1}:
            a0, a1, n = int(s.cu[b]), int(s.cu[b + 1]), int(s.kv[b])
            want, absv, reach, _ = po.attend(q[a0:a1].double().cpu().numpy(), k, v, [0, a1 - a0], [n], s.table[b:b + 1], 16, **kw)
            tol = bound(dtype, dim, n, want, absv, reach, 0.0) + (n * vmax * 2.0 ** -34 if dtype == F16 else 0.0)
            err = np.abs(out[a0:a1].double().cpu().numpy() - want)
            assert (err <= tol).all(), (b, float((err / tol).max()), float(err.max()), float(np.abs(want).max()))


def test_attend_pages_that_do_not_exist(pkg, ctx):
    """-1 and numbers past the pool are pages that were given back; a length past the table's width has no pages there."""
    s = Setup(pkg, ctx, [(300, 1), (200, 40), (170, 3), (64, 2)], BF16, None, 64, 2, 16, seed=3)
    s.table[0, 2:9], s.table[1, 1], s.table[2, :5] = -1, 1 << 30, s.cache.n_pages
    s.table[3, :] = -1
    s.table[1, 11:12] = -2147483648
    q = s.rows(s.n, 4)
    out = s.cache.attend(q, *s.plan())
    check_attend(s, q, out)
    assert bool((out[-2:] == 0).all())
    s.kv = np.array([300 + 5000, 200, 170, 64])
    check_attend(s, q, s.cache.attend(q, *s.plan()))
    check_attend(s, q, s.cache.attend(q, *s.plan(), window=100, sinks=20), window=100, sinks=20)


def test_attend_far_offsets(pkg, ctx):
    """Pages past 4 GiB into the pool."""
    page, heads, dim = 256, 8, 128
    n_pages = (1 << 32) // (page * heads * dim * 2) + 300
    k, v = (torch.empty((n_pages, heads, page, dim), dtype=F16, device="cuda") for _ in range(2))
    s = Setup(pkg, ctx, [(300, 2), (600, 1)], F16, None, dim, heads, page, seed=1)
    far = pkg.PagedKvCache(ctx, k, v)
    table = np.where(s.table >= 0, n_pages - 1 - 37 * s.table, -1)
    new_k, new_v = s.rows(903, heads), s.rows(903, heads)
    lens = i32([300, 600])
    far.append(new_k[:900], new_v[:900], i32([0, 300, 900]), lens, i32(table))
    near = s.cache
    near.append(new_k[:900], new_v[:900], i32([0, 300, 900]), lens, i32(s.table))
    q = s.rows(s.n, heads)
    out = far.attend(q, i32(s.cu), lens, i32(table))
    check_attend(s, q, out)
    assert torch.equal(out, near.attend(q, *s.plan()))
    a, b = far.read(lens, i32(table), 600), near.read(lens, i32(s.table), 600)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("store", [None, E4M3], ids=["16", "e4m3"])
@pytest.mark.parametrize("rows", [(3, 1), (40, 3), (320, 4)], ids=["tokens", "chunk", "tiles of 128"])
def test_far_rows_and_far_pages(pkg, ctx, rows, store):
    """Rows of every operand 32 MiB apart (past 4 GiB with 320 of them), in pages past 4 GiB into each pool: as near ones."""
    new, group = rows
    page, heads, dim, kv = 256, 8, 128, 600
    assert new < 300 or repeats([(kv, new)], heads, group, bool(store), 256) == 1
    n_pages = (1 << 32) // (page * heads * dim * (1 if store else 2)) + 300
    s = Setup(pkg, ctx, [(kv, new), (300, 1)], BF16, store, dim, heads, page, seed=new)
    far = pkg.PagedKvCache.allocate(ctx, n_pages, page, heads, dim, store or BF16)
    table = np.where(s.table >= 0, n_pages - 1 - 37 * s.table, -1)
    for name in ("k", "v") + (("k_exp", "v_exp") if store else ()):
        a, b = getattr(far, name).view(torch.uint8), getattr(s.cache, name).view(torch.uint8)
        for x, y in zip(table.reshape(-1), s.table.reshape(-1)):
            if y >= 0:
                a[int(x)] = b[int(y)]
    wide = torch.zeros(s.n << 24, dtype=BF16, device="cuda").view(s.n, 1 << 24)
    cu, lens, near_table = s.plan()

    def apart(n_heads, place):
        return wide[:, place << 16:(place << 16) + n_heads * dim].view(s.n, n_heads, dim)

    q, k, v, out = apart(heads * group, 0), apart(heads, 1), apart(heads, 2), apart(heads * group, 3)
    for t in (q, k, v):
        t.copy_(s.rows(s.n, t.shape[1]))
    far.append(k, v, cu, lens, i32(table))
    s.cache.append(k.contiguous(), v.contiguous(), cu, lens, near_table)
    far.attend(q, cu, lens, i32(table), out=out)
    assert torch.equal(out, s.cache.attend(q.contiguous(), cu, lens, near_table))
    for a, b in zip(far.read(lens, i32(table), kv, dtype=BF16), s.cache.read(lens, near_table, kv, dtype=BF16)):
        assert torch.equal(a, b)
    assert not bool(wide[:, 1 << 18:].any())
    check_attend(s, q, out)


# ---- writing and reading back -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, store, dim", [(F16, None, 64), (BF16, None, 128), (F16, E4M3, 128), (BF16, E4M3, 64)],
                         ids=["f16", "bf16", "f16-e4m3", "bf16-e4m3"])
@pytest.mark.parametrize("heads", [1, 3, 8])
@pytest.mark.parametrize("lens", [[(1, 1)], [(77, 1), (16, 1), (17, 1), (200, 1)], [(90, 90), (33, 5), (0, 0), (64, 64), (3, 7)]])
def test_append_writes_its_rows_and_nothing_else(pkg, ctx, lens, heads, dtype, store, dim):
    s = Setup(pkg, ctx, lens, dtype, store, dim, heads, 16, seed=heads)
    names = ("k", "v") if store is None else ("k", "v", "k_exp", "v_exp")
    raw = {n: getattr(s.cache, n).view(torch.uint8).cpu().numpy().copy() if store else getattr(s.cache, n).cpu().clone() for n in names}
    qkv = s.rows(s.n + 1, 2 + 2 * heads, 3.0)
    # rows of very different size, zeros, and what a conversion has to survive
    qkv *= torch.exp2(torch.randint(-14, 6, qkv.shape[:2], generator=s.g, device="cuda").float())[..., None].to(dtype)
    qkv[0, 2] = 0
    qkv[0, 2 + heads, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")], device="cuda").to(dtype)
    new = {"k": qkv[:, 2:2 + heads], "v": qkv[:, 2 + heads:]}
    s.cache.append(new["k"], new["v"], *s.plan())
    for name in ("k", "v"):
        x = new[name].cpu()
        for t, b, p in po.new_positions(s.cu, s.kv):
            page, at = s.table[b, p // 16], p % 16
            if store is None:
                raw[name][page, :, at] = x[t]
            else:
                codes, exps = po.quantise(x[t].double().numpy())
                raw[name][page, :, at], raw[name + "_exp"][page, :, at] = codes, exps
    for name in names:
        got = getattr(s.cache, name)
        if store is None:
            assert torch.equal(got.cpu().view(torch.int16), raw[name].view(torch.int16))
        else:
            got = got.view(torch.uint8).cpu().numpy()
            if name in ("k", "v"):  # (the sign of a NaN is free)
                nan = (raw[name] & 0x7f) == 0x7f
                assert ((got[nan] & 0x7f) == 0x7f).all()
                got, want = got[~nan], raw[name][~nan]
            else:
                want = raw[name]
            np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_code_reads_back_exactly(pkg, ctx, dtype):
    """All 256 codes under scales from the smallest to the largest: exact in bf16; in fp16 rounded to nearest and kept inside
    its range."""
    c = pkg.PagedKvCache.allocate(ctx, 8, 16, 4, 128, E4M3)
    codes = torch.arange(256, dtype=torch.uint8).repeat(8 * 4 * 16 // 2)
    exps = torch.arange(8 * 4 * 16) % 256
    exps[exps == 255] = 120
    for name in ("k", "v"):
        getattr(c, name).view(torch.uint8).copy_(codes.view(8, 4, 16, 128))
        getattr(c, name + "_exp").copy_(exps.to(torch.uint8).view(8, 4, 16))
    k, v = c.read(i32([128]), i32([list(range(8))]), 128, dtype=dtype)
    want = po.dequantise(c.k.view(torch.uint8).cpu().numpy(), c.k_exp.cpu().numpy())
    want = torch.from_numpy(want).permute(0, 2, 1, 3).reshape(1, 128, 4, 128)
    fine = torch.isfinite(want)
    # (2^-127 and its multiples below 2^-126 are subnormal in fp32 and bf16: they may be flushed)
    fine &= (want.abs() >= 2.0 ** -126) | (want == 0)
    w = want.float() if dtype == BF16 else want.float().clamp(-65504, 65504)
    big = want.abs() > 3e38  # past bf16's and fp32's own range: not a value any row of theirs is stored as
    fine &= ~big
    for got in (k, v):
        assert torch.equal(got.cpu()[fine], w.to(dtype)[fine])
        assert bool(torch.isnan(got.cpu()[torch.isnan(want)]).all())


def test_read_lengths_pages_and_types(pkg, ctx):
    for store in (None, E4M3):
        s = Setup(pkg, ctx, [(50, 1), (0, 0), (33, 1), (200, 1)], BF16, store, 64, 3, 32, seed=2)
        s.table[3, 1], s.table[3, 3] = -1, s.cache.n_pages + 5
        for t_max in (1, 33, 230):
            k, v = s.cache.read(i32(s.kv), i32(s.table), t_max, dtype=BF16)
            for got, name in ((k, "k"), (v, "v")):
                for b in range(4):
                    want, _ = po.dense(values_of(s.cache, name), s.table, 32, b, min(t_max, int(s.kv[b])))
                    assert np.array_equal(got[b, :len(want)].double().cpu().numpy(), want)
                    assert not bool(got[b, len(want):].any())
    k, v = s.cache.read(i32([]), torch.empty(0, 2, dtype=torch.int32, device="cuda"), 5)
    assert k.shape == (0, 5, 3, 64)


@pytest.mark.parametrize("store", [None, E4M3], ids=["16", "e4m3"])
@pytest.mark.parametrize("heads, dim", [(1, 64), (2, 64), (3, 64), (5, 64), (1, 128), (2, 128), (3, 128)])
def test_few_heads_share_a_wave(pkg, ctx, heads, dim, store):
    """Neighbouring positions of a wave may belong to several sequences, have other pages, or none."""
    lens = [(5, 1), (1, 1), (0, 0), (40, 2), (17, 1), (2, 2), (3, 1), (33, 1), (16, 1), (9, 1), (1, 1), (20, 3), (64, 1)]
    s = Setup(pkg, ctx, lens, F16, store, dim, heads, 16, seed=heads)
    s.table[6, 0] = -1
    for t_max in (1, 2, 3, 21):
        got = s.cache.read(i32(s.kv), i32(s.table), t_max)
        for name, t in zip("kv", got):
            want = np.zeros((len(lens), t_max, heads, dim))
            x = values_of(s.cache, name)
            for b in range(len(lens)):
                for j in range(min(t_max, int(s.kv[b]))):
                    if s.table[b, j // 16] >= 0:
                        want[b, j] = x[s.table[b, j // 16], :, j % 16]
            np.testing.assert_array_equal(t.double().cpu().numpy(), want)
    k, v = s.rows(s.n + 9, heads), s.rows(s.n + 9, heads)
    before = values_of(s.cache, "k"), values_of(s.cache, "v")
    s.cache.append(k, v, *s.plan())
    for x, new, name in ((before[0], k, "k"), (before[1], v, "v")):
        new = new.double().cpu().numpy()
        for b in range(len(lens)):
            for i in range(int(s.nq[b])):
                j = int(s.kv[b] - s.nq[b]) + i
                if s.table[b, j // 16] >= 0:
                    row = new[s.cu[b] + i]
                    if store:
                        row = po.dequantise(*po.quantise(row))
                    x[s.table[b, j // 16], :, j % 16] = row
        np.testing.assert_array_equal(values_of(s.cache, name), x)


@pytest.mark.parametrize("store", [None, E4M3], ids=["16", "e4m3"])
@pytest.mark.parametrize("heads", [1, 8])
def test_thousands_of_sequences(pkg, ctx, heads, store):
    """The search for a row's sequence takes three steps; many sequences have no new rows, the first and the last among them."""
    rng = np.random.default_rng(heads)
    batch = 9001 if heads == 1 else 4500
    kv = rng.integers(0, 34, batch)
    q = np.minimum(kv, rng.choice([0, 0, 1, 2, 7], batch))
    q[:70] = q[-70:] = 0
    s = Setup(pkg, ctx, list(zip(kv.tolist(), q.tolist())), F16, store, 64, heads, 16, seed=heads)
    k, v = s.rows(s.n + 3, heads), s.rows(s.n + 3, heads)
    want = [values_of(s.cache, x) for x in "kv"]
    s.cache.append(k, v, *s.plan())
    for x, new in zip(want, (k, v)):
        new = new.double().cpu().numpy()
        new = po.dequantise(*po.quantise(new)) if store else new
        for t, b, p in po.new_positions(s.cu, s.kv):
            x[s.table[b, p // 16], :, p % 16] = new[t]
    for x, name in zip(want, "kv"):
        np.testing.assert_array_equal(values_of(s.cache, name), x)
    queries = s.rows(s.n + 3, 2 * heads)
    out = torch.full_like(queries, 7.0)
    s.cache.attend(queries, *s.plan(), out=out)
    check_attend(s, queries, out, untouched=7.0)
    got = s.cache.read(i32(s.kv), i32(s.table), 3)
    for x, t in zip(want, got):
        dense = np.stack([po.dense(x, s.table, 16, b, 3)[0] * (np.arange(3) < s.kv[b])[:, None, None] for b in range(batch)])
        np.testing.assert_array_equal(t.double().cpu().numpy(), dense)


def test_append_of_bad_pages_writes_nothing(pkg, ctx):
    s = Setup(pkg, ctx, [(40, 40), (20, 20)], F16, None, 64, 2, 16, seed=4)
    s.table[0, 1], s.table[1, 0] = -1, 1 << 29
    before = s.cache.k.clone()
    x = s.rows(s.n, 2)
    s.kv[1] = 20 + 16 * 7  # its last rows lie past the table
    s.cache.append(x, x, *s.plan())
    want = before.clone()
    for t, b, p in po.new_positions(s.cu, s.kv):
        page = po.page_at(s.table, s.cache.n_pages, 16, b, p)
        if page >= 0:
            want[page, :, p % 16] = x[t]
    assert torch.equal(s.cache.k, want)


# ---- as a program uses them -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("store", [None, E4M3], ids=["16", "e4m3"])
def test_steps_of_a_decoder(pkg, ctx, store):
    """A prompt and then single tokens: append, attend, project, sample; every step's attention is held against the oracle on
    what the cache holds, and the chosen ids against the oracle on the step's logits."""
    torch.manual_seed(0)
    heads, group, dim, page, vocab = 2, 2, 64, 16, 301
    s = Setup(pkg, ctx, [(35, 35), (9, 9), (20, 20)], F16, store, dim, heads, page, seed=6, spare=40)
    pages = list(s.free)
    s.table = np.concatenate([s.table, np.full((3, 3), -1)], axis=1)
    w = torch.randn(heads * group * dim, vocab, device="cuda") * 0.1
    emb = torch.randn(vocab, (heads * group + 2 * heads) * dim, device="cuda")
    ids = torch.randint(vocab, (s.n,), device="cuda")
    for step in range(6):
        qkv = emb[ids.long()].view(len(ids), -1, dim).to(F16)
        q, k, v = qkv[:, :heads * group], qkv[:, heads * group:heads * (group + 1)], qkv[:, heads * (group + 1):]
        s.cache.append(k, v, *s.plan())
        out = s.cache.attend(q, *s.plan(), window=24, sinks=2)
        check_attend(s, q, out, window=24, sinks=2)
        last = out[torch.from_numpy(s.cu[1:] - 1).cuda()].float().reshape(3, -1)
        logits = last @ w
        u = torch.rand(3, device="cuda")
        ids, lp = pkg.sample_tokens(ctx, logits, u, temperature=0.8, top_k=40, top_p=0.95)
        for r in range(3):
            want, wlp, _ = po.sample_row(logits[r].double().cpu().numpy(), float(u[r]), float(np.float32(0.8)), 40, float(np.float32(0.95)))
            assert int(ids[r]) == want and abs(float(lp[r]) - wlp) <= 1e-5 * max(1.0, abs(wlp))
        s.kv = s.kv + 1
        s.nq = np.ones(3, dtype=np.int64)
        s.cu, s.n = np.arange(4), 3
        for b in range(3):
            if s.table[b, (s.kv[b] - 1) // page] < 0:
                s.table[b, (s.kv[b] - 1) // page] = pages.pop()


def test_attend_and_append_on_another_stream_and_in_graphs(pkg, ctx):
    """Two captured graphs of different sizes over one cache, replayed in turn with eager calls between, and calls on two
    streams at once: every result equals the eager one, bit for bit."""
    s = Setup(pkg, ctx, [(5000, 1), (3000, 1)], F16, None, 128, 2, 64, seed=8)
    t = Setup(pkg, ctx, [(700, 1)] * 8, F16, None, 128, 2, 64, seed=9)
    plans = [x.plan() for x in (s, t)]
    qs = [x.rows(x.n, 8) for x in (s, t)]
    new = [x.rows(x.n, 2) for x in (s, t)]

    def step(i):
        (s, t)[i].cache.append(new[i], new[i], *plans[i])
        return (s, t)[i].cache.attend(qs[i], *plans[i], window=0)

    want = [step(0).clone(), step(1).clone()]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for i in range(2):
            step(i)
    side.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for r in range(4):
        for i in (0, 1, 1, 0):
            outs[i].zero_()
            graphs[i].replay()
            eager = step(1 - i)
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i]) and torch.equal(eager, want[1 - i])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for r in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("store", [None, E4M3], ids=["16", "e4m3"])
@pytest.mark.parametrize("kw", [{}, dict(window=100, sinks=5), dict(causal=False)], ids=["plain", "window", "whole"])
@pytest.mark.parametrize("n, heads, group, width", [(4, 2, 4, 200), (60, 2, 1, 60), (300, 8, 4, 90), (200, 1, 2, 500)],
                         ids=["tokens", "chunks", "prompts", "prompts in parts"])
def test_a_captured_step_follows_its_buffers(pkg, ctx, n, heads, group, width, kw, store):
    """One graph of append, attend and read back, replayed while the batch in its buffers changes: other lengths, other shares of the rows, empty
    sequences, rows that belong to nobody, pages given back.  Every replay equals an eager call on the same buffers, and the
    definition."""
    s = Setup(pkg, ctx, [(16 * width, n // 4)] * 4, F16, store, 64, heads, 16, seed=n)
    c, (cu, lens, table) = s.cache, s.plan()
    full = s.table.copy()
    q, k, v = s.rows(n, heads * group), s.rows(n, heads), s.rows(n, heads)
    out = torch.zeros_like(q)

    def step():
        c.append(k, v, cu, lens, table)
        c.attend(q, cu, lens, table, out=out, **kw)
        return c.read(lens, table, 40)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    rng = np.random.default_rng(n)
    for r in range(5):
        last = n - (0, 3)[r % 2]
        s.cu = np.minimum([0, *np.sort(rng.integers(0, n + 1, 3)), last], last) if r else np.array([0, 0, n // 2, n // 2, n])
        s.nq = np.diff(s.cu)
        s.kv = rng.integers(0, 16 * width + 1, 4)
        s.kv[r % 4] = s.nq[r % 4]
        s.n = int(s.cu[-1])
        s.table = np.where(rng.random(full.shape) < (0.1 if r == 3 else 0.0), -1, full)
        for t, x in ((cu, s.cu), (lens, s.kv), (table, s.table)):
            t.copy_(i32(x))
        for t in (q, k, v):
            t.copy_(s.rows(n, t.shape[1]))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, pages = out.clone(), [t.clone() for t in held]
        out.fill_(7.0)
        eager = step()
        assert torch.equal(got, out) and all(torch.equal(a, b) for a, b in zip(pages, eager))
        assert bool((got[s.n:] == 7).all())
        check_attend(s, q[:s.n], got[:s.n], **kw)


def test_python_refusals(pkg, ctx):
    s = Setup(pkg, ctx, [(20, 2)], F16, None, 64, 2, 16)
    c, (cu, lens, table), q = s.cache, s.plan(), s.rows(2, 4)
    k = s.rows(2, 2)
    bad = [
        lambda: c.attend(q.float(), cu, lens, table), lambda: c.attend(q.to(BF16), cu, lens, table), lambda: c.attend(q[:, :3], cu, lens, table),
        lambda: c.attend(q[:, :0], cu, lens, table), lambda: c.attend(q.cpu(), cu, lens, table), lambda: c.attend(q, cu.long(), lens, table),
        lambda: c.attend(q, cu[:1], lens, table), lambda: c.attend(q, cu, lens, table[0]), lambda: c.attend(q, cu, lens, table, window=-1),
        lambda: c.attend(q, cu, lens, table, sinks=-1), lambda: c.attend(q, cu, lens, table, out=q[:1]),
        lambda: c.attend(q.transpose(1, 2).contiguous().transpose(1, 2), cu, lens, table), lambda: c.attend(q[..., :32], cu, lens, table),
        lambda: c.attend(s.rows(2, 9).view(-1)[4:4 + 512].view(2, 4, 64), cu, lens, table),
        lambda: c.append(k, k[:1], cu, lens, table), lambda: c.append(q, q, cu, lens, table), lambda: c.append(k, k.to(BF16), cu, lens, table),
        lambda: c.append(k, k, cu, lens.cpu(), table), lambda: c.read(lens, table, 4, dtype=BF16), lambda: c.read(lens, table, 4, dtype=torch.float32),
        lambda: pkg.PagedKvCache(ctx, c.k.transpose(0, 1), c.v.transpose(0, 1)),
    ]
    for call in bad:
        with pytest.raises(ValueError, match="PagedKvCache"):
            call()
    for kw in (dict(scale=float("nan")), dict(scale=float("inf")), dict(max_kv=-1)):
        with pytest.raises((ValueError, pkg.AsrfeError)):
            c.attend(q, cu, lens, table, **kw)
    assert c.attend(q[:0], cu, lens, table).shape == (0, 4, 64)


def test_numbers_past_32_bits_and_overlapping_results(pkg, ctx):
    s = Setup(pkg, ctx, [(40, 3), (25, 1)], F16, None, 64, 2, 16)
    c, (cu, lens, table), q = s.cache, s.plan(), s.rows(4, 4)
    want = c.attend(q, cu, lens, table)
    assert torch.equal(c.attend(q, cu, lens, table, max_kv=(1 << 32) + 8), want)
    assert torch.equal(c.attend(q, cu, lens, table, window=1 << 32), want)
    assert torch.equal(c.attend(q, cu, lens, table, window=5, sinks=(1 << 32) + 1), want)  # every position is a sink
    buf = torch.zeros(4, 4, 64, dtype=F16, device="cuda")
    for out in (buf[:1].expand(4, 4, 64), buf[:, :1].expand(4, 4, 64), buf.view(-1).as_strided((4, 4, 64), (256, 32, 1))):
        with pytest.raises(ValueError, match="overlap"):
            c.attend(q, cu, lens, table, out=out)


def test_more_threads_than_a_launch_holds_are_refused(pkg, ctx):
    """65535 sequences on 256 heads of keys are more row tiles than one launch takes (the queries repeat one row: no memory)."""
    n, heads = 65535, 256
    cache = pkg.PagedKvCache.allocate(ctx, 1, 16, heads, 64)
    q = torch.zeros(1, 1, 64, dtype=F16, device="cuda").expand(n, heads, 64)
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    lens, table = torch.ones(n, dtype=torch.int32, device="cuda"), torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(pkg.AsrfeError, match="too many"):
        cache.attend(q, cu, lens, table)
