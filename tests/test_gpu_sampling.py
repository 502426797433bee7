"""The choice of a token on the device against its definition in 64 bits (oracle/paged_oracle.py)."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    import toolbox_for_asr_and_tts_amd as p

    p.load()
    return p


@pytest.fixture(scope="module")
def ctx(pkg):
    return pkg.Context()


def check(pkg, ctx, logits, u, border=1e-8, **settings):
    """Every row's id equals the definition's unless the number lies within `border` of the edge between two ids (sums and
    weights are held to errors below 1e-9); the log-probability is fp32: half a step of its value, and the weights'
    1e-9."""
    ids, lp = pkg.sample_tokens(ctx, logits, u, **settings)
    again, lp2 = pkg.sample_tokens(ctx, logits, u, **settings)
    assert torch.equal(ids, again) and torch.equal(lp.nan_to_num(1.0), lp2.nan_to_num(1.0))
    x, uu = logits.double().cpu().numpy(), u.double().cpu().numpy()
    ids, lp = ids.cpu().numpy(), lp.double().cpu().numpy()

    def of(name, r):
        v = settings.get(name)
        d = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)[name]
        if v is None:
            return d
        return v[r].item() if isinstance(v, torch.Tensor) else (int(v) if name == "top_k" else float(np.float32(v)))

    skipped = 0
    for r in range(x.shape[0]):
        want, wlp, dist = po.sample_row(x[r], uu[r], of("temperature", r), of("top_k", r), of("top_p", r), of("min_p", r))
        if dist < border and 0 < uu[r] < 1:
            skipped += 1
            continue
        assert ids[r] == want, (r, ids[r], want, dist)
        assert lp[r] == wlp or abs(lp[r] - wlp) <= 2.0 ** -24 * abs(wlp) + 2e-9, (r, lp[r], wlp)
    assert skipped <= max(1, x.shape[0] // 50)


def make(rows, vocab, dtype, seed, pad=0, sharp=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rank = torch.rand(rows, vocab + pad, generator=g, device="cuda") * vocab
    x = 6 - sharp * torch.log1p(rank) + 0.3 * torch.randn(rank.shape, generator=g, device="cuda")
    return x.to(dtype)[:, :vocab], torch.rand(rows, generator=g, device="cuda")


SETTINGS = {
    "plain": {}, "cold": dict(temperature=0.1), "hot": dict(temperature=30.0), "greedy": dict(temperature=0.0), "top_k": dict(top_k=17),
    "top_k 1": dict(top_k=1), "top_k past the vocabulary": dict(top_k=1 << 30), "top_p": dict(top_p=0.7), "top_p tiny": dict(top_p=1e-6),
    "top_p zero": dict(top_p=0.0), "top_p near one": dict(top_p=0.9999), "min_p": dict(min_p=0.03), "min_p one": dict(min_p=1.0), "min_p above one": dict(min_p=2.0),
    "all": dict(temperature=0.7, top_k=50, top_p=0.9, min_p=0.01), "hot and all": dict(temperature=4.0, top_k=400, top_p=0.95, min_p=1e-4),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", SETTINGS)
def test_settings(pkg, ctx, name, dtype):
    x, u = make(24, 8404, dtype, seed=len(name), pad=44)
    check(pkg, ctx, x, u, **SETTINGS[name])


@pytest.mark.parametrize("vocab, pad", [(1, 0), (2, 0), (3, 1), (63, 0), (64, 0), (65, 7), (1000, 0), (1023, 1), (1025, 0), (4097, 3), (32000, 0), (50001, 0),
                                        (131072, 0), (262144, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vocabularies_and_strides(pkg, ctx, vocab, pad, dtype):
    rows = 9 if vocab < 40000 else 3
    x, u = make(rows, vocab, dtype, seed=vocab, pad=pad)
    check(pkg, ctx, x, u, top_p=0.95, temperature=1.1)
    check(pkg, ctx, x, u, temperature=1.5)
    check(pkg, ctx, x, u, top_k=40, min_p=0.001)


def test_per_row_settings_and_many_rows(pkg, ctx):
    rows = 700
    x, u = make(rows, 517, torch.float32, seed=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(len(v), (rows,), generator=g, device="cuda")]  # noqa: E731
    check(pkg, ctx, x, u, temperature=pick(0.0, 0.5, 1.0, 2.0, -1.0), top_k=pick(0, 1, 5, 100, -3).int(), top_p=pick(0.1, 0.5, 0.9, 1.0, 1.5),
          min_p=pick(0.0, 0.01, 0.2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_index(pkg, ctx, dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(0, 4, (40, 3001), generator=g, device="cuda").to(dtype)  # few values, many of each
    u = torch.rand(40, generator=g, device="cuda")
    for settings in (dict(top_k=5), dict(top_k=900), dict(top_p=0.3), dict(top_p=0.6, top_k=1200), dict(min_p=0.1), dict(temperature=0.0),
                     dict(temperature=2.0, top_p=0.999)):
        check(pkg, ctx, x, u, **settings)
    flat = torch.zeros(4, 2048, dtype=dtype, device="cuda")
    ends = torch.tensor([0.0, 0.25, 0.5, 1 - 2.0 ** -24], device="cuda")
    ids, lp = pkg.sample_tokens(ctx, flat, ends)
    assert ids.tolist() == [0, 512, 1024, 2047] and torch.allclose(lp, torch.full_like(lp, -np.log(2048.0)), rtol=1e-6)
    ids, _ = pkg.sample_tokens(ctx, flat, ends, top_k=8)
    assert ids.tolist() == [0, 2, 4, 7]
    ids, _ = pkg.sample_tokens(ctx, -flat, ends, top_p=0.5)  # (-0 and +0 are equal)
    assert ids.tolist() == [0, 256, 512, 1023]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ties", [3, 300, 3000])
def test_min_p_above_one_keeps_the_first_alone(pkg, ctx, dtype, ties):
    g = torch.Generator(device="cuda").manual_seed(ties)
    x = torch.randn(6, 3000, generator=g, device="cuda").clamp(max=2.0).to(dtype)
    at = torch.rand(x.shape, generator=g, device="cuda").argsort(1)[:, :ties]
    x.scatter_(1, at, torch.full(at.shape, 3.0, device="cuda", dtype=dtype))
    u = torch.rand(6, generator=g, device="cuda") * 0.5 + 0.5
    for settings in ({}, dict(top_k=2), dict(top_k=300), dict(top_k=2500), dict(top_p=0.05), dict(top_p=0.9), dict(top_k=1000, top_p=0.5)):
        check(pkg, ctx, x, u, min_p=2.0, **settings)
        ids, lp = pkg.sample_tokens(ctx, x, u, min_p=2.0, **settings)
        assert torch.equal(ids.long(), at.min(1).values) and not bool(lp.any())


def test_rows_with_infinities_and_nan(pkg, ctx):
    inf, nan = float("inf"), float("nan")
    x, u = make(12, 700, torch.float32, seed=5)
    x[0] = -inf
    x[1] = nan
    x[2, :600] = -inf
    x[3, ::2] = nan
    x[4, 77] = x[4, 400] = inf
    x[5] = -inf
    x[5, 699] = -3e38
    x[6] = 3.4e38
    x[7, 5] = nan
    x[8] = torch.finfo(torch.float32).min
    x[9, 1:] = torch.finfo(torch.float32).min
    for settings in ({}, dict(top_k=3), dict(top_p=0.5), dict(min_p=0.5), dict(temperature=0.0), dict(top_k=650, top_p=0.99, min_p=1e-9)):
        check(pkg, ctx, x, u, **settings)
    ids, lp = pkg.sample_tokens(ctx, x[:2], u[:2])
    assert ids.tolist() == [0, 0] and lp.tolist() == [-inf, -inf]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("left", [1, 3, 300, 2500])
def test_rows_that_a_mask_leaves_little_of(pkg, ctx, dtype, left):
    x, u = make(12, 40000, dtype, seed=left)
    g = torch.Generator(device="cuda").manual_seed(left)
    keep = torch.rand(x.shape, generator=g, device="cuda").argsort(1) < left
    low = torch.tensor([-float("inf"), torch.finfo(dtype).min, -60000.0], device="cuda").to(dtype).repeat(4)
    x = torch.where(keep, x, low[:, None])
    for settings in (dict(top_k=50), dict(top_k=200, top_p=0.9), dict(top_k=1000), dict(top_p=0.8), dict(min_p=0.05), dict(top_k=7, temperature=1e5), {}):
        check(pkg, ctx, x, u, **settings)


@pytest.mark.parametrize("rows, vocab", [(300, 9001), (770, 33001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_many_rows(pkg, ctx, rows, vocab, dtype):
    x, u = make(rows, vocab, dtype, seed=vocab, pad=5)
    g = torch.Generator(device="cuda").manual_seed(7)
    pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(len(v), (rows,), generator=g, device="cuda")]  # noqa: E731
    check(pkg, ctx, x, u, temperature=pick(0.0, 0.7, 1.0, 1.6), top_k=pick(0, 0, 20, 200, 700).int(), top_p=pick(0.3, 0.9, 0.97, 1.0),
          min_p=pick(0.0, 0.0, 0.02, 0.2))


def test_rows_far_apart(pkg, ctx):
    """Rows a gigabyte apart, the last ones past 8 GiB, give what they give side by side."""
    x, u = make(10, 9001, torch.float32, seed=21)
    far = torch.zeros(10 << 28, device="cuda").view(10, 1 << 28)[:, 3:9004]
    far.copy_(x)
    for settings in (dict(top_k=40, top_p=0.9), dict(top_p=0.97), dict(temperature=0.0), dict(min_p=0.01)):
        check(pkg, ctx, far, u, **settings)
        for a, b in zip(pkg.sample_tokens(ctx, far, u, **settings), pkg.sample_tokens(ctx, x, u, **settings)):
            assert torch.equal(a, b)


def test_numbers_at_the_ends(pkg, ctx):
    """u = 0 takes the first kept token; a number outside [0, 1), which no generator gives, takes an end instead of running on."""
    x, _ = make(5, 900, torch.float32, seed=8)
    for settings in ({}, dict(top_k=9), dict(top_p=0.5)):
        first, _ = pkg.sample_tokens(ctx, x, torch.zeros(5, device="cuda"), **settings)
        last, _ = pkg.sample_tokens(ctx, x, torch.full((5,), 1 - 2.0 ** -24, device="cuda"), **settings)
        for v, want in ((-1.0, first), (float("nan"), first), (1.0, None), (5.0, None), (float("inf"), None)):
            got, lp = pkg.sample_tokens(ctx, x, torch.full((5,), v, device="cuda"), **settings)
            assert bool(((got >= 0) & (got < 900)).all()) and bool(torch.isfinite(lp).all())
            assert torch.equal(got, want) if want is not None else bool((got >= last).all())


def test_temperatures_that_are_no_numbers_or_have_no_end(pkg, ctx):
    x, _ = make(4, 3000, torch.float32, seed=17)
    u = torch.tensor([0.9, 0.9, 0.9, 0.25], device="cuda")
    t = torch.tensor([float("nan"), -1.0, 0.0, float("inf")], device="cuda")
    ids, lp = pkg.sample_tokens(ctx, x, u, temperature=t)
    assert ids[:3].tolist() == x[:3].argmax(1).tolist() and lp[:3].tolist() == [0.0, 0.0, 0.0]
    assert int(ids[3]) == 750 and abs(float(lp[3]) + np.log(3000.0)) < 1e-6  # all weights are one: the 751st sum is the first above 750


@pytest.mark.parametrize("vocab", [1000, 1 << 18])
def test_many_weights_below_the_last_place_of_the_sum(pkg, ctx, vocab):
    """Weights of 2^-45.2 round to zero, of 2^-44.4 to 2^-44: the sums are off by n 2^-45 at most, and so is the share."""
    for nats in (31.32, 30.78):
        x = torch.full((2, vocab), -nats, device="cuda")
        x[:, vocab // 2] = 0.0
        ids, lp = pkg.sample_tokens(ctx, x, torch.full((2,), 0.5, device="cuda"))
        want = -np.log1p((vocab - 1) * np.exp(float(x[0, 0])))
        assert ids.tolist() == [vocab // 2] * 2
        assert (np.abs(lp.double().cpu().numpy() - want) <= vocab * 2.0 ** -45 + 1e-11).all()


def test_temperatures_past_the_largest(pkg, ctx):
    """They count as 1e30: what a mask of the type's lowest value hides stays hidden in 32 bits."""
    x, u = make(6, 2000, torch.float32, seed=3)
    x[:, ::3] = torch.finfo(torch.float32).min
    t = torch.tensor([1e30, 2e30, 1e36, 3e38, float("inf"), 1e29], device="cuda")
    ids, lp = pkg.sample_tokens(ctx, x, u, temperature=t)
    kept = torch.arange(2000, device="cuda")[torch.arange(2000, device="cuda") % 3 != 0]
    assert torch.equal(ids.long(), kept[(u.double() * len(kept)).long()])
    assert torch.allclose(lp, torch.full_like(lp, -np.log(len(kept))), rtol=1e-6)


@pytest.mark.parametrize("dtype, rows", [(torch.float32, 9), (torch.float16, 9), (torch.bfloat16, 9), (torch.float16, 300), (torch.bfloat16, 300)])
def test_a_cut_just_below_zero(pkg, ctx, dtype, rows):
    """Zeros of both signs above the cut, the least negative values at and below it: bins of keys that end right below zero
    hold no zeros.  (The maxima differ by row, so that bins end at every distance from zero; the first one's keys end
    there in 32 bits, too.)"""
    vocab, g = 3000, torch.Generator(device="cuda").manual_seed(3)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the least subnormal
    x = torch.full((rows, vocab), -1.0, device="cuda", dtype=torch.float64)
    x[:, 100:300] = 0.0
    x[:, 200:300] *= -1
    x[:, 300:1000] = -tiny * torch.randint(1, 64 if dtype is not torch.float32 else 1 << 22, (rows, 700), generator=g, device="cuda")
    x = x.to(dtype)
    bits = torch.int32 if dtype is torch.float32 else torch.int16
    top = {torch.float32: 0x3fffffff, torch.float16: 0x3fff, torch.bfloat16: 0x3fff}[dtype]
    x[:, 0] = (top - torch.arange(rows, device="cuda")).to(bits).view(dtype)
    x = x[:, torch.randperm(vocab, generator=g, device="cuda")].contiguous()
    u = torch.rand(rows, generator=g, device="cuda")
    for settings in (dict(top_k=650), dict(top_p=0.2), dict(top_k=2000, top_p=0.3)):
        for temperature in (1.0, 100.0):
            check(pkg, ctx, x, u, temperature=temperature, **settings)


def test_rows_behind_an_utterances_tokens(pkg, ctx):
    x, u = make(15, 300, torch.float16, seed=4)
    num = torch.tensor([5, 0, 3], dtype=torch.int32, device="cuda")
    ids, lp = pkg.sample_tokens(ctx, x, u, top_k=10, token_num=num)
    free, flp = pkg.sample_tokens(ctx, x, u, top_k=10)
    keep = torch.arange(5, device="cuda").repeat(3) < num.repeat_interleave(5)
    assert torch.equal(ids, torch.where(keep, free, -1)) and torch.equal(lp, torch.where(keep, flp, 0.0))


def test_a_captured_call_and_another_stream(pkg, ctx):
    x, u = make(30, 20000, torch.bfloat16, seed=6)
    kw = dict(temperature=torch.full((30,), 0.9, device="cuda"), top_p=torch.full((30,), 0.9, device="cuda"))
    want = pkg.sample_tokens(ctx, x, u, **kw)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = pkg.sample_tokens(ctx, x, u, **kw)
    side.synchronize()
    assert torch.equal(got[0], want[0])
    with torch.cuda.graph(g):
        got = pkg.sample_tokens(ctx, x, u, **kw)
    for i in range(4):
        u.copy_(torch.rand(30, device="cuda"))
        want = pkg.sample_tokens(ctx, x, u, **kw)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_recogniser_draws_its_tokens(pkg):
    """ParaformerHead with sampling: ids drawn from its own logits row by row; the arg-max again with temperature 0."""
    from oracle import paraformer_decoder_oracle as do
    from oracle import sanm_oracle as so

    cfg = do.DecoderConfig(num_blocks=2, vocab_size=500)
    head = pkg.ParaformerHead(pkg.Context(), num_blocks=2, vocab_size=500)
    head.load_state_dict(do.make_state_dict(cfg, seed=1))
    enc = so.synth_feats(2, 40, 512, seed=3).cuda().float().contiguous()
    lens = torch.tensor([40, 25], dtype=torch.int32)
    n_max = 41
    plain = head.forward(enc, lens, return_logits=True)
    u = torch.rand(2, n_max, device="cuda")
    got = head.forward(enc, lens, return_logits=True, sampling=dict(u=u, temperature=0.0))
    assert torch.equal(got["token_ids"], plain["token_ids"]) and torch.equal(got["token_num"], plain["token_num"])
    got = head.forward(enc, lens, return_logits=True, sampling=dict(u=u, temperature=1.2, top_k=20, top_p=0.9))
    assert "logits" not in head.forward(enc, lens, sampling=dict(u=u)) and "logprobs" not in plain
    for b in range(2):
        for i in range(n_max):
            if i >= int(plain["token_num"][b]):
                assert int(got["token_ids"][b, i]) == -1 and float(got["logprobs"][b, i]) == 0.0
                continue
            want, lp, dist = po.sample_row(got["logits"][b, i].double().cpu().numpy(), float(u[b, i]), float(np.float32(1.2)), 20, float(np.float32(0.9)))
            assert dist < 1e-8 or int(got["token_ids"][b, i]) == want
    with pytest.raises(ValueError, match="sampling"):
        head.forward(enc, lens, sampling=dict(u=u[:1]))
    with pytest.raises(ValueError, match="sampling"):
        head.forward(enc, lens, sampling=dict(u=u, beam=3))


def test_python_refusals(pkg, ctx):
    x, u = make(4, 50, torch.float32, seed=1)
    for call in (lambda: pkg.sample_tokens(ctx, x.double(), u), lambda: pkg.sample_tokens(ctx, x[0], u), lambda: pkg.sample_tokens(ctx, x, u[:3]),
                 lambda: pkg.sample_tokens(ctx, x, u.double()), lambda: pkg.sample_tokens(ctx, x.t(), torch.rand(50, device="cuda")),
                 lambda: pkg.sample_tokens(ctx, x[:1].expand(4, 50), u), lambda: pkg.sample_tokens(ctx, x, u, top_k=torch.ones(4, device="cuda")),
                 lambda: pkg.sample_tokens(ctx, x, u, top_p=torch.ones(3, device="cuda")), lambda: pkg.sample_tokens(ctx, x[:, :0], u),
                 lambda: pkg.sample_tokens(ctx, x, u, token_num=torch.ones(3, dtype=torch.int32, device="cuda")),
                 lambda: pkg.sample_tokens(ctx, x, u, ids=torch.zeros(4, device="cuda")), lambda: pkg.sample_tokens(ctx, x, u, min_p=u.cpu())):
        with pytest.raises(ValueError, match="sample_tokens"):
            call()
    ids, lp = pkg.sample_tokens(ctx, x[:0], u[:0])
    assert ids.shape == (0,) and lp.shape == (0,)
