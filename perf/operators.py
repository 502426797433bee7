"""Cases of the streaming decoder operators: what they are given, their plain form in elementary torch operations, and the
calls a program makes of the package for the same work.

Four operators share one set of cases:

* ``append``: the keys and values of new tokens are written into a paged cache, either as they are (16 bit) or as e4m3
  bytes with one power-of-two scale per token and head;
* ``read``: the cache's pages are read back as dense 16-bit keys and values;
* ``attend``: the new tokens of every sequence attend to their sequence's pages (one token per sequence, a chunk of
  frames, or a long prompt), with an optional sliding window, a few first tokens that stay visible (sinks) and, for
  chunks that see themselves whole, without the causal mask;
* ``sample``: a token is chosen per row of logits with temperature, top-k, top-p and min-p from a given random number.

A cache is ``k``, ``v`` [pages, heads, page, dim] and, for e4m3, the biased exponents of the scales ``k_exp``, ``v_exp``
[pages, heads, page]: a stored value is code * 2 ** (exp - 127).  A batch is ``cu_q`` [B + 1] (rows of the packed new
tokens), ``kv_lens`` [B] (positions in the cache, the new tokens among them: they are the last ones) and ``block_table``
[B, n] (page numbers).
"""
import math

import numpy as np
import torch

own = False

DEVICE = torch.device("cuda" if torch.cuda.is_available() else "cpu")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one streaming session asks for its next step: 4 heads of 128 over the 500 frames of a 30 s clip
        dict(name="attend one stream", op="attend", batch=1, q=1, kv=500, spread=0.0, kv_heads=4, group=1, dim=128, page=64,
             dtype="f16", fmt="16", window=0, sinks=0, causal=True),
        # a serving step: every sequence of a mixed batch decodes one token with grouped heads
        dict(name="attend 64 streams", op="attend", batch=64, q=1, kv=8192, spread=0.9, kv_heads=8, group=4, dim=128, page=64,
             dtype="bf16", fmt="16", window=0, sinks=0, causal=True),
        # few sequences with very long caches, held in 8 bits
        dict(name="attend long e4m3", op="attend", batch=8, q=1, kv=131072, spread=0.5, kv_heads=2, group=8, dim=128, page=128,
             dtype="f16", fmt="e4m3", window=0, sinks=0, causal=True),
        # 256 sessions hand in a chunk of 10 frames each; a frame sees its whole chunk and the four chunks before it
        dict(name="attend stream chunks", op="attend", batch=256, q=10, kv=500, spread=0.95, kv_heads=4, group=1, dim=128, page=16,
             dtype="f16", fmt="16", window=50, sinks=0, causal=False),
        # two prompts are worked through in chunks of 2048 tokens, the last chunks against a cache of 16 k
        dict(name="attend prompt chunk", op="attend", batch=2, q=2048, kv=16384, spread=0.3, kv_heads=4, group=4, dim=128, page=64,
             dtype="bf16", fmt="16", window=0, sinks=0, causal=True),
        # prompts under a sliding window of 1024 with four sinks, heads of 64
        dict(name="attend prompt window", op="attend", batch=4, q=4096, kv=6000, spread=0.4, kv_heads=8, group=2, dim=64, page=32,
             dtype="f16", fmt="16", window=1024, sinks=4, causal=True),
        # the step's new token of eight sequences goes into an 8-bit cache
        dict(name="append tokens", op="append", batch=8, q=1, kv=777, spread=0.8, kv_heads=8, dim=128, page=64, dtype="bf16",
             fmt="e4m3"),
        # a batch of prompts goes into an 8-bit cache
        dict(name="append prompts", op="append", batch=8, q=4096, kv=5000, spread=0.6, kv_heads=8, dim=128, page=64, dtype="bf16",
             fmt="e4m3"),
        # a few short sequences are read back from a 16-bit cache
        dict(name="read short", op="read", batch=4, kv=300, spread=0.7, kv_heads=4, dim=64, page=16, dtype="f16", fmt="16"),
        # long sequences are read back from an 8-bit cache
        dict(name="read long", op="read", batch=16, kv=8192, spread=0.5, kv_heads=8, dim=128, page=64, dtype="bf16", fmt="e4m3"),
        # one row of the recogniser's vocabulary
        dict(name="sample one row", op="sample", rows=1, vocab=8404, pad=44, dtype="f32", sharp=1.5, filters="all"),
        # a serving batch over a large vocabulary, every row with its own settings
        dict(name="sample batch", op="sample", rows=256, vocab=131072, pad=0, dtype="bf16", sharp=1.2, filters="mixed"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "read", "sample"])
    if op == "sample":
        vocab = _log_int(rng, 300, 131072)
        rows = _log_int(rng, 1, max(1, min(4096, (1 << 25) // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 7, 44, 64]), dtype=rng.choice(["f32", "f16", "bf16"]),
                    sharp=round(rng.uniform(0.6, 2.5), 2), filters=rng.choice(["all", "mixed", "none", "top_k", "top_p", "min_p"]))
    case = dict(op=op, kv_heads=rng.choice([1, 2, 3, 4, 8]), dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                dtype=rng.choice(["f16", "bf16"]), fmt=rng.choice(["16", "e4m3"]), spread=round(rng.uniform(0.0, 0.95), 2))
    if op == "read":
        kv = _log_int(rng, 20, 16384)
        case.update(kv=kv, batch=_log_int(rng, 1, max(1, min(64, (1 << 20) // (kv * case["kv_heads"])))))
        return case
    if op == "append":
        q = rng.choice([1, _log_int(rng, 2, 4096)])
        kv = q + rng.randint(0, 1500)
        case.update(q=q, kv=kv, batch=_log_int(rng, 1, max(1, min(256, (1 << 18) // (kv * case["kv_heads"])))))
        return case
    kind = rng.choice(["token", "chunk", "prompt"])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    if kind == "token":
        q, kv = 1, _log_int(rng, 30, 65536)
        batch = _log_int(rng, 1, max(1, min(256, (1 << 21) // (kv * case["kv_heads"]))))
    elif kind == "chunk":
        q = rng.randint(2, 65)
        kv = q + _log_int(rng, 1, 4096)
        batch = _log_int(rng, 1, max(1, min(256, (1 << 25) // (kv * q * case["kv_heads"] * group))))
    else:
        kv = _log_int(rng, 200, 12288)
        q = _log_int(rng, 100, min(4096, kv, (1 << 29) // (kv * case["kv_heads"] * group)))
        batch = max(1, min(8, (1 << 29) // (kv * q * case["kv_heads"] * group)))
    window = rng.choice([0, 0, _log_int(rng, 2, kv)])
    case.update(q=q, kv=kv, batch=batch, group=group, window=window, sinks=rng.choice([0, 4, 17]) if window else 0,
                causal=rng.choice([True, True, False]))
    return case


def _lengths(case):
    """Positions and new tokens of every sequence: the first one has the case's full lengths, the others are spread below it."""
    kv, q = [], []
    for b in range(case["batch"]):
        part = 1.0 - case["spread"] * ((b * 0.6180339887498949) % 1.0)
        kv.append(max(1, int(case["kv"] * part)))
        q.append(max(1, min(kv[-1], int(case.get("q", 0) * part))))
    return kv, q


def _visible(case, kv, q):
    """Visible (row, key) pairs of one sequence, and the keys that at least one row sees."""
    window, sinks, causal = case["window"], case["sinks"], case["causal"]
    pos = np.arange(kv - q, kv, dtype=np.int64)
    hi = pos + 1 if causal else np.full_like(pos, kv)
    lo = np.maximum(0, pos - window + 1) if window else np.zeros_like(pos)
    pairs = int((hi - lo).sum() + np.minimum(lo, sinks).sum())
    first = int(lo.min())
    return pairs, int(hi.max()) - first + min(first, sinks)


def work(case):
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * TYPES[case["dtype"]].itemsize + case["rows"] * 28, "flops": 3 * n}
    kv, q = _lengths(case)
    row = case["kv_heads"] * case["dim"]
    stored = 2 * case["kv_heads"] * (case["dim"] + 1 if case["fmt"] == "e4m3" else 2 * case["dim"])  # bytes of a position
    table = 4 * sum(-(-n // case["page"]) for n in kv) + 8 * case["batch"]
    if op == "append":
        return {"bytes": sum(q) * (2 * 2 * row + stored) + table, "flops": 4 * sum(q) * row}
    if op == "read":
        return {"bytes": sum(kv) * stored + 2 * 2 * row * case["batch"] * case["kv"] + table, "flops": 2 * sum(kv) * row}
    pairs = keys = 0
    for n, m in zip(kv, q):
        p, k = _visible(case, n, m)
        pairs, keys = pairs + p, keys + k
    heads = case["kv_heads"] * case["group"]
    return {"bytes": keys * stored + 2 * 2 * sum(q) * heads * case["dim"] + table, "flops": 4 * pairs * heads * case["dim"]}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEVICE) * scale).to(dtype)


def _pages(case, gen, kv):
    """A pool of pages in use, in no order, and each sequence's table."""
    page = case["page"]
    need = [-(-n // page) for n in kv]
    total = sum(need)
    order = torch.randperm(total + 3, generator=gen, device=DEVICE)[:total].to(torch.int32).cpu()
    table = torch.zeros(len(kv), max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return total + 3, table.to(DEVICE)


def _cache(case, gen, pages):
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    k, v = _normal(gen, *shape, dtype=torch.float16 if case["fmt"] == "e4m3" else TYPES[case["dtype"]]), None
    if case["fmt"] != "e4m3":
        return {"k": k, "v": _normal(gen, *shape, dtype=k.dtype), "k_exp": None, "v_exp": None}
    # codes that fill the format's range, with scales around those that values of size one get
    k = (k.float() * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)
    v = (_normal(gen, *shape) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)
    k_exp, v_exp = (torch.randint(118, 122, shape[:3], generator=gen, device=DEVICE, dtype=torch.uint8) for _ in range(2))
    return {"k": k, "v": v, "k_exp": k_exp, "v_exp": v_exp}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = dict(case=case)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        rank = torch.rand(rows, vocab + case["pad"], generator=gen, device=DEVICE) * vocab
        logits = -case["sharp"] * torch.log1p(rank) + 0.3 * torch.randn(rank.shape, generator=gen, device=DEVICE)
        state["logits"] = (logits + 8.0).to(TYPES[case["dtype"]])[:, :vocab]  # rows may be padded, as the recogniser's are
        pick = lambda *v: torch.tensor(v, device=DEVICE)[torch.randint(len(v), (rows,), generator=gen, device=DEVICE)]  # noqa: E731
        use, mixed = case["filters"], case["filters"] == "mixed"
        off_k, off_p, off_m = [0] * mixed, [1.0] * mixed, [0.0] * mixed
        state["temperature"] = pick(0.6, 0.8, 1.0, 1.3, *[0.0] * mixed)
        state["top_k"] = (pick(20, 50, 200, *off_k) if use in ("all", "mixed", "top_k") else pick(0)).to(torch.int32)
        state["top_p"] = pick(0.8, 0.9, 0.95, *off_p) if use in ("all", "mixed", "top_p") else pick(1.0)
        state["min_p"] = pick(0.02, 0.05, 0.1, *off_m) if use in ("all", "mixed", "min_p") else pick(0.0)
        state["u"] = torch.rand(rows, generator=gen, device=DEVICE)
        return state
    kv, q = _lengths(case)
    pages, state["block_table"] = _pages(case, gen, kv)
    state.update(_cache(case, gen, pages))
    state["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device=DEVICE)
    if case["op"] == "read":
        return state
    state["cu_q"] = torch.tensor([0] + np.cumsum(q).tolist(), dtype=torch.int32, device=DEVICE)
    state["max_q"] = max(q)
    # the new tokens' projections come out of one product, side by side: q | k | v
    heads = case["kv_heads"] * case.get("group", 0)
    qkv = _normal(gen, sum(q), heads + 2 * case["kv_heads"], case["dim"], dtype=TYPES[case["dtype"]])
    state["q"] = qkv[:, :heads]
    if case["op"] == "append":
        state["new_k"], state["new_v"] = qkv[:, heads:heads + case["kv_heads"]], qkv[:, heads + case["kv_heads"]:]
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _positions(state):
    """Sequence and position of every packed new token."""
    cu, kv = state["cu_q"].long(), state["kv_lens"].long()
    n = state["q"].shape[0]
    t = torch.arange(n, device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, kv[b] - cu[b + 1] + t


def _quantise(x):
    """Rows of 32-bit values -> e4m3 codes and the biased exponents of their scales, the least power of two that brings a
    row's largest magnitude to 448 or below."""
    top = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m * 2 ** e, m in [0.5, 1)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    e = torch.where(top > 0, e, torch.zeros_like(e))
    return torch.ldexp(x, -e).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).squeeze(-1)


def _append(state):
    b, pos = _positions(state)
    page = state["case"]["page"]
    at, row = state["block_table"].long()[b, pos // page], pos % page
    for name in ("k", "v"):
        x = state["new_" + name]
        if state["k_exp"] is None:
            state[name][at, :, row] = x
        else:
            codes, exps = _quantise(x.float())
            state[name].view(torch.uint8)[at, :, row] = codes.view(torch.uint8)
            state[name + "_exp"][at, :, row] = exps
    return _buffers(state)


def _buffers(state):
    return {name: state[name] for name in ("k", "v", "k_exp", "v_exp") if state[name] is not None}


def _dense(state, name):
    """[B, heads, positions, dim] in 32 bits; positions past a sequence's end are zero."""
    table, case = state["block_table"].long(), state["case"]
    x = state[name].view(torch.uint8)[table].view(state[name].dtype).float() if state["k_exp"] is not None else state[name][table].float()
    if state["k_exp"] is not None:
        x = torch.ldexp(x, state[name + "_exp"][table].int().unsqueeze(-1) - 127)
    x = x.transpose(1, 2).reshape(table.shape[0], case["kv_heads"], -1, case["dim"])
    there = torch.arange(x.shape[2], device=x.device) < state["kv_lens"][:, None]
    return x.masked_fill_(~there[:, None, :, None], 0.0)


def _read(state):
    case = state["case"]
    return {name: _dense(state, name)[:, :, :case["kv"]].transpose(1, 2).to(TYPES[case["dtype"]]).contiguous() for name in ("k", "v")}


def _attend(state):
    case, q = state["case"], state["q"]
    batch, heads, group, dim = case["batch"], case["kv_heads"], case["group"], case["dim"]
    k, v = _dense(state, "k"), _dense(state, "v")
    b, pos = _positions(state)
    i = torch.arange(q.shape[0], device=q.device) - state["cu_q"].long()[b]
    rows = torch.zeros(batch, state["max_q"], heads, group, dim, device=q.device)
    rows[b, i] = q.float().view(-1, heads, group, dim)
    at = torch.full((batch, state["max_q"]), -1, device=q.device)
    at[b, i] = pos
    key = torch.arange(k.shape[2], device=q.device)
    see = (key < state["kv_lens"][:, None])[:, None, :] & (at >= 0)[:, :, None]
    if case["causal"]:
        see = see & (key <= at[:, :, None])
    if case["window"]:
        see = see & ((key > at[:, :, None] - case["window"]) | (key < case["sinks"]))
    s = torch.matmul(rows.permute(0, 2, 3, 1, 4).reshape(batch, heads, -1, dim), k.transpose(2, 3).contiguous())
    s = s.view(batch, heads, group, state["max_q"], -1).mul_(1.0 / math.sqrt(dim)).masked_fill_(~see[:, None, None], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = s.sum(-1, keepdim=True)
    out = torch.matmul(s.view(batch, heads, -1, s.shape[-1]), v).view(batch, heads, group, state["max_q"], dim) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4)[b, i].reshape(q.shape).to(q.dtype)


def _sample(state):
    logits, temperature = state["logits"].double(), state["temperature"].double()[:, None]
    vocab = logits.shape[1]
    greedy = temperature <= 0
    value, index = torch.sort(logits, dim=1, descending=True, stable=True)
    w = torch.exp((value - value[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature))
    rank = torch.arange(vocab, device=logits.device)
    top_k = state["top_k"].long()[:, None]
    keep = (rank < torch.where(top_k > 0, top_k, vocab)) & (~greedy | (rank == 0))
    w = w * keep
    before = torch.cumsum(w, 1) - w
    top_p = state["top_p"].double()[:, None]
    keep &= (before < top_p * w.sum(1, keepdim=True)) | (top_p >= 1) | (rank == 0)
    keep &= (w >= state["min_p"].double()[:, None]) | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, index, w * keep)  # in the order of the vocabulary again
    upto = torch.cumsum(kept, 1)
    total = upto[:, -1:]
    over = (upto > state["u"].double()[:, None] * total) & (kept > 0)
    token = torch.argmax(over.to(torch.uint8), dim=1)
    logprob = torch.log(kept.gather(1, token[:, None]) / total).squeeze(1)
    return {"token": token.to(torch.int32), "logprob": logprob.float()}


# ---- the package's calls ----------------------------------------------------------------------------------------------
_handle = None


def _context():
    global _handle
    if _handle is None:
        import toolbox_for_asr_and_tts_amd as pkg

        _handle = pkg.Context()
    return _handle


def _own_cache(state):
    """The cache object that a program keeps beside its buffers."""
    if "cache" not in state:
        import toolbox_for_asr_and_tts_amd as pkg

        state["cache"] = pkg.PagedKvCache(_context(), state["k"], state["v"], state["k_exp"], state["v_exp"])
    return state["cache"]


def _own_run(state):
    case = state["case"]
    if case["op"] == "sample":
        import toolbox_for_asr_and_tts_amd as pkg

        token, logprob = pkg.sample_tokens(_context(), state["logits"], state["u"], temperature=state["temperature"],
                                           top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
        return {"token": token, "logprob": logprob}
    cache = _own_cache(state)
    if case["op"] == "append":
        cache.append(state["new_k"], state["new_v"], state["cu_q"], state["kv_lens"], state["block_table"])
        return _buffers(state)
    if case["op"] == "read":
        k, v = cache.read(state["kv_lens"], state["block_table"], case["kv"], dtype=TYPES[case["dtype"]])
        return {"k": k, "v": v}
    return cache.attend(state["q"], state["cu_q"], state["kv_lens"], state["block_table"], window=case["window"],
                        sinks=case["sinks"], causal=case["causal"])


def run(state):
    if own:
        return _own_run(state)
    return {"append": _append, "read": _read, "attend": _attend, "sample": _sample}[state["case"]["op"]](state)


# ---- the definitions in 64 bits, sequence by sequence and row by row -----------------------------------------------------
def _exact_values(state, name, b, lo, hi):
    """Positions lo .. hi - 1 of sequence b as [positions, heads, dim]."""
    page = state["case"]["page"]
    pos = torch.arange(lo, hi, device=DEVICE)
    at = state["block_table"][b].long()[torch.div(pos, page, rounding_mode="floor")]
    x = state[name].view(torch.uint8)[at, :, pos % page].view(state[name].dtype).double() if state["k_exp"] is not None \
        else state[name][at, :, pos % page].double()
    if state["k_exp"] is not None:
        x = x * torch.exp2(state[name + "_exp"][at, :, pos % page].double() - 127.0).unsqueeze(-1)
    return x


def _exact_attend(state):
    case = state["case"]
    heads, group, dim = case["kv_heads"], case["group"], case["dim"]
    kv, nq = _lengths(case)
    out, start = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE), 0
    for b in range(case["batch"]):
        k, v = _exact_values(state, "k", b, 0, kv[b]), _exact_values(state, "v", b, 0, kv[b])
        step = max(1, (1 << 27) // kv[b])
        for h in range(heads * group):
            kh, vh = k[:, h // group].contiguous(), v[:, h // group].contiguous()
            for r0 in range(0, nq[b], step):
                r1 = min(nq[b], r0 + step)
                pos = torch.arange(kv[b] - nq[b] + r0, kv[b] - nq[b] + r1, device=DEVICE)[:, None]
                key = torch.arange(kv[b], device=DEVICE)[None, :]
                hidden = torch.zeros(r1 - r0, kv[b], dtype=torch.bool, device=DEVICE)
                if case["causal"]:
                    hidden |= key > pos
                if case["window"]:
                    hidden |= (key <= pos - case["window"]) & (key >= case["sinks"])
                s = state["q"][start + r0:start + r1, h].double() @ kh.t().contiguous() / dim ** 0.5
                out[start + r0:start + r1, h] = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1) @ vh
        start += nq[b]
    return out


def _exact_e4m3(x):
    """Rows of 64-bit values -> the nearest e4m3 values under the row's scale (ties to even), and the scale's exponent."""
    top = np.abs(x).max(axis=-1, keepdims=True)
    with np.errstate(divide="ignore"):
        e = np.ceil(np.log2(top / 448.0))
    e = np.where(top > 0, np.maximum(e, -126), 0)
    # (a quotient right at a power of two: decided by the products, which are exact)
    e = np.where((top > 0) & (448.0 * np.exp2(e - 1) >= top) & (e > -126), e - 1, e)
    e = np.where((top > 0) & (448.0 * np.exp2(e) < top), e + 1, e)
    y = x / np.exp2(e)
    with np.errstate(divide="ignore"):
        step = np.exp2(np.maximum(np.floor(np.log2(np.abs(y))), -6) - 3)
    return np.rint(y / step) * step, e[..., 0] + 127


def _exact_append(state):
    case = state["case"]
    kv, nq = _lengths(case)
    table = state["block_table"].cpu().numpy()
    got = {}
    for name in ("k", "v"):
        buf = state[name].double().cpu().numpy()
        exps = None if state["k_exp"] is None else state[name + "_exp"].cpu().numpy().astype(np.int64)
        new, start = state["new_" + name].double().cpu().numpy(), 0
        for b in range(case["batch"]):
            pos = np.arange(kv[b] - nq[b], kv[b])
            at, row = table[b][pos // case["page"]], pos % case["page"]
            x = new[start:start + nq[b]]
            if exps is not None:
                x, e = _exact_e4m3(x)
                exps[at, :, row] = e
            buf[at, :, row] = x
            start += nq[b]
        got[name] = buf
        if exps is not None:
            got[name + "_exp"] = exps
    return got


def _exact_read(state):
    case = state["case"]
    kv, _ = _lengths(case)
    got = {}
    for name in ("k", "v"):
        got[name] = torch.zeros(case["batch"], case["kv"], case["kv_heads"], case["dim"], dtype=torch.float64, device=DEVICE)
        for b in range(case["batch"]):
            got[name][b, :kv[b]] = _exact_values(state, name, b, 0, kv[b])
    return got


def _exact_sample(state):
    case = state["case"]
    logits = state["logits"].double().cpu().numpy()
    temperature, top_k, top_p, min_p, u = (state[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    token, logprob = np.zeros(case["rows"], dtype=np.int64), np.zeros(case["rows"])
    for r in range(case["rows"]):
        best = int(np.argmax(logits[r]))
        if temperature[r] <= 0:
            token[r] = best
            continue
        w = np.exp((logits[r] - logits[r][best]) / temperature[r])
        order = np.lexsort((np.arange(w.size), -logits[r]))
        n = int(top_k[r]) if 0 < top_k[r] < w.size else w.size
        mass = np.cumsum(w[order[:n]])
        if top_p[r] < 1:
            n = min(n, 1 + int(np.searchsorted(mass, top_p[r] * mass[-1], side="left")))
        n = max(1, min(n, int(np.count_nonzero(w[order[:n]] >= min_p[r]))))
        chosen = np.sort(order[:n])
        mass = np.cumsum(w[chosen])
        token[r] = chosen[min(n - 1, int(np.searchsorted(mass, u[r] * mass[-1], side="right")))]
        logprob[r] = math.log(w[token[r]] / mass[-1])
    return {"token": token, "logprob": logprob}


def exact(case, seed):
    if case["op"] == "attend" and work(case)["flops"] > 2e12:
        return None
    state = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](state)
