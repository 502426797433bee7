"""CPU tests of the paged cache, its attention and the choice of a token: refusals of both layers before anything touches a
device, and the oracle against independent statements (torch's own e4m3 conversion, its softmax, known answers)."""
import ctypes as C
import glob
import os
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

from oracle import paged_oracle as po  # noqa: E402


@pytest.fixture(scope="module")
def pkg():
    import toolbox_for_asr_and_tts_amd as p

    p.load()
    return p


# ---- the C entry points refuse bad arguments before they touch the context, the stream or the device -------------------------
class _Abi:
    """Calls with good numbers and one of them changed.  The context is a block of zeros and the pointers are numbers: a
    refusal reads neither."""

    def __init__(self, pkg):
        self.lib, self.L = pkg.load(), pkg._lib
        self.block = C.create_string_buffer(1 << 16)
        self.ctx = C.cast(self.block, C.c_void_p)

    def error(self):
        return self.lib.asrfe_last_error(self.ctx).decode()

    def cache(self, **kw):
        f = dict(k=1 << 20, v=1 << 21, k_exp=None, v_exp=None, n_pages=4, page_size=16, n_heads=4, head_dim=128, dtype=self.L.DT_F16)
        f.update(kw)
        return self.L.KvCache(*f.values())

    def append(self, cache=None, **kw):
        f = dict(k=4096, v=8192, dtype=self.L.DT_F16, kts=512, khs=128, vts=512, vhs=128, n=3, cu=64, lens=64, table=64, stride=2,
                 batch=1, stream=None)
        f.update(kw)
        return self.lib.asrfe_kv_append(self.ctx, C.byref(cache or self.cache()), *f.values())

    def read(self, cache=None, **kw):
        f = dict(lens=64, table=64, stride=2, batch=1, t_max=5, k=4096, v=8192, dtype=self.L.DT_F16, stream=None)
        f.update(kw)
        return self.lib.asrfe_kv_read(self.ctx, C.byref(cache or self.cache()), *f.values())

    def attend(self, cache=None, **kw):
        f = dict(q=4096, dtype=self.L.DT_F16, qts=512, qhs=128, n=3, heads=4, cu=64, lens=64, table=64, stride=2, batch=1, max_kv=32,
                 window=0, sinks=0, causal=1, scale=0.1, out=8192, ots=512, ohs=128, ws=None, nbytes=0, stream=None)
        f.update(kw)
        return self.lib.asrfe_paged_attention(self.ctx, C.byref(cache or self.cache()), *f.values())

    def sample(self, **kw):
        f = dict(logits=4096, dtype=self.L.DT_F32, ld=100, rows=2, vocab=100, u=64, t=None, k=None, p=None, m=None, num=None, per=0,
                 ids=64, logprobs=None, stream=None)
        f.update(kw)
        return self.lib.asrfe_sample_tokens(self.ctx, *f.values())


@pytest.fixture(scope="module")
def abi(pkg):
    return _Abi(pkg)


BAD, SHAPE = -1, -2


@pytest.mark.parametrize("field, value, code", [
    ("dtype", 0, BAD), ("dtype", 7, BAD), ("head_dim", 96, SHAPE), ("head_dim", 0, SHAPE), ("page_size", 48, SHAPE), ("page_size", 8, SHAPE),
    ("page_size", 512, SHAPE), ("page_size", 0, SHAPE), ("n_heads", 0, SHAPE), ("n_heads", 257, SHAPE), ("n_pages", 0, SHAPE), ("k", None, BAD),
    ("v", None, BAD), ("k", 1 << 20 | 8, BAD), ("v", 1 << 21 | 4, BAD), ("k_exp", 64, BAD), ("v_exp", 64, BAD), ("dtype", 3, BAD)])
def test_every_entry_point_refuses_a_bad_cache(abi, field, value, code):
    for call in (abi.append, abi.read, abi.attend):
        assert call(abi.cache(**{field: value})) == code
        assert abi.error().startswith("asrfe_")


@pytest.mark.parametrize("kw, code", [
    (dict(dtype=0), BAD), (dict(dtype=1), BAD), (dict(dtype=3), BAD), (dict(batch=-1), SHAPE), (dict(batch=65536), SHAPE), (dict(stride=-1), SHAPE),
    (dict(stride=1 << 27), SHAPE)])
def test_every_entry_point_refuses_a_bad_batch(abi, kw, code):
    for call in (abi.append, abi.read, abi.attend):
        assert call(**kw) == code


def _reaches_the_device_check(abi, rc):
    """Good arguments get as far as the comparison of devices, which a block of zeros fails where there is no GPU; with one
    (device 0, as the zeros say) the call would run on made-up pointers, so these are asked for without a GPU only."""
    assert rc == BAD and "device" in abi.error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="would run on made-up pointers")
def test_good_arguments_pass_the_checks(abi):
    for call in (abi.append, abi.read, abi.attend, abi.sample):
        _reaches_the_device_check(abi, call())


def test_null_contexts_and_caches_are_refused(pkg):
    lib = pkg.load()
    abi = _Abi(pkg)
    good = C.byref(abi.cache())
    assert lib.asrfe_kv_append(None, good, 16, 16, 2, 8, 8, 8, 8, 1, 16, 16, 16, 1, 1, None) == BAD
    assert lib.asrfe_kv_read(None, good, 16, 16, 1, 1, 1, 16, 16, 2, None) == BAD
    assert lib.asrfe_sample_tokens(None, 16, 0, 8, 1, 8, 16, None, None, None, None, None, 0, 16, None, None) == BAD
    assert lib.asrfe_kv_append(abi.ctx, None, 16, 16, 2, 8, 8, 8, 8, 1, 16, 16, 16, 1, 1, None) == BAD
    assert lib.asrfe_paged_attention_workspace_bytes(abi.ctx, None, 1, 1, 1, 1) == -1
    assert lib.asrfe_paged_attention_workspace_bytes(None, good, 1, 4, 1, 1) == -1
    for args in ((-1, 4, 1, 1), (1, 5, 1, 1), (1, 0, 1, 1), (1, 4, -1, 1), (1, 4, 1, -1), (1, 4, 65536, 1), ((1 << 24) + 1, 4, 1, 1), (1, 4 * 257, 1, 1)):
        assert lib.asrfe_paged_attention_workspace_bytes(abi.ctx, good, *args) == -1


@pytest.mark.parametrize("n, heads, ts, hs", [
    (3, 4, 128, 128), (3, 4, 256, 128), (3, 4, 512, 0), (3, 4, 512, 64), (3, 4, 384, 128), (2, 4, 504, 128), (3, 4, 128, 256), (4, 3, 320, 640),
    (9, 2, 136, 1024), (2, 8, 128 * 9 + 64, 384), (2, 2, 1 << 62, 1 << 62), (1, 4, 0, 120), (2, 1, 120, 0)])
def test_results_that_overlap_are_refused(abi, n, heads, ts, hs):
    assert abi.attend(n=n, heads=heads, ots=ts, ohs=hs, cache=abi.cache(n_heads=1)) == BAD and "overlap" in abi.error()


ROWS_APART = [(3, 4, 512, 128), (3, 4, 128, 384), (1, 4, 0, 128), (4, 1, 128, 0), (2, 8, 128 * 9, 256), (4, 3, 256, 384 + 512), (2, 3, 3 * 128 + 8, 1024)]


@pytest.mark.skipif(torch.cuda.is_available(), reason="would run on made-up pointers")
@pytest.mark.parametrize("n, heads, ts, hs", ROWS_APART)
def test_results_that_do_not_overlap_are_taken(abi, n, heads, ts, hs):
    _reaches_the_device_check(abi, abi.attend(n=n, heads=heads, ots=ts, ohs=hs, cache=abi.cache(n_heads=1)))


def test_overlap_by_its_definition(pkg):
    """Both layers' rule against a count of the elements, over all small layouts."""
    from toolbox_for_asr_and_tts_amd.paged import _rows_apart

    for n in range(1, 5):
        for heads in range(1, 5):
            for ts in range(0, 34):
                for hs in range(0, 34):
                    at = [t * ts + h * hs + d for t in range(n) for h in range(heads) for d in range(3)]
                    assert _rows_apart(n, heads, 3, ts, hs) == (len(set(at)) == len(at)), (n, heads, ts, hs)


@pytest.mark.parametrize("kw, code", [
    (dict(dtype=3), BAD), (dict(dtype=9), BAD), (dict(rows=-1), SHAPE), (dict(vocab=0), SHAPE), (dict(vocab=(1 << 18) + 1, ld=1 << 20), SHAPE),
    (dict(ld=99), SHAPE), (dict(num=64, per=0), SHAPE), (dict(rows=(1 << 24) + 1), SHAPE)])
def test_sample_refuses(abi, kw, code):
    assert abi.sample(**kw) == code


@pytest.mark.parametrize("rc", [lambda a: a.read(batch=1 << 10, t_max=1 << 16), lambda a: a.read(batch=1, t_max=1 << 26), lambda a: a.sample(rows=(1 << 23) + 1)])
def test_more_threads_than_a_launch_holds_are_refused(abi, rc):
    assert rc(abi) == SHAPE


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan"), 2.4e38, -3e38])
def test_scales_that_are_not_finite_in_base_two_are_refused(abi, scale):
    assert abi.attend(scale=scale) == BAD and "scale" in abi.error()


def test_documents_fill_the_cache_structure_in_its_order(pkg):
    """The examples that build it from its fields one after the other, evaluated."""
    names = [n for n, _ in pkg._lib.KvCache._fields_]
    given = dict(zip(names, (64, 128, 192, 256, 7, 16, 3, 128, pkg._lib.DT_E4M3)))
    scope = dict(given, **{n: getattr(pkg._lib, "DT_E4M3") for n in ("DT_E4M3", "ASRFE_DT_E4M3")}, KvCache=pkg._lib.KvCache)
    calls = [m for path in glob.glob(os.path.join(ROOT, "*.md")) for m in re.findall(r"(?<![A-Za-z])KvCache\([^()]*\)", open(path).read())]
    assert calls
    for call in calls:
        built = eval(call, {}, scope)
        assert {n: getattr(built, n) for n in names} == given, call


# ---- the Python layer ---------------------------------------------------------------------------------------------------------
def test_cache_refuses_bad_buffers(pkg):
    def make(shape=(2, 4, 16, 64), dtype=torch.float16, **kw):
        return pkg.PagedKvCache(None, torch.zeros(shape).to(dtype), torch.zeros(shape).to(dtype), **kw)

    for kw in (dict(dtype=torch.float32), dict(shape=(2, 4, 17, 64)), dict(shape=(2, 4, 16, 80)), dict(shape=(0, 4, 16, 64)),
               dict(shape=(2, 0, 16, 64)), dict(shape=(4, 16, 64)), dict(dtype=torch.float8_e4m3fn),
               dict(k_exp=torch.zeros(2, 4, 16, dtype=torch.uint8)), dict()):  # the last: good, but on the CPU
        with pytest.raises(ValueError, match="PagedKvCache"):
            make(**kw)
    with pytest.raises(ValueError, match="uint8"):
        make(dtype=torch.float8_e4m3fn, k_exp=torch.zeros(2, 4, 16), v_exp=torch.zeros(2, 4, 16))


def test_lengths_given_as_offsets_are_refused(pkg):
    """One tensor as kv_lens and cu_q has an entry too few: the kernels would read past its end."""
    c = pkg.PagedKvCache.__new__(pkg.PagedKvCache)
    c._index, c.device = -1, torch.device("cpu")  # (a host tensor's device index)
    lens, table, x = torch.ones(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 4, 64)
    for call in (lambda: c.append(x, x, lens, lens, table), lambda: c.attend(x, lens, lens, table)):
        with pytest.raises(ValueError, match="one entry more"):
            call()


def test_sample_tokens_refuses_host_tensors(pkg):
    with pytest.raises(ValueError, match="CUDA"):
        pkg.sample_tokens(None, torch.zeros(2, 8), torch.zeros(2))


# ---- the oracle ----------------------------------------------------------------------------------------------------------
def test_oracle_e4m3_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    v = codes.view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(po.E4M3, v)
    rng = np.random.default_rng(0)
    for scale in (1e-30, 1e-3, 1.0, 300.0, 1e20):
        x = torch.from_numpy(rng.standard_normal((50, 64)) * scale).float()
        got, exps = po.quantise(x.double().numpy())
        e = torch.from_numpy(exps.astype(np.int32)) - 127
        want = torch.ldexp(x, -e[:, None]).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        np.testing.assert_array_equal(got, want)
        y = np.abs(x.double().numpy()).max(1) / np.exp2(e.numpy().astype(np.float64))
        assert (y <= 448).all() and (y > 224).all()


def test_oracle_e4m3_special_rows():
    x = np.zeros((6, 8))
    x[1, 0], x[2, :3], x[3, 0], x[4, 0], x[5, :2] = 448.0, [np.inf, -np.inf, 1.0], 1e-45, 448.0 * 2 + 1, [np.nan, 3.0]
    codes, exps = po.quantise(x)
    assert exps.tolist() == [127, 127, 127 - 8, 1, 129, 127 - 7]
    assert codes[2, :2].tolist() == [0x7e, 0xfe] and codes[5, 0] & 0x7f == 0x7f
    assert po.dequantise(codes, exps)[2, 2] == 1.0 and po.dequantise(codes, exps)[5, 1] == 3.0


def test_oracle_attention_is_softmax_attention():
    rng = np.random.default_rng(1)
    n, h, d, page = 37, 2, 64, 16
    k, v = rng.standard_normal((2, 3, h, page, d))
    table = np.array([[2, 0, 1]])
    q = rng.standard_normal((5, 4, d))
    out, _, _, owned = po.attend(q, k, v, [0, 5], [n], table, page)
    kd = torch.from_numpy(k[table[0]]).transpose(0, 1).reshape(h, -1, d)[:, :n].repeat_interleave(2, 0)
    vd = torch.from_numpy(v[table[0]]).transpose(0, 1).reshape(h, -1, d)[:, :n].repeat_interleave(2, 0)
    mask = torch.ones(5, n, dtype=torch.bool).tril(n - 5)
    want = torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q).transpose(0, 1), kd, vd, attn_mask=mask)
    assert owned.all() and np.abs(out - want.transpose(0, 1).numpy()).max() < 1e-12


def test_oracle_masks():
    assert po.visible(5, 8, 0, 0, True).tolist() == [True] * 6 + [False] * 2
    assert po.visible(5, 8, 2, 1, True).tolist() == [True, False, False, False, True, True, False, False]
    assert po.visible(5, 8, 2, 0, False).tolist() == [False] * 4 + [True] * 4
    assert not po.visible(-1, 8, 0, 4, False).any()


def test_oracle_sampling_known_answers():
    l = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert [po.sample_row(l, u)[0] for u in (0.0, 0.05, 0.15, 0.55, 0.65, 0.75, 0.99)] == [0, 0, 1, 2, 2, 3, 3]
    assert po.sample_row(l, 0.5, top_k=1)[:2] == (1, 0.0)
    assert [po.sample_row(l, u, top_p=0.6)[0] for u in (0.1, 0.5, 0.6, 0.9)] == [1, 1, 3, 3]      # 0.4 + 0.3 reach 0.6
    assert [po.sample_row(l, u, min_p=0.49)[0] for u in (0.0, 0.44, 0.45, 0.6)] == [1, 1, 2, 2]
    assert po.sample_row(np.zeros(5), 0.99, top_k=2)[0] == 1                                      # equal ones: lowest indices
    assert po.sample_row(np.full(4, -np.inf), 0.5)[:2] == (0, -np.inf)
    assert po.sample_row(np.array([np.nan, -np.inf, 2.0]), 0.9)[0] == 2
    assert po.sample_row(np.array([1.0, np.inf, 3.0, np.inf]), 0.6)[0] == 3
    assert po.sample_row(l, 0.9, temperature=0.0)[0] == 1


# ---- the generated code ---------------------------------------------------------------------------------------------------
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc to generate the kernels' assembly")
@pytest.mark.parametrize("source", ["paged_kernels.hip", "paged_attention.hip", "sampling_kernels.hip"])
def test_generated_code(tmp_path, source):
    """With the Makefile's flags: no packed fp32 arithmetic, no flat access of memory (the LDS counter would wait for it), and
    LDS-DMA loads that keep their distance from the M0 write in front of them."""
    from tools import check_vm_queue as cq

    csrc = os.path.join(ROOT, "toolbox-for-asr-and-tts_amd", "csrc")
    path = str(tmp_path / "kernels.s")
    subprocess.check_call([HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                           "-I" + os.path.join(ROOT, "include"), "-I" + csrc, "-S", "--cuda-device-only", "-o", path,
                           os.path.join(csrc, source)], stderr=subprocess.DEVNULL)
    text = open(path).read()
    assert not re.findall(r"\bv_pk_(?:add|mul|fma)_f32", text)
    if source == "paged_attention.hip":
        assert cq.check_m0(path) == []
    assert not re.findall(r"\bflat_(?:load|store)", text)
