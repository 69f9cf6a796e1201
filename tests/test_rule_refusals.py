"""Refusals of the norm + rotation and score-rule entry points, their workspace queries and the rotations' frequencies:
on the CPU, before any launch."""
import ctypes
import math

import pytest
import torch

from delta_amd import _lib
from delta_amd import kernels as K

A = 1 << 20  # stand-in address, never dereferenced
NO_GPU = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="stand-in addresses: validation-only, run where no GPU is visible")


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not _lib.LIB_PATH.exists():
        from delta_amd import build
        build.build()
    return _lib.load()


def rot(turns=A, dim=128, inter=0, factor=1.0):
    return ctypes.byref(_lib.RotaryC(turns, dim, inter, factor))


def norm(q=A, k=A, eps=1e-6):
    return ctypes.byref(_lib.HeadNormC(q, k, eps))


def rule(cap=0.0, slopes=None, window=0, begin=None, end=None):
    return ctypes.byref(_lib.ScoreRuleC(cap, slopes, window, begin, end))


def rope(r=rot(), n=norm(), q=A, qs=4096, k=A, ks=1024, qo=A, qos=4096, ko=A, kos=1024, ip=A, off=A, nnz=5, batch=2, hq=32,
         hkv=8, hd=128, dt=0):
    return (r, n, q, qs, k, ks, qo, qos, ko, kos, ip, off, nnz, batch, hq, hkv, hd, dt, None)


def append(r=rot(), n=norm(), q=A, v=A, vs=1024, ip=A, cache=A, pages=16, ind=A, ilen=16, kip=A, last=A, nnz=5, batch=2, hd=128, dt=0):
    return (r, n, q, 4096, A, 1024, v, vs, A, 4096, ip, A, cache, pages, ind, ilen, kip, last, nnz, batch, 32, 8, hd, dt, None)


def decode(r=rule(), q=A, sb=4096, kv=A, pages=16, ip=A, ilen=16, o=A, batch=2, hq=32, hkv=8, hd=128, dt=0, mp=64, ws=A, wsb=1 << 40):
    return (r, q, sb, 128, kv, pages, ip, A, ilen, A, o, 4096, 128, None, batch, hq, hkv, hd, dt, 1.0, mp, ws, wsb, None)


def prefill(r=rule(), q=A, st=4096, kv=A, pages=16, qo=A, ilen=4096, o=A, os=4096, batch=2, tokens=5, mq=5, hq=32, hkv=8, hd=128, dt=0,
            ws=A, wsb=1 << 40):
    return (r, q, st, 128, kv, pages, qo, A, A, ilen, A, o, os, 128, None, batch, tokens, mq, hq, hkv, hd, dt, 1.0, ws, wsb, None)


def rejects(name, args, match):
    with pytest.raises(_lib.DeltaHipError, match=match):
        _lib.call(name, *args)


def test_empty_calls_return_before_touching_pointers():
    _lib.call("delta_qk_norm_rope", *rope(q=None, nnz=0))
    _lib.call("delta_qk_norm_rope", *rope(q=None, batch=0))
    _lib.call("delta_qk_norm_rope_append", *append(q=None, nnz=0))
    _lib.call("delta_paged_decode_rule", *decode(r=None, q=None, batch=0))
    _lib.call("delta_paged_prefill_rule", *prefill(r=None, q=None, batch=0))
    _lib.call("delta_paged_prefill_rule", *prefill(r=None, q=None, tokens=0))
    _lib.call("delta_paged_prefill_rule", *prefill(r=None, q=None, mq=0))


@NO_GPU
@pytest.mark.parametrize("args,match", [
    (dict(hd=64), "head_dim must be 128"),
    (dict(dt=7), "bad dtype"),
    (dict(hq=0), "bad head counts"),
    (dict(hkv=-1), "bad head counts"),
    (dict(nnz=(1 << 23) + 1), "more than 2\\^23 tokens"),
    (dict(q=None), "null pointer"),
    (dict(ip=None), "null pointer"),
    (dict(off=None), "null pointer"),
    (dict(q=A + 8), "16-byte aligned"),
    (dict(ks=1028), "multiples of 8"),
    (dict(qos=4097), "multiples of 8"),
    (dict(ko=None), "k_out null"),
    (dict(ko=A + 4), "k_out null or not 16-byte aligned"),
    (dict(r=rot(dim=130)), "rotary_dim must be even"),
    (dict(r=rot(dim=-2)), "rotary_dim must be even"),
    (dict(r=rot(dim=33)), "rotary_dim must be even"),
    (dict(r=rot(turns=None)), "turns null"),
    (dict(r=rot(turns=A + 4)), "turns null or not 8-byte aligned"),
    (dict(n=norm(q=None)), "norm weights null"),
    (dict(n=norm(k=A + 2)), "norm weights null or not 16-byte aligned"),
    (dict(n=norm(eps=-1.0)), "bad eps"),
    (dict(n=norm(eps=math.nan)), "bad eps"),
])
def test_rope(args, match):
    rejects("delta_qk_norm_rope", rope(**args), match)


@NO_GPU
@pytest.mark.parametrize("args,match", [
    (dict(hd=64), "head_dim must be 128"),
    (dict(v=None), "null pointer"),
    (dict(cache=None), "null pointer"),
    (dict(kip=None), "null pointer"),
    (dict(v=A + 8), "16-byte aligned"),
    (dict(vs=1001), "v stride"),
    (dict(pages=0), "empty cache"),
    (dict(ilen=-1), "empty cache"),
    (dict(r=rot(dim=200)), "rotary_dim"),
])
def test_append(args, match):
    rejects("delta_qk_norm_rope_append", append(**args), match)


RULES = [
    (dict(r=None), "null score rule"),
    (dict(r=rule(cap=-1.0)), "softcap must be 0"),
    (dict(r=rule(cap=math.nan)), "softcap must be 0"),
    (dict(r=rule(cap=math.inf)), "softcap must be 0"),
    (dict(r=rule(cap=1e-35)), "softcap too small"),
    (dict(r=rule(window=-1)), "window must be 0"),
    (dict(r=rule(slopes=A + 2)), "4-byte aligned"),
    (dict(r=rule(begin=A + 1)), "4-byte aligned"),
    (dict(r=rule(end=A + 3)), "4-byte aligned"),
    (dict(hd=64), "head_dim must be 128"),
    (dict(hq=12), "multiple of num_kv_heads"),
    (dict(hq=72), "group size 9 > 8"),
    (dict(dt=7), "dtype"),
    (dict(q=None), "null"),
    (dict(o=None), "null"),
    (dict(q=A + 8), "16-byte aligned"),
    (dict(pages=0), "empty cache"),
    (dict(ilen=-1), "empty cache"),
]


@NO_GPU
@pytest.mark.parametrize("args,match", RULES + [
    (dict(sb=4100), "multiples of 8"),
    (dict(ws=None), "workspace of .* bytes needed"),
    (dict(wsb=1000), "workspace of .* bytes needed, 1000 given"),
    (dict(ws=A + 16), "workspace must be 256-byte aligned"),
])
def test_decode_rule(args, match):
    rejects("delta_paged_decode_rule", decode(**args), match)


@NO_GPU
@pytest.mark.parametrize("args,match", RULES + [
    (dict(st=4100), "multiples of 8"),
    (dict(o=A + 4), "o 8-byte aligned"),
    (dict(os=4098), "multiples of 4"),
    (dict(qo=None), "null"),
    (dict(tokens=(1 << 23) + 1), "more than 2\\^23 tokens"),
    (dict(ilen=(1 << 26) + 1), "2\\^26 pages"),
    (dict(ws=None), "workspace of .* bytes needed"),
    (dict(wsb=1000), "workspace of .* bytes needed, 1000 given"),
    (dict(ws=A + 16), "workspace must be 256-byte aligned"),
])
def test_prefill_rule(args, match):
    rejects("delta_paged_prefill_rule", prefill(**args), match)


def test_workspace_queries(lib):
    p = lib.delta_paged_prefill_rule_workspace_bytes
    assert p(0, 1, 32, 8, 1, 100, 0) == 0 and p(5, 1, 12, 8, 5, 100, 0) == 0 and p(5, 1, 72, 8, 5, 100, 0) == 0
    assert p(8192, 1, 32, 8, 8192, 512, 0) == 0   # tiles enough: nothing is cut
    assert p(40, 1, 32, 8, 40, 40, 0) == 0        # a short cache
    assert p(40, 1, 32, 8, 40, 4096, 64) == 0     # a short window
    sizes = [p(t, 4, 28, 4, t, 4096, 0) for t in (1, 8, 48, 300, 4000)]
    assert all(s > 0 and s % 256 == 0 and s < 64 << 20 for s in sizes)
    d = lib.delta_paged_decode_rule_workspace_bytes
    assert d(2, 32, 8, 1000, 0) == lib.delta_paged_decode_workspace_bytes(2, 32, 8, 1000)
    # a window of 33 tokens lies in at most 3 pages
    assert d(2, 32, 8, 1000, 33) == lib.delta_paged_decode_workspace_bytes(2, 32, 8, 3)
    assert d(0, 32, 8, 1000, 0) == 0


def test_frequencies():
    f, factor = K.rotary_frequencies(128, rope_theta=1e4)
    assert factor == 1.0 and f[0] == 1.0 and f[63] == pytest.approx(1e4 ** (-126 / 128), rel=1e-15)
    g, _ = K.rotary_frequencies(128, rope_theta=1e4, rope_scale=4.0)
    assert g == [x / 4 for x in f]
    n, _ = K.rotary_frequencies(128, rope_theta=1e4, rope_scale=4.0, scaling="ntk")
    assert n[0] == 1.0 and n[63] == pytest.approx(f[63] / 4, rel=1e-12)
    y, factor = K.rotary_frequencies(128, rope_theta=1e4, rope_scale=4.0, old_context_len=4096.0, scaling="yarn")
    assert factor == pytest.approx(0.1 * math.log(4) + 1)
    for a, b in zip(f, y):
        turns = 4096.0 * a / (2 * math.pi)
        assert b == (a if turns >= 32 else pytest.approx(a / 4) if turns <= 1 else pytest.approx(a / 4 + (a - a / 4) * (turns - 1) / 31))
    # the blend that rope applies, at the two borders and inside
    m, _ = K.rotary_frequencies(128, rope_theta=5e5, rope_scale=8.0, low_freq_factor=1.0, high_freq_factor=4.0, old_context_len=8192.0)
    from oracle import delta_oracle as O
    want = O.rope_frequencies(128, 8.0, 5e5, 1.0, 4.0, 8192)
    assert torch.allclose(torch.tensor(m, dtype=torch.float64), torch.as_tensor(want).double(), rtol=1e-5)


def test_turns_are_exact_fractions():
    r = K.rotary(4, frequencies=[2 * math.pi / 4, -2 * math.pi / 8], device="cpu")
    turns = [t % (1 << 64) for t in r.turns.tolist()]
    assert abs(turns[0] - (1 << 62)) <= 1 << 10 and abs(turns[1] - ((1 << 64) - (1 << 61))) <= 1 << 10
    assert (r.rotary_dim, r.interleaved, r.factor, r.c.rotary_dim, r.c.turns) == (4, False, 1.0, 4, r.turns.data_ptr())


@pytest.mark.parametrize("args,match", [
    (dict(rotary_dim=127), "rotary_dim"), (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=256), "rotary_dim"),
    (dict(rope_theta=0.0), "positive"), (dict(rope_scale=-1.0), "positive"), (dict(rope_theta=math.nan), "positive"),
    (dict(scaling="x"), "unknown scaling"), (dict(rotary_dim=2, scaling="ntk"), "over 2"),
    (dict(scaling="yarn"), "old_context_len"), (dict(scaling="yarn", old_context_len=10.0, beta_slow=40.0), "low < high"),
    (dict(scaling="llama31", old_context_len=10.0), "low < high"),
    (dict(rotary_dim=4, frequencies=[1.0]), "2 frequencies"), (dict(rotary_dim=2, frequencies=[math.inf]), "finite"),
    (dict(rotary_dim=2, frequencies=[1.0], rope_theta=3.0), "no scaling"), (dict(factor=math.nan), "factor"),
])
def test_rotary_refusals(args, match):
    with pytest.raises(ValueError, match=match):
        K.rotary(device="cpu", **args)


def test_wrappers_refuse_host_tensors():
    q, k = torch.zeros(1, 4, 128, dtype=torch.bfloat16), torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    ip, one = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([0], dtype=torch.int32)
    cache = torch.zeros(2, 2, 16, 2, 128, dtype=torch.bfloat16)
    r = K.rotary(device="cpu")
    with pytest.raises(ValueError, match="GPU tensors"):
        K.qk_norm_rope(q, k, ip, one, r)
    with pytest.raises(ValueError, match="GPU tensors"):
        K.qk_norm_rope_append(q, k, k, ip, one, cache, one, ip, one, r)
    with pytest.raises(ValueError, match="GPU tensors"):
        K.paged_decode_rule(q, cache, ip, one, one, K.ScoreRule(), max_pages_per_row=1)
    with pytest.raises(ValueError, match="GPU tensors"):
        K.paged_prefill_rule(q, cache, ip, ip, one, one, K.ScoreRule(), max_qo_len=1)


@pytest.mark.parametrize("dim,theta,context,scale", [(128, 1e6, 32768, 4.0), (128, 5e5, 8192, 16.0), (64, 1e4, 4096, 16.0), (96, 1e4, 64, 4.0),
                                                     (128, 1e6, 1 << 20, 2.0)])
def test_yarn_over_the_pairs(dim, theta, context, scale):
    """The blend linear in the pair's index between the last pair of at least 32 turns and the first of at most one, as yarn
    checkpoints have it, found here by counting each pair's turns."""
    args = dict(rope_theta=theta, rope_scale=scale, old_context_len=float(context), scaling="yarn")
    got, factor = K.rotary_frequencies(dim, ramp="pairs", **args)
    plain, _ = K.rotary_frequencies(dim, rope_theta=theta)
    turns = [context * theta ** (-2 * j / dim) / (2 * math.pi) for j in range(dim)]
    first, last = max([j for j in range(dim) if turns[j] >= 32], default=0), min([j for j in range(dim) if turns[j] <= 1], default=dim - 1)
    assert factor == pytest.approx(0.1 * math.log(scale) + 1)
    for j, (f, g) in enumerate(zip(plain, got)):
        slow = min(max((j - first) / (last - first), 0), 1)
        assert g == pytest.approx(f * ((1 - slow) + slow / scale), rel=1e-12)
    same, _ = K.rotary_frequencies(dim, ramp="turns", **args)
    assert same == K.rotary_frequencies(dim, **args)[0] and same != got


@pytest.mark.parametrize("args,match", [
    (dict(ramp="index"), "ramp must be"), (dict(ramp="pairs"), "ramp must be"),
    (dict(ramp="pairs", scaling="llama31", low_freq_factor=1.0, high_freq_factor=4.0, old_context_len=10.0), "ramp must be"),
    (dict(ramp="pairs", scaling="yarn"), "old_context_len"), (dict(ramp="pairs", scaling="yarn", old_context_len=10.0, rope_theta=1.0), "over 1"),
])
def test_ramp_refusals(args, match):
    with pytest.raises(ValueError, match=match):
        K.rotary_frequencies(128, **args)


def test_padded_token_buffers_are_cut_all_the_same(lib):
    """Few real tokens over a long cache (max_qo_len tokens a row at most) in a buffer of more: what a buffer of the real size needs."""
    p = lib.delta_paged_prefill_rule_workspace_bytes
    for batch, most, pages in ((2, 7, 189), (1, 64, 563), (16, 1, 4096), (4, 40, 300)):
        for tokens in range(batch * most, 40 * pages, 37):
            assert p(tokens, batch, 12, 2, most, pages, 0) > 0 and p(tokens, batch, 32, 8, most, pages, 0) > 0, (tokens, batch, most, pages)
    for batch, most, tokens in ((12, 166, 12 * 166), (3, 40, 70), (30, 400, 30 * 400)):  # whole prompts are not
        assert p(tokens, batch, 40, 8, most, sum(-(-tokens // batch // 16) for _ in range(batch)), 0) == 0


@NO_GPU
@pytest.mark.parametrize("hkv", [17, 32, 40])
def test_decode_of_more_than_16_kv_heads(hkv):
    """Refused by the decode call, with every other argument right, and by name."""
    rejects("delta_paged_decode_rule", decode(hq=hkv, hkv=hkv), f"num_kv_heads {hkv} > 16 unsupported")
