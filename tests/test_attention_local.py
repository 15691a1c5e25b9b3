"""The 64-bit reference of the attention with window, sinks, position bias and dropout
(attention_reference.py) against autograd and differences; the bucket tables; the refusals of
the Python and C entry points (all on the CPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import attention_reference as ref
from genet5_amd import _lib, attention, residual

CASES = [
    dict(),
    dict(window=(3, 2), sinks=2),
    dict(window=(0, -1), sinks=0, slopes=[0.3, -0.1, 0.0, 1.0]),
    dict(window=(-1, 0), sinks=4, table=(8, 5)),
    dict(table=(16, 20), p=0.3),
    dict(window=(6, 6), sinks=1, slopes=[0.5, 0.25, 0.125, 0.0625], p=0.5),
]


def make(case, T=29, H=4, Hkv=2, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    kw = dict(case)
    if "table" in kw:
        nb, far = kw["table"]
        kw["table"], kw["max_distance"] = r(nb, H), far
    return r(T, H, 8), r(T, Hkv, 8), r(T, Hkv, 8), r(T, H, 8), kw


@pytest.mark.parametrize("case", CASES)
def test_reference_gradients_are_differences(case):
    """Central differences of <dout, out> along random directions in 64 bits."""
    cu = [0, 1, 1, 12, 29]
    q, k, v, do, kw = make(case)
    r = ref.attention(q, k, v, cu, 0.35, do, seed=99, **kw)

    def value(q, k, v, kw):
        return (do * ref.attention(q, k, v, cu, 0.35, seed=99, **kw)["out"]).sum().item()

    g = torch.Generator().manual_seed(7)
    for name, t in (("dq", q), ("dk", k), ("dv", v), ("dtable", kw.get("table"))):
        if t is None:
            continue
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        h = 1e-5
        sides = []
        for s in (h, -h):
            moved = dict(q=q, k=k, v=v)
            kk = dict(kw)
            if name == "dtable":
                kk["table"] = t + s * d
            else:
                moved[name[1]] = t + s * d
            sides.append(value(moved["q"], moved["k"], moved["v"], kk))
        diff = (sides[0] - sides[1]) / (2 * h)
        want = (r[name] * d).sum().item()
        # second order: h^2 = 1e-10 times third derivatives of order one; cancellation
        # 2^-52 / h = 2e-11 times the value
        assert abs(diff - want) <= 1e-6 * max(1.0, abs(want)), (name, diff, want)


def test_reference_without_options_is_the_oracle():
    import oracle
    q, k, v, _, _ = make({})
    cu = [0, 5, 5, 29]
    sl = [0.3, 0.2, 0.1, 0.05]
    want = oracle.attention_varlen(q.numpy(), k.numpy(), v.numpy(), cu, 0.35, sl)
    got = ref.attention(q, k, v, cu, 0.35, slopes=sl)["out"].numpy()
    np.testing.assert_allclose(got, want, rtol=1e-12, atol=1e-13)


@pytest.mark.parametrize("nb,far", [(32, 128), (16, 64), (64, 512), (8, 20), (32, 1000), (4, 2),
                                    (6, 7), (256, 1024)])
def test_bucket_tables(nb, far):
    t = attention.relative_buckets(nb, far)
    assert t.dtype == torch.int32 and t.shape == (2 * far + 1,)
    assert t.tolist() == [ref.bucket(r, nb, far) for r in range(-far, far + 1)]
    assert t[far] == 0 and t[0] == nb // 2 - 1 and t[2 * far] == nb - 1
    # steps of one distance up to half / 2, monotone beyond
    right = t[far + 1:].tolist()
    assert right == sorted(right)
    e = nb // 4
    assert [x - nb // 2 for x in right[: e - 1]] == list(range(1, e))


def test_bucket_borders_are_exact():
    # powers of two of the 32 / 128 table start buckets: log2(n / 8) * 2
    t = attention.relative_buckets(32, 128).tolist()
    side = lambda n: t[128 - n]
    assert [side(n) for n in (8, 15, 16, 31, 32, 63, 64, 127, 128)] == \
        [8, 9, 10, 11, 12, 13, 14, 15, 15]


@pytest.mark.parametrize("args,error,match", [
    (dict(causal=True), NotImplementedError, "causal"),
    (dict(window_size=(3,)), ValueError, "window_size"),
    (dict(window_size=(-2, 3)), ValueError, "window_size"),
    (dict(window_size=(1.5, 3)), ValueError, "window_size"),
    (dict(sink_tokens=-1), ValueError, "sink_tokens"),
    (dict(dropout_p=1.5), ValueError, "dropout_p"),
    (dict(dropout_p=-0.1), ValueError, "dropout_p"),
    (dict(dropout_p=float("nan")), ValueError, "dropout_p"),
    (dict(dropout_seed=-1), ValueError, "dropout_seed"),
    (dict(dropout_seed=2 ** 63), ValueError, "dropout_seed"),
    (dict(window_size=(4, 4)), RuntimeError, "GPU only"),
    (dict(relative_bias=torch.zeros(32, 2)), RuntimeError, "GPU only"),
    (dict(dropout_p=0.1), NotImplementedError, "dropout"),
])
def test_python_refusals(args, error, match):
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(error, match=match):
        attention.flash_attn_varlen_func(q, q, q, cu, cu, 4, 4, **args)


@pytest.mark.parametrize("bias,far,slopes,error,match", [
    (torch.zeros(32, 3), 128, None, ValueError, "shape"),
    (torch.zeros(32), 128, None, ValueError, "shape"),
    (torch.zeros(32, 2, dtype=torch.float16), 128, None, TypeError, "dtype"),
    (torch.zeros(31, 2), 128, None, ValueError, "num_buckets"),
    (torch.zeros(2, 2), 128, None, ValueError, "num_buckets"),
    (torch.zeros(32, 2), 8, None, ValueError, "max_distance"),
    (torch.zeros(32, 2), 1025, None, ValueError, "max_distance"),
    (torch.zeros(32, 2), 128, torch.zeros(2), ValueError, "exclude"),
    (None, 128, torch.zeros(3), ValueError, "alibi_slopes"),
    (None, 128, torch.zeros(2, dtype=torch.float64), ValueError, "alibi_slopes"),
])
def test_position_refusals(bias, far, slopes, error, match):
    with pytest.raises(error, match=match):
        attention._check_position(slopes, bias, far, 2, torch.device("cpu"))


def _shape(**kw):
    base = dict(n_seqs=1, max_seqlen=8, total_tokens=8, n_heads=4, n_kv_heads=2, head_dim=64)
    base.update(kw)
    s = _lib.AttnShape(**base)
    for f in ("q", "k", "v", "o"):
        setattr(s, f + "_token_stride", kw.get("stride", 256))
        setattr(s, f + "_head_stride", 64)
    return s


def _opts(**kw):
    o = _lib.AttnOptions(-1, -1, 0, 0, 0, 0, _lib.Dropout(0.0, 0, 0, 0), 0)
    for n, v in kw.items():
        if n == "p":
            o.dropout.p = v
        else:
            setattr(o, n, v)
    return o


FAKE = 1 << 20  # a 16-byte aligned address that no check reads


@pytest.mark.parametrize("opts,shape,ptrs,scale,match", [
    (dict(window_left=-2), {}, {}, 0.1, "window_left"),
    (dict(sink_tokens=-1), {}, {}, 0.1, "sink_tokens"),
    (dict(reserved=1), {}, {}, 0.1, "reserved"),
    (dict(p=1.5), {}, {}, 0.1, "dropout.p"),
    (dict(p=float("nan")), {}, {}, 0.1, "dropout.p"),
    ({}, {}, {}, float("nan"), "softmax_scale"),
    ({}, {}, {}, float("inf"), "softmax_scale"),
    ({}, dict(head_dim=32), {}, 0.1, "head_dim"),
    ({}, dict(n_kv_heads=3), {}, 0.1, "n_kv_heads"),
    ({}, dict(stride=250), {}, 0.1, "stride"),
    ({}, {}, dict(q=None), 0.1, "q is NULL"),
    ({}, {}, dict(cu=None), 0.1, "cu_seqlens is NULL"),
    ({}, {}, dict(k=FAKE + 2), 0.1, "aligned"),
    (dict(bias_buckets=8, bias_distance=4), {}, dict(table=FAKE), 0.1, "bucket_of"),
    (dict(bias_buckets=0, bias_distance=4), {}, dict(table=FAKE, lut=FAKE), 0.1, "bias_buckets"),
    (dict(bias_buckets=8, bias_distance=0), {}, dict(table=FAKE, lut=FAKE), 0.1, "bias_distance"),
    (dict(bias_buckets=8, bias_distance=1025), {}, dict(table=FAKE, lut=FAKE), 0.1,
     "bias_distance"),
    (dict(bias_buckets=8, bias_distance=4, bias_dtype=2), {}, dict(table=FAKE, lut=FAKE), 0.1,
     "bias_dtype"),
    (dict(bias_buckets=8, bias_distance=4), {}, dict(table=FAKE, lut=FAKE, slopes=FAKE), 0.1,
     "exclude"),
])
def test_c_refusals(g5lib, opts, shape, ptrs, scale, match):
    at = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, cu=FAKE, slopes=None, table=None, lut=None)
    at.update(ptrs)
    o, s = _opts(**opts), _shape(**shape)
    with pytest.raises(_lib.G5MoEError, match=match):
        _lib.call("g5moe_attn_local_fwd", at["q"], at["k"], at["v"], at["out"], at["cu"],
                  at["slopes"], at["table"], at["lut"], scale, None, None, None, ctypes.byref(o),
                  ctypes.byref(s), None)
    with pytest.raises(_lib.G5MoEError, match=match):
        _lib.call("g5moe_attn_bwd", FAKE, at["q"], at["k"], at["v"], at["out"], None, FAKE, at["cu"],
                  at["slopes"], at["table"], at["lut"], scale, FAKE, FAKE, FAKE, None, None, FAKE,
                  ctypes.byref(o), ctypes.byref(s), ctypes.byref(_shape(**shape)), None)


def test_c_backward_refusals(g5lib):
    o, s = _opts(), _shape()

    def call(dbias=None, grad=s, ws=FAKE, lse=FAKE):
        _lib.call("g5moe_attn_bwd", FAKE, FAKE, FAKE, FAKE, FAKE, None, lse, FAKE, None, None, None,
                  0.1, FAKE, FAKE, FAKE, dbias, None, ws, ctypes.byref(o), ctypes.byref(s),
                  ctypes.byref(grad), None)

    with pytest.raises(_lib.G5MoEError, match="softmax_lse"):   # out_low without it
        _lib.call("g5moe_attn_local_fwd", FAKE, FAKE, FAKE, FAKE, FAKE, None, None, None, 0.1,
                  None, FAKE, None, ctypes.byref(o), ctypes.byref(s), None)
    with pytest.raises(_lib.G5MoEError, match="aligned"):
        _lib.call("g5moe_attn_local_fwd", FAKE, FAKE, FAKE, FAKE, FAKE, None, None, None, 0.1,
                  FAKE, FAKE + 2, None, ctypes.byref(o), ctypes.byref(s), None)
    for kw, match in ((dict(dbias=FAKE), "dbias"), (dict(grad=_shape(total_tokens=9)), "strides"),
                      (dict(ws=None), "ws is NULL"), (dict(lse=None), "softmax_lse")):
        with pytest.raises(_lib.G5MoEError, match=match):
            call(**kw)


def test_c_empty_calls_do_nothing(g5lib):
    for kw in (dict(n_seqs=0), dict(max_seqlen=0), dict(total_tokens=0)):
        s = _shape(**kw)
        _lib.call("g5moe_attn_local_fwd", None, None, None, None, None, None, None, None, 0.1,
                  None, None, None, None, ctypes.byref(s), None)
        _lib.call("g5moe_attn_bwd", None, None, None, None, None, None, None, None, None, None, None,
                  0.1, None, None, None, None, None, None, None, ctypes.byref(s), ctypes.byref(s),
                  None)


def test_workspace_size_counts_what_the_backward_keeps(g5lib):
    n = ctypes.c_size_t()

    def size(o, **kw):
        _lib.call("g5moe_attn_bwd_workspace_size", ctypes.byref(o), ctypes.byref(_shape(**kw)),
                  ctypes.byref(n))
        return n.value

    # 40,000 tokens keep every workgroup busy without a split
    up = lambda floats: (floats * 4 + 255) // 256 * 256
    T, blocks = 40000, 20 * 16                     # 16 sequences of 2,500: 20 blocks each
    kw = dict(total_tokens=T, max_seqlen=2500, n_seqs=16, n_heads=8, n_kv_heads=4)
    base = 2 * up(8 * T) + up(4 * T // 64) + up(2 * blocks * 8)
    assert size(_opts(), **kw) == base
    assert size(_opts(p=0.1), **kw) == base + up(8 * T)
    assert size(_opts(bias_buckets=8, bias_distance=10), **kw) == \
        base + up(blocks * 8 * 21)
    # sinks under a window: their 128 keys' tiles in pieces of the window's length
    all_steps, window = 40 * 2 + 1, ((100 + 128) // 64 + 1) * 2 + 1
    pieces = -(-all_steps // window)
    assert size(_opts(window_left=50, window_right=50, sink_tokens=3), **kw) == \
        base + up(16 * pieces * 4 * 128 * 128)
    # few tokens: blocks of 64 keys, and each one's tiles split over workgroups
    kw.update(total_tokens=1000, max_seqlen=1000, n_seqs=1)
    assert size(_opts(), **kw) == 2 * up(8000) + up(4 * 16) + up(2 * 16 * 8) + up(2 * 4 * 1000 * 128)


@pytest.mark.parametrize("args,match", [
    (dict(p=1.5), "dropout.p"), (dict(d=0), "d 0"), (dict(rows=-1), "rows"),
    (dict(dtype=3), "dtype"), (dict(x=None), "x is NULL"), (dict(out=None), "out is NULL"),
    (dict(residual=None), "residual is NULL"), (dict(rows=1 << 42), "exceed"),
])
def test_dropout_add_c_refusals(g5lib, args, match):
    a = dict(x=FAKE, residual=FAKE, out=FAKE, p=0.1, rows=4, d=8, dtype=0)
    a.update(args)
    drop = _lib.make_dropout(a["p"], 5)
    with pytest.raises(_lib.G5MoEError, match=match):
        _lib.call("g5moe_dropout_add", a["x"], a["residual"], a["out"], ctypes.byref(drop), 1.0,
                  a["rows"], a["d"], a["dtype"], None)


@pytest.mark.parametrize("x,r,p,seed,error,match", [
    (torch.zeros(2, 4), torch.zeros(2, 4), 0.1, None, RuntimeError, "GPU only"),
])
def test_dropout_add_refuses_the_cpu(x, r, p, seed, error, match):
    with pytest.raises(error, match=match):
        residual.dropout_add(x, r, p, seed=seed)


def test_mask_statistics():
    """The generator's kept share and its independence along rows, columns and heads: within
    five standard deviations of a Bernoulli mask's."""
    keep, up = ref.keep_mask(np.arange(512), 1024, (123 << 32) + 77, 0.25)
    n = keep.size
    sd = math.sqrt(0.25 * 0.75 / n)
    assert abs(keep.mean() - 0.75) <= 5 * sd and up == 65536 / (65536 - 16384)
    x = keep - 0.75
    for a, b in ((x[:, 1:], x[:, :-1]), (x[1:], x[:-1]), (x[12:], x[:-12]), (x[:, 2:], x[:, :-2])):
        assert abs((a * b).mean()) <= 5 * 0.25 * 0.75 / math.sqrt(a.size)
