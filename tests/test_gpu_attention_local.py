"""The attention with window, sinks, bucketed position bias and dropout on the GPU, forward
and backward, against the 64-bit reference, every element within the bound that the
roundings allow (attention_reference.py)."""
import math

import pytest
import torch

import attention_reference as ref
from genet5_amd import attention

pytestmark = pytest.mark.gpu


def inputs(T, H, Hkv, seed, dev, scale=1.0, table=None, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, m=1.0: (torch.randn(*s, generator=g) * m).to(torch.bfloat16).to(dev)
    q, k, v, do = r(T, H, 64, m=scale), r(T, Hkv, 64, m=scale), r(T, Hkv, 64), r(T, H, 64)
    tab = None
    if table is not None:
        tab = torch.randn(table, H, generator=g).to(dtype).to(dev)
    return q, k, v, do, tab


def cu_tensor(cu, dev):
    return torch.tensor(cu, dtype=torch.int32, device=dev)


def run(q, k, v, do, cu, scale=0.125, table=None, max_len=None, grads=True, **kw):
    """out, lse and gradients through the public entry point."""
    q, k, v = (t.detach().requires_grad_(grads) for t in (q, k, v))
    tab = None if table is None else table.detach().requires_grad_(grads)
    top = max_len or max(b - a for a, b in zip(cu[:-1], cu[1:]))
    c = cu_tensor(cu, q.device)
    out, lse, _ = attention.flash_attn_varlen_func(q, k, v, c, c, top, top, softmax_scale=scale,
                                                   relative_bias=tab, return_attn_probs=True, **kw)
    res = dict(out=out.detach(), lse=lse)
    if grads:
        leaves = [t for t in (q, k, v, tab) if t is not None]
        for n, g in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, do)):
            res[n] = g
    torch.cuda.synchronize()
    return res


def compare(res, want, what, rows=None):
    """rows: those of the sequences (softmax_lse is not written behind them)."""
    T = want["out"].shape[0]
    for n in ("out", "dq", "dk", "dv", "dtable"):
        if n in res:
            ref.check(res[n], want, n, what)
    lse, got = want["lse"][:, :rows], res["lse"].double().cpu()[:, :rows]
    fin = torch.isfinite(lse)
    assert ((got - lse)[fin].abs() <= 2 * ref.SLACK * (1 + lse[fin].abs())).all()
    assert T == res["out"].shape[0]


EDGES = [1, 0, 31, 32, 33, 63, 64, 65, 127, 128, 129, 193, 257]


def packed(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


CASES = {
    "full": dict(),
    "full_alibi": dict(slopes=[0.5, 0.03, 0.0, -0.01]),
    "window": dict(window=(40, 17)),
    "window_zero": dict(window=(0, 0)),
    "window_sinks": dict(window=(20, 0), sinks=5),
    "past_only": dict(window=(-1, 0)),
    "future_and_sinks": dict(window=(0, -1), sinks=70),
    "wide_window": dict(window=(100, 130), sinks=130, slopes=[0.1, 0.2, 0.0, 0.004]),
    "buckets": dict(table=32, far=128),
    "buckets_near": dict(table=8, far=20),
    "buckets_far": dict(table=64, far=1000),
    "buckets_window": dict(table=16, far=64, window=(50, 50), sinks=3),
    "dropout": dict(p=0.3),
    "dropout_alibi": dict(p=0.1, slopes=[0.5, 0.03, 0.0, 0.01]),
    "all": dict(table=32, far=100, window=(70, 33), sinks=9, p=0.2),
}


def call_args(case, dev):
    kw = {}
    if "window" in case:
        kw["window_size"] = case["window"]
    if "sinks" in case:
        kw["sink_tokens"] = case["sinks"]
    if "slopes" in case:
        kw["alibi_slopes"] = torch.tensor(case["slopes"], device=dev)
    if "far" in case:
        kw["max_distance"] = case["far"]
    if "p" in case:
        kw.update(dropout_p=case["p"], dropout_seed=(77 << 33) + 5)
    return kw


def ref_args(case):
    return dict(window=case.get("window", (-1, -1)), sinks=case.get("sinks", 0),
                slopes=None if "slopes" not in case else torch.tensor(case["slopes"]),
                max_distance=case.get("far", 128), p=case.get("p", 0.0), seed=(77 << 33) + 5)


@pytest.mark.parametrize("hkv", [4, 2, 1])
@pytest.mark.parametrize("name", list(CASES))
def test_block_edges(cuda_device, name, hkv):
    """Lengths around every tile edge, and zero and one, in one packed call."""
    case = CASES[name]
    cu = packed(EDGES)
    print(f"attention local edges {name} hkv={hkv}", flush=True)
    q, k, v, do, tab = inputs(cu[-1], 4, hkv, 3, cuda_device, table=case.get("table"))
    res = run(q, k, v, do, cu, table=tab, **call_args(case, cuda_device))
    want = ref.attention(q, k, v, cu, 0.125, do, table=tab, **ref_args(case))
    compare(res, want, name)


@pytest.mark.parametrize("name", ["window_sinks", "wide_window", "buckets", "all", "full_alibi"])
@pytest.mark.parametrize("scale", [0.5, 0.0, -0.125])
def test_scales(cuda_device, name, scale):
    case = CASES[name]
    cu = [0, 300, 333]
    print(f"attention local scale {scale} {name}", flush=True)
    # scores of a scale of 0.5: sum |q_d k_d| scale stays below the reference's 25
    q, k, v, do, tab = inputs(cu[-1], 4, 2, 5, cuda_device, scale=0.7, table=case.get("table"))
    res = run(q, k, v, do, cu, scale=scale, table=tab, **call_args(case, cuda_device))
    want = ref.attention(q, k, v, cu, scale, do, table=tab, **ref_args(case))
    compare(res, want, f"{name} {scale}")


@pytest.mark.parametrize("name", ["window_sinks", "wide_window", "buckets", "buckets_near",
                                  "buckets_window", "all", "dropout_alibi", "past_only"])
def test_long_sequences(cuda_device, name):
    """Many tiles before, inside and after the window, plain and far ones among them."""
    case = CASES[name]
    cu = [0, 1111, 1111, 1650]
    print(f"attention local long {name}", flush=True)
    q, k, v, do, tab = inputs(cu[-1], 4, 2, 7, cuda_device, table=case.get("table"))
    res = run(q, k, v, do, cu, table=tab, max_len=1300, **call_args(case, cuda_device))
    want = ref.attention(q, k, v, cu, 0.125, do, table=tab, **ref_args(case))
    compare(res, want, name)


def test_fp32_table(cuda_device):
    cu = [0, 200, 329]
    q, k, v, do, tab = inputs(cu[-1], 4, 4, 9, cuda_device, table=32, dtype=torch.float32)
    res = run(q, k, v, do, cu, table=tab)
    assert res["dtable"].dtype == torch.float32
    compare(res, ref.attention(q, k, v, cu, 0.125, do, table=tab), "fp32 table")


def test_rows_that_see_nothing(cuda_device):
    """Bias entries of -inf: buckets that no query may use, and rows with no key left (the
    window keeps only the query itself, whose bucket is -inf): out 0, lse -inf, gradients 0
    and finite everywhere."""
    cu = [0, 150, 151, 251]
    q, k, v, do, tab = inputs(cu[-1], 4, 4, 11, cuda_device, table=32)
    t1 = tab.clone()
    t1[3] = t1[20] = -math.inf
    res = run(q, k, v, do, cu, table=t1)
    compare(res, ref.attention(q, k, v, cu, 0.125, do, table=t1), "-inf buckets")
    t2 = tab.clone()
    t2[0, 1] = -math.inf                       # distance 0, head 1
    res = run(q, k, v, do, cu, table=t2, window_size=(0, 0), sink_tokens=0)
    want = ref.attention(q, k, v, cu, 0.125, do, table=t2, window=(0, 0))
    compare(res, want, "empty rows")
    assert (res["out"][:, 1] == 0).all() and (res["lse"][1] == -math.inf).all()
    assert (res["dq"][:, 1] == 0).all() and (res["dk"][:, 1] == 0).all()
    # with sinks only queries past the first tokens see another key
    res = run(q, k, v, do, cu, table=t2, window_size=(0, 0), sink_tokens=1)
    want = ref.attention(q, k, v, cu, 0.125, do, table=t2, window=(0, 0), sinks=1)
    compare(res, want, "empty first rows")


def test_most_negative_bias_is_a_number(cuda_device):
    """The type's lowest value in a bucket masks it (exp underflows) without NaN."""
    cu = [0, 150]
    q, k, v, do, tab = inputs(150, 4, 4, 13, cuda_device, table=32, dtype=torch.float32)
    tab[5:9] = torch.finfo(torch.float32).min / 4
    res = run(q, k, v, do, cu, table=tab)
    compare(res, ref.attention(q, k, v, cu, 0.125, do, table=tab), "lowest")


def test_dropout_of_everything(cuda_device):
    cu = [0, 70]
    q, k, v, do, _ = inputs(70, 4, 2, 15, cuda_device)
    res = run(q, k, v, do, cu, dropout_p=1.0, dropout_seed=3)
    for n in ("out", "dq", "dk", "dv"):
        assert (res[n] == 0).all(), n


@pytest.mark.parametrize("name", ["full_alibi", "window_sinks", "buckets", "all"])
def test_rows_behind_the_last_sequence(cuda_device, name):
    """A padded batch: zeros in out and in every gradient behind the last sequence, whatever
    the inputs hold there, and the other rows as without the padding, bit for bit."""
    case = CASES[name]
    cu = [0, 70, 140]
    q, k, v, do, tab = inputs(200, 4, 2, 17, cuda_device, table=case.get("table"))
    kw = call_args(case, cuda_device)
    want = run(q[:140], k[:140], v[:140], do[:140], cu, table=tab, **kw)
    for t in (q, k, v, do):
        t[140:] = float("nan")
    got = run(q, k, v, do, cu, table=tab, **kw)
    for n in ("out", "dq", "dk", "dv"):
        assert torch.equal(got[n][:140], want[n]), n
        assert (got[n][140:] == 0).all(), n
    if tab is not None:
        assert torch.equal(got["dtable"], want["dtable"])


@pytest.mark.parametrize("name", ["full_alibi", "window_sinks", "buckets", "all"])
def test_other_sequences_stay_out(cuda_device, name):
    """NaN and infinities in the neighbours leave a sequence's results as they were: bit for
    bit, or for the full attention, whose key-norm bounds take whole 64-token blocks of the
    packed batch and only choose between loops of equal results, within the bound."""
    case = CASES[name]
    cu = [0, 70, 140, 333]
    q, k, v, do, _ = inputs(cu[-1], 4, 2, 19, cuda_device)
    tab = None if "table" not in case else inputs(1, 4, 2, 19, cuda_device,
                                                  table=case["table"])[4]
    kw = call_args(case, cuda_device)
    want = run(q, k, v, do, cu, table=tab, **kw)
    exact = ref.attention(q, k, v, cu, 0.125, do, table=tab, **ref_args(case))
    for a, b in ((0, 70), (140, 333)):
        q[a:b], k[a:b], v[a:b], do[a:b] = float("inf"), float("nan"), float("inf"), float("nan")
    got = run(q, k, v, do, cu, table=tab, **kw)
    for n in ("out", "dq", "dk", "dv"):
        if name == "full_alibi":
            ref.check(got[n][70:140], {m: exact[m][70:140] for m in (n, n + "_tol")}, n, name)
        else:
            assert torch.equal(got[n][70:140], want[n][70:140]), n


def test_tiles_out_of_the_window_stay_out(cuda_device):
    """Within a sequence: NaN keys and values in tiles that no key of the window touches."""
    cu = [0, 640]
    q, k, v, do, _ = inputs(640, 4, 4, 21, cuda_device)
    kw = dict(window_size=(64, 64))
    want = run(q, k, v, do, cu, **kw)
    k2, v2 = k.clone(), v.clone()
    k2[:128], v2[:128] = float("nan"), float("inf")
    got = run(q, k2, v2, do, cu, **kw)
    # queries from 256 on see keys from 192 on
    assert torch.equal(got["out"][256:], want["out"][256:])
    assert torch.equal(got["dq"][256:], want["dq"][256:])


def test_strided_views_and_broadcast_gradients(cuda_device):
    """q, k, v as views of one projection's output, dout as a transposed and as an expanded
    tensor: the same bits as from contiguous tensors."""
    T, H = 333, 4
    cu = [0, 100, 333]
    g = torch.Generator().manual_seed(23)
    qkv = torch.randn(T, 3, H, 64, generator=g).to(torch.bfloat16).to(cuda_device)
    q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
    do = torch.randn(H, T, 64, generator=g).to(torch.bfloat16).to(cuda_device).transpose(0, 1)
    kw = dict(window_size=(50, 60), sink_tokens=4)
    a = run(q, k, v, do, cu, **kw)
    b = run(q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous(), cu, **kw)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    one = torch.ones((), dtype=torch.bfloat16, device=cuda_device).expand(T, H, 64)
    a = run(q, k, v, one, cu, **kw)
    b = run(q, k, v, torch.ones(T, H, 64, dtype=torch.bfloat16, device=cuda_device), cu, **kw)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    # one key/value head expanded over the heads: its gradient is the heads' sum
    k1 = k[:, :1].contiguous().requires_grad_(True)
    c = cu_tensor(cu, cuda_device)
    out = attention.flash_attn_varlen_func(q, k1.expand(T, H, 64), v, c, c, 233, 233, **kw)
    (dk1,) = torch.autograd.grad(out, (k1,), do)
    assert dk1.shape == k1.shape and torch.isfinite(dk1).all()


def test_wide_token_strides(cuda_device):
    """Token strides too large for 32-bit offsets inside a tile (2^24 elements)."""
    T, stride = 70, 1 << 24
    q, k, v, do, _ = inputs(T, 1, 1, 25, cuda_device)
    buf = torch.empty((T * stride,), dtype=torch.bfloat16, device=cuda_device)
    wide = [buf.as_strided((T, 1, 64), (stride, 64, 1), storage_offset=64 * i) for i in range(4)]
    for w, t in zip(wide, (q, k, v, do)):
        w.copy_(t)
    a = run(q, k, v, do, [0, T], window_size=(30, 30))
    b = run(*wide, [0, T], window_size=(30, 30))
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_every_result_repeats(cuda_device):
    cu = packed([700, 33, 400])
    q, k, v, do, tab = inputs(cu[-1], 4, 2, 27, cuda_device, table=32)
    kw = call_args(CASES["all"], cuda_device)
    first = run(q, k, v, do, cu, table=tab, **kw)
    for _ in range(4):
        again = run(q, k, v, do, cu, table=tab, **kw)
        for n in first:
            assert torch.equal(first[n], again[n]), n


def test_seeds(cuda_device):
    """torch.manual_seed reproduces a drawn mask; calls draw new ones; forward and backward
    use the same one (the gradients of a repeated call are equal)."""
    cu = [0, 200]
    q, k, v, do, _ = inputs(200, 4, 4, 29, cuda_device)
    torch.manual_seed(5)
    a = run(q, k, v, do, cu, dropout_p=0.2)
    b = run(q, k, v, do, cu, dropout_p=0.2)
    torch.manual_seed(5)
    c = run(q, k, v, do, cu, dropout_p=0.2)
    assert not torch.equal(a["out"], b["out"])
    for n in a:
        assert torch.equal(a[n], c[n]), n


def test_inference_equals_the_training_forward(cuda_device):
    cu = [0, 300, 333]
    q, k, v, do, tab = inputs(333, 4, 2, 31, cuda_device, table=32)
    for name in ("window_sinks", "buckets", "all"):
        kw = call_args(CASES[name], cuda_device)
        t = tab if "table" in CASES[name] else None
        a = run(q, k, v, do, cu, table=t, **kw)
        b = run(q, k, v, do, cu, table=t, grads=False, **kw)
        assert torch.equal(a["out"], b["out"]) and torch.equal(a["lse"], b["lse"])
    # a long call without any option keeps the inference kernel's results under a gradient
    # (max_seqlen and the rows of the batch, not the lengths, decide)
    q, k, v, do, _ = inputs(2100, 4, 2, 32, cuda_device)
    a = run(q, k, v, do, cu, max_len=3000)
    compare(a, ref.attention(q, k, v, cu, 0.125, do), "long", rows=333)
    with torch.no_grad():
        c = cu_tensor(cu, cuda_device)
        b = attention.flash_attn_varlen_func(q, k, v, c, c, 3000, 3000, softmax_scale=0.125)
    assert torch.equal(a["out"][:333], b[:333])


def test_fixed_length_entry_point(cuda_device):
    B, L, H = 3, 100, 4
    q, k, v, do, tab = inputs(B * L, H, 2, 33, cuda_device, table=16)
    a = run(q, k, v, do, [0, 100, 200, 300], table=tab, window_size=(30, 20), max_distance=50)
    four = lambda t: t.view(B, L, *t.shape[1:])
    b = attention.flash_attn_func(four(q), four(k), four(v), softmax_scale=0.125,
                                  window_size=(30, 20), relative_bias=tab, max_distance=50)
    torch.cuda.synchronize()
    assert torch.equal(a["out"], b.reshape(B * L, H, 64))


def test_streams(cuda_device):
    """Two different calls on two streams at once, each with its own workspace."""
    cu = packed([600, 500])
    sets = [inputs(cu[-1], 4, 2, 35 + i, cuda_device, table=32) for i in range(2)]
    kws = [call_args(CASES["all"], cuda_device), dict()]
    want = [run(*s[:4], cu, table=s[4], **kw) for s, kw in zip(sets, kws)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    c = cu_tensor(cu, cuda_device)
    torch.cuda.synchronize()
    got = []
    for rep in range(3):
        for s, kw, st in zip(sets, kws, streams):
            with torch.cuda.stream(st):
                leaves = [t.detach().requires_grad_(True) for t in (*s[:3], s[4])]
                out = attention.flash_attn_varlen_func(
                    *leaves[:3], c, c, 600, 600, softmax_scale=0.125, relative_bias=leaves[3], **kw)
                got.append((out, torch.autograd.grad(out, leaves, s[3])))
    torch.cuda.synchronize()
    for i, (out, grads) in enumerate(got):
        w = want[i % 2]
        assert torch.equal(out, w["out"])
        for g, n in zip(grads, ("dq", "dk", "dv", "dtable")):
            assert torch.equal(g, w[n]), n


@pytest.mark.parametrize("name", ["full_alibi", "window_sinks", "all"])
def test_graph_replays(cuda_device, name):
    """Forward and backward captured in one graph, replayed on new inputs with eager work
    between the replays."""
    case = CASES[name]
    cu = packed([300, 77])
    kw = call_args(case, cuda_device)
    sets = [inputs(cu[-1], 4, 2, 41 + i, cuda_device, table=case.get("table")) for i in range(3)]
    want = [run(*s[:4], cu, table=s[4], **kw) for s in sets]
    static = [None if t is None else t.clone() for t in sets[0]]
    c = cu_tensor(cu, cuda_device)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (*static[:3], static[4])
                  if t is not None]
        out = attention.flash_attn_varlen_func(
            *leaves[:3], c, c, 300, 300, softmax_scale=0.125,
            relative_bias=leaves[3] if len(leaves) > 3 else None, **kw)
        return (out.detach(),) + torch.autograd.grad(out, leaves, static[3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for rep in range(6):
        s = sets[rep % 3]
        for a, b in zip(static, s):
            if a is not None:
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        w = want[rep % 3]
        for got, n in zip(res, ("out", "dq", "dk", "dv", "dtable")):
            assert torch.equal(got, w[n]), (rep, n)
        eager = run(*s[:4], cu, table=s[4], **kw)
        assert torch.equal(eager["dq"], w["dq"])


def test_nothing_to_do(cuda_device):
    """No sequence, or none with a token: zeros, and gradients of zeros."""
    q, k, v, do, tab = inputs(5, 4, 2, 51, cuda_device, table=32)
    for cu, top in (([0], 0), ([0, 0, 0], 0), ([0, 0], 4)):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, tab)]
        c = cu_tensor(cu, cuda_device)
        out = attention.flash_attn_varlen_func(*leaves[:3], c, c, top, top,
                                               relative_bias=leaves[3])
        grads = torch.autograd.grad(out, leaves, do)
        torch.cuda.synchronize()
        for t in (out, *grads):
            assert (t == 0).all()
    e = attention.flash_attn_varlen_func(q[:0], k[:0], v[:0], c, c, 0, 0, window_size=(3, 3))
    assert e.shape == (0, 4, 64)


@pytest.mark.parametrize("name", ["full_alibi", "window_sinks", "all"])
def test_many_sequences(cuda_device, name):
    """More sequences than lanes of a wave, empty ones among them (at both ends too), one long."""
    case = CASES[name]
    lens = [0, 0] + [(7 * i) % 11 for i in range(62)] + [300] + [(5 * i) % 4 for i in range(90)] + [0]
    cu = packed(lens)
    print(f"attention local {len(lens)} sequences {name}", flush=True)
    q, k, v, do, tab = inputs(cu[-1] + 5, 4, 2, 61, cuda_device, table=case.get("table"))
    res = run(q, k, v, do, cu, table=tab, **call_args(case, cuda_device))
    want = ref.attention(q, k, v, cu, 0.125, do, table=tab, **ref_args(case))
    compare(res, want, name, rows=cu[-1])
    assert (res["out"][cu[-1]:] == 0).all() and (res["dk"][cu[-1]:] == 0).all()


def test_a_cu_seqlens_that_breaks_its_contract_stays_in_bounds(cuda_device):
    """Falling, negative and too large entries are clamped on the device: no result is promised,
    but every access stays inside the buffers and the call ends."""
    q, k, v, do, tab = inputs(300, 4, 2, 63, cuda_device, table=32)
    for bad in ([0, 200, 100, 300], [0, -5, 400, 250], [50, 60, 2 ** 30, 300], [7, 7, 7, 7]):
        c = cu_tensor(bad, cuda_device)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, tab)]
        out = attention.flash_attn_varlen_func(*leaves[:3], c, c, 300, 300, window_size=(30, 30),
                                               sink_tokens=3, relative_bias=leaves[3])
        grads = torch.autograd.grad(out, leaves, do)
        torch.cuda.synchronize()
        assert out.shape == q.shape and grads[3].shape == tab.shape


def test_windows_beyond_every_position(cuda_device):
    """Windows, sinks and lengths that pass 32 bits mean all keys."""
    cu = [0, 200]
    q, k, v, do, _ = inputs(200, 4, 2, 65, cuda_device)
    want = run(q, k, v, do, cu, window_size=(1000, 1000))
    for w in ((2 ** 31 - 1, 2 ** 31), (2 ** 32 + 5, 2 ** 40)):
        got = run(q, k, v, do, cu, window_size=w, max_len=2 ** 33)
        for n in want:
            assert torch.equal(got[n], want[n]), n
    a = run(q, k, v, do, cu, window_size=(3, 3), sink_tokens=2 ** 32)
    for n in want:
        ref.check(a[n], {**ref.attention(q, k, v, cu, 0.125, do)}, n) if n != "lse" else None


def test_bucket_table_before_a_capture(cuda_device):
    """A table that no call has built yet is refused under capture, which stays valid."""
    q, k, v, do, tab = inputs(64, 4, 4, 67, cuda_device, table=32)
    c = cu_tensor([0, 64], cuda_device)
    attention._BUCKETS.pop((32, 777, q.device), None)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captur"):
            attention.flash_attn_varlen_func(q, k, v, c, c, 64, 64, relative_bias=tab,
                                             max_distance=777)
        out = q * 2
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, q * 2)


def test_fixed_length_calls_of_changing_sizes_under_graphs(cuda_device):
    """A captured fixed-length call keeps its own sequence bounds when calls of other sizes
    come between its replays."""
    g = torch.Generator().manual_seed(69)
    r = lambda B, L: torch.randn(B, L, 4, 64, generator=g).to(torch.bfloat16).to(cuda_device)
    x = r(3, 70)
    f = lambda t: attention.flash_attn_func(t, t, t, window_size=(20, 20))
    with torch.no_grad():
        want = f(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f(x)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(x)
        for rep in range(5):
            f(r(2 + rep, 33 + rep))
            junk = [torch.full((4,), 2 ** 30, dtype=torch.int32, device=cuda_device)
                    for _ in range(64)]
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), rep
            del junk


@pytest.mark.parametrize("name,L", [("full", 2100), ("full_alibi", 600), ("window_sinks", 300),
                                    ("buckets", 77), ("dropout", 600)])
def test_what_the_rounding_of_out_left_over(cuda_device, name, L):
    """out_low is off out by at most half a step of bf16 (2^-8 relative), and out + out_low is
    nearer to the 64-bit value than out (2,100 tokens without an option: the full attention's
    kernel)."""
    case = CASES[name]
    cu = [0, L, L + 40]
    print(f"attention out_low {name} {L}", flush=True)
    q, k, v, do, tab = inputs(cu[-1], 4, 2, 21, cuda_device, table=case.get("table"))
    kw = call_args(case, cuda_device)
    out, lse, low, _ = attention.attn_local_fwd(
        q, k, v, cu_tensor(cu, cuda_device), L, 0.125, kw.get("alibi_slopes"), tab,
        kw.get("max_distance", 128), kw.get("window_size", (-1, -1)), kw.get("sink_tokens", 0),
        kw.get("dropout_p", 0.0), kw.get("dropout_seed", 0), for_backward=True)
    assert torch.equal(out, run(q, k, v, do, cu, grads=False, table=tab, **kw)["out"]) or \
        name in ("full", "full_alibi")   # inference without options keeps its kernel
    assert (low.double().abs() <= out.double().abs() * 2.0 ** -8).all()
    want = ref.attention(q, k, v, cu, 0.125, None, table=tab, **ref_args(case))["out"]
    a, b = (((x.double().cpu() - want).norm() / want.norm()).item()
            for x in (out, out.double() + low.double()))
    assert b < a, (a, b)


@pytest.mark.parametrize("name", ["alibi", "alibi_dropout", "buckets"])
def test_gradients_carry_two_roundings(cuda_device, name):
    """dq and dk against the formula in 64 bits, by norm.  A value's rounding to bf16 has the
    relative root mean square 1.66e-3: the error of a mantissa m in [1, 2) is uniform in
    +-2^-8, its root mean square 2^-8 / sqrt 3, and the mean of 1 / m^2 is 3 / (8 ln 2) over
    the density 1 / (m ln 2).  dS and the result are rounded: 2.35e-3; 6 % are left for the
    probabilities' rounding in out.  With the rounding of out itself in delta it would be
    2.6e-3."""
    H, L = 12, 600
    case = {"alibi": dict(slopes=attention.alibi_slopes(H)),
            "alibi_dropout": dict(slopes=attention.alibi_slopes(H), p=0.1),
            "buckets": dict(table=32, far=128)}[name]
    cu = [0, L]
    print(f"attention two roundings {name}", flush=True)
    q, k, v, do, tab = inputs(L, H, H, 22, cuda_device, table=case.get("table"))
    res = run(q, k, v, do, cu, table=tab, **call_args(case, cuda_device))
    want = ref.attention(q, k, v, cu, 0.125, do, table=tab, **ref_args(case))
    for n in ("dq", "dk"):
        rel = ((res[n].double().cpu() - want[n]).norm() / want[n].norm()).item()
        print(n, rel, flush=True)
        assert rel <= 2.5e-3, (n, rel)


@pytest.mark.parametrize("slopes", [None, [0.5, 0.03]])
def test_sinks_longer_than_most_sequences(cuda_device, slopes):
    """Many short sequences and one long one with 700 sinks: the sinks' key blocks are not
    numbered for every sequence."""
    lens = [i % 4 for i in range(600)] + [1500] + [3, 0, 2] * 100
    cu = packed(lens)
    print(f"attention sinks of many sequences {slopes}", flush=True)
    case = dict(window=(20, 20), sinks=700)
    if slopes:
        case["slopes"] = slopes
    q, k, v, do, _ = inputs(cu[-1], 2, 1, 23, cuda_device)
    res = run(q, k, v, do, cu, **call_args(case, cuda_device))
    want = ref.attention(q, k, v, cu, 0.125, do, **ref_args(case))
    compare(res, want, "sinks of many sequences")


@pytest.mark.parametrize("buckets,far,p,lens", [(8, 20, 0.25, (1500, 1100)), (16, 64, 0.0, (2300,)),
                                                (32, 128, 0.0, (700, 900))])
def test_bias_gradient_where_one_bucket_holds_most(cuda_device, buckets, far, p, lens):
    """The end buckets hold most of a row's probability, and their terms nearly cancel, so an
    error of delta shows there: by norm at most half more than the result's own rounding to
    bf16 (1.66e-3)."""
    case = dict(table=buckets, far=far, **(dict(p=p) if p else {}))
    cu = packed(lens)
    print(f"attention bias gradient {buckets} {far} {lens}", flush=True)
    q, k, v, do, tab = inputs(cu[-1], 4, 2, 24, cuda_device, table=buckets)
    res = run(q, k, v, do, cu, table=tab, **call_args(case, cuda_device))
    want = ref.attention(q, k, v, cu, 0.125, do, table=tab, **ref_args(case))["dtable"]
    rel = ((res["dtable"].double().cpu() - want).norm() / want.norm()).item()
    print("dtable", rel, flush=True)
    assert rel <= 2.5e-3


def test_second_derivatives_are_refused(cuda_device):
    q, k, v, do, _ = inputs(70, 4, 2, 25, cuda_device)
    q = q.requires_grad_()
    c = cu_tensor([0, 70], cuda_device)
    out = attention.flash_attn_varlen_func(q, k, v, c, c, 70, 70)
    plain = torch.autograd.grad(out, q, do, retain_graph=True)[0]
    dq = torch.autograd.grad(out, q, do, create_graph=True)[0]
    assert torch.equal(plain, dq)
    with pytest.raises(RuntimeError):  # dq has no graph: nothing else of it required a gradient
        torch.autograd.grad(dq.float().sum(), q)


@pytest.mark.parametrize("name", ["window_sinks", "dropout_alibi", "buckets"])
def test_saved_tensors_that_come_back_with_other_strides(cuda_device, name):
    """Hooks that keep saved tensors elsewhere give back contiguous copies of strided views."""
    case = CASES[name]
    cu = [0, 150, 380]
    print(f"attention saved tensors {name}", flush=True)
    _, _, _, do, tab = inputs(cu[-1], 4, 4, 26, cuda_device, table=case.get("table"))
    qkv = inputs(cu[-1], 12, 12, 27, cuda_device)[0].requires_grad_()
    c = cu_tensor(cu, cuda_device)

    def grad():
        q, k, v = qkv[:, :4], qkv[:, 4:8], qkv[:, 8:]
        out = attention.flash_attn_varlen_func(q, k, v, c, c, 230, 230, relative_bias=tab,
                                               **call_args(case, cuda_device))
        return torch.autograd.grad(out, qkv, do)[0]

    want = grad()
    with torch.autograd.graph.save_on_cpu():
        got = grad()
    assert torch.equal(got, want)
